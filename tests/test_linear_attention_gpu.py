"""Linear attention from and into fp32 states against its plain 64-bit form: types, decays, sizes, strides, slots, unusual values."""

import pytest
import torch

from linquant_amd.kernels.zoo.linear_attention import linear_attention_prompt, linear_attention_step
from tests.attention_cases import attention_inputs, attention_ref, out_rel, state_rel
from tests.serving_cases import assert_near, starts_of

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
NAN, INF = float("nan"), float("inf")


def _to(cuda, *ts):
    return [None if t is None else t.to(cuda) for t in ts]


def _check_prompt(cuda, lens, H, K, V, dtype, g="token", seed=0, scale=None, packed=True, with_state=True, g_mean=2.0):
    T, n = sum(lens), len(lens)
    q, k, v, gd = attention_inputs(T, H, K, V, dtype, g, seed, g_mean)
    gen = torch.Generator().manual_seed(seed + 1)
    state = torch.randn(n + 2, H, K, V, generator=gen)
    slots = torch.randperm(n + 2, generator=gen)[:n].to(torch.int32)
    first = state[slots.long()] if with_state else torch.zeros(n, H, K, V)
    s = K ** -0.5 if scale is None else scale
    o, mag, S, Sm, most = attention_ref(q, k, v, gd, s, lens, first)
    dq, dk, dv, dg, dst, dsl = _to(cuda, q, k, v, gd, state, slots)
    if not packed:
        dq, dk, dv = (t.unflatten(0, (n, lens[0])) for t in (dq, dk, dv))
        dg = dg if dg is None or dg.dim() == 1 else dg.unflatten(0, (n, lens[0]))
    got = linear_attention_prompt(dq, dk, dv, dg, scale=scale, state=dst if with_state else None, slots=dsl if with_state else None,
                                  seq_starts=starts_of(lens, cuda) if packed else None)
    assert got.shape == dv.shape and got.dtype == dtype and got.is_contiguous()
    assert_near(got.flatten(0, -3), o, mag, out_rel(lens, most, dtype), "o")
    if with_state:
        want, wm = state.double().clone(), state.double().abs()
        want[slots.long()], wm[slots.long()] = S, Sm
        assert_near(dst, want, wm, state_rel(lens, most), "state")
        rest = [i for i in range(n + 2) if i not in slots.tolist()]
        assert torch.equal(dst[rest].cpu(), state[rest])


@pytest.mark.parametrize("K,V", [(8, 8), (64, 64), (128, 128), (128, 64), (64, 200), (96, 40), (136, 72), (256, 32), (40, 328)])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("g", ["token", "head", "none"])
def test_prompt_dims(cuda, K, V, dtype, g):
    _check_prompt(cuda, [70, 0, 1, 129], 3, K, V, dtype, g, seed=K + V)


@pytest.mark.parametrize("lens", [[1], [2], [63], [64], [65], [127], [128], [200], [5, 64, 0, 0, 192, 1], [0, 0, 3], [1] * 70, [300, 17, 64]])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_prompt_lengths(cuda, lens, dtype):
    _check_prompt(cuda, lens, 2, 64, 64, dtype, seed=len(lens))


@pytest.mark.parametrize("L", [1, 64, 100, 260])
@pytest.mark.parametrize("g", ["token", "head", "fast", "none"])
@pytest.mark.parametrize("with_state", [True, False])
def test_prompts_of_one_length(cuda, L, g, with_state):
    _check_prompt(cuda, [L] * 3, 4, 128, 128, BF16, g, seed=L, packed=False, with_state=with_state)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("H,lens", [(1, [2500]), (2, [1900, 30]), (3, [1024, 1024]), (1, [64 * 31])])
@pytest.mark.parametrize("g", ["token", "head"])
def test_long_prompts_of_few_heads(cuda, H, lens, dtype, g):
    """Few heads: prompts are cut into segments."""
    _check_prompt(cuda, lens, H, 64, 64, dtype, g, seed=7, g_mean=4.0)


def test_long_prompts_of_one_length(cuda):
    _check_prompt(cuda, [1500, 1500], 2, 128, 128, F16, "head", seed=8, packed=False)
    _check_prompt(cuda, [1500, 1500], 2, 128, 128, BF16, "none", seed=9, packed=False, with_state=False)


def test_prompt_in_parts_and_steps(cuda):
    """A prompt in two calls, then single tokens: the whole prompt's outputs and state."""
    H, K, V, lens = 3, 128, 64, [150]
    q, k, v, g = attention_inputs(150, H, K, V, F16, seed=3)
    o, mag, S, Sm, most = attention_ref(q, k, v, g, K ** -0.5, lens, torch.zeros(1, H, K, V))
    dq, dk, dv, dg = _to(cuda, q, k, v, g)
    state = torch.zeros(1, H, K, V, device=cuda)
    parts = [linear_attention_prompt(*(t[None, a:b] for t in (dq, dk, dv, dg)), state=state)[0] for a, b in ((0, 77), (77, 140))]
    parts += [linear_attention_step(state, *(t[i:i + 1] for t in (dq, dk, dv, dg))) for i in range(140, 150)]
    assert_near(torch.cat(parts), o, mag, out_rel(lens, most, F16), "o")
    assert_near(state, S, Sm, state_rel(lens, most), "state")


@pytest.mark.parametrize("B,H,K,V", [(1, 1, 8, 8), (3, 5, 96, 40), (2, 4, 128, 128), (70, 16, 128, 128), (40, 20, 256, 72), (5, 300, 64, 200), (600, 2, 40, 328), (260, 3, 64, 64), (300, 2, 200, 16)])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("g", ["token", "head", "none"])
def test_step(cuda, B, H, K, V, dtype, g):
    q, k, v, gd = attention_inputs(B, H, K, V, dtype, g, seed=B)
    gen = torch.Generator().manual_seed(5)
    state = torch.randn(B + 3, H, K, V, generator=gen)
    slots = torch.randperm(B + 3, generator=gen)[:B].to(torch.int32)
    gb = gd if gd is None or gd.dim() == 2 else gd.expand(B, H)
    o, mag, S, Sm, _ = attention_ref(q, k, v, gb, 0.3, [1] * B, state[slots.long()])
    dst = state.to(cuda)
    got = linear_attention_step(dst, *_to(cuda, q, k, v, gd), scale=0.3, slots=slots.to(cuda))
    # decay by 2 units of 2^-24 and its product, k v and the sum a rounding each; q scaled, its product, sums of up to 256
    assert_near(got, o, mag, 2.0 ** -24 * 16 + 2.0 ** -24 * 256, "o")
    want, wm = state.double().clone(), state.double().abs()
    want[slots.long()], wm[slots.long()] = S, Sm
    assert_near(dst, want, wm, 2.0 ** -24 * 6, "state")


def test_strides_and_types_of_g(cuda):
    """Slices of a projection, heads in another order, a state with room between its slots; g in 16 bits reads as its value."""
    H, K, V, n, L = 4, 64, 72, 2, 90
    gen = torch.Generator().manual_seed(1)
    wide = torch.randn(n, L, H * (2 * K + V) + 24, generator=gen).to(BF16).to(cuda)
    q, k, v = (t.unflatten(-1, (H, -1)) for t in wide[..., 8:-16].split([H * K, H * K, H * V], -1))
    q = q.flip(2)                                                                       # copied by the wrapper
    g = torch.nn.functional.logsigmoid(torch.randn(L, n, H + 3, generator=gen)).to(BF16).to(cuda).transpose(0, 1)[..., 2:2 + H]
    big = torch.randn(3, 2, H, K, V, generator=gen).to(cuda)
    keep = big.clone()
    state = big[:, 1]
    slots = torch.tensor([2, 0], dtype=torch.int32, device=cuda)
    o, mag, S, Sm, most = attention_ref(*(t.cpu().flatten(0, 1) for t in (q, k, v)), g.cpu().reshape(-1, H), K ** -0.5, [L] * n, state[slots.long()].cpu())
    got = linear_attention_prompt(q, k, v, g, state=state, slots=slots)
    assert_near(got.flatten(0, 1), o, mag, out_rel([L], most, BF16), "o")
    assert_near(state[slots.long()], S, Sm, state_rel([L], most), "state")
    assert torch.equal(big[:, 0], keep[:, 0]) and torch.equal(big[1], keep[1])
    one = state.clone()
    want = linear_attention_step(one, q[:, 0].contiguous(), k[:, 0].contiguous(), v[:, 0].contiguous(), g[:, 0].contiguous(), slots=slots)
    assert torch.equal(linear_attention_step(state, q[:, 0], k[:, 0], v[:, 0], g[:, 0], slots=slots), want) and torch.equal(state[slots.long()], one[slots.long()])


def test_slots_padding_and_out_of_range(cuda):
    H, K, V = 2, 64, 64
    q, k, v, g = _to(cuda, *attention_inputs(30, H, K, V, F16, seed=4))
    state = torch.randn(3, H, K, V, device=cuda)
    before = state.clone()
    slots = torch.tensor([-1, 9, 1], dtype=torch.int32, device=cuda)
    starts = starts_of([10, 10, 8], cuda)
    got = linear_attention_prompt(q, k, v, g, state=state, slots=slots, seq_starts=starts)
    assert torch.isnan(got[10:20]).all() and not torch.isnan(got[:10]).any() and not torch.isnan(got[20:28]).any()
    assert torch.equal(got[:10], linear_attention_prompt(q[None, :10], k[None, :10], v[None, :10], g[None, :10])[0])
    assert torch.equal(state[[0, 2]], before[[0, 2]]) and not torch.equal(state[1], before[1])
    after = state.clone()
    y = linear_attention_step(state, q[:3], k[:3], v[:3], g[:3], slots=slots)
    assert (y[0] == 0).all() and torch.isnan(y[1]).all() and not torch.isnan(y[2]).any()
    assert torch.equal(state[[0, 2]], after[[0, 2]]) and not torch.equal(state[1], after[1])
    assert linear_attention_prompt(q[None, :0], k[None, :0], v[None, :0], None, state=state[:1]).shape == (1, 0, H, V)


def test_tokens_outside_every_prompt_do_not_matter(cuda):
    H, K, V = 2, 128, 64
    q, k, v, g = _to(cuda, *attention_inputs(200, H, K, V, BF16, seed=5))
    starts = starts_of([60, 40], cuda, first=30)
    want = linear_attention_prompt(q, k, v, g, seq_starts=starts)[30:130].clone()
    for t in (q, k, v, g):
        t[:30], t[130:] = NAN, INF
    assert torch.equal(linear_attention_prompt(q, k, v, g, seq_starts=starts)[30:130], want)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("what", ["q", "k", "v", "g", "state"])
@pytest.mark.parametrize("value", [NAN, INF])
@pytest.mark.parametrize("at", [0, 70, 100])
def test_values_that_are_no_numbers(cuda, dtype, what, value, at):
    """They reach what the formula has them reach, and nothing in front of them, in another head or in another sequence."""
    H, K, V, lens = 2, 64, 72, [130, 80]
    q, k, v, g = attention_inputs(210, H, K, V, dtype, seed=6)
    state = torch.randn(2, H, K, V, generator=torch.Generator().manual_seed(6))
    if what == "state":
        state[0, 1, 3, 5] = value
    elif what == "g":
        if value == INF:
            value = -INF                                                                # a decay to nothing
        g[at, 1] = value
    else:
        {"q": q, "k": k, "v": v}[what][at, 1, 5] = value
    o, mag, S, Sm, most = attention_ref(q, k, v, g, K ** -0.5, lens, state)
    bad = lambda t: torch.where(torch.isfinite(t), t, NAN)  # noqa: E731
    dst = state.to(cuda)
    got = linear_attention_prompt(*_to(cuda, q, k, v, g), state=dst, seq_starts=starts_of(lens, cuda))
    most = min(most, 64 * 160.0)
    assert_near(bad(got.cpu()), bad(o), bad(mag), out_rel(lens, most + 160, dtype), "o")
    assert_near(bad(dst.cpu()), bad(S), bad(Sm), state_rel(lens, most + 160), "state")


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_decays_from_nothing_to_all(cuda, dtype):
    """Decays that leave nothing, sums far below the smallest number, above zero (no decay), and denormal ones."""
    H, K, V, lens = 6, 64, 64, [140]
    q, k, v, _ = attention_inputs(140, H, K, V, dtype, "none", seed=11)
    g = torch.zeros(140, H)
    g[:, 0], g[:, 1], g[:, 2], g[:, 3] = -1e30, -30.0, 5.0, -1e-42
    g[::7, 4], g[::64, 5] = -1e4, -INF
    o, mag, S, Sm, _ = attention_ref(q, k, v, g, 1.0, lens, torch.ones(1, H, K, V))
    dst = torch.ones(1, H, K, V, device=cuda)
    got = linear_attention_prompt(*_to(cuda, q[None], k[None], v[None], g[None]), scale=1.0, state=dst)
    # a factor below 2^-160 counts as 2^-160, so sums of log2 over 64 tokens reach 160 a token
    assert_near(got[0], o, mag, out_rel(lens, 160.0 * 64 / 8, dtype), "o")
    assert_near(dst, S, Sm, state_rel(lens, 160.0 * 64 / 8), "state")


def test_fp16_sizes_far_apart(cuda):
    """Nothing overflows or underflows in fp16 that does not in the formula: channels and states of very different sizes."""
    H, K, V, lens = 2, 64, 64, [150]
    q, k, v, g = attention_inputs(150, H, K, V, F16, "token", seed=12, g_mean=5.0)
    q, k = (q.float() * 2.0 ** -6).half(), (k.float() * 2.0 ** 6).half()
    v[:, :, 3] = (v[:, :, 3].float() * 2.0 ** 12).half()
    v[:, :, 4] = (v[:, :, 4].float() * 2.0 ** -12).half()
    state = torch.randn(1, H, K, V, generator=torch.Generator().manual_seed(1))
    state[..., 3] *= 2.0 ** 30
    state[..., 4] *= 2.0 ** -20
    o, mag, S, Sm, most = attention_ref(q, k, v, g, 2.0 ** -16, lens, state)
    dst = state.to(cuda)
    got = linear_attention_prompt(*_to(cuda, q[None], k[None], v[None], g[None]), scale=2.0 ** -16, state=dst)
    assert_near(got[0], o, mag, out_rel(lens, most, F16), "o")
    assert_near(dst, S, Sm, state_rel(lens, most), "state")
    big = _to(cuda, *(torch.full((1, 70, 1, 64), 60000.0).half() for _ in range(3)))
    y = linear_attention_prompt(*big, scale=2.0 ** -46, state=(s := torch.zeros(1, 1, 64, 64, device=cuda)))
    want = 60000.0 ** 2 * torch.arange(1, 71).double()
    assert_near(y[0, :, 0, 0], want * 60000.0 * 64 * 2.0 ** -46, want * 60000.0 * 64 * 2.0 ** -46, out_rel([70], 0, F16), "o")
    assert_near(s[0, 0], want[-1].expand(64, 64), want[-1].expand(64, 64), state_rel([70], 0), "state")


def test_capture_replay_and_streams(cuda):
    H, K, V = 4, 128, 128
    q, k, v, g = _to(cuda, *attention_inputs(300, H, K, V, BF16, seed=13))
    starts = starts_of([200, 100], cuda)
    state, expect = torch.zeros(2, H, K, V, device=cuda), torch.zeros(2, H, K, V, device=cuda)
    sq = [t[:2].clone() for t in (q, k, v, g)]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        warm = state.clone()
        linear_attention_prompt(q, k, v, g, state=warm, seq_starts=starts)
        linear_attention_step(warm, *sq)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a = linear_attention_prompt(q, k, v, g, state=state, seq_starts=starts)
        b = linear_attention_step(state, *sq)
    for i in range(4):
        v.mul_(0.5 + 0.25 * i)
        graph.replay()
        torch.cuda.synchronize()
        wa = linear_attention_prompt(q, k, v, g, state=expect, seq_starts=starts)
        wb = linear_attention_step(expect, *sq)
        assert torch.equal(a, wa) and torch.equal(b, wb) and torch.equal(state, expect)


def test_states_past_32_bits(cuda):
    """Slots whose offset in entries does not fit 32 bits."""
    H, K, V = 32, 128, 128
    n = 2 ** 31 // (H * K * V) + 3
    state = torch.empty(n, H, K, V, device=cuda)
    q, k, v, g = _to(cuda, *attention_inputs(70, H, K, V, BF16, seed=14))
    slots = torch.tensor([n - 1, 1], dtype=torch.int32, device=cuda)
    small = torch.randn(2, H, K, V, device=cuda)
    state[n - 1], state[1] = small[0], small[1]
    small = small.clone()
    for call in (lambda s, sl: linear_attention_prompt(q, k, v, g, state=s, slots=sl, seq_starts=starts_of([40, 30], cuda)),
                 lambda s, sl: linear_attention_step(s, q[:2], k[:2], v[:2], g[:2], slots=sl)):
        assert torch.equal(call(state, slots), call(small, None))
        assert torch.equal(state[slots.long()], small)
