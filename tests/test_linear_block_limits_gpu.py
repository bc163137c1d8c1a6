"""A linear attention block's operators at the limits of what they take: sizes and magnitudes where a variant, a unit or a workspace changes."""

import pytest
import torch

from linquant_amd.kernels.zoo.linear_attention import linear_attention_prompt
from linquant_amd.w8a8_linear import LowRankAdapters, W8A8Linear
from tests.attention_cases import attention_inputs, attention_ref, out_rel, state_rel
from tests.serving_cases import assert_near, starts_of

pytestmark = pytest.mark.gpu

F16, BF16, F32, I8, I32 = torch.float16, torch.bfloat16, torch.float32, torch.int8, torch.int32


def test_widths_behind_the_padding_are_told_apart(cuda):
    """250 features lie in rows of 256 bytes, as 256 do."""
    lin = {k: W8A8Linear(torch.ones(8, k, dtype=I8), torch.ones(8)).to(cuda) for k in (250, 256)}
    ad = {k: LowRankAdapters(torch.ones(2, 4, k).half(), torch.ones(2, 8, 4).half()).to(cuda) for k in (250, 256)}
    ids = torch.zeros(3, dtype=I32, device=cuda)
    for w in (250, 256):
        for a in (250, 256):
            for k in (250, 256):
                x, codes = torch.ones(3, k, device=cuda).half(), torch.ones(3, k, dtype=I8, device=cuda)
                for call in (lambda: lin[w](x, adapters=ad[a], ids=ids), lambda: lin[w].forward_int8(codes, torch.ones(3, device=cuda), adapters=ad[a], ids=ids)):
                    if w == a == k:
                        assert call().shape == (3, 8)
                    else:
                        with pytest.raises(AssertionError):
                            call()


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("half", [0, 4])
def test_large_values_beside_one_that_is_no_number(cuda, half, value):
    """fp16, a small chunk in front of a large one, whose large values of v stand in one half of the wave's tokens with a value that is no number
    behind them: the tokens in front of it keep their outputs."""
    H, K, V, L = 1, 64, 64, 200
    q, k, v, _ = attention_inputs(L, H, K, V, F16, "none", seed=half)
    v = (v.float().clamp(-2, 2) * 1e-4).half()
    v[[t for t in range(64, 128) if t % 8 // 4 * 4 == half]] = 20.0
    v[64 + 56 + half, 0, 5] = value
    o, mag, S, Sm, most = attention_ref(q, k, v, None, 0.125, [L], torch.zeros(1, H, K, V))
    bad = lambda t: torch.where(torch.isfinite(t), t, float("nan"))  # noqa: E731
    state = torch.zeros(1, H, K, V, device=cuda)
    got = linear_attention_prompt(q[None].to(cuda), k[None].to(cuda), v[None].to(cuda), scale=0.125, state=state)
    assert_near(bad(got[0].cpu()), bad(o), bad(mag), out_rel([L], most, F16), "o")
    assert_near(bad(state.cpu()), bad(S), bad(Sm), state_rel([L], most), "state")


def _weights_off(q, k, v, g, scale, rel):
    """What outputs lose where weighted q . k is off by ``rel`` of the largest of its token's row within the chunk of 64: (T, H, V)."""
    T, H = q.shape[:2]
    g = torch.zeros(T, H).double() if g is None else g.double().expand(T, H)
    off = torch.zeros(T, H, v.shape[2]).double()
    for a in range(0, T, 64):
        c = torch.cumsum(g[a:a + 64], 0)
        w = abs(scale) * (q[a:a + 64].double()[:, None] * k[a:a + 64].double()[None]).sum(-1).abs() * torch.exp((c[:, None] - c[None]).clamp(max=0.0))
        w = w * torch.ones(w.shape[:2]).tril().double()[..., None]
        size = torch.cumsum(v[a:a + 64].double().abs(), 0)                              # of the tokens up to each one
        off[a:a + 64] = rel * w.amax(1)[..., None] * size
    return off


@pytest.mark.parametrize("L", [64, 128, 200])
@pytest.mark.parametrize("size", [0.01, 1e-4])
@pytest.mark.parametrize("near", [2.0 ** -4, 2.0 ** -8, 1.0])
def test_fp16_old_tokens_of_large_v(cuda, L, size, near):
    """Weighted q . k of tokens whose v is far above the later ones' keeps its bits while they count; q and k of several sizes."""
    H, K, V = 2, 64, 64
    gen = torch.Generator().manual_seed(L)
    rn = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    q, k = (near * (1 + 0.1 * rn(L, H, K))).half(), (2.0 ** -5 * (1 + 0.1 * rn(L, H, K))).half()
    v = (size * rn(L, H, V)).half()
    v[torch.arange(L) % 64 < 24] = 200.0
    g = torch.full((L, H), -0.6)
    g[:, 1] = -0.3
    o, mag, S, Sm, most = attention_ref(q, k, v, g, 2.0 ** -4, [L], torch.zeros(1, H, K, V))
    got = linear_attention_prompt(q[None].to(cuda), k[None].to(cuda), v[None].to(cuda), g[None].to(cuda), scale=2.0 ** -4)
    assert_near(got[0], o, out_rel([L], most, F16) * mag + _weights_off(q, k, v, g, 2.0 ** -4, 2.0 ** -29), 1.0, "o")


def _state_off(k, v, g, rel):
    """What a state loses where a chunk's weighted v is off by ``rel`` of the largest of its channel: (H, K, V)."""
    T, H = k.shape[:2]
    g = torch.zeros(T, H).double() if g is None else g.double().expand(T, H)
    off = torch.zeros(H, k.shape[2], v.shape[2]).double()
    for a in range(0, T, 64):
        c = torch.cumsum(g[a:a + 64], 0)
        top = (torch.exp(c[-1] - c)[..., None] * v[a:a + 64].double().abs()).amax(0)                  # (H, V)
        off = off * torch.exp(c[-1])[:, None, None] + rel * k[a:a + 64].double().abs().sum(0)[..., None] * top[:, None]
    return off


def _check_sizes(cuda, q, k, v, g, state, scale=0.125):
    L, H = v.shape[:2]
    o, mag, S, Sm, most = attention_ref(q, k, v, g, scale, [L], state)
    got_state = state.to(cuda)
    got = linear_attention_prompt(q[None].to(cuda), k[None].to(cuda), v[None].to(cuda), None if g is None else g[None].to(cuda), scale=scale, state=got_state)
    off = _state_off(k, v, g, 2.0 ** -26) if state.abs().max() == 0 else 0.0
    bad = lambda t: torch.where(torch.isfinite(t), t, float("nan"))  # noqa: E731  (an infinity counts as a NaN)
    assert_near(bad(got_state[0].cpu()), bad(S[0]), bad(state_rel([L], most) * Sm[0] + off), 1.0, "state")
    got = got[0].cpu()
    near = (o.abs() > 65000) & (o.abs() < 66000)                                       # (fp16 ends at 65504: beyond it, infinities)
    got, o = torch.where(near, 0.0, got), torch.where(near, 0.0, torch.where(o.abs() > 65504, float("inf"), o))
    assert_near(bad(got), bad(o), bad(out_rel([L], most, F16) * mag + _weights_off(q, k, v, g, scale, 2.0 ** -29)), 1.0, "o")


@pytest.mark.parametrize("L", [64, 200, 1500])
@pytest.mark.parametrize("size", [2.0 ** -11, 2.0 ** -14, 2.0 ** -18, 2.0 ** 8])
@pytest.mark.parametrize("K,V", [(64, 64), (128, 72)])
def test_fp16_small_values_behind_a_large_one_that_decays(cuda, L, size, K, V):
    """The first token of each chunk is large and decays to nothing inside it: the later ones' part of the state keeps its bits."""
    H = 2
    q, k, v, _ = attention_inputs(L, H, K, V, F16, "none", seed=L)
    v = (v.float() * size).half()
    v[::64] = 1.0
    g = torch.full((L, H), -0.6931)
    g[:, 1] = -0.2
    _check_sizes(cuda, q, k, v, g, torch.zeros(1, H, K, V))


@pytest.mark.parametrize("decay", [0.0, -0.02, -0.4, -3.0])
@pytest.mark.parametrize("first", [0.0, 1.0, 1e-30, 2.0 ** 60])
@pytest.mark.parametrize("up", [1, -1])
def test_fp16_sizes_that_change_from_chunk_to_chunk(cuda, decay, first, up):
    """Chunks and channels of v of many sizes (upwards some are infinite), from states of many sizes."""
    H, K, V, L = 2, 64, 96, 640
    q, k, v, _ = attention_inputs(L, H, K, V, F16, "none", seed=3)
    sizes = 2.0 ** torch.tensor([0.0, -12, -12, 8, -18, 0, 12, 12, -6, -14])
    v = v.float().clamp(-3, 3) * sizes.repeat_interleave(64)[:, None, None] * 2.0 ** (up * (-torch.arange(V) % 5 * (torch.arange(V) // 32)))
    state = first * torch.randn(1, H, K, V, generator=torch.Generator().manual_seed(4))
    _check_sizes(cuda, q, k, v.half(), torch.full((L, H), decay), state)


def test_fp16_states_next_to_the_largest_numbers(cuda):
    H, K, V, L = 1, 64, 64, 70
    q, k, v, _ = attention_inputs(L, H, K, V, F16, "none", seed=5)
    _check_sizes(cuda, (q.float() * 2.0 ** -5).half(), k, v, torch.full((L, H), -0.5), torch.full((1, H, K, V), 3e38), scale=2.0 ** -126)


@pytest.mark.parametrize("size", [2.0 ** -4, 2.0 ** -2, 1.0, 40.0, 2.0 ** -30])
@pytest.mark.parametrize("below", [2.0 ** -10, 2.0 ** -13, 2.0 ** -16])
def test_fp16_small_rows_of_a_state(cuda, size, below):
    """q that reads only the rows of the state that are far below its others: off by half a step, or 2^-25 of the channel's largest entry."""
    H, K, V, L = 2, 64, 64, 130
    q, k, v, g = attention_inputs(L, H, K, V, F16, seed=7, g_mean=5.0)
    q[:, :, :32], v[:] = 0.0, 0.0
    state = size * (1 + torch.rand(1, H, K, V, generator=torch.Generator().manual_seed(8)))
    state[:, :, 32:] *= below
    o, mag, S, Sm, most = attention_ref(q, k, v, g, 0.125 / below, [L], state)
    got = linear_attention_prompt(q[None].to(cuda), k[None].to(cuda), v[None].to(cuda), g[None].to(cuda), scale=0.125 / below, state=state.to(cuda))
    decay = torch.exp(torch.cumsum(g.double(), 0))[..., None]
    off = 2.0 ** -25 * 0.125 / below * decay * state[0].double().amax(1) * q.double().abs().sum(-1, keepdim=True)
    assert_near(got[0], o, out_rel([L], most, F16) * mag + off, 1.0, "o")


@pytest.mark.parametrize("dtype,log", [(BF16, -116), (BF16, -60), (BF16, 70), (F16, -44), (F16, 90)])
@pytest.mark.parametrize("decay", [0.0, -0.3, -2.0])
def test_scales_far_from_one(cuda, dtype, log, decay):
    """Such a scale takes nothing from the weights of old tokens."""
    H, K, V, L = 2, 64, 64, 200
    q, k, v, _ = attention_inputs(L, H, K, V, dtype, "none", seed=-log)
    up = -log - 26 if dtype == BF16 else 0
    v = (v.float() * 2.0 ** up).to(dtype)
    state = torch.randn(1, H, K, V, generator=torch.Generator().manual_seed(9)) * 2.0 ** (up if dtype == BF16 else -log)
    g, scale = torch.full((L, H), decay), -1.3 * 2.0 ** log
    if dtype == F16:
        v = v * 0.0 if log > 0 else v
    o, mag, S, Sm, most = attention_ref(q, k, v, g, scale, [L], state)
    got = linear_attention_prompt(q[None].to(cuda), k[None].to(cuda), v[None].to(cuda), g[None].to(cuda), scale=scale, state=state.to(cuda))
    assert_near(got[0], o, mag, out_rel([L], most, dtype), "o")


@pytest.mark.parametrize("L", [64, 200, 1500])
@pytest.mark.parametrize("decay", [0.0, -0.05, -0.3, -2.0])
@pytest.mark.parametrize("size", [100, 116])
def test_bf16_has_the_range_of_fp32(cuda, L, decay, size):
    """Nothing overflows that the formula leaves below 2^128: v, and k v with large k, next to that."""
    H, K, V = 2, 64, 64
    q, k, v, _ = attention_inputs(L, H, K, V, BF16, "none", seed=L)
    v = v.float()
    v[:, 0] *= 2.0 ** size
    k[:, 1] = (k[:, 1].float() * 2.0 ** (size - 20)).to(BF16)
    v[:, 1] *= 2.0 ** 20
    v, g = v.to(BF16), torch.full((L, H), decay)
    o, mag, S, Sm, most = attention_ref(q, k, v, g, 2.0 ** -size, [L], torch.zeros(1, H, K, V))
    state = torch.zeros(1, H, K, V, device=cuda)
    got = linear_attention_prompt(q[None].to(cuda), k[None].to(cuda), v[None].to(cuda), g[None].to(cuda), scale=2.0 ** -size, state=state)
    assert_near(got[0], o, mag, out_rel([L], most, BF16), "o")
    assert_near(state, S, Sm, state_rel([L], most), "state")


@pytest.mark.parametrize("seed", range(8))
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_packed_prompts_cut_at_every_place(cuda, seed, dtype):
    """Prompts around whole segments among empty and single ones, more than 64 of them; each segment's state lies where its neighbours expect it."""
    gen = torch.Generator().manual_seed(seed)
    pick = lambda n: int(torch.randint(0, n, (1,), generator=gen))  # noqa: E731
    choices = [0, 0, 1, 1, 2, 63, 64, 65, 127, 128, 129, 192, 193, 256, 257, 384, 385, 512, 513, 1025]
    lens = [choices[pick(len(choices) if i % 3 == 0 else 6)] for i in range([5, 9, 30, 70, 130, 3, 200, 12][seed])] + [600 + pick(400)]
    first, H, K, V = [0, 64, 5, 0, 63, 200, 0, 1][seed], 1 + seed % 2, 64, 64
    T, n = sum(lens), len(lens)
    q, k, v, g = attention_inputs(T, H, K, V, dtype, seed=seed, g_mean=5.0)
    state = torch.randn(n, H, K, V, generator=gen)
    o, mag, S, Sm, most = attention_ref(q, k, v, g, 0.125, lens, state)
    room = lambda t: torch.cat([torch.full((first, *t.shape[1:]), float("nan")).to(t.dtype), t]).to(cuda)  # noqa: E731
    got_state = state.to(cuda)
    got = linear_attention_prompt(*(room(t) for t in (q, k, v, g)), scale=0.125, state=got_state, seq_starts=starts_of(lens, cuda, first=first))
    assert_near(got[first:], o, mag, out_rel(lens, most, dtype), "o")
    assert_near(got_state, S, Sm, state_rel(lens, most), "state")
