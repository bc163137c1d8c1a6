"""The serving operators at the edges of what they take: one row of a wide tensor, prompts in each way of being cut, steps that let a
state grow, magnitudes far apart, values that are no numbers."""

import pytest
import torch

from linquant_amd import _lib
from linquant_amd.kernels.mamba2.conv1d_state import conv1d_prompt, conv1d_step
from linquant_amd.kernels.mamba2.ssm import ssm_prompt, ssm_step
from linquant_amd.norm import residual_rmsnorm, rmsnorm_gated, rmsnorm_gated_qhad
from linquant_amd.hadamard_utils import qhad_transform
from linquant_amd.w8a8_linear import W8A8Linear, int8_matmul, quantize_rows
from tests.serving_cases import assert_near, ssm_inputs, ssm_ref, ssm_rel, ssm_y_rel, starts_of
from tests.test_serving_mixer_gpu import build, check_call, snapshot, tokens

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
NAN, INF = float("nan"), float("inf")


def _gen(seed=0):
    return torch.Generator().manual_seed(seed)


def _rn(*shape, seed=0):
    return torch.randn(*shape, generator=_gen(seed))


# --------------------------------------------------------------------------------------------- one row of a wide tensor
def _one(t, pitch, dim=0):
    """``t``, one entry long along ``dim``, as a view whose stride there is ``pitch``."""
    strides = list(t.stride())
    strides[dim] = pitch
    return t.as_strided(t.shape, strides)


@pytest.mark.parametrize("pitch", [77, 1 << 24, (1 << 24) + 1])
def test_one_row_at_any_distance(cuda, pitch):
    """The stride along a dimension of length one is no distance between entries: any is taken."""
    x, w = _rn(1, 64).half().to(cuda), _rn(64, 4, seed=1).half().to(cuda)
    st = [torch.zeros(1, 3, 64, dtype=F16, device=cuda) for _ in range(2)]
    assert torch.equal(conv1d_step(_one(x, pitch), st[0], w), conv1d_step(x, st[1], w)) and torch.equal(*st)
    starts = starts_of([1], cuda)
    assert torch.equal(conv1d_prompt(_one(x, pitch), w, state=st[0], seq_starts=starts), conv1d_prompt(x, w, state=st[1], seq_starts=starts))
    assert torch.equal(conv1d_prompt(_one(_one(x[None], pitch), pitch, 1), w), conv1d_prompt(x[None], w))
    a, b = (torch.randint(-127, 128, (1, 64), generator=_gen(i)).to(torch.int8).to(cuda) for i in (2, 3))
    assert torch.equal(int8_matmul(_one(a, pitch), _one(b, pitch), 1.0, 1.0), int8_matmul(a, b, 1.0, 1.0))
    q = W8A8Linear(b, torch.ones(1), input_scale=0.05).to(cuda)
    assert torch.equal(q(_one(x, pitch)), q(x))
    assert all(torch.equal(i, j) for i, j in zip(quantize_rows(_one(x, pitch)), quantize_rows(x)))
    assert all(torch.equal(i, j) for i, j in zip(residual_rmsnorm(_one(x, pitch), x[0], _one(x, pitch)), residual_rmsnorm(x, x[0], x)))
    v = {k: t.to(cuda) for k, t in ssm_inputs(1, 2, 64, 1, 64, F16).items()}
    far = {k: t if k == "A" else _one(t, pitch) for k, t in v.items() if k in ("x", "dt", "A", "B", "C")}
    near = {k: v[k] for k in far}
    s = [torch.ones(1, 2, 64, 64, device=cuda) for _ in range(2)]
    assert torch.equal(ssm_step(s[0], **far), ssm_step(s[1], **near)) and torch.equal(*s)
    assert torch.equal(ssm_prompt(**far, state=s[0], seq_starts=starts), ssm_prompt(**near, state=s[1], seq_starts=starts)) and torch.equal(*s)
    batch = lambda d, p: {k: t if k == "A" else (_one(t[None], p) if p else t[None]) for k, t in d.items()}  # noqa: E731
    assert torch.equal(ssm_prompt(**batch(far, pitch), state=s[0]), ssm_prompt(**batch(near, 0), state=s[1])) and torch.equal(*s)


def test_norms_of_one_row_of_a_wide_tensor(cuda):
    x, z, w = _rn(1, 512).half().to(cuda), _rn(1, 1540, seed=1).half().to(cuda)[:, :512], torch.ones(512, device=cuda)
    assert torch.equal(rmsnorm_gated(x, z, w), rmsnorm_gated(x, z.clone(), w))
    assert torch.equal(rmsnorm_gated_qhad(x, z, w, 0.05)[0], rmsnorm_gated_qhad(x, z.clone(), w, 0.05)[0])
    odd = _one(x, 517)
    assert torch.equal(rmsnorm_gated(odd, z, w), rmsnorm_gated(x, z, w)) and torch.equal(qhad_transform(odd, 0.05)[0], qhad_transform(x, 0.05)[0])


@pytest.mark.parametrize("rows", [True, False])
def test_mixer_with_one_sequence(cuda, rows):
    """Four heads: a token's projected row is no multiple of 16 bytes, and one sequence has one of them."""
    m = build(W8A8Linear, 2, 4, 128, rows=rows)
    st = m.allocate_state(2)
    slots = torch.tensor([1], dtype=torch.int32, device=cuda)
    wide = torch.zeros(1, m.d_model + 3, dtype=F16, device=cuda)   # the activations as such a row, too
    wide[:, :m.d_model] = tokens(1, m, 1).cuda()
    one = wide[:, :m.d_model]

    def run(call, hidden):
        before, dbg = snapshot(st), {}
        call(hidden, dbg)
        if rows:
            check_call(m, hidden.cpu(), dbg, [1], before, snapshot(st), [1], slice(None))
        assert torch.isfinite(dbg["out"]).all()

    run(lambda h, dbg: m.prefill(h, st, slots, starts_of([1], cuda), _debug=dbg), one)
    run(lambda h, dbg: m.step(h, st, slots, _debug=dbg), one)
    run(lambda h, dbg: m.prefill(h, st, slots, _debug=dbg), one[None])


# ----------------------------------------------------------------------------------------------------- shapes and types
@pytest.mark.parametrize("K", [32, 21])
def test_a_single_row_without_a_leading_dimension(cuda, K):
    x = _rn(K).half().to(cuda)
    q, s = quantize_rows(x)
    q2, s2 = quantize_rows(x[None])
    assert q.shape == (K,) and s.shape == () and torch.equal(q, q2[0]) and torch.equal(s, s2[0])
    b = torch.randint(-127, 128, (5, K), generator=_gen(1)).to(torch.int8).to(cuda)
    assert torch.equal(int8_matmul(q, b, s, 1.0), int8_matmul(q2, b, s2, 1.0)[0])


@pytest.mark.parametrize("wt,pt", [(F16, F32), (BF16, F32), (F32, F16), (F16, BF16), (BF16, F16)])
def test_norm_weights_of_two_types(cuda, wt, pt):
    """Each weight enters as it is: nothing of the wider type's bits or range is lost to the other's."""
    x, w = _rn(3, 264).half(), (1 + 0.1 * _rn(264, seed=1)).to(wt)
    post = (1 + 0.1 * _rn(264, seed=2)).to(pt)
    post[:8] *= 2.0 ** (30 if pt != F16 else 12)
    y, r = residual_rmsnorm(x.to(cuda), w.to(cuda), post_weight=post.to(cuda), residual_dtype=F32)
    u = x.double()
    want = u * torch.rsqrt(u.square().mean(-1, keepdim=True) + 1e-5) * post.double()
    # the mean's sum over 264 in four waves, its square root and three products: fewer than 32 roundings
    assert_near(r, want, want.abs(), 32 * 2.0 ** -24, "r")
    f = torch.rsqrt(want.square().mean(-1, keepdim=True) + 1e-5) * w.double()
    assert_near(y, f * want, (f * want).abs(), 64 * 2.0 ** -24, "y")


# ------------------------------------------------------------------------------------------------------------- the scan
def _scan(cuda, v, lens, *, packed=True, state=None, slots=None, **kw):
    """(y, state behind, the formula's y, its magnitudes, state and magnitudes, the most that |d A| sums to in a chunk); the formula in 64
    bits on the GPU, where the token loop is quicker."""
    d = {k: t.to(cuda) for k, t in v.items()}
    n = len(lens)
    st = None if state is None else state.to(cuda)
    call = dict(D=d["D"], dt_bias=d.get("dt_bias"), state=st, slots=None if slots is None else torch.tensor(slots, dtype=torch.int32, device=cuda), **kw)
    args = [d[k] for k in ("x", "dt", "A", "B", "C")]
    if packed:
        y = ssm_prompt(*args, **call, seq_starts=starts_of(lens, cuda))
    else:
        y = ssm_prompt(*(a if a is d["A"] else a.unflatten(0, (n, lens[0])) for a in args), **call).flatten(0, 1)
    H, P, N = v["x"].shape[1], v["x"].shape[2], v["B"].shape[2]
    use = list(range(n)) if slots is None else slots
    first = torch.stack([torch.zeros(H, P, N) if state is None or s < 0 else state[s] for s in use]).to(cuda)
    ref = ssm_ref(*args, d["D"], d.get("dt_bias"), kw.get("dt_softplus", True), kw.get("dt_limit", (0.0, INF)), lens, first)
    return (y, st, *ref)


def _near_where_finite(y, want, mag, rel):
    """``assert_near`` where even the largest error that it allows, half a step of fp16 and rel * mag, leaves a number of fp16 (or bf16): a result that
    may be off past 65504 may be an infinity."""
    fits = want.abs() * (1 + 2.0 ** -8) + 1.01 * rel * mag < torch.finfo(y.dtype).max
    assert_near(torch.where(fits, y, 0.0), torch.where(fits, want, 0.0), torch.where(fits, mag, 0.0), rel, "y")


def _plan(lens, packed, H, P, G, N, dtype):
    import ctypes

    st = _lib.fill("lq_ssm_prompt_args", nseq=len(lens), seqlen=0 if packed else lens[0], tokens=sum(lens) if packed else 0,
                   seq_starts=16 if packed else None, nheads=H, headdim=P, ngroups=G, dstate=N,
                   dtype=_lib.LQ_DT_F16 if dtype == F16 else _lib.LQ_DT_BF16)
    out = (ctypes.c_int64 * 3)()
    assert _lib.load().lq_ssm_prompt_plan(ctypes.byref(st), ctypes.byref(out)) == 0
    return list(out)[1:]


# H, P, G, N; lengths, packed; a segment's chunks and pieces.  Nearly all leave a last segment that is shorter and a last chunk that is not full.
CUT = [((80, 64, 1, 128), [2500] * 2, False, [14, 2]), ((16, 64, 2, 128), [2500] * 2, False, [3, 1]), ((40, 64, 2, 64), [2500] * 2, False, [7, 1]),
       ((64, 64, 8, 128), [3999] * 2, False, [16, 2]), ((128, 8, 1, 8), [2300, 1200, 70, 0, 1900, 1500, 1400, 1230], True, [14, 2]),
       ((64, 64, 8, 128), [900, 2100, 130], True, [6, 1]), ((32, 32, 4, 16), [4000] * 2, False, [2, 1])]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dims,lens,packed,cut", CUT, ids=lambda c: str(c))
def test_prompts_cut_into_segments_of_several_chunks(cuda, dims, lens, packed, cut, dtype):
    """States pass, join and the segments that start inside a prompt, as long prompts of many heads take them: little decay, so that what one
    segment leaves is most of what the next one has; carried-in states, and a prompt that starts from zero and leaves nothing."""
    H, P, G, N = dims
    assert _plan(lens, packed, *dims, dtype) == cut
    v = ssm_inputs(sum(lens), H, P, G, N, dtype, seed=len(lens), a_max=1.3, dt_mean=-6.0)
    n = len(lens)
    state = _rn(n + 1, H, P, N, seed=5)
    slots = [n - i for i in range(n)]
    slots[1] = -1
    y, st, wy, mag, ws, smag, most = _scan(cuda, v, lens, packed=packed, state=state, slots=slots)
    assert_near(y, wy, mag, ssm_y_rel(lens, most, dtype), "y")
    for i, s in enumerate(slots):
        if s >= 0:
            assert_near(st[s], ws[i], smag[i], ssm_rel(lens, most), f"state {i}")
    for s in set(range(n + 1)) - set(slots):
        assert torch.equal(st[s].cpu(), state[s])


def _growing(dtype, T, turn, bits):
    """Steps that are negative for `turn` tokens, so that a state grows by 2^bits over them, and as positive for the next."""
    H, P, G, N = 3, 40, 1, 64
    v = ssm_inputs(T, H, P, G, N, dtype, seed=9)
    v["A"] = torch.full((H,), -1.0)
    v["dt"] = (torch.full((T, H), bits / turn / 1.4427) * torch.where(torch.arange(T) // turn % 2 == 0, -1.0, 1.0)[:, None]).float()
    del v["dt_bias"]
    return v


@pytest.mark.parametrize("dtype,turn,bits,scale", [(BF16, 32, 45, 0), (BF16, 64, 60, 0), (BF16, 7, 20, 0), (F16, 32, 26, -14), (F16, 64, 24, -14), (F16, 7, 8, 0)])
def test_steps_that_let_the_state_grow(cuda, dtype, turn, bits, scale):
    """Negative steps, where ``dt_limit`` lets them through: the weights of a chunk's tokens grow along it."""
    v = _growing(dtype, 200, turn, bits)
    v["B"], v["C"], v["x"] = v["B"] * 2.0 ** scale, v["C"] * 2.0 ** scale, v["x"] * 2.0 ** -(scale // 2)
    state = _rn(1, 3, 40, 64, seed=3) * 2.0 ** -8
    y, st, wy, mag, ws, smag, most = _scan(cuda, v, [200], state=state, dt_softplus=False, dt_limit=(-INF, INF))
    assert (wy.abs() < 60000).all() or dtype == BF16
    assert_near(y, wy, mag, ssm_y_rel([200], most, dtype), "y")
    assert_near(st[0], ws[0], smag[0], ssm_rel([200], most), "state")
    d = {k: t.to(cuda) for k, t in v.items()}
    one = state.to(cuda)
    for t in range(70):                                             # token by token
        ssm_step(one, d["x"][t:t + 1], d["dt"][t:t + 1], d["A"], d["B"][t:t + 1], d["C"][t:t + 1], dt_softplus=False, dt_limit=(-INF, INF))
    part = {k: x if k in ("A", "D") else x[:70] for k, x in v.items()}
    y, st, wy, mag, ws, smag, most = _scan(cuda, part, [70], state=state, dt_softplus=False, dt_limit=(-INF, INF))
    assert_near(one[0], ws[0], smag[0], ssm_rel([70], most), "state of single tokens")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("carried", [0, 20, 60])
@pytest.mark.parametrize("T", [1, 150])
def test_channels_far_apart(cuda, dtype, carried, T):
    """One channel of a head far above the others, by its activations (2^26) and by what it carries in: the others are as if it was not there."""
    H, P, G, N = 2, 64, 1, 128
    v = ssm_inputs(T, H, P, G, N, dtype, seed=13, a_max=1.3, dt_mean=-4.5)
    v["x"] = v["x"] * 2.0 ** -12
    v["x"][:, :, 5] = v["x"][:, :, 5] * 2.0 ** 25
    state = _rn(1, H, P, N, seed=4) * 2.0 ** -14
    state[:, :, 37] *= 2.0 ** carried
    y, st, wy, mag, ws, smag, most = _scan(cuda, v, [T], state=state)
    assert_near(st[0], ws[0], smag[0], ssm_rel([T], most), "state")
    _near_where_finite(y, wy, mag, ssm_y_rel([T], most, dtype))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("what", ["x", "dt", "B", "C", "state"])
@pytest.mark.parametrize("value", [NAN, INF, -INF])
@pytest.mark.parametrize("T,at", [(200, 70), (200, 127), (200, 191), (64, 0), (40, 39)])
def test_values_that_are_no_numbers(cuda, dtype, what, value, T, at):
    """They reach what the formula has them reach, and nothing else: no token in front, no other channel, head or sequence.  (A raw step of minus
    infinity is a step of zero, a number.)"""
    H, P, G, N = 4, 40, 2, 72
    lens = [30, T, 9]
    v = ssm_inputs(sum(lens), H, P, G, N, dtype, seed=21, a_max=2.0, dt_mean=-3.0)
    state = _rn(3, H, P, N, seed=6)
    clean = _scan(cuda, v, lens, state=state)
    t = 30 + at
    {"x": lambda: v["x"][t, 2].__setitem__(7, value), "dt": lambda: v["dt"][t].__setitem__(1, value), "B": lambda: v["B"][t, 1].__setitem__(66, value),
     "C": lambda: v["C"][t, 0].__setitem__(3, value), "state": lambda: state[1, 3, 33].__setitem__(70, value)}[what]()
    y, st, wy, mag, ws, smag, most = _scan(cuda, v, lens, state=state)
    reach, gone = ~torch.isfinite(wy), ~torch.isfinite(ws)
    number = what == "dt" and value == -INF
    assert reach.any() == (not number) and torch.equal(~torch.isfinite(y), reach) and torch.equal(~torch.isfinite(st), gone)
    if not number:
        wy, mag, ws, smag, most = clean[2:]
    assert_near(torch.where(reach, 0.0, y), torch.where(reach, 0.0, wy), mag, ssm_y_rel(lens, most, dtype), "y elsewhere")
    assert_near(torch.where(gone, 0.0, st), torch.where(gone, 0.0, ws), smag, ssm_rel(lens, most), "state elsewhere")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("N", [8, 24, 40, 96, 128, 200])
def test_single_tokens_and_infinite_entries(cuda, dtype, N):
    """An infinite entry of the state gives its row's output its sign; the row's length need be no multiple of what a wave reads."""
    H, P = 2, 16
    v = {k: t.to(cuda) for k, t in ssm_inputs(1, H, P, 1, N, dtype, seed=22).items()}
    for n in sorted({0, N // 2, N - 4, N - 1}):
        st = torch.ones(1, H, P, N, device=cuda)
        st[0, 1, 3, n], st[0, 0, 9, n] = INF, NAN
        y = ssm_step(st, v["x"], v["dt"], v["A"], v["B"], v["C"])
        assert float(y[0, 1, 3]) == float(v["C"][0, 0, n].sign()) * INF, n
        assert torch.isnan(y[0, 0, 9])
        y[0, 1, 3] = y[0, 0, 9] = 0.0
        assert torch.isfinite(y).all()
        st[0, 1, 3, n] = st[0, 0, 9, n] = 0.0
        assert torch.isfinite(st).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("at", [20, 63, 64, 100])
@pytest.mark.parametrize("T", [110, 600])
def test_tokens_far_apart(cuda, dtype, at, T):
    """A token far above those in front of it, which read a small state: they are as if it was not there.  And a prompt that goes on in front of a state far
    above it."""
    H, P, G, N = 2, 64, 1, 64
    v = ssm_inputs(T, H, P, G, N, dtype, seed=14, a_max=1.3, dt_mean=-4.5)
    v["x"] = v["x"] * 2.0 ** -12
    v["x"][at] = v["x"][at] * 2.0 ** 25
    for up in (-14, 30):
        state = _rn(1, H, P, N, seed=4) * 2.0 ** up
        y, st, wy, mag, ws, smag, most = _scan(cuda, v, [T], state=state)
        assert_near(st[0], ws[0], smag[0], ssm_rel([T], most), "state")
        _near_where_finite(y, wy, mag, ssm_y_rel([T], most, dtype))


def test_starts_that_name_more_segments_than_32_bits_count(cuda):
    """60,000 prompts of the same 2^24 tokens: the segments in front of the later ones come to 2^33.  Nothing is touched out of range, and the first
    one's state is what it is by itself."""
    H, P, G, N, T, n = 1, 8, 1, 8, 1 << 24, 120001
    v = {k: t.repeat(*([1] if k in ("A", "D", "dt_bias") else [T // 4096] + [1] * (t.dim() - 1))).to(cuda) for k, t in ssm_inputs(4096, H, P, G, N, F16, seed=32).items()}
    args = [v[k] for k in ("x", "dt", "A", "B", "C")]
    starts = torch.zeros(n + 1, dtype=torch.int32, device=cuda)
    starts[1::2] = T
    st, alone = torch.zeros(n, H, P, N, device=cuda), torch.zeros(1, H, P, N, device=cuda)
    ssm_prompt(*args, state=st, seq_starts=starts)
    ssm_prompt(*args, state=alone, seq_starts=starts_of([T], cuda))
    torch.cuda.synchronize()
    assert torch.isfinite(alone).all() and ((st[0] - alone[0]).abs().max() <= 2.0 ** -9 * alone.abs().max()).all()   # (cut into other segments)


@pytest.mark.parametrize("rows", [True, False])
def test_mixer_calls_without_tokens(cuda, rows):
    """No tokens, no sequences: nothing comes out and no state is touched."""
    from linquant_amd.quantized_mamba2 import Mamba2Block

    m = build(W8A8Linear, rows=rows)
    b = Mamba2Block(m, torch.ones(m.d_model).half().cuda())
    st = m.allocate_state(3)
    for t in st:
        t.fill_(1.5)
    none, starts = torch.zeros(0, m.d_model, dtype=F16, device=cuda), torch.zeros(4, dtype=torch.int32, device=cuda)
    for hidden in (none, (torch.zeros(0, m.d_model, dtype=torch.int8, device=cuda), torch.ones((), device=cuda))):
        assert m.prefill(hidden, st, None, starts).shape == none.shape and m.step(hidden, st).shape == none.shape
    assert m.prefill(none.view(3, 0, m.d_model), st).shape == (3, 0, m.d_model)
    x, r = b.step(none, None, st)
    assert x.shape == r.shape == none.shape and b.prefill(x, r, st, None, starts)[0].shape == none.shape
    torch.cuda.synchronize()
    assert all((t == 1.5).all() for t in st)
