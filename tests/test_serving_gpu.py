"""The serving operators against their plain 64-bit forms: types, odd sizes, strides, slots, empty prompts, unusual values."""

import pytest
import torch

from linquant_amd.kernels.mamba2.conv1d_state import conv1d_prompt, conv1d_step
from linquant_amd.kernels.mamba2.ssm import ssm_prompt, ssm_step
from linquant_amd.norm import residual_rmsnorm
from linquant_amd.w8a8_linear import W8A8Linear, int8_matmul, quantize_rows
from tests.serving_cases import HALF_STEP, assert_near, conv_ref, ssm_inputs, ssm_ref, ssm_rel, ssm_y_rel, starts_of

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
NAN = float("nan")


def _gen(seed=0):
    return torch.Generator().manual_seed(seed)


# ------------------------------------------------------------------------------------------------------------ projections
def _codes(shape, gen):
    return torch.randint(-127, 128, shape, generator=gen).to(torch.int8)


@pytest.mark.parametrize("M,K,N", [(1, 16, 1), (1, 2560, 640), (3, 48, 33), (16, 256, 100), (17, 1040, 777), (33, 128, 256), (64, 640, 129),
                                   (65, 640, 500), (127, 144, 31), (128, 128, 128), (129, 272, 257), (300, 1024, 260), (513, 2560, 300)])
@pytest.mark.parametrize("out_dtype", [F16, BF16, F32])
def test_int8_matmul(cuda, M, K, N, out_dtype):
    gen = _gen(M + K + N)
    a, b = _codes((M, K), gen), _codes((N, K), gen)
    sa, sb = torch.rand(M, generator=gen) * 1e-3 + 1e-4, torch.rand(N, generator=gen) * 1e-2 + 1e-3
    bias = torch.randn(N, generator=gen)
    got = int8_matmul(a.to(cuda), b.to(cuda), sa.to(cuda), sb.to(cuda), bias=bias.to(out_dtype).to(cuda), out_dtype=out_dtype)
    exact = (a.double() @ b.double().T) * sa.double()[:, None] * sb.double()
    want = exact + bias.to(out_dtype).double()
    # the sum's conversion, the product of the scales, its product with the sum and the bias: a rounding each
    assert_near(got, want, exact.abs() + bias.abs(), 4 * 2.0 ** -24, "product")


def test_int8_matmul_sums_are_exact(cuda):
    """Extreme codes over the longest row that a sum in 32 bits allows, and differences of one in it."""
    K = 131056
    a = torch.full((2, K), -128, dtype=torch.int8, device=cuda)
    b = torch.full((3, K), -128, dtype=torch.int8, device=cuda)
    a[1, -1], b[2] = 127, 127
    got = int8_matmul(a, b, 1.0, 1.0, out_dtype=F32)
    want = a.double() @ b.double().T
    assert torch.equal(got, want.float())


def test_int8_matmul_strides_scales_and_out(cuda):
    gen = _gen(1)
    wide_a, wide_b = _codes((40, 96), gen).to(cuda), _codes((50, 128), gen).to(cuda)
    a, b = wide_a[::2, 16:80], wide_b[1::3, 32:96]
    want = a.double() @ b.double().T
    buf = torch.full((20, 40), 7.0, dtype=F32, device=cuda)
    out = buf[:, 3:3 + b.shape[0]]
    assert int8_matmul(a, b, 1.0, torch.ones((), device=cuda), out_dtype=F32, out=out) is out
    assert torch.equal(out, want.float()) and (buf[:, :3] == 7).all() and (buf[:, 3 + b.shape[0]:] == 7).all()
    half = int8_matmul(a, b, torch.full((20,), 0.5, dtype=F16, device=cuda), 2.0, out_dtype=F32)   # a 16-bit scale is read as its value
    assert torch.equal(half, want.float())
    odd = int8_matmul(wide_a[:, 5:26], wide_b[:, 5:26], 1.0, 1.0, out_dtype=F32)                  # rows of 21 bytes
    assert torch.equal(odd, (wide_a[:, 5:26].double() @ wide_b[:, 5:26].double().T).float())
    lead = int8_matmul(wide_a.view(2, 4, 5, 96), wide_b[:, :96], 1.0, 1.0, out_dtype=F32)
    assert lead.shape == (2, 4, 5, 50) and torch.equal(lead.view(40, 50), (wide_a.double() @ wide_b[:, :96].double().T).float())
    assert int8_matmul(wide_a[:0, :64], b, 1.0, 1.0).shape == (0, b.shape[0])


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 64), (2, 2560), (1025, 2560), (1030, 512), (1024, 4096), (7, 4099), (2, 16384), (2000, 5120)])
def test_quantize_rows(cuda, dtype, rows, cols):
    x = (torch.randn(rows, cols, generator=_gen(2)) * 3).to(dtype)
    x[0] = 0.0
    q, s = quantize_rows(x.to(cuda))
    xf = x.float()
    want = xf.abs().amax(1) / 127.0
    assert torch.equal(s.cpu(), want)
    codes = torch.round(xf / torch.where(want > 0, want, 1.0)[:, None]).to(torch.int8)  # IEEE division, half to even
    assert torch.equal(q.cpu(), codes) and int(q[-1].abs().max()) == (127 if rows > 1 else 0)


def test_quantize_rows_unusual_values(cuda):
    x = torch.randn(8, 40, dtype=F32, generator=_gen(3))
    x[0, 3], x[1, 5], x[2, 7] = NAN, float("inf"), -float("inf")
    x[3] *= 1e-38                                       # a scale in the subnormals
    x[4] *= 1e37
    wide = torch.zeros(8, 100)
    wide[:, 3:43] = x
    q, s = quantize_rows(wide.to(cuda)[:, 3:43].view(2, 4, 40))
    assert q.shape == (2, 4, 40) and s.shape == (2, 4)
    q, s = q.reshape(8, 40).cpu(), s.reshape(8).cpu()
    assert torch.isnan(s[:3]).all() and (q[:3] == 0).all()
    ref = x[4:].abs().amax(1) / 127.0
    assert torch.equal(s[4:], ref) and torch.equal(q[4:], torch.round(x[4:] / ref[:, None]).to(torch.int8))
    assert (s[3] * q[3].double() - x[3].double()).abs().max() <= 2.0 ** -133 + x[3].double().abs().max() / 254 * 1.01 + 127 * 2.0 ** -149


@pytest.mark.parametrize("K,N", [(256, 96), (250, 33)])
def test_w8a8_linear(cuda, K, N):
    gen = _gen(4)
    lin = torch.nn.Linear(K, N)
    with torch.no_grad():
        lin.weight.copy_(torch.randn(N, K, generator=gen) / K ** 0.5)
        lin.weight[3] = 0.0
    x = torch.randn(2, 5, K, generator=gen).half()
    m = W8A8Linear.from_fp16(lin).to(cuda)
    got = m(x.to(cuda))
    q, s = quantize_rows(x.to(cuda))
    w = m.weight[:, :K].double().cpu() * m.weight_scale.double().cpu()[:, None]
    terms = q.double().cpu() * s.double().cpu()[..., None]
    want = terms @ w.T + lin.bias.detach().double()
    assert_near(got, want, (terms @ w.T).abs() + lin.bias.detach().abs(), 4 * 2.0 ** -24, "linear")
    assert torch.equal(m.forward_int8(q, s), got)
    if K % 8 == 0:
        st = W8A8Linear.from_fp16(lin, input_scale=torch.tensor(0.03)).to(cuda)
        codes = torch.clamp(torch.round(x.float() / 0.03), -128, 127).to(torch.int8)
        assert torch.equal(st(x.to(cuda)), st.forward_int8(codes.to(cuda), 0.03))


# ------------------------------------------------------------------------------------------------------------------- norm
def _norm_ref(x, weight, residual, gate, scale, post, eps):
    u = x.double()
    if post is not None:
        u = u * torch.rsqrt(u.square().mean(-1, keepdim=True) + eps) * post.double()
    if gate is not None:
        u = u * gate.double()
    r0 = torch.zeros_like(u) if residual is None else residual.double()
    r = r0 + scale * u
    f, mag = torch.rsqrt(r.square().mean(-1, keepdim=True) + eps) * weight.double(), r0.abs() + (scale * u).abs()
    # y = f r: what r may be off by (a multiple of mag, also where its terms cancel to nothing) times |f|, and a multiple of y for f itself,
    # which |f| mag covers since |r| <= mag
    return f * r, r, mag, f.abs() * mag


@pytest.mark.parametrize("dtype,res", [(F16, F16), (F16, F32), (BF16, BF16), (BF16, F32), (F16, None)])
@pytest.mark.parametrize("gate,post", [("none", False), ("channel", True), ("full", True), ("sequence", False)])
@pytest.mark.parametrize("B,L,D", [(1, 1, 8), (2, 3, 2560), (3, 500, 1536), (2, 700, 2560), (2, 5, 4099), (1, 2, 16384), (1, 1100, 4096)])
def test_residual_rmsnorm(cuda, dtype, res, gate, post, B, L, D):
    gen = _gen(D + L)
    rn = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    x, w = rn(B, L, D).to(dtype), (1 + 0.1 * rn(D))
    residual = None if res is None else (2 * rn(B, L, D)).to(res)
    g = {"none": lambda: None, "channel": lambda: rn(D), "full": lambda: rn(B, L, D), "sequence": lambda: rn(B, 1, D)}[gate]()
    g = None if g is None else g.to(dtype)
    pw = (1 + 0.1 * rn(D)) if post else None
    dev = lambda t: None if t is None else t.to(cuda)  # noqa: E731
    y, r = residual_rmsnorm(dev(x), dev(w), dev(residual), 1e-5, gate=dev(g), scale=0.7, post_weight=dev(pw))
    want_y, want_r, mag, ymag = _norm_ref(x, w, residual, g, 0.7, pw, 1e-5)
    # a mean's sum over D and the chain of a handful of products: D / 64 additions a lane and seven rounds of exchanges are fewer than
    # 256 + 16 roundings, half of them in the square root's argument
    rel = 2.0 ** -24 * 288
    assert_near(r, want_r, mag, rel, "r")
    assert_near(y, want_y, ymag, 2 * rel, "y")
    assert y.dtype == dtype and r.dtype == (res or dtype)


@pytest.mark.parametrize("rows,D", [(4, 2560), (1500, 2560), (3, 1001)])
def test_residual_rmsnorm_codes(cuda, rows, D):
    gen = _gen(5)
    x, res, w = (torch.randn(rows, D, generator=gen).half().to(cuda), torch.randn(rows, D, generator=gen).to(cuda), (1 + 0.1 * torch.randn(D, generator=gen)).to(cuda))
    y, r = residual_rmsnorm(x, w, res)
    q, s, r2 = residual_rmsnorm(x, w, res, quantize="rows")
    assert torch.equal(r, r2) and q.shape == x.shape and s.shape == (rows,)
    want, _, _, _ = _norm_ref(x.cpu(), w.cpu(), res.cpu(), None, 1.0, None, 1e-5)
    # the row's scale, and codes whose value is within half a step of it (and what fp32 may move a tie by)
    assert ((s.double().cpu() * 127 - want.abs().amax(1)).abs() <= 2.0 ** -15 * want.abs().amax(1)).all()
    assert ((q.double() * s.double()[:, None]).cpu() - want).abs().le(0.5001 * s.double().cpu()[:, None] + 2.0 ** -15 * want.abs()).all()
    static = torch.tensor(0.025, device=cuda)
    q3, s3, r3 = residual_rmsnorm(x, w, res, quantize=static)
    assert s3 is static and torch.equal(r3, r)
    ref = want / static.double().cpu()
    assert (q3.double().cpu() - ref.clamp(-128, 127)).abs().max() <= 0.501


def test_residual_rmsnorm_unusual_rows(cuda):
    x = torch.randn(6, 64, dtype=F32, generator=_gen(6)).half()
    x[0], x[1, 3], x[2, 3] = 0.0, NAN, float("inf")
    y, r = residual_rmsnorm(x.to(cuda), torch.ones(64, device=cuda))
    assert (y[0] == 0).all() and torch.isnan(y[1]).all() and torch.equal(r.cpu().isnan(), x.isnan()) and torch.equal(r[3:].cpu(), x[3:])
    q, s, _ = residual_rmsnorm(x.to(cuda), torch.ones(64, device=cuda), quantize="rows")
    assert s[0] == 0 and (q[:3] == 0).all() and torch.isnan(s[1:3]).all() and torch.isfinite(s[3:]).all()
    assert residual_rmsnorm(x[:0].to(cuda), torch.ones(64, device=cuda))[0].shape == (0, 64)
    wide = torch.randn(6, 100, generator=_gen(7)).to(BF16).to(cuda)                # rows off the 16-byte grid, post weight of another type
    a, ra = residual_rmsnorm(wide[:, 3:67], torch.ones(64, device=cuda), wide[:, 20:84], post_weight=torch.ones(64, dtype=F16, device=cuda))
    b, rb = residual_rmsnorm(wide[:, 3:67].clone(), torch.ones(64, device=cuda), wide[:, 20:84].clone(), post_weight=torch.ones(64, device=cuda))
    assert_near(a, b.double(), b.double().abs(), 2 * HALF_STEP[BF16], "strided")
    assert_near(ra, rb.double(), rb.double().abs(), 2 * HALF_STEP[BF16], "strided")


# ------------------------------------------------------------------------------------------------------------ convolution
CONV_REL = 2.0 ** -20    # four taps and a bias, and SiLU on the exp2 and reciprocal units: fewer than sixteen roundings


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("W,bias,act", [(4, True, "silu"), (3, False, "silu"), (2, True, None)])
@pytest.mark.parametrize("lens", [[1], [5], [16], [17, 0, 1, 2, 3, 64, 0, 31], [0, 0], [100] * 3, [1] * 130, [2, 40] * 40])
def test_conv1d_prompt_packed(cuda, dtype, W, bias, act, lens):
    gen = _gen(sum(lens) + W)
    D, n, T = 536, len(lens), sum(lens)
    wide = torch.randn(T + 7, D + 16, generator=gen).to(dtype)
    x = wide.to(cuda)[:, 8:8 + D]
    w, b = (torch.randn(D, W, generator=gen) * 0.5).to(dtype), torch.randn(D, generator=gen).to(dtype) if bias else None
    state = torch.randn(n + 2, W - 1, D, generator=gen).to(dtype)
    slots = torch.randperm(n + 2, generator=gen)[:n].to(torch.int32)
    st = state.to(cuda)
    out = conv1d_prompt(x, w.to(cuda), None if b is None else b.to(cuda), activation=act, state=st, slots=slots.to(cuda),
                        seq_starts=starts_of(lens, cuda, first=3))               # tokens in front and behind belong to nobody
    y, mag, after = conv_ref(wide[3:3 + T, 8:8 + D], w, b, act is not None, lens, state[slots.long()])
    if T:
        assert_near(out[3:3 + T], y, mag, CONV_REL, "y")
    want = state.clone()
    want[slots.long()] = after.to(dtype)
    assert torch.equal(st.cpu(), want)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("L", [1, 2, 3, 15, 16, 33])
def test_conv1d_prompt_batch(cuda, dtype, L):
    """One length, with and without a state; without one it is the convolution that there was."""
    from linquant_amd.kernels.mamba2.causal_conv1d import causal_conv1d_fn

    gen = _gen(L)
    x, w, b = torch.randn(3, L, 64, generator=gen).to(dtype).to(cuda), torch.randn(64, 4, generator=gen).to(dtype).to(cuda), torch.randn(64, generator=gen).to(dtype).to(cuda)
    out = conv1d_prompt(x, w, b, activation="silu")
    if dtype == F16:
        assert torch.equal(out, causal_conv1d_fn(x.transpose(1, 2), w, b, activation="silu").transpose(1, 2))
    st = torch.zeros(3, 3, 64, dtype=dtype, device=cuda)
    assert torch.equal(conv1d_prompt(x, w, b, activation="silu", state=st), out)
    line = torch.cat([torch.zeros(3, 3, 64, dtype=dtype, device=cuda), x], 1)
    assert torch.equal(st, line[:, -3:])


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("W,D", [(4, 1032), (3, 8), (2, 5376)])
def test_conv1d_step(cuda, dtype, W, D):
    """Token after token is what one call over all of them gives, bit for bit; padding entries and slots out of range."""
    gen = _gen(W)
    n, L = 5, 7
    x = torch.randn(n, L, D, generator=gen).to(dtype).to(cuda)
    w, b = torch.randn(D, W, generator=gen).to(dtype).to(cuda), torch.randn(D, generator=gen).to(dtype).to(cuda)
    first = torch.randn(n + 1, W - 1, D, generator=gen).to(dtype).to(cuda)
    slots = torch.tensor([4, 0, 2, 5, 1], dtype=torch.int32, device=cuda)
    whole, parts = first.clone(), first.clone()
    y = conv1d_prompt(x, w, b, activation="silu", state=whole, slots=slots)
    for t in range(L):
        assert torch.equal(conv1d_step(x[:, t], parts, w, b, activation="silu", slots=slots), y[:, t])
    assert torch.equal(whole, parts)
    odd = torch.tensor([4, -1, 6, 99, 0], dtype=torch.int32, device=cuda)
    before = parts.clone()
    out = conv1d_step(x[:, 0], parts, w, b, activation="silu", slots=odd)
    assert (out[1] == 0).all() and torch.isnan(out[2:4]).all() and torch.isfinite(out[[0, 4]]).all()
    assert torch.equal(parts[[1, 2, 3, 5]], before[[1, 2, 3, 5]])


def test_conv1d_prompt_slots_out_of_range(cuda):
    x, w = torch.randn(4, 20, 64, generator=_gen(8)).half().to(cuda), torch.randn(64, 4, generator=_gen(9)).half().to(cuda)
    st = torch.randn(4, 3, 64, generator=_gen(10)).half().to(cuda)
    before = st.clone()
    out = conv1d_prompt(x, w, state=st, slots=torch.tensor([1, -1, 4, 1 << 30], dtype=torch.int32, device=cuda))
    assert torch.isnan(out[2:]).all() and torch.equal(out[1], conv1d_prompt(x[1:2], w)[0])
    assert torch.equal(st[[0, 2, 3]], before[[0, 2, 3]]) and torch.equal(st[1], x[0, -3:])


# ------------------------------------------------------------------------------------------------------------------- scan
def _dev(d, cuda):
    return {k: v.to(cuda) for k, v in d.items()}


def _check_scan(cuda, lens, H, P, G, N, dtype, *, packed=True, softplus=True, limit=(0.0, float("inf")), with_state=True, dt32=False, dhp=False,
                seed=0, **regime):
    T, n = sum(lens), len(lens)
    v = ssm_inputs(T, H, P, G, N, dtype, seed=seed, **regime)
    if dt32:
        v["dt"] = v["dt"].float()
    if not softplus:
        v["dt"] = v["dt"].abs() * 0.1
    if dhp:
        v["D"] = torch.randn(H, P, generator=_gen(seed + 1))
    state = 0.5 * torch.randn(n + 2, H, P, N, generator=_gen(seed + 2)) if with_state else None
    slots = torch.randperm(n + 2, generator=_gen(seed + 3))[:n].to(torch.int32)
    d = _dev(v, cuda)
    kw = dict(D=d["D"], dt_bias=d["dt_bias"] if softplus else None, dt_softplus=softplus, dt_limit=limit)
    args = [d[k] for k in ("x", "dt", "A", "B", "C")]
    st = None
    if with_state:
        st = state.to(cuda)
        kw.update(state=st, slots=slots.to(cuda))
    if packed:
        y = ssm_prompt(*args, **kw, seq_starts=starts_of(lens, cuda))
    else:
        y = ssm_prompt(*(a if a is d["A"] else a.unflatten(0, (n, lens[0])) for a in args), **kw).flatten(0, 1)
    first = state[slots.long()] if with_state else torch.zeros(n, H, P, N)
    wy, mag, ws, smag, most = ssm_ref(v["x"], v["dt"], v["A"], v["B"], v["C"], v["D"], v["dt_bias"] if softplus else None, softplus, limit, lens, first)
    rel = ssm_rel(lens, most)
    assert_near(y, wy, mag, ssm_y_rel(lens, most, dtype), "y")
    if with_state:
        assert_near(st[slots.long()], ws, smag, rel, "state")
        rest = [i for i in range(n + 2) if i not in slots.tolist()]
        assert torch.equal(st[rest].cpu(), state[rest])


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("lens", [[1], [2, 0, 63, 64, 65], [130], [0], [257, 1, 1, 40], [5] * 70, [600, 33]])
def test_ssm_prompt_lengths(cuda, dtype, lens):
    _check_scan(cuda, lens, H=4, P=64, G=1, N=128, dtype=dtype, seed=len(lens))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("H,P,G,N", [(1, 8, 1, 8), (6, 16, 2, 16), (3, 64, 1, 64), (8, 64, 8, 128), (5, 64, 1, 128), (2, 128, 1, 64), (4, 32, 2, 128),
                                     (3, 40, 1, 96), (2, 64, 1, 256), (7, 24, 7, 24), (2, 200, 1, 40)])
def test_ssm_prompt_shapes(cuda, dtype, H, P, G, N):
    _check_scan(cuda, [70, 3, 129], H, P, G, N, dtype, seed=H)


@pytest.mark.parametrize("form", [dict(with_state=False), dict(packed=False), dict(packed=False, with_state=False), dict(dt32=True), dict(dhp=True),
                                  dict(softplus=False), dict(limit=(0.01, 0.1)), dict(a_max=1.3, dt_mean=-4.5), dict(a_max=40.0, dt_mean=2.0)],
                         ids=lambda f: ",".join(f))
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_ssm_prompt_forms(cuda, dtype, form):
    _check_scan(cuda, [150, 150, 150], H=4, P=64, G=2, N=128, dtype=dtype, seed=11, **form)


def test_ssm_prompt_long(cuda):
    """Enough tokens that a sequence's work is divided, with strong and hardly any decay."""
    _check_scan(cuda, [2500], H=2, P=64, G=1, N=64, dtype=F16, seed=12)
    _check_scan(cuda, [1100, 2300, 17], H=2, P=64, G=1, N=128, dtype=BF16, seed=13, a_max=1.01, dt_mean=-7.0)


def test_ssm_prompt_views_and_tokens_of_nobody(cuda):
    """x, B and C as views of one row, dt as a slice; tokens outside the prompts are neither read nor written."""
    H, P, G, N, T = 4, 64, 1, 128, 200
    gen = _gen(14)
    xBC = torch.randn(T, H * P + 2 * G * N, generator=gen).half()
    raw = (torch.randn(T, H + 9, generator=gen) - 2).half()
    A = -torch.rand(H, generator=gen) - 1
    cut = lambda t: t.split([H * P, G * N, G * N], dim=-1)  # noqa: E731
    poisoned, praw = xBC.clone(), raw.clone()
    for t in (poisoned, praw):
        t[:10], t[110:] = NAN, NAN
    x, B, C = cut(poisoned.to(cuda))
    st = torch.zeros(2, H, P, N, device=cuda)
    y = ssm_prompt(x.view(T, H, P), praw.to(cuda)[:, 9:], A.to(cuda), B.view(T, G, N), C.view(T, G, N), state=st,
                   seq_starts=torch.tensor([10, 80, 110], dtype=torch.int32, device=cuda))
    x, B, C = (t[10:110] for t in cut(xBC))
    wy, mag, ws, smag, most = ssm_ref(x.reshape(-1, H, P), raw[10:110, 9:], A, B.reshape(-1, G, N), C.reshape(-1, G, N), None, None, True, (0.0, float("inf")),
                                      [70, 30], torch.zeros(2, H, P, N))
    assert_near(y[10:110], wy, mag, ssm_y_rel([70], most, F16), "y")
    assert_near(st, ws, smag, ssm_rel([70], most), "state")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("H,P,G,N", [(80, 64, 1, 128), (6, 16, 2, 8), (3, 40, 1, 96), (2, 64, 1, 256), (5, 8, 5, 16)])
def test_ssm_step(cuda, dtype, H, P, G, N):
    n = 5
    v = ssm_inputs(n, H, P, G, N, dtype, seed=15)
    state = torch.randn(n + 2, H, P, N, generator=_gen(16))
    slots = torch.tensor([6, 0, 3, 1, 4], dtype=torch.int32)
    d, st = _dev(v, cuda), state.to(cuda)
    y = ssm_step(st, d["x"], d["dt"], d["A"], d["B"], d["C"], D=d["D"], dt_bias=d["dt_bias"], slots=slots.to(cuda))
    wy, mag, ws, smag, _ = ssm_ref(v["x"], v["dt"], v["A"], v["B"], v["C"], v["D"], v["dt_bias"], True, (0.0, float("inf")), [1] * n, state[slots.long()])
    rel = 2.0 ** -20     # d by 4 units, its exponential by 6, a product and a sum; a sum over N in eight lanes
    assert_near(y, wy, mag, rel, "y")
    assert_near(st[slots.long()], ws, smag, rel, "state")
    assert torch.equal(st[[2, 5]].cpu(), state[[2, 5]])


def test_ssm_slots_out_of_range(cuda):
    v = _dev(ssm_inputs(80, 2, 64, 1, 128, F16, seed=17), cuda)
    st = torch.randn(3, 2, 64, 128, generator=_gen(18)).to(cuda)
    before = st.clone()
    bad = torch.tensor([1, -5, 3, 1 << 30], dtype=torch.int32, device=cuda)
    y = ssm_step(st, v["x"][:4], v["dt"][:4], v["A"], v["B"][:4], v["C"][:4], slots=bad)
    assert torch.isfinite(y[0]).all() and (y[1] == 0).all() and torch.isnan(y[2:]).all()
    assert torch.equal(st[[0, 2]], before[[0, 2]]) and not torch.equal(st[1], before[1])
    st = before.clone()
    args = [v[k] if k == "A" else v[k].unflatten(0, (4, 20)) for k in ("x", "dt", "A", "B", "C")]
    y = ssm_prompt(*args, state=st, slots=bad)
    assert torch.isnan(y[2:]).all() and torch.isfinite(y[:2]).all()
    assert torch.equal(y[1], ssm_prompt(*args)[1]) and torch.equal(st[[0, 2]], before[[0, 2]])


def test_ssm_large_steps_and_values(cuda):
    """d A far below the exponent's range (the state is forgotten), d of zero (nothing changes), and the largest activations."""
    v = ssm_inputs(96, 2, 64, 1, 64, F16, seed=19)
    v["dt"][10:20], v["dt"][40:50] = 60000.0, -60000.0
    v["x"][60], v["B"][61] = 60000.0, 60000.0
    v["x"] *= 2.0 ** -6
    d = _dev(v, cuda)
    st = torch.ones(1, 2, 64, 64, device=cuda)
    y = ssm_prompt(d["x"], d["dt"], d["A"], d["B"], d["C"], state=st, seq_starts=starts_of([96], cuda))
    wy, mag, ws, smag, most = ssm_ref(v["x"], v["dt"], v["A"], v["B"], v["C"], None, None, True, (0.0, float("inf")), [96], torch.ones(1, 2, 64, 64))
    assert_near(st, ws, smag, ssm_rel([96], 200.0), "state")   # (beyond 200 a weight is zero in 32 bits)
    fits = wy.abs() < 60000
    assert_near(torch.where(fits, y.cpu(), 0.0), torch.where(fits, wy, 0.0), mag, ssm_y_rel([96], 200.0, F16), "y")


@pytest.mark.parametrize("T", [100, 2500])
def test_starts_that_do_not_ascend(cuda, T):
    """Prompts that name the same tokens again and again: more chunks than there is workspace for.  Nothing is touched out of range, and
    the first one's state is what it is by itself."""
    v = _dev(ssm_inputs(T, 2, 64, 1, 64, F16, seed=31), cuda)
    args = [v[k] for k in ("x", "dt", "A", "B", "C")]
    st, alone = torch.zeros(16, 2, 64, 64, device=cuda), torch.zeros(1, 2, 64, 64, device=cuda)
    ssm_prompt(*args, state=st, seq_starts=torch.tensor([0, T] * 8 + [0], dtype=torch.int32, device=cuda))
    ssm_prompt(*args, state=alone, seq_starts=starts_of([T], cuda))
    torch.cuda.synchronize()
    scale = alone.abs().max()
    assert ((st[0] - alone[0]).abs().max() <= 2.0 ** -9 * scale).all()   # (cut into other segments, perhaps)
    x = v["x"].flatten(1)
    cst = torch.zeros(16, 3, 128, dtype=F16, device=cuda)
    conv1d_prompt(x, torch.ones(128, 4, device=cuda).half(), state=cst, seq_starts=torch.tensor([0, T] * 8 + [0], dtype=torch.int32, device=cuda))
    assert torch.equal(cst[0], x[T - 3:])


def test_ssm_nan_stays_in_its_sequence_and_head(cuda):
    v = ssm_inputs(300, 4, 64, 1, 128, BF16, seed=20)
    clean = _dev(v, cuda)
    run = lambda d, st: ssm_prompt(d["x"], d["dt"], d["A"], d["B"], d["C"], state=st, seq_starts=starts_of([100, 100, 100], cuda))  # noqa: E731
    s0 = torch.zeros(3, 4, 64, 128, device=cuda)
    y0 = run(clean, s0)
    d = {k: t.clone() for k, t in clean.items()}
    d["x"][150, 2, 5] = NAN
    d["dt"][250, 1] = NAN
    s1 = torch.zeros_like(s0)
    y1 = run(d, s1)
    assert torch.equal(y1[:100], y0[:100]) and torch.equal(s1[0], s0[0])
    assert torch.equal(y1[100:200, [0, 1, 3]], y0[100:200, [0, 1, 3]]) and torch.isnan(y1[150:200, 2, 5]).all()
    assert torch.equal(y1[200:, [0, 2, 3]], y0[200:, [0, 2, 3]]) and torch.isnan(y1[250:, 1]).all() and torch.isnan(s1[2, 1]).all()


# --------------------------------------------------------------------------------------------------- long offsets, streams
def test_states_past_32_bit_offsets(cuda):
    """A state pool of more than 2^31 entries and 2^33 bytes; the last slot is used."""
    H, P, N = 80, 64, 128
    slots = 2 ** 31 // (H * P * N) + 2
    st = torch.empty(slots, H, P, N, device=cuda)
    st[-1], st[-2] = 1.0, 2.0
    v = _dev(ssm_inputs(1, H, P, 1, N, F16, seed=21), cuda)
    small = torch.ones(1, H, P, N, device=cuda)
    y0 = ssm_step(small, v["x"], v["dt"], v["A"], v["B"], v["C"])
    last = torch.tensor([slots - 1], dtype=torch.int32, device=cuda)
    assert torch.equal(ssm_step(st, v["x"], v["dt"], v["A"], v["B"], v["C"], slots=last), y0) and torch.equal(st[-1], small[0]) and (st[-2] == 2.0).all()
    small.fill_(1.0)
    st[-1] = 1.0
    y0 = ssm_prompt(v["x"], v["dt"], v["A"], v["B"], v["C"], state=small, seq_starts=starts_of([1], cuda))
    y1 = ssm_prompt(v["x"], v["dt"], v["A"], v["B"], v["C"], state=st, slots=last, seq_starts=starts_of([1], cuda))
    assert torch.equal(y0, y1) and torch.equal(st[-1], small[0]) and (st[-2] == 2.0).all()


def test_rows_past_32_bit_offsets(cuda):
    """Rows far enough apart that the last ones lie past 2^31 elements."""
    rows, D = 70, 2560
    big = torch.zeros((rows - 1) * (1 << 25) + D, dtype=F16, device=cuda)
    x = big.as_strided((rows, D), (1 << 25, 1))
    x.copy_(torch.randn(rows, D, generator=_gen(22)).half().to(cuda))
    w = torch.ones(D, device=cuda)
    assert torch.equal(residual_rmsnorm(x, w)[0], residual_rmsnorm(x.clone(), w)[0])
    assert torch.equal(quantize_rows(x)[0], quantize_rows(x.clone())[0])
    taps = torch.randn(D, 4, generator=_gen(23)).half().to(cuda)
    assert torch.equal(conv1d_prompt(x.unsqueeze(0), taps), conv1d_prompt(x.clone().unsqueeze(0), taps))
    st = torch.zeros(rows, 3, D, dtype=F16, device=cuda)
    assert torch.equal(conv1d_step(x, st, taps), conv1d_step(x.clone(), torch.zeros_like(st), taps))


def test_calls_on_two_streams_and_in_a_graph(cuda):
    """Two calls at once on streams of their own, and a graph of all operators replayed with eager work in between."""
    v = _dev(ssm_inputs(700, 4, 64, 1, 128, F16, seed=24), cuda)
    starts = starts_of([300, 400], cuda)
    w = torch.randn(64, 4, generator=_gen(25)).half().to(cuda)
    wq = _codes((96, 64), _gen(26)).to(cuda)
    ws = torch.full((96,), 0.01, device=cuda)
    nw = torch.ones(64, device=cuda)

    def work(conv, ssm):
        x = v["x"].flatten(0, 1)[:700]
        y, r = residual_rmsnorm(x, nw)
        c = conv1d_prompt(y, w, activation="silu", state=conv, seq_starts=starts)
        q, s = quantize_rows(c)
        p = int8_matmul(q, wq, s, ws)
        t = ssm_prompt(v["x"], v["dt"], v["A"], v["B"], v["C"], state=ssm, seq_starts=starts)
        u = ssm_step(ssm, v["x"][:2], v["dt"][:2], v["A"], v["B"][:2], v["C"][:2])
        return [y, r, c, p, t, u, conv1d_step(y[:2], conv, w)]

    def fresh():
        return torch.zeros(2, 3, 64, dtype=F16, device=cuda), torch.zeros(2, 4, 64, 128, device=cuda)

    st = fresh()
    want = [t.clone() for t in work(*st)] + [t.clone() for t in st]
    torch.cuda.synchronize()
    streams, got, states = [torch.cuda.Stream(), torch.cuda.Stream()], [None, None], [fresh(), fresh()]
    torch.cuda.synchronize()
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            got[i] = work(*states[i])
    torch.cuda.synchronize()
    for i in range(2):
        for a, b in zip([*got[i], *states[i]], want):
            assert torch.equal(a, b)
    st = fresh()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = work(*st)
    for _ in range(4):
        for t in st:
            t.zero_()
        for t in captured:
            t.fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip([*captured, *st], want):
            assert torch.equal(a, b)
        other = fresh()
        for a, b in zip([*work(*other), *other], want):
            assert torch.equal(a, b)
