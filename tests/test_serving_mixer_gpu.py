"""The mixer's serving calls: prompts in parts, packed and padded, then single tokens, each stage against a plain form on the tensors
that the mixer itself fed it; two blocks in a row, eager and as a graph; and the operators' native short calls against their
general path."""

import pytest
import torch

from linquant_amd.kernels.mamba2.conv1d_state import conv1d_prompt, conv1d_step
from linquant_amd.kernels.mamba2.ssm import ssm_prompt, ssm_step
from linquant_amd.norm import RMSNormGated, residual_rmsnorm, rmsnorm_gated_qhad
from linquant_amd.quantized_mamba2 import Int8InputLinear, Mamba2Block, QuantizedMamba2, random_calibrated_mixer
from linquant_amd.w8a8_linear import W8A8Linear, int8_matmul, quantize_rows
from tests.serving_cases import HALF_STEP, assert_near, conv_ref, ssm_inputs, ssm_ref, ssm_rel, ssm_y_rel, starts_of
from tests.test_native_calls_gpu import _both, _unaligned

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
CONV_REL = 2.0 ** -20     # as for the convolution alone
LINEAR_REL = 2.0 ** -22   # an exact sum times two scales, one after the other, and a bias


def build(linear=W8A8Linear, ngroups=1, nheads=8, d_state=64, rows=True, seed=3):
    """A mixer that is not calibrated, which serving does not need."""
    gen = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    d_model, headdim = 264, 512 // nheads
    d_ssm = 512   # with four heads, projected rows are not whole 16-byte pieces
    conv_dim = d_ssm + 2 * ngroups * d_state
    proj = [torch.nn.Linear(d_model, d_ssm + conv_dim + nheads, bias=False), torch.nn.Linear(d_ssm, d_model, bias=False)]
    for p in proj:
        p.weight.data.copy_(rn(*p.weight.shape) / p.in_features ** 0.5)
    conv = torch.nn.Conv1d(conv_dim, conv_dim, 4, groups=conv_dim)
    conv.weight.data.copy_(rn(conv_dim, 1, 4) * 0.5)
    conv.bias.data.copy_(rn(conv_dim) * 0.1)
    norm = RMSNormGated(d_ssm, group_size=d_ssm // ngroups)
    norm.weight.data.copy_(1 + 0.1 * rn(d_ssm))
    m = QuantizedMamba2(d_model=d_model, d_ssm=d_ssm, nheads=nheads, headdim=headdim, d_state=d_state, ngroups=ngroups, d_conv=4, chunk_size=64,
                        in_proj=linear.from_fp16(proj[0], None if rows and linear is W8A8Linear else torch.tensor(0.03)),
                        out_proj=linear.from_fp16(proj[1], torch.tensor(0.04)), conv1d=conv.half(), norm=norm,
                        A_log=torch.randint(0, 128, (nheads,), generator=gen).to(torch.int8), D=torch.randint(60, 128, (nheads,), generator=gen).to(torch.int8).cuda(),
                        dt_bias=torch.full((nheads,), -2.0).cuda())
    m.register_buffer("A_log_scale", torch.tensor(2.75 / 127))
    m.register_buffer("D_scale", torch.tensor(0.01))
    m.register_buffer("comp_out", (rn(d_model) * 0.01).half())
    return m.cuda()


def tokens(n, m, seed):
    return (torch.randn(n, m.d_model, generator=torch.Generator().manual_seed(seed)) * 0.9).half()


def check_linear(lin, codes, scale, got, what, extra=None):
    codes, w = codes.double().cpu(), lin.weight[:, :lin.in_features].double().cpu()
    want = codes @ w.T * torch.as_tensor(scale).double().cpu().reshape(-1, 1) * lin.weight_scale.double().cpu()
    if extra is None:
        return assert_near(got, want, want.abs(), LINEAR_REL, what)
    # the sum of two fp16 numbers: the product's rounding comes before the sum's
    assert_near(got, want + extra.double().cpu(), want.abs(), HALF_STEP[F16] * 1.01, what)


def check_call(m, hidden, dbg, lens, before, after, slots, rows):
    """One call, its stages on the mixer's own tensors.  ``rows``: the rows of the call's tokens that belong to the sequences;
    before, after: the state on the CPU in front of the call and behind it; slots: (n,) a negative one without a state."""
    t = {k: v.detach().cpu().reshape(-1, v.shape[-1] if k not in ("y",) else m.d_ssm)[rows] for k, v in dbg.items()}
    if isinstance(m.in_proj, W8A8Linear):
        codes, scale = quantize_rows(hidden.cuda())
        check_linear(m.in_proj, codes.reshape(-1, m.d_model)[rows], scale.flatten()[rows], t["projected"], "in_proj")
        check_linear(m.out_proj, t["y_i8"], m.out_proj.input_scale, t["out"], "out_proj", m.comp_out)
    p, H, G, N = t["projected"], m.nheads, m.ngroups, m.d_state
    z, xBC, dt = p[:, :m.d_ssm], p[:, m.d_ssm:m.d_ssm + m.conv_dim], p[:, m.d_ssm + m.conv_dim:]
    assert dt.shape[1] == H and torch.equal(dt, t["dt"]) and torch.equal(z, t["z"])

    conv = torch.stack([before.conv[s] if s >= 0 else torch.zeros_like(before.conv[0]) for s in slots])
    ssm = torch.stack([before.ssm[s] if s >= 0 else torch.zeros_like(before.ssm[0]) for s in slots])
    y, mag, conv_after = conv_ref(xBC, m.conv1d.weight.detach().cpu().reshape(m.conv_dim, -1), m.conv1d.bias.detach().cpu(), True, lens, conv)
    assert_near(t["xBC"], y, mag, CONV_REL, "conv")

    A = -torch.exp(m.A_log.float() * m.A_log_scale.float()).cpu()
    D = (m.D.float() * m.D_scale.float()).cpu()
    x, B, C = t["xBC"].split([m.d_ssm, G * N, G * N], 1)
    T = len(x)
    y, mag, ssm_after, smag, most = ssm_ref(x.reshape(T, H, -1), dt, A, B.reshape(T, G, N), C.reshape(T, G, N), D, m.dt_bias.cpu(), True,
                                            m.dt_limit, lens, ssm)
    # A and D come from the exponential and a product in fp32, the oracle's from the same fp32 numbers
    rel = ssm_rel(lens, most)
    assert_near(t["y"], y.reshape(T, -1), mag.reshape(T, -1), ssm_y_rel(lens, most, F16), "scan")
    y_i8, _ = rmsnorm_gated_qhad(t["y"].cuda(), t["z"].cuda(), m.norm.weight, m.out_proj.input_scale, m.norm.eps, m.norm.group_size)
    assert torch.equal(y_i8.cpu(), t["y_i8"])

    kept = set()
    for i, s in enumerate(slots):
        if s >= 0:
            kept.add(s)
            assert torch.equal(after.conv[s], conv_after[i].half())
            assert_near(after.ssm[s], ssm_after[i], smag[i], rel, "state")
    for s in range(len(before.conv)):
        if s not in kept:
            assert torch.equal(after.conv[s], before.conv[s]) and torch.equal(after.ssm[s], before.ssm[s])


def snapshot(state):
    return type(state)(*(t.cpu() for t in state))


@pytest.mark.parametrize("linear", [W8A8Linear, Int8InputLinear])
@pytest.mark.parametrize("ngroups,nheads,d_state", [(1, 8, 64), (2, 4, 128)])
def test_prompts_in_parts_then_tokens(cuda, linear, ngroups, nheads, d_state):
    m = build(linear, ngroups, nheads, d_state)
    st = m.allocate_state(6)
    for lens, slots, front, seed in [([70, 1, 0, 33], [4, 0, 2, 5], 2, 1), ([3, 64, 65, 5], [2, 4, -1, 0], 0, 2)]:
        hidden, before, dbg = tokens(front + sum(lens) + 1, m, seed), snapshot(st), {}
        out = m.prefill(hidden.cuda(), st, torch.tensor(slots, dtype=torch.int32, device=cuda), starts_of(lens, cuda, first=front), _debug=dbg)
        assert out.shape == hidden.shape and out.dtype == F16
        check_call(m, hidden, dbg, lens, before, snapshot(st), slots, slice(front, front + sum(lens)))
    for seed in (3, 4):
        hidden, before, dbg, slots = tokens(5, m, seed), snapshot(st), {}, [5, 2, -1, 4, 0]
        out = m.step(hidden.cuda(), st, torch.tensor(slots, dtype=torch.int32, device=cuda), _debug=dbg)
        assert out.shape == hidden.shape and torch.isfinite(out).all()
        real = [i for i, s in enumerate(slots) if s >= 0]
        check_call(m, hidden, dbg, [1] * len(real), before, snapshot(st), [slots[i] for i in real], real)


def test_batch_without_slots_and_bf16(cuda):
    m = build(ngroups=2)
    st = m.allocate_state(3)
    hidden, dbg = tokens(3 * 40, m, 5).view(3, 40, -1).bfloat16(), {}
    before = snapshot(st)
    out = m.prefill(hidden.cuda(), st, _debug=dbg)
    assert out.shape == hidden.shape and out.dtype == F16
    check_call(m, hidden.half(), dbg, [40] * 3, before, snapshot(st), [0, 1, 2], slice(None))
    again = m.allocate_state(3)
    assert torch.equal(m.prefill(quantize_rows(hidden.half().cuda()), again), out)      # codes in place of activations
    assert all(torch.equal(a, b) for a, b in zip(again, st))


def test_static_scales_and_the_int8_forward(cuda):
    """One input scale for the tensor; ``forward`` runs on the same projections."""
    m, _ = random_calibrated_mixer(d_model=264, nheads=8, headdim=64, d_state=64, ngroups=1, chunk_size=64, seqlen=128, linear=W8A8Linear)
    m.register_buffer("comp_out", torch.linspace(-0.02, 0.02, 264).half().cuda())
    hidden, dbg = tokens(2 * 64, m, 6).view(2, 64, -1).cuda(), {}
    out = m(hidden, _debug=dbg)
    assert torch.isfinite(out).all()
    check_linear(m.in_proj, dbg["h_i8"].reshape(-1, m.d_model), m.in_proj.input_scale, dbg["projected"].reshape(128, -1), "in_proj")
    check_linear(m.out_proj, dbg["y_i8"].reshape(128, -1), m.out_proj.input_scale, dbg["out"].reshape(128, -1), "out_proj", m.comp_out)
    st, served = m.allocate_state(2), {}
    m.prefill(hidden, st, _debug=served)
    assert torch.equal(served["projected"], dbg["projected"])
    m.in_proj.input_scale = None
    m(hidden, _debug=dbg)                                          # a scale for each row
    assert dbg["h_i8"] is None
    codes, scale = quantize_rows(hidden)
    check_linear(m.in_proj, codes.reshape(128, -1), scale.flatten(), dbg["projected"].reshape(128, -1), "in_proj")


@pytest.mark.parametrize("rows", [True, False])
def test_blocks_as_a_model_runs_them(cuda, rows):
    """Two blocks: packed prompts, then tokens, eager and as a graph that is replayed with eager work between the replays."""
    gen = torch.Generator().manual_seed(7)
    blocks = [Mamba2Block(m, (1 + 0.1 * torch.randn(m.d_model, generator=gen)).half().cuda()) for m in (build(rows=rows, seed=3), build(rows=rows, seed=8))]
    lens, slots = [30, 65, 2], torch.tensor([2, 0, 3], dtype=torch.int32, device=cuda)
    starts = starts_of(lens, cuda)
    prompt, steps = tokens(sum(lens), blocks[0].mixer, 9).cuda(), tokens(3 * 4, blocks[0].mixer, 10).view(4, 3, -1).cuda()

    def plain(block, x, residual, state, call):
        """The block without its fusion."""
        r = x.float() + (0 if residual is None else residual)
        m = block.mixer
        codes, scale, r2 = residual_rmsnorm(x, block.norm_weight, residual, quantize="rows" if rows else m.in_proj.input_scale, residual_dtype=torch.float32 if residual is None else None)
        assert torch.equal(r, r2)
        return call(m, (codes, scale), state), r2

    states = [b.mixer.allocate_state(4) for b in blocks]
    other = [b.mixer.allocate_state(4) for b in blocks]
    x, r, u, v = prompt, None, prompt, None
    for b, s, o in zip(blocks, states, other):
        x, r = b.prefill(x, r, s, slots, starts)
        u, v = plain(b, u, v, o, lambda m, h, q: m.prefill(h, q, slots, starts))
        assert torch.equal(x, u) and torch.equal(r, v) and r.dtype == torch.float32
    after_prompt = [[t.clone() for t in s] for s in states]

    def token(x, sts):
        r = None
        for b, s in zip(blocks, sts):
            x, r = b.step(x, r, s, slots)
        return x, r

    want = [tuple(t.clone() for t in token(h, states)) for h in steps]
    # the same from a graph
    held = steps[0].clone()
    graph = torch.cuda.CUDAGraph()
    token(held, other)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = token(held, other)
    for o, s in zip(other, after_prompt):
        for a, b in zip(o, s):
            a.copy_(b)
    for h, (x, r) in zip(steps, want):
        held.copy_(h)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], x) and torch.equal(got[1], r)
        token(h, [b.mixer.allocate_state(4) for b in blocks])
        got[0].fill_(3.0)
    for o, s in zip(other, states):
        assert all(torch.equal(a, b) for a, b in zip(o, s))


# ------------------------------------------------------------------------------------------------- native short calls
def _scan_case(cuda, form):
    v = {k: t.to(cuda) for k, t in ssm_inputs(40, 4, 16, 2, 32, BF16 if form == "bf16" else F16, seed=1).items()}
    if form == "dt fp32":
        v["dt"] = v["dt"].float()
    if form == "A unaligned":
        v["A"] = _unaligned(v["A"])
    if form == "D of heads and rows":
        v["D"] = v["D"][:, None] + torch.zeros(4, 16, device=cuda)
    if form == "A fp16":
        v["A"] = v["A"].half()
    if form == "x unaligned":
        v["x"] = _unaligned(v["x"])
    if form == "x of views":
        v["x"] = torch.cat([v["x"], v["x"]], -1)[..., :16]
    kw = dict(D=None if form == "no D" else v["D"], dt_bias=None if form == "no bias" else v["dt_bias"])
    if form == "limit":
        kw.update(dt_softplus=False, dt_limit=(0.0, 0.05))
    return [v[k] for k in ("x", "dt", "A", "B", "C")], kw


SCAN = {"plain": True, "bf16": True, "dt fp32": True, "no D": True, "no bias": True, "limit": True, "D of heads and rows": True,
        "x of views": True, "x unaligned": False, "A fp16": False, "A unaligned": True, "slots": True, "no state": None}


@pytest.mark.parametrize("form", list(SCAN))
def test_native_scan(cuda, monkeypatch, form):
    args, kw = _scan_case(cuda, form)
    starts, state = starts_of([30, 0, 10], cuda), torch.randn(4, 4, 16, 32, generator=torch.Generator().manual_seed(2)).to(cuda)
    if form == "slots":
        kw["slots"] = torch.tensor([3, -1, 0], dtype=torch.int32, device=cuda)

    def prompt():
        s = state.clone()
        return ssm_prompt(*args, **kw, **({} if form == "no state" else dict(state=s)), seq_starts=starts), s

    if SCAN[form] is None:
        y = prompt()[0]
        monkeypatch.setattr("linquant_amd._lib.native", lambda: pytest.fail("offered"))
        assert torch.equal(prompt()[0], y)
        return
    _both(monkeypatch, "ssm_prompt", prompt, SCAN[form])

    def step():
        s = state.clone()
        x, dt, A, B, C = args
        return ssm_step(s, *(t if t is A else t[:3] for t in (x, dt, A, B, C)), **kw), s

    _both(monkeypatch, "ssm_step", step, SCAN[form])


@pytest.mark.parametrize("form,native", [("plain", True), ("bf16", True), ("no bias", True), ("no activation", True), ("slots", True), ("weight fp32", False),
                                         ("weight unaligned", False), ("x unaligned", False), ("x of views", True)])
def test_native_convolution(cuda, monkeypatch, form, native):
    gen = torch.Generator().manual_seed(4)
    dtype = BF16 if form == "bf16" else F16
    x, w, b = (torch.randn(*s, generator=gen).to(dtype).to(cuda) for s in ((50, 64), (64, 4), (64,)))
    state = torch.randn(4, 3, 64, generator=gen).to(dtype).to(cuda)
    w = w.float() if form == "weight fp32" else _unaligned(w) if form == "weight unaligned" else w
    x = _unaligned(x) if form == "x unaligned" else torch.cat([x, x], 1)[:, :64] if form == "x of views" else x
    bias, act = None if form == "no bias" else b, None if form == "no activation" else "silu"
    slots = torch.tensor([2, -3, 0], dtype=torch.int32, device=cuda) if form == "slots" else None

    def prompt():
        s = state.clone()
        return conv1d_prompt(x, w, bias, act, state=s, slots=slots, seq_starts=starts_of([20, 3, 27], cuda)), s

    def step():
        s = state.clone()
        return conv1d_step(x[:3], s, w, bias, act, slots=slots), s

    _both(monkeypatch, "conv1d_prompt", prompt, native)
    _both(monkeypatch, "conv1d_step", step, native)


@pytest.mark.parametrize("form,native", [("plain", True), ("rows", True), ("fp32 stream", True), ("gates", True), ("gate of a channel", True), ("post", True),
                                         ("gate of a prompt", False), ("post of another type", False), ("x of views", False), ("no residual", False)])
def test_native_norm(cuda, monkeypatch, form, native):
    gen = torch.Generator().manual_seed(5)
    rn = lambda *s: torch.randn(*s, generator=gen).half().to(cuda)  # noqa: E731
    x, res, w = rn(3, 7, 136), rn(3, 7, 136), rn(136)
    kw = {"rows": dict(quantize="rows"), "gates": dict(gate=rn(3, 7, 136), scale=0.5), "gate of a channel": dict(gate=rn(136)), "post": dict(post_weight=rn(136)),
          "gate of a prompt": dict(gate=rn(3, 1, 136)), "post of another type": dict(post_weight=rn(136).float())}.get(form, {})
    if form == "x of views":
        x = torch.cat([x, x], -1)[..., :136]
    residual = None if form == "no residual" else res.float() if form == "fp32 stream" else res
    _both(monkeypatch, "residual_rmsnorm", lambda: residual_rmsnorm(x, w, residual, 1e-5, **kw), native)


@pytest.mark.parametrize("form,native", [("plain", True), ("bias", True), ("bf16", True), ("one scale", True), ("number", False), ("unaligned", False), ("ragged", False),
                                         ("batch", False)])
def test_native_linear(cuda, monkeypatch, form, native):
    gen = torch.Generator().manual_seed(6)
    K = 100 if form == "ragged" else 96
    a, b = (torch.randint(-128, 128, s, generator=gen).to(torch.int8).to(cuda) for s in ((33, K), (72, K)))
    xs, ws = torch.rand(33, generator=gen).to(cuda), torch.rand(72, generator=gen).to(cuda)
    xs = 0.25 if form == "number" else xs[:1] if form == "one scale" else xs
    a = _unaligned(a) if form == "unaligned" else a[:32].view(2, 16, K) if form == "batch" else a
    xs = xs[:32] if form == "batch" else xs
    bias = torch.randn(72, generator=gen).to(cuda) if form == "bias" else None
    _both(monkeypatch, "int8_matmul", lambda: int8_matmul(a, b, xs, ws, bias, BF16 if form == "bf16" else F16), native)
    x = torch.randn(33, K, generator=gen).half().to(cuda)
    x = x.view(3, 11, K) if form == "batch" else x
    _both(monkeypatch, "quantize_rows", lambda: quantize_rows(x), form != "batch")
