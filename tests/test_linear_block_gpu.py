"""A linear attention block that answers for many requests, its operators together: projections with an adapter for each request, prompts and
single tokens from slots, the gated group norm, slots forked and compacted; and their native short calls against the general path."""

import pytest
import torch

from linquant_amd import _lib
from linquant_amd.kernels.zoo import linear_attention_prompt, linear_attention_step
from linquant_amd.norm import groupnorm_gated
from linquant_amd.quantized_mamba2 import Mamba2State
from linquant_amd.slots import copy_slots
from linquant_amd.w8a8_linear import LowRankAdapters, W8A8Linear, quantize_rows
from tests.attention_cases import adapters_ref, attention_inputs, attention_ref, norm_ref, out_rel, state_rel
from tests.serving_cases import assert_near, starts_of

pytestmark = pytest.mark.gpu

F16, BF16, F32, I32 = torch.float16, torch.bfloat16, torch.float32, torch.int32


class _Block:
    """Two projections with adapters around linear attention of 4 heads with a decay each; every stage gives what it took and gave."""

    def __init__(self, cuda, dtype, seed=0, D=256, H=4, K=64, V=72, R=8, n=3):
        gen = torch.Generator().manual_seed(seed)
        self.H, self.K, self.V, self.dtype = H, K, V, dtype
        self.wide = H * (2 * K + 2 * V)
        self.g = torch.log1p(-torch.exp2(-2.0 - torch.arange(H))).to(cuda)
        self.norm_w = (1 + 0.2 * torch.randn(H * V, generator=gen)).to(dtype).to(cuda)
        self.proj = []
        for k, m in ((D, self.wide), (H * V, D)):
            w = torch.randn(m, k, generator=gen) / k ** 0.5
            ws = w.abs().amax(1) / 127.0
            codes = torch.round(w / ws[:, None]).to(torch.int8)
            a, b = (torch.randn(n, R, k, generator=gen) / k ** 0.5).to(dtype), (torch.randn(n, m, R, generator=gen) / R ** 0.5).to(dtype)
            s = 0.25 + torch.rand(n, generator=gen)
            self.proj.append((W8A8Linear(codes, ws).to(cuda), LowRankAdapters(a, b, s).to(cuda), (codes, ws, a, b, s)))

    def state(self, slots, cuda):
        return torch.zeros(slots, self.H, self.K, self.V, device=cuda)

    def __call__(self, x, ids, state, slots, starts=None):
        (inp, a1, _), (out, a2, _) = self.proj
        H, K, V = self.H, self.K, self.V
        y = inp(x, adapters=a1, ids=ids)
        q, k, v, z = y.split([H * K, H * K, H * V, H * V], -1)
        q, k, v = (t.unflatten(-1, (H, -1)) for t in (q, k, v))
        if starts is None:
            o = linear_attention_step(state, q, k, v, self.g, slots=slots)
        else:
            o = linear_attention_prompt(q, k, v, self.g, state=state, slots=slots, seq_starts=starts)
        n = groupnorm_gated(o.flatten(-2), z, self.norm_w, num_groups=H)
        return y, o, n, out(n, adapters=a2, ids=ids)


def _check_stages(block, x, ids, lens, before, after, got, step):
    """Each stage against the plain form of what it took; ``before``, ``after`` (n, H, K, V): the sequences' states."""
    y, o, n, out = got
    H, K, V = block.H, block.K, block.V
    ids = ids.cpu()
    for i, (taken, gave) in enumerate(((x, y), (n, out))):
        codes, ws, a, b, s = block.proj[i][2]
        q, qs = quantize_rows(taken)
        want, mag, low = adapters_ref(q.cpu(), qs.cpu(), codes, ws, None, taken.cpu(), a, b, s, ids)
        # as for the adapters alone: sums of K and R terms in 32 bits, h in two pieces
        assert_near(gave, want, mag * 4 * 2.0 ** -24 + low * (2.0 ** -24 * (taken.shape[-1] / 8 + a.shape[1] + 16) + 2.0 ** -14), 1.0, f"projection {i}")
    q, k, v, z = y.cpu().split([H * K, H * K, H * V, H * V], -1)
    q, k, v = (t.unflatten(-1, (H, -1)) for t in (q, k, v))
    want, mag, S, Sm, most = attention_ref(q, k, v, block.g.cpu(), K ** -0.5, lens, before)
    rel, srel = (2.0 ** -24 * (16 + K), 2.0 ** -24 * 6) if step else (out_rel(lens, most, block.dtype), state_rel(lens, most))
    assert_near(o, want, mag, rel, "o")
    assert_near(after, S, Sm, srel, "state")
    want, off = norm_ref(o.cpu().flatten(-2), z, block.norm_w.cpu(), None, H, 1e-5, "silu")
    assert_near(n, want, off, 2.0 ** -24, "norm")


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_requests_from_prompt_to_fork_to_compaction(cuda, dtype):
    gen = torch.Generator().manual_seed(1)
    block = _Block(cuda, dtype)
    state = block.state(6, cuda)
    state[4] = 3.0                                                                       # (a slot of an earlier request)
    idx = lambda *i: torch.tensor(i, dtype=I32, device=cuda)  # noqa: E731
    copy_slots(state, idx(-1), idx(4))
    assert (state == 0).all()
    lens, slots = [70, 1, 130], [4, 0, 2]
    x = torch.randn(sum(lens), 256, generator=gen).to(dtype).to(cuda)
    ids = torch.repeat_interleave(torch.tensor([2, -1, 0], dtype=I32), torch.tensor(lens)).to(cuda)
    got = block(x, ids, state, idx(*slots), starts_of(lens, cuda))
    _check_stages(block, x, ids, lens, torch.zeros(3, *state.shape[1:]), state[slots], got, False)
    assert (state[[1, 3, 5]] == 0).all()
    copy_slots(state, idx(2, 2, 4), idx(1, 5, 3))                                        # request 2 in three beams, request 0 in two
    assert all(torch.equal(state[a], state[b]) for a, b in ((1, 2), (5, 2), (3, 4)))
    slots, who = [4, 0, 2, 1, -1, 5, 3], [2, -1, 0, 0, 1, 1, 2]                          # (a padding entry among them; one beam takes another adapter)
    for t in range(3):
        x = torch.randn(7, 256, generator=gen).to(dtype).to(cuda)
        live = [i for i in range(7) if slots[i] >= 0]
        before = state[[max(s, 0) for s in slots]].clone()
        got = block(x, idx(*who), state, idx(*slots))
        assert (got[1][4] == 0).all()
        _check_stages(block, x[live], idx(*who)[live], [1] * 6, before[live].cpu(), state[[slots[i] for i in live]], [g[live] for g in got], True)
    kept = state.clone()
    copy_slots(state, idx(5, 3, 0, -1, -1, -1), idx(0, 1, 2, 3, 4, 5))                   # the three that go on move to the front
    assert torch.equal(state[:3], kept[[5, 3, 0]]) and (state[3:] == 0).all()


def test_captured_steps_over_changing_requests(cuda):
    """A step and a move of slots in a graph, replayed with other requests, adapters and moves; the program works between the replays."""
    gen = torch.Generator().manual_seed(2)
    block = _Block(cuda, F16)
    state = torch.randn(block.state(8, cuda).shape, generator=gen).to(cuda)
    expect = state.clone()
    x = torch.randn(5, 256, generator=gen).half().to(cuda)
    ids, slots, src, dst = (torch.tensor(t, dtype=I32, device=cuda) for t in ([0, 1, 2, -1, 0], [0, 1, 2, 3, -1], [0, -1], [7, 6]))
    block(x, ids, block.state(8, cuda), slots)
    copy_slots(block.state(8, cuda), src, dst)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = block(x, ids, state, slots)
        copy_slots([state], src, dst)
    for i in range(4):
        x.normal_()
        ids.copy_(torch.randint(-1, 3, (5,), generator=gen))
        slots.copy_(torch.randperm(8, generator=gen)[:5])
        src.copy_(torch.randint(-1, 8, (2,), generator=gen)), dst.copy_(torch.randperm(8, generator=gen)[:2])
        graph.replay()
        torch.cuda.synchronize()
        want = block(x, ids, expect, slots)
        copy_slots([expect], src, dst)
        assert all(torch.equal(a, b) for a, b in zip(out, want)) and torch.equal(state, expect)


def test_two_graphs_and_two_streams(cuda):
    """Prompts cut into segments, whose calls have workspaces, captured twice and run on two streams side by side."""
    block = _Block(cuda, BF16)
    gen = torch.Generator().manual_seed(3)
    xs = [torch.randn(2200, 256, generator=gen).to(BF16).to(cuda) for _ in range(2)]
    ids, starts, slot = torch.zeros(2200, dtype=I32, device=cuda), starts_of([2000, 200], cuda), torch.tensor([1, 0], dtype=I32, device=cuda)
    want = []
    for x in xs:
        s = block.state(2, cuda)
        want.append((block(x, ids, s, slot, starts)[-1], s))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    for i in range(3):
        got = []
        for x, stream in zip(xs, streams):
            with torch.cuda.stream(stream):
                s = block.state(2, cuda)
                got.append((block(x, ids, s, slot, starts)[-1], s))
        torch.cuda.synchronize()
        assert all(torch.equal(a[j], b[j]) for a, b in zip(got, want) for j in (0, 1))
    graphs, got = [], []
    for x in xs:
        s, graph = block.state(2, cuda), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = block(x, ids, s, slot, starts)[-1]
        graphs.append(graph), got.append((y, s))
    torch.cuda.synchronize()
    for i in range(3):
        for _, s in got:
            s.zero_()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a[j], b[j]) for a, b in zip(got, want) for j in (0, 1))


def test_slots_of_a_mixers_state(cuda):
    """The states of two mixers, each a convolution's and a scan's, and tensors whose slots lie between each other's."""
    gen = torch.Generator().manual_seed(4)
    layers = [Mamba2State(torch.randn(5, 3, 40, generator=gen).half().to(cuda), torch.randn(5, 2, 8, 16, generator=gen).to(cuda)) for _ in range(2)]
    both = torch.randn(5, 2, 36, generator=gen).to(cuda)
    old = [(c.clone(), s.clone()) for c, s in layers], both.clone()
    src, dst = (torch.tensor(t, dtype=I32, device=cuda) for t in ([0, 0, 4, -1], [1, 2, 0, 4]))
    copy_slots([layers, both[:, 0], both[:, 1]], src, dst)
    take = [4, 0, 0, 3]
    for (c, s), (c0, s0) in zip(layers, old[0]):
        assert torch.equal(c[:4], c0[take]) and torch.equal(s[:4], s0[take]) and not c[4].any() and not s[4].any()
    assert torch.equal(both[:4], old[1][take]) and not both[4].any()
    with pytest.raises(AssertionError, match="overlap"):
        copy_slots([both[:, 0], both], src, dst)
    loop = [both]
    loop.append(loop)
    with pytest.raises(RecursionError):
        copy_slots(loop, src, dst)


@pytest.mark.parametrize("M,K,n", [(65, 128, 3), (130, 250, 70), (256, 128, 2000), (257, 128, 5), (511, 64, 40), (700, 128, 2000), (1300, 130, 6), (1537, 64, 900)])
@pytest.mark.parametrize("ids", ["in turn", "random", "far apart", "few changes", "pairs"])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_rows_of_many_adapters_in_any_order(cuda, M, K, n, ids, dtype):
    """Rows are taken in an order by their adapters and come back in their own; twice the same."""
    gen = torch.Generator().manual_seed(M + n)
    N, R = 70, 16
    codes = torch.randint(-127, 128, (N, K), generator=gen).to(torch.int8)
    ws = torch.rand(N, generator=gen) / 1000
    a, b, s = (torch.randn(n, R, K, generator=gen) / K ** 0.5).to(dtype), (torch.randn(n, N, R, generator=gen) / 4).to(dtype), 0.25 + torch.rand(n, generator=gen)
    lin, ad = W8A8Linear(codes, ws).to(cuda), LowRankAdapters(a, b, s).to(cuda)
    x = torch.randn(M, K, generator=gen).to(dtype)
    t = torch.arange(M)
    idx = {"in turn": t % n, "random": torch.randint(-1, n + 1, (M,), generator=gen), "far apart": (t * 512 + t // 3 * 7) % n, "few changes": t * 9 // M % n,
           "pairs": t // 2 * 5 % n}[ids].to(I32)
    q, qs = quantize_rows(x.to(cuda))
    want, mag, low = adapters_ref(q.cpu(), qs.cpu(), codes, ws, None, x, a, b, s, idx)
    got = lin(x.to(cuda), adapters=ad, ids=idx.to(cuda))
    # as for a few adapters: sums of K and R terms in 32 bits, h in two pieces
    assert_near(got, want, mag * 4 * 2.0 ** -24 + low * (2.0 ** -24 * (K / 8 + R + 16) + 2.0 ** -14), 1.0, "adapted")
    assert torch.equal(torch.nan_to_num(lin(x.to(cuda), adapters=ad, ids=idx.to(cuda))), torch.nan_to_num(got))


@pytest.mark.parametrize("M", [300, 4113])
@pytest.mark.parametrize("R", [16, 32, 40, 64, 72, 96, 112, 128])
@pytest.mark.parametrize("dtype,coded", [(F16, False), (BF16, True), (F16, True)])
def test_every_rank_over_prompts(cuda, M, R, dtype, coded):
    """Contractions of several stages, the last one cut short; workgroups few and many to a compute unit."""
    gen = torch.Generator().manual_seed(M + R)
    K, N, n = 1872, 40, 3
    codes = torch.randint(-127, 128, (N, K), generator=gen).to(torch.int8)
    ws = torch.rand(N, generator=gen) / 1000
    a, b, s = (torch.randn(n, R, K, generator=gen) / K ** 0.5).to(dtype), (torch.randn(n, N, R, generator=gen) / R ** 0.5).to(dtype), 0.25 + torch.rand(n, generator=gen)
    lin, ad = W8A8Linear(codes, ws).to(cuda), LowRankAdapters(a, b, s).to(cuda)
    x = torch.randn(M, K, generator=gen).to(dtype)
    idx = torch.sort(torch.randint(-1, n + 1, (M,), generator=gen)).values.roll(M // 5).to(I32)
    q, qs = quantize_rows(x.to(cuda))
    got = lin.forward_int8(q, qs, dtype, adapters=ad, ids=idx.to(cuda)) if coded else lin(x.to(cuda), adapters=ad, ids=idx.to(cuda))
    want, mag, low = adapters_ref(q.cpu(), qs.cpu(), codes, ws, None, q.cpu().double() * qs.cpu().double()[:, None] if coded else x, a, b, s, idx)
    # as for few rows: sums of K and R terms in 32 bits, h in two pieces
    assert_near(got, want, mag * 4 * 2.0 ** -24 + low * (2.0 ** -24 * (K / 8 + R + 16) + 2.0 ** -14), 1.0, "adapted")


@pytest.mark.parametrize("M", [32, 33, 48, 64])
@pytest.mark.parametrize("R", [16, 64, 128])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_few_rows_of_wide_results(cuda, M, R, dtype):
    """Up to 64 rows on either side of what the kernel of few rows takes."""
    gen = torch.Generator().manual_seed(M + R)
    K, N, n = 272, 9100, 7
    codes = torch.randint(-127, 128, (N, K), generator=gen).to(torch.int8)
    ws = torch.rand(N, generator=gen) / 1000
    a, b, s = (torch.randn(n, R, K, generator=gen) / K ** 0.5).to(dtype), (torch.randn(n, N, R, generator=gen) / R ** 0.5).to(dtype), 0.25 + torch.rand(n, generator=gen)
    lin, ad = W8A8Linear(codes, ws).to(cuda), LowRankAdapters(a, b, s).to(cuda)
    x = torch.randn(M, K, generator=gen).to(dtype)
    for idx in (torch.arange(M) % (n + 2) - 1, torch.full((M,), 3)):
        q, qs = quantize_rows(x.to(cuda))
        want, mag, low = adapters_ref(q.cpu(), qs.cpu(), codes, ws, None, x, a, b, s, idx)
        got = lin(x.to(cuda), adapters=ad, ids=idx.to(I32).to(cuda))
        # as for other sizes: sums of K and R terms in 32 bits, h in two pieces
        assert_near(got, want, mag * 4 * 2.0 ** -24 + low * (2.0 ** -24 * (K / 8 + R + 16) + 2.0 ** -14), 1.0, "adapted")


@pytest.mark.parametrize("n", [3, 64, 65, 700, 5000, 8192])
@pytest.mark.parametrize("kind", ["all to one", "a few", "far apart", "every one twice"])
def test_many_entries_with_one_destination(cuda, n, kind):
    """The last entry of a destination counts, however many there are and however their numbers lie."""
    gen = torch.Generator().manual_seed(n)
    slots = 9000
    t = torch.arange(slots, device=cuda)[:, None].repeat(1, 3)
    dst = {"all to one": torch.full((n,), 5), "a few": torch.randint(0, 7, (n,), generator=gen) * 1024, "far apart": torch.randperm(9, generator=gen)[torch.arange(n) % 9] * 1000 % slots,
           "every one twice": torch.randperm(slots, generator=gen)[:(n + 1) // 2].repeat(2)[:n]}[kind]
    src = torch.randint(0, slots, (n,), generator=gen)
    want = t.cpu().clone()
    for s, d in zip(src.tolist(), dst.tolist()):
        want[d] = s
    copy_slots(t, src.to(I32).to(cuda), dst.to(I32).to(cuda))
    assert torch.equal(t.cpu(), want)


def _prompts(cuda, lens, H, K, V, dtype, g, slots, num_slots, seed):
    """Packed prompts against the plain form; slots: negative ones start from zero and keep nothing, ones beyond the state give NaN."""
    T = sum(lens)
    q, k, v, gd = attention_inputs(T, H, K, V, dtype, g, seed)
    state = torch.randn(num_slots, H, K, V, generator=torch.Generator().manual_seed(seed + 1))
    first = torch.stack([state[s] if 0 <= s < num_slots else torch.zeros(H, K, V) for s in slots])
    o, mag, S, Sm, most = attention_ref(q, k, v, gd, K ** -0.5, lens, first)
    at = 0
    for n, s in zip(lens, slots):
        if s >= num_slots:
            o[at:at + n] = float("nan")
        at += n
    dst = state.to(cuda)
    got = linear_attention_prompt(*(None if t is None else t.to(cuda) for t in (q, k, v, gd)), state=dst, slots=torch.tensor(slots, dtype=I32, device=cuda),
                                  seq_starts=starts_of(lens, cuda))
    assert_near(got, o, mag, out_rel(lens, most, dtype), "o")
    live = [i for i, s in enumerate(slots) if 0 <= s < num_slots]
    want, wm = state.double().clone(), state.double().abs()
    for i in live:
        want[slots[i]], wm[slots[i]] = S[i], Sm[i]
    assert_near(dst, want, wm, state_rel(lens, most), "state")
    rest = [i for i in range(num_slots) if i not in slots]
    assert torch.equal(dst[rest].cpu(), state[rest])


@pytest.mark.parametrize("K", [24, 64, 128, 200])
@pytest.mark.parametrize("V", [40, 200])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("g", ["token", "none"])
def test_prompts_in_segments_of_every_width(cuda, K, V, dtype, g):
    _prompts(cuda, [700, 3, 1, 1000], 2, K, V, dtype, g, [1, 0, 3, 2], 5, 11)


@pytest.mark.parametrize("lens", [[600, 800, 700, 64], [1] * 130 + [900] + [2] * 70, [0] * 65 + [1500]])
def test_segments_of_padding_and_slots_that_do_not_exist(cuda, lens):
    n = len(lens)
    _prompts(cuda, lens, 1, 64, 72, F16, "token", ([-1, 99, 0, 1] if n == 4 else [i if i % 9 else -1 - i for i in range(n)]), n, 12)


# ---------------------------------------------------------------------------------------------- native and general calls
def _both_ways(monkeypatch, name, call, native):
    """The call as it is and without its native form: the same bits; whether the native form served it."""
    served, fn = [], getattr(_lib.native(), name)
    with monkeypatch.context() as m:
        m.setattr(_lib.native(), name, lambda *a: served.append(fn(*a)) or served[-1])
        here = call()
        m.setattr(_lib.native(), name, lambda *a: None)
        there = call()
    assert [r is not None for r in served] in ([[True]] if native else [[False], []])
    for a, b in zip(here, there):
        assert a.dtype == b.dtype and a.shape == b.shape and a.stride() == b.stride() and torch.equal(a, b)


@pytest.mark.parametrize("form", ["plain", "head", "none", "packed", "slots", "g 16 bits", "q reversed", "v unaligned", "scale"])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("L", [90, 1500])
def test_native_attention(cuda, monkeypatch, form, dtype, L):
    H, K, V = 3, 64, 40
    q, k, v, g = (None if t is None else t.to(cuda) for t in attention_inputs(2 * L, H, K, V, dtype, form if form in ("head", "none") else "token", 5))
    if form == "q reversed":
        q = q.flip(-1)[..., ::1].transpose(1, 2).contiguous().transpose(1, 2)               # (channels with a stride)
    if form == "v unaligned":
        v = torch.cat([v.new_zeros(1), v.flatten()])[1:].view(v.shape)
    if form == "g 16 bits":
        g = g.to(dtype)
    kw = dict(scale=0.3) if form == "scale" else {}
    packed = form == "packed"
    native = form not in ("g 16 bits", "q reversed", "v unaligned")
    slots = torch.tensor([3, 1], dtype=I32, device=cuda) if form == "slots" else None

    def prompt():
        state = torch.ones(4, H, K, V, device=cuda)
        args = (q, k, v, g) if packed else tuple(t if t is None or t.dim() == 1 else t.unflatten(0, (2, L)) for t in (q, k, v, g))
        return linear_attention_prompt(*args, state=state, slots=slots, seq_starts=starts_of([L, L], cuda) if packed else None, **kw), state

    def step():
        state = torch.ones(4, H, K, V, device=cuda)
        return linear_attention_step(state, *(t if t is None or t.dim() == 1 else t[5:7] for t in (q, k, v, g)), slots=slots, **kw), state

    _both_ways(monkeypatch, "linear_attention_prompt", prompt, native)
    _both_ways(monkeypatch, "linear_attention_step", step, native)


@pytest.mark.parametrize("form", ["plain", "bare", "no gate", "x strided", "two types", "z slice", "x and z slices", "z reversed", "one row", "z expanded", "z of one row"])
def test_native_norm(cuda, monkeypatch, form):
    gen = torch.Generator().manual_seed(6)
    x, z, w, b = (torch.randn(*s, generator=gen).to(BF16).to(cuda) for s in ((3, 7, 96), (3, 7, 96), (96,), (96,)))
    x = x.transpose(0, 1) if form == "x strided" else x
    z = None if form in ("bare", "no gate") else z.transpose(0, 1) if form == "x strided" else z
    w, b = (None, None) if form == "bare" else (w, b.float() if form == "two types" else b)
    wide = torch.randn(3, 7, 300, generator=gen).to(BF16).to(cuda)
    if form in ("z slice", "x and z slices"):
        z = wide[..., 200:296]
    if form == "x and z slices":
        x = wide[..., 5:101]                                                                # (not on a 16-byte boundary)
    if form == "z reversed":
        z = z.flip(-1).transpose(-1, -2).contiguous().transpose(-1, -2)                     # (channels with a stride)
    if form == "z expanded":
        z = wide[:, :1, 100:196].expand(3, 7, 96)                                           # (rows not equally far apart)
    if form == "z of one row":
        z = wide[:1, :1, 100:196].expand(3, 7, 96)
    if form == "one row":
        x, z = x[1:2, 2:3], wide[:1, ::7, 100:196]
    _both_ways(monkeypatch, "groupnorm_gated", lambda: [groupnorm_gated(x, z, w, b, num_groups=6)], form not in ("x strided", "two types", "z reversed", "z expanded"))


@pytest.mark.parametrize("form", ["plain", "codes", "one scale", "K not padded", "static scale", "x strided", "scale number"])
@pytest.mark.parametrize("M", [5, 300])
def test_native_adapters(cuda, monkeypatch, form, M):
    gen = torch.Generator().manual_seed(7)
    K, N, R = 250 if form == "K not padded" else 256, 96, 24
    codes = torch.randint(-127, 128, (N, K), generator=gen).to(torch.int8)
    lin = W8A8Linear(codes, torch.rand(N, generator=gen) / 1000, torch.tensor(0.02) if form == "static scale" else None, torch.randn(N, generator=gen).half()).to(cuda)
    ad = LowRankAdapters(torch.randn(3, R, K, generator=gen).half() / 16, torch.randn(3, N, R, generator=gen).half() / 4).to(cuda)
    x, ids = torch.randn(M, K, generator=gen).half().to(cuda), torch.randint(-1, 4, (M,), generator=gen).to(I32).to(cuda)
    q, qs = quantize_rows(x)
    if form == "x strided":
        x = torch.cat([x, x], 1)[:, :K]
    call = {"codes": lambda: lin.forward_int8(q, qs, F16, adapters=ad, ids=ids), "one scale": lambda: lin.forward_int8(q, qs[:1].clone(), F32, adapters=ad, ids=ids),
            "scale number": lambda: lin.forward_int8(q, 0.02, F16, adapters=ad, ids=ids)}.get(form, lambda: lin(x, adapters=ad, ids=ids))
    _both_ways(monkeypatch, "adapted", lambda: [torch.nan_to_num(call())], form in ("plain", "codes", "one scale"))


@pytest.mark.parametrize("form", ["plain", "nested", "room between", "one slot", "interleaved", "src strided"])
def test_native_slots(cuda, monkeypatch, form):
    gen = torch.Generator().manual_seed(8)
    n = 1 if form == "one slot" else 6
    src, dst = (torch.tensor(t, dtype=I32, device=cuda) for t in ([0, 3, -1, 7], [1, 0, 2, 5]))
    if form == "src strided":
        src = src.repeat_interleave(2)[::2]

    def call():
        wide = torch.arange(n * 200.0, device=cuda).view(n, 2, 100).clone()
        t = wide[:, 0] if form in ("room between", "interleaved") else wide
        copy_slots([[t], (wide[:, 1],)] if form == "interleaved" else [[t]] if form == "nested" else t, src, dst)
        return [torch.nan_to_num(wide)]

    _both_ways(monkeypatch, "copy_slots", call, form not in ("interleaved", "src strided"))
