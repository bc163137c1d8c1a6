"""Low-rank adapters beside an INT8 projection, moves between slots and the gated group norm against plain forms."""

import pytest
import torch

from linquant_amd.norm import groupnorm_gated
from linquant_amd.slots import copy_slots
from linquant_amd.w8a8_linear import LowRankAdapters, W8A8Linear, quantize_rows
from tests.attention_cases import adapters_ref, norm_ref
from tests.serving_cases import HALF_STEP, TINY, assert_near

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
NAN, INF = float("nan"), float("inf")


# ------------------------------------------------------------------------------------------------------------- group norm
@pytest.mark.parametrize("rows,groups,size", [(1, 1, 1), (3, 4, 8), (5, 7, 99), (16, 32, 128), (300, 5, 40), (9, 3, 64), (4, 2, 200), (3, 1, 513), (2, 3, 1000),
                                              (3, 2, 2048), (2, 1, 2560), (2, 2, 4096), (1, 1, 8192), (2, 1, 16384), (2, 1, 16383), (3, 2, 260), (1025, 2, 136)])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("gate,affine,act", [(True, True, "silu"), (False, True, "silu"), (True, False, "sigmoid"), (False, False, None), (True, True, None), (False, False, "sigmoid")])
def test_groupnorm_gated(cuda, rows, groups, size, dtype, gate, affine, act):
    gen = torch.Generator().manual_seed(rows + size)
    D = groups * size
    x, z = (1.5 * torch.randn(rows, D, generator=gen) + 0.4).to(dtype), (2 * torch.randn(rows, D, generator=gen)).to(dtype)
    w, b = 1 + 0.2 * torch.randn(D, generator=gen), 0.3 * torch.randn(D, generator=gen)
    z, w, b = z if gate else None, w.to(dtype) if affine else None, b if affine else None     # (weight and bias of two types)
    want, off = norm_ref(x, z, w, b, groups, 1e-5, act)
    got = groupnorm_gated(x.to(cuda), None if z is None else z.to(cuda), None if w is None else w.to(cuda), None if b is None else b.to(cuda), num_groups=groups, activation=act)
    _near(got, want, off)


def _near(got, want, off):
    assert_near(got, want, off, 2.0 ** -24, "norm")


def test_groupnorm_strides_and_lead_dimensions(cuda):
    gen = torch.Generator().manual_seed(3)
    wide = torch.randn(2, 6, 3, 200, generator=gen).half().to(cuda)
    for cut in (slice(8, 136), slice(3, 131), slice(0, 198)):
        x, z = wide[:, ::2, 0, cut], wide[:, 1::2, 2, cut]
        want, off = norm_ref(x.cpu(), z.cpu(), None, None, 2, 1e-3, "silu")
        _near(groupnorm_gated(x, z, num_groups=2, eps=1e-3), want, off)
    assert groupnorm_gated(wide[:, :0], num_groups=2).shape == (2, 0, 3, 200)
    one = groupnorm_gated(wide[0, 0, 0], num_groups=2)
    assert one.shape == (200,)


def test_groupnorm_unusual_values(cuda):
    """A group of one value, large values, and values that are no numbers, which stay in their group."""
    x = torch.randn(4, 3, 64, generator=torch.Generator().manual_seed(4)).half()
    x[0, 0] = 7.0
    x[1] = 60000.0
    x[1, :, 1] = -60000.0
    x[2, 1, 5], x[3, 2, 0] = NAN, INF
    want, off = norm_ref(x.flatten(1), None, None, None, 3, 1e-5, None)
    got = groupnorm_gated(x.flatten(1).to(cuda), num_groups=3, activation=None)
    assert torch.isnan(got[2, 64:128]).all() and torch.isnan(got[3, 128:]).all()
    keep = torch.isfinite(want)
    assert_near(got.cpu()[keep], want[keep], off[keep], 2.0 ** -24, "norm")
    z = torch.tensor([-INF, INF, NAN, -100.0, -88.0, 65504.0, 0.0, 1.0]).half().repeat(2, 1)
    y = groupnorm_gated(torch.arange(16.0).view(2, 8).half().to(cuda), z.to(cuda), num_groups=1, activation="sigmoid").float().cpu()
    n = groupnorm_gated(torch.arange(16.0).view(2, 8).half().to(cuda), num_groups=1, activation=None).float().cpu()
    assert (y[:, 0] == 0).all() and torch.isnan(y[:, 2]).all() and (y[:, 3:5].abs() < 1e-30).all() and (y[:, 1] - n[:, 1]).abs().max() < 2e-3


# --------------------------------------------------------------------------------------------------------------- adapters
def _linear(K, N, gen, bias=True, input_scale=None):
    w = torch.randn(N, K, generator=gen) / K ** 0.5
    ws = w.abs().amax(1) / 127.0
    codes = torch.round(w / ws[:, None]).to(torch.int8)
    b = torch.randn(N, generator=gen) if bias else None
    return codes, ws, b, W8A8Linear(codes, ws, input_scale, b)


def _adapters(n, R, K, N, dtype, gen):
    return (torch.randn(n, R, K, generator=gen) / K ** 0.5).to(dtype), (torch.randn(n, N, R, generator=gen) / R ** 0.5).to(dtype), 0.25 + torch.rand(n, generator=gen)


def _rel(K, R):
    """fp32 sums over K and R terms as trees or chains of fused steps of at most K / 8 and R; h in two pieces 2^-17 of its row's largest,
    which is at most the sum of magnitudes of any of them times sqrt-free bound: taken as 2^-14 of the terms; the product's part: 4 roundings."""
    return 2.0 ** -24 * (K / 8 + R + 16) + 2.0 ** -14


@pytest.mark.parametrize("M,K,N,R,n", [(1, 256, 96, 8, 1), (3, 1040, 777, 12, 4), (16, 2560, 640, 16, 16), (33, 128, 256, 32, 3), (64, 640, 129, 64, 5), (65, 640, 500, 16, 9),
                                       (127, 144, 31, 128, 2), (257, 272, 257, 24, 7), (300, 1024, 260, 48, 4), (513, 512, 300, 96, 40), (700, 256, 640, 1, 3), (600, 250, 33, 16, 5)])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("order", ["runs", "mixed"])
@pytest.mark.parametrize("coded", [False, True])
def test_adapters(cuda, M, K, N, R, n, dtype, order, coded):
    gen = torch.Generator().manual_seed(M + K + R)
    codes_w, ws, bias, lin = _linear(K, N, gen)
    a, b, s = _adapters(n, R, K, N, dtype, gen)
    x = torch.randn(M, K, generator=gen).to(dtype)
    ids = torch.randint(-1, n, (M,), generator=gen).to(torch.int32)
    if order == "runs":
        ids = ids.sort().values
    if M > 2:
        ids[M // 2], ids[-1] = n, 2 ** 31 - 1                                               # beyond the adapters
    lin, ad = lin.to(cuda), LowRankAdapters(a, b, s).to(cuda)
    q, qs = quantize_rows(x.to(cuda))
    if coded:
        got = lin.forward_int8(q, qs, dtype, adapters=ad, ids=ids.to(cuda))
        xa = q.cpu().double() * qs.cpu().double()[:, None]
    else:
        got = lin(x.to(cuda), adapters=ad, ids=ids.to(cuda))
        xa = x
    want, mag, low = adapters_ref(q.cpu(), qs.cpu(), codes_w, ws, bias, xa, a, b, s, ids)
    assert_near(got, want, mag * 4 * 2.0 ** -24 + low * _rel(K, R), 1.0, "adapted")


def test_adapters_static_scale_lead_dimensions_and_out_types(cuda):
    gen = torch.Generator().manual_seed(8)
    codes_w, ws, bias, lin = _linear(256, 96, gen, input_scale=0.03)
    a, b, s = _adapters(3, 16, 256, 96, F16, gen)
    lin, ad = lin.to(cuda), LowRankAdapters(a, b, s).to(cuda)
    x = torch.randn(2, 5, 256, generator=gen).half()
    ids = torch.randint(-1, 3, (2, 5), generator=gen).to(torch.int32)
    got = lin(x.to(cuda), adapters=ad, ids=ids.to(cuda))
    codes = torch.clamp(torch.round(x.float() / 0.03), -128, 127).to(torch.int8).view(10, 256)
    scale = torch.full((10,), 0.03)
    want, mag, low = adapters_ref(codes, scale, codes_w, ws, bias, x.view(10, 256), a, b, s, ids.view(-1))
    assert got.shape == (2, 5, 96)
    assert_near(got.view(10, 96), want, mag * 4 * 2.0 ** -24 + low * _rel(256, 16), 1.0, "adapted")
    got = lin.forward_int8(codes.view(2, 5, 256).to(cuda), 0.03, F32, adapters=ad, ids=ids.to(cuda))
    want, mag, low = adapters_ref(codes, scale, codes_w, ws, bias, codes.double() * float(torch.tensor(0.03)), a, b, s, ids.view(-1))
    assert got.dtype == F32
    assert_near(got.view(10, 96), want, mag * 4 * 2.0 ** -24 + low * _rel(256, 16), 1.0, "adapted")
    assert lin(x[:, :0].to(cuda), adapters=ad, ids=ids[:, :0].to(cuda)).shape == (2, 0, 96)
    strided = torch.randn(10, 300, generator=gen).half().to(cuda)[:, 20:276]
    ids = ids.view(-1).to(cuda)
    assert torch.equal(lin(strided, adapters=ad, ids=ids), lin(strided.contiguous(), adapters=ad, ids=ids))


@pytest.mark.parametrize("M", [20, 400])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_adapters_keep_to_their_rows(cuda, M, dtype):
    """Values that are no numbers in one request's row or adapter do not reach another's; sizes far apart neither overflow nor vanish."""
    gen = torch.Generator().manual_seed(9)
    K, N, R, n = 256, 160, 16, 4
    codes_w, ws, bias, lin = _linear(K, N, gen)
    a, b, s = _adapters(n, R, K, N, dtype, gen)
    ids = (torch.arange(M) % n).to(torch.int32)
    x = torch.randn(M, K, generator=gen).to(dtype)
    lin = lin.to(cuda)
    q, qs = quantize_rows(x.to(cuda))
    want = lin.forward_int8(q, qs, dtype, adapters=LowRankAdapters(a, b, s).to(cuda), ids=ids.to(cuda)).cpu()
    a2, b2 = a.clone(), b.clone()
    a2[1, 3, 7], b2[2, 5, 1] = INF, NAN
    got = lin.forward_int8(q, qs, dtype, adapters=LowRankAdapters(a2, b2, s).to(cuda), ids=ids.to(cuda)).cpu()
    assert torch.equal(got[ids == 0], want[ids == 0]) and torch.equal(got[ids == 3], want[ids == 3])
    assert not torch.isfinite(got[ids == 1]).any() and torch.isnan(got[ids == 2][:, 5]).all()
    others = [c for c in range(N) if c != 5]
    assert torch.equal(got[ids == 2][:, others], want[ids == 2][:, others])
    x2 = x.clone()
    x2[5, 9] = NAN
    y = lin(x2.to(cuda), adapters=LowRankAdapters(a, b, s).to(cuda), ids=ids.to(cuda)).cpu()
    z = lin(x.to(cuda), adapters=LowRankAdapters(a, b, s).to(cuda), ids=ids.to(cuda)).cpu()
    rest = [m for m in range(M) if m != 5]
    assert torch.isnan(y[5]).all() and torch.equal(y[rest], z[rest])
    big = torch.tensor([2.0 ** 12, 2.0 ** -12, 1.0, 2.0 ** 13])
    if dtype == F16:
        a3, b3 = (a.float() * 2.0 ** 9).half(), (b.float() * 2.0 ** -9).half()
        ref, mag, low = adapters_ref(q.cpu(), qs.cpu(), codes_w, ws, bias, q.cpu().double() * qs.cpu().double()[:, None], a3, b3, s * big, ids)
        got = lin.forward_int8(q, qs, F32, adapters=LowRankAdapters(a3, b3, s * big).to(cuda), ids=ids.to(cuda))
        assert_near(got, ref, mag * 4 * 2.0 ** -24 + low * _rel(K, R), 1.0, "adapted")


def test_adapters_capture(cuda):
    gen = torch.Generator().manual_seed(10)
    _, _, _, lin = _linear(256, 96, gen)
    ad = LowRankAdapters(*_adapters(3, 16, 256, 96, F16, gen)).to(cuda)
    lin = lin.to(cuda)
    x, ids = torch.randn(20, 256, generator=gen).half().to(cuda), torch.zeros(20, dtype=torch.int32, device=cuda)
    lin(x, adapters=ad, ids=ids)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = lin(x, adapters=ad, ids=ids)
    for i in range(4):
        ids.copy_((torch.arange(20, device=cuda) + i) % 4 - 1)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, lin(x, adapters=ad, ids=ids))


# ------------------------------------------------------------------------------------------------------------------ slots
def _move_ref(t, src, dst):
    old, new = t.clone(), t.clone()
    for s, d in zip(src, dst):
        if 0 <= d < t.shape[0]:
            if s >= t.shape[0]:
                new[d] = torch.full_like(old[0].view(torch.uint8), 255).view(t.dtype)
            else:
                new[d] = old[s] if s >= 0 else 0
    return new


def _check_moves(cuda, states, src, dst):
    want = [_move_ref(t.cpu(), src, dst) for t in states]
    copy_slots(states, torch.tensor(src, dtype=torch.int32, device=cuda), torch.tensor(dst, dtype=torch.int32, device=cuda))
    for t, w in zip(states, want):
        assert torch.equal(t.cpu().contiguous().view(torch.uint8), w.contiguous().view(torch.uint8))


SHAPES = [((3, 40), F16), ((5, 8, 16), F32), ((7,), BF16), ((3,), torch.int8), ((1000,), F32), ((1,), torch.int64)]


@pytest.mark.parametrize("n,slots", [(1, 1), (1, 3), (4, 9), (8, 8), (63, 70), (64, 64), (65, 200), (129, 150), (257, 300), (700, 700), (2100, 2500), (8192, 8200)])
@pytest.mark.parametrize("kind", ["permutation", "fork", "mixed"])
def test_copy_slots(cuda, n, slots, kind):
    gen = torch.Generator().manual_seed(n)
    states = [torch.randint(-100, 100, (slots, *shape), generator=gen).to(dt).to(cuda) for shape, dt in SHAPES]
    dst = torch.randperm(slots, generator=gen)[:n]
    src = {"permutation": dst[torch.randperm(n, generator=gen)], "fork": torch.randint(0, min(slots, 3), (n,), generator=gen),
           "mixed": torch.randint(-2, slots + 2, (n,), generator=gen)}[kind]
    if kind == "mixed":
        dst = torch.where(torch.rand(n, generator=gen) < 0.2, torch.randint(-3, slots + 3, (n,), generator=gen), dst)   # (some twice, some nowhere)
    _check_moves(cuda, states, src.tolist(), dst.tolist())


def test_copy_slots_nested_strided_many_and_large(cuda):
    big = torch.randn(6, 2, 500, device=cuda)
    keep = big[:, 1].clone()
    nested = [(big[:, 0], torch.randn(6, 33, device=cuda).half()), [torch.randn(6, 4, device=cuda)]]
    flat = [nested[0][0], nested[0][1], nested[1][0]]
    want = [_move_ref(t.cpu(), [0, 5, 1], [5, 0, 2]) for t in flat]
    copy_slots(nested, torch.tensor([0, 5, 1], dtype=torch.int32, device=cuda), torch.tensor([5, 0, 2], dtype=torch.int32, device=cuda))
    assert all(torch.equal(t.cpu(), w) for t, w in zip(flat, want)) and torch.equal(big[:, 1], keep)
    _check_moves(cuda, [torch.randn(4, 5 + i, device=cuda) for i in range(150)], [1, 0], [0, 3])     # more tensors than a launch takes
    _check_moves(cuda, [torch.randn(5, 80, 64, 128, device=cuda)], [4, 2, -1], [2, 4, 0])
    one = torch.randn(1, 8, device=cuda)
    copy_slots(one, torch.full((1,), -1, dtype=torch.int32, device=cuda), torch.zeros(1, dtype=torch.int32, device=cuda))
    assert (one == 0).all()
    copy_slots([], torch.zeros(1, dtype=torch.int32, device=cuda), torch.zeros(1, dtype=torch.int32, device=cuda))
    copy_slots(one, torch.zeros(0, dtype=torch.int32, device=cuda), torch.zeros(0, dtype=torch.int32, device=cuda))


def test_copy_slots_past_32_bits(cuda):
    n = 2 ** 33 // (4 * 65536) + 2
    t = torch.empty(n, 65536, device=cuda)
    t[0], t[n - 1] = 1.0, 2.0
    copy_slots(t, torch.tensor([0, n - 1], dtype=torch.int32, device=cuda), torch.tensor([n - 1, 0], dtype=torch.int32, device=cuda))
    assert (t[0] == 2).all() and (t[n - 1] == 1).all()


def test_copy_slots_capture(cuda):
    t = torch.arange(6.0, device=cuda)[:, None].repeat(1, 100)
    src, dst = torch.tensor([0, 1, 2], dtype=torch.int32, device=cuda), torch.tensor([1, 2, 0], dtype=torch.int32, device=cuda)
    graph = torch.cuda.CUDAGraph()
    copy_slots(t, src, src)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        copy_slots(t, src, dst)
    for i in range(1, 5):
        graph.replay()
        torch.cuda.synchronize()
        assert t[:, 0].tolist() == [(0 - i) % 3, (1 - i) % 3, (2 - i) % 3, 3, 4, 5]
