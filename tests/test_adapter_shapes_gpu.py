"""Low-rank adapters beside an INT8 projection in every shape of the product's tiles and of the first half, against a plain 64-bit form on the GPU."""

import pytest
import torch

from linquant_amd.w8a8_linear import LowRankAdapters, W8A8Linear, quantize_rows
from tests.serving_cases import HALF_STEP, TINY

pytestmark = pytest.mark.gpu

F16, BF16, F32, I32 = torch.float16, torch.bfloat16, torch.float32, torch.int32


def _ids(kind, M, n, gen):
    """Adapters by row: none (-1) and one beyond the last (n) among them."""
    if kind == "turn":
        return (torch.arange(M) % (n + 2) - 1).to(I32)
    if kind == "runs":
        return torch.sort(torch.randint(-1, n + 1, (M,), generator=gen)).values.roll(M // 3).to(I32)
    return torch.randint(-1, n + 1, (M,), generator=gen).to(I32)


def _ref(x, base, base_mag, a, b, s, ids):
    """x (M, K), base (M, N) and its magnitudes in 64 bits -> with the adapters, and the magnitudes of what they add; NaN where an id is beyond them."""
    y, low, h = base.clone(), torch.zeros_like(base), torch.zeros(x.shape[0], a.shape[1], dtype=torch.float64, device=x.device)
    top = h.clone()
    for j in range(a.shape[0]):
        rows = (ids == j).nonzero()[:, 0]
        if len(rows):
            aj, bj, xj = a[j].double(), b[j].double(), x[rows]
            h[rows], top[rows] = s[j].double() * (xj @ aj.t().contiguous()), s[j].double().abs() * (xj.abs() @ aj.abs().t().contiguous())
            y[rows] += h[rows] @ bj.t().contiguous()
            low[rows] = top[rows] @ bj.abs().t().contiguous()
    beyond = ids >= a.shape[0]
    y[beyond], h[beyond] = float("nan"), float("nan")
    return y, low, h, top


def _near(got, want, slack, what):
    g = got.double()
    assert torch.equal(g.isnan(), want.isnan()), f"{what}: NaN in other places"
    off = (g - want).abs() - (HALF_STEP[got.dtype] * (want.abs() + slack) + TINY[got.dtype] + slack)
    off = torch.nan_to_num(off, nan=-1.0)
    at = off.argmax()
    assert (off <= 0).all(), f"{what}: {got.flatten()[at]} for {want.flatten()[at]}, too far by {off.flatten()[at]}"


def _check(cuda, M, K, N, R, n, kind, dtype, coded, bias, out_dtype=None):
    gen = torch.Generator().manual_seed(M + N + R)
    codes = torch.randint(-127, 128, (N, K), generator=gen).to(torch.int8)
    ws = torch.rand(N, generator=gen) / 1000
    b0 = torch.randn(N, generator=gen) if bias else None
    a, b, s = (torch.randn(n, R, K, generator=gen) / K ** 0.5).to(dtype), (torch.randn(n, N, R, generator=gen) / R ** 0.5).to(dtype), 0.25 + torch.rand(n, generator=gen)
    lin, ad = W8A8Linear(codes, ws, bias=b0).to(cuda), LowRankAdapters(a, b, s).to(cuda)
    x = torch.randn(M, K, generator=gen).to(dtype).to(cuda)
    ids = _ids(kind, M, n, gen).to(cuda)
    q, qs = quantize_rows(x)
    taken = q.double() * qs.double()[:, None] if coded else x.double()
    w = codes.to(cuda).double().t().contiguous()
    scale = qs.double()[:, None] * ws.to(cuda).double()
    base, mag = (q.double() @ w) * scale, (q.double() @ w).abs() * scale
    if bias:
        base, mag = base + b0.to(cuda).double(), mag + b0.to(cuda).double().abs()
    want, low, h, top = _ref(taken, base, mag, a.to(cuda), b.to(cuda), s.to(cuda), ids)
    # the first half: products and sums of K terms in 32 bits, its scales a rounding each
    got_h, order = ad._down(q if coded else x, qs if coded else None, ids)
    _near(got_h[:, :R], h, top * 2.0 ** -24 * (K / 8 + 16), "h")
    assert not torch.nan_to_num(got_h[:, R:]).any()
    assert order is None or torch.equal(torch.sort(order).values, torch.arange(M, dtype=I32, device=cuda))
    got = lin.forward_int8(q, qs, out_dtype or dtype, adapters=ad, ids=ids) if coded else lin(x, adapters=ad, ids=ids)
    # the product exact, its scales and the bias a rounding each; h in two pieces of 16 bits and sums of R terms in 32 bits
    _near(got, want, mag * 4 * 2.0 ** -24 + low * (2.0 ** -24 * (K / 8 + R + 16) + 2.0 ** -14), "adapted")


@pytest.mark.parametrize("M,N", [(1100, 1200), (449, 2560), (2305, 4200), (1537, 3333), (4113, 6200), (5000, 5001)])   # 64 x 128, 128 x 128, 128 x 256
@pytest.mark.parametrize("kind", ["runs", "turn", "random"])
@pytest.mark.parametrize("dtype,coded,bias", [(F16, False, True), (BF16, True, False)])
@pytest.mark.parametrize("R", [16, 40])
def test_every_tile_of_the_product(cuda, M, N, kind, dtype, coded, bias, R):
    """Odd rows and columns behind the last whole tile, and contractions of two stages, the second cut short."""
    _check(cuda, M, 144, N, R, 5, kind, dtype, coded, bias)


@pytest.mark.parametrize("M,N", [(130, 100), (1100, 1200), (2305, 4200), (4113, 6200)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_every_tile_in_32_bits(cuda, M, N, dtype):
    _check(cuda, M, 64, N, 128, 3, "runs", dtype, True, True, F32)


@pytest.mark.parametrize("K", [250, 122, 1001])
@pytest.mark.parametrize("M,R", [(1100, 16), (600, 32), (400, 48), (300, 64), (300, 80), (700, 96), (515, 128)])
@pytest.mark.parametrize("dtype,coded", [(F16, False), (BF16, False), (F16, True), (BF16, True)])
def test_first_half_of_rows_that_are_no_whole_eights(cuda, M, K, R, dtype, coded):
    """Rows that are read one entry at a time, every number of sums of a tile; from rank 80 on in windows of 256 rows."""
    _check(cuda, M, K, 70, R, 4, "random", dtype, coded, False)


@pytest.mark.parametrize("M,K,R", [(1100, 248, 16), (600, 72, 32), (400, 24, 48), (300, 1000, 64), (700, 248, 96), (515, 8, 128)])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("kind", ["runs", "turn"])
def test_first_half_from_codes_of_whole_eights(cuda, M, K, R, dtype, kind):
    """Rows of whole eights of codes that are no whole 16 bytes."""
    _check(cuda, M, K, 70, R, 4, kind, dtype, True, False)
