"""Plain 64-bit forms of the serving operators and the bounds that follow from how the kernels round, for the tests.

``Bound`` of a sum: a kernel's result may be off by the rounding of the output, half a step of its type relative to the value, and
by what its fp32 arithmetic loses, which is proportional to the sum of the terms' magnitudes (``mag``), not to the result."""

from __future__ import annotations

import torch

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}   # half the spacing of subnormals


def assert_near(got, want, mag, rel, what):
    """|got - want| <= half a step of got's type + rel * mag, entry by entry; NaN where want is NaN."""
    w, g = want.double().cpu(), got.double().cpu()
    m = mag.double().cpu() if isinstance(mag, torch.Tensor) else torch.full_like(w, float(mag))
    assert g.shape == w.shape, (what, g.shape, w.shape)
    assert torch.equal(torch.isnan(g), torch.isnan(w)), f"{what}: NaN in other places"
    if not w.numel():
        return
    slack = rel * m
    limit = HALF_STEP[got.dtype] * (w.abs() + slack) + TINY[got.dtype] + slack
    off = torch.nan_to_num((g - w).abs() - limit, nan=-1.0)
    worst = off.argmax()
    assert (off <= 0).all(), f"{what}: {g.flatten()[worst]} for {w.flatten()[worst]}, may be off by {limit.flatten()[worst]}"


def lengths(starts):
    return [int(b - a) for a, b in zip(starts[:-1], starts[1:])]


def conv_ref(x, weight, bias, silu, lens, before):
    """x (T, D) of sequences of the given lengths, before (n, W-1, D).  -> y, magnitudes, the new inputs in front."""
    W = weight.shape[1]
    x, w = x.double(), weight.double()
    ys, mags, after, at = [], [], [], 0
    for n, front in zip(lens, before.double()):
        line = torch.cat([front, x[at:at + n]])
        terms = [w[:, j] * line[j:j + n] for j in range(W)]
        b = torch.zeros_like(w[:, 0]) if bias is None else bias.double()
        y, m = b + sum(terms), b.abs() + sum(t.abs() for t in terms)
        ys.append(y * torch.sigmoid(y) if silu else y)
        mags.append(m)
        after.append(line[n:])
        at += n
    return torch.cat(ys), torch.cat(mags), torch.stack(after)


def ssm_ref(x, dt, A, B, C, D, dt_bias, softplus, limit, lens, state):
    """x (T, H, P), dt (T, H), B, C (T, G, N), state (n, H, P, N), 64 bits on the CPU, token by token.
    -> y, its magnitudes, state, its magnitudes, the most that |d A| sums to over 64 tokens of a sequence."""
    x, dt, A, B, C, S = (t.double() for t in (x, dt, A, B, C, state))
    H, G = x.shape[1], B.shape[1]
    B, C = (t.repeat_interleave(H // G, dim=1) for t in (B, C))
    d = dt + (0.0 if dt_bias is None else dt_bias.double())
    if softplus:
        d = torch.nn.functional.softplus(d, threshold=500.0)
    d = d.clamp(*limit)
    Dv = torch.zeros(H, 1).double() if D is None else (D.double()[:, None] if D.dim() == 1 else D.double())
    y, mag, out, outm, at, most = torch.empty_like(x), torch.empty_like(x), [], [], 0, 0.0
    for n, s in zip(lens, S):
        s, m = s.clone(), s.abs()
        run = torch.zeros(1)
        for t in range(at, at + n):
            a = torch.exp(d[t] * A)[:, None, None]
            u = (d[t][:, None] * x[t])[..., None] * B[t][:, None]
            s, m = a * s + u, a * m + u.abs()
            y[t] = (s * C[t][:, None]).sum(-1) + Dv * x[t]
            mag[t] = (m * C[t][:, None].abs()).sum(-1) + (Dv * x[t]).abs()
        if n:
            run = (d[at:at + n] * A).abs()
            run = torch.nn.functional.pad(run, (0, 0, 0, -n % 64)).view(-1, 64, H).sum(1)
        most = max(most, float(run.max()))
        out.append(s)
        outm.append(m)
        at += n
    return y, mag, torch.stack(out), torch.stack(outm), most


def ssm_rel(lens, most):
    """What fp32 loses of a scan's terms.  Weights are products or exponentials of sums of d A: each of up to max(lens) factors is off by
    a few units of 2^-24 (d by 4, exp by 2, the product by 1: 2^-21 together), an exponential of a sum of up to `most` by 2^-23 of that;
    a product of two operands that are split into 16 bits loses at most 2^-16 of each, three such products to a term."""
    return 2.0 ** -21 * (max(lens) + 8) + 2.0 ** -22 * most + 2.0 ** -14


def ssm_y_rel(lens, most, dtype):
    """The same for the outputs of a prompt.  What the activations multiply there, an entry of the state and a weight of C B^T, is rounded
    to their type once more: (1 + e) of each term, |e| half a step, so the sum is off by at most half a step of the sum of magnitudes.
    (In fp16 that holds for entries above 2^-14 of a unit that the largest of 32 channels fills up to 2^13: down to 2^-27 of it.)"""
    return ssm_rel(lens, most) + HALF_STEP[dtype]


def starts_of(lens, device="cpu", first=0):
    at = [first]
    for n in lens:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device=device)


def ssm_inputs(T, H, P, G, N, dtype, seed=0, a_max=16.0, dt_mean=-2.0):
    """What a call takes, on the CPU."""
    gen = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    return dict(x=rn(T, H, P).to(dtype), dt=(dt_mean + 0.5 * rn(T, H)).to(dtype), A=-(1 + (a_max - 1) * torch.rand(H, generator=gen)),
                B=rn(T, G, N).to(dtype), C=rn(T, G, N).to(dtype), D=1 + 0.1 * rn(H), dt_bias=0.1 * rn(H))
