"""Plain 64-bit forms of the operators of a linear attention block that answers, and the bounds that follow from how the kernels round."""

from __future__ import annotations

import torch

from tests.serving_cases import HALF_STEP


def attention_ref(q, k, v, g, scale, lens, state):
    """q, k (T, H, K), v (T, H, V), g None, (H,) or (T, H), state (n, H, K, V), 64 bits on the CPU, token by token.
    -> o, its magnitudes, state, its magnitudes, the most that |g| sums to over 64 tokens of a sequence."""
    q, k, v, S = (t.double().cpu() for t in (q, k, v, state))
    T, H = q.shape[:2]
    g = torch.zeros(T, H).double() if g is None else g.double().cpu().clamp(max=0.0).expand(T, H)
    o, mag, out, outm, at, most = torch.empty_like(v), torch.empty_like(v), [], [], 0, 0.0
    for n, s in zip(lens, S):
        s, m = s.clone(), s.abs()
        for t in range(at, at + n):
            a, u = torch.exp(g[t])[:, None, None], k[t][..., None] * v[t][:, None]
            s, m = a * s + u, a * m + u.abs()
            o[t] = scale * (s * q[t][..., None]).sum(1)
            mag[t] = abs(scale) * (m * q[t].abs()[..., None]).sum(1)
        if n:
            run = torch.nn.functional.pad(g[at:at + n].abs(), (0, 0, 0, -n % 64)).view(-1, 64, H).sum(1)
            most = max(most, float(torch.nan_to_num(run, nan=0.0, posinf=0.0).max()))
        out.append(s)
        outm.append(m)
        at += n
    return o, mag, torch.stack(out), torch.stack(outm), most


def state_rel(lens, most):
    """What the state loses of its terms.  A weight is the product of, or an exponential of the sum of, up to max(lens) decays: each off by a
    few units of 2^-24 (exp by 2, the product by 1), an exponential of a sum of up to `most` by 2^-23 of that; an operand in two pieces of
    16 bits is off by 2^-17 of itself, and sums over up to 256 entries in 32 bits by 2^-16 of their terms."""
    return 2.0 ** -22 * (max(lens) + 8) + 2.0 ** -22 * most + 2.0 ** -15


def out_rel(lens, most, dtype):
    """The same for the outputs of a prompt: the weighted q . k and the state that q multiplies enter their products rounded to the activations'
    type once, half a step of each term."""
    return state_rel(lens, most) + HALF_STEP[dtype]


def attention_inputs(T, H, K, V, dtype, g="token", seed=0, g_mean=2.0):
    gen = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    q, k, v = rn(T, H, K).to(dtype), rn(T, H, K).to(dtype), rn(T, H, V).to(dtype)
    decay = {"token": lambda: torch.nn.functional.logsigmoid(g_mean + rn(T, H)), "head": lambda: torch.log1p(-torch.exp2(-5.0 - torch.arange(H) % 8)),
             "fast": lambda: -3.0 * torch.rand(H, generator=gen) - 0.5, "none": lambda: None}[g]()
    return q, k, v, decay


def norm_ref(x, z, weight, bias, groups, eps, act):
    """-> y, and a bound of what its fp32 arithmetic may be off by, apart from the rounding of the output, in units of 2^-24.

    mean: n terms summed, off by at most 2^-24 n mean|x| (taken whole; the sums are trees) -> a shift of the differences; the differences themselves
    by one rounding; var and rsqrt relative: n + 8 units; weight, bias, the activation (hardware exp2 and reciprocal: 8 units of its value or
    of 1) and the product with the gate a rounding or two each."""
    D = x.shape[-1]
    n = D // groups
    xd = x.double().unflatten(-1, (groups, n))
    mean = xd.mean(-1, keepdim=True)
    d = xd - mean
    rs = torch.rsqrt(d.square().mean(-1, keepdim=True) + eps)
    m = xd.abs().mean(-1, keepdim=True)
    logs = n.bit_length() + 8
    off = ((logs * m + xd.abs() + mean.abs()) * rs + (logs + 8) * d.abs() * rs).flatten(-2)
    y = (d * rs).flatten(-2)
    if weight is not None:
        y, off = y * weight.double(), off * weight.double().abs()
        off = off + 2 * y.abs()
    if bias is not None:
        y = y + bias.double()
        off = off + 2 * y.abs()
    f = {"silu": lambda u: u * torch.sigmoid(u), "sigmoid": torch.sigmoid, None: lambda u: u}[act]
    # both activations change by at most 1.1 times their argument's change; exp2's argument is off by 2 units of itself
    if z is None:
        return f(y), 1.1 * off + (0 if act is None else 1) * (16 * f(y).abs() + 4 * y.abs() * torch.sigmoid(y) * (1 + y.abs())) if act else off
    a = f(z.double())
    err_a = 0 if act is None else 16 * a.abs() + 4 * z.double().abs() * a.abs()
    return y * a, off * a.abs() + y.abs() * err_a + 2 * (y * a).abs()


def adapters_ref(codes, code_scale, w, w_scale, bias, x, a, b, scaling, ids):
    """-> y, magnitudes of the product and of what the adapters add.  ``x`` the adapters' activations (M, K)."""
    base = (codes.double() @ w.double().T) * code_scale.double().reshape(-1, 1) * w_scale.double()
    y, mag, low = base.clone(), base.abs(), torch.zeros_like(base)
    for m in range(y.shape[0]):
        j = int(ids[m])
        if j >= a.shape[0]:
            y[m] = float("nan")
        elif j >= 0:
            h = a[j].double() @ x[m].double() * scaling[j].double()
            top = (a[j].double().abs() @ x[m].double().abs()) * scaling[j].double().abs()
            y[m] += b[j].double() @ h
            low[m] = b[j].double().abs() @ top
    if bias is not None:
        y, mag = y + bias.double(), mag + bias.double().abs()
    return y, mag, low
