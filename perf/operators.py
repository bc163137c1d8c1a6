"""The operators with which a quantized Mamba-2 block serves, as cases that can be timed and compared.

  linear    rows quantized to INT8 with a scale each, then the INT8 matrix product with a scale for each row and output channel
  norm      the residual stream between two blocks: optional norm after a block, gate and residual scale, norm before the next
  conv      the short causal convolution that carries its last inputs from call to call: prompts and single tokens
  scan      the selective state space scan that carries its state from call to call: prompts of one length or ragged ones
  step      the same scan for one token of each sequence

Sizes are those of the repository's benchmark layer (d_model 2560, 80 heads of 64, state 128, convolution over 5376 channels)
and its tests' neighbours: 64 heads, 8 groups, state 64.  Activations are drawn as the benchmark draws them: SiLU of normal
values behind the convolution, raw dt around -2 with A in [-16, -1] ("strong") or around -4.5 with A in [-1.3, -1] ("weak").
"""

from __future__ import annotations

import math

import torch
import torch.nn.functional as Fn

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
REGIMES = {"strong": (-2.0, 16.0), "weak": (-4.5, 1.3)}
CHUNK = 64


def _linear(M, K, N, *, dtype="fp16", bias=False, name=None):
    c = dict(op="linear", M=M, K=K, N=N, dtype=dtype, bias=bias)
    return c if name is None else dict(c, name=name)


def _norm(rows, D, *, dtype="fp16", residual="fp32", gate="none", post=False, scale=1.0, name=None):
    c = dict(op="norm", rows=rows, D=D, dtype=dtype, residual=residual, gate=gate, post=post, scale=scale)
    return c if name is None else dict(c, name=name)


def _conv(lens, D, *, W=4, dtype="fp16", packed=True, single=False, name=None):
    c = dict(op="conv", lens=lens, D=D, W=W, dtype=dtype, packed=packed, single=single)
    return c if name is None else dict(c, name=name)


def _scan(lens, H, *, P=64, G=1, N=128, dtype="fp16", packed=True, decay="strong", name=None):
    c = dict(op="scan", lens=lens, H=H, P=P, G=G, N=N, dtype=dtype, packed=packed, decay=decay)
    return c if name is None else dict(c, name=name)


def _step(batch, H, *, P=64, G=1, N=128, dtype="fp16", decay="strong", name=None):
    c = dict(op="step", batch=batch, H=H, P=P, G=G, N=N, dtype=dtype, decay=decay)
    return c if name is None else dict(c, name=name)


def _same(n, length):
    return ",".join([str(length)] * n)


def listed():
    return [
        # the projection into the mixer for 16 sequences that answer, one token each
        _linear(16, 2560, 10576, name="linear_in_decode_b16"),
        # the projection out of it for a few prompts, a token count off every tile
        _linear(3001, 5120, 2560, dtype="bf16", bias=True, name="linear_out_m3001"),
        # the projection into it at the prefill that the benchmark is quoted on
        _linear(32768, 2560, 10576, name="linear_in_b4_l8192"),
        # one token of 16 sequences between two blocks, the stream kept in 32 bits
        _norm(16, 2560, dtype="bf16", name="norm_decode_b16"),
        # prompts: norm after the block, a gate for each channel, residual scale, norm before the next block
        _norm(32768, 2560, residual="fp16", gate="channel", post=True, scale=0.5, name="norm_sandwich_b4_l8192"),
        # 64 sequences that answer
        _conv(_same(64, 1), 5376, dtype="bf16", single=True, name="conv_step_b64"),
        # a ragged batch of prompts, an empty one and a single token among them
        _conv("1200,1,64,2047,0,333,4096,3,777,1500", 5376, name="conv_prompt_ragged"),
        # few and many sequences that answer
        _step(4, 80, name="step_b4"),
        _step(256, 80, dtype="bf16", decay="weak", name="step_b256"),
        # one short prompt: launches and the chain of chunks count
        _scan("384", 80, packed=False, name="scan_b1_l384"),
        # a ragged batch of prompts with 8 groups, some going on from a state
        _scan("1200,1,64,2047,0,333,1024,3,777,1500", 64, G=8, dtype="bf16", decay="weak", name="scan_ragged_g8"),
        # the prefill that the benchmark is quoted on
        _scan(_same(4, 8192), 80, packed=False, name="scan_b4_l8192"),
    ]


def _log(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def _draw_lens(rng, tokens, ragged):
    tokens = int(tokens)
    if not ragged:
        n = rng.choice([b for b in (1, 2, 3, 4, 8) if b <= tokens])
        return _same(n, max(1, tokens // n))
    lens, left = [], tokens
    while left > 0 and len(lens) < 12:
        lens.append(min(left, int(_log(rng, 1, 3000))))
        left -= lens[-1]
    if rng.random() < 0.3:
        lens.insert(rng.randrange(len(lens) + 1), 0)
    return ",".join(map(str, lens))


def draw(rng):
    op = rng.choice(["linear", "norm", "conv", "scan", "step"])
    dtype = rng.choice(["fp16", "bf16"])
    if op == "linear":
        K, N = rng.choice([(2560, 10576), (5120, 2560), (2048, 8512), (4096, 2048), (1040, 777)])
        return _linear(int(_log(rng, 1, 32768)), K, N, dtype=dtype, bias=rng.random() < 0.5)
    if op == "norm":
        return _norm(int(_log(rng, 1, 32768)), rng.choice([768, 1000, 2048, 2560, 5120, 4099]), dtype=dtype,
                     residual=rng.choice(["fp32", dtype]), gate=rng.choice(["none", "channel", "full"]), post=rng.random() < 0.5,
                     scale=rng.choice([1.0, 0.5]))
    if op == "conv":
        D, W = rng.choice([5376, 4352, 7168, 1032]), rng.choice([4, 4, 3, 2])
        if rng.random() < 0.4:
            return _conv(_same(int(_log(rng, 1, 512)), 1), D, W=W, dtype=dtype, single=True)
        ragged = rng.random() < 0.6
        return _conv(_draw_lens(rng, _log(rng, 1, 32768), ragged), D, W=W, dtype=dtype, packed=ragged)
    H, G = rng.choice([(80, 1), (64, 1), (64, 8), (24, 1), (32, 2), (5, 1)])
    P, N = rng.choice([(64, 128), (64, 128), (64, 64), (32, 128), (128, 64)])
    decay = rng.choice(["strong", "weak"])
    if op == "step":
        return _step(int(_log(rng, 1, 256)), H, P=P, G=G, N=N, dtype=dtype, decay=decay)
    ragged = rng.random() < 0.6
    return _scan(_draw_lens(rng, _log(rng, 1, 32768), ragged), H, P=P, G=G, N=N, dtype=dtype, packed=ragged, decay=decay)


# ------------------------------------------------------------------------------------------------------------- inputs
def _lens(c):
    return [int(n) for n in c["lens"].split(",")]


def _starts(lens, device="cuda"):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device=device)


def prepare(case, seed):
    c = case
    dt = DTYPES[c["dtype"]]
    gen = torch.Generator(device="cuda").manual_seed(seed % (1 << 62))
    rn = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    un = lambda *shape: torch.rand(*shape, generator=gen, device="cuda")  # noqa: E731
    if c["op"] == "linear":
        M, K, N = c["M"], c["K"], c["N"]
        w = rn(N, K) / math.sqrt(K)
        ws = w.abs().amax(1) / 127.0
        return dict(c=c, x=(rn(M, K) * (0.5 + un(M, 1))).to(dt), w=torch.round(w / ws[:, None]).to(torch.int8), w_scale=ws,
                    bias=rn(N).to(dt) if c["bias"] else None)
    if c["op"] == "norm":
        rows, D = c["rows"], c["D"]
        gate = {"none": lambda: None, "channel": lambda: (0.5 + un(D)).to(dt), "full": lambda: (0.5 + un(rows, D)).to(dt)}[c["gate"]]()
        return dict(c=c, x=rn(rows, D).to(dt), residual=(2 * rn(rows, D)).to(DTYPES[c["residual"]]), weight=(1 + 0.1 * rn(D)).to(dt),
                    post=(1 + 0.1 * rn(D)).to(dt) if c["post"] else None, gate=gate)
    if c["op"] == "conv":
        lens, D, W = _lens(c), c["D"], c["W"]
        n, T = len(lens), sum(lens)
        wide = rn(T, D + 64).to(dt)                      # the channels are a slice of the projection
        x = wide[:, 32:32 + D]
        slots = torch.randperm(n + 3, generator=gen, device="cuda")[:n].to(torch.int32)
        s = dict(c=c, wide=wide, x=x, weight=(0.5 * rn(D, W)).to(dt), bias=(0.1 * rn(D)).to(dt), slots=slots,
                 state=rn(n + 3, W - 1, D).to(dt), starts=_starts(lens))
        if not c["packed"] and not c["single"]:
            s["x"] = wide.view(n, lens[0], D + 64)[..., 32:32 + D]
        return s
    H, P, G, N = c["H"], c["P"], c["G"], c["N"]
    mean, a_max = REGIMES[c["decay"]]
    n = c["batch"] if c["op"] == "step" else len(_lens(c))
    T = c["batch"] if c["op"] == "step" else sum(_lens(c))
    xBC = Fn.silu(rn(T, H * P + 2 * G * N)).to(dt)       # x, B and C are views of what the convolution gives
    raw = (mean + 0.5 * rn(T, H + 40)).to(dt)            # dt is a slice of the projection
    x, B, C = xBC.split([H * P, G * N, G * N], dim=-1)
    s = dict(c=c, xBC=xBC, x=x.view(T, H, P), B=B.view(T, G, N), C=C.view(T, G, N), dt=raw[:, 40:], A=-(1 + (a_max - 1) * un(H)),
             D=1 + 0.1 * rn(H), dt_bias=0.1 * rn(H), slots=torch.randperm(n + 3, generator=gen, device="cuda")[:n].to(torch.int32),
             state=0.3 * rn(n + 3, H, P, N))
    if c["op"] == "scan":
        lens = _lens(c)
        s.update(starts=_starts(lens), longest=max(lens))
        if not c["packed"]:
            L = lens[0]
            for k in ("x", "B", "C", "dt"):
                s[k] = s[k].unflatten(0, (n, L))
    return s


# ---------------------------------------------------------------------------------------------------------- plain forms
def _plain_linear(s):
    x = s["x"].float()
    xs = x.abs().amax(1, keepdim=True) / 127.0
    q = torch.round(x / torch.where(xs > 0, xs, 1.0))
    y = (q @ s["w"].float().T) * (xs * s["w_scale"])
    return (y if s["bias"] is None else y + s["bias"].float()).to(s["x"].dtype)


def _plain_norm(s):
    x, r = s["x"].float(), s["residual"].float()
    if s["post"] is not None:
        x = x * torch.rsqrt(x.square().mean(1, keepdim=True) + 1e-5) * s["post"].float()
    if s["gate"] is not None:
        x = x * s["gate"].float()
    r = r + s["c"]["scale"] * x
    y = r * torch.rsqrt(r.square().mean(1, keepdim=True) + 1e-5) * s["weight"].float()
    return y.to(s["x"].dtype), r.to(s["residual"].dtype)


def _plain_conv(s):
    c, D, W = s["c"], s["c"]["D"], s["c"]["W"]
    x, n = s["x"].reshape(-1, D), s["slots"].numel()
    T, starts, slots = x.shape[0], s["starts"].long(), s["slots"].long()
    # every sequence's state in front of its tokens, one sequence behind the other
    seq = torch.searchsorted(starts[1:], torch.arange(T, device=x.device), right=True)
    at = torch.arange(T, device=x.device) + (seq + 1) * (W - 1)
    before = (starts[:-1] + torch.arange(n, device=x.device) * (W - 1))[:, None] + torch.arange(W - 1, device=x.device)
    line = torch.empty(T + n * (W - 1), D, dtype=x.dtype, device=x.device)
    line[at] = x
    line[before.reshape(-1)] = s["state"][slots].reshape(-1, D)
    w = s["weight"].float()
    y = s["bias"].float() + sum(w[:, j] * line[at - (W - 1) + j].float() for j in range(W))
    after = (starts[1:] + torch.arange(n, device=x.device) * (W - 1))[:, None] + torch.arange(W - 1, device=x.device)
    s["state"][slots] = line[after.reshape(-1)].view(n, W - 1, D)
    return (y * torch.sigmoid(y)).to(x.dtype).view(s["x"].shape), s["state"]


def _softplus(v):
    return torch.where(v > 20.0, v, torch.log1p(torch.exp(v.clamp(max=20.0))))


def _plain_step(s):
    c, slots = s["c"], s["slots"].long()
    H, G = c["H"], c["G"]
    x, B, C = s["x"].float(), s["B"].float(), s["C"].float()
    d = _softplus(s["dt"].float() + s["dt_bias"])
    B, C = (t.repeat_interleave(H // G, dim=1) for t in (B, C))
    S = s["state"][slots] * torch.exp(d * s["A"])[..., None, None] + (d[..., None] * x)[..., None] * B[:, :, None]
    y = (S * C[:, :, None]).sum(-1) + s["D"][:, None] * x
    s["state"][slots] = S
    return y.to(s["x"].dtype), s["state"]


def _plain_scan(s):
    c, slots, n = s["c"], s["slots"].long(), s["slots"].numel()
    H, P, G, N, Q = c["H"], c["P"], c["G"], c["N"], CHUNK
    flat = lambda t, *tail: t.reshape(-1, *tail)  # noqa: E731
    x, B, C, raw = flat(s["x"], H, P), flat(s["B"], G, N), flat(s["C"], G, N), flat(s["dt"], H)
    T, L = x.shape[0], -(-s["longest"] // Q) * Q
    # every sequence padded to whole chunks by tokens with dt = 0, which change nothing
    pos = torch.arange(L, device=x.device)
    lens = (s["starts"][1:] - s["starts"][:-1]).long()
    real = pos < lens[:, None]
    at = (s["starts"][:-1].long()[:, None] + pos).clamp(max=T - 1)
    x, B, C = (t[at].float() * real[..., None, None] for t in (x, B, C))
    d = _softplus(raw[at].float() + s["dt_bias"]) * real[..., None]
    nc = L // Q
    x, B, C, d = x.view(n, nc, Q, H, P), B.view(n, nc, Q, G, N), C.view(n, nc, Q, G, N), d.view(n, nc, Q, H)
    cum = torch.cumsum((d * s["A"]).double(), 2).permute(0, 3, 1, 2)                        # (n, H, nc, Q), long sums in 64 bits
    u = (d[..., None] * x).permute(0, 3, 1, 2, 4)                                            # (n, H, nc, Q, P)
    B, C = (t.permute(0, 3, 1, 2, 4).repeat_interleave(H // G, dim=1) for t in (B, C))       # (n, H, nc, Q, N)
    later = torch.ones(Q, Q, dtype=torch.bool, device=x.device).tril()
    w = torch.where(later, torch.exp(torch.where(later, cum[..., :, None] - cum[..., None, :], 0.0).float()), 0.0)
    y = ((C @ B.transpose(-1, -2)) * w) @ u
    last = cum[..., -1]
    local = (u * torch.exp((last[..., None] - cum).float())[..., None]).transpose(-1, -2) @ B   # (n, H, nc, P, N)
    # states in front of each chunk: the chunks' own and the first one, decayed
    ends = torch.cat([torch.zeros_like(last[..., :1]), torch.cumsum(last, -1)], -1)         # (n, H, nc + 1)
    later = torch.ones(nc + 1, nc + 1, dtype=torch.bool, device=x.device).tril()
    w = torch.where(later, torch.exp(torch.where(later, ends[..., :, None] - ends[..., None, :], 0.0).float()), 0.0)
    first = s["state"][slots][:, :, None]
    S = (w @ torch.cat([first, local], 2).flatten(3)).unflatten(3, (P, N))                   # (n, H, nc + 1, P, N)
    y = y + (C * torch.exp(cum.float())[..., None]) @ S[:, :, :-1].transpose(-1, -2)
    y = y + s["D"][:, None, None, None] * x.permute(0, 3, 1, 2, 4)
    y = y.permute(0, 2, 3, 1, 4).reshape(n, L, H, P)
    s["state"][slots] = S[:, :, -1]
    return y[real].to(s["x"].dtype).view(s["x"].shape), s["state"]


# ------------------------------------------------------------------------------------------------------------ own calls
def _own_linear(s):
    from linquant_amd.w8a8_linear import int8_matmul, quantize_rows

    q, qs = quantize_rows(s["x"])
    return int8_matmul(q, s["w"], qs, s["w_scale"], bias=s["bias"], out_dtype=s["x"].dtype)


def _own_norm(s):
    from linquant_amd.norm import residual_rmsnorm

    return residual_rmsnorm(s["x"], s["weight"], s["residual"], eps=1e-5, gate=s["gate"], scale=s["c"]["scale"], post_weight=s["post"])


def _own_conv(s):
    from linquant_amd.kernels.mamba2.conv1d_state import conv1d_prompt, conv1d_step

    if s["c"]["single"]:
        return conv1d_step(s["x"], s["state"], s["weight"], s["bias"], activation="silu", slots=s["slots"]), s["state"]
    return conv1d_prompt(s["x"], s["weight"], s["bias"], activation="silu", state=s["state"], slots=s["slots"],
                         seq_starts=s["starts"] if s["c"]["packed"] else None), s["state"]


def _own_step(s):
    from linquant_amd.kernels.mamba2.ssm import ssm_step

    return ssm_step(s["state"], s["x"], s["dt"], s["A"], s["B"], s["C"], D=s["D"], dt_bias=s["dt_bias"], dt_softplus=True,
                    slots=s["slots"]), s["state"]


def _own_scan(s):
    from linquant_amd.kernels.mamba2.ssm import ssm_prompt

    return ssm_prompt(s["x"], s["dt"], s["A"], s["B"], s["C"], D=s["D"], dt_bias=s["dt_bias"], dt_softplus=True, state=s["state"],
                      slots=s["slots"], seq_starts=s["starts"] if s["c"]["packed"] else None), s["state"]


def run(state):
    op = state["c"]["op"]
    if own:
        return {"linear": _own_linear, "norm": _own_norm, "conv": _own_conv, "step": _own_step, "scan": _own_scan}[op](state)
    return {"linear": _plain_linear, "norm": _plain_norm, "conv": _plain_conv, "step": _plain_step, "scan": _plain_scan}[op](state)


def work(case):
    """Bytes: every input once, every output once, the state of the sequences read and written.  Operations: multiplications and
    additions of the definition, the scan's by its recurrence."""
    c = case
    if c["op"] == "linear":
        M, K, N = c["M"], c["K"], c["N"]
        return {"bytes": 2 * M * K + N * K + 4 * N + (2 * N if c["bias"] else 0) + 2 * M * N, "flops": 2 * M * N * K}
    if c["op"] == "norm":
        rows, D = c["rows"], c["D"]
        res = 4 if c["residual"] == "fp32" else 2
        full = rows * D * (2 + 2 + 2 * res + (2 if c["gate"] == "full" else 0))
        return {"bytes": full + 2 * D * (1 + c["post"] + (c["gate"] == "channel")), "flops": rows * D * (6 + 4 * c["post"] + (c["gate"] != "none"))}
    if c["op"] == "conv":
        lens, D, W = _lens(c), c["D"], c["W"]
        n, T = sum(v > 0 for v in lens), sum(lens)
        return {"bytes": 2 * D * (2 * T + 2 * n * (W - 1) + W + 1), "flops": T * D * (2 * W + 4)}
    H, P, G, N = c["H"], c["P"], c["G"], c["N"]
    n, T = (c["batch"], c["batch"]) if c["op"] == "step" else (sum(v > 0 for v in _lens(c)), sum(_lens(c)))
    return {"bytes": T * 2 * (2 * H * P + 2 * G * N + H) + 8 * n * H * P * N + 12 * H, "flops": T * H * (5 * P * N + 4 * P)}


# ----------------------------------------------------------------------------------------------- definition in 64 bits
def exact(case, seed):
    s, c = prepare(case, seed), case
    f = lambda t: t.double()  # noqa: E731
    if c["op"] == "linear":
        # codes are whole numbers of the 32-bit quotient by definition: the 64-bit part is the product
        x = s["x"].float()
        top = x.abs().max(dim=1).values / 127.0
        codes = torch.where(top[:, None] > 0, (x / top[:, None]).round(), torch.zeros_like(x))
        y = torch.mm(f(codes), f(s["w"]).t()) * f(top)[:, None] * f(s["w_scale"])[None]
        return y if s["bias"] is None else y + f(s["bias"])
    if c["op"] == "norm":
        u, r = f(s["x"]), f(s["residual"])
        if c["post"]:
            u = u / (u.pow(2).sum(-1, keepdim=True) / c["D"] + 1e-5).sqrt() * f(s["post"])
        r = r + c["scale"] * u * (1.0 if s["gate"] is None else f(s["gate"]))
        return r / (r.pow(2).sum(-1, keepdim=True) / c["D"] + 1e-5).sqrt() * f(s["weight"]), r
    slots = s["slots"].tolist()
    if c["op"] == "conv":
        W, at, parts, state = c["W"], 0, [], f(s["state"])
        x = f(s["x"]).reshape(-1, c["D"])
        for slot, n in zip(slots, _lens(c)):
            line = torch.cat([state[slot], x[at:at + n]])
            y = f(s["bias"]).expand(n, -1).clone()
            for j in range(W):
                y += f(s["weight"])[:, j] * line[j:j + n]
            parts.append(y / (1 + (-y).exp()))
            state[slot] = line[n:]
            at += n
        return torch.cat(parts).view(s["x"].shape), state
    H, P, G, N = c["H"], c["P"], c["G"], c["N"]
    lens = [1] * c["batch"] if c["op"] == "step" else _lens(c)
    if max(lens) > 40000:
        return None
    x, B, C = f(s["x"]).reshape(-1, H, P), f(s["B"]).reshape(-1, G, N), f(s["C"]).reshape(-1, G, N)
    d = Fn.softplus(f(s["dt"]).reshape(-1, H) + f(s["dt_bias"]), threshold=200.0)
    y, state = torch.empty_like(x), f(s["state"])
    # token by token, over the sequences that still have one
    order = sorted(range(len(lens)), key=lambda i: -lens[i])
    begin = [sum(lens[:i]) for i in range(len(lens))]
    idx = torch.tensor([slots[i] for i in order], device="cuda")
    row = torch.tensor([begin[i] for i in order], device="cuda")
    S, A, D = state[idx], f(s["A"]), f(s["D"])
    group = torch.arange(H, device="cuda") // (H // G)
    live = len(order)
    for t in range(max(lens)):
        while live and lens[order[live - 1]] <= t:
            live -= 1
        r = row[:live] + t
        S[:live] *= torch.exp(d[r] * A)[:, :, None, None]
        S[:live] += torch.einsum("bhp,bhn->bhpn", d[r][..., None] * x[r], B[r][:, group])
        y[r] = torch.einsum("bhpn,bhn->bhp", S[:live], C[r][:, group]) + D[:, None] * x[r]
    state[idx] = S
    return y.view(s["x"].shape), state
