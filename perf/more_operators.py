"""The operators with which a linear attention block answers for many requests, as cases that can be timed and compared.

  prompt    linear attention with a decay for each head (or head and token) over prompts, from and into fp32 states in slots
  step      the same for one token of each sequence
  norm      group norm of each token's heads, channels last, with scale, shift and a gate behind an activation
  adapters  an INT8 projection and, beside it, the low-rank adapter that each row's request names
  slots     states copied, exchanged, compacted and freed between slots, every tensor of several layers in one call

Sizes are those of the repository's configurations: 16 or 32 heads of 128 by 128 with prompts of 4096 or 8192 tokens, projections of
2560 by 10576 and 5120 by 2560, a mixer's state of (3, 5376) in fp16 and (80, 64, 128) in fp32; and their tests' neighbours.
Decays: "retention", one for each head, 1 - 2^-5 to 1 - 2^-13; "strong" and "weak", for each token, log-sigmoid(N(2, 1)) and a
sixteenth of it; "none".
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
CHUNK = 64


def _prompt(lens, H, *, K=128, V=128, dtype="fp16", packed=True, decay="retention", name=None):
    c = dict(op="prompt", lens=lens, H=H, K=K, V=V, dtype=dtype, packed=packed, decay=decay)
    return c if name is None else dict(c, name=name)


def _step(batch, H, *, K=128, V=128, dtype="fp16", decay="retention", name=None):
    c = dict(op="step", batch=batch, H=H, K=K, V=V, dtype=dtype, decay=decay)
    return c if name is None else dict(c, name=name)


def _norm(rows, H, V, *, dtype="fp16", gate=True, affine=True, act="silu", name=None):
    c = dict(op="norm", rows=rows, H=H, V=V, dtype=dtype, gate=gate, affine=affine, act=act)
    return c if name is None else dict(c, name=name)


def _adapters(M, K, N, *, R=16, count=8, run=1, coded=False, dtype="fp16", bias=False, name=None):
    c = dict(op="adapters", M=M, K=K, N=N, R=R, count=count, run=run, coded=coded, dtype=dtype, bias=bias)
    return c if name is None else dict(c, name=name)


def _slots(moves, slots, layers, *, kind="mixer", freed=0.0, inplace=False, name=None):
    c = dict(op="slots", moves=moves, slots=slots, layers=layers, kind=kind, freed=freed, inplace=inplace)
    return c if name is None else dict(c, name=name)


def _same(n, length):
    return ",".join([str(length)] * n)


def listed():
    return [
        # one short prompt: launches and the chain of chunks count
        _prompt("500", 16, dtype="bf16", packed=False, name="prompt_b1_l500"),
        # a ragged batch of prompts, an empty one and a single token among them, some going on from a state; a decay of each token
        _prompt("1200,1,64,2047,0,333,1024,3,777,1500", 16, decay="strong", name="prompt_ragged_h16"),
        # long prompts at the largest zoo configuration
        _prompt(_same(2, 8192), 32, packed=False, name="prompt_b2_l8192_h32"),
        # few and many sequences that answer
        _step(4, 16, name="step_b4"),
        _step(256, 32, dtype="bf16", decay="weak", name="step_b256"),
        # one token of 16 sequences, norm of 32 heads of 128 with a gate
        _norm(16, 32, 128, dtype="bf16", name="norm_decode_b16"),
        # the same over prompts
        _norm(16384, 32, 128, name="norm_b2_l8192"),
        # the projection into a mixer for 16 sequences that answer, a request each
        _adapters(16, 2560, 10576, count=16, name="adapters_in_decode_b16"),
        # the projection out of it for a few prompts, a token count off every tile, codes in hand
        _adapters(3001, 5120, 2560, R=32, run=700, coded=True, dtype="bf16", bias=True, name="adapters_out_m3001"),
        # the projection into it over long prompts of eight requests
        _adapters(16384, 2560, 10576, run=2048, name="adapters_in_m16384"),
        # one sequence's state forked to four, one layer
        _slots(4, 16, 1, kind="heads", name="slots_fork_4"),
        # 64 sequences of four layers in a new order, some ended
        _slots(64, 72, 4, freed=0.1, inplace=True, name="slots_reorder_64"),
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
    op = rng.choice(["prompt", "step", "norm", "adapters", "slots"])
    dtype = rng.choice(["fp16", "bf16"])
    if op in ("prompt", "step"):
        H, decay = rng.choice([32, 16, 8, 5]), rng.choice(["retention", "strong", "weak", "none"])
        K, V = rng.choice([(128, 128), (128, 128), (64, 64), (64, 128), (128, 256), (256, 128), (96, 40), (32, 72)])
        if op == "step":
            return _step(int(_log(rng, 1, 256 if K * V <= 128 * 128 else 128)), H, K=K, V=V, dtype=dtype, decay=decay)
        ragged = rng.random() < 0.6
        return _prompt(_draw_lens(rng, _log(rng, 1, 16384 if K * V <= 128 * 128 else 8192), ragged), H, K=K, V=V, dtype=dtype, packed=ragged, decay=decay)
    if op == "norm":
        H, V = rng.choice([(32, 128), (16, 128), (16, 256), (8, 64), (5, 40), (7, 99), (1, 2560)])
        return _norm(int(_log(rng, 1, 16384)), H, V, dtype=dtype, gate=rng.random() < 0.7, affine=rng.random() < 0.7,
                     act=rng.choice(["silu", "silu", "sigmoid", "none"]))
    if op == "adapters":
        K, N = rng.choice([(2560, 10576), (5120, 2560), (2048, 8512), (4096, 2048), (1040, 777)])
        M = int(_log(rng, 1, 16384))
        return _adapters(M, K, N, R=rng.choice([8, 16, 16, 32, 64, 12]), count=rng.choice([1, 4, 8, 16]), run=int(_log(rng, 1, max(1.5, M))),
                         coded=rng.random() < 0.4, dtype=dtype, bias=rng.random() < 0.5)
    kind = rng.choice(["mixer", "heads", "odd"])
    moves = int(_log(rng, 1, 64))
    return _slots(moves, 2 * moves + rng.randrange(8), rng.choice([1, 2, 3]), kind=kind, freed=rng.choice([0.0, 0.2]), inplace=rng.random() < 0.6)


# ------------------------------------------------------------------------------------------------------------- inputs
KINDS = {"mixer": [((3, 5376), torch.float16), ((80, 64, 128), torch.float32)],     # a Mamba-2 mixer's
         "heads": [((32, 128, 128), torch.float32)],                                # a linear attention's
         "odd": [((3, 1032), torch.bfloat16), ((5, 96, 40), torch.float32), ((7,), torch.float16)]}


def _lens(c):
    return [int(n) for n in c["lens"].split(",")]


def _starts(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed % (1 << 62))
    rn = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    un = lambda *shape: torch.rand(*shape, generator=gen, device="cuda")  # noqa: E731
    perm = lambda n: torch.randperm(n, generator=gen, device="cuda").to(torch.int32)  # noqa: E731
    if c["op"] == "slots":
        n, total = c["moves"], c["slots"]
        states = [[rn(total, *shape).to(dt) for shape, dt in KINDS[c["kind"]]] for _ in range(c["layers"])]
        dst = perm(total)[:n]
        # in place: the sources are the destinations in another order; else one of three sequences is forked, from a slot that is kept
        src = dst[perm(n).long()] if c["inplace"] else perm(total)[torch.randint(0, min(3, total), (n,), generator=gen, device="cuda")]
        return dict(c=c, states=states, dst=dst, src=torch.where(un(n) < c["freed"], -1, src).to(torch.int32))
    dt = DTYPES[c["dtype"]]
    if c["op"] == "norm":
        rows, D = c["rows"], c["H"] * c["V"]
        return dict(c=c, x=((0.5 + un(rows, 1)) * (rn(rows, D) + 0.3)).to(dt), z=rn(rows, D).to(dt) if c["gate"] else None,
                    weight=(1 + 0.1 * rn(D)).to(dt) if c["affine"] else None, bias=(0.1 * rn(D)).to(dt) if c["affine"] else None)
    if c["op"] == "adapters":
        M, K, N, R, n = c["M"], c["K"], c["N"], c["R"], c["count"]
        w = rn(N, K) / math.sqrt(K)
        ws = w.abs().amax(1) / 127.0
        s = dict(c=c, w=torch.round(w / ws[:, None]).to(torch.int8), w_scale=ws, bias=rn(N).to(dt) if c["bias"] else None,
                 a=(rn(n, R, K) / math.sqrt(K)).to(dt), b=(rn(n, N, R) / math.sqrt(R)).to(dt), scaling=0.25 + 0.5 * un(n))
        # a request's rows lie together; the last request has no adapter
        runs = -(-M // c["run"])
        of = (torch.arange(runs, device="cuda") + torch.randint(0, n, (1,), generator=gen, device="cuda")) % n
        if runs > 1:
            of[-1] = -1
        s["ids"] = of.repeat_interleave(c["run"])[:M].to(torch.int32)
        x = rn(M, K) * (0.5 + un(M, 1))
        if c["coded"]:
            s["x_scale"] = x.abs().amax(1) / 127.0
            s["x"] = torch.round(x / s["x_scale"][:, None]).to(torch.int8)
        else:
            s["x"] = x.to(dt)
        if own:  # weights laid out once
            from linquant_amd.w8a8_linear import LowRankAdapters, W8A8Linear

            s["linear"] = W8A8Linear(s["w"], s["w_scale"], bias=s["bias"])
            s["adapters"] = LowRankAdapters(s["a"], s["b"], s["scaling"])
        return s
    H, K, V = c["H"], c["K"], c["V"]
    n = c["batch"] if c["op"] == "step" else len(_lens(c))
    T = c["batch"] if c["op"] == "step" else sum(_lens(c))
    wide = rn(T, H * (2 * K + V)).to(dt)                 # q, k and v are views of what the projection gives
    q, k, v = (t.unflatten(1, (H, -1)) for t in wide.split([H * K, H * K, H * V], dim=1))
    g = {"retention": lambda: torch.log1p(-torch.exp2(-5.0 - 8.0 * torch.arange(H, device="cuda") / H)),
         "strong": lambda: -torch.log1p(torch.exp(-(2 + rn(T, H)))), "weak": lambda: -torch.log1p(torch.exp(-(2 + rn(T, H)))) / 16,
         "none": lambda: None}[c["decay"]]()
    s = dict(c=c, q=q, k=k, v=v, g=g, slots=perm(n + 3)[:n], state=rn(n + 3, H, K, V))
    if c["op"] == "prompt":
        lens = _lens(c)
        s.update(starts=_starts(lens), longest=max(lens))
        if not c["packed"]:
            for key in ("q", "k", "v") + (("g",) if g is not None and g.dim() == 2 else ()):
                s[key] = s[key].unflatten(0, (n, lens[0]))
    return s


# ---------------------------------------------------------------------------------------------------------- plain forms
def _plain_prompt(s):
    c, slots, n = s["c"], s["slots"].long(), s["slots"].numel()
    H, K, V, Q = c["H"], c["K"], c["V"], CHUNK
    q, k, v = (s[key].reshape(-1, H, d) for key, d in (("q", K), ("k", K), ("v", V)))
    T, L = q.shape[0], -(-s["longest"] // Q) * Q
    # every sequence padded to whole chunks by tokens with k = 0 and no decay, which change nothing
    pos = torch.arange(L, device=q.device)
    lens = (s["starts"][1:] - s["starts"][:-1]).long()
    real = pos < lens[:, None]
    at = (s["starts"][:-1].long()[:, None] + pos).clamp(max=T - 1)
    if s["g"] is None:
        g = torch.zeros(n, L, H, device=q.device)
    else:
        g = (s["g"].expand(n, L, H) if s["g"].dim() == 1 else s["g"].reshape(T, H)[at]) * real[..., None]
    nc = L // Q
    q, k, v = ((t[at].float() * real[..., None, None]).view(n, nc, Q, H, -1).permute(0, 3, 1, 2, 4) for t in (q, k, v))   # (n, H, nc, Q, .)
    cum = torch.cumsum(g.view(n, nc, Q, H).double(), 2).permute(0, 3, 1, 2)                 # long sums in 64 bits
    later = torch.ones(Q, Q, dtype=torch.bool, device=q.device).tril()
    w = torch.where(later, torch.exp(torch.where(later, cum[..., :, None] - cum[..., None, :], 0.0).float()), 0.0)
    o = ((q @ k.transpose(-1, -2)) * w) @ v
    last = cum[..., -1]
    local = (k * torch.exp((last[..., None] - cum).float())[..., None]).transpose(-1, -2) @ v    # (n, H, nc, K, V)
    # the states in front of the chunks, chunk by chunk
    S, before = s["state"][slots], []
    for i in range(nc):
        before.append(S)
        S = S * torch.exp(last[:, :, i].float())[..., None, None] + local[:, :, i]
    o = o + (q * torch.exp(cum.float())[..., None]) @ torch.stack(before, 2)
    o = (o * K ** -0.5).permute(0, 2, 3, 1, 4).reshape(n, L, H, V)
    s["state"][slots] = S
    return o[real].to(s["v"].dtype).view(s["v"].shape), s["state"]


def _plain_step(s):
    slots, g = s["slots"].long(), s["g"]
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    S = s["state"][slots]
    if g is not None:
        S = S * torch.exp(g)[..., None, None]
    S = S + k[..., None] * v[:, :, None]
    o = (S * q[..., None]).sum(2) * s["c"]["K"] ** -0.5
    s["state"][slots] = S
    return o.to(s["v"].dtype), s["state"]


def _act(u, act):
    return {"silu": lambda: u * torch.sigmoid(u), "sigmoid": lambda: torch.sigmoid(u), "none": lambda: u}[act]()


def _plain_norm(s):
    c = s["c"]
    x = s["x"].float().view(-1, c["H"], c["V"])
    mean = x.mean(-1, keepdim=True)
    y = ((x - mean) * torch.rsqrt((x - mean).square().mean(-1, keepdim=True) + 1e-5)).view(s["x"].shape)
    if s["weight"] is not None:
        y = y * s["weight"].float() + s["bias"].float()
    y = _act(y, c["act"]) if s["z"] is None else y * _act(s["z"].float(), c["act"])
    return y.to(s["x"].dtype)


def _plain_adapters(s):
    c, dt = s["c"], DTYPES[s["c"]["dtype"]]
    if c["coded"]:
        codes, xs = s["x"].float(), s["x_scale"][:, None]
        x = codes * xs
    else:
        x = s["x"].float()
        xs = x.abs().amax(1, keepdim=True) / 127.0
        codes = torch.round(x / torch.where(xs > 0, xs, 1.0))
    y = (codes @ s["w"].float().T) * (xs * s["w_scale"])
    # each row against all adapters, those of other requests left out
    n, R = c["count"], c["R"]
    mine = s["ids"][:, None] == torch.arange(n, device=x.device)
    h = (x @ s["a"].float().flatten(0, 1).T).view(-1, n, R) * (mine * s["scaling"])[..., None]
    y = y + h.flatten(1) @ s["b"].float().permute(0, 2, 1).flatten(0, 1)
    return (y if s["bias"] is None else y + s["bias"].float()).to(dt)


def _plain_slots(s):
    src, dst = s["src"].long(), s["dst"].long()
    for layer in s["states"]:
        for t in layer:
            kept = (src >= 0).view(-1, *[1] * (t.dim() - 1))
            t[dst] = torch.where(kept, t[src.clamp(min=0)], 0.0)
    return s["states"]


# ------------------------------------------------------------------------------------------------------------ own calls
def _own_prompt(s):
    from linquant_amd.kernels.zoo.linear_attention import linear_attention_prompt

    return linear_attention_prompt(s["q"], s["k"], s["v"], s["g"], state=s["state"], slots=s["slots"],
                                   seq_starts=s["starts"] if s["c"]["packed"] else None), s["state"]


def _own_step(s):
    from linquant_amd.kernels.zoo.linear_attention import linear_attention_step

    return linear_attention_step(s["state"], s["q"], s["k"], s["v"], s["g"], slots=s["slots"]), s["state"]


def _own_norm(s):
    from linquant_amd.norm import groupnorm_gated

    c = s["c"]
    return groupnorm_gated(s["x"], s["z"], s["weight"], s["bias"], num_groups=c["H"], eps=1e-5, activation=None if c["act"] == "none" else c["act"])


def _own_adapters(s):
    if s["c"]["coded"]:
        return s["linear"].forward_int8(s["x"], s["x_scale"], DTYPES[s["c"]["dtype"]], adapters=s["adapters"], ids=s["ids"])
    return s["linear"](s["x"], adapters=s["adapters"], ids=s["ids"])


def _own_slots(s):
    from linquant_amd.slots import copy_slots

    copy_slots(s["states"], s["src"], s["dst"])
    return s["states"]


def run(state):
    op = state["c"]["op"]
    if own:
        return {"prompt": _own_prompt, "step": _own_step, "norm": _own_norm, "adapters": _own_adapters, "slots": _own_slots}[op](state)
    return {"prompt": _plain_prompt, "step": _plain_step, "norm": _plain_norm, "adapters": _plain_adapters, "slots": _plain_slots}[op](state)


def work(case):
    """Bytes: every input once, every output once, the states of the sequences read and written.  Operations: multiplications and
    additions of the definition, the attention's by its recurrence."""
    c = case
    if c["op"] == "slots":
        size = sum(math.prod(shape) * (4 if dt == torch.float32 else 2) for shape, dt in KINDS[c["kind"]]) * c["layers"]
        return {"bytes": int(size * c["moves"] * (2 - c["freed"])) + 8 * c["moves"], "flops": 0}
    if c["op"] == "norm":
        n, D = c["rows"] * c["H"] * c["V"], c["H"] * c["V"]
        return {"bytes": 2 * n * (3 if c["gate"] else 2) + (4 * D if c["affine"] else 0), "flops": n * (5 + 2 * c["affine"] + (0 if c["act"] == "none" else 4) + c["gate"])}
    if c["op"] == "adapters":
        M, K, N, R = c["M"], c["K"], c["N"], c["R"]
        runs = -(-M // c["run"])
        used, rows = (min(c["count"], runs - 1), (runs - 1) * c["run"]) if runs > 1 else (1, M)
        return {"bytes": M * K * (1 if c["coded"] else 2) + (4 * M if c["coded"] else 0) + N * K + 4 * N + (2 * N if c["bias"] else 0) + 4 * M + 2 * M * N + used * (2 * R * (K + N) + 4),
                "flops": 2 * M * N * K + 2 * rows * R * (K + N)}
    H, K, V = c["H"], c["K"], c["V"]
    n, T = (c["batch"], c["batch"]) if c["op"] == "step" else (sum(v > 0 for v in _lens(c)), sum(_lens(c)))
    g = {"retention": 4 * H, "none": 0}.get(c["decay"], 4 * T * H)
    return {"bytes": 2 * T * H * (2 * K + 2 * V) + g + 8 * n * H * K * V, "flops": T * H * 5 * K * V}


# ----------------------------------------------------------------------------------------------- definition in 64 bits
def exact(case, seed):
    s, c = prepare(case, seed), case
    f = lambda t: t.double()  # noqa: E731
    if c["op"] == "slots":
        src, dst = s["src"].tolist(), s["dst"].tolist()
        out = []
        for layer in s["states"]:
            new = [t.clone() for t in layer]
            for i, j in zip(src, dst):
                for t, u in zip(layer, new):
                    u[j] = t[i] if i >= 0 else 0.0
            out.append(new)
        return out
    act = {"silu": lambda u: u / (1 + (-u).exp()), "sigmoid": lambda u: 1 / (1 + (-u).exp()), "none": lambda u: u}
    if c["op"] == "norm":
        x = f(s["x"]).unflatten(1, (c["H"], c["V"]))
        d = x - x.sum(-1, keepdim=True) / c["V"]
        y = (d / (d.pow(2).sum(-1, keepdim=True) / c["V"] + 1e-5).sqrt()).flatten(1)
        if c["affine"]:
            y = y * f(s["weight"]) + f(s["bias"])
        return act[c["act"]](y) if s["z"] is None else y * act[c["act"]](f(s["z"]))
    if c["op"] == "adapters":
        # codes are whole numbers of the 32-bit quotient by definition: the 64-bit part is the products
        if c["coded"]:
            codes, top = s["x"], s["x_scale"]
            x = f(codes) * f(top)[:, None]
        else:
            x32 = s["x"].float()
            top = x32.abs().max(dim=1).values / 127.0
            codes = torch.where(top[:, None] > 0, (x32 / top[:, None]).round(), torch.zeros_like(x32))
            x = f(x32)
        y = torch.mm(f(codes), f(s["w"]).t()) * f(top)[:, None] * f(s["w_scale"])[None]
        if c["bias"]:
            y += f(s["bias"])
        ids = s["ids"].cpu()
        for j in sorted(set(ids.tolist()) - {-1}):
            rows = (ids == j).nonzero()[:, 0].cuda()
            y[rows] += f(s["scaling"])[j] * torch.mm(torch.mm(x[rows], f(s["a"][j]).t()), f(s["b"][j]).t())
        return y
    H, K, V = c["H"], c["K"], c["V"]
    lens = [1] * c["batch"] if c["op"] == "step" else _lens(c)
    if max(lens) > 40000:
        return None
    q, k, v = f(s["q"]).reshape(-1, H, K) * K ** -0.5, f(s["k"]).reshape(-1, H, K), f(s["v"]).reshape(-1, H, V)
    T = q.shape[0]
    decay = torch.ones(T, H, device="cuda").double() if s["g"] is None else f(s["g"]).exp().reshape(-1, H).expand(T, H)
    o, state = torch.empty_like(v), f(s["state"])
    # token by token, over the sequences that still have one
    order = sorted(range(len(lens)), key=lambda i: -lens[i])
    begin = [sum(lens[:i]) for i in range(len(lens))]
    slots = s["slots"].tolist()
    idx = torch.tensor([slots[i] for i in order], device="cuda")
    row = torch.tensor([begin[i] for i in order], device="cuda")
    S, live = state[idx], len(order)
    for t in range(max(lens)):
        while live and lens[order[live - 1]] <= t:
            live -= 1
        r = row[:live] + t
        S[:live] *= decay[r][:, :, None, None]
        S[:live] += k[r][..., None] * v[r][:, :, None]
        o[r] = (S[:live] * q[r][..., None]).sum(2)
    state[idx] = S
    return o.view(s["v"].shape), state
