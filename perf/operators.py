"""Cases and plain forms of the sequence-model operators: leaky attention
(linear attention with a decay for each head), the fused norm / gate /
residual of a block, and the embedding with its gradient.

`own` chooses what `run` calls: the framework's operators, or the same
mathematics in elementary torch operations, in fp32, rounded once at the end.
"""
import math

import torch

own = False

_DT = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    return [
        # one sequence answering token by token: latency of one layer's state update
        dict(name="step one sequence", op="step", B=1, slots=1, H=4, Hk=4, Dk=64, Dv=64, dtype="bfloat16"),
        # a serving batch over a cache of states, a few of its places empty
        dict(name="step full batch", op="step", B=190, slots=203, H=16, Hk=16, Dk=128, Dv=128, dtype="bfloat16"),
        # one long prompt with shared key/value heads, continuing a state and leaving one
        dict(name="prompt one long", op="prompt", B=1, T=16381, H=16, Hk=4, Dk=128, Dv=128, dtype="bfloat16",
             ragged=False, state=True),
        # a batch of prompts of unequal length, one of them empty, padded to the longest
        dict(name="prompts ragged", op="prompt", B=24, T=2047, H=8, Hk=8, Dk=64, Dv=64, dtype="bfloat16",
             ragged=True, state=True),
        # a training step's attention: forward, and the gradients of q, k, v
        dict(name="attention train", op="attn_train", B=8, T=4096, H=16, Hk=16, Dk=128, Dv=128, dtype="bfloat16",
             ragged=False, state=False),
        # the same in fp32 at the spiking network's size: T = 1024, batch 64, width 256 as 4 heads
        dict(name="attention train fp32", op="attn_train", B=64, T=1024, H=4, Hk=4, Dk=64, Dv=64, dtype="float32",
             ragged=False, state=False),
        # the norms of a block for one token
        dict(name="norm one token", op="norm", R=1, D=256, gate="full", act="silu", dtype="bfloat16"),
        # the norms of a wide block in training, an elementwise gate
        dict(name="norm train wide", op="norm_train", R=32768, D=2048, gate="full", act="silu", dtype="bfloat16"),
        # the spiking network's rows (1024 steps x batch 64) and width, one gate value for each row
        dict(name="norm train fp32", op="norm_train", R=65536, D=256, gate="row", act="sigmoid", dtype="float32"),
        # the tokens of one serving step
        dict(name="embed step", op="embed", n=64, V=700, D=256, dtype="float32", zipf=False),
        # the spiking network's 700 input channels as tokens: few rows, each used often
        dict(name="embed train channels", op="embed_train", n=65536, V=700, D=256, dtype="float32", zipf=False),
        # a text-sized vocabulary: a few tokens very often, most rows not at all
        dict(name="embed train text", op="embed_train", n=32768, V=50001, D=1024, dtype="bfloat16", zipf=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["step", "prompt", "prompt", "attn_train", "attn_train", "norm", "norm_train", "norm_train",
                     "embed", "embed_train"])
    if op in ("step", "prompt", "attn_train"):
        dt = rng.choice(["bfloat16", "bfloat16", "float32"])
        H = rng.choice([1, 2, 3, 4, 6, 8, 12, 16])
        Hk = rng.choice([h for h in range(1, H + 1) if H % h == 0 and (h == H or H // h <= 8)] + [H, H])
        c = dict(op=op, H=H, Hk=Hk, Dk=rng.choice([16, 32, 40, 64, 64, 80, 96, 128, 128]),
                 Dv=rng.choice([16, 32, 48, 64, 64, 72, 112, 128, 128]), dtype=dt)
        if op == "step":
            c["B"] = _log_int(rng, 1, 190)
            c["slots"] = c["B"] + rng.randrange(14)
            return c
        # at most 2^23.. elements of q (fp32: 2^22..), the listed training cases' order
        most = (1 << 25) if dt == "bfloat16" else (1 << 23)
        T = _log_int(rng, 1, 16381 if op == "prompt" else 6000)
        B = max(1, min(64, most // (T * H * 128)))
        c.update(B=_log_int(rng, 1, B), T=T, ragged=rng.random() < 0.3, state=rng.random() < 0.5)
        return c
    if op in ("norm", "norm_train"):
        D = _log_int(rng, 32, 6000)
        if rng.random() < 0.7:
            D = max(8, D // 8 * 8)
        R = _log_int(rng, 1, max(2, (1 << 25) // D) if op == "norm_train" else 300)
        return dict(op=op, R=R, D=D, gate=rng.choice(["full", "full", "row", "none"]),
                    act=rng.choice(["silu", "sigmoid"]), dtype=rng.choice(["float32", "bfloat16", "float16"]))
    V = _log_int(rng, 20, 50001)
    D = _log_int(rng, 32, 1024)
    if rng.random() < 0.7:
        D = max(8, D // 8 * 8)
    n = _log_int(rng, 1, 65536 if D <= 512 else 32768) if op == "embed_train" else _log_int(rng, 1, 4096)
    return dict(op=op, n=n, V=V, D=D, dtype=rng.choice(["float32", "bfloat16", "float16"]), zipf=rng.random() < 0.5)


def _lengths(case):
    """Valid tokens of each sequence: all, or spread over 0..T by the golden ratio."""
    B, T = case["B"], case["T"]
    if not case["ragged"]:
        return [T] * B
    n = [int((0.6180339887 * (b + 1)) % 1.0 * T) for b in range(B)]
    n[0] = T
    if B > 1:
        n[-1] = 0
    return n


def _log_decay(H, dev):
    # memories from a few tokens to tens of thousands; the last head of several forgets nothing
    e = torch.linspace(1.0, 14.0, H, device=dev)
    ld = torch.log1p(-torch.exp2(-e))
    if H > 2:
        ld[-1] = 0.0
    return ld


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = _DT[case["dtype"]]

    def rand(*shape, mean=0.0, sd=1.0, dtype=dt):
        return (torch.randn(*shape, device=dev, generator=g) * sd + mean).to(dtype)

    op = case["op"]
    s = {"op": op, "case": case}
    if op in ("step", "prompt", "attn_train"):
        B, H, Hk, Dk, Dv = (case[k] for k in ("B", "H", "Hk", "Dk", "Dv"))
        lead = (B,) if op == "step" else (B, case["T"])
        s["q"], s["k"], s["v"] = rand(*lead, H, Dk), rand(*lead, Hk, Dk, sd=Dk ** -0.5), rand(*lead, Hk, Dv, mean=0.1)
        s["log_decay"] = _log_decay(H, dev)
        if op == "step":
            s["state"] = rand(case["slots"], H, Dk, Dv, dtype=torch.float32)
            order = torch.randperm(case["slots"], device=dev, generator=g)[:B].to(torch.int32)
            if B > 8:
                order[torch.randint(0, B, (2,), device=dev, generator=g)] = -1  # places without a sequence
            s["slots"] = order
        else:
            s["state"] = rand(B, H, Dk, Dv, dtype=torch.float32) if case["state"] else None
            s["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device=dev) if case["ragged"] else None
        if op == "attn_train":
            s["do"] = rand(B, case["T"], H, Dv, sd=0.1)
            for k in ("q", "k", "v") + (("state",) if case["state"] else ()):
                s[k].requires_grad_()
    elif op in ("norm", "norm_train"):
        R, D = case["R"], case["D"]
        s["x"], s["h"] = rand(R, D), rand(R, D, sd=2.0)
        s["gate"] = None if case["gate"] == "none" else rand(R, D if case["gate"] == "full" else 1)
        s["post"], s["pre"] = (rand(D, mean=1.0, sd=0.1, dtype=torch.float32) for _ in range(2))
        if op == "norm_train":
            s["dx"], s["dn"] = rand(R, D, sd=0.1), rand(R, D, sd=0.1)
            for k in ("x", "h", "post", "pre") + (("gate",) if s["gate"] is not None else ()):
                s[k].requires_grad_()
    else:
        n, V, D = case["n"], case["V"], case["D"]
        if case["zipf"]:
            u = torch.rand(n, device=dev, generator=g)
            tok = torch.exp(u * math.log(V)).long().clamp_(1, V) - 1
            tok = (tok * 7919) % V if V % 7919 else tok  # the frequent ones spread over the table
        else:
            tok = torch.randint(0, V, (n,), device=dev, generator=g)
        if n > 16:
            tok[torch.randint(0, n, (n // 16,), device=dev, generator=g)] = -1  # padding
        s["tokens"], s["weight"] = tok, rand(V, D)
        if op == "embed_train":
            s["dy"] = rand(n, D, sd=0.1)
            s["weight"].requires_grad_()
    return s


_RES_SCALE, _EPS = 0.5, 1e-6


def run(s):
    case = s["case"]
    op = s["op"]
    if op == "step":
        return _step_own(s) if own else _step_plain(s)
    if op in ("prompt", "attn_train"):
        o, st = _attention_own(s) if own else _attention_plain(s)
        if op == "prompt":
            return {"o": o, "state": st}
        wrt = [s["q"], s["k"], s["v"]] + ([s["state"]] if case["state"] else [])
        gr = torch.autograd.grad(o, wrt, s["do"])
        return {"o": o.detach(), **dict(zip(("dq", "dk", "dv", "dstate"), gr))}
    if op in ("norm", "norm_train"):
        x, n = _norm_own(s) if own else _norm_plain(s)
        if op == "norm":
            return {"x": x, "n": n}
        names = ["x", "h", "post", "pre"] + (["gate"] if s["gate"] is not None else [])
        gr = torch.autograd.grad((x, n), [s[k] for k in names], (s["dx"], s["dn"]))
        return {"x": x.detach(), "n": n.detach(), **{"d" + k: v for k, v in zip(names, gr)}}
    y = _embed_own(s) if own else _embed_plain(s)
    if op == "embed":
        return {"y": y}
    return {"y": y.detach(), "dweight": torch.autograd.grad(y, s["weight"], s["dy"])[0]}


# ---- the framework's operators

def _step_own(s):
    from hard_resets_compose_b200 import leakyattn
    o = leakyattn.leaky_attention_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"], slots=s["slots"])
    return {"o": o, "state": s["state"]}


def _attention_own(s):
    from hard_resets_compose_b200 import leakyattn
    if s["op"] == "prompt":
        return leakyattn.leaky_attention(s["q"], s["k"], s["v"], s["log_decay"], state=s["state"],
                                         lengths=s["lengths"], return_state=True)
    return leakyattn.leaky_attention(s["q"], s["k"], s["v"], s["log_decay"], state=s["state"],
                                     lengths=s["lengths"]), None


def _norm_own(s):
    from hard_resets_compose_b200 import normgate
    return normgate.norm_gate_residual(s["x"], s["h"], s["gate"], s["post"], s["pre"], residual_scale=_RES_SCALE,
                                       act=s["case"]["act"], eps=_EPS)


def _embed_own(s):
    from hard_resets_compose_b200 import embed
    return embed.embedding(s["tokens"], s["weight"], scale=s["case"]["D"] ** 0.5)


# ---- the plain forms

def _step_plain(s):
    c, st = s["case"], s["state"]
    grp = c["H"] // c["Hk"]
    slot = s["slots"].long()
    live = (slot >= 0)[:, None, None]
    at = slot.clamp(min=0)
    q = s["q"].float() * c["Dk"] ** -0.5
    k, v = s["k"].float().repeat_interleave(grp, 1), s["v"].float().repeat_interleave(grp, 1)
    new = torch.exp(s["log_decay"])[:, None, None] * st[at] + k[..., :, None] * v[..., None, :]
    o = torch.where(live, (q[..., :, None] * new).sum(-2), 0.0)
    keep = torch.where(slot >= 0, slot, st.shape[0])  # an empty place writes past the cache's end
    wide = torch.cat([st, st[:1]])
    wide[keep] = new
    st.copy_(wide[:-1])
    return {"o": o.to(s["q"].dtype), "state": st}


def _attention_plain(s):
    """Chunks of 64 tokens: scores within a chunk, states between chunks joined by a matrix of decays."""
    c = s["case"]
    B, T, H, grp, C = c["B"], c["T"], c["H"], c["H"] // c["Hk"], 64
    dev = s["q"].device
    nc = -(-T // C)
    length = s["lengths"].long() if s["lengths"] is not None else torch.full((B,), T, device=dev)
    valid = torch.arange(nc * C, device=dev)[None] < length[:, None]

    def chunks(x, rep):
        x = torch.nn.functional.pad(x.float(), (0, 0, 0, 0, 0, nc * C - T))
        x = torch.where(valid[..., None, None], x, 0.0)
        return x.repeat_interleave(rep, 2).transpose(1, 2).reshape(B, H, nc, C, -1)

    q, k, v = chunks(s["q"], 1) * c["Dk"] ** -0.5, chunks(s["k"], grp), chunks(s["v"], grp)
    ld = s["log_decay"].float()
    i = torch.arange(C, device=dev)
    dist = (i[:, None] - i[None, :]).clamp(min=0)
    mask = torch.where(i[:, None] >= i[None, :], torch.exp(ld[:, None, None] * dist), 0.0)
    o = ((q @ k.transpose(-1, -2)) * mask[:, None]) @ v
    # state after a chunk's n valid tokens: sum of b^(n-1-j) k_j v_j, and b^n of the state before
    start = (torch.arange(nc + 1, device=dev) * C)[None].minimum(length[:, None])  # [B, nc + 1]
    n = start[:, 1:] - start[:, :-1]
    left = (n[:, None, :, None] - 1 - i).clamp(min=0)  # [B, 1, nc, C]
    kv = (k * torch.exp(ld[:, None, None] * left)[..., None]).transpose(-1, -2) @ v
    at = torch.arange(nc + 1, device=dev)
    gap = (start[:, None, :, None] - start[:, None, None, 1:]).clamp(min=0)  # chunk boundary after chunk
    join = torch.where((at[:, None] > at[None, :-1]), torch.exp(ld[:, None, None] * gap), 0.0)  # [B, H, nc + 1, nc]
    st = (join @ kv.reshape(B, H, nc, -1)).reshape(B, H, nc + 1, c["Dk"], c["Dv"])
    if s["state"] is not None:
        st = st + torch.exp(ld[:, None] * start[:, None])[..., None, None] * s["state"][:, :, None]
    o = o + (q * torch.exp(ld[:, None] * (i + 1))[:, None, :, None]) @ st[:, :, :-1]
    o = o.reshape(B, H, nc * C, -1)[:, :, :T].transpose(1, 2)
    o = torch.where(valid[:, :T, None, None], o, 0.0)
    return o.to(s["q"].dtype), st[:, :, -1].contiguous()


def _rms(x, w):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * w


def _norm_plain(s):
    y = _rms(s["h"].float(), s["post"])
    if s["gate"] is not None:
        g = s["gate"].float()
        sg = 1.0 / (1.0 + torch.exp(-g))
        y = y * (g * sg if s["case"]["act"] == "silu" else sg)
    x = s["x"].float() + _RES_SCALE * y
    return x.to(s["x"].dtype), _rms(x, s["pre"]).to(s["x"].dtype)


def _embed_plain(s):
    tok = s["tokens"]
    y = s["weight"].float()[tok.clamp(min=0)] * s["case"]["D"] ** 0.5
    return torch.where((tok >= 0)[:, None], y, 0.0).to(s["weight"].dtype)


# ---- what a pass cannot do without

def work(case):
    e = 4 if case["dtype"] == "float32" else 2
    op = case["op"]
    if op == "step":
        B, H, Hk, Dk, Dv = (case[k] for k in ("B", "H", "Hk", "Dk", "Dv"))
        io = B * (H * Dk + Hk * Dk + Hk * Dv + H * Dv) * e
        return {"bytes": io + 8 * B * H * Dk * Dv, "flops": 5 * B * H * Dk * Dv}
    if op in ("prompt", "attn_train"):
        B, T, H, Hk, Dk, Dv = (case[k] for k in ("B", "T", "H", "Hk", "Dk", "Dv"))
        n = sum(_lengths(case))
        q, kv, o = H * Dk * e, Hk * (Dk + Dv) * e, H * Dv * e
        st = 4 * B * H * Dk * Dv
        if op == "prompt":
            return {"bytes": n * (q + kv) + B * T * o + st * (1 + case["state"]), "flops": 4 * n * H * Dk * Dv}
        return {"bytes": n * (q + kv + o) + B * T * (q + kv + o) + 2 * st * case["state"],
                "flops": 14 * n * H * Dk * Dv}
    if op in ("norm", "norm_train"):
        R, D = case["R"], case["D"]
        g = R * {"full": D, "row": 1, "none": 0}[case["gate"]] * e
        if op == "norm":
            return {"bytes": 4 * R * D * e + g + 8 * D, "flops": 12 * R * D}
        return {"bytes": 8 * R * D * e + 2 * g + 16 * D, "flops": 40 * R * D}
    n, V, D = case["n"], case["V"], case["D"]
    if op == "embed":
        return {"bytes": (min(n, V) + n) * D * e + 8 * n, "flops": n * D}
    return {"bytes": (min(n, V) + 2 * n + V) * D * e + 8 * n, "flops": 2 * n * D}


# ---- the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    s = {k: v.detach() if isinstance(v, torch.Tensor) else v for k, v in s.items()}
    op = case["op"]
    with torch.no_grad():
        if op in ("step", "prompt", "attn_train"):
            return _exact_attention(case, s)
        if op in ("norm", "norm_train"):
            return _exact_norm(case, s)
        return _exact_embed(case, s)


def _exact_attention(case, s):
    """The recurrence itself, token by token, in both directions."""
    q, k, v = (s[n].double() for n in ("q", "k", "v"))
    H, rep, scale = case["H"], case["H"] // case["Hk"], 1.0 / math.sqrt(case["Dk"])
    b = s["log_decay"].double().exp()[None, :, None, None]
    if case["op"] == "step":
        S = s["state"].double()
        out = torch.zeros(case["B"], H, case["Dv"], dtype=torch.float64, device=q.device)
        for i, slot in enumerate(s["slots"].tolist()):
            if slot >= 0:
                for h in range(H):
                    S[slot, h] = b[0, h] * S[slot, h] + torch.outer(k[i, h // rep], v[i, h // rep])
                    out[i, h] = scale * (q[i, h] @ S[slot, h])
        return {"o": out, "state": S}
    B, T = case["B"], case["T"]
    of = torch.arange(H, device=q.device) // rep
    n = s["lengths"].long() if s["lengths"] is not None else torch.full((B,), T, device=q.device)
    live = (torch.arange(T, device=q.device)[:, None] < n)[:, :, None, None, None]  # [T, B, 1, 1, 1]
    first = s["state"].double() if s["state"] is not None else q.new_zeros(B, H, case["Dk"], case["Dv"])
    train = case["op"] == "attn_train"
    o, S = q.new_zeros(B, T, H, case["Dv"]), first.clone()
    dq = torch.zeros_like(q) if train else None
    do = s["do"].double() if train else None
    for t in range(T):
        S = torch.where(live[t], b * S + k[:, t, of][..., None] * v[:, t, of][:, :, None], S)
        o[:, t] = live[t, ..., 0] * scale * (q[:, t, :, None] @ S)[:, :, 0]
        if train:
            dq[:, t] = live[t, ..., 0] * scale * (S @ do[:, t, :, :, None])[..., 0]
    if not train:
        return {"o": o, "state": S}
    dk, dv, dS = torch.zeros_like(k), torch.zeros_like(v), torch.zeros_like(S)
    for t in reversed(range(T)):
        dS = torch.where(live[t], dS + scale * q[:, t, :, :, None] * do[:, t, :, None], dS)
        gk = live[t, ..., 0] * (dS @ v[:, t, of][..., None])[..., 0]
        gv = live[t, ..., 0] * (k[:, t, of][:, :, None] @ dS)[:, :, 0]
        dk[:, t] = gk.reshape(B, case["Hk"], rep, -1).sum(2)
        dv[:, t] = gv.reshape(B, case["Hk"], rep, -1).sum(2)
        dS = torch.where(live[t], b * dS, dS)
    r = {"o": o, "dq": dq, "dk": dk, "dv": dv}
    return {**r, "dstate": dS} if case["state"] else r


def _exact_norm(case, s):
    x, h, post, pre = (s[k].double() for k in ("x", "h", "post", "pre"))
    D = case["D"]
    rh = 1.0 / torch.sqrt(h.pow(2).sum(-1, keepdim=True) / D + _EPS)
    hh = h * rh
    if s["gate"] is None:
        a = da = None
        y = _RES_SCALE * hh * post
    else:
        g = s["gate"].double()
        sg = torch.sigmoid(g)
        silu = case["act"] == "silu"
        a, da = (g * sg, sg * (1 + g * (1 - sg))) if silu else (sg, sg * (1 - sg))
        y = _RES_SCALE * a * hh * post
    x = x + y
    rx = 1.0 / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / D + _EPS)
    xh = x * rx
    r = {"x": x, "n": xh * pre}
    if case["op"] == "norm":
        return r
    dn = s["dn"].double()
    u = dn * pre
    dx = s["dx"].double() + rx * (u - xh * (u * xh).sum(-1, keepdim=True) / D)
    dy = _RES_SCALE * dx if a is None else _RES_SCALE * a * dx
    w = dy * post
    r.update(dx=dx, dpre=(dn * xh).sum(0), dpost=(dy * hh).sum(0),
             dh=rh * (w - hh * (w * hh).sum(-1, keepdim=True) / D))
    if a is not None:
        dg = _RES_SCALE * dx * hh * post * da
        r["dgate"] = dg if case["gate"] == "full" else dg.sum(-1, keepdim=True)
    return r


def _exact_embed(case, s):
    tok, W = s["tokens"], s["weight"].double()
    scale = math.sqrt(case["D"])
    live = tok >= 0
    y = torch.zeros(case["n"], case["D"], dtype=torch.float64, device=W.device)
    y[live] = W[tok[live]] * scale
    if case["op"] == "embed":
        return {"y": y}
    dW = torch.zeros_like(W)
    dW.index_put_((tok[live],), s["dy"].double()[live] * scale, accumulate=True)
    return {"y": y, "dweight": dW}
