"""The language-model operators whose speed is measured: attention over packed sequences with its
gradient, rotary positions, the norms around a block with their gradient, and the clipping of
gradients by their global norm.

``own`` chooses between the plain form (elementary torch operations in 32 bits, rounded once at the
end) and the framework's calls.  A case is one call (attention's training step: the forward and the
backward call) on device tensors that a program has in hand.

``draw`` spreads over the same ranges: both types, heads of 16 to 128 with odd widths among them,
one to 64 sequences of one to some thousand tokens, shared key heads, rows of 64 to 8192 channels,
one to hundreds of gradient tensors.
"""
import math

import torch

own = False

EPS = 1e-6  # of the norms, and of the clip's quotient
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def _attn(name, mode, dtype, q, k, heads, kv_heads, dim, causal=True, slot=0):
    """q, k: the sequences' lengths; slot: tokens that a cache keeps for each sequence (0: packed)."""
    case = dict(kind="attention", mode=mode, dtype=dtype, q=q, k=k, heads=heads, kv_heads=kv_heads,
                dim=dim, causal=causal, slot=slot)
    return dict(case, name=name) if name else case


def _rotary(name, dtype, tokens, heads, kv_heads, dim, rot, interleaved, inverse, length, factor):
    case = dict(kind="rotary", dtype=dtype, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim,
                rot=rot, interleaved=interleaved, inverse=inverse, length=length, factor=factor)
    return dict(case, name=name) if name else case


def _norm(name, mode, dtype, rows, cols, gate, post, alpha):
    case = dict(kind="norm", mode=mode, dtype=dtype, rows=rows, cols=cols, gate=gate, post=post,
                alpha=alpha)
    return dict(case, name=name) if name else case


def _clip(name, dtype, layers, width, vocab, max_norm):
    case = dict(kind="clip", dtype=dtype, layers=layers, width=width, vocab=vocab,
                max_norm=max_norm)
    return dict(case, name=name) if name else case


def listed():
    return [
        # One request's next token over a short cache: the smallest call, where launches are all.
        _attn("decode_one", "forward", "bf16", "1", "777", 8, 2, 64),
        # Next tokens of 32 requests, each over its part of a long cache of 8192 tokens a slot:
        # bound by reading the cache.
        _attn("decode_batch", "forward", "bf16", ",".join(["1"] * 32),
              ",".join(str(1500 + 6151 * (7 * i % 32) // 31) for i in range(32)), 32, 8, 128,
              slot=8192),
        # Prompts of several requests, some continued after a cached part, in the framework's own
        # type; one request has nothing to compute.
        _attn("prompt_chunks", "forward", "f32", "1,37,513,0,200", "640,37,1025,5,200", 8, 2, 64),
        # One long prompt.
        _attn("prompt_long", "forward", "bf16", "8192", "8192", 16, 4, 128),
        # A training step on documents packed into one batch.
        _attn("train_packed", "train", "bf16", "2711,1024,1777,488", "2711,1024,1777,488", 16, 4,
              128),
        # The same for a small model in float32, with a head width that is no power of two.
        _attn("train_odd", "train", "f32", "129,577,40,301", "129,577,40,301", 6, 3, 80),
        # Rotation of 32 requests' next tokens, far into a context scaled to four times its length.
        _rotary("rotary_decode", "bf16", 32, 32, 8, 128, 128, False, False, 32768, 4.0),
        # The gradient's rotation in a training step: half of each head rotates, in pairs.
        _rotary("rotary_train", "f32", 16384, 16, 4, 128, 64, True, True, 4096, 1.0),
        # Between two blocks of a small model, forward.
        _norm("norm_forward", "forward", "f32", 4096, 2048, "channel", True, 0.7),
        # The gradient there in a larger model's training step, with a gate for every element.
        _norm("norm_backward", "backward", "bf16", 8192, 4096, "element", True, 1.0),
        # Gradients of a small model, as the training step ends.
        _clip("clip_small", "f32", 4, 256, 1001, 1.0),
        # Gradients of a larger one: more than any cache holds.
        _clip("clip_large", "bf16", 16, 2048, 32000, 1.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


MAX_ATTN_FLOPS = 2.7e11   # the long prompt
MAX_ATTN_BYTES = 6e8      # the batch of single tokens
MAX_PADDED = 2e9          # heads * longest query * longest key * sequences: the plain form's scores


def draw(rng):
    kind = rng.choice(["decode", "prompt", "train", "train", "rotary", "norm", "norm", "clip"])
    dtype = rng.choice(["f32", "bf16"])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 8])
    dim = rng.choice([16, 32, 40, 64, 64, 72, 80, 96, 112, 128, 128])
    if kind in ("decode", "prompt", "train"):
        while True:
            n = _log(rng, 1, 64 if kind == "decode" else 12)
            causal, slot = True, 0
            if kind == "decode":
                k = [_log(rng, 1, 9000) for _ in range(n)]
                q = [1] * n
                slot = rng.choice([0, max(k) + rng.randrange(64)])
            else:
                q = [_log(rng, 1, 6000) for _ in range(n)]
                k = list(q)
                if kind == "prompt":
                    causal = rng.random() < 0.8
                    k = [i + rng.choice([0, 0, _log(rng, 1, 3000)]) for i in q]
            case = _attn(None, "train" if kind == "train" else "forward", dtype,
                         ",".join(map(str, q)), ",".join(map(str, k)), heads, kv_heads, dim,
                         causal, slot)
            w = work(case)
            rate = 16 if dtype == "f32" else 1  # float32 products cost that much more
            if (w["flops"] * rate < MAX_ATTN_FLOPS and w["bytes"] < MAX_ATTN_BYTES
                    and n * max(q) * max(k) * heads < MAX_PADDED):
                return case
    if kind == "rotary":
        tokens = _log(rng, 1, 16384)
        rot = rng.choice([dim, dim // 2])
        return _rotary(None, dtype, tokens, min(heads, 16), min(kv_heads, 4), dim, rot,
                       rng.random() < 0.5, rng.random() < 0.5, _log(rng, 64, 65536),
                       rng.choice([1.0, 1.0, 2.0, 8.0]))
    if kind == "norm":
        cols = rng.choice([_log(rng, 64, 8192), 64 * rng.randint(1, 128)])
        rows = _log(rng, 1, 1 << 14)
        rows = min(rows, (1 << 25) // (cols * (2 if dtype == "f32" else 1)))
        return _norm(None, rng.choice(["forward", "backward"]), dtype, rows, cols,
                     rng.choice(["none", "channel", "element"]), rng.random() < 0.7,
                     rng.choice([1.0, 0.5, 0.22]))
    return _clip(None, dtype, _log(rng, 1, 24), _log(rng, 32, 1024), _log(rng, 100, 32000),
                 rng.choice([1.0, 0.1, 1e6]))


def _lens(text):
    return [int(t) for t in text.split(",")]


def _pairs(case):
    """Visible (query, key) pairs of one head."""
    total = 0
    for lq, lk in zip(_lens(case["q"]), _lens(case["k"])):
        if case["causal"]:
            lo, hi = max(0, lk - lq + 1), lk  # of the first and the last row that see a key
            total += (lo + hi) * (hi - lo + 1) // 2 if hi >= lo else 0
        else:
            total += lq * lk
    return total


def _shapes(case):
    w, kv = case["width"], case["width"] // 4 + 1
    shapes = [(case["vocab"], w)]
    for _ in range(case["layers"]):
        shapes += [(w,), (w, w + 2 * kv), (w, w), (w,), (w, 4 * w), (4 * w, w)]
    return shapes + [(w,)]


def work(case):
    b = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "attention":
        nq, nk = sum(_lens(case["q"])), sum(_lens(case["k"]))
        qo, kv = nq * case["heads"] * case["dim"] * b, nk * case["kv_heads"] * case["dim"] * b
        flops = 4 * _pairs(case) * case["heads"] * case["dim"]
        if case["mode"] == "forward":
            return {"bytes": 2 * qo + 2 * kv, "flops": flops}
        # dout as well, and three gradients; five products more
        return {"bytes": 4 * qo + 4 * kv, "flops": flops * 7 // 2}
    if case["kind"] == "rotary":
        n = case["tokens"] * (case["heads"] + case["kv_heads"])
        table = min(case["tokens"], case["length"]) * case["rot"] * 4
        return {"bytes": 2 * n * case["dim"] * b + table + 4 * case["tokens"],
                "flops": 3 * n * case["rot"]}
    if case["kind"] == "norm":
        n = case["rows"] * case["cols"]
        gate = {"none": 0, "channel": case["cols"], "element": n}[case["gate"]]
        if case["mode"] == "forward":
            return {"bytes": (4 * n + gate) * b, "flops": 10 * n}
        return {"bytes": (6 * n + 2 * gate) * b, "flops": 24 * n}
    n = sum(math.prod(s) for s in _shapes(case))
    return {"bytes": 2 * n * b, "flops": 3 * n}


def _starts(lens, dev):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return torch.tensor(out, dtype=torch.int32, device=dev)


def _table(length, rot, factor, dev):
    """cos and sin [length, rot] of the positions' angles, as a program keeps them: wavelengths that
    fit 1/32 of the context stay, those beyond it are stretched by the factor, those between are mixed."""
    i = torch.arange(0, rot, 2, dtype=torch.float64, device=dev)
    freq = 10000.0 ** (-i / rot)
    amp = 1.0
    if factor != 1.0:
        turns = length / factor * freq / (2 * math.pi)
        keep = ((turns - 1.0) / 31.0).clamp(0, 1)
        freq = freq * (keep + (1 - keep) / factor)
        amp = 0.1 * math.log(factor) + 1.0
    angle = torch.arange(length, dtype=torch.float64, device=dev)[:, None] * freq
    return (torch.cat([angle.cos(), angle.sin()], 1) * amp).float()


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0, dtype=dt):
        t = torch.empty(shape, dtype=torch.float32 if math.prod(shape) < 1 << 28 else dtype,
                        device=dev)
        return t.normal_(mean, std, generator=gen).to(dtype)

    s = dict(case)
    if case["kind"] == "attention":
        q, k = _lens(case["q"]), _lens(case["k"])
        slot = case["slot"]
        nk = slot * len(k) if slot else sum(k)
        s["qlens"], s["klens"] = q, k
        s["cu_q"] = _starts(q, dev)
        s["cu_k"] = _starts([slot] * len(k) if slot else k, dev)
        s["k_lens"] = torch.tensor(k, dtype=torch.int32, device=dev) if slot else None
        # Scores of standard deviation 1.5: attention that prefers some keys.
        s["q"] = normal(sum(q), case["heads"], case["dim"], std=1.5)
        s["k"] = normal(nk, case["kv_heads"], case["dim"])
        s["v"] = normal(nk, case["kv_heads"], case["dim"])
        if case["mode"] == "train":
            s["dout"] = normal(sum(q), case["heads"], case["dim"], std=0.1)
    elif case["kind"] == "rotary":
        s["q"] = normal(case["tokens"], case["heads"], case["dim"])
        s["k"] = normal(case["tokens"], case["kv_heads"], case["dim"])
        s["table"] = _table(case["length"], case["rot"], case["factor"], dev)
        s["positions"] = torch.randint(0, case["length"], (case["tokens"],), dtype=torch.int32,
                                       device=dev, generator=gen)
    elif case["kind"] == "norm":
        shape = (case["rows"], case["cols"])
        s["o"] = normal(*shape, std=0.5)
        s["w_pre"] = normal(case["cols"], mean=1.0, std=0.1)
        s["w_post"] = normal(case["cols"], mean=1.0, std=0.1) if case["post"] else None
        gates = {"none": None, "channel": shape[1:], "element": shape}[case["gate"]]
        s["gate"] = normal(*gates, mean=0.5, std=0.3) if gates else None
        if case["mode"] == "forward":
            s["x"] = normal(*shape, std=2.0)
        else:  # what the forward call left: its output y, and the rows' 1/rms of o and y
            s["y"] = normal(*shape, std=2.0)
            s["dy"], s["dh"] = normal(*shape, std=0.1), normal(*shape, std=0.1)
            s["stats"] = torch.stack([(t.double().square().mean(1) + EPS).rsqrt().float()
                                      for t in (s["o"], s["y"])])
    else:
        shapes = _shapes(case)
        s["grads"] = [normal(*t, std=1e-3) for t in shapes]
        sizes = [math.prod(t) for t in shapes]
        s["flat"] = torch.empty(sum(sizes), dtype=dt, device=dev)  # where the clipped ones go
        s["outs"] = [t.view(shape) for t, shape in zip(s["flat"].split(sizes), shapes)]
    return s


# ---- the plain forms ----

def _padded(cu, lens, most):
    """Token numbers [sequences, most] of packed sequences, and which of them exist."""
    j = torch.arange(most, device=cu.device)
    real = j < lens[:, None]
    return torch.where(real, cu[:-1, None] + j, 0), real


def _plain_attention(s):
    heads, kv, dim = s["heads"], s["kv_heads"], s["dim"]
    group, dt = heads // kv, s["q"].dtype
    n, lq, lk = len(s["qlens"]), max(s["qlens"]), max(s["klens"])
    cu_q = s["cu_q"].long()
    qlens = cu_q.diff()
    klens = s["k_lens"].long() if s["slot"] else s["cu_k"].long().diff()
    iq, real_q = _padded(cu_q, qlens, lq)
    ik, real_k = _padded(s["cu_k"].long(), klens, lk)
    seen = (real_q[:, :, None] & real_k[:, None, :])[:, None, None]
    if s["causal"]:
        last = torch.arange(lq, device=cu_q.device) + (klens - qlens)[:, None]
        seen = seen & (torch.arange(lk, device=cu_q.device) <= last[:, :, None])[:, None, None]

    def rows(t):   # [tokens, heads, dim] -> [sequences, key heads, group * lq, dim]
        t = t.float()[iq].view(n, lq, kv, group, dim)
        return t.permute(0, 2, 3, 1, 4).reshape(n, kv, group * lq, dim)

    def keys(t):
        return t.float()[ik].transpose(1, 2).contiguous()

    def packed(t, cu, idx_len, total):  # the padded rows' values at the packed tokens
        tok = torch.arange(total, device=cu.device)
        seq = torch.searchsorted(cu, tok, right=True) - 1
        return t.reshape((n * idx_len,) + t.shape[2:])[seq * idx_len + tok - cu[seq]]

    def unrows(t):
        t = t.view(n, kv, group, lq, dim).permute(0, 3, 1, 2, 4).reshape(n, lq, heads, dim)
        return packed(t, cu_q, lq, s["q"].shape[0]).to(dt)

    scale = dim ** -0.5
    q, k, v = rows(s["q"]), keys(s["k"]), keys(s["v"])
    x = (q @ k.transpose(2, 3) * scale).view(n, kv, group, lq, lk)
    x = x.masked_fill(~seen, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = (x - top.masked_fill(top == -math.inf, 0.0)).exp()
    total = p.sum(-1, keepdim=True)
    p = (p / total.masked_fill(total == 0, 1.0)).view(n, kv, group * lq, lk)
    o = p @ v
    if s["mode"] == "forward":
        return {"out": unrows(o)}
    do = rows(s["dout"])
    dp = do @ v.transpose(2, 3)
    ds = p * (dp - (do * o).sum(-1, keepdim=True)) * scale
    cu_k = s["cu_k"].long()

    def unkeys(t):
        return packed(t.transpose(1, 2), cu_k, lk, s["k"].shape[0]).to(dt)

    return {"out": unrows(o), "dq": unrows(ds @ k), "dk": unkeys(ds.transpose(2, 3) @ q),
            "dv": unkeys(p.transpose(2, 3) @ do)}


def _plain_rotate(t, s):
    rot, half = s["rot"], s["rot"] // 2
    cos, sin = s["table"][s["positions"].long()][:, None].split(half, -1)
    sin = -sin if s["inverse"] else sin
    x = t.float()
    if s["interleaved"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:rot]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([turned, x[..., rot:]], -1).to(t.dtype)


def _plain_norm(s):
    dt = s["o"].dtype
    o, w_pre, alpha = s["o"].float(), s["w_pre"].float(), s["alpha"]
    w_post = s["w_post"].float() if s["post"] else None
    gate = s["gate"].float() if s["gate"] is not None else None
    if s["mode"] == "forward":
        b = o * (o.square().mean(1, keepdim=True) + EPS).rsqrt() * w_post if s["post"] else o
        b = b * gate if gate is not None else b
        y = s["x"].float() + alpha * b
        h = y * (y.square().mean(1, keepdim=True) + EPS).rsqrt() * w_pre
        return {"y": y.to(dt), "h": h.to(dt)}
    r_o, r_y = s["stats"][:, :, None]
    dh = s["dh"].float()
    yn, gw = s["y"].float() * r_y, dh * w_pre
    gy = s["dy"].float() + r_y * (gw - yn * (gw * yn).mean(1, keepdim=True))
    out = {"dx": gy.to(dt), "dw_pre": (dh * yn).sum(0).to(dt)}
    on = o * r_o if s["post"] else o
    if gate is not None:
        dg = alpha * gy * (on * w_post if s["post"] else on)
        out["dgate"] = (dg.sum(0) if gate.dim() == 1 else dg).to(dt)
    db = alpha * gy * gate if gate is not None else alpha * gy
    if s["post"]:
        out["dw_post"] = (db * on).sum(0).to(dt)
        gw = db * w_post
        db = r_o * (gw - on * (gw * on).mean(1, keepdim=True))
    out["do"] = db.to(dt)
    return out


def _plain_clip(s):
    norm = torch.stack([g.float().square().sum() for g in s["grads"]]).sum().sqrt()
    coef = (s["max_norm"] / (norm + EPS)).clamp(max=1.0)
    flat = torch.cat([g.reshape(-1) for g in s["grads"]])
    s["flat"].copy_(flat.float() * coef)
    return {"norm": norm.view(1), "grads": s["flat"]}


# ---- the framework's calls ----

def _own(s):
    from katsu_amd import ops
    if s["kind"] == "attention":
        out, lse = ops.attention(s["q"], s["k"], s["v"], cu_q=s["cu_q"], cu_k=s["cu_k"],
                                 k_lens=s["k_lens"], causal=s["causal"])
        if s["mode"] == "forward":
            return {"out": out}
        dq, dk, dv = ops.attention_backward(s["dout"], s["q"], s["k"], s["v"], out, lse,
                                            cu_q=s["cu_q"], cu_k=s["cu_k"], causal=s["causal"])
        return {"out": out, "dq": dq, "dk": dk, "dv": dv}
    if s["kind"] == "rotary":
        q, k = ops.rotary(s["q"], s["k"], s["table"], s["positions"],
                          interleaved=s["interleaved"], inverse=s["inverse"])
        return {"q": q, "k": k}
    if s["kind"] == "norm":
        if s["mode"] == "forward":
            y, h, _ = ops.block_norm(s["x"], s["o"], gate=s["gate"], w_post=s["w_post"],
                                     w_pre=s["w_pre"], alpha=s["alpha"], eps=EPS)
            return {"y": y, "h": h}
        dx, do, dgate, dw_post, dw_pre = ops.block_norm_backward(
            s["dy"], s["dh"], s["y"], s["o"], s["stats"], gate=s["gate"], w_post=s["w_post"],
            w_pre=s["w_pre"], alpha=s["alpha"])
        return {"dx": dx, "do": do, "dgate": dgate, "dw_post": dw_post, "dw_pre": dw_pre}
    norm = ops.clip_grad_norm(s["grads"], s["max_norm"], out=s["outs"])
    return {"norm": norm, "grads": s["flat"]}


def run(state):
    if own:
        return _own(state)
    if state["kind"] == "attention":
        return _plain_attention(state)
    if state["kind"] == "rotary":
        return {"q": _plain_rotate(state["q"], state), "k": _plain_rotate(state["k"], state)}
    return _plain_norm(state) if state["kind"] == "norm" else _plain_clip(state)


# ---- from the definitions, in 64 bits ----

def _exact_attention(s):
    train = s["mode"] == "train"
    group, scale = s["heads"] // s["kv_heads"], 1.0 / math.sqrt(s["dim"])
    new = {"out": torch.zeros_like(s["q"], dtype=torch.float64)}
    if train:
        new.update({"d" + t: torch.zeros_like(s[t], dtype=torch.float64) for t in "qkv"})
    qa = ka = 0
    for lq, lk in zip(s["qlens"], s["klens"]):
        for h in range(s["heads"]):
            at_q, at_k = (slice(qa, qa + lq), h), (slice(ka, ka + lk), h // group)
            q, k, v = s["q"][at_q].double(), s["k"][at_k].double(), s["v"][at_k].double()
            x = torch.mm(q, k.t()) * scale
            if s["causal"]:
                x += torch.full_like(x, -math.inf).triu(lk - lq + 1)
            p = x.softmax(1).nan_to_num(0.0) if lk else x
            new["out"][at_q] = torch.mm(p, v)
            if train:
                g = s["dout"][at_q].double()
                dp = torch.mm(g, v.t())
                dx = p * (dp - (p * dp).sum(1, keepdim=True)) * scale
                new["dq"][at_q] = torch.mm(dx, k)
                new["dk"][at_k] += torch.mm(dx.t(), q)
                new["dv"][at_k] += torch.mm(p.t(), g)
        qa, ka = qa + lq, ka + (s["slot"] or lk)
    return new


def _exact_rotary(t, s):
    half = s["rot"] // 2
    table = s["table"].double()[s["positions"].long()]
    turn = torch.complex(table[:, :half], table[:, half:])[:, None]
    turn = turn.conj() if s["inverse"] else turn
    x = t.double()
    pairs = (x[..., :s["rot"]].unflatten(-1, (half, 2)) if s["interleaved"]
             else x[..., :s["rot"]].unflatten(-1, (2, half)).transpose(-1, -2))
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    x[..., :s["rot"]] = (z if s["interleaved"] else z.transpose(-1, -2)).flatten(-2)
    return x


def _exact_norm(s):
    wide = {k: t.double() for k, t in s.items() if isinstance(t, torch.Tensor)}
    one = torch.ones((), dtype=torch.float64, device=s["o"].device)
    gate, w_post, w_pre = (wide.get(k, one) for k in ("gate", "w_post", "w_pre"))

    if s["mode"] == "forward":
        def rms(t):
            return (t.square().sum(-1, keepdim=True) / t.shape[-1] + EPS).sqrt()
        o = wide["o"]
        y = wide["x"] + s["alpha"] * gate * (o / rms(o) * w_post if s["post"] else o)
        return {"y": y, "h": y / rms(y) * w_pre}

    # The given 1/rms r is a function of its row: dr/dt_i = -r^3 t_i / C.
    def back(g, t, r):
        c = t.shape[-1]
        return r * g - r ** 3 * t * ((g * t).sum(-1, keepdim=True) / c)

    r_o, r_y = wide["stats"][0][:, None], wide["stats"][1][:, None]
    o, y, dh = wide["o"], wide["y"], wide["dh"]
    dx = wide["dy"] + back(dh * w_pre, y, r_y)
    branch = o * r_o * w_post if s["post"] else o
    out = {"dx": dx, "dw_pre": (dh * y * r_y).sum(0)}
    dg = s["alpha"] * dx * branch
    if s["gate"] is not None:
        out["dgate"] = dg.sum(0) if s["gate"].dim() == 1 else dg
    db = s["alpha"] * dx * gate
    if s["post"]:
        out["dw_post"] = (db * o * r_o).sum(0)
    out["do"] = back(db * w_post, o, r_o) if s["post"] else db
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "attention":
        return _exact_attention(s)
    if case["kind"] == "rotary":
        return {"q": _exact_rotary(s["q"], s), "k": _exact_rotary(s["k"], s)}
    if case["kind"] == "norm":
        return _exact_norm(s)
    total = math.fsum(float((g.double() ** 2).sum()) for g in s["grads"])
    coef = min(1.0, case["max_norm"] / (math.sqrt(total) + EPS))
    return {"norm": torch.tensor([math.sqrt(total)], dtype=torch.float64, device="cuda"),
            "grads": torch.cat([(g.double() * coef).reshape(-1) for g in s["grads"]])}
