"""The operators at the two ends of a language model's training step and before its attention, whose
speed is measured: embedding with its gradient, the norm of each query and key head with the position
rotation, with its gradient, and the loss against a teacher's top logits with its gradient.

``own`` chooses between the plain form (elementary torch operations in 32 bits, rounded once at the
end) and the framework's calls.  A case is one call on device tensors that a program has in hand.

``draw`` spreads over the same ranges: both types, one to some ten thousand tokens, vocabularies of a
hundred to over a hundred thousand with odd ones among them, rows of 32 to 4096 channels, heads of 16
to 256 with odd widths, one to 256 of the teacher's logits.
"""
import math

import torch

own = False

EPS = 1e-6  # of the heads' norms
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def _embed(name, mode, dtype, tokens, vocab, cols, scale, pad):
    """pad: the share of tokens that are padding, ids of -1."""
    case = dict(kind="embed", mode=mode, dtype=dtype, tokens=tokens, vocab=vocab, cols=cols,
                scale=scale, pad=pad)
    return dict(case, name=name) if name else case


def _heads(name, mode, dtype, tokens, heads, kv_heads, dim, rot, interleaved, length):
    case = dict(kind="heads", mode=mode, dtype=dtype, tokens=tokens, heads=heads,
                kv_heads=kv_heads, dim=dim, rot=rot, interleaved=interleaved, length=length)
    return dict(case, name=name) if name else case


def _distill(name, mode, dtype, rows, vocab, top, tau):
    case = dict(kind="distill", mode=mode, dtype=dtype, rows=rows, vocab=vocab, top=top, tau=tau)
    return dict(case, name=name) if name else case


def listed():
    return [
        # The next tokens of 32 requests: the smallest call, where launches are all.
        _embed("embed_next", "forward", "bf16", 32, 32000, 2048, 1.0, 0.0),
        # A training batch's tokens, scaled by the root of the width.
        _embed("embed_batch", "forward", "f32", 16384, 32000, 2048, 45.25, 0.03),
        # The gradient in a small model's step, documents of some 250 tokens in all.
        _embed("embed_grad_small", "backward", "f32", 252, 1001, 256, 16.0, 0.0),
        # The gradient in a larger model's step: words as frequent as in text, the batch padded.
        _embed("embed_grad", "backward", "bf16", 16384, 32000, 2048, 45.25, 0.03),
        # The next tokens of 32 requests, far into their contexts.
        _heads("heads_next", "forward", "bf16", 32, 32, 8, 128, 128, False, 32768),
        # One long prompt.
        _heads("heads_prompt", "forward", "bf16", 8192, 16, 4, 128, 128, False, 8192),
        # A training step on 6000 packed tokens.
        _heads("heads_grad", "backward", "bf16", 6000, 16, 4, 128, 128, False, 4096),
        # The same for a small model in float32: an odd width, half of which turns, in pairs.
        _heads("heads_grad_odd", "backward", "f32", 1047, 6, 3, 80, 40, True, 1024),
        # Loss and gradient in a small model's step.
        _distill("distill_small", "step", "f32", 252, 1001, 8, 1.0),
        # The loss alone, on tokens held out.
        _distill("distill_eval", "forward", "bf16", 4096, 32000, 64, 1.0),
        # The gradient of a loss that something else weighed; a vocabulary of odd size, in float32.
        _distill("distill_grad", "backward", "f32", 1000, 32001, 100, 2.0),
        # Loss and gradient in a larger model's step: more logits than any cache holds.
        _distill("distill_step", "step", "bf16", 8192, 32000, 32, 2.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


MAX_BYTES = 1 << 30  # of the largest listed case


def draw(rng):
    kind = rng.choice(["embed", "heads", "distill"])
    dtype = rng.choice(["f32", "bf16"])
    while True:
        if kind == "embed":
            case = _embed(None, rng.choice(["forward", "backward"]), dtype, _log(rng, 1, 32768),
                          _log(rng, 100, 130000), _log(rng, 32, 4096),
                          rng.choice([1.0, 11.3, 64.0]), rng.choice([0.0, 0.1, 0.5]))
            fits = case["vocab"] * case["cols"] < 1 << 27
        elif kind == "heads":
            kv = rng.choice([1, 2, 3, 4, 8])
            dim = rng.choice([16, 40, 64, 64, 72, 80, 96, 112, 128, 128, 256])
            case = _heads(None, rng.choice(["forward", "backward", "backward"]), dtype,
                          _log(rng, 1, 16384), kv * rng.choice([1, 2, 3, 4, 5, 8]), kv, dim,
                          rng.choice([dim, dim // 2]), rng.random() < 0.4, _log(rng, 64, 65536))
            fits = True
        else:
            vocab = _log(rng, 100, 130000)
            case = _distill(None, rng.choice(["forward", "backward", "step", "step"]), dtype,
                            _log(rng, 1, 8192), vocab, min(_log(rng, 1, 256), vocab // 2),
                            rng.choice([0.5, 1.0, 1.0, 2.0, 4.0]))
            fits = True
        w = work(case)
        if fits and w["bytes"] * (1 if dtype == "bf16" else 2) < MAX_BYTES:
            return case


def work(case):
    b = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "embed":
        n = case["tokens"] * case["cols"]
        if case["mode"] == "forward":  # no row of the table more than once
            rows = min(case["tokens"], case["vocab"])
            return {"bytes": (n + rows * case["cols"]) * b + 4 * case["tokens"], "flops": n}
        return {"bytes": (n + case["vocab"] * case["cols"]) * b + 4 * case["tokens"],
                "flops": n + case["vocab"] * case["cols"]}
    if case["kind"] == "heads":
        n = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        table = min(case["tokens"], case["length"]) * case["rot"] * 4 + 4 * case["tokens"]
        if case["mode"] == "forward":
            return {"bytes": 2 * n * b + table, "flops": 8 * n}
        return {"bytes": 3 * n * b + table, "flops": 16 * n}
    n = (case["rows"] - case["rows"] // 16) * case["vocab"]  # padding rows' logits say nothing
    side = case["rows"] * (case["top"] * (4 + b) + 12)
    out = 0 if case["mode"] == "forward" else case["rows"] * case["vocab"]
    return {"bytes": (n + out) * b + side,
            "flops": n * (4 if case["mode"] == "forward" else 7)}


def _table(length, rot, dev):
    """cos and sin [length, rot] of the positions' angles, as a program keeps them."""
    freq = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=dev) / rot)
    angle = torch.arange(length, dtype=torch.float64, device=dev)[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0):
        return torch.empty(shape, device=dev).normal_(mean, std, generator=gen).to(dt)

    s = dict(case)
    if case["kind"] == "embed":
        n, vocab = case["tokens"], case["vocab"]
        # As frequent as words: the i-th has a share of about 1 / (i + 1), in an order of its own.
        u = torch.rand(n, device=dev, generator=gen, dtype=torch.float64)
        rank = ((vocab + 1.0) ** u - 1.0).long().clamp(0, vocab - 1)
        ids = torch.randperm(vocab, device=dev, generator=gen)[rank]
        pad = torch.rand(n, device=dev, generator=gen) < case["pad"]
        s["ids"] = torch.where(pad, -1, ids).int()
        if case["mode"] == "forward":
            s["table"] = normal(vocab, case["cols"], std=0.02)
        else:
            s["dout"] = normal(n, case["cols"], std=0.1)
    elif case["kind"] == "heads":
        h, kv, dim = case["heads"], case["kv_heads"], case["dim"]
        # q and k are parts of one projection, beside the values.
        qkv = normal(case["tokens"], h + 2 * kv, dim, std=1.7)
        s["q"], s["k"] = qkv[:, :h], qkv[:, h:h + kv]
        s["w_q"], s["w_k"] = normal(dim, mean=1.0, std=0.2), normal(dim, mean=1.0, std=0.2)
        s["table"] = _table(case["length"], case["rot"], dev)
        s["positions"] = torch.randint(0, case["length"], (case["tokens"],), dtype=torch.int32,
                                       device=dev, generator=gen)
        if case["mode"] == "backward":
            s["dq"] = normal(case["tokens"], h, dim, std=0.1)
            s["dk"] = normal(case["tokens"], kv, dim, std=0.1)
    else:
        rows, vocab, top = case["rows"], case["vocab"], case["top"]
        z = s["logits"] = torch.empty((rows, vocab), dtype=dt, device=dev)
        s["ids"] = torch.empty((rows, top), dtype=torch.int32, device=dev)
        s["teacher"] = torch.empty((rows, top), dtype=dt, device=dev)
        # What the forward call left: each row's largest logit, and one over its total.
        s["stats"] = torch.empty((2, rows), device=dev)
        for at in range(0, rows, 512):
            part = slice(at, min(at + 512, rows))
            z[part] = normal(part.stop - at, vocab, std=2.5)
            wide = z[part].float()
            # The teacher agrees with the model by and large.
            best = (wide + torch.randn(wide.shape, device=dev, generator=gen)).topk(top, dim=1)
            s["teacher"][part], s["ids"][part] = best.values.to(dt), best.indices.int()
            m = wide.amax(1)
            s["stats"][0, part] = m
            total = ((wide - m[:, None]).double() / case["tau"]).exp().sum(1)
            s["stats"][1, part] = (1.0 / total).float()
        # The last rows are padding: the teacher says nothing there.
        s["ids"][rows - rows // 16:] = -1
        s["dloss"] = torch.full((rows,), 1.0 / rows, device=dev)
    return s


# ---- the plain forms ----

def _plain_embed(s):
    real = s["ids"] >= 0
    ids = s["ids"].long().clamp(min=0)
    if s["mode"] == "forward":
        out = s["table"][ids].float() * s["scale"]
        return {"out": out.masked_fill(~real[:, None], 0.0).to(s["table"].dtype)}
    total = torch.zeros((s["vocab"], s["cols"]), device=ids.device)
    total.index_add_(0, ids, s["dout"].float().masked_fill(~real[:, None], 0.0))
    return {"dtable": (total * s["scale"]).to(s["dout"].dtype)}


def _plain_turn(x, s, sign):
    rot, half = s["rot"], s["rot"] // 2
    cos, sin = s["table"][s["positions"].long()][:, None].split(half, -1)
    sin = sin * sign
    if s["interleaved"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:rot]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _plain_heads(x, w, dy, s):
    wide, w = x.float(), w.float()
    r = (wide.square().mean(-1, keepdim=True) + EPS).rsqrt()
    n = wide * r
    if dy is None:
        return _plain_turn(n * w, s, 1.0).to(x.dtype)
    g = _plain_turn(dy.float(), s, -1.0)
    dw = (g * n).sum((0, 1))
    g = g * w
    return (r * (g - n * (g * n).mean(-1, keepdim=True))).to(x.dtype), dw.to(x.dtype)


def _plain_distill(s):
    tau, z = s["tau"], s["logits"].float()
    real = s["ids"] >= 0
    ids = s["ids"].long().clamp(min=0)
    some = real.any(1)
    t = (s["teacher"].float() / tau).masked_fill(~real, -math.inf)
    t = (t - t.amax(1, keepdim=True)).masked_fill(~some[:, None], 0.0)
    p = t.exp().masked_fill(~real, 0.0)
    total = p.sum(1, keepdim=True).masked_fill(~some[:, None], 1.0)
    p = p / total
    if s["mode"] == "backward":
        m, inv = s["stats"][0][:, None], s["stats"][1][:, None]
        e = ((z - m) / tau).exp()
    else:
        m = z.amax(1, keepdim=True)
        e = ((z - m) / tau).exp()
        student = e.sum(1, keepdim=True)
        inv = 1.0 / student
        log_s = (z.gather(1, ids) - m) / tau - student.log()
        log_p = (t - total.log()).masked_fill(~real, 0.0)
        out = {"loss": tau * tau * (p * (log_p - log_s)).sum(1)}
        if s["mode"] == "forward":
            return dict(out, largest=m[:, 0].masked_fill(~some, 0.0),
                        inverse=inv[:, 0].masked_fill(~some, 0.0))
    e = (e * inv).masked_fill(~some[:, None], 0.0)
    e.scatter_add_(1, ids, -p)
    dz = (e * (tau * s["dloss"])[:, None]).to(s["logits"].dtype)
    return {"dlogits": dz} if s["mode"] == "backward" else dict(out, dlogits=dz)


# ---- the framework's calls ----

def _own(s):
    from katsu_amd import ops
    if s["kind"] == "embed":
        if s["mode"] == "forward":
            return {"out": ops.embedding(s["ids"], s["table"], scale=s["scale"])}
        return {"dtable": ops.embedding_backward(s["dout"], s["ids"], s["vocab"],
                                                 scale=s["scale"])}
    if s["kind"] == "heads":
        how = dict(w_q=s["w_q"], w_k=s["w_k"], eps=EPS, interleaved=s["interleaved"])
        if s["mode"] == "forward":
            q, k = ops.qk_norm_rotary(s["q"], s["k"], s["table"], s["positions"], **how)
            return {"q": q, "k": k}
        dq, dk, dw_q, dw_k = ops.qk_norm_rotary_backward(s["dq"], s["dk"], s["q"], s["k"],
                                                         s["table"], s["positions"], **how)
        return {"dq": dq, "dk": dk, "dw_q": dw_q, "dw_k": dw_k}
    z, ids, teacher, tau = s["logits"], s["ids"], s["teacher"], s["tau"]
    if s["mode"] == "forward":
        loss, stats = ops.distillation(z, ids, teacher, temperature=tau)
        return {"loss": loss, "largest": stats[0], "inverse": stats[1]}
    if s["mode"] == "backward":
        return {"dlogits": ops.distillation_backward(s["dloss"], z, ids, teacher, s["stats"],
                                                     temperature=tau)}
    loss, dz = ops.distillation_step(z, ids, teacher, s["dloss"], temperature=tau)
    return {"loss": loss, "dlogits": dz}


def run(state):
    if own:
        return _own(state)
    if state["kind"] == "embed":
        return _plain_embed(state)
    if state["kind"] == "distill":
        return _plain_distill(state)
    if state["mode"] == "forward":
        return {t: _plain_heads(state[t], state["w_" + t], None, state) for t in "qk"}
    out = {}
    for t in "qk":
        out["d" + t], out["dw_" + t] = _plain_heads(state[t], state["w_" + t], state["d" + t],
                                                    state)
    return {key: out[key] for key in ("dq", "dk", "dw_q", "dw_k")}


# ---- from the definitions, in 64 bits ----

def _exact_embed(s):
    ids = s["ids"].long()
    at = torch.nonzero(ids >= 0).squeeze(1)
    if s["mode"] == "forward":
        out = torch.zeros((s["tokens"], s["cols"]), dtype=torch.float64, device=ids.device)
        out[at] = s["table"][ids[at]].double() * s["scale"]
        return {"out": out}
    out = torch.zeros((s["vocab"], s["cols"]), dtype=torch.float64, device=ids.device)
    out.index_put_((ids[at],), s["dout"][at].double() * s["scale"], accumulate=True)
    return {"dtable": out}


def _exact_heads(x, w, dy, s):
    rot, half = s["rot"], s["rot"] // 2
    angles = s["table"].double()[s["positions"].long()][:, None]
    turn = torch.complex(angles[..., :half].contiguous(), angles[..., half:].contiguous())

    def turned(t, by):
        pairs = (t[..., :rot].unflatten(-1, (half, 2)) if s["interleaved"]
                 else t[..., :rot].unflatten(-1, (2, half)).transpose(-1, -2))
        u = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * by)
        u = (u if s["interleaved"] else u.transpose(-1, -2)).flatten(-2)
        return torch.cat((u, t[..., rot:]), -1)

    x, w = x.double(), w.double()
    rms = (x.pow(2).sum(-1, keepdim=True) / s["dim"] + EPS).sqrt()
    if dy is None:
        return turned(x / rms * w, turn)
    g = turned(dy.double(), turn.conj())
    # d(1/rms)/dx_i = -x_i / (D rms^3)
    dx = g * w / rms - x * ((g * w * x).sum(-1, keepdim=True) / (s["dim"] * rms.pow(3)))
    return dx, (g * x / rms).flatten(0, 1).sum(0)


def _exact_distill(s):
    rows, tau = s["rows"], s["tau"]
    dev, parts = s["ids"].device, []
    for at in range(0, rows, 256):
        part = slice(at, min(at + 256, rows))
        z, ids = s["logits"][part].double(), s["ids"][part].long()
        real = (ids >= 0) & (ids < s["vocab"])
        some = real.any(1)
        log_p = (s["teacher"][part].double() / tau).masked_fill(~real, -math.inf)
        log_p = (log_p - torch.logsumexp(log_p, 1, keepdim=True)).masked_fill(~real, 0.0)
        p = log_p.exp() * real
        log_all = (z / tau).log_softmax(1)
        loss = (p * (log_p - log_all.gather(1, ids.clamp(min=0)))).sum(1) * tau ** 2
        if s["mode"] == "backward":  # with the statistics that are given
            m, inv = s["stats"].double()[:, part, None]
            all_p = ((z - m) / tau).exp() * inv
        else:
            all_p = log_all.exp()
        want = torch.zeros_like(z)
        row = torch.arange(len(z), device=dev)[:, None].expand_as(ids)
        want.index_put_((row[real], ids[real]), p[real], accumulate=True)
        dz = (all_p - want) * some[:, None] * (tau * s["dloss"][part].double())[:, None]
        parts.append((loss, dz, z.amax(1) * some, log_all.amax(1).exp() * some))
    out = {"loss": torch.cat([v[0] for v in parts])}
    if s["mode"] == "forward":
        out["largest"], out["inverse"] = (torch.cat([v[i] for v in parts]) for i in (2, 3))
    else:
        out["dlogits"] = torch.cat([v[1] for v in parts])
        if s["mode"] == "backward":
            del out["loss"]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "embed":
        return _exact_embed(s)
    if case["kind"] == "distill":
        return _exact_distill(s)
    if case["mode"] == "forward":
        return {t: _exact_heads(s[t], s["w_" + t], None, s) for t in "qk"}
    (dq, dw_q), (dk, dw_k) = (_exact_heads(s[t], s["w_" + t], s["d" + t], s) for t in "qk")
    return {"dq": dq, "dk": dk, "dw_q": dw_q, "dw_k": dw_k}
