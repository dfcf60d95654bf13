"""The operators of a token model around the recurrent layers, as measurable cases.

A token model feeds token ids through an embedding table into a stack of recurrent layers, each between two norms and a
residual connection, multiplies the result with an output matrix and scores it against the next tokens.  Kinds of case:

  embed_fwd     rows of the table by token id, scaled
  embed_bwd     gradient of the table, overwritten: for each token the sum over the frames that hold it
  logprob_fwd   log probability of one given token per row of logits; entropy and the most likely tokens where asked for
  logprob_bwd   gradient of those log probabilities (and of the entropy) with respect to the logits
  clip          the norm over all gradients of a model, and the gradients scaled down to a largest norm
  norm_fwd      y = x + a * gate * norm(f) and h = norm(y): the end of one residual block and the start of the next
  norm_bwd      the gradients of that

Rows are the frames of a fraction, time-major with the parallel sequences interleaved; padding frames have the token -1.
"""
import math
import os
import random
import sys

import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # one new token for each of 64 running sequences: launch and host work count
        dict(name="embed step 64x512", kind="embed_fwd", rows=64, vocab=32000, dim=512, table="f32", out="f32", pad=0.0),
        # two utterances of quantised targets, as the example log has them: a small table that every frame hits often
        dict(name="embed grad 1516x259x128", kind="embed_bwd", rows=1516, vocab=259, dim=128, grad="f32", out="f32", pad=0.05),
        # a training batch of text: few frequent tokens, a long tail, most of the table without a frame
        dict(name="embed grad 32768x50000x1024", kind="embed_bwd", rows=32768, vocab=50000, dim=1024, grad="bf16", out="f32", pad=0.03),
        # sampling for eight sequences, some tokens ruled out for all
        dict(name="logprob step 8x131072 top8", kind="logprob_fwd", rows=8, vocab=131072, ld=131072, type="bf16", top=8, entropy=True,
             mask="shared", scale=1.25, pad=0.0),
        # a fraction of 32 utterances scored over quantised amplitude classes; odd width, fp32 as the layers write it
        dict(name="logprob 38400x259", kind="logprob_fwd", rows=38400, vocab=259, ld=259, type="f32", top=0, entropy=True, mask="none",
             scale=1.0, pad=0.35),
        # scoring a training batch over a large vocabulary, with alternatives
        dict(name="logprob 8192x50001 top4", kind="logprob_fwd", rows=8192, vocab=50001, ld=50048, type="bf16", top=4, entropy=True,
             mask="none", scale=1.0, pad=0.03),
        # the gradient of such a batch; rows that start anywhere
        dict(name="logprob grad 8192x32003", kind="logprob_bwd", rows=8192, vocab=32003, ld=32003, type="bf16", dentropy=True, mask="none",
             scale=1.0, pad=0.03),
        # the weights of the acoustic model (feed-forward 382-512-512, two blstm layers of 256 units per direction, 187 outputs)
        dict(name="clip acoustic 5", kind="clip", sizes="acoustic", over=True),
        # many tensors of all sizes, two types
        dict(name="clip 240 tensors", kind="clip", sizes="many", tensors=240, total=260_000_000, over=True),
        # one new token for each of 64 sequences
        dict(name="norm step 64x1024", kind="norm_fwd", rows=64, dim=1024, type="bf16", ln=False, gate_rows=1, pad=0.0),
        # a fraction of 32 sequences, a gate for each sequence
        dict(name="norm 38400x512", kind="norm_fwd", rows=38400, dim=512, type="f32", ln=True, gate_rows=32, pad=0.35),
        # a training batch backwards, a gate for each frame
        dict(name="norm grad 16384x2048", kind="norm_bwd", rows=16384, dim=2048, type="bf16", ln=False, gate_rows=16384, pad=0.03),
    ]


# ---- drawn cases -----------------------------------------------------------------------------------------------------
def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_MOST = 1.7e9   # bytes of the largest listed case, roughly


def draw(rng):
    while True:
        kind = rng.choice(["embed_fwd", "embed_bwd", "logprob_fwd", "logprob_bwd", "clip", "norm_fwd", "norm_bwd"])
        pad = rng.choice([0.0, 0.03, 0.35])
        t = rng.choice(["f32", "bf16", "bf16", "f16"])
        if kind in ("embed_fwd", "embed_bwd"):
            c = dict(kind=kind, rows=_log_int(rng, 16, 65536), vocab=_log_int(rng, 20, 130000), dim=_log_int(rng, 16, 2048), out=rng.choice(["f32", t]),
                     pad=pad)
            c["table" if kind == "embed_fwd" else "grad"] = t
        elif kind in ("logprob_fwd", "logprob_bwd"):
            v = _log_int(rng, 16, 200000)
            c = dict(kind=kind, rows=_log_int(rng, 1, 65536), vocab=v, ld=rng.choice([v, (v + 63) // 64 * 64]), type=t,
                     mask=rng.choice(["none", "none", "shared", "rows"]), scale=rng.choice([1.0, 1.0, 0.7, 1.25]), pad=pad)
            if kind == "logprob_fwd":
                c.update(top=rng.choice([0, 1, 4, 8, 20]), entropy=rng.random() < 0.6)
            else:
                c.update(dentropy=rng.random() < 0.4)
        elif kind == "clip":
            n = _log_int(rng, 1, 240)
            c = dict(kind=kind, sizes="many", tensors=n, total=max(n * 20, _log_int(rng, 10000, 260_000_000)), over=rng.random() < 0.7)
        else:
            p = _log_int(rng, 1, 64)
            rows = p * _log_int(rng, 1, max(1, 65536 // p))
            c = dict(kind=kind, rows=rows, dim=_log_int(rng, 16, 8192), type=t, ln=rng.random() < 0.4, gate_rows=rng.choice([0, 1, p, rows]), pad=pad)
        w = work(c)
        if w["bytes"] <= _MOST and w["flops"] <= 2.5e9 and c.get("rows", 1) * c.get("vocab" if kind.startswith("logprob") else "dim", 1) <= 4.2e8:
            return c


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------
def work(c):
    k = c["kind"]
    if k == "embed_fwd":
        n = c["rows"] * c["dim"]
        return dict(bytes=c["rows"] * 4 + min(c["rows"], c["vocab"]) * c["dim"] * _SIZE[c["table"]] + n * _SIZE[c["out"]], flops=n)
    if k == "embed_bwd":
        n = c["rows"] * c["dim"]
        return dict(bytes=c["rows"] * 4 + n * _SIZE[c["grad"]] + c["vocab"] * c["dim"] * _SIZE[c["out"]], flops=2 * n)
    if k in ("logprob_fwd", "logprob_bwd"):
        n = c["rows"] * c["vocab"]
        mask = 0 if c["mask"] == "none" else c["vocab"] if c["mask"] == "shared" else n
        if k == "logprob_fwd":
            return dict(bytes=n * _SIZE[c["type"]] + mask + c["rows"] * (12 + 4 * c["entropy"] + 8 * c["top"]), flops=(6 if c["entropy"] else 4) * n)
        return dict(bytes=2 * n * _SIZE[c["type"]] + mask + c["rows"] * (12 + 8 * c["dentropy"]), flops=(8 if c["dentropy"] else 5) * n)
    if k == "clip":
        b = sum(n * _SIZE[t] for n, t in _tensors(c))
        return dict(bytes=2 * b, flops=3 * sum(n for n, _ in _tensors(c)))
    n, e = c["rows"] * c["dim"], _SIZE[c["type"]]
    gate = c["gate_rows"] * c["dim"] * e
    if k == "norm_fwd":
        return dict(bytes=4 * n * e + gate + 16 * c["rows"], flops=16 * n)
    return dict(bytes=6 * n * e + 2 * gate + 16 * c["rows"], flops=36 * n)


def _tensors(c):
    """(elements, type) of every tensor of a clip case; the same for every seed"""
    if c["sizes"] == "acoustic":
        return [(n, "f32") for n in (196096, 262656, 1579520, 1579520, 95931)]
    r = random.Random(c["tensors"] * 1000003 + c["total"])
    share = [math.exp(r.gauss(0.0, 2.0)) for _ in range(c["tensors"])]
    s = sum(share)
    return [(max(1, int(c["total"] * x / s)), r.choice(["f32", "bf16"])) for x in share]


def _room(n):
    return (n + 63) // 64 * 64


def _slices(c, flat):
    at, out = dict.fromkeys(flat, 0), []
    for n, t in _tensors(c):
        out.append(flat[t][at[t]:at[t] + n])
        at[t] += _room(n)
    return out


# ---- inputs ------------------------------------------------------------------------------------------------------------------
def _tokens(c, gen, zipf):
    """token ids, frequent ones first drawn by a 1/rank law and spread over the table; -1 for padding frames"""
    u = torch.rand(c["rows"], device="cuda", generator=gen, dtype=torch.float64)
    v = c["vocab"]
    if zipf:
        t = (torch.exp(u * math.log(v + 1.0)) - 1.0).floor().clamp(0, v - 1).long()
        t = torch.randperm(v, device="cuda", generator=gen)[t]
    else:
        t = (u * v).floor().clamp(0, v - 1).long()
    t[torch.rand(c["rows"], device="cuda", generator=gen) < c["pad"]] = -1
    return t.int()


def _normal(gen, shape, dtype, std=1.0):
    return (torch.randn(shape, device="cuda", generator=gen) * std).to(dtype)


def prepare(c, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(c)
    k = c["kind"]
    if k == "embed_fwd":
        s["tokens"] = _tokens(c, gen, True)
        s["weights"] = _normal(gen, (c["vocab"], c["dim"]), _DT[c["table"]], 0.02)
        s["result"] = torch.empty(c["rows"], c["dim"], device="cuda", dtype=_DT[c["out"]])
        s["factor"] = math.sqrt(c["dim"])
    elif k == "embed_bwd":
        s["tokens"] = _tokens(c, gen, True)
        s["dout"] = _normal(gen, (c["rows"], c["dim"]), _DT[c["grad"]], 0.01)
        s["result"] = torch.empty(c["vocab"], c["dim"], device="cuda", dtype=_DT[c["out"]])
        s["factor"] = math.sqrt(c["dim"])
    elif k in ("logprob_fwd", "logprob_bwd"):
        rows, v = c["rows"], c["vocab"]
        # rows of different sharpness: spreads between 0.5 and 4, as a model has them on easy and hard frames
        spread = 0.5 + 3.5 * torch.rand(rows, 1, device="cuda", generator=gen)
        x = torch.empty(rows, c["ld"], device="cuda", dtype=_DT[c["type"]])
        for a in range(0, rows, 4096):
            b = min(rows, a + 4096)
            x[a:b] = torch.randn(b - a, c["ld"], device="cuda", generator=gen).mul_(spread[a:b])
        s["logits"] = x[:, :v]
        s["tokens"] = _tokens(c, gen, False)
        s["allowed"] = None
        if c["mask"] != "none":
            s["allowed"] = torch.rand(1 if c["mask"] == "shared" else rows, v, device="cuda", generator=gen) < 0.9
            if c["mask"] == "shared":
                s["allowed"] = s["allowed"][0]
                s["allowed"][v // 2] = True
            # the given tokens are allowed ones
            on = s["tokens"].long().clamp(min=0)
            if c["mask"] == "rows":
                s["allowed"].scatter_(1, on[:, None], True)
            else:
                s["allowed"][on] = True
            s["allowed"] = s["allowed"].to(torch.uint8)
        f = lambda *shape: torch.empty(*shape, device="cuda")  # noqa: E731
        if k == "logprob_fwd":
            s["logprob"], s["lse"] = f(rows), f(rows)
            s["H"] = f(rows) if c["entropy"] else None
            s["top_lp"] = f(rows, c["top"]) if c["top"] else None
            s["top_tok"] = torch.empty(rows, c["top"], device="cuda", dtype=torch.int32) if c["top"] else None
        else:
            # what the forward pass left
            s["lse"], s["H"] = f(rows), f(rows)
            for a in range(0, rows, 4096):
                b = min(rows, a + 4096)
                z = s["logits"][a:b].float() * c["scale"]
                if s["allowed"] is not None:
                    z = z.masked_fill((s["allowed"] if c["mask"] == "shared" else s["allowed"][a:b]) == 0, -math.inf)
                lse = torch.logsumexp(z.double(), 1)
                lp = z.double() - lse[:, None]
                s["lse"][a:b] = lse
                s["H"][a:b] = -(lp.exp() * lp.clamp(min=-1e30)).sum(1)
            s["g"] = torch.where(s["tokens"] >= 0, -1.0 / rows, 0.0) * (0.5 + torch.rand(rows, device="cuda", generator=gen))
            s["h"] = 0.01 / rows * torch.rand(rows, device="cuda", generator=gen) if c["dentropy"] else None
            s["dlogits"] = torch.empty_like(x)[:, :v]
    elif k == "clip":
        s["grads"] = [_normal(gen, (n,), _DT[t], math.exp(random.Random(i).uniform(-7, -3))) for i, (n, t) in enumerate(_tensors(c))]
        # the scaled gradients go into one buffer for each type, where an optimizer has its own copies
        s["flat"] = {t: torch.zeros(sum(_room(n) for n, u in _tensors(c) if u == t), device="cuda", dtype=_DT[t])
                     for t in sorted({u for _, u in _tensors(c)})}
        s["clipped"] = _slices(c, s["flat"])
        norm = math.sqrt(sum(float((g.double() ** 2).sum()) for g in s["grads"]))
        s["max_norm"] = norm * (0.37 if c["over"] else 1.9)
        s["norm"] = torch.empty(1, device="cuda")
    else:
        rows, d, dt = c["rows"], c["dim"], _DT[c["type"]]
        s["x"], s["f"] = _normal(gen, (rows, d), dt, 2.0), _normal(gen, (rows, d), dt, 0.7)
        s["gate"] = (torch.rand(c["gate_rows"], d, device="cuda", generator=gen) * 1.2 - 0.1).to(dt) if c["gate_rows"] else None
        s["w1"], s["w2"] = (1.0 + 0.2 * torch.randn(d, device="cuda", generator=gen) for _ in range(2))
        s["b1"], s["b2"] = ((0.1 * torch.randn(d, device="cuda", generator=gen) for _ in range(2)) if c["ln"] else (None, None))
        s["real"] = (torch.rand(rows, device="cuda", generator=gen) >= c["pad"]).to(torch.int8) * 2   # pattern types: 0 padding, 2 inner frame
        s["eps"], s["a"] = 1e-5, 0.5
        e = lambda *shape, dtype=dt: torch.empty(*shape, device="cuda", dtype=dtype)  # noqa: E731
        s["y"], s["h"], s["stats"] = e(rows, d), e(rows, d), e(rows, 4, dtype=torch.float32)
        if k == "norm_bwd":
            # what the forward pass left: y and the statistics, in 64 bits and rounded once
            y, _, st = _norm_forward64(s)
            s["y"].copy_(y)
            s["stats"].copy_(_stats_of(s, s["y"].double(), st))
            s["dy"], s["dh"] = _normal(gen, (rows, d), dt, 0.01), _normal(gen, (rows, d), dt, 0.01)
            s["dx"], s["df"] = e(rows, d), e(rows, d)
            s["dgate"] = torch.empty_like(s["gate"]) if c["gate_rows"] else None
            s["dw1"], s["dw2"] = e(d, dtype=torch.float32), e(d, dtype=torch.float32)
            s["db1"], s["db2"] = (e(d, dtype=torch.float32), e(d, dtype=torch.float32)) if c["ln"] else (None, None)
    s["work"] = _workspace(s)
    return s


def _workspace(s):
    """the scratch a program keeps for the call, where the framework's operators ask for one"""
    if not own:
        return None
    b2 = _b2()
    k = s["kind"]
    if k == "embed_bwd":
        n = b2.embedding_backward_workspace(s["rows"], s["vocab"], s["dim"])
    elif k == "clip":
        s["list"] = b2.TensorList(s["grads"], s["clipped"])
        n = b2.gradient_norm_workspace()
    elif k == "norm_bwd":
        n = b2.block_norm_backward_workspace(s["rows"], s["dim"], s["gate_rows"])
    else:
        return None
    return torch.empty(max(n, 1), device="cuda", dtype=torch.uint8)


_module = None


def _b2():
    global _module
    if _module is None:
        sys.path.insert(0, os.path.join(os.getcwd(), "project-currennt-public_b200"))
        import b2lstm
        _module = b2lstm
    return _module


# ---- one pass ----------------------------------------------------------------------------------------------------------------
def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    b2, k = _b2(), s["kind"]
    st = torch.cuda.current_stream().cuda_stream
    if k == "embed_fwd":
        b2.embedding_forward(s["result"], s["weights"], s["tokens"], s["factor"], stream=st)
        return s["result"]
    if k == "embed_bwd":
        b2.embedding_backward(s["result"], s["dout"], s["tokens"], s["factor"], workspace=s["work"], stream=st)
        return s["result"]
    if k == "logprob_fwd":
        b2.logprob_forward(s["logits"], s["tokens"], s["logprob"], s["lse"], entropy=s["H"], top_tokens=s["top_tok"], top_logprobs=s["top_lp"],
                           mask=s["allowed"], scale=s["scale"], stream=st)
        return {n: s[n] for n in ("logprob", "lse", "H", "top_tok", "top_lp") if s[n] is not None}
    if k == "logprob_bwd":
        b2.logprob_backward(s["dlogits"], s["logits"], s["tokens"], s["lse"], s["g"], entropy=s["H"] if s["dentropy"] else None, dentropy=s["h"],
                            mask=s["allowed"], scale=s["scale"], stream=st)
        return s["dlogits"]
    if k == "clip":
        b2.gradient_clip(s["list"], s["max_norm"], s["norm"], workspace=s["work"], stream=st)
        return dict(s["flat"], norm=s["norm"])
    if k == "norm_fwd":
        b2.block_norm_forward(s["x"], s["f"], s["y"], s["h"], w_pre=s["w1"], b_pre=s["b1"], w_post=s["w2"], b_post=s["b2"], gate=s["gate"],
                              stats=s["stats"], pat_types=s["real"], layer_norm=s["ln"], eps=s["eps"], residual_scale=s["a"], stream=st)
        return dict(y=s["y"], h=s["h"], stats=s["stats"])
    b2.block_norm_backward(s["dx"], s["df"], s["dy"], s["dh"], s["y"], s["f"], s["stats"], w_pre=s["w1"], w_post=s["w2"], b_post=s["b2"],
                           gate=s["gate"], dgate=s["dgate"], dw_pre=s["dw1"], db_pre=s["db1"], dw_post=s["dw2"], db_post=s["db2"],
                           pat_types=s["real"], layer_norm=s["ln"], residual_scale=s["a"], workspace=s["work"], stream=st)
    return {n: s[n] for n in ("dx", "df", "dgate", "dw1", "db1", "dw2", "db2") if s[n] is not None}


def _run_plain(s):
    k = s["kind"]
    if k == "embed_fwd":
        tok = s["tokens"].long()
        rows = s["weights"][tok.clamp(min=0)].float() * s["factor"]
        return torch.where(tok[:, None] >= 0, rows, 0.0).to(s["result"].dtype)
    if k == "embed_bwd":
        tok = s["tokens"].long()
        d = torch.where(tok[:, None] >= 0, s["dout"].float(), 0.0) * s["factor"]
        return torch.zeros(s["vocab"], s["dim"], device="cuda").index_add_(0, tok.clamp(min=0), d).to(s["result"].dtype)
    if k in ("logprob_fwd", "logprob_bwd"):
        z = s["logits"].float() * s["scale"]
        if s["allowed"] is not None:
            z = torch.where(s["allowed"] != 0, z, -math.inf)
        tok = s["tokens"].long()
        real = tok >= 0
        if k == "logprob_bwd":
            lp = z - s["lse"][:, None]
            p = torch.exp(lp)
            d = -s["g"][:, None] * p
            if s["dentropy"]:
                d = d - s["h"][:, None] * torch.where(p > 0, p * (lp + s["H"][:, None]), 0.0)
            d.scatter_add_(1, tok.clamp(min=0)[:, None], torch.where(real, s["g"], 0.0)[:, None])
            return torch.where(real[:, None], d * s["scale"], 0.0).to(s["dlogits"].dtype)
        m = z.amax(1, keepdim=True)
        e = torch.exp(z - m)
        total = e.sum(1)
        lse = m[:, 0] + torch.log(total)
        out = dict(logprob=torch.where(real, z.gather(1, tok.clamp(min=0)[:, None])[:, 0] - lse, 0.0), lse=lse)
        if s["entropy"]:
            out["H"] = torch.log(total) - torch.where(e > 0, e * (z - m), 0.0).sum(1) / total
        if s["top"]:
            value, index = torch.sort(z, dim=1, descending=True, stable=True)
            value, index = value[:, :s["top"]], index[:, :s["top"]]
            if value.shape[1] < s["top"]:
                more = s["top"] - value.shape[1]
                value = torch.nn.functional.pad(value, (0, more), value=-math.inf)
                index = torch.nn.functional.pad(index, (0, more), value=-1)
            none = value == -math.inf
            out["top_tok"] = torch.where(none, -1, index).int()
            out["top_lp"] = torch.where(none, -math.inf, value - lse[:, None])
        return out
    if k == "clip":
        g32 = [g.float() for g in s["grads"]]
        norm = torch.stack([(g * g).sum() for g in g32]).sum().sqrt()
        coef = torch.where(norm > s["max_norm"], s["max_norm"] / norm, 1.0)
        for to, x in zip(s["clipped"], g32):
            to.copy_(x * coef)
        return dict(s["flat"], norm=norm.reshape(1))
    if k == "norm_fwd":
        return _norm_forward32(s)
    return _norm_backward32(s)


def _gate32(s):
    if s["gate"] is None:
        return 1.0
    return s["gate"].float().repeat(s["rows"] // s["gate_rows"], 1)


def _norm32(v, ln, eps):
    mean = v.mean(1, keepdim=True) if ln else torch.zeros(v.shape[0], 1, device="cuda")
    d = v - mean
    rstd = torch.rsqrt((d * d).mean(1, keepdim=True) + eps)
    return d * rstd, mean[:, 0], rstd[:, 0]


def _affine32(v, w, b):
    return v * w if b is None else v * w + b


def _norm_forward32(s):
    real = (s["real"] != 0)[:, None]
    n, m2, r2 = _norm32(s["f"].float(), s["ln"], s["eps"])
    y = s["x"].float() + s["a"] * _gate32(s) * _affine32(n, s["w2"], s["b2"])
    y = torch.where(real, y, 0.0).to(s["y"].dtype)
    n, m1, r1 = _norm32(y.float(), s["ln"], s["eps"])
    h = torch.where(real, _affine32(n, s["w1"], s["b1"]), 0.0).to(s["h"].dtype)
    return dict(y=y, h=h, stats=torch.where(real, torch.stack([m2, r2, m1, r1], 1), 0.0))


def _back32(d, v, w, rstd, ln):
    """gradient of w * v + b, v = (input - mean) * rstd, with respect to the input"""
    u = d * w
    out = u - v * (u * v).mean(1, keepdim=True)
    if ln:
        out = out - u.mean(1, keepdim=True)
    return out * rstd


def _norm_backward32(s):
    real = (s["real"] != 0)[:, None]
    m2, r2, m1, r1 = (t[:, None] for t in s["stats"].unbind(1))
    dh, dy = torch.where(real, s["dh"].float(), 0.0), torch.where(real, s["dy"].float(), 0.0)
    v1, v2 = (s["y"].float() - m1) * r1, (s["f"].float() - m2) * r2
    dt = dy + _back32(dh, v1, s["w1"], r1, s["ln"])
    gate = _gate32(s)
    dn = dt * s["a"] * gate
    out = dict(dx=torch.where(real, dt, 0.0).to(s["dx"].dtype), df=torch.where(real, _back32(dn, v2, s["w2"], r2, s["ln"]), 0.0).to(s["df"].dtype))
    if s["gate"] is not None:
        dg = torch.where(real, dt * s["a"] * _affine32(v2, s["w2"], s["b2"]), 0.0)
        out["dgate"] = dg.view(-1, s["gate_rows"], s["dim"]).sum(0).to(s["dgate"].dtype)
    out["dw1"] = (dh * v1).sum(0)
    if s["ln"]:
        out["db1"] = dh.sum(0)
    out["dw2"] = (torch.where(real, dn * v2, 0.0)).sum(0)
    if s["ln"]:
        out["db2"] = torch.where(real, dn, 0.0).sum(0)
    return out


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------------------
def _stats_of(s, y, st2):
    mean = y.mean(1) if s["ln"] else torch.zeros_like(y[:, 0])
    var = ((y - mean[:, None]) ** 2).mean(1)
    out = torch.stack([st2[0], st2[1], mean, 1.0 / torch.sqrt(var + s["eps"])], 1)
    out[s["real"] == 0] = 0.0
    return out


def _rows64(v, ln, eps):
    mean = v.mean(1) if ln else torch.zeros_like(v[:, 0])
    var = (v * v).mean(1) if not ln else v.var(1, unbiased=False)
    return mean, 1.0 / torch.sqrt(var + eps)


def _gate64(s):
    if s["gate"] is None:
        return torch.ones(1, 1, device="cuda", dtype=torch.float64)
    at = torch.arange(s["rows"], device="cuda") % s["gate_rows"]
    return s["gate"].double()[at]


def _norm_forward64(s):
    pad = s["real"] == 0
    f = s["f"].double()
    mean, rstd = _rows64(f, s["ln"], s["eps"])
    n = (f - mean[:, None]) * rstd[:, None] * s["w2"].double()
    if s["b2"] is not None:
        n = n + s["b2"].double()
    y = s["x"].double() + s["a"] * _gate64(s) * n
    y[pad] = 0.0
    yr = y.to(s["y"].dtype).double()          # the block's output is held in the tensors' type, and the next norm reads that
    m1, r1 = _rows64(yr, s["ln"], s["eps"])
    h = (yr - m1[:, None]) * r1[:, None] * s["w1"].double()
    if s["b1"] is not None:
        h = h + s["b1"].double()
    h[pad] = 0.0
    return y, h, (mean, rstd)


def exact(c, seed):
    if c["kind"] in ("logprob_fwd", "logprob_bwd") and c["rows"] * c["vocab"] > 5e8:
        return None
    s = prepare(c, seed)
    k = c["kind"]
    if k == "embed_fwd":
        out = torch.zeros(c["rows"], c["dim"], device="cuda", dtype=torch.float64)
        real = s["tokens"] >= 0
        out[real] = s["weights"].double()[s["tokens"][real].long()] * s["factor"]
        return out
    if k == "embed_bwd":
        real = s["tokens"] >= 0
        tok, order = torch.sort(s["tokens"][real].long())
        out = torch.zeros(c["vocab"], c["dim"], device="cuda", dtype=torch.float64)
        d = s["dout"][real][order].double()
        sums = torch.cat([torch.zeros(1, c["dim"], device="cuda", dtype=torch.float64), d.cumsum(0)])
        ids, counts = torch.unique_consecutive(tok, return_counts=True)
        end = counts.cumsum(0)
        out[ids] = (sums[end] - sums[end - counts]) * s["factor"]
        return out
    if k == "logprob_fwd":
        names = ["logprob", "lse"] + (["H"] if c["entropy"] else []) + (["top_tok", "top_lp"] if c["top"] else [])
        parts = {n: [] for n in names}
        for a in range(0, c["rows"], 1024):
            b = min(c["rows"], a + 1024)
            z = s["logits"][a:b].double() * c["scale"]
            if s["allowed"] is not None:
                z[((s["allowed"] if c["mask"] == "shared" else s["allowed"][a:b]) == 0).expand(b - a, c["vocab"])] = -math.inf
            lse = torch.logsumexp(z, 1)
            tok = s["tokens"][a:b].long()
            lp = z - lse[:, None]
            parts["lse"].append(lse)
            parts["logprob"].append(torch.where(tok >= 0, lp[torch.arange(b - a, device="cuda"), tok.clamp(min=0)], 0.0))
            if c["entropy"]:
                parts["H"].append(torch.special.entr(lp.exp()).sum(1))
            if c["top"]:
                best = torch.topk(lp, min(c["top"], c["vocab"]), dim=1)[0]
                parts["top_lp"].append(torch.nn.functional.pad(best, (0, c["top"] - best.shape[1]), value=-math.inf))
        return {n: torch.cat(parts[n]) if parts[n] else None for n in names}
    if k == "logprob_bwd":
        out = torch.zeros(c["rows"], c["vocab"], device="cuda", dtype=torch.float64)
        for a in range(0, c["rows"], 1024):
            b = min(c["rows"], a + 1024)
            z = s["logits"][a:b].double() * c["scale"]
            off = torch.zeros_like(z, dtype=torch.bool)
            if s["allowed"] is not None:
                off = ((s["allowed"] if c["mask"] == "shared" else s["allowed"][a:b]) == 0).expand(b - a, c["vocab"])
            lp = z - s["lse"][a:b, None].double()
            p = lp.exp()
            tok = s["tokens"][a:b].long()
            hot = torch.zeros_like(z)
            hot[torch.arange(b - a, device="cuda"), tok.clamp(min=0)] = 1.0
            d = s["g"][a:b, None].double() * (hot - p)
            if c["dentropy"]:
                d -= s["h"][a:b, None].double() * p * (lp + s["H"][a:b, None].double())
            d[off] = 0.0
            d[tok < 0] = 0.0
            out[a:b] = d * c["scale"]
        return out
    if k == "clip":
        norm = math.sqrt(math.fsum(float((g.double() ** 2).sum()) for g in s["grads"]))
        coef = min(1.0, s["max_norm"] / norm)
        flat = {t: x.double().zero_() for t, x in s["flat"].items()}
        for to, g in zip(_slices(c, flat), s["grads"]):
            to.copy_(g.double() * coef)
        return dict(flat, norm=torch.tensor([norm], dtype=torch.float64))
    if k == "norm_fwd":
        y, h, st = _norm_forward64(s)
        return dict(y=y, h=h, stats=_stats_of(s, y.to(s["y"].dtype).double(), st))
    pad = s["real"] == 0
    dh, dy = s["dh"].double(), s["dy"].double()
    dh[pad] = 0.0
    dy[pad] = 0.0
    m2, r2, m1, r1 = (t[:, None] for t in s["stats"].double().unbind(1))

    def through(d, v, m, r, w):
        # with u = (v - m) r the gradient of w u is r (w d - [mean(w d)] - u mean(w d u))
        u, wd = (v - m) * r, d * w.double()
        g = wd - u * (wd * u).mean(1, keepdim=True)
        return u, r * (g - wd.mean(1, keepdim=True) if c["ln"] else g)

    u1, back1 = through(dh, s["y"].double(), m1, r1, s["w1"])
    dt = dy + back1
    dn = dt * (s["a"] * _gate64(s))
    u2, df = through(dn, s["f"].double(), m2, r2, s["w2"])
    n = u2 * s["w2"].double() + (0.0 if s["b2"] is None else s["b2"].double())
    dg = dt * s["a"] * n
    dg[pad] = 0.0
    out = dict(dx=dt, df=df)
    if s["gate"] is not None:
        out["dgate"] = torch.zeros(c["gate_rows"], c["dim"], device="cuda", dtype=torch.float64)
        out["dgate"].index_add_(0, torch.arange(c["rows"], device="cuda") % c["gate_rows"], dg)
    out["dw1"] = (dh * u1).sum(0)
    if c["ln"]:
        out["db1"] = dh.sum(0)
    out["dw2"] = (dn * u2).sum(0)
    if c["ln"]:
        out["db2"] = dn.sum(0)
    return out
