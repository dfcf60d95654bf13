"""The operators with which a token model answers and learns from another one, as measurable cases.

A token model writes by beam search: a step's logits come from a product of the last layer's outputs with a large matrix, held in 8 bits; the best
continuations over all beams of a sequence and all tokens go on, and the states and histories of the beams follow them.  A small model learns from a
large one by the large one's most likely tokens and their log probabilities.  Kinds of case:

  distill_fwd   divergence of a model's tokens from a teacher's most likely ones, for each row of logits
  distill_bwd   its gradient with respect to the logits
  select        the best continuations of the beams of each sequence, with their scores, beams and tokens
  reorder       states and histories of the beams by the beams that go on
  quantize      rows in 8-bit integers with a scale for each row
  product       activations times a matrix in 8-bit integers with a scale for each token and each channel; the activations are quantised in the call

Rows of logits are frames (padding frames have the token -1), or the beams of all sequences one after the other.
"""
import math
import os
import sys

import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}
_REST = 2.0 ** -20    # a rest of the teacher's probability below this is none: its log probabilities are fp32


def listed():
    return [
        # two utterances of quantised targets learnt from a larger model
        dict(name="distill 1516x259 top8", kind="distill_fwd", rows=1516, vocab=259, ld=259, type="f32", top=8, rest=False, scale=1.0, pad=0.05),
        # a training batch over a large vocabulary, the rest of the vocabulary as one more outcome
        dict(name="distill 8192x50001 top32", kind="distill_fwd", rows=8192, vocab=50001, ld=50048, type="bf16", top=32, rest=True, scale=1.0, pad=0.03),
        # a fraction of 32 utterances backwards, small odd vocabulary
        dict(name="distill grad 38400x259 top16", kind="distill_bwd", rows=38400, vocab=259, ld=259, type="f32", top=16, rest=True, scale=1.0, pad=0.35),
        # a training batch backwards at temperature 2, rows that start anywhere
        dict(name="distill grad 8192x32003 top64", kind="distill_bwd", rows=8192, vocab=32003, ld=32003, type="bf16", top=64, rest=True, scale=0.5, pad=0.03),
        # one sequence with four beams: latency counts
        dict(name="select 1x4x32000 top8", kind="select", groups=1, beams=4, vocab=32000, ld=32000, type="f32", top=8, mask="none", scale=1.0, done=0.0),
        # sixty-four sequences with eight beams, some tokens ruled out, some beams at their end
        dict(name="select 64x8x50001 top16", kind="select", groups=64, beams=8, vocab=50001, ld=50048, type="bf16", top=16, mask="shared", scale=1.25, done=0.1),
        # states of two layers and the tokens so far, of one sequence
        dict(name="reorder 1x4", kind="reorder", groups=1, beams=4, states=4, dim=512, type="f32", steps=200, frames=0),
        # states of three layers, the tokens so far and the frames of a layer, of sixty-four sequences
        dict(name="reorder 64x8 with frames", kind="reorder", groups=64, beams=8, states=6, dim=1024, type="bf16", steps=200, frames=512),
        # a step's activations
        dict(name="quantize 64x1024", kind="quantize", rows=64, dim=1024, type="bf16"),
        # an output matrix, once when a model is loaded
        dict(name="quantize 50001x1024", kind="quantize", rows=50001, dim=1024, type="f32"),
        # logits of a step of eight beams
        dict(name="product 8x50001x1024", kind="product", rows=8, channels=50001, dim=1024, type="bf16", out="f32", bias=True),
        # logits of a whole batch, scored in 8 bits
        dict(name="product 8192x50001x1024", kind="product", rows=8192, channels=50001, dim=1024, type="bf16", out="bf16", bias=False),
    ]


# ---- drawn cases -----------------------------------------------------------------------------------------------------
def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        kind = rng.choice(["distill_fwd", "distill_bwd", "select", "reorder", "quantize", "product"])
        t = rng.choice(["f32", "bf16", "bf16", "f16"])
        if kind in ("distill_fwd", "distill_bwd"):
            v = _log_int(rng, 16, 200000)
            c = dict(kind=kind, rows=_log_int(rng, 1, 65536), vocab=v, ld=rng.choice([v, (v + 63) // 64 * 64]), type=t, top=min(v, _log_int(rng, 1, 128)),
                     rest=rng.random() < 0.6, scale=rng.choice([1.0, 1.0, 0.5, 0.7]), pad=rng.choice([0.0, 0.03, 0.35]))
            if c["rows"] * v > 4.1e8:
                continue
        elif kind == "select":
            v, b = _log_int(rng, 16, 200000), _log_int(rng, 1, 32)
            c = dict(kind=kind, groups=_log_int(rng, 1, 256), beams=b, vocab=v, ld=rng.choice([v, (v + 63) // 64 * 64]), type=t, top=rng.choice([b, 2 * b]),
                     mask=rng.choice(["none", "none", "shared", "rows"]), scale=rng.choice([1.0, 1.0, 0.7, 1.25]), done=rng.choice([0.0, 0.1]))
            if c["groups"] * b * v > 2.6e7:
                continue
        elif kind == "reorder":
            c = dict(kind=kind, groups=_log_int(rng, 1, 256), beams=_log_int(rng, 1, 32), states=rng.randrange(1, 13), dim=_log_int(rng, 16, 4096), type=t,
                     steps=_log_int(rng, 1, 1000), frames=rng.choice([0, 0, _log_int(rng, 16, 1024)]))
        elif kind == "quantize":
            c = dict(kind=kind, rows=_log_int(rng, 1, 65536), dim=_log_int(rng, 16, 8192), type=t)
        else:
            c = dict(kind=kind, rows=_log_int(rng, 1, 16384), channels=_log_int(rng, 16, 65536), dim=_log_int(rng, 16, 8192), type=t,
                     out=rng.choice(["f32", t]), bias=rng.random() < 0.5)
            if c["rows"] * c["channels"] > 4.1e8:
                continue
        w = work(c)
        if w["bytes"] <= 1.7e9 and w["flops"] <= (8.4e11 if kind == "product" else 4e9):
            return c


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------
def work(c):
    k = c["kind"]
    if k in ("distill_fwd", "distill_bwd"):
        n, each = c["rows"] * c["vocab"], c["rows"] * (8 * c["top"] + 8 + 4 * c["rest"])
        if k == "distill_fwd":
            return dict(bytes=n * _SIZE[c["type"]] + each, flops=4 * n)
        return dict(bytes=2 * n * _SIZE[c["type"]] + each, flops=(8 if c["rest"] else 5) * n)
    if k == "select":
        rows = c["groups"] * c["beams"]
        n = rows * c["vocab"]
        mask = 0 if c["mask"] == "none" else c["vocab"] if c["mask"] == "shared" else n
        return dict(bytes=n * _SIZE[c["type"]] + mask + 9 * rows + 12 * c["groups"] * c["top"], flops=5 * n)
    if k == "reorder":
        rows = c["groups"] * c["beams"]
        n = rows * (_SIZE[c["type"]] * (c["states"] * c["dim"] + c["steps"] * c["frames"]) + 4 * c["steps"])
        return dict(bytes=2 * n + 4 * rows, flops=0)
    n = c["rows"] * c["dim"]
    if k == "quantize":
        return dict(bytes=n * _SIZE[c["type"]] + n + 4 * c["rows"], flops=3 * n)
    m = c["channels"] * c["dim"]
    return dict(bytes=n * _SIZE[c["type"]] + m + 4 * c["channels"] * (1 + c["bias"]) + c["rows"] * c["channels"] * _SIZE[c["out"]], flops=2 * c["rows"] * m)


# ---- inputs ------------------------------------------------------------------------------------------------------------------
def _normal(gen, shape, dtype, std=1.0):
    return (torch.randn(shape, device="cuda", generator=gen) * std).to(dtype)


def _logits(gen, rows, ld, dtype):
    """rows of different sharpness: spreads between 0.5 and 4, as a model has them on easy and hard frames"""
    spread = 0.5 + 3.5 * torch.rand(rows, 1, device="cuda", generator=gen)
    return torch.randn(rows, ld, device="cuda", generator=gen).mul_(spread).to(dtype), spread


def _room(n):
    """bytes from row to row of a matrix in 8-bit integers"""
    return (n + 15) // 16 * 16


def prepare(c, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(c)
    k = c["kind"]
    f = lambda *shape: torch.empty(*shape, device="cuda")  # noqa: E731
    i = lambda *shape: torch.empty(*shape, device="cuda", dtype=torch.int32)  # noqa: E731
    rand = lambda *shape: torch.rand(*shape, device="cuda", generator=gen)  # noqa: E731
    if k in ("distill_fwd", "distill_bwd"):
        rows, v, top = c["rows"], c["vocab"], c["top"]
        x, spread = _logits(gen, rows, c["ld"], _DT[c["type"]])
        s["logits"] = x[:, :v]
        # the teacher's list: a model near the student's, its most likely tokens; some rows have fewer, padding frames none
        s["tokens"], s["teacher"], lse, rest = i(rows, top), f(rows, top), f(rows), f(rows)
        step = max(1, min(rows, 2 ** 26 // v))
        few = torch.where(rand(rows) < 0.1, (rand(rows) * top).long() + 1, top)
        few[rand(rows) < c["pad"]] = 0
        for a in range(0, rows, step):
            b = min(rows, a + step)
            z = s["logits"][a:b].float().mul_(c["scale"])
            t = torch.randn(b - a, v, device="cuda", generator=gen).mul_(spread[a:b] * (0.6 * c["scale"])).add_(z, alpha=0.8)
            value, index = torch.topk(t, top, dim=1)
            none = torch.arange(top, device="cuda") >= few[a:b, None]
            s["tokens"][a:b] = torch.where(none, -1, index)
            s["teacher"][a:b] = torch.where(none, -math.inf, value - torch.logsumexp(t, 1, keepdim=True))
            if k == "distill_bwd":
                # what the forward pass left
                lse[a:b] = torch.logsumexp(z.double(), 1)
                pad = torch.nn.functional.pad(z, (0, 1))
                pad.scatter_(1, torch.where(none, v, index), -math.inf)
                rest[a:b] = torch.logsumexp(pad[:, :v].double(), 1)
        s["loss"], s["lse"], s["lse_rest"] = f(rows), lse, rest if c["rest"] else None
        if k == "distill_bwd":
            # the mean over the frames; scaled up where 16 bits of a small range hold the gradient
            s["dloss"] = (0.5 + rand(rows)) * ((1024.0 if c["type"] == "f16" else 1.0) / rows)
            s["dlogits"] = torch.empty_like(x)[:, :v]
    elif k == "select":
        rows, v = c["groups"] * c["beams"], c["vocab"]
        s["logits"] = _logits(gen, rows, c["ld"], _DT[c["type"]])[0][:, :v]
        s["scores"] = -20.0 * rand(rows)
        # beams at their end, and the factors of a length penalty: such beams are shorter than the others
        s["finished"] = (rand(rows) < c["done"]).to(torch.uint8) if c["done"] else None
        s["weights"] = torch.where(s["finished"] != 0, 0.05 + 0.05 * rand(rows), 0.05) if c["done"] else None
        s["end"] = v // 3
        s["allowed"] = None
        if c["mask"] != "none":
            s["allowed"] = (rand(*((v,) if c["mask"] == "shared" else (rows, v))) < 0.9).to(torch.uint8)
            s["allowed"][..., v // 2] = 1
        s["best"], s["from"], s["token"] = f(c["groups"], c["top"]), i(c["groups"], c["top"]), i(c["groups"], c["top"])
    elif k == "reorder":
        rows, dt = c["groups"] * c["beams"], _DT[c["type"]]
        s["states"] = [_normal(gen, (rows, c["dim"]), dt, 0.5) for _ in range(c["states"])]
        s["states"].append((rand(c["steps"], rows) * 32000).int())
        if c["frames"]:
            s["states"].append(_normal(gen, (c["steps"], rows, c["frames"]), dt, 0.5))
        s["axes"] = [0] * c["states"] + [1] * (2 if c["frames"] else 1)
        s["parents"] = (rand(c["groups"], c["beams"]) * c["beams"]).int().clamp(max=c["beams"] - 1)
        # a program swaps two sets of buffers from step to step
        s["next"] = [torch.empty_like(t) for t in s["states"]]
    else:
        rows, d = c["rows"], c["dim"]
        # rows of different magnitude, a few large channels
        s["x"] = _normal(gen, (rows, d), torch.float32).mul_(0.3 + 2.0 * rand(rows, 1)).mul_(torch.where(rand(d) < 0.01, 8.0, 1.0)).to(_DT[c["type"]])
        if k == "quantize":
            s["q"] = torch.empty(rows, _room(d), device="cuda", dtype=torch.int8)[:, :d]
            s["s"] = f(rows)
        else:
            n = c["channels"]
            s["w"] = torch.empty(n, _room(d), device="cuda", dtype=torch.int8)[:, :d]
            s["w"].copy_(torch.randn(n, d, device="cuda", generator=gen).mul_(32.0).round_().clamp_(-127, 127))
            s["ws"] = (0.5 + rand(n)) / (32.0 * math.sqrt(d))
            s["b"] = _normal(gen, (n,), torch.float32, 0.1) if c["bias"] else None
            s["result"] = torch.empty(rows, n, device="cuda", dtype=_DT[c["out"]])
    _keep(s)
    return s


def _keep(s):
    """the scratch and the lists a program keeps for the call, where the framework's operators ask for one"""
    if not own:
        return
    b2, k, n = _b2(), s["kind"], 0
    if k == "select":
        n = b2.beam_select_workspace(s["groups"], s["beams"], s["vocab"], s["top"])
    elif k == "product":
        n = b2.int8_product_workspace(s["rows"], s["channels"], s["dim"])
    elif k == "reorder":
        s["list"] = b2.StateList(s["states"], s["axes"], s["next"])
    s["work"] = torch.empty(max(n, 1), device="cuda", dtype=torch.uint8)


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
    if k == "distill_fwd":
        b2.distill_forward(s["logits"], s["tokens"], s["teacher"], s["loss"], s["lse"], lse_rest=s["lse_rest"], scale=s["scale"], stream=st)
        return dict(loss=s["loss"], lse=s["lse"], **({"lse_rest": s["lse_rest"]} if s["rest"] else {}))
    if k == "distill_bwd":
        b2.distill_backward(s["dlogits"], s["logits"], s["tokens"], s["teacher"], s["lse"], s["dloss"], lse_rest=s["lse_rest"], scale=s["scale"], stream=st)
        return s["dlogits"]
    if k == "select":
        b2.beam_select(s["logits"], s["scores"], s["best"], s["from"], s["token"], finished=s["finished"], weights=s["weights"], end_token=s["end"],
                       mask=s["allowed"], scale=s["scale"], workspace=s["work"], stream=st)
        return {"score": s["best"], "from": s["from"], "token": s["token"]}
    if k == "reorder":
        b2.beam_reorder(s["list"], s["parents"], stream=st)
        return s["next"]
    if k == "quantize":
        b2.int8_quantize(s["q"], s["s"], s["x"], stream=st)
        return dict(q=s["q"], scale=s["s"])
    b2.int8_product(s["result"], s["x"], s["w"], s["ws"], bias=s["b"], workspace=s["work"], stream=st)
    return s["result"]


def _lse32(z):
    m = z.amax(1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    return m[:, 0] + torch.log(torch.exp(z - m).sum(1))


def _teacher32(s):
    """probabilities of the listed tokens and of the rest, and where a place of the list holds a token"""
    there = s["tokens"] >= 0
    lp = torch.where(there, s["teacher"], -math.inf)
    if s["rest"]:
        q = torch.exp(lp)
        left = (1.0 - q.double().sum(1)).float()
        return q, torch.where(there.any(1) & (left >= _REST), left, 0.0), there
    most = lp.amax(1, keepdim=True)
    e = torch.exp(lp - torch.where(most == -math.inf, 0.0, most))
    return torch.where(there, e / e.sum(1, keepdim=True), 0.0), torch.zeros_like(s["lse"]), there


def _quantize32(x):
    most = x.float().abs().amax(1)
    top = torch.full_like(most, 127.0)      # a tensor: divisions by and of a number become products with a reciprocal
    inv = torch.where(most > 0, top / most, 0.0)
    # a value next to the middle of two integers: the product in 64 bits, rounded once
    return torch.round(x.double() * inv.double()[:, None]).float(), most / top


def _run_plain(s):
    k = s["kind"]
    if k in ("distill_fwd", "distill_bwd"):
        z = s["logits"].float() * s["scale"]
        q, left, there = _teacher32(s)
        at = torch.where(there, s["tokens"], 0).long()
        known = there.any(1)
        if k == "distill_bwd":
            d = torch.exp(z - s["lse"][:, None])
            p = d.gather(1, at)
            if s["rest"]:
                d = d - torch.where(left > 0, left, 0.0)[:, None] * torch.exp(z - torch.where(left > 0, s["lse_rest"], 0.0)[:, None])
            # places without a token write behind the row
            d = torch.nn.functional.pad(d, (0, 1)).scatter_(1, torch.where(there, at, s["vocab"]), p - q)[:, :-1]
            return torch.where(known[:, None], d * (s["dloss"] * s["scale"])[:, None], 0.0).to(s["dlogits"].dtype)
        lse = _lse32(z)
        gap = torch.log(q) - (z.gather(1, at) - lse[:, None])
        loss = torch.where(q > 0, q * gap, 0.0).sum(1)
        out = dict(lse=lse)
        if s["rest"]:
            others = torch.nn.functional.pad(z, (0, 1)).scatter_(1, torch.where(there, at, s["vocab"]), -math.inf)[:, :-1]
            out["lse_rest"] = _lse32(others)
            loss = loss + torch.where(left > 0, left * (torch.log(left) - (out["lse_rest"] - lse)), 0.0)
        return dict(loss=torch.where(known, loss, 0.0), **out)
    if k == "select":
        z = s["logits"].float() * s["scale"]
        if s["allowed"] is not None:
            z = torch.where(s["allowed"] != 0, z, -math.inf)
        # scores of different beams meet: 64 bits
        z = z.double()
        m = z.amax(1, keepdim=True)
        score = z + (s["scores"].double()[:, None] - m - torch.log(torch.exp(z - m).sum(1, keepdim=True)))
        if s["finished"] is not None:
            end = torch.where(torch.arange(s["vocab"], device="cuda") == s["end"], s["scores"].double()[:, None], -math.inf)
            score = torch.where(s["finished"][:, None] != 0, end, score)
        rank = score if s["weights"] is None else score * s["weights"].double()[:, None]
        order = torch.sort(rank.view(s["groups"], -1), dim=1, descending=True, stable=True)[1][:, :s["top"]]
        best = score.view(s["groups"], -1).gather(1, order)
        best, order = (torch.nn.functional.pad(t, (0, s["top"] - t.shape[1]), value=w) for t, w in ((best, -math.inf), (order, 0)))
        none = best == -math.inf
        return {"score": best.float(), "from": torch.where(none, -1, order // s["vocab"]).int(), "token": torch.where(none, -1, order % s["vocab"]).int()}
    if k == "reorder":
        rows = (s["parents"].long() + torch.arange(s["groups"], device="cuda")[:, None] * s["beams"]).view(-1)
        return [t.index_select(a, rows) for t, a in zip(s["states"], s["axes"])]
    q, scale = _quantize32(s["x"])
    if k == "quantize":
        return dict(q=q.to(torch.int8), scale=scale)
    y = (q @ s["w"].float().t()) * (scale[:, None] * s["ws"])
    return (y if s["b"] is None else y + s["b"]).to(s["result"].dtype)


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------------------
def exact(c, seed):
    k = c["kind"]
    if k == "reorder":
        return None
    if k in ("distill_fwd", "distill_bwd") and c["rows"] * c["vocab"] > 4.2e8:
        return None
    s = prepare(c, seed)
    if k in ("distill_fwd", "distill_bwd"):
        rows, v = c["rows"], c["vocab"]
        loss, lse, rest = (torch.zeros(rows, device="cuda", dtype=torch.float64) for _ in range(3))
        grad = torch.zeros(rows, v, device="cuda", dtype=torch.float64) if k == "distill_bwd" else None
        step = max(1, min(rows, 2 ** 25 // v))
        for a in range(0, rows, step):
            b = min(rows, a + step)
            z = (s["logits"][a:b].float() * c["scale"]).double()
            tok, lp = s["tokens"][a:b].long(), s["teacher"][a:b].double()
            have = tok >= 0
            lp = lp.masked_fill(~have, -math.inf)
            on = torch.zeros(b - a, v + 1, device="cuda", dtype=torch.bool)
            on.scatter_(1, tok.masked_fill(~have, v), True)
            on = on[:, :v]
            total = torch.logsumexp(z, 1)
            others = torch.logsumexp(z.masked_fill(on, -math.inf), 1)
            if c["rest"]:
                r = 1.0 - lp.exp().sum(1)
                r = torch.where(r < _REST, 0.0, r)
            else:
                lp = lp - torch.logsumexp(lp, 1, keepdim=True)
                r = torch.zeros_like(total)
            empty = ~have.any(1)
            r[empty] = 0.0
            q = lp.exp().masked_fill(~have, 0.0)
            if k == "distill_fwd":
                zk = z.gather(1, tok.clamp(min=0))
                part = torch.special.xlogy(q, q) - q * (zk - total[:, None])
                loss[a:b] = part.masked_fill(~have, 0.0).sum(1)
                some = r > 0
                loss[a:b][some] += (r * (torch.log(r) - others + total))[some]
                loss[a:b][empty] = 0.0
                lse[a:b], rest[a:b] = total, others
                continue
            p = (z - s["lse"][a:b, None].double()).exp()
            want = torch.zeros(b - a, v + 1, device="cuda", dtype=torch.float64)
            want.scatter_(1, tok.masked_fill(~have, v), q)
            want = want[:, :v]
            if c["rest"]:
                tail = (z - s["lse_rest"][a:b, None].double()).exp() * r[:, None]
                tail[r == 0] = 0.0
                want = torch.where(on, want, tail)
            g = (p - want) * (s["dloss"][a:b, None].double() * c["scale"])
            g[empty] = 0.0
            grad[a:b] = g
        if k == "distill_bwd":
            return grad
        return dict(loss=loss, lse=lse, **({"lse_rest": rest} if c["rest"] else {}))
    if k == "select":
        best = []
        for g in range(c["groups"]):
            a, b = g * c["beams"], (g + 1) * c["beams"]
            z = (s["logits"][a:b].float() * c["scale"]).double()
            if s["allowed"] is not None:
                z = z.masked_fill((s["allowed"] if c["mask"] == "shared" else s["allowed"][a:b]) == 0, -math.inf)
            total = torch.log_softmax(z, 1) + s["scores"][a:b, None].double()
            if s["finished"] is not None:
                over = s["finished"][a:b] != 0
                total[over] = -math.inf
                total[over, s["end"]] = s["scores"][a:b][over].double()
            rank = total if s["weights"] is None else total * s["weights"][a:b, None].double()
            at = torch.topk(rank.reshape(-1), min(c["top"], rank.numel()))[1]
            best.append(torch.nn.functional.pad(total.reshape(-1)[at], (0, c["top"] - at.numel()), value=-math.inf))
        return {"score": torch.stack(best), "from": None, "token": None}
    # the scale is what 32 bits hold; the integers go by it
    x = s["x"].double()
    most = x.abs().max(1)[0]
    inv = (127.0 / most).float().double()
    inv[most == 0] = 0.0
    if k == "quantize":
        return dict(q=None, scale=most / 127.0)
    y = torch.empty(c["rows"], c["channels"], device="cuda", dtype=torch.float64)
    w = s["w"].double().t()
    for a in range(0, c["rows"], 2048):
        b = min(c["rows"], a + 2048)
        y[a:b] = torch.mm((x[a:b] * inv[a:b, None]).round(), w)
    y *= (most / 127.0)[:, None]
    y *= s["ws"].double()
    if s["b"] is not None:
        y += s["b"].double()
    return y
