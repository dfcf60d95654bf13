"""The kernels of the token operators that only calls with many rows reach, against plain implementations in 64 bits (on the GPU, by elementary operations).
Tolerances as in test_gpu_token_operators.py: error bounds, element by element; u is the unit roundoff of fp32."""
import math

import pytest

from test_gpu_token_operators import TINY, TYPES, U, _dt, _out, _untouched, tm, u  # noqa: F401

pytestmark = pytest.mark.gpu


def _randn(torch, rows, cols, t, seed, std=1.0, pad=0, shift=0):
    """[rows, cols] made on the GPU; rows `pad` elements apart beyond their columns, starting `shift` elements behind an aligned address"""
    g = torch.Generator(device="cuda").manual_seed(seed)
    view = torch.full((rows * (cols + pad) + shift,), float("nan"), dtype=_dt(torch, t), device="cuda")[shift:].view(rows, cols + pad)[:, :cols]
    view.copy_((torch.randn(rows, cols, generator=g, device="cuda") * std).to(view.dtype))
    return view


def _near(torch, got, want, tol):
    """equal where the wanted value is no finite number, within tol elsewhere"""
    got = got.double()
    fin = torch.isfinite(want)
    assert got.shape == want.shape and torch.equal(torch.isfinite(got), fin), "finite in other places"
    assert torch.equal(torch.nan_to_num(got[~fin], nan=7.0), torch.nan_to_num(want[~fin], nan=7.0))
    over = torch.where(fin, (got - want).abs() - tol, torch.zeros_like(want)) if want.numel() else want
    assert over.numel() == 0 or over.max() <= 0, "off by %g more than allowed at %s" % (over.max().item(), divmod(int(over.argmax()), want.shape[-1]))


# ---- embedding ----------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("n,vocab,dim,pad,shift", [(70000, 3000, 64, 0, 0), (20000, 500, 130, 2, 2), (20000, 500, 1023, 0, 0), (9000, 100, 2056, 8, 8), (40000, 70, 36, 0, 4)])
@pytest.mark.parametrize("t,o", [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16"), ("f16", "bf16"), ("f32", "f16")])
def test_lookup_of_many_rows(tm, n, vocab, dim, pad, shift, t, o):  # noqa: F811
    torch, b2 = tm
    table = _randn(torch, vocab, dim, t, 1, 0.5, pad, shift)
    tok = torch.randint(-1, vocab, (n,), generator=torch.Generator().manual_seed(2)).int().cuda()
    full, out = _out(torch, (n, dim), o, pad, shift)
    b2.embedding_forward(out, table, tok, 1.7)
    # one product in fp32 and one rounding: the bits are determined
    want = torch.where((tok >= 0)[:, None], table[tok.long().clamp(min=0)].float() * torch.tensor(1.7, device="cuda"), torch.zeros((), device="cuda")).to(out.dtype)
    assert torch.equal(out, want)
    _untouched(torch, full, out)


@pytest.mark.parametrize("n,vocab,dim,kind", [(270000, 259, 8, "zipf"), (400000, 60000, 5, "zipf"), (400000, 3, 24, "uniform"), (310000, 200000, 2, "sorted"), (33000, 5000, 1100, "zipf")])
@pytest.mark.parametrize("t,o", [("f32", "f32"), ("bf16", "f32"), ("f16", "f16")])
def test_table_gradient_of_many_rows(tm, n, vocab, dim, kind, t, o):  # noqa: F811
    """pieces of 64 rows, tiles of more keys than the least, rows of several tiles of columns"""
    torch, b2 = tm
    r = torch.rand(n, generator=torch.Generator().manual_seed(n)).double()
    tok = ((vocab + 1.0) ** r - 1).clamp(max=vocab - 1) if kind == "zipf" else (r * vocab).floor().clamp(max=vocab - 1)
    tok = (tok.sort()[0] if kind == "sorted" else tok).int().cuda()
    tok[torch.rand(n, generator=torch.Generator().manual_seed(1)).cuda() < 0.1] = -1
    dout = _randn(torch, n, dim, t, 3, 0.3)
    full, out = _out(torch, (vocab, dim), o)
    ws = torch.full((b2.embedding_backward_workspace(n, vocab, dim),), 0xA5, dtype=torch.uint8, device="cuda")
    b2.embedding_backward(out, dout, tok, 0.75, workspace=ws)
    real = tok >= 0
    at, d = tok[real].long(), dout[real].double() * 0.75
    want = torch.zeros(vocab, dim, dtype=torch.float64, device="cuda").index_add_(0, at, d)
    mass = torch.zeros_like(want).index_add_(0, at, d.abs())
    # chains of at most 64 rows, their sums by at least 8 phases in turn, the phases in turn
    chain = 64 + math.ceil(n / 32 / 8) + 256 / 8 + 4
    count = torch.zeros(vocab, dtype=torch.float64, device="cuda").index_add_(0, at, torch.ones_like(at, dtype=torch.float64))[:, None]
    _near(torch, out, want, torch.minimum(count + 2, torch.tensor(chain, device="cuda")) * u * mass + U[o] * want.abs() + TINY[o])
    _untouched(torch, full, out)
    first = out.clone()
    b2.embedding_backward(out, dout, tok, 0.75, workspace=ws)
    assert torch.equal(first, out)


# ---- log probabilities ----------------------------------------------------------------------------------------------------------------
# rows a group of lanes (up to 1024 columns) and a warp each there; a block of 8, of 4, a warp, by the number of rows, with masks read by vectors and by bytes
FORWARD = [(500, 40, 0, 0), (300, 259, 3, 1), (301, 1000, 0, 0), (60, 3001, 0, 0), (700, 3001, 0, 3), (700, 3008, 0, 0), (2500, 1501, 1, 1), (2500, 3008, 0, 0), (3000, 1100, 0, 0)]


def _logits(torch, rows, vocab, t, pad, shift):
    """ordinary rows, and some at which a kernel can go wrong"""
    x = _randn(torch, rows, vocab, t, vocab + rows, 2.0, pad, shift)
    low = torch.finfo(x.dtype).min
    x[0, vocab // 2] = float("nan")
    x[1, vocab // 3] = float("inf")
    x[2] = -float("inf")
    x[3, 1:] = low
    x[4] = low
    x[5] = 1.5
    x[6], x[7] = x[6].sort()[0], x[7].sort(descending=True)[0]
    x[8, : vocab - 1] = -float("inf")
    x[9, vocab - 1] = float("nan")
    x[10] = x[10] + (1000 if t != "f16" else 500)
    return x


def _allowed(torch, rows, vocab, kind):
    if kind == "none":
        return None
    g = torch.Generator(device="cuda").manual_seed(9)
    if kind == "shared":
        m = (torch.rand(vocab, generator=g, device="cuda") < 0.6).to(torch.uint8) * 3
        m[vocab // 2] = 1
        return m
    m = (torch.rand(rows, vocab, generator=g, device="cuda") < 0.6).to(torch.uint8)
    m[9] = 1
    m[9, vocab - 1] = 0                                      # the row's only NaN is ruled out
    m[11] = 0
    m[12] = 0
    m[12, vocab - 1] = 1
    return m


def _definition(torch, x, mask, scale):
    """z, the largest of a row, S, log S, p, in 64 bits of z as fp32 gives it"""
    z = (x.float() * torch.tensor(scale, device="cuda")).double()
    if mask is not None:
        z = torch.where(mask.expand(z.shape) != 0, z, -math.inf)
    m = torch.where(z.isnan().any(1), math.nan, z.nan_to_num(nan=-math.inf, posinf=math.inf, neginf=-math.inf).amax(1))
    m = torch.where(m == math.inf, math.nan, m)              # a row with +inf has no log probabilities
    e = torch.where(z == -math.inf, 0.0, torch.exp(z - torch.where(m == -math.inf, 0.0, m)[:, None]))
    S = e.sum(1)
    d = torch.where(z == -math.inf, 0.0, z - m[:, None])
    return z, m, S, d, e / S[:, None]


@pytest.mark.parametrize("rows,vocab,pad,shift", FORWARD)
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("top", [0, 4, 32])
@pytest.mark.parametrize("kind,scale", [("none", 1.0), ("none", 0.7), ("shared", 1.25), ("rows", 1.0)])
def test_log_probabilities_of_many_rows(tm, rows, vocab, pad, shift, t, top, kind, scale):  # noqa: F811
    torch, b2 = tm
    x, mask = _logits(torch, rows, vocab, t, pad, shift), _allowed(torch, rows, vocab, kind)
    tok = torch.randint(-1, vocab, (rows,), generator=torch.Generator().manual_seed(rows)).cuda()
    f = lambda *s: torch.full(s, 9.5, device="cuda")  # noqa: E731
    lp, lse, H = f(rows), f(rows), f(rows)
    tt, tl = (torch.full((rows, top), -5, dtype=torch.int32, device="cuda"), f(rows, top)) if top else (None, None)
    b2.logprob_forward(x, tok.int(), lp, lse, entropy=H, top_tokens=tt, top_logprobs=tl, mask=mask, scale=scale)
    z, m, S, d, p = _definition(torch, x, mask, scale)
    none = m == -math.inf
    ls = torch.where(none, 0.0, torch.log(S))
    zt = z.gather(1, tok.clamp(min=0)[:, None])[:, 0]
    w_lse = torch.where(none, -math.inf, m + ls)
    w_lp = torch.where(tok < 0, 0.0, torch.where(m.isnan(), math.nan, torch.where(zt == -math.inf, -math.inf, zt - m - ls)))
    w_H = torch.where(none, 0.0, ls - torch.where(p > 0, p * d, 0.0).sum(1))
    # An exponential is off by 4 u and 3 u |d| (its argument); a thread adds at most 100 parts one after another, 16 more in the joins.  So log S is off by
    # 120 u + 3 u E|d|, and E |d| by that of each term: (120 + 3 |d|) u |d|; then a few roundings of what is written.
    p = torch.where(p > 0, p, 0.0)
    D = torch.where(p > 0, d.abs(), 0.0)
    Ed, Ed2 = (p * D).sum(1), (p * D * D).sum(1)
    size = lambda v: v.abs().nan_to_num(nan=0.0, posinf=0.0, neginf=0.0)  # noqa: E731
    off = u * (120 + 3 * Ed).nan_to_num()
    _near(torch, lse, w_lse, off + u * size(ls) + u * size(w_lse))
    _near(torch, lp, w_lp, off + 2 * u * size(ls) + 2 * u * size(w_lp))
    _near(torch, H, w_H, off * (1 + size(Ed)) + u * (120 * size(Ed) + 3 * size(Ed2)) + 2 * u * (size(ls) + size(Ed)))
    if top:
        order = torch.sort(z, dim=1, descending=True, stable=True)
        best, at = order.values[:, :top], order.indices[:, :top].int()
        at = torch.where(best == -math.inf, -1, at)
        assert torch.equal(tt, at)
        w_tl = torch.where(best == -math.inf, -math.inf, torch.where(m.isnan()[:, None], math.nan, best - m[:, None] - ls[:, None]))
        _near(torch, tl, w_tl, (off + 2 * u * size(ls))[:, None] + 2 * u * size(w_tl))
        assert not (tl > 0).any()
    assert not (lp > 0).any()


# as many vectors as give a thread 8 of them (4 with a mask), rows of several blocks and of parts of one
@pytest.mark.parametrize("rows,vocab,pad,shift,out_pad,out_shift", [(2500, 3001, 0, 0, 0, 0), (2500, 3008, 0, 0, 0, 0), (16000, 331, 1, 1, 2, 3), (600, 20011, 5, 1, 5, 1), (250000, 17, 0, 0, 0, 0)])
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("kind,ent,scale", [("none", False, 1.0), ("none", True, 0.7), ("shared", True, 1.25), ("rows", False, 1.0), ("rows", True, 1.0)])
def test_log_probability_gradients_of_many_rows(tm, rows, vocab, pad, shift, out_pad, out_shift, t, kind, ent, scale):  # noqa: F811
    torch, b2 = tm
    x, mask = _logits(torch, rows, vocab, t, pad, shift), _allowed(torch, rows, vocab, kind)
    x[0], x[1], x[9, vocab - 1] = 0.25, 0.5, -1.0            # NaN and inf give NaN all over: see below
    tok = torch.randint(-1, vocab, (rows,), generator=torch.Generator().manual_seed(rows)).cuda()
    z, m, S, d, p = _definition(torch, x, mask, scale)
    none = m == -math.inf
    # what a forward pass leaves, from the definition
    lse = torch.where(none, -math.inf, m + torch.log(S)).float()
    H = torch.where(none, 0.0, torch.log(S) - (p * d).nan_to_num().sum(1)).float()
    gen = torch.Generator(device="cuda").manual_seed(4)
    g, h = torch.randn(rows, generator=gen, device="cuda"), torch.randn(rows, generator=gen, device="cuda")
    full, out = _out(torch, (rows, vocab), t, out_pad, out_shift)
    kw = dict(mask=mask, scale=scale, **(dict(entropy=H, dentropy=h) if ent else {}))
    b2.logprob_backward(out, x, tok.int(), lse, g, **kw)
    logp = z - lse.double()[:, None]
    p = torch.where(z == -math.inf, 0.0, torch.exp(logp))
    want = -g.double()[:, None] * p
    size = want.abs()
    if ent:
        hd, Hd = h.double()[:, None], H.double()[:, None]
        want = want - hd * torch.where(p > 0, p * (logp + Hd), 0.0)
        size = size + hd.abs() * torch.where(p > 0, p * (logp.abs() + Hd.abs() + 1), 0.0)
    hot = torch.zeros_like(want).scatter_(1, tok.clamp(min=0)[:, None], 1.0)
    if mask is not None:
        hot = torch.where(mask.expand(hot.shape) != 0, hot, 0.0)
    want, size = want + g.double()[:, None] * hot, size + g.double().abs()[:, None] * hot
    off = ((tok < 0) | none)[:, None]
    want, size = torch.where(off, 0.0, want) * scale, torch.where(off, 0.0, size) * scale
    # log p is a rounding of itself away (z is exact), its product with log2 e and the exponential 4 u more
    far = torch.where(p > 0, logp.abs(), 0.0)
    _near(torch, out, want, u * (4 * far + 32) * size + U[t] * want.abs() + TINY[t])
    _untouched(torch, full, out)
    b2.logprob_backward(x, x, tok.int(), lse, g, **kw)        # in place
    assert torch.equal(x, out)


def test_log_probability_gradient_of_rows_without_a_number(tm):  # noqa: F811
    """NaN or +inf among a row's allowed logits: NaN in that row and nowhere else; ruled out or in padding: nothing of it"""
    torch, b2 = tm
    rows, vocab = 2500, 3001
    x = _randn(torch, rows, vocab, "bf16", 1)
    x[::5, 7], x[1::5, 8] = math.nan, math.inf
    tok = torch.full((rows,), 5, dtype=torch.int32, device="cuda")
    tok[::10] = -1
    mask = torch.ones(rows, vocab, dtype=torch.uint8, device="cuda")
    mask[1::10, 8] = 0
    lp, lse, out = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda"), torch.empty_like(x)
    b2.logprob_forward(x, tok, lp, lse, mask=mask)
    b2.logprob_backward(out, x, tok, lse, torch.ones(rows, device="cuda"), mask=mask)
    bad = torch.zeros(rows, dtype=torch.bool, device="cuda")
    bad[5::10] = bad[6::10] = True
    assert torch.equal(lse.isnan(), bad | (torch.arange(rows, device="cuda") % 10 == 0))
    assert torch.equal(out.isnan().all(1), bad) and not out[~bad].isnan().any() and (out[::10] == 0).all() and (out[1::10, 8] == 0).all()


# ---- norms around a block ------------------------------------------------------------------------------------------------------------
# rows of 16-byte vectors, several for every worker: widths that fill the threads of a row and widths that do not, a warp to 1024 threads a row
@pytest.mark.parametrize("rows,dim", [(16000, 40), (16000, 128), (12000, 200), (12000, 256), (8000, 264), (8000, 512), (8000, 1000), (8000, 1024), (3000, 1032), (3000, 2048), (1600, 2056), (1600, 4096),
                                      (1000, 4104), (1000, 8192)])
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("ln,bias,gate", [(False, False, "rows"), (True, True, "sequences"), (True, True, "none"), (False, False, "one"), (False, True, "sequences"), (True, False, "rows")])
def test_block_norm_of_many_rows(tm, rows, dim, t, ln, bias, gate):  # noqa: F811
    torch, b2 = tm
    eps, a, P = 1e-5, 0.5, 8
    x, f, dy, dh = (_randn(torch, rows, dim, t, i, s) for i, s in enumerate((2.0, 0.7, 0.3, 0.4)))
    if ln:
        f += 1.5
    gate_rows = {"none": 0, "one": 1, "sequences": P, "rows": rows}[gate]
    g = _randn(torch, gate_rows, dim, t, 8) if gate_rows else None
    gen = torch.Generator(device="cuda").manual_seed(dim)
    vec = lambda std, at: at + std * torch.randn(dim, generator=gen, device="cuda")  # noqa: E731
    w1, w2, b1, b2_ = vec(0.2, 1), vec(0.2, 1), vec(0.1, 0) if bias else None, vec(0.1, 0) if bias else None
    pat = torch.where(torch.rand(rows, generator=gen, device="cuda") < 0.2, 0, 2).to(torch.int8)
    real = (pat != 0)[:, None]
    fy, y = _out(torch, (rows, dim), t)
    fh, h = _out(torch, (rows, dim), t)
    stats = torch.full((rows, 4), math.nan, device="cuda")
    kw = dict(w_pre=w1, w_post=w2, b_post=b2_, gate=g, pat_types=pat, layer_norm=ln, residual_scale=a)
    b2.block_norm_forward(x, f, y, h, b_pre=b1, eps=eps, stats=stats, **kw)
    eps = float(torch.tensor(eps))
    X, F, W1, W2 = x.double(), f.double(), w1.double(), w2.double()
    B1, B2 = (b1.double(), b2_.double()) if bias else (torch.zeros(dim, device="cuda").double(),) * 2
    G = 1.0 if g is None else g.double()[torch.arange(rows, device="cuda") % gate_rows]
    G = torch.ones(1, 1, device="cuda").double() if g is None else G

    def norm(v):
        mean = v.mean(1) if ln else torch.zeros(rows, device="cuda").double()
        return mean, 1 / torch.sqrt(((v - mean[:, None]) ** 2).mean(1) + eps)

    def own(v, r):      # as in test_block_norm: a mean of squares of at most 32 terms a thread and 10 steps between them
        return 60 * u * (((v - v.mean(1, keepdim=True) * ln) * r[:, None]).abs() + (v.abs().mean(1) * r)[:, None] * ln)

    m2, r2 = norm(F)
    n = (F - m2[:, None]) * r2[:, None] * W2 + B2
    want = torch.where(real, X + a * G * n, 0.0)
    _near(torch, y, want, real * (4 * u * (X.abs() + (a * G * n).abs()) + (a * G).abs() * (own(F, r2) * W2.abs() + u * B2.abs())) + U[t] * want.abs() + TINY[t])
    Y = y.double()
    m1, r1 = norm(Y)
    want = torch.where(real, (Y - m1[:, None]) * r1[:, None] * W1 + B1, 0.0)
    _near(torch, h, want, real * (own(Y, r1) * W1.abs() + 4 * u * (want.abs() + B1.abs())) + U[t] * want.abs() + TINY[t])
    on = real[:, 0]
    S = stats.double()
    for k, (v, ref, size) in enumerate([(F, m2, F.abs().mean(1)), (F, r2, r2), (Y, m1, Y.abs().mean(1)), (Y, r1, r1)]):
        extra = 0.0 if k % 2 == 0 else ref * (60 * u * v.abs().mean(1) * ref) ** 2
        _near(torch, S[on, k], ref[on], (60 * u * size + extra)[on] + 1e-300)
    assert (S[~on] == 0).all()
    _untouched(torch, fy, y)
    _untouched(torch, fh, h)

    # Backward: y and the statistics from the definition (y as the type holds it), not from what the forward pass left
    stats = torch.where(real, torch.stack([m2, r2, m1, r1], 1), 0.0).float()
    outs = {k: _out(torch, (rows, dim), t) for k in ("dx", "df")}
    dgate = _out(torch, (gate_rows, dim), t) if gate_rows else (None, None)
    sums = {k: torch.full((dim,), math.nan, device="cuda") if bias or k[1] == "w" else None for k in ("dw_pre", "db_pre", "dw_post", "db_post")}
    ws = torch.full((b2.block_norm_backward_workspace(rows, dim, gate_rows),), 0xA5, dtype=torch.uint8, device="cuda")
    call = lambda: b2.block_norm_backward(outs["dx"][1], outs["df"][1], dy, dh, y, f, stats, dgate=dgate[1], workspace=ws, **sums, **kw)  # noqa: E731
    call()
    DY, DH = torch.where(real, dy.double(), 0.0), torch.where(real, dh.double(), 0.0)
    s2, q2, s1, q1 = (c[:, None] for c in stats.double().unbind(1))
    v1, v2 = (Y - s1) * q1, (F - s2) * q2

    def back(d, v, w, r):
        wd = d * w
        grad = r * (wd - v * (wd * v).mean(1, keepdim=True) - (wd.mean(1, keepdim=True) if ln else 0.0))
        return grad, r * (wd.abs() + v.abs() * (wd * v).abs().mean(1, keepdim=True) + (wd.abs().mean(1, keepdim=True) if ln else 0.0))

    grad, size = back(DH, v1, W1, q1)
    dt, M = DY + grad, DY.abs() + size                       # what the terms of dt add up to; every one is off by 100 u of its size
    dn, Mn = a * G * dt, (a * G).abs() * M
    dF, _ = back(dn, v2, W2, q2)
    _, MF = back(Mn, v2.abs(), W2.abs(), q2)
    _near(torch, outs["dx"][1], torch.where(real, dt, 0.0), real * (100 * u * M + U[t] * dt.abs()) + TINY[t])
    _near(torch, outs["df"][1], torch.where(real, dF, 0.0), real * (300 * u * MF + U[t] * dF.abs()) + TINY[t])
    n, Nn = v2 * W2 + B2, (v2 * W2).abs() + B2.abs()
    if gate_rows:
        per = lambda v: torch.where(real, v, 0.0).view(-1, gate_rows, dim).sum(0)  # noqa: E731
        want, size = per(a * dt * n), per(a * M * Nn)
        # a worker adds its rows in turn, at most rows / 148 of them (one block a multiprocessor), the join 32 chains
        terms = min(rows / gate_rows, rows / 148 + 2) + 100
        _near(torch, dgate[1], want, (300 + terms) * u * size + U[t] * want.abs() + TINY[t])
        _untouched(torch, *dgate)
    for k, v, s in (("dw_pre", DH * v1, (DH * v1).abs()), ("db_pre", DH, DH.abs()), ("dw_post", dn * v2, Mn * v2.abs()), ("db_post", dn, Mn)):
        if sums[k] is not None:
            _near(torch, sums[k], torch.where(real, v, 0.0).sum(0), (300 + rows / 148 + 100) * u * torch.where(real, s, 0.0).sum(0) + 1e-300)
    first = [v.clone() for v in (outs["dx"][1], outs["df"][1], *(s for s in sums.values() if s is not None))]
    call()
    assert all(torch.equal(p, q) for p, q in zip(first, (outs["dx"][1], outs["df"][1], *(s for s in sums.values() if s is not None))))
    for k in outs:
        _untouched(torch, *outs[k])


@pytest.mark.parametrize("t,dim", [("bf16", 512), ("bf16", 2048), ("f32", 512), ("f16", 333), ("f32", 3000)])
def test_block_norm_parts_of_many_rows(tm, t, dim):  # noqa: F811
    """a norm alone, no norm behind, in place, without statistics; gradients of parts, in place: the same bits as of the whole"""
    torch, b2 = tm
    rows = 6000
    x, f, dy, dh = (_randn(torch, rows, dim, t, i, s) for i, s in enumerate((2.0, 0.7, 0.3, 0.4)))
    g = _randn(torch, 6, dim, t, 8)
    w1, w2 = torch.rand(dim, device="cuda") + 0.5, torch.rand(dim, device="cuda") + 0.5
    new = lambda: torch.full((rows, dim), math.nan, dtype=x.dtype, device="cuda")  # noqa: E731
    st, st2 = torch.empty(rows, 4, device="cuda"), torch.empty(rows, 4, device="cuda")
    kw = dict(w_post=w2, gate=g, residual_scale=0.5)
    y, h, y2, h2, h3 = new(), new(), x.clone(), new(), new()
    b2.block_norm_forward(x, f, y, h, stats=st, w_pre=w1, **kw)
    b2.block_norm_forward(y2, f, y2, h2, w_pre=w1, **kw)
    assert torch.equal(y2, y) and torch.equal(h2, h)
    y3 = new()
    b2.block_norm_forward(x, f, y3, None, **kw)
    b2.block_norm_forward(y, None, None, h3, stats=st2, w_pre=w1)
    assert torch.equal(y3, y) and torch.equal(h3, h) and torch.equal(st2[:, 2:], st[:, 2:]) and (st2[:, :2] == 0).all()
    ws = torch.empty(b2.block_norm_backward_workspace(rows, dim, 6), dtype=torch.uint8, device="cuda")
    dx, df, dw, dg = new(), new(), torch.empty(dim, device="cuda"), torch.empty_like(g)
    b2.block_norm_backward(dx, df, dy, dh, y, f, st, dw_pre=dw, dgate=dg, w_pre=w1, workspace=ws, **kw)
    a, c = dy.clone(), dh.clone()
    b2.block_norm_backward(a, c, a, c, y, f, st, w_pre=w1, workspace=ws, **kw)
    assert torch.equal(a, dx) and torch.equal(c, df)
    e = new()
    b2.block_norm_backward(e, None, dy, dh, y, None, st, w_pre=w1, workspace=ws)
    assert torch.equal(e, dx)
    only = torch.empty_like(g)
    b2.block_norm_backward(None, None, dy, dh, y, f, st, dgate=only, w_pre=w1, workspace=ws, **kw)
    assert torch.equal(only, dg)


@pytest.mark.parametrize("t,dim", [("bf16", 512), ("f16", 333), ("f32", 2000)])
def test_block_norm_gradients_in_place_of_a_gate_for_every_frame(tm, t, dim):  # noqa: F811
    torch, b2 = tm
    rows = 5000
    y, f, dy, dh = (_randn(torch, rows, dim, t, i, s) for i, s in enumerate((2.0, 0.7, 0.3, 0.4)))
    g = _randn(torch, rows, dim, t, 8)
    st = torch.rand(rows, 4, device="cuda")
    ws = torch.empty(b2.block_norm_backward_workspace(rows, dim, rows), dtype=torch.uint8, device="cuda")
    run = lambda dx, df, gate, dgate: b2.block_norm_backward(dx, df, dy, dh, y, f, st, gate=gate, dgate=dgate, workspace=ws)  # noqa: E731
    dx, df, dg = (torch.empty_like(y) for _ in range(3))
    run(dx, df, g, dg)
    a, b, c, other = g.clone(), g.clone(), g.clone(), torch.empty_like(y)
    run(a, other, a, None)
    run(other, b, b, None)
    run(other, torch.empty_like(y), c, c)
    assert torch.equal(a, dx) and torch.equal(b, df) and torch.equal(c, dg)
