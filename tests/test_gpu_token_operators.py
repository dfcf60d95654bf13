"""GPU tests of the token operators (include/b2lstm.h: b2_embedding_*, b2_block_norm_*, b2_logprob_*, b2_gradient_*) against plain
implementations in 64 bits on the host.

Tolerances are error bounds, written down per case: u = 2^-24 is the unit roundoff of fp32, U[type] that of a tensor's type (the one rounding
of a result), TINY[type] half of its smallest number.  A sum of n terms x in fp32 is off by at most (n + 1) u sum|x| in any order."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
u = 2.0 ** -24
U = {"f32": 0.0, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}      # fp32 results: covered by the bound of the arithmetic
TINY = {"f32": 2.0 ** -149, "bf16": 2.0 ** -134, "f16": 2.0 ** -25}
TYPES = ["f32", "bf16", "f16"]


@pytest.fixture(scope="module")
def tm():
    import torch
    import b2lstm
    return torch, b2lstm


def _dt(torch, t):
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[t]


def _host(t):
    return t.detach().double().cpu().numpy()


def _rand(torch, shape, t, seed, std=1.0, pad=0, shift=0):
    """[rows, cols] on the GPU; rows `pad` elements apart beyond their columns and starting `shift` elements behind an aligned address"""
    g = torch.Generator().manual_seed(seed)
    rows, cols = shape
    full = torch.full((rows * (cols + pad) + shift,), float("nan"), dtype=_dt(torch, t), device="cuda")
    view = full[shift:shift + rows * (cols + pad)].view(rows, cols + pad)[:, :cols]
    view.copy_((torch.randn(rows, cols, generator=g) * std).to(_dt(torch, t)).cuda())
    return view


def _out(torch, shape, t, pad=0, shift=0):
    """the same, filled with NaN: what a call does not write shows; and what lies between the rows has to stay NaN"""
    rows, cols = shape
    full = torch.full((rows * (cols + pad) + shift + 8,), float("nan"), dtype=_dt(torch, t), device="cuda")
    return full, full[shift:shift + rows * (cols + pad)].view(rows, cols + pad)[:, :cols]


def _untouched(torch, full, view):
    keep = full.clone()
    n = view.numel()
    inside = torch.isnan(view).sum().item()
    assert torch.isnan(keep).sum().item() == keep.numel() - n + inside


def _close(got, want, tol):
    got, want, tol = np.asarray(got, np.float64), np.asarray(want, np.float64), np.broadcast_to(tol, np.shape(want))
    assert got.shape == want.shape
    fin = np.isfinite(want)
    assert np.array_equal(fin, np.isfinite(got)), "finite in other places"
    assert np.array_equal(got[~fin & ~np.isnan(want)], want[~fin & ~np.isnan(want)]) and np.array_equal(np.isnan(got), np.isnan(want))
    over = np.abs(got - want)[fin] - tol[fin]
    assert over.size == 0 or over.max() <= 0, "off by %g, allowed %g" % (np.abs(got - want)[fin].flat[over.argmax()], tol[fin].flat[over.argmax()])


# ---- embedding ------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("n,vocab,dim,pad,shift", [(1, 1, 1, 0, 0), (7, 5, 3, 2, 1), (64, 300, 512, 0, 0), (33, 40, 1077, 0, 0), (100, 17, 24, 8, 8),
                                                   (70, 9, 130, 0, 3), (5, 4, 4100, 0, 0)])
@pytest.mark.parametrize("t,o", [("f32", "f32"), ("bf16", "f32"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16"), ("f16", "bf16")])
def test_embedding_forward(tm, n, vocab, dim, pad, shift, t, o):
    torch, b2 = tm
    table = _rand(torch, (vocab, dim), t, 1, 0.5, pad, shift)
    tok = torch.randint(-1, vocab, (n,), generator=torch.Generator().manual_seed(2)).int()
    full, out = _out(torch, (n, dim), o, pad, shift)
    b2.embedding_forward(out, table, tok.cuda(), 1.7)
    s = float(np.float32(1.7))
    want = np.where(tok.numpy()[:, None] >= 0, _host(table)[tok.clamp(min=0).numpy()] * s, 0.0)
    _close(_host(out), want, (U[o] + 2 * u) * np.abs(want) + TINY[o])
    _untouched(torch, full, out)


def test_embedding_forward_marks_tokens_beyond_the_table(tm):
    torch, b2 = tm
    out = torch.zeros(4, 5, device="cuda")
    b2.embedding_forward(out, torch.ones(3, 5, device="cuda"), torch.tensor([2, 3, -7, 2 ** 31 - 1], dtype=torch.int32, device="cuda"))
    got = _host(out)
    assert (got[0] == 1).all() and np.isnan(got[1]).all() and (got[2] == 0).all() and np.isnan(got[3]).all()


def _embedding_gradient(dout, tok, vocab, scale):
    want, mass, count = np.zeros((vocab, dout.shape[1])), np.zeros((vocab, dout.shape[1])), np.zeros(vocab)
    for r, v in enumerate(tok):
        if 0 <= v < vocab:
            want[v] += dout[r] * scale
            mass[v] += np.abs(dout[r]) * abs(scale)
            count[v] += 1
    return want, mass, count


# around the borders of a piece (8, 16, 32 rows), of the one-block sort (4096), of its digits (512) and of a tile (2048)
@pytest.mark.parametrize("n,vocab,dim,kind", [(1, 1, 1, "uniform"), (7, 3, 5, "uniform"), (8, 2, 8, "one"), (9, 2, 8, "one"), (300, 259, 128, "zipf"),
                                              (1516, 511, 12, "zipf"), (1000, 512, 33, "uniform"), (2000, 70000, 4, "zipf"), (4096, 300, 6, "zipf"),
                                              (4097, 300, 6, "zipf"), (5000, 1, 40, "one"), (9000, 262144, 3, "zipf"), (6000, 1000, 260, "padding"),
                                              (20000, 50, 16, "sorted"), (40000, 5000, 2, "zipf"), (4500, 4, 130, "none"), (33, 4, 2050, "uniform")])
@pytest.mark.parametrize("t,o", [("f32", "f32"), ("bf16", "f32"), ("f16", "f16")])
def test_embedding_backward(tm, n, vocab, dim, kind, t, o):
    torch, b2 = tm
    r = np.random.default_rng(n + vocab)
    if kind == "zipf":
        tok = np.minimum((vocab + 1.0) ** r.random(n) - 1, vocab - 1).astype(np.int32)
    elif kind == "one":
        tok = np.full(n, vocab - 1, np.int32)
    elif kind == "none":
        tok = np.where(r.random(n) < 0.5, -1, vocab).astype(np.int32)      # padding, and tokens beyond the table
    else:
        tok = r.integers(0, vocab, n).astype(np.int32)
    if kind == "padding":
        tok[r.random(n) < 0.7] = -1
    if kind == "sorted":
        tok = np.sort(tok)
    dout = _rand(torch, (n, dim), t, 3, 0.3)
    tokens = torch.from_numpy(tok).cuda()
    ws = torch.full((b2.embedding_backward_workspace(n, vocab, dim),), 0xA5, dtype=torch.uint8, device="cuda")
    full, out = _out(torch, (vocab, dim), o)
    b2.embedding_backward(out, dout, tokens, 0.75, workspace=ws)
    want, mass, count = _embedding_gradient(_host(dout), tok, vocab, 0.75)
    _close(_host(out), want, (count[:, None] + 2) * u * mass + U[o] * np.abs(want) + TINY[o])
    _untouched(torch, full, out)
    first = out.clone()
    out.fill_(7.0)
    b2.embedding_backward(out, dout, tokens, 0.75, workspace=ws)       # the workspace as the first call left it
    assert torch.equal(out, first)
    # added to what is there; rows without a frame keep their bits
    out.fill_(1.0)
    b2.embedding_backward(out, dout, tokens, 0.75, accumulate=True, workspace=ws)
    _close(_host(out), want + 1, (count[:, None] + 3) * u * (mass + 1) * (count[:, None] > 0) + U[o] * np.abs(want + 1) * (count[:, None] > 0) + TINY[o])


@pytest.mark.parametrize("dim,pad,shift", [(16, 16, 8), (24, 0, 1), (7, 2, 3)])
def test_embedding_backward_over_strides_and_alignments(tm, dim, pad, shift):
    torch, b2 = tm
    tok = np.random.default_rng(5).integers(-1, 20, 200).astype(np.int32)
    for t, o in (("bf16", "bf16"), ("f32", "f32"), ("bf16", "f32")):
        dout = _rand(torch, (200, dim), t, 4, 1.0, pad, shift)
        full, out = _out(torch, (20, dim), o, pad, shift)
        ws = torch.empty(b2.embedding_backward_workspace(200, 20, dim), dtype=torch.uint8, device="cuda")
        b2.embedding_backward(out, dout, torch.from_numpy(tok).cuda(), -1.25, workspace=ws)
        want, mass, count = _embedding_gradient(_host(dout), tok, 20, -1.25)
        _close(_host(out), want, (count[:, None] + 2) * u * mass + U[o] * np.abs(want))
        _untouched(torch, full, out)


def test_embedding_of_no_tokens(tm):
    torch, b2 = tm
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    out = torch.full((5, 4), 3.0, device="cuda")
    b2.embedding_forward(torch.zeros(0, 4, device="cuda"), out, none)
    b2.embedding_backward(out, torch.zeros(0, 4, device="cuda"), none, accumulate=True)
    assert (out == 3).all()
    b2.embedding_backward(out, torch.zeros(0, 4, device="cuda"), none)
    assert (out == 0).all()


def test_embedding_gradient_against_differences(tm):
    """<dtable, v> against the change of sum(dout * out) along v: the operator is linear, so only rounding separates them"""
    torch, b2 = tm
    tok = torch.randint(-1, 30, (500,), generator=torch.Generator().manual_seed(1)).int().cuda()
    table, v, dout = (_rand(torch, s, "f32", i) for i, s in enumerate([(30, 20), (30, 20), (500, 20)]))
    outs = []
    for t in (table + v, table - v):
        o = torch.empty(500, 20, device="cuda")
        b2.embedding_forward(o, t.contiguous(), tok, 0.5)
        outs.append(_host(o))
    grad = torch.empty(30, 20, device="cuda")
    b2.embedding_backward(grad, dout, tok, 0.5, workspace=torch.empty(b2.embedding_backward_workspace(500, 30, 20), dtype=torch.uint8, device="cuda"))
    change = ((outs[0] - outs[1]) / 2 * _host(dout)).sum()
    slack = 8 * u * (np.abs(outs[0]) + np.abs(outs[1]) + 1).sum() * np.abs(_host(dout)).max() + 600 * u * np.abs(_host(dout)).sum() * np.abs(_host(v)).max()
    assert abs(change - (_host(grad) * _host(v)).sum()) <= slack


# ---- log probabilities ----------------------------------------------------------------------------------------------------------------
def _logprob(x, mask, tok, scale, top):
    """plain form in 64 bits"""
    z = x * scale
    if mask is not None:
        z = np.where(np.broadcast_to(mask, z.shape) != 0, z, -np.inf)
    with np.errstate(all="ignore"):
        m = z.max(1, keepdims=True)
        e = np.where(z == -np.inf, 0.0, np.exp(z - np.where(m == -np.inf, 0.0, m)))
        s = e.sum(1)
        lse = m[:, 0] + np.log(s)
        lp = (z - m) - np.log(s)[:, None]                  # z - lse would lose log s beside a large m, in 64 bits too
        p = np.where(z == -np.inf, 0.0, np.exp(lp))
        H = -(p * np.where(p > 0, lp, 0.0)).sum(1)
    H = np.where(np.isnan(lse), np.nan, np.where(lse == -np.inf, 0.0, H))
    given = np.array([0.0 if t < 0 else np.nan if t >= z.shape[1] else (-np.inf if z[r, t] == -np.inf and not np.isnan(lse[r]) else z[r, t] - lse[r])
                      for r, t in enumerate(tok)])
    order = np.argsort(np.where(np.isnan(z), -np.inf, -z), axis=1, kind="stable")[:, :top]      # NaN first, then by value, then by index
    best = np.take_along_axis(z, order, 1)
    pad = top - order.shape[1]
    if pad > 0:
        order, best = np.pad(order, ((0, 0), (0, pad))), np.pad(best, ((0, 0), (0, pad)), constant_values=-np.inf)
    with np.errstate(all="ignore"):
        return z, lse, given, H, np.where(best == -np.inf, -1, order), np.where(best == -np.inf, -np.inf, best - lse[:, None])


def _run_logprob(tm, x, tok, mask, scale, top, entropy=True):
    torch, b2 = tm
    rows = x.shape[0]
    f = lambda *s: torch.full(s, 9.5, device="cuda")  # noqa: E731
    lp, lse, H = f(rows), f(rows), f(rows) if entropy else None
    tt, tl = (torch.full((rows, top), -5, dtype=torch.int32, device="cuda"), f(rows, top)) if top else (None, None)
    b2.logprob_forward(x, torch.as_tensor(tok, dtype=torch.int32).cuda(), lp, lse, entropy=H, top_tokens=tt, top_logprobs=tl, mask=mask, scale=scale)
    return lp, lse, H, tt, tl


def _check_logprob(tm, x, tok, mask, scale, top):
    torch, b2 = tm
    lp, lse, H, tt, tl = _run_logprob(tm, x, tok, mask, scale, top)
    s = float(np.float32(scale))
    # the kernel ranks z as fp32 gives it
    z32 = (x.float().cpu().numpy() * np.float32(s)).astype(np.float64)
    z, w_lse, w_lp, w_H, w_tt, w_tl = _logprob(z32, None if mask is None else mask.cpu().numpy(), tok, 1.0, top)
    big = np.abs(np.where(np.isfinite(z), z, 0.0)).max(1)
    # lse: hardware exponential 4 u, argument 3 u |d| with |d| <= 2 max|z|, sums of at most 100 partial steps, and its own rounding
    tol = u * (8 * big + 200)
    _close(_host(lse), w_lse, tol)
    _close(_host(lp), w_lp, tol + u * np.abs(np.where(np.isfinite(w_lp), w_lp, 0)))
    _close(_host(H), w_H, tol * (2 + 2 * big))
    if top:
        assert np.array_equal(tt.cpu().numpy(), w_tt)
        _close(_host(tl), w_tl, (tol + u * (big + 1))[:, None] * 2)


# widths around a warp, the limits of its registers (128, 320, 576, 1024), one vector, one batch of a block (8192 entries of 16 bits)
@pytest.mark.parametrize("rows,vocab,pad,shift", [(1, 1, 0, 0), (3, 2, 1, 1), (9, 31, 0, 0), (8, 33, 0, 1), (17, 128, 0, 0), (5, 129, 2, 0), (11, 259, 0, 0), (6, 320, 0, 0),
                                                  (6, 321, 0, 0), (4, 577, 0, 0), (4, 1024, 0, 0), (4, 1025, 0, 0), (3, 1025, 7, 5), (2, 4099, 1, 3),
                                                  (3, 8192, 0, 0), (3, 8193, 0, 0), (2, 20011, 5, 1), (1, 131072, 0, 0), (1, 100003, 0, 2), (200, 9000, 0, 0), (400, 2500, 0, 0)])
@pytest.mark.parametrize("t,top", [("f32", 0), ("f32", 5), ("bf16", 1), ("bf16", 8), ("f16", 32)])
def test_logprob_forward(tm, rows, vocab, pad, shift, t, top):
    torch, b2 = tm
    x = _rand(torch, (rows, vocab), t, vocab + rows, 3.0, pad, shift)
    tok = np.random.default_rng(rows).integers(-1, vocab, rows)
    _check_logprob(tm, x, tok, None, 1.0, top)
    _check_logprob(tm, x, tok, None, 0.37, top)


@pytest.mark.parametrize("vocab", [5, 200, 1000, 1500, 9001, 70000])
@pytest.mark.parametrize("kind", ["shared", "rows", "strided"])
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_logprob_forward_with_masks(tm, vocab, kind, t):
    torch, b2 = tm
    rows = 6
    x = _rand(torch, (rows, vocab), t, 8, 2.0, 3, 1)
    r = np.random.default_rng(vocab)
    if kind == "shared":
        mask = torch.from_numpy((r.random(vocab) < 0.5).astype(np.uint8)).cuda()
    else:
        m = (r.random((rows, vocab)) < 0.5).astype(np.uint8)
        m[1] = 0                                          # nothing allowed
        m[2] = 0
        m[2, vocab - 1] = 1                               # one token
        m[3] = 2                                          # everything
        full = torch.zeros(rows, vocab + (13 if kind == "strided" else 0), dtype=torch.uint8, device="cuda")
        mask = full[:, :vocab]
        mask.copy_(torch.from_numpy(m).cuda())
    _check_logprob(tm, x, r.integers(-1, vocab, rows), mask, 1.25, 4)


@pytest.mark.parametrize("vocab", [40, 1000, 5000, 50000])
def test_logprob_forward_of_special_rows(tm, vocab):
    """the type's lowest value as a mask, -inf, +inf and NaN, equal values, ordered values, -0 and 0"""
    torch, b2 = tm
    x = np.random.default_rng(vocab).standard_normal((12, vocab)).astype(np.float32)
    low = np.finfo(np.float32).min
    x[0, 1:] = low
    x[1, :] = low                                         # every entry: all tokens are equally likely
    x[2, :] = -np.inf
    x[3, 1:] = -np.inf
    x[4, vocab // 2] = np.nan
    x[5, vocab // 2] = np.inf
    x[6, :] = 1.5
    x[7] = np.sort(x[7])
    x[8] = np.sort(x[8])[::-1]
    x[9, ::2], x[9, 1::2] = 0.0, -0.0
    x[10, :] = -np.inf
    x[10, vocab - 3] = np.nan
    x[11, : vocab - 1] = 3e38
    x[11, vocab - 1] = -3e38
    tok = np.array([0, 3, 1, 5, 0, 0, 2, 1, 0, 4, 0, vocab - 1])
    xt = torch.from_numpy(x).cuda()
    lp, lse, H, tt, tl = _run_logprob(tm, xt, tok, None, 1.0, 6)
    _, w_lse, w_lp, w_H, w_tt, w_tl = _logprob(x.astype(np.float64), None, tok, 1.0, 6)
    w_lse[[4, 5, 10]] = w_lp[[4, 5, 10]] = w_H[[4, 5, 10]] = np.nan
    w_tl[[4, 5, 10]] = np.where(w_tt[[4, 5, 10]] >= 0, np.nan, -np.inf)
    big = np.array([1e1] * 12)
    big[[0, 1, 11]] = 3.4e38
    tol = u * (8 * big + 200)
    _close(_host(lse), w_lse, tol)
    with np.errstate(all="ignore"):
        # row 11: 3e38 and -3e38 are further apart than fp32 reaches
        w_lp = w_lp.astype(np.float32).astype(np.float64)
    _close(_host(lp), w_lp, tol)
    # a row of equal values has the entropy log n whatever their size; elsewhere the differences to the maximum are small or weightless
    _close(_host(H), w_H, u * 600)
    assert np.array_equal(tt.cpu().numpy(), w_tt)


# a row a group of lanes, a warp, a block of 8, of 4 and of 1 warps, and a cluster
ROW_KERNELS = [(64, 40), (64, 3000), (700, 1500), (2500, 1500), (3, 70001)]


@pytest.mark.parametrize("rows,vocab", ROW_KERNELS)
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("top", [0, 3])
def test_a_certain_token_has_the_log_probability_0(tm, rows, vocab, t, top):
    """one token allowed, its logit large and the scale no power of two: z is one number everywhere, so z - lse is 0 and so are entropy and gradient"""
    torch, b2 = tm
    x = _rand(torch, (rows, vocab), t, 3, 4.0)
    tok = np.random.default_rng(vocab).integers(0, vocab, rows)
    at = torch.from_numpy(tok).cuda()
    r = torch.arange(rows, device="cuda")
    x[r, at] = (torch.rand(rows, generator=torch.Generator().manual_seed(4)) * 7000 - 2000).cuda().to(x.dtype)
    mask = torch.zeros(rows, vocab, dtype=torch.uint8, device="cuda")
    mask[r, at] = 1
    lp, lse, H, tt, tl = _run_logprob(tm, x, tok, mask, 0.7, top)
    assert (lp == 0).all() and (H == 0).all() and torch.equal(lse, x[r, at].float() * np.float32(0.7))
    if top:
        assert torch.equal(tt[:, 0].long(), at) and (tl[:, 0] == 0).all() and (tt[:, 1:] == -1).all()
    d = torch.full_like(x, 9.0)
    b2.logprob_backward(d, x, torch.from_numpy(tok).int().cuda(), lse, torch.ones(rows, device="cuda"), mask=mask, scale=0.7)
    assert (d == 0).all()


@pytest.mark.parametrize("rows,vocab", ROW_KERNELS)
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("top", [0, 4])
@pytest.mark.parametrize("masked", [False, True])
def test_logprob_of_large_logits_close_together(tm, rows, vocab, t, top, masked):
    """logits near 9000 a few apart: what is lost must follow from their differences, not from their size"""
    torch, b2 = tm
    x = _rand(torch, (rows, vocab), t, 6, 2.0)
    x.copy_((x.float().clamp(-8, 8) + 9000).to(x.dtype))
    tok = np.random.default_rng(vocab).integers(0, vocab, rows)
    mask = None
    if masked:
        m = (np.random.default_rng(7).random(vocab) < 0.7).astype(np.uint8)
        m[[0, vocab - 1]] = 1
        mask = torch.from_numpy(m).cuda()
    lp, lse, H, tt, tl = _run_logprob(tm, x, tok, mask, 0.7, top)
    z = (x.float().cpu().numpy() * np.float32(0.7)).astype(np.float64)
    if masked:
        z = np.where(m != 0, z, -np.inf)
    best = z.max(1, keepdims=True)
    S = np.exp(z - best).sum(1)
    # z - m is exact to a rounding of itself: bf16 logits near 9000 are 64 apart (scaled 45), the others within 16 + 8.  The exponential is off by 4 u and by 3 u |d| of its argument
    # (weights e^d |d| <= 1/e beyond 1), sums of 100 partial steps, log S and the difference by a rounding each
    want = np.where(z[np.arange(rows), tok] == -np.inf, -np.inf, z[np.arange(rows), tok] - best[:, 0] - np.log(S))
    size = np.where(np.isfinite(want), np.abs(want), 0.0)
    _close(_host(lp), want, u * (200 + 2 * size))
    assert (lp <= 0).all()
    if top:
        order = np.argsort(-z, axis=1, kind="stable")[:, :top]
        assert np.array_equal(tt.cpu().numpy(), order)
        w = np.take_along_axis(z, order, 1) - best - np.log(S)[:, None]
        _close(_host(tl), w, u * (200 + 2 * np.abs(w)))
        assert (tl <= 0).all()


def test_logprob_forward_marks_tokens_beyond_the_vocabulary(tm):
    torch, b2 = tm
    for vocab in (10, 3000):
        x = torch.zeros(3, vocab, device="cuda")
        lp, lse, H, _, _ = _run_logprob(tm, x, np.array([vocab, -2, 0]), None, 1.0, 0)
        got = _host(lp)
        assert np.isnan(got[0]) and got[1] == 0 and abs(got[2] + math.log(vocab)) < 1e-5
        assert np.abs(_host(lse) - math.log(vocab)).max() < 1e-5


def test_logprob_forward_is_the_same_every_time_and_on_another_stream(tm):
    torch, b2 = tm
    for rows, vocab in ((4, 60000), (300, 3000), (50, 200)):
        x = _rand(torch, (rows, vocab), "bf16", 3, 1.0)
        tok = np.arange(rows) % vocab
        first = _run_logprob(tm, x, tok, None, 1.0, 7)
        st = torch.cuda.Stream()
        tokens = torch.as_tensor(tok, dtype=torch.int32).cuda()
        out = [torch.empty_like(t) for t in first]
        torch.cuda.synchronize()
        b2.logprob_forward(x, tokens, out[0], out[1], entropy=out[2], top_tokens=out[3], top_logprobs=out[4], stream=st.cuda_stream)
        st.synchronize()
        for a, b in zip(first, out):
            assert torch.equal(a, b)


def _logprob_gradient(z, lse, H, tok, g, h, scale):
    """formula in 64 bits, and a bound of the terms' size for the tolerance"""
    with np.errstate(all="ignore"):
        lp = z - lse[:, None]
        p = np.where(z == -np.inf, 0.0, np.exp(lp))
        d = -g[:, None] * p
        size = np.abs(d)
        if h is not None:
            e = np.where(p > 0, p * (lp + H[:, None]), 0.0)
            d = d - h[:, None] * e
            size = size + np.abs(h[:, None]) * np.where(p > 0, p * (np.abs(lp) + np.abs(H[:, None]) + 1), 0.0)
    for r, t in enumerate(tok):
        if t >= 0:
            d[r, t] += g[r]
            size[r, t] += abs(g[r])
    none = (np.asarray(tok) < 0) | (lse == -np.inf)
    d[none] = size[none] = 0.0
    return d * scale, size * scale


@pytest.mark.parametrize("rows,vocab,pad,shift", [(1, 1, 0, 0), (5, 7, 2, 1), (40, 259, 0, 0), (9, 1024, 0, 0), (4, 4097, 0, 0), (3, 8193, 5, 3), (2, 70001, 0, 1)])
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("mask_kind,ent", [("none", False), ("none", True), ("shared", True), ("rows", False)])
def test_logprob_backward(tm, rows, vocab, pad, shift, t, mask_kind, ent):
    torch, b2 = tm
    r = np.random.default_rng(vocab)
    x = _rand(torch, (rows, vocab), t, 5, 2.0, pad, shift)
    tok = r.integers(-1, vocab, rows)
    mask = None
    if mask_kind != "none":
        m = (r.random((vocab,) if mask_kind == "shared" else (rows, vocab)) < 0.6).astype(np.uint8)
        for k, v in enumerate(tok):
            m[(v,) if mask_kind == "shared" else (k, v)] = 1
        if mask_kind == "rows":
            m[0] = 0
            tok[0] = -1
        mask = torch.from_numpy(m).cuda()
    scale = 1.25
    lp, lse, H, _, _ = _run_logprob(tm, x, tok, mask, scale, 0)
    g, h = (torch.from_numpy(r.standard_normal(rows).astype(np.float32)).cuda() for _ in range(2))
    tokens = torch.as_tensor(tok, dtype=torch.int32).cuda()
    full, d = _out(torch, (rows, vocab), t, pad, shift)
    kw = dict(entropy=H, dentropy=h) if ent else {}
    b2.logprob_backward(d, x, tokens, lse, g, mask=mask, scale=scale, **kw)
    z = (x.float().cpu().numpy() * np.float32(scale)).astype(np.float64)
    if mask is not None:
        z = np.where(np.broadcast_to(mask.cpu().numpy(), z.shape) != 0, z, -np.inf)
    want, size = _logprob_gradient(z, _host(lse), _host(H), tok, _host(g), _host(h) if ent else None, scale)
    big = np.abs(np.where(np.isfinite(z), z, 0.0)).max(1, keepdims=True) + np.log(vocab)
    # p: rounding of log p (2 u (|z| + |lse|)), of its product with log2 e and of the exponential; then a few operations
    _close(_host(d), want, u * (8 * big + 32) * size + U[t] * np.abs(want) + TINY[t])
    _untouched(torch, full, d)
    keep = d.clone()
    b2.logprob_backward(x, x, tokens, lse, g, mask=mask, scale=scale, **kw)        # in place
    assert torch.equal(x, keep)


def test_logprob_backward_with_rows_apart_differently(tm):
    """gradient and logits whose rows do not start at the same place of a 16-byte vector"""
    torch, b2 = tm
    x = _rand(torch, (5, 1003), "bf16", 5, 2.0, 5, 1)
    tok = np.array([3, 0, 1002, -1, 77])
    lp, lse, H, _, _ = _run_logprob(tm, x, tok, None, 1.0, 0)
    g = torch.ones(5, device="cuda")
    tokens = torch.as_tensor(tok, dtype=torch.int32).cuda()
    full, d = _out(torch, (5, 1003), "bf16", 2, 3)
    b2.logprob_backward(d, x, tokens, lse, g)
    same = torch.empty(5, 1003, dtype=torch.bfloat16, device="cuda")
    b2.logprob_backward(same, x.contiguous(), tokens, lse, g)
    assert torch.equal(d.contiguous(), same)
    _untouched(torch, full, d)


def test_logprob_gradient_against_differences(tm):
    torch, b2 = tm
    rows, vocab, eps = 6, 50, 2.0 ** -6
    x, v = _rand(torch, (rows, vocab), "f32", 1, 1.0), _rand(torch, (rows, vocab), "f32", 2, 1.0)
    tok = np.array([0, 49, -1, 7, 7, 20])
    g, h = np.linspace(-1, 2, rows), np.linspace(1, -0.5, rows)
    g[2] = h[2] = 0.0
    value = []
    for s in (1, -1):
        lp, lse, H, _, _ = _run_logprob(tm, (x + s * eps * v).contiguous(), tok, None, 0.8, 0)
        value.append((_host(lp) * g + _host(H) * h).sum())
    lp, lse, H, _, _ = _run_logprob(tm, x, tok, None, 0.8, 0)
    d = torch.empty_like(x)
    f = lambda a: torch.from_numpy(a.astype(np.float32)).cuda()  # noqa: E731
    b2.logprob_backward(d, x, torch.as_tensor(tok, dtype=torch.int32).cuda(), lse, f(g), entropy=H, dentropy=f(h), scale=0.8)
    slope = (value[0] - value[1]) / (2 * eps)
    # central differences: third derivatives of both functions stay below 8 max|v|^3 a row; the values carry u (8 max|z| + 200)
    vmax = np.abs(_host(v)).max()
    slack = rows * 2 * (8 * (0.8 * vmax) ** 3 * eps ** 2 / 6 + u * 300 * 6 / eps)
    assert abs(slope - (_host(d) * _host(v)).sum()) <= slack


# ---- gradient norm and clipping ---------------------------------------------------------------------------------------------------------
def _tensors(torch, sizes, types, seed, std=1.0, shift=0):
    return [_rand(torch, (1, n), t, seed + i, std, 0, shift)[0] for i, (n, t) in enumerate(zip(sizes, types))]


@pytest.mark.parametrize("sizes", [[1], [5], [4096], [4095, 4097, 1], [0, 3, 0, 100000], [100003] * 3 + [7] * 40, [17] * 33, [9] * 700 + [5000] * 600, [3000001]])
@pytest.mark.parametrize("shift", [0, 1, 3])
def test_gradient_norm_and_clip(tm, sizes, shift):
    torch, b2 = tm
    types = [TYPES[i % 3] for i in range(len(sizes))]
    ts = _tensors(torch, sizes, types, 11, 0.1, shift)
    ref = math.sqrt(math.fsum(float((_host(t) ** 2).sum()) for t in ts))
    ws = torch.full((b2.gradient_norm_workspace(),), 0xA5, dtype=torch.uint8, device="cuda")
    norm = torch.full((1,), -1.0, device="cuda")
    b2.gradient_norm(b2.TensorList(ts), norm, workspace=ws)
    assert abs(norm.item() - ref) <= 2 * u * ref
    outs = _tensors(torch, sizes, [TYPES[(i + 1) % 3] for i in range(len(sizes))], 99, 1.0, (shift * 2) % 5)      # other types and alignments
    for most, coef in ((ref * 0.25, 0.25), (ref * 4, 1.0)):
        most = float(np.float32(most))
        norm.fill_(-1)
        b2.gradient_clip(b2.TensorList(ts, outs), most, norm, workspace=ws)
        assert abs(norm.item() - ref) <= 2 * u * ref
        c = min(1.0, most / ref)
        for i, (a, b) in enumerate(zip(ts, outs)):
            want = _host(a) * c
            o = TYPES[(i + 1) % 3]
            _close(_host(b), want, (U[o] + 4 * u) * np.abs(want) + TINY[o])
    same = [t.clone() for t in ts]
    b2.gradient_clip(b2.TensorList(same), ref * 4, norm, workspace=ws)       # in place, nothing to do
    assert all(torch.equal(a, b) for a, b in zip(same, ts))
    b2.gradient_clip(b2.TensorList(same), ref / 8, norm, workspace=ws)
    for i, (a, b) in enumerate(zip(ts, same)):
        want = _host(a) * (float(np.float32(ref / 8)) / ref)
        _close(_host(b), want, (U[types[i]] + 4 * u) * np.abs(want) + TINY[types[i]])


def test_gradient_norm_of_extreme_values(tm):
    torch, b2 = tm
    ws, norm = torch.empty(b2.gradient_norm_workspace(), dtype=torch.uint8, device="cuda"), torch.zeros(1, device="cuda")
    for value, want in ((1e30, 1e32), (1e-30, 1e-28), (0.0, 0.0)):
        t = torch.full((10000,), value, device="cuda")
        ref = math.sqrt(float((_host(t) ** 2).sum()))
        b2.gradient_clip(b2.TensorList([t]), ref / 2, norm, workspace=ws)
        assert abs(norm.item() - ref) <= 2 * u * ref and abs(ref - want) <= 1e-6 * want
        _close(_host(t), np.full(10000, float(np.float32(value)) / (2 if value else 1)), 4 * u * value)
    for bad in (float("nan"), float("inf"), -float("inf")):
        t = torch.ones(5000, device="cuda")
        t[77] = bad
        keep = t.clone()
        out = torch.zeros_like(t)
        b2.gradient_clip(b2.TensorList([t], [out]), 1.0, norm, workspace=ws)
        got = norm.item()
        assert math.isnan(got) if math.isnan(bad) else got == math.inf
        assert torch.equal(torch.nan_to_num(out, nan=5.0), torch.nan_to_num(keep, nan=5.0))
    b2.gradient_clip(b2.TensorList([]), 1.0, norm, workspace=ws)
    assert norm.item() == 0
    t = torch.ones(100, device="cuda")
    b2.gradient_clip(b2.TensorList([t]), 0.0, norm, workspace=ws)
    assert (t == 0).all() and norm.item() == 10


def test_gradient_clip_at_the_ends_of_the_floats(tm):
    """a norm beyond the largest float is reported as infinite and scales nothing; a factor too small for a normal number loses nothing"""
    torch, b2 = tm
    ws, norm = torch.empty(b2.gradient_norm_workspace(), dtype=torch.uint8, device="cuda"), torch.zeros(1, device="cuda")
    t = torch.full((10000,), 1e37, device="cuda")
    out = torch.zeros_like(t)
    b2.gradient_clip(b2.TensorList([t], [out]), 1.0, norm, workspace=ws)
    assert norm.item() == math.inf and torch.equal(out, t)
    for value, most in ((1e36, 1e-3), (3e36, 1e-20), (1e36, 1e-1), (1e-2, 3e-38), (1e30, 2.0)):
        t = torch.full((10000,), value, device="cuda")
        t[1::2] = -value / 3
        ref = math.sqrt(float((_host(t) ** 2).sum()))
        b2.gradient_clip(b2.TensorList([t], [out]), most, norm, workspace=ws)
        assert abs(norm.item() - ref) <= 2 * u * ref
        want = _host(t) * (float(np.float32(most)) / ref)
        # the norm, its quotient (or the root of it, twice) and two products are rounded; numbers below the normal ones by their own unit
        _close(_host(out), want, 6 * u * np.abs(want) + 2 * TINY["f32"])


@pytest.mark.parametrize("t", TYPES)
def test_gradient_clip_takes_its_factor_from_the_norm_it_reports(tm, t):
    torch, b2 = tm
    x = _rand(torch, (1, 70001), t, 5, 0.1)[0]
    out, ws, norm = torch.empty(70001, device="cuda"), torch.empty(b2.gradient_norm_workspace(), dtype=torch.uint8, device="cuda"), torch.zeros(1, device="cuda")
    for most in (0.37, 1.0, 3.3, 7.7, 11.1, 20.2):
        b2.gradient_clip(b2.TensorList([x], [out]), most, norm, workspace=ws)
        factor = np.float32(most) / norm.cpu().numpy()[0]
        assert factor < 1 and np.array_equal(out.cpu().numpy(), x.float().cpu().numpy() * factor)


# ---- norms around a block ------------------------------------------------------------------------------------------------------------------
def _norm64(v, ln, eps):
    mean = v.mean(1) if ln else np.zeros(len(v))
    var = ((v - mean[:, None]) ** 2).mean(1)
    return mean, 1 / np.sqrt(var + eps)


def _gate_rows(gate, rows):
    return 1.0 if gate is None else gate[np.arange(rows) % len(gate)]


DIMS = [1, 7, 32, 33, 128, 257, 513, 1024, 1077, 2048, 4100, 8192, 8191]


def _norm_case(tm, rows, dim, t, ln, gate_rows, pad, shift, seed=0, padding=0.2):
    torch, b2 = tm
    r = np.random.default_rng(dim + rows)
    c = {n: _rand(torch, (rows, dim), t, seed + i, s, pad, shift) for i, (n, s) in enumerate([("x", 2.0), ("f", 0.7), ("dy", 0.3), ("dh", 0.4)])}
    if ln:
        c["f"] += 1.5                                    # a mean that is worth taking off
    c["gate"] = _rand(torch, (gate_rows, dim), t, seed + 8, 1.0, pad, shift) if gate_rows else None
    f = lambda std, at: torch.from_numpy((at + std * r.standard_normal(dim)).astype(np.float32)).cuda()  # noqa: E731
    c["w1"], c["w2"], c["b1"], c["b2"] = f(0.2, 1), f(0.2, 1), f(0.1, 0) if ln else None, f(0.1, 0) if ln else None
    pat = np.where(r.random(rows) < padding, 0, 2).astype(np.int8)
    pat[0] = 1
    c["pat"] = torch.from_numpy(pat).cuda()
    return c


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("t,ln,gate_rows,pad,shift", [("f32", True, 0, 0, 0), ("bf16", False, 12, 0, 0), ("f16", True, 1, 3, 1), ("bf16", True, 4, 8, 8), ("f32", False, 6, 0, 2)])
def test_block_norm(tm, dim, t, ln, gate_rows, pad, shift):
    torch, b2 = tm
    rows, eps, a = 12, 1e-5, 0.5
    c = _norm_case(tm, rows, dim, t, ln, gate_rows, pad, shift)
    real = (c["pat"].cpu().numpy() != 0)[:, None]
    fy, y = _out(torch, (rows, dim), t, pad, shift)
    fh, h = _out(torch, (rows, dim), t, pad, shift)
    stats = torch.full((rows, 4), float("nan"), device="cuda")
    kw = dict(w_pre=c["w1"], w_post=c["w2"], b_post=c["b2"], gate=c["gate"], stats=stats, pat_types=c["pat"], layer_norm=ln, residual_scale=a)
    b2.block_norm_forward(c["x"], c["f"], y, h, b_pre=c["b1"], eps=eps, **kw)
    eps = float(np.float32(eps))
    X, F, w1, w2 = (_host(c[n]) for n in ("x", "f", "w1", "w2"))
    b1, b_2 = (_host(c[n]) if ln else np.zeros(dim) for n in ("b1", "b2"))
    gate = _gate_rows(None if c["gate"] is None else _host(c["gate"]), rows)
    m2, r2 = _norm64(F, ln, eps)
    v2 = (F - m2[:, None]) * r2[:, None]
    n = v2 * w2 + b_2
    # 1/deviation: half the error of a mean of squares (per thread at most 32 terms, 10 steps of shuffles), a few roundings; the mean is off by
    # 60 u mean|v|, which 1/deviation scales
    own = lambda v, rs: 60 * u * (np.abs((v - v.mean(1, keepdims=True) * ln) * rs[:, None]) + (np.abs(v).mean(1) * rs)[:, None] * ln)  # noqa: E731
    want = np.where(real, X + a * gate * n, 0.0)
    _close(_host(y), want, real * (4 * u * (np.abs(X) + np.abs(a * gate * n)) + np.abs(a * gate) * (own(F, r2) * np.abs(w2) + u * np.abs(b_2))) + U[t] * np.abs(want) + TINY[t])
    Y = _host(y)
    m1, r1 = _norm64(Y, ln, eps)
    v1 = (Y - m1[:, None]) * r1[:, None]
    want = np.where(real, v1 * w1 + b1, 0.0)
    _close(_host(h), want, real * (own(Y, r1) * np.abs(w1) + 4 * u * (np.abs(want) + np.abs(b1))) + U[t] * np.abs(want) + TINY[t])
    S = _host(stats)
    on = real[:, 0]
    for k, (v, ref, size) in enumerate([(F, m2, np.abs(F).mean(1)), (F, r2, r2), (Y, m1, np.abs(Y).mean(1)), (Y, r1, r1)]):
        # with a mean that is off by 60 u mean|v| the deviation is off by its square at most, relative to the variance
        extra = 0.0 if k % 2 == 0 else r1 * 0 + ref * ((60 * u * np.abs(v).mean(1) * ref) ** 2)
        _close(S[on, k], ref[on], (60 * u * size + extra)[on] + 1e-300)
    assert (S[~on] == 0).all()
    _untouched(torch, fy, y)
    _untouched(torch, fh, h)

    # backward, from the y and the statistics that the forward pass left
    outs = {k: _out(torch, (rows, dim), t, pad, shift) for k in ("dx", "df")}
    dgate = _out(torch, (gate_rows, dim), t, pad, shift) if gate_rows else (None, None)
    sums = {k: torch.full((dim,), float("nan"), device="cuda") for k in ("dw_pre", "db_pre", "dw_post", "db_post")}
    if not ln:
        sums["db_pre"] = sums["db_post"] = None
    ws = torch.full((b2.block_norm_backward_workspace(rows, dim, gate_rows),), 0xA5, dtype=torch.uint8, device="cuda")
    kw.pop("stats")
    call = lambda: b2.block_norm_backward(outs["dx"][1], outs["df"][1], c["dy"], c["dh"], y, c["f"], stats, dgate=dgate[1], workspace=ws, **sums, **kw)  # noqa: E731
    call()
    dy, dh = np.where(real, _host(c["dy"]), 0.0), np.where(real, _host(c["dh"]), 0.0)
    m2, r2, m1, r1 = (S[:, k:k + 1] for k in range(4))
    v1, v2 = (Y - m1) * r1, (F - m2) * r2

    def back(d, v, w, rs):
        wd = d * w
        g = rs * (wd - v * (wd * v).mean(1, keepdims=True) - (wd.mean(1, keepdims=True) if ln else 0.0))
        size = rs * (np.abs(wd) + np.abs(v) * np.abs(wd * v).mean(1, keepdims=True) + (np.abs(wd).mean(1, keepdims=True) if ln else 0.0))
        return g, size

    g, size = back(dh, v1, w1, r1)
    dt, M = dy + g, np.abs(dy) + size                    # M: what the terms of dt add up to; every one of them is off by 100 u of its size
    dn, Mn = a * gate * dt, np.abs(a * gate) * M
    dF, _ = back(dn, v2, w2, r2)
    _, MF = back(Mn, np.abs(v2), np.abs(w2), r2)
    _close(_host(outs["dx"][1]), np.where(real, dt, 0.0), real * 100 * u * M + U[t] * np.abs(dt) * real + TINY[t])
    _close(_host(outs["df"][1]), np.where(real, dF, 0.0), real * 300 * u * MF + U[t] * np.abs(dF) * real + TINY[t])
    n, Nn = v2 * w2 + b_2, np.abs(v2 * w2) + np.abs(b_2)
    if gate_rows:
        at = np.arange(rows) % gate_rows
        want, size = np.zeros((gate_rows, dim)), np.zeros((gate_rows, dim))
        np.add.at(want, at, np.where(real, a * dt * n, 0.0))
        np.add.at(size, at, np.where(real, a * M * Nn, 0.0))
        _close(_host(dgate[1]), want, (300 + rows) * u * size + U[t] * np.abs(want) + TINY[t])
        _untouched(torch, *dgate)
    for k, x, s in (("dw_pre", dh * v1, np.abs(dh * v1)), ("db_pre", dh, np.abs(dh)), ("dw_post", dn * v2, Mn * np.abs(v2)), ("db_post", dn, Mn)):
        if sums[k] is not None:
            _close(_host(sums[k]), np.where(real, x, 0.0).sum(0), (300 + rows) * u * np.where(real, s, 0.0).sum(0) + 1e-300)
    first = [t_.clone() for t_ in (outs["dx"][1], outs["df"][1], *(s for s in sums.values() if s is not None))]
    call()
    for p, q in zip(first, (outs["dx"][1], outs["df"][1], *(s for s in sums.values() if s is not None))):
        assert torch.equal(p, q)


@pytest.mark.parametrize("rows,dim,gate_rows", [(5000, 64, 1), (5000, 64, 8), (3000, 520, 3), (20000, 24, 10000), (20000, 24, 5000), (700, 2048, 700), (2000, 4099, 2), (1, 300, 1)])
def test_block_norm_backward_over_many_rows(tm, rows, dim, gate_rows):
    """every way of sharing the rows out: sums over workers, over groups, rows of the gate that one worker finishes"""
    torch, b2 = tm
    c = _norm_case(tm, rows, dim, "f32", True, gate_rows, 0, 0, padding=0.3)
    y, h, stats = torch.empty(rows, dim, device="cuda"), torch.empty(rows, dim, device="cuda"), torch.empty(rows, 4, device="cuda")
    kw = dict(w_pre=c["w1"], w_post=c["w2"], b_post=c["b2"], gate=c["gate"], pat_types=c["pat"], layer_norm=True, residual_scale=1.5)
    b2.block_norm_forward(c["x"], c["f"], y, h, b_pre=c["b1"], stats=stats, **kw)
    real = c["pat"].cuda().bool()[:, None]
    v1, v2 = (y.double() - stats[:, 2:3]) * stats[:, 3:4], (c["f"].double() - stats[:, 0:1]) * stats[:, 1:2]
    dh, dy = c["dh"].double() * real, c["dy"].double() * real

    def back(d, v, w, rs):
        wd = d * w
        return rs * (wd - v * (wd * v).mean(1, keepdim=True) - wd.mean(1, keepdim=True))

    dt = dy + back(dh, v1, c["w1"].double(), stats[:, 3:4].double())
    gate = c["gate"].double().repeat(rows // gate_rows, 1)
    dn = 1.5 * gate * dt
    n = v2 * c["w2"].double() + c["b2"].double()
    want = dict(dx=dt, df=back(dn, v2, c["w2"].double(), stats[:, 1:2].double()) * real, dgate=(1.5 * dt * n * real).view(-1, gate_rows, dim).sum(0), dw_pre=(dh * v1).sum(0),
                db_pre=dh.sum(0), dw_post=(dn * v2 * real).sum(0), db_post=(dn * real).sum(0))
    got = {k: torch.full(v.shape, float("nan"), device="cuda") for k, v in want.items()}
    ws = torch.empty(b2.block_norm_backward_workspace(rows, dim, gate_rows), dtype=torch.uint8, device="cuda")
    b2.block_norm_backward(got["dx"], got["df"], c["dy"], c["dh"], y, c["f"], stats, dgate=got["dgate"], dw_pre=got["dw_pre"], db_pre=got["db_pre"], dw_post=got["dw_post"],
                           db_post=got["db_post"], workspace=ws, **kw)
    # terms of size up to 30, at most `rows` of them in a sum: their roundings (300 u) and those of the sums in 2-norm
    for k in want:
        terms = 1 if k in ("dx", "df") else rows // gate_rows if k == "dgate" else rows
        off = (got[k].double() - want[k]).norm() / want[k].norm()
        assert off <= (300 + math.sqrt(terms)) * u * 4, (k, off.item())


@pytest.mark.parametrize("dim", [1, 45, 102, 127, 128, 129, 202, 255, 256, 257, 405])
@pytest.mark.parametrize("t,ln,pad,shift", [("f32", True, 1, 1), ("f32", False, 2, 2), ("bf16", True, 1, 1), ("f16", False, 1, 1), ("bf16", False, 2, 2)])
def test_block_norm_of_many_narrow_rows(tm, dim, t, ln, pad, shift):
    """rows that no 16-byte access fits, more of them than the kernel for few rows takes: the columns a thread has change with the width.
    The bounds are those of test_block_norm: a thread's terms are no more than there."""
    torch, b2 = tm
    rows, eps, a = 400000 // dim, 1e-5, 0.5
    c = _norm_case(tm, rows, dim, t, ln, 0, pad, shift, padding=0.1)
    real = (c["pat"].cpu().numpy() != 0)[:, None]
    fy, y = _out(torch, (rows, dim), t, pad, shift)
    fh, h = _out(torch, (rows, dim), t, pad, shift)
    stats = torch.full((rows, 4), float("nan"), device="cuda")
    kw = dict(w_pre=c["w1"], w_post=c["w2"], b_post=c["b2"], pat_types=c["pat"], layer_norm=ln, residual_scale=a)
    b2.block_norm_forward(c["x"], c["f"], y, h, b_pre=c["b1"], eps=eps, stats=stats, **kw)
    eps = float(np.float32(eps))
    X, F, w1, w2 = (_host(c[n]) for n in ("x", "f", "w1", "w2"))
    b1, b_2 = (_host(c[n]) if ln else np.zeros(dim) for n in ("b1", "b2"))
    own = lambda v, rs: 60 * u * (np.abs((v - v.mean(1, keepdims=True) * ln) * rs[:, None]) + (np.abs(v).mean(1) * rs)[:, None] * ln)  # noqa: E731
    m2, r2 = _norm64(F, ln, eps)
    n = (F - m2[:, None]) * r2[:, None] * w2 + b_2
    want = np.where(real, X + a * n, 0.0)
    _close(_host(y), want, real * (4 * u * (np.abs(X) + np.abs(a * n)) + a * (own(F, r2) * np.abs(w2) + u * np.abs(b_2))) + U[t] * np.abs(want) + TINY[t])
    Y = _host(y)
    m1, r1 = _norm64(Y, ln, eps)
    want = np.where(real, (Y - m1[:, None]) * r1[:, None] * w1 + b1, 0.0)
    _close(_host(h), want, real * (own(Y, r1) * np.abs(w1) + 4 * u * (np.abs(want) + np.abs(b1))) + U[t] * np.abs(want) + TINY[t])
    _untouched(torch, fy, y)
    _untouched(torch, fh, h)

    outs = {k: _out(torch, (rows, dim), t, pad, shift) for k in ("dx", "df")}
    sums = {k: torch.full((dim,), float("nan"), device="cuda") if ln or k[1] == "w" else None for k in ("dw_pre", "db_pre", "dw_post", "db_post")}
    ws = torch.full((b2.block_norm_backward_workspace(rows, dim, 0),), 0xA5, dtype=torch.uint8, device="cuda")
    b2.block_norm_backward(outs["dx"][1], outs["df"][1], c["dy"], c["dh"], y, c["f"], stats, workspace=ws, **sums, **kw)
    dy, dh = np.where(real, _host(c["dy"]), 0.0), np.where(real, _host(c["dh"]), 0.0)
    m2, r2, m1, r1 = (_host(stats)[:, k:k + 1] for k in range(4))
    v1, v2 = (Y - m1) * r1, (F - m2) * r2

    def back(d, v, w, rs):
        wd = d * w
        g = rs * (wd - v * (wd * v).mean(1, keepdims=True) - (wd.mean(1, keepdims=True) if ln else 0.0))
        size = rs * (np.abs(wd) + np.abs(v) * np.abs(wd * v).mean(1, keepdims=True) + (np.abs(wd).mean(1, keepdims=True) if ln else 0.0))
        return g, size

    g, size = back(dh, v1, w1, r1)
    dt, M = dy + g, np.abs(dy) + size
    dn, Mn = a * dt, a * M
    dF, _ = back(dn, v2, w2, r2)
    _, MF = back(Mn, np.abs(v2), np.abs(w2), r2)
    _close(_host(outs["dx"][1]), np.where(real, dt, 0.0), real * 100 * u * M + U[t] * np.abs(dt) * real + TINY[t])
    _close(_host(outs["df"][1]), np.where(real, dF, 0.0), real * 300 * u * MF + U[t] * np.abs(dF) * real + TINY[t])
    for k, x, s in (("dw_pre", dh * v1, np.abs(dh * v1)), ("db_pre", dh, np.abs(dh)), ("dw_post", dn * v2, Mn * np.abs(v2)), ("db_post", dn, Mn)):
        if sums[k] is not None:
            # a worker adds at most rows / 148 of them in turn, the join 32 chains of at most 148
            _close(_host(sums[k]), np.where(real, x, 0.0).sum(0), (300 + rows / 148 + 40) * u * np.where(real, s, 0.0).sum(0) + 1e-300)
    for k in outs:
        _untouched(torch, *outs[k])


def test_block_norm_parts(tm):
    """without a block (first norm), without a norm behind (last block), in place, without statistics, gradients left out"""
    torch, b2 = tm
    rows, dim = 6, 320
    c = _norm_case(tm, rows, dim, "f32", False, 1, 0, 0, padding=0.0)
    y, h = torch.empty(rows, dim, device="cuda"), torch.empty(rows, dim, device="cuda")
    kw = dict(w_pre=c["w1"], w_post=c["w2"], gate=c["gate"], residual_scale=0.5)
    st = torch.empty(rows, 4, device="cuda")
    b2.block_norm_forward(c["x"], c["f"], y, h, stats=st, **kw)
    x = c["x"].clone()
    h2 = torch.empty_like(h)
    b2.block_norm_forward(x, c["f"], x, h2, **kw)                              # in place, no statistics
    assert torch.equal(x, y) and torch.equal(h2, h)
    y2 = torch.empty_like(y)
    b2.block_norm_forward(c["x"], c["f"], y2, None, **kw)                      # last block
    assert torch.equal(y2, y)
    h3, st3 = torch.empty_like(h), torch.empty_like(st)
    b2.block_norm_forward(y, None, None, h3, stats=st3, w_pre=c["w1"])         # a norm alone
    assert torch.equal(h3, h) and torch.equal(st3[:, 2:], st[:, 2:]) and (st3[:, :2] == 0).all()
    ws = torch.empty(b2.block_norm_backward_workspace(rows, dim, 1), dtype=torch.uint8, device="cuda")
    dx, df, dw = torch.empty_like(y), torch.empty_like(y), torch.empty(dim, device="cuda")
    b2.block_norm_backward(dx, df, c["dy"], c["dh"], y, c["f"], st, dw_pre=dw, workspace=ws, **kw)
    a, b = torch.empty_like(y), torch.empty(dim, device="cuda")
    b2.block_norm_backward(a, None, None, c["dh"], y, None, st, dw_pre=b, w_pre=c["w1"], workspace=ws)       # the norm alone
    assert torch.equal(b, dw)
    _close(_host(a) + _host(c["dy"]), _host(dx), 8 * u * (np.abs(_host(a)) + np.abs(_host(c["dy"]))))
    e, g = torch.empty_like(y), torch.empty_like(y)
    b2.block_norm_backward(e, g, dx, None, None, c["f"], st, w_post=c["w2"], gate=c["gate"], residual_scale=0.5, workspace=ws)      # the block alone
    assert torch.equal(e, dx) and torch.equal(g, df)
    dh = c["dh"].clone()
    dy = c["dy"].clone()
    b2.block_norm_backward(dy, dh, dy, dh, y, c["f"], st, workspace=ws, **kw)                                # gradients in place of what came in
    assert torch.equal(dy, dx) and torch.equal(dh, df)


def test_block_norm_gradient_against_differences(tm):
    torch, b2 = tm
    rows, dim, eps = 4, 24, 2.0 ** -7
    c = _norm_case(tm, rows, dim, "f32", True, 2, 0, 0, padding=0.0)
    names = ("x", "f", "gate", "w1", "b1", "w2", "b2")
    v = {k: torch.randn(c[k].shape, generator=torch.Generator().manual_seed(i)).cuda() for i, k in enumerate(names)}

    def forward(s):
        q = {k: (c[k] + s * eps * v[k]).contiguous() for k in names}
        y, h, st = torch.empty(rows, dim, device="cuda"), torch.empty(rows, dim, device="cuda"), torch.empty(rows, 4, device="cuda")
        b2.block_norm_forward(q["x"], q["f"], y, h, w_pre=q["w1"], b_pre=q["b1"], w_post=q["w2"], b_post=q["b2"], gate=q["gate"], stats=st, layer_norm=True, residual_scale=0.7)
        return y, h, st, (_host(y) * _host(c["dy"])).sum() + (_host(h) * _host(c["dh"])).sum()

    y, h, st, _ = forward(0)
    slope = (forward(1)[3] - forward(-1)[3]) / (2 * eps)
    g = {k: torch.empty_like(c[k]) for k in names}
    ws = torch.empty(b2.block_norm_backward_workspace(rows, dim, 2), dtype=torch.uint8, device="cuda")
    b2.block_norm_backward(g["x"], g["f"], c["dy"], c["dh"], y, c["f"], st, w_pre=c["w1"], w_post=c["w2"], b_post=c["b2"], gate=c["gate"], dgate=g["gate"], dw_pre=g["w1"], db_pre=g["b1"],
                           dw_post=g["w2"], db_post=g["b2"], layer_norm=True, residual_scale=0.7, workspace=ws)
    total = sum((_host(g[k]) * _host(v[k])).sum() for k in names)
    # the values: rows * dim terms of size up to 3, each off by 200 u; the curve: third derivatives of order 100 a term over eps^2 / 6
    n = rows * dim
    slack = math.sqrt(n) * 3 * 200 * u / eps + math.sqrt(n) * 100 * eps ** 2 / 6
    assert abs(slope - total) <= slack, (slope, total, slack)


# ---- refusals ----------------------------------------------------------------------------------------------------------------------------------
def test_refusals(tm):
    torch, b2 = tm
    f = lambda *s, dtype=None: torch.zeros(*s, device="cuda", dtype=dtype)  # noqa: E731
    tok, ws = f(4, dtype=torch.int32), torch.zeros(1 << 22, dtype=torch.uint8, device="cuda")
    E = b2.B2Error

    def refuses(text, fn, *a, **k):
        with pytest.raises(E, match=text):
            fn(*a, **k)

    refuses("shape", b2.embedding_forward, f(3, 8), f(10, 8), tok)
    refuses("shape", b2.embedding_forward, f(4, 9), f(10, 8), tok)
    refuses("element type", b2.embedding_forward, f(4, 8), f(10, 8), tok.long())
    refuses("element type", b2.embedding_forward, f(4, 8), f(10, 8, dtype=torch.float64), tok)
    refuses("strides", b2.embedding_forward, f(4, 8), f(8, 10).t(), tok)
    refuses("not on the GPU", b2.embedding_forward, torch.zeros(4, 8), f(10, 8), tok)
    refuses("workspace|null", b2.embedding_backward, f(10, 8), f(4, 8), tok)
    refuses("are needed", b2.embedding_backward, f(10, 8), f(4, 8), tok, workspace=ws[:256])
    refuses("256 bytes", b2.embedding_backward, f(10, 8), f(4, 8), tok, workspace=ws[16:])
    refuses("scale", b2.logprob_forward, f(4, 8), tok, f(4), f(4), scale=0.0)
    refuses("scale", b2.logprob_forward, f(4, 8), tok, f(4), f(4), scale=float("nan"))
    refuses("null", b2.logprob_forward, f(4, 8), tok, f(4), None)
    refuses("alternatives", b2.logprob_forward, f(4, 8), tok, f(4), f(4), top_tokens=f(4, 33, dtype=torch.int32), top_logprobs=f(4, 33))
    refuses("null", b2.logprob_forward, f(4, 8), tok, f(4), f(4), top_tokens=f(4, 3, dtype=torch.int32))
    refuses("shape", b2.logprob_forward, f(4, 8), tok, f(4), f(4), mask=f(4, 7, dtype=torch.uint8))
    refuses("element type", b2.logprob_forward, f(4, 8), tok, f(4), f(4), mask=f(4, 8))
    refuses("null", b2.logprob_backward, f(4, 8), f(4, 8), tok, f(4), f(4), dentropy=f(4))
    refuses("element type", b2.logprob_backward, f(4, 8, dtype=torch.bfloat16), f(4, 8), tok, f(4), f(4))
    refuses("largest norm", b2.gradient_clip, b2.TensorList([f(5)]), -1.0, f(1), workspace=ws)
    refuses("largest norm", b2.gradient_clip, b2.TensorList([f(5)]), float("nan"), f(1), workspace=ws)
    refuses("workspace", b2.gradient_clip, b2.TensorList([f(5)]), 1.0, f(1))
    refuses("are needed", b2.gradient_norm, b2.TensorList([f(5)]), f(1), workspace=ws[:64])
    refuses("elements", b2.gradient_clip, b2.TensorList([f(5)], [f(6)]), 1.0, f(1), workspace=ws)
    x = f(4, 16)
    refuses("at most", b2.block_norm_forward, f(2, 8193), None, None, f(2, 8193))
    refuses("gate", b2.block_norm_forward, x, f(4, 16), f(4, 16), f(4, 16), gate=f(3, 16))
    refuses("null", b2.block_norm_forward, x, f(4, 16), None, f(4, 16))
    refuses("null", b2.block_norm_forward, x, None, None, None)
    refuses("place of x", b2.block_norm_forward, x, None, None, x)
    refuses("epsilon", b2.block_norm_forward, x, None, None, f(4, 16), eps=-1.0)
    st = f(4, 4)
    refuses("need f", b2.block_norm_backward, f(4, 16), f(4, 16), x, None, None, None, st, workspace=ws)
    refuses("need dh", b2.block_norm_backward, f(4, 16), None, x, None, None, None, st, dw_pre=f(16), workspace=ws)
    refuses("gate", b2.block_norm_backward, f(4, 16), f(4, 16), x, None, None, f(4, 16), st, dgate=f(0, 16), workspace=ws)
    refuses("workspace", b2.block_norm_backward, f(4, 16), f(4, 16), x, x, x, f(4, 16), st)
    refuses("are needed", b2.block_norm_backward, f(4, 16), f(4, 16), x, x, x, f(4, 16), st, workspace=ws[:64])
    # the library itself, past the binding's checks
    L = b2.lib()
    assert L.b2_embedding_forward(x.data_ptr(), 7, 16, x.data_ptr(), 0, 16, 4, 16, tok.data_ptr(), 4, 1.0, None) == -5
    assert L.b2_embedding_forward(x.data_ptr() + 2, 0, 16, x.data_ptr(), 0, 16, 4, 16, tok.data_ptr(), 1, 1.0, None) == -5
    assert L.b2_embedding_forward(x.data_ptr(), 0, 15, x.data_ptr(), 0, 16, 4, 16, tok.data_ptr(), 1, 1.0, None) == -5
    assert L.b2_embedding_forward(x.data_ptr(), 0, 16, x.data_ptr(), 0, 16, 0, 16, tok.data_ptr(), 1, 1.0, None) == -1
    assert L.b2_logprob_forward(x.data_ptr(), 0, -1, 16, 16, None, 0, 1.0, None, None, st.data_ptr(), None, 0, None, None, None) == -1
    assert L.b2_logprob_forward(x.data_ptr(), 0, 4, 16, 15, None, 0, 1.0, None, None, st.data_ptr(), None, 0, None, None, None) == -5
    assert L.b2_gradient_norm(None, 3, st.data_ptr(), ws.data_ptr(), ws.numel(), None) == -5


# ---- large buffers, streams --------------------------------------------------------------------------------------------------------------------
def test_offsets_beyond_32_bits(tm):
    """rows 2^30 and more elements apart, a tensor of more than 2^32 elements: the last rows and elements are the ones that would go astray"""
    torch, b2 = tm
    ld, dim = (1 << 30) + 8, 72

    def wide(rows, cols, seed, dtype=torch.bfloat16):
        t = torch.empty(rows * ld, dtype=dtype, device="cuda").view(rows, ld)[:, :cols]
        t.copy_(torch.randn(rows, cols, generator=torch.Generator().manual_seed(seed)).to(dtype))
        return t

    tok = torch.tensor([2, 0, 3, 3], dtype=torch.int32, device="cuda")
    table, out = wide(4, dim, 1), wide(4, dim, 2)
    b2.embedding_forward(out, table, tok, 2.0)
    assert torch.equal(out.contiguous(), table.contiguous()[tok.long()] * 2)
    ws = torch.empty(b2.embedding_backward_workspace(4, 4, dim), dtype=torch.uint8, device="cuda")
    b2.embedding_backward(table, out, tok, 1.0, workspace=ws)
    want = torch.zeros(4, dim, device="cuda").index_add_(0, tok.long(), out.float())
    assert torch.equal(table.float(), want.to(torch.bfloat16).float())
    # rows of logits, and their gradient in place
    x, small = wide(4, 3000, 3), None
    small = x.contiguous()
    for a in (x, small):
        r = _run_logprob(tm, a, tok.cpu().numpy(), None, 1.0, 5)
        b2.logprob_backward(a, a, tok, r[1], torch.ones(4, device="cuda"))
        if a is x:
            first = r
    assert all(torch.equal(p, q) for p, q in zip(first, r)) and torch.equal(x.contiguous(), small)
    del table, out, x, small
    # norms
    f, y, h = wide(3, dim, 4), wide(3, dim, 5), wide(3, dim, 6)
    st, st2 = torch.empty(3, 4, device="cuda"), torch.empty(3, 4, device="cuda")
    fs, ys, hs = (t.contiguous() for t in (f, y, h))
    b2.block_norm_forward(y, f, y, h, stats=st)
    b2.block_norm_forward(ys, fs, ys, hs, stats=st2)
    assert torch.equal(y.contiguous(), ys) and torch.equal(h.contiguous(), hs) and torch.equal(st, st2)
    ws = torch.empty(b2.block_norm_backward_workspace(3, dim), dtype=torch.uint8, device="cuda")
    b2.block_norm_backward(h, f, h, None, None, f, st, workspace=ws)
    b2.block_norm_backward(hs, fs, hs, None, None, fs, st2, workspace=ws)
    assert torch.equal(h.contiguous(), hs) and torch.equal(f.contiguous(), fs)
    del f, y, h
    big = torch.zeros((1 << 32) + 21, dtype=torch.bfloat16, device="cuda")
    big[0], big[-1], big[1 << 31] = 2.0, 3.0, 6.0
    norm, ws = torch.zeros(1, device="cuda"), torch.empty(b2.gradient_norm_workspace(), dtype=torch.uint8, device="cuda")
    b2.gradient_clip(b2.TensorList([big]), 3.5, norm, workspace=ws)
    assert norm.item() == 7.0 and big[0] == 1.0 and big[-1] == 1.5 and big[1 << 31] == 3.0 and big[1:1 << 31].sum() == 0


def test_every_operator_runs_on_the_callers_stream(tm):
    """work on a side stream, behind a kernel that keeps it busy and writes the inputs last: an operator that ran elsewhere would read them too early"""
    torch, b2 = tm
    side = torch.cuda.Stream()
    n, vocab, dim = 5000, 3000, 96
    g = torch.Generator().manual_seed(3)
    src = {"table": torch.randn(vocab, dim, generator=g).cuda(), "x": torch.randn(n, dim, generator=g).cuda(), "logits": torch.randn(n, vocab, generator=g).cuda()}
    tok = torch.randint(-1, vocab, (n,), generator=g).int().cuda()
    ws = torch.empty(max(b2.embedding_backward_workspace(n, vocab, dim), b2.block_norm_backward_workspace(n, dim), b2.gradient_norm_workspace()), dtype=torch.uint8, device="cuda")

    def run(late, handle):
        t = {k: torch.zeros_like(v) for k, v in src.items()}
        o = {k: torch.zeros(s, device="cuda") for k, s in dict(e=(n, dim), y=(n, dim), h=(n, dim), st=(n, 4), lp=(n,), lse=(n,), dt=(vocab, dim), dx=(n, dim), df=(n, dim),
                                                               norm=(1,), dl=(n, vocab)).items()}
        torch.cuda.synchronize()
        with torch.cuda.stream(side if handle else torch.cuda.current_stream()):
            if late:
                torch.cuda._sleep(20_000_000)
            for k in src:
                t[k].copy_(src[k])
            b2.embedding_forward(o["e"], t["table"], tok, stream=handle)
            b2.block_norm_forward(t["x"], o["e"], o["y"], o["h"], stats=o["st"], stream=handle)
            b2.logprob_forward(t["logits"], tok, o["lp"], o["lse"], stream=handle)
            b2.logprob_backward(o["dl"], t["logits"], tok, o["lse"], o["lp"], stream=handle)
            b2.block_norm_backward(o["dx"], o["df"], o["h"], o["y"], o["y"], o["e"], o["st"], workspace=ws, stream=handle)
            b2.embedding_backward(o["dt"], o["df"], tok, workspace=ws, stream=handle)
            b2.gradient_clip(b2.TensorList([o["dt"], o["dx"], o["dl"]]), 1.0, o["norm"], workspace=ws, stream=handle)
        torch.cuda.synchronize()
        return o

    want, got = run(False, None), run(True, side.cuda_stream)
    for k in want:
        assert torch.equal(want[k], got[k]), k


@pytest.mark.parametrize("n,vocab", [(600, 259), (5000, 259), (6000, 60000)])
def test_calls_that_follow_each_other_closely(tm, n, vocab):
    """the launches of a call overlap with those before: other inputs in the same buffers and workspace every time, nothing waited for between"""
    torch, b2 = tm
    dim, calls = 40, 24
    g = torch.Generator().manual_seed(n)
    toks = torch.randint(-1, vocab, (calls, n), generator=g).int().cuda()
    grads = torch.randn(calls, n, dim, generator=g).cuda()
    sizes = [70001, 5, 300000]
    lists = [[(torch.randn(s, generator=g) * (k + 1)).cuda() for s in sizes] for k in range(calls)]
    new = lambda: torch.empty(b2.embedding_backward_workspace(n, vocab, dim), dtype=torch.uint8, device="cuda")  # noqa: E731
    small = lambda: torch.empty(b2.gradient_norm_workspace(), dtype=torch.uint8, device="cuda")  # noqa: E731
    tok, dout, ts = torch.empty_like(toks[0]), torch.empty_like(grads[0]), [torch.empty(s, device="cuda") for s in sizes]
    ws, ws2, tables = new(), small(), torch.empty(calls, vocab, dim, device="cuda")
    outs, norms = [[torch.empty(s, device="cuda") for s in sizes] for _ in range(calls)], torch.empty(calls, 1, device="cuda")
    tl = [b2.TensorList(ts, o) for o in outs]
    torch.cuda.synchronize()
    for k in range(calls):
        tok.copy_(toks[k])
        dout.copy_(grads[k])
        b2.embedding_backward(tables[k], dout, tok, 1.0, workspace=ws)
        for a, b in zip(ts, lists[k]):
            a.copy_(b)
        b2.gradient_clip(tl[k], 100.0, norms[k], workspace=ws2)
    torch.cuda.synchronize()
    for k in range(calls):
        want, norm = torch.empty(vocab, dim, device="cuda"), torch.empty(1, device="cuda")
        b2.embedding_backward(want, grads[k], toks[k], 1.0, workspace=new())
        alone = [torch.empty(s, device="cuda") for s in sizes]
        b2.gradient_clip(b2.TensorList(lists[k], alone), 100.0, norm, workspace=small())
        torch.cuda.synchronize()
        assert torch.equal(want, tables[k]) and torch.equal(norm, norms[k]) and all(torch.equal(a, b) for a, b in zip(alone, outs[k])), k
        ref = math.sqrt(math.fsum(float((t.double() ** 2).sum()) for t in lists[k]))
        assert abs(norm.item() - ref) <= 2 * u * ref
        real = toks[k] >= 0
        plain = torch.zeros(vocab, dim, device="cuda", dtype=torch.float64).index_add_(0, toks[k][real].long(), grads[k][real].double())
        mass = torch.zeros(vocab, dim, device="cuda", dtype=torch.float64).index_add_(0, toks[k][real].long(), grads[k][real].double().abs())
        assert ((want.double() - plain).abs() <= (n + 1) * u * mass).all()
