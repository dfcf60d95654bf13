"""GPU tests of the divergence from a teacher's most likely tokens (b2_distill_*) against plain implementations in 64 bits on the host.

Tolerances are error bounds, written down beside the oracle: u = 2^-24 is the unit roundoff of fp32, U[type] that of a tensor's type (the one rounding of
a result), TINY[type] half of its smallest number."""
import math

import numpy as np
import pytest

from test_gpu_token_operators import TINY, TYPES, U, _close, _host, _out, _rand, _untouched, tm, u  # noqa: F401

pytestmark = pytest.mark.gpu
REST = 2.0 ** -20


def _lse(z):
    m = z.max(-1, keepdims=True)
    m = np.where(np.isfinite(m), m, 0.0)
    with np.errstate(divide="ignore"):
        return (m + np.log(np.exp(z - m).sum(-1, keepdims=True)))[..., 0]


def _teacher(tok, lp, rest):
    """settled places, their probabilities, the rest's, log q of the places"""
    have = [k for k in range(len(tok)) if tok[k] >= 0 and tok[k] not in tok[:k]]
    lp = lp[have].astype(np.float64)
    if not have or (not rest and (lp == -np.inf).all()):
        return None
    if not rest:
        lp = lp - _lse(lp)
        return have, np.exp(lp), 0.0, lp
    q_rest = 1.0 - np.exp(lp).sum()
    return have, np.exp(lp), (q_rest if q_rest >= REST else 0.0), lp


def _forward(z, tok, lp, rest):
    """loss, lse, lse_rest of one row of z in 64 bits, and how far each may be off.

    The sum of n exponentials: every lane adds up to n / 32 + 32 of them (errors u each), every exponential has the hardware's 2^-22, the rounding of its
    argument's product with log2(e) (0.37 u at most, weighted with the exponential) and that of the difference (as much); each of the n / 512 + 8 times that
    a lane's or a warp's maximum rises costs one more exponential and product: 2^-21.  log adds an ulp, and the sum with the maximum u |lse|.  In the loss a
    place's q is off by (K + 6) 2 u relative to it, log q by 4 u (|lp| + 1), log p as lse and by 2 u (|z| + |lse|); q_rest by (K + 6) 2 u."""
    n, K = len(z), len(tok)
    have = _teacher(tok, lp, rest)
    listed = [tok[k] for k in range(K) if tok[k] >= 0]
    lse = _lse(z)
    others = z.copy()
    others[listed] = -np.inf
    lse_rest = _lse(others)
    e = (n / 32 + 32) * u + 2.0 ** -22 + u + (n / 512 + 8) * 2.0 ** -21
    size = np.abs(z[np.isfinite(z)]).max(initial=0.0)
    t_lse = e + 2 * u * (1 + size + math.log(n))
    if have is None:
        return 0.0, lse, lse_rest, 0.0, t_lse, t_lse
    at, q, q_rest, lq = have
    if lse == -np.inf:
        return np.inf, lse, lse_rest, 0.0, t_lse, t_lse
    lp_s = z[tok[at]] - lse
    on = q > 0
    loss = (q[on] * (lq[on] - lp_s[on])).sum()
    t_q = (K + 6) * 2 * u
    tol = (q[on] * (t_q * np.abs(lq[on] - lp_s[on]) + 4 * u * (np.abs(lq[on]) + np.abs(lp[at][on]) + 2) + t_lse + 2 * u * (size + abs(lse)))).sum() if np.isfinite(loss) else 0.0
    tol += K * u * np.abs(q[on] * (lq[on] - lp_s[on])).sum() if np.isfinite(loss) else 0.0
    if q_rest > 0:
        gap = math.log(q_rest) - (lse_rest - lse)
        loss += q_rest * gap
        if np.isfinite(gap):
            tol += t_q * (abs(gap) + 1) + q_rest * (4 * u * (abs(math.log(q_rest)) + 1) + 2 * t_lse + 2 * u * (size + abs(lse)))
    return loss, lse, lse_rest, tol + 2 * u * abs(loss) if np.isfinite(loss) else 0.0, t_lse, t_lse


def _list(torch, rows, vocab, top, seed, kind):
    """a teacher's list: tokens and log probabilities of random rows, some places empty; kinds with tokens twice, certain teachers, and all of a small vocabulary"""
    r = np.random.default_rng(seed)
    t = r.normal(size=(rows, min(vocab, 4096))) * (0.5 + 3.5 * r.random((rows, 1)))
    t = t - _lse(t)[:, None]
    tok = np.full((rows, top), -1, np.int32)
    lp = np.full((rows, top), -np.inf, np.float32)
    for i in range(rows):
        order = np.argsort(-t[i])[:top]
        n = len(order) if r.random() < 0.7 else int(r.integers(0, len(order) + 1))
        spread = r.permutation(vocab)[:t.shape[1]] if vocab > t.shape[1] else np.arange(vocab)
        tok[i, :n] = spread[order[:n]]
        lp[i, :n] = t[i, order[:n]]
    if kind == "twice":
        for i in range(rows):
            for _ in range(3):
                a, b = r.integers(0, top, 2)
                tok[i, a], lp[i, a] = tok[i, b], lp[i, b] - 1.0
    if kind == "certain":
        tok[:, 0] = r.integers(0, vocab, rows)
        tok[:, 1:] = -1
        lp[:, 0] = 0.0
    if kind == "holes":
        hole = r.random((rows, top)) < 0.4
        tok[hole] = -5
        lp[hole] = np.nan                       # nobody looks at an empty place's
        lp[r.random((rows, top)) < 0.1] = -np.inf
    return tok, lp


SIZES = [(1, 1, 1, 0, 0), (5, 2, 2, 0, 1), (3, 7, 3, 0, 0), (9, 16, 16, 0, 0), (40, 33, 8, 3, 1), (17, 259, 8, 0, 0), (70, 259, 33, 1, 3), (8, 1000, 128, 0, 5), (300, 1030, 20, 2, 0),
         (4, 2049, 64, 0, 1), (3, 5003, 100, 5, 3), (2, 40000, 31, 0, 0), (1, 131072, 128, 0, 0)]
KINDS = ["plain", "twice", "certain", "holes"]


@pytest.mark.parametrize("rows,vocab,top,pad,shift", SIZES)
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rest,scale", [(False, 1.0), (True, 0.5), (True, 0.7)])
def test_forward(tm, rows, vocab, top, pad, shift, t, rest, scale):  # noqa: F811
    torch, b2 = tm
    kind = KINDS[(rows + vocab + top + rest) % 4] if top > 1 else "plain"
    x = _rand(torch, (rows, vocab), t, rows + vocab, 2.5, pad, shift)
    if vocab > 20 and rows > 2:
        x[1, ::3] = -math.inf
        x[2] = torch.finfo(x.dtype).min
    tok, lp = _list(torch, rows, vocab, top, 7 + vocab, kind)
    if vocab > 20 and rows > 2:                 # no certain divergence from tokens that can not be
        tok[1][tok[1] % 3 == 0] = -1
    loss, lse, other = (torch.full((rows,), 7.0, device="cuda") for _ in range(3))
    b2.distill_forward(x, torch.from_numpy(tok).cuda(), torch.from_numpy(lp).cuda(), loss, lse, lse_rest=other if rest else None, scale=scale)
    z = (x.float() * scale).double().cpu().numpy()
    want = [_forward(z[i], tok[i], lp[i], rest) for i in range(rows)]
    _close(_host(lse), [w[1] for w in want], [w[4] for w in want])
    _close(_host(loss), [w[0] for w in want], [w[3] for w in want])
    if rest:
        _close(_host(other), [w[2] for w in want], [w[5] for w in want])
    again = [torch.full((rows,), 3.0, device="cuda") for _ in range(3)]
    b2.distill_forward(x, torch.from_numpy(tok).cuda(), torch.from_numpy(lp).cuda(), again[0], again[1], lse_rest=again[2] if rest else None, scale=scale)
    assert torch.equal(again[0], loss) and torch.equal(again[1], lse)


@pytest.mark.parametrize("rows,vocab,top,rest", [(2500, 300, 12, True), (2400, 2100, 40, False), (1300, 259, 70, True), (2370, 4500, 9, True), (2400, 9001, 20, True), (5000, 31, 6, True),
                                                 (2400, 1100, 128, False)])
def test_forward_of_many_rows(tm, rows, vocab, top, rest):  # noqa: F811
    """more rows than run at a time, rows that start anywhere"""
    torch, b2 = tm
    x = _rand(torch, (rows, vocab), "bf16", 3, 2.0, 3, 1)
    tok, lp = _list(torch, rows, vocab, top, 11, "holes")
    loss, lse, other = (torch.empty(rows, device="cuda") for _ in range(3))
    b2.distill_forward(x, torch.from_numpy(tok).cuda(), torch.from_numpy(lp).cuda(), loss, lse, lse_rest=other if rest else None)
    z = x.double().cpu().numpy()
    pick = np.unique(np.concatenate([np.arange(0, rows, 37), [rows - 1]]))
    want = [_forward(z[i], tok[i], lp[i], rest) for i in pick]
    _close(_host(loss)[pick], [w[0] for w in want], [w[3] for w in want])
    _close(_host(lse)[pick], [w[1] for w in want], [w[4] for w in want])
    # every row by itself, as the only one of a call: the kernel for few rows
    for i in pick[::9]:
        a, b, c = (torch.empty(1, device="cuda") for _ in range(3))
        b2.distill_forward(x[i:i + 1], torch.from_numpy(tok[i:i + 1]).cuda(), torch.from_numpy(lp[i:i + 1]).cuda(), a, b, lse_rest=c if rest else None)
        w = _forward(z[i], tok[i], lp[i], rest)
        _close(_host(a), [w[0]], [w[3]])


def test_special_rows(tm):  # noqa: F811
    torch, b2 = tm
    inf, nan = math.inf, math.nan
    V = 40
    x = torch.randn(12, V, generator=torch.Generator().manual_seed(1))
    tok = torch.tensor([[3, 5, -1]] * 12, dtype=torch.int32)
    lp = torch.tensor([[-1.0, -2.0, nan]] * 12)
    tok[0] = -1                                  # nothing listed
    x[1] = -inf                                  # nothing possible
    x[2, 7] = nan
    x[3, 7] = inf
    x[4, 3] = -inf                               # the teacher's token can not be
    tok[5, 1] = V                                # beyond the vocabulary
    lp[6, 0] = nan
    lp[7, 0] = inf
    lp[8] = torch.tensor([-inf, -inf, 0.0])      # nothing with a probability
    x[9] = -inf
    x[9, [3, 5]] = 1.0                           # no rest
    tok[10] = torch.tensor([3, 3, 5])
    lp[10] = torch.tensor([-1.0, 9.0, -2.0])     # the second 3 is not looked at
    tok[11] = -1
    x[11] = nan                                  # padding with anything in it
    x, tok, lp = x.cuda(), tok.cuda(), lp.cuda()
    loss, lse, other = (torch.full((12,), 5.0, device="cuda") for _ in range(3))
    b2.distill_forward(x, tok, lp, loss, lse, lse_rest=other)
    got = _host(loss)
    assert got[0] == 0 and got[1] == inf and np.isnan(got[[2, 3, 5, 6, 7]]).all() and got[4] == inf and got[9] == inf and got[11] == 0
    assert _host(lse)[1] == -inf and _host(other)[1] == -inf and np.isnan(_host(lse)[[2, 3, 11]]).all() and _host(other)[9] == -inf
    z = x[8].double().cpu().numpy()
    want = _forward(z, tok[8].cpu().numpy(), lp[8].cpu().numpy(), True)
    assert abs(got[8] - want[0]) <= want[3] and want[0] > 0                   # all of the teacher's mass off the list
    plain = got[10]
    tok[10, 1] = -1
    b2.distill_forward(x, tok, lp, loss, lse, lse_rest=other)
    assert loss[10].item() == plain
    b2.distill_forward(x, tok, lp, loss, lse)
    got = _host(loss)
    assert got[0] == 0 and got[1] == inf and np.isnan(got[[2, 3, 5, 6, 7]]).all() and got[4] == inf and got[8] == 0 and np.isfinite(got[9]) and got[11] == 0
    # gradients of the same rows
    g = torch.ones(12, device="cuda")
    for rest in (True, False):
        b2.distill_forward(x, tok, lp, loss, lse, lse_rest=other if rest else None)
        d = torch.full_like(x, 9.0)
        b2.distill_backward(d, x, tok, lp, lse, g, lse_rest=other if rest else None)
        d = _host(d)
        assert (d[[0, 1, 11]] == 0).all() and np.isnan(d[[2, 5]]).all() and np.isfinite(d[[4, 9, 10]]).all()
        assert np.isnan(d[6, 3]) or np.isnan(d[6]).all()
        if not rest:
            assert (d[8] == 0).all()
        assert abs(d[10].sum()) < 1e-5


def _backward(z, tok, lp, lse, lse_rest, weight, rest, vocab):
    """the gradient of one row over its scale, and how far it may be off: exponentials with 2^-21 (and 2^-22 of the hardware's) and the roundings of their arguments, the
    teacher's probabilities as in the forward pass, the row's factor p_rest - q_rest by the errors of both"""
    K = len(tok)
    want, tol = np.zeros(vocab), np.zeros(vocab)
    have = _teacher(tok, lp, rest)
    if have is None or lse == -np.inf:
        return want, tol
    at, q, q_rest, _ = have
    zf = np.where(np.isfinite(z), z, 0.0)
    e = 2.0 ** -20 + 4 * u * (np.abs(zf) + abs(lse) + (abs(lse_rest) if np.isfinite(lse_rest) else 0.0))
    t_q = (K + 6) * 2 * u
    p = np.exp(z - lse)
    if rest and np.isfinite(lse_rest):
        given = np.exp(z - lse_rest)
        p_rest = math.exp(lse_rest - lse)
        want = given * (p_rest - q_rest)
        tol = e * np.abs(want) + given * (t_q + p_rest * (2.0 ** -20 + 4 * u * (abs(lse) + abs(lse_rest))))
    else:
        want, tol = p.copy(), p * e
    listed = tok[at]
    want[listed] = p[listed] - q
    tol[listed] = p[listed] * e[listed] + q * (t_q + 4 * u * (np.abs(np.where(np.isfinite(lp[at]), lp[at], 0.0)) + 4))
    return weight * want, abs(weight) * (tol + 4 * u * np.abs(want))


@pytest.mark.parametrize("rows,vocab,top,pad,shift", SIZES)
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rest,scale,add", [(False, 1.0, False), (True, 0.5, False), (True, 0.7, True), (False, 1.3, True)])
def test_backward(tm, rows, vocab, top, pad, shift, t, rest, scale, add):  # noqa: F811
    torch, b2 = tm
    kind = KINDS[(rows + vocab + top + add) % 4] if top > 1 else "plain"
    x = _rand(torch, (rows, vocab), t, rows + vocab, 2.5, pad, shift)
    if vocab > 20 and rows > 2:
        x[1, ::3] = -math.inf
    tok, lp = _list(torch, rows, vocab, top, 7 + vocab, kind)
    z = (x.float() * scale).double().cpu().numpy()
    lse = np.array([_lse(r) for r in z], np.float32)
    others = z.copy()
    for i in range(rows):
        others[i, tok[i][tok[i] >= 0]] = -np.inf
    other = np.array([_lse(r) for r in others], np.float32)
    g = np.random.default_rng(3).normal(size=rows).astype(np.float32)
    cu = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    full, d = _out(torch, (rows, vocab), t, pad, shift)
    before = np.zeros((rows, vocab))
    if add:
        d.copy_(_rand(torch, (rows, vocab), t, 5))
        before = _host(d)
    args = [cu(tok), cu(lp), cu(lse), cu(g)]
    b2.distill_backward(d, x, *args, lse_rest=cu(other) if rest else None, scale=scale, accumulate=add)
    both = [_backward(z[i], tok[i], lp[i], float(lse[i]), float(other[i]), float(g[i]) * float(np.float32(scale)), rest, vocab) for i in range(rows)]
    want, tol = before + np.array([b[0] for b in both]), np.array([b[1] for b in both])
    _close(_host(d), want, tol + (U[t] + (2 * u if add else 0)) * np.abs(want) + 2 * u * np.abs(want) + TINY[t])
    if not add:
        _untouched(torch, full, d)
        once = d.clone()
        b2.distill_backward(x, x, *args, lse_rest=cu(other) if rest else None, scale=scale)          # in place
        assert torch.equal(x, once)
    else:
        for i in range(rows):
            if _teacher(tok[i], lp[i], rest) is None:
                assert np.array_equal(_host(d)[i], before[i])


@pytest.mark.parametrize("rows,vocab,top", [(4000, 3001, 40), (40000, 30, 5), (9000, 520, 128)])
def test_backward_of_many_rows(tm, rows, vocab, top):  # noqa: F811
    torch, b2 = tm
    x = _rand(torch, (rows, vocab), "bf16", 3, 2.0, 1, 1)
    tok, lp = _list(torch, rows, vocab, top, 11, "holes")
    tok, lp = torch.from_numpy(tok).cuda(), torch.from_numpy(lp).cuda()
    loss, lse, other = (torch.empty(rows, device="cuda") for _ in range(3))
    b2.distill_forward(x, tok, lp, loss, lse, lse_rest=other)
    g = torch.rand(rows, device="cuda")
    d = torch.full_like(x, math.nan)
    b2.distill_backward(d, x, tok, lp, lse, g, lse_rest=other)
    z, f = x.double().cpu().numpy(), lambda t: _host(t)  # noqa: E731
    for i in list(range(0, rows, max(1, rows // 60))) + [rows - 1]:
        want, tol = _backward(z[i], tok[i].cpu().numpy(), lp[i].cpu().numpy(), float(lse[i]), float(other[i]), float(g[i]), True, vocab)
        _close(f(d[i]), want, tol + (U["bf16"] + 2 * u) * np.abs(want) + TINY["bf16"])


@pytest.mark.parametrize("rest", [False, True])
def test_gradient_against_differences(tm, rest):  # noqa: F811
    """central differences of the loss in 64 bits (the oracle's) against the kernel's gradient: step h = 1e-4, error h^2 times third derivatives (below 1)"""
    torch, b2 = tm
    rows, vocab, top = 3, 30, 6
    x = _rand(torch, (rows, vocab), "f32", 2, 1.5)
    tok, lp = _list(torch, rows, vocab, top, 5, "plain")
    tt, tl = torch.from_numpy(tok).cuda(), torch.from_numpy(lp).cuda()
    loss, lse, other = (torch.empty(rows, device="cuda") for _ in range(3))
    b2.distill_forward(x, tt, tl, loss, lse, lse_rest=other if rest else None, scale=0.8)
    d = torch.empty_like(x)
    b2.distill_backward(d, x, tt, tl, lse, torch.ones(rows, device="cuda"), lse_rest=other if rest else None, scale=0.8)
    xs, h = x.double().cpu().numpy(), 1e-4
    s = float(np.float32(0.8))
    for i in range(rows):
        for j in range(vocab):
            up, down = xs[i].copy(), xs[i].copy()
            up[j] += h
            down[j] -= h
            slope = (_forward(up * s, tok[i], lp[i], rest)[0] - _forward(down * s, tok[i], lp[i], rest)[0]) / (2 * h)
            assert abs(slope - d[i, j].item()) <= h * h + 40 * u


def test_on_a_stream_and_in_a_graph(tm):  # noqa: F811
    torch, b2 = tm
    rows, vocab, top = 64, 3000, 16
    x = _rand(torch, (rows, vocab), "bf16", 2, 2.0)
    tok, lp = (torch.from_numpy(a).cuda() for a in _list(torch, rows, vocab, top, 5, "plain"))
    g = torch.rand(rows, device="cuda")
    out = [torch.empty(rows, device="cuda") for _ in range(3)]
    d = torch.empty_like(x)

    def both(st):
        b2.distill_forward(x, tok, lp, out[0], out[1], lse_rest=out[2], stream=st)
        b2.distill_backward(d, x, tok, lp, out[1], g, lse_rest=out[2], stream=st)
    both(None)
    torch.cuda.synchronize()
    want = [t.clone() for t in out + [d]]
    st = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        both(st.cuda_stream)
    keep = x.clone()
    x.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert not torch.equal(d, want[3])
    x.copy_(keep)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out + [d], want))


def test_offsets_beyond_32_bits(tm):  # noqa: F811
    torch, b2 = tm
    rows, vocab, ld = 3, 1000, (1 << 30) + 8
    x = torch.empty(rows * ld, dtype=torch.bfloat16, device="cuda").view(rows, ld)[:, :vocab]
    x.copy_(_rand(torch, (rows, vocab), "bf16", 4, 2.0))
    tok, lp = (torch.from_numpy(a).cuda() for a in _list(torch, rows, vocab, 9, 5, "plain"))
    near = x.clone()
    res = []
    for v in (x, near):
        loss, lse, other = (torch.empty(rows, device="cuda") for _ in range(3))
        b2.distill_forward(v, tok, lp, loss, lse, lse_rest=other)
        b2.distill_backward(v, v, tok, lp, lse, torch.ones(rows, device="cuda"), lse_rest=other)
        res.append((loss, lse, other, v.clone()))
    assert all(torch.equal(a, b) for a, b in zip(*res))
