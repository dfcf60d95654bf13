"""GPU tests of the divergence from a teacher's most likely tokens (b2_distill_*) where rows, lists and numbers end: listed tokens among a row's last entries, NaN in the
middle of long rows, logits that a scale takes to -inf.  Oracles and error bounds are those of test_gpu_distill.py."""
import math

import numpy as np
import pytest

from test_gpu_distill import _backward, _forward, _list
from test_gpu_token_operators import TINY, U, _close, _host, _rand, tm, u  # noqa: F401

pytestmark = pytest.mark.gpu


# segments of 512 vectors in small calls and of 2048 in large ones: more blocks than run at a time, and rows that start and end anywhere
@pytest.mark.parametrize("rows,vocab,pad,shift,t", [(3000, 20011, 0, 0, "bf16"), (1500, 50001, 47, 0, "bf16"), (1500, 9002, 0, 3, "f32"), (700, 20011, 2, 5, "f16"), (40, 20011, 0, 1, "bf16"),
                                                    (3, 4099, 0, 0, "f32")])
@pytest.mark.parametrize("rest", [True, False])
def test_gradient_of_listed_tokens_at_the_ends_of_wide_rows(tm, rows, vocab, pad, shift, t, rest):  # noqa: F811
    """The first and the last three tokens are in every list.  In place and added to zeros gives the bits that a buffer of its own gets, and that is right; so is what is
    added to other numbers."""
    torch, b2 = tm
    x = _rand(torch, (rows, vocab), t, 3, 2.0, pad, shift)
    tok, lp = _list(torch, rows, vocab, 12, 5, "plain")
    ends = np.array([vocab - 1, vocab - 2, vocab - 3, 0, 1, 2], np.int32)
    tok[:, 6:], lp[:, 6:] = ends, np.float32(-3.0) - 0.5 * np.arange(6, dtype=np.float32)
    tokens, lps = torch.from_numpy(tok).cuda(), torch.from_numpy(lp).cuda()
    loss, lse, other = (torch.empty(rows, device="cuda") for _ in range(3))
    kw = dict(lse_rest=other) if rest else {}
    b2.distill_forward(x, tokens, lps, loss, lse, **kw)
    g = torch.rand(rows, device="cuda", generator=torch.Generator("cuda").manual_seed(7)) + 0.5
    d = torch.full_like(x, math.nan)
    b2.distill_backward(d, x, tokens, lps, lse, g, **kw)
    old = _rand(torch, (rows, vocab), t, 4, 0.01, pad, shift)
    added = [torch.zeros_like(x), old.clone()]
    for a in added:
        b2.distill_backward(a, x, tokens, lps, lse, g, accumulate=True, **kw)
    pick = sorted(set(range(0, rows, max(1, rows // 40))) | {rows - 1})
    z = x[pick].double().cpu().numpy()
    b2.distill_backward(x, x, tokens, lps, lse, g, **kw)                     # in place
    assert torch.equal(x, d) and torch.equal(added[0], d)
    got, sums, before = _host(d[pick]), _host(added[1][pick]), _host(old[pick])
    for i, r in enumerate(pick):
        want, tol = _backward(z[i], tok[r], lp[r], float(lse[r]), float(other[r]), float(g[r]), rest, vocab)
        _close(got[i], want, tol + (U[t] + 2 * u) * np.abs(want) + TINY[t])
        _close(sums[i], before[i] + want, tol + (U[t] + 4 * u) * np.abs(before[i] + want) + 2 * u * np.abs(want) + TINY[t])


@pytest.mark.parametrize("vocab,t", [(3 * 1024 + 40, "bf16"), (9 * 1024 + 200, "bf16"), (10 * 1024, "f16"), (2 * 512 + 9, "f32"), (9 * 512 + 100, "f32"), (25001, "bf16"), (259, "f32")])
@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("behind", ["nothing", "more", "much more"])
def test_nan_anywhere_in_a_row(tm, vocab, t, many, behind):  # noqa: F811
    """A NaN makes its row's sums NaN whatever comes behind it: logits that can not be, the end of the row, logits of which the one before is nothing.  The other rows are
    as right as ever."""
    torch, b2 = tm
    at = np.unique(np.concatenate([np.arange(5, vocab, 197), vocab - 1 - np.arange(0, vocab // 2, 331)]))
    rows = 2 * len(at)                                          # every second one without a NaN
    x = _rand(torch, (rows, vocab), t, 3, 2.0)
    for i, p in enumerate(at):
        for r in (2 * i, 2 * i + 1):
            if behind == "nothing":
                x[r, p + 1:] = -math.inf
            elif behind == "much more":
                x[r, p + 1:] += 100.0
                x[r, p + 1 + (vocab - p) // 2:] += 100.0
        x[2 * i, p] = math.nan
    tok, lp = _list(torch, rows, vocab, 8, 5, "plain")
    if behind == "nothing":
        tok[:, :] = -1
        tok[:, 0] = 0
        lp[:, 0] = -0.5
    tok[tok[:, 0] < 0, 0] = 1
    lp[lp[:, 0] == -np.inf, 0] = -1.0
    times = 2368 // rows + 1 if many else 1                     # a warp a row, or a block
    xs = x.repeat(times, 1)
    tokens, lps = torch.from_numpy(np.tile(tok, (times, 1))).cuda(), torch.from_numpy(np.tile(lp, (times, 1))).cuda()
    z = x.double().cpu().numpy()
    for rest in (True, False):
        loss, lse, other = (torch.full((rows * times,), 7.0, device="cuda") for _ in range(3))
        b2.distill_forward(xs, tokens, lps, loss, lse, lse_rest=other if rest else None)
        got = [_host(v).reshape(times, rows) for v in (loss, lse)]
        assert np.isnan(got[0][:, ::2]).all() and np.isnan(got[1][:, ::2]).all()
        for r in range(1, rows, 2):
            w = _forward(z[r], tok[r], lp[r], rest)
            for c in range(times):
                _close(got[0][c, r], w[0], w[3])
                _close(got[1][c, r], w[1], w[4])


@pytest.mark.parametrize("rows,vocab,shift", [(5, 1031, 3), (2400, 1031, 1), (7, 9005, 0), (2400, 2101, 5)])
@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("rest", [True, False])
def test_the_lowest_value_at_the_ends_of_a_row_and_a_scale_above_1(tm, rows, vocab, shift, t, rest):  # noqa: F811
    """logits that the scale takes to -inf add nothing, wherever they stand: in front of the first whole vector and behind the last one too"""
    torch, b2 = tm
    x = _rand(torch, (rows, vocab), t, 3, 2.0, 2, shift)
    x[:, :9] = torch.finfo(x.dtype).min
    x[:, -9:] = torch.finfo(x.dtype).min
    x[1, 20:] = torch.finfo(x.dtype).min
    x[2] = torch.finfo(x.dtype).min                            # nothing that can be
    tok, lp = _list(torch, rows, vocab, 6, 5, "plain")
    tok[(tok < 9) | (tok >= vocab - 9)] = -1
    tok[1:3] = -1
    tok[1:3, 0], lp[1:3, 0] = 12, -0.25
    loss, lse, other = (torch.full((rows,), 7.0, device="cuda") for _ in range(3))
    b2.distill_forward(x, torch.from_numpy(tok).cuda(), torch.from_numpy(lp).cuda(), loss, lse, lse_rest=other if rest else None, scale=2.0)
    z = (x.float() * 2.0).double().cpu().numpy()
    assert (z[:, -9:] == -math.inf).all()
    for r in sorted({0, 1, 2, 3, 4, rows - 1} | set(range(5, rows, 61))):
        w = _forward(z[r], tok[r], lp[r], rest)
        _close(_host(loss[r]), w[0], w[3])
        _close(_host(lse[r]), w[1], w[4])
        if rest:
            _close(_host(other[r]), w[2], w[5])
