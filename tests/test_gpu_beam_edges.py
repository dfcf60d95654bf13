"""GPU tests of the selection of beam search (b2_beam_select) where many continuations are close to each other: the ways of its second kernel to find the best ones.  The
oracle and the bounds of a score's error are those of test_gpu_beam.py."""
import math

import numpy as np
import pytest

from test_gpu_beam import _run, _same, _select
from test_gpu_token_operators import _host, tm, u  # noqa: F401

pytestmark = pytest.mark.gpu


def _near(got, z, scores, groups, top):
    """Beams whose log sums differ may swap places where their scores are closer than these are exact.  Every candidate's score is off by e at most (as _same says), so the k-th best is,
    and so is each one's own; no place is left empty, and none is there twice."""
    rows, vocab = z.shape
    beams = rows // groups
    best, beam, token = _host(got[0]), got[1].cpu().numpy(), got[2].cpu().numpy()
    m = z.max(1)
    all_of = (np.asarray(scores, np.float64) - m - np.log(np.exp(z - m[:, None]).sum(1)))[:, None] + z
    for g in range(groups):
        mine = all_of[g * beams:(g + 1) * beams]
        n = min(top, mine.size)
        want = np.sort(mine.reshape(-1))[::-1][:n]
        e = (vocab / 64 + 64) * u + 2.0 ** -20 + 2 * u * np.abs(want)
        assert (beam[g, :n] >= 0).all() and (beam[g, n:] == -1).all() and (best[g, n:] == -math.inf).all(), "sequence %d: %d of %d" % (g, (beam[g] >= 0).sum(), n)
        assert (np.abs(best[g, :n] - want) <= e).all()
        assert (np.abs(best[g, :n] - mine[beam[g, :n], token[g, :n]]) <= e).all()
        assert (np.diff(best[g, :n]) <= 0).all() and len(set(zip(beam[g, :n], token[g, :n]))) == n


def _beams(torch, groups, beams, vocab, spread, at, seed):
    """logits and scores that differ by `spread`, the scores around `at`"""
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(groups * beams, vocab, generator=g) * spread).cuda()
    return x, (at + torch.randn(groups * beams, generator=g) * spread).cuda()


@pytest.mark.parametrize("groups,beams,vocab,top", [(150, 64, 259, 64), (40, 16, 2000, 32), (60, 8, 5000, 64)])
def test_beams_of_different_strength_again_and_again(tm, groups, beams, vocab, top):  # noqa: F811
    """continuations that are found by their ranks' first two digits: the same ones in every pass"""
    torch, b2 = tm
    x, scores = _beams(torch, groups, beams, vocab, 2.0, -20.0, 1)
    first = _run(torch, b2, x, scores, groups, top)
    _near(first, x.double().cpu().numpy(), scores.cpu().numpy(), groups, top)
    for _ in range(100):
        assert all(torch.equal(a, b) for a, b in zip(first, _run(torch, b2, x, scores, groups, top)))


@pytest.mark.parametrize("vocab,t", [(200, "float32"), (131, "float32"), (249, "float32"), (300, "bfloat16"), (500, "float16")])
@pytest.mark.parametrize("top", [33, 64])
@pytest.mark.parametrize("masked", [False, True])
def test_two_warps_of_a_row_and_many_continuations(tm, vocab, t, top, masked):  # noqa: F811
    """rows of 33 to 63 vectors, which have no bound for more than 32 continuations: every entry is of interest from the start"""
    torch, b2 = tm
    rows = 1200
    x = (torch.randn(rows, vocab, generator=torch.Generator().manual_seed(vocab)) * 3).to(getattr(torch, t)).cuda()
    scores = torch.zeros(rows, device="cuda")
    mask = torch.ones(vocab, dtype=torch.uint8, device="cuda")
    if masked:
        mask[::7] = 0
    z = x.double().cpu().numpy()
    z[:, (mask == 0).cpu().numpy()] = -math.inf
    want = _select(z, scores.cpu().numpy(), None, None, 0, rows, top)
    for _ in range(5):
        _same(_run(torch, b2, x, scores, rows, top, mask=mask if masked else None), want, 0, vocab)


@pytest.mark.parametrize("groups,beams,vocab,top", [(4, 64, 259, 64), (2, 16, 50001, 32), (6, 32, 1000, 32), (5, 8, 5000, 64), (7, 64, 300, 16)])
@pytest.mark.parametrize("spread", [1e-3, 0.01, 0.1])
@pytest.mark.parametrize("at", [-20.0, -100.0, -1000.0])
def test_continuations_next_to_each_other(tm, groups, beams, vocab, top, spread, at):  # noqa: F811
    """ranks that have the bits of their first two digits in common: no place stays empty"""
    torch, b2 = tm
    x, scores = _beams(torch, groups, beams, vocab, spread, at, 5)
    _near(_run(torch, b2, x, scores, groups, top), x.double().cpu().numpy(), scores.cpu().numpy(), groups, top)


@pytest.mark.parametrize("beams,vocab,top", [(64, 260, 64), (16, 50000, 32), (32, 1000, 48)])
@pytest.mark.parametrize("spread,at", [(1e-3, -20.0), (0.01, -100.0), (0.1, -1000.0)])
def test_the_order_of_continuations_next_to_each_other(tm, beams, vocab, top, spread, at):  # noqa: F811
    """beams with the same logits have the same log sum, whatever its error: their continuations' order is exact"""
    torch, b2 = tm
    groups = 3
    x = torch.cat([_beams(torch, 1, 1, vocab, spread, at, s)[0].repeat(beams, 1) for s in range(groups)])
    scores = _beams(torch, groups, beams, 1, spread, at, 9)[1]
    z, sc = x.double().cpu().numpy(), scores.cpu().numpy()
    for g in range(groups):                                   # no two of them are closer than the roundings in 64 bits
        ranks = np.sort((sc[g * beams:(g + 1) * beams, None].astype(np.float64) + z[g * beams]).reshape(-1))[::-1][:top + 1]
        assert (-np.diff(ranks) > 1e-11).all()
    got, want = _run(torch, b2, x, scores, groups, top), _select(z, sc, None, None, 0, groups, top)
    _same(got, want, 0, vocab)


@pytest.mark.parametrize("t", ["bfloat16", "float32"])
@pytest.mark.parametrize("behind", ["nothing", "masked", "more", "much more"])
@pytest.mark.parametrize("beams", [64, 5])
def test_nan_anywhere_in_a_row(tm, t, behind, beams):  # noqa: F811
    """a beam with a NaN among its allowed logits has no continuations, whatever comes behind it; the others have theirs"""
    torch, b2 = tm
    chunk = 1024 * (4 if t == "float32" else 8)
    vocab = 2 * chunk + chunk // 3
    x = (torch.randn(beams, vocab, generator=torch.Generator().manual_seed(4)) * 2.5).to(getattr(torch, t)).cuda()
    at = np.linspace(3, vocab - 1, beams).astype(int)
    allowed = np.ones((beams, vocab), np.uint8)
    for b in range(0, beams, 2):
        p = at[b]
        if behind == "nothing":
            x[b, p + 1:] = -math.inf
        elif behind == "masked":
            allowed[b, p + 1:] = 0
        elif behind == "much more":
            x[b, p + 1:] += 100.0
            x[b, p + 1 + (vocab - p) // 2:] += 100.0
        x[b, p] = math.nan
    scores = -torch.rand(beams, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    mask = torch.from_numpy(allowed).cuda() if behind == "masked" else None
    got = _run(torch, b2, x, scores, 1, 24, mask=mask)
    z = x.double().cpu().numpy()
    z[allowed == 0] = -math.inf
    want = _select(z, scores.cpu().numpy(), None, None, 0, 1, 24)
    assert (want[1] % 2 == 1).all()
    _same(got, want, 0, vocab)


@pytest.mark.parametrize("lo,hi", [(0, 16384), (0, 20000), (0, 40000), (8192, 50001), (16384, 16385), (10000, 49990)])
@pytest.mark.parametrize("t", ["bfloat16", "float32"])
def test_a_range_of_tokens_ruled_out(tm, lo, hi, t):  # noqa: F811
    """rows of one slice whose mask leaves nothing in whole chunks, first, last or between"""
    torch, b2 = tm
    beams, vocab, top = 40, 50001, 24
    x = (torch.randn(beams, vocab, generator=torch.Generator().manual_seed(6)) * 2.5).to(getattr(torch, t)).cuda()
    scores = -torch.rand(beams, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    mask = torch.ones(vocab, dtype=torch.bool, device="cuda")
    mask[lo:hi] = False
    got = _run(torch, b2, x, scores, 1, top, mask=mask)
    z = x.double().cpu().numpy()
    z[:, lo:hi] = -math.inf
    _same(got, _select(z, scores.cpu().numpy(), None, None, 0, 1, top), 0, vocab)
