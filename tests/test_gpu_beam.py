"""GPU tests of a step of beam search (b2_beam_select, b2_beam_reorder) against plain implementations in 64 bits on the host."""
import math

import numpy as np
import pytest

from test_gpu_token_operators import TYPES, _host, _rand, tm, u  # noqa: F401

pytestmark = pytest.mark.gpu


def _select(z, scores, finished, weights, end, groups, top):
    """scores, beams and tokens in the order of ranks: rank, beam, logit, token; z [rows, vocab] in 64 bits, -inf where not allowed"""
    rows, vocab = z.shape
    beams = rows // groups
    best, beam, token = np.full((groups, top), -np.inf), np.full((groups, top), -1), np.full((groups, top), -1)
    for g in range(groups):
        cand = []
        for b in range(beams):
            r = g * beams + b
            s, w = float(scores[r]), 1.0 if weights is None else float(weights[r])
            if not (-np.inf < s < np.inf) or not (0 < w < np.inf):
                continue
            if finished is not None and finished[r]:
                cand.append((-(w * s), b, 0.0, end, s))
                continue
            row = z[r]
            if np.isnan(row).any() or (row == np.inf).any() or (row == -np.inf).all():
                continue
            m = row.max()
            off = s - m - math.log(np.exp(row - m).sum())
            for v in np.lexsort((np.arange(vocab), -row))[:top]:
                if row[v] > -np.inf:
                    cand.append((-(w * (off + row[v])), b, -row[v], int(v), off + row[v]))
        for k, c in enumerate(sorted(cand)[:top]):
            best[g, k], beam[g, k], token[g, k] = c[4], c[1], c[3]
    return best, beam, token


def _run(torch, b2, x, scores, groups, top, stream=None, **k):
    best = torch.full((groups, top), 7.0, device="cuda")
    beam, token = (torch.full((groups, top), 77, dtype=torch.int32, device="cuda") for _ in range(2))
    ws = torch.full((b2.beam_select_workspace(groups, x.shape[0] // groups, x.shape[1], top),), 0xA5, dtype=torch.uint8, device="cuda")
    b2.beam_select(x, scores, best, beam, token, workspace=ws, stream=stream, **k)
    return best, beam, token


def _same(got, want, x_size, vocab):
    """the order exactly; a score is a sum of three terms in 64 bits, its log sum's fp32 parts off by (vocab / 64 + 64) u + 2^-21, rounded once"""
    assert np.array_equal(got[1].cpu().numpy(), want[1]) and np.array_equal(got[2].cpu().numpy(), want[2])
    s = _host(got[0])
    fin = np.isfinite(want[0])
    assert np.array_equal(s[~fin], want[0][~fin])
    assert (np.abs(s - want[0])[fin] <= (vocab / 64 + 64) * u + 2.0 ** -20 + 2 * u * np.abs(want[0][fin])).all()


SIZES = [(1, 1, 1, 1, 0, 0), (1, 1, 5, 2, 0, 0), (2, 3, 7, 8, 0, 1), (3, 4, 16, 64, 0, 0), (5, 2, 259, 4, 0, 0), (2, 64, 33, 64, 3, 1), (1, 4, 32000, 8, 0, 0), (7, 5, 1031, 10, 1, 3),
         (2, 8, 50001, 16, 47, 0), (1, 64, 9000, 64, 0, 5), (1, 2, 200000, 33, 0, 0), (40, 6, 500, 12, 0, 0), (1, 1, 3000, 50, 0, 7)]


@pytest.mark.parametrize("groups,beams,vocab,top,pad,shift", SIZES)
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("mask,done,scale", [(None, 0.0, 1.0), ("shared", 0.2, 0.7), ("rows", 0.0, 1.25), (None, 0.3, 0.5)])
def test_select(tm, groups, beams, vocab, top, pad, shift, t, mask, done, scale):  # noqa: F811
    torch, b2 = tm
    rows = groups * beams
    x = _rand(torch, (rows, vocab), t, vocab + top, 2.5, pad, shift)
    r = np.random.default_rng(rows + vocab)
    scores = (-10 * r.random(rows)).astype(np.float32)
    finished = (r.random(rows) < done).astype(np.uint8) if done else None
    weights = (0.05 + 0.1 * r.random(rows)).astype(np.float32) if done else None
    allowed = None
    if mask:
        allowed = (r.random((rows, vocab) if mask == "rows" else vocab) < 0.8).astype(np.uint8)
        if mask == "rows":
            allowed[0] = 0                                 # nothing allowed
    cu = lambda a: None if a is None else torch.from_numpy(a).cuda()  # noqa: E731
    got = _run(torch, b2, x, cu(scores), groups, top, finished=cu(finished), weights=cu(weights), end_token=vocab // 2, mask=cu(allowed), scale=scale)
    z = (x.float() * scale).double().cpu().numpy()
    if mask:
        z = np.where(np.broadcast_to(allowed, z.shape) != 0, z, -np.inf)
    _same(got, _select(z, scores, finished, weights, vocab // 2, groups, top), 0, vocab)
    again = _run(torch, b2, x, cu(scores), groups, top, finished=cu(finished), weights=cu(weights), end_token=vocab // 2, mask=cu(allowed), scale=scale)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


def test_the_first_step_and_dead_beams(tm):  # noqa: F811
    """all beams alike and only the first alive; beams that have no continuations"""
    torch, b2 = tm
    vocab, inf, nan = 3000, math.inf, math.nan
    x = _rand(torch, (1, vocab), "bf16", 1, 2.0).repeat(8, 1)
    scores = torch.tensor([0.0] + [-inf] * 3 + [nan, inf, -1.0, -2.0], device="cuda")
    weights = torch.tensor([1, 1, 1, 1, 1, 1, 0.0, nan], device="cuda")
    got = _run(torch, b2, x, scores, 2, 6, weights=weights)
    want = _select(x.double().cpu().numpy(), scores.cpu().numpy(), None, weights.cpu().numpy(), 0, 2, 6)
    assert (want[1][0] == 0).all() and (want[1][1] == -1).all()
    _same(got, want, 0, vocab)
    for bad in (nan, inf):
        y = x.clone()
        y[0, 77] = bad
        got = _run(torch, b2, y, scores, 2, 6, weights=weights)
        assert (got[1] == -1).all() and (got[2] == -1).all() and (got[0] == -inf).all()
    # NaN where nothing is allowed, and the lowest value
    y = x.clone()
    y[:, 5] = nan
    y[:, 6] = inf
    y[:, 7] = torch.finfo(torch.bfloat16).min
    m = torch.ones(vocab, dtype=torch.bool, device="cuda")
    m[5:7] = False
    got = _run(torch, b2, y, scores, 2, 6, weights=weights, mask=m)
    z = y.double().cpu().numpy()
    z[:, 5:7] = -inf
    _same(got, _select(z, scores.cpu().numpy(), None, weights.cpu().numpy(), 0, 2, 6), 0, vocab)


@pytest.mark.parametrize("vocab", [40, 5000, 70000])
@pytest.mark.parametrize("t", ["bf16", "f32"])
def test_equal_continuations(tm, vocab, t):  # noqa: F811
    """rows of one value, of few values, and beams that are copies: the lower beam, then the lower token"""
    torch, b2 = tm
    row = torch.zeros(vocab)
    few = torch.randint(0, 3, (vocab,), generator=torch.Generator().manual_seed(3)).float()
    for base in (row, few):
        x = base.repeat(6, 1).to({"bf16": torch.bfloat16, "f32": torch.float32}[t]).cuda()
        scores = torch.full((6,), -3.0, device="cuda")
        got = _run(torch, b2, x, scores, 2, 40)
        _same(got, _select(x.double().cpu().numpy(), scores.cpu().numpy(), None, None, 0, 2, 40), 0, vocab)
    # a token in all blocks of a row and the rest impossible
    x = torch.full((2, vocab), -math.inf, device="cuda")
    x[:, :: max(1, vocab // 37)] = 0.25
    got = _run(torch, b2, x, torch.zeros(2, device="cuda"), 1, 60)
    _same(got, _select(x.double().cpu().numpy(), [0.0, 0.0], None, None, 0, 1, 60), 0, vocab)


def test_all_finished_and_negative_zero(tm):  # noqa: F811
    torch, b2 = tm
    x = torch.full((4, 100), math.nan, device="cuda")                 # nobody looks
    scores = torch.tensor([-3.0, -1.0, -2.0, -1.0], device="cuda")
    got = _run(torch, b2, x, scores, 1, 6, finished=torch.ones(4, dtype=torch.bool, device="cuda"), end_token=42)
    assert got[1].tolist() == [[1, 3, 2, 0, -1, -1]] and got[2].tolist() == [[42] * 4 + [-1] * 2] and got[0].tolist() == [[-1.0, -1.0, -2.0, -3.0, -math.inf, -math.inf]]
    x = torch.full((1, 64), -5.0, device="cuda")
    x[0, 9], x[0, 3], x[0, 20] = -0.0, 0.0, 0.0
    got = _run(torch, b2, x, torch.zeros(1, device="cuda"), 1, 3)
    assert got[2].tolist() == [[3, 9, 20]]


def test_select_on_a_stream_in_a_graph_and_twice_at_once(tm):  # noqa: F811
    torch, b2 = tm
    groups, beams, vocab, top = 4, 8, 20000, 16
    xs = [_rand(torch, (groups * beams, vocab), "bf16", s, 2.0) for s in (1, 2)]
    scores = -torch.rand(groups * beams, device="cuda")
    torch.cuda.synchronize()
    want = [_run(torch, b2, x, scores, groups, top) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    bufs = [[torch.empty(groups, top, device="cuda"), *(torch.empty(groups, top, dtype=torch.int32, device="cuda") for _ in range(2)),
             torch.empty(b2.beam_select_workspace(groups, beams, vocab, top), dtype=torch.uint8, device="cuda")] for _ in xs]
    torch.cuda.synchronize()
    for _ in range(20):
        for x, st, b in zip(xs, streams, bufs):
            b2.beam_select(x, scores, *b[:3], workspace=b[3], stream=st.cuda_stream)
    torch.cuda.synchronize()
    for b, w in zip(bufs, want):
        assert all(torch.equal(i, j) for i, j in zip(b, w))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=streams[0]):
        for x, b in zip(xs, bufs):                                     # one workspace for both, in turn
            b2.beam_select(x, scores, *b[:3], workspace=bufs[0][3], stream=streams[0].cuda_stream)
    for b in bufs:
        for t in b[:3]:
            t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    for b, w in zip(bufs, want):
        assert all(torch.equal(i, j) for i, j in zip(b, w))


def test_select_with_offsets_beyond_32_bits(tm):  # noqa: F811
    torch, b2 = tm
    rows, vocab, ld = 3, 20000, (1 << 30) + 8
    x = torch.empty(rows * ld, dtype=torch.bfloat16, device="cuda").view(rows, ld)[:, :vocab]
    x.copy_(_rand(torch, (rows, vocab), "bf16", 4, 2.0))
    scores = torch.zeros(rows, device="cuda")
    assert all(torch.equal(a, b) for a, b in zip(_run(torch, b2, x, scores, 1, 9), _run(torch, b2, x.clone(), scores, 1, 9)))


# ---- reordering ----------------------------------------------------------------------------------------------------------------------------
def _reorder(t, axis, parents, beams):
    rows = parents.numel()
    p = parents.view(-1).long()
    ok = (p >= 0) & (p < beams)
    import torch
    index = torch.where(ok, p, 0) + (torch.arange(rows, device=t.device) // beams) * beams
    out = t.index_select(axis, index)
    shape = [1] * t.dim()
    shape[axis] = rows
    return torch.where(ok.view(shape), out, torch.zeros_like(out))


@pytest.mark.parametrize("groups,beams", [(1, 1), (1, 4), (3, 5), (2, 8), (5, 16), (2, 17), (3, 64), (200, 3)])
@pytest.mark.parametrize("place", [False, True])
def test_reorder(tm, groups, beams, place):  # noqa: F811
    """states and time-major frames of all element sizes and alignments; parents that are twice there, in a ring, negative and too large"""
    torch, b2 = tm
    rows = groups * beams
    g = torch.Generator().manual_seed(beams)
    tensors, axes = [], []
    for dtype in (torch.float32, torch.bfloat16, torch.int32, torch.uint8, torch.float64):
        for shape, axis in (((rows, 1), 0), ((rows, 7), 0), ((rows, 512), 0), ((4, rows, 33), 1), ((13, rows), 1), ((2, 3, rows, 130), 2)):
            tensors.append((torch.randn(shape, generator=g) * 50).to(dtype).cuda())
            axes.append(axis)
    off = (torch.randn(rows * 24 + 3, generator=g) * 50).to(torch.bfloat16).cuda()[3:].view(rows, 24)        # rows of 48 bytes that start at 6
    tensors.append(off)
    axes.append(0)
    tensors.append(torch.empty(0, rows, 5, device="cuda"))
    axes.append(1)
    kinds = [torch.randint(0, beams, (groups, beams), generator=g), (torch.arange(beams) + 1).remainder(beams).repeat(groups, 1), torch.arange(beams).repeat(groups, 1),
             torch.randint(-2, beams + 2, (groups, beams), generator=g), torch.full((groups, beams), beams - 1)]
    for k, parents in enumerate(kinds):
        parents = parents.int().cuda()
        if place:
            mine = [t.clone() for t in tensors]
            states = b2.StateList(mine, axes)
        else:
            mine = [torch.full_like(t, 99) for t in tensors]
            states = b2.StateList(tensors, axes, mine)
        keep = [t.clone() for t in tensors]
        b2.beam_reorder(states, parents)
        for t, a, o in zip(keep, axes, mine):
            assert torch.equal(o, _reorder(t, a, parents, beams)), (k, t.dtype, t.shape)
        assert all(torch.equal(t, o) for t, o in zip(tensors, keep))


def test_reorder_beyond_32_bits(tm):  # noqa: F811
    torch, b2 = tm
    x = torch.zeros(5, 4, (1 << 28) + 16, dtype=torch.uint8, device="cuda")          # 5.4 GB
    x[:, :, -3:] = torch.arange(60, dtype=torch.uint8, device="cuda").view(5, 4, 3)
    parents = torch.tensor([[2, 0, 3, 3]], dtype=torch.int32, device="cuda")
    want = x[:, :, -3:].index_select(1, parents[0].long())
    b2.beam_reorder(b2.StateList([x], 1), parents)
    assert torch.equal(x[:, :, -3:], want) and not x[:, :, :-3].any()


def test_reorder_of_many_tensors_on_a_stream(tm):  # noqa: F811
    torch, b2 = tm
    tensors = [torch.randn(6, 10 + i, device="cuda") for i in range(75)]
    parents = torch.tensor([[1, 1, 0], [2, 0, 2]], dtype=torch.int32, device="cuda")
    want = [_reorder(t, 0, parents, 3) for t in tensors]
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    b2.beam_reorder(b2.StateList(tensors), parents, stream=st.cuda_stream)
    st.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(tensors, want))
