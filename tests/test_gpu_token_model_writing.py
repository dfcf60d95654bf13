"""The operators that learn from another model and write by beam search, run together as a program does (examples/token_model.py)."""
import os
import sys

import numpy as np
import pytest

from test_gpu_beam import _select
from test_gpu_int8 import _quantized

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "project-currennt-public_b200", "examples"))


def test_the_gradient_of_learning_from_another_model_against_differences():
    """As for the model's own loss: central differences with steps of 2^-6 of a weight's norm in random directions"""
    import torch
    import token_model as tm
    g = torch.Generator().manual_seed(5)
    teacher, model = tm.TokenModel(24, 48, 1, 4, 10, seed=8), tm.TokenModel(24, 32, 2, 4, 10, seed=3)
    tokens, _ = tm.batch(4, 10, 24, g)
    teacher.load(tokens)
    teacher.forward()
    taught = teacher.teach(6, scale=0.5)

    def loss():
        model.load(tokens)
        model.forward()
        return float(model.divergence(taught, scale=0.5).double())

    start = loss()
    assert start > 0
    model.backward_divergence(taught, scale=0.5)
    model.synchronize()
    for name in model.w:
        v = torch.randn(model.w[name].shape, generator=g).cuda()
        v *= model.w[name].norm() / v.norm()
        slope = (model.g[name].double() * v.double()).sum().item()
        eps, keep, ends = 2.0 ** -6, model.w[name].clone(), []
        for s in (1, -1):
            model.w[name].copy_(keep + s * eps * v)
            ends.append(loss())
        model.w[name].copy_(keep)
        # the losses carry 2^-22 each (roundings of a mean over 40 rows of fp32 values below 4), a third derivative below 8 costs eps^2 8 / 6 of the step's scale
        assert abs((ends[0] - ends[1]) / (2 * eps) - slope) <= 4 * 2.0 ** -22 / eps + eps * eps * 2 * max(1.0, start), name


def test_a_model_learns_from_another():
    import torch
    import token_model as tm
    teacher, model = tm.TokenModel(24, 48, 1, 4, 12, seed=8), tm.TokenModel(24, 32, 1, 4, 12, seed=3)
    before = {k: v.clone() for k, v in model.w.items()}
    kept = {k: v.clone() for k, v in teacher.w.items()}
    for s in range(3):
        loss = model.learn(teacher, tm.batch(4, 12, 24, torch.Generator().manual_seed(s))[0], 0.1, 1.0, top=5)
        assert torch.isfinite(loss)
    model.synchronize()
    assert all(torch.isfinite(v).all() for v in model.w.values()) and any((v != before[k]).any() for k, v in model.w.items())
    assert all(torch.equal(v, kept[k]) for k, v in teacher.w.items())


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("end,power,ruled_out", [(None, 0.0, False), (7, 0.0, False), (7, 0.6, True)])
def test_beam_search_against_a_plain_one(eight, end, power, ruled_out):
    """The same search on the host, over the logits that the model gives for the host's histories"""
    import torch
    import token_model as tm
    V, beams, groups, steps = 24, 4, 3, 8
    model = tm.TokenModel(V, 40, 1, groups * beams, 16, seed=3)
    if eight:
        model.quantize()
    start = torch.randint(0, V, (3, groups), generator=torch.Generator().manual_seed(2), dtype=torch.int32).cuda()
    allowed = None
    if ruled_out:
        allowed = torch.ones(V, dtype=torch.uint8, device="cuda")
        allowed[::5] = 0
    written, scores = model.write(start, beams, steps, end=end, length_power=power, allowed=allowed)
    model.synchronize()
    rows = groups * beams
    history = start.cpu().numpy().repeat(beams, 1)
    score = np.full(rows, -np.inf, np.float32)
    score[::beams] = 0.0
    done, length = np.zeros(rows, bool), np.ones(rows)
    for _ in range(steps):
        model.load(torch.from_numpy(history.astype(np.int32)).cuda())
        z = model.last_logits().double().cpu().numpy()
        if ruled_out:
            z[:, ::5] = -np.inf
        w = (torch.from_numpy(length).float().cuda() ** -power).cpu().numpy()
        best, parent, token = _select(z, score, done if end is not None else None, w, end or 0, groups, beams)
        take = (parent.clip(min=0) + np.arange(groups)[:, None] * beams).reshape(-1)
        gone = (parent < 0).reshape(-1)
        history, done, length = history[:, take], done[take] & ~gone, np.where(gone, 0.0, length[take])
        history[:, gone] = 0
        score, token = best.reshape(-1).astype(np.float32), token.reshape(-1).clip(min=0)
        if end is not None:
            done = done | (token == end)
        length = length + (1.0 - done)
        history = np.concatenate([history, token[None]])
    assert np.array_equal(written.cpu().numpy(), history[3:])
    fin = np.isfinite(score)
    assert np.array_equal(np.isfinite(scores.cpu().numpy()), fin)
    # each step adds the roundings of one score: 2^-20 of its log sum (24 exponentials) and half an ulp of values below 64
    assert (np.abs(scores.cpu().numpy() - score)[fin] <= steps * (2.0 ** -20 + 2.0 ** -18)).all()


def test_logits_in_8_bits():
    """the model's last logits in 8-bit integers are those of its outputs and matrix, quantised"""
    import torch
    import token_model as tm
    model = tm.TokenModel(30, 40, 1, 6, 8, seed=3)
    model.quantize()
    tokens = torch.randint(0, 30, (5, 6), generator=torch.Generator().manual_seed(2), dtype=torch.int32).cuda()
    model.load(tokens)
    got = model.last_logits().double().cpu().numpy()
    h = model.h[model.L][:model.n][-6:].double().cpu().numpy()
    q, s = _quantized(h)
    qw, sw = _quantized(model.w["out"].double().cpu().numpy())
    want = (q @ qw.T) * s.astype(np.float64)[:, None] * sw.astype(np.float64)
    assert (np.abs(got - want) <= 4 * 2.0 ** -24 * np.abs(want)).all()
    exact = h @ model.w["out"].double().cpu().numpy().T
    # a value is off by half a step of its row: sums of 40 products with errors of at most s / 2 * |w| + sw / 2 * |h| + s sw / 4
    assert (np.abs(got - exact) <= 0.5 * (s[:, None] * np.abs(qw * sw[:, None].astype(np.float64)).sum(1) + np.abs(h).sum(1)[:, None] * sw) + 10.0 * s[:, None] * sw).all()
