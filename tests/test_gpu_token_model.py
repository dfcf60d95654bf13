"""The token operators used together (examples/token_model.py), and clipping inside the network's own update."""
import os
import sys

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "project-currennt-public_b200", "examples"))


def test_the_model_learns_and_writes():
    import torch
    import token_model as tm
    model, losses = tm.train(700)
    # it starts near the log of the vocabulary and predicts all but the first turn of every word: 3 to 6 of 16 to 32 tokens cost log 24 each
    assert abs(losses[0] - np.log(24)) < 0.5
    assert np.mean(losses[-20:]) < 0.45 * losses[0]
    again, same = tm.train(20)
    assert same == losses[:20]                           # the same bits every time
    # the last token of sequences it has not seen: far more often right than the 1 in 24 of a guess
    tokens, targets = tm.batch(model.P, 24, 24, torch.Generator().manual_seed(123))
    whole = (tokens >= 0).all(0)
    hits = []
    for t in range(16, 24):
        best, lp = model.next_tokens(tokens[:t].clamp(min=0).contiguous(), top=3)
        want = targets.view(24, model.P)[t - 1]
        hits.append((best[:, 0] == want)[whole].float())
        assert (lp[:, 0] >= lp[:, 1]).all() and (lp[:, 1] >= lp[:, 2]).all() and (best[:, 0] != best[:, 1]).all()
    assert torch.cat(hits).mean() > 0.4
    allowed = torch.ones(24, dtype=torch.uint8, device="cuda")
    allowed[int(best[0, 0])] = 0
    other, _ = model.next_tokens(tokens[:23].clamp(min=0).contiguous(), top=3, allowed=allowed)
    assert (other != best[0, 0]).all() and other[0, 0] == best[0, 1]


def test_the_models_gradient_against_differences():
    import torch
    import token_model as tm
    g = torch.Generator().manual_seed(5)
    model = tm.TokenModel(24, 32, 2, 4, 10, seed=3)
    tokens, targets = tm.batch(4, 10, 24, g)

    def loss():
        model.load(tokens)
        model.forward()
        return float(model.loss(targets).double())

    loss()
    model.backward(targets)
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
        # a loss of about 3 in fp32, off by some 20 roundings: 20 * 3 * 2^-24 / eps; and curvature over steps of 1/64 of the weights
        slack = 20 * 3 * 2.0 ** -24 / eps + 0.02 * abs(slope) + 20 * eps ** 2
        assert abs((ends[0] - ends[1]) / (2 * eps) - slope) <= slack, (name, slope, (ends[0] - ends[1]) / (2 * eps))


def test_clipping_in_the_networks_update():
    import b2lstm
    from b2lstm import workloads
    layers = [dict(type="input", size=16), dict(type="blstm", size=24, bias=1.0), dict(type="feedforward_identity", size=5, bias=1.0), dict(type="sse", size=5)]
    lens = np.array([20, 20, 11], np.int32)
    x, tg = workloads.make_fraction(16, 5, 3, lens, 1, 2)
    w = workloads.make_weights(layers, 3, 0.1)

    def net():
        n = b2lstm.Net(layers, 3, 20)
        for i, wi in w.items():
            n.set_weights(i, wi)
        n.load_fraction(lens, x, tg)
        n.forward()
        n.backward()
        return n

    plain = net()
    g = {i: plain.weight_updates(i).astype(np.float64) for i in w}
    norm = np.sqrt(sum((v ** 2).sum() for v in g.values()))
    with pytest.raises(b2lstm.B2Error, match="not clipped"):
        plain.gradient_norm()
    with pytest.raises(b2lstm.B2Error, match="largest norm"):
        plain.set_gradient_clipping(-1.0)
    plain.update_weights(0.01, 0.0)
    for factor in (0.25, 4.0, 0.0):
        n = net()
        n.set_gradient_clipping(factor * norm)
        n.update_weights(0.01, 0.0)
        if factor:
            assert abs(n.gradient_norm() - norm) <= 2.0 ** -22 * norm
        for i in w:
            if factor == 0.25:
                want = w[i] - 0.01 * g[i] * factor
                # the factor, the product, the step and the sum are rounded once each
                assert np.abs(n.get_weights(i) - want).max() <= 2.0 ** -22 * (np.abs(want) + np.abs(0.01 * g[i])).max()
            else:
                assert np.array_equal(n.get_weights(i), plain.get_weights(i))     # nothing to scale: the plain update's bits
        n.close()
    plain.close()
