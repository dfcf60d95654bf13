"""A model over tokens from the library's pieces: embedding -> [norm, lstm layer, norm * gate + residual] x L -> product -> log probabilities.

    python examples/token_model.py [--steps 200]

trains it to continue periodic sequences and lets it write one.  Every step runs the forward and the backward pass on the caller's own
(torch) buffers through b2lstm: embedding_forward, block_norm_forward, LstmLayer.forward, matrix_multiply, logprob_forward, their gradients in
reverse order, gradient_clip, and a plain update.  Frames are time-major with the parallel sequences interleaved (row t*P + p);
padding frames have the token -1 and the pattern type 0.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
import b2lstm  # noqa: E402


class TokenModel:
    def __init__(self, vocab, dim, layers, parallel_sequences, max_len, seed=1):
        g = torch.Generator().manual_seed(seed)
        rand = lambda *shape, std: (torch.randn(*shape, generator=g) * std).cuda()  # noqa: E731
        self.V, self.D, self.L, self.P, self.maxT = vocab, dim, layers, parallel_sequences, max_len
        self.scale = dim ** 0.5
        self.lstm = [b2lstm.LstmLayer(parallel_sequences, max_len, dim, dim, False) for _ in range(layers)]
        one = lambda: torch.ones(dim, device="cuda")  # noqa: E731
        # norm i stands before layer i (and the last one before the product); post i and gate i behind layer i
        self.w = {"table": rand(vocab, dim, std=dim ** -0.5), "out": rand(vocab, dim, std=dim ** -0.5), "norm0": one()}
        for i in range(layers):
            self.w["lstm%d" % i] = rand(self.lstm[i].num_weights, std=0.08)
            self.w["post%d" % i], self.w["gate%d" % i], self.w["norm%d" % (i + 1)] = one(), one(), one()
        self.g = {k: torch.zeros_like(v) for k, v in self.w.items()}
        frames = max_len * parallel_sequences
        new = lambda n=dim: torch.empty(frames, n, device="cuda")  # noqa: E731
        self.x, self.h, self.f = ([new() for _ in range(layers + 1)] for _ in range(3))
        self.stats = [new(4) for _ in range(layers + 1)]
        self.dx, self.dh, self.df = new(), new(), new()
        self.logits = new(vocab)
        self.logprob, self.lse, self.entropy = (torch.empty(frames, device="cuda") for _ in range(3))
        self.norm = torch.zeros(1, device="cuda")
        self.grads = b2lstm.TensorList(list(self.g.values()))
        size = max(b2lstm.embedding_backward_workspace(frames, vocab, dim), b2lstm.block_norm_backward_workspace(frames, dim, 1),
                   b2lstm.block_norm_backward_workspace(frames, dim, 0), b2lstm.gradient_norm_workspace())
        self.work = torch.empty(size, dtype=torch.uint8, device="cuda")

    def load(self, tokens):
        """tokens: int32 [T, P] on the GPU, -1 behind a sequence's end"""
        self.T = tokens.shape[0]
        self.n = self.T * self.P
        self.tokens = tokens.reshape(-1).contiguous()
        lens = (tokens >= 0).sum(0)
        t = torch.arange(self.T, device="cuda")[:, None]
        pat = torch.where(t >= lens, 0, torch.where(t == 0, 1, torch.where(t == lens - 1, 3, 2)))
        self.pat = pat.to(torch.int8).reshape(-1).contiguous()
        for layer in self.lstm:
            layer.load_sequences(self.T, int(lens.min()), self.pat)

    def forward(self):
        """logits of the loaded tokens' successors"""
        n, w = self.n, self.w
        b2lstm.embedding_forward(self.x[0][:n], w["table"], self.tokens, self.scale)
        b2lstm.block_norm_forward(self.x[0][:n], None, None, self.h[0][:n], w_pre=w["norm0"], stats=self.stats[0][:n], pat_types=self.pat)
        for i, layer in enumerate(self.lstm):
            layer.forward(w["lstm%d" % i], self.h[i], self.f[i])
            b2lstm.block_norm_forward(self.x[i][:n], self.f[i][:n], self.x[i + 1][:n], self.h[i + 1][:n], w_pre=w["norm%d" % (i + 1)],
                                      w_post=w["post%d" % i], gate=w["gate%d" % i].view(1, -1), stats=self.stats[i + 1][:n], pat_types=self.pat)
        # logits [n][V] = h [n][D] out [V][D]^T, as the column-major product (V x D) (D x n)
        b2lstm.matrix_multiply(self.logits, self.V, w["out"], self.D, True, self.h[self.L], self.D, False, self.V, n, self.D)
        return self.logits[:n]

    def loss(self, targets):
        """mean of -log p(target) over the frames that have one (targets int32 [T * P], -1 elsewhere)"""
        n = self.n
        b2lstm.logprob_forward(self.logits[:n], targets, self.logprob[:n], self.lse[:n], entropy=self.entropy[:n])
        return -self.logprob[:n].sum() / (targets >= 0).sum()

    def backward(self, targets):
        """gradients of loss() with respect to all weights, in self.g"""
        n, w, g = self.n, self.w, self.g
        dlogits = self.logits[:n]                                        # in place
        b2lstm.logprob_backward(dlogits, dlogits, targets, self.lse[:n], torch.where(targets >= 0, -1.0, 0.0) / (targets >= 0).sum())
        b2lstm.matrix_multiply(self.dh, self.D, w["out"], self.D, False, dlogits, self.V, False, self.D, n, self.V)
        b2lstm.matrix_multiply(g["out"], self.D, self.h[self.L], self.D, False, dlogits, self.V, True, self.D, self.V, n)
        dx, dh, df = self.dx[:n], self.dh[:n], self.df[:n]
        for i in reversed(range(self.L)):
            last = i == self.L - 1
            b2lstm.block_norm_backward(dx, df, None if last else dx, dh, self.x[i + 1][:n], self.f[i][:n], self.stats[i + 1][:n], w_pre=w["norm%d" % (i + 1)],
                                       w_post=w["post%d" % i], gate=w["gate%d" % i].view(1, -1), dgate=g["gate%d" % i].view(1, -1),
                                       dw_pre=g["norm%d" % (i + 1)], dw_post=g["post%d" % i], pat_types=self.pat, workspace=self.work)
            self.lstm[i].backward(w["lstm%d" % i], self.h[i], self.f[i], df, dh, g["lstm%d" % i])
        b2lstm.block_norm_backward(dx, None, dx if self.L else None, dh, self.x[0][:n], None, self.stats[0][:n], w_pre=w["norm0"], dw_pre=g["norm0"],
                                   pat_types=self.pat, workspace=self.work)
        b2lstm.embedding_backward(g["table"], dx, self.tokens, self.scale, workspace=self.work)

    def step(self, tokens, targets, lr, max_norm):
        """one training step; the loss stays on the GPU"""
        self.load(tokens)
        self.forward()
        loss = self.loss(targets)
        self.backward(targets)
        b2lstm.gradient_clip(self.grads, max_norm, self.norm, workspace=self.work)
        for k, w in self.w.items():
            w.add_(self.g[k], alpha=-lr)
        return loss

    def next_tokens(self, tokens, top=1, allowed=None):
        """the most likely successors (tokens, log probabilities) of the last token of every sequence of tokens [T, P]"""
        self.load(tokens)
        logits = self.forward()[(self.T - 1) * self.P:]
        out, lp = torch.empty(self.P, top, dtype=torch.int32, device="cuda"), torch.empty(self.P, top, device="cuda")
        b2lstm.logprob_forward(logits, None, None, self.lse[:self.P], top_tokens=out, top_logprobs=lp, mask=allowed)
        return out, lp

    def synchronize(self):
        for layer in self.lstm:
            layer.synchronize()


def batch(P, T, vocab, generator):
    """sequences that repeat a random word of 3 to 6 tokens, of different lengths: tokens [T, P] and their successors [T * P]"""
    rows = torch.full((T + 1, P), -1, dtype=torch.int32)
    for p in range(P):
        n = T if p == 0 else int(torch.randint(T // 2, T + 1, (1,), generator=generator))
        word = torch.randint(0, vocab, (int(torch.randint(3, 7, (1,), generator=generator)),), generator=generator)
        rows[:n + 1, p] = word.repeat(n // len(word) + 1)[:n + 1].int()
        rows[n + 1:, p] = -1
    tokens, targets = rows[:-1].clone(), rows[1:].clone()
    tokens[targets < 0] = -1
    return tokens.cuda(), targets.reshape(-1).cuda()


def train(steps, vocab=24, dim=64, layers=2, P=16, T=32, lr=0.5, max_norm=1.0, seed=1, report=None):
    g = torch.Generator().manual_seed(seed)
    model = TokenModel(vocab, dim, layers, P, T, seed)
    losses = []
    for s in range(steps):
        losses.append(model.step(*batch(P, T, vocab, g), lr, max_norm))
        if report and (s + 1) % report == 0:
            print("step %4d  loss %.4f  gradient norm %.3f" % (s + 1, losses[-1].item(), model.norm.item()))
    model.synchronize()
    return model, [float(x) for x in losses]


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=400)
    model, losses = train(ap.parse_args().steps, report=50)
    tokens = batch(model.P, 12, model.V, torch.Generator().manual_seed(99))[0][:6].clone()
    for _ in range(12):
        best, _ = model.next_tokens(tokens)
        tokens = torch.cat([tokens, best.view(1, -1)])
    print("given 6 tokens, written 12 (first sequence):", tokens[:, 0].tolist())
