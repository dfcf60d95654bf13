"""A model over tokens from the library's pieces: embedding -> [norm, lstm layer, norm * gate + residual] x L -> product -> log probabilities.

    python examples/token_model.py [--steps 200]

trains it to continue periodic sequences, lets it write one, and lets a smaller model learn from it.  Every step runs the forward and the backward pass on the caller's own
(torch) buffers through b2lstm: embedding_forward, block_norm_forward, LstmLayer.forward, matrix_multiply, logprob_forward, their gradients in
reverse order, gradient_clip, and a plain update.  A model learns from a larger one by that one's most likely tokens (logprob_forward's alternatives into
distill_forward and distill_backward), and writes by beam search: beam_select over the last frames' logits, beam_reorder on the tokens so far; the
product with the output matrix may then run in 8-bit integers (int8_quantize once, int8_product).  Frames are time-major with the parallel sequences interleaved (row t*P + p);
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
        self.out8 = None

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

    def hidden(self):
        """what the output matrix is multiplied with: [T * P, D] of the loaded tokens"""
        n, w = self.n, self.w
        b2lstm.embedding_forward(self.x[0][:n], w["table"], self.tokens, self.scale)
        b2lstm.block_norm_forward(self.x[0][:n], None, None, self.h[0][:n], w_pre=w["norm0"], stats=self.stats[0][:n], pat_types=self.pat)
        for i, layer in enumerate(self.lstm):
            layer.forward(w["lstm%d" % i], self.h[i], self.f[i])
            b2lstm.block_norm_forward(self.x[i][:n], self.f[i][:n], self.x[i + 1][:n], self.h[i + 1][:n], w_pre=w["norm%d" % (i + 1)],
                                      w_post=w["post%d" % i], gate=w["gate%d" % i].view(1, -1), stats=self.stats[i + 1][:n], pat_types=self.pat)
        return self.h[self.L][:n]

    def forward(self):
        """logits of the loaded tokens' successors"""
        self.hidden()
        # logits [n][V] = h [n][D] out [V][D]^T, as the column-major product (V x D) (D x n)
        b2lstm.matrix_multiply(self.logits, self.V, self.w["out"], self.D, True, self.h[self.L], self.D, False, self.V, self.n, self.D)
        return self.logits[:self.n]

    def quantize(self):
        """the output matrix in 8-bit integers, for last_logits; from then on an update quantises it anew"""
        pitch = (self.D + 15) // 16 * 16
        self.out8 = torch.empty(self.V, pitch, dtype=torch.int8, device="cuda")[:, :self.D], torch.empty(self.V, device="cuda")
        b2lstm.int8_quantize(*self.out8, self.w["out"])
        self.work8 = torch.empty(b2lstm.int8_product_workspace(self.P, self.V, self.D), dtype=torch.uint8, device="cuda")

    def last_logits(self):
        """logits [P, V] of the successors of the last loaded token of every sequence"""
        h = self.hidden()[(self.T - 1) * self.P:]
        if self.out8:
            b2lstm.int8_product(self.logits[:self.P], h, *self.out8, workspace=self.work8)
        else:
            b2lstm.matrix_multiply(self.logits, self.V, self.w["out"], self.D, True, h, self.D, False, self.V, self.P, self.D)
        return self.logits[:self.P]

    def loss(self, targets):
        """mean of -log p(target) over the frames that have one (targets int32 [T * P], -1 elsewhere)"""
        n = self.n
        b2lstm.logprob_forward(self.logits[:n], targets, self.logprob[:n], self.lse[:n], entropy=self.entropy[:n])
        return -self.logprob[:n].sum() / (targets >= 0).sum()

    def teach(self, top, scale=1.0):
        """what another model learns from after forward(): the `top` most likely tokens of every frame and their log probabilities, none for padding"""
        n = self.n
        tok, lp = torch.empty(n, top, dtype=torch.int32, device="cuda"), torch.empty(n, top, device="cuda")
        b2lstm.logprob_forward(self.logits[:n], None, None, self.lse[:n], top_tokens=tok, top_logprobs=lp, scale=scale)
        tok[self.tokens < 0] = -1
        return tok, lp

    def divergence(self, taught, scale=1.0):
        """mean over the frames with a list of the divergence from a teacher (teach())"""
        n, (tok, lp) = self.n, taught
        self.rest = torch.empty(n, device="cuda")
        b2lstm.distill_forward(self.logits[:n], tok, lp, self.logprob[:n], self.lse[:n], lse_rest=self.rest, scale=scale)
        return self.logprob[:n].sum() / (tok[:, 0] >= 0).sum()

    def backward(self, targets):
        """gradients of loss() with respect to all weights, in self.g"""
        dlogits = self.logits[:self.n]                                   # in place
        b2lstm.logprob_backward(dlogits, dlogits, targets, self.lse[:self.n], torch.where(targets >= 0, -1.0, 0.0) / (targets >= 0).sum())
        self.backward_from(dlogits)

    def backward_divergence(self, taught, scale=1.0):
        """gradients of divergence()"""
        dlogits, (tok, lp) = self.logits[:self.n], taught
        each = (1.0 / (tok[:, 0] >= 0).sum()).expand(self.n).contiguous()
        b2lstm.distill_backward(dlogits, dlogits, tok, lp, self.lse[:self.n], each, lse_rest=self.rest, scale=scale)
        self.backward_from(dlogits)

    def backward_from(self, dlogits):
        n, w, g = self.n, self.w, self.g
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
        self.update(lr, max_norm)
        return loss

    def learn(self, teacher, tokens, lr, max_norm, top=8, scale=1.0):
        """one step of learning from another model of the same vocabulary"""
        teacher.load(tokens)
        teacher.forward()
        taught = teacher.teach(top, scale)
        self.load(tokens)
        self.forward()
        loss = self.divergence(taught, scale)
        self.backward_divergence(taught, scale)
        self.update(lr, max_norm)
        return loss

    def update(self, lr, max_norm):
        b2lstm.gradient_clip(self.grads, max_norm, self.norm, workspace=self.work)
        for k, w in self.w.items():
            w.add_(self.g[k], alpha=-lr)
        if self.out8:
            b2lstm.int8_quantize(*self.out8, self.w["out"])

    def write(self, tokens, beams, steps, end=None, length_power=0.0, allowed=None):
        """Beam search from tokens [T, P / beams] (no padding): the `steps` tokens of every beam [steps, P], best first within a sequence, and their log probabilities
        [P].  A beam that writes `end` is at its end (its further tokens are `end`); beams are ranked by log probability / (written tokens) ** length_power."""
        groups = self.P // beams
        history = tokens.repeat_interleave(beams, 1).contiguous()
        scores = torch.full((groups, beams), -float("inf"), device="cuda")
        scores[:, 0] = 0.0                                                # the beams are alike at first: one of them goes on
        done, length = torch.zeros(self.P, dtype=torch.uint8, device="cuda"), torch.ones(self.P, device="cuda")
        best, parent, token = torch.empty(groups, beams, device="cuda"), *(torch.empty(groups, beams, dtype=torch.int32, device="cuda") for _ in range(2))
        work = torch.empty(b2lstm.beam_select_workspace(groups, beams, self.V, beams), dtype=torch.uint8, device="cuda")
        for _ in range(steps):
            self.load(history)
            logits = self.last_logits()
            b2lstm.beam_select(logits, scores.view(-1), best, parent, token, finished=done if end is not None else None, weights=length ** -length_power,
                               end_token=end or 0, mask=allowed, workspace=work)
            # a copy of each: the states of a list are reordered in place
            b2lstm.beam_reorder(b2lstm.StateList([history, done, length], [1, 0, 0]), parent)
            scores.copy_(best)
            token.clamp_(min=0)                                           # beams without a continuation (score -inf)
            if end is not None:
                done |= (token.view(-1) == end).to(torch.uint8)
            length += 1.0 - done.float()
            history = torch.cat([history, token.view(1, -1)])
        return history[tokens.shape[0]:], scores.view(-1)

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
    model.quantize()
    start = batch(model.P // 4, 12, model.V, torch.Generator().manual_seed(99))[0][:6].clone()
    written, scores = model.write(start, 4, 12)
    print("by beam search, product in 8-bit integers:", start[:, 0].tolist() + written[:, 0].tolist(), "log probability %.3f" % scores[0].item())
    small = TokenModel(model.V, 32, 1, model.P, model.maxT, seed=5)
    g = torch.Generator().manual_seed(7)
    for s in range(ap.parse_args().steps):
        loss = small.learn(model, batch(model.P, model.maxT, model.V, g)[0], 0.5, 1.0)
    small.synchronize()
    print("a smaller model's divergence from this one after as many steps: %.4f" % loss.item())
