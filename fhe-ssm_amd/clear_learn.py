"""A drafting model that learns in the clear, from the tokens that encrypted steps answered: the operators of clear_ops.py that
score and train together, as they are used.

A small recurrent language model.  With n = norm(x), per layer

    z, v, s = W_in n;  h = gated recurrence (z + b, v) with the state carried;  x <- x + W_out (h silu(s))

from x = scale E[token], and in the end logits = W_head norm(x).  Parameters are float32, their products are taken in `dtype`
by torch; AdamW writes both.  Every position of a text predicts its next token; what lies past a lane's length counts for
nothing.

    python fhe-ssm_amd/clear_learn.py --lanes 32 --tokens 256 --steps 20
"""
from __future__ import annotations

import argparse
import time

import torch

import clear_ops
import rwkv_model as M


def _bytes(need: int):
    return torch.empty(need, dtype=torch.uint8, device="cuda") if need else None


class Learner:
    """the model, its optimizer, and between steps of one token the lanes' states (reset makes them)"""

    ROWS = 8192  # whose logits are held at once
    # What a position counts on its way back in float16, whose numbers end at 6e-8 and at 65,504: 1 / 65,536 of it, a token's
    # probability, keeps all its bits, and 4,096 times as much is in range.  The sums over positions are float32.
    WEIGHT_16 = 16.0

    def __init__(self, layers: int = 2, d: int = M.D, vocab: int = M.VOCAB, seed: int = 7, dtype=torch.bfloat16, bits: int = 32,
                 betas=(0.9, 0.99), weight_decay: float = 0.01):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.d, self.vocab, self.dtype, self.scale = d, vocab, dtype, d**0.5

        def matrix(rows, columns):
            return torch.randn((rows, columns), generator=gen, device="cuda") / columns**0.5

        self.matrices = [matrix(vocab, d), matrix(vocab, d)]  # embedding, head, then each layer's W_in and W_out
        for _ in range(layers):
            self.matrices += [matrix(3 * d, d), matrix(d, d)]
        ones, zeros = torch.ones(d, device="cuda"), torch.zeros(d, device="cuda")
        self.vectors = [ones.clone(), zeros.clone()]  # the last norm's weight and bias, then each layer's and its gates' bias
        for _ in range(layers):
            self.vectors += [ones.clone(), zeros.clone(), torch.linspace(0, 6, d, device="cuda")]
        copies = None if dtype == torch.float32 else [w.to(dtype) for w in self.matrices]
        self.weights = self.matrices if copies is None else copies  # what products are taken with
        self._adamw = (clear_ops.AdamW(self.matrices, betas=betas, weight_decay=weight_decay, bits=bits, copies=copies),
                       clear_ops.AdamW(self.vectors, betas=betas, weight_decay=0.0))
        self.steps, self.states = 0, []

    def _layers(self):
        """each layer's W_in, W_out, norm weight, norm bias and gates' bias"""
        w, v = self.weights, self.vectors
        return [(w[i], w[i + 1], *v[j:j + 3]) for i, j in zip(range(2, len(w), 2), range(2, len(v), 3))]

    # -------------------------------------------------------------------------------------------- forward
    def _norm(self, x, w, b, kept=None):
        rows, out = x.view(-1, self.d), torch.empty_like(x)
        mean, rstd = (torch.empty(len(rows), device="cuda") for _ in range(2)) if kept is not None else (None, None)
        clear_ops.layer_norm(rows, w, b, out.view(-1, self.d), mean, rstd)
        if kept is not None:
            kept.append((rows, w, mean, rstd))
        return out

    def _run(self, tokens, lengths=None, states=None, kept=None):
        """Hidden rows [..., d] of tokens [lanes, n] or, for one step, [lanes]; states are carried on in place; kept receives what
        the backward pass takes."""
        x = torch.empty((*tokens.shape, self.d), dtype=self.dtype, device="cuda")
        clear_ops.embedding(tokens.contiguous().view(-1), self.weights[0], x.view(-1, self.d), scale=self.scale)
        for i, (w_in, w_out, nw, nb, bias) in enumerate(self._layers()):
            n = self._norm(x, nw, nb, kept)
            z, v, s = (n @ w_in.t()).split(self.d, -1)
            z = z + bias.to(self.dtype)
            h, state = torch.empty_like(x), None if states is None else states[i]
            if tokens.dim() == 1:
                clear_ops.gated_recurrence_step(z, v, state, state, h)
            else:
                saved = _bytes(clear_ops.gated_recurrence_saved(z)) if kept is not None else None
                clear_ops.gated_recurrence(z, v, state, state, h, lengths=lengths, saved=saved,
                                           workspace=_bytes(clear_ops.gated_recurrence_workspace(z)))
            gate = torch.sigmoid(s.float())
            u = (h.float() * s.float() * gate).to(self.dtype)
            if kept is not None:
                kept.append((n, z, v, s, h, u, saved))
            x = x + u @ w_out.t()
        return self._norm(x, *self.vectors[:2], kept)

    def _targets(self, tokens, lengths):
        """the next token of every position, -1 where there is none of the vocabulary"""
        n = tokens.shape[1]
        ends = n if lengths is None else lengths.clamp(0, n)[:, None]
        after = torch.cat((tokens[:, 1:], tokens[:, :1]), 1)
        there = (torch.arange(1, n + 1, device="cuda")[None] < ends) & (after >= 0) & (after < self.vocab)
        return torch.where(there, after, -1)

    # -------------------------------------------------------------------------------------------- scoring
    def score(self, tokens, lengths=None, top: int = 0):
        """Of tokens [lanes, n] the log-probabilities and entropies [lanes, n] of what follows each position (0 where no token of the
        vocabulary does), with `top` the likeliest tokens and their log-probabilities [lanes, n, top] too, of every position."""
        lanes, n = tokens.shape
        rows, targets = self._run(tokens, lengths).view(-1, self.d), self._targets(tokens, lengths).reshape(-1)
        out = [torch.empty(len(rows), device="cuda") for _ in range(2)]
        if top:
            out += [torch.empty((len(rows), top), dtype=torch.int64, device="cuda"), torch.empty((len(rows), top), device="cuda")]
        for i in range(0, len(rows), self.ROWS):
            logits = rows[i:i + self.ROWS] @ self.weights[1].t()
            logprobs, entropy, *likeliest = (t[i:i + self.ROWS] for t in out)
            clear_ops.token_logprobs(logits, targets[i:i + self.ROWS], logprobs, entropy, None, *likeliest,
                                     workspace=_bytes(clear_ops.token_logprobs_workspace(logits, top)))
        out[1].masked_fill_(targets < 0, 0.0)  # the operator gives every row's
        return tuple(t.view(lanes, n, *t.shape[1:]) for t in out)

    # -------------------------------------------------------------------------------------------- learning
    def _sum(self, a, b):
        """a^T b, a matrix' gradient"""
        return a.t() @ b if self.dtype != torch.float16 else torch.mm(a.t(), b, out_dtype=torch.float32)

    def gradients(self, tokens, lengths=None):
        """The mean negative log-probability of what follows each position, and its gradients: of the matrices in dtype, for
        float16 in float32, of the vectors in float32."""
        kept: list = []
        rows, targets = self._run(tokens, lengths, kept=kept).view(-1, self.d), self._targets(tokens, lengths).reshape(-1)
        half, each = self.dtype == torch.float16, 1.0 / (targets >= 0).sum().clamp_min(1)
        weights = torch.full((len(targets),), -self.WEIGHT_16, device="cuda") if half else (-each).float().expand(len(targets)).contiguous()
        logprobs, drows = torch.empty(len(rows), device="cuda"), torch.empty_like(rows)
        dhead = torch.zeros((self.vocab, self.d), device="cuda")
        for i in range(0, len(rows), self.ROWS):
            part = slice(i, i + self.ROWS)
            logits = rows[part] @ self.weights[1].t()
            clear_ops.token_logprobs(logits, targets[part], logprobs[part], weights=weights[part], gradient=logits,
                                     workspace=_bytes(clear_ops.token_logprobs_workspace(logits)))
            drows[part] = logits @ self.weights[1]
            dhead += self._sum(logits, rows[part])
        dmatrices, dvectors = [None] * len(self.matrices), [None] * len(self.vectors)
        dmatrices[1] = dhead if half else dhead.to(self.dtype)

        def through_norm(dy, j):
            x, w, mean, rstd = kept.pop()
            dx, dvectors[j], dvectors[j + 1] = torch.empty_like(x), torch.empty_like(w), torch.empty_like(w)
            clear_ops.layer_norm_backward(dy.reshape(x.shape), x, w, mean, rstd, dx, dvectors[j], dvectors[j + 1],
                                          workspace=_bytes(clear_ops.layer_norm_workspace(x)))
            return dx

        dx = through_norm(drows, 0)
        for i, (w_in, w_out, *_) in reversed(list(enumerate(self._layers()))):
            n, z, v, s, h, u, saved = kept.pop()
            du = (dx @ w_out).float().view(s.shape)
            dmatrices[2 * i + 3] = self._sum(dx, u.view(-1, self.d))
            gate = torch.sigmoid(s.float())
            dh = (du * s.float() * gate).to(self.dtype)
            dzvs = torch.empty((*z.shape[:-1], 3 * self.d), dtype=self.dtype, device="cuda")
            dz, dv, ds = dzvs.split(self.d, -1)
            clear_ops.gated_recurrence_backward(z, v, saved, dh, None, dz, dv, lengths=lengths,
                                                workspace=_bytes(clear_ops.gated_recurrence_workspace(z)))
            ds.copy_(du * h.float() * gate * (1 + s.float() * (1 - gate)))
            dvectors[3 * i + 4] = dz.float().sum((0, 1))
            dzvs = dzvs.view(-1, 3 * self.d)
            dmatrices[2 * i + 2] = self._sum(dzvs, n.view(-1, self.d))
            dx = dx + through_norm(dzvs @ w_in, 3 * i + 2)
        flat = tokens.contiguous().view(-1)
        if lengths is not None:  # what lies past a lane's length is no token
            there = torch.arange(tokens.shape[1], device="cuda")[None] < lengths[:, None]
            flat = torch.where(there, tokens, -1).reshape(-1)
        dmatrices[0] = torch.empty_like(self.matrices[0] if half else self.weights[0])
        clear_ops.embedding_gradient(flat, dx, dmatrices[0], scale=self.scale,
                                     workspace=_bytes(clear_ops.embedding_gradient_workspace(flat, dmatrices[0])))
        if half:
            for g in dmatrices + dvectors:
                g *= each / self.WEIGHT_16
        return -logprobs.sum() / (targets >= 0).sum().clamp_min(1), dmatrices, dvectors

    def learn(self, tokens, lengths=None, lr: float = 1e-3):
        """One step on texts tokens [lanes, n]; their loss before it, on the GPU."""
        loss, *gradients = self.gradients(tokens, lengths)
        self.steps += 1
        for optimizer, g in zip(self._adamw, gradients):
            optimizer.step(g, lr=lr, step=self.steps, seed=self.steps)
        return loss

    # -------------------------------------------------------------------------------------------- drafting
    def reset(self, lanes: int) -> None:
        self.states = [torch.zeros((lanes, self.d), device="cuda") for _ in self._layers()]

    def _logits(self, hidden):
        return hidden @ self.weights[1].t()

    def prompt(self, tokens, lengths=None):
        """tokens [lanes, n], of lane b the first lengths[b]: the logits after each lane's last token, zeros for a lane that has none;
        the states are carried on"""
        if len(self.states) != len(self._layers()):
            raise clear_ops.ClearError("reset(lanes) makes the states that prompt and step carry on")
        hidden, n = self._run(tokens, lengths, states=self.states), tokens.shape[1]
        if n == 0:
            return self._logits(hidden.new_zeros((len(hidden), self.d)))
        last = torch.full((len(tokens),), n, device="cuda") if lengths is None else lengths.long().clamp(0, n)
        rows = hidden[torch.arange(len(tokens), device="cuda"), (last - 1).clamp_min(0)]
        return self._logits(torch.where((last > 0)[:, None], rows, 0.0))

    def step(self, tokens):
        """one token [lanes] for every lane: the logits after it"""
        if len(self.states) != len(self._layers()):
            raise clear_ops.ClearError("reset(lanes) makes the states that prompt and step carry on")
        return self._logits(self._run(tokens, states=self.states))

    def generate(self, tokens, count: int, draws, lengths=None, **filters):
        """`count` tokens after each lane's prompt: [lanes, count], drawn with draws [count, lanes]; filters are
        clear_ops.sample's"""
        self.reset(len(tokens))
        logits, out = self.prompt(tokens, lengths), []
        for i in range(count):
            out.append(torch.empty(len(tokens), dtype=torch.int64, device="cuda"))
            clear_ops.sample(logits, draws[i], out[-1], **filters)
            if i + 1 < count:
                logits = self.step(out[-1])
        return torch.stack(out, 1) if out else tokens.new_empty((len(tokens), 0))


def main() -> None:
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    p.add_argument("--lanes", type=int, default=M.LANES)
    p.add_argument("--tokens", type=int, default=256)
    p.add_argument("--steps", type=int, default=20)
    p.add_argument("--layers", type=int, default=2)
    p.add_argument("--bits", type=int, default=32, help="of the optimizer's states: 32 or 8")
    a = p.parse_args()
    model = Learner(layers=a.layers, bits=a.bits)
    gen = torch.Generator(device="cuda").manual_seed(1)
    follows = torch.randint(0, model.vocab, (model.vocab, 2), generator=gen, device="cuda")  # texts where two tokens may follow each
    texts = [torch.randint(0, model.vocab, (a.lanes,), generator=gen, device="cuda")]
    for _ in range(a.tokens - 1):
        texts.append(follows[texts[-1], torch.randint(0, 2, (a.lanes,), generator=gen, device="cuda")])
    texts = torch.stack(texts, 1)
    model.learn(texts)
    torch.cuda.synchronize()
    t = time.perf_counter()
    losses = [model.learn(texts) for _ in range(a.steps)]
    torch.cuda.synchronize()
    t = (time.perf_counter() - t) / max(1, a.steps)
    print(f"{a.lanes} texts of {a.tokens} tokens: {t * 1e3:.2f} ms a step, {a.lanes * a.tokens / t:.0f} tokens/s")
    print("loss:", " ".join(f"{x.item():.3f}" for x in losses))


if __name__ == "__main__":
    main()
