"""A small recurrent language model in the clear, which drafts tokens between encrypted steps, and the client's answer to a
decrypted step: the operators of clear_ops.py together, as they are used.

The model has the shape of rwkv_model.py's (768 channels, 12 heads of 64, 65536 tokens) with fewer layers and linear
attention with a decay for each head in place of its time mixing; weights are seeded and random, held in 4 bits.  Per layer

    n = norm(x);  q, k, v, s = W n  (one product);  o = linear attention (q, k, v) with the state carried;  x <- x + W_o (o silu(s))

and in the end logits = W_head norm(x).  A prompt runs by chunks for all lanes at once, each of its own length; then every
token is one step.

    python fhe-ssm_amd/clear_draft.py --lanes 32 --prompt 200 --tokens 32
"""
from __future__ import annotations

import argparse
import time

import numpy as np
import torch

import clear_ops
import rwkv_model as M


def matrix(rng: np.random.Generator, out: int, n_in: int, group: int = 64, scale: float = 1.0) -> clear_ops.Q4Matrix:
    """a random 4-bit matrix whose products keep the size of their input times `scale`"""
    w = (scale / np.sqrt(n_in)) * rng.standard_normal((out, n_in), dtype=np.float32)
    codes, scales, _ = clear_ops.quantize_q4(w, group)
    return clear_ops.Q4Matrix(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda(), in_features=n_in, group=group)


def answer(hidden, head: clear_ops.Q4Matrix, draws, logprobs=None, **filters):
    """The client's answer to a step: rows of hidden states [lanes, channels] as ckks_decrypt_decode gives them (float64 on the
    host, or a device tensor) to tokens [lanes].  draws and filters are clear_ops.sample's."""
    x = torch.as_tensor(hidden)
    if not x.is_cuda or x.dtype == torch.float64:
        x = x.to("cuda", torch.float32)
    logits = torch.empty((x.shape[0], head.out_features), dtype=x.dtype, device="cuda")
    tokens = torch.empty(x.shape[0], dtype=torch.int64, device="cuda")
    head.product(x, logits)
    clear_ops.sample(logits, draws, tokens, logprobs, **filters)
    return tokens


class Draft:
    """the model and, between calls, the lanes' states (reset makes them)"""

    def __init__(self, layers: int = 2, d: int = M.D, heads: int = M.HEADS, vocab: int = M.VOCAB, seed: int = 7,
                 dtype=torch.bfloat16):
        rng = np.random.default_rng(seed)
        self.d, self.heads, self.hs, self.vocab, self.dtype = d, heads, d // heads, vocab, dtype
        self.w_in = [matrix(rng, 4 * d, d) for _ in range(layers)]
        self.w_out = [matrix(rng, d, d, scale=0.5) for _ in range(layers)]
        self.head = matrix(rng, vocab, d, scale=3.0)
        self.embedding = torch.from_numpy(0.5 * rng.standard_normal((vocab, d), dtype=np.float32)).cuda().to(dtype)
        self.log_decay = -torch.exp2(-torch.linspace(3, 8, heads, device="cuda"))  # one for each head, at every token
        self.states: list = []

    def _zeros(self, lanes: int) -> list:
        return [torch.zeros((lanes, self.heads, self.hs, self.hs), device="cuda") for _ in self.w_in]

    def reset(self, lanes: int) -> None:
        self.states = self._zeros(lanes)

    def _product(self, m, x):
        rows = x.reshape(-1, x.shape[-1])
        out = torch.empty((rows.shape[0], m.out_features), dtype=self.dtype, device="cuda")
        m.product(rows, out)
        return out.view(*x.shape[:-1], m.out_features)

    def _norm(self, x):
        f = x.float()
        return (f * torch.rsqrt(f.square().mean(-1, keepdim=True) + 1e-5)).to(self.dtype)

    def _run(self, tokens, lengths, states=None, x=None):
        """tokens [lanes, n] or, for one step, [lanes]: hidden rows of the same shape, the states (the lanes' own, unless others are
        given) carried on; x: the tokens' rows, where they are known"""
        states = self.states if states is None else states
        if len(states) != len(self.w_in):
            raise clear_ops.ClearError("reset(lanes) makes the states that prompt and step carry on")
        x = self.embedding[tokens].float() if x is None else x
        for w_in, w_out, state in zip(self.w_in, self.w_out, states):
            q, k, v, gate = self._product(w_in, self._norm(x)).unflatten(-1, (4, self.heads, self.hs)).unbind(-3)
            o = torch.empty(v.shape, dtype=self.dtype, device="cuda")
            if tokens.dim() == 1:
                clear_ops.linear_attention_step(q, k, v, self.log_decay, state, state, o, scale=self.hs**-0.5)
            else:
                need = clear_ops.linear_attention_workspace(q, k, v)
                work = torch.empty(need, dtype=torch.uint8, device="cuda") if need else None
                clear_ops.linear_attention_prompt(q, k, v, self.log_decay, state, state, o, scale=self.hs**-0.5,
                                                  lengths=lengths, workspace=work)
            o = self._norm(o) * torch.nn.functional.silu(gate.float())
            x = x + self._product(w_out, o.flatten(-2).to(self.dtype)).float()
        return self._norm(x)

    def prompt(self, tokens, lengths=None):
        """tokens [lanes, n], of lane b the first lengths[b] (int32, held to [0, n]): the hidden rows after each lane's last
        token, zeros for a lane that has none"""
        h = self._run(tokens, lengths)
        if h.shape[1] == 0:
            return h.new_zeros((len(h), h.shape[2]))
        if lengths is None:
            return h[:, -1]
        last = lengths.long().clamp(0, h.shape[1]) - 1
        rows = h[torch.arange(len(h), device=h.device), last.clamp_min(0)]
        return torch.where((last >= 0)[:, None], rows, 0.0)

    def step(self, tokens):
        """one token [lanes] for every lane: the hidden rows after it"""
        return self._run(tokens, None)

    def score(self, tokens, lengths=None, top: int = 0):
        """What the model makes of texts tokens [lanes, n], of lane b the first lengths[b]: the log-probability of every token after
        those before it and the entropy there, [lanes, n - 1] (log-probabilities past a length, and of tokens outside the
        vocabulary, are 0; entropies are of every position), with `top` the likeliest tokens and their log-probabilities
        [lanes, n - 1, top] too.  To what follows it a token outside the vocabulary is a row of zeros.  Lanes' states are left
        alone: a score may run beside steps."""
        lanes, n = len(tokens), max(1, tokens.shape[1])
        before = tokens[:, :-1].contiguous()
        x = torch.empty((*before.shape, self.d), device="cuda")
        clear_ops.embedding(before.view(-1), self.embedding, x.view(-1, self.d))
        hidden = self._run(before, None if lengths is None else (lengths - 1).clamp(min=0), self._zeros(lanes), x)
        rows, next_tokens = hidden.flatten(0, 1), tokens[:, 1:]
        if lengths is not None:
            next_tokens = torch.where(torch.arange(1, n, device=tokens.device)[None] < lengths[:, None], next_tokens, -1)
        next_tokens = next_tokens.reshape(-1)
        out = [torch.empty(len(rows), device="cuda") for _ in range(2)]
        if top:
            out += [torch.empty((len(rows), top), dtype=torch.int64, device="cuda"), torch.empty((len(rows), top), device="cuda")]
        for i in range(0, len(rows), 8192):  # so many rows' logits are held at once
            logits = self._product(self.head, rows[i:i + 8192])
            need = clear_ops.token_logprobs_workspace(logits, top)
            logprobs, entropy, *likeliest = (t[i:i + 8192] for t in out)
            clear_ops.token_logprobs(logits, next_tokens[i:i + 8192], logprobs, entropy, None, *likeliest,
                                     workspace=torch.empty(need, dtype=torch.uint8, device="cuda") if need else None)
        return tuple(t.view(lanes, n - 1, *t.shape[1:]) for t in out)

    def generate(self, tokens, count: int, draws, lengths=None, **filters):
        """`count` tokens after each lane's prompt: [lanes, count], drawn with draws [count, lanes]"""
        self.reset(len(tokens))
        hidden, out = self.prompt(tokens, lengths), []
        for i in range(count):
            out.append(answer(hidden, self.head, draws[i], **filters))
            if i + 1 < count:
                hidden = self.step(out[-1])
        return torch.stack(out, 1) if out else tokens.new_empty((len(tokens), 0))


def main() -> None:
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    p.add_argument("--lanes", type=int, default=M.LANES)
    p.add_argument("--prompt", type=int, default=200)
    p.add_argument("--tokens", type=int, default=32)
    p.add_argument("--layers", type=int, default=2)
    a = p.parse_args()
    model = Draft(layers=a.layers)
    gen = torch.Generator(device="cuda").manual_seed(1)
    tokens = torch.randint(0, model.vocab, (a.lanes, a.prompt), generator=gen, device="cuda")
    draws = torch.rand((a.tokens, a.lanes), generator=gen, device="cuda")
    filters = dict(temperature=torch.full((a.lanes,), 0.8, device="cuda"), top_p=torch.full((a.lanes,), 0.9, device="cuda"))
    for what in ("first", "second"):
        torch.cuda.synchronize()
        t = time.perf_counter()
        out = model.generate(tokens, a.tokens, draws, **filters)
        torch.cuda.synchronize()
        t = time.perf_counter() - t
        print(f"{what} run: {a.lanes} lanes, {a.prompt} tokens of prompt, {a.tokens} drafted: {t * 1e3:.1f} ms, "
              f"{a.lanes * a.tokens / t:.0f} drafted tokens/s")
    print("lane 0:", out[0].tolist())


if __name__ == "__main__":
    main()
