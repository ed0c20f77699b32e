"""What a client computes in the clear to score tokens with its drafting model and to train it on them, through clear_ops.py:
layer norm, the gated linear recurrence, the embedding, log-probabilities of given tokens, each with its gradient, and the
AdamW step over the model's tensors.

Each operator is here twice: `run` with `own` false computes it from elementary torch operations in 32 bits, with `own`
true it calls the framework; `exact` computes it in 64 bits.  Sizes are those of the repository's model (768 channels, 32
lanes, 65536 tokens), or generic ones around them.
"""
import math
import os
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
BLOCK = 256  # entries of an 8-bit state that share a power of two


def _ops():
    """the framework's module (its folder's name is no Python identifier)"""
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fhe-ssm_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import clear_ops
    return clear_ops


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # the norm before one token's product, for every lane of a step: all latency
        {"name": "norm step", "op": "norm", "rows": 32, "channels": 768, "train": False, "type": "bf16"},
        # a training batch of 32 conversations of 1024 tokens
        {"name": "norm train", "op": "norm", "rows": 32768, "channels": 768, "train": True, "type": "bf16"},
        # a small batch in full precision, rows that fill no vector
        {"name": "norm odd", "op": "norm", "rows": 2999, "channels": 1101, "train": True, "type": "f32"},
        # one token of every lane while the draft generates
        {"name": "recurrence step", "op": "step", "lanes": 32, "channels": 768, "type": "f32"},
        # the training batch, each conversation of its own length
        {"name": "recurrence lanes", "op": "recurrence", "lanes": 32, "tokens": 1024, "channels": 768, "ragged": True,
         "type": "bf16"},
        # one long text, where only the token axis has work to spread
        {"name": "recurrence long", "op": "recurrence", "lanes": 1, "tokens": 16384, "channels": 768, "ragged": False,
         "type": "f32"},
        # the training batch's tokens, as frequent as words are, the ends of conversations padded
        {"name": "embedding train", "op": "embedding", "tokens": 32768, "vocab": 65536, "channels": 768, "pad": True,
         "add": False, "type": "bf16"},
        # a few hundred answered tokens, added to the gradient that other batches left
        {"name": "embedding few", "op": "embedding", "tokens": 701, "vocab": 50277, "channels": 1101, "pad": False,
         "add": True, "type": "f32"},
        # the draft's view of the answered tokens of all lanes, with the alternatives that a client shows
        {"name": "score lanes", "op": "score", "rows": 32, "vocab": 65536, "top": 20, "train": False, "later": False,
         "type": "f32"},
        # the loss of a part of the training batch, and its gradient with weights that are known before
        {"name": "score train", "op": "score", "rows": 4096, "vocab": 65536, "top": 0, "train": True, "later": False,
         "type": "bf16"},
        # the step of a small model's tensors, among them many short ones, in float32
        {"name": "adamw 32", "op": "adamw", "bits": 32, "count": 40, "most": 2359296, "type": "f32"},
        # the step of a large model's, its states in 8 bits
        {"name": "adamw 8", "op": "adamw", "bits": 8, "count": 12, "most": 50331648, "type": "bf16"},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "step", "recurrence", "recurrence", "embedding", "score", "score", "adamw", "adamw"])
    case = {"op": op, "type": rng.choice(["f32", "bf16", "f16"])}
    if op == "norm":
        channels = rng.choice([768, 1024, _log(rng, 8, 8192), _log(rng, 8, 8192)])
        return {**case, "channels": channels, "rows": _log(rng, 1, min(65536, (1 << 24) // channels)),
                "train": rng.random() < 0.7}
    if op == "step":
        return {**case, "lanes": _log(rng, 1, 256), "channels": _log(rng, 8, 8192)}
    if op == "recurrence":
        channels = rng.choice([768, _log(rng, 8, 4096)])
        tokens = _log(rng, 1, 16384)
        return {**case, "channels": channels, "tokens": tokens,
                "lanes": _log(rng, 1, max(1, min(256, (1 << 24) // (channels * tokens)))), "ragged": rng.random() < 0.5}
    if op == "embedding":
        vocab = _log(rng, 100, 131072)
        channels = rng.choice([768, _log(rng, 8, 4096)])
        vocab = min(vocab, (50 << 20) // channels)
        return {**case, "vocab": vocab, "channels": channels, "tokens": _log(rng, 1, min(65536, (25 << 20) // channels)),
                "pad": rng.random() < 0.5, "add": rng.random() < 0.5}
    if op == "score":
        vocab = _log(rng, 100, 131072)
        return {**case, "vocab": vocab, "rows": _log(rng, 1, min(16384, (1 << 27) // vocab)),
                "top": min(rng.choice([0, 1, 5, 20, 32]), vocab // 97), "train": rng.random() < 0.5,
                "later": rng.random() < 0.3}
    most = _log(rng, 300, 1 << 24)
    return {**case, "bits": rng.choice([8, 32]), "most": most, "count": _log(rng, 1, 60 if most < (1 << 21) else 6)}


# ------------------------------------------------------------------------------------------------ inputs
class State:
    pass


def _norm_inputs(case, gen):
    """rows with a mean and a size of their own and some channels that stand out, as a residual stream has them"""
    rows, channels, kind = case["rows"], case["channels"], TYPES[case["type"]]
    x = torch.randn((rows, channels), generator=gen, device="cuda")
    x = x * (0.5 + torch.rand((rows, 1), generator=gen, device="cuda")) + torch.randn((rows, 1), generator=gen, device="cuda")
    x[:, ::97] *= 8
    w = 1 + 0.1 * torch.randn(channels, generator=gen, device="cuda")
    b = 0.1 * torch.randn(channels, generator=gen, device="cuda")
    dy = torch.randn((rows, channels), generator=gen, device="cuda") if case["train"] else None
    return x.to(kind), w, b, None if dy is None else dy.to(kind)


def _recurrence_inputs(case, gen):
    """gates whose channels remember from two to some hundred tokens, values of unit size, a state that some text left"""
    lanes, channels, kind = case["lanes"], case["channels"], TYPES[case["type"]]
    shape = (lanes, channels) if case["op"] == "step" else (lanes, case["tokens"], channels)

    def normal(*s):
        return torch.randn(s, generator=gen, device="cuda")

    z = (normal(*shape) + torch.linspace(0, 6, channels, device="cuda")).to(kind)
    x, state = normal(*shape).to(kind), normal(lanes, channels)
    if case["op"] == "step":
        return z, x, state
    lengths = None
    if case["ragged"]:
        lengths = torch.randint(case["tokens"] // 2, case["tokens"] + 1, (lanes,), generator=gen, device="cuda",
                                dtype=torch.int32)
    return z, x, state, lengths, normal(*shape).to(kind), normal(lanes, channels)


def _tokens(n, vocab, gen):
    """token i about as often as 1 / (i + 1), the numbers shuffled"""
    u = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64)
    at = ((vocab + 1.0) ** u).long().sub_(1).clamp_(0, vocab - 1)
    return torch.randperm(vocab, generator=gen, device="cuda")[at]


def _embedding_inputs(case, gen):
    n, vocab, channels, kind = case["tokens"], case["vocab"], case["channels"], TYPES[case["type"]]
    tokens = _tokens(n, vocab, gen)
    if case["pad"]:
        tokens[torch.arange(n, device="cuda") % 1024 >= 900] = -1
    table = 0.5 * torch.randn((vocab, channels), generator=gen, device="cuda")
    dy = torch.randn((n, channels), generator=gen, device="cuda").to(kind)
    before = torch.randn((vocab, channels), generator=gen, device="cuda") if case["add"] else None
    return tokens, table.to(kind), dy, before


def _score_inputs(case, gen):
    """logits as a language model leaves them: a wide bulk, some tens of likely tokens well above it, a few banned ones; the
    given tokens are mostly likely ones, a few positions are padding"""
    rows, vocab, kind = case["rows"], case["vocab"], TYPES[case["type"]]

    def uniform(*shape):
        return torch.rand(shape, generator=gen, device="cuda")

    logits = torch.randn((rows, vocab), generator=gen, device="cuda").mul_(2)
    likely = torch.randint(0, vocab, (rows, 32), generator=gen, device="cuda")
    logits.scatter_(-1, likely, 7 - 2.5 * uniform(rows, 32).clamp_min_(1e-6).log())
    logits[:, ::97] = -math.inf
    tokens = torch.where(uniform(rows) < 0.8, likely[:, 0], torch.randint(0, vocab, (rows,), generator=gen, device="cuda"))
    tokens = torch.where(tokens % 97 == 0, tokens + 1, tokens).clamp_(max=vocab - 1)
    tokens[torch.arange(rows, device="cuda") % 16 == 11] = -1
    weight = -(0.5 + uniform(rows)) if case["train"] else None
    weight_entropy = 0.1 * uniform(rows) if case["train"] else None
    return logits.to(kind), tokens, weight, weight_entropy


def _adamw_sizes(case):
    """the entries of each tensor: every second one a vector, the others falling from the largest"""
    count, most = case["count"], case["most"]
    return [max(1, most // (1 + 3 * (i // 2))) if i % 2 == 0 else max(1, int(math.sqrt(most)) // 2 - 7 * (i % 5))
            for i in range(count)]


def _starts(case):
    """where each tensor begins in the one buffer that holds them all, and the buffer's length: whole blocks"""
    starts, at = [], 0
    for n in _adamw_sizes(case):
        starts.append(at)
        at += -(-n // BLOCK) * BLOCK
    return starts, at


ADAMW = {"lr": 1e-3, "beta1": 0.9, "beta2": 0.99, "eps": 1e-8, "decay": 0.01, "step": 57, "seed": 12345}


def _adamw_inputs(case, gen):
    """weights, gradients whose size differs from channel to channel, and the moments that earlier steps left; 8-bit ones as
    rounding down leaves them.  What lies between two tensors is 0."""
    starts, length = _starts(case)
    sizes = torch.tensor(_adamw_sizes(case), device="cuda")
    whole = -(-sizes // BLOCK) * BLOCK
    local = torch.arange(length, device="cuda") - torch.tensor(starts, device="cuda").repeat_interleave(whole)
    there = local < sizes.repeat_interleave(whole)
    del local

    def normal():
        return torch.randn(length, generator=gen, device="cuda") * there

    size = torch.exp2(-8 * torch.rand(length // 64, generator=gen, device="cuda")).repeat_interleave(64) * 0.01
    p, g = 0.05 * normal(), (size * normal()).to(TYPES[case["type"]])
    m, v = 0.3 * size * normal(), (size * normal().abs_().clamp_min_(0.05)) ** 2 * there
    if case["bits"] == 32:
        return p, g, (m, v)
    none = torch.zeros(1, dtype=torch.int64, device="cuda")
    return p, g, _to_8_bits(m, _field(m), none, False) + _to_8_bits(v.sqrt(), (_field(v) + 127) >> 1, none, True)


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    make = {"norm": _norm_inputs, "step": _recurrence_inputs, "recurrence": _recurrence_inputs,
            "embedding": _embedding_inputs, "score": _score_inputs, "adamw": _adamw_inputs}
    return make[case["op"]](case, gen)


def prepare(case, seed):
    """the call's tensors; with the framework also what its user keeps: outputs, workspaces, the optimizer with its states"""
    st = State()
    st.case, st.inputs = case, _inputs(case, seed)
    if not own:
        return st
    ops = st.ops = _ops()
    op = case["op"]
    if op == "norm":
        x, w, _, dy = st.inputs
        st.out, st.mean, st.rstd = torch.empty_like(x), x.new_empty(len(x), dtype=torch.float32), None
        if case["train"]:
            st.rstd, st.dx, st.dw, st.db = torch.empty_like(st.mean), torch.empty_like(x), torch.empty_like(w), torch.empty_like(w)
            st.workspace = _bytes(ops.layer_norm_workspace(x))
    elif op == "step":
        z, x, state = st.inputs
        st.out, st.next = torch.empty_like(x), torch.empty_like(state)
    elif op == "recurrence":
        z, x, state = st.inputs[:3]
        st.out, st.dz, st.dx, st.next, st.dstate = (torch.empty_like(t) for t in (x, x, x, state, state))
        st.saved, st.workspace = _bytes(ops.gated_recurrence_saved(z)), _bytes(ops.gated_recurrence_workspace(z))
    elif op == "embedding":
        tokens, table, dy, before = st.inputs
        st.out = torch.empty_like(dy)
        st.grad = torch.empty(table.shape, device="cuda") if before is None else before
        st.workspace = _bytes(ops.embedding_gradient_workspace(tokens, st.grad))
    elif op == "score":
        logits = st.inputs[0]
        rows = len(logits)
        st.logprobs, st.entropy, st.stats = (torch.empty(n, device="cuda") for n in (rows, rows, (rows, 2)))
        st.top = torch.empty((rows, case["top"]), dtype=torch.int64, device="cuda") if case["top"] else None
        st.top_logprobs = torch.empty((rows, case["top"]), device="cuda") if case["top"] else None
        st.workspace = _bytes(ops.token_logprobs_workspace(logits, case["top"]))
        st.grad = torch.empty_like(logits) if case["train"] else None
    else:
        p, g, states = st.inputs
        starts, sizes = _starts(case)[0], _adamw_sizes(case)

        def parts(flat):
            return [flat[a:a + n] for a, n in zip(starts, sizes)]

        if case["bits"] == 8:
            m, me, r, re = states
            st.exponents = torch.stack((me, re), -1)
            states = (parts(m), parts(r), [st.exponents[a // BLOCK:-(-(a + n) // BLOCK)] for a, n in zip(starts, sizes)])
        else:
            states = tuple(parts(s) for s in states)
        st.copy = torch.zeros(len(p), dtype=torch.bfloat16, device="cuda") if case["bits"] == 8 else None
        st.grads = parts(g)
        st.optimizer = ops.AdamW(parts(p), betas=(ADAMW["beta1"], ADAMW["beta2"]), eps=ADAMW["eps"], weight_decay=ADAMW["decay"],
                                 bits=case["bits"], states=states, copies=None if st.copy is None else parts(st.copy))
    return st


def _bytes(need):
    return torch.empty(need, dtype=torch.uint8, device="cuda") if need else None


# ------------------------------------------------------------------------------------------------ one pass
def run(st):
    return _own(st) if own else _PLAIN[st.case["op"]](st)


def _own(st):
    ops, case, op = st.ops, st.case, st.case["op"]
    if op == "norm":
        x, w, b, dy = st.inputs
        if not case["train"]:
            ops.layer_norm(x, w, b, st.out)
            return st.out
        ops.layer_norm(x, w, b, st.out, st.mean, st.rstd)
        ops.layer_norm_backward(dy, x, w, st.mean, st.rstd, st.dx, st.dw, st.db, workspace=st.workspace)
        return {"out": st.out, "dx": st.dx, "dw": st.dw, "db": st.db}
    if op == "step":
        z, x, state = st.inputs
        ops.gated_recurrence_step(z, x, state, st.next, st.out)
        return {"out": st.out, "state": st.next}
    if op == "recurrence":
        z, x, state, lengths, dy, dlast = st.inputs
        ops.gated_recurrence(z, x, state, st.next, st.out, lengths=lengths, saved=st.saved, workspace=st.workspace)
        ops.gated_recurrence_backward(z, x, st.saved, dy, dlast, st.dz, st.dx, st.dstate, lengths=lengths,
                                      workspace=st.workspace)
        return {"out": st.out, "state": st.next, "dz": st.dz, "dx": st.dx, "dstate": st.dstate}
    if op == "embedding":
        tokens, table, dy, before = st.inputs
        ops.embedding(tokens, table, st.out, scale=2.0)
        ops.embedding_gradient(tokens, dy, st.grad, scale=2.0, accumulate=before is not None, workspace=st.workspace)
        return {"out": st.out, "grad": st.grad}
    if op == "score":
        logits, tokens, weight, weight_entropy = st.inputs
        known = {} if not case["train"] or case["later"] else \
            {"weights": weight, "entropy_weights": weight_entropy, "gradient": st.grad}
        ops.token_logprobs(logits, tokens, st.logprobs, st.entropy, st.stats, st.top, st.top_logprobs, workspace=st.workspace,
                           **known)
        out = {"logprobs": st.logprobs, "entropy": st.entropy}
        if case["top"]:
            out.update(top=st.top, top_logprobs=st.top_logprobs)
        if case["train"]:
            if case["later"]:  # weights that hang on the log-probabilities
                ops.token_logprobs_gradient(logits, tokens, st.stats, weight, st.grad, weight_entropy, st.entropy)
            out["grad"] = st.grad
        return out
    p, _, states = st.inputs
    st.optimizer.step(st.grads, lr=ADAMW["lr"], step=ADAMW["step"], seed=ADAMW["seed"])
    if case["bits"] == 8:
        return {"p": p, "copy": st.copy, "m": states[0], "root": states[2], "exponents": st.exponents}
    return {"p": p, "m": states[0], "v": states[1]}


def _plain_norm(st):
    x, w, b, dy = st.inputs
    f = x.float()
    f = f - f.mean(-1, keepdim=True)
    rstd = (f.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
    hat = f * rstd
    out = (hat * w + b).to(x.dtype)
    if dy is None:
        return out
    dy = dy.float()
    dh = dy * w
    dx = rstd * (dh - dh.mean(-1, keepdim=True) - hat * (dh * hat).mean(-1, keepdim=True))
    return {"out": out, "dx": dx.to(x.dtype), "dw": (dy * hat).sum(0), "db": dy.sum(0)}


def _plain_step(st):
    z, x, state = st.inputs
    z, x = z.float(), x.float()
    new = state * torch.sigmoid(z) + x * torch.sigmoid(-z)
    return {"out": new.to(st.inputs[1].dtype), "state": new}


def _scan(a, b):
    """b_t + a_t b_{t-1} + a_t a_{t-1} b_{t-2} + ... along axis 1, over spans that double"""
    a, b = a.clone(), b.clone()
    n = 1
    while n < a.shape[1]:
        b = torch.cat((b[:, :n], b[:, n:] + a[:, n:] * b[:, :-n]), 1)
        a = torch.cat((a[:, :n], a[:, n:] * a[:, :-n]), 1)
        n *= 2
    return b


def _plain_recurrence(st):
    z, x, state, lengths, dy, dlast = st.inputs
    kind, tokens = x.dtype, x.shape[1]
    at = torch.arange(tokens, device=x.device)
    last = torch.full((len(x),), tokens, device=x.device) if lengths is None else lengths.long()
    there = (at[None] < last[:, None])[..., None]
    z, x, dy = z.float(), x.float(), torch.where(there, dy.float(), 0.0)
    a, rest = torch.where(there, torch.sigmoid(z), 1.0), torch.where(there, torch.sigmoid(-z), 0.0)
    b = rest * x
    b[:, 0] += a[:, 0] * state
    h = _scan(a, b)
    before = torch.cat((state[:, None], h[:, :-1]), 1)
    # the gradient runs from the end: d_t = dy_t + a_{t+1} d_{t+1}, after the last token what the last state is given
    after = torch.cat((a[:, 1:], torch.ones_like(a[:, :1])), 1)
    d = dy.clone()
    d[:, -1] += dlast
    d = _scan(after.flip(1), d.flip(1)).flip(1)
    dz = d * (before - x) * a * rest
    return {"out": torch.where(there, h, 0.0).to(kind), "state": h[:, -1], "dz": dz.to(kind), "dx": (d * rest).to(kind),
            "dstate": d[:, 0] * a[:, 0]}


def _plain_embedding(st):
    tokens, table, dy, before = st.inputs
    there = (tokens >= 0)[:, None]
    at = tokens.clamp_min(0)
    out = torch.where(there, table[at].float() * 2.0, 0.0).to(table.dtype)
    grad = torch.zeros(table.shape, device=table.device) if before is None else before
    grad.index_add_(0, at, torch.where(there, dy.float() * 2.0, 0.0))
    return {"out": out, "grad": grad}


def _plain_score(st):
    logits, tokens, weight, weight_entropy = st.inputs
    x, there, at = logits.float(), tokens >= 0, tokens.clamp_min(0)[:, None]
    m = x.amax(-1, keepdim=True)
    e = (x - m).exp_()
    total = e.sum(-1, keepdim=True)
    lse = m + total.log()
    p = e.div_(total)
    logs = x - lse
    entropy = -(p * torch.where(p > 0, logs, 0.0)).sum(-1)
    out = {"logprobs": torch.where(there, logs.gather(-1, at)[:, 0], 0.0), "entropy": entropy}
    if st.case["top"]:
        top, index = (t[:, :st.case["top"]].contiguous() for t in x.sort(dim=-1, descending=True, stable=True))
        out.update(top=index, top_logprobs=top - lse)
    if weight is not None:
        weight = torch.where(there, weight, 0.0)
        grad = (weight_entropy[:, None] * (torch.where(p > 0, logs, 0.0) + entropy[:, None])).add_(weight[:, None]).mul_(p).neg_()
        grad.scatter_add_(-1, at, weight[:, None])
        out["grad"] = grad.to(logits.dtype)
    return out


def _mixed(x):
    """the 32 bits that a counter stands for"""
    x = ((x ^ (x >> 16)) * 0x9E3779B1) & 0xffffffff
    x = ((x ^ (x >> 15)) * 0xB7E15163) & 0xffffffff
    return x ^ (x >> 16)


def _field(x):
    """the exponent field of each block's largest"""
    return x.abs().view(-1, BLOCK).amax(-1, keepdim=True).view(torch.int32).long() >> 23


def _to_8_bits(x, field, draws, keep):
    """Blocks of x as float8_e4m3fn times the power of two that brings 2^(field - 127) to 2^7.  A magnitude is cut off, after a
    16-bit draw, in units of the first 16 bits that are cut off, was added to it; with `keep` what is above 0 stays above 0."""
    field = field.clamp_min(16)
    bits = x.abs().view(torch.int32).long().view(-1, BLOCK)
    up = (bits >> 23) - field + 13  # binades above the lowest whole one
    shift = (-up).clamp_min(0)
    draws = draws.view(-1, BLOCK) if draws.numel() > 1 else draws
    code = ((bits & 0x7fffff) + 0x800000 + (draws << (4 + shift).clamp(max=32))) >> (20 + shift).clamp(max=60)
    code = torch.where((bits >= 0x800000) & (shift < 12), up.clamp_min(0) * 8 + code, 0)
    if keep:
        code = torch.where((bits > 0) & (code == 0), 1, code)
    code |= (x.view(-1, BLOCK) < 0).long() << 7
    return code.to(torch.uint8).view(-1).view(torch.float8_e4m3fn), field[:, 0].to(torch.uint8)


def _of_8_bits(codes, exponent):
    return (codes.float().view(-1, BLOCK) * torch.exp2(exponent.float() - 134.0)[:, None]).view(-1)


def _draws(case, device):
    """two times 16 bits for every entry, by the step, its tensor's place and its own"""
    starts, length = _starts(case)
    begin = torch.tensor(starts, device=device)
    whole = torch.diff(begin, append=begin.new_tensor([length]))
    key = _mixed(ADAMW["seed"] + 0xB7E15163 * ADAMW["step"] + 0x9E3779B1 * torch.arange(len(starts), device=device) & 0xffffffff)
    local = torch.arange(length, device=device) - begin.repeat_interleave(whole)
    h = _mixed(key.repeat_interleave(whole) + local & 0xffffffff)
    return h & 0xffff, h >> 16


def _plain_adamw(st):
    p, g, states = st.inputs
    c, bits = ADAMW, st.case["bits"]
    if bits == 8:
        m, root = _of_8_bits(*states[:2]), _of_8_bits(*states[2:])
        v = root * root
    else:
        m, v = states
    g = g.float()
    m = m * c["beta1"] + g * (1 - c["beta1"])
    v = v * c["beta2"] + (g * g) * (1 - c["beta2"])
    root = v.sqrt()
    first, second = 1 - c["beta1"] ** c["step"], math.sqrt(1 - c["beta2"] ** c["step"])
    p.sub_(p * (c["lr"] * c["decay"]) + (c["lr"] / first) * m / (root / second + c["eps"]))
    if bits == 32:
        for old, new in zip(states, (m, v)):
            old.copy_(new)
        return {"p": p, "m": states[0], "v": states[1]}
    low, high = _draws(st.case, p.device)
    new = _to_8_bits(m, _field(m), low, False) + _to_8_bits(root, (_field(v) + 127) >> 1, high, True)
    for old, new in zip(states, new):
        old.copy_(new)
    return {"p": p, "copy": p.bfloat16(), "m": states[0], "root": states[2], "exponents": torch.stack(states[1::2], -1)}


_PLAIN = {"norm": _plain_norm, "step": _plain_step, "recurrence": _plain_recurrence, "embedding": _plain_embedding,
          "score": _plain_score, "adamw": _plain_adamw}


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    inputs = _inputs(case, seed)
    return _EXACT[case["op"]](case, *inputs)


def _exact_norm(case, x, w, b, dy):
    x, w, b = x.double(), w.double(), b.double()
    n = x.shape[1]
    mean = x.sum(1) / n
    rstd = (((x - mean[:, None]) ** 2).sum(1) / n + 1e-5) ** -0.5
    hat = (x - mean[:, None]) * rstd[:, None]
    out = hat * w + b
    if dy is None:
        return out
    dy = dy.double()
    along, flat = ((dy * w) * hat).sum(1) / n, (dy * w).sum(1) / n
    return {"out": out, "dx": rstd[:, None] * (dy * w - flat[:, None] - hat * along[:, None]), "dw": (dy * hat).sum(0),
            "db": dy.sum(0)}


def _exact_step(case, z, x, state):
    a = 1 / (1 + (-z.double()).exp())
    new = a * state.double() + (1 - a) * x.double()
    return {"out": new, "state": new}


def _exact_recurrence(case, z, x, state, lengths, dy, dlast):
    """token by token, as the recurrence is defined, and back"""
    lanes, tokens = x.shape[:2]
    ends = torch.full((lanes,), tokens, device=x.device) if lengths is None else lengths
    h, hs = state.double(), []
    out, dz, dx = (torch.zeros(x.shape, dtype=torch.float64, device=x.device) for _ in range(3))
    gate = 1 / (1 + (-z.double()).exp())
    rest = 1 / (1 + z.double().exp())
    for t in range(tokens):
        hs.append(h)
        there = (ends > t)[:, None]
        h = torch.where(there, gate[:, t] * h + rest[:, t] * x[:, t].double(), h)
        out[:, t] = torch.where(there, h, 0.0)
    d = dlast.double()
    for t in range(tokens - 1, -1, -1):
        there = (ends > t)[:, None]
        now = torch.where(there, d + dy[:, t].double(), 0.0)
        dx[:, t] = now * rest[:, t]
        dz[:, t] = now * (hs[t] - x[:, t].double()) * gate[:, t] * rest[:, t]
        d = torch.where(there, now * gate[:, t], d)
    return {"out": out, "state": h, "dz": dz, "dx": dx, "dstate": d}


def _exact_embedding(case, tokens, table, dy, before):
    """a stable order of the tokens, then differences of running sums over it, 64 channels at a time"""
    there = tokens >= 0
    out = 2 * table.double()[tokens.clamp_min(0)] * there[:, None]
    grad = torch.zeros(table.shape, dtype=torch.float64, device=table.device) if before is None else before.double()
    order = torch.sort(tokens[there], stable=True)
    ids, counts = torch.unique_consecutive(order.values, return_counts=True)
    if len(ids):
        ends = counts.cumsum(0)
        sums = dy[there][order.indices].double().cumsum(0)[ends - 1]
        grad[ids] += 2 * (sums - torch.cat((torch.zeros_like(sums[:1]), sums[:-1])))
    return {"out": out, "grad": grad}


def _exact_score(case, logits, tokens, weight, weight_entropy):
    x = logits.double()
    logs = x - torch.logsumexp(x, -1, keepdim=True)
    p = logs.exp()
    entropy = -torch.special.xlogy(p, p).sum(-1)
    rows = torch.arange(len(x), device=x.device)
    there = tokens >= 0
    out = {"logprobs": torch.where(there, logs[rows, tokens.clamp_min(0)], 0.0), "entropy": entropy}
    if case["top"]:
        order = torch.sort(-x, dim=-1, stable=True).indices[:, :case["top"]]
        out.update(top=order.contiguous(), top_logprobs=logs.gather(-1, order))
    if weight is not None:
        weight = weight.double() * there
        one = torch.zeros_like(x)
        one[rows, tokens.clamp_min(0)] = 1.0
        grad = weight[:, None] * (one - p)
        grad -= weight_entropy.double()[:, None] * (torch.special.xlogy(p, p) + p * entropy[:, None])
        out["grad"] = grad
    return out


def _exact_adamw(case, p, g, states):
    c = ADAMW
    if case["bits"] == 8:
        scale = [(2.0 ** (e.double() - 134))[:, None] for e in states[1::2]]
        m, root = ((s.double().view(-1, BLOCK) * e).view(-1) for s, e in zip(states[::2], scale))
        v = root ** 2
    else:
        m, v = (s.double() for s in states)
    p, g = p.double(), g.double()
    m, v = c["beta1"] * m + (1 - c["beta1"]) * g, c["beta2"] * v + (1 - c["beta2"]) * g ** 2
    first, second = 1 - c["beta1"] ** c["step"], 1 - c["beta2"] ** c["step"]
    p = p * (1 - c["lr"] * c["decay"]) - c["lr"] * (m / first) / ((v / second) ** 0.5 + c["eps"])
    if case["bits"] == 32:
        return {"p": p, "m": m, "v": v}
    # the moments before they are rounded: an 8-bit one is up to a step of its own away
    out = {"p": p, "copy": p, "exponents": None}
    for name, x in (("m", m), ("root", v.sqrt())):
        x = x.view(-1, BLOCK)
        _, e = torch.frexp(x.abs().amax(-1, keepdim=True))
        out[name] = torch.ldexp(x, 8 - e).view(-1)
    return out


_EXACT = {"norm": _exact_norm, "step": _exact_step, "recurrence": _exact_recurrence, "embedding": _exact_embedding,
          "score": _exact_score, "adamw": _exact_adamw}


# ------------------------------------------------------------------------------------------------ what it takes
def work(case):
    size, op = BYTES[case["type"]], case["op"]
    if op == "norm":
        n = case["rows"] * case["channels"]
        return {"bytes": (4 if case["train"] else 2) * n * size + (16 if case["train"] else 8) * case["channels"],
                "flops": (24 if case["train"] else 8) * n}
    if op == "step":
        return {"bytes": case["lanes"] * case["channels"] * (3 * size + 8), "flops": 8 * case["lanes"] * case["channels"]}
    if op == "recurrence":
        n = case["lanes"] * case["tokens"] * case["channels"] * (0.75 if case["ragged"] else 1)
        return {"bytes": 6 * n * size + 16 * case["lanes"] * case["channels"], "flops": 24 * n}
    if op == "embedding":
        n, table = case["tokens"] * case["channels"], case["vocab"] * case["channels"]
        used = min(n, table)
        return {"bytes": 8 * case["tokens"] + used * size + 2 * n * size + (8 * used if case["add"] else 4 * table),
                "flops": 3 * n}
    if op == "score":
        n = case["rows"] * case["vocab"]
        return {"bytes": (2 if case["train"] else 1) * n * size + case["rows"] * (28 + 12 * case["top"]),
                "flops": (12 if case["train"] else 6) * n}
    n = sum(_adamw_sizes(case))
    return {"bytes": n * (size + (14 if case["bits"] == 8 else 24)), "flops": 14 * n}
