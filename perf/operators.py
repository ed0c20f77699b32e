"""What a client of the encrypted decode step computes in the clear, through clear_ops.py: the recurrence of the small
model that drafts tokens (linear attention with a decay for each head, over a prompt and over one token), products with
4-bit weights (that model's projections, and the vocabulary head that turns decrypted rows into logits), and the draw
of the next token.

Each operator is here twice: `run` with `own` false computes it from elementary torch operations in 32 bits, with `own`
true it calls the framework; `exact` computes it in 64 bits.  Sizes are those of the repository's model (12 heads of 64,
768 channels, 32 lanes, 65536 tokens), or generic ones around them.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}


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
        # one token of one conversation in one layer: the smallest call of a draft, all latency
        {"name": "step one lane", "op": "step", "lanes": 1, "heads": 12, "key_heads": 12, "dk": 64, "dv": 64,
         "type": "bf16"},
        # one token of each of the 32 conversations that an encrypted step carries
        {"name": "step lanes", "op": "step", "lanes": 32, "heads": 12, "key_heads": 12, "dk": 64, "dv": 64,
         "type": "f32"},
        # one long prompt, where only the token axis has work to spread
        {"name": "prompt long", "op": "prompt", "lanes": 1, "tokens": 8192, "heads": 12, "key_heads": 12, "dk": 64,
         "dv": 64, "type": "bf16", "ragged": False},
        # the prompts of 32 conversations, each of its own length
        {"name": "prompt lanes", "op": "prompt", "lanes": 32, "tokens": 1024, "heads": 12, "key_heads": 12, "dk": 64,
         "dv": 64, "type": "bf16", "ragged": True},
        # a few short prompts in full precision, keys shared by all heads, sizes that fill no tile
        {"name": "prompt odd", "op": "prompt", "lanes": 3, "tokens": 777, "heads": 5, "key_heads": 1, "dk": 48,
         "dv": 80, "type": "f32", "ragged": True},
        # the vocabulary head for one decrypted row, and for all lanes of a step
        {"name": "head one row", "op": "product", "rows": 1, "out": 65536, "in": 768, "group": 64, "zeros": False,
         "type": "f32"},
        {"name": "head lanes", "op": "product", "rows": 32, "out": 65536, "in": 768, "group": 64, "zeros": False,
         "type": "bf16"},
        # a projection of odd sizes, the last group cut short, with zero points
        {"name": "projection odd", "op": "product", "rows": 5, "out": 1999, "in": 1101, "group": 32, "zeros": True,
         "type": "f16"},
        # the products of a large draft model
        {"name": "projection large", "op": "product", "rows": 16, "out": 16384, "in": 8192, "group": 128,
         "zeros": False, "type": "bf16"},
        # one conversation's draw with every filter on
        {"name": "draw one", "op": "draw", "rows": 1, "vocab": 65536, "filters": "all", "type": "f32"},
        # every lane's draw from its nucleus
        {"name": "draw lanes", "op": "draw", "rows": 32, "vocab": 65536, "filters": "nucleus", "type": "f32"},
        # draws for many drafted positions at once, each row with parameters of its own, an odd vocabulary
        {"name": "draw many", "op": "draw", "rows": 300, "vocab": 50277, "filters": "mixed", "type": "bf16"},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["step", "prompt", "prompt", "product", "product", "draw", "draw"])
    kind = rng.choice(["f32", "bf16", "f16"])
    if op in ("step", "prompt"):
        heads = rng.choice([1, 2, 3, 5, 8, 12, 16])
        case = {"op": op, "heads": heads, "key_heads": rng.choice([d for d in (1, 2, 3, 4, 8, heads) if heads % d == 0]),
                "dk": rng.choice([64, 64, 128, 32, rng.randint(8, 128)]),
                "dv": rng.choice([64, 64, 128, 32, rng.randint(8, 160)]), "type": kind}
        if op == "step":
            return {**case, "lanes": _log(rng, 1, 64)}
        tokens = _log(rng, 2, 8192 if kind != "f32" else 2048)
        most = max(1, min(32, int(4e8 / (heads * tokens * tokens))))  # what the plain form's square of scores allows
        return {**case, "lanes": _log(rng, 1, most), "tokens": tokens, "ragged": rng.random() < 0.5}
    if op == "product":
        rows, group = _log(rng, 1, 64), rng.choice([32, 64, 128])
        n_in = _log(rng, 64, 16384)
        return {"op": op, "rows": rows, "in": n_in, "out": _log(rng, 64, min(65536, (1 << 26) // n_in)), "group": group,
                "zeros": rng.random() < 0.5, "type": kind}
    vocab = _log(rng, 500, 131072)
    return {"op": op, "vocab": vocab, "rows": _log(rng, 1, min(300, (1 << 24) // vocab)),
            "filters": rng.choice(["none", "nucleus", "top-k", "all", "mixed"]), "type": kind}


# ------------------------------------------------------------------------------------------------ inputs
class State:
    pass


def _attention_inputs(case, gen):
    """queries, keys and values of unit size; decays that differ from head to head, from about 1/8 to 1/512 a token, and
    from token to token; a state that some earlier text left"""
    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)

    kind, lanes, heads, shared = TYPES[case["type"]], case["lanes"], case["heads"], case["key_heads"]
    shape = (lanes,) if case["op"] == "step" else (lanes, case["tokens"])
    q, k = normal(*shape, shared, case["dk"]).to(kind), normal(*shape, shared, case["dk"]).to(kind)
    v = normal(*shape, heads, case["dv"]).to(kind)
    rate = torch.exp2(-torch.linspace(3, 9, heads, device="cuda"))
    g = -rate * (0.5 + torch.rand(shape + (heads,), generator=gen, device="cuda"))
    state = 2 * normal(lanes, heads, case["dk"], case["dv"])
    lengths = None
    if case.get("ragged"):
        lengths = torch.randint(case["tokens"] // 2, case["tokens"] + 1, (lanes,), generator=gen, device="cuda",
                                dtype=torch.int32)
    return q, k, v, g, state, lengths


def _product_inputs(case, gen):
    """rows of unit size, codes as rounding a Gaussian weight leaves them, scales that keep the outputs of unit size"""
    out, n_in, group = case["out"], case["in"], case["group"]
    groups = -(-n_in // group)
    x = torch.randn((case["rows"], n_in), generator=gen, device="cuda").to(TYPES[case["type"]])
    codes = torch.randn((out, 2 * (-(-n_in // 2))), generator=gen, device="cuda").mul_(3).add_(8).round_().clamp_(0, 15)
    codes = codes.to(torch.uint8)
    codes = codes[:, 0::2] | (codes[:, 1::2] << 4)
    scales = ((0.5 + torch.rand((out, groups), generator=gen, device="cuda")) / (3 * math.sqrt(n_in))).half()
    zeros = torch.randint(4, 12, (out, groups), generator=gen, device="cuda", dtype=torch.uint8) if case["zeros"] else None
    return x, codes, scales, zeros


def _settle(logits, temperature, top_k, top_p, min_p, draws):
    """The parameters moved off the places where the answer hangs on the last bit: top-p and min-p to the middle of the
    gap they fall into, a draw to the inner half of its token's interval.  On such a place 32 bits have no right answer."""
    x, at = logits.double().sort(dim=-1, descending=True, stable=True)
    hot = (temperature > 0)[:, None]
    t = torch.where(hot, temperature[:, None], 1.0).double()
    e = ((x - x[:, :1]) / t).exp()
    rank = torch.arange(x.shape[1], device=x.device)[None]
    e = torch.where((top_k[:, None] <= 0) | (rank < top_k[:, None]), e, 0.0)
    sums = e.cumsum(-1)
    before, total = sums - e, sums[:, -1:]
    n = (before < top_p[:, None].double() * total).sum(-1, keepdim=True).clamp(1)
    middle = (before.gather(-1, n - 1) + 0.5 * e.gather(-1, n - 1)) / total
    top_p = torch.where(top_p < 1, middle[:, 0].float(), top_p)
    m = (e >= min_p[:, None]).sum(-1, keepdim=True).clamp(1)
    below = e.gather(-1, m.clamp(max=e.shape[1] - 1))
    gap = (e.gather(-1, m - 1) * below).sqrt()
    min_p = torch.where((min_p > 0) & (below > 0)[:, 0], gap[:, 0].float(), min_p)
    n = torch.where(top_p[:, None] < 1, n, e.shape[1])
    m = torch.where(min_p[:, None] > 0, m, e.shape[1])
    e = torch.where(rank < torch.where(hot, torch.minimum(n, m), 1), e, 0.0)
    w = torch.zeros_like(e).scatter_(-1, at, e)
    sums = w.cumsum(-1)
    total = sums[:, -1:]
    token = (sums <= draws[:, None].double() * total).sum(-1, keepdim=True).clamp(max=e.shape[1] - 1)
    wide = w.gather(-1, token) >= 1e-5 * total
    token = torch.where(wide, token, w.argmax(-1, keepdim=True))
    low = sums.gather(-1, token) - w.gather(-1, token)
    draws = (low + w.gather(-1, token) * (0.25 + 0.5 * draws[:, None])) / total
    return top_p, min_p, draws[:, 0].float()


def _draw_inputs(case, gen):
    """logits as a language model leaves them: a wide bulk, some tens of likely tokens well above it, a few banned ones"""
    rows, vocab = case["rows"], case["vocab"]

    def uniform(*shape):
        return torch.rand(shape, generator=gen, device="cuda")

    logits = 2 * torch.randn((rows, vocab), generator=gen, device="cuda")
    part = vocab // 48  # one likely token in each 48th of the vocabulary
    likely = torch.randint(0, part, (rows, 48), generator=gen, device="cuda") + part * torch.arange(48, device="cuda")
    logits.scatter_(-1, likely, 7 - 2.5 * uniform(rows, 48).clamp_min_(1e-6).log())
    logits[:, ::97] = -math.inf
    logits = logits.to(TYPES[case["type"]])
    kind, ones = case["filters"], torch.ones(rows, device="cuda")
    temperature, top_p, min_p = 0.6 + 0.6 * uniform(rows), ones.clone(), 0 * ones
    top_k = torch.zeros(rows, device="cuda", dtype=torch.int32)
    each = torch.arange(rows, device="cuda")
    if kind in ("all", "top-k", "mixed"):
        top_k = torch.randint(1, 100, (rows,), generator=gen, device="cuda", dtype=torch.int32)
        top_k = torch.where(each % 3 == 1, 0, top_k) if kind == "mixed" else top_k
    if kind in ("all", "nucleus", "mixed"):
        top_p = 0.7 + 0.29 * uniform(rows)
        top_p = torch.where(each % 4 == 2, 1.0, top_p) if kind == "mixed" else top_p
    if kind in ("all", "mixed"):
        min_p = 0.005 + 0.1 * uniform(rows)
        min_p = torch.where(each % 5 > 0, 0.0, min_p) if kind == "mixed" else min_p
    if kind == "mixed":
        temperature = torch.where(each % 7 == 3, 0.0, temperature)
    top_p, min_p, draws = _settle(logits, temperature, top_k, top_p, min_p, uniform(rows))
    return logits, draws, temperature, top_k, top_p, min_p


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    make = {"step": _attention_inputs, "prompt": _attention_inputs, "product": _product_inputs, "draw": _draw_inputs}
    return make[case["op"]](case, gen)


def prepare(case, seed):
    """the call's tensors; with the framework also what its user keeps: the weights laid out once, the workspace, the
    output buffers"""
    st = State()
    st.case, st.inputs = case, _inputs(case, seed)
    st.scale = case["dk"] ** -0.5 if "dk" in case else 1.0
    if not own:
        return st
    st.ops, kind = _ops(), TYPES[case["type"]]
    if case["op"] in ("step", "prompt"):
        q, k, v, g, state, lengths = st.inputs
        st.out, st.next = torch.empty_like(v), torch.empty_like(state)
        if case["op"] == "prompt":
            need = st.ops.linear_attention_workspace(q, k, v)
            st.workspace = torch.empty(need, dtype=torch.uint8, device="cuda") if need else None
    elif case["op"] == "product":
        x, codes, scales, zeros = st.inputs
        st.weights = st.ops.Q4Matrix(codes, scales, zeros, in_features=case["in"], group=case["group"])
        st.out = torch.empty((case["rows"], case["out"]), dtype=kind, device="cuda")
    else:
        st.tokens = torch.empty(case["rows"], dtype=torch.int64, device="cuda")
        st.logprobs = torch.empty(case["rows"], dtype=torch.float32, device="cuda")
    return st


# ------------------------------------------------------------------------------------------------ one pass
def run(st):
    return _own(st) if own else _PLAIN[st.case["op"]](st)


def _own(st):
    ops, op = st.ops, st.case["op"]
    if op == "product":
        st.weights.product(st.inputs[0], st.out)
        return st.out
    if op == "draw":
        logits, draws, temperature, top_k, top_p, min_p = st.inputs
        ops.sample(logits, draws, st.tokens, st.logprobs, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
        return {"tokens": st.tokens, "logprobs": st.logprobs}
    q, k, v, g, state, lengths = st.inputs
    if op == "step":
        ops.linear_attention_step(q, k, v, g, state, st.next, st.out, scale=st.scale)
    else:
        ops.linear_attention_prompt(q, k, v, g, state, st.next, st.out, scale=st.scale, lengths=lengths,
                                    workspace=st.workspace)
    return {"out": st.out, "state": st.next}


def _plain_step(st):
    q, k, v, g, state, _ = st.inputs
    each = st.case["heads"] // st.case["key_heads"]
    q, k = (x.float().repeat_interleave(each, 1) for x in (q, k))
    new = state * g.exp()[..., None, None] + k[..., :, None] * v.float()[..., None, :]
    out = (q[..., :, None] * new).sum(-2) * st.scale
    return {"out": out.to(v.dtype), "state": new}


def _plain_prompt(st):
    q, k, v, g, state, lengths = st.inputs
    tokens, each = st.case["tokens"], st.case["heads"] // st.case["key_heads"]
    at = torch.arange(tokens, device=v.device)
    there = torch.ones((v.shape[0], tokens), dtype=torch.bool, device=v.device) if lengths is None \
        else at[None] < lengths[:, None]
    there = there[:, None, :]  # lanes, heads, tokens
    q, k = (x.float().repeat_interleave(each, 2).transpose(1, 2) for x in (q, k))
    values = v.float().transpose(1, 2).contiguous()
    g = torch.where(there, g.transpose(1, 2), 0.0)
    k = torch.where(there[..., None], k, 0.0)
    sums = g.cumsum(-1)
    decay = (sums[..., :, None] - sums[..., None, :]).masked_fill_(at[None] > at[:, None], -math.inf).exp_()
    scores = (q @ k.transpose(-1, -2).contiguous()).mul_(decay)
    out = (scores @ values + (q * sums.exp()[..., None]) @ state) * st.scale
    out = torch.where(there[..., None], out, 0.0).transpose(1, 2)
    left = g.flip(-1).cumsum(-1).flip(-1) - g  # the decay from after a token to the end
    new = (k * left.exp()[..., None]).transpose(-1, -2).contiguous() @ values + state * sums[..., -1:, None].exp()
    return {"out": out.to(v.dtype).contiguous(), "state": new}


def _plain_product(st):
    x, codes, scales, zeros = st.inputs
    n_in, group = st.case["in"], st.case["group"]
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(1)[:, :n_in].float()
    z = 8.0 if zeros is None else zeros.float().repeat_interleave(group, 1)[:, :n_in]
    w = (c - z) * scales.float().repeat_interleave(group, 1)[:, :n_in]
    return (x.float() @ w.t().contiguous()).to(x.dtype)


def _plain_draw(st):
    logits, draws, temperature, top_k, top_p, min_p = (x[:, None] if x.dim() == 1 else x for x in st.inputs)
    x = logits.float()
    v, at = x.sort(dim=-1, descending=True, stable=True)
    hot = temperature > 0
    t = torch.where(hot, temperature, 1.0)
    e = ((v - v[:, :1]) / t).exp()
    rank = torch.arange(x.shape[1], device=x.device)[None]
    e = torch.where((top_k <= 0) | (rank < top_k), e, 0.0)
    sums = e.cumsum(-1)
    keep = ((top_p >= 1) | (sums - e < top_p * sums[:, -1:])) & ((min_p <= 0) | (e >= min_p))
    e = torch.where(torch.where(hot, keep, rank == 0), e, 0.0)
    sums = torch.zeros_like(e).scatter_(-1, at, e).cumsum(-1)
    token = (sums <= draws * sums[:, -1:]).sum(-1, keepdim=True)
    logprob = (x.gather(-1, token) - v[:, :1]) / t - e[:, 1:].sum(-1, keepdim=True).log1p()  # e of the largest is 1
    return {"tokens": token[:, 0], "logprobs": logprob[:, 0]}


_PLAIN = {"step": _plain_step, "prompt": _plain_prompt, "product": _plain_product, "draw": _plain_draw}


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    inputs = _inputs(case, seed)
    if case["op"] in ("step", "prompt"):
        return _exact_recurrence(case, *inputs)
    if case["op"] == "product":
        return _exact_product(case, *inputs)
    return _exact_draw(*(x.double().cpu().numpy() for x in inputs))


def _exact_recurrence(case, q, k, v, g, state, lengths):
    """token by token, as the recurrence is defined"""
    if case["op"] == "step":
        q, k, v, g = q[:, None], k[:, None], v[:, None], g[:, None]
    each = case["heads"] // case["key_heads"]
    state, outs = state.double(), []
    for t in range(v.shape[1]):
        kt, qt = (x[:, t].double().repeat_interleave(each, 1).unsqueeze(-1) for x in (k, q))
        new = state * g[:, t].double().exp()[:, :, None, None] + kt * v[:, t].double().unsqueeze(-2)
        out = (qt * new).sum(-2) / math.sqrt(case["dk"])
        if lengths is not None:
            there = (lengths > t)[:, None, None]
            new, out = torch.where(there[..., None], new, state), torch.where(there, out, 0.0)
        state = new
        outs.append(out)
    out = torch.stack(outs, 1)
    return {"out": out[:, 0] if case["op"] == "step" else out, "state": state}


def _exact_product(case, x, codes, scales, zeros):
    """group by group: the scale times what the codes give, less the zero point times the group's sum"""
    group, n_in, rows = case["group"], case["in"], case["rows"]
    total = torch.zeros((rows, case["out"]), dtype=torch.float64, device=x.device)
    for n, start in enumerate(range(0, n_in, group)):
        j = torch.arange(start, min(start + group, n_in), device=x.device)
        c = ((codes[:, j // 2] >> (4 * (j % 2)).to(torch.uint8)) & 15).double()
        part = x[:, j].double()
        z = 8.0 if zeros is None else zeros[:, n].double()
        total += scales[:, n].double() * (part @ c.t().contiguous() - z * part.sum(-1, keepdim=True))
    return total


def _exact_draw(logits, draws, temperature, top_k, top_p, min_p):
    """row by row, as the draw is defined"""
    tokens, logprobs = [], []
    for r, x in enumerate(logits):
        order = np.argsort(-x, kind="stable")
        if temperature[r] <= 0:
            tokens.append(int(order[0]))
            logprobs.append(0.0)
            continue
        order = order[:int(top_k[r])] if top_k[r] > 0 else order
        p = np.exp((x[order] - x[order[0]]) / temperature[r])
        p /= p.sum()
        kept = np.ones(len(p), dtype=bool)
        if top_p[r] < 1:
            kept &= np.concatenate(([0.0], np.cumsum(p)[:-1])) < top_p[r]
        if min_p[r] > 0:
            kept &= p >= min_p[r] * p[0]
        weight = np.zeros(len(x))
        weight[order[kept]] = p[kept] / p[kept].sum()
        token = int(np.searchsorted(np.cumsum(weight), draws[r], side="right"))
        tokens.append(token)
        logprobs.append(math.log(weight[token]))
    return {"tokens": np.array(tokens, dtype=np.int64), "logprobs": np.array(logprobs)}


# ------------------------------------------------------------------------------------------------ what it takes
def work(case):
    size = BYTES[case["type"]]
    if case["op"] in ("step", "prompt"):
        tokens = 1 if case["op"] == "step" else 0.75 * case["tokens"] if case["ragged"] else case["tokens"]
        one = 2 * case["key_heads"] * case["dk"] * size + 2 * case["heads"] * case["dv"] * size + 4 * case["heads"]
        square = case["heads"] * case["dk"] * case["dv"]
        return {"bytes": case["lanes"] * (tokens * one + 8 * square), "flops": case["lanes"] * tokens * 4 * square}
    if case["op"] == "product":
        rows, out, n_in, groups = case["rows"], case["out"], case["in"], -(-case["in"] // case["group"])
        weights = out * (n_in / 2 + groups * (3 if case["zeros"] else 2))
        return {"bytes": weights + rows * (n_in + out) * size, "flops": 2 * rows * out * n_in}
    return {"bytes": case["rows"] * (case["vocab"] * size + 32), "flops": 4 * case["rows"] * case["vocab"]}
