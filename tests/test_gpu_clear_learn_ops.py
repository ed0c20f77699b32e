"""GPU tests of what scores and trains the drafting model (layer norm, gated recurrence, embedding, token log-probabilities,
AdamW through clear_ops.py) against their definitions in 64 bits.

Tolerances are derived from the arithmetic, not from results, at each check: a float32 sum of n rounded terms is off by at most
about n 2^-24 of the sum of their magnitudes, and an output in a 16-bit type is rounded once more (test_gpu_clear_ops.py).
"""
import math

import numpy as np
import pytest

from engine_loader import load_module
from test_gpu_clear_ops import LOWEST, ROUNDING, TYPES, assert_near

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

U = 2.0**-24


def ops():
    return load_module("clear_ops")


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def workspace(need):
    return torch.full((need,), 255, dtype=torch.uint8, device="cuda") if need else None


def assert_within(got, want, allowed):
    """got within `allowed` of want, and one rounding to its type"""
    g = got.double()
    assert torch.isfinite(g).all()
    allowed = allowed * (1 + ROUNDING[got.dtype]) + ROUNDING[got.dtype] * want.abs() + LOWEST[got.dtype]
    worst = ((g - want).abs() / allowed).max().item() if g.numel() else 0.0
    assert worst <= 1, f"{worst} times the allowed error"


# ------------------------------------------------------------------------------------------------ layer norm
def norm_case(rows, d, kind, seed, offset=0.0):
    gen = generator(seed)
    x = (normal(gen, rows, d) * (0.2 + torch.rand((rows, 1), generator=gen, device="cuda")) + offset).to(kind)
    return x, 1 + 0.3 * normal(gen, d), 0.3 * normal(gen, d), normal(gen, rows, d).to(kind)


def check_norm(x, w, b, dy, eps=1e-5, out=None, dx=None):
    """A lane adds up to 32 elements and the lanes' sums meet in 10 steps more, so the mean is off by 44 2^-24 mean|x| (called q
    once it is times rstd), rstd by as much of itself and a few roundings: h by 64 2^-24 (|h| + q)."""
    c = ops()
    rows, d = x.shape
    X, W = x.double(), torch.ones(d, dtype=torch.float64, device="cuda") if w is None else w.double()
    B = torch.zeros(d, dtype=torch.float64, device="cuda") if b is None else b.double()
    mean = X.mean(1, keepdim=True)
    rstd = ((X - mean).square().mean(1, keepdim=True) + eps) ** -0.5
    h, q = (X - mean) * rstd, rstd * X.abs().mean(1, keepdim=True)
    out = torch.full_like(x, 7.0) if out is None else out
    m, r = torch.full((rows,), 7.0, device="cuda"), torch.full((rows,), 7.0, device="cuda")
    c.layer_norm(x, w, b, out, m, r, eps=eps)
    assert_within(out, h * W + B, 64 * U * (W.abs() * (h.abs() + q) + B.abs()))
    # dx: t = dy w, its mean, and h times the mean of t h, each factor off by 64 2^-24 of |h| + q
    T = dy.double() * W
    want = rstd * (T - T.mean(1, keepdim=True) - h * (T * h).mean(1, keepdim=True))
    H = h.abs() + q
    size = rstd * (T.abs() + T.abs().mean(1, keepdim=True) + H * (T.abs() * H).mean(1, keepdim=True))
    dx = torch.full_like(x, 7.0) if dx is None else dx
    dw, db = torch.full((d,), 7.0, device="cuda"), torch.full((d,), 7.0, device="cuda")
    c.layer_norm_backward(dy, x, w, m, r, dx, dw, db, workspace=workspace(c.layer_norm_workspace(x)))
    assert_within(dx, want, 160 * U * size)
    assert_within(dw, (dy.double() * h).sum(0), (rows + 128) * U * (dy.double().abs() * H).sum(0))
    assert_within(db, dy.double().sum(0), (rows + 64) * U * dy.double().abs().sum(0))
    return out, dx, dw, db, m, r


@pytest.mark.parametrize("d", [1, 2, 15, 16, 64, 65, 128, 129, 256, 257, 512, 513, 768, 1024, 1025, 1101, 2048, 2049, 4095, 4096,
                               8192, 8200, 16383, 16384])
@pytest.mark.parametrize("kind", TYPES)
def test_norm_channels(d, kind):
    print(f"{d} channels, {kind}", flush=True)
    for rows in (1, 37):
        check_norm(*norm_case(rows, d, TYPES[kind], d + rows))


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 31, 33, 700, 4097, 9001])
@pytest.mark.parametrize("d", [48, 768, 2300])
def test_norm_rows(rows, d):
    check_norm(*norm_case(rows, d, torch.bfloat16, rows + d))


@pytest.mark.parametrize("kind", TYPES)
def test_norm_rows_far_from_zero(kind):
    """a mean of 3000 over rows of size 1: what a difference of two sums of squares would lose (of float16 the rows' own bits
    are what is left)"""
    check_norm(*norm_case(50, 768, TYPES[kind], 3, offset=3000.0 if kind == "f32" else 60.0))


def test_norm_without_weight_or_bias_and_with_weights_of_the_rows_type():
    x, w, b, dy = norm_case(40, 768, torch.bfloat16, 5)
    for weight, bias in ((None, None), (w, None), (None, b), (w.bfloat16(), b.bfloat16()), (w.bfloat16(), None)):
        check_norm(x, weight, bias, dy)


@pytest.mark.parametrize("kind", TYPES)
def test_norm_strides(kind):
    """columns of a wider matrix at an odd place, one row for all, outputs with gaps that stay as they were"""
    gen, d = generator(8), 321
    wide = normal(gen, 20, 3 * d + 5).to(TYPES[kind])
    x, dy = wide[:, 3:3 + d], wide[:1, 3 + d:3 + 2 * d].expand(20, d)
    w, b = 1 + 0.1 * normal(gen, d), normal(gen, d)
    gaps = torch.full((20, 2 * d + 3), 7.0, device="cuda").to(TYPES[kind])
    check_norm(x, w, b, dy, out=gaps[:, 1:1 + d], dx=gaps[:, 2 + d:2 + 2 * d])
    assert (gaps[:, 0] == 7).all() and (gaps[:, 1 + d] == 7).all() and (gaps[:, -1] == 7).all()


def test_norm_in_place_and_parts_of_the_outputs():
    c = ops()
    x, w, b, dy = norm_case(300, 768, torch.bfloat16, 9)
    out, dx, dw, db, m, r = check_norm(x, w, b, dy)
    y = x.clone()
    c.layer_norm(y, w, b, y)
    assert torch.equal(y, out)
    need = workspace(c.layer_norm_workspace(x))
    g, one = dy.clone(), torch.empty_like(dw)
    c.layer_norm_backward(g, x, w, m, r, g, workspace=None)
    assert torch.equal(g, dx)
    c.layer_norm_backward(dy, x, w, m, r, g, dweight=one, workspace=need)
    assert torch.equal(one, dw)
    c.layer_norm_backward(dy, x, w, m, r, g, dbias=one, workspace=need)
    assert torch.equal(one, db)


def test_norm_of_equal_channels_and_of_no_rows():
    c = ops()
    x = torch.full((3, 100), 2.5, device="cuda")
    b = torch.arange(100.0, device="cuda")
    out, m, r = torch.empty_like(x), torch.empty(3, device="cuda"), torch.empty(3, device="cuda")
    c.layer_norm(x, None, b, out, m, r)
    assert torch.equal(out, b.expand(3, 100)) and (m == 2.5).all()
    none = x[:0]
    dw, db = torch.full((100,), 7.0, device="cuda"), torch.full((100,), 7.0, device="cuda")
    c.layer_norm(none, None, b, out[:0])
    c.layer_norm_backward(none, none, None, m[:0], r[:0], none.clone(), dw, db)
    assert (dw == 0).all() and (db == 0).all()


def test_norm_of_a_row_that_is_not_finite():
    c = ops()
    x, w, b, _ = norm_case(9, 500, torch.float32, 2)
    want = torch.empty_like(x)
    c.layer_norm(x, w, b, want)
    x[3, 17], x[6, 499] = math.nan, math.inf
    out = torch.empty_like(x)
    c.layer_norm(x, w, b, out)
    keep = torch.tensor([i not in (3, 6) for i in range(9)], device="cuda")
    assert torch.isnan(out[3]).all() and torch.isnan(out[6]).all() and torch.equal(out[keep], want[keep])


# ------------------------------------------------------------------------------------------------ gated recurrence
def recurrence(z, x, state, lengths, dy, dlast):
    """the definition, token by token in 64 bits, and back"""
    B, T, C = x.shape
    z, x, h, dy, d = z.double(), x.double(), state.double(), dy.double(), dlast.double()
    a, r = torch.sigmoid(z), torch.sigmoid(-z)
    out, dz, dx = (torch.zeros((B, T, C), dtype=torch.float64, device="cuda") for _ in range(3))
    hs = []
    for t in range(T):
        hs.append(h)
        there = (lengths > t)[:, None]
        h = torch.where(there, a[:, t] * h + r[:, t] * x[:, t], h)
        out[:, t] = torch.where(there, h, 0.0)
    for t in range(T - 1, -1, -1):
        there = (lengths > t)[:, None]
        now = torch.where(there, d + dy[:, t], 0.0)
        dx[:, t] = now * r[:, t]
        dz[:, t] = now * a[:, t] * r[:, t] * (hs[t] - x[:, t])
        d = torch.where(there, now * a[:, t], d)
    return out, h, dz, dx, d, hs


def gates_case(B, T, C, kind, seed, shift=2.0):
    gen = generator(seed)
    return ((normal(gen, B, T, C) + shift).to(kind), normal(gen, B, T, C).to(kind), normal(gen, B, C),
            normal(gen, B, T, C).to(kind), normal(gen, B, C))


def run_recurrence(z, x, state, dy, dlast, lengths=None, out=None, dz=None, dx=None):
    c = ops()
    B, T, C = x.shape
    out, dz, dx = (torch.full((B, T, C), 7.0, device="cuda").to(x.dtype) if t is None else t for t in (out, dz, dx))
    last, dstate = torch.full((B, C), 7.0, device="cuda"), torch.full((B, C), 7.0, device="cuda")
    saved, work = workspace(c.gated_recurrence_saved(z)), workspace(c.gated_recurrence_workspace(z))
    if saved is None:
        saved = torch.empty(0, dtype=torch.uint8, device="cuda")
    c.gated_recurrence(z, x, state, last, out, lengths=lengths, saved=saved, workspace=work)
    if work is not None:
        work.fill_(255)
    c.gated_recurrence_backward(z, x, saved, dy, dlast, dz, dx, dstate, lengths=lengths, workspace=work)
    torch.cuda.synchronize()
    return out, last, dz, dx, dstate


def check_recurrence(z, x, state, dy, dlast, lengths=None, **more):
    """Gates are off by (|z| + 4) 2^-24 of themselves at most where they are small and by 4 2^-24 near 1, a term of a state by its
    gates', of which up to T stand in a product, and two roundings a token; dz takes a product of a state and a gradient."""
    B, T, C = x.shape
    full = torch.full((B,), T, device="cuda") if lengths is None else lengths.clamp(0, T)
    zero = torch.zeros((B, C), device="cuda")
    want = recurrence(z, x, zero if state is None else state, full, torch.zeros_like(x) if dy is None else dy,
                      zero if dlast is None else dlast)
    size = recurrence(z, x.abs(), (zero if state is None else state).abs(), full, (torch.zeros_like(x) if dy is None else dy).abs(),
                      (zero if dlast is None else dlast).abs())
    got = run_recurrence(z, x, state, dy, dlast, lengths, **more)
    most = z.double().abs().clamp(max=100).max().item() if z.numel() else 0.0
    terms = 8 * T + 2 * most + 64
    assert_within(got[0], want[0], terms * U * size[0])
    assert_within(got[1], want[1], terms * U * size[1])
    assert_within(got[3], want[3], terms * U * size[3])
    assert_within(got[4], want[4], terms * U * size[4])
    if T:
        Z = z.double()
        both = size[3] * torch.sigmoid(Z) * (torch.stack(size[5], 1) + x.double().abs())
        assert_within(got[2], want[2], 2 * terms * U * both)
    return got


@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 31, 127, 128, 129, 255, 256, 257, 500, 1100])
@pytest.mark.parametrize("kind", TYPES)
def test_recurrence_lengths(T, kind):
    print(f"{T} tokens, {kind}", flush=True)
    check_recurrence(*gates_case(2, T, 70, TYPES[kind], T))


@pytest.mark.parametrize("C", [1, 2, 63, 64, 65, 768, 1000])
def test_recurrence_channels(C):
    for T in (3, 300):
        check_recurrence(*gates_case(3, T, C, torch.bfloat16, C + T))


@pytest.mark.parametrize("lanes, T", [(1, 5000), (3, 2100), (40, 200), (150, 9)])
def test_recurrence_lanes_few_and_many(lanes, T):
    """long texts in segments, and lanes that fill the GPU"""
    check_recurrence(*gates_case(lanes, T, 128, torch.float32, lanes, shift=4.0))


@pytest.mark.parametrize("T", [11, 12, 13, 24, 35, 36, 37, 95, 96, 97])
@pytest.mark.parametrize("kind", TYPES)
def test_recurrence_short_texts(T, kind):
    """around what one wave, three and eight take, with lengths of their own, and gradients of the state or of the outputs alone"""
    lengths = torch.tensor([T, 0, T - 1, 1, T // 2], dtype=torch.int32, device="cuda")
    z, x, state, dy, dlast = gates_case(5, T, 65, TYPES[kind], T)
    check_recurrence(z, x, state, dy, dlast, lengths)
    check_recurrence(z, x, None, None, dlast)
    check_recurrence(z, x, state, dy, None)


@pytest.mark.parametrize("T", [7, 130, 900])
def test_recurrence_ragged_lengths_hide_what_lies_behind(T):
    lengths = torch.tensor([0, 1, T // 2, T - 1, T, T + 5, -3], dtype=torch.int32, device="cuda")
    z, x, state, dy, dlast = gates_case(len(lengths), T, 66, torch.float32, T)
    want = check_recurrence(z, x, state, dy, dlast, lengths)
    for b, n in enumerate(lengths.clamp(0, T).tolist()):
        z[b, n:], x[b, n:], dy[b, n:] = math.nan, math.inf, math.nan
    got = run_recurrence(z, x, state, dy, dlast, lengths)
    assert all(torch.equal(g, w) for g, w in zip(got, want))
    assert torch.equal(got[1][0], state[0]) and torch.equal(got[4][0], dlast[0]) and (got[2][0] == 0).all()


def test_recurrence_of_no_tokens_hands_the_state_on():
    z, x, state, dy, dlast = gates_case(2, 0, 40, torch.bfloat16, 1)
    out, last, _, _, dstate = run_recurrence(z, x, state, dy, dlast)
    assert out.numel() == 0 and torch.equal(last, state) and torch.equal(dstate, dlast)
    ops().gated_recurrence_backward(z, x, None, dy, dlast, z.clone(), z.clone(), dstate.fill_(7))  # nothing is saved of nothing
    assert torch.equal(dstate, dlast)


@pytest.mark.parametrize("T", [40, 700])
def test_recurrence_states(T):
    """none before, none kept, no gradient from behind or of the outputs, the same buffer for both"""
    c = ops()
    z, x, state, dy, dlast = gates_case(1, T, 64, torch.bfloat16, T)
    check_recurrence(z, x, None, dy, None)
    check_recurrence(z, x, state, None, dlast)
    want = check_recurrence(z, x, state, dy, dlast)
    saved, work = workspace(c.gated_recurrence_saved(z)), workspace(c.gated_recurrence_workspace(z))
    assert (work is not None) == (T == 700)
    kept, out, dkept, dz, dx = state.clone(), torch.empty_like(x), dlast.clone(), torch.empty_like(x), torch.empty_like(x)
    c.gated_recurrence(z, x, kept, kept, out, saved=saved, workspace=work)
    c.gated_recurrence_backward(z, x, saved, dy, dkept, dz, dx, dkept, workspace=work)
    assert all(torch.equal(a, b) for a, b in zip((out, kept, dz, dx, dkept), want))
    c.gated_recurrence(z, x, state, None, out, workspace=work)  # serving: nothing kept for a backward pass
    assert torch.equal(out, want[0])
    c.gated_recurrence_backward(z, x, saved, dy, dlast, dz, dx, workspace=work)
    assert torch.equal(dz, want[2]) and torch.equal(dx, want[3])


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_recurrence_gates_at_their_ends(kind):
    """gates that keep everything or nothing, and infinite ones"""
    z, x, state, dy, dlast = gates_case(2, 300, 6, TYPES[kind], 4)
    z[:, :, 0], z[:, ::3, 1], z[:, :, 2], z[:, 1::4, 3], z[:, ::5, 4] = 30.0, -30.0, -80.0, 80.0, -math.inf
    z[:, ::7, 5] = math.inf
    check_recurrence(z, x, state, dy, dlast)


@pytest.mark.parametrize("T", [100, 600])
def test_recurrence_values_that_are_not_finite_stay_in_their_future(T):
    z, x, state, dy, dlast = gates_case(1, T, 70, torch.float32, T)
    want = run_recurrence(z, x, state, dy, dlast)
    x[0, T // 2, 7], x[0, T - 1, 69] = math.nan, math.inf
    got = run_recurrence(z, x, state, dy, dlast)
    keep = torch.ones(70, dtype=torch.bool, device="cuda")
    keep[[7, 69]] = False
    assert all(torch.equal(g[..., keep], w[..., keep]) for g, w in zip(got, want))
    assert torch.equal(got[0][0, :T // 2, 7], want[0][0, :T // 2, 7]) and not torch.isfinite(got[0][0, T // 2:, 7]).any()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("T", [9, 260])
def test_recurrence_strides(T, kind):
    """slices of one projection's rows, tokens before lanes, one lane's values for all, gaps in the outputs"""
    B, C, gen = 3, 50, generator(T)
    rows = normal(gen, T, B, 3 + 3 * C + 5).to(TYPES[kind]).transpose(0, 1)
    z, x, dy = rows[..., 3:3 + C], rows[:1, :, 3 + C:3 + 2 * C].expand(B, T, C), rows[..., 3 + 2 * C:3 + 3 * C]
    gaps = [torch.full((T, B, C + 3), 7.0, device="cuda").to(TYPES[kind]) for _ in range(3)]
    out, dz, dx = (g[..., 1:1 + C].transpose(0, 1) for g in gaps)
    check_recurrence(z, x, normal(gen, B, C), dy, normal(gen, B, C), out=out, dz=dz, dx=dx)
    for g in gaps:
        assert (g[..., 0] == 7).all() and (g[..., 1 + C:] == 7).all()


def test_recurrence_offsets_past_32_bits():
    """a lane whose rows begin past 2^32 bytes and past 2^31 elements"""
    B, T, C = 2, 140, 64
    far = (1 << 31) + 4096
    pool = torch.zeros(far + T * C, dtype=torch.bfloat16, device="cuda")
    z, x, state, dy, dlast = gates_case(B, T, C, torch.bfloat16, 5)
    want = check_recurrence(z, x, state, dy, dlast)
    view = pool.as_strided((B, T, C), (far, C, 1))
    for name, t in (("z", z), ("x", x), ("dy", dy)):
        view.copy_(t)
        got = run_recurrence(view if name == "z" else z, view if name == "x" else x, state, view if name == "dy" else dy, dlast)
        assert all(torch.equal(g, w) for g, w in zip(got, want))
    for i, name in ((0, "out"), (2, "dz"), (3, "dx")):
        run_recurrence(z, x, state, dy, dlast, **{name: view})
        assert torch.equal(view, want[i])


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("lanes, C", [(1, 1), (32, 768), (5, 100)])
def test_recurrence_step(lanes, C, kind):
    c = ops()
    z, x, state, dy, dlast = gates_case(lanes, 1, C, TYPES[kind], lanes + C)
    want, left, *_ = recurrence(z, x, state, torch.ones(lanes, device="cuda"), dy, dlast)
    out, into = torch.full_like(x[:, 0], 7.0), torch.full_like(state, 7.0)
    c.gated_recurrence_step(z[:, 0], x[:, 0], state, into, out)
    size = (state.abs() + x[:, 0].abs()).double()
    assert_within(out, want[:, 0], 80 * U * size)
    assert_within(into, left, 80 * U * size)
    again = state.clone()
    c.gated_recurrence_step(z[:, 0], x[:, 0], again, again, out)
    assert torch.equal(again, into)


def test_recurrence_steps_continue_a_prompt():
    T, more = 130, 5
    z, x, state, dy, dlast = gates_case(2, T + more, 64, torch.float32, 8)
    want = check_recurrence(z, x, state, dy, dlast)
    _, into, *_ = run_recurrence(z[:, :T], x[:, :T], state, dy[:, :T], dlast)
    out = torch.empty_like(x[:, 0])
    for t in range(T, T + more):
        ops().gated_recurrence_step(z[:, t], x[:, t], into, into, out)
        assert ((out - want[0][:, t]).abs() <= 2 * (8 * (T + more) + 80) * U * 5).all()
    assert ((into - want[1]).abs() <= 2 * (8 * (T + more) + 80) * U * 5).all()


def test_recurrence_gradients_against_differences():
    """central differences of the outputs in 64 bits, weighted, at a few entries: what the formulas of `recurrence` say"""
    z, x, state, dy, dlast = gates_case(1, 40, 3, torch.float32, 6)
    full = torch.full((1,), 40, device="cuda")
    _, _, dz, dx, dstate = run_recurrence(z, x, state, dy, dlast)

    def value(z, x, state):
        out, last, *_ = recurrence(z, x, state, full, dy, dlast)
        return ((out * dy.double()).sum() + (last * dlast.double()).sum()).item()

    step = 2.0**-12  # what is left is of its square, the next derivatives (below 10), and 2^-53 of the value over it
    for name, at in (("z", (0, 0, 0)), ("z", (0, 17, 2)), ("z", (0, 39, 1)), ("x", (0, 0, 1)), ("x", (0, 38, 0)), ("state", (0, 2))):
        ends = []
        for sign in (1, -1):
            v = {"z": z.double(), "x": x.double(), "state": state.double()}
            v[name] = v[name].clone()
            v[name][at] += sign * step
            ends.append(value(**v))
        got = {"z": dz, "x": dx, "state": dstate}[name][at].item()
        assert abs(got - (ends[0] - ends[1]) / (2 * step)) <= 10 * step**2 + 1e-4, (name, at)


# ------------------------------------------------------------------------------------------------ embedding
def run_gradient(tokens, dout, dtable, scale=1.0, accumulate=False):
    c = ops()
    c.embedding_gradient(tokens, dout, dtable, scale=scale, accumulate=accumulate,
                         workspace=workspace(c.embedding_gradient_workspace(tokens, dtable)))
    torch.cuda.synchronize()
    return dtable


def check_embedding(tokens, table, dout, scale=1.0, kind=torch.float32):
    """the lookup is one product and one rounding; a row's sum of n rows is off by n 2^-24 of their magnitudes"""
    c = ops()
    vocab, d = table.shape
    n = len(tokens)
    there = ((tokens >= 0) & (tokens < vocab))[:, None]
    at = tokens.clamp(0, vocab - 1)
    out = torch.full((n, d), 7.0, device="cuda").to(dout.dtype)
    c.embedding(tokens, table, out, scale=scale)
    assert torch.equal(out, torch.where(there, table[at].float() * scale, 0.0).to(dout.dtype))
    want, size = (torch.zeros((vocab, d), dtype=torch.float64, device="cuda") for _ in range(2))
    rows = torch.where(there, dout.double() * scale, 0.0)
    want.index_add_(0, at, rows)
    size.index_add_(0, at, rows.abs())
    count = torch.zeros(vocab, device="cuda").index_add_(0, at, there[:, 0].float())[:, None]
    grad = run_gradient(tokens, dout, torch.full((vocab, d), 7.0, device="cuda").to(kind), scale)
    assert_within(grad, want, (count + 2) * U * size)
    assert (grad[(count == 0)[:, 0]] == 0).all()
    # rows that are added up in 16 bits are rounded once more; what no token names stays as it was
    before = normal(generator(1), vocab, d).to(kind)
    more = run_gradient(tokens, dout, before.clone(), scale, accumulate=True)
    assert_within(more, before.double() + want, (count + 3) * U * (size + before.double().abs()))
    assert torch.equal(more[(count == 0)[:, 0]], before[(count == 0)[:, 0]])
    assert torch.equal(run_gradient(tokens, dout, torch.empty_like(grad), scale), grad)  # whatever runs when
    return grad


def some_tokens(n, vocab, seed, shape):
    gen = generator(seed)
    if shape == "all":
        t = torch.randint(0, vocab, (n,), generator=gen, device="cuda")
    elif shape == "one":
        t = torch.full((n,), vocab - 1, dtype=torch.int64, device="cuda")
    elif shape == "few":
        t = torch.randint(0, min(vocab, 3), (n,), generator=gen, device="cuda") * (vocab // 3)
        t.clamp_(max=vocab - 1)
    else:  # often small, some outside
        t = (torch.exp(torch.rand(n, generator=gen, device="cuda", dtype=torch.float64) * math.log(vocab + 1)) - 1).long()
        t[::9] = -1
        t[4::11] = vocab + 3
    return t


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 700, 1023, 1025, 4096, 8191, 8192])
@pytest.mark.parametrize("shape", ["all", "one", "few", "padded"])
def test_embedding_tokens(n, shape):
    print(f"{n} tokens, {shape}", flush=True)
    gen = generator(n)
    check_embedding(some_tokens(n, 1000, n, shape), normal(gen, 1000, 40), normal(gen, n, 40), scale=1.5)


@pytest.mark.parametrize("n", [8193, 12288, 12289, 70001])
@pytest.mark.parametrize("shape", ["all", "one", "few", "padded"])
def test_embedding_many_tokens(n, shape):
    print(f"{n} tokens, {shape}", flush=True)
    gen = generator(n)
    check_embedding(some_tokens(n, 5003, n, shape), normal(gen, 5003, 24).bfloat16(), normal(gen, n, 24).bfloat16())


def test_embedding_of_more_tokens_than_tiles_of_a_part():
    """256 parts of two tiles each"""
    n = 256 * 4096 + 77
    gen = generator(3)
    check_embedding(some_tokens(n, 3001, 1, "padded"), normal(gen, 3001, 8), normal(gen, n, 8))


@pytest.mark.parametrize("vocab", [1, 2, 3, 1023, 1024, 65536, 262143, 262144])
def test_embedding_vocabularies(vocab):
    gen = generator(vocab)
    for n in (300, 9000):
        check_embedding(some_tokens(n, vocab, vocab, "padded"), normal(gen, vocab, 8), normal(gen, n, 8))


@pytest.mark.parametrize("d", [1, 3, 8, 16, 17, 64, 130, 768, 1024, 1025, 2056, 4100])
@pytest.mark.parametrize("kind", TYPES)
def test_embedding_channels(d, kind):
    print(f"{d} channels, {kind}", flush=True)
    gen = generator(d)
    tokens = some_tokens(200, 50, d, "padded")
    check_embedding(tokens, normal(gen, 50, d).to(TYPES[kind]), normal(gen, 200, d).to(TYPES[kind]), scale=0.5)
    check_embedding(tokens, normal(gen, 50, d), normal(gen, 200, d).to(TYPES[kind]), kind=TYPES[kind])


def test_embedding_types_on_either_side():
    c, gen = ops(), generator(4)
    tokens = some_tokens(100, 60, 2, "padded")
    there, at = ((tokens >= 0) & (tokens < 60))[:, None], tokens.clamp(0, 59)
    for table in TYPES.values():
        for rows in TYPES.values():
            for d in (7, 64):
                t, out = normal(gen, 60, d).to(table), torch.empty((100, d), device="cuda").to(rows)
                c.embedding(tokens, t, out, scale=3.0)
                assert torch.equal(out, torch.where(there, t[at].float() * 3, 0.0).to(rows))


@pytest.mark.parametrize("d", [33, 64])
def test_embedding_strides(d):
    """a table inside a wider one, rows inside wider ones, a gradient that begins anywhere, with what lies around it kept"""
    c, gen = ops(), generator(d)
    tokens = some_tokens(500, 40, d, "all")
    table = normal(gen, 40, d + 9)[:, 5:5 + d]
    rows = normal(gen, 500, 2 * d + 1).bfloat16()[:, 1 + d:1 + 2 * d]
    gaps = torch.full((500, d + 3), 7.0, device="cuda").bfloat16()
    c.embedding(tokens, table, gaps[:, 2:2 + d])
    assert torch.equal(gaps[:, 2:2 + d], table[tokens].bfloat16()) and (gaps[:, :2] == 7).all() and (gaps[:, -1] == 7).all()
    want = check_embedding(tokens, table.contiguous(), rows.contiguous())
    for shift in (1, 2, 3):
        flat = torch.full((40 * d + 8,), 7.0, device="cuda")
        got = run_gradient(tokens, rows, flat[shift:shift + 40 * d].view(40, d))
        assert torch.equal(got, want) and (flat[:shift] == 7).all() and (flat[shift + 40 * d:] == 7).all()
    short = torch.full((40 * d + 16,), 7.0, device="cuda").bfloat16()
    got = run_gradient(tokens, rows, short[3:3 + 40 * d].view(40, d))
    assert torch.equal(got, run_gradient(tokens, rows, torch.empty((40, d), device="cuda").bfloat16()))
    assert (short[:3] == 7).all() and (short[3 + 40 * d:] == 7).all()


def test_embedding_of_no_tokens():
    none = torch.zeros(0, dtype=torch.int64, device="cuda")
    grad = torch.full((50, 33), 7.0, device="cuda")
    rows = torch.zeros((0, 33), device="cuda")
    ops().embedding(none, grad, rows)
    assert (run_gradient(none, rows, grad.clone(), accumulate=True) == 7).all()
    assert (run_gradient(none, rows, grad) == 0).all()


def test_embedding_rows_that_are_not_finite_stay_in_their_token():
    gen = generator(2)
    tokens, rows = some_tokens(3000, 200, 2, "all"), normal(gen, 3000, 16)
    want = run_gradient(tokens, rows, torch.empty((200, 16), device="cuda"))
    rows[77, 3] = math.nan
    got = run_gradient(tokens, rows, torch.empty((200, 16), device="cuda"))
    hit = torch.zeros_like(want, dtype=torch.bool)
    hit[tokens[77], 3] = True
    assert torch.isnan(got[hit]).all() and torch.equal(got[~hit], want[~hit])


def test_embedding_offsets_past_32_bits():
    """a table and its gradient past 2^32 bytes"""
    vocab, d = 1 << 18, 4224
    table = torch.zeros((vocab, d), device="cuda")
    tokens = torch.tensor([vocab - 1, 0, vocab - 1, 260000, vocab], device="cuda")
    rows = normal(generator(1), 5, d)
    run_gradient(tokens, rows, table)
    assert torch.equal(table[-1], rows[0] + rows[2]) and torch.equal(table[260000], rows[3]) and torch.equal(table[0], rows[1])
    assert (table[1:260000].abs().amax() == 0).item() and (table[260001:-1].abs().amax() == 0).item()
    out = torch.empty((5, d), device="cuda")
    ops().embedding(tokens, table, out)
    assert torch.equal(out[0], table[-1]) and (out[4] == 0).all()


# ------------------------------------------------------------------------------------------------ log-probabilities
def score_case(rows, vocab, kind, seed):
    gen = generator(seed)
    logits = 2 * normal(gen, rows, vocab)
    logits[:, ::7] += 6
    if vocab > 5:
        logits[:, 3::97] = -math.inf
    tokens = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
    tokens[2::5] = -1
    tokens[4::7] = vocab
    return logits.to(kind), tokens, normal(gen, rows), normal(gen, rows)


def score(logits, tokens, k=0, weights=None, entropy_weights=None, at_once=False, gradient=None):
    c = ops()
    rows, vocab = logits.shape
    lp, entropy, stats = (torch.full(s, 7.0, device="cuda") for s in ((rows,), (rows,), (rows, 2)))
    top, top_lp = (torch.full((rows, k), 7, dtype=torch.int64, device="cuda"), torch.full((rows, k), 7.0, device="cuda")) if k else (None, None)
    gradient = torch.full((rows, vocab), 7.0, device="cuda").to(logits.dtype) if gradient is None else gradient
    known = dict(weights=weights, entropy_weights=entropy_weights, gradient=gradient) if at_once else {}
    c.token_logprobs(logits, tokens, lp if tokens is not None else None, entropy, stats, top, top_lp,
                     workspace=workspace(c.token_logprobs_workspace(logits, k)), **known)
    if not at_once and (weights is not None or entropy_weights is not None):
        c.token_logprobs_gradient(logits, tokens, stats, weights, gradient, entropy_weights, entropy)
    torch.cuda.synchronize()
    return lp, entropy, stats, top, top_lp, gradient


def check_score(logits, tokens, weights, entropy_weights, k=0):
    """A thread adds up to vocab / 256 exponentials, and the threads' sums meet in 20 steps more: S is off by (vocab / 256 + 64)
    2^-24 of itself, each exponential by its exponent's rounding.  The entropy's sum goes by differences from a reference up to 6
    below the largest.  Alternatives are places: they have to be equal."""
    rows, vocab = logits.shape
    x = logits.double()
    m = x.amax(1, keepdim=True)
    logs = torch.log(torch.exp(x - m).sum(1, keepdim=True))
    log_p = (x - m) - logs
    p = log_p.exp()
    plp = torch.where(p > 0, p * log_p, 0.0)
    H = -plp.sum(1)
    there = (tokens >= 0) & (tokens < vocab)
    at = tokens.clamp(0, vocab - 1)[:, None]
    want = torch.where(there, log_p.gather(1, at)[:, 0], 0.0)
    n = vocab / 256 + 64
    lp, entropy, stats, top, top_lp, gradient = score(logits, tokens, k, weights, entropy_weights)
    finite = torch.isfinite(want)
    assert torch.equal(lp[~finite].double(), want[~finite])
    assert_within(lp[finite], want[finite], U * (3 * want.abs() + 3 * logs[:, 0] + n)[finite])
    assert_within(entropy, H, U * (n * (14 + 2 * H + 2 * logs[:, 0])))
    assert torch.equal(stats[:, 0].double(), m[:, 0])
    assert_within(stats[:, 1], logs[:, 0], U * (n + 3 * logs[:, 0]))
    if k:
        order = torch.sort(-x, dim=1, stable=True).indices[:, :k]
        have = torch.isfinite(x.gather(1, order))
        order, like = torch.where(have, order, -1), log_p.gather(1, order)
        assert torch.equal(top[:, :order.shape[1]], order) and (top[:, order.shape[1]:] == -1).all()
        assert torch.equal(torch.isfinite(top_lp[:, :order.shape[1]]), have)
        assert ((top_lp[:, :order.shape[1]].double() - like).abs()[have] <= (U * (3 * like.abs() + 3 * logs + n))[have]).all()
    one = torch.zeros_like(x)
    one[torch.arange(rows), at[:, 0]] = there.double()
    w, u = torch.where(there, weights, 0.0).double()[:, None], entropy_weights.double()[:, None]
    grad = w * (one - p) - u * (plp + p * H[:, None])
    safe = torch.where(p > 0, log_p, 0.0).abs()
    size = w.abs() * (one + p) + u.abs() * p * (safe + H[:, None])
    # p is off by the error of its exponent; the entropy beside log p by its own
    off = U * (n + 4 * safe + 4 * logs) * size + u.abs() * p * (U * n * (14 + 2 * H + 2 * logs[:, 0]))[:, None]
    assert_within(gradient, grad, off)
    at_once = score(logits, tokens, k, weights, entropy_weights, at_once=True)
    assert_within(at_once[5], grad, off)
    assert torch.equal(at_once[0], lp) and torch.equal(at_once[1], entropy)
    place = logits.clone()  # the gradient in the logits' place; a clone's rows may begin elsewhere, and sums go by vectors
    apart = score(place, tokens, k, weights, entropy_weights, at_once=True)[5]
    assert torch.equal(score(place, tokens, k, weights, entropy_weights, at_once=True, gradient=place)[5], apart)
    return lp, entropy, top


@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 31, 255, 257, 1000, 4096, 4097, 8192, 20011, 65536, 262144])
@pytest.mark.parametrize("kind", TYPES)
def test_score_vocabularies(vocab, kind):
    print(f"vocabulary {vocab}, {kind}", flush=True)
    check_score(*score_case(9, vocab, TYPES[kind], vocab), k=20)


@pytest.mark.parametrize("rows", [1, 2, 300, 1000])
@pytest.mark.parametrize("k", [0, 1, 5, 32])
def test_score_rows_and_alternatives(rows, k):
    check_score(*score_case(rows, 5000, torch.bfloat16, rows + k), k=k)


@pytest.mark.parametrize("kind", TYPES)
def test_score_strides(kind):
    """rows at every alignment, the gradient at another"""
    gen = generator(4)
    wide = normal(gen, 11, 3001).to(TYPES[kind])
    logits = wide[:, 7:2907]
    assert logits.stride()[0] % 8 == 1
    tokens = torch.randint(0, 2900, (11,), generator=gen, device="cuda")
    w, u = normal(gen, 11), normal(gen, 11)
    check_score(logits, tokens, w, u, k=9)
    gaps = torch.full((11, 2911), 7.0, device="cuda").to(TYPES[kind])
    for at_once in (False, True):
        want = score(logits, tokens, 0, w, u, at_once=at_once)[5]
        got = score(logits, tokens, 0, w, u, at_once=at_once, gradient=gaps[:, 3:2903])[5]
        assert torch.equal(got, want)  # where it goes does not change it
        assert (gaps[:, :3] == 7).all() and (gaps[:, 2903:] == 7).all()


@pytest.mark.parametrize("vocab", [50, 3000, 70000])
def test_score_equal_logits_go_by_their_index(vocab):
    for kind in TYPES.values():
        x = torch.zeros((3, vocab), device="cuda").to(kind)
        x[1, vocab // 2:] = 1.0
        x[2, ::3] = -math.inf
        tokens = torch.tensor([0, vocab - 1, 1], device="cuda")
        _, entropy, top = check_score(x, tokens, torch.ones(3, device="cuda"), torch.ones(3, device="cuda"), k=min(32, vocab // 2))
        assert top[0].tolist() == list(range(len(top[0]))) and top[1, 0].item() == vocab // 2


@pytest.mark.parametrize("rows", [2, 300])
@pytest.mark.parametrize("kind", TYPES)
def test_score_large_logits_that_lie_together(rows, kind):
    """rising and falling rows, and thousands of large logits in the strips of a few threads: more than the list holds"""
    vocab = 60000
    x = torch.zeros((rows, vocab), device="cuda")
    x[0] = torch.arange(vocab, device="cuda") / 4096
    x[1] = -torch.arange(vocab, device="cuda") / 4096
    if rows > 2:
        v = 16 // torch.empty(0, dtype=TYPES[kind]).element_size()
        index = torch.arange(vocab, device="cuda")
        for r, threads in ((2, 256), (3, 1024)):
            x[r] = torch.where(index // v % threads < 40, 5 + torch.rand(vocab, generator=generator(r), device="cuda"), 0.0)
    x = x.to(TYPES[kind])
    tokens = torch.arange(rows, device="cuda")
    check_score(x, tokens, torch.ones(rows, device="cuda"), torch.zeros(rows, device="cuda"), k=32)


@pytest.mark.parametrize("kind", TYPES)
def test_score_rows_of_nothing_and_of_lowest_values(kind):
    c, kind = ops(), TYPES[kind]
    lowest = torch.finfo(kind).min
    x = torch.full((6, 5000), -math.inf, device="cuda").to(kind)
    x[1] = lowest           # all alike
    x[2, 4321] = lowest     # the only one
    x[3], x[3, 77] = lowest, 2.0
    x[4, 10:13] = 1.0
    tokens = torch.tensor([5, 5, 4321, 77, 11, -1], device="cuda")
    ones = torch.ones(6, device="cuda")
    for at_once in (False, True):
        lp, entropy, stats, top, top_lp, grad = score(x, tokens, 4, ones, ones, at_once=at_once)
        third = math.log(3)
        want = torch.tensor([-math.inf, -math.log(5000), 0.0, 0.0, -third, 0.0], device="cuda")
        assert torch.allclose(lp, want, rtol=1e-5, atol=0) and lp[0].item() == -math.inf
        assert torch.allclose(entropy, torch.tensor([0.0, math.log(5000), 0.0, 0.0, third, 0.0], device="cuda"), rtol=1e-5, atol=1e-6)
        assert top[0].tolist() == [-1] * 4 and top[2].tolist() == [4321, -1, -1, -1] and top[4].tolist() == [10, 11, 12, -1]
        assert (top_lp[0] == -math.inf).all() and top_lp[2, 0].item() == 0
        assert (grad[0] == 0).all() and (grad[5] == 0).all() and (grad[2].abs() <= 1e-6).all() and torch.isfinite(grad).all()
        assert (grad[1].double().sum().abs() <= 5000 * 2.0**-8 / 5000 + 1e-3).item()


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("rows", [5, 400])
def test_score_of_a_row_that_is_not_finite(rows, value):
    logits, tokens, w, u = score_case(rows, 6000, torch.float32, 1)
    want = score(logits, tokens, 3, w, u)
    logits[1, 4444] = value
    tokens[1] = 17
    got = score(logits, tokens, 3, w, u)
    keep = torch.arange(rows, device="cuda") != 1
    assert all(torch.equal(g[keep], t[keep]) for g, t in zip(got, want))
    assert torch.isnan(got[0][1]) and torch.isnan(got[1][1]) and torch.isnan(got[5][1]).all()
    assert (got[3][1][0].item() == 4444) == (value == math.inf)
    w[1] = u[1] = 0
    assert (score(logits, tokens, 3, w, u)[5][1] == 0).all()  # a masked position
    assert (score(logits, tokens, 3, w, u, at_once=True)[5][1] == 0).all()


@pytest.mark.parametrize("rows", [3, 600])
def test_score_of_nan_beside_logits_out_of_all_proportion(rows):
    """a NaN stays one whatever follows it: logits of 2^120, later and larger ones, rows of nothing but them"""
    x = torch.zeros((rows, 9000), device="cuda")
    x[:, 5], x[:, 4000:4004], x[:, 8000] = math.nan, 2.0**120, 2.0**121
    x[1, 5] = 0.0
    lp, entropy, _, top, _, grad = score(x, torch.full((rows,), 8000, device="cuda"), 2, torch.ones(rows, device="cuda"))
    keep = torch.arange(rows, device="cuda") != 1
    assert torch.isnan(lp[keep]).all() and torch.isnan(entropy[keep]).all() and torch.isnan(grad[keep]).all()
    assert lp[1].item() == 0 and entropy[1].item() == 0 and (grad[1] == 0).all()
    assert (top == torch.tensor([8000, 4000], device="cuda")).all()


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [20, 600])
def test_score_alternatives_are_scored_like_given_tokens(rows, kind):
    """bit for bit, whichever threads find them"""
    logits = (3 * normal(generator(rows), rows, 40000)).to(kind)
    _, _, _, top, top_logprobs, _ = score(logits, torch.zeros(rows, dtype=torch.int64, device="cuda"), 7)
    for j in range(7):
        logprobs, *_ = score(logits, top[:, j].contiguous(), 7)
        assert torch.equal(logprobs, top_logprobs[:, j])


@pytest.mark.parametrize("vocab, rows", [(1024, 30), (1025, 30), (2048, 30), (2049, 30), (2048, 1100), (4096, 1100), (4097, 1025), (97, 1100)])
@pytest.mark.parametrize("kind", [torch.float32, torch.float16])
@pytest.mark.parametrize("k", [0, 16, 17])
def test_score_short_rows(vocab, rows, kind, k):
    """around what a wave takes by itself"""
    check_score(*score_case(rows, vocab, kind, vocab), k)


@pytest.mark.parametrize("vocab", [300, 2000])
def test_score_short_rows_of_logits_that_lie_together(vocab):
    """more entries at the bound than the list holds, and equal ones"""
    logits = torch.full((1200, vocab), 2.0, dtype=torch.bfloat16, device="cuda")
    logits[::3, 5::2] = 2.015625
    logits[1::3, -1] = 3
    tokens = torch.arange(1200, device="cuda") % vocab
    top = score(logits, tokens, 4)[3]
    want = torch.sort(logits.double(), dim=-1, descending=True, stable=True).indices[:, :4]
    assert torch.equal(top, want)


def test_score_without_tokens():
    logits, _, _, u = score_case(7, 900, torch.float32, 1)
    got, want = score(logits, None, 4), score(logits, torch.zeros(7, dtype=torch.int64, device="cuda"), 4)
    assert torch.equal(got[1], want[1]) and torch.equal(got[3], want[3])
    assert torch.equal(score(logits, None, 0, None, u)[5], score(logits, torch.zeros(7, dtype=torch.int64, device="cuda"), 0, 0 * u, u)[5])


def test_score_gradient_against_differences():
    logits, tokens, w, u = score_case(3, 40, torch.float32, 2)
    tokens = tokens.clamp(0, 39)
    logits = logits.clamp(min=-3.0)
    grad = score(logits, tokens, 0, w, u)[5]

    def value(x):
        log_p = torch.log_softmax(x, 1)
        return ((w.double() * log_p.gather(1, tokens[:, None])[:, 0]).sum() - (u.double() * (log_p.exp() * log_p).sum(1)).sum()).item()

    step = 2.0**-12
    for at in ((0, 0), (1, 7), (2, 39), (0, tokens[0].item())):
        ends = []
        for sign in (1, -1):
            x = logits.double().clone()
            x[at] += sign * step
            ends.append(value(x))
        assert abs(grad[at].item() - (ends[0] - ends[1]) / (2 * step)) <= 10 * step**2 + 1e-4


# ------------------------------------------------------------------------------------------------ AdamW
BETAS, EPS = (0.9, 0.99), 1e-8


def adamw_case(sizes, kind, seed):
    gen = generator(seed)
    params = [0.1 * normal(gen, n) for n in sizes]
    grads = [(0.01 * normal(gen, n)).to(kind) for n in sizes]
    m = [0.003 * normal(gen, n) for n in sizes]
    v = [(0.01 * normal(gen, n)).square() for n in sizes]
    return params, grads, m, v


def adamw_64(p, g, m, v, lr, decay, step, scale=1.0):
    p, g, m, v = (t.double() for t in (p, g, m, v))
    g = g * scale
    m, v = BETAS[0] * m + (1 - BETAS[0]) * g, BETAS[1] * v + (1 - BETAS[1]) * g * g
    move = m / (1 - BETAS[0]**step) / ((v / (1 - BETAS[1]**step)).sqrt() + EPS)
    return p - lr * (decay * p + move), m, v, lr * (decay * p.abs() + move.abs())


SIZES = [1, 3, 4, 255, 256, 257, 1000, 1024, 4095, 4096, 4097, 10000]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("step", [1, 57, 100000])
def test_adamw_in_32_bits(kind, step):
    """A moment is two products and a sum, 3 2^-24 of their magnitudes (and of b and 1 - b, which are rounded to float32: 2 more);
    the update adds the root, the reciprocal and the corrections of both betas: 40 2^-24 of itself and of where the moments'
    roundings leave it."""
    c = ops()
    params, grads, m, v = adamw_case(SIZES, TYPES[kind], step)
    decay = [0.0 if i % 2 else 0.1 for i in range(len(SIZES))]
    want = [adamw_64(p, g, a, b, 1e-3, d, step) for p, g, a, b, d in zip(params, grads, m, v, decay)]
    mags = [(BETAS[0] * a.abs() + (1 - BETAS[0]) * g.abs()).double() for a, g in zip(m, grads)]
    copies = [torch.empty_like(p, dtype=torch.bfloat16) for p in params]
    opt = c.AdamW(params, betas=BETAS, eps=EPS, weight_decay=decay, copies=copies, states=(m, v))
    opt.step(grads, lr=1e-3, step=step)
    first, second = 1 - BETAS[0]**step, math.sqrt(1 - BETAS[1]**step)
    for i in range(len(SIZES)):
        wp, wm, wv, size = want[i]
        lost = 5 * U * mags[i] / first / (wv.sqrt() / second + EPS) * 1e-3  # what m's rounding moves
        assert_within(m[i], wm, 5 * U * mags[i])
        assert_within(v[i], wv, 6 * U * wv)
        assert_within(params[i], wp, 40 * U * size + lost + U * wp.abs())
        assert torch.equal(copies[i], params[i].bfloat16())


def test_adamw_of_more_tensors_than_a_launch_takes_and_of_empty_ones():
    c = ops()
    sizes = [(37 * i) % 301 for i in range(130)]
    params, grads, m, v = adamw_case(sizes, torch.float32, 4)
    want = [adamw_64(p, g, a, b, 1e-2, 0.01, 3) for p, g, a, b in zip(params, grads, m, v)]
    c.AdamW(params, betas=BETAS, eps=EPS, states=(m, v)).step(grads, lr=1e-2, step=3)
    for p, a, w in zip(params, m, want):
        assert ((p.double() - w[0]).abs() <= 1e-5 * w[3] + 2 * U * w[0].abs()).all()
        assert ((a.double() - w[1]).abs() <= 1e-5 * 0.01).all()


def test_adamw_of_a_large_tensor():
    """chunks longer than the least"""
    n = 80_000_001
    p = torch.zeros(n, device="cuda")
    g = torch.arange(n, device="cuda").remainder_(251).sub_(125).bfloat16()
    opt = ops().AdamW([p], betas=BETAS, eps=EPS, weight_decay=0.0)
    opt.step([g], lr=1.0, step=1)
    assert ((p + g.float().sign()).abs() <= 1e-5).all()  # m / sqrt(v) of one gradient is its sign


def test_adamw_at_other_addresses():
    """tensors at odd places of one buffer, with what lies between kept"""
    c, gen = ops(), generator(1)
    for bits in (32, 8):
        flat = torch.full((5000,), 7.0, device="cuda")
        g = normal(gen, 4990).bfloat16()
        params = [torch.full((n,), 0.5, device="cuda") for n in (1500, 900)]
        a = c.AdamW(params, bits=bits)
        views = [flat[3:1503], flat[1601:2501]]
        for x in views:
            x.fill_(0.5)
        copies = torch.full((5000,), 7.0, device="cuda").half()
        grads = [g[1:1501], g[1777:2677]]
        b = c.AdamW(views, bits=bits, copies=[copies[5:1505], copies[1603:2503]])
        for step in (1, 2):
            a.step([x.clone() for x in grads], lr=0.01, step=step, seed=5)
            b.step(grads, lr=0.01, step=step, seed=5)
        for x, y, s, t in zip(params, views, a.states[0], b.states[0]):
            assert torch.equal(x, y) and torch.equal(s.float(), t.float())
        assert (flat[:3] == 7).all() and (flat[1503:1601] == 7).all() and (flat[2501:] == 7).all()
        assert torch.equal(copies[5:1505], views[0].half()) and (copies[1505:1603] == 7).all()


def test_adamw_reads_its_numbers_on_the_device():
    c = ops()
    a, b = (adamw_case([5000], torch.float32, 2) for _ in range(2))
    lr, step, scale = torch.tensor([0.01], device="cuda"), torch.tensor([7], dtype=torch.int32, device="cuda"), torch.tensor([0.25], device="cuda")
    c.AdamW(a[0], betas=BETAS, states=a[2:]).step(a[1], lr=0.01, step=7, scale=scale)
    c.AdamW(b[0], betas=BETAS, states=b[2:]).step([0.25 * b[1][0]], lr=lr, step=step)
    assert torch.equal(a[0][0], b[0][0]) and torch.equal(a[3][0], b[3][0])


def mixed(x):
    x = ((x ^ (x >> 16)) * 0x9E3779B1) & 0xffffffff
    x = ((x ^ (x >> 15)) * 0xB7E15163) & 0xffffffff
    return x ^ (x >> 16)


def codes_of(x, field, draws, keep):
    """8-bit codes of float32 values (numpy, whole blocks) by the definition, in whole numbers"""
    out = np.zeros(x.shape, np.uint8)
    power = np.maximum(field, 16)
    for i, (value, draw) in enumerate(zip(x, draws)):
        bits = int(np.float32(abs(value)).view(np.uint32))
        e = (bits >> 23) - int(power[i // 256]) + 7  # of the value under the power
        mantissa, cut = (bits & 0x7fffff) | 0x800000, 20 + max(0, -6 - e)
        code = 0
        if bits >= 0x800000 and cut < 32:
            whole = (mantissa + (int(draw) << (cut - 16))) >> cut
            code = whole + 8 * max(0, e + 6)
        if keep and bits and not code:
            code = 1
        out[i] = code | (0x80 if value < 0 else 0)
    return out, power.astype(np.uint8)


@pytest.mark.parametrize("n", [1, 255, 256, 257, 5000])
def test_adamw_8_bit_states_are_rounded_as_defined(n):
    """codes and powers equal the definition's; of the root one in 2^20 may be the next code, as its last bit may differ"""
    c = ops()
    gen = generator(n)
    spread = torch.exp2(-30 * torch.rand(n, generator=gen, device="cuda"))
    g = normal(gen, n) * spread
    g[::50] = 0
    p, opt = torch.zeros(n, device="cuda"), None
    opt = c.AdamW([torch.zeros(3, device="cuda"), p], betas=BETAS, bits=8)
    opt.step([torch.zeros(3, device="cuda"), g], lr=0.1, step=9, seed=77)
    f = np.float32
    pad = -n % 256
    gn = np.pad(g.cpu().numpy(), (0, pad))
    m, v = gn * f(1 - BETAS[0]), (gn * gn) * f(1 - BETAS[1])
    key = mixed((77 + 0xB7E15163 * 9 + 0x9E3779B1 * 1) & 0xffffffff)
    draws = np.array([mixed((key + i) & 0xffffffff) for i in range(n + pad)], np.uint64)

    def field(x):
        return np.abs(x).reshape(-1, 256).max(1).astype(f).view(np.uint32).astype(np.int64) >> 23

    want_m, power_m = codes_of(m, field(m), draws & 0xffff, False)
    want_r, power_r = codes_of(np.sqrt(v), (field(v) + 127) >> 1, draws >> 16, True)
    got_m, got_r = (s[1].view(torch.uint8).cpu().numpy() for s in opt.states[:2])
    powers = opt.states[2][1].cpu().numpy()
    assert (powers == np.stack((power_m, power_r), 1)).all()
    assert ((got_m == want_m[:n]) | ((got_m & 127 == 0) & (want_m[:n] & 127 == 0))).all()
    assert (got_r != want_r[:n]).sum() <= 1 and (np.abs(got_r.astype(int) - want_r[:n]) <= 1).all()
    assert (got_r[(gn[:n] != 0) & (v[:n] > 0)] > 0).all()


def test_adamw_8_bit_states_are_right_on_average():
    """one gradient under many seeds: the mean of the rounded moments is the moment.  A rounding is off by less than a step, 1/8
    of the value (a step of the smallest in the range below), its mean over 4,000 by 5 / sqrt(4000) of half of that, 8 %"""
    c = ops()
    n, tries = 256, 4000
    g = normal(generator(3), n) * torch.exp2(-9 * torch.rand(n, generator=generator(4), device="cuda"))
    sums = torch.zeros((2, n), dtype=torch.float64, device="cuda")
    for seed in range(tries):
        opt = c.AdamW([torch.zeros(n, device="cuda")], betas=BETAS, bits=8)
        opt.step([g], lr=0.0, step=1, seed=seed)
        for i in range(2):
            sums[i] += opt.states[i][0].double() * 2.0**(opt.states[2][0][0, i].double() - 134)
    step = torch.tensor([2.0**-9, 2.0**-9], device="cuda").double() * 2.0**(opt.states[2][0][0].double() - 134)
    for i, want in ((0, (1 - BETAS[0]) * g.double()), (1, (math.sqrt(1 - BETAS[1]) * g.double()).abs())):
        assert ((sums[i] / tries - want).abs() <= 0.08 * (want.abs() / 8 + step[i])).all()


def test_adamw_8_bit_updates_use_the_moments_before_they_are_rounded():
    """the first step moves every entry by lr sign(g), as in 32 bits; the next ones by what the rounded states say"""
    c = ops()
    gen = generator(5)
    grads = [normal(gen, 3000) * 10 for _ in range(6)]
    a, b = torch.zeros(3000, device="cuda"), torch.zeros(3000, device="cuda")
    eight, full = c.AdamW([a], betas=BETAS, weight_decay=0.0, bits=8), c.AdamW([b], betas=BETAS, weight_decay=0.0)
    for i, g in enumerate(grads):
        eight.step([g], lr=0.01, step=i + 1, seed=1)
        full.step([g], lr=0.01, step=i + 1)
        if i == 0:
            assert (a - b).abs().max().item() <= 1e-7
    # moments rounded by up to 1/8 of themselves (a sum of five such m's by less than 5/8 of the largest), the root by 1/8: an
    # update, below 1/0.1 lr, is off by less than itself
    assert (a - b).abs().max().item() <= 6 * 0.01 * 2
    again = c.AdamW([torch.zeros(3000, device="cuda")], betas=BETAS, weight_decay=0.0, bits=8)
    for i, g in enumerate(grads):
        again.step([g], lr=0.01, step=i + 1, seed=1)
    assert torch.equal(again.params[0], a) and torch.equal(again.states[2][0], eight.states[2][0])


def test_adamw_gradients_that_are_not_finite():
    """in 32 bits the entry is lost, in 8 its block of 256; others are not"""
    c = ops()
    for bits in (32, 8):
        grads = [normal(generator(1), 2000) for _ in range(2)]
        clean, p = torch.zeros(2000, device="cuda"), torch.zeros(2000, device="cuda")
        a, b = c.AdamW([clean], bits=bits), c.AdamW([p], bits=bits)
        a.step(grads[:1], lr=0.01, step=1)
        bad = grads[0].clone()
        bad[700] = math.nan
        bad[1500] = math.inf
        b.step([bad], lr=0.01, step=1)
        for opt in (a, b):
            opt.step(grads[1:], lr=0.01, step=2)
        hit = torch.zeros(2000, dtype=torch.bool, device="cuda")
        if bits == 32:
            hit[[700, 1500]] = True
        else:
            hit[512:768] = hit[1280:1536] = True
        assert torch.equal(p[~hit], clean[~hit]) and torch.isnan(p[hit]).all()
