"""GPU tests of every form that the kernels of the operators in the clear are built in, at the smallest sizes whose rules of
dispatch reach it: tiles of 64 and 32 state columns, alone and in segments, for each head size and type; 4-bit products whose
rows share a read of the weights, for each type, group and kind of scales, over one chunk of rows in LDS and over several; draws
for more rows than compute units.

Largest errors are bounded as in test_gpu_clear_ops.py.  Root mean squares are bounded by what sums of n terms of random signs,
each cut off at 2^-23 of the sum, leave: sqrt(n) 2^-23 of the result's own."""
import math

import numpy as np
import pytest

from engine_loader import load_module
from test_gpu_clear_ops import (ROUNDING, TYPES, attention_case, check_product, check_prompt, kept_weights, product_case,
                                recurrence, run_prompt, run_sample, spread)

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

# lanes, heads, tokens, and what they reach.  64 columns: more than 192 tiles of 64, or more than 384 chunks of them; segments:
# fewer than 256 workgroups and four chunks.  float32 always takes 32 columns.
SHAPES = {"64 columns": (100, 4, 70), "64 columns in two segments": (50, 4, 260), "64 columns in many segments": (1, 12, 2177),
          "32 columns": (2, 3, 100), "32 columns in segments": (1, 2, 600)}


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dk", [20, 32, 64, 100, 128])
@pytest.mark.parametrize("kind", TYPES)
def test_prompt_forms(shape, dk, kind):
    lanes, heads, tokens = SHAPES[shape]
    print(shape, dk, kind, flush=True)
    check_prompt(*attention_case(lanes, tokens, heads, heads, 1, dk, 64, TYPES[kind], dk), scale=dk**-0.5)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("kind", TYPES)
def test_prompt_forms_with_columns_left_over(shape, kind):
    lanes, heads, tokens = SHAPES[shape]
    for dv in (33, 80):
        check_prompt(*attention_case(lanes, tokens, heads, 1, heads, 64, dv, TYPES[kind], dv), scale=0.125)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dk", [64, 128])
@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_prompt_forms_of_ragged_lengths(shape, dk, kind):
    """NaN behind every lane's length, lengths that end in the first, a middle and the last chunk, and none"""
    lanes, heads, tokens = SHAPES[shape]
    q, k, v, g, state = attention_case(lanes, tokens, heads, heads, heads, dk, 64, TYPES[kind], 9)
    lengths = (torch.arange(lanes, device="cuda") * 37 % (tokens + 1)).int() if lanes > 1 else torch.tensor(
        [tokens // 2 + 5], dtype=torch.int32, device="cuda")
    want, left = check_prompt(q, k, v, g, state, lengths, scale=dk**-0.5)
    behind = torch.arange(tokens, device="cuda")[None] >= lengths[:, None]
    for x in (q, k, v, g):
        x[behind] = math.nan
    out, into = run_prompt(q, k, v, g, state, lengths, dk**-0.5)
    assert torch.equal(out, want) and torch.equal(into, left)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dk", [32, 64, 128])
@pytest.mark.parametrize("kind", TYPES)
def test_prompt_forms_keep_what_is_not_finite_in_its_future(shape, dk, kind):
    lanes, heads, tokens = SHAPES[shape]
    q, k, v, g, state = attention_case(lanes, tokens, heads, heads, heads, dk, 64, TYPES[kind], tokens)
    want, left = run_prompt(q, k, v, g, state)
    hit, hit_state = torch.zeros_like(want, dtype=torch.bool), torch.zeros_like(left, dtype=torch.bool)
    for b, t, h, c, x in ((0, tokens // 2, 1, 7, math.inf), (lanes - 1, tokens - 1, 0, 3, math.nan), (0, tokens // 3, 0, 63, -math.inf)):
        v[b, t, h, c] = x
        hit[b, t:, h, c], hit_state[b, h, :, c] = True, True
    out, into = run_prompt(q, k, v, g, state)
    assert not torch.isfinite(out[hit]).any() and not torch.isfinite(into[hit_state]).any()
    # elsewhere the same sums in another order
    full = torch.full((lanes,), tokens, device="cuda")
    size, size_left = recurrence(q.abs(), k.abs(), v.nan_to_num(0, 0, 0).abs(), g, state.abs(), full, 1.0)
    allowed = (2 * (4 * tokens + dk + 64) * 2.0**-24) * size + 2 * ROUNDING[out.dtype] * want.double().abs()
    assert ((out.double() - want.double()).abs() <= allowed)[~hit].all()
    assert ((into.double() - left.double()).abs() <= 2 * (4 * tokens + dk + 64) * 2.0**-24 * size_left)[~hit_state].all()


def rms(x):
    return x.square().mean().sqrt().item()


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dk", [32, 64, 128])
@pytest.mark.parametrize("kind", TYPES)
def test_prompt_forms_round_as_float32_does(shape, dk, kind):
    """Sums over dk channels make scores and read the state, sums over 64 tokens of a chunk read the scores, sums over all
    tokens make the state.  A third piece left out of any operand, or a state joined in 16 bits, is 2^-16 to 2^-9 instead."""
    lanes, heads, tokens = SHAPES[shape]
    q, k, v, g, state = attention_case(lanes, tokens, heads, heads, heads, dk, 64, TYPES[kind], dk + 1, decay=0.03)
    out, into = run_prompt(q, k, v, g, state)
    want, left = recurrence(q, k, v, g, state, torch.full((lanes,), tokens, device="cuda"), 1.0)
    carried = 2 * math.sqrt(tokens) + 4  # and the decays' exponentials
    assert rms(into.double() - left) <= carried * 2.0**-23 * rms(left)
    own = 0.0 if kind == "f32" else ROUNDING[TYPES[kind]] * rms(want)
    assert rms(out.double() - want) <= (2 * math.sqrt(dk) + 8 + carried) * 2.0**-23 * rms(want) + own


@pytest.mark.parametrize("T", [5, 64, 300])
def test_float32_prompts_keep_the_third_piece(T):
    """a and -a cut to 16 bits: their sum is the third of a's three pieces of 8 bits, below 2^-15.  As two keys' channels, as two
    rows of the state, as two tokens' values.  Every product is one with 1 or -1; the sum of the first pieces, two of below 2, is
    off by at most 2^-23 of 4."""
    close = dict(rtol=0, atol=2.0**-21)
    B, H = 4, 8
    gen = torch.Generator(device="cuda").manual_seed(T)
    a = 1 + torch.rand((B, H), generator=gen, device="cuda")
    cut = (a.view(torch.int32) & ~255).view(torch.float32)
    low = (a.double() - cut.double())
    assert (low >= 0).all() and (low < 2.0**-15).all() and low.max() > 2.0**-16
    zero, ones = torch.zeros((B, T, H), device="cuda"), torch.ones((B, T, H, 2), device="cuda")
    first, v = torch.zeros((B, T, H, 2), device="cuda"), torch.ones((B, T, H, 16), device="cuda")
    first[:, 0] = torch.stack((a, -cut), -1)
    out, into = run_prompt(ones, first, v, zero, None)  # the key of the first token, read by all
    torch.testing.assert_close(out.double(), low[:, None, :, None].expand(out.shape), **close)
    torch.testing.assert_close(into.double().sum(2), low[..., None].expand(B, H, 16), **close)
    rows = torch.stack((a, -cut), -1)[..., None].expand(B, H, 2, 16).contiguous()
    out, into = run_prompt(ones, 0 * ones, v, zero, rows)
    torch.testing.assert_close(out.double(), low[:, None, :, None].expand(out.shape), **close)
    assert torch.equal(into, rows)
    two = torch.zeros((B, T, H, 16), device="cuda")
    two[:, 0], two[:, 1] = a[..., None], -cut[..., None]
    out, into = run_prompt(ones[..., :1], ones[..., :1], two, zero, None)
    torch.testing.assert_close(out[:, 1:].double(), low[:, None, :, None].expand(B, T - 1, H, 16), **close)
    torch.testing.assert_close(into.double(), low[..., None, None].expand(into.shape), **close)


# ------------------------------------------------------------------------------------------------ 4-bit products
@pytest.mark.parametrize("rows", [20, 40, 70])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("scales", ["f16", "f16 and zeros", "f32 and zeros"])
@pytest.mark.parametrize("kind", TYPES)
def test_product_forms_of_rows_that_share_a_read(rows, group, scales, kind):
    """1,025 tiles of outputs: two or four tiles of rows take one read of the weights"""
    print(rows, group, scales, kind, flush=True)
    check_product(*product_case(rows, 16391, 700, group, TYPES[kind], TYPES[scales[:3]], "zeros" in scales, rows), group)


@pytest.mark.parametrize("rows, out, n_in", [(6, 500, 8192), (20, 16400, 2100), (40, 16400, 2100), (16, 16400, 4096), (64, 100, 9000)])
@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("kind", TYPES)
def test_product_forms_over_several_chunks_of_rows(rows, out, n_in, group, kind):
    """rows longer than LDS holds, with and without columns split over waves"""
    check_product(*product_case(rows, out, n_in, group, TYPES[kind], torch.float16, True, rows), group)


@pytest.mark.parametrize("rows", [1, 5, 6, 17, 40, 70])
@pytest.mark.parametrize("out", [20, 16391])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_float32_products_keep_the_third_piece(rows, out, group):
    """Weights of 1 and pairs a, -a cut to 16 bits: the result is the sum of the third pieces, 16 of 2^-16 on average.  Sums of
    the first pieces are whole multiples of 2^-7 below 2^11 and exact; those of the second, below 2^-7 each, go through 25 and 24
    times their size and are cut off at 2^-23 of it at every term."""
    n = 32
    gen = torch.Generator(device="cuda").manual_seed(rows)
    a = 1 + torch.rand((rows, n // 2), generator=gen, device="cuda")
    cut = (a.view(torch.int32) & ~255).view(torch.float32)
    x = torch.stack((a, -cut), -1).flatten(1).contiguous()
    codes = torch.full((out, n // 2), 0x99, dtype=torch.uint8, device="cuda")
    y = torch.empty((rows, out), device="cuda")
    load_module("clear_ops").Q4Matrix(codes, torch.ones((out, 1), device="cuda"), group=group).product(x, y)
    want = x.double().sum(1, keepdim=True)
    allowed = n * 2.0**-23 * (25 + 24) * n * 2.0**-7
    assert (want > 2 * allowed).all()
    assert ((y.double() - want).abs() <= allowed).all()


# ------------------------------------------------------------------------------------------------ sampling
@pytest.mark.parametrize("kind", TYPES)
def test_sample_form_of_many_rows(kind):
    """More rows than the GPU has compute units: each row's token is the one it gives in a call of its own few, and for the row
    that all of them share, draws in the middle of entries' intervals give those entries.  Filters that go by a short list, a
    long one, a histogram, and none."""
    x = torch.from_numpy(spread(20011, 5, "flat") / 3).cuda().to(TYPES[kind])
    for params in ({}, dict(top_k=40), dict(top_k=700), dict(top_k=9000, top_p=0.9003), dict(top_p=0.2003), dict(min_p=0.3), dict(temperature=0.0)):
        w = kept_weights(x.double().cpu().numpy(), params.get("temperature", 1.0), params.get("top_k", 0),
                         float(np.float32(params.get("top_p", 1.0))), float(np.float32(params.get("min_p", 0.0))))
        at = np.flatnonzero(w > 2.0**-18)
        at = at[np.linspace(0, len(at) - 1, 300).astype(int)]
        draws = np.cumsum(w)[at] - w[at] / 2
        tokens, logprobs = run_sample(x[None].expand(300, len(x)), draws, **params)
        assert np.array_equal(tokens, at) and np.abs(logprobs - np.log(w[at])).max() <= 2.0**-20
        few, logs = run_sample(x[None].expand(60, len(x)), draws[:60], **params)
        assert np.array_equal(few, at[:60]) and np.array_equal(logs, logprobs[:60])
