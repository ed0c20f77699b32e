"""GPU tests of what the operators in the clear keep of their inputs: results that live in the low bits of large operands, as
they do where a sum cancels, operands at the ends of their range, draws near 0 from entries that hardly weigh.  Bounds are
derived at each test, from sums that are cut off rather than rounded at worst (2^-23 of what is summed each)."""
import math

import numpy as np
import pytest

from engine_loader import load_module
from test_gpu_clear_ops import TYPES, ROUNDING, check_product, product_case, run_prompt, run_sample

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ linear attention
@pytest.mark.parametrize("T, dv", [(5, 16), (63, 64), (130, 64), (300, 96)])
@pytest.mark.parametrize("kind", TYPES)
def test_prompt_outputs_read_the_whole_state(T, dv, kind):
    """Two rows of the state near 1000 that differ by up to 1/4, read with q = (1, -1): their difference.  Products with 1 are
    exact; two rows of three pieces at most are six terms, each sum off by at most 2^-23 of 2,000."""
    kind, B, H = TYPES[kind], 3, 4
    gen = torch.Generator(device="cuda").manual_seed(T)
    low = 900 + 100 * torch.rand((B, H, 1, dv), generator=gen, device="cuda")
    state = torch.cat((low, low + torch.rand((B, H, 1, dv), generator=gen, device="cuda") / 4), 2)
    q = torch.tensor([1.0, -1.0], device="cuda").to(kind).expand(B, T, H, 2).contiguous()
    k, v = torch.zeros((B, T, H, 2), device="cuda").to(kind), torch.zeros((B, T, H, dv), device="cuda").to(kind)
    out, into = run_prompt(q, k, v, torch.zeros((B, T, H), device="cuda"), state)
    want = (state[:, :, 0].double() - state[:, :, 1].double())[:, None].expand(B, T, H, dv)
    assert ((out.double() - want).abs() <= 6 * 2.0**-23 * 2000 + ROUNDING[kind] * want.abs()).all()
    assert torch.equal(into, state)


@pytest.mark.parametrize("T", [5, 64, 200])
@pytest.mark.parametrize("kind", TYPES)
def test_prompt_outputs_read_whole_scores(T, kind):
    """Scores 1000 + x_j against values 1 and -1 in turn: after two tokens x_0 - x_1, after four the sum of two differences.  A
    score is one sum of two exact products (its pieces: six terms at most, the largest 1,000), and is read as three pieces."""
    kind, B, H, dv = TYPES[kind], 8, 8, 32
    gen = torch.Generator(device="cuda").manual_seed(T)
    x = torch.rand((B, T, H), generator=gen, device="cuda").to(kind)
    k = torch.stack((torch.full_like(x, 1000.0), x), -1)  # 1000 and the x are numbers of the type
    q = torch.ones((B, T, H, 2), device="cuda").to(kind)
    sign = (1.0 - 2.0 * (torch.arange(T, device="cuda") % 2))[None, :, None]
    v = sign[..., None].expand(B, T, H, dv).contiguous().to(kind)
    out, _ = run_prompt(q, k, v, torch.zeros((B, T, H), device="cuda"), None)
    want = ((1000 + x.double()) * sign.double()).cumsum(1)
    for t in (1, 3):
        allowed = (6 + 3) * (t + 1) * 2.0**-23 * 1001 + ROUNDING[kind] * want[:, t, :, None].abs()
        assert ((out[:, t].double() - want[:, t, :, None]).abs() <= allowed).all(), t


@pytest.mark.parametrize("T", [5, 100])
def test_prompt_takes_float16_inputs_below_the_normal_ones(T):
    """queries of 2^-20 and 3 2^-24 with keys of 2^10, and the other way round: exact products, one a token"""
    small = torch.tensor([2.0**-20, 3 * 2.0**-24], device="cuda").half().reshape(1, 1, 2, 1).expand(1, T, 2, 1).contiguous()
    large = torch.full((1, T, 2, 1), 1024.0, device="cuda").half()
    v = torch.ones((1, T, 2, 16), device="cuda").half()
    g = torch.full((1, T, 2), -math.inf, device="cuda")
    want = (small.float() * large.float()).expand(v.shape)
    for q, k in ((small, large), (large, small)):
        out, into = run_prompt(q, k, v, g, None)
        assert torch.equal(out.float(), want)
        assert torch.equal(into, k[:, -1].float()[..., None].expand(into.shape))


@pytest.mark.parametrize("T", [5, 64, 300])
def test_prompt_keeps_the_products_of_low_pieces(T):
    """x = 1 + 2^-7 - 2^-23, whose three pieces of 8 bits are 1, 2^-7 - 2^-15 and 2^-15 - 2^-23: the products of its second and
    third are 2^-21 of x x.  As a score, as what goes into the state, as what the state gives: a product is a sum of its
    pieces' products, of which those left out are below 2^-30, off by at most 2^-23 of itself, twice for outputs by scores."""
    x = 1 + 2.0**-7 - 2.0**-23
    B, H, zero = 2, 3, torch.zeros((2, T, 3), device="cuda")
    one = torch.zeros((B, T, H, 1), device="cuda")
    one[:, 0] = 1
    q, v = torch.full((B, T, H, 1), x, device="cuda"), torch.ones((B, T, H, 8), device="cuda")
    out, _ = run_prompt(q, one * x, v, zero, None)  # a key at the first token only
    assert ((out.double() - x * x).abs() <= 2.5 * 2.0**-23 * x * x).all()
    _, into = run_prompt(q, one * x, x * v, zero, None)
    assert ((into.double() - x * x).abs() <= 1.5 * 2.0**-23 * x * x).all()
    out, into = run_prompt(q, 0 * one, v, zero, torch.full((B, H, 1, 8), x, device="cuda"))
    assert ((out.double() - x * x).abs() <= 1.5 * 2.0**-23 * x * x).all()
    assert (into == x).all()


# ------------------------------------------------------------------------------------------------ sampling
def drawn(x, draws, **params):
    rows = torch.from_numpy(np.asarray(x, dtype=np.float32)).cuda()[None].expand(len(draws), len(x))
    return run_sample(rows, draws, **params)[0].tolist()


FORMS = [{}, dict(min_p=1e-30), dict(top_p=0.99999), dict(top_k=60000), dict(top_k=50), dict(top_p=0.5), dict(temperature=0.9)]


@pytest.mark.parametrize("params", FORMS, ids=str)
@pytest.mark.parametrize("front", [1, 700, 8192, 65000])
def test_sample_draws_near_0_pass_over_entries_that_weigh_nothing(front, params):
    """entries 55 and more powers of two below the largest stand before all others: no draw, 0 itself included, takes them"""
    x = np.full(65536, -40.0)
    x[front:] = -np.arange(65536 - front) / 65536  # the largest first
    assert drawn(x, [0.0, 1e-30, 1e-12], **params) == [front] * 3


def test_sample_draws_near_0_between_entries_that_weigh_nothing():
    """one light entry far along, none else beside the largest at the end"""
    x = np.full(50277, -np.inf)
    x[::3] = -45.0
    x[30000], x[50000] = -10.0, 0.0
    assert drawn(x, [0.0, 1e-20, 1e-3, 0.5]) == [30000, 30000, 50000, 50000]


@pytest.mark.parametrize("params", [{}, dict(min_p=1e-25), dict(top_k=5), dict(top_k=5, min_p=1e-25)], ids=str)
def test_sample_what_weighs_does_not_hang_on_the_filters(params):
    """44 powers of two below the largest is where weights end, whatever filter keeps the entry: of 30.4 (43.86 powers of two)
    and 30.6 (44.15) below it, before it, draw 0 takes the first and not the second"""
    assert drawn([-30.4, 0.0, -1.0, -2.0, -3.0, -50.0], [0.0], **params) == [0]
    assert drawn([-30.6, 0.0, -1.0, -2.0, -3.0, -50.0], [0.0], **params) == [1]


def test_sample_what_weighs_among_thousands_of_equal_entries():
    for light, token in ((-30.4, 0), (-30.6, 1)):
        x = np.zeros(3005)
        x[0], x[3001:] = light, -np.inf
        for params in ({}, dict(min_p=1e-25), dict(top_k=3004), dict(top_k=3003, min_p=1e-25)):
            assert drawn(x, [0.0], **params) == [token], (light, params)


# ------------------------------------------------------------------------------------------------ 4-bit products
@pytest.mark.parametrize("rows", [1, 3, 20, 70])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_product_of_very_large_rows(rows, kind):
    """magnitudes that sum to just below 2^122 in every group, scales that bring the results back: sums of 62 times as much at
    most stay below 2^128"""
    for group, zeros in ((32, True), (128, False)):
        x, codes, scales, z = product_case(rows, 50, 384, group, TYPES[kind], torch.float16, zeros, rows)
        signs = torch.where(x > 0, 1.0, -1.0)
        x = (signs * (2.0**122 / group) * (0.5 + x.abs().clamp(max=2) / 4.1)).to(TYPES[kind])
        x[:, ::7] = x[:, ::7].abs()
        assert (x.double().abs().reshape(rows, -1, group).sum(-1) < 2.0**122).all()
        check_product(x, codes, (scales / 1024).float(), z, group)


@pytest.mark.parametrize("rows", [3, 20, 70])
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_product_of_a_row_that_is_not_finite(rows, kind, value):
    x, codes, scales, z = product_case(rows, 50, 300, 64, TYPES[kind], torch.float16, True, rows)
    want = check_product(x, codes, scales, z, 64)
    x[1, 217] = value
    y = torch.empty_like(want)
    load_module("clear_ops").Q4Matrix(codes, scales, z, in_features=300, group=64).product(x, y)
    assert torch.isnan(y[1]).all()
    keep = torch.arange(rows) != 1
    assert torch.equal(y[keep], want[keep])
