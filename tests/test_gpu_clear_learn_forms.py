"""GPU tests of the forms of the kernels that score and train which long rows, wide and odd channels, 16-bit gradients and the model's
own slices take, against the definitions in 64 bits of test_gpu_clear_learn_ops.py, with its tolerances."""
import math

import pytest

from test_gpu_clear_learn_ops import (TYPES, check_embedding, check_recurrence, check_score, generator, normal, run_gradient, score,
                                      score_case, some_tokens)

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

ROWS = 520  # from 512 on rows are not cut into parts


# ------------------------------------------------------------------------------------------------ whole long rows by 1,024 threads
@pytest.mark.parametrize("vocab", [8193, 9001, 20011, 32768])
@pytest.mark.parametrize("kind", TYPES)
def test_score_of_many_long_rows(vocab, kind):
    """the row's end in every group of the threads' vectors; the gradient by itself, at once and in the logits' place"""
    print(f"vocabulary {vocab}, {kind}", flush=True)
    check_score(*score_case(ROWS, vocab, TYPES[kind], vocab))


@pytest.mark.parametrize("kind", TYPES)
def test_score_of_many_long_rows_at_every_alignment(kind):
    vocab, gen = 9002, generator(5)
    wide = normal(gen, ROWS, vocab + 7).to(TYPES[kind])
    logits = wide[:, 3:3 + vocab]
    assert logits.stride()[0] % 8 == 1
    tokens, w, u = torch.randint(0, vocab, (ROWS,), generator=gen, device="cuda"), normal(gen, ROWS), normal(gen, ROWS)
    check_score(logits, tokens, w, u)
    want = score(logits, tokens, 0, w, u, at_once=True)
    gaps = torch.full((ROWS, vocab + 9), 7.0, device="cuda").to(TYPES[kind])
    assert torch.equal(score(logits, tokens, 0, w, u, at_once=True, gradient=gaps[:, 5:5 + vocab])[5], want[5])
    assert (gaps[:, :5] == 7).all() and (gaps[:, 5 + vocab:] == 7).all()
    around = wide.clone()
    got = score(logits, tokens, 0, w, u, at_once=True, gradient=logits)
    assert all(torch.equal(got[i], want[i]) for i in (0, 1, 2, 5)) and torch.equal(logits, want[5])
    assert torch.equal(wide[:, :3], around[:, :3]) and torch.equal(wide[:, 3 + vocab:], around[:, 3 + vocab:])


@pytest.mark.parametrize("kind", TYPES)
def test_score_of_many_long_rows_with_masked_values(kind):
    kind = TYPES[kind]
    vocab, lowest = 9000, torch.finfo(kind).min
    x = torch.full((ROWS, vocab), -math.inf, device="cuda").to(kind)
    x[1::6] = lowest          # all alike
    x[2::6, 8321] = lowest    # the only one
    x[3::6], x[3::6, 77] = lowest, 2.0
    x[4::6, 4090:4093] = 1.0
    x[5::6, 100:] = 0.0
    tokens = torch.tensor([5, 5, 8321, 77, 4091, -1], device="cuda").repeat(ROWS)[:ROWS]
    ones = torch.ones(ROWS, device="cuda")
    third, all_, most = math.log(3), math.log(vocab), math.log(vocab - 100)
    want = torch.tensor([[-math.inf, -all_, 0.0, 0.0, -third, 0.0], [0.0, all_, 0.0, 0.0, third, most]], device="cuda").repeat(1, ROWS)[:, :ROWS]
    for at_once in (False, True):
        lp, entropy, _, _, _, grad = score(x, tokens, 0, ones, ones, at_once=at_once)
        # a sum of 9,000 equal terms by 1,024 threads is exact up to its logarithm
        assert torch.allclose(lp, want[0], rtol=1e-5, atol=0) and torch.allclose(entropy, want[1], rtol=1e-5, atol=1e-6)
        assert torch.isfinite(grad).all() and (grad[0::6] == 0).all() and (grad[2::6].abs() <= 1e-6).all()
        assert (grad[3::6].abs() <= 1e-6).all() and (grad[5::6, :100] == 0).all()


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("at", [0, 4444, 8999])
def test_score_of_long_rows_that_are_not_finite(value, at):
    logits, tokens, w, u = score_case(ROWS, 9000, torch.bfloat16, 1)
    for at_once in (False, True):
        w[1] = u[1] = 1
        x = logits.clone()
        want = score(x, tokens, 0, w, u, at_once=at_once)
        x[1, at] = value
        tokens[1] = 17
        got = score(x, tokens, 0, w, u, at_once=at_once)
        keep = torch.arange(ROWS, device="cuda") != 1
        assert all(torch.equal(got[i][keep], want[i][keep]) for i in (0, 1, 2, 5))
        assert torch.isnan(got[0][1]) and torch.isnan(got[1][1]) and torch.isnan(got[5][1]).all()
        w[1] = u[1] = 0
        assert (score(x, tokens, 0, w, u, at_once=at_once)[5][1] == 0).all()


def test_score_of_long_rows_with_nan_beside_logits_out_of_all_proportion():
    x = torch.zeros((ROWS, 9000), device="cuda")
    x[:, 5], x[:, 4000:4004], x[:, 8000] = math.nan, 2.0**120, 2.0**121
    x[1, 5] = 0.0
    for at_once in (False, True):
        lp, entropy, _, _, _, grad = score(x, torch.full((ROWS,), 8000, device="cuda"), 0, torch.ones(ROWS, device="cuda"), at_once=at_once)
        keep = torch.arange(ROWS, device="cuda") != 1
        assert torch.isnan(lp[keep]).all() and torch.isnan(entropy[keep]).all() and torch.isnan(grad[keep]).all()
        assert lp[1].item() == 0 and entropy[1].item() == 0 and (grad[1] == 0).all()


# ------------------------------------------------------------------------------------------------ large and masked logits
# by a wave, by 256 threads, in parts or by 1,024 threads
SHAPES = [(4, 300), (4, 5000), (4, 20011), (600, 300), (600, 5000), (520, 20011)]


@pytest.mark.parametrize("rows, vocab", SHAPES)
@pytest.mark.parametrize("k", [0, 5])
def test_score_of_logits_masked_by_large_numbers(rows, vocab, k):
    """before the others, behind them, among them, all of a row and all but one of it"""
    w, u = normal(generator(1), rows), normal(generator(2), rows)
    tokens = torch.randint(0, vocab, (rows,), generator=generator(3), device="cuda")
    for mask in (-1e4, -1e9, -1e10, -1e20, -1e30, -3e38, 5e8, 1e10, 1e30):
        for kind in (torch.float32, torch.bfloat16):
            print(f"{mask}, {kind}", flush=True)
            x = 2 * normal(generator(vocab), rows, vocab)
            x[0::4, :vocab // 2], x[1::4, vocab // 3:], x[2::4], x[3::4, ::3] = mask, mask, mask, mask
            x[1::8, 5::7] = mask
            x[2::8, vocab - 2] = mask + abs(mask) / 64
            check_score(x.to(kind), tokens, w, u, k)


@pytest.mark.parametrize("rows, vocab", SHAPES)
def test_score_of_rising_logits_far_from_zero(rows, vocab):
    """the largest moves up again and again, by more and by less than the logits' own steps at that size"""
    ramp = torch.arange(vocab, device="cuda") * (60.0 / vocab) + normal(generator(4), rows, vocab)
    w, u = normal(generator(1), rows), normal(generator(2), rows)
    tokens = torch.randint(0, vocab, (rows,), generator=generator(3), device="cuda")
    for offset in (1e3, 1e4, 1e5, -1e5, 3e7, -3e8, 2.0**29, -2.0**29, 2.0**30, 2e12, -1e25):
        print(offset, flush=True)
        x = (ramp.double() + offset).float()
        x[::3] = (offset + 64.0 * ramp[::3].double().round()).float()
        check_score(x, tokens, w, u)


# ------------------------------------------------------------------------------------------------ the gradient of sorted tokens
@pytest.mark.parametrize("d", [1, 3, 130, 513, 768, 1025, 2056, 4091])
@pytest.mark.parametrize("kind", TYPES)
def test_embedding_gradient_of_sorted_tokens_and_wide_rows(d, kind):
    """single elements and vectors, several groups of channels and several passes over them, in short and long runs; tables of
    float32 and of the rows' type, where they lie on vectors and where not"""
    kind = TYPES[kind]
    for n, shape in ((1025, "padded"), (3000, "few"), (3000, "one"), (9000, "padded")):
        print(f"{n} tokens, {shape}, {d} channels, {kind}", flush=True)
        gen = generator(n + d)
        tokens, rows = some_tokens(n, 300, d, shape), normal(gen, n, d).to(kind)
        for table in {torch.float32, kind}:
            want = check_embedding(tokens, normal(gen, 300, d), rows, scale=0.5, kind=table)
            flat = torch.full((300 * d + 8,), 7.0, device="cuda").to(table)
            # at an odd place by single elements; a column's rows meet in the same order
            got = run_gradient(tokens, rows, flat[1:1 + 300 * d].view(300, d), scale=0.5)
            assert torch.equal(got, want) and (flat[:1] == 7).all() and (flat[1 + 300 * d:] == 7).all()


# ------------------------------------------------------------------------------------------------ the model's slices
@pytest.mark.parametrize("lanes, T", [(32, 64), (2, 300), (1, 2000)])
@pytest.mark.parametrize("kind", TYPES)
def test_recurrence_of_slices_of_one_projection(lanes, T, kind):
    """as clear_learn.Learner hands them over: values and both gradients are slices of rows of three times 768"""
    C, gen = 768, generator(lanes)
    z, zvs, dzvs = ((2 * normal(gen, lanes, T, w)).to(TYPES[kind]) for w in (C, 3 * C, 3 * C))
    dz, dv, ds = dzvs.split(C, -1)
    kept = ds.clone()
    lengths = torch.randint(0, T + 1, (lanes,), generator=gen, device="cuda").int()
    lengths[0] = T
    check_recurrence(z + 2, zvs.split(C, -1)[1], None, normal(gen, lanes, T, C).to(TYPES[kind]), None, lengths, dz=dz, dx=dv)
    assert torch.equal(ds, kept)
