"""GPU tests of the drafting model that learns (clear_learn.py), and of the drafting model's scores: the operators that score and
train together, against the same model in 64 bits."""
import math

import pytest

from engine_loader import load_module

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

LAYERS, D, VOCAB = 2, 128, 700

# A product sums up to 700 float32 terms, off by sqrt(700) 2^-24 = 1.6e-6 of their size where roundings fall as they may; a dozen
# of such stages follow each other, and a gradient may be a tenth of what its terms are: 2e-4.
CLOSE = 1e-3
# in bf16 every stage is rounded to 2^-9 of its size on average; a dozen and their sums
CLOSE_16 = 0.1


def learner(**more):
    return load_module("clear_learn").Learner(layers=LAYERS, d=D, vocab=VOCAB, seed=3, **{"dtype": torch.float32, **more})


def texts(lanes, n, seed=1):
    return torch.randint(0, VOCAB, (lanes, n), generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def plain(matrices, vectors, tokens, lengths):
    """the model's logits in 64 bits, [lanes, n, vocab], by torch's autograd"""
    lanes, n = tokens.shape

    def norm(x, w, b):
        x = x - x.mean(-1, keepdim=True)
        return x / (x.square().mean(-1, keepdim=True) + 1e-5).sqrt() * w + b

    x = matrices[0][tokens] * D**0.5
    for i in range(LAYERS):
        w_in, w_out = matrices[2 + 2 * i:4 + 2 * i]
        nw, nb, bias = vectors[2 + 3 * i:5 + 3 * i]
        z, v, s = (norm(x, nw, nb) @ w_in.t()).split(D, -1)
        gate, h, out = torch.sigmoid(z + bias), torch.zeros((lanes, D), dtype=torch.float64, device="cuda"), []
        for t in range(n):
            there = (lengths > t)[:, None]
            h = torch.where(there, gate[:, t] * h + (1 - gate[:, t]) * v[:, t], h)
            out.append(torch.where(there, h, torch.zeros_like(h)))
        x = x + (torch.stack(out, 1) * torch.nn.functional.silu(s)) @ w_out.t()
    return norm(x, *vectors[:2]) @ matrices[1].t()


def plain_loss(matrices, vectors, tokens, lengths):
    n = tokens.shape[1]
    logp = torch.log_softmax(plain(matrices, vectors, tokens, lengths), -1)
    there = torch.arange(1, n, device="cuda")[None] < lengths[:, None]
    return -(logp[:, :-1].gather(-1, tokens[:, 1:, None])[..., 0] * there).sum() / there.sum()


def in_64(model):
    return [[t.double().requires_grad_() for t in ts] for ts in (model.matrices, model.vectors)]


CASES = [(3, 37, None), (4, 150, (150, 1, 0, 77)), (1, 2, None), (9, 300, None)]


@pytest.mark.parametrize("lanes, n, lengths", CASES, ids=str)
def test_gradients_against_autograd_in_64_bits(lanes, n, lengths):
    model, tokens = learner(), texts(lanes, n)
    lengths = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    matrices, vectors = in_64(model)
    full = torch.full((lanes,), n, device="cuda") if lengths is None else lengths
    want = plain_loss(matrices, vectors, tokens, full)
    grads = torch.autograd.grad(want, matrices + vectors)
    loss, dmatrices, dvectors = model.gradients(tokens, lengths)
    assert abs(loss.item() - want.item()) <= CLOSE * want.item()
    for i, (got, g) in enumerate(zip(dmatrices + dvectors, grads)):
        assert (got.double() - g).norm() <= CLOSE * g.norm() + 1e-12, i


def test_gradients_in_bf16_and_the_rows_of_several_products():
    model, tokens = learner(dtype=torch.bfloat16), texts(5, 90)
    matrices, vectors = in_64(model)
    grads = torch.autograd.grad(plain_loss(matrices, vectors, tokens, torch.full((5,), 90, device="cuda")), matrices + vectors)
    for rows in (8192, 128):
        model.ROWS = rows
        _, dmatrices, dvectors = model.gradients(tokens)
        for i, (got, g) in enumerate(zip(dmatrices + dvectors, grads)):
            assert (got.double() - g).norm() <= CLOSE_16 * g.norm(), (rows, i)


def test_texts_of_no_and_of_one_token_and_tokens_outside():
    model = learner()
    for n in (0, 1):
        loss, dmatrices, dvectors = model.gradients(texts(3, n))
        assert loss.item() == 0 and all((g == 0).all() for g in dmatrices + dvectors)
        assert model.score(texts(3, n))[0].shape == (3, n)
    tokens = texts(2, 20)
    tokens[0, 7] = VOCAB + 5  # as what follows it counts for nothing, as a token it is a row of zeros
    want = model.score(tokens)[0]
    assert want[0, 6] == 0 and torch.isfinite(want).all()
    assert abs(model.gradients(tokens)[0].item() + want.sum().item() / 37) <= CLOSE


def test_a_step_moves_the_parameters_as_adamw_says():
    """the first step's moments are the gradient's: every entry moves by lr, against it, where the gradient is not tiny"""
    model, tokens = learner(), texts(3, 40)
    before = [w.clone() for w in model.matrices]
    _, grads, _ = model.gradients(tokens)
    grads = [g.clone() for g in grads]
    model.learn(tokens, lr=0.01)
    for w, b, g in zip(model.matrices, before, grads):
        large = g.abs() > 1e-5  # eps of 1e-8 is 1e-3 of that
        moved = b - 0.01 * (0.01 * b + g.sign())
        assert ((w - moved).abs()[large] <= 0.01 * 2e-3).all()


@pytest.mark.parametrize("bits, dtype", [(32, torch.float32), (32, torch.bfloat16), (8, torch.float16)], ids=str)
def test_learning_runs_and_is_the_same_again(bits, dtype):
    tokens, ends = texts(6, 70), []
    lengths = torch.tensor([70, 3, 50, 0, 1, 70], dtype=torch.int32, device="cuda")
    for _ in range(2):
        model = learner(bits=bits, dtype=dtype)
        losses = [model.learn(tokens, lengths).item() for _ in range(4)]
        assert all(math.isfinite(x) for x in losses)
        ends.append((losses, [w.clone() for w in model.matrices + model.vectors]))
    assert ends[0][0] == ends[1][0] and all(torch.equal(a, b) for a, b in zip(ends[0][1], ends[1][1]))
    if dtype != torch.float32:
        assert all(torch.equal(w, p.to(dtype)) for w, p in zip(model.weights, model.matrices))


def test_scores_against_64_bits():
    model, tokens = learner(), texts(4, 60)
    lengths = torch.tensor([60, 1, 0, 33], dtype=torch.int32, device="cuda")
    matrices, vectors = in_64(model)
    logits = plain(matrices, vectors, tokens, lengths).detach()
    logp = torch.log_softmax(logits, -1)
    logprobs, entropy, top, top_logprobs = model.score(tokens, lengths, top=5)
    for lane, n in enumerate(lengths.tolist()):
        for t in range(max(0, n - 1)):
            row = logp[lane, t]
            assert abs(logprobs[lane, t].item() - row[tokens[lane, t + 1]].item()) <= 10 * CLOSE
            assert abs(entropy[lane, t].item() + (row.exp() * row).sum().item()) <= 10 * CLOSE
            assert (row[top[lane, t]] - row.topk(5).values).abs().max() <= 10 * CLOSE
            assert (top_logprobs[lane, t].double() - row[top[lane, t]]).abs().max() <= 10 * CLOSE
        assert (logprobs[lane, max(0, n - 1):] == 0).all()


def test_steps_continue_a_prompt():
    """a text as a prompt and single tokens gives the logits of the whole text"""
    model, tokens = learner(), texts(3, 50)
    matrices, vectors = in_64(model)
    lengths = torch.tensor([44, 1, 20], dtype=torch.int32, device="cuda")
    model.reset(3)
    got = [model.prompt(tokens[:, :44], lengths)]
    for t in range(44, 50):
        got.append(model.step(tokens[:, t]))
    for lane, n in enumerate(lengths.tolist()):
        text = torch.cat((tokens[lane, :n], tokens[lane, 44:]))[None]
        want = plain(matrices, vectors, text, torch.tensor([text.shape[1]], device="cuda")).detach()[0, n - 1:]
        for i, row in enumerate(want):
            assert (got[i][lane].double() - row).abs().max() <= 10 * CLOSE * row.square().mean().sqrt(), (lane, i)


def test_generate_draws_the_largest_logits():
    model, tokens = learner(), texts(2, 30)
    matrices, vectors = in_64(model)
    out = model.generate(tokens, 5, torch.zeros((5, 2), device="cuda"), temperature=torch.zeros(2, device="cuda"))
    full = torch.cat((tokens, out), 1)
    logits = plain(matrices, vectors, full, torch.full((2,), 35, device="cuda")).detach()
    for lane in range(2):
        for i in range(5):
            row = logits[lane, 29 + i]
            assert row[out[lane, i]] >= row.max() - 20 * CLOSE * row.square().mean().sqrt()
    with pytest.raises(load_module("clear_ops").ClearError):
        learner().step(tokens[:, 0])


def test_the_drafting_models_scores_against_64_bits():
    """clear_draft.Draft's, with its 4-bit head"""
    from test_gpu_clear_draft import D as draft_d, HEADS, LAYERS as draft_layers, VOCAB as draft_vocab, plain_logits
    draft = load_module("clear_draft").Draft(layers=draft_layers, d=draft_d, heads=HEADS, vocab=draft_vocab, seed=3, dtype=torch.float32)
    tokens = torch.randint(0, draft_vocab, (3, 40), generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
    lengths = torch.tensor([40, 1, 22], dtype=torch.int32, device="cuda")
    draft.reset(3)
    draft.prompt(tokens)
    before = [s.clone() for s in draft.states]
    logprobs, entropy, top, _ = draft.score(tokens, lengths, top=3)
    assert all(torch.equal(a, b) for a, b in zip(before, draft.states))  # scoring is beside the lanes' conversations
    assert logprobs.shape == (3, 39) and top.shape == (3, 39, 3)
    for lane, n in enumerate(lengths.tolist()):
        want = torch.log_softmax(torch.from_numpy(plain_logits(tokens[lane, :n].tolist())), -1)
        size = want.sub(want.mean()).square().mean().sqrt()
        for t in range(n - 1):
            # logits of prompt and steps are within 1e-3 of their size (test_gpu_clear_use.py); a difference of two, and the sum
            assert abs(logprobs[lane, t].item() - want[t, tokens[lane, t + 1]].item()) <= 3e-3 * size
            assert abs(entropy[lane, t].item() + (want[t].exp() * want[t]).sum().item()) <= 2e-2 * size
        assert (logprobs[lane, max(0, n - 1):] == 0).all()
    assert [t.shape[1] for t in draft.score(tokens[:, :1])] == [0, 0]


def test_the_drafting_models_scores_of_padding_outside_the_vocabulary_and_after_an_error():
    from test_gpu_clear_draft import D as draft_d, HEADS, LAYERS as draft_layers, VOCAB as draft_vocab
    draft = load_module("clear_draft").Draft(layers=draft_layers, d=draft_d, heads=HEADS, vocab=draft_vocab, seed=3, dtype=torch.float32)
    draft.reset(2)
    states = draft.states
    tokens, lengths = texts(2, 9) % draft_vocab, torch.tensor([9, 4], dtype=torch.int32, device="cuda")
    want = draft.score(tokens, lengths)
    for pad in (-1, -100, draft_vocab, 1 << 40):
        padded = tokens.clone()
        padded[1, 4:] = pad
        assert all(torch.equal(a[0], b[0]) and torch.equal(a[1, :3], b[1, :3]) for a, b in zip(draft.score(padded, lengths), want))
    with pytest.raises(load_module("clear_ops").ClearError):
        draft.score(tokens, lengths.long())
    assert draft.states is states and all(not s.any() for s in states)
