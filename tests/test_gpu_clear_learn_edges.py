"""GPU tests of the learning and the drafting model (clear_learn.py, clear_draft.py) and of AdamW where calls come to the edge of
what they take."""
import pytest

from engine_loader import load_module
from test_gpu_clear_learn import CLOSE_16, D, LAYERS, in_64, learner, plain_loss, texts

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

# float16 has three bits more than bfloat16, whose bound is CLOSE_16
CLOSE_F16 = CLOSE_16 / 8


def float16_gradients(tokens, lengths=None):
    """loss and gradients of a float16 model of all 65,536 tokens and those of the same model in 64 bits"""
    model = load_module("clear_learn").Learner(layers=LAYERS, d=D, seed=3, dtype=torch.float16)
    matrices, vectors = in_64(model)
    full = torch.full((len(tokens),), tokens.shape[1], device="cuda") if lengths is None else lengths
    want = plain_loss(matrices, vectors, tokens, full)
    grads = torch.autograd.grad(want, matrices + vectors)
    loss, dmatrices, dvectors = model.gradients(tokens, lengths)
    assert abs(loss.item() - want.item()) <= CLOSE_F16 * want.item()
    return dmatrices + dvectors, grads


@pytest.mark.parametrize("lengths", [None, "ragged"])
def test_gradients_in_float16_of_many_positions(lengths):
    """a position's weight times a token's probability is 1 / (4,096 65,536) = 4e-9, float16's smallest number 6e-8"""
    tokens = torch.randint(0, 65536, (64, 65), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    if lengths is not None:
        lengths = (torch.arange(64, device="cuda") + 2).int()
    got, want = float16_gradients(tokens, lengths)
    for i, (g, w) in enumerate(zip(got, want)):
        assert (g.double() - w).norm() <= CLOSE_F16 * w.norm(), i
    assert got[1].any(1).all()  # every row of the head learns


def test_gradients_in_float16_of_one_token_all_along():
    """8,192 positions whose gradients add up"""
    got, want = float16_gradients(torch.full((64, 129), 77, device="cuda"))
    for i, (g, w) in enumerate(zip(got, want)):
        assert torch.isfinite(g).all() and (g.double() - w).norm() <= CLOSE_F16 * w.norm() + 1e-12, i


@pytest.mark.parametrize("lanes, n", [(3, 0), (0, 5), (3, 1), (1, 2)])
def test_gradients_in_float16_of_hardly_any_positions(lanes, n):
    model, tokens = learner(dtype=torch.float16), texts(lanes, n)
    used = [torch.full_like(w, 7.0) for w in model.matrices for _ in range(4)]
    del used  # what is not written is not 0
    loss, dmatrices, dvectors = model.gradients(tokens)
    assert all(torch.isfinite(g).all() and g.dtype == torch.float32 for g in dmatrices + dvectors)
    assert n == 2 or loss.item() == 0 and not any(g.any() for g in dmatrices + dvectors)


def test_scores_where_nothing_follows_are_zeros():
    model, tokens = learner(), texts(4, 30)
    tokens[0, 9] = -5  # no token follows position 8, nor the last of a text
    lengths = torch.tensor([30, 1, 0, 12], dtype=torch.int32, device="cuda")
    logprobs, entropy = model.score(tokens, lengths)
    nothing = torch.arange(1, 31, device="cuda")[None] >= lengths[:, None]
    nothing[0, 8] = True
    assert (logprobs[nothing] == 0).all() and (entropy[nothing] == 0).all()
    assert (logprobs[~nothing] < 0).all() and (entropy[~nothing] > 0).all()


@pytest.mark.parametrize("lengths", [None, (0, 3)])
def test_a_prompt_of_no_tokens_gives_the_logits_of_rows_of_zeros(lengths):
    """as one whose lengths are 0 does, and leaves the states"""
    model = learner()
    model.reset(2)
    for s in model.states:
        s.fill_(0.5)
    lengths = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    logits = model.prompt(texts(2, 0), lengths)
    assert logits.shape == (2, 700) and not logits.any() and all((s == 0.5).all() for s in model.states)
    assert model.generate(texts(2, 0), 3, torch.full((3, 2), 0.5, device="cuda")).shape == (2, 3)


def draft():
    from test_gpu_clear_draft import D as d, HEADS, LAYERS as layers, VOCAB as vocab
    return load_module("clear_draft").Draft(layers=layers, d=d, heads=HEADS, vocab=vocab, seed=3, dtype=torch.float32), vocab


def test_a_score_leaves_the_drafting_models_states_alone_while_it_runs(monkeypatch):
    """another thread's step meets its own lanes"""
    model, vocab = draft()
    model.reset(2)
    states, ops, calls = model.states, load_module("clear_draft").clear_ops, []
    prompt = ops.linear_attention_prompt

    def during(*args, **more):
        calls.append(model.states is states)
        return prompt(*args, **more)

    monkeypatch.setattr(ops, "linear_attention_prompt", during)
    model.score(texts(3, 9) % vocab)
    assert len(calls) == len(states) and all(calls)


def test_a_token_outside_the_vocabulary_is_a_row_of_zeros_to_the_drafting_models_scores():
    """whichever it is; it takes no other token's place"""
    model, vocab = draft()
    tokens = texts(1, 12) % vocab
    scores = []
    for outside in (-1, vocab, 1 << 40, -(1 << 40)):
        tokens[0, 5] = outside
        logprobs, entropy = model.score(tokens)
        assert logprobs[0, 4].item() == 0 and torch.isfinite(logprobs).all()
        scores.append((logprobs, entropy))
    assert all(torch.equal(a, b) for s in scores[1:] for a, b in zip(s, scores[0]))
    model.embedding = torch.cat((model.embedding, torch.zeros_like(model.embedding[:1])))  # the last token's row
    tokens[0, 5] = vocab
    assert torch.equal(model.score(tokens)[1], scores[0][1])


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("before", [0, -1, -(1 << 31)])
def test_adamw_of_a_step_on_the_device_before_the_first_changes_nothing(bits, before):
    c = load_module("clear_ops")
    gen = torch.Generator(device="cuda").manual_seed(bits)
    p, g = torch.randn(5000, generator=gen, device="cuda"), torch.randn(5000, generator=gen, device="cuda")
    copy = torch.full((5000,), 7.0, device="cuda").bfloat16()
    opt = c.AdamW([p], bits=bits, copies=[copy])
    opt.step([g], lr=0.1, step=1)
    kept = [t.clone().view(torch.uint8) for t in (p, copy, *(s[0] for s in opt.states))]
    step = torch.tensor([before], dtype=torch.int32, device="cuda")
    opt.step([g], lr=0.1, step=step)
    assert all(torch.equal(t.view(torch.uint8), k) for t, k in zip((p, copy, *(s[0] for s in opt.states)), kept))
    step.fill_(2)
    opt.step([g], lr=0.1, step=step)
    assert torch.isfinite(p).all() and not torch.equal(p.view(torch.uint8), kept[0])


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("g", [1e-15, 1e-18, 3e-19, 1e-19, 3e-20])
def test_adamw_of_gradients_whose_squares_are_below_the_normal_numbers(bits, g):
    """beside an eps that is smaller still: the first step moves by lr.  The square and v lie on steps of 2^-149 there, which is
    half of that over v in the root, and the rest is 40 2^-24 as for other gradients"""
    p = torch.zeros(1029, device="cuda")
    grad = torch.full((1029,), g, device="cuda")
    opt = load_module("clear_ops").AdamW([p], betas=(0.9, 0.99), eps=1e-30, weight_decay=0.0, bits=bits)
    opt.step([grad], lr=1.0, step=1)
    off = 40 * 2.0**-24 + 0.5 * 1.01 * 2.0**-150 / (0.01 * g * g)
    assert ((p + 1).abs() <= off).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_of_a_gradient_whose_square_overflows(bits):
    """in 32 bits its v is infinite and its entry stays where it is from then on, in 8 its block of 256 is lost"""
    c = load_module("clear_ops")
    gen = torch.Generator(device="cuda").manual_seed(1)
    first, second = torch.randn(2000, generator=gen, device="cuda"), torch.randn(2000, generator=gen, device="cuda")
    large = first.clone()
    large[700] = 1e20
    clean, p = torch.zeros(2000, device="cuda"), torch.zeros(2000, device="cuda")
    for param, gradients in ((clean, (first, second)), (p, (large, second))):
        opt = c.AdamW([param], bits=bits)
        for i, g in enumerate(gradients):
            opt.step([g], lr=0.01, step=i + 1)
    hit = torch.zeros(2000, dtype=torch.bool, device="cuda")
    if bits == 32:
        hit[700] = True
        assert p[700].item() == 0
    else:
        hit[512:768] = True
        assert torch.isnan(p[hit]).all()
    assert torch.equal(p[~hit], clean[~hit])
