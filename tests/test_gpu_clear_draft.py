"""GPU tests of the drafting model (clear_draft.py): the operators in the clear together, against the same model in 64 bits."""
import numpy as np
import pytest

from engine_loader import load_module

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

LAYERS, D, HEADS, VOCAB = 2, 128, 2, 700


@pytest.fixture(scope="module")
def draft():
    return load_module("clear_draft").Draft(layers=LAYERS, d=D, heads=HEADS, vocab=VOCAB, seed=3, dtype=torch.float32)


def plain_weights():
    """the model's matrices in 64 bits, made from the same seed in the same order"""
    ops = load_module("clear_ops")
    rng = np.random.default_rng(3)

    def matrix(out, n_in, scale=1.0):
        w = (scale / np.sqrt(n_in)) * rng.standard_normal((out, n_in), dtype=np.float32)
        codes, scales, _ = ops.quantize_q4(w, 64)
        c = np.stack((codes & 15, codes >> 4), -1).reshape(out, -1)[:, :n_in].astype(np.float64) - 8
        return c * np.repeat(scales.astype(np.float64), 64, 1)[:, :n_in]

    w_in = [matrix(4 * D, D) for _ in range(LAYERS)]
    w_out = [matrix(D, D, 0.5) for _ in range(LAYERS)]
    head = matrix(VOCAB, D, 3.0)
    embedding = (0.5 * rng.standard_normal((VOCAB, D), dtype=np.float32)).astype(np.float64)
    return w_in, w_out, head, embedding


def plain_logits(tokens):
    """the logits after every token of one lane, token by token in 64 bits"""
    w_in, w_out, head, embedding = plain_weights()
    hs = D // HEADS
    decay = np.exp(-np.exp2(-np.linspace(3, 8, HEADS)))
    states = [np.zeros((HEADS, hs, hs)) for _ in range(LAYERS)]

    def norm(x):
        return x / np.sqrt(np.mean(x * x, axis=-1, keepdims=True) + 1e-5)

    out = []
    for t in tokens:
        x = embedding[t]
        for i in range(LAYERS):
            q, k, v, gate = (w_in[i] @ norm(x)).reshape(4, HEADS, hs)
            states[i] = states[i] * decay[:, None, None] + k[:, :, None] * v[:, None, :]
            o = norm(np.einsum("hd,hdc->hc", q, states[i]) * hs**-0.5) * (gate / (1 + np.exp(-gate)))
            x = x + w_out[i] @ o.reshape(-1)
        out.append(head @ norm(x))
    return np.array(out)


def logits_of(draft, hidden):
    out = torch.empty((len(hidden), VOCAB), device="cuda")
    draft.head.product(hidden, out)
    return out.double().cpu().numpy()


# Products of 128 columns lose up to 2 (64 + 18) 2^-24 of magnitudes 32 times the codes' and about 10 times the result's: 3e-3 of
# an output's size where every rounding falls the same way, 1e-4 where they fall as they may; three in a row and the norms.
CLOSE = 1e-3


def test_prompt_and_steps_against_64_bits(draft):
    rng = np.random.default_rng(1)
    lengths = [70, 1, 33]
    tokens = rng.integers(0, VOCAB, (3, 75))
    draft.reset(3)
    hidden = draft.prompt(torch.from_numpy(tokens[:, :70]).cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    got = [logits_of(draft, hidden)]
    for t in range(5):
        got.append(logits_of(draft, draft.step(torch.from_numpy(tokens[:, 70 + t]).cuda())))
    for lane, n in enumerate(lengths):
        want = plain_logits(np.concatenate((tokens[lane, :n], tokens[lane, 70:])))[n - 1:]
        for step in range(6):
            off = np.abs(got[step][lane] - want[step]).max()
            assert off <= CLOSE * np.sqrt(np.mean(want[step] ** 2)) * 10, (lane, step, off)


def test_generate_draws_what_the_logits_say(draft):
    """greedy: every token is the largest of its 64-bit logits, up to a gap that rounding may close"""
    rng = np.random.default_rng(2)
    prompt = rng.integers(0, VOCAB, (2, 40))
    out = draft.generate(torch.from_numpy(prompt).cuda(), 6, torch.zeros((6, 2), device="cuda"),
                         temperature=torch.zeros(2, device="cuda")).cpu().numpy()
    for lane in range(2):
        want = plain_logits(np.concatenate((prompt[lane], out[lane])))
        for i, token in enumerate(out[lane]):
            row = want[39 + i]
            assert row[token] >= row.max() - 20 * CLOSE * np.sqrt(np.mean(row**2))


def test_generate_is_the_same_again_and_follows_its_draws(draft):
    gen = torch.Generator(device="cuda").manual_seed(5)
    tokens = torch.randint(0, VOCAB, (4, 20), generator=gen, device="cuda")
    draws = torch.rand((8, 4), generator=gen, device="cuda")
    filters = dict(temperature=torch.full((4,), 1.0, device="cuda"), top_k=torch.full((4,), 50, dtype=torch.int32, device="cuda"))
    first = draft.generate(tokens, 8, draws, **filters)
    assert torch.equal(draft.generate(tokens, 8, draws, **filters), first)
    assert not torch.equal(draft.generate(tokens, 8, 1 - draws, **filters), first)
    assert ((first >= 0) & (first < VOCAB)).all()


def test_answer_takes_decrypted_rows(draft):
    """float64 rows on the host, as decryption gives them, and the same rows on the GPU"""
    rows = np.random.default_rng(4).standard_normal((32, D))
    answer = load_module("clear_draft").answer
    draws = torch.full((32,), 0.25, device="cuda")
    kept = torch.full((32,), 0.8, device="cuda")
    got = answer(rows, draft.head, draws, top_p=kept)
    again = answer(torch.from_numpy(rows).cuda().float(), draft.head, draws, top_p=kept)
    assert torch.equal(got, again)
