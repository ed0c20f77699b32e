"""GPU tests of the drafting model as it is used: on a stream of its own, with lanes that have no tokens, in what it refuses."""
import pytest

from engine_loader import load_module

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

D, HEADS, VOCAB = 128, 2, 700


def make():
    return load_module("clear_draft").Draft(layers=2, d=D, heads=HEADS, vocab=VOCAB, seed=3, dtype=torch.float32)


def test_model_built_and_run_on_a_side_stream():
    """while the null stream is busy with other work, which a side stream does not wait for"""
    gen = torch.Generator(device="cuda").manual_seed(5)
    tokens, draws = torch.randint(0, VOCAB, (4, 70), generator=gen, device="cuda"), torch.rand((6, 4), generator=gen, device="cuda")
    kept = torch.full((4,), 0.8, device="cuda")
    want = make().generate(tokens, 6, draws, top_p=kept)
    big = torch.zeros((8192, 8192), device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(8):
        big @ big
    with torch.cuda.stream(side):
        got = make().generate(tokens, 6, draws, top_p=kept)
        side.synchronize()
    assert torch.equal(got, want)
    torch.cuda.synchronize()


def test_calls_are_recorded_with_the_current_stream():
    """a graph takes up calls that name no stream"""
    c = load_module("clear_ops")
    gen = torch.Generator(device="cuda").manual_seed(1)
    logits, draws = torch.randn((5, 1000), generator=gen, device="cuda"), torch.rand(5, generator=gen, device="cuda")
    tokens = torch.full((5,), -7, dtype=torch.int64, device="cuda")
    c.sample(logits, draws, tokens)
    want = tokens.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.sample(logits, draws, tokens)
    for _ in range(3):
        tokens.fill_(-7)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(tokens, want)
        c.sample(logits, draws, tokens)
        torch.cuda.synchronize()


@pytest.mark.parametrize("where", ["cpu", "cuda"])
@pytest.mark.parametrize("kind", [torch.float64, torch.float32, torch.bfloat16])
def test_answer_takes_rows_of_every_kind(where, kind):
    """rows of decrypted values as they come, on the host or on the GPU: the tokens of the same values in float32"""
    d = load_module("clear_draft")
    head = d.matrix(d.np.random.default_rng(3), VOCAB, D, scale=3.0)
    rows = torch.randn((9, D), generator=torch.Generator().manual_seed(4), dtype=torch.float64).to(torch.bfloat16)
    draws = torch.rand(9, generator=torch.Generator().manual_seed(5)).cuda()
    want = d.answer(rows.float().cuda(), head, torch.zeros(9, device="cuda"), temperature=torch.zeros(9, device="cuda"))
    got = d.answer(rows.to(kind).to(where), head, draws, temperature=torch.zeros(9, device="cuda"))
    if kind == torch.bfloat16 and where == "cuda":  # logits of that type
        assert ((got >= 0) & (got < VOCAB)).all()
    else:
        assert torch.equal(got, want)


def test_matrices_of_one_row_and_of_one_byte_a_row():
    """strides of axes that have one entry say nothing, and must not be refused"""
    c = load_module("clear_ops")
    gen = torch.Generator(device="cuda").manual_seed(6)
    column = torch.randint(0, 256, (32, 1), generator=gen, device="cuda", dtype=torch.uint8)
    codes = torch.stack((column & 15, column >> 4), -1).double() - 8  # [32, 1, 2]
    one_row = column.t()  # [1, 32], one byte from row to row
    assert one_row.stride() == (1, 1)
    x, y = torch.randn((3, 64), generator=gen, device="cuda"), torch.empty((3, 1), device="cuda")
    c.Q4Matrix(one_row, torch.ones((1, 2), device="cuda"), group=32).product(x, y)
    want = x.double() @ codes.reshape(64, 1)
    assert ((y.double() - want).abs() <= 2 * (32 + 2 + 16) * 2.0**-24 * 32 * x.double().abs().sum(1, keepdim=True)).all()
    wide = torch.zeros((32, 40), dtype=torch.uint8, device="cuda")
    wide[:, 7:8] = column
    x, y = torch.randn((3, 2), generator=gen, device="cuda"), torch.empty((3, 32), device="cuda")
    c.Q4Matrix(wide[:, 7:8], torch.ones((32, 1), device="cuda"), group=32).product(x, y)
    want = x.double() @ codes.reshape(32, 2).t().contiguous()
    assert ((y.double() - want).abs() <= 2 * (2 + 1 + 16) * 2.0**-24 * 32 * x.double().abs().sum(1, keepdim=True)).all()


def test_logits_of_prompt_and_steps_are_float32s():
    """What CLOSE of test_gpu_clear_draft.py derives, 1e-4 for each of three products in a row where roundings fall as they may
    and the norms between them, without a factor on it"""
    from test_gpu_clear_draft import CLOSE, plain_logits
    model, gen = make(), torch.Generator(device="cuda").manual_seed(8)
    tokens = torch.randint(0, VOCAB, (3, 75), generator=gen, device="cuda")
    lengths = torch.tensor([70, 1, 33], dtype=torch.int32, device="cuda")
    model.reset(3)
    hidden = [model.prompt(tokens[:, :70], lengths)] + [model.step(tokens[:, 70 + t]) for t in range(5)]
    logits = torch.stack([torch.stack([h[lane] for h in hidden]) for lane in range(3)])  # lane, step, channel
    out = torch.empty((18, VOCAB), device="cuda")
    model.head.product(logits.flatten(0, 1), out)
    for lane, n in enumerate(lengths.tolist()):
        rows = torch.cat((tokens[lane, :n], tokens[lane, 70:])).tolist()
        want = torch.from_numpy(plain_logits(rows)[n - 1:])
        off = (out.view(3, 6, VOCAB)[lane].double().cpu() - want).abs().amax(1)
        assert (off <= CLOSE * want.square().mean(1).sqrt()).all(), (lane, off)


def test_lanes_without_tokens_draft_like_any_other():
    """a lane of length 0 begins from zeros; the others are not touched by it"""
    gen = torch.Generator(device="cuda").manual_seed(9)
    tokens, draws = torch.randint(0, VOCAB, (3, 20), generator=gen, device="cuda"), torch.rand((4, 3), generator=gen, device="cuda")
    lengths = torch.tensor([20, 0, 7], dtype=torch.int32, device="cuda")
    model = make()
    out = model.generate(tokens, 4, draws, lengths=lengths)
    assert ((out >= 0) & (out < VOCAB)).all()
    keep = torch.tensor([0, 2], device="cuda")
    assert torch.equal(model.generate(tokens[keep], 4, draws[:, keep], lengths=lengths[keep]), out[keep])
    assert model.generate(tokens[:, :0], 2, draws[:2]).shape == (3, 2)
    model.reset(2)
    with pytest.raises(load_module("clear_ops").ClearError):
        model.step(tokens[:, 0])  # three lanes for two states
