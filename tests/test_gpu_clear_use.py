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
