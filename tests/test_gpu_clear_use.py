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
