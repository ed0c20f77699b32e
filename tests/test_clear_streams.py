"""CPU-side checks of the stream that a call from Python goes to: the one it is given, else torch's current one, as the tensors
that torch made on it may still be in the making, and may be handed on by its allocator, there and nowhere else."""
import pytest

from engine_loader import load_module

torch = pytest.importorskip("torch")

CURRENT = 0x5eed00


class OnGpu(torch.Tensor):
    """a tensor that says it is on the GPU"""
    is_cuda = True


def on_gpu(t):
    return t.as_subclass(OnGpu)


@pytest.fixture
def ops(monkeypatch):
    """clear_ops over a library that only notes the stream, its calls' last argument"""
    ops = load_module("clear_ops")

    class Library:
        streams = []

        def __getattr__(self, name):
            def call(*args):
                if name in ("fhe_ssm_q4_bytes", "fhe_ssm_linear_attention_workspace"):
                    args[1]._obj.value = 4096
                else:
                    self.streams.append(args[-1])
                return 0
            return call

    monkeypatch.setattr(ops, "_lib", Library())
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: CURRENT, raising=False)
    return ops


def calls(ops, **stream):
    """one call of every kind"""
    x, h = on_gpu(torch.zeros(1, 2, 3, 4)), on_gpu(torch.zeros(1, 3, 4))
    g, s = on_gpu(torch.zeros(3)), on_gpu(torch.zeros(1, 3, 4, 4))
    ops.linear_attention_prompt(x, x, x, g, None, s, x, workspace=on_gpu(torch.zeros(4096, dtype=torch.uint8)), **stream)
    ops.linear_attention_step(h, h, h, g, s, s, h, **stream)
    m = ops.Q4Matrix(on_gpu(torch.zeros(8, 32, dtype=torch.uint8)), on_gpu(torch.zeros(8, 1)), group=64, **stream)
    m.product(on_gpu(torch.zeros(2, 64)), on_gpu(torch.zeros(2, 8)), **stream)
    ops.sample(on_gpu(torch.zeros(2, 9)), on_gpu(torch.zeros(2)), on_gpu(torch.zeros(2, dtype=torch.int64)), **stream)
    return ops._lib.streams


def test_calls_go_to_torchs_current_stream(ops):
    assert calls(ops) == [CURRENT] * 5


@pytest.mark.parametrize("given", [0, 0xabc0])
def test_calls_go_to_the_stream_they_are_given(ops, given):
    assert calls(ops, stream=given) == [given] * 5


def test_the_drafting_model_lays_its_matrices_out_on_the_current_stream(ops, monkeypatch):
    draft = load_module("clear_draft")
    monkeypatch.setattr(torch.Tensor, "cuda", on_gpu)
    draft.matrix(load_module("clear_draft").np.random.default_rng(1), 4, 64)
    assert ops._lib.streams == [CURRENT]
