"""CPU-side checks of what the operators that score and train refuse, from Python and through the C ABI, before anything reaches a
GPU (there is none here), of what they must not refuse, and of the streams that their calls go to."""
import ctypes

import pytest

from test_clear_abi import clear, refused
from test_clear_streams import CURRENT, on_gpu

torch = pytest.importorskip("torch")

F = 256  # an address that nothing reads


@pytest.fixture
def library(monkeypatch):
    """clear_ops over a library that answers questions of sizes by 4,096 bytes, and else only notes the stream, its last argument"""
    ops, _ = clear()

    class Library:
        streams = []

        def __getattr__(self, name):
            def call(*args):
                if name.endswith("workspace"):
                    for a in args[1:]:
                        if a is not None:
                            a._obj.value = 4096
                else:
                    self.streams.append(args[-1])
                return 0
            return call

    monkeypatch.setattr(ops, "_lib", Library())
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: CURRENT, raising=False)
    return ops


def sizes(ops, kind, **change):
    a = {"norm": lambda: ops.LayerNormSizes(ops.BF16, ops.F32, 4, 64, 1e-5, 64, 64, 64),
         "recurrence": lambda: ops.GatedRecurrenceSizes(ops.BF16, 2, 5, 64, *[(320, 64)] * 6),
         "embedding": lambda: ops.EmbeddingSizes(ops.F32, ops.F32, 7, 100, 64, 1.0, 64, 64),
         "logprobs": lambda: ops.TokenLogprobsSizes(ops.F32, 4, 1000, 5, 1000, 1000),
         "adamw": lambda: ops.AdamWSizes(ops.F32, ops.BF16, 32, 1, 0, 1e-3, 1e-8, 0.9, 0.99)}[kind]()
    for name, value in change.items():
        setattr(a, name, value)
    return ctypes.byref(a)


@pytest.mark.parametrize("change, words", [
    (dict(type=3), "unknown type"), (dict(weight_type=2), "weights of type"), (dict(channels=0), "0 channels"),
    (dict(channels=16385), "16385 channels"), (dict(rows=1 << 31), "too many rows"), (dict(out_stride=63), "overlap"),
    (dict(x_stride=-64), "negative stride"), (dict(dy_stride=-1), "negative stride"), (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps")])
def test_layer_norm_refusals(change, words):
    ops, lib = clear()
    a, n = sizes(ops, "norm", **change), ctypes.c_size_t()
    refused(lib, lib.fhe_ssm_layer_norm_workspace(a, ctypes.byref(n)), words)
    refused(lib, lib.fhe_ssm_layer_norm_forward(a, F, None, None, F, None, None, None), words)
    refused(lib, lib.fhe_ssm_layer_norm_backward(a, F, F, None, F, F, F, None, None, None, 0, None), words)


def test_layer_norm_refuses_null_and_small_workspaces():
    ops, lib = clear()
    a, n = sizes(ops, "norm", rows=5000), ctypes.c_size_t()
    refused(lib, lib.fhe_ssm_layer_norm_workspace(None, None), "null")
    refused(lib, lib.fhe_ssm_layer_norm_workspace(a, None), "null")
    assert lib.fhe_ssm_layer_norm_workspace(a, ctypes.byref(n)) == 0 and n.value > 0
    refused(lib, lib.fhe_ssm_layer_norm_forward(a, None, None, None, F, None, None, None), "null")
    refused(lib, lib.fhe_ssm_layer_norm_backward(a, F, F, None, None, F, F, None, None, None, 0, None), "null")
    for address, size in ((None, n.value), (F, n.value - 1), (F + 8, n.value)):
        refused(lib, lib.fhe_ssm_layer_norm_backward(a, F, F, None, F, F, F, F, None, address, size, None), "workspace")
    assert lib.fhe_ssm_layer_norm_forward(sizes(ops, "norm", rows=0), None, None, None, None, None, None, None) == 0


@pytest.mark.parametrize("change, words", [
    (dict(type=3), "unknown type"), (dict(channels=0), "no channels"), (dict(tokens=(1 << 24) + 1), "too many"),
    (dict(channels=(1 << 24) + 1), "too many"), (dict(lanes=1 << 23), "too many"), (dict(lanes=1 << 18, channels=1 << 11), "too many"),
    (dict(lanes=0xffffffff, channels=1 << 24), "too many")])
def test_gated_recurrence_refusals(change, words):
    ops, lib = clear()
    a, n = sizes(ops, "recurrence", **change), ctypes.c_size_t()
    refused(lib, lib.fhe_ssm_gated_recurrence_workspace(a, ctypes.byref(n), None), words)
    refused(lib, lib.fhe_ssm_gated_recurrence_prompt(a, F, F, None, None, None, F, None, None, 0, None), words)
    refused(lib, lib.fhe_ssm_gated_recurrence_backward(a, F, F, None, F, F, None, F, F, None, None, 0, None), words)


@pytest.mark.parametrize("stride", [(320, 63), (64, 64), (0, 64), (320, 0), (320, -64), (63, 126), (319, 64)])
def test_gated_recurrence_refuses_output_rows_that_overlap(stride):
    ops, lib = clear()
    refused(lib, lib.fhe_ssm_gated_recurrence_prompt(sizes(ops, "recurrence", out_stride=stride), F, F, None, None, None, F, None, None, 0, None), "overlap")
    for name in ("dz_stride", "dx_stride"):
        refused(lib, lib.fhe_ssm_gated_recurrence_backward(sizes(ops, "recurrence", **{name: stride}), F, F, None, F, F, None, F, F, None, None, 0, None), "overlap")
    refused(lib, lib.fhe_ssm_gated_recurrence_step(sizes(ops, "recurrence", tokens=1, out_stride=(63, 0)), F, F, None, None, F, None), "overlap")


def test_gated_recurrence_refuses_null_long_steps_and_small_workspaces():
    ops, lib = clear()
    a = sizes(ops, "recurrence")
    refused(lib, lib.fhe_ssm_gated_recurrence_workspace(None, None, None), "null")
    refused(lib, lib.fhe_ssm_gated_recurrence_prompt(a, None, F, None, None, None, F, None, None, 0, None), "null")
    refused(lib, lib.fhe_ssm_gated_recurrence_backward(a, F, F, None, None, F, None, F, F, None, None, 0, None), "null")
    refused(lib, lib.fhe_ssm_gated_recurrence_step(a, F, F, None, None, F, None), "one token")
    refused(lib, lib.fhe_ssm_gated_recurrence_step(sizes(ops, "recurrence", tokens=1), F, None, None, None, F, None), "null")
    a, work, saved = sizes(ops, "recurrence", tokens=4000, out_stride=(256000, 64)), ctypes.c_size_t(), ctypes.c_size_t()
    assert lib.fhe_ssm_gated_recurrence_workspace(a, ctypes.byref(work), ctypes.byref(saved)) == 0
    assert work.value > 0 and saved.value >= 4000 // 128 * 2 * 64 * 4
    for address, size in ((None, work.value), (F, work.value - 1), (F + 4, work.value)):
        refused(lib, lib.fhe_ssm_gated_recurrence_prompt(a, F, F, None, None, None, F, None, address, size, None), "workspace")
    assert lib.fhe_ssm_gated_recurrence_prompt(sizes(ops, "recurrence", lanes=0), None, None, None, None, None, None, None, None, 0, None) == 0


@pytest.mark.parametrize("change, words", [
    (dict(table_type=3), "unknown type"), (dict(row_type=9), "unknown type"), (dict(vocab=0), "vocabulary of 0"),
    (dict(vocab=(1 << 18) + 1), "vocabulary"), (dict(channels=0), "0 channels"), (dict(channels=(1 << 20) + 1), "channels"),
    (dict(tokens=(1 << 26) + 1), "too many")])
def test_embedding_refusals(change, words):
    ops, lib = clear()
    a, n = sizes(ops, "embedding", **change), ctypes.c_size_t()
    refused(lib, lib.fhe_ssm_embedding_workspace(a, ctypes.byref(n)), words)
    refused(lib, lib.fhe_ssm_embedding_lookup(a, F, F, F, None), words)
    refused(lib, lib.fhe_ssm_embedding_gradient(a, F, F, F, 0, None, 0, None), words)


def test_embedding_refuses_null_strides_and_small_workspaces():
    ops, lib = clear()
    a, n = sizes(ops, "embedding", tokens=5000), ctypes.c_size_t()
    refused(lib, lib.fhe_ssm_embedding_lookup(a, None, F, F, None), "null")
    refused(lib, lib.fhe_ssm_embedding_lookup(sizes(ops, "embedding", table_stride=63), F, F, F, None), "overlap")
    refused(lib, lib.fhe_ssm_embedding_lookup(sizes(ops, "embedding", row_stride=63), F, F, F, None), "overlap")
    refused(lib, lib.fhe_ssm_embedding_gradient(a, F, None, F, 0, None, 0, None), "null")
    refused(lib, lib.fhe_ssm_embedding_gradient(sizes(ops, "embedding", table_type=1, row_type=2), F, F, F, 0, None, 0, None), "float32 or of the rows")
    refused(lib, lib.fhe_ssm_embedding_gradient(sizes(ops, "embedding", row_stride=-1), F, F, F, 0, None, 0, None), "negative")
    refused(lib, lib.fhe_ssm_embedding_gradient(sizes(ops, "embedding"), F, F, F + 2, 0, None, 0, None), "between elements")
    assert lib.fhe_ssm_embedding_workspace(a, ctypes.byref(n)) == 0 and n.value > 0
    for address, size in ((None, n.value), (F, n.value - 1), (F + 8, n.value)):
        refused(lib, lib.fhe_ssm_embedding_gradient(a, F, F, F, 0, address, size, None), "workspace")
    none = sizes(ops, "embedding", tokens=0)
    assert lib.fhe_ssm_embedding_lookup(none, None, None, None, None) == 0
    assert lib.fhe_ssm_embedding_gradient(none, None, None, F, 1, None, 0, None) == 0  # nothing to add


@pytest.mark.parametrize("change, words", [
    (dict(type=3), "unknown type"), (dict(vocab=0), "vocabulary of 0"), (dict(vocab=(1 << 18) + 1), "vocabulary"),
    (dict(top=33), "33 alternatives"), (dict(rows=1 << 22), "too many"), (dict(row_stride=-1), "negative")])
def test_token_logprobs_refusals(change, words):
    ops, lib = clear()
    a, n = sizes(ops, "logprobs", **change), ctypes.c_size_t()
    refused(lib, lib.fhe_ssm_token_logprobs_workspace(a, ctypes.byref(n)), words)
    refused(lib, lib.fhe_ssm_token_logprobs_forward(a, F, F, F, None, None, F, F, None, None, None, None, 0, None), words)
    refused(lib, lib.fhe_ssm_token_logprobs_gradient(a, F, F, F, None, F, None, F, None), words)


def test_token_logprobs_refuses_null_strides_and_small_workspaces():
    ops, lib = clear()
    a, n = sizes(ops, "logprobs"), ctypes.c_size_t()
    call = lib.fhe_ssm_token_logprobs_forward
    refused(lib, call(a, None, F, F, None, None, F, F, None, None, None, None, 0, None), "null")
    refused(lib, call(a, F, None, F, None, None, F, F, None, None, None, None, 0, None), "null")     # log-probabilities of no tokens
    refused(lib, call(a, F, F, F, None, None, F, None, None, None, None, None, 0, None), "null")     # alternatives by half
    refused(lib, call(a, F, None, None, None, None, F, F, F, None, F, None, 0, None), "null")        # weights of no tokens
    refused(lib, call(sizes(ops, "logprobs", gradient_stride=999), F, F, F, None, None, F, F, F, None, 2 * F, None, 0, None), "overlap")
    refused(lib, call(sizes(ops, "logprobs", gradient_stride=1001), F, F, F, None, None, F, F, F, None, F, None, 0, None), "their stride")
    refused(lib, lib.fhe_ssm_token_logprobs_gradient(a, F, F, None, None, F, None, F, None), "null")
    refused(lib, lib.fhe_ssm_token_logprobs_gradient(a, F, F, F, None, F, F, F, None), "null")       # an entropy's weight without it
    assert lib.fhe_ssm_token_logprobs_workspace(a, ctypes.byref(n)) == 0 and n.value == 0
    a = sizes(ops, "logprobs", vocab=60000, row_stride=60000)
    assert lib.fhe_ssm_token_logprobs_workspace(a, ctypes.byref(n)) == 0 and n.value > 0
    for address, size in ((None, n.value), (F, n.value - 1), (F + 8, n.value)):
        refused(lib, call(a, F, F, F, None, None, F, F, None, None, None, address, size, None), "workspace")
    assert call(sizes(ops, "logprobs", rows=0), None, None, None, None, None, None, None, None, None, None, None, 0, None) == 0


@pytest.mark.parametrize("change, words", [
    (dict(gradient_type=3), "type of gradients"), (dict(copy_type=0), "copies are"), (dict(state_bits=16), "16 bits"),
    (dict(beta1=1.0), "beta"), (dict(beta2=-0.1), "beta"), (dict(beta1=float("nan")), "beta"), (dict(eps=0.0), "eps"),
    (dict(step=0), "count from 1")])
def test_adamw_refusals(change, words):
    ops, lib = clear()
    t = ops.AdamWTensor(F, F, F, F, F, None, 10, 0.0)
    refused(lib, lib.fhe_ssm_adamw_step(sizes(ops, "adamw", **change), 1, ctypes.byref(t), None), words)


def test_adamw_refuses_null_and_large_tensors():
    ops, lib = clear()
    a = sizes(ops, "adamw")
    refused(lib, lib.fhe_ssm_adamw_step(None, 0, None, None), "null")
    refused(lib, lib.fhe_ssm_adamw_step(a, 1, None, None), "null")
    for i in range(4):
        fields = [F, F, F, F, None, None, 10, 0.0]
        fields[i] = None
        refused(lib, lib.fhe_ssm_adamw_step(a, 1, ctypes.byref(ops.AdamWTensor(*fields)), None), "null argument in tensor 0")
    refused(lib, lib.fhe_ssm_adamw_step(a, 1, ctypes.byref(ops.AdamWTensor(F, F, F, F, None, None, 1 << 32, 0.0)), None), "2^32")
    eight = sizes(ops, "adamw", state_bits=8)
    refused(lib, lib.fhe_ssm_adamw_step(eight, 1, ctypes.byref(ops.AdamWTensor(F, F, F, F, None, None, 10, 0.0)), None), "null")
    refused(lib, lib.fhe_ssm_adamw_step(eight, 1, ctypes.byref(ops.AdamWTensor(F, F, F, F, F + 1, None, 10, 0.0)), None), "odd address")
    assert lib.fhe_ssm_adamw_step(a, 0, None, None) == 0
    assert lib.fhe_ssm_adamw_step(a, 1, ctypes.byref(ops.AdamWTensor(None, None, None, None, None, None, 0, 0.0)), None) == 0


def test_python_refuses_tensors_that_are_not_on_the_gpu():
    ops, _ = clear()
    x, v = torch.zeros(2, 8), torch.zeros(2)
    calls = [lambda: ops.layer_norm(x, None, None, x), lambda: ops.layer_norm_backward(x, x, None, v, v, x),
             lambda: ops.gated_recurrence_step(x, x, x, x, x), lambda: ops.embedding(torch.zeros(2, dtype=torch.int64), x, x),
             lambda: ops.token_logprobs(x, None, None, v), lambda: ops.token_logprobs_gradient(x, None, x, None, x),
             lambda: ops.AdamW([x])]
    for call in calls:
        with pytest.raises(ops.ClearError, match="on the GPU"):
            call()


def test_python_refuses_shapes_types_and_strides(library):
    z = lambda *s, dtype=torch.float32: on_gpu(torch.zeros(s, dtype=dtype))  # noqa: E731
    x, v, ids = z(4, 8), z(4), z(4, dtype=torch.int64)
    p3 = z(2, 3, 8)
    saved = z(4096, dtype=torch.uint8)
    bad = [
        lambda: library.layer_norm(z(8), None, None, z(8)), lambda: library.layer_norm(x, z(7), None, x),
        lambda: library.layer_norm(x, z(8), z(8, dtype=torch.bfloat16), x), lambda: library.layer_norm(x, None, None, z(4, 8, dtype=torch.float16)),
        lambda: library.layer_norm(x.t(), None, None, x.t()), lambda: library.layer_norm(x, None, None, x, mean=z(5)),
        lambda: library.layer_norm(z(4, 8, dtype=torch.float64), None, None, x),
        lambda: library.layer_norm_backward(z(3, 8), x, None, v, v, x), lambda: library.layer_norm_backward(x, x, None, v, v, x, dweight=z(4)),
        lambda: library.layer_norm_backward(x, x, None, v, v, x, workspace=on_gpu(torch.zeros(1)).expand(4096)),
        lambda: library.gated_recurrence(p3, z(2, 3, 7), None, None, p3), lambda: library.gated_recurrence(p3, p3, z(2, 7), None, p3),
        lambda: library.gated_recurrence(p3, p3, None, None, p3, lengths=z(2, dtype=torch.int64)),
        lambda: library.gated_recurrence(p3, p3, None, None, p3, saved=saved[:8]), lambda: library.gated_recurrence(x, x, None, None, x),
        lambda: library.gated_recurrence_backward(p3, p3, None, p3, None, p3, p3),
        lambda: library.gated_recurrence_step(p3, p3, None, None, p3),
        lambda: library.embedding(v, x, x), lambda: library.embedding(ids, x, z(3, 8)), lambda: library.embedding(ids, x.t(), z(4, 4)),
        lambda: library.embedding_gradient(ids, x, z(8, 9).t()), lambda: library.embedding_gradient(ids, z(4, 7), x),
        lambda: library.token_logprobs(x, ids, z(3)), lambda: library.token_logprobs(x, ids[:3], v),
        lambda: library.token_logprobs(x, ids, v, top_tokens=z(4, 2, dtype=torch.int64)),
        lambda: library.token_logprobs(x, ids, v, top_tokens=z(4, 2), top_logprobs=z(4, 2)),
        lambda: library.token_logprobs(x, ids, v, statistics=v), lambda: library.token_logprobs(x, ids, v, gradient=z(4, 8, dtype=torch.float16)),
        lambda: library.token_logprobs_gradient(x, ids, v, v, x),
        lambda: library.AdamW([]), lambda: library.AdamW([z(4, dtype=torch.bfloat16)]), lambda: library.AdamW([x.t()]),
        lambda: library.AdamW([x], bits=4), lambda: library.AdamW([x], weight_decay=[0.1, 0.1]), lambda: library.AdamW([x], copies=[x]),
        lambda: library.AdamW([x], states=([x], [v])), lambda: library.AdamW([x], copies=[z(4, 8, dtype=torch.float16)] * 2),
    ]
    for i, call in enumerate(bad):
        try:
            call()
        except library.ClearError:
            continue
        raise AssertionError(f"call {i} is not refused")
    a = library.AdamW([x, v])
    for gradients in ([x], [x, z(5)], [x, z(4, dtype=torch.bfloat16)], [x.t().contiguous().t(), v], [torch.zeros(4, 8), v]):
        with pytest.raises(library.ClearError):
            a.step(gradients, lr=0.1, step=1)
    with pytest.raises(library.ClearError, match="lr must be"):
        a.step([x, v], lr=torch.zeros(1), step=1)
    with pytest.raises(library.ClearError, match="step must be"):
        a.step([x, v], lr=0.1, step=z(1))


def test_adamw_refuses_steps_before_the_first_and_tensors_with_other_memory(library):
    z = lambda *s, dtype=torch.float32: on_gpu(torch.zeros(s, dtype=dtype))  # noqa: E731
    for bits in (32, 8):
        p, c, g = z(4, 8), z(4, 8, dtype=torch.bfloat16), z(4, 8)
        a = library.AdamW([p], copies=[c], bits=bits)
        for step in (0, -1, 1 << 32):
            with pytest.raises(library.ClearError, match="steps count from 1"):
                a.step([g], lr=0.1, step=step)
        a.step([g], lr=0.1, step=(1 << 32) - 1)
        was, p.data = p.data, torch.zeros(4, 8)
        with pytest.raises(library.ClearError, match="other memory"):
            a.step([g], lr=0.1, step=1)
        p.data = was
        a.step([g], lr=0.1, step=1)
        c.data = torch.zeros(4, 8, dtype=torch.bfloat16)
        with pytest.raises(library.ClearError, match="other memory"):
            a.step([g], lr=0.1, step=1)
    assert len(library._lib.streams) == 4


def test_what_is_refused_once_is_refused_again_and_what_is_not_goes_through(library):
    x = on_gpu(torch.zeros(4, 8))
    for _ in range(2):
        with pytest.raises(library.ClearError):
            library.layer_norm(x, on_gpu(torch.zeros(7)), None, x)
        library.layer_norm(x, on_gpu(torch.zeros(8)), None, x)
        library.layer_norm(x[:, 1:4], None, None, x[:, 4:7])
        library.layer_norm(x[:1], None, None, x[3:])
        library.embedding(on_gpu(torch.zeros(2, dtype=torch.int64)), x[:1].expand(1, 8), on_gpu(torch.zeros(2, 8)))
    assert len(library._lib.streams) == 8


@pytest.mark.parametrize("stream", [{}, {"stream": 0}, {"stream": 0xabc0}])
def test_calls_go_to_the_current_stream_or_the_one_they_are_given(library, stream):
    z = lambda *s, dtype=torch.float32: on_gpu(torch.zeros(s, dtype=dtype))  # noqa: E731
    x, v, p3, ids, saved = z(4, 8), z(4), z(2, 3, 8), z(4, dtype=torch.int64), z(4096, dtype=torch.uint8)
    library.layer_norm(x, None, None, x, **stream)
    library.layer_norm_backward(x, x, None, v, v, x, **stream)
    library.gated_recurrence(p3, p3, None, None, p3, **stream)
    library.gated_recurrence_backward(p3, p3, saved, p3, None, p3, p3, **stream)
    library.gated_recurrence_step(x, x, None, None, x, **stream)
    library.embedding(ids, x, x, **stream)
    library.embedding_gradient(ids, x, x, **stream)
    library.token_logprobs(x, ids, v, **stream)
    library.token_logprobs_gradient(x, ids, z(4, 2), v, x, **stream)
    library.AdamW([x]).step([x], lr=0.1, step=1, **stream)
    assert library._lib.streams == [stream.get("stream", CURRENT)] * 10


def test_adamw_refuses_tensors_that_share_memory(library):
    """a parameter twice, parts of one another, states or copies of two parameters: what one entry's thread writes another reads"""
    z = lambda *s, dtype=torch.float32: on_gpu(torch.zeros(s, dtype=dtype))  # noqa: E731
    a, b, half, flat = z(8), z(8), z(8, dtype=torch.bfloat16), torch.zeros(20)
    bad = [
        lambda: library.AdamW([a, a]), lambda: library.AdamW([a, b, a], bits=8),
        lambda: library.AdamW([on_gpu(flat[:8]), on_gpu(flat[7:15])]), lambda: library.AdamW([on_gpu(flat), on_gpu(flat[:1])]),
        lambda: library.AdamW([a], states=([b], [b])), lambda: library.AdamW([a], states=([a], [b])),
        lambda: library.AdamW([a, b], states=([z(8)] * 2, [z(8), z(8)])), lambda: library.AdamW([a, b], copies=[half, half]),
        lambda: library.AdamW([a], copies=[on_gpu(a.view(torch.bfloat16)[:8])]),
    ]
    for i, call in enumerate(bad):
        try:
            call()
        except library.ClearError as e:
            assert "share memory" in str(e), i
            continue
        raise AssertionError(f"call {i} is not refused")
    library.AdamW([on_gpu(flat[:8]), on_gpu(flat[8:15]), on_gpu(flat[3:3])], bits=8, copies=[half, z(7, dtype=torch.bfloat16), half[:0]])
    library.AdamW([a]).step([a], lr=0.1, step=1)  # a gradient is only read, each entry by the thread that writes it
