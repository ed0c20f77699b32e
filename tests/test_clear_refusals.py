"""CPU-side checks of what the operators in the clear refuse, and of what they must not, from Python and through the C ABI."""
import pytest

from test_clear_abi import attention_sizes, clear, refused
from test_clear_streams import on_gpu, ops as library

torch = pytest.importorskip("torch")


def test_rows_that_are_no_matrix_are_refused(library):
    m = library.Q4Matrix(on_gpu(torch.zeros(8, 32, dtype=torch.uint8)), on_gpu(torch.zeros(8, 1)), group=64)
    for x, out in (((64,), (8,)), ((64,), (1, 8)), ((1, 64), (8,)), ((1, 1, 64), (1, 1, 8))):
        with pytest.raises(library.ClearError, match=r"\[rows, columns\]"):
            m.product(on_gpu(torch.zeros(x)), on_gpu(torch.zeros(out)))
    for shape in ((9,), (1, 1, 9), ()):
        with pytest.raises(library.ClearError, match=r"\[rows, vocab\]"):
            library.sample(on_gpu(torch.zeros(shape)), on_gpu(torch.zeros(1)), on_gpu(torch.zeros(1, dtype=torch.int64)))


def test_a_workspace_that_is_smaller_than_its_shape_is_refused(library):
    """an expanded tensor has many elements and little memory"""
    x, g = on_gpu(torch.zeros(1, 2, 3, 4)), on_gpu(torch.zeros(3))
    few = on_gpu(torch.zeros(1, dtype=torch.uint8)).expand(4096)
    with pytest.raises(library.ClearError, match="workspace must be contiguous"):
        library.linear_attention_prompt(x, x, x, g, None, None, x, workspace=few)


def test_rows_of_one_byte_have_any_stride_inside(library):
    library.Q4Matrix(on_gpu(torch.zeros(8, 40, dtype=torch.uint8))[:, 7:8], on_gpu(torch.zeros(8, 1)), group=32, in_features=2)
    library.Q4Matrix(on_gpu(torch.zeros(1, 8, dtype=torch.uint8).t()), on_gpu(torch.zeros(8, 1)), group=32, in_features=1)


@pytest.mark.parametrize("stride", [(0, 256, 64), (1024, 0, 64), (1024, 256, 0), (1024, 256, 63), (1024, -63, 64), (1, 256, 64)])
def test_rows_of_attention_outputs_that_overlap_are_refused(stride):
    """two workgroups would write one place; the other strides may share rows"""
    ops, lib = clear()
    a = attention_sizes(ops)
    a._obj.out_stride = stride
    refused(lib, lib.fhe_ssm_linear_attention_prompt(a, 256, 256, 256, 256, None, None, None, 256, None, 0, None), "overlap")
    a = attention_sizes(ops, tokens=1)
    a._obj.out_stride = (stride[0], 0, stride[2])
    if stride[0] >= 64 and stride[2] >= 64:  # a stride of the one token says nothing: what is refused is something else
        refused(lib, lib.fhe_ssm_linear_attention_step(a, None, 256, 256, 256, None, None, 256, None), "null")
    else:
        refused(lib, lib.fhe_ssm_linear_attention_step(a, 256, 256, 256, 256, None, None, 256, None), "overlap")
