"""CPU-side checks of libfhe_ssm_clear.so: it exports what include/fhe_ssm_clear.h declares, stands without the engine and
the oracle, and refuses what a host can see to be wrong before anything reaches a GPU (there is none here)."""
import ctypes
import os
import re
import subprocess

import numpy as np
import pytest

from conftest import REPO
from engine_loader import load_module

def clear():
    ops = load_module("clear_ops")
    return ops, ops.load()


def declared():
    text = open(os.path.join(REPO, "include", "fhe_ssm_clear.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    return sorted(set(re.findall(r"\b(fhe_ssm_\w+)\s*\(", text)))


def test_library_exports_its_header():
    ops, _ = clear()
    out = subprocess.run(["nm", "-D", "--defined-only", ops.LIB_PATH], capture_output=True, text=True).stdout
    assert set(declared()) == set(ops.SIGNATURES)
    assert set(declared()) <= set(re.findall(r"\bT (fhe_ssm_\w+)", out))


def test_library_needs_neither_engine_nor_oracle():
    ops, _ = clear()
    ldd = subprocess.run(["ldd", ops.LIB_PATH], capture_output=True, text=True).stdout
    assert "libckks_hip" not in ldd and "liboracle" not in ldd
    undefined = subprocess.run(["nm", "-D", "--undefined-only", ops.LIB_PATH], capture_output=True, text=True).stdout
    assert not re.search(r"\b(ckks_|rocblas|hipblas|miopen)", undefined)


def refused(lib, rc, words):
    assert rc != 0
    assert words in lib.fhe_ssm_clear_last_error().decode(), lib.fhe_ssm_clear_last_error()


def attention_sizes(ops, **change):
    a = ops.LinearAttentionSizes(ops.BF16, 2, 3, 4, 2, 1, 64, 64, 1.0)
    for name, value in change.items():
        setattr(a, name, value)
    return ctypes.byref(a)


@pytest.mark.parametrize("change, words", [
    (dict(type=3), "unknown type"), (dict(dk=0), "dk 0"), (dict(dk=129), "dk 129"), (dict(dv=0), "at least 1"),
    (dict(heads=0), "at least 1"), (dict(q_heads=3), "cannot share"), (dict(k_heads=0), "cannot share"),
    (dict(lanes=1 << 31), "too many"), (dict(tokens=(1 << 24) + 1), "too many")])
def test_attention_refusals(change, words):
    ops, lib = clear()
    n = ctypes.c_size_t()
    a = attention_sizes(ops, **change)
    refused(lib, lib.fhe_ssm_linear_attention_workspace(a, ctypes.byref(n)), words)
    refused(lib, lib.fhe_ssm_linear_attention_prompt(a, None, None, None, None, None, None, None, None, None, 0, None),
            words)


def test_attention_refuses_null_and_long_steps():
    ops, lib = clear()
    refused(lib, lib.fhe_ssm_linear_attention_workspace(None, None), "null")
    refused(lib, lib.fhe_ssm_linear_attention_prompt(attention_sizes(ops), None, None, None, None, None, None, None, None,
                                                     None, 0, None), "null")
    refused(lib, lib.fhe_ssm_linear_attention_step(attention_sizes(ops), None, None, None, None, None, None, None, None),
            "one token")
    # no lanes: nothing to do, and nothing that a pointer is needed for
    assert lib.fhe_ssm_linear_attention_prompt(attention_sizes(ops, lanes=0), None, None, None, None, None, None, None,
                                               None, None, 0, None) == 0


@pytest.mark.parametrize("sizes, words", [
    ((0, 64, 32, 0, 0), "matrix of"), ((64, 0, 32, 0, 0), "matrix of"), ((64, 64, 48, 0, 0), "group 48"),
    ((64, 64, 0, 0, 0), "group 0"), ((64, 64, 96, 0, 0), "group 96"), ((64, 64, 32, 3, 0), "type of scales"),
    ((0x7fffff00, 0x7fffff00, 128, 0, 0), "too large")])
def test_q4_refusals(sizes, words):
    ops, lib = clear()
    n = ctypes.c_size_t()
    m = ctypes.byref(ops.Q4Sizes(*sizes))
    refused(lib, lib.fhe_ssm_q4_bytes(m, ctypes.byref(n)), words)
    refused(lib, lib.fhe_ssm_q4_arrange(m, 256, 512, 256, None, 256, None), words)
    refused(lib, lib.fhe_ssm_q4_product(m, 256, 0, 1, 256, 64, 256, 64, None), words)


def test_q4_refuses_pointers_and_strides():
    ops, lib = clear()
    m = ctypes.byref(ops.Q4Sizes(64, 65, 32, ops.F16, 0))
    refused(lib, lib.fhe_ssm_q4_arrange(m, None, 33, 256, None, 256, None), "null")
    refused(lib, lib.fhe_ssm_q4_arrange(m, 256, 33, 256, 256, 256, None), "zero points")
    refused(lib, lib.fhe_ssm_q4_arrange(m, 256, 32, 256, None, 256, None), "overlap")
    refused(lib, lib.fhe_ssm_q4_arrange(m, 256, 33, 256, None, 260, None), "256 bytes")
    refused(lib, lib.fhe_ssm_q4_product(m, 256, 3, 1, 256, 65, 256, 64, None), "unknown type")
    refused(lib, lib.fhe_ssm_q4_product(m, 260, 0, 1, 256, 65, 256, 64, None), "256 bytes")
    refused(lib, lib.fhe_ssm_q4_product(m, 256, 0, 2, 256, 65, 256, 63, None), "overlap")
    refused(lib, lib.fhe_ssm_q4_product(m, 256, 0, 1, None, 65, 256, 64, None), "null")
    assert lib.fhe_ssm_q4_product(m, 256, 0, 0, None, 65, None, 64, None) == 0  # no rows


@pytest.mark.parametrize("args, words", [
    ((3, 256, 1, 10, 10), "unknown type"), ((0, 256, 1, 0, 10), "vocabulary of 0"),
    ((0, 256, 1, (1 << 18) + 1, 10), "vocabulary"), ((0, None, 1, 10, 10), "null"), ((0, 256, 1, 10, -1), "negative"),
    ((0, 256, 1 << 31, 10, 10), "too many")])
def test_sample_refusals(args, words):
    ops, lib = clear()
    p = ctypes.byref(ops.SampleParams())
    refused(lib, lib.fhe_ssm_sample(*args, 256, p, 256, None, None), words)


def test_python_refuses_tensors_that_are_not_on_the_gpu():
    torch = pytest.importorskip("torch")
    ops, _ = clear()
    x = torch.zeros(1, 2, 3, 4)
    with pytest.raises(ops.ClearError, match="on the GPU"):
        ops.linear_attention_prompt(x, x, x, torch.zeros(3), None, None, x)
    with pytest.raises(ops.ClearError, match="on the GPU"):
        ops.Q4Matrix(torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(4, 1))
    with pytest.raises(ops.ClearError, match="on the GPU"):
        ops.sample(torch.zeros(2, 5), torch.zeros(2), torch.zeros(2, dtype=torch.int64))


def unpacked(codes, n_in):
    c = np.stack((codes & 15, codes >> 4), -1).reshape(codes.shape[0], -1)
    return c[:, :n_in].astype(np.float64)


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("shape, group", [((3, 64), 32), ((5, 101), 32), ((2, 128), 64), ((4, 300), 128), ((1, 1), 32)])
def test_quantize_q4_is_near_the_matrix(shape, group, zeros):
    """A code is at most half a step off inside the range that its group's scale spans.  The scale is rounded to float16
    (2^-11 of it, at most 15 steps of it in a code), which moves the range's end by up to 15 2^-11 of a step, and a zero point
    is rounded to a whole step (half a step more, at the clipped end)."""
    ops, _ = clear()
    w = np.random.default_rng(3).standard_normal(shape).astype(np.float32)
    codes, scales, zero = ops.quantize_q4(w, group, zeros)
    groups = -(-shape[1] // group)
    assert codes.shape == (shape[0], (shape[1] + 1) // 2) and scales.shape == (shape[0], groups)
    s = np.repeat(scales.astype(np.float64), group, 1)[:, :shape[1]]
    z = np.repeat(zero.astype(np.float64), group, 1)[:, :shape[1]] if zeros else 8.0
    off = np.abs((unpacked(codes, shape[1]) - z) * s - w) / s
    assert off.max() <= (1.0 if zeros else 0.5) + 16 * 2.0**-11


def test_quantize_q4_of_a_zero_matrix():
    ops, _ = clear()
    codes, scales, _ = ops.quantize_q4(np.zeros((2, 40), np.float32), 32)
    assert (codes == 0x88).all() and np.isfinite(scales.astype(np.float32)).all() and (scales > 0).all()


def test_sizes_that_pass_32_bits_are_refused():
    """counts of workgroups and groups near 2^32, which must not wrap around"""
    ops, lib = clear()
    n = ctypes.c_size_t()
    for change in (dict(dv=0xffffffff), dict(dv=0xffffffe1), dict(lanes=1 << 22, heads=8, q_heads=2, k_heads=2)):
        refused(lib, lib.fhe_ssm_linear_attention_workspace(attention_sizes(ops, **change), ctypes.byref(n)), "too many")
    refused(lib, lib.fhe_ssm_q4_bytes(ctypes.byref(ops.Q4Sizes(1 << 20, 1 << 19, 128, 0, 0)), ctypes.byref(n)), "too large")
    # a group far longer than a row: one group a row
    one, far = ctypes.c_size_t(), ctypes.c_size_t()
    assert lib.fhe_ssm_q4_bytes(ctypes.byref(ops.Q4Sizes(16, 256, 256, 0, 0)), ctypes.byref(one)) == 0
    assert lib.fhe_ssm_q4_bytes(ctypes.byref(ops.Q4Sizes(16, 256, 0xffffff80, 0, 0)), ctypes.byref(far)) == 0
    assert far.value == one.value
