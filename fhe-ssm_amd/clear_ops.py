"""ctypes front end of libfhe_ssm_clear.so (include/fhe_ssm_clear.h): what a client of the encrypted step computes in the
clear -- linear attention with a decay for each head, products with 4-bit weights, the draw of a token.

Arguments are device tensors (torch's, or anything with data_ptr, dtype, shape and stride); outputs are tensors that the
caller brings.  Calls go to `stream` (a hipStream_t as an int, for torch `stream.cuda_stream`; 0 is the null stream; None is
torch's current stream, and the null stream for tensors that are not torch's) and return without waiting, so the tensors must
stay until that stream has passed them.  Shapes, types and strides are checked here and ClearError raised; there is no
fallback: if the library is missing, loading raises.
"""
from __future__ import annotations

import ctypes
import os
import sys

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libfhe_ssm_clear.so")

_vp = ctypes.c_void_p
_u32 = ctypes.c_uint32
_i64 = ctypes.c_int64
_int = ctypes.c_int
_size = ctypes.c_size_t

F32, BF16, F16 = 0, 1, 2


class LinearAttentionSizes(ctypes.Structure):
    """fhe_ssm_linear_attention"""
    _fields_ = [("type", _u32), ("lanes", _u32), ("tokens", _u32), ("heads", _u32), ("q_heads", _u32), ("k_heads", _u32),
                ("dk", _u32), ("dv", _u32), ("scale", ctypes.c_float), ("q_stride", _i64 * 3), ("k_stride", _i64 * 3),
                ("v_stride", _i64 * 3), ("decay_stride", _i64 * 3), ("out_stride", _i64 * 3)]


class Q4Sizes(ctypes.Structure):
    """fhe_ssm_q4_matrix"""
    _fields_ = [("out", _u32), ("in_", _u32), ("group", _u32), ("scale_type", _u32), ("has_zeros", _u32)]


class SampleParams(ctypes.Structure):
    """fhe_ssm_sample_params"""
    _fields_ = [("temperature", _vp), ("top_k", _vp), ("top_p", _vp), ("min_p", _vp)]


# name -> (restype, argtypes); the exported C ABI (kept in step with include/fhe_ssm_clear.h)
SIGNATURES = {
    "fhe_ssm_clear_last_error": (ctypes.c_char_p, []),
    "fhe_ssm_linear_attention_workspace": (_int, [_vp, ctypes.POINTER(_size)]),
    "fhe_ssm_linear_attention_prompt": (_int, [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _size, _vp]),
    "fhe_ssm_linear_attention_step": (_int, [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp]),
    "fhe_ssm_q4_bytes": (_int, [_vp, ctypes.POINTER(_size)]),
    "fhe_ssm_q4_arrange": (_int, [_vp, _vp, _i64, _vp, _vp, _vp, _vp]),
    "fhe_ssm_q4_product": (_int, [_vp, _vp, _u32, _u32, _vp, _i64, _vp, _i64, _vp]),
    "fhe_ssm_sample": (_int, [_u32, _vp, _u32, _u32, _i64, _vp, _vp, _vp, _vp, _vp]),
}


class ClearError(RuntimeError):
    pass


_lib = None


def load(path: str = LIB_PATH):
    """Load the library (raises if it was not built)."""
    global _lib
    if _lib is None:
        if not os.path.exists(path):
            raise ClearError(f"{path} is missing: build it with __graft_entry__.build() (make -C fhe-ssm_amd)")
        lib = ctypes.CDLL(path)
        for name, (res, args) in SIGNATURES.items():
            f = getattr(lib, name)
            f.restype = res
            f.argtypes = args
        _lib = lib
    return _lib


def check(rc: int) -> None:
    if rc:
        raise ClearError(f"clear error {rc}: {load().fhe_ssm_clear_last_error().decode()}")


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ClearError(what)


_TYPE_NAMES = {"torch.float32": F32, "torch.bfloat16": BF16, "torch.float16": F16}
_types: dict = {}


def _type(t) -> int:
    """the code of a tensor's element type"""
    code = _types.get(t.dtype)
    if code is None:
        code = _TYPE_NAMES.get(str(t.dtype))
        _need(code is not None, f"element type {t.dtype} is none of float32, bfloat16, float16")
        _types[t.dtype] = code
    return code


_names: dict = {}


def _is(t, dtype: str) -> bool:
    name = _names.get(t.dtype)
    if name is None:
        name = _names[t.dtype] = str(t.dtype)
    return name == dtype


def _on_device(*tensors) -> None:
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise ClearError("tensors must be on the GPU")


def _queue(stream, t):
    """the stream of a call on tensor t"""
    if stream is not None:
        return stream
    torch = sys.modules.get("torch")
    if torch is None or not isinstance(t, torch.Tensor):
        return None
    return torch._C._cuda_getCurrentRawStream(t.get_device())  # current_stream() makes an object a call


def _ptr(t):
    return None if t is None else t.data_ptr()


# ------------------------------------------------------------------------------------------------ linear attention
_attention: dict = {}  # sizes, types and strides of a call -> its checked description


def _rows(t, name: str, tokens_axis: bool):
    """(lane, token, head) strides of a [lanes, (tokens,) heads, channels] tensor"""
    s = t.stride()
    _need(t.shape[-1] <= 1 or s[-1] == 1, f"{name}: channels must be contiguous")
    return (s[0], s[1], s[2]) if tokens_axis else (s[0], 0, s[1])


def _describe(q, k, v, g, state_in, state_out, out, scale, tokens_axis):
    n = 4 if tokens_axis else 3
    _need(len(q.shape) == len(k.shape) == len(v.shape) == n,
          "q, k and v are [lanes, tokens, heads, channels], of one token [lanes, heads, channels]")
    lead = tuple(v.shape[:-2])
    heads, dv = v.shape[-2:]
    q_heads, dk = q.shape[-2:]
    k_heads = k.shape[-2]
    _need(tuple(q.shape[:-2]) == lead and tuple(k.shape[:-2]) == lead and k.shape[-1] == dk,
          "q, k and v differ in lanes or tokens, or q and k in channels")
    _need(_type(q) == _type(k) == _type(v), "q, k and v differ in type")
    _need(q_heads >= 1 and k_heads >= 1 and heads % q_heads == 0 and heads % k_heads == 0,
          f"{heads} heads cannot share {q_heads} query and {k_heads} key heads")
    lanes, tokens = lead[0], lead[1] if tokens_axis else 1
    a = LinearAttentionSizes(_type(v), lanes, tokens, heads, q_heads, k_heads, dk, dv, scale)
    a.q_stride, a.k_stride, a.v_stride = _rows(q, "q", tokens_axis), _rows(k, "k", tokens_axis), _rows(v, "v", tokens_axis)
    if g is not None:  # None: only the workspace is asked for
        _need(_is(g, "torch.float32"), "log_decay must be float32")
        if len(g.shape) == 1:  # one decay per head, the same at every token
            _need(g.shape[0] == heads, "log_decay has one entry per head")
            a.decay_stride = (0, 0, g.stride()[0])
        else:
            _need(tuple(g.shape) == lead + (heads,), "log_decay is [heads] or [lanes, tokens, heads]")
            s = g.stride()
            a.decay_stride = (s[0], s[1], s[2]) if tokens_axis else (s[0], 0, s[1])
        _need(_type(out) == _type(v) and out.shape == v.shape, "out must be like v")
        a.out_stride = _rows(out, "out", tokens_axis)
        for name, s in (("state_in", state_in), ("state_out", state_out)):
            _need(s is None or (tuple(s.shape) == (lanes, heads, dk, dv) and _is(s, "torch.float32") and s.is_contiguous()),
                  f"{name} must be contiguous float32 [lanes, heads, dk, dv]")
    return a, ctypes.addressof(a)


def _described(q, k, v, g, state_in, state_out, out, scale, tokens_axis):
    key = (q.dtype, q.shape, q.stride(), k.dtype, k.shape, k.stride(), v.dtype, v.shape, v.stride(), scale, tokens_axis)
    if g is not None:
        key += (g.dtype, g.shape, g.stride(), out.dtype, out.shape, out.stride(),
                state_in is not None and (state_in.dtype, state_in.shape, state_in.stride()),
                state_out is not None and (state_out.dtype, state_out.shape, state_out.stride()))
    a = _attention.get(key)
    if a is None:
        if len(_attention) >= 256:
            _attention.clear()
        a = _attention[key] = _describe(q, k, v, g, state_in, state_out, out, scale, tokens_axis)
    return a  # the description, which its caller holds while it is used, and its address


def linear_attention_workspace(q, k, v) -> int:
    """device bytes that linear_attention_prompt needs for tensors of these shapes (0 for many)"""
    n = _size()
    a = _described(q, k, v, None, None, None, None, 1.0, True)
    check(load().fhe_ssm_linear_attention_workspace(a[1], ctypes.byref(n)))
    return n.value


def linear_attention_prompt(q, k, v, log_decay, state_in, state_out, out, scale: float = 1.0, lengths=None,
                            workspace=None, stream=None) -> None:
    """S_t = exp(log_decay_t) S_{t-1} + k_t v_t^T and out_t = scale q_t S_t over a prompt, per lane and head.

    q [lanes, tokens, query heads, dk], k [lanes, tokens, key heads, dk], v and out [lanes, tokens, heads, dv]; log_decay
    float32 [lanes, tokens, heads] or [heads]; states float32 [lanes, heads, dk, dv] (state_in None: zero; state_out None:
    not kept; both may be one tensor); lengths int32 [lanes]: tokens past a lane's length change nothing and give zeros;
    workspace: a uint8 tensor of linear_attention_workspace(q, k, v) bytes, None where that is 0."""
    _on_device(q, k, v, log_decay, state_in, state_out, out, lengths, workspace)
    if lengths is not None:
        _need(_is(lengths, "torch.int32") and tuple(lengths.shape) == (v.shape[0],) and lengths.is_contiguous(),
              "lengths must be contiguous int32 [lanes]")
    _need(workspace is None or workspace.is_contiguous(), "workspace must be contiguous")
    a = _described(q, k, v, log_decay, state_in, state_out, out, scale, True)
    check(load().fhe_ssm_linear_attention_prompt(
        a[1], q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(), _ptr(lengths), _ptr(state_in), _ptr(state_out),
        out.data_ptr(), _ptr(workspace), 0 if workspace is None else workspace.numel() * workspace.element_size(),
        _queue(stream, v)))


def linear_attention_step(q, k, v, log_decay, state_in, state_out, out, scale: float = 1.0, stream=None) -> None:
    """linear_attention_prompt for one token of every lane: the same tensors without the token axis"""
    _on_device(q, k, v, log_decay, state_in, state_out, out)
    a = _described(q, k, v, log_decay, state_in, state_out, out, scale, False)
    check(load().fhe_ssm_linear_attention_step(a[1], q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(),
                                               _ptr(state_in), _ptr(state_out), out.data_ptr(), _queue(stream, v)))


# ------------------------------------------------------------------------------------------------ 4-bit products
def quantize_q4(w: np.ndarray, group: int, zeros: bool = False):
    """A float matrix [out, in] as 4-bit codes with float16 scales, rounded to nearest: (codes uint8 [out, ceil(in / 2)],
    scales float16 [out, groups], zero points uint8 [out, groups] or None).  A group is the weights' range mapped to the
    codes 0..15 (zeros) or its largest magnitude to 7 steps either side of 8 (no zeros); the last group may be short."""
    w = np.asarray(w, dtype=np.float32)
    out, n_in = w.shape
    groups = -(-n_in // group)
    padded = np.full((out, groups * group), np.nan, dtype=np.float32)
    padded[:, :n_in] = w
    parts = padded.reshape(out, groups, group)
    if zeros:
        low, high = np.minimum(np.nanmin(parts, -1), 0), np.maximum(np.nanmax(parts, -1), 0)
        scales = np.maximum((high - low) / 15, 2.0**-24).astype(np.float16)
        zero = np.clip(np.rint(-low / scales.astype(np.float32)), 0, 15)
    else:
        scales = np.maximum(np.nanmax(np.abs(parts), -1) / 7, 2.0**-24).astype(np.float16)
        zero = np.full((out, groups), 8.0)
    codes = np.rint(np.nan_to_num(parts) / scales.astype(np.float32)[..., None]) + zero[..., None]
    codes = np.clip(codes, 0, 15).astype(np.uint8).reshape(out, -1)[:, :n_in]
    codes = np.pad(codes, ((0, 0), (0, n_in % 2)))
    return codes[:, 0::2] | (codes[:, 1::2] << 4), scales, zero.astype(np.uint8) if zeros else None


class Q4Matrix:
    """A matrix [out, in_features] of 4-bit weights, laid out once on the GPU for products with rows.

    codes: uint8 [out, ceil(in_features / 2)], two codes in a byte, the lower index in the low four bits; scales: float32,
    bfloat16 or float16 [out, groups]; zeros: uint8 [out, groups], or None: 8 throughout.  group: 32, 64 or a multiple of
    128.  None of the three is needed after the layout has run on the stream."""

    def __init__(self, codes, scales, zeros=None, in_features: int | None = None, group: int = 64, stream=None):
        _on_device(codes, scales, zeros)
        _need(_is(codes, "torch.uint8") and len(codes.shape) == 2 and (codes.stride()[1] == 1 or codes.shape[1] == 1),
              "codes must be uint8 rows")
        out, row = codes.shape
        n_in = 2 * row if in_features is None else in_features
        _need((n_in + 1) // 2 == row, f"rows of {row} bytes do not hold {n_in} codes")
        m = self.sizes = Q4Sizes(out, n_in, group, _type(scales), zeros is not None)
        n = _size()
        check(load().fhe_ssm_q4_bytes(ctypes.byref(m), ctypes.byref(n)))
        groups = -(-n_in // group)
        for name, t in (("scales", scales), ("zeros", zeros)):
            _need(t is None or (tuple(t.shape) == (out, groups) and t.is_contiguous()),
                  f"{name} must be contiguous [{out}, {groups}]")
        _need(zeros is None or _is(zeros, "torch.uint8"), "zeros must be uint8")
        self.weights = codes.new_empty((n.value + 255,))  # the layout starts on 256 bytes
        self._at = -(-self.weights.data_ptr() // 256) * 256
        self.out_features, self.in_features, self._m = out, n_in, ctypes.addressof(m)
        check(load().fhe_ssm_q4_arrange(self._m, codes.data_ptr(), codes.stride()[0], scales.data_ptr(), _ptr(zeros),
                                        self._at, _queue(stream, codes)))

    def product(self, x, out, stream=None) -> None:
        """out[r] = matrix times x[r] for rows x [rows, in_features], out [rows, out_features] of one type"""
        _on_device(x, out)
        _need(len(x.shape) == len(out.shape) == 2, "x and out are [rows, columns]")
        kind = _type(x)
        rows, n_in = x.shape
        (xs, x1), (ys, y1) = x.stride(), out.stride()
        _need(kind == _type(out) and n_in == self.in_features and tuple(out.shape) == (rows, self.out_features),
              f"x must be [rows, {self.in_features}] and out [rows, {self.out_features}], of one type")
        _need((x1 == 1 or n_in == 1) and (y1 == 1 or self.out_features == 1), "rows must be contiguous")
        check(load().fhe_ssm_q4_product(self._m, self._at, kind, rows, x.data_ptr(), xs, out.data_ptr(), ys,
                                          _queue(stream, x)))


# ------------------------------------------------------------------------------------------------ sampling
def sample(logits, draws, tokens, logprobs=None, temperature=None, top_k=None, top_p=None, min_p=None, stream=None) -> None:
    """Draws a token for every row of logits [rows, vocab] with the given random numbers draws in [0, 1).

    tokens: int64 [rows]; logprobs: float32 [rows] or None, the log-probability among what the filters keep.  temperature,
    top_p, min_p: float32 [rows]; top_k: int32 [rows]; None turns a filter off (temperature: 1).  What they keep, and which
    token a number draws, is defined in include/fhe_ssm_clear.h."""
    _on_device(logits, draws, tokens, logprobs, temperature, top_k, top_p, min_p)
    _need(len(logits.shape) == 2, "logits are [rows, vocab]")
    rows, vocab = logits.shape
    stride = logits.stride()
    _need(vocab == 1 or stride[1] == 1, "rows of logits must be contiguous")
    for name, t, dtype in (("draws", draws, "torch.float32"), ("tokens", tokens, "torch.int64"),
                           ("logprobs", logprobs, "torch.float32"), ("temperature", temperature, "torch.float32"),
                           ("top_k", top_k, "torch.int32"), ("top_p", top_p, "torch.float32"),
                           ("min_p", min_p, "torch.float32")):
        if t is not None and not (_is(t, dtype) and t.shape == (rows,) and t.is_contiguous()):
            raise ClearError(f"{name} must be contiguous {dtype[6:]} [{rows}]")
    p = SampleParams(_ptr(temperature), _ptr(top_k), _ptr(top_p), _ptr(min_p))
    check(load().fhe_ssm_sample(_type(logits), logits.data_ptr(), rows, vocab, stride[0], draws.data_ptr(),
                                ctypes.addressof(p), tokens.data_ptr(), _ptr(logprobs),
                                _queue(stream, logits)))
