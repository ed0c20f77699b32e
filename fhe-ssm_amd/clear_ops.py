"""ctypes front end of libfhe_ssm_clear.so (include/fhe_ssm_clear.h): what a client of the encrypted step computes in the
clear -- linear attention with a decay for each head, products with 4-bit weights, the draw of a token; and what scores and
trains its drafting model: layer norm, a gated linear recurrence, the embedding, log-probabilities of given tokens, each with
its gradient, and the AdamW step.

Arguments are device tensors (torch's, or anything with data_ptr, dtype, shape and stride); outputs are tensors that the
caller brings.  Calls go to `stream` (a hipStream_t as an int, for torch `stream.cuda_stream`; 0 is the null stream; None is
torch's current stream, and the null stream for tensors that are not torch's) and return without waiting, so the tensors must
stay until that stream has passed them.  Shapes, types and strides are checked here and ClearError raised; there is no
fallback: if the library is missing, loading raises.  What scores and trains is asked for get_device() of its tensors too: they
lie on one device, the current one.
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


class LayerNormSizes(ctypes.Structure):
    """fhe_ssm_layer_norm"""
    _fields_ = [("type", _u32), ("weight_type", _u32), ("rows", _u32), ("channels", _u32), ("eps", ctypes.c_float),
                ("x_stride", _i64), ("out_stride", _i64), ("dy_stride", _i64)]


class GatedRecurrenceSizes(ctypes.Structure):
    """fhe_ssm_gated_recurrence"""
    _fields_ = [("type", _u32), ("lanes", _u32), ("tokens", _u32), ("channels", _u32), ("z_stride", _i64 * 2),
                ("x_stride", _i64 * 2), ("out_stride", _i64 * 2), ("dout_stride", _i64 * 2), ("dz_stride", _i64 * 2),
                ("dx_stride", _i64 * 2)]


class EmbeddingSizes(ctypes.Structure):
    """fhe_ssm_embedding"""
    _fields_ = [("table_type", _u32), ("row_type", _u32), ("tokens", _u32), ("vocab", _u32), ("channels", _u32),
                ("scale", ctypes.c_float), ("table_stride", _i64), ("row_stride", _i64)]


class TokenLogprobsSizes(ctypes.Structure):
    """fhe_ssm_token_logprobs"""
    _fields_ = [("type", _u32), ("rows", _u32), ("vocab", _u32), ("top", _u32), ("row_stride", _i64),
                ("gradient_stride", _i64)]


class AdamWSizes(ctypes.Structure):
    """fhe_ssm_adamw"""
    _fields_ = [("gradient_type", _u32), ("copy_type", _u32), ("state_bits", _u32), ("step", _u32), ("seed", _u32),
                ("lr", ctypes.c_float), ("eps", ctypes.c_float), ("beta1", ctypes.c_double), ("beta2", ctypes.c_double),
                ("lr_at", _vp), ("scale_at", _vp), ("step_at", _vp)]


class AdamWTensor(ctypes.Structure):
    """fhe_ssm_adamw_tensor"""
    _fields_ = [("param", _vp), ("gradient", _vp), ("first", _vp), ("second", _vp), ("powers", _vp), ("copy", _vp),
                ("n", ctypes.c_uint64), ("weight_decay", ctypes.c_float)]


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
    "fhe_ssm_layer_norm_workspace": (_int, [_vp, ctypes.POINTER(_size)]),
    "fhe_ssm_layer_norm_forward": (_int, [_vp] * 8),
    "fhe_ssm_layer_norm_backward": (_int, [_vp] * 10 + [_size, _vp]),
    "fhe_ssm_gated_recurrence_workspace": (_int, [_vp, ctypes.POINTER(_size), ctypes.POINTER(_size)]),
    "fhe_ssm_gated_recurrence_prompt": (_int, [_vp] * 9 + [_size, _vp]),
    "fhe_ssm_gated_recurrence_backward": (_int, [_vp] * 11 + [_size, _vp]),
    "fhe_ssm_gated_recurrence_step": (_int, [_vp] * 7),
    "fhe_ssm_embedding_lookup": (_int, [_vp] * 5),
    "fhe_ssm_embedding_workspace": (_int, [_vp, ctypes.POINTER(_size)]),
    "fhe_ssm_embedding_gradient": (_int, [_vp, _vp, _vp, _vp, _int, _vp, _size, _vp]),
    "fhe_ssm_token_logprobs_workspace": (_int, [_vp, ctypes.POINTER(_size)]),
    "fhe_ssm_token_logprobs_forward": (_int, [_vp] * 12 + [_size, _vp]),
    "fhe_ssm_token_logprobs_gradient": (_int, [_vp] * 9),
    "fhe_ssm_adamw_step": (_int, [_vp, _u32, _vp, _vp]),
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


# ------------------------------------------------------------------------------------------------ what the operators below share
_calls: dict = {}  # an operator's name, and sizes, types, strides and devices of a call's tensors -> its checked description


def _like(t):
    """all that is checked of a tensor; one on the host, whose device is -1, is refused when its description would be made"""
    return None if t is None else (t.dtype, t.shape, t.stride(), t.get_device())


def _kept(key, a):
    """keeps a call's checked description: the structure, which the caller holds while it is used, and its address"""
    _need(len({k[3] for k in key if type(k) is tuple}) <= 1, "tensors lie on different devices")
    if len(_calls) >= 512:
        _calls.clear()
    a = _calls[key] = a, ctypes.addressof(a)
    return a


def _bytes_of(workspace, t) -> int:
    """the size of the workspace of a call on tensor t, which is checked here too"""
    if workspace is None:
        return 0
    _need(workspace.is_contiguous() and workspace.get_device() == t.get_device(), "workspace must be contiguous, on the tensors' device")
    return workspace.numel() * workspace.element_size()


def _here(stream, t):
    """the stream of a call on tensor t, which has to lie on the current device: kernels are launched there"""
    torch = sys.modules.get("torch")
    if torch is not None and isinstance(t, torch.Tensor):
        device = t.get_device()
        if device >= 0 and device != torch._C._cuda_getDevice():
            raise ClearError(f"tensors lie on device {device}, which is not the current one")
    return _queue(stream, t)


def _floats(shape, **tensors) -> None:
    """each is None or contiguous float32 of the shape"""
    for name, t in tensors.items():
        if t is not None and not (t.shape == shape and _is(t, "torch.float32") and t.is_contiguous()):
            raise ClearError(f"{name} must be contiguous float32 {list(shape)}")


def _matrix(t, name: str):
    """the stride of the rows of a [rows, columns] tensor with contiguous rows"""
    _need(len(t.shape) == 2, f"{name} must be [rows, columns]")
    s = t.stride()
    _need(s[1] == 1 or t.shape[1] <= 1, f"rows of {name} must be contiguous")
    return s[0]


def _token_ids(tokens, rows=None):
    _need(_is(tokens, "torch.int64") and len(tokens.shape) == 1 and tokens.is_contiguous()
          and (rows is None or tokens.shape[0] == rows), "tokens must be contiguous int64, one for each row")


# ------------------------------------------------------------------------------------------------ layer norm
def _norm_sizes(x, out, weight, bias, eps=0.0, dy=None):
    rows, channels = x.shape if len(x.shape) == 2 else (0, 0)
    a = LayerNormSizes(_type(x), F32, rows, channels, eps, _matrix(x, "x"), 0, 0)
    if out is not None:
        _need(out.shape == x.shape and out.dtype == x.dtype, "the output must be like x")
        a.out_stride = _matrix(out, "the output")
    if dy is not None:
        _need(dy.shape == x.shape and dy.dtype == x.dtype, "dy must be like x")
        a.dy_stride = _matrix(dy, "dy")
    kinds = {_type(t) for t in (weight, bias) if t is not None}
    _need(len(kinds) < 2, "weight and bias differ in type")
    a.weight_type = kinds.pop() if kinds else F32
    for name, t in (("weight", weight), ("bias", bias)):
        _need(t is None or (tuple(t.shape) == (channels,) and t.is_contiguous()), f"{name} must be contiguous [{channels}]")
    return a


def layer_norm_workspace(x) -> int:
    """device bytes that layer_norm_backward needs for the weight's gradient of rows x (0 for few)"""
    a, n = _norm_sizes(x, None, None, None), _size()
    a.out_stride = a.channels
    check(load().fhe_ssm_layer_norm_workspace(ctypes.addressof(a), ctypes.byref(n)))
    return n.value


def layer_norm(x, weight, bias, out, mean=None, rstd=None, eps: float = 1e-5, stream=None) -> None:
    """out = (x - mean) rstd weight + bias over the channels of x [rows, channels], rstd = 1 / sqrt(variance + eps).

    out like x, or x itself; weight and bias [channels], float32 or of x's type, None: 1 and 0; mean and rstd float32 [rows] or
    None: what layer_norm_backward takes."""
    key = ("norm", eps, _like(x), _like(weight), _like(bias), _like(out), _like(mean), _like(rstd))
    a = _calls.get(key)
    if a is None:
        _on_device(x, weight, bias, out, mean, rstd)
        sizes = _norm_sizes(x, out, weight, bias, eps)
        _floats((sizes.rows,), mean=mean, rstd=rstd)
        a = _kept(key, sizes)
    check(load().fhe_ssm_layer_norm_forward(a[1], x.data_ptr(), _ptr(weight), _ptr(bias), out.data_ptr(), _ptr(mean),
                                            _ptr(rstd), _here(stream, x)))


def layer_norm_backward(dy, x, weight, mean, rstd, dx, dweight=None, dbias=None, workspace=None, stream=None) -> None:
    """The gradients of layer_norm from that of its output: dx like x (it may be dy), dweight and dbias float32 [channels] where
    they are given.  workspace: a uint8 tensor of layer_norm_workspace(x) bytes, needed for dweight and dbias."""
    key = ("norm back", _like(x), _like(weight), _like(dx), _like(dy), _like(mean), _like(rstd), _like(dweight), _like(dbias))
    a = _calls.get(key)
    if a is None:
        _on_device(dy, x, weight, mean, rstd, dx, dweight, dbias)
        sizes = _norm_sizes(x, dx, weight, None, dy=dy)
        _floats((sizes.rows,), mean=mean, rstd=rstd)
        _floats((sizes.channels,), dweight=dweight, dbias=dbias)
        a = _kept(key, sizes)
    check(load().fhe_ssm_layer_norm_backward(
        a[1], dy.data_ptr(), x.data_ptr(), _ptr(weight), mean.data_ptr(), rstd.data_ptr(), dx.data_ptr(),
        _ptr(dweight), _ptr(dbias), _ptr(workspace), _bytes_of(workspace, x), _here(stream, x)))


# ------------------------------------------------------------------------------------------------ gated recurrence
def _recurrence_sizes(z, tokens_axis, **others):
    """others: names of the description's strides -> tensors like z, or None"""
    n = 3 if tokens_axis else 2
    shape = z.shape
    _need(len(shape) == n, "z is [lanes, tokens, channels], of one token [lanes, channels]")
    a = GatedRecurrenceSizes(_type(z), shape[0], shape[1] if tokens_axis else 1, shape[-1])
    for name, t in (("z", z), *others.items()):
        if t is None:
            continue
        _need(t.shape == shape and t.dtype == z.dtype, f"{name} must be like z")
        s = t.stride()
        _need(s[-1] == 1 or shape[-1] <= 1, f"{name}: channels must be contiguous")
        setattr(a, name + "_stride", (s[0], s[1]) if tokens_axis else (s[0], 0))
    return a


def _lengths(lengths, lanes) -> None:
    _need(lengths is None or (_is(lengths, "torch.int32") and tuple(lengths.shape) == (lanes,) and lengths.is_contiguous()),
          "lengths must be contiguous int32 [lanes]")


def _recurrence_bytes(z):
    work, saved = _size(), _size()
    a = _recurrence_sizes(z, True)
    check(load().fhe_ssm_gated_recurrence_workspace(ctypes.addressof(a), ctypes.byref(work), ctypes.byref(saved)))
    return work.value, saved.value


def gated_recurrence_workspace(z) -> int:
    """device bytes that gated_recurrence and its backward pass need for gates of this shape (0 for many)"""
    return _recurrence_bytes(z)[0]


def gated_recurrence_saved(z) -> int:
    """device bytes that gated_recurrence saves for its backward pass"""
    return _recurrence_bytes(z)[1]


def _saved(saved, a, needed: bool = False) -> None:
    need = _size()
    check(load().fhe_ssm_gated_recurrence_workspace(ctypes.addressof(a), None, ctypes.byref(need)))
    if saved is None:
        _need(not needed or need.value == 0, "the backward pass needs what the prompt saved")
    else:
        _need(saved.is_contiguous() and saved.numel() * saved.element_size() >= need.value,
              f"saved must have {need.value} bytes, contiguous")


def gated_recurrence(z, x, state_in, state_out, out, lengths=None, saved=None, workspace=None, stream=None) -> None:
    """h_t = sigmoid(z_t) h_{t-1} + sigmoid(-z_t) x_t over a prompt, per lane and channel; out_t = h_t.

    z, x and out [lanes, tokens, channels]; states float32 [lanes, channels] (state_in None: zero; state_out None: not kept; both
    may be one tensor); lengths int32 [lanes]: tokens past a lane's length change nothing and give zeros; saved: None, or a uint8
    tensor of gated_recurrence_saved(z) bytes for the backward pass; workspace: one of gated_recurrence_workspace(z) bytes, None
    where that is 0."""
    key = ("recurrence", _like(z), _like(x), _like(state_in), _like(state_out), _like(out), _like(lengths), _like(saved))
    a = _calls.get(key)
    if a is None:
        _on_device(z, x, state_in, state_out, out, lengths, saved)
        sizes = _recurrence_sizes(z, True, x=x, out=out)
        _floats((sizes.lanes, sizes.channels), state_in=state_in, state_out=state_out)
        _lengths(lengths, sizes.lanes)
        _saved(saved, sizes)
        a = _kept(key, sizes)
    check(load().fhe_ssm_gated_recurrence_prompt(
        a[1], z.data_ptr(), x.data_ptr(), _ptr(lengths), _ptr(state_in), _ptr(state_out), out.data_ptr(),
        _ptr(saved), _ptr(workspace), _bytes_of(workspace, z), _here(stream, z)))


def gated_recurrence_backward(z, x, saved, dout, dstate_out, dz, dx, dstate_in=None, lengths=None, workspace=None,
                              stream=None) -> None:
    """The gradients of gated_recurrence: dz and dx like z, dstate_in float32 [lanes, channels] where it is given, from those of
    out and of state_out (None: zeros).  z, x, lengths and saved are the prompt's; dstate_in may be dstate_out."""
    key = ("recurrence back", _like(z), _like(x), _like(saved), _like(dout), _like(dstate_out), _like(dz), _like(dx),
           _like(dstate_in), _like(lengths))
    a = _calls.get(key)
    if a is None:
        _on_device(z, x, saved, dout, dstate_out, dz, dx, dstate_in, lengths)
        sizes = _recurrence_sizes(z, True, x=x, dout=dout, dz=dz, dx=dx)
        _floats((sizes.lanes, sizes.channels), dstate_in=dstate_in, dstate_out=dstate_out)
        _lengths(lengths, sizes.lanes)
        _saved(saved, sizes, needed=True)
        a = _kept(key, sizes)
    check(load().fhe_ssm_gated_recurrence_backward(
        a[1], z.data_ptr(), x.data_ptr(), _ptr(lengths), _ptr(saved), _ptr(dout), _ptr(dstate_out),
        dz.data_ptr(), dx.data_ptr(), _ptr(dstate_in), _ptr(workspace), _bytes_of(workspace, z), _here(stream, z)))


def gated_recurrence_step(z, x, state_in, state_out, out, stream=None) -> None:
    """gated_recurrence for one token of every lane: the same tensors without the token axis"""
    key = ("recurrence step", _like(z), _like(x), _like(state_in), _like(state_out), _like(out))
    a = _calls.get(key)
    if a is None:
        _on_device(z, x, state_in, state_out, out)
        sizes = _recurrence_sizes(z, False, x=x, out=out)
        _floats((sizes.lanes, sizes.channels), state_in=state_in, state_out=state_out)
        a = _kept(key, sizes)
    check(load().fhe_ssm_gated_recurrence_step(a[1], z.data_ptr(), x.data_ptr(), _ptr(state_in), _ptr(state_out),
                                               out.data_ptr(), _here(stream, z)))


# ------------------------------------------------------------------------------------------------ embedding
def embedding(tokens, table, out, scale: float = 1.0, stream=None) -> None:
    """out[t] = scale table[tokens[t]]; zeros for a token outside the table.  tokens int64 [n], table [vocab, channels], out
    [n, channels], each of any of the three types."""
    key = ("embedding", scale, _like(tokens), _like(table), _like(out))
    a = _calls.get(key)
    if a is None:
        _on_device(tokens, table, out)
        _token_ids(tokens)
        n = tokens.shape[0]
        strides = _matrix(table, "table"), _matrix(out, "out")
        vocab, channels = table.shape
        _need(tuple(out.shape) == (n, channels), f"out must be [{n}, {channels}]")
        a = EmbeddingSizes(_type(table), _type(out), n, vocab, channels, scale, *strides)
        if vocab == 1:  # the stride of the one row says nothing
            a.table_stride = channels
        a = _kept(key, a)
    check(load().fhe_ssm_embedding_lookup(a[1], tokens.data_ptr(), table.data_ptr(), out.data_ptr(),
                                          _here(stream, table)))


def _embedding_gradient_sizes(tokens, dtable, scale=1.0):
    _token_ids(tokens)
    _need(len(dtable.shape) == 2 and dtable.is_contiguous(), "dtable must be contiguous [vocab, channels]")
    vocab, channels = dtable.shape
    return EmbeddingSizes(_type(dtable), F32, tokens.shape[0], vocab, channels, scale, channels, channels)


def embedding_gradient_workspace(tokens, dtable) -> int:
    """device bytes that embedding_gradient needs (0 for few tokens)"""
    n = _size()
    a = _embedding_gradient_sizes(tokens, dtable)
    check(load().fhe_ssm_embedding_workspace(ctypes.addressof(a), ctypes.byref(n)))
    return n.value


def embedding_gradient(tokens, dout, dtable, scale: float = 1.0, accumulate: bool = False, workspace=None, stream=None) -> None:
    """dtable[v] = scale times the sum of dout[t] over the t with tokens[t] = v, the same in equal calls; with `accumulate` added to
    what is there.  dout [n, channels]; dtable contiguous [vocab, channels], float32 or of dout's type; workspace: a uint8 tensor of
    embedding_gradient_workspace(tokens, dtable) bytes, None where that is 0."""
    key = ("embedding back", scale, _like(tokens), _like(dout), _like(dtable))
    a = _calls.get(key)
    if a is None:
        _on_device(tokens, dout, dtable)
        a = _embedding_gradient_sizes(tokens, dtable, scale)
        a.row_type, a.row_stride = _type(dout), _matrix(dout, "dout")
        _need(tuple(dout.shape) == (a.tokens, a.channels), f"dout must be [{a.tokens}, {a.channels}]")
        a = _kept(key, a)
    check(load().fhe_ssm_embedding_gradient(a[1], tokens.data_ptr(), dout.data_ptr(), dtable.data_ptr(),
                                            bool(accumulate), _ptr(workspace), _bytes_of(workspace, dout), _here(stream, dout)))


# ------------------------------------------------------------------------------------------------ log-probabilities
def _logprobs_sizes(logits, top=0, gradient=None):
    stride = _matrix(logits, "logits")
    rows, vocab = logits.shape
    a = TokenLogprobsSizes(_type(logits), rows, vocab, top, stride, 0)
    if gradient is not None:
        _need(gradient.shape == logits.shape and gradient.dtype == logits.dtype, "the gradient must be like logits")
        a.gradient_stride = _matrix(gradient, "the gradient")
    return a


def token_logprobs_workspace(logits, top: int = 0) -> int:
    """device bytes that token_logprobs needs for logits of this shape and so many alternatives (0 for many)"""
    a, n = _logprobs_sizes(logits, top), _size()
    check(load().fhe_ssm_token_logprobs_workspace(ctypes.addressof(a), ctypes.byref(n)))
    return n.value


def token_logprobs(logits, tokens, logprobs, entropy=None, statistics=None, top_tokens=None, top_logprobs=None, workspace=None,
                   weights=None, entropy_weights=None, gradient=None, stream=None) -> None:
    """Log-probabilities of given tokens under softmax of logits [rows, vocab], with the rows' entropy and the alternatives.

    tokens int64 [rows], one outside the vocabulary is a padded position; logprobs and entropy float32 [rows], statistics float32
    [rows, 2]: what token_logprobs_gradient takes; top_tokens int64 and top_logprobs float32 [rows, k], k <= 32, in the order of
    falling logits, equal ones by rising index.  gradient (like logits, or logits itself) receives that of
    sum(weights logprobs + entropy_weights entropy) in the same call, with weights float32 [rows].  All but logits may be None.
    workspace: a uint8 tensor of token_logprobs_workspace(logits, k) bytes, None where that is 0."""
    key = ("logprobs", _like(logits), _like(tokens), _like(logprobs), _like(entropy), _like(statistics), _like(top_tokens),
           _like(top_logprobs), _like(weights), _like(entropy_weights), _like(gradient))
    a = _calls.get(key)
    if a is None:
        _on_device(logits, tokens, logprobs, entropy, statistics, top_tokens, top_logprobs, weights, entropy_weights, gradient)
        top = 0
        if top_tokens is not None or top_logprobs is not None:
            _need(top_tokens is not None and top_logprobs is not None, "top_tokens and top_logprobs come together")
            _need(_is(top_tokens, "torch.int64") and len(top_tokens.shape) == 2 and top_tokens.is_contiguous()
                  and top_tokens.shape[0] == logits.shape[0], "top_tokens must be contiguous int64 [rows, k]")
            top = top_tokens.shape[1]
        a = _logprobs_sizes(logits, top, gradient)
        if tokens is not None:
            _token_ids(tokens, a.rows)
        _floats((a.rows,), logprobs=logprobs, entropy=entropy, weights=weights, entropy_weights=entropy_weights)
        _floats((a.rows, 2), statistics=statistics)
        _floats((a.rows, top), top_logprobs=top_logprobs)
        a = _kept(key, a)
    check(load().fhe_ssm_token_logprobs_forward(
        a[1], logits.data_ptr(), _ptr(tokens), _ptr(logprobs), _ptr(entropy), _ptr(statistics),
        _ptr(top_tokens), _ptr(top_logprobs), _ptr(weights), _ptr(entropy_weights), _ptr(gradient), _ptr(workspace),
        _bytes_of(workspace, logits), _here(stream, logits)))


def token_logprobs_gradient(logits, tokens, statistics, weights, gradient, entropy_weights=None, entropy=None,
                            stream=None) -> None:
    """The gradient that token_logprobs writes, where its weights were not known then: from the statistics, and the entropy if it
    has weights."""
    key = ("logprobs back", _like(logits), _like(tokens), _like(statistics), _like(weights), _like(gradient),
           _like(entropy_weights), _like(entropy))
    a = _calls.get(key)
    if a is None:
        _on_device(logits, tokens, statistics, weights, gradient, entropy_weights, entropy)
        a = _logprobs_sizes(logits, 0, gradient)
        if tokens is not None:
            _token_ids(tokens, a.rows)
        _floats((a.rows,), weights=weights, entropy_weights=entropy_weights, entropy=entropy)
        _floats((a.rows, 2), statistics=statistics)
        a = _kept(key, a)
    check(load().fhe_ssm_token_logprobs_gradient(
        a[1], logits.data_ptr(), _ptr(tokens), statistics.data_ptr(), _ptr(entropy), _ptr(weights),
        _ptr(entropy_weights), gradient.data_ptr(), _here(stream, logits)))


# ------------------------------------------------------------------------------------------------ AdamW
class AdamW:
    """The AdamW step over a model's tensors, and its states.

    params: contiguous float32 tensors, updated in place.  weight_decay: one for all, or one for each.  copies: bfloat16 or
    float16 tensors (one type) that receive the parameters after every step, or None.  bits: 32 for states in float32, 8 for
    states in 8-bit floats with a power of two for each 256 entries: m and the root of v as float8_e4m3fn, and the powers.
    states: (m, v) or (m, root, powers), lists of tensors like params (powers uint8 [blocks, 2]); None begins with zeros.  No two of
    all these tensors may share memory."""

    BLOCK = 256

    def __init__(self, params, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay=0.01, bits: int = 32, copies=None, states=None):
        self.params, n = list(params), len(params)
        _need(n > 0, "no parameters")
        _on_device(*self.params)
        for p in self.params:
            _need(_is(p, "torch.float32") and p.is_contiguous(), "parameters must be contiguous float32")
            _need(p.device == self.params[0].device, "parameters lie on different devices")
        _need(bits in (8, 32), f"states have 8 or 32 bits, not {bits}")
        self.bits, self.copies = bits, None if copies is None else list(copies)
        decay = [float(weight_decay)] * n if isinstance(weight_decay, (int, float)) else [float(w) for w in weight_decay]
        _need(len(decay) == n, "one weight_decay for all, or one for each parameter")
        if states is None:
            states = self._zeros()
        _need(len(states) == (2 if bits == 32 else 3) and all(len(s) == n for s in states), "states are lists as long as params")
        self.states = tuple(list(s) for s in states)
        kind = "torch.float32" if bits == 32 else "torch.float8_e4m3fn"
        for name, s in zip(("the first state", "the second state"), self.states):
            for p, t in zip(self.params, s):
                _need(t.device == p.device and t.shape == p.shape and _is(t, kind) and t.is_contiguous(),
                      f"{name} must be contiguous {kind[6:]} like its parameter")
        if bits == 8:
            for p, t in zip(self.params, self.states[2]):
                blocks = -(-p.numel() // self.BLOCK)
                _need(t.device == p.device and tuple(t.shape) == (blocks, 2) and _is(t, "torch.uint8") and t.is_contiguous(),
                      "powers must be contiguous uint8 [blocks, 2]")
        copy_type = BF16
        if self.copies is not None:
            _need(len(self.copies) == n, "one copy for each parameter")
            copy_type = _type(self.copies[0])
            _need(copy_type != F32, "copies are bfloat16 or float16")
            for p, t in zip(self.params, self.copies):
                _need(t.device == p.device and t.shape == p.shape and t.dtype == self.copies[0].dtype and t.is_contiguous(),
                      "copies must be contiguous bfloat16 or float16 like their parameters")
        spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size())
                       for ts in (self.params, *self.states, self.copies or ()) for t in ts if t.numel())
        _need(all(a[1] <= b[0] for a, b in zip(spans, spans[1:])), "parameters, states or copies share memory")
        self._sizes = AdamWSizes(F32, copy_type, bits, 0, 0, 0.0, eps, *betas)
        self._tensors = (AdamWTensor * n)()
        for i, (t, p) in enumerate(zip(self._tensors, self.params)):
            t.param, t.first, t.second, t.n = p.data_ptr(), self.states[0][i].data_ptr(), self.states[1][i].data_ptr(), p.numel()
            t.weight_decay = decay[i]
            if bits == 8:
                t.powers = self.states[2][i].data_ptr()
            if self.copies is not None:
                t.copy = self.copies[i].data_ptr()
        self._gradients = np.frombuffer(self._tensors, np.uint64).reshape(n, -1)[:, 1]
        # the memory stays while this does, and whose tensors the caller gave other memory is told at the next step
        self._memory = [t.detach() for ts in (self.params, *self.states, self.copies or ()) for t in ts]
        self._theirs = self.params + (self.copies or [])
        self._at, self._shapes = [t.data_ptr() for t in self._theirs], [p.shape for p in self.params]

    def _zeros(self):
        if self.bits == 32:
            return [p.new_zeros(p.shape) for p in self.params], [p.new_zeros(p.shape) for p in self.params]
        import torch
        codes = [[p.new_zeros(p.shape, dtype=torch.uint8).view(torch.float8_e4m3fn) for p in self.params] for _ in range(2)]
        return *codes, [p.new_zeros((-(-p.numel() // self.BLOCK), 2), dtype=torch.uint8) for p in self.params]

    def step(self, gradients, lr, step, seed: int = 0, scale=None, stream=None) -> None:
        """One step with the gradients, contiguous tensors of one type like the parameters.  lr: a number or a float32 tensor of
        one; step, from 1: a number or an int32 tensor of one; scale: a float32 tensor of one that the gradients are multiplied
        by, or None.  Tensors are read when the step runs, so that a recorded one follows them; one of a step below 1 leaves all as
        it is.  seed goes, with the step, into how 8-bit states are rounded."""
        _need(len(gradients) == len(self.params), f"{len(self.params)} gradients are needed")
        kind, at = gradients[0].dtype, self.params[0].get_device()
        for g, shape in zip(gradients, self._shapes):
            if not (g.is_cuda and g.get_device() == at and g.dtype == kind and g.shape == shape and g.is_contiguous()):
                raise ClearError("gradients must be contiguous tensors of one type, like their parameters, on the GPU")
        if [t.data_ptr() for t in self._theirs] != self._at:
            raise ClearError("a parameter or copy has other memory than it had; an AdamW of them and of these states goes on")
        if isinstance(step, int) and not 1 <= step < 1 << 32:
            raise ClearError(f"steps count from 1, not {step}")
        a = self._sizes
        a.gradient_type, a.seed = _type(gradients[0]), seed & 0xffffffff
        a.lr, a.lr_at = (lr, None) if isinstance(lr, (int, float)) else (0.0, self._one(lr, "lr", "torch.float32", at))
        a.step, a.step_at = (step, None) if isinstance(step, int) else (0, self._one(step, "step", "torch.int32", at))
        a.scale_at = None if scale is None else self._one(scale, "scale", "torch.float32", at)
        self._gradients[:] = [g.data_ptr() for g in gradients]
        check(load().fhe_ssm_adamw_step(ctypes.addressof(a), len(self.params), ctypes.addressof(self._tensors),
                                        _here(stream, self.params[0])))

    @staticmethod
    def _one(t, name: str, dtype: str, at: int):
        _need(hasattr(t, "data_ptr") and t.is_cuda and t.get_device() == at and _is(t, dtype) and t.numel() == 1,
              f"{name} must be a number or a {dtype[6:]} tensor of one, on the parameters' GPU")
        return t.data_ptr()
