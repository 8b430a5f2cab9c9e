"""A decoder layer's operators on decoded weights: matrix products with their
epilogue, over 16-bit weights or INT4 buffers (hh_linear), the gated
feed-forward's two in one launch (hh_gated_linear), the norms between them and
rotary positions (hh_norm, hh_rotary), all three with their gradients, and a
paged 8-bit key / value cache with its plan, append, read, attention and
differential attention (hh_kv_*).

Tensors are torch tensors on the context's device.  Calls run on torch's
current stream, where their results are allocated, and don't synchronise.
Calls on several streams need no order but their tensors' own; captured calls
keep what they use of the context's memory for as long as the context lives, whatever is called later (graphs
captured on one stream must not run beside each other).
What a call can't take raises HaagentiError before anything is launched;
gradients are calls of their own (norm_backward, gated_linear_backward,
rotary's inverse) that autograd doesn't know, so tensors that require them are taken under
torch.no_grad() only."""
import ctypes as C
import struct

import torch

from . import BF16, F16, F32, INVALID_ARGUMENT, UNSUPPORTED, HaagentiError, _check, _i32, _sig, _u32, _vp

INT4 = 16

NORMS = {"layer": 0, "rms": 1}
ACTIVATIONS = {"none": 0, None: 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
_CODE = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
_HALF = {torch.float16: F16, torch.bfloat16: BF16}

# The argument structures, packed as the header lays them out (natural
# alignment, no gaps; a step's calls are a few microseconds each, and a packed
# string costs a quarter of a ctypes structure).
_LINEAR = struct.Struct("=6Q6Q3I4i4x")      # hh_linear_args
_NORM = struct.Struct("=4Q2Q2If3i")         # hh_norm_args
_NORM_GRADS = struct.Struct("=6Q")          # hh_norm_grads
_ROTARY = struct.Struct("=4Q5Q8I3i4x")      # hh_rotary_args
_GATED = struct.Struct("=7Q6Q3I4i4x")       # hh_gated_args
_GATED_GRADS = struct.Struct("=6Q4Q")       # hh_gated_grads
_CACHE = struct.Struct("=4Q4I")             # hh_kv_cache
_PLAN = struct.Struct("=10QQ5I4x")          # hh_kv_plan_args
_ATTENTION = struct.Struct("=5Q5Q6Ifi")     # hh_kv_attention_args
_DIFF = struct.Struct("=2Q2f")              # hh_kv_diff_args

_u64, _bytes = C.c_uint64, C.c_char_p
_linear = _sig("hh_linear", _i32, [_vp, _bytes, _vp])
_norm = _sig("hh_norm", _i32, [_vp, _bytes, _vp])
_norm_backward = _sig("hh_norm_backward", _i32, [_vp, _bytes, _bytes, _vp])
_rotary = _sig("hh_rotary", _i32, [_vp, _bytes, _vp])
_gated = _sig("hh_gated_linear", _i32, [_vp, _bytes, _vp])
_gated_backward = _sig("hh_gated_linear_backward", _i32, [_vp, _bytes, _bytes, _vp])
_plan = _sig("hh_kv_plan", _i32, [_vp, _bytes, _vp])
_append = _sig("hh_kv_append", _i32, [_vp, _bytes, _vp, _vp, _i32, _u64, _u64, _u64, _u64, _vp, _u32, _vp])
_read = _sig("hh_kv_read", _i32, [_vp, _bytes, _vp, _u32, _i32, _vp, _vp, _vp])
_diff_attention = _sig("hh_kv_diff_attention", _i32, [_vp, _bytes, _bytes, _bytes, _vp])
_attention = _sig("hh_kv_attention", _i32, [_vp, _bytes, _bytes, _vp])

# torch.cuda.current_stream(device).cuda_stream without the Stream object
_stream = torch._C._cuda_getCurrentRawStream


def _refuse(code, what):
    raise HaagentiError(code, what)


def _no_grad(what):
    """For a tensor that requires gradients: refuses it where autograd is asked to follow."""
    if torch.is_grad_enabled():
        _refuse(UNSUPPORTED, f"{what}: no gradients (call it under torch.no_grad())")


def _on(dev, what, *tensors):
    for t in tensors:
        if t is not None and t.get_device() != dev:
            _refuse(INVALID_ARGUMENT, f"{what}: tensors must be on the context's device")


def _ints(what, *tensors):
    for t in tensors:
        if t.dtype != torch.int32 or not t.is_contiguous():
            _refuse(INVALID_ARGUMENT, f"{what}: contiguous int32 tensors")


class Int4Weight:
    """An n x k weight as its INT4 buffer (quantize_int4 of its values in row
    order: ceil(n k / 32) f16 scales, then ceil(n k / 2) bytes of nibbles), a
    uint8 device tensor."""

    def __init__(self, data, n, k):
        if data.dtype != torch.uint8 or not data.is_contiguous():
            _refuse(INVALID_ARGUMENT, "Int4Weight: a contiguous uint8 tensor")
        self.data, self.n, self.k = data, int(n), int(k)
        if self.n < 0 or self.k < 0:
            _refuse(INVALID_ARGUMENT, "Int4Weight: a negative size")


def _rows(t, m, n, dev, what, of="linear"):
    """Row stride of an m x n matrix on the device whose rows are contiguous."""
    shape, stride = t.shape, t.stride()
    if len(shape) != 2 or shape[0] != m or shape[1] != n or (n > 1 and stride[1] != 1 and m):
        _refuse(INVALID_ARGUMENT, f"{of}: {what} is {m} x {n} with contiguous rows, got {tuple(shape)}")
    if t.get_device() != dev:
        _refuse(INVALID_ARGUMENT, f"{of}: {what} must be on the context's device")
    return stride[0] if m > 1 else n


def _apart(a, b):
    """Whether two matrices with contiguous rows share no memory (columns of
    one buffer's rows side by side are apart)."""
    spans = []
    for t in (a, b):
        size = t.element_size()
        rows, width = (t.shape[0], t.shape[1]) if t.dim() == 2 else (1, t.numel())
        stride = t.stride(0) if rows > 1 else width
        if not rows or not width:
            return True
        spans.append((t.data_ptr(), stride * size, width * size, t.data_ptr() + ((rows - 1) * stride + width) * size))
    (a0, a_step, a_width, a1), (b0, b_step, b_width, b1) = spans
    if a1 <= b0 or b1 <= a0:
        return True
    if a_step != b_step or not a_step:
        return False
    between = (b0 - a0) % a_step
    return between >= a_width and between + b_width <= a_step


def linear(ctx, x, w, bias=None, act=None, mul=None, residual=None, out=None, out_dtype=None):
    """act(x w^T + bias) * mul + residual (hh_linear).  x: m x k, float16 or
    bfloat16; w: n x k of x's type, or an Int4Weight; bias n values, mul and
    residual m x n, of x's type.  act: a key of ACTIVATIONS.  Rows are
    contiguous, any stride apart.  Returns out (m x n of out_dtype, by default
    x's type; float32 is allowed), which may be residual or mul."""
    dtype, dev, shape = x.dtype, ctx.device, x.shape
    dt = _HALF.get(dtype)
    if dt is None:
        _refuse(UNSUPPORTED, f"linear: {dtype} (float16 or bfloat16)")
    if len(shape) != 2:
        _refuse(INVALID_ARGUMENT, "linear: x is m x k")
    m, k = shape
    if isinstance(w, Int4Weight):
        n, w_dtype, w_stride, w_bytes = w.n, INT4, 0, w.data.numel()
        if w.k != k:
            _refuse(INVALID_ARGUMENT, f"linear: x has {k} columns, the weight {w.k}")
        w = w.data
        _on(dev, "linear", w)
    else:
        if w.dtype != dtype or w.dim() != 2:
            _refuse(INVALID_ARGUMENT, "linear: w is n x k of x's type, or an Int4Weight")
        n, w_dtype, w_bytes = w.shape[0], dt, 0
        w_stride = _rows(w, n, k, dev, "w")
    if x.requires_grad or w.requires_grad:
        _no_grad("linear")
    code = ACTIVATIONS.get(act)
    if code is None:
        _refuse(UNSUPPORTED, f"linear: activation {act!r}")
    x_stride = _rows(x, m, k, dev, "x")
    if out is None:
        y_dtype, y_stride = out_dtype or dtype, n
        if y_dtype is not dtype and y_dtype is not torch.float32:
            _refuse(UNSUPPORTED, f"linear: output {y_dtype}")
        out = x.new_empty((m, n), dtype=y_dtype)
    else:
        y_dtype = out.dtype
        if y_dtype is not dtype and y_dtype is not torch.float32:
            _refuse(UNSUPPORTED, f"linear: output {y_dtype}")
        if out_dtype is not None and y_dtype is not out_dtype:
            _refuse(INVALID_ARGUMENT, "linear: out has another type than out_dtype")
        y_stride = _rows(out, m, n, dev, "out")
        for t in (x, w, bias, mul, residual):
            # (a weight's buffer is compared whole)
            if t is not None and not _apart(out, t) and not (
                    (t is mul or t is residual) and t.data_ptr() == out.data_ptr() and t.dtype is y_dtype
                    and (m == 1 or t.stride(0) == y_stride)):
                _refuse(INVALID_ARGUMENT, "linear: out lies over what is read (other than mul or residual itself)")
        if out.requires_grad:
            _no_grad("linear")
    b = c = d = c_stride = d_stride = 0
    if bias is not None:
        if bias.dim() != 1 or bias.shape[0] != n or bias.dtype is not dtype or not bias.is_contiguous():
            _refuse(INVALID_ARGUMENT, "linear: bias is n contiguous values of x's type")
        _on(dev, "linear", bias)
        if bias.requires_grad:
            _no_grad("linear")
        b = bias.data_ptr()
    if mul is not None:
        c, c_stride = mul.data_ptr(), _rows(mul, m, n, dev, "mul")
        if mul.dtype is not dtype:
            _refuse(INVALID_ARGUMENT, "linear: mul has x's type")
        if mul.requires_grad:
            _no_grad("linear")
    if residual is not None:
        d, d_stride = residual.data_ptr(), _rows(residual, m, n, dev, "residual")
        if residual.dtype is not dtype:
            _refuse(INVALID_ARGUMENT, "linear: residual has x's type")
        if residual.requires_grad:
            _no_grad("linear")
    try:
        args = _LINEAR.pack(x.data_ptr(), w.data_ptr(), b, c, d, out.data_ptr(), x_stride, w_stride, c_stride, d_stride,
                            y_stride, w_bytes, m, n, k, dt, w_dtype, _CODE[y_dtype], code)
    except struct.error:
        _refuse(INVALID_ARGUMENT, f"linear: {m} x {n} x {k}")
    rc = _linear(ctx.handle, args, _stream(dev))
    if rc:
        _check(rc, "hh_linear")
    return out


def _same(a, b, m):
    """Whether two m x n matrices of one type are the same memory in the same order."""
    return a.data_ptr() == b.data_ptr() and a.dtype is b.dtype and (m <= 1 or a.stride(0) == b.stride(0))


def _out_rows(out, m, n, dtype, dev, of, reads, over=()):
    """Row stride of a given output: of this type, apart from `reads`, and from `over` unless it is one of these itself."""
    if out.dtype is not dtype:
        _refuse(INVALID_ARGUMENT, f"{of}: out is {dtype}")
    stride = _rows(out, m, n, dev, "out", of)
    if m > 1 and stride < n:
        _refuse(INVALID_ARGUMENT, f"{of}: rows of out overlap")
    if out.requires_grad:
        _no_grad(of)
    for t in reads:
        if t is not None and not _apart(out, t):
            _refuse(INVALID_ARGUMENT, f"{of}: out lies over what is read")
    for t in over:
        if t is not None and not _same(out, t, m) and not _apart(out, t):
            _refuse(INVALID_ARGUMENT, f"{of}: out lies over part of what is read")
    return stride


def _norm_args(what, ctx, x, weight, bias, kind, eps):
    """The checks that both passes share: (rows, n, code of x's type, the weights' code, kind)."""
    dev, dt = ctx.device, _CODE.get(x.dtype)
    if dt is None:
        _refuse(UNSUPPORTED, f"{what}: {x.dtype} (float32, float16 or bfloat16)")
    if kind not in NORMS:
        _refuse(UNSUPPORTED, f"{what}: kind {kind!r}")
    if x.dim() != 2:
        _refuse(INVALID_ARGUMENT, f"{what}: x is rows x n")
    rows, n = x.shape
    wt = dt
    for t in (weight, bias):
        if t is None:
            continue
        if t.dim() != 1 or t.shape[0] != n or not t.is_contiguous() or (t.dtype is not x.dtype and t.dtype is not torch.float32):
            _refuse(INVALID_ARGUMENT, f"{what}: weight and bias are n contiguous values of x's type or float32")
        _on(dev, what, t)
        if t.requires_grad:
            _no_grad(what)
        wt = _CODE[t.dtype]
    if weight is not None and bias is not None and weight.dtype is not bias.dtype:
        _refuse(INVALID_ARGUMENT, f"{what}: weight and bias have one type")
    if x.requires_grad:
        _no_grad(what)
    return rows, n, dt, wt, NORMS[kind]


def norm(ctx, x, weight=None, bias=None, kind="layer", eps=1e-5, out=None):
    """Layer norm of the rows of x, or with kind "rms" the root mean square
    norm (hh_norm): (x - mean) / sqrt(variance + eps) * weight + bias.  x:
    rows x n, float32, float16 or bfloat16, rows contiguous, any stride apart;
    weight and bias n values of x's type or float32.  Returns out, of x's type,
    which may be x itself."""
    rows, n, dt, wt, code = _norm_args("norm", ctx, x, weight, bias, kind, eps)
    dev = ctx.device
    x_stride = _rows(x, rows, n, dev, "x", "norm")
    if out is None:
        out, y_stride = x.new_empty((rows, n)), n
    else:
        y_stride = _out_rows(out, rows, n, x.dtype, dev, "norm", (weight, bias), (x,))
    try:
        args = _NORM.pack(x.data_ptr(), 0 if weight is None else weight.data_ptr(), 0 if bias is None else bias.data_ptr(),
                          out.data_ptr(), x_stride, y_stride, rows, n, eps, dt, wt, code)
    except (struct.error, OverflowError):
        _refuse(INVALID_ARGUMENT, f"norm: {rows} x {n}, eps {eps!r}")
    rc = _norm(ctx.handle, args, _stream(dev))
    if rc:
        _check(rc, "hh_norm")
    return out


def norm_backward(ctx, dy, x, weight=None, bias=False, kind="layer", eps=1e-5, add=None, out=None):
    """The gradients of norm from dy, that of its output, and its x and weight
    (hh_norm_backward): (dx, dweight, dbias).  dx is of x's type, `add` (rows x
    n of that type; what else flows back into x) on top, and may be given as
    out: dy, x or add itself; dweight (with a weight) and dbias (with bias
    true) are float32, else None."""
    rows, n, dt, wt, code = _norm_args("norm_backward", ctx, x, weight, None, kind, eps)
    dev = ctx.device
    x_stride = _rows(x, rows, n, dev, "x", "norm_backward")
    strides = []
    for t, name in ((dy, "dy"), (add, "add")):
        if t is None:
            strides.append(0)
            continue
        if t.dtype is not x.dtype:
            _refuse(INVALID_ARGUMENT, f"norm_backward: {name} has x's type")
        strides.append(_rows(t, rows, n, dev, name, "norm_backward"))
        if t.requires_grad:
            _no_grad("norm_backward")
    if out is None:
        out, y_stride = x.new_empty((rows, n)), n
    else:
        y_stride = _out_rows(out, rows, n, x.dtype, dev, "norm_backward", (weight,), (x, dy, add))
    dweight = None if weight is None else x.new_empty(n, dtype=torch.float32)
    dbias = x.new_empty(n, dtype=torch.float32) if bias else None
    try:
        args = _NORM.pack(x.data_ptr(), 0 if weight is None else weight.data_ptr(), 0, out.data_ptr(), x_stride, y_stride, rows,
                          n, eps, dt, wt, code)
    except (struct.error, OverflowError):
        _refuse(INVALID_ARGUMENT, f"norm_backward: {rows} x {n}, eps {eps!r}")
    grads = _NORM_GRADS.pack(dy.data_ptr(), 0 if add is None else add.data_ptr(), 0 if dweight is None else dweight.data_ptr(),
                             0 if dbias is None else dbias.data_ptr(), *strides)
    rc = _norm_backward(ctx.handle, args, grads, _stream(dev))
    if rc:
        _check(rc, "hh_norm_backward")
    return out, dweight, dbias


def rotary(ctx, x, positions, inv_freq, sections=None, interleaved=False, inverse=False, out=None):
    """Rotary positions on x (tokens x heads x dim, float32, float16 or
    bfloat16; any token and head strides, so the query and key heads of a joint
    projection are one call) (hh_rotary).  positions: int32, axes x tokens (or
    tokens, for one axis); inv_freq: float32, one frequency per pair of
    dimensions; sections: how many of the pairs, in order, each axis turns
    (default: all the first).  Pair j is dimensions (j, j + pairs), interleaved
    (2 j, 2 j + 1); dimensions past the pairs are copied.  inverse turns back:
    the gradient's way.  Returns out, of x's type, which may be x itself."""
    dev, dt, shape, stride = ctx.device, _CODE.get(x.dtype), x.shape, x.stride()
    if dt is None:
        _refuse(UNSUPPORTED, f"rotary: {x.dtype} (float32, float16 or bfloat16)")
    if len(shape) != 3 or (shape[2] > 1 and stride[2] != 1 and shape[0] and shape[1]):
        _refuse(INVALID_ARGUMENT, "rotary: x is tokens x heads x dim, contiguous dimensions")
    tokens, heads, dim = shape
    if positions.dim() == 1:
        positions = positions[None]
    if positions.dtype != torch.int32 or positions.dim() != 2 or positions.shape[1] != tokens \
            or (tokens > 1 and positions.stride(1) != 1):
        _refuse(INVALID_ARGUMENT, "rotary: positions are int32, axes x tokens with contiguous rows")
    if inv_freq.dtype != torch.float32 or inv_freq.dim() != 1 or not inv_freq.is_contiguous():
        _refuse(INVALID_ARGUMENT, "rotary: inv_freq is contiguous float32, one per pair")
    axes = positions.shape[0]
    sections = [inv_freq.numel()] if sections is None else list(sections)
    if len(sections) != axes or not 1 <= axes <= 4:
        _refuse(INVALID_ARGUMENT, "rotary: a section for each of 1 to 4 axes of positions")
    if any(s < 0 for s in sections) or sum(sections) != inv_freq.numel() or 2 * sum(sections) > dim:
        _refuse(INVALID_ARGUMENT, "rotary: sections add up to inv_freq's pairs, at most half of dim")
    _on(dev, "rotary", x, positions, inv_freq)
    if x.requires_grad or inv_freq.requires_grad:
        _no_grad("rotary")
    if out is None:
        out = x.new_empty((tokens, heads, dim))
        yt, yh = heads * dim, dim
    else:
        if out.dtype is not x.dtype or out.shape != shape or (dim > 1 and out.stride(2) != 1 and tokens and heads):
            _refuse(INVALID_ARGUMENT, "rotary: out is like x")
        _on(dev, "rotary", out)
        if out.requires_grad:
            _no_grad("rotary")
        yt, yh = out.stride(0), out.stride(1)
        same = out.data_ptr() == x.data_ptr() and (tokens <= 1 or yt == stride[0]) and (heads <= 1 or yh == stride[1])
        if any(not _spans_apart(out, t) for t in ((positions, inv_freq) if same else (positions, inv_freq, x))):
            _refuse(INVALID_ARGUMENT, "rotary: out is x itself or lies apart from what is read")
    try:
        args = _ROTARY.pack(x.data_ptr(), out.data_ptr(), positions.data_ptr(), inv_freq.data_ptr(), stride[0], stride[1], yt, yh,
                            positions.stride(0) if axes > 1 else tokens, tokens, heads, dim, axes,
                            *(sections + [0] * (4 - axes)), bool(interleaved), bool(inverse), dt)
    except struct.error:
        _refuse(INVALID_ARGUMENT, f"rotary: {tuple(shape)}")
    rc = _rotary(ctx.handle, args, _stream(dev))
    if rc:
        _check(rc, "hh_rotary")
    return out


def _spans_apart(a, b):
    """Whether the memory from the first to the last element of two tensors is apart."""
    if not a.numel() or not b.numel():
        return True
    end = [t.data_ptr() + (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))) * t.element_size() for t in (a, b)]
    return end[0] <= b.data_ptr() or end[1] <= a.data_ptr()



def _gated_args(what, ctx, x, gate, up, act):
    """The checks that both passes share: (m, n, k, x's code, the weights' code, the pointers, strides and buffer sizes)."""
    dev, dt = ctx.device, _HALF.get(x.dtype)
    if dt is None:
        _refuse(UNSUPPORTED, f"{what}: {x.dtype} (float16 or bfloat16)")
    if x.dim() != 2:
        _refuse(INVALID_ARGUMENT, f"{what}: x is m x k")
    m, k = x.shape
    if isinstance(gate, Int4Weight) != isinstance(up, Int4Weight):
        _refuse(INVALID_ARGUMENT, f"{what}: gate and up are both tensors or both Int4Weights")
    if isinstance(gate, Int4Weight):
        if (gate.n, gate.k) != (up.n, up.k) or gate.k != k:
            _refuse(INVALID_ARGUMENT, f"{what}: x has {k} columns, the weights {gate.k} and {up.k}, of {gate.n} and {up.n} rows")
        n, wt, strides, sizes, held = gate.n, INT4, (0, 0), (gate.data.numel(), up.data.numel()), (gate.data, up.data)
        _on(dev, what, *held)
    else:
        if gate.dtype is not x.dtype or up.dtype is not x.dtype or gate.dim() != 2:
            _refuse(INVALID_ARGUMENT, f"{what}: gate and up are n x k of x's type, or Int4Weights")
        n, wt, sizes, held = gate.shape[0], dt, (0, 0), (gate, up)
        strides = _rows(gate, n, k, dev, "gate", what), _rows(up, n, k, dev, "up", what)
    code = ACTIVATIONS.get(act)
    if code is None:
        _refuse(UNSUPPORTED, f"{what}: activation {act!r}")
    if x.requires_grad or held[0].requires_grad or held[1].requires_grad:
        _no_grad(what)
    return m, n, k, dt, wt, code, held, (_rows(x, m, k, dev, "x", what), *strides), sizes


def gated_linear(ctx, x, gate, up, gate_bias=None, up_bias=None, act="silu", save=False, out=None, out_dtype=None):
    """act(x gate^T + gate_bias) * (x up^T + up_bias) in one launch
    (hh_gated_linear).  x: m x k, float16 or bfloat16; gate and up: n x k of
    x's type, or two Int4Weights; biases n values of x's type.  act: a key of
    ACTIVATIONS.  Returns out (m x n of out_dtype, by default x's type; float32
    is allowed), with save (out, saved): saved is what
    gated_linear_backward takes, m x 2 n float32."""
    m, n, k, dt, wt, code, held, strides, sizes = _gated_args("gated_linear", ctx, x, gate, up, act)
    dev, dtype = ctx.device, x.dtype
    biases = []
    for b in (gate_bias, up_bias):
        if b is None:
            biases.append(0)
            continue
        if b.dim() != 1 or b.shape[0] != n or b.dtype is not dtype or not b.is_contiguous():
            _refuse(INVALID_ARGUMENT, "gated_linear: biases are n contiguous values of x's type")
        _on(dev, "gated_linear", b)
        if b.requires_grad:
            _no_grad("gated_linear")
        biases.append(b.data_ptr())
    if out is None:
        y_dtype, y_stride = out_dtype or dtype, n
        if y_dtype is not dtype and y_dtype is not torch.float32:
            _refuse(UNSUPPORTED, f"gated_linear: output {y_dtype}")
        out = x.new_empty((m, n), dtype=y_dtype)
    else:
        y_dtype = out.dtype
        if y_dtype is not dtype and y_dtype is not torch.float32:
            _refuse(UNSUPPORTED, f"gated_linear: output {y_dtype}")
        y_stride = _out_rows(out, m, n, out_dtype or y_dtype, dev, "gated_linear", (x, *held, gate_bias, up_bias))
    saved = x.new_empty((m, 2 * n), dtype=torch.float32) if save else None
    try:
        args = _GATED.pack(x.data_ptr(), held[0].data_ptr(), held[1].data_ptr(), *biases, out.data_ptr(),
                           saved.data_ptr() if save else 0, *strides, y_stride, *sizes, m, n, k, dt, wt, _CODE[y_dtype], code)
    except struct.error:
        _refuse(INVALID_ARGUMENT, f"gated_linear: {m} x {n} x {k}")
    rc = _gated(ctx.handle, args, _stream(dev))
    if rc:
        _check(rc, "hh_gated_linear")
    return (out, saved) if save else out



class GatedGrads:
    """What gated_linear_backward gives: dx, dgate, dup (of x's type) and the biases' dgate_bias, dup_bias (float32); None for
    what was not asked for."""
    __slots__ = ("dx", "dgate", "dup", "dgate_bias", "dup_bias")

    def __init__(self, dx, dgate, dup, dgate_bias, dup_bias):
        self.dx, self.dgate, self.dup, self.dgate_bias, self.dup_bias = dx, dgate, dup, dgate_bias, dup_bias


def gated_linear_backward(ctx, dy, x, gate, up, saved, act="silu", dx=True, dw=True, bias=False):
    """The gradients of gated_linear from dy, that of its output (m x n of x's
    type), its x, gate and up (16-bit tensors), act, and what it saved
    (hh_gated_linear_backward).  dx, dw (both weights'), bias (both): which are
    computed.  Returns GatedGrads."""
    what = "gated_linear_backward"
    if isinstance(gate, Int4Weight) or isinstance(up, Int4Weight):
        _refuse(UNSUPPORTED, f"{what}: 16-bit weights")
    m, n, k, dt, wt, code, held, strides, sizes = _gated_args(what, ctx, x, gate, up, act)
    dev = ctx.device
    if dy.dtype is not x.dtype:
        _refuse(INVALID_ARGUMENT, f"{what}: dy has x's type")
    dy_stride = _rows(dy, m, n, dev, "dy", what)
    if saved.dtype != torch.float32 or tuple(saved.shape) != (m, 2 * n) or not saved.is_contiguous():
        _refuse(INVALID_ARGUMENT, f"{what}: saved is what gated_linear gave, {m} x {2 * n}")
    _on(dev, what, saved)
    if dy.requires_grad or saved.requires_grad:
        _no_grad(what)
    gx = x.new_empty((m, k)) if dx else None
    gw = x.new_empty((2, n, k)).unbind(0) if dw else (None, None)
    gb = saved.new_empty((2, n)).unbind(0) if bias else (None, None)
    at = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    try:
        args = _GATED.pack(x.data_ptr(), held[0].data_ptr(), held[1].data_ptr(), 0, 0, 0, saved.data_ptr(), *strides, n, *sizes,
                           m, n, k, dt, wt, dt, code)
    except struct.error:
        _refuse(INVALID_ARGUMENT, f"{what}: {m} x {n} x {k}")
    rc = _gated_backward(ctx.handle, args, _GATED_GRADS.pack(dy.data_ptr(), at(gx), at(gw[0]), at(gw[1]), at(gb[0]), at(gb[1]),
                                                             dy_stride, k, k, k), _stream(dev))
    if rc:
        _check(rc, "hh_gated_linear_backward")
    return GatedGrads(gx, *gw, *gb)



class Plan:
    """What kv_plan gives: start, kv_len, slots, status, state (the free
    queue's next state)."""
    __slots__ = ("start", "kv_len", "slots", "status", "state")

    def __init__(self, start, kv_len, slots, status, state):
        self.start, self.kv_len, self.slots, self.status, self.state = start, kv_len, slots, status, state


def free_ring(num_blocks, device="cuda"):
    """The queue of free blocks of a new cache: (ring, state)."""
    return (torch.arange(num_blocks, dtype=torch.int32, device=device),
            torch.tensor([0, num_blocks], dtype=torch.int32, device=device))


def kv_plan(ctx, lens, new, table, ring, state, block_size, tokens):
    """One step's plan from request lengths (hh_kv_plan): int32 device tensors
    lens, new (requests), table (requests x width, updated), ring and state
    (the free queue; ring is updated, the next state returned).  tokens: room
    for the step's new rows."""
    requests, dev, shape = lens.numel(), ctx.device, table.shape
    _ints("kv_plan", lens, new, ring, state)
    if (table.dtype != torch.int32 or len(shape) != 2 or shape[0] != requests or new.shape != lens.shape or lens.dim() != 1
            or state.numel() != 2 or (requests and shape[1] > 1 and table.stride(1) != 1)):
        _refuse(INVALID_ARGUMENT, "kv_plan: lens and new per request, table requests x width, state of 2")
    _on(dev, "kv_plan", lens, new, table, ring, state)
    if not 0 <= tokens < 1 << 31 or not 0 <= block_size < 1 << 31:
        _refuse(INVALID_ARGUMENT, "kv_plan: sizes below 2^31")
    # one allocation: start, kv_len, status, state, slots
    buf = lens.new_empty(3 * requests + 3 + tokens)
    at = buf.data_ptr()
    rc = _plan(ctx.handle, _PLAN.pack(lens.data_ptr(), new.data_ptr(), table.data_ptr(), ring.data_ptr(), state.data_ptr(),
                                      at, at + 4 * requests + 4, at + 12 * requests + 12, at + 8 * requests + 4,
                                      at + 12 * requests + 4, table.stride(0) if requests > 1 else shape[1], requests,
                                      shape[1], ring.numel(), block_size, tokens), _stream(dev))
    if rc:
        _check(rc, "hh_kv_plan")
    start, kv_len, status, after, slots = buf.split_with_sizes((requests + 1, requests, requests, 2, tokens))
    return Plan(start, kv_len, slots, status, after)


class KvCache:
    """A paged 8-bit cache over its tensors: k uint8 (blocks, heads,
    block_size, dim), v uint8 (blocks, heads, dim, block_size), scales float32
    (blocks, heads); byte c stands for (c - 128) * scale."""

    def __init__(self, ctx, k, v, k_scale, v_scale):
        if k.dim() != 4:
            _refuse(INVALID_ARGUMENT, "KvCache: k is blocks x heads x block_size x dim")
        blocks, heads, block_size, dim = k.shape
        if k.dtype != torch.uint8 or v.dtype != torch.uint8 or k_scale.dtype != torch.float32 \
                or v_scale.dtype != torch.float32:
            _refuse(INVALID_ARGUMENT, "KvCache: uint8 codes and float32 scales")
        if tuple(v.shape) != (blocks, heads, dim, block_size) or tuple(k_scale.shape) != (blocks, heads) \
                or tuple(v_scale.shape) != (blocks, heads):
            _refuse(INVALID_ARGUMENT, "KvCache: shapes of v and the scales must match k's")
        if not all(t.is_contiguous() for t in (k, v, k_scale, v_scale)):
            _refuse(INVALID_ARGUMENT, "KvCache: contiguous tensors")
        _on(ctx.device, "KvCache", k, v, k_scale, v_scale)
        self.ctx, self.k, self.v, self.k_scale, self.v_scale = ctx, k, v, k_scale, v_scale
        self.num_blocks, self.kv_heads, self.block_size, self.head_dim = blocks, heads, block_size, dim
        self._c = _CACHE.pack(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), blocks, block_size,
                              heads, dim)

    @classmethod
    def create(cls, ctx, num_blocks, block_size, kv_heads, head_dim):
        """A new cache (its contents are written before they are read)."""
        dev = f"cuda:{ctx.device}"
        shape = (num_blocks, kv_heads)
        return cls(ctx, torch.empty(shape + (block_size, head_dim), dtype=torch.uint8, device=dev),
                   torch.empty(shape + (head_dim, block_size), dtype=torch.uint8, device=dev),
                   torch.empty(shape, dtype=torch.float32, device=dev),
                   torch.empty(shape, dtype=torch.float32, device=dev))

    def _heads(self, t, rows, heads, what):
        """Row and head strides of rows x heads x head_dim on the device."""
        shape, stride = t.shape, t.stride()
        if len(shape) != 3 or shape[0] != rows or shape[1] != heads or shape[2] != self.head_dim or (stride[2] != 1 and rows):
            _refuse(INVALID_ARGUMENT, f"{what}: {rows} x {heads} x {self.head_dim}, contiguous dimensions")
        if t.get_device() != self.ctx.device:
            _refuse(INVALID_ARGUMENT, f"{what} must be on the context's device")
        return stride[0], stride[1]

    def append(self, k, v, slots):
        """Rows k and v (rows x kv_heads x head_dim; any row and head strides)
        at slots (hh_kv_append)."""
        ctx, rows, dt = self.ctx, slots.numel(), _HALF.get(k.dtype)
        if dt is None:
            _refuse(UNSUPPORTED, f"append: {k.dtype} (float16 or bfloat16)")
        if k.requires_grad or v.requires_grad:
            _no_grad("append")
        tk, hk = self._heads(k, rows, self.kv_heads, "append: k")
        tv, hv = self._heads(v, rows, self.kv_heads, "append: v")
        if v.dtype is not k.dtype or slots.dim() != 1:
            _refuse(INVALID_ARGUMENT, "append: k, v and slots have the same rows, k and v the same type")
        _ints("append", slots)
        _on(ctx.device, "append", slots)
        rc = _append(ctx.handle, self._c, k.data_ptr(), v.data_ptr(), dt, tk, hk, tv, hv, slots.data_ptr(), rows,
                     _stream(ctx.device))
        if rc:
            _check(rc, "hh_kv_append")

    def read(self, blocks, dtype=torch.float32):
        """The values of whole blocks (int32 ids): k and v as n x block_size x
        kv_heads x head_dim of dtype (hh_kv_read)."""
        ctx, code = self.ctx, _CODE.get(dtype)
        if code is None:
            _refuse(UNSUPPORTED, f"read: {dtype}")
        _ints("read", blocks)
        _on(ctx.device, "read", blocks)
        n = blocks.numel()
        k, v = self.k_scale.new_empty((2, n, self.block_size, self.kv_heads, self.head_dim), dtype=dtype).unbind(0)
        rc = _read(ctx.handle, self._c, blocks.data_ptr(), n, code, k.data_ptr(), v.data_ptr(), _stream(ctx.device))
        if rc:
            _check(rc, "hh_kv_read")
        return k, v

    def _attention_args(self, what, q, table, start, kv_len, max_q, max_kv, scale, out):
        """The checks and arguments of an attention call: (out, packed)."""
        ctx, shape, dt = self.ctx, q.shape, _HALF.get(q.dtype)
        if dt is None:
            _refuse(UNSUPPORTED, f"{what}: {q.dtype} (float16 or bfloat16)")
        if len(shape) != 3:
            _refuse(INVALID_ARGUMENT, f"{what}: q is rows x q_heads x head_dim")
        if q.requires_grad or (out is not None and out.requires_grad):
            _no_grad(what)
        tokens, heads = shape[0], shape[1]
        tq, hq = self._heads(q, tokens, heads, f"{what}: q")
        if out is None:
            out = q.new_empty((tokens, heads, self.head_dim))
            to, ho = heads * self.head_dim, self.head_dim
        else:
            to, ho = self._heads(out, tokens, heads, f"{what}: out")
            if out.dtype is not q.dtype:
                _refuse(INVALID_ARGUMENT, f"{what}: out is like q")
        _ints(what, start, kv_len)
        requests, tshape, tstride = kv_len.numel(), table.shape, table.stride()
        if (kv_len.dim() != 1 or table.dtype != torch.int32 or len(tshape) != 2 or tshape[0] != requests or start.numel() != requests + 1
                or (requests and tshape[1] > 1 and tstride[1] != 1)):
            _refuse(INVALID_ARGUMENT, f"{what}: table requests x width, start requests + 1")
        _on(ctx.device, what, table, start, kv_len)
        width = tshape[1]
        try:
            args = _ATTENTION.pack(
                q.data_ptr(), out.data_ptr(), table.data_ptr(), start.data_ptr(), kv_len.data_ptr(), tq, hq, to, ho,
                tstride[0] if requests > 1 else width, requests, tokens, heads, width, tokens if max_q is None else max_q,
                min(width * self.block_size, 1 << 30) if max_kv is None else max_kv,
                scale, dt)
        except struct.error:
            _refuse(INVALID_ARGUMENT, f"{what}: max_q, max_kv and scale are numbers in range")
        return out, args

    def attention(self, q, table, start, kv_len, max_q=None, max_kv=None, scale=None, out=None):
        """softmax(scale q K^T) V of each request's new rows over its tokens
        (hh_kv_attention): q rows x q_heads x head_dim; table (requests x
        width), start and kv_len as kv_plan leaves them.  max_q and max_kv
        bound a request's rows and tokens (default: q's rows, the table's
        width; rows beyond give zeros, tokens beyond are not seen); scale defaults to head_dim ** -0.5."""
        out, args = self._attention_args("attention", q, table, start, kv_len, max_q, max_kv,
                                         self.head_dim ** -0.5 if scale is None else scale, out)
        rc = _attention(self.ctx.handle, self._c, args, _stream(self.ctx.device))
        if rc:
            _check(rc, "hh_kv_attention")
        return out

    def diff_attention(self, q, lam, table, start, kv_len, max_q=None, max_kv=None, scale=None, norm_weight=None, eps=1e-5,
                       gain=1.0, out=None):
        """Differential attention (hh_kv_diff_attention): a head's dimensions
        are two halves with a softmax map each,
        softmax(scale q1 K1^T) V - lam softmax(scale q2 K2^T) V over all of V's
        dimensions; with norm_weight (head_dim float32 values) the root mean
        square norm of each head's outputs times norm_weight, then times gain.
        lam: q_heads float32 values; scale defaults to (head_dim / 2) ** -0.5;
        out lies, from its first to its last element, apart from what is read;
        the rest as for attention."""
        what, ctx = "diff_attention", self.ctx
        if q.dim() != 3:
            _refuse(INVALID_ARGUMENT, f"{what}: q is rows x q_heads x head_dim")
        for t, n, name in ((lam, q.shape[1], "lam"), (norm_weight, self.head_dim, "norm_weight")):
            if t is None and name == "norm_weight":
                continue
            if t.dtype != torch.float32 or t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
                _refuse(INVALID_ARGUMENT, f"{what}: {name} is {n} contiguous float32 values")
            _on(ctx.device, what, t)
            if t.requires_grad:
                _no_grad(what)
        if out is not None and any(t is not None and not _spans_apart(out, t) for t in (q, lam, norm_weight, table, start, kv_len,
                                                                                       self.k, self.v, self.k_scale, self.v_scale)):
            _refuse(INVALID_ARGUMENT, f"{what}: out lies over what is read")
        out, args = self._attention_args(what, q, table, start, kv_len, max_q, max_kv,
                                         (self.head_dim / 2) ** -0.5 if scale is None else scale, out)
        try:
            diff = _DIFF.pack(lam.data_ptr(), 0 if norm_weight is None else norm_weight.data_ptr(), eps, gain)
        except (struct.error, OverflowError):
            _refuse(INVALID_ARGUMENT, f"{what}: eps and gain are numbers in range")
        rc = _diff_attention(ctx.handle, self._c, args, diff, _stream(ctx.device))
        if rc:
            _check(rc, "hh_kv_diff_attention")
        return out
