"""A decoder layer's operators on decoded weights (hh_linear, hh_kv_*): matrix
products with their epilogue, over 16-bit weights or INT4 buffers, and a
paged 8-bit key / value cache with its plan, append, read and attention.

Tensors are torch tensors on the context's device.  Calls run on torch's
current stream, where their results are allocated, and don't synchronise.
Calls on several streams need no order but their tensors' own; captured calls
keep what they use of the context's memory for as long as the context lives, whatever is called later (graphs
captured on one stream must not run beside each other).
What a call can't take raises HaagentiError before anything is launched;
there are no gradients, so tensors that require them are taken under
torch.no_grad() only."""
import ctypes as C
import struct

import torch

from . import BF16, F16, F32, INVALID_ARGUMENT, UNSUPPORTED, HaagentiError, _check, _i32, _sig, _u32, _vp

INT4 = 16

ACTIVATIONS = {"none": 0, None: 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
_CODE = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
_HALF = {torch.float16: F16, torch.bfloat16: BF16}

# The argument structures, packed as the header lays them out (natural
# alignment, no gaps; a step's calls are a few microseconds each, and a packed
# string costs a quarter of a ctypes structure).
_LINEAR = struct.Struct("=6Q6Q3I4i4x")      # hh_linear_args
_CACHE = struct.Struct("=4Q4I")             # hh_kv_cache
_PLAN = struct.Struct("=10QQ5I4x")          # hh_kv_plan_args
_ATTENTION = struct.Struct("=5Q5Q6Ifi")     # hh_kv_attention_args

_u64, _bytes = C.c_uint64, C.c_char_p
_linear = _sig("hh_linear", _i32, [_vp, _bytes, _vp])
_plan = _sig("hh_kv_plan", _i32, [_vp, _bytes, _vp])
_append = _sig("hh_kv_append", _i32, [_vp, _bytes, _vp, _vp, _i32, _u64, _u64, _u64, _u64, _vp, _u32, _vp])
_read = _sig("hh_kv_read", _i32, [_vp, _bytes, _vp, _u32, _i32, _vp, _vp, _vp])
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


def _rows(t, m, n, dev, what):
    """Row stride of an m x n matrix on the device whose rows are contiguous."""
    shape, stride = t.shape, t.stride()
    if len(shape) != 2 or shape[0] != m or shape[1] != n or (n > 1 and stride[1] != 1 and m):
        _refuse(INVALID_ARGUMENT, f"linear: {what} is {m} x {n} with contiguous rows, got {tuple(shape)}")
    if t.get_device() != dev:
        _refuse(INVALID_ARGUMENT, f"linear: {what} must be on the context's device")
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

    def attention(self, q, table, start, kv_len, max_q=None, max_kv=None, scale=None, out=None):
        """softmax(scale q K^T) V of each request's new rows over its tokens
        (hh_kv_attention): q rows x q_heads x head_dim; table (requests x
        width), start and kv_len as kv_plan leaves them.  max_q and max_kv
        bound a request's rows and tokens (default: q's rows, the table's
        width; rows beyond give zeros, tokens beyond are not seen); scale defaults to head_dim ** -0.5."""
        ctx, shape, dt = self.ctx, q.shape, _HALF.get(q.dtype)
        if dt is None:
            _refuse(UNSUPPORTED, f"attention: {q.dtype} (float16 or bfloat16)")
        if len(shape) != 3:
            _refuse(INVALID_ARGUMENT, "attention: q is rows x q_heads x head_dim")
        if q.requires_grad or (out is not None and out.requires_grad):
            _no_grad("attention")
        tokens, heads = shape[0], shape[1]
        tq, hq = self._heads(q, tokens, heads, "attention: q")
        if out is None:
            out = q.new_empty((tokens, heads, self.head_dim))
            to, ho = heads * self.head_dim, self.head_dim
        else:
            to, ho = self._heads(out, tokens, heads, "attention: out")
            if out.dtype is not q.dtype:
                _refuse(INVALID_ARGUMENT, "attention: out is like q")
        _ints("attention", start, kv_len)
        requests, tshape, tstride = kv_len.numel(), table.shape, table.stride()
        if (kv_len.dim() != 1 or table.dtype != torch.int32 or len(tshape) != 2 or tshape[0] != requests or start.numel() != requests + 1
                or (requests and tshape[1] > 1 and tstride[1] != 1)):
            _refuse(INVALID_ARGUMENT, "attention: table requests x width, start requests + 1")
        _on(ctx.device, "attention", table, start, kv_len)
        width = tshape[1]
        try:
            args = _ATTENTION.pack(
                q.data_ptr(), out.data_ptr(), table.data_ptr(), start.data_ptr(), kv_len.data_ptr(), tq, hq, to, ho,
                tstride[0] if requests > 1 else width, requests, tokens, heads, width, tokens if max_q is None else max_q,
                min(width * self.block_size, 1 << 30) if max_kv is None else max_kv,
                self.head_dim ** -0.5 if scale is None else scale, dt)
        except struct.error:
            _refuse(INVALID_ARGUMENT, "attention: max_q, max_kv and scale are numbers in range")
        rc = _attention(ctx.handle, self._c, args, _stream(ctx.device))
        if rc:
            _check(rc, "hh_kv_attention")
        return out
