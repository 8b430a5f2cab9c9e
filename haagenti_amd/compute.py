"""A decoder layer's operators on decoded weights (hh_linear, hh_kv_*): matrix
products with their epilogue, over 16-bit weights or INT4 buffers, and a
paged 8-bit key / value cache with its plan, append, read and attention.

Tensors are torch tensors on the context's device.  Calls run on torch's
current stream, where their results are allocated, and don't synchronise.
What a call can't take raises HaagentiError before anything is launched."""
import ctypes as C

import torch

from . import BF16, F16, F32, INVALID_ARGUMENT, UNSUPPORTED, HaagentiError, _check, _i32, _sig, _sz, _u32, _vp

_u64 = C.c_uint64
INT4 = 16

ACTIVATIONS = {"none": 0, None: 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
_CODE = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}


class _LinearArgs(C.Structure):
    _fields_ = ([(n, _vp) for n in ("d_x", "d_w", "d_bias", "d_mul", "d_residual", "d_y")]
                + [(n, _u64) for n in ("x_stride", "w_stride", "mul_stride", "residual_stride", "y_stride", "w_bytes")]
                + [(n, _u32) for n in ("m", "n", "k")]
                + [(n, _i32) for n in ("dtype", "w_dtype", "y_dtype", "activation")])


class _Cache(C.Structure):
    _fields_ = ([(n, _vp) for n in ("d_k", "d_v", "d_k_scale", "d_v_scale")]
                + [(n, _u32) for n in ("num_blocks", "block_size", "kv_heads", "head_dim")])


class _PlanArgs(C.Structure):
    _fields_ = ([(n, _vp) for n in ("d_len", "d_new", "d_table", "d_ring", "d_state", "d_start", "d_kv_len", "d_slots",
                                    "d_status", "d_state_out")]
                + [("table_stride", _u64)]
                + [(n, _u32) for n in ("requests", "table_width", "ring_capacity", "block_size", "tokens")])


class _AttentionArgs(C.Structure):
    _fields_ = ([(n, _vp) for n in ("d_q", "d_out", "d_table", "d_start", "d_kv_len")]
                + [(n, _u64) for n in ("q_token_stride", "q_head_stride", "out_token_stride", "out_head_stride",
                                       "table_stride")]
                + [(n, _u32) for n in ("requests", "tokens", "q_heads", "table_width", "max_q", "max_kv")]
                + [("scale", C.c_float), ("dtype", _i32)])


_linear = _sig("hh_linear", _i32, [_vp, C.POINTER(_LinearArgs), _vp])
_plan = _sig("hh_kv_plan", _i32, [_vp, C.POINTER(_PlanArgs), _vp])
_append = _sig("hh_kv_append", _i32, [_vp, C.POINTER(_Cache), _vp, _vp, _i32, _u64, _u64, _u64, _u64, _vp, _u32, _vp])
_read = _sig("hh_kv_read", _i32, [_vp, C.POINTER(_Cache), _vp, _u32, _i32, _vp, _vp, _vp])
_attention = _sig("hh_kv_attention", _i32, [_vp, C.POINTER(_Cache), C.POINTER(_AttentionArgs), _vp])


def _refuse(code, what):
    raise HaagentiError(code, what)


def _on(ctx, what, *tensors):
    for t in tensors:
        if t is not None and (not t.is_cuda or t.get_device() != ctx.device):
            _refuse(INVALID_ARGUMENT, f"{what}: tensors must be on the context's device")


def _stream(ctx):
    return torch.cuda.current_stream(ctx.device).cuda_stream


def _half(t, what):
    if t.dtype not in (torch.float16, torch.bfloat16):
        _refuse(UNSUPPORTED, f"{what}: {t.dtype} (float16 or bfloat16)")
    return _CODE[t.dtype]


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


def _rows(t, m, n, what):
    """Row stride of an m x n matrix whose rows are contiguous."""
    if t.dim() != 2 or t.shape[0] != m or t.shape[1] != n or (n > 1 and t.stride(1) != 1):
        _refuse(INVALID_ARGUMENT, f"{what}: {m} x {n} with contiguous rows, got {tuple(t.shape)}")
    return t.stride(0) if m > 1 else max(n, 1)


def linear(ctx, x, w, bias=None, act=None, mul=None, residual=None, out=None, out_dtype=None):
    """act(x w^T + bias) * mul + residual (hh_linear).  x: m x k, float16 or
    bfloat16; w: n x k of x's type, or an Int4Weight; bias n values, mul and
    residual m x n, of x's type.  act: a key of ACTIVATIONS.  Rows are
    contiguous, any stride apart.  Returns out (m x n of out_dtype, by default
    x's type; float32 is allowed), which may be residual or mul."""
    dt = _half(x, "linear")
    if x.dim() != 2:
        _refuse(INVALID_ARGUMENT, "linear: x is m x k")
    m, k = x.shape
    a = _LinearArgs()
    if isinstance(w, Int4Weight):
        n, wt = w.n, w.data
        if w.k != k:
            _refuse(INVALID_ARGUMENT, f"linear: x has {k} columns, the weight {w.k}")
        a.w_dtype, a.w_bytes = INT4, wt.numel()
    else:
        if w.dim() != 2 or w.dtype != x.dtype:
            _refuse(INVALID_ARGUMENT, "linear: w is n x k of x's type, or an Int4Weight")
        n, wt = w.shape[0], w
        a.w_dtype, a.w_stride = dt, _rows(w, n, k, "linear: w")
    if act not in ACTIVATIONS:
        _refuse(UNSUPPORTED, f"linear: activation {act!r}")
    if out is None:
        out = torch.empty((m, n), dtype=out_dtype or x.dtype, device=x.device)
    elif out_dtype is not None and out.dtype != out_dtype:
        _refuse(INVALID_ARGUMENT, "linear: out has another type than out_dtype")
    if out.dtype not in (x.dtype, torch.float32):
        _refuse(UNSUPPORTED, f"linear: output {out.dtype}")
    _on(ctx, "linear", x, wt, bias, mul, residual, out)
    a.x_stride, a.y_stride = _rows(x, m, k, "linear: x"), _rows(out, m, n, "linear: out")
    a.d_x, a.d_w, a.d_y = x.data_ptr(), wt.data_ptr(), out.data_ptr()
    if bias is not None:
        if bias.dim() != 1 or bias.shape[0] != n or bias.dtype != x.dtype or not bias.is_contiguous():
            _refuse(INVALID_ARGUMENT, "linear: bias is n contiguous values of x's type")
        a.d_bias = bias.data_ptr()
    if mul is not None:
        a.d_mul, a.mul_stride = mul.data_ptr(), _rows(mul, m, n, "linear: mul")
    if residual is not None:
        a.d_residual, a.residual_stride = residual.data_ptr(), _rows(residual, m, n, "linear: residual")
    for t in (mul, residual):
        if t is not None and t.dtype != x.dtype:
            _refuse(INVALID_ARGUMENT, "linear: mul and residual have x's type")
    a.m, a.n, a.k, a.dtype, a.y_dtype, a.activation = m, n, k, dt, _CODE[out.dtype], ACTIVATIONS[act]
    _check(_linear(ctx.handle, C.byref(a), _stream(ctx)), "hh_linear")
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
    requests = lens.shape[0]
    _ints("kv_plan", lens, new, ring, state)
    if (table.dtype != torch.int32 or table.dim() != 2 or (table.shape[1] > 1 and table.stride(1) != 1)
            or table.shape[0] != requests or new.shape != lens.shape or lens.dim() != 1 or state.numel() != 2):
        _refuse(INVALID_ARGUMENT, "kv_plan: lens and new per request, table requests x width, state of 2")
    _on(ctx, "kv_plan", lens, new, table, ring, state)
    tokens = int(tokens)
    # one allocation: start, kv_len, status, state, slots
    buf = torch.empty(3 * requests + 3 + tokens, dtype=torch.int32, device=lens.device)
    at = buf.data_ptr()
    a = _PlanArgs(lens.data_ptr(), new.data_ptr(), table.data_ptr(), ring.data_ptr(), state.data_ptr(), at,
                  at + 4 * (requests + 1), at + 4 * (3 * requests + 3), at + 4 * (2 * requests + 1),
                  at + 4 * (3 * requests + 1), table.stride(0) if requests > 1 else table.shape[1], requests,
                  table.shape[1], ring.numel(), int(block_size), tokens)
    _check(_plan(ctx.handle, C.byref(a), _stream(ctx)), "hh_kv_plan")
    start, kv_len, status, after, slots = buf.split_with_sizes([requests + 1, requests, requests, 2, tokens])
    return Plan(start, kv_len, slots, status, after)


class KvCache:
    """A paged 8-bit cache over its tensors: k uint8 (blocks, heads,
    block_size, dim), v uint8 (blocks, heads, dim, block_size), scales float32
    (blocks, heads); byte c stands for (c - 128) * scale."""

    def __init__(self, ctx, k, v, k_scale, v_scale):
        blocks, heads, block_size, dim = k.shape
        if k.dtype != torch.uint8 or v.dtype != torch.uint8 or k_scale.dtype != torch.float32 \
                or v_scale.dtype != torch.float32:
            _refuse(INVALID_ARGUMENT, "KvCache: uint8 codes and float32 scales")
        if tuple(v.shape) != (blocks, heads, dim, block_size) or tuple(k_scale.shape) != (blocks, heads) \
                or tuple(v_scale.shape) != (blocks, heads):
            _refuse(INVALID_ARGUMENT, "KvCache: shapes of v and the scales must match k's")
        if not all(t.is_contiguous() for t in (k, v, k_scale, v_scale)):
            _refuse(INVALID_ARGUMENT, "KvCache: contiguous tensors")
        _on(ctx, "KvCache", k, v, k_scale, v_scale)
        self.ctx, self.k, self.v, self.k_scale, self.v_scale = ctx, k, v, k_scale, v_scale
        self.num_blocks, self.kv_heads, self.block_size, self.head_dim = blocks, heads, block_size, dim
        self._c = _Cache(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), blocks, block_size, heads,
                         dim)
        self._p = C.byref(self._c)

    @classmethod
    def create(cls, ctx, num_blocks, block_size, kv_heads, head_dim):
        """A new cache (its contents are written before they are read)."""
        dev = f"cuda:{ctx.device}"
        shape = (num_blocks, kv_heads)
        return cls(ctx, torch.empty(shape + (block_size, head_dim), dtype=torch.uint8, device=dev),
                   torch.empty(shape + (head_dim, block_size), dtype=torch.uint8, device=dev),
                   torch.empty(shape, dtype=torch.float32, device=dev),
                   torch.empty(shape, dtype=torch.float32, device=dev))

    def _heads(self, t, heads, what):
        if t.dim() != 3 or t.shape[1] != heads or t.shape[2] != self.head_dim or t.stride(2) != 1:
            _refuse(INVALID_ARGUMENT, f"{what}: rows x {heads} x {self.head_dim}, contiguous dimensions")

    def append(self, k, v, slots):
        """Rows k and v (rows x kv_heads x head_dim; any row and head strides)
        at slots (hh_kv_append)."""
        self._heads(k, self.kv_heads, "append: k")
        self._heads(v, self.kv_heads, "append: v")
        dt = _half(k, "append")
        if v.dtype != k.dtype or v.shape[0] != k.shape[0] or slots.dim() != 1 or slots.shape[0] != k.shape[0]:
            _refuse(INVALID_ARGUMENT, "append: k, v and slots have the same rows, k and v the same type")
        _ints("append", slots)
        _on(self.ctx, "append", k, v, slots)
        _check(_append(self.ctx.handle, self._p, k.data_ptr(), v.data_ptr(), dt, k.stride(0), k.stride(1), v.stride(0),
                       v.stride(1), slots.data_ptr(), k.shape[0], _stream(self.ctx)), "hh_kv_append")

    def read(self, blocks, dtype=torch.float32):
        """The values of whole blocks (int32 ids): k and v as n x block_size x
        kv_heads x head_dim of dtype (hh_kv_read)."""
        if dtype not in _CODE:
            _refuse(UNSUPPORTED, f"read: {dtype}")
        _ints("read", blocks)
        _on(self.ctx, "read", blocks)
        n = blocks.numel()
        k, v = torch.empty((2, n, self.block_size, self.kv_heads, self.head_dim), dtype=dtype,
                           device=self.k.device).unbind(0)
        _check(_read(self.ctx.handle, self._p, blocks.data_ptr(), n, _CODE[dtype], k.data_ptr(), v.data_ptr(),
                     _stream(self.ctx)), "hh_kv_read")
        return k, v

    def attention(self, q, table, start, kv_len, max_q=None, max_kv=None, scale=None, out=None):
        """softmax(scale q K^T) V of each request's new rows over its tokens
        (hh_kv_attention): q rows x q_heads x head_dim; table (requests x
        width), start and kv_len as kv_plan leaves them.  max_q and max_kv
        bound a request's rows and tokens (default: q's rows, the table's
        width); scale defaults to head_dim ** -0.5."""
        dt = _half(q, "attention")
        if q.dim() != 3:
            _refuse(INVALID_ARGUMENT, "attention: q is rows x q_heads x head_dim")
        tokens, heads = q.shape[0], q.shape[1]
        self._heads(q, heads, "attention: q")
        if out is None:
            out = torch.empty((tokens, heads, self.head_dim), dtype=q.dtype, device=q.device)
        else:
            self._heads(out, heads, "attention: out")
            if out.dtype != q.dtype or out.shape[0] != tokens:
                _refuse(INVALID_ARGUMENT, "attention: out is like q")
        requests = kv_len.shape[0]
        _ints("attention", start, kv_len)
        if (table.dtype != torch.int32 or table.dim() != 2 or table.shape[0] != requests
                or (table.shape[1] > 1 and table.stride(1) != 1) or start.numel() != requests + 1):
            _refuse(INVALID_ARGUMENT, "attention: table requests x width, start requests + 1")
        _on(self.ctx, "attention", q, table, start, kv_len, out)
        width = table.shape[1]
        a = _AttentionArgs(q.data_ptr(), out.data_ptr(), table.data_ptr(), start.data_ptr(), kv_len.data_ptr(),
                           q.stride(0), q.stride(1), out.stride(0), out.stride(1),
                           table.stride(0) if requests > 1 else width, requests, tokens, heads, width,
                           tokens if max_q is None else int(max_q),
                           width * self.block_size if max_kv is None else int(max_kv),
                           self.head_dim ** -0.5 if scale is None else float(scale), dt)
        _check(_attention(self.ctx.handle, self._p, C.byref(a), _stream(self.ctx)), "hh_kv_attention")
        return out
