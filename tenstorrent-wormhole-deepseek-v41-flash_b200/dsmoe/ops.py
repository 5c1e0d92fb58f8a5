"""8-bit operators around the expert products, and tokens to experts and back.

What stands between a layer's residual stream and its quantized products, beside the kernel surface's
``act_quant`` / ``fp8_gemm`` / ``fp4_gemm`` and the fused layer (``MoE``), which keeps these steps inside
its kernels:

* ``rms_norm_quant``      residual added, RMS norm, 8-bit rows with scales (e4m3 per 128, or int8 per row)
* ``int8_gemm``           product of int8 rows, one scale for each token and channel
* ``int8_grouped_gemm``   the same with every expert's weights over rows sorted by expert
* ``swiglu_quant``        the expert FFN's activation to 8-bit rows, between two such products
* ``sort_tokens``, ``dispatch_tokens``, ``combine_tokens``   tokens sorted by expert and back, with the
  gradients of tokens, expert rows and weights

CUDA tensors only, on the tensors' current stream; every call can be captured into a CUDA graph and
none keeps anything between calls. Inputs that are not contiguous are copied. The 8-bit operators
have no gradient and refuse tensors that require one.
"""
from typing import NamedTuple, Optional

import torch

from . import _lib as L

BLOCK = 128        # values per e4m3 scale
MAX_EXPERTS = 1024
MAX_TOPK = 64
MAX_ROW = 16384    # values per row of rms_norm_quant / swiglu_quant
MAX_K = 131071     # int8 products summed exactly in 32 bits

_FLOATS = {torch.float32: L.DTYPE_F32, torch.bfloat16: L.DTYPE_BF16}
_FMTS = {"fp8": (L.DTYPE_E4M3, torch.float8_e4m3fn), "int8": (L.DTYPE_I8, torch.int8)}


class NormQuant(NamedTuple):
    q: torch.Tensor                   # 8-bit rows, the shape of x
    s: torch.Tensor                   # fp32 scales: [..., hidden / 128] (fp8) or [...] (int8)
    residual: Optional[torch.Tensor]  # x + residual, the new residual stream (None without residual)
    normed: Optional[torch.Tensor]    # the normed rows in x's dtype (None unless asked for)


class TokenOrder(NamedTuple):
    pos: torch.Tensor      # [tokens, k] int32: sorted row of each choice, -1 where it was dropped
    src: torch.Tensor      # [tokens * k] int32: choice (token * k + j) of each row, -1 behind the last
    offsets: torch.Tensor  # [n_experts + 1] int32: first row of each expert


# Small calls are bound by the host, so the checks below are few and flat, and outputs are allocated by the
# cheapest form for their shape (on the host of a B200 box: empty_like 1.3 us, new_empty with sizes 1.4 us,
# torch.empty with a shape tuple and a device 2.5 us; the stream's raw handle 0.1 us, as an object 1.3 us).
_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else \
    lambda i: torch.cuda.current_stream(i).cuda_stream


def _call(fn, t: torch.Tensor, *args) -> None:
    """The entry point on t's device and that device's current stream."""
    i = t.get_device()
    if torch.cuda.current_device() == i:
        rc = fn(*args, _stream(i))
    else:
        with torch.cuda.device(i):
            rc = fn(*args, _stream(i))
    if rc:
        L.check(rc)


def _same_device(*ts) -> None:
    i = ts[0].get_device()
    for t in ts:
        if t is not None:
            j = t.get_device()
            if j < 0 or not t.is_cuda:
                raise ValueError("dsmoe kernels take CUDA tensors only")
            if j != i:
                raise ValueError(f"tensors on {ts[0].device} and {t.device}")


def _no_grad(name: str, *ts) -> None:
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                raise ValueError(f"{name} has no gradient: detach its inputs or call it under torch.no_grad()")


def _dense(t: torch.Tensor) -> torch.Tensor:
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _want(name: str, t: torch.Tensor, what: str, dtype, shape) -> None:
    if t.dtype != dtype:
        raise TypeError(f"{name}: {what} must be {dtype}, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name}: {what} must be {list(shape)}, got {list(t.shape)}")


def _quant_out(name: str, fmt: str, scale_fmt, like: torch.Tensor, n: int):
    """(dtype code, codes [..., n], scales) for rows of ``like`` [..., *]."""
    if fmt not in _FMTS:
        raise ValueError(f"{name}: fmt must be one of {sorted(_FMTS)}, got {fmt!r}")
    if scale_fmt is not None and fmt != "fp8":
        raise ValueError(f"{name}: power-of-2 scales (scale_fmt) are for fmt 'fp8'")
    if not 0 < n <= MAX_ROW:
        raise ValueError(f"{name}: rows of {n} values (1..{MAX_ROW})")
    if fmt == "fp8" and n % BLOCK:
        raise ValueError(f"{name}: fmt 'fp8' needs rows of a multiple of {BLOCK} values, got {n}")
    code, dtype = _FMTS[fmt]
    lead = like.shape[:-1]
    if like.shape[-1] == n:
        q = torch.empty_like(like, dtype=dtype, memory_format=torch.contiguous_format)
    else:
        q = like.new_empty(*lead, n, dtype=dtype)
    if fmt == "fp8":
        return code, q, like.new_empty(*lead, n // BLOCK, dtype=torch.float32)
    return code, q, like.new_empty(lead, dtype=torch.float32)


def rms_norm_quant(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, *, eps: float = 1e-6,
                   fmt: str = "fp8", scale_fmt=None, normed: bool = False, inplace: bool = False) -> NormQuant:
    """r = x + residual (rounded to x's dtype); v = r / sqrt(mean(r^2) + eps) * weight; v to 8 bits.

    x, residual [..., hidden] bf16 or fp32, weight [hidden] bf16 or fp32. ``fmt`` "fp8": e4m3 with one
    scale per 128 values, ``act_quant``'s rule (``scale_fmt`` not None: power-of-2 scales), the input of
    ``fp8_gemm`` / ``fp4_gemm``. "int8": one scale per row, s = max(amax, 1e-4) / 127, the input of
    ``int8_gemm``. ``normed``: also v in x's dtype (the router's input). ``inplace``: the new residual is
    written over ``residual``, which must be contiguous.

    v is quantized from fp32. A row (fp8: a block of 128) holding an infinity or NaN has the scale NaN."""
    name = "rms_norm_quant"
    _same_device(x, weight, residual)
    _no_grad(name, x, weight, residual)
    if x.dtype not in _FLOATS or weight.dtype not in _FLOATS:
        raise TypeError(f"{name}: x and weight must be bfloat16 or float32, got {x.dtype}, {weight.dtype}")
    if x.dim() < 1:
        raise ValueError(f"{name}: x must be [..., hidden]")
    h = x.shape[-1]
    _want(name, weight, "weight", weight.dtype, (h,))
    if residual is not None:
        _want(name, residual, "residual", x.dtype, x.shape)
    if inplace and (residual is None or not residual.is_contiguous()):
        raise ValueError(f"{name}: inplace needs a contiguous residual")
    code, q, s = _quant_out(name, fmt, scale_fmt, x, h)
    x, weight = _dense(x), _dense(weight)
    out = keep = None
    if residual is not None:
        keep, residual = residual, _dense(residual)
        out = residual if inplace else torch.empty_like(residual)
    y = torch.empty_like(x) if normed else None
    if x.numel():
        _call(L.lib.dsmoe_rms_norm_quant, x, x.data_ptr(), _FLOATS[x.dtype], L.ptr(residual), weight.data_ptr(),
              _FLOATS[weight.dtype], x.numel() // h, h, eps, code, 1 if scale_fmt is not None else 0, q.data_ptr(),
              s.data_ptr(), L.ptr(out), L.ptr(y))
        if inplace and out is not keep and out.data_ptr() != keep.data_ptr():  # it was not 16-byte aligned
            keep.copy_(out)
    return NormQuant(q, s, keep if inplace else out, y)


def swiglu_quant(gu: torch.Tensor, row_weight: Optional[torch.Tensor] = None, *, limit: float = 10.0, fmt: str = "int8",
                 scale_fmt=None):
    """(q, s) of silu(min(g, limit)) * clamp(u, -limit, limit) * row_weight for gu [..., 2 * inter] = g | u.

    The activation of ``Expert`` (dsv41/tt/moe.py:133-139) between two 8-bit products; formats and scales
    as in ``rms_norm_quant``. ``row_weight`` [...] fp32 (e.g. routing weights) is applied before the
    quantization."""
    name = "swiglu_quant"
    _same_device(gu, row_weight)
    _no_grad(name, gu, row_weight)
    if gu.dtype not in _FLOATS:
        raise TypeError(f"{name}: gu must be bfloat16 or float32, got {gu.dtype}")
    if gu.dim() < 1 or gu.shape[-1] % 2:
        raise ValueError(f"{name}: gu must be [..., 2 * inter], got {list(gu.shape)}")
    if not limit > 0:
        raise ValueError(f"{name}: limit must be positive, got {limit}")
    if row_weight is not None:
        _want(name, row_weight, "row_weight", torch.float32, gu.shape[:-1])
        row_weight = row_weight.contiguous()
    n = gu.shape[-1] // 2
    code, q, s = _quant_out(name, fmt, scale_fmt, gu, n)
    gu = _dense(gu)
    if gu.numel():
        _call(L.lib.dsmoe_swiglu_quant, gu, gu.data_ptr(), _FLOATS[gu.dtype], L.ptr(row_weight), gu.numel() // (2 * n), n,
              limit, code, 1 if scale_fmt is not None else 0, q.data_ptr(), s.data_ptr())
    return q, s


def _product(name: str, a, a_s, b, b_s, offsets, out_dtype, out):
    _no_grad(name, a_s, b_s, out)
    if a.dtype != torch.int8 or b.dtype != torch.int8:
        raise TypeError(f"{name}: a and b must be int8, got {a.dtype}, {b.dtype}")
    K = a.shape[-1] if a.dim() else 0
    N = b.shape[-2]
    if b.shape[-1] != K or not 0 < K <= MAX_K or K % 16:
        raise ValueError(f"{name}: a {list(a.shape)} and b {list(b.shape)} need one K, a multiple of 16, at most {MAX_K}")
    _want(name, a_s, "a_s", torch.float32, a.shape[:-1])
    _want(name, b_s, "b_s", torch.float32, b.shape[:-1])
    shape = (*a.shape[:-1], N)
    if out is not None:
        if out_dtype is not None and out_dtype != out.dtype:
            raise TypeError(f"{name}: out is {out.dtype}, out_dtype {out_dtype}")
        out_dtype = out.dtype
        if out.shape != shape or not out.is_contiguous():
            raise ValueError(f"{name}: out must be a contiguous {list(shape)} tensor")
    elif out_dtype is None:
        out_dtype = torch.get_default_dtype()
    if out_dtype not in _FLOATS:
        raise TypeError(f"{name}: output dtype must be bfloat16 or float32, got {out_dtype}")
    if out is None:
        out = a_s.new_empty(*shape, dtype=out_dtype)
    M = a.numel() // K
    if M and N:
        a, b, a_s, b_s = _dense(a), _dense(b), a_s.contiguous(), b_s.contiguous()
        if offsets is None:
            _call(L.lib.dsmoe_int8_gemm, a, a.data_ptr(), a_s.data_ptr(), M, K, b.data_ptr(), b_s.data_ptr(), N,
                  out.data_ptr(), _FLOATS[out_dtype])
        else:
            _call(L.lib.dsmoe_int8_grouped_gemm, a, a.data_ptr(), a_s.data_ptr(), M, K, b.data_ptr(), b_s.data_ptr(),
                  b.shape[0], N, offsets.data_ptr(), out.data_ptr(), _FLOATS[out_dtype])
    return out


def int8_gemm(a: torch.Tensor, a_s: torch.Tensor, b: torch.Tensor, b_s: torch.Tensor, out_dtype=None,
              out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """(a @ b^T) * a_s * b_s: a [..., K] int8 with one scale per token (a_s [...]), b [N, K] int8 with one per
    channel (b_s [N]), beside ``fp8_gemm`` / ``fp4_gemm``. The integer sum is exact; the product with the
    scales is rounded once to ``out_dtype`` (default: the default dtype, as there; bf16 or fp32). K is a
    multiple of 16."""
    _same_device(a, a_s, b, b_s, out)
    if b.dim() != 2:
        raise ValueError(f"int8_gemm: b must be [N, K], got {list(b.shape)}")
    return _product("int8_gemm", a, a_s, b, b_s, None, out_dtype, out)


def int8_grouped_gemm(a: torch.Tensor, a_s: torch.Tensor, b: torch.Tensor, b_s: torch.Tensor, offsets: torch.Tensor,
                      out_dtype=None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``int8_gemm`` of each expert's rows: rows offsets[e]..offsets[e+1]-1 of a [rows, K] times b[e] of
    b [E, N, K], b_s [E, N]; offsets [E + 1] int32 on the GPU (``TokenOrder.offsets``). Rows at and behind
    offsets[E] come out as zeros; offsets that do not rise from 0 to at most rows give NaN throughout."""
    name = "int8_grouped_gemm"
    _same_device(a, a_s, b, b_s, offsets, out)
    if b.dim() != 3 or a.dim() != 2:
        raise ValueError(f"{name}: a must be [rows, K] and b [E, N, K], got {list(a.shape)}, {list(b.shape)}")
    if not 0 < b.shape[0] <= MAX_EXPERTS:
        raise ValueError(f"{name}: {b.shape[0]} experts (1..{MAX_EXPERTS})")
    _want(name, offsets, "offsets", torch.int32, (b.shape[0] + 1,))
    return _product(name, a, a_s, b, b_s, offsets.contiguous(), out_dtype, out)


# ------------------------------------------------------------------ tokens to experts and back

def sort_tokens(idx: torch.Tensor, n_experts: int) -> TokenOrder:
    """The order of (expert, token, choice) of routing choices idx [tokens, k] int64 (``MoE.route``'s).

    Choices outside 0..n_experts-1 (e.g. -1 for padding) are dropped: their ``pos`` is -1, and the sorted
    rows behind offsets[n_experts] belong to nobody. Nothing is read back to the host."""
    _same_device(idx)
    if idx.dtype != torch.int64 or idx.dim() != 2:
        raise TypeError(f"sort_tokens: idx must be [tokens, k] int64, got {list(idx.shape)} {idx.dtype}")
    P, k = idx.shape
    if not 0 < k <= MAX_TOPK:
        raise ValueError(f"sort_tokens: {k} choices per token (1..{MAX_TOPK})")
    if not 0 < n_experts <= MAX_EXPERTS:
        raise ValueError(f"sort_tokens: {n_experts} experts (1..{MAX_EXPERTS})")
    idx = idx.contiguous()
    pos = torch.empty_like(idx, dtype=torch.int32)
    src = idx.new_empty(P * k, dtype=torch.int32)
    if P == 0:
        return TokenOrder(pos, src, idx.new_zeros(n_experts + 1, dtype=torch.int32))
    offsets = idx.new_empty(n_experts + 1, dtype=torch.int32)
    _call(L.lib.dsmoe_sort_tokens, idx, idx.data_ptr(), P, k, n_experts, pos.data_ptr(), src.data_ptr(), offsets.data_ptr())
    return TokenOrder(pos, src, offsets)


def _check_order(name: str, order: TokenOrder) -> None:
    pos, _, offsets = order
    if pos.dtype != torch.int32 or offsets.dtype != torch.int32 or pos.dim() != 2 or offsets.dim() != 1 \
            or not pos.is_contiguous() or not offsets.is_contiguous() or not 1 <= pos.shape[1] <= MAX_TOPK \
            or not 2 <= offsets.shape[0] <= MAX_EXPERTS + 1:
        raise ValueError(f"{name}: order must come from sort_tokens")


def _eager_leaf(name: str, *ts):
    """A gradient captured into a CUDA graph must not reach a leaf whose accumulation node belongs to a
    live eager graph: autograd runs that node on the stream it was made on, outside the capture. The
    node carries a mark from the eager call, so that the captured call can refuse. Returns the nodes,
    which live only as long as something holds them: hold them until the call's own graph does."""
    capturing = torch.cuda.is_current_stream_capturing()
    nodes = []
    for t in ts:
        if t is not None and t.requires_grad and t.is_leaf:
            node = torch.autograd.graph.get_gradient_edge(t).node
            nodes.append(node)
            if not capturing:
                node.metadata["dsmoe_eager"] = True
            elif node.metadata.get("dsmoe_eager"):
                raise RuntimeError(f"{name}: an eager graph of this leaf is still alive; delete its outputs before "
                                   "capturing a backward pass")
    return nodes


def _dispatch(x, pos, offsets, scales):
    P, k = pos.shape
    n = P * k
    x = x.contiguous()
    xs = x.new_empty(n, x.shape[1])
    ss = None
    if scales is not None:
        scales = scales.contiguous()
        ss = scales.new_empty(n)
    if n:
        _call(L.lib.dsmoe_dispatch_rows, x, x.data_ptr(), L.ptr(scales), pos.data_ptr(), offsets.data_ptr(),
              offsets.shape[0] - 1, P, k, x.shape[1] * x.element_size(), xs.data_ptr(), L.ptr(ss))
    return xs, ss


def _combine(ys, pos, wt):
    P, k = pos.shape
    ys = ys.contiguous()
    y = ys.new_empty(P, ys.shape[1])
    if P:
        _call(L.lib.dsmoe_combine_rows, ys, ys.data_ptr(), _FLOATS[ys.dtype], pos.data_ptr(), L.ptr(wt), P, k, ys.shape[1],
              y.data_ptr())
    return y


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, pos, offsets):
        ctx.save_for_backward(pos)
        return _dispatch(x, pos, offsets, None)[0]

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dxs):
        return _combine(dxs, ctx.saved_tensors[0], None), None, None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ys, pos, offsets, wt):
        ctx.save_for_backward(ys if ctx.needs_input_grad[3] else None, pos, offsets, wt)
        return _combine(ys, pos, wt)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        ys, pos, offsets, wt = ctx.saved_tensors
        P, k = pos.shape
        dy = dy.contiguous()
        H = dy.shape[1]
        dys = dy.new_empty(P * k, H) if ctx.needs_input_grad[0] else None
        dwt = dy.new_empty(P, k, dtype=torch.float32) if ctx.needs_input_grad[3] else None
        if P:
            ys = ys.contiguous() if ys is not None else None
            _call(L.lib.dsmoe_combine_grad, dy, dy.data_ptr(), L.ptr(ys), _FLOATS[dy.dtype], pos.data_ptr(), L.ptr(wt),
                  offsets.data_ptr(), offsets.shape[0] - 1, P, k, H, L.ptr(dys), L.ptr(dwt))
        return dys, None, None, dwt


def dispatch_tokens(x: torch.Tensor, order: TokenOrder, scales: Optional[torch.Tensor] = None):
    """xs [tokens * k, width]: row order.pos[t, j] is x[t]; rows behind the last are zero.

    x [tokens, width] of any dtype. With ``scales`` [tokens] fp32 (8-bit rows) returns (xs, scales of xs).
    The gradient of x (bf16 or fp32) is the sum of its rows' gradients, in fp32, in order of j."""
    name = "dispatch_tokens"
    _same_device(x, order.pos, order.offsets, scales)
    _check_order(name, order)
    if x.dim() != 2 or x.shape[0] != order.pos.shape[0] or x.shape[1] == 0:
        raise ValueError(f"{name}: x must be [{order.pos.shape[0]}, width], got {list(x.shape)}")
    if scales is not None:
        _want(name, scales, "scales", torch.float32, x.shape[:1])
        _no_grad(name, x, scales)
        return _dispatch(x, order.pos, order.offsets, scales)
    if torch.is_grad_enabled() and x.requires_grad:
        if x.dtype not in _FLOATS:
            raise TypeError(f"{name}: a gradient needs bfloat16 or float32, got {x.dtype}")
        nodes = _eager_leaf(name, x)  # noqa: F841  (held over the call)
        return _Dispatch.apply(x, order.pos, order.offsets)
    return _dispatch(x, order.pos, order.offsets, None)[0]


def combine_tokens(ys: torch.Tensor, order: TokenOrder, wt: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y [tokens, width] = sum over j of wt[t, j] * ys[order.pos[t, j]]: summed in fp32 in order of j, rounded
    once to ys's dtype (bf16 or fp32). Dropped choices add nothing. wt [tokens, k] fp32, None: ones.

    Differentiable in ys (rows behind the last get zero) and wt."""
    name = "combine_tokens"
    _same_device(ys, order.pos, order.offsets, wt)
    _check_order(name, order)
    if ys.dtype not in _FLOATS:
        raise TypeError(f"{name}: ys must be bfloat16 or float32, got {ys.dtype}")
    n = order.pos.numel()
    if ys.dim() != 2 or ys.shape[0] != n or ys.shape[1] == 0:
        raise ValueError(f"{name}: ys must be [{n}, width], got {list(ys.shape)}")
    if wt is not None:
        _want(name, wt, "wt", torch.float32, order.pos.shape)
    if torch.is_grad_enabled() and (ys.requires_grad or (wt is not None and wt.requires_grad)):
        nodes = _eager_leaf(name, ys, wt)  # noqa: F841  (held over the call)
        return _Combine.apply(ys, order.pos, order.offsets, wt if wt is None else wt.contiguous())
    return _combine(ys, order.pos, wt if wt is None else wt.contiguous())
