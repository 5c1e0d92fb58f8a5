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

CUDA tensors only, on the tensors' device and that device's current stream; every call can be captured into a CUDA graph and
none keeps anything between calls. Inputs that are not contiguous are copied. The 8-bit operators
have no gradient and refuse tensors that require one; none has a forward-mode derivative, and all refuse tensors that
carry a tangent. Checks, allocations and the C ABI call of each
operator are native (csrc/pyops.cpp, module ``dsmoe._ops``): there is no fallback if it is missing. It is
built for one PyTorch and loaded by the first call, so the rest of the package does not need it.
"""
import importlib
from typing import NamedTuple, Optional

import torch

from . import _lib as L


class _Native:
    """Stands in for the module until the first operator is called."""

    def __getattr__(self, name):
        global _ops
        if name.startswith("__"):  # whoever looks at objects in general
            raise AttributeError(name)
        try:
            native = importlib.import_module("._ops", __package__)
        except ImportError as e:
            raise ImportError(f"dsmoe.ops needs dsmoe/_ops.so, built for this PyTorch ({torch.__version__}): run make in csrc "
                              f"({e})") from e
        native.set_error_type(L.DsmoeError)
        _ops = native
        return getattr(native, name)


_ops = _Native()


class NormQuant(NamedTuple):
    q: torch.Tensor                   # 8-bit rows, the shape of x
    s: torch.Tensor                   # fp32 scales: [..., hidden / 128] (fp8) or [...] (int8)
    residual: Optional[torch.Tensor]  # x + residual, the new residual stream (None without residual)
    normed: Optional[torch.Tensor]    # the normed rows in x's dtype (None unless asked for)


class TokenOrder(NamedTuple):
    pos: torch.Tensor      # [tokens, k] int32: sorted row of each choice, -1 where it was dropped
    src: torch.Tensor      # [tokens * k] int32: choice (token * k + j) of each row, -1 behind the last
    offsets: torch.Tensor  # [n_experts + 1] int32: first row of each expert


def rms_norm_quant(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, *, eps: float = 1e-6,
                   fmt: str = "fp8", scale_fmt=None, normed: bool = False, inplace: bool = False) -> NormQuant:
    """r = x + residual (rounded to x's dtype); v = r / sqrt(mean(r^2) + eps) * weight; v to 8 bits.

    x, residual [..., hidden] bf16 or fp32 (hidden <= 16384), weight [hidden] bf16 or fp32. ``fmt`` "fp8":
    e4m3 with one scale per 128 values, ``act_quant``'s rule (``scale_fmt`` not None: power-of-2 scales), the
    input of ``fp8_gemm`` / ``fp4_gemm``. "int8": one scale per row, s = max(amax, 1e-4) / 127, the input of
    ``int8_gemm``. ``normed``: also v in x's dtype (the router's input). ``inplace``: the new residual is
    written over ``residual``, which must be contiguous.

    v is quantized from fp32; a scale is the quotient rounded once (``act_quant``'s, bit for bit, for the same v), a code
    v times the scale's reciprocal, rounded: beside a tie it may be the other neighbour of v / s. A row holding an infinity or NaN, or whose squares overflow fp32, has NaN scales."""
    return NormQuant._make(_ops.rms_norm_quant(x, weight, residual, eps, fmt, scale_fmt is not None, bool(normed),
                                               bool(inplace)))


def swiglu_quant(gu: torch.Tensor, row_weight: Optional[torch.Tensor] = None, *, limit: float = 10.0, fmt: str = "int8",
                 scale_fmt=None):
    """(q, s) of silu(min(g, limit)) * clamp(u, -limit, limit) * row_weight for gu [..., 2 * inter] = g | u.

    The activation of ``Expert`` (dsv41/tt/moe.py:133-139) between two 8-bit products; formats and scales
    as in ``rms_norm_quant``; a row (fp8: a block) whose amax is not finite has the scale NaN (a gate of -inf among them, as
    silu(-inf) is NaN; every finite one down to the type's lowest value gives its silu, 0). ``row_weight``
    [...] fp32 (e.g. routing weights) is applied before the quantization."""
    return _ops.swiglu_quant(gu, row_weight, limit, fmt, scale_fmt is not None)


def int8_gemm(a: torch.Tensor, a_s: torch.Tensor, b: torch.Tensor, b_s: torch.Tensor, out_dtype=None,
              out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """(a @ b^T) * a_s * b_s: a [..., K] int8 with one scale per token (a_s [...]), b [N, K] int8 with one per
    channel (b_s [N]), beside ``fp8_gemm`` / ``fp4_gemm``. The integer sum is exact; it is taken to fp32, times
    b_s, times a_s, and rounded to ``out_dtype`` (default: the default dtype, as there; bf16 or fp32). K is a
    multiple of 16, at most 131071. ``out``: contiguous, sharing no memory with the inputs."""
    return _ops.int8_product(a, a_s, b, b_s, None, out_dtype, out)


def int8_grouped_gemm(a: torch.Tensor, a_s: torch.Tensor, b: torch.Tensor, b_s: torch.Tensor, offsets: torch.Tensor,
                      out_dtype=None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``int8_gemm`` of each expert's rows: rows offsets[e]..offsets[e+1]-1 of a [rows, K] times b[e] of
    b [E, N, K], b_s [E, N]; offsets [E + 1] int32 on the GPU (``TokenOrder.offsets``). Rows at and behind
    offsets[E] come out as zeros; offsets that do not rise from 0 to at most rows give NaN throughout."""
    if offsets is None:
        raise TypeError("int8_grouped_gemm: offsets is required")
    return _ops.int8_product(a, a_s, b, b_s, offsets, out_dtype, out)


# ------------------------------------------------------------------ tokens to experts and back

def sort_tokens(idx: torch.Tensor, n_experts: int) -> TokenOrder:
    """The order of (expert, token, choice) of routing choices idx [tokens, k] int64 (``MoE.route``'s).

    Choices outside 0..n_experts-1 (e.g. -1 for padding) are dropped: their ``pos`` is -1, and the sorted
    rows behind offsets[n_experts] belong to nobody. Nothing is read back to the host."""
    return TokenOrder._make(_ops.sort_tokens(idx, n_experts))


def dispatch_tokens(x: torch.Tensor, order: TokenOrder, scales: Optional[torch.Tensor] = None):
    """xs [tokens * k, width]: row order.pos[t, j] is x[t]; rows behind the last are zero.

    x [tokens, width] of any dtype. With ``scales`` [tokens] fp32 (8-bit rows) returns (xs, scales of xs).
    The gradient of x (bf16 or fp32) is the sum of its rows' gradients, in fp32, in order of j. It can be captured
    into a CUDA graph; a capture beside a live eager graph of the same leaves is refused. Differentiable once."""
    return _ops.dispatch_tokens(x, order.pos, order.offsets, scales)


def combine_tokens(ys: torch.Tensor, order: TokenOrder, wt: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y [tokens, width] = sum over j of wt[t, j] * ys[order.pos[t, j]]: summed in fp32 in order of j, rounded
    once to ys's dtype (bf16 or fp32). Dropped choices add nothing. wt [tokens, k] fp32, None: ones.

    Differentiable (once) in ys (rows behind the last get zero) and wt; captures as in ``dispatch_tokens``."""
    return _ops.combine_tokens(ys, order.pos, order.offsets, wt)
