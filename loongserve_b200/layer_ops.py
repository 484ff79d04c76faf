"""Element-wise layer ops with the reference's names (the pybind functions of ``longserve_cuda_kernels``,
longserve_cuda_kernels/src/entrypoints.cpp:15-101): ``rms_norm``, ``rotary_emb``, ``silu_and_mul_inplace`` and the
host-level fusion ``ffn_block``.  Matrix products are cuBLAS through ``torch.mm`` as in the reference."""
from __future__ import annotations

import torch

from . import _lib
from ._util import dtype16_tag, dtype_tag, need_cuda, need_here, ptr, stream_of, stream_ptr


@torch.inference_mode()
def rms_norm(input: torch.Tensor, weight: torch.Tensor, eps: float, out=None) -> torch.Tensor:
    need_cuda(input, weight)
    assert input.dim() == 2 and weight.dim() == 1 and input.size(1) == weight.size(0)
    assert input.is_contiguous() and weight.is_contiguous() and weight.dtype == input.dtype
    output = torch.empty_like(input) if out is None else out
    rc = _lib.attn().esp_rms_norm(ptr(output), ptr(input), ptr(weight), input.size(0), input.size(1), float(eps),
                                  dtype_tag(input), stream_ptr())
    _lib.check(rc, "esp_rms_norm")
    return output


def _rotary_single(x, cos, sin):
    assert x.dim() == 3 and x.stride(2) == 1
    tokens, heads, head_dim = x.shape
    assert cos.shape == sin.shape == (tokens, head_dim // 2) and cos.is_contiguous() and sin.is_contiguous()
    assert cos.dtype == x.dtype and sin.dtype == x.dtype
    rc = _lib.attn().esp_rotary_emb(ptr(x), ptr(cos), ptr(sin), x.stride(0), x.stride(1), tokens, heads, head_dim,
                                    dtype_tag(x), stream_ptr())
    _lib.check(rc, "esp_rotary_emb")


@torch.inference_mode()
def rotary_emb(q: torch.Tensor, k: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> None:
    """In place on q and k (k may be the K half of a [tokens, 2*Hkv, D] cache view)."""
    need_cuda(q, k, cos, sin)
    _rotary_single(q, cos, sin)
    _rotary_single(k, cos, sin)


@torch.inference_mode()
def silu_and_mul_inplace(io: torch.Tensor) -> None:
    need_cuda(io)
    assert io.dim() == 2 and io.is_contiguous()
    rc = _lib.attn().esp_silu_and_mul_inplace(ptr(io), io.size(0), io.size(1) // 2, dtype_tag(io), stream_ptr())
    _lib.check(rc, "esp_silu_and_mul_inplace")


@torch.inference_mode()
def ffn_block(input_embds, norm_weight, norm_eps: float, gate_up_proj, down_proj) -> torch.Tensor:
    """rms_norm -> mm(gate_up) -> silu*mul -> mm(down), reusing the norm buffer as the output
    (entrypoints.cpp:89-101)."""
    input_normed = rms_norm(input_embds, norm_weight, norm_eps)
    up_gate_out = torch.mm(input_normed, gate_up_proj)
    silu_and_mul_inplace(up_gate_out)
    torch.mm(up_gate_out[:, : up_gate_out.size(-1) // 2], down_proj, out=input_normed)
    return input_normed


# ---------------------------------------------------------------------------------------- 8-bit rows
# A row of int8 codes has one fp32 scale: scale = max(max|y|, 2^-100) / 127, code = rint(y * fl32(127 / max|y|)).  A row with an
# infinity or a NaN gets codes 0 and scale NaN.
# (These wrappers stand in front of launches of a few microseconds: shapes are read once, and nothing is wrapped in a mode.)
def _rows_out(like, codes, scale, rows, cols):
    if codes is None:
        codes = like.new_empty((rows, cols), dtype=torch.int8)
    else:
        assert codes.shape == (rows, cols) and codes.dtype == torch.int8 and codes.is_contiguous()
    if scale is None:
        scale = like.new_empty(rows, dtype=torch.float32)
    else:
        assert scale.shape == (rows,) and scale.dtype == torch.float32 and scale.is_contiguous()
    return codes, scale


def _norm_args(input, residual, weight):
    """(tokens, hidden, dtype tag) of a norm's arguments."""
    shape = input.shape
    tokens, hidden = shape if len(shape) == 2 else (0, -1)
    assert hidden >= 0 and weight.shape == (hidden,), "expected input [tokens, hidden] and weight [hidden]"
    assert input.is_contiguous() and weight.is_contiguous() and weight.dtype == input.dtype
    if residual is not None:
        assert residual.shape == shape and residual.dtype == input.dtype and residual.is_contiguous()
    return tokens, hidden, dtype16_tag(input)


def add_rms_norm(input: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, eps: float, out=None) -> torch.Tensor:
    """residual += input (in place), and the RMSNorm of the sum.  The norm is taken of the fp32 sum before it is rounded into
    ``residual``; the output is rounded once."""
    dev = need_here(input, residual, weight, out)
    tokens, hidden, tag = _norm_args(input, residual, weight)
    if out is None:
        out = torch.empty_like(input)
    else:
        assert out.shape == input.shape and out.dtype == input.dtype and out.is_contiguous()
    rc = _lib.attn().esp_add_rms_norm(out.data_ptr(), residual.data_ptr(), input.data_ptr(), weight.data_ptr(), tokens, hidden, eps, tag,
                                      stream_of(dev))
    if rc:
        _lib.check(rc, "esp_add_rms_norm")
    return out


def add_rms_norm_quant(input: torch.Tensor, residual, weight: torch.Tensor, eps: float, out=None, out_scale=None):
    """``add_rms_norm`` whose output is int8 rows: (codes [tokens, hidden], scale [tokens]).  ``residual`` None: the norm of
    ``input`` alone."""
    dev = need_here(input, residual, weight, out, out_scale)
    tokens, hidden, tag = _norm_args(input, residual, weight)
    codes, scale = _rows_out(input, out, out_scale, tokens, hidden)
    rc = _lib.attn().esp_add_rms_norm_q8(codes.data_ptr(), scale.data_ptr(), ptr(residual), input.data_ptr(), weight.data_ptr(), tokens,
                                         hidden, eps, tag, stream_of(dev))
    if rc:
        _lib.check(rc, "esp_add_rms_norm_q8")
    return codes, scale


def silu_and_mul_quant(io: torch.Tensor, out=None, out_scale=None):
    """int8 rows of silu(io[:, :F]) * io[:, F:]: (codes [tokens, F], scale [tokens]).  ``io`` is left as it was."""
    dev = need_here(io, out, out_scale)
    shape = io.shape
    assert len(shape) == 2 and shape[1] % 2 == 0 and io.is_contiguous()
    tokens, ffn = shape[0], shape[1] // 2
    tag = dtype16_tag(io)
    codes, scale = _rows_out(io, out, out_scale, tokens, ffn)
    rc = _lib.attn().esp_silu_and_mul_q8(codes.data_ptr(), scale.data_ptr(), io.data_ptr(), tokens, ffn, tag, stream_of(dev))
    if rc:
        _lib.check(rc, "esp_silu_and_mul_q8")
    return codes, scale


def quantize_rows(x: torch.Tensor, out=None, out_scale=None):
    """int8 rows of x [rows, cols]: (codes, scale [rows]).  Also lays out weights for ``mm_w8a8``: ``quantize_rows(w.t().contiguous())``
    of a [in, out] weight gives its output channels as rows."""
    dev = need_here(x, out, out_scale)
    shape = x.shape
    assert len(shape) == 2 and x.stride(1) == 1
    rows, cols = shape
    tag = dtype16_tag(x)
    codes, scale = _rows_out(x, out, out_scale, rows, cols)
    rc = _lib.attn().esp_quantize_rows(codes.data_ptr(), scale.data_ptr(), x.data_ptr(), x.stride(0) if rows > 1 else cols, rows, cols, tag,
                                       stream_of(dev))
    if rc:
        _lib.check(rc, "esp_quantize_rows")
    return codes, scale


def dequantize_rows(codes: torch.Tensor, scale: torch.Tensor, dtype=torch.bfloat16, out=None) -> torch.Tensor:
    """codes * scale per row, rounded to ``dtype``."""
    dev = need_here(codes, scale, out)
    shape = codes.shape
    assert len(shape) == 2 and codes.dtype == torch.int8 and codes.is_contiguous()
    assert scale.shape == shape[:1] and scale.dtype == torch.float32 and scale.is_contiguous()
    if out is None:
        out = torch.empty_like(codes, dtype=dtype)
    else:
        assert out.shape == shape and out.is_contiguous()
    rc = _lib.attn().esp_dequantize_rows(out.data_ptr(), codes.data_ptr(), scale.data_ptr(), shape[0], shape[1], dtype_tag(out), stream_of(dev))
    if rc:
        _lib.check(rc, "esp_dequantize_rows")
    return out


def mm_w8a8(a: torch.Tensor, a_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, out_dtype=torch.bfloat16, out=None):
    """(a @ w.T) * a_scale[:, None] * w_scale[None]: int8 rows of tokens [M, K] and of output channels [N, K], exact integer sums,
    then fp32 (the sum, two products) and the rounding to the output type.  K a multiple of 16, at most 131071."""
    dev = need_here(a, a_scale, w, w_scale, out)
    sa, sw = a.shape, w.shape
    assert len(sa) == 2 and len(sw) == 2 and sa[1] == sw[1]
    if a.dtype != torch.int8 or w.dtype != torch.int8 or a_scale.dtype != torch.float32 or w_scale.dtype != torch.float32:
        raise TypeError("mm_w8a8 takes int8 codes and fp32 scales")
    (m, k), n = sa, sw[0]
    (la, ca), (lw, cw) = a.stride(), w.stride()
    assert ca == 1 and cw == 1
    assert a_scale.shape == (m,) and w_scale.shape == (n,) and a_scale.is_contiguous() and w_scale.is_contiguous()
    if out is None:
        out = a_scale.new_empty((m, n), dtype=out_dtype)
        lo = n
    else:
        assert out.shape == (m, n) and (n == 1 or out.stride(1) == 1)
        lo = out.stride(0) if m > 1 else n
    # a single row's stride says nothing
    rc = _lib.attn().esp_mm_w8a8(out.data_ptr(), lo, a.data_ptr(), la if m > 1 else k, a_scale.data_ptr(), w.data_ptr(),
                                 lw if n > 1 else k, w_scale.data_ptr(), m, n, k, dtype_tag(out), stream_of(dev))
    if rc:
        _lib.check(rc, "esp_mm_w8a8")
    return out
