"""Element-wise layer ops with the reference's names (the pybind functions of ``longserve_cuda_kernels``,
longserve_cuda_kernels/src/entrypoints.cpp:15-101): ``rms_norm``, ``rotary_emb``, ``silu_and_mul_inplace`` and the
host-level fusion ``ffn_block``.  Matrix products are cuBLAS through ``torch.mm`` as in the reference."""
from __future__ import annotations

import torch

from . import _lib
from ._util import dtype16_tag, dtype_tag, need_cuda, need_here, ptr, stream_ptr


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
def _rows_out(codes, scale, rows, cols, device):
    if codes is None:
        codes = torch.empty((rows, cols), dtype=torch.int8, device=device)
    if scale is None:
        scale = torch.empty((rows,), dtype=torch.float32, device=device)
    assert codes.shape == (rows, cols) and codes.dtype == torch.int8 and codes.is_contiguous()
    assert scale.shape == (rows,) and scale.dtype == torch.float32 and scale.is_contiguous()
    return codes, scale


def _norm_args(input, residual, weight):
    assert input.dim() == 2 and weight.dim() == 1 and input.size(1) == weight.size(0)
    assert input.is_contiguous() and weight.is_contiguous() and weight.dtype == input.dtype
    if residual is not None:
        assert residual.shape == input.shape and residual.dtype == input.dtype and residual.is_contiguous()


@torch.inference_mode()
def add_rms_norm(input: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, eps: float, out=None) -> torch.Tensor:
    """residual += input (in place), and the RMSNorm of the sum.  The norm is taken of the fp32 sum before it is rounded into
    ``residual``; the output is rounded once."""
    need_here(input, residual, weight, out)
    _norm_args(input, residual, weight)
    output = torch.empty_like(input) if out is None else out
    assert output.shape == input.shape and output.dtype == input.dtype and output.is_contiguous()
    rc = _lib.attn().esp_add_rms_norm(output.data_ptr(), residual.data_ptr(), input.data_ptr(), weight.data_ptr(), input.size(0),
                                      input.size(1), float(eps), dtype16_tag(input), stream_ptr())
    _lib.check(rc, "esp_add_rms_norm")
    return output


@torch.inference_mode()
def add_rms_norm_quant(input: torch.Tensor, residual, weight: torch.Tensor, eps: float, out=None, out_scale=None):
    """``add_rms_norm`` whose output is int8 rows: (codes [tokens, hidden], scale [tokens]).  ``residual`` None: the norm of
    ``input`` alone."""
    need_here(input, residual, weight, out, out_scale)
    _norm_args(input, residual, weight)
    tokens, hidden = input.shape
    codes, scale = _rows_out(out, out_scale, tokens, hidden, input.device)
    rc = _lib.attn().esp_add_rms_norm_q8(codes.data_ptr(), scale.data_ptr(), ptr(residual), input.data_ptr(), weight.data_ptr(), tokens,
                                         hidden, float(eps), dtype16_tag(input), stream_ptr())
    _lib.check(rc, "esp_add_rms_norm_q8")
    return codes, scale


@torch.inference_mode()
def silu_and_mul_quant(io: torch.Tensor, out=None, out_scale=None):
    """int8 rows of silu(io[:, :F]) * io[:, F:]: (codes [tokens, F], scale [tokens]).  ``io`` is left as it was."""
    need_here(io, out, out_scale)
    assert io.dim() == 2 and io.is_contiguous() and io.size(1) % 2 == 0
    tokens, ffn = io.size(0), io.size(1) // 2
    codes, scale = _rows_out(out, out_scale, tokens, ffn, io.device)
    rc = _lib.attn().esp_silu_and_mul_q8(codes.data_ptr(), scale.data_ptr(), io.data_ptr(), tokens, ffn, dtype16_tag(io), stream_ptr())
    _lib.check(rc, "esp_silu_and_mul_q8")
    return codes, scale


@torch.inference_mode()
def quantize_rows(x: torch.Tensor, out=None, out_scale=None):
    """int8 rows of x [rows, cols]: (codes, scale [rows]).  Also lays out weights for ``mm_w8a8``: ``quantize_rows(w.t().contiguous())``
    of a [in, out] weight gives its output channels as rows."""
    need_here(x, out, out_scale)
    assert x.dim() == 2 and x.stride(1) == 1
    codes, scale = _rows_out(out, out_scale, x.size(0), x.size(1), x.device)
    rc = _lib.attn().esp_quantize_rows(codes.data_ptr(), scale.data_ptr(), x.data_ptr(), x.stride(0), x.size(0), x.size(1), dtype16_tag(x),
                                       stream_ptr())
    _lib.check(rc, "esp_quantize_rows")
    return codes, scale


@torch.inference_mode()
def dequantize_rows(codes: torch.Tensor, scale: torch.Tensor, dtype=torch.bfloat16, out=None) -> torch.Tensor:
    """codes * scale per row, rounded to ``dtype``."""
    need_here(codes, scale, out)
    assert codes.dim() == 2 and codes.dtype == torch.int8 and codes.is_contiguous()
    assert scale.shape == (codes.size(0),) and scale.dtype == torch.float32 and scale.is_contiguous()
    o = torch.empty(codes.shape, dtype=dtype, device=codes.device) if out is None else out
    assert o.shape == codes.shape and o.is_contiguous()
    rc = _lib.attn().esp_dequantize_rows(o.data_ptr(), codes.data_ptr(), scale.data_ptr(), codes.size(0), codes.size(1), dtype_tag(o),
                                         stream_ptr())
    _lib.check(rc, "esp_dequantize_rows")
    return o


@torch.inference_mode()
def mm_w8a8(a: torch.Tensor, a_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, out_dtype=torch.bfloat16, out=None):
    """(a @ w.T) * a_scale[:, None] * w_scale[None]: int8 rows of tokens [M, K] and of output channels [N, K], exact integer sums,
    one rounding to the output type.  K a multiple of 16, at most 131071."""
    need_here(a, a_scale, w, w_scale, out)
    assert a.dim() == 2 and w.dim() == 2 and a.size(1) == w.size(1)
    if a.dtype != torch.int8 or w.dtype != torch.int8 or a_scale.dtype != torch.float32 or w_scale.dtype != torch.float32:
        raise TypeError("mm_w8a8 takes int8 codes and fp32 scales")
    m, k = a.shape
    n = w.size(0)
    assert a.stride(1) == 1 and w.stride(1) == 1
    assert a_scale.shape == (m,) and w_scale.shape == (n,) and a_scale.is_contiguous() and w_scale.is_contiguous()
    o = torch.empty((m, n), dtype=out_dtype, device=a.device) if out is None else out
    assert o.shape == (m, n) and (n == 1 or o.stride(1) == 1)
    rc = _lib.attn().esp_mm_w8a8(o.data_ptr(), o.stride(0), a.data_ptr(), a.stride(0), a_scale.data_ptr(), w.data_ptr(), w.stride(0),
                                 w_scale.data_ptr(), m, n, k, dtype_tag(o), stream_ptr())
    _lib.check(rc, "esp_mm_w8a8")
    return o
