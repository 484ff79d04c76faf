"""Distributed flash-decoding ops with the reference's names and argument order.

``flash_decoding_stage1`` / ``flash_decoding_stage2`` correspond to the pybind functions of
``longserve_cuda_kernels`` (longserve_cuda_kernels/src/entrypoints.cpp:103-221); the
``longserve_*`` wrappers to loongserve/models/llama/triton_kernel/longserve_flash_decoding*.py.
"""
from __future__ import annotations

import torch

from . import _lib
from ._util import code_tag, dtype16_tag, dtype_tag, need_cuda, need_here, need_i32, ptr, stream_of, stream_ptr


@torch.inference_mode()
def flash_decoding_stage1(mid_o, mid_o_logexpsum, q, k, v, req_to_tokens, b_req_idx, b_seqlen,
                          max_len_in_batch: int, seq_block_size: int, sm_scale: float = 0.0):
    need_cuda(mid_o, mid_o_logexpsum, q, k, v, req_to_tokens, b_req_idx, b_seqlen)
    assert mid_o.is_contiguous() and mid_o_logexpsum.is_contiguous() and q.is_contiguous()
    assert k.stride(2) == 1 and v.stride(2) == 1 and req_to_tokens.is_contiguous()
    assert mid_o.dim() == 4 and mid_o_logexpsum.dim() == 3 and q.dim() == 3 and k.dim() == 3 and v.dim() == 3
    assert mid_o.dtype == torch.float32 and mid_o_logexpsum.dtype == torch.float32
    assert k.dtype == q.dtype and v.dtype == q.dtype and req_to_tokens.dtype == torch.int32
    need_i32(b_req_idx, b_seqlen)
    nblk = (int(max_len_in_batch) + int(seq_block_size) - 1) // int(seq_block_size)
    assert mid_o.shape[0] >= nblk and mid_o.shape[1] == q.shape[0] and mid_o.shape[2] == q.shape[1]
    rc = _lib.attn().esp_decode_stage1(
        ptr(mid_o), ptr(mid_o_logexpsum), ptr(q), ptr(k), ptr(v), k.stride(0), k.stride(1), v.stride(0),
        v.stride(1), ptr(req_to_tokens), req_to_tokens.stride(0), ptr(b_req_idx), ptr(b_seqlen),
        q.shape[0], q.shape[1], k.shape[1], q.shape[2], int(max_len_in_batch), int(seq_block_size),
        dtype_tag(q), float(sm_scale), min(k.shape[0], v.shape[0]), stream_ptr())
    _lib.check(rc, "esp_decode_stage1")


@torch.inference_mode()
def flash_decoding_stage2(o, out_logexpsum, b_seqlen, mid_o, mid_o_logexpsum, block_seq: int):
    need_cuda(o, out_logexpsum, b_seqlen, mid_o, mid_o_logexpsum)
    assert o.is_contiguous() and out_logexpsum.is_contiguous() and mid_o.is_contiguous() and mid_o_logexpsum.is_contiguous()
    assert o.dim() == 3 and out_logexpsum.dim() == 2 and mid_o.dim() == 4 and mid_o_logexpsum.dim() == 3
    assert out_logexpsum.dtype == torch.float32 and mid_o.dtype == torch.float32
    need_i32(b_seqlen)
    rc = _lib.attn().esp_decode_merge(ptr(o), ptr(out_logexpsum), ptr(b_seqlen), ptr(mid_o), ptr(mid_o_logexpsum),
                                      o.shape[0], o.shape[1], o.shape[2], mid_o.shape[0], int(block_seq),
                                      dtype_tag(o), stream_ptr())
    _lib.check(rc, "esp_decode_merge")


def _q8_args(q, k, k_scale, v, v_scale, req_to_tokens, b_req_idx, b_seqlen):
    """The arguments of the C calls from q to b_seqlen and the sizes behind them, checked."""
    qs, ks, vs = q.shape, k.shape, v.shape
    assert len(qs) == 3 and len(ks) == 3 and len(vs) == 3 and q.is_contiguous()
    (kt, kh, kd), (vt, vh, vd) = k.stride(), v.stride()
    assert kd == 1 and vd == 1 and ks[1:] == vs[1:] and ks[2] == qs[2] and k_scale.shape == ks[:2] and v_scale.shape == vs[:2]
    (kst, ksh), (vst, vsh) = k_scale.stride(), v_scale.stride()
    assert ks[1] == 1 or (ksh == 1 and vsh == 1)
    if k_scale.dtype != torch.float32 or v_scale.dtype != torch.float32 or v.dtype != k.dtype or req_to_tokens.dtype != torch.int32:
        raise TypeError("k and v hold codes of one type, their scales are fp32, req_to_tokens is int32")
    ts = req_to_tokens.shape
    assert len(ts) == 2 and req_to_tokens.stride(1) == 1
    need_i32(b_req_idx, b_seqlen)
    assert b_req_idx.shape == qs[:1] and b_seqlen.shape == qs[:1]
    return (q.data_ptr(), k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), kt, kh, vt, vh, kst, vst,
            req_to_tokens.data_ptr(), req_to_tokens.stride(0), ts[0], ts[1], b_req_idx.data_ptr(), b_seqlen.data_ptr(), qs[0], qs[1],
            ks[1], qs[2]), min(ks[0], vs[0])


def flash_decoding_stage1_q8(mid_o, mid_o_logexpsum, q, k, k_scale, v, v_scale, req_to_tokens, b_req_idx, b_seqlen,
                             max_len_in_batch: int, seq_block_size: int, sm_scale: float = 0.0):
    """``flash_decoding_stage1`` over a pool held in 8 bits: k, v int8 or e4m3 codes [slots, Hkv, 128], k_scale, v_scale fp32
    [slots, Hkv].  The partials go to ``flash_decoding_stage2`` unchanged."""
    dev = need_here(q, mid_o, mid_o_logexpsum, k, k_scale, v, v_scale, req_to_tokens, b_req_idx, b_seqlen)
    args, slots = _q8_args(q, k, k_scale, v, v_scale, req_to_tokens, b_req_idx, b_seqlen)
    assert mid_o.is_contiguous() and mid_o_logexpsum.is_contiguous()
    assert mid_o.dim() == 4 and mid_o_logexpsum.dim() == 3 and mid_o.dtype == mid_o_logexpsum.dtype == torch.float32
    nblk = (int(max_len_in_batch) + int(seq_block_size) - 1) // int(seq_block_size)
    assert mid_o.shape[0] >= nblk and mid_o.shape[1:] == q.shape
    assert mid_o_logexpsum.shape[0] >= nblk and mid_o_logexpsum.shape[1:] == q.shape[:2]
    rc = _lib.attn().esp_decode_stage1_q8(mid_o.data_ptr(), mid_o_logexpsum.data_ptr(), *args, int(max_len_in_batch), int(seq_block_size),
                                          dtype16_tag(q), code_tag(k), sm_scale, slots, stream_of(dev))
    if rc:
        _lib.check(rc, "esp_decode_stage1_q8")


Q8_MAX_EVEN = 384          # requests whose tokens one call divides evenly


def q8_block_seq(batch: int, kv_heads: int, group: int, max_len_in_batch: int) -> int:
    """Tokens per split, where splits have a fixed length: eight times as many (split, heads) items as the GPU holds CTAs, within 128
    and 512 tokens.  Shorter splits cost partials, longer ones leave a tail: 32 requests x 32 heads, 287567 tokens, take 467 / 410 / 389 /
    399 / 420 us with 128 / 256 / 512 / 1024 / 2048."""
    tiles = batch * kv_heads * ((group + 7) // 8)
    splits = max(1, -(-148 * 3 * 8 * 4 // max(1, tiles)))
    return min(512, max(128, -(-max(int(max_len_in_batch), 1) // splits // 128) * 128))


def token_decode_attention_q8(q, cache_k, k_scale, cache_v, v_scale, req_to_token_indexs, b_req_idx, b_seq_len,
                              max_len_in_batch: int, block_seq=None, out=None, out_logexpsum=None, sm_scale: float = 0.0):
    """Decode attention over a pool held in 8 bits, splits and merge in one call: (o like q unless ``out`` is given, lse fp32).
    ``block_seq``: tokens per split; by default the tokens of up to 384 requests are divided evenly over the GPU (392 us for 32 requests
    x 32 heads, 287567 tokens, 185 us for 2 x 8, 501702 tokens; with the best fixed length 389 and 195).  A request of length zero gets
    o = 0, lse = -inf."""
    dev = need_here(q, cache_k, k_scale, cache_v, v_scale, req_to_token_indexs, b_req_idx, b_seq_len, out, out_logexpsum)
    args, slots = _q8_args(q, cache_k, k_scale, cache_v, v_scale, req_to_token_indexs, b_req_idx, b_seq_len)
    batch, hq, hkv, dim = args[-4:]
    max_len = int(max_len_in_batch)
    if out is None:
        out = torch.empty_like(q)
    else:
        assert out.shape == q.shape and out.is_contiguous()
    if out_logexpsum is None:
        out_logexpsum = k_scale.new_empty((batch, hq))
    else:
        assert out_logexpsum.shape == (batch, hq) and out_logexpsum.is_contiguous()
        if out_logexpsum.dtype != torch.float32:
            raise TypeError("out_logexpsum is fp32")
    tags = dtype16_tag(q), dtype_tag(out), code_tag(cache_k)
    if block_seq is None and (batch <= Q8_MAX_EVEN or max_len <= 512):
        block = 0
        floats = (min(444, (batch * max_len + 63) // 64) + batch) * hq * (dim + 1) + 2 * batch if 256 < max_len and batch <= Q8_MAX_EVEN else 0
    else:
        block = int(block_seq) if block_seq is not None else q8_block_seq(batch, hkv, hq // max(hkv, 1), max_len)
        assert block > 0
        nblk = (max_len + block - 1) // block
        floats = nblk * batch * hq * (dim + 1) if nblk > 1 else 0
    work = k_scale.new_empty(floats) if floats else None
    rc = _lib.attn().esp_decode_attention_q8(out.data_ptr(), out_logexpsum.data_ptr(), ptr(work), *args, max_len, block, *tags, sm_scale,
                                             slots, stream_of(dev))
    if rc:
        _lib.check(rc, "esp_decode_attention_q8")
    return out, out_logexpsum


def longserve_flash_decode_stage1(q, k, v, Req_to_tokens, B_req_idx, B_Seqlen, max_len_in_batch, mid_out,
                                  mid_out_logsumexp, block_seq):
    """longserve_flash_decoding_stage1.py:78-88."""
    flash_decoding_stage1(mid_out, mid_out_logsumexp, q, k, v, Req_to_tokens, B_req_idx, B_Seqlen,
                          max_len_in_batch, block_seq)


def longserve_flash_decode_stage2(mid_out, mid_out_logexpsum, B_Seqlen, O, out_logexpsum, block_seq):
    """longserve_flash_decoding_stage2.py:53-61."""
    flash_decoding_stage2(O, out_logexpsum, B_Seqlen, mid_out, mid_out_logexpsum, block_seq)


def longserve_token_decode_attention_flash_decoding(q, req_to_token_indexs, b_req_idx, b_seq_len, mid_o,
                                                    mid_o_logexpsum, batch_size, max_len_in_batch, q_head_num,
                                                    head_dim, cache_k, cache_v, BLOCK_SEQ, out=None,
                                                    o_logexpsum=None):
    """Peer-side stage 1 + stage 2 for foreign queries -> (o fp32, lse fp32)
    (longserve_flash_decoding.py:3-28)."""
    shape = (-1, q_head_num, head_dim)
    o_tensor = torch.empty_like(q, dtype=torch.float32) if out is None else out
    out_lse = torch.empty([batch_size, q_head_num], dtype=torch.float32, device=q.device) if o_logexpsum is None else o_logexpsum
    longserve_flash_decode_stage1(q.view(shape), cache_k, cache_v, req_to_token_indexs, b_req_idx, b_seq_len,
                                  max_len_in_batch, mid_o, mid_o_logexpsum, BLOCK_SEQ)
    longserve_flash_decode_stage2(mid_o, mid_o_logexpsum, b_seq_len, o_tensor.view(shape), out_lse, BLOCK_SEQ)
    return o_tensor, out_lse


def device_status(clear: bool = True):
    """(code, block, which, value) of the decode kernels and flag waits on the current device: code 0, or
    ESP_ERR_DEVICE_TIMEOUT (-4) for a flag wait that ran out, or ESP_ERR_BAD_SLOT (-8) for a slot id outside the pool
    (that token was left out).  Synchronises the device."""
    import ctypes as C
    buf = (C.c_int32 * 4)()
    _lib.check(_lib.attn().esp_decode_device_status(buf, 1 if clear else 0), "esp_decode_device_status")
    return tuple(buf)


def set_wait_limit_cycles(cycles: int):
    """Limit of every bounded in-kernel wait on the current device, in SM cycles (default 2e9, about a second)."""
    _lib.check(_lib.attn().esp_set_wait_limit_cycles(int(cycles)), "esp_set_wait_limit_cycles")
