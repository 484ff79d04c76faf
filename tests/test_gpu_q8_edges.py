"""Edges of the 8-bit operators beside those of tests/test_gpu_q8.py, with its definitions, inputs and tolerances unless a test derives
its own."""
import pytest
import torch

from test_gpu_q8 import BF16, D, DEV, E4M3, INT8, check_decode, decode_case, decode_exact
from test_gpu_q8_runtime import exact_over_pool, i32, make_runtime, prefill, rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("code", [INT8, E4M3])
@pytest.mark.parametrize("hq,hkv", [(2, 2), (8, 2), (10, 2), (16, 2)])
def test_decode_with_the_largest_queries(code, hq, hkv):
    """+-finfo(bf16).max in a query, K scales of 2^-126 that bring the scores back to about a hundred: signs and sizes hold, in the
    digits of groups of up to four heads and of more."""
    from loongserve_b200 import flash_decoding as fd
    c = decode_case([40, 300], hq, hkv, BF16, code, 17)
    top = torch.finfo(BF16).max
    c["scales"][:, :hkv] = 2.0 ** -126
    c["q"][0, 0, 3] = top
    c["q"][0, -1, 0] = -top; c["q"][0, -1, 127] = top
    c["q"][1, 0, 64] = -top
    c["q"][1, -1] = top
    out = torch.empty(2, hq, D, device=DEV); lse = torch.empty(2, hq, device=DEV)
    for block in (None, 64):
        fd.token_decode_attention_q8(c["q"], c["codes"][:, :hkv], c["scales"][:, :hkv], c["codes"][:, hkv:], c["scales"][:, hkv:], c["table"],
                                     c["rows"], c["lens"], 300, block, out, lse)
        check_decode(out, lse, decode_exact(c), 300)


def test_a_layer_of_no_tokens():
    """The 8-bit layer of an instance that holds no token of a prefill: every operator takes zero rows."""
    from types import SimpleNamespace
    from loongserve_b200.llama_stack import LlamaConfig, LlamaESPStack, LlamaW8A8Weights, LlamaWeights
    cfg = LlamaConfig(num_layers=2, hidden=256, num_q_heads=4, num_kv_heads=2, head_dim=128, ffn=320, vocab=50)
    scratch = torch.zeros(1, 4, D, dtype=BF16, device=DEV)
    rt = SimpleNamespace(pre_cache_kv=lambda st, li: scratch, context_attention=lambda q, st, li: torch.empty_like(q))
    stack = LlamaESPStack(cfg, LlamaW8A8Weights(cfg, LlamaWeights(cfg, BF16, DEV, seed=1)), rt)
    none = torch.empty(0, dtype=torch.int64, device=DEV)
    assert stack.prefill(none, none, None).shape == (0, 256) and stack.prefill(none, none, None, last_token_rows=none).shape == (0, 50)
    torch.cuda.synchronize()


def test_keep_range_write_refuses_vectors_of_the_host():
    from loongserve_b200 import kv_ops
    from test_gpu_q8 import pool
    dev = lambda *x, dtype=torch.int32: torch.tensor(x, dtype=dtype, device=DEV)
    raw, codes, scales = pool(8, 2, INT8)
    before = raw.clone()
    a = [1, dev(2), dev(0), dev(2), dev(2, dtype=torch.int64), torch.randn(4, 2, D, device=DEV).to(BF16), dev(0), dev(0), dev(3, 1, dtype=torch.int64),
         codes, scales, torch.zeros(2, 8, dtype=torch.int32, device=DEV), dev(0), 0, 2, True]
    for i in (1, 2, 3, 4, 6, 7, 8, 11, 12):
        with pytest.raises(RuntimeError, match="CUDA"):
            kv_ops.destindex_copy_quantize_and_register_kv(*a[:i], a[i].cpu(), *a[i + 1:])
    with pytest.raises(AssertionError):
        kv_ops.destindex_copy_quantize_and_register_kv(2, *a[1:])
    assert torch.equal(raw, before)
    kv_ops.destindex_copy_quantize_and_register_kv(*a)
    assert not torch.equal(raw[[1, 3]], before[[1, 3]]) and a[11][0, :2].tolist() == [3, 1]


@pytest.mark.parametrize("block", [None, 32, 100])
def test_a_decode_step_with_splits_of_its_own(block):
    g = torch.Generator().manual_seed(3)
    lens = [300, 7, 130]
    rt = make_runtime(INT8, decode_block_seq=block)
    b_req, _, _ = prefill(rt, lens, rows(437, 2, 8, g), rows(437, 2, 4, g))
    lens = [n + 1 for n in lens]
    st = rt.prepare_decode(3, 3, max(lens), b_req, i32(lens), i32([n - 1 for n in lens]), 0, [0], 0)
    q, kv = torch.randn(3, 8, D, generator=g).to(BF16).to(DEV), torch.randn(3, 4, D, generator=g).to(BF16).to(DEV)
    for layer in range(2):
        rt.decode_cache_kv(st, layer).copy_(kv)
        rt.post_decode_cache_kv(st, layer)
        check_decode(rt.token_attention(q, st, layer), st.global_out_logexpsum, exact_over_pool(rt, layer, q, b_req, lens), max(lens))
    rt.check_device_status()
