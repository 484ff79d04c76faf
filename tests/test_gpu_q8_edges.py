"""Edges of the 8-bit operators beside those of tests/test_gpu_q8.py, with its definitions, inputs and tolerances unless a test derives
its own."""
import pytest
import torch

from test_gpu_q8 import BF16, D, DEV, E4M3, F16, INT8, U32, check_decode, decode_case, decode_exact
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


def launch_shapes(test):
    """Groups of up to four heads (rests in the columns of heads 4 to 7) and of more (a second product), one, two and four kv heads to
    a CTA."""
    return pytest.mark.parametrize("code", [INT8, E4M3])(pytest.mark.parametrize("hq,hkv,batch", [
        (8, 2, 4), (32, 32, 10), (32, 32, 20), (10, 2, 4), (16, 2, 4), (160, 32, 10), (256, 32, 20), (20, 1, 4)])(test))


@launch_shapes
def test_decode_weights_keep_both_their_f16_numbers(code, hq, hkv, batch):
    """K scales of zero make every score 0 and every p exactly 1, so nothing covers the weights' own error.

    Roundings, relative to the mean of |v|: a weight is vs * (4096 / v_ref), 2; held as an f16 number and the f16 rounding of its rest,
    2^-22 (and 2^-25 absolute next to weights of 128 at least); 2n terms (both numbers of n weights) are added up, at most 2^-23
    each where the sum is cut instead of rounded; moving the reference, twice 1; the shares of four warps, three times 4; the two
    halves, the factor and its product, 4."""
    from loongserve_b200 import flash_decoding as fd
    lens = [17, 1, 3, 16] * (batch // 4) + [5] * (batch % 4)
    c = decode_case(lens, hq, hkv, BF16, code, hq + batch)
    g = torch.Generator().manual_seed(batch)
    c["scales"][:, :hkv] = 0.0
    c["scales"][:, hkv:] = (1 + 7 * torch.rand(c["scales"].shape[0], hkv, generator=g)).to(DEV)
    out = torch.empty(batch, hq, D, device=DEV); lse = torch.empty(batch, hq, device=DEV)
    fd.token_decode_attention_q8(c["q"], c["codes"][:, :hkv], c["scales"][:, :hkv], c["codes"][:, hkv:], c["scales"][:, hkv:], c["table"], c["rows"],
                                 c["lens"], 17, None, out, lse)
    n = torch.tensor(lens, dtype=torch.float64)[:, None]
    ro, _, wabs, _, _, _ = decode_exact(c)
    tol = (2.0 ** -22 + 2.0 ** -32 + 2 * n * 2.0 ** -23 + 20 * U32)[..., None] * wabs
    assert bool(((out.double().cpu() - ro).abs() <= tol).all()), ((out.double().cpu() - ro).abs() / tol).max()
    assert bool(((lse.double().cpu() - n.log()).abs() <= 4 * U32 * n.log() + 2.0 ** -30).all())
    # the bound is of use: weights without their rests do not keep it
    worst = 0.0
    for b, m in enumerate(lens):
        slots = c["table"][int(c["rows"][b]), :m].long()
        vs = c["scales"][slots, hkv:].double().cpu()                                             # [m, hkv]
        w = (vs * (1024 / vs.amax(0))).to(F16).double() * vs.amax(0) / 1024
        v = c["codes"].view(torch.uint8)[slots].view(code)[:, hkv:].double().cpu() * w[..., None]
        off = (v.mean(0).repeat_interleave(hq // hkv, 0) - ro[b]).abs() / tol[b]
        worst = max(worst, float(off.max()))
    assert worst > 4


@launch_shapes
def test_decode_scores_of_single_tokens(code, hq, hkv, batch):
    """A request of one token: p is exactly 1, and lse is the score itself.

    Roundings.  The factor sm_scale * log2(e), its two constants and the way back to natural logarithms: 6, and 2 of the K scale's
    products, relative to the score.  int8: the sum over the query's integer is exact; its digits meet in 3 roundings of sums
    below sum|q k| and what a lower digit can have more than its place (2^-6 of the largest element); the integer is off by half
    of 2^-29 (groups of up to four) or 2^-21 of the largest.  e4m3: 128 exact products are added up, at most 2^-23 each; elements below
    2^-21 of the largest are rounded by 2^-32 of it."""
    from loongserve_b200 import flash_decoding as fd
    c = decode_case([1] * batch, hq, hkv, BF16, code, hq - batch)
    out = torch.empty(batch, hq, D, device=DEV); lse = torch.empty(batch, hq, device=DEV)
    fd.token_decode_attention_q8(c["q"], c["codes"][:, :hkv], c["scales"][:, :hkv], c["codes"][:, hkv:], c["scales"][:, hkv:], c["table"], c["rows"],
                                 c["lens"], 1, None, out, lse)
    ro, rl, wabs, sabs, qabs, _ = decode_exact(c)
    if code is INT8:
        ds = 3 * U32 * (sabs + 2.0 ** -6 * qabs) + (2.0 ** -30 if hq // hkv <= 4 else 2.0 ** -22) * qabs
    else:
        ds = 128 * 2.0 ** -23 * sabs + 2.0 ** -32 * qabs
    tol = 8 * U32 * rl.abs() + ds
    assert bool(((lse.double().cpu() - rl).abs() <= tol).all()), ((lse.double().cpu() - rl).abs() / tol).max()
    assert bool(((out.double().cpu() - ro).abs() <= (2.0 ** -22 + 12 * U32) * wabs).all())


def test_silu_where_the_denominator_nears_the_end_of_the_range():
    """Gates from -88.5 to -87 give 1 + exp(-g) of 2^125 to 2^128; next to up values of 1e36 and more the products are ordinary
    numbers.  exp(-g) is off by 2 + 1.173 * 88.5 ulp, its reciprocal by one; then two products: within 2^-16 relative."""
    from loongserve_b200 import layer_ops as ops
    g = torch.Generator().manual_seed(2)
    gate = torch.linspace(-88.5, -87.0, 256).to(BF16)
    up = (torch.randn(3, 256, generator=g) * torch.tensor([[1e36], [1e37], [3e37]])).to(BF16)
    io = torch.cat([gate.expand(3, -1), up], 1).contiguous()
    codes, scale = ops.silu_and_mul_quant(io.to(DEV))
    y = gate.double() * torch.sigmoid(gate.double()) * up.double()
    s = y.abs().amax(-1) / 127
    assert bool(((scale.double().cpu() - s).abs() <= (2.0 ** -16 + 2 * U32) * s).all())
    v = codes.double().cpu() * scale.double().cpu()[:, None]
    assert bool(((v - y).abs() <= (0.5 + 127 * 2.0 ** -15) * s[:, None]).all())
