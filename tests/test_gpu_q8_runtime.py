"""The 8-bit serving path in the framework's own runtime on one GPU: the pool in 8 bits behind ESPAttentionRuntime (prefill, keep-range
write, decode, the message exchange, migration) and the Llama stack with 8-bit projections.

What decode reads is what the pool holds, so decode is checked against attention over ``read_kv`` in 64 bits with the roundings
of tests/test_gpu_q8.py; prefill attends to 16-bit rows and has to give the same bits as with a 16-bit pool."""
import pytest
import torch

from oracle import esp_oracle as O
from test_gpu_q8 import BF16, D, E4M3, F16, INT8, check_decode, decode_exact

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make_runtime(kv_dtype, dtype=BF16, L=2, Hq=8, Hkv=2, slots=1024, **kw):
    from loongserve_b200.attention_runtime import ESPAttentionRuntime
    return ESPAttentionRuntime(layers_num=L, q_head_num=Hq, kv_head_num=Hkv, head_dim=D, max_total_token_num=slots, max_req_num=8,
                               max_seq_length=512, dtype=dtype, kv_dtype=kv_dtype, **kw)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def prefill(rt, lens, q, kv, **kw):
    B = len(lens)
    b_req = rt.req_manager.alloc(B).to(torch.int32)
    b_len = i32(lens)
    b_start = torch.cumsum(b_len, 0, dtype=torch.int32) - b_len
    st = rt.prepare_prefill(B, sum(lens), sum(lens), max(lens), b_req, b_start, b_len, i32([0] * B), [0], 0, **kw)
    outs = []
    for layer in range(rt.layers_num):
        rt.pre_cache_kv(st, layer)[:sum(lens)].copy_(kv[layer])
        outs.append(rt.context_attention(q[layer], st, layer))
    return b_req, st, outs


def exact_over_pool(rt, layer, q, b_req, lens):
    lay = rt.mem_manager.layer(layer)
    return decode_exact(dict(q=q, codes=lay.codes, scales=lay.scales, table=rt.req_manager.req_to_token_indexs, rows=b_req,
                             lens=i32(lens), hkv=rt.tp_k_head_num_))


def rows(n, layers, heads, g, dtype=BF16):
    return [torch.randn(n, heads, D, generator=g).to(dtype).to(DEV) for _ in range(layers)]


@pytest.mark.parametrize("kv_dtype", [INT8, E4M3])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_prefill_then_decode(kv_dtype, dtype):
    g = torch.Generator().manual_seed(31)
    lens = [301, 6, 130]
    rt, plain = make_runtime(kv_dtype, dtype), make_runtime(None, dtype)
    q, kv = rows(sum(lens), 2, 8, g, dtype), rows(sum(lens), 2, 4, g, dtype)
    b_req, st, outs = prefill(rt, lens, q, kv)
    _, _, outs16 = prefill(plain, lens, q, kv)
    assert not st.mem_is_contiguous
    for layer in range(2):
        assert torch.equal(outs[layer], outs16[layer])                      # prefill attends to the 16-bit rows
        back = rt.read_kv(st.mem_index, layer)
        amax = kv[layer].float().abs().amax(-1, keepdim=True)               # half a step of int8, or 2^-4 relative (2^-10 of amax near 0)
        off = (back.float() - kv[layer].float()).abs()
        lim = (amax / 254 if kv_dtype is INT8 else torch.maximum(kv[layer].float().abs() / 16, amax * 2.0 ** -9 / 448)) * 1.02
        assert bool((off <= lim + torch.finfo(dtype).eps * kv[layer].float().abs()).all())
    for step in range(3):                                                    # three decode steps, each over what the pool then holds
        lens = [n + 1 for n in lens]
        dst = rt.prepare_decode(3, 3, max(lens), b_req, i32(lens), i32([n - 1 for n in lens]), 0, [0], 0)
        for layer in range(2):
            new_q, new_kv = torch.randn(3, 8, D, generator=g).to(dtype).to(DEV), torch.randn(3, 4, D, generator=g).to(dtype).to(DEV)
            rt.decode_cache_kv(dst, layer).copy_(new_kv)
            rt.post_decode_cache_kv(dst, layer)
            o = rt.token_attention(new_q, dst, layer)
            check_decode(o, dst.global_out_logexpsum, exact_over_pool(rt, layer, new_q, b_req, lens), max(lens))
            given = torch.empty_like(new_q)
            assert rt.token_attention(new_q, dst, layer, out=given) is given and torch.equal(given, o)
    rt.check_device_status()
    assert rt.mem_manager.can_use_mem_size == 1024 - sum(lens)


def test_keep_range_prefill_fills_the_pool():
    """A scale-down batch (need_context_migration): the ring's keep step quantises the kept rows and registers their slots."""
    g = torch.Generator().manual_seed(5)
    lens, begin, end = [200, 37, 64], [20, 0, 10], [180, 37, 10]
    rt = make_runtime(INT8)
    q, kv = rows(sum(lens), 2, 8, g), rows(sum(lens), 2, 4, g)
    b_req, st, outs = prefill(rt, lens, q, kv, need_context_migration=True, kv_cache_index_begin=i32(begin), kv_cache_index_end=i32(end))
    start = [0, 200, 237]
    for layer in range(2):
        ro, _ = O.full_causal_attention(q[layer].cpu(), kv[layer][:, :2].cpu(), kv[layer][:, 2:].cpu(), lens)
        assert bool(((outs[layer].float().cpu() - ro).abs() <= 2e-2 + 1e-2 * ro.abs()).all())
        at = 0
        for b in range(3):
            n = end[b] - begin[b]
            slots = rt.req_manager.req_to_token_indexs[int(b_req[b]), :n]
            assert torch.equal(slots.long(), st.mem_index[at:at + n])
            if n:
                want = kv[layer][start[b] + begin[b]:start[b] + end[b]].float()
                off = (rt.read_kv(slots, layer).float() - want).abs()
                assert bool((off <= want.abs().amax(-1, keepdim=True) / 254 * 1.01 + 2.0 ** -8 * want.abs()).all())
            at += n


class Mail:
    """Stands for the communicator of two instances that run one after the other in this process."""

    def __init__(self):
        self.box, self.sent = [], []

    def nccl_group_start(self): pass
    def nccl_group_end(self): pass
    def wait_for_default_stream(self): pass
    def let_default_stream_wait(self): pass

    def nccl_send(self, t, peer):
        self.sent.append(t.clone())

    def nccl_recv(self, t, peer):
        t.copy_(self.box.pop(0))


@pytest.mark.parametrize("kv_dtype", [INT8, E4M3])
def test_message_exchange_over_two_instances(kv_dtype):
    """A batch whose tokens lie on two instances: the peer's partial over its 8-bit pool, merged by the master."""
    from loongserve_b200 import ring
    g = torch.Generator().manual_seed(6)
    master, peer = make_runtime(kv_dtype, L=1), make_runtime(kv_dtype, L=1)
    lens_m, lens_p = [120, 33, 200], [64, 90, 1]
    q1, kv_m, kv_p = rows(3, 1, 8, g)[0], rows(sum(lens_m), 1, 4, g), rows(sum(lens_p), 1, 4, g)
    req_m, _, _ = prefill(master, lens_m, rows(sum(lens_m), 1, 8, g), kv_m)
    req_p, _, _ = prefill(peer, lens_p, rows(sum(lens_p), 1, 8, g), kv_p)
    f = lambda *s: torch.empty(*s, device=DEV)
    bs = 64
    mail = Mail()
    mail.box = [q1]
    pp = ring.PeerPlan([0], [(0, 3)], torch.empty_like(q1), req_p, i32(lens_p), max(lens_p), bs, f(2, 3, 8, D), f(2, 3, 8), f(3, 8, D), f(3, 8))
    peer.sp_comm = mail
    from loongserve_b200.attention_runtime import LongServeLlamaInferStateInfo
    st = LongServeLlamaInferStateInfo(peer_plan=pp, master_plan=None, logical_sp_peer_ranks=[0, 1])
    assert peer.token_attention(None, st, 0) is None and len(mail.sent) == 2
    nblk = (max(lens_m) + bs - 1) // bs
    mlen = i32([1 + (n + bs - 1) // bs for n in lens_m])
    mp = ring.MasterPlan([0, 1], req_m, i32(lens_m), max(lens_m), bs, f(1 + nblk, 3, 8, D), f(1 + nblk, 3, 8), mlen, f(3, 8))
    mail2 = Mail()
    mail2.box = mail.sent
    master.sp_comm = mail2
    o = master.token_attention(q1, LongServeLlamaInferStateInfo(peer_plan=None, master_plan=mp, logical_sp_peer_ranks=[0, 1]), 0)
    # one pool that holds both instances' rows
    lay = [r.mem_manager.layer(0) for r in (master, peer)]
    n0 = lay[0].shape[0]
    both = dict(q=q1, codes=torch.cat([x.codes.view(torch.uint8) for x in lay]).view(kv_dtype), scales=torch.cat([x.scales for x in lay]), hkv=2,
                rows=i32([0, 1, 2]), lens=i32([a + b for a, b in zip(lens_m, lens_p)]), table=torch.zeros(3, 300, dtype=torch.int32, device=DEV))
    for b in range(3):
        both["table"][b, :lens_m[b]] = master.req_manager.req_to_token_indexs[int(req_m[b]), :lens_m[b]]
        both["table"][b, lens_m[b]:lens_m[b] + lens_p[b]] = n0 + peer.req_manager.req_to_token_indexs[int(req_p[b]), :lens_p[b]]
    check_decode(o, mp.global_out_lse, decode_exact(both), 300)


@pytest.mark.parametrize("kv_dtype", [INT8, E4M3])
def test_migration_moves_codes_and_scales(kv_dtype):
    g = torch.Generator().manual_seed(7)
    a, b = make_runtime(kv_dtype), make_runtime(kv_dtype)
    lens, mig = [100, 40], [60, 40]
    req_a, st, _ = prefill(a, lens, rows(140, 2, 8, g), rows(140, 2, 4, g))
    req_b = b.req_manager.alloc(2).to(torch.int32)
    want = [torch.cat([a.read_kv(a.req_manager.req_to_token_indexs[int(req_a[r]), lens[r] - mig[r]:lens[r]], layer) for r in range(2)]) for layer in range(2)]
    a.sp_comm = Mail()
    a.decoding_stage_migration(False, req_a, i32(mig), i32(lens), 1, sum(mig), max(mig))
    b.sp_comm = Mail()
    b.sp_comm.box = a.sp_comm.sent
    b.decoding_stage_migration(True, req_b, i32(mig), i32([0, 0]), 0, sum(mig), max(mig))
    for layer in range(2):
        got = torch.cat([b.read_kv(b.req_manager.req_to_token_indexs[int(req_b[r]), :mig[r]], layer) for r in range(2)])
        assert torch.equal(got, want[layer])
    assert a.mem_manager.can_use_mem_size == 1024 - 40 and b.mem_manager.can_use_mem_size == 1024 - 100


@pytest.mark.parametrize("kv_dtype", [None, INT8, E4M3])
def test_llama_stack_with_8_bit_projections(kv_dtype):
    """Prefill and three decode steps.  Against the oracle stack on the same 8-bit weights (activations not quantised): int8 rows of
    activations lose about 0.009 of a row's rms per projection (a step is max/127 of 3-4 sigma; step / sqrt(12)), e4m3 rows of the
    pool 0.027 (2^-4 half step, uniform: / sqrt(3) of a quarter binade on average), four of them per layer and two layers."""
    from loongserve_b200.llama_stack import LlamaConfig, LlamaESPStack, LlamaW8A8Weights, LlamaWeights
    cfg = LlamaConfig(num_layers=2, hidden=512, num_q_heads=4, num_kv_heads=4, head_dim=128, ffn=1040, vocab=1000)
    w16 = LlamaWeights(cfg, BF16, DEV, seed=3)
    w8 = LlamaW8A8Weights(cfg, w16)
    rt = make_runtime(kv_dtype, Hq=4, Hkv=4, slots=2048)
    stack = LlamaESPStack(cfg, w8, rt)
    g = torch.Generator().manual_seed(5)
    full = [203, 36, 132]
    starts = [0, 203, 239]
    ids = torch.randint(0, cfg.vocab, (sum(full),), generator=g)
    pos = torch.cat([torch.arange(n) for n in full])
    wl = [dict(att_norm=lw["att_norm"].cpu(), ffn_norm=lw["ffn_norm"].cpu(),
               **{n: (lw[n][0].float() * lw[n][1][:, None]).t().cpu() for n in ("q", "kv", "o", "gate_up", "down")}) for lw in w8.layers]
    x = w16.embed.cpu()[ids].float()
    for lw in wl:
        x, _, _ = O.llama_layer(x, pos, full, lw, cfg.rms_eps, 4, 4, 128, BF16)
    ref_logits = O.rms_norm(x, w16.final_norm.cpu(), cfg.rms_eps).float() @ w16.lm_head.cpu().float()
    pre = [n - 3 for n in full]
    pre_rows = torch.cat([torch.arange(s, s + n) for s, n in zip(starts, pre)])
    b_req = rt.req_manager.alloc(3).to(torch.int32)
    b_len = i32(pre); b_start = torch.cumsum(b_len, 0, dtype=torch.int32) - b_len
    st = rt.prepare_prefill(3, sum(pre), sum(pre), max(pre), b_req, b_start, b_len, i32([0] * 3), [0], 0)
    last = (b_start + b_len - 1)
    logits = stack.prefill(ids[pre_rows].to(DEV), pos[pre_rows].to(DEV), st, last_token_rows=last)
    close = lambda got, want, lim: float((got.float().cpu() - want).norm() / want.norm()) < lim
    assert close(logits, ref_logits[torch.tensor([s + n - 1 for s, n in zip(starts, pre)])], 0.05)
    hidden = stack.prefill(ids[pre_rows].to(DEV), pos[pre_rows].to(DEV), rt.prepare_prefill(
        3, sum(pre), sum(pre), max(pre), rt.req_manager.alloc(3).to(torch.int32), b_start, b_len, i32([0] * 3), [0], 0))
    assert close(hidden, x[pre_rows], 0.05)
    for step in range(3):
        lens = [n + step + 1 for n in pre]
        new = torch.tensor([s + n - 1 for s, n in zip(starts, lens)])
        dst = rt.prepare_decode(3, 3, max(lens), b_req, i32(lens), i32([n - 1 for n in lens]), 0, [0], 0)
        logits = stack.decode(ids[new].to(DEV), pos[new].to(DEV), dst)
        assert close(logits, ref_logits[new], 0.08 if kv_dtype is E4M3 else 0.06)
    rt.check_device_status()


def test_what_the_8_bit_runtime_refuses():
    from loongserve_b200.llama_stack import GraphedDecode, LlamaConfig, LlamaESPStack, LlamaWeights
    with pytest.raises(ValueError, match="message exchange"):
        make_runtime(INT8, peer_memory_decode=True)
    with pytest.raises(TypeError):
        make_runtime(torch.uint8)
    rt = make_runtime(INT8)
    with pytest.raises(ValueError):
        rt.enable_peer_memory_decode(0, None, 4)
    cfg = LlamaConfig(num_layers=1, hidden=256, num_q_heads=2, num_kv_heads=2, ffn=256, vocab=64)
    stack = LlamaESPStack(cfg, LlamaWeights(cfg), rt)

    class Group:
        rank = master = 0
    with pytest.raises(ValueError):
        GraphedDecode(stack, Group(), i32([0]), i32([4]), positions=i32([4]))
