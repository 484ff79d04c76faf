"""Host side of the 8-bit serving path: the Llama stack's glue around the operators, on stand-ins of their shapes, and checks that are
made before a launch (no GPU needed)."""
from types import SimpleNamespace

import pytest
import torch

from loongserve_b200 import llama_stack


class Ops:
    """The layer operators by their shapes."""

    @staticmethod
    def add_rms_norm_quant(x, residual, weight, eps):
        assert residual is None or residual.shape == x.shape
        return torch.zeros(x.shape, dtype=torch.int8), torch.ones(x.shape[0])

    @staticmethod
    def add_rms_norm(x, residual, weight, eps):
        assert residual.shape == x.shape
        return torch.zeros_like(x)

    @staticmethod
    def mm_w8a8(a, a_scale, w, w_scale, out_dtype=torch.bfloat16, out=None):
        assert a.shape[1] == w.shape[1] and a_scale.shape == a.shape[:1]
        if out is None:
            return torch.zeros(a.shape[0], w.shape[0], dtype=out_dtype)
        assert out.shape == (a.shape[0], w.shape[0])
        return out.zero_()

    @staticmethod
    def quantize_rows(x):
        return torch.zeros(x.shape, dtype=torch.int8), torch.ones(x.shape[0])

    @staticmethod
    def silu_and_mul_quant(io):
        return torch.zeros(io.shape[0], io.shape[1] // 2, dtype=torch.int8), torch.ones(io.shape[0])

    @staticmethod
    def rotary_emb(q, k, cos, sin):
        assert q.shape[0] == k.shape[0] == cos.shape[0]


def stack_on_stand_ins(monkeypatch, max_tokens):
    monkeypatch.setattr(llama_stack, "layer_ops", Ops)
    cfg = llama_stack.LlamaConfig(num_layers=2, hidden=64, num_q_heads=4, num_kv_heads=2, head_dim=128, ffn=96, vocab=10)
    q8 = lambda n, k: (torch.zeros(n, k, dtype=torch.int8), torch.ones(n))
    layer = dict(att_norm=torch.ones(64), ffn_norm=torch.ones(64), q=q8(512, 64), kv=q8(512, 64), o=q8(64, 512), gate_up=q8(192, 64), down=q8(64, 96))
    weights = SimpleNamespace(w8a8=True, embed=torch.zeros(10, 64), final_norm=torch.ones(64), lm_head=torch.zeros(64, 10), layers=[layer, layer])
    scratch = torch.zeros(max_tokens, 4, 128)
    rt = SimpleNamespace(pre_cache_kv=lambda st, li: scratch, context_attention=lambda q, st, li: torch.empty_like(q))
    return llama_stack.LlamaESPStack(cfg, weights, rt)


@pytest.mark.parametrize("n", [0, 1, 3])
def test_a_prefill_of_which_an_instance_holds_few_tokens_or_none(monkeypatch, n):
    """Striped placement leaves the higher instances without tokens where all prompts are shorter than the ring."""
    stack = stack_on_stand_ins(monkeypatch, 4)
    hidden = stack.prefill(torch.zeros(n, dtype=torch.long), torch.arange(n), None)
    assert hidden.shape == (n, 64)
    assert stack.prefill(torch.zeros(n, dtype=torch.long), torch.arange(n), None, last_token_rows=torch.arange(n)).shape == (n, 10)


def keep_range_args(batch):
    i32 = lambda n: torch.zeros(n, dtype=torch.int32)
    lay = dict(codes=torch.zeros(9, 2, 128, dtype=torch.int8), scales=torch.zeros(9, 2))
    vectors = dict(new_len=i32(batch), begin=i32(batch), end=i32(batch), start=i32(batch), cur=i32(batch), b_req=i32(batch))
    rest = dict(cumsum=torch.zeros(batch, dtype=torch.int64), kv=torch.zeros(4, 2, 128, dtype=torch.bfloat16), mem=torch.zeros(4, dtype=torch.int64),
                table=torch.zeros(3, 8, dtype=torch.int32))
    return {**lay, **vectors, **rest}


def keep_range(a, batch):
    from loongserve_b200 import kv_ops
    kv_ops.destindex_copy_quantize_and_register_kv(batch, a["new_len"], a["begin"], a["end"], a["cumsum"], a["kv"], a["start"], a["cur"], a["mem"],
                                                   a["codes"], a["scales"], a["table"], a["b_req"], 0, 4, True)


def test_the_keep_range_write_looks_where_every_tensor_lies(monkeypatch):
    """The kernel reads all of them: a vector left on the host must not get as far as the launch."""
    from loongserve_b200 import kv_ops
    a = keep_range_args(2)
    seen = []
    monkeypatch.setattr(kv_ops, "need_here", lambda *ts: seen.extend(id(t) for t in ts))
    monkeypatch.setattr(kv_ops, "need_i32", lambda *ts: (_ for _ in ()).throw(InterruptedError))
    with pytest.raises(InterruptedError):
        keep_range(a, 2)
    assert {k for k, t in a.items() if id(t) not in seen} == set()


@pytest.mark.parametrize("short", ["new_len", "begin", "end", "start", "cur", "b_req", "cumsum"])
def test_the_keep_range_write_wants_an_entry_for_every_request(monkeypatch, short):
    from loongserve_b200 import kv_ops
    a = keep_range_args(3)
    a[short] = a[short][:2]
    monkeypatch.setattr(kv_ops, "need_here", lambda *ts: 0)
    monkeypatch.setattr(kv_ops._lib, "attn", lambda: pytest.fail("a launch"))
    with pytest.raises(AssertionError, match="every request"):
        keep_range(a, 3)


def decode_step(monkeypatch, peers, **kw):
    """A decode step of two requests on an 8-bit pool, without its kernels: (state, arguments that attention got)."""
    from loongserve_b200 import attention_runtime as ar
    monkeypatch.setattr(ar.kv_ops, "copy_kv_index_to_req", lambda *a: None)
    got = []
    monkeypatch.setattr(ar.fd, "token_decode_attention_q8", lambda q, *a, **k: (got.append((a, k)), (q, None))[1])
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)
    rt = ar.ESPAttentionRuntime(layers_num=1, q_head_num=4, kv_head_num=2, head_dim=128, max_total_token_num=2048, max_req_num=4, max_seq_length=1024,
                                device="cpu", kv_dtype=torch.int8, **kw)
    st = rt.prepare_decode(2, 2, 700, i32(0, 1), i32(700, 30), i32(699, 29), 0, peers, 0)
    if len(peers) == 1:
        rt.token_attention(torch.zeros(2, 4, 128, dtype=torch.bfloat16), st, 0)
    return st, got


@pytest.mark.parametrize("block", [None, 64, 100])
def test_splits_asked_for_reach_attention_over_an_8_bit_pool(monkeypatch, block):
    st, got = decode_step(monkeypatch, [0], decode_block_seq=block)
    (args, kw), = got
    assert kw["block_seq"] == block and args[-1] == 700 and kw["out_logexpsum"] is st.global_out_logexpsum


def test_a_step_of_one_instance_holds_no_partials_that_nothing_reads(monkeypatch):
    st, _ = decode_step(monkeypatch, [0])
    assert st.global_mid_o is None and st.global_mid_o_logexpsum is None and st.global_out_logexpsum.shape == (2, 4)
    st, _ = decode_step(monkeypatch, [0, 1], sp_world_size=2)
    assert st.global_mid_o.shape == (1 + 3, 2, 4, 128) and st.master_plan.global_mid_lse.shape == (1 + 3, 2, 4)


@pytest.mark.parametrize("words,names", [
    ([[(-4, 3, 101, 7)], [], []], ["8-bit product"]), ([[(-4, 3, 6, 7)], [], []], ["prefill kernel"]),
    ([[(-4, 3, 6, 7), (-4, 0, 104, 1)], [(-4, 1, 2, 5), (-4, 1, 9, 5)], [(-8, 1, 0, 3), (-8, 6, 0, 3)]],
     ["prefill kernel", "8-bit product", "decode kernels / flag waits", "8-bit decode kernel", "KV pool kernels", "8-bit KV pool kernels"]),
    ([[], [(-8, 0, 0, 99)], [(-8, 7, 2, -1)]], ["decode kernels / flag waits", "8-bit KV pool kernels"]), ([[], [], []], [])])
def test_the_device_status_names_every_kernel_that_reported(monkeypatch, words, names):
    from loongserve_b200 import attention_runtime as ar
    for mod, left in zip((ar.ca, ar.fd, ar.kv_ops), words):
        monkeypatch.setattr(mod, "device_status", lambda clear=True, left=list(left): left.pop(0) if left else (0, 0, 0, 0))
    check = lambda: ar.ESPAttentionRuntime.check_device_status(SimpleNamespace())
    if names:
        with pytest.raises(RuntimeError) as e:
            check()
        assert [part.split(":")[0] for part in str(e.value).removeprefix("ESP attention device status, ").split("; ")] == names
    check()                                     # all of it has been read
