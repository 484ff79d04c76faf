"""Argument checks of the 8-bit serving path: every refusal is decided on the host, before any CUDA call (no GPU needed)."""
import ctypes as C

import pytest
import torch

BAD, ALIGN, UNSUP, LARGE = -1, -2, -5, -7
P = 0x10000            # an aligned address that no refused call looks behind


@pytest.fixture(scope="module")
def lib():
    from loongserve_b200 import _lib, build
    build.build_attention(force=False)
    return _lib.attn()


def call(fn, base, **change):
    args = dict(base)
    assert set(change) <= set(args), "unknown argument"
    args.update(change)
    return fn(*args.values())


SCATTER = dict(src=P, src_row=256, src_head=128, codes=P, codes_row=272, codes_head=128, scales=P, scales_row=68, dest=P, idx64=1, n=4, heads2=2,
               head_dim=128, dtype=1, code=0, pool_rows=9, stream=None)


@pytest.mark.parametrize("change,rc", [
    (dict(n=0), 0), (dict(n=-1), BAD), (dict(src=None), BAD), (dict(codes=None), BAD), (dict(scales=None), BAD), (dict(dest=None), BAD),
    (dict(heads2=0), BAD), (dict(head_dim=0), BAD), (dict(head_dim=272), UNSUP), (dict(head_dim=24), ALIGN), (dict(dtype=2), BAD), (dict(dtype=7), BAD),
    (dict(code=2), BAD), (dict(code=-1), BAD), (dict(pool_rows=0), BAD), (dict(src=P + 8), ALIGN), (dict(src_row=252), ALIGN), (dict(src_head=4), ALIGN),
    (dict(codes=P + 4), ALIGN), (dict(codes_row=264), ALIGN), (dict(codes_head=120), ALIGN), (dict(scales=P + 2), BAD), (dict(scales_row=1), BAD)])
def test_scatter(lib, change, rc):
    assert call(lib.esp_kv_scatter_q8, SCATTER, **change) == rc


GATHER = dict(out=P, out_row=256, out_head=128, codes=P, codes_row=272, codes_head=128, scales=P, scales_row=68, src=P, idx64=0, n=4, heads2=2, head_dim=128,
              dtype=1, code=0, pool_rows=9, stream=None)


@pytest.mark.parametrize("change,rc", [
    (dict(n=0), 0), (dict(n=-3), BAD), (dict(out=None), BAD), (dict(src=None), BAD), (dict(dtype=3), BAD), (dict(code=5), BAD), (dict(out=P + 2), ALIGN),
    (dict(out_row=4), ALIGN), (dict(dtype=2, out_row=2), ALIGN), (dict(codes_row=8), ALIGN), (dict(head_dim=1024), UNSUP), (dict(pool_rows=-1), BAD)])
def test_gather(lib, change, rc):
    assert call(lib.esp_kv_gather_q8, GATHER, **change) == rc


REGISTER = dict(batch=2, new_len=P, begin=P, end=P, cumsum=P, kv=P, kv_row=256, kv_head=128, start=P, cur=P, mem=P, idx64=0, codes=P, codes_row=272,
                codes_head=128, scales=P, scales_row=68, table=P, table_row=8, b_req=P, used=0, max_len=5, register=1, heads2=2, head_dim=128, dtype=1,
                code=0, pool_rows=9, stream=None)


@pytest.mark.parametrize("change,rc", [
    (dict(batch=0), 0), (dict(max_len=0), 0), (dict(batch=-1), BAD), (dict(batch=70000), LARGE), (dict(new_len=None), BAD), (dict(cumsum=None), BAD),
    (dict(table=None), BAD), (dict(b_req=None), BAD), (dict(cur=None), BAD), (dict(kv=P + 2), ALIGN), (dict(kv_row=3), ALIGN), (dict(dtype=2), BAD),
    (dict(code=9), BAD), (dict(codes_row=100), ALIGN)])
def test_scatter_register(lib, change, rc):
    assert call(lib.esp_kv_scatter_register_q8, REGISTER, **change) == rc


DECODE = dict(mid_o=P, mid_lse=P, q=P, k=P, v=P, ks=P, vs=P, kst=528, ksh=128, vst=528, vsh=128, kss=132, vss=132, table=P, table_row=64, rows=4, cols=64,
              b_req=P, b_len=P, batch=2, hq=8, hkv=2, dim=128, max_len=50, block=16, dtype=1, code=0, sm=C.c_float(0.0), pool=100, stream=None)


@pytest.mark.parametrize("change,rc", [
    (dict(batch=0), 0), (dict(max_len=0), 0), (dict(batch=-2), BAD), (dict(mid_o=None), BAD), (dict(q=None), BAD), (dict(k=None), BAD), (dict(vs=None), BAD),
    (dict(table=None), BAD), (dict(b_len=None), BAD), (dict(hq=9), BAD), (dict(hkv=0), BAD), (dict(block=0), BAD), (dict(rows=0), BAD), (dict(cols=0), BAD),
    (dict(pool=0), BAD), (dict(dtype=2), BAD), (dict(code=2), BAD), (dict(dim=64), UNSUP), (dict(batch=65536), LARGE), (dict(hq=65536, hkv=1), LARGE),
    (dict(q=P + 8), ALIGN), (dict(k=P + 8), ALIGN), (dict(kst=520), ALIGN), (dict(vsh=8), ALIGN), (dict(ks=P + 1), ALIGN),
    (dict(mid_o=P + 4), ALIGN), (dict(mid_lse=P + 2), ALIGN)])
def test_decode_stage1(lib, change, rc):
    assert call(lib.esp_decode_stage1_q8, DECODE, **change) == rc


@pytest.mark.parametrize("change,rc", [
    (dict(batch=0), 0), (dict(o=None), BAD), (dict(lse=None), BAD), (dict(work=None), BAD), (dict(work=P + 4), ALIGN), (dict(o=P + 8), ALIGN), (dict(lse=P + 1), ALIGN), (dict(block=-1), BAD),
    (dict(max_len=-1), BAD), (dict(odt=3), BAD), (dict(batch=385), LARGE), (dict(batch=384, max_len=2147483647), LARGE), (dict(hq=0), BAD),
    (dict(q=None), BAD), (dict(kst=520), ALIGN), (dict(dim=64), UNSUP), (dict(block=16, work=None), BAD)])
def test_decode_attention(lib, change, rc):
    """block 0: the tokens are divided evenly."""
    base = dict(o=P, lse=P, work=P, **{k: v for k, v in DECODE.items() if k not in ("mid_o", "mid_lse")})
    base.update(max_len=5000, block=0)
    keys = list(base); at = keys.index("dtype") + 1
    base = {**{k: base[k] for k in keys[:at]}, "odt": 1, **{k: base[k] for k in keys[at:]}}
    assert call(lib.esp_decode_attention_q8, base, **change) == rc


@pytest.mark.parametrize("change,rc", [
    (dict(tokens=0), 0), (dict(tokens=-1), BAD), (dict(hidden=0), BAD), (dict(hidden=60), ALIGN), (dict(hidden=65544), LARGE), (dict(dtype=2), BAD),
    (dict(inp=None), BAD), (dict(weight=None), BAD), (dict(residual=P + 4), ALIGN), (dict(inp=P + 2), ALIGN), (dict(weight=P + 8), ALIGN),
    (dict(tokens=1 << 31), LARGE)])
def test_norms(lib, change, rc):
    base = dict(out=P, residual=P, inp=P, weight=P, tokens=3, hidden=64, eps=C.c_float(1e-5), dtype=1, stream=None)
    assert call(lib.esp_add_rms_norm, base, **change) == rc
    base = dict(codes=P, scale=P, residual=P, inp=P, weight=P, tokens=3, hidden=64, eps=C.c_float(1e-5), dtype=1, stream=None)
    assert call(lib.esp_add_rms_norm_q8, base, **change) == rc
    assert call(lib.esp_add_rms_norm_q8, base, codes=None) == BAD and call(lib.esp_add_rms_norm_q8, base, scale=None) == BAD
    assert call(lib.esp_add_rms_norm_q8, base, codes=P + 8) == ALIGN


def test_row_quantisers(lib):
    silu = dict(codes=P, scale=P, io=P, tokens=3, ffn=64, dtype=0, stream=None)
    assert [call(lib.esp_silu_and_mul_q8, silu, **c) for c in (dict(tokens=0), dict(io=None), dict(ffn=4), dict(ffn=65544), dict(dtype=2), dict(io=P + 4))] == \
        [0, BAD, ALIGN, LARGE, BAD, ALIGN]
    rows = dict(codes=P, scale=P, x=P, x_row=64, rows=3, cols=64, dtype=0, stream=None)
    assert [call(lib.esp_quantize_rows, rows, **c) for c in (dict(rows=0), dict(x=None), dict(cols=4), dict(x_row=60), dict(dtype=2), dict(x=P + 4))] == \
        [0, BAD, ALIGN, ALIGN, BAD, ALIGN]
    back = dict(out=P, codes=P, scale=P, rows=3, cols=64, dtype=2, stream=None)
    assert [call(lib.esp_dequantize_rows, back, **c) for c in (dict(rows=0), dict(out=None), dict(cols=4), dict(dtype=3), dict(out=P + 4), dict(codes=P + 4))] == \
        [0, BAD, ALIGN, BAD, ALIGN, ALIGN]


@pytest.mark.parametrize("change,rc", [
    (dict(m=0), 0), (dict(n=0), 0), (dict(m=-1), BAD), (dict(k=0), BAD), (dict(out=None), BAD), (dict(sa=None), BAD), (dict(w=None), BAD), (dict(ldo=7), BAD),
    (dict(lda=16), BAD), (dict(ldw=16), BAD), (dict(k=24, lda=32, ldw=32), ALIGN), (dict(lda=40), ALIGN), (dict(ldw=72), ALIGN), (dict(a=P + 8), ALIGN),
    (dict(w=P + 1), ALIGN), (dict(k=131072, lda=131072, ldw=131072), LARGE), (dict(dtype=4), BAD), (dict(dtype=-1), BAD), (dict(m=1 << 40), LARGE)])
def test_mm(lib, change, rc):
    base = dict(out=P, ldo=8, a=P, lda=32, sa=P, w=P, ldw=32, sw=P, m=4, n=8, k=32, dtype=1, stream=None)
    assert call(lib.esp_mm_w8a8, base, **change) == rc


# ---------------------------------------------------------------------------------------- the Python entry points
def test_python_entry_points_refuse_cpu_tensors():
    from loongserve_b200 import flash_decoding as fd, kv_ops, layer_ops as ops
    x, c, s = torch.zeros(2, 2, 128, dtype=torch.bfloat16), torch.zeros(4, 2, 128, dtype=torch.int8), torch.zeros(4, 2)
    r, i = torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int32)
    c2, s2, w = torch.zeros(2, 64, dtype=torch.int8), torch.zeros(2), torch.zeros(64, dtype=torch.bfloat16)
    for fn in (lambda: kv_ops.destindex_copy_quantize_kv(x, i, c, s), lambda: kv_ops.gather_dequantize_kv(c, s, i), lambda: ops.add_rms_norm(r, r, w, 1e-5),
               lambda: ops.add_rms_norm_quant(r, None, w, 1e-5), lambda: ops.silu_and_mul_quant(r), lambda: ops.quantize_rows(r),
               lambda: ops.dequantize_rows(c2, s2), lambda: ops.mm_w8a8(c2, s2, c2, s2),
               lambda: fd.token_decode_attention_q8(x, c[:, :1], s[:, :1], c[:, 1:], s[:, 1:], torch.zeros(2, 8, dtype=torch.int32), i, i, 4)):
        with pytest.raises(RuntimeError, match="CUDA"):
            fn()


class _On:
    """Stands for a tensor on a given CUDA device."""

    def __init__(self, index):
        self.is_cuda, self.device, self.index = True, f"cuda:{index}", index

    def get_device(self):
        return self.index


def test_tensors_of_another_device_are_refused(monkeypatch):
    from loongserve_b200 import _util
    monkeypatch.setattr(_util, "current_device", lambda: 0)
    _util.need_here(_On(0), None, _On(0))
    with pytest.raises(RuntimeError, match="current CUDA device"):
        _util.need_here(_On(0), _On(1))
    with pytest.raises(RuntimeError, match="current CUDA device"):
        _util.need_here(_On(1), _On(1))


@pytest.fixture
def no_device_check(monkeypatch):
    """Lets the shape checks of the wrappers be reached with CPU tensors; none of the calls below gets past them."""
    from loongserve_b200 import flash_decoding, kv_ops, layer_ops
    for mod in (flash_decoding, kv_ops, layer_ops):
        monkeypatch.setattr(mod, "need_here", lambda *a: None)
        monkeypatch.setattr(mod, "stream_of", lambda device: 0)

    class Refuse:
        def __getattr__(self, name):
            def reached(*args):
                raise AssertionError("a refused call reached the library")
            return reached
    for mod in (flash_decoding, kv_ops, layer_ops):
        monkeypatch.setattr(mod._lib, "attn", lambda: Refuse())


def test_python_entry_points_check_shapes_and_types(no_device_check):
    from loongserve_b200 import flash_decoding as fd, kv_ops, layer_ops as ops
    bf = torch.bfloat16
    x, c, s, i = torch.zeros(2, 2, 128, dtype=bf), torch.zeros(4, 2, 128, dtype=torch.int8), torch.zeros(4, 2), torch.zeros(2, dtype=torch.int32)
    bad = [
        lambda: kv_ops.destindex_copy_quantize_kv(x, i, c[:, :1], s[:, :1]), lambda: kv_ops.destindex_copy_quantize_kv(x, i, c, s[:3]),
        lambda: kv_ops.destindex_copy_quantize_kv(x, torch.zeros(3, dtype=torch.int32), c, s), lambda: kv_ops.destindex_copy_quantize_kv(x, i, c, s.double()),
        lambda: kv_ops.destindex_copy_quantize_kv(x, i, c.to(torch.uint8), s), lambda: kv_ops.destindex_copy_quantize_kv(x, i.float(), c, s),
        lambda: kv_ops.destindex_copy_quantize_kv(x.double(), i, c, s), lambda: kv_ops.destindex_copy_quantize_kv(x.transpose(1, 2), i, c, s),
        lambda: kv_ops.destindex_copy_quantize_kv(x, i, c, torch.zeros(2, 4).t()),
        lambda: kv_ops.gather_dequantize_kv(c, s, i, torch.float64), lambda: kv_ops.gather_dequantize_kv(c, s, i, out=torch.zeros(3, 2, 128)),
        lambda: kv_ops.gather_dequantize_kv(c, s, i, bf, out=torch.zeros(2, 2, 128)), lambda: kv_ops.gather_dequantize_kv(c, s, i[None]),
    ]
    r, w = torch.zeros(2, 64, dtype=bf), torch.zeros(64, dtype=bf)
    c2, s2 = torch.zeros(2, 64, dtype=torch.int8), torch.zeros(2)
    bad += [
        lambda: ops.add_rms_norm(r, r[:1], w, 1e-5), lambda: ops.add_rms_norm(r, r.half(), w, 1e-5), lambda: ops.add_rms_norm(r, r, w[:32], 1e-5),
        lambda: ops.add_rms_norm(r, r, w.float(), 1e-5), lambda: ops.add_rms_norm(r.t(), r.t(), w[:2], 1e-5), lambda: ops.add_rms_norm(r, r, w, 1e-5, out=r.float()),
        lambda: ops.add_rms_norm_quant(r, None, w, 1e-5, out=r), lambda: ops.add_rms_norm_quant(r, None, w, 1e-5, out=c2, out_scale=s2[:1]),
        lambda: ops.add_rms_norm(r.float(), r.float(), w.float(), 1e-5),
        lambda: ops.silu_and_mul_quant(r[:, :63]), lambda: ops.silu_and_mul_quant(r.t()), lambda: ops.silu_and_mul_quant(r, out=c2),
        lambda: ops.quantize_rows(r.t()), lambda: ops.quantize_rows(r.float()), lambda: ops.dequantize_rows(c2, s2[:1]), lambda: ops.dequantize_rows(c2.float(), s2),
        lambda: ops.dequantize_rows(c2, s2, torch.float64),
        lambda: ops.mm_w8a8(c2, s2, c2[:, :32], s2), lambda: ops.mm_w8a8(c2, s2[:1], c2, s2), lambda: ops.mm_w8a8(c2, s2, c2, s2.double()),
        lambda: ops.mm_w8a8(c2.float(), s2, c2, s2), lambda: ops.mm_w8a8(c2.t(), torch.zeros(64), c2.t(), torch.zeros(64)),
        lambda: ops.mm_w8a8(c2, s2, c2, s2, out=torch.zeros(3, 2)), lambda: ops.mm_w8a8(c2, s2, c2, s2, out_dtype=torch.float64),
    ]
    t = torch.zeros(2, 8, dtype=torch.int32)
    good = dict(q=x, cache_k=c[:, :1], k_scale=s[:, :1], cache_v=c[:, 1:], v_scale=s[:, 1:], req_to_token_indexs=t, b_req_idx=i, b_seq_len=i, max_len_in_batch=4)
    for change in (dict(b_req_idx=i.long()), dict(b_seq_len=i[:1]), dict(k_scale=s[:3, :1]), dict(v_scale=s[:, 1:].half()), dict(cache_v=c[:, 1:].view(torch.float8_e4m3fn)),
                   dict(req_to_token_indexs=t.long()), dict(q=x.float()), dict(q=torch.zeros(2, 2, 64, dtype=bf)), dict(cache_k=c[:, :1].float(), cache_v=c[:, 1:].float()),
                   dict(req_to_token_indexs=t.t()), dict(out=x.double()), dict(out=x[:1])):
        bad.append(lambda change=change: fd.token_decode_attention_q8(**{**good, **change}))
    for n, fn in enumerate(bad):
        with pytest.raises((AssertionError, TypeError)) as e:
            fn()
        assert "reached the library" not in str(e.value), n
