"""The 8-bit serving path on one GPU, each operator against its definition in 64 bits: the KV pool held in 8 bits (quantising
write, keep-range write, read-back, decode attention), the row-quantising layer kernels and the 8-bit integer product, and
a run of them together.

Tolerances count roundings: half a step of the output type (finfo.eps / 2, relative), 2^-24 per fp32 operation, and for
codes half a step of the row's scale.  Whole numbers (codes, int32 sums) and scales of stored rows have to be equal."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
D = 128
TINY = 2.0 ** -100
F16, BF16 = torch.float16, torch.bfloat16
INT8, E4M3 = torch.int8, torch.float8_e4m3fn
TOP = {INT8: 127.0, E4M3: 448.0}
U32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def quantise(x, code):
    """Codes and scales of the rows of x by the definition: fp32 scale and factor, int8 products rounded once (64 bits)."""
    amax = x.float().abs().amax(-1, keepdim=True)
    bad = ~torch.isfinite(x.float()).all(-1, keepdim=True)
    amax = torch.where(bad, torch.ones_like(amax), amax).clamp_min(TINY)
    inv = torch.tensor(TOP[code], dtype=torch.float32) / amax.cpu()
    scale = (amax.cpu() / torch.tensor(TOP[code], dtype=torch.float32))
    xs = torch.where(bad, torch.zeros_like(x.float()), x.float()).cpu()
    c = torch.round(xs.double() * inv.double()).to(INT8) if code is INT8 else (xs * inv).to(E4M3)
    return c, torch.where(bad.cpu(), torch.full_like(scale, math.nan), scale).squeeze(-1)


def pool(rows, heads2, code, head_dim=D, pad=0, fill=7):
    """Codes [rows, heads2, head_dim] and scales [rows, heads2] as views of one byte row per slot; `pad` more bytes per row."""
    width = (heads2 * (head_dim + 4) + 15) // 16 * 16 + pad
    raw = torch.full((rows, width), fill, dtype=torch.uint8, device=DEV)
    codes = raw[:, :heads2 * head_dim].view(code).unflatten(1, (heads2, head_dim))
    return raw, codes, raw[:, heads2 * head_dim:heads2 * (head_dim + 4)].view(torch.float32)


def bits(t):
    return t.contiguous().view(torch.uint8).cpu()


# ------------------------------------------------------------------------------------------------ writing and reading back
@pytest.mark.parametrize("code", [INT8, E4M3])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n,heads2,head_dim,idx", [(1, 2, 128, torch.int64), (37, 6, 128, torch.int32), (300, 64, 128, torch.int64),
                                                   (33, 4, 80, torch.int32), (9, 2, 16, torch.int64), (5, 2, 256, torch.int64),
                                                   (3, 2, 208, torch.int32), (1025, 2, 64, torch.int64)])
def test_write_and_read_back(code, dtype, n, heads2, head_dim, idx):
    from loongserve_b200 import kv_ops
    g = torch.Generator().manual_seed(n * 7 + heads2)
    rows = n + 13
    src = (torch.randn(n + 2, heads2 + 1, head_dim + 16, generator=g) * torch.exp(2 * torch.randn(n + 2, heads2 + 1, 1, generator=g))).to(dtype)
    src_g = src.to(DEV)[:n, 1:, 8:8 + head_dim]                                # strided on every level, 16-byte aligned
    src = src[:n, 1:, 8:8 + head_dim]
    dest = torch.randperm(rows, generator=g)[:n].to(idx)
    raw, codes, scales = pool(rows, heads2, code, head_dim, pad=32)
    before = raw.clone()
    kv_ops.destindex_copy_quantize_kv(src_g, dest.to(DEV), codes, scales)
    rc, rs = quantise(src, code)
    d = dest.long()
    assert torch.equal(bits(codes)[d], bits(rc)) and torch.equal(scales.cpu()[d], rs)
    untouched = torch.ones(rows, dtype=torch.bool); untouched[d] = False
    assert torch.equal(raw.cpu()[untouched], before.cpu()[untouched])          # other slots keep every byte
    assert torch.equal(raw[:, heads2 * (head_dim + 4):], before[:, heads2 * (head_dim + 4):])   # and the padding of a row
    for odt in (F16, BF16, torch.float32):
        back = kv_ops.gather_dequantize_kv(codes, scales, dest.to(DEV), odt).cpu().double()
        want = rc.double() * rs.double()[..., None]
        tiny = 2.0 ** -25 if odt is F16 else 0.0                                # fp16 goes subnormal below 2^-14
        fit = want.abs() < torch.finfo(odt).max
        assert bool(((back - want).abs() <= (half_step(odt) + U32) * want.abs() + tiny)[fit].all())
    wide = torch.full((n, heads2 + 1, head_dim + 8), 5.0, dtype=dtype, device=DEV)
    kv_ops.gather_dequantize_kv(codes, scales, dest.to(DEV), out=wide[:, :heads2, :head_dim])
    assert bool((wide[:, heads2:] == 5).all()) and bool((wide[:, :, head_dim:] == 5).all())
    assert torch.equal(wide[:, :heads2, :head_dim], kv_ops.gather_dequantize_kv(codes, scales, dest.to(DEV), dtype))
    assert kv_ops.device_status()[0] == 0


@pytest.mark.parametrize("code", [INT8, E4M3])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_rows_at_the_ends_of_the_range(code, dtype):
    """Zeros, the smallest and the largest finite numbers, ties between two codes, infinities and NaN."""
    from loongserve_b200 import kv_ops
    fi = torch.finfo(dtype)
    x = torch.zeros(9, 2, D, dtype=dtype)
    x[1] = fi.tiny
    x[2, :, ::2] = fi.max; x[2, :, 1::2] = -fi.max / 2
    x[3, :, 0] = 127.0; x[3, :, 1:120] = torch.arange(119) / 2.0            # with amax = 127 every odd half is a tie
    x[4] = torch.randn(2, D); x[4, 0, 5] = math.inf
    x[5] = torch.randn(2, D); x[5, 1, 127] = math.nan
    x[6] = torch.randn(2, D); x[6, 0, 64] = -math.inf; x[6, 0, 65] = math.nan
    x[7, :, 3] = -1.0; x[7, :, 4] = 0.5
    x[8, :, 0] = 448.0; x[8, :, 1:] = torch.linspace(-448, 448, D - 1)
    raw, codes, scales = pool(9, 2, code)
    kv_ops.destindex_copy_quantize_kv(x.to(DEV), torch.arange(9, device=DEV), codes, scales)
    rc, rs = quantise(x, code)
    assert torch.equal(bits(codes), bits(rc))
    assert torch.equal(scales.cpu().isnan(), rs.isnan()) and torch.equal(scales.cpu().nan_to_num(-1), rs.nan_to_num(-1))
    assert rs.isnan().tolist() == [[False] * 2] * 4 + [[True, False], [False, True], [True, False]] + [[False] * 2] * 2
    back = kv_ops.gather_dequantize_kv(codes, scales, torch.arange(9, device=DEV), torch.float32).cpu()
    assert bool(back[4, 0].isnan().all()) and not bool(back[4, 1].isnan().any())
    assert bool((back[0] == 0).all())


def test_slots_outside_the_pool_are_skipped_and_reported():
    from loongserve_b200 import kv_ops
    kv_ops.device_status()
    x = torch.randn(4, 2, D, dtype=torch.float32).to(BF16).to(DEV)
    raw, codes, scales = pool(10, 2, INT8)
    before = raw.clone()
    kv_ops.destindex_copy_quantize_kv(x, torch.tensor([3, -1, 2147483647, 10], device=DEV), codes, scales)
    st = kv_ops.device_status()
    assert st[0] == -8 and st[1] == 5 and st[3] in (-1, 2147483647, 10)
    keep = [i for i in range(10) if i != 3]
    assert torch.equal(raw[keep], before[keep]) and torch.equal(bits(codes[3]), bits(quantise(x[:1].cpu(), INT8)[0][0]))
    back = kv_ops.gather_dequantize_kv(codes, scales, torch.tensor([3, 10, -5], device=DEV), torch.float32)
    assert kv_ops.device_status()[:2] == (-8, 7) and kv_ops.device_status()[0] == 0
    assert bool((back[1:] == 0).all()) and bool((back[0] != 0).any())


@pytest.mark.parametrize("code", [INT8, E4M3])
def test_keep_range_write_equals_the_16_bit_form(code):
    """Same rows, same registrations as destindex_copy_and_register_kv, quantised."""
    from loongserve_b200 import kv_ops
    g = torch.Generator().manual_seed(3)
    lens, P, heads2 = [700, 1, 300, 64, 5], 3, 4
    B = len(lens)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    begin, end, first = i32([10, 0, 30, 0, 9]), i32([600, 2, 200, 0, 9]), i32([1, 0, 2, 1, 0])
    rb, re, nl = kv_ops.pre_copy_and_register_kv(begin, end, first, P)
    cs = torch.cumsum(nl, 0, dtype=torch.int64)
    total = int(cs[-1])
    start = torch.cumsum(i32(lens), 0, dtype=torch.int32) - i32(lens)
    kv = torch.randn(sum(lens), heads2, D, generator=g).to(BF16).to(DEV)
    mem = torch.randperm(total + 40, generator=g).to(DEV)
    b_req, cur = i32([4, 1, 0, 6, 2]), i32([2, 0, 5, 0, 1])
    tables = [torch.full((7, 800), 2147483647, dtype=torch.int32, device=DEV) for _ in range(2)]
    full = torch.zeros(total + 40, heads2, D, dtype=BF16, device=DEV)
    raw, codes, scales = pool(total + 40, heads2, code, fill=0)
    args = (B, nl, rb, re, cs, kv, start, cur, mem)
    kv_ops.destindex_copy_and_register_kv(*args, full, tables[0], b_req, 3, max(lens), True)
    kv_ops.destindex_copy_quantize_and_register_kv(*args, codes, scales, tables[1], b_req, 3, max(lens), True)
    assert torch.equal(tables[0], tables[1])
    kept = mem[3:3 + total]
    rc, rs = quantise(full[kept].cpu(), code)
    assert total > 200 and torch.equal(bits(codes[kept]), bits(rc)) and torch.equal(scales[kept].cpu(), rs)
    rest = torch.ones(total + 40, dtype=torch.bool, device=DEV); rest[kept] = False
    assert bool((raw[rest] == 0).all())


# ------------------------------------------------------------------------------------------------ decode attention
def decode_case(lens, hq, hkv, dtype, code, seed, q_scale=1.5, pool_extra=3):
    g = torch.Generator().manual_seed(seed)
    B, total = len(lens), sum(lens)
    kv = torch.randn(total + pool_extra, 2 * hkv, D, generator=g) * torch.exp(0.7 * torch.randn(total + pool_extra, 2 * hkv, 1, generator=g))
    rc, rs = quantise(kv.to(dtype), code)
    raw, codes, scales = pool(total + pool_extra, 2 * hkv, code)
    codes.copy_(rc.to(DEV)); scales.copy_(rs.to(DEV))
    table = torch.full((B + 2, max(max(lens), 1) + 3), 2147483647, dtype=torch.int32)
    rows = torch.randperm(B + 2, generator=g)[:B].to(torch.int32)
    perm = torch.randperm(total + pool_extra, generator=g).to(torch.int32)
    at = 0
    for b, n in enumerate(lens):
        table[int(rows[b]), :n] = perm[at:at + n]; at += n
    q = (q_scale * torch.randn(B, hq, D, generator=g)).to(dtype)
    return dict(q=q.to(DEV), codes=codes, scales=scales, table=table.to(DEV), rows=rows.to(DEV), lens=torch.tensor(lens, dtype=torch.int32, device=DEV),
                hkv=hkv, raw=raw)


def decode_exact(c, lens=None, sm_scale=None):
    """(o, lse, sum p|v| / sum p, max over tokens of sum|q k| * sm_scale, the same of max|q| * sum|k|, tokens * largest v scale * top
    code) in 64 bits."""
    B, hq, _ = c["q"].shape
    hkv = c["hkv"]
    sm = sm_scale or D ** -0.5
    o = torch.zeros(B, hq, D, dtype=torch.float64); lse = torch.full((B, hq), -math.inf, dtype=torch.float64)
    wabs = torch.zeros_like(o); sabs = torch.zeros(B, hq, dtype=torch.float64)
    floor = torch.zeros(B, hq, 1, dtype=torch.float64); qabs = torch.zeros_like(sabs)
    for b, n in enumerate(lens if lens is not None else c["lens"].tolist()):
        if n == 0:
            continue
        slots = c["table"][int(c["rows"][b]), :n].long()
        slots = slots[(slots >= 0) & (slots < c["codes"].shape[0])]
        if len(slots) == 0:
            continue
        x = c["codes"].view(torch.uint8)[slots].view(c["codes"].dtype).double() * c["scales"][slots].double()[..., None]
        k, v = x[:, :hkv].repeat_interleave(hq // hkv, 1), x[:, hkv:].repeat_interleave(hq // hkv, 1)      # [n, hq, D]
        q = c["q"][b].double()
        s = (q[None] * k).sum(-1) * sm
        p = torch.softmax(s, 0)
        o[b] = (p[..., None] * v).sum(0).cpu(); wabs[b] = (p[..., None] * v.abs()).sum(0).cpu()
        lse[b] = torch.logsumexp(s, 0).cpu()
        sabs[b] = ((q[None] * k).abs().sum(-1) * sm).amax(0).cpu()
        qabs[b] = (q.abs().amax(-1)[None] * k.abs().sum(-1) * sm).amax(0).cpu()
        top = c["scales"][slots, hkv:].double().amax(0).repeat_interleave(hq // hkv) * TOP[c["codes"].dtype]
        floor[b, :, 0] = len(slots) * top.cpu()
    return o, lse, wabs, sabs, qabs, floor


def check_decode(o, lse, ref, n_max):
    """Roundings.  A score is a sum of 128 products and three factors, at most 131 * 2^-24 of sum|q k|, of a query whose
    elements are held to 2^-22 of the largest (int8 codes: rounded to integers, the largest at least 2^21 of them; e4m3: f16, the largest
    scaled to [2^7, 2^8), exact but below f16's normal range, 2^-25 * 2^-7).  p carries the score's error and one more of 2^-22 (ex2).  The weight p * v_scale * 2^12 / v_ref with v_ref <= 4 * the
    largest v_scale, while some p is 1 and so sum p >= 1, is held as the f16 rounding of itself and of what that left (2^-22 relative;
    below f16's normal range 2^-25 absolute: at most 2^-25 * 4 / 2^12 = 2^-35 of the largest v_scale * top code for each of n tokens).
    Sums of n terms in fp32 lose at most n * 2^-24 of the sum of magnitudes; the output is rounded once."""
    ro, rl, wabs, sabs, qabs, floor = ref
    ds = 131 * U32 * sabs + 2.0 ** -22 * qabs
    tol = ((2.0 ** -22 + 2.0 ** -20 + 2 * min(n_max, 4096) * U32) + 2 * ds)[..., None] * wabs
    tol = tol + 2.0 ** -35 * floor + (half_step(o.dtype) if o.dtype != torch.float32 else U32) * ro.abs() * 1.01 + 1e-30
    if o.dtype == F16:
        tol = tol + 2.0 ** -25
    err = (o.double().cpu() - ro).abs()
    assert bool((err <= tol).all()), ((err / tol).max(), err.max())
    fin = torch.isfinite(rl)
    assert torch.equal(torch.isfinite(lse.cpu()), fin)
    ltol = ds + 2.0 ** -20 + 4 * U32 * rl.abs()
    lerr = (lse.double().cpu() - rl).abs()
    assert bool((lerr[fin] <= ltol[fin]).all()), (lerr[fin] / ltol[fin]).max()


@pytest.mark.parametrize("code", [INT8, E4M3])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hq,hkv", [(32, 32), (8, 2), (10, 2), (16, 1), (3, 3), (20, 1), (12, 4), (48, 3)])
def test_decode_attention_matches_the_definition(code, dtype, hq, hkv):
    from loongserve_b200 import flash_decoding as fd
    lens = [1, 300, 0, 257, 1025, 64, 15, 17]
    c = decode_case(lens, hq, hkv, dtype, code, seed=hq * 100 + hkv)
    k, v, ks, vs = c["codes"][:, :hkv], c["codes"][:, hkv:], c["scales"][:, :hkv], c["scales"][:, hkv:]
    ref = decode_exact(c)
    for block in (None, 16, 100, 256, 2000):
        for odt in (dtype, torch.float32):
            out = torch.full((len(lens), hq, D), 9.0, dtype=odt, device=DEV)
            lse = torch.full((len(lens), hq), 9.0, device=DEV)
            fd.token_decode_attention_q8(c["q"], k, ks, v, vs, c["table"], c["rows"], c["lens"], max(lens), block, out, lse)
            check_decode(out, lse, ref, max(lens))
            assert bool((out[2] == 0).all()) and bool((lse[2] == -math.inf).all())
    assert fd.device_status()[0] == 0


@pytest.mark.parametrize("code", [INT8, E4M3])
def test_decode_partials_are_the_blocks_own_attention(code):
    """Stage 1 writes block j of a request from its tokens alone, and leaves blocks behind the length as they were."""
    from loongserve_b200 import flash_decoding as fd
    lens, bs, hq, hkv = [130, 1, 0, 64], 64, 8, 2
    c = decode_case(lens, hq, hkv, BF16, code, 5)
    nblk = 3
    mid_o = torch.full((nblk, 4, hq, D), math.nan, device=DEV); mid_l = torch.full((nblk, 4, hq), math.nan, device=DEV)
    fd.flash_decoding_stage1_q8(mid_o, mid_l, c["q"], c["codes"][:, :hkv], c["scales"][:, :hkv], c["codes"][:, hkv:], c["scales"][:, hkv:],
                                c["table"], c["rows"], c["lens"], max(lens), bs)
    for b, n in enumerate(lens):
        for j in range(nblk):
            m = min(bs, n - j * bs)
            if m <= 0:
                assert bool(mid_o[j, b].isnan().all()) and bool(mid_l[j, b].isnan().all())
                continue
            part = dict(c, table=c["table"][:, j * bs:], q=c["q"][b:b + 1], rows=c["rows"][b:b + 1])
            check_decode(mid_o[j, b:b + 1], mid_l[j, b:b + 1], decode_exact(part, [m]), m)


@pytest.mark.parametrize("code,hq,hkv,lens", [
    (INT8, 32, 32, [5000, 0, 1, 129, 700, 0, 2600]), (E4M3, 8, 1, [9000]), (INT8, 4, 4, [40] * 200 + [0, 0, 7] + [3000, 2999]),
    (E4M3, 16, 2, [0] * 5 + [129] + [0] * 5), (INT8, 24, 8, [128 * (i % 5) + i for i in range(384)]), (INT8, 8, 8, [33 * (i % 9) for i in range(385)]),
    (E4M3, 32, 4, [1] * 300 + [4096]), (INT8, 8, 2, [20000, 64, 20001]), (INT8, 449, 449, [600, 70]), (E4M3, 4, 4, [500] * 390)])
def test_decode_pieces_across_requests(code, hq, hkv, lens):
    """Divided evenly, a piece ends anywhere in a request and holds the ends of several."""
    from loongserve_b200 import flash_decoding as fd
    c = decode_case(lens, hq, hkv, BF16, code, seed=len(lens) + hq)
    out = torch.full((len(lens), hq, D), 9.0, device=DEV); lse = torch.full((len(lens), hq), 9.0, device=DEV)
    fd.token_decode_attention_q8(c["q"], c["codes"][:, :hkv], c["scales"][:, :hkv], c["codes"][:, hkv:], c["scales"][:, hkv:], c["table"], c["rows"],
                                 c["lens"], max(lens), None, out, lse)
    check_decode(out, lse, decode_exact(c), max(lens))
    assert fd.device_status()[0] == 0


def test_decode_pieces_follow_the_lengths_of_a_replay():
    """Captured once; lengths, rows and tokens are read when the graph runs.  Two graphs have a workspace each."""
    from loongserve_b200 import flash_decoding as fd
    hq, hkv = 8, 4
    c = decode_case([900, 31, 1500, 2], hq, hkv, BF16, INT8, 77)
    a = (c["codes"][:, :hkv], c["scales"][:, :hkv], c["codes"][:, hkv:], c["scales"][:, hkv:], c["table"], c["rows"], c["lens"], 1500)
    fd.token_decode_attention_q8(c["q"], *a)
    torch.cuda.synchronize()
    q2 = c["q"].flip(0).contiguous()
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    res = []
    for gr, q in zip(graphs, (c["q"], q2)):
        with torch.cuda.graph(gr):
            res.append(fd.token_decode_attention_q8(q, *a))
    for lens in ([900, 31, 1500, 2], [1, 0, 1499, 2], [0, 0, 0, 0], [128, 31, 129, 1]):
        c["lens"].copy_(torch.tensor(lens, dtype=torch.int32))
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        torch.cuda.synchronize()
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        for (o, lse), q in zip(res, (c["q"], q2)):
            check_decode(o, lse, decode_exact(dict(c, q=q)), 1500)


def test_decode_pieces_stop_at_the_given_longest():
    """No token behind max_len_in_batch is read; slots and rows outside are reported and left out, as with splits."""
    from loongserve_b200 import flash_decoding as fd
    fd.device_status()
    c = decode_case([600, 400, 500], 8, 2, BF16, E4M3, 13)
    r0 = int(c["rows"][0])
    a = (c["codes"][:, :2], c["scales"][:, :2], c["codes"][:, 2:], c["scales"][:, 2:], c["table"])
    out = torch.empty(3, 8, D, device=DEV); lse = torch.empty(3, 8, device=DEV)
    fd.token_decode_attention_q8(c["q"], *a, c["rows"], c["lens"], 450, None, out, lse)
    check_decode(out, lse, decode_exact(c, [450, 400, 450]), 450)
    assert fd.device_status()[0] == 0
    fd.token_decode_attention_q8(c["q"], *a, c["rows"], c["lens"], 100, None, out, lse)
    check_decode(out, lse, decode_exact(c, [100, 100, 100]), 100)
    buf = torch.zeros(3 * 8 * D + 1, dtype=BF16, device=DEV)
    with pytest.raises(RuntimeError):                                                          # rows are written 16 bytes at a time
        fd.token_decode_attention_q8(c["q"], *a, c["rows"], c["lens"], 100, None, buf[1:].view(3, 8, D), lse)
    with pytest.raises(AssertionError):
        fd.token_decode_attention_q8(c["q"], *a, c["rows"], c["lens"], 600, 0, out, lse)
    c["table"][r0, 5] = 2147483647; c["table"][r0, 400] = -3; c["table"][r0, 599] = c["codes"].shape[0]
    fd.token_decode_attention_q8(c["q"], *a, c["rows"], c["lens"], 600, None, out, lse)
    check_decode(out, lse, decode_exact(c), 600)
    st = fd.device_status()
    assert st[0] == -8 and st[2] == 0 and st[3] in (2147483647, -3, c["codes"].shape[0])
    rows = c["rows"].clone(); rows[1] = 99; rows[2] = -1
    lens = c["lens"].clone(); lens[0] = c["table"].shape[1] + 1                                # longer than the table is wide
    fd.token_decode_attention_q8(c["q"], *a, rows, lens, 600, None, out, lse)
    assert fd.device_status()[0] == -8
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())


def test_decode_scores_and_scales_of_every_size():
    """Scores that grow by hundreds from token to token, token scales from 1e-20 to 1e20, zero rows, a NaN row."""
    from loongserve_b200 import flash_decoding as fd
    for code in (INT8, E4M3):
        c = decode_case([513, 200, 90], 4, 2, BF16, code, 9, q_scale=40.0)
        g = torch.Generator().manual_seed(1)
        n = c["scales"].shape[0]
        c["scales"][:, 2:] *= torch.exp(20 * torch.randn(n, 2, generator=g)).to(DEV)       # V scales far apart
        k, v, ks, vs = c["codes"][:, :2], c["codes"][:, 2:], c["scales"][:, :2], c["scales"][:, 2:]
        out = torch.empty(3, 4, D, device=DEV); lse = torch.empty(3, 4, device=DEV)
        fd.token_decode_attention_q8(c["q"], k, ks, v, vs, c["table"], c["rows"], c["lens"], 513, 128, out, lse)
        check_decode(out, lse, decode_exact(c), 513)
        c["scales"][:, :2] = 0.0                                                              # all scores zero: the mean of the values
        c["scales"][:, 2:] = 0.5
        fd.token_decode_attention_q8(c["q"], k, ks, v, vs, c["table"], c["rows"], c["lens"], 513, 128, out, lse)
        check_decode(out, lse, decode_exact(c), 513)
        c["scales"][int(c["table"][int(c["rows"][1]), 77]), 0] = math.nan                     # one K row of request 1, kv head 0
        fd.token_decode_attention_q8(c["q"], k, ks, v, vs, c["table"], c["rows"], c["lens"], 513, 128, out, lse)
        assert bool(out[1, :2].isnan().all()) and not bool(out[1, 2:].isnan().any()) and not bool(out[[0, 2]].isnan().any())
        c["scales"][int(c["table"][int(c["rows"][1]), 77]), 0] = 0.0
        c["scales"][int(c["table"][int(c["rows"][2]), 3]), 3] = math.nan                      # one V row of request 2, kv head 1
        fd.token_decode_attention_q8(c["q"], k, ks, v, vs, c["table"], c["rows"], c["lens"], 513, 128, out, lse)
        assert bool(out[2, 2:].isnan().all()) and not bool(out[2, :2].isnan().any()) and not bool(out[:2].isnan().any())


def test_decode_query_range():
    """Queries at the ends of bf16's range next to ordinary ones: what is representable comes out, per head."""
    from loongserve_b200 import flash_decoding as fd
    c = decode_case([40, 33], 8, 2, BF16, INT8, 21)
    c["q"][0, 0] = 0.0
    c["q"][0, 1] *= 2.0 ** -60
    c["q"][0, 2] *= 2.0 ** 60
    c["scales"][:, 0] *= 2.0 ** -60                                                            # heads 0..3 read kv head 0
    c["q"][1, 4, 5] = 2.0 ** 9; c["q"][1, 4, 6] = 2.0 ** -30                                   # far apart within one query
    out = torch.empty(2, 8, D, device=DEV); lse = torch.empty(2, 8, device=DEV)
    fd.token_decode_attention_q8(c["q"], c["codes"][:, :2], c["scales"][:, :2], c["codes"][:, 2:], c["scales"][:, 2:], c["table"], c["rows"],
                                 c["lens"], 40, None, out, lse)
    check_decode(out, lse, decode_exact(c), 40)


def test_decode_bad_slots_rows_and_lengths():
    from loongserve_b200 import flash_decoding as fd
    fd.device_status()
    c = decode_case([100, 70, 50], 8, 2, BF16, E4M3, 13)
    r0 = int(c["rows"][0])
    c["table"][r0, 5] = 2147483647; c["table"][r0, 40] = -3; c["table"][r0, 99] = c["codes"].shape[0]
    a = (c["codes"][:, :2], c["scales"][:, :2], c["codes"][:, 2:], c["scales"][:, 2:], c["table"])
    out = torch.empty(3, 8, D, device=DEV); lse = torch.empty(3, 8, device=DEV)
    fd.token_decode_attention_q8(c["q"], *a, c["rows"], c["lens"], 100, 64, out, lse)
    check_decode(out, lse, decode_exact(c), 100)                                               # the three tokens are left out
    st = fd.device_status()
    assert st[0] == -8 and st[2] == 0 and st[3] in (2147483647, -3, c["codes"].shape[0])
    rows = c["rows"].clone(); rows[1] = 99; rows[2] = -1
    fd.token_decode_attention_q8(c["q"], *a, rows, c["lens"], 100, 64, out, lse)
    assert fd.device_status()[0] == -8
    assert bool((out[1:] == 0).all()) and bool((lse[1:] == -math.inf).all())                   # rows outside the table: nothing is read
    c["table"][r0, :100] = -1                                                                  # no token of the request is left
    fd.token_decode_attention_q8(c["q"], *a, c["rows"], c["lens"], 100, 64, out, lse)
    assert bool((out[0] == 0).all()) and bool((lse[0] == -math.inf).all()) and fd.device_status()[0] == -8
    assert fd.device_status()[0] == 0


def test_decode_offsets_beyond_32_bits():
    """A pool whose rows lie more than 2^31 bytes apart from its start."""
    from loongserve_b200 import flash_decoding as fd
    rows = 600000                                                                              # x 4224 B = 2.5 GB
    raw, codes, scales = pool(rows, 32, INT8, fill=0)
    g = torch.Generator().manual_seed(2)
    kv = torch.randn(50, 32, D, generator=g).to(BF16)
    from loongserve_b200 import kv_ops
    slots = (rows - 1 - 7 * torch.arange(50)).to(DEV)
    kv_ops.destindex_copy_quantize_kv(kv.to(DEV), slots, codes, scales)
    assert torch.equal(bits(codes[slots]), bits(quantise(kv, INT8)[0]))
    c = dict(q=torch.randn(1, 16, D, generator=g).to(BF16).to(DEV), codes=codes, scales=scales, table=slots.to(torch.int32)[None].contiguous(),
             rows=torch.zeros(1, dtype=torch.int32, device=DEV), lens=torch.tensor([50], dtype=torch.int32, device=DEV), hkv=16)
    o, lse = fd.token_decode_attention_q8(c["q"], codes[:, :16], scales[:, :16], codes[:, 16:], scales[:, 16:], c["table"], c["rows"], c["lens"], 50)
    check_decode(o, lse, decode_exact(c), 50)
    assert bool((kv_ops.gather_dequantize_kv(codes, scales, slots, BF16) != 0).any())


# ------------------------------------------------------------------------------------------------ row kernels
SHAPES = [(1, 8), (3, 24), (5, 128), (64, 4096), (33, 1144), (7, 8200), (2, 11008), (3, 16384), (2, 65536), (300, 512)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("tokens,hidden", SHAPES)
def test_add_rms_norm(dtype, tokens, hidden):
    from loongserve_b200 import layer_ops as ops
    g = torch.Generator().manual_seed(hidden)
    x = torch.randn(tokens, hidden, generator=g).to(dtype); r = (2 * torch.randn(tokens, hidden, generator=g)).to(dtype)
    w = (1 + 0.2 * torch.randn(hidden, generator=g)).to(dtype)
    t = x.double() + r.double()
    y = t / torch.sqrt(t.square().mean(-1, keepdim=True) + 1e-5) * w.double()
    # the sum of squares (all terms positive) is off by at most hidden/threads + 10 roundings, halved by the root; then rsqrt (2 ulp), two products
    rel = (hidden / 256 + 16) * U32
    rg = r.to(DEV)
    out = ops.add_rms_norm(x.to(DEV), rg, w.to(DEV), 1e-5)
    assert torch.equal(rg.cpu(), (x.float() + r.float()).to(dtype))
    tiny = 2.0 ** -25 if dtype is F16 else 0.0
    assert bool(((out.cpu().double() - y).abs() <= (half_step(dtype) + rel) * y.abs() + tiny).all())
    for residual in (True, False):
        rg = r.to(DEV) if residual else None
        src = x if residual else (x.float() + r.float()).to(dtype)
        yy = y
        if not residual:
            tt = src.double(); yy = tt / torch.sqrt(tt.square().mean(-1, keepdim=True) + 1e-5) * w.double()
        codes, scale = ops.add_rms_norm_quant(src.to(DEV), rg, w.to(DEV), 1e-5)
        if residual:
            assert torch.equal(rg.cpu(), (x.float() + r.float()).to(dtype))
        check_rows(codes, scale, yy, rel)


def check_rows(codes, scale, y, rel):
    """Codes stand for y (64 bits, known up to `rel` of its value) within half a step; the scale is max|y| / 127."""
    s = y.abs().amax(-1).clamp_min(TINY) / 127
    assert bool(((scale.cpu().double() - s).abs() <= (rel + 4 * U32) * s).all())
    v = codes.cpu().double() * scale.cpu().double()[:, None]
    assert bool(((v - y).abs() <= (0.5 + 127 * (2 * rel + 4 * U32)) * s[:, None] + rel * y.abs()).all())
    assert bool((codes.cpu().abs().amax(-1) == 127)[y.abs().amax(-1) > 1e-20].all())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("tokens,ffn", SHAPES)
def test_silu_and_mul_quant(dtype, tokens, ffn):
    from loongserve_b200 import layer_ops as ops
    g = torch.Generator().manual_seed(ffn + 1)
    io = (1.5 * torch.randn(tokens, 2 * ffn, generator=g)).to(dtype)
    gate, up = io.double().chunk(2, -1)
    iog = io.to(DEV)
    codes, scale = ops.silu_and_mul_quant(iog)
    assert torch.equal(iog.cpu(), io)
    # exp(-x), |x| <= 8 here: 2 + 1.173 * |x| ulp; a sum, a division (2 ulp) and a product
    check_rows(codes, scale, gate * torch.sigmoid(gate) * up, 24 * 2 * U32)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("tokens,cols", SHAPES)
def test_quantize_and_dequantize_rows(dtype, tokens, cols):
    from loongserve_b200 import layer_ops as ops
    g = torch.Generator().manual_seed(cols + 2)
    x = torch.randn(tokens, cols + 16, generator=g).to(dtype)
    if tokens > 2:
        x[0] = 0; x[1, 11 if cols > 8 else 8] = math.inf
    codes, scale = ops.quantize_rows(x.to(DEV)[:, 8:8 + cols])
    rc, rs = quantise(x[:, 8:8 + cols], INT8)
    assert torch.equal(codes.cpu(), rc) and torch.equal(scale.cpu().nan_to_num(-1), rs.nan_to_num(-1))
    for odt in (F16, BF16, torch.float32):
        back = ops.dequantize_rows(codes, scale, odt).cpu().double()
        want = rc.double() * rs.double()[:, None]
        ok = ((back - want).abs() <= (half_step(odt) + U32) * want.abs() + 2.0 ** -25 * (odt is F16)) | want.isnan() & back.isnan()
        assert bool(ok.all())


def test_row_kernels_at_the_ends_of_the_range():
    from loongserve_b200 import layer_ops as ops
    x = torch.ones(4, 256, dtype=BF16); x[1, 3] = math.nan; x[2, 5] = math.inf; x[3] = 0
    r = torch.zeros(4, 256, dtype=BF16)
    w = torch.ones(256, dtype=BF16)
    codes, scale = ops.add_rms_norm_quant(x.to(DEV), r.to(DEV), w.to(DEV), 1e-5)
    assert scale.isnan().tolist() == [False, True, True, False] and bool((codes[1:] == 0).all())
    io = torch.zeros(4, 512, dtype=F16)
    io[0, :256] = -60000.0; io[0, 256:] = 3.0                # silu goes to -0 without overflow
    io[1, :256] = 60000.0; io[1, 256:] = 60000.0             # the product is beyond fp16, not beyond fp32
    io[2, 7] = math.nan; io[2, 256:] = 1.0
    codes, scale = ops.silu_and_mul_quant(io.to(DEV))
    assert bool((codes[0] == 0).all()) and bool((codes[1] == 127).all()) and abs(float(scale[1]) * 127 / 3.6e9 - 1) < 1e-3
    assert scale.isnan().tolist() == [False, False, True, False]


# ------------------------------------------------------------------------------------------------ the integer product
MM = [(1, 1, 16), (1, 4096, 4096), (3, 129, 48), (16, 100, 208), (17, 257, 1040), (64, 4096, 11008), (65, 640, 128), (128, 128, 128),
      (129, 1000, 4112), (255, 300, 272), (256, 256, 256), (300, 517, 1552), (1000, 22, 64), (2049, 777, 400), (5000, 333, 512), (70, 5000, 144)]


@pytest.mark.parametrize("m,n,k", MM)
@pytest.mark.parametrize("odt", [F16, BF16, torch.float32])
def test_mm_w8a8(m, n, k, odt):
    from loongserve_b200 import layer_ops as ops
    g = torch.Generator(device=DEV).manual_seed(m * 3 + n + k)
    a = torch.randint(-128, 128, (m, k), generator=g, device=DEV, dtype=torch.int8)
    w = torch.randint(-128, 128, (n, k), generator=g, device=DEV, dtype=torch.int8)
    sa = torch.rand(m, generator=g, device=DEV) * 0.01 + 1e-4; sw = torch.rand(n, generator=g, device=DEV) * 0.01 + 1e-4
    want = (a.double() @ w.double().t()) * sa.double()[:, None] * sw.double()[None]
    got = ops.mm_w8a8(a, sa, w, sw, out_dtype=odt)
    fit = want.abs() < torch.finfo(odt).max
    tol = (half_step(odt) + 3 * U32) * want.abs() + (2.0 ** -25 if odt is F16 else 0.0)        # sum to fp32, two products, the output
    assert bool(((got.double() - want).abs() <= tol)[fit].all()), (got.double() - want).abs().max()


def test_mm_w8a8_strides_rows_behind_and_extremes():
    from loongserve_b200 import layer_ops as ops
    g = torch.Generator(device=DEV).manual_seed(4)
    for m, n, k in ((5, 70, 96), (200, 300, 512), (600, 513, 4096)):
        abig = torch.randint(-128, 128, (m + 1, k + 48), generator=g, device=DEV, dtype=torch.int8)
        wbig = torch.randint(-128, 128, (n + 1, k + 16), generator=g, device=DEV, dtype=torch.int8)
        a, w = abig[1:, 16:16 + k], wbig[1:, 16:16 + k]
        sa = torch.rand(m, generator=g, device=DEV); sw = torch.rand(n, generator=g, device=DEV)
        want = (a.double() @ w.double().t()) * sa.double()[:, None] * sw.double()[None]
        for off in (0, 1, 3):
            out = torch.full((m + 2, n + 7), 3.0, dtype=BF16, device=DEV)
            ops.mm_w8a8(a, sa, w, sw, out=out[1:m + 1, off:off + n])
            assert bool(((out[1:m + 1, off:off + n].double() - want).abs() <= (half_step(BF16) + 3 * U32) * want.abs()).all())
            assert bool((out[0] == 3).all()) and bool((out[m + 1] == 3).all()) and bool((out[:, off + n:] == 3).all()) and bool((out[:, :off] == 3).all())
    # the largest sum: every product is 128 * 128 over the largest K
    k = 131056
    a = torch.full((2, k), -128, dtype=torch.int8, device=DEV)
    got = ops.mm_w8a8(a, torch.ones(2, device=DEV), torch.cat([a, -a - 1]), torch.ones(4, device=DEV), out_dtype=torch.float32)
    assert got.tolist() == [[16384.0 * k] * 2 + [float(torch.tensor(-128 * 127 * k, dtype=torch.int64).float())] * 2] * 2
    # a scale of NaN (a row that had no scale) reaches its row or its column and no other
    a = torch.randint(-5, 6, (20, 64), device=DEV, dtype=torch.int8); w = torch.randint(-5, 6, (40, 64), device=DEV, dtype=torch.int8)
    sa, sw = torch.ones(20, device=DEV), torch.ones(40, device=DEV)
    sa[3] = math.nan; sw[39] = math.nan
    got = ops.mm_w8a8(a, sa, w, sw).isnan()
    want = torch.zeros(20, 40, dtype=torch.bool, device=DEV); want[3] = True; want[:, 39] = True
    assert torch.equal(got, want)


# ------------------------------------------------------------------------------------------------ together
def test_a_layer_in_8_bits_captured_and_on_another_stream():
    """norm -> qkv product -> cache write -> attention over the cache -> product -> add + norm -> gate/up -> SiLU -> down, eager on
    the default stream, eager on another stream, and as a replayed graph: the same bits each time, and near 64 bits."""
    from loongserve_b200 import flash_decoding as fd, kv_ops, layer_ops as ops
    g = torch.Generator().manual_seed(8)
    B, H, hq, hkv, F, L = 5, 512, 4, 2, 768, 100
    rnd = lambda *s, k=1.0: (k * torch.randn(*s, generator=g)).to(BF16).to(DEV)
    w = {n: ops.quantize_rows(rnd(*s, k=0.05)) for n, s in dict(q=(hq * D, H), kv=(2 * hkv * D, H), o=(H, hq * D), gu=(2 * F, H), dn=(H, F)).items()}
    n1, n2 = (1 + 0.1 * torch.randn(H, generator=g)).to(BF16).to(DEV), (1 + 0.1 * torch.randn(H, generator=g)).to(BF16).to(DEV)
    x0, d0 = rnd(B, H), rnd(B, H)
    raw, codes, scales = pool(B * L + 9, 2 * hkv, INT8, fill=0)
    old = rnd(B * (L - 1), 2 * hkv, D)
    slots = torch.randperm(B * L + 9, generator=g)[:B * L].to(DEV)
    kv_ops.destindex_copy_quantize_kv(old, slots[:B * (L - 1)].contiguous(), codes, scales)
    table = torch.cat([slots[:B * (L - 1)].view(B, L - 1), slots[B * (L - 1):].view(B, 1)], 1).to(torch.int32).contiguous()
    rows, lens, new = torch.arange(B, dtype=torch.int32, device=DEV), torch.full((B,), L, dtype=torch.int32, device=DEV), slots[B * (L - 1):].contiguous()

    def layer(x, delta):
        h, hs = ops.add_rms_norm_quant(delta, x, n1, 1e-5)
        q = ops.mm_w8a8(h, hs, *w["q"]).view(B, hq, D)
        kv_ops.destindex_copy_quantize_kv(ops.mm_w8a8(h, hs, *w["kv"]).view(B, 2 * hkv, D), new, codes, scales)
        o, lse = fd.token_decode_attention_q8(q, codes[:, :hkv], scales[:, :hkv], codes[:, hkv:], scales[:, hkv:], table, rows, lens, L)
        h, hs = ops.add_rms_norm_quant(ops.mm_w8a8(*ops.quantize_rows(o.view(B, hq * D)), *w["o"]), x, n2, 1e-5)
        return q, o, lse, ops.mm_w8a8(*ops.silu_and_mul_quant(ops.mm_w8a8(h, hs, *w["gu"])), *w["dn"])

    x = x0.clone()
    first = [t.clone() for t in layer(x, d0)] + [x.clone()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x = x0.clone()
        second = list(layer(x, d0)) + [x]
    side.synchronize()
    xs, ds = x0.clone(), d0.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = layer(xs, ds)
    for _ in range(3):
        xs.copy_(x0)
        graph.replay()
    torch.cuda.synchronize()
    for a, b, c in zip(first, second, list(held) + [xs]):
        assert torch.equal(a, b) and torch.equal(a, c)
    # the same layer in 64 bits from the 8-bit weights, activations not quantised: apart by what 8-bit rows lose (a step of 1/127 of
    # a row's maximum of about 4 sigma is 0.03 sigma, 0.009 sigma rms; five of them in a row and 16-bit outputs)
    deq = {n: c.double() * s.double()[:, None] for n, (c, s) in w.items()}
    norm = lambda t, nw: t / torch.sqrt(t.square().mean(-1, keepdim=True) + 1e-5) * nw.double()
    t = x0.double() + d0.double()
    h = norm(t, n1)
    case = dict(q=(h @ deq["q"].t()).view(B, hq, D), codes=codes, scales=scales, table=table, rows=rows, lens=lens, hkv=hkv)
    ro = decode_exact(case)[0].to(DEV)
    t = t + ro.view(B, -1) @ deq["o"].t()
    gate, up = (norm(t, n2) @ deq["gu"].t()).chunk(2, -1)
    y = (gate * torch.sigmoid(gate) * up) @ deq["dn"].t()
    assert (first[3].double() - y).norm() / y.norm() < 0.05 and (first[4].double() - t).norm() / t.norm() < 0.02


def test_empty_batches_do_nothing():
    from loongserve_b200 import flash_decoding as fd, kv_ops, layer_ops as ops
    raw, codes, scales = pool(4, 2, INT8)
    before = raw.clone()
    none = torch.empty(0, dtype=torch.int64, device=DEV)
    kv_ops.destindex_copy_quantize_kv(torch.empty(0, 2, D, dtype=BF16, device=DEV), none, codes, scales)
    assert torch.equal(raw, before) and kv_ops.gather_dequantize_kv(codes, scales, none, F16).shape == (0, 2, D)
    e = torch.empty(0, 64, dtype=BF16, device=DEV)
    w = torch.ones(64, dtype=BF16, device=DEV)
    assert ops.add_rms_norm(e, e.clone(), w, 1e-5).shape == (0, 64) and ops.add_rms_norm_quant(e, None, w, 1e-5)[0].shape == (0, 64)
    c, s = ops.silu_and_mul_quant(e)
    assert c.shape == (0, 32) and ops.dequantize_rows(c, s).shape == (0, 32)
    wq, ws = ops.quantize_rows(torch.ones(16, 32, dtype=BF16, device=DEV))
    assert ops.mm_w8a8(c, s, wq, ws).shape == (0, 16)
    o, lse = fd.token_decode_attention_q8(torch.empty(0, 4, D, dtype=BF16, device=DEV), codes[:, :1], scales[:, :1], codes[:, 1:], scales[:, 1:],
                                          torch.zeros(2, 8, dtype=torch.int32, device=DEV), none.int(), none.int(), 0)
    assert o.shape == (0, 4, D)
    o, lse = fd.token_decode_attention_q8(torch.ones(2, 4, D, dtype=BF16, device=DEV), codes[:, :1], scales[:, :1], codes[:, 1:], scales[:, 1:],
                                          torch.zeros(2, 8, dtype=torch.int32, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV),
                                          torch.zeros(2, dtype=torch.int32, device=DEV), 0)
    assert bool((o == 0).all()) and bool((lse == -math.inf).all())


@pytest.mark.parametrize("tokens", [1, 16, 64])
def test_row_kernels_and_products_in_a_chain(tokens):
    """A layer's norm, product, SiLU and product, three layers in one graph over shared buffers: every product waits for its rows, and
    every row kernel for the product before it."""
    from loongserve_b200 import layer_ops as ops
    H, Fn = 1024, 2816
    g = torch.Generator().manual_seed(tokens)
    w1 = ops.quantize_rows((torch.randn(2 * Fn, H, generator=g) * H ** -0.5).to(BF16).to(DEV))
    w2 = ops.quantize_rows((torch.randn(H, Fn, generator=g) * Fn ** -0.5).to(BF16).to(DEV))
    nw = torch.rand(H, generator=g).to(BF16).to(DEV)
    x = torch.empty(tokens, H, dtype=BF16, device=DEV); res = torch.empty_like(x)
    codes, scale = torch.empty(tokens, H, dtype=INT8, device=DEV), torch.empty(tokens, device=DEV)
    gu = torch.empty(tokens, 2 * Fn, dtype=BF16, device=DEV)
    codes2, scale2 = torch.empty(tokens, Fn, dtype=INT8, device=DEV), torch.empty(tokens, device=DEV)

    def layers(sync):
        for _ in range(3):
            for f in (lambda: ops.add_rms_norm_quant(x, res, nw, 1e-5, codes, scale), lambda: ops.mm_w8a8(codes, scale, *w1, out=gu),
                      lambda: ops.silu_and_mul_quant(gu, codes2, scale2), lambda: ops.mm_w8a8(codes2, scale2, *w2, out=x)):
                f()
                if sync:
                    torch.cuda.synchronize()

    x.normal_(); res.normal_()
    layers(True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layers(False)
    for seed in range(4):
        g.manual_seed(seed)
        a, b = torch.randn(tokens, H, generator=g).to(BF16).to(DEV), torch.randn(tokens, H, generator=g).to(BF16).to(DEV)
        x.copy_(a); res.copy_(b)
        layers(True)
        want = x.clone(), res.clone(), codes2.clone(), scale2.clone()
        for run in (graph.replay, lambda: layers(False)):
            x.copy_(a); res.copy_(b)
            run()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(want, (x, res, codes2, scale2)))


@pytest.mark.parametrize("code", [INT8, E4M3])
@pytest.mark.parametrize("lens", [[40, 9], [3000, 1200, 1, 700]])
def test_pool_writes_and_decode_in_a_chain(code, lens):
    """A step's rows are written, attended to with a query that the step before made, three times in one graph: each kernel waits for the
    one ahead of it, and calls that take turns on one workspace do not meet."""
    from loongserve_b200 import flash_decoding as fd, kv_ops
    hq, hkv = 8, 4
    B = len(lens)
    c = decode_case(lens, hq, hkv, BF16, code, 31)
    a = (c["codes"][:, :hkv], c["scales"][:, :hkv], c["codes"][:, hkv:], c["scales"][:, hkv:], c["table"], c["rows"], c["lens"], max(lens))
    last = torch.stack([c["table"][int(c["rows"][b]), n - 1] for b, n in enumerate(lens)]).to(torch.int64)
    kv = torch.empty(B, 2 * hkv, D, dtype=BF16, device=DEV); q = torch.empty(B, hq, D, dtype=BF16, device=DEV)
    lse = torch.empty(B, hq, device=DEV)

    def steps(sync):
        for _ in range(3):
            for f in (lambda: kv_ops.destindex_copy_quantize_kv(kv, last, c["codes"], c["scales"]),
                      lambda: fd.token_decode_attention_q8(q, *a, out=q, out_logexpsum=lse), lambda: kv.copy_(q[:, :2 * hkv])):
                f()
                if sync:
                    torch.cuda.synchronize()

    kv.normal_(); q.normal_()
    steps(True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        steps(False)
    g = torch.Generator()
    for seed in range(4):
        g.manual_seed(seed)
        x, y = torch.randn(B, 2 * hkv, D, generator=g).to(BF16).to(DEV), torch.randn(B, hq, D, generator=g).to(BF16).to(DEV)
        kv.copy_(x); q.copy_(y)
        steps(True)
        want = q.clone(), lse.clone(), kv.clone()
        for run in (graph.replay, lambda: steps(False)):
            kv.copy_(x); q.copy_(y)
            run()
            torch.cuda.synchronize()
            assert all(torch.equal(m, n) for m, n in zip(want, (q, lse, kv)))
