"""What the 8-bit product and decode kernels do once a bounded wait has run out, on their own code with waits that can be made short
(tests/csrc/short_waits.cu): they return, the status names the wait, what they write is right or not written at all, a later call
writes nothing until the status has been read, and after that everything works.  Nothing hangs or faults: every wait is bounded, and
the kernels wait for their own copies and products before they leave."""
import ctypes as C

import pytest
import torch

from test_gpu_q8 import BF16, DEV, E4M3, INT8, decode_case

pytestmark = pytest.mark.gpu
FULL = 2_000_000_000
TIMEOUT = -4


@pytest.fixture(scope="module")
def lib():
    from loongserve_b200 import _lib, build
    short = C.CDLL(build.build_short_waits())
    for name in ("esp_mm_w8a8", "esp_decode_attention_q8", "esp_decode_stage1_q8"):
        getattr(short, name).argtypes = _lib.ATTN_SIGNATURES[name]
        getattr(short, name).restype = C.c_int32
    short.esp_short_limit.argtypes = [C.c_int64]
    yield short
    short.esp_short_limit(FULL)


def status(lib):
    buf = (C.c_int32 * 8)()
    assert lib.esp_short_status(buf) == 0
    return tuple(buf[:4]), tuple(buf[4:])


def run_out(lib, call, results, want, which, sure=True):
    """call() with limits from one cycle to some twenty thousand; results: what it writes, want: what it should.  A wait of one cycle runs
    out at its second poll; sure: with many waits in the call, some of them for copies that have just been started, one does."""
    status(lib)
    ran_out = 0
    for limit in (1, 300, 1000, 2000, 4000, 8000, 20000, 1):
        for r in results:
            r.fill_(7.0)
        assert lib.esp_short_limit(limit) == 0
        call()
        torch.cuda.synchronize()
        for r, w in zip(results, want):
            assert bool(((r == 7.0) | (r == w)).all())                # what is written is right
        again = [r.clone() for r in results]
        call()                                                         # once the status is set nothing is started
        st = status(lib)
        if st[which][0]:
            assert st[which][0] == TIMEOUT
            ran_out += 1
        else:
            assert all(torch.equal(r, w) for r, w in zip(results, want))
        if limit == 1 and st[which][0]:
            assert all(torch.equal(r, a) for r, a in zip(results, again))
        assert lib.esp_short_limit(FULL) == 0
        call()
        torch.cuda.synchronize()
        assert all(torch.equal(r, w) for r, w in zip(results, want)) and status(lib)[which][0] == 0
    assert ran_out >= 2 or not sure


# few tokens: 1, 2 and 8 splits of K, tiles of 16 to 128 tokens; pairs over 256 and 128 channels, one tile each and several
@pytest.mark.parametrize("m,n,k", [(1, 100, 112), (16, 4096, 4096), (33, 300, 11008), (64, 4096, 11008), (200, 600, 8000), (512, 4096, 1280),
                                   (300, 22016, 4096), (5000, 333, 512), (2049, 5000, 400)])
def test_products(lib, m, n, k):
    from loongserve_b200 import layer_ops as ops
    g = torch.Generator(device=DEV).manual_seed(m + n)
    a = torch.randint(-128, 128, (m, k), generator=g, device=DEV, dtype=torch.int8)
    w = torch.randint(-128, 128, (n, k), generator=g, device=DEV, dtype=torch.int8)
    sa, sw = torch.rand(m, generator=g, device=DEV) + 0.1, torch.rand(n, generator=g, device=DEV) + 0.1
    want = ops.mm_w8a8(a, sa, w, sw, out_dtype=torch.float32)
    out = torch.empty_like(want)
    s = torch.cuda.current_stream().cuda_stream

    def call():
        assert lib.esp_mm_w8a8(out.data_ptr(), n, a.data_ptr(), k, sa.data_ptr(), w.data_ptr(), k, sw.data_ptr(), m, n, k, 2, s) == 0
    run_out(lib, call, [out], [want], 0, sure=m > 1)


@pytest.mark.parametrize("code", [INT8, E4M3])
@pytest.mark.parametrize("lens,hq,hkv", [([300], 8, 2), ([5000, 0, 1, 700], 8, 2), ([40] * 100 + [3000], 16, 16), ([200] * 40, 20, 2)])
def test_decode(lib, code, lens, hq, hkv):
    from loongserve_b200 import _lib, flash_decoding as fd
    c = decode_case(lens, hq, hkv, BF16, code, 3)
    a = (c["codes"][:, :hkv], c["scales"][:, :hkv], c["codes"][:, hkv:], c["scales"][:, hkv:], c["table"], c["rows"], c["lens"], max(lens))
    out, lse = torch.empty(len(lens), hq, 128, dtype=torch.float32, device=DEV), torch.empty(len(lens), hq, device=DEV)
    want = [t.clone() for t in fd.token_decode_attention_q8(c["q"], *a, None, out, lse)]
    real = _lib.attn
    try:
        _lib.attn = lambda: lib
        run_out(lib, lambda: fd.token_decode_attention_q8(c["q"], *a, None, out, lse), [out, lse], want, 1)
    finally:
        _lib.attn = real
