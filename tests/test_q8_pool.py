"""Host side of the pool in 8 bits: the row layout, its views, slicing, resizing, and what is refused (no GPU needed)."""
import pytest
import torch

from loongserve_b200.mem_manager import LongServeMemoryManager, QuantizedKVMemoryManager, QuantizedPoolLayer


@pytest.fixture(scope="module", autouse=True)
def built():
    from loongserve_b200 import build
    build.build_attention(force=False)


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("heads,dim,row", [(32, 128, 8448), (8, 128, 2112), (1, 128, 272), (3, 128, 800), (5, 80, 848), (1, 16, 48)])
def test_a_row_keeps_codes_and_scales(dtype, heads, dim, row):
    m = QuantizedKVMemoryManager(10, dtype, heads, dim, 2, num_idle_slots=3, device="cpu")
    assert m.row_bytes == row and m.kv_buffer.shape == (2, 13, row) and m.kv_buffer.dtype == torch.uint8
    m.kv_buffer.zero_()
    lay = m.layer(1)
    assert lay.shape == (13, 2 * heads, dim) and lay.codes.dtype == dtype and lay.scales.shape == (13, 2 * heads) and lay.scales.dtype == torch.float32
    assert lay.codes.data_ptr() % 16 == 0 and lay.codes.stride(0) % 16 == 0 and lay.codes.stride(2) == 1 and lay.scales.stride(1) == 1
    lay.codes.view(torch.uint8).fill_(255)
    lay.scales.view(torch.int32).fill_(-1)
    used = 2 * heads * (dim + 4)
    assert bool((m.kv_buffer[1, :, :used] == 255).all()) and bool((m.kv_buffer[1, :, used:] == 0).all()) and bool((m.kv_buffer[0] == 0).all())
    v = lay[:, heads:, :]
    assert isinstance(v, QuantizedPoolLayer) and torch.equal(v.codes.view(torch.uint8), lay.codes.view(torch.uint8)[:, heads:]) and v.scales.shape == (13, heads)
    assert m.layer(1) is lay and m.migration_view.shape == (2, 13, 1, row)


def test_slots_and_resizing_as_in_the_16_bit_pool():
    a, b = LongServeMemoryManager(20, torch.float16, 2, 128, 1, device="cpu"), QuantizedKVMemoryManager(20, torch.int8, 2, 128, 1, device="cpu")
    assert torch.equal(a.alloc(5), b.alloc(5)) and a.alloc_contiguous(4)[1:] == b.alloc_contiguous(4)[1:]
    assert a.can_use_mem_size == b.can_use_mem_size == 11
    old = b.layer(0)
    b.resize_mem(40)
    assert b.can_use_mem_size == 40 and b.layer(0).shape[0] == 40 and b.layer(0) is not old
    assert a.layer(0).data_ptr() == a.kv_buffer[0].data_ptr() and a.migration_view is a.kv_buffer


def test_refusals():
    for bad in (torch.uint8, torch.float16, torch.float8_e5m2):
        with pytest.raises(TypeError):
            QuantizedKVMemoryManager(4, bad, 1, 128, 1, device="cpu")
    with pytest.raises(ValueError):
        QuantizedKVMemoryManager(4, torch.int8, 1, 72, 1, device="cpu")
    lay = QuantizedKVMemoryManager(4, torch.int8, 1, 128, 1, device="cpu").layer(0)
    for index in ((slice(0, 2), slice(None), slice(None)), (slice(None), 1, slice(None)), (slice(None), slice(None), slice(0, 8))):
        with pytest.raises(AssertionError):
            lay[index]
    from loongserve_b200.llama_stack import LlamaConfig, LlamaW8A8Weights
    with pytest.raises(ValueError):
        LlamaW8A8Weights(LlamaConfig(hidden=4096, ffn=1000), None)


def test_the_keep_step_and_stage_1_reach_the_8_bit_kernels(monkeypatch):
    """The runtime's adapters hand a layer's codes and scales on in the argument order of the ring."""
    from loongserve_b200 import attention_runtime as ar
    seen = {}
    monkeypatch.setattr(ar.kv_ops, "destindex_copy_quantize_and_register_kv", lambda *a: seen.setdefault("keep", a))
    monkeypatch.setattr(ar.fd, "flash_decoding_stage1_q8", lambda *a: seen.setdefault("stage1", a))
    lay = QuantizedKVMemoryManager(4, torch.int8, 2, 128, 1, device="cpu").layer(0)
    ar._keep_quantized(1, 2, 3, 4, 5, 6, 7, 8, 9, lay, 10, 11, 12, 13, True)
    assert seen["keep"] == (1, 2, 3, 4, 5, 6, 7, 8, 9, lay.codes, lay.scales, 10, 11, 12, 13, True)
    k, v = lay[:, :2, :], lay[:, 2:, :]
    ar._stage1_quantized(1, 2, 3, k, v, 4, 5, 6, 7, 8)
    assert seen["stage1"][:3] == (1, 2, 3) and seen["stage1"][3] is k.codes and seen["stage1"][6] is v.scales and seen["stage1"][7:] == (4, 5, 6, 7, 8)
