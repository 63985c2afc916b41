"""Refusals of the 8-bit cache's entry points, and its cache engine, without a GPU."""
import ctypes

import pytest
import torch

from apt_serve_b200 import _native as N
from apt_serve_b200 import attention as A
from apt_serve_b200 import ops
from apt_serve_b200.cache_engine import CacheEngine
from apt_serve_b200.layers import OPTAttention

E4M3 = torch.float8_e4m3fn


def address(offset=0):
    address.buf = getattr(address, "buf", None) or (ctypes.c_char * 8192)()
    return (ctypes.addressof(address.buf) + 255) // 256 * 256 + offset


def write(**kw):
    p = address()
    a = dict(key=p, value=p, kc=p, vc=p, ks=p, vs=p, slots=p, t=2, h=2, d=64, bs=16, nb=4, s_k=128, s_v=128, block=2048, s_s=2, ws=p, ws_bytes=1 << 40, dtype=1)
    a.update(kw)
    return N.lib().aps_kv8_write(*a.values(), 0)


def attend(**kw):
    p = address()
    a = dict(out=p, q=p, kc=p, vc=p, ks=p, vs=p, bt=p, starts=p, sl=p, b=2, t=5, most=3, width=4, h=2, d=64, bs=16, nb=4, s_q=128, s_o=128,
             block=2048, s_s=2, scale=1.0, ws=p, ws_bytes=1 << 40, dtype=1)
    a.update(kw)
    return N.lib().aps_kv8_attention(*a.values(), 0)


@pytest.mark.parametrize("status,kw", [
    (N.APS_ERR_DTYPE, dict(dtype=3)), (N.APS_ERR_UNSUPPORTED, dict(d=96)), (N.APS_ERR_UNSUPPORTED, dict(bs=8)),
    (N.APS_ERR_UNSUPPORTED, dict(bs=1040, block=1040 * 128)), (N.APS_ERR_SHAPE, dict(h=0)), (N.APS_ERR_SHAPE, dict(t=-1)),
    (N.APS_ERR_SHAPE, dict(s_k=64)), (N.APS_ERR_SHAPE, dict(block=1024)), (N.APS_ERR_SHAPE, dict(s_s=1)), (N.APS_ERR_SHAPE, dict(nb=1 << 28)),
    (N.APS_ERR_NULL_POINTER, dict(ks=0)), (N.APS_ERR_NULL_POINTER, dict(slots=0)), (N.APS_ERR_MISALIGNED, dict(kc=address(2))),
    (N.APS_ERR_MISALIGNED, dict(block=2050)), (N.APS_ERR_MISALIGNED, dict(key=address(1))), (N.APS_OK, dict(t=0, key=0)),
    (N.APS_ERR_WORKSPACE, dict(t=1025, ws=0)), (N.APS_ERR_WORKSPACE, dict(t=1025, ws_bytes=1025 * 4)),
])
def test_write_refuses(status, kw):
    assert write(**kw) == status


@pytest.mark.parametrize("status,kw", [
    (N.APS_ERR_DTYPE, dict(dtype=3)), (N.APS_ERR_UNSUPPORTED, dict(d=80)), (N.APS_ERR_UNSUPPORTED, dict(bs=20, block=4000)),
    (N.APS_ERR_SHAPE, dict(width=0)), (N.APS_ERR_SHAPE, dict(b=-1)), (N.APS_ERR_SHAPE, dict(s_q=127)), (N.APS_ERR_SHAPE, dict(starts=0)),
    (N.APS_ERR_SHAPE, dict(width=1 << 28)), (N.APS_ERR_NULL_POINTER, dict(bt=0)), (N.APS_ERR_NULL_POINTER, dict(out=0)),
    (N.APS_ERR_MISALIGNED, dict(vc=address(8))), (N.APS_ERR_MISALIGNED, dict(block=2056)), (N.APS_ERR_WORKSPACE, dict(width=4000, ws_bytes=64)),
    (N.APS_ERR_WORKSPACE, dict(width=4000, ws=0)), (N.APS_OK, dict(t=0, q=0)), (N.APS_OK, dict(b=0, bt=0)),
])
def test_attention_refuses(status, kw):
    assert attend(**kw) == status


def test_python_refusals():
    kc, s = torch.zeros(4, 16, 2, 64, dtype=E4M3), torch.zeros(4, 2)
    x, slots = torch.zeros(3, 2, 64, dtype=torch.float16), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="k_scale and v_scale"):
        ops.reshape_and_cache_flash(x, x, kc, kc, slots, "fp8")
    with pytest.raises(ValueError, match="float8_e4m3fn or uint8"):
        ops.reshape_and_cache_flash(x, x, kc.half(), kc.half(), slots, "fp8", s, s)
    with pytest.raises(ValueError, match="not supported"):
        ops.reshape_and_cache_flash(x, x, kc, kc, slots, "fp8_e5m2", s, s)
    for bad in (s[:3], s.double(), torch.zeros(2, 4).t()):
        with pytest.raises(RuntimeError, match="scale must be float32"):
            ops.reshape_and_cache_flash(x, x, kc, kc, slots, "fp8", bad, bad)
    with pytest.raises(RuntimeError, match="contiguous"):
        ops.reshape_and_cache_flash(x, x, kc[..., :32], kc[..., :32], slots, "fp8", s, s)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ops.reshape_and_cache_flash(x, x, kc, kc, slots, "fp8", s, s)
    q, bt, sl = torch.zeros(3, 128), torch.zeros(3, 2, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="k_scale and v_scale"):
        A.paged_decode_attention(q, kc, kc, bt, sl, 1.0)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        A.paged_prefix_attention(q, kc, kc, bt, sl, sl, 1, 1.0, s, s)


def test_hidden_cached_requests_are_refused():
    class Config:
        cache_dtype, sliding_window = "fp8", None
    layer = OPTAttention(128, 2, torch.zeros(384, 128), None, torch.zeros(128, 128), None, cache_config=Config)

    class Meta:
        num_hidden_cache_tokens, num_decode_tokens, num_prefill_tokens = 3, 2, 0
    with pytest.raises(ValueError, match="hidden-cached"):
        layer(torch.zeros(2, 128), None, None, Meta)
    x = torch.zeros(2, 128)
    with pytest.raises(ValueError, match="hidden-cached"):
        layer.attn.impl.forward(x, x, x, None, None, Meta)


def test_decode_tokens_without_a_cache_are_refused():
    class Meta:
        num_hidden_cache_tokens, num_decode_tokens, num_prefill_tokens, num_prefills = 0, 2, 0, 0
        block_tables = seq_lens_tensor = slot_mapping = None
    x = torch.zeros(2, 128)
    with pytest.raises(ValueError, match="need a kv_cache"):
        A.FlashAttentionImpl(2, 64, 1.0, 2, None, None, "fp8").forward(x, x, x, None, None, Meta)


def test_cache_engine_moves_the_scales_with_the_blocks():
    engine = CacheEngine(2, 4, 64, 16, 8, 4, E4M3, device="cpu", pin_memory=False, hidden_size=512)
    assert engine.gpu_hidden_cache is None and engine.gpu_cache[0].dtype == E4M3 and engine.gpu_scale[1].shape == (2, 8, 4)
    engine.gpu_scale[1][:, 3], engine.gpu_cache[1][:, 3] = 2.0, 3.0
    engine.swap_out(torch.tensor([[3, 1]]))
    assert (engine.cpu_scale[1][:, 1] == 2).all() and (engine.cpu_cache[1][:, 1].float() == 3).all()
    engine.swap_in(torch.tensor([[1, 6]]))
    assert (engine.gpu_scale[1][:, 6] == 2).all() and (engine.gpu_cache[1][:, 6].float() == 3).all()
    assert CacheEngine.get_cache_block_size(2, 4, 64, 16, E4M3, 512) == 2 * (2 * 16 * 4 * 64 + 2 * 4 * 4)
    assert CacheEngine.num_blocks_for_budget(10 * 16448, 2, 4, 64, 16, E4M3) == 10
    with pytest.raises(ValueError, match="shared cache"):
        CacheEngine(1, 4, 64, 16, 8, 4, E4M3, device="cpu", with_shared_cache=True, pin_memory=False)


def test_scratch_is_that_of_the_kernel_that_runs():
    """Parts of rows are held where the tokens are cut, which long chunks' are not: no row of theirs needs a place for each part that a
    few rows would be cut into."""
    def size(batch, rows, most, blocks, heads, d, dtype=torch.float16):
        return N.lib().aps_kv8_attention_workspace_bytes(batch, rows, most, blocks, 16, heads, d, N.DTYPE_ENUM[dtype])
    for dtype in (torch.float16, torch.bfloat16, torch.float32):
        assert size(1, 2048, 2048, 1001, 32, 64, dtype) == size(1, 8192, 8192, 2048, 40, 128, dtype) == 256   # the header alone
        for batch in (1, 2, 7, 60, 300):
            for most in (17, 100, 129, 600, 5000):
                # twice as many CTAs as SMs at most, 128 rows and heads' parts each
                assert size(batch, batch * most, most, 2048, 12, 128, dtype) <= 256 * 2 + 2 * 148 * 128 * 130 * 4
    # a few rows' parts: what the streaming kernel takes, for drafted tokens and for one row of each request
    assert size(64, 320, 5, 128, 40, 128) == size(64, 320, 16, 128, 40, 128) > size(64, 320, 17, 128, 40, 128)
    assert size(256, 256, 1, 128, 40, 128) == size(256, 256, 300, 128, 40, 128) < 32 << 20   # 300: without starts a row for each
    assert size(256, 256, 1, 128, 12, 64, torch.float32) <= size(256, 256, 1, 128, 12, 64)
    assert size(0, 5, 1, 4, 2, 64) == size(2, 0, 1, 4, 2, 64) == size(2, 5, -1, 4, 2, 64) == 0


def test_scratch_sizes_are_kept_for_each_device(monkeypatch):
    """They follow the current device's number of SMs."""
    class Lib:
        sms = 148

        def aps_kv8_attention_workspace_bytes(self, *sizes):
            return self.sms * 1000
    lib = Lib()
    monkeypatch.setattr(N, "lib", lambda: lib)
    sizes = (3, 3, 1, 4001, 16, 3, 64, 1)
    first = A._fp8_scratch_bytes(0, *sizes)
    lib.sms = 160
    assert A._fp8_scratch_bytes(1, *sizes) == 160000 and A._fp8_scratch_bytes(0, *sizes) == first == 148000
    A._fp8_scratch_bytes.cache_clear()


def test_a_16_bit_cache_takes_the_number_one_as_a_scale():
    """As a tensor, too; not the scales of an 8-bit cache."""
    class Meta:
        num_hidden_cache_tokens = num_decode_tokens = num_prefill_tokens = num_prefills = num_tot_tokens = 0
        block_tables = seq_lens_tensor = prefill_metadata = decode_metadata = None
        slot_mapping = torch.zeros(0, dtype=torch.int64)
    x, impl = torch.zeros(0, 128), A.FlashAttentionImpl(2, 64, 1.0, 2, None, None, "auto")
    for one in (1.0, 1, torch.tensor(1.0), torch.ones(1)):
        assert impl.forward(x, x, x, None, None, Meta, one).shape == (0, 128)
    for other in (0.5, torch.tensor(2.0), torch.ones(2, 4, 2)):
        with pytest.raises(AssertionError, match="kv_scale"):
            impl.forward(x, x, x, None, None, Meta, other)
