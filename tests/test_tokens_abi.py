"""CPU: what the per-token and cache entry points refuse before they touch a device, and that they fail with a CUDA status, never
a host computation, where there is none."""
import ctypes as C

import pytest


def cache_desc(**kw):
    from ltq._binding import KVCacheDesc
    d = dict(k_dev=4096, k_qp_dev=4096, v_dev=4096, v_qp_dev=4096, blocks=4, kv_heads=2, block_tokens=16, head_dim=64)
    d.update(kw)
    return C.byref(KVCacheDesc(*d.values()))


def append(L, cache=None, k=4096, v=4096, dtype=0, ld=128, tokens=3, offsets=4096, lengths=4096, table=4096, seqs=1, width=2, max_new=3):
    return L.ltq_cache_append(cache or cache_desc(), k, v, dtype, ld, tokens, offsets, lengths, table, seqs, width, max_new, 0, None)


def attention(L, cache=None, q=4096, dtype=2, ld=256, tokens=3, heads=4, offsets=4096, lengths=4096, table=4096, seqs=1, width=2, max_new=3,
              scale=0.1, out=4096, ws=4096, ws_bytes=1 << 30):
    return L.ltq_cache_attention(cache or cache_desc(), q, dtype, ld, tokens, heads, offsets, lengths, table, seqs, width, max_new, scale, out, ws,
                                 ws_bytes, 0, None)


def test_tokens_arguments():
    import ltq
    L = ltq.lib()
    quant = lambda x=4096, dtype=0, m=2, k=8, ld=8, q=4096, qp=4096, s=4096: L.ltq_quantize_tokens_u8(x, dtype, m, k, ld, q, qp, s, 0, None)  # noqa: E731
    assert quant(x=None) == quant(q=None) == quant(qp=None) == -1
    assert quant(dtype=3) == quant(dtype=-1) == quant(k=0) == quant(ld=7) == -1
    assert quant(x=4098) == quant(x=4097, dtype=1) == quant(qp=4098) == quant(s=4099) == -1
    assert quant(k=1 << 31, ld=1 << 31) == -6
    assert quant(m=0) == 0 and quant(m=0, ld=0) == 0
    deq = lambda x=4096, dtype=0, ld=8, q=4096, qp=4096, m=2, k=8: L.ltq_dequantize_tokens_u8(x, dtype, ld, q, qp, m, k, 0, None)  # noqa: E731
    assert deq(x=None) == deq(q=None) == deq(qp=None) == deq(dtype=7) == deq(ld=3) == deq(x=4098) == -1
    assert deq(m=0) == 0


def test_layer_entry_points_need_a_layer():
    import ltq
    L = ltq.lib()
    assert L.ltq_layer_set_channel_qparams(None, 4096, None, None) == -1
    assert L.ltq_layer_forward_tokens(None, 4096, 4096, 4096, 1, 0, 0, 4096, 8, None) == -1
    assert L.ltq_layer_forward_float(None, 4096, 0, 8, 1, 0, 0, 4096, 8, 4096, 1 << 20, None) == -1
    assert L.ltq_layer_float_workspace(None, 5) == 0


@pytest.mark.parametrize("call", [append, attention])
def test_cache_arguments(call):
    import ltq
    L = ltq.lib()
    for name in ("k_dev", "v_dev", "k_qp_dev", "v_qp_dev"):
        assert call(L, cache_desc(**{name: None})) == -1
        assert call(L, cache_desc(**{name: 4100 if "qp" in name else 4104})) == -1, "misaligned"
    assert call(L, cache_desc(blocks=0)) == call(L, cache_desc(blocks=1 << 31)) == call(L, cache_desc(kv_heads=0)) == -1
    for bt in (0, 8, 24, 256):
        assert call(L, cache_desc(block_tokens=bt)) == -2
    for d in (0, 16, 80, 512):
        assert call(L, cache_desc(head_dim=d)) == -2
    assert call(L, dtype=3) == -1
    assert call(L, offsets=None) == call(L, lengths=None) == call(L, table=None) == call(L, lengths=4098) == -1
    assert call(L, seqs=65536) == -6
    assert call(L, max_new=4) == -1, "more new tokens in a sequence than rows"
    assert call(L, width=1 << 27) == -1, "positions beyond 2^31"
    assert call(L, ld=100) == -1
    for n in ("tokens", "seqs", "max_new"):
        assert call(L, **{n: 0, **({"max_new": 0} if n == "tokens" else {})}) == 0


def test_attention_arguments():
    import ltq
    L = ltq.lib()
    assert attention(L, heads=3) == attention(L, heads=0) == attention(L, heads=4096, ld=1 << 20) == -1
    assert attention(L, scale=float("inf")) == attention(L, scale=float("nan")) == -1
    assert attention(L, q=None) == attention(L, out=None) == attention(L, ws=4104) == attention(L, q=4097) == -1


def test_no_cpu_fallback():
    import torch
    if torch.cuda.is_available():
        pytest.skip("a CUDA device is present")
    import ltq
    L = ltq.lib()
    assert append(L) == attention(L) == -3
    assert L.ltq_quantize_tokens_u8(4096, 0, 2, 8, 8, 4096, 4096, None, 0, None) == -3
    assert L.ltq_cache_attention_workspace(cache_desc(), 3, 4, 1, 2, 3, 0) == 0


def test_python_checks():
    import torch
    import ltq
    with pytest.raises(ValueError, match="CUDA"):
        ltq.quantize_tokens(torch.zeros(2, 8))
    with pytest.raises(ValueError, match="CUDA"):
        ltq.dequantize_tokens(torch.zeros(2, 8, dtype=torch.uint8), torch.zeros(2, 8, dtype=torch.uint8))
    with pytest.raises(ValueError, match="CUDA"):
        ltq.FullyConnected_t(torch.zeros(2, 8, dtype=torch.uint8), torch.zeros(2, 8, dtype=torch.uint8))
    with pytest.raises(ValueError, match="CUDA"):
        ltq.KVCache.empty(2, 1, 16, 32, device="cpu")
