"""FlashSVDKV4Cache on the CPU, its operators replaced by the definition in 64 bits: storage, positions in any order, what update() returns, refusals."""
from types import SimpleNamespace

import pytest
import torch

from tests import kv4_reference as R

BF16 = torch.bfloat16
CFG = SimpleNamespace(num_hidden_layers=2, rope_theta=10000.0)


def _pack(values, size):
    """Codes uint8 [.., Dh / 2] of values [.., Dh] that are code * size."""
    table = torch.cat((R.CODES, -R.CODES))
    y = values / size
    code = (y.abs()[..., None] - R.CODES).abs().argmin(-1) | torch.where(y.signbit(), 8, 0)
    assert torch.equal(table[code], y)
    return (code[..., 0::2] | code[..., 1::2] << 4).to(torch.uint8)


@pytest.fixture
def cache(monkeypatch):
    from flashsvd_amd import hip_ops
    from flashsvd_amd.runtime import FlashSVDKV4Cache

    def append(k, v, k_cache, v_cache, k_scale, v_scale, positions, *, cos=None, sin=None, rows=None):
        for x, codes, scales in ((k, k_cache, k_scale), (v, v_cache, v_scale)):
            for b in range(x.shape[0]):
                values = R.unpack(codes[b], scales[b])
                R.append(values, scales[b], x[b], int(positions[b]), x.shape[1])
                size = torch.exp2(scales[b].double() - 127).movedim(-1, -3).repeat_interleave(32, -1)
                codes[b].copy_(_pack(values, size))

    def dequantize(k_cache, v_cache, k_scale, v_scale, *, length, dtype):
        return tuple(R.unpack(c, s)[:, :length].to(dtype) for c, s in ((k_cache, k_scale), (v_cache, v_scale)))

    monkeypatch.setattr(hip_ops, "kv4_append", append)
    monkeypatch.setattr(hip_ops, "kv4_dequantize", dequantize)
    return FlashSVDKV4Cache(CFG, max_batch_size=2, max_cache_len=70, dtype=BF16)


def _rows(n, seed, dh=64):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(2, 3, n, dh, generator=g).to(BF16) for _ in range(2)]


def _rounded(x):
    flat = x.double().reshape(-1, 32)
    return torch.stack([R.group_values(r)[1] for r in flat]).view(x.shape).to(BF16)


def test_storage():
    from flashsvd_amd.runtime import FlashSVDKV4Cache, FlashSVDV15DenseKVCache
    c = FlashSVDKV4Cache(CFG, max_batch_size=3, max_cache_len=70)
    assert not isinstance(c, FlashSVDV15DenseKVCache) and len(c) == 2 and c.max_cache_len == 70
    c._ensure_layer_spec(1, h=4, dh=64)
    k, v, ks, vs = c.operands(1, 2)
    assert k.shape == v.shape == (2, 128, 4, 32) and k.dtype == ks.dtype == torch.uint8 and k.stride(3) == 1 and k.stride(1) == 32
    assert ks.shape == vs.shape == (2, 4, 2, 128) and ks.stride(3) == 1
    assert c.key_cache[0].shape == (3, 128, 0, 0)
    assert k.data_ptr() != v.data_ptr() and ks.data_ptr() != vs.data_ptr()
    c._ensure_layer_spec(1, h=2, dh=128)                   # nothing written: the shape may still change
    assert c.operands(1, 1)[0].shape == (1, 128, 2, 64)
    for dh in (32, 96, 256, 65):
        with pytest.raises(ValueError, match="64 or 128"):
            c._ensure_layer_spec(0, h=2, dh=dh)


def test_updates_in_any_order(cache):
    k, v = _rows(20, 1)
    K, V = cache.update(k, v, 0, {"cache_position": torch.arange(20)})
    assert torch.equal(K, _rounded(k)) and torch.equal(V, _rounded(v)) and cache.get_seq_length() == 20
    k2, v2 = _rows(5, 2)
    at = [3, 4, 25, 3, 69]                                  # a gap, the same position twice, the last one
    K, V = cache.update(k2, v2, 0, {"cache_position": torch.tensor(at)})
    assert K.shape == (2, 3, 70, 64) and cache.get_seq_length() == 70
    want = torch.zeros(2, 3, 70, 64, dtype=BF16)
    want[:, :, :20] = _rounded(k)
    for i, p in enumerate(at):
        want[:, :, p] = _rounded(k2)[:, :, i]
    assert torch.equal(K, want)
    K, V = cache.update(k2, v2, 1)                          # without positions: from the start; layer 0 counts
    assert torch.equal(V, _rounded(v2)) and cache.get_seq_length() == 70
    cache.reset()
    K, V = cache.update(k2[:1], v2[:1], 0)                  # fewer sequences than the cache has
    assert K.shape == (1, 3, 5, 64) and cache.get_seq_length() == 5


def test_refusals(cache):
    k, v = _rows(4, 3)
    for at in ([67, 68, 69, 70], [-1, 0, 1, 2]):
        with pytest.raises(IndexError, match="out of range"):
            cache.update(k, v, 0, {"cache_position": torch.tensor(at)})
    with pytest.raises(ValueError, match="a position for each"):
        cache.update(k, v, 0, {"cache_position": torch.arange(3)})
    cache.update(k, v, 0)
    with pytest.raises(RuntimeError, match="shape changed"):
        cache.update(*(x.repeat(1, 2, 1, 1) for x in (k, v)), 0)
    K, V = cache.update(k[:, :, :0], v[:, :, :0], 0, {"cache_position": torch.arange(0)})
    assert K.shape[2] == 4


def test_the_serving_functions_take_one_cache():
    from flashsvd_amd import api
    from flashsvd_amd.runtime import FlashSVDKV4Cache
    model = torch.nn.Linear(2, 2)
    model.config = CFG
    with pytest.raises(ValueError, match="mutually exclusive"):
        api._build_generation_cache(model, prompt_len=3, max_new_tokens=3, batch_size=1, device="cpu", kv8_cache=True, kv4_cache=True)
    c, _ = api._build_generation_cache(model, prompt_len=3, max_new_tokens=3, batch_size=1, device="cpu", kv4_cache=True)
    assert isinstance(c, FlashSVDKV4Cache) and c.max_cache_len == 10
    for other in ("kv8_cache", "lowrank_cache", "flashsvd_dense_cache", "baseline_dense_kvcache"):
        with pytest.raises(ValueError, match="mutually exclusive"):
            api.decode_kvcache_eval(model, kv4_cache=True, **{other: True})
    for n in (-1, 65):
        with pytest.raises(ValueError, match="logprobs"):
            api.generate_text(model, None, prompt="x", logprobs=n)


def test_without_a_gpu_nothing_runs():
    from flashsvd_amd.runtime import FlashSVDKV4Cache
    c = FlashSVDKV4Cache(CFG, max_batch_size=2, max_cache_len=70, dtype=BF16)
    with pytest.raises(ValueError, match="GPU|device"):
        c.update(*_rows(2, 1), 0)
