"""What the operators of the KV cache in 8 bits and the draw of a token refuse, and their shapes, without a GPU."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from flashsvd_amd import _lib, hip_ops

BF16, F8 = torch.bfloat16, torch.float8_e4m3fn


def _on(i, dtype, *shape):
    return torch.empty(*shape, dtype=dtype, device=f"cuda:{i}")


def _cache(B=2, S=40, Hk=2, Dh=64, block=16, i=0):
    return [_on(i, F8, B, S, Hk, Dh), _on(i, F8, B, S, Hk, Dh), _on(i, torch.float32, B, -(-S // block), Hk), _on(i, torch.float32, B, -(-S // block), Hk)]


def _refused(call, match):
    with pytest.raises((ValueError, TypeError), match=match):
        call()


def test_caches_that_are_refused():
    with FakeTensorMode():
        k = _on(0, BF16, 2, 3, 2, 64)
        pos = _on(0, torch.int32, 2)
        call = lambda c, kk=k, vv=k, p=pos, block=16, cos=None, sin=None, rows=None: hip_ops._kv8_append_impl(kk, vv, *c, p, block, cos, sin, rows)      # noqa: E731
        c = _cache()
        _refused(lambda: call(c, block=24), "block must be")
        _refused(lambda: call(c, block=32), "scales must be")
        _refused(lambda: call([c[0].view(torch.uint8), *c[1:]]), "k_cache must be torch.float8")
        _refused(lambda: call([c[0], c[1][:, :39], *c[2:]]), "matching")
        _refused(lambda: call([*c[:3], c[3].half()]), "v_scale must be")
        _refused(lambda: call(_cache(B=1)), "caches must be")
        _refused(lambda: call([*_cache(i=1)]), "on cuda:1")
        _refused(lambda: call([c[0], c[1], c[2], _cache(i=1)[3]]), "one device")
        _refused(lambda: call([t[:1].expand(2, *t.shape[1:]) for t in c]), "expanded")
        _refused(lambda: call([c[0], c[1], c[2][:, :, :1].expand(-1, -1, 2), c[3][:, :, :1].expand(-1, -1, 2)]), "expanded")
        _refused(lambda: call(c, kk=k.half()), "v must be torch.float16")
        _refused(lambda: call(c, vv=k[:, :2]), "k and v must be")
        _refused(lambda: call(c, p=pos.long()), "positions must be")
        _refused(lambda: call(c, p=_on(0, torch.int32, 3)), "positions must be")
        _refused(lambda: call(c, p=_on(0, torch.int32, 4)[::2]), "positions must be")
        _refused(lambda: call(c, rows=_on(1, torch.int32, 2)), "rows must be")
        _refused(lambda: call(c, cos=_on(0, BF16, 9, 32)), "cos and sin")
        _refused(lambda: call(c, cos=_on(0, BF16, 9, 32), sin=_on(1, BF16, 9, 32)), "cos and sin")
        _refused(lambda: call(c, cos=_on(0, BF16, 9, 64), sin=_on(0, BF16, 9, 64)), "tables")


def test_attention_calls_that_are_refused():
    with FakeTensorMode():
        c, n = _cache(), _on(0, torch.int32, 2)
        q, k = _on(0, BF16, 2, 4, 64), _on(0, BF16, 2, 2, 64)
        call = lambda q=q, n=n, k=None, v=None, out=None, c=c, cos=None, sin=None: hip_ops._attn_decode_kv8_impl(q, *c, n, 16, k, v, cos, sin, 0, None, None, out)      # noqa: E731
        _refused(lambda: call(q=_on(0, BF16, 2, 3, 64)), "does not match")
        _refused(lambda: call(q=_on(0, BF16, 2, 4, 128)), "does not match")
        _refused(lambda: call(q=_on(1, BF16, 2, 4, 64)), "does not match")
        _refused(lambda: call(q=_on(0, torch.float32, 2, 4, 64)), "bfloat16 or torch.float16")
        _refused(lambda: call(q=_on(0, BF16, 2, 4, 128)[..., ::2]), "unit inner stride")
        _refused(lambda: call(n=_on(0, torch.int64, 2)), "cache_seqlens")
        _refused(lambda: call(k=k), "go together")
        _refused(lambda: call(k=k, v=k[:, :1]), "k_new/v_new")
        _refused(lambda: call(k=k, v=_on(1, BF16, 2, 2, 64)), "k_new/v_new")
        _refused(lambda: call(k=k, v=k, c=[t[:1].expand(2, *t.shape[1:]) for t in c]), "expanded")
        _refused(lambda: call(out=_on(0, BF16, 2, 4, 32)), "out must be")
        p = _on(0, BF16, 2, 5, 4, 64)
        chunk = lambda q=p, n=n, rows=None, out=None: hip_ops._attn_prefill_kv8_impl(q, *c, n, 16, rows, None, None, None, out)      # noqa: E731
        _refused(lambda: chunk(q=p[..., ::2]), "unit inner stride")
        _refused(lambda: chunk(q=p[:, :, :3]), "does not match")
        _refused(lambda: chunk(rows=_on(0, torch.int32, 3)), "rows must be")
        _refused(lambda: chunk(out=p[:1]), "out must be")


def test_draws_that_are_refused():
    with FakeTensorMode():
        x, u, t, p = _on(0, BF16, 2, 50), _on(0, torch.float32, 2), _on(0, torch.long, 2, 1), _on(0, torch.int32, 2)
        call = lambda x=x, u=u, t=t, p=p, ts=None, ks=None, ps=None, ms=None: hip_ops._sample_token_impl(x, u, t, p, 1.0, 0, 1.0, 0.0, ts, ks, ps, ms)      # noqa: E731
        _refused(lambda: call(x=_on(0, torch.float32, 2, 50)), "bfloat16 or torch.float16")
        _refused(lambda: call(x=_on(0, BF16, 50, 2).t()), "unit inner stride")
        _refused(lambda: call(u=u.double()), "uniforms")
        _refused(lambda: call(u=_on(0, torch.float32, 3)), "uniforms")
        _refused(lambda: call(t=_on(0, torch.int32, 2, 1)), "tokens")
        _refused(lambda: call(t=_on(0, torch.long, 1, 2)), "tokens")
        _refused(lambda: call(t=_on(1, torch.long, 2, 1)), "one device")
        _refused(lambda: call(p=_on(1, torch.int32, 2)), "positions")
        for name in ("ts", "ps", "ms"):
            _refused(lambda: call(**{name: _on(0, torch.float64, 2)}), "contiguous")
        _refused(lambda: call(ks=_on(0, torch.int64, 2)), "top_k")


def test_shapes_and_what_is_written():
    ops = torch.ops.flashsvd_hip
    m = lambda dt, *s: torch.empty(*s, dtype=dt, device="meta")      # noqa: E731
    c = [m(F8, 2, 40, 2, 64), m(F8, 2, 40, 2, 64), m(torch.float32, 2, 3, 2), m(torch.float32, 2, 3, 2)]
    n = m(torch.int32, 2)
    assert ops.attn_decode_kv8(m(BF16, 2, 4, 64), *c, n, 16).shape == (2, 4, 64)
    assert ops.attn_prefill_kv8(m(BF16, 2, 9, 4, 64), *c, n, 16).shape == (2, 9, 4, 64)
    assert ops.kv8_append(m(BF16, 2, 9, 2, 64), m(BF16, 2, 9, 2, 64), *c, n, 16) is None
    for name, args in (("kv8_append", "abcd"), ("attn_decode_kv8", "abcd")):
        schema = str(getattr(ops, name).default._schema)
        for a, t in zip(args, ("k_cache", "v_cache", "k_scale", "v_scale")):
            assert f"Tensor({a}!) {t}" in schema
    assert "Tensor(a!) tokens" in str(ops.sample_token_.default._schema)


def test_refusals_of_the_c_abi():
    """Bad descriptors come back as status codes with a message; nothing is launched."""
    lib = _lib.load()
    p = 1 << 20
    good = dict(k=p, v=p, k_scale=p, v_scale=p, sc_b=40 * 128, sc_s=128, sc_h=64, ss_b=6, ss_n=2, ss_h=1, S=40, Hk=2, Dh=64, block=16)
    append = lambda c, B=1, T=1, dt=0, k=p, cos=None, rope=0: lib.fsvd_kv8_append(c, k, 64, 64, 64, p, 64, 64, 64, p, None, cos, cos, rope, B, T, dt, None)      # noqa: E731
    cache = lambda **kw: _lib.Kv8Cache(**(good | kw))      # noqa: E731
    for kw, code in ((dict(k=None), -4), (dict(v_scale=None), -4), (dict(Dh=96), -1), (dict(block=8), -1), (dict(S=0), -1), (dict(k=p + 8), -2),
                     (dict(sc_s=72), -2), (dict(sc_b=-16), -1), (dict(ss_n=(1 << 26) + 1), -1), (dict(sc_s=(1 << 26) + 16), -1)):
        assert append(cache(**kw)) == code, kw
        assert b"fsvd_kv8_append" in lib.fsvd_last_error()
    assert append(cache(), B=0) == -1 and append(cache(), T=-1) == -1 and append(cache(), dt=2) == -3 and append(cache(), k=None) == -4
    assert append(cache(), cos=p) == -4 and append(None) == -4
    assert append(cache(), T=0) == 0                      # nothing to write
    decode = lambda H=2, out=p, v=None, c=cache(): lib.fsvd_attn_decode_kv8(c, p, 128, 64, p if v else None, 64, 64, None, 64, 64, p, 0, None, None, 0, out, 128, 64, None, 0, 1, H, 0, 0.0, 0, None)      # noqa: E731
    assert decode(H=3) == -1 and decode(out=None) == -4 and decode(v=True) == -4 and decode(c=cache(Dh=32)) == -1
    chunk = lambda H=2, M=1, q=p: lib.fsvd_attn_prefill_kv8(cache(), q, 128, 128, 64, p, None, None, None, 0, p, 128, 128, 64, None, 0, 1, M, H, 0.0, 0, None)      # noqa: E731
    assert chunk(H=3) == -1 and chunk(M=-1) == -1 and chunk(q=None) == -4 and chunk(M=0) == 0
    draw = lambda x=p, B=1, V=8, dt=0: lib.fsvd_sample_token(x, 8, p, p, 1, None, 1.0, None, 0, None, 1.0, None, 0.0, None, B, V, dt, None)      # noqa: E731
    assert draw(x=None) == -4 and draw(B=0) == -1 and draw(V=0) == -1 and draw(V=(1 << 24) + 1) == -1 and draw(dt=2) == -3 and draw(x=p + 1) == -2


def test_tensors_that_a_call_writes_are_not_expanded():
    lib = _lib.load()
    p = 1 << 20
    good = dict(k=p, v=p, k_scale=p, v_scale=p, sc_b=40 * 128, sc_s=128, sc_h=64, ss_b=6, ss_n=2, ss_h=1, S=40, Hk=2, Dh=64, block=16)
    for kw in (dict(sc_b=0), dict(ss_b=0), dict(sc_h=0), dict(ss_h=0), dict(ss_n=0)):
        c = _lib.Kv8Cache(**(good | kw))
        assert lib.fsvd_kv8_append(c, p, 64, 64, 64, p, 64, 64, 64, p, None, None, None, 0, 2, 1, 0, None) == -1
        assert b"expanded" in lib.fsvd_last_error()
        assert lib.fsvd_attn_decode_kv8(c, p, 128, 64, p, 64, 64, p, 64, 64, p, 0, None, None, 0, p, 128, 64, p, 1 << 30, 2, 2, 0, 0.0, 0, None) == -1
        assert b"expanded" in lib.fsvd_last_error()
    c = _lib.Kv8Cache(**good)
    for so in ((0, 64), (128, 0)):
        assert lib.fsvd_attn_decode_kv8(c, p, 128, 64, None, 0, 0, None, 0, 0, p, 0, None, None, 0, p, *so, p, 1 << 30, 2, 2, 0, 0.0, 0, None) == -1
        assert b"out must not" in lib.fsvd_last_error()
    for so in ((0, 128, 64), (640, 0, 64), (640, 128, 0)):
        assert lib.fsvd_attn_prefill_kv8(c, p, 640, 128, 64, p, None, None, None, 0, p, *so, p, 1 << 30, 2, 5, 2, 0.0, 0, None) == -1
        assert b"out must not" in lib.fsvd_last_error()
    assert lib.fsvd_sample_token(p, 8, p, p, 0, None, 1.0, None, 0, None, 1.0, None, 0.0, None, 2, 8, 0, None) == -1
    assert b"tokens must not" in lib.fsvd_last_error()
    with FakeTensorMode():                                 # no rows: nothing to do
        none = lambda dt, *s: _on(0, dt, *s)      # noqa: E731
        hip_ops._sample_token_impl(none(BF16, 0, 9), none(torch.float32, 0), none(torch.long, 0, 1), None, 1.0, 0, 1.0, 0.0, None, None, None, None)


def test_the_cache_object_without_a_gpu():
    from types import SimpleNamespace
    from flashsvd_amd.runtime import FlashSVDKV8Cache, FlashSVDV15DenseKVCache
    cfg = SimpleNamespace(num_hidden_layers=2, rope_theta=10000.0)
    with pytest.raises(ValueError, match="block_size"):
        FlashSVDKV8Cache(cfg, max_batch_size=1, max_cache_len=8, block_size=24)
    c = FlashSVDKV8Cache(cfg, max_batch_size=3, max_cache_len=70, block_size=32)
    assert not isinstance(c, FlashSVDV15DenseKVCache) and len(c) == 2 and c.max_cache_len == 70
    c._ensure_layer_spec(1, h=4, dh=64)
    k, v, ks, vs = c.operands(1, 2)
    assert k.shape == v.shape == (2, 70, 4, 64) and k.dtype == F8 and k.stride(3) == 1 and k.stride(1) == 64
    assert ks.shape == vs.shape == (2, 3, 4) and ks.dtype == torch.float32
    assert c.key_cache[0].shape == (3, 70, 0, 0)
    K, V = c.dequantize(1, length=5)
    assert K.shape == (3, 5, 4, 64) and not bool(K.any()) and not bool(V.any())
    with pytest.raises(IndexError):
        c.update(torch.zeros(1, 4, 3, 64), torch.zeros(1, 4, 3, 64), 1, {"cache_position": torch.arange(68, 71)})
    with pytest.raises(ValueError, match="consecutive"):
        c.update(torch.zeros(1, 4, 2, 64), torch.zeros(1, 4, 2, 64), 1, {"cache_position": torch.tensor([4, 6])})
    with pytest.raises(ValueError, match="GPU tensor"):
        c.update(torch.zeros(1, 4, 2, 64), torch.zeros(1, 4, 2, 64), 1)
