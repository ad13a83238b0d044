"""What the operators of the KV cache in 4 bits and the log probabilities refuse, and their shapes, without a GPU."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from flashsvd_amd import _lib, hip_ops

BF16, U8 = torch.bfloat16, torch.uint8


def _on(i, dtype, *shape):
    return torch.empty(*shape, dtype=dtype, device=f"cuda:{i}")


def _cache(B=2, S=64, Hk=2, Dh=64, i=0):
    return [_on(i, U8, B, S, Hk, Dh // 2), _on(i, U8, B, S, Hk, Dh // 2), _on(i, U8, B, Hk, Dh // 32, S), _on(i, U8, B, Hk, Dh // 32, S)]


def _refused(call, match):
    with pytest.raises((ValueError, TypeError, _lib.FlashSVDHipError), match=match):
        call()


def test_caches_that_are_refused():
    with FakeTensorMode():
        k = _on(0, BF16, 2, 3, 2, 64)
        pos = _on(0, torch.int32, 2)
        call = lambda c, kk=k, vv=k, p=pos, cos=None, sin=None, rows=None: hip_ops._kv4_append_impl(kk, vv, *c, p, cos, sin, rows)      # noqa: E731
        c = _cache()
        _refused(lambda: call([c[0].view(torch.float8_e4m3fn), *c[1:]]), "k_cache must be torch.uint8")
        _refused(lambda: call([c[0], c[1][:, :48], *c[2:]]), "matching")
        _refused(lambda: call([*c[:3], c[3].float()]), "v_scale must be")
        _refused(lambda: call([*c[:2], *_cache(S=128)[2:]]), "scales must be")
        _refused(lambda: call([*c[:2], *(t.transpose(2, 3).contiguous().transpose(2, 3) for t in c[2:])]), "unit inner stride")
        _refused(lambda: call(_cache(B=1)), "caches must be")
        _refused(lambda: call([_on(0, U8, 2, 64, 2, 24), _on(0, U8, 2, 64, 2, 24), *c[2:]]), "caches must be")
        _refused(lambda: call([*_cache(i=1)]), "on cuda:1")
        _refused(lambda: call([c[0], c[1], c[2], _cache(i=1)[3]]), "one device")
        _refused(lambda: call([t[:1].expand(2, *t.shape[1:]) for t in c]), "expanded")
        _refused(lambda: call([*(t[:, :1].expand(-1, 64, -1, -1) for t in c[:2]), *c[2:]]), "expanded")
        _refused(lambda: call(c, kk=k.half()), "v must be torch.float16")
        _refused(lambda: call(c, vv=k[:, :2]), "k and v must be")
        _refused(lambda: call(c, p=pos.long()), "positions must be")
        _refused(lambda: call(c, p=_on(0, torch.int32, 3)), "positions must be")
        _refused(lambda: call(c, p=_on(0, torch.int32, 4)[::2]), "positions must be")
        _refused(lambda: call(c, rows=_on(1, torch.int32, 2)), "rows must be")
        _refused(lambda: call(c, cos=_on(0, BF16, 9, 32)), "cos and sin")
        _refused(lambda: call(c, cos=_on(0, BF16, 9, 64), sin=_on(0, BF16, 9, 64)), "tables")
        read = lambda length=None, dtype=BF16: hip_ops._kv4_dequantize_impl(*c, length, dtype)      # noqa: E731
        _refused(lambda: read(length=65), "length must be")
        _refused(lambda: read(length=-1), "length must be")
        _refused(lambda: read(dtype=torch.float32), "bfloat16 or torch.float16")


def test_attention_calls_that_are_refused():
    with FakeTensorMode():
        c, n = _cache(), _on(0, torch.int32, 2)
        q, k = _on(0, BF16, 2, 4, 64), _on(0, BF16, 2, 2, 64)
        call = lambda q=q, n=n, k=None, v=None, out=None, c=c, cos=None, sin=None, add=0: hip_ops._attn_decode_kv4_impl(q, *c, n, k, v, cos, sin, add, None, None, out)      # noqa: E731
        _refused(lambda: call(q=_on(0, BF16, 2, 3, 64)), "does not match")
        _refused(lambda: call(q=_on(0, BF16, 2, 4, 128)), "does not match")
        _refused(lambda: call(q=_on(1, BF16, 2, 4, 64)), "does not match")
        _refused(lambda: call(q=_on(0, torch.float32, 2, 4, 64)), "bfloat16 or torch.float16")
        _refused(lambda: call(q=_on(0, BF16, 2, 4, 128)[..., ::2]), "unit inner stride")
        _refused(lambda: call(n=_on(0, torch.int64, 2)), "cache_seqlens")
        _refused(lambda: call(add=1 << 31), "32-bit")
        _refused(lambda: call(k=k), "go together")
        _refused(lambda: call(k=k, v=k[:, :1]), "k_new/v_new")
        _refused(lambda: call(k=k, v=_on(1, BF16, 2, 2, 64)), "k_new/v_new")
        _refused(lambda: call(k=k, v=k, c=[t[:1].expand(2, *t.shape[1:]) for t in c]), "expanded")
        _refused(lambda: call(out=_on(0, BF16, 2, 4, 32)), "out must be")
        p = _on(0, BF16, 2, 5, 4, 64)
        chunk = lambda q=p, n=n, rows=None, out=None: hip_ops._attn_prefill_kv4_impl(q, *c, n, rows, None, None, None, out)      # noqa: E731
        _refused(lambda: chunk(q=p[..., ::2]), "unit inner stride")
        _refused(lambda: chunk(q=p[:, :, :3]), "does not match")
        _refused(lambda: chunk(rows=_on(0, torch.int32, 3)), "rows must be")
        _refused(lambda: chunk(out=p[:1]), "out must be")


def test_log_probabilities_that_are_refused():
    with FakeTensorMode():
        x, t = _on(0, BF16, 2, 3, 50), _on(0, torch.long, 2, 3)
        call = lambda x=x, t=t, top=0: hip_ops._token_logprobs_impl(x, t, top)      # noqa: E731
        _refused(lambda: call(x=x.double()), "bfloat16 or torch.float16")
        _refused(lambda: call(x=x[0, 0], t=t[0, 0]), "logits must be")
        _refused(lambda: call(x=x[..., ::2]), "unit inner stride")
        _refused(lambda: call(x=x[..., :0]), "logits must be")
        _refused(lambda: call(t=t.int()), "tokens must be")
        _refused(lambda: call(t=t[:1]), "tokens must be")
        _refused(lambda: call(t=_on(1, torch.long, 2, 3)), "tokens must be")
        _refused(lambda: call(top=51), "top must be 0 to 50")
        _refused(lambda: call(top=-1), "top must be")
        _refused(lambda: call(x=_on(0, BF16, 2, 3, 100), top=65), "top must be 0 to 64")
        out = call(x=x[:0], t=t[:0], top=4)                       # no rows
        assert [tuple(o.shape) for o in out] == [(0, 3), (0, 3), (0, 3, 4), (0, 3, 4)]


def test_shapes_and_what_is_written():
    ops = torch.ops.flashsvd_hip
    m = lambda dt, *s: torch.empty(*s, dtype=dt, device="meta")      # noqa: E731
    c = [m(U8, 2, 64, 2, 32), m(U8, 2, 64, 2, 32), m(U8, 2, 2, 2, 64), m(U8, 2, 2, 2, 64)]
    n = m(torch.int32, 2)
    assert ops.attn_decode_kv4(m(BF16, 2, 4, 64), *c, n).shape == (2, 4, 64)
    assert ops.attn_prefill_kv4(m(BF16, 2, 9, 4, 64), *c, n).shape == (2, 9, 4, 64)
    assert ops.kv4_append(m(BF16, 2, 9, 2, 64), m(BF16, 2, 9, 2, 64), *c, n) is None
    k, v = ops.kv4_dequantize(*c, 7, torch.float16)
    assert k.shape == v.shape == (2, 7, 2, 64) and k.dtype == torch.float16 and ops.kv4_dequantize(*c)[0].shape == (2, 64, 2, 64)
    out = ops.token_logprobs(m(BF16, 4, 6, 50), m(torch.long, 4, 6), 3)
    assert [(tuple(o.shape), o.dtype) for o in out] == [((4, 6), torch.float32)] * 2 + [((4, 6, 3), torch.long), ((4, 6, 3), torch.float32)]
    for name in ("kv4_append", "attn_decode_kv4"):
        schema = str(getattr(ops, name).default._schema)
        for a, t in zip("abcd", ("k_cache", "v_cache", "k_scale", "v_scale")):
            assert f"Tensor({a}!) {t}" in schema


GOOD = dict(k=1 << 20, v=1 << 20, k_scale=1 << 20, v_scale=1 << 20, sc_b=64 * 64, sc_s=64, sc_h=32, ss_b=256, ss_h=128, ss_g=64, S=64, Hk=2, Dh=64)


def test_refusals_of_the_c_abi():
    """Bad descriptors come back as status codes with a message; nothing is launched."""
    lib = _lib.load()
    p = 1 << 20
    append = lambda c, B=1, T=1, dt=0, k=p, cos=None, rope=0: lib.fsvd_kv4_append(c, k, 64, 64, 64, p, 64, 64, 64, p, None, cos, cos, rope, B, T, dt, None)      # noqa: E731
    cache = lambda **kw: _lib.Kv4Cache(**(GOOD | kw))      # noqa: E731
    for kw, code in ((dict(k=None), -4), (dict(v_scale=None), -4), (dict(Dh=96), -1), (dict(S=0), -1), (dict(S=80), -1), (dict(Hk=0), -1), (dict(k=p + 8), -2),
                     (dict(k_scale=p + 1), -2), (dict(sc_s=72), -2), (dict(ss_g=72), -2), (dict(ss_g=48), -1), (dict(sc_s=16), -1), (dict(sc_b=-16), -1),
                     (dict(ss_h=-16), -1), (dict(sc_s=(1 << 24) + 16), -1)):
        assert append(cache(**kw)) == code, kw
        assert b"fsvd_kv4_append" in lib.fsvd_last_error()
    assert append(cache(), B=0) == -1 and append(cache(), B=65536) == -1 and append(cache(), T=-1) == -1 and append(cache(), dt=2) == -3
    assert append(cache(), k=None) == -4 and append(cache(), cos=p) == -4 and append(None) == -4
    assert append(cache(), T=0) == 0                      # nothing to write
    read = lambda L=64, B=1, dt=0, k=p, so=(8192, 128, 64): lib.fsvd_kv4_dequantize(cache(), k, p, *so, B, L, dt, None)      # noqa: E731
    assert read(L=65) == -1 and read(L=-1) == -1 and read(B=0) == -1 and read(dt=2) == -3 and read(k=None) == -4 and read(L=0, k=None) == 0
    assert read(so=(8192, 0, 64)) == -1 and read(so=(0, 128, 64), B=2) == -1 and read(so=(8192, 128, 0)) == -1
    decode = lambda H=2, out=p, v=None, c=cache(): lib.fsvd_attn_decode_kv4(c, p, 128, 64, p if v else None, 64, 64, None, 64, 64, p, 0, None, None, 0, out, 128, 64, None, 0, 1, H, 0, 0.0, 0, None)      # noqa: E731
    assert decode(H=3) == -1 and decode(out=None) == -4 and decode(v=True) == -4 and decode(c=cache(Dh=32)) == -1
    chunk = lambda H=2, M=1, q=p: lib.fsvd_attn_prefill_kv4(cache(), q, 128, 128, 64, p, None, None, None, 0, p, 128, 128, 64, None, 0, 1, M, H, 0.0, 0, None)      # noqa: E731
    assert chunk(H=3) == -1 and chunk(M=-1) == -1 and chunk(q=None) == -4 and chunk(M=0) == 0
    lp = lambda x=p, B=1, T=1, V=8, top=0, dt=0, ids=None: lib.fsvd_token_logprobs(x, 8, 8, p, p, p, ids, ids, None, 0, B, T, V, top, dt, None)      # noqa: E731
    assert lp(x=None) == -4 and lp(B=-1) == -1 and lp(V=0) == -1 and lp(V=(1 << 24) + 1) == -1 and lp(dt=2) == -3 and lp(x=p + 1) == -2
    assert lp(top=1) == -4 and lp(top=9, ids=p) == -1 and lp(V=100, top=65, ids=p) == -1 and lp(top=-1) == -1 and lp(B=0) == 0 and lp(T=0, x=None) == 0
    assert lp(B=1 << 16, T=1 << 16) == -1
    assert lp(B=1 << 11, T=1 << 11) == -1 and b"rows" in lib.fsvd_last_error()      # more workgroups than a launch has


def test_tensors_that_a_call_writes_are_not_expanded():
    lib = _lib.load()
    p = 1 << 20
    for kw in (dict(sc_b=0), dict(ss_b=0), dict(sc_h=0), dict(ss_h=0)):
        c = _lib.Kv4Cache(**(GOOD | kw))
        assert lib.fsvd_kv4_append(c, p, 64, 64, 64, p, 64, 64, 64, p, None, None, None, 0, 2, 1, 0, None) == -1
        assert b"expanded" in lib.fsvd_last_error()
        assert lib.fsvd_attn_decode_kv4(c, p, 128, 64, p, 64, 64, p, 64, 64, p, 0, None, None, 0, p, 128, 64, p, 1 << 30, 2, 2, 0, 0.0, 0, None) == -1
        assert b"expanded" in lib.fsvd_last_error()
    c = _lib.Kv4Cache(**GOOD)
    for so in ((0, 64), (128, 0)):
        assert lib.fsvd_attn_decode_kv4(c, p, 128, 64, None, 0, 0, None, 0, 0, p, 0, None, None, 0, p, *so, p, 1 << 30, 2, 2, 0, 0.0, 0, None) == -1
        assert b"out must not" in lib.fsvd_last_error()
    for so in ((0, 128, 64), (640, 0, 64), (640, 128, 0)):
        assert lib.fsvd_attn_prefill_kv4(c, p, 640, 128, 64, p, None, None, None, 0, p, *so, p, 1 << 30, 2, 5, 2, 0.0, 0, None) == -1
        assert b"out must not" in lib.fsvd_last_error()
