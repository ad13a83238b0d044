"""The limit of the operators over the cache in 4 bits, what it refuses and what FlashSVDKV4Cache gives them, without a GPU."""
from types import SimpleNamespace

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from flashsvd_amd import _lib, hip_ops
from tests.test_kv4_host import BF16, GOOD, _cache, _on

CFG = SimpleNamespace(num_hidden_layers=1, rope_theta=10000.0)


def test_limits_that_are_refused():
    with FakeTensorMode():
        c, n = _cache(), _on(0, torch.int32, 2)
        k, q, p = _on(0, BF16, 2, 3, 2, 64), _on(0, BF16, 2, 4, 64), _on(0, BF16, 2, 5, 4, 64)
        for limit in (0, -1, 65):
            for call in (lambda: hip_ops._kv4_append_impl(k, k, *c, n, None, None, None, limit),
                         lambda: hip_ops._attn_decode_kv4_impl(q, *c, n, None, None, None, None, 0, None, None, None, limit),
                         lambda: hip_ops._attn_prefill_kv4_impl(p, *c, n, None, None, None, None, None, limit)):
                with pytest.raises(ValueError, match="limit must be 1 to 64"):
                    call()


def test_refusals_of_the_c_abi():
    lib, p = _lib.load(), 1 << 20
    for limit in (-1, 65):
        c = _lib.Kv4Cache(**(GOOD | dict(limit=limit)))
        assert lib.fsvd_kv4_append(c, p, 64, 64, 64, p, 64, 64, 64, p, None, None, None, 0, 1, 1, 0, None) == -1
        assert b"limit" in lib.fsvd_last_error()
    assert lib.fsvd_kv4_append(_lib.Kv4Cache(**(GOOD | dict(limit=64))), p, 64, 64, 64, p, 64, 64, 64, p, None, None, None, 0, 1, 0, 0, None) == 0


@pytest.mark.parametrize("length,limit", [(70, 70), (128, None), (1, 1)])
def test_the_cache_gives_its_length(length, limit, monkeypatch):
    from flashsvd_amd.runtime import FlashSVDKV4Cache
    seen = []
    for name in ("kv4_append", "attn_decode_kv4", "attn_prefill_kv4"):
        monkeypatch.setattr(hip_ops, name, lambda *a, limit, **k: seen.append(limit))
    c = FlashSVDKV4Cache(CFG, max_batch_size=2, max_cache_len=length, dtype=BF16)
    c.append(0, torch.zeros(2, 1, 2, 64), torch.zeros(2, 1, 2, 64), None)
    c.attend_token(0, torch.zeros(2, 2, 64), None)
    c.attend_chunk(0, torch.zeros(2, 1, 2, 64), None)
    assert seen == [limit] * 3
