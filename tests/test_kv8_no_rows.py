"""Calls of the KV cache in 8 bits without rows: an empty tensor has no address, and there is nothing to do."""
import pytest
import torch

from flashsvd_amd import _lib

BF16, F8 = torch.bfloat16, torch.float8_e4m3fn


def test_no_rows_need_no_buffers():
    lib = _lib.load()
    p = 1 << 20
    c = _lib.Kv8Cache(k=p, v=p, k_scale=p, v_scale=p, sc_b=40 * 128, sc_s=128, sc_h=64, ss_b=6, ss_n=2, ss_h=1, S=40, Hk=2, Dh=64, block=16)
    append = lambda T, k, pos: lib.fsvd_kv8_append(c, k, 64, 64, 64, k, 64, 64, 64, pos, None, None, None, 0, 1, T, 0, None)      # noqa: E731
    assert append(0, None, p) == 0 and append(1, None, p) == -4 and append(0, None, None) == -4 and append(-1, p, p) == -1
    chunk = lambda M, q, pos: lib.fsvd_attn_prefill_kv8(c, q, 128, 128, 64, pos, None, None, None, 0, q, 128, 128, 64, None, 0, 1, M, 2, 0.0, 0, None)      # noqa: E731
    assert chunk(0, None, p) == 0 and chunk(1, None, p) == -4 and chunk(0, None, None) == -4 and chunk(-1, p, p) == -1


@pytest.mark.gpu
def test_empty_chunks_leave_everything_as_it_was():
    from flashsvd_amd import hip_ops
    c = [torch.ones(2, 40, 2, 64, device="cuda").to(F8), torch.ones(2, 40, 2, 64, device="cuda").to(F8), torch.ones(2, 3, 2, device="cuda"),
         torch.ones(2, 3, 2, device="cuda")]
    pos = torch.tensor([3, 9], dtype=torch.int32, device="cuda")
    k = torch.zeros(2, 0, 2, 64, dtype=BF16, device="cuda")
    hip_ops.kv8_append(k, k, *c, pos, block=16)
    for rows in (None, torch.zeros(2, dtype=torch.int32, device="cuda")):
        assert hip_ops.attn_prefill_kv8(torch.zeros(2, 0, 4, 64, dtype=BF16, device="cuda"), *c, pos, block=16, rows=rows).shape == (2, 0, 4, 64)
    torch.cuda.synchronize()
    assert all(bool((t.float() == 1).all()) for t in c)
