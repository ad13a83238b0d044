"""Scores beyond 32 bits: keys whose score is -infinity in fp32 have no weight beside others, wherever they stand among the steps and ranges of a call."""
import pytest
import torch

from tests import kv4_reference as R
from tests.test_gpu_kv4 import HALF_PART, TWO_PARTS, Cache, _close
from tests.util import form_taken

pytestmark = pytest.mark.gpu


def _cache(S, Dh, low, seed=8, B=1, Hk=1):
    """Keys of -6 * 2^125 at `low`, which a query of positive numbers scores below -2^128."""
    c = Cache(B, S, Hk, Dh, seed=seed)
    c.t[0][:, low] = 0xff
    c.t[2][..., low] = 252
    return c


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("G", [4, 12])
@pytest.mark.parametrize("Dh", [64, 128])
@pytest.mark.parametrize("low", [slice(0, 64), slice(0, 256), slice(64, 700), slice(0, 1030), slice(1990, 2048), slice(3, 2047)])
def test_decode(low, Dh, G, dt):
    from flashsvd_amd import hip_ops
    S = 2048
    c = _cache(S, Dh, low)
    k, v = (x[0, :, 0] for x in c.values())
    q = torch.rand(1, G, Dh, generator=torch.Generator().manual_seed(3)).add(0.5).to(dt)
    keep = torch.ones(S, dtype=torch.bool)
    keep[low] = False
    n = torch.tensor([S], dtype=torch.int32, device="cuda")
    for nsplit in (1, 3, 8, None):
        out = hip_ops.attn_decode_kv4(q.cuda(), *c.t, n, nsplit=nsplit)
        for h in range(G):
            want, room = R.attend(q[0, h].double(), k[keep], v[keep], Dh ** -0.5, TWO_PARTS, TWO_PARTS)
            _close(out[0, h], want, room, dt, f"{low} in {nsplit} ranges")


@pytest.mark.parametrize("Dh", [64, 128])
@pytest.mark.parametrize("B,Hk,M,S,name", [(8, 32, 130, 320, "kv4 prompt 128"), (8, 25, 70, 128, "kv4 prompt 64"), (1, 1, 9, 2048, "kv4 prompt 64 halves ranges"),
                                           (2, 2, 40, 192, "kv4 prompt 64 halves")])
def test_prompts(B, Hk, M, S, name, Dh):
    from flashsvd_amd import hip_ops
    dt = torch.bfloat16
    for low in (slice(0, 64), slice(0, S - M - 1), slice(1, S - 3)):
        c = _cache(S, Dh, low, B=B, Hk=Hk)
        k, v = c.values()
        q = torch.rand(B, M, Hk, Dh, generator=torch.Generator().manual_seed(3)).add(0.5).to(dt)
        out = hip_ops.attn_prefill_kv4(q.cuda(), *c.t, torch.full((B,), S - M, dtype=torch.int32, device="cuda"))
        if name != "kv4 prompt 64":
            assert form_taken() == name or Dh == 64
        for m in (0, M // 2, M - 1):
            sees = torch.arange(S) <= S - M + m
            sees[low] = False
            for h in {0, Hk - 1}:
                want, room = R.attend(q[B - 1, m, h].double(), k[B - 1, sees, h], v[B - 1, sees, h], Dh ** -0.5, TWO_PARTS, HALF_PART)
                _close(out[B - 1, m, h], want, room, dt, f"{low} row {m} head {h}")
