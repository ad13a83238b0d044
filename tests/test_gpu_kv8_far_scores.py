"""Scores beyond 32 bits over the cache in 8 bits: keys whose score is -infinity in fp32 have no weight beside others, and a wave whose keys are all NaN makes NaN."""
import pytest
import torch

from tests import kv8_reference as R
from tests.test_gpu_kv4 import TWO_PARTS, _close
from tests.test_gpu_kv8 import Cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("G", [4, 12])
@pytest.mark.parametrize("Dh", [64, 128])
@pytest.mark.parametrize("low", [slice(0, 32), slice(0, 128), slice(64, 704), slice(0, 1024), slice(1984, 2048), slice(32, 2016)])
def test_decode(low, Dh, G, dt):
    from flashsvd_amd import hip_ops
    S, block = 2048, 32
    c = Cache(1, S, 1, Dh, block, seed=8).finite()
    c.t[0].view(torch.uint8)[:, low] = 0xfe                 # -448, times 2^119
    c.t[2][:, low.start // block:low.stop // block] = 2.0 ** 119
    k, v = (x[0, :, 0] for x in c.values())
    q = torch.rand(1, G, Dh, generator=torch.Generator().manual_seed(3)).add(0.5).to(dt)
    keep = torch.ones(S, dtype=torch.bool)
    keep[low] = False
    n = torch.tensor([S], dtype=torch.int32, device="cuda")
    for nsplit in (1, 3, 16, None):
        out = hip_ops.attn_decode_kv8(q.cuda(), *c.t, n, block=block, nsplit=nsplit)
        for h in range(G):
            want, room = R.attend(q[0, h].double(), k[keep], v[keep], Dh ** -0.5, TWO_PARTS, TWO_PARTS)
            _close(out[0, h], want, room, dt, f"{low} in {nsplit} ranges")


@pytest.mark.parametrize("first,last", [(0, 32), (0, 128), (512, 1024), (1990, 2048), (3, 4)])
def test_keys_that_are_nan(first, last):
    from flashsvd_amd import hip_ops
    S, Dh = 2048, 128
    c = Cache(1, S, 1, Dh, 16, seed=8).finite()
    c.t[0].view(torch.uint8)[:, first:last, 0, 5] = 0x7f
    q = torch.ones(1, 4, Dh, dtype=torch.bfloat16, device="cuda")
    n = torch.tensor([S], dtype=torch.int32, device="cuda")
    for nsplit in (None, 1, 3, 16):
        assert bool(hip_ops.attn_decode_kv8(q, *c.t, n, block=16, nsplit=nsplit).isnan().all())
