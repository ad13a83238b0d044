"""FlashSVDKV4Cache.update with positions on the GPU: the held length is that of the largest position, as with positions on the host."""
from types import SimpleNamespace

import pytest
import torch

from tests import kv4_reference as R

pytestmark = pytest.mark.gpu
CFG = SimpleNamespace(num_hidden_layers=2, rope_theta=10000.0)


@pytest.mark.parametrize("device", ["cpu", "cuda"])
def test_updates_in_any_order(device):
    from flashsvd_amd.runtime import FlashSVDKV4Cache
    c = FlashSVDKV4Cache(CFG, max_batch_size=2, max_cache_len=70, device="cuda", dtype=torch.bfloat16)
    g = torch.Generator().manual_seed(8)
    k, v = (torch.randn(2, 2, 7, 64, generator=g).to(torch.bfloat16) for _ in range(2))
    held = torch.zeros(2, 2, 70, 64, dtype=torch.double)
    for at, n in (([0, 1, 2, 3, 4, 5, 6], 7), ([5], 7), ([3, 2], 7), ([7, 39, 5], 40), ([39, 39], 40), ([69, 0], 70), ([], 70)):
        rows = [x[:, :, :len(at)].contiguous() for x in (k, v)]
        K, V = c.update(*(x.cuda() for x in rows), 0, {"cache_position": torch.tensor(at, dtype=torch.long, device=device)})
        for t, p in enumerate(at):
            for b in range(2):
                for h in range(2):
                    held[b, h, p] = torch.cat([R.group_values(r)[1] for r in rows[0][b, h, t].double().view(2, 32)])
        assert c.get_seq_length() == n and K.shape == V.shape == (2, 2, n, 64)
        assert torch.equal(K.cpu().double(), held[:, :, :n])
    K, V = c.update(k[:, :, :2].cuda(), v[:, :, :2].cuda(), 1, {"cache_position": torch.tensor([4, 5], device=device)})      # layer 0 counts
    assert K.shape == (2, 2, 70, 64) and c.get_seq_length() == 70
