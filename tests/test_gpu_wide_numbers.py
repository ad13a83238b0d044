"""Numbers of a call that 32 bits do not hold: they are what they say or are refused, and never what is left of them in 32 bits."""
import pytest
import torch

from tests import kv8_reference as R
from tests.test_gpu_kv8 import Cache
from tests.test_gpu_sample import _draw

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("top_k,kept", [(2 ** 32 + 1, 0), (10 ** 12, 0), (2 ** 31, 0), (-2 ** 32 + 2, 0), (-1, 0), (2 ** 31 - 1, 0), (300, 0), (299, 299)])
def test_top_k_of_any_size(top_k, kept):
    x = torch.randn(9, 300, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    u = torch.linspace(0, 0.999, 9)
    got = _draw(x.cuda(), u.cuda(), top_k=top_k)
    assert got == [R.draw(x[b], float(u[b]), 1.0, kept, 1.0, 0.0) for b in range(9)]


def test_ranges_and_keys_of_any_number():
    from flashsvd_amd import hip_ops
    c = Cache(1, 600, 1, 64, 16, seed=3).finite()
    q = torch.randn(1, 2, 64, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
    n = torch.tensor([7], dtype=torch.int32, device="cuda")
    call = lambda **kw: hip_ops.attn_decode_kv8(q, *c.t, n, block=16, **kw)      # noqa: E731
    assert torch.equal(call(nsplit=2 ** 32 + 1), call(nsplit=600)) and torch.equal(call(nsplit=-2 ** 32 + 3), call())
    assert torch.equal(call(seqlen_add=2 ** 31 - 1), call(seqlen_add=593)) and not bool(call(seqlen_add=-2 ** 31 + 1).any())
    for add in (2 ** 31, 2 ** 32 + 1, -2 ** 31, -2 ** 40):
        with pytest.raises(ValueError, match="32-bit"):
            call(seqlen_add=add)
