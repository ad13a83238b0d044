"""Groups of zeros among the values of long chunks: float16 holds them whatever their scale, so they change no rounding of what stands beside them."""
import pytest
import torch

from tests.test_gpu_kv4 import Cache, _check_rows
from tests.util import form_taken

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("Dh", [64, 128])
@pytest.mark.parametrize("byte", [0, 2, 90, 141, 252])
@pytest.mark.parametrize("where", [slice(0, 1), slice(5, 70), slice(300, 301), slice(899, 900)])
def test_zeros_of_any_scale_are_alike(where, byte, Dh):
    """Byte 2 is what an append writes for zeros, 0 what a new cache holds.  The output is that of the same zeros with a scale of 1, bit for bit."""
    from flashsvd_amd import hip_ops
    B, Hk, H, M, past, dt = 8, 16, 32, 300, 600, torch.bfloat16
    g = torch.Generator().manual_seed(72)
    q = (torch.randn(B, M, H, Dh, generator=g) * 0.7).to(dt)
    pos = torch.full((B,), past, dtype=torch.int32, device="cuda")
    outs = []
    for scale in (127, byte):
        c = Cache(B, past + M, Hk, Dh, seed=9)
        for b, hk, group in ((1, 3, 1), (6, slice(None), 0)):
            c.t[1][b, where, hk, 16 * group:16 * group + 16] &= 0x88          # zeros of either sign
            c.t[3][b, hk, group, where] = scale
        outs.append(hip_ops.attn_prefill_kv4(q.cuda(), *c.t, pos).cpu())
        assert form_taken() == "kv4 prompt 128"
    assert torch.equal(*outs)
    picked = [(b, m) for b in (0, 1, 6) for m in (0, 97, 299)]
    _check_rows(c, torch.stack([q[b, m] for b, m in picked]), torch.stack([outs[1][b, m] for b, m in picked]), [(b, past + m + 1) for b, m in picked], Dh ** -0.5, dt,
                what=f"byte {byte}", heads=[6, 7, 31])


@pytest.mark.parametrize("Dh", [64, 128])
def test_one_number_beside_zeros_counts(Dh):
    """A group of one code that is no zero and a scale beyond float16, the first or the last of its tile or of its sixteen tokens, among groups of zeros."""
    from flashsvd_amd import hip_ops
    B, Hk, H, M, past, dt = 8, 16, 32, 300, 600, torch.bfloat16
    g = torch.Generator().manual_seed(73)
    q = (torch.randn(B, M, H, Dh, generator=g) * 0.7).to(dt)
    for n in (64, 79, 80, 127, 640, 895):
        for byte in (1, 252):
            c = Cache(B, past + M, Hk, Dh, seed=9)
            c.t[1][:, n // 16 * 16:n // 16 * 16 + 16, :, :16] = 0
            c.t[3][:, :, 0, n // 16 * 16:n // 16 * 16 + 16] = 2
            c.t[1][:, n, :, 15], c.t[3][:, :, 0, n] = 0x70, byte
            out = hip_ops.attn_prefill_kv4(q.cuda(), *c.t, torch.full((B,), past, dtype=torch.int32, device="cuda")).cpu()
            picked = [(1, 0), (6, 40), (7, 299)]
            _check_rows(c, torch.stack([q[b, m] for b, m in picked]), torch.stack([out[b, m] for b, m in picked]), [(b, past + m + 1) for b, m in picked], Dh ** -0.5, dt,
                        what=f"{byte} at {n}", heads=[0, 31])
