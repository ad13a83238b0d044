"""Key ranges far below the others: a weight that 32 bits do not hold is nothing of a number, however large, in how many ranges the keys ever stand."""
import pytest
import torch

from tests import kv4_reference as R4
from tests import kv8_reference as R8
from tests.test_gpu_kv4 import HALF_PART, TWO_PARTS, Cache, _close
from tests.test_gpu_kv8 import Cache as Cache8
from tests.util import form_taken

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn


def _far_below(S, Dh, far):
    """A cache in 4 bits and its rows without the range `far`: keys of 48, which a query of ones scores 384 or 543, and values of 0; in the range keys of 0, e^-384 of
    the others' weight (2^119 * 2^-554 is no number of 32 bits), and values of 6 * 2^116, up to a thousand of which fp32 sums."""
    c = Cache(1, S, 1, Dh, seed=8)
    c.t[0].fill_(0x77)
    c.t[2].fill_(130)
    c.t[1].zero_()
    c.t[0][:, far] = 0
    c.t[1][:, far] = 0x77
    c.t[3][..., far] = 243
    keep = torch.ones(S, dtype=torch.bool)
    keep[far] = False
    return c, *(x[0, :, 0] for x in c.values()), keep


@pytest.mark.parametrize("Dh", [64, 128])
@pytest.mark.parametrize("S,splits", [(2048, (1, 2, 3, 8, None)), (16896, (1, 8, 33, 66, None))])
def test_decode_over_4_bits(S, splits, Dh):
    from flashsvd_amd import hip_ops
    dt = torch.bfloat16
    q = torch.ones(1, 4, Dh, dtype=dt, device="cuda")
    n = torch.tensor([S], dtype=torch.int32, device="cuda")
    for far in (slice(0, 256), slice(512, 1024), slice(S - 256, S)):
        c, k, v, keep = _far_below(S, Dh, far)
        want, room = R4.attend(torch.ones(Dh, dtype=torch.double), k[keep], v[keep], Dh ** -0.5, TWO_PARTS, TWO_PARTS)
        for nsplit in splits:
            out = hip_ops.attn_decode_kv4(q, *c.t, n, nsplit=nsplit)
            for h in range(4):
                _close(out[0, h], want, room, dt, f"{far} in {nsplit} ranges")


@pytest.mark.parametrize("Dh", [64, 128])
@pytest.mark.parametrize("M,Hk,G,name", [(9, 1, 2, "kv4 prompt 64 halves ranges"), (300, 8, 4, "kv4 prompt 128 ranges")])
def test_prompts_over_4_bits(M, Hk, G, name, Dh):
    from flashsvd_amd import hip_ops
    S, dt, H = 4800, torch.bfloat16, Hk * G
    c, k, v, keep = _far_below(S, Dh, slice(1600, 2560))
    held = [t.repeat_interleave(Hk, 2 if i < 2 else 1) for i, t in enumerate(c.t)]
    q = torch.ones(1, M, H, Dh, dtype=dt, device="cuda")
    out = hip_ops.attn_prefill_kv4(q, *held, torch.tensor([S - M], dtype=torch.int32, device="cuda"))
    assert form_taken() == name
    for m in (0, M // 2, M - 1):
        sees = keep & (torch.arange(S) <= S - M + m)
        want, room = R4.attend(torch.ones(Dh, dtype=torch.double), k[sees], v[sees], Dh ** -0.5, TWO_PARTS, HALF_PART)
        for h in (0, H - 1):
            _close(out[0, m, h], want, room, dt, f"row {m} head {h}")


@pytest.mark.parametrize("Dh", [64, 128])
def test_decode_over_8_bits(Dh):
    """The same of the cache in 8 bits, values of 448 and a scale of 2^109 beside zeros."""
    from flashsvd_amd import hip_ops
    S, block, dt = 2048, 32, torch.bfloat16
    c = Cache8(1, S, 1, Dh, block, seed=5).finite()
    far = slice(512, 1024)
    ones = torch.ones(1, S, 1, Dh, device="cuda")
    c.t[0].copy_((48 * ones).to(F8))
    c.t[0][:, far].copy_((0 * ones[:, far]).to(F8))
    c.t[1].copy_((0 * ones).to(F8))
    c.t[1][:, far].copy_((448 * ones[:, far]).to(F8))
    c.t[2].fill_(1.0)
    c.t[3].fill_(2.0 ** 109)
    k, v = (x[0, :, 0] for x in c.values())
    q = torch.ones(1, 4, Dh, dtype=dt, device="cuda")
    n = torch.tensor([S], dtype=torch.int32, device="cuda")
    keep = torch.ones(S, dtype=torch.bool)
    keep[far] = False
    want, room = R8.attend(torch.ones(Dh, dtype=torch.double), k[keep], v[keep], Dh ** -0.5, TWO_PARTS, TWO_PARTS)
    for nsplit in (1, 2, 4, 16, None):
        out = hip_ops.attn_decode_kv8(q, *c.t, n, block=block, nsplit=nsplit)
        for h in range(4):
            _close(out[0, h], want, room, dt, f"{nsplit} ranges")


def test_a_nan_in_a_range_that_weighs_nothing():
    """It reaches the output in its group of channels, beside ranges without keys."""
    from flashsvd_amd import hip_ops
    S, Dh = 2048, 128
    q = torch.ones(1, 4, Dh, dtype=torch.bfloat16, device="cuda")
    for room in (S, 4096):
        c, *_ = _far_below(room, Dh, slice(512, 1024))
        c.t[3][:, :, 2, 700] = 255
        for t in c.t[2:]:
            t[..., S:] = 255                                # what no query sees
        n = torch.tensor([S], dtype=torch.int32, device="cuda")
        for nsplit in (1, 2, 8, 16, None):
            nan = hip_ops.attn_decode_kv4(q, *c.t, n, nsplit=nsplit).isnan()
            assert bool(nan[..., 64:96].all()) and not bool(nan[..., :64].any()) and not bool(nan[..., 96:].any())
