"""How few bits the attention over the KV cache in 8 bits may lose (csrc/kv8_attn.hip): the weights go into the 16-bit products as two parts, so what one
16-bit rounding of them would leave is over the bounds here.  Inputs are made so that such roundings add up instead of averaging out."""
import math

import pytest
import torch

from tests import kv8_reference as R
from tests.test_gpu_kv8 import F8, _close

pytestmark = pytest.mark.gpu

# shapes on the far side of each threshold of the prompt kernel's forms, and one whose keys are cut into ranges
PROMPTS = {
    "128 rows": dict(B=8, Hk=32, G=1, M=130, past=7),
    "128 rows of two heads": dict(B=16, Hk=16, G=2, M=70, past=40),
    "64 rows": dict(B=8, Hk=25, G=1, M=70, past=33),
    "64 rows in halves": dict(B=2, Hk=2, G=2, M=40, past=90),
    "64 rows in halves and ranges": dict(B=1, Hk=2, G=3, M=21, past=1200),
}
TWO_PARTS = 2.0 ** -16                                   # of two bf16 parts: the second is rounded by at most 2^-8 of the at most 2^-8 that the first leaves


def _held(B, S, Hk, Dh, block):
    """Codes and scales of one, to be filled; codes as floats."""
    k, v = torch.zeros(B, S, Hk, Dh), torch.zeros(B, S, Hk, Dh)
    scale = torch.ones(B, -(-S // block), Hk)
    return k, v, scale


def _varied(Dh):
    """Codes whose multiples fall everywhere between two numbers of a 16-bit type."""
    return (1 + (torch.arange(Dh) % 8) / 8) * torch.exp2((torch.arange(Dh) // 8 % 4).float())


def _weights_case(B, S, Hk, Dh, block=32):
    """Keys of score 0 with values 0, and one of sixteen with weight w = 0.98 of a half step of bf16 over 2^-5: the output is c n w / (m + n w), off by nearly
    2^-8 of itself if w is rounded to bf16."""
    k, v, scale = _held(B, S, Hk, Dh, block)
    k[:, 5::16, :, 0] = -1.0
    v[:, 5::16] = _varied(Dh)
    return k, v, scale, -math.log((1 + 0.98 / 256) * 2.0 ** -5)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Dh", [64, 128])
@pytest.mark.parametrize("form", PROMPTS)
def test_prompt_weights_are_two_parts(form, Dh, dt):
    from flashsvd_amd import hip_ops
    p = PROMPTS[form]
    B, Hk, M, past, H = p["B"], p["Hk"], p["M"], p["past"], p["Hk"] * p["G"]
    k, v, scale, by = _weights_case(B, past + M, Hk, Dh)
    q = torch.zeros(B, M, H, Dh, dtype=dt, device="cuda")
    q[..., 0] = 1.0
    pos = torch.full((B,), past, dtype=torch.int32, device="cuda")
    out = hip_ops.attn_prefill_kv8(q, k.to(F8).cuda(), v.to(F8).cuda(), scale.cuda(), scale.cuda(), pos, block=32, softmax_scale=by).cpu()
    for b, m, h in [(0, 0, 0), (0, M - 1, H - 1), (B - 1, 13, 0), (B - 1, M // 2, H // 2), (B // 2, M - 2, 1)]:
        n, hk = past + m + 1, h // p["G"]
        want, room = R.attend(q[b, m, h].cpu().double(), k[b, :n, hk].double(), v[b, :n, hk].double(), by, 0.0, TWO_PARTS)
        _close(out[b, m, h], want, room, dt, f"{form}: row {m} of head {h}")


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Dh,H,Hk,lens", [(64, 8, 8, [137, 40]), (128, 8, 2, [900, 77]), (128, 40, 2, [200])])
def test_decode_weights_are_two_parts(Dh, H, Hk, lens, dt):
    from flashsvd_amd import hip_ops
    B, S = len(lens), max(lens)
    k, v, scale, by = _weights_case(B, S, Hk, Dh)
    q = torch.zeros(B, H, Dh, dtype=dt, device="cuda")
    q[..., 0] = 1.0
    for nsplit in (None, 1, 3):
        out = hip_ops.attn_decode_kv8(q, k.to(F8).cuda(), v.to(F8).cuda(), scale.cuda(), scale.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"),
                                      block=32, softmax_scale=by, nsplit=nsplit).cpu()
        for b, n in enumerate(lens):
            for h in (0, H - 1):
                hk = h // (H // Hk)
                want, room = R.attend(q[b, h].cpu().double(), k[b, :n, hk].double(), v[b, :n, hk].double(), by, 0.0, TWO_PARTS)
                _close(out[b, h], want, room, dt, f"{n} keys, head {h}, in {nsplit}")
