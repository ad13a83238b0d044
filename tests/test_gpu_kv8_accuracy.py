"""How few bits the attention over the KV cache in 8 bits may lose (csrc/kv8_attn.hip): weights and a q that the call rotates go into the 16-bit products as
two parts, so what a 16-bit rounding of either would leave is over the bounds here.  Inputs are made so that such roundings add up instead of averaging out."""
import math

import pytest
import torch

from tests import kv8_reference as R
from tests.test_gpu_kv8 import F8, _close, half_step, tables

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


SHARP = 4.0                                              # softmax scale of the cases below


def _against_rounding(x, cos, sin, pos, dt):
    """(key, error of q's elements): codes +-1 that follow the signs of what a 16-bit rounding of x, rotated at pos, leaves of its elements, as many as keep the
    score near 0, and the relative error of an element as two parts: 2^-2p of the rounding, 2^-22 of the rotated pair for the rotation in fp32."""
    y = R.rotate(x.double(), cos, sin, pos)
    left = y.to(dt).double() - y
    part = left.sign() * y                               # of the score
    up, down = ([d for d in part.abs().argsort().tolist() if part[d] * s > 0 and abs(y[d]) > 0.2] for s in (1, -1))
    key, run = torch.zeros_like(y), 0.0
    while up if run <= 0 else down:
        d = (up if run <= 0 else down).pop()
        if abs(run + float(part[d])) <= 1.0:
            key[d], run = left[d].sign(), run + float(part[d])
    pair = x.double().abs()
    pair = pair + pair.roll(len(y) // 2)
    used = key != 0
    error = half_step(dt) ** 2 + 2.0 ** -22 * float((pair[used] / y[used].abs()).max())
    shift, bound = SHARP * float((key * left).sum()), SHARP * float(key.abs() @ y.abs()) * (error + len(y) * 2.0 ** -23)
    assert shift > 3 * bound + 4 * half_step(dt), "the case would not tell one rounding from two"
    return key, error


def _away_from_zero(g, dt, Dh):
    return ((0.5 + torch.rand(Dh, generator=g)) * torch.where(torch.rand(Dh, generator=g) < 0.5, -1.0, 1.0)).to(dt)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Dh", [64, 128])
@pytest.mark.parametrize("form", PROMPTS)
def test_a_rotated_prompt_query_is_two_parts(form, Dh, dt):
    """One key against the roundings of the row that it is made for; its score would be off by the sum of them all."""
    from flashsvd_amd import hip_ops
    p = PROMPTS[form]
    B, Hk, M, past, H = p["B"], p["Hk"], p["M"], p["past"], p["Hk"] * p["G"]
    g = torch.Generator().manual_seed(61)
    cos, sin = tables(past + M, Dh, dt)
    x = _away_from_zero(g, dt, Dh)
    q = x.expand(B, M, H, Dh).contiguous().cuda()
    pos = torch.full((B,), past, dtype=torch.int32, device="cuda")
    for b, m, h in [(0, 5, 0), (B - 1, M - 1, H - 1)]:
        k, v, scale = _held(B, past + M, Hk, Dh, 32)
        hk = h // p["G"]
        key, error = _against_rounding(x, cos, sin, past + m, dt)
        k[b, 3, hk] = key.float()
        v[b, 3, hk] = _varied(Dh)
        out = hip_ops.attn_prefill_kv8(q, k.to(F8).cuda(), v.to(F8).cuda(), scale.cuda(), scale.cuda(), pos, block=32, cos=cos.cuda(), sin=sin.cuda(),
                                       softmax_scale=SHARP).cpu()
        n = past + m + 1
        want, room = R.attend(R.rotate(x.double(), cos, sin, past + m), k[b, :n, hk].double(), v[b, :n, hk].double(), SHARP, error, TWO_PARTS)
        _close(out[b, m, h], want, room, dt, f"{form}: row {m} of head {h}")


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Dh,H,Hk,n", [(64, 8, 8, 137), (128, 8, 2, 900), (128, 4, 4, 30), (64, 40, 2, 200)])
def test_a_rotated_decode_query_is_two_parts(Dh, H, Hk, n, dt):
    from flashsvd_amd import hip_ops
    g = torch.Generator().manual_seed(62)
    cos, sin = tables(n + 1, Dh, dt)
    x = _away_from_zero(g, dt, Dh)
    key, error = _against_rounding(x, cos, sin, n, dt)
    k, v, scale = _held(1, n, Hk, Dh, 32)
    k[0, 3], v[0, 3] = key.float(), _varied(Dh)
    q = x.expand(1, H, Dh).contiguous().cuda()
    out = hip_ops.attn_decode_kv8(q, k.to(F8).cuda(), v.to(F8).cuda(), scale.cuda(), scale.cuda(), torch.tensor([n], dtype=torch.int32, device="cuda"), block=32,
                                  cos=cos.cuda(), sin=sin.cuda(), softmax_scale=SHARP).cpu()
    for h in (0, H - 1):
        want, room = R.attend(R.rotate(x.double(), cos, sin, n), k[0, :, 0].double(), v[0, :, 0].double(), SHARP, error, TWO_PARTS)
        _close(out[0, h], want, room, dt, f"head {h}")


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Dh", [64, 128])
@pytest.mark.parametrize("form", PROMPTS)
def test_scales_that_are_no_power_of_two(form, Dh, dt):
    """value = code * scale for any scale: 0.98 of a half step of bf16 above 1, with powers of two and zeros among the blocks; a value rounded to bf16 would be off
    by nearly 2^-8 of itself."""
    from flashsvd_amd import hip_ops
    p = PROMPTS[form]
    B, Hk, M, past, H = p["B"], p["Hk"], p["M"], p["past"], p["Hk"] * p["G"]
    block = 16
    k, v, scale = _held(B, past + M, Hk, Dh, block)
    k[:, 5::16, :, 0] = -1.0
    v[:, 5::16] = torch.exp2((torch.arange(Dh) % 4).float())
    ks, vs = scale * 1.37, scale * torch.tensor([1 + 0.98 / 256, 1.0, 0.0, 2.0 * (1 + 0.98 / 256)]).repeat(scale.shape[1])[:scale.shape[1], None]
    by = 5 * math.log(2) / 1.37
    q = torch.zeros(B, M, H, Dh, dtype=dt, device="cuda")
    q[..., 0] = 1.0
    out = hip_ops.attn_prefill_kv8(q, k.to(F8).cuda(), v.to(F8).cuda(), ks.cuda(), vs.cuda(), torch.full((B,), past, dtype=torch.int32, device="cuda"),
                                   block=block, softmax_scale=by).cpu()
    b, h = B - 1, H - 1
    full = lambda s: s[b, :, h // p["G"], None].double().repeat_interleave(block, 0)[:past + M]      # noqa: E731
    kk, vv = k[b, :, h // p["G"]].double() * full(ks), v[b, :, h // p["G"]].double() * full(vs)
    for m in range(M):
        want, room = R.attend(q[b, m, h].cpu().double(), kk[:past + m + 1], vv[:past + m + 1], by, 0.0, TWO_PARTS)
        _close(out[b, m, h], want, room, dt, f"{form}: row {m}")
    one = hip_ops.attn_decode_kv8(q[:, M - 1], k.to(F8).cuda(), v.to(F8).cuda(), ks.cuda(), vs.cuda(), torch.full((B,), past + M, dtype=torch.int32, device="cuda"),
                                  block=block, softmax_scale=by).cpu()
    _close(one[b, h], want, room, dt, f"{form}: a token behind it")


@pytest.mark.parametrize("Dh", [64, 128])
@pytest.mark.parametrize("form", PROMPTS)
def test_a_rotation_beyond_the_range_of_float16(form, Dh):
    """Pairs of elements near the end of float16 turn to elements of up to 92600, which the first part of q does not hold (65504); the remainder, at most 27100, is
    rounded by 2^-11 of itself, 2^-12.2 of the element."""
    from flashsvd_amd import hip_ops
    p = PROMPTS[form]
    B, Hk, M, past, H = p["B"], p["Hk"], p["M"], p["past"], p["Hk"] * p["G"]
    g = torch.Generator().manual_seed(63)
    cos, sin = tables(past + M, Dh, torch.float16)
    x = (_away_from_zero(g, torch.float16, Dh).sign() * (65504 - 2000 * torch.rand(Dh, generator=g))).half()
    k, v, scale = _held(B, past + M, Hk, Dh, 32)
    k[:] = torch.randn(past + M, Hk, Dh, generator=g).to(F8).float()
    v[:] = torch.randn(past + M, Hk, Dh, generator=g).to(F8).float()
    kw = dict(block=32, cos=cos.cuda(), sin=sin.cuda(), softmax_scale=1e-6)
    c = [k.to(F8).cuda(), v.to(F8).cuda(), scale.cuda(), scale.cuda()]
    pos = torch.full((B,), past, dtype=torch.int32, device="cuda")
    out = hip_ops.attn_prefill_kv8(x.expand(B, M, H, Dh).contiguous().cuda(), *c, pos, **kw).cpu()
    one = hip_ops.attn_decode_kv8(x.expand(B, H, Dh).contiguous().cuda(), *c, pos + M - 1, seqlen_add=1, **kw).cpu()
    beyond = 0
    for b, m, h in [(0, 0, 0), (B - 1, M - 1, H - 1), (B // 2, M // 2, 0)]:
        y, n, hk = R.rotate(x.double(), cos, sin, past + m), past + m + 1, h // p["G"]
        beyond += int((y.abs() > 65520).sum())
        want, room = R.attend(y, k[b, :n, hk].double(), v[b, :n, hk].double(), 1e-6, 2.0 ** -12.2, TWO_PARTS)
        _close(out[b, m, h], want, room, torch.float16, f"{form}: row {m} of head {h}")
        if m == M - 1:
            _close(one[b, h], want, room, torch.float16, f"{form}: one token")
    assert beyond
