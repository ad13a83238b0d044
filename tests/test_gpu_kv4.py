"""The KV cache in 4 bits (csrc/kv4.hip, csrc/kv4_attn.hip) against its definition in 64 bits: what an append leaves in the cache, attention of single
tokens and of chunks over it, and all of them together as a decode loop uses them, captured and not."""
import math

import pytest
import torch

from tests import kv4_reference as R
from tests.test_gpu_kv8 import _same, half_step, tables
from tests.util import form_taken

pytestmark = pytest.mark.gpu


class Cache:
    """Codes and bytes with something in every row, on the GPU; layout "head": a head's rows side by side, "token": a row's heads."""

    def __init__(self, B, S, Hk, Dh, seed, layout="head", zero=False):
        g = torch.Generator().manual_seed(seed)
        room = -(-S // 64) * 64
        order = (B, Hk, room, Dh // 2) if layout == "head" else (B, room, Hk, Dh // 2)
        codes = [torch.randint(0, 256, order, generator=g, dtype=torch.uint8) for _ in range(2)]
        scale = [torch.randint(123, 127, (B, Hk, Dh // 32, room), generator=g, dtype=torch.uint8) for _ in range(2)]
        if zero:
            codes, scale = [c * 0 for c in codes], [s * 0 for s in scale]
        self.t = [*(c.cuda().transpose(1, 2) if layout == "head" else c.cuda() for c in codes), *(s.cuda() for s in scale)]

    def values(self):
        return R.unpack(self.t[0], self.t[2]), R.unpack(self.t[1], self.t[3])

    def spoil(self, lens):
        """A NaN for every group of rows that no query may see."""
        for b, n in enumerate(lens):
            for t in self.t[2:]:
                t[b, :, :, max(n, 0):] = 255


TWO_PARTS = 2.0 ** -16                                   # of two bf16 parts: the second is rounded by at most 2^-8 of the at most 2^-8 that the first leaves
HALF_PART = 2.0 ** -11                                   # of one float16: half a step


def _close(got, want, room, dt, what):
    """Within `room` before the last rounding, of half a step: 2^-p of the value, and below the smallest normal number, where steps stay the same (2^-24 in
    float16), half of such a step.  A code of zero for the key that has nearly all the weight leaves outputs as small as that."""
    got = got.double().cpu()
    assert bool(torch.isfinite(got).all()), what
    step = torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    over = (got - want).abs() - (want.abs() * half_step(dt) + step / 2 + room * (1 + half_step(dt)) + 1e-30)
    assert float(over.max()) <= 0, f"{what}: {float(over.max()):.3g} over the bound"


def _check_rows(c, q, out, lens, scale, dt, cos=None, sin=None, pos=None, what="", heads=None):
    """q, out [rows, H, Dh] of rows (sequence b, keys n, position): one query each.  A q that the call rotates and the weights are two parts of 8 bits at least,
    and the rotation in fp32 leaves 2^-22 of the rotated pair.  The weights of long chunks in bf16 are one float16, smallest number 2^-24 where the largest weight is
    2^7 at least: they lose 2^-32 of the largest."""
    one = dt == torch.bfloat16 and form_taken().startswith("kv4 prompt 128")
    k, v = c.values()
    H, Hk = q.shape[1], k.shape[2]
    for i, (b, n) in enumerate(lens):
        for h in range(H) if heads is None else heads:
            x = q[i, h].double()
            y = R.rotate(x, cos, sin, pos[i] if pos else 0)
            hk = h // (H // Hk)
            kk = k[b, :n, hk]
            pair = x.abs() + x.abs().roll(len(x) // 2)
            turned = 2.0 ** -22 * float(((kk.abs() @ pair) / (kk.abs() @ y.abs()).clamp_min(1e-30)).max()) if cos is not None and n else 0.0
            want, room = R.attend(y, kk, v[b, :n, hk], scale, TWO_PARTS + turned, HALF_PART if one else TWO_PARTS)
            if one and n:
                room = room + n * 2.0 ** -32 * v[b, :n, hk].abs().amax(0)
            _close(out[i, h], want, room, dt, f"{what} row {i} head {h} of {n} keys")


# ------------------------------------------------------------------ append
APPENDS = [
    (128, 2, "head", 1, [0, 5, 15, 63, 47], None),
    (64, 3, "token", 1, [0, 31, 32, 46, 7], None),
    (128, 1, "head", 7, [0, 3, 30, 25, 41], None),
    (64, 2, "head", 33, [0, 1, 15, 31, 7], [33, 0, 1, 17, 32]),
    (128, 2, "token", 40, [0, 8, 5, 1, 3], [40, 40, 0, 3, 39]),
    (128, 1, "head", 65, [0, 60, 1, 127, 64], [65, 1, 64, 65, 63]),
    # outside the cache: dropped in front of it and behind it
    (64, 2, "head", 5, [-3, 126, 128, 300, -9], None),
]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("turn", [False, True])
@pytest.mark.parametrize("Dh,Hk,layout,T,at,rows", APPENDS)
def test_append_holds_what_the_definition_says(dt, turn, Dh, Hk, layout, T, at, rows):
    """Codes go by the exact rotated value, so values and bytes are equal, rotated or not; every other row is as it was."""
    from flashsvd_amd import hip_ops
    B, S = len(at), 128
    c = Cache(B, S, Hk, Dh, seed=T + Dh, layout=layout)
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(B, T, Hk, Dh, generator=g) * torch.exp2(torch.randint(-3, 3, (B, T, Hk, 1), generator=g).float())).to(dt), torch.randn(B, T, Hk, Dh, generator=g).to(dt)
    k[..., ::7] = (k[..., ::7].float() * 4).round().to(dt) / 4       # ties among them
    cos, sin = tables(S - 3, Dh, dt) if turn else (None, None)       # the last positions take the last row of the tables
    values, bytes_ = c.values(), [t.cpu().clone() for t in c.t[2:]]
    for b in range(B):
        n = T if rows is None else rows[b]
        R.append(values[0][b], bytes_[0][b], k[b], at[b], n, cos, sin)
        R.append(values[1][b], bytes_[1][b], v[b], at[b], n)
    wide = torch.zeros(B, T, Hk, 2 * Dh + 1, dtype=dt, device="cuda")               # rows inside longer ones, at odd elements
    wide[..., :Dh], wide[..., Dh + 1:] = k.cuda(), v.cuda()
    hip_ops.kv4_append(wide[..., :Dh], wide[..., Dh + 1:], *c.t, torch.tensor(at, dtype=torch.int32, device="cuda"), cos=cos.cuda() if turn else None,
                       sin=sin.cuda() if turn else None, rows=None if rows is None else torch.tensor(rows, dtype=torch.int32, device="cuda"))
    for got, want, name in zip((*c.values(), *(t.cpu() for t in c.t[2:])), (*values, *bytes_), ("k", "v", "k_scale", "v_scale")):
        assert _same(got, want) if got.is_floating_point() else torch.equal(got, want), f"{name}: {int((got != want).sum())} of {got.numel()} differ"


@pytest.mark.parametrize("T", [1, 9])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_append_at_the_ends_of_the_numbers(dt, T):
    """Zeros, the smallest and the largest numbers of the type, infinities and NaN, and groups at the borders between two exponents."""
    from flashsvd_amd import hip_ops
    Dh, Hk, S = 64, 1, 64
    big, small = float(torch.finfo(dt).max), float(torch.finfo(dt).smallest_normal)
    g = torch.Generator().manual_seed(8)
    rows = []
    for size in (0.0, small, small / 64, 1e-3, 6.0, 7.0, 7.0 * (1 + 2 * half_step(dt)), 1.75, 14.0, big, big / 2, math.inf, math.nan):
        row = torch.rand(Hk, Dh, generator=g) * (size if math.isfinite(size) else 1.0)
        row[..., 5], row[..., 40] = -size, size
        rows.append(row.to(dt))
    rows = torch.stack(rows)
    c = Cache(1, S, Hk, Dh, seed=9, zero=True)
    values, bytes_ = c.values(), [t.cpu().clone() for t in c.t[2:]]
    R.append(values[0][0], bytes_[0][0], rows, 0, len(rows))
    R.append(values[1][0], bytes_[1][0], -rows, 0, len(rows))
    for i in range(0, len(rows), T):
        x = rows[None, i:i + T].cuda()
        hip_ops.kv4_append(x, -x, *c.t, torch.tensor([i], dtype=torch.int32, device="cuda"))
    for got, want in zip((*c.values(), *(t.cpu() for t in c.t[2:])), (*values, *bytes_)):
        assert _same(got, want) if got.is_floating_point() else torch.equal(got, want)


@pytest.mark.parametrize("T", [1, 5])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_rotated_keys_at_the_ends_of_the_numbers(dt, T):
    """A rotated pair of the largest bf16 numbers is beyond 32 bits and still a number that decides the scale; infinities of the input do not."""
    from flashsvd_amd import hip_ops
    Dh, S = 64, 64
    big = float(torch.finfo(dt).max)
    cos, sin = tables(S, Dh, dt)
    g = torch.Generator().manual_seed(12)
    k = torch.rand(1, 20, 1, Dh, generator=g).sub(0.5).to(dt)
    for t in range(20):                                              # channels 3 and 35 are a pair, 9 and 41 too
        k[0, t, 0, 3], k[0, t, 0, 35] = big * (-1) ** (t // 2), big * (-1) ** t
        if t % 5 == 4:
            k[0, t, 0, 9], k[0, t, 0, 41] = (math.inf, 0.5) if t % 2 else (1.0, -math.inf)
    c = Cache(1, S, 1, Dh, seed=9, zero=True)
    values, bytes_ = c.values(), [t.cpu().clone() for t in c.t[2:]]
    R.append(values[0][0], bytes_[0][0], k[0], 3, 20, cos, sin)
    R.append(values[1][0], bytes_[1][0], k[0], 3, 20)
    for i in range(0, 20, T):
        hip_ops.kv4_append(k[:, i:i + T].cuda(), k[:, i:i + T].cuda(), *c.t, torch.tensor([3 + i], dtype=torch.int32, device="cuda"), cos=cos.cuda(), sin=sin.cuda())
    for got, want in zip((*c.values(), *(t.cpu() for t in c.t[2:])), (*values, *bytes_)):
        assert _same(got, want) if got.is_floating_point() else torch.equal(got, want)


def test_appends_row_by_row_and_at_once_are_alike():
    from flashsvd_amd import hip_ops
    B, T, Hk, Dh, S = 2, 70, 2, 128, 128
    dt = torch.bfloat16
    g = torch.Generator().manual_seed(4)
    k, v = (torch.randn(B, T, Hk, Dh, generator=g).to(dt).cuda() for _ in range(2))
    cos, sin = (t.cuda() for t in tables(S, Dh, dt))
    a, b = (Cache(B, S, Hk, Dh, seed=1) for _ in range(2))
    at = lambda n: torch.tensor([n, n + 9], dtype=torch.int32, device="cuda")      # noqa: E731
    hip_ops.kv4_append(k, v, *a.t, at(3), cos=cos, sin=sin)
    for t in range(T):
        hip_ops.kv4_append(k[:, t:t + 1], v[:, t:t + 1], *b.t, at(3 + t), cos=cos, sin=sin)
    assert all(torch.equal(x, y) for x, y in zip(a.t, b.t))


# ------------------------------------------------------------------ reading it back
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Dh,Hk,layout,B,S,length", [(128, 2, "head", 3, 128, None), (64, 3, "token", 2, 64, 37), (128, 1, "token", 1, 192, 1), (64, 1, "head", 5, 64, 0)])
def test_what_the_cache_holds(dt, Dh, Hk, layout, B, S, length):
    from flashsvd_amd import hip_ops
    c = Cache(B, S, Hk, Dh, seed=5, layout=layout)
    c.t[2][0, 0, 0, 0], c.t[3][-1, -1, -1, :5] = 255, torch.tensor([0, 1, 140, 255, 100], dtype=torch.uint8)
    L = S if length is None else length
    for got, want in zip(hip_ops.kv4_dequantize(*c.t, length=length, dtype=dt), c.values()):
        assert got.shape == (B, L, Hk, Dh) and got.dtype == dt
        want = want[:, :L].to(dt)
        assert _same(got.cpu().double(), want.double())


def test_the_largest_exponents_read_as_bf16():
    """Every byte from 1 to 252 with every code is exact in bf16."""
    from flashsvd_amd import hip_ops
    c = Cache(1, 256, 1, 64, seed=6)
    c.t[0][0, :, 0] = torch.arange(32, dtype=torch.uint8, device="cuda") * 8 + 3
    c.t[2][0, 0] = torch.arange(256, device="cuda").to(torch.uint8)
    k, _ = hip_ops.kv4_dequantize(*c.t)
    want = c.values()[0]
    assert torch.equal(k[:, 1:253].cpu().double(), want[:, 1:253])
    assert bool(k[:, 255].isnan().all())


# ------------------------------------------------------------------ attention
DECODES = [
    (128, 4, 4, "head", [1, 33, 0, 70], 96),
    (128, 8, 2, "token", [95, 16, 17, 15], 96),
    (64, 8, 8, "head", [137], 160),
    (64, 6, 2, "head", [64, 65, 129], 130),
    (128, 5, 1, "token", [127, 128, 129, 200], 200),
    (128, 7, 1, "head", [31], 40),
    (64, 16, 1, "head", [100, 1], 112),
    (64, 40, 2, "head", [61], 64),
    (128, 34, 2, "token", [300, 7], 301),
    (128, 2, 2, "head", [1500, 3, 700], 1501),
    (128, 8, 1, "head", [4097], 4100),
    (64, 20, 1, "head", [900, 0, 513], 1000),              # more than 16 heads of a kv head over key ranges
    (128, 1, 1, "head", [500, 0, -4, 9999], 256),          # a negative length, and one beyond the cache
]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Dh,H,Hk,layout,lens,S", DECODES)
def test_decode_attention(dt, Dh, H, Hk, layout, lens, S):
    from flashsvd_amd import hip_ops
    B = len(lens)
    c = Cache(B + 1, S, Hk, Dh, seed=S + H, layout=layout)
    room = c.t[0].shape[1]
    keys = [min(max(n, 0), room) for n in lens]
    c.spoil(keys)
    g = torch.Generator().manual_seed(7)
    q = (torch.randn(B, H, Dh, generator=g) * 0.7).to(dt)
    wide = torch.zeros(B, H + 1, Dh + 8, dtype=dt, device="cuda")
    wide[:, :H, :Dh] = q.cuda()
    n32 = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = hip_ops.attn_decode_kv4(wide[:, :H, :Dh], *c.t, n32)
    _check_rows(c, q, out, list(enumerate(keys)), Dh ** -0.5, dt, what="decode")
    for nsplit in (1, 3, 7, 64):                          # any cut of the keys is within the same bound; `out` inside longer rows
        into = torch.full((B, H + 2, Dh + 4), 7.0, dtype=dt, device="cuda")
        hip_ops.attn_decode_kv4(wide[:, :H, :Dh], *c.t, n32, nsplit=nsplit, out=into[:, 1:H + 1, :Dh], softmax_scale=0.2)
        _check_rows(c, q, into[:, 1:H + 1, :Dh], list(enumerate(keys)), 0.2, dt, what=f"decode in {nsplit}")
        assert bool((into[:, 0] == 7).all() and (into[:, H + 1] == 7).all() and (into[:, :, Dh:] == 7).all())


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Dh,H,Hk,at,S", [
    (128, 8, 2, [0, 5, 31, 32, 100], 128),
    (64, 8, 8, [137, 0], 144),
    (128, 4, 4, [63, 64, 699], 700),
    (64, 9, 1, [130, 127, 128, 50, 40, 1], 200),
    (64, 20, 1, [900, 0, 513], 1000),
    (128, 4, 2, [127, 128, 383, 384, 511, 1151], 1152),      # a new row at the ends of ranges
    (128, 4, 1, [64, -1, 256, 255], 256),                    # two of the rows outside the cache: dropped
])
def test_decode_attention_appends_its_token(dt, Dh, H, Hk, at, S):
    """The call against an append of its own followed by attention: the same cache, bit for bit, and the output within the bound over it."""
    from flashsvd_amd import hip_ops
    B = len(at)
    cos, sin = tables(S, Dh, dt)
    c, other = (Cache(B, S, Hk, Dh, seed=11) for _ in range(2))
    room = c.t[0].shape[1]
    g = torch.Generator().manual_seed(12)
    q, k, v = ((torch.randn(B, h, Dh, generator=g) * f).to(dt) for h, f in ((H, 0.7), (Hk, 20.0), (Hk, 1.0)))
    pos = torch.tensor(at, dtype=torch.int32, device="cuda")
    kw = dict(cos=cos.cuda(), sin=sin.cuda())
    out = hip_ops.attn_decode_kv4(q.cuda(), *c.t, pos, k_new=k.cuda(), v_new=v.cuda(), **kw)
    hip_ops.kv4_append(k.cuda()[:, None], v.cuda()[:, None], *other.t, pos, **kw)
    assert all(torch.equal(x, y) for x, y in zip(c.t, other.t))
    seen = [(b, min(n + 1, room)) for b, n in enumerate(at)]
    _check_rows(c, q, out, seen, Dh ** -0.5, dt, cos, sin, at, "append and decode")
    again = hip_ops.attn_decode_kv4(q.cuda(), *other.t, pos, seqlen_add=1, **kw)
    _check_rows(other, q, again, seen, Dh ** -0.5, dt, cos, sin, at, "decode behind an append")


PROMPTS = [
    (128, 4, 4, "head", 1, [0, 40], None),
    (128, 4, 2, "token", 17, [0, 5, 100], [17, 0, 9]),
    (64, 8, 2, "head", 33, [0, 31], None),
    (64, 2, 2, "head", 130, [0, 3], [130, 65]),
    (128, 6, 1, "head", 77, [211, 0, 64], [77, 1, 76]),
    (128, 1, 1, "token", 150, [0], None),
    (64, 3, 1, "head", 64, [64], None),
    (128, 2, 1, "head", 40, [500, 1], None),
    (128, 4, 2, "head", 9, [900, 3, 650], [9, 9, 0]),      # in ranges of the keys
    (64, 2, 2, "token", 3, [1500], None),
]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Dh,H,Hk,layout,M,start,rows", PROMPTS)
def test_prompt_attention(dt, Dh, H, Hk, layout, M, start, rows):
    from flashsvd_amd import hip_ops
    B = len(start)
    n = rows or [M] * B
    S = max(p + t for p, t in zip(start, n)) + 3
    c = Cache(B, S, Hk, Dh, seed=M + H, layout=layout)
    c.spoil([p + t for p, t in zip(start, n)])
    cos, sin = tables(S, Dh, dt)
    g = torch.Generator().manual_seed(13)
    q = (torch.randn(B, M, H, Dh, generator=g) * 0.7).to(dt)
    p32 = torch.tensor(start, dtype=torch.int32, device="cuda")
    r32 = None if rows is None else torch.tensor(rows, dtype=torch.int32, device="cuda")
    for rope in ((None, None), (cos, sin)):
        into = torch.full((B, M + 1, H, Dh + 4), 7.0, dtype=dt, device="cuda")
        hip_ops.attn_prefill_kv4(q.cuda(), *c.t, p32, rows=r32, cos=None if rope[0] is None else cos.cuda(),
                                 sin=None if rope[0] is None else sin.cuda(), out=into[:, :M, :, :Dh])
        flat = [(b, m) for b in range(B) for m in range(n[b])]
        picked = flat if len(flat) <= 60 else flat[:8] + flat[8:-8:max(1, len(flat) // 40)] + flat[-8:]
        _check_rows(c, torch.stack([q[b, m] for b, m in picked]), torch.stack([into[b, m, :, :Dh].cpu() for b, m in picked]),
                    [(b, start[b] + m + 1) for b, m in picked], Dh ** -0.5, dt, *rope, [start[b] + m for b, m in picked], "prompt")
        for b in range(B):
            assert bool((into[b, n[b]:] == 7).all()), "rows behind the last one"
        assert bool((into[..., Dh:] == 7).all())
    zeros = hip_ops.attn_prefill_kv4(q.cuda(), *c.t, p32, rows=r32)
    assert bool(torch.isfinite(zeros).all())
    for b in range(B):
        assert not bool(zeros[b, n[b]:].any())


@pytest.mark.parametrize("Dh,H,Hk,M,start", [
    (128, 32, 32, 130, [0, 3, 64, 200]),       # 128 rows of a workgroup
    (64, 64, 32, 70, [0, 1, 31, 77]),
    (128, 40, 40, 50, [5, 0, 63, 64]),         # 64 rows, no key ranges
])
def test_prompt_attention_of_many_heads(Dh, H, Hk, M, start):
    from flashsvd_amd import hip_ops
    dt, B = torch.float16, len(start)
    c = Cache(B, max(start) + M, Hk, Dh, seed=M)
    g = torch.Generator().manual_seed(14)
    q = (torch.randn(B, M, H, Dh, generator=g) * 0.7).to(dt)
    out = hip_ops.attn_prefill_kv4(q.cuda(), *c.t, torch.tensor(start, dtype=torch.int32, device="cuda")).cpu()
    picked = [(0, 0), (0, M - 1), (1, 15), (1, 16), (2, 63 if M > 63 else 31), (3, M // 2), (3, M - 1)]
    _check_rows(c, torch.stack([q[b, m] for b, m in picked]), torch.stack([out[b, m] for b, m in picked]),
                [(b, start[b] + m + 1) for b, m in picked], Dh ** -0.5, dt, what="prompt")


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Dh,H,Hk,M,start,B", [(128, 2, 1, 90, 37, 1), (64, 3, 3, 40, 100, 2), (128, 32, 32, 130, 3, 4), (64, 4, 2, 70, 400, 1), (128, 4, 2, 70, 700, 1)])
def test_a_nan_stays_in_what_sees_it(dt, Dh, H, Hk, M, start, B):
    """A NaN among the values of a later token leaves the rows before it and the other groups of channels as they are; one among its keys leaves the
    rows before it."""
    from flashsvd_amd import hip_ops
    S = start + M
    clean, c = (Cache(B, S, Hk, Dh, seed=41) for _ in range(2))
    g = torch.Generator().manual_seed(42)
    q = (torch.randn(B, M, H, Dh, generator=g) * 0.7).to(dt)
    pos = torch.full((B,), start, dtype=torch.int32, device="cuda")
    last = Dh // 32 - 1
    marks = [(0, start + 11, 0, 0), (0, start + 30, 0, 1), (0, start + 12, 0, 0), (B - 1, start + M - 1, Hk - 1, last), (B - 1, start, Hk - 1, last)]
    for b, n, hk, d in marks:                             # the clean cache holds zeros there: what else goes into the sums is alike
        for x in (clean, c):
            x.t[1][b, n, hk, 16 * d:16 * d + 16] = 0
        c.t[3][b, hk, d, n] = 255
    want, got = (hip_ops.attn_prefill_kv4(q.cuda(), *x.t, pos).float().cpu() for x in (clean, c))
    per = H // Hk
    for b, n, hk, d in marks:
        want[b, n - start:, hk * per:(hk + 1) * per, 32 * d:32 * d + 32] = float("nan")
    assert _same(got.double(), want.double())
    one, seen = torch.full((B,), start + 12, dtype=torch.int32, device="cuda"), hip_ops.attn_decode_kv4
    want, got = (seen(q[:, 0].cuda(), *x.t, one).float().cpu() for x in (clean, c))
    for b, n, hk, d in marks:
        if n < start + 12:
            want[b, hk * per:(hk + 1) * per, 32 * d:32 * d + 32] = float("nan")
    assert _same(got.double(), want.double())

    base = hip_ops.attn_prefill_kv4(q.cuda(), *clean.t, pos).float().cpu()
    clean.t[2][0, 0, 1, start + 20] = 255
    got = hip_ops.attn_prefill_kv4(q.cuda(), *clean.t, pos).float().cpu()
    assert bool(got[0, 20:, :per].isnan().all())
    assert torch.equal(got[0, :20], base[0, :20]) and torch.equal(got[0, :, per:], base[0, :, per:]) and torch.equal(got[1:], base[1:])
    for n, nsplit in ((start + 20, 0), (start + 21, 0), (start + 21, 1)):
        got = seen(q[:, 0].cuda(), *clean.t, torch.full((B,), n, dtype=torch.int32, device="cuda"), nsplit=nsplit or None).float().cpu()
        assert bool(got[0, :per].isnan().all()) == (n > start + 20) and not bool(got[0, per:].isnan().any() or got[1:].isnan().any())


def test_positions_at_the_end_of_the_integers():
    """Lengths and positions far beyond the cache see all of it."""
    from flashsvd_amd import hip_ops
    c = Cache(3, 64, 1, 64, seed=51)
    g = torch.Generator().manual_seed(52)
    q = (torch.randn(3, 9, 2, 64, generator=g) * 0.7).to(torch.bfloat16).cuda()
    far, end = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([2 ** 31 - 1, -2 ** 31, 2 ** 31 - 5], [64, 0, 64]))
    for add in (0, 1, 100):
        want = hip_ops.attn_decode_kv4(q[:, 0], *c.t, end)
        got = hip_ops.attn_decode_kv4(q[:, 0], *c.t, far, seqlen_add=add)
        assert torch.equal(got, want) and not bool(got[1].any())
    near = torch.tensor([63, -9, 63], dtype=torch.int32, device="cuda")
    got, want = (hip_ops.attn_prefill_kv4(q, *c.t, n) for n in (far, near))
    assert torch.equal(got, want) and not bool(got[1].any()) and bool(got[0].any())
    rows = torch.randn(3, 2, 1, 64, generator=g).to(torch.bfloat16).cuda()
    held = [t.clone() for t in c.t]
    hip_ops.kv4_append(rows, rows, *c.t, far)
    assert all(torch.equal(a, b) for a, b in zip(c.t, held))


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_a_decode_loop_captured_and_not(dt):
    """A prompt written and attended to, then tokens: append and attention, the draw of a token and its log probability, eagerly and as a captured graph that is
    replayed with the program's own work between the replays; both leave the same cache, tokens and numbers."""
    from flashsvd_amd import hip_ops
    B, H, Hk, Dh, S, T, V, steps = 3, 4, 2, 64, 128, 21, 1000, 6
    cos, sin = (t.cuda() for t in tables(S, Dh, dt))
    g = torch.Generator().manual_seed(21)
    new = lambda *s: torch.randn(*s, generator=g).to(dt).cuda()      # noqa: E731
    kp, vp, qp = new(B, T, Hk, Dh), new(B, T, Hk, Dh), new(B, T, H, Dh)
    n = torch.tensor([21, 4, 13], dtype=torch.int32, device="cuda")
    head = new(V, H * Dh)
    rows = [(new(B, H, Dh), new(B, Hk, Dh), new(B, Hk, Dh), torch.rand(B, generator=g).cuda()) for _ in range(steps)]

    def fresh():
        c = Cache(B, S, Hk, Dh, seed=1, zero=True)
        zero = torch.zeros(B, dtype=torch.int32, device="cuda")
        hip_ops.kv4_append(kp, vp, *c.t, zero, cos=cos, sin=sin, rows=n)
        first = hip_ops.attn_prefill_kv4(qp, *c.t, zero, cos=cos, sin=sin, rows=n)
        return c, first, n.clone(), torch.zeros(B, 1, dtype=torch.long, device="cuda")

    def step(c, q, k, v, u, pos, tokens):
        o = hip_ops.attn_decode_kv4(q, *c.t, pos, k_new=k, v_new=v, cos=cos, sin=sin)
        logits = hip_ops.linear(o.view(B, H * Dh), head)
        hip_ops.sample_token_(logits, u, tokens, pos, temperature=0.8, top_k=40, top_p=0.9)
        return (o, *hip_ops.token_logprobs(logits, tokens[:, 0], top=5))

    c, first, pos, tokens = fresh()
    eager = []
    for r in rows:
        o = step(c, *r, pos, tokens)
        eager.append(([x.clone() for x in o], tokens.clone()))
    c2, first2, pos2, tokens2 = fresh()
    assert torch.equal(first, first2)
    static = [t.clone() for t in rows[0]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        spare = fresh()
        step(spare[0], *static, spare[2], spare[3])
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(c2, *static, pos2, tokens2)
    for r, (o, t) in zip(rows, eager):
        for s, x in zip(static, r):
            s.copy_(x)
        graph.replay()
        hip_ops.attn_decode_kv4(r[0], *c.t, pos)            # other work of the program
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, o)) and torch.equal(tokens2, t)
    assert torch.equal(pos, pos2) and pos.tolist() == [27, 10, 19]
    assert all(torch.equal(a, b) for a, b in zip(c.t, c2.t))


def test_two_streams_at_once():
    """Calls with key ranges on two streams use scratch of their own."""
    from flashsvd_amd import hip_ops
    c = Cache(2, 3000, 2, 128, seed=31)
    g = torch.Generator().manual_seed(32)
    q = (torch.randn(2, 8, 128, generator=g) * 0.7).to(torch.bfloat16).cuda()
    lens = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([2999, 1000], [17, 2500])]
    want = [hip_ops.attn_decode_kv4(q, *c.t, n) for n in lens]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in lens]
    got = [[], []]
    for _ in range(20):
        for s, n, g_ in zip(streams, lens, got):
            with torch.cuda.stream(s):
                g_.append(hip_ops.attn_decode_kv4(q, *c.t, n))
    torch.cuda.synchronize()
    for g_, w in zip(got, want):
        assert all(torch.equal(x, w) for x in g_)


def test_opcheck_of_the_operators():
    """Schemas and fake tensors against what the kernels do."""
    from flashsvd_amd import hip_ops      # noqa: F401  (registers them)
    ops, checks = torch.ops.flashsvd_hip, ("test_schema", "test_faketensor")
    c = Cache(2, 700, 2, 64, seed=51).t
    g = torch.Generator().manual_seed(52)
    rand = lambda *shape: torch.randn(*shape, generator=g).to(torch.bfloat16).cuda()      # noqa: E731
    n = torch.tensor([600, 5], dtype=torch.int32, device="cuda")
    torch.library.opcheck(ops.kv4_append.default, (rand(2, 9, 2, 64), rand(2, 9, 2, 64), *c, n), test_utils=checks)
    torch.library.opcheck(ops.kv4_dequantize.default, (*c, 70, torch.float16), test_utils=checks)
    q, out = rand(2, 4, 64), rand(2, 4, 64)
    torch.library.opcheck(ops.attn_decode_kv4.default, (q, *c, n), dict(k_new=rand(2, 2, 64), v_new=rand(2, 2, 64)), test_utils=checks)
    torch.library.opcheck(ops.attn_decode_kv4.out, (q, *c, n), dict(out=out), test_utils=checks)
    q, out = rand(2, 9, 4, 64), rand(2, 9, 4, 64)
    torch.library.opcheck(ops.attn_prefill_kv4.default, (q, *c, n), test_utils=checks)
    torch.library.opcheck(ops.attn_prefill_kv4.out, (q, *c, n), dict(rows=torch.tensor([3, 9], dtype=torch.int32, device="cuda"), out=out), test_utils=checks)
    x, t = rand(3, 5, 40000), torch.randint(0, 40000, (3, 5), generator=g).cuda()
    for top in (0, 4):
        torch.library.opcheck(ops.token_logprobs.default, (x, t, top), test_utils=checks)
