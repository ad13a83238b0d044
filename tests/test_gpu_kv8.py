"""The KV cache in 8 bits (csrc/kv8.hip, csrc/kv8_attn.hip) against its definition in 64 bits: what an append leaves in the cache, attention of single
tokens and of chunks over it, and all of them together as a decode loop uses them, captured and not."""
import math

import pytest
import torch

from tests import kv8_reference as R

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn


class Cache:
    """Codes and scales with something in every row, on the GPU, and their doubles here."""

    def __init__(self, B, S, Hk, Dh, block, seed, layout="head", zero=False):
        g = torch.Generator().manual_seed(seed)
        n = -(-S // block)
        order = (B, Hk, S, Dh) if layout == "head" else (B, S, Hk, Dh)
        x = torch.randn(order, generator=g) * 100.0
        s = torch.exp2(torch.randint(-9, -4, (B, Hk, n) if layout == "head" else (B, n, Hk), generator=g).float())
        if zero:
            x, s = x * 0, s * 0
        k, v = x.to(F8), x.flip(-1).to(F8)
        self.t = [t.cuda().transpose(1, 2) if layout == "head" else t.cuda() for t in (k, v, s, 2 * s)]
        self.block = block

    def finite(self):
        """Without the few codes of NaN that the conversion of the largest random numbers left."""
        for t in self.t[:2]:
            w = t.view(torch.uint8)
            w.masked_fill_((w & 0x7f) == 0x7f, 0x7e)
        return self

    def doubles(self):
        return [t.cpu().float().double() for t in self.t]

    def values(self):
        k, v, ks, vs = self.doubles()
        S = k.shape[1]
        full = lambda s: s.repeat_interleave(self.block, 1)[:, :S, :, None]      # noqa: E731
        return k * full(ks), v * full(vs)


def tables(length, Dh, dt):
    ang = torch.arange(length)[:, None].double() * 10000.0 ** (-torch.arange(Dh // 2).double() / (Dh // 2))
    return ang.cos().to(dt), ang.sin().to(dt)


def _same(a, b):
    return torch.equal(a.nan_to_num(-1e9), b.nan_to_num(-1e9))


def half_step(dt):
    return torch.finfo(dt).eps / 2


# ------------------------------------------------------------------ append
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Dh,Hk,block,layout,T,at,rows", [
    (128, 2, 16, "head", 1, [0, 5, 15, 16, 47], None),
    (64, 3, 32, "token", 1, [0, 31, 32, 46, 7], None),
    (128, 1, 32, "head", 7, [0, 3, 30, 25, 41], None),
    (64, 2, 16, "head", 33, [0, 1, 15, 14, 7], [33, 0, 1, 17, 32]),
    (128, 2, 64, "token", 40, [0, 8, 5, 1, 3], [40, 40, 0, 3, 39]),
    (64, 1, 128, "head", 48, [0, 0, 0, 0, 0], [48, 1, 2, 47, 0]),
    # outside the cache: dropped in front of it and behind it
    (64, 2, 16, "head", 5, [-3, 46, 48, 100, -9], None),
])
def test_append_holds_what_the_definition_says(dt, Dh, Hk, block, layout, T, at, rows):
    """Without a rotation every step is exact but the one rounding: codes and scales are equal."""
    from flashsvd_amd import hip_ops
    B, S = len(at), 48
    c = Cache(B, S, Hk, Dh, block, seed=T + Dh, layout=layout)
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(B, T, Hk, Dh, generator=g) * torch.exp2(torch.randint(-3, 3, (B, T, Hk, 1), generator=g).float())).to(dt), torch.randn(B, T, Hk, Dh, generator=g).to(dt)
    want = c.doubles()
    for b in range(B):
        n = T if rows is None else rows[b]
        R.append(want[0][b], want[2][b], k[b], at[b], n, block)
        R.append(want[1][b], want[3][b], v[b], at[b], n, block)
    wide = torch.zeros(B, T, Hk, 2 * Dh, dtype=dt, device="cuda")               # rows inside longer ones
    wide[..., :Dh], wide[..., Dh:] = k.cuda(), v.cuda()
    hip_ops.kv8_append(wide[..., :Dh], wide[..., Dh:], *c.t, torch.tensor(at, dtype=torch.int32, device="cuda"), block=block,
                       rows=None if rows is None else torch.tensor(rows, dtype=torch.int32, device="cuda"))
    for got, w, name in zip(c.doubles(), want, ("k", "v", "k_scale", "v_scale")):
        assert _same(got, w), f"{name}: {int((got != w).sum())} of {w.numel()} differ"


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Dh,block,T,at", [(128, 32, 1, [0, 9, 40]), (64, 16, 21, [0, 11, 26]), (128, 64, 50, [0, 1, 13])])
def test_append_rotates_keys(dt, Dh, block, T, at):
    """The rotated key is rounded once: at most half a step of a code (2^-4 of the value, 2^-10 of the scale among the subnormals) and what two products and a
    sum in fp32 leave, 2^-22 of the pair's magnitudes."""
    from flashsvd_amd import hip_ops
    B, S, Hk = len(at), 64, 2
    cos, sin = tables(S - 3, Dh, dt)                     # the last positions take the last row of the tables
    c = Cache(B, S, Hk, Dh, block, seed=5, zero=True)
    g = torch.Generator().manual_seed(4)
    k, v = torch.randn(B, T, Hk, Dh, generator=g).to(dt), torch.randn(B, T, Hk, Dh, generator=g).to(dt)
    hip_ops.kv8_append(k.cuda(), v.cuda(), *c.t, torch.tensor(at, dtype=torch.int32, device="cuda"), block=block, cos=cos.cuda(), sin=sin.cuda())
    kv, vv = c.values()
    for b in range(B):
        for t in range(T):
            p = at[b] + t
            x = R.rotate(k[b, t].double(), cos, sin, p)
            size = c.t[2][b, p // block].cpu().double()[:, None]
            mag = k[b, t].double().abs()
            room = x.abs() * 2.0 ** -4 + size * 2.0 ** -10 + 2.0 ** -22 * (mag + mag.roll(Dh // 2, -1))
            assert bool(((kv[b, p] - x).abs() <= room).all()), f"key of {b}, {p}"
            y, vsize = v[b, t].double(), c.t[3][b, p // block].cpu().double()[:, None]
            assert bool(((vv[b, p] - y).abs() <= y.abs() * 2.0 ** -4 + vsize * 2.0 ** -10).all()), f"value of {b}, {p}"


def test_append_token_by_token_grows_a_block():
    """Rows of rising magnitude, one call each: the scale of the block rises with them and the rows that it holds move to it exactly as the definition has it,
    values of 2^-126 and of the largest 16-bit floats, zeros, infinities and NaN among them."""
    from flashsvd_amd import hip_ops
    Dh, Hk, block, S = 64, 1, 16, 32
    for dt in (torch.bfloat16, torch.float16):
        c = Cache(1, S, Hk, Dh, block, seed=9, zero=True)
        want = c.doubles()
        g = torch.Generator().manual_seed(8)
        small = float(torch.finfo(dt).smallest_normal)
        for t, size in enumerate([0.0, small, 1e-3, 1e-3, 0.5, 0.0, 447.0, 448.0, 449.0, 1e4, 2.0, float(torch.finfo(dt).max), 1.0, float("inf"), float("nan"), 3.0, 4.0, 1.0]):
            row = torch.rand(1, 1, Hk, Dh, generator=g)
            if math.isfinite(size):
                row = row * size
                row[..., 5] = -size
            else:
                row[..., 3], row[..., 4] = size, -size
            row = row.to(dt)
            R.append(want[0][0], want[2][0], row[0], t, 1, block)
            R.append(want[1][0], want[3][0], -row[0], t, 1, block)
            hip_ops.kv8_append(row.cuda(), -row.cuda(), *c.t, torch.tensor([t], dtype=torch.int32, device="cuda"), block=block)
            for got, w, name in zip(c.doubles(), want, ("k", "v", "k_scale", "v_scale")):
                assert _same(got, w), f"{dt} {name} after row {t}"


# ------------------------------------------------------------------ attention
def _spoil(c, lens):
    """NaN in every row that no query may see, and in the scales of blocks without a visible row."""
    for b, n in enumerate(lens):
        n = max(n, 0)
        for t in c.t[:2]:
            t.view(torch.uint8)[b, n:] = 0x7f
        for t in c.t[2:]:
            t[b, -(-n // c.block):] = float("nan")


def _close(got, want, room, dt, what):
    got = got.double().cpu()
    assert bool(torch.isfinite(got).all()), what
    over = (got - want).abs() - (want.abs() * half_step(dt) + room * (1 + half_step(dt)) + 1e-30)
    assert float(over.max()) <= 0, f"{what}: {float(over.max()):.3g} over the bound"


def _errors(dt, rotated):
    """Relative rounding of q (16 bits where the call rotates it) and of the softmax weights (16 bits)."""
    return half_step(dt) if rotated else 0.0, half_step(torch.bfloat16)


def _check_rows(c, q, out, lens, scale, dt, cos=None, sin=None, pos=None, what=""):
    """q, out [rows, H, Dh] of rows (sequence b, keys n, position): one query each."""
    k, v = c.values()
    H, Hk = q.shape[1], k.shape[2]
    qe, we = _errors(dt, cos is not None)
    for i, (b, n) in enumerate(lens):
        for h in range(H):
            x = R.rotate(q[i, h].double(), cos, sin, pos[i] if pos else 0)
            hk = h // (H // Hk)
            want, room = R.attend(x, k[b, :n, hk], v[b, :n, hk], scale, qe, we)
            _close(out[i, h], want, room, dt, f"{what} row {i} head {h} of {n} keys")


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Dh,H,Hk,block,layout,lens,S", [
    (128, 4, 4, 32, "head", [1, 33, 0, 70], 96),
    (128, 8, 2, 16, "token", [95, 16, 17, 15], 96),
    (64, 8, 8, 32, "head", [137], 160),
    (64, 6, 2, 64, "head", [64, 65, 129], 130),
    (128, 5, 1, 128, "token", [127, 128, 129, 200], 200),
    (128, 7, 1, 16, "head", [31], 40),
    (64, 16, 1, 16, "head", [100, 1], 112),
    (64, 40, 2, 32, "head", [61], 64),
    (128, 34, 2, 16, "token", [300, 7], 301),
    (128, 2, 2, 32, "head", [1500, 3, 700], 1501),
    (128, 8, 1, 64, "head", [4097], 4100),
    (64, 20, 1, 32, "head", [900, 0, 513], 1000),          # more than 16 heads of a kv head over key ranges
    (128, 1, 1, 16, "head", [500, 0, -4, 9999], 256),      # a negative length, and one beyond the cache
])
def test_decode_attention(dt, Dh, H, Hk, block, layout, lens, S):
    from flashsvd_amd import hip_ops
    B = len(lens)
    c = Cache(B + 1, S, Hk, Dh, block, seed=S + H, layout=layout).finite()
    keys = [min(max(n, 0), S) for n in lens]
    _spoil(c, keys)
    g = torch.Generator().manual_seed(7)
    q = (torch.randn(B, H, Dh, generator=g) * 0.7).to(dt)
    wide = torch.zeros(B, H + 1, Dh + 8, dtype=dt, device="cuda")
    wide[:, :H, :Dh] = q.cuda()
    n32 = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = hip_ops.attn_decode_kv8(wide[:, :H, :Dh], *c.t, n32, block=block)
    _check_rows(c, q, out, list(enumerate(keys)), Dh ** -0.5, dt, what="decode")
    for nsplit in (1, 3, 7, 64):                          # any cut of the keys is within the same bound; `out` inside longer rows
        into = torch.full((B, H + 2, Dh + 4), 7.0, dtype=dt, device="cuda")
        hip_ops.attn_decode_kv8(wide[:, :H, :Dh], *c.t, n32, block=block, nsplit=nsplit, out=into[:, 1:H + 1, :Dh], softmax_scale=0.2)
        _check_rows(c, q, into[:, 1:H + 1, :Dh], list(enumerate(keys)), 0.2, dt, what=f"decode in {nsplit}")
        assert bool((into[:, 0] == 7).all() and (into[:, H + 1] == 7).all() and (into[:, :, Dh:] == 7).all())


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Dh,H,Hk,block,at,S", [
    (128, 8, 2, 32, [0, 5, 31, 32, 100], 128),
    (64, 8, 8, 16, [137, 0], 144),
    (128, 4, 4, 64, [63, 64, 699], 700),
    (64, 9, 1, 128, [130, 127, 128, 50, 40, 1], 200),
    (64, 20, 1, 32, [900, 0, 513], 1000),
    (128, 4, 2, 128, [127, 128, 383, 384, 511, 1151], 1152),      # a new row at the ends of ranges
])
def test_decode_attention_appends_its_token(dt, Dh, H, Hk, block, at, S):
    """The call against an append of its own followed by attention: the same cache, bit for bit, and the output within the bound over it."""
    from flashsvd_amd import hip_ops
    B = len(at)
    cos, sin = tables(S, Dh, dt)
    c, other = (Cache(B, S, Hk, Dh, block, seed=11).finite() for _ in range(2))
    g = torch.Generator().manual_seed(12)
    q, k, v = ((torch.randn(B, h, Dh, generator=g) * f).to(dt) for h, f in ((H, 0.7), (Hk, 20.0), (Hk, 1.0)))
    pos = torch.tensor(at, dtype=torch.int32, device="cuda")
    kw = dict(block=block, cos=cos.cuda(), sin=sin.cuda())
    out = hip_ops.attn_decode_kv8(q.cuda(), *c.t, pos, k_new=k.cuda(), v_new=v.cuda(), **kw)
    hip_ops.kv8_append(k.cuda()[:, None], v.cuda()[:, None], *other.t, pos, **kw)
    for a, b in zip(c.doubles(), other.doubles()):
        assert torch.equal(a, b)
    _check_rows(c, q, out, [(b, n + 1) for b, n in enumerate(at)], Dh ** -0.5, dt, cos, sin, at, "append and decode")
    again = hip_ops.attn_decode_kv8(q.cuda(), *other.t, pos, seqlen_add=1, **kw)
    _check_rows(other, q, again, [(b, n + 1) for b, n in enumerate(at)], Dh ** -0.5, dt, cos, sin, at, "decode behind an append")


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Dh,H,Hk,block,layout,M,start,rows", [
    (128, 4, 4, 32, "head", 1, [0, 40], None),
    (128, 4, 2, 16, "token", 17, [0, 5, 100], [17, 0, 9]),
    (64, 8, 2, 32, "head", 33, [0, 31], None),
    (64, 2, 2, 64, "head", 130, [0, 3], [130, 65]),
    (128, 6, 1, 128, "head", 77, [211, 0, 64], [77, 1, 76]),
    (128, 1, 1, 16, "token", 150, [0], None),
    (64, 3, 1, 16, "head", 64, [64], None),
    (128, 2, 1, 32, "head", 40, [500, 1], None),
    (128, 4, 2, 32, "head", 9, [900, 3, 650], [9, 9, 0]),      # in ranges of the keys
    (64, 2, 2, 128, "token", 3, [1500], None),
])
def test_prompt_attention(dt, Dh, H, Hk, block, layout, M, start, rows):
    from flashsvd_amd import hip_ops
    B = len(start)
    n = rows or [M] * B
    S = max(p + t for p, t in zip(start, n)) + 3
    c = Cache(B, S, Hk, Dh, block, seed=M + H, layout=layout).finite()
    _spoil(c, [p + t for p, t in zip(start, n)])
    cos, sin = tables(S, Dh, dt)
    g = torch.Generator().manual_seed(13)
    q = (torch.randn(B, M, H, Dh, generator=g) * 0.7).to(dt)
    p32 = torch.tensor(start, dtype=torch.int32, device="cuda")
    r32 = None if rows is None else torch.tensor(rows, dtype=torch.int32, device="cuda")
    for rope in ((None, None), (cos, sin)):
        into = torch.full((B, M + 1, H, Dh + 4), 7.0, dtype=dt, device="cuda")
        hip_ops.attn_prefill_kv8(q.cuda(), *c.t, p32, block=block, rows=r32, cos=None if rope[0] is None else cos.cuda(),
                                 sin=None if rope[0] is None else sin.cuda(), out=into[:, :M, :, :Dh])
        flat = [(b, m) for b in range(B) for m in range(n[b])]
        picked = flat if len(flat) <= 60 else flat[:8] + flat[8:-8:max(1, len(flat) // 40)] + flat[-8:]
        _check_rows(c, torch.stack([q[b, m] for b, m in picked]), torch.stack([into[b, m, :, :Dh].cpu() for b, m in picked]),
                    [(b, start[b] + m + 1) for b, m in picked], Dh ** -0.5, dt, *rope, [start[b] + m for b, m in picked], "prompt")
        for b in range(B):
            assert bool((into[b, n[b]:] == 7).all()), "rows behind the last one"
        assert bool((into[..., Dh:] == 7).all())
    zeros = hip_ops.attn_prefill_kv8(q.cuda(), *c.t, p32, block=block, rows=r32)
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
    c = Cache(B, max(start) + M, Hk, Dh, 32, seed=M).finite()
    g = torch.Generator().manual_seed(14)
    q = (torch.randn(B, M, H, Dh, generator=g) * 0.7).to(dt)
    out = hip_ops.attn_prefill_kv8(q.cuda(), *c.t, torch.tensor(start, dtype=torch.int32, device="cuda"), block=32).cpu()
    picked = [(0, 0), (0, M - 1), (1, 15), (1, 16), (2, 63 if M > 63 else 31), (3, M // 2), (3, M - 1)]
    _check_rows(c, torch.stack([q[b, m] for b, m in picked]), torch.stack([out[b, m] for b, m in picked]),
                [(b, start[b] + m + 1) for b, m in picked], Dh ** -0.5, dt, what="prompt")


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Dh,H,Hk,M,start,B", [(128, 2, 1, 90, 37, 1), (64, 3, 3, 40, 100, 2), (128, 32, 32, 130, 3, 4), (64, 4, 2, 70, 400, 1), (128, 4, 2, 70, 700, 1)])
def test_a_nan_stays_in_what_sees_it(dt, Dh, H, Hk, M, start, B):
    """A NaN among the values of a later token leaves the rows before it as they are, in every dimension; so does one among its keys."""
    from flashsvd_amd import hip_ops
    S = start + M
    clean = Cache(B, S, Hk, Dh, 16, seed=41).finite()
    g = torch.Generator().manual_seed(42)
    q = (torch.randn(B, M, H, Dh, generator=g) * 0.7).to(dt)
    pos = torch.full((B,), start, dtype=torch.int32, device="cuda")
    marks = [(0, start + 11, 0, 5), (0, start + 30, 0, 0), (0, start + 12, 0, 5), (B - 1, start + M - 1, Hk - 1, Dh - 1), (B - 1, start, Hk - 1, 2)]
    for b, n, hk, d in marks:                             # the clean cache holds zeros there: what else goes into the sums is alike
        clean.t[1].view(torch.uint8)[b, n, hk, d] = 0
    c = Cache(B, S, Hk, Dh, 16, seed=41).finite()
    for t, u in zip(c.t, clean.t):
        t.copy_(u) if t.dtype is not F8 else t.view(torch.uint8).copy_(u.view(torch.uint8))
    for b, n, hk, d in marks:
        c.t[1].view(torch.uint8)[b, n, hk, d] = 0xff if d else 0x7f
    want, got = (hip_ops.attn_prefill_kv8(q.cuda(), *x.t, pos, block=16).float().cpu() for x in (clean, c))
    per = H // Hk
    for b, n, hk, d in marks:
        want[b, n - start:, hk * per:(hk + 1) * per, d] = float("nan")
    assert _same(got.double(), want.double())
    one, seen = torch.full((B,), start + 12, dtype=torch.int32, device="cuda"), hip_ops.attn_decode_kv8
    want, got = (seen(q[:, 0].cuda(), *x.t, one, block=16).float().cpu() for x in (clean, c))
    for b, n, hk, d in marks:
        if n < start + 12:
            want[b, hk * per:(hk + 1) * per, d] = float("nan")
    assert _same(got.double(), want.double())

    base = hip_ops.attn_prefill_kv8(q.cuda(), *clean.t, pos, block=16).float().cpu()
    clean.t[0].view(torch.uint8)[0, start + 20, 0, 3] = 0x7f
    got = hip_ops.attn_prefill_kv8(q.cuda(), *clean.t, pos, block=16).float().cpu()
    assert bool(got[0, 20:, :per].isnan().all())
    assert torch.equal(got[0, :20], base[0, :20]) and torch.equal(got[0, :, per:], base[0, :, per:]) and torch.equal(got[1:], base[1:])
    for n, nsplit in ((start + 20, 0), (start + 21, 0), (start + 21, 1)):
        got = seen(q[:, 0].cuda(), *clean.t, torch.full((B,), n, dtype=torch.int32, device="cuda"), block=16, nsplit=nsplit or None).float().cpu()
        assert bool(got[0, :per].isnan().all()) == (n > start + 20) and not bool(got[0, per:].isnan().any() or got[1:].isnan().any())


def test_positions_at_the_end_of_the_integers():
    """Lengths and positions far beyond the cache see all of it."""
    from flashsvd_amd import hip_ops
    c = Cache(3, 40, 1, 64, 16, seed=51).finite()
    g = torch.Generator().manual_seed(52)
    q = (torch.randn(3, 9, 2, 64, generator=g) * 0.7).to(torch.bfloat16).cuda()
    far, end = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([2 ** 31 - 1, -2 ** 31, 2 ** 31 - 5], [40, 0, 40]))
    for add in (0, 1, 100):
        want = hip_ops.attn_decode_kv8(q[:, 0], *c.t, end, block=16)
        got = hip_ops.attn_decode_kv8(q[:, 0], *c.t, far, block=16, seqlen_add=add)
        assert torch.equal(got, want) and not bool(got[1].any())
    near = torch.tensor([39, -9, 39], dtype=torch.int32, device="cuda")
    got, want = (hip_ops.attn_prefill_kv8(q, *c.t, n, block=16) for n in (far, near))
    assert torch.equal(got, want) and not bool(got[1].any()) and bool(got[0].any())


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_a_decode_loop_captured_and_not(dt):
    """A prompt written and attended to, then tokens: append and attention and the draw of a token, eagerly and as a captured graph that is replayed with the
    program's own work between the replays; both leave the same cache and tokens."""
    from flashsvd_amd import hip_ops
    B, H, Hk, Dh, block, S, T, V, steps = 3, 4, 2, 64, 16, 80, 21, 1000, 6
    cos, sin = (t.cuda() for t in tables(S, Dh, dt))
    g = torch.Generator().manual_seed(21)
    new = lambda *s: torch.randn(*s, generator=g).to(dt).cuda()      # noqa: E731
    kp, vp, qp = new(B, T, Hk, Dh), new(B, T, Hk, Dh), new(B, T, H, Dh)
    n = torch.tensor([21, 4, 13], dtype=torch.int32, device="cuda")
    head = new(V, H * Dh)
    rows = [(new(B, H, Dh), new(B, Hk, Dh), new(B, Hk, Dh), torch.rand(B, generator=g).cuda()) for _ in range(steps)]

    def fresh():
        c = Cache(B, S, Hk, Dh, block, seed=1, zero=True)
        zero = torch.zeros(B, dtype=torch.int32, device="cuda")
        hip_ops.kv8_append(kp, vp, *c.t, zero, block=block, cos=cos, sin=sin, rows=n)
        first = hip_ops.attn_prefill_kv8(qp, *c.t, zero, block=block, cos=cos, sin=sin, rows=n)
        return c, first, n.clone(), torch.zeros(B, 1, dtype=torch.long, device="cuda")

    def step(c, q, k, v, u, pos, tokens):
        o = hip_ops.attn_decode_kv8(q, *c.t, pos, block=block, k_new=k, v_new=v, cos=cos, sin=sin)
        logits = hip_ops.linear(o.view(B, H * Dh), head)
        hip_ops.sample_token_(logits, u, tokens, pos, temperature=0.8, top_k=40, top_p=0.9)
        return o

    c, first, pos, tokens = fresh()
    eager = []
    for r in rows:
        o = step(c, *r, pos, tokens)
        eager.append((o.clone(), tokens.clone()))
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
        hip_ops.attn_decode_kv8(r[0], *c.t, pos, block=block)            # other work of the program
        torch.cuda.synchronize()
        assert torch.equal(out, o) and torch.equal(tokens2, t)
    assert torch.equal(pos, pos2) and pos.tolist() == [27, 10, 19]
    for a, b in zip(c.doubles(), c2.doubles()):
        assert torch.equal(a, b)


def test_two_streams_at_once():
    """Calls with key ranges on two streams use scratch of their own."""
    from flashsvd_amd import hip_ops
    c = Cache(2, 3000, 2, 128, 32, seed=31).finite()
    g = torch.Generator().manual_seed(32)
    q = (torch.randn(2, 8, 128, generator=g) * 0.7).to(torch.bfloat16).cuda()
    lens = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([2999, 1000], [17, 2500])]
    want = [hip_ops.attn_decode_kv8(q, *c.t, n, block=32) for n in lens]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in lens]
    got = [[], []]
    for _ in range(20):
        for s, n, g_ in zip(streams, lens, got):
            with torch.cuda.stream(s):
                g_.append(hip_ops.attn_decode_kv8(q, *c.t, n, block=32))
    torch.cuda.synchronize()
    for g_, w in zip(got, want):
        assert all(torch.equal(x, w) for x in g_)
