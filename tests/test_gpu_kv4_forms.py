"""Every kernel form of the KV cache in 4 bits and of the log probabilities, by name: shapes on either side of each rule, against the definitions in 64 bits, and how
few bits the weights of the attention may lose."""
import math

import pytest
import torch

from tests import kv4_reference as R
from tests.test_gpu_kv4 import HALF_PART, TWO_PARTS, Cache, _check_rows, _close
from tests.test_gpu_kv8 import _same, tables
from tests.util import form_taken

pytestmark = pytest.mark.gpu

# the name of the form, the heads' dimensions that take it, what a call takes, and rows of a sequence that are real (of M)
SHAPES = [
    ("kv4 prompt 128", (64, 128), dict(B=8, Hk=32, G=1, M=130, past=7, rows=[130, 129, 128, 65, 64, 1, 0, 130])),
    ("kv4 prompt 128", (64, 128), dict(B=16, Hk=16, G=2, M=70, past=40, rows=None)),
    ("kv4 prompt 128", (64, 128), dict(B=1, Hk=8, G=6, M=1400, past=300, rows=None)),
    ("kv4 prompt 128", (128,), dict(B=8, Hk=25, G=1, M=70, past=133, rows=[70, 64, 63, 17, 16, 1, 0, 70])),
    ("kv4 prompt 128 ranges", (64, 128), dict(B=1, Hk=8, G=4, M=300, past=4400, rows=None)),
    ("kv4 prompt 128 ranges", (64, 128), dict(B=2, Hk=4, G=4, M=300, past=4400, rows=[299, 3])),
    ("kv4 prompt 128 ranges", (64, 128), dict(B=1, Hk=8, G=8, M=400, past=3800, rows=None)),
    ("kv4 prompt 64", (64, 128), dict(B=8, Hk=25, G=1, M=70, past=33, rows=[70, 64, 63, 17, 16, 1, 0, 70])),
    ("kv4 prompt 64", (64, 128), dict(B=2, Hk=5, G=3, M=850, past=0, rows=None)),
    ("kv4 prompt 64 halves", (64, 128), dict(B=2, Hk=2, G=2, M=40, past=90, rows=[39, 40])),
    ("kv4 prompt 64 halves", (64, 128), dict(B=3, Hk=29, G=1, M=256, past=0, rows=None)),
    ("kv4 prompt 64 halves ranges", (64, 128), dict(B=1, Hk=2, G=3, M=21, past=1200, rows=None)),
    ("kv4 prompt 64 halves ranges", (64, 128), dict(B=3, Hk=1, G=1, M=64, past=700, rows=[64, 2, 0])),
]
PROMPTS = [(name, p, Dh) for name, dims, p in SHAPES for Dh in dims]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("turn", [False, True])
@pytest.mark.parametrize("name,p,Dh", PROMPTS)
def test_prompt_forms(name, p, turn, Dh, dt):
    """Rows of unequal numbers, NaN in every row that none sees, an out whose rows stand at odd elements, scores with and without a rotation."""
    from flashsvd_amd import hip_ops
    B, Hk, M, past, H = p["B"], p["Hk"], p["M"], p["past"], p["Hk"] * p["G"]
    n = p["rows"] or [M] * B
    c = Cache(B, past + M, Hk, Dh, seed=M + Dh)
    c.spoil([past + t for t in n])
    g = torch.Generator().manual_seed(71)
    q = (torch.randn(B, M, H, Dh, generator=g) * 0.7).to(dt)
    cos, sin = tables(past + M, Dh, dt) if turn else (None, None)
    into = torch.full((B, M, H, Dh + 3), 7.0, dtype=dt, device="cuda")
    hip_ops.attn_prefill_kv4(q.cuda(), *c.t, torch.full((B,), past, dtype=torch.int32, device="cuda"),
                             rows=None if p["rows"] is None else torch.tensor(n, dtype=torch.int32, device="cuda"),
                             cos=cos.cuda() if turn else None, sin=sin.cuda() if turn else None, out=into[..., 1:Dh + 1])
    assert form_taken() == name
    out = into.cpu()
    assert bool((out[..., 0] == 7).all() and (out[..., Dh + 1:] == 7).all())
    for b in range(B):
        assert bool((out[b, n[b]:] == 7).all()), "rows behind the last one"
    picked = [(b, m) for b in {0, B // 2, B - 1} for m in sorted({0, n[b] // 3, n[b] // 2, n[b] - 1}) if 0 <= m < n[b]]
    heads = sorted({0, H // 2, H - 1})
    _check_rows(c, torch.stack([q[b, m] for b, m in picked]), torch.stack([out[b, m, :, 1:Dh + 1] for b, m in picked]),
                [(b, past + m + 1) for b, m in picked], Dh ** -0.5, dt, cos, sin, [past + m for b, m in picked], name, heads)


@pytest.mark.parametrize("Dh", [64, 128])
@pytest.mark.parametrize("where", [[5], [300], [64, 127], [700, 701], [897], [0, 899]])
@pytest.mark.parametrize("byte", [1, 90, 103, 104, 140, 141, 200, 252])
def test_values_that_float16_does_not_hold(byte, where, Dh):
    """Long chunks in bf16 keep V in float16 up to the first tile with a scale that it does not hold (below 2^-23, above 2^13): rows on either side of such tokens."""
    from flashsvd_amd import hip_ops
    B, Hk, H, M, past, dt = 8, 16, 32, 300, 600, torch.bfloat16
    c = Cache(B, past + M, Hk, Dh, seed=byte)
    g = torch.Generator().manual_seed(72)
    q = (torch.randn(B, M, H, Dh, generator=g) * 0.7).to(dt)
    for n in where:
        c.t[3][1, 3, 1, n] = byte
        c.t[3][6, :, :, n] = byte
    out = hip_ops.attn_prefill_kv4(q.cuda(), *c.t, torch.full((B,), past, dtype=torch.int32, device="cuda")).cpu()
    assert form_taken() == "kv4 prompt 128"
    picked = [(b, m) for b in (0, 1, 6) for m in (0, 30, 97, 98, 200, 297, 299)]
    _check_rows(c, torch.stack([q[b, m] for b, m in picked]), torch.stack([out[b, m] for b, m in picked]), [(b, past + m + 1) for b, m in picked], Dh ** -0.5, dt,
                what=f"byte {byte}", heads=[6, 7, 31])


@pytest.mark.parametrize("name,p,Dh", PROMPTS[4:])
def test_the_largest_values_do_not_become_infinite(name, p, Dh):
    """A value near the largest number of float32 at a key whose score is well above the scores before it."""
    from flashsvd_amd import hip_ops
    B, Hk, M, past, H, dt = p["B"], p["Hk"], p["M"], p["past"], p["Hk"] * p["G"], torch.bfloat16
    c = Cache(B, past + M, Hk, Dh, seed=6)
    at = (past + M) // 2
    c.t[3][:, :, :, at] = 252
    c.t[2][:, :, :, at] += 2
    g = torch.Generator().manual_seed(74)
    q = (torch.randn(B, M, H, Dh, generator=g) * 0.7).to(dt)
    out = hip_ops.attn_prefill_kv4(q.cuda(), *c.t, torch.full((B,), past, dtype=torch.int32, device="cuda")).cpu()
    assert form_taken() == name
    picked = [(b, m) for b in {0, B - 1} for m in (0, M // 2, M - 1)]
    _check_rows(c, torch.stack([q[b, m] for b, m in picked]), torch.stack([out[b, m] for b, m in picked]), [(b, past + m + 1) for b, m in picked], Dh ** -0.5, dt,
                what=name, heads=[0, H - 1])


@pytest.mark.parametrize("byte", [1, 103, 141, 252])
@pytest.mark.parametrize("name,p,Dh", PROMPTS[7:])
def test_values_far_apart_in_the_other_forms(name, p, byte, Dh):
    """A value of another size in the first tile, in a middle one and in the last: halves and ranges with and without it are joined."""
    from flashsvd_amd import hip_ops
    B, Hk, M, past, H, dt = p["B"], p["Hk"], p["M"], p["past"], p["Hk"] * p["G"], torch.bfloat16
    for at in (2, past + M // 2, past + M - 2):
        c = Cache(B, past + M, Hk, Dh, seed=6)
        c.t[3][:, Hk // 2, 1, at] = byte
        g = torch.Generator().manual_seed(75)
        q = (torch.randn(B, M, H, Dh, generator=g) * 0.7).to(dt)
        out = hip_ops.attn_prefill_kv4(q.cuda(), *c.t, torch.full((B,), past, dtype=torch.int32, device="cuda")).cpu()
        assert form_taken() == name
        picked = [(b, m) for b in {0, B - 1} for m in (0, M // 2, M - 1)]
        _check_rows(c, torch.stack([q[b, m] for b, m in picked]), torch.stack([out[b, m] for b, m in picked]), [(b, past + m + 1) for b, m in picked], Dh ** -0.5, dt,
                    what=name, heads=sorted({0, H // 2, H - 1}))


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Dh", [64, 128])
def test_a_room_that_is_nearly_empty(Dh, dt):
    """Key ranges by the room's length where sequences hold little of it or nothing: ranges without keys, rows that see none."""
    from flashsvd_amd import hip_ops
    for name, B, Hk, G, M, starts in (("kv4 prompt 128 ranges", 2, 4, 4, 300, [0, 77]), ("kv4 prompt 64 halves ranges", 3, 1, 2, 40, [0, 300, 5])):
        room = 4800
        c = Cache(B, room, Hk, Dh, seed=3)
        c.spoil([s + M for s in starts])
        g = torch.Generator().manual_seed(77)
        q = (torch.randn(B, M, Hk * G, Dh, generator=g) * 0.7).to(dt)
        rows = [M, M - 7, 0][:B]
        out = hip_ops.attn_prefill_kv4(q.cuda(), *c.t, torch.tensor(starts, dtype=torch.int32, device="cuda"), rows=torch.tensor(rows, dtype=torch.int32, device="cuda"))
        assert form_taken() == name
        out = out.cpu()
        for b in range(B):
            assert not bool(out[b, rows[b]:].any())
        picked = [(b, m) for b in range(B) for m in (0, 1, 31, 63, 64, 200, rows[b] - 1) if 0 <= m < rows[b]]
        _check_rows(c, torch.stack([q[b, m] for b, m in picked]), torch.stack([out[b, m] for b, m in picked]), [(b, starts[b] + m + 1) for b, m in picked], Dh ** -0.5, dt,
                    what=name, heads=sorted({0, Hk * G - 1}))
        before = hip_ops.attn_prefill_kv4(q.cuda(), *c.t, torch.tensor([-M - 3] * B, dtype=torch.int32, device="cuda"))       # in front of the cache: no key
        assert not bool(before.any())


def test_small_weights_of_many_keys_are_kept():
    """One key of weight 1 and thousands of 2^-14 to 2^-20 of it, whose values alone are not zero: float16 holds such weights as it holds larger ones."""
    from flashsvd_amd import hip_ops
    Dh, Hk, M, past, dt = 128, 32, 260, 3836, torch.bfloat16
    S = past + M
    for down in (14, 17, 20):
        c = Cache(6, S, Hk, Dh, seed=3, zero=True)
        c.t[2].fill_(127), c.t[3].fill_(127)
        c.t[1].fill_(0x22)                                          # values of 1
        c.t[1][:, 17] = 0
        c.t[0][:, 17, :, 0] = 2                                     # score 1 for one key
        q = torch.zeros(6, M, Hk, Dh, dtype=dt, device="cuda")
        q[..., 0] = 1.0
        by = down * math.log(2.0)
        out = hip_ops.attn_prefill_kv4(q, *c.t, torch.full((6,), past, dtype=torch.int32, device="cuda"), softmax_scale=by).cpu()
        assert form_taken() == "kv4 prompt 128"
        picked = [(0, 0), (1, 100), (3, M - 1)]
        _check_rows(c, torch.stack([q[b, m].cpu() for b, m in picked]), torch.stack([out[b, m] for b, m in picked]), [(b, past + m + 1) for b, m in picked], by, dt,
                    heads=[0, 31])


def _weights_case(B, S, Hk, Dh):
    """Keys of score 0 with values 0, and one of sixteen with weight w = 0.98 of a half step of bf16 over 2^-5: the output is c n w / (m + n w), off by nearly
    2^-8 of itself if w is rounded to bf16."""
    c = Cache(B, S, Hk, Dh, seed=1, zero=True)
    for t in c.t[2:]:
        t.fill_(127)
    c.t[0][:, 5::16, :, 0] = 2 | 8                                  # -1 in the first channel
    varied = torch.tensor([(1 + i % 7) | (1 + (i + 3) % 7) << 4 for i in range(Dh // 2)], dtype=torch.uint8, device="cuda")
    c.t[1][:, 5::16] = varied
    return c, -math.log((1 + 0.98 / 256) * 2.0 ** -5)


ACCURATE = [("kv4 prompt 128", dict(B=8, Hk=32, G=1, M=130, past=7), 64), ("kv4 prompt 128", dict(B=8, Hk=32, G=1, M=130, past=7), 128),
            ("kv4 prompt 128 ranges", dict(B=1, Hk=8, G=4, M=300, past=4400), 64), ("kv4 prompt 128 ranges", dict(B=1, Hk=8, G=4, M=300, past=4400), 128),
            ("kv4 prompt 64", dict(B=8, Hk=25, G=1, M=70, past=33), 64), ("kv4 prompt 64", dict(B=8, Hk=25, G=1, M=70, past=33), 128),
            ("kv4 prompt 64 halves", dict(B=2, Hk=2, G=2, M=40, past=90), 64), ("kv4 prompt 64 halves", dict(B=2, Hk=2, G=2, M=40, past=90), 128),
            ("kv4 prompt 64 halves ranges", dict(B=1, Hk=2, G=3, M=21, past=1200), 64), ("kv4 prompt 64 halves ranges", dict(B=1, Hk=2, G=3, M=21, past=1200), 128)]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("name,p,Dh", ACCURATE)
def test_prompt_weights_keep_their_bits(name, p, Dh, dt):
    from flashsvd_amd import hip_ops
    B, Hk, M, past, H = p["B"], p["Hk"], p["M"], p["past"], p["Hk"] * p["G"]
    c, by = _weights_case(B, past + M, Hk, Dh)
    q = torch.zeros(B, M, H, Dh, dtype=dt, device="cuda")
    q[..., 0] = 1.0
    out = hip_ops.attn_prefill_kv4(q, *c.t, torch.full((B,), past, dtype=torch.int32, device="cuda"), softmax_scale=by).cpu()
    assert form_taken() == name
    picked = [(0, 0), (0, M - 1), (B - 1, 13), (B - 1, M // 2), (B // 2, M - 2)]
    _check_rows(c, torch.stack([q[b, m].cpu() for b, m in picked]), torch.stack([out[b, m] for b, m in picked]), [(b, past + m + 1) for b, m in picked], by, dt,
                what=name, heads=sorted({0, H // 2, H - 1}))


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Dh", [64, 128])
@pytest.mark.parametrize("G", [1, 3, 8, 9, 16, 20])
def test_decode_weights_and_a_rotated_q_keep_their_bits(G, Dh, dt):
    from flashsvd_amd import hip_ops
    B, S, Hk = 2, 1000, 2
    c, by = _weights_case(B, S, Hk, Dh)
    n = torch.tensor([S, 333], dtype=torch.int32, device="cuda")
    q = torch.zeros(B, Hk * G, Dh, dtype=dt, device="cuda")
    q[..., 0] = 1.0
    for nsplit in (1, None):
        out = hip_ops.attn_decode_kv4(q, *c.t, n, softmax_scale=by, nsplit=nsplit)
        assert form_taken() == ("kv4 decode" if nsplit else "kv4 decode ranges")
        _check_rows(c, q.cpu(), out, [(0, S), (1, 333)], by, dt, heads=sorted({0, G - 1, 2 * G - 1}))
    # pairs of channels whose rotation has more bits than the type: every key sees their sum, large against the differences that decide the weights
    cos, sin = tables(S + 1, Dh, dt)
    c = Cache(B, S, Hk, Dh, seed=4)
    g = torch.Generator().manual_seed(73)
    q = (torch.randn(B, Hk * G, Dh, generator=g) * 2).to(dt)
    out = hip_ops.attn_decode_kv4(q.cuda(), *c.t, n, cos=cos.cuda(), sin=sin.cuda())
    _check_rows(c, q, out, [(0, S), (1, 333)], Dh ** -0.5, dt, cos, sin, [S, 333], heads=sorted({0, G - 1, 2 * G - 1}))


def test_a_range_of_nans_alone():
    """Every key of a range a NaN: the joined output is NaN, whatever the other ranges hold; the same for a wave's and a half's keys."""
    from flashsvd_amd import hip_ops
    Dh, Hk, S = 128, 1, 2048
    for first, last in ((0, 256), (512, 1024), (1990, 2048), (64, 128), (3, 4)):
        c = Cache(1, S, Hk, Dh, seed=8)
        c.t[2][:, :, 2, first:last] = 255
        q = torch.ones(1, 4, Dh, dtype=torch.bfloat16, device="cuda")
        n = torch.tensor([S], dtype=torch.int32, device="cuda")
        for nsplit in (None, 1, 3, 8):
            assert bool(hip_ops.attn_decode_kv4(q, *c.t, n, nsplit=nsplit).isnan().all())
        out = hip_ops.attn_prefill_kv4(q[:, None], *c.t, n - 1)
        assert bool(out.isnan().all())


def test_a_nan_of_a_value_that_weighs_nothing():
    """A weight that 32 bits do not hold is above zero, so a NaN among the values that it stands before is one of the output, in how many ranges of keys ever."""
    from flashsvd_amd import hip_ops
    Dh, S = 128, 2048
    c = Cache(1, S, 1, Dh, seed=8)
    c.t[0].zero_()
    c.t[0][:, :256], c.t[2][..., :256] = 0x77, 130                  # the first 256 keys 48, the others 0: scores of 543 and 0
    c.t[3][:, :, 1, 1500] = 255
    q = torch.ones(1, 4, Dh, dtype=torch.bfloat16, device="cuda")
    n = torch.tensor([S], dtype=torch.int32, device="cuda")
    for out in [hip_ops.attn_decode_kv4(q, *c.t, n, nsplit=nsplit) for nsplit in (None, 1, 3, 8)] + [hip_ops.attn_prefill_kv4(q[:, None], *c.t, n - 1)[:, 0]]:
        nan = out.isnan()
        assert bool(nan[..., 32:64].all()) and not bool(nan[..., :32].any()) and not bool(nan[..., 64:].any())


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_append_forms_are_alike(dt):
    """Many rows at once, four heads of a workgroup, against the same rows in shorter calls."""
    from flashsvd_amd import hip_ops
    for Dh, Hk, B, T, S in ((128, 32, 8, 2048, 2112), (64, 24, 16, 1500, 1620)):
        g = torch.Generator(device="cuda").manual_seed(9)
        k, v = (torch.randn(B, T, Hk, Dh, generator=g, device="cuda").to(dt) for _ in range(2))
        cos, sin = (t.cuda() for t in tables(S, Dh, dt))
        a, b = (Cache(B, S, Hk, Dh, seed=2) for _ in range(2))
        at = torch.arange(B, dtype=torch.int32, device="cuda") * 7
        rows = torch.tensor(([T, T - 1, 70, 0, 1, T, 33, 5] * 2)[:B], dtype=torch.int32, device="cuda")
        hip_ops.kv4_append(k, v, *a.t, at, cos=cos, sin=sin, rows=rows)
        assert form_taken() == "kv4 rows of 4 heads"
        for t in range(0, T, 100):
            hip_ops.kv4_append(k[:, t:t + 100], v[:, t:t + 100], *b.t, at + t, cos=cos, sin=sin, rows=rows - t)
        assert form_taken() == "kv4 rows"
        assert all(torch.equal(x, y) for x, y in zip(a.t, b.t))
        hip_ops.kv4_append(k[:, :1], v[:, :1], *a.t, at, cos=cos, sin=sin)
        assert form_taken() == "kv4 row"


@pytest.mark.parametrize("B,T,V,name", [(600, 1, 2049, "logprobs 256"), (2, 256, 32000, "logprobs 256"), (512, 1, 32769, "logprobs 1024"), (256, 1, 4096, "logprobs 256"), (256, 1, 4097, "logprobs 1024"), (257, 1, 4097, "logprobs 256"),
                                        (1, 1, 32768, "logprobs 1024"), (1, 1, 32769, "logprobs parts"), (1, 2, 131073, "logprobs parts"),
                                        (16, 8, 40001, "logprobs parts"), (129, 1, 40001, "logprobs 1024"), (300, 1, 131073, "logprobs parts"), (1, 1, 2500001, "logprobs long parts")])
def test_logprob_forms(B, T, V, name):
    from flashsvd_amd import hip_ops
    from tests.test_gpu_logprobs import _check
    g = torch.Generator(device="cuda").manual_seed(V)
    x = (torch.randn(B, T, V, generator=g, device="cuda") * 3).to(torch.bfloat16)
    t = torch.randint(0, V, (B, T), generator=g, device="cuda")
    out = hip_ops.token_logprobs(x, t, top=min(9, V))
    assert form_taken() == name
    pick = sorted({0, B // 2, B - 1})
    _check(x[pick], t[pick], min(9, V), [o[pick] for o in out])


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("top", [0, 1, 20, 33, 64])
def test_parts_of_rows_with_ties_masks_and_nans(top, dt):
    """Equal logits across the borders of parts, parts of -inf alone, fewer logits that are not -inf than alternatives, a NaN in one part, an infinity in another."""
    from flashsvd_amd import hip_ops
    from tests.test_gpu_logprobs import _check
    V = 40003
    g = torch.Generator().manual_seed(top)
    x = torch.zeros(9, V)
    x[1] = torch.randn(V, generator=g).mul(2).round()               # many equal ones
    x[2] = -math.inf
    x[2, [3, 20000, 20001, V - 1]] = torch.tensor([1.0, 1.0, 2.0, 1.0])
    x[3] = torch.randn(V, generator=g)
    x[3, :30000] = -math.inf
    x[4] = torch.randn(V, generator=g)
    x[4, 35000] = math.nan
    x[5] = torch.randn(V, generator=g)
    x[5, 100] = math.inf
    x[6] = -math.inf
    x[7] = -0.0
    x[7, ::3] = 0.0
    x[8] = torch.randn(V, generator=g) * 30
    x = x.to(dt).cuda()
    t = torch.tensor([V - 1, 0, 20001, 39999, 35000, 100, 5, -1, V], device="cuda")
    out = hip_ops.token_logprobs(x, t, top=top)
    assert form_taken() == "logprobs parts"
    _check(x, t, top, out)


@pytest.mark.parametrize("Dh", [64, 128])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_rows_of_the_output_at_odd_elements(dt, Dh):
    """Every form of a prompt writes rows of any distance at any element; what stands between them is left as it was."""
    from flashsvd_amd import hip_ops
    B, M, H, Hk = 8, 200, 32, 32
    c = Cache(B, 256, Hk, Dh, seed=61)
    g = torch.Generator(device="cuda").manual_seed(62)
    q = (torch.randn(B, M, H, Dh, generator=g, device="cuda") * 0.7).to(dt)
    names = set()
    for n, rows in ((8, 200), (4, 200), (4, 70), (1, 70), (1, 9)):
        pos = torch.arange(n, dtype=torch.int32, device="cuda") * 3
        args = (q[:n, :rows], *(t[:n] for t in c.t), pos)
        want = hip_ops.attn_prefill_kv4(*args)
        names.add(form_taken())
        into = torch.full((n, rows, H, Dh + 3), 7.0, dtype=dt, device="cuda")
        hip_ops.attn_prefill_kv4(*args, out=into[..., 1:Dh + 1])
        assert torch.equal(into[..., 1:Dh + 1], want) and bool((into[..., 0] == 7).all()) and bool((into[..., Dh + 1:] == 7).all())
    assert names >= {"kv4 prompt 128", "kv4 prompt 64", "kv4 prompt 64 halves"}
