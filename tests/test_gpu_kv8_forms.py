"""Every kernel form of the KV cache in 8 bits and of the draw of a token, by name: shapes on either side of each rule, against the definitions in 64 bits."""
import pytest
import torch

from tests import kv8_reference as R
from tests import test_gpu_kv8 as base
from tests.test_gpu_kv8 import Cache, _close, _same, half_step, tables
from tests.test_gpu_kv8_accuracy import TWO_PARTS
from tests.test_gpu_sample import _draw
from tests.util import form_taken

pytestmark = pytest.mark.gpu

# what a call takes, its name, and rows of a sequence that are real (of M)
PROMPTS = [
    ("kv8 prompt 128", dict(B=8, Hk=32, G=1, M=130, past=7, rows=[130, 129, 128, 65, 64, 1, 0, 130])),
    ("kv8 prompt 128", dict(B=16, Hk=16, G=2, M=70, past=40, rows=None)),
    ("kv8 prompt 128", dict(B=1, Hk=8, G=6, M=1400, past=300, rows=None)),
    ("kv8 prompt 64", dict(B=8, Hk=25, G=1, M=70, past=33, rows=[70, 64, 63, 17, 16, 1, 0, 70])),
    ("kv8 prompt 64", dict(B=2, Hk=5, G=3, M=850, past=0, rows=None)),
    ("kv8 prompt 64 halves", dict(B=2, Hk=2, G=2, M=40, past=90, rows=[39, 40])),
    ("kv8 prompt 64 halves", dict(B=3, Hk=32, G=1, M=256, past=0, rows=None)),
    ("kv8 prompt 64 halves ranges", dict(B=1, Hk=2, G=3, M=21, past=1200, rows=None)),
    ("kv8 prompt 64 halves ranges", dict(B=3, Hk=1, G=1, M=64, past=700, rows=[64, 2, 0])),
]


def _q_error(x, y, k, dt):
    """Error of a q that the call rotates to y as two parts of its type, relative to the sums |k| |y| of its scores: 2^-2p of an element for the second
    rounding, and 2^-22 of the rotated pair for the rotation in fp32."""
    pair = x.double().abs()
    pair = pair + pair.roll(len(x) // 2)
    k = k.abs()
    return half_step(dt) ** 2 + 2.0 ** -22 * float(((k @ pair) / (k @ y.abs()).clamp_min(1e-30)).max())


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Dh,block", [(64, 16), (128, 32), (128, 128)])
@pytest.mark.parametrize("turn", [False, True])
@pytest.mark.parametrize("name,p", PROMPTS)
def test_prompt_forms(name, p, turn, Dh, block, dt):
    """Rows of unequal numbers, NaN in every row that none sees, an out whose rows stand at odd elements, scores with and without a rotation."""
    from flashsvd_amd import hip_ops
    B, Hk, M, past, H = p["B"], p["Hk"], p["M"], p["past"], p["Hk"] * p["G"]
    n = p["rows"] or [M] * B
    c = Cache(B, past + M, Hk, Dh, block, seed=M + Dh).finite()
    base._spoil(c, [past + t for t in n])
    g = torch.Generator().manual_seed(71)
    q = (torch.randn(B, M, H, Dh, generator=g) * 0.7).to(dt)
    cos, sin = tables(past + M, Dh, dt) if turn else (None, None)
    into = torch.full((B, M, H, Dh + 3), 7.0, dtype=dt, device="cuda")
    hip_ops.attn_prefill_kv8(q.cuda(), *c.t, torch.full((B,), past, dtype=torch.int32, device="cuda"), block=block,
                             rows=None if p["rows"] is None else torch.tensor(n, dtype=torch.int32, device="cuda"),
                             cos=cos.cuda() if turn else None, sin=sin.cuda() if turn else None, out=into[..., 1:Dh + 1])
    assert form_taken() == name
    out = into.cpu()
    assert bool((out[..., 0] == 7).all() and (out[..., Dh + 1:] == 7).all())
    for b in range(B):
        assert bool((out[b, n[b]:] == 7).all()), "rows behind the last one"
    k, v = c.values()
    picked = {(b, m, (7 * b + m) % H) for b in {0, B // 2, B - 1} for m in (0, 1, 15, 16, 63, 64, 127, 128, M // 2, M - 1) if m < n[b]}
    for b, m, h in sorted(picked):
        x, hk, end = q[b, m, h], h // p["G"], past + m + 1
        y = R.rotate(x.double(), cos, sin, past + m)
        kk = k[b, :end, hk]
        want, room = R.attend(y, kk, v[b, :end, hk], Dh ** -0.5, _q_error(x, y, kk, dt) if turn else 0.0, TWO_PARTS)
        _close(out[b, m, h, 1:Dh + 1], want, room, dt, f"row {m} of sequence {b}, head {h}")


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Dh", [64, 128])
@pytest.mark.parametrize("name,H,Hk,M,start,B", [("kv8 prompt 128", 32, 32, 130, 3, 8), ("kv8 prompt 128", 32, 16, 70, 40, 16), ("kv8 prompt 64", 25, 25, 70, 33, 8),
                                                 ("kv8 prompt 64", 50, 25, 40, 33, 8)])
def test_a_nan_stays_in_what_sees_it_in_every_form(name, H, Hk, M, start, B, Dh, dt):
    from flashsvd_amd import hip_ops
    c = Cache(B, start + M, Hk, Dh, 16, seed=41).finite()
    hip_ops.attn_prefill_kv8(torch.zeros(B, M, H, Dh, dtype=dt, device="cuda"), *c.t, torch.full((B,), start, dtype=torch.int32, device="cuda"), block=16)
    assert form_taken() == name
    base.test_a_nan_stays_in_what_sees_it(Dh=Dh, H=H, Hk=Hk, M=M, start=start, B=B, dt=dt)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("name,Dh,Hk,block,T,at,rows", [
    ("kv8 rows 4", 128, 2, 128, 150, [0, 5, 127, 128, 200, -30, 260], None),
    ("kv8 rows 4", 128, 1, 128, 300, [0, 1, 90, 100, 50, 255, 0], [300, 0, 127, 128, 1, 300, 129]),
    ("kv8 rows 2", 128, 2, 64, 131, [0, 63, 64, 65, 260, 10, 200], None),
    ("kv8 rows 2", 64, 3, 128, 129, [0, 5, 127, 128, 200, 17, 260], [129, 128, 1, 127, 100, 0, 5]),
    ("kv8 rows 1", 128, 2, 32, 100, [0, 31, 32, 33, 250, 7, 100], None),
    ("kv8 rows 1", 64, 1, 16, 77, [0, 1, 15, 16, 250, 240, 9], [77, 76, 1, 2, 40, 0, 16]),
])
def test_append_forms(name, Dh, Hk, block, T, at, rows, dt):
    """Rows over several workgroups, blocks that are open in front and left open behind."""
    from flashsvd_amd import hip_ops
    B, S = len(at), 300
    c = Cache(B, S, Hk, Dh, block, seed=T + Dh)
    g = torch.Generator().manual_seed(73)
    k = (torch.randn(B, T, Hk, Dh, generator=g) * torch.exp2(torch.randint(-3, 3, (B, T, Hk, 1), generator=g).float())).to(dt)
    v = torch.randn(B, T, Hk, Dh, generator=g).to(dt)
    want = c.doubles()
    for b in range(B):
        for x, i in ((k, 0), (v, 1)):
            R.append(want[i][b], want[i + 2][b], x[b], at[b], T if rows is None else rows[b], block)
    hip_ops.kv8_append(k.cuda(), v.cuda(), *c.t, torch.tensor(at, dtype=torch.int32, device="cuda"), block=block,
                       rows=None if rows is None else torch.tensor(rows, dtype=torch.int32, device="cuda"))
    assert form_taken() == name
    for got, w, what in zip(c.doubles(), want, ("k", "v", "k_scale", "v_scale")):
        assert _same(got, w), f"{what}: {int((got != w).sum())} of {w.numel()} differ"


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Dh,H,Hk,lens,S,splits", [
    (128, 8, 4, [8450], 8470, {None: 67, 65: 65, 64: 64, 9: 9, 8: 8, 1: 1}),
    (64, 4, 1, [8700, 0, 130], 8701, {65: 65, 66: 66, 67: 67, 68: 68}),
    (128, 2, 2, [16500, 8300], 16500, {None: 128, 129: 129}),
])
def test_decode_over_many_ranges(Dh, H, Hk, lens, S, splits, dt):
    """More ranges than a wave has lanes, with one to four in the last pass of the join."""
    from flashsvd_amd import hip_ops
    B = len(lens)
    c = Cache(B, S, Hk, Dh, 32, seed=S).finite()
    base._spoil(c, lens)
    g = torch.Generator().manual_seed(74)
    q = (torch.randn(B, H, Dh, generator=g) * 0.7).to(dt)
    k, v = c.values()
    rooms = {(b, h): R.attend(q[b, h].double(), k[b, :n, h * Hk // H], v[b, :n, h * Hk // H], Dh ** -0.5, 0.0, TWO_PARTS) for b, n in enumerate(lens) for h in range(H)}
    for nsplit, ranges in splits.items():
        out = hip_ops.attn_decode_kv8(q.cuda(), *c.t, torch.tensor(lens, dtype=torch.int32, device="cuda"), block=32, nsplit=nsplit).cpu()
        assert form_taken() == "kv8 decode" + ("" if ranges == 1 else " ranges" if ranges <= 8 else " ranges 9" if ranges <= 64 else " ranges 65")
        for (b, h), (want, room) in rooms.items():
            _close(out[b, h], want, room, dt, f"{lens[b]} keys of head {h} in {ranges}")


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V,name", [(16384, "draw 2"), (16385, "draw 4"), (32768, "draw 4"), (32769, "draw 8"), (50257, "draw 8"), (65535, "draw 8"),
                                    (65536, "draw 16"), (131072, "draw 16"), (131073, "draw")])
def test_draw_forms(V, name, dt):
    """Rows at the ends of each form: spread logits, all of them equal, two values, and one that stands alone at the end."""
    g = torch.Generator().manual_seed(V)
    x = torch.randn(5, V, generator=g) * 2.5
    x[1] = -1.5
    x[2] = torch.where(torch.arange(V) % 3 == 0, 1.0, 0.5)
    x[3] = 0.25
    x[3, V - 1] = 30.0
    x = x.to(dt)
    for u in (0.0, 0.3, 0.75, 1 - 2.0 ** -24):
        for f in (dict(), dict(top_p=0.9, top_k=V - 2, temperature=0.8), dict(min_p=0.02)):
            got = _draw(x.cuda(), torch.full((5,), u, device="cuda"), **f)
            assert form_taken() == name
            full = dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) | f
            assert got == [R.draw(x[b], u, **full) for b in range(5)], (u, f)
