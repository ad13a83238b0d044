"""The draw of a token (csrc/sample.hip) against its definition in 64 bits: whole numbers, so they agree exactly."""
import pytest
import torch

from tests import kv8_reference as R

pytestmark = pytest.mark.gpu


def _draw(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, positions=None):
    from flashsvd_amd import hip_ops
    tokens = torch.full((x.shape[0], 1), -7, dtype=torch.long, device="cuda")
    hip_ops.sample_token_(x, u, tokens, positions, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    return tokens[:, 0].tolist()


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V,off", [(1, 0), (2, 1), (7, 0), (8, 3), (9, 0), (1023, 1), (8192, 0), (8200, 5), (32000, 0), (65537, 2), (128256, 0)])
@pytest.mark.parametrize("filters", [dict(), dict(temperature=0.7, top_k=50, top_p=0.9375, min_p=0.03125), dict(top_k=3), dict(top_p=0.5), dict(min_p=0.25),
                                     dict(temperature=3.0, top_p=0.99), dict(temperature=0.0), dict(top_p=0.0), dict(temperature=1e-9), dict(temperature=1e6, min_p=1.0)])
def test_draw_of_every_row(dt, V, off, filters):
    B = 6
    g = torch.Generator().manual_seed(V + off)
    x = torch.randn(B, V + off + 3, generator=g) * 2.5
    x[1] = x[1].round()                                  # many equal values
    x[2, V // 2] += 12.0                                 # one that nearly always wins
    x = x.to(dt)[:, off:off + V]
    u = torch.tensor([0.0, 0.5, 0.25, 1 - 2.0 ** -24, 0.9, 0.37])
    pos = torch.arange(B, dtype=torch.int32, device="cuda")
    wide = torch.zeros(B, V + off + 3, dtype=dt, device="cuda")
    wide[:, off:off + V] = x.cuda()
    got = _draw(wide[:, off:off + V], u.cuda(), positions=pos, **filters)
    full = dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) | filters
    assert got == [R.draw(x[b], float(u[b]), **full) for b in range(B)]
    assert pos.tolist() == list(range(1, B + 1))


def test_filters_of_every_row():
    B, V = 64, 5003
    g = torch.Generator().manual_seed(2)
    x = (torch.randn(B, V, generator=g) * 3).to(torch.bfloat16)
    r = torch.rand(5, B, generator=g)
    u, t, k, p, m = r[0], 2 * r[1] - 0.2, (r[2] * 200 - 60).int(), r[3] * 1.2, (r[4] - 0.6).clamp_min(0.0)
    got = _draw(x.cuda(), u.cuda(), t.cuda(), k.cuda(), p.cuda(), m.cuda())
    assert got == [R.draw(x[b], *(float(v[b]) for v in (u, t)), int(k[b]), float(p[b]), float(m[b])) for b in range(B)]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V", [5, 4096, 70001, 200003])
def test_rows_that_are_not_ordinary(dt, V):
    """Equal logits (more of them than 16 bits count), only masked ones, masks of -inf and of the lowest value, zeros of both signs, NaN, infinities, and
    values from the smallest to the largest of the type."""
    fi = torch.finfo(dt)
    x = torch.zeros(12, V)
    x[1] = -3.0
    x[2] = float("-inf")
    x[3, :] = float("-inf")
    x[3, V // 2:] = 1.0
    x[4] = fi.min
    x[4, [1, V - 1]] = 2.0
    x[5, ::2] = -0.0
    x[6] = torch.randn(V, generator=torch.Generator().manual_seed(1))
    x[6, V - 2] = float("nan")
    x[7] = x[6].nan_to_num()
    x[7, [V // 3, V - 1]] = float("inf")
    x[8] = fi.max
    x[8, 0] = fi.min
    x[9] = torch.linspace(-1, 1, V) * fi.tiny
    x[10] = fi.min                                       # nothing but the lowest finite value
    x[11] = torch.where(torch.arange(V) % 3 == 0, 1.0, 0.5)
    x = x.to(dt)
    for u in (0.0, 0.5, 0.75, 1 - 2.0 ** -24):
        for f in (dict(), dict(top_p=0.5), dict(top_k=V - 1, min_p=0.5, temperature=0.5)):
            full = dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) | f
            got = _draw(x.cuda(), torch.full((12,), u, device="cuda"), **f)
            assert got == [R.draw(x[b], u, **full) for b in range(12)], (u, f)


def test_shares_follow_the_weights():
    """Draws at evenly spread numbers hit every kept token as often as its weight says, to one draw."""
    V, n = 257, 4096
    x = (torch.randn(1, V, generator=torch.Generator().manual_seed(5)) * 1.5).to(torch.float16)
    u = (torch.arange(n, dtype=torch.float32) + 0.5) / n
    got = torch.tensor(_draw(x.expand(n, V).contiguous().cuda(), u.cuda(), top_k=100))
    w = torch.exp(x[0].double())
    w[torch.sort(x[0].double(), descending=True, stable=True).indices[100:]] = 0
    share = w / w.sum() * n
    assert float((torch.bincount(got, minlength=V).double() - share).abs().max()) <= 1.0
