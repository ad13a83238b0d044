"""Log probabilities of given tokens, entropies and the likeliest alternatives (csrc/logprobs.hip) against their definition in 64 bits."""
import math

import pytest
import torch

from tests import kv4_reference as R

pytestmark = pytest.mark.gpu


def _room(x, value, entropy):
    """How far an fp32 result may be from the exact one.  Weights are off by 2^-21 of themselves or less (2^-23 |x| e^x for the rounding of an argument x <= 0, and the
    exponential's own), their sums by 2^-24 for each of the V / 256 + 16 additions in a row, the logarithm of the sum by that and its own rounding; a log
    probability by half a step of each of two subtractions besides.  The entropy also has the mean of |x|, up to log V and the entropy in size, from two sums."""
    V = x.numel()
    rel = 2.0 ** -21 + 2.0 ** -24 * (V / 256 + 16)
    size = math.log(V) + 1 + abs(value)
    return rel * (1 + 2 * size) + 2.0 ** -22 * size if entropy else rel + 2.0 ** -22 * size


def _check(logits, tokens, top, out):
    rows, ids = logits.cpu().flatten(0, -2), tokens.cpu().flatten()
    lp, ent, best, best_lp = (o.cpu() for o in out)
    assert lp.shape == ent.shape == tokens.shape and best.shape == best_lp.shape == (*tokens.shape, top)
    lp, ent, best, best_lp = lp.flatten(), ent.flatten(), best.view(len(rows), top), best_lp.view(len(rows), top)
    for i in range(len(rows)):
        a, h, order, b = R.logprobs(rows[i], int(ids[i]), top)
        assert best[i].tolist() == order.tolist(), f"row {i}"
        x = rows[i].double()
        for got, want, kind in [(float(lp[i]), a, False), (float(ent[i]), h, True), *((y, z, False) for y, z in zip(best_lp[i].tolist(), b.tolist()))]:
            if math.isfinite(want):
                assert abs(got - want) <= _room(x, want, kind), f"row {i}: {got} for {want}"
            else:
                assert got == want or (math.isnan(got) and math.isnan(want)), f"row {i}: {got} for {want}"


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,V,top", [(1, 1, 1), (1, 2, 0), (3, 7, 7), (2, 63, 5), (5, 64, 64), (4, 257, 20), (3, 1000, 1), (2, 2049, 64), (2, 8191, 33), (1, 32000, 20),
                                     (2, 32001, 5), (2, 50257, 3), (1, 65536, 64), (2, 128256, 20), (1, 200003, 7)])
def test_against_the_definition(dt, N, V, top):
    from flashsvd_amd import hip_ops
    g = torch.Generator().manual_seed(V + top)
    x = (torch.randn(N, V + 3, generator=g) * 3).to(dt).cuda()[:, 1:V + 1]        # rows at odd elements, of odd distances
    t = torch.randint(0, V, (N,), generator=g).cuda()
    _check(x, t, top, hip_ops.token_logprobs(x, t, top=top))


@pytest.mark.parametrize("V", [300, 4096, 40000, 150000])
def test_ties_go_to_the_lowest_index(V):
    """Rows of few values, so that the alternatives are chosen by index alone; all equal; the ones at the ends."""
    from flashsvd_amd import hip_ops
    g = torch.Generator().manual_seed(V)
    x = torch.stack((torch.randint(-2, 2, (V,), generator=g).float(), torch.zeros(V), -torch.zeros(V), torch.arange(V) // (V // 3 + 1) * 1.0,
                     torch.where(torch.arange(V) % 2 == 0, 0.0, -0.0), -torch.arange(V).float().clamp_max(20.0))).to(torch.bfloat16)
    t = torch.tensor([0, V - 1, 5, V // 2, 1, 2])
    _check(x.cuda(), t.cuda(), 64, hip_ops.token_logprobs(x.cuda(), t.cuda(), top=64))


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V", [40, 5000, 70000])
def test_numbers_that_are_none(dt, V):
    """-inf has no weight; a row with a NaN or infinity, or of -inf alone, has no distribution but an order; a token below 0 is none, one from V on has none."""
    from flashsvd_amd import hip_ops
    g = torch.Generator().manual_seed(V)
    x = torch.randn(9, V, generator=g)
    x[0, ::2] = -math.inf
    x[1, 5:] = -math.inf                                    # five left, and alternatives among the others
    x[2] = -math.inf
    x[3, 17] = math.inf
    x[4, 3], x[4, 9] = math.nan, math.inf
    x[5, V - 1] = math.nan
    x[6] = torch.finfo(dt).min                              # the type's lowest value as a mask, and one that stands out
    x[7] = torch.finfo(dt).min
    x[7, 11] = 1.0
    x = x.to(dt)
    x.view(torch.int16)[4, 30] = -1                         # a NaN with its sign set
    t = torch.tensor([0, 1, 0, 17, 2, 1, 3, 11, 4])
    _check(x.cuda(), t.cuda(), 20, hip_ops.token_logprobs(x.cuda(), t.cuda(), top=20))
    t = torch.tensor([-1, -100, V, V + 7, -5, 2 ** 40, -2 ** 40, -1, V - 1])
    _check(x.cuda(), t.cuda(), 0, hip_ops.token_logprobs(x.cuda(), t.cuda()))


def test_a_sharp_distribution_and_wide_numbers():
    """One token far above the rest, rows of large offsets, and rows whose logits span the type."""
    from flashsvd_amd import hip_ops
    g = torch.Generator().manual_seed(5)
    V = 32000
    x = torch.randn(4, V, generator=g)
    x[0, 777] = 40.0
    x[1] += 30000.0
    x[2] *= 10000.0
    x[3] = -60000.0 + x[3] * 8
    for dt in (torch.bfloat16, torch.float16):
        y = x.to(dt).cuda()
        t = torch.tensor([777, 5, 6, 7]).cuda()
        _check(y, t, 10, hip_ops.token_logprobs(y, t, top=10))


def test_rows_of_a_longer_tensor_and_streams():
    """[B, T, V] with rows of other tokens between, tokens of their own strides, a stream of its own, and a captured call."""
    from flashsvd_amd import hip_ops
    g = torch.Generator().manual_seed(6)
    whole = (torch.randn(3, 6, 900, generator=g) * 2).to(torch.bfloat16).cuda()
    x, t = whole[:, :-1, 4:], torch.randint(0, 896, (5, 3), generator=g).cuda().t()
    want = hip_ops.token_logprobs(x, t, top=4)
    _check(x, t, 4, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = hip_ops.token_logprobs(x, t, top=4)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph, static = torch.cuda.CUDAGraph(), x.contiguous()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = hip_ops.token_logprobs(static, t, top=4)
    for i in range(3):
        static.copy_(x.roll(i, -1))
        graph.replay()
        eager = hip_ops.token_logprobs(static, t, top=4)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager))


def test_many_rows():
    """The bounds of _room for 777 logits, log probabilities down to -20 and entropies up to log 777."""
    from flashsvd_amd import hip_ops
    g = torch.Generator(device="cuda").manual_seed(7)
    x = (torch.randn(3000, 777, generator=g, device="cuda") * 2).to(torch.float16)
    t = torch.randint(0, 777, (3000,), generator=g, device="cuda")
    lp, ent, ids, best = hip_ops.token_logprobs(x, t, top=3)
    ref = torch.log_softmax(x.double(), 1)
    assert float((lp.double() - ref.gather(1, t[:, None])[:, 0]).abs().max()) < 9e-6
    assert float((ent.double() + (ref.exp() * ref).sum(1)).abs().max()) < 5.2e-5
    order = torch.sort(x.double(), dim=1, descending=True, stable=True).indices[:, :3]
    assert torch.equal(ids, order) and float((best.double() - ref.gather(1, order)).abs().max()) < 9e-6


@pytest.mark.parametrize("V,top", [(1000, 5), (70000, 20)])
def test_captured_and_replayed(V, top):
    """One workgroup a row and rows in parts, whose scratch is the graph's; other calls of the program between the replays."""
    from flashsvd_amd import hip_ops
    g = torch.Generator().manual_seed(V)
    rows = [(torch.randn(3, V, generator=g) * 3).to(torch.bfloat16).cuda() for _ in range(4)]
    ids = [torch.randint(-1, V, (3,), generator=g).cuda() for _ in range(4)]
    x, t = rows[0].clone(), ids[0].clone()
    hip_ops.token_logprobs(x, t, top=top)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = hip_ops.token_logprobs(x, t, top=top)
    for a, b in zip(rows, ids):
        x.copy_(a)
        t.copy_(b)
        graph.replay()
        other = hip_ops.token_logprobs(a.flip(0).contiguous(), b.flip(0), top=top)
        torch.cuda.synchronize()
        want = hip_ops.token_logprobs(a, b, top=top)
        for got, w, o in zip(out, want, other):
            assert torch.equal(got, w) and torch.equal(o.flip(0), w)
