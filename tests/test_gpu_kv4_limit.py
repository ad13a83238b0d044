"""Rows from the limit on in a cache in 4 bits, whose room is rounded up: dropped by every form that writes, seen by none that reads, in the operators and in a
model that decodes to the end of its cache and beyond."""
import pytest
import torch

from tests.test_gpu_kv4 import Cache, _check_rows
from tests.test_gpu_kv8 import tables
from tests.test_gpu_kv8_model import _model
from tests.util import form_taken

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("Dh", [64, 128])
@pytest.mark.parametrize("T,Hk,form", [(1, 2, "kv4 row"), (9, 2, "kv4 rows"), (600, 32, "kv4 rows of 4 heads")])
@pytest.mark.parametrize("limit", [1, 70, 127, 128])
def test_append(limit, T, Hk, form, Dh):
    from flashsvd_amd import hip_ops
    B, dt = 32 if T == 600 else 4, torch.bfloat16
    room = 128 if T < 600 else 704
    limit += room - 128
    c, whole = (Cache(B, room, Hk, Dh, seed=1) for _ in range(2))
    g = torch.Generator(device="cuda").manual_seed(2)
    k, v = (torch.randn(B, T, Hk, Dh, generator=g, device="cuda").to(dt) for _ in range(2))
    at = torch.tensor([limit - 1, limit, room - 1, 0] * (B // 4), dtype=torch.int32, device="cuda")
    hip_ops.kv4_append(k, v, *whole.t, at)
    want = [t.clone() for t in c.t]
    for w, t in zip(want[:2], whole.t[:2]):
        w[:, :limit] = t[:, :limit]
    for w, t in zip(want[2:], whole.t[2:]):
        w[..., :limit] = t[..., :limit]
    hip_ops.kv4_append(k, v, *c.t, at, limit=limit)
    assert form_taken() == form
    assert all(torch.equal(a, b) for a, b in zip(c.t, want))


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Dh,H,Hk", [(128, 4, 2), (64, 12, 1), (128, 20, 1)])
@pytest.mark.parametrize("limit", [1, 65, 1000, 1024])
def test_decode(limit, Dh, H, Hk, dt):
    """Rows behind the limit are NaN and seen by no query; a token there is dropped and sees what lies before."""
    from flashsvd_amd import hip_ops
    at = [0, limit - 1, limit, 1023, 5000, -1]
    B, S = len(at), 1024
    cos, sin = tables(S, Dh, dt)
    g = torch.Generator().manual_seed(12)
    q, k, v = ((torch.randn(B, h, Dh, generator=g) * f).to(dt) for h, f in ((H, 0.7), (Hk, 4.0), (Hk, 1.0)))
    pos = torch.tensor(at, dtype=torch.int32, device="cuda")
    kw = dict(cos=cos.cuda(), sin=sin.cuda(), limit=limit)
    for nsplit in (None, 1, 3):
        c, other = (Cache(B, S, Hk, Dh, seed=11) for _ in range(2))
        for x in (c, other):
            x.spoil([limit] * B)
        held = [t.clone() for t in c.t]
        out = hip_ops.attn_decode_kv4(q.cuda(), *c.t, pos, k_new=k.cuda(), v_new=v.cuda(), nsplit=nsplit, **kw)
        hip_ops.kv4_append(k.cuda()[:, None], v.cuda()[:, None], *other.t, pos, **kw)
        assert all(torch.equal(x, y) for x, y in zip(c.t, other.t))
        for b, n in enumerate(at):
            assert torch.equal(c.t[0][b], held[0][b]) == (not 0 <= n < limit)
        _check_rows(c, q, out, [(b, min(n + 1, limit)) for b, n in enumerate(at)], Dh ** -0.5, dt, cos, sin, at, f"{nsplit} ranges")
        again = hip_ops.attn_decode_kv4(q.cuda(), *c.t, pos, seqlen_add=1, nsplit=nsplit, **kw)
        _check_rows(c, q, again, [(b, min(n + 1, limit)) for b, n in enumerate(at)], Dh ** -0.5, dt, cos, sin, at, "behind an append")


@pytest.mark.parametrize("Dh", [64, 128])
@pytest.mark.parametrize("B,Hk,G,M,past,name", [(8, 32, 1, 130, 20, "kv4 prompt 128"), (1, 8, 4, 300, 4400, "kv4 prompt 128 ranges"), (8, 25, 1, 70, 33, "kv4 prompt 64"),
                                                (2, 2, 2, 40, 90, "kv4 prompt 64 halves"), (1, 2, 3, 21, 1200, "kv4 prompt 64 halves ranges")])
def test_prompts(B, Hk, G, M, past, name, Dh):
    from flashsvd_amd import hip_ops
    dt, H = torch.bfloat16, Hk * G
    c = Cache(B, past + M, Hk, Dh, seed=M)
    g = torch.Generator().manual_seed(13)
    q = (torch.randn(B, M, H, Dh, generator=g) * 0.7).to(dt)
    pos = torch.full((B,), past, dtype=torch.int32, device="cuda")
    limit = past + M // 2 + 1
    c.spoil([limit] * B)
    out = hip_ops.attn_prefill_kv4(q.cuda(), *c.t, pos, limit=limit).cpu()
    assert form_taken() == name
    picked = [(b, m) for b in {0, B - 1} for m in (0, M // 2, M - 1)]
    _check_rows(c, torch.stack([q[b, m] for b, m in picked]), torch.stack([out[b, m] for b, m in picked]), [(b, min(past + m + 1, limit)) for b, m in picked], Dh ** -0.5,
                dt, what=name, heads=sorted({0, H - 1}))
    assert bool(hip_ops.attn_prefill_kv4(q.cuda(), *c.t, pos).isnan().any())


@pytest.mark.parametrize("captured", [False, True])
def test_a_model_at_the_end_of_its_cache(captured):
    """A step at a position behind max_cache_len, which only a caller of decode_step can make, changes nothing and sees the cache as it is."""
    from flashsvd_amd import hip_ops
    from flashsvd_amd.graphs import GraphedDecoder
    from flashsvd_amd.runtime.cache import FlashSVDKV4Cache
    model, S, T = _model(128), 70, 70
    ids = torch.randint(0, 512, (2, T), generator=torch.Generator().manual_seed(2)).cuda()
    c = FlashSVDKV4Cache(model.config, max_batch_size=2, max_cache_len=S, device="cuda", dtype=torch.bfloat16)
    model(ids, past_key_values=c, cache_position=torch.arange(T))
    held = [t.clone() for i in range(2) for t in c.operands(i, 2)]
    token = torch.full((2, 1), 7, device="cuda")
    seen, run = [], hip_ops.attn_decode_kv4

    def watched(q, *a, **k):
        out = run(q, *a, **k)
        turn = {n: k[n] for n in ("cos", "sin")}
        seen.append((out, run(q, *a[:4], torch.full_like(a[4], S), **turn)))
        return out

    if captured:
        dec = GraphedDecoder(model, c, 2)
        dec.set_state(token, S - 1)
        dec.capture()                                       # its warm-ups lie behind the room
        for at in ([S, 75], [127, S]):
            dec.positions.copy_(torch.tensor(at, dtype=torch.int32))
            dec.graph.replay()
        with pytest.raises(IndexError, match="outside the cache"):
            dec.set_state(token, S)
    else:
        hip_ops.attn_decode_kv4 = watched
        try:
            for at in ([S, 75], [127, 128], [S, 5000]):
                model.decode_step(token, c, torch.tensor(at, dtype=torch.int32, device="cuda"))
        finally:
            hip_ops.attn_decode_kv4 = run
        for out, want in seen:                              # positions behind the tables take their last row
            assert torch.equal(out, want)
    assert all(torch.equal(a, b) for a, b in zip(held, [t for i in range(2) for t in c.operands(i, 2)]))
