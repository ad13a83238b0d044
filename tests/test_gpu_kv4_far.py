"""The KV cache in 4 bits where its rows, heads, groups and sequences lie further apart than 32 bits count: the same bits as over one whose rows lie side by side."""
import pytest
import torch

from tests.test_gpu_kv4 import Cache
from tests.test_gpu_kv8 import tables
from tests.util import form_taken

pytestmark = pytest.mark.gpu

B, S, Hk, Dh = 3, 320, 2, 128
LAYOUTS = {
    "tokens": ((128, 1 << 24, 64), (2048, 1024, 1 << 28)),                        # the most that a token and a group may be apart
    "sequences": (((1 << 31) + 4096, 64, S * 64), ((1 << 31) + 64, 4 * S, S)),
    "heads": ((64 * S, 64, (1 << 32) + 64), (4 * S, (1 << 32) + 16, S)),
}


def _apart(tensors, layout):
    """The four tensors of a cache, copied into views whose strides are the layout's."""
    (sb, ss, sh), (gb, gh, gg) = LAYOUTS[layout]
    strides = [(sb, ss, sh, 1)] * 2 + [(gb, gh, gg, 1)] * 2
    out = []
    for t, st in zip(tensors, strides):
        store = torch.empty(sum((n - 1) * s for n, s in zip(t.shape, st)) + 1, dtype=torch.uint8, device="cuda")
        view = store.as_strided(t.shape, st)
        view.copy_(t)
        out.append(view)
    return out


@pytest.mark.parametrize("layout", list(LAYOUTS))
def test_far_apart(layout):
    from flashsvd_amd import hip_ops
    near = [t.contiguous() for t in Cache(B, S, Hk, Dh, seed=5).t]
    far = _apart(near, layout)
    g = torch.Generator().manual_seed(6)
    cos, sin = (t.cuda() for t in tables(S, Dh, torch.bfloat16))
    kw = dict(cos=cos, sin=sin)
    rand = lambda *shape: torch.randn(*shape, generator=g).to(torch.bfloat16).cuda()      # noqa: E731
    for T, at in ((300, [0, 20, 7]), (1, [319, 0, 200]), (9, [311, 100, -3])):
        k, v, pos = rand(B, T, Hk, Dh), rand(B, T, Hk, Dh), torch.tensor(at, dtype=torch.int32, device="cuda")
        for c in (near, far):
            hip_ops.kv4_append(k, v, *c, pos, **kw)
        assert all(torch.equal(a, b) for a, b in zip(near, far))
    for a, b in zip(hip_ops.kv4_dequantize(*near), hip_ops.kv4_dequantize(*far)):
        assert torch.equal(a, b)
    lens = torch.tensor([300, 319, 64], dtype=torch.int32, device="cuda")
    for H in (2, 8, 24, 64):
        q, k, v = rand(B, H, Dh), rand(B, Hk, Dh), rand(B, Hk, Dh)
        for nsplit in (1, 2):
            a, b = (hip_ops.attn_decode_kv4(q, *c, lens, k_new=k, v_new=v, nsplit=nsplit, **kw) for c in (near, far))
            assert torch.equal(a, b)
        assert all(torch.equal(x, y) for x, y in zip(near, far))
    forms = set()
    for M, H, at in ((1, 2, [319, 0, 100]), (70, 2, [250, 0, 31]), (300, 8, [20, 0, 7]), (300, 64, [20, 0, 7])):
        q, pos = rand(B, M, H, Dh), torch.tensor(at, dtype=torch.int32, device="cuda")
        a, b = (hip_ops.attn_prefill_kv4(q, *c, pos, **kw) for c in (near, far))
        forms.add(form_taken())
        assert torch.equal(a, b)
    assert "kv4 prompt 128" in forms and any(f.startswith("kv4 prompt 64") for f in forms)
