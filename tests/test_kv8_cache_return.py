"""A cache in 8 bits whose caller goes back to an earlier position: the rows behind the last one written are given up, in what update() returns and in the
length that the next call continues from.  The append itself is the definition in 64 bits, so no GPU is needed."""
from types import SimpleNamespace

import pytest
import torch

from tests import kv8_reference as R

BF16 = torch.bfloat16


@pytest.fixture
def cache(monkeypatch):
    from flashsvd_amd import hip_ops
    from flashsvd_amd.runtime import FlashSVDKV8Cache

    def append(k, v, k_cache, v_cache, k_scale, v_scale, positions, *, block, cos=None, sin=None, rows=None):
        for x, codes, scales in ((k, k_cache, k_scale), (v, v_cache, v_scale)):
            for b in range(x.shape[0]):
                c, s = codes[b].float().double(), scales[b].double()
                R.append(c, s, x[b], int(positions[b]), x.shape[1], block)
                codes[b].view(torch.uint8).copy_(c.to(codes.dtype).view(torch.uint8))
                scales[b].copy_(s)

    monkeypatch.setattr(hip_ops, "kv8_append", append)
    return FlashSVDKV8Cache(SimpleNamespace(num_hidden_layers=2, rope_theta=10000.0), max_batch_size=2, max_cache_len=64, block_size=16, dtype=BF16)


def _rows(n, size, seed):
    g = torch.Generator().manual_seed(seed)
    return [((torch.rand(2, 3, n, 64, generator=g) + 0.5) * size).to(BF16) for _ in range(2)]


@pytest.mark.parametrize("layers", [(0, 1), (1, 0)])
@pytest.mark.parametrize("back,n,size", [(0, 1, 1000.0), (0, 5, 0.001), (16, 3, 500.0), (21, 4, 300.0), (21, 1, 1e-3), (39, 1, 77.0)])
def test_update_returns_what_is_still_valid(cache, back, n, size, layers):
    """Every row returned is within a half step of a code (2^-4 of the value, 2^-10 of the block's scale) for each time it was rounded: once, and once more
    where its block moved to a larger scale."""
    held = {i: _rows(40, 1.0, seed=i) for i in layers}
    for i in layers:
        cache.update(*held[i], i, {"cache_position": torch.arange(40)})
    for i in layers:
        new = _rows(n, size, seed=9 + i)
        got = cache.update(*new, i, {"cache_position": torch.arange(back, back + n)})
        assert got[0].shape == got[1].shape == (2, 3, back + n, 64)
        for x, old, rows, scale in zip(got, held[i], new, (cache.key_scale[i], cache.value_scale[i])):
            want = torch.cat((old[:, :, :back], rows), 2).double()
            steps = scale.double().transpose(1, 2).repeat_interleave(16, 2)[:, :, :back + n, None]
            assert bool(((x.double() - want).abs() <= 2 * (want.abs() * 2.0 ** -4 + steps * 2.0 ** -10)).all())
    assert cache.get_seq_length() == back + n


def test_length_follows_the_last_write(cache):
    cache.update(*_rows(30, 1.0, 1), 0)
    assert cache.get_seq_length() == 30
    cache.update(*_rows(7, 1.0, 2), 0)                     # without positions: from the start
    assert cache.get_seq_length() == 7
    cache.update(*_rows(2, 1.0, 3), 1, {"cache_position": torch.arange(7, 9)})
    assert cache.get_seq_length() == 7                     # layer 0 counts
    cache.update(*_rows(2, 1.0, 3), 0, {"cache_position": torch.arange(7, 9)})
    assert cache.get_seq_length() == 9
    for at, want in ((None, 10), (torch.tensor([4]), 5), (torch.tensor([6, 8]), 9), (3, 4)):
        cache.advance_after_fa2(1, q_len=1, cache_position=at)
        cache.advance_after_fa2(0, q_len=1, cache_position=at)
        assert cache.get_seq_length() == want
    cache._note_seen(0, 5, torch.arange(2, 7))
    assert cache.get_seq_length() == 7
    none = cache.update(*_rows(0, 1.0, 4), 0)               # no rows: nothing is written, nothing given up
    assert none[0].shape == (2, 3, 0, 64) and cache.get_seq_length() == 7
    with pytest.raises(ValueError, match="consecutive"):
        cache.update(*_rows(2, 1.0, 3), 0, {"cache_position": torch.arange(0)})


@pytest.mark.gpu
def test_a_model_continues_from_where_it_went_back_to():
    """Tokens written again from the start of a block on: lengths, logits and cached rows are those of a cache that never held the others."""
    from flashsvd_amd.graphs import GraphedDecoder
    from tests.test_gpu_kv8_model import _cache, _model
    model, S = _model(128), 96
    ids = torch.randint(0, 512, (1, 60), generator=torch.Generator().manual_seed(3)).cuda()
    again, fresh = _cache(model, 1, S), _cache(model, 1, S)
    model(ids[:, :40], past_key_values=again, cache_position=torch.arange(40))
    out = []
    for c in (again, fresh):
        if c is fresh:
            model(ids[:, :16], past_key_values=c, cache_position=torch.arange(16))
        else:
            dec = GraphedDecoder(model, c, 1)              # some tokens that are given up too
            dec.set_state(ids[:, 50:51], 40)
            dec.step()
            assert c.get_seq_length() == 41
        logits = model(ids[:, 40:60], past_key_values=c, cache_position=torch.arange(16, 36, device="cuda")).logits[:, -1]
        assert c.get_seq_length() == 36
        dec = GraphedDecoder(model, c, 1)
        dec.set_state(logits.argmax(-1, keepdim=True), 36)
        tokens = [int(dec.step()) for _ in range(5)]
        assert c.get_seq_length() == 41
        out.append((logits, tokens, [t[0, :41].float() for t in c.key_cache + c.value_cache]))
    assert torch.equal(out[0][0], out[1][0]) and out[0][1] == out[1][1]
    for a, b in zip(out[0][2], out[1][2]):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("sampling", [None, dict(temperature=0.9, top_k=20)])
def test_a_capture_leaves_the_cache_as_it_was(sampling):
    """Captured before the first state is set as well as behind it, and again in between: the tokens of a decoder that runs eagerly."""
    from flashsvd_amd.graphs import GraphedDecoder
    from tests.test_gpu_kv8_model import _cache, _model
    model, S = _model(128), 64
    ids = torch.randint(0, 512, (2, 20), generator=torch.Generator().manual_seed(5)).cuda()
    out = []
    for captures in ((), (0,), (1, 4)):
        c = _cache(model, 2, S)
        first = model(ids, past_key_values=c, cache_position=torch.arange(20)).logits[:, -1].argmax(-1, keepdim=True)
        dec = GraphedDecoder(model, c, 2, sampling=sampling, generator=torch.Generator(device="cuda").manual_seed(7))

        def capture():
            buffers = c.key_cache + c.value_cache + c.key_scale + c.value_scale
            before = [t.view(torch.uint8).clone() if t.element_size() == 1 else t.clone() for t in buffers]
            dec.capture()
            for t, w in zip(buffers, before):
                assert torch.equal(t.view(torch.uint8) if t.element_size() == 1 else t, w)

        if 0 in captures:
            capture()
        dec.set_state(first, 20)
        got = []
        for i in range(1, 8):
            if i in captures:
                capture()
            got.append((dec.step() if captures else dec.eager_step()).tolist())
        assert c.get_seq_length() == 27
        out.append(got)
    assert out[0] == out[1] == out[2]
