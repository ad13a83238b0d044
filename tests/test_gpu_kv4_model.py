"""The low-rank Llama modules over the KV cache in 4 bits and the log probabilities of what they generate: what a prompt leaves in the cache, decoding eagerly and
captured, and the serving functions that take them."""
import math

import pytest
import torch

from tests import kv4_reference as R
from tests.test_gpu_kv8_model import _Tok, _model

pytestmark = pytest.mark.gpu


def _cache(model, B, length, dt=torch.bfloat16):
    from flashsvd_amd.runtime.cache import FlashSVDKV4Cache
    return FlashSVDKV4Cache(model.config, max_batch_size=B, max_cache_len=length, device="cuda", dtype=dt)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Dh,T", [(128, 40), (64, 40), (128, 5), (64, 16)])
def test_prompt_leaves_the_rounded_rows_in_the_cache(Dh, T, dt):
    """Layer 0 sees the same input whatever the cache: its rows are those of the dense cache, rounded.  Where the same kernels make them (128 dimensions, 16 rows
    and more) the codes are equal; else the rows come from other sums and are rotated in fp32 instead of 16 bits with a rounding for each of three operations.  The
    steps of a code are 0.5, 1 and 2 of the group's power of two below 2, 4 and above: a value is off by a fourth of it or of the power at most."""
    from flashsvd_amd.runtime.cache import FlashSVDV15DenseKVCache
    model, B, S = _model(Dh, dt), 2, 64
    ids = torch.randint(0, 512, (B, T), generator=torch.Generator().manual_seed(1)).cuda()
    c4, c16 = _cache(model, B, S, dt), FlashSVDV15DenseKVCache(model.config, max_batch_size=B, max_cache_len=S, device="cuda", dtype=dt)
    for c in (c4, c16):
        model(ids, past_key_values=c, cache_position=torch.arange(T))
        assert c.get_seq_length() == T
    for codes, bytes_, dense in ((c4.key_cache[0], c4.key_scale[0], c16.key_cache[0]), (c4.value_cache[0], c4.value_scale[0], c16.value_cache[0])):
        got, rows = R.unpack(codes, bytes_), dense.cpu()
        assert not bool(codes[:, T:].any()) and not bool(bytes_[..., T:].any())
        for b in range(B):
            if Dh == 128 and T >= 16:
                want, size = torch.zeros_like(got[b]), torch.zeros_like(bytes_[b].cpu())
                R.append(want, size, rows[b, :T], 0, T)
                assert torch.equal(got[b], want) and torch.equal(bytes_[b].cpu(), size)
            else:
                power = torch.exp2(bytes_[b, :, :, :T].cpu().double() - 127).movedim(-1, -3).repeat_interleave(32, -1)
                x = rows[b, :T].double()
                other = 4 * torch.finfo(dt).eps / 2 * x.abs().amax(-1, keepdim=True) * 2
                assert bool(((got[b, :T] - x).abs() <= torch.maximum(x.abs() + other, power) / 4 + other).all())


@pytest.mark.parametrize("Dh,B", [(128, 1), (64, 3)])
def test_decode_captured_is_decode_eager(Dh, B):
    from flashsvd_amd.graphs import GraphedDecoder
    model, T, S, steps = _model(Dh), 21, 64, 8
    ids = torch.randint(0, 512, (B, T), generator=torch.Generator().manual_seed(2)).cuda()
    outs = []
    for captured in (False, True):
        c = _cache(model, B, S)
        first = model(ids, past_key_values=c, cache_position=torch.arange(T)).logits[:, -1].argmax(-1, keepdim=True)
        dec = GraphedDecoder(model, c, B)
        dec.set_state(first, T)
        if captured:
            dec.capture()
        got = []
        for _ in range(steps):
            t = dec.step() if captured else dec.eager_step()
            got.append((t.clone(), dec.logits.clone()))
            torch.zeros(1000, device="cuda").sum()          # the program's own work between the steps
            torch.cuda.synchronize()
        outs.append((got, c))
    for (a, la), (b, lb) in zip(outs[0][0], outs[1][0]):
        assert torch.equal(a, b) and torch.equal(la, lb)
    for i in range(2):
        for name in ("key_cache", "value_cache", "key_scale", "value_scale"):
            x, y = (getattr(o[1], name)[i] for o in outs)
            assert torch.equal(x, y)


@pytest.mark.parametrize("S", [64, 100])
def test_a_capture_before_the_state_is_set_leaves_the_cache_as_it_was(S):
    from flashsvd_amd.graphs import GraphedDecoder
    model, T = _model(128), 21
    ids = torch.randint(0, 512, (2, T), generator=torch.Generator().manual_seed(2)).cuda()
    c = _cache(model, 2, S)
    first = model(ids, past_key_values=c, cache_position=torch.arange(T)).logits[:, -1].argmax(-1, keepdim=True)
    held = [t.clone() for name in ("key_cache", "value_cache", "key_scale", "value_scale") for t in getattr(c, name)]
    dec = GraphedDecoder(model, c, 2)
    dec.capture()
    assert all(torch.equal(a, b) for a, b in zip(held, [t for name in ("key_cache", "value_cache", "key_scale", "value_scale") for t in getattr(c, name)]))
    dec.set_state(first, T)
    got = [dec.step().clone() for _ in range(3)]
    other = GraphedDecoder(model, c, 2)
    other.set_state(first, T)
    assert all(torch.equal(a, other.eager_step()) for a in got)


def test_decode_sees_the_dense_rows_rounded():
    """One layer, a prompt and one token: the attention's output over the 4-bit cache against the formula in 64 bits over what the cache holds."""
    from flashsvd_amd import hip_ops
    model, B, T, S = _model(128, layers=1), 2, 33, 64
    ids = torch.randint(0, 512, (B, T), generator=torch.Generator().manual_seed(4)).cuda()
    c = _cache(model, B, S)
    model(ids, past_key_values=c, cache_position=torch.arange(T))
    seen = {}
    run = hip_ops.attn_decode_kv4

    def watched(q, *a, **k):
        seen.update(q=q.clone(), **{n: v for n, v in k.items() if n in ("cos", "sin")})
        seen["out"] = run(q, *a, **k)
        return seen["out"]

    hip_ops.attn_decode_kv4 = watched
    try:
        model.decode_step(torch.full((B, 1), 7, device="cuda"), c, torch.full((B,), T, dtype=torch.int32, device="cuda"))
    finally:
        hip_ops.attn_decode_kv4 = run
    k, v = (x.cpu().double() for x in c.dequantize(0, batch_size=B, length=T + 1))
    half = torch.finfo(torch.bfloat16).eps / 2
    for b in range(B):
        for h in range(4):
            q = R.rotate(seen["q"][b, h].cpu().double(), seen["cos"].cpu(), seen["sin"].cpu(), T)
            want, room = R.attend(q, k[b, :, h // 2], v[b, :, h // 2], 128 ** -0.5, half, half)
            assert bool(((seen["out"][b, h].cpu().double() - want).abs() <= want.abs() * half + room * (1 + half)).all())


def test_chunks_of_a_prompt_and_int4_factors():
    """A prompt in two chunks, the second from the middle of a tile on, and a model of int4 factors: both decode on, eagerly as captured."""
    from flashsvd_amd import quant
    from flashsvd_amd.graphs import GraphedDecoder
    for int4 in (False, True):
        model, B, S = _model(128), 1, 96
        if int4:
            quant.replace_linears_with_packed_quant_inplace(model, module_names=quant.factor_linear_names(model), bits=4, group_size=32, sym=False)
        ids = torch.randint(0, 512, (B, 53), generator=torch.Generator().manual_seed(6)).cuda()
        outs = []
        for captured in (False, True):
            c = _cache(model, B, S)
            model(ids[:, :21], past_key_values=c, cache_position=torch.arange(21))
            first = model(ids[:, 21:], past_key_values=c, cache_position=torch.arange(21, 53)).logits[:, -1].argmax(-1, keepdim=True)
            assert c.get_seq_length() == 53
            dec = GraphedDecoder(model, c, B)
            dec.set_state(first, 53)
            outs.append([(dec.step() if captured else dec.eager_step()).item() for _ in range(5)])
        assert outs[0] == outs[1]


@pytest.mark.parametrize("captured", [False, True])
def test_sampled_generation_with_log_probabilities(captured):
    """The cache, the draw and the log probabilities together: a seed gives the same tokens and numbers eagerly and captured, and the numbers are those of the
    logits that the tokens were drawn from."""
    from flashsvd_amd import api, hip_ops
    from tests.test_gpu_logprobs import _check
    model, seen, run = _model(128), [], hip_ops.token_logprobs

    def watched(logits, tokens, *, top):
        out = run(logits, tokens, top=top)
        seen.append((logits.clone(), tokens.clone(), out))
        return out

    kw = dict(prompt="x", max_new_tokens=12, kv4_cache=True, do_sample=True, temperature=3.0, top_p=0.98, top_k=300, seed=5, logprobs=4)
    plain = api.generate_text(model, _Tok(), use_graph=False, **(kw | dict(logprobs=None)))
    hip_ops.token_logprobs = watched
    try:
        out = api.generate_text(model, _Tok(), use_graph=captured, **kw)
    finally:
        hip_ops.token_logprobs = run
    assert out["completion_ids"] == plain["completion_ids"] and len(out["completion_ids"]) == 12 and not set(out) & {"logprobs"} and "completion_logprobs" not in plain
    assert [int(t) for _, t, _ in seen] == out["completion_ids"] and len(out["completion_logprobs"]) == len(out["completion_entropies"]) == 12
    for (logits, tokens, o), lp, ent, top in zip(seen, out["completion_logprobs"], out["completion_entropies"], out["completion_top_logprobs"]):
        _check(logits, tokens, 4, o)
        assert lp == o[0].item() and ent == o[1].item() and [t for t, _ in top] == o[2][0].tolist() and [p for _, p in top] == o[3][0].tolist()
    assert len({tuple(x) for x in out["completion_top_logprobs"]}) > 1          # not one step's numbers for all
    greedy = api.generate_text(model, _Tok(), prompt="x", max_new_tokens=5, kv4_cache=True, use_graph=captured, logprobs=1)
    assert [t[0][1] for t in greedy["completion_top_logprobs"]] == greedy["completion_logprobs"]
    bare = api.generate_text(model, _Tok(), prompt="x", max_new_tokens=5, kv4_cache=True, use_graph=captured, logprobs=0)
    assert bare["completion_logprobs"] == greedy["completion_logprobs"] and bare["completion_top_logprobs"] == [[]] * 5


def test_scores_of_a_text():
    from flashsvd_amd import api
    from tests.test_gpu_logprobs import _room
    model = _model(64)
    out = api.score_text(model, _Tok(), text="x", top=3)
    ids = torch.arange(1, 20)[None].cuda()
    with torch.no_grad():
        logits = model(input_ids=ids).logits[0].cpu()
    assert out["ids"] == ids[0].tolist() and len(out["logprobs"]) == 18
    for t in range(18):
        lp, ent, best, best_lp = R.logprobs(logits[t], int(ids[0, t + 1]), 3)
        assert [i for i, _ in out["top_logprobs"][t]] == best.tolist()
        for got, want, kind in ((out["logprobs"][t], lp, False), (out["entropies"][t], ent, True), *((p, x, False) for (_, p), x in zip(out["top_logprobs"][t], best_lp.tolist()))):
            assert abs(got - want) <= _room(logits[t].double(), want, kind)
    assert out["sum"] == math.fsum(out["logprobs"]) and abs(out["perplexity"] - math.exp(-out["sum"] / 18)) <= 1e-12 * out["perplexity"]
    with pytest.raises(ValueError, match="top"):
        api.score_text(model, _Tok(), text="x", top=65)


def test_serving_functions_and_the_cache_api():
    from flashsvd_amd import api
    model = _model(64)
    out = api.decode_kvcache_eval(model, prompt_len=16, new_tokens=4, warmup=2, batch_size=2, kv4_cache=True)
    assert out["kv4_cache"] and not out["kv8_cache"] and out["decode_engine"] == "graph" and not out["flashsvd_dense_cache"]
    c = _cache(model, 2, 40)
    g = torch.Generator().manual_seed(8)
    k, v = (torch.randn(2, 2, 7, 64, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    K, V = c.update(k, v, 0)
    assert K.shape == (2, 2, 7, 64) and c.get_seq_length() == 7
    K, V = c.update(k[:, :, :3], v[:, :, :3], 0, {"cache_position": torch.tensor([7, 39, 5])})
    assert K.shape == (2, 2, 40, 64) and c.get_seq_length() == 40
    for got, x in ((K, k), (V, v)):
        for p, t in ((0, 0), (4, 4), (5, 2), (6, 6), (7, 0), (39, 1)):
            for b in range(2):
                for h in range(2):
                    want = torch.cat([R.group_values(r)[1] for r in x[b, h, t].cpu().double().view(2, 32)])
                    assert torch.equal(got[b, h, p].cpu().double(), want)
    with pytest.raises(IndexError, match="out of range"):
        c.update(k, v, 0, {"cache_position": torch.arange(36, 43)})


def test_more_positions_than_sequences_in_use():
    """Decoding with fewer sequences than the cache has, each at a position of its own, the last one at the end of the cache's length."""
    model, S = _model(128, layers=1), 70
    c = _cache(model, 4, S)
    ids = torch.randint(0, 512, (2, 30), generator=torch.Generator().manual_seed(9)).cuda()
    model(ids, past_key_values=c, cache_position=torch.arange(30))
    before = [t.clone() for t in c.operands(0, 4)]
    model.decode_step(torch.tensor([[3], [4]], device="cuda"), c, torch.tensor([11, S - 1], dtype=torch.int32, device="cuda"))
    for t, old in zip(c.operands(0, 4), before):
        rows, kept = (t, old) if t.shape[1] == 128 else (t.permute(0, 3, 1, 2), old.permute(0, 3, 1, 2))       # rows second
        same = (rows == kept).flatten(2).all(-1)
        assert [p for p in range(128) if not bool(same[0, p])] == [11] and [p for p in range(128) if not bool(same[1, p])] == [S - 1]
        assert bool(same[2:].all())
