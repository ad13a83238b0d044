"""The low-rank Llama modules over the KV cache in 8 bits, and sampled generation: what a prompt leaves in the cache, decoding eagerly and captured, and
the serving functions that take them."""
import pytest
import torch

from tests import kv8_reference as R

pytestmark = pytest.mark.gpu
SHAPES = {64: dict(hidden_size=256, num_heads=4, num_kv_heads=2, head_dim=64, intermediate_size=512), 128: dict(hidden_size=256, num_heads=4, num_kv_heads=2, head_dim=128, intermediate_size=512)}


def _model(Dh, dt=torch.bfloat16, layers=2, seed=3):
    from flashsvd_amd import llama
    m = llama.build_model(**SHAPES[Dh], num_layers=layers, vocab_size=512, attn_rank=64, mlp_rank=128)
    return llama.materialize(m, "cuda", dt, seed=seed, std=0.08)


def _cache(model, B, length, dt=torch.bfloat16, block=16):
    from flashsvd_amd.runtime.cache import FlashSVDKV8Cache
    return FlashSVDKV8Cache(model.config, max_batch_size=B, max_cache_len=length, block_size=block, device="cuda", dtype=dt)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Dh,T", [(128, 40), (64, 40), (128, 5), (64, 16)])
def test_prompt_leaves_the_rounded_rows_in_the_cache(Dh, T, dt):
    """Layer 0 sees the same input whatever the cache: its rows are those of the dense cache, rounded.  Where the same kernels make them (128 dimensions, 16 rows
    and more) the codes are equal; else the rows come from other sums and are rotated in fp32 instead of 16 bits with a rounding for each of three operations, so a
    code is off by its half step (2^-4 of the value, 2^-10 of the scale) and four half steps of the 16-bit type of the row's largest magnitudes."""
    from flashsvd_amd.runtime.cache import FlashSVDV15DenseKVCache
    model, B, S = _model(Dh, dt), 2, 64
    ids = torch.randint(0, 512, (B, T), generator=torch.Generator().manual_seed(1)).cuda()
    c8, c16 = _cache(model, B, S, dt), FlashSVDV15DenseKVCache(model.config, max_batch_size=B, max_cache_len=S, device="cuda", dtype=dt)
    for c in (c8, c16):
        model(ids, past_key_values=c, cache_position=torch.arange(T))
        assert c.get_seq_length() == T
    for codes, scale, dense in ((c8.key_cache[0], c8.key_scale[0], c16.key_cache[0]), (c8.value_cache[0], c8.value_scale[0], c16.value_cache[0])):
        got, size, rows = codes.cpu().float().double(), scale.cpu().double(), dense.cpu()
        assert not bool(got[:, T:].any())
        for b in range(B):
            if Dh == 128 and T >= 16:
                want, s = torch.zeros_like(got[b]), torch.zeros_like(size[b])
                R.append(want, s, rows[b, :T], 0, T, 16)
                assert torch.equal(got[b], want) and torch.equal(size[b], s)
            else:
                full = size[b].repeat_interleave(16, 0)[:T, :, None]
                x = rows[b, :T].double()
                room = x.abs() * 2.0 ** -4 + full * 2.0 ** -10 + 4 * torch.finfo(dt).eps / 2 * x.abs().amax(-1, keepdim=True) * 2
                assert bool(((got[b, :T] * full - x).abs() <= room).all())


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
            assert torch.equal(x.float(), y.float())


def test_decode_sees_the_dense_rows_rounded():
    """One layer, a prompt and one token: the attention's output over the 8-bit cache against the formula in 64 bits over what the cache holds."""
    from flashsvd_amd import hip_ops
    model, B, T, S = _model(128, layers=1), 2, 33, 64
    ids = torch.randint(0, 512, (B, T), generator=torch.Generator().manual_seed(4)).cuda()
    c = _cache(model, B, S)
    model(ids, past_key_values=c, cache_position=torch.arange(T))
    seen = {}
    run = hip_ops.attn_decode_kv8

    def watched(q, *a, **k):
        seen.update(q=q.clone(), **{n: v for n, v in k.items() if n in ("cos", "sin")})
        seen["out"] = run(q, *a, **k)
        return seen["out"]

    hip_ops.attn_decode_kv8 = watched
    try:
        model.decode_step(torch.full((B, 1), 7, device="cuda"), c, torch.full((B,), T, dtype=torch.int32, device="cuda"))
    finally:
        hip_ops.attn_decode_kv8 = run
    k, v = (x.cpu().double() for x in c.dequantize(0, batch_size=B, length=T + 1))
    half = torch.finfo(torch.bfloat16).eps / 2
    for b in range(B):
        for h in range(4):
            q = R.rotate(seen["q"][b, h].cpu().double(), seen["cos"].cpu(), seen["sin"].cpu(), T)
            want, room = R.attend(q, k[b, :, h // 2], v[b, :, h // 2], 128 ** -0.5, half, half)
            assert bool(((seen["out"][b, h].cpu().double() - want).abs() <= want.abs() * half + room * (1 + half)).all())


def test_chunks_of_a_prompt_and_int4_factors():
    """A prompt in two chunks, the second across a block that the first left open, and a model of int4 factors: both decode on, eagerly as captured."""
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


class _Tok:
    pad_token_id = eos_token_id = None

    def __call__(self, prompt, return_tensors=None, add_special_tokens=False):
        return {"input_ids": torch.arange(1, 20)[None]}

    def decode(self, ids, skip_special_tokens=False):
        return " ".join(map(str, ids))


@pytest.mark.parametrize("kv8", [False, True])
def test_sampled_generation(kv8):
    """A seed gives the same tokens eagerly and captured, another seed others; top_k = 1 gives the greedy ones."""
    from flashsvd_amd import api
    model = _model(128)
    kw = dict(prompt="x", max_new_tokens=12, kv8_cache=kv8, do_sample=True, temperature=3.0, top_p=0.98, top_k=300, min_p=0.001)
    a, b, other = (api.generate_text(model, _Tok(), seed=s, use_graph=g, **kw)["completion_ids"] for s, g in ((5, False), (5, True), (6, True)))
    assert a == b and a != other and len(a) == 12
    one = api.generate_text(model, _Tok(), seed=1, use_graph=True, **(kw | dict(top_k=1)))["completion_ids"]
    greedy = api.generate_text(model, _Tok(), prompt="x", max_new_tokens=12, kv8_cache=kv8, use_graph=False)["completion_ids"]
    assert one == greedy


def test_serving_functions_and_the_cache_api():
    from flashsvd_amd import api
    model = _model(64)
    out = api.decode_kvcache_eval(model, prompt_len=16, new_tokens=4, warmup=2, batch_size=2, kv8_cache=True)
    assert out["kv8_cache"] and out["decode_engine"] == "graph" and not out["flashsvd_dense_cache"]
    with pytest.raises(ValueError, match="mutually exclusive"):
        api.decode_kvcache_eval(model, prompt_len=8, new_tokens=1, warmup=0, kv8_cache=True, lowrank_cache=True)
    c = _cache(model, 2, 40)
    g = torch.Generator().manual_seed(8)
    k, v = (torch.randn(2, 2, 7, 64, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    K, V = c.update(k, v, 0)
    assert K.shape == (2, 2, 7, 64) and c.get_seq_length() == 7
    K, V = c.update(k[:, :, :3], v[:, :, :3], 0, {"cache_position": torch.arange(7, 10)})
    assert K.shape == (2, 2, 10, 64) and c.get_seq_length() == 10
    for got, x in ((K, k), (V, v)):
        want = torch.cat((x, x[:, :, :3]), 2).float()
        scale = c.key_scale[0].max() if got is K else c.value_scale[0].max()
        assert bool(((got.float() - want).abs() <= want.abs() * 2.0 ** -4 + scale * 2.0 ** -10).all())
    with pytest.raises(RuntimeError, match="shape changed"):
        c.update(k[..., :32].repeat(1, 2, 1, 1), v[..., :32].repeat(1, 2, 1, 1), 0)
    with pytest.raises(ValueError, match="consecutive"):
        c.update(k[:, :, :2], v[:, :, :2], 0, {"cache_position": torch.tensor([3, 9])})
    with pytest.raises(IndexError, match="out of range"):
        c.update(k, v, 0, {"cache_position": torch.arange(36, 43)})
