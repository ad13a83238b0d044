"""A text's log probabilities over the caches in 8 and 4 bits: those of the logits that the model's own pass over such a cache gives."""
import pytest
import torch

from tests import kv4_reference as R
from tests.test_gpu_kv8_model import _model
from tests.test_gpu_logprobs import _room


class _Text:
    """A tokenizer whose texts are numbers of tokens."""

    def __call__(self, text, **kw):
        return {"input_ids": torch.randint(0, 512, (1, int(text)), generator=torch.Generator().manual_seed(1))}

    def decode(self, ids, **kw):
        return ""


@pytest.mark.gpu
@pytest.mark.parametrize("Dh", [64, 128])
@pytest.mark.parametrize("which", ["kv8_cache", "kv4_cache"])
@pytest.mark.parametrize("n", [1, 2, 61, 200])
def test_scores_over_a_smaller_cache(n, which, Dh):
    from flashsvd_amd import api
    from flashsvd_amd.runtime.cache import FlashSVDKV4Cache, FlashSVDKV8Cache
    model, kind = _model(Dh), FlashSVDKV4Cache if which == "kv4_cache" else FlashSVDKV8Cache
    out, plain = (api.score_text(model, _Text(), text=str(n), top=3, **kw) for kw in ({which: True}, {}))
    assert out["ids"] == plain["ids"] and len(out["logprobs"]) == len(out["top_logprobs"]) == n - 1
    if n == 1:
        return
    ids = torch.tensor(out["ids"])[None].cuda()
    c = kind(model.config, max_batch_size=1, max_cache_len=n + 4, device="cuda", dtype=torch.bfloat16)
    logits = model(ids, past_key_values=c, cache_position=torch.arange(n)).logits[0].cpu()
    for t in range(n - 1):
        lp, ent, best, best_lp = R.logprobs(logits[t], out["ids"][t + 1], 3)
        assert [i for i, _ in out["top_logprobs"][t]] == best.tolist()
        assert abs(out["logprobs"][t] - lp) <= _room(logits[t].double(), lp, False) and abs(out["entropies"][t] - ent) <= _room(logits[t].double(), ent, True)
        for (_, p), x in zip(out["top_logprobs"][t], best_lp.tolist()):
            assert abs(p - x) <= _room(logits[t].double(), x, False)
    assert n == 2 or out["logprobs"] != plain["logprobs"]   # not the 16-bit cache's numbers


def test_one_cache_at_a_time():
    from types import SimpleNamespace

    from flashsvd_amd import api
    model = torch.nn.Linear(2, 2)
    model.config = SimpleNamespace(num_hidden_layers=2, rope_theta=10000.0)
    with pytest.raises(ValueError, match="mutually exclusive"):
        api.score_text(model, _Text(), text="5", kv8_cache=True, kv4_cache=True)
    assert api.score_text(model, _Text(), text="1", kv4_cache=True)["logprobs"] == []
