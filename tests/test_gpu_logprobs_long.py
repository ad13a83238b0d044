"""Log probabilities of rows whose parts no registers hold, which are read again: masks of the type's lowest value and of -inf in front of other logits, ties, a NaN."""
import math

import pytest
import torch

from tests.test_gpu_logprobs import _check
from tests.util import form_taken

pytestmark = pytest.mark.gpu
V = 2 ** 21 + 13                                            # sixteen parts of 16386 pieces of eight logits


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("mask", ["lowest", "-inf"])
def test_masks_in_front_of_other_logits(mask, dt):
    """A thread that has summed masked logits alone moves its sums to a larger one: e^x of the distance is 0 and so are they, however large the distance."""
    from flashsvd_amd import hip_ops
    g = torch.Generator().manual_seed(3)
    x = torch.randn(5, V, generator=g) * 2
    low = torch.finfo(dt).min if mask == "lowest" else -math.inf
    piece = torch.arange(V) // 8
    x[0, :V * 3 // 5] = low                                 # the front of the row, up to the middle of a part
    x[1, piece % 16386 < 8200] = low                        # the front of every part
    x[2, piece // 1024 % 2 == 0] = low                      # every other piece of a thread
    x[3] = low                                              # one that stands out, the last a thread reads
    x[3, V - 1] = 1.0
    x[4, ::2] = low
    x = x.to(dt)
    t = torch.tensor([V - 2, 5, 9000, V - 1, 1])
    out = hip_ops.token_logprobs(x.cuda(), t.cuda(), top=4)
    assert form_taken() == "logprobs long parts"
    _check(x, t, 4, out)


def test_ties_and_numbers_that_are_none():
    from flashsvd_amd import hip_ops
    g = torch.Generator().manual_seed(4)
    x = torch.stack((torch.randn(V, generator=g).mul(2).round(), torch.zeros(V), torch.full((V,), -math.inf), torch.randn(V, generator=g),
                     torch.randn(V, generator=g))).to(torch.bfloat16)
    x[3, V // 2] = math.nan
    x[4, 70001] = math.inf
    t = torch.tensor([V - 1, 0, 3, 5, -1])
    out = hip_ops.token_logprobs(x.cuda(), t.cuda(), top=20)
    assert form_taken() == "logprobs long parts"
    _check(x, t, 20, out)
