"""The KV cache in 4 bits and the log probabilities of tokens in 64 bits on the CPU, written from their definitions."""
import math

import torch

from tests.kv8_reference import attend, rotate      # noqa: F401  (what the two caches share)

CODES = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.double)


def exponent_for(amax: float) -> int:
    """The smallest e from -125 to 125 for which 7 * 2^e >= amax."""
    e = -125
    while e < 125 and amax > math.ldexp(7.0, e):
        e += 1
    return e


def group_values(x):
    """What a group of values [32] (double) becomes: its byte and the values that its codes stand for."""
    finite = x[x.isfinite()].abs()
    e = exponent_for(float(finite.max()) if len(finite) else 0.0)
    if bool(x.isnan().any()):
        return 255, torch.full_like(x, math.nan)
    y = (x.abs() / math.ldexp(1.0, e)).clamp_max(7.0)
    away = (y[:, None] - CODES).abs()
    nearest = away.amin(1, keepdim=True)
    code = torch.where(away == nearest, torch.arange(8), 99)
    low, high = code.amin(1), torch.where(away == nearest, torch.arange(8), -1).amax(1)
    code = torch.where(low % 2 == 0, low, high)                    # on a tie they are neighbours: the even one
    return e + 127, torch.where(x.signbit(), -1.0, 1.0) * CODES[code] * math.ldexp(1.0, e)


def append(values, bytes_, rows, p, n, cos=None, sin=None):
    """rows [T, Hk, Dh] (any float type) to positions p .. p + n - 1 of one sequence's values [S, Hk, Dh] (double) and bytes [Hk, Dh / 32, S], in place."""
    S, Hk, Dh = values.shape
    for r in range(max(p, 0), min(p + n, S)):
        for h in range(Hk):
            x = rotate(rows[r - p, h].double(), cos, sin, r)
            for g in range(Dh // 32):
                bytes_[h, g, r], values[r, h, 32 * g:32 * g + 32] = group_values(x[32 * g:32 * g + 32])


def unpack(codes, bytes_):
    """The values [.., S, Hk, Dh] (double) of codes [.., S, Hk, Dh / 2] and bytes [.., Hk, Dh / 32, S]."""
    table = torch.cat((CODES, -CODES))
    c = codes.cpu().long()
    x = torch.stack((table[c & 15], table[c >> 4]), -1).flatten(-2)
    b = bytes_.cpu().double()
    size = torch.where(b == 255, math.nan, torch.exp2(b - 127)).movedim(-1, -3)
    return x * size.repeat_interleave(32, -1)


def logprobs(logits, tokens, top):
    """One row [V] and its token: log probability, entropy, the likeliest tokens and their log probabilities."""
    x = logits.double()
    most = x.amax() if not bool(x.isnan().any()) else torch.tensor(math.nan)
    ranked = torch.sort(torch.where(x.isnan(), math.inf, x), descending=True, stable=True).indices
    if bool(x.isnan().any()):                                       # a NaN ranks above infinity
        nan = x[ranked].isnan()
        ranked = torch.cat((ranked[nan], ranked[~nan]))
    ranked = ranked[:top]
    if not bool(torch.isfinite(most)):
        lp = torch.full_like(x, math.nan)
        entropy = math.nan
    else:
        lp = x - most - torch.log(torch.exp(x - most).sum())
        p = torch.exp(lp)
        entropy = float(-(torch.where(p > 0, p * lp, 0.0)).sum())
    one = 0.0 if tokens < 0 else math.nan if tokens >= len(x) else float(lp[tokens])
    return one, entropy, ranked, lp[ranked]
