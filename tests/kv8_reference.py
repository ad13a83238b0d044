"""The KV cache in 8 bits and the draw of a token in 64 bits on the CPU, written from their definitions."""
import math

import torch

F8 = torch.float8_e4m3fn


def scale_for(amax: float) -> float:
    """2^e with the smallest e >= -126 for which 448 * 2^e >= amax."""
    e = -126
    while amax > math.ldexp(448.0, e):
        e += 1
    return math.ldexp(1.0, e)


def nearest_code(x: torch.Tensor) -> torch.Tensor:
    """The e4m3 value nearest to x (double), ties to even; infinities become the largest, a NaN stays one."""
    e = (torch.frexp(x.nan_to_num(0.0, 0.0, 0.0))[1].double() - 1).clamp_min(-6.0)
    step = torch.exp2(e - 3.0)
    return torch.where(x.isinf(), x.sign() * 448.0, torch.clamp(torch.round(x / step) * step, -448.0, 448.0))


def rotate(x, cos, sin, pos):
    """x [.., Dh] (double) rotated at position pos, table rows clamped as the kernels do."""
    if cos is None:
        return x
    p = min(max(int(pos), 0), cos.shape[0] - 1)
    c, s = cos[p].double(), sin[p].double()
    a, b = x.chunk(2, -1)
    return torch.cat((a * c - b * s, a * s + b * c), -1)


def append(codes, scales, rows, p, n, block, cos=None, sin=None):
    """rows [T, Hk, Dh] (any float type) to positions p .. p + n - 1 of one sequence's codes [S, Hk, Dh] and scales [N, Hk], both double, in place."""
    S, Hk, _ = codes.shape
    first, last = max(p, 0), min(p + n, S)
    for blk in range(first // block, (last - 1) // block + 1 if last > first else 0):
        n0, n1 = max(first, blk * block), min(last, (blk + 1) * block)
        for h in range(Hk):
            new = torch.stack([rotate(rows[r - p, h].double(), cos, sin, r) for r in range(n0, n1)])
            size = scale_for(float(new.masked_fill(~new.isfinite(), 0.0).abs().max()))
            if n0 > blk * block:
                old = float(scales[blk, h])
                size = max(size, old)
                if size > old:
                    held = codes[blk * block:n0, h]
                    held.copy_(nearest_code(held * (old / size)))
            scales[blk, h] = size
            codes[n0:n1, h] = nearest_code(new / size)


def attend(q, k, v, scale, q_error, weight_error):
    """softmax(scale * q K^T) V for one query [Dh] over k, v [n, Dh] (all double): the output and how far a kernel may be from it before its last rounding.

    q_error: the relative rounding of q's elements, weight_error that of the softmax weights.  A score is off by at most
    d = scale * sum |q k| * (q_error + Dh * 2^-23) (fp32 sums of Dh products), a weight then by expm1(2 d) of itself, by 2^-20 for its
    exponential (argument and result in fp32 for arguments down to -90: 90 * 2^-23 < 2^-16 only where the weight is below e^-80, 2^-20 near
    the largest) and by weight_error, and sums of n terms in fp32 by n * 2^-23."""
    if len(k) == 0:
        return torch.zeros_like(q), torch.zeros_like(q)
    s = scale * (k @ q)
    w = torch.softmax(s, 0)
    d = float((scale * (k.abs() @ q.abs())).max()) * (q_error + q.numel() * 2.0 ** -23)
    rel = math.expm1(2 * d) + weight_error + 2.0 ** -18 + float(s.max() - s.min()) * 2.0 ** -22 + len(k) * 2.0 ** -23
    return w @ v, rel * (w @ v.abs())


def draw(logits, u, temperature, top_k, top_p, min_p) -> int:
    """The token of one row; numbers as Python floats."""
    x = logits.double()
    top = x.max() if not x.isnan().any() else torch.tensor(float("nan"))
    if not temperature > 0 or not torch.isfinite(top):
        return int(x.isnan().float().argmax()) if x.isnan().any() else int((x == x.max()).float().argmax())
    order = torch.sort(x, descending=True, stable=True).indices
    w = torch.exp((x[order] - top) / temperature)
    c = torch.cumsum(w, 0)
    k = min(top_k, len(x)) if top_k > 0 else len(x)
    n = min(k, int((c <= top_p * c[k - 1]).sum()) + 1, int((w >= min_p).sum()))
    n = max(n, 1)
    return int(order[min(int((c <= u * c[n - 1]).sum()), n - 1)])
