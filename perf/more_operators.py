"""Serving from a KV cache in 4 bits and the log probabilities of tokens, as cases that can be timed and compared: rows appended to the cache and
what it holds then ("append"), one query token per sequence over it ("decode"), a chunk of a prompt over it ("prompt"), and log probabilities
of given tokens with the entropy and the likeliest alternatives ("logprobs").

The cache holds e2m1 codes, two a byte with the even channel in the low bits, [B, S, Hk, Dh / 2], and one byte for each token, kv head and 32 channels,
[B, Hk, Dh / 32, S]: ``value = code * 2 ** (byte - 127)``.  The exponent of a group is the smallest from -125 to 125 whose 7-fold covers the group (7 lies halfway
between the largest code, 6, and what would follow it); a value goes to the nearest code, ties to the even one.

A case names sizes only: ``batch`` sequences with up to ``context`` cached tokens (``ragged``: of unequal lengths), ``tokens`` new rows,
``heads`` / ``kv_heads`` / ``head_dim``, ``dtype``, ``rotate`` (rotary tables are applied by the call); ``batch`` rows of ``vocab`` logits and ``top`` alternatives.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
GROUP = 32
CODES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)

# head layouts of the model shapes in cases.py: the one-block configuration, the 7B shape, the same with a quarter of the kv heads
SMALL = dict(heads=8, kv_heads=8, head_dim=64)
WIDE = dict(heads=32, kv_heads=32, head_dim=128)
GROUPED = dict(heads=32, kv_heads=8, head_dim=128)


def listed():
    append = dict(kind="append", dtype="bf16", rotate=True, ragged=False)
    decode = dict(kind="decode", tokens=1, dtype="bf16", rotate=True, ragged=False)
    prompt = dict(kind="prompt", dtype="bf16", rotate=False, ragged=False)
    logprobs = dict(kind="logprobs", dtype="bf16")
    return [
        # the next token of four short conversations written behind their caches and the caches handed on in 16 bits
        dict(append, name="append_tokens", **GROUPED, batch=4, context=120, tokens=1) | dict(ragged=True),
        # the stress configuration's prompts written in one call and handed on in 16 bits
        dict(append, name="append_prompts", **WIDE, batch=8, context=0, tokens=2048),
        # one token of the small model: all latency
        dict(decode, name="decode_small", **SMALL, batch=1, context=137),
        # one long conversation of a grouped-query model in float16
        dict(decode, name="decode_one_long", **GROUPED, batch=1, context=16001) | dict(dtype="fp16"),
        # sixteen conversations of unequal lengths of a grouped-query model
        dict(decode, name="decode_batch", **GROUPED, batch=16, context=4001) | dict(ragged=True),
        # the stress configuration's decode step: as many kv heads as query heads
        dict(decode, name="decode_stress", **WIDE, batch=16, context=4090),
        # the 7B shape's prompt of 512 tokens
        dict(prompt, name="prompt_512", **WIDE, batch=1, context=0, tokens=512),
        # the next turn of two conversations, of unequal lengths, in float16
        dict(prompt, name="prompt_chunk", **GROUPED, batch=2, context=1411, tokens=77) | dict(dtype="fp16", ragged=True, rotate=True),
        # the stress configuration's prompts: the largest call
        dict(prompt, name="prompt_stress", **WIDE, batch=8, context=0, tokens=2048),
        # an answer's token with what else it could have been
        dict(logprobs, name="logprobs_one", batch=1, vocab=32000, top=20),
        # a batch of requests over a large vocabulary
        dict(logprobs, name="logprobs_batch", batch=64, vocab=128256, top=5) | dict(dtype="fp16"),
        # the scores of eight texts of 512 tokens
        dict(logprobs, name="logprobs_texts", batch=4096, vocab=32000, top=1),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "append", "decode", "decode", "decode", "prompt", "prompt", "logprobs", "logprobs"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if kind == "logprobs":
        vocab = _log(rng, 500, 130000)
        return dict(kind=kind, dtype=dtype, batch=_log(rng, 1, max(1, min(8192, 4096 * 32000 // vocab))), vocab=vocab, top=rng.choice([0, 1, 5, 20, _log(rng, 2, 64)]))
    kv_heads = rng.choice([1, 2, 4, 8, 8, 16, 32])
    case = dict(kind=kind, dtype=dtype, head_dim=rng.choice([64, 128, 128]), kv_heads=kv_heads,
                heads=kv_heads * rng.choice([g for g in (1, 2, 4, 6, 8) if g * kv_heads <= 48]), rotate=rng.choice([True, False]), ragged=rng.choice([True, False]))
    row = kv_heads * case["head_dim"]
    if kind == "append":
        case["tokens"], case["context"] = rng.choice([1, _log(rng, 2, 2048)]), rng.choice([0, _log(rng, 1, 2000)])
        case["batch"] = _log(rng, 1, max(1, min(64, 8 * 2048 * 4096 // (row * _room(case)))))
    elif kind == "decode":
        case.update(tokens=1, context=_log(rng, 1, 16000))
        case["batch"] = _log(rng, 1, max(1, min(64, 16 * 4090 * 4096 // (row * case["context"]))))
    else:
        case["tokens"], case["context"] = _log(rng, 2, 2048), rng.choice([0, _log(rng, 1, 3000)])
        pairs = case["heads"] * case["tokens"] * (case["context"] + case["tokens"] // 2 + 1)
        case["batch"] = _log(rng, 1, max(1, min(16, 8 * 32 * 1024 * 2048 // pairs)))
    return case


# ------------------------------------------------------------------ sizes that follow from a case
def _contexts(case):
    """Cached tokens of every sequence: the first has them all, the others of a ragged batch down to a quarter."""
    n = case["context"]
    return [n - (613 * b) % (3 * n // 4 + 1) if case["ragged"] else n for b in range(case["batch"])]


def _rows(case):
    """New rows of every sequence (a ragged chunk is padded behind them)."""
    t = case["tokens"]
    return [t - (29 * b) % ((t + 1) // 2) if case["ragged"] else t for b in range(case["batch"])]


def _room(case):
    """Cache rows of a sequence: a multiple of 64 with room for the new ones."""
    return (case["context"] + case["tokens"] + 63) // 64 * 64


def work(case):
    if case["kind"] == "logprobs":
        return {"bytes": case["batch"] * (2.0 * case["vocab"] + 16 + 12.0 * case["top"]), "flops": 4.0 * case["batch"] * case["vocab"]}
    row = case["kv_heads"] * case["head_dim"]
    past, new = _contexts(case), _rows(case)
    held = 2.0 * row * (0.5 + 1.0 / GROUP)                          # of a token, keys and values
    if case["kind"] == "append":
        return {"bytes": sum(new) * (4.0 * row + held) + case["batch"] * _room(case) * (held + 4.0 * row), "flops": (6.0 * sum(new) + 2.0 * case["batch"] * _room(case)) * row}
    q = 4.0 * sum(new) * case["heads"] * case["head_dim"]          # 16 bits in and out
    if case["kind"] == "decode":
        return {"bytes": sum(past) * held + q, "flops": 4.0 * sum(past) * case["heads"] * case["head_dim"]}
    pairs = sum(t * c + t * (t + 1) // 2 for c, t in zip(past, new))
    return {"bytes": sum(c + t for c, t in zip(past, new)) * held + q, "flops": 4.0 * pairs * case["heads"] * case["head_dim"]}


# ------------------------------------------------------------------ inputs
def _cache(gen, case, spread):
    """Codes [B, S, Hk, Dh / 2] and bytes [B, Hk, Dh / 32, S] of a cache that has been in use: every row holds something."""
    B, S, Hk, Dh = case["batch"], _room(case), case["kv_heads"], case["head_dim"]
    codes = torch.empty(B, Hk, S, Dh // 2, dtype=torch.uint8, device="cuda")
    scale = torch.empty(B, Hk, Dh // GROUP, S, dtype=torch.uint8, device="cuda")
    for b in range(B):
        c, e = _coded(torch.randn(Hk, S, Dh, generator=gen, device="cuda") * spread)
        codes[b], scale[b] = c, e.transpose(1, 2)
    return codes.transpose(1, 2), scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]
    B = case["batch"]
    if case["kind"] == "logprobs":
        V = case["vocab"]
        # most of a vocabulary far below a few candidates, as a language model leaves it; the token is one of the likelier ones
        x = torch.randn(B, V, generator=gen, device="cuda") * 2.5
        x += 4.0 * torch.rand(B, V, generator=gen, device="cuda").pow(12) * torch.rand(B, 1, generator=gen, device="cuda")
        tokens = torch.where(x > 5.0, torch.rand(B, V, generator=gen, device="cuda"), -x.abs()).argmax(1)
        return dict(case=case, logits=x.to(dt), tokens=tokens)
    H, Hk, Dh, T, S = case["heads"], case["kv_heads"], case["head_dim"], case["tokens"], _room(case)
    # keys with a few strong channels, values without
    strong = 1.0 + 3.0 * (torch.rand(Hk, 1, Dh, generator=gen, device="cuda") > 0.95)
    s = dict(case=case)
    s["k"], s["k_scale"] = _cache(gen, case, strong)
    s["v"], s["v_scale"] = _cache(gen, case, 1.0)
    s["positions"] = torch.tensor(_contexts(case), dtype=torch.int32, device="cuda")
    s["rows"] = torch.tensor(_rows(case), dtype=torch.int32, device="cuda") if case["ragged"] and T > 1 else None
    ang = torch.arange(S, device="cuda")[:, None].double() * 10000.0 ** (-torch.arange(Dh // 2, device="cuda").double() / (Dh // 2))
    s["cos"], s["sin"] = (ang.cos().to(dt), ang.sin().to(dt)) if case["rotate"] else (None, None)
    if case["kind"] == "append":
        s["k_new"] = (torch.randn(B, T, Hk, Dh, generator=gen, device="cuda") * strong[:, 0] * 1.5).to(dt)
        s["v_new"] = (torch.randn(B, T, Hk, Dh, generator=gen, device="cuda") * 1.5).to(dt)
    else:
        # scores of a standard deviation of about two
        shape = (B, H, Dh) if case["kind"] == "decode" else (B, T, H, Dh)
        s["q"] = (torch.randn(shape, generator=gen, device="cuda") * 1.5).to(dt)
        s["out"] = torch.zeros_like(s["q"])
    return s


# ------------------------------------------------------------------ the operators
def run(state):
    return {"append": _append, "decode": _decode, "prompt": _prompt, "logprobs": _logprobs}[state["case"]["kind"]](state)


def _append(s):
    held, dt = (s["k"], s["v"], s["k_scale"], s["v_scale"]), DTYPES[s["case"]["dtype"]]
    if own:
        from flashsvd_amd import hip_ops
        hip_ops.kv4_append(s["k_new"], s["v_new"], *held, s["positions"], cos=s["cos"], sin=s["sin"], rows=s["rows"])
        k, v = hip_ops.kv4_dequantize(*held, dtype=dt)
    else:
        T = s["k_new"].shape[1]
        t = torch.arange(T, device="cuda")
        at = s["positions"].long()[:, None] + t
        new = torch.ones_like(at, dtype=torch.bool) if s["rows"] is None else t < s["rows"][:, None]
        b, i = new.nonzero(as_tuple=True)
        for name, x in (("k", _rotated(s, s["k_new"].double(), at)), ("v", s["v_new"].double())):
            codes, scale = _coded(x[b, i])
            s[name][b, at[b, i]] = codes
            s[name + "_scale"].permute(0, 3, 1, 2)[b, at[b, i]] = scale
        k, v = (_values(s, name, s["k"].shape[1]).to(dt) for name in ("k", "v"))
    return {"k": k, "v": v}


def _decode(s):
    if own:
        from flashsvd_amd import hip_ops
        return hip_ops.attn_decode_kv4(s["q"], s["k"], s["v"], s["k_scale"], s["v_scale"], s["positions"], cos=s["cos"], sin=s["sin"])
    lens = s["positions"].long()[:, None]
    return _plain_attend(s, _rotated(s, s["q"][:, None].float(), lens), lens, s["case"]["context"])[:, 0].to(s["q"].dtype)


def _prompt(s):
    if own:
        from flashsvd_amd import hip_ops
        return hip_ops.attn_prefill_kv4(s["q"], s["k"], s["v"], s["k_scale"], s["v_scale"], s["positions"], rows=s["rows"], cos=s["cos"], sin=s["sin"], out=s["out"])
    M = s["q"].shape[1]
    at = s["positions"].long()[:, None] + torch.arange(M, device="cuda")
    o = _plain_attend(s, _rotated(s, s["q"].float(), at), at + 1, s["case"]["context"] + M).to(s["q"].dtype)
    if s["rows"] is not None:
        o = torch.where((torch.arange(M, device="cuda") < s["rows"][:, None])[..., None, None], o, s["out"])
    return s["out"].copy_(o)


def _logprobs(s):
    if own:
        from flashsvd_amd import hip_ops
        lp, entropy, top, top_lp = hip_ops.token_logprobs(s["logits"], s["tokens"], top=s["case"]["top"])
    else:
        x = s["logits"].float()
        V = x.shape[1]
        x = x - x.amax(1, keepdim=True)
        w = x.exp()
        z = w.sum(1, keepdim=True)
        entropy = (z.log() - (w * x).sum(1, keepdim=True) / z)[:, 0]
        lp = (x.gather(1, s["tokens"][:, None]) - z.log())[:, 0]
        # whole numbers in the order of the logits, equal ones by index
        bits = s["logits"].view(torch.int16).int()
        order = torch.where(bits >= 0, bits, -32768 - bits).long() * V + torch.arange(V - 1, -1, -1, device="cuda")
        top = V - 1 - order.topk(s["case"]["top"], dim=1).values.remainder(V)
        top_lp = x.gather(1, top) - z.log()
    return {"logprobs": lp, "entropy": entropy, "top": top, "top_logprobs": top_lp}


# ------------------------------------------------------------------ plain forms
def _rotated(s, x, at):
    """x [B, T, heads, Dh] rotated at positions at [B, T]; the two halves of a head are the pairs."""
    if s["cos"] is None:
        return x
    c, n = (t[at.clamp_max(len(t) - 1)].to(x.dtype)[:, :, None] for t in (s["cos"], s["sin"]))
    a, b = x.chunk(2, -1)
    return torch.cat((a * c - b * n, a * n + b * c), -1)


def _coded(x):
    """Codes [.., Dh / 2] and bytes [.., Dh / 32] of values [.., Dh]."""
    g = x.unflatten(-1, (-1, GROUP))
    amax = g.abs().amax(-1)
    mant, ex = torch.frexp(amax)                                    # amax = mant * 2 ** ex, 1/2 <= mant < 1; 7 = 7/8 * 2 ** 3
    e = torch.where(amax > 0, ex - 3 + (mant > 0.875).int(), -125).clamp(-125, 125)
    z = torch.ldexp(g.abs(), -e[..., None]).clamp_max(7.0)
    step = torch.where(z < 2, 0.5, torch.where(z < 4, 1.0, 2.0))
    z = (torch.round(z / step) * step).clamp_max(6.0)
    code = torch.where(z <= 2, 2 * z, torch.where(z <= 4, z + 2, 7.0)).to(torch.uint8) + 8 * (g < 0).to(torch.uint8)
    code = code.flatten(-2).unflatten(-1, (-1, 2))
    return code[..., 0] + 16 * code[..., 1], (e + 127).to(torch.uint8)


def _values(s, name, most):
    """The first `most` rows of the cache in 32 bits, [B, most, Hk, Dh]."""
    table = torch.tensor(CODES + tuple(-c for c in CODES), device="cuda")
    c = s[name][:, :most].int()
    x = torch.stack((table[c & 15], table[c >> 4]), -1).flatten(-2)
    power = (s[name + "_scale"][..., :most].int() << 23).view(torch.float32).permute(0, 3, 1, 2)
    return (x.unflatten(-1, (-1, GROUP)) * power[..., None]).flatten(-2)


def _plain_attend(s, q, lens, most):
    """softmax(q K^T / sqrt(Dh)) V in 32 bits: q [B, M, H, Dh], row m of b over the first lens[b, m] cached rows, none of them beyond `most`."""
    B, M, H, Dh = q.shape
    Hk = s["case"]["kv_heads"]
    k, v = (_values(s, x, most).transpose(1, 2).contiguous() for x in ("k", "v"))
    q = q.transpose(1, 2).reshape(B, Hk, H // Hk * M, Dh)
    w = torch.matmul(q, k.transpose(2, 3).contiguous()).div_(math.sqrt(Dh)).view(B, H, M, most)
    w.masked_fill_((torch.arange(most, device="cuda") >= lens[..., None])[:, None], -math.inf)
    w.sub_(w.amax(-1, keepdim=True).clamp_min(-1e30)).exp_()
    total = w.sum(-1, keepdim=True)
    o = torch.matmul(w.view(B, Hk, -1, most), v).view(B, H, M, Dh) / torch.where(total > 0, total, 1.0)
    return o.transpose(1, 2)


# ------------------------------------------------------------------ in 64 bits, from the definition
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "logprobs":
        out = {"logprobs": [], "entropy": [], "top": None, "top_logprobs": []}
        for rows, tokens in zip(s["logits"].split(256), s["tokens"].split(256)):
            lp = torch.log_softmax(rows.double(), 1)
            out["logprobs"].append(lp[torch.arange(len(lp)), tokens])
            out["entropy"].append(-(lp.exp() * lp).sum(1))
            out["top_logprobs"].append(torch.sort(lp, 1, descending=True).values[:, :case["top"]])
        return {k: torch.cat(v) if v is not None else None for k, v in out.items()}
    B, Dh, Hk = case["batch"], case["head_dim"], case["kv_heads"]
    turn = torch.complex(s["cos"].double(), s["sin"].double()) if case["rotate"] else None

    def rotate(x, first):
        """x [T, heads, Dh] whose first row stands at position `first`"""
        x = x.double()
        if turn is None:
            return x
        z = torch.complex(x[..., : Dh // 2], x[..., Dh // 2:]) * turn[(first + torch.arange(len(x), device="cuda")).clamp_max(len(turn) - 1), None]
        return torch.cat((z.real, z.imag), -1)

    def held(name, b):
        """what the cache of sequence b stands for, [S, Hk, Dh]"""
        c = s[name][b].long()
        x = torch.empty(*c.shape[:2], Dh, dtype=torch.double, device="cuda")
        for i, half in enumerate((c % 16, c // 16)):
            size = torch.tensor(CODES, dtype=torch.double, device="cuda")[half % 8]
            x[..., i::2] = torch.where(half > 7, -size, size)
        return x * torch.exp2(s[name + "_scale"][b].double() - 127.0).permute(2, 0, 1).repeat_interleave(GROUP, 2)

    past, new = _contexts(case), _rows(case)
    if case["kind"] == "append":
        grid = torch.tensor(CODES, dtype=torch.double, device="cuda")
        middle = (grid[1:] + grid[:-1]) / 2                         # a tie goes to the code with the even number
        powers = torch.exp2(torch.arange(-125, 126, device="cuda").double())
        out = {"k": [], "v": []}
        for b in range(B):
            p, t = past[b], new[b]
            for name, rows in (("k", rotate(s["k_new"][b, :t], p)), ("v", s["v_new"][b, :t].double())):
                x = rows.view(t, Hk, Dh // GROUP, GROUP)
                size = powers[torch.searchsorted(7.0 * powers, x.abs().amax(-1))][..., None]
                y = x.abs() / size
                up, down = torch.bucketize(y, middle, right=True), torch.bucketize(y, middle)        # they differ on a tie
                value = torch.where(up % 2 == 0, grid[up], grid[down]) * size
                whole = held(name, b)
                whole[p:p + t] = torch.where(x < 0, -value, value).view(t, Hk, Dh)
                out[name].append(whole)
        return {k: torch.stack(v) for k, v in out.items()}
    H, M = case["heads"], case["tokens"]
    out = torch.zeros(B, M, H, Dh, dtype=torch.double, device="cuda")
    q_all = s["q"].view(B, M, H, Dh)
    for b in range(B):
        p, t = past[b], new[b]
        L = p + (t if case["kind"] == "prompt" else 0)
        if L == 0:
            continue
        k, v = (held(x, b)[:L] for x in ("k", "v"))
        q = rotate(q_all[b, :t], p)
        seen = p + torch.arange(t, device="cuda") + (1 if case["kind"] == "prompt" else 0)
        unseen = torch.arange(L, device="cuda") >= seen[:, None]
        for h in range(H):
            hk = h // (H // Hk)
            a = q[:, h] @ k[:, hk].t() / Dh ** 0.5
            out[b, :t, h] = torch.softmax(a.masked_fill(unseen, -math.inf), 1) @ v[:, hk]
    return out.view(s["q"].shape)
