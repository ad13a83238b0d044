"""KV caches of the decode path.

``FlashSVDV15DenseKVCache`` keeps post-RoPE K and V per layer as [Bmax, Smax, Hk, Dh]
(runtime/cache/attn_dense_kv.py:7-357 of the reference); ``FlashSVDLegacySparseKVCache`` keeps
the pre-RoPE rank coefficients Pk, Pv per layer as [Bmax, Smax, R]
(runtime/cache/attn_legacy_sparse_kv.py:22-257).  ``FlashSVDKV8Cache`` keeps K and V in 8 bits, ``FlashSVDKV4Cache`` in 4.  All are plain Python objects (no dependency
on the transformers ``Cache`` base class) with the method names, return values and error
behaviour the reference's callers rely on.  Storage is allocated once at full size so that
decode kernels can write in place and a captured HIP graph keeps valid pointers.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Any, Optional

import torch


def _as_device(d) -> torch.device:
    return torch.device("cuda", d) if isinstance(d, int) else torch.device(d)


def _rope_tables(cache: dict, seqlen: int, head_dim: int, theta: float, device, dtype):
    key = (int(seqlen), int(head_dim), float(theta), dtype, torch.device(device))
    hit = cache.get(key)
    if hit is not None:
        return hit
    if head_dim % 2:
        raise ValueError(f"head_dim must be even, got {head_dim}")
    half = head_dim // 2
    pos = torch.arange(int(seqlen), device=device, dtype=torch.float32)
    inv_freq = 1.0 / (float(theta) ** (torch.arange(0, half, device=device, dtype=torch.float32) / half))
    ang = pos[:, None] * inv_freq[None, :]
    pair = (torch.cos(ang).to(dtype).contiguous(), torch.sin(ang).to(dtype).contiguous())
    cache[key] = pair
    return pair


class _CacheBase:
    is_compileable = False

    def __init__(self, config, max_batch_size: int, max_cache_len: int, device, dtype, layer_device_map):
        self._config = config
        self._max_batch_size = int(max_batch_size)
        self._max_cache_len = int(max_cache_len)
        self._dtype = dtype
        self._rope_theta = float(getattr(config, "rope_theta", 10000.0))
        self._seen_tokens = 0
        self._rope_cache: dict = {}
        n_layers = int(getattr(config, "num_hidden_layers", 0))
        base = torch.device(device) if device is not None else torch.device("cpu")
        self._layer_device = [
            _as_device(layer_device_map[i]) if layer_device_map is not None else base for i in range(n_layers)]
        self._layer_initialized = [False] * n_layers
        self.key_cache: list[torch.Tensor] = []
        self.value_cache: list[torch.Tensor] = []

    max_batch_size = property(lambda self: self._max_batch_size)
    max_cache_len = property(lambda self: self._max_cache_len)

    def __len__(self) -> int:
        return len(self.key_cache)

    def get_seq_length(self, layer_idx: Optional[int] = 0) -> int:
        return int(self._seen_tokens)

    def get_max_cache_shape(self) -> Optional[int]:
        return self._max_cache_len

    def get_mask_sizes(self, cache_position: torch.Tensor, layer_idx: int) -> tuple[int, int]:
        return int(cache_position.shape[0]) + int(self._seen_tokens), 0

    def get_rope_tables(self, *, seqlen: int, head_dim: int, device, dtype):
        """(cos, sin), each [seqlen, head_dim/2]: fp32 angles pos * theta^(-i/half) cast to ``dtype``."""
        return _rope_tables(self._rope_cache, seqlen, head_dim, self._rope_theta, device, dtype)

    def _note_seen(self, layer_idx: int, q_len: int, cache_position) -> None:
        """Only layer 0 advances the token count; exact for host positions, sequential otherwise."""
        if int(layer_idx) != 0:
            return
        if cache_position is None:
            self._seen_tokens = max(self._seen_tokens, int(q_len))
        elif torch.is_tensor(cache_position) and not cache_position.is_cuda and cache_position.numel() > 0:
            self._seen_tokens = max(self._seen_tokens, int(cache_position.max()) + 1)
        else:
            self._seen_tokens = self._seen_tokens + int(q_len)

    def reset(self) -> None:
        self._seen_tokens = 0


class _HeadCacheBase(_CacheBase):
    """What the caches of whole heads share: head counts learnt from the first write, the device buffers of the decoded positions."""

    def __init__(self, config, max_batch_size: int, max_cache_len: int, device, dtype, layer_device_map):
        super().__init__(config, max_batch_size, max_cache_len, device, dtype, layer_device_map)
        self._layer_heads = [0] * len(self._layer_device)
        self._layer_head_dim = [0] * len(self._layer_device)
        self._seqlens: dict[tuple[int, int], torch.Tensor] = {}

    def _seqlens_buffer(self, layer_idx: int, batch_size: int) -> torch.Tensor:
        key = (int(layer_idx), int(batch_size))
        dev = self.key_cache[int(layer_idx)].device
        buf = self._seqlens.get(key)
        if buf is None or buf.device != dev:
            buf = torch.empty((int(batch_size),), device=dev, dtype=torch.int32)
            self._seqlens[key] = buf
        return buf

    @staticmethod
    def _fill_cache_seqlens_buffer(cache_seqlens: torch.Tensor, *, seen_tokens: int, cache_position=None) -> torch.Tensor:
        if cache_position is None:
            cache_seqlens.fill_(int(seen_tokens))
        elif torch.is_tensor(cache_position):
            pos = cache_position.to(device=cache_seqlens.device, dtype=torch.int32).reshape(-1)
            if pos.numel() == 0:
                cache_seqlens.zero_()
            elif pos.numel() == 1:
                cache_seqlens.copy_(pos.expand_as(cache_seqlens))
            else:
                cache_seqlens.copy_(pos[: cache_seqlens.shape[0]])
        else:
            cache_seqlens.fill_(int(cache_position))
        return cache_seqlens

    def advance_after_fa2(self, layer_idx: int, *, q_len: int, cache_position) -> None:
        if int(layer_idx) != 0:
            return
        if cache_position is not None and torch.is_tensor(cache_position) and not cache_position.is_cuda \
                and cache_position.numel() > 0:
            self._seen_tokens = max(self._seen_tokens, int(cache_position.max()) + 1)
        else:
            self._seen_tokens = self._seen_tokens + int(q_len)


class FlashSVDV15DenseKVCache(_HeadCacheBase):
    """Dense KV cache, [B, S, Hk, Dh] per layer, K stored after RoPE."""

    def __init__(self, config, *, max_batch_size: int, max_cache_len: int, device=None,
                 dtype: torch.dtype = torch.float16, layer_device_map: Optional[dict] = None) -> None:
        super().__init__(config, max_batch_size, max_cache_len, device, dtype, layer_device_map)
        for dev in self._layer_device:
            # shaped lazily: head count / head_dim are learnt from the first write
            self.key_cache.append(torch.zeros((self._max_batch_size, self._max_cache_len, 0, 0), dtype=dtype, device=dev))
            self.value_cache.append(torch.zeros((self._max_batch_size, self._max_cache_len, 0, 0), dtype=dtype, device=dev))

    # -- storage ---------------------------------------------------------------------------
    def _ensure_layer_spec(self, layer_idx: int, *, h: int, dh: int) -> None:
        layer_idx, h, dh = int(layer_idx), int(h), int(dh)
        cur = self.key_cache[layer_idx]
        if (cur.shape[2], cur.shape[3]) == (h, dh):
            return
        if self._layer_initialized[layer_idx]:
            raise RuntimeError(
                f"FlashSVDV15DenseKVCache shape changed after init for layer {layer_idx}: "
                f"old={(int(cur.shape[2]), int(cur.shape[3]))}, new={(h, dh)}")
        shape = (self._max_batch_size, self._max_cache_len, h, dh)
        self.key_cache[layer_idx] = torch.zeros(shape, dtype=self._dtype, device=self._layer_device[layer_idx])
        self.value_cache[layer_idx] = torch.zeros(shape, dtype=self._dtype, device=self._layer_device[layer_idx])
        self._layer_heads[layer_idx], self._layer_head_dim[layer_idx] = h, dh

    # -- HF-style update (prefill copy or positional scatter) -------------------------------
    def update(self, key_states: torch.Tensor, value_states: torch.Tensor, layer_idx: int,
               cache_kwargs: Optional[dict[str, Any]] = None):
        """key/value_states are [B, Hk, T, Dh]; returns the valid cache prefix as [B, Hk, L, Dh]."""
        layer_idx = int(layer_idx)
        cache_position = (cache_kwargs or {}).get("cache_position")
        self._ensure_layer_spec(layer_idx, h=key_states.shape[1], dh=key_states.shape[-1])
        kc, vc = self.key_cache[layer_idx], self.value_cache[layer_idx]
        k_bshd = key_states.to(device=kc.device, dtype=kc.dtype).transpose(1, 2)
        v_bshd = value_states.to(device=vc.device, dtype=vc.dtype).transpose(1, 2)
        b, t = k_bshd.shape[0], k_bshd.shape[1]
        if cache_position is None:
            kc[:b, :t].copy_(k_bshd)
            vc[:b, :t].copy_(v_bshd)
        else:
            idx = cache_position.to(device=kc.device)
            kc[:b].index_copy_(1, idx, k_bshd.contiguous())
            vc[:b].index_copy_(1, idx, v_bshd.contiguous())
        self._layer_initialized[layer_idx] = True
        self._note_seen(layer_idx, t, cache_position)
        n = t if cache_position is None else int(self.get_seq_length())
        return kc[:b, :n].transpose(1, 2).contiguous(), vc[:b, :n].transpose(1, 2).contiguous()

    # -- decode-step helpers ------------------------------------------------------------------
    def prepare_fa2_step(self, layer_idx: int, *, batch_size: int, cache_position=None):
        """(k_cache[:B], v_cache[:B], cache_seqlens int32 [B]) for an attend-with-append kernel."""
        layer_idx, batch_size = int(layer_idx), int(batch_size)
        lens = self._seqlens_buffer(layer_idx, batch_size)
        self._fill_cache_seqlens_buffer(lens, seen_tokens=self.get_seq_length(), cache_position=cache_position)
        return self.key_cache[layer_idx][:batch_size], self.value_cache[layer_idx][:batch_size], lens

    def get_fa2_kvcache(self, layer_idx: int, *, batch_size: int):
        return self.prepare_fa2_step(layer_idx, batch_size=batch_size, cache_position=None)

    def prepare_fa2_direct_write_step(self, layer_idx: int, *, batch_size: int, num_heads: int, head_dim: int,
                                      q_len: int, cache_position=None):
        """Views for writing the current token straight into the cache: (k_cache, v_cache,
        k_slot, v_slot, cache_seqlens = start + q_len).  None unless q_len == 1 and all
        positions are equal; IndexError if the slot is outside the cache."""
        layer_idx, batch_size, q_len = int(layer_idx), int(batch_size), int(q_len)
        if q_len != 1:
            return None
        self._ensure_layer_spec(layer_idx, h=num_heads, dh=head_dim)
        if cache_position is None:
            start = int(self.get_seq_length())
        elif torch.is_tensor(cache_position):
            pos = cache_position.reshape(-1)
            if pos.numel() == 0:
                return None
            vals = pos.tolist()  # one host read, like the reference
            if any(v != vals[0] for v in vals):
                return None
            start = int(vals[0])
        else:
            start = int(cache_position)
        if start < 0 or start + q_len > self._max_cache_len:
            raise IndexError(
                f"FlashSVDV15DenseKVCache write position out of range: start={start} q_len={q_len} max={self._max_cache_len}")
        kc, vc = self.key_cache[layer_idx][:batch_size], self.value_cache[layer_idx][:batch_size]
        lens = self._seqlens_buffer(layer_idx, batch_size)
        lens.fill_(start + q_len)
        self._layer_initialized[layer_idx] = True
        return kc, vc, kc[:, start:start + q_len], vc[:, start:start + q_len], lens

    def clone_for_autotune(self, *, layer_idx: int, batch_size: int) -> "FlashSVDV15DenseKVCache":
        """A scratch copy holding only ``layer_idx``'s first ``batch_size`` rows."""
        layer_idx, batch_size = int(layer_idx), int(batch_size)
        other = type(self)(self._config, max_batch_size=self._max_batch_size, max_cache_len=self._max_cache_len,
                           device=self._layer_device[0] if self._layer_device else None, dtype=self._dtype,
                           layer_device_map=dict(enumerate(self._layer_device)))
        other._seen_tokens = self._seen_tokens
        h, dh = self._layer_heads[layer_idx], self._layer_head_dim[layer_idx]
        if h > 0 and dh > 0:
            other._ensure_layer_spec(layer_idx, h=h, dh=dh)
            other.key_cache[layer_idx][:batch_size].copy_(self.key_cache[layer_idx][:batch_size])
            other.value_cache[layer_idx][:batch_size].copy_(self.value_cache[layer_idx][:batch_size])
            other._layer_initialized[layer_idx] = self._layer_initialized[layer_idx]
        return other


class _CodesCacheBase(_HeadCacheBase):
    """What the caches of codes and scales share: storage by the head count of the first write, the operands of the operators."""

    def _make_lists(self) -> None:
        self.key_scale: list[torch.Tensor] = []
        self.value_scale: list[torch.Tensor] = []
        for dev in self._layer_device:
            codes, scale = self._storage(0, 0, dev)
            self.key_cache.append(codes)
            self.value_cache.append(codes)
            self.key_scale.append(scale)
            self.value_scale.append(scale)

    def _ensure_layer_spec(self, layer_idx: int, *, h: int, dh: int) -> None:
        layer_idx, h, dh = int(layer_idx), int(h), int(dh)
        old = (self._layer_heads[layer_idx], self._layer_head_dim[layer_idx])
        if old == (h, dh):
            return
        if self._layer_initialized[layer_idx]:
            raise RuntimeError(f"{type(self).__name__} shape changed after init for layer {layer_idx}: old={old}, new={(h, dh)}")
        dev = self._layer_device[layer_idx]
        self.key_cache[layer_idx], self.key_scale[layer_idx] = self._storage(h, dh, dev)
        self.value_cache[layer_idx], self.value_scale[layer_idx] = self._storage(h, dh, dev)
        self._layer_heads[layer_idx], self._layer_head_dim[layer_idx] = h, dh

    def operands(self, layer_idx: int, batch_size: int):
        """(key codes, value codes, key scales, value scales) of the first ``batch_size`` sequences, as the operators take them."""
        i, b = int(layer_idx), int(batch_size)
        return self.key_cache[i][:b], self.value_cache[i][:b], self.key_scale[i][:b], self.value_scale[i][:b]


class FlashSVDKV8Cache(_CodesCacheBase):
    """Dense KV cache in 8 bits: per layer e4m3 codes [B, S, Hk, Dh] of K (after RoPE) and V, and one float32 power of two for each
    block of ``block_size`` tokens (16, 32, 64 or 128) of a kv head, [B, ceil(S / block_size), Hk]; ``value = code * scale``.

    Half the bytes of :class:`FlashSVDV15DenseKVCache` and its method names where they make sense; rows are written by
    ``hip_ops.kv8_append`` and read by ``hip_ops.attn_decode_kv8`` / ``attn_prefill_kv8``.  ``dtype`` is that of the activations.  A row's
    tokens stand side by side for each head in memory (the kernels take any strides).  Writing a position makes it the last valid one
    of its block, so rows are written in order: a write at an earlier position gives up the rows behind it, and the held length
    (``get_seq_length()``) is what it leaves, where the caches of 16 bits keep the largest.  A token whose position is on the device
    counts as one further.  No counterpart in the reference, whose caches are of 16 bits."""

    def __init__(self, config, *, max_batch_size: int, max_cache_len: int, block_size: int = 32, device=None, dtype: torch.dtype = torch.float16,
                 layer_device_map: Optional[dict] = None) -> None:
        super().__init__(config, max_batch_size, max_cache_len, device, dtype, layer_device_map)
        if int(block_size) not in (16, 32, 64, 128):
            raise ValueError(f"block_size must be 16, 32, 64 or 128 tokens, got {block_size}")
        self.block_size = int(block_size)
        self._make_lists()

    def _storage(self, h: int, dh: int, dev):
        codes = torch.zeros((self._max_batch_size, h, self._max_cache_len, dh), dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
        scale = torch.zeros((self._max_batch_size, h, -(-self._max_cache_len // self.block_size)), dtype=torch.float32, device=dev)
        return codes.transpose(1, 2), scale.transpose(1, 2)

    def _note_seen(self, layer_idx: int, q_len: int, cache_position) -> None:
        if int(layer_idx) != 0 or int(q_len) == 0:
            return
        if cache_position is None:
            self._seen_tokens = int(q_len)
            return
        pos = torch.as_tensor(cache_position).reshape(-1)
        if int(q_len) != 1:                                # a chunk: its first position
            self._seen_tokens = (int(pos[0]) if pos.numel() else self._seen_tokens) + int(q_len)
        elif pos.is_cuda:
            self._seen_tokens += 1
        else:
            self._seen_tokens = int(pos.max()) + 1

    def advance_after_fa2(self, layer_idx: int, *, q_len: int, cache_position) -> None:
        self._note_seen(layer_idx, q_len, self._seen_tokens if cache_position is None else cache_position)

    def append(self, layer_idx: int, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, *, cos=None, sin=None, rows=None) -> None:
        """``hip_ops.kv8_append`` of rows k, v [B, T, Hk, Dh] at positions int32 [B] of this layer."""
        from .. import hip_ops
        self._ensure_layer_spec(layer_idx, h=k.shape[2], dh=k.shape[3])
        hip_ops.kv8_append(k, v, *self.operands(layer_idx, k.shape[0]), positions, block=self.block_size, cos=cos, sin=sin, rows=rows)
        self._layer_initialized[int(layer_idx)] = True

    def attend_token(self, layer_idx: int, q: torch.Tensor, positions: torch.Tensor, **kw) -> torch.Tensor:
        """``hip_ops.attn_decode_kv8`` of one query token per sequence, q [B, H, Dh], over this layer."""
        from .. import hip_ops
        return hip_ops.attn_decode_kv8(q, *self.operands(layer_idx, q.shape[0]), positions, block=self.block_size, **kw)

    def attend_chunk(self, layer_idx: int, q: torch.Tensor, positions: torch.Tensor, **kw) -> torch.Tensor:
        """``hip_ops.attn_prefill_kv8`` of a chunk q [B, M, H, Dh] that the cache holds, over this layer."""
        from .. import hip_ops
        return hip_ops.attn_prefill_kv8(q, *self.operands(layer_idx, q.shape[0]), positions, block=self.block_size, **kw)

    def dequantize(self, layer_idx: int, *, batch_size: Optional[int] = None, length: Optional[int] = None):
        """(K, V) of the first ``length`` positions as ``dtype`` [B, L, Hk, Dh]."""
        i = int(layer_idx)
        b = self._max_batch_size if batch_size is None else int(batch_size)
        n = self._max_cache_len if length is None else int(length)
        out = []
        for codes, scale in ((self.key_cache[i], self.key_scale[i]), (self.value_cache[i], self.value_scale[i])):
            full = scale[:b].repeat_interleave(self.block_size, 1)[:, :n, :, None]
            out.append((codes[:b, :n].float() * full).to(self._dtype))
        return out[0], out[1]

    def update(self, key_states: torch.Tensor, value_states: torch.Tensor, layer_idx: int, cache_kwargs: Optional[dict[str, Any]] = None):
        """key/value_states are [B, Hk, T, Dh] (keys rotated) for consecutive positions; returns what the cache holds then, up to the last row
        written, as [B, Hk, L, Dh]."""
        cache_position = (cache_kwargs or {}).get("cache_position")
        t, start = key_states.shape[2], 0
        if cache_position is not None:
            pos = cache_position.reshape(-1).tolist()
            if not pos or pos != list(range(pos[0], pos[0] + t)):
                raise ValueError("FlashSVDKV8Cache takes consecutive positions: a block's scale is that of the rows up to the last one written")
            start = pos[0]
        if start < 0 or start + t > self._max_cache_len:
            raise IndexError(f"FlashSVDKV8Cache write position out of range: start={start} q_len={t} max={self._max_cache_len}")
        dev = self._layer_device[int(layer_idx)]
        k, v = (x.to(device=dev, dtype=self._dtype).transpose(1, 2) for x in (key_states, value_states))
        k, v = (x if x.stride(-1) == 1 else x.contiguous() for x in (k, v))
        self.append(layer_idx, k, v, torch.full((k.shape[0],), start, dtype=torch.int32, device=dev))
        self._note_seen(layer_idx, t, torch.tensor([start]))
        k, v = self.dequantize(layer_idx, batch_size=k.shape[0], length=start + t)
        return k.transpose(1, 2).contiguous(), v.transpose(1, 2).contiguous()


class FlashSVDKV4Cache(_CodesCacheBase):
    """Dense KV cache in 4 bits: per layer two e2m1 codes a byte, [B, S, Hk, Dh / 2], of K (after RoPE) and V, and one byte for each 32 channels of a token,
    [B, Hk, Dh / 32, S]; ``value = code * 2 ** (byte - 127)``: 4.25 bits a number.

    Heads of 64 or 128 dimensions.  A row's codes and scales are its own, so positions are written in any order, again too, and the held length is that of
    :class:`FlashSVDV15DenseKVCache`.  Rows are written by ``hip_ops.kv4_append`` and read by ``hip_ops.attn_decode_kv4`` / ``attn_prefill_kv4``.  ``dtype`` is that
    of the activations.  S is ``max_cache_len`` rounded up to 64 tokens, the operators' tile; rows behind ``max_cache_len`` are dropped and not seen.  No counterpart in
    the reference, whose caches are of 16 bits."""

    TILE = 64

    def __init__(self, config, *, max_batch_size: int, max_cache_len: int, device=None, dtype: torch.dtype = torch.float16,
                 layer_device_map: Optional[dict] = None) -> None:
        super().__init__(config, max_batch_size, max_cache_len, device, dtype, layer_device_map)
        self._limit = self._max_cache_len if self._max_cache_len % self.TILE else None      # for the operators, of the room
        self._make_lists()

    def _storage(self, h: int, dh: int, dev):
        if dh not in (0, 64, 128):
            raise ValueError(f"FlashSVDKV4Cache takes heads of 64 or 128 dimensions, got {dh}")
        room = -(-self._max_cache_len // self.TILE) * self.TILE
        codes = torch.zeros((self._max_batch_size, h, room, dh // 2), dtype=torch.uint8, device=dev)
        return codes.transpose(1, 2), torch.zeros((self._max_batch_size, h, dh // 32, room), dtype=torch.uint8, device=dev)

    def append(self, layer_idx: int, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, *, cos=None, sin=None, rows=None) -> None:
        """``hip_ops.kv4_append`` of rows k, v [B, T, Hk, Dh] at positions int32 [B] of this layer."""
        self._write(layer_idx, k, v, positions, cos=cos, sin=sin, rows=rows, limit=self._limit)

    def _write(self, layer_idx: int, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, **kw) -> None:
        from .. import hip_ops
        self._ensure_layer_spec(layer_idx, h=k.shape[2], dh=k.shape[3])
        hip_ops.kv4_append(k, v, *self.operands(layer_idx, k.shape[0]), positions, **kw)
        self._layer_initialized[int(layer_idx)] = True

    def attend_token(self, layer_idx: int, q: torch.Tensor, positions: torch.Tensor, **kw) -> torch.Tensor:
        """``hip_ops.attn_decode_kv4`` of one query token per sequence, q [B, H, Dh], over this layer."""
        from .. import hip_ops
        return hip_ops.attn_decode_kv4(q, *self.operands(layer_idx, q.shape[0]), positions, limit=self._limit, **kw)

    def attend_chunk(self, layer_idx: int, q: torch.Tensor, positions: torch.Tensor, **kw) -> torch.Tensor:
        """``hip_ops.attn_prefill_kv4`` of a chunk q [B, M, H, Dh] that the cache holds, over this layer."""
        from .. import hip_ops
        return hip_ops.attn_prefill_kv4(q, *self.operands(layer_idx, q.shape[0]), positions, limit=self._limit, **kw)

    def dequantize(self, layer_idx: int, *, batch_size: Optional[int] = None, length: Optional[int] = None):
        """(K, V) of the first ``length`` positions as ``dtype`` [B, L, Hk, Dh] (``hip_ops.kv4_dequantize``)."""
        from .. import hip_ops
        b = self._max_batch_size if batch_size is None else int(batch_size)
        n = self._max_cache_len if length is None else int(length)
        return hip_ops.kv4_dequantize(*self.operands(layer_idx, b), length=n, dtype=self._dtype)

    def update(self, key_states: torch.Tensor, value_states: torch.Tensor, layer_idx: int, cache_kwargs: Optional[dict[str, Any]] = None):
        """key/value_states are [B, Hk, T, Dh] (keys rotated), row t for position ``cache_position[t]`` (t without it); returns what the cache holds then as
        [B, Hk, L, Dh]."""
        cache_position = (cache_kwargs or {}).get("cache_position")
        t = key_states.shape[2]
        pos = list(range(t)) if cache_position is None else cache_position.reshape(-1).tolist()
        if len(pos) != t:
            raise ValueError(f"FlashSVDKV4Cache needs a position for each of {t} rows, got {len(pos)}")
        if pos and (min(pos) < 0 or max(pos) >= self._max_cache_len):
            raise IndexError(f"FlashSVDKV4Cache write position out of range: positions {min(pos)} to {max(pos)} max={self._max_cache_len}")
        dev = self._layer_device[int(layer_idx)]
        k, v = (x.to(device=dev, dtype=self._dtype).transpose(1, 2) for x in (key_states, value_states))
        k, v = (x if x.stride(-1) == 1 else x.contiguous() for x in (k, v))
        b, first = k.shape[0], 0
        self._ensure_layer_spec(layer_idx, h=k.shape[2], dh=k.shape[3])
        for i in range(1, t + 1):                          # a call for each run of consecutive positions
            if i == t or pos[i] != pos[i - 1] + 1:
                self._write(layer_idx, k[:, first:i], v[:, first:i], torch.full((b,), pos[first], dtype=torch.int32, device=dev))      # inside: checked above
                first = i
        self._note_seen(layer_idx, t, None if cache_position is None else torch.tensor(pos, dtype=torch.long))      # on the host, where they have been read
        n = t if cache_position is None else int(self.get_seq_length())
        k, v = self.dequantize(layer_idx, batch_size=b, length=min(n, self._max_cache_len))
        return k.transpose(1, 2).contiguous(), v.transpose(1, 2).contiguous()


@dataclass
class _DecodeWorkspace:
    """Split-K scratch of the rank-space decode kernel: running max / sum [B,H,S] fp32, rank-space
    accumulator [B,H,S,R] fp32 and the two pre-rotated query halves [B,H,Dh/2]."""
    M: torch.Tensor
    L: torch.Tensor
    Acc: torch.Tensor
    Q0: torch.Tensor
    Q1: torch.Tensor


class FlashSVDLegacySparseKVCache(_CacheBase):
    """Rank-space KV cache: Pk = X @ k_v^T and Pv = X @ v_v^T (pre-RoPE), [B, S, R] per layer.
    K/V heads are rebuilt inside the decode kernel from the per-head bases."""

    def __init__(self, config, *, max_batch_size: int, max_cache_len: int, rank: Optional[int] = None,
                 rank_k: Optional[int] = None, rank_v: Optional[int] = None, device=None,
                 dtype: torch.dtype = torch.float16, layer_device_map: Optional[dict] = None) -> None:
        super().__init__(config, max_batch_size, max_cache_len, device, dtype, layer_device_map)
        if rank is not None:
            rank_k = rank_v = int(rank)
        rk, rv = int(rank_k or 0), int(rank_v or 0)
        self.rank = int(rk or rv or 0)  # hint only; per-layer ranks may differ
        for dev in self._layer_device:
            self.key_cache.append(torch.zeros((self._max_batch_size, self._max_cache_len, rk), dtype=dtype, device=dev))
            self.value_cache.append(torch.zeros((self._max_batch_size, self._max_cache_len, rv), dtype=dtype, device=dev))
        self._layer_key_rank = [rk] * len(self._layer_device)
        self._layer_value_rank = [rv] * len(self._layer_device)
        self._decode_workspaces: dict = {}

    def ensure_layer_ranks(self, layer_idx: int, k_rank: int, v_rank: int) -> None:
        layer_idx, k_rank, v_rank = int(layer_idx), int(k_rank), int(v_rank)
        kc, vc = self.key_cache[layer_idx], self.value_cache[layer_idx]
        if kc.shape[-1] == k_rank and vc.shape[-1] == v_rank:
            return
        if self._layer_initialized[layer_idx]:
            raise RuntimeError(
                "FlashSVDLegacySparseKVCache rank changed after initialization for layer "
                f"{layer_idx}: cache.key_rank={int(kc.shape[-1])} cache.value_rank={int(vc.shape[-1])} "
                f"but got key rank {k_rank}, value rank {v_rank}.")
        dev = self._layer_device[layer_idx]
        self.key_cache[layer_idx] = torch.zeros((self._max_batch_size, self._max_cache_len, k_rank), dtype=self._dtype, device=dev)
        self.value_cache[layer_idx] = torch.zeros((self._max_batch_size, self._max_cache_len, v_rank), dtype=self._dtype, device=dev)
        self._layer_key_rank[layer_idx], self._layer_value_rank[layer_idx] = k_rank, v_rank
        self.rank = int(self.rank or k_rank or v_rank)

    def update(self, key_states: torch.Tensor, value_states: torch.Tensor, layer_idx: int,
               cache_kwargs: Optional[dict[str, Any]] = None):
        """key/value_states are rank coefficients [B, T, R]; returned unchanged (cast to the cache dtype)."""
        layer_idx = int(layer_idx)
        cache_position = (cache_kwargs or {}).get("cache_position")
        self.ensure_layer_ranks(layer_idx, key_states.shape[-1], value_states.shape[-1])
        kc, vc = self.key_cache[layer_idx], self.value_cache[layer_idx]
        key_states = key_states.to(dtype=kc.dtype, device=kc.device)
        value_states = value_states.to(dtype=vc.dtype, device=vc.device)
        self._layer_initialized[layer_idx] = True
        b, t = key_states.shape[0], key_states.shape[1]
        if cache_position is None:
            kc[:b, :t].copy_(key_states)
            vc[:b, :t].copy_(value_states)
        else:
            idx = cache_position.to(device=kc.device)
            kc[:b].index_copy_(1, idx, key_states)
            vc[:b].index_copy_(1, idx, value_states)
        self._note_seen(layer_idx, t, cache_position)
        return key_states, value_states

    def get_decode_workspace(self, *, batch_size: int, num_heads: int, rank: int, head_dim: int, max_splits: int,
                             device, dtype) -> _DecodeWorkspace:
        key = (int(batch_size), int(num_heads), int(rank), int(max_splits), dtype, torch.device(device))
        ws = self._decode_workspaces.get(key)
        if ws is None:
            if head_dim % 2:
                raise ValueError(f"head_dim must be even, got {head_dim}")
            b, h, r, s = key[:4]
            f32 = dict(device=device, dtype=torch.float32)
            ws = _DecodeWorkspace(M=torch.empty((b, h, s), **f32), L=torch.empty((b, h, s), **f32),
                                  Acc=torch.empty((b, h, s, r), **f32),
                                  Q0=torch.empty((b, h, head_dim // 2), device=device, dtype=dtype),
                                  Q1=torch.empty((b, h, head_dim // 2), device=device, dtype=dtype))
            self._decode_workspaces[key] = ws
        return ws


# names kept for older imports
FlashSVDDenseKVCache = FlashSVDV15DenseKVCache
LowRankKVCache = FlashSVDLegacySparseKVCache
