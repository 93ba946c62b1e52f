"""Preallocated, API-compatible KV caches, in bf16 and in 4 bits.

The reference passes ``past_kv = (past_k, past_v)`` to the attention and
builds ``k = cat(past_k, k)`` every step (REF modules/attention.py:89-93),
copying the whole history (1.07 GB per layer per step at 64 sequences x 8192
positions).  ``LayerKVCache`` holds one layer's K/V in buffers of a fixed
capacity, ``[B, Hkv, capacity, D]`` bf16; ``CudaFullAttention`` appends the new
rows in place (``q35_kv_append``) and attends over the buffers directly (the
attention kernels take the capacity as the per-head row stride).
``Q4LayerKVCache`` holds the same rows as 4-bit codes (0.31 of the bytes at
head_dim 128 and groups of 32).

Compatibility: a ``LayerKVCache`` unpacks and indexes like the ``(k, v)``
tuple of the reference API -- ``k, v = cache`` and ``cache[0]`` give the valid
rows ``[B, Hkv, length, D]`` (views; bf16 copies for a 4-bit cache) -- and it is
what the attention returns as ``new_kv``.  ``KVCache`` / ``Q4KVCache`` are the
per-model lists (``past_key_values``).

The length advances on the host when the attention runs, so a cache is meant
for eager decode loops, one forward at a time.  A 4-bit cache can instead keep a
length per sequence on the device (``set_lengths``): sequences of different
lengths then decode together, and a captured decode step advances on replay.
"""
from __future__ import annotations

import torch


class LayerKVCache:
    lengths: torch.Tensor | None = None  # per-sequence lengths (4-bit caches only)

    def __init__(self, batch: int, num_kv_heads: int, capacity: int, head_dim: int,
                 device, dtype: torch.dtype = torch.bfloat16):
        if capacity < 1:
            raise ValueError("capacity must be positive")
        # zero-initialised: the last key tile of an attention call reads rows
        # past the valid length (masked), which must hold finite values
        self.k = torch.zeros(batch, num_kv_heads, capacity, head_dim, device=device, dtype=dtype)
        self.v = torch.zeros_like(self.k)
        self.length = 0

    @property
    def capacity(self) -> int:
        return self.k.shape[2]

    def views(self) -> tuple[torch.Tensor, torch.Tensor]:
        return self.k[:, :, :self.length], self.v[:, :, :self.length]

    def append_attend(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float,
                      causal: bool) -> torch.Tensor:
        """Appends k/v (B,Hkv,S,D), advances the length and attends q (B,Hq,S,D)
        over all rows; returns the token-major (B,S,Hq*D)."""
        from . import kernels as K
        Sk = self._room(k.shape[2])
        K.kv_append(k, v, self.k, self.v, self.length)
        out = K.attention_cache(q, self.k, self.v, Sk, scale, causal)
        self.length = Sk
        return out

    @property
    def empty(self) -> bool:
        """Whether no sequence holds a row (known on the host)."""
        return self.length == 0

    def _room(self, S: int) -> int:
        if self.length + S > self.capacity:
            raise RuntimeError(f"KV cache full: {self.length} + {S} > {self.capacity}")
        return self.length + S

    def save_length(self):
        """The cache's length(s), for ``restore_length``."""
        return self.length

    def restore_length(self, saved) -> None:
        self.length = saved

    def __iter__(self):
        return iter(self.views())

    def __getitem__(self, i):
        return self.views()[i]

    def __len__(self) -> int:
        return 2

    def reset(self) -> None:
        self.length = 0


class Q4LayerKVCache(LayerKVCache):
    """One layer's K/V as 4-bit codes with a (scale, minimum) pair per group of
    ``group_size`` channels (32, 64 or 128; smaller groups are more exact:
    0.31 / 0.28 / 0.27 of the bf16 bytes at head_dim 128).

    A first chunk of two tokens or more attends over its own exact k/v (not when a
    length per sequence was set before it); later calls, and a first chunk of one
    token, attend over the stored rows, their own included.

    ``set_lengths(lengths)`` switches to a length per sequence, held on the
    device in ``lengths``: appends go behind each sequence's own rows and
    attention stops at them.  The usual way is a right-padded prompt batch,
    then ``set_lengths`` with the prompts' true lengths.  Nothing checks the
    capacity on the host then; a step that passes it attends over the rows within
    it and is recorded as a device error (``kernels.device_error_check``), while
    ``lengths`` goes on counting until ``set_lengths`` or ``reset``."""

    def __init__(self, batch: int, num_kv_heads: int, capacity: int, head_dim: int, device,
                 group_size: int = 32):
        if capacity < 1:
            raise ValueError("capacity must be positive")
        if head_dim not in (32, 64, 128):
            raise ValueError(f"head_dim {head_dim} unsupported (32, 64 or 128)")
        if group_size not in (32, 64, 128) or group_size > head_dim:
            raise ValueError(f"group_size {group_size} unsupported (32, 64 or 128, at most head_dim)")
        self._capacity = capacity
        self.head_dim, self.group_size = head_dim, group_size
        rows = -(-capacity // 16) * 16  # the kernels' row granularity
        self.k_codes = torch.zeros(batch, num_kv_heads, rows, head_dim // 2, device=device,
                                   dtype=torch.uint8)
        self.k_scales = torch.zeros(batch, num_kv_heads, rows, head_dim // group_size, 2,
                                    device=device, dtype=torch.bfloat16)
        self.v_codes = torch.zeros_like(self.k_codes)
        self.v_scales = torch.zeros_like(self.k_scales)
        self._length = 0
        self._lengths: torch.Tensor | None = None
        self._empty = True  # of the sequences behind _lengths

    @property
    def capacity(self) -> int:
        return self._capacity

    @property
    def length(self) -> int:
        """Valid rows; with per-sequence lengths the longest (synchronises)."""
        return self._length if self.lengths is None else int(self.lengths.max())

    @length.setter
    def length(self, n: int) -> None:
        if self.lengths is not None:
            raise RuntimeError("this cache keeps a length per sequence: use set_lengths")
        self._length = n

    @property
    def empty(self) -> bool:
        return self._length == 0 if self.lengths is None else self._empty

    @property
    def buffers(self) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
        """(k_codes, k_scales, v_codes, v_scales), as the *_q4 kernels take them."""
        return self.k_codes, self.k_scales, self.v_codes, self.v_scales

    def set_lengths(self, lengths: torch.Tensor) -> None:
        """Keeps a length per sequence from here on (copied to an int32 device tensor)."""
        B = self.k_codes.shape[0]
        if lengths.shape != (B,) or lengths.is_floating_point():
            raise ValueError(f"expected {B} integer lengths, got {tuple(lengths.shape)} {lengths.dtype}")
        lo, hi = (int(lengths.min()), int(lengths.max())) if B else (0, 0)
        if lo < 0 or hi > self.capacity:
            raise ValueError(f"lengths {lo}..{hi} outside the capacity {self.capacity}")
        if self._lengths is None:
            self._lengths = torch.empty(B, device=self.k_codes.device, dtype=torch.int32)
        # always the same tensor: captured graphs read and advance it
        self._lengths.copy_(lengths)
        self._empty = hi == 0
        self.lengths = self._lengths

    def read(self, start: int, length: int) -> tuple[torch.Tensor, torch.Tensor]:
        """Rows [start, start+length) of every sequence as bf16 k, v."""
        from . import kernels as K
        return K.kv_read_q4(*self.buffers, start, length)

    def views(self) -> tuple[torch.Tensor, torch.Tensor]:
        """The valid rows as bf16 copies."""
        if self.lengths is not None:
            raise RuntimeError("this cache keeps a length per sequence: use read()")
        return self.read(0, self._length)

    def append_attend(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float,
                      causal: bool) -> torch.Tensor:
        from . import kernels as K
        S = k.shape[2]
        if self.lengths is not None:
            K.kv_append_q4(k, v, *self.buffers, self.lengths)
            self.lengths.add_(S)
            self._empty = self._empty and S == 0
            return K.attention_cache_q4(q, *self.buffers, self.lengths, scale, causal,
                                        max_kv_len=self.capacity)
        past, Sk = self._length, self._room(S)
        K.kv_append_q4(k, v, *self.buffers, past)
        if past == 0 and S > 1:
            out = K.attention_tokens(q, k, v, scale, causal)
        else:
            out = K.attention_cache_q4(q, *self.buffers, Sk, scale, causal)
        self._length = Sk
        return out

    def save_length(self):
        return self._length if self.lengths is None else (self.lengths.clone(), self._empty)

    def restore_length(self, saved) -> None:
        if self.lengths is None:
            self._length = saved
        else:
            self.lengths.copy_(saved[0])
            self._empty = saved[1]

    def reset(self) -> None:
        self.lengths = None
        self._length = 0


class KVCache:
    """One ``LayerKVCache`` per attention layer; pass as ``past_key_values``."""

    def __init__(self, num_layers: int, batch: int, num_kv_heads: int, capacity: int,
                 head_dim: int, device, dtype: torch.dtype = torch.bfloat16):
        self.layers = [LayerKVCache(batch, num_kv_heads, capacity, head_dim, device, dtype)
                       for _ in range(num_layers)]

    def __getitem__(self, i) -> LayerKVCache:
        return self.layers[i]

    def __len__(self) -> int:
        return len(self.layers)

    def __iter__(self):
        return iter(self.layers)

    @property
    def length(self) -> int:
        return self.layers[0].length if self.layers else 0

    def reset(self) -> None:
        for layer in self.layers:
            layer.reset()


class Q4KVCache(KVCache):
    """One ``Q4LayerKVCache`` per attention layer; pass as ``past_key_values``."""

    def __init__(self, num_layers: int, batch: int, num_kv_heads: int, capacity: int,
                 head_dim: int, device, group_size: int = 32):
        self.layers = [Q4LayerKVCache(batch, num_kv_heads, capacity, head_dim, device, group_size)
                       for _ in range(num_layers)]

    def set_lengths(self, lengths: torch.Tensor) -> None:
        """A length per sequence in every layer (``Q4LayerKVCache.set_lengths``)."""
        for layer in self.layers:
            layer.set_lengths(lengths)
