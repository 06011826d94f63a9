"""The 8-bit key/value cache of one attention layer.

A row (one token's key or value of one kv head) is held as whole numbers
-127 .. 127 and one fp32 scale, max|x| / 127: 64 + 4 bytes for 128 bytes of
bf16 at head dim 64.  The kernels' layout (csrc/kv_cache.h) is described at
KVCache's fields; read values back with kv_cache_read_hip.
"""
from __future__ import annotations

import operator

import torch

from .kernels import padded_head_dim

BLOCK = 64  # tokens of a block; a capacity is rounded up to a multiple of it


class KVCache:
    """Room for `capacity` tokens (rounded up to a multiple of 64) of `batch`
    sequences, with n_kv_head heads of head_dim values (at most 128).

    Tokens lie where kv_cache_write_hip is told to put them: the cache keeps no
    lengths, so one tensor of positions can serve all layers of a model, on the
    device, inside a captured graph.  Positions never written read as zeros.

      k        uint8 (batch, n_kv_head, capacity / 16, D / 16, 16, 16):
               whole numbers + 128, [token / 16][dim / 16][token % 16][dim % 16]
      v        uint8 (batch, n_kv_head, capacity / 64, D / 16, 4, 16, 16):
               [dim / 16][token / 4 % 4][dim % 16][4 (token / 16 % 4) + token % 4]
      k_scale, v_scale  float32 (batch, n_kv_head, capacity)

    D is 64 or 128: other head dims are held zero-padded to the next of them,
    as attention() runs them.
    """

    def __init__(self, batch: int, capacity: int, n_kv_head: int, head_dim: int, device: torch.device | str = "cuda") -> None:
        batch, capacity, n_kv_head, head_dim = map(operator.index, (batch, capacity, n_kv_head, head_dim))
        for name, n in (("batch", batch), ("capacity", capacity), ("n_kv_head", n_kv_head)):
            if n < 1:
                raise RuntimeError(f"{name} must be at least 1, got {n}")
        self.batch, self.n_kv_head, self.head_dim = batch, n_kv_head, head_dim
        self.kernel_dim = padded_head_dim(head_dim, head_dim)
        self.capacity = -(-capacity // BLOCK) * BLOCK
        if self.capacity > 1 << 24:
            raise RuntimeError(f"capacity {capacity} is beyond {1 << 24} tokens")
        shape = (self.batch, self.n_kv_head, self.capacity)
        pieces = self.kernel_dim // 16
        self.k = torch.empty((*shape[:2], self.capacity // 16, pieces, 16, 16), dtype=torch.uint8, device=device)
        self.v = torch.empty((*shape[:2], self.capacity // BLOCK, pieces, 4, 16, 16), dtype=torch.uint8, device=device)
        self.k_scale = torch.zeros(shape, dtype=torch.float32, device=device)  # a scale of zero is a row of zeros
        self.v_scale = torch.zeros(shape, dtype=torch.float32, device=device)

    @property
    def device(self) -> torch.device:
        return self.k.device

    @property
    def nbytes(self) -> int:
        """Device bytes held."""
        return sum(t.numel() * t.element_size() for t in self.tensors())

    def tensors(self) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
        return self.k, self.v, self.k_scale, self.v_scale
