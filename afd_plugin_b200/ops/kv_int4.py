"""The paged 4-bit KV cache of grouped-query attention.

Per block, KV head and position the cache holds ``d / 2`` bytes of codes (dim ``2 i`` in the low
nibble of byte ``i``) and, per 64 dims, a bf16 ``(step, zero)``; a code ``c`` stands for
``zero + c * step``: 4.5 bits per value.  Tensors are head-major inside a block, so the rows that
one (sequence, KV head) reads are contiguous.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from afd_plugin_b200.ops.reference import INT4_GROUP

INT4_HEAD_DIMS = (64, 128, 256)


class Int4KV(NamedTuple):
    """One layer's cache: codes ``[blocks, kv_heads, block_size, d / 2]`` uint8 and ``(step, zero)``
    ``[blocks, kv_heads, block_size, d / 64, 2]`` bf16 for K and for V."""

    k: torch.Tensor
    k_scale: torch.Tensor
    v: torch.Tensor
    v_scale: torch.Tensor

    @property
    def num_blocks(self) -> int:
        return self.k.shape[0]

    @property
    def block_size(self) -> int:
        return self.k.shape[2]


def int4_kv_cache(num_blocks: int, block_size: int, kv_heads: int, head_dim: int,
                  device: torch.device | str = "cuda") -> Int4KV:
    """A zeroed cache (every stored value is 0)."""
    if head_dim not in INT4_HEAD_DIMS:
        raise ValueError(f"the 4-bit KV cache takes head dims {INT4_HEAD_DIMS}, got {head_dim}")
    if block_size % 16 or block_size <= 0:
        raise ValueError(f"the 4-bit KV cache needs a block size that is a multiple of 16, got {block_size}")

    def one():
        return (torch.zeros(num_blocks, kv_heads, block_size, head_dim // 2, dtype=torch.uint8, device=device),
                torch.zeros(num_blocks, kv_heads, block_size, head_dim // INT4_GROUP, 2, dtype=torch.bfloat16,
                            device=device))

    return Int4KV(*one(), *one())


def check_cache(op: str, kv: Int4KV, scores: torch.Tensor | None = None) -> None:
    """The shape and type rules of the CUDA entry points, for tensors of any device."""
    d = kv.k.shape[-1] * 2
    if kv.k.dim() != 4 or d not in INT4_HEAD_DIMS or kv.block_size % 16 or not kv.block_size:
        raise ValueError(f"{op}: codes [blocks, kv_heads, block_size (a multiple of 16), dim / 2] for dims "
                         f"{INT4_HEAD_DIMS}, got {tuple(kv.k.shape)}")
    pairs = (*kv.k.shape[:3], d // INT4_GROUP, 2)
    for codes, scale in ((kv.k, kv.k_scale), (kv.v, kv.v_scale)):
        if codes.dtype != torch.uint8 or codes.shape != kv.k.shape:
            raise ValueError(f"{op}: uint8 codes of one shape")
        if scale.dtype != torch.bfloat16 or tuple(scale.shape) != pairs:
            raise ValueError(f"{op}: bf16 (step, zero) pairs {pairs}, got {tuple(scale.shape)} {scale.dtype}")
        if not (codes.is_contiguous() and scale.is_contiguous()):
            raise ValueError(f"{op}: contiguous cache tensors")
    if scores is not None and (scores.dtype != torch.float32 or scores.shape != kv.k.shape[:3]
                               or not scores.is_contiguous()):
        raise ValueError(f"{op}: fp32 contiguous scores {tuple(kv.k.shape[:3])}")


def check_rows(op: str, kv: Int4KV, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    want = (slots.shape[0], kv.k.shape[1], kv.k.shape[3] * 2)
    if tuple(k.shape) != want or tuple(v.shape) != want or k.dtype != v.dtype:
        raise ValueError(f"{op}: k / v {want} of one type, got {tuple(k.shape)} and {tuple(v.shape)}")
    if k.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise ValueError(f"{op}: bf16, fp16 or fp32 rows, got {k.dtype}")
    check_slots(op, slots)


def check_slots(op: str, slots: torch.Tensor) -> None:
    if slots.dtype != torch.int64 or slots.dim() != 1:
        raise ValueError(f"{op}: int64 slots [tokens]")


def check_batch(op: str, block_table: torch.Tensor, seq_lens: torch.Tensor, batch: int) -> None:
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.shape[0] != batch:
        raise ValueError(f"{op}: int32 block_table [batch, blocks]")
    if seq_lens.dtype != torch.int32 or tuple(seq_lens.shape) != (batch,):
        raise ValueError(f"{op}: int32 seq_lens [batch]")


def check_query(op: str, kv: Int4KV, q: torch.Tensor) -> None:
    if q.dim() != 3 or q.shape[2] != kv.k.shape[3] * 2 or q.shape[1] % kv.k.shape[1] or not q.shape[1]:
        raise ValueError(f"{op}: q [batch, heads (a multiple of {kv.k.shape[1]}), {kv.k.shape[3] * 2}], "
                         f"got {tuple(q.shape)}")


__all__ = ["INT4_HEAD_DIMS", "Int4KV", "int4_kv_cache"]
