"""8-bit KV arena: e4m3 codes with one power-of-two scale byte per token and head.

``kv8_arena(num_blocks, n_layers, n_kv_heads)`` allocates a page-first arena
uint8 [blocks, layers, kv_heads, 2 (K, V), 16 * head_dim + 16]: for every page, layer,
head and side the 16 tokens' codes, then the page's scale line of 16 bytes b;
``value = code * 2^(b - 127)``. A token's b is the smallest that keeps its largest
element within e4m3's 448 (at least 1), b = 255 marks a row that held an infinity or a
NaN: it reads back as NaN. A page takes 1032 bytes per token of 4 KV heads where the bf16
arena takes 2048, so a pool holds nearly twice the tokens and attention reads half the bytes.

The scale belongs to the token, not to the page, so that a row's bytes depend on that row
alone: pages are shared by the hash of their tokens, and a page must not differ by how its
prompt was chunked or by a draft that was rejected.

The bf16 arena's entry points take this arena too, told apart by its dtype: ``linear_qkv``
(its epilogue quantises K and V from the fp32 accumulators), ``paged_decode_attention`` and
``paged_prefill_attention``; so do ``page_copy`` and the pool agents, which move whole pages.
``kv8_write`` and ``kv8_read`` move dense rows in and out. An engine takes it with
``LLMEngine(..., kv_dtype="fp8")``.
"""
from __future__ import annotations

import torch

from ..oracle import ops_ref as ref
from . import core
from ._ext import native

is_kv8 = ref.is_kv8


def kv8_arena(num_blocks: int, n_layers: int, n_kv_heads: int, head_dim: int = ref.HEAD_DIM,
              device: torch.device | str = "cuda") -> torch.Tensor:
    """Zero-filled 8-bit KV arena (pages of 16 tokens). The kernels take head_dim 128; the CPU
    oracle any multiple of 16."""
    if head_dim % 16 or head_dim <= 0:
        raise ValueError(f"head_dim must be a multiple of 16, got {head_dim}")
    return torch.zeros(num_blocks, n_layers, n_kv_heads, 2, ref.PAGE * head_dim + ref.PAGE, dtype=torch.uint8,
                       device=device)


def kv8_write(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, arena: torch.Tensor, layer: int) -> None:
    """Quantise rows of K and V [T, kv_heads * head_dim] (bf16 on the GPU; rows may be strided views
    of a packed projection) into the arena at `slots` (int64 [T], page * 16 + offset; < 0: skipped).

    Slots of one call are distinct; a slot past the arena is reported in the status word and
    skipped."""
    if arena.is_cuda:
        native().kv8_write(k, v, slots, arena, layer, core.status_word(arena.device))
        core.LAUNCHES[0] += slots.numel() > 0
        return
    d = ref.arena_head_dim(arena)
    h = arena.shape[2]
    ref.write_kv(arena, layer, slots, k.reshape(-1, h, d), v.reshape(-1, h, d))


def kv8_read(arena: torch.Tensor, layer: int, slots: torch.Tensor, k_out: torch.Tensor | None = None,
             v_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The cached K and V of `slots` (int64 [T]) as dense bf16 rows [T, kv_heads * head_dim]; a
    negative slot gives a row of zeros (so does one past the arena, which is reported). On the GPU
    outputs that are not given are views of one allocation."""
    if arena.is_cuda:
        got = native().kv8_read(arena, layer, slots, k_out, v_out, core.status_word(arena.device))
        core.LAUNCHES[0] += slots.numel() > 0
        return got
    shape = (slots.shape[0], arena.shape[2] * ref.arena_head_dim(arena))
    if k_out is None:
        k_out = torch.empty(shape, dtype=torch.bfloat16)
    if v_out is None:
        v_out = torch.empty(shape, dtype=torch.bfloat16)
    x = ref.kv8_rows(arena, layer, slots)
    k_out.copy_(x[:, :, 0].reshape(shape).to(k_out.dtype))
    v_out.copy_(x[:, :, 1].reshape(shape).to(v_out.dtype))
    return k_out, v_out
