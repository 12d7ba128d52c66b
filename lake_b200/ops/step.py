"""Tables of an engine step, built on the device from request lengths.

For a caller that keeps one row of page ids per request in a device table, and appends to it when a
request takes a page: a step then needs only which rows it runs and how many tokens each has
and gets, not every sequence's whole block table again. (The engine's runner packs its tables on
the host.)
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from ..oracle import ops_ref as ref
from . import core
from ._ext import native


class StepTables(NamedTuple):
    block_tables: torch.Tensor  # int32 [S, max_blocks]: each sequence's pages, 0 past them
    seq_lens: torch.Tensor      # int32 [S]: tokens after the step
    query_start: torch.Tensor   # int32 [S + 1]
    positions: torch.Tensor     # int32 [max_tokens], 0 for rows past the step's tokens
    slots: torch.Tensor         # int64 [max_tokens] KV slot, -1 for rows past the step's tokens
    tiles: torch.Tensor         # int32 [max_tiles, 4] (seq, first row, rows, first position), 0 past the step's
    counts: torch.Tensor        # int32 [2]: tokens, tiles


def build_step_tables(pages: torch.Tensor, rows: torch.Tensor, context_lens: torch.Tensor, new_lens: torch.Tensor,
                      max_tokens: int, max_tiles: int, n_decode: int = 0, block_size: int = ref.PAGE,
                      tile: int = core.PREFILL_TILE) -> StepTables:
    """The tables of a step over the sequences `rows` (int32 [S], rows of `pages` int32
    [requests, max_blocks]), which have `context_lens` tokens in the cache and get `new_lens` more.

    The first `n_decode` sequences are decode rows and get no query tiles; the others' tokens are
    cut into tiles of up to `tile` rows. Every output has its full size whatever the lengths are
    (nothing waits for the device), so a call can be captured into a graph and replayed with other
    lengths. More tokens or tiles than max_tokens / max_tiles, a negative length, a request row
    outside `pages`, or a token whose page is missing (negative, or past the row's end) is reported
    (the status word on the GPU, ValueError on the CPU); on the GPU such a token gets slot -1.

    On the GPU the seven tables are views of one allocation: keeping one keeps all of them."""
    if pages.is_cuda:
        core.LAUNCHES[0] += 1
        return StepTables._make(native().step_tables(pages, rows, context_lens, new_lens, max_tokens, max_tiles, n_decode,
                                                block_size, tile, core.status_word(pages.device)))
    if max_tokens < 0 or max_tiles < 0:
        raise ValueError(f"max_tokens and max_tiles must not be negative, got {max_tokens} and {max_tiles}")
    return StepTables(*ref.step_tables(pages, rows, context_lens, new_lens, max_tokens, max_tiles, n_decode,
                                       block_size, tile))
