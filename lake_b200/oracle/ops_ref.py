"""fp32 PyTorch reference implementations of every kernel in ``csrc/kernels``.

These are the correctness oracle for the CUDA kernels (tests compare against
them) and the CPU execution path of :mod:`lake_b200.ops`. Semantics follow the
reference model's intended forward (python/lake/engine/model_executor/models/
qwen/qwen3.py:85-259 describes the module tree; the reference never executes it)
and the pure-Python attention oracle (python/lake/kernels/attn_ref.py:13-56).
"""
from __future__ import annotations

import math

import torch

PAGE = 16
HEAD_DIM = 128


def linear(a: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    return a.float() @ w.float().t()


def swiglu_from_interleaved(acc: torch.Tensor, tile: int = 256) -> torch.Tensor:
    """acc [M, 2I] with rows of each 256-wide tile laid out [gate 128 | up 128]."""
    m, n = acc.shape
    t = acc.view(m, n // tile, 2, tile // 2)
    g, u = t[:, :, 0, :], t[:, :, 1, :]
    return (torch.nn.functional.silu(g) * u).reshape(m, n // 2)


def interleave_gate_up(gate: torch.Tensor, up: torch.Tensor, tile: int = 256) -> torch.Tensor:
    """Stack gate [I, H] and up [I, H] into the tile-interleaved layout the SwiGLU epilogue reads."""
    i, h = gate.shape
    half = tile // 2
    assert i % half == 0
    g = gate.view(i // half, half, h)
    u = up.view(i // half, half, h)
    return torch.stack([g, u], dim=1).reshape(2 * i, h).contiguous()


def rope_cache(max_pos: int, theta: float, head_dim: int = HEAD_DIM, scaling: dict | None = None,
               device=None) -> torch.Tensor:
    """[max_pos, head_dim/2, 2] fp32 (cos, sin) for rotate-half RoPE.

    ``scaling`` supports the "llama3" frequency-band rule (factor, low/high
    frequency factors, original max positions).
    """
    half = head_dim // 2
    inv = 1.0 / (theta ** (torch.arange(0, half, dtype=torch.float64) * 2.0 / head_dim))
    if scaling and scaling.get("rope_type", scaling.get("type")) == "llama3":
        factor = scaling["factor"]
        lo = scaling.get("low_freq_factor", 1.0)
        hi = scaling.get("high_freq_factor", 4.0)
        orig = scaling.get("original_max_position_embeddings", 8192)
        lo_wl, hi_wl = orig / lo, orig / hi
        wl = 2 * math.pi / inv
        smooth = (orig / wl - lo) / (hi - lo)
        scaled = torch.where(wl > lo_wl, inv / factor, inv)
        mid = (wl <= lo_wl) & (wl >= hi_wl)
        scaled = torch.where(mid, (1 - smooth) * inv / factor + smooth * inv, scaled)
        inv = scaled
    pos = torch.arange(max_pos, dtype=torch.float64)
    ang = pos[:, None] * inv[None, :]
    cs = torch.stack([torch.cos(ang), torch.sin(ang)], dim=-1).float()
    return cs.to(device) if device is not None else cs


def apply_rope(x: torch.Tensor, positions: torch.Tensor, cs: torch.Tensor) -> torch.Tensor:
    """x [T, H, D] fp32, rotate-half convention."""
    half = x.shape[-1] // 2
    c = cs[positions.long(), :, 0][:, None, :]
    s = cs[positions.long(), :, 1][:, None, :]
    x1, x2 = x[..., :half], x[..., half:]
    return torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], dim=-1)


def rms_norm(x: torch.Tensor, w: torch.Tensor, eps: float) -> torch.Tensor:
    xf = x.float()
    return xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps) * w.float()


# ------------------------------------------------------------------ 8-bit KV arena
def is_kv8(arena: torch.Tensor) -> bool:
    """Whether `arena` is an 8-bit KV arena (uint8 [blocks, layers, kv_heads, 2, 16 * D + 16])."""
    return arena.dtype == torch.uint8


def arena_head_dim(arena: torch.Tensor) -> int:
    return arena.shape[-1] // PAGE - 1 if is_kv8(arena) else arena.shape[-1]


def kv8_quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows [..., D] -> (e4m3 codes uint8 [..., D], scale bytes uint8 [...]): the scale is 2^(b - 127)
    with the smallest b >= 1 that keeps the row's largest element within 448; b = 255 and codes 0 for a
    row with an infinity or a NaN."""
    x = x.float()
    fine = torch.isfinite(x).all(-1)
    x = torch.where(fine[..., None], x, torch.zeros_like(x))
    amax = x.abs().amax(-1)
    m, e = torch.frexp(amax)  # amax = m * 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(amax > 0, (e - 9 + (m > 0.875).to(e.dtype)).clamp_min(-126), torch.full_like(e, -126))
    q = torch.ldexp(x, -e[..., None]).to(torch.float8_e4m3fn).view(torch.uint8)
    return q, torch.where(fine, e + 127, torch.full_like(e, 255)).to(torch.uint8)


def kv8_scale(b: torch.Tensor) -> torch.Tensor:
    """Scale bytes -> fp32 2^(b - 127); 255 -> NaN, 0 (never written) -> 0."""
    return torch.where(b == 255, torch.full(b.shape, float("nan"), device=b.device),
                       (b.to(torch.int32) << 23).view(torch.float32))


def _kv8_cols(tok: torch.Tensor, d: int) -> torch.Tensor:
    """Byte offsets [N, d] of the codes of tokens `tok` (offsets in the page): 16-byte chunk c of
    token t lies at chunk c ^ (t & (p - 1)), p the power of two in the row's chunks, at most 8."""
    n = d // 16
    c = torch.arange(n, device=tok.device)[None, :] ^ (tok[:, None] & (min(n & -n, 8) - 1))
    return (tok[:, None, None] * d + c[:, :, None] * 16 + torch.arange(16, device=tok.device)).reshape(-1, d)


def kv8_rows(arena: torch.Tensor, layer: int, slots: torch.Tensor) -> torch.Tensor:
    """fp32 values [N, Hkv, 2 (K, V), D] of cached tokens (negative slots: zeros)."""
    d = arena_head_dim(arena)
    sl = slots.long().clamp_min(0)
    blk, tok = sl // PAGE, sl % PAGE
    raw = arena[blk, layer]  # [N, Hkv, 2, 16 * D + 16]
    at = _kv8_cols(tok, d)[:, None, None, :].expand(-1, raw.shape[1], 2, -1)
    q = raw.gather(-1, at).view(torch.float8_e4m3fn).float()
    b = raw.gather(-1, (PAGE * d + tok)[:, None, None, None].expand(-1, raw.shape[1], 2, 1))
    x = q * kv8_scale(b)
    return torch.where((slots >= 0)[:, None, None, None], x, torch.zeros_like(x))


def _kv8_put(arena: torch.Tensor, layer: int, slots: torch.Tensor, x: torch.Tensor) -> None:
    """x [N, Hkv, 2, D] into the arena at slots [N] (all >= 0)."""
    d = arena_head_dim(arena)
    q, b = kv8_quantize(x)
    blk, tok = slots // PAGE, slots % PAGE
    h = torch.arange(arena.shape[2], device=slots.device)[None, :, None]
    kv = torch.arange(2, device=slots.device)[None, None, :]
    arena[blk[:, None, None, None], layer, h[..., None], kv[..., None], _kv8_cols(tok, d)[:, None, None, :]] = q
    arena[blk[:, None, None], layer, h, kv, (PAGE * d + tok)[:, None, None]] = b


def write_kv(arena: torch.Tensor, layer: int, slots: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> None:
    """k, v [T, Hkv, D]; slots [T] (block*16+offset, <0 skipped)."""
    sl = slots.long()
    keep = sl >= 0
    sl = sl[keep]
    if is_kv8(arena):
        _kv8_put(arena, layer, sl, torch.stack([k[keep].float(), v[keep].float()], dim=2))
        return
    page = arena.shape[4]
    blk, off = sl // page, sl % page
    arena[blk, layer, 0, :, off, :] = k[keep].to(arena.dtype)
    arena[blk, layer, 1, :, off, :] = v[keep].to(arena.dtype)


def gather_kv(arena: torch.Tensor, layer: int, block_table: torch.Tensor, length: int):
    """Return K, V [length, Hkv, D] fp32 for one sequence."""
    if is_kv8(arena):
        j = torch.arange(length, device=arena.device)
        x = kv8_rows(arena, layer, block_table.long()[j // PAGE] * PAGE + j % PAGE)
        return x[:, :, 0], x[:, :, 1]
    page = arena.shape[4]
    nb = (length + page - 1) // page
    ids = block_table[:nb].long()
    k = arena[ids, layer, 0].float()  # [nb, Hkv, 16, D]
    v = arena[ids, layer, 1].float()
    k = k.permute(0, 2, 1, 3).reshape(nb * page, -1, k.shape[-1])[:length]
    v = v.permute(0, 2, 1, 3).reshape(nb * page, -1, v.shape[-1])[:length]
    return k, v


def attention_one(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_pos: torch.Tensor, scale: float):
    """q [Tq, Hq, D], k/v [Tk, Hkv, D] (fp32), causal by absolute position: key j visible iff j <= q_pos."""
    hq, hkv = q.shape[1], k.shape[1]
    g = hq // hkv
    k = k.repeat_interleave(g, dim=1)
    v = v.repeat_interleave(g, dim=1)
    s = torch.einsum("qhd,khd->hqk", q.float(), k) * scale
    kp = torch.arange(k.shape[0], device=q.device)
    mask = kp[None, :] > q_pos.long()[:, None]
    s = s.masked_fill(mask[None], float("-inf"))
    p = torch.softmax(s, dim=-1)
    return torch.einsum("hqk,khd->qhd", p, v)


def paged_attention(q: torch.Tensor, arena: torch.Tensor, layer: int, block_tables: torch.Tensor,
                    seq_lens: torch.Tensor, query_start: torch.Tensor, positions: torch.Tensor,
                    n_q_heads: int, n_kv_heads: int, scale: float) -> torch.Tensor:
    """Generic paged attention: rows [query_start[s], query_start[s+1]) belong to sequence s."""
    d = arena_head_dim(arena)
    out = torch.zeros(q.shape[0], n_q_heads * d, dtype=torch.float32, device=q.device)
    qs = query_start.tolist()
    lens = seq_lens.tolist()
    for s in range(len(lens)):
        a, b = qs[s], qs[s + 1]
        if b <= a or lens[s] <= 0:
            continue
        k, v = gather_kv(arena, layer, block_tables[s], lens[s])
        qq = q[a:b].float().view(b - a, n_q_heads, d)
        o = attention_one(qq, k, v, positions[a:b], scale)
        out[a:b] = o.reshape(b - a, -1)
    return out


def step_tables(pages: torch.Tensor, rows: torch.Tensor, context_lens: torch.Tensor, new_lens: torch.Tensor,
                max_tokens: int, max_tiles: int, n_decode: int = 0, block_size: int = PAGE, tile: int = 128):
    """Tables of an engine step by plain loops (see ops.build_step_tables); raises ValueError where
    the kernel reports through the status word."""
    r, ctx, new = rows.tolist(), context_lens.tolist(), new_lens.tolist()
    n, maxb = len(r), pages.shape[1]
    if len(ctx) != n or len(new) != n:
        raise ValueError("one context and one new length per sequence")
    if not 0 <= n_decode <= n:
        raise ValueError(f"n_decode {n_decode} of {n} sequences")
    if any(x < 0 for x in new) or any(x < 0 for x in ctx):
        raise ValueError("negative length")
    if any(not 0 <= x < pages.shape[0] for x in r):
        raise ValueError("request row outside the page table")
    bt = torch.zeros(n, maxb, dtype=torch.int32)
    start, positions, slots, tiles = [0], [], [], []
    for s in range(n):
        nb = (ctx[s] + new[s] + block_size - 1) // block_size
        if nb > maxb:
            raise ValueError(f"sequence {s} needs {nb} pages, its row has {maxb}")
        own = pages[r[s], :nb]
        if bool((own < 0).any()):
            raise ValueError(f"sequence {s} has a token without a page")
        bt[s, :nb] = own
        ids = own.tolist()
        for j in range(new[s]):
            p = ctx[s] + j
            positions.append(p)
            slots.append(ids[p // block_size] * block_size + p % block_size)
        if s >= n_decode:
            for at in range(0, new[s], tile):
                tiles.append((s, start[-1] + at, min(tile, new[s] - at), ctx[s] + at))
        start.append(start[-1] + new[s])
    if start[-1] > max_tokens or len(tiles) > max_tiles:
        raise ValueError(f"{start[-1]} tokens and {len(tiles)} tiles, room for {max_tokens} and {max_tiles}")
    counts = [start[-1], len(tiles)]
    positions += [0] * (max_tokens - len(positions))
    slots += [-1] * (max_tokens - len(slots))
    tiles += [(0, 0, 0, 0)] * (max_tiles - len(tiles))
    i32 = torch.int32
    return (bt, torch.tensor([a + b for a, b in zip(ctx, new)], dtype=i32), torch.tensor(start, dtype=i32),
            torch.tensor(positions, dtype=i32), torch.tensor(slots, dtype=torch.int64),
            torch.tensor(tiles, dtype=i32).reshape(max_tiles, 4), torch.tensor(counts, dtype=i32))


def greedy(logits: torch.Tensor, bitmask: torch.Tensor | None = None) -> torch.Tensor:
    lg = logits.float()
    if bitmask is not None:
        lg = apply_bitmask(lg, bitmask)
    return lg.argmax(dim=-1).to(torch.int32)


def bitmask_to_bool(bitmask: torch.Tensor, vocab: int) -> torch.Tensor:
    words = bitmask.to(torch.int64) & 0xFFFFFFFF
    bits = (words[:, :, None] >> torch.arange(32, device=bitmask.device)[None, None, :]) & 1
    return bits.reshape(bitmask.shape[0], -1)[:, :vocab].bool()


def apply_bitmask(logits: torch.Tensor, bitmask: torch.Tensor) -> torch.Tensor:
    allow = bitmask_to_bool(bitmask, logits.shape[-1])
    return logits.masked_fill(~allow, float("-inf"))


def chain_reject(draft: list[list[int]], target: list[list[int]]) -> list[list[int]]:
    """Greedy chain verification: accept matching drafts, then the target token at the first mismatch,
    or the bonus token after a fully accepted chain (target has len(draft)+1 entries per request)."""
    out = []
    for d, t in zip(draft, target):
        acc = []
        for i, tok in enumerate(d):
            acc.append(t[i])
            if t[i] != tok:
                break
        else:
            acc.append(t[len(d)])
        out.append(acc)
    return out
