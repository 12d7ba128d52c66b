"""Cases of the 8-bit KV cache operators: writing rows into the paged cache, reading them back,
decode and prefill attention over it, and the step tables (slots, positions, block tables, query
tiles) built from request lengths.

The cache is a uint8 tensor [blocks, layers, kv_heads, 2 (K, V), 16 * 128 + 16]: the 16 tokens'
e4m3 codes of one page, layer, head and side, then one power-of-two scale byte b per token
(value = code * 2^(b - 127); b = 255: the row is NaN). Token t's 16-byte chunk c is stored at
chunk c ^ (t & 7).
"""
import math

import torch

own = False

D = 128
PAGE = 16
TILE = 128
SIDE = PAGE * D + PAGE
BF = torch.bfloat16
DEV = "cuda"


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step of 256 running sequences (the engine's default batch), 32q/8kv heads
        dict(name="write_decode_256", op="write", seqs=256, lo=1, hi=1, hq=32, hkv=8, layers=2),
        # a full prefill step of prompts and chunks: 8192 tokens, the engine's step budget
        dict(name="write_prompts_8192", op="write", seqs=7, lo=248, hi=2916, hq=32, hkv=8, layers=2),
        # one cached prefix handed to a bf16 instance
        dict(name="read_prefix_2000", op="read", seqs=1, lo=2000, hi=2000, hkv=8, layers=2),
        # the prefixes of a batch, odd lengths
        dict(name="read_batch_ragged", op="read", seqs=24, lo=33, hi=4097, hkv=8, layers=2),
        # a few short chats: latency counts
        dict(name="decode_4_short", op="decode", seqs=4, pad=0, lo=1, hi=200, hq=16, hkv=8, layers=2),
        # the steady state of the serving benchmark: 256 sequences of 2048 + 256 tokens
        dict(name="decode_256x2304", op="decode", seqs=256, pad=0, lo=2304, hi=2304, hq=32, hkv=8, layers=2),
        # few sequences of very different length in a padded graph bucket, 64q/8kv heads
        dict(name="decode_ragged_long", op="decode", seqs=13, pad=3, lo=100, hi=40960, hq=64, hkv=8, layers=2),
        # verification of drafts: five query rows behind each context
        dict(name="prefill_verify_16x5", op="prefill", seqs=16, new_lo=5, new_hi=5, pre_lo=300, pre_hi=2000, hq=32,
             hkv=8, layers=2),
        # chunks of prompts behind cached prefixes, odd sizes
        dict(name="prefill_chunks_ragged", op="prefill", seqs=6, new_lo=17, new_hi=1500, pre_lo=1, pre_hi=6001, hq=64,
             hkv=8, layers=2),
        # one fresh prompt of the model's whole window
        dict(name="prefill_8192", op="prefill", seqs=1, new_lo=8192, new_hi=8192, pre_lo=0, pre_hi=0, hq=32, hkv=8,
             layers=2),
        # the tables of a pure decode step
        dict(name="tables_decode_256", op="tables", seqs=256, decode=256, lo=1, hi=1, ctx_hi=2304, maxb=512, tokens=256),
        # the tables of a mixed step: decode rows and prompt chunks in a step of 8448 rows
        dict(name="tables_mixed_8448", op="tables", seqs=264, decode=250, lo=130, hi=1400, ctx_hi=8000, maxb=2560,
             tokens=8448),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["write", "read", "decode", "prefill", "tables"])
    hq, hkv = rng.choice([(32, 8), (64, 8), (16, 8), (8, 1), (4, 2), (4, 4), (16, 2)])
    layers = rng.choice([1, 2, 3])
    if op == "write":
        hi = _log(rng, 1, 4000)
        seqs = _log(rng, 1, max(1, min(256, 8000 // hi)))
        return dict(op=op, seqs=seqs, lo=rng.randint(1, hi), hi=hi, hq=hq, hkv=hkv, layers=layers)
    if op == "read":
        hi = _log(rng, 1, 8000)
        seqs = _log(rng, 1, max(1, min(256, 16000 // hi)))
        return dict(op=op, seqs=seqs, lo=rng.randint(1, hi), hi=hi, hkv=hkv, layers=layers)
    if op == "decode":
        hi = _log(rng, 1, 40960)
        seqs = _log(rng, 1, max(1, min(256, 256 * 2304 // hi)))
        return dict(op=op, seqs=seqs, pad=rng.choice([0, 0, 1, 5]), lo=rng.randint(1, hi), hi=hi, hq=hq, hkv=hkv,
                    layers=layers)
    if op == "prefill":
        new_hi, pre_hi = _log(rng, 1, 2048), rng.choice([0, _log(rng, 1, 6000)])
        pairs = new_hi * (new_hi + pre_hi) * hq
        seqs = _log(rng, 1, max(1, min(32, 4096 // new_hi, 16 * 4096 * 8192 // pairs)))
        return dict(op=op, seqs=seqs, new_lo=rng.randint(1, new_hi), new_hi=new_hi, pre_lo=rng.randint(0, pre_hi),
                    pre_hi=pre_hi, hq=hq, hkv=hkv, layers=layers)
    decode = _log(rng, 1, 256)
    more = rng.choice([0, 0, _log(rng, 1, 8)])
    hi = _log(rng, 2, 1000)
    tokens = decode + more * hi + rng.choice([0, 1, 77])
    return dict(op=op, seqs=decode + more, decode=decode, lo=rng.randint(1, hi), hi=hi, ctx_hi=_log(rng, 16, 8000),
                maxb=(8000 + 1000 + 15) // PAGE + rng.randint(0, 900), tokens=tokens)


def _spread(n, lo, hi):
    """n lengths from lo to hi, evenly spread over their logarithm, odd ones among them."""
    if n <= 1 or lo == hi:
        return [hi] * n
    a, b = math.log(max(lo, 1)), math.log(hi)
    got = [int(round(math.exp(a + (b - a) * i / (n - 1)))) for i in range(n)]
    got[0], got[-1] = lo, hi
    return got


def _lens(c):
    """(new tokens, cached tokens before them) of each sequence, by the case alone."""
    if c["op"] == "write":
        new = _spread(c["seqs"], c["lo"], c["hi"])
        return new, [(37 * i + 5) % 200 for i in range(len(new))]
    if c["op"] == "read":
        return _spread(c["seqs"], c["lo"], c["hi"]), [0] * c["seqs"]
    if c["op"] == "decode":
        lens = _spread(c["seqs"], c["lo"], c["hi"])
        return [1] * len(lens) + [0] * c["pad"], [x - 1 for x in lens] + [0] * c["pad"]
    if c["op"] == "prefill":
        return _spread(c["seqs"], c["new_lo"], c["new_hi"]), _spread(c["seqs"], c["pre_lo"], c["pre_hi"])[::-1]
    more = c["seqs"] - c["decode"]
    return [1] * c["decode"] + _spread(more, c["lo"], c["hi"]), _spread(c["seqs"], 1, c["ctx_hi"])


# ------------------------------------------------------------------ plain form of the format
def _swizzle(device):
    t = torch.arange(PAGE, device=device)
    return t[:, None], torch.arange(D // 16, device=device)[None, :] ^ (t[:, None] & 7)


def _codes(x):
    """fp32 rows [..., 128] -> (e4m3 codes uint8 [..., 128], scale bytes uint8 [...])."""
    fine = torch.isfinite(x).all(-1)
    amax = x.abs().amax(-1)
    amax = torch.where(fine, amax, torch.zeros_like(amax))
    m, e = torch.frexp(amax)
    e = torch.where(amax > 0, (e - 9 + (m > 0.875).to(e.dtype)).clamp_min(-126), torch.full_like(e, -126))
    q = torch.ldexp(torch.where(fine[..., None], x, torch.zeros_like(x)), -e[..., None])
    q = q.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)
    return q, torch.where(fine, e + 127, torch.full_like(e, 255)).to(torch.uint8)


def _scales(b):
    """Scale bytes -> fp32 powers of two (255: NaN)."""
    return torch.where(b == 255, torch.full(b.shape, float("nan"), device=b.device),
                       (b.to(torch.int32) << 23).view(torch.float32))


def _pages_of_rows(x):
    """fp32 [blocks, 16, heads, 2, 128] -> the cache bytes [blocks, heads, 2, SIDE] of one layer."""
    q, b = _codes(x)
    n, _, h = x.shape[:3]
    t, c = _swizzle(x.device)
    q = q.permute(0, 2, 3, 1, 4).reshape(n, h, 2, PAGE, D // 16, 16)
    out = torch.empty(n, h, 2, SIDE, dtype=torch.uint8, device=x.device)
    out[..., : PAGE * D] = q[..., t, c, :].reshape(n, h, 2, PAGE * D)
    out[..., PAGE * D:] = b.permute(0, 2, 3, 1)
    return out


def _rows(arena, layer, slots):
    """fp32 values [N, heads, 2, 128] of the cached tokens at `slots` (all >= 0)."""
    blk, tok = slots // PAGE, slots % PAGE
    c = torch.arange(D // 16, device=slots.device)
    at = ((tok[:, None] * D + (c[None, :] ^ (tok[:, None] & 7)) * 16)[:, :, None]
          + torch.arange(16, device=slots.device)).reshape(-1, D)
    side = arena[:, layer]
    h = torch.arange(side.shape[1], device=slots.device)
    kv = torch.arange(2, device=slots.device)
    q = side[blk[:, None, None, None], h[:, None, None], kv[:, None], at[:, None, None, :]]
    b = side[blk[:, None, None], h[:, None], kv, (PAGE * D + tok)[:, None, None]]
    return q.view(torch.float8_e4m3fn).float() * _scales(b)[..., None]


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _kv_rows(n, heads, g, side):
    """K or V rows as a model makes them: K with a few strong channels per head, tokens of varied norm."""
    x = torch.randn(n, heads, D, device=DEV, generator=g)
    ch = torch.randn(heads, D, device=DEV, generator=g).mul_(0.6 if side == 0 else 0.2).exp_()
    tok = torch.randn(n, heads, 1, device=DEV, generator=g).mul_(0.3).exp_()
    return x.mul_(ch).mul_(tok).mul_(1.0 if side == 0 else 0.4)


def _cache(blocks, layers, layer, heads, g):
    arena = torch.zeros(blocks, layers, heads, 2, SIDE, dtype=torch.uint8, device=DEV)
    step = max(1, (1 << 28) // (PAGE * heads * 2 * D))
    for a in range(0, blocks, step):
        n = min(step, blocks - a)
        rows = [_kv_rows(n * PAGE, heads, g, s).view(n, PAGE, heads, D) for s in (0, 1)]
        arena[a:a + n, layer] = _pages_of_rows(torch.stack(rows, 3).to(BF).float())
    return arena


def _tables(lens, g, extra=2):
    """Block tables [S, widest] over a shuffled pool of pages, and the pool's size."""
    nb = [-(-x // PAGE) for x in lens]
    total = sum(nb)
    ids = torch.randperm(total + extra, device=DEV, generator=g)[:total].to(torch.int32)
    bt = torch.zeros(len(lens), max(max(nb), 1), dtype=torch.int32, device=DEV)
    used = torch.arange(bt.shape[1], device=DEV)[None, :] < torch.tensor(nb, device=DEV)[:, None]
    bt[used] = ids
    return bt, total + extra


def prepare(case, seed):
    g = _gen(seed)
    new, pre = _lens(case)
    lens = [a + b for a, b in zip(new, pre)]
    dev = dict(device=DEV)
    if case["op"] == "tables":
        r = case["seqs"] + 9
        pages = torch.randint(0, 1 << 20, (r, case["maxb"]), dtype=torch.int32, generator=g, **dev)
        rows = torch.randperm(r, generator=g, **dev)[: case["seqs"]].to(torch.int32)
        order = torch.randperm(case["decode"], generator=g, **dev)
        ctx = torch.tensor(pre, dtype=torch.int32, **dev)
        ctx[: case["decode"]] = ctx[: case["decode"]][order]
        tiles = sum(-(-x // TILE) for x in new[case["decode"]:]) + 3
        return dict(op="tables", pages=pages, rows=rows, ctx=ctx, new=torch.tensor(new, dtype=torch.int32, **dev),
                    n_decode=case["decode"], tokens=case["tokens"], tiles=tiles)
    h, layers = case["hkv"], case["layers"]
    layer = layers - 1
    bt, blocks = _tables(lens, g)
    arena = _cache(blocks, layers, layer, h, g)
    seq_lens = torch.tensor(lens, dtype=torch.int32, **dev)
    st = dict(op=case["op"], arena=arena, layer=layer, hkv=h)
    if case["op"] in ("write", "read"):
        slots = torch.cat([bt[s].long().repeat_interleave(PAGE)[a:a + n] * PAGE
                           + torch.arange(a, a + n, **dev) % PAGE for s, (n, a) in enumerate(zip(new, pre))])
        if case["op"] == "read":
            return dict(st, slots=slots)
        # rows of a packed QKV projection; the first row of a step of several rows is a padding row
        qkv = torch.randn(slots.numel(), (case["hq"] + 2 * h) * D, generator=g, **dev).to(BF)
        k, v = qkv[:, case["hq"] * D:(case["hq"] + h) * D], qkv[:, (case["hq"] + h) * D:]
        k.copy_(_kv_rows(slots.numel(), h, g, 0).view(-1, h * D))
        v.copy_(_kv_rows(slots.numel(), h, g, 1).view(-1, h * D))
        touched = torch.unique(slots // PAGE)
        back = (touched[:, None] * PAGE + torch.arange(PAGE, **dev)).reshape(-1)
        if slots.numel() > 4:
            slots[0] = -1
        return dict(st, k=k, v=v, slots=slots, back=back)
    scale = 1.0 / math.sqrt(D)
    hq = case["hq"]
    q = torch.randn(sum(new) if case["op"] == "prefill" else len(lens), hq * D, generator=g, **dev).mul_(1.5).to(BF)
    st.update(q=q, bt=bt, seq_lens=seq_lens, hq=hq, scale=scale)
    if case["op"] == "decode":
        return st
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    tiles = [(s, starts[s] + t, min(TILE, n - t), pre[s] + t) for s, n in enumerate(new) for t in range(0, n, TILE)]
    pos = torch.cat([torch.arange(a, a + n, dtype=torch.int32, **dev) for n, a in zip(new, pre)])
    return dict(st, tiles=torch.tensor(tiles, dtype=torch.int32, **dev), positions=pos, most_new=max(new),
                query_start=torch.tensor(starts, dtype=torch.int32, **dev))


# ------------------------------------------------------------------ plain operators
def _plain_write(s):
    slots, arena, layer = s["slots"], s["arena"], s["layer"]
    keep = slots >= 0
    sl = slots[keep]
    x = torch.stack([s["k"].float().view(-1, s["hkv"], D), s["v"].float().view(-1, s["hkv"], D)], 2)[keep]
    q, b = _codes(x)
    blk, tok = sl // PAGE, sl % PAGE
    dev = sl.device
    at = ((tok[:, None] * D + (torch.arange(D // 16, device=dev)[None, :] ^ (tok[:, None] & 7)) * 16)[:, :, None]
          + torch.arange(16, device=dev)).reshape(-1, D)
    h, kv = torch.arange(s["hkv"], device=dev), torch.arange(2, device=dev)
    side = arena[:, layer]
    side[blk[:, None, None, None], h[:, None, None], kv[:, None], at[:, None, None, :]] = q
    side[blk[:, None, None], h[:, None], kv, (PAGE * D + tok)[:, None, None]] = b


def _plain_read(arena, layer, slots):
    x = _rows(arena, layer, slots)
    x = torch.where((slots >= 0)[:, None, None, None], x, torch.zeros_like(x)).to(BF)
    return x[:, :, 0].reshape(slots.numel(), -1), x[:, :, 1].reshape(slots.numel(), -1)


def _padded_kv(s):
    """K, V fp32 [S, heads, keys, 128] of the tables' pages (0 past a sequence's end) and the key mask [S, keys]."""
    n, nb = s["bt"].shape
    raw = s["arena"][s["bt"].long(), s["layer"]]
    t, c = _swizzle(DEV)
    x = raw[..., : PAGE * D].view(n, nb, s["hkv"], 2, PAGE, D // 16, 16)[..., t, c, :].flatten(-2)
    x = x.view(torch.float8_e4m3fn).float() * _scales(raw[..., PAGE * D:])[..., None]
    ok = torch.arange(nb * PAGE, device=DEV)[None, :] < s["seq_lens"][:, None]
    x.masked_fill_(~ok.view(n, nb, 1, 1, PAGE, 1), 0.0)
    x = x.permute(3, 0, 2, 1, 4, 5).reshape(2, n, s["hkv"], nb * PAGE, D)
    return x[0], x[1], ok


def _plain_decode(s):
    n, hq, hkv = s["seq_lens"].shape[0], s["hq"], s["hkv"]
    k, v, ok = _padded_kv(s)
    q = s["q"].float().view(n, hkv, hq // hkv, D) * s["scale"]
    a = torch.matmul(q, k.transpose(2, 3))
    a = a.masked_fill(~ok[:, None, None, :], float("-inf"))
    m = a.amax(-1, keepdim=True)
    p = torch.exp(a - torch.where(torch.isinf(m), torch.zeros_like(m), m))
    o = torch.matmul(p, v)
    z = p.sum(-1, keepdim=True)
    return torch.where(z == 0, torch.zeros_like(o), o / z).reshape(n, hq * D).to(BF)


def _plain_prefill(s):
    n, hq, hkv = s["seq_lens"].shape[0], s["hq"], s["hkv"]
    most = s["most_new"]
    i = torch.arange(most, device=DEV)
    qs = s["query_start"].long()
    real = i[None, :] < (qs[1:] - qs[:-1])[:, None]
    row = torch.where(real, qs[:-1, None] + i[None, :], torch.zeros_like(i))
    q = s["q"].float()[row].view(n, most, hkv, hq // hkv, D).permute(0, 2, 3, 1, 4) * s["scale"]
    k, v, ok = _padded_kv(s)
    a = torch.matmul(q.reshape(n, hkv, -1, D), k.transpose(2, 3)).view(n, hkv, hq // hkv, most, -1)
    pos = s["positions"].long()[row]
    see = ok[:, None, :] & (torch.arange(k.shape[2], device=DEV)[None, None, :] <= pos[:, :, None])
    a.masked_fill_(~see[:, None, None], float("-inf"))
    a.sub_(a.amax(-1, keepdim=True)).exp_()
    z = a.sum(-1, keepdim=True)
    o = torch.matmul(a.view(n, hkv, -1, a.shape[-1]), v).view(n, hkv, hq // hkv, most, D) / z
    out = torch.empty(s["q"].shape[0], hq * D, dtype=BF, device=DEV)
    out[row[real]] = o.permute(0, 3, 1, 2, 4).reshape(n, most, hq * D)[real].to(BF)
    return out


def _plain_tables(s):
    rows, ctx, new, pages = s["rows"].long(), s["ctx"].long(), s["new"].long(), s["pages"]
    lens = ctx + new
    start = torch.cat([torch.zeros(1, dtype=torch.int64, device=DEV), new.cumsum(0)])
    t = torch.arange(s["tokens"], device=DEV)
    seq = torch.searchsorted(start[1:], t, right=True).clamp_max(rows.numel() - 1)
    real = t < start[-1]
    pos = torch.where(real, ctx[seq] + t - start[seq], torch.zeros_like(t))
    slots = torch.where(real, pages[rows[seq], pos // PAGE].long() * PAGE + pos % PAGE, torch.full_like(t, -1))
    used = torch.arange(pages.shape[1], device=DEV)[None, :] < ((lens + PAGE - 1) // PAGE)[:, None]
    bt = torch.where(used, pages[rows], torch.zeros_like(pages[:1, :1]))
    many = torch.where(torch.arange(rows.numel(), device=DEV) < s["n_decode"], torch.zeros_like(new),
                       (new + TILE - 1) // TILE)
    first = torch.cat([torch.zeros(1, dtype=torch.int64, device=DEV), many.cumsum(0)])
    j = torch.arange(s["tiles"], device=DEV)
    q = torch.searchsorted(first[1:], j, right=True).clamp_max(rows.numel() - 1)
    at = (j - first[q]) * TILE
    tiles = torch.stack([q, start[q] + at, (new[q] - at).clamp_max(TILE), ctx[q] + at], 1)
    tiles = torch.where((j < first[-1])[:, None], tiles, torch.zeros_like(tiles))
    i32 = torch.int32
    return (bt, lens.to(i32), start.to(i32), pos.to(i32), slots, tiles.to(i32),
            torch.stack([start[-1], first[-1]]).to(i32))


def run(state):
    s, op = state, state["op"]
    if own:
        from lake_b200 import ops

        if op == "write":
            ops.kv8_write(s["k"], s["v"], s["slots"], s["arena"], s["layer"])
            return ops.kv8_read(s["arena"], s["layer"], s["back"])
        if op == "read":
            return ops.kv8_read(s["arena"], s["layer"], s["slots"])
        if op == "decode":
            return ops.paged_decode_attention(s["q"], s["arena"], s["layer"], s["bt"], s["seq_lens"], s["hq"],
                                              s["hkv"], s["scale"])
        if op == "prefill":
            return ops.paged_prefill_attention(s["q"], s["arena"], s["layer"], s["bt"], s["seq_lens"], s["tiles"],
                                               s["query_start"], s["positions"], s["hq"], s["hkv"], s["scale"])
        return tuple(ops.build_step_tables(s["pages"], s["rows"], s["ctx"], s["new"], s["tokens"], s["tiles"],
                                           n_decode=s["n_decode"]))
    if op == "write":
        _plain_write(s)
        return _plain_read(s["arena"], s["layer"], s["back"])
    if op == "read":
        return _plain_read(s["arena"], s["layer"], s["slots"])
    return {"decode": _plain_decode, "prefill": _plain_prefill, "tables": _plain_tables}[op](s)


# ------------------------------------------------------------------ work
def work(case):
    new, pre = _lens(case)
    lens = [a + b for a, b in zip(new, pre)]
    if case["op"] == "tables":
        nb = sum(-(-x // PAGE) for x in lens)
        tiles = sum(-(-x // TILE) for x in new[case["decode"]:]) + 3
        return {"bytes": 4 * nb + 4 * case["seqs"] * case["maxb"] + 12 * case["tokens"] + 16 * tiles
                + 20 * case["seqs"], "flops": 0}
    h = case["hkv"]
    cached = 2 * h * (D + 1)  # codes and scale byte of one token, K and V
    dense = 2 * h * D * 2
    if case["op"] == "write":
        t = sum(new) - (1 if sum(new) > 4 else 0)
        back = sum((-(-(a + n) // PAGE) - a // PAGE) * PAGE for n, a in zip(new, pre))
        return {"bytes": (t + back) * (cached + dense) + 8 * (sum(new) + back), "flops": 0}
    if case["op"] == "read":
        return {"bytes": sum(new) * (cached + dense + 8), "flops": 0}
    hq = case["hq"]
    rows = sum(new) if case["op"] == "prefill" else len(lens)
    pairs = sum(n * a + n * (n + 1) // 2 for n, a in zip(new, pre))
    return {"bytes": sum(lens) * cached + rows * hq * D * 4 + sum(-(-x // PAGE) for x in lens) * 4,
            "flops": 4 * hq * D * pairs}


# ------------------------------------------------------------------ 64-bit results
def _cached64(arena, layer, bt, length):
    """K, V in 64 bits [heads, length, 128] of one sequence, page by page from the format's definition."""
    nb = -(-length // PAGE)
    raw = arena[bt[:nb].long(), layer]
    codes = raw[..., : PAGE * D].view(torch.float8_e4m3fn).double().view(nb, -1, 2, PAGE, D // 16, 16)
    tok = [codes[:, :, :, t][:, :, :, [c ^ (t & 7) for c in range(D // 16)]].flatten(3) for t in range(PAGE)]
    x = torch.stack(tok, 3) * torch.exp2(raw[..., PAGE * D:].double() - 127.0)[..., None]
    x = x.permute(2, 1, 0, 3, 4).reshape(2, raw.shape[1], nb * PAGE, D)[:, :, :length]
    return x[0], x[1]


def _write64(s):
    """The values that a write leaves at `back`, by the quantisation's definition in 64 bits."""
    arena, layer, h = s["arena"], s["layer"], s["hkv"]
    page = (s["back"][::PAGE] // PAGE).to(torch.int32)
    k, v = _cached64(arena, layer, page, page.numel() * PAGE)
    where = {int(p): i for i, p in enumerate(page.tolist())}
    slots = s["slots"].tolist()
    rows = [i for i, sl in enumerate(slots) if sl >= 0]
    at = torch.tensor([where[slots[i] // PAGE] * PAGE + slots[i] % PAGE for i in rows], device=DEV)
    rows = torch.tensor(rows, device=DEV)
    out = []
    for old, x in ((k, s["k"]), (v, s["v"])):
        x = x[rows].double().view(-1, h, D)
        top = x.abs().amax(-1, keepdim=True)
        e = torch.ceil(torch.log2(top / 448.0)).clamp(-126, 200)
        e = torch.where(top / 448.0 <= torch.exp2(e - 1), e - 1, e)
        e = torch.where(top > 448.0 * torch.exp2(e), e + 1, e)
        y = x / torch.exp2(e)
        ulp = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)  # 3 mantissa bits, 2^-9 at least
        old[:, at] = (torch.round(y / ulp) * ulp * torch.exp2(e)).transpose(0, 1)
        out.append(old.transpose(0, 1).reshape(-1, h * D))
    return tuple(out)


def _attend64(q, k, v, pos, scale):
    """q [n, hq, 128], k and v [heads, length, 128], causal by position: [n, hq * 128] in 64 bits."""
    n, hq = q.shape[:2]
    g = hq // k.shape[0]
    out = torch.empty(n, hq, D, dtype=torch.float64, device=DEV)
    step = max(1, (1 << 27) // max(1, k.shape[1]))
    key = torch.arange(k.shape[1], device=DEV)
    for h in range(hq):
        for a in range(0, n, step):
            z = q[a:a + step, h] @ k[h // g].t() * scale
            z = z.masked_fill(key[None, :] > pos[a:a + step, None], float("-inf"))
            out[a:a + step, h] = torch.softmax(z, -1) @ v[h // g]
    return out.view(n, hq * D)


def exact(case, seed):
    if case["op"] == "tables":
        return None
    s = prepare(case, seed)
    if case["op"] == "write":
        return _write64(s)
    if case["op"] == "read":
        new, _ = _lens(case)
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        k, v = [], []
        for a, b in zip(starts, starts[1:]):
            kk, vv = _cached64(s["arena"], s["layer"], s["slots"][a:b:PAGE] // PAGE, b - a)
            k.append(kk.transpose(0, 1).reshape(b - a, -1))
            v.append(vv.transpose(0, 1).reshape(b - a, -1))
        return torch.cat(k), torch.cat(v)
    new, pre = _lens(case)
    out = []
    at = 0
    for i, (n, a) in enumerate(zip(new, pre)):
        rows = n if case["op"] == "prefill" else 1
        q = s["q"][at:at + rows].double().view(rows, s["hq"], D)
        at += rows
        if n + a == 0:
            out.append(torch.zeros(rows, s["hq"] * D, dtype=torch.float64, device=DEV))
            continue
        k, v = _cached64(s["arena"], s["layer"], s["bt"][i], n + a)
        out.append(_attend64(q, k, v, torch.arange(a, a + rows, device=DEV), s["scale"]))
    return torch.cat(out)
