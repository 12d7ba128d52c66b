"""8-bit KV arena: rows in and out, decode and prefill attention over it, against 64-bit results
computed here from the format's definition."""
import math

import pytest
import torch

from lake_b200 import ops
from lake_b200.oracle import ops_ref as ref

BF = torch.bfloat16
PAGE = 16


# ------------------------------------------------------------------ definitions in 64 bits
def quantize64(x):
    """The value that a cached row stands for, element by element in 64 bits ([..., D])."""
    x = x.double()
    fine = torch.isfinite(x).all(-1, keepdim=True)
    x0 = torch.where(fine, x, torch.zeros_like(x))
    top = x0.abs().amax(-1, keepdim=True)
    e = torch.full_like(top, -126.0)
    for k in range(-126, 129):  # the smallest e with top <= 448 * 2^e
        e = torch.where((top > 448.0 * 2.0 ** (k - 1)) & (top <= 448.0 * 2.0 ** k) & (k > -126),
                        torch.full_like(e, float(k)), e)
    y = x0 * torch.exp2(-e)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)  # e4m3: 3 bits, 2^-9 at least
    y = torch.round(y / step) * step * torch.exp2(e)
    return torch.where(fine, y, torch.full_like(y, float("nan")))


def stored64(arena, layer, page, tok):
    """[heads, 2, D] of one cached token, byte by byte from the layout."""
    d = arena.shape[-1] // PAGE - 1
    n = d // 16
    swz = min(n & -n, 8) - 1
    raw = arena[page, layer].cpu()
    out = torch.empty(raw.shape[0], 2, d, dtype=torch.float64)
    for c in range(n):
        at = tok * d + (c ^ (tok & swz)) * 16
        out[:, :, 16 * c:16 * c + 16] = raw[:, :, at:at + 16].contiguous().view(torch.float8_e4m3fn).double()
    b = raw[:, :, PAGE * d + tok].double()
    scale = torch.where(b == 255, torch.full_like(b, float("nan")), torch.exp2(b - 127))
    scale = torch.where(b == 0, torch.zeros_like(b), scale)
    return out * scale[..., None]


def attend64(q, k, v, lim, scale):
    """q [n, hq, D], k/v [L, hkv, D] in 64 bits, row i sees keys [0, lim[i]): the result, the mean of
    |v| under the same weights, and the largest sum of |q_d k_d| * scale of a row."""
    g = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    z = torch.einsum("nhd,lhd->nhl", q, k) * scale
    mask = torch.arange(k.shape[0], device=q.device)[None, :] >= lim[:, None]
    z = z.masked_fill(mask[:, None], float("-inf"))
    none = (lim <= 0)[:, None, None]
    p = torch.where(none, torch.zeros_like(z), torch.softmax(z.masked_fill(none, 0.0), -1))
    p = torch.where(mask[:, None], torch.zeros_like(p), p)
    # a key that a row does not see counts for nothing, whatever it holds
    o = torch.stack([torch.einsum("hl,lhd->hd", p[i, :, :int(lim[i])], v[:int(lim[i])]) for i in range(len(lim))])
    w = torch.stack([torch.einsum("hl,lhd->hd", p[i, :, :int(lim[i])], v[:int(lim[i])].abs())
                     for i in range(len(lim))])
    size = torch.einsum("nhd,lhd->nhl", q.abs(), k.abs()) * scale
    size = size.masked_fill(mask[:, None], 0.0).amax(-1) if k.shape[0] else torch.zeros_like(o[..., 0])
    return o, w, size


def attention_tolerance(o, w, size, vmax):
    """How far a kernel's bf16 result may be from o:
    the final rounding, half a bf16 step: 2^-8 |o|;
    P rounded to fp16, half a step each: 2^-11 of the mean |v|;
    scores: fp32 sums of 128 exact products and their scaling, at most (128 + 4) 2^-24 of
    sum |q_d k_d| each, which moves p by that part in the numerator and in the denominator: 2^-15 size;
    ex2.approx (2^-22) and the rounding of its argument (2^-24 of at most ~2 size / ln 2): within 2^-15 (1 + size);
    P below fp16's normal range, or V below it where the kernel scales V by tile: 2^-17 of the largest |v|."""
    return 2.0 ** -8 * o.abs() + (2.0 ** -11 + 2.0 ** -14 * (1 + size[..., None])) * w + 2.0 ** -17 * vmax


# ------------------------------------------------------------------ inputs
def rows(n, heads, d, g, spread=0.3):
    x = torch.randn(n, heads, d, generator=g, dtype=torch.float32)
    return x * torch.exp(spread * torch.randn(n, heads, 1, generator=g))


def special_rows(heads, d, g):
    """Rows at the edges of the format (each repeated over the heads with another order of elements)."""
    f = torch.finfo(BF)
    out = []
    for kind in ("zero", "one", "top448", "over448", "tiny", "subnormal", "huge", "ties", "wide", "inf", "nan",
                 "negative"):
        x = torch.zeros(heads, d)
        if kind == "one":
            x[:, 3] = 1.0
        elif kind == "top448":
            x[:] = 448.0 * torch.sign(torch.randn(heads, d, generator=g))
        elif kind == "over448":
            x[:, 0] = 450.0
            x[:, 1:] = torch.randn(heads, d - 1, generator=g)
        elif kind == "tiny":
            x[:] = torch.randn(heads, d, generator=g) * f.tiny
        elif kind == "subnormal":
            x[:, ::2] = 2.0 ** -133
            x[:, 1] = 2.0 ** -128
        elif kind == "huge":
            x[:] = torch.randn(heads, d, generator=g).clamp(-2, 2) * 2.0 ** 125
        elif kind == "ties":  # halfway between two codes
            x[:] = (torch.arange(d) % 8 + 8 + 0.5)[None] * 16.0
        elif kind == "wide":
            x[:] = torch.exp2(-torch.arange(d).float() / 4)[None]
        elif kind == "inf":
            x[:] = torch.randn(heads, d, generator=g)
            x[:, d // 2] = float("-inf")
        elif kind == "nan":
            x[:] = torch.randn(heads, d, generator=g)
            x[:, d - 1] = float("nan")
        elif kind == "negative":
            x[:] = -torch.rand(heads, d, generator=g)
        out.append(x)
    return torch.stack(out).to(BF).float()


def same(a, b):
    return torch.equal(torch.nan_to_num(a, nan=12345.0), torch.nan_to_num(b, nan=12345.0)) \
        and torch.equal(torch.isnan(a), torch.isnan(b))


def build(lens, hq, hkv, layers, layer, g, device, d=128, spread=0.3, garbage=True, extra_cols=0):
    """An arena with shuffled pages holding the sequences' random K and V, bytes past their ends
    random (garbage) where asked; the block tables and the cached values in 64 bits per sequence."""
    nb = [-(-x // PAGE) for x in lens]
    blocks = sum(nb) + 3
    arena = ops.kv8_arena(blocks, layers, hkv, head_dim=d, device="cpu")
    if garbage:
        arena.copy_(torch.randint(0, 256, arena.shape, generator=g, dtype=torch.uint8))
    perm = torch.randperm(blocks, generator=g)
    bt = torch.full((len(lens), max(nb + [1]) + extra_cols), blocks - 1, dtype=torch.int32)
    cached, at = [], 0
    for s, n in enumerate(lens):
        bt[s, :nb[s]] = perm[at:at + nb[s]].to(torch.int32)
        at += nb[s]
        k, v = rows(n, hkv, d, g, spread).to(BF), rows(n, hkv, d, g, spread).to(BF)
        j = torch.arange(n)
        ops.kv8_write(k.reshape(n, hkv * d), v.reshape(n, hkv * d), bt[s].long()[j // PAGE] * PAGE + j % PAGE, arena, layer)
        cached.append((quantize64(k), quantize64(v)))
    return arena.to(device), bt.to(device), cached


# ------------------------------------------------------------------ rows, CPU
@pytest.mark.parametrize("d", [16, 48, 64, 128, 256])
def test_rows_round_trip_cpu(d):
    g = torch.Generator().manual_seed(d)
    heads = 3
    x = torch.cat([special_rows(heads, d, g), rows(30, heads, d, g).to(BF).float()])
    y = torch.cat([rows(30, heads, d, g).to(BF).float(), special_rows(heads, d, g)])
    t = x.shape[0]
    arena = ops.kv8_arena(6, 2, heads, head_dim=d, device="cpu")
    slots = torch.randperm(6 * PAGE, generator=g)[:t]
    slots[4] = -1
    ops.kv8_write(x.reshape(t, -1), y.reshape(t, -1), slots, arena, 1)
    k, v = ops.kv8_read(arena, 1, slots)
    keep = slots >= 0
    assert same(k.view(t, heads, d).double()[keep], quantize64(x)[keep].to(BF).double())
    assert same(v.view(t, heads, d).double()[keep], quantize64(y)[keep].to(BF).double())
    assert not k[4].any() and not v[4].any()
    for i in (0, 7, 12, 40):
        if slots[i] >= 0:
            got = stored64(arena, 1, int(slots[i]) // PAGE, int(slots[i]) % PAGE)
            assert same(got[:, 0], quantize64(x)[i]) and same(got[:, 1], quantize64(y)[i])
    assert not arena[:, 0].any()  # the other layer is left as it was
    fresh = ops.kv8_read(ops.kv8_arena(2, 1, heads, head_dim=d, device="cpu"), 0, torch.arange(5))
    assert not fresh[0].any()


def test_quantisation_error_is_half_a_step():
    g = torch.Generator().manual_seed(0)
    x = rows(200, 2, 128, g).to(BF)
    err = (quantize64(x) - x.double()).abs()
    top = x.double().abs().amax(-1, keepdim=True)
    # e4m3 rounds by at most 2^-4 of the value, or by half of its smallest step, 2^-10 * 2^e, 2^e < top / 224
    assert bool((err <= torch.maximum(2.0 ** -4 * x.double().abs(), 2.0 ** -10 * top / 224)).all())


def test_row_bytes_do_not_depend_on_the_page():
    """Token by token, in one chunk, and after rows that were overwritten: the same bytes."""
    g = torch.Generator().manual_seed(1)
    k, v = rows(16, 2, 128, g).to(BF).reshape(16, -1), rows(16, 2, 128, g).to(BF).reshape(16, -1)
    big = 1000 * k
    a, b, c = (ops.kv8_arena(1, 1, 2, device="cpu") for _ in range(3))
    ops.kv8_write(k, v, torch.arange(16), a, 0)
    for i in range(16):
        ops.kv8_write(k[i:i + 1], v[i:i + 1], torch.tensor([i]), b, 0)
    ops.kv8_write(big, big, torch.arange(16), c, 0)
    ops.kv8_write(k, v, torch.arange(16), c, 0)
    assert torch.equal(a, b) and torch.equal(a, c)


def test_arena_refusals_cpu():
    with pytest.raises(ValueError):
        ops.kv8_arena(2, 1, 1, head_dim=100, device="cpu")
    a = ops.kv8_arena(2, 1, 1, device="cpu")
    with pytest.raises(IndexError):
        ops.kv8_write(torch.zeros(1, 128), torch.zeros(1, 128), torch.tensor([99]), a, 0)


# ------------------------------------------------------------------ attention, CPU
@pytest.mark.parametrize("d", [64, 128])
def test_decode_and_prefill_cpu(d):
    g = torch.Generator().manual_seed(2)
    lens, hq, hkv = [0, 1, 16, 17, 50], 4, 2
    arena, bt, cached = build(lens, hq, hkv, 2, 1, g, "cpu", d=d, garbage=False)
    scale = 1 / math.sqrt(d)
    q = torch.randn(len(lens), hq * d, generator=g)
    out = ops.paged_decode_attention(q, arena, 1, bt, torch.tensor(lens, dtype=torch.int32), hq, hkv, scale)
    for s, n in enumerate(lens):
        o, _, _ = attend64(q[s:s + 1].double().view(1, hq, d), *cached[s], torch.tensor([n]), scale)
        assert torch.allclose(out[s].double(), o.flatten(), atol=1e-5, rtol=1e-5)
    new = [0, 1, 5, 3, 20]
    qs = torch.tensor([0, 0, 1, 6, 9, 29], dtype=torch.int32)
    pos = torch.cat([torch.arange(n - m, n, dtype=torch.int32) for n, m in zip(lens, new)])
    q = torch.randn(29, hq * d, generator=g)
    out = ops.paged_prefill_attention(q, arena, 1, bt, torch.tensor(lens, dtype=torch.int32), None, qs, pos, hq, hkv,
                                      scale)
    for s in range(len(lens)):
        a, b = int(qs[s]), int(qs[s + 1])
        if b > a:
            o, _, _ = attend64(q[a:b].double().view(b - a, hq, d), *cached[s], pos[a:b].long() + 1, scale)
            assert torch.allclose(out[a:b].double(), o.reshape(b - a, -1), atol=1e-5, rtol=1e-5)


def test_linear_qkv_cpu_writes_the_8bit_arena():
    g = torch.Generator().manual_seed(3)
    t, hid, hq, hkv, d = 5, 32, 4, 2, 64
    a, w = torch.randn(t, hid, generator=g), torch.randn((hq + 2 * hkv) * d, hid, generator=g)
    cs = ref.rope_cache(64, 10000.0, d)
    pos = torch.tensor([3, 4, 5, 0, 9], dtype=torch.int32)
    slots = torch.tensor([3, 4, 5, -1, 25])
    arena = ops.kv8_arena(2, 1, hkv, head_dim=d, device="cpu")
    dense = torch.zeros(2, 1, 2, hkv, PAGE, d)
    qa, qb = torch.empty(t, hq * d), torch.empty(t, hq * d)
    ops.linear_qkv(a, w, qa, cs, pos, slots, arena, 0, hq, hkv)
    ops.linear_qkv(a, w, qb, cs, pos, slots, dense, 0, hq, hkv)
    assert torch.equal(qa, qb)
    k, v = ref.gather_kv(arena, 0, torch.tensor([0, 1]), 32)
    kd, vd = ref.gather_kv(dense, 0, torch.tensor([0, 1]), 32)
    at = slots[slots >= 0]
    assert same(k[at].double(), quantize64(kd[at])) and same(v[at].double(), quantize64(vd[at]))


# ------------------------------------------------------------------ rows, GPU
@pytest.mark.gpu
@pytest.mark.parametrize("heads", [1, 2, 8])
def test_rows_round_trip_gpu(cuda_dev, heads):
    g = torch.Generator().manual_seed(heads)
    x = torch.cat([special_rows(heads, 128, g), rows(70, heads, 128, g).to(BF).float()]).to(BF)
    y = torch.cat([rows(70, heads, 128, g).to(BF).float(), special_rows(heads, 128, g)]).to(BF)
    t = x.shape[0]
    slots = torch.randperm(8 * PAGE, generator=g)[:t]
    slots[3] = -1
    base = torch.randint(0, 255, (8, 3, heads, 2, 2064), generator=g, dtype=torch.uint8)
    want = base.clone()
    ops.kv8_write(x.reshape(t, -1).float(), y.reshape(t, -1).float(), slots, want, 1)
    # K and V as strided views of one packed projection, behind q columns
    packed = torch.zeros(t, (4 + 2 * heads) * 128, dtype=BF)
    packed[:, 512:512 + heads * 128] = x.reshape(t, -1)
    packed[:, 512 + heads * 128:] = y.reshape(t, -1)
    packed = packed.to(cuda_dev)
    arena = base.to(cuda_dev)
    ops.kv8_write(packed[:, 512:512 + heads * 128], packed[:, 512 + heads * 128:], slots.to(cuda_dev), arena, 1)
    assert torch.equal(arena.cpu(), want)  # the same bytes, and nothing else touched
    k, v = ops.kv8_read(arena, 1, slots.to(cuda_dev))
    kc, vc = ops.kv8_read(want, 1, slots)
    assert same(k.cpu().float(), kc.float()) and same(v.cpu().float(), vc.float())
    keep = slots >= 0
    assert same(k.cpu().view(t, heads, 128).double()[keep], quantize64(x)[keep].to(BF).double())
    assert not k[3].any() and not v[3].any()
    wide = torch.full((t, heads * 256), 7.0, dtype=BF, device=cuda_dev)
    ops.kv8_read(arena, 1, slots.to(cuda_dev), k_out=wide[:, :heads * 128], v_out=wide[:, heads * 128:])
    assert same(wide[:, :heads * 128].float(), k.float()) and same(wide[:, heads * 128:].float(), v.float())
    empty = torch.empty(0, heads * 128, dtype=BF, device=cuda_dev)
    ops.kv8_write(empty, empty, torch.empty(0, dtype=torch.int64, device=cuda_dev), arena, 1)
    assert ops.kv8_read(arena, 1, torch.empty(0, dtype=torch.int64, device=cuda_dev))[0].shape == (0, heads * 128)
    ops.core.check_status(cuda_dev)


@pytest.mark.gpu
def test_all_codes_and_scales_read_exactly(cuda_dev):
    arena = ops.kv8_arena(16, 1, 1, device=cuda_dev)
    codes = torch.arange(256, dtype=torch.uint8).view(2, 128)
    for page in range(16):
        for t in range(PAGE):
            at = ref._kv8_cols(torch.tensor([t]), 128)[0].to(cuda_dev)
            arena[page, 0, 0, 0, at] = codes[0].to(cuda_dev)
            arena[page, 0, 0, 1, at] = codes[1].to(cuda_dev)
            arena[page, 0, 0, :, 2048 + t] = page * 16 + t
    slots = torch.arange(256, device=cuda_dev)
    k, v = ops.kv8_read(arena, 0, slots)
    kc, vc = ops.kv8_read(arena.cpu(), 0, slots.cpu())
    assert same(k.cpu().float(), kc.float()) and same(v.cpu().float(), vc.float())


@pytest.mark.gpu
def test_rows_refusals_gpu(cuda_dev):
    a = ops.kv8_arena(2, 1, 2, device=cuda_dev)
    x = torch.zeros(3, 256, dtype=BF, device=cuda_dev)
    s = torch.tensor([0, 40, 1], device=cuda_dev)  # 40: past the arena's 32 slots
    for bad in (dict(k=x.float()), dict(k=x[:, :128]), dict(slots=s.int()), dict(slots=s[:2]), dict(layer=1),
                dict(layer=-1), dict(arena=a[:, :, :1]), dict(arena=a.view(torch.int8)), dict(k=x.cpu()),
                dict(slots=s.cpu())):
        kw = dict(k=x, v=x, slots=s, arena=a, layer=0) | bad
        with pytest.raises(RuntimeError):
            ops.kv8_write(**kw)
    odd = ops.kv8_arena(2, 1, 2, head_dim=64, device=cuda_dev)
    with pytest.raises(RuntimeError, match="head_dim"):
        ops.kv8_write(x[:, :128], x[:, :128], s, odd, 0)
    ops.core.check_status(cuda_dev)
    ops.kv8_write(x + 1, x + 2, s, a, 0)
    with pytest.raises(ops.core.KernelError, match="out of bounds"):
        ops.core.check_status(cuda_dev)
    k, v = ops.kv8_read(a, 0, s)
    with pytest.raises(ops.core.KernelError, match="out of bounds"):
        ops.core.check_status(cuda_dev)
    assert k[0, 0] == 1 and v[2, 5] == 2 and not k[1].any()


# ------------------------------------------------------------------ decode, GPU
def check_decode(dev, lens, hq, hkv, seed, layers=2, layer=1, spread=0.3, qscale=1.5, **kw):
    g = torch.Generator().manual_seed(seed)
    arena, bt, cached = build(lens, hq, hkv, layers, layer, g, dev, spread=spread, **kw)
    scale = 1 / math.sqrt(128)
    q = (torch.randn(len(lens), hq * 128, generator=g) * qscale).to(BF)
    sl = torch.tensor(lens, dtype=torch.int32, device=dev)
    out = ops.paged_decode_attention(q.to(dev), arena, layer, bt, sl, hq, hkv, scale)
    ops.core.check_status(dev)
    again = ops.paged_decode_attention(q.to(dev), arena, layer, bt, sl, hq, hkv, scale)
    assert torch.equal(out, again)
    for s, n in enumerate(lens):
        k, v = (x.to(dev) for x in cached[s])
        o, w, size = attend64(q[s:s + 1].to(dev).double().view(1, hq, 128), k, v, torch.tensor([n], device=dev), scale)
        vmax = v.abs().amax() if n else torch.zeros((), device=dev)
        err = (out[s].double().view(1, hq, 128) - o).abs()
        tol = attention_tolerance(o, w, size, vmax)
        assert bool((err <= tol).all()), (s, n, float((err - tol).amax()), float(err.amax()))


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv", [(1, 1), (4, 4), (4, 2), (8, 2), (6, 2), (16, 2), (7, 1), (24, 2), (40, 1), (128, 1)])
def test_decode_heads(cuda_dev, hq, hkv):
    check_decode(cuda_dev, [1, 33, 200], hq, hkv, 10 + hq)


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[0], [1], [0, 0, 5, 0], [15, 16, 17], [63, 64, 65], [320, 321, 319], [1000], [4097],
                                  [3] * 70, [1, 5000, 2, 700, 0, 64], [257] * 40 + [0] * 9])
def test_decode_lengths(cuda_dev, lens):
    check_decode(cuda_dev, lens, 8, 2, 100 + len(lens) + lens[0], extra_cols=3)


@pytest.mark.gpu
@pytest.mark.parametrize("lens,hq,hkv", [([200, 16, 0, 700], 8, 2), ([5], 16, 1), ([0, 0], 8, 2), ([768] * 12, 8, 2),
                                         ([30] * 148, 4, 2), ([30] * 149, 4, 2), ([17] * 300, 2, 1), ([769, 20], 8, 2)])
def test_decode_few_pages_in_a_wide_table(cuda_dev, lens, hq, hkv):
    """Segments that are not cut although the table is wide, and the first that are."""
    check_decode(cuda_dev, lens, hq, hkv, 70 + len(lens), extra_cols=80)


@pytest.mark.gpu
@pytest.mark.parametrize("spread,qscale", [(3.0, 1.0), (0.3, 40.0), (8.0, 0.01), (0.0, 1e-20)])
def test_decode_values(cuda_dev, spread, qscale):
    """Rows whose scales differ by many octaves, sharp and flat softmax, tiny queries."""
    check_decode(cuda_dev, [90, 700], 8, 2, 7, spread=spread, qscale=qscale)


@pytest.mark.gpu
def test_decode_strided_rows_and_unseen_pages(cuda_dev):
    """q and out as views of wider rows; table entries past a sequence's pages name no page at all."""
    g = torch.Generator().manual_seed(5)
    lens, hq, hkv = [40, 0, 7], 8, 2
    arena, bt, cached = build(lens, hq, hkv, 1, 0, g, cuda_dev, extra_cols=2)
    sl = torch.tensor(lens, dtype=torch.int32, device=cuda_dev)
    for s, n in enumerate(lens):
        bt[s, -(-n // PAGE):] = -7
    wide = torch.randn(4, 3 * hq * 128, generator=g).to(BF).to(cuda_dev)
    q = wide[:, hq * 128:2 * hq * 128]
    res = torch.full((5, 2 * hq * 128), 3.0, dtype=BF, device=cuda_dev)
    ops.paged_decode_attention(q, arena, 0, bt, sl, hq, hkv, 0.1, out=res[:, :hq * 128])
    ops.core.check_status(cuda_dev)
    plain = ops.paged_decode_attention(q[:3].contiguous(), arena, 0, bt, sl, hq, hkv, 0.1)
    assert torch.equal(res[:3, :hq * 128], plain) and not plain[1].any()
    assert bool((res[3:] == 3.0).all()) and bool((res[:, hq * 128:] == 3.0).all())


@pytest.mark.gpu
def test_decode_non_finite_rows(cuda_dev):
    """A NaN or infinite row reaches what sees it and nothing else."""
    g = torch.Generator().manual_seed(6)
    lens, hq, hkv = [50, 50, 50], 8, 2
    arena, bt, cached = build(lens, hq, hkv, 1, 0, g, cuda_dev)
    q = torch.randn(3, hq * 128, generator=g).to(BF).to(cuda_dev)
    sl = torch.tensor(lens, dtype=torch.int32, device=cuda_dev)
    clean = ops.paged_decode_attention(q, arena, 0, bt, sl, hq, hkv, 0.1)
    at = int(bt[1, 2]) * PAGE + 5
    k, v = ops.kv8_read(arena, 0, torch.tensor([at], device=cuda_dev))
    v[0, 130] = float("inf")  # KV head 1
    ops.kv8_write(k, v, torch.tensor([at], device=cuda_dev), arena, 0)
    out = ops.paged_decode_attention(q, arena, 0, bt, sl, hq, hkv, 0.1)
    assert torch.equal(out[0], clean[0]) and torch.equal(out[2], clean[2]) and torch.equal(out[1, :512], clean[1, :512])
    assert bool(torch.isnan(out[1, 512:]).all())
    sl[1] = 37  # the row is no longer seen
    short = ops.paged_decode_attention(q, arena, 0, bt, sl, hq, hkv, 0.1)
    assert bool(torch.isfinite(short.float()).all())


@pytest.mark.gpu
def test_decode_refusals_and_bad_pages(cuda_dev):
    g = torch.Generator().manual_seed(8)
    arena, bt, _ = build([40, 20], 8, 2, 1, 0, g, cuda_dev)
    q = torch.zeros(2, 1024, dtype=BF, device=cuda_dev)
    sl = torch.tensor([40, 20], dtype=torch.int32, device=cuda_dev)
    for bad in (dict(q=q.float()), dict(q=q[:1]), dict(q=q[:, :512]), dict(layer=3), dict(block_tables=bt.long()),
                dict(block_tables=bt[:1]), dict(seq_lens=sl.long()), dict(n_kv_heads=4), dict(n_q_heads=7),
                dict(block_tables=bt.cpu()), dict(seq_lens=sl.cpu()), dict(n_q_heads=0)):
        kw = dict(q=q, arena=arena, layer=0, block_tables=bt, seq_lens=sl, n_q_heads=8, n_kv_heads=2, scale=0.1) | bad
        with pytest.raises(RuntimeError):
            ops.paged_decode_attention(**kw, out=torch.empty(2, 1024, dtype=BF, device=cuda_dev))
    ops.core.check_status(cuda_dev)
    good = ops.paged_decode_attention(q, arena, 0, bt, sl, 8, 2, 0.1)
    for page in (arena.shape[0], -1, 2 ** 31 - 1):
        worse = bt.clone()
        worse[0, 1] = page
        out = ops.paged_decode_attention(q, arena, 0, worse, sl, 8, 2, 0.1)
        with pytest.raises(ops.core.KernelError, match="out of bounds"):
            ops.core.check_status(cuda_dev)
        assert torch.equal(out[1], good[1])


# ------------------------------------------------------------------ prefill, GPU
def check_prefill(dev, lens, new, hq, hkv, seed, layers=2, layer=1, tile=128, spread=0.3, qscale=1.5, pad_tiles=0):
    g = torch.Generator().manual_seed(seed)
    arena, bt, cached = build(lens, hq, hkv, layers, layer, g, dev, spread=spread)
    scale = 1 / math.sqrt(128)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    t = starts[-1]
    q = (torch.randn(t + 2, hq * 128, generator=g) * qscale).to(BF).to(dev)
    pos = torch.cat([torch.arange(n - m, n, dtype=torch.int32) for n, m in zip(lens, new)]).to(dev)
    qs = torch.tensor(starts, dtype=torch.int32, device=dev)
    sl = torch.tensor(lens, dtype=torch.int32, device=dev)
    tiles = ops.build_prefill_tiles(starts, [n - m for n, m in zip(lens, new)], tile=tile, device=dev)
    if pad_tiles:
        tiles = torch.cat([tiles, torch.zeros(pad_tiles, 4, dtype=torch.int32, device=dev)])
    out = torch.full((t + 2, hq * 128), 5.0, dtype=BF, device=dev)
    ops.paged_prefill_attention(q, arena, layer, bt, sl, tiles, qs, pos, hq, hkv, scale, out=out)
    ops.core.check_status(dev)
    assert bool((out[t:] == 5.0).all())  # rows behind the last sequence
    again = torch.full_like(out, 5.0)
    ops.paged_prefill_attention(q, arena, layer, bt, sl, tiles, qs, pos, hq, hkv, scale, out=again)
    assert torch.equal(out, again)
    for s, n in enumerate(lens):
        a, b = starts[s], starts[s + 1]
        if b == a:
            continue
        k, v = (x.to(dev) for x in cached[s])
        o, w, size = attend64(q[a:b].double().view(b - a, hq, 128), k, v, pos[a:b].long() + 1, scale)
        err = (out[a:b].double().view(b - a, hq, 128) - o).abs()
        tol = attention_tolerance(o, w, size, v.abs().amax())
        assert bool((err <= tol).all()), (s, n, float((err - tol).amax()), float(err.amax()))


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv", [(1, 1), (4, 4), (4, 2), (8, 2), (6, 2), (16, 2), (5, 1), (24, 2), (40, 1), (64, 1),
                                    (96, 1), (128, 1), (256, 1)])
def test_prefill_heads(cuda_dev, hq, hkv):
    check_prefill(cuda_dev, [140, 33], [140, 7], hq, hkv, 20 + hq)


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv", [(32, 8), (64, 8), (40, 8), (24, 8), (16, 16), (128, 2)])
def test_prefill_more_tiles_than_half_the_gpu(cuda_dev, hq, hkv):
    """(the launches above have one product in a CTA, these two)"""
    check_prefill(cuda_dev, [700, 900, 300], [640, 515, 300], hq, hkv, 60 + hq)
    check_prefill(cuda_dev, [1300], [1201], hq, hkv, 61 + hq)


@pytest.mark.gpu
@pytest.mark.parametrize("lens,new", [([1], [1]), ([16], [16]), ([17], [1]), ([127], [127]), ([128], [128]),
                                      ([129], [129]), ([300], [172]), ([700, 5, 90], [300, 5, 1]),
                                      ([40, 0, 60], [5, 0, 5]), ([513], [257]), ([1030, 2, 2], [6, 2, 1]),
                                      ([1500], [640]), ([200] * 12, [5] * 12), ([256, 2000], [256, 3]),
                                      # few rows beside many: of so many keys that they go by themselves, or not
                                      ([300, 5000], [300, 20]), ([40, 2000, 1900], [20, 640, 513]),
                                      ([60] * 300 + [900, 0], [40] * 300 + [7, 0])])
def test_prefill_lengths(cuda_dev, lens, new):
    check_prefill(cuda_dev, lens, new, 8, 2, 200 + lens[0], pad_tiles=2)


@pytest.mark.gpu
@pytest.mark.parametrize("spread,qscale", [(1.5, 1.0), (0.3, 40.0), (0.0, 1e-20)])
def test_prefill_values(cuda_dev, spread, qscale):
    check_prefill(cuda_dev, [400, 150], [300, 9], 8, 2, 9, spread=spread, qscale=qscale)


@pytest.mark.gpu
@pytest.mark.parametrize("tile", [5, 64])
def test_prefill_smaller_tiles(cuda_dev, tile):
    check_prefill(cuda_dev, [150, 70], [150, 33], 8, 2, 11, tile=tile)


@pytest.mark.gpu
def test_prefill_non_finite_rows(cuda_dev):
    """A row that is not finite reaches the rows that see it: those before it in the chunk stay as they were."""
    g = torch.Generator().manual_seed(12)
    n, hq, hkv = 200, 8, 2
    arena, bt, _ = build([n], hq, hkv, 1, 0, g, cuda_dev)
    q = torch.randn(n, hq * 128, generator=g).to(BF).to(cuda_dev)
    sl = torch.tensor([n], dtype=torch.int32, device=cuda_dev)
    qs, pos = torch.tensor([0, n], dtype=torch.int32, device=cuda_dev), torch.arange(n, dtype=torch.int32, device=cuda_dev)
    tiles = ops.build_prefill_tiles([0, n], [0], device=cuda_dev)
    args = (bt, sl, tiles, qs, pos, hq, hkv, 0.1)
    clean = ops.paged_prefill_attention(q, arena, 0, *args)
    for side in (0, 1):
        for tok in (37, 150):
            a2 = arena.clone()
            at = torch.tensor([int(bt[0, tok // PAGE]) * PAGE + tok % PAGE], device=cuda_dev)
            kv = ops.kv8_read(arena, 0, at)
            kv[side][0, 5] = float("nan")  # KV head 0
            ops.kv8_write(*kv, at, a2, 0)
            out = ops.paged_prefill_attention(q, a2, 0, *args)
            assert torch.equal(out[:tok], clean[:tok]) and torch.equal(out[:, 512:], clean[:, 512:])
            assert bool(torch.isnan(out[tok:, :512]).all())


@pytest.mark.gpu
def test_prefill_refusals(cuda_dev):
    g = torch.Generator().manual_seed(13)
    arena, bt, _ = build([40], 8, 2, 1, 0, g, cuda_dev)
    q = torch.zeros(40, 1024, dtype=BF, device=cuda_dev)
    sl = torch.tensor([40], dtype=torch.int32, device=cuda_dev)
    tiles = ops.build_prefill_tiles([0, 40], [0], device=cuda_dev)
    for bad in (dict(q=q.float()), dict(tiles=tiles.long()), dict(tiles=tiles[:, :3]), dict(tiles=tiles.cpu()),
                dict(layer=1), dict(n_kv_heads=1), dict(n_q_heads=4)):
        kw = dict(q=q, arena=arena, layer=0, block_tables=bt, seq_lens=sl, tiles=tiles, query_start=None,
                  positions=None, n_q_heads=8, n_kv_heads=2, scale=0.1) | bad
        with pytest.raises(RuntimeError):
            ops.paged_prefill_attention(**kw, out=torch.empty(40, 1024, dtype=BF, device=cuda_dev))
    bt[0, 1] = arena.shape[0] + 3
    ops.paged_prefill_attention(q, arena, 0, bt, sl, tiles, None, None, 8, 2, 0.1)
    with pytest.raises(ops.core.KernelError, match="out of bounds"):
        ops.core.check_status(cuda_dev)
    none = ops.paged_prefill_attention(q[:0], arena, 0, bt, sl, tiles[:0], None, None, 8, 2, 0.1)
    assert none.shape == (0, 1024)
    for table in (bt, bt[:, :1].expand(1, 80).contiguous()):  # no rows, tiles that are all padding
        none = ops.paged_prefill_attention(q[:0], arena, 0, table, sl, torch.zeros_like(tiles), None, None, 8, 2, 0.1)
        assert none.shape == (0, 1024)
    ops.core.check_status(cuda_dev)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [3, 200])  # both kernels
@pytest.mark.parametrize("case", ["values grow", "values fall", "keys near the smallest"])
def test_far_apart_magnitudes(cuda_dev, rows, case):
    """V rows 2^160 apart in one sequence, and K rows of e4m3's smallest scale under queries that make up for it."""
    g = torch.Generator().manual_seed(19)
    n, hq, hkv, scale = 500, 8, 2, 0.09
    arena, bt, _ = build([n], hq, hkv, 1, 0, g, cuda_dev)
    j = torch.arange(n)
    slots = bt[0].cpu().long()[j // PAGE] * PAGE + j % PAGE
    k, v = torch.randn(n, hkv, 128, generator=g), torch.randn(n, hkv, 128, generator=g)
    q = torch.randn(rows, hq, 128, generator=g)
    if case == "values grow":
        v[:300] *= 2.0 ** -70
        v[300:] *= 2.0 ** 90
    elif case == "values fall":
        v[:300] *= 2.0 ** 90
        v[300:] *= 2.0 ** -70
    else:
        k *= 2.0 ** -122
        q *= 2.0 ** 121
    k, v, q = k.to(BF), v.to(BF), q.to(BF)
    ops.kv8_write(k.view(n, -1).to(cuda_dev), v.view(n, -1).to(cuda_dev), slots.to(cuda_dev), arena, 0)
    sl = torch.tensor([n], dtype=torch.int32, device=cuda_dev)
    tiles = ops.build_prefill_tiles([0, rows], [n - rows], device=cuda_dev)
    out = ops.paged_prefill_attention(q.view(rows, -1).to(cuda_dev), arena, 0, bt, sl, tiles, None, None, hq, hkv, scale)
    ops.core.check_status(cuda_dev)
    k64, v64 = quantize64(k).to(cuda_dev), quantize64(v).to(cuda_dev)
    lim = torch.arange(n - rows + 1, n + 1, device=cuda_dev)
    o, w, size = attend64(q.double().to(cuda_dev), k64, v64, lim, scale)
    # a row's own largest value: those that it does not see do not count for its error
    big = torch.stack([v64[:int(x)].abs().amax() for x in lim])
    tol = torch.stack([attention_tolerance(o[i:i + 1], w[i:i + 1], size[i:i + 1], big[i])[0] for i in range(rows)])
    err = (out.double().view(rows, hq, 128) - o).abs()
    assert bool((err <= tol).all()), float((err / tol).amax())


def check_contributions(out, q, k, v, lim, scale):
    """`out` [n, hq, 128] against 64-bit attention, held to what a row's own keys add to it:
    the final rounding, P's and the scores' as in attention_tolerance, with |v| weighted and the scores' size that
    of the keys whose weight is at least 2^-40 (the others are below every bound here);
    P below fp16's normal range: half of its smallest step, 2^-25, where the largest P |v| has a P of at least
    2^-1 and both |v| are codes of at most 448 against one of at least 224: 2^-23 of the largest p |v| for each key."""
    g = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    for i in range(q.shape[0]):
        n = int(lim[i])
        z = torch.einsum("hd,lhd->hl", q[i], k[:n]) * scale
        p = torch.softmax(z, -1)
        size = (torch.einsum("hd,lhd->hl", q[i].abs(), k[:n].abs()) * scale).masked_fill(p < 2.0 ** -40, 0.0).amax(-1)
        o, w = (torch.einsum("hl,lhd->hd", p, x) for x in (v[:n], v[:n].abs()))
        top = (p * v[:n].abs().amax(-1).t()).amax(-1)[:, None]
        tol = 2.0 ** -8 * o.abs() + (2.0 ** -11 + 2.0 ** -14 * (1 + size[:, None])) * w + n * 2.0 ** -23 * top + 2.0 ** -134
        err = (out[i].double() - o).abs()
        assert bool((err <= tol).all()), (i, n, float((err / tol).nan_to_num(nan=float("inf")).amax()))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [4, 230])  # both kernels
@pytest.mark.parametrize("octaves", [7, 9, 14, 17, 26, 60, 110])
@pytest.mark.parametrize("side", ["k", "v"])
def test_a_large_key_counts_for_the_rows_that_see_it(cuda_dev, rows, octaves, side):
    """One key of the chunk is 2^octaves times the others: rows before it come out as if it were not there, to
    the accuracy of their own keys, and rows that see it with hardly any weight as well."""
    g = torch.Generator().manual_seed(23)
    n, hq, hkv, scale = 300, 8, 2, 0.09
    arena, bt, _ = build([n], hq, hkv, 1, 0, g, cuda_dev)
    j = torch.arange(n)
    slots = bt[0].cpu().long()[j // PAGE] * PAGE + j % PAGE
    k, v = torch.randn(n, hkv, 128, generator=g), torch.randn(n, hkv, 128, generator=g)
    q = torch.randn(rows, hq, 128, generator=g)
    q[..., 0] = 3.0
    for at, head in ((n - 2, 0), (n - rows // 2, 1)):
        if side == "k":  # a score far below the others for the rows that see it
            k[at, head] = 0.0
            k[at, head, 0] = -(2.0 ** octaves)
        else:  # a weight that the value does not make up for: 2^-160, octaves < 160
            k[at, head] = 0.0
            k[at, head, 0] = -420.0
            v[at, head] *= 2.0 ** octaves
    k, v, q = k.to(BF), v.to(BF), q.to(BF)
    ops.kv8_write(k.view(n, -1).to(cuda_dev), v.view(n, -1).to(cuda_dev), slots.to(cuda_dev), arena, 0)
    sl = torch.tensor([n], dtype=torch.int32, device=cuda_dev)
    tiles = ops.build_prefill_tiles([0, rows], [n - rows], device=cuda_dev)
    out = ops.paged_prefill_attention(q.view(rows, -1).to(cuda_dev), arena, 0, bt, sl, tiles, None, None, hq, hkv, scale)
    ops.core.check_status(cuda_dev)
    check_contributions(out.view(rows, hq, 128), q.double().to(cuda_dev), quantize64(k).to(cuda_dev),
                        quantize64(v).to(cuda_dev), torch.arange(n - rows + 1, n + 1), scale)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n", [(5, 400), (5, 1300), (400, 400)])  # few rows (whole; cut between CTAs), many
@pytest.mark.parametrize("case", ["mixed", "zero rows", "falling", "rising", "tiny", "huge", "never written"])
def test_scales_over_the_whole_range(cuda_dev, rows, n, case):
    """Rows of one call over all of e4m3's and the scale's range, in any order: each counts by its own value."""
    g = torch.Generator().manual_seed(24)
    hq, hkv, scale = 8, 2, 0.09
    arena, bt, _ = build([n], hq, hkv, 1, 0, g, cuda_dev, garbage=False)
    j = torch.arange(n)
    slots = bt[0].cpu().long()[j // PAGE] * PAGE + j % PAGE
    k, v = torch.randn(n, hkv, 128, generator=g), torch.randn(n, hkv, 128, generator=g)
    q = torch.randn(rows, hq, 128, generator=g)
    at = torch.arange(n).float()
    if case == "mixed":  # neighbours far apart; keys' large ones score low or high
        v *= torch.exp2(torch.randint(-124, 118, (n, hkv, 1), generator=g).float())
        k *= torch.exp2(torch.randint(-60, 6, (n, hkv, 1), generator=g).float())
    elif case == "zero rows":  # of K and of V, alone and over a whole tile of keys
        zk, zv = (torch.rand(n, hkv, 1, generator=g) < 0.3 for _ in range(2))
        zv[128:256] = True
        zk[256:384] = True
        k, v = torch.where(zk, 0.0, k), torch.where(zv, 0.0, v)
    elif case == "falling":
        v *= torch.exp2(110 - at * (220 / n))[:, None, None]
    elif case == "rising":
        v *= torch.exp2(-110 + at * (220 / n))[:, None, None]
    elif case == "tiny":
        v *= 2.0 ** -122
    elif case == "huge":
        v *= 2.0 ** 124
    k, v, q = k.to(BF), v.to(BF), q.to(BF)
    k64, v64 = quantize64(k), quantize64(v)
    if case == "never written":  # pages as they were allocated: zeros
        arena[:, 0] = 0
        keep = (j // PAGE) % 3 != 1
        k64[~keep], v64[~keep] = 0.0, 0.0
    else:
        keep = j >= 0
    ops.kv8_write(k[keep].view(-1, hkv * 128).to(cuda_dev), v[keep].view(-1, hkv * 128).to(cuda_dev),
                  slots[keep].to(cuda_dev), arena, 0)
    sl = torch.tensor([n], dtype=torch.int32, device=cuda_dev)
    tiles = ops.build_prefill_tiles([0, rows], [n - rows], device=cuda_dev)
    out = ops.paged_prefill_attention(q.view(rows, -1).to(cuda_dev), arena, 0, bt, sl, tiles, None, None, hq, hkv, scale)
    one = ops.paged_decode_attention(q[-1:].view(1, -1).to(cuda_dev), arena, 0, bt, sl, hq, hkv, scale)
    ops.core.check_status(cuda_dev)
    lim = torch.arange(n - rows + 1, n + 1)
    args = q.double().to(cuda_dev), k64.to(cuda_dev), v64.to(cuda_dev)
    check_contributions(out.view(rows, hq, 128), *args, lim, scale)
    check_contributions(one.view(1, hq, 128), args[0][-1:], *args[1:], lim[-1:], scale)


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv", [(8, 2), (3, 1)])
def test_wide_and_narrow_tiles_in_turn(cuda_dev, hq, hkv):
    """Long sequences whose tiles of keys change between far-apart and near scales, NaN rows among them: right, and
    bit for bit the same when calls follow one another on two streams."""
    g = torch.Generator().manual_seed(29)
    n, rows, scale = 2900, 640, 0.09
    arena, bt, _ = build([n], hq, hkv, 1, 0, g, cuda_dev)
    j = torch.arange(n)
    slots = bt[0].cpu().long()[j // PAGE] * PAGE + j % PAGE
    k, v = torch.randn(n, hkv, 128, generator=g), torch.randn(n, hkv, 128, generator=g)
    q = torch.randn(rows, hq, 128, generator=g)
    wide = torch.rand(-(-n // 64), 2, generator=g) < 0.4  # of K, of V, by 64 keys
    up = torch.exp2(torch.randint(-30, 1, (n, hkv, 2), generator=g).float())
    up = torch.where(wide[j // 64][:, None, :], up, torch.ones_like(up))
    k, v = (k * up[..., :1]).to(BF), (v * up[..., 1:]).to(BF)
    at = n - rows + 77  # seen by the rows from here on
    v[at, 0, 3] = float("nan")
    q = q.to(BF)
    ops.kv8_write(k.view(n, -1).to(cuda_dev), v.view(n, -1).to(cuda_dev), slots.to(cuda_dev), arena, 0)
    sl = torch.tensor([n], dtype=torch.int32, device=cuda_dev)
    tiles = ops.build_prefill_tiles([0, rows], [n - rows], device=cuda_dev)
    qd = q.view(rows, -1).to(cuda_dev)
    call = lambda: ops.paged_prefill_attention(qd, arena, 0, bt, sl, tiles, None, None, hq, hkv, scale)  # noqa: E731
    out = call()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    more = []
    for i in range(16):
        with torch.cuda.stream(streams[i % 2]):
            more.append(call())
    torch.cuda.synchronize()
    ops.core.check_status(cuda_dev)
    bits = out.view(torch.int16)
    assert all(torch.equal(x.view(torch.int16), bits) for x in more)
    out = out.view(rows, hq, 128)
    g0 = hq // hkv  # heads of KV head 0
    assert bool(torch.isnan(out[77:, :g0]).all()) and bool(torch.isfinite(out[:77].float()).all())
    pick = torch.cat([torch.arange(0, 77, 5), torch.arange(77, rows, 23)])
    v64 = quantize64(v).nan_to_num(nan=0.0)
    lim = torch.arange(n - rows + 1, n + 1)
    args = q.double().to(cuda_dev), quantize64(k).to(cuda_dev), v64.to(cuda_dev)
    before = pick[pick < 77]
    check_contributions(out[before], args[0][before], *args[1:], lim[before], scale)
    if hkv > 1:  # the NaN is KV head 0's alone
        check_contributions(out[pick][:, g0:], args[0][pick][:, g0:], args[1][:, 1:], args[2][:, 1:], lim[pick], scale)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [3, 150])  # both kernels
def test_scores_too_small_for_their_factor(cuda_dev, rows):
    """Queries of zeros beside keys near fp32's smallest, and a scale of 0: every seen key weighs the same."""
    g = torch.Generator().manual_seed(17)
    n, hq, hkv = 150, 8, 2
    arena, bt, _ = build([n], hq, hkv, 1, 0, g, cuda_dev)
    j = torch.arange(n, device=cuda_dev)
    slots = bt[0].long()[j // PAGE] * PAGE + j % PAGE
    k = (torch.randn(n, hkv * 128, generator=g) * 1e-36).to(BF).to(cuda_dev)
    v = torch.randn(n, hkv * 128, generator=g).to(BF).to(cuda_dev)
    ops.kv8_write(k, v, slots, arena, 0)
    sl = torch.tensor([n], dtype=torch.int32, device=cuda_dev)
    tiles = ops.build_prefill_tiles([0, rows], [n - rows], device=cuda_dev)
    cached = ops.kv8_read(arena, 0, slots)[1].double().view(n, hkv, 128)
    lim = torch.arange(n - rows + 1, n + 1, device=cuda_dev)
    want = cached.cumsum(0)[lim - 1] / lim[:, None, None]
    # the weights are 2^0 up to an exponential's error and fp16's rounding (2^-11), the output is a bf16 number
    tol = want.abs() * 2 ** -8 + 4 * 2 ** -11 * cached.abs().amax()
    for q, scale in ((torch.zeros(rows, hq * 128), 0.09), (torch.randn(rows, hq * 128, generator=g), 0.0)):
        out = ops.paged_prefill_attention(q.to(BF).to(cuda_dev), arena, 0, bt, sl, tiles, None, None, hq, hkv, scale)
        ops.core.check_status(cuda_dev)
        err = (out.double().view(rows, hkv, hq // hkv, 128) - want[:, :, None]).abs()
        assert bool((err <= tol[:, :, None]).all())
    for scale in (-0.1, float("nan"), float("inf")):
        with pytest.raises(RuntimeError, match="scale"):
            ops.paged_prefill_attention(q.to(BF).to(cuda_dev), arena, 0, bt, sl, tiles, None, None, hq, hkv, scale)
        with pytest.raises(RuntimeError, match="scale"):
            ops.paged_decode_attention(q[:1].to(BF).to(cuda_dev), arena, 0, bt, sl, hq, hkv, scale)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [2, 200])  # both kernels
def test_prefill_bad_tiles_are_reported_and_skipped(cuda_dev, rows):
    g = torch.Generator().manual_seed(14)
    arena, bt, _ = build([rows, 30], 8, 2, 1, 0, g, cuda_dev)
    n = rows + 2
    q = torch.randn(n, 1024, generator=g).to(BF).to(cuda_dev)
    sl = torch.tensor([rows, 30], dtype=torch.int32, device=cuda_dev)
    tiles = ops.build_prefill_tiles([0, rows, n], [0, 28], device=cuda_dev)
    args = (bt, sl)
    good = ops.paged_prefill_attention(q, arena, 0, *args, tiles, None, None, 8, 2, 0.1)
    ops.core.check_status(cuda_dev)
    for bad in ([2, 0, 1, 0], [-1, 0, 1, 0], [0, n, 1, 0], [0, -1, 1, 0], [0, n - 1, 2, 0], [0, 0, 129, 0],
                [0, 0, 2 ** 31 - 1, 0], [0, 0, 1, -1], [0, 0, 1, 2 ** 31 - 1]):
        t2 = torch.cat([tiles, torch.tensor([bad], dtype=torch.int32, device=cuda_dev)])
        out = ops.paged_prefill_attention(q, arena, 0, *args, t2, None, None, 8, 2, 0.1)
        with pytest.raises(ops.core.KernelError, match="out of bounds"):
            ops.core.check_status(cuda_dev)
        assert torch.equal(out, good), bad


def check_rows(out, q, cached, lens, new, hkv, scale):
    """Rows of `out` (packed prefill rows, the last `new` of each sequence) against 64-bit attention; what a row
    does not see counts neither for its result nor for its error."""
    dev, hq, at = out.device, q.shape[1] // 128, 0
    for s, (n, m) in enumerate(zip(lens, new)):
        k, v = (x.to(dev) for x in cached[s])
        lim = torch.arange(n - m + 1, n + 1, device=dev)
        o, w, size = attend64(q[at:at + m].double().view(m, hq, 128), k, v, lim, scale)
        top = v.abs().amax((1, 2)).cummax(0).values[lim - 1][:, None, None] if m else torch.zeros(0, 1, 1, device=dev)
        err = (out[at:at + m].double().view(m, hq, 128) - o).abs()
        tol = attention_tolerance(o, w, size, top)
        assert bool((err <= tol).all()), (s, float((err / tol).nan_to_num(nan=float("inf")).amax()))
        at += m


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [5, 80])  # whole segments, and segments that are cut
@pytest.mark.parametrize("lens,new", [([40, 30], [3, 2]), ([200, 30], [200, 30]), ([300, 5000], [300, 20])])
def test_padding_tiles_name_no_sequence(cuda_dev, cols, lens, new):
    """Tiles of no rows may hold anything else."""
    g = torch.Generator().manual_seed(22)
    arena, bt, cached = build(lens, 8, 2, 1, 0, g, cuda_dev, extra_cols=cols)
    starts = [0, new[0], sum(new)]
    q = torch.randn(starts[-1], 1024, generator=g).to(BF).to(cuda_dev)
    sl = torch.tensor(lens, dtype=torch.int32, device=cuda_dev)
    tiles = ops.build_prefill_tiles(starts, [a - b for a, b in zip(lens, new)], device=cuda_dev)
    odd = torch.tensor([[x, y, z, w] for x, y, w in ((-1, -1, -1), (2, 0, 0), (2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1),
                                                     (-2 ** 31, 5, 7), (10 ** 6, 0, 3)) for z in (0, -1, -2 ** 31)],
                       dtype=torch.int32, device=cuda_dev)
    for t2 in (torch.cat([tiles, odd]), torch.cat([odd, tiles])):
        out = ops.paged_prefill_attention(q, arena, 0, bt, sl, t2, None, None, 8, 2, 0.1)
        ops.core.check_status(cuda_dev)
        check_rows(out, q, cached, lens, new, 2, 0.1)


@pytest.mark.gpu
@pytest.mark.parametrize("maxb", [5, 80])
@pytest.mark.parametrize("n", [0, 3, 600])
def test_a_step_of_no_sequences(cuda_dev, maxb, n):
    """The tables of no sequences are padding alone; attention over them touches nothing."""
    i32 = dict(dtype=torch.int32, device=cuda_dev)
    t = ops.build_step_tables(torch.zeros(4, maxb, **i32), *(torch.zeros(0, **i32) for _ in range(3)), n, 3)
    arena = ops.kv8_arena(2, 1, 2, device=cuda_dev)
    q = torch.ones(n, 1024, dtype=BF, device=cuda_dev)
    out = torch.full_like(q, 4.0)
    ops.paged_prefill_attention(q, arena, 0, t.block_tables, t.seq_lens, t.tiles, t.query_start, t.positions, 8, 2, 0.1,
                                out=out)
    ops.paged_decode_attention(q, arena, 0, t.block_tables, t.seq_lens, 8, 2, 0.1, out=out)
    ops.core.check_status(cuda_dev)
    assert bool((out == 4.0).all())
    if n:  # a tile with rows names a sequence that is not there
        t.tiles[0, 2] = 1
        ops.paged_prefill_attention(q, arena, 0, t.block_tables, t.seq_lens, t.tiles, None, None, 8, 2, 0.1, out=out)
        with pytest.raises(ops.core.KernelError, match="out of bounds"):
            ops.core.check_status(cuda_dev)
        assert bool((out == 4.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("n", [304, 1600])  # whole segments, and segments that may be cut
@pytest.mark.parametrize("new", [[1, 1], [5, 2], [140, 130], [300, 20]])  # decode, few rows, many, both
def test_lengths_past_the_block_table_are_reported(cuda_dev, new, n):
    """What the table holds is attended to, the other sequence is as ever, and the caller hears of it."""
    g = torch.Generator().manual_seed(25)
    hq, hkv = 8, 2
    arena, bt, cached = build([n, 150], hq, hkv, 1, 0, g, cuda_dev)
    cap = bt.shape[1] * PAGE
    assert cap == n
    q = torch.randn(sum(new), hq * 128, generator=g).to(BF).to(cuda_dev)
    tiles = ops.build_prefill_tiles([0, new[0], sum(new)], [n - new[0], 150 - new[1]], device=cuda_dev)

    def call(lens):
        sl = torch.tensor(lens, dtype=torch.int32, device=cuda_dev)
        if new == [1, 1]:
            return ops.paged_decode_attention(q, arena, 0, bt, sl, hq, hkv, 0.1)
        return ops.paged_prefill_attention(q, arena, 0, bt, sl, tiles, None, None, hq, hkv, 0.1)

    good = call([cap, 150])
    ops.core.check_status(cuda_dev)
    check_rows(good, q, cached, [n, 150], new, hkv, 0.1)
    for bad in (cap + 1, 2 ** 31 - 1):
        out = call([bad, 150])
        with pytest.raises(ops.core.KernelError, match="out of bounds"):
            ops.core.check_status(cuda_dev)
        assert torch.equal(out, good)
    for bad in (-1, -2 ** 31):
        out = call([cap, bad])
        with pytest.raises(ops.core.KernelError, match="out of bounds"):
            ops.core.check_status(cuda_dev)
        assert not out[new[0]:].any() and torch.equal(out[:new[0]], call([cap, 0])[:new[0]])
        ops.core.check_status(cuda_dev)


@pytest.mark.gpu
def test_calls_that_are_refused_for_their_size_or_memory(cuda_dev):
    arena = ops.kv8_arena(1, 1, 1, device=cuda_dev)
    sl = torch.ones(1, dtype=torch.int32, device=cuda_dev)
    q = torch.zeros(1, 1024, dtype=BF, device=cuda_dev)
    tiles = torch.tensor([[0, 0, 1, 0]], dtype=torch.int32, device=cuda_dev)
    wide = torch.zeros(1, 600_000, dtype=torch.int32, device=cuda_dev)  # 32 such tiles could pass 32 bits of pages
    with pytest.raises(RuntimeError):
        ops.paged_prefill_attention(q, arena, 0, wide, sl, tiles, None, None, 8, 1, 0.1)
    ops.paged_prefill_attention(q, arena, 0, wide[:, :500_000], sl, tiles, None, None, 8, 1, 0.1)
    ops.paged_decode_attention(q, arena, 0, wide, sl, 8, 1, 0.1)
    for f in (lambda: ops.paged_prefill_attention(q, arena, 0, wide[:, :4], sl, tiles, None, None, 8, 1, 0.1, out=q),
              lambda: ops.paged_decode_attention(q, arena, 0, wide[:, :4], sl, 8, 1, 0.1, out=q)):
        with pytest.raises(RuntimeError, match="out must not be q"):
            f()
    ops.core.check_status(cuda_dev)
    empty = ops.kv8_arena(2, 1, 0, device=cuda_dev)  # no heads
    for n in (1, 3):
        none, at = torch.zeros(n, 0, dtype=BF, device=cuda_dev), torch.arange(n, device=cuda_dev)
        with pytest.raises(RuntimeError):
            ops.kv8_write(none, none, at, empty, 0)
        with pytest.raises(RuntimeError):
            ops.kv8_read(empty, 0, at)


@pytest.mark.gpu
def test_out_beside_q_but_not_over_it(cuda_dev):
    """q and out in one buffer: side by side they are as good as apart, over each other they are refused."""
    g = torch.Generator().manual_seed(27)
    lens, hq, hkv = [40, 300, 7], 8, 2
    arena, bt, cached = build(lens, hq, hkv, 1, 0, g, cuda_dev)
    sl = torch.tensor(lens, dtype=torch.int32, device=cuda_dev)
    w = hq * 128
    buf = torch.randn(8, 2 * w, generator=g).to(BF).to(cuda_dev)
    flat, keep = buf.view(-1), buf.clone()
    tiles = ops.build_prefill_tiles([0, 1, 2, 3], [n - 1 for n in lens], device=cuda_dev)

    def calls(q, out):
        yield lambda: ops.paged_decode_attention(q, arena, 0, bt, sl, hq, hkv, 0.1, out=out)
        yield lambda: ops.paged_prefill_attention(q, arena, 0, bt, sl, tiles, None, None, hq, hkv, 0.1, out=out)

    q = buf[:3, :w]
    for out in (buf[:3, w:], buf[3:6, :w], buf[4:7, w:], flat[7 * w:10 * w].view(3, w)):
        for call in calls(q, out):
            check_rows(call(), q, cached, lens, [1, 1, 1], hkv, 0.1)
            buf.copy_(keep)
    for out in (buf[1:4, :w], buf[2:5, :w], buf[:3, 8:8 + w], buf[:3, w - 8:2 * w - 8], flat[8:8 + 3 * w].view(3, w),
                flat[w:4 * w].view(3, w), flat[:w].expand(3, w), flat[6 * w:7 * w].expand(3, w)):
        for call in calls(q, out):
            with pytest.raises(RuntimeError, match="out must not|must not overlap"):
                call()
    assert torch.equal(buf, keep)
    ops.core.check_status(cuda_dev)


@pytest.mark.gpu
def test_an_arena_of_no_pages(cuda_dev):
    """Attention refuses it (there is no page to read in place of one that is not there); rows are reported."""
    arena = ops.kv8_arena(0, 1, 1, device=cuda_dev)
    i32 = dict(dtype=torch.int32, device=cuda_dev)
    q, bt, sl = torch.zeros(1, 128, dtype=BF, device=cuda_dev), torch.zeros(1, 2, **i32), torch.ones(1, **i32)
    with pytest.raises(RuntimeError, match="no pages"):
        ops.paged_decode_attention(q, arena, 0, bt, sl, 1, 1, 0.1)
    with pytest.raises(RuntimeError, match="no pages"):
        ops.paged_prefill_attention(q, arena, 0, bt, sl, torch.tensor([[0, 0, 1, 0]], **i32), None, None, 1, 1, 0.1)
    ops.core.check_status(cuda_dev)
    at = torch.zeros(1, dtype=torch.int64, device=cuda_dev)
    for call in (lambda: ops.kv8_write(q, q, at, arena, 0), lambda: ops.kv8_read(arena, 0, at)):
        call()
        with pytest.raises(ops.core.KernelError, match="out of bounds"):
            ops.core.check_status(cuda_dev)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [3, 200])  # both kernels
def test_one_query_row_broadcast_to_all(cuda_dev, rows):
    """q may be a view whose rows are one row."""
    g = torch.Generator().manual_seed(28)
    arena, bt, cached = build([250], 8, 2, 1, 0, g, cuda_dev)
    q = torch.randn(1, 1024, generator=g).to(BF).to(cuda_dev).expand(rows, -1)
    sl = torch.tensor([250], dtype=torch.int32, device=cuda_dev)
    tiles = ops.build_prefill_tiles([0, rows], [250 - rows], device=cuda_dev)
    out = ops.paged_prefill_attention(q, arena, 0, bt, sl, tiles, None, None, 8, 2, 0.1)
    check_rows(out, q, cached, [250], [rows], 2, 0.1)
    out = ops.paged_decode_attention(q[:3], arena, 0, bt.expand(3, -1), sl.expand(3).contiguous(), 8, 2, 0.1)
    for i in range(3):
        check_rows(out[i:i + 1], q[:1], cached, [250], [1], 2, 0.1)
    ops.core.check_status(cuda_dev)


@pytest.mark.gpu
def test_decode_more_sequences_than_a_grid_axis(cuda_dev):
    n = 70_000
    g = torch.Generator().manual_seed(15)
    arena, bt, _ = build([16], 4, 1, 1, 0, g, cuda_dev)
    q = torch.randn(16, 512, generator=g).to(BF).to(cuda_dev)
    lens = torch.arange(1, 17, dtype=torch.int32, device=cuda_dev)
    few = ops.paged_decode_attention(q, arena, 0, bt.expand(16, -1), lens, 4, 1, 0.1)
    pick = torch.randint(0, 16, (n,), generator=g).to(cuda_dev)
    many = ops.paged_decode_attention(q[pick], arena, 0, bt.expand(n, -1), lens[pick], 4, 1, 0.1)
    ops.core.check_status(cuda_dev)
    assert torch.equal(many, few[pick])


@pytest.mark.gpu
@pytest.mark.parametrize("lens,new,hq,hkv", [([256], [256], 2, 1), ([1500], [640], 8, 2), ([3000, 40], [640, 20], 8, 2),
                                             ([700] * 6, [129] * 6, 10, 2), ([2500] * 3, [3, 9, 5], 8, 2),
                                             ([300, 5000], [300, 20], 16, 2), ([40, 900, 900], [20, 640, 513], 16, 2)])
def test_prefill_repeats_bit_for_bit(cuda_dev, lens, new, hq, hkv):
    """Back to back, without a wait between the calls: a hand-off that is early by one phase shows here."""
    g = torch.Generator().manual_seed(16)
    arena, bt, _ = build(lens, hq, hkv, 1, 0, g, cuda_dev)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    q = (torch.randn(starts[-1], hq * 128, generator=g) * 1.5).to(BF).to(cuda_dev)
    sl = torch.tensor(lens, dtype=torch.int32, device=cuda_dev)
    tiles = ops.build_prefill_tiles(starts, [n - m for n, m in zip(lens, new)], device=cuda_dev)
    outs = [ops.paged_prefill_attention(q, arena, 0, bt, sl, tiles, None, None, hq, hkv, 0.09) for _ in range(16)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for i in range(12):  # two at once
        with torch.cuda.stream(streams[i % 2]):
            outs.append(ops.paged_prefill_attention(q, arena, 0, bt, sl, tiles, None, None, hq, hkv, 0.09))
    torch.cuda.synchronize()
    ops.core.check_status(cuda_dev)
    for o in outs[1:]:
        assert torch.equal(o, outs[0])


# ------------------------------------------------------------------ streams, graphs, sizes
@pytest.mark.gpu
def test_two_streams_and_a_replayed_graph(cuda_dev):
    """Calls on two streams at once and a captured call replayed with other lengths give what single
    calls give."""
    g = torch.Generator().manual_seed(14)
    lens, hq, hkv = [700, 90, 1500, 1], 8, 2
    arena, bt, _ = build(lens, hq, hkv, 1, 0, g, cuda_dev)
    sl = torch.tensor(lens, dtype=torch.int32, device=cuda_dev)
    qs = [torch.randn(4, 1024, generator=g).to(BF).to(cuda_dev) for _ in range(4)]
    want = [ops.paged_decode_attention(q, arena, 0, bt, sl, hq, hkv, 0.1) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[] for _ in qs]
    for _ in range(20):
        for i, q in enumerate(qs):
            with torch.cuda.stream(streams[i % 2]):
                got[i].append(ops.paged_decode_attention(q, arena, 0, bt, sl, hq, hkv, 0.1))
    torch.cuda.synchronize()
    for i in range(4):
        assert all(torch.equal(x, want[i]) for x in got[i])
    q, lens_buf = qs[0].clone(), sl.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.paged_decode_attention(q, arena, 0, bt, lens_buf, hq, hkv, 0.1)
    graph.replay()
    assert torch.equal(out, want[0])
    q.copy_(qs[1])
    lens_buf.copy_(torch.tensor([3, 0, 1499, 1], device=cuda_dev))
    graph.replay()
    assert torch.equal(out, ops.paged_decode_attention(qs[1], arena, 0, bt, lens_buf, hq, hkv, 0.1))
    ops.core.check_status(cuda_dev)


@pytest.mark.gpu
@pytest.mark.parametrize("lens,new,hq,hkv", [([700, 90, 1500], None, 8, 2), ([200, 90, 16], None, 8, 2),
                                             ([700, 90, 1500], [5, 2, 3], 8, 2), ([700, 90, 5000], [300, 20, 30], 16, 2),
                                             ([400, 90, 250], [300, 20, 30], 16, 2)])
@pytest.mark.parametrize("graph", [False, True])
def test_attention_right_behind_its_writers(cuda_dev, lens, new, hq, hkv, graph):
    """Keys, queries, lengths and pages written by the kernels just before, on this stream and on one that
    joins it, without a wait between the rounds; the outputs and the buffers are used again at once."""
    g = torch.Generator().manual_seed(18)
    rounds, total = 6, sum(lens)
    arena, bt, _ = build(lens, hq, hkv, 1, 0, g, cuda_dev)
    slots = torch.cat([bt[i].long()[torch.arange(n, device=cuda_dev) // PAGE] * PAGE + torch.arange(n, device=cuda_dev) % PAGE
                       for i, n in enumerate(lens)])
    starts = [0]
    for n in new or [1] * len(lens):
        starts.append(starts[-1] + n)
    k, v, q = (torch.randn(rounds, n, w * 128, generator=g).to(BF).to(cuda_dev)
               for n, w in ((total, hkv), (total, hkv), (starts[-1], hq)))
    full = torch.tensor(lens, dtype=torch.int32, device=cuda_dev)
    sls = [full - (i % 2) * 3 for i in range(rounds)]
    tiles = ops.build_prefill_tiles(starts, [a - b for a, b in zip(lens, new or lens)], device=cuda_dev)
    qb, slb, btb, tb = torch.zeros_like(q[0]), torch.zeros_like(full), torch.zeros_like(bt), torch.zeros_like(tiles)
    side = torch.cuda.Stream()

    def attend():
        if new is None:
            return ops.paged_decode_attention(qb, arena, 0, btb, slb, hq, hkv, 0.1)
        return ops.paged_prefill_attention(qb, arena, 0, btb, slb, tb, None, None, hq, hkv, 0.1)

    def one(i, split):
        main = torch.cuda.current_stream()
        if split:
            side.wait_stream(main)
        with torch.cuda.stream(side if split else main):
            ops.kv8_write(k[i], v[i], slots, arena, 0)
        tb.copy_(tiles)
        btb.copy_(bt)
        qb.copy_(q[i])
        if split and i % 2:
            main.wait_stream(side)
        slb.copy_(sls[i])
        if split:
            main.wait_stream(side)
        out = attend()
        qb.zero_()
        slb.zero_()
        return out

    want = []
    for i in range(rounds):
        ops.kv8_write(k[i], v[i], slots, arena, 0)
        for b, x in ((tb, tiles), (btb, bt), (qb, q[i]), (slb, sls[i])):
            b.copy_(x)
        torch.cuda.synchronize()
        want.append(attend())
        torch.cuda.synchronize()
    if graph:
        run = torch.cuda.CUDAGraph()
        with torch.cuda.graph(run):
            got = [one(i, split) for split in (False, True) for i in range(rounds)]
        for _ in range(3):
            run.replay()
    else:
        got = [one(i, split) for split in (False, True) for i in range(rounds)]
    torch.cuda.synchronize()
    ops.core.check_status(cuda_dev)
    for i, o in enumerate(got):
        assert torch.equal(o, want[i % rounds]), i


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [0, 100])  # block tables of few pages and of many
def test_launches_are_counted(cuda_dev, cols):
    """The count that the benchmarks report grows by the kernels that a call really launches (those in its graph)."""
    rt = pytest.importorskip("cuda.bindings.runtime")
    g = torch.Generator().manual_seed(26)
    lens = [300, 900, 40]
    arena, bt, _ = build(lens, 8, 2, 1, 0, g, cuda_dev, extra_cols=cols)
    sl = torch.tensor(lens, dtype=torch.int32, device=cuda_dev)
    q = torch.randn(700, 1024, generator=g).to(BF).to(cuda_dev)
    rows = torch.randn(5, 256, generator=g).to(BF).to(cuda_dev)
    slots, at = torch.arange(5, device=cuda_dev), torch.arange(3, dtype=torch.int32, device=cuda_dev)
    zero, out = torch.zeros_like(at), torch.empty_like(q)

    def prefill(new):
        starts = [sum(new[:i]) for i in range(4)]
        tiles = ops.build_prefill_tiles(starts, [a - b for a, b in zip(lens, new)], device=cuda_dev)
        return lambda: ops.paged_prefill_attention(q[:starts[-1]], arena, 0, bt, sl, tiles, None, None, 8, 2, 0.1, out=out)

    calls = [prefill(x) for x in ([5, 3, 1], [20, 640, 30], [300, 300, 40], [0, 0, 0])]
    calls += [lambda: ops.paged_decode_attention(q[:3], arena, 0, bt, sl, 8, 2, 0.1, out=out),
              lambda: ops.paged_decode_attention(q[:0], arena, 0, bt, sl[:0], 8, 2, 0.1, out=out),
              lambda: ops.kv8_write(rows, rows, slots, arena, 0),
              lambda: ops.kv8_write(rows[:0], rows[:0], slots[:0], arena, 0), lambda: ops.kv8_read(arena, 0, slots),
              lambda: ops.kv8_read(arena, 0, slots[:0]),
              lambda: ops.build_step_tables(bt, at, zero, sl, 2000, 32)]
    counts = []
    for call in calls:
        call()  # (what a first call sets up is none of its launches)
        graph = torch.cuda.CUDAGraph(keep_graph=True)
        with torch.cuda.graph(graph):
            before = ops.core.LAUNCHES[0]
            call()
            counted = ops.core.LAUNCHES[0] - before
        raw = rt.cudaGraph_t(graph.raw_cuda_graph())
        err, _, n = rt.cudaGraphGetNodes(raw)
        assert int(err) == 0
        err, nodes, n = rt.cudaGraphGetNodes(raw, n) if n else (0, [], 0)
        kinds = [rt.cudaGraphNodeGetType(x)[1] for x in nodes[:n]]
        launched = sum(k == rt.cudaGraphNodeType.cudaGraphNodeTypeKernel for k in kinds)
        counts.append((counted, launched))
    assert all(a == b for a, b in counts), counts
    assert max(b for _, b in counts) == (3 if cols else 1)
    ops.core.check_status(cuda_dev)


@pytest.mark.gpu
def test_offsets_past_32_bits(cuda_dev):
    """Pages beyond 4 GiB of the arena are written, read and attended to."""
    blocks = (1 << 32) // (4128 * 2) + 64
    arena = torch.zeros(blocks, 1, 2, 2, 2064, dtype=torch.uint8, device=cuda_dev)
    g = torch.Generator().manual_seed(15)
    n, hq = 50, 8
    k, v = (rows(n, 2, 128, g).to(BF).reshape(n, -1).to(cuda_dev) for _ in range(2))
    small = ops.kv8_arena(4, 1, 2, device=cuda_dev)
    j = torch.arange(n, device=cuda_dev)
    far = (blocks - 4) * PAGE + j
    ops.kv8_write(k, v, far, arena, 0)
    ops.kv8_write(k, v, j, small, 0)
    assert torch.equal(arena[blocks - 4:], small)
    assert torch.equal(ops.kv8_read(arena, 0, far)[0], ops.kv8_read(small, 0, j)[0])
    q = torch.randn(n, hq * 128, generator=g).to(BF).to(cuda_dev)
    sl = torch.tensor([n], dtype=torch.int32, device=cuda_dev)
    near = torch.arange(4, dtype=torch.int32, device=cuda_dev)[None]
    args = (sl, hq, 2, 0.1)
    assert torch.equal(ops.paged_decode_attention(q[:1], arena, 0, near + (blocks - 4), *args),
                       ops.paged_decode_attention(q[:1], small, 0, near, *args))
    tiles = ops.build_prefill_tiles([0, n], [0], device=cuda_dev)
    a = ops.paged_prefill_attention(q, arena, 0, near + (blocks - 4), sl, tiles, None, None, hq, 2, 0.1)
    b = ops.paged_prefill_attention(q, small, 0, near, sl, tiles, None, None, hq, 2, 0.1)
    assert torch.equal(a, b)
    ops.core.check_status(cuda_dev)


# ------------------------------------------------------------------ QKV projection and engine
@pytest.mark.gpu
@pytest.mark.parametrize("t,norm", [(1, False), (70, False), (70, True), (600, False)])  # 600: two-SM kernel
def test_linear_qkv_writes_the_8bit_arena(cuda_dev, t, norm):
    """Cached rows are within a quantisation step of the fp32 rows, q is what the bf16 arena's call gives."""
    g = torch.Generator(device=cuda_dev).manual_seed(21)
    hid, hq, hkv = 512, 4, 2
    a = torch.randn(t, hid, device=cuda_dev, generator=g).to(BF)
    w = (torch.randn((hq + 2 * hkv) * 128, hid, device=cuda_dev, generator=g) / 20).to(BF)
    cs = ref.rope_cache(4096, 500000.0, device=cuda_dev)
    pos = torch.randint(0, 4000, (t,), device=cuda_dev, dtype=torch.int32, generator=g)
    slots = torch.randperm(64 * 16, device=cuda_dev, generator=g)[:t]
    if t > 5:
        slots[5] = -1
    nw = [(1 + 0.1 * torch.randn(128, device=cuda_dev, generator=g)).to(BF) for _ in range(2)] if norm else [None] * 2
    arena = ops.kv8_arena(64, 3, hkv, device=cuda_dev)
    peer = ops.kv8_arena(64, 3, hkv, device=cuda_dev)
    dense = torch.zeros(64, 3, 2, hkv, 16, 128, dtype=BF, device=cuda_dev)
    qa, qb = torch.empty(t, hq * 128, dtype=BF, device=cuda_dev), torch.empty(t, hq * 128, dtype=BF, device=cuda_dev)
    peer_slots = torch.where(slots >= 0, (slots + 16) % 1024, slots)
    ops.linear_qkv(a, w, qa, cs, pos, slots, arena, 1, hq, hkv, peer, peer_slots, *nw)
    ops.linear_qkv(a, w, qb, cs, pos, slots, dense, 1, hq, hkv, None, None, *nw)
    ops.core.check_status(cuda_dev)
    assert torch.equal(qa, qb)
    assert not arena[:, 0].any() and not arena[:, 2].any()
    acc = a.double() @ w.double().t()
    k, v = acc[:, hq * 128:(hq + hkv) * 128].view(t, hkv, 128), acc[:, (hq + hkv) * 128:].view(t, hkv, 128)
    if norm:
        k = k * torch.rsqrt(k.pow(2).mean(-1, keepdim=True) + 1e-6) * nw[1].double()
    k = ref.apply_rope(k, pos, cs.double())
    keep = slots >= 0
    for side, got in zip((k, v), ops.kv8_read(arena, 1, slots)):
        got, want = got.view(t, hkv, 128).double()[keep], side[keep]
        top = want.abs().amax(-1, keepdim=True)
        # half a step of e4m3: 2^-4 of the value, at least half its smallest, 2^-10 2^e with 2^e <= top / 224; the
        # fp32 sums of 512 products move the value by less than 2^-12 of the row's largest and may move it over a step
        assert bool(((got - want).abs() <= 2.0 ** -4 * want.abs() + 2.0 ** -10 * top / 224 + 2.0 ** -12 * top).all())
    assert not ops.kv8_read(arena, 1, slots)[0][~keep].any()
    for x, y in zip(ops.kv8_read(arena, 1, slots), ops.kv8_read(peer, 1, peer_slots)):
        assert torch.equal(x, y)
    with pytest.raises(RuntimeError, match="another type"):
        ops.linear_qkv(a, w, qa, cs, pos, slots, arena, 1, hq, hkv, dense, slots)
    with pytest.raises(RuntimeError, match="layer"):
        ops.linear_qkv(a, w, qa, cs, pos, slots, arena, 3, hq, hkv)
    far = slots.clone()
    far[0] = 64 * 16
    ops.linear_qkv(a, w, qa, cs, pos, far, arena, 1, hq, hkv)
    with pytest.raises(ops.core.KernelError, match="out of bounds"):
        ops.core.check_status(cuda_dev)


@pytest.mark.gpu
def test_linear_qkv_refuses_a_peer_arena_of_other_heads(cuda_dev):
    """(its rows would land in the next layer, or past the arena's end)"""
    a = torch.zeros(3, 256, dtype=BF, device=cuda_dev)
    w = torch.zeros(8 * 128, 256, dtype=BF, device=cuda_dev)
    q = torch.empty(3, 512, dtype=BF, device=cuda_dev)
    pos, slots = torch.zeros(3, dtype=torch.int32, device=cuda_dev), torch.arange(3, device=cuda_dev)
    cs = ref.rope_cache(16, 10000.0, device=cuda_dev)
    arena = ops.kv8_arena(1, 1, 2, device=cuda_dev)
    for peer, at in ((ops.kv8_arena(1, 1, 1, device=cuda_dev), slots), (ops.kv8_arena(1, 1, 4, device=cuda_dev), slots),
                     (ops.kv8_arena(1, 1, 2, device=cuda_dev), slots[:2]), (arena, slots.int())):
        with pytest.raises(RuntimeError):
            ops.linear_qkv(a, w, q, cs, pos, slots, arena, 0, 4, 2, peer, at)
    ops.linear_qkv(a, w, q, cs, pos, slots, arena, 0, 4, 2, ops.kv8_arena(1, 1, 2, device=cuda_dev), slots)
    ops.core.check_status(cuda_dev)


def _engine(device, model, **kw):
    from lake_b200.engine.llm_engine import LLMEngine

    return LLMEngine(model, device=device, max_running=8, max_batched_tokens=256, max_model_len=512, num_blocks=128, **kw)


def _prompts(n, vocab, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, vocab, (x,), generator=g).tolist() for x in n]


def test_engine_8bit_kv_cpu():
    """The CPU engine with an 8-bit cache: chunked prefill, decode and a reused prefix give what one
    prefill of the same tokens gives, since a row's bytes do not depend on how its page was filled."""
    prompts = _prompts([5, 40, 33, 100], 1024)
    eng = _engine("cpu", "tiny", kv_dtype="fp8")
    assert eng.arena.dtype == torch.uint8 and eng.arena.shape == (128, 2, 2, 2, 16 * 64 + 16)
    out = eng.generate(prompts, max_new_tokens=6)
    chunked = _engine("cpu", "tiny", kv_dtype="fp8", long_prefill_threshold=16)
    assert chunked.generate(prompts, max_new_tokens=6) == out
    assert eng.generate([prompts[3]], max_new_tokens=6) == [out[3]] and eng.pool.stats["hits"] > 0
    from lake_b200.engine.llm_engine import page_bytes

    assert page_bytes(eng.cfg, 16, kv8=True) == eng.arena[0].numel()


def test_engine_8bit_kv_refusals():
    for bad in (dict(kv_dtype="int4"), dict(kv_dtype="fp8", block_size=32), dict(kv_dtype="fp8", model_impl="library")):
        with pytest.raises(ValueError):
            _engine("cpu", "tiny", **bad)


def test_worker_config_takes_kv_dtype(monkeypatch):
    from lake_b200.runtime.config import RoleConfig
    from lake_b200.runtime.worker_engine import build_engine

    monkeypatch.setenv("LAKE_KV_DTYPE", "FP8")
    cfg = RoleConfig.from_env()
    cfg.model_backend, cfg.num_blocks, cfg.max_running_reqs, cfg.max_model_length = "mock", 64, 4, 256
    assert cfg.kv_dtype == "fp8" and build_engine(cfg).arena.dtype == torch.uint8


@pytest.mark.gpu
@pytest.mark.parametrize("model", ["tiny-gpu", "qwen"])
def test_engine_8bit_kv_gpu(cuda_dev, model):
    """The engine's steps over the 8-bit cache (mixed steps, graph decode, prefix reuse, drafts) against the
    model run by the CPU oracle's ops on the same weights and the same cached values: logits of every
    position agree within bf16 activations' rounding, and tokens where the oracle's are clear."""
    over = {} if model == "tiny-gpu" else dict(qk_norm=True, n_q_heads=8, n_kv_heads=1)
    prompts = _prompts([7, 130, 64, 200], 2048, 3)
    eng = _engine(cuda_dev, "tiny-gpu", kv_dtype="fp8", model_overrides=over)
    out = eng.generate(prompts, max_new_tokens=12)
    eager = _engine(cuda_dev, "tiny-gpu", kv_dtype="fp8", model_overrides=over, use_cuda_graphs=False,
                    long_prefill_threshold=32)
    out2 = eager.generate(prompts, max_new_tokens=12)
    ops.core.check_status(cuda_dev)
    cpu = _engine("cpu", "tiny-gpu", kv_dtype="fp8", model_overrides=over)
    for k, w in eng.model.w.items():
        cpu.model.w[k].copy_(w.float().cpu())
    # teacher-forced logits of the oracle for prompt + output: the engine's token is within the rounding of the
    # largest logit (bf16 activations over two layers: 2^-8 a rounding, under 32 of them, of logits ~ |h| |w|)
    for p, o in zip(prompts, out):
        lg = _logits(cpu, p + o[:-1])[len(p) - 1:]
        top = lg.amax(-1)
        got = lg[torch.arange(len(o)), torch.tensor(o)]
        assert bool((top - got <= 32 * 2.0 ** -8 * lg.std(-1)).all())
    same_first = sum(a[0] == b[0] for a, b in zip(out, out2))
    assert same_first >= 3 and all(len(o) == 12 for o in out2)
    assert eng.generate([prompts[3]], max_new_tokens=3)[0][0] == out[3][0] and eng.pool.stats["hits"] > 0


def _logits(eng, tokens):
    from lake_b200.models.llama import ForwardBatch

    t = len(tokens)
    blocks = eng.reserve_blocks(t)
    pos = torch.arange(t, dtype=torch.int32)
    bt = torch.tensor([blocks], dtype=torch.int32)
    b = ForwardBatch(input_ids=torch.tensor(tokens, dtype=torch.int32), positions=pos,
                     slots=bt[0].long()[pos.long() // 16] * 16 + pos.long() % 16, block_tables=bt,
                     seq_lens=torch.tensor([t], dtype=torch.int32), n_decode=0,
                     prefill_tiles=ops.build_prefill_tiles([0, t], [0]),
                     query_start=torch.tensor([0, t], dtype=torch.int32), sample_rows=pos.long(), want_logits=True)
    ws = eng.model.new_workspace(t, t, 1)
    lg = eng.model.forward(b, eng.arena, ws)
    eng.release_blocks(blocks)
    return lg


@pytest.mark.gpu
def test_one_step_from_the_tables_on(cuda_dev):
    """A mixed step as they are used together: tables from lengths, rows written, decode rows and prompt
    chunks attended, against 64-bit attention over what the cache holds."""
    g = torch.Generator().manual_seed(31)
    hq, hkv, nd = 8, 2, 3
    ctx = [40, 0, 333, 100, 0, 7]
    new = [1, 1, 1, 70, 140, 2]
    lens = [a + b for a, b in zip(ctx, new)]
    pages = torch.randperm(128, generator=g)[:8 * 16].view(8, 16).to(torch.int32)
    pages = torch.cat([pages, torch.full((8, 9), -1, dtype=torch.int32)], 1)
    pages[2, 16:22] = torch.arange(128, 134)
    rows_of = torch.tensor([4, 0, 2, 5, 1, 7], dtype=torch.int32)
    dev = [x.to(cuda_dev) for x in (pages, rows_of, torch.tensor(ctx, dtype=torch.int32), torch.tensor(new, dtype=torch.int32))]
    arena = torch.randint(0, 256, (134, 2, hkv, 2, 2064), generator=g, dtype=torch.uint8).to(cuda_dev)
    # what was cached before the step
    old = ops.build_step_tables(dev[0], dev[1], torch.zeros_like(dev[2]), dev[2], sum(ctx), 8)
    k, v = (torch.randn(sum(ctx), hkv * 128, generator=g).to(BF).to(cuda_dev) for _ in range(2))
    ops.kv8_write(k, v, old.slots, arena, 1)
    t = ops.build_step_tables(*dev, sum(new) + 5, 8, n_decode=nd)
    qkv = torch.randn(sum(new) + 5, (hq + 2 * hkv) * 128, generator=g).to(BF).to(cuda_dev)
    q, kn, vn = qkv[:, :hq * 128], qkv[:, hq * 128:(hq + hkv) * 128], qkv[:, (hq + hkv) * 128:]
    ops.kv8_write(kn, vn, t.slots, arena, 1)
    out = torch.full((sum(new) + 5, hq * 128), 9.0, dtype=BF, device=cuda_dev)
    ops.paged_decode_attention(q[:nd], arena, 1, t.block_tables[:nd], t.seq_lens[:nd], hq, hkv, 0.09, out=out[:nd])
    ops.paged_prefill_attention(q, arena, 1, t.block_tables, t.seq_lens, t.tiles, t.query_start, t.positions, hq, hkv,
                                0.09, out=out)
    ops.core.check_status(cuda_dev)
    assert bool((out[sum(new):] == 9.0).all())
    starts, o0 = t.query_start.tolist(), 0
    for s, n in enumerate(lens):
        j = torch.arange(n)
        slots = pages[rows_of[s]].long()[j // PAGE] * PAGE + j % PAGE
        kk, vv = (x.view(n, hkv, 128).double() for x in ops.kv8_read(arena, 1, slots.to(cuda_dev)))
        a, b = starts[s], starts[s + 1]
        lim = torch.arange(ctx[s], n, device=cuda_dev) + 1
        o, w, size = attend64(q[a:b].double().view(b - a, hq, 128), kk, vv, lim, 0.09)
        err = (out[a:b].double().view(b - a, hq, 128) - o).abs()
        assert bool((err <= attention_tolerance(o, w, size, vv.abs().amax())).all()), s
