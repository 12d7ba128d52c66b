"""Step tables from request lengths: the kernel against the plain loops, and both against what the
engine packs on the host."""
import pytest
import torch

from lake_b200 import ops


def make(decode, prompts, ctx_hi, maxb, seed, rows=None):
    g = torch.Generator().manual_seed(seed)
    n = decode + len(prompts)
    new = torch.tensor([1] * decode + prompts, dtype=torch.int32)
    ctx = torch.randint(0, ctx_hi + 1, (n,), generator=g, dtype=torch.int32)
    r = rows or n + 3
    pages = torch.randint(0, 1 << 24, (r, maxb), generator=g, dtype=torch.int32)
    order = torch.randperm(r, generator=g)[:n].to(torch.int32)
    return pages, order, ctx, new


CASES = [(1, [], 0, 1), (0, [1], 0, 4), (0, [128, 129, 127], 100, 40), (3, [0, 300, 0, 1], 500, 80),
         (256, [], 2304, 160), (250, [1400, 7, 900, 513], 4000, 400), (700, [33], 50, 16), (0, [0, 0], 9, 3), (0, [], 0, 2)]


@pytest.mark.parametrize("decode,prompts,ctx_hi,maxb", CASES)
def test_tables_cpu(decode, prompts, ctx_hi, maxb):
    pages, rows, ctx, new = make(decode, prompts, ctx_hi, maxb, 1)
    total = int(new.sum())
    t = ops.build_step_tables(pages, rows, ctx, new, total + 3, 40, n_decode=decode)
    n = rows.numel()
    assert t.counts.tolist()[0] == total and t.seq_lens.tolist() == (ctx + new).tolist()
    starts = t.query_start.tolist()
    want = ops.build_prefill_tiles(starts, ctx.tolist())
    want = want[want[:, 0] >= decode]
    assert torch.equal(t.tiles[: want.shape[0]], want) and not t.tiles[want.shape[0]:].any()
    assert t.counts.tolist()[1] == want.shape[0]
    for s in range(n):
        nb = (int(ctx[s] + new[s]) + 15) // 16
        assert torch.equal(t.block_tables[s, :nb], pages[rows[s], :nb]) and not t.block_tables[s, nb:].any()
        for j in range(0, int(new[s]), 37):
            p = int(ctx[s]) + j
            assert int(t.positions[starts[s] + j]) == p
            assert int(t.slots[starts[s] + j]) == int(pages[rows[s], p // 16]) * 16 + p % 16
    assert t.slots[total:].tolist() == [-1] * 3 and t.positions[total:].tolist() == [0] * 3


def test_refusals_cpu():
    pages, rows, ctx, new = make(2, [20], 30, 8, 2)
    good = dict(pages=pages, rows=rows, context_lens=ctx, new_lens=new, max_tokens=30, max_tiles=2, n_decode=2)
    ops.build_step_tables(**good)
    gone = pages.clone()
    gone[rows[0], 0] = -1
    for bad in (dict(max_tokens=21), dict(max_tiles=0), dict(new_lens=-new), dict(context_lens=ctx + 500),
                dict(rows=rows + 100), dict(rows=-rows - 1), dict(n_decode=4), dict(n_decode=-1), dict(pages=gone),
                dict(max_tokens=-1), dict(context_lens=ctx[:1])):
        with pytest.raises(ValueError):
            ops.build_step_tables(**(good | bad))


@pytest.mark.gpu
@pytest.mark.parametrize("decode,prompts,ctx_hi,maxb", CASES + [(0, [3] * 1500, 60, 8), (0, [20000], 5000, 1600)])
def test_tables_gpu(cuda_dev, decode, prompts, ctx_hi, maxb):
    pages, rows, ctx, new = make(decode, prompts, ctx_hi, maxb, 3)
    for extra, tiles in ((0, sum((x + 127) // 128 for x in prompts)), (77, 1600)):
        total = int(new.sum()) + extra
        want = ops.build_step_tables(pages, rows, ctx, new, total, tiles, n_decode=decode)
        wide = torch.cat([pages, pages], 1).to(cuda_dev)[:, :maxb]  # a view with a longer row stride
        for p in (pages.to(cuda_dev), wide):
            got = ops.build_step_tables(p, rows.to(cuda_dev), ctx.to(cuda_dev), new.to(cuda_dev), total, tiles,
                                        n_decode=decode)
            for a, b in zip(got, want):
                assert torch.equal(a.cpu(), b)
    ops.core.check_status(cuda_dev)


@pytest.mark.gpu
@pytest.mark.parametrize("block_size,tile", [(16, 64), (32, 128), (5, 3)])
def test_tables_gpu_other_sizes(cuda_dev, block_size, tile):
    pages, rows, ctx, new = make(4, [70, 1, 9], 200, 90, 4)
    want = ops.build_step_tables(pages, rows, ctx, new, 90, 40, 4, block_size, tile)
    got = ops.build_step_tables(*(x.to(cuda_dev) for x in (pages, rows, ctx, new)), 90, 40, 4, block_size, tile)
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b)


@pytest.mark.gpu
def test_reports_gpu(cuda_dev):
    pages, rows, ctx, new = (x.to(cuda_dev) for x in make(2, [20], 30, 8, 2))
    good = dict(pages=pages, rows=rows, context_lens=ctx, new_lens=new, max_tokens=30, max_tiles=2, n_decode=2)
    ok = ops.build_step_tables(**good)
    ops.core.check_status(cuda_dev)
    gone = pages.clone()
    gone[rows[0].long(), 0] = -1
    for bad in (dict(max_tokens=21), dict(max_tiles=0), dict(new_lens=-new), dict(context_lens=ctx + 500),
                dict(rows=rows + 100), dict(rows=-rows - 1), dict(pages=gone)):
        got = ops.build_step_tables(**(good | bad))
        with pytest.raises(ops.core.KernelError):
            ops.core.check_status(cuda_dev)
        if "pages" in bad:  # the other sequences are as they should be
            assert torch.equal(got.slots[1:], ok.slots[1:])
    # lengths that no row of pages holds, of sequences without new tokens as well
    for c, n in ((-1, 0), (129, 0), (2 ** 31 - 1, 0), (2 ** 31 - 1, 1), (5, 2 ** 31 - 1), (2 ** 30, 2 ** 30)):
        c2, n2 = ctx.clone(), new.clone()
        c2[0], n2[0] = c, n
        ops.build_step_tables(**(good | dict(context_lens=c2, new_lens=n2)))
        with pytest.raises(ops.core.KernelError):
            ops.core.check_status(cuda_dev)
    many = torch.full((3,), 2 ** 31 - 1, dtype=torch.int32, device=cuda_dev)  # sums past 32 bits
    ops.build_step_tables(**(good | dict(new_lens=many)))
    with pytest.raises(ops.core.KernelError):
        ops.core.check_status(cuda_dev)
    with pytest.raises(RuntimeError):
        ops.build_step_tables(**(good | dict(max_tokens=2 ** 29)))
    for bad in (dict(rows=rows.long()), dict(n_decode=4), dict(context_lens=ctx[:1]), dict(new_lens=new.cpu()),
                dict(block_size=0), dict(pages=pages.long())):
        with pytest.raises(RuntimeError):
            ops.build_step_tables(**(good | bad))


@pytest.mark.gpu
def test_graph_replay_with_other_lengths(cuda_dev):
    pages, rows, ctx, new = make(3, [200, 10], 300, 40, 5)
    bufs = [x.to(cuda_dev) for x in (pages, rows, ctx, new)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.build_step_tables(*bufs, 260, 6, n_decode=3)
    for shift in (0, 17):
        new2 = new.clone()
        new2[3] -= shift
        bufs[3].copy_(new2)
        bufs[2].copy_(ctx + shift)
        graph.replay()
        for a, b in zip(out, ops.build_step_tables(pages, rows, ctx + shift, new2, 260, 6, n_decode=3)):
            assert torch.equal(a.cpu(), b)
