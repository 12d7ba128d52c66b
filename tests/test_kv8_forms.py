"""The 8-bit KV cache under the framework's other settings: fp8 weights, the host cache and its kernel
write-behind, durable and remote pools, and prefill and decode on separate instances."""
import json
import os
import random

import numpy as np
import pytest
import torch
import torch.multiprocessing as mp

from lake_b200 import ops
from lake_b200.engine.block_pool import chain_block_hashes
from lake_b200.engine.llm_engine import LLMEngine
from lake_b200.oracle import ops_ref as ref
from lake_b200.pool.pool_iface import PoolIface

BF = torch.bfloat16


def _tiny(**kw):
    return LLMEngine("tiny", device="cpu", max_running=4, max_batched_tokens=128, max_model_len=512, kv_dtype="fp8", **kw)


# ------------------------------------------------------------------ host cache and pools, CPU
def test_host_cache_and_durable_tier_cpu(tmp_path):
    """Pages leave the arena as bytes, by the epilogue's second target and by copy, reach durable records,
    and come back: the same tokens as an engine that kept them."""
    from lake_b200.pool.agents.durable import DurableTier
    from lake_b200.pool.agents.hostcache import HostCacheAgent

    rng = np.random.default_rng(5)
    first = rng.integers(0, 1024, 40).tolist()
    eng = _tiny(num_blocks=24)
    page_bytes = eng.arena[0].numel()
    tier = DurableTier("tiny", page_bytes, eng.cfg.n_layers, 16, l2_blocks=256, storage_dir=str(tmp_path))
    agent = HostCacheAgent(eng, l1_blocks=10, durable=tier)
    eng.attach_pool(PoolIface(agent))
    assert agent.mirror_arena.dtype == torch.uint8 and agent.mirror_arena.shape[1:] == eng.arena.shape[1:]
    out = eng.generate([first], max_new_tokens=60)[0]
    assert agent.stats["kernel_written_blocks"] == 3 and agent.stats["copied_blocks"] == 3
    tier.flush()
    hashes = chain_block_hashes((first + out)[:6 * 16], 16, full_only=True)
    for h in hashes:
        assert torch.equal(agent.l1[agent.slot_of[h]], eng.arena[eng.pool.block_of[h]].view(-1))
    for p in [rng.integers(0, 1024, 150).tolist() for _ in range(2)]:  # out of the arena and of the 10 slots
        eng.generate([p], max_new_tokens=2)
    tier.flush()
    follow = first + out + rng.integers(0, 1024, 7).tolist()
    got = eng.generate([follow], max_new_tokens=5)[0]
    assert agent.stats["l2_promoted_blocks"] > 0
    assert got == _tiny(num_blocks=64).generate([follow], max_new_tokens=5)[0]
    tier.close()


def test_native_pool_agent_cpu(tmp_path):
    """One pool node that two engines share: what the first wrote back, the second promotes."""
    from lake_b200 import _host as H
    from lake_b200.pool.agents.native import NativeAgent, make_pool_node

    a, b = _tiny(num_blocks=64), _tiny(num_blocks=64)
    node = make_pool_node("tiny", a.arena[0].numel(), a.pool.num_blocks, l1_blocks=8, l2_blocks=2, storage_dir=str(tmp_path))
    authority = H.Authority()
    agents = [NativeAgent(e, "n0", authority=authority, shared_tiers=node) for e in (a, b)]
    for e, ag in zip((a, b), agents):
        e.attach_pool(PoolIface(ag, node_id="n0"))
    prompt = list(range(3, 3 + 5 * 16 + 1))
    want = a.generate([prompt], max_new_tokens=4)
    assert b.generate([prompt], max_new_tokens=4) == want and agents[1].stats["promoted_blocks"] == 5
    for h in chain_block_hashes(prompt, 16, full_only=True)[:5]:
        assert torch.equal(a.arena[a.pool.block_of[h]], b.arena[b.pool.block_of[h]])


@pytest.mark.parametrize("second", ["fp8", "bf16"])
def test_remote_pool_cpu(second):
    """Worker B pulls what worker A wrote back; a worker of the other cache takes no page of another size and
    computes its own."""
    from concurrent import futures

    import grpc

    from lake_b200.api import proto
    from lake_b200.runtime.config import RoleConfig
    from lake_b200.runtime.worker import remote_pool_factory
    from lake_b200.runtime.worker_engine import WorkerEngine, build_engine
    from lake_b200.services.controlplane import ControlPlane
    from lake_b200.services.kvpool import serve as serve_kvpool

    cp = ControlPlane()
    server = grpc.server(futures.ThreadPoolExecutor(max_workers=8), options=proto.message_options())
    proto.add_service(server, "ControlPlaneService", cp)
    port = server.add_insecure_port("127.0.0.1:0")
    server.start()
    kv_server, kv_port = serve_kvpool("127.0.0.1:0", max_workers=8)

    def cfg(kv):
        return RoleConfig(model_backend="mock", served_model_name="tiny", device="cpu", max_running_reqs=4,
                          max_num_scheduled_tokens=128, max_model_length=512, num_blocks=64, enable_overlap=False, kv_dtype=kv)

    workers = []
    try:
        for node, kv in (("wA", "fp8"), ("wB", second)):
            we = WorkerEngine(cfg(kv), node_id=node, pool_factory=remote_pool_factory(
                f"127.0.0.1:{port}", f"127.0.0.1:{kv_port}", node, "tiny"))
            we.start()
            workers.append(we)
        prompt = np.random.default_rng(1).integers(0, 1024, 100).tolist()
        ra = workers[0].submit("r-a", prompt, 4)
        assert ra.output_tokens == build_engine(cfg("fp8")).generate([prompt], max_new_tokens=4)[0]
        follow = prompt + np.random.default_rng(2).integers(0, 1024, 20).tolist()
        rb = workers[1].submit("r-b", follow, 4)
        assert rb.output_tokens == build_engine(cfg(second)).generate([follow], max_new_tokens=4)[0]
        stats = workers[1].pool.agent.stats
        assert stats["pulled_blocks"] == (6 if second == "fp8" else 0)
        assert stats["missing_bytes"] == (0 if second == "fp8" else 1)
    finally:
        for we in workers:
            we.stop(drain=False)
        cp.stop()
        server.stop(0)
        kv_server.stop(0)


# ------------------------------------------------------------------ prefill and decode instances, CPU
def _free_port():
    import socket

    s = socket.socket()
    s.bind(("127.0.0.1", 0))
    p = s.getsockname()[1]
    s.close()
    return p


def _pd_prompts():
    rng = random.Random(5)
    prefix = [rng.randrange(1024) for _ in range(48)]
    return [prefix + [rng.randrange(1024) for _ in range(n)] for n in (3, 20, 40, 1)]


def _pd_worker(rank, port, out_dir):
    import torch.distributed as dist

    from lake_b200.parallel import pd
    from lake_b200.parallel.peer import unlink_shared

    os.environ["MASTER_ADDR"] = "127.0.0.1"
    os.environ["MASTER_PORT"] = str(port)
    dist.init_process_group("gloo", rank=rank, world_size=2)
    role = "prefill" if rank == 0 else "decode"
    eng = _tiny(num_blocks=96, shared_arena=(role == "decode"))
    side = pd.connect_pair(eng, role, rank, 1 - rank, None, job=f"k8{port}", shm_path=eng.arena_path)
    if role == "prefill":
        pd.serve_prefill(side)
    else:
        prompts = _pd_prompts()
        rids = [side.submit(p, 8) for p in prompts]
        while side.inflight:
            side.poll()
            eng.step()
        outs = [eng.requests[r].output for r in rids]
        want = _tiny(num_blocks=96).generate(prompts, max_new_tokens=8)
        side.shutdown()
        with open(os.path.join(out_dir, "res.json"), "w") as f:
            json.dump({"outs": outs, "want": want, "kv_bytes": side.kv_bytes, "page": side.page_bytes}, f)
    dist.barrier()
    side.close()
    dist.destroy_process_group()
    if eng.arena_path:
        unlink_shared(eng.arena_path)


def test_prefill_instance_writes_the_decode_instances_arena_cpu(tmp_path):
    mp.spawn(_pd_worker, args=(_free_port(), str(tmp_path)), nprocs=2, join=True)
    res = json.load(open(tmp_path / "res.json"))
    assert res["outs"] == res["want"] and res["kv_bytes"] > 0
    assert res["page"] == _tiny(num_blocks=4).arena[0].numel()


# ------------------------------------------------------------------ fp8 weights, GPU
@pytest.mark.gpu
@pytest.mark.parametrize("t,w8a8", [(1, False), (70, False), (300, False), (70, True), (300, True), (1000, True)])
@pytest.mark.parametrize("norm", [False, True])
def test_linear_qkv_of_fp8_weights_writes_the_8bit_arena(cuda_dev, t, w8a8, norm):
    """W8A16 and W8A8 sums reach the quantising epilogue as the bf16 arena's calls see them: q is the same, the
    cached rows are within a quantisation step of the rows that the same call leaves in a bf16 arena."""
    from lake_b200.ops._ext import native
    from lake_b200.ops.fp8 import quantize_blockwise

    g = torch.Generator(device=cuda_dev).manual_seed(t)
    hid, hq, hkv, layers = 512, 4, 2, 2
    a = (torch.randn(t, hid, device=cuda_dev, generator=g) * 0.5).to(BF)
    w = quantize_blockwise(torch.randn((hq + 2 * hkv) * 128, hid, device=cuda_dev, generator=g) / 20)
    cs = ref.rope_cache(4096, 500000.0, device=cuda_dev)
    pos = torch.randint(0, 4000, (t,), device=cuda_dev, dtype=torch.int32, generator=g)
    slots = torch.randperm(64 * 16, device=cuda_dev, generator=g)[:t]
    if t > 5:
        slots[5] = -1
    back = torch.where(slots >= 0, 64 * 16 - 1 - slots, slots)
    nw = [(1 + 0.1 * torch.randn(128, device=cuda_dev, generator=g)).to(BF) for _ in range(2)] if norm else [None] * 2
    arena, peer = (ops.kv8_arena(64, layers, hkv, device=cuda_dev) for _ in range(2))
    dense = torch.zeros(64, layers, 2, hkv, 16, 128, dtype=BF, device=cuda_dev)
    qa, qb = (torch.empty(t, hq * 128, dtype=BF, device=cuda_dev) for _ in range(2))
    native().set_gemm_w8a8_min_m(1 if w8a8 else 0)
    try:
        if w8a8:
            assert native().gemm_w8a8_reserve(t, hid)
        for _ in range(3):  # back to back: a hand-over that is early shows as another row
            ops.linear_qkv(a, w, qa, cs, pos, slots, arena, 1, hq, hkv, peer, back, *nw)
        ops.linear_qkv(a, w, qb, cs, pos, slots, dense, 1, hq, hkv, None, None, *nw)
        ops.core.check_status(cuda_dev)
    finally:
        native().set_gemm_w8a8_min_m(256)
    keep = slots >= 0
    sl = slots[keep]
    # (the split of a small product's K adds in any order: fp32 sums of 512 products, 2^-12 of the row's largest,
    # which may also move q over a bf16 step)
    assert bool(((qa.float() - qb.float()).abs() <= 2.0 ** -7 * qb.float().abs() + 2.0 ** -12 * qb.float().abs().amax()).all())
    assert not arena[:, 0].any()
    for side, got in enumerate(ops.kv8_read(arena, 1, slots)):
        got = got.view(t, hkv, 128).double()[keep]
        want = dense[sl // 16, 1, side, :, sl % 16].double()
        top = want.abs().amax(-1, keepdim=True)
        # half a step of e4m3 (2^-4 of the value, 2^-10 2^e at least, 2^e <= top / 224, twice that for the roundings of
        # top itself), half a bf16 step (2^-8), the sums' order (2^-12, twice)
        assert bool(((got - want).abs() <= (2.0 ** -4 + 2.0 ** -8) * want.abs() + 2.0 ** -9 * top / 224 + 2.0 ** -11 * top).all())
    for x, y in zip(ops.kv8_read(arena, 1, slots), ops.kv8_read(peer, 1, back)):
        assert torch.equal(x, y)


@pytest.mark.gpu
@pytest.mark.parametrize("w8a8", [False, True])
def test_engine_of_fp8_weights_and_8bit_kv_gpu(cuda_dev, w8a8):
    """Both settings at once, in eager and graph steps: teacher-forced oracle logits on the dequantised weights and
    an 8-bit cache put the engine's tokens within the roundings of the largest logit."""
    from lake_b200.models.llama import ForwardBatch
    from lake_b200.ops._ext import native
    from lake_b200.ops.fp8 import Fp8Weight

    kw = dict(max_running=8, max_batched_tokens=256, max_model_len=512, num_blocks=128, kv_dtype="fp8")
    native().set_gemm_w8a8_min_m(1 if w8a8 else 256)
    try:
        eng = LLMEngine("tiny-gpu", device=cuda_dev, weight_dtype="fp8", use_cuda_graphs=not w8a8, **kw)
        rng = random.Random(8)
        prompts = [[rng.randrange(eng.cfg.vocab) for _ in range(n)] for n in (5, 70, 130)]
        outs = eng.generate(prompts, max_new_tokens=6)
        torch.cuda.synchronize()
        ops.core.check_status(cuda_dev)
    finally:
        native().set_gemm_w8a8_min_m(256)
    cpu = LLMEngine("tiny-gpu", device="cpu", **kw)
    for k, v in eng.model.w.items():
        cpu.model.w[k].copy_((v.dequant(torch.bfloat16, swiglu_tile=256) if isinstance(v, Fp8Weight) else v).float().cpu())
    for p, o in zip(prompts, outs):
        toks = p + o[:-1]
        t = len(toks)
        blocks = cpu.reserve_blocks(t)
        pos, bt = torch.arange(t, dtype=torch.int32), torch.tensor([blocks], dtype=torch.int32)
        b = ForwardBatch(input_ids=torch.tensor(toks, dtype=torch.int32), positions=pos,
                         slots=bt[0].long()[pos.long() // 16] * 16 + pos.long() % 16, block_tables=bt,
                         seq_lens=torch.tensor([t], dtype=torch.int32), n_decode=0,
                         prefill_tiles=ops.build_prefill_tiles([0, t], [0]),
                         query_start=torch.tensor([0, t], dtype=torch.int32), sample_rows=pos.long(), want_logits=True)
        lg = cpu.model.forward(b, cpu.arena, cpu.model.new_workspace(t, t, 1))[len(p) - 1:]
        cpu.release_blocks(blocks)
        got = lg[torch.arange(len(o)), torch.tensor(o)]
        # bf16 activations: under 32 roundings of 2^-8 over two layers; W8A8 rounds the input of every projection to
        # e4m3 as well, 2^-4 an element, independent ones, of which a sum keeps its relative size: eight, in quadrature
        tol = 32 * 2.0 ** -8 + (8 ** 0.5 * 2.0 ** -4 if w8a8 else 0.0)
        assert bool((lg.amax(-1) - got <= tol * lg.std(-1)).all()), float(((lg.amax(-1) - got) / lg.std(-1)).amax())


# ------------------------------------------------------------------ host cache, GPU
@pytest.mark.gpu
@pytest.mark.parametrize("graphs", [False, True])
def test_kernel_write_behind_gpu(cuda_dev, graphs):
    """The epilogue writes generated tokens' rows into the pinned host slab beside the arena: the same bytes, and
    pages that come back from there are those that left."""
    from lake_b200.pool.agents.hostcache import HostCacheAgent

    rng = np.random.default_rng(9)
    first = rng.integers(0, 2048, 40).tolist()
    eng = LLMEngine("tiny-gpu", device=cuda_dev, max_running=4, max_batched_tokens=256, max_model_len=1024, num_blocks=40,
                    kv_dtype="fp8", use_cuda_graphs=graphs)
    agent = HostCacheAgent(eng, l1_blocks=128)
    eng.attach_pool(PoolIface(agent))
    if graphs:
        eng.runner.capture_graphs()
    out = eng.generate([first], max_new_tokens=60)[0]
    torch.cuda.synchronize()
    assert agent.stats["kernel_written_blocks"] == 3 and not agent.reserved
    hashes = chain_block_hashes((first + out)[:6 * 16], 16, full_only=True)
    left = {h: agent.l1[agent.slot_of[h]].clone() for h in hashes}
    for h in hashes:
        assert torch.equal(left[h], eng.arena[eng.pool.block_of[h]].view(-1).cpu())
    for p in [rng.integers(0, 2048, 200).tolist() for _ in range(3)]:
        eng.generate([p], max_new_tokens=2)
    follow = first + out + rng.integers(0, 2048, 9).tolist()
    eng.generate([follow], max_new_tokens=6)
    torch.cuda.synchronize()
    assert agent.stats["promoted_blocks"] >= 5
    back = [h for h in hashes if h in eng.pool.block_of]
    assert len(back) >= 5 and all(torch.equal(left[h], eng.arena[eng.pool.block_of[h]].view(-1).cpu()) for h in back)
    ops.core.check_status(cuda_dev)
