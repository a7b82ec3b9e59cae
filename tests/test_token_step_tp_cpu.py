"""Token steps at tensor parallelism 2, on CPU (two ``gloo`` ranks): the row-parallel layers' step forms against
the whole product, with the matrix-vector kernel stood in for by its formula, and the calls that
``IncrementalEmbedder`` makes on every rank against a recording stand-in for the library."""
import datetime
import os
import socket
import sys

import numpy as np
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
import __graft_entry__  # noqa: E402  (spawned ranks import this module by name)

__graft_entry__.load_package()

from mes_b200 import _C, synthetic  # noqa: E402
from mes_b200.core.incremental import IncrementalEmbedder  # noqa: E402
from mes_b200.layers.linear import RowParallelLinear  # noqa: E402
from mes_b200.models import Qwen2ForCausalLM, Qwen3ForCausalLM  # noqa: E402
from mes_b200.schemas.config import MESConfig  # noqa: E402
from oracle import awq as oawq  # noqa: E402

K, N, GROUP = 512, 72, 128


class _RecordingLib:
    def __init__(self, real):
        self.real, self.calls = real, []

    def __getattr__(self, name):
        if name.endswith("_size") or name == "mes_status_string":
            return getattr(self.real, name)

        def launch(*args):
            self.calls.append(name)
            return 0
        return launch


def _weights():
    rng = np.random.default_rng(3)
    q, z = rng.integers(0, 16, (K, N), dtype=np.uint8), rng.integers(0, 16, (K // GROUP, N), dtype=np.uint8)
    s = rng.uniform(0.002, 0.02, (K // GROUP, N)).astype(np.float16)
    bias = torch.from_numpy(rng.uniform(50, 100, N)).to(torch.bfloat16)      # counted twice, it would show
    return (torch.from_numpy(oawq.awq_pack(q)), torch.from_numpy(oawq.awq_pack(z)), torch.from_numpy(s), bias,
            (q.astype(np.float64) - np.repeat(z, GROUP, 0)) * np.repeat(s.astype(np.float64), GROUP, 0))


def _layer(rows):
    """Distances of ``step`` and ``step_residual`` from ``x W + b`` over their bound, and whether the residual was left."""
    qw, qz, s, bias, w = _weights()
    layer = RowParallelLinear(K, N, bias=True)
    for param, full in ((layer.qweight, qw), (layer.qzeros, qz), (layer.scales, s), (layer.bias, bias)):
        layer.weight_loader(param, full)
    used = []

    def gemv(x, qm, zeros, scales, b=None, group_size=GROUP):
        used.append(x.shape)
        c = oawq.mes_unpack(qm.numpy()).astype(np.float64) - np.repeat(oawq.awq_unpack(zeros.numpy()).astype(np.float64), group_size, 0)
        y = x.double().numpy() @ (c * np.repeat(scales.view(torch.float16).double().numpy(), group_size, 0))
        return torch.from_numpy(y if b is None else y + b.double().numpy()).to(torch.bfloat16)
    saved = _C.awq_repack, _C.awq_gemv
    _C.awq_repack, _C.awq_gemv = lambda t: torch.from_numpy(oawq.mes_repack(t.numpy())), gemv
    try:
        x = torch.randn(rows, K, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
        rank, half = dist.get_rank(), K // 2
        mine = x[:, rank * half:(rank + 1) * half]
        residual = torch.randn(rows, N, generator=torch.Generator().manual_seed(2))
        before = residual.clone()
        a, b = layer.step(mine), layer.step_residual(mine, residual)
    finally:
        _C.awq_repack, _C.awq_gemv = saved
    xd, bd = x.double().numpy(), bias.double().numpy()
    parts = [xd[:, i * half:(i + 1) * half] @ w[i * half:(i + 1) * half] for i in range(2)]
    parts[0] = parts[0] + bd
    want = parts[0] + parts[1]
    # two roundings to bf16 and that of their sum
    bound = 2.0 ** -8 * (np.abs(parts[0]) + np.abs(parts[1]) + np.abs(want))
    off = max(float((np.abs(t.double().numpy() - want) / bound).max()) for t in (a, b))
    return off, torch.equal(residual, before), used


def _embedder(cls, cfg):
    fake = _RecordingLib(_C.lib())
    _C.lib = lambda: fake
    _C._stream = lambda t: 0
    emb = IncrementalEmbedder(cls(MESConfig(model_config=cfg)), num_pages=30, page_size=16, budget=32, observe=4)
    handles, out = emb.add([np.arange(40), np.arange(3)])
    shapes = [tuple(out.shape)]
    first = list(fake.calls)
    fake.calls.clear()
    shapes.append(tuple(emb.extend(handles, [[1], [2, 3]]).shape))        # few rows, and an eviction
    few = list(fake.calls)
    fake.calls.clear()
    shapes.append(tuple(emb.extend(handles, [[1] * 9, [2] * 11]).shape))  # more than the matrix-vector kernel takes
    return shapes, first, few, list(fake.calls), [emb.cached_tokens(h) for h in handles], emb.caches[0].codes.shape[2]


def _rank(rank, world, port, q):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world, timeout=datetime.timedelta(seconds=120))
    torch.set_num_threads(2)
    try:
        layer = [_layer(rows) for rows in (1, 5, 16)]
        models = [_embedder(cls, make(num_hidden_layers=2, vocab_size=1000)) for cls, make in
                  ((Qwen3ForCausalLM, synthetic.qwen3_0_6b), (Qwen2ForCausalLM, synthetic.qwen2_1_5b))]
        q.put((rank, layer, models))
    finally:
        dist.destroy_process_group()


def test_two_ranks():
    with socket.socket() as sk:
        sk.bind(("127.0.0.1", 0))
        port = sk.getsockname()[1]
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    procs = [ctx.Process(target=_rank, args=(r, 2, port, q)) for r in range(2)]
    for p in procs:
        p.start()
    results = [q.get(timeout=300) for _ in procs]
    for p in procs:
        p.join(timeout=60)
    assert all(p.exitcode == 0 for p in procs), [p.exitcode for p in procs]
    for rank, layer, models in results:
        for rows, (off, residual_left, used) in zip((1, 5, 16), layer):
            assert off <= 1 and residual_left and used == [(rows, K // 2)] * 2, (rank, rows, off)
        for (shapes, first, few, many, cached, kv_heads), (hidden, heads) in zip(models, ((1024, 8), (1536, 2))):
            assert shapes == [(2, hidden)] * 3 and kv_heads == heads // 2 and cached == [32, 16]
            # the sums of the ranks' parts are added to the residual by the norm that follows
            assert few.count("mes_awq_gemv") == 2 * 4 and "mes_awq_gemm_ws" not in few
            assert few.count("mes_add_rmsnorm_f32res") == 4 and few.count("mes_kv8_evict") == 2
            assert "mes_awq_gemv" not in first + many and {"mes_awq_gemm_ws", "mes_kv8_attention"} <= set(many)
    # every rank made the same calls
    assert [m[1:4] for m in results[0][2]] == [m[1:4] for m in results[1][2]]
