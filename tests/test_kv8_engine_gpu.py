"""8-bit KV arenas under the engine on the GPU."""

import numpy as np
import pytest
import torch

from quail_b200 import ops
from quail_b200.engine.arena import KVArena
from quail_b200.engine.chunk import ChunkPacker, SeqSpec
from quail_b200.models.config import QWEN3_GPU_TINY_GQA4

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0) if torch.cuda.is_available() else None


def test_decode_graphs_hold_the_form_for_few_keys_and_the_other():
    # a graph's page list has spare entries, so its decode goes by the keys the packer counted; a row that
    # passes the limit goes to a graph of its own (bounds as for an eager pass, see test_kv8_model_gpu.py)
    from quail_b200.engine.graphs import DecodeGraphs
    from quail_b200.models.build import build_pipeline
    cfg = QWEN3_GPU_TINY_GQA4.with_(weight_dtype="bf16")
    pipe = build_pipeline(cfg, device=DEV, seed=0, answer_ids=(1, 2, 3, 4))
    arena = KVArena(cfg.layers, 64, 128, cfg.num_kv_heads, cfg.head_dim, device=DEV, dtype=torch.int8)
    packer, graphs = ChunkPacker(arena.pool, DEV), DecodeGraphs(pipe, arena, DEV)
    rng = np.random.default_rng(3)
    lens = (ops.KV8_FEW_KEYS - 2, 1, 64)
    for i, n in enumerate(lens):
        arena.pool.alloc(i, n, capacity=n + 8)
    pipe.forward_chunk(packer.pack([SeqSpec([], i, 0, rng.integers(0, 1000, n).astype(np.int32), 0, readout=True)
                                    for i, n in enumerate(lens)]), arena)
    for step in range(5):
        specs = [SeqSpec([], i, n + step, rng.integers(0, 1000, 1).astype(np.int32), n + step, readout=True)
                 for i, n in enumerate(lens)]
        eager = pipe.forward_chunk(packer.pack(specs), arena).float()
        got = graphs.run(packer.host_parts(specs)[0], False)[0].float()
        assert torch.allclose(got, eager, atol=0.02 * float(eager.abs().max()))
        # 1023 and 1024 keys in the longest row, then more
        assert (graphs.captures, graphs.replays) == ((1, step) if step < 2 else (2, step - 1))
    assert sorted(at[3] for at in graphs.entries) == [ops.KV8_FEW_KEYS, ops.KV8_FEW_KEYS + 1]
    assert ops.read_and_clear_error(0) == 0
