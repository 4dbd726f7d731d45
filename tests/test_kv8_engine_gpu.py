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


def session(kind, **kw):
    import pyarrow as pa

    import quail_b200 as quail
    rng = np.random.default_rng(0)
    words = ["ending", "music", "cast", "plot", "money", "great", "bad", "long"]
    bodies = [" ".join(rng.choice(words, size=int(rng.integers(3, 40)))) for _ in range(40)]
    s = quail.Session(config=quail.EngineConfig(model="qwen3-gpu-tiny-gqa4", device="b200", chunk_tokens=2048,
                                                kv_dtype=kind, **kw))
    s.register("t", pa.table({"id": list(range(40)), "body": bodies}))
    return s, bodies


@pytest.mark.parametrize("kind", ["int8", "fp8"])
def test_sessions_answer_every_kind_of_call(kind):
    s, bodies = session(kind)
    with s:
        t = s.sql("""
            SELECT id, AI.SCORE(PROMPT('Positive? {0}', body)) AS s,
                   AI.CLASSIFY(body, ['praise', 'complaint'], {'probabilities': true}) AS k,
                   AI.MAP(body, 'Summarize.', 4) AS m, AI.EXTRACT(body, ['What is it about?']) AS e
            FROM t ORDER BY id""").collect()
        kept = s.sql("SELECT id FROM t WHERE AI.IF(PROMPT('Is it about music? {0}', body)) ORDER BY id").collect()
        flags = s.sql("SELECT id, AI.IF(PROMPT('Is it about music? {0}', body)) AS f FROM t ORDER BY id").collect()
        assert s.engine().executor.stats.reused >= 40
    assert t.num_rows == 40 and all(0.0 < x < 1.0 for x in t.column("s").to_pylist())
    assert set(t.column("k").to_pylist()) <= {"praise", "complaint"}
    assert all(isinstance(m, str) for m in t.column("m").to_pylist())
    for body, e in zip(bodies, t.column("e").to_pylist()):
        assert all(x is None or x.strip() in body for x in e)
    want = [i for i, f in zip(flags.column("id").to_pylist(), flags.column("f").to_pylist()) if f]
    assert kept.column("id").to_pylist() == want


@pytest.mark.parametrize("kind", ["int8", "fp8"])
def test_retained_documents_are_the_same_whatever_was_asked(kind):
    asked = ("SELECT id, AI.IF(PROMPT('Would somebody who wrote this go again? {0}', body)) AS m FROM t ORDER BY id",
             "SELECT id, AI.IF(PROMPT('Is it about music? {0}', body)) AS f FROM t ORDER BY id")
    held = []
    for queries in (asked, asked[::-1], asked[1:]):
        s, _ = session(kind)
        with s:
            for q in queries:
                s.sql(q).collect()
            arena = s.engine().arena
            got = {}
            for key in arena.pool.retained:
                pages, n = arena.pool.owned[key], arena.pool.tokens[key]
                parts = []
                for i in range(arena.num_layers):
                    for p in arena.layer(i):
                        codes = torch.cat([p.codes[g].view(torch.uint8) for g in pages], dim=1)[:, :n]
                        parts += [codes, torch.cat([p.bytes[g] for g in pages], dim=1)[:, :-(-n // 16)]]
                got[key] = [x.cpu() for x in parts]
            held.append(got)
    assert len(held[0]) >= 35 and held[0].keys() == held[1].keys() == held[2].keys()
    for other in held[1:]:
        for key, parts in held[0].items():
            assert all(torch.equal(x, y) for x, y in zip(parts, other[key]))
