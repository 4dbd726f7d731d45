"""What a region leaves in an 8-bit arena: a retained document's pages hold its own tokens' values and no trace of
the questions asked of it. A stub model writes K and V that depend on the token alone, so they can be compared
bit for bit."""

import numpy as np
import pytest
import torch

from quail_b200.engine.arena import KVArena
from quail_b200.engine.region import Call, RegionRun
from quail_b200.engine.stage_executor import StageExecutor
from quail_b200.ops import KV8_DTYPES
from quail_b200.ops import reference as ref

VOCAB, KH, D, P = 64, 2, 64, 16
LOUD, BROKEN = 60, 61                # tokens with very large K and V, and with ones that are not finite


class Stub:
    """Writes a token's own K and V; logits by the token at each readout row."""

    def __init__(self, width):
        g = torch.Generator().manual_seed(0)
        self.k, self.v = (torch.randn(VOCAB, KH, D, generator=g) for _ in range(2))
        for x in (self.k, self.v):
            x[LOUD] *= 1e4
            x[BROKEN] = float("nan")
        self.out = torch.randn(VOCAB, width, generator=g)

    def forward_chunk(self, chunk, arena):
        for i in range(arena.num_layers):
            for x, p in zip((self.k, self.v), arena.layer(i)):
                ref.kv8_write(x[chunk.ids.long()], chunk.slots, p.codes, p.bytes)
        return self.out[chunk.ids.long()[chunk.final_rows.long()]] if chunk.final_rows.numel() else None


def executor(kind="int8", pages=64, chunk_tokens=256):
    arena = KVArena(1, pages, P, KH, D, device="cpu", dtype=KV8_DTYPES[kind])
    return StageExecutor(Stub(6), arena, chunk_tokens)


def score(name, suffix):
    return Call(kind="score", suffix=np.asarray(suffix, np.int32), true_cols=[0], false_cols=[1], name=name)


def run(ex, docs, calls, retain=True):
    r = RegionRun(ex, np.arange(1, 20, dtype=np.int32), docs, calls, answer_width=4)
    if retain:
        r.retain_key = lambda i: ("kept", i)
    r.run()
    ex.pool.check()
    return r


def held(ex, key, doc):
    """A key's codes and bytes of its document's tokens."""
    pages, n = ex.pool.owned[key], len(doc)
    out = []
    for p in ex.arena.layer(0):
        c = torch.cat([p.codes.view(torch.uint8)[g] for g in pages], dim=1)[:, :n]
        b = torch.cat([p.bytes[g] for g in pages], dim=1)[:, :-(-n // 16)]
        out += [c, b]
    return out


def alone(doc, kind):
    """The same of a document written by itself, whole blocks at a time."""
    arena = KVArena(1, 8, P, KH, D, device="cpu", dtype=KV8_DTYPES[kind])
    m = Stub(6)
    out = []
    for x, p in zip((m.k, m.v), arena.layer(0)):
        ref.kv8_write(x[torch.as_tensor(doc).long()], torch.arange(len(doc), dtype=torch.int32), p.codes, p.bytes)
        n = len(doc)
        c = torch.cat(list(p.codes.view(torch.uint8)), dim=1)[:, :n]
        out += [c, torch.cat(list(p.bytes), dim=1)[:, :-(-n // 16)]]
    return out


DOCS = [np.asarray([(7 * i + j) % 50 + 1 for j in range(n)], np.int32) for i, n in enumerate((5, 16, 21, 33, 100))]


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("suffix", [[3, 4], [LOUD, 4], [BROKEN, 5]])
def test_a_retained_document_has_no_trace_of_its_questions(kind, suffix):
    ex = executor(kind)
    run(ex, DOCS, [score("a", suffix), score("b", [9, LOUD, BROKEN])])
    for i, doc in enumerate(DOCS):
        assert all(torch.equal(x, y) for x, y in zip(held(ex, ("kept", i), doc), alone(doc, kind)))
    again = run(ex, DOCS, [score("c", [LOUD])])
    assert ex.stats.reused == len(DOCS) and all("c" in x.values for x in again.results)
    for i, doc in enumerate(DOCS):
        assert all(torch.equal(x, y) for x, y in zip(held(ex, ("kept", i), doc), alone(doc, kind)))


def test_the_answers_are_those_of_one_sequence():
    # the document and its first question as one sequence, or apart: the stub's answers go by the last token
    ex = executor()
    got = run(ex, DOCS, [score("a", [3, 4]), score("b", [9])], retain=False)
    logits = ex.model.out.double().numpy()
    for res in got.results:
        for name, tok in (("a", 4), ("b", 9)):
            m = logits[tok][0] - logits[tok][1]
            assert abs(res.values[name] - 1 / (1 + np.exp(-m))) < 1e-6
    assert ex.pool.free_pages == ex.pool.num_pages


def test_decoding_and_classifying_over_apart_documents():
    ex = executor()
    calls = [Call(kind="map", suffix=np.asarray([3], np.int32), max_tokens=4, stop_ids=(99,), name="m"),
             Call(kind="classify", suffix=np.asarray([5, 6], np.int32), labels=[[1, 2], [3], [4, 5, 6]],
                  label_cols=[[0, 1], [2], [1, 2, 3]], name="c")]
    ex.model.out[:, 4] = (torch.arange(VOCAB) % 7 + 1).float()          # the argmax column: a token to go on with
    got = run(ex, DOCS, calls)
    assert all(len(r.values["m"]) == 4 and r.values["c"] in (0, 1, 2) for r in got.results)
    for i, doc in enumerate(DOCS):
        assert all(torch.equal(x, y) for x, y in zip(held(ex, ("kept", i), doc), alone(doc, "int8")))


def test_max_pooled_features_read_the_documents_rows_too():
    # packed readout rows: ids, then strengths; every own token of the document and of the question is read
    def rows(ex):
        ex.model.out[:, :3] = torch.arange(VOCAB)[:, None].float() * 3 + torch.arange(3)
        ex.model.out[:, 3:] = 1.0 + torch.arange(VOCAB)[:, None].float() + torch.tensor([0.0, 0.1, 0.2])
    ex = executor()
    rows(ex)
    call = Call(kind="features", suffix=np.asarray([3, 4], np.int32), pooling="max", name="f")
    got = run(ex, DOCS, [call, score("b", [9])])
    for doc, res in zip(DOCS, got.results):
        want = {int(t) * 3 + j for t in list(doc) + [3, 4] for j in range(3)}
        assert {i for i, _ in res.values["f"]} == want


def test_many_documents_in_a_small_arena_leave_room_for_their_questions():
    # more documents than pages: admitted documents must not take the pages their questions need
    ex = executor(pages=24, chunk_tokens=4096)
    docs = [np.asarray([i % 50 + 1] * 10, np.int32) for i in range(200)]
    got = run(ex, docs, [score("a", [3, 4])], retain=False)
    assert all("a" in r.values for r in got.results) and ex.pool.free_pages == ex.pool.num_pages
    got = run(ex, docs, [score("a", [3, 4]), score("b", [9])])
    assert all("b" in r.values for r in got.results)


def test_no_copy_drafts_over_8_bit_pages():
    # a draft's rejected tokens share blocks with the tokens before them
    doc = DOCS[3]
    call = Call(kind="extract", suffix=np.asarray([3], np.int32), copy=True, name="x")
    for kind, want in (("int8", ()), (None, tuple(int(t) for t in doc[2:6]))):
        arena = KVArena(1, 64, P, KH, D, device="cpu", dtype=KV8_DTYPES[kind] if kind else torch.float32)
        r = RegionRun(StageExecutor(Stub(6), arena, 256), np.arange(1, 20, dtype=np.int32), [doc], [call], answer_width=4)
        r._copies[(0, 0)] = np.asarray([2])
        assert r._draft(0, 0, 4) == want


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("chunk_tokens", [17, 70, 100])
def test_pieces_of_a_document_end_where_a_block_does(kind, chunk_tokens):
    # a block written in two pieces would be rounded twice, by where the piece happened to end
    ex = executor(kind, chunk_tokens=chunk_tokens)
    docs = [*DOCS, np.asarray([LOUD if j % 11 == 10 else j % 50 + 1 for j in range(90)], np.int32)]
    run(ex, docs, [score("a", [3, 4])])
    assert max(ex.stats.pass_tokens) <= chunk_tokens and ex.stats.passes > len(docs) // 2
    for i, doc in enumerate(docs):
        assert all(torch.equal(x, y) for x, y in zip(held(ex, ("kept", i), doc), alone(doc, kind)))


def test_a_pass_smaller_than_a_block_still_gets_on():
    ex = executor(chunk_tokens=5)
    got = run(ex, DOCS, [score("a", [3, 4])], retain=False)
    assert all("a" in r.values for r in got.results)
