"""What decides between the two forms of decode over the 8-bit cache, and what the packer tells it."""

import numpy as np

from quail_b200.engine.arena import PagePool
from quail_b200.engine.chunk import ChunkPacker, SeqSpec
from quail_b200.ops.kv8 import KV8_FEW_KEYS, _few_keys


def test_the_rule_goes_by_the_longest_row():
    # a padded page list (a captured graph's) says nothing where the caller knows the keys
    assert _few_keys(8, 1025, 128, 230) and _few_keys(8, 1025, 128, KV8_FEW_KEYS)
    assert not _few_keys(8, 20, 128, KV8_FEW_KEYS + 1)
    # one long row among short ones has a long list, though its average is short
    assert not _few_keys(55, 54 + -(-20000 // 128), 128, None)
    # one long shared document, listed once for all its readers
    assert not _few_keys(8, 8 + -(-7000 // 128), 128, None)
    assert _few_keys(8, 8 * 2 + 1, 128, None) and _few_keys(30, 30 * 7, 16, None) and _few_keys(40, 40 * 2, 128, None)
    # one row: its keys are the list's
    assert _few_keys(1, 8, 128, None) and not _few_keys(1, 9, 128, None)


def test_a_chunk_carries_the_most_keys_of_its_one_token_rows():
    pool = PagePool(64, 16)
    pool.alloc("p", 40)
    for k, n in (("a", 101), ("b", 7), ("c", 300)):
        pool.alloc(k, n)
    packer = ChunkPacker(pool, "cpu")
    one = np.zeros(1, np.int32)
    specs = [SeqSpec([("p", 40)], "a", 100, one, 140), SeqSpec([("p", 40)], "b", 6, one, 46),
             SeqSpec([("p", 40)], "c", 0, np.zeros(300, np.int32), 40)]
    assert packer.pack(specs).dkeys == 141
    assert packer.pack(specs[1:2]).dkeys == 47 and packer.pack(specs[2:]).dkeys == 0
