"""The 8-bit KV cache's statements at the ends of their range."""

import pytest
import torch

from quail_b200.ops import KV8_DTYPES, Pages8
from quail_b200.ops import reference as ref


@pytest.mark.parametrize("kind", ["int8", "fp8"])
def test_every_finite_value_is_stored_as_a_bf16_number(kind):
    dtype = KV8_DTYPES[kind]
    x = torch.tensor([torch.finfo(torch.float32).max, torch.finfo(torch.bfloat16).max, 2.0 ** 127 * 127 / 64,
                      2.0 ** 127 * 1.875, 2.0 ** 127, 3.3e38, 1.0, 0.0])
    p = Pages8.zeros(1, 16, 1, 64, dtype, "cpu")
    rows = torch.zeros(8, 1, 64)
    rows[:, 0, 0], rows[:, 0, 1] = x, -x
    ref.kv8_write(rows, torch.arange(8, dtype=torch.int32), p.codes, p.bytes)
    got = ref.kv8_values(p.codes, p.bytes)[0, :8, 0]
    assert bool((got.abs() < 2.0 ** 128).all()) and torch.equal(got, got.float().bfloat16().double())
    assert torch.equal(got[:, 0], -got[:, 1])
    top = 2.0 ** 127 * (127 / 64 if kind == "int8" else 1.875)
    assert got[0, 0] == got[1, 0] == top and got[4, 0] == 2.0 ** 127


@pytest.mark.parametrize("kind", ["int8", "fp8"])
def test_a_row_written_before_kept_rows_of_its_block_leaves_their_values(kind):
    p = Pages8.zeros(1, 16, 2, 64, KV8_DTYPES[kind], "cpu")
    ref.kv8_write(torch.ones(16, 2, 64), torch.arange(16, dtype=torch.int32), p.codes, p.bytes)
    ref.kv8_write(torch.full((1, 2, 64), 8.0), torch.tensor([3], dtype=torch.int32), p.codes, p.bytes)
    want = torch.ones(16, 2, 64, dtype=torch.float64)
    want[3] = 8
    assert torch.equal(ref.kv8_values(p.codes, p.bytes)[0], want)


@pytest.mark.parametrize("name,device,chunk", [("qwen3-4b-fp8", "b200", None), ("qwen3-8b-bf16", "b200", None),
                                               ("qwen3-32b-fp8", "b200", None), ("qwen3-4b-fp8", "b200", 65_536),
                                               ("qwen3-32b-fp8", "h100-sxm", 65_536), ("qwen3-tiny", "cpu", None)])
def test_the_engines_arena_of_8_bit_pages_holds_twice_the_tokens(name, device, chunk, monkeypatch):
    from quail_b200.models.config import MODEL_CONFIGS
    from quail_b200.planner.budgets import Budgets
    monkeypatch.delenv("QUAIL_KV_POOL_TOKENS", raising=False)
    cfg = MODEL_CONFIGS[name]

    def pages(kv):
        return Budgets.for_model(cfg, device, chunk_tokens=chunk, kv_dtype=kv).arena_pages(128)
    # a byte and 1/16 of one per head_dim values against two, both rounded down to whole pages
    ratio = 2 / (1 + 1 / (16 * cfg.head_dim))
    for kind in ("int8", "fp8"):
        assert abs(pages(kind) - ratio * pages("bf16")) <= ratio + 1


def test_unshare_refuses_a_place_the_key_does_not_have():
    from quail_b200.engine.arena import PagePool
    p = PagePool(8, 16)
    p.alloc("p", 32)
    assert p.fork("p", "c") == []
    for tokens in (-1, 33):
        with pytest.raises(ValueError, match="tokens"):
            p.unshare("c", tokens)
        p.check()
    assert len(p.unshare("c", 31)) == 1
    p.check()


@pytest.mark.parametrize("kind", ["int8", "fp8"])
def test_infinity_beside_nan_marks_its_block_too(kind):
    p = Pages8.zeros(1, 16, 3, 64, KV8_DTYPES[kind], "cpu")
    rows = torch.ones(4, 3, 64)
    rows[1, 0, 5], rows[2, 1, 6] = float("nan"), float("-inf")
    ref.kv8_write(rows, torch.arange(4, dtype=torch.int32), p.codes, p.bytes)
    assert p.bytes[0, :, 0].tolist() == [255, 255, 121 if kind == "int8" else 119]
