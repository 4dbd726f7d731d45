"""What the 8-bit KV operators refuse or report because a kernel would otherwise read or write out of range."""

import pytest
import torch

from quail_b200 import ops

pytestmark = pytest.mark.gpu

DEV = "cuda"
I32 = dict(dtype=torch.int32, device=DEV)
GEOMETRIES = [(8, 2, 128), (4, 2, 128), (4, 1, 256)]      # tcgen05 and mma.sync prefill


@pytest.fixture(autouse=True)
def _no_kernel_errors():
    torch.manual_seed(0)
    yield
    assert ops.read_and_clear_error(0) == 0


def one_sequence(QH, KH, D, pages=4, P=16, tokens=6, length=20, kind="int8"):
    kp, vp = (ops.Pages8.zeros(pages, P, KH, D, ops.KV8_DTYPES[kind], DEV) for _ in range(2))
    q = torch.randn(tokens, QH, D, device=DEV).bfloat16()
    seqs = torch.tensor([[0, tokens, 1, 0, length, 0, 0, 0, 0, 0, 0, 0]], **I32)
    return q, kp, vp, seqs, torch.zeros(1, 2, **I32), torch.arange(-(-length // P), **I32)


@pytest.mark.parametrize("QH,KH,D", GEOMETRIES)
def test_a_cache_without_pages_is_refused(QH, KH, D):
    # a key whose page is out of range is reported and page 0 read instead: there has to be one
    q, kp, vp, seqs, blocks, pl = one_sequence(QH, KH, D, pages=0)
    with pytest.raises(RuntimeError, match="at least one page"):
        ops.prefill_attention_kv8(q, kp, vp, seqs, blocks, pl, 0.1)
    with pytest.raises(RuntimeError, match="at least one page"):
        ops.decode_attention_kv8(q, kp, vp, seqs, torch.zeros(1, **I32), pl, 0.1)
    # the write and the read report every slot of it
    rows = torch.randn(2, KH, D, device=DEV).bfloat16()
    ops.kv8_write(rows, rows, torch.tensor([0, 5], **I32), kp, vp)
    assert ops.read_and_clear_error(0) == 5
    k, v = ops.kv8_read(kp, vp, torch.tensor([0, 5], **I32))
    assert ops.read_and_clear_error(0) == 5 and not bool(k.any()) and not bool(v.any())


@pytest.mark.parametrize("QH,KH,D", GEOMETRIES)
def test_scale_bytes_elsewhere_or_unaligned_are_refused(QH, KH, D):
    q, kp, vp, seqs, blocks, pl = one_sequence(QH, KH, D)
    n = ops.sf_bytes(q.shape[0], QH * D)
    dseqs = torch.zeros(1, **I32)
    for sf in (torch.zeros(n, dtype=torch.uint8), torch.zeros(n + 1, dtype=torch.uint8, device=DEV)[1:]):
        with pytest.raises(RuntimeError, match="scale bytes"):
            ops.prefill_attention_kv8(q, kp, vp, seqs, blocks, pl, 0.1, fp8_out=True, out_scale=sf)
        with pytest.raises(RuntimeError, match="scale bytes"):
            ops.decode_attention_kv8(q, kp, vp, seqs, dseqs, pl, 0.1, fp8_out=True, out_scale=sf)


@pytest.mark.parametrize("QH,KH,D", GEOMETRIES)
@pytest.mark.parametrize("start,count", [(2 ** 31 - 4, 6), (1, 2 ** 31 - 1), (2 ** 31 - 1, 2 ** 31 - 1), (3, 6), (-1, 6),
                                         (0, -2 ** 31), (7, 0)])
def test_query_rows_out_of_range_are_reported(QH, KH, D, start, count):
    # also where first row + rows is past 32 bits
    q, kp, vp, seqs, blocks, pl = one_sequence(QH, KH, D)
    seqs[0, 0], seqs[0, 1] = start, count
    out = torch.full((q.shape[0], QH * D), 7.0, dtype=torch.bfloat16, device=DEV)
    ops.prefill_attention_kv8(q, kp, vp, seqs, blocks, pl, 0.1, out=out)
    assert ops.read_and_clear_error(0) == 5 and bool((out == 7).all())
    if count > 0:
        ops.decode_attention_kv8(q, kp, vp, seqs, torch.zeros(1, **I32), pl, 0.1, out=out)
        assert ops.read_and_clear_error(0) == 5 and bool((out == 7).all())


@pytest.mark.parametrize("QH,KH,D", GEOMETRIES)
def test_a_block_before_its_sequence_is_reported(QH, KH, D):
    q, kp, vp, seqs, blocks, pl = one_sequence(QH, KH, D)
    out = torch.full((q.shape[0], QH * D), 7.0, dtype=torch.bfloat16, device=DEV)
    blocks[0, 1] = -64
    ops.prefill_attention_kv8(q, kp, vp, seqs, blocks, pl, 0.1, out=out)
    assert ops.read_and_clear_error(0) == 5 and bool((out == 7).all())


@pytest.mark.parametrize("QH,KH,D", GEOMETRIES)
@pytest.mark.parametrize("length,off", [(33, 0), (2 ** 31 - 1, 0), (2 ** 31 - 1, 1), (17, 1), (1, 2), (20, -1),
                                        (1, -2 ** 31), (20, 2 ** 31 - 1)])
def test_a_segment_past_the_page_list_is_reported_and_empty(QH, KH, D, length, off):
    # its keys would be looked up outside the list, and lengths like these pass 32 bits when summed
    q, kp, vp, seqs, blocks, pl = one_sequence(QH, KH, D)
    for p in (kp, vp):
        p.codes.random_(-127, 128)
        p.bytes.fill_(120)
    seqs[0, 2], seqs[0, 4], seqs[0, 8], seqs[0, 5], seqs[0, 9] = 2, length, off, 20, 0
    alone = seqs.clone()
    alone[0, 2], alone[0, 4], alone[0, 8] = 1, 20, 0
    n = 40
    many = seqs.expand(n, -1).contiguous()
    dseqs = torch.arange(n, **I32)
    got = ops.prefill_attention_kv8(q, kp, vp, seqs, blocks, pl, 0.1)
    assert ops.read_and_clear_error(0) == 5
    want = ops.prefill_attention_kv8(q, kp, vp, alone, blocks, pl, 0.1)
    assert ops.read_and_clear_error(0) == 0 and torch.equal(got, want)
    got = torch.zeros_like(want)
    ops.decode_attention_kv8(q, kp, vp, many, dseqs, pl, 0.1, out=got)
    assert ops.read_and_clear_error(0) == 5
    want = torch.zeros_like(want)
    ops.decode_attention_kv8(q, kp, vp, alone.expand(n, -1).contiguous(), dseqs, pl, 0.1, out=want)
    assert ops.read_and_clear_error(0) == 0 and torch.equal(got, want)


def test_a_page_list_past_32_bit_sums_is_refused():
    q, kp, vp, seqs, blocks, pl = one_sequence(8, 2, 128)
    pl = torch.zeros(2 ** 25 + 1, **I32)
    with pytest.raises(RuntimeError, match="page list"):
        ops.prefill_attention_kv8(q, kp, vp, seqs, blocks, pl, 0.1)
    with pytest.raises(RuntimeError, match="page list"):
        ops.decode_attention_kv8(q, kp, vp, seqs, torch.zeros(1, **I32), pl, 0.1)
    # the largest one allowed: a launch takes as many rows as 32-bit counts of its tiles allow
    pl = torch.zeros(2 ** 25 - 1, **I32)
    n = 100
    out = torch.zeros(q.shape[0], 8 * 128, dtype=torch.bfloat16, device=DEV)
    ops.decode_attention_kv8(q, kp, vp, seqs.expand(n, -1).contiguous(), torch.arange(n, **I32), pl, 0.1, out=out)
    ops.prefill_attention_kv8(q, kp, vp, seqs, blocks, pl, 0.1)
