"""8-bit KV operators on values, scales and masks at the ends of their ranges, against the 64-bit statements
(bounds as in test_kv8_gpu.py)."""

import math

import pytest
import torch

from quail_b200 import ops
from quail_b200.ops import reference as ref
from test_kv8_gpu import DEV, KINDS, blocks_of, check_rows, layout, random_pages, write_both

pytestmark = pytest.mark.gpu

GEOMETRIES = [(8, 2, 128), (16, 2, 128), (4, 2, 128), (4, 1, 256), (4, 4, 64)]      # tcgen05 and mma.sync prefill
TOP = {d: torch.finfo(d).max for d in (torch.bfloat16, torch.float32)}


@pytest.fixture(autouse=True)
def _no_kernel_errors():
    torch.manual_seed(0)
    yield
    assert ops.read_and_clear_error(0) == 0


# ------------------------------------------------------------------ write and read
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_the_largest_finite_values_stay_finite(kind, dtype):
    P, KH, D = 16, 2, 128
    kp, vp = (ops.Pages8.zeros(3, P, KH, D, ops.KV8_DTYPES[kind], DEV) for _ in range(2))
    rows = torch.randn(32, KH, D, device=DEV).to(dtype)
    rows[3, 0, 5], rows[4, 0, 6], rows[20, 1, 0] = TOP[dtype], -TOP[dtype], 3.38e38
    rows[5, 0] = 0
    slots = torch.arange(32, dtype=torch.int32, device=DEV)
    write_both(rows, -rows, slots, kp, vp)
    k, v = ops.kv8_read(kp, vp, slots)
    assert bool(torch.isfinite(k).all()) and bool(torch.isfinite(v).all()) and not bool(k[5, 0].any())
    # int8: half a step of 2^(byte - 127), a whole one for fp32 values past 127.5 of them; e4m3: 4 significant bits
    # and steps of 2^-9, and its largest value below 2^128 is 1.875 * 2^127
    step = torch.exp2(kp.bytes[:2].double() - 127).permute(0, 2, 1).repeat_interleave(16, dim=1).reshape(32, KH, 1)
    x = rows.double()
    bound = (0.5 if dtype == torch.bfloat16 else 1.0) * step if kind == "int8" else x.abs() * 2 ** -4 + step * 2 ** -10
    assert bool(((k.double() - x).abs() <= bound).all()) and bool(((v.double() + x).abs() <= bound).all())


@pytest.mark.parametrize("kind", KINDS)
def test_a_row_written_before_kept_rows_of_its_block_leaves_their_values(kind):
    P, KH, D = 16, 2, 128
    for first in (1, 3, 14):
        kp, vp = (ops.Pages8.zeros(3, P, KH, D, ops.KV8_DTYPES[kind], DEV) for _ in range(2))
        ones = torch.ones(16, KH, D, device=DEV).bfloat16()
        write_both(ones, ones, torch.arange(16, 32, dtype=torch.int32, device=DEV), kp, vp)
        big = 8 * ones[:1]
        write_both(big, -big, torch.tensor([16 + first], dtype=torch.int32, device=DEV), kp, vp)
        k, v = ops.kv8_read(kp, vp, torch.arange(16, 32, dtype=torch.int32, device=DEV))
        want = torch.ones(16, KH, D, device=DEV).bfloat16()
        want[first] = 8
        assert torch.equal(k, want)
        want[first] = -8
        assert torch.equal(v, want)


# ------------------------------------------------------------------ attention
def both(q, kp, vp, seqs, pl, scale):
    """Prefill and decode against the statement; decode once as few short rows and once over a long page list."""
    lse = torch.empty(q.shape[0], q.shape[1], device=DEV)
    out = ops.prefill_attention_kv8(q, kp, vp, seqs, blocks_of(seqs), pl, scale, lse=lse)
    check_rows(out, lse, q, kp, vp, seqs, pl, scale)
    dseqs = torch.arange(seqs.shape[0], dtype=torch.int32, device=DEV)
    last = (seqs[:, 0] + seqs[:, 1] - 1).long()
    for table in (pl, torch.cat([pl, pl.new_zeros(8192)])):
        dec = torch.zeros_like(out)
        ops.decode_attention_kv8(q, kp, vp, seqs, dseqs, table, scale, out=dec, lse=lse)
        check_rows(dec, lse, q, kp, vp, seqs, pl, scale, last)
    return out


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("QH,KH,D", GEOMETRIES)
@pytest.mark.parametrize("top", [2.0 ** 100, 2.0 ** 122, 3.38e38])
def test_attention_over_large_values(kind, QH, KH, D, top):
    # the mean of values near the largest number is finite, though their sum is not, nor p 2^8 times one of them
    # (a running maximum may be that far behind)
    P, pages = 64, 16
    kp, vp = (ops.Pages8.zeros(pages, P, KH, D, ops.KV8_DTYPES[kind], DEV) for _ in range(2))
    seqs, pl, T = layout([(70, [200, 70]), (3, [130]), (1, [1])], P, pages)
    n = 200 + 70 + 130 + 1
    g = torch.arange(n, device=DEV).view(-1, 1, 1) % 200
    k = (0.3 + 0.004 * g + 0.01 * torch.rand(n, KH, D, device=DEV)).bfloat16()          # scores grow slowly
    v = (top * (0.6 + 0.4 * torch.rand(n, KH, D, device=DEV))).clamp(max=TOP[torch.bfloat16]).bfloat16()
    v[::7] = -v[::7]
    v[1::2] *= 2.0 ** -30
    order = []
    for row in seqs.tolist():
        for i in range(row[2]):
            order += [int(pl[row[8 + i] + j // P]) * P + j % P for j in range(row[4 + i])]
    slots = torch.tensor(order, dtype=torch.int32, device=DEV)
    ops.kv8_write(k, v, slots, kp, vp)
    q = (0.5 + torch.rand(T, QH, D, device=DEV)).bfloat16()
    out = both(q, kp, vp, seqs, pl, 1 / math.sqrt(D))
    assert bool(torch.isfinite(out).all())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("QH,KH,D", GEOMETRIES)
def test_attention_over_blocks_never_written(kind, QH, KH, D):
    # zeros with an exponent byte of 0: keys and values of 0, in and beyond a causal mask's edge
    P, pages = 64, 16
    kp, vp = random_pages(pages, KH, P, D, kind, 41), random_pages(pages, KH, P, D, kind, 42)
    seqs, pl, T = layout([(100, [30, 100]), (20, [90, 20]), (1, [70])], P, pages)
    q = torch.randn(T, QH, D, device=DEV).bfloat16()
    for blank in ([0, 1, 2, 3], [1]):
        for p in (kp, vp):
            for e in pl.tolist():
                p.codes[e, :, :].view(torch.uint8).view(KH, P // 16, 16, D)[:, blank] = 0
                p.bytes[e][:, blank] = 0
        both(q, kp, vp, seqs, pl, 0.1)
        kp, vp = random_pages(pages, KH, P, D, kind, 43), random_pages(pages, KH, P, D, kind, 44)


@pytest.mark.parametrize("QH,KH,D", GEOMETRIES)
def test_a_softmax_scale_of_zero_is_the_mean(QH, KH, D):
    P, pages = 64, 12
    kp, vp = random_pages(pages, KH, P, D, "int8", 45), random_pages(pages, KH, P, D, "int8", 46)
    seqs, pl, T = layout([(100, [30, 100]), (1, [70])], P, pages)
    q = torch.randn(T, QH, D, device=DEV).bfloat16()
    both(q, kp, vp, seqs, pl, 0.0)
    both(q, kp, vp, seqs, pl, 1e-30)


def test_a_softmax_scale_that_is_negative_or_not_finite_is_refused():
    P, pages, QH, KH, D = 64, 12, 8, 2, 128
    kp, vp = random_pages(pages, KH, P, D, "int8", 45), random_pages(pages, KH, P, D, "int8", 46)
    seqs, pl, T = layout([(100, [30, 100]), (1, [70])], P, pages)
    q = torch.randn(T, QH, D, device=DEV).bfloat16()
    for scale in (-0.1, float("nan"), float("inf"), 1e39):
        with pytest.raises(RuntimeError, match="scale"):
            ops.prefill_attention_kv8(q, kp, vp, seqs, blocks_of(seqs), pl, scale)
        with pytest.raises(RuntimeError, match="scale"):
            ops.decode_attention_kv8(q, kp, vp, seqs, torch.zeros(1, dtype=torch.int32, device=DEV), pl, scale)


@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("QH,KH,D", GEOMETRIES)
def test_a_window_that_leaves_a_block_leaves_what_it_holds(which, QH, KH, D):
    # rows 7 to 12 see nothing of the 10-token segment before them, though their window ends in its block
    P, pages = 64, 12
    kp, vp = random_pages(pages, KH, P, D, "int8", 47), random_pages(pages, KH, P, D, "int8", 48)
    seqs, pl, T = layout([(64, [10, 64]), (40, [75, 40])], P, pages, flags=(8 << 8) | (1 << 24))
    for e in (int(pl[0]), int(pl[3])):
        (kp if which == "k" else vp).bytes[e, 0, 0] = 255
    q = torch.randn(T, QH, D, device=DEV).bfloat16()
    want, _ = ref.segmented_attention_kv8(q, kp, vp, seqs, pl, 0.1, torch.float64)
    out = ops.prefill_attention_kv8(q, kp, vp, seqs, blocks_of(seqs), pl, 0.1)
    assert torch.equal(torch.isnan(out.double()), torch.isnan(want))
    assert bool(torch.isnan(out[:7]).any(dim=1).all()) and not bool(torch.isnan(out[7:64]).any())


def test_decode_of_more_rows_than_one_launch_takes():
    P, QH, KH, D, n = 16, 4, 1, 128, 2900
    specs = [(1, [1 + (7 * i) % 37]) for i in range(n)]
    pages = sum(-(-ln // P) for _, (ln,) in specs)
    kp, vp = random_pages(pages, KH, P, D, "int8", 49), random_pages(pages, KH, P, D, "int8", 50)
    seqs, pl, T = layout(specs, P, pages)
    q = torch.randn(T, QH, D, device=DEV).bfloat16()
    dseqs = torch.randperm(n, device=DEV).int()
    lse = torch.empty(T, QH, device=DEV)
    out = ops.decode_attention_kv8(q, kp, vp, seqs, dseqs, pl, 0.1, lse=lse)
    check_rows(out, lse, q, kp, vp, seqs, pl, 0.1)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("QH,KH,D", GEOMETRIES)
def test_decode_gives_the_same_whatever_is_said_of_its_rows(kind, QH, KH, D):
    # a hint that is too small or too large changes the time only; a long row among short ones, a padded list
    P, pages = 16, 250
    kp, vp = random_pages(pages, KH, P, D, kind, 51), random_pages(pages, KH, P, D, kind, 52)
    seqs, pl, T = layout([(1, [48, 30]), (1, [48, 2500]), (1, [48, 1]), (1, [48, 600])], P, pages, prefix_shared=True)
    q = torch.randn(T, QH, D, device=DEV).bfloat16()
    dseqs = torch.arange(4, dtype=torch.int32, device=DEV)
    for table in (pl, torch.cat([pl, pl.new_zeros(5000)])):
        for most in (None, 1, 2548, 1 << 40):
            lse = torch.empty(T, QH, device=DEV)
            out = ops.decode_attention_kv8(q, kp, vp, seqs, dseqs, table, 0.1, lse=lse, max_keys=most)
            check_rows(out, lse, q, kp, vp, seqs, pl, 0.1)
