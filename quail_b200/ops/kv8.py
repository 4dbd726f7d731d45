"""The 8-bit KV cache: pages of codes with an exponent byte per 16 tokens and head.

A layer's K (or V) is a `Pages8`: `codes` [pages, KH, P, D] int8 or e4m3 and
`bytes` [pages, KH, P / 16] uint8; a value is code * 2^(byte - 127). Half the
memory of the bf16 arena (a byte and 1/2048 of one per value at head_dim 128
against two), so twice the documents stay resident, and decode attention
reads half the bytes. int8 codes keep 7 bits under a block's largest value;
e4m3 codes keep 4 significant bits of every value, which suits keys with a few
very wide channels.

Kernels: csrc/kv8_cache.cu (write, read, page copies), csrc/attention_kv8_tc.cu
and csrc/attention_kv8.cu (prefill), csrc/attention_kv8_decode.cu; layout and
conversions in csrc/kv8.cuh. Sequence tables, blocks,
dseqs and page lists are those of the bf16 attentions (engine/chunk.py).
"""

from __future__ import annotations

import torch

from quail_b200.ops import kernels as K

KV8_BLOCK = 16                            # tokens that share an exponent byte
KV8_DTYPES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
KV8_HEAD_DIMS = frozenset({64, 128, 256})
KV8_FEW_KEYS = 1024                       # up to this many keys a row, few rows take a CTA per row and KV head


class Pages8:
    """One layer's K or V pages in 8 bits (the tensors are the arena's, not copies)."""

    __slots__ = ("codes", "bytes")

    def __init__(self, codes: torch.Tensor, bytes: torch.Tensor):
        self.codes = codes
        self.bytes = bytes

    @classmethod
    def zeros(cls, num_pages: int, page_tokens: int, kv_heads: int, head_dim: int, dtype=torch.int8,
              device="cuda") -> "Pages8":
        check_kv8(dtype, page_tokens, head_dim)
        return cls(torch.zeros(num_pages, kv_heads, page_tokens, head_dim, dtype=dtype, device=device),
                   torch.zeros(num_pages, kv_heads, page_tokens // KV8_BLOCK, dtype=torch.uint8, device=device))

    @property
    def num_pages(self) -> int:
        return self.codes.shape[0]

    @property
    def kv_heads(self) -> int:
        return self.codes.shape[1]

    @property
    def page_tokens(self) -> int:
        return self.codes.shape[2]

    @property
    def head_dim(self) -> int:
        return self.codes.shape[3]

    @property
    def dtype(self) -> torch.dtype:
        return self.codes.dtype


def check_kv8(dtype, page_tokens: int, head_dim: int) -> None:
    """Refuse a geometry the 8-bit cache is not built for."""
    if dtype not in KV8_DTYPES.values():
        raise ValueError(f"8-bit KV pages are int8 or float8_e4m3fn, not {dtype}")
    if head_dim not in KV8_HEAD_DIMS:
        raise ValueError(f"8-bit KV pages: head_dim {head_dim} is not built; built: {sorted(KV8_HEAD_DIMS)}")
    if page_tokens < KV8_BLOCK or page_tokens & (page_tokens - 1):
        raise ValueError(f"8-bit KV pages hold a power of two of at least {KV8_BLOCK} tokens, not {page_tokens}")


def _check_heads(what: str, q: torch.Tensor, pages: Pages8) -> None:
    if q.dim() != 3 or q.shape[2] != pages.codes.shape[3] or q.shape[2] not in KV8_HEAD_DIMS:
        raise ValueError(f"{what}: q {tuple(q.shape)} over pages of head_dim {pages.codes.shape[3]}; "
                         f"built: {sorted(KV8_HEAD_DIMS)}")
    if q.shape[1] % pages.codes.shape[1]:
        raise ValueError(f"{what}: {q.shape[1]} q heads over {pages.codes.shape[1]} KV heads")


def kv8_write(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, k_pages: Pages8, v_pages: Pages8) -> None:
    """Quantize rows k, v [T, KH, D] (bf16, fp16 or fp32, any token and head strides) into the cache.

    slots int32 [T]: page * P + offset, -1 to skip a row. The rows of one 16-token block are
    adjacent in the call (a sequence's new tokens in order are), with fewer than 16 skipped
    rows between them. A block's exponent grows to what its largest value needs, and the
    codes of all its other rows are rescaled (rounded once); a write at a block's offset 0
    begins it anew, and its other rows are lost. A value that is not finite marks its block:
    attention over it gives NaN.
    """
    K.count_launch()
    K.native().kv8_write(k, v, slots, k_pages.codes, k_pages.bytes, v_pages.codes, v_pages.bytes)


def kv8_read(k_pages: Pages8, v_pages: Pages8, slots: torch.Tensor, k_out=None, v_out=None):
    """The cached values of slots int32 [n] (-1: zeros): (k, v) bf16 [n, KH, D]."""
    n = slots.numel()
    _, KH, _, D = k_pages.codes.shape
    if k_out is None:
        k_out = torch.empty(n, KH, D, dtype=torch.bfloat16, device=slots.device)
    if v_out is None:
        v_out = torch.empty(n, KH, D, dtype=torch.bfloat16, device=slots.device)
    K.count_launch()
    K.native().kv8_read(k_pages.codes, k_pages.bytes, v_pages.codes, v_pages.bytes, slots, k_out, v_out)
    return k_out, v_out


def _outputs(q, fp8_out, out, out_scale):
    T, QH, D = q.shape
    if out is None:
        out = torch.empty(T, QH * D, dtype=torch.float8_e4m3fn if fp8_out else torch.bfloat16, device=q.device)
    if fp8_out and out_scale is None:
        out_scale = torch.empty(K.sf_bytes(T, QH * D), dtype=torch.uint8, device=q.device)
    return out, out_scale


def prefill_attention_kv8(q, k_pages: Pages8, v_pages: Pages8, seqs, blocks, page_list, softmax_scale: float, *,
                          fp8_out: bool = False, out=None, out_scale=None, lse=None):
    """Attention of packed prompts over the 8-bit cache -> [T, QH * D].

    blocks [m, 2] int32: (sequence, first query token) per 64-token block (a chunk's `blocks`);
    rows no block covers are not written. Returns bf16, or with fp8_out (e4m3, UE8M0 scale bytes
    in the MX atom layout). A row that sees no key is 0 (and -inf in `lse`, fp32 [T, QH], which
    goes with a bf16 output). softmax_scale is finite and at least 0.
    """
    _check_heads("prefill_attention_kv8", q, k_pages)
    out, out_scale = _outputs(q, fp8_out, out, out_scale)
    K.count_launch()
    K.native().prefill_attention_kv8(q, k_pages.codes, k_pages.bytes, v_pages.codes, v_pages.bytes, seqs, blocks,
                                     page_list, softmax_scale, out, out_scale, lse)
    return (out, out_scale) if fp8_out else out


def _few_keys(rows: int, listed: int, page_tokens: int, max_keys: int | None) -> bool:
    """Whether no row of a decode has many keys, by what the host knows.

    Without `max_keys`, by the page list: the rows' average, and what one row can have of it, as
    every other row has a page of its own there. That bound is several times what most rows have,
    so it may be six times as large: the worst case, one row of 5900 keys among short ones, takes
    67 us for 26, while 4 to 40 rows of 60 to 250 keys take 10 to 19 us for 17 to 27.
    """
    if max_keys is not None:
        return max_keys <= KV8_FEW_KEYS
    return listed <= rows * KV8_FEW_KEYS // page_tokens and (listed - rows + 1) * page_tokens <= 6 * KV8_FEW_KEYS


def decode_attention_kv8(q, k_pages: Pages8, v_pages: Pages8, seqs, dseqs, page_list, softmax_scale: float, *,
                         fp8_out: bool = False, out=None, out_scale=None, lse=None, max_keys: int | None = None):
    """Attention of the last query token of the sequences dseqs int32 [n] over the 8-bit cache.

    Outputs as prefill_attention_kv8; only those tokens' rows are written. `max_keys`: the most
    keys one of the rows reads, where the caller knows it. It changes the time and the order of
    fp32 sums, not what is computed.
    """
    _check_heads("decode_attention_kv8", q, k_pages)
    out, out_scale = _outputs(q, fp8_out, out, out_scale)
    if dseqs.numel():
        K.count_launch()
        K.native().decode_attention_kv8(q, k_pages.codes, k_pages.bytes, v_pages.codes, v_pages.bytes, seqs, dseqs,
                                        page_list, softmax_scale, out, out_scale, lse,
                                        _few_keys(dseqs.numel(), page_list.numel(), k_pages.page_tokens, max_keys))
    return (out, out_scale) if fp8_out else out


def kv_copy_pages(pools, src: torch.Tensor, dst: torch.Tensor) -> None:
    """Copy whole pages inside an arena, in every layer's K and V, in one launch.

    pools: tensors [layers, 2, pages, ...] of one arena (codes and exponent bytes, or bf16 pages);
    src, dst int32 [n]: page dst[i] becomes a copy of page src[i] in each of them. No page is in
    both lists and none is twice in dst (KVArena's fork, unshare and compact keep to that).
    """
    if src.numel():
        K.count_launch()
        K.native().kv_copy_pages(list(pools), src, dst)


_ROWS: dict = {}      # device -> [0, 1, ...] tensors, the largest last (all kept: graphs may read them)


def _row_numbers(n: int, device) -> torch.Tensor:
    have = _ROWS.setdefault(device, [])
    if not have or have[-1].numel() < n:
        have.append(torch.arange(max(n, 16384), dtype=torch.int32, device=device))
        torch.cuda.current_stream(device).synchronize()      # other streams may read it
    return have[-1][:n]


def qk_norm_rope_kv8(qkv, positions, q_norm_w, k_norm_w, cos_sin, slots, k_pages: Pages8, v_pages: Pages8,
                     num_q_heads: int, num_kv_heads: int, eps: float):
    """ops.qk_norm_rope_kv into 8-bit pages (head_dim 128): per-head q/k RMSNorm and NeoX RoPE, q returned
    as [T, QH, 128]; k and v rows (bf16) quantized into the slots' blocks. An fp8 model's Q, K and V come
    here rounded to bf16, which its GEMM's fused epilogue (for bf16 pages) norms and rotates in fp32: a
    block's exponent needs all its rows, so K and V cannot be written from that epilogue."""
    T = qkv.shape[0]
    q = torch.empty(T, num_q_heads, 128, dtype=torch.bfloat16, device=qkv.device)
    # k and v as pages of one token each, row t in page t, then into the cache
    k = torch.empty(T, 1, num_kv_heads, 128, dtype=torch.bfloat16, device=qkv.device)
    v = torch.empty_like(k)
    rows = _row_numbers(T, qkv.device)
    K.qk_norm_rope_kv(qkv, positions, q_norm_w, k_norm_w, cos_sin, rows, k, v, num_q_heads, num_kv_heads, eps,
                      q_out=q)
    kv8_write(k[:, 0], v[:, 0], slots, k_pages, v_pages)
    return q


def chunk_attention_kv8(q, k_pages: Pages8, v_pages: Pages8, chunk, softmax_scale: float, *, mx: bool, out=None,
                        out_scale=None):
    """ops.chunk_attention over 8-bit pages; a chunk with a tree is read in two passes merged by their
    log-sum-exps, as there."""
    T, QH, D = q.shape
    tree = getattr(chunk, "tree", None)
    dseqs, dkeys = getattr(chunk, "dseqs", None), getattr(chunk, "dkeys", None)
    if tree is not None and chunk.tiles.shape[0] > 0:
        o_a = torch.empty(T, QH * D, dtype=torch.bfloat16, device=q.device)
        lse_a = torch.empty(T, QH, dtype=torch.float32, device=q.device)
        prefill_attention_kv8(q, k_pages, v_pages, tree["seqs_a"], tree["blocks_a"], chunk.page_list, softmax_scale,
                              out=o_a, lse=lse_a)
        if dseqs is not None:
            decode_attention_kv8(q, k_pages, v_pages, chunk.seqs, dseqs, chunk.page_list, softmax_scale, out=o_a,
                                 max_keys=dkeys)
        rows = tree["rows"]
        o_b = torch.empty(rows.numel(), QH * D, dtype=torch.bfloat16, device=q.device)
        lse_b = torch.empty(rows.numel(), QH, dtype=torch.float32, device=q.device)
        prefill_attention_kv8(q.index_select(0, rows.long()), k_pages, v_pages, tree["seqs_b"], tree["blocks_b"],
                              chunk.page_list, softmax_scale, out=o_b, lse=lse_b)
        return K.attention_merge(o_a, lse_a, o_b, lse_b, tree["source"], fp8_out=mx, out=out, out_scale=out_scale)
    out, out_scale = _outputs(q, mx, out, out_scale)
    if chunk.tiles.shape[0] > 0:
        prefill_attention_kv8(q, k_pages, v_pages, chunk.seqs, chunk.blocks, chunk.page_list, softmax_scale,
                              fp8_out=mx, out=out, out_scale=out_scale)
    if dseqs is not None:
        decode_attention_kv8(q, k_pages, v_pages, chunk.seqs, dseqs, chunk.page_list, softmax_scale, fp8_out=mx,
                             out=out, out_scale=out_scale, max_keys=dkeys)
    return (out, out_scale) if mx else out
