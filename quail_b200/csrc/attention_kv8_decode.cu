// Decode attention over the 8-bit paged KV cache: the last query token of each
// sequence, all query heads of a KV head together (up to 8 at a time).
//
// What bounds it is the bytes of the codes, so the kernel is built to keep
// loads in flight and to spend few instructions on a code:
//   * Every warp works alone, on a contiguous range of 32-key tiles of the
//     flattened list (sequence, KV head, tile). Ranges are equal, whatever the
//     lengths, so ragged batches and one long sequence alike keep every SM
//     busy to the end; a range that cuts an item leaves a partial result (m,
//     l, O), joined by the second kernel in the order of the ranges (no
//     atomics, the same sum every time).
//   * A warp's tiles arrive by cp.async into its own ring of stages; the next
//     tiles are in flight while it computes, across the ends of items, and it
//     never waits for another warp. Page numbers are read a tile earlier still.
//   * S^T = K Q^T and O^T = V^T P^T with mma.sync m16n8k16: keys (then
//     columns of V) are the 16 rows, heads the 8 columns, so no row of a tile is
//     padding. Which of a row's columns is the k-th of a product is free as
//     long as both operands agree, so a lane takes 16 contiguous codes of a
//     key for K and of four keys for V and pairs them with byte permutes: no
//     transposing load. P^T comes out of S^T by movmatrix, rounded to bf16 (the sum of p is taken before that).
//   * Codes become 16-bit numbers in integer instructions, and the integer
//     pipe, which runs at half rate, is what is scarce: 3 of them for 4 int8
//     codes of K as f16, 4 for V as bf16 (kv8.cuh). K may be f16 because q,
//     scaled per head by the power of two that brings its largest value to
//     [2^14, 2^15), loses nothing but what is below 2^-39 of that. V may not:
//     P 2^e needs more range than f16 has (a column in which the heaviest keys
//     have the code 0 is made of keys of any smaller weight).
//   * A stage's 16-byte chunks are XOR-swizzled by the key so that the 8 lanes
//     of a load's phase meet in no bank, for K and for V.
// tcgen05 has no place here: its 128-row tile would be 8 rows of heads, and
// the codes would have to go through shared memory a second time as f16.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "kv8.cuh"
#include "mx_common.cuh"

namespace qb {

int num_sms(int dev);
Kv8Attn kv8_args(const char* what, const torch::Tensor& q, const torch::Tensor& kc, const torch::Tensor& kb,
                 const torch::Tensor& vc, const torch::Tensor& vb, const torch::Tensor& seqs,
                 const torch::Tensor& page_list, double scale, torch::Tensor& out,
                 const c10::optional<torch::Tensor>& out_sf, const c10::optional<torch::Tensor>& lse);

namespace {

constexpr int kTile = 32;             // keys of a stage: two exponent blocks
constexpr int kHeads = 8;             // query heads of one KV head per item

template <int D>
struct DecGeom {
  static constexpr int kWarps = D == 256 ? 6 : 4;
  static constexpr int kStages = 2;
  static constexpr int kSide = kTile * D;
  static constexpr int kStageBytes = 2 * kSide;                // K, V
  static constexpr int kRing = kWarps * kStages * kStageBytes;
  static constexpr int kBlocksPerSm = D == 64 ? 5 : D == 128 ? 3 : 1;
  static constexpr int kPartial = kHeads * D + 2 * kHeads;     // floats of a partial result: O, m, l
  static constexpr int kFixed = kRing + kWarps * kKv8MaxSeg * 16 + 32;
  // Sequences of one launch: their prefix sums are in shared memory, beside which kBlocksPerSm CTAs still have to
  // fit (228 KB an SM, 1 KB of each CTA's reserved), as the ranges are made for one wave. head_dim 128: 2743.
  static constexpr int kFit = (233472 / kBlocksPerSm - 1024 - kFixed) / 4 - 1;
  static constexpr int kMaxRows = kFit < 4096 ? kFit : 4096;
  static_assert(kBlocksPerSm * (kFixed + (kMaxRows + 1) * 4 + 1024) <= 233472, "a full launch keeps its CTAs an SM");
};

__device__ __forceinline__ uint32_t movm(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
template <bool F16>
__device__ __forceinline__ void mma_dec(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  if constexpr (F16)
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the first product of a sum
__device__ __forceinline__ void mma_dec0(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t pack_bf(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

__device__ __forceinline__ void copy16(uint32_t dst, const uint8_t* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// Place of 16-byte chunk c of key r in a side of a stage (keys of D bytes, 128-byte lines): the chunk's
// index in its line is XORed with bits of the key, so that K loads (two keys 4p, 4p + 1, four neighbouring
// chunks) and V loads (keys 4t + k for t = 0..3, two neighbouring chunks) each touch all 32 banks once.
template <int D>
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
  if constexpr (D == 64) return (r >> 1) * 128 + ((((r & 1) * 4 + c) ^ (((r >> 2) & 3) << 1)) << 4);
  return r * D + (((c & ~7) | ((c ^ ((((r >> 2) ^ ((r & 1) << 1)) & 3) << 1)) & 7)) << 4);
}

// Keys [lo, hi) of segment `seg` the sequence's last token sees.
__device__ __forceinline__ void last_span(const Kv8Seq& s, int seg, int& len, int& off, int& lo, int& hi) {
  int base = 0;
  len = off = 0;
#pragma unroll
  for (int i = 0; i < kKv8MaxSeg; ++i) {
    if (i < seg) base += s.len[i];
    if (i == seg) {
      len = s.len[i];
      off = s.off[i];
    }
  }
  kv8_span(s, seg, len, base, s.own_len - 1, lo, hi);
}

// Tiles of a sequence; at least 1, so that a sequence that sees nothing is written too.
__device__ __forceinline__ int seq_tiles(const Kv8Seq& s) {
  int n = 0;
#pragma unroll
  for (int i = 0; i < kKv8MaxSeg; ++i) {
    if (i >= s.nseg) break;
    int len, off, lo, hi;
    last_span(s, i, len, off, lo, hi);
    if (hi > lo) n += (hi + kTile - 1) / kTile - lo / kTile;
  }
  return max(n, 1);
}

// The row a sequence's output goes to, or -1 (and the error word) when its entry is out of range.
__device__ __forceinline__ int seq_row(const Kv8Attn& a, const Kv8Seq& s) {
  const int row = s.q_start + s.q_len - 1;
  if (s.q_len <= 0) return -1;
  if (s.q_start < 0 || row >= a.T || row < 0) {
    kv8_error(a.err, kErrBadShape);
    return -1;
  }
  return row;
}

__device__ __forceinline__ bool load_dseq(const Kv8Attn& a, int i, Kv8Seq& s) {
  const int seq = a.blocks[i];
  if ((unsigned)seq < (unsigned)a.n_seqs) {
    kv8_load_seq(s, a, seq);
    return true;
  }
  kv8_error(a.err, kErrBadShape);
  s.nseg = 0;
  s.q_start = s.q_len = s.own_len = s.before = s.win = 0;
  s.bidir = s.win_all = false;
#pragma unroll
  for (int k = 0; k < kKv8MaxSeg; ++k) s.len[k] = s.off[k] = 0;
  return false;
}

// An item that several ranges have: what the join needs. Written for every range; i < 0 where the join
// that starts at this range's first tile has nothing to do.
struct Cut {
  int i, hg;                          // sequence and head group
  int w0, w1, per, row;               // first and last range, tiles of a range, output row (-1: none)
  int64_t first, last;                // its tiles [first, last) of the flattened list
};
// Whether all the ranges of the CTA of range w lie in tiles [first, last): it has joined them then.
__device__ __forceinline__ bool cta_inside(int w, int warps, int per, int64_t first, int64_t last) {
  const int64_t x = (int64_t)(w / warps) * warps * per;
  return x >= first && x + (int64_t)warps * per <= last;
}

// One head's D / 32 columns per lane out: bf16, or e4m3 with a UE8M0 byte per 32 columns.
template <int D, bool MX, int N>
__device__ __forceinline__ void emit_cols(const Kv8Attn& a, int row, int head, int col, const float* v, int group_lanes,
                                          int lane_step, bool first) {
  if constexpr (!MX) {
    __nv_bfloat16* dst = a.o + ((size_t)row * a.QH + head) * D + col;
    if constexpr (N == 2) {
      *reinterpret_cast<uint32_t*>(dst) = pack_bf(v[0], v[1]);
    } else if constexpr (N == 4) {
      *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf(v[0], v[1]), pack_bf(v[2], v[3]));
    } else {
#pragma unroll
      for (int i = 0; i < N; i += 8) st_bf16x8(dst + i, v + i);
    }
  } else {
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) amax = fmaxf(amax, fabsf(v[i]));
    for (int x = 1; x < group_lanes; x <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, x * lane_step));
    const uint8_t e = ue8m0_of(amax);
    const float f = ue8m0_inv(e);
    uint8_t* dst = a.o8 + ((size_t)row * a.QH + head) * D + col;
    if (row >= 0) {
#pragma unroll
      for (int i = 0; i < N; i += 2)
        *reinterpret_cast<__nv_fp8x2_storage_t*>(dst + i) =
            __nv_cvt_float2_to_fp8x2(make_float2(v[i] * f, v[i + 1] * f), __NV_SATFINITE, __NV_E4M3);
      if (first) {
        const int c = head * D + col;
        a.osf[((size_t)(row >> 7) * (a.QH * D / 128) + c / 128) * 512 + (row & 31) * 16 + ((row & 127) >> 5) * 4 +
              (c % 128) / 32] = e;
      }
    }
  }
}

}  // namespace

// A lane's 4 codes of a key's column range: two f16 pairs (codes 0, 2 and 1, 3 of the word for int8; 0, 1
// and 2, 3 for e4m3), each two neighbouring k of a product. load_q takes the same columns of Q.
template <bool FP8>
__device__ __forceinline__ void k_pairs(uint32_t w, uint32_t& p0, uint32_t& p1) {
  if constexpr (FP8) {
    p0 = kv8_half2<true>(w);
    p1 = kv8_half2<true>(w >> 16);
  } else {
    p0 = kv8_half2<false>(w);
    p1 = kv8_half2<false>(w >> 8);
  }
}

// Codes of one column range (4 columns) of two keys -> the bf16 pairs (key x, key y) of each column.
template <bool FP8>
__device__ __forceinline__ void v_pairs(uint32_t x, uint32_t y, uint32_t* p) {
  p[0] = kv8_pair<FP8>(__byte_perm(x, y, 0x4400));
  p[1] = kv8_pair<FP8>(__byte_perm(x, y, 0x5511));
  p[2] = kv8_pair<FP8>(__byte_perm(x, y, 0x6622));
  p[3] = kv8_pair<FP8>(__byte_perm(x, y, 0x7733));
}

__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// What the consumer needs to know of a tile in flight.
struct TileInfo {
  int row;         // output row, -1: none
  int hg;          // KV head and head group
  int span;        // first visible key | one past the last << 8 | the item's last tile << 16
  int byte;        // lanes 0..3: exponent bytes K0, K1, V0, V1 of the two blocks
};

// SMALL: pages of 16 tokens, so that a tile is in two pages. ITEM: a CTA per item, its warps sharing
// the item's tiles and joining in shared memory: one launch and no scan over the batch, for few short items.
template <int D, bool FP8, bool MX, bool SMALL, bool ITEM>
__global__ void __launch_bounds__(DecGeom<D>::kWarps * 32, DecGeom<D>::kBlocksPerSm)
    decode_kv8_kernel(const __grid_constant__ Kv8Attn a, int n, int min_tiles, Cut* __restrict__ cuts,
                      float* __restrict__ ws) {
  using Gm = DecGeom<D>;
  constexpr int kWarps = Gm::kWarps, NS = Gm::kStages, KK = D / 16, KCH = D / 64, JT = D / 16;
  extern __shared__ __align__(128) uint8_t smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t4 = lane & 3;
  int4* segs = reinterpret_cast<int4*>(smem + Gm::kRing) + warp * kKv8MaxSeg;     // off, lo, hi, tiles before
  int* scan = reinterpret_cast<int*>(smem + Gm::kRing) + kWarps * kKv8MaxSeg * 4;
  int* prefix = scan + 8;                                                  // [n + 1]

  // tiles before each sequence: every CTA scans the batch itself
  if constexpr (!ITEM) {
    asm volatile("griddepcontrol.launch_dependents;");                     // the join's CTAs may come and wait
    constexpr int kT = kWarps * 32;
#pragma unroll 4
    for (int i = tid; i < n; i += kT) {
      Kv8Seq s;
      load_dseq(a, i, s);
      prefix[i] = seq_tiles(s);
    }
    __syncthreads();
    const int each = (n + kT - 1) / kT;
    int sum = 0;
    for (int k = 0; k < each; ++k)
      if (tid * each + k < n) sum += prefix[tid * each + k];
    int inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += x;
    }
    if (lane == 31) scan[warp] = inc;
    __syncthreads();
    int run = inc - sum;
    for (int w = 0; w < warp; ++w) run += scan[w];
    for (int k = 0; k < each; ++k) {
      const int i = tid * each + k;
      if (i < n) {
        const int t = prefix[i];
        prefix[i] = run;
        run += t;
        if (i == n - 1) prefix[n] = run;
      }
    }
    __syncthreads();
  }

  const int G = a.QH / a.KH, HG = (G + kHeads - 1) / kHeads, KHG = a.KH * HG;
  const int range = blockIdx.x * kWarps + warp;
  int pi = 0, per, count, p_nt, into, phg;
  int64_t x0;
  // ---- the producer's cursor: sequence pi, head group phg, segment ps, tile of the segment
  if constexpr (ITEM) {
    pi = blockIdx.x / KHG;
    phg = blockIdx.x % KHG;
    Kv8Seq s;
    load_dseq(a, pi, s);
    p_nt = seq_tiles(s);
    per = (p_nt + kWarps - 1) / kWarps;
    x0 = into = warp * per;
    count = max(0, min(per, p_nt - into));
  } else {
    const int64_t total = (int64_t)prefix[n] * KHG;
    const int ranges = gridDim.x * kWarps;
    per = (int)max((total + ranges - 1) / ranges, (int64_t)min_tiles);
    x0 = (int64_t)range * per;
    count = (int)max((int64_t)0, min((int64_t)per, total - x0));
    int hi = n;                                                            // prefix[pi] * KHG <= x0 < prefix[hi] * KHG
    while (hi - pi > 1) {
      const int mid = (pi + hi) >> 1;
      if ((int64_t)prefix[mid] * KHG <= x0) pi = mid; else hi = mid;
    }
    p_nt = prefix[pi + 1] - prefix[pi];
    into = (int)((x0 - (int64_t)prefix[pi] * KHG) % p_nt);
    phg = (int)((x0 - (int64_t)prefix[pi] * KHG) / p_nt);
  }
  int p_left = p_nt - into;                                                // tiles of the item from here on
  // the first item's tiles in the flattened list, and whether this CTA is all inside it
  const int64_t item_first = x0 - into, item_last = item_first + p_nt;
  const int hg0 = phg;
  const bool inside = ITEM || (count > 0 && cta_inside(range, kWarps, per, item_first, item_last));
  int row0 = -1;                                                           // the first item's output row
  if (!ITEM && count > 0 && into > 0) {
    Kv8Seq s;
    if (load_dseq(a, pi, s)) row0 = seq_row(a, s);
  }
  if (!ITEM && lane == 0) {
    Cut c;
    c.w0 = (int)(item_first / per);
    c.w1 = (int)((item_last - 1) / per);
    c.i = count > 0 && into > 0 && c.w0 == range - 1 ? pi : -1;
    c.hg = phg;
    c.per = per;
    c.row = c.i >= 0 ? row0 : -1;
    c.first = item_first;
    c.last = item_last;
    cuts[range] = c;
  }
  int p_row = -1, p_nseg = 0, ptile = 0;
  int4 ps = make_int4(0, 0, 0, 0);                                         // the current segment
  auto open = [&]() {                                                      // the sequence's segments into shared memory
    Kv8Seq s;
    load_dseq(a, pi, s);
    p_row = seq_row(a, s);
    p_nseg = s.nseg;
    __syncwarp();
    if (lane < kKv8MaxSeg) {
      int before = 0, len = 0, off = 0, lo = 0, hi = 0;
#pragma unroll
      for (int i = 0; i < kKv8MaxSeg; ++i) {
        if (i > lane || i >= s.nseg) continue;
        before += hi > lo ? (hi + kTile - 1) / kTile - lo / kTile : 0;
        last_span(s, i, len, off, lo, hi);
      }
      if (lane >= s.nseg || hi <= lo) lo = hi = 0;
      segs[lane] = make_int4(off, lo, hi, before);
    }
    __syncwarp();
  };
  auto seek = [&](int t) {                                                 // to the item's tile t
    ps = segs[0];
    for (int i = 1; i < p_nseg; ++i) {
      const int4 x = segs[i];
      if (x.z > x.y && (x.w <= t || ps.z <= ps.y)) ps = x;
    }
    ptile = ps.y / kTile + t - ps.w;
  };

  const uint32_t ring = smem_u32(smem + warp * NS * Gm::kStageBytes);
  const int pshift = __ffs(a.P) - 1, pmask = a.P - 1;
  // a lane's chunk of the first 512 bytes of a side; the others are 512 bytes on, with bits 5 and 6 changed
  constexpr int kRows = 512 / D;                                           // keys a warp's copy covers
  const uint32_t mine = ring + chunk_at<D>(lane / (D / 16), lane % (D / 16));
  const uint8_t *kcl = a.kc + lane * 16, *vcl = a.vc + lane * 16;
  const uint8_t* bytes = lane & 2 ? a.vb : a.kb;
  // the cursor's page (and its second one, if SMALL), looked up a tile ahead
  int page[SMALL ? 2 : 1];
  auto lookup = [&]() {
#pragma unroll
    for (int h = 0; h < (SMALL ? 2 : 1); ++h) {
      const int j = ptile * kTile + h * 16, e = ps.x + (j >> pshift);
      page[h] = 0;
      if (j < ps.z) page[h] = a.page_list[e];
    }
  };
  uint32_t blk[2] = {0, 0};                                                // the cursor's blocks of 16 keys
  int run = 0;                                                             // whole tiles that follow in its page

  // Issue the cursor's tile into stage st, then move the cursor.
  auto issue = [&](int st) -> TileInfo {
    TileInfo info;
    info.row = p_row;
    info.hg = phg;
    info.span = kTile << 8;
    bool second = true, any = true;
    if (run > 0) {
      blk[0] += 2;
      blk[1] = blk[0] + 1;
      --run;
    } else {
      const int j0 = ptile * kTile, left = ps.z - j0;
      any = left > 0;
      second = left > 16;
      info.span = max(ps.y - j0, 0) | max(min(left, kTile), 0) << 8;
#pragma unroll
      for (int h = 0; h < (SMALL ? 2 : 1); ++h) {
        int pg = page[h];
        if ((unsigned)pg >= (unsigned)a.pages) {
          kv8_error(a.err, kErrBadShape);
          pg = 0;
        }
        blk[h] = ((uint32_t)(pg * a.KH + phg / HG) << (pshift - 4)) + (SMALL ? 0 : (j0 & pmask) >> 4);
      }
      if (!SMALL) {
        blk[1] = blk[0] + 1;
        run = max(min(min((a.P - (j0 & pmask)) / kTile, left / kTile), p_left) - 1, 0);
      }
    }
    info.byte = 127;
    const uint32_t to = mine + st * Gm::kStageBytes;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (h == 0 ? any : second) {
        const uint8_t* ks = kcl + (size_t)blk[h] * (16 * D);
        const uint8_t* vs = vcl + (size_t)blk[h] * (16 * D);
#pragma unroll
        for (int i = 0; i < 16 / kRows; ++i) {
          // key i * kRows of the block: what its bits change in the swizzle
          const uint32_t at = to ^ ((((uint32_t)(i * kRows) >> 2) & 3) << 5);
          copy16(at + h * 16 * D + i * 512, ks + i * 512);
          copy16(at + h * 16 * D + i * 512 + Gm::kSide, vs + i * 512);
        }
      }
    }
    if (lane < 4 && (lane & 1 ? second : any)) info.byte = bytes[lane & 1 ? blk[1] : blk[0]];
    asm volatile("cp.async.commit_group;" ::: "memory");
    if (--p_left > 0) {
      ++ptile;
      if (run == 0) {
        if (ptile * kTile >= ps.z) seek(p_nt - p_left);
        lookup();
      }
    } else {
      info.span |= 1 << 16;
      if (ITEM) return info;
      if (++phg == KHG) {
        phg = 0;
        if (++pi < n) {
          p_nt = prefix[pi + 1] - prefix[pi];
          open();
        }
      }
      p_left = p_nt;
      seek(0);
      lookup();
    }
    return info;
  };

  TileInfo queue[NS];                                                      // the tiles in flight, the oldest first
  int issued = 0;
  if (count > 0) {
    open();
    seek(into);
    lookup();
  }
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    if (issued < count) {
      queue[s] = issue(s);
      ++issued;
    } else {
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
  }

  uint32_t qb[KK][2];
  float qs[2];                                                             // scores are the products times this
  float o[JT][4], m[2], l[2];
  bool fresh = true, first_item = true, cut = into != 0;
  int st = 0;
  for (int done = 0; done < count; ++done) {
    const TileInfo ti = queue[0];
    if (fresh) {
      // Q^T columns: head g; in each step the 4 columns lane t4 takes of K
      const int h0 = (ti.hg / HG) * G + (ti.hg % HG) * kHeads;
      const bool have = g < G - (ti.hg % HG) * kHeads && ti.row >= 0;
      const __nv_bfloat16* qp = a.q + ((size_t)max(ti.row, 0) * a.QH + h0 + g) * D + t4 * 16;
      uint2 w[KK];
      uint32_t top = 0;
#pragma unroll
      for (int k = 0; k < KK; ++k) {
        w[k] = make_uint2(0, 0);
        if (have) w[k] = __ldg(reinterpret_cast<const uint2*>(qp + (k >> 2) * 64 + (k & 3) * 4));
      }
#pragma unroll
      for (int k = 0; k < KK; ++k)
        top = max(top, max(max(w[k].x & 0x7fffu, (w[k].x >> 16) & 0x7fffu),
                           max(w[k].y & 0x7fffu, (w[k].y >> 16) & 0x7fffu)));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int ex = (int)(top >> 7);                                      // exponent of the head's largest value
      const int up = ex == 255 || top == 0 ? 127 : min(max(127 + 14 + 127 - ex, 1), 253);
      const float f = __uint_as_float((uint32_t)up << 23);
#pragma unroll
      for (int k = 0; k < KK; ++k) {
        const float c0 = __uint_as_float(w[k].x << 16) * f, c1 = __uint_as_float(w[k].x & 0xffff0000u) * f;
        const float c2 = __uint_as_float(w[k].y << 16) * f, c3 = __uint_as_float(w[k].y & 0xffff0000u) * f;
        qb[k][0] = FP8 ? pack_half(c0, c1) : pack_half(c0, c2);
        qb[k][1] = FP8 ? pack_half(c2, c3) : pack_half(c1, c3);
      }
      const float down = __uint_as_float((uint32_t)(254 - up) << 23);
      qs[0] = __shfl_sync(0xffffffffu, down, t4 * 8) * a.sl2;
      qs[1] = __shfl_sync(0xffffffffu, down, t4 * 8 + 4) * a.sl2;
#pragma unroll
      for (int j = 0; j < JT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[j][i] = 0.f;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        m[i] = -INFINITY;
        l[i] = 0.f;
      }
      fresh = false;
    }
    asm volatile("cp.async.wait_group %0;" ::"n"(NS - 1) : "memory");
    __syncwarp();
    const int lo = ti.span & 0xff, hi = (ti.span >> 8) & 0xff;
    if (hi > lo) {
      const bool full = lo == 0 && hi == kTile;
      const uint8_t* sk = smem + (warp * NS + st) * Gm::kStageBytes;
      const uint8_t* sv = sk + Gm::kSide;
      const float mine_scale = kv8_scale(ti.byte) * (lane & 2 ? kKv8Down / kv8_unit<FP8> : 1.f);
      // row g of a block's product is key kg of the block, row g + 8 key kg + 2
      const int kg = (g >> 1) * 4 + (g & 1);
      float s[2][4];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
#pragma unroll
        for (int u = 0; u < KCH; ++u) {
          const uint8_t* k0 = sk + b * 16 * D + chunk_at<D>(kg, u * 4 + t4);
          const uint4 x = *reinterpret_cast<const uint4*>(k0);
          const uint4 y = *reinterpret_cast<const uint4*>(k0 + 2 * D);
          const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            uint32_t x0p, x1p, y0p, y1p;
            k_pairs<FP8>(xs[w], x0p, x1p);
            k_pairs<FP8>(ys[w], y0p, y1p);
            if (u == 0 && w == 0)
              mma_dec0(s[b], x0p, y0p, x1p, y1p, qb[0][0], qb[0][1]);
            else
              mma_dec<true>(s[b], x0p, y0p, x1p, y1p, qb[u * 4 + w][0], qb[u * 4 + w][1]);
          }
        }
      }
      float f[2][2];                                                       // score units of each block and head
      float mx[2] = {m[0], m[1]};
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const float ks = __shfl_sync(0xffffffffu, mine_scale, b);
        if (!full) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int kx = b * 16 + kg + (i >> 1) * 2;
            if (kx < lo || kx >= hi) s[b][i] = -INFINITY;
          }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          f[b][i] = ks * qs[i];
          mx[i] = fmaxf(mx[i], fmaxf(s[b][i], s[b][i + 2]) * f[b][i]);
        }
      }
      // the maximum of all lanes only where one of them has a larger one
      if (__any_sync(0xffffffffu, mx[0] > m[0] || mx[1] > m[1])) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) {
          mx[0] = fmaxf(mx[0], __shfl_xor_sync(0xffffffffu, mx[0], x));
          mx[1] = fmaxf(mx[1], __shfl_xor_sync(0xffffffffu, mx[1], x));
        }
        float c[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          c[i] = m[i] == -INFINITY ? 0.f : kv8_ex2(m[i] - mx[i]);
          m[i] = mx[i];
          l[i] *= c[i];
        }
#pragma unroll
        for (int j = 0; j < JT; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[j][i] *= c[i & 1];
      }
      const float r[2] = {m[0] == -INFINITY ? 0.f : -m[0], m[1] == -INFINITY ? 0.f : -m[1]};
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const float vs = __shfl_sync(0xffffffffu, mine_scale, 2 + b);
        float p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float e = kv8_ex2(fmaf(s[b][i], f[b][i & 1], r[i & 1]));
          p[i] = e * vs;
          if (!full) {
            const int kx = b * 16 + kg + (i >> 1) * 2;
            if (kx < lo || kx >= hi) e = p[i] = 0.f;                       // also where a scale is NaN
          }
          l[i & 1] += e;
        }
        const uint32_t p0 = movm(pack_bf(p[0], p[1])), p1 = movm(pack_bf(p[2], p[3]));
        constexpr int VW = D == 64 ? 2 : 4;                                // words of a lane's columns per part
#pragma unroll
        for (int u = 0; u < (D == 256 ? 2 : 1); ++u) {
          uint32_t v[4][VW];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            // keys 4 t4 + k: rows 2 t4, 2 t4 + 1, 2 t4 + 8 and 2 t4 + 9 of the product
            const uint8_t* vp = sv + b * 16 * D;
            if constexpr (VW == 2) {
              const uint2 x = *reinterpret_cast<const uint2*>(vp + chunk_at<D>(t4 * 4 + k, g >> 1) + (g & 1) * 8);
              v[k][0] = x.x;
              v[k][1] = x.y;
            } else {
              const uint4 x = *reinterpret_cast<const uint4*>(vp + chunk_at<D>(t4 * 4 + k, u * 8 + g));
              v[k][0] = x.x;
              v[k][1] = x.y;
              v[k][2] = x.z;
              v[k][3] = x.w;
            }
          }
#pragma unroll
          for (int w = 0; w < VW; ++w) {
            uint32_t lo4[4], hi4[4];
            v_pairs<FP8>(v[0][w], v[1][w], lo4);
            v_pairs<FP8>(v[2][w], v[3][w], hi4);
            float(*oj)[4] = &o[u * 8 + 2 * w];
            mma_dec<false>(oj[0], lo4[0], lo4[1], hi4[0], hi4[1], p0, p1);
            mma_dec<false>(oj[1], lo4[2], lo4[3], hi4[2], hi4[3], p0, p1);
          }
        }
      }
    }
    __syncwarp();
    const bool end = (ti.span >> 16) != 0;
    if (end || done == count - 1) {
      const int h0 = (ti.hg / HG) * G + (ti.hg % HG) * kHeads;             // first query head
      const int heads = min(kHeads, G - (ti.hg % HG) * kHeads);
      float ls[2] = {l[0], l[1]};
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) {
        ls[0] += __shfl_xor_sync(0xffffffffu, ls[0], x);
        ls[1] += __shfl_xor_sync(0xffffffffu, ls[1], x);
      }
      const bool whole = !ITEM && end && !cut;
      // where a partial result goes: the CTA's shared memory (this warp's stages, all read) if it joins
      // its own ranges, else the workspace
      float* dst = inside ? reinterpret_cast<float*>(smem + warp * NS * Gm::kStageBytes)
                          : ws + ((size_t)range * 2 + (first_item ? 0 : 1)) * Gm::kPartial;
      constexpr int C = D == 64 ? 8 : 16;                                  // lane g's neighbouring columns of a part
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        const int hl = 2 * t4 + hh;
        const float inv = !whole ? 1.f : ls[hh] == 0.f ? 0.f : kKv8Up / ls[hh];
#pragma unroll
        for (int u = 0; u < (D == 256 ? 2 : 1); ++u) {
          float v[C];
#pragma unroll
          for (int c = 0; c < C; c += 2) {
            v[c] = o[u * 8 + c / 2][hh] * inv;
            v[c + 1] = o[u * 8 + c / 2][2 + hh] * inv;
          }
          const int col = (u * 8 + g) * C;
          if (whole) {
            const bool write = hl < heads && ti.row >= 0;
            if constexpr (MX) {
              emit_cols<D, true, C>(a, write ? ti.row : -1, h0 + hl, col, v, 32 / C, 4, (g % (32 / C)) == 0);
            } else {
              if (write) emit_cols<D, false, C>(a, ti.row, h0 + hl, col, v, 0, 0, false);
            }
          } else if (hl < heads) {
#pragma unroll
            for (int c = 0; c < C; c += 4)
              *reinterpret_cast<float4*>(dst + hl * D + col + c) = make_float4(v[c], v[c + 1], v[c + 2], v[c + 3]);
            if (g == 0 && u == 0) {
              dst[kHeads * D + hl] = m[hh];
              dst[kHeads * D + kHeads + hl] = ls[hh];
            }
          }
        }
        if (whole && a.lse != nullptr && g == 0 && hl < heads && ti.row >= 0)
          a.lse[(size_t)ti.row * a.QH + h0 + hl] =
              ls[hh] == 0.f ? -INFINITY : (m[hh] + __log2f(ls[hh])) * 0.69314718055994531f;
      }
      fresh = true;
      first_item = cut = false;
    }
#pragma unroll
    for (int i = 0; i + 1 < NS; ++i) queue[i] = queue[i + 1];
    if (issued < count) {
      queue[NS - 1] = issue(st);
      ++issued;
    } else {
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
    st = st + 1 == NS ? 0 : st + 1;
  }

  if constexpr (ITEM) {
    // a warp without tiles adds nothing
    if (count == 0) {
      float* dst = reinterpret_cast<float*>(smem + warp * NS * Gm::kStageBytes);
      for (int x = lane; x < Gm::kPartial; x += 32) dst[x] = x >= kHeads * D && x < kHeads * D + kHeads ? -INFINITY : 0.f;
      open();                                                              // for the output row
    }
    __syncthreads();
    const int heads = min(kHeads, G - (hg0 % HG) * kHeads), h0 = (hg0 / HG) * G + (hg0 % HG) * kHeads;
    auto part = [&](int w) { return reinterpret_cast<const float*>(smem + w * NS * Gm::kStageBytes); };
    constexpr int N = D / 32;
    for (int hl = warp; hl < heads; hl += kWarps) {
      float top = -INFINITY, l_ = 0.f, v[N];
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, part(w)[kHeads * D + hl]);
#pragma unroll
      for (int k = 0; k < N; ++k) v[k] = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float mw = part(w)[kHeads * D + hl], c = mw == -INFINITY ? 0.f : kv8_ex2(mw - top);
        l_ += part(w)[kHeads * D + kHeads + hl] * c;
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] += part(w)[hl * D + lane * N + k] * c;
      }
      const float inv = l_ == 0.f ? 0.f : kKv8Up / l_;
#pragma unroll
      for (int k = 0; k < N; ++k) v[k] *= inv;
      if (p_row < 0) break;                                                // alike in the CTA
      emit_cols<D, MX, N>(a, p_row, h0 + hl, lane * N, v, 32 / N, 1, lane % (32 / N) == 0);
      if (a.lse != nullptr && lane == 0)
        a.lse[(size_t)p_row * a.QH + h0 + hl] = l_ == 0.f ? -INFINITY : (top + __log2f(l_)) * 0.69314718055994531f;
    }
  } else if (inside) {                                                     // alike in every warp of the CTA
    __syncthreads();
    const int heads = min(kHeads, G - (hg0 % HG) * kHeads);
    float* dst = ws + (size_t)blockIdx.x * kWarps * 2 * Gm::kPartial;
    auto part = [&](int w) { return reinterpret_cast<const float*>(smem + w * NS * Gm::kStageBytes); };
    for (int x = tid; x < kHeads * D; x += kWarps * 32) {
      const int hl = x / D;
      if (hl >= heads) break;
      float top = -INFINITY, v = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, part(w)[kHeads * D + hl]);
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float mw = part(w)[kHeads * D + hl], c = mw == -INFINITY ? 0.f : kv8_ex2(mw - top);
        v += part(w)[x] * c;
        sum += part(w)[kHeads * D + kHeads + hl] * c;
      }
      dst[x] = v;
      if (x % D == 0) {
        dst[kHeads * D + hl] = top;
        dst[kHeads * D + kHeads + hl] = sum;
      }
    }
  }
}

// Join the partial results of every item that more than one range has: the CTA of the item's second
// range; its warps take a head each, or several share one, and go through the ranges in order.
// (8 warps a CTA; 16 where items are few and each has many ranges: one row of 131k keys 74.9 us with 8, 73.5)
template <int D, bool MX, int kJoinWarps>
__global__ void __launch_bounds__(kJoinWarps * 32)
    decode_kv8_join_kernel(const __grid_constant__ Kv8Attn a, const Cut* __restrict__ cuts,
                           const float* __restrict__ ws) {
  using Gm = DecGeom<D>;
  constexpr int N = D / 32;
  __shared__ float acc[kJoinWarps][D + 2];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Cut c = cuts[blockIdx.x];
  if (c.i < 0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = a.QH / a.KH, HG = (G + kHeads - 1) / kHeads;
  const int heads = min(kHeads, G - (c.hg % HG) * kHeads);
  const int hp = heads <= 1 ? 1 : heads <= 2 ? 2 : heads <= 4 ? 4 : 8, parts = kJoinWarps / hp;
  const int hl = warp % hp, part = warp / hp;
  constexpr int W = Gm::kWarps;
  const int c0 = c.w0 / W, c1 = c.w1 / W;
  auto joined = [&](int cta) { return cta_inside(cta * W, W, c.per, c.first, c.last); };
  // range w's partial result: its first item's unless the item began inside it
  auto at = [&](int w) {
    return ws + ((size_t)w * 2 + ((int64_t)w * c.per < c.first ? 1 : 0)) * Gm::kPartial;
  };
  float v[N], l = 0.f, top = -INFINITY;
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = 0.f;
  if (hl < heads) {
    for (int x = c0 + lane; x <= c1; x += 32) {
      if (joined(x)) {
        top = fmaxf(top, at(x * W)[kHeads * D + hl]);
      } else {
        for (int w = max(c.w0, x * W); w <= min(c.w1, x * W + W - 1); ++w) top = fmaxf(top, at(w)[kHeads * D + hl]);
      }
    }
    top = warp_max(top);
    auto add = [&](int w) {
      const float* p = at(w);
      const float mw = p[kHeads * D + hl], f = mw == -INFINITY ? 0.f : kv8_ex2(mw - top);
      l += p[kHeads * D + kHeads + hl] * f;
      const float* src = p + hl * D + lane * N;
#pragma unroll
      for (int k = 0; k < N; k += 2) {
        const float2 x = *reinterpret_cast<const float2*>(src + k);
        v[k] += x.x * f;
        v[k + 1] += x.y * f;
      }
    };
    // the ends' ranges one by one, the joined CTAs between them in turn
    if (part == 0) {
      for (int x = c0; x <= c1; x = x == c0 && c1 > c0 ? c1 : c1 + 1)
        if (!joined(x))
          for (int w = max(c.w0, x * W); w <= min(c.w1, x * W + W - 1); ++w) add(w);
    }
    const int j0 = c0 + (joined(c0) ? 0 : 1), j1 = c1 - (joined(c1) ? 0 : 1);
#pragma unroll 8
    for (int x = j0 + part; x <= j1; x += parts) add(x * W);
  }
#pragma unroll
  for (int k = 0; k < N; ++k) acc[warp][lane * N + k] = v[k];
  if (lane == 0) acc[warp][D] = l;
  __syncthreads();
  if (part != 0 || hl >= heads) return;
  for (int k = 1; k < parts; ++k) {
    l += acc[hl + k * hp][D];
#pragma unroll
    for (int x = 0; x < N; ++x) v[x] += acc[hl + k * hp][lane * N + x];
  }
  const int row = c.row;
  if (row < 0) return;
  const float inv = l == 0.f ? 0.f : kKv8Up / l;
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] *= inv;
  const int head = (c.hg / HG) * G + (c.hg % HG) * kHeads + hl;
  emit_cols<D, MX, N>(a, row, head, lane * N, v, 32 / N, 1, lane % (32 / N) == 0);
  if (a.lse != nullptr && lane == 0)
    a.lse[(size_t)row * a.QH + head] = l == 0.f ? -INFINITY : (top + __log2f(l)) * 0.69314718055994531f;
}

// ------------------------------------------------------------------ host side

template <int D, bool FP8, bool MX, bool SMALL, bool ITEM>
static void launch_decode_p(const Kv8Attn& a, int n, cudaStream_t st, int dev, const torch::Tensor& like) {
  using Gm = DecGeom<D>;
  constexpr int kMinTiles = 2;
  const int smem = Gm::kFixed + (n + 1) * 4;
  static bool configured[64] = {false};
  if (!configured[dev]) {
    C10_CUDA_CHECK(cudaFuncSetAttribute(decode_kv8_kernel<D, FP8, MX, SMALL, ITEM>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        Gm::kFixed + (Gm::kMaxRows + 1) * 4));
    configured[dev] = true;
  }
  if constexpr (ITEM) {
    const int G = a.QH / a.KH, items = n * a.KH * ((G + kHeads - 1) / kHeads);
    decode_kv8_kernel<D, FP8, MX, SMALL, true><<<items, Gm::kWarps * 32, smem, st>>>(a, n, kMinTiles, nullptr, nullptr);
    return;
  }
  const int grid = num_sms(dev) * Gm::kBlocksPerSm, ranges = grid * Gm::kWarps;
  constexpr int kCutFloats = sizeof(Cut) / 4;
  torch::Tensor ws = torch::empty({(int64_t)ranges * (2 * Gm::kPartial + kCutFloats)}, like.options().dtype(at::kFloat));
  float* part = ws.data_ptr<float>();
  Cut* cuts = reinterpret_cast<Cut*>(part + (int64_t)ranges * 2 * Gm::kPartial);
  decode_kv8_kernel<D, FP8, MX, SMALL, false><<<grid, Gm::kWarps * 32, smem, st>>>(a, n, kMinTiles, cuts, part);
  // the join may be put on the SMs while the first kernel runs; it waits for its end there
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ranges);
  const int G = a.QH / a.KH, items = n * a.KH * ((G + kHeads - 1) / kHeads);
  const bool many = items * 16 <= ranges;
  cfg.blockDim = dim3(many ? 512 : 256);
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, many ? decode_kv8_join_kernel<D, MX, 16> : decode_kv8_join_kernel<D, MX, 8>, a,
                                    (const Cut*)cuts, (const float*)part));
}

template <int D, bool FP8, bool MX>
static void launch_decode(const Kv8Attn& a, int n, bool few_keys, cudaStream_t st, int dev,
                          const torch::Tensor& like) {
  // A CTA per item where they are one wave of CTAs at most and no row has many keys (ops/kv8.py says what the
  // caller knows of that): a row of 1000 keys is 8 tiles for each of its CTA's warps. 32 query and 8 KV heads of
  // 128, in us, so and as equal ranges with a join: 8 rows of 230 keys 13.2, 21.4; of 1000 keys 20.5, 25.6; 55 rows
  // of 1000 keys 37.8, 48.1; but a row of 2000 keys among 7 of 100 29.5, 23.6; of 4000 keys 49.2, 25.6.
  const int G = a.QH / a.KH;
  const int64_t items = (int64_t)n * a.KH * ((G + kHeads - 1) / kHeads);
  const bool item = few_keys && items <= (int64_t)num_sms(dev) * DecGeom<D>::kBlocksPerSm;
  if (item)
    a.P < kTile ? launch_decode_p<D, FP8, MX, true, true>(a, n, st, dev, like)
                : launch_decode_p<D, FP8, MX, false, true>(a, n, st, dev, like);
  else
    a.P < kTile ? launch_decode_p<D, FP8, MX, true, false>(a, n, st, dev, like)
                : launch_decode_p<D, FP8, MX, false, false>(a, n, st, dev, like);
}

// dseqs [n] int32: the sequences whose last query token is read; few_keys: none of them has many keys (a hint)
void decode_attention_kv8(const torch::Tensor& q, const torch::Tensor& kc, const torch::Tensor& kb,
                          const torch::Tensor& vc, const torch::Tensor& vb, const torch::Tensor& seqs,
                          const torch::Tensor& dseqs, const torch::Tensor& page_list, double scale,
                          torch::Tensor& out, const c10::optional<torch::Tensor>& out_sf,
                          const c10::optional<torch::Tensor>& lse, bool few_keys) {
  const char* what = "decode_attention_kv8";
  Kv8Attn a = kv8_args(what, q, kc, kb, vc, vb, seqs, page_list, scale, out, out_sf, lse);
  TORCH_CHECK(dseqs.scalar_type() == at::kInt && dseqs.is_contiguous() && dseqs.device() == q.device(), what,
              ": dseqs int32");
  const int total = (int)dseqs.numel();
  if (total == 0 || a.T == 0) return;
  const int dev = q.get_device();
  c10::cuda::CUDAGuard guard(dev);
  cudaStream_t st = at::cuda::getCurrentCUDAStream(dev);
  const bool fp8 = kc.scalar_type() == at::kFloat8_e4m3fn, mx = a.o8 != nullptr;
  const int D = (int)q.size(2);
  // the tiles of a launch are counted in 32 bits: a row has at most 4 times the page list's
  const int64_t row_tiles = kKv8MaxSeg * ((int64_t)a.n_list * a.P / kTile + 1);
  const int fit = D == 64 ? DecGeom<64>::kMaxRows : D == 128 ? DecGeom<128>::kMaxRows : DecGeom<256>::kMaxRows;
  const int most = (int)std::max<int64_t>(1, std::min<int64_t>(fit, INT32_MAX / row_tiles));
  const int launches = (total + most - 1) / most, each = (total + launches - 1) / launches;
  for (int first = 0; first < total; first += each) {
    const int n = std::min(each, total - first);
    a.blocks = dseqs.data_ptr<int>() + first;
#define QB_DEC8(DD)                                                                                     \
  if (D == DD) {                                                                                        \
    if (fp8)                                                                                            \
      mx ? launch_decode<DD, true, true>(a, n, few_keys, st, dev, q)                                    \
         : launch_decode<DD, true, false>(a, n, few_keys, st, dev, q);                                  \
    else                                                                                                \
      mx ? launch_decode<DD, false, true>(a, n, few_keys, st, dev, q)                                   \
         : launch_decode<DD, false, false>(a, n, few_keys, st, dev, q);                                 \
  }
    QB_DEC8(64)
    QB_DEC8(128)
    QB_DEC8(256)
#undef QB_DEC8
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  }
}

}  // namespace qb
