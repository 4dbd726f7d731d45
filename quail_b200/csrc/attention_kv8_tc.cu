// Packed-prompt attention over the 8-bit paged KV cache on the tcgen05 tensor
// cores: head_dim 128, groups of 4 query heads of one KV head.
//
// One CTA per SM walks a list of work items (64-token query block, group of 4
// heads); the block's 64 tokens x 4 heads are two 128-row query tiles, A and
// B, that read the same K/V tiles of 64 keys. Warp roles (512 threads):
//   warp 0       loader: works out each item's geometry, ahead of the others, which
//                read it from a ring of descriptors; the codes of K and V by bulk
//                copies into a 2-stage ring (a head's tokens of a page are
//                contiguous), the pages and exponents of 8 tiles looked up at a time
//   warp 1       MMA issuer (one thread): S_t(j + 1) = Q_t K^T before
//                O_t += P_t(j) V, with S double-buffered in TMEM, so that a
//                softmax warp finds its next scores waiting
//   warp 2       Q by TMA, brought to L2 while the previous item's is in use
//   warps 4-7    softmax and epilogue of tile A, one thread per row
//   warps 8-11   the same for tile B
//   warps 12-15  converters: codes to bf16 (exactly, kv8.cuh) in the
//                128-byte-swizzled operand layout, 3 stages; and each block's
//                exponents as floats
// The K exponent of a 16-key block scales 16 columns of S: it multiplies the
// block's maximum and is the factor of the multiply-add under 2^x. The V
// exponent is added in that same multiply-add, so p 2^e comes out of 2^x
// itself, is summed (fp32) per block and brought back by 2^-e once a block:
// neither costs an instruction per score.
//
// P is rounded to bf16 (8 bits of p; its sum is taken before that), the heaviest p too, as the maximum may be 2^8
// behind: the error against 64 bits is 0.0022 of the output where its own rounding to bf16 makes 0.0017.
//
// The tensor work is done on 16-bit operands, as for a bf16 cache, because
// 8-bit products would need q and p cut to 8 bits too; what the 8-bit cache
// saves here is its bytes. What bounds the kernel is the softmax: 64 x 256
// exponentials per tile pair at 16 per clock and SM are 1024 cycles, the
// matrix products 1024. They do not overlap fully: without the 2^x the long case takes 15 % less, without the
// conversion 8 %. Letting tile B start half a step after A was slower (1672 us against 1596).
//
// TMEM: S of tile t, buffer b at columns (2 t + b) 64; O of tile t at 256 +
// 128 t. O is rescaled only when a row's maximum grows by more than 2^8.
// Registers: 128 a thread at launch, of which the loader's and the converters' warpgroups keep 88 and 72 and
// the two softmax groups take 176: with 128 the scores spilled (16k-token chunk 244 us, with 176 187; 4096 tokens
// over 12k resident 1591 us and 1325; now 192 and 1341, with the checks of ranges since). One setmaxnreg a warpgroup, before its warps part into roles.
// Every wait is bounded (common.cuh); on expiry a role records an error code
// and stops, and the kernel drains its copies and MMAs before it frees TMEM.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "gemm_sm100.h"
#include "kv8.cuh"
#include "mx_common.cuh"

namespace qb {

int num_sms(int dev);
int* device_error_word(int dev);
CUtensorMap make_tmap_3d_bf16(const void* ptr, int64_t d0, int64_t d1, int64_t d2, int64_t stride1_bytes,
                              int64_t stride2_bytes, int box0, int box1, int box2);

namespace {

constexpr int kRows = 128, kKeys = 64, kD = 128;
constexpr int kRaw = 2, kStages = 3;
constexpr int kQBytes = kRows * 256;           // a tile: two 64-dim atoms of 128 rows
constexpr int kTileBytes = kKeys * 256;        // K or V as bf16: two atoms of 64 rows
constexpr int kRawBytes = 2 * kKeys * kD;      // codes of K, then of V
constexpr int kPBytes = kRows * 128;
constexpr int kScaleFloats = 20;               // per stage: K units [4], V log2 [4], V inverses [4], masks [3], tops [4]
constexpr int kItems = 4;                     // item descriptors in flight
constexpr int kBarBytes = 1024;
constexpr int kSmem = 2 * kQBytes + kStages * 2 * kTileBytes + kRaw * kRawBytes + 2 * kPBytes + kBarBytes + 1024;
constexpr int kThreads = 512;

// Shared-memory operand descriptors (128-byte swizzle, 8 rows of 128 bytes every 1024): the high word is a
// constant, the low word the address / 16 and the leading offset, so that stepping through a tile adds a
// constant to one register. One thread issues every product: what it computes for each is what bounds it.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
constexpr uint32_t kLeadK = 1u << 16;                             // K-major: unused
constexpr uint32_t kLeadV = (uint32_t)(kKeys * 128 >> 4) << 16;   // MN-major: the second 64 columns
__device__ __forceinline__ void umma(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
      "mov.b64 da, {%1, %5};\n\t"
      "mov.b64 db, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d),
      "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(kDescHigh)
      : "memory");
}
constexpr uint32_t idesc_bf16(int M, int N, int b_mn_major) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)b_mn_major << 16) | ((uint32_t)(N >> 3) << 17) |
         ((uint32_t)(M >> 4) << 24);
}

#define QB_TMEM_ST16_K8(taddr, r)                                                                       \
  asm volatile(                                                                                         \
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "                                                   \
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),                         \
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), \
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])                 \
      : "memory")

__device__ __forceinline__ void tma_prefetch_3d(const CUtensorMap* map, int c0, int c1, int c2) {
  asm volatile("cp.async.bulk.prefetch.tensor.3d.L2.global [%0, {%1, %2, %3}];" ::"l"(reinterpret_cast<uint64_t>(map)),
               "r"(c0), "r"(c1), "r"(c2)
               : "memory");
}
// A bounded wait that sleeps between its looks (about `ns` each): for a warp that waits most of the time, whose
// polling would take issue slots from the softmax warps of its quarter of the SM (without it the 16k-token chunk
// takes 191.9 us for 191.2, 4096 tokens over 12k resident 1345 us for 1340).
__device__ __forceinline__ bool mbar_wait_idle(uint64_t* bar, uint32_t parity, int* err, int code, uint32_t ns) {
  const uint32_t addr = smem_u32(bar);
  const long long start = clock64(), budget = wait_budget(err);
  while (!mbar_try_wait(addr, parity)) {
    if (clock64() - start > budget) {
      if (err) atomicCAS(err, 0, code);
      return false;
    }
    __nanosleep(ns);
  }
  return true;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ uint64_t pack_f2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpack_f2(uint64_t x, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(x));
}
__device__ __forceinline__ uint64_t fma_f2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add_f2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint32_t pack_bf2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// p reaches 2^8 (the running maximum may be that far behind), a code 2 (int8) or 2^9 (e4m3), and 2^24 keys may add up
// below 2^128: where the V exponent is above this, the running maximum is taken that much higher.
template <bool FP8>
constexpr int kTopShift = FP8 ? 84 : 92;

// A work item's geometry, as the loader hands it to the other roles.
struct Item {
  int tok, head0;              // first query row and head
  int rows_a, rows_b;          // valid query tokens of tiles A and B
  int pos;                     // own-segment position of the block's first token
  int n_a, n_b;                // K/V tiles each query tile reads; the shorter list is the longer one's beginning
  int pad;
};

}  // namespace

template <bool FP8, bool MX>
__global__ void __launch_bounds__(kThreads, 1)
    prefill_kv8_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ Kv8Attn a, int n_items) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw0 = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw0 + 1023u) & ~1023u) - raw0);
  uint8_t* sQ = smem;                                   // [2][kQBytes]
  uint8_t* sKV = sQ + 2 * kQBytes;                      // [kStages][K, V]
  uint8_t* sP = sKV + kStages * 2 * kTileBytes;         // [2][kPBytes]
  uint8_t* sRaw = sP + 2 * kPBytes;                     // [kRaw][kRawBytes]
  uint64_t* bars = reinterpret_cast<uint64_t*>(sRaw + kRaw * kRawBytes);
  uint64_t* q_full = bars + 0;
  uint64_t* q_empty = bars + 1;
  uint64_t* mma_idle = bars + 2;
  uint64_t* raw_full = bars + 3;                        // [kRaw]
  uint64_t* raw_empty = raw_full + kRaw;                // [kRaw] count 128
  uint64_t* kv_full = raw_empty + kRaw;                 // [kStages] count 128
  uint64_t* kv_empty = kv_full + kStages;               // [kStages]
  uint64_t* s_full = kv_empty + kStages;                // [2][2]: tile, buffer
  uint64_t* p_full = s_full + 4;                        // [2] count 128
  uint64_t* o_done = p_full + 2;                        // [2]
  uint64_t* o_free = o_done + 2;                        // [2] count 128
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_free + 2);
  uint64_t* item_full = bars + 24;                      // [kItems]
  uint64_t* item_empty = item_full + kItems;            // [kItems] count 14: every warp but the loader
  int* raw_info = reinterpret_cast<int*>(bars + 32);    // [kRaw][8]: 4 bytes of K, 4 of V, and the masks' numbers
  float* scales = reinterpret_cast<float*>(bars + 40);  // [kStages][kScaleFloats]
  Item* items = reinterpret_cast<Item*>(bars + 72);     // [kItems]

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int groups = a.QH / 4;
  int* err = a.err;

  if (tid == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    mbar_init(mma_idle, 1);
    for (int i = 0; i < kRaw; ++i) {
      mbar_init(&raw_full[i], 1);
      mbar_init(&raw_empty[i], 128);
    }
    for (int i = 0; i < kItems; ++i) {
      mbar_init(&item_full[i], 1);
      mbar_init(&item_empty[i], 14);
    }
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&kv_full[i], 128);
      mbar_init(&kv_empty[i], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&s_full[2 * t], 1);
      mbar_init(&s_full[2 * t + 1], 1);
      mbar_init(&p_full[t], 128);
      mbar_init(&o_done[t], 1);
      mbar_init(&o_free[t], 128);
    }
    fence_barrier_init();
  }
  if (warp == 1) tmem_alloc<512>(tmem_slot);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  // A warpgroup's registers are set by one setmaxnreg that all of its warps execute: under separate ones in the
  // branches of its warps the instruction is undefined, and the raise to 176 waits for what the others give up.
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == 0) {
      // ------------------------------------------------------------------ loader
      const int pshift = __ffs(a.P) - 1, pmask = a.P - 1;
      int it_raw = 0, idx = 0;
      bool ok = true;
      // (sequence, first token) of the items after this one, and the next one's row, are read ahead
      auto block_of = [&](int item) -> int2 {
        const int* b = a.blocks + 2 * (item / groups);
        return item < n_items ? make_int2(b[0], b[1]) : make_int2(0, 0);
      };
      auto row_of = [&](int seq) { return (unsigned)seq < (unsigned)a.n_seqs ? seq : 0; };
      int2 b0 = block_of(blockIdx.x), b1 = block_of(blockIdx.x + gridDim.x);
      Kv8Seq s;
      kv8_load_seq(s, a, row_of(b0.x));
      for (int item = blockIdx.x; item < n_items && ok; item += gridDim.x, ++idx) {
        const int q0 = b0.y;
        const bool good = (unsigned)b0.x < (unsigned)a.n_seqs && q0 >= 0 && kv8_rows_ok(s, a.T);
        if (!good && lane == 0) kv8_error(err, kErrBadShape);
        Item it;
        it.head0 = item % groups * 4;
        const int kvh = it.head0 / (a.QH / a.KH);
        const int left = good ? s.q_len - q0 : 0;
        it.tok = s.q_start + q0;
        it.rows_a = max(0, min(32, left));
        it.rows_b = max(0, min(32, left - 32));
        it.pos = s.own_len - s.q_len + q0;
        it.n_a = it.n_b = it.pad = 0;
        int before[kKv8MaxSeg], first[kKv8MaxSeg], cum[kKv8MaxSeg];      // keys and tiles before a segment
        {
          int base = 0, n = 0;
  #pragma unroll
          for (int i = 0; i < kKv8MaxSeg; ++i) {
            // the first row reaches furthest back, each tile's last row furthest ahead (earlier segments
            // are seen alike, so only in the last one, the own, do the two tiles' ends differ)
            int lo, hi, lo2, end_a, end_b;
            kv8_span(s, i, s.len[i], base, it.pos, lo, hi);
            kv8_span(s, i, s.len[i], base, it.pos + it.rows_a - 1, lo2, end_a);
            kv8_span(s, i, s.len[i], base, it.pos + 31 + it.rows_b, lo2, end_b);
            const bool there = i < s.nseg;
            const int f = lo / kKeys;
            const int e_a = there && it.rows_a > 0 && end_a > lo ? (end_a + kKeys - 1) / kKeys : f;
            const int e_b = there && it.rows_b > 0 && end_b > lo ? (end_b + kKeys - 1) / kKeys : f;
            before[i] = base;
            first[i] = f;
            cum[i] = n;
            it.n_a += e_a - f;
            it.n_b += e_b - f;
            n += max(e_a, e_b) - f;
            base += s.len[i];
          }
        }
        const int nmax = max(it.n_a, it.n_b);
        // the next item's row, and the block after it: not needed before this item's copies are issued
        const int2 b2 = block_of(item + 2 * gridDim.x);
        Kv8Seq next;
        kv8_load_seq(next, a, row_of(b1.x));
        // 8 tiles at a time: lane 4 k + b looks up block b of tile k
        struct Look {
          uint32_t blk;
          int bytes, x, y, z, blocks;
        };
        auto look = [&](int jb) -> Look {
          Look r;
          r.blk = 0;
          r.bytes = 127 | 127 << 8;
          r.blocks = 0;
          const int j = jb + (lane >> 2);
          int sg = 0;
  #pragma unroll
          for (int i = 1; i < kKv8MaxSeg; ++i)
            if (i < s.nseg && j >= cum[i]) sg = i;
          int len = 0, off = 0, f = 0, base = 0, c = 0;
  #pragma unroll
          for (int i = 0; i < kKv8MaxSeg; ++i)
            if (i == sg) {
              len = s.len[i];
              off = s.off[i];
              f = first[i];
              base = before[i];
              c = cum[i];
            }
          const int j0 = (f + j - c) * kKeys, key = j0 + (lane & 3) * 16, e = off + (key >> pshift);
          const bool own = sg == s.nseg - 1;
          // a row at own position p sees columns [p + z, min(x, p + y)) of the tile
          r.x = len - j0;
          r.y = own && !s.bidir ? 1 - j0 : 1 << 29;
          r.z = s.win > 0 && (own ? !s.bidir : s.win_all) ? s.before - s.win + 1 - base - j0 : -(1 << 30);
          if (j < nmax) {
            r.blocks = min(4, (len - j0 + 15) / 16);       // 16-key blocks of the tile that exist
            if ((lane & 3) < r.blocks) {
              int page = a.page_list[e];
              if ((unsigned)page >= (unsigned)a.pages) {
                kv8_error(err, kErrBadShape);
                page = 0;
              }
              r.blk = ((uint32_t)(page * a.KH + kvh) << (pshift - 4)) + ((key & pmask) >> 4);
              r.bytes = a.kb[r.blk] | (int)a.vb[r.blk] << 8;
            }
          }
          return r;
        };
        Look cur = look(0);
        if (lane == 0) {
          const int sl = idx % kItems;
          ok = mbar_wait(&item_empty[sl], (uint32_t)((idx / kItems) & 1) ^ 1, err, kErrTimeoutProducer);
          if (ok) {
            items[sl] = it;
            mbar_arrive(&item_full[sl]);
          }
        }
        ok = __shfl_sync(0xffffffffu, ok, 0);
        for (int jb = 0; jb < nmax && ok; jb += 8) {
          const Look then = look(jb + 8);
          const int cnt = min(8, nmax - jb);
          for (int k = 0; k < cnt && ok; ++k) {
            const bool mine = (lane >> 2) == k;
            const int at8 = 8 * (lane & 3);
            const uint32_t k4 = __reduce_or_sync(0xffffffffu, mine ? (uint32_t)(cur.bytes & 0xff) << at8 : 0u);
            const uint32_t v4 = __reduce_or_sync(0xffffffffu, mine ? (uint32_t)(cur.bytes >> 8) << at8 : 0u);
            const int blocks = __shfl_sync(0xffffffffu, cur.blocks, 4 * k);
            const int st = it_raw % kRaw;
            if (mine && (lane & 3) == 0) {
              ok = mbar_wait(&raw_empty[st], (uint32_t)((it_raw / kRaw) & 1) ^ 1, err, kErrTimeoutProducer);
              if (ok) {
                int* info = raw_info + 8 * st;
                info[0] = (int)k4;
                info[1] = (int)v4;
                info[2] = cur.x;
                info[3] = cur.y;
                info[4] = cur.z;
                mbar_arrive_expect_tx(&raw_full[st], 2 * blocks * 16 * kD);
              }
            }
            ok = __shfl_sync(0xffffffffu, ok, 4 * k);
            if (!ok) break;
            uint8_t* dst = sRaw + st * kRawBytes + (lane & 3) * 16 * kD;
            // in pages of 64 tokens and more a tile is one run of keys
            if (mine && (lane & 3) < (a.P >= kKeys ? 1 : blocks)) {
              const uint32_t bytes = (a.P >= kKeys ? blocks : 1) * 16 * kD;
              bulk_load(dst, a.kc + (size_t)cur.blk * (16 * kD), bytes, &raw_full[st]);
              bulk_load(dst + kKeys * kD, a.vc + (size_t)cur.blk * (16 * kD), bytes, &raw_full[st]);
            }
            ++it_raw;
          }
          cur = then;
        }
        s = next;
        b0 = b1;
        b1 = b2;
      }
      if (!ok && lane == 0) {
        // stopped early: wait (bounded) for the copies already issued into shared memory
        for (int k = max(0, it_raw - kRaw); k < it_raw; ++k)
          mbar_wait(&raw_full[k % kRaw], (uint32_t)((k / kRaw) & 1), err, kErrTimeoutProducer);
      }
    } else if (warp == 1) {
      // ------------------------------------------------------------------ MMA issuer
      if (elect_one()) {
        constexpr uint32_t IS = idesc_bf16(128, kKeys, 0);
        constexpr uint32_t IO = idesc_bf16(128, kD, 1);
        const uint32_t q_lo = (smem_u32(sQ) >> 4) | kLeadK, kv_lo = (smem_u32(sKV) >> 4) | kLeadK,
                       p_lo = (smem_u32(sP) >> 4) | kLeadK;
        int kv_base = 0, q_it = 0, idx = 0;
        int s_cnt[2] = {0, 0}, p_cnt[2] = {0, 0}, free_cnt[2] = {0, 0};
        bool had[2] = {false, false};
        bool ok = true;
        auto kv_ready = [&](int j) -> bool {
          const int st = (kv_base + j) % kStages;
          if (!mbar_wait(&kv_full[st], (uint32_t)(((kv_base + j) / kStages) & 1), err, kErrTimeoutMma)) return false;
          tc_fence_after();
          return true;
        };
        auto issue_s = [&](int t, int j) {
          const uint32_t qa = q_lo + t * (kQBytes >> 4);
          const uint32_t kb = kv_lo + (uint32_t)((kv_base + j) % kStages) * (2 * kTileBytes >> 4);
          const uint32_t d = tmem + (uint32_t)((2 * t + (s_cnt[t] & 1)) * 64);
  #pragma unroll
          for (int ks = 0; ks < 8; ++ks)
            umma(d, qa + (ks >> 2) * (kRows * 128 >> 4) + (ks & 3) * 2,
                 kb + (ks >> 2) * (kKeys * 128 >> 4) + (ks & 3) * 2, IS, ks > 0 ? 1u : 0u);
          tc_commit(&s_full[2 * t + (s_cnt[t] & 1)]);
          ++s_cnt[t];
        };
        for (int item = blockIdx.x; item < n_items && ok; item += gridDim.x) {
          const int sl = idx % kItems;
          if (!mbar_wait(&item_full[sl], (uint32_t)((idx / kItems) & 1), err, kErrTimeoutMma)) {
            ok = false;
            break;
          }
          ++idx;
          const int nt[2] = {items[sl].n_a, items[sl].n_b};
          mbar_arrive(&item_empty[sl]);
          const int nmax = max(nt[0], nt[1]);
          if (nmax == 0) continue;
          if (!mbar_wait(q_full, (uint32_t)(q_it & 1), err, kErrTimeoutMma)) {
            ok = false;
            break;
          }
          ++q_it;
          tc_fence_after();
          ok = kv_ready(0);
          if (!ok) break;
  #pragma unroll
          for (int t = 0; t < 2; ++t)
            if (nt[t] > 0) issue_s(t, 0);
          if (nmax == 1) tc_commit(q_empty);
          for (int j = 0; j < nmax && ok; ++j) {
            if (j + 1 < nmax) {
              // the other S buffer was read before P(j - 1) was handed over
              ok = kv_ready(j + 1);
              if (!ok) break;
  #pragma unroll
              for (int t = 0; t < 2; ++t)
                if (j + 1 < nt[t]) issue_s(t, j + 1);
              if (j + 2 == nmax) tc_commit(q_empty);
            }
            const int st = (kv_base + j) % kStages;
  #pragma unroll
            for (int t = 0; t < 2; ++t) {
              if (j >= nt[t] || !ok) continue;
              if (!mbar_wait(&p_full[t], (uint32_t)(p_cnt[t] & 1), err, kErrTimeoutMma)) {
                ok = false;
                continue;
              }
              ++p_cnt[t];
              if (j == 0 && had[t]) {
                // the previous item's epilogue has read O_t out of TMEM
                if (!mbar_wait(&o_free[t], (uint32_t)(free_cnt[t] & 1), err, kErrTimeoutMma)) {
                  ok = false;
                  continue;
                }
                ++free_cnt[t];
              }
              tc_fence_after();
              const uint32_t pa = p_lo + t * (kPBytes >> 4);
              const uint32_t vb = kv_lo + (uint32_t)st * (2 * kTileBytes >> 4) + (kTileBytes >> 4) + (kLeadV - kLeadK);
  #pragma unroll
              for (int ks = 0; ks < 4; ++ks)
                umma(tmem + 256u + (uint32_t)(t * 128), pa + ks * 2, vb + ks * (16 * 128 >> 4), IO,
                     (j > 0 || ks > 0) ? 1u : 0u);
              tc_commit(&o_done[t]);
            }
            if (ok) tc_commit(&kv_empty[st]);
          }
          if (!ok) break;
          had[0] = had[0] || nt[0] > 0;
          had[1] = had[1] || nt[1] > 0;
          kv_base += nmax;
        }
        tc_commit(mma_idle);
        mbar_wait(mma_idle, 0, err, kErrTimeoutMma);
      }
    } else if (warp == 2) {
      // ------------------------------------------------------------------ Q
      if (lane == 0) {
        tma_prefetch_desc(&tmQ);
        int q_it = 0, idx = 0;
        bool ok = true;
        for (int item = blockIdx.x; item < n_items; item += gridDim.x, ++idx) {
          const int sl = idx % kItems;
          ok = mbar_wait_idle(&item_full[sl], (uint32_t)((idx / kItems) & 1), err, kErrTimeoutProducer, 200);
          if (!ok) break;
          const int tok = items[sl].tok, head0 = items[sl].head0;
          const bool any = max(items[sl].n_a, items[sl].n_b) > 0;
          mbar_arrive(&item_empty[sl]);
          if (!any) continue;
          tma_prefetch_3d(&tmQ, 0, head0, tok);
          tma_prefetch_3d(&tmQ, 64, head0, tok);
          tma_prefetch_3d(&tmQ, 0, head0, tok + 32);
          tma_prefetch_3d(&tmQ, 64, head0, tok + 32);
          ok = mbar_wait_idle(q_empty, (uint32_t)((q_it & 1) ^ 1), err, kErrTimeoutProducer, 100);
          if (!ok) break;
          mbar_arrive_expect_tx(q_full, 2 * kQBytes);
          tma_load_3d(&tmQ, q_full, sQ, 0, head0, tok);
          tma_load_3d(&tmQ, q_full, sQ + kQBytes / 2, 64, head0, tok);
          tma_load_3d(&tmQ, q_full, sQ + kQBytes, 0, head0, tok + 32);
          tma_load_3d(&tmQ, q_full, sQ + kQBytes + kQBytes / 2, 64, head0, tok + 32);
          ++q_it;
        }
        // stopped early: wait (bounded) for the copies already issued into shared memory
        if (!ok && q_it > 0) mbar_wait(q_full, (uint32_t)((q_it - 1) & 1), err, kErrTimeoutProducer);
      }
    }
  } else if (warp >= 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    // ------------------------------------------------------------------ converters
    const int ct = tid - 384;
    // lane: 16 codes of row ct / 4 (+ 32), columns 16 (ct % 4) (+ 64)
    int cnt = 0, idx = 0;
    bool ok = true;
    for (int item = blockIdx.x; item < n_items && ok; item += gridDim.x) {
      const int sl = idx % kItems;
      ok = mbar_wait(&item_full[sl], (uint32_t)((idx / kItems) & 1), err, kErrTimeoutProducer);
      if (!ok) break;
      ++idx;
      const int tiles = max(items[sl].n_a, items[sl].n_b);
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[sl]);
      for (int j = 0; j < tiles; ++j, ++cnt) {
        const int rs = cnt % kRaw, st = cnt % kStages;
        ok = mbar_wait(&raw_full[rs], (uint32_t)((cnt / kRaw) & 1), err, kErrTimeoutProducer) &&
             mbar_wait(&kv_empty[st], (uint32_t)((cnt / kStages) & 1) ^ 1, err, kErrTimeoutProducer);
        if (!ok) break;
        const uint8_t* src = sRaw + rs * kRawBytes;
        const uint32_t dst = smem_u32(sKV + st * 2 * kTileBytes);
#pragma unroll
        for (int half = 0; half < 2; ++half) {          // K, V
          uint4 w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            w[i] = *reinterpret_cast<const uint4*>(src + half * kKeys * kD + ((ct >> 2) + 32 * (i >> 1)) * kD +
                                                   ((ct & 3) + 4 * (i & 1)) * 16);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = (ct >> 2) + 32 * (i >> 1), c = 2 * (ct & 3);
            const uint32_t at = dst + half * kTileBytes + (i & 1) * (kKeys * 128) + r * 128;
            const uint32_t ws[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
            for (int u = 0; u < 2; ++u)
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at + (((c + u) ^ (r & 7)) << 4)),
                           "r"(kv8_lo<FP8>(ws[2 * u])), "r"(kv8_hi<FP8>(ws[2 * u])), "r"(kv8_lo<FP8>(ws[2 * u + 1])),
                           "r"(kv8_hi<FP8>(ws[2 * u + 1]))
                           : "memory");
          }
        }
        if (ct < 4) {
          const int kb = (raw_info[8 * rs] >> (8 * ct)) & 0xff;
          // a block never written has a byte of 0 and codes of 0: no byte below the smallest that is written,
          // as p 2^(byte - 127) would underflow and the block's share of the sum with it
          const int vb = max((raw_info[8 * rs + 1] >> (8 * ct)) & 0xff, kKv8MinByte);
          float* sc = scales + st * kScaleFloats;
          // never 0 (a softmax scale of 0, a byte of 0): a masked score is -inf, and has to stay that
          sc[ct] = kb == kKv8Nan ? kv8_scale(kb) : fmaxf(kv8_scale(kb) * (a.sl2 / kv8_unit<FP8>), 1.1754943508222875e-38f);
          // p is stored times 2^(vb - 127) / unit
          const int shift = vb - 127 + (FP8 ? 0 : 6);
          sc[4 + ct] = vb == kKv8Nan ? __int_as_float(0x7fc00000) : (float)shift;
          sc[8 + ct] = vb == kKv8Nan ? __int_as_float(0x7fc00000) : scalbnf(1.f, -shift);   // 2^-127 too
          sc[16 + ct] = (float)max(shift - kTopShift<FP8>, 0);
          if (ct < 3) sc[12 + ct] = __int_as_float(raw_info[8 * rs + 2 + ct]);
        }
        fence_proxy_async_smem();
        mbar_arrive(&kv_full[st]);
        mbar_arrive(&raw_empty[rs]);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 176;");
    // ------------------------------------------------------------------ softmax + epilogue
    const int t = (warp - 4) >> 2;                      // tile A (warps 4-7) or B (warps 8-11)
    const int quarter = warp & 3;                       // TMEM lane quarter this warp may access
    const int row = quarter * 32 + lane;
    const int tok = row >> 2, hh = row & 3;
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const uint32_t tO = tmem + lane_base + 256u + (uint32_t)(t * 128);
    const uint32_t p_row = smem_u32(sP + t * kPBytes) + row * 128;
    int s_cnt = 0, o_cnt = 0, kv_base = 0, idx = 0;
    bool ok = true;
    for (int item = blockIdx.x; item < n_items && ok; item += gridDim.x) {
      int n, pos, head, nmax, rows;
      size_t t_out;
      bool valid;
      {
        const int sl = idx % kItems;
        ok = mbar_wait(&item_full[sl], (uint32_t)((idx / kItems) & 1), err, kErrTimeoutEpilogue);
        if (!ok) break;
        ++idx;
        const Item it = items[sl];
        __syncwarp();
        if (lane == 0) mbar_arrive(&item_empty[sl]);
        n = t ? it.n_b : it.n_a;
        nmax = max(it.n_a, it.n_b);
        rows = t ? it.rows_b : it.rows_a;
        valid = tok < rows;
        pos = it.pos + 32 * t + tok;                    // own-segment position
        head = it.head0 + hh;
        t_out = (size_t)it.tok + 32 * t + tok;
      }
      float m_ref = -INFINITY, l = 0.f;
      for (int j = 0; j < n; ++j) {
        const int st = (kv_base + j) % kStages;
        // the stage's scales, then its scores
        if (!mbar_wait(&kv_full[st], (uint32_t)(((kv_base + j) / kStages) & 1), err, kErrTimeoutEpilogue) ||
            !mbar_wait(&s_full[2 * t + (s_cnt & 1)], (uint32_t)((s_cnt >> 1) & 1), err, kErrTimeoutEpilogue)) {
          ok = false;
          break;
        }
        const uint32_t tS = tmem + lane_base + (uint32_t)((2 * t + (s_cnt & 1)) * 64);
        ++s_cnt;
        tc_fence_after();
        uint32_t sv[64];
        QB_TMEM_LD32(tS, sv);
        QB_TMEM_LD32(tS + 32, (sv + 32));
        const float4 kf = *reinterpret_cast<const float4*>(scales + st * kScaleFloats);
        const float4 vf = *reinterpret_cast<const float4*>(scales + st * kScaleFloats + 4);
        const float4 vi = *reinterpret_cast<const float4*>(scales + st * kScaleFloats + 8);
        const float kfs[4] = {kf.x, kf.y, kf.z, kf.w}, vfs[4] = {vf.x, vf.y, vf.z, vf.w};
        const float vis[4] = {vi.x, vi.y, vi.z, vi.w};
        const float4 vt = *reinterpret_cast<const float4*>(scales + st * kScaleFloats + 16);
        const float vts[4] = {vt.x, vt.y, vt.z, vt.w};
        const int4 mk = *reinterpret_cast<const int4*>(scales + st * kScaleFloats + 12);
        const int lo = pos + mk.z, end = valid ? min(mk.x, pos + mk.y) : 0;
        const int hi = end > lo ? end : 0;              // a window may end before its tile's first key, or after its last
        const bool full = __all_sync(0xffffffffu, lo <= 0 && hi >= kKeys);
        tmem_ld_wait();
        if (!full) {
#pragma unroll
          for (int i = 0; i < 64; ++i)
            if (i < lo || i >= hi) sv[i] = 0xff800000u;               // -inf
        }
        float tmax = -INFINITY;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const uint32_t* x = sv + 16 * b;
          float y[5];
#pragma unroll
          for (int i = 0; i < 5; ++i)
            y[i] = max3(__uint_as_float(x[3 * i]), __uint_as_float(x[3 * i + 1]), __uint_as_float(x[3 * i + 2]));
          const float z = max3(max3(y[0], y[1], y[2]), max3(y[3], y[4], __uint_as_float(x[15])), -INFINITY);
          tmax = fmaxf(tmax, fmaf(z, kfs[b], vts[b]));
        }
        float corr = 1.f;
        if (tmax > m_ref + 8.f) {
          corr = (m_ref == -INFINITY) ? 0.f : kv8_ex2(m_ref - tmax);
          m_ref = tmax;
        }
        if (j > 0) {
          // P_{j-1} V_{j-1} is done: the P buffer is free and O is stable
          if (!mbar_wait(&o_done[t], (uint32_t)(o_cnt & 1), err, kErrTimeoutEpilogue)) {
            ok = false;
            break;
          }
          ++o_cnt;
          tc_fence_after();
          if (__any_sync(0xffffffffu, corr != 1.f)) {
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              uint32_t ov[16];
              QB_TMEM_LD16(tO + c * 16, ov);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * corr);
              QB_TMEM_ST16_K8(tO + c * 16, ov);
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
          }
        }
        l *= corr;
        const float mref = (m_ref == -INFINITY) ? 0.f : m_ref;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          // a block the row sees nothing of has only -inf: its scales, which may be anything, are not used
          const bool seen = 16 * b < hi && 16 * b + 16 > lo;
          const float mul = seen ? kfs[b] : 1.f, add = seen ? vfs[b] - mref : 0.f;
          const uint64_t f2 = pack_f2(mul, mul), a2 = pack_f2(add, add);
          uint64_t sum = 0;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int e = 16 * b + 8 * h + 2 * i;
              float p0, p1;
              unpack_f2(fma_f2(pack_f2(__uint_as_float(sv[e]), __uint_as_float(sv[e + 1])), f2, a2), p0, p1);
              p0 = kv8_ex2(p0);
              p1 = kv8_ex2(p1);
              sum = add_f2(sum, pack_f2(p0, p1));
              w[i] = pack_bf2(p0, p1);
            }
            const uint32_t dst = p_row + (((2 * b + h) ^ (row & 7)) << 4);
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                         "r"(w[3])
                         : "memory");
          }
          float s0, s1;
          unpack_f2(sum, s0, s1);
          s0 += s1;
          if (seen) l += s0 * vis[b];
        }
        fence_proxy_async_smem();
        tc_fence_before();
        mbar_arrive(&p_full[t]);
      }
      kv_base += nmax;
      if (!ok) break;
      if (n > 0) {
        if (!mbar_wait(&o_done[t], (uint32_t)(o_cnt & 1), err, kErrTimeoutEpilogue)) {
          ok = false;
          break;
        }
        ++o_cnt;
        tc_fence_after();
      }
      // ---- epilogue: O / l (rows that see no key: 0)
      const float inv = l == 0.f ? 0.f : 1.f / l;
      // A warp's 32 rows go through its part of the (now unused) P buffer, 128 bytes of each at a time, so
      // that a store writes whole rows of 128 bytes. Rows 4 k .. 4 k + 3 are a token's 4 heads.
      {
        uint32_t word = 0;
        uint8_t* stage = sP + t * kPBytes + quarter * 32 * 128;
        auto flush = [&](uint8_t* out, size_t row_bytes, int col) {
          __syncwarp();
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int r = 4 * k + (lane >> 3);
            const uint4 x = *reinterpret_cast<const uint4*>(stage + r * 128 + (((lane & 7) ^ (r & 7)) << 4));
            if (quarter * 8 + k < rows)
              *reinterpret_cast<uint4*>(out + ((t_out - tok + quarter * 8 + k) * a.QH + head - hh + (r & 3)) * row_bytes +
                                        col + (lane & 7) * 16) = x;
          }
          __syncwarp();
        };
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t ov[32];
          if (n > 0) {
            QB_TMEM_LD32(tO + c * 32, ov);
            tmem_ld_wait();
          }
          float v[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = n == 0 || l == 0.f ? 0.f : __uint_as_float(ov[i]) * inv;
          if constexpr (!MX) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              st_bf16x8(reinterpret_cast<__nv_bfloat16*>(stage + lane * 128 + ((((c & 1) * 4 + i) ^ (lane & 7)) << 4)),
                        v + 8 * i);
            if (c & 1) flush(reinterpret_cast<uint8_t*>(a.o), 256, (c >> 1) * 128);
          } else {
            float amax = 0.f;
#pragma unroll
            for (int i = 0; i < 32; ++i) amax = fmaxf(amax, fabsf(v[i]));
            const uint8_t e = ue8m0_of(amax);
            const float sc = ue8m0_inv(e);
            word |= (uint32_t)e << (8 * c);
#pragma unroll
            for (int i = 0; i < 32; i += 16) {
              __align__(16) __nv_fp8x4_e4m3 pk[4];
#pragma unroll
              for (int k = 0; k < 4; ++k)
                pk[k] = __nv_fp8x4_e4m3(make_float4(v[i + 4 * k] * sc, v[i + 4 * k + 1] * sc, v[i + 4 * k + 2] * sc,
                                                    v[i + 4 * k + 3] * sc));
              *reinterpret_cast<uint4*>(stage + lane * 128 + (((2 * c + i / 16) ^ (lane & 7)) << 4)) =
                  *reinterpret_cast<const uint4*>(pk);
            }
            if (c == 3) flush(a.o8, 128, 0);
          }
        }
        if constexpr (MX) {
          if (valid)
            *reinterpret_cast<uint32_t*>(a.osf + ((t_out >> 7) * a.QH + head) * 512 + (t_out & 31) * 16 +
                                         ((t_out & 127) >> 5) * 4) = word;
        }
        if (a.lse != nullptr && valid)
          a.lse[t_out * a.QH + head] = l == 0.f ? -INFINITY : (m_ref + __log2f(l)) * 0.69314718055994531f;
      }
      if (n > 0) {
        tc_fence_before();
        mbar_arrive(&o_free[t]);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc<512>(tmem);
  }
}

// ------------------------------------------------------------------ host side

template <bool FP8, bool MX>
static void launch_tc(const CUtensorMap& tq, const Kv8Attn& a, int n_items, int grid, cudaStream_t st, int dev) {
  static bool configured[64] = {false};
  if (!configured[dev]) {
    C10_CUDA_CHECK(cudaFuncSetAttribute(prefill_kv8_tc_kernel<FP8, MX>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        kSmem));
    configured[dev] = true;
  }
  prefill_kv8_tc_kernel<FP8, MX><<<grid, kThreads, kSmem, st>>>(tq, a, n_items);
}

// head_dim 128 and a multiple of 4 query heads per KV head; a.blocks: n 64-token blocks
void prefill_kv8_tc(const Kv8Attn& a, bool fp8, int n, cudaStream_t st, int dev) {
  // Q: dims {128, QH, T}, box {64, 4, 32}
  const CUtensorMap tq = make_tmap_3d_bf16(a.q, kD, a.QH, a.T, 256, (int64_t)a.QH * 256, 64, 4, 32);
  const int items = n * (a.QH / 4), grid = std::min(items, num_sms(dev));
  if (a.o8 != nullptr)
    fp8 ? launch_tc<true, true>(tq, a, items, grid, st, dev) : launch_tc<false, true>(tq, a, items, grid, st, dev);
  else
    fp8 ? launch_tc<true, false>(tq, a, items, grid, st, dev) : launch_tc<false, false>(tq, a, items, grid, st, dev);
}

}  // namespace qb
