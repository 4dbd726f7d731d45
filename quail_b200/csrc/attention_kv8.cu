// Attention over the 8-bit paged KV cache (kv8.cuh), any head geometry: mma.sync tiles. head_dim 128 with a
// multiple of 4 query heads per KV head goes to the tcgen05 kernel (a 16k-token chunk: 192 us there, 648 here).
//
// For a row with query q over its visible keys, with codes ck, cv and the
// exponents ek, ev of their blocks of 16 tokens:
//   s_j = scale * 2^ek_j * (q . ck_j),  o = sum_j e^(s_j - m) 2^ev_j cv_j / sum_j e^(s_j - m)
// The products run on the codes themselves, which bf16 holds exactly; the K
// exponent multiplies 16 columns of S, the V exponent 16 columns of P before P
// is rounded to bf16 (8 bits of p; the sum of p is taken before that rounding,
// in fp32, as are the maxima and O). One pass over the keys with the running
// maximum and sum of an online softmax.
//
// A CTA of 4 warps takes 64 rows (query token x head of one KV head's group)
// and walks the keys in tiles: the next tile's codes are in registers while
// this one's, converted to bf16 in shared memory once for all 64 rows, feed
// ldmatrix and mma.sync m16n8k16.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <cmath>

#include "kv8.cuh"
#include "mx_common.cuh"

namespace qb {

int* device_error_word(int dev);
void check_pages8(const torch::Tensor& codes, const torch::Tensor& bytes, const char* what);
void prefill_kv8_tc(const Kv8Attn& a, bool fp8, int n, cudaStream_t st, int dev);

namespace {

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(addr));
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(addr));
}
__device__ __forceinline__ void mma_bf16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

}  // namespace

// blocks [n, 2]: (sequence, first query token), 64 tokens each. MX: e4m3 out + UE8M0 atoms, else bf16.
template <int D, bool FP8, bool MX>
__global__ void __launch_bounds__(128) attn_kv8_kernel(const __grid_constant__ Kv8Attn a) {
  constexpr int BK = D == 256 ? 32 : 64;
  constexpr int kRow = 2 * D + 16;                       // bytes of a padded bf16 row
  constexpr int kChunks = BK * D / 16 / 128;             // 16-byte code chunks per thread, of K and of V
  constexpr int kPerRow = D / 16;
  constexpr int NT = BK / 8, DT = D / 8, KS = D / 16;
  extern __shared__ __align__(16) uint8_t smem[];
  uint8_t* sK = smem;
  uint8_t* sV = sK + BK * kRow;
  float* sScale = reinterpret_cast<float*>(sV + BK * kRow);   // [2][BK / 16]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t4 = lane & 3;
  const int kvh = blockIdx.y, G = a.QH / a.KH;

  const int seq = a.blocks[2 * blockIdx.x];
  if ((unsigned)seq >= (unsigned)a.n_seqs) {
    if (tid == 0) kv8_error(a.err, kErrBadShape);
    return;
  }
  Kv8Seq s;
  kv8_load_seq(s, a, seq);
  const int q0 = a.blocks[2 * blockIdx.x + 1];
  if (q0 < 0 || !kv8_rows_ok(s, a.T)) {
    if (tid == 0) kv8_error(a.err, kErrBadShape);
    return;
  }
  const int tokens = min(64, s.q_len - q0);                // of the block
  const int row0 = blockIdx.z * 64;                        // first of this CTA's rows in the block
  if (row0 >= tokens * G) return;
  const int last_row = min(row0 + 64, tokens * G) - 1;
  const int shift = s.own_len - s.q_len + q0;              // own position of the block's first token
  const int pos_first = shift + row0 / G, pos_last = shift + last_row / G;

  // this lane's two rows: token, head, own position
  int tok[2], head[2], pos[2];
  bool valid[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = row0 + warp * 16 + g + 8 * i;
    valid[i] = r <= last_row;
    tok[i] = s.q_start + q0 + r / G;
    head[i] = kvh * G + r % G;
    pos[i] = shift + r / G;
  }
  uint32_t qa[KS][4];
#pragma unroll
  for (int kk = 0; kk < KS; ++kk)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = i & 1;
      const __nv_bfloat16* p = a.q + ((size_t)tok[r] * a.QH + head[r]) * D + kk * 16 + t4 * 2 + (i >> 1) * 8;
      qa[kk][i] = valid[r] ? *reinterpret_cast<const uint32_t*>(p) : 0u;
    }

  const int pshift = __ffs(a.P) - 1, pmask = a.P - 1;
  // tiles [first, end) of a segment that some row of the CTA sees
  auto tiles_of = [&](int seg, int& first, int& end, int& base, int& len, int& off) {
    base = 0;
    len = off = 0;
#pragma unroll
    for (int i = 0; i < kKv8MaxSeg; ++i) {
      if (i < seg) base += s.len[i];
      if (i == seg) {
        len = s.len[i];
        off = s.off[i];
      }
    }
    int lo, hi, lo2, hi2;
    kv8_span(s, seg, len, base, pos_first, lo, hi);
    kv8_span(s, seg, len, base, pos_last, lo2, hi2);
    first = lo / BK;
    end = hi2 > lo ? (hi2 + BK - 1) / BK : first;
  };
  int seg = -1, tile = 0, end = 0, base = 0, len = 0, off = 0;
  auto advance = [&]() -> bool {       // to the next tile; false past the last one
    ++tile;
    while (tile >= end) {
      if (++seg >= s.nseg) return false;
      tiles_of(seg, tile, end, base, len, off);
    }
    return true;
  };

  uint4 rk[kChunks], rv[kChunks];
  int rbyte = 0;
  auto fetch = [&]() {                 // the current tile's codes, and one exponent byte per thread
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const int idx = c * 128 + tid, r = idx / kPerRow, col = idx % kPerRow;
      const int j = tile * BK + r;
      rk[c] = rv[c] = make_uint4(0, 0, 0, 0);
      if (j < len) {
        const int e = off + (j >> pshift);
        const int page = a.page_list[e];
        if ((unsigned)page < (unsigned)a.pages) {
          const size_t at = (((size_t)page * a.KH + kvh) * a.P + (j & pmask)) * D + col * 16;
          rk[c] = *reinterpret_cast<const uint4*>(a.kc + at);
          rv[c] = *reinterpret_cast<const uint4*>(a.vc + at);
        } else {
          kv8_error(a.err, kErrBadShape);
        }
      }
    }
    rbyte = 127;
    if (tid < 2 * (BK / 16)) {
      const int j = tile * BK + (tid % (BK / 16)) * 16;
      const int e = off + (j >> pshift);
      if (j < len) {
        const int page = a.page_list[e];
        if ((unsigned)page < (unsigned)a.pages)
          rbyte = (tid < BK / 16 ? a.kb : a.vb)[((size_t)page * a.KH + kvh) * (a.P / 16) + ((j & pmask) >> 4)];
      }
    }
  };

  float oacc[DT][4];
#pragma unroll
  for (int n = 0; n < DT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) oacc[n][i] = 0.f;
  float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};
  const uint32_t k_s = smem_u32(sK), v_s = smem_u32(sV);

  bool more = advance();
  if (more) fetch();
  while (more) {
    const int j0 = tile * BK, cur_seg = seg, cur_len = len, cur_base = base;
    __syncthreads();                   // the previous tile has been read
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const int idx = c * 128 + tid, r = idx / kPerRow, col = idx % kPerRow;
      const uint32_t wk[4] = {rk[c].x, rk[c].y, rk[c].z, rk[c].w}, wv[4] = {rv[c].x, rv[c].y, rv[c].z, rv[c].w};
      uint4* dk = reinterpret_cast<uint4*>(sK + r * kRow + col * 32);
      uint4* dv = reinterpret_cast<uint4*>(sV + r * kRow + col * 32);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        dk[u] = make_uint4(kv8_lo<FP8>(wk[2 * u]), kv8_hi<FP8>(wk[2 * u]), kv8_lo<FP8>(wk[2 * u + 1]),
                           kv8_hi<FP8>(wk[2 * u + 1]));
        dv[u] = make_uint4(kv8_lo<FP8>(wv[2 * u]), kv8_hi<FP8>(wv[2 * u]), kv8_lo<FP8>(wv[2 * u + 1]),
                           kv8_hi<FP8>(wv[2 * u + 1]));
      }
    }
    if (tid < 2 * (BK / 16))
      sScale[tid] = kv8_scale(rbyte) * ((tid < BK / 16 ? 1.f : kKv8Down) / kv8_unit<FP8>);
    __syncthreads();
    more = advance();
    if (more) fetch();

    float sc[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int i = 0; i < 4; ++i) sc[n][i] = 0.f;
#pragma unroll
      for (int kk = 0; kk < KS; kk += 2) {
        uint32_t b0, b1, b2, b3;
        ldsm4(k_s + (n * 8 + (lane & 7)) * kRow + (kk * 16 + (lane >> 3) * 8) * 2, b0, b1, b2, b3);
        mma_bf16(sc[n], qa[kk], b0, b1);
        mma_bf16(sc[n], qa[kk + 1], b2, b3);
      }
    }
    int lo[2], hi[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      kv8_span(s, cur_seg, cur_len, cur_base, pos[i], lo[i], hi[i]);
      lo[i] -= j0;
      hi[i] = valid[i] ? hi[i] - j0 : 0;
    }
    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float ks = sScale[n >> 1] * a.sl2;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int col = n * 8 + t4 * 2 + (i & 1), r = i >> 1;
        sc[n][i] = col >= lo[r] && col < hi[r] ? sc[n][i] * ks : -INFINITY;
        mx[r] = fmaxf(mx[r], sc[n][i]);
      }
    }
    float corr[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
      mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
      const float mnew = fmaxf(m_run[r], mx[r]);
      corr[r] = m_run[r] == -INFINITY ? 0.f : kv8_ex2(m_run[r] - mnew);
      m_run[r] = mnew;
      l_run[r] *= corr[r];
    }
#pragma unroll
    for (int n = 0; n < DT; ++n) {
      oacc[n][0] *= corr[0];
      oacc[n][1] *= corr[0];
      oacc[n][2] *= corr[1];
      oacc[n][3] *= corr[1];
    }
#pragma unroll
    for (int n = 0; n < NT; n += 2) {
      const float vs = sScale[BK / 16 + (n >> 1)];
      float p[2][4];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int col = (n + u) * 8 + t4 * 2 + (i & 1), r = i >> 1;
          const float x = sc[n + u][i];
          const bool see = col >= lo[r] && col < hi[r];
          const float e = see ? kv8_ex2(x - (m_run[r] == -INFINITY ? 0.f : m_run[r])) : 0.f;
          l_run[r] += e;
          p[u][i] = see ? e * vs : 0.f;
        }
      const uint32_t pa[4] = {pack2(p[0][0], p[0][1]), pack2(p[0][2], p[0][3]), pack2(p[1][0], p[1][1]),
                              pack2(p[1][2], p[1][3])};
#pragma unroll
      for (int d = 0; d < DT; d += 2) {
        uint32_t b0, b1, b2, b3;
        ldsm4_t(v_s + (n * 8 + (lane & 7) + ((lane >> 3) & 1) * 8) * kRow + (d + (lane >> 4)) * 16, b0, b1, b2, b3);
        mma_bf16(oacc[d], pa, b0, b1);
        mma_bf16(oacc[d + 1], pa, b2, b3);
      }
    }
  }

#pragma unroll
  for (int r = 0; r < 2; ++r) {
    float l = l_run[r];
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    const float inv = l == 0.f ? 0.f : kKv8Up / l;   // no visible key: 0; NaN stays NaN
    const size_t row = (size_t)tok[r] * a.QH + head[r];
    if constexpr (!MX) {
      if (valid[r]) {
        __nv_bfloat16* dst = a.o + row * D + t4 * 2;
#pragma unroll
        for (int d = 0; d < DT; ++d)
          *reinterpret_cast<uint32_t*>(dst + d * 8) = pack2(oacc[d][2 * r] * inv, oacc[d][2 * r + 1] * inv);
      }
    } else {
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        float amax = 0.f;
#pragma unroll
        for (int d = 0; d < 4; ++d)
          amax = fmaxf(amax, fmaxf(fabsf(oacc[4 * c + d][2 * r]), fabsf(oacc[4 * c + d][2 * r + 1])) * inv);
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        const uint8_t e = ue8m0_of(amax);
        const float f = ue8m0_inv(e);                // not times inv, which may pass fp32
        if (valid[r]) {
          uint8_t* dst = a.o8 + row * D + c * 32 + t4 * 2;
#pragma unroll
          for (int d = 0; d < 4; ++d)
            *reinterpret_cast<__nv_fp8x2_storage_t*>(dst + d * 8) = __nv_cvt_float2_to_fp8x2(
                make_float2(oacc[4 * c + d][2 * r] * inv * f, oacc[4 * c + d][2 * r + 1] * inv * f), __NV_SATFINITE,
                __NV_E4M3);
          if (t4 == 0) {
            const int col = head[r] * D + c * 32, t = tok[r];
            a.osf[((size_t)(t >> 7) * (a.QH * D / 128) + col / 128) * 512 + (t & 31) * 16 + ((t & 127) >> 5) * 4 +
                  (col % 128) / 32] = e;
          }
        }
      }
    }
    if (a.lse != nullptr && valid[r] && t4 == 0)
      a.lse[row] = l == 0.f ? -INFINITY : (m_run[r] + __log2f(l)) * 0.69314718055994531f;
  }
}

// ------------------------------------------------------------------ host side

template <int D, bool FP8, bool MX>
static void launch_kv8(const Kv8Attn& a, int n, cudaStream_t st, int dev) {
  constexpr int BK = D == 256 ? 32 : 64;
  constexpr int kSmem = 2 * BK * (2 * D + 16) + 2 * (BK / 16) * 4;
  static bool configured[64] = {false};
  if (!configured[dev]) {
    C10_CUDA_CHECK(cudaFuncSetAttribute(attn_kv8_kernel<D, FP8, MX>,
                                        cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
    configured[dev] = true;
  }
  const int G = a.QH / a.KH;
  const dim3 grid(n, a.KH, G);
  attn_kv8_kernel<D, FP8, MX><<<grid, 128, kSmem, st>>>(a);
}

template <bool FP8, bool MX>
static void launch_kv8_d(const Kv8Attn& a, int D, int n, cudaStream_t st, int dev) {
  if (D == 64) return launch_kv8<64, FP8, MX>(a, n, st, dev);
  if (D == 128) return launch_kv8<128, FP8, MX>(a, n, st, dev);
  return launch_kv8<256, FP8, MX>(a, n, st, dev);
}

// Checks shared by the kv8 attentions; fills everything but `blocks`.
Kv8Attn kv8_args(const char* what, const torch::Tensor& q, const torch::Tensor& kc, const torch::Tensor& kb,
                        const torch::Tensor& vc, const torch::Tensor& vb, const torch::Tensor& seqs,
                        const torch::Tensor& page_list, double scale, torch::Tensor& out,
                        const c10::optional<torch::Tensor>& out_sf, const c10::optional<torch::Tensor>& lse) {
  check_pages8(kc, kb, what);
  check_pages8(vc, vb, what);
  TORCH_CHECK(kc.sizes() == vc.sizes() && kc.scalar_type() == vc.scalar_type() && kc.device() == vc.device(), what,
              ": K and V pages alike");
  TORCH_CHECK(q.dim() == 3 && q.is_contiguous() && q.scalar_type() == at::kBFloat16 && q.device() == kc.device(), what,
              ": q [T, QH, D] bf16 beside the pages");
  const int64_t T = q.size(0), QH = q.size(1), D = q.size(2), KH = kc.size(1);
  TORCH_CHECK(D == kc.size(3) && (D == 64 || D == 128 || D == 256), what, ": head_dim 64, 128 or 256, as the pages'");
  TORCH_CHECK(KH > 0 && QH > 0 && QH % KH == 0, what, ": q heads must be a multiple of KV heads");
  // where a page number is out of range the kernels report it and read page 0 instead
  TORCH_CHECK(kc.size(0) > 0, what, ": at least one page");
  TORCH_CHECK(seqs.dim() == 2 && seqs.size(1) == kKv8SeqInts && seqs.scalar_type() == at::kInt &&
                  seqs.is_contiguous() && seqs.device() == q.device() && seqs.size(0) > 0,
              what, ": seqs [S, 12] int32, at least one");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0 && reinterpret_cast<uintptr_t>(out.data_ptr()) % 16 == 0,
              what, ": q and out are 16-byte aligned");
  TORCH_CHECK(page_list.scalar_type() == at::kInt && page_list.is_contiguous() && page_list.device() == q.device(), what,
              ": page_list int32");
  TORCH_CHECK(out.dim() == 2 && out.size(0) == T && out.size(1) == QH * D && out.is_contiguous() &&
                  out.device() == q.device(),
              what, ": out [T, QH*D]");
  // a row's largest score is found before the scale is applied
  TORCH_CHECK(scale >= 0 && std::isfinite((float)(scale * 1.4426950408889634)), what,
              ": the softmax scale is finite and not negative");
  // the kernels sum a sequence's (at most 4) segments, none longer than the list, in 32 bits
  TORCH_CHECK(page_list.numel() <= INT32_MAX / kKv8MaxSeg / kc.size(2), what, ": the page list passes 2^29 tokens");
  Kv8Attn a;
  a.q = reinterpret_cast<const __nv_bfloat16*>(q.data_ptr());
  a.kc = static_cast<const uint8_t*>(kc.data_ptr());
  a.kb = kb.data_ptr<uint8_t>();
  a.vc = static_cast<const uint8_t*>(vc.data_ptr());
  a.vb = vb.data_ptr<uint8_t>();
  a.seqs = seqs.data_ptr<int>();
  a.page_list = page_list.data_ptr<int>();
  a.T = (int)T;
  a.n_seqs = (int)seqs.size(0);
  a.n_list = (int)page_list.numel();
  a.pages = (int)kc.size(0);
  a.P = (int)kc.size(2);
  a.QH = (int)QH;
  a.KH = (int)KH;
  a.sl2 = (float)(scale * 1.4426950408889634);
  a.o = nullptr;
  a.o8 = a.osf = nullptr;
  a.lse = nullptr;
  a.err = device_error_word(q.get_device());
  if (out.scalar_type() == at::kFloat8_e4m3fn) {
    TORCH_CHECK(QH * D % 128 == 0 && out_sf.has_value() && out_sf->scalar_type() == at::kByte &&
                    out_sf->is_contiguous() && out_sf->numel() >= (T + 127) / 128 * (QH * D / 128) * 512,
                what, ": e4m3 output needs its MX scale bytes");
    // the tcgen05 prefill stores a row's four scale bytes as a word
    TORCH_CHECK(out_sf->device() == q.device() && reinterpret_cast<uintptr_t>(out_sf->data_ptr()) % 4 == 0, what,
                ": the MX scale bytes are 4-byte aligned and beside q");
    TORCH_CHECK(!lse.has_value(), what, ": a log-sum-exp output goes with a bf16 out");
    a.o8 = static_cast<uint8_t*>(out.data_ptr());
    a.osf = out_sf->data_ptr<uint8_t>();
  } else {
    TORCH_CHECK(out.scalar_type() == at::kBFloat16, what, ": bf16 or e4m3 output");
    a.o = reinterpret_cast<__nv_bfloat16*>(out.data_ptr());
  }
  if (lse.has_value()) {
    TORCH_CHECK(lse->scalar_type() == at::kFloat && lse->is_contiguous() && lse->numel() >= T * QH &&
                    lse->device() == q.device(),
                what, ": lse fp32 [T, QH]");
    a.lse = lse->data_ptr<float>();
  }
  return a;
}

// blocks [n, 2] int32 (sequence, first token of a 64-token block); rows no block covers are not written
void prefill_attention_kv8(const torch::Tensor& q, const torch::Tensor& kc, const torch::Tensor& kb,
                           const torch::Tensor& vc, const torch::Tensor& vb, const torch::Tensor& seqs,
                           const torch::Tensor& blocks, const torch::Tensor& page_list, double scale,
                           torch::Tensor& out, const c10::optional<torch::Tensor>& out_sf,
                           const c10::optional<torch::Tensor>& lse) {
  const char* what = "prefill_attention_kv8";
  Kv8Attn a = kv8_args(what, q, kc, kb, vc, vb, seqs, page_list, scale, out, out_sf, lse);
  TORCH_CHECK(blocks.dim() == 2 && blocks.size(1) == 2 && blocks.scalar_type() == at::kInt && blocks.is_contiguous() &&
                  blocks.device() == q.device(),
              what, ": blocks [n, 2] int32");
  const int n = (int)blocks.size(0);
  if (n == 0 || a.T == 0) return;
  const int dev = q.get_device();
  c10::cuda::CUDAGuard guard(dev);
  cudaStream_t st = at::cuda::getCurrentCUDAStream(dev);
  a.blocks = blocks.data_ptr<int>();
  const bool fp8 = kc.scalar_type() == at::kFloat8_e4m3fn;
  const int D = (int)q.size(2);
  if (D == 128 && (a.QH / a.KH) % 4 == 0) {
    prefill_kv8_tc(a, fp8, n, st, dev);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
    return;
  }
  if (a.o8 != nullptr)
    fp8 ? launch_kv8_d<true, true>(a, D, n, st, dev) : launch_kv8_d<false, true>(a, D, n, st, dev);
  else
    fp8 ? launch_kv8_d<true, false>(a, D, n, st, dev) : launch_kv8_d<false, false>(a, D, n, st, dev);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

}  // namespace qb
