// The 8-bit KV cache's data movement: the quantizing write of new rows, the
// read back of rows, and the copy of whole pages (of any cache).
//
// Write. A block (16 tokens of one head) has one exponent byte, so the unit of
// work is a run: the call's rows of one block, which are adjacent in the call
// (but for fewer than 16 skipped rows among them).
// One warp owns a run of K or of V of one head: it takes the largest magnitude
// (an integer max over |x| bits), grows the block's byte if it has to, rescales
// the block's other codes when the byte grew, and writes the new codes.
// No two warps touch one block, so there are no atomics and the result does not
// depend on timing. Bound by the bytes: each row is read (bf16) and half as
// many bytes are written.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_fp16.h>

#include "kv8.cuh"

namespace qb {

int num_sms(int dev);
int* device_error_word(int dev);

namespace {

template <typename T>
__device__ __forceinline__ float to_f32(T x) {
  return static_cast<float>(x);
}

// a lane's N values of a row; VEC: one aligned load
template <typename T, int N, bool VEC>
__device__ __forceinline__ void load_vals(const T* p, float* v) {
  if constexpr (VEC) {
    constexpr int kBytes = N * (int)sizeof(T);
    __align__(16) T raw[N];
    if constexpr (kBytes == 4) {
      *reinterpret_cast<uint32_t*>(raw) = __ldg(reinterpret_cast<const uint32_t*>(p));
    } else if constexpr (kBytes == 8) {
      *reinterpret_cast<uint2*>(raw) = __ldg(reinterpret_cast<const uint2*>(p));
    } else {
#pragma unroll
      for (int i = 0; i < kBytes / 16; ++i)
        reinterpret_cast<uint4*>(raw)[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = to_f32(raw[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = to_f32(p[i]);
  }
}

template <typename T, int N>
struct __align__(N * sizeof(T)) Raw {
  T v[N];
};
template <typename T, int N>
__device__ __forceinline__ Raw<T, N> ldg_raw(const T* p) {
  Raw<T, N> r;
  if constexpr (N * sizeof(T) == 4)
    *reinterpret_cast<uint32_t*>(&r) = __ldg(reinterpret_cast<const uint32_t*>(p));
  else if constexpr (N * sizeof(T) == 8)
    *reinterpret_cast<uint2*>(&r) = __ldg(reinterpret_cast<const uint2*>(p));
  else if constexpr (N * sizeof(T) == 16)
    *reinterpret_cast<uint4*>(&r) = __ldg(reinterpret_cast<const uint4*>(p));
  return r;
}

template <bool FP8>
__device__ __forceinline__ uint8_t encode(float y) {
  if constexpr (FP8) {
    return (uint8_t)__nv_cvt_float_to_fp8(y, __NV_SATFINITE, __NV_E4M3);
  } else {
    return (uint8_t)(int8_t)__float2int_rn(y);
  }
}

template <bool FP8>
__device__ __forceinline__ float decode(uint8_t c) {
  if constexpr (FP8) {
    __nv_fp8_e4m3 f;
    f.__x = c;
    return static_cast<float>(f);
  } else {
    return (float)(int8_t)c;
  }
}

template <int N>
struct Codes {
  uint8_t c[N];
};

template <int N>
__device__ __forceinline__ void store_codes(uint8_t* p, const uint8_t* c) {
  if constexpr (N == 2) *reinterpret_cast<uint16_t*>(p) = *reinterpret_cast<const uint16_t*>(c);
  if constexpr (N == 4) *reinterpret_cast<uint32_t*>(p) = *reinterpret_cast<const uint32_t*>(c);
  if constexpr (N == 8) *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(c);
}

struct WriteArgs {
  const void* x[2];        // K rows, V rows
  int64_t st[2], sh[2];    // their token and head strides, in elements
  uint8_t* codes[2];
  uint8_t* bytes[2];
  const int* slots;
  int T, KH, P;
  int64_t slots_total;
  int* err;
};

}  // namespace

// GROUP tokens per warp: 1 (few rows: every row's own warp) or 16 (a packed
// chunk: at most two runs begin in 16 adjacent rows of one sequence).
// Four CTAs an SM are kept up to head_dim 128 (the compiler's own 136 registers leave three: write and read of 16k
// tokens 81 us, with four 73); at 256 the rows held would spill.
template <typename T, int D, bool FP8, bool VEC, int GROUP>
__global__ void __launch_bounds__(128, D == 256 ? 1 : 4) kv8_write_kernel(const __grid_constant__ WriteArgs a) {
  constexpr int N = D / 32;
  const int lane = threadIdx.x & 31;
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int side = (int)(unit & 1);
  const int64_t rest = unit >> 1;
  const int h = (int)(rest % a.KH);
  const int64_t t0 = rest / a.KH * GROUP;
  if (t0 >= a.T) return;
  // slots of rows t0 - 32 .. t0 + 63: a run begins in the group and ends within 32 rows of its first
  auto slot_at = [&](int64_t t) -> int {
    const int x = t >= 0 && t < a.T ? a.slots[t] : -1;
    if (x < a.slots_total) return x;
    kv8_error(a.err, kErrBadShape);
    return -1;
  };
  const int slot = slot_at(t0 + lane), slot2 = GROUP == 1 ? -1 : slot_at(t0 + 32 + lane);
  const int blk = slot >= 0 ? slot / kKv8Block : -1, blk2 = slot2 >= 0 ? slot2 / kKv8Block : -1;
  const int back = slot_at(t0 - 32 + lane);
  const int blk0 = back >= 0 ? back / kKv8Block : -1;
  const uint32_t there = __ballot_sync(0xffffffffu, blk >= 0), there0 = __ballot_sync(0xffffffffu, blk0 >= 0);
  // the block of the last kept row before this lane's: skipped rows do not end a run
  const uint32_t below = there & ((1u << lane) - 1);
  const int in_group = __shfl_sync(0xffffffffu, blk, below ? 31 - __clz(below) : 0);
  const int in_back = __shfl_sync(0xffffffffu, blk0, there0 ? 31 - __clz(there0) : 0);
  const int prev = below ? in_group : there0 ? in_back : -1;
  uint32_t leaders = __ballot_sync(0xffffffffu, blk >= 0 && blk != prev) & (GROUP == 1 ? 1u : 0xffffu);
  const T* x = static_cast<const T*>(a.x[side]) + h * a.sh[side] + lane * N;
  const int per = a.P / kKv8Block;
  while (leaders) {
    const int l0 = __ffs(leaders) - 1;
    leaders &= leaders - 1;
    const int b = __shfl_sync(0xffffffffu, blk, l0);
    // bit i: row t0 + l0 + i is one of the run's (up to the first kept row of another block)
    auto window = [&](bool lo, bool hi) -> uint32_t {
      const uint32_t w0 = __ballot_sync(0xffffffffu, lo), w1 = __ballot_sync(0xffffffffu, hi);
      return __funnelshift_r(w0, w1, l0);
    };
    uint32_t run = window(blk == b, blk2 == b);
    const uint32_t other = window(blk >= 0 && blk != b, blk2 >= 0 && blk2 != b);
    if (other) run &= (other & (0u - other)) - 1;
    const int span = 32 - __clz(run);
    const int page = b / per, at = b % per;
    uint8_t* codes = a.codes[side] + (((size_t)page * a.KH + h) * a.P + (size_t)at * kKv8Block) * D + lane * N;
    uint8_t* byte_p = a.bytes[side] + ((size_t)page * a.KH + h) * per + at;
    // which of the block's rows are new
    const int s0 = __shfl_sync(0xffffffffu, slot, (l0 + lane) & 31);
    const int s1 = __shfl_sync(0xffffffffu, slot2, (l0 + lane) & 31);
    const int off = (l0 + lane < 32 ? s0 : s1) & (kKv8Block - 1);      // of row t0 + l0 + lane
    const uint32_t fresh = __reduce_or_sync(0xffffffffu, (run >> lane) & 1 ? 1u << off : 0u);
    const int first = __ffs(fresh) - 1;
    // a run without skipped rows of at most 256 bytes a row is read once, all 16 rows in flight
    constexpr bool kHold = VEC && N * sizeof(T) <= 16;
    const bool held = kHold && run == (0xffffffffu >> (32 - span)) && span <= kKv8Block;
    Raw<T, N> raw[kHold ? kKv8Block : 1];
    uint32_t amax = 0;
    if constexpr (kHold) {
      if (held) {
        const T* p = x + (t0 + l0) * a.st[side];
#pragma unroll
        for (int r = 0; r < kKv8Block; ++r)
          if (r < span) raw[r] = ldg_raw<T, N>(p + r * a.st[side]);
#pragma unroll
        for (int r = 0; r < kKv8Block; ++r)
          if (r < span) {
#pragma unroll
            for (int i = 0; i < N; ++i) amax = max(amax, __float_as_uint(to_f32(raw[r].v[i])) & 0x7fffffffu);
          }
      }
    }
#pragma unroll 4
    for (int r = 0; r < (held ? 0 : span); ++r) {
      if (!((run >> r) & 1)) continue;
      float v[N];
      load_vals<T, N, VEC>(x + (t0 + l0 + r) * a.st[side], v);
#pragma unroll
      for (int i = 0; i < N; ++i) amax = max(amax, __float_as_uint(v[i]) & 0x7fffffffu);
    }
    amax = __reduce_max_sync(0xffffffffu, amax);
    int byte = kv8_byte<FP8>(amax);
    if (first > 0) {
      const int old = *byte_p;
      byte = max(byte, old);
      if (byte != old) {
        // the block's scale grew: all its other rows, those after the new ones too, move to the new one, rounded once
        const int d = old - byte;
        const float f = d < -126 ? 0.f : __uint_as_float((uint32_t)(127 + d) << 23);
#pragma unroll 4
        for (int r = 0; r < kKv8Block; ++r) {
          if ((fresh >> r) & 1) continue;
          Codes<N> c;
          __align__(8) uint8_t y[N];
          c = *reinterpret_cast<const Codes<N>*>(codes + (size_t)r * D);
#pragma unroll
          for (int i = 0; i < N; ++i) y[i] = byte == kKv8Nan ? 0 : encode<FP8>(decode<FP8>(c.c[i]) * f);
          store_codes<N>(codes + (size_t)r * D, y);
        }
      }
    }
    const float inv = byte == kKv8Nan ? 0.f : __uint_as_float((uint32_t)(254 - byte) << 23);
    auto put = [&](float* v, int o) {
      __align__(8) uint8_t y[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        v[i] = fminf(fmaxf(v[i], -kv8_top<FP8>), kv8_top<FP8>);
        y[i] = byte == kKv8Nan ? 0 : encode<FP8>(v[i] * inv);
      }
      store_codes<N>(codes + (size_t)o * D, y);
    };
    if constexpr (kHold) {
      if (held) {
#pragma unroll
        for (int r = 0; r < kKv8Block; ++r) {
          const int o = __shfl_sync(0xffffffffu, off, r);
          if (r < span) {
            float v[N];
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = to_f32(raw[r].v[i]);
            put(v, o);
          }
        }
      }
    }
#pragma unroll 4
    for (int r = 0; r < (held ? 0 : span); ++r) {
      if (!((run >> r) & 1)) continue;
      float v[N];
      load_vals<T, N, VEC>(x + (t0 + l0 + r) * a.st[side], v);
      put(v, __shfl_sync(0xffffffffu, off, r));
    }
    __syncwarp();
    if (lane == 0) *byte_p = (uint8_t)byte;
  }
}

// out[i] = the cache's values of slot i: thread per 16 columns, both caches in one launch. 32-bit
// indices (the host splits longer calls): a 64-bit division per thread cost as much as its bytes.
template <bool FP8>
__global__ void __launch_bounds__(256)
    kv8_read_kernel(const uint8_t* __restrict__ kc, const uint8_t* __restrict__ kb, const uint8_t* __restrict__ vc,
                    const uint8_t* __restrict__ vb, const int* __restrict__ slots, uint32_t n, int KH, int D,
                    int pshift, int64_t slots_total, __nv_bfloat16* __restrict__ ko, __nv_bfloat16* __restrict__ vo,
                    int* err) {
  const uint32_t c16 = D / 16, per = KH * c16;
  const uint32_t i = blockIdx.x * 256 + threadIdx.x, row = i / per;
  if (row >= n) return;
  const uint32_t rem = i - row * per, h = rem / c16, c = (rem - h * c16) * 16;
  const int slot = slots[row];
  const bool is_v = blockIdx.y != 0;
  uint4 w[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
  if (slot >= slots_total) kv8_error(err, kErrBadShape);
  if (slot >= 0 && slot < slots_total) {
    const int page = slot >> pshift, at = slot & ((1 << pshift) - 1);
    const size_t head = (size_t)page * KH + h;
    const uint4 q = __ldg(reinterpret_cast<const uint4*>((is_v ? vc : kc) + ((head << pshift) + at) * D + c));
    const float s = kv8_scale((is_v ? vb : kb)[(head << (pshift - 4)) + at / kKv8Block]) / kv8_unit<FP8>;
    const uint32_t in[4] = {q.x, q.y, q.z, q.w};
    __align__(16) __nv_bfloat162 o[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t x = j & 1 ? kv8_hi<FP8>(in[j / 2]) : kv8_lo<FP8>(in[j / 2]);
      const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&x));
      o[j] = __floats2bfloat162_rn(f.x * s, f.y * s);
    }
    w[0] = reinterpret_cast<const uint4*>(o)[0];
    w[1] = reinterpret_cast<const uint4*>(o)[1];
  }
  uint4* dst = reinterpret_cast<uint4*>((is_v ? vo : ko) + ((size_t)row * KH + h) * D + c);
  dst[0] = w[0];
  dst[1] = w[1];
}

namespace {
constexpr int kMaxPools = 8;
struct CopyPool {
  uint8_t* base;
  int64_t page_bytes;      // one page of one layer's K or V
  int64_t outer_stride;    // bytes between two layers' (or K's and V's) pools
  int64_t first_block;     // of the launch's blocks
  int outer;               // layers x 2
  int unit;                // bytes one thread moves at a time: 16, 4 or 1
};
struct CopyArgs {
  CopyPool pool[kMaxPools];
  const int* src;
  const int* dst;
  int pools, moves, pages;
  int* err;
};

template <typename U>
__device__ __forceinline__ void copy_units(const CopyPool& p, const CopyArgs& a, int64_t blk) {
  // 256 threads x 4 units, over (layer, move, unit) flattened
  const int64_t upp = p.page_bytes / (int64_t)sizeof(U);
  const int64_t total = upp * a.moves * p.outer;
  U v[4];
  U* to[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    to[k] = nullptr;
    const int64_t i = (blk * 4 + k) * 256 + threadIdx.x;
    if (i >= total) continue;
    const int64_t pm = i / upp, u = i - pm * upp;
    const int64_t o = pm / a.moves;
    const int m = (int)(pm - o * a.moves);
    const int s = a.src[m], d = a.dst[m];
    if ((unsigned)s >= (unsigned)a.pages || (unsigned)d >= (unsigned)a.pages) {
      kv8_error(a.err, kErrBadShape);
      continue;
    }
    uint8_t* base = p.base + o * p.outer_stride;
    v[k] = reinterpret_cast<const U*>(base + s * p.page_bytes)[u];
    to[k] = reinterpret_cast<U*>(base + d * p.page_bytes) + u;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (to[k] != nullptr) *to[k] = v[k];
}
}  // namespace

__global__ void __launch_bounds__(256) kv_copy_pages_kernel(const __grid_constant__ CopyArgs a) {
  int k = 0;
  while (k + 1 < a.pools && (int64_t)blockIdx.x >= a.pool[k + 1].first_block) ++k;
  const CopyPool& p = a.pool[k];
  const int64_t blk = (int64_t)blockIdx.x - p.first_block;
  if (p.unit == 16)
    copy_units<uint4>(p, a, blk);
  else if (p.unit == 4)
    copy_units<uint32_t>(p, a, blk);
  else
    copy_units<uint8_t>(p, a, blk);
}

// ------------------------------------------------------------------ host side

// codes [pages, KH, P, D] int8 / e4m3 and bytes [pages, KH, P / 16] of one cache
void check_pages8(const torch::Tensor& codes, const torch::Tensor& bytes, const char* what) {
  TORCH_CHECK(codes.dim() == 4 && codes.is_contiguous() &&
                  (codes.scalar_type() == at::kChar || codes.scalar_type() == at::kFloat8_e4m3fn) && codes.is_cuda(),
              what, ": codes [pages, KH, P, D] int8 or e4m3 on the GPU, contiguous");
  const int64_t P = codes.size(2);
  TORCH_CHECK(P >= kKv8Block && (P & (P - 1)) == 0, what, ": page tokens are a power of two, at least 16");
  TORCH_CHECK(bytes.dim() == 3 && bytes.is_contiguous() && bytes.scalar_type() == at::kByte &&
                  bytes.device() == codes.device() && bytes.size(0) == codes.size(0) &&
                  bytes.size(1) == codes.size(1) && bytes.size(2) == P / kKv8Block,
              what, ": exponent bytes [pages, KH, P / 16] uint8 beside the codes");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(codes.data_ptr()) % 16 == 0, what, ": codes are 16-byte aligned");
  TORCH_CHECK(codes.size(0) * P <= INT32_MAX, what, ": slots are 32-bit");
}

template <typename T, int D, bool FP8>
static void launch_write(const WriteArgs& a, bool vec, cudaStream_t st) {
  // One warp a row up to 4096 rows: decode steps, where each row is its own run. Above, 16 rows a
  // warp: a packed chunk has one run in 16 rows, and fifteen of sixteen one-row warps would only exit.
  const int group = a.T <= 4096 ? 1 : 16;
  const int64_t warps = (int64_t)((a.T + group - 1) / group) * a.KH * 2;
  const int grid = (int)((warps + 3) / 4);
#define QB_W(V, G) kv8_write_kernel<T, D, FP8, V, G><<<grid, 128, 0, st>>>(a)
  if (vec)
    group == 1 ? QB_W(true, 1) : QB_W(true, 16);
  else
    group == 1 ? QB_W(false, 1) : QB_W(false, 16);
#undef QB_W
}

template <typename T, bool FP8>
static void launch_write_d(const WriteArgs& a, int D, bool vec, cudaStream_t st) {
  if (D == 64) return launch_write<T, 64, FP8>(a, vec, st);
  if (D == 128) return launch_write<T, 128, FP8>(a, vec, st);
  return launch_write<T, 256, FP8>(a, vec, st);
}

// k, v [T, KH, D] (bf16, fp16 or fp32; any token and head strides) -> the slots' blocks.
// slots int32 [T], -1 to skip; rows of one block are adjacent.
void kv8_write(const torch::Tensor& k, const torch::Tensor& v, const torch::Tensor& slots, torch::Tensor& kc,
               torch::Tensor& kb, torch::Tensor& vc, torch::Tensor& vb) {
  check_pages8(kc, kb, "kv8_write K");
  check_pages8(vc, vb, "kv8_write V");
  TORCH_CHECK(kc.sizes() == vc.sizes() && kc.scalar_type() == vc.scalar_type() && kc.device() == vc.device(),
              "kv8_write: K and V pages alike");
  const int64_t KH = kc.size(1), D = kc.size(3), T = k.size(0);
  TORCH_CHECK(D == 64 || D == 128 || D == 256, "kv8_write: head_dim 64, 128 or 256");
  TORCH_CHECK(k.dim() == 3 && k.size(1) == KH && k.size(2) == D && v.sizes() == k.sizes() &&
                  v.scalar_type() == k.scalar_type(),
              "kv8_write: k and v [T, KH, D] of one type");
  TORCH_CHECK(k.device() == kc.device() && v.device() == kc.device() && slots.device() == kc.device(),
              "kv8_write: one device");
  TORCH_CHECK(k.stride(2) == 1 && v.stride(2) == 1, "kv8_write: a head's columns are contiguous");
  TORCH_CHECK(slots.scalar_type() == at::kInt && slots.is_contiguous() && slots.numel() == T, "kv8_write: slots int32 [T]");
  TORCH_CHECK(T <= INT32_MAX / 2, "kv8_write: T");
  if (T == 0) return;
  const int dev = kc.get_device();
  c10::cuda::CUDAGuard guard(dev);
  cudaStream_t st = at::cuda::getCurrentCUDAStream(dev);
  WriteArgs a;
  const torch::Tensor* xs[2] = {&k, &v};
  const int64_t item = k.element_size();
  const int64_t lane_bytes = std::min<int64_t>(16, D / 32 * item);
  bool vec = true;
  for (int i = 0; i < 2; ++i) {
    a.x[i] = xs[i]->data_ptr();
    a.st[i] = xs[i]->stride(0);
    a.sh[i] = xs[i]->stride(1);
    vec = vec && reinterpret_cast<uintptr_t>(a.x[i]) % lane_bytes == 0 && a.st[i] * item % lane_bytes == 0 &&
          a.sh[i] * item % lane_bytes == 0;
  }
  a.codes[0] = static_cast<uint8_t*>(kc.data_ptr());
  a.codes[1] = static_cast<uint8_t*>(vc.data_ptr());
  a.bytes[0] = kb.data_ptr<uint8_t>();
  a.bytes[1] = vb.data_ptr<uint8_t>();
  a.slots = slots.data_ptr<int>();
  a.T = (int)T;
  a.KH = (int)KH;
  a.P = (int)kc.size(2);
  a.slots_total = kc.size(0) * kc.size(2);
  a.err = device_error_word(dev);
  const bool fp8 = kc.scalar_type() == at::kFloat8_e4m3fn;
  if (k.scalar_type() == at::kBFloat16)
    fp8 ? launch_write_d<__nv_bfloat16, true>(a, D, vec, st) : launch_write_d<__nv_bfloat16, false>(a, D, vec, st);
  else if (k.scalar_type() == at::kHalf)
    fp8 ? launch_write_d<__half, true>(a, D, vec, st) : launch_write_d<__half, false>(a, D, vec, st);
  else if (k.scalar_type() == at::kFloat)
    fp8 ? launch_write_d<float, true>(a, D, vec, st) : launch_write_d<float, false>(a, D, vec, st);
  else
    TORCH_CHECK(false, "kv8_write: k and v are bf16, fp16 or fp32");
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

void kv8_read(const torch::Tensor& kc, const torch::Tensor& kb, const torch::Tensor& vc, const torch::Tensor& vb,
              const torch::Tensor& slots, torch::Tensor& ko, torch::Tensor& vo) {
  check_pages8(kc, kb, "kv8_read K");
  check_pages8(vc, vb, "kv8_read V");
  TORCH_CHECK(kc.sizes() == vc.sizes() && kc.scalar_type() == vc.scalar_type() && kc.device() == vc.device(),
              "kv8_read: K and V pages alike");
  const int64_t n = slots.numel(), KH = kc.size(1), D = kc.size(3), P = kc.size(2);
  TORCH_CHECK(D % 16 == 0, "kv8_read: head_dim");
  TORCH_CHECK(slots.scalar_type() == at::kInt && slots.is_contiguous() && slots.device() == kc.device(),
              "kv8_read: slots int32");
  for (const torch::Tensor* o : {&ko, &vo})
    TORCH_CHECK(o->scalar_type() == at::kBFloat16 && o->is_contiguous() && o->device() == kc.device() &&
                    o->numel() == n * KH * D && reinterpret_cast<uintptr_t>(o->data_ptr()) % 16 == 0,
                "kv8_read: out [n, KH, D] bf16, 16-byte aligned");
  if (n == 0) return;
  const int dev = kc.get_device();
  c10::cuda::CUDAGuard guard(dev);
  cudaStream_t st = at::cuda::getCurrentCUDAStream(dev);
  auto p8 = [](const torch::Tensor& t) { return static_cast<const uint8_t*>(t.data_ptr()); };
  auto bf = [](torch::Tensor& t) { return reinterpret_cast<__nv_bfloat16*>(t.data_ptr()); };
  int* err = device_error_word(dev);
  const int pshift = __builtin_ctzll((unsigned long long)P);
  const int64_t per = KH * (D / 16), most = std::max<int64_t>(1, ((int64_t)1 << 31) / per);   // rows of a launch
  for (int64_t r0 = 0; r0 < n; r0 += most) {
    const int64_t rows = std::min(most, n - r0);
    const dim3 grid((unsigned)((rows * per + 255) / 256), 2);
    const int* sl = slots.data_ptr<int>() + r0;
    __nv_bfloat16 *ro = bf(ko) + r0 * KH * D, *so = bf(vo) + r0 * KH * D;
    if (kc.scalar_type() == at::kFloat8_e4m3fn)
      kv8_read_kernel<true><<<grid, 256, 0, st>>>(p8(kc), p8(kb), p8(vc), p8(vb), sl, (uint32_t)rows, KH, D, pshift,
                                                  kc.size(0) * P, ro, so, err);
    else
      kv8_read_kernel<false><<<grid, 256, 0, st>>>(p8(kc), p8(kb), p8(vc), p8(vb), sl, (uint32_t)rows, KH, D, pshift,
                                                   kc.size(0) * P, ro, so, err);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  }
}

// pools: tensors [layers, 2, pages, ...] (one arena's; all with the same number of pages);
// in each, page dst[i] of every layer's K and V becomes a copy of page src[i]. No page is in
// both lists, and none twice in dst.
void kv_copy_pages(std::vector<torch::Tensor> pools, const torch::Tensor& src, const torch::Tensor& dst) {
  TORCH_CHECK(!pools.empty() && (int)pools.size() <= kMaxPools, "kv_copy_pages: 1 to 8 pools");
  TORCH_CHECK(src.scalar_type() == at::kInt && dst.scalar_type() == at::kInt && src.is_contiguous() &&
                  dst.is_contiguous() && src.numel() == dst.numel() && src.device() == pools[0].device() &&
                  dst.device() == pools[0].device(),
              "kv_copy_pages: src and dst int32, of one length, beside the pools");
  CopyArgs a;
  a.moves = (int)src.numel();
  a.pages = (int)pools[0].size(2);
  int64_t blocks = 0;
  int n = 0;
  for (const torch::Tensor& t : pools) {
    TORCH_CHECK(t.is_cuda() && t.dim() >= 3 && t.is_contiguous() && t.device() == pools[0].device() &&
                    t.size(2) == pools[0].size(2),
                "kv_copy_pages: pools [layers, 2, pages, ...], contiguous, of one number of pages");
    const int64_t outer = t.size(0) * t.size(1);
    if (t.numel() == 0) continue;
    CopyPool& p = a.pool[n++];
    p.base = static_cast<uint8_t*>(t.data_ptr());
    p.page_bytes = t.stride(2) * t.element_size();
    p.outer = (int)outer;
    p.outer_stride = t.stride(1) * t.element_size();
    const int64_t al = (int64_t)(reinterpret_cast<uintptr_t>(p.base) | (uintptr_t)p.page_bytes);
    p.unit = al % 16 == 0 ? 16 : al % 4 == 0 ? 4 : 1;
    p.first_block = blocks;
    blocks += (p.page_bytes / p.unit * a.moves * outer + 1023) / 1024;
  }
  a.pools = n;
  if (a.moves == 0 || n == 0) return;
  TORCH_CHECK(blocks <= INT32_MAX, "kv_copy_pages: too many pages in one call");
  const int dev = pools[0].get_device();
  c10::cuda::CUDAGuard guard(dev);
  cudaStream_t st = at::cuda::getCurrentCUDAStream(dev);
  a.src = src.data_ptr<int>();
  a.dst = dst.data_ptr<int>();
  a.err = device_error_word(dev);
  kv_copy_pages_kernel<<<(unsigned)blocks, 256, 0, st>>>(a);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

}  // namespace qb
