// The 8-bit KV cache: layout, code conversion and the segment walk its
// kernels share.
//
// One layer's K (or V) is codes [pages, KH, P, D] (int8 or e4m3) and exponent
// bytes [pages, KH, P / 16]: a value is code * 2^(byte - 127), with one byte
// for 16 consecutive tokens of one head. Byte 255 marks a block that was given
// a value that is not finite; its values read as NaN. Pages are head-major, so
// a head's tokens of a page are one contiguous run (the unit a bulk copy
// moves), and a 64-token tile's four bytes are one aligned word.
//
// The scale is a power of two so that every step but the final rounding is
// exact: a write has one right answer bit for bit, a block's scale can grow
// when a later token needs it with an exact rescale of the old codes (one
// rounding), and in attention it is an exponent added where an exponent is
// computed anyway. It costs int8 up to one bit of the 7 against amax / 127
// (a block's largest code is 64..127). The smallest byte written is 67
// (2^-60): below it, attention's p * 2^(byte - 127) would underflow and lose
// that block's share of the softmax sum.
#pragma once

#include "common.cuh"

namespace qb {

constexpr int kKv8Block = 16;        // tokens per exponent byte
constexpr int kKv8MinByte = 67;
constexpr int kKv8TopByte = 248;       // of int8; e4m3 needs no more than 247
constexpr int kKv8Nan = 255;
constexpr int kKv8SeqInts = 12;
constexpr int kKv8MaxSeg = 4;

// Exponent byte for a block whose largest magnitude has these fp32 bits: the
// smallest power of two with 127 * 2^e (int8) or 448 * 2^e (e4m3) >= amax.
// 127 = 1.984375 * 2^6 and 448 = 1.75 * 2^8, so a compare of the mantissa decides.
// int8's 249 is not used: its codes from 64 on would stand for 2^128 and more, past fp32 and bf16 (kv8_top).
template <bool FP8>
__device__ __forceinline__ int kv8_byte(uint32_t amax_bits) {
  if (amax_bits >= 0x7f800000u) return kKv8Nan;
  const int x = (int)(amax_bits >> 23);
  const uint32_t frac = amax_bits & 0x7fffffu;
  const int b = FP8 ? x - 8 + (frac > 0x600000u) : min(x - 6 + (frac > 0x7e0000u), kKv8TopByte);
  return max(b, kKv8MinByte);
}

// The largest magnitude that is stored; finite values above it become it. int8: 127 * 2^(248 - 127), within half a
// step of bf16's largest number. e4m3's 4 bits would round a magnitude from 1.9375 * 2^127 up to 2^128, which no
// reader's bf16 holds: 1.875 * 2^127 is the largest code below it.
template <bool FP8>
constexpr float kv8_top = FP8 ? 3.1901471898837980e38f : 3.3762391092936860e38f;

// 2^(byte - 127) as fp32; NaN for 255
__device__ __forceinline__ float kv8_scale(int byte) {
  return byte == kKv8Nan ? __int_as_float(0x7fc00000) : __uint_as_float((uint32_t)byte << 23);
}

// Two codes, each doubled into both bytes of a half word ([c0, c0, c1, c1]), to two bf16 values,
// exactly, times kv8_unit.
//   int8: the 16-bit pattern of a whole number u < 256 is the bf16 number u * 2^-133 (the subnormals and
//         the first binade have one spacing), so with u = c + 128 one fused multiply-add, u * 2^-133 *
//         2^127 - 2, leaves c * 2^-6.
//   e4m3: sign, exponent and mantissa moved into place read as value * 2^-120
//         (the biases differ by 120; e4m3 subnormals become bf16 subnormals,
//         which bf16x2 arithmetic keeps), then times 2^120.
template <bool FP8>
constexpr float kv8_unit = FP8 ? 1.f : 0.015625f;
template <bool FP8>
__device__ __forceinline__ uint32_t kv8_pair(uint32_t x) {
  uint32_t r;
  if constexpr (FP8) {
    const uint32_t bits = ((x >> 4) & 0x07f007f0u) | (x & 0x80008000u);
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(bits), "r"(0x7b807b80u));
  } else {
    const uint32_t u = (x & 0x00ff00ffu) ^ 0x00800080u;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(u), "r"(0x7f007f00u), "r"(0xc000c000u));
  }
  return r;
}

// codes i and i + 1 of a word (i = 0 or 2) as bf16x2
template <bool FP8>
__device__ __forceinline__ uint32_t kv8_lo(uint32_t w) {
  return kv8_pair<FP8>(__byte_perm(w, 0, 0x1100));
}
template <bool FP8>
__device__ __forceinline__ uint32_t kv8_hi(uint32_t w) {
  return kv8_pair<FP8>(__byte_perm(w, 0, 0x3322));
}

// The same to two f16 values, exactly (half the ALU work of bf16, whose 7 explicit bits do not hold
// 1024 + a byte). `x` has the codes in bytes 0 and 2 for int8, in bytes 0 and 1 for e4m3.
//   int8: 0x6400 | (c ^ 128) is 1024 + 128 + c in f16
//   e4m3: the hardware's conversion
template <bool FP8>
__device__ __forceinline__ uint32_t kv8_half2(uint32_t x) {
  uint32_t r;
  if constexpr (FP8) {
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(x));
  } else {
    const uint32_t u = (x & 0x00ff00ffu) ^ 0x64806480u;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(u), "r"(0x64806480u));
  }
  return r;
}

// A mean of values near fp32's largest is finite, their sum is not: the mma.sync kernels take V's scales times 2^-24
// and their results times 2^24, which is room for 2^24 keys. (The tcgen05 kernel raises its running maximum instead.)
constexpr float kKv8Down = 5.9604644775390625e-8f, kKv8Up = 16777216.f;

__device__ __forceinline__ float kv8_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void kv8_error(int* err, int code) {
  if (err != nullptr) atomicCAS(err, 0, code);
}

// What every attention over the cache gets.
struct Kv8Attn {
  const __nv_bfloat16* q;
  const uint8_t *kc, *kb, *vc, *vb;
  const int *seqs, *blocks, *page_list;   // blocks: the prefill's blocks, or the decode's sequences
  int T, n_seqs, n_list, pages, P, QH, KH;
  float sl2;
  __nv_bfloat16* o;
  uint8_t *o8, *osf;
  float* lse;
  int* err;
};


// One sequence's segments and what its queries see. Flags: bit 0, the own
// segment is read both ways; bits 8..23, a sliding window over the own segment
// (0: none); bit 24, the window spans the earlier segments too (with bit 0 only
// those). Keys of earlier segments are read whole unless bit 24 is set.
struct Kv8Seq {
  int q_start, q_len, nseg, own_len, before, win;
  bool bidir, win_all;
  int len[kKv8MaxSeg], off[kKv8MaxSeg];
};

// Segments that reach past the page list are reported and count as empty, so that every key's place in the list is
// inside it, and the sums of a table's lengths (which the host bounds by the list's) stay in 32 bits.
__device__ __forceinline__ void kv8_load_seq(Kv8Seq& s, const Kv8Attn& a, int seq) {
  const int* sd = a.seqs + (size_t)seq * kKv8SeqInts;    // a view of a packed buffer: 4-byte aligned
  int v[kKv8SeqInts];
#pragma unroll
  for (int i = 0; i < kKv8SeqInts; ++i) v[i] = __ldg(sd + i);
  s.q_start = v[0];
  s.q_len = v[1];
  s.nseg = min(max(v[2], 0), kKv8MaxSeg);
  s.bidir = (v[3] & 1) != 0;
  s.win = (v[3] >> 8) & 0xffff;
  s.win_all = (v[3] >> 24) & 1;
  const int pshift = __ffs(a.P) - 1;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < kKv8MaxSeg; ++i) {
    s.len[i] = i < s.nseg ? max(v[4 + i], 0) : 0;
    s.off[i] = v[4 + kKv8MaxSeg + i];
    const bool past = s.len[i] > 0 && (s.off[i] < 0 || (s.len[i] - 1) >> pshift >= a.n_list - s.off[i]);
    if (past) s.len[i] = 0;
    bad |= past;
  }
  if (bad) kv8_error(a.err, kErrBadShape);
  s.own_len = 0;
  s.before = 0;
#pragma unroll
  for (int i = 0; i < kKv8MaxSeg; ++i) {
    if (i == s.nseg - 1) s.own_len = s.len[i];
    if (i < s.nseg - 1) s.before += s.len[i];
  }
}

// Whether a sequence's query rows are among the T there are (their sum may pass 32 bits).
__device__ __forceinline__ bool kv8_rows_ok(const Kv8Seq& s, int T) {
  return s.q_start >= 0 && s.q_len >= 0 && s.q_len <= T - s.q_start;
}

// Keys [lo, hi) of segment `seg` (with `base` keys before it) that a query at
// own-segment position `pos` sees.
__device__ __forceinline__ void kv8_span(const Kv8Seq& s, int seg, int seg_len, int base, int pos, int& lo, int& hi) {
  const bool own = seg == s.nseg - 1;
  hi = own && !s.bidir ? min(seg_len, pos + 1) : seg_len;
  lo = 0;
  if (s.win > 0 && (own ? !s.bidir : s.win_all)) lo = max(0, s.before + pos - s.win + 1 - base);
}

}  // namespace qb
