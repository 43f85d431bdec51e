// Device code shared by the e4m3 products (fp8.hip, fp8_gemm.hip).
#pragma once

#include "fp8.hpp"
#include "mfma.hpp"
#include "scores.hpp"

namespace uocr {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// A raw buffer resource for loads: those at or past `bytes` give zeros.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t read_rsrc(const void* base, uint32_t bytes) {
  return store_rsrc(const_cast<void*>(base), bytes);
}

constexpr int kCus = 256, kMostLds = 160 << 10;

// What a product leaves: its values in f32 or bf16, or its rows' statistics.
enum { kOutF32, kOutBf16, kOutScores };

struct ProductOut {
  void* y;              // [m, n]
  ScorePart* parts;     // [column tiles][m]
  const int32_t* tokens;
  float* given;         // [m] logits of the given tokens
};

// Eight e4m3 values (two words) as bf16, which holds them exactly.
__device__ __forceinline__ bf16x8 widen_fp8x8(uint32_t lo, uint32_t hi) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
  return (bf16x8){a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Four adjacent columns of row `row`, from column col on.
template <int OUT>
__device__ __forceinline__ void store_columns(const Fp8Product& p, void* y, int row, int col, f32x4 v) {
  if (row >= p.m || col >= p.n) return;
  const size_t at = (size_t)row * p.n + col;
  if (p.n % 4 == 0) {  // four whole columns; y is aligned to its element, so is any of its rows to four
    if (OUT == kOutF32) {
      __builtin_memcpy(static_cast<float*>(y) + at, &v, 16);
    } else {
      const uint2 b = make_uint2(bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3]));
      __builtin_memcpy(static_cast<uint16_t*>(y) + at, &b, 8);
    }
    return;
  }
#pragma unroll
  for (int r = 0; r < 4; r++) {
    if (col + r >= p.n) return;
    if (OUT == kOutF32)
      static_cast<float*>(y)[at + r] = v[r];
    else
      static_cast<uint16_t*>(y)[at + r] = bf16_bits(v[r]);
  }
}

// The statistics of one row's logits in a wave: lane l holds columns col + STRIDE i +
// r of row l % 16 (v[i][r]; col differs by 4 between the four lanes of a row) or, with a
// STRIDE of 8, of row l % 32 (two lanes). Every lane of the row gets them. The lane with
// the given token's column keeps its logit. FULL: all of the columns are below n.
template <int COUNT, bool FULL, int STRIDE>
__device__ __forceinline__ ScorePart row_statistics(const f32x4 (&v)[COUNT], int col, int n, int token,
                                                    float* given) {
  ScorePart q = empty_part();
  float most = -INFINITY;
#pragma unroll
  for (int i = 0; i < COUNT; i++)
#pragma unroll
    for (int r = 0; r < 4; r++) most = FULL || col + STRIDE * i + r < n ? fmaxf(most, v[i][r]) : most;
  if (STRIDE == 16) most = fmaxf(most, __shfl_xor(most, 16));
  most = fmaxf(most, __shfl_xor(most, 32));
  // d = log2(e) x - r2 in one instruction; r2's rounding c, the same for all of the
  // row's logits here, is put right at the end: the terms are 2^(d + c). Beyond 1e9 c is
  // large enough for 2^c to overflow or vanish, which ends as a row without distribution.
  q.r = fminf(fmaxf(most, -1e38f), 1e38f);
  const float r2 = q.r * kLog2e;
#pragma unroll
  for (int i = 0; i < COUNT; i++)
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const float d = FULL || col + STRIDE * i + r < n ? fmaf(v[i][r], kLog2e, -r2) : -1000.0f;
      const float e = __builtin_amdgcn_exp2f(d);
      q.s += e;
      q.t = fmaf(e, d, q.t);
    }
  const uint32_t off = (uint32_t)(token - col);
  if (off < (uint32_t)STRIDE * COUNT && (off & (STRIDE - 4u)) == 0 && token < n) {
    float g = 0.0f;
#pragma unroll
    for (int i = 0; i < COUNT; i++)
#pragma unroll
      for (int r = 0; r < 4; r++) g = off == (uint32_t)STRIDE * i + r ? v[i][r] : g;
    *given = g;
  }
#pragma unroll
  for (int o = STRIDE == 16 ? 16 : 32; o <= 32; o <<= 1) {
    q.s += __shfl_xor(q.s, o);
    q.t += __shfl_xor(q.t, o);
  }
  const float c = fmaf(-q.r, kLog2e, r2);
  const float e = __builtin_amdgcn_exp2f(c);
  q.t = fmaf(q.s, c, q.t) * e;
  q.s *= e;
  return q;
}
// The same, whether or not the wave's columns (from n0 on) end below n.
template <int COUNT, int STRIDE = 16>
__device__ __forceinline__ ScorePart row_statistics(const f32x4 (&v)[COUNT], int n0, int fg, int n, int token,
                                                    float* given) {
  return n0 + STRIDE * COUNT <= n ? row_statistics<COUNT, true, STRIDE>(v, n0 + 4 * fg, n, token, given)
                                  : row_statistics<COUNT, false, STRIDE>(v, n0 + 4 * fg, n, token, given);
}

// fp8_gemm.hip: the product of many rows.
// Parts per row that scores leave (ProductOut::parts), and the launch.
int fp8_gemm_parts(const Fp8Product& p);
// `work` may be any size: without room for partial sums the depth is not split.
void launch_fp8_gemm(const Fp8Product& p, const ProductOut& out, int kind, void* work, size_t work_bytes,
                     hipStream_t s);
void fp8_gemm_init_attributes();
// The launch's modelled time in units of 0.1 us (whole_chunks only).
double fp8_gemm_time(const Fp8Product& p, bool widen, size_t work_bytes);

// Rows at any address are read by aligned words, one more than the bytes wanted, and moved
// to their places (loads at addresses that are no multiple of 4 take some three times as
// long). A resource of `bytes` bytes from p on then starts at p's word and ends with the
// last byte's; each word of a 16-byte load is checked for itself.
__device__ __forceinline__ uint32_t misaligned(const void* p) { return (uint32_t)reinterpret_cast<uintptr_t>(p) & 3; }
template <bool WHOLE>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t word_rsrc(const uint8_t* p, uint32_t bytes) {
  if (WHOLE) return read_rsrc(p, bytes);
  const uint32_t by = misaligned(p);
  return read_rsrc(p - by, bytes ? (bytes + by + 3) & ~3u : 0);  // no byte, no word
}
__device__ __forceinline__ u32x4 shift_bytes(u32x4 v, uint32_t next, uint32_t by) {
  by &= 3;
  return (u32x4){__builtin_amdgcn_alignbyte(v.y, v.x, by), __builtin_amdgcn_alignbyte(v.z, v.y, by),
                 __builtin_amdgcn_alignbyte(v.w, v.z, by), __builtin_amdgcn_alignbyte(next, v.w, by)};
}
// The first `left` bytes, zeros behind them.
__device__ __forceinline__ u32x4 first_bytes(u32x4 v, int left) {
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int bits = min(max(left - 4 * i, 0), 4) * 8;
    v[i] = bits == 32 ? v[i] : v[i] & ((1u << bits) - 1);
  }
  return v;
}

// Bytes of fp8_pack_bytes' copy.
size_t fp8_packed_size(const Fp8Product& p);

// Whole 16-byte chunks of rows at aligned addresses.
inline bool whole_chunks(const Fp8Product& p) {
  return p.k % 16 == 0 && reinterpret_cast<uintptr_t>(p.x) % 16 == 0 && reinterpret_cast<uintptr_t>(p.w) % 16 == 0;
}

}  // namespace uocr
