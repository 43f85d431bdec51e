// 8-bit floating point (e4m3) with a scale per block of 128: rows quantised,
// and the product of such rows with a matrix of 128 x 128 tiles.
//
//   y[i][j] = sum_b xs[i][b] ws[j / 128][b] sum_{k in block b} x[i][k] w[j][k]
//
// No counterpart in the reference, whose overlay is int8 with blocks of 32
// (src/cpu/quantized.rs:9-237); these stand beside its operators.
#include <algorithm>

#include "fp8_device.hpp"

namespace uocr {

// ------------------------------------------------------------- quantisation

// The scale of a block whose largest magnitude has the bits `most`: the least
// power of two s with most / s <= 448 = 1.75 * 2^8, at least 2^-126; 1 for a
// block of zeros. As biased exponents; a power of two makes x / s exact, so the
// only rounding is the one to e4m3, and costs nothing against most / 448: the
// relative step of a floating format does not depend on the scale.
__device__ __forceinline__ uint32_t scale_exponent(uint32_t most) {
  if (most == 0) return 127;
  const int e = (int)(most >> 23) - 8 + ((most & 0x7fffffu) > 0x600000u);
  return (uint32_t)max(e, 1);
}

template <typename T>
__device__ __forceinline__ float widen(T v);
template <>
__device__ __forceinline__ float widen<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ float widen<uint16_t>(uint16_t v) {
  return __uint_as_float((uint32_t)v << 16);
}

__device__ __forceinline__ uint32_t max_u32(uint32_t a, uint32_t b) { return a > b ? a : b; }

// Eight values of one lane as e4m3 (round to nearest even), two words.
__device__ __forceinline__ uint2 to_fp8x8(const float (&v)[8], float inverse) {
  int lo = 0, hi = 0;
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inverse, v[1] * inverse, lo, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * inverse, v[3] * inverse, lo, true);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[4] * inverse, v[5] * inverse, hi, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[6] * inverse, v[7] * inverse, hi, true);
  return make_uint2((uint32_t)lo, (uint32_t)hi);
}

// Eight consecutive elements at p, of which `have` exist (zeros behind them).
template <typename T, bool WIDE>
__device__ __forceinline__ void load8(const T* p, int have, float (&v)[8]) {
  if (WIDE) {
    if (have > 0) {
      if constexpr (sizeof(T) == 4) {
        const float4 a = reinterpret_cast<const float4*>(p)[0];
        const float4 b = reinterpret_cast<const float4*>(p)[1];
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
        v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
      } else {
        const uint4 a = *reinterpret_cast<const uint4*>(p);
        v[0] = bf16_lo(a.x), v[1] = bf16_hi(a.x), v[2] = bf16_lo(a.y), v[3] = bf16_hi(a.y);
        v[4] = bf16_lo(a.z), v[5] = bf16_hi(a.z), v[6] = bf16_lo(a.w), v[7] = bf16_hi(a.w);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] = 0.0f;
    }
  } else if (have >= 8) {
    if constexpr (sizeof(T) == 4) {
      __builtin_memcpy(v, p, 32);
    } else {  // aligned words, five where the first element is the second of its word
      const uint32_t by = misaligned(p);
      const auto* at = reinterpret_cast<const uint32_t*>(reinterpret_cast<const uint8_t*>(p) - by);
      u32x4 a;
      __builtin_memcpy(&a, __builtin_assume_aligned(at, 4), 16);
      a = shift_bytes(a, by ? at[4] : 0, by);
#pragma unroll
      for (int j = 0; j < 4; j++) v[2 * j] = bf16_lo(a[j]), v[2 * j + 1] = bf16_hi(a[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = j < have ? widen<T>(p[j]) : 0.0f;
  }
}

template <bool WIDE>
__device__ __forceinline__ void store8(uint8_t* q, int have, uint2 b) {
  if (WIDE) {
    if (have > 0) *reinterpret_cast<uint2*>(q) = b;
  } else if (have >= 8) {
    __builtin_memcpy(q, &b, 8);
  } else {
#pragma unroll
    for (int j = 0; j < 8; j++)
      if (j < have) q[j] = (uint8_t)((j < 4 ? b.x : b.y) >> (8 * (j & 3)));
  }
}

__device__ __forceinline__ uint32_t largest_bits(const float (&v)[8]) {
  uint32_t most = 0;
#pragma unroll
  for (int j = 0; j < 8; j++) most = max_u32(most, __float_as_uint(v[j]) & 0x7fffffffu);
  return most;
}

// Sixteen lanes hold one block, eight columns each. The block's largest
// magnitude is compared as bits: a NaN is above infinity is above all numbers.
// WIDE: rows and columns allow 16-byte loads and 8-byte stores (cols a multiple
// of 8, so a lane's columns exist all or not at all); otherwise elements move one by
// one at a row's end and eight at a time before it. 4096 x 6848 bf16 15.4 us, 6847
// columns 17.7 (42 one by one); f32 23.4 and 23.5.
template <typename T, bool WIDE>
__global__ __launch_bounds__(256) void fp8_quantize_kernel(const T* __restrict__ x, size_t items,
                                                           int cols, size_t ld,
                                                           uint8_t* __restrict__ q,
                                                           float* __restrict__ scales, int* err) {
  const int nb = (cols + kFp8Block - 1) / kFp8Block;
  const size_t item = ((size_t)blockIdx.x * 256 + threadIdx.x) / 16;
  if (item >= items) return;
  const size_t row = item / nb;
  const int b = (int)(item % nb);
  const int c = b * kFp8Block + (threadIdx.x & 15) * 8;
  float v[8];
  load8<T, WIDE>(x + row * ld + c, cols - c, v);
  uint32_t most = largest_bits(v);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) most = max_u32(most, (uint32_t)__shfl_xor((int)most, o));
  const uint32_t e = scale_exponent(most);
  store8<WIDE>(q + row * cols + c, cols - c, to_fp8x8(v, __uint_as_float((254u - e) << 23)));
  if ((threadIdx.x & 15) == 0) {
    scales[item] = __uint_as_float(e << 23);
    if (most >= 0x7f800000u) raise_error(err, kErrNumerical);
  }
}

void launch_fp8_quantize(const void* x, int type, size_t rows, int cols, size_t ld, uint8_t* q,
                         float* scales, int* err, hipStream_t s) {
  const size_t nb = ((size_t)cols + kFp8Block - 1) / kFp8Block;
  const size_t items = rows * nb;
  const size_t size = type == kTypeF32 ? 4 : 2;
  const bool wide = cols % 8 == 0 && (rows == 1 || ld * size % 16 == 0) &&
                    reinterpret_cast<uintptr_t>(x) % 16 == 0 &&
                    reinterpret_cast<uintptr_t>(q) % 8 == 0;
  const dim3 grid((unsigned)((items + 15) / 16)), block(256);
  if (type == kTypeF32) {
    if (wide)
      fp8_quantize_kernel<float, true><<<grid, block, 0, s>>>((const float*)x, items, cols, ld, q, scales, err);
    else
      fp8_quantize_kernel<float, false><<<grid, block, 0, s>>>((const float*)x, items, cols, ld, q, scales, err);
  } else {
    if (wide)
      fp8_quantize_kernel<uint16_t, true><<<grid, block, 0, s>>>((const uint16_t*)x, items, cols, ld, q, scales, err);
    else
      fp8_quantize_kernel<uint16_t, false><<<grid, block, 0, s>>>((const uint16_t*)x, items, cols, ld, q, scales, err);
  }
}

// One workgroup per 128 x 128 tile of a matrix (laid out once, not in a
// serving path): sixteen lanes per row of the tile, sixteen rows per pass.
template <typename T>
__global__ __launch_bounds__(256) void fp8_quantize_tiles_kernel(const T* __restrict__ x, int rows,
                                                                 int cols, size_t ld,
                                                                 uint8_t* __restrict__ q,
                                                                 float* __restrict__ scales,
                                                                 int* err) {
  __shared__ uint32_t wave_most[4];
  const int c = (int)blockIdx.x * kFp8Block + (threadIdx.x & 15) * 8;
  const int r0 = (int)blockIdx.y * kFp8Block + (threadIdx.x >> 4);
  float v[8][8];
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const int r = r0 + 16 * i;
    load8<T, false>(x + (size_t)r * ld + c, r < rows ? cols - c : 0, v[i]);
    most = max_u32(most, largest_bits(v[i]));
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) most = max_u32(most, (uint32_t)__shfl_xor((int)most, o));
  if ((threadIdx.x & 63) == 0) wave_most[threadIdx.x >> 6] = most;
  __syncthreads();
  most = max_u32(max_u32(wave_most[0], wave_most[1]), max_u32(wave_most[2], wave_most[3]));
  const uint32_t e = scale_exponent(most);
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const int r = r0 + 16 * i;
    store8<false>(q + (size_t)r * cols + c, r < rows ? cols - c : 0,
                  to_fp8x8(v[i], __uint_as_float((254u - e) << 23)));
  }
  if (threadIdx.x == 0) {
    scales[(size_t)blockIdx.y * gridDim.x + blockIdx.x] = __uint_as_float(e << 23);
    if (most >= 0x7f800000u) raise_error(err, kErrNumerical);
  }
}

void launch_fp8_quantize_tiles(const void* x, int type, int rows, int cols, size_t ld, uint8_t* q,
                               float* scales, int* err, hipStream_t s) {
  const dim3 grid((unsigned)((cols + kFp8Block - 1) / kFp8Block),
                  (unsigned)((rows + kFp8Block - 1) / kFp8Block));
  if (type == kTypeF32)
    fp8_quantize_tiles_kernel<float><<<grid, 256, 0, s>>>((const float*)x, rows, cols, ld, q, scales, err);
  else
    fp8_quantize_tiles_kernel<uint16_t><<<grid, 256, 0, s>>>((const uint16_t*)x, rows, cols, ld, q, scales, err);
}

// ------------------------------------------------------------------ product

// ---- few rows: the matrix is streamed from memory straight to the registers of the
// wave that multiplies it, two scale blocks in flight; x comes from the caches. A wave
// takes 16 RG columns of y (rows of the matrix) and up to 64 of x's rows, as MB blocks of
// 16 (more rows: more workgroups, in the grid's second dimension); KS waves of a
// workgroup share a group's depth and add up in LDS, in order. Lane l reads the bytes
// [16 (l / 16), +16) and 64 bytes on of row l % 16 in each block: a load instruction
// covers 64-byte runs. Rows that are not whole chunks (WHOLE false; the same in the kernel
// below) are read where they are, by aligned words: 1 x 1280 x 6847 11.0 us against 7.2 at
// 6848, 16 x 6848 x 1279 7.6 against 5.8.
constexpr int kStreamRows = 64;
// More than 64 rows come here only up to this many rows (whole 64) x columns x blocks.
constexpr size_t kStreamMost = (size_t)4 << 20;

struct StreamShape {
  int ks, waves;  // waves that share a group's depth, waves per workgroup
};

// Blocks in flight.
constexpr int kStreamDepth = 2;
// Most waves of a workgroup, by the registers that a wave then may have: 128 where
// x has one or two blocks of rows, 256 otherwise.
constexpr int stream_waves(int mb) { return mb <= 2 ? 16 : 8; }

template <int MB, int RG, int OUT, bool WHOLE>
__global__ __launch_bounds__(64 * stream_waves(MB), 2) void fp8_stream_kernel(Fp8Product p, ProductOut out,
                                                                                  StreamShape shape) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int fr = lane & 15, fg = lane >> 4;
  // This workgroup's rows become the product's.
  const int m0 = (int)blockIdx.y * kStreamRows, rows = p.m;
  p.x += (size_t)m0 * p.k;
  p.xs += (size_t)m0 * p.kblocks();
  p.m = min(kStreamRows, rows - m0);
  const int groups = shape.waves / shape.ks;  // of this workgroup
  const int slot = wave / shape.ks, k0 = wave % shape.ks;
  const int n0 = ((int)blockIdx.x * groups + slot) * 16 * RG;
  const int K = p.k, nkb = p.kblocks();

  struct Stage {
    u32x4 w[RG][2], x[MB][2];
    uint32_t w_next[WHOLE ? 1 : RG][2], x_next[WHOLE ? 1 : MB][2];
    float xs[MB], ws;
  };
  f32x4 acc[RG][MB];
#pragma unroll
  for (int i = 0; i < RG; i++)
#pragma unroll
    for (int j = 0; j < MB; j++) acc[i][j] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};

  if (n0 < p.n) {
    // Rows past the last one and chunks past a row's end are out of the resources'
    // ranges: zeros, without a branch around the loads (as in the kernel below).
    const uint8_t* w0 = p.w + (size_t)n0 * K;
    const __amdgpu_buffer_rsrc_t rw = word_rsrc<WHOLE>(w0, (uint32_t)min(16 * RG, p.n - n0) * K);
    const __amdgpu_buffer_rsrc_t rx = word_rsrc<WHOLE>(p.x, (uint32_t)p.m * K);
    // Where rows start, in bytes from the resources' first words.
    const uint32_t at_w = (WHOLE ? 0 : misaligned(w0)) + (uint32_t)fr * K;
    const uint32_t at_x = (WHOLE ? 0 : misaligned(p.x)) + (uint32_t)fr * K;
    const __amdgpu_buffer_rsrc_t rs = read_rsrc(p.xs, (uint32_t)(p.m * nkb) * 4u);
    const __amdgpu_buffer_rsrc_t rt = read_rsrc(p.ws + (size_t)(n0 / kFp8Block) * nkb, (uint32_t)nkb * 4u);
    auto load = [&](Stage& s, int kb) {
      const int k = kb * kFp8Block + 16 * fg;
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const uint32_t out_of = k + 64 * h < K ? 0 : kDmaOut;
#pragma unroll
        for (int i = 0; i < RG; i++) {
          const uint32_t at = at_w + (uint32_t)(16 * i) * K + k + 64 * h;
          s.w[i][h] = __builtin_amdgcn_raw_buffer_load_b128(rw, (WHOLE ? at : at & ~3u) | out_of, 0, 0);
          if (!WHOLE) s.w_next[i][h] = __builtin_amdgcn_raw_buffer_load_b32(rw, ((at & ~3u) + 16) | out_of, 0, 0);
        }
#pragma unroll
        for (int j = 0; j < MB; j++) {
          const uint32_t at = at_x + (uint32_t)(16 * j) * K + k + 64 * h;
          s.x[j][h] = __builtin_amdgcn_raw_buffer_load_b128(rx, (WHOLE ? at : at & ~3u) | out_of, 0, 0);
          if (!WHOLE) s.x_next[j][h] = __builtin_amdgcn_raw_buffer_load_b32(rx, ((at & ~3u) + 16) | out_of, 0, 0);
        }
      }
      const int past = kb < nkb ? 0 : (int)kDmaOut;
#pragma unroll
      for (int j = 0; j < MB; j++)
        s.xs[j] =
            __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rs, ((16 * j + fr) * nkb + kb) * 4 | past, 0, 0));
      s.ws = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rt, kb * 4 | past, 0, 0));
    };
    auto multiply = [&](Stage& s, int kb) {
      if constexpr (!WHOLE) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
#pragma unroll
          for (int i = 0; i < RG; i++) s.w[i][h] = shift_bytes(s.w[i][h], s.w_next[i][h], at_w + 16 * i * K);
#pragma unroll
          for (int j = 0; j < MB; j++) s.x[j][h] = shift_bytes(s.x[j][h], s.x_next[j][h], at_x + 16 * j * K);
        }
        if (kb == nkb - 1) {
          const int left = K - (kb * kFp8Block + 16 * fg);
#pragma unroll
          for (int h = 0; h < 2; h++) {
#pragma unroll
            for (int i = 0; i < RG; i++) s.w[i][h] = first_bytes(s.w[i][h], left - 64 * h);
#pragma unroll
            for (int j = 0; j < MB; j++) s.x[j][h] = first_bytes(s.x[j][h], left - 64 * h);
          }
        }
      }
      bf16x8 fw[RG][4];
#pragma unroll
      for (int i = 0; i < RG; i++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
          fw[i][2 * h] = widen_fp8x8(s.w[i][h].x, s.w[i][h].y);
          fw[i][2 * h + 1] = widen_fp8x8(s.w[i][h].z, s.w[i][h].w);
        }
#pragma unroll
      for (int j = 0; j < MB; j++) {
        const float sc = s.xs[j] * s.ws;
        bf16x8 fx[4];
#pragma unroll
        for (int h = 0; h < 2; h++) {
          fx[2 * h] = widen_fp8x8(s.x[j][h].x, s.x[j][h].y);
          fx[2 * h + 1] = widen_fp8x8(s.x[j][h].z, s.x[j][h].w);
        }
#pragma unroll
        for (int i = 0; i < RG; i++) {
          f32x4 d = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int h = 0; h < 4; h++) d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fw[i][h], fx[h], d, 0, 0, 0);
#pragma unroll
          for (int r = 0; r < 4; r++) acc[i][j][r] = fmaf(d[r], sc, acc[i][j][r]);
        }
      }
    };
    constexpr int D = kStreamDepth;
    Stage ring[D];
#pragma unroll
    for (int d = 0; d < D; d++) load(ring[d], k0 + d * shape.ks);
    for (int kb = k0; kb < nkb; kb += D * shape.ks) {
#pragma unroll
      for (int d = 0; d < D; d++) {  // those past the last block multiply zeros
        multiply(ring[d], kb + d * shape.ks);
        load(ring[d], kb + (d + D) * shape.ks);
      }
    }
  }

  // The waves of a group add up into its first one.
  if (shape.ks > 1) {
    f32x4* held = reinterpret_cast<f32x4*>(lds);
    if (k0 > 0)
#pragma unroll
      for (int i = 0; i < RG; i++)
#pragma unroll
        for (int j = 0; j < MB; j++) held[(wave * RG * MB + i * MB + j) * 64 + lane] = acc[i][j];
    __syncthreads();
    if (k0 == 0)
      for (int w = 1; w < shape.ks; w++)
#pragma unroll
        for (int i = 0; i < RG; i++)
#pragma unroll
          for (int j = 0; j < MB; j++) {
            const f32x4 o = held[((wave + w) * RG * MB + i * MB + j) * 64 + lane];
#pragma unroll
            for (int r = 0; r < 4; r++) acc[i][j][r] += o[r];
          }
  }
  if constexpr (OUT == kOutScores) {
    // One part per workgroup and row: the groups' join in LDS.
    ScorePart* held = reinterpret_cast<ScorePart*>(lds);
    if (shape.ks > 1) __syncthreads();
    if (k0 == 0)
#pragma unroll
      for (int j = 0; j < MB; j++) {
        const int row = 16 * j + fr;
        const int token = out.tokens && row < p.m ? out.tokens[m0 + row] : -1;
        f32x4 v[RG];
#pragma unroll
        for (int i = 0; i < RG; i++) v[i] = acc[i][j];
        const ScorePart q = row_statistics<RG>(v, n0, fg, p.n, token, out.given + m0 + row);
        if (fg == 0) held[slot * (16 * MB) + row] = n0 < p.n ? q : empty_part();
      }
    __syncthreads();
    if (tid < 16 * MB && tid < p.m) {
      ScorePart q = held[tid];
      for (int g = 1; g < groups; g++) q = join(q, held[g * (16 * MB) + tid]);
      out.parts[(size_t)blockIdx.x * rows + m0 + tid] = q;
    }
  } else {
    char* y = static_cast<char*>(out.y) + (size_t)m0 * p.n * (OUT == kOutF32 ? 4 : 2);
    if (k0 == 0)
#pragma unroll
      for (int j = 0; j < MB; j++)
#pragma unroll
        for (int i = 0; i < RG; i++) store_columns<OUT>(p, y, 16 * j + fr, n0 + 16 * i + 4 * fg, acc[i][j]);
  }
}

struct StreamPlan {
  int rg, mb;
  StreamShape shape;
  dim3 grid;
  size_t lds;
};
static StreamPlan plan_stream(const Fp8Product& p, bool scores) {
  StreamPlan s;
  const int chunks = (p.m + kStreamRows - 1) / kStreamRows;
  s.mb = (std::min(p.m, kStreamRows) + 15) / 16;
  // Two groups of columns to a wave, which reads x half as often, where whole 64 rows are
  // enough work for half of the CUs all the same.
  s.rg = chunks > 1 && (p.n + 31) / 32 * chunks >= 128 ? 2 : 1;
  const int groups = (p.n + 16 * s.rg - 1) / (16 * s.rg);
  // Waves of a group: as many as fill the card, then as few as leave each the same
  // whole rounds of kStreamDepth blocks.
  const int want = std::min({stream_waves(s.mb), p.kblocks(), (2048 + groups * chunks - 1) / (groups * chunks)});
  int each = (p.kblocks() + want - 1) / want;
  each = (each + kStreamDepth - 1) / kStreamDepth * kStreamDepth;
  const int ks = (p.kblocks() + each - 1) / each;
  const int per = std::max(1, 4 / ks);
  s.shape.ks = ks;
  s.shape.waves = per * ks;
  s.grid = dim3((unsigned)((groups + per - 1) / per), (unsigned)chunks);
  s.lds = ks > 1 ? (size_t)s.shape.waves * s.rg * s.mb * 64 * sizeof(f32x4) : 0;
  if (scores) s.lds = std::max(s.lds, (size_t)per * 16 * s.mb * sizeof(ScorePart));
  return s;
}

// Few rows, or a small product, where the tiles would leave most of the card idle: by a
// model of both times. A CU's loads set the time here, 25 bytes per ns of x and of the
// matrix; measured against the model 0.75 to 1.2. f32 results here and on tiles: 16 x
// 6848 x 1280 5.7 and 8.3 us, 64 x 1280 x 1280 7.1 and 7.5, 48 x 4096 x 4096 13.8 and
// 12.8, 64 x 1280 x 6848 19.5 and 12.7, 512 x 896 x 1280 8.7 and 11.2, 512 x 1280 x 896
// 10.4 and 8.9, 1 x 20000 x 1280 8.8 and 10.7, 32 x 20000 x 1280 16.2 and 11.5.
static bool takes_stream(const Fp8Product& p, int kind, size_t work_bytes) {
  const size_t rows = (size_t)(p.m + kStreamRows - 1) / kStreamRows * kStreamRows;
  if (rows / kStreamRows > 65535) return false;  // a grid's second dimension
  if (p.m > kStreamRows && rows * (size_t)p.n * p.kblocks() > kStreamMost) return false;
  const StreamPlan t = plan_stream(p, kind == kOutScores);
  const size_t rounds = ((size_t)t.grid.x * t.grid.y + kCus - 1) / kCus;
  const size_t bytes =
      rounds * (t.shape.waves / t.shape.ks) * (16 * t.rg + std::min(p.m, kStreamRows)) * (size_t)p.k;
  const bool whole = whole_chunks(p);
  // The tiles' copy takes a launch, and its bytes each way at 3.3 TB/s.
  const double copy = whole ? 0.0 : 25 + 2.0 * fp8_packed_size(p) / 3.3e5;
  return 26 + bytes * (whole ? 4e-4 : 5e-4) <= copy + fp8_gemm_time(p, kind != kOutBf16, work_bytes);
}

template <int MB, int RG, bool WHOLE>
static void run_stream(const Fp8Product& p, const ProductOut& out, int kind, const StreamPlan& t, hipStream_t s) {
  const dim3 grid = t.grid, block(64 * t.shape.waves);
  if (kind == kOutF32)
    fp8_stream_kernel<MB, RG, kOutF32, WHOLE><<<grid, block, t.lds, s>>>(p, out, t.shape);
  else if (kind == kOutBf16)
    fp8_stream_kernel<MB, RG, kOutBf16, WHOLE><<<grid, block, t.lds, s>>>(p, out, t.shape);
  else
    fp8_stream_kernel<MB, RG, kOutScores, WHOLE><<<grid, block, t.lds, s>>>(p, out, t.shape);
}
template <bool WHOLE>
static void run_stream_rows(const Fp8Product& p, const ProductOut& out, int kind, const StreamPlan& t, hipStream_t s) {
  if (t.rg == 2) {
    run_stream<4, 2, WHOLE>(p, out, kind, t, s);
    return;
  }
  if (t.mb == 1) run_stream<1, 1, WHOLE>(p, out, kind, t, s);
  if (t.mb == 2) run_stream<2, 1, WHOLE>(p, out, kind, t, s);
  if (t.mb == 3) run_stream<3, 1, WHOLE>(p, out, kind, t, s);
  if (t.mb == 4) run_stream<4, 1, WHOLE>(p, out, kind, t, s);
}

// ---- few rows and many columns (a vocabulary): persistent workgroups of eight
// waves, one per CU, hold x in LDS and stream the matrix with kWideDepth scale
// blocks of 32 columns in flight per wave, across the ends of groups. Scores stay
// in registers until the last group: one part per workgroup and row.
// 129280 x 1280 (165 MB), scores: one row 33 us (5.0 TB/s; the same loads alone take
// 28.5), 48 rows 38.6 us. Four or five blocks in flight are 2 to 3 us slower, as are two
// workgroups per CU; waves that load x from the caches instead take 39 and 66 us. With
// 1279 columns 51 and 57 us, joins and all, against 37 and 40.
constexpr int kWideWaves = 8, kWideDepth = 2, kWideCols = 32;

struct WideShape {
  int groups;  // of kWideCols columns
};

constexpr size_t kWideParts = (size_t)kWideWaves * kStreamRows * sizeof(ScorePart);
static size_t wide_lds(const Fp8Product& p) {
  const size_t rows = (size_t)(p.m + 15) / 16 * 16;
  return rows * p.kblocks() * (kFp8Block + sizeof(float)) + kWideParts;
}

template <int MB, int OUT, bool WHOLE>
__global__ __launch_bounds__(64 * kWideWaves, 2) void fp8_wide_kernel(Fp8Product p, ProductOut out, WideShape shape) {
  constexpr int D = kWideDepth, R = kWideCols / 16;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int fr = lane & 15, fg = lane >> 4;
  const int K = p.k, nkb = p.kblocks();
  char* xl = lds;                                                        // [kb][16 MB rows][128]
  float* xsl = reinterpret_cast<float*>(lds + (size_t)nkb * MB * 16 * kFp8Block);  // [kb][16 MB rows]
  ScorePart* held = reinterpret_cast<ScorePart*>(xsl + nkb * MB * 16);

  struct Stage {
    u32x4 w[R][2];
    uint32_t next[WHOLE ? 1 : R][2];
    float ws;
  };
  // Every load is issued whatever is left to do, without a branch: what lies past a
  // row's last chunk, a group's last row or the wave's last group is out of its
  // resource's range and comes as zeros. Around a branch the compiler waits for all
  // loads instead of the oldest block's (37 -> 35 us for 129280 x 1280 and one row).
  // The tile scales come by vector loads for the same reason: scalar ones return in
  // no order, so each would be waited for with all others.
  const int tiles = (p.n + kFp8Block - 1) / kFp8Block;
  const __amdgpu_buffer_rsrc_t rt = read_rsrc(p.ws, (uint32_t)(tiles * nkb) * 4u);
  auto load = [&](Stage& s, int g, int kb) {
    const int n0 = g * kWideCols, k = kb * kFp8Block + 16 * fg;
    const int rows = g < shape.groups ? min(kWideCols, p.n - n0) : 0;
    const uint8_t* w0 = p.w + (size_t)n0 * K;
    const __amdgpu_buffer_rsrc_t rs = word_rsrc<WHOLE>(w0, (uint32_t)rows * K);
    const uint32_t at_w = (WHOLE ? 0 : misaligned(w0)) + (uint32_t)fr * K;
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int i = 0; i < R; i++) {
        const uint32_t at = at_w + (uint32_t)(16 * i) * K + k + 64 * h, out_of = k + 64 * h < K ? 0 : kDmaOut;
        s.w[i][h] = __builtin_amdgcn_raw_buffer_load_b128(rs, (WHOLE ? at : at & ~3u) | out_of, 0, 0);
        if (!WHOLE) s.next[i][h] = __builtin_amdgcn_raw_buffer_load_b32(rs, ((at & ~3u) + 16) | out_of, 0, 0);
      }
    const int at = g < shape.groups ? ((n0 / kFp8Block) * nkb + kb) * 4 : (int)kDmaOut;
    s.ws = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rt, at, 0, 0));
  };
  const int stride = (int)gridDim.x * kWideWaves;
  int g = (int)blockIdx.x * kWideWaves + wave;
  const int blocks = g < shape.groups ? ((shape.groups - 1 - g) / stride + 1) * nkb : 0;  // of this wave
  Stage ring[D];
  int next_g = g, next_kb = 0;
  auto load_next = [&](Stage& s) {
    load(s, next_g, next_kb);
    next_kb++;
    next_g = next_kb == nkb ? next_g + stride : next_g;
    next_kb = next_kb == nkb ? 0 : next_kb;
  };

  // x: chunk c of a row's 128 bytes at c ^ (row % 8), so that the sixteen rows of
  // a fragment read spread over all banks; zeros behind the last row and column.
  // The matrix's first loads are issued behind x's last ones, which return first:
  // in front of them, LDS would be filled only when the matrix has come.
  constexpr int kChunks = 3 * MB, kStep = 64 * kWideWaves;
  const __amdgpu_buffer_rsrc_t rx = word_rsrc<WHOLE>(p.x, (uint32_t)p.m * K);
  const __amdgpu_buffer_rsrc_t rxs = read_rsrc(p.xs, (uint32_t)(p.m * nkb) * 4u);
  const int chunks = nkb * MB * 16 * 8;
  u32x4 xv[kChunks];
  uint32_t x_next[WHOLE ? 1 : kChunks];
  auto load_x = [&](int c0) {
#pragma unroll
    for (int i = 0; i < kChunks; i++) {
      const int c = c0 + i * kStep + tid, k = c / (MB * 16 * 8) * kFp8Block + 16 * (c & 7);
      const int row = c / 8 % (MB * 16);
      const uint32_t at = (WHOLE ? 0 : misaligned(p.x)) + (uint32_t)row * K + k, out_of = k < K ? 0 : kDmaOut;
      xv[i] = __builtin_amdgcn_raw_buffer_load_b128(rx, (WHOLE ? at : at & ~3u) | out_of, 0, 0);
      if (!WHOLE) x_next[i] = __builtin_amdgcn_raw_buffer_load_b32(rx, ((at & ~3u) + 16) | out_of, 0, 0);
    }
  };
  auto store_x = [&](int c0) {
#pragma unroll
    for (int i = 0; i < kChunks; i++) {
      const int c = c0 + i * kStep + tid, row = c / 8;
      if constexpr (!WHOLE) {
        const int k = c / (MB * 16 * 8) * kFp8Block + 16 * (c & 7);
        xv[i] = first_bytes(shift_bytes(xv[i], x_next[i], misaligned(p.x) + row % (MB * 16) * K), K - k);
      }
      if (c < chunks) *reinterpret_cast<u32x4*>(xl + (size_t)row * 128 + 16 * ((c & 7) ^ (row & 7))) = xv[i];
    }
  };
  for (int c = tid; c < nkb * MB * 16; c += kStep) {
    const int row = c % (MB * 16);
    xsl[c] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(
        rxs, row < p.m ? (row * nkb + c / (MB * 16)) * 4 : (int)kDmaOut, 0, 0));
  }
  int c0 = 0;
  for (; c0 + kChunks * kStep < chunks; c0 += kChunks * kStep) {
    load_x(c0);
    store_x(c0);
  }
  load_x(c0);
#pragma unroll
  for (int d = 0; d < D; d++) load_next(ring[d]);
  store_x(c0);
  __syncthreads();

  ScorePart sum[MB];
  int token[MB];
  if constexpr (OUT == kOutScores)
#pragma unroll
    for (int j = 0; j < MB; j++) {
      sum[j] = empty_part();
      token[j] = out.tokens && 16 * j + fr < p.m ? out.tokens[16 * j + fr] : -1;
    }
  auto finish = [&](const f32x4 (&acc)[R][MB], int g) {
    const int n0 = g * kWideCols;
#pragma unroll
    for (int j = 0; j < MB; j++) {
      if constexpr (OUT == kOutScores) {
        f32x4 v[R];
#pragma unroll
        for (int i = 0; i < R; i++) v[i] = acc[i][j];
        sum[j] = join(sum[j], row_statistics<R>(v, n0, fg, p.n, token[j], out.given + 16 * j + fr));
      } else {
#pragma unroll
        for (int i = 0; i < R; i++) store_columns<OUT>(p, out.y, 16 * j + fr, n0 + 16 * i + 4 * fg, acc[i][j]);
      }
    }
  };
  f32x4 acc[R][MB];
#pragma unroll
  for (int i = 0; i < R; i++)
#pragma unroll
    for (int j = 0; j < MB; j++) acc[i][j] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
  int kb = 0;
  for (int at = 0; at < blocks; at += D) {
#pragma unroll
    for (int d = 0; d < D; d++) {  // those past the last block multiply zeros
      Stage& s = ring[d];
      if constexpr (!WHOLE) {
        const uint32_t by = misaligned(p.w + (size_t)g * kWideCols * K) + fr * K;
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
          for (int i = 0; i < R; i++) s.w[i][h] = shift_bytes(s.w[i][h], s.next[i][h], by + 16 * i * K);
        if (kb == nkb - 1)
#pragma unroll
          for (int h = 0; h < 2; h++)
#pragma unroll
            for (int i = 0; i < R; i++) s.w[i][h] = first_bytes(s.w[i][h], K - (kb * kFp8Block + 16 * fg + 64 * h));
      }
      bf16x8 fw[R][4];
#pragma unroll
      for (int i = 0; i < R; i++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
          fw[i][2 * h] = widen_fp8x8(s.w[i][h].x, s.w[i][h].y);
          fw[i][2 * h + 1] = widen_fp8x8(s.w[i][h].z, s.w[i][h].w);
        }
      const float ws = s.ws;
      load_next(ring[d]);
      const char* xb = xl + (size_t)kb * MB * 16 * 128;
#pragma unroll
      for (int j = 0; j < MB; j++) {
        const int row = 16 * j + fr;
        bf16x8 fx[4];
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const uint4 v = *reinterpret_cast<const uint4*>(xb + row * 128 + 16 * ((fg + 4 * h) ^ (row & 7)));
          fx[2 * h] = widen_fp8x8(v.x, v.y);
          fx[2 * h + 1] = widen_fp8x8(v.z, v.w);
        }
        const float sc = xsl[kb * MB * 16 + row] * ws;
#pragma unroll
        for (int i = 0; i < R; i++) {
          f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int h = 0; h < 4; h++) v = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fw[i][h], fx[h], v, 0, 0, 0);
#pragma unroll
          for (int r = 0; r < 4; r++) acc[i][j][r] = fmaf(v[r], sc, acc[i][j][r]);
        }
      }
      if (++kb == nkb) {
        if (at + d < blocks) finish(acc, g);
#pragma unroll
        for (int i = 0; i < R; i++)
#pragma unroll
          for (int j = 0; j < MB; j++) acc[i][j] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
        kb = 0;
        g += stride;
      }
    }
  }
  if constexpr (OUT == kOutScores) {
#pragma unroll
    for (int j = 0; j < MB; j++)
      if (fg == 0) held[wave * (16 * MB) + 16 * j + fr] = sum[j];
    __syncthreads();
    // Four threads to a row, two waves' parts each.
    static_assert(kWideWaves == 8, "two parts to a thread");
    const int row = tid / 4, w = 2 * (tid & 3);
    if (row < 16 * MB) {
      ScorePart q = join(held[w * (16 * MB) + row], held[(w + 1) * (16 * MB) + row]);
      q = join(q, shfl_xor(q, 1));
      q = join(q, shfl_xor(q, 2));
      if ((tid & 3) == 0 && row < p.m) out.parts[(size_t)blockIdx.x * p.m + row] = q;
    }
  }
}

template <int MB, bool WHOLE>
static void run_wide(const Fp8Product& p, const ProductOut& out, int kind, hipStream_t s) {
  const dim3 grid(kCus), block(64 * kWideWaves);
  const WideShape shape{(p.n + kWideCols - 1) / kWideCols};
  const size_t lds = wide_lds(p);
  if (kind == kOutF32)
    fp8_wide_kernel<MB, kOutF32, WHOLE><<<grid, block, lds, s>>>(p, out, shape);
  else if (kind == kOutBf16)
    fp8_wide_kernel<MB, kOutBf16, WHOLE><<<grid, block, lds, s>>>(p, out, shape);
  else
    fp8_wide_kernel<MB, kOutScores, WHOLE><<<grid, block, lds, s>>>(p, out, shape);
}

template <bool WHOLE>
static void run_wide_rows(const Fp8Product& p, const ProductOut& out, int kind, hipStream_t s) {
  const int mb = (p.m + 15) / 16;
  if (mb == 1) run_wide<1, WHOLE>(p, out, kind, s);
  if (mb == 2) run_wide<2, WHOLE>(p, out, kind, s);
  if (mb == 3) run_wide<3, WHOLE>(p, out, kind, s);
  if (mb == 4) run_wide<4, WHOLE>(p, out, kind, s);
}

template <int MB, bool WHOLE = true>
static void wide_attributes() {
  if (WHOLE) wide_attributes<MB, false>();
  const void* kernels[] = {(const void*)fp8_wide_kernel<MB, kOutF32, WHOLE>,
                           (const void*)fp8_wide_kernel<MB, kOutBf16, WHOLE>,
                           (const void*)fp8_wide_kernel<MB, kOutScores, WHOLE>};
  for (const void* k : kernels) (void)hipFuncSetAttribute(k, hipFuncAttributeMaxDynamicSharedMemorySize, kMostLds);
}
void fp8_init_attributes() {
  wide_attributes<1>();
  wide_attributes<2>();
  wide_attributes<3>();
  wide_attributes<4>();
  fp8_gemm_init_attributes();
  (void)hipGetLastError();  // a refused attribute surfaces at launch instead
}

// Enough columns to keep every wave at work, and x fits into LDS.
static bool takes_wide(const Fp8Product& p) {
  return p.m <= kStreamRows && p.n >= kCus * kWideWaves * kWideCols && wide_lds(p) <= (size_t)kMostLds;
}

static void launch_product(const Fp8Product& p, const ProductOut& out, int kind, void* work, size_t work_bytes,
                           hipStream_t s) {
  if (takes_wide(p)) {
    whole_chunks(p) ? run_wide_rows<true>(p, out, kind, s) : run_wide_rows<false>(p, out, kind, s);
  } else if (takes_stream(p, kind, work_bytes)) {
    const StreamPlan t = plan_stream(p, kind == kOutScores);
    whole_chunks(p) ? run_stream_rows<true>(p, out, kind, t, s) : run_stream_rows<false>(p, out, kind, t, s);
  } else {
    launch_fp8_gemm(p, out, kind, work, work_bytes, s);
  }
}

size_t fp8_pack_bytes(const Fp8Product& p, int ytype, size_t work_bytes) {
  if (whole_chunks(p) || takes_wide(p) || takes_stream(p, ytype == kTypeF32 ? kOutF32 : kOutBf16, work_bytes)) return 0;
  return fp8_packed_size(p);
}

void launch_fp8_linear(const Fp8Product& p, void* y, int ytype, void* work, size_t work_bytes, hipStream_t s) {
  launch_product(p, {y, nullptr, nullptr, nullptr}, ytype == kTypeF32 ? kOutF32 : kOutBf16, work, work_bytes, s);
}

// ------------------------------------------------- scores from the product

// Parts per row.
static int score_tiles(const Fp8Product& p) {
  if (takes_wide(p)) return kCus;
  return takes_stream(p, kOutScores, 0) ? (int)plan_stream(p, true).grid.x : fp8_gemm_parts(p);
}

size_t fp8_score_bytes(const Fp8Product& p) {
  // Room for p.m rows or fewer, whichever kernel takes them.
  const size_t most = kStreamMost / ((size_t)p.n * p.kblocks()) / kStreamRows * kStreamRows;
  const size_t streamed = std::min<size_t>(p.m, std::max<size_t>(most, kStreamRows));
  return std::max((size_t)fp8_gemm_parts(p) * p.m, (size_t)((p.n + 15) / 16) * streamed) * sizeof(ScorePart) +
         (size_t)p.m * 4;
}

// Joins the column tiles' statistics of each row. A workgroup of sixteen waves
// takes R rows (1, 4, 16 or 64, the wave's lanes being R rows of 64 / R tiles each,
// so that adjacent lanes read adjacent rows' parts): every thread some tiles, four
// loads in flight, then the lanes and the waves of a row, in trees. With one row or
// some dozens each thread has about one part: two dependent reads of memory in all.
// 256 parts of one row 4.8 us, of 48 rows 5.1 us, mostly the launch and those reads;
// 1010 of 4096 rows 22 us.
constexpr int kJoinWaves = 16;

template <int R>
__global__ __launch_bounds__(64 * kJoinWaves) void join_parts_kernel(const ScorePart* __restrict__ parts,
                                                                     int tiles, int m, int vocab,
                                                                     const float* __restrict__ given,
                                                                     TokenScores out, int* err) {
  __shared__ ScorePart held[kJoinWaves][R];
  constexpr int kStep = 64 * kJoinWaves / R;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane % R, row = (int)blockIdx.x * R + r;
  const int token = row < m && out.tokens ? out.tokens[row] : 0;
  const float logit = row < m && out.logprobs && token >= 0 && token < vocab ? given[row] : 0.0f;
  ScorePart p = empty_part();
  if (row < m) {
    const ScorePart* at = parts + row;
    for (int t = threadIdx.x / R; t < tiles; t += 4 * kStep) {
      ScorePart q[4];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        q[i] = empty_part();
        if (t + i * kStep < tiles) q[i] = at[(size_t)(t + i * kStep) * m];
      }
      p = join(p, join(join(q[0], q[1]), join(q[2], q[3])));
    }
  }
  p = lanes_join<R>(p);
  if (lane < R) held[wave][lane] = p;
  __syncthreads();
  if (wave > 0) return;
  // The waves' parts likewise: 64 / R lanes to a row.
  p = empty_part();
#pragma unroll
  for (int w = 0; w < kJoinWaves; w += 64 / R)
    if (w + lane / R < kJoinWaves) p = join(p, held[w + lane / R][r]);
  p = lanes_join<R>(p);
  if (lane >= R || row >= m) return;
  if (token < 0) {  // a padding row
    if (out.logprobs) out.logprobs[row] = 0.0f;
    if (out.entropy) out.entropy[row] = 0.0f;
    return;
  }
  write_scores(out, row, token, vocab, p, logit, err);
}

void launch_fp8_scores(const Fp8Product& p, const TokenScores& out, void* work, int* err,
                       hipStream_t s) {
  const int tiles = score_tiles(p);
  auto* parts = static_cast<ScorePart*>(work);
  auto* given = reinterpret_cast<float*>(parts + (size_t)tiles * p.m);
  const ProductOut po{nullptr, parts, out.logprobs ? out.tokens : nullptr, given};
  launch_product(p, po, kOutScores, nullptr, 0, s);
#define UOCR_JOIN(R)                                                                               \
  join_parts_kernel<R><<<(unsigned)((p.m + R - 1) / R), 64 * kJoinWaves, 0, s>>>(parts, tiles, p.m, p.n, \
                                                                                 given, out, err)
  if (p.m < 4)
    UOCR_JOIN(1);
  else if (p.m < 64)
    UOCR_JOIN(4);
  else if (p.m < 1024)
    UOCR_JOIN(16);
  else
    UOCR_JOIN(64);
#undef UOCR_JOIN
}

}  // namespace uocr
