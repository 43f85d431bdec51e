// The e4m3 product of many rows, on tiles that are staged through LDS.
#include <algorithm>

#include "fp8_device.hpp"

namespace uocr {

// Sixteen bytes of a row of K bytes from byte k, zeros behind the row's end.
// Rows start at any address where K is not a multiple of 16.
__device__ __forceinline__ uint4 load_chunk(const uint8_t* row, int k, int K) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (k + 16 <= K) {
    __builtin_memcpy(&v, row + k, 16);
  } else {
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 16; j++)
      if (k + j < K) w[j / 4] |= (uint32_t)row[k + j] << (8 * (j & 3));
    v = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return v;
}

// The product of rows whose bytes may start at any address (K no multiple of 16):
// 128 x 128 outputs per workgroup of four waves, 64 x 64 each, staged through
// registers. Not tuned.
template <int OUT>
__global__ __launch_bounds__(256) void fp8_bytes_kernel(Fp8Product p, ProductOut out) {
  constexpr int kT = 128;
  __shared__ __attribute__((aligned(16))) uint8_t lds_w[kT * 128], lds_x[kT * 128];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int n0 = (int)blockIdx.x * kT, m0 = (int)blockIdx.y * kT;
  const int wn = n0 + 64 * (wave & 1), wm = m0 + 64 * (wave >> 1);
  const int fr = lane & 15, fg = lane >> 4;
  const int K = p.k, nkb = p.kblocks();
  f32x4 acc[4][4];  // [16 columns][16 rows]
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int j = 0; j < 4; j++) acc[i][j] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};

  // Byte k of row r lies at chunk (k / 16) ^ (r % 8) of the row's 128 bytes:
  // the sixteen rows of a fragment read then spread over all banks.
  for (int kb = 0; kb < nkb; kb++) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int chunk = tid + 256 * i, r = chunk >> 3, c = chunk & 7;
      const int at = r * 128 + 16 * (c ^ (r & 7));
      uint4 a = make_uint4(0, 0, 0, 0), b = a;
      if (n0 + r < p.n) a = load_chunk(p.w + (size_t)(n0 + r) * K, kb * 128 + 16 * c, K);
      if (m0 + r < p.m) b = load_chunk(p.x + (size_t)(m0 + r) * K, kb * 128 + 16 * c, K);
      *reinterpret_cast<uint4*>(lds_w + at) = a;
      *reinterpret_cast<uint4*>(lds_x + at) = b;
    }
    __syncthreads();
    const float ws = p.ws[(size_t)(n0 / kFp8Block) * nkb + kb];
    // Lane group g takes chunks g and g + 4 of both operands: the order of
    // the 128 products inside a block is free.
    struct Fragment {
      bf16x8 part[4];
    };
    auto fragment = [&](const uint8_t* tile, int r) {
      const uint4 lo = *reinterpret_cast<const uint4*>(tile + r * 128 + 16 * (fg ^ (r & 7)));
      const uint4 hi = *reinterpret_cast<const uint4*>(tile + r * 128 + 16 * ((fg + 4) ^ (r & 7)));
      return Fragment{{widen_fp8x8(lo.x, lo.y), widen_fp8x8(lo.z, lo.w), widen_fp8x8(hi.x, hi.y),
                       widen_fp8x8(hi.z, hi.w)}};
    };
    Fragment fw[4];
#pragma unroll
    for (int i = 0; i < 4; i++) fw[i] = fragment(lds_w, wn - n0 + 16 * i + fr);
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const Fragment fx = fragment(lds_x, wm - m0 + 16 * j + fr);
      const int row = wm + 16 * j + fr;
      const float sc = row < p.m ? p.xs[(size_t)row * nkb + kb] * ws : 0.0f;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        f32x4 d = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int h = 0; h < 4; h++) d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fw[i].part[h], fx.part[h], d, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 4; r++) acc[i][j][r] = fmaf(d[r], sc, acc[i][j][r]);
      }
    }
  }

  if constexpr (OUT == kOutScores) {
    if (wn >= p.n) return;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int row = wm + 16 * j + fr;
      const int token = out.tokens && row < p.m ? out.tokens[row] : -1;
      const f32x4 v[4] = {acc[0][j], acc[1][j], acc[2][j], acc[3][j]};
      const ScorePart q = row_statistics<4>(v, wn, fg, p.n, token, out.given + row);
      if (fg == 0 && row < p.m) out.parts[(size_t)(wn / 64) * p.m + row] = q;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
      for (int i = 0; i < 4; i++) store_columns<OUT>(p, out.y, wm + 16 * j + fr, wn + 16 * i + 4 * fg, acc[i][j]);
  }
}

// ---- whole 16-byte chunks: TM x TN outputs per workgroup, 16 XB rows x 64 columns
// per wave. A stage is one scale block deep: TM + TN rows of 128 bytes, brought by
// global->LDS loads into one of two buffers while the other is multiplied. The
// matrix is the matrix instruction's first operand: lane l then holds four adjacent
// columns of y for row l % 16, whose x scale it needs as one value.
//
// WIDEN: the matrix cores' e4m3 instructions bring each group of eight products to
// the largest one's exponent and cut them off 13 bits below it (measured: 2^16 -
// 2^16 + v keeps multiples of 8; 1.3e-5 of a Gaussian block's sum). Results in f32
// and scores widen the operands to bf16 instead, whose products are summed to f32's
// last bit (1e-8): a scale block is a chain of four v_mfma_f32_16x16x32_bf16 from
// zero. bf16 results, rounded to 2^-9 anyway, take v_mfma_f32_16x16x128_f8f6f4, one
// per scale block, at twice the rate. Either way a block's sum is scaled into the f32
// accumulators when it is done.
template <int WAVES_M, int WAVES_N, int XB_>
struct TileShape {
  static constexpr int kWm = WAVES_M, kWn = WAVES_N, kWaves = WAVES_M * WAVES_N, XB = XB_;
  static constexpr int TM = WAVES_M * 16 * XB, TN = WAVES_N * 64;
  static constexpr uint32_t kStage = (TM + TN) * 128u;
  static constexpr size_t kLds = 2 * kStage;
};

template <class S, bool WIDEN, int OUT>
__global__ __launch_bounds__(64 * S::kWaves, 2) void fp8_tile_kernel(Fp8Product p, ProductOut out) {
  constexpr int XB = S::XB, TM = S::TM, TN = S::TN;
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int fr = lane & 15, fg = lane >> 4;
  const int K = p.k, nkb = p.kblocks();
  const int m0 = (int)blockIdx.y * TM, n0 = (int)blockIdx.x * TN;
  const int wm = wave / S::kWn * (16 * XB), wn = wave % S::kWn * 64;

  // Loads: a wave instruction brings 8 rows of 128 bytes; chunk c of row r lies at c
  // ^ (r % 8), which spreads a fragment read's sixteen rows over all banks.
  constexpr int kSegX = TM / 8 / S::kWaves, kSegW = TN / 8 / S::kWaves;
  const i32x4 rx = buffer_rsrc(p.x + (size_t)m0 * K, (uint32_t)min(TM, p.m - m0) * K);
  const i32x4 rw = buffer_rsrc(p.w + (size_t)n0 * K, (uint32_t)min(TN, p.n - n0) * K);
  const int chunk = (lane & 7) ^ (lane >> 3);
  const uint32_t xat = (uint32_t)(wave * kSegX * 8 + (lane >> 3)) * K + 16 * chunk;
  const uint32_t wat = (uint32_t)(wave * kSegW * 8 + (lane >> 3)) * K + 16 * chunk;
  const uint32_t lds0 = (uint32_t)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)lds);
  auto issue = [&](int buf, int kb) {
    const uint32_t k = (uint32_t)kb * 128u;
    const uint32_t past = (int)k + 16 * chunk < K ? 0u : kDmaOut;
    const uint32_t to = __builtin_amdgcn_readfirstlane(lds0 + (uint32_t)buf * S::kStage);
#pragma unroll
    for (int i = 0; i < kSegX; i++)
      buffer_load_lds16(rx, to + (uint32_t)(wave * kSegX + i) * 1024u, (xat + (uint32_t)(8 * i) * K + k) | past);
#pragma unroll
    for (int i = 0; i < kSegW; i++)
      buffer_load_lds16(rw, to + TM * 128u + (uint32_t)(wave * kSegW + i) * 1024u,
                        (wat + (uint32_t)(8 * i) * K + k) | past);
  };
  // Scales of the wave's rows (lane l: row l % 16 of each block) and of its columns,
  // which lie in one tile of the matrix.
  const __amdgpu_buffer_rsrc_t rxs = read_rsrc(p.xs + (size_t)m0 * nkb, (uint32_t)(min(TM, p.m - m0) * nkb) * 4u);
  const __amdgpu_buffer_rsrc_t rws =
      read_rsrc(p.ws, (uint32_t)((p.n + kFp8Block - 1) / kFp8Block * nkb) * 4u);
  const int wsat = (n0 + wn) / kFp8Block * nkb;
  struct Scales {
    float x[XB], w;
  };
  auto load_scales = [&](Scales& s, int kb) {
#pragma unroll
    for (int j = 0; j < XB; j++)
      s.x[j] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rxs, ((wm + 16 * j + fr) * nkb + kb) * 4, 0, 0));
    s.w = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rws, (wsat + kb) * 4, 0, 0));
  };

  f32x4 acc[4][XB];
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int j = 0; j < XB; j++) acc[i][j] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
  auto chunk_at = [&](const char* tile, int r, int c) {
    return *reinterpret_cast<const u32x4*>(tile + r * 128 + 16 * (c ^ (r & 7)));
  };
  // Lane group g takes chunks g and g + 4 of both operands: the order of the 128
  // products inside a block is free.
  struct Wide {
    bf16x8 part[4];
  };
  auto widen = [&](u32x4 lo, u32x4 hi) {
    return Wide{{widen_fp8x8(lo.x, lo.y), widen_fp8x8(lo.z, lo.w), widen_fp8x8(hi.x, hi.y), widen_fp8x8(hi.z, hi.w)}};
  };
  auto join8 = [&](u32x4 lo, u32x4 hi) {
    return (i32x8){(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w, (int)hi.x, (int)hi.y, (int)hi.z, (int)hi.w};
  };
  auto multiply = [&](int buf, const Scales& s) {
    const char* xt = lds + (size_t)buf * S::kStage;
    const char* wt = xt + TM * 128;
    if constexpr (WIDEN) {
      Wide fw[4];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int r = wn + 16 * i + fr;
        fw[i] = widen(chunk_at(wt, r, fg), chunk_at(wt, r, fg + 4));
      }
#pragma unroll
      for (int j = 0; j < XB; j++) {
        const int r = wm + 16 * j + fr;
        const Wide fx = widen(chunk_at(xt, r, fg), chunk_at(xt, r, fg + 4));
        const float sc = s.x[j] * s.w;
        f32x4 d[4];
#pragma unroll
        for (int i = 0; i < 4; i++) d[i] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int h = 0; h < 4; h++)
#pragma unroll
          for (int i = 0; i < 4; i++)
            d[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fw[i].part[h], fx.part[h], d[i], 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
          for (int r4 = 0; r4 < 4; r4++) acc[i][j][r4] = fmaf(d[i][r4], sc, acc[i][j][r4]);
      }
    } else {
      i32x8 fw[4];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int r = wn + 16 * i + fr;
        fw[i] = join8(chunk_at(wt, r, fg), chunk_at(wt, r, fg + 4));
      }
#pragma unroll
      for (int j = 0; j < XB; j++) {
        const int r = wm + 16 * j + fr;
        const i32x8 fx = join8(chunk_at(xt, r, fg), chunk_at(xt, r, fg + 4));
        const float sc = s.x[j] * s.w;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
          const f32x4 d = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fw[i], fx, zero, 0, 0, 0, 0, 0, 0);
#pragma unroll
          for (int r4 = 0; r4 < 4; r4++) acc[i][j][r4] = fmaf(d[r4], sc, acc[i][j][r4]);
        }
      }
    }
  };

  Scales now, next;
  issue(0, 0);
  load_scales(now, 0);
  __builtin_amdgcn_s_waitcnt(vmcnt_only(0));
  __syncthreads();
  for (int kb = 0; kb < nkb; kb++) {
    if (kb + 1 < nkb) {
      issue((kb + 1) & 1, kb + 1);
      load_scales(next, kb + 1);
    }
    multiply(kb & 1, now);
    now = next;
    __builtin_amdgcn_s_waitcnt(vmcnt_only(0));
    __syncthreads();
  }

  if constexpr (OUT == kOutScores) {
    // One part per tile and row: the columns' waves join in LDS.
    ScorePart* held = reinterpret_cast<ScorePart*>(lds);
#pragma unroll
    for (int j = 0; j < XB; j++) {
      const int r = wm + 16 * j + fr, row = m0 + r;
      const int token = out.tokens && row < p.m ? out.tokens[row] : -1;
      const f32x4 v[4] = {acc[0][j], acc[1][j], acc[2][j], acc[3][j]};
      ScorePart q = empty_part();
      if (n0 + wn < p.n) q = row_statistics<4>(v, n0 + wn, fg, p.n, token, out.given + row);
      if (fg == 0) held[wave % S::kWn * TM + r] = q;
    }
    __syncthreads();
    for (int r = tid; r < TM && m0 + r < p.m; r += 64 * S::kWaves) {
      ScorePart q = held[r];
      for (int w = 1; w < S::kWn; w++) q = join(q, held[w * TM + r]);
      out.parts[(size_t)blockIdx.x * p.m + m0 + r] = q;
    }
  } else {
#pragma unroll
    for (int j = 0; j < XB; j++)
#pragma unroll
      for (int i = 0; i < 4; i++)
        store_columns<OUT>(p, out.y, m0 + wm + 16 * j + fr, n0 + wn + 16 * i + 4 * fg, acc[i][j]);
  }
}

using Tile256 = TileShape<2, 4, 8>;
using Tile128 = TileShape<2, 2, 4>;

template <class S, bool WIDEN, int OUT>
static void run_tiles(const Fp8Product& p, const ProductOut& out, hipStream_t s) {
  const dim3 grid((unsigned)((p.n + S::TN - 1) / S::TN), (unsigned)((p.m + S::TM - 1) / S::TM));
  fp8_tile_kernel<S, WIDEN, OUT><<<grid, 64 * S::kWaves, S::kLds, s>>>(p, out);
}

using ScoreTile = Tile128;

int fp8_gemm_parts(const Fp8Product& p) {
  return whole_chunks(p) ? (p.n + ScoreTile::TN - 1) / ScoreTile::TN : (p.n + 63) / 64;
}

void fp8_gemm_init_attributes() {
  const void* kernels[] = {(const void*)fp8_tile_kernel<Tile256, false, kOutBf16>,
                           (const void*)fp8_tile_kernel<Tile128, true, kOutF32>,
                           (const void*)fp8_tile_kernel<ScoreTile, true, kOutScores>};
  for (const void* k : kernels) (void)hipFuncSetAttribute(k, hipFuncAttributeMaxDynamicSharedMemorySize, kMostLds);
}

void launch_fp8_gemm(const Fp8Product& p, const ProductOut& out, int kind, hipStream_t s) {
  if (!whole_chunks(p)) {
    const dim3 grid((unsigned)((p.n + 127) / 128), (unsigned)((p.m + 127) / 128));
    if (kind == kOutF32)
      fp8_bytes_kernel<kOutF32><<<grid, 256, 0, s>>>(p, out);
    else if (kind == kOutBf16)
      fp8_bytes_kernel<kOutBf16><<<grid, 256, 0, s>>>(p, out);
    else
      fp8_bytes_kernel<kOutScores><<<grid, 256, 0, s>>>(p, out);
  } else if (kind == kOutF32) {
    run_tiles<Tile128, true, kOutF32>(p, out, s);
  } else if (kind == kOutBf16) {
    run_tiles<Tile256, false, kOutBf16>(p, out, s);
  } else {
    run_tiles<ScoreTile, true, kOutScores>(p, out, s);
  }
}

}  // namespace uocr
