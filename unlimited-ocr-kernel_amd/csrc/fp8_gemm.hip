// The e4m3 product of many rows, on tiles that are staged through LDS.
#include <algorithm>

#include "fp8_device.hpp"

namespace uocr {

// Sixteen bytes of a row of K bytes from byte k, zeros behind the row's end, of rows that
// start at any address: by the aligned words that hold any of them.
__device__ __forceinline__ uint4 load_chunk(const uint8_t* row, int k, int K) {
  if (k >= K) return make_uint4(0, 0, 0, 0);
  const int left = min(K - k, 16), by = (int)misaligned(row + k);
  const auto* at = reinterpret_cast<const uint32_t*>(row + k - by);
  const int words = (by + left + 3) / 4;
  u32x4 v = {0, 0, 0, 0};
  if (words >= 4) {
    __builtin_memcpy(&v, __builtin_assume_aligned(at, 4), 16);
  } else {
#pragma unroll
    for (int i = 0; i < 3; i++)
      if (i < words) v[i] = at[i];
  }
  v = first_bytes(shift_bytes(v, words == 5 ? at[4] : 0, by), left);
  return make_uint4(v.x, v.y, v.z, v.w);
}

// Both operands with rows of whole chunks, a chunk per thread. 4096 x 6848 x 1279 f32:
// 219 us on the kernel below, 99 with such a copy and its tiles; 277 x 1280 x 6847 194 and
// 26.
__global__ __launch_bounds__(256) void fp8_pack_kernel(Fp8Product p, uint8_t* __restrict__ x, uint8_t* __restrict__ w) {
  const uint32_t chunks = (p.k + 15) / 16, all_x = p.m * chunks, all = all_x + p.n * chunks;
  uint32_t c = blockIdx.x * 256 + threadIdx.x;
  if (c >= all) return;
  const bool second = c >= all_x;
  if (second) c -= all_x;
  const uint4 v = load_chunk((second ? p.w : p.x) + (size_t)(c / chunks) * p.k, (int)(c % chunks) * 16, p.k);
  reinterpret_cast<uint4*>(second ? w : x)[c] = v;
}

// A thread per chunk, counted in 32 bits: larger copies have no room anywhere.
constexpr size_t kMostPacked = (size_t)1 << 35;
static size_t pack_part(int rows, int k) { return ((size_t)rows * ((k + 15) / 16) * 16 + 255) / 256 * 256; }
size_t fp8_packed_size(const Fp8Product& p) {
  const size_t bytes = pack_part(p.m, p.k) + pack_part(p.n, p.k);
  return bytes < kMostPacked ? bytes : SIZE_MAX / 2;
}
Fp8Product launch_fp8_pack(const Fp8Product& p, void* work, hipStream_t s) {
  auto* x = static_cast<uint8_t*>(work);
  uint8_t* w = x + pack_part(p.m, p.k);
  const size_t chunks = ((size_t)p.m + p.n) * ((p.k + 15) / 16);
  fp8_pack_kernel<<<(unsigned)((chunks + 255) / 256), 256, 0, s>>>(p, x, w);
  return {x, p.xs, w, p.ws, p.m, p.n, (p.k + 15) / 16 * 16};
}

// The product of rows whose bytes may start at any address (K no multiple of 16), where
// there is no room for a copy: 128 x 128 outputs per workgroup of four waves, 64 x 64
// each, staged through registers. Not tuned.
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

// ---- whole 16-byte chunks: 128 x 128 or 64 x 128 outputs per workgroup of four waves,
// 64 x 64 or 32 x 64 each. A stage is one scale block deep: the tile's rows and columns,
// 128 bytes of each, brought by global->LDS loads into a ring of buffers ahead of the one
// that is multiplied. The matrix is the matrix instruction's first operand: lane l then
// holds groups of four adjacent columns of y for one row of x, whose scale it needs as one
// value.
//
// WIDEN: the matrix cores' e4m3 instructions bring each group of eight products to
// the largest one's exponent and cut them off 13 bits below it (measured: 2^16 -
// 2^16 + v keeps multiples of 8; 1.3e-5 of a Gaussian block's sum). Results in f32
// and scores widen the operands to bf16 instead, whose products are summed to f32's
// last bit (1e-8): a scale block is a chain of eight v_mfma_f32_32x32x16_bf16 from zero
// (four v_mfma_f32_16x16x32_bf16 are twice the instructions to issue: 277 x 1280 x 6848
// 16.4 -> 15.6 us, 100 x 20000 x 1280 scores 16.0 -> 14.2). bf16 results, rounded to 2^-9 anyway, take v_mfma_f32_16x16x128_f8f6f4, one
// per scale block, at twice the rate. Either way a block's sum is scaled into the f32
// accumulators when it is done.
//
// BUFS stages of LDS, so that workgroups share a CU and hide each other's waits: two
// stages with tiles of 128 rows, two workgroups to a CU; with tiles of 64 rows two stages
// and three workgroups (WIDEN: 600 x 6848 x 1280 scores 24.2 us with three stages, 21.2
// with two), or three stages and two workgroups (bf16 results, whose steps are shorter:
// 2048 x 1280 x 6848 41 and 43.5 us). The smaller tiles are taken where all of them fit
// the card at once: more of them, less padding (277 x 1280 x 6848 f32 20.9 -> 16.8 us,
// 1024 x 1280 x 896 bf16 9.6 -> 7.1, 3500 x 1280 x 6848 f32 100 -> 92; beyond, 1024 x
// 6848 x 1280 f32 is 26.7 us with 128 rows and 29.9 with 64). Few tiles of a long depth
// are also split along it: each split leaves f32 partial sums in memory, and a second
// launch adds them in order.
//
// 4096 x 6848 x 1280 bf16 55 us (1310 TFLOP/s): the loads bring 17 TB/s into LDS, which is
// what bounds the steps, and the stores take 10 us. 4096 x 129280 x 1280 scores 1246 us
// (1090 TFLOP/s): the vector instructions (3.4 to 16 x 16 x 32 products, of them 2 of
// widening and 1 of scaling, and the statistics') share the issue with the products.
constexpr int kCols = 128;  // columns of a tile
constexpr int short_bufs(bool widen) { return widen ? 2 : 3; }
constexpr int short_per_cu(bool widen) { return widen ? 3 : 2; }
constexpr int tile_rows(int xb) { return 32 * xb; }  // for xb blocks of 16 rows in each of two waves
constexpr uint32_t stage_bytes(int xb) { return (tile_rows(xb) + kCols) * 128u; }
// Scales of eight blocks: x's [8][rows of the tile], the matrix's [8].
constexpr uint32_t scale_bytes(int xb) { return (8 * tile_rows(xb) + 8) * 4u; }
constexpr size_t tile_lds(int bufs, int xb) { return bufs * stage_bytes(xb) + 2 * scale_bytes(xb); }

// Workgroups reach the 8 XCDs round-robin, each XCD with an L2 of its own. They are
// renumbered so that an XCD takes a contiguous run of tiles, and tiles run down strips
// of kStrip row tiles: the tiles at work on an XCD at once are near square, so that
// together they read the fewest rows of x and w.
constexpr int kStrip = 8;
struct TileAt {
  int m, n;
};
__device__ __forceinline__ TileAt tile_of(int id, int tiles_m, int tiles_n) {
  const int total = tiles_m * tiles_n, xcd = id % kXcds, each = total / kXcds, more = total % kXcds;
  const int at = xcd * each + min(xcd, more) + id / kXcds;
  const int strip = at / (kStrip * tiles_n), in = at % (kStrip * tiles_n);
  const int rows = min(kStrip, tiles_m - strip * kStrip);
  return {strip * kStrip + in % rows, in / rows};
}

// Blocks [split * each, + each) of the depth; a split's results go to its own [m, n]
// of y.
struct Splits {
  int count, each;
};

// Four adjacent columns of a 32 x 32 block's sixteen.
__device__ __forceinline__ f32x4 quarter(const f32x16& v, int i) {
  return (f32x4){v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]};
}

template <bool WIDEN, int OUT, int BUFS, int XB>
__global__ __launch_bounds__(256, 2) void fp8_tile_kernel(Fp8Product p, ProductOut out, Splits splits) {
  constexpr int kRows = tile_rows(XB);
  constexpr uint32_t kStage = stage_bytes(XB), kScales = scale_bytes(XB);
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int fr = lane & 15, fg = lane >> 4;
  const int K = p.k, nkb = p.kblocks();
  const int tiles_m = (p.m + kRows - 1) / kRows, tiles_n = (p.n + kCols - 1) / kCols;
  // The splits of a tile lie far apart: an XCD works on neighbouring tiles at one depth.
  const int split = (int)blockIdx.x / (tiles_m * tiles_n);
  const TileAt tile = tile_of((int)blockIdx.x % (tiles_m * tiles_n), tiles_m, tiles_n);
  const int first = split * splits.each, last = min(nkb, first + splits.each);
  const int m0 = tile.m * kRows, n0 = tile.n * kCols;
  const int wm = wave / 2 * (16 * XB), wn = wave % 2 * 64;

  // Loads: a wave instruction brings 8 rows of 128 bytes; chunk c of row r lies at c
  // ^ (r / 2 % 8), which spreads a fragment read's rows, sixteen of two chunks or 32 of
  // one, over all banks (two rows fill them).
  constexpr int kSegsX = kRows / 8 / 4, kSegsW = kCols / 8 / 4, kLoads = kSegsX + kSegsW;
  const i32x4 rx = buffer_rsrc(p.x + (size_t)m0 * K, (uint32_t)min(kRows, p.m - m0) * K);
  const i32x4 rw = buffer_rsrc(p.w + (size_t)n0 * K, (uint32_t)min(kCols, p.n - n0) * K);
  static_assert(kSegsX % 2 == 0 && kSegsW % 2 == 0, "a wave's first rows are a multiple of 16");
  const uint32_t chunk[2] = {(uint32_t)((lane & 7) ^ (lane >> 4)) * 16, (uint32_t)((lane & 7) ^ (lane >> 4) ^ 4) * 16};
  const uint32_t at_x = (uint32_t)(wave * kSegsX * 8 + (lane >> 3)) * K;
  const uint32_t at_w = (uint32_t)(wave * kSegsW * 8 + (lane >> 3)) * K;
  const uint32_t lds0 = (uint32_t)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)lds);
  auto issue = [&](int kb) {
    const uint32_t k = (uint32_t)kb * 128u;
    uint32_t at[2];
#pragma unroll
    for (int i = 0; i < 2; i++) at[i] = (k + chunk[i]) | ((int)(k + chunk[i]) < K ? 0u : kDmaOut);
    const uint32_t to = __builtin_amdgcn_readfirstlane(lds0 + (uint32_t)(kb % BUFS) * kStage);
#pragma unroll
    for (int i = 0; i < kSegsW; i++) {
      if (i < kSegsX)
        buffer_load_lds16(rx, to + (uint32_t)(wave * kSegsX + i) * 1024u, at_x + (uint32_t)(8 * i) * K + at[i & 1]);
      buffer_load_lds16(rw, to + kRows * 128u + (uint32_t)(wave * kSegsW + i) * 1024u,
                        at_w + (uint32_t)(8 * i) * K + at[i & 1]);
    }
  };
  // Scales of eight blocks at a time, in LDS beside the stages. A thread brings four
  // blocks of one row of x (16 bytes; a lane per row and block, 4 bytes each of a line
  // of its own, took as long as the stages), some one of the matrix's.
  const __amdgpu_buffer_rsrc_t rxs = read_rsrc(p.xs + (size_t)m0 * nkb, (uint32_t)(min(kRows, p.m - m0) * nkb) * 4u);
  const __amdgpu_buffer_rsrc_t rws = read_rsrc(p.ws + (size_t)tile.n * nkb, (uint32_t)nkb * 4u);
  struct Scales {
    u32x4 x;
    uint32_t w;
  };
  auto load_scales = [&](int eighth) {  // blocks past the last one: anything
    Scales s;
    s.x = __builtin_amdgcn_raw_buffer_load_b128(rxs, ((tid >> 1) * nkb + 8 * eighth + 4 * (tid & 1)) * 4, 0, 0);
    s.w = __builtin_amdgcn_raw_buffer_load_b32(rws, (8 * eighth + (tid & 7)) * 4, 0, 0);
    return s;
  };
  auto scales_at = [&](int eighth) { return reinterpret_cast<float*>(lds + BUFS * kStage + (eighth & 1) * kScales); };
  auto store_scales = [&](int eighth, const Scales& s) {
    float* to = scales_at(eighth);
    if (kRows == 128 || tid < 2 * kRows)
#pragma unroll
      for (int i = 0; i < 4; i++) to[(4 * (tid & 1) + i) * kRows + (tid >> 1)] = __uint_as_float(s.x[i]);
    if (tid < 8) to[8 * kRows + tid] = __uint_as_float(s.w);
  };

  // WIDEN: blocks of 32 x 32 (twice XB / 2 of them in a wave), whose lane l has row l % 32
  // of x and columns 8 i + 4 (l / 32) + r; otherwise of 16 x 16.
  constexpr int JB = XB / 2;
  const int r32 = lane & 31, half = lane >> 5;
  f32x4 acc[4][XB];
  f32x16 wide[2][JB];
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int j = 0; j < XB; j++) acc[i][j] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < 2; i++)
#pragma unroll
    for (int j = 0; j < JB; j++)
#pragma unroll
      for (int r = 0; r < 16; r++) wide[i][j][r] = 0.0f;
  auto chunk_at = [&](const char* tile, int r, int c) {
    return *reinterpret_cast<const u32x4*>(tile + r * 128 + 16 * (c ^ (r / 2 & 7)));
  };
  // One stage. The order of the 128 products inside a block is free, so lanes take whole
  // chunks of their rows. What stands between products is held there by sched_barrier:
  // left to itself the compiler waits for each product before it scales it.
  auto multiply = [&](int kb) {
    const char* xt = lds + (size_t)(kb % BUFS) * kStage;
    const char* wt = xt + kRows * 128;
    const float* xs = scales_at(kb >> 3) + (kb & 7) * kRows + wm;
    const float ws = scales_at(kb >> 3)[8 * kRows + (kb & 7)];
    if constexpr (WIDEN) {
      // Lane half g takes chunks 4 g to 4 g + 3, eight bytes to a product; the operands
      // of the next eight are widened under the products of these.
      u32x4 w4[2][4], x4[JB][4];
#pragma unroll
      for (int t = 0; t < 4; t++) {
#pragma unroll
        for (int j = 0; j < JB; j++) x4[j][t] = chunk_at(xt, wm + 32 * j + r32, 4 * half + t);
#pragma unroll
        for (int i = 0; i < 2; i++) w4[i][t] = chunk_at(wt, wn + 32 * i + r32, 4 * half + t);
      }
      float sc[JB];
#pragma unroll
      for (int j = 0; j < JB; j++) sc[j] = xs[32 * j + r32] * ws;
      auto part = [&](const u32x4 (&v)[4], int u) { return widen_fp8x8(v[u / 2][2 * (u & 1)], v[u / 2][2 * (u & 1) + 1]); };
      bf16x8 fw[2][2], fx[2][JB];
      f32x16 d[2][JB];
#pragma unroll
      for (int j = 0; j < JB; j++) fx[0][j] = part(x4[j], 0);
#pragma unroll
      for (int i = 0; i < 2; i++) fw[0][i] = part(w4[i], 0);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int u = 0; u < 8; u++) {
#pragma unroll
        for (int j = 0; j < JB; j++)
#pragma unroll
          for (int i = 0; i < 2; i++) {
            if (u == 0)
#pragma unroll
              for (int r = 0; r < 16; r++) d[i][j][r] = 0.0f;
            d[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fw[u & 1][i], fx[u & 1][j], d[i][j], 0, 0, 0);
            if (u < 7) {
              if (j == 0) fw[(u + 1) & 1][i] = part(w4[i], u + 1);
              if (j == JB - 1 && i < JB) fx[(u + 1) & 1][i] = part(x4[i], u + 1);
            }
            __builtin_amdgcn_sched_barrier(0);
          }
      }
#pragma unroll
      for (int j = 0; j < JB; j++)
#pragma unroll
        for (int i = 0; i < 2; i++) {
#pragma unroll
          for (int r = 0; r < 16; r++) wide[i][j][r] = fmaf(d[i][j][r], sc[j], wide[i][j][r]);
          asm volatile("" : "+v"(wide[i][j]));  // here, not sunk behind the loop's next branch
        }
    } else {
      // Lane group g takes chunks g and g + 4. While row block j is multiplied, block j - 1's
      // sums are scaled and block j + 1's fragment is read.
      struct Raw {
        u32x4 half[2];
      };
      auto read = [&](const char* tile, int r) { return Raw{{chunk_at(tile, r, fg), chunk_at(tile, r, fg + 4)}}; };
      auto scale = [&](f32x4& a, const f32x4& d, float sc) {
#pragma unroll
        for (int r = 0; r < 4; r++) a[r] = fmaf(d[r], sc, a[r]);
        asm volatile("" : "+v"(a));
      };
      float sc[2];
      f32x4 d[2][4];
      auto whole = [&](const Raw& v) {
        return (i32x8){(int)v.half[0].x, (int)v.half[0].y, (int)v.half[0].z, (int)v.half[0].w,
                       (int)v.half[1].x, (int)v.half[1].y, (int)v.half[1].z, (int)v.half[1].w};
      };
      Raw fw[4], fx[2];
      fx[0] = read(xt, wm + fr);
#pragma unroll
      for (int i = 0; i < 4; i++) fw[i] = read(wt, wn + 16 * i + fr);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < XB; j++) {
        if (j + 1 < XB) fx[(j + 1) & 1] = read(xt, wm + 16 * (j + 1) + fr);
        sc[j & 1] = xs[16 * j + fr] * ws;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
          d[j & 1][i] =
              __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(whole(fw[i]), whole(fx[j & 1]), zero, 0, 0, 0, 0, 0, 0);
          if (j > 0) scale(acc[i][j - 1], d[(j - 1) & 1][i], sc[(j - 1) & 1]);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; i++) scale(acc[i][XB - 1], d[(XB - 1) & 1][i], sc[(XB - 1) & 1]);
    }
  };

  // Stage kb is multiplied while the BUFS - 1 behind it are on their way. A wave's loads
  // return in order, so its own part of stage kb is there when at most those of the
  // later stages are outstanding; the barrier then publishes every wave's, and says
  // that stage kb - 1, whose buffer the next loads fill, has been read.
  constexpr int kAhead = BUFS - 1;
  Scales next = load_scales(first >> 3);
  for (int i = 0; i < kAhead; i++)
    if (first + i < last) issue(first + i);
  store_scales(first >> 3, next);
  next = load_scales((first >> 3) + 1);
  for (int kb = first; kb < last; kb++) {
    if (kb + kAhead <= last)
      __builtin_amdgcn_s_waitcnt(vmcnt_only((kAhead - 1) * kLoads));
    else
      __builtin_amdgcn_s_waitcnt(vmcnt_only(0));
    __syncthreads();
    if (kb + kAhead < last) issue(kb + kAhead);
    __builtin_amdgcn_sched_barrier(0);
    multiply(kb);
    __builtin_amdgcn_sched_barrier(0);
    // The other eight blocks' scales were last read a step or more ago.
    if ((kb & 7) == 7) {
      store_scales((kb >> 3) + 1, next);
      next = load_scales((kb >> 3) + 2);
    }
  }

  if constexpr (OUT == kOutScores) {
    // One part per tile and row: the two waves of a row join in LDS.
    ScorePart* held = reinterpret_cast<ScorePart*>(lds);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < JB; j++) {
      const int r = wm + 32 * j + r32, row = m0 + r;
      const int token = out.tokens && row < p.m ? out.tokens[row] : -1;
      f32x4 v[8];
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] = quarter(wide[i / 4][j], i % 4);
      ScorePart q = empty_part();
      if (n0 + wn < p.n) q = row_statistics<8, 8>(v, n0 + wn, half, p.n, token, out.given + row);
      if (half == 0) held[wave % 2 * kRows + r] = q;
    }
    __syncthreads();
    if (tid < kRows && m0 + tid < p.m)
      out.parts[(size_t)tile.n * p.m + m0 + tid] = join(held[tid], held[kRows + tid]);
  } else {
    char* y = static_cast<char*>(out.y) + (size_t)split * p.m * p.n * (OUT == kOutF32 ? 4 : 2);
    if constexpr (WIDEN) {
#pragma unroll
      for (int j = 0; j < JB; j++)
#pragma unroll
        for (int i = 0; i < 8; i++)
          store_columns<OUT>(p, y, m0 + wm + 32 * j + r32, n0 + wn + 8 * i + 4 * half, quarter(wide[i / 4][j], i % 4));
      return;
    }
#pragma unroll
    for (int j = 0; j < XB; j++)
#pragma unroll
      for (int i = 0; i < 4; i++)
        store_columns<OUT>(p, y, m0 + wm + 16 * j + fr, n0 + wn + 16 * i + 4 * fg, acc[i][j]);
  }
}

// Adds the splits' partial sums in order.
template <int OUT>
__global__ __launch_bounds__(256) void add_splits_kernel(const float* __restrict__ parts, size_t count, int splits,
                                                         void* __restrict__ y) {
  const size_t i = ((size_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= count) return;
  if (i + 4 <= count) {
    f32x4 a;
    __builtin_memcpy(&a, parts + i, 16);
#pragma unroll 4
    for (int s = 1; s < splits; s++) {
      f32x4 b;
      __builtin_memcpy(&b, parts + s * count + i, 16);
#pragma unroll
      for (int r = 0; r < 4; r++) a[r] += b[r];
    }
    if (OUT == kOutF32) {
      __builtin_memcpy(static_cast<float*>(y) + i, &a, 16);
    } else {
      const uint2 b = make_uint2(bf16_pair(a[0], a[1]), bf16_pair(a[2], a[3]));
      __builtin_memcpy(static_cast<uint16_t*>(y) + i, &b, 8);
    }
    return;
  }
  for (size_t e = i; e < count; e++) {
    float a = parts[e];
    for (int s = 1; s < splits; s++) a += parts[s * count + e];
    if (OUT == kOutF32)
      static_cast<float*>(y)[e] = a;
    else
      static_cast<uint16_t*>(y)[e] = bf16_bits(a);
  }
}

static size_t tiles_of(const Fp8Product& p, int rows) {
  return (size_t)((p.n + kCols - 1) / kCols) * ((p.m + rows - 1) / rows);
}

template <bool WIDEN, int OUT, int BUFS, int XB>
static void run_tiles(const Fp8Product& p, const ProductOut& out, const Splits& splits, hipStream_t s) {
  fp8_tile_kernel<WIDEN, OUT, BUFS, XB>
      <<<(unsigned)(tiles_of(p, tile_rows(XB)) * splits.count), 256, tile_lds(BUFS, XB), s>>>(p, out, splits);
}
// Tiles of 128 rows, or (more of them, with less padding) of 64.
template <bool WIDEN, int OUT>
static void run_tall(const Fp8Product& p, const ProductOut& out, hipStream_t s) {
  run_tiles<WIDEN, OUT, 2, 4>(p, out, {1, p.kblocks()}, s);
}
template <bool WIDEN, int OUT>
static void run_short(const Fp8Product& p, const ProductOut& out, const Splits& splits, hipStream_t s) {
  run_tiles<WIDEN, OUT, short_bufs(WIDEN), 2>(p, out, splits, s);
}

// Short tiles are taken as long as they all fit the card at once.
static bool takes_tall(const Fp8Product& p, bool widen) {
  return tiles_of(p, tile_rows(2)) > (size_t)short_per_cu(widen) * kCus;
}

// A model of the time in units of 0.1 us, with what was measured for its parts: a
// workgroup's start and end 35; a step of one that has a CU to itself 7.7 (WIDEN) or 4.5,
// of two that share one 12 or 7, of three 17; with tall tiles twice that.
static double tiles_time(size_t workgroups, int steps, bool widen, bool tall) {
  static const double kStep[2][3] = {{4.5, 7.0, 0.0}, {7.7, 12.0, 17.0}};
  const int most = tall ? 2 : short_per_cu(widen);
  const size_t full = workgroups / (most * kCus), rest = workgroups % (most * kCus);
  const double unit = steps * (tall ? 2.0 : 1.0);
  double time = full * (35 + kStep[widen][most - 1] * unit);
  if (rest) time += 35 + kStep[widen][(rest - 1) / kCus] * unit;
  return time;
}

// How many ways to split the depth, and the modelled time: the second launch takes 30 and
// its traffic 5 GB/ms each way. Of 1 to 10 ways this takes the best or one within 3%.
constexpr int kMostSplits = 64;
struct TilePlan {
  Splits splits;
  double time;
};
static TilePlan plan_splits(const Fp8Product& p, bool widen, size_t work_bytes) {
  const int nkb = p.kblocks();
  const size_t tiles = tiles_of(p, tile_rows(2)), bytes = (size_t)p.m * p.n * 4;
  TilePlan best{{1, nkb}, tiles_time(tiles, nkb, widen, false)};
  for (int ways = 2; ways <= std::min(kMostSplits, nkb / 2); ways++) {
    const int each = (nkb + ways - 1) / ways, count = (nkb + each - 1) / each;
    if (count * bytes > work_bytes) break;
    const double time = tiles_time(tiles * count, each, widen, false) + 30 + 2.0 * count * bytes / 5e5;
    if (time < best.time) best = {{count, each}, time};
  }
  return best;
}

double fp8_gemm_time(const Fp8Product& p, bool widen, size_t work_bytes) {
  return takes_tall(p, widen) ? tiles_time(tiles_of(p, tile_rows(4)), p.kblocks(), widen, true)
                              : plan_splits(p, widen, work_bytes).time;
}

int fp8_gemm_parts(const Fp8Product& p) {
  return whole_chunks(p) ? (p.n + kCols - 1) / kCols : (p.n + 63) / 64;
}

template <bool WIDEN, int OUT, int BUFS, int XB>
static void tile_attributes() {
  (void)hipFuncSetAttribute((const void*)fp8_tile_kernel<WIDEN, OUT, BUFS, XB>,
                            hipFuncAttributeMaxDynamicSharedMemorySize, kMostLds);
}
void fp8_gemm_init_attributes() {
  tile_attributes<false, kOutBf16, 2, 4>();
  tile_attributes<true, kOutF32, 2, 4>();
  tile_attributes<true, kOutScores, 2, 4>();
  tile_attributes<false, kOutBf16, short_bufs(false), 2>();
  tile_attributes<false, kOutF32, short_bufs(false), 2>();
  tile_attributes<true, kOutF32, short_bufs(true), 2>();
  tile_attributes<true, kOutScores, short_bufs(true), 2>();
}

void launch_fp8_gemm(const Fp8Product& p, const ProductOut& out, int kind, void* work, size_t work_bytes,
                     hipStream_t s) {
  if (!whole_chunks(p)) {
    const dim3 grid((unsigned)((p.n + 127) / 128), (unsigned)((p.m + 127) / 128));
    if (kind == kOutF32)
      fp8_bytes_kernel<kOutF32><<<grid, 256, 0, s>>>(p, out);
    else if (kind == kOutBf16)
      fp8_bytes_kernel<kOutBf16><<<grid, 256, 0, s>>>(p, out);
    else
      fp8_bytes_kernel<kOutScores><<<grid, 256, 0, s>>>(p, out);
    return;
  }
  if (takes_tall(p, kind != kOutBf16)) {
    if (kind == kOutF32)
      run_tall<true, kOutF32>(p, out, s);
    else if (kind == kOutBf16)
      run_tall<false, kOutBf16>(p, out, s);
    else
      run_tall<true, kOutScores>(p, out, s);
    return;
  }
  if (kind == kOutScores) {
    run_short<true, kOutScores>(p, out, {1, p.kblocks()}, s);
    return;
  }
  const Splits splits = plan_splits(p, kind == kOutF32, work_bytes).splits;
  if (splits.count == 1) {
    kind == kOutF32 ? run_short<true, kOutF32>(p, out, splits, s) : run_short<false, kOutBf16>(p, out, splits, s);
    return;
  }
  const ProductOut parts{work, nullptr, nullptr, nullptr};
  const size_t count = (size_t)p.m * p.n;
  const unsigned grid = (unsigned)((count + 1023) / 1024);
  if (kind == kOutF32) {
    run_short<true, kOutF32>(p, parts, splits, s);
    add_splits_kernel<kOutF32><<<grid, 256, 0, s>>>((const float*)work, count, splits.count, out.y);
  } else {
    run_short<false, kOutF32>(p, parts, splits, s);
    add_splits_kernel<kOutBf16><<<grid, 256, 0, s>>>((const float*)work, count, splits.count, out.y);
  }
}

}  // namespace uocr
