// Interface of the 8-bit floating point operators (fp8.hip) and of token
// scoring (score.hip) towards the C-ABI layer.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace uocr {

constexpr int kFp8Block = 128;  // scale block: columns of a row, rows and columns of a matrix tile

// Element types, as uocr_dtype numbers them.
constexpr int kTypeBf16 = 0, kTypeF16 = 1, kTypeF32 = 2;

// fp8.hip: rows [rows, cols] (row stride ld elements; bf16 or f32) to e4m3
// with a power-of-two scale per (row, 128 columns), or per 128 x 128 tile.
void launch_fp8_quantize(const void* x, int type, size_t rows, int cols, size_t ld, uint8_t* q,
                         float* scales, int* err, hipStream_t s);
void launch_fp8_quantize_tiles(const void* x, int type, int rows, int cols, size_t ld, uint8_t* q,
                               float* scales, int* err, hipStream_t s);

// Once per process, before the first launch.
void fp8_init_attributes();

// One product: x [m, k] e4m3 rows with scales [m, blocks(k)], w [n, k] with
// scales [blocks(n), blocks(k)].
struct Fp8Product {
  const uint8_t* x;
  const float* xs;
  const uint8_t* w;
  const float* ws;
  int m, n, k;
  __host__ __device__ int kblocks() const { return (k + kFp8Block - 1) / kFp8Block; }
};
// Tiles are staged from rows of whole 16-byte chunks at aligned addresses. Where p's are
// not and tiles are what takes it, a copy of both operands that are, with zeros behind each
// row's end: its bytes (0 where it needs none), and the launch that makes it at `work`
// (256-byte aligned). ytype and work_bytes are those of the launch below; scores, kTypeF32
// and 0.
size_t fp8_pack_bytes(const Fp8Product& p, int ytype, size_t work_bytes);
Fp8Product launch_fp8_pack(const Fp8Product& p, void* work, hipStream_t s);
// `work`: room for partial sums where the depth is split; any size will do.
void launch_fp8_linear(const Fp8Product& p, void* y, int ytype, void* work, size_t work_bytes, hipStream_t s);

// Scores of the product's rows without the logits in memory: partial
// statistics per (column tile, row) and the given tokens' logits go to
// `work` (fp8_score_bytes of it), and a second launch joins them.
struct TokenScores {
  const int32_t* tokens;  // [rows], negative: a padding row; may be null with logprobs
  float* logprobs;        // [rows] or null
  float* entropy;         // [rows] or null
  int32_t* top_ids;       // [rows, top] or null
  float* top_logprobs;    // [rows, top] or null
  int top;
};
size_t fp8_score_bytes(const Fp8Product& p);
void launch_fp8_scores(const Fp8Product& p, const TokenScores& out, void* work, int* err,
                       hipStream_t s);

// score.hip: scores of logits [rows, vocab] (row stride ld elements).
constexpr int kMaxTop = 64;
size_t token_score_bytes(size_t rows, int vocab, int type, int top);
// Most rows of one launch (fewer than 2^32 threads).
size_t token_score_rows(int vocab, int type);
void launch_token_scores(const void* logits, int type, size_t rows, int vocab, size_t ld,
                         const TokenScores& out, void* work, int* err, hipStream_t s);

}  // namespace uocr
