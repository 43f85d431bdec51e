// Scores of logits in memory: the log probability of each row's given token,
// the entropy of its distribution, and its most probable tokens.
//
// One pass over the logits (scores.hpp has the mathematics) leaves, per wave's
// chunk of a row, its statistics and, where alternatives are asked for, the largest
// logit of every group of 16 lanes' columns (64 or 128). The second launch, one
// workgroup per row, joins the statistics and finds the alternatives from the
// maxima without ordering them: with tau the n-th largest of its threads' maxima, at
// least n logits are not below tau, so the n largest logits are among the logits
// that are not below tau in the groups whose maximum is not. Those are few unless
// many are equal; each is ranked by counting the ones before it.
#include <algorithm>

#include "fp8.hpp"
#include "scores.hpp"

namespace uocr {

constexpr int kScoreThreads = 256;

template <typename T>
struct Logits;
template <>
struct Logits<float> {
  static constexpr int kVec = 4;
  static __device__ __forceinline__ float widen(float v) { return v; }
};
struct Bf16 {
  uint16_t bits;
};
template <>
struct Logits<Bf16> {
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float widen(Bf16 v) { return __uint_as_float((uint32_t)v.bits << 16); }
};
template <>
struct Logits<_Float16> {
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float widen(_Float16 v) { return (float)v; }
};

static int vec_of(int type) { return type == kTypeF32 ? 4 : 8; }
static int group_of(int type) { return 16 * vec_of(type); }

// Vectors per lane of a wave's chunk, all in flight at once: eight where there are
// many rows, fewer where a few rows have to fill the card (some 2048 waves).
constexpr int kMostVectors = 8;
static size_t chunks_of(int vocab, int type, int vectors) {
  const size_t chunk = (size_t)64 * vec_of(type) * vectors;
  return ((size_t)vocab + chunk - 1) / chunk;
}

struct ScorePlan {
  int vectors, chunks, groups;
  size_t maxima_at, bytes;
};
static ScorePlan plan_scores(size_t rows, int vocab, int type, int top) {
  ScorePlan p;
  p.vectors = kMostVectors;
  while (p.vectors > 1 && rows * chunks_of(vocab, type, p.vectors) < 2048) p.vectors /= 2;
  p.chunks = (int)chunks_of(vocab, type, p.vectors);
  p.groups = (int)(((size_t)vocab + group_of(type) - 1) / group_of(type));
  // Room for `rows` rows or fewer: fewer rows may take smaller chunks (at most
  // 2 * 2047 of them in all, or one vector per lane each).
  const size_t most = std::max(rows * chunks_of(vocab, type, kMostVectors),
                               std::min<size_t>(4096, rows * chunks_of(vocab, type, 1)));
  p.maxima_at = most * sizeof(ScorePart);
  p.bytes = p.maxima_at + (top ? rows * p.groups * sizeof(float) : 0);
  return p;
}

size_t token_score_bytes(size_t rows, int vocab, int type, int top) {
  return plan_scores(rows, vocab, type, top).bytes;
}

size_t token_score_rows(int vocab, int type) {
  const size_t chunks = chunks_of(vocab, type, kMostVectors);
  const size_t rows = (((size_t)1 << 26) - 1) / chunks;  // 64 threads each
  return std::min(std::max<size_t>(rows, 1), (size_t)1 << 22);
}

// One vector of a row as f32, -inf behind the row's end. Rows may start at any
// element.
template <typename T>
__device__ __forceinline__ void load_logits(const T* row, int c, int vocab, float (&v)[Logits<T>::kVec]) {
  constexpr int kVec = Logits<T>::kVec;
  if (c + kVec <= vocab) {
    T raw[kVec];
    __builtin_memcpy(raw, row + c, sizeof raw);
#pragma unroll
    for (int j = 0; j < kVec; j++) v[j] = Logits<T>::widen(raw[j]);
  } else {
#pragma unroll
    for (int j = 0; j < kVec; j++) v[j] = c + j < vocab ? Logits<T>::widen(row[c + j]) : -INFINITY;
  }
}

// Largest of the sixteen lanes of a row of lanes, in each of them.
__device__ __forceinline__ float row16_max(float v) {
  v = fmaxf(v, dpp_move<0xB1>(v));   // quad_perm [1,0,3,2]
  v = fmaxf(v, dpp_move<0x4E>(v));   // quad_perm [2,3,0,1]
  v = fmaxf(v, dpp_move<0x141>(v));  // row_half_mirror
  v = fmaxf(v, dpp_move<0x140>(v));  // row_mirror
  return v;
}

// A lane's statistics of its values, with the reference `most`, which none is above.
template <int V, int VEC>
__device__ __forceinline__ ScorePart lane_statistics(const float (&v)[V][VEC], float most) {
  // Banned words only have no reference; with 0 in its place every term vanishes (and
  // a NaN stays one).
  const float r = most == -INFINITY ? 0.0f : most;
  float s[2] = {0.0f, 0.0f}, t[2] = {0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < V; i++)
#pragma unroll
    for (int j = 0; j < VEC; j++) {
      // A banned word's distance is brought to where 2^d is 0 and 0 times d too.
      const float d = (v[i][j] - r) * kLog2e;
      const float e = __builtin_amdgcn_exp2f(d);
      s[j & 1] += e;
      t[j & 1] = fmaf(e, fmaxf(d, -1000.0f), t[j & 1]);
    }
  return {most, s[0] + s[1], t[0] + t[1], 0.0f};
}

template <typename T, int V>
__global__ __launch_bounds__(kScoreThreads) void score_chunks_kernel(
    const T* __restrict__ logits, size_t items, int vocab, size_t ld, const int32_t* __restrict__ tokens,
    int chunks, ScorePart* __restrict__ parts, float* __restrict__ maxima, int groups) {
  constexpr int kVec = Logits<T>::kVec;
  const int lane = threadIdx.x & 63;
  const size_t item = (size_t)blockIdx.x * (kScoreThreads / 64) +
                      (size_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  if (item >= items) return;
  const size_t row = item / (unsigned)chunks;
  const int chunk = (int)(item % (unsigned)chunks);
  if (tokens && tokens[row] < 0) return;  // a padding row is not read
  const T* x = logits + row * ld;
  const int c0 = (chunk * V * 64 + lane) * kVec;
  float v[V][kVec];
#pragma unroll
  for (int i = 0; i < V; i++) load_logits<T>(x, c0 + i * 64 * kVec, vocab, v[i]);
  float most = -INFINITY;
#pragma unroll
  for (int i = 0; i < V; i++) {
    float g = v[i][0];
#pragma unroll
    for (int j = 1; j < kVec; j++) g = fmaxf(g, v[i][j]);
    g = row16_max(g);
    most = fmaxf(most, g);
    const int c = c0 + i * 64 * kVec;
    if (maxima && (lane & 15) == 0 && c < vocab) maxima[row * groups + c / (16 * kVec)] = g;
  }
  most = fmaxf(most, __shfl_xor(most, 16));
  most = fmaxf(most, __shfl_xor(most, 32));
  ScorePart p = lane_statistics<V, kVec>(v, most);
  auto add = [](float a, float b) { return a + b; };
  p.s = lanes_reduce<1>(p.s, add);
  p.t = lanes_reduce<1>(p.t, add);
  if (lane == 0) parts[item] = p;
}

// The workgroup's largest key.
__device__ __forceinline__ unsigned long long block_max(unsigned long long key,
                                                        unsigned long long* held) {
  key = wave_max_u64(key);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) held[threadIdx.x >> 6] = key;
  __syncthreads();
  unsigned long long best = held[0];
#pragma unroll
  for (int w = 1; w < kScoreThreads / 64; w++) best = held[w] > best ? held[w] : best;
  return best;
}

// Groups and candidates that the short way holds; more (many equal logits) take
// the long one, which passes over the row once for each alternative.
constexpr int kMostGroups = 512, kMostCandidates = 1024;
// Group maxima that a thread keeps in registers (rows of up to 131072 or 262144
// logits); those of longer rows are read twice.
constexpr int kHeldMaxima = 8;
constexpr int kScorer = kScoreThreads - 64;  // first thread of the last wave, which writes a row's scores

// What a padding row gets.
__device__ __forceinline__ void write_padding(const TokenScores& out, size_t row, int tid) {
  if (tid == 0 && out.logprobs) out.logprobs[row] = 0.0f;
  if (tid == 0 && out.entropy) out.entropy[row] = 0.0f;
  for (int i = tid; i < out.top; i += kScoreThreads) {
    out.top_ids[row * out.top + i] = -1;
    out.top_logprobs[row * out.top + i] = -INFINITY;
  }
}

// A row's outputs from its threads' statistics p and its groups' maxima, of which g are
// this thread's first and group_max(at) gives any. `most` is the largest of some logits
// of this thread's own, which the first `filled` threads have; `given` the given token's
// logit in the last wave's first thread.
// A chain of dependent reads (the maxima; then the candidates' logits) and barriers,
// which is what it takes: everything that can be read early is, and nothing that can
// wait stands before a barrier.
template <typename T, class GroupMax>
__device__ __forceinline__ void finish_row(const T* x, size_t row, int vocab, int groups, ScorePart p,
                                           const float (&g)[kHeldMaxima], const GroupMax& group_max, float most,
                                           int filled, int token, float given, const TokenScores& out, int* err) {
  constexpr int kVec = Logits<T>::kVec, kGroup = 16 * kVec;
  __shared__ ScorePart held[kScoreThreads / 64];
  __shared__ unsigned long long keys[kMostCandidates];
  __shared__ int listed[kMostGroups];
  __shared__ __attribute__((aligned(16))) float mine[kScoreThreads];
  __shared__ uint32_t tau_at;
  __shared__ int counts[2];
  __shared__ float normalizer[2];
  __shared__ bool good;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int top = out.top;
  // tau is chosen from the maxima of four, two or single threads each: fewer to rank,
  // as long as they are as many as the alternatives.
  const int share = 4 * top <= filled ? 4 : 2 * top <= filled ? 2 : 1;
  if (share >= 2) most = fmaxf(most, dpp_move<0xB1>(most));
  if (share == 4) most = fmaxf(most, dpp_move<0x4E>(most));
  if (tid % share == 0) mine[tid / share] = most;
  p = lanes_join<1>(p);
  if (lane == 0) held[wave] = p;
  if (tid < 2) counts[tid] = 0;
  if (tid == 0) tau_at = ~0u;
  __syncthreads();
  // The n-th largest is the least of those that fewer than n are larger than.
  const int many = kScoreThreads / share;
  if (top && tid < many) {
    const float v = mine[tid];
    int larger = 0;
#pragma unroll 8
    for (int i = 0; i < many; i += 4) {
      const float4 o = *reinterpret_cast<const float4*>(mine + i);
      larger += (o.x > v) + (o.y > v) + (o.z > v) + (o.w > v);
    }
    if (larger < top) atomicMin(&tau_at, (uint32_t)(order_key(v, 0) >> 32));
  }
  // The last wave, which has no maximum to rank where threads share one, joins the
  // waves' statistics meanwhile.
  if (tid >= kScorer) {
    p = lanes_join<1>(lane < kScoreThreads / 64 ? held[lane] : empty_part());
    if (lane == 0) {
      write_scores(out, row, token, vocab, p, given, err);
      good = has_distribution(p);
      normalizer[0] = p.r;
      normalizer[1] = kLn2 * log2f(p.s);
    }
  }
  if (top == 0) return;
  __syncthreads();
  if (!good) {
    for (int i = tid; i < top; i += kScoreThreads) {
      out.top_ids[row * top + i] = -1;
      out.top_logprobs[row * top + i] = __uint_as_float(0x7fc00000u);
    }
    return;
  }
  const float tau = key_value((unsigned long long)tau_at << 32);
  // With tau -inf (fewer finite logits than alternatives, or nearly): all finite
  // logits, and the first columns' banned ones to fill up with.
  const bool finite = tau > -INFINITY;
  auto list = [&](int at, float v) {
    if (at >= groups || !(finite ? v >= tau : v > -INFINITY || at == 0)) return;
    const int to = atomicAdd(&counts[0], 1);
    if (to < kMostGroups) listed[to] = at;
  };
#pragma unroll
  for (int i = 0; i < kHeldMaxima; i++) list(tid + i * kScoreThreads, g[i]);
  for (int at = tid + kHeldMaxima * kScoreThreads; at < groups; at += kScoreThreads) list(at, group_max(at));
  __syncthreads();
  const int some = counts[0];
  if (some <= kMostGroups) {
    // Sixteen threads to a group, a vector each; two groups' loads in flight.
    auto consider = [&](int c, const float (&v)[kVec]) {
#pragma unroll
      for (int j = 0; j < kVec; j++)
        if (c + j < vocab && (finite ? v[j] >= tau : v[j] > -INFINITY || c + j < top)) {
          const int to = atomicAdd(&counts[1], 1);
          if (to < kMostCandidates) keys[to] = order_key(v[j], (uint32_t)(c + j));
        }
    };
    constexpr int kPass = kScoreThreads / 16;
    for (int i = tid / 16; i < some; i += 2 * kPass) {
      const int ca = listed[i] * kGroup + (tid & 15) * kVec;
      const int cb = i + kPass < some ? listed[i + kPass] * kGroup + (tid & 15) * kVec : vocab;
      float a[kVec], b[kVec];
      load_logits<T>(x, ca, vocab, a);
      load_logits<T>(x, cb, vocab, b);
      consider(ca, a);
      consider(cb, b);
    }
    __syncthreads();
  }
  auto write = [&](int at, unsigned long long key) {
    out.top_ids[row * top + at] = (int32_t)key_index(key);
    out.top_logprobs[row * top + at] = key_value(key) - normalizer[0] - normalizer[1];
  };
  const int found = counts[1];
  if (some <= kMostGroups && found <= kMostCandidates) {
    // The order of the list differs from run to run; the ranks do not.
    for (int i = tid; i < found; i += kScoreThreads) {
      const unsigned long long key = keys[i];
      int before = 0;
      for (int j = 0; j < found; j++) before += keys[j] > key;
      if (before < top) write(before, key);
    }
    return;
  }
  // The long way: one alternative after the other, each the largest below the one
  // before it.
  __syncthreads();
  unsigned long long last = ~0ull;
  for (int i = 0; i < top; i++) {
    unsigned long long best = 0;
    for (int c = tid * kVec; c < vocab; c += kScoreThreads * kVec) {
      float v[kVec];
      load_logits<T>(x, c, vocab, v);
#pragma unroll
      for (int j = 0; j < kVec; j++) {
        const unsigned long long key = order_key(v[j], (uint32_t)(c + j));
        if (c + j < vocab && key < last && key > best) best = key;
      }
    }
    last = block_max(best, keys);
    if (tid == 0) write(i, last);
  }
}

// One row of 129280 f32 6.1 us: 1.7 to the maxima, 0.7 to tau, 0.6 to the list, 1.2 to
// the candidates, 0.5 to the ranks.
template <typename T>
__global__ __launch_bounds__(kScoreThreads) void score_rows_kernel(
    const T* __restrict__ logits, int vocab, size_t ld, int chunks,
    const ScorePart* __restrict__ parts, const float* __restrict__ maxima, int groups,
    TokenScores out, int* err) {
  const size_t row = blockIdx.x;
  const int tid = threadIdx.x;
  const float* gmax = maxima + row * groups;
  float g[kHeldMaxima];
#pragma unroll
  for (int i = 0; i < kHeldMaxima; i++) {
    const int at = tid + i * kScoreThreads;
    g[i] = out.top && at < groups ? gmax[at] : -INFINITY;
  }
  ScorePart p = empty_part();
  for (int c = tid; c < chunks; c += kScoreThreads) p = join(p, parts[row * chunks + c]);
  const int token = out.tokens ? out.tokens[row] : 0;
  if (token < 0) {  // what was read of it is not used
    write_padding(out, row, tid);
    return;
  }
  const T* x = logits + row * ld;
  const float given = tid == kScorer && out.logprobs && token < vocab ? Logits<T>::widen(x[token]) : 0.0f;
  float most = g[0];
#pragma unroll
  for (int i = 1; i < kHeldMaxima; i++) most = fmaxf(most, g[i]);
  if (out.top)
    for (int at = tid + kHeldMaxima * kScoreThreads; at < groups; at += kScoreThreads) most = fmaxf(most, gmax[at]);
  finish_row<T>(x, row, vocab, groups, p, g, [&](int at) { return gmax[at]; }, most, min(groups, kScoreThreads), token,
                given, out, err);
}

// Short rows (up to kWholeVocab logits) are read by the workgroup that finishes them: no
// second launch, the groups' maxima stay in LDS, and tau comes from every thread's logits,
// which are more than the groups. 61 x 5000 f32 8.2 -> 7.2 us, 512 x 8192 bf16 10.4 ->
// 8.1; with 20 alternatives 61 x 1000 f32 65 -> 7.1 (fewer groups than alternatives). 61
// x 12000 would be 6% faster too, 61 x 16384 not, 61 x 129280 39 us against 14.7.
constexpr int kWholeVectors = 4, kWholeVocab = 8192;
template <typename T>
__global__ __launch_bounds__(kScoreThreads) void score_short_rows_kernel(const T* __restrict__ logits, int vocab,
                                                                         size_t ld, int groups, TokenScores out,
                                                                         int* err) {
  constexpr int kVec = Logits<T>::kVec, V = kWholeVectors;
  __shared__ float gmax[kWholeVocab / (16 * kVec)];
  const size_t row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63;
  const int token = out.tokens ? out.tokens[row] : 0;
  if (token < 0) {  // not read
    write_padding(out, row, tid);
    return;
  }
  const T* x = logits + row * ld;
  const float given = tid == kScorer && out.logprobs && token < vocab ? Logits<T>::widen(x[token]) : 0.0f;
  ScorePart p = empty_part();
  float largest = -INFINITY;
  // Whole waves: row16_max reads all sixteen lanes.
  for (int c0 = tid * kVec; c0 - lane * kVec < vocab; c0 += kScoreThreads * V * kVec) {
    float v[V][kVec];
#pragma unroll
    for (int i = 0; i < V; i++) load_logits<T>(x, c0 + i * kScoreThreads * kVec, vocab, v[i]);
    float most = -INFINITY;
#pragma unroll
    for (int i = 0; i < V; i++) {
      float m = v[i][0];
#pragma unroll
      for (int j = 1; j < kVec; j++) m = fmaxf(m, v[i][j]);
      most = fmaxf(most, m);
      if (out.top) {
        m = row16_max(m);
        const int c = c0 + i * kScoreThreads * kVec;
        if ((lane & 15) == 0 && c < vocab) gmax[c / (16 * kVec)] = m;
      }
    }
    p = join(p, lane_statistics<V, kVec>(v, most));
    largest = fmaxf(largest, most);
  }
  __syncthreads();
  float g[kHeldMaxima];
#pragma unroll
  for (int i = 0; i < kHeldMaxima; i++) {
    const int at = tid + i * kScoreThreads;
    g[i] = out.top && at < groups ? gmax[at] : -INFINITY;
  }
  finish_row<T>(x, row, vocab, groups, p, g, [&](int at) { return gmax[at]; }, largest,
                min((vocab + kVec - 1) / kVec, kScoreThreads), token, given, out, err);
}

template <typename T>
static void launch(const T* logits, size_t rows, int vocab, size_t ld, const ScorePlan& plan,
                   const TokenScores& out, void* work, int* err, hipStream_t s) {
  auto* parts = static_cast<ScorePart*>(work);
  float* maxima = out.top ? reinterpret_cast<float*>(static_cast<char*>(work) + plan.maxima_at) : nullptr;
  if (vocab <= kWholeVocab) {
    score_short_rows_kernel<T><<<(unsigned)rows, kScoreThreads, 0, s>>>(logits, vocab, ld, plan.groups, out, err);
    return;
  }
  const size_t items = rows * plan.chunks;
  const dim3 grid((unsigned)((items + kScoreThreads / 64 - 1) / (kScoreThreads / 64))), block(kScoreThreads);
#define UOCR_CHUNKS(V)                                                                             \
  score_chunks_kernel<T, V><<<grid, block, 0, s>>>(logits, items, vocab, ld, out.tokens, plan.chunks, \
                                                   parts, maxima, plan.groups)
  if (plan.vectors == 8)
    UOCR_CHUNKS(8);
  else if (plan.vectors == 4)
    UOCR_CHUNKS(4);
  else if (plan.vectors == 2)
    UOCR_CHUNKS(2);
  else
    UOCR_CHUNKS(1);
#undef UOCR_CHUNKS
  score_rows_kernel<T><<<(unsigned)rows, kScoreThreads, 0, s>>>(logits, vocab, ld, plan.chunks, parts,
                                                                maxima, plan.groups, out, err);
}

void launch_token_scores(const void* logits, int type, size_t rows, int vocab, size_t ld,
                         const TokenScores& out, void* work, int* err, hipStream_t s) {
  const ScorePlan plan = plan_scores(rows, vocab, type, out.top);
  if (type == kTypeF32)
    launch((const float*)logits, rows, vocab, ld, plan, out, work, err, s);
  else if (type == kTypeBf16)
    launch((const Bf16*)logits, rows, vocab, ld, plan, out, work, err, s);
  else
    launch((const _Float16*)logits, rows, vocab, ld, plan, out, work, err, s);
}

}  // namespace uocr
