// Attention of M rows over a paged cache (fp16, or 8-bit codes) under a sliding window with sinks: row m at position
// p = *pos + m attends the tokens t <= p with t > p - window or t < sinks (window 0: all t <= p). Shared by the kernel of many
// columns (attention_window.hip) and the one of few (attention_few.hip); a column is a (row, query head) pair of one kv head.
//
// Both hold a column's weights as p = 2^(c2 (s - ref) + kWinLift), c2 = log2(e) / sqrt(D), computed as c2 s + lift: one
// multiply-add. The reference is a maximum of scores seen so far, not the running one: it moves to a tile's maximum where a sum
// of p passes kWinMost, so that p fits fp16 and no maximum is taken otherwise; what fp16 cannot hold of a small p is 2^-32 of p
// at the reference. lift holds c2 ref to half a step of fp32, as a score of that size is held. From kWinFar on equal scores
// would weigh visibly apart in tiles of different references: there lift is infinite, every tile's first weights overflow, and
// the second ones are taken from s - ref, exact at the reference. Scores, sums and outputs are fp32.
// Where a weight meets V it is two fp16 numbers, hi and what hi leaves, both to nearest (2^-22), as in the attention of a
// prompt and of a decode step elsewhere in the library. Many columns over codes are the exception: there hi alone (2^-11,
// unbiased; its sum is taken unrounded), because the second product costs 30% (4096 rows of a prompt, e4m3: 193 us instead of
// 148) and V's codes are themselves off by up to 2^-8 of their block's largest value (int8) or 2^-4 of their own (e4m3). Over
// fp16, where V is exact and the output's rounding is the only one of that size, it costs 2 to 32% (8 x 4 heads of 128: 4096
// rows 195 us instead of 149, 512 rows 16 instead of 14, 4096 under a window of 1024 114 instead of 92); of few columns 2% at
// most (one token at 131072).
#pragma once
#include "kv8.hpp"

namespace dk {

// Reference maximum of a column that has seen no token: a finite stand-in for -infinity (no -inf - (-inf)).
constexpr float kWinNoMax = -1e30f;
constexpr float kWinLift = 7.0f;     // p's exponent at the reference maximum
constexpr float kWinMost = 32768.f;  // the reference moves where a lane's sum of p over its part of a tile passes this
constexpr float kWinFar = 4096.f;    // a reference further from 0 than this (log2 units) is taken off the score itself

constexpr int kWinMaxSplits = 64;

struct WinArgs {
  const f16* q;
  long long q_stride;
  const int32_t* pos;
  const int32_t* bt;
  const uint8_t* kc;
  const uint8_t* vc;
  const float* ks;
  const float* vs;
  int n_pages, n_bt, log2P, n_kv, lhpg, M, cap;  // cap: tokens at and past it do not exist
  int window, sinks, splits;
  float c2;  // log2(e) / sqrt(D)
  f16* out;  // [M, n_q D]
  float4* part_o;   // [splits][n_kv][column waves][D / 8][64 lanes]: the accumulators as the lanes hold them
  float2* part_ml;  // [splits][n_kv][column waves][32]: reference maximum, sum
};

// The tokens of one row: [lo, lim] and [0, sinks). (The position of a row that exists fits 32 bits without a sign.)
struct Sight {
  int lim, lo;
};
__device__ __forceinline__ Sight sight_of(int pos, int m, int window, int cap) {
  const uint32_t p = (uint32_t)pos + (uint32_t)m;
  const bool none = pos < 0 && (int)p < 0;
  const int lim = none ? -1 : (int)min(p, (uint32_t)cap - 1);
  const int lo = none || window == 0 || p < (uint32_t)window ? 0 : (int)min(p + 1 - (uint32_t)window, (uint32_t)cap);
  return {lim, lo};
}

// 16 bytes with a half that is no finite number.
__device__ __forceinline__ bool has_nonfinite(u32x4 v) {
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    bad = bad || (v[i] & 0x7C00u) == 0x7C00u || (v[i] & 0x7C000000u) == 0x7C000000u;
  return bad;
}

// The tokens that a block of `rows` rows can see at most.
inline long long win_tokens(long long rows, int max_ctx, int window, int sinks) {
  return window == 0 ? max_ctx : min((long long)max_ctx, (long long)window + rows + sinks + 32);
}

// The kernel of few columns: at most kFewCols of a kv head, tiles of kFewTile tokens.
constexpr int kFewCols = 16;
constexpr int kFewTile = 32;
// Whether the kernel of few columns takes a call. Pages of fewer than 16 tokens are left to the other one.
inline bool win_few(int M, int n_q, int n_kv, int log2P) { return (long long)M * (n_q / n_kv) <= kFewCols && log2P >= 4; }

// The RoPE of one token and its append, in front of its attention (8-bit caches, one row; a.q is then the fused qkv vector).
struct WinDecode {
  const float* cos_t;
  const float* sin_t;
  int max_pos;
};
// attention_few.hip: the splits that a call can use, and its launch (dec null: attention alone).
int attention_few_splits(int M, int n_kv, int head_dim, int max_ctx, int window, int sinks, int cache);
void launch_attention_few(const WindowAttn& w, const WinArgs& a, const WinDecode* dec, hipStream_t st);

}  // namespace dk
