// Log probabilities of given tokens, entropy and the k largest of each row of logits, from one read of the logits.
//   m = max x;  l = sum e^(x - m);  s = sum e^(x - m) (x - m);  log p_v = (x_v - m) - log l;  H = log l - s / l
// all in fp32 whatever the logits' type; a term with x = -inf is 0 in both sums.
//
// A row is cut into `splits` slices, a workgroup each; a workgroup walks its slice in blocks of 8192 values (2048 where
// there are few), the next block's 16-byte loads in flight while the current one sits in registers. Every lane keeps its
// own running (m, l, s), rescaled once per block, and the lanes meet once at the end. The k largest need no second look at
// the data: in the first block the lanes form 64 groups, and the k-th largest of the groups' maxima is a lower bound T of
// the k-th largest value, so the values >= T go to a list in LDS, hardly more than k of a block. The list is ranked by
// counting, and cut to its k largest, at the end, whenever it is half full and behind a block whose candidates it could not
// take; T is then what follows the k-th. With more than one slice the (m, l, s) and k keys of each go to the workspace and
// a second launch joins them in slice order.
// Measured (captured, us): 512 x 128256 fp32 46 with one alternative (5.8 TB/s), 57 with 5, 62 with 20, 64 with 32; fp16 35,
// 50, 55, 57; bf16 32, 50, 55, 57; 61 x 128256 fp16 and bf16 13 with one, 17 with 5, 19 with 20, fp32 14, 18, 20; 1 x 128256
// 9, 10, 13; 1 x 32000 8 (one launch), 10, 13 (two, of a memory round trip each). What the alternatives cost at 512 rows is
// the barrier per block that the list needs; one slice per row is the fastest there (two 65-79, four 68-83, sixteen 96-114
// with 2 to 20), eight of two blocks at 61 rows. Two passes (maximum and sums, then one pass per alternative) took 5175 at
// 512 x 128256 fp32 with 20.
// Rows at odd addresses: 16-byte chunks lie on 16-byte boundaries, the first and last one are read value by value.
#include "common.hpp"
#include "launch.hpp"

namespace dk {
namespace {

constexpr int kLpJoinThreads = 256;
constexpr int kLpGroups = 64;  // groups of lanes, one per lane of a wave
constexpr int kLpList = 512;  // candidates that the list takes; a block with more gives its k largest one after the other
static_assert(kLogprobsMaxK <= kLpGroups, "k group maxima bound the k-th largest value");
constexpr float kLog2e = 1.44269504088896341f;

struct f16_t {
  static constexpr int EPC = 8;
  static constexpr uint32_t kNegInf = 0xFC00u;
  static __device__ __forceinline__ void unpack(u32x4 v, float* x) { unpack8(v, x); }
  static __device__ __forceinline__ float max_of(u32x4 v) {  // (a NaN loses against any number)
    const f16x2 a = __builtin_elementwise_max(as_f16x2(v[0]), as_f16x2(v[1]));
    const f16x2 b = __builtin_elementwise_max(as_f16x2(v[2]), as_f16x2(v[3]));
    const f16x2 c = __builtin_elementwise_max(a, b);
    return fmaxf((float)c.x, (float)c.y);
  }
};
struct bf16_t {
  static constexpr int EPC = 8;
  static constexpr uint32_t kNegInf = 0xFF80u;
  static __device__ __forceinline__ void unpack(u32x4 v, float* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(v[i] << 16);
      x[2 * i + 1] = __uint_as_float(v[i] & 0xFFFF0000u);
    }
  }
  static __device__ __forceinline__ float max_of(u32x4 v) {
    float x[8];
    unpack(v, x);
    return fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
  }
};
struct f32_t {
  static constexpr int EPC = 4;
  static constexpr uint32_t kNegInf = 0xFF800000u;
  static __device__ __forceinline__ void unpack(u32x4 v, float* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(v[i]);
  }
  static __device__ __forceinline__ float max_of(u32x4 v) {
    return fmaxf(fmaxf(__uint_as_float(v[0]), __uint_as_float(v[1])), fmaxf(__uint_as_float(v[2]), __uint_as_float(v[3])));
  }
};

template <class T>
__device__ __forceinline__ float lp_value(const void* row, size_t i) {
  if constexpr (T::EPC == 4) {
    return reinterpret_cast<const float*>(row)[i];
  } else {
    float x[8];
    T::unpack(u32x4{reinterpret_cast<const uint16_t*>(row)[i], 0u, 0u, 0u}, x);
    return x[0];
  }
}

// The 16-byte chunk that holds values [i0, i0 + EPC) of a row of V (byte offsets fit 32 bits: V <= 2^24).
template <class T>
__device__ __forceinline__ u32x4 lp_chunk(const void* row, int i0) {
  return *reinterpret_cast<const u32x4*>(reinterpret_cast<const uint8_t*>(row) + (uint32_t)i0 * (16 / T::EPC));
}
// The same where parts of it (or all) may lie outside the row: those values read as -inf. One value after the other.
template <class T>
__device__ __forceinline__ u32x4 lp_edge_chunk(const void* row, int i0, int V) {
  if (i0 >= 0 && i0 + T::EPC <= V) return lp_chunk<T>(row, i0);
  constexpr int kBits = 128 / T::EPC;
  uint64_t lo = 0, hi = 0;
#pragma unroll 1
  for (int e = 0; e < T::EPC; ++e) {
    const int i = i0 + e;
    uint64_t w = T::kNegInf;
    if (i >= 0 && i < V) {
      if constexpr (T::EPC == 4)
        w = reinterpret_cast<const uint32_t*>(row)[i];
      else
        w = reinterpret_cast<const uint16_t*>(row)[i];
    }
    const int at = e * kBits;
    if (at < 64)
      lo |= w << at;
    else
      hi |= w << (at - 64);
  }
  return u32x4{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
}

// The value whose ordered bits (the high word of an argmax key) these are, the zero of either sign as +0.
__device__ __forceinline__ float ordered_value(uint32_t u) {
  return __uint_as_float(u & 0x80000000u ? u & 0x7FFFFFFFu : ~u);
}
__device__ __forceinline__ float key_value(uint64_t key) { return ordered_value((uint32_t)(key >> 32)); }
__device__ __forceinline__ uint64_t shfl_max_key(uint64_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint64_t w = __shfl_xor((unsigned long long)v, o, kWave);
    v = w > v ? w : v;
  }
  return v;
}

// Partial sums about a maximum, and their join: sums about m move to M with e^(m - M).
struct Sums {
  float m, l, s;
};
__device__ __forceinline__ float finite_or_zero(float m) { return m == -INFINITY ? 0.f : m; }
__device__ __forceinline__ void move_sums(Sums& a, float M) {  // M >= a.m
  const float d = a.m == -INFINITY ? 0.f : a.m - finite_or_zero(M);
  const float w = __builtin_amdgcn_exp2f(d * kLog2e);
  // w is 0 below -200; there d l may pass the range (sums about a mask's lowest value), and 0 times infinity is NaN
  a.s = w * fmaf(fmaxf(d, -200.f), a.l, a.s);
  a.l *= w;
  a.m = M;
}

// Row results from the joined sums and the k keys (descending) in LDS; called by a whole workgroup.
template <class T>
__device__ __forceinline__ void lp_finish(const Sums& a, const void* row, int r, const int64_t* tokens, float* logprobs,
                                          float* entropy, int64_t* top_ids, float* top_logprobs, int V, int k,
                                          const uint64_t* keys) {
  const int tid = threadIdx.x;
  // NaN or +inf among the logits made l NaN, nothing but -inf left it 0
  const bool bad = !(a.l > 0.f);
  const float ll = logf(a.l);
  if (tid < k) {
    top_ids[(size_t)r * k + tid] = (int64_t)(uint32_t)~(uint32_t)keys[tid];
    top_logprobs[(size_t)r * k + tid] = bad ? NAN : (key_value(keys[tid]) - a.m) - ll;
  }
  if (tid == kWave) {
    if (logprobs) {
      const int64_t t = tokens[r];
      const bool in = t >= 0 && t < V;
      const float x = lp_value<T>(row, in ? (size_t)t : 0);
      logprobs[r] = bad || !in ? NAN : (x - a.m) - ll;
    }
    if (entropy) entropy[r] = bad ? NAN : ll - a.s / a.l;
  }
}

// Entries [0, n) of list ranked by counting; the k largest to out in descending order, 0 behind the last.
__device__ __forceinline__ void rank_list(const uint64_t* list, int n, uint64_t* out, int k) {
  for (int i = threadIdx.x; i < max(n, k); i += blockDim.x) {
    if (i >= n) {
      out[i] = 0;
      continue;
    }
    const uint64_t key = list[i];
    int rank = 0;
#pragma unroll 4
    for (int j = 0; j < n; ++j) rank += list[j] > key;
    if (rank < k) out[rank] = key;
  }
}

// T: the logits' type; NT: threads; CPT: 16-byte chunks per thread and block; TOP: k >= 2 (otherwise each lane keeps its
// best key).
template <class T, int NT, int CPT, bool TOP>
__global__ void __launch_bounds__(NT, 4)
logprobs_kernel(const void* __restrict__ logits, long long ld, const int64_t* __restrict__ tokens,
                float* __restrict__ logprobs, float* __restrict__ entropy, int64_t* __restrict__ top_ids,
                float* __restrict__ top_logprobs, int V, int k, int per, int extra, Sums* __restrict__ ws_sums,
                uint64_t* __restrict__ ws_keys) {
  constexpr int EPC = T::EPC, E = CPT * EPC, kBlock = NT * E, kLpWaves = NT / kWave;
  constexpr int kGroup = NT / kLpGroups;  // lanes per group
  static_assert(E <= 32 && kGroup >= 1 && kGroup <= 16, "one bit per value of a lane; groups inside a wave");
  __shared__ uint64_t s_list[TOP ? kLpList + kLogprobsMaxK : 1];
  __shared__ float s_x[TOP ? E : 1][NT];  // a lane's values, where it has to look at them one by one
  __shared__ uint64_t s_top[kLogprobsMaxK];
  __shared__ uint64_t s_key[kLpWaves];
  __shared__ uint32_t s_max[TOP ? kLpGroups : 1];
  __shared__ Sums s_sums[kLpWaves];
  __shared__ int s_n, s_hits[2][kLpWaves];  // (s_hits by the block's parity: a wave is at most one barrier ahead)
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int r = blockIdx.x, slice = blockIdx.y, splits = gridDim.y;
  const uint8_t* row = reinterpret_cast<const uint8_t*>(logits) + (size_t)r * (size_t)ld * (16 / EPC);
  const int off = (int)((reinterpret_cast<uintptr_t>(row) & 15u) / (16 / EPC));  // values of chunk 0 ahead of the row
  const int b0 = slice * per + min(slice, extra), b1 = b0 + per + (slice < extra);  // the first `extra` slices have one more

  // value e of a lane lies at i0 + place(e) of the row
  auto place = [](int e) { return (e / EPC) * (NT * EPC) + e % EPC; };
  u32x4 raw[CPT];
  auto fetch = [&](int b) {
    const int first = b * kBlock - off;
    if (first >= 0 && first + kBlock <= V) {  // uniform
#pragma unroll
      for (int j = 0; j < CPT; ++j) raw[j] = lp_chunk<T>(row, first + (j * NT + tid) * EPC);
    } else {
#pragma unroll
      for (int j = 0; j < CPT; ++j) raw[j] = lp_edge_chunk<T>(row, first + (j * NT + tid) * EPC, V);
    }
  };
  Sums a = {-INFINITY, 0.f, 0.f};
  uint64_t best = 0;       // !TOP: this lane's largest key
  float best_v = -INFINITY;
  int n = 0;               // TOP: entries of the list (uniform)
  uint32_t t = 0;          // TOP: T in ordered bits (uniform)
  if (TOP && tid == 0) s_n = 0;
  fetch(b0);
  for (int b = b0; b < b1; ++b) {
    u32x4 now[CPT];
#pragma unroll
    for (int j = 0; j < CPT; ++j) now[j] = raw[j];
    if (b + 1 < b1) fetch(b + 1);
    const int i0 = b * kBlock + tid * EPC - off;
    // ---- the lane's sums about its running maximum
    float bm = T::max_of(now[0]);
#pragma unroll
    for (int j = 1; j < CPT; ++j) bm = fmaxf(bm, T::max_of(now[j]));
    move_sums(a, fmaxf(a.m, bm));
    const float ms = finite_or_zero(a.m);
    float l[4] = {0.f, 0.f, 0.f, 0.f}, s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < CPT; ++j) {
      float x[EPC];
      T::unpack(now[j], x);
#pragma unroll
      for (int e = 0; e < EPC; ++e) {
        const float d = x[e] - ms;  // NaN stays NaN, in l; e^-200 is 0 in fp32, so the bound changes no term of s
        const float p = __builtin_amdgcn_exp2f(d * kLog2e);
        l[e & 3] += p;
        s[e & 3] = fmaf(p, fmaxf(d, -200.f), s[e & 3]);
      }
    }
    const float bl = (l[0] + l[1]) + (l[2] + l[3]);
    a.l += bl;
    a.s += (s[0] + s[1]) + (s[2] + s[3]);
    const bool nan = bl != bl;  // a NaN or +inf in this block
    if constexpr (!TOP) {
      if (k > 0 && (b == b0 || bm > best_v || nan)) {  // equal values later in the row rank behind
        best_v = bm;
        int at = 0;
        float val = bm;
#pragma unroll
        for (int j = CPT - 1; j >= 0; --j) {
          float x[EPC];
          T::unpack(now[j], x);
#pragma unroll
          for (int e = EPC - 1; e >= 0; --e) at = x[e] == bm ? place(j * EPC + e) : at;
        }
        if (nan) {  // the lane's first NaN of this block, if it has one
#pragma unroll
          for (int j = CPT - 1; j >= 0; --j) {
            float x[EPC];
            T::unpack(now[j], x);
#pragma unroll
            for (int e = EPC - 1; e >= 0; --e) {
              at = x[e] != x[e] ? place(j * EPC + e) : at;
              val = x[e] != x[e] ? x[e] : val;
            }
          }
        }
        // what lies outside the row reads as -inf: ahead of it only in the chunk that holds value 0
        const int i = max(i0 + at, 0);
        const uint64_t key = argmax_key(val, i);
        best = i < V && key > best ? key : best;
      }
    } else {
      if (b == b0) {
        // T: the k-th largest group maximum, bit by bit until it is exact or k groups pass
        const float gm = group_max<kGroup>(bm);
        if (lane % kGroup == 0) s_max[tid / kGroup] = (uint32_t)(argmax_key(gm, 0) >> 32);
        __syncthreads();
        const uint32_t v = s_max[lane];
        int groups = kLpGroups;
        for (int bit = 31; bit >= 0 && groups != k; --bit) {
          const int c = __popcll(__ballot(v >= (t | 1u << bit)));
          if (c >= k) {
            t |= 1u << bit;
            groups = c;
          }
        }
      }
      // ---- the values >= T, into the list
      const float tv = ordered_value(t);
      uint32_t hit = 0;
      if (bm >= tv) {
#pragma unroll
        for (int j = 0; j < CPT; ++j) {
          float x[EPC];
          T::unpack(now[j], x);
#pragma unroll
          for (int e = 0; e < EPC; ++e) {
            hit |= x[e] >= tv ? 1u << (j * EPC + e) : 0u;
            s_x[j * EPC + e][tid] = x[e];
          }
        }
        if (i0 < 0 || i0 + place(E - 1) >= V) {  // what lies outside the row
          for (int e = 0; e < E; ++e)
            if (i0 + place(e) < 0 || i0 + place(e) >= V) hit &= ~(1u << e);
        }
        int at = hit ? atomicAdd(&s_n, __popc(hit)) : 0;
        for (uint32_t h = hit; h != 0; h &= h - 1, ++at) {
          const int e = __builtin_ctz(h);
          if (at < kLpList) s_list[at] = argmax_key(s_x[e][tid], i0 + place(e));
        }
      }
      int hits = __any(nan) ? kLpList + 1 : 0;
      if (__any(hit != 0)) hits += (int)group_sum<64>((float)__popc(hit));
      if (lane == 0) s_hits[b & 1][wave] = hits;
      __syncthreads();
      hits = 0;
#pragma unroll
      for (int w = 0; w < kLpWaves; ++w) hits += s_hits[b & 1][w];
      const bool over = n + hits > kLpList;  // uniform
      if (!over) {
        n += hits;
      } else {
        // NaN, or more candidates than the list takes (equal values by the hundred): the block's k largest one after the
        // other, in the place of what it has put into the list
#pragma unroll
        for (int j = 0; j < CPT; ++j) {
          float x[EPC];
          T::unpack(now[j], x);
#pragma unroll
          for (int e = 0; e < EPC; ++e) s_x[j * EPC + e][tid] = x[e];
        }
        uint64_t prev = ~0ull;
        int found = 0;
        for (; found < k; ++found) {
          uint64_t mine = 0;
          for (int e = 0; e < E; ++e) {
            const int i = i0 + place(e);
            const uint64_t key = argmax_key(s_x[e][tid], i);
            mine = i >= 0 && i < V && key < prev && key > mine ? key : mine;
          }
          mine = shfl_max_key(mine);
          if (lane == 0) s_key[wave] = mine;
          __syncthreads();
#pragma unroll
          for (int w = 0; w < kLpWaves; ++w) mine = s_key[w] > mine ? s_key[w] : mine;
          __syncthreads();
          prev = mine;
          if (mine == 0) break;  // uniform
          if (tid == 0) s_list[n + found] = mine;
        }
        n += found;
        __syncthreads();
      }
      // uniform: the list's k largest, and T from the k-th. Also behind an overflow, which leaves s_n past the list's end:
      // places in the next block start at the s_n that is set here.
      if (n > kLpList / 2 || b + 1 == b1 || over) {
        rank_list(s_list, n, s_top, k);
        __syncthreads();
        const uint64_t kth = s_top[k - 1];
        if (tid < k) s_list[tid] = s_top[tid];
        n = min(n, k);
        // equal values further on rank behind (NaN: nothing follows)
        t = kth == 0 ? 0 : max((uint32_t)(kth >> 32), (uint32_t)(kth >> 32) + 1);
        if (tid == 0) s_n = n;
        __syncthreads();
      }
    }
  }
  // ---- the lanes meet
  const float wm = group_max<64>(a.m);
  move_sums(a, wm);
  a.l = group_sum<64>(a.l);
  a.s = group_sum<64>(a.s);
  if (lane == 0) s_sums[wave] = a;
  if constexpr (!TOP) {
    best = shfl_max_key(best);
    if (lane == 0) s_key[wave] = best;
  }
  __syncthreads();
  float M = -INFINITY;
#pragma unroll
  for (int w = 0; w < kLpWaves; ++w) M = fmaxf(M, s_sums[w].m);
  Sums tot = {M, 0.f, 0.f};
#pragma unroll
  for (int w = 0; w < kLpWaves; ++w) {
    Sums p = s_sums[w];
    move_sums(p, M);
    tot.l += p.l;
    tot.s += p.s;
  }
  if constexpr (!TOP) {
    if (tid == 0 && k > 0) {
      uint64_t key = 0;
#pragma unroll
      for (int w = 0; w < kLpWaves; ++w) key = s_key[w] > key ? s_key[w] : key;
      s_top[0] = key;
    }
    __syncthreads();
  }
  if (splits == 1) {
    lp_finish<T>(tot, row, r, tokens, logprobs, entropy, top_ids, top_logprobs, V, k, s_top);
    return;
  }
  const size_t part = (size_t)r * splits + slice;
  if (tid == 0) ws_sums[part] = tot;
  if (tid < k) ws_keys[part * k + tid] = s_top[tid];
}

// Joins the slices of a row: sums in slice order, the k largest of the slices' k.
template <class T>
__global__ void __launch_bounds__(kLpJoinThreads)
logprobs_join_kernel(const void* __restrict__ logits, long long ld, const int64_t* __restrict__ tokens,
                     float* __restrict__ logprobs, float* __restrict__ entropy, int64_t* __restrict__ top_ids,
                     float* __restrict__ top_logprobs, int V, int k, int splits, const Sums* __restrict__ ws_sums,
                     const uint64_t* __restrict__ ws_keys) {
  __shared__ uint64_t s_list[kLogprobsMaxSplits * kLogprobsMaxK], s_top[kLogprobsMaxK];
  __shared__ Sums s_sums;
  __shared__ int s_n;
  const int r = blockIdx.x, tid = threadIdx.x;
  const uint64_t* keys = ws_keys + (size_t)r * splits * k;
  if (tid == 0) s_n = 0;
  // A lower bound of the row's k-th key: the q-th largest of the slices' j-th keys, q j >= k (0 stands for a key that a short
  // slice does not have, and bounds nothing).
  uint64_t floor_key = 0;
  if (k > 0) {
    const int j = (k + splits - 1) / splits, q = (k + j - 1) / j;
    const int slice = tid & 63;
    const uint64_t mine = slice < splits ? keys[(size_t)slice * k + j - 1] : 0;
    if (tid < kWave) s_list[tid] = mine;
    __syncthreads();
    int rank = 0;
#pragma unroll 8
    for (int i = 0; i < kWave; ++i) rank += s_list[i] > mine;
    floor_key = shfl_max_key(rank >= q - 1 ? mine : 0);
    __syncthreads();
  }
  Sums a = {-INFINITY, 0.f, 0.f};
  if (tid < splits) a = ws_sums[(size_t)r * splits + tid];
  __syncthreads();
  for (int i = tid; i < splits * k; i += kLpJoinThreads) {
    const uint64_t key = keys[i];
    if (key != 0 && key >= floor_key) s_list[atomicAdd(&s_n, 1)] = key;
  }
  if (tid < kWave) {  // splits <= 64: one slice per lane
    move_sums(a, group_max<64>(a.m));
    a.l = group_sum<64>(a.l);
    a.s = group_sum<64>(a.s);
    if (tid == 0) s_sums = a;
  }
  __syncthreads();
  rank_list(s_list, s_n, s_top, k);
  __syncthreads();
  lp_finish<T>(s_sums, reinterpret_cast<const uint8_t*>(logits) + (size_t)r * (size_t)ld * (16 / T::EPC), r, tokens,
               logprobs, entropy, top_ids, top_logprobs, V, k, s_top);
}

// Blocks of a row: one workgroup and launch takes up to four full ones (512 threads, 8192 values), two where k asks for a
// list: 32000 fp16 values with k 1 in 7.9 us for one row and 8.2 for 61, split 8.2 and 10.0 (called eagerly 7.4 and 7.9 : 9.9
// and 10.2); 16000 with k 5 8.7 and 9.5 : 10.3 and 11.5; past that 64000 with k 1 11.6 : 8.5, 32000 with k 5 11.5 : 10.1.
// Longer rows are split, in small blocks (256 threads, a chunk each) while a launch of full ones would leave CUs idle; a row
// that has to run unsplit takes full ones (128256 fp16 values, k 5: 33 us, small ones 74).
constexpr int kLpFullThreads = 512, kLpSmallThreads = 256;
constexpr int lp_full_chunks(int dtype) { return dtype == 2 ? 4 : 2; }
struct LpPlan {
  bool small;
  int blocks, splits;
};
int lp_blocks(int V, int dtype, int size) {  // of `size` 16-byte chunks
  const int epc = dtype == 2 ? 4 : 8;
  const long long chunks = ((long long)V + epc - 1) / epc + 1;  // one more where the row starts inside a chunk
  return (int)((chunks + size - 1) / size);
}
LpPlan lp_unsplit(int V, int dtype) { return {false, lp_blocks(V, dtype, kLpFullThreads * lp_full_chunks(dtype)), 1}; }
LpPlan lp_plan(int M, int V, int k, int dtype) {
  LpPlan p = lp_unsplit(V, dtype);
  if (p.blocks <= (k >= 2 ? 2 : 4)) return p;
  if ((long long)M * p.blocks < 256) p = {true, lp_blocks(V, dtype, kLpSmallThreads), 0};
  // slices for as many workgroups as are resident at once (two of 512 threads or four of 256 per CU), of equal length
  int want = (p.small ? 1024 : 512) / M;
  want = want < 1 ? 1 : want > kLogprobsMaxSplits ? kLogprobsMaxSplits : want;
  const int per = (p.blocks + want - 1) / want;
  p.splits = (p.blocks + per - 1) / per;
  return p;
}

template <class T, int DTYPE>
void launch_lp(const Logprobs& a, hipStream_t st) {
  LpPlan p = lp_plan(a.M, a.V, a.k, a.dtype);
  const int S = a.splits;
  if (S == 1) p = lp_unsplit(a.V, a.dtype);
  Sums* sums = reinterpret_cast<Sums*>(a.ws);
  uint64_t* keys = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(a.ws) + logprobs_sums_bytes(a.M, S));
  auto go = [&](auto kernel, int threads) {
    hipLaunchKernelGGL(kernel, dim3(a.M, S), dim3(threads), 0, st, a.logits, a.ld, a.tokens, a.logprobs, a.entropy,
                       a.top_ids, a.top_logprobs, a.V, a.k, p.blocks / S, p.blocks % S, sums, keys);
  };
  constexpr int kFull = lp_full_chunks(DTYPE);
  if (p.small)
    a.k >= 2 ? go(logprobs_kernel<T, kLpSmallThreads, 1, true>, kLpSmallThreads)
             : go(logprobs_kernel<T, kLpSmallThreads, 1, false>, kLpSmallThreads);
  else
    a.k >= 2 ? go(logprobs_kernel<T, kLpFullThreads, kFull, true>, kLpFullThreads)
             : go(logprobs_kernel<T, kLpFullThreads, kFull, false>, kLpFullThreads);
  if (S > 1)
    hipLaunchKernelGGL(logprobs_join_kernel<T>, dim3(a.M), dim3(kLpJoinThreads), 0, st, a.logits, a.ld, a.tokens, a.logprobs,
                       a.entropy, a.top_ids, a.top_logprobs, a.V, a.k, S, sums, keys);
}

}  // namespace

int token_logprobs_splits(int M, int V, int k, int dtype) { return lp_plan(M, V, k, dtype).splits; }
size_t logprobs_sums_bytes(int M, int splits) {
  return ((size_t)M * splits * sizeof(Sums) + 15) & ~(size_t)15;
}
size_t token_logprobs_ws_bytes(int M, int k, int splits) {
  return logprobs_sums_bytes(M, splits) + (((size_t)M * splits * k * 8 + 15) & ~(size_t)15);
}

void launch_token_logprobs(const Logprobs& a, hipStream_t st) {
  if (a.dtype == 0)
    launch_lp<f16_t, 0>(a, st);
  else if (a.dtype == 1)
    launch_lp<bf16_t, 1>(a, st);
  else
    launch_lp<f32_t, 2>(a, st);
}

}  // namespace dk
