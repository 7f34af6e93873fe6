// Log probabilities of given tokens, entropy and the k largest of each row of logits, from one read of the logits.
//   m = max x;  l = sum e^(x - m);  s = sum e^(x - m) (x - m);  log p_v = (x_v - m) - log l;  H = log l - s / l
// all in fp32 whatever the logits' type; a term with x = -inf is 0 in both sums.
//
// A row is cut into `splits` slices, a workgroup each; a workgroup walks its slice in blocks of 256 threads x kPerThread
// values, the next block's 16-byte loads in flight while the values of the current one sit in registers. Every lane keeps
// its own running (m, l, s), rescaled once per block, and the lanes meet once at the end. The k largest need no second
// look at the data: the k-th largest of the 256 lane maxima is a lower bound T of the block's k-th largest value, so the
// values >= T, a few more than k, go to a list in LDS whose entries are ranked by counting. After the first block T is
// the k-th largest so far, and a block without a larger value ends with one comparison per lane. With more than one slice
// the (m, l, s) and k keys of each go to the workspace and a second launch joins them in slice order.
// Rows at odd addresses: 16-byte chunks lie on 16-byte boundaries, the first and last one are read value by value.
#include "common.hpp"
#include "launch.hpp"

namespace dk {
namespace {

constexpr int kLpThreads = 256, kLpWaves = kLpThreads / kWave;
constexpr int kLpListLanes = 64;  // lanes whose values the list has room for
constexpr float kLog2e = 1.44269504088896341f;

struct f16_t {
  static constexpr int EPC = 8;
  static constexpr uint32_t kNegInf = 0xFC00u;
  static __device__ __forceinline__ void unpack(u32x4 v, float* x) { unpack8(v, x); }
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
};
struct f32_t {
  static constexpr int EPC = 4;
  static constexpr uint32_t kNegInf = 0xFF800000u;
  static __device__ __forceinline__ void unpack(u32x4 v, float* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(v[i]);
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

// The 16-byte chunk that holds values [i0, i0 + EPC) of a row of V; `edge`: parts of it (or all) may lie outside the row and
// read as -inf.
template <class T>
__device__ __forceinline__ u32x4 lp_chunk(const void* row, int i0, int V, bool edge) {
  if (!edge) {
    if constexpr (T::EPC == 4)
      return *reinterpret_cast<const u32x4*>(reinterpret_cast<const float*>(row) + i0);
    else
      return *reinterpret_cast<const u32x4*>(reinterpret_cast<const uint16_t*>(row) + i0);
  }
  uint32_t w[T::EPC];
#pragma unroll
  for (int e = 0; e < T::EPC; ++e) {
    const int i = min(max(i0 + e, 0), V - 1);
    if constexpr (T::EPC == 4)
      w[e] = reinterpret_cast<const uint32_t*>(row)[i];
    else
      w[e] = reinterpret_cast<const uint16_t*>(row)[i];
    w[e] = i == i0 + e ? w[e] : T::kNegInf;
  }
  if constexpr (T::EPC == 4)
    return u32x4{w[0], w[1], w[2], w[3]};
  else
    return u32x4{w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16};
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
  a.s = w * fmaf(d, a.l, a.s);
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
  for (int i = threadIdx.x; i < max(n, k); i += kLpThreads) {
    if (i >= n) {
      out[i] = 0;
      continue;
    }
    const uint64_t key = list[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += list[j] > key;
    if (rank < k) out[rank] = key;
  }
}

// T: the logits' type; CPT: 16-byte chunks per thread and block; TOP: k >= 2 (otherwise each lane keeps its best key).
template <class T, int CPT, bool TOP>
__global__ void __launch_bounds__(kLpThreads, 4)
logprobs_kernel(const void* __restrict__ logits, long long ld, const int64_t* __restrict__ tokens,
                float* __restrict__ logprobs, float* __restrict__ entropy, int64_t* __restrict__ top_ids,
                float* __restrict__ top_logprobs, int V, int k, int per, int extra, Sums* __restrict__ ws_sums,
                uint64_t* __restrict__ ws_keys) {
  constexpr int EPC = T::EPC, E = CPT * EPC, kBlock = kLpThreads * E;
  static_assert(E <= 32, "one bit per value of a lane");
  __shared__ uint64_t s_list[TOP ? kLpListLanes * E + kLogprobsMaxK : 1];
  __shared__ float s_x[TOP ? E : 1][kLpThreads];  // a lane's values, where it has to look at them one by one
  __shared__ uint64_t s_top[2][kLogprobsMaxK];
  __shared__ uint64_t s_key[kLpWaves];
  __shared__ uint32_t s_max[TOP ? kLpThreads : 1];
  __shared__ Sums s_sums[kLpWaves];
  __shared__ int s_n;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int r = blockIdx.x, slice = blockIdx.y, splits = gridDim.y;
  const uint8_t* row = reinterpret_cast<const uint8_t*>(logits) + (size_t)r * (size_t)ld * (16 / EPC);
  const int off = (int)((reinterpret_cast<uintptr_t>(row) & 15u) / (16 / EPC));  // values of chunk 0 ahead of the row
  const int b0 = slice * per + min(slice, extra), b1 = b0 + per + (slice < extra);  // the first `extra` slices have one more

  // value e of a lane lies at i0 + place(e) of the row
  auto place = [](int e) { return (e / EPC) * (kLpThreads * EPC) + e % EPC; };
  u32x4 raw[CPT];
  auto fetch = [&](int b) {
    const int first = b * kBlock - off;
    if (first >= 0 && first + kBlock <= V) {  // uniform
#pragma unroll
      for (int j = 0; j < CPT; ++j) raw[j] = lp_chunk<T>(row, first + (j * kLpThreads + tid) * EPC, V, false);
    } else {
#pragma unroll
      for (int j = 0; j < CPT; ++j) raw[j] = lp_chunk<T>(row, first + (j * kLpThreads + tid) * EPC, V, true);
    }
  };
  Sums a = {-INFINITY, 0.f, 0.f};
  uint64_t best = 0;       // !TOP: this lane's largest key
  float best_v = -INFINITY;
  int cur = 0;             // TOP: s_top[cur] holds the k largest so far
  if (TOP && tid < k) s_top[0][tid] = 0;
  fetch(b0);
  for (int b = b0; b < b1; ++b) {
    float x[E];
#pragma unroll
    for (int j = 0; j < CPT; ++j) T::unpack(raw[j], x + j * EPC);
    if (b + 1 < b1) fetch(b + 1);
    const int i0 = b * kBlock + tid * EPC - off;
    // ---- the lane's sums about its running maximum
    float bm = x[0];
#pragma unroll
    for (int e = 1; e < E; ++e) bm = fmaxf(bm, x[e]);
    move_sums(a, fmaxf(a.m, bm));
    const float ms = finite_or_zero(a.m);
    float l[4] = {0.f, 0.f, 0.f, 0.f}, s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float d = x[e] - ms;  // NaN stays NaN, in l; e^-200 is 0 in fp32, so the bound changes no term of s
      const float p = __builtin_amdgcn_exp2f(d * kLog2e);
      l[e & 3] += p;
      s[e & 3] = fmaf(p, fmaxf(d, -200.f), s[e & 3]);
    }
    a.l += (l[0] + l[1]) + (l[2] + l[3]);
    a.s += (s[0] + s[1]) + (s[2] + s[3]);
    const bool nan = a.l != a.l;
    if constexpr (!TOP) {
      if (k > 0 && (b == b0 || bm > best_v || nan)) {  // equal values later in the row rank behind
        best_v = bm;
        int at = 0;
        float val = bm;
#pragma unroll
        for (int e = E - 1; e >= 0; --e) at = x[e] == bm ? place(e) : at;
        if (nan) {  // the lane's first NaN of this block, if it has one
#pragma unroll
          for (int e = E - 1; e >= 0; --e) {
            at = x[e] != x[e] ? place(e) : at;
            val = x[e] != x[e] ? x[e] : val;
          }
        }
        // what lies outside the row reads as -inf: ahead of it only in the chunk that holds value 0
        const int i = max(i0 + at, 0);
        const uint64_t key = argmax_key(val, i);
        best = i < V && key > best ? key : best;
      }
    } else {
      const uint64_t kth = s_top[cur][k - 1];  // 0: fewer than k so far
      const float kth_v = kth ? key_value(kth) : -INFINITY;
      const uint32_t order = (uint32_t)(argmax_key(bm, 0) >> 32);
      s_max[tid] = order;
      if (tid == 0) s_n = 0;
      // (the barrier also ends the reads of s_top[cur] above ahead of its next writer)
      if (!__syncthreads_or(nan || kth == 0 || bm > kth_v)) continue;
      // ---- T, in ordered bits: every one of the k largest values is >= T and lies in a lane whose maximum is. Past the
      // first block what follows the k-th value so far; otherwise, or where that leaves too many lanes, the k-th largest
      // lane maximum, found bit by bit until it is exact or k lanes pass
      uint32_t v[kLpWaves];
#pragma unroll
      for (int w = 0; w < kLpWaves; ++w) v[w] = s_max[w * kWave + lane];
      auto passing = [&](uint32_t probe) {
        int n = 0;
#pragma unroll
        for (int w = 0; w < kLpWaves; ++w) n += __popcll(__ballot(v[w] >= probe));
        return n;
      };
      uint32_t t = kth ? (uint32_t)(kth >> 32) + 1 : 0;
      int lanes = passing(t);
      if (lanes > kLpListLanes) {
        t = 0;
        lanes = kLpThreads;
        for (int bit = 31; bit >= 0 && lanes != k; --bit) {
          const int n = passing(t | 1u << bit);
          if (n >= k) {
            t |= 1u << bit;
            lanes = n;
          }
        }
      }
      const bool slow = __syncthreads_or(nan) || lanes > kLpListLanes;  // uniform
      // ---- the candidates, into the list
      if (!slow) {
        uint32_t hit = 0;
        if (order >= t) {
          const float tv = ordered_value(t);
#pragma unroll
          for (int e = 0; e < E; ++e) hit |= x[e] >= tv ? 1u << e : 0u;
        }
        if (hit != 0) {
#pragma unroll
          for (int e = 0; e < E; ++e) s_x[e][tid] = x[e];
          for (; hit != 0; hit &= hit - 1) {
            const int e = __builtin_ctz(hit), i = i0 + place(e);
            const uint64_t key = argmax_key(s_x[e][tid], i);
            if (key > kth && i >= 0 && i < V) s_list[atomicAdd(&s_n, 1)] = key;
          }
        }
      } else {
        // NaN, or more equal lane maxima than the list takes: the k largest one after the other
#pragma unroll
        for (int e = 0; e < E; ++e) s_x[e][tid] = x[e];
        uint64_t prev = ~0ull;
        for (int j = 0; j < k; ++j) {
          uint64_t mine = 0;
          for (int e = 0; e < E; ++e) {
            const int i = i0 + place(e);
            const uint64_t key = argmax_key(s_x[e][tid], i);
            mine = i >= 0 && i < V && key < prev && key > kth && key > mine ? key : mine;
          }
          mine = shfl_max_key(mine);
          if (lane == 0) s_key[wave] = mine;
          __syncthreads();
#pragma unroll
          for (int w = 0; w < kLpWaves; ++w) mine = s_key[w] > mine ? s_key[w] : mine;
          __syncthreads();
          prev = mine;
          if (mine == 0) break;  // uniform
          if (tid == 0) s_list[s_n++] = mine;
        }
      }
      __syncthreads();
      // ---- the k largest of the list and the k so far
      const int n0 = s_n;
      const uint64_t kept = lane < k ? s_top[cur][lane] : 0;
      const int had = __popcll(__ballot(kept != 0));
      if (wave == 0 && kept != 0) s_list[n0 + lane] = kept;
      __syncthreads();
      rank_list(s_list, n0 + had, s_top[cur ^ 1], k);
      __syncthreads();
      cur ^= 1;
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
      s_top[0][0] = key;
    }
    __syncthreads();
  }
  if (splits == 1) {
    lp_finish<T>(tot, row, r, tokens, logprobs, entropy, top_ids, top_logprobs, V, k, s_top[cur]);
    return;
  }
  const size_t part = (size_t)r * splits + slice;
  if (tid == 0) ws_sums[part] = tot;
  if (tid < k) ws_keys[part * k + tid] = s_top[cur][tid];
}

// Joins the slices of a row: sums in slice order, the k largest of the slices' k.
template <class T>
__global__ void __launch_bounds__(kLpThreads)
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
  // a slice's k-th key bounds the row's k-th from below: every wave takes the largest of them
  const uint64_t last = k > 0 && (tid & 63) < splits ? keys[(size_t)(tid & 63) * k + k - 1] : 0;
  Sums a = {-INFINITY, 0.f, 0.f};
  if (tid < splits) a = ws_sums[(size_t)r * splits + tid];
  const uint64_t floor_key = shfl_max_key(last);
  __syncthreads();
  for (int i = tid; i < splits * k; i += kLpThreads) {
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

// Blocks of a row: small ones (a chunk per thread) while a launch of them would leave CUs idle.
struct LpPlan {
  int cpt, blocks, splits;
};
LpPlan lp_plan(int M, int V, int dtype) {
  const int epc = dtype == 2 ? 4 : 8, full = dtype == 2 ? 8 : 4;
  const long long chunks = ((long long)V + epc - 1) / epc + 1;  // one more where the row starts inside a chunk
  auto blocks_of = [&](int cpt) { return (int)((chunks + (long long)kLpThreads * cpt - 1) / ((long long)kLpThreads * cpt)); };
  LpPlan p = {full, blocks_of(full), 0};
  if ((long long)M * p.blocks < 256) p = {1, blocks_of(1), 0};
  const long long want = (2048 + M - 1) / M;  // slices per row for eight workgroups per CU
  p.splits = (int)(want < 1 ? 1 : want);
  if (p.splits > p.blocks) p.splits = p.blocks;
  if (p.splits > kLogprobsMaxSplits) p.splits = kLogprobsMaxSplits;
  return p;
}

template <class T, int FULL>
void launch_lp(const Logprobs& a, hipStream_t st) {
  LpPlan p = lp_plan(a.M, a.V, a.dtype);
  const int S = a.splits;
  Sums* sums = reinterpret_cast<Sums*>(a.ws);
  uint64_t* keys = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(a.ws) + logprobs_sums_bytes(a.M, S));
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(a.M, S), dim3(kLpThreads), 0, st, a.logits, a.ld, a.tokens, a.logprobs, a.entropy,
                       a.top_ids, a.top_logprobs, a.V, a.k, p.blocks / S, p.blocks % S, sums, keys);
  };
  if (p.cpt == 1)
    a.k >= 2 ? go(logprobs_kernel<T, 1, true>) : go(logprobs_kernel<T, 1, false>);
  else
    a.k >= 2 ? go(logprobs_kernel<T, FULL, true>) : go(logprobs_kernel<T, FULL, false>);
  if (S > 1)
    hipLaunchKernelGGL(logprobs_join_kernel<T>, dim3(a.M), dim3(kLpThreads), 0, st, a.logits, a.ld, a.tokens, a.logprobs,
                       a.entropy, a.top_ids, a.top_logprobs, a.V, a.k, S, sums, keys);
}

}  // namespace

int token_logprobs_splits(int M, int V, int, int dtype) { return lp_plan(M, V, dtype).splits; }
size_t logprobs_sums_bytes(int M, int splits) {
  return ((size_t)M * splits * sizeof(Sums) + 15) & ~(size_t)15;
}
size_t token_logprobs_ws_bytes(int M, int k, int splits) {
  return logprobs_sums_bytes(M, splits) + (((size_t)M * splits * k * 8 + 15) & ~(size_t)15);
}

void launch_token_logprobs(const Logprobs& a, hipStream_t st) {
  if (a.dtype == 0)
    launch_lp<f16_t, 4>(a, st);
  else if (a.dtype == 1)
    launch_lp<bf16_t, 4>(a, st);
  else
    launch_lp<f32_t, 8>(a, st);
}

}  // namespace dk
