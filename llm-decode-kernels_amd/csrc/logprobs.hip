// Log probabilities of given tokens, entropy and the k largest of each row of logits.
//   m = max x;  l = sum e^(x - m);  s = sum e^(x - m) (x - m);  log p_v = (x_v - m) - log l;  H = log l - s / l
// all in fp32 whatever the logits' type; a term with x = -inf is 0 in both sums.
#include "common.hpp"
#include "launch.hpp"

namespace dk {
namespace {

constexpr int kLpThreads = 256;

__device__ __forceinline__ float lp_load(const void* x, int dtype, size_t i) {
  if (dtype == 0) return (float)reinterpret_cast<const f16*>(x)[i];
  if (dtype == 1) return __builtin_bit_cast(float, (uint32_t)reinterpret_cast<const uint16_t*>(x)[i] << 16);
  return reinterpret_cast<const float*>(x)[i];
}

// One workgroup per row: the maximum, the sums, then one pass per alternative.
__global__ void __launch_bounds__(kLpThreads)
logprobs_row_kernel(const void* __restrict__ logits, int dtype, long long ld, const int64_t* __restrict__ tokens,
                    float* __restrict__ logprobs, float* __restrict__ entropy, int64_t* __restrict__ top_ids,
                    float* __restrict__ top_logprobs, int V, int k) {
  __shared__ float s_f[2][kLpThreads / kWave];
  __shared__ unsigned long long s_k[kLpThreads / kWave];
  const int row = blockIdx.x, tid = threadIdx.x;
  const size_t r0 = (size_t)row * ld;
  float m = -INFINITY;
  bool nan = false;
  for (int v = tid; v < V; v += kLpThreads) {
    const float x = lp_load(logits, dtype, r0 + v);
    nan = nan || x != x;
    m = fmaxf(m, x);
  }
  m = nan ? INFINITY : m;  // +inf marks a row without a distribution
  m = group_max<64>(m);
  if ((tid & 63) == 0) s_f[0][tid >> 6] = m;
  __syncthreads();
  for (int w = 0; w < kLpThreads / kWave; ++w) m = fmaxf(m, s_f[0][w]);
  __syncthreads();
  float l = 0.f, s = 0.f;
  for (int v = tid; v < V; v += kLpThreads) {
    const float d = lp_load(logits, dtype, r0 + v) - m, e = expf(d);
    l += e;
    s += d == -INFINITY ? 0.f : e * d;
  }
  l = group_sum<64>(l);
  s = group_sum<64>(s);
  if ((tid & 63) == 0) {
    s_f[0][tid >> 6] = l;
    s_f[1][tid >> 6] = s;
  }
  __syncthreads();
  l = s = 0.f;
  for (int w = 0; w < kLpThreads / kWave; ++w) {
    l += s_f[0][w];
    s += s_f[1][w];
  }
  const bool bad = !(m > -INFINITY && m < INFINITY);
  const float ll = logf(l);
  if (tid == 0) {
    if (logprobs) {
      const int64_t t = tokens[row];
      logprobs[row] = bad || t < 0 || t >= V ? NAN : (lp_load(logits, dtype, r0 + (size_t)t) - m) - ll;
    }
    if (entropy) entropy[row] = bad ? NAN : ll - s / l;
  }
  unsigned long long prev = ~0ull;
  for (int j = 0; j < k; ++j) {
    unsigned long long best = 0;
    for (int v = tid; v < V; v += kLpThreads) {
      const unsigned long long key = argmax_key(lp_load(logits, dtype, r0 + v), v);
      if (key < prev || j == 0) best = max(best, key);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) best = max(best, (unsigned long long)__shfl_xor(best, o, kWave));
    __syncthreads();
    if ((tid & 63) == 0) s_k[tid >> 6] = best;
    __syncthreads();
    for (int w = 0; w < kLpThreads / kWave; ++w) best = max(best, s_k[w]);
    prev = best;
    if (tid == 0) {
      const int64_t id = (uint32_t)~(uint32_t)best;
      top_ids[(size_t)row * k + j] = id;
      top_logprobs[(size_t)row * k + j] = bad ? NAN : (lp_load(logits, dtype, r0 + (size_t)id) - m) - ll;
    }
  }
}

}  // namespace

int token_logprobs_splits(int, int, int, int) { return 1; }
size_t token_logprobs_ws_bytes(int, int, int) { return 0; }

void launch_token_logprobs(const Logprobs& a, hipStream_t st) {
  hipLaunchKernelGGL(logprobs_row_kernel, dim3(a.M), dim3(kLpThreads), 0, st, a.logits, a.dtype, a.ld, a.tokens,
                     a.logprobs, a.entropy, a.top_ids, a.top_logprobs, a.V, a.k);
}

}  // namespace dk
