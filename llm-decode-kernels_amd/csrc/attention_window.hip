// Attention of M rows over a paged cache (fp16, or 8-bit codes) under a sliding window with sinks: row m at position
// p = *pos + m attends the tokens t <= p with t > p - window or t < sinks (window 0: all t <= p).
//
// A wave owns one (row, query head). By 64 tokens: a lane has a token's score (dot over its K row), the wave the running
// maximum and sum; then a lane has D / 64 dims of the output and adds p V over the 64 tokens. All in fp32.
#include "kv8.hpp"

namespace dk {
namespace {

constexpr float kWinNoMax = -1e30f;  // a finite stand-in for -infinity (no -inf - (-inf))

struct WinArgs {
  const f16* q;
  long long q_stride;
  const int32_t* pos;
  const int32_t* bt;
  const uint8_t* kc;
  const uint8_t* vc;
  const float* ks;
  const float* vs;
  int n_pages, log2P, n_kv, lhpg, M, cap, window, sinks;
  float c2;
  f16* out;
};

template <int D, int CACHE>
__global__ void __launch_bounds__(64) attn_window_kernel(const WinArgs a) {
  constexpr int DPL = D / 64;
  __shared__ float s_q[D], s_p[64];
  __shared__ long long s_at[64];
  const int lane = threadIdx.x;
  const int n_q = a.n_kv << a.lhpg;
  const int hd = blockIdx.x % n_q, m = blockIdx.x / n_q, kvh = hd >> a.lhpg;
  const long long p = (long long)*a.pos + m;
  for (int d = lane; d < D; d += 64) s_q[d] = (float)a.q[(size_t)m * a.q_stride + (size_t)hd * D + d];
  __syncthreads();
  const long long end = min(p + 1, (long long)a.cap);  // tokens [0, end)
  const long long lo = a.window ? max(0LL, p - a.window + 1) : 0;
  float mx = kWinNoMax, l = 0.f, acc[DPL] = {};
  auto value = [&](const uint8_t* c, const float* sc, long long at, int d) -> float {  // row at, dim d
    if constexpr (CACHE == kCacheF16) {
      return (float)reinterpret_cast<const f16*>(c)[at * D + d];
    } else {
      const uint8_t b = c[at * D + d];
      const u32x4 x = kv8_decode8<CACHE>(u32x2{b, 0u}, sc[at >> 4]);
      return (float)as_f16x2(x[0])[0];
    }
  };
  auto tokens = [&](long long t0, long long t1) {
    for (long long b = t0; b < t1; b += 64) {
      const long long t = b + lane;
      const int page = t < t1 ? a.bt[t >> a.log2P] : -1;
      const bool see = (unsigned)page < (unsigned)a.n_pages;
      const long long at = see ? ((((long long)page * a.n_kv + kvh) << a.log2P) + (t & ((1 << a.log2P) - 1))) : -1;
      float s = -INFINITY;
      if (see) {
        s = 0.f;
        for (int d = 0; d < D; ++d) s = fmaf(s_q[d], value(a.kc, a.ks, at, d), s);
      }
      float top = s;
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, kWave));
      const float to = fmaxf(mx, top), alpha = __builtin_amdgcn_exp2f((mx - to) * a.c2);
      const float w = see ? __builtin_amdgcn_exp2f((s - to) * a.c2) : 0.f;
      mx = to;
      l = l * alpha + w;
      s_p[lane] = w;
      s_at[lane] = at;
      __syncthreads();
      for (int i = 0; i < DPL; ++i) acc[i] *= alpha;
      for (int j = 0; j < 64; ++j) {
        if (s_at[j] < 0) continue;
        for (int i = 0; i < DPL; ++i) acc[i] = fmaf(s_p[j], value(a.vc, a.vs, s_at[j], DPL * lane + i), acc[i]);
      }
      __syncthreads();
    }
  };
  if (a.window) tokens(0, min(min((long long)a.sinks, lo), end));
  tokens(lo, end);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o, kWave);
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  for (int i = 0; i < DPL; ++i) a.out[((size_t)m * n_q + hd) * D + DPL * lane + i] = (f16)(acc[i] * inv);
}

template <int D, int CACHE>
void launch(const WindowAttn& w, hipStream_t st) {
  int lhpg = 0;
  while ((w.n_kv << lhpg) < w.n_q) ++lhpg;
  const WinArgs a{(const f16*)w.q, w.q_stride, w.pos, w.bt, (const uint8_t*)w.kc, (const uint8_t*)w.vc, w.ks, w.vs, w.n_pages,
                  w.log2P, w.n_kv, lhpg, w.M, (int)min((long long)w.max_ctx, (long long)w.n_bt << w.log2P), w.window, w.sinks,
                  (float)(1.4426950408889634 / sqrt((double)D)), (f16*)w.out};
  hipLaunchKernelGGL((attn_window_kernel<D, CACHE>), dim3((unsigned)(w.M * w.n_q)), dim3(64), 0, st, a);
}

template <int D>
void launch_cache(const WindowAttn& w, hipStream_t st) {
  if (w.cache == kCacheF16)
    launch<D, kCacheF16>(w, st);
  else if (w.cache == kCacheInt8)
    launch<D, kCacheInt8>(w, st);
  else
    launch<D, kCacheE4m3>(w, st);
}

}  // namespace

int attention_window_splits(int, int, int, int, int, int, int, int) { return 1; }
size_t attention_window_part_bytes(int M, int n_q, int, int head_dim) { return (size_t)M * n_q * (head_dim + 2) * 4; }

void launch_attention_window(const WindowAttn& a, hipStream_t st) {
  if (a.head_dim == 64)
    launch_cache<64>(a, st);
  else
    launch_cache<128>(a, st);
}

}  // namespace dk
