// The small operators around a drafted token tree: per-head norm + RoPE + append of its rows, and the greedy walk down
// the verified tree with the move of the accepted cache rows.
#include "common.hpp"
#include "launch.hpp"
#include "attn_common.hpp"

namespace dk {
namespace {

// ---------------------------------------------------------------------------------------------------------------
// Per-head RMSNorm of q and k, RoPE (rotate_half pairs (i, i + D/2)) and paged append.
//   y = x w / sqrt(mean(x^2) + eps);  (a, b) -> (a c - b s, b c + a s);  fp32 throughout, rounded to fp16 once at the end
// (the products and sums of the rotation rounded separately, so that without weights the result is rope_append_rows's).
// D / 16 lanes hold a head, lane c its dims [8c, 8c + 8) and their partners D/2 further: every load and store is 16 bytes,
// a rotation pair sits in one lane and the mean needs 2 (D 64) or 3 (D 128) DPP steps.
template <int D>
__global__ void __launch_bounds__(256)
qk_norm_rope_kernel(const f16* qkv, f16* q_out, long long q_stride, const int32_t* __restrict__ pos_ptr,
                    const int32_t* __restrict__ depth, const int32_t* __restrict__ bt, const f16* __restrict__ q_w,
                    const f16* __restrict__ k_w, float eps, const float* __restrict__ cos_t,
                    const float* __restrict__ sin_t, f16* __restrict__ kc, f16* __restrict__ vc, int M, int n_q,
                    int n_kv, int groups, int log2P, int max_pos, int n_pages, int n_bt) {
#pragma clang fp contract(off)
  constexpr int LPH = D / 16, HPW = kWave / LPH;  // lanes per head, heads per wave
  const int wave = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int m = wave / groups, grp = wave - m * groups;
  if (m >= M) return;  // uniform per wave
  const int c = lane % LPH;
  const int head = grp * HPW + lane / LPH, heads = n_q + 2 * n_kv;
  const long long t = (long long)*pos_ptr + m;
  const long long rot = depth ? (long long)*pos_ptr + depth[m] : t;
  if (t < 0 || rot < 0 || rot >= max_pos) return;
  const bool live = head < heads;
  const f16* src = qkv + ((size_t)m * heads + (live ? head : 0)) * D + 8 * c;
  const u32x4 lo = *reinterpret_cast<const u32x4*>(src), hi = *reinterpret_cast<const u32x4*>(src + D / 2);
  const long long lp = t >> log2P;
  const int page = lp < n_bt ? bt[lp] : -1;
  const bool mapped = (unsigned)page < (unsigned)n_pages;
  const int kvh = head < n_q + n_kv ? head - n_q : head - n_q - n_kv;
  const size_t slot = ((((size_t)(mapped ? page : 0) * n_kv + kvh) << log2P) + (size_t)(t & ((1 << log2P) - 1))) * D + 8 * c;
  if (head >= n_q + n_kv) {  // v: copied
    if (live && mapped) {
      *reinterpret_cast<u32x4*>(vc + slot) = lo;
      *reinterpret_cast<u32x4*>(vc + slot + D / 2) = hi;
    }
    return;
  }
  float a[8], b[8];
  unpack8(lo, a);
  unpack8(hi, b);
  if (q_w) {
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss += a[e] * a[e] + b[e] * b[e];
    ss = group_sum<LPH>(ss);
    const float r = 1.0f / sqrtf(ss / (float)D + eps);
    const f16* w = (head < n_q ? q_w : k_w) + 8 * c;
    float wa[8], wb[8];
    unpack8(*reinterpret_cast<const u32x4*>(w), wa);
    unpack8(*reinterpret_cast<const u32x4*>(w + D / 2), wb);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      a[e] = a[e] * r * wa[e];
      b[e] = b[e] * r * wb[e];
    }
  }
  const float* cs = cos_t + (size_t)rot * (D / 2) + 8 * c;
  const float* sn = sin_t + (size_t)rot * (D / 2) + 8 * c;
  u32x4 ol, oh;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    f16 l2[2], h2[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int i = 2 * k + e;
      const float ac = a[i] * cs[i], bs = b[i] * sn[i], bc = b[i] * cs[i], as = a[i] * sn[i];
      l2[e] = (f16)(ac - bs);
      h2[e] = (f16)(bc + as);
    }
    ol[k] = as_u32(f16x2{l2[0], l2[1]});
    oh[k] = as_u32(f16x2{h2[0], h2[1]});
  }
  if (head < n_q) {
    f16* dst = q_out + (size_t)m * q_stride + (size_t)head * D + 8 * c;
    *reinterpret_cast<u32x4*>(dst) = ol;
    *reinterpret_cast<u32x4*>(dst + D / 2) = oh;
  } else if (mapped) {
    *reinterpret_cast<u32x4*>(kc + slot) = ol;
    *reinterpret_cast<u32x4*>(kc + slot + D / 2) = oh;
  }
}

// ---------------------------------------------------------------------------------------------------------------
// The greedy walk, done by every workgroup for itself (a second launch or a wait between workgroups would cost more than
// the walk), and the move of the accepted rows. A thread owns one 16-byte chunk of a row in one cache and moves it for
// every accepted token in order: targets never lie ahead of a later source (path[t] >= t, strictly increasing), and no
// other thread touches the chunk.
__global__ void __launch_bounds__(256)
tree_accept_kernel(const int64_t* __restrict__ tokens, const int32_t* __restrict__ parents,
                   const int64_t* __restrict__ picks, long long picks_stride, int M, const int32_t* __restrict__ pos_ptr,
                   const int32_t* __restrict__ bt, int n_bt, uint8_t* kv, long long chunks, int n_pages, int n_kv,
                   int log2P, int log2C, int32_t* __restrict__ path, int32_t* __restrict__ count,
                   int64_t* __restrict__ tok) {
  __shared__ int64_t s_tok[kTreeMaxNodes], s_pick[kTreeMaxNodes];
  __shared__ int s_par[kTreeMaxNodes], s_path[kTreeMaxNodes], s_n;
  const int tid = threadIdx.x;
  for (int i = tid; i < M; i += 256) {
    s_tok[i] = tokens[i];
    s_pick[i] = picks[i * picks_stride];
    s_par[i] = parents[i];
  }
  __syncthreads();
  if (tid < kWave) {
    int cur = 0, n = 1;
    if (tid == 0) s_path[0] = 0;
    for (int base = 1; base < M;) {  // children lie behind their parent: cur only grows
      const int c = base + tid;
      const uint64_t hit = __ballot(c < M && s_par[c < M ? c : 0] == cur && s_tok[c < M ? c : 0] == s_pick[cur]);
      if (hit == 0) {
        base += kWave;
        continue;
      }
      cur = base + __builtin_ctzll(hit);
      base = cur + 1;
      if (tid == 0) s_path[n] = cur;
      ++n;
    }
    if (tid == 0) s_n = n;
  }
  __syncthreads();
  const int n = s_n;
  if (blockIdx.x == 0) {
    for (int i = tid; i < M; i += 256) path[i] = i < n ? s_path[i] : -1;
    if (tid == 0) {
      *count = n;
      *tok = s_pick[s_path[n - 1]];
    }
  }
  const long long id = (long long)blockIdx.x * 256 + tid;
  if (id >= chunks) return;
  const long long P = 1ll << log2P, cap = (long long)n_bt << log2P;
  const int ch = (int)(id & ((1 << log2C) - 1));
  const long long hc = id >> log2C;
  const int kvh = (int)(hc % n_kv);
  const size_t base = (size_t)(hc / n_kv) * n_pages;
  auto row = [&](long long t) -> uint8_t* {  // token t's chunk, null where it has no page
    if (t < 0 || t >= cap) return nullptr;
    const int p = bt[t >> log2P];
    if ((unsigned)p >= (unsigned)n_pages) return nullptr;
    return kv + (((((base + p) * n_kv + kvh) << log2P) + (size_t)(t & (P - 1))) << (log2C + 4)) + 16 * ch;
  };
  const long long pos = *pos_ptr;
  for (int i = 1; i < n; ++i) {
    const int from = s_path[i];
    if (from == i) continue;
    const uint8_t* src = row(pos + from);
    uint8_t* dst = row(pos + i);
    if (src && dst) *reinterpret_cast<u32x4*>(dst) = *reinterpret_cast<const u32x4*>(src);
  }
}

}  // namespace

void launch_qk_norm_rope(const QkNormRope& a, hipStream_t st) {
  const int hpw = kWave / (a.head_dim / 16);
  const int groups = (a.n_q + 2 * a.n_kv + hpw - 1) / hpw;
  const unsigned blocks = (unsigned)(((long long)a.M * groups + 3) / 4);
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(256), 0, st, (const f16*)a.qkv, (f16*)a.q_out, a.q_stride, a.pos,
                       a.depth, a.bt, (const f16*)a.q_w, (const f16*)a.k_w, a.eps, a.cos_t, a.sin_t, (f16*)a.kc,
                       (f16*)a.vc, a.M, a.n_q, a.n_kv, groups, a.log2P, a.max_pos, a.n_pages, a.n_bt);
  };
  if (a.head_dim == 64)
    go(qk_norm_rope_kernel<64>);
  else
    go(qk_norm_rope_kernel<128>);
}

void launch_tree_accept(const TreeAccept& a, hipStream_t st) {
  const int log2C = a.head_dim == 64 ? 3 : 4;  // 16-byte chunks of a row
  const long long chunks = ((long long)a.n_caches * a.n_kv) << log2C;
  const unsigned blocks = (unsigned)(chunks > 0 ? (chunks + 255) / 256 : 1);
  hipLaunchKernelGGL(tree_accept_kernel, dim3(blocks), dim3(256), 0, st, a.tokens, a.parents, a.picks, a.picks_stride,
                     a.M, a.pos, a.bt, a.n_bt, (uint8_t*)a.kv, chunks, a.n_pages, a.n_kv, a.log2P, log2C, a.path,
                     a.count, a.tok);
}

}  // namespace dk
