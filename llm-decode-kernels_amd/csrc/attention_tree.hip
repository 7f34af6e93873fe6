// Attention of the nodes of a drafted token tree over the paged cache: node i (row i of q) attends the committed tokens
// [0, *pos) and the nodes (tokens *pos + j) whose bit is set in its mask row.
#include "common.hpp"
#include "launch.hpp"
#include "attn_common.hpp"

namespace dk {
namespace {

constexpr int kTreeThreads = 256;

// One workgroup per (node, query head): scores of 256 tokens at a time into LDS, online softmax over the blocks, then
// thread (g, d) adds the tokens t % G == g of dim d.
template <int D>
__global__ void __launch_bounds__(kTreeThreads)
tree_attn_simple_kernel(const f16* __restrict__ q, long long q_stride, const int64_t* __restrict__ mask,
                        const int32_t* __restrict__ pos_ptr, const int32_t* __restrict__ bt, int n_bt,
                        const f16* __restrict__ kc, const f16* __restrict__ vc, int n_pages, int log2P, int hpg,
                        int n_kv, int M, int max_ctx, float scale, f16* __restrict__ out) {
  constexpr int G = kTreeThreads / D;
  __shared__ float s_p[kTreeThreads], s_red[kTreeThreads / kWave], s_acc[G][D];
  __shared__ int s_pg[kTreeThreads];
  const int head = blockIdx.x, i = blockIdx.y, kvh = head / hpg, tid = threadIdx.x, W = (M + 63) >> 6;
  const long long pos = *pos_ptr, cap = min((long long)max_ctx, (long long)n_bt << log2P);
  const int ctx = pos < 0 ? 0 : (int)min(pos + M, cap);
  const f16* qh = q + (size_t)i * q_stride + (size_t)head * D;
  const int g = tid / D, d = tid % D;
  float m = -INFINITY, l = 0.f, acc = 0.f;
  for (int t0 = 0; t0 < ctx; t0 += kTreeThreads) {
    const int t = t0 + tid;
    bool see = t < ctx;
    if (see && t >= pos) {
      const int j = (int)(t - pos);
      see = mask ? (mask[(size_t)i * W + (j >> 6)] >> (j & 63)) & 1 : j <= i;
    }
    const int page = see ? bt[t >> log2P] : -1;
    see = see && (unsigned)page < (unsigned)n_pages;
    float sc = -INFINITY;
    if (see) {
      const f16* kr = kc + ((((size_t)page * n_kv + kvh) << log2P) + (t & ((1 << log2P) - 1))) * D;
      float a = 0.f;
      for (int e = 0; e < D; ++e) a = fmaf((float)qh[e], (float)kr[e], a);
      sc = a * scale;
    }
    s_pg[tid] = see ? page : -1;
    const float wm = group_max<64>(sc);
    if ((tid & 63) == 0) s_red[tid >> 6] = wm;
    __syncthreads();
    float mn = m;
    for (int w = 0; w < kTreeThreads / kWave; ++w) mn = fmaxf(mn, s_red[w]);
    const float alpha = mn == -INFINITY ? 0.f : expf(m - mn);
    const float p = see ? expf(sc - mn) : 0.f;
    s_p[tid] = p;
    m = mn;
    const float ws = group_sum<64>(p);
    __syncthreads();
    if ((tid & 63) == 0) s_red[tid >> 6] = ws;
    __syncthreads();
    l *= alpha;
    for (int w = 0; w < kTreeThreads / kWave; ++w) l += s_red[w];
    acc *= alpha;
    for (int k = g; k < kTreeThreads; k += G) {
      if (s_pg[k] < 0) continue;
      const f16* vr = vc + ((((size_t)s_pg[k] * n_kv + kvh) << log2P) + ((t0 + k) & ((1 << log2P) - 1))) * D;
      acc = fmaf(s_p[k], (float)vr[d], acc);
    }
    __syncthreads();
  }
  s_acc[g][d] = acc;
  __syncthreads();
  if (g == 0) {
    for (int k = 1; k < G; ++k) acc += s_acc[k][d];
    out[((size_t)i * n_kv * hpg + head) * D + d] = (f16)(l == 0.f ? 0.f : acc / l);
  }
}

}  // namespace

int attention_tree_splits(int, int, int, int, int) { return 1; }
size_t attention_tree_part_bytes(int M, int n_q, int, int head_dim) { return (size_t)M * n_q * (head_dim + 2) * 4; }

void launch_attention_tree(const TreeAttn& a, hipStream_t st) {
  const float scale = 1.0f / sqrtf((float)a.head_dim);
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(a.n_q, a.M), dim3(kTreeThreads), 0, st, (const f16*)a.q, a.q_stride, a.mask, a.pos,
                       a.bt, a.n_bt, (const f16*)a.kc, (const f16*)a.vc, a.n_pages, a.log2P, a.n_q / a.n_kv, a.n_kv, a.M,
                       a.max_ctx, scale, (f16*)a.out);
  };
  if (a.head_dim == 64)
    go(tree_attn_simple_kernel<64>);
  else
    go(tree_attn_simple_kernel<128>);
}

}  // namespace dk
