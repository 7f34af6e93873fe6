// The 8-bit cache, written and read back: RoPE of rows and their K / V as codes (kv8.hpp), and codes as fp16 rows.
#include "kv8.hpp"

namespace dk {
namespace {

// The rotation of dk_rope_append: (a, b) -> (a c - b s, b c + a s) for dims [8 c, 8 c + 8) and their partners D / 2 further,
// products and sums rounded one by one in fp32, the result rounded to fp16.
struct Turn {
  float cs[8], sn[8];
};
__device__ __forceinline__ Turn load_turn(const float* cos_t, const float* sin_t, size_t at) {
  Turn t;
#pragma unroll
  for (int e = 0; e < 8; e += 4) {
    *reinterpret_cast<f4*>(&t.cs[e]) = *reinterpret_cast<const f4*>(cos_t + at + e);
    *reinterpret_cast<f4*>(&t.sn[e]) = *reinterpret_cast<const f4*>(sin_t + at + e);
  }
  return t;
}
__device__ __forceinline__ void rotate(u32x4& lo, u32x4& hi, const Turn& t) {
#pragma clang fp contract(off)
  float a[8], b[8];
  unpack8(lo, a);
  unpack8(hi, b);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    f16 l2[2], h2[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int i = 2 * k + e;
      const float ac = a[i] * t.cs[i], bs = b[i] * t.sn[i], bc = b[i] * t.cs[i], as = a[i] * t.sn[i];
      l2[e] = (f16)(ac - bs);
      h2[e] = (f16)(bc + as);
    }
    lo[k] = as_u32(f16x2{l2[0], l2[1]});
    hi[k] = as_u32(f16x2{h2[0], h2[1]});
  }
}

// ---------------------------------------------------------------------------------------------------------------
// Append. D / 16 lanes hold a row, lane c its dims [8 c, 8 c + 8) and their partners D / 2 further: every load is 16 bytes and
// a rotation pair sits in one lane. A wave owns one block of 16 tokens of one kv head, of K or of V, so that the block's
// largest value is a reduction inside the wave and nothing is shared between waves. K is rotated and rounded to fp16; that
// value is what is quantized. The waves behind those rotate q: `per` sets of heads of one row, whose tables they load once.
//   scale = that of the new rows' largest value; where the block holds rows ahead of the new ones, the larger of that and
//   the one it had. If it grows, those rows' codes are taken anew from their values.
// What bounds it: 4096 rows, 8 x 4 heads of 128, move 94 MB in 17 us from a warm cache and 22 from a cold one (floor 19 at the
// rate of a large copy); with a chunk of a row per lane, its partner by a shuffle and the tables read per chunk 24 and 26. One
// row takes 4 us traced: position, then rows, tables and page, then the block's scale. No gain: q's waves first (25 us instead
// of 22.6 with the read back), two sets of heads per wave, stores past the cache, 64 registers for eight waves per SIMD (26).
template <int D, int CACHE>
__device__ __forceinline__ void append_block(const Kv8Append& a, long long pos, int blk, int kvh, bool is_v, int lane) {
  constexpr int LPR = D / 16, RPP = kWave / LPR, NP = 16 / RPP;  // lanes per row, rows per pass, passes
  const int c = lane % LPR;
  const long long first = (pos & ~15LL) + 16LL * blk;             // the block's first token
  const long long end = min(pos + a.M, (long long)a.max_pos);     // tokens that are appended: [max(pos, 0), end)
  if (first < 0 || max(first, pos) >= end) return;                // uniform: none of its tokens is new
  // the page, whose scale waits for it, then rows and tables, which do not
  const long long lp = first >> a.log2P;
  const int page = lp < a.n_bt ? a.bt[lp] : -1;
  const int heads = a.n_q + 2 * a.n_kv, head = a.n_q + (is_v ? a.n_kv : 0) + kvh;
  u32x4 lo[NP], hi[NP];
  Turn turn[NP];
  bool mine[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const long long t = first + RPP * i + lane / LPR;
    mine[i] = t >= pos && t < end;
    const f16* row = a.qkv + ((size_t)(mine[i] ? t - pos : 0) * heads + head) * D + 8 * c;
    lo[i] = *reinterpret_cast<const u32x4*>(row);
    hi[i] = *reinterpret_cast<const u32x4*>(row + D / 2);
    if (!is_v && a.cos_t) turn[i] = load_turn(a.cos_t, a.sin_t, (size_t)(mine[i] ? t : 0) * (D / 2) + 8 * c);  // uniform
  }
  if ((unsigned)page >= (unsigned)a.n_pages) return;
  const size_t tile = (((size_t)page * a.n_kv + kvh) << a.log2P) + (size_t)(first & ((1 << a.log2P) - 1));  // its first row
  uint8_t* codes = (is_v ? a.vc : a.kc) + tile * D + 8 * c;
  float* scale = (is_v ? a.vs : a.ks) + (tile >> 4);
  const float had = first < pos ? *scale : 0.f;
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    if (!is_v && a.cos_t) rotate(lo[i], hi[i], turn[i]);
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) most = kv8_top(hi[i][j], kv8_top(lo[i][j], most));
    top = max(top, mine[i] ? most : 0u);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, kWave));
  const float need = kv8_scale<CACHE>((float)as_f16x2(top)[0]);
  const float s = kv8_grown(had, need), inv = 1.0f / s, big = kv8_big<CACHE>(s, inv);
  const bool grows = first < pos && had != s;  // uniform: the rows before pos take the new scale
  const float ratio = had * inv;
  auto put = [&](uint8_t* at, const u32x4& x) __attribute__((always_inline)) {
    *reinterpret_cast<u32x2*>(at) = u32x2{kv8_code4<CACHE>(x[0], x[1], inv, big), kv8_code4<CACHE>(x[2], x[3], inv, big)};
  };
  auto again = [&](uint8_t* at) __attribute__((always_inline)) {
    const u32x2 w = *reinterpret_cast<const u32x2*>(at);
    *reinterpret_cast<u32x2*>(at) = u32x2{kv8_recode4<CACHE>(w[0], ratio, big), kv8_recode4<CACHE>(w[1], ratio, big)};
  };
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int row = RPP * i + lane / LPR;
    uint8_t* at = codes + row * D;
    if (mine[i]) {
      put(at, lo[i]);
      put(at + D / 2, hi[i]);
    } else if (grows && first + row < pos) {
      again(at);
      again(at + D / 2);
    }
  }
  if (lane == 0) *scale = s;
}

constexpr int kQSets = 4;  // sets of heads of q in flight per wave

template <int D, int CACHE>
__global__ void __launch_bounds__(256) kv8_append_kernel(const Kv8Append a, int kv_waves, int q_waves, int per) {
  constexpr int LPR = D / 16, HPW = kWave / LPR;
  const int lane = threadIdx.x & 63;
  int wave = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long long pos = *a.pos;
  if (wave < kv_waves) {
    const int at = wave % (2 * a.n_kv);
    append_block<D, CACHE>(a, pos, wave / (2 * a.n_kv), at % a.n_kv, at >= a.n_kv, lane);
    return;
  }
  wave -= kv_waves;
  if (wave >= q_waves) return;
  const int sets = (a.n_q + HPW - 1) / HPW, wpr = (sets + per - 1) / per;  // sets of heads, waves of a row
  const int m = wave / wpr, c = lane % LPR;
  const long long t = pos + m;
  if (t < 0 || t >= a.max_pos) return;  // uniform
  const int s0 = (wave - m * wpr) * per, s1 = min(s0 + per, sets);
  const f16* src = a.qkv + (size_t)m * (a.n_q + 2 * a.n_kv) * D + 8 * c;
  f16* dst = a.q_out + (size_t)m * a.q_stride + 8 * c;
  Turn turn;
  if (a.cos_t) turn = load_turn(a.cos_t, a.sin_t, (size_t)t * (D / 2) + 8 * c);  // uniform
  for (int s = s0; s < s1; s += kQSets) {
    u32x4 lo[kQSets], hi[kQSets];
#pragma unroll
    for (int k = 0; k < kQSets; ++k) {
      const int head = (s + k) * HPW + lane / LPR;
      if (s + k < s1 && head < a.n_q) {
        lo[k] = *reinterpret_cast<const u32x4*>(src + (size_t)head * D);
        hi[k] = *reinterpret_cast<const u32x4*>(src + (size_t)head * D + D / 2);
      }
    }
#pragma unroll
    for (int k = 0; k < kQSets; ++k) {
      const int head = (s + k) * HPW + lane / LPR;
      if (s + k < s1 && head < a.n_q) {
        if (a.cos_t) rotate(lo[k], hi[k], turn);
        *reinterpret_cast<u32x4*>(dst + (size_t)head * D) = lo[k];
        *reinterpret_cast<u32x4*>(dst + (size_t)head * D + D / 2) = hi[k];
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------
// Read back: a lane turns eight codes into 16 bytes of an fp16 row, SETS times, 256 chunks apart. Tokens without a page read
// as zeros. 16001 tokens of 8 heads of 128 take 17 us warm, 20 cold (98 MB, at the rate of a large copy; with one chunk per
// lane 23); 61 of 4 heads of 64 take 2.6.
template <int D, int CACHE, int SETS>
__global__ void __launch_bounds__(256) kv8_read_kernel(const Kv8Read a, long long chunks) {
  constexpr int CPL = D / 8;
  const bool is_v = blockIdx.y != 0;
  const uint8_t* codes = is_v ? a.vc : a.kc;
  const float* scales = is_v ? a.vs : a.ks;
  f16* out = is_v ? a.v_out : a.k_out;
  const long long i0 = (long long)blockIdx.x * (256 * SETS) + threadIdx.x;
  int page[SETS];
  size_t slot[SETS];
#pragma unroll
  for (int k = 0; k < SETS; ++k) {
    const long long i = min(i0 + 256 * k, chunks - 1), row = i / CPL, n = row / a.n_kv;
    const int t = a.start + (int)n, lp = t >> a.log2P;
    page[k] = lp < a.n_bt ? a.bt[lp] : -1;
    slot[k] = ((size_t)(row - n * a.n_kv) << a.log2P) + (t & ((1 << a.log2P) - 1));
  }
  u32x2 w[SETS];
  float s[SETS];
#pragma unroll
  for (int k = 0; k < SETS; ++k) {
    const bool ok = (unsigned)page[k] < (unsigned)a.n_pages;
    const size_t at = ((size_t)(ok ? page[k] : 0) * a.n_kv << a.log2P) + slot[k];
    w[k] = *reinterpret_cast<const u32x2*>(codes + at * D + 8 * (threadIdx.x % CPL));
    s[k] = scales[at >> 4];
    if (!ok) {
      w[k] = u32x2{0u, 0u};
      s[k] = 1.0f;
    }
  }
#pragma unroll
  for (int k = 0; k < SETS; ++k)
    if (i0 + 256 * k < chunks) *reinterpret_cast<u32x4*>(out + (size_t)(i0 + 256 * k) * 8) = kv8_decode8<CACHE>(w[k], s[k]);
}

template <int D, int CACHE>
void append(const Kv8Append& a, hipStream_t st) {
  // blocks that M rows can touch, wherever in its block the first of them lies
  const int blocks = (int)(((long long)a.M + 30) / 16), kv_waves = 2 * a.n_kv * blocks;
  const int sets = (a.n_q + kWave / (D / 16) - 1) / (kWave / (D / 16));
  const bool turns = a.cos_t || a.q_out != a.qkv;
  // a wave takes one set of heads of a row while that leaves CUs idle, else kQSets
  const int per = (long long)a.M * sets <= 2048 ? 1 : kQSets;
  const int q_waves = turns ? a.M * ((sets + per - 1) / per) : 0;
  hipLaunchKernelGGL((kv8_append_kernel<D, CACHE>), dim3((kv_waves + q_waves + 3) / 4), dim3(256), 0, st, a, kv_waves, q_waves,
                     per);
}

template <int D, int CACHE>
void read_back(const Kv8Read& a, hipStream_t st) {
  const long long chunks = (long long)a.n * a.n_kv * (D / 8), groups = (chunks + 255) / 256;
  if (groups <= 512)  // fewer workgroups than the CUs hold at once: a short chain for each
    hipLaunchKernelGGL((kv8_read_kernel<D, CACHE, 1>), dim3((unsigned)groups, 2), dim3(256), 0, st, a, chunks);
  else
    hipLaunchKernelGGL((kv8_read_kernel<D, CACHE, 4>), dim3((unsigned)((groups + 3) / 4), 2), dim3(256), 0, st, a, chunks);
}

}  // namespace

void launch_kv8_append(const Kv8Append& a, int head_dim, int cache, hipStream_t st) {
  if (head_dim == 64)
    cache == kCacheInt8 ? append<64, kCacheInt8>(a, st) : append<64, kCacheE4m3>(a, st);
  else
    cache == kCacheInt8 ? append<128, kCacheInt8>(a, st) : append<128, kCacheE4m3>(a, st);
}

void launch_kv8_read(const Kv8Read& a, int head_dim, int cache, hipStream_t st) {
  if (head_dim == 64)
    cache == kCacheInt8 ? read_back<64, kCacheInt8>(a, st) : read_back<64, kCacheE4m3>(a, st);
  else
    cache == kCacheInt8 ? read_back<128, kCacheInt8>(a, st) : read_back<128, kCacheE4m3>(a, st);
}

}  // namespace dk
