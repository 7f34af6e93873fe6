// The 8-bit cache, written and read back: RoPE of rows and their K / V as codes (kv8.hpp), and codes as fp16 rows.
#include "kv8.hpp"

namespace dk {
namespace {

// ---------------------------------------------------------------------------------------------------------------
// Append. A wave owns one block of 16 tokens of one kv head, of K or of V: D / 8 lanes hold a row, eight values each, so
// that every load is 16 bytes and the block's largest value is a reduction inside the wave. K is rotated as
// dk_rope_append rotates it and rounded to fp16; that value is what is quantized. The waves behind those rotate q.
//   scale = that of the new rows' largest value; where the block holds rows ahead of the new ones, the larger of that and
//   the one it had. If it grows, those rows' codes are taken anew from their values.
// (A block belongs to one wave, so nothing is shared between waves.)
template <int D, int CACHE>
__device__ __forceinline__ void append_block(const Kv8Append& a, long long pos, int blk, int kvh, bool is_v, int lane) {
  constexpr int CPL = D / 8, RPP = kWave / CPL, NP = 16 / RPP;  // lanes per row, rows per pass, passes
  const int c = lane % CPL;
  const long long first = (pos & ~15LL) + 16LL * blk;  // the block's first token
  if (first + 15 < 0 || first >= pos + a.M) return;     // uniform
  const long long lp = first >> a.log2P;
  const int page = first >= 0 && lp < a.n_bt ? a.bt[lp] : -1;
  if ((unsigned)page >= (unsigned)a.n_pages) return;
  const int slot = (int)(first & ((1 << a.log2P) - 1));
  const size_t tile = (((size_t)page * a.n_kv + kvh) << a.log2P) + slot;  // the block's first row in the cache
  uint8_t* codes = (is_v ? a.vc : a.kc) + tile * D + 8 * c;
  float* scale = (is_v ? a.vs : a.ks) + (tile >> 4);
  const int heads = a.n_q + 2 * a.n_kv, head = a.n_q + (is_v ? a.n_kv : 0) + kvh;
  const long long end = min(pos + a.M, (long long)a.max_pos);  // tokens that are appended: [max(pos, 0), end)
  if (first >= end) return;
  const float had = first < pos ? *scale : 0.f;
  u32x4 x[NP];
  bool mine[NP];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const long long t = first + RPP * i + lane / CPL;
    mine[i] = t >= max(pos, 0LL) && t < end;
    const f16* row = a.qkv + ((size_t)(mine[i] ? t - pos : 0) * heads + head) * D + 8 * c;
    x[i] = mine[i] ? *reinterpret_cast<const u32x4*>(row) : u32x4{0u, 0u, 0u, 0u};
    if (!is_v && a.cos_t) {  // uniform
      u32x4 other;
#pragma unroll
      for (int j = 0; j < 4; ++j) other[j] = __shfl_xor(x[i][j], CPL / 2, kWave);
      const size_t at = (size_t)(mine[i] ? t : 0) * (D / 2) + 8 * (c % (CPL / 2));
      float cs[8], sn[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        cs[e] = a.cos_t[at + e];
        sn[e] = a.sin_t[at + e];
      }
      x[i] = rope_slice<D>(x[i], other, cs, sn, c < CPL / 2);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        uint32_t m = (x[i][j] >> (16 * e)) & 0x7FFFu;
        m = m == 0x7C00u ? 0x7BFFu : m;  // an infinity is stored as the largest fp16 value
        if (m < 0x7C00u && mine[i]) top = max(top, m);
      }
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, kWave));
  const float need = kv8_scale<CACHE>((float)as_f16x2(top)[0]);
  // (a scale that this library did not write is not taken further than its own go)
  const float s = had > need && had <= kKv8MaxScale ? had : need, inv = 1.0f / s;
  using Codes = Kv8Codes<CACHE>;
  const float big = s == Codes::top_scale ? Codes::top_code : Codes::most;
  const bool grows = first < pos && had != s;  // uniform: the rows before pos take the new scale
  const float ratio = had * inv;
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int row = RPP * i + lane / CPL;
    float v[8];
    bool put = mine[i];
    if (grows && first + row < pos) {
      const u32x2 old = *reinterpret_cast<const u32x2*>(codes + row * D);
      unpack8(kv8_decode8<CACHE>(old, 1.0f), v);  // the codes themselves
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= ratio;
      put = true;
    } else {
      unpack8(x[i], v);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= inv;
    }
    float lo[4] = {v[0], v[1], v[2], v[3]}, hi[4] = {v[4], v[5], v[6], v[7]};
    if (put) *reinterpret_cast<u32x2*>(codes + row * D) = u32x2{kv8_encode4<CACHE>(lo, big), kv8_encode4<CACHE>(hi, big)};
  }
  if (lane == 0) *scale = s;
}

template <int D, int CACHE>
__global__ void __launch_bounds__(256) kv8_append_kernel(const Kv8Append a, int kv_waves, int q_waves) {
  constexpr int CPL = D / 8, HPW = kWave / CPL;
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
  const long long i = (long long)wave * HPW + lane / CPL;  // (row, query head)
  const int c = lane % CPL;
  const long long m = i / a.n_q, t = pos + m;
  const int head = (int)(i - m * a.n_q);
  const bool live = m < a.M && t >= 0 && t < a.max_pos;
  const f16* src = a.qkv + ((size_t)(live ? m : 0) * (a.n_q + 2 * a.n_kv) + (live ? head : 0)) * D + 8 * c;
  u32x4 x = *reinterpret_cast<const u32x4*>(src);
  if (a.cos_t) {  // uniform
    u32x4 other;
#pragma unroll
    for (int j = 0; j < 4; ++j) other[j] = __shfl_xor(x[j], CPL / 2, kWave);
    const size_t at = (size_t)(live ? t : 0) * (D / 2) + 8 * (c % (CPL / 2));
    float cs[8], sn[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      cs[e] = a.cos_t[at + e];
      sn[e] = a.sin_t[at + e];
    }
    x = rope_slice<D>(x, other, cs, sn, c < CPL / 2);
  }
  if (live) *reinterpret_cast<u32x4*>(a.q_out + (size_t)m * a.q_stride + (size_t)head * D + 8 * c) = x;
}

// ---------------------------------------------------------------------------------------------------------------
// Read back: a lane turns eight codes into 16 bytes of an fp16 row. Tokens without a page read as zeros.
template <int D, int CACHE>
__global__ void __launch_bounds__(256) kv8_read_kernel(const Kv8Read a, long long chunks) {
  constexpr int CPL = D / 8;
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= chunks) return;
  const bool is_v = blockIdx.y != 0;
  const int c = (int)(i % CPL);
  const long long row = i / CPL, n = row / a.n_kv;
  const int kvh = (int)(row - n * a.n_kv);
  const int t = a.start + (int)n, lp = t >> a.log2P;
  const int page = lp < a.n_bt ? a.bt[lp] : -1;
  u32x4 x = {0u, 0u, 0u, 0u};
  if ((unsigned)page < (unsigned)a.n_pages) {
    const size_t at = (((size_t)page * a.n_kv + kvh) << a.log2P) + (t & ((1 << a.log2P) - 1));
    const u32x2 w = *reinterpret_cast<const u32x2*>((is_v ? a.vc : a.kc) + at * D + 8 * c);
    x = kv8_decode8<CACHE>(w, (is_v ? a.vs : a.ks)[at >> 4]);
  }
  *reinterpret_cast<u32x4*>((is_v ? a.v_out : a.k_out) + (size_t)row * D + 8 * c) = x;
}

template <int D, int CACHE>
void append(const Kv8Append& a, hipStream_t st) {
  // blocks that M rows can touch, wherever in its block the first of them lies
  const int blocks = (int)(((long long)a.M + 30) / 16), kv_waves = 2 * a.n_kv * blocks;
  const int per = kWave / (D / 8);
  const bool turns = a.cos_t || a.q_out != a.qkv;
  const int q_waves = turns ? (int)(((long long)a.M * a.n_q + per - 1) / per) : 0;
  hipLaunchKernelGGL((kv8_append_kernel<D, CACHE>), dim3((kv_waves + q_waves + 3) / 4), dim3(256), 0, st, a, kv_waves, q_waves);
}

template <int D, int CACHE>
void read_back(const Kv8Read& a, hipStream_t st) {
  const long long chunks = (long long)a.n * a.n_kv * (D / 8);
  hipLaunchKernelGGL((kv8_read_kernel<D, CACHE>), dim3((unsigned)((chunks + 255) / 256), 2), dim3(256), 0, st, a, chunks);
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
