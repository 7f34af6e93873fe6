// Windowed attention of few columns: at most 16 (row, query head) pairs of a kv head, as in a decode step.
//
// Nothing is shared between waves, so K and V go from the cache to registers, a tile ahead of its products. The waves of all
// splits take the tiles of 32 tokens in turn, so that without a window the first tile's pages are looked up beside the position
// instead of behind it, and any context spreads evenly. Per tile:
//   * S^T = K . Q^T on v_mfma_f32_16x16x32_f16, 16 tokens at a time: lane (g, c) feeds token c of K and column c of Q over the
//     same dims (any order of the dims serves that both operands keep): 16 bytes of a row are one k step of fp16 values or
//     two of codes, which become fp16 with their scale here. It receives the scores of tokens 4 g + v for column c.
//   * the weights (attn_window.hpp); the first tile brings the reference at once.
//   * O^T += V^T . P^T over the 32 tokens: the weights, as two fp16 numbers, are the B operands as they are (k slot 4 s + v of
//     lane group g is token 16 s + 4 g + v). For A lane (g, r) loads dims [r D / 16, (r + 1) D / 16) of those 8 tokens' rows and transposes
//     them in registers; output tile t holds dim r D / 16 + t, so that lane (g, c) ends with D / 4 dims in a row of column c.
// Tiles that some column does not see whole: 32 token bits per column; V of tokens that do not exist is zeroed, and where the
// words hold anything that may be NaN or infinite such values are taken out of the products and added one by one for the
// columns that see their token.
//
// What bounds it: one int8 token at 131072, 8 x 4 heads of 128, takes 48 us for 269 MB, 5.6 TB/s. Small ones are launch and a
// chain of dependent loads (position and page, K / V), the waves' merge in LDS, and where they are split the join: captured,
// 4.9 us at 300 tokens of 4 x 8 heads of 64 (one launch), 7.7 at 4096 of 8 x 4 heads of 128 (traced 5.3 and 3.4). Masks as
// compares and the look for NaN on unpacked values cost 1 us (every decode step's last tile takes that path), reductions
// through LDS and a second copy of the tile's code 0.2. No gain: 16 waves (the registers of a tile do not fit).
#include "attn_window.hpp"

namespace dk {
namespace {

// Over the lanes c, c + 16, c + 32, c + 48 of a wave, by swapping rows and halves of two registers (LDS is not touched).
template <class F>
__device__ __forceinline__ float over_rows(float v, F f) {
  const uint32_t u = __float_as_uint(v);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t a0 = a[0], a1 = a[1];
  const uint32_t w = __float_as_uint(f(__uint_as_float(a0), __uint_as_float(a1)));
  const auto b = __builtin_amdgcn_permlane32_swap(w, w, false, false);
  const uint32_t b0 = b[0], b1 = b[1];
  return f(__uint_as_float(b0), __uint_as_float(b1));
}

// A value that the whole wave reads and that nothing writes ahead of that read, through the scalar cache. Elsewhere a load like
// it is a vector load wherever the kernel may store or an asm block stands between, and those return in order: a page looked
// up behind a tile's loads would come only after all of them.
template <class T>
__device__ __forceinline__ T load_scalar(const T* p) {
  return *(const __attribute__((address_space(4))) T*)p;
}

template <int D, int CACHE>
struct FewShape {
  static constexpr bool F16 = CACHE == kCacheF16;
  static constexpr int ES = F16 ? 2 : 1;        // bytes of a value in the cache
  static constexpr int KW = D * ES / 64;        // 16-byte loads of a K row per lane
  static constexpr int DPL = D / 16;            // dims of a V row per lane
  static constexpr int VW = DPL * ES / 4;       // their words
};

// Largest value over the 16 lanes of a row.
__device__ __forceinline__ float over_lanes16(float v) {
  v = fmaxf(v, DK_DPP_F32(v, 0xB1, 0xF));   // quad_perm [1,0,3,2]
  v = fmaxf(v, DK_DPP_F32(v, 0x4E, 0xF));   // quad_perm [2,3,0,1]
  v = fmaxf(v, DK_DPP_F32(v, 0x141, 0xF));  // row_half_mirror
  return fmaxf(v, DK_DPP_F32(v, 0x140, 0xF));
}

// DECODE: one row, whose q is rotated here and whose K / V are appended by the wave that has their tile: it takes the new
// row's codes into the tile that it has loaded, takes the block's others anew where its scale grows, and stores them. So the
// append adds no launch and no round trip to the cache, only this wave's arithmetic: in a decode step of 8 layers of 8 x 4
// heads of 128 at 512 tokens, e4m3, the step takes 341 us, with the append in a launch of its own 354 (at 65536 502 and 529).
template <int D, int CACHE, int NW, bool NT, bool DECODE>
__global__ void __launch_bounds__(NW * kWave, 2)
attn_few_kernel(const WinArgs a, const WinDecode dec) {
  using S = FewShape<D, CACHE>;
  constexpr bool F16 = S::F16;
  constexpr int ES = S::ES, KW = S::KW, DPL = S::DPL, VW = S::VW, KS = D / 32;
  __shared__ float s_m[NW][kFewCols], s_l[NW][kFewCols];
  __shared__ __align__(16) float s_o[NW][kFewCols][D];
  const int kvh = blockIdx.x, split = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int P = 1 << a.log2P;
  const int i0 = split * NW + wave, step = a.splits * NW;  // the wave's tiles: i0 and every step-th from there
  // pages of tile i0 as they are without a window, beside the position
  struct Pages {
    int p[2];
  };
  auto pages_at = [&](int t) __attribute__((always_inline)) {
    return Pages{{load_scalar(a.bt + min(t >> a.log2P, a.n_bt - 1)), load_scalar(a.bt + min((t + 16) >> a.log2P, a.n_bt - 1))}};
  };
  const int pos = *a.pos;
  Pages pg = pages_at(kFewTile * i0);
  const int n_q = a.n_kv << a.lhpg, cols = a.M << a.lhpg;
  const int cc = min(c, cols - 1);              // columns past the last repeat it
  const int m = cc >> a.lhpg, hd = (kvh << a.lhpg) + (cc & ((1 << a.lhpg) - 1));
  h8 q[KS];
  {
    const f16* qh = a.q + (size_t)m * a.q_stride + (size_t)hd * D;
#pragma unroll
    for (int k = 0; k < KS; ++k)  // the dims of K's k step
      q[k] = __builtin_bit_cast(
          h8, *reinterpret_cast<const u32x4*>(qh + (F16 ? 32 * k + 8 * g : 64 * (k >> 1) + 16 * g + 8 * (k & 1))));
  }
  __builtin_amdgcn_sched_barrier(0);            // (those loads go out before the position is waited for)
  if (DECODE && (pos < 0 || pos >= dec.max_pos)) return;  // uniform: nothing is touched
  const Sight mine = sight_of(pos, m, a.window, a.cap);
  const Sight s0 = sight_of(pos, 0, a.window, a.cap), s1 = sight_of(pos, a.M - 1, a.window, a.cap);
  const int ctx = s1.lim + 1;                   // tokens [0, ctx) are read
  // tiles: those of the sinks, then those of the window, nt in all
  const int all = (ctx + kFewTile - 1) / kFewTile, wt = min(s0.lo / kFewTile, all);
  const int ns = a.window > 0 ? min((min(a.sinks, ctx) + kFewTile - 1) / kFewTile, wt) : 0;
  const int nt = ns + all - wt;
  // DECODE: one more where the position is past all of them (max_ctx is): a tile that is not attended
  const int nd = DECODE && pos / kFewTile >= all ? nt + 1 : nt;
  auto tile_at = [&](int i) __attribute__((always_inline)) {
    return DECODE && i == nd - 1 ? pos & -kFewTile : kFewTile * (i < ns ? i : i + (wt - ns));
  };

  typedef uint32_t vrow __attribute__((ext_vector_type(VW)));
  struct Tile {
    int t0;
    u32x4 k[2][KW];   // by 16 tokens
    vrow v[2][4];
    float ks[2], vs[2];
    bool ok[2];       // the page is mapped; uniform
  };
  auto lookup = [&](int i) __attribute__((always_inline)) { return pages_at(tile_at(i)); };
  auto load = [&](int i, const Pages& w) __attribute__((always_inline)) {
    Tile x;
    x.t0 = tile_at(i);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      x.ok[s] = (unsigned)w.p[s] < (unsigned)a.n_pages;
      // (16 tokens lie in one page; without one, rows of a page that exists)
      const size_t row = (((size_t)(x.ok[s] ? w.p[s] : 0) * a.n_kv + kvh) << a.log2P) + ((x.t0 + 16 * s) & (P - 1));
      const uint8_t* kr = a.kc + row * (D * ES) + c * (D * ES) + 16 * g;
      const uint8_t* vr = a.vc + row * (D * ES) + 4 * g * (D * ES) + c * (DPL * ES);
#pragma unroll
      for (int j = 0; j < KW; ++j) {
        const u32x4* p = reinterpret_cast<const u32x4*>(kr + 64 * j);
        x.k[s][j] = NT ? load_stream(p) : *p;
      }
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const vrow* p = reinterpret_cast<const vrow*>(vr + v * (D * ES));
        x.v[s][v] = NT ? __builtin_nontemporal_load(p) : *p;
      }
      if constexpr (!F16) {
        x.ks[s] = load_scalar(a.ks + (row >> 4));
        x.vs[s] = load_scalar(a.vs + (row >> 4));
      }
    }
    return x;
  };

  float ref = kWinNoMax, lift = -kWinNoMax, l = 0.f;  // as in the kernel of many columns
  f4 acc[DPL];
#pragma unroll
  for (int t = 0; t < DPL; ++t) acc[t] = f4{0.f, 0.f, 0.f, 0.f};

  // the V operand of output tile t: dim DPL r + t of the 8 tokens
  auto operand = [&](const Tile& x, const uint32_t (&tr)[2][VW][4], int t) __attribute__((always_inline)) -> u32x4 {
    if constexpr (F16) {
      const uint32_t sel = (t & 1) ? 0x07060302u : 0x05040100u;
      u32x4 r;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        r[2 * s] = __builtin_amdgcn_perm(x.v[s][1][t >> 1], x.v[s][0][t >> 1], sel);
        r[2 * s + 1] = __builtin_amdgcn_perm(x.v[s][3][t >> 1], x.v[s][2][t >> 1], sel);
      }
      return r;
    } else {
      const u32x2 lo = kv8_decode4<CACHE>(tr[0][t >> 2][t & 3], x.vs[0]);
      const u32x2 hi = kv8_decode4<CACHE>(tr[1][t >> 2][t & 3], x.vs[1]);
      return u32x4{lo[0], lo[1], hi[0], hi[1]};
    }
  };
  auto finite = [](u32x4 x) __attribute__((always_inline)) -> u32x4 {  // zero for what is no finite number
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if ((x[i] & 0x7C00u) == 0x7C00u) x[i] &= 0xFFFF0000u;
      if ((x[i] & 0x7C000000u) == 0x7C000000u) x[i] &= 0xFFFFu;
    }
    return x;
  };
  // ---- DECODE: q's rotation, and this token's K and V in the layouts of the operands
  const bool owner = DECODE && i0 == (nd - 1) % step;  // uniform per wave
  h8 kn[DECODE ? KS : 1];
  typedef uint32_t vnew __attribute__((ext_vector_type(DPL / 2)));
  vnew vn;
  if constexpr (DECODE) {
    static_assert(!F16, "the append is the 8-bit one");
    if (owner) {
      const f16* kr = a.q + (size_t)(n_q + kvh) * D;
#pragma unroll
      for (int k = 0; k < KS; ++k)
        kn[k] = __builtin_bit_cast(h8, *reinterpret_cast<const u32x4*>(kr + 64 * (k >> 1) + 16 * g + 8 * (k & 1)));
      vn = *reinterpret_cast<const vnew*>(a.q + (size_t)(n_q + a.n_kv + kvh) * D + DPL * c);
    }
    // dims 64 (k / 2) + 16 g + 8 (k % 2): the partner D / 2 further is k ^ 2 of the lane (D 128) or k of lane group g ^ 2 (D 64)
    float cs[2][8], sn[2][8];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const size_t at = (size_t)pos * (D / 2) + (16 * g + 8 * k) % (D / 2);
#pragma unroll
      for (int e = 0; e < 8; e += 4) {
        *reinterpret_cast<f4*>(&cs[k][e]) = *reinterpret_cast<const f4*>(dec.cos_t + at + e);
        *reinterpret_cast<f4*>(&sn[k][e]) = *reinterpret_cast<const f4*>(dec.sin_t + at + e);
      }
    }
    auto turn = [&](h8* f) __attribute__((always_inline)) {
      u32x4 own[KS], other[KS];
#pragma unroll
      for (int k = 0; k < KS; ++k) own[k] = __builtin_bit_cast(u32x4, f[k]);
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        if constexpr (D == 128) {
          other[k] = own[k ^ 2];
        } else {
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const uint32_t u = own[k][w];
            const auto both = __builtin_amdgcn_permlane32_swap(u, u, false, false);
            const uint32_t lo = both[0], hi = both[1];
            other[k][w] = lane < 32 ? hi : lo;
          }
        }
      }
#pragma unroll
      for (int k = 0; k < KS; ++k)
        f[k] = __builtin_bit_cast(h8, rope_slice<D>(own[k], other[k], cs[k & 1], sn[k & 1], D == 128 ? k < 2 : g < 2));
    };
    turn(q);
    if (owner) turn(kn);
  }
  auto append = [&](Tile& x) __attribute__((always_inline)) {
    if constexpr (DECODE) {
      const int row = pos & 15, page = load_scalar(a.bt + min(pos >> a.log2P, a.n_bt - 1));
      if (pos >> a.log2P >= a.n_bt || (unsigned)page >= (unsigned)a.n_pages) return;  // uniform
      const size_t at = (((size_t)page * a.n_kv + kvh) << a.log2P) + (pos & (P - 1) & ~15);  // the block's first row
      uint8_t* kb = const_cast<uint8_t*>(a.kc) + at * D + c * D + 16 * g;
      uint8_t* vb = const_cast<uint8_t*>(a.vc) + at * D + c * DPL;
      const auto larger = [](float x, float y) { return fmaxf(x, y); };
      uint32_t tk = 0, tv = 0;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const u32x4 w = __builtin_bit_cast(u32x4, kn[k]);
#pragma unroll
        for (int j = 0; j < 4; ++j) tk = kv8_top(w[j], tk);
      }
#pragma unroll
      for (int j = 0; j < DPL / 2; ++j) tv = kv8_top(vn[j], tv);
      const float need_k = kv8_scale<CACHE>(over_rows((float)as_f16x2(tk)[0], larger));
      const float need_v = kv8_scale<CACHE>(over_lanes16((float)as_f16x2(tv)[0]));
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        if (((pos >> 4) & 1) != s) continue;  // uniform
        const float had_k = row ? x.ks[s] : 0.f, had_v = row ? x.vs[s] : 0.f;
        const float sk = kv8_grown(had_k, need_k), sv = kv8_grown(had_v, need_v);
        const float ik = 1.0f / sk, iv = 1.0f / sv, big_k = kv8_big<CACHE>(sk, ik), big_v = kv8_big<CACHE>(sv, iv);
        if (row && had_k != sk) {             // uniform
          const float ratio = had_k * ik;
#pragma unroll
          for (int j = 0; j < KW; ++j) {
            if (c < row) {
#pragma unroll
              for (int w = 0; w < 4; ++w) x.k[s][j][w] = kv8_recode4<CACHE>(x.k[s][j][w], ratio, big_k);
              *reinterpret_cast<u32x4*>(kb + 64 * j) = x.k[s][j];
            }
          }
        }
        if (row && had_v != sv) {
          const float ratio = had_v * iv;
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            if (4 * g + v < row) {
#pragma unroll
              for (int w = 0; w < VW; ++w) x.v[s][v][w] = kv8_recode4<CACHE>(x.v[s][v][w], ratio, big_v);
              *reinterpret_cast<vrow*>(vb + (4 * g + v) * D) = x.v[s][v];
            }
          }
        }
        if (c == row) {
#pragma unroll
          for (int j = 0; j < KW; ++j) {
            const u32x4 lo = __builtin_bit_cast(u32x4, kn[2 * j]), hi = __builtin_bit_cast(u32x4, kn[2 * j + 1]);
            x.k[s][j] = u32x4{kv8_code4<CACHE>(lo[0], lo[1], ik, big_k), kv8_code4<CACHE>(lo[2], lo[3], ik, big_k),
                              kv8_code4<CACHE>(hi[0], hi[1], ik, big_k), kv8_code4<CACHE>(hi[2], hi[3], ik, big_k)};
            *reinterpret_cast<u32x4*>(kb + 64 * j) = x.k[s][j];
          }
        }
        vrow code;
#pragma unroll
        for (int w = 0; w < VW; ++w) code[w] = kv8_code4<CACHE>(vn[2 * w], vn[2 * w + 1], iv, big_v);
#pragma unroll
        for (int v = 0; v < 4; ++v)
          if (4 * g + v == row) {
            x.v[s][v] = code;
            *reinterpret_cast<vrow*>(vb + row * D) = code;
          }
        x.ks[s] = sk;
        x.vs[s] = sv;
        if (lane == 0) {
          const_cast<float*>(a.ks)[at >> 4] = sk;
          const_cast<float*>(a.vs)[at >> 4] = sv;
        }
      }
    }
  };
  auto compute = [&](Tile& x, bool first) __attribute__((always_inline)) {
    const int t0 = x.t0;
    // every column sees every token; uniform per wave
    const bool plain = x.ok[0] && x.ok[1] && t0 + kFewTile - 1 <= s0.lim && (t0 >= s1.lo || t0 + kFewTile <= a.sinks);
    f4 sc[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      sc[s] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < KW; ++j) {
        if constexpr (F16) {
          sc[s] = mfma16x32(__builtin_bit_cast(h8, x.k[s][j]), q[j], sc[s]);
        } else {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const u32x4 k = kv8_decode8<CACHE>(u32x2{x.k[s][j][2 * e], x.k[s][j][2 * e + 1]}, x.ks[s]);
            sc[s] = mfma16x32(__builtin_bit_cast(h8, k), q[2 * j + e], sc[s]);
          }
        }
      }
    }
    if (!plain) {
      asm volatile("");  // stays a branch
      auto low = [](int n) __attribute__((always_inline)) -> uint32_t { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1; };
      // tokens of the tile that exist (uniform), and those that the column sees, from this lane's first one on
      const uint32_t there = low(ctx - t0) & ((x.ok[0] ? 0xFFFFu : 0u) | (x.ok[1] ? 0xFFFF0000u : 0u));
      const uint32_t seen = (there & low(mine.lim + 1 - t0) & (~low(mine.lo - t0) | low(a.sinks - t0))) >> (4 * g);
      const uint32_t real = there >> (4 * g);
#pragma unroll
      for (int s = 0; s < 2; ++s) {
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          if (!(seen & (1u << (16 * s + v)))) sc[s][v] = -INFINITY;
          if (!(real & (1u << (16 * s + v)))) x.v[s][v] = vrow(0u);  // (its V must not meet a p of 0)
        }
        if constexpr (!F16) x.vs[s] = there & (1u << (16 * s)) ? x.vs[s] : 1.f;
      }
    }
    float p[2][4];
    auto weigh = [&](float off, float lift) __attribute__((always_inline)) -> float {
      float sum = 0.f;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          p[s][v] = __builtin_amdgcn_exp2f(fmaf(sc[s][v] - off, a.c2, lift));
          sum += p[s][v];
        }
      }
      return sum;
    };
    float sum = INFINITY;            // (the first tile brings the reference)
    if (!first) sum = weigh(0.f, lift);
    if (__any(!(sum <= kWinMost))) {  // the reference moves to this tile's maximum where that is higher
      asm volatile("");
      float mx = sc[0][0];
#pragma unroll
      for (int s = 0; s < 2; ++s) {
#pragma unroll
        for (int v = 0; v < 4; ++v) mx = fmaxf(mx, sc[s][v]);
      }
      const auto larger = [](float x, float y) { return fmaxf(x, y); };
      mx = fmaxf(ref, over_rows(mx, larger));
      mx = over_rows(sum <= kWinMost ? 0.f : 1.f, larger) != 0.f ? mx : ref;  // in any of the column's four lanes
      const float alpha = __builtin_amdgcn_exp2f((ref - mx) * a.c2);  // 1 for a column that stays
      if (mx != ref) lift = fabsf(mx * a.c2) > kWinFar ? INFINITY : kWinLift - mx * a.c2;
      ref = mx;
      l *= alpha;
#pragma unroll
      for (int t = 0; t < DPL; ++t) acc[t] *= alpha;
      sum = weigh(lift == INFINITY ? ref : 0.f, lift == INFINITY ? kWinLift : lift);
    }
    l += sum;
    h8 ph, pl;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int v = 0; v < 4; v += 2) {
        const h2 hi = __builtin_convertvector(f2{p[s][v], p[s][v + 1]}, h2);
        const uint32_t pair = __builtin_bit_cast(uint32_t, hi);
        const h2 lo = __builtin_convertvector(f2{minus_lo(p[s][v], pair), minus_hi(p[s][v + 1], pair)}, h2);
        ph[4 * s + v] = hi[0];
        ph[4 * s + v + 1] = hi[1];
        pl[4 * s + v] = lo[0];
        pl[4 * s + v + 1] = lo[1];
      }
    }
    auto weighted = [&](u32x4 v, f4 c) __attribute__((always_inline)) {
      return mfma16x32(__builtin_bit_cast(h8, v), pl, mfma16x32(__builtin_bit_cast(h8, v), ph, c));
    };
    // codes: bytes of four tokens' words to words of four tokens
    uint32_t tr[2][VW][4];
    if constexpr (!F16) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
#pragma unroll
        for (int w = 0; w < VW; ++w) {
          const uint32_t al = __builtin_amdgcn_perm(x.v[s][1][w], x.v[s][0][w], 0x05010400u);
          const uint32_t ah = __builtin_amdgcn_perm(x.v[s][1][w], x.v[s][0][w], 0x07030602u);
          const uint32_t bl = __builtin_amdgcn_perm(x.v[s][3][w], x.v[s][2][w], 0x05010400u);
          const uint32_t bh = __builtin_amdgcn_perm(x.v[s][3][w], x.v[s][2][w], 0x07030602u);
          tr[s][w][0] = __builtin_amdgcn_perm(bl, al, 0x05040100u);
          tr[s][w][1] = __builtin_amdgcn_perm(bl, al, 0x07060302u);
          tr[s][w][2] = __builtin_amdgcn_perm(bh, ah, 0x05040100u);
          tr[s][w][3] = __builtin_amdgcn_perm(bh, ah, 0x07060302u);
        }
      }
    }
    bool dirty = false;  // NaN or infinity in V of a tile that not every column sees whole; uniform
    if (!plain) {
      asm volatile("");
      // a look at the words first: fp16 with all exponent bits, e4m3's NaN, a scale that takes a code past fp16
      uint32_t odd = 0;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
#pragma unroll
        for (int v = 0; v < 4; ++v) {
#pragma unroll
          for (int w = 0; w < VW; ++w) {
            if constexpr (F16)
              odd |= ((x.v[s][v][w] & 0x7C007C00u) + 0x04000400u) & 0x80008000u;
            else if constexpr (CACHE == kCacheE4m3)
              odd |= ((x.v[s][v][w] & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
          }
        }
        if constexpr (!F16) odd |= x.vs[s] <= (CACHE == kCacheInt8 ? 512.f : 128.f) ? 0u : 1u;
      }
      if (__any(odd != 0)) {
        asm volatile("");
#pragma unroll
        for (int t = 0; t < DPL; ++t) dirty = dirty || has_nonfinite(operand(x, tr, t));
        dirty = __any(dirty);
      }
    }
    if (!dirty) {
#pragma unroll
      for (int t = 0; t < DPL; ++t) acc[t] = weighted(operand(x, tr, t), acc[t]);
      return;
    }
    asm volatile("");
    if constexpr (DECODE) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "agent");  // V is read again, the appended row with it
#pragma unroll
    for (int t = 0; t < DPL; ++t) acc[t] = weighted(finite(operand(x, tr, t)), acc[t]);
    // the values left out, for the columns that see their token
    for (int i = 0; i < kFewTile; ++i) {
      const int t = t0 + i, s = i >> 4;
      if (!((s ? x.ok[1] : x.ok[0]) && t < ctx)) continue;  // uniform
      const bool see = t <= mine.lim && (t >= mine.lo || t < a.sinks);
      float w = 0.f;                        // p of token i: in lane group i / 4 % 4, element (s, i % 4)
#pragma unroll
      for (int e = 0; e < 8; ++e) w = e == 4 * s + (i & 3) ? p[e >> 2][e & 3] : w;
      w = __shfl(w, 16 * ((i >> 2) & 3) + c, kWave);
      const size_t at = (((size_t)a.bt[t >> a.log2P] * a.n_kv + kvh) << a.log2P) + (t & (P - 1));
#pragma unroll
      for (int v = 0; v < 4; ++v) {
#pragma unroll
        for (int d = 0; d < DPL; d += 4) {
          const size_t off = at * D + (size_t)(4 * g + v) * DPL + d;
          u32x2 b;
          if constexpr (F16)
            b = *reinterpret_cast<const u32x2*>(a.vc + 2 * off);
          else
            b = kv8_decode4<CACHE>(*reinterpret_cast<const uint32_t*>(a.vc + off), s ? x.vs[1] : x.vs[0]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float f = (float)as_f16x2(b[e >> 1])[e & 1];
            if (see && !(fabsf(f) <= 65504.f)) acc[d + e][v] = fmaf(w, f, acc[d + e][v]);
          }
        }
      }
    }
  };

  if (i0 < nd) {  // uniform per wave
    if (a.window > 0 || (DECODE && i0 >= nt)) pg = lookup(i0);
    // the next tile's loads go out ahead of a tile's products; behind the last one every wave's are of tile 0, from a cache
    auto live = [&](int i) __attribute__((always_inline)) { return i < nd ? i : 0; };
    Tile x = load(i0, pg);
    pg = lookup(live(i0 + step));
#pragma unroll 1
    for (int i = i0; i < nd; i += step) {
      const Tile y = load(live(i + step), pg);
      pg = lookup(live(i + 2 * step));
      if (DECODE && i == nd - 1) append(x);
      compute(x, i == i0);
      x = y;
    }
  }
  l = over_rows(l, [](float x, float y) { return x + y; });
  // ---- the waves meet in LDS, in order: column c's dims [D / 4 g, + D / 4), acc[t][v] dim D / 4 g + DPL v + t
  if (g == 0) {
    s_m[wave][c] = ref;
    s_l[wave][c] = l;
  }
  if (c < cols) {
#pragma unroll
    for (int v = 0; v < 4; ++v) {
#pragma unroll
      for (int t = 0; t < DPL; t += 4)
        *reinterpret_cast<f4*>(&s_o[wave][c][D / 4 * g + DPL * v + t]) =
            f4{acc[t][v], acc[t + 1][v], acc[t + 2][v], acc[t + 3][v]};
    }
  }
  __syncthreads();
  const size_t part = (size_t)split * a.n_kv + kvh;
  const bool none = split * NW >= nt;  // a split without tokens: the join reads no output of it
  for (int j = tid; j < cols * (D / 4); j += NW * kWave) {
    const int col = j / (D / 4), d = 4 * (j % (D / 4));
    float mx = kWinNoMax, L = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) mx = fmaxf(mx, s_m[w][col]);
    f4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      // a wave that saw no token weighs 0 beside one that did
      const float f = __builtin_amdgcn_exp2f((s_m[w][col] - mx) * a.c2);
      L = fmaf(f, s_l[w][col], L);
      const f4 y = *reinterpret_cast<const f4*>(&s_o[w][col][d]);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = fmaf(f, y[e], o[e]);
    }
    if (a.splits > 1) {
      if (d == 0) a.part_ml[part * kFewCols + col] = none ? float2{kWinNoMax, 0.f} : float2{mx, L};
      if (!none) store_through16(a.part_o + part * kFewCols * (D / 4), 4 * (col * D + d), __builtin_bit_cast(u32x4, o));
      continue;
    }
    const float inv = L == 0.f ? 0.f : 1.0f / L;  // a NaN stays
    const int mo = col >> a.lhpg, ho = (kvh << a.lhpg) + (col & ((1 << a.lhpg) - 1));
    *reinterpret_cast<u32x2*>(a.out + ((size_t)mo * n_q + ho) * D + d) =
        u32x2{as_u32(f16x2{(f16)(o[0] * inv), (f16)(o[1] * inv)}), as_u32(f16x2{(f16)(o[2] * inv), (f16)(o[3] * inv)})};
  }
}

// Joins the splits of one column, in split order: groups of D / 4 threads take the splits i, i + G, ..., then meet in LDS.
template <int D>
__global__ void __launch_bounds__(256)
attn_few_join_kernel(const f4* __restrict__ part_o, const float2* __restrict__ part_ml, int lhpg, int n_kv, int splits,
                     float c2, f16* __restrict__ out, const int32_t* __restrict__ pos, int max_pos) {
  if (pos && (*pos < 0 || *pos >= max_pos)) return;  // uniform: nothing was written
  constexpr int T = D / 4, G = 256 / T;
  __shared__ float s_w[kWinMaxSplits];
  __shared__ float s_l;
  __shared__ f4 s_o[G][T];
  const int kvh = blockIdx.x, col = blockIdx.y, tid = threadIdx.x, d = tid % T, grp = tid / T;
  const size_t step = (size_t)n_kv * kFewCols, first = (size_t)kvh * kFewCols + col;
  constexpr int NB = kWinMaxSplits / G;
  f4 x[NB];
#pragma unroll
  for (int k = 0; k < NB; ++k) {
    const int s = grp + G * k;
    if (s < splits) x[k] = part_o[((size_t)s * step + first) * T + d];
  }
  if (tid < kWave) {
    const float2 ml = tid < splits ? part_ml[(size_t)tid * step + first] : float2{kWinNoMax, 0.f};
    const bool saw = ml.x != kWinNoMax || ml.y != 0.f;  // (a NaN sum counts)
    const float mx = group_max<kWave>(ml.x);
    const float w = __builtin_amdgcn_exp2f((ml.x - mx) * c2);
    const float L = group_sum<kWave>(saw ? w * ml.y : 0.f);
    s_w[tid] = saw ? w : -1.f;
    if (tid == 0) s_l = L;
  }
  __syncthreads();
  f4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int k = 0; k < NB; ++k) {
    const int s = grp + G * k;
    const float w = s < splits ? s_w[s] : -1.f;
    if (w < 0.f) continue;  // (its output was not written)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = fmaf(w, x[k][e], o[e]);
  }
  s_o[grp][d] = o;
  __syncthreads();
  if (grp > 0) return;
#pragma unroll
  for (int k = 1; k < G; ++k) {
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += s_o[k][d][e];
  }
  const float inv = s_l == 0.f ? 0.f : 1.0f / s_l;  // a NaN stays
  const int m = col >> lhpg, hd = (kvh << lhpg) + (col & ((1 << lhpg) - 1));
  *reinterpret_cast<u32x2*>(out + ((size_t)m * (n_kv << lhpg) + hd) * D + 4 * d) =
      u32x2{as_u32(f16x2{(f16)(o[0] * inv), (f16)(o[1] * inv)}), as_u32(f16x2{(f16)(o[2] * inv), (f16)(o[3] * inv)})};
}

// Waves of a workgroup and splits of a call of few columns. A short context is not split, one launch instead of two: up to 512
// tokens in e4m3, 384 in int8 (more arithmetic per code) and 256 in fp16 (twice the bytes) at D 128, twice that at D 64. From
// there to 4096 tiles over all kv heads workgroups of four waves, so that one tile per wave reaches twice the CUs; then of
// eight. At most one workgroup per CU, none with less than a tile per wave. Captured, in us, one token, e4m3 if nothing else:
//   8 x 4 heads of 128   384 tokens unsplit 6.4, split 7.3 | 512: 7.5, 7.2 | int8 384: 7.0, 7.6 | 448: 8.2, 7.6
//                        fp16 256: 7.4, 7.8 | 320: 7.9, 7.9 | 4096: waves 4 7.8, 8 9.1 | 16384: 12.8, 12.2 | 32768: 21.7, 18.8
//   4 x 8 heads of 64    768 tokens unsplit 5.8, split 6.8 | 1024: 6.6, 6.8 | int8 768: 6.8, 7.0 | 1024: 7.8, 7.0
//                        fp16 512: 6.7, 7.1 | 640: 7.4, 7.1 | 16384: waves 4 and 8 7.9 | 32768: 9.4, 9.0
// One or two kv heads of a long cache reach kWinMaxSplits and leave CUs idle: one e4m3 token at 131072 takes 21 us with one kv
// head, 23 with two, 29 with four, 49 with eight.
struct FewPlan {
  int waves, splits;
};
FewPlan few_plan(int M, int n_kv, int D, int max_ctx, int window, int sinks, int cache) {
  const long long tiles = (win_tokens(M, max_ctx, window, sinks) + kFewTile - 1) / kFewTile;
  const int alone = cache == kCacheE4m3 ? 16 : cache == kCacheInt8 ? 12 : 8;
  if (tiles * D <= alone * 128) return {8, 1};
  const int waves = tiles * n_kv < 4096 ? 4 : 8;
  const long long want = max(1LL, min((long long)kWinMaxSplits, 256LL / n_kv));
  const long long per = max((tiles + want - 1) / want, (long long)waves);
  return {waves, (int)((tiles + per - 1) / per)};
}

template <int D, int CACHE, bool DECODE>
void launch(const WindowAttn& w, WinArgs a, const WinDecode& dec, hipStream_t st) {
  a.part_ml = (float2*)(a.part_o + (size_t)w.splits * w.n_kv * kFewCols * (D / 4));
  const FewPlan p = few_plan(w.M, w.n_kv, D, w.max_ctx, w.window, w.sinks, w.cache);
  // K and V that may fill half of the last cache (256 MB) are not kept there for the next call. max_ctx decides, not the
  // position, which the host does not know: 16 e4m3 caches of 8 heads of 128 in turn, max_ctx 131072, take 49.5 us a token at
  // 131072 (from the cache 54.3), 13.6 at 16384 (14.8), and short contexts pay for it: 10.3 at 4096 (9.7), 8.9 at 512 (8.7)
  const long long bytes = win_tokens(w.M, w.max_ctx, w.window, w.sinks) * w.n_kv * 2 * D * (CACHE == kCacheF16 ? 2 : 1);
  const dim3 grid(w.n_kv, w.splits);
  if (p.waves == 4)
    hipLaunchKernelGGL((attn_few_kernel<D, CACHE, 4, false, DECODE>), grid, dim3(4 * kWave), 0, st, a, dec);
  else if (bytes < (128LL << 20))
    hipLaunchKernelGGL((attn_few_kernel<D, CACHE, 8, false, DECODE>), grid, dim3(8 * kWave), 0, st, a, dec);
  else
    hipLaunchKernelGGL((attn_few_kernel<D, CACHE, 8, true, DECODE>), grid, dim3(8 * kWave), 0, st, a, dec);
  if (w.splits > 1)
    hipLaunchKernelGGL(attn_few_join_kernel<D>, dim3(w.n_kv, (unsigned)(w.M << a.lhpg)), dim3(256), 0, st,
                       (const f4*)a.part_o, a.part_ml, a.lhpg, w.n_kv, w.splits, a.c2, (f16*)w.out,
                       DECODE ? a.pos : nullptr, dec.max_pos);
}

template <int D>
void launch_cache(const WindowAttn& w, const WinArgs& a, const WinDecode* dec, hipStream_t st) {
  if (dec && w.cache == kCacheInt8)
    launch<D, kCacheInt8, true>(w, a, *dec, st);
  else if (dec)
    launch<D, kCacheE4m3, true>(w, a, *dec, st);
  else if (w.cache == kCacheF16)
    launch<D, kCacheF16, false>(w, a, {}, st);
  else if (w.cache == kCacheInt8)
    launch<D, kCacheInt8, false>(w, a, {}, st);
  else
    launch<D, kCacheE4m3, false>(w, a, {}, st);
}

}  // namespace

int attention_few_splits(int M, int n_kv, int D, int max_ctx, int window, int sinks, int cache) {
  return few_plan(M, n_kv, D, max_ctx, window, sinks, cache).splits;
}

void launch_attention_few(const WindowAttn& w, const WinArgs& a, const WinDecode* dec, hipStream_t st) {
  if (w.head_dim == 64)
    launch_cache<64>(w, a, dec, st);
  else
    launch_cache<128>(w, a, dec, st);
}

}  // namespace dk
