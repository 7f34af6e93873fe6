// Windowed attention of many columns. A wave has 32 columns, so every column does work at any GQA ratio. A workgroup has CW
// waves of columns, KVS times: group g of KVS takes the blocks of BT tokens with index % KVS == g, so that K / V in LDS once
// serve CW waves, and few columns still fill a workgroup. The tokens are further split over `splits` workgroups in whole
// rounds of KVS blocks; the ends follow *pos, so one captured launch serves every position. The kv head is the fastest grid
// index: with 8 of them each XCD's L2 holds one head's K / V for all its workgroups.
//
// The tokens of a workgroup are those of its rows' windows behind those of the sinks, as one list of 32-token tiles
// ("places"): a round is taken from the list, so a handful of sinks costs one tile, and the window's start is aligned to a
// tile. (As whole rounds of their own 4 sinks cost a round of 128 tokens: 4096 rows under a window of 1024 took 110 us instead
// of 102 in that shape.)
// A round's K / V lie in LDS as fp16, double-buffered. fp16 caches are loaded straight into LDS (buffer loads, spread over the
// products of the round before); codes go to registers in the first half of that round's products and are turned to fp16, with
// their scale, on the way to LDS behind them: CW waves share that work, 1 / CW of a conversion per weight and wave. 4096 rows
// take 149 us over e4m3, 195 over fp16 (149 with one product of V per weight).
//
// Per tile of 32 tokens, on v_mfma_f32_32x32x16_f16:
//   * S^T = K . Q^T: A = the tile's rows of K from LDS, B = the wave's Q columns (registers). Lane (h, r) receives column r,
//     tokens 8 q + 4 h + v: a column's scores, sum and output live in the lane pair (r, r + 32).
//   * the weights (attn_window.hpp), while the next tile's products run;
//   * O^T += V^T . P^T: the score accumulator, rounded to fp16, is the B operand as it is (over fp16 caches a second time, with
//     what the rounding left); V^T comes out of the row-major V tile through the transposing LDS read.
// Masks cost nothing where every column of the wave sees the whole block and every page of the split is mapped (asked once).
// Elsewhere a lane compares its column's bounds to 32 token bits per tile. Scores of tokens that are not seen become -inf
// whatever K holds; their p is an exact 0. Since 0 times NaN or infinity is NaN, V chunks of tokens that do not exist are
// zeroed on the way, and those with such values in rounds that some column does not see whole; the latter are added behind the
// block, value by value, for the columns that see their token.
//
// What bounds it: 4096 rows of e4m3 at 0, 8 x 4 heads of 128, take 148-155 us, 0.89-0.93 PFLOP/s of what they need, against
// 117 at the rate of a large matrix product: the softmax and LDS reads beside the products at the clock that the card keeps up
// under them, and blocks on the diagonal that are computed whole. Over fp16, whose weights meet V twice, they take 195. Under a
// window of 1024 fp16 takes 115 (floor 51, with the second product 77), e4m3 96: two turns of 18 rounds of 64 tokens, 16 of
// them needed, and about 8 us each to start. 100 rows behind 8000 tokens take 31 (floor 11): 78% of the columns are real, four
// rounds in 256 workgroups (17 us), 10 for launch and first loads, 28 MB of partials.
// No gain: tiles that no column of a wave sees left out (the accumulators meet at the branch: 10 to 250 registers spilled);
// blocks of 64 tokens for eight waves (157 us instead of 150); the halves of V's codes in another order for every other row, so
// that their writes to LDS conflict no more (17% of LDS's cycles; 152 us instead of 147).
//
// LDS: rows of 2 D bytes without padding. K chunk q (16 bytes) of row t at q ^ (t & 15) (D 128) or q ^ ((t >> 1) & 7) (D 64),
// V in 64-byte units, unit u of row t at u ^ (t & 3) (D 128) or u ^ ((t >> 1) & 1) (D 64): reads fall in distinct banks.
// The groups of a workgroup meet in LDS, the splits in the workspace and a second launch, both in order.
#include <type_traits>

#include "attn_window.hpp"

namespace dk {
namespace {

template <int D, int CACHE, int CW, int KVS, int BT, bool UP>
__global__ void __launch_bounds__(CW * KVS * kWave, 2) attn_window_kernel(const WinArgs a) {
  constexpr bool F16 = CACHE == kCacheF16;
  constexpr int NTH = CW * KVS * kWave;
  constexpr int RB = 2 * D;                     // bytes of a row in LDS
  constexpr int GB = F16 ? 2 * D : D;           // bytes of a row in the cache
  constexpr int CH = GB / 16;                   // its 16-byte loads
  constexpr int SB = BT * KVS;                  // tokens per round
  constexpr int LPT = SB * CH / NTH;            // 16-byte K (and V) loads per thread per round
  constexpr int RPI = NTH / CH;                 // token rows covered per load index
  constexpr int RPW = kWave / CH;               // rows per load instruction of a wave
  constexpr int NT = BT / 32, DT = D / 32;      // 32-token score tiles per block, 32-dim output tiles
  constexpr int KS = D / 16;                    // k steps of the scores
  static_assert(LPT >= 1 && LPT * RPI == SB && RPI % 16 == 0, "staging covers a round");
  static_assert(F16 || UP, "8-bit pages hold 16 tokens or more");
  constexpr int kTile = SB * RB;                // bytes of one K (or V) buffer
  static_assert((KVS == 1 || KVS * CW * kWave * 16 * DT <= kTile) && 4 % KVS == 0,
                "a merge row set fits a buffer, a wave's rows whole ones");
  __shared__ __align__(16) uint8_t s_k0[kTile], s_k1[kTile], s_v0[kTile], s_v1[kTile];
  __shared__ float s_m[KVS > 1 ? KVS * CW * 32 : 1], s_l[KVS > 1 ? KVS * CW * 32 : 1];
  // tokens of a round (by 32, in the slot of the round's number modulo 3) of which V chunks were taken out (checked)
  __shared__ uint32_t s_bad[3][SB / 32];
  __shared__ int s_holes;  // a page of this split's tokens is not mapped

  // the kv head is the fastest grid index; of the column blocks those with the most tokens come first
  const int kvh = blockIdx.x % a.n_kv, split = blockIdx.y;
  const int cb = (int)gridDim.x / a.n_kv - 1 - blockIdx.x / a.n_kv;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int grp = wave / CW, gw = wave % CW;  // group, and the wave's columns within it
  const int r = lane & 31, h = lane >> 5;
  const int P = 1 << a.log2P;
  const int pos = *a.pos;
  const int n_q = a.n_kv << a.lhpg, cols = a.M << a.lhpg;
  // this lane's column: row m, head hd; columns past the last repeat it
  const int col = (cb * CW + gw) * 32 + r;
  const int cc = min(col, cols - 1);
  const int m = cc >> a.lhpg, hd = (kvh << a.lhpg) + (cc & ((1 << a.lhpg) - 1));
  auto row_of = [&](int c) { return min(c, cols - 1) >> a.lhpg; };
  const Sight mine = sight_of(pos, m, a.window, a.cap);
  const Sight w0 = sight_of(pos, row_of((cb * CW + gw) * 32), a.window, a.cap);       // the wave's first and last rows
  const Sight w1 = sight_of(pos, row_of((cb * CW + gw) * 32 + 31), a.window, a.cap);
  const Sight g0 = sight_of(pos, row_of(cb * CW * 32), a.window, a.cap);              // the workgroup's
  const Sight g1 = sight_of(pos, row_of((cb + 1) * CW * 32 - 1), a.window, a.cap);
  const int ctx = g1.lim + 1;                   // tokens [0, ctx) are read
  // The tokens in the order in which they are taken ("places"): the sinks, in whole tiles of 32, then those from the window's
  // first tile on; place v is token v below ns and v + gap from there.
  const int all = (ctx + 31) / 32, wt = min(g0.lo / 32, all);
  const int ns = a.window > 0 ? 32 * min((min(a.sinks, ctx) + 31) / 32, wt) : 0, gap = 32 * wt - ns;
  auto token = [&](int v) __attribute__((always_inline)) { return v < ns ? v : v + gap; };
  // this split's rounds [r0, r1): the first nr % splits splits have one more
  const unsigned nr = (unsigned)(32 * all - gap + SB - 1) / SB;
  const unsigned per = nr / (unsigned)a.splits, more = nr - per * (unsigned)a.splits;
  const int r0 = (int)(split * per + min((unsigned)split, more)), r1 = r0 + (int)per + ((unsigned)split < more);
  h8 q[KS];
  auto load_q = [&]() __attribute__((always_inline)) {
    const f16* qh = a.q + (size_t)m * a.q_stride + (size_t)hd * D + 8 * h;
#pragma unroll
    for (int s = 0; s < KS; ++s) q[s] = __builtin_bit_cast(h8, *reinterpret_cast<const u32x4*>(qh + 16 * s));
  };

  // Thread's share of a round: 16-byte piece tid % CH of token rows tid / CH + RPI i. Pages are looked up a round ahead of
  // the K / V loads; tokens without a page, or past ctx, read a row that exists; their V is zeroed on the way. UP: a load
  // instruction's rows lie in one page, lane i looks up the page of load i, and the base is a scalar.
  const int sch = tid % CH, sr = tid / CH;
  constexpr int NP = UP ? 1 : LPT;
  const uint64_t page_bytes = (uint64_t)a.n_kv * GB << a.log2P;
  const uint64_t head_bytes = (uint64_t)kvh * GB << a.log2P;
  const uint8_t* kp = a.kc + head_bytes;
  const uint8_t* vp = a.vc + head_bytes;
  // swizzles of row sr (those of row sr + RPI i are the same): K chunk c of a row at c ^ ksw_, V's 64-byte unit u at u ^ vsw_
  const int sksw = D == 128 ? sr & 15 : (sr >> 1) & 7, svsw = D == 128 ? sr & 3 : (sr >> 1) & 1;
  // fp16: lane j of a load fills bytes [16 j, 16 j + 16) of the load's rows in LDS, with the chunk that belongs there
  const uint32_t row_off = UP ? (lane / CH) * GB : 0;
  const uint32_t k_place = row_off + 16 * (F16 ? sch ^ sksw : sch);
  const uint32_t v_place = row_off + (F16 ? 64 * ((sch >> 2) ^ svsw) + 16 * (sch & 3) : 16 * sch);
  int pg[NP];             // pages of the loads
  struct Rows {           // where a round's rows lie (UP: lane i's those of load i), and 8-bit: their scales
    uint64_t base[NP];
    float ks, vs;
  };
  bool whole = true;      // every page with a token of this split that some column can see is mapped; uniform
  auto mapped = [&](int t) __attribute__((always_inline)) { return (unsigned)a.bt[t >> a.log2P] < (unsigned)a.n_pages; };
  auto first_row = [&](int rnd, int i) __attribute__((always_inline)) {  // (a load's rows lie in one tile)
    return token(rnd * SB + (UP ? RPW * wave : sr) + RPI * i);
  };
  auto lookup = [&](int rnd) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NP; ++i) pg[i] = a.bt[min(first_row(rnd, UP ? lane % LPT : i), ctx - 1) >> a.log2P];
  };
  auto locate = [&](int rnd) __attribute__((always_inline)) {  // from the looked-up pages
    Rows w;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int t = first_row(rnd, UP ? lane % LPT : i);
      const uint64_t page = (uint64_t)(uint32_t)((unsigned)pg[i] < (unsigned)a.n_pages ? pg[i] : 0);
      w.base[i] = page * page_bytes + (uint64_t)(uint32_t)(t & (P - 1)) * GB;  // (a page may pass 4 GiB)
      if constexpr (!F16) {
        const size_t block = (((page * a.n_kv + kvh) << a.log2P) + (uint32_t)(t & (P - 1))) >> 4;
        w.ks = a.ks[block];
        w.vs = a.vs[block];
      }
    }
    return w;
  };
  auto rows_of = [&](const Rows& w, int i) __attribute__((always_inline)) -> uint64_t {  // bytes ahead of the rows of load i
    return UP ? (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(w.base[0] >> 32), i) << 32 |
                    (uint32_t)__builtin_amdgcn_readlane((int)w.base[0], i)
              : w.base[UP ? 0 : i];
  };
  // load i of a round: fp16 straight into LDS, codes into registers
  u32x4 kk[F16 ? 1 : LPT], vv[F16 ? 1 : LPT];
  auto fetch = [&](const uint8_t* cache, const Rows& w, int i, uint32_t place, uint8_t* buf, u32x4* reg)
                   __attribute__((always_inline)) {
    typedef __attribute__((address_space(1))) const void* gptr;
    typedef __attribute__((address_space(3))) void* lptr;
    if constexpr (F16) {
      lptr at = (lptr)(buf + (RPI * i + RPW * wave) * RB);
      if constexpr (UP) {
        const __amdgpu_buffer_rsrc_t res =
            __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(cache) + rows_of(w, i), 0, RPW * GB, 0x00020000);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(res, at, 16, (int)place, 0, 0, 0);
      } else {
        __builtin_amdgcn_global_load_lds((gptr)(cache + rows_of(w, i) + place), at, 16, 0, 0);
      }
    } else {
      reg[i] = *reinterpret_cast<const u32x4*>(cache + rows_of(w, i) + place);
    }
  };
  // A round in which some column does not see some token (uniform in the workgroup).
  auto partial = [&](int rnd) __attribute__((always_inline)) {
    const int t0 = rnd * SB + gap, t1 = t0 + SB;
    return rnd * SB < ns || t1 > g0.lim + 1 || (t0 < g1.lo && t1 > a.sinks);
  };
  // A V chunk (8 dims of token t) that must not meet a p of 0 is taken out: one of a token that does not exist, and one with
  // NaN or infinity in a round that not every column sees whole.
  auto checked = [&](u32x4 x, int rnd, int row) __attribute__((always_inline)) -> u32x4 {
    const int t = token(rnd * SB + row);
    const bool ok = t < ctx && (whole || mapped(t));
    const bool bad = ok && has_nonfinite(x);
    if (bad) atomicOr(&s_bad[(unsigned)rnd % 3u][row / 32], 1u << (row % 32));
    return ok && !bad ? x : u32x4{0u, 0u, 0u, 0u};
  };

  // the column's reference maximum (a score), kWinLift less its c2 fold (infinite: far), and this lane's half of its sum
  float ref = kWinNoMax, lift = -kWinNoMax, l = 0.f;
  f32x16 acc[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) acc[t] = f32x16{};

  // LDS addresses: K row r of the group's block (chunk bits apart), and the lane's row of a transposing V read
  const int krow = (grp * BT + r) * RB, ksw = D == 128 ? r & 15 : (r >> 1) & 7;
  const int vt = 4 * h + ((lane & 15) >> 2);               // token (of 8) that the lane addresses
  const int vd = 32 * ((lane >> 4) & 1) + 8 * (lane & 3);  // byte of its 4 dims within the 64-byte unit
  const int vrow = (grp * BT + vt) * RB + vd, vsw = D == 128 ? vt & 3 : (vt >> 1) & 1;

  // bits of tokens [t0, t0 + 32) that this lane's column sees by position
  auto seen_bits = [&](int t0) __attribute__((always_inline)) -> uint32_t {
    auto low = [](int n) -> uint32_t { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1; };
    return low(mine.lim + 1 - t0) & (~low(mine.lo - t0) | low(a.sinks - t0));
  };
  // ---- a block, by tiles of 32 tokens
  f32x16 sc[2];        // scores of a tile and the next
  u32x4 pw[2];         // p in fp16: the B operand of the output's products
  u32x4 pl[2];         // fp16 caches: what pw leaves of p
  constexpr int RA = 4;  // K fragments in flight from LDS
  u32x4 ka[RA + 1];
  h8 va[2][DT];        // V fragments: 16 tokens, in two sets
  float psum[2];       // sums of p over the tile
  // p of scores x, y, the scores e, e + 1 of a tile
  auto weigh = [&](float x, float y, int e, float lift) __attribute__((always_inline)) {
    const float p0 = __builtin_amdgcn_exp2f(fmaf(x, a.c2, lift)), p1 = __builtin_amdgcn_exp2f(fmaf(y, a.c2, lift));
    psum[0] = e == 0 ? p0 : psum[0] + p0;
    psum[1] = e == 0 ? p1 : psum[1] + p1;
    const h2 p = __builtin_convertvector(f2{p0, p1}, h2);
    uint32_t pair = __builtin_bit_cast(uint32_t, p);
    asm volatile("" : "+v"(pair), "+v"(psum[0]), "+v"(psum[1]));  // here, beside the products, not where they are used
    pw[e >> 3][(e & 7) >> 1] = pair;
    if constexpr (F16) {
      const h2 rest = __builtin_convertvector(f2{minus_lo(p0, pair), minus_hi(p1, pair)}, h2);
      uint32_t word = __builtin_bit_cast(uint32_t, rest);
      asm volatile("" : "+v"(word));
      pl[e >> 3][(e & 7) >> 1] = word;
    }
  };
  auto block = [&](int rnd, const uint8_t* kb, const uint8_t* vb, auto send) __attribute__((always_inline)) {
    const int v0 = (rnd * KVS + grp) * BT, t0 = v0 + gap;
    // every token is seen; uniform per wave (a block with sinks counts as one that is not seen whole)
    const bool plain = whole && v0 >= ns && t0 + BT - 1 <= w0.lim && (t0 >= w1.lo || t0 + BT <= a.sinks);
    uint32_t vis[NT];
    if (!plain) {
      asm volatile("");  // stays a branch
#pragma unroll
      for (int c = 0; c < NT; ++c) {
        const int ts = token(v0 + 32 * c);
        vis[c] = (uint32_t)__ballot(ts + r < ctx && (whole || mapped(ts + r))) & seen_bits(ts);
      }
    }
    int kat = krow + ((h ^ ksw) << 4), vat = vrow + (vsw << 6);
    asm volatile("" : "+v"(kat), "+v"(vat));  // (the chunks' places are worked out per block: all of them held would not fit)
    auto read_k = [&](int f) __attribute__((always_inline)) {  // k step f % KS of tile f / KS
      ka[f % (RA + 1)] = *reinterpret_cast<const u32x4*>(kb + f / KS * 32 * RB + (kat ^ (f % KS << 5)));
    };
    auto read_v = [&](int ks) __attribute__((always_inline)) {  // 16 tokens
#pragma unroll
      for (int t = 0; t < DT; ++t) {
        const uint8_t* src = vb + ks * 16 * RB + (vat ^ (t << 6));
        const u32x2 x = read_tr(src), y = read_tr(src + 8 * RB);
        va[ks & 1][t] = __builtin_bit_cast(h8, u32x4{x[0], x[1], y[0], y[1]});
      }
    };
    // scores of tile tt, with after(k) behind product k
    auto scores = [&](int tt, auto after) __attribute__((always_inline)) {
      sc[tt & 1] = f32x16{};
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const int f = tt * KS + k;
        if (k + RA < KS) read_k(f + RA);
        sc[tt & 1] = mfma32x32(__builtin_bit_cast(h8, ka[f % (RA + 1)]), q[k], sc[tt & 1]);
        send(f);
        after(k);
        __builtin_amdgcn_sched_barrier(0);  // in this order
      }
      if (!plain) {
        asm volatile("");
        const uint32_t bits = vis[tt] >> (4 * h);
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (!(bits & (1u << (8 * (i >> 2) + (i & 3))))) sc[tt & 1][i] = -INFINITY;
      }
    };
    auto ahead_k = [&](int tt) __attribute__((always_inline)) {
#pragma unroll
      for (int k = 0; k < (RA < KS ? RA : KS); ++k) read_k(tt * KS + k);
    };
    ahead_k(0);
    scores(0, [](int) {});
    if (NT > 1) ahead_k(1);
#pragma unroll
    for (int tt = 0; tt < NT; ++tt) {
      const f32x16& s = sc[tt & 1];
      read_v(2 * tt);
      if (tt + 1 < NT) {
        scores(tt + 1, [&](int k) __attribute__((always_inline)) {
          constexpr int NE = 16 / KS;
#pragma unroll
          for (int e = 0; e < NE; e += 2) weigh(s[NE * k + e], s[NE * k + e + 1], NE * k + e, lift);
        });
      } else {
#pragma unroll
        for (int e = 0; e < 16; e += 2) weigh(s[e], s[e + 1], e, lift);
      }
      float sum = psum[0] + psum[1];
      if (__any(!(sum <= kWinMost))) {  // the reference moves to this tile's maximum where that is higher
        asm volatile("");
        float mx = s[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
        mx = fmaxf(ref, fmaxf(mx, __shfl_xor(mx, 32, kWave)));
        // (a column decides by itself: its result does not depend on what else shares its wave)
        const int over = !(sum <= kWinMost);
        mx = over | __shfl_xor(over, 32, kWave) ? mx : ref;
        const float alpha = __builtin_amdgcn_exp2f((ref - mx) * a.c2);  // 1 for a column that stays
        if (mx != ref) lift = fabsf(mx * a.c2) > kWinFar ? INFINITY : kWinLift - mx * a.c2;
        ref = mx;
        const float off = lift == INFINITY ? ref : 0.f, up = lift == INFINITY ? kWinLift : lift;
        l *= alpha;
#pragma unroll
        for (int t = 0; t < DT; ++t) {
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[t][i] *= alpha;
        }
#pragma unroll
        for (int e = 0; e < 16; e += 2) weigh(s[e] - off, s[e + 1] - off, e, up);
        sum = psum[0] + psum[1];
      }
      l += sum;
      if (tt + 2 < NT) ahead_k(tt + 2);
      read_v(2 * tt + 1);
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
        for (int t = 0; t < DT; ++t) acc[t] = mfma32x32(va[ks][t], __builtin_bit_cast(h8, pw[ks]), acc[t]);
        if constexpr (F16) {
#pragma unroll
          for (int t = 0; t < DT; ++t) acc[t] = mfma32x32(va[ks][t], __builtin_bit_cast(h8, pl[ks]), acc[t]);
        }
      }
    }
    if (!whole || partial(rnd)) {  // uniform in the workgroup
      // the chunks that were taken out, from the cache, for the columns that see their token; its weight once more from q and
      // k, as in the loop and so the same to the last bit
      for (int w = 0; w < BT / 32; ++w) {
        uint32_t bad = __builtin_amdgcn_readfirstlane(s_bad[(unsigned)rnd % 3u][grp * (BT / 32) + w]);
        if (bad == 0) continue;
        const int ts = token(v0 + 32 * w);
        const uint32_t seen = seen_bits(ts);
        f32x16 st = {};
#pragma unroll
        for (int k = 0; k < KS; ++k)
          st = mfma32x32(__builtin_bit_cast(h8, *reinterpret_cast<const u32x4*>(kb + w * 32 * RB + (kat ^ (k << 5)))), q[k],
                         st);
        for (; bad != 0; bad &= bad - 1) {
          const int i = __builtin_ctz(bad), t = ts + i;            // a token in this set is inside the context
          const int page = a.bt[t >> a.log2P];
          if ((unsigned)page >= (unsigned)a.n_pages) continue;     // (nobody sees it)
          const size_t at = (((size_t)page * a.n_kv + kvh) << a.log2P) + (t & (P - 1));
          float dot = 0.f;  // in element 4 (i / 8) + i % 4 of the half i / 4 % 2
#pragma unroll
          for (int e = 0; e < 16; ++e) dot = e == 4 * (i >> 3) + (i & 3) ? st[e] : dot;
          dot = __shfl(dot, r + 32 * ((i >> 2) & 1), kWave);
          const float p = __builtin_amdgcn_exp2f(lift == INFINITY ? fmaf(dot - ref, a.c2, kWinLift) : fmaf(dot, a.c2, lift));
          const bool see = (seen >> i) & 1;
#pragma unroll
          for (int c = 0; c < D / 8; ++c) {
            u32x4 x;
            if constexpr (F16)
              x = *reinterpret_cast<const u32x4*>(a.vc + at * GB + 16 * c);
            else
              x = kv8_decode8<CACHE>(*reinterpret_cast<const u32x2*>(a.vc + at * GB + 8 * c), a.vs[at >> 4]);
            if (!has_nonfinite(x) || !see) continue;
            const f16x2 lo = as_f16x2(h ? x[2] : x[0]), hi = as_f16x2(h ? x[3] : x[1]);
            const float f[4] = {(float)lo[0], (float)lo[1], (float)hi[0], (float)hi[1]};
#pragma unroll
            for (int v = 0; v < 4; ++v) acc[c / 4][4 * (c % 4) + v] = fmaf(p, f[v], acc[c / 4][4 * (c % 4) + v]);
          }
        }
      }
    }
  };

  // Round rnd, in buffer B: the loads of round rnd + 1 go out, into the other buffer (every wave finished reading it before
  // the last barrier).
  Rows rows;
  auto start = [&](int j, uint8_t* k, uint8_t* v) __attribute__((always_inline)) {  // load j of K's and V's 2 LPT
    if (j < LPT)
      fetch(kp, rows, j, k_place, k, kk);
    else
      fetch(vp, rows, j - LPT, v_place, v, vv);
  };
  auto finish = [&](int rnd, uint8_t* k, uint8_t* v) __attribute__((always_inline)) {
    const bool check = rnd < r1 && (!whole || partial(rnd));  // uniform
    if constexpr (F16) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      if (check) {
        asm volatile("");  // stays a branch
#pragma unroll
        for (int i = 0; i < LPT; ++i) {
          const int row = sr + RPI * i;
          u32x4* x = reinterpret_cast<u32x4*>(v + row * RB + 16 * sch);
          *x = checked(*x, rnd, row);
        }
      }
    } else {
      // codes to fp16, 16 of one row: two K chunks, half a V unit
#pragma unroll
      for (int i = 0; i < LPT; ++i) {
        const float s = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, rows.ks), i));
        uint8_t* at = k + (sr + RPI * i) * RB;
#pragma unroll
        for (int e = 0; e < 2; ++e)
          *reinterpret_cast<u32x4*>(at + (((2 * sch + e) ^ sksw) << 4)) =
              kv8_decode8<CACHE>(u32x2{kk[i][2 * e], kk[i][2 * e + 1]}, s);
      }
#pragma unroll
      for (int i = 0; i < LPT; ++i) {
        const float s = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, rows.vs), i));
        u32x4* at = reinterpret_cast<u32x4*>(v + (sr + RPI * i) * RB + (((sch >> 1) ^ svsw) << 6) + 32 * (sch & 1));
        u32x4 x[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) x[e] = kv8_decode8<CACHE>(u32x2{vv[i][2 * e], vv[i][2 * e + 1]}, s);
        if (check) {
          asm volatile("");  // stays a branch
          for (int e = 0; e < 2; ++e) x[e] = checked(x[e], rnd, sr + RPI * i);
        }
        at[0] = x[0];
        at[1] = x[1];
      }
    }
    __syncthreads();
  };
  auto round = [&](int rnd, auto B) __attribute__((always_inline)) {
    constexpr bool odd = decltype(B)::value;
    uint8_t *kb = odd ? s_k1 : s_k0, *vb = odd ? s_v1 : s_v0, *kn = odd ? s_k0 : s_k1, *vn = odd ? s_v0 : s_v1;
    rows = locate(rnd + 1);  // past the end: rows that are never computed on
    // the slot of the round before this one, for the one after the next: nobody reads or writes it now
    if (tid < SB / 32) s_bad[(unsigned)(rnd + 2) % 3u][tid] = 0u;
    // spread over the products: issued in a row they hold a wave up while the other waves' are taken in
    constexpr int NF = KS * NT, NL = 2 * LPT;
    block(rnd, kb, vb, [&](int f) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < NL; ++j)
        if (f == j * (F16 ? NF : NF / 2) / NL) start(j, kn, vn);
      if (f == NF - 1) lookup(rnd + 2);
    });
    pf_fence();
    finish(rnd + 1, kn, vn);
  };
  if (r0 < r1) {  // uniform
    lookup(r0);
    if (tid < 3 * (SB / 32)) s_bad[tid / (SB / 32)][tid % (SB / 32)] = 0u;
    if (tid == 0) s_holes = 0;
    rows = locate(r0);
#pragma unroll
    for (int j = 0; j < 2 * LPT; ++j) start(j, s_k0, s_v0);
    pf_fence();  // (loads return in order: what is wanted later goes out later)
    lookup(r0 + 1);
    load_q();
    pf_fence();
    auto scan = [&](int t0, int t1) __attribute__((always_inline)) {  // tokens [t0, t1)
      for (int p = (t0 >> a.log2P) + tid; p <= (t1 - 1) >> a.log2P; p += NTH)
        whole = whole && (unsigned)a.bt[p] < (unsigned)a.n_pages;
    };
    // (pages between the sinks and the window may be gone; sinks that reach past 32 wt are in the window's places)
    if (r0 * SB < ns) scan(r0 * SB, min(min(r1 * SB, ns), min(a.sinks, ctx)));
    const int from = a.sinks > 32 * wt ? 0 : min(g0.lo, ctx);
    if (r1 * SB > ns) scan(max(max(r0 * SB, ns) + gap, from), min(r1 * SB + gap, ctx));
    __syncthreads();  // (s_bad, s_holes)
    if (!whole) s_holes = 1;
    __syncthreads();
    whole = __builtin_amdgcn_readfirstlane(s_holes) == 0;
    finish(r0, s_k0, s_v0);
    for (int rnd = r0; rnd < r1; rnd += 2) {
      round(rnd, std::false_type{});
      if (rnd + 1 < r1) round(rnd + 1, std::true_type{});
    }
  }
  l += __shfl_xor(l, 32, kWave);
  // ---- output: acc[t][4 q + v] = O[column r][dim 32 t + 8 q + 4 h + v], row 4 t + q of a wave's 4 DT rows of float4. The
  // groups leave theirs in LDS (over the K / V buffers, which every wave has finished reading at the last barrier), with
  // maximum and sum per column; then each takes 1 / KVS of the rows, over all groups in order.
  const int waves = (cols + 31) >> 5;
  const size_t part = ((size_t)split * a.n_kv + kvh) * waves + (cb * CW + gw);
  if (a.splits > 1 && r0 >= r1) {  // a split without tokens: the join reads no accumulator of it
    if (grp == 0 && h == 0 && col < cols) a.part_ml[part * 32 + r] = float2{kWinNoMax, 0.f};
    return;
  }
  constexpr int kRows = 4 * DT / KVS;
  float mx = ref, L = l, w[KVS];
  auto own_row = [&](int i) __attribute__((always_inline)) {
    const f32x16& x = acc[i / 4];
    return float4{x[4 * (i % 4)], x[4 * (i % 4) + 1], x[4 * (i % 4) + 2], x[4 * (i % 4) + 3]};
  };
  auto merge_row = [&](int quarter, int i, int g) __attribute__((always_inline)) {  // row DT quarter + i of group g
    uint8_t* buf = quarter == 0 ? s_k0 : quarter == 1 ? s_k1 : quarter == 2 ? s_v0 : s_v1;
    return reinterpret_cast<float4*>(buf) + ((i * KVS + g) * CW + gw) * kWave + lane;
  };
  if constexpr (KVS > 1) {
    if (h == 0) {
      s_m[(grp * CW + gw) * 32 + r] = ref;
      s_l[(grp * CW + gw) * 32 + r] = l;
    }
#pragma unroll
    for (int i = 0; i < 4 * DT; ++i) *merge_row(i / DT, i % DT, grp) = own_row(i);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < KVS; ++k) mx = fmaxf(mx, s_m[(k * CW + gw) * 32 + r]);
    L = 0.f;
#pragma unroll
    for (int k = 0; k < KVS; ++k) {
      // a group that saw no token weighs 0 beside one that did
      w[k] = __builtin_amdgcn_exp2f((s_m[(k * CW + gw) * 32 + r] - mx) * a.c2);
      L = fmaf(w[k], s_l[(k * CW + gw) * 32 + r], L);
    }
  }
  if (col >= cols) return;
  if (a.splits > 1 && grp == 0 && h == 0) a.part_ml[part * 32 + r] = float2{mx, L};
  const float inv = L == 0.f ? 0.f : 1.0f / L;  // a NaN stays
  f16* out = a.out + ((size_t)m * n_q + hd) * D + 4 * h;
  float4* dst = a.part_o + part * (DT * 4 * kWave);  // uniform per wave
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    float4 o;
    if constexpr (KVS > 1) {
      o = float4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < KVS; ++k) {
        const float4 x = *merge_row(grp * (4 / KVS) + i / DT, i % DT, k);
        o = float4{fmaf(w[k], x.x, o.x), fmaf(w[k], x.y, o.y), fmaf(w[k], x.z, o.z), fmaf(w[k], x.w, o.w)};
      }
    } else {
      o = own_row(i);
    }
    const int row = grp * kRows + i;
    if (a.splits == 1)
      *reinterpret_cast<u32x2*>(out + 32 * (row >> 2) + 8 * (row & 3)) =
          u32x2{as_u32(f16x2{(f16)(o.x * inv), (f16)(o.y * inv)}), as_u32(f16x2{(f16)(o.z * inv), (f16)(o.w * inv)})};
    else
      store_through16(dst, (uint32_t)((row * kWave + lane) * 16), __builtin_bit_cast(u32x4, f4{o.x, o.y, o.z, o.w}));
  }
}

// Joins the splits of a column in split order. A workgroup takes kRows of the D / 8 accumulator rows of one wave's 32
// columns, a thread one float4 of it (4 dims of a column). The first kBatch partials are loaded ahead of the maxima and
// sums, so that one memory round trip covers both; the accumulator of a split that saw no token was not written and is
// dropped.
constexpr int kWinJoinRows = 4;
template <int D>
__global__ void __launch_bounds__(kWinJoinRows * kWave)
attn_window_join_kernel(const float4* __restrict__ part_o, const float2* __restrict__ part_ml, int cols, int lhpg, int n_kv,
                        int splits, float c2, f16* __restrict__ out) {
  constexpr int kRows = kWinJoinRows, kBatch = 8, kGroups = 2 * kRows;  // kGroups threads share a column's maxima and sums
  __shared__ float s_w[kWinMaxSplits][32];          // a split's weight in a column, -1 where it saw no token
  __shared__ float s_l[32];
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 31, h = lane >> 5;
  const int kvh = blockIdx.x, row = (blockIdx.y % (D / 8 / kRows)) * kRows + (tid >> 6);
  const int waves = gridDim.y / (D / 8 / kRows), cw = blockIdx.y / (D / 8 / kRows), col = cw * 32 + r;
  const bool live = col < cols;
  const size_t wave = (size_t)kvh * waves + cw, wstep = (size_t)n_kv * waves;  // per split
  const float4* src = part_o + (wave * (D / 8) + row) * kWave + lane;
  const size_t step = wstep * (D / 8) * kWave;
  float4 p[kBatch];
  auto load = [&](int s0) {
#pragma unroll
    for (int k = 0; k < kBatch; ++k) p[k] = src[(size_t)min(s0 + k, splits - 1) * step];
  };
  if (live) load(0);
  // weights: thread (column c, g) takes splits g, g + 8, ...
  {
    const int c = tid / kGroups, g = tid % kGroups;
    constexpr int kMl = kWinMaxSplits / kGroups;
    float2 ml[kMl];
    float mx = kWinNoMax;
#pragma unroll
    for (int j = 0; j < kMl; ++j) {
      const int s = g + kGroups * j;
      ml[j] = s < splits ? part_ml[((size_t)s * wstep + wave) * 32 + c] : float2{kWinNoMax, 0.f};
      mx = fmaxf(mx, ml[j].x);
    }
    mx = group_max<kGroups>(mx);
    float L = 0.f;
#pragma unroll
    for (int j = 0; j < kMl; ++j) {
      const int s = g + kGroups * j;
      const bool saw = ml[j].x != kWinNoMax || ml[j].y != 0.f;  // (a NaN sum counts)
      const float w = __builtin_amdgcn_exp2f((ml[j].x - mx) * c2);
      L = saw ? fmaf(w, ml[j].y, L) : L;
      if (s < splits) s_w[s][c] = saw ? w : -1.f;
    }
    L = group_sum<kGroups>(L);
    if (g == 0) s_l[c] = L;
  }
  __syncthreads();
  if (!live) return;
  float4 o = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < splits; s0 += kBatch) {
    if (s0 > 0) load(s0);
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const float w = s0 + k < splits ? s_w[s0 + k][r] : -1.f;
      if (w < 0.f) continue;
      o.x = fmaf(w, p[k].x, o.x);
      o.y = fmaf(w, p[k].y, o.y);
      o.z = fmaf(w, p[k].z, o.z);
      o.w = fmaf(w, p[k].w, o.w);
    }
  }
  const float L = s_l[r], inv = L == 0.f ? 0.f : 1.0f / L;  // a NaN stays
  const int m = col >> lhpg, hd = (kvh << lhpg) + (col & ((1 << lhpg) - 1));
  f16* dst = out + ((size_t)m * (n_kv << lhpg) + hd) * D + 32 * (row >> 2) + 8 * (row & 3) + 4 * h;
  *reinterpret_cast<u32x2*>(dst) =
      u32x2{as_u32(f16x2{(f16)(o.x * inv), (f16)(o.y * inv)}), as_u32(f16x2{(f16)(o.z * inv), (f16)(o.w * inv)})};
}

// Shape of the workgroup (CW, KVS, BT), and the splits that it can use: at most one workgroup per CU, of equal length.
struct WinShape {
  int cw, kvs, bt, splits;
};
constexpr WinShape kWinShapes[4] = {{2, 4, 32, 1}, {4, 1, 64, 1}, {4, 2, 64, 1}, {8, 1, 128, 1}};

// The shape with the least estimated time: a fixed part, a round's time times the rounds of the longest workgroup, or of all
// of them over the CUs with what it takes to start each. Fitted to the times of all four shapes in 75 cases (8 to 4096 rows
// behind 0 to 30000 tokens, windows of 256 to 2048 and none, five head layouts), before weights met fp16 caches' V twice; as it
// stands the choice is 0.6% above the best of the four in the geometric mean for e4m3 and 0.9% for fp16, 7% at worst. In us,
// D 128 (e4m3, 8 x 4 heads):
//                              (2,4,32) (4,1,64) (4,2,64) (8,1,128)
//   512 rows at 0                15.3     19.2     19.3     20.5
//   64 behind 4000               18.4     19.3     19.7     23.7
//   1024 at 0                    30.2     32.1     28.1     33.5
//   256 behind 8000              62.9     59.5     52.0     49.1
//   4096 at 0                   262      171      185      150
//   4096, window 1024           172       97      121      103
WinShape win_shape(int M, int n_q, int n_kv, int D, int max_ctx, int window, int sinks) {
  const double rounds[2][4] = {{0.96, 1.0, 1.42, 2.39}, {1.62, 1.49, 2.52, 4.3}};  // us of a round, D 64 and 128
  const double paired[2] = {1.24, 2.32};                                            // (4,1,64): of two workgroups of a CU
  const double fixed[4] = {7.89, 8.49, 8.88, 10.19}, join = 2.9, start = 7.68;
  const int hpg = n_q / n_kv, d = D == 128;
  const long long waves = ((long long)M * hpg + 31) / 32;
  WinShape best = {};
  double least = 0;
  for (int i = 0; i < 4; ++i) {
    WinShape s = kWinShapes[i];
    const long long blocks = (waves + s.cw - 1) / s.cw * n_kv, round = s.bt * s.kvs;
    const long long span = win_tokens(min((long long)M, 32LL * s.cw / hpg), max_ctx, window, sinks);
    const long long all = (span + round - 1) / round, want = max(1LL, min((long long)kWinMaxSplits, 256 / blocks));
    const long long per = (all + want - 1) / want;
    s.splits = (int)((all + per - 1) / per);
    // tokens of a row in the mean: min(p, span) over the positions p of the rows
    const double lo = max(0, max_ctx - M), hi = max_ctx, w = (double)span;
    const double mean = w >= hi ? (lo + hi) / 2 : w <= lo ? w : ((w * w - lo * lo) / 2 + w * (hi - w)) / (hi - lo);
    const double groups = (double)blocks * s.splits;
    const bool two = i == 1 && groups > 256;
    const double us = two ? paired[d] : rounds[d][i];
    double turns = groups / (two ? 512 : 256);
    if (w < 1.3 * mean) turns = ceil(turns);  // workgroups alike end together
    const double time = fixed[i] + (s.splits > 1 ? join : 0) +
                        max(us * per, turns * (us * (mean / round / s.splits + 0.5) + start) - start);
    if (i == 0 || time < least) {
      least = time;
      best = s;
    }
  }
  return best;
}

}  // namespace

// (The query does not know the page: where a cache of small pages keeps few columns from their kernel, the other one runs that
// many splits.)
int attention_window_splits(int M, int n_q, int n_kv, int D, int max_ctx, int window, int sinks, int cache) {
  return win_few(M, n_q, n_kv, 4) ? attention_few_splits(M, n_kv, D, max_ctx, window, sinks, cache)
                                  : win_shape(M, n_q, n_kv, D, max_ctx, window, sinks).splits;
}
size_t attention_window_part_bytes(int M, int n_q, int n_kv, int head_dim) {
  return (size_t)n_kv * (((size_t)M * (n_q / n_kv) + 31) / 32) * 32 * (head_dim + 2) * sizeof(float);
}

namespace {

template <int D, int CACHE, int CW, int KVS, int BT>
void launch_shape(const WinArgs& a, long long cols, hipStream_t st) {
  const dim3 grid((unsigned)(a.n_kv * ((cols + 32 * CW - 1) / (32 * CW))), a.splits), block(CW * KVS * kWave);
  if (CACHE != kCacheF16 || (1 << a.log2P) >= 512 / D)
    hipLaunchKernelGGL((attn_window_kernel<D, CACHE, CW, KVS, BT, true>), grid, block, 0, st, a);
  else if constexpr (CACHE == kCacheF16)
    hipLaunchKernelGGL((attn_window_kernel<D, CACHE, CW, KVS, BT, false>), grid, block, 0, st, a);
}

template <int D>
WinArgs window_args(const WindowAttn& w) {
  int lhpg = 0;
  while ((w.n_kv << lhpg) < w.n_q) ++lhpg;
  const long long waves = (((long long)w.M << lhpg) + 31) / 32;
  float4* part_o = (float4*)w.ws;
  return {(const f16*)w.q, w.q_stride, w.pos, w.bt, (const uint8_t*)w.kc, (const uint8_t*)w.vc, w.ks, w.vs, w.n_pages,
                  w.n_bt, w.log2P, w.n_kv, lhpg, w.M, (int)min((long long)w.max_ctx, (long long)w.n_bt << w.log2P), w.window,
                  w.sinks, w.splits, (float)(1.4426950408889634 / sqrt((double)D)), (f16*)w.out, part_o,
                  (float2*)(part_o + (size_t)w.splits * w.n_kv * waves * 8 * D)};
}

template <int D, int CACHE>
void launch(const WindowAttn& w, const WinArgs& a, hipStream_t st) {
  const long long cols = (long long)w.M << a.lhpg, waves = (cols + 31) / 32;
  const WinShape s = win_shape(w.M, w.n_q, w.n_kv, D, w.max_ctx, w.window, w.sinks);
  if (s.cw == 2)
    launch_shape<D, CACHE, 2, 4, 32>(a, cols, st);
  else if (s.cw == 8)
    launch_shape<D, CACHE, 8, 1, 128>(a, cols, st);
  else if (s.kvs == 1)
    launch_shape<D, CACHE, 4, 1, 64>(a, cols, st);
  else
    launch_shape<D, CACHE, 4, 2, 64>(a, cols, st);
  if (w.splits > 1)
    hipLaunchKernelGGL(attn_window_join_kernel<D>, dim3(w.n_kv, (unsigned)(waves * (D / 8 / kWinJoinRows))),
                       dim3(kWinJoinRows * kWave), 0, st, a.part_o, a.part_ml, (int)cols, a.lhpg, w.n_kv, w.splits, a.c2,
                       (f16*)w.out);
}

template <int D>
void launch_cache(const WindowAttn& w, const WinDecode* dec, hipStream_t st) {
  const WinArgs a = window_args<D>(w);
  if (dec || win_few(w.M, w.n_q, w.n_kv, w.log2P))
    launch_attention_few(w, a, dec, st);
  else if (w.cache == kCacheF16)
    launch<D, kCacheF16>(w, a, st);
  else if (w.cache == kCacheInt8)
    launch<D, kCacheInt8>(w, a, st);
  else
    launch<D, kCacheE4m3>(w, a, st);
}

}  // namespace

void launch_attention_window(const WindowAttn& a, hipStream_t st) {
  if (a.head_dim == 64)
    launch_cache<64>(a, nullptr, st);
  else
    launch_cache<128>(a, nullptr, st);
}

void launch_attention_kv8_decode(const WindowAttn& a, const float* cos_t, const float* sin_t, int max_pos, hipStream_t st) {
  const WinDecode dec{cos_t, sin_t, max_pos};
  if (a.head_dim == 64)
    launch_cache<64>(a, &dec, st);
  else
    launch_cache<128>(a, &dec, st);
}

}  // namespace dk
