// Attention of the nodes of a drafted token tree over the paged cache on gfx950: node i (row i of q) attends the committed
// tokens [0, *pos) and the nodes (tokens *pos + j) whose bit is set in its mask row.
//
// A column is a (node, query head) pair of one kv head; a wave has 32 columns, so every column does work at any GQA ratio.
// A workgroup has CW waves of columns, KVS times: group g of KVS takes the token blocks b (of BT tokens) with b % KVS == g,
// so K / V in LDS once serve CW waves, and few columns still fill a workgroup. The context is further split over `splits`
// workgroups in whole rounds of KVS blocks; the ends follow *pos, so one captured launch serves every position. The kv head
// is the fastest grid index: with 8 of them each XCD's L2 holds one head's K / V for all its workgroups, and its partials
// for the join.
// K / V go from the cache straight into LDS (16-byte loads), double-buffered: a round's loads go out between the products of
// the round before it, spread, since a wave that issues them in a row waits for the other waves' to be taken in (250 nodes at
// 32768 tokens: 155.9 -> 154.5 us). As buffer loads, whose base is a scalar where a load's rows lie in one page: behind
// global loads to LDS the compiler waits for every LDS read in flight instead of the one it needs (159.6 -> 156.7).
//
// Per tile of 32 tokens, on v_mfma_f32_32x32x16_f16:
//   * S^T = K . Q^T: A = the tile's rows of K from LDS, B = the wave's Q columns (registers). Lane (h, r) receives column r,
//     tokens 8 q + 4 h + v: a column's scores, sum and output live in the lane pair (r, r + 32).
//   * p = 2^(c2 (s - ref) + kTreeLift), c2 = log2(e) / sqrt(D), as c2 s + lift: one multiply-add, while the next tile's
//     products run. The reference is a maximum of scores seen so far, not the running one: it moves to the tile's maximum
//     where a sum of p in the column's two lanes passes kTreeMost, so that p fits fp16 and no maximum is taken otherwise;
//     what fp16 cannot hold of a small p is 2^-32 of p at the reference. (With a maximum per block of 64 tokens ahead of its
//     weights 156.7 -> 153.3 us.) lift holds c2 ref to half a step of fp32. From kTreeFar on that would be more than p's own
//     half step in fp16 (and at 2^26 p could overflow at the reference): there lift is infinite, every tile's first weights
//     overflow, and the second ones are taken from s - ref, exact at the reference.
//   * O^T += V^T . P^T: the score accumulator, rounded to fp16 to nearest, is the B operand as it is; V^T comes out of the
//     row-major V tile through the transposing LDS read. One fp16 part of p instead of two: its 2^-11, unbiased and beside
//     an output that is rounded to fp16 itself, against a half more of the products. The sum of the weights keeps fp32.
//
// Masks cost nothing where every column of the wave sees the whole block: all before *pos, all mapped, which a workgroup asks
// once for its split (per block 151.8 us instead of 148.0). In the others a lane holds its column's 64 token bits: mapped
// tokens inside the context, and for tokens from *pos on the node bits of the mask row, shifted to the block. Scores of
// tokens that are not seen become -inf whatever K holds; their p is an exact 0.
// Since 0 times NaN or infinity is NaN, check_v zeroes in LDS the V chunks of tokens that do not exist, and those with such
// values in blocks that reach *pos; the latter are added at the end, value by value, for the columns that see their token.
//
// What bounds it (250 nodes at 32768 tokens, 8 x 4 heads of 128: 140-146 us against 114 at the rate of a large matrix product,
// 0.93-0.97 PFLOP/s): the work beside the products, at the 2.0 GHz that the card keeps up under them. Per product a wave
// issues 4 instructions of its softmax, 1.5 LDS reads and its share of the addresses; a loop of nothing but that, two waves
// per SIMD, runs a product and those in 45 cycles, the product alone in 33. With blocks of 64 tokens, 156 us: without the
// exponentials it takes 139, without reading V 142, without both 119 and without loads too 100; the products' own time is
// 62. Barriers and waits taken out changed nothing, 5% fewer cycles save 2% of the time. 64 columns per wave would halve
// the reads, but then scores lie in accumulation registers, which the softmax cannot use.
// 64 nodes at 16001 take 30-32 (floor 14; traced 26.5 and 6 for the join), of which about 18 are this and the rest launch,
// first loads and 17 MB of partials.
// Small ones are launch, a chain of dependent loads (position, page, K / V: 3 us to the first product), partials and the
// join: 26 nodes at 4096 16, 5 at 300, unsplit, 6.7.
// No gain: two halves of the workgroup half a block apart, so that one's softmax meets the other's products; a block's
// weights behind the next one's scores; wave priorities; 168 registers for three waves per SIMD; sums of p by dot products;
// the first pages looked up ahead of the position; the first two rounds' loads sent together.
//
// LDS: rows of 2 D bytes without padding. K chunk q (16 bytes) of row t at q ^ (t & 15) (D 128) or q ^ ((t >> 1) & 7) (D 64),
// V in 64-byte units, unit u of row t at u ^ (t & 3) (D 128) or u ^ ((t >> 1) & 1) (D 64): reads fall in distinct banks
// (the lane that loads a chunk picks the one that belongs at its place). The groups of a workgroup meet in LDS, the splits
// in the workspace and a second launch, both in order.
#include <limits.h>

#include <type_traits>

#include "common.hpp"
#include "launch.hpp"
#include "attn_common.hpp"

namespace dk {
namespace {

// Reference maximum of a column that has seen no token: a finite stand-in for -infinity (no -inf - (-inf)).
constexpr float kTreeNoMax = -1e30f;
constexpr float kTreeLift = 7.0f;     // p's exponent at the reference maximum
constexpr float kTreeMost = 32768.f;  // the reference moves where a lane's sum of p over its part of a tile passes this
constexpr float kTreeFar = 4096.f;    // a reference further from 0 than this (log2 units) is taken off the score itself

constexpr int kTreeMaxSplits = 64;

struct TreeArgs {
  const f16* q;
  long long q_stride;
  const int64_t* mask;
  const int32_t* pos;
  const int32_t* bt;
  const f16* kc;
  const f16* vc;
  int n_pages, log2P, n_kv, lhpg, M, cap;  // cap: tokens at and past it do not exist
  int splits;
  float c2;  // log2(e) / sqrt(D)
  f16* out;  // [M, n_q D]
  float4* part_o;   // [splits][n_kv][column waves][D / 8][64 lanes]: the accumulators as the lanes hold them
  float2* part_ml;  // [splits][n_kv][column waves][32]: reference maximum, sum
};

// Tokens that exist: [0, ctx).
__device__ __forceinline__ int tree_context(long long pos, int M, int cap) {
  return pos < 0 ? 0 : (int)min(pos + M, (long long)cap);
}

// 16 bytes with a half that is no finite number.
__device__ __forceinline__ bool has_nonfinite(u32x4 v) {
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    bad = bad || (v[i] & 0x7C00u) == 0x7C00u || (v[i] & 0x7C000000u) == 0x7C000000u;
  return bad;
}

template <int D, int CW, int KVS, int BT, bool UP>
__global__ void __launch_bounds__(CW * KVS * kWave, 2)
attn_tree_kernel(const TreeArgs a) {
  constexpr int NTH = CW * KVS * kWave;      // threads
  constexpr int CH = D / 8;                  // 16-byte chunks per K / V row
  constexpr int RB = 2 * D;                  // bytes per row
  constexpr int SB = BT * KVS;               // tokens per round (one block per group)
  constexpr int LPT = SB * CH / NTH;         // 16-byte K (and V) loads per thread per round
  constexpr int RPI = NTH / CH;              // token rows covered per load index
  constexpr int NT = BT / 32, DT = D / 32;   // 32-token score tiles per block, 32-dim output tiles
  constexpr int KS = D / 16;                 // k steps of the scores
  static_assert(LPT * RPI == SB && RPI % 16 == 0, "staging covers a round");
  constexpr int kTile = SB * RB;             // bytes of one K (or V) buffer
  // K and V buffers as arrays of their own: the compiler then knows that the loads which fill one in flight touch no other.
  // In the end the groups' accumulators, DT of their 4 DT rows in each.
  static_assert(KVS * CW * kWave * 16 * DT <= kTile && 4 % KVS == 0, "a merge row set fits a buffer, a wave's rows whole ones");
  __shared__ __align__(16) uint8_t s_k0[kTile], s_k1[kTile], s_v0[kTile], s_v1[kTile];
  __shared__ float s_m[KVS > 1 ? KVS * CW * 32 : 1], s_l[KVS > 1 ? KVS * CW * 32 : 1];
  // by 32 tokens from those of *pos on: the tokens that have V chunks which check_v took out
  constexpr int kBadWords = kTreeMaxNodes / 32 + 1;
  __shared__ uint32_t s_bad[kBadWords];
  __shared__ int s_holes;  // a page of this split's tokens is not mapped

  const int kvh = blockIdx.x, cb = blockIdx.y, split = blockIdx.z;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int grp = wave / CW, gw = wave % CW;  // group, and the wave's columns within it
  const int r = lane & 31, h = lane >> 5;
  const int P = 1 << a.log2P;
  const long long pos = *a.pos;
  const int ctx = tree_context(pos, a.M, a.cap);
  const int tail = pos < ctx ? (int)(pos / 32) : INT_MAX / 2;  // the first 32 tokens with some that not every column sees
  // this split's rounds [r0, r1): the first nr % splits splits have one more
  const unsigned nr = (ctx + SB - 1u) / SB, per = nr / (unsigned)a.splits, more = nr - per * (unsigned)a.splits;
  const int r0 = (int)(split * per + min((unsigned)split, more)), r1 = r0 + (int)per + ((unsigned)split < more);
  const int n_q = a.n_kv << a.lhpg, cols = a.M << a.lhpg;
  // this lane's column: node m, head hd; columns past the last repeat it
  const int col = (cb * CW + gw) * 32 + r;
  const int cc = min(col, cols - 1);
  const int m = cc >> a.lhpg, hd = (kvh << a.lhpg) + (cc & ((1 << a.lhpg) - 1));
  h8 q[KS];
  auto load_q = [&]() __attribute__((always_inline)) {
    const f16* qh = a.q + (size_t)m * a.q_stride + (size_t)hd * D + 8 * h;
#pragma unroll
    for (int s = 0; s < KS; ++s) q[s] = __builtin_bit_cast(h8, *reinterpret_cast<const u32x4*>(qh + 16 * s));
  };

  // Thread's share of a round: chunk tid % CH of token rows tid / CH + RPI i. Pages are looked up a round ahead of the K / V
  // loads; tokens without a page, or past ctx, read a row that exists; check_v zeroes it. UP: a load
  // instruction's rows lie in one page, lane i looks up the page of load i, and the base is a scalar.
  const int sch = tid % CH, sr = tid / CH;
  constexpr int RPW = kWave / CH;            // rows per load instruction of a wave
  constexpr int NP = UP ? 1 : LPT;
  const uint64_t page_bytes = (uint64_t)a.n_kv << a.log2P << (D == 128 ? 8 : 7);
  const uint64_t head_bytes = (uint64_t)kvh << a.log2P << (D == 128 ? 8 : 7);
  const uint8_t* kp = reinterpret_cast<const uint8_t*>(a.kc) + head_bytes;
  const uint8_t* vp = reinterpret_cast<const uint8_t*>(a.vc) + head_bytes;
  // lane j of a load fills bytes [16 j, 16 j + 16) of the load's rows in LDS: with the chunk that belongs there
  const uint32_t row_off = UP ? (lane / CH) * RB : 0;
  const uint32_t k_place = row_off + 16 * (D == 128 ? sch ^ (sr & 15) : sch ^ ((sr >> 1) & 7));
  const uint32_t v_place = row_off + 64 * ((sch >> 2) ^ (D == 128 ? sr & 3 : (sr >> 1) & 1)) + 16 * (sch & 3);
  int pg[NP];             // pages of the loads
  struct Rows {           // where a round's rows lie (UP: lane i's those of load i)
    uint64_t base[NP];
  };
  bool whole = true;      // every page of this split's tokens is mapped; uniform
  auto mapped = [&](int t) __attribute__((always_inline)) { return (unsigned)a.bt[t >> a.log2P] < (unsigned)a.n_pages; };
  auto lookup = [&](int rnd) __attribute__((always_inline)) {
    const int last = ctx - 1;
    if constexpr (UP) {
      pg[0] = a.bt[min(rnd * SB + RPW * wave + RPI * (lane % LPT), last) >> a.log2P];
    } else {
#pragma unroll
      for (int i = 0; i < LPT; ++i) pg[i] = a.bt[min(rnd * SB + sr + RPI * i, last) >> a.log2P];
    }
  };
  auto locate = [&](int rnd) __attribute__((always_inline)) {  // from the looked-up pages
    Rows w;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int t = UP ? rnd * SB + RPW * wave + RPI * (lane % LPT) : rnd * SB + sr + RPI * i;
      w.base[i] = (uint64_t)(uint32_t)((unsigned)pg[i] < (unsigned)a.n_pages ? pg[i] : 0) * page_bytes +
                  (uint64_t)(uint32_t)(t & (P - 1)) * RB;  // (a page may pass 4 GiB)
    }
    return w;
  };
  auto rows_of = [&](const Rows& w, int i) __attribute__((always_inline)) -> uint64_t {  // bytes ahead of the rows of load i
    return UP ? (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(w.base[0] >> 32), i) << 32 |
                    (uint32_t)__builtin_amdgcn_readlane((int)w.base[0], i)
              : w.base[UP ? 0 : i];
  };
  // load i of a round
  auto fetch = [&](const uint8_t* cache, const Rows& w, int i, uint32_t place, uint8_t* buf) __attribute__((always_inline)) {
    typedef __attribute__((address_space(1))) const void* gptr;
    typedef __attribute__((address_space(3))) void* lptr;
    lptr at = (lptr)(buf + (RPI * i + RPW * wave) * RB);
    if constexpr (UP) {
      const __amdgpu_buffer_rsrc_t res =
          __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(cache) + rows_of(w, i), 0, RPW * RB, 0x00020000);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(res, at, 16, (int)place, 0, 0, 0);
    } else {
      __builtin_amdgcn_global_load_lds((gptr)(cache + rows_of(w, i) + place), at, 16, 0, 0);
    }
  };
  // V chunks that must not meet a p of 0, looked over in LDS by the lane that loaded them: those of tokens that do not exist,
  // and those with NaN or infinity of tokens that not every column sees
  auto check_v = [&](int rnd, uint8_t* buf) __attribute__((always_inline)) {
    const bool reaches = (rnd + 1) * (long long)SB > min(pos, (long long)ctx);  // uniform
    if (!reaches && whole) return;
    asm volatile("");  // stays a branch
#pragma unroll
    for (int i = 0; i < LPT; ++i) {
      const int row = sr + RPI * i, t = rnd * SB + row, word = t / 32 - tail;
      u32x4* x = reinterpret_cast<u32x4*>(buf + row * RB + 16 * sch);
      const bool ok = t < ctx && (whole || mapped(t));
      const bool bad = ok && word >= 0 && has_nonfinite(*x);
      if (bad) atomicOr(&s_bad[word], 1u << (t % 32));
      if (!ok || bad) *x = u32x4{0u, 0u, 0u, 0u};
    }
  };

  // the column's reference maximum (a score), kTreeLift less its c2 fold (infinite: far), and this lane's half of its sum
  float ref = kTreeNoMax, lift = -kTreeNoMax, l = 0.f;
  f32x16 acc[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) acc[t] = f32x16{};

  // LDS addresses: K row r of the group's block (chunk bits apart), and the lane's row of a transposing V read
  const int krow = (grp * BT + r) * RB, ksw = D == 128 ? r & 15 : (r >> 1) & 7;
  const int vt = 4 * h + ((lane & 15) >> 2);               // token (of 8) that the lane addresses
  const int vd = 32 * ((lane >> 4) & 1) + 8 * (lane & 3);  // byte of its 4 dims within the 64-byte unit
  const int vrow = (grp * BT + vt) * RB + vd, vsw = D == 128 ? vt & 3 : (vt >> 1) & 1;

  // bits of tokens [t0, t0 + 64) that column node m sees by position and mask
  auto seen_bits = [&](int t0) __attribute__((always_inline)) -> uint64_t {
    const long long d = (long long)t0 - pos;  // node index of token t0
    int m = cc;
    asm volatile("" : "+v"(m));  // nothing of this is kept in registers around the loop
    m >>= a.lhpg;
    auto low = [](long long n) -> uint64_t { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1; };
    if (a.mask == nullptr) return low(m + 1 - d);
    const int W = (a.M + 63) >> 6;
    const int64_t* row = a.mask + (size_t)m * W;
    if (d <= 0) return d <= -64 ? ~0ull : low(-d) | (uint64_t)row[0] << (int)-d;
    const int w = (int)(d >> 6), sh = (int)(d & 63);
    uint64_t bits = w < W ? (uint64_t)row[w] >> sh : 0ull;
    if (sh != 0 && w + 1 < W) bits |= (uint64_t)row[w + 1] << (64 - sh);
    return bits;
  };
  auto block_start = [&](int rnd) __attribute__((always_inline)) { return (rnd * KVS + grp) * BT; };
  // ---- a block, by tiles of 32 tokens
  f32x16 sc[2];        // scores of a tile and the next
  u32x4 pw[2];         // p in fp16: the B operand of the output's products
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
    // here, beside the products (148.6 -> 145.2 us), not where they are used
    asm volatile("" : "+v"(pair), "+v"(psum[0]), "+v"(psum[1]));
    pw[e >> 3][(e & 7) >> 1] = pair;
  };
  auto block = [&](int rnd, const uint8_t* kb, const uint8_t* vb, auto send) __attribute__((always_inline)) {
    const int t0 = block_start(rnd);
    // every token is seen; uniform per wave
    const bool plain = whole && t0 + (long long)BT <= min(pos, (long long)ctx);
    constexpr int NB = (BT + 63) / 64;
    uint64_t vis[NB];
    if (!plain) {
      asm volatile("");  // stays a branch
#pragma unroll
      for (int c = 0; c < NB; ++c) {
        const int t = t0 + 64 * c + lane % BT;
        vis[c] = __ballot(t < ctx && lane < BT && (whole || mapped(t))) & seen_bits(t0 + 64 * c);
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
        const uint32_t bits = (uint32_t)(vis[tt / 2] >> (32 * (tt & 1))) >> (4 * h);
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
      if (__any(!(sum <= kTreeMost))) {  // the reference moves to this tile's maximum where that is higher
        asm volatile("");
        float mx = s[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
        mx = fmaxf(ref, fmaxf(mx, __shfl_xor(mx, 32, kWave)));
        // (a column decides by itself: its result does not depend on what else shares its wave)
        const int over = !(sum <= kTreeMost);
        mx = over | __shfl_xor(over, 32, kWave) ? mx : ref;
        const float alpha = __builtin_amdgcn_exp2f((ref - mx) * a.c2);  // 1 for a column that stays
        if (mx != ref) lift = fabsf(mx * a.c2) > kTreeFar ? INFINITY : kTreeLift - mx * a.c2;
        ref = mx;
        const float off = lift == INFINITY ? ref : 0.f, up = lift == INFINITY ? kTreeLift : lift;
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
      }
    }
  };

  // Round rnd, in buffer B: the loads of round rnd + 1 go out, straight into the other buffer (every wave finished reading
  // it before the last barrier).
  Rows rows;
  auto start = [&](int j, uint8_t* k, uint8_t* v) __attribute__((always_inline)) {  // load j of K's and V's 2 LPT
    if (j < LPT)
      fetch(kp, rows, j, k_place, k);
    else
      fetch(vp, rows, j - LPT, v_place, v);
  };
  auto finish = [&](int rnd, uint8_t* v) __attribute__((always_inline)) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (rnd < r1) check_v(rnd, v);
    __syncthreads();
  };
  auto round = [&](int rnd, auto B) __attribute__((always_inline)) {
    constexpr bool odd = decltype(B)::value;
    uint8_t *kb = odd ? s_k1 : s_k0, *vb = odd ? s_v1 : s_v0, *kn = odd ? s_k0 : s_k1, *vn = odd ? s_v0 : s_v1;
    rows = locate(rnd + 1);  // past the end: rows that are never computed on
    // spread over the products: issued in a row they hold a wave up while the other waves' are taken in
    constexpr int NF = KS * NT, NL = 2 * LPT;
    block(rnd, kb, vb, [&](int f) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < NL; ++j)
        if (f == j * NF / NL) start(j, kn, vn);
      if (f == NF - 1) lookup(rnd + 2);
    });
    pf_fence();
    finish(rnd + 1, vn);
  };
  if (r0 < r1) {  // uniform
    lookup(r0);
    if (tid < kBadWords) s_bad[tid] = 0u;
    if (tid == 0) s_holes = 0;
    rows = locate(r0);
#pragma unroll
    for (int j = 0; j < 2 * LPT; ++j) start(j, s_k0, s_v0);
    pf_fence();  // (loads return in order: what is wanted later goes out later)
    lookup(r0 + 1);
    load_q();
    pf_fence();
    const int last_page = (min(r1 * SB, ctx) - 1) >> a.log2P;
    for (int p = (r0 * SB >> a.log2P) + tid; p <= last_page; p += NTH) whole = whole && (unsigned)a.bt[p] < (unsigned)a.n_pages;
    __syncthreads();  // (s_bad, s_holes)
    if (!whole) s_holes = 1;
    __syncthreads();
    whole = __builtin_amdgcn_readfirstlane(s_holes) == 0;
    finish(r0, s_v0);
    for (int rnd = r0; rnd < r1; rnd += 2) {
      round(rnd, std::false_type{});
      if (rnd + 1 < r1) round(rnd + 1, std::true_type{});
    }
    // ---- add_bad_rows: the chunks that check_v took out, from the cache, for the columns that see their token; its weight
    // once more from q and k
    for (int word = max(tail, r0 * (SB / 32)); word < min(r1 * (SB / 32), (ctx + 31) / 32); ++word) {
      if (word * 32 / BT % KVS != grp) continue;
      uint32_t bad = __builtin_amdgcn_readfirstlane(s_bad[word - tail]);
      if (bad == 0) continue;
      const uint64_t vis = seen_bits(word * 32);
      // the scores of the 32 tokens, as in the loop and so the same to the last bit (tokens that do not exist: of any row)
      const int tk = min(word * 32 + r, ctx - 1), pk = a.bt[tk >> a.log2P];
      const size_t kat = ((((size_t)((unsigned)pk < (unsigned)a.n_pages ? pk : 0) * a.n_kv + kvh) << a.log2P) + (tk & (P - 1))) * D;
      f32x16 st = {};
#pragma unroll
      for (int k = 0; k < KS; ++k)
        st = mfma32x32(__builtin_bit_cast(h8, *reinterpret_cast<const u32x4*>(a.kc + kat + 16 * k + 8 * h)), q[k], st);
      for (; bad != 0; bad &= bad - 1) {
        const int i = __builtin_ctz(bad), t = word * 32 + i;
        const int page = a.bt[t >> a.log2P];  // a token in this set is mapped and inside the context
        const size_t at = ((((size_t)page * a.n_kv + kvh) << a.log2P) + (t & (P - 1))) * D;
        float dot = 0.f;  // in element 4 (i / 8) + i % 4 of the half i / 4 % 2
#pragma unroll
        for (int e = 0; e < 16; ++e) dot = e == 4 * (i >> 3) + (i & 3) ? st[e] : dot;
        dot = __shfl(dot, r + 32 * ((i >> 2) & 1), kWave);
        const float p = __builtin_amdgcn_exp2f(lift == INFINITY ? fmaf(dot - ref, a.c2, kTreeLift) : fmaf(dot, a.c2, lift));
        const bool see = (vis >> i) & 1;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          const u32x4 x = *reinterpret_cast<const u32x4*>(a.vc + at + 8 * c);
          if (!has_nonfinite(x) || !see) continue;
          const f16x2 lo = as_f16x2(h ? x[2] : x[0]), hi = as_f16x2(h ? x[3] : x[1]);
          const float f[4] = {(float)lo[0], (float)lo[1], (float)hi[0], (float)hi[1]};
#pragma unroll
          for (int v = 0; v < 4; ++v) acc[c / 4][4 * (c % 4) + v] = fmaf(p, f[v], acc[c / 4][4 * (c % 4) + v]);
        }
      }
    }
  }
  l += __shfl_xor(l, 32, kWave);
  // ---- output: acc[t][4 q + v] = O[column r][dim 32 t + 8 q + 4 h + v], row 4 t + q of a wave's 4 DT rows of float4. The
  // groups leave theirs in LDS (over the K / V buffers, which every wave has finished reading at the last barrier), with
  // maximum and sum per column; then each takes 1 / KVS of the rows, over all groups in order.
  const int waves = (cols + 31) >> 5;
  const size_t part = ((size_t)split * a.n_kv + kvh) * waves + (cb * CW + gw);
  if (a.splits > 1 && r0 >= r1) {  // a split without tokens: the join reads no accumulator of it
    if (grp == 0 && h == 0 && col < cols) a.part_ml[part * 32 + r] = float2{kTreeNoMax, 0.f};
    return;
  }
  constexpr int kRows = 4 * DT / KVS;
  float mx = ref, L = l, w[KVS];
  auto own_row = [&](int i) __attribute__((always_inline)) {
    return float4{acc[i / 4][4 * (i % 4)], acc[i / 4][4 * (i % 4) + 1], acc[i / 4][4 * (i % 4) + 2], acc[i / 4][4 * (i % 4) + 3]};
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
constexpr int kTreeJoinRows = 4;
template <int D>
__global__ void __launch_bounds__(kTreeJoinRows * kWave)
attn_tree_join_kernel(const float4* __restrict__ part_o, const float2* __restrict__ part_ml, int cols, int lhpg, int n_kv,
                      int splits, float c2, f16* __restrict__ out) {
  constexpr int kRows = kTreeJoinRows, kBatch = 8, kGroups = 2 * kRows;  // kGroups threads share a column's maxima and sums
  __shared__ float s_w[kTreeMaxSplits][32];          // a split's weight in a column, -1 where it saw no token
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
    constexpr int kMl = kTreeMaxSplits / kGroups;
    float2 ml[kMl];
    float mx = kTreeNoMax;
#pragma unroll
    for (int j = 0; j < kMl; ++j) {
      const int s = g + kGroups * j;
      ml[j] = s < splits ? part_ml[((size_t)s * wstep + wave) * 32 + c] : float2{kTreeNoMax, 0.f};
      mx = fmaxf(mx, ml[j].x);
    }
    mx = group_max<kGroups>(mx);
    float L = 0.f;
#pragma unroll
    for (int j = 0; j < kMl; ++j) {
      const int s = g + kGroups * j;
      const bool saw = ml[j].x != kTreeNoMax || ml[j].y != 0.f;  // (a NaN sum counts)
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

// Workgroup shape (CW, KVS, BT) by the column waves of a kv head and the longest context. Each shape's time against the best
// of seven, geometric mean / worst over 288 cases (1-250 nodes, six head layouts, contexts of 500 to 32000):
//             to 4 waves: 1000, 4000, 8000, from 16000   5 to 8: the same                        9 and more: the same
//   D 128
//   (4,1,64)  1.00/1.00 1.06/1.21 1.03/1.18 1.03/1.09   1.00/1.00 1.05/1.12 1.02/1.06 1.08/1.16   1.04/1.17 1.11 1.09 1.19
//   (2,4,32)  1.11/1.21 1.05/1.12 1.03/1.11 1.02/1.10   1.05/1.08 1.03/1.07 1.02/1.04 1.08/1.16   1.06/1.11 1.06 1.09 1.18
//   (4,2,64)  1.10/1.18 1.05/1.11 1.07/1.27 1.02/1.11   1.07/1.09 1.05/1.08 1.03/1.08 1.00/1.02   1.02/1.05 1.01 1.02 1.02
//   (8,1,128) 1.16/1.30 1.13/1.22 1.16/1.28 1.23/1.44   1.15/1.19 1.28/1.39 1.19/1.31 1.08/1.21   1.13/1.18 1.14 1.03 1.02
//             (250 nodes, 8 x 4 heads: (4,2,64) 80.7 us at 16000, 150.6 at 32000, (8,1,128) 80.4, 140.1)
//   D 64
//   (2,4,32)  1.05/1.12 1.02/1.09 1.01/1.03 1.00/1.06   1.00/1.00 1.00/1.00 1.00/1.01 1.04/1.13   1.02/1.09 1.03 1.05 1.13
//   (4,2,64)  1.06/1.13 1.05/1.11 1.05/1.26 1.05/1.19   1.05/1.07 1.08/1.19 1.12/1.30 1.04/1.22   1.04/1.10 1.07 1.04 1.02
// A context that four groups of 32 tokens get through in three rounds (D 64) or two (D 128) is not split: one launch instead
// of two. 26 nodes, 4 x 8 heads of 64: at 100 tokens 6.9 us against 9.4 split, at 300 8.8 : 9.7, at 500 10.7 : 10.6 (250
// nodes 11.3 : 13.0, 13.0 : 14.6, 13.8 : 15.1); 8 x 4 heads of 128: at 100 10.7 : 11.7, at 200 12.0 : 11.9, at 300 13.4 : 11.9.
// Called eagerly the second launch costs another 3 us of host time.
struct TreeShape {
  int cw, kvs, bt;
  bool split = true;
};
TreeShape tree_shape(int M, int n_q, int n_kv, int D, int max_ctx) {
  const int waves = (M * (n_q / n_kv) + 31) / 32;
  if (D == 128) {
    if (max_ctx <= 2 * 128) return {2, 4, 32, false};
    if (waves <= 8 && max_ctx <= 2048) return {4, 1, 64};
    if (waves <= 4) return {2, 4, 32};
    return waves > 8 && max_ctx >= 20000 ? TreeShape{8, 1, 128} : TreeShape{4, 2, 64};
  }
  if (max_ctx <= 3 * 128) return {1, 4, 32, false};
  return waves > 8 && max_ctx >= 8000 ? TreeShape{4, 2, 64} : TreeShape{2, 4, 32};
}

}  // namespace

// At most one workgroup per CU, in splits of equal length: exactly one where blocks * n_kv divides 256, and fewer elsewhere
// (11 blocks of 8 heads: two splits, 176 workgroups).
int attention_tree_splits(int M, int n_q, int n_kv, int D, int max_ctx) {
  const TreeShape s = tree_shape(M, n_q, n_kv, D, max_ctx);
  if (!s.split) return 1;
  const int blocks = (M * (n_q / n_kv) + 32 * s.cw - 1) / (32 * s.cw), round = s.bt * s.kvs;
  const int rounds = max_ctx / round + (max_ctx % round != 0);
  int want = 256 / (blocks * n_kv);
  want = want < 1 ? 1 : want > kTreeMaxSplits ? kTreeMaxSplits : want;
  const int per = rounds / want + (rounds % want != 0);
  return (rounds + per - 1) / per;
}
size_t attention_tree_part_bytes(int M, int n_q, int n_kv, int head_dim) {
  return (size_t)n_kv * ((M * (n_q / n_kv) + 31) / 32) * 32 * (head_dim + 2) * sizeof(float);
}

template <int D, int CW, int KVS, int BT>
static void launch_tree_shape(const TreeArgs& a, int cols, hipStream_t st) {
  const dim3 grid(a.n_kv, (cols + 32 * CW - 1) / (32 * CW), a.splits), block(CW * KVS * kWave);
  if ((1 << a.log2P) >= 512 / D)
    hipLaunchKernelGGL((attn_tree_kernel<D, CW, KVS, BT, true>), grid, block, 0, st, a);
  else
    hipLaunchKernelGGL((attn_tree_kernel<D, CW, KVS, BT, false>), grid, block, 0, st, a);
}

template <int D>
static void launch_tree(const TreeAttn& t, hipStream_t st) {
  int lhpg = 0;
  while ((t.n_kv << lhpg) < t.n_q) ++lhpg;
  const int cols = t.M << lhpg, waves = (cols + 31) / 32;
  float4* part_o = (float4*)t.ws;
  TreeArgs a{(const f16*)t.q, t.q_stride, t.mask, t.pos, t.bt, (const f16*)t.kc, (const f16*)t.vc, t.n_pages, t.log2P,
             t.n_kv, lhpg, t.M, (int)min((long long)t.max_ctx, (long long)t.n_bt << t.log2P), t.splits,
             (float)(1.4426950408889634 / sqrt((double)D)), (f16*)t.out, part_o,
             (float2*)(part_o + (size_t)t.splits * t.n_kv * waves * 8 * D)};
  const TreeShape s = tree_shape(t.M, t.n_q, t.n_kv, D, t.max_ctx);
  if constexpr (D == 128) {
    if (s.cw == 2)
      launch_tree_shape<D, 2, 4, 32>(a, cols, st);
    else if (s.cw == 8)
      launch_tree_shape<D, 8, 1, 128>(a, cols, st);
    else if (s.kvs == 1)
      launch_tree_shape<D, 4, 1, 64>(a, cols, st);
    else
      launch_tree_shape<D, 4, 2, 64>(a, cols, st);
  } else {
    if (s.cw == 1)
      launch_tree_shape<D, 1, 4, 32>(a, cols, st);
    else if (s.cw == 2)
      launch_tree_shape<D, 2, 4, 32>(a, cols, st);
    else
      launch_tree_shape<D, 4, 2, 64>(a, cols, st);
  }
  if (t.splits > 1)
    hipLaunchKernelGGL(attn_tree_join_kernel<D>, dim3(t.n_kv, waves * (D / 8 / kTreeJoinRows)), dim3(kTreeJoinRows * kWave),
                       0, st, part_o, a.part_ml, cols, lhpg, t.n_kv, t.splits, a.c2, (f16*)t.out);
}

void launch_attention_tree(const TreeAttn& a, hipStream_t st) {
  if (a.head_dim == 64)
    launch_tree<64>(a, st);
  else
    launch_tree<128>(a, st);
}

}  // namespace dk
