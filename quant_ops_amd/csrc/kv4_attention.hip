// Causal attention over the 4-bit cache of kv4_common.h, on its codes: with k = lo + s c,
// q . k = s (q . c) + lo sum(q), and with v = mid + s (c - 8), mid = lo + 8 s, sum_t p v =
// sum_t (p s) (c - 8) + sum_t p mid: both products run on the codes, which fp16 holds exactly,
// and the parameters are applied to scores, in float32. Values are taken from their middle so
// that the sums hold no large terms that cancel.
//
// A wave takes 64 tokens a step (four tiles of 16) and up to 16 rows. v_mfma_f32_16x16x32_f16 computes S^T = K Q^T (A: codes of 16
// tokens, B: queries) and O^T += V^T P^T (A: codes of 16 pairs' values, B: weights). Lane
// l = r + 16 g of an operand holds eight consecutive k of row r, a lane of the result rows
// 4 g .. 4 g + 3 of column r; the order of k is free as long as both operands have it. So
//   * S^T's row 4 a + i of its tile u is token 16 a + 4 u + i: lane group g ends up with tokens
//     16 g .. 16 g + 15, the k that it supplies to the second product from the 16 bytes of
//     tile g of the values, and the weights never change lanes;
//   * values of a vector (k of the first product) and tokens (of the second) come in the order
//     in which masks take codes out of a word, and the queries and weights are put in it.
//
// For 16-bit queries a key's code is made fp16 by masking alone: its four bits at the bottom of an fp16
// are the subnormal c 2^-24, at bits 4 .. 7 c 2^-20 (five instructions for eight codes). The matrix
// core keeps subnormals, but what it drops of a sum of products (probed) goes by an exponent that a
// subnormal's leading zeros do not lower: sums are off by 1e-7 of their terms' magnitudes. Values
// meet weights of very different sizes, where that costs much more (2e-6 of the terms, all of one
// sign, at 33210 tokens), so their codes less 8 are normal numbers (nine instructions for eight),
// and float32 queries have keys' codes as those too.
//
// Rows that are few (FOLD times 16 / FOLD of them) stand in every 16 / FOLD columns again, and the lanes
// of those columns share a row's scores: each takes 16 / FOLD of its group's tokens from the scores
// to the weights, which then go back to the first columns. Second parts (of float32 queries, of weights) then
// stand in columns 8 .. 15: one product makes the sums of both parts, in half the instructions and registers, and the two
// meet by a rotation of lanes (24 sequences of 1024 tokens, float32 of 256: 32 -> 26 us;
// 16 x 2048 tokens of 32 heads, fp16: 25 -> 24).
//
// Queries: brought by a power of two for each row to a largest magnitude in [2^14, 2^15), 16-bit
// values are exact in fp16 (those below 2^-28 of the largest lose bits); float32 takes two fp16
// parts (22 bits). Weights: p s 2^14 / S, where p is 1 at the row's largest score so far and S a
// power of two that no scale of the tokens so far exceeds, is at most 2^14, in two fp16 parts (22 bits; with one a
// bf16 output in twenty is a step off, and the second costs 2 to 3 % up to eight rows a sequence, 3 to 7 % up to 32). In
// float32 the second parts have sums of their own: added to the first parts' they would lose what is below 2^-24 of
// those. Weights p s below 2^-28 of S lose bits (in kv4_prefill.hip below 2^-20). Maximum, sums and outputs are float32.
//
// What bounds it: one sequence of 131072 tokens (64 heads on 8 of 128, bf16, 142 MB) takes 33 us, 4.3 TB/s; 64 sequences of
// 2098 tokens (32 on 8 heads, 146 MB) take 30 us, 4.9 TB/s, where a copy reaches 5.1. The same tokens in sequences of 100 to
// 4096 take 43 us: a workgroup each, the longest twice an even share. Loads a step ahead were worth 100 -> 55 us there,
// lanes that share scores 55 -> 46.
#include "dispatch_rules.h"
#include "kv4_attention.h"

namespace qo {

namespace {

// And over lanes r, r + CW, .. of a row of 16.
template <int CW, class F>
__device__ inline uint32_t row_reduce(uint32_t u, F f) {
  if constexpr (CW <= 4) u = f(u, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u, 0x124, 0xF, 0xF, false));   // row_ror:4
  if constexpr (CW <= 8) u = f(u, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u, 0x128, 0xF, 0xF, false));   // row_ror:8
  return groups_reduce(u, f);
}

// v from another lane of the row of 16 (CTRL) in lanes of the banks of four of BANKS, elsewhere old.
template <int CTRL, int BANKS>
__device__ inline uint32_t merge(uint32_t old, uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)old, (int)v, CTRL, 0xF, BANKS, false);
}
constexpr int kStay = 0xE4, kRor8 = 0x128, kShl4 = 0x104, kShl12 = 0x10C, kShr4 = 0x114;   // quad_perm, row_ror, row_shl, row_shr

// The eight codes of a key's word in the order of kCodeOrder: even ones times kEven, odd ones times
// kOdd, all less kLess.
template <bool FINE>
struct Codes {
  static constexpr float kEven = FINE ? 1.f : 0x1p-24f, kOdd = 16.f * kEven, kLess = FINE ? 8.f : 0.f;
  __device__ static inline v8h of(uint32_t w, uint32_t e) {
    const uint32_t h = w >> 8;
    if constexpr (FINE) return __builtin_bit_cast(v8h, (v4u){less_low(w, e), less_high(w, e), less_low(h, e), less_high(h, e)});
    else return __builtin_bit_cast(v8h, (v4u){w & kLow, w & kHigh, h & kLow, h & kHigh});
  }
};

// The low (odd: high) halves of eight bytes of values, in the order 0, 2, 1, 3, 4, 6, 5, 7.
__device__ inline v8h values_even(uint32_t a, uint32_t b, uint32_t e) {
  return __builtin_bit_cast(v8h, (v4u){less_low(a, e), less_low(a >> 8, e), less_low(b, e), less_low(b >> 8, e)});
}
__device__ inline v8h values_odd(uint32_t a, uint32_t b, uint32_t e) {
  return __builtin_bit_cast(v8h, (v4u){less_high(a, e), less_high(a >> 8, e), less_high(b, e), less_high(b >> 8, e)});
}

template <class D, int DIM, int FOLD, int NQ, bool FINE>
__global__ void __launch_bounds__(256, DIM <= (FOLD > 1 ? 256 : FINE ? 96 : 192) ? 2 : 1)
kv4_attention_kernel(Attention a) {
  constexpr bool PACK = FOLD > 1;     // second parts in columns 8 .. 15
  constexpr int NQF = PACK ? 1 : NQ;
  constexpr int NS = DIM / 32;        // k-steps of a score, words of a key's codes in a lane
  constexpr int NF = DIM / 32;        // blocks of 16 pairs of values
  constexpr int CW = 16 / FOLD;       // columns with rows of their own, and tokens of a step for a lane's softmax
  constexpr int TILE = 4 * CW;
  constexpr int APART = FINE && !PACK;   // second parts of weights have sums of their own
  using C = Codes<FINE>;
  using T = typename D::T;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  const int heads = a.cache.heads;
  const int head = blockIdx.x % heads, split = blockIdx.x / heads / a.tiles;
  const Rows w = find_rows<TILE>(a, blockIdx.x / heads % a.tiles);
  if (!w.all) return;
  const int row0 = w.index * TILE, rows = min(w.all - row0, TILE);

  // The waves' rows; waves with the same rows take turns at their tokens.
  const int blocks = (rows + CW - 1) / CW;
  const int sharing = blocks == 1 ? 4 : blocks == 2 ? 2 : 1;
  const int mine = wave / sharing, turn_of = wave % sharing;
  const bool active = mine < blocks;
  const int first_row = row0 + (active ? mine : 0) * CW;
  const int last_row = min(first_row + CW, row0 + rows) - 1;
  const int row = min(first_row + r % CW, last_row);
  const Sees top = sees(a, w, first_row), bottom = sees(a, w, last_row), see = sees(a, w, row);

  // The query as fp16 parts in the order of Codes::of, the odd codes' factor taken out.
  v8h qf[NQF][NS];
  float factor, qsum;   // of the exponent of two; sum of the query, in units of its scores
  {
    const T* q = reinterpret_cast<const T*>(a.q) + (w.start + row / a.group) * a.q_token + (head * a.group + row % a.group) * a.q_head;
    float x[NS][8], most = 0.f;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      T t[8];
      __builtin_memcpy(t, q + (g * NS + s) * 8, sizeof(t));
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[s][i] = D::to_f(t[i]);
        most = fmaxf(most, fabsf(x[s][i]));
      }
    }
    most = bits_float(groups_reduce(float_bits(most), FMax{}));
    const int e = query_exponent(most);
    float sum = 0.f;
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float v = ldexpf(x[s][kCodeOrder[i]], e);
        sum += v;
        const float part = opaque(kCodeOrder[i] & 1 ? v * (C::kEven / C::kOdd) : v);
        const _Float16 hi = (_Float16)part;
        qf[0][s][i] = hi;
        if constexpr (NQ > 1) {
          const _Float16 lo = (_Float16)(part - (float)hi);
          if constexpr (PACK) qf[0][s][i] = r & 8 ? lo : hi;
          else qf[1][s][i] = lo;
        }
      }
    sum = bits_float(groups_reduce(float_bits(sum), FAdd{}));
    qsum = most < kInf ? sum * C::kEven : __builtin_nanf("");   // an infinity's scores are NaN
    factor = score_factor(a.scale, e, 1.f / C::kEven);
  }

  v4f o[APART + 1][NF][2];
  float most = -kInf, at = 0.f, total = 0.f, middles = 0.f;   // largest score, as an exponent; sums of weights, and times middles
#pragma unroll
  for (int h = 0; h <= APART; ++h)
#pragma unroll
    for (int f = 0; f < NF; ++f) o[h][f][0] = o[h][f][1] = v4f{0.f, 0.f, 0.f, 0.f};
  int scale_exp = -14;
  bool far = false;   // some row's exponent is kFar or more

  const int begin = top.first & ~63;
  const int steps = bottom.last > begin ? (bottom.last - begin + 63) / 64 : 0;
  const int per_split = (steps + a.splits - 1) / a.splits;
  const int to = (split + 1) * per_split < steps ? (split + 1) * per_split : steps;
  const int32_t* table = a.table + (w.b < a.sequences ? w.b : 0) * a.table_ld;
  const Pages pages(a.cache, head, DIM);

  // A step's loads go out a step ahead: its pages two, its keys as soon as the scores of the step
  // before are made, its values after that step's second product.
  // The lane's tokens of a step, from the scores to the weights: 16 g + own ..; their parameters in pairs.
  const int own = r / CW * CW;
  uint32_t kw[4][NS], ks[CW / 2], kl[CW / 2], vs[CW / 2], vl[CW / 2];
  v4u vw[NF];
  Tile kt, vt;
  bool bad = false;               // the lane's tokens stand on a page outside the cache
  auto find = [&](int step) {
    // keys: lane row r reads token 16 (r / 4) + 4 u + r % 4 of tile u, its words of group g
    kt = tile_at(a, table, begin + 64 * step + 16 * (r >> 2));
    vt = tile_at(a, table, begin + 64 * step + 16 * g);
  };
  auto load_keys = [&] {
    const uint8_t* p = pages.k + (uint64_t)(uint32_t)kt.page * pages.codes + ((kt.place + (r & 3)) * (DIM / 2) + g * (4 * NS));
    const uint8_t* par = pages.params + (uint64_t)(uint32_t)vt.page * pages.param_bytes + (vt.place * 4 + own * 2);
#pragma unroll
    for (int u = 0; u < 4; ++u) __builtin_memcpy(kw[u], p + u * 4 * (DIM / 2), sizeof(kw[u]));
    __builtin_memcpy(ks, par, sizeof(ks));
    __builtin_memcpy(kl, par + 32, sizeof(kl));
  };
  auto load_values = [&] {
    const uint8_t* p = pages.v + (uint64_t)(uint32_t)vt.page * pages.codes + (vt.place * (DIM / 2) + r * 16);
    const uint8_t* par = pages.params + (uint64_t)(uint32_t)vt.page * pages.param_bytes + pages.param_values + (vt.place * 4 + own * 2);
    __builtin_memcpy(vs, par, sizeof(vs));
    __builtin_memcpy(vl, par + 32, sizeof(vl));
#pragma unroll
    for (int f = 0; f < NF; ++f) vw[f] = *reinterpret_cast<const v4u*>(p + f * 256);
  };
  const uint32_t exponents = exponents_of_1024();

  const int first_step = split * per_split + turn_of;
  if (active && first_step < to) {
    find(first_step);
    bad = vt.bad;
    load_keys();
    load_values();
    find(first_step + sharing);
  }
  for (int step = first_step; active && step < to; step += sharing) {
    const int t0 = begin + 64 * step;
    const bool more = step + sharing < to;
    const bool whole = t0 + 64 <= top.last && t0 >= bottom.first && !__any(bad);
    // scores
    v4f sc[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      v4f rest = {0.f, 0.f, 0.f, 0.f};
      sc[u] = rest;
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        const v8h c = C::of(kw[u][s], exponents);
        sc[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(c, qf[0][s], sc[u], 0, 0, 0);
        if constexpr (NQF > 1) rest = __builtin_amdgcn_mfma_f32_16x16x32_f16(c, qf[1][s], rest, 0, 0, 0);
      }
      if constexpr (NQF > 1) {
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[u][i] += rest[i];
      }
    }
    float x[CW];   // of the lane's tokens
#pragma unroll
    for (int t = 0; t < CW; ++t) {
      auto at_token = [&](int i) { return float_bits(sc[i / 4][i % 4]); };
      auto pick = [&](int first) {   // token first + t of the lane's own, of columns with the same values
        const int n = FOLD - 1;
        uint32_t y = at_token(first + t);
        if constexpr (FOLD == 2) y = merge<kStay, 0xC>(y, at_token((first + CW & n * CW) + t));
        if constexpr (FOLD == 4) {
          y = merge<kStay, 2>(y, at_token((first + CW & n * CW) + t));
          y = merge<kStay, 4>(y, at_token((first + 2 * CW & n * CW) + t));
          y = merge<kStay, 8>(y, at_token((first + 3 * CW & n * CW) + t));
        }
        return y;
      };
      uint32_t y = pick(0);
      // the other part's share comes from the column 8 apart
      if constexpr (PACK && NQ > 1) y = float_bits(bits_float(y) + bits_float(merge<kRor8, 0xF>(0, pick(8))));
      const float s = half_of(ks, t), lo = half_of(kl, t);
      x[t] = fmaf(s, bits_float(y), fmaf(C::kLess, s, lo) * qsum);
    }
    __builtin_amdgcn_sched_barrier(0);
    const bool bad_now = bad;
    if (more) {
      bad = vt.bad;
      load_keys();
    }
    if (!whole) {
      // Tokens that the row does not see get no weight, whatever stands there. A NaN (or a page outside the
      // cache) that it sees makes its sum NaN; a value's parameters are then 0, for the rows that do not.
#pragma unroll
      for (int t = 0; t < CW; ++t) {
        const int at_t = t0 + 16 * g + own + t;
        const bool finite = fabsf(half_of(vs, t)) < kInf && fabsf(half_of(vl, t)) < kInf && !bad_now;
        const bool any = at_t >= top.first && at_t < bottom.last, seen = at_t >= see.first && at_t < see.last;
        x[t] = seen ? x[t] : -kInf;
        if (seen && !finite) total = __builtin_nanf("");
        if (!finite || !any) {
          const uint32_t keep = t & 1 ? 0x0000FFFFu : 0xFFFF0000u;
          vs[t / 2] &= keep;
          vl[t / 2] &= keep;
        }
      }
    }
    // the exponent of the largest scale, over the step's tokens (as bits, which order like it)
    uint32_t big = 0;
#pragma unroll
    for (int i = 0; i < CW / 2; ++i) big = pk_max_u16(big, vs[i] & 0x7FFF7FFFu);
    const uint32_t field = row_reduce<CW>(max(big & 0xFFFFu, big >> 16) >> 10, UMax{});
    const int exp_now = max(scale_exp, __builtin_amdgcn_readfirstlane((int)field) - 14);
    // s becomes s 2^14 / S, exactly, in one packed product or (scales below 1/4) two
    const int up = 14 - exp_now;
    auto by_power = [&](int e) {
      const _Float16 f = (_Float16)power_of_two(e);
#pragma unroll
      for (int i = 0; i < CW / 2; ++i) vs[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, vs[i]) * (v2h){f, f});
    };
    by_power(min(up, 15));
    if (up > 15) by_power(up - 15);
    const float eight = power_of_two(3 - up);   // 8 of the scale as it was
    float now = most;
#pragma unroll
    for (int t = 0; t < CW; ++t) now = fmaxf(now, x[t]);
    now = bits_float(row_reduce<CW>(float_bits(now), FMax{}));
    if (__any(now > most) || exp_now > scale_exp) {
      const float next = now == -kInf ? 0.f : factor * now;
      const float shrink = most == -kInf ? 1.f : __builtin_amdgcn_exp2f(at - next);   // before: all sums 0
      const float shrink_o = shrink * power_of_two(scale_exp - exp_now);
      most = now;
      at = next;
      far = __any(fabsf(at) >= kFar);
      total *= shrink;
      middles *= shrink;
#pragma unroll
      for (int h = 0; h <= APART; ++h)
#pragma unroll
        for (int f = 0; f < NF; ++f) {
          o[h][f][0] *= shrink_o;
          o[h][f][1] *= shrink_o;
        }
    }
    if (far) {
#pragma unroll
      for (int t = 0; t < CW; ++t) x[t] *= factor;
    }
    const float slope = far ? 1.f : factor;
    uint32_t wh[CW / 2], wl[CW / 2];   // weights, in the order of values_even
    {
      _Float16 hi[CW], lo[CW];
#pragma unroll
      for (int t = 0; t < CW; ++t) {
        constexpr int kSlot[4] = {0, 2, 1, 3};
        const int j = t / 4 * 4 + kSlot[t % 4];
        const float p = __builtin_amdgcn_exp2f(fmaf(slope, x[t], -at));
        const float s = half_of(vs, t);
        total += p;
        middles = fmaf(p, fmaf(eight, s, half_of(vl, t)), middles);   // what code 8 stands for
        hi[j] = (_Float16)fmaf(p, s, 0.f);
        // one and the same rounding in both parts: the product rounded twice (to float32 first)
        // or once differ by a step of h where it is next to a tie
        asm("" : "+v"(hi[j]));
        lo[j] = (_Float16)fmaf(p, s, -(float)hi[j]);
      }
      __builtin_memcpy(wh, hi, sizeof(wh));
      __builtin_memcpy(wl, lo, sizeof(wl));
    }
    scale_exp = exp_now;
    __builtin_amdgcn_sched_barrier(0);
    // Tokens 8 z .. 8 z + 7 of the group.
    auto weights = [&](const uint32_t* x, int z) {
      return __builtin_bit_cast(v8h, (v4u){x[4 * z], x[4 * z + 1], x[4 * z + 2], x[4 * z + 3]});
    };
    // The same of both parts, the second in columns 8 ..
    auto both = [&](int z) {
      v4u v;
      if constexpr (PACK && FOLD == 2) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = z == 0 ? merge<kRor8, 0xC>(wh[i], wl[i]) : merge<kRor8, 0x3>(wl[i], wh[i]);
      }
      if constexpr (PACK && FOLD == 4) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          v[i] = z == 0 ? merge<kRor8, 0x4>(wh[i], wl[i]) : merge<kRor8, 0x1>(wl[i], wh[i]);
          v[2 + i] = z == 0 ? merge<kShr4, 0x4>(merge<kShl4, 0xF>(0, wh[i]), wl[i])
                            : merge<kShl12, 0x1>(merge<kShl4, 0xF>(0, wl[i]), wh[i]);
        }
      }
      return __builtin_bit_cast(v8h, v);
    };
    v8h ph[2], pl[2];
#pragma unroll
    for (int z = 0; z < 2; ++z) {
      if constexpr (PACK) {
        ph[z] = both(z);
      } else {
        ph[z] = weights(wh, z);
        pl[z] = weights(wl, z);
      }
    }
#pragma unroll
    for (int f = 0; f < NF; ++f)
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        const v8h even = values_even(vw[f][2 * z], vw[f][2 * z + 1], exponents), odd = values_odd(vw[f][2 * z], vw[f][2 * z + 1], exponents);
        v4f(&hi)[2] = o[0][f], (&lo)[2] = o[APART][f];
        hi[0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(even, ph[z], hi[0], 0, 0, 0);
        hi[1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(odd, ph[z], hi[1], 0, 0, 0);
        if constexpr (!PACK) {
          lo[0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(even, pl[z], lo[0], 0, 0, 0);
          lo[1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(odd, pl[z], lo[1], 0, 0, 0);
        }
      }
    __builtin_amdgcn_sched_barrier(0);
    if (more) {
      load_values();
      find(step + 2 * sharing);
    }
  }

  // Outputs in units of the weights, and the sums of all lanes. A wave that saw nothing has
  // the exponent -inf, so that it counts for nothing beside another.
  const float unit = power_of_two(scale_exp - 14);
  total = bits_float(row_reduce<CW>(float_bits(total), FAdd{}));
  middles = bits_float(row_reduce<CW>(float_bits(middles), FAdd{}));
  if (most == -kInf && total == 0.f) at = -kInf;
  if (w.poison) total = __builtin_nanf(""), at = 0.f;
#pragma unroll
  for (int f = 0; f < NF; ++f)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (PACK) {
        for (int h = 0; h < 2; ++h) {
          const float first = o[0][f][h][i];
          o[0][f][h][i] = first + bits_float(merge<kRor8, 0xF>(0, float_bits(first)));
        }
      }
      if constexpr (APART) o[0][f][0][i] += o[1][f][0][i], o[0][f][1][i] += o[1][f][1][i];
      o[0][f][0][i] = fmaf(o[0][f][0][i], unit, middles);
      o[0][f][1][i] = fmaf(o[0][f][1][i], 0.0625f * unit, middles);
    }
  // Waves that shared rows: half of them hand theirs to the others, twice for four.
  __shared__ float join[2][64][NF * 8 + 3];   // an odd number: lanes in different banks
  for (int step = sharing / 2; step > 0; step /= 2) {
    // of two waves that share rows and stand `step` turns apart the later gives
    const int slot = sharing == 4 ? (turn_of % step) : mine;
    float* box = join[slot & 1][lane];
    if (active && turn_of >= step && turn_of < 2 * step) {
      box[0] = at;
      box[1] = total;
#pragma unroll
      for (int f = 0; f < NF; ++f)
#pragma unroll
        for (int i = 0; i < 8; ++i) box[2 + f * 8 + i] = o[0][f][i >> 2][i & 3];
    }
    __syncthreads();
    if (active && turn_of < step) {
      const float other = box[0], both = fmaxf(at, other);
      const float x = at == -kInf ? 0.f : __builtin_amdgcn_exp2f(at - both);
      const float y = other == -kInf ? 0.f : __builtin_amdgcn_exp2f(other - both);
      at = both;
      total = total * x + box[1] * y;
#pragma unroll
      for (int f = 0; f < NF; ++f)
#pragma unroll
        for (int i = 0; i < 8; ++i) o[0][f][i >> 2][i & 3] = o[0][f][i >> 2][i & 3] * x + box[2 + f * 8 + i] * y;
    }
    __syncthreads();
  }
  if (!active || turn_of || r >= CW || first_row + r > last_row) return;
  const int64_t total_rows = (int64_t)a.tokens * a.q_heads;   // of all heads
  const int64_t at_row = (int64_t)(w.start + row / a.group) * a.q_heads + head * a.group + row % a.group;
  float v[NF][8];
#pragma unroll
  for (int f = 0; f < NF; ++f)
#pragma unroll
    for (int i = 0; i < 8; ++i) v[f][i] = o[0][f][i & 1][i >> 1];
  if (a.splits > 1) {
    const int64_t slot = split * total_rows + at_row;
#pragma unroll
    for (int f = 0; f < NF; ++f) __builtin_memcpy(a.part + slot * DIM + 32 * f + 8 * g, v[f], sizeof(v[f]));
    if (g == 0) {
      float* ml = a.part + a.splits * total_rows * DIM + slot * 2;
      ml[0] = at;
      ml[1] = total;
    }
  } else {
    T* to_o = reinterpret_cast<T*>(a.out) + at_row * DIM;
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      T out[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) out[i] = D::from_f(total == 0.f ? 0.f : v[f][i] / total);
      __builtin_memcpy(to_o + 32 * f + 8 * g, out, sizeof(out));
    }
  }
}

// Parts of a row's tokens to its output, a row to a workgroup: a lane of the first wave weighs a part,
// then DIM / 4 lanes (four values each) take a part's values, in GROUPS whose sums meet in LDS.
constexpr int kMostSplits = 64;
template <class D, int DIM, int GROUPS>
__global__ void __launch_bounds__((GROUPS * DIM / 4 + 63) / 64 * 64)
kv4_attention_join(const float* __restrict__ part, int splits, int64_t rows, typename D::T* __restrict__ out) {
  constexpr int LANES = DIM / 4;
  __shared__ float weight[kMostSplits], box[GROUPS][4][LANES], sum_of_weights;
  const int64_t row = blockIdx.x;
  const int d = threadIdx.x % LANES, group = threadIdx.x / LANES;
  v4f v[2];   // under way while the weights are made
  auto load = [&](int s) { return *reinterpret_cast<const v4f*>(part + (s * rows + row) * DIM + d * 4); };
  const bool mine = group < GROUPS;
#pragma unroll
  for (int i = 0; i < 2; ++i) v[i] = mine && group + i * GROUPS < splits ? load(group + i * GROUPS) : v4f{0.f, 0.f, 0.f, 0.f};
  if (threadIdx.x < 64) {
    const int s = threadIdx.x;
    const float* ml = part + splits * rows * DIM + (s * rows + row) * 2;
    const float at = s < splits ? ml[0] : -kInf, total = s < splits ? ml[1] : 0.f;
    const float most = wave_max(at);
    const float w = at == -kInf ? 0.f : __builtin_amdgcn_exp2f(at - most);
    float sum = w * total;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    weight[s] = w;
    if (s == 0) sum_of_weights = sum;
  }
  __syncthreads();
  v4f sum = {0.f, 0.f, 0.f, 0.f};
  auto add = [&](int s, const v4f& x) {
    const float w = weight[s];
    if (w == 0.f) return;   // a part without tokens holds nothing
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[j] = fmaf(w, x[j], sum[j]);
  };
  if (mine) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (group + i * GROUPS < splits) add(group + i * GROUPS, v[i]);
#pragma unroll 4
    for (int s = group + 2 * GROUPS; s < splits; s += GROUPS) add(s, load(s));
#pragma unroll
    for (int j = 0; j < 4; ++j) box[group][j][d] = sum[j];
  }
  __syncthreads();
  if (group) return;
#pragma unroll
  for (int i = 1; i < GROUPS; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[j] += box[i][j][d];
  const float total = sum_of_weights;
  typename D::T t[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) t[j] = D::from_f(total == 0.f ? 0.f : sum[j] / total);
  __builtin_memcpy(out + row * DIM + d * 4, t, sizeof(t));
}

// The same of a few parts: DIM / 4 lanes have a row and weigh its parts themselves, 256 / (DIM / 4) rows to a workgroup.
constexpr int kFewSplits = 4;
template <class D, int DIM>
__global__ void __launch_bounds__(256)
kv4_attention_join_few(const float* __restrict__ part, int splits, int64_t rows, typename D::T* __restrict__ out) {
  constexpr int LANES = DIM / 4, ROWS = 256 / LANES;
  const int d = threadIdx.x % LANES;
  const int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / LANES;
  if ((int)threadIdx.x >= ROWS * LANES || row >= rows) return;
  float at[kFewSplits], total[kFewSplits], most = -kInf;
  v4f v[kFewSplits];
#pragma unroll
  for (int s = 0; s < kFewSplits; ++s) {
    const bool there = s < splits;
    const int64_t slot = there ? s * rows + row : row;
    const float* ml = part + splits * rows * DIM + slot * 2;
    at[s] = there ? ml[0] : -kInf;
    total[s] = ml[1];
    v[s] = *reinterpret_cast<const v4f*>(part + slot * DIM + d * 4);
    most = fmaxf(most, at[s]);
  }
  float all = 0.f;
  v4f sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < kFewSplits; ++s) {
    if (at[s] == -kInf) continue;   // a part without tokens holds nothing
    const float w = __builtin_amdgcn_exp2f(at[s] - most);
    all = fmaf(w, total[s], all);
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[j] = fmaf(w, v[s][j], sum[j]);
  }
  typename D::T t[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) t[j] = D::from_f(all == 0.f ? 0.f : sum[j] / all);
  __builtin_memcpy(out + row * DIM + d * 4, t, sizeof(t));
}

template <class F>
void with_dim(int dim, F&& f) {
  if (dim == 64) f(std::integral_constant<int, 64>{});
  else if (dim == 96) f(std::integral_constant<int, 96>{});
  else if (dim == 128) f(std::integral_constant<int, 128>{});
  else if (dim == 192) f(std::integral_constant<int, 192>{});
  else f(std::integral_constant<int, 256>{});
}

}  // namespace

}  // namespace qo

extern "C" int64_t qo_kv4_attention_workspace_size(const qo_kv4_cache* cache, int dtype, int64_t tokens, int q_heads,
                                                   int64_t table_width, int64_t sequences, int has_starts,
                                                   int64_t window) {
  using namespace qo;
  if (!cache || cache->kv_heads < 1 || tokens < 1 || q_heads < cache->kv_heads || sequences < 1) return 0;
  const Kv4Plan p = kv4_plan(tokens, q_heads, cache->kv_heads, cache->head_dim, table_width * cache->page_size,
                             sequences, has_starts != 0, window, dtype == QO_DTYPE_F32, device_cu_count());
  return p.splits > 1 ? p.splits * tokens * q_heads * (cache->head_dim + 2) * 4 : 0;
}

extern "C" int qo_kv4_attention(const qo_kv4_cache* cache, const qo_heads* q, int dtype, int64_t tokens, int q_heads,
                                const int32_t* page_table, int64_t table_ld, int64_t table_width,
                                const int32_t* lengths, const int32_t* q_starts, int64_t sequences, float scale,
                                int64_t window, void* out, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace qo;
  const char* fn = "qo_kv4_attention";
  KV4 c;
  const int st = kv4_cache(fn, cache, &c);
  if (st != QO_OK) return st;
  if (tokens < 0 || tokens > QO_KV4_MAX_TOKENS || sequences < 0 || sequences > QO_KV4_MAX_TOKENS || table_width < 0 ||
      table_width > INT32_MAX || table_ld < table_width) {
    qo_set_error("%s: invalid sizes tokens=%lld sequences=%lld table %lld wide, row stride %lld", fn, (long long)tokens,
                 (long long)sequences, (long long)table_width, (long long)table_ld);
    return QO_ERR_SHAPE;
  }
  if (q_heads < 1 || q_heads > 16384 || q_heads % c.heads != 0) {
    qo_set_error("%s: q_heads (%d) must be a multiple of kv_heads (%d)", fn, q_heads, c.heads);
    return QO_ERR_SHAPE;
  }
  if (!q_starts && (sequences == 0 ? tokens != 0 : tokens % sequences != 0)) {
    qo_set_error("%s: %lld queries of %lld sequences need q_starts", fn, (long long)tokens, (long long)sequences);
    return QO_ERR_SHAPE;
  }
  if (!(scale > 0.f && scale < 3.4e38f) || window < 0) {
    qo_set_error("%s: scale must be positive and window not negative, got %g and %lld", fn, (double)scale,
                 (long long)window);
    return QO_ERR_SHAPE;
  }
  if (dtype != QO_DTYPE_F32 && dtype != QO_DTYPE_F16 && dtype != QO_DTYPE_BF16) {
    qo_set_error("%s: unsupported dtype code %d", fn, dtype);
    return QO_ERR_DTYPE;
  }
  if (tokens == 0) return QO_OK;
  if (!q || !q->data || !out || (sequences && !lengths) || (sequences && table_width && !page_table)) {
    qo_set_error("%s: NULL pointer argument", fn);
    return QO_ERR_NULL_POINTER;
  }
  if (workspace && (uintptr_t)workspace % 16 != 0) {
    qo_set_error("%s: workspace must be 16-byte aligned", fn);
    return QO_ERR_ALIGNMENT;
  }
  Kv4Plan plan = kv4_plan(tokens, q_heads, c.heads, cache->head_dim, table_width * cache->page_size, sequences,
                          q_starts != nullptr, window, dtype == QO_DTYPE_F32, device_cu_count());
  if (plan.splits > 1 &&
      (!workspace || workspace_bytes < plan.splits * tokens * q_heads * (cache->head_dim + 2) * 4))
    plan.splits = 1;
  const int64_t grid = plan.tiles * c.heads * plan.splits;
  // rows of a KV head, threads (512 a workgroup at most) and a page's bytes take 32 bits
  if (tokens * (q_heads / c.heads) > (1 << 30) || grid > (1 << 23) - 1) {
    qo_set_error("%s: too many rows for one call (%lld queries of %d heads)", fn, (long long)tokens, q_heads);
    return QO_ERR_SHAPE;
  }
  if ((int64_t)c.heads * cache->page_size * cache->head_dim > INT32_MAX) {
    qo_set_error("%s: pages of %d tokens of %d heads are too large", fn, (int)cache->page_size, c.heads);
    return QO_ERR_SHAPE;
  }
  const Attention a = {c, q->data, q->token_stride, q->head_stride, out, page_table, table_ld,
                       c.pages ? (int)table_width : 0,   // without pages there is nothing to read
                       lengths, q_starts, (int)tokens, (int)sequences, sequences ? (int)(tokens / sequences) : 0, q_heads,
                       q_heads / c.heads, scale, window < kMostTokens ? (int)window : 0, (int)plan.tiles, plan.splits,
                       reinterpret_cast<float*>(workspace)};
  launch_begin();
  auto go = [&](auto d, auto parts_q, auto fine) {
    using D = decltype(d);
    constexpr int NQ = decltype(parts_q)::value;
    constexpr bool FINE = decltype(fine)::value;
    with_dim(cache->head_dim, [&](auto dim) {
      constexpr int DIM = decltype(dim)::value;
      hipStream_t s = reinterpret_cast<hipStream_t>(stream);
      auto attend = [&](auto kernel) { launch(kernel, dim3((unsigned)grid), dim3(256), 0, s, a); };
      if (plan.rows == 4) attend(kv4_attention_kernel<D, DIM, 4, NQ, FINE>);
      else if (plan.rows == 8) attend(kv4_attention_kernel<D, DIM, 2, NQ, FINE>);
      else if (plan.rows == 16) attend(kv4_attention_kernel<D, DIM, 1, NQ, FINE>);
      else kv4_prefill(a, dtype, DIM, 4 * plan.rows, grid, s);
      if (plan.splits > 1) {
        const int64_t rows = tokens * q_heads;
        const float* parts = reinterpret_cast<const float*>(workspace);
        auto* to = reinterpret_cast<typename D::T*>(out);
        constexpr int GROUPS = 8, ROWS = 256 / (DIM / 4);
        if (plan.splits <= kFewSplits)
          launch(kv4_attention_join_few<D, DIM>, dim3((unsigned)((rows + ROWS - 1) / ROWS)), dim3(256), 0, s, parts, plan.splits,
                 rows, to);
        else
          launch(kv4_attention_join<D, DIM, GROUPS>, dim3((unsigned)rows), dim3((GROUPS * DIM / 4 + 63) / 64 * 64), 0, s, parts,
                 plan.splits, rows, to);
      }
    });
  };
  using One = std::integral_constant<int, 1>;
  using Two = std::integral_constant<int, 2>;
  if (dtype == QO_DTYPE_BF16) go(BF16T{}, One{}, std::false_type{});
  else if (dtype == QO_DTYPE_F16) go(F16T{}, One{}, std::false_type{});
  else go(F32T{}, Two{}, std::true_type{});
  return launch_result(fn);
}
