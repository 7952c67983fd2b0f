// Attention over the 4-bit cache for sequences of many rows (prompts and their chunks), 16-bit types:
// the mathematics of kv4_attention.hip with the codes unpacked once for a workgroup.
//
// Waves of 32 rows share tiles of 64 tokens: while they multiply one, each unpacks a part of the next (its
// codes on their way to registers since a tile before) into the other half of LDS, as fragments of
// v_mfma_f32_32x32x16_f16 that a wave reads with consecutive 16-byte reads. Eight waves have two tiles of 128 rows:
// the first four one tile and the keys' unpacking, the others the tile that mirrors it from the sequence's end and
// the values' (half the unpacking a row, and under a causal mask every workgroup the same work); fewer rows, and head
// sizes whose outputs leave no room for two waves on a SIMD, have four. Fragments: lane
// l = r + 32 g of an operand holds eight consecutive k of row r, a lane of the result rows 8 m + 4 g + i
// (register 4 m + i) of column r. S^T = K Q^T (rows: 32 tokens), O^T += V^T P^T (rows: the even and then
// the odd values of 16 pairs): lane half g has tokens 8 m + 4 g + i of a tile's weights, in the order in which
// the values' fragments hold them, so that weights stay in their lanes.
//
// Codes less 8 are multiplied as they are, whatever a key's offset or outliers and a value's size: the parameters are applied to
// scores and weights in float32, as in kv4_attention.hip. They come from LDS as float32, and the power of two that brings weights
// times scales into fp16 stands in the exponent's argument. A weight is rounded to fp16 once for bf16 (half a step 2^-11, beside
// the output's 2^-8: 0.00167 of the outputs' norm where the output's rounding alone is 0.00166; a second part brings the two
// together and takes 190 us where one takes 161) and has two parts for fp16.
//
// A wave's 32 x 64 scores take 208 vector instructions and 32 exponentials beside 32 products (128 values,
// bf16), on the same SIMD: products run beside the other half's softmax, but the two overlap in part only. 2048
// queries of 32 heads on 4096 tokens (8 heads): of 128 164 us in bf16 (628 TFLOP/s of the pairs that a causal mask
// leaves, 52% of a large product's rate) and 195 in fp16, of 64 143 and 162. Keys and values unpacked to what they stand for
// in fp16 take the parameters out of the softmax (131 us in bf16), but a key's rounding then counts with its offset and
// outliers, in an exponent: twenty times the output's own for keys about 100.
#include "kv4_attention.h"

namespace qo {

namespace {

// A weight at the row's reference, in fp16, and how far (exponents) a larger score may pass the reference before
// sums and outputs move to it: each row's maximum grows now and then, some row's of 32 nearly every step.
constexpr int kAtRest = 6;
constexpr float kSlack = 8.f;

typedef float v16f __attribute__((ext_vector_type(16)));

template <class D, int DIM, int NP, int WAVES>
__global__ void __launch_bounds__(64 * WAVES, DIM <= 128 ? 2 : 1)
kv4_prefill_kernel(Attention a) {
  constexpr int NS = DIM / 16;        // k-steps of a score
  constexpr int NF = DIM / 32;        // blocks of 32 values
  constexpr int NW = DIM / 32;        // words of a key's codes that a lane unpacks
  constexpr int NV = (DIM / 2 + 63) / 64;   // pairs of values (16 tokens of each) that a lane unpacks
  constexpr int TILE = 32 * WAVES;
  using T = typename D::T;
  struct Stage {
    v4u k[2][NS][64];      // fragments: 32 tokens, k-step
    v4u v[NF][4][64];      // block of values, 16 tokens
    v4f params[4][2][8];   // keys' scale and middle, values' middle and scale; lane half g; its 32 tokens
    int largest[4];        // of 16 values' scales, the exponent's bits
  };
  __shared__ Stage stage[2];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 31, g = lane >> 5;
  const int heads = a.cache.heads;
  const int head = blockIdx.x % heads, split = blockIdx.x / heads / a.tiles;
  const Rows w = find_rows<TILE>(a, blockIdx.x / heads % a.tiles);
  if (!w.all) return;

  // Waves 0 .. 3 have one tile of 128 rows, 4 .. 7 another: its mirror image from the sequence's end, so that all
  // workgroups have the same work (with a window the next one, which sees the same tokens).
  const int tiles = (w.all + 127) / 128;
  int mine = w.index, other = w.index;
  if constexpr (WAVES == 8) {
    const int a_tile = a.window ? 2 * w.index : w.index, b_tile = a.window ? 2 * w.index + 1 : tiles - 1 - w.index;
    mine = wave < 4 ? b_tile : a_tile;
    other = wave < 4 ? a_tile : b_tile;
  }
  const bool active = mine * 128 + 32 * (wave & 3) < w.all && (wave < 4 || mine != other);
  const int first_row = min(mine * 128 + 32 * (wave & 3), w.all - 1), last_row = min(first_row + 31, w.all - 1);
  const int row = min(first_row + r, last_row);
  const Sees top = sees(a, w, first_row), bottom = sees(a, w, last_row), see = sees(a, w, row);
  const Sees all_top = sees(a, w, min(min(mine, other) * 128, w.all - 1));
  const Sees all_bottom = sees(a, w, min(max(mine, other) * 128 + 127, w.all - 1));

  // The query in fp16, brought to 2^14 .. 2^15, in the order in which a word gives a key's codes.
  v8h qf[NS];
  float factor, qsum;
  {
    const T* q = reinterpret_cast<const T*>(a.q) + (w.start + row / a.group) * a.q_token + (head * a.group + row % a.group) * a.q_head;
    T t[NS][8];
    float most = 0.f;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      __builtin_memcpy(t[s], q + (2 * s + g) * 8, sizeof(t[s]));
#pragma unroll
      for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(D::to_f(t[s][i])));
    }
    most = bits_float(halves_reduce(float_bits(most), FMax{}));
    const int e = query_exponent(most);
    float sum = 0.f;
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float v = ldexpf(D::to_f(t[s][kCodeOrder[i]]), e);
        sum += v;
        qf[s][i] = (_Float16)(kCodeOrder[i] & 1 ? v * 0.0625f : v);
      }
    sum = bits_float(halves_reduce(float_bits(sum), FAdd{}));
    qsum = most < kInf ? sum : __builtin_nanf("");   // an infinity's scores are NaN
    factor = score_factor(a.scale, e, 1.f);
  }

  v16f o[NF];
#pragma unroll
  for (int f = 0; f < NF; ++f)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[f][i] = 0.f;
  float most = -kInf, slope = factor, offset = 0.f, middles = 0.f;   // a weight is 2^(slope score + offset)
  float total = qsum != qsum && see.last > see.first ? qsum : 0.f;   // infinite queries: NaN, also where all scores are -inf
  int scale_exp = -14;   // every scale so far is below two to it
  bool far = false;      // some row's exponent is kFar or more

  auto exponent = [&](float score) { return score == -kInf ? 0.f : factor * score; };

  const int begin = all_top.first & ~63;
  const int steps = all_bottom.last > begin ? (all_bottom.last - begin + 63) / 64 : 0;
  const int per_split = (steps + a.splits - 1) / a.splits;
  const int from = split * per_split, to = min(from + per_split, steps);
  const int32_t* table = a.table + (w.b < a.sequences ? w.b : 0) * a.table_ld;
  const Pages pages(a.cache, head, DIM);
  const uint32_t exponents = exponents_of_1024();

  // Unpacking: wave i takes tile i % 4 of a step's four tiles of 16 tokens, of eight waves the first its keys and
  // the others its values. Keys: lane c + 16 d token c, words NW d ..;
  // values: a lane the 16 tokens of pair `lane` (+ 64).
  const int c = lane & 15, d = lane >> 4, part = wave & 3;
  const bool keys = WAVES == 4 || wave < 4, values_too = WAVES == 4 || wave >= 4;
  uint32_t kw[NW], key_s, key_lo, value_s, value_lo;   // the lane's token's parameters (16 bits)
  v4u vw[NV];
  Tile tile;
  bool bad = false;
  auto find = [&](int step) { tile = tile_at(a, table, begin + 64 * step + 16 * part); };
  auto load = [&] {
    bad = tile.bad;
    const uint8_t* kp = pages.k + (uint64_t)(uint32_t)tile.page * pages.codes + ((tile.place + c) * (DIM / 2) + d * (4 * NW));
    const uint8_t* vp = pages.v + (uint64_t)(uint32_t)tile.page * pages.codes + (tile.place * (DIM / 2) + lane * 16);
    const uint8_t* par = pages.params + (uint64_t)(uint32_t)tile.page * pages.param_bytes + tile.place * 4;
    if (keys) __builtin_memcpy(kw, kp, sizeof(kw));
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (values_too && 64 * i + lane < DIM / 2) vw[i] = *reinterpret_cast<const v4u*>(vp + 1024 * i);
    if (keys) {
      const uint16_t* ks = reinterpret_cast<const uint16_t*>(par) + c;
      const uint16_t* vs = reinterpret_cast<const uint16_t*>(par + pages.param_values) + c;
      key_s = ks[0], key_lo = ks[16], value_s = vs[0], value_lo = vs[16];
    }
  };
  auto unpack = [&](Stage& st, int step) {
    if (keys) {
#pragma unroll
      for (int i = 0; i < NW; ++i) {
        const int word = d * NW + i;   // of the token's row: dims 8 word ..
        const uint32_t x = kw[i], h = x >> 8;
        st.k[part >> 1][word >> 1][(part & 1) * 16 + c + 32 * (word & 1)] =
            (v4u){less_low(x, exponents), less_high(x, exponents), less_low(h, exponents), less_high(h, exponents)};
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (values_too && 64 * i + lane < DIM / 2) {
        const int pair = 64 * i + lane;
        v4u even[2], odd[2];   // of lane half g: tokens 4 g .. and 8 + 4 g ..
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int h = 0; h < 2; ++h) {   // tokens 4 q + 2 h, and the next
            const uint32_t two = __builtin_amdgcn_perm(0, vw[i][q], h ? 0x0C030C02u : 0x0C010C00u);
            even[q & 1][2 * (q >> 1) + h] = less_low(two, exponents);
            odd[q & 1][2 * (q >> 1) + h] = less_high(two, exponents);
          }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          st.v[pair >> 4][part][(pair & 15) + 32 * h] = even[h];
          st.v[pair >> 4][part][(pair & 15) + 16 + 32 * h] = odd[h];
        }
      }
    // The parameters, as float32: of token 16 part + c of the step, of lane half (c / 4) % 2 its token 8 part + 4 (c / 8) + c % 4.
    if (keys && d == 0) {
      // A value that is no number (or on a page outside the cache) becomes 0 and its key NaN: the rows that see the
      // token are NaN then, and the others are not. Values that no row sees are 0 too: they have no say in S.
      const bool finite = (value_s & 0x7C00u) != 0x7C00u && (value_lo & 0x7C00u) != 0x7C00u && !bad;
      if (!finite) key_s = key_lo = 0x7E00u;
      const int t = begin + 64 * step + 16 * part + c;
      if (!(finite && t >= all_top.first && t < all_bottom.last)) value_s = value_lo = 0u;
      const int half_of_c = c >> 2 & 1, place = 8 * part + 4 * (c >> 3) + (c & 3);
      auto put = [&](int which, float x) { reinterpret_cast<float*>(&st.params[which][half_of_c][0])[place] = x; };
      const float ks = half_of(&key_s, 0), vs = half_of(&value_s, 0);
      put(0, ks);
      put(1, fmaf(8.f, ks, half_of(&key_lo, 0)));
      put(2, fmaf(8.f, vs, half_of(&value_lo, 0)));
      put(3, vs);
      uint32_t top_of = value_s & 0x7FFFu;
      auto with = [&](int other) { top_of = max(top_of, (uint32_t)other); };
      with(__builtin_amdgcn_update_dpp(0, (int)top_of, 0xB1, 0xF, 0xF, false));    // quad_perm 1,0,3,2
      with(__builtin_amdgcn_update_dpp(0, (int)top_of, 0x4E, 0xF, 0xF, false));    // quad_perm 2,3,0,1
      with(__builtin_amdgcn_update_dpp(0, (int)top_of, 0x141, 0xF, 0xF, false));   // row_half_mirror
      with(__builtin_amdgcn_update_dpp(0, (int)top_of, 0x140, 0xF, 0xF, false));   // row_mirror
      if (c == 0) st.largest[part] = (int)(top_of >> 10);
    }
  };

  if (from < to) {
    find(from);
    load();
    find(from + 1);
    unpack(stage[0], from);
    if (from + 1 < to) {
      load();
      find(from + 2);
    }
    lds_barrier();
  }
  for (int step = from; step < to; ++step) {
    const Stage& st = stage[(step - from) & 1];
    if (step + 1 < to) {
      unpack(stage[(step - from + 1) & 1], step + 1);
      if (step + 2 < to) {
        load();
        find(step + 3);
      }
    }
    const int t0 = begin + 64 * step;
    if (active && t0 < bottom.last && t0 + 64 > top.first) {
      v16f sc[2];
      v8h ph[4], pl[4];
      // The scores of 32 tokens.
      auto scores = [&](int u) {
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[u][i] = 0.f;
#pragma unroll
        for (int k = 0; k < NS; ++k)
          sc[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, st.k[u][k][lane]), qf[k], sc[u], 0, 0, 0);
      };
      // Their weights' product with the values.
      auto values = [&](int u) {
#pragma unroll
        for (int f = 0; f < NF; ++f)
#pragma unroll
          for (int i = 2 * u; i < 2 * u + 2; ++i) {
            const v8h v = __builtin_bit_cast(v8h, st.v[f][i][lane]);
            o[f] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, ph[i], o[f], 0, 0, 0);
            if constexpr (NP > 1) o[f] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, pl[i], o[f], 0, 0, 0);
          }
      };
      float shrink_o = 1.f;
      // A parameter of the lane's 16 tokens of a half.
      auto params = [&](int which, int u, float(&x)[16]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const v4f four = st.params[which][g][4 * u + i];
#pragma unroll
          for (int j = 0; j < 4; ++j) x[4 * i + j] = four[j];
        }
      };
      // Parameters, masks and the largest score; sums follow a larger one, and outputs do in rescale(), once the
      // weights made before it are in them.
      auto largest = [&](int u) {
        float ks[16], middle[16];
        params(0, u, ks);
        params(1, u, middle);
#pragma unroll
        for (int t = 0; t < 16; ++t) sc[u][t] = fmaf(ks[t], sc[u][t], middle[t] * qsum);
        const int field = max(st.largest[2 * u], st.largest[2 * u + 1]);
        const int exp_now = max(scale_exp, __builtin_amdgcn_readfirstlane(field) - 14);
        if (!(t0 + 32 * u + 32 <= top.last && t0 + 32 * u >= bottom.first)) {   // some row does not see some token
#pragma unroll
          for (int t = 0; t < 16; ++t) {
            const int at_t = t0 + 32 * u + t / 4 * 8 + 4 * g + t % 4;
            if (at_t < see.first || at_t >= see.last) sc[u][t] = -kInf;
          }
        }
        float now = -kInf;
#pragma unroll
        for (int t = 0; t < 16; ++t) now = fmaxf(now, sc[u][t]);
        now = bits_float(halves_reduce(float_bits(now), FMax{}));
        if (__any(factor * (now - most) > kSlack) || exp_now > scale_exp || far) {
          now = fmaxf(now, most);
          const float at = exponent(most), next = exponent(now), rest = (float)(kAtRest - exp_now);
          const bool now_far = __any(fabsf(next) >= kFar);
          const float by = far || now_far ? (at - next) + (float)(scale_exp - exp_now) : (rest - next) - offset;
          shrink_o = most == -kInf ? 1.f : __builtin_amdgcn_exp2f(by);   // before: all sums 0
          most = now;
          slope = now_far ? 1.f : factor;
          offset = now_far ? rest : rest - next;
          far = now_far;
          total *= shrink_o;
          middles *= shrink_o;
          scale_exp = exp_now;
          if (far) {
#pragma unroll
            for (int t = 0; t < 16; ++t) sc[u][t] = factor * sc[u][t] - next;
          }
          return true;
        }
        return false;
      };
      auto rescale = [&](bool larger) {
        if (larger) {
#pragma unroll
          for (int f = 0; f < NF; ++f) o[f] *= shrink_o;
        }
        __builtin_amdgcn_sched_barrier(0);
      };
      auto weights = [&](int u) {
        float middle[16], vs[16];
        params(2, u, middle);
        params(3, u, vs);
#pragma unroll
        for (int t = 0; t < 16; ++t) {
          const float p = __builtin_amdgcn_exp2f(fmaf(slope, sc[u][t], offset));
          total += p;
          middles = fmaf(p, middle[t], middles);
          _Float16 h = (_Float16)fmaf(p, vs[t], 0.f);
          if constexpr (NP > 1) {
            asm("" : "+v"(h));   // one and the same rounding in both parts
            pl[2 * u + t / 8][t % 8] = (_Float16)fmaf(p, vs[t], -(float)h);
          }
          ph[2 * u + t / 8][t % 8] = h;
        }
        // here and not where the product takes them
#pragma unroll
        for (int i = 2 * u; i < 2 * u + 2; ++i) {
          asm volatile("" : "+v"(ph[i]));
          if constexpr (NP > 1) asm volatile("" : "+v"(pl[i]));
        }
      };
      // Products of one half beside the softmax of the other: reads of four fragments, then a product, a read and
      // some VALU instructions in turn.
      auto beside = [&](auto products, auto valu) {
        constexpr int N = decltype(products)::value, V = decltype(valu)::value;
        __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
          if (V) {
            __builtin_amdgcn_sched_group_barrier(0x002, V, 0);
            __builtin_amdgcn_sched_group_barrier(0x400, 2, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, V, 0);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      };
      scores(0);
      beside(std::integral_constant<int, NS>{}, std::integral_constant<int, 0>{});
      rescale(largest(0));
      scores(1);
      weights(0);
      beside(std::integral_constant<int, NS>{}, std::integral_constant<int, 3>{});
      const bool larger = largest(1);
      __builtin_amdgcn_sched_barrier(0);
      values(0);
      weights(1);
      beside(std::integral_constant<int, 2 * NF * NP>{}, std::integral_constant<int, 3>{});
      rescale(larger);
      values(1);
      beside(std::integral_constant<int, 2 * NF * NP>{}, std::integral_constant<int, 0>{});
    }
    lds_barrier();
  }
  if (!active) return;

  total = bits_float(halves_reduce(float_bits(total), FAdd{}));
  middles = bits_float(halves_reduce(float_bits(middles), FAdd{}));
  // The sums are in units of 2^at, or else of 2^(at - offset).
  float at = far ? exponent(most) : -offset;
  const float unit = far ? power_of_two(scale_exp - kAtRest) : 1.f;
  if (most == -kInf && total == 0.f) at = -kInf;
  if (w.poison) total = __builtin_nanf(""), at = 0.f;
  if (first_row + r > last_row) return;
  const int64_t total_rows = (int64_t)a.tokens * a.q_heads;   // of all heads
  const int64_t at_row = (int64_t)(w.start + row / a.group) * a.q_heads + head * a.group + row % a.group;
#pragma unroll
  for (int f = 0; f < NF; ++f)
#pragma unroll
    for (int m = 0; m < 2; ++m) {   // values 32 f + 16 m + 8 g ..: pairs 16 f + 8 m + 4 g + i
      float v[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = o[f][4 * m + i] + middles;
        v[2 * i + 1] = fmaf(o[f][8 + 4 * m + i], 0.0625f, middles);
      }
      if (a.splits > 1) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= unit;
        __builtin_memcpy(a.part + (split * total_rows + at_row) * DIM + 32 * f + 16 * m + 8 * g, v, sizeof(v));
      } else {
        T out[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) out[i] = D::from_f(total == 0.f ? 0.f : v[i] / total);
        __builtin_memcpy(reinterpret_cast<T*>(a.out) + at_row * DIM + 32 * f + 16 * m + 8 * g, out, sizeof(out));
      }
    }
  if (a.splits > 1 && g == 0) {
    float* ml = a.part + a.splits * total_rows * DIM + (split * total_rows + at_row) * 2;
    ml[0] = at;
    ml[1] = total * unit;
  }
}

}  // namespace

void kv4_prefill(const Attention& a, int dtype, int dim, int tile, int64_t grid, hipStream_t stream) {
  auto go = [&](auto n) {
    constexpr int DIM = decltype(n)::value;
    auto attend = [&](auto kernel) { launch(kernel, dim3((unsigned)grid), dim3(2 * tile), 0, stream, a); };
    const bool bf16 = dtype == QO_DTYPE_BF16;
    if constexpr (DIM <= 128) {
      if (tile == 256) return bf16 ? attend(kv4_prefill_kernel<BF16T, DIM, 1, 8>) : attend(kv4_prefill_kernel<F16T, DIM, 2, 8>);
    }
    if (bf16) attend(kv4_prefill_kernel<BF16T, DIM, 1, 4>);
    else attend(kv4_prefill_kernel<F16T, DIM, 2, 4>);
  };
  if (dim == 64) go(std::integral_constant<int, 64>{});
  else if (dim == 96) go(std::integral_constant<int, 96>{});
  else if (dim == 128) go(std::integral_constant<int, 128>{});
  else if (dim == 192) go(std::integral_constant<int, 192>{});
  else go(std::integral_constant<int, 256>{});
}

}  // namespace qo
