// What the kernels of attention over the 4-bit cache (kv4_attention.hip, kv4_prefill.hip) share:
// their arguments, where a workgroup's rows and tokens are, codes as fp16, reductions.
//
// A row is one query of one of the heads that share a KV head: row i of a sequence is its query
// i / group, head i % group.
#pragma once

#include "kv4_common.h"

namespace qo {

typedef unsigned v4u __attribute__((ext_vector_type(4)));
typedef unsigned v2u __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.44269504f;
constexpr float kInf = __builtin_inff();
constexpr int kMostTokens = 0x7FFFF000;   // of a sequence: positions take 32 bits, those a few steps ahead too

struct Attention {
  KV4 cache;
  const void* q;
  int64_t q_token, q_head;
  void* out;
  const int32_t* table;
  int64_t table_ld;
  int width;                  // pages of a row of the table
  const int32_t* lengths;
  const int32_t* q_starts;    // or null: `each` queries a sequence
  int tokens, sequences, each;
  int q_heads, group;
  float scale;
  int window;                 // 0: none
  int tiles;                  // row tiles of all sequences
  int splits;
  float* part;                // [splits][tokens * q_heads][DIM], then [splits][tokens * q_heads][2]
};

__device__ inline float bits_float(uint32_t u) { return __builtin_bit_cast(float, u); }
__device__ inline uint32_t float_bits(float f) { return __builtin_bit_cast(uint32_t, f); }
__device__ inline float power_of_two(int e) { return bits_float((uint32_t)(127 + e) << 23); }
__device__ inline float half_of(const uint32_t* pairs, int t) {
  const uint32_t w = pairs[t / 2];
  return (float)__builtin_bit_cast(v2h, w)[t & 1];
}
__device__ inline uint32_t pk_max_u16(uint32_t a, uint32_t b) {
  typedef unsigned short v2u16 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(v2u16, a), __builtin_bit_cast(v2u16, b)));
}

struct FMax {
  __device__ uint32_t operator()(uint32_t a, uint32_t b) const { return float_bits(fmaxf(bits_float(a), bits_float(b))); }
};
struct FAdd {
  __device__ uint32_t operator()(uint32_t a, uint32_t b) const { return float_bits(bits_float(a) + bits_float(b)); }
};
struct UMax {
  __device__ uint32_t operator()(uint32_t a, uint32_t b) const { return max(a, b); }
};
// Over lanes l and l + 32, and over lanes r, r + 16, r + 32, r + 48.
template <class F>
__device__ inline uint32_t halves_reduce(uint32_t u, F f) {
  const v2u a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return f(a[0], a[1]);
}
template <class F>
__device__ inline uint32_t groups_reduce(uint32_t u, F f) {
  const uint32_t w = halves_reduce(u, f);
  const v2u b = __builtin_amdgcn_permlane16_swap(w, w, false, false);
  return f(b[0], b[1]);
}

// Codes less 8 as fp16 (those at bits 4 .. 7 times 16): with the exponent of 1024 in front, an
// fp16's lowest bits count in ones.
constexpr uint32_t kLow = 0x000F000Fu, kHigh = 0x00F000F0u;
__device__ inline uint32_t less(uint32_t w, uint32_t mask, uint32_t exponents, _Float16 n) {
  const v2h v = __builtin_bit_cast(v2h, (w & mask) | exponents) - (v2h){n, n};
  return __builtin_bit_cast(uint32_t, v);
}
__device__ inline uint32_t less_low(uint32_t w, uint32_t e) { return less(w, kLow, e, (_Float16)1032.f); }
__device__ inline uint32_t less_high(uint32_t w, uint32_t e) { return less(w, kHigh, e, (_Float16)1152.f); }
// The exponents in a vector register: a mask and they are then one instruction's operands.
__device__ inline uint32_t exponents_of_1024() {
  uint32_t e = 0x64006400u;
  asm("" : "+v"(e));
  return e;
}
constexpr int kCodeOrder[8] = {0, 4, 1, 5, 2, 6, 3, 7};   // of a word's codes, as masks and shifts by 8 take them out

// Where a workgroup's rows are: sequence b (or, b = sequences, behind the last), whose queries are start .. start +
// count - 1, and the number `index` of its tiles of TILE rows (below 0 or past the last: nothing). Tiles of ragged
// sequences are counted from q_starts[b] * group / TILE + b on, which leaves room for every one's last.
struct Rows {
  int b, start, count, index, all, length;   // all: rows of the sequence
  bool poison;                               // the sequence is longer than its row of the table
};
template <int TILE>
__device__ inline Rows find_rows(const Attention& a, int tile) {
  Rows w;
  auto begin_of = [&](int i) {   // sequence 0 starts at 0
    const int s = i == 0 ? 0 : a.q_starts[i];
    return s < 0 ? 0 : s > a.tokens ? a.tokens : s;
  };
  if (a.q_starts) {
    int n = 0;
    for (int base = 0; base <= a.sequences; base += 64) {
      const int i = base + (int)(threadIdx.x & 63);
      const bool before = i <= a.sequences && begin_of(i) * a.group / TILE + i <= tile;
      const int got = __popcll(__ballot(before));
      n += got;
      if (got < 64) break;
    }
    w.b = n - 1;
    w.start = begin_of(w.b);
    const int end = w.b < a.sequences ? begin_of(w.b + 1) : a.tokens;
    w.count = end > w.start ? end - w.start : 0;
    w.index = tile - (w.start * a.group / TILE + w.b);   // below 0: q_starts that do not ascend
  } else {
    const int per = (a.each * a.group + TILE - 1) / TILE;
    w.b = tile / per;
    w.start = w.b * a.each;
    w.count = a.each;
    w.index = tile % per;
  }
  w.all = w.count * a.group;
  if (w.index < 0 || (int64_t)w.index * TILE >= w.all) w.all = 0;
  w.length = w.all && w.b < a.sequences ? a.lengths[w.b] : 0;
  const int shift = a.cache.shift, pages = w.length >> shift;
  w.poison = w.length > kMostTokens || pages > a.width || (pages == a.width && (w.length & ((1 << shift) - 1)));
  if (w.length < 0 || w.poison) w.length = 0;
  return w;
}

// The first token that a row sees and the one after the last.
struct Sees {
  int first, last;
};
__device__ inline Sees sees(const Attention& a, const Rows& w, int row) {
  const int p = w.length - w.count + row / a.group;
  return Sees{a.window && p + 1 > a.window ? p + 1 - a.window : 0, w.length && p >= 0 ? p + 1 : 0};
}

// One head's pages: where page 0 starts and the bytes from page to page (below 2^32: the host's check).
struct Pages {
  const uint8_t* k;
  const uint8_t* v;
  const uint8_t* params;   // of keys; those of values stand param_values further
  uint32_t codes, param_bytes, param_values;

  __device__ Pages(const KV4& c, int head, int dim)
      : k(c.k + ((int64_t)head << c.shift) * (dim / 2)),
        v(c.v + ((int64_t)head << c.shift) * (dim / 2)),
        params(reinterpret_cast<const uint8_t*>(c.params) + ((int64_t)head << (c.shift - 4)) * 64),
        codes((uint32_t)(c.heads << c.shift) * (dim / 2)),
        param_bytes((uint32_t)(c.heads << (c.shift - 4)) * 128),
        param_values(param_bytes / 2) {}
};

// Where a tile of 16 tokens stands: its page (0 for one outside the cache) and the place of its first token.
struct Tile {
  int page, place;
  bool bad;
};
__device__ inline Tile tile_at(const Attention& a, const int32_t* table, int t) {
  const int at = t >> a.cache.shift;
  const int page = at < a.width ? table[at] : 0;   // beyond: past the tokens, masked
  const bool bad = page < 0 || page >= (int)a.cache.pages;
  return {bad ? 0 : page, t & ((1 << a.cache.shift) - 1), bad};
}

// A weight is 2^(factor x - at), at the rounded factor x of the row's largest score, by one fma. It is 1 for that score, up
// to at's rounding, which is the same for all of a row's weights and at most 2^-3 below kFar. From there on the
// products are rounded before the difference, as at is.
constexpr float kFar = 0x1p22f;

// The power of two that brings a row's largest magnitude into [2^14, 2^15).
__device__ inline int query_exponent(float most) { return most > 0.f && most < kInf ? 15 - __builtin_amdgcn_frexp_expf(most) : 0; }

// What brings such a row's scores, times `unit`, to exponents of two. 0 would make no number of a masked score, and
// no exponent below 2^-80 differs from 0; an infinite one would make none of a score of 0, and at the largest
// number any two scores that differ are as far apart as they need to be.
__device__ inline float score_factor(float scale, int e, float unit) {
  return fminf(fmaxf(ldexpf(scale, -e) * kLog2e * unit, 0x1p-126f), 0x1.fffffep127f);
}

// Starts the kernel for many rows a sequence (16-bit types), in tiles of 128 or 256; the grid is that of kv4_plan.
void kv4_prefill(const Attention& a, int dtype, int dim, int tile, int64_t grid, hipStream_t stream);

}  // namespace qo
