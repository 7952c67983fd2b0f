// The 4-bit key/value cache of qo_kv4_cache: one vector of D values per token and KV head,
// v read as lo + s c with c = 0 .. 15, s and lo in fp16. Pages of P tokens:
//
//   k_codes  [pages, heads, P, D/2]         a token's codes in a row: a product over the values
//                                           of a vector reads 16 bytes of a token at a time
//   v_codes  [pages, heads, P/16, D/2, 16]  16 tokens of a pair of values in a row: a product
//                                           over tokens reads 16 bytes of a pair, and appending a
//                                           token changes whole bytes
//   params   [pages, 2, heads, P/16, 2, 16] the 16 scales and the 16 minima of a tile of tokens
#pragma once

#include "common.h"

namespace qo {

constexpr float kKV4Most = 65504.f;   // values are clamped to fp16's range

struct KV4 {
  uint8_t* k;
  uint8_t* v;
  _Float16* params;
  int64_t pages;
  int shift;   // log2 of the page size
  int heads;

  __device__ inline int64_t slots() const { return pages << shift; }
  // Token `place` of a page: its key's codes, its value's tile (16 tokens) and its tiles of parameters.
  __device__ inline uint8_t* key(int64_t page, int head, int place, int dim) const {
    return k + (((page * heads + head) << shift) + place) * (dim / 2);
  }
  __device__ inline uint8_t* value_tile(int64_t page, int head, int place, int dim) const {
    return v + (((page * heads + head) << (shift - 4)) + (place >> 4)) * (dim * 8);
  }
  __device__ inline _Float16* param_tile(int64_t page, int which, int head, int place) const {
    return params + ((((page * 2 + which) * heads + head) << (shift - 4)) + (place >> 4)) * 32;
  }
};

// Vectors [tokens, heads, D] with unit inner stride.
template <class T>
struct Heads {
  const T* data;
  int64_t token, head;
  __device__ inline const T* at(int64_t t, int h) const { return data + t * token + h * head; }
};

inline bool kv4_head_dim(int d) { return d == 64 || d == 96 || d == 128 || d == 192 || d == 256; }

// The cache's sizes and pointers as an entry point's call has them; QO_OK with *out set.
int kv4_cache(const char* fn, const qo_kv4_cache* cache, KV4* out);

}  // namespace qo
