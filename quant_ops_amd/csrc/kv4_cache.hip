// Appending keys and values to the 4-bit cache of kv4_common.h, with the position rotation on
// the way, and reading them back.
#include "kv4_common.h"

namespace qo {

int kv4_cache(const char* fn, const qo_kv4_cache* c, KV4* out) {
  if (!c) {
    qo_set_error("%s: NULL cache", fn);
    return QO_ERR_NULL_POINTER;
  }
  if (!kv4_head_dim(c->head_dim)) {
    qo_set_error("%s: head_dim must be 64, 96, 128, 192 or 256, got %d", fn, (int)c->head_dim);
    return QO_ERR_SHAPE;
  }
  const int p = c->page_size;
  if (p < 16 || p > QO_KV4_MAX_PAGE || (p & (p - 1))) {
    qo_set_error("%s: page_size must be a power of two from 16 to %d, got %d", fn, QO_KV4_MAX_PAGE, p);
    return QO_ERR_SHAPE;
  }
  if (c->pages < 0 || c->pages > INT32_MAX || c->kv_heads < 1 || c->kv_heads > 16384) {
    qo_set_error("%s: invalid sizes pages=%lld kv_heads=%d", fn, (long long)c->pages, (int)c->kv_heads);
    return QO_ERR_SHAPE;
  }
  if (c->pages && (!c->k_codes || !c->v_codes || !c->params)) {
    qo_set_error("%s: NULL pointer in the cache", fn);
    return QO_ERR_NULL_POINTER;
  }
  if (((uintptr_t)c->k_codes | (uintptr_t)c->v_codes | (uintptr_t)c->params) % 16 != 0) {
    qo_set_error("%s: the cache's pointers must be 16-byte aligned", fn);
    return QO_ERR_ALIGNMENT;
  }
  int shift = 4;
  while ((1 << shift) < p) ++shift;
  *out = {reinterpret_cast<uint8_t*>(c->k_codes), reinterpret_cast<uint8_t*>(c->v_codes),
          reinterpret_cast<_Float16*>(c->params), c->pages, shift, c->kv_heads};
  return QO_OK;
}

namespace {

// Lanes of a vector: eight values each, a power of two of them (those past the vector idle).
template <int DIM>
constexpr int kLanes = DIM <= 64 ? 8 : DIM <= 128 ? 16 : 32;

// Over the LANES lanes of a vector.
template <int LANES, class F>
__device__ inline float lanes_reduce(float v, F&& f) {
  auto with = [&](int other) { v = f(v, __builtin_bit_cast(float, other)); };
  with(__builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0xB1, 0xF, 0xF, false));    // quad_perm 1,0,3,2
  with(__builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x4E, 0xF, 0xF, false));    // quad_perm 2,3,0,1
  with(__builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x141, 0xF, 0xF, false));   // row_half_mirror
  if constexpr (LANES > 8) with(__builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x140, 0xF, 0xF, false));   // row_mirror
  if constexpr (LANES > 16) with(__builtin_amdgcn_ds_swizzle(__builtin_bit_cast(int, v), 0x401F));   // lanes 16 apart
  return v;
}

// A token's rotation: angles of position p, or NaN where the table does not reach.
struct Angles {
  const int64_t* positions;
  const float* cos_;
  const float* sin_;
  int64_t rows;
  int rot;
};

// Eight values of a vector and where they stand: `at` the first four, `more` the others. In
// the rotated part a lane has four pairs.
struct Place {
  int at, more;
  bool turned;
};
template <bool PAIRS>
__device__ inline Place place_of(int lane, int rot) {
  if (8 * lane >= rot || PAIRS) return {8 * lane, 8 * lane + 4, 8 * lane < rot};
  return {4 * lane, rot / 2 + 4 * lane, true};
}

// (a, b) -> (a cos - b sin, b cos + a sin). A product of two float32 is exact in 64 bits, so
// the results are the formula's, rounded to 64 bits and then to 32: whoever computes it in
// 64 bits gets the same codes.
__device__ inline void turn(float& a, float& b, double c, double s) {
  const double x = (double)a * c - (double)b * s, y = (double)b * c + (double)a * s;
  a = (float)x;
  b = (float)y;
}

// Codes of a vector's eight values (in the low bytes of words: two by two) and its parameters. A code is the whole number
// nearest to an estimate (v - lo) / s, which is off by 2^-18 at most (15 1/2 times the difference's 2^-24 and the scale's
// reciprocal's 2^-23), unless that lies within 2^-17 of a border between codes or outside them. There (one value in 10^5,
// exact ties, vectors whose size is far above their range) 64 bits decide: with n the whole number below the border,
// v - lo against s (n + 1/2), which is exact but for the difference's rounding to 64 bits (where v is below 2^-29 of lo).
template <int LANES>
__device__ inline void quantize(const float (&v)[8], bool there, uint32_t (&two)[4], _Float16& scale, _Float16& least) {
  float lo = v[0], hi = v[0];   // hi: NaN for a NaN
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    lo = fminf(lo, v[i]);
    hi = __builtin_elementwise_maximum(hi, v[i]);
  }
  if (!there) lo = __builtin_inff(), hi = -__builtin_inff();
  lo = lanes_reduce<LANES>(lo, [](float a, float b) { return fminf(a, b); });
  hi = lanes_reduce<LANES>(hi, [](float a, float b) { return __builtin_elementwise_maximum(a, b); });
  const bool finite = lo > -__builtin_inff() && hi < __builtin_inff();
  lo = fmaxf(lo, -kKV4Most);
  hi = fminf(hi, kKV4Most);
  least = (_Float16)fminf(lo, kKV4Most);
  const float l = (float)least;
  const double d = (double)fmaxf(hi, -kKV4Most) - (double)l, q = d * (1.0 / 15.0);
  const float range = (float)fma(fma(-15.0, q, d), 1.0 / 15.0, q);   // the quotient, rounded to float32, then to fp16
  scale = (_Float16)fmaxf(range, 0.f);
  const float s = (float)scale;
  const float inverse = s > 0.f ? __builtin_amdgcn_rcpf(s) : 0.f;
  constexpr float kRound = 12582912.f;   // 1.5 2^23: a sum with it is a whole number, in its low bits
  float near = 0.f, m[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float x = v[i] - l;
    m[i] = fmaf(x, inverse, kRound);
    near = fmaxf(near, fabsf(fmaf(x, inverse, -(m[i] - kRound))));
  }
  // beyond a border lies what is above 15 1/2 or below -1/2, values past fp16 among them
  const float high = fmaxf((hi - l) * inverse - 15.f, (l - lo) * inverse);
  if (__any(!(fmaxf(near, high) < 0.5f - 0x1p-17f) || !finite || s == 0.f || hi == kKV4Most || lo == -kKV4Most)) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float u = __builtin_amdgcn_fmed3f(v[i], -kKV4Most, kKV4Most);
      const float n = floorf(__builtin_amdgcn_fmed3f((u - l) * inverse, 0.f, 15.f));
      const double over = ((double)u - (double)l) - (double)s * ((double)n + 0.5);
      const bool up = over > 0.0 || (over == 0.0 && ((int)n & 1));
      m[i] = (s > 0.f && finite ? fminf(n + (up ? 1.f : 0.f), 15.f) : 0.f) + kRound;
    }
    if (!finite) scale = least = (_Float16)__builtin_nanf("");
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    two[i] = __builtin_bit_cast(uint32_t, m[2 * i + 1]) << 4 | __builtin_bit_cast(uint32_t, m[2 * i]);
}

// Where values' bytes of TOKENS tokens go from a box in LDS: a thread has a byte (a pair of values) of four
// tokens, which share a word of the cache where their slots do; four threads have 16 tokens of a pair, so that
// single bytes too go to whole lines. A head's bytes stand head_bytes behind those of the head before.
template <int DIM, int TOKENS>
struct ValueBytes {
  uint8_t* at[4];   // null: no such token
  bool beside, there;
  int pair, t;
  int64_t head_bytes;

  __device__ ValueBytes(const KV4& cache, int head, const int64_t* token_slots) {
    pair = threadIdx.x / (TOKENS / 4), t = 4 * (threadIdx.x % (TOKENS / 4));
    there = pair < DIM / 2;
    head_bytes = (int64_t)DIM / 2 << cache.shift;
    const int64_t first = token_slots[t];
    beside = there && first >= 0 && (first & 3) == 0;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int64_t slot = token_slots[t + n];
      const int place = (int)(slot & ((1 << cache.shift) - 1));
      at[n] = there && slot >= 0 ? cache.value_tile(slot >> cache.shift, head, place, DIM) + pair * 16 + (place & 15) : nullptr;
      beside = beside && slot == first + n;
    }
  }
  __device__ inline void next_head() {
#pragma unroll
    for (int n = 0; n < 4; ++n)
      if (at[n]) at[n] += head_bytes;
  }
  __device__ inline void put(uint32_t four) const {
    if (beside) {
      *reinterpret_cast<uint32_t*>(at[0]) = four;
    } else {
#pragma unroll
      for (int n = 0; n < 4; ++n)
        if (at[n]) *at[n] = (uint8_t)(four >> (8 * n));
    }
  }
};

// A workgroup of 256 threads takes 256 / LANES consecutive tokens of `per` heads in turn, of the queries, the keys or the
// values (blockIdx.y counts groups of heads); a token's angles are read once for them all, and a head's values are on
// their way while those of the head before are worked on. 8192 tokens of 32 + 8 + 8 heads of 128, bf16 (178 MB from memory):
// 46 us; the 16 heads with codes alone 22 (44 MB), a copy of the queries alone 25 (67 MB read and 67 written). The codes'
// part is bound by its arithmetic, 230 vector instructions for eight values, half of them in the way through 64 bits.
template <class D, int DIM, bool PAIRS>
__global__ void __launch_bounds__(256)
kv4_append_kernel(KV4 cache, Heads<typename D::T> q, Heads<typename D::T> k, Heads<typename D::T> v, int64_t tokens,
                  int q_heads, int per, const int64_t* __restrict__ slots, Angles angles, typename D::T* __restrict__ q_out) {
  using T = typename D::T;
  constexpr int LANES = kLanes<DIM>, TOKENS = 256 / LANES;
  __shared__ __align__(4) uint8_t bytes[2][DIM / 2][TOKENS];
  __shared__ int64_t token_slots[TOKENS];
  const int lane = threadIdx.x % LANES, mine = threadIdx.x / LANES;
  const int64_t token = (int64_t)blockIdx.x * TOKENS + mine;
  const bool there = token < tokens && 8 * lane < DIM;
  const int64_t row = token < tokens ? token : 0;
  const int q_groups = (q_heads + per - 1) / per, groups = (cache.heads + per - 1) / per;
  int group = blockIdx.y;
  const int kind = group < q_groups ? 0 : group < q_groups + groups ? 1 : 2;
  group -= kind == 0 ? 0 : kind == 1 ? q_groups : q_groups + groups;
  const int first = group * per, last = min(first + per, kind == 0 ? q_heads : cache.heads);

  Place p = {8 * lane, 8 * lane + 4, false};
  if (kind < 2) p = place_of<PAIRS>(lane, angles.rot);
  const Heads<T> source = kind == 0 ? q : kind == 1 ? k : v;
  const T* src = source.at(row, first);
  T raw[8];
  auto load = [&] {
    if (there) {
      __builtin_memcpy(raw, src + p.at, 4 * sizeof(T));
      __builtin_memcpy(raw + 4, src + p.more, 4 * sizeof(T));
    }
    src += source.head;
  };
  load();
  double c[4], s[4];
  if (p.turned && there) {
    const int64_t pos = angles.positions[row];
    const bool known = pos >= 0 && pos < angles.rows;
    const int64_t at = (known ? pos : 0) * (angles.rot / 2) + 4 * lane;   // the first pair's angle
    float a[4], b[4];
    __builtin_memcpy(a, angles.cos_ + at, sizeof(a));
    __builtin_memcpy(b, angles.sin_ + at, sizeof(b));
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = known ? a[i] : __builtin_nanf(""), s[i] = b[i];
  }
  // The lane's vector x of the next head, turned where it is.
  auto take = [&](bool more, float(&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = there ? D::to_f(raw[i]) : 0.f;
    if (more) load();
    if (p.turned && there) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (PAIRS) turn(x[2 * i], x[2 * i + 1], c[i], s[i]);
        else turn(x[i], x[4 + i], c[i], s[i]);
      }
    }
  };
  if (kind == 0) {
    T* to = q_out + (token * q_heads + first) * DIM;
    for (int head = first; head < last; ++head, to += DIM) {
      float x[8];
      take(head + 1 < last, x);
      if (!there) continue;
      T out[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) out[i] = D::from_f(x[i]);
      __builtin_memcpy(to + p.at, out, 4 * sizeof(T));
      __builtin_memcpy(to + p.more, out + 4, 4 * sizeof(T));
    }
    return;
  }

  const int64_t slot = token < tokens ? slots[row] : -1;
  const bool known = slot >= 0 && slot < cache.slots(), kept = there && known;
  const int64_t page = known ? slot >> cache.shift : 0;
  const int place = known ? (int)(slot & ((1 << cache.shift) - 1)) : 0;
  _Float16* par = cache.param_tile(page, kind - 1, first, place) + (place & 15);
  const int64_t head_params = (int64_t)2 << cache.shift;
  auto parameters = [&](_Float16 scale, _Float16 least) {
    if (kept && lane == 0) par[0] = scale, par[16] = least;
    par += head_params;
  };
  if (kind == 1) {
    uint8_t* to = cache.key(page, first, place, DIM);
    for (int head = first; head < last; ++head, to += (int64_t)DIM / 2 << cache.shift) {
      float x[8];
      take(head + 1 < last, x);
      uint32_t two[4];
      _Float16 scale, least;
      quantize<LANES>(x, there, two, scale, least);
      if (kept) {
        *reinterpret_cast<uint16_t*>(to + p.at / 2) = (uint16_t)__builtin_amdgcn_perm(two[1], two[0], 0x0C0C0400u);
        *reinterpret_cast<uint16_t*>(to + p.more / 2) = (uint16_t)__builtin_amdgcn_perm(two[3], two[2], 0x0C0C0400u);
      }
      parameters(scale, least);
    }
    return;
  }
  if (lane == 0) token_slots[mine] = known ? slot : -1;
  __syncthreads();
  ValueBytes<DIM, TOKENS> to(cache, first, token_slots);
  for (int head = first; head < last; ++head) {
    float x[8];
    take(head + 1 < last, x);
    uint32_t two[4];
    _Float16 scale, least;
    quantize<LANES>(x, there, two, scale, least);
    uint8_t(*box)[TOKENS] = bytes[(head - first) & 1];
    if (there) {
#pragma unroll
      for (int i = 0; i < 4; ++i) box[4 * lane + i][mine] = (uint8_t)two[i];
    }
    lds_barrier();   // the other box is written next: one barrier a head
    if (to.there) to.put(*reinterpret_cast<const uint32_t*>(&box[to.pair][to.t]));
    to.next_head();
    parameters(scale, least);
  }
}

// A thread reads eight values of a vector; blockIdx.y counts key heads, then value heads. 8192 tokens, 8 heads of
// 128 to bf16: 15.4 us for 43 MB, 2.8 TB/s (at random slots 18.7): 8192 workgroups whose threads wait for a slot, then for
// codes and parameters, and store 16 bytes once, with nothing under way beside it but other workgroups. A lane's four bytes of a value's codes are loads of their own: the lanes of 16
// tokens share their lines, and the same through words and LDS, as they were written, took 19 us (22).
template <class D, int DIM>
__global__ void __launch_bounds__(256)
kv4_read_kernel(KV4 cache, const int64_t* __restrict__ slots, int64_t tokens, typename D::T* __restrict__ k_out,
                typename D::T* __restrict__ v_out) {
  constexpr int LANES = kLanes<DIM>, TOKENS = 256 / LANES;
  const int lane = threadIdx.x % LANES;
  const int64_t token = (int64_t)blockIdx.x * TOKENS + threadIdx.x / LANES;
  if (token >= tokens || 8 * lane >= DIM) return;
  const bool values = blockIdx.y >= (unsigned)cache.heads;
  const int head = values ? blockIdx.y - cache.heads : blockIdx.y;
  const int64_t slot = slots[token];
  typename D::T out[8] = {};
  if (slot >= 0 && slot < cache.slots()) {
    const int64_t page = slot >> cache.shift;
    const int place = (int)(slot & ((1 << cache.shift) - 1));
    uint32_t w = 0;
    if (values) {
      const uint8_t* from = cache.value_tile(page, head, place, DIM) + (place & 15) + 4 * lane * 16;
#pragma unroll
      for (int i = 0; i < 4; ++i) w |= (uint32_t)from[16 * i] << (8 * i);
    } else {
      w = *reinterpret_cast<const uint32_t*>(cache.key(page, head, place, DIM) + 4 * lane);
    }
    const _Float16* par = cache.param_tile(page, values, head, place) + (place & 15);
    const float s = (float)par[0], lo = (float)par[16];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = fmaf(s, (float)(w >> (4 * i) & 15u), lo);
      // the largest code may stand for half a step more than fp16 holds
      out[i] = D::from_f(D::code == QO_DTYPE_F16 && fabsf(x) > kKV4Most ? copysignf(kKV4Most, x) : x);
    }
  }
  __builtin_memcpy((values ? v_out : k_out) + (token * cache.heads + head) * DIM + 8 * lane, out, sizeof(out));
}

template <class F>
bool with_dtype(int code, F&& f) {
  if (code == QO_DTYPE_F32) f(F32T{});
  else if (code == QO_DTYPE_F16) f(F16T{});
  else if (code == QO_DTYPE_BF16) f(BF16T{});
  else return false;
  return true;
}
template <class F>
void with_dim(int dim, F&& f) {
  if (dim == 64) f(std::integral_constant<int, 64>{});
  else if (dim == 96) f(std::integral_constant<int, 96>{});
  else if (dim == 128) f(std::integral_constant<int, 128>{});
  else if (dim == 192) f(std::integral_constant<int, 192>{});
  else f(std::integral_constant<int, 256>{});
}

int check_tokens(const char* fn, int64_t tokens, int dtype) {
  if (tokens < 0 || tokens > QO_KV4_MAX_TOKENS) {
    qo_set_error("%s: invalid number of tokens %lld", fn, (long long)tokens);
    return QO_ERR_SHAPE;
  }
  if (dtype != QO_DTYPE_F32 && dtype != QO_DTYPE_F16 && dtype != QO_DTYPE_BF16) {
    qo_set_error("%s: unsupported dtype code %d", fn, dtype);
    return QO_ERR_DTYPE;
  }
  return QO_OK;
}

// Heads that a workgroup takes in turn: as many as leave four workgroups for each CU, eight at most (8192 tokens of 48
// heads of 128, bf16: one 74 us, two 60, four and eight 44 to 54).
int heads_per_group(int64_t blocks, int heads) {
  const int64_t n = blocks * heads / (4 * device_cu_count());
  return n < 1 ? 1 : n > 8 ? 8 : (int)n;
}

int null_pointer(const char* fn) {
  qo_set_error("%s: NULL pointer argument", fn);
  return QO_ERR_NULL_POINTER;
}

}  // namespace

}  // namespace qo

extern "C" int qo_kv4_append(const qo_kv4_cache* cache, const qo_heads* q, const qo_heads* k, const qo_heads* v,
                             int dtype, int64_t tokens, int q_heads, const int64_t* slots, const int64_t* positions,
                             const float* cos_, const float* sin_, int64_t table_rows, int rot, int interleaved,
                             void* q_out, void* stream) {
  using namespace qo;
  const char* fn = "qo_kv4_append";
  KV4 c;
  int st = kv4_cache(fn, cache, &c);
  if (st == QO_OK) st = check_tokens(fn, tokens, dtype);
  if (st != QO_OK) return st;
  if (rot < 0 || rot > cache->head_dim || rot % 8 != 0 || table_rows < 0) {
    qo_set_error("%s: rot must be a multiple of 8 from 0 to head_dim (%d), got %d", fn, (int)cache->head_dim, rot);
    return QO_ERR_SHAPE;
  }
  if (q && (rot == 0 || q_heads < 1 || q_heads > 16384)) {
    qo_set_error("%s: q needs a rotation and from 1 to 16384 heads, got rot %d and %d heads", fn, rot, q_heads);
    return QO_ERR_SHAPE;
  }
  if (tokens == 0) return QO_OK;
  if (!k || !v || !k->data || !v->data || !slots || (q && (!q->data || !q_out))) return null_pointer(fn);
  if (rot && (!positions || (table_rows && (!cos_ || !sin_)))) return null_pointer(fn);
  if (table_rows == 0 && rot) {
    qo_set_error("%s: the table of angles is empty", fn);
    return QO_ERR_SHAPE;
  }
  if (!q) q_heads = 0;
  launch_begin();
  with_dtype(dtype, [&](auto d) {
    using D = decltype(d);
    using T = typename D::T;
    with_dim(cache->head_dim, [&](auto dim) {
      constexpr int DIM = decltype(dim)::value, TOKENS = 256 / kLanes<DIM>;
      auto heads = [](const qo_heads* h) {
        return h ? Heads<T>{reinterpret_cast<const T*>(h->data), h->token_stride, h->head_stride} : Heads<T>{};
      };
      const int64_t blocks = (tokens + TOKENS - 1) / TOKENS;
      const int per = heads_per_group(blocks, q_heads + 2 * c.heads);
      const dim3 grid((unsigned)blocks, (unsigned)((q_heads + per - 1) / per + 2 * ((c.heads + per - 1) / per)));
      launch(interleaved ? kv4_append_kernel<D, DIM, true> : kv4_append_kernel<D, DIM, false>, grid, dim3(256), 0,
             reinterpret_cast<hipStream_t>(stream), c, heads(q), heads(k), heads(v), tokens, q_heads, per, slots,
             Angles{positions, cos_, sin_, table_rows, rot}, reinterpret_cast<T*>(q_out));
    });
  });
  return launch_result(fn);
}

extern "C" int qo_kv4_read(const qo_kv4_cache* cache, const int64_t* slots, int64_t tokens, void* k_out, void* v_out,
                           int out_dtype, void* stream) {
  using namespace qo;
  const char* fn = "qo_kv4_read";
  KV4 c;
  int st = kv4_cache(fn, cache, &c);
  if (st == QO_OK) st = check_tokens(fn, tokens, out_dtype);
  if (st != QO_OK) return st;
  if (tokens == 0) return QO_OK;
  if (!slots || !k_out || !v_out) return null_pointer(fn);
  launch_begin();
  with_dtype(out_dtype, [&](auto d) {
    using D = decltype(d);
    using T = typename D::T;
    with_dim(cache->head_dim, [&](auto dim) {
      constexpr int DIM = decltype(dim)::value, TOKENS = 256 / kLanes<DIM>;
      launch(kv4_read_kernel<D, DIM>, dim3((unsigned)((tokens + TOKENS - 1) / TOKENS), (unsigned)(2 * c.heads)), dim3(256),
             0, reinterpret_cast<hipStream_t>(stream), c, slots, tokens, reinterpret_cast<T*>(k_out),
             reinterpret_cast<T*>(v_out));
    });
  });
  return launch_result(fn);
}
