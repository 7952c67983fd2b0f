// Quantizing to the microscaled formats of mx_common.h and back: as it is, after
// the RMS norm (with the residual's addition), and after the SwiGLU gate. All
// of them are bound by HBM: a thread holds eight consecutive values of a row
// (one or two 16-byte loads), four lanes share a block's maximum by DPP, and the
// conversions to and from codes are one instruction for two values.
#include "mx_common.h"

namespace qo {

namespace {

// A workgroup of 256 threads takes 256 / TPR rows (TPR: a power of two) by TPR
// chunks of a row: blockIdx.x counts chunk columns, blockIdx.y groups of rows. One
// chunk a thread: several rows a thread with their loads issued together measured
// slower (quantize 14336 x 4096 bf16 30.2 us; two rows 30.5, four 31.1).
struct RowMap {
  int shift;   // log2(TPR)
  int chunks;  // of a row
};

template <class F>
__device__ inline void for_rows(const RowMap& map, int64_t tokens, F&& f) {
  const int tpr = 1 << map.shift, rows = 256 >> map.shift;
  const int c = blockIdx.x * tpr + (threadIdx.x & (tpr - 1));
  if (c >= map.chunks) return;   // whole quads: tpr and chunks of quantizing kernels are multiples of 4
  for (int64_t row = (int64_t)blockIdx.y * rows + (threadIdx.x >> map.shift); row < tokens; row += (int64_t)gridDim.y * rows)
    f(row, c);
}

// 14336 x 4096 bf16 to FP4: 29-30 us, 5.0 TB/s (a large read and write 6.2). Codes and scales
// are plain stores, since a product reads them next: non-temporal ones gave nothing here
// and cost the reader a trip to memory.
template <class D, class Q, bool WHOLE>
__global__ void __launch_bounds__(256)
mx_quantize_kernel(const typename D::T* __restrict__ x, int64_t ld, int64_t tokens, int64_t features, int blocks,
                   RowMap map, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, int64_t scales_ld) {
  for_rows(map, tokens, [&](int64_t row, int c) {
    float v[8];
    values8<D, WHOLE>(load8<D, WHOLE>(x + row * ld, c, features), c, features, v);
    mx_store8<Q>(v, codes, scales, scales_ld, row, blocks, c);
  });
}

// g / (1 + exp(-g)) to a few units of float32, in a third of the instructions of
// expf and a full division (which bound the kernel). The power's argument -g log2(e)
// is split in its rounded product and the rest; above 128 the power is
// infinite and the quotient 0, as the formula has it. From g = 128 on the power adds
// nothing to 1: the argument stops there, so that the split of the largest g is no
// inf - inf. The reciprocal is taken of a quarter of the sum, so that it never
// leaves the normal range.
__device__ inline float mx_silu(float g) {
  constexpr float kLog2e = 1.44269502f, kRest = 1.92596303e-8f, kLn2 = 0.693147182f;   // log2(e) = kLog2e + kRest
  const float t = fminf(g, 128.f);   // a NaN is in the last line's g still
  const float hi = -t * kLog2e;
  const float lo = fmaf(-t, kRest, fmaf(-t, kLog2e, -hi));
  const float p = __builtin_amdgcn_exp2f(hi);
  const float e = hi >= 128.f ? __builtin_inff() : fmaf(p, lo * kLn2, p);
  return (0.25f * g) * __builtin_amdgcn_rcpf(fmaf(e, 0.25f, 0.25f));
}

// y = silu(g) u of the gate g and its factor u, which stand `features` apart in a row.
// 2048 x 14336 fp16 to FP8: 25 us, 5.9 TB/s.
template <class D, class Q, bool WHOLE>
__global__ void __launch_bounds__(256)
swiglu_mx_kernel(const typename D::T* __restrict__ x, int64_t ld, int64_t tokens, int64_t features, int blocks,
                 RowMap map, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, int64_t scales_ld) {
  for_rows(map, tokens, [&](int64_t row, int c) {
    const typename D::T* p = x + row * ld;
    const Raw8<D> g = load8<D, WHOLE>(p, c, features), u = load8<D, WHOLE>(p + features, c, features);
    float v[8], w[8];
    values8<D, WHOLE>(g, c, features, v);
    values8<D, WHOLE>(u, c, features, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = mx_silu(v[i]) * w[i];
    mx_store8<Q>(v, codes, scales, scales_ld, row, blocks, c);
  });
}

// A lane writes 16 bytes of values (a wave 1 KiB of a row): eight of 16 bits, four
// float32. NT: as non-temporal stores, which stream to memory instead of waiting in
// L2: 14336 x 4096 FP4 to bf16 39.9 -> 21.8 us (6.8 TB/s).
template <class D, class Q, bool NT>
__global__ void __launch_bounds__(256)
mx_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int64_t scales_ld,
                     int64_t tokens, int64_t features, int blocks, RowMap map, typename D::T* __restrict__ out) {
  constexpr int N = 16 / sizeof(typename D::T), BYTES = N * Q::words / 2;   // values and their codes' bytes
  constexpr int PER = 8 / Q::words;                                         // values of a word
  for_rows(map, tokens, [&](int64_t row, int c) {
    uint32_t w[2] = {0, 0};
    __builtin_memcpy(w, codes + row * blocks * 16 * Q::words + (int64_t)c * BYTES, BYTES);
    const uint32_t byte = scales[row * scales_ld + c * N / 32];
    float v[N];
#pragma unroll
    for (int h = 0; h < (N + PER - 1) / PER; ++h) {
      float t[PER];
      mx_word_values<Q>(w[h], byte, t);
#pragma unroll
      for (int i = 0; i < PER && h * PER + i < N; ++i) v[h * PER + i] = t[i];
    }
    store_row<D, N, NT>(out + row * features + (int64_t)c * N, features - (int64_t)c * N, v);
  });
}

// One row per workgroup, in registers: h = x + residual, the mean of h^2, then
// y = h / sqrt(mean + eps) * weight and its codes. h and y are float32. The sum of
// squares and the mean are held in 64 bits, and the factor 1 / sqrt and its products with h
// carry their roundings along, so y is the formula's value rounded once, also where the
// squares leave float32 (beside memory's time at no cost: 8192 x 4096 as with float32 sums;
// products in 64 bits 15 % more). h is rounded once, to x's type, where it is stored. Of T
// threads (a multiple of 64 up to MOST), thread t holds chunks t, t + T, .. (NV of them, T
// the least that covers the row); rows longer than that, or of no whole pieces, are read
// twice (NV = 0). 8192 x 4096 bf16 with a residual: 46 us, 5.2 TB/s, on 512 threads of one
// chunk (256 of two 50, 128 of four 60, 1024, half of them idle, 106; read twice 59).
template <class D, class Q, int MOST, int NV>
__global__ void __launch_bounds__(MOST)
rms_norm_mx_kernel(const typename D::T* __restrict__ x, int64_t ld, const typename D::T* res, int64_t res_ld,
                   const void* __restrict__ weight, int weight_dtype, int64_t tokens, int64_t features, int blocks,
                   float eps, double per_feature, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                   int64_t scales_ld, typename D::T* res_out) {
  constexpr int N = NV ? NV : 1;
  constexpr bool WHOLE = NV > 0;
  __shared__ double part[MOST / 64];
  const int tid = threadIdx.x, T = blockDim.x, chunks = 4 * blocks;
  auto weights = [&](int c, float(&w)[8]) {
    if (weight_dtype == QO_DTYPE_F32) values8<F32T, WHOLE>(load8<F32T, WHOLE>(reinterpret_cast<const float*>(weight), c, features), c, features, w);
    else if (weight_dtype == QO_DTYPE_F16) values8<F16T, WHOLE>(load8<F16T, WHOLE>(reinterpret_cast<const _Float16*>(weight), c, features), c, features, w);
    else values8<BF16T, WHOLE>(load8<BF16T, WHOLE>(reinterpret_cast<const __bf16*>(weight), c, features), c, features, w);
  };
  for (int64_t row = blockIdx.x; row < tokens; row += gridDim.x) {
    Raw8<D> rx[N], rr[N];
    double sum = 0.0;
    auto load = [&](int c, int j) {
      rx[j] = load8<D, WHOLE>(x + row * ld, c, features);
      if (res) rr[j] = load8<D, WHOLE>(res + row * res_ld, c, features);
    };
    auto add = [&](int c, int j, float(&v)[8]) {
      values8<D, WHOLE>(rx[j], c, features, v);
      if (res) {
        float r[8];
        values8<D, WHOLE>(rr[j], c, features, r);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += r[i];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = opaque(v[i]);   // else all chunks of h become one tuple, which spills
    };
    auto squares = [&](const float(&v)[8]) {
#pragma unroll
      for (int i = 0; i < 8; ++i) sum = fma((double)v[i], (double)v[i], sum);
    };
    float h[N][8];
    if constexpr (NV > 0) {
#pragma unroll
      for (int j = 0; j < NV; ++j) load(tid + j * T, j);   // past the row's chunks: nothing (zeros)
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        add(tid + j * T, j, h[j]);
        squares(h[j]);
      }
    } else {
      for (int c = tid; c < chunks; c += T) {
        load(c, 0);
        add(c, 0, h[0]);
        squares(h[0]);
      }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    if (T > 64) {
      if ((tid & 63) == 0) part[tid >> 6] = sum;
      __syncthreads();
      sum = 0.0;
      for (int i = 0; i < T >> 6; ++i) sum += part[i];
      __syncthreads();   // part is written again for the next row
    }
    // 1 / sqrt(mean + eps) = fit (r + rest): the rest by a Newton step in 64 bits, which leaves 2^-45 of
    // it (0 where r is 0 or infinite). fit is 1, or the power of two that brings the squares into float32.
    const double mean = sum * per_feature + (double)eps;
    const float fit = mean > 0x1p100 ? 0x1p-80f : mean < 0x1p-100 ? 0x1p96f : 1.f;
    const double m = mean * fit * fit;
    const float r = __builtin_amdgcn_rsqf((float)m);
    const float step = (float)(0.5 * r * (1.0 - m * r * r)), rest = step == step ? step : 0.f;
    auto finish = [&](int c, const float(&v)[8]) {
      // whole pieces stream to memory (16-byte aligned: the host's check)
      if (res_out && 8 * c < features) store_row<D, 8, WHOLE>(res_out + row * features + 8 * c, WHOLE ? 8 : features - 8 * c, v);
      float w[8], y[8];
      weights(c, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) {   // (u r + its rounding + u rest) w
        const float u = v[i] * fit, q = u * r, more = fmaf(u, rest, fmaf(u, r, -q));
        y[i] = fmaf(q, w[i], more * w[i]);
      }
      mx_store8<Q>(y, codes, scales, scales_ld, row, blocks, c);
    };
    if constexpr (NV > 0) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (tid + j * T < chunks) finish(tid + j * T, h[j]);
    } else {
      for (int c = tid; c < chunks; c += T) {
        load(c, 0);
        add(c, 0, h[0]);
        finish(c, h[0]);
      }
    }
  }
}

struct Grid {
  RowMap map;
  dim3 grid;
};

// TPR: the power of two from 4 to 256 that covers a row's chunks, or 256.
Grid row_grid(int64_t tokens, int64_t chunks) {
  int shift = 2;
  while (shift < 8 && (1 << shift) < chunks) ++shift;
  const int64_t per = 256 >> shift;
  const int64_t y = (tokens + per - 1) / per;
  return {{shift, (int)chunks}, dim3((unsigned)((chunks + (1 << shift) - 1) >> shift), (unsigned)(y < 65535 ? y : 65535))};
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
void with_format(int code, F&& f) {
  if (code == QO_MX_FP4) f(FP4{});
  else f(FP8{});
}

bool known_dtype(int c) { return c == QO_DTYPE_F32 || c == QO_DTYPE_F16 || c == QO_DTYPE_BF16; }
bool known_format(int c) { return c == QO_MX_FP4 || c == QO_MX_FP8; }

// Checks that the entry points share; QO_OK with *empty set where there is nothing to do.
int check(const char* fn, int64_t tokens, int64_t features, int dtype, int format, int64_t scales_ld, bool* empty) {
  if (tokens < 0 || features < 0 || features > QO_MX_MAX_FEATURES) {
    qo_set_error("%s: invalid sizes tokens=%lld features=%lld", fn, (long long)tokens, (long long)features);
    return QO_ERR_SHAPE;
  }
  if (scales_ld < (features + 31) / 32) {
    qo_set_error("%s: scales_ld %lld below the %lld blocks of a row", fn, (long long)scales_ld,
                 (long long)((features + 31) / 32));
    return QO_ERR_SHAPE;
  }
  if (!known_dtype(dtype)) {
    qo_set_error("%s: unsupported dtype code %d", fn, dtype);
    return QO_ERR_DTYPE;
  }
  if (!known_format(format)) {
    qo_set_error("%s: unknown MX format code %d", fn, format);
    return QO_ERR_DTYPE;
  }
  *empty = tokens == 0 || features == 0;
  return QO_OK;
}

int null_pointer(const char* fn) {
  qo_set_error("%s: NULL pointer argument", fn);
  return QO_ERR_NULL_POINTER;
}

int misaligned(const char* fn, const char* what) {
  qo_set_error("%s: %s must be 8-byte aligned", fn, what);
  return QO_ERR_ALIGNMENT;
}

}  // namespace

}  // namespace qo

extern "C" int qo_mx_quantize(const void* x, int x_dtype, int64_t tokens, int64_t features, int64_t x_ld, int format,
                              void* codes, uint8_t* scales, int64_t scales_ld, void* stream) {
  using namespace qo;
  const char* fn = "qo_mx_quantize";
  bool empty;
  const int st = check(fn, tokens, features, x_dtype, format, scales_ld, &empty);
  if (st != QO_OK) return st;
  if (x_ld < features) {
    qo_set_error("%s: row stride %lld below row length %lld", fn, (long long)x_ld, (long long)features);
    return QO_ERR_SHAPE;
  }
  if (empty) return QO_OK;
  if (!x || !codes || !scales) return null_pointer(fn);
  if ((uintptr_t)codes % 8 != 0) return misaligned(fn, "codes");
  const int blocks = (int)((features + 31) / 32);
  launch_begin();
  with_dtype(x_dtype, [&](auto d) {
    using D = decltype(d);
    with_format(format, [&](auto q) {
      using Q = decltype(q);
      const Grid g = row_grid(tokens, 4 * blocks);
      launch(features % 8 == 0 ? mx_quantize_kernel<D, Q, true> : mx_quantize_kernel<D, Q, false>, g.grid, dim3(256), 0,
             reinterpret_cast<hipStream_t>(stream), reinterpret_cast<const typename D::T*>(x), x_ld, tokens, features,
             blocks, g.map, reinterpret_cast<uint8_t*>(codes), scales, scales_ld);
    });
  });
  return launch_result(fn);
}

extern "C" int qo_mx_dequantize(const void* codes, const uint8_t* scales, int64_t scales_ld, int format,
                                int64_t tokens, int64_t features, void* out, int out_dtype, void* stream) {
  using namespace qo;
  const char* fn = "qo_mx_dequantize";
  bool empty;
  const int st = check(fn, tokens, features, out_dtype, format, scales_ld, &empty);
  if (st != QO_OK) return st;
  if (empty) return QO_OK;
  if (!codes || !scales || !out) return null_pointer(fn);
  if ((uintptr_t)codes % 8 != 0) return misaligned(fn, "codes");
  const int blocks = (int)((features + 31) / 32);
  launch_begin();
  with_dtype(out_dtype, [&](auto d) {
    using D = decltype(d);
    with_format(format, [&](auto q) {
      using Q = decltype(q);
      constexpr int N = 16 / sizeof(typename D::T);
      const Grid g = row_grid(tokens, (features + N - 1) / N);
      const bool aligned = (uintptr_t)out % 16 == 0 && features % N == 0;
      launch(aligned ? mx_dequantize_kernel<D, Q, true> : mx_dequantize_kernel<D, Q, false>, g.grid, dim3(256), 0,
             reinterpret_cast<hipStream_t>(stream), reinterpret_cast<const uint8_t*>(codes), scales, scales_ld, tokens,
             features, blocks, g.map, reinterpret_cast<typename D::T*>(out));
    });
  });
  return launch_result(fn);
}

extern "C" int qo_swiglu_mx_quantize(const void* gate_up, int dtype, int64_t tokens, int64_t features, int64_t ld,
                                     int format, void* codes, uint8_t* scales, int64_t scales_ld, void* stream) {
  using namespace qo;
  const char* fn = "qo_swiglu_mx_quantize";
  bool empty;
  const int st = check(fn, tokens, features, dtype, format, scales_ld, &empty);
  if (st != QO_OK) return st;
  if (ld < 2 * features) {
    qo_set_error("%s: row stride %lld below row length %lld", fn, (long long)ld, (long long)(2 * features));
    return QO_ERR_SHAPE;
  }
  if (empty) return QO_OK;
  if (!gate_up || !codes || !scales) return null_pointer(fn);
  if ((uintptr_t)codes % 8 != 0) return misaligned(fn, "codes");
  const int blocks = (int)((features + 31) / 32);
  launch_begin();
  with_dtype(dtype, [&](auto d) {
    using D = decltype(d);
    with_format(format, [&](auto q) {
      using Q = decltype(q);
      const Grid g = row_grid(tokens, 4 * blocks);
      launch(features % 8 == 0 ? swiglu_mx_kernel<D, Q, true> : swiglu_mx_kernel<D, Q, false>, g.grid, dim3(256), 0,
             reinterpret_cast<hipStream_t>(stream), reinterpret_cast<const typename D::T*>(gate_up), ld, tokens, features,
             blocks, g.map, reinterpret_cast<uint8_t*>(codes), scales, scales_ld);
    });
  });
  return launch_result(fn);
}

extern "C" int qo_rms_norm_mx_quantize(const void* x, const void* residual, int x_dtype, int64_t tokens,
                                       int64_t features, int64_t x_ld, int64_t residual_ld, const void* weight,
                                       int weight_dtype, float eps, int format, void* codes, uint8_t* scales,
                                       int64_t scales_ld, void* residual_out, void* stream) {
  using namespace qo;
  const char* fn = "qo_rms_norm_mx_quantize";
  bool empty;
  const int st = check(fn, tokens, features, x_dtype, format, scales_ld, &empty);
  if (st != QO_OK) return st;
  if (!known_dtype(weight_dtype)) {
    qo_set_error("%s: unsupported weight dtype code %d", fn, weight_dtype);
    return QO_ERR_DTYPE;
  }
  if (x_ld < features || (residual && residual_ld < features)) {
    qo_set_error("%s: row stride below row length (x %lld, residual %lld, features %lld)", fn, (long long)x_ld,
                 (long long)residual_ld, (long long)features);
    return QO_ERR_SHAPE;
  }
  if (empty) return QO_OK;
  if (!x || !weight || !codes || !scales || (residual && !residual_out)) return null_pointer(fn);
  if ((uintptr_t)codes % 8 != 0) return misaligned(fn, "codes");
  const int blocks = (int)((features + 31) / 32);
  launch_begin();
  with_dtype(x_dtype, [&](auto d) {
    using D = decltype(d);
    using T = typename D::T;
    with_format(format, [&](auto q) {
      const dim3 grid((unsigned)(tokens < (1 << 20) ? tokens : (1 << 20)));
      auto go = [&](auto kernel, int threads) {
        launch(kernel, grid, dim3(threads), 0, reinterpret_cast<hipStream_t>(stream), reinterpret_cast<const T*>(x),
               x_ld, reinterpret_cast<const T*>(residual), residual_ld, weight, weight_dtype, tokens, features, blocks,
               eps, 1.0 / (double)features, reinterpret_cast<uint8_t*>(codes), scales, scales_ld,
               residual ? reinterpret_cast<T*>(residual_out) : nullptr);
      };
      using Q = decltype(q);
      const int chunks = 4 * blocks;
      const bool whole = features % 8 == 0 && (!residual || (uintptr_t)residual_out % 16 == 0);
      auto threads = [&](int nv) { return ((chunks + nv - 1) / nv + 63) / 64 * 64; };
      if (whole && chunks <= 512) go(rms_norm_mx_kernel<D, Q, 512, 1>, threads(1));
      else if (whole && chunks <= 1024) go(rms_norm_mx_kernel<D, Q, 512, 2>, threads(2));
      else if (whole && chunks <= 2048) go(rms_norm_mx_kernel<D, Q, 1024, 2>, threads(2));
      else if (whole && chunks <= 3072) go(rms_norm_mx_kernel<D, Q, 1024, 3>, threads(3));
      else if (whole && chunks <= 4096) go(rms_norm_mx_kernel<D, Q, 1024, 4>, threads(4));
      else if (chunks <= 1024) go(rms_norm_mx_kernel<D, Q, 256, 0>, 256);
      else go(rms_norm_mx_kernel<D, Q, 1024, 0>, 1024);
    });
  });
  return launch_result(fn);
}
