// Quantizing to the microscaled formats of mx_common.h and back: as it is, after
// the RMS norm (with the residual's addition), and after the SwiGLU gate. All
// of them are bound by HBM: a thread holds eight consecutive values of a row
// (one or two 16-byte loads), four lanes share a block's maximum by DPP, and the
// conversions to and from codes are one instruction for two values.
#include "mx_common.h"

namespace qo {

namespace {

// A workgroup of 256 threads takes 256 / TPR rows (TPR: a power of two) by TPR
// chunks of eight values; blockIdx.x counts chunk columns, blockIdx.y groups of
// U row groups, whose loads are all issued before the first is used.
struct RowMap {
  int shift;   // log2(TPR)
  int chunks;  // of a row: 4 * blocks, or those of its features
};

template <int U, class F>
__device__ inline void for_rows(const RowMap& map, int64_t tokens, F&& f) {
  const int tpr = 1 << map.shift, rows = 256 >> map.shift;
  const int c = blockIdx.x * tpr + (threadIdx.x & (tpr - 1));
  if (c >= map.chunks) return;   // whole quads: tpr and chunks of quantizing kernels are multiples of 4
  for (int64_t r0 = (int64_t)blockIdx.y * U * rows; r0 < tokens; r0 += (int64_t)gridDim.y * U * rows)
    f(r0 + (threadIdx.x >> map.shift), rows, c);
}

template <class D, class Q, int U>
__global__ void __launch_bounds__(256)
mx_quantize_kernel(const typename D::T* __restrict__ x, int64_t ld, int64_t tokens, int64_t features, int blocks,
                   RowMap map, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, int64_t scales_ld) {
  for_rows<U>(map, tokens, [&](int64_t row, int step, int c) {
    float v[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (row + u * step < tokens) load8<D>(x + (row + u * step) * ld + 8 * c, features - 8 * c, v[u]);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (row + u * step < tokens) mx_store8<Q>(v[u], codes, scales, scales_ld, row + u * step, blocks, c);
  });
}

// y = g / (1 + exp(-g)) u of the gate g and its factor u, which stand
// `features` apart in a row.
template <class D, class Q, int U>
__global__ void __launch_bounds__(256)
swiglu_mx_kernel(const typename D::T* __restrict__ x, int64_t ld, int64_t tokens, int64_t features, int blocks,
                 RowMap map, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, int64_t scales_ld) {
  for_rows<U>(map, tokens, [&](int64_t row, int step, int c) {
    float g[U][8], up[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (row + u * step < tokens) {
        const typename D::T* p = x + (row + u * step) * ld + 8 * c;
        load8<D>(p, features - 8 * c, g[u]);
        load8<D>(p + features, features - 8 * c, up[u]);
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (row + u * step < tokens) {
#pragma unroll
        for (int i = 0; i < 8; ++i) g[u][i] = g[u][i] / (1.f + expf(-g[u][i])) * up[u][i];
        mx_store8<Q>(g[u], codes, scales, scales_ld, row + u * step, blocks, c);
      }
  });
}

template <class D, class Q, int U>
__global__ void __launch_bounds__(256)
mx_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int64_t scales_ld, int64_t tokens,
                     int64_t features, int blocks, RowMap map, typename D::T* __restrict__ out) {
  for_rows<U>(map, tokens, [&](int64_t row, int step, int c) {
    uint32_t w[U][Q::words], byte[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (row + u * step < tokens) {
        const int64_t r = row + u * step;
        __builtin_memcpy(w[u], codes + (r * blocks * 4 + c) * (4 * Q::words), sizeof(w[u]));
        byte[u] = scales[r * scales_ld + (c >> 2)];
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (row + u * step < tokens) {
        float v[8];
        mx_values8<Q>(w[u], byte[u], v);
        store8<D>(out + (row + u * step) * features + 8 * c, features - 8 * c, v);
      }
  });
}

// One row per workgroup, in registers: h = x + residual, the mean of h^2, then
// y = h / sqrt(mean + eps) * weight and its codes. Statistics, h and y are
// float32; h is rounded once, to x's type, where it is stored. Thread t holds
// chunks t, t + THREADS, .. (NV of them); rows longer than that are read twice
// (NV = 0).
template <class D, class Q, int THREADS, int NV>
__global__ void __launch_bounds__(THREADS)
rms_norm_mx_kernel(const typename D::T* __restrict__ x, int64_t ld, const typename D::T* res,
                   int64_t res_ld, const void* __restrict__ weight, int weight_dtype, int64_t tokens,
                   int64_t features, int blocks, float eps, uint8_t* __restrict__ codes,
                   uint8_t* __restrict__ scales, int64_t scales_ld, typename D::T* res_out) {
  constexpr int W = THREADS / 64, N = NV ? NV : 1;
  __shared__ float part[W];
  const int tid = threadIdx.x, chunks = 4 * blocks;
  auto weights = [&](int c, float(&w)[8]) {
    const int64_t n = features - 8 * c;
    if (weight_dtype == QO_DTYPE_F32) load8<F32T>(reinterpret_cast<const float*>(weight) + 8 * c, n, w);
    else if (weight_dtype == QO_DTYPE_F16) load8<F16T>(reinterpret_cast<const _Float16*>(weight) + 8 * c, n, w);
    else load8<BF16T>(reinterpret_cast<const __bf16*>(weight) + 8 * c, n, w);
  };
  for (int64_t row = blockIdx.x; row < tokens; row += gridDim.x) {
    float h[N][8], sum = 0.f;
    auto load = [&](int c, float(&v)[8]) {
      load8<D>(x + row * ld + 8 * c, features - 8 * c, v);
      if (res) {
        float r[8];
        load8<D>(res + row * res_ld + 8 * c, features - 8 * c, r);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += r[i];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) sum = fmaf(v[i], v[i], sum);
    };
    if constexpr (NV > 0) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (tid + j * THREADS < chunks) load(tid + j * THREADS, h[j]);
    } else {
      for (int c = tid; c < chunks; c += THREADS) load(c, h[0]);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    if constexpr (W > 1) {
      if ((tid & 63) == 0) part[tid >> 6] = sum;
      __syncthreads();
      sum = 0.f;
#pragma unroll
      for (int i = 0; i < W; ++i) sum += part[i];
      __syncthreads();   // part is written again for the next row
    }
    const float r = 1.f / sqrtf(sum / (float)features + eps);
    auto finish = [&](int c, float(&v)[8]) {
      if (res_out && 8 * c < features) store8<D>(res_out + row * features + 8 * c, features - 8 * c, v);
      float w[8];
      weights(c, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = v[i] * r * w[i];
      mx_store8<Q>(v, codes, scales, scales_ld, row, blocks, c);
    };
    if constexpr (NV > 0) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (tid + j * THREADS < chunks) finish(tid + j * THREADS, h[j]);
    } else {
      for (int c = tid; c < chunks; c += THREADS) {
        load(c, h[0]);
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
Grid row_grid(int64_t tokens, int64_t chunks, int U) {
  int shift = 2;
  while (shift < 8 && (1 << shift) < chunks) ++shift;
  const int64_t per = (int64_t)U * (256 >> shift);
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
      const Grid g = row_grid(tokens, 4 * blocks, 1);
      launch(mx_quantize_kernel<D, decltype(q), 1>, g.grid, dim3(256), 0, reinterpret_cast<hipStream_t>(stream),
             reinterpret_cast<const typename D::T*>(x), x_ld, tokens, features, blocks, g.map,
             reinterpret_cast<uint8_t*>(codes), scales, scales_ld);
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
      const Grid g = row_grid(tokens, (features + 7) / 8, 1);
      launch(mx_dequantize_kernel<D, decltype(q), 1>, g.grid, dim3(256), 0, reinterpret_cast<hipStream_t>(stream),
             reinterpret_cast<const uint8_t*>(codes), scales, scales_ld, tokens, features, blocks, g.map,
             reinterpret_cast<typename D::T*>(out));
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
      const Grid g = row_grid(tokens, 4 * blocks, 1);
      launch(swiglu_mx_kernel<D, decltype(q), 1>, g.grid, dim3(256), 0, reinterpret_cast<hipStream_t>(stream),
             reinterpret_cast<const typename D::T*>(gate_up), ld, tokens, features, blocks, g.map,
             reinterpret_cast<uint8_t*>(codes), scales, scales_ld);
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
               eps, reinterpret_cast<uint8_t*>(codes), scales, scales_ld,
               residual ? reinterpret_cast<T*>(residual_out) : nullptr);
      };
      using Q = decltype(q);
      go(rms_norm_mx_kernel<D, Q, 256, 0>, 256);
    });
  });
  return launch_result(fn);
}
