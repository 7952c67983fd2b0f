// The product of microscaled operands (mx_common.h) on gfx950's scaled matrix
// cores: out[m, n] = rnd(sum_k a[m, k] b[n, k] + bias[n]), a in FP4 or FP8, the
// weight b in FP4, each value its code times its block's scale.
// v_mfma_scale_f32_16x16x128_f8f6f4 takes both formats and the scale bytes as
// they are and sums in float32.
//
// Fragments of 16 rows x 128 values (four blocks): lane l = r + 16 g has row r.
// FP4: the 16 bytes of block g. FP8: bytes 16 g .. of the row's 128 and 64 + 16 g ..
// (half of two blocks each). Either way its scale operand is block g's.
#include "int4_common.h"
#include "mx_common.h"

namespace qo {

namespace {

typedef int v8i __attribute__((ext_vector_type(8)));

struct MxOperand {
  const uint8_t* codes;
  int64_t ld;            // bytes between rows of codes
  const uint8_t* scales;
  int64_t scales_ld;
  int rows;
};

// What the matrix core does with an FP8 operand (found by probing it with
// terms of chosen sizes): of each eight consecutive products it drops the bits
// below 2^-13 of 2^(largest exponent sum of the eight). FP4 products span too
// few binades to lose any. On activations with outlier channels (0.5 %, x30)
// that is 2.3e-5 of the result's norm, far below a 16-bit output's rounding,
// but above float32's. For float32 outputs FP8 fragments are therefore
// multiplied in two halves, codes of magnitude 2 and up (exponent field 8 ..
// 15) and below: within each the lowest bit of any product stands above the
// cut (2^-3 against 2^-3, 2^-10 against 2^-11), so nothing is dropped.
template <class QA, class OT>
constexpr bool kSplitFp8 = QA::code == QO_MX_FP8 && sizeof(typename OT::T) == 4;

template <class Q>
constexpr int kMfmaFormat = Q::code == QO_MX_FP4 ? 4 : 0;

// MFMA of weight fragment b (output columns) and activation fragment a
// (rows): lane l's four sums are row l % 16, columns 4 (l / 16) + 0 .. 3. SEL: the
// byte of the scale operands.
template <class QA, int SEL>
__device__ inline v4f mx_mfma(const v8i& b, const v8i& a, v4f acc, uint32_t sb, uint32_t sa) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b, a, acc, 4, kMfmaFormat<QA>, SEL, (int)sb, SEL, (int)sa);
}

// mx_mfma, FP8 fragments in two halves where OT asks for it.
template <class QA, class OT, int SEL>
__device__ inline v4f mx_mac(const v8i& b, const v8i& a, v4f acc, uint32_t sb, uint32_t sa) {
  if constexpr (kSplitFp8<QA, OT>) {
    v8i hi, lo;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t w = (uint32_t)a[i], top = w & 0x40404040u;   // exponent field's high bit
      const uint32_t mask = (top << 1) | (top + (top - (top >> 6)));   // 0xFF in each byte that has it
      hi[i] = (int)(w & mask);
      lo[i] = (int)(w & ~mask);
    }
    acc = mx_mfma<QA, SEL>(b, lo, acc, sb, sa);
    return mx_mfma<QA, SEL>(b, hi, acc, sb, sa);
  } else {
    return mx_mfma<QA, SEL>(b, a, acc, sb, sa);
  }
}

// The output's four values of one row from column n on, + bias, rounded once.
template <class OT>
__device__ inline void mx_store4(v4f v, typename OT::T* out, int64_t ldc, const typename OT::T* bias, int M, int N,
                                 int m, int n) {
  if (m >= M || n >= N) return;
  typename OT::T t[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) t[r] = OT::cvt(v[r] + (bias ? (float)bias[min(n + r, N - 1)] : 0.f));
  typename OT::T* o = out + (int64_t)m * ldc + n;
  if (n + 4 <= N) {
    __builtin_memcpy(o, t, sizeof(t));
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (n + r < N) o[r] = t[r];
  }
}

// ---------------------------------------------------------------------------
// mx_gemm_stream: a workgroup makes 16 FM x 16 FN outputs; its W waves split the
// k-steps (of 128) in contiguous runs, load their fragments straight into
// registers, U steps at a time, and add their sums in LDS in a fixed order.
// ---------------------------------------------------------------------------
template <class QA, class OT, int FM, int FN, int U, int W>
__global__ void __launch_bounds__(64 * W)
mx_gemm_stream(MxOperand a, MxOperand b, int blocks, typename OT::T* __restrict__ out, int64_t ldc,
               const typename OT::T* __restrict__ bias) {
  constexpr int F = FM * FN;
  __shared__ __align__(16) v4f part[W][F][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int li = lane & 15, lg = lane >> 4;
  const int tiles_n = (b.rows + 16 * FN - 1) / (16 * FN);
  const int m0 = (int)(blockIdx.x / tiles_n) * 16 * FM, n0 = (int)(blockIdx.x % tiles_n) * 16 * FN;

  // rows past the edge read the last row; their sums are not stored
  const uint8_t *ac[FM], *as[FM], *bc[FN], *bs[FN];
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int64_t r = min(m0 + 16 * i + li, a.rows - 1);
    ac[i] = a.codes + r * a.ld + 16 * lg;
    as[i] = a.scales + r * a.scales_ld;
  }
#pragma unroll
  for (int j = 0; j < FN; ++j) {
    const int64_t r = min(n0 + 16 * j + li, b.rows - 1);
    bc[j] = b.codes + r * b.ld + 16 * lg;
    bs[j] = b.scales + r * b.scales_ld;
  }

  v4f acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};

  // step t's fragment; past the last block: zeros with scale 1
  auto frag4 = [&](const uint8_t* p, int t) -> v8i {
    v4i x = {0, 0, 0, 0};
    if (4 * t + lg < blocks) x = *reinterpret_cast<const v4i*>(p + 64 * (int64_t)t);
    return v8i{x[0], x[1], x[2], x[3], 0, 0, 0, 0};
  };
  auto frag8 = [&](const uint8_t* p, int t) -> v8i {
    v4i x = {0, 0, 0, 0}, y = {0, 0, 0, 0};
    if (4 * t + (lg >> 1) < blocks) x = *reinterpret_cast<const v4i*>(p + 128 * (int64_t)t);
    if (4 * t + 2 + (lg >> 1) < blocks) y = *reinterpret_cast<const v4i*>(p + 128 * (int64_t)t + 64);
    return v8i{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
  };
  auto scale = [&](const uint8_t* p, int t) -> uint32_t { return 4 * t + lg < blocks ? p[4 * t + lg] : 127u; };

  const int nk = (blocks + 3) >> 2;
  const int t0 = (int)((int64_t)nk * wave / W), t1 = (int)((int64_t)nk * (wave + 1) / W);
  for (int t = t0; t < t1; ++t) {
    v8i fa[FM], fb[FN];
    uint32_t sa[FM], sb[FN];
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      fb[j] = frag4(bc[j], t);
      sb[j] = scale(bs[j], t);
    }
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      if constexpr (QA::code == QO_MX_FP4) fa[i] = frag4(ac[i], t);
      else fa[i] = frag8(ac[i], t);
      sa[i] = scale(as[i], t);
    }
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int i = 0; i < FM; ++i) acc[i][j] = mx_mac<QA, OT, 0>(fb[j], fa[i], acc[i][j], sb[j], sa[i]);
  }
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) part[wave][i * FN + j][lane] = acc[i][j];
  __syncthreads();
  for (int f = wave; f < F; f += W) {
    v4f v = part[0][f][lane];
#pragma unroll
    for (int w = 1; w < W; ++w) v += part[w][f][lane];
    mx_store4<OT>(v, out, ldc, bias, a.rows, b.rows, m0 + 16 * (f / FN) + li, n0 + 16 * (f % FN) + 4 * lg);
  }
}

template <class QA, class OT>
void mx_gemm_launch(const MxOperand& a, const MxOperand& b, int blocks, void* out, int64_t ldc, const void* bias,
                    hipStream_t stream) {
  using T = typename OT::T;
  T* o = reinterpret_cast<T*>(out);
  const T* bi = reinterpret_cast<const T*>(bias);
  auto go = [&](auto kernel, int bm, int bn, int threads) {
    const int64_t tiles = ((int64_t)(a.rows + bm - 1) / bm) * ((b.rows + bn - 1) / bn);
    launch(kernel, dim3((unsigned)tiles), dim3(threads), 0, stream, a, b, blocks, o, ldc, bi);
  };
  if (a.rows <= 16) go(mx_gemm_stream<QA, OT, 1, 1, 1, 8>, 16, 16, 512);
  else go(mx_gemm_stream<QA, OT, 4, 2, 1, 4>, 64, 32, 256);
}

}  // namespace

}  // namespace qo

extern "C" int qo_mx_gemm(const void* a, int64_t lda, int a_format, const uint8_t* a_scales, int64_t a_scales_ld,
                          const void* b, int64_t ldb, const uint8_t* b_scales, int64_t b_scales_ld, const void* bias,
                          void* out, int out_dtype, int64_t ldc, int64_t M, int64_t N, int64_t K, void* stream) {
  using namespace qo;
  const char* fn = "qo_mx_gemm";
  if (M < 0 || N < 0 || K < 0 || K % 32 != 0 || M > QO_MX_MAX_FEATURES || N > QO_MX_MAX_FEATURES ||
      K > QO_MX_MAX_FEATURES) {
    qo_set_error("%s: invalid sizes M=%lld N=%lld K=%lld (K a multiple of 32)", fn, (long long)M, (long long)N,
                 (long long)K);
    return QO_ERR_SHAPE;
  }
  if (a_format != QO_MX_FP4 && a_format != QO_MX_FP8) {
    qo_set_error("%s: unknown MX format code %d", fn, a_format);
    return QO_ERR_DTYPE;
  }
  if (out_dtype != QO_DTYPE_F32 && out_dtype != QO_DTYPE_F16 && out_dtype != QO_DTYPE_BF16) {
    qo_set_error("%s: unsupported output dtype code %d", fn, out_dtype);
    return QO_ERR_DTYPE;
  }
  const int64_t row_a = a_format == QO_MX_FP4 ? K / 2 : K;
  if (lda < row_a || ldb < K / 2 || a_scales_ld < K / 32 || b_scales_ld < K / 32 || ldc < N) {
    qo_set_error("%s: row stride below row length (a %lld, b %lld, scales %lld and %lld, out %lld)", fn, (long long)lda,
                 (long long)ldb, (long long)a_scales_ld, (long long)b_scales_ld, (long long)ldc);
    return QO_ERR_SHAPE;
  }
  if (M == 0 || N == 0) return QO_OK;
  if (!out || (K > 0 && (!a || !b || !a_scales || !b_scales))) {
    qo_set_error("%s: NULL pointer argument", fn);
    return QO_ERR_NULL_POINTER;
  }
  if (K > 0 && ((uintptr_t)a % 16 != 0 || (uintptr_t)b % 16 != 0 || lda % 16 != 0 || ldb % 16 != 0)) {
    qo_set_error("%s: codes and their row strides must be multiples of 16 bytes", fn);
    return QO_ERR_ALIGNMENT;
  }
  const MxOperand A = {reinterpret_cast<const uint8_t*>(a), lda, a_scales, a_scales_ld, (int)M};
  const MxOperand B = {reinterpret_cast<const uint8_t*>(b), ldb, b_scales, b_scales_ld, (int)N};
  launch_begin();
  auto with_out = [&](auto q) {
    using QA = decltype(q);
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    const int blocks = (int)(K / 32);
    if (out_dtype == QO_DTYPE_F32) mx_gemm_launch<QA, OutF32>(A, B, blocks, out, ldc, bias, s);
    else if (out_dtype == QO_DTYPE_F16) mx_gemm_launch<QA, OutF16>(A, B, blocks, out, ldc, bias, s);
    else mx_gemm_launch<QA, OutBF16>(A, B, blocks, out, ldc, bias, s);
  };
  if (a_format == QO_MX_FP4) with_out(FP4{});
  else with_out(FP8{});
  return launch_result(fn);
}
