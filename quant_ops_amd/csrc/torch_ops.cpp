// torch operator registration for the quant_ops namespace, backed by the C ABI
// of libquant_ops_hip.so.
//
// Schemas are those of the reference (flatquant/kernels/cuda_quant_kernel.cu:407-409,
// int4_matmul/kernels/cuda_int4_matmul_kernel.cu:207-209), so callers of
// torch.ops.quant_ops.* and graph captures see the same operators. The others
// are additions of this build: int4_matmul_ex (output dtype choice),
// int4_matmul_bias (bias in the epilogue), w4a4_linear (the linear layer's
// quantize + GEMM as one operator), dequantize_int4 (a device kernel
// for the reference's Python function) and the microscaled operators (mx_*,
// *_mx_quantize).
//
// Unlike the reference, kernels go to the caller's current HIP stream and the
// host is never synchronised (cuda_quant_kernel.cu:379-385 synchronised the
// stream after launching on the legacy default stream).
#include <ATen/ATen.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>

#include "quant_ops_hip.h"

namespace {

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return QO_DTYPE_F32;
    case at::kHalf: return QO_DTYPE_F16;
    case at::kBFloat16: return QO_DTYPE_BF16;
    default: return -1;
  }
}

void check_status(int st, const char* op) {
  TORCH_CHECK(st == QO_OK, op, " failed: ", qo_status_string(st), ": ", qo_last_error());
}

void* current_stream(const at::Tensor& t) {
  return reinterpret_cast<void*>(c10::hip::getCurrentHIPStream(t.device().index()).stream());
}

// The FP6 route's workspace from the caching allocator (its blocks are 512-byte
// aligned); undefined where no byte is needed, or where memory does not allow
// it: the GEMM then takes the kernels that need none, with the same results.
at::Tensor gemm_workspace(int64_t bytes, const at::Tensor& like) {
  if (bytes <= 0) return at::Tensor();
  try {
    return at::empty({bytes}, like.options().dtype(at::kByte));
  } catch (const c10::OutOfMemoryError&) {
    return at::Tensor();
  }
}

// Same checks as cuda_kronecker_quant_int8 (cuda_quant_kernel.cu:324-329), plus
// the dtype agreement torch::matmul enforces there.
std::tuple<at::Tensor, at::Tensor> flatquant_dynamic_quantize(const at::Tensor& input, const at::Tensor& left_trans,
                                                              const at::Tensor& right_trans, double clip_ratio,
                                                              bool pack_int32) {
  TORCH_CHECK(input.dim() == 2, "flatquant_dynamic_quantize: input must be 2-D [tokens, features], got ",
              input.sizes());
  TORCH_CHECK(left_trans.dim() == 2 && left_trans.size(0) == left_trans.size(1),
              "flatquant_dynamic_quantize: left_trans must be square [M, M]");
  TORCH_CHECK(right_trans.dim() == 2 && right_trans.size(0) == right_trans.size(1),
              "flatquant_dynamic_quantize: right_trans must be square [N, N]");
  const int64_t T = input.size(0);
  const int64_t M = left_trans.size(0), N = right_trans.size(0), F = M * N;
  TORCH_CHECK(input.size(-1) == F, "Input last dimension must equal M*N");
  TORCH_CHECK(F % 8 == 0 || !pack_int32, "Features must be divisible by 8 for int32 packing");
  const int code = dtype_code(input.scalar_type());
  TORCH_CHECK(code >= 0, "flatquant_dynamic_quantize: input dtype must be float32, float16 or bfloat16, got ",
              input.scalar_type());
  TORCH_CHECK(left_trans.scalar_type() == input.scalar_type() && right_trans.scalar_type() == input.scalar_type(),
              "flatquant_dynamic_quantize: left_trans / right_trans must have the input dtype ",
              input.scalar_type());
  TORCH_CHECK(input.is_cuda(), "flatquant_dynamic_quantize: input must be a GPU tensor");
  c10::DeviceGuard guard(input.device());

  at::Tensor x = input.stride(1) == 1 && input.stride(0) >= F ? input : input.contiguous();
  at::Tensor L = left_trans.to(input.device()).contiguous();
  at::Tensor R = right_trans.to(input.device()).contiguous();
  at::Tensor scales = at::empty({T}, input.options().dtype(at::kFloat));
  at::Tensor codes = pack_int32 ? at::empty({T, F / 8}, input.options().dtype(at::kInt))
                                : at::empty({T, F}, input.options().dtype(at::kChar));
  const int64_t ld = T > 0 ? x.stride(0) : F;
  check_status(qo_flatquant_quantize(x.data_ptr(), code, T, ld, L.data_ptr(), R.data_ptr(), (int)M, (int)N,
                                     (float)clip_ratio, pack_int32 ? 1 : 0, codes.data_ptr(),
                                     scales.data_ptr<float>(), current_stream(input)),
               "flatquant_dynamic_quantize");
  return {codes, scales};
}

// Same checks as cuda_int4_matmul (cuda_int4_matmul_kernel.cu:136-153); scales
// may also be float16 / bfloat16 (the fallback promotes them), and b may be the
// transposed view of a [N, K/8] weight.
at::Tensor int4_matmul_impl(const at::Tensor& a, const at::Tensor& b, const at::Tensor& scale_a,
                            const at::Tensor& scale_b, at::ScalarType out_dtype,
                            const std::optional<at::Tensor>& bias = std::nullopt) {
  TORCH_CHECK(a.is_cuda(), "a_packed must be on CUDA");
  TORCH_CHECK(b.is_cuda(), "b_packed must be on CUDA");
  TORCH_CHECK(scale_a.is_cuda(), "scale_a must be on CUDA");
  TORCH_CHECK(scale_b.is_cuda(), "scale_b must be on CUDA");
  TORCH_CHECK(a.scalar_type() == at::kInt, "a_packed must be int32");
  TORCH_CHECK(b.scalar_type() == at::kInt, "b_packed must be int32");
  const int sad = dtype_code(scale_a.scalar_type()), sbd = dtype_code(scale_b.scalar_type());
  TORCH_CHECK(sad >= 0, "scale_a must be float32, float16 or bfloat16");
  TORCH_CHECK(sbd >= 0, "scale_b must be float32, float16 or bfloat16");
  const int od = dtype_code(out_dtype);
  TORCH_CHECK(od >= 0, "out_dtype must be float16, bfloat16 or float32");
  TORCH_CHECK(a.dim() == 2 && b.dim() == 2, "a_packed and b_packed must be 2-D");
  const int64_t M = a.size(0), KP = a.size(1), N = b.size(1), K = KP * 8;
  TORCH_CHECK(b.size(0) == KP, "Matrix dimensions mismatch");
  TORCH_CHECK(scale_a.size(0) == M && scale_a.numel() == M, "scale_a dimension mismatch");
  TORCH_CHECK(scale_b.size(0) == N && scale_b.numel() == N, "scale_b dimension mismatch");
  c10::DeviceGuard guard(a.device());

  at::Tensor A = (a.stride(1) == 1 && (M <= 1 || a.stride(0) >= KP)) ? a : a.contiguous();
  at::Tensor B = b;
  if (!(b.stride(0) == 1 || b.stride(1) == 1)) B = b.contiguous();
  at::Tensor sa = scale_a.contiguous(), sb = scale_b.contiguous();
  at::Tensor out = at::empty({M, N}, a.options().dtype(out_dtype));
  int64_t bsp = B.stride(0), bsn = B.stride(1);
  if (KP == 1) bsp = 1;     // a single packed row: either stride works
  if (N == 1) bsn = 1;
  const int64_t lda = M > 0 ? A.stride(0) : KP;
  at::Tensor bv;
  if (bias.has_value()) {
    TORCH_CHECK(bias->is_cuda() && bias->numel() == N, "bias must be a GPU tensor of N elements");
    // the reference adds bias.to(output dtype) to the output
    bv = bias->to(out_dtype).contiguous();
  }
  const int64_t ws_bytes = qo_int4_gemm_workspace_needed(A.data_ptr<int32_t>(), lda, B.data_ptr<int32_t>(), bsp, bsn,
                                                         out.data_ptr(), od, N, M, N, K);
  at::Tensor ws = gemm_workspace(ws_bytes, a);
  check_status(qo_int4_gemm_ws(A.data_ptr<int32_t>(), lda, B.data_ptr<int32_t>(), bsp, bsn, sa.data_ptr(), sad,
                               sb.data_ptr(), sbd, bv.defined() ? bv.data_ptr() : nullptr, out.data_ptr(), od, N, M,
                               N, K, ws.defined() ? ws.data_ptr() : nullptr, ws_bytes, current_stream(a)),
               bias.has_value() ? "int4_matmul_bias" : "int4_matmul");
  return out;
}

at::Tensor int4_matmul(const at::Tensor& a, const at::Tensor& b, const at::Tensor& scale_a,
                       const at::Tensor& scale_b) {
  return int4_matmul_impl(a, b, scale_a, scale_b, at::kHalf);
}

at::Tensor int4_matmul_ex(const at::Tensor& a, const at::Tensor& b, const at::Tensor& scale_a,
                          const at::Tensor& scale_b, std::optional<at::ScalarType> out_dtype) {
  return int4_matmul_impl(a, b, scale_a, scale_b, out_dtype.value_or(at::kHalf));
}

at::Tensor int4_matmul_bias(const at::Tensor& a, const at::Tensor& b, const at::Tensor& scale_a,
                            const at::Tensor& scale_b, const at::Tensor& bias,
                            std::optional<at::ScalarType> out_dtype) {
  return int4_matmul_impl(a, b, scale_a, scale_b, out_dtype.value_or(at::kHalf), bias);
}

// The W4A4 linear layer (w4a4_flatquant_dynamic.py:168-266 on the GPU path):
// x [T, M*N], weight_packed int32 [out, M*N/8] (the GEMM uses its W.t() view),
// weight_scale [out] (float32 / float16 / bfloat16), optional bias; output in
// x's dtype.
at::Tensor w4a4_linear(const at::Tensor& x, const at::Tensor& left_trans, const at::Tensor& right_trans,
                       const at::Tensor& weight_packed, const at::Tensor& weight_scale, double clip_ratio,
                       const std::optional<at::Tensor>& bias) {
  TORCH_CHECK(x.dim() == 2, "w4a4_linear: x must be 2-D [tokens, features], got ", x.sizes());
  TORCH_CHECK(left_trans.dim() == 2 && left_trans.size(0) == left_trans.size(1),
              "w4a4_linear: left_trans must be square [M, M]");
  TORCH_CHECK(right_trans.dim() == 2 && right_trans.size(0) == right_trans.size(1),
              "w4a4_linear: right_trans must be square [N, N]");
  const int64_t T = x.size(0), M = left_trans.size(0), N = right_trans.size(0), F = M * N;
  TORCH_CHECK(x.size(1) == F, "Input last dimension must equal M*N");
  TORCH_CHECK(F % 8 == 0, "Features must be divisible by 8 for int32 packing");
  const int code = dtype_code(x.scalar_type());
  TORCH_CHECK(code >= 0, "w4a4_linear: x dtype must be float32, float16 or bfloat16, got ", x.scalar_type());
  TORCH_CHECK(left_trans.scalar_type() == x.scalar_type() && right_trans.scalar_type() == x.scalar_type(),
              "w4a4_linear: left_trans / right_trans must have x's dtype ", x.scalar_type());
  TORCH_CHECK(weight_packed.scalar_type() == at::kInt && weight_packed.dim() == 2 && weight_packed.size(1) * 8 == F,
              "w4a4_linear: weight_packed must be int32 [out_features, M*N/8]");
  const int64_t NO = weight_packed.size(0);
  const int swd = dtype_code(weight_scale.scalar_type());
  TORCH_CHECK(swd >= 0, "w4a4_linear: weight_scale must be float32, float16 or bfloat16");
  TORCH_CHECK(weight_scale.numel() == NO, "w4a4_linear: weight_scale must hold one value per output channel");
  TORCH_CHECK(x.is_cuda() && weight_packed.is_cuda() && weight_scale.is_cuda(),
              "w4a4_linear: x, weight_packed and weight_scale must be GPU tensors");
  c10::DeviceGuard guard(x.device());

  at::Tensor X = x.stride(1) == 1 && x.stride(0) >= F ? x : x.contiguous();
  at::Tensor L = left_trans.to(x.device()).contiguous();
  at::Tensor R = right_trans.to(x.device()).contiguous();
  at::Tensor W = weight_packed.stride(1) == 1 && weight_packed.stride(0) >= F / 8 ? weight_packed
                                                                                  : weight_packed.contiguous();
  at::Tensor sw = weight_scale.reshape({NO}).contiguous();
  at::Tensor bv;
  if (bias.has_value()) {
    TORCH_CHECK(bias->is_cuda() && bias->numel() == NO, "bias must be a GPU tensor of out_features elements");
    bv = bias->to(x.scalar_type()).reshape({NO}).contiguous();   // the reference adds bias.to(dtype)
  }
  at::Tensor codes = at::empty({T, F / 8}, x.options().dtype(at::kInt));
  at::Tensor scales = at::empty({T}, x.options().dtype(at::kFloat));
  at::Tensor out = at::empty({T, NO}, x.options());
  // the GEMM's FP6 route (0 bytes: not taken)
  const int64_t ws_bytes =
      qo_int4_gemm_workspace_needed(codes.data_ptr<int32_t>(), F / 8, W.data_ptr<int32_t>(), 1,
                                    NO > 0 ? W.stride(0) : F / 8, out.data_ptr(), code, NO, T, NO, F);
  at::Tensor ws = gemm_workspace(ws_bytes, x);
  check_status(qo_w4a4_linear_ws(X.data_ptr(), code, T, T > 0 ? X.stride(0) : F, L.data_ptr(), R.data_ptr(), (int)M,
                                 (int)N, (float)clip_ratio, W.data_ptr<int32_t>(), NO > 0 ? W.stride(0) : F / 8, NO,
                                 sw.data_ptr(), swd, bv.defined() ? bv.data_ptr() : nullptr,
                                 codes.data_ptr<int32_t>(), scales.data_ptr<float>(), out.data_ptr(), NO,
                                 ws.defined() ? ws.data_ptr() : nullptr, ws_bytes, current_stream(x)),
               "w4a4_linear");
  return out;
}

at::Tensor dequantize_int4(const at::Tensor& quantized, const at::Tensor& scales, bool packed_int32) {
  TORCH_CHECK(quantized.is_cuda() && scales.is_cuda(), "dequantize_int4: tensors must be on the GPU");
  TORCH_CHECK(quantized.dim() == 2, "dequantize_int4: quantized must be 2-D");
  TORCH_CHECK(quantized.scalar_type() == (packed_int32 ? at::kInt : at::kChar),
              "dequantize_int4: quantized must be ", packed_int32 ? "int32" : "int8");
  const int sd = dtype_code(scales.scalar_type());
  TORCH_CHECK(sd >= 0, "dequantize_int4: scales must be float32, float16 or bfloat16");
  const int64_t T = quantized.size(0);
  const int64_t F = packed_int32 ? quantized.size(1) * 8 : quantized.size(1);
  TORCH_CHECK(scales.numel() == T, "dequantize_int4: scales must hold one value per token");
  c10::DeviceGuard guard(quantized.device());
  at::Tensor q = quantized.contiguous();
  at::Tensor s = scales.contiguous();
  at::Tensor out = at::empty({T, F}, quantized.options().dtype(at::kFloat));
  check_status(qo_dequantize_int4(q.data_ptr(), packed_int32 ? 1 : 0, s.data_ptr(), sd, T, F,
                                  out.data_ptr<float>(), current_stream(quantized)),
               "dequantize_int4");
  return out;
}

// ---------------------------------------------------------------------------
// Microscaled formats: codes are uint8 (FP4, two per byte) or float8_e4m3fn
// (FP8), scales uint8, one per 32 values; rows are padded to whole blocks.
// ---------------------------------------------------------------------------
int mx_format(c10::string_view fmt, const char* op) {
  if (fmt == "mxfp4") return QO_MX_FP4;
  TORCH_CHECK(fmt == "mxfp8", op, ": fmt must be \"mxfp4\" or \"mxfp8\", got \"", fmt, "\"");
  return QO_MX_FP8;
}

int mx_codes_format(const at::Tensor& codes, const char* op, const char* name) {
  if (codes.scalar_type() == at::kByte) return QO_MX_FP4;
  TORCH_CHECK(codes.scalar_type() == at::kFloat8_e4m3fn, op, ": ", name,
              " must be uint8 (FP4 codes) or float8_e4m3fn (FP8 codes), got ", codes.scalar_type());
  return QO_MX_FP8;
}

// Uninitialized rows from the caching allocator, without the dispatcher's way to it (of the
// host's time of a small call, which bounds it, a tenth).
at::Tensor mx_empty(int64_t rows, int64_t columns, at::ScalarType dtype, at::Device device) {
  return at::detail::empty_cuda({rows, columns}, dtype, device, std::nullopt);
}

// Empty codes and scales for [tokens, features]. Rows of scales stand a multiple of
// 16 bytes apart, as mx_matmul reads them: the tensor is made with the padding and narrowed.
std::tuple<at::Tensor, at::Tensor> mx_outputs(const at::Tensor& like, int64_t tokens, int64_t features, int format) {
  const int64_t blocks = (features + 31) / 32, pad = (blocks + 15) / 16 * 16;
  at::Tensor codes = format == QO_MX_FP4 ? mx_empty(tokens, 16 * blocks, at::kByte, like.device())
                                         : mx_empty(tokens, 32 * blocks, at::kFloat8_e4m3fn, like.device());
  at::Tensor scales = mx_empty(tokens, pad, at::kByte, like.device());
  if (pad != blocks) scales.unsafeGetTensorImpl()->set_sizes_and_strides(at::IntArrayRef{tokens, blocks}, at::IntArrayRef{pad, 1});
  return {std::move(codes), std::move(scales)};
}
int64_t mx_scales_ld(const at::Tensor& s) { return std::max(s.stride(0), s.size(1)); }

void check_rows(const at::Tensor& x, const char* op, const char* name) {
  TORCH_CHECK(x.dim() == 2, op, ": ", name, " must be 2-D [tokens, features], got ", x.sizes());
  TORCH_CHECK(x.is_cuda(), op, ": ", name, " must be a GPU tensor");
  TORCH_CHECK(dtype_code(x.scalar_type()) >= 0, op, ": ", name, " dtype must be float32, float16 or bfloat16, got ",
              x.scalar_type());
}

// Rows with unit inner stride that do not overlap; x itself where it has them.
at::Tensor mx_rows(const at::Tensor& x) {
  return x.stride(1) == 1 && (x.size(0) <= 1 || x.stride(0) >= x.size(1)) ? x : x.contiguous();
}
int64_t mx_ld(const at::Tensor& x) { return x.size(0) > 1 ? x.stride(0) : x.size(1); }

std::tuple<at::Tensor, at::Tensor> mx_quantize(const at::Tensor& input, c10::string_view fmt) {
  check_rows(input, "mx_quantize", "input");
  const int format = mx_format(fmt, "mx_quantize");
  c10::DeviceGuard guard(input.device());
  at::Tensor x = mx_rows(input);
  auto [codes, scales] = mx_outputs(x, x.size(0), x.size(1), format);
  check_status(qo_mx_quantize(x.data_ptr(), dtype_code(x.scalar_type()), x.size(0), x.size(1), mx_ld(x), format,
                              codes.data_ptr(), scales.data_ptr<uint8_t>(), mx_scales_ld(scales), current_stream(x)),
               "mx_quantize");
  return {codes, scales};
}

at::Tensor mx_dequantize(const at::Tensor& codes, const at::Tensor& scales, std::optional<int64_t> features,
                         std::optional<at::ScalarType> out_dtype) {
  TORCH_CHECK(codes.is_cuda() && scales.device() == codes.device(), "mx_dequantize: tensors must be on one GPU");
  TORCH_CHECK(codes.dim() == 2 && scales.dim() == 2, "mx_dequantize: codes and scales must be 2-D");
  const int format = mx_codes_format(codes, "mx_dequantize", "codes");
  TORCH_CHECK(scales.scalar_type() == at::kByte, "mx_dequantize: scales must be uint8");
  const int64_t T = codes.size(0), blocks = scales.size(1);
  TORCH_CHECK(scales.size(0) == T && codes.size(1) == blocks * (format == QO_MX_FP4 ? 16 : 32),
              "mx_dequantize: codes ", codes.sizes(), " and scales ", scales.sizes(), " do not match");
  const int64_t F = features.value_or(32 * blocks);
  TORCH_CHECK((F + 31) / 32 == blocks && F >= 0, "mx_dequantize: features (", F, ") must fill the ", blocks, " blocks of a row");
  const at::ScalarType dtype = out_dtype.value_or(at::kFloat);
  TORCH_CHECK(dtype_code(dtype) >= 0, "mx_dequantize: out_dtype must be float32, float16 or bfloat16");
  c10::DeviceGuard guard(codes.device());
  at::Tensor q = codes.contiguous(), s = mx_rows(scales);
  if (reinterpret_cast<uintptr_t>(q.data_ptr()) % 8 != 0) q = q.clone();
  at::Tensor out = mx_empty(T, F, dtype, codes.device());
  check_status(qo_mx_dequantize(q.data_ptr(), s.data_ptr<uint8_t>(), mx_scales_ld(s), format, T, F, out.data_ptr(), dtype_code(dtype),
                                current_stream(codes)),
               "mx_dequantize");
  return out;
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> rms_norm_mx_impl(const at::Tensor& input, const at::Tensor* residual,
                                                                const at::Tensor& weight, double eps,
                                                                c10::string_view fmt, const char* op) {
  check_rows(input, op, "x");
  const int format = mx_format(fmt, op);
  const int64_t T = input.size(0), F = input.size(1);
  TORCH_CHECK(weight.dim() == 1 && weight.size(0) == F, op, ": weight must hold one value per feature (", F, "), got ",
              weight.sizes());
  TORCH_CHECK(weight.device() == input.device() && dtype_code(weight.scalar_type()) >= 0, op,
              ": weight must be float32, float16 or bfloat16 on x's device");
  if (residual)
    TORCH_CHECK(residual->sizes() == input.sizes() && residual->scalar_type() == input.scalar_type() &&
                    residual->device() == input.device(),
                op, ": residual must have x's shape, dtype and device");
  c10::DeviceGuard guard(input.device());
  at::Tensor x = mx_rows(input), w = weight.contiguous(), res, h;
  if (residual) {
    res = mx_rows(*residual);
    h = mx_empty(T, F, input.scalar_type(), input.device());
  }
  auto [codes, scales] = mx_outputs(x, T, F, format);
  check_status(qo_rms_norm_mx_quantize(x.data_ptr(), residual ? res.data_ptr() : nullptr, dtype_code(x.scalar_type()),
                                       T, F, mx_ld(x), residual ? mx_ld(res) : 0, w.data_ptr(),
                                       dtype_code(w.scalar_type()), (float)eps, format, codes.data_ptr(),
                                       scales.data_ptr<uint8_t>(), mx_scales_ld(scales), residual ? h.data_ptr() : nullptr,
                                       current_stream(x)),
               op);
  return {codes, scales, h};
}

std::tuple<at::Tensor, at::Tensor> rms_norm_mx_quantize(const at::Tensor& x, const at::Tensor& weight, double eps,
                                                        c10::string_view fmt) {
  auto [codes, scales, h] = rms_norm_mx_impl(x, nullptr, weight, eps, fmt, "rms_norm_mx_quantize");
  return {codes, scales};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> add_rms_norm_mx_quantize(const at::Tensor& x, const at::Tensor& residual,
                                                                        const at::Tensor& weight, double eps,
                                                                        c10::string_view fmt) {
  return rms_norm_mx_impl(x, &residual, weight, eps, fmt, "add_rms_norm_mx_quantize");
}

std::tuple<at::Tensor, at::Tensor> swiglu_mx_quantize(const at::Tensor& gate_up, c10::string_view fmt) {
  check_rows(gate_up, "swiglu_mx_quantize", "gate_up");
  const int format = mx_format(fmt, "swiglu_mx_quantize");
  TORCH_CHECK(gate_up.size(1) % 2 == 0, "swiglu_mx_quantize: gate_up must hold two halves, got ", gate_up.sizes());
  c10::DeviceGuard guard(gate_up.device());
  at::Tensor x = mx_rows(gate_up);
  const int64_t T = x.size(0), F = x.size(1) / 2;
  auto [codes, scales] = mx_outputs(x, T, F, format);
  check_status(qo_swiglu_mx_quantize(x.data_ptr(), dtype_code(x.scalar_type()), T, F, mx_ld(x), format,
                                     codes.data_ptr(), scales.data_ptr<uint8_t>(), mx_scales_ld(scales), current_stream(x)),
               "swiglu_mx_quantize");
  return {codes, scales};
}

// Codes whose rows the GEMM can read: 16-byte aligned, unit inner stride, not overlapping.
at::Tensor mx_gemm_rows(const at::Tensor& codes) {
  const bool fits = codes.stride(1) == 1 && reinterpret_cast<uintptr_t>(codes.data_ptr()) % 16 == 0 &&
                    (codes.size(0) <= 1 || (codes.stride(0) >= codes.size(1) && codes.stride(0) % 16 == 0));
  return fits ? codes : codes.clone(at::MemoryFormat::Contiguous);
}

// Scales as the GEMM of `rows` rows reads them: with many, 16-byte aligned rows that are
// readable up to a multiple of 16 bytes.
at::Tensor mx_gemm_scales(const at::Tensor& scales, int64_t rows) {
  at::Tensor s = mx_rows(scales);
  if (rows <= QO_MX_GEMM_FEW_ROWS) return s;
  const int64_t n = s.size(0), blocks = s.size(1), pad = (blocks + 15) / 16 * 16;
  const int64_t stored = (int64_t)s.storage().nbytes() - s.storage_offset();
  if (reinterpret_cast<uintptr_t>(s.data_ptr()) % 16 == 0 && mx_scales_ld(s) % 16 == 0 &&
      (n - 1) * mx_scales_ld(s) + pad <= stored)
    return s;
  at::Tensor padded = at::empty({n, pad}, s.options());
  at::Tensor view = padded.narrow(1, 0, blocks);
  view.copy_(s);
  return view;
}

at::Tensor mx_matmul(const at::Tensor& a, const at::Tensor& a_scales, const at::Tensor& b, const at::Tensor& b_scales,
                     const std::optional<at::Tensor>& bias, std::optional<at::ScalarType> out_dtype) {
  TORCH_CHECK(a.is_cuda() && a_scales.device() == a.device() && b.device() == a.device() &&
                  b_scales.device() == a.device(),
              "mx_matmul: a, b and their scales must be on one GPU");
  TORCH_CHECK(a.dim() == 2 && a_scales.dim() == 2 && b.dim() == 2 && b_scales.dim() == 2,
              "mx_matmul: a, b and their scales must be 2-D");
  const int format = mx_codes_format(a, "mx_matmul", "a");
  TORCH_CHECK(b.scalar_type() == at::kByte, "mx_matmul: b must be uint8 (FP4 codes), got ", b.scalar_type());
  TORCH_CHECK(a_scales.scalar_type() == at::kByte && b_scales.scalar_type() == at::kByte,
              "mx_matmul: scales must be uint8");
  const int64_t M = a.size(0), N = b.size(0), blocks = a_scales.size(1), K = 32 * blocks;
  TORCH_CHECK(a_scales.size(0) == M && a.size(1) == (format == QO_MX_FP4 ? K / 2 : K), "mx_matmul: a ", a.sizes(),
              " and a_scales ", a_scales.sizes(), " do not match");
  TORCH_CHECK(b_scales.size(0) == N && b_scales.size(1) == blocks && b.size(1) == K / 2, "mx_matmul: b ", b.sizes(),
              " and b_scales ", b_scales.sizes(), " do not match a's ", blocks, " blocks");
  const at::ScalarType dtype = out_dtype.value_or(at::kBFloat16);
  const int od = dtype_code(dtype);
  TORCH_CHECK(od >= 0, "mx_matmul: out_dtype must be float16, bfloat16 or float32");
  c10::DeviceGuard guard(a.device());
  at::Tensor A = mx_gemm_rows(a), B = mx_gemm_rows(b), sa = mx_gemm_scales(a_scales, M), sb = mx_gemm_scales(b_scales, M), bv;
  if (bias.has_value()) {
    TORCH_CHECK(bias->device() == a.device() && bias->numel() == N, "mx_matmul: bias must hold N (", N,
                ") elements on a's device");
    bv = bias->to(dtype).reshape({N}).contiguous();
  }
  at::Tensor out = mx_empty(M, N, dtype, a.device());
  const int64_t ws_bytes = qo_mx_gemm_workspace_size(M, N, K, format);
  at::Tensor ws = gemm_workspace(ws_bytes, a);
  check_status(qo_mx_gemm(A.data_ptr(), mx_ld(A), format, sa.data_ptr<uint8_t>(), mx_scales_ld(sa), B.data_ptr(),
                          mx_ld(B), sb.data_ptr<uint8_t>(), mx_scales_ld(sb), bv.defined() ? bv.data_ptr() : nullptr, out.data_ptr(), od,
                          N, M, N, K, ws.defined() ? ws.data_ptr() : nullptr, ws_bytes, current_stream(a)),
               "mx_matmul");
  return out;
}

}  // namespace

TORCH_LIBRARY(quant_ops, m) {
  m.def(
      "flatquant_dynamic_quantize(Tensor input, Tensor left_trans, Tensor right_trans, float clip_ratio=1, "
      "bool pack_int32=False) -> (Tensor, Tensor)");
  m.def("int4_matmul(Tensor a, Tensor b, Tensor scale_a, Tensor scale_b) -> Tensor");
  m.def("int4_matmul_ex(Tensor a, Tensor b, Tensor scale_a, Tensor scale_b, ScalarType? out_dtype=None) -> Tensor");
  m.def("dequantize_int4(Tensor quantized, Tensor scales, bool packed_int32=False) -> Tensor");
  m.def(
      "int4_matmul_bias(Tensor a, Tensor b, Tensor scale_a, Tensor scale_b, Tensor bias, "
      "ScalarType? out_dtype=None) -> Tensor");
  m.def(
      "w4a4_linear(Tensor x, Tensor left_trans, Tensor right_trans, Tensor weight_packed, Tensor weight_scale, "
      "float clip_ratio=1, Tensor? bias=None) -> Tensor");
  m.def("mx_quantize(Tensor input, str fmt=\"mxfp4\") -> (Tensor, Tensor)");
  m.def("mx_dequantize(Tensor codes, Tensor scales, int? features=None, ScalarType? out_dtype=None) -> Tensor");
  m.def("rms_norm_mx_quantize(Tensor x, Tensor weight, float eps=1e-06, str fmt=\"mxfp8\") -> (Tensor, Tensor)");
  m.def(
      "add_rms_norm_mx_quantize(Tensor x, Tensor residual, Tensor weight, float eps=1e-06, str fmt=\"mxfp8\") -> "
      "(Tensor, Tensor, Tensor)");
  m.def("swiglu_mx_quantize(Tensor gate_up, str fmt=\"mxfp8\") -> (Tensor, Tensor)");
  m.def(
      "mx_matmul(Tensor a, Tensor a_scales, Tensor b, Tensor b_scales, Tensor? bias=None, "
      "ScalarType? out_dtype=None) -> Tensor");
}

TORCH_LIBRARY_IMPL(quant_ops, CUDA, m) {
  m.impl("flatquant_dynamic_quantize", &flatquant_dynamic_quantize);
  m.impl("int4_matmul", &int4_matmul);
  m.impl("int4_matmul_ex", &int4_matmul_ex);
  m.impl("dequantize_int4", &dequantize_int4);
  m.impl("int4_matmul_bias", &int4_matmul_bias);
  m.impl("w4a4_linear", &w4a4_linear);
  m.impl("mx_quantize", &mx_quantize);
  m.impl("mx_dequantize", &mx_dequantize);
  m.impl("rms_norm_mx_quantize", &rms_norm_mx_quantize);
  m.impl("add_rms_norm_mx_quantize", &add_rms_norm_mx_quantize);
  m.impl("swiglu_mx_quantize", &swiglu_mx_quantize);
  m.impl("mx_matmul", &mx_matmul);
}
