"""Fake (meta) kernels so FakeTensor / torch.compile can trace the operators.

Shapes and dtypes follow the reference (``src/quant_ops/meta_ops.py:22-37``):
int4_matmul -> float16 [M, N]; flatquant_dynamic_quantize -> int32 [T, F/8] or
int8 [T, F] plus float32 scales [T]. The operators this build adds get
fakes of their own. Registered only when the native library defined the
schemas.
"""
import torch

from . import _loader

if _loader.KERNELS_AVAILABLE:

    @torch.library.register_fake("quant_ops::int4_matmul")
    def _int4_matmul_fake(a, b, scale_a, scale_b):
        return a.new_empty((a.size(0), b.size(1)), dtype=torch.float16)

    @torch.library.register_fake("quant_ops::int4_matmul_ex")
    def _int4_matmul_ex_fake(a, b, scale_a, scale_b, out_dtype=None):
        return a.new_empty((a.size(0), b.size(1)), dtype=out_dtype or torch.float16)

    # defined by libraries built from this version on (a stale build lacks it)
    if hasattr(torch.ops.quant_ops, "int4_matmul_bias"):

        @torch.library.register_fake("quant_ops::int4_matmul_bias")
        def _int4_matmul_bias_fake(a, b, scale_a, scale_b, bias, out_dtype=None):
            return a.new_empty((a.size(0), b.size(1)), dtype=out_dtype or torch.float16)

    if hasattr(torch.ops.quant_ops, "w4a4_linear"):

        @torch.library.register_fake("quant_ops::w4a4_linear")
        def _w4a4_linear_fake(x, left_trans, right_trans, weight_packed, weight_scale, clip_ratio=1.0, bias=None):
            return x.new_empty((x.size(0), weight_packed.size(0)), dtype=x.dtype)

    @torch.library.register_fake("quant_ops::flatquant_dynamic_quantize")
    def _flatquant_fake(input_tensor, left_trans, right_trans, clip_ratio=1.0, pack_int32=False):
        tokens, feats = input_tensor.shape
        if pack_int32:
            codes = input_tensor.new_empty((tokens, feats // 8), dtype=torch.int32)
        else:
            codes = input_tensor.new_empty((tokens, feats), dtype=torch.int8)
        return codes, input_tensor.new_empty((tokens,), dtype=torch.float32)

    @torch.library.register_fake("quant_ops::dequantize_int4")
    def _dequant_fake(quantized, scales, packed_int32=False):
        feats = quantized.size(1) * (8 if packed_int32 else 1)
        return quantized.new_empty((quantized.size(0), feats), dtype=torch.float32)

    if hasattr(torch.ops.quant_ops, "mx_quantize"):

        def _mx_outputs(like, tokens, feats, fmt):
            blocks = (feats + 31) // 32
            codes = (like.new_empty((tokens, 16 * blocks), dtype=torch.uint8) if fmt == "mxfp4"
                     else like.new_empty((tokens, 32 * blocks), dtype=torch.float8_e4m3fn))
            return codes, like.new_empty((tokens, (blocks + 15) // 16 * 16), dtype=torch.uint8)[:, :blocks]

        @torch.library.register_fake("quant_ops::mx_quantize")
        def _mx_quantize_fake(input, fmt="mxfp4"):
            return _mx_outputs(input, input.size(0), input.size(1), fmt)

        @torch.library.register_fake("quant_ops::mx_dequantize")
        def _mx_dequantize_fake(codes, scales, features=None, out_dtype=None):
            feats = scales.size(1) * 32 if features is None else features
            return codes.new_empty((codes.size(0), feats), dtype=out_dtype or torch.float32)

        @torch.library.register_fake("quant_ops::rms_norm_mx_quantize")
        def _rms_norm_mx_fake(x, weight, eps=1e-6, fmt="mxfp8"):
            return _mx_outputs(x, x.size(0), x.size(1), fmt)

        @torch.library.register_fake("quant_ops::add_rms_norm_mx_quantize")
        def _add_rms_norm_mx_fake(x, residual, weight, eps=1e-6, fmt="mxfp8"):
            return (*_mx_outputs(x, x.size(0), x.size(1), fmt), x.new_empty(tuple(x.shape)))

        @torch.library.register_fake("quant_ops::swiglu_mx_quantize")
        def _swiglu_mx_fake(gate_up, fmt="mxfp8"):
            return _mx_outputs(gate_up, gate_up.size(0), gate_up.size(1) // 2, fmt)

        @torch.library.register_fake("quant_ops::mx_matmul")
        def _mx_matmul_fake(a, a_scales, b, b_scales, bias=None, out_dtype=None):
            return a.new_empty((a.size(0), b.size(0)), dtype=out_dtype or torch.bfloat16)

    if hasattr(torch.ops.quant_ops, "kv4_append"):

        @torch.library.register_fake("quant_ops::kv4_append")
        def _kv4_append_fake(k_codes, v_codes, params, k, v, slots, positions=None, cos=None, sin=None, q=None,
                             interleaved=False):
            return k.new_empty((0, 0) if q is None else tuple(q.shape))

        @torch.library.register_fake("quant_ops::kv4_read")
        def _kv4_read_fake(k_codes, v_codes, params, slots, out_dtype=None):
            shape = (slots.size(0), k_codes.size(1), 2 * k_codes.size(3))
            dtype = out_dtype or torch.float32
            return params.new_empty(shape, dtype=dtype), params.new_empty(shape, dtype=dtype)

        @torch.library.register_fake("quant_ops::kv4_attention")
        def _kv4_attention_fake(q, k_codes, v_codes, params, page_table, lengths, scale, q_starts=None, window=0):
            return q.new_empty(tuple(q.shape))
