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
// (rows): lane l's four sums are row l % 16, columns 4 (l / 16) + 0 .. 3. SB, SA:
// the byte of the scale operands.
template <class QA, int SB, int SA>
__device__ inline v4f mx_mfma(const v8i& b, const v8i& a, v4f acc, uint32_t sb, uint32_t sa) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b, a, acc, 4, kMfmaFormat<QA>, SB, (int)sb, SA, (int)sa);
}

// mx_mfma, FP8 fragments in two halves where OT asks for it.
template <class QA, class OT, int SB, int SA>
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
    acc = mx_mfma<QA, SB, SA>(b, lo, acc, sb, sa);
    return mx_mfma<QA, SB, SA>(b, hi, acc, sb, sa);
  } else {
    return mx_mfma<QA, SB, SA>(b, a, acc, sb, sa);
  }
}

// 32 x 32 blocks of FP4 fragments of 32 rows x 64: lane l has row l % 32, the 16 bytes
// of block l / 32 and that block's scale in byte S of its operands; its sums
// are row l % 32, columns 8 e + 4 (l / 32) + 0 .. 3, e = 0 .. 3.
typedef float v16f __attribute__((ext_vector_type(16)));
template <int S>
__device__ inline v16f mx_mfma32(const v8i& b, const v8i& a, v16f acc, uint32_t sb, uint32_t sa) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(b, a, acc, 4, 4, S, (int)sb, S, (int)sa);
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
      for (int i = 0; i < FM; ++i) acc[i][j] = mx_mac<QA, OT, 0, 0>(fb[j], fa[i], acc[i][j], sb[j], sa[i]);
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

// ---------------------------------------------------------------------------
// Scale operands of a wave's fragments. Lane r loads the 16 bytes of a quad of
// k-steps (16 blocks) of row r of 64: dword s holds step s's blocks, byte j block j.
// ---------------------------------------------------------------------------

// Blocks 16 q .. of the row at p; blocks past the last are 0.
__device__ inline v4i mx_load_scales(const uint8_t* p, int q, int blocks) {
  v4i v = {0, 0, 0, 0};
  p += 16 * (int64_t)q;
  const int left = blocks - 16 * q;
  if (left >= 16) {
    __builtin_memcpy(&v, p, 16);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (left >= 4 * i + 4) {
        int d;
        __builtin_memcpy(&d, p + 4 * i, 4);
        v[i] = d;
      } else {
#pragma unroll
        for (int j = 0; j < 3; ++j)
          if (4 * i + j < left) v[i] |= (int)p[4 * i + j] << (8 * j);
      }
    }
  }
  return v;
}

// The same where the row has 16 blocks or more, as one load whatever q (q's
// blocks, or the row's last 16), and how far to shift what it gave.
__device__ inline v4i mx_load_scales_end(const uint8_t* p, int q, int blocks) {
  v4i v;
  __builtin_memcpy(&v, p + min(16 * q, blocks - 16), 16);
  return v;
}
__device__ inline void mx_shift_scales(v4i& v, int bytes) {   // 1 .. 15, zeros come in
  const int d = bytes >> 2, r = bytes & 3;
  uint32_t x[5];
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = i + d == 0 ? v[0] : i + d == 1 ? v[1] : i + d == 2 ? v[2] : i + d == 3 ? v[3] : 0;
  x[4] = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = (int)__builtin_amdgcn_alignbyte(x[i + 1], x[i], r);
}

struct MxScales {
  uint32_t w[4];
};

// For fragments of 16 rows x 128: the MFMA of step s and fragment f wants in lane
// g * 16 + r byte g of row 16 f + r, so bytes and groups of 16 lanes change places:
// two rounds of byte permutes and lane swaps, for two steps at a time. Word 2 (s / 2)
// + f % 2 then holds step s, fragment f in byte 2 (s % 2) + f / 2.
__device__ inline MxScales mx_scales16(const v4i& v) {
  MxScales s;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t x = (uint32_t)v[2 * h], y = (uint32_t)v[2 * h + 1];
    // (x's low half, y's low half) and the high ones; halves of the upper lane groups change sides
    const auto p = __builtin_amdgcn_permlane32_swap(__builtin_amdgcn_perm(y, x, 0x05040100u),
                                                    __builtin_amdgcn_perm(y, x, 0x07060302u), false, false);
    const auto u = __builtin_amdgcn_permlane16_swap(__builtin_amdgcn_perm(p[1], p[0], 0x06020400u),
                                                    __builtin_amdgcn_perm(p[1], p[0], 0x07030501u), false, false);
    s.w[2 * h] = u[0];
    s.w[2 * h + 1] = u[1];
  }
  return s;
}

// For fragments of 32 rows x 64 (half t of a step): lane g * 32 + r wants byte 2 t + g of
// row 32 f + r. Word 2 (s / 2) + f holds step s, half t in byte 2 (s % 2) + t.
__device__ inline MxScales mx_scales32(const v4i& v) {
  MxScales s;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t x = (uint32_t)v[2 * h], y = (uint32_t)v[2 * h + 1];
    const auto p = __builtin_amdgcn_permlane32_swap(__builtin_amdgcn_perm(y, x, 0x06040200u),
                                                    __builtin_amdgcn_perm(y, x, 0x07050301u), false, false);
    s.w[2 * h] = p[0];
    s.w[2 * h + 1] = p[1];
  }
  return s;
}

// ---------------------------------------------------------------------------
// mx_gemm_tile: 256 x 256 tiles, eight waves as 4 x 2, each 64 x 128 of the output
// in 4 x 8 blocks of 16 x 16. Operand rows go from memory into LDS as they are
// (LDS-DMA), KS k-steps a stage on a ring of STAGES. Waves 0 .. 3 and 4 .. 7
// alternate, one slot apart, between a load slot (a k-step's LDS reads, the
// copies of a later stage) and a compute slot (its MFMAs), with a workgroup
// barrier between slots.
//
// A row of a stage is 64 bytes (FP4, one k-step) or 128 (two, or FP8). Its 16-byte
// chunk c stands at slot c ^ f(row), so that the 16 rows a fragment read touches at
// once fall into different banks; the copies' source addresses do the
// permutation, within each row's 64 or 128 contiguous bytes.
// ---------------------------------------------------------------------------
template <class Q, int KS>
struct MxRow {
  static constexpr int bytes = KS * (Q::code == QO_MX_FP4 ? 64 : 128);
  static_assert(bytes == 64 || bytes == 128, "row of a stage");
  static constexpr int per_copy = 1024 / bytes;   // rows of one 64-lane copy
  // what the slot of row r's chunks is XORed with
  __device__ static inline int swizzle(int r) { return bytes == 128 ? (r >> 1) & 7 : (r >> 2) & 2; }
};

template <class QA, class OT, int KS, int STAGES>
__global__ void __launch_bounds__(512, 1)
mx_gemm_tile(MxOperand a, MxOperand b, int blocks, typename OT::T* __restrict__ out, int64_t ldc,
             const typename OT::T* __restrict__ bias, int tiles_m) {
  using T = typename OT::T;
  using RA = MxRow<QA, KS>;
  using RB = MxRow<FP4, KS>;
  constexpr int BM = 256, BN = 256, W = 8;
  constexpr bool k32 = QA::code == QO_MX_FP4;   // 32 x 32 x 64 MFMAs
  constexpr int A_BYTES = BM * RA::bytes, BYTES = A_BYTES + BN * RB::bytes;
  constexpr int TA = A_BYTES / 1024 / W, TB = (BYTES - A_BYTES) / 1024 / W, PER = TA + TB;
  constexpr bool k16 = sizeof(T) == 2;   // 16-bit outputs go through LDS, float32 from registers
  constexpr int C_PITCH = BN * 2 + 16;
  constexpr int RING = STAGES * BYTES, CTILE = k16 ? BM * C_PITCH : 0;
  static_assert(PER * (STAGES - 1) < 60, "vmcnt range");
  __shared__ __align__(16) unsigned char ring[RING > CTILE ? RING : CTILE];
  __shared__ __align__(16) float s_bias[BN];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 1, wn = wave & 1, li = lane & 15, lg = lane >> 4;
  const bool grp1 = wave >= W / 2;
  const int M = a.rows, N = b.rows;

  // Each XCD (workgroup j runs on XCD j % 8) a contiguous run of tiles, in groups
  // of 4 row tiles x every column tile.
  const int nblk = gridDim.x, xcd = blockIdx.x & 7;
  const int pid = xcd * (nblk >> 3) + min(xcd, nblk & 7) + (int)(blockIdx.x >> 3);
  constexpr int GM = 4;
  const int tiles_n = (N + BN - 1) / BN;
  const int g = pid / (GM * tiles_n), w = pid % (GM * tiles_n);
  const int gm = min(GM, tiles_m - g * GM);
  const int m0 = (g * GM + w % gm) * BM, n0 = (w / gm) * BN;

  // Copy t of this wave fills bytes 1024 (wave + 8 t) .. of its operand's part of
  // the stage. Rows past the edge repeat the last one (their sums are not
  // stored); past a row's end its last chunk is repeated (its scales are 0 there).
  const uint8_t* const a_base = a.codes + (int64_t)m0 * a.ld;
  const uint8_t* const b_base = b.codes + (int64_t)n0 * b.ld;
  const int a_end = blocks * (QA::code == QO_MX_FP4 ? 16 : 32) - 16, b_end = blocks * 16 - 16;
  uint32_t voff[PER];
  auto copy_row = [&](auto rowc, int t) -> int { return (wave + W * t) * decltype(rowc)::per_copy + lane / (decltype(rowc)::bytes / 16); };
  auto copy_chunk = [&](auto rowc, int row) -> int { return (lane & (decltype(rowc)::bytes / 16 - 1)) ^ decltype(rowc)::swizzle(row); };
  const int ca = 16 * copy_chunk(RA{}, copy_row(RA{}, 0)), cb = 16 * copy_chunk(RB{}, copy_row(RB{}, 0));   // the same for every t
#pragma unroll
  for (int t = 0; t < PER; ++t)
    voff[t] = t < TA ? (uint32_t)min(copy_row(RA{}, t), M - 1 - m0) * (uint32_t)a.ld + ca
                     : (uint32_t)min(copy_row(RB{}, t - TA), N - 1 - n0) * (uint32_t)b.ld + cb;
  const int nk = (blocks + 3) >> 2, ns = (nk + KS - 1) / KS;
  const uint32_t ring0 = lds_addr(ring) + 1024 * wave;
  auto issue = [&](int st, uint32_t buf) {
    const int oa = st * RA::bytes, ob = st * RB::bytes;
    // how far this lane's chunk lies past its row's end (0 but in a last, partial stage)
    const uint32_t over_a = max(oa + ca - a_end, 0), over_b = max(ob + cb - b_end, 0);
#pragma unroll
    for (int t = 0; t < PER; ++t) {
      const uint32_t dst = ring0 + buf + (t < TA ? 8192 * t : A_BYTES + 8192 * (t - TA));
      if (t < TA) dma16_s(voff[t] - over_a, a_base + oa, __builtin_amdgcn_readfirstlane(dst));
      else dma16_s(voff[t] - over_b, b_base + ob, __builtin_amdgcn_readfirstlane(dst));
    }
  };

  const uint8_t* sp[3];   // scale rows of this lane: A's 64, B's first and second 64
  sp[0] = a.scales + (int64_t)min(m0 + 64 * wm + lane, M - 1) * a.scales_ld;
#pragma unroll
  for (int h = 0; h < 2; ++h) sp[1 + h] = b.scales + (int64_t)min(n0 + 128 * wn + 64 * h + lane, N - 1) * b.scales_ld;
  v4i raw[3];
  MxScales sc[3];

  // This lane's place in a fragment read (k-step 0 of a stage): its row of the
  // first fragment, and its chunk.
  const int lr = k32 ? lane & 31 : li, lc = k32 ? lane >> 5 : lg;
  const uint32_t xa = (64 * wm + lr) * RA::bytes + 16 * (lc ^ RA::swizzle(lr));
  const uint32_t xb = A_BYTES + (128 * wn + lr) * RB::bytes + 16 * (lc ^ RB::swizzle(lr));
  v8i fa[4], fb[8];   // 16 rows each; 32 x 64: halves 0 and 1 of 32 rows
  auto chunk = [&](uint32_t at) -> v4i { return *reinterpret_cast<const v4i*>(ring + at); };
  auto load_regs = [&](uint32_t buf, int h) {   // k-step h of the stage: chunks 4 h .., one bit of the slot
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (k32) {
        const v4i x = chunk(buf + 32 * (i / 2) * RA::bytes + (xa ^ (64 * h + 32 * (i % 2))));
        fa[i] = v8i{x[0], x[1], x[2], x[3], 0, 0, 0, 0};
      } else {
        const v4i x = chunk(buf + 16 * i * RA::bytes + xa), y = chunk(buf + 16 * i * RA::bytes + (xa ^ 64));
        fa[i] = v8i{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const v4i x = k32 ? chunk(buf + 32 * (j / 2) * RB::bytes + (xb ^ (64 * h + 32 * (j % 2))))
                        : chunk(buf + 16 * j * RB::bytes + (xb ^ (64 * h)));
      fb[j] = v8i{x[0], x[1], x[2], x[3], 0, 0, 0, 0};
    }
  };
  auto bar = [&]() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };

  // 16 x 16: acc[i][j] (4 x 8 blocks); 32 x 32: acc32[i][j] (2 x 4)
  v4f acc[k32 ? 1 : 4][k32 ? 1 : 8];
  v16f acc32[k32 ? 2 : 1][k32 ? 4 : 1];
#pragma unroll
  for (auto& row : acc)
#pragma unroll
    for (auto& v : row) v = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (auto& row : acc32)
#pragma unroll
    for (auto& v : row)
#pragma unroll
      for (int r = 0; r < 16; ++r) v[r] = 0.f;

#pragma unroll
  for (int i = 0; i < 3; ++i) raw[i] = mx_load_scales(sp[i], 0, blocks);
  if (tid < BN) s_bias[tid] = bias ? (float)bias[min(n0 + tid, N - 1)] : 0.f;
#pragma unroll
  for (int st = 0; st < STAGES - 1 + (KS == 2); ++st)
    if (st < ns) issue(st, st * BYTES);
  if constexpr (KS == 2) gemm_wait_groups<PER, STAGES - 1>(ns - 1);
  else gemm_wait_groups<PER, STAGES - 2>(ns - 1);
  lds_barrier();
  if (grp1) bar();

  uint32_t buf = 0;   // of the current stage
  int st = 0;
  // k-step 4 q + s: load slot, compute slot
  auto phase = [&](int q, auto stepc) {
    constexpr int s = decltype(stepc)::value, h = s % KS;
    const int k = 4 * q + s;
    if constexpr (s == 0) {
      const int past = 16 * (q + 1) - blocks;   // of this quad's blocks
      if (q > 0 && past > 0) {
#pragma unroll
        for (int i = 0; i < 3; ++i) mx_shift_scales(raw[i], past);
      }
#pragma unroll
      for (int i = 0; i < 3; ++i) sc[i] = k32 ? mx_scales32(raw[i]) : mx_scales16(raw[i]);
    }
    load_regs(buf, h);
    if constexpr (h == 0) {
      // the stage before this one has been read by every wave: its slot is free
      const bool first = KS == 2 && st == 0;   // its later stages are under way already
      const int next = st + STAGES - 1;
      if (!first && next < ns) issue(next, buf >= BYTES ? buf - BYTES : buf + (STAGES - 1) * BYTES);
    }
    if constexpr (s == 0) {
      if (k + 4 < nk) {
#pragma unroll
        for (int i = 0; i < 3; ++i) raw[i] = mx_load_scales_end(sp[i], q + 1, blocks);
      }
    }
    const bool last = h == KS - 1 || k == nk - 1;   // of its stage
    if (last) gemm_wait_groups<PER, STAGES - 2>(ns - 2 - st);   // stage st + 1 has landed
    __builtin_amdgcn_s_waitcnt(0xC07F);   // lgkmcnt(0)
    bar();
    constexpr int word = 2 * (s / 2), byte = 2 * (s % 2);
    if constexpr (k32) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t sb = sc[1 + j / 2].w[word + j % 2], sa = sc[0].w[word + i];
            acc32[i][j] = t == 0 ? mx_mfma32<byte>(fb[2 * j], fa[2 * i], acc32[i][j], sb, sa)
                                 : mx_mfma32<byte + 1>(fb[2 * j + 1], fa[2 * i + 1], acc32[i][j], sb, sa);
          }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t sb = sc[1 + j / 4].w[word + j % 2], sa = sc[0].w[word + i % 2];
          const int e = (j % 4) / 2, f = i / 2;   // byte + e of sb, byte + f of sa
          if (e == 0 && f == 0) acc[i][j] = mx_mac<QA, OT, byte, byte>(fb[j], fa[i], acc[i][j], sb, sa);
          else if (e == 0) acc[i][j] = mx_mac<QA, OT, byte, byte + 1>(fb[j], fa[i], acc[i][j], sb, sa);
          else if (f == 0) acc[i][j] = mx_mac<QA, OT, byte + 1, byte>(fb[j], fa[i], acc[i][j], sb, sa);
          else acc[i][j] = mx_mac<QA, OT, byte + 1, byte + 1>(fb[j], fa[i], acc[i][j], sb, sa);
        }
    }
    bar();
    if (last) {
      ++st;
      buf = buf == (STAGES - 1) * BYTES ? 0 : buf + BYTES;
    }
  };
  for (int q = 0; 4 * q < nk; ++q) {
    phase(q, std::integral_constant<int, 0>{});
    if (4 * q + 1 < nk) phase(q, std::integral_constant<int, 1>{});
    if (4 * q + 2 < nk) phase(q, std::integral_constant<int, 2>{});
    if (4 * q + 3 < nk) phase(q, std::integral_constant<int, 3>{});
  }

  // Each lane's sums come in fours of consecutive columns: 16 x 16 blocks hold row
  // 16 i + li, columns 16 j + 4 lg ..; 32 x 32 row 32 i + lane % 32, columns 32 j + 8 e +
  // 4 (lane / 32) .., e = 0 .. 3.
  auto fours = [&](auto&& f) {
    if constexpr (k32) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const v16f& v = acc32[i][j];
            f(32 * i + lr, 32 * j + 8 * e + 4 * lc, v4f{v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]});
          }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) f(16 * i + li, 16 * j + 4 * lg, acc[i][j]);
    }
  };
  // Group 0 is one slot ahead: it stages its rows while group 1 runs its last
  // compute slot, and copies them out while group 1 stages its own.
  if constexpr (k16) {
    unsigned char* const c_wave = ring + wm * 64 * C_PITCH + wn * 256;
    fours([&](int row, int col, const v4f& x) {
      const v4f bb = *reinterpret_cast<const v4f*>(s_bias + 128 * wn + col);
      T v[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = OT::cvt(x[r] + bb[r]);
      *reinterpret_cast<v2i*>(c_wave + row * C_PITCH + 2 * col) =
          v2i{(int)(out_bits<OT>(v[0]) | out_bits<OT>(v[1]) << 16), (int)(out_bits<OT>(v[2]) | out_bits<OT>(v[3]) << 16)};
    });
    lds_barrier();
    const int half = grp1 ? BM / 2 : 0;
    copy_out_c<BM / 2, BN, 256, OT, true>(ring + half * C_PITCH, C_PITCH, out, ldc, M, N, m0 + half, n0, tid & 255);
  } else {
    fours([&](int row, int col, const v4f& x) {
      const v4f bb = *reinterpret_cast<const v4f*>(s_bias + 128 * wn + col);
      mx_store4<OT>(x + bb, out, ldc, nullptr, M, N, m0 + 64 * wm + row, n0 + 128 * wn + col);
    });
    lds_barrier();
  }
  if (!grp1) bar();
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
  constexpr int KS = QA::code == QO_MX_FP4 ? 2 : 1, STAGES = QA::code == QO_MX_FP4 ? 2 : 3;
  if (a.rows > 64 && blocks > 0 && a.ld < (1 << 23) && b.ld < (1 << 23)) {   // 32-bit offsets within a tile
    const int tm = (a.rows + 255) / 256, tn = (b.rows + 255) / 256;
    launch(mx_gemm_tile<QA, OT, KS, STAGES>, dim3((unsigned)(tm * tn)), dim3(512), 0, stream, a, b, blocks, o, ldc, bi, tm);
    return;
  }
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
  if (((M + 63) / 64) * ((N + 31) / 32) > INT32_MAX) {   // more tiles than a grid takes
    qo_set_error("%s: output too large (M=%lld N=%lld)", fn, (long long)M, (long long)N);
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
