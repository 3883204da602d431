// FP8 (OCP e4m3fn) quantisation in groups of 128 consecutive values of a row, one fp32 scale a group: alone, behind silu(gate) * up, and
// behind RMSNorm (+ residual).  The activations' side of fp8_block_mm.hip.
//
//   y  = x                                                       (group_quant_kernel)
//      = g / (1 + exp(-g)) * u                                   (the same, SILU)
//      = (x [+ residual]) * rsqrt(mean of their squares + eps) * weight      (rms_norm_group_quant_kernel)
//   s  = max(max|y| over the group, 1e-10) / 448,   code = e4m3(y / s)
// y and the statistics are fp32 throughout: a y rounded to 16 bits ahead of the maximum would put 2^-9 of error into every scale, and with
// it into every product with the group.  What is rounded: the code, and the new residual to the type of the old one.  Behind silu and norm the code rounds y times 1 / s, which is off
// from y / s by 2^-23 and only moves codes of values that near to a tie; y itself carries a few such roundings there.
// The maximum is taken over the magnitudes' bit patterns, which order like the magnitudes with NaN above infinity: a group with a NaN has
// scale NaN and codes NaN, one with an infinity scale infinity, codes 0 for what is finite and NaN for the infinities, as x / s says.
// No clamp: |y / s| is at most 448 (1 + 2^-22), which rounds to 448.
//
// A lane holds 8 consecutive values (16 bytes of a 16-bit row), 16 lanes a group: the maximum is four rotations inside a row of 16 lanes, without
// LDS.  The scales are written where the caller's strides say; the package lays a group's scales of all tokens next to each other, which is
// how the product reads them.
//
// All three are bound by memory with many rows; each value is read once and written once.  Calls over the same tensors (a copy of 1 GiB moves 5.1 TB/s here):
//   4096 x 14336 bf16 33.0 us = 5.4 TB/s (28.7 of them kernel), silu of 2048 x 2 x 14336 26.9 us = 5.5 TB/s, norm of 3333 x 5120 with a residual 23.0 us = 5.2 TB/s.
//   4096 x 14336 fp32 44.9 us (part of it from the last-level cache); norm of 3333 x 5120 without a residual 15.3 us = 3.4 TB/s.
// A token of 4096 takes 2.4 us of kernel, of which one round trip to memory is most; the call, 4.7 us, is then bound by the host.
// Rows whose length or offset is no multiple of 8 are read value by value; above 4096 values the norm keeps them in 1024 threads of 64 values, of which 72 .. 84 registers spill with a
// residual: 64 x 5125 13.8 us, 21.0 with a residual.
#include "vaq_common.h"

#include <string.h>

namespace vaq {

namespace {

constexpr int GROUP = 128;
constexpr float GQ_MAX = 448.0f, GQ_LEAST = 1e-10f;
constexpr int GQ_T = 256;            // threads of a workgroup: 4 wavefronts
constexpr int GQ_ROWS = 4;           // rows of a wavefront, all requested ahead of the first use

// DT is VAQ_F16, VAQ_BF16 or VAQ_F32
template <int DT>
struct Raw8 {
  static constexpr int SIZE = DT == VAQ_F32 ? 4 : 2;
  v4u w[SIZE / 2];
};

// Values e .. e + 7 of a row, `left` of which are in it.  VEC: rows are 16-byte aligned multiples of 8, so that either all are or none.
template <int DT, bool VEC>
__device__ inline Raw8<DT> load8(const void* row, int64_t e, int left) {
  Raw8<DT> r = {};
  if constexpr (VEC) {
    if (left > 0) {
      const v4u* p = reinterpret_cast<const v4u*>((const char*)row + e * Raw8<DT>::SIZE);
#pragma unroll
      for (int i = 0; i < Raw8<DT>::SIZE / 2; ++i) r.w[i] = p[i];
    }
  } else {
    uint32_t* w = reinterpret_cast<uint32_t*>(r.w);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) {
        if constexpr (DT == VAQ_F32) w[i] = reinterpret_cast<const uint32_t*>(row)[e + i];
        else w[i / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(row)[e + i] << (16 * (i & 1));
      }
  }
  return r;
}

template <int DT>
__device__ inline void unpack8(const Raw8<DT>& r, float (&f)[8]) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(r.w);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (DT == VAQ_F32) f[i] = __builtin_bit_cast(float, w[i]);
    else f[i] = F16Traits<DT == VAQ_BF16>::to_float((uint16_t)(w[i / 2] >> (16 * (i & 1))));
  }
}

__device__ inline uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }
__device__ inline uint32_t magnitude(const float (&f)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = umax(m, __builtin_bit_cast(uint32_t, f[i]) & 0x7fffffffu);
  return m;
}
// the largest of 16 lanes (a row of the wavefront), in all of them
__device__ inline uint32_t row16_umax(uint32_t v) {
  v = umax(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x128, 0xf, 0xf, true));      // row_ror:8
  v = umax(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x124, 0xf, 0xf, true));
  v = umax(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x122, 0xf, 0xf, true));
  return umax(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x121, 0xf, 0xf, true));
}
__device__ inline float scale_of(uint32_t magnitude_bits) {
  return __builtin_bit_cast(float, umax(magnitude_bits, __builtin_bit_cast(uint32_t, GQ_LEAST))) / GQ_MAX;
}

// eight values -> eight codes, stored at `to`; `left` of them are in the row
template <bool VEC, typename F>
__device__ inline void store_codes(uint8_t* to, int left, const float (&y)[8], F&& over_scale) {
  uint32_t o[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(over_scale(y[4 * h]), over_scale(y[4 * h + 1]), 0, false) & 0xffffu;
    const uint32_t hi = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(over_scale(y[4 * h + 2]), over_scale(y[4 * h + 3]), 0, false) & 0xffffu;
    o[h] = lo | hi << 16;
  }
  if constexpr (VEC) {
    if (left > 0) *reinterpret_cast<v2u*>(to) = v2u{o[0], o[1]};
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) to[i] = (uint8_t)(o[i / 4] >> (8 * (i & 3)));
  }
}

// Bound by memory: every value is read once.  A workgroup takes 16 rows x 512 columns; 16 rows' scales of a group are 64 contiguous bytes in the
// package's layout.  Quotients: of 16-bit values the correctly rounded one (div16_exact; the same codes as IEEE division), of fp32 values the
// IEEE division, of silu(g) u the product with 1 / s.
// (What the first requests need arrives in registers with the launch, as one vector: the host's cost of a launch grows with the number of arguments.)
struct QuantTo {
  uint8_t* out;
  int64_t out_stride;
  float* scales;
  int64_t scale_row, scale_group;
};
__device__ inline int64_t join(uint32_t lo, uint32_t hi) { return (int64_t)((uint64_t)hi << 32 | lo); }
template <int DT, bool VEC, bool SILU>
__global__ __launch_bounds__(GQ_T) void group_quant_kernel(const v8u head, const QuantTo to) {
  constexpr int SIZE = Raw8<DT>::SIZE;
  const char* const in = head_ptr<char>(head[0], head[1]);
  const int64_t in_stride = join(head[2], head[3]), rows = join(head[4], head[5]);
  const int hidden = (int)head[6];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int e = ((int)blockIdx.x * 64 + lane) * 8, left = hidden - e;
  const int64_t step = (int64_t)gridDim.y * (GQ_T / 64 * GQ_ROWS);
  for (int64_t r0 = ((int64_t)blockIdx.y * (GQ_T / 64) + wave) * GQ_ROWS; r0 < rows; r0 += step) {
    Raw8<DT> a[GQ_ROWS], b[SILU ? GQ_ROWS : 1];
#pragma unroll
    for (int i = 0; i < GQ_ROWS; ++i) {
      const char* row = in + (r0 + i) * in_stride * SIZE;
      const int n = r0 + i < rows ? left : 0;
      a[i] = load8<DT, VEC>(row, e, n);
      if constexpr (SILU) b[i] = load8<DT, VEC>(row, (int64_t)hidden + e, n);
    }
    float mine = 0.f;
#pragma unroll
    for (int i = 0; i < GQ_ROWS; ++i) {
      if (r0 + i >= rows) break;
      float y[8];
      unpack8<DT>(a[i], y);
      if constexpr (SILU) {
        // (hardware exponential and reciprocal, one unit in the last place each, and |g| 6e-8 from the exponential's argument)
        float u[8];
        unpack8<DT>(b[i], u);
#pragma unroll
        for (int k = 0; k < 8; ++k) y[k] = y[k] * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * y[k])) * u[k];
      }
      const float s = scale_of(row16_umax(magnitude(y))), r = 1.0f / s;
      uint8_t* const codes = to.out + (r0 + i) * to.out_stride + e;
      if constexpr (SILU) store_codes<VEC>(codes, left, y, [&](float v) { return v * r; });
      else if constexpr (DT == VAQ_F32) store_codes<VEC>(codes, left, y, [&](float v) { return v / s; });
      else if (s < __builtin_inff()) store_codes<VEC>(codes, left, y, [&](float v) { return div16_exact(v, s, r); });
      else store_codes<VEC>(codes, left, y, [&](float v) { return v / s; });
      mine = (lane & 15) == i ? s : mine;
    }
    const int64_t row = r0 + (lane & 15), g = (int64_t)blockIdx.x * 4 + (lane >> 4);
    if ((lane & 15) < GQ_ROWS && row < rows && g * GROUP < hidden) to.scales[row * to.scale_row + g * to.scale_group] = mine;
  }
}

// One row a workgroup, which stays in registers from the sum of squares to the codes.  Bound by memory with many rows; with few by one round trip
// for row, residual and weight (all requested together) and one meeting of the wavefronts.
struct NormTo {
  uint8_t* out;
  float* scales;
  int64_t scale_row, scale_group;
  uint16_t* residual_out;
};
template <bool BF16, bool VEC, bool RES, int TPB, int NV>
__global__ __launch_bounds__(TPB) void rms_norm_group_quant_kernel(const v8u head, const v2u head2, const NormTo to) {
  const uint16_t* const input = head_ptr<uint16_t>(head[0], head[1]);
  const uint16_t* const residual = head_ptr<uint16_t>(head[2], head[3]);
  const uint16_t* const weight = head_ptr<uint16_t>(head[4], head[5]);
  const int64_t in_stride = join(head[6], head[7]);
  const int hidden = (int)head2[0];
  const float eps = __builtin_bit_cast(float, (uint32_t)head2[1]);
  constexpr int DT = BF16 ? VAQ_BF16 : VAQ_F16;
  using T = F16Traits<BF16>;
  __shared__ float smem[TPB / 64];
  const int64_t row = blockIdx.x;
  const uint16_t* const x_row = input + row * in_stride;
  Raw8<DT> xr[NV], rr[RES ? NV : 1], wr[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int e = ((int)threadIdx.x + v * TPB) * 8;
    xr[v] = load8<DT, VEC>(x_row, e, hidden - e);
    if constexpr (RES) rr[v] = load8<DT, VEC>(residual + row * hidden, e, hidden - e);
  }
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int e = ((int)threadIdx.x + v * TPB) * 8;
    wr[v] = load8<DT, VEC>(weight, e, hidden - e);
  }
  float x[NV][8], ss = 0.f;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    unpack8<DT>(xr[v], x[v]);
    if constexpr (RES) {
      const int e = ((int)threadIdx.x + v * TPB) * 8;
      float r[8];
      unpack8<DT>(rr[v], r);
      uint16_t z[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[v][i] += r[i];
        z[i] = T::from_float(x[v][i]);
      }
      uint16_t* const sum = to.residual_out + row * hidden + e;
      if constexpr (VEC) {
        if (e < hidden)
          *reinterpret_cast<v4u*>(sum) = v4u{(uint32_t)z[0] | (uint32_t)z[1] << 16, (uint32_t)z[2] | (uint32_t)z[3] << 16,
                                            (uint32_t)z[4] | (uint32_t)z[5] << 16, (uint32_t)z[6] | (uint32_t)z[7] << 16};
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (e + i < hidden) sum[i] = z[i];
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) ss += x[v][i] * x[v][i];
  }
  ss = block_sum<TPB>(ss, smem);
  const float rms = rsqrtf(ss / (float)hidden + eps);
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int c = (int)threadIdx.x + v * TPB, e = c * 8;
    float w[8], y[8];
    unpack8<DT>(wr[v], w);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = e + i < hidden ? x[v][i] * rms * w[i] : 0.f;      // (0 * infinity behind the row)
    const float s = scale_of(row16_umax(magnitude(y))), r = 1.0f / s;
    store_codes<VEC>(to.out + row * hidden + e, hidden - e, y, [&](float f) { return f * r; });
    if ((c & 15) == 0 && e < hidden) to.scales[row * to.scale_row + (int64_t)(c >> 4) * to.scale_group] = s;
  }
}

template <int DT, bool SILU>
void launch_quant(bool vec, const void* in, int64_t in_stride, int64_t rows, int64_t hidden, uint8_t* out, int64_t out_stride, float* scales,
                  int64_t scale_row, int64_t scale_group, hipStream_t s) {
  const int64_t row_blocks = (rows + GQ_T / 64 * GQ_ROWS - 1) / (GQ_T / 64 * GQ_ROWS);
  const dim3 grid((unsigned)((hidden + 511) / 512), (unsigned)(row_blocks < 65535 ? row_blocks : 65535));
  const uint64_t in_s = (uint64_t)in_stride, n = (uint64_t)rows;
  const v8u head{ptr_lo(in), ptr_hi(in), (uint32_t)in_s, (uint32_t)(in_s >> 32), (uint32_t)n, (uint32_t)(n >> 32), (uint32_t)hidden, 0u};
  const QuantTo to{out, out_stride, scales, scale_row, scale_group};
  if (vec) group_quant_kernel<DT, true, SILU><<<grid, GQ_T, 0, s>>>(head, to);
  else group_quant_kernel<DT, false, SILU><<<grid, GQ_T, 0, s>>>(head, to);
}

struct NormArgs {
  const uint16_t *input, *residual, *weight;
  int64_t in_stride, tokens, hidden;
  float eps;
  uint8_t* out;
  float* scales;
  int64_t scale_row, scale_group;
  uint16_t* residual_out;
};
template <bool BF16, bool VEC, int TPB, int NV>
void launch_norm(const NormArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)a.tokens);
  const uint64_t in_s = (uint64_t)a.in_stride;
  const v8u head{ptr_lo(a.input), ptr_hi(a.input), ptr_lo(a.residual), ptr_hi(a.residual), ptr_lo(a.weight), ptr_hi(a.weight), (uint32_t)in_s, (uint32_t)(in_s >> 32)};
  uint32_t eps_bits;
  memcpy(&eps_bits, &a.eps, sizeof(eps_bits));
  const v2u head2{(uint32_t)a.hidden, eps_bits};
  const NormTo to{a.out, a.scales, a.scale_row, a.scale_group, a.residual_out};
  if (a.residual) rms_norm_group_quant_kernel<BF16, VEC, true, TPB, NV><<<grid, TPB, 0, s>>>(head, head2, to);
  else rms_norm_group_quant_kernel<BF16, VEC, false, TPB, NV><<<grid, TPB, 0, s>>>(head, head2, to);
}
constexpr int64_t NORM_MAX = 1024 * 8 * 8;      // values of a row that a workgroup holds
template <bool BF16>
void launch_norm_type(bool vec, const NormArgs& a, hipStream_t s) {
  if (!vec) {
    if (a.hidden <= 4096) launch_norm<BF16, false, 256, 2>(a, s);
    else launch_norm<BF16, false, 1024, 8>(a, s);
  } else if (a.hidden <= 2048) launch_norm<BF16, true, 256, 1>(a, s);
  else if (a.hidden <= 4096) launch_norm<BF16, true, 256, 2>(a, s);
  else if (a.hidden <= 8192) launch_norm<BF16, true, 512, 2>(a, s);
  else if (a.hidden <= 16384) launch_norm<BF16, true, 512, 4>(a, s);
  else launch_norm<BF16, true, 1024, 8>(a, s);
}

bool aligned(const void* p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) == 0; }
constexpr int64_t MOST = (int64_t)1 << 30;      // values of a row, tokens
constexpr int64_t NORM_GRID = (int64_t)1 << 21;      // rows of a launch, whose threads are below 2^32

int quant_common(const char* who, const void* in, int in_dtype, int64_t in_stride, int64_t row_values, uint8_t* out, int64_t out_stride, float* scales,
                 int64_t rows, int64_t hidden) {
  VAQ_CHECK_ARG(rows >= 0 && hidden >= 0 && rows <= MOST && hidden <= MOST, "%s: rows = %lld, hidden = %lld", who, (long long)rows, (long long)hidden);
  if (rows == 0 || hidden == 0) return VAQ_OK;
  VAQ_CHECK_ARG(in && out && scales, "%s: null pointer", who);
  VAQ_CHECK_ARG(rows == 1 || (in_stride >= row_values && out_stride >= hidden), "%s: row strides %lld, %lld below the rows' lengths", who,
                (long long)in_stride, (long long)out_stride);
  VAQ_CHECK_ARG(aligned(in, in_dtype == VAQ_F32 ? 4 : 2) && aligned(scales, 4), "%s: pointers are not aligned to their types", who);
  return VAQ_OK;
}

}  // namespace

}  // namespace vaq

using namespace vaq;

extern "C" int vaq_fp8_group_quant(const void* in, int in_dtype, int64_t in_row_stride, uint8_t* out, int64_t out_row_stride, float* scales,
                                   int64_t scale_row_stride, int64_t scale_group_stride, int64_t rows, int64_t hidden, void* stream) {
  VAQ_CHECK_ARG(in_dtype == VAQ_F16 || in_dtype == VAQ_BF16 || in_dtype == VAQ_F32, "fp8_group_quant: in_dtype = %d", in_dtype);
  if (const int rc = quant_common("fp8_group_quant", in, in_dtype, in_row_stride, hidden, out, out_row_stride, scales, rows, hidden); rc != VAQ_OK) return rc;
  if (rows == 0 || hidden == 0) return VAQ_OK;
  const int size = in_dtype == VAQ_F32 ? 4 : 2;
  const bool vec = hidden % 8 == 0 && aligned(in, 16) && aligned(out, 8) && (rows == 1 || (in_row_stride * size % 16 == 0 && out_row_stride % 8 == 0));
  hipStream_t s = (hipStream_t)stream;
  if (in_dtype == VAQ_F16) launch_quant<VAQ_F16, false>(vec, in, in_row_stride, rows, hidden, out, out_row_stride, scales, scale_row_stride, scale_group_stride, s);
  else if (in_dtype == VAQ_BF16) launch_quant<VAQ_BF16, false>(vec, in, in_row_stride, rows, hidden, out, out_row_stride, scales, scale_row_stride, scale_group_stride, s);
  else launch_quant<VAQ_F32, false>(vec, in, in_row_stride, rows, hidden, out, out_row_stride, scales, scale_row_stride, scale_group_stride, s);
  VAQ_CHECK_LAUNCH("fp8_group_quant");
  return VAQ_OK;
}

extern "C" int vaq_silu_and_mul_fp8_group_quant(const void* in, int dtype, int64_t in_row_stride, uint8_t* out, int64_t out_row_stride, float* scales,
                                                int64_t scale_row_stride, int64_t scale_group_stride, int64_t rows, int64_t d, void* stream) {
  VAQ_CHECK_ARG(dtype == VAQ_F16 || dtype == VAQ_BF16, "silu_and_mul_fp8_group_quant: dtype = %d", dtype);
  if (const int rc = quant_common("silu_and_mul_fp8_group_quant", in, dtype, in_row_stride, 2 * d, out, out_row_stride, scales, rows, d); rc != VAQ_OK) return rc;
  if (rows == 0 || d == 0) return VAQ_OK;
  const bool vec = d % 8 == 0 && aligned(in, 16) && aligned(out, 8) && (rows == 1 || (in_row_stride % 8 == 0 && out_row_stride % 8 == 0));
  hipStream_t s = (hipStream_t)stream;
  if (dtype == VAQ_F16) launch_quant<VAQ_F16, true>(vec, in, in_row_stride, rows, d, out, out_row_stride, scales, scale_row_stride, scale_group_stride, s);
  else launch_quant<VAQ_BF16, true>(vec, in, in_row_stride, rows, d, out, out_row_stride, scales, scale_row_stride, scale_group_stride, s);
  VAQ_CHECK_LAUNCH("silu_and_mul_fp8_group_quant");
  return VAQ_OK;
}

extern "C" int vaq_rms_norm_fp8_group_quant(uint8_t* out, float* scales, int64_t scale_row_stride, int64_t scale_group_stride, const void* input,
                                            int64_t in_row_stride, const void* weight, float epsilon, const void* residual, void* residual_out,
                                            int dtype, int64_t tokens, int64_t hidden, void* stream) {
  VAQ_CHECK_ARG(dtype == VAQ_F16 || dtype == VAQ_BF16, "rms_norm_fp8_group_quant: dtype = %d", dtype);
  if (const int rc = quant_common("rms_norm_fp8_group_quant", input, dtype, in_row_stride, hidden, out, hidden, scales, tokens, hidden); rc != VAQ_OK) return rc;
  if (tokens == 0 || hidden == 0) return VAQ_OK;
  VAQ_CHECK_SUPPORTED(hidden <= NORM_MAX, "rms_norm_fp8_group_quant: hidden = %lld, at most %lld are built", (long long)hidden, (long long)NORM_MAX);
  VAQ_CHECK_ARG(weight && (residual == nullptr) == (residual_out == nullptr), "rms_norm_fp8_group_quant: null pointer");
  VAQ_CHECK_ARG(aligned(weight, 2) && aligned(residual, 2) && aligned(residual_out, 2), "rms_norm_fp8_group_quant: pointers are not aligned to their types");
  const bool vec = hidden % 8 == 0 && aligned(input, 16) && aligned(weight, 16) && aligned(residual, 16) && aligned(residual_out, 16) && aligned(out, 8) &&
                   (tokens == 1 || in_row_stride % 8 == 0);
  for (int64_t t = 0; t < tokens; t += NORM_GRID) {
    const NormArgs a{(const uint16_t*)input + t * in_row_stride, residual ? (const uint16_t*)residual + t * hidden : nullptr, (const uint16_t*)weight, in_row_stride,
                     tokens - t < NORM_GRID ? tokens - t : NORM_GRID, hidden, epsilon, out + t * hidden, scales + t * scale_row_stride, scale_row_stride,
                     scale_group_stride, residual ? (uint16_t*)residual_out + t * hidden : nullptr};
    if (dtype == VAQ_BF16) launch_norm_type<true>(vec, a, (hipStream_t)stream);
    else launch_norm_type<false>(vec, a, (hipStream_t)stream);
    VAQ_CHECK_LAUNCH("rms_norm_fp8_group_quant");
  }
  return VAQ_OK;
}
