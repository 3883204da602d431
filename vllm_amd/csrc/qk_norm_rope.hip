// RMSNorm of every query and key head of a qkv projection's result and the rotation by the token's position, in one pass:
//   y = x * rsqrt(mean of the head's squares + eps) * weight            (fp32)
//   (u, v) -> (u cos - v sin, v cos + u sin)                            over pairs of the first `rotary` values, cos and sin from the position's row
// and one rounding to the activations' type.  Pairs are (i, i + rotary / 2), or neighbours (2 i, 2 i + 1).
//
// Bound by memory: 2 bytes in and 2 out for each value, the row of cos and sin once a token.  A workgroup takes a token; a lane holds 8 consecutive values of a head
// (16 bytes) and a head takes the next power of two of lanes, so that a wavefront has 512 values of several heads, and its sum of squares is a butterfly inside them.  cos, sin
// and both weights stay in registers over the token's heads.  With pairs half the rotated width apart the partner's values come from the lane `rotary / 16` on.
// 5001 tokens of 48 heads of 128: 22.4 us of kernel, the call 23.1 = 5.3 TB/s (a copy of 1 GiB: 5.1); with q and k given 20.9 .. 21.7, pairs of either kind, over all of the head or a quarter of it.  With sums through LDS permutes and cos and sin loaded one by one
// it was 35.5: arithmetic, not memory.  32 tokens of 40 heads: 3.7 us of kernel, a chain of position, cos and sin, store; positions are requested ahead of everything, and
// nothing waits for the kernel's arguments (4.1 us where it did).
#include "vaq_common.h"

namespace vaq {

namespace {

constexpr int QK_T = 256, QK_AHEAD = 4;      // threads; rounds of heads that are requested together
constexpr int64_t QK_GRID = (int64_t)1 << 22;      // tokens of a launch, whose threads are below 2^32

struct QkArgs {
  const uint16_t* qkv;
  uint16_t *q, *k;
  const uint16_t *q_weight, *k_weight;
  const void* cache;
  const int64_t* positions;
  int64_t stride, cache_stride, cache_rows;
  int heads_q, heads_k, head_dim, rotary, lanes_log2;      // lanes: of a head
  float eps;
};
// What the first requests need arrives in registers with the launch: rows and positions, then the cache.
__device__ inline int64_t join(uint32_t lo, uint32_t hi) { return (int64_t)((uint64_t)hi << 32 | lo); }
inline KernelHead head_of_launch(const QkArgs& a) {
  const uint64_t stride = (uint64_t)a.stride, cache_stride = (uint64_t)a.cache_stride;
  return KernelHead{v8u{ptr_lo(a.qkv), ptr_hi(a.qkv), ptr_lo(a.positions), ptr_hi(a.positions), (uint32_t)stride, (uint32_t)(stride >> 32),
                        (uint32_t)a.heads_q | (uint32_t)(a.head_dim / 8) << 20 | (uint32_t)a.lanes_log2 << 28, (uint32_t)a.heads_k},
                    v4u{ptr_lo(a.cache), ptr_hi(a.cache), (uint32_t)cache_stride, (uint32_t)(cache_stride >> 32)}, v2u{}};
}

template <bool BF16>
__device__ inline void unpack(v4u r, float (&f)[8]) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = F16Traits<BF16>::to_float((uint16_t)(w[i / 2] >> (16 * (i & 1))));
}

// The sum over groups of 2^log2 lanes, in every lane of the group, in registers: pairs inside four lanes, mirrors of 8 and 16, swaps of rows of 16 and of halves.
__device__ inline float group_sum(float v, int log2) {
  auto f = [](auto u) { return __builtin_bit_cast(float, (uint32_t)u); };
  auto u = [](float x) { return __builtin_bit_cast(uint32_t, x); };
  if (log2 > 0) v += f(__builtin_amdgcn_mov_dpp((int)u(v), 0xb1, 0xf, 0xf, true));       // quad_perm 1 0 3 2
  if (log2 > 1) v += f(__builtin_amdgcn_mov_dpp((int)u(v), 0x4e, 0xf, 0xf, true));       // quad_perm 2 3 0 1
  if (log2 > 2) v += f(__builtin_amdgcn_mov_dpp((int)u(v), 0x141, 0xf, 0xf, true));      // row_half_mirror
  if (log2 > 3) v += f(__builtin_amdgcn_mov_dpp((int)u(v), 0x140, 0xf, 0xf, true));      // row_mirror
  if (log2 > 4) {
    const auto s = __builtin_amdgcn_permlane16_swap(u(v), u(v), false, false);
    v = f(s[0]) + f(s[1]);
  }
  if (log2 > 5) {
    const auto s = __builtin_amdgcn_permlane32_swap(u(v), u(v), false, false);
    v = f(s[0]) + f(s[1]);
  }
  return v;
}

// N consecutive numbers of a row of cos and sin, aligned to their type only
template <bool CACHE32, bool BF16, int N>
__device__ inline void angles(const void* row, int at, float (&to)[8], int first) {
  if constexpr (CACHE32) {
    typedef float vec __attribute__((ext_vector_type(N), aligned(4)));
    const vec v = *reinterpret_cast<const vec*>((const float*)row + at);
#pragma unroll
    for (int i = 0; i < N; ++i) to[first + i] = v[i];
  } else {
    typedef uint16_t vec __attribute__((ext_vector_type(N), aligned(2)));
    const vec v = *reinterpret_cast<const vec*>((const uint16_t*)row + at);
#pragma unroll
    for (int i = 0; i < N; ++i) to[first + i] = F16Traits<BF16>::to_float(v[i]);
  }
}

template <bool BF16, bool CACHE32, bool HALVES>
__global__ __launch_bounds__(QK_T) void qk_norm_rope_kernel(const v8u head, const v4u head2, const QkArgs p) {
  using T = F16Traits<BF16>;
  const int heads_q = (int)(head[6] & 0xfffffu), heads_k = (int)head[7], head_dim = (int)(head[6] >> 20 & 0xffu) * 8, lanes_log2 = (int)(head[6] >> 28);
  const int64_t token = blockIdx.x, position = head_ptr<int64_t>(head[2], head[3])[token];
  __builtin_amdgcn_sched_barrier(0);      // (the first request: cos and sin wait for it)
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int lanes = 1 << lanes_log2, per_wave = 64 >> lanes_log2;
  const int e = (lane & (lanes - 1)) * 8;      // first of this lane's values in a head
  const bool in_head = e < head_dim;
  const int heads = heads_q + heads_k, rounds = (heads + per_wave - 1) / per_wave;
  const uint16_t* const row = head_ptr<uint16_t>(head[0], head[1]) + token * join(head[4], head[5]);

  v4u x[QK_AHEAD];
  auto head_of = [&](int round) { return round * per_wave + (lane >> lanes_log2); };
  auto request = [&](int first) {
#pragma unroll
    for (int i = 0; i < QK_AHEAD; ++i)      // (without a branch: a lane behind the head or the heads reads the last one)
      x[i] = *reinterpret_cast<const v4u*>(row + (int64_t)min(head_of(first + i * (QK_T / 64)), heads - 1) * head_dim + min(e, head_dim - 8));
  };
  int round = wave;
  request(round);      // (ahead of the wait for the position)
  const v4u raw_q = *reinterpret_cast<const v4u*>(p.q_weight + min(e, head_dim - 8)), raw_k = *reinterpret_cast<const v4u*>(p.k_weight + min(e, head_dim - 8));
  const bool written = position >= 0 && position < p.cache_rows;      // (or not a token of a sequence: its rows stay as they are.  A branch here would have the requests wait for it)

  // cos and sin of this lane's values; values that are not rotated have cos 1 and sin 0.  The second of a pair has + sin, the first - sin.
  float c[8], s[8], wq[8], wk[8];
  const int half = p.rotary / 2;
  const void* const angle = head_ptr<char>(head2[0], head2[1]) + (written ? position : 0) * join(head2[2], head2[3]) * (CACHE32 ? 4 : 2);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    c[i] = 1.f;
    s[i] = 0.f;
  }
  if constexpr (HALVES) {
    if (half > 0) {      // (both halves are whole lanes; a lane behind them reads the first one's)
      const int at = e >= p.rotary ? 0 : e >= half ? e - half : e;
      angles<CACHE32, BF16, 8>(angle, at, c, 0);
      angles<CACHE32, BF16, 8>(angle, half + at, s, 0);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        c[i] = e < p.rotary ? c[i] : 1.f;
        s[i] = e < half ? -s[i] : e < p.rotary ? s[i] : 0.f;
      }
    }
  } else {
    float cc[8], ss[8];
    if (e + 8 <= p.rotary) {
      angles<CACHE32, BF16, 4>(angle, e / 2, cc, 0);
      angles<CACHE32, BF16, 4>(angle, half + e / 2, ss, 0);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (e + 2 * i < p.rotary) {
        if (e + 8 > p.rotary) {      // the last rotated values end inside the lane's
          angles<CACHE32, BF16, 1>(angle, e / 2 + i, cc, i);
          angles<CACHE32, BF16, 1>(angle, half + e / 2 + i, ss, i);
        }
        c[2 * i] = c[2 * i + 1] = cc[i];
        s[2 * i] = -ss[i];
        s[2 * i + 1] = ss[i];
      }
  }
  unpack<BF16>(raw_q, wq);
  unpack<BF16>(raw_k, wk);
  const int partner = !HALVES || e >= p.rotary ? lane : e < half ? lane + half / 8 : lane - half / 8;
  const float over_dim = 1.0f / (float)head_dim;

  for (; round < rounds; round += QK_AHEAD * (QK_T / 64)) {
    if (round != wave) request(round);
#pragma unroll
    for (int i = 0; i < QK_AHEAD; ++i) {
      if (round + i * (QK_T / 64) >= rounds) break;      // (the same for the whole wavefront)
      const int h = head_of(round + i * (QK_T / 64));
      float y[8], ss = 0.f;
      unpack<BF16>(x[i], y);
#pragma unroll
      for (int j = 0; j < 8; ++j) ss += y[j] * y[j];
      ss = in_head ? ss : 0.f;
      const float rms = rsqrtf(group_sum(ss, lanes_log2) * over_dim + p.eps);
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = y[j] * rms * (h < heads_q ? wq[j] : wk[j]);
      float z[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float other = HALVES ? __shfl(y[j], partner) : y[j ^ 1];
        z[j] = y[j] * c[j];
        if (e + j < p.rotary) z[j] += other * s[j];      // (a value that is not rotated stays what it is, whatever its neighbours are)
      }
      if (written && h < heads && in_head) {
        uint32_t o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = (uint32_t)T::from_float(z[2 * j]) | (uint32_t)T::from_float(z[2 * j + 1]) << 16;
        uint16_t* const to = h < heads_q ? p.q + (token * heads_q + h) * head_dim : p.k + (token * heads_k + h - heads_q) * head_dim;
        *reinterpret_cast<v4u*>(to + e) = v4u{o[0], o[1], o[2], o[3]};
      }
    }
  }
}

template <bool BF16>
void launch(const QkArgs& a, bool cache32, bool halves, int64_t tokens, hipStream_t s) {
  const dim3 grid((unsigned)tokens);
  const KernelHead h = head_of_launch(a);
  if (cache32 && halves) qk_norm_rope_kernel<BF16, true, true><<<grid, QK_T, 0, s>>>(h.a, h.b, a);
  else if (cache32) qk_norm_rope_kernel<BF16, true, false><<<grid, QK_T, 0, s>>>(h.a, h.b, a);
  else if (halves) qk_norm_rope_kernel<BF16, false, true><<<grid, QK_T, 0, s>>>(h.a, h.b, a);
  else qk_norm_rope_kernel<BF16, false, false><<<grid, QK_T, 0, s>>>(h.a, h.b, a);
}

}  // namespace

}  // namespace vaq

using namespace vaq;

extern "C" int vaq_qk_norm_rope(const void* qkv, int64_t qkv_row_stride, void* q_out, void* k_out, int64_t heads_q, int64_t heads_k, int64_t head_dim,
                                float epsilon, const void* q_weight, const void* k_weight, const void* cos_sin, int cos_sin_dtype,
                                int64_t cos_sin_row_stride, int64_t cos_sin_rows, int64_t rotary_dim, int interleaved, const int64_t* positions,
                                int dtype, int64_t tokens, void* stream) {
  VAQ_CHECK_ARG(dtype == VAQ_F16 || dtype == VAQ_BF16, "qk_norm_rope: dtype = %d", dtype);
  VAQ_CHECK_ARG(cos_sin_dtype == VAQ_F32 || cos_sin_dtype == dtype, "qk_norm_rope: cos and sin are fp32 or of the type of qkv, not %d", cos_sin_dtype);
  VAQ_CHECK_ARG(tokens >= 0 && tokens < (1ll << 31) && heads_q >= 0 && heads_k >= 0 && heads_q + heads_k > 0 && heads_q + heads_k <= 65536,
                "qk_norm_rope: tokens = %lld, heads = %lld, %lld", (long long)tokens, (long long)heads_q, (long long)heads_k);
  VAQ_CHECK_ARG(head_dim > 0 && rotary_dim >= 0 && rotary_dim <= head_dim && rotary_dim % 2 == 0, "qk_norm_rope: head_dim = %lld, rotary_dim = %lld",
                (long long)head_dim, (long long)rotary_dim);
  VAQ_CHECK_SUPPORTED(head_dim % 8 == 0 && head_dim <= 512, "qk_norm_rope: head_dim = %lld, a multiple of 8 up to 512 is built", (long long)head_dim);
  VAQ_CHECK_SUPPORTED(interleaved || rotary_dim % 16 == 0, "qk_norm_rope: rotary_dim = %lld, pairs of halves need a multiple of 16", (long long)rotary_dim);
  if (tokens == 0) return VAQ_OK;
  VAQ_CHECK_ARG(qkv && (q_out || !heads_q) && (k_out || !heads_k) && q_weight && k_weight && positions && (cos_sin || !rotary_dim), "qk_norm_rope: null pointer");
  VAQ_CHECK_ARG(tokens == 1 || qkv_row_stride >= (heads_q + heads_k) * head_dim, "qk_norm_rope: row stride %lld below the heads' values", (long long)qkv_row_stride);
  VAQ_CHECK_ARG(cos_sin_rows >= 0 && (cos_sin_rows <= 1 || cos_sin_row_stride >= rotary_dim), "qk_norm_rope: cos_sin rows %lld, stride %lld",
                (long long)cos_sin_rows, (long long)cos_sin_row_stride);
  VAQ_CHECK_ARG((((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)k_out | (uintptr_t)q_weight | (uintptr_t)k_weight) & 15) == 0 && (tokens == 1 || qkv_row_stride % 8 == 0),
                "qk_norm_rope: rows and weights must be aligned to 16 bytes");
  if (cos_sin_rows == 0) return VAQ_OK;      // every position lies outside
  QkArgs a{(const uint16_t*)qkv, (uint16_t*)q_out, (uint16_t*)k_out, (const uint16_t*)q_weight, (const uint16_t*)k_weight, cos_sin, positions, qkv_row_stride,
           cos_sin_row_stride, cos_sin_rows, (int)heads_q, (int)heads_k, (int)head_dim, (int)rotary_dim, 0, epsilon};
  while ((8 << a.lanes_log2) < head_dim) ++a.lanes_log2;
  for (int64_t left = tokens; left > 0; left -= QK_GRID) {
    const int64_t n = left < QK_GRID ? left : QK_GRID;
    if (dtype == VAQ_BF16) launch<true>(a, cos_sin_dtype == VAQ_F32, !interleaved, n, (hipStream_t)stream);
    else launch<false>(a, cos_sin_dtype == VAQ_F32, !interleaved, n, (hipStream_t)stream);
    VAQ_CHECK_LAUNCH("qk_norm_rope");
    a.qkv += n * a.stride;
    if (a.q) a.q += n * heads_q * head_dim;
    if (a.k) a.k += n * heads_k * head_dim;
    a.positions += n;
  }
  return VAQ_OK;
}
