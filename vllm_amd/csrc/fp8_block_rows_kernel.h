// FP8 product with a scale for each block of 128 (fp8_block_mm.h): few rows, bound by the weights' way from memory.
//
//  * A wavefront multiplies one step of 256 bytes of K of MB * 16 rows with J neighbouring n-tiles of 16 columns; the NW wavefronts of a workgroup take a range of
//    K each and share nothing until their sums meet in LDS: no barrier in the K loop, no hand-over between workgroups, no scratch.
//  * Both operands come by direct-to-LDS loads of 4 rows x 256 contiguous bytes into a piece of LDS of the wavefront's own, activations one step ahead, weights
//    AHEAD = one or two: two where the weights' way from memory counts, one where the LDS has room for larger results instead.
//  * A wavefront's scales for all of its K range are requested between the first step's weights and activations, into LDS of its own: a request behind another is
//    answered behind it, so that the first step's wait covers them and no step waits for scales.
//  * Rows beyond MB * 16 are a further block of rows with workgroups of their own, side by side on the same XCD, so that they find the weights in its L2.
//
// 32 rows against 4096 x 28672: 22.0 us of kernel, the call 22.9 = 5.2 TB/s, what a copy reaches.  One row against 2048 x 2048: 2.9 .. 3.4 us, a launch, one round trip to
// memory and the meeting.  Eight wavefronts to a range of K shorten the chain of layers that are narrow; four read wide ones at the same rate with half the meeting.
#pragma once
#include "fp8_block_mm.h"

namespace vaq {

constexpr int F8BR_STEP = 256;
__host__ __device__ inline int f8br_steps(int K, int nw) { return ((K + F8BR_STEP - 1) / F8BR_STEP + nw - 1) / nw; }      // of a wavefront, at most
__host__ __device__ inline int f8br_scales_a(int steps, int mb) { return (steps * 2 * mb * 16 + 63) / 64 * 64; }                  // floats; a load writes 64
__host__ __device__ inline int f8br_scales_b(int steps) { return (steps * 2 + 63) / 64 * 64; }
constexpr size_t f8br_operand_bytes(int mb, int j, int ahead) { return (size_t)(mb + ahead * j) * 16 * F8BR_STEP; }              // of a wavefront
inline size_t f8br_lds_bytes(int64_t K, int mb, int j, int ahead, int nw) {
  const int steps = f8br_steps((int)K, nw);
  const size_t run = nw * (f8br_operand_bytes(mb, j, ahead) + 4 * (size_t)(f8br_scales_a(steps, mb) + f8br_scales_b(steps)));
  const size_t sums = (size_t)nw * j * mb * 1024;
  return run > sums ? run : sums;
}

// A workgroup's range of n-tiles and block of rows: the row blocks of a range are neighbours on one XCD.
struct F8brUnit {
  uint32_t range, rows;
};
__host__ __device__ inline F8brUnit f8br_unit(uint32_t block, uint32_t ranges, uint32_t row_blocks) {      // range >= ranges: none
  const uint32_t unit = (block & 7u) * ((ranges * row_blocks + 7) / 8) + (block >> 3);
  return F8brUnit{unit / row_blocks, unit % row_blocks};
}

// TAIL: K ends inside a step; of the last one each lane asks for the chunks before K, and the rest of both operands arrives as zeros.
template <bool BF16, int MB, int J, int AHEAD, int NW, bool TAIL>
__global__ __launch_bounds__(NW * 64, NW == 4 && MB * J >= 12 ? 1 : 2) void fp8_block_rows_kernel(const v8u head, const Fp8BlockParams p) {
  using T = F16Traits<BF16>;
  constexpr int KT = F8BR_STEP, R = (J * MB + NW - 1) / NW, TB = 16 * KT, LI = TB / 1024, U = KT / F8B;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds8[];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), q = lane >> 4, r16 = lane & 15;
  // (what the first request of the weights needs arrives in registers with the launch)
  const uint8_t* const weights = head_ptr<uint8_t>(head[0], head[1]);
  const uint32_t ldb = head[2], ranges = head[6], row_blocks = head[7];
  const int K = (int)head[3], N = (int)head[4], M = (int)head[5];
  const F8brUnit unit = f8br_unit(blockIdx.x, ranges, row_blocks);
  if (unit.range >= ranges) return;
  const int n0 = (int)unit.range * J * 16, row0 = (int)unit.rows * MB * 16;
  const uint32_t rows = (uint32_t)min(MB * 16, M - row0), columns = (uint32_t)min(J * 16, N - n0);
  const int all = (K + KT - 1) / KT, per = f8br_steps(K, NW), first = w * per, last = min(first + per, all);      // this wavefront's steps

  typedef __attribute__((address_space(3))) void* lds_ptr_t;
  const int scales_a = f8br_scales_a(per, MB), scales_b = f8br_scales_b(per);
  uint8_t* const mine = lds8 + (size_t)w * (f8br_operand_bytes(MB, J, AHEAD) + 4 * (size_t)(scales_a + scales_b));
  float* const sa_lds = reinterpret_cast<float*>(mine + f8br_operand_bytes(MB, J, AHEAD));
  float* const sb_lds = sa_lds + scales_a;

  // a load fetches four whole rows of a tile of 16; their 16-byte chunk c is at place c ^ row: the 16 rows of an operand read hit all banks
  const uint32_t a_extent = (rows - 1) * p.lda + (uint32_t)K, b_extent = (columns - 1) * ldb + (uint32_t)K, rest = (uint32_t)K % KT;
  const uint8_t *const a = p.a + (int64_t)row0 * p.lda, *const b = weights + (int64_t)n0 * ldb;
  uint32_t vo_a[LI * MB], vo_w[LI];
#pragma unroll
  for (int i = 0; i < LI * MB; ++i) {
    const int r = i * 4 + q;
    vo_a[i] = (uint32_t)min(r, (int)rows - 1) * p.lda + (uint32_t)((r16 ^ (r & 15)) * 16);
  }
#pragma unroll
  for (int i = 0; i < LI; ++i) {
    const int r = i * 4 + q;
    vo_w[i] = (uint32_t)r * ldb + (uint32_t)((r16 ^ r) * 16);
  }
  // A step past the last has no extent and starts at 0 (vaq_common.h): its requests fetch nothing and keep the count of requests under way.
  auto place = [&](uint32_t vo, int r, int g) {
    if constexpr (TAIL) return g == all - 1 && (uint32_t)((r16 ^ (r & 15)) * 16) >= rest ? F8B_NOWHERE : vo;
    return vo;
  };
  auto load_act = [&](int g) {
    const __amdgpu_buffer_rsrc_t ra = f8b_rsrc(a, g < last ? a_extent : 0u);
#pragma unroll
    for (int i = 0; i < LI * MB; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (lds_ptr_t)(mine + i * 1024), 16, (int)place(vo_a[i], i * 4 + q, g), g < last ? g * KT : 0, 0, 0);
  };
  auto load_w = [&](int s, int g) {
    const __amdgpu_buffer_rsrc_t rb = f8b_rsrc(b, g < last ? b_extent : 0u);
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int so = g < last ? (int)(min((uint32_t)(j * 16), columns - 16) * ldb + (uint32_t)(g * KT)) : 0;
#pragma unroll
      for (int i = 0; i < LI; ++i)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, (lds_ptr_t)(mine + (MB + s * J + j) * TB + i * 1024), 16, (int)place(vo_w[i], i * 4 + q, g), so, 0, 2);
    }
  };
  // scales: [block of K][row], then [block of K]; blocks past K and past this wavefront's arrive as zeros
  const int blocks = (K + F8B - 1) / F8B, kb0 = first * U, kb_n = max(0, min(last * U, blocks) - kb0);
  auto load_scales = [&] {
    const __amdgpu_buffer_rsrc_t rsa = f8b_rsrc(p.sa + (int64_t)row0 * p.sa_row, 0x7ffffffcu), rsb = f8b_rsrc(p.sb + (int64_t)(n0 / F8B) * p.sb_n, 0x7ffffffcu);
    for (int i = 0; i < scales_a; i += 64) {
      const int kb = (i + lane) / (MB * 16), row = (i + lane) % (MB * 16);
      const uint32_t at = (uint32_t)min(row, (int)rows - 1) * (uint32_t)p.sa_row * 4u + (uint32_t)(kb0 + kb) * p.sa_block * 4u;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsa, (lds_ptr_t)(sa_lds + i), 4, (int)(kb < kb_n ? at : F8B_NOWHERE), 0, 0, 0);
    }
    for (int i = 0; i < scales_b; i += 64)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsb, (lds_ptr_t)(sb_lds + i), 4, (int)(i + lane < kb_n ? (uint32_t)(kb0 + i + lane) * p.sb_block * 4u : F8B_NOWHERE), 0, 0, 0);
  };
  v4f acc[J][MB];
#pragma unroll
  for (int j = 0; j < J; ++j)
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) acc[j][mb] = v4f{0.f, 0.f, 0.f, 0.f};
  auto operand = [&](const uint8_t* at, int u) {
    const v4i lo = *reinterpret_cast<const v4i*>(at + r16 * KT + ((u * 8 + q) ^ r16) * 16);
    const v4i hi = *reinterpret_cast<const v4i*>(at + r16 * KT + ((u * 8 + 4 + q) ^ r16) * 16);
    return v8i{lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
  };
  auto tile = [&](int s, int g, bool refill_act, bool refill_w) {
    v8i act[U][MB], wop[U][J];
    float scale[U][MB];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int kb = (g - first) * U + u;
      const float sb = sb_lds[kb];
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) {
        act[u][mb] = operand(mine + mb * TB, u);
        scale[u][mb] = sa_lds[(kb * MB + mb) * 16 + r16] * sb;
      }
#pragma unroll
      for (int j = 0; j < J; ++j) wop[u][j] = operand(mine + (MB + s * J + j) * TB, u);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");      // this step's are in registers
    __builtin_amdgcn_sched_barrier(0);
    if (refill_act) load_act(g + 1);
    __builtin_amdgcn_sched_barrier(0);
    if (refill_w) load_w(s, g + AHEAD);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      v4f part[J][MB];
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) part[j][mb] = mfma_fp8_block(wop[u][j], act[u][mb]);
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[j][mb][e] = __builtin_fmaf(scale[u][mb], part[j][mb][e], acc[j][mb][e]);
    }
  };

  int g = first;
  load_w(0, g);
  __builtin_amdgcn_sched_barrier(0);
  load_scales();
  __builtin_amdgcn_sched_barrier(0);
  load_act(g);
  __builtin_amdgcn_sched_barrier(0);
  if constexpr (AHEAD == 1) {
    // W(0) A(0) | A(1) W(1) | A(2) W(2) | ..., `|` = a step: it starts when everything has been answered
#pragma unroll 1
    for (; g + 1 < last; ++g) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      tile(0, g, true, true);
    }
    if (g < last) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      tile(0, g, false, false);
    }
  } else {
    // W(0) A(0) W(1) | A(1) W(2) | A(2) W(3) | ..., it starts when all but the weights requested behind its activations have been answered
    auto wait = [&] { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(J * LI) : "memory"); };
    load_w(1, g + 1);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll 1
    for (; g + 2 < last; g += 2) {
      wait();
      tile(0, g, true, true);
      wait();
      tile(1, g + 1, true, true);
    }
    if (g + 1 < last) {
      wait();
      tile(0, g, true, false);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      tile(1, g + 1, false, false);
    } else if (g < last) {
      wait();
      tile(0, g, false, false);
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");      // (what is requested past the end writes zeros into LDS)

  v4f* const red = reinterpret_cast<v4f*>(lds8);      // [NW][J * MB][64], on top of the operands
  __syncthreads();
#pragma unroll
  for (int j = 0; j < J; ++j)
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) red[(w * (J * MB) + j * MB + mb) * 64 + lane] = acc[j][mb];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int u = w + i * NW, j = u / MB, mb = u - j * MB, n = n0 + j * 16 + q * 4, m = row0 + mb * 16 + r16;
    if (u >= J * MB || n >= N || m >= M) continue;
    v4f val = red[u * 64 + lane];
#pragma unroll
    for (int ww = 1; ww < NW; ++ww) val += red[(ww * (J * MB) + u) * 64 + lane];
    uint16_t o[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = T::from_float(val[e] + (p.bias ? T::to_float(p.bias[n + e]) : 0.f));
    *reinterpret_cast<v2u*>(p.out + (int64_t)m * p.ldc + n) = v2u{(uint32_t)o[0] | (uint32_t)o[1] << 16, (uint32_t)o[2] | (uint32_t)o[3] << 16};
  }
}

constexpr bool f8br_built(int mb, int j, int ahead, int nw) {
  return mb >= 1 && mb <= 4 && (j == 1 || j == 2 || (j == 4 && ahead == 1)) && (ahead == 1 || ahead == 2) && (nw == 4 || (nw == 8 && j == 1)) &&
         nw * f8br_operand_bytes(mb, j, ahead) < 160 * 1024;
}

}  // namespace vaq
