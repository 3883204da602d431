// FP8 product with a scale for each block of 128 (fp8_block_mm.h): tiles.
//
//  * BM x BN results a workgroup; a step is one block of K.  Both operands come by direct-to-LDS loads of whole 128-byte lines (8 rows an instruction) into a
//    ring of NST stages; chunk c of a row lies at place c ^ (row / 2 & 7) of its 128 bytes, so that the 16 lanes that are served together hit all banks.
//  * A wavefront holds its TM rows' scales of the step in registers, one load for 64 rows, multiplied by the weight's scale and spread over the four groups of
//    16 lanes by swaps: no LDS for scales, and no place in the ring.
//  * The products of 16 rows are issued ahead of the multiply-adds of the 16 rows before them, which then find their results ready: four multiply-adds go beside an
//    instruction that keeps the matrix core for 32 cycles.
#pragma once
#include "fp8_block_mm.h"

namespace vaq {

// What a workgroup computes: one contiguous range of tile positions an XCD (its L2 then holds what neighbours share), positions in bands of 4 tile rows.
struct F8bTile {
  int m0, n0;
};
__host__ __device__ inline uint32_t f8b_position(uint32_t block, uint32_t total) {      // total or more: none
  return (block & 7u) * ((total + 7) / 8) + (block >> 3);
}
__host__ __device__ inline F8bTile f8b_tile(uint32_t position, uint32_t tiles_m, uint32_t tiles_n, int BM, int BN) {
  const uint32_t band = position / (4 * tiles_n), in_band = position - band * 4 * tiles_n;
  const uint32_t height = tiles_m - band * 4 < 4 ? tiles_m - band * 4 : 4, column = in_band / height;
  return F8bTile{(int)((band * 4 + in_band - column * height) * BM), (int)(column * BN)};
}

template <bool BF16, int BM, int BN, int WAVES_M, int WAVES_N, int NST, bool TAIL>
__global__ __launch_bounds__(WAVES_M * WAVES_N * 64) void fp8_block_tile_kernel(const Fp8BlockParams p, const uint32_t tiles_m, const uint32_t tiles_n) {
  using T = F16Traits<BF16>;
  constexpr int NW = WAVES_M * WAVES_N, TM = BM / WAVES_M, TN = BN / WAVES_N, MT = TM / 16, NT = TN / 16;
  constexpr int A_LD = BM / (8 * NW), B_LD = BN / (8 * NW), STAGE = (BM + BN) * 128;
  constexpr int SL = TM <= 64 ? 1 : TM / 64;      // loads of row scales
  static_assert(A_LD >= 1 && B_LD >= 1 && (TM == 32 || TM % 64 == 0) && TN <= F8B && F8B % TN == 0, "tile shape");
  extern __shared__ __attribute__((aligned(16))) uint8_t lds8[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WAVES_N, wn = wave % WAVES_N, q = lane >> 4, r16 = lane & 15;
  const uint32_t position = f8b_position(blockIdx.x, tiles_m * tiles_n);
  if (position >= tiles_m * tiles_n) return;
  const F8bTile tile = f8b_tile(position, tiles_m, tiles_n, BM, BN);
  const int m0 = tile.m0, n0 = tile.n0;

  // operands: descriptors of this tile's rows, so that no offset passes 32 bits whatever the whole operand is
  const uint32_t rows_a = (uint32_t)min(BM, p.M - m0), rows_b = (uint32_t)min(BN, p.N - n0), K = (uint32_t)p.K;
  const __amdgpu_buffer_rsrc_t ra = f8b_rsrc(p.a + (int64_t)m0 * p.lda, (rows_a - 1) * p.lda + K);
  const __amdgpu_buffer_rsrc_t rb = f8b_rsrc(p.b + (int64_t)n0 * p.ldb, (rows_b - 1) * p.ldb + K);
  // a load: lane l writes place l & 7 of row r0 + l / 8, r0 = 8 times the instruction's number; odd numbers differ by 4 in the place's XOR.
  // (A row past the last counts as the last, see vaq_common.h: the first eight lanes ask for that one over again, the others for nothing.)
  const uint32_t lrow = (uint32_t)lane >> 3, lbyte = (uint32_t)(((lane & 7) ^ (lane >> 4)) * 16);
  const uint32_t va = lrow * p.lda, vb = lrow * p.ldb;
  typedef __attribute__((address_space(3))) void* lds_ptr_t;
  auto request = [&](uint32_t k, uint8_t* at) {
    auto offset = [&](uint32_t row, uint32_t byte) { return (int)(!TAIL || k + byte < K ? row + byte : F8B_NOWHERE); };
    const int a0 = offset(va, lbyte), a1 = offset(va, lbyte ^ 64u), b0 = offset(vb, lbyte), b1 = offset(vb, lbyte ^ 64u);
#pragma unroll
    for (int i = 0; i < A_LD; ++i) {
      const uint32_t r0 = (uint32_t)(wave * A_LD + i) * 8;
      const bool odd = A_LD % 2 == 0 ? i & 1 : (r0 & 8) != 0;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (lds_ptr_t)(at + r0 * 128), 16, odd ? a1 : a0, (int)(min(r0, rows_a - 1) * p.lda + k), 0, 0);
    }
#pragma unroll
    for (int i = 0; i < B_LD; ++i) {
      const uint32_t r0 = (uint32_t)(wave * B_LD + i) * 8;
      const bool odd = B_LD % 2 == 0 ? i & 1 : (r0 & 8) != 0;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, (lds_ptr_t)(at + BM * 128 + r0 * 128), 16, odd ? b1 : b0, (int)(min(r0, rows_b - 1) * p.ldb + k), 0, 0);
    }
  };
  // scales of a step: rows (lane: row i * 64 + lane of the wavefront's; 32 rows twice) and the columns' one
  const __amdgpu_buffer_rsrc_t rsa = f8b_rsrc(p.sa + (int64_t)m0 * p.sa_row, 0x7ffffffcu);
  const __amdgpu_buffer_rsrc_t rsb = f8b_rsrc(p.sb + (int64_t)((n0 + wn * TN < p.N ? n0 + wn * TN : n0) / F8B) * p.sb_n, 0x7ffffffcu);
  uint32_t vsa[SL];
#pragma unroll
  for (int i = 0; i < SL; ++i)
    vsa[i] = min((uint32_t)(wm * TM + (TM == 32 ? lane & 31 : i * 64 + lane)), rows_a - 1) * (uint32_t)p.sa_row * 4u;
  struct Scales {
    float a[SL], b;
  };
  auto request_scales = [&](uint32_t kb) {
    Scales s;
#pragma unroll
    for (int i = 0; i < SL; ++i) s.a[i] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rsa, (int)vsa[i], (int)(kb * p.sa_block * 4u), 0));
    s.b = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rsb, 0, (int)(kb * p.sb_block * 4u), 0));
    return s;
  };
  // -> scale[i]: that of row i * 16 + r16 of the wavefront's, in all four groups of lanes
  auto spread = [&](const Scales& s, float (&scale)[MT]) {
    auto u = [](float x) { return __builtin_bit_cast(uint32_t, x); };
    auto f = [](auto x) { return __builtin_bit_cast(float, (uint32_t)x); };
#pragma unroll
    for (int i = 0; i < SL; ++i) {
      const uint32_t v = u(s.a[i] * s.b);
      const auto h = __builtin_amdgcn_permlane16_swap(v, v, false, false);      // groups of lanes 0 0 2 2, and 1 1 3 3
      if constexpr (TM == 32) {
        scale[0] = f(h[0]);
        scale[1] = f(h[1]);
      } else {
        const auto e = __builtin_amdgcn_permlane32_swap((uint32_t)h[0], (uint32_t)h[0], false, false);
        const auto o = __builtin_amdgcn_permlane32_swap((uint32_t)h[1], (uint32_t)h[1], false, false);
        scale[4 * i] = f(e[0]);
        scale[4 * i + 1] = f(o[0]);
        scale[4 * i + 2] = f(e[1]);
        scale[4 * i + 3] = f(o[1]);
      }
    }
  };

  v4f acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};

  // a fragment: 16 rows from a multiple of 16 on; chunks q and q + 4 lie 64 bytes apart, one way or the other
  const uint32_t lo = (uint32_t)(r16 * 128 + ((q ^ (r16 >> 1)) * 16)), hi = lo ^ 64u;
  auto fragment = [&](const uint8_t* rows) {
    const v4i x = *reinterpret_cast<const v4i*>(rows + lo), y = *reinterpret_cast<const v4i*>(rows + hi);
    return v8i{x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
  };
  auto compute = [&](const uint8_t* at, const Scales& s) {
    float scale[MT];
    spread(s, scale);
    v8i w[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) w[j] = fragment(at + BM * 128 + (wn * TN + j * 16) * 128);
    v4f part[2][NT];
#pragma unroll
    for (int i = 0; i <= MT; ++i) {
      if (i < MT) {
        const v8i x = fragment(at + (wm * TM + i * 16) * 128);
#pragma unroll
        for (int j = 0; j < NT; ++j) part[i & 1][j] = mfma_fp8_block(w[j], x);
      }
      if (i > 0) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i - 1][j][e] = __builtin_fmaf(scale[i - 1], part[(i - 1) & 1][j][e], acc[i - 1][j][e]);
      }
    }
  };

  const int steps = (p.K + F8B - 1) / F8B;
  constexpr int OPS = A_LD + B_LD, SCALES = SL + 1;      // requests of a step
  // Behind a step's operands come those of the next NST - 2 steps and at least so many steps' scales: what may be under way when that step begins.
  constexpr int BEHIND = (NST - 2) * OPS + (NST - 2 < 2 ? NST - 2 : 2) * SCALES;
  static_assert(BEHIND <= 63, "wait counter range");
#pragma unroll
  for (int s = 0; s < NST - 1; ++s)
    if (s < steps) request((uint32_t)s * F8B, lds8 + s * STAGE);
  Scales now = request_scales(0);
  if (steps >= NST - 1) asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((NST - 2) * OPS + SCALES) : "memory");
  else asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
  // Step s: its operands have landed for everybody and stage s - 1 has been read by everybody (the barrier ahead of it); the scales of step s + 1
  // and the operands of step s + NST - 1 are requested.
  int stage = 0;
  for (int s = 0; s < steps; ++s) {
    const Scales next = request_scales((uint32_t)min(s + 1, steps - 1));
    if (s + NST - 1 < steps) request((uint32_t)(s + NST - 1) * F8B, lds8 + (stage == 0 ? NST - 1 : stage - 1) * STAGE);
    compute(lds8 + stage * STAGE, now);
    if (s + NST <= steps) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(BEHIND) : "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    now = next;
    stage = stage + 1 == NST ? 0 : stage + 1;
  }

  // four neighbouring columns of a row a lane
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int n = n0 + wn * TN + j * 16 + q * 4;
    if (n >= p.N) continue;
    float bias[4] = {0.f, 0.f, 0.f, 0.f};
    if (p.bias) {
#pragma unroll
      for (int e = 0; e < 4; ++e) bias[e] = T::to_float(p.bias[n + e]);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int m = m0 + wm * TM + i * 16 + r16;
      if (m >= p.M) continue;
      uint16_t o[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = T::from_float(acc[i][j][e] + bias[e]);
      *reinterpret_cast<v2u*>(p.out + (int64_t)m * p.ldc + n) = v2u{(uint32_t)o[0] | (uint32_t)o[1] << 16, (uint32_t)o[2] | (uint32_t)o[3] << 16};
    }
  }
}

}  // namespace vaq
