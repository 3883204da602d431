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

// A wavefront's part of a tile: TM x TN results, from fragments of both operands in LDS rows of 128 bytes.
template <bool BF16, int TM, int TN>
struct F8bWave {
  static constexpr int MT = TM / 16, NT = TN / 16, SL = TM <= 64 ? 1 : TM / 64;      // SL: loads of row scales
  static_assert((TM == 32 || TM % 64 == 0) && TN <= F8B && F8B % TN == 0, "shape of a wavefront");
  struct Scales {
    float a[SL], b;
  };
  v4f acc[MT][NT], part[NT];      // part, pend: the last products, which the next ones' multiply-adds add
  float scale[MT], pend;
  uint32_t lo, hi;                // a fragment: chunks q and q + 4 of 16 rows, 64 bytes apart one way or the other
  __amdgpu_buffer_rsrc_t rsa, rsb;
  uint32_t vsa[SL], sa_step, sb_step;

  // rows from `row` on of the tile's first, `rows` of them in it; columns from n on
  __device__ inline void start(const Fp8BlockParams& p, int m0, int row, int rows, int n, int n_tile) {
    const int lane = threadIdx.x & 63, q = lane >> 4, r16 = lane & 15;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      part[j] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < MT; ++i) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
    }
    pend = 0.f;
    lo = (uint32_t)(r16 * 128 + ((q ^ (r16 >> 1)) * 16));
    hi = lo ^ 64u;
    rsa = f8b_rsrc(p.sa + (int64_t)m0 * p.sa_row, 0x7ffffffcu);
    rsb = f8b_rsrc(p.sb + (int64_t)((n < p.N ? n : n_tile) / F8B) * p.sb_n, 0x7ffffffcu);
#pragma unroll
    for (int i = 0; i < SL; ++i) vsa[i] = (uint32_t)min(row + (TM == 32 ? lane & 31 : i * 64 + lane), rows - 1) * (uint32_t)p.sa_row * 4u;
    sa_step = p.sa_block * 4u;
    sb_step = p.sb_block * 4u;
  }
  // scales of block kb: of the rows (lane: row i * 64 + lane; 32 rows twice) and of the columns
  __device__ inline Scales request_scales(uint32_t kb) const {
    Scales s;
#pragma unroll
    for (int i = 0; i < SL; ++i) s.a[i] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rsa, (int)vsa[i], (int)(kb * sa_step), 0));
    s.b = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rsb, 0, (int)(kb * sb_step), 0));
    return s;
  }
  // -> scale[i]: that of row i * 16 + r16, in all four groups of 16 lanes
  __device__ inline void spread(const Scales& s) {
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
  }
  __device__ inline v8i fragment(const uint8_t* rows) const {
    const v4i x = *reinterpret_cast<const v4i*>(rows + lo), y = *reinterpret_cast<const v4i*>(rows + hi);
    return v8i{x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
  }
  // Products of 16 rows (number i) with all columns.  Each takes the place of the one before it in `part`, behind the four multiply-adds that add that one: its result is
  // NT instructions old by then.
  __device__ inline void add(int i, float s) {
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][j][e] = __builtin_fmaf(s, part[j][e], acc[i][j][e]);
  }
  __device__ inline void multiply(int i, const v8i (&w)[NT], const v8i& x) {
    const int before = i == 0 ? MT - 1 : i - 1;
    const float s = i == 0 ? pend : scale[before];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[before][j][e] = __builtin_fmaf(s, part[j][e], acc[before][j][e]);
      part[j] = mfma_fp8_block(w[j], x);
    }
    if (i == MT - 1) pend = scale[MT - 1];
  }
  // four neighbouring columns of a row a lane
  __device__ inline void store(const Fp8BlockParams& p, int m, int n) {
    using T = F16Traits<BF16>;
    add(MT - 1, pend);
    const int lane = threadIdx.x & 63;
    m += lane & 15;
    n += (lane >> 4) * 4;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      if (n + j * 16 >= p.N) continue;
      float bias[4] = {0.f, 0.f, 0.f, 0.f};
      if (p.bias) {
#pragma unroll
        for (int e = 0; e < 4; ++e) bias[e] = T::to_float(p.bias[n + j * 16 + e]);
      }
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        if (m + i * 16 >= p.M) continue;
        uint16_t o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = T::from_float(acc[i][j][e] + bias[e]);
        *reinterpret_cast<v2u*>(p.out + (int64_t)(m + i * 16) * p.ldc + n + j * 16) = v2u{(uint32_t)o[0] | (uint32_t)o[1] << 16, (uint32_t)o[2] | (uint32_t)o[3] << 16};
      }
    }
  }
};

// The compiler's schedule of a run of products: four multiply-adds, one product, `reads` LDS reads behind each row of them but the last.
template <int ROWS, int NT, int READS>
__device__ inline void f8b_order() {
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      __builtin_amdgcn_sched_group_barrier(0x2, 4, 0);
      __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
    }
    if (READS && i + 1 < ROWS) __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
  }
}

// A barrier under a condition that the whole wavefront shares, without a branch that the compiler sees: it moves multiply-adds behind one, out of the
// products' shadow.
__device__ inline void f8b_barrier_if(bool condition) {
#ifdef __HIP_DEVICE_COMPILE__
  asm volatile("s_cmp_eq_u32 %0, 0\n\ts_cbranch_scc1 .Lno_barrier%=\n\ts_barrier\n.Lno_barrier%=:" ::"s"(__builtin_amdgcn_readfirstlane((uint32_t)condition)) : "scc", "memory");
#endif
}

// Requests for a tile's rows of one operand: ROWS rows by NW wavefronts, 8 rows of 128 bytes an instruction.  Lane l writes place l & 7 of row r0 + l / 8, r0 = 8 times
// the instruction's number; odd numbers differ by 4 in the place's XOR.  (A row past the last counts as the last, see vaq_common.h: the first eight lanes ask for that one
// over again, the others for nothing.)  A step past K asks for nothing, and keeps the count of requests under way what it is on every path.  TAIL: K ends inside a step.
template <int ROWS, int NW, bool TAIL>
struct F8bOperand {
  static constexpr int LD = ROWS / (8 * NW);
  static_assert(LD >= 1, "fewer rows than the wavefronts ask for");
  __amdgpu_buffer_rsrc_t r;
  uint32_t row, lbyte, pitch, last, K;
  int wave;
  __device__ inline void start(const uint8_t* base, int64_t first, int rows, uint32_t pitch_, int K_, int wave_) {
    const uint32_t lane = threadIdx.x & 63;
    pitch = pitch_;
    K = (uint32_t)K_;
    last = (uint32_t)rows - 1;
    wave = wave_;
    r = f8b_rsrc(base + first * pitch, last * pitch + K);      // (the tile's own rows: no offset passes 32 bits)
    row = (lane >> 3) * pitch;
    lbyte = ((lane & 7) ^ (lane >> 4)) * 16;
  }
  __device__ inline void request(uint32_t k, uint8_t* at) const {
    typedef __attribute__((address_space(3))) void* lds_ptr_t;
    auto offset = [&](uint32_t byte) { return (int)((TAIL ? k + byte : k) < K ? row + byte : F8B_NOWHERE); };
    const int v0 = offset(lbyte), v1 = offset(lbyte ^ 64u);
    k = k < K ? k : 0;
#pragma unroll
    for (int i = 0; i < LD; ++i) {
      const uint32_t r0 = (uint32_t)(wave * LD + i) * 8;
      const bool odd = LD % 2 == 0 ? i & 1 : (r0 & 8) != 0;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr_t)(at + r0 * 128), 16, odd ? v1 : v0, (int)(min(r0, last) * pitch + k), 0, 0);
    }
  }
};

template <bool BF16, int BM, int BN, int WAVES_M, int WAVES_N, int NST, bool TAIL>
__global__ __launch_bounds__(WAVES_M * WAVES_N * 64) void fp8_block_tile_kernel(const Fp8BlockParams p, const uint32_t tiles_m, const uint32_t tiles_n) {
  constexpr int NW = WAVES_M * WAVES_N, TM = BM / WAVES_M, TN = BN / WAVES_N, STAGE = (BM + BN) * 128;
  using Wave = F8bWave<BF16, TM, TN>;
  constexpr int MT = Wave::MT, NT = Wave::NT;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds8[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / WAVES_N, wn = wave % WAVES_N;
  const uint32_t position = f8b_position(blockIdx.x, tiles_m * tiles_n);
  if (position >= tiles_m * tiles_n) return;
  const F8bTile tile = f8b_tile(position, tiles_m, tiles_n, BM, BN);
  const int m0 = tile.m0, n0 = tile.n0, rows = min(BM, p.M - m0);

  F8bOperand<BM, NW, TAIL> a;
  F8bOperand<BN, NW, TAIL> b;
  a.start(p.a, m0, rows, p.lda, p.K, wave);
  b.start(p.b, n0, min(BN, p.N - n0), p.ldb, p.K, wave);
  Wave w;
  w.start(p, m0, wm * TM, rows, n0 + wn * TN, n0);
  auto request = [&](int step, uint8_t* at) {
    a.request((uint32_t)step * F8B, at);
    b.request((uint32_t)step * F8B, at + BM * 128);
  };
  auto compute = [&](const uint8_t* at, const typename Wave::Scales& s) {
    v8i cols[NT], row[2];
#pragma unroll
    for (int j = 0; j < NT; ++j) cols[j] = w.fragment(at + BM * 128 + (wn * TN + j * 16) * 128);
    row[0] = w.fragment(at + wm * TM * 128);
    w.spread(s);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      if (i + 1 < MT) row[(i + 1) & 1] = w.fragment(at + (wm * TM + (i + 1) * 16) * 128);
      w.multiply(i, cols, row[i & 1]);
    }
    __builtin_amdgcn_sched_group_barrier(0x100, 2 * NT + 4, 0);
    f8b_order<MT, NT, 2>();
  };

  const int steps = (p.K + F8B - 1) / F8B;
  constexpr int OPS = a.LD + b.LD, SCALES = Wave::SL + 1;      // requests of a step
  // Behind a step's operands come those of the next NST - 2 steps and at least so many steps' scales: what may be under way when that step begins.
  constexpr int BEHIND = (NST - 2) * OPS + (NST - 2 < 2 ? NST - 2 : 2) * SCALES;
  static_assert(BEHIND <= 63, "wait counter range");
#pragma unroll
  for (int s = 0; s < NST - 1; ++s) request(s, lds8 + s * STAGE);
  typename Wave::Scales now = w.request_scales(0);
  asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((NST - 2) * OPS + SCALES) : "memory");
  // Step s: its operands have landed for everybody and stage s - 1 has been read by everybody (the barrier ahead of it); the scales of step s + 1
  // and the operands of step s + NST - 1 are requested.
  int stage = 0;
#pragma unroll 1
  for (int s = 0; s < steps; ++s) {
    __builtin_amdgcn_sched_barrier(0);
    const typename Wave::Scales next = w.request_scales((uint32_t)min(s + 1, steps - 1));
    __builtin_amdgcn_sched_barrier(0);
    request(s + NST - 1, lds8 + (stage == 0 ? NST - 1 : stage - 1) * STAGE);
    __builtin_amdgcn_sched_barrier(0);
    compute(lds8 + stage * STAGE, now);
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(BEHIND) : "memory");
    now = next;
    stage = stage + 1 == NST ? 0 : stage + 1;
  }
  w.store(p, m0 + wm * TM, n0 + wn * TN);
}

// 256 x 256 results by eight wavefronts of 128 x 64 in alternating phases: of the two that share a SIMD one reads its fragments and requests operands while
// the other one's products and multiply-adds run.  The LDS has five places for an operand of a step, which weights and activations take in turn, B(0) A(0) B(1) A(1) ...: a
// step's weights are free behind its first phase, the activations behind its second, and each is at once replaced by what comes two and a half steps later.
// A step of a wavefront is [read columns and rows 0 .. 63, request B(s + 2)] barrier [products] barrier [read rows 64 .. 127, request A(s + 2), wait for what step s + 1
// reads] barrier [products] barrier; the late half of the workgroup passes one extra barrier first and skips its last one, so that every wavefront passes the same number.
template <bool BF16, bool TAIL>
__global__ __launch_bounds__(512) void fp8_block_tile256_kernel(const Fp8BlockParams p, const uint32_t tiles_m, const uint32_t tiles_n) {
  constexpr int B = 256, NW = 8, TM = 128, TN = 64, PLACE = B * 128;
  using Wave = F8bWave<BF16, TM, TN>;
  constexpr int NT = Wave::NT;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds8[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave >> 2, wn = wave & 3;
  const bool late = wave >= 4;      // wavefronts w and w + 4 share a SIMD
  const uint32_t position = f8b_position(blockIdx.x, tiles_m * tiles_n);
  if (position >= tiles_m * tiles_n) return;
  const F8bTile tile = f8b_tile(position, tiles_m, tiles_n, B, B);
  const int m0 = tile.m0, n0 = tile.n0, rows = min(B, p.M - m0);

  F8bOperand<B, NW, TAIL> a, b;
  a.start(p.a, m0, rows, p.lda, p.K, wave);
  b.start(p.b, n0, min(B, p.N - n0), p.ldb, p.K, wave);
  Wave w;
  w.start(p, m0, wm * TM, rows, n0 + wn * TN, n0);
  constexpr int LD = a.LD;      // requests of a wavefront for an operand

  const int steps = (p.K + F8B - 1) / F8B;
  int qb = 0;      // place of this step's weights
  auto place = [&](int ahead) {
    const int q = qb + ahead;
    return lds8 + (q >= 5 ? q - 5 : q) * PLACE;
  };
  typename Wave::Scales now = w.request_scales(0);
  b.request(0, place(0));
  a.request(0, place(1));
  b.request(F8B, place(2));
  a.request(F8B, place(3));
  asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(2 * LD) : "memory");
  if (late) asm volatile("s_barrier" ::: "memory");
  v8i cols[NT], row[4];
  auto products = [&](int first) {
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 4; ++i) w.multiply(first + i, cols, row[i]);
    f8b_order<4, NT, 0>();
    __builtin_amdgcn_sched_barrier(0);
  };
#pragma unroll 1
  for (int s = 0; s < steps; ++s) {
    const uint8_t* const at_b = place(0) + wn * TN * 128;
    const uint8_t* const at_a = place(1) + wm * TM * 128;
#pragma unroll
    for (int j = 0; j < NT; ++j) cols[j] = w.fragment(at_b + j * 2048);
#pragma unroll
    for (int i = 0; i < 4; ++i) row[i] = w.fragment(at_a + i * 2048);
    w.spread(now);
    __builtin_amdgcn_sched_barrier(0);
    now = w.request_scales((uint32_t)min(s + 1, steps - 1));
    __builtin_amdgcn_sched_barrier(0);
    b.request((uint32_t)(s + 2) * F8B, place(4));
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    products(0);
    asm volatile("s_barrier" ::: "memory");
#pragma unroll
    for (int i = 0; i < 4; ++i) row[i] = w.fragment(at_a + (4 + i) * 2048);
    __builtin_amdgcn_sched_barrier(0);
    a.request((uint32_t)(s + 2) * F8B, place(0));
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(2 * LD) : "memory");
    products(4);
    f8b_barrier_if(!late || s + 1 < steps);
    qb = qb >= 3 ? qb - 3 : qb + 2;
  }
  w.store(p, m0 + wm * TM, n0 + wn * TN);
}

}  // namespace vaq
