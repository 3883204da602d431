// FP8 product with a scale for each block of 128 (fp8_block_mm.h): tiles.
//
//  * BM x BN results a workgroup; a step is one block of K.  Both operands come by direct-to-LDS loads of whole 128-byte lines (8 rows an instruction) into a
//    ring of NST stages; chunk c of a row lies at place c ^ (row / 2 & 7) of its 128 bytes, so that the 16 lanes that are served together hit all banks.
//  * A product is issued behind the four multiply-adds that add the one before it in its registers: they find their result ready, and run beside an instruction
//    that keeps the matrix core for 32 cycles (measured without a loss of the product's rate).
//
// 4096 x 4096 x 28672: 400 .. 420 us by 256 x 256 tiles = 2.3 PFLOP/s, the rate of the library's 8192^3 product without block scales (2.25 .. 2.31), and the card's power limit
// (zeros run a quarter faster).  That is the rate of a steady stream of calls: behind an idle device the first three take as long, the next ones 440 .. 580 us until the power control has
// settled, some 70 calls later (profiles/block_fp8_kernels.txt).  333 rows, K = 2976, N = 10240, by 128 x 128 tiles on 240 of 256 compute units: 18.8 .. 20 us in a stream of calls over
// the same weights, 22.7 in a graph of them, 24.8 in a graph with cold weights; bytes 7.5, products 9.
// What the smaller tiles wait for is the operands' way into a compute unit, in part: 790 KB there, for which reads alone (profiles/fp8_128x128_tiles_read_probe.txt) take 10.4 us of weights that
// the launch before read (76 bytes/ns) and 16.8 of cold ones (47).  The other 8 us of either are not explained by it.
// Measured without gain: two groups of four wavefronts with half of K each on a compute unit (12.6 us for 12.6 at 128 x 4096 x 4096, 64 x 64 tiles), less LDS traffic by four wavefronts of
// 64 x 64 (3 % either way), weights from memory straight into registers (1.0 .. 1.3 x the time), two blocks of K a step (level), fewer stages and two workgroups on a
// compute unit (8 .. 60 % slower where there is one tile for each).
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
  static constexpr int MT = TM / 16, NT = TN / 16;
  static_assert(TN <= F8B && F8B % TN == 0, "the columns of a wavefront share their scale");
  v4f acc[MT][NT], part[NT];      // part, pend: the last products, which the next ones' multiply-adds add
  float scale[MT], pend;
  uint32_t lo, hi;                // a fragment: chunks q and q + 4 of 16 rows, 64 bytes apart one way or the other

  __device__ inline void start() {
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
  // The products stand ahead of this, not behind the barrier that follows: the compiler may move what only a later phase uses.  (Nothing reads the registers here, so nothing
  // waits for them.)
  __device__ inline void hold() {
#ifdef __HIP_DEVICE_COMPILE__
#pragma unroll
    for (int j = 0; j < NT; ++j) asm volatile("" : "+v"(part[j]));
#endif
  }
  // Results of the wavefront's part, which begins at (m, n).  They cross a piece of LDS of the wavefront's own (LDS_BYTES; everybody is done with the operands), 16 rows at a time, so
  // that they leave as 16-byte stores, whole lines of 128 bytes.  As they lie in registers, a store of 8 bytes a lane touches 16 rows with 32 bytes each, and the
  // requests of a device that finishes its tiles at the same time took 13 us.  Where the output is not aligned to 16 bytes they leave that way.
  static constexpr int PITCH = TN * 2 + 16, LDS_BYTES = 16 * PITCH;
  __device__ inline void store(const Fp8BlockParams& p, int m, int n, uint8_t* lds) {
    using T = F16Traits<BF16>;
    add(MT - 1, pend);
    const int lane = threadIdx.x & 63, q = lane >> 4, r16 = lane & 15;
    float bias[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int c = n + j * 16 + q * 4 + e;
        bias[j][e] = p.bias && c < p.N ? T::to_float(p.bias[c]) : 0.f;
      }
    const bool lines = ((uintptr_t)p.out & 15) == 0 && p.ldc % 8 == 0;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        uint16_t o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = T::from_float(acc[i][j][e] + bias[j][e]);
        const v2u four{(uint32_t)o[0] | (uint32_t)o[1] << 16, (uint32_t)o[2] | (uint32_t)o[3] << 16};
        if (lines) *reinterpret_cast<v2u*>(lds + r16 * PITCH + (j * 16 + q * 4) * 2) = four;
        else if (m + i * 16 + r16 < p.M && n + j * 16 < p.N) *reinterpret_cast<v2u*>(p.out + (int64_t)(m + i * 16 + r16) * p.ldc + n + j * 16 + q * 4) = four;
      }
      if (lines) {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_wave_barrier();      // lanes exchange data through LDS; its operations run in program order
        constexpr int CHUNKS = TN / 8;        // of 16 bytes in a row
        static_assert(16 * CHUNKS % 64 == 0, "whole wavefronts");
#pragma unroll
        for (int c = 0; c < 16 * CHUNKS; c += 64) {
          const int row = (c + lane) / CHUNKS, chunk = (c + lane) % CHUNKS;
          const v4u eight = *reinterpret_cast<const v4u*>(lds + row * PITCH + chunk * 16);
          if (m + i * 16 + row < p.M && n + chunk * 8 < p.N) *reinterpret_cast<v4u*>(p.out + (int64_t)(m + i * 16 + row) * p.ldc + n + chunk * 8) = eight;
        }
        asm volatile("" ::: "memory");
        __builtin_amdgcn_wave_barrier();
      }
    }
  }
};

// The same with the rows' scales in registers: one load for 64 rows, multiplied by the columns' scale and spread over the four groups of 16 lanes by swaps.
template <bool BF16, int TM, int TN>
struct F8bWaveScales : F8bWave<BF16, TM, TN> {
  using Base = F8bWave<BF16, TM, TN>;
  static constexpr int SL = TM / 64;      // loads of row scales
  static_assert(TM % 64 == 0, "scales are loaded for 64 rows");
  struct Scales {
    float a[SL], b;
  };
  __amdgpu_buffer_rsrc_t rsa, rsb;
  uint32_t vsa[SL], sa_step, sb_step;
  // rows from `row` on of the tile's, which begin at m0 and are `rows`; columns from n on
  __device__ inline void start(const Fp8BlockParams& p, int m0, int row, int rows, int n, int n_tile) {
    const int lane = threadIdx.x & 63;
    Base::start();
    rsa = f8b_rsrc(p.sa + (int64_t)m0 * p.sa_row, 0x7ffffffcu);
    rsb = f8b_rsrc(p.sb + (int64_t)((n < p.N ? n : n_tile) / F8B) * p.sb_n, 0x7ffffffcu);
#pragma unroll
    for (int i = 0; i < SL; ++i) vsa[i] = (uint32_t)min(row + i * 64 + lane, rows - 1) * (uint32_t)p.sa_row * 4u;
    sa_step = p.sa_block * 4u;
    sb_step = p.sb_block * 4u;
  }
  // scales of block kb: of the rows (lane: row i * 64 + lane) and of the columns
  __device__ inline Scales request_scales(uint32_t kb) const {
    Scales s;
#pragma unroll
    for (int i = 0; i < SL; ++i) s.a[i] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rsa, (int)vsa[i], (int)(kb * sa_step), 0));
    s.b = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rsb, 0, (int)(kb * sb_step), 0));
    return s;
  }
  // -> scale[i]: that of row i * 16 + r16, in all four groups of 16 lanes
  __device__ inline void spread(const Scales& s, float (&scale)[TM / 16]) const {
    auto u = [](float x) { return __builtin_bit_cast(uint32_t, x); };
    auto f = [](auto x) { return __builtin_bit_cast(float, (uint32_t)x); };
#pragma unroll
    for (int i = 0; i < SL; ++i) {
      const uint32_t v = u(s.a[i] * s.b);
      const auto h = __builtin_amdgcn_permlane16_swap(v, v, false, false);      // groups of lanes 0 0 2 2, and 1 1 3 3
      const auto e = __builtin_amdgcn_permlane32_swap((uint32_t)h[0], (uint32_t)h[0], false, false);
      const auto o = __builtin_amdgcn_permlane32_swap((uint32_t)h[1], (uint32_t)h[1], false, false);
      scale[4 * i] = f(e[0]);
      scale[4 * i + 1] = f(o[0]);
      scale[4 * i + 2] = f(e[1]);
      scale[4 * i + 3] = f(o[1]);
    }
  }
};

// The compiler's schedule of N products, each behind four multiply-adds: READS LDS reads, the same number beside each of the first WITH products, and requests beside the others.
template <int N, int READS, int WITH, int REQUESTS>
__device__ inline void f8b_order() {
  constexpr int R = WITH ? (READS + WITH - 1) / (WITH ? WITH : 1) : 0, Q = N > WITH ? (REQUESTS + N - WITH - 1) / (N > WITH ? N - WITH : 1) : 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x2, 4, 0);
    __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
    if (i < WITH) __builtin_amdgcn_sched_group_barrier(0x100, R, 0);
    else if (REQUESTS) __builtin_amdgcn_sched_group_barrier(0x10, Q, 0);
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

// The same with all of a lane's offsets in registers, so that a request is one instruction and its LDS address.
template <int ROWS, int NW, bool TAIL>
struct F8bOperandOffsets {
  static constexpr int LD = ROWS / (8 * NW);
  static_assert(LD >= 1, "fewer rows than the wavefronts ask for");
  const uint8_t* base;
  uint32_t v[LD], extent, lbyte, K;
  int wave;
  __device__ inline void start(const uint8_t* operand, int64_t first, int rows, uint32_t pitch, int K_, int wave_) {
    const uint32_t lane = threadIdx.x & 63;
    K = (uint32_t)K_;
    wave = wave_;
    base = operand + first * pitch;
    extent = (uint32_t)(rows - 1) * pitch + K;
    lbyte = ((lane & 7) ^ (lane >> 4)) * 16;
#pragma unroll
    for (int i = 0; i < LD; ++i) {
      const uint32_t r0 = (uint32_t)(wave * LD + i) * 8, row = r0 + (lane >> 3);
      v[i] = row < (uint32_t)rows ? row * pitch + (lbyte ^ (r0 & 8 ? 64u : 0u)) : F8B_NOWHERE;
    }
  }
  // k = K: nothing
  __device__ inline void request(uint32_t k, uint8_t* at) const {
    typedef __attribute__((address_space(3))) void* lds_ptr_t;
    const bool some = k < K;
    const __amdgpu_buffer_rsrc_t r = f8b_rsrc(base, some ? extent : 0u);
    const int so = some ? (int)k : 0;
#pragma unroll
    for (int i = 0; i < LD; ++i) {
      const uint32_t r0 = (uint32_t)(wave * LD + i) * 8;
      const bool odd = LD % 2 == 0 ? i & 1 : (r0 & 8) != 0;
      uint32_t offset = v[i];
      if constexpr (TAIL) offset = k + (lbyte ^ (odd ? 64u : 0u)) < K ? offset : F8B_NOWHERE;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr_t)(at + r0 * 128), 16, (int)offset, so, 0, 0);
    }
  }
};

// What the first requests need, which arrives in registers with the launch.
struct F8bHead {
  const uint8_t *a, *b;
  uint32_t lda, ldb, tiles_m, tiles_n;
  int K, M, N;
};
inline KernelHead f8b_head(const Fp8BlockParams& p, uint32_t tiles_m, uint32_t tiles_n) {
  return KernelHead{v8u{ptr_lo(p.a), ptr_hi(p.a), ptr_lo(p.b), ptr_hi(p.b), p.lda, p.ldb, (uint32_t)p.K, (uint32_t)p.M}, v4u{(uint32_t)p.N, tiles_m, tiles_n, 0u}, v2u{}};
}
__device__ inline F8bHead f8b_head_of(v8u h, v4u h2) {
  return F8bHead{head_ptr<uint8_t>(h[0], h[1]), head_ptr<uint8_t>(h[2], h[3]), h[4], h[5], h2[1], h2[2], (int)h[6], (int)h[7], (int)h2[0]};
}

// BM x BN results through a ring of NST stages.  A step's fragments are in registers when it begins; its products run while the next step's fragments are read,
// and its stage, which nobody needs any more, takes the operands NST steps on.  So NST - 1 steps are under way, and a step costs the longer of its LDS traffic and its products, and one
// barrier.  The rows' scales travel with the operands (a load of four bytes a lane into the stage): loaded into registers a step ahead they would be answered behind
// the operands of all steps under way, which the wait for them would then be a wait for.  The columns' scales of all of K are requested once, behind the first step's operands.
template <int BM, int BN, int NST>
struct F8bRing {
  static constexpr int SCALES = BM * 128 + BN * 128, STAGE = SCALES + BM * 4;
  static inline size_t lds_bytes(int64_t K) { return (size_t)NST * STAGE + (BN + F8B - 1) / F8B * 4 * (size_t)sb_floats((int)K); }
  __host__ __device__ static inline int sb_floats(int K) { return ((K + F8B - 1) / F8B + 1 + 63) / 64 * 64; }      // of a block of columns: one past K, which is zero
};
template <bool BF16, int BM, int BN, int WAVES_M, int WAVES_N, int NST, bool TAIL>
__global__ __launch_bounds__(WAVES_M * WAVES_N * 64, 2) void fp8_block_tile_kernel(const v8u head, const v4u head2, const Fp8BlockParams p) {
  constexpr int NW = WAVES_M * WAVES_N, TM = BM / WAVES_M, TN = BN / WAVES_N;
  using Wave = F8bWave<BF16, TM, TN>;
  using Ring = F8bRing<BM, BN, NST>;
  constexpr int MT = Wave::MT, NT = Wave::NT, NB = (BN + F8B - 1) / F8B;
  static_assert(BM <= 64 * NW, "each wavefront asks for the scales of 64 rows");
  extern __shared__ __attribute__((aligned(16))) uint8_t lds8[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / WAVES_N, wn = wave % WAVES_N;
  const F8bHead h = f8b_head_of(head, head2);
  const uint32_t position = f8b_position(blockIdx.x, h.tiles_m * h.tiles_n);
  if (position >= h.tiles_m * h.tiles_n) return;
  const F8bTile tile = f8b_tile(position, h.tiles_m, h.tiles_n, BM, BN);
  const int m0 = tile.m0, n0 = tile.n0, rows = min(BM, h.M - m0), steps = (h.K + F8B - 1) / F8B;
  F8bOperandOffsets<BM, NW, TAIL> a;
  F8bOperandOffsets<BN, NW, TAIL> b;
  a.start(h.a, m0, rows, h.lda, h.K, wave);
  b.start(h.b, n0, min(BN, h.N - n0), h.ldb, h.K, wave);
  Wave w;
  w.start();
  typedef __attribute__((address_space(3))) void* lds_ptr_t;
  const int sb_floats = Ring::sb_floats(h.K);
  float* const sb_lds = reinterpret_cast<float*>(lds8 + NST * Ring::STAGE);      // [block of columns][block of K]
  auto request_columns_scales = [&] {
    // (every wavefront asks for all of them: each then waits for its own requests only)
    const int nb0 = n0 / F8B, nb_n = (h.N + F8B - 1) / F8B - nb0;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
      for (int i = 0; i < sb_floats; i += 64)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(f8b_rsrc(p.sb + (int64_t)(nb0 + (nb < nb_n ? nb : 0)) * p.sb_n, 0x7ffffffcu), (lds_ptr_t)(sb_lds + nb * sb_floats + i), 4,
                                                 (int)(i + lane < steps ? (uint32_t)(i + lane) * p.sb_block * 4u : F8B_NOWHERE), 0, 0, 0);
  };
  const int sa_first = wave % (BM / 64) * 64;
  const uint32_t vsa = (uint32_t)min(sa_first + lane, rows - 1) * (uint32_t)p.sa_row * 4u, sa_step = p.sa_block * 4u;
  uint32_t k = 0, sa_next = 0;      // the block that is requested next; past K: nothing
  auto request = [&](uint8_t* at) {
    const bool some = k < (uint32_t)h.K;
    a.request(k, at);
    b.request(k, at + BM * 128);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(f8b_rsrc(p.sa + (int64_t)m0 * p.sa_row, some ? 0x7ffffffcu : 0u), (lds_ptr_t)(at + Ring::SCALES + sa_first * 4), 4, (int)vsa,
                                             (int)(some ? sa_next : 0u), 0, 0);
    k += F8B;
    sa_next += sa_step;
  };
  struct Step {
    v8i cols[NT], row[MT];
    float sa[MT], sb;
  };
  const uint8_t* const my_b = lds8 + BM * 128 + wn * TN * 128;
  const uint8_t* const my_a = lds8 + wm * TM * 128;
  const uint8_t* const my_sa = lds8 + Ring::SCALES + (wm * TM + (lane & 15)) * 4;
  const float* const my_sb = sb_lds + wn * TN / F8B * sb_floats;
  int kb_read = 0;
  auto read = [&](Step& f, int at) {
#pragma unroll
    for (int j = 0; j < NT; ++j) f.cols[j] = w.fragment(my_b + at + j * 2048);
#pragma unroll
    for (int i = 0; i < MT; ++i) f.row[i] = w.fragment(my_a + at + i * 2048);
#pragma unroll
    for (int i = 0; i < MT; ++i) f.sa[i] = *reinterpret_cast<const float*>(my_sa + at + i * 64);
    f.sb = my_sb[min(kb_read++, steps)];      // (past K: zero)
  };
  // Behind a step's operands come those of the next NST - 2 steps.
  constexpr int OPS = a.LD + b.LD + 1;
  static_assert((NST - 1) * OPS <= 63, "wait counter range");
  request(lds8);
  __builtin_amdgcn_sched_barrier(0);
  request_columns_scales();
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int s = 1; s < NST; ++s) request(lds8 + s * Ring::STAGE);
  asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((NST - 1) * OPS) : "memory");
  Step even, odd;
  int stage = 0;      // in bytes
  read(even, 0);
  // One step: its fragments are here (lgkmcnt) and everybody's, so that its stage is free; the next one's operands have landed for everybody.
  auto step = [&](Step& now, Step& next) {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((NST - 2) * OPS) : "memory");
    __builtin_amdgcn_sched_barrier(0);
    uint8_t* const free_stage = lds8 + stage;
    stage = stage + Ring::STAGE == NST * Ring::STAGE ? 0 : stage + Ring::STAGE;
    read(next, stage);
#pragma unroll
    for (int i = 0; i < MT; ++i) w.scale[i] = now.sa[i] * now.sb;
#pragma unroll
    for (int i = 0; i < MT; ++i) w.multiply(i, now.cols, now.row[i]);
    request(free_stage);
    f8b_order<MT * NT, 2 * (NT + MT) + MT + 1, MT * NT / 4, OPS>();      // (reads beside three quarters of the products: 128 x 256 tiles 3 % slower)
    __builtin_amdgcn_sched_barrier(0);
  };
  // (an odd number of steps ends with one of zeros)
#pragma unroll 1
  for (int s = 0; s < steps; s += 2) {
    step(even, odd);
    step(odd, even);
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");      // (requests for nothing write zeros)
  static_assert(NST * Ring::STAGE >= NW * Wave::LDS_BYTES, "room for the results");
  w.store(p, m0 + wm * TM, n0 + wn * TN, lds8 + wave * Wave::LDS_BYTES);
}

// 256 x 256 results by eight wavefronts of 128 x 64 in alternating phases: of the two that share a SIMD one reads its fragments and requests operands while
// the other one's products and multiply-adds run.  The LDS has five places for an operand of a step, which weights and activations take in turn, B(0) A(0) B(1) A(1) ...: a
// step's weights are free behind its first phase, the activations behind its second, and each is at once replaced by what comes two and a half steps later.
// A step of a wavefront is [read columns and rows 0 .. 31, request B(s + 2)] barrier [products of rows 0 .. 63, read rows 32 .. 95] barrier [read rows 96 .. 127, request A(s + 2),
// wait for what step s + 1 reads] barrier [products of rows 64 .. 127] barrier; the late half of the workgroup passes one extra barrier first and skips its last one, so that every wavefront passes the same number.
template <bool BF16, bool TAIL>
__global__ __launch_bounds__(512) void fp8_block_tile256_kernel(const v8u head, const v4u head2, const Fp8BlockParams p) {
  constexpr int B = 256, NW = 8, TM = 128, TN = 64, PLACE = B * 128;
  using Wave = F8bWaveScales<BF16, TM, TN>;
  constexpr int NT = Wave::NT;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds8[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave >> 2, wn = wave & 3;
  const bool late = wave >= 4;      // wavefronts w and w + 4 share a SIMD
  const F8bHead h = f8b_head_of(head, head2);
  const uint32_t position = f8b_position(blockIdx.x, h.tiles_m * h.tiles_n);
  if (position >= h.tiles_m * h.tiles_n) return;
  const F8bTile tile = f8b_tile(position, h.tiles_m, h.tiles_n, B, B);
  const int m0 = tile.m0, n0 = tile.n0, rows = min(B, h.M - m0);

  F8bOperand<B, NW, TAIL> a, b;
  a.start(h.a, m0, rows, h.lda, h.K, wave);
  b.start(h.b, n0, min(B, h.N - n0), h.ldb, h.K, wave);
  constexpr int LD = a.LD;      // requests of a wavefront for an operand

  const int steps = (h.K + F8B - 1) / F8B;
  int qb = 0;      // place of this step's weights
  auto place = [&](int ahead) {
    const int q = qb + ahead;
    return lds8 + (q >= 5 ? q - 5 : q) * PLACE;
  };
  b.request(0, place(0));
  a.request(0, place(1));
  __builtin_amdgcn_sched_barrier(0);      // (what follows waits for arguments)
  Wave w;
  w.start(p, m0, wm * TM, rows, n0 + wn * TN, n0);
  typename Wave::Scales first = w.request_scales(0), now = w.request_scales((uint32_t)min(1, steps - 1));
  __builtin_amdgcn_sched_barrier(0);
  b.request(F8B, place(2));
  a.request(F8B, place(3));
  asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(2 * LD) : "memory");
  if (late) asm volatile("s_barrier" ::: "memory");
  v8i cols[NT], row[4];
  float scale[Wave::MT];      // of the step to come
  w.spread(first, scale);
#pragma unroll 1
  for (int s = 0; s < steps; ++s) {
    const uint8_t* const at_b = place(0) + wn * TN * 128;
    const uint8_t* const at_a = place(1) + wm * TM * 128;
#pragma unroll
    for (int j = 0; j < NT; ++j) cols[j] = w.fragment(at_b + j * 2048);
    row[0] = w.fragment(at_a);
    row[1] = w.fragment(at_a + 2048);
#pragma unroll
    for (int i = 0; i < Wave::MT; ++i) w.scale[i] = scale[i];
    __builtin_amdgcn_sched_barrier(0);
    b.request((uint32_t)(s + 2) * F8B, place(4));
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(1);
    row[2] = w.fragment(at_a + 2 * 2048);
    row[3] = w.fragment(at_a + 3 * 2048);
    w.multiply(0, cols, row[0]);
    w.multiply(1, cols, row[1]);
    row[0] = w.fragment(at_a + 4 * 2048);
    row[1] = w.fragment(at_a + 5 * 2048);
    w.multiply(2, cols, row[2]);
    w.multiply(3, cols, row[3]);
    w.hold();
    f8b_order<NT, NT, NT, 0>();
    f8b_order<NT, 0, 0, 0>();
    f8b_order<NT, NT, NT, 0>();
    f8b_order<NT, 0, 0, 0>();
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(0);
    asm volatile("s_barrier" ::: "memory");
    row[2] = w.fragment(at_a + 6 * 2048);
    row[3] = w.fragment(at_a + 7 * 2048);
    __builtin_amdgcn_sched_barrier(0);
    const typename Wave::Scales next = w.request_scales((uint32_t)min(s + 2, steps - 1));
    __builtin_amdgcn_sched_barrier(0);
    a.request((uint32_t)(s + 2) * F8B, place(0));
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(2 * LD + Wave::SL + 1) : "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int i = 0; i < 4; ++i) w.multiply(4 + i, cols, row[i]);
    w.spread(now, scale);      // (requested a step ago: ahead of everything that is still under way)
    now = next;
#ifdef __HIP_DEVICE_COMPILE__
#pragma unroll
    for (int i = 0; i < Wave::MT; ++i) asm volatile("" : "+v"(scale[i]));
#endif
    w.hold();
    f8b_order<4 * NT, 0, 0, 0>();
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(0);
    f8b_barrier_if(!late || s + 1 < steps);
    qb = qb >= 3 ? qb - 3 : qb + 2;
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");      // (requests for nothing write zeros)
  static_assert(5 * PLACE >= NW * Wave::LDS_BYTES, "room for the results");
  w.store(p, m0 + wm * TM, n0 + wn * TN, lds8 + wave * Wave::LDS_BYTES);
}

}  // namespace vaq
