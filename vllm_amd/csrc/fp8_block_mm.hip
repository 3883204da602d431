// FP8 product with a scale for each block of 128 (fp8_block_mm.h): arguments, choice of the kernel, launch of the tiles.
#include "fp8_block_tile_kernel.h"

#include <math.h>

namespace vaq {

template <int BM, int BN, int WAVES, typename Kernel>
static int launch_tiles(const Fp8BlockParams& p, size_t lds, Kernel kern, size_t (&reserved)[VAQ_MAX_DEVICES], hipStream_t s) {
  const uint32_t tiles_m = ((uint32_t)p.M + BM - 1) / BM, tiles_n = ((uint32_t)p.N + BN - 1) / BN;
  if (const int rc = reserve_dynamic_lds(reinterpret_cast<const void*>(kern), lds, reserved, "fp8_block_scaled_mm"); rc != VAQ_OK) return rc;
  const KernelHead h = f8b_head(p, tiles_m, tiles_n);
  hipLaunchKernelGGL(kern, dim3((tiles_m * tiles_n + 7) / 8 * 8), dim3(WAVES * 64), lds, s, h.a, h.b, p);
  return VAQ_OK;
}
// tile shapes: rows, columns, wavefronts along both, stages of the ring
template <bool BF16, int BM, int BN, int WAVES_M, int WAVES_N, int NST>
static int launch_shape(const Fp8BlockParams& p, hipStream_t s) {
  static size_t whole[VAQ_MAX_DEVICES], tail[VAQ_MAX_DEVICES];
  const size_t lds = F8bRing<BM, BN, NST>::lds_bytes(p.K);
  constexpr int W = WAVES_M * WAVES_N;
  return p.K % F8B != 0 ? launch_tiles<BM, BN, W>(p, lds, fp8_block_tile_kernel<BF16, BM, BN, WAVES_M, WAVES_N, NST, true>, tail, s)
                        : launch_tiles<BM, BN, W>(p, lds, fp8_block_tile_kernel<BF16, BM, BN, WAVES_M, WAVES_N, NST, false>, whole, s);
}
template <bool BF16>
static int launch_256(const Fp8BlockParams& p, hipStream_t s) {
  static size_t whole[VAQ_MAX_DEVICES], tail[VAQ_MAX_DEVICES];
  constexpr size_t LDS = 5 * 256 * F8B;
  return p.K % F8B != 0 ? launch_tiles<256, 256, 8>(p, LDS, fp8_block_tile256_kernel<BF16, true>, tail, s)
                        : launch_tiles<256, 256, 8>(p, LDS, fp8_block_tile256_kernel<BF16, false>, whole, s);
}

template <bool BF16>
static int launch_type(const Fp8BlockParams& p, int shape, hipStream_t s) {
  switch (shape) {
    case 0: return launch_shape<BF16, 64, 64, 2, 2, 6>(p, s);
    case 1: return launch_shape<BF16, 64, 128, 2, 4, 6>(p, s);
    case 2: return launch_shape<BF16, 128, 128, 2, 4, 4>(p, s);
    case 3: return launch_shape<BF16, 128, 256, 2, 4, 3>(p, s);
    case 4: return launch_shape<BF16, 256, 128, 4, 2, 3>(p, s);
    case 6: return launch_shape<BF16, 128, 64, 4, 2, 6>(p, s);
    default: return launch_256<BF16>(p, s);
  }
}
int fp8_block_tile_launch(const Fp8BlockParams& p, bool bf16, int shape, hipStream_t s) {
  return bf16 ? launch_type<true>(p, shape, s) : launch_type<false>(p, shape, s);
}

// ----------------------------------------------------------------------------- choice of the kernel
// The cheapest plan by price, in us.  Rows: a step is a latency, the bytes into the compute unit or the products, whichever is longest; a workgroup is its start, its steps and its
// meeting; beside all of them the weights from memory, once and a share for every further block of rows.  Tiles: rounds of workgroups (a last, partly filled one costs a share of
// a full one), each a start and its steps, longer where few tiles of a column share the weights they read; beside them the weights from memory.  Fitted to the cold times of 4031
// problems (M 1 .. 8192, K 512 .. 14336, N 512 .. 28672; profiles/plan_prices/fp8_block_fit.csv.gz): of each the plans for few rows of at most eight blocks of rows, the 64-row tiles from
// 9 rows on and the others from a quarter of their rows on.  Over 1730 problems that the fit did not see (fp8_block.csv.gz) the cheapest plan takes 1.011 of the time of the fastest one timed
// in the mean; without eight wavefronts 1.018, without any one of the tile shapes 1.012 .. 1.033.  (profiles/plan_prices/fp8_block.py: the fit, from these constants on, gives them back.)
constexpr double ROWS_PRICE[4][9] = {      // by steps ahead and wavefronts: 1, 4; 1, 8; 2, 4; 2, 8
    {0.7038, 0.217, 0.08696, 0.3525, 0.1332, 0.1972, 0.3488, 1.744, 8.075e-08},
    {0.6413, 0.1219, 0.2373, 0.8801, 3.759e-09, 0.2089, 0.458, 1.845, 0.6726},
    {0.4628, 0.2024, 0.123, 0.8821, 0.06831, 0.2003, 0.3304, 1.504, 0.3148},
    {0.1983, 0.1981, 0.09101, 1.083, 6.719e-09, 0.2081, 0.4423, 1.482, 0.3933},
};
constexpr double TILE_PRICE[F8B_SHAPES][8] = {
    {0.8069, 2.116, 0.2367, 0.1964, 0.3056, 1.63, 0.2593, 0.1684},
    {0.7361, 1.904, 0.3832, 0.1829, 0.2016, 2.272, 0.4499, 0.301},
    {0.743, 2.82, 0.5552, 0.1841, 0.2579, 2.002, 0.1814, 0.1479},
    {0.7305, 4.074, 0.8848, 0.2526, 0.09163, 2.121, 0.2139, 0.1661},
    {0.771, 4.56, 0.8191, 0.1713, 0.7118, 1.68, 0.183, 0.07507},
    {0.8033, 5.69, 1.438, 0.1896, 0.57, 2.301, 0.1616, 0.05301},
    {0.7719, 2.926, 0.364, 0.1916, 0.3317, 1.662, 0.1059, 0.1476},
};
constexpr int TILE_ROWS[F8B_SHAPES] = {64, 64, 128, 128, 256, 256, 128}, TILE_COLUMNS[F8B_SHAPES] = {64, 128, 128, 256, 128, 256, 64};
static double cubes(double a, double b, double c = 0) { return cbrt(a * a * a + b * b * b + c * c * c); }

static double rows_us(const F8bRows& r, double M, double N, double K, int cus) {
  const double* const c = ROWS_PRICE[(r.ahead - 1) * 2 + (r.waves == 8)];
  const double blocks = ceil(M / 16 / r.mb), per_cu = ceil(ceil(N / 16 / r.j) * blocks / cus);
  const double slots = fmin(floor(160.0 * 1024 / fp8_block_rows_lds_bytes((int64_t)K, r)), 16 / r.waves), w = r.waves / 4.0;
  const double side = fmin(per_cu, slots) * w, rounds = fmax(per_cu / slots, 1.0);
  const double step = cubes(c[0], c[1] * side * (r.mb + r.j), c[2] * side * r.mb * r.j);
  const double core = rounds * (c[3] + ceil(ceil(K / 256) / r.waves) * step + c[4] * r.mb * r.j * w);
  return c[7] + cubes(core, c[5] * 1e-6 * K * N * (1 + c[6] * (blocks - 1))) + c[8] * 1e-6 * M * N;
}
static double tile_us(int shape, double M, double N, double K, int cus) {
  const double* const c = TILE_PRICE[shape];
  const double down = ceil(M / TILE_ROWS[shape]), across = ceil(N / TILE_COLUMNS[shape]);
  const double full = floor(down * across / cus), rest = down * across / cus - full;
  const double rounds = full + (rest > 0 ? c[0] + (1 - c[0]) * rest : 0);
  const double core = rounds * (c[1] + ceil(K / F8B) * c[2] * (1 + c[7] / down));
  return c[5] + cubes(core, c[3] * 1e-6 * K * N * (1 + c[4] * (down - 1))) + c[6] * 1e-6 * M * N;
}

struct F8bPlan {
  F8bRows rows;      // mb = 0: tiles
  int shape = 0;
  double us = -1;
};
// Plans for few rows have at most eight blocks of rows, so at most 512 rows: none of more was timed.  (At 385 .. 512 rows they are the fastest of 25 problems in 182.)
constexpr int ROW_BLOCKS = 8;
static F8bPlan cheapest(int64_t M, int64_t N, int64_t K, int cus) {
  F8bPlan best;
  auto offer = [&](const F8bRows& r, int shape, double us) {
    if (best.us >= 0 && best.us <= us) return;
    best.rows = r;
    best.shape = shape;
    best.us = us;
  };
  for (int shape = 0; shape < F8B_SHAPES; ++shape) offer(F8bRows{}, shape, tile_us(shape, (double)M, (double)N, (double)K, cus));
  for (int mb = 1; mb <= 4 && (mb == 1 || M > 16 * (mb - 1)); ++mb) {
    if (M > ROW_BLOCKS * 16 * mb) continue;
    for (int j = 1; j <= 4; j *= 2)
      for (int ahead = 1; ahead <= 2; ++ahead)
        for (int waves = 4; waves <= 8; waves += 4)
          if (const F8bRows r{mb, j, ahead, waves}; fp8_block_rows_fits(K, r)) offer(r, 0, rows_us(r, (double)M, (double)N, (double)K, cus));
  }
  return best;
}
// Plans of recent problems, by size (a search costs 3 us).  Direct mapped, one table per thread.
static const F8bPlan& plan_of(int64_t M, int64_t N, int64_t K) {
  struct Entry {
    int64_t M = -1, N = 0, K = 0;
    int cus = 0;
    F8bPlan plan;
  };
  static thread_local Entry table[256];
  const int cus = num_cus_current_device();
  const uint64_t h = (uint64_t)M * 0x9e3779b97f4a7c15ull ^ (uint64_t)N * 0xc2b2ae3d27d4eb4full ^ (uint64_t)K * 0x165667b19e3779f9ull;
  Entry& e = table[h >> 56];
  if (e.M != M || e.N != N || e.K != K || e.cus != cus) {
    e.M = -1;
    e.plan = cheapest(M, N, K, cus);
    e.N = N; e.K = K; e.cus = cus; e.M = M;
  }
  return e.plan;
}

static int block_scaled_mm(const Fp8BlockParams& p, bool bf16, hipStream_t s) {
  const VaqTuning& t = tuning();
  F8bPlan plan = plan_of(p.M, p.N, p.K);
  if (t.fp8_path == 1) {
    plan.rows = F8bRows{t.exp[11] >> 4 & 15, t.exp[11] & 15, t.exp[11] >> 8 & 15, t.exp[11] >> 12};
    VAQ_CHECK_SUPPORTED(fp8_block_rows_fits(p.K, plan.rows), "fp8_block_scaled_mm: no such plan for few rows");
  } else if (t.fp8_path == 2) {
    plan.rows = F8bRows{};
    plan.shape = t.fp8_tile_cfg - 1;
    VAQ_CHECK_SUPPORTED(plan.shape >= 0 && plan.shape < F8B_SHAPES, "fp8_block_scaled_mm: no such tile shape");
  }
  const int64_t units = plan.rows.mb > 0 ? (p.M + 16 * (int64_t)plan.rows.mb - 1) / (16 * plan.rows.mb) * ((p.N + 16 * (int64_t)plan.rows.j - 1) / (16 * plan.rows.j))
                                         : (p.M + (int64_t)TILE_ROWS[plan.shape] - 1) / TILE_ROWS[plan.shape] *
                                               ((p.N + (int64_t)TILE_COLUMNS[plan.shape] - 1) / TILE_COLUMNS[plan.shape]);
  VAQ_CHECK_SUPPORTED(units < (1 << 23) - 8, "fp8_block_scaled_mm: M = %d, N = %d need more than a launch's 2^32 threads", p.M, p.N);      // (512 each)
  if (plan.rows.mb > 0) {
    if (!fp8_block_rows_launch(p, bf16, plan.rows, s)) return VAQ_ERR_LAUNCH;
  } else if (const int rc = fp8_block_tile_launch(p, bf16, plan.shape, s); rc != VAQ_OK) {
    return rc;
  }
  VAQ_CHECK_LAUNCH("fp8_block_scaled_mm");
  return VAQ_OK;
}

}  // namespace vaq

using namespace vaq;

extern "C" int vaq_fp8_block_scaled_mm_tuned(const uint8_t* a, int64_t lda, const uint8_t* b, int64_t ldb, const float* sa, int64_t sa_row_stride,
                                             int64_t sa_block_stride, const float* sb, int64_t sb_k_stride, int64_t sb_n_stride, const void* bias, void* out,
                                             int64_t ldc, int out_dtype, int64_t size_m, int64_t size_n, int64_t size_k, void* stream, const VaqTuning* tuning) {
  VAQ_CHECK_ARG(out_dtype == VAQ_F16 || out_dtype == VAQ_BF16, "fp8_block_scaled_mm: out_dtype = %d", out_dtype);
  VAQ_CHECK_ARG(size_m >= 0 && size_n > 0 && size_k > 0 && size_m < (1ll << 31) && size_n < (1ll << 31) && size_k < (1ll << 31),
                "fp8_block_scaled_mm: M = %lld, N = %lld, K = %lld", (long long)size_m, (long long)size_n, (long long)size_k);
  VAQ_CHECK_ARG(size_k % 16 == 0 && size_n % 16 == 0, "fp8_block_scaled_mm: K = %lld and N = %lld must be multiples of 16", (long long)size_k, (long long)size_n);
  if (size_m == 0) return VAQ_OK;
  VAQ_CHECK_ARG(a && b && sa && sb && out, "fp8_block_scaled_mm: null pointer");
  VAQ_CHECK_ARG((((uintptr_t)a | (uintptr_t)b) & 15) == 0 && ((uintptr_t)out & 7) == 0 && (((uintptr_t)sa | (uintptr_t)sb) & 3) == 0 && ((uintptr_t)bias & 1) == 0,
                "fp8_block_scaled_mm: a and b must be aligned to 16 bytes, out to 8, scales to 4");
  if (size_m == 1) {      // (the strides of a single row say nothing)
    lda = size_k;
    ldc = size_n;
    sa_row_stride = 0;
  }
  VAQ_CHECK_ARG(lda % 16 == 0 && ldb % 16 == 0 && ldc % 4 == 0 && lda >= size_k && ldb >= size_k && ldc >= size_n,
                "fp8_block_scaled_mm: row strides lda = %lld, ldb = %lld (multiples of 16, at least K), ldc = %lld (a multiple of 4, at least N)", (long long)lda,
                (long long)ldb, (long long)ldc);
  const int64_t blocks = (size_k + F8B - 1) / F8B, limit = (int64_t)1 << 31;
  if (blocks == 1) sa_block_stride = sb_k_stride = 0;
  // (a tile is at most 256 rows of each operand: their offsets fit in 31 bits)
  VAQ_CHECK_SUPPORTED(lda <= (1 << 22) && ldb <= (1 << 22), "fp8_block_scaled_mm: rows more than 4 MiB apart are not built (lda = %lld, ldb = %lld)", (long long)lda,
                      (long long)ldb);
  VAQ_CHECK_ARG(sa_row_stride >= 0 && sa_block_stride >= 0 && sb_k_stride >= 0 && sb_n_stride >= 0, "fp8_block_scaled_mm: negative stride of the scales");
  VAQ_CHECK_SUPPORTED(sa_row_stride <= (1 << 20) && sa_block_stride < limit && sb_k_stride < limit && (256 * sa_row_stride + blocks * sa_block_stride) * 4 < limit &&
                          blocks * sb_k_stride * 4 < limit,
                      "fp8_block_scaled_mm: scales of 256 rows or of a block of columns lie more than 2 GiB apart");
  VAQ_CHECK_SUPPORTED(size_k <= 131072, "fp8_block_scaled_mm: K = %lld, at most 131072 is built", (long long)size_k);      // (the scales of a block of columns are in LDS)
  const Fp8BlockParams p{a, b, sa, sb, (const uint16_t*)bias, (uint16_t*)out, sa_row_stride, sb_n_stride, (uint32_t)sa_block_stride, (uint32_t)sb_k_stride,
                         (uint32_t)lda, (uint32_t)ldb, ldc, (int)size_m, (int)size_n, (int)size_k};
  TuningScope scope(tuning);
  return block_scaled_mm(p, out_dtype == VAQ_BF16, (hipStream_t)stream);
}

extern "C" int vaq_fp8_block_scaled_mm(const uint8_t* a, int64_t lda, const uint8_t* b, int64_t ldb, const float* sa, int64_t sa_row_stride,
                                       int64_t sa_block_stride, const float* sb, int64_t sb_k_stride, int64_t sb_n_stride, const void* bias, void* out,
                                       int64_t ldc, int out_dtype, int64_t size_m, int64_t size_n, int64_t size_k, void* stream) {
  return vaq_fp8_block_scaled_mm_tuned(a, lda, b, ldb, sa, sa_row_stride, sa_block_stride, sb, sb_k_stride, sb_n_stride, bias, out, ldc, out_dtype, size_m,
                                       size_n, size_k, stream, nullptr);
}

extern "C" int vaq_fp8_block_plan(int64_t size_m, int64_t size_n, int64_t size_k, double* plan) {
  VAQ_CHECK_ARG(plan && size_m > 0 && size_n > 0 && size_k > 0, "fp8_block_plan: no problem");
  const F8bPlan p = cheapest(size_m, size_n, size_k, num_cus_current_device());
  const double out[6] = {(double)p.rows.mb, (double)p.rows.j, (double)p.rows.ahead, (double)p.rows.waves, (double)p.shape, p.us};
  for (int i = 0; i < 6; ++i) plan[i] = out[i];
  return VAQ_OK;
}
