// FP8 product with a scale for each block of 128 (fp8_block_mm.h): arguments, choice of the kernel, launch of the tiles.
#include "fp8_block_tile_kernel.h"

namespace vaq {

template <int BM, int BN, int WAVES, typename Kernel>
static int launch_tiles(const Fp8BlockParams& p, size_t lds, Kernel kern, size_t (&reserved)[VAQ_MAX_DEVICES], hipStream_t s) {
  const uint32_t tiles_m = ((uint32_t)p.M + BM - 1) / BM, tiles_n = ((uint32_t)p.N + BN - 1) / BN;
  if (const int rc = reserve_dynamic_lds(reinterpret_cast<const void*>(kern), lds, reserved, "fp8_block_scaled_mm"); rc != VAQ_OK) return rc;
  hipLaunchKernelGGL(kern, dim3((tiles_m * tiles_n + 7) / 8 * 8), dim3(WAVES * 64), lds, s, p, tiles_m, tiles_n);
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
    default: return launch_256<BF16>(p, s);
  }
}
int fp8_block_tile_launch(const Fp8BlockParams& p, bool bf16, int shape, hipStream_t s) {
  return bf16 ? launch_type<true>(p, shape, s) : launch_type<false>(p, shape, s);
}

// The kernel of a problem.
struct F8bPlan {
  F8bRows rows;      // mb = 0: tiles
  int shape = 0;
};
static F8bPlan plan_of(int64_t M, int64_t N, int64_t K, bool rows_ok) {
  F8bPlan plan;
  const int cus = num_cus_current_device();
  if (rows_ok && M <= 64) {
    const int mb = (int)((M + 15) / 16);
    // as many n-tiles a workgroup as leave every compute unit one
    for (int j = 4; j >= 1; j /= 2)
      if (const F8bRows r{mb, j, 2, 4}; fp8_block_rows_fits(K, r) && (j == 1 || (N + 16 * j - 1) / (16 * j) >= cus)) {
        plan.rows = r;
        return plan;
      }
  }
  auto tiles = [&](int64_t bm, int64_t bn) { return ((M + bm - 1) / bm) * ((N + bn - 1) / bn); };
  plan.shape = tiles(256, 256) >= cus ? 5 : tiles(128, 256) >= cus ? 3 : tiles(128, 128) >= cus / 2 ? 2 : tiles(64, 128) >= cus / 2 ? 1 : 0;
  return plan;
}

static int block_scaled_mm(const Fp8BlockParams& p, bool bf16, hipStream_t s) {
  const VaqTuning& t = tuning();
  // the kernel for few rows counts its scales' offsets from the first row on, in 31 bits
  const int64_t blocks = (p.K + F8B - 1) / F8B;
  const bool rows_ok = (64 * p.sa_row + blocks * p.sa_block) * 4 < ((int64_t)1 << 31);
  F8bPlan plan = plan_of(p.M, p.N, p.K, rows_ok);
  if (t.fp8_path == 1) {
    plan.rows = F8bRows{t.exp[11] >> 4 & 15, t.exp[11] & 15, t.exp[11] >> 8 & 15, t.exp[11] >> 12};
    VAQ_CHECK_SUPPORTED(rows_ok && fp8_block_rows_fits(p.K, plan.rows), "fp8_block_scaled_mm: no such plan for few rows");
  } else if (t.fp8_path == 2) {
    plan.rows = F8bRows{};
    plan.shape = t.fp8_tile_cfg - 1;
    VAQ_CHECK_SUPPORTED(plan.shape >= 0 && plan.shape < F8B_SHAPES, "fp8_block_scaled_mm: no such tile shape");
  }
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
  VAQ_CHECK_ARG(lda % 16 == 0 && ldb % 16 == 0 && ldc % 4 == 0 && lda >= size_k && ldb >= size_k && ldc >= size_n,
                "fp8_block_scaled_mm: row strides lda = %lld, ldb = %lld (multiples of 16, at least K), ldc = %lld (a multiple of 4, at least N)", (long long)lda,
                (long long)ldb, (long long)ldc);
  const int64_t blocks = (size_k + F8B - 1) / F8B, limit = (int64_t)1 << 31;
  // (a tile is at most 256 rows of each operand: their offsets fit in 31 bits)
  VAQ_CHECK_SUPPORTED(lda <= (1 << 22) && ldb <= (1 << 22), "fp8_block_scaled_mm: rows more than 4 MiB apart are not built (lda = %lld, ldb = %lld)", (long long)lda,
                      (long long)ldb);
  VAQ_CHECK_ARG(sa_row_stride >= 0 && sa_block_stride >= 0 && sb_k_stride >= 0 && sb_n_stride >= 0, "fp8_block_scaled_mm: negative stride of the scales");
  VAQ_CHECK_SUPPORTED(sa_row_stride <= (1 << 20) && sa_block_stride < limit && sb_k_stride < limit && (256 * sa_row_stride + blocks * sa_block_stride) * 4 < limit &&
                          blocks * sb_k_stride * 4 < limit,
                      "fp8_block_scaled_mm: scales of 256 rows or of a block of columns lie more than 2 GiB apart");
  VAQ_CHECK_SUPPORTED(size_k <= 131072, "fp8_block_scaled_mm: K = %lld, at most 131072 is built", (long long)size_k);      // (the scales of a block of columns are in LDS)
  const int64_t most = (int64_t)1 << 31;
  VAQ_CHECK_SUPPORTED(((size_m + 15) / 16) * ((size_n + 15) / 16) < most, "fp8_block_scaled_mm: M = %lld, N = %lld", (long long)size_m, (long long)size_n);
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
