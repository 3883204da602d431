// Launch of the block-scaled FP8 product's kernel for few rows (fp8_block_rows_kernel.h).
#include "fp8_block_rows_kernel.h"

namespace vaq {

bool fp8_block_rows_fits(int64_t K, int mb, int j) { return f8br_built(mb, j) && f8br_lds_bytes(K, mb, j) <= 160 * 1024; }

template <bool BF16, int MB, int J, bool TAIL>
static bool launch(const Fp8BlockParams& p, hipStream_t s) {
  const uint32_t ranges = ((uint32_t)p.N + 16 * J - 1) / (16 * J), row_blocks = ((uint32_t)p.M + MB * 16 - 1) / (MB * 16);
  const size_t lds = f8br_lds_bytes(p.K, MB, J);
  auto kern = fp8_block_rows_kernel<BF16, MB, J, TAIL>;
  static size_t reserved[VAQ_MAX_DEVICES];
  if (reserve_dynamic_lds(reinterpret_cast<const void*>(kern), lds, reserved, "fp8_block_scaled_mm") != VAQ_OK) return false;
  hipLaunchKernelGGL(kern, dim3((ranges * row_blocks + 7) / 8 * 8), dim3(F8BR_WAVES * 64), lds, s, p, ranges, row_blocks);
  return true;
}

template <bool BF16, int MB, int J>
static bool launch(const Fp8BlockParams& p, hipStream_t s) {
  if constexpr (!f8br_built(MB, J)) return false;
  else return p.K % F8BR_STEP != 0 ? launch<BF16, MB, J, true>(p, s) : launch<BF16, MB, J, false>(p, s);
}

template <bool BF16, int MB>
static bool launch_mb(const Fp8BlockParams& p, int j, hipStream_t s) {
  return j == 1 ? launch<BF16, MB, 1>(p, s) : j == 2 ? launch<BF16, MB, 2>(p, s) : j == 4 ? launch<BF16, MB, 4>(p, s) : false;
}

template <bool BF16>
static bool launch_type(const Fp8BlockParams& p, int mb, int j, hipStream_t s) {
  return mb == 1 ? launch_mb<BF16, 1>(p, j, s) : mb == 2 ? launch_mb<BF16, 2>(p, j, s) : mb == 3 ? launch_mb<BF16, 3>(p, j, s) : mb == 4 ? launch_mb<BF16, 4>(p, j, s) : false;
}

bool fp8_block_rows_launch(const Fp8BlockParams& p, bool bf16, int mb, int j, hipStream_t s) {
  if (!fp8_block_rows_fits(p.K, mb, j)) return false;
  return bf16 ? launch_type<true>(p, mb, j, s) : launch_type<false>(p, mb, j, s);
}

}  // namespace vaq
