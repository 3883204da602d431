// Launch of the block-scaled FP8 product's kernel for few rows (fp8_block_rows_kernel.h).
#include "fp8_block_rows_kernel.h"

namespace vaq {

size_t fp8_block_rows_lds_bytes(int64_t K, const F8bRows& r) { return f8br_lds_bytes(K, r.mb, r.j, r.ahead, r.waves); }
bool fp8_block_rows_fits(int64_t K, const F8bRows& r) { return f8br_built(r.mb, r.j, r.ahead, r.waves) && f8br_lds_bytes(K, r.mb, r.j, r.ahead, r.waves) <= 160 * 1024; }

template <bool BF16, int MB, int J, int AHEAD, int NW, bool TAIL>
static bool launch(const Fp8BlockParams& p, hipStream_t s) {
  const uint32_t ranges = ((uint32_t)p.N + 16 * J - 1) / (16 * J), row_blocks = ((uint32_t)p.M + MB * 16 - 1) / (MB * 16);
  const size_t lds = f8br_lds_bytes(p.K, MB, J, AHEAD, NW);
  auto kern = fp8_block_rows_kernel<BF16, MB, J, AHEAD, NW, TAIL>;
  static size_t reserved[VAQ_MAX_DEVICES];
  if (reserve_dynamic_lds(reinterpret_cast<const void*>(kern), lds, reserved, "fp8_block_scaled_mm") != VAQ_OK) return false;
  hipLaunchKernelGGL(kern, dim3((ranges * row_blocks + 7) / 8 * 8), dim3(NW * 64), lds, s,
                     v8u{ptr_lo(p.b), ptr_hi(p.b), p.ldb, (uint32_t)p.K, (uint32_t)p.N, (uint32_t)p.M, ranges, row_blocks}, p);
  return true;
}

template <int MB, int J, int AHEAD, int NW>
static bool launch_plan(const Fp8BlockParams& p, bool bf16, hipStream_t s) {
  if constexpr (!f8br_built(MB, J, AHEAD, NW)) {
    return false;
  } else {
    const bool tail = p.K % F8BR_STEP != 0;
    if (bf16) return tail ? launch<true, MB, J, AHEAD, NW, true>(p, s) : launch<true, MB, J, AHEAD, NW, false>(p, s);
    return tail ? launch<false, MB, J, AHEAD, NW, true>(p, s) : launch<false, MB, J, AHEAD, NW, false>(p, s);
  }
}
template <int MB, int AHEAD, int NW>
static bool launch_j(const Fp8BlockParams& p, bool bf16, int j, hipStream_t s) {
  return j == 1 ? launch_plan<MB, 1, AHEAD, NW>(p, bf16, s) : j == 2 ? launch_plan<MB, 2, AHEAD, NW>(p, bf16, s) : launch_plan<MB, 4, AHEAD, NW>(p, bf16, s);
}
template <int AHEAD, int NW>
static bool launch_mb(const Fp8BlockParams& p, bool bf16, int mb, int j, hipStream_t s) {
  return mb == 1 ? launch_j<1, AHEAD, NW>(p, bf16, j, s) : mb == 2 ? launch_j<2, AHEAD, NW>(p, bf16, j, s) : mb == 3 ? launch_j<3, AHEAD, NW>(p, bf16, j, s) : launch_j<4, AHEAD, NW>(p, bf16, j, s);
}

bool fp8_block_rows_launch(const Fp8BlockParams& p, bool bf16, const F8bRows& r, hipStream_t s) {
  if (!fp8_block_rows_fits(p.K, r)) return false;
  if (r.waves == 8) return r.ahead == 1 ? launch_mb<1, 8>(p, bf16, r.mb, r.j, s) : launch_mb<2, 8>(p, bf16, r.mb, r.j, s);
  return r.ahead == 1 ? launch_mb<1, 4>(p, bf16, r.mb, r.j, s) : launch_mb<2, 4>(p, bf16, r.mb, r.j, s);
}

}  // namespace vaq
