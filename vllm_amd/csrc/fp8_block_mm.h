// FP8 product with a scale for each block of 128: what its kernels share.
//     out[m, n] = round( sum over blocks kb of K of  sa[m, kb] * sb[kb, n / 128] * (sum over k in kb of a[m, k] b[k, n])  + bias[n] )
// a is [M, K] row-major, b is [K, N] column-major (= weight [N, K] row-major); the last blocks of K and N may be shorter.
//
// A block of K is one v_mfma_f32_16x16x128_f8f6f4 of 16 x 16 results, which starts from zero: the sum over the block is exact up to the instruction's own
// fp32 accumulation, and one fused multiply-add for each result adds it, times both scales, to an fp32 sum over the blocks.  The weights are the instruction's A
// operand: a lane's four results are neighbouring columns of one row of the output, so that they take the same scale.
// A lane's 32 bytes of an operand are chunks q and q + 4 (of 16 bytes, q = lane / 16) of the block, the same in both operands.
#pragma once
#include "vaq_common.h"

namespace vaq {

constexpr int F8B = 128;      // values of K and columns of the weight that share a scale

struct Fp8BlockParams {
  const uint8_t* a;
  const uint8_t* b;
  const float* sa;
  const float* sb;
  const uint16_t* bias;
  uint16_t* out;
  int64_t sa_row, sb_n;          // elements from row to row of `sa`, from block to block of N in `sb`
  uint32_t sa_block, sb_block;   // from block to block of K
  uint32_t lda, ldb;
  int64_t ldc;
  int M, N, K;
};

__device__ inline v4f mfma_fp8_block(v8i a, v8i b) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, v4f{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
}
__device__ inline __amdgpu_buffer_rsrc_t f8b_rsrc(const void* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, (int)bytes, 0x00020000);
}
constexpr uint32_t F8B_NOWHERE = 0x80000000u;      // an offset past every operand: arrives as zeros

// few rows (fp8_block_rows_kernel.h): blocks of 16 rows and n-tiles of a workgroup, steps that weights are ahead, wavefronts.  false: not built, or no room in LDS
struct F8bRows {
  int mb = 0, j = 0, ahead = 0, waves = 0;
};
size_t fp8_block_rows_lds_bytes(int64_t K, const F8bRows& r);
bool fp8_block_rows_fits(int64_t K, const F8bRows& r);
bool fp8_block_rows_launch(const Fp8BlockParams& p, bool bf16, const F8bRows& r, hipStream_t s);
// tiles (fp8_block_tile_kernel.h)
constexpr int F8B_SHAPES = 7;
int fp8_block_tile_launch(const Fp8BlockParams& p, bool bf16, int shape, hipStream_t s);

}  // namespace vaq
