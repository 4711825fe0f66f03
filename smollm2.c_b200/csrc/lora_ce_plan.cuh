// lora_ce_plan.cuh — host-side planning that the translation units of the
// LoRA head share: tensor maps, the rank a step runs at, how its rank term
// joins the MMA, and how tiles split over the resident CTAs.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <type_traits>

#include "lora_ce_kernels.cuh"

namespace {

using namespace lce;

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                  const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  if (!fn) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(p);
  }
  return fn;
}

// [rows][d] f16 row-major, read in boxes of 64 x box_rows with 128 B swizzle.
inline bool make_map(CUtensorMap* m, const void* base, long long rows, int d, int box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  cuuint64_t dims[2] = {(cuuint64_t)d, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)d * 2};
  cuuint32_t box[2] = {(cuuint32_t)kBK, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(base), dims, strides, box,
            estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) ==
         CUDA_SUCCESS;
}

// [rows][width] f16 with a row stride of ld elements (ld % 8 == 0), read in
// boxes of 64 x box_rows with 128 B swizzle; columns past width read as 0.
inline bool make_map_ld(CUtensorMap* m, const void* base, long long rows, long long width, long long ld,
                 int box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  cuuint64_t dims[2] = {(cuuint64_t)width, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
  cuuint32_t box[2] = {(cuuint32_t)kBK, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(base), dims, strides, box,
            estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) ==
         CUDA_SUCCESS;
}

inline long long round_up(long long x, long long m) { return (x + m - 1) / m * m; }

// Largest number of CTA segments any resident tile's run of n_b tiles is
// split into, for n_a x n_b tiles over G CTAs.
inline int max_segments(int n_a, int n_b, int G) {
  const long long total = (long long)n_a * n_b;
  int best = 1;
  for (int a = 0; a < n_a; ++a) {
    const int s0 = tile_owner((long long)a * n_b, total, G);
    const int s1 = tile_owner((long long)a * n_b + n_b - 1, total, G);
    if (s1 - s0 + 1 > best) best = s1 - s0 + 1;
  }
  return best;
}

// The rank the kernels run at: the adapter's rank rounded up.
inline int kernel_rank(int r) {
  return r <= 4 ? 4 : r <= 8 ? 8 : r <= 16 ? 16 : r <= 32 ? 32 : r <= 64 ? 64 : r <= 128 ? 128 : 256;
}

// Largest rank of the fused passes; ranks above it take the wide-rank path.
constexpr int kMaxFusedRank = 64;
constexpr int kMaxRank = 256;  // LORA_MAX_RANK (src/train.c:20)

// The same decisions at run time, for sizing a handle's buffers.
inline int aug_width_of(int R) {
  if (R < LCE_AUG_MIN_RANK) return 0;
  return R <= 16 ? 64 : (2 * R + 63) / 64 * 64;
}

// Everything a kernel rank decides.  Ranks up to 16 run each pass once;
// ranks 32 and 64 run each pass once per chunk of 16 ranks (the epilogue's
// accumulators for 16 ranks are what fits in registers), with the full-rank
// logit term in the MMA either way.
//   augmentation layout 0: none (rank 4: the term is epilogue FMAs)
//   layout 1: one 64-wide block, [sU_hi | sU_hi | sU_lo] . [B_hi | B_lo | B_hi]
//   layout 2: [sU_hi | sU_lo] . [B_hi | B_lo], 2R columns, K-steps pairing
//             hi.hi, hi.lo and lo.hi slices
template <int R>
struct RankPlan {
  static constexpr bool kChunked = R > 16;
  static constexpr int kRC = kChunked ? 16 : R;  // ranks per pass
  using EL = std::conditional_t<kChunked, EpiLse<16, true, true>, EpiLse<R>>;
  using EG = std::conditional_t<kChunked, EpiGrad<16, true, true>, EpiGrad<R>>;
  static constexpr bool kAug = EL::kAug;
  static constexpr int kLayout = !kAug ? 0 : kChunked ? 2 : 1;
  static constexpr int kAugWidth = kLayout == 2 ? (2 * R + 63) / 64 * 64 : kLayout == 1 ? 64 : 0;
  static constexpr int kAugBlocks = kAugWidth / 64;
  static_assert(EG::kAug == kAug, "both passes augment the rank term or neither");
  static void schedule(GemmArgs& g) {
    g.n_aug = 0;
    if constexpr (kLayout == 1) {
      for (int s = 0; s < (3 * R + 15) / 16; ++s) {
        g.aug_a[g.n_aug] = (uint8_t)s;
        g.aug_b[g.n_aug++] = (uint8_t)s;
      }
    } else if constexpr (kLayout == 2) {
      constexpr int q = R / 16;
      for (int k = 0; k < q; ++k) {
        const uint8_t pa[3] = {(uint8_t)k, (uint8_t)k, (uint8_t)(q + k)};
        const uint8_t pb[3] = {(uint8_t)k, (uint8_t)(q + k), (uint8_t)k};
        for (int m = 0; m < 3; ++m) {
          g.aug_a[g.n_aug] = pa[m];
          g.aug_b[g.n_aug++] = pb[m];
        }
      }
    }
  }
};

}  // namespace
