// lora_head.cu — host side of the operators declared in include/lora_head.h:
// argument checks, workspace layout and the launch sequences.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <map>
#include <mutex>
#include <string>
#include <tuple>

#include "lora_ce_kernels.cuh"
#include "lora_ce_plan.cuh"
#include "lora_ce_tc.cuh"
#include "lora_head.cuh"
#include "lora_head.h"
#include "lora_head_core.h"

using namespace lce;

namespace {

thread_local std::string g_head_error;

int hfail(int code, const char* msg) {
  g_head_error = msg;
  return code;
}

// A C entry's body: no exception leaves it, and a failed call leaves no CUDA error
// behind for the caller's next check.
template <class F>
int entry(F&& body) {
  int rc = LORA_CE_ENOMEM;
  try {
    rc = body();
  } catch (...) {
    g_head_error.clear();
  }
  if (rc) cudaGetLastError();
  return rc;
}

// How the rank term joins the MMA: one K-block up to rank 16, 2R columns above; not
// at all up to rank 4, where the epilogues add it in f32.
// Its operands are only as wide as they are used (a multiple of 16 bytes); the
// loads fill the rest of a 64-column block with zeros.
struct Aug {
  int R = 0, layout = 0, width = 0;
};
Aug aug_of(int r) {
  Aug a;
  if (r == 0) return a;
  a.R = kernel_rank(r);
  if (a.R == 4) return a;
  a.layout = a.R <= 16 ? 1 : 2;
  a.width = a.R <= 16 ? (3 * a.R + 7) / 8 * 8 : 2 * a.R;
  return a;
}
void aug_schedule(GemmArgs& g, const Aug& a) {
  switch (a.R) {
    case 8: RankPlan<8>::schedule(g); break;
    case 16: RankPlan<16>::schedule(g); break;
    case 32: RankPlan<32>::schedule(g); break;
    case 64: RankPlan<64>::schedule(g); break;
    default: g.n_aug = 0;
  }
}

// The share by which the accumulator of a large logit falls short where its partial
// sums grow evenly (lora_head.cuh): partial sums at 1/n, 2/n .. 1 of it over the n K-steps of
// h . W, then at all of it over the rank term's.
double acc_short(int n, int n_aug) {
  return 0.79 * (0.5 * (n + 1) + n_aug) * std::ldexp(1.0, -25) / std::log(2.0);
}

// Co-resident owners (CTA pairs) of a kernel on the current device, found once
// per device, kernel and shared-memory size; also lets the kernel use that
// much shared memory.
int resident_pairs(const void* kern, int threads, int smem) {
  static std::mutex mu;
  static std::map<std::tuple<int, const void*, int>, int> known;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  std::lock_guard<std::mutex> lock(mu);
  const auto key = std::make_tuple(dev, kern, smem);
  const auto it = known.find(key);
  if (it != known.end()) return it->second;
  // the attribute keeps the largest size that any call has asked for
  cudaFuncAttributes fa;
  if (cudaFuncGetAttributes(&fa, kern) != cudaSuccess) return 0;
  if (fa.maxDynamicSharedSizeBytes < smem &&
      cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
    return 0;
  int sms = 0;
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  cudaLaunchConfig_t lc = {};
  lc.gridDim = dim3((unsigned)(sms / 2 * 2));
  lc.blockDim = dim3((unsigned)threads);
  lc.dynamicSmemBytes = (size_t)smem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  lc.attrs = attr;
  lc.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, kern, &lc) != cudaSuccess || n < 1) return 0;
  known[key] = n;
  return n;
}

// Same for kernels without clusters: only the shared-memory attribute.  48 KB need
// none, which a kernel's static arrays (up to 8 KB here) share.
bool allow_smem(const void* kern, size_t smem) {
  if (smem <= 40 * 1024) return true;
  static std::mutex mu;
  static std::map<std::pair<int, const void*>, size_t> known;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  std::lock_guard<std::mutex> lock(mu);
  size_t& have = known[std::make_pair(dev, kern)];
  if (have >= smem) return true;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) !=
      cudaSuccess)
    return false;
  have = smem;
  return true;
}

int sm_count() {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess)
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

// An upper bound on the owners, the same on every call, for sizing partials.
constexpr int kMaxPairs = 80;

// Most slots per row of a pass whose owners are at most kMaxPairs.
int most_segments(int n_a, int n_b) {
  const long long total = (long long)n_a * n_b;
  // an owner's run is at least floor(total / G) tiles, so a row of n_b tiles
  // meets at most n_b / run + 2 owners
  const int G = (int)std::min<long long>(kMaxPairs, total);
  const long long run = total / G;
  return (int)std::min<long long>(G, n_b / run + 2);
}

// Most where, of n_a (or n_b) tiles of positions, as few as a quarter may run
// (active_tiles).
int most_segments_by_a(int n_a, int n_b) {
  return std::max(most_segments(n_a, n_b), most_segments((n_a + 3) / 4, n_b));
}
int most_segments_by_b(int n_a, int n_b) {
  return std::max(most_segments(n_a, n_b), most_segments(n_a, (n_b + 3) / 4));
}

struct Carve {
  uint8_t* base;
  size_t off = 0;
  template <class T>
  T* take(size_t count) {
    const size_t at = off;
    off = (off + count * sizeof(T) + 255) / 256 * 256;
    return base ? reinterpret_cast<T*>(base + at) : nullptr;
  }
};

// A GEMM pass on CTA pairs, all but launched.
struct Pass {
  const void* kern = nullptr;
  int threads = 0, smem = 0, G = 0;
  int n_maps = 0;
  CUtensorMap maps[5];
  GemmArgs g{};
};

// Launch with a programmatic dependency on the kernel ahead (whose end the kernel
// waits for by itself, grid_wait).
bool launch_pass(Pass& p, cudaStream_t st) {
  cudaLaunchConfig_t lc = {};
  lc.gridDim = dim3((unsigned)(2 * p.G));
  lc.blockDim = dim3((unsigned)p.threads);
  lc.dynamicSmemBytes = (size_t)p.smem;
  lc.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  lc.attrs = attr;
  lc.numAttrs = 2;
  void* args[6];
  for (int i = 0; i < p.n_maps; ++i) args[i] = &p.maps[i];
  args[p.n_maps] = &p.g;
  return cudaLaunchKernelExC(&lc, p.kern, args) == cudaSuccess;
}

// A kernel that waits for all that is ahead of it in the stream.
template <class K, class... Args>
bool launch_plain(K kern, int blocks, int threads, size_t smem, cudaStream_t st,
                  const Args&... args) {
  cudaLaunchConfig_t lc = {};
  lc.gridDim = dim3((unsigned)blocks);
  lc.blockDim = dim3((unsigned)threads);
  lc.dynamicSmemBytes = smem;
  lc.stream = st;
  return cudaLaunchKernelEx(&lc, kern, args...) == cudaSuccess;
}

// One that waits by itself (grid_wait).
template <class K, class... Args>
bool launch_after(K kern, int blocks, int threads, size_t smem, cudaStream_t st,
                  const Args&... args) {
  cudaLaunchConfig_t lc = {};
  lc.gridDim = dim3((unsigned)blocks);
  lc.blockDim = dim3((unsigned)threads);
  lc.dynamicSmemBytes = smem;
  lc.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  lc.attrs = attr;
  lc.numAttrs = 1;
  return cudaLaunchKernelEx(&lc, kern, args...) == cudaSuccess;
}

using PassKernel = void (*)(const CUtensorMap, const CUtensorMap, const CUtensorMap,
                            const CUtensorMap, const GemmArgs);

struct PassPlan {
  PassKernel kern = nullptr;
  int threads = 0, smem = 0;
};

// EpiScore with the largest ring that fits beside the resident K-blocks (and, up to
// rank 4, two tiles of staged rows of B).
template <class Epi>
PassPlan plan_of(int kblocks) {
  constexpr bool kStaged = Epi::kRec != 0;
  return PassPlan{lce_gemm_kernel<Epi, kStaged, 2>, block_threads(Epi::kWarps),
                  SmemLayout::bytes(kblocks, Epi::kRec * Epi::kRecBufs, Epi::kRing)};
}
template <int kSub>
PassPlan score_plan(int kblocks, bool r4) {
  if (r4)
    return kblocks <= 9 ? plan_of<EpiScore<65536, kSub, true>>(kblocks)
                        : plan_of<EpiScore<49152, kSub, true>>(kblocks);
  return kblocks <= 10   ? plan_of<EpiScore<65536, kSub, false>>(kblocks)
         : kblocks == 11 ? plan_of<EpiScore<49152, kSub, false>>(kblocks)
                         : plan_of<EpiScore<32768, kSub, false>>(kblocks);
}
PassPlan score_plan(int kblocks, int sub, bool r4) {
  return sub == 64  ? score_plan<64>(kblocks, r4)
         : sub == 8 ? score_plan<8>(kblocks, r4)
         : sub == 1 ? score_plan<1>(kblocks, r4) : score_plan<0>(kblocks, r4);
}

// Columns per record: the widest that leaves four records per alternative.
int record_columns(int V, int top_k) {
  const int want = 4 * std::max(top_k, kMinPick);
  return (V + 63) / 64 >= want ? 64 : (V + 7) / 8 >= want ? 8 : 1;
}

// The passes of ranks 4 and 8 (rank sums in the epilogue): records staged in
// shared memory where they fit.
template <class Epi>
PassPlan sums_plan(int kblocks) {
  PassPlan p;
  p.threads = block_threads(Epi::kWarps);
  p.smem = SmemLayout::bytes(kblocks, Epi::kRec * Epi::kRecBufs, Epi::kRing);
  if (p.smem <= kMaxDynSmem) {
    p.kern = lce_gemm_kernel<Epi, true, 2>;
  } else {
    p.smem = SmemLayout::bytes(kblocks, 0, Epi::kRing);
    p.kern = lce_gemm_kernel<Epi, false, 2>;
  }
  return p;
}

// Tiles, partials and temperature factors of a pass whose resident rows are
// positions.
void fill_pass1(GemmArgs& g, const HeadCore& hd, const Aug& aug, int T, float tau) {
  g.kmain = hd.d / kBK;
  g.kblocks = g.kstr = g.kmain + (aug.width + kBK - 1) / kBK;
  aug_schedule(g, aug);
  g.rank_total = g.R = aug.R;
  g.T = T;
  g.V = hd.V;
  g.Vpad = round_up(hd.V, kBN);
  g.n_a = (T + 2 * kBM - 1) / (2 * kBM);
  g.Tcap = (long long)g.n_a * 2 * kBM;
  const double shortfall = acc_short(4 * g.kmain, g.kblocks > g.kmain ? g.n_aug : 0);
  g.lg = (float)((1.0 + shortfall) / (std::log(2.0) * tau));
  g.lazy = 8.0f * tau;
  g.redo = 80.0f * tau;
}

// lh_prep over positions and vocab rows: a block per position up to two an SM,
// else kTileRows positions per block.
struct PrepPlan {
  void (*kern)(PrepArgs, PackArgs, NormArgs, int, int, int) = nullptr;
  int norm_blocks = 0, prep_blocks = 0, max_blocks = 0, pack_blocks = 0;
  size_t smem = 0;
  bool ok = false;
};
PrepPlan plan_prep(const PrepArgs& pa, const PackArgs& pk, const NormArgs& na, bool rows,
                   int max_blocks, bool pack, int sms) {
  PrepPlan p;
  const bool tiles = pa.Tpad > 2 * sms;
  p.kern = lh_prep<-1>;
  if (tiles) {
    switch (pa.R) {
      case 0: p.kern = lh_prep<0>; break;
      case 4: p.kern = lh_prep<4>; break;
      case 8: p.kern = lh_prep<8>; break;
      case 16: p.kern = lh_prep<16>; break;
      case 32: p.kern = lh_prep<32>; break;
      default: p.kern = lh_prep<64>; break;
    }
  }
  p.norm_blocks = na.out ? kNormBlocks + (na.r ? 1 : 0) : 0;
  p.prep_blocks = !rows ? 0 : tiles ? (pa.Tpad + kTileRows - 1) / kTileRows : pa.Tpad;
  p.max_blocks = max_blocks;
  p.pack_blocks = pack ? (int)(pk.Vpad / kPackRows) : 0;
  p.smem = std::max(!rows ? 0 : tiles ? prep_tile_smem(pa.R, pa.d) : (size_t)(pa.d + 264) * 4,
                    pack ? (size_t)pk.R * (kPackRows + 1) * 4 : 0);
  p.ok = allow_smem(reinterpret_cast<const void*>(p.kern), p.smem);
  return p;
}
bool launch_prep(const PrepPlan& p, const PrepArgs& pa, const PackArgs& pk, const NormArgs& na,
                 cudaStream_t st) {
  return launch_plain(p.kern, p.norm_blocks + p.prep_blocks + p.max_blocks + p.pack_blocks, 256,
                      p.smem, st, pa, pk, na, p.norm_blocks, p.prep_blocks, p.max_blocks);
}

// The pass for few positions, one slot per 128 vocab rows.  Its time grows with
// positions and ranks, that of the tensor-core passes does not.  V = 49152, d = 576,
// whole calls in us, L2 flushed, at 8 / 16 / 24 / 32 positions: scoring (8
// alternatives) rank 4 41 / 41 / 45 / 49 against 53 / 51 / 51 / 49, rank 16 43 / 45 /
// 51 / 55 against 55 / 53 / 53 / 51, rank 64 51 / 57 / 76 / 82 against 70 / 68 / 68 /
// 66; distillation with gradients, at 8 / 16 / 32, rank 4 51 / 55 / 70 against 82,
// rank 16 65 / 72 / 92 against 112, rank 64 123 / 139 / 211 against 172 (its own
// forward and backward passes and no partial gradients, so a higher limit).
// Scoring: where records have 64 columns.
constexpr int kFewMax = 32;
bool few_score(int T, int R, int sub) { return T <= (R <= 16 ? 24 : 16) && sub == 64; }
bool few_distill(int T, int R) { return T <= (R <= 16 ? kFewMax : 16); }
int few_blocks(int V) { return (V + kFewRows - 1) / kFewRows; }

FewArgs few_args(const HeadCore& hd, int R, int T, const __half* h16, const float* sU, float lg) {
  FewArgs f{};
  f.W = hd.W;
  f.h16 = h16;
  f.sU = sU;
  f.B = BView{hd.B, hd.V, hd.r, R, hd.layout};
  f.T = T;
  f.V = hd.V;
  f.d = hd.d;
  f.r = hd.r;
  f.R = R;
  f.lg = lg;
  f.ld = round_up(T, 8);
  return f;
}

struct FewPlan {
  void (*kern)(FewArgs) = nullptr;
  size_t smem = 0;
  bool ok = true;
};
template <int kMode>
FewPlan plan_few(const FewArgs& f) {
  const int nt = (f.T + 7) / 8, NT = nt <= 2 ? nt : 4;
  FewPlan p;
  p.kern = NT == 1 ? lh_few<1, kMode> : NT == 2 ? lh_few<2, kMode> : lh_few<4, kMode>;
  p.smem = few_smem(NT, f.d, f.R);
  p.ok = allow_smem(reinterpret_cast<const void*>(p.kern), p.smem);
  return p;
}
bool launch_few(const FewPlan& p, const FewArgs& f, int blocks, cudaStream_t st) {
  return launch_after(p.kern, blocks, 256, p.smem, st, f);
}

struct ScoreWs {
  int* stats;
  __half *h16, *haug, *waug;
  float *sU, *Bt, *norms, *hn, *p_max, *p_sum, *p_ent, *sub_max, *sub_second, *sub_rest;
  uint8_t *sub_arg, *sub_arg2;
  int sub, n_sub;
  size_t bytes;
};

ScoreWs score_ws(const HeadCore& hd, int T, int top_k, void* ws) {
  const Aug aug = aug_of(hd.r);
  ScoreWs w{};
  Carve c{static_cast<uint8_t*>(ws)};
  const long long Vpad = round_up(hd.V, kBN);
  const int n_a = (T + 2 * kBM - 1) / (2 * kBM), n_b = (int)(Vpad / kBN);
  w.sub = record_columns(hd.V, top_k);
  const bool few = few_score(T, aug.R, w.sub);
  const size_t part = few ? (size_t)few_blocks(hd.V) * kFewMax
                          : (size_t)4 * most_segments(n_a, n_b) * n_a * 2 * kBM;
  w.n_sub = (hd.V + w.sub - 1) / w.sub;
  w.stats = c.take<int>(kStatWords);
  w.h16 = c.take<__half>((size_t)T * hd.d);
  w.sU = c.take<float>((size_t)T * aug.R);
  w.haug = c.take<__half>((size_t)T * aug.width);
  w.waug = c.take<__half>((size_t)Vpad * aug.width);
  w.Bt = c.take<float>(aug.R == 4 && !few && !hd.layout ? (size_t)Vpad * 4 : 0);
  w.norms = c.take<float>(2 * kNormBlocks + 1);
  w.hn = c.take<float>(T);
  w.p_max = c.take<float>(part);
  w.p_sum = c.take<float>(part);
  w.p_ent = c.take<float>(part);
  const size_t recs = (size_t)w.n_sub * round_up(T, 8);
  w.sub_max = c.take<float>(recs);
  w.sub_second = c.take<float>(w.sub == 64 ? recs : 0);
  w.sub_rest = c.take<float>(w.sub > 1 ? recs : 0);
  w.sub_arg = c.take<uint8_t>(w.sub > 1 ? recs : 0);
  w.sub_arg2 = c.take<uint8_t>(w.sub == 64 ? recs : 0);
  w.bytes = c.off;
  return w;
}

struct DistillWs {
  int* stats;
  __half *h16, *haug, *waug, *xv, *xt;
  float *sU, *wt, *p_max, *p_sum, *p_q, *tok, *Bt, *nml, *xs, *dU, *gAp, *gBp;
  float2* ref;
  int* order;
  unsigned* masks;
  unsigned long long* corr;
  size_t zero_bytes;  // stats and corr: cleared by every call
  size_t bytes;
};

DistillWs distill_ws(const HeadCore& hd, int T, bool grads, void* ws) {
  const Aug aug = aug_of(hd.r);
  const int R = aug.R;
  const bool tc = R >= 16;
  DistillWs w{};
  Carve c{static_cast<uint8_t*>(ws)};
  const long long Vpad = round_up(hd.V, kBN), Tpad = round_up(T, kBN);
  const int bn = grads && tc ? tc_bn(R) : kBN;
  const int n_a = (T + 2 * kBM - 1) / (2 * kBM), n_b = (hd.V + bn - 1) / bn;
  const size_t part = (size_t)(grads && tc ? 2 : 4) * most_segments_by_a(n_a, n_b) * n_a * 2 * kBM;
  w.stats = c.take<int>(kStatWords);
  if (grads) w.corr = c.take<unsigned long long>((size_t)Vpad * R);
  w.zero_bytes = c.off;
  w.h16 = c.take<__half>((size_t)T * hd.d);
  w.sU = c.take<float>((size_t)T * R);
  w.wt = c.take<float>(T);
  if (few_distill(T, R)) {
    const size_t slots = (size_t)few_blocks(hd.V) * round_up(T, 8);
    w.p_max = c.take<float>(slots);
    w.p_sum = c.take<float>(slots);
    w.p_q = c.take<float>(grads ? slots * R : 0);
    w.ref = c.take<float2>(T);
    w.dU = c.take<float>((size_t)T * R);
    w.bytes = c.off;
    return w;
  }
  w.order = c.take<int>(T);
  w.masks = c.take<unsigned>((T + 31) / 32);
  w.haug = c.take<__half>((size_t)T * aug.width);
  w.waug = c.take<__half>((size_t)Vpad * aug.width);
  w.p_max = c.take<float>(part);
  w.p_sum = c.take<float>(part);
  if (grads || R == 4) w.Bt = c.take<float>(hd.layout ? 0 : (size_t)Vpad * R);
  if (grads) {
    // chunks of four or eight epilogue columns a row: up to 4 slots per owner
    const int n_a2 = (hd.V + 2 * kBM - 1) / (2 * kBM), n_b2 = (T + bn - 1) / bn;
    const size_t segs = (size_t)(tc ? 1 : 4) * most_segments_by_b(n_a2, n_b2);
    w.p_q = c.take<float>(part * R);
    w.tok = c.take<float>(tc ? 0 : (size_t)Tpad * tok_stride(R));
    w.xv = c.take<__half>(tc ? (size_t)2 * R * Vpad : 0);
    w.xt = c.take<__half>(tc ? (size_t)2 * R * Tpad : 0);
    w.nml = c.take<float>(tc ? (size_t)Tpad + kMaxBNT : 0);
    w.xs = c.take<float>(tc ? T : 0);
    w.dU = c.take<float>((size_t)T * R);
    w.gAp = c.take<float>((size_t)((T + kDAChunk - 1) / kDAChunk) * hd.d * R);
    w.gBp = c.take<float>(segs * Vpad * R);
  }
  w.bytes = c.off;
  return w;
}

LogitArgs logit_args(const HeadCore& hd, const Aug& aug, int T, const __half* h16,
                     const float* sU, const __half* haug, const __half* waug) {
  LogitArgs z{};
  z.W = hd.W;
  z.h16 = h16;
  z.sU = sU;
  z.haug = haug;
  z.waug = aug.width ? waug : nullptr;
  z.aug_layout = aug.layout;
  z.aug_width = aug.width;
  z.A = hd.A;
  z.lda = hd.lda;
  z.scale = hd.scale;
  z.B = BView{hd.B, hd.V, hd.r, aug.R, hd.layout};
  z.T = T;
  z.V = hd.V;
  z.d = hd.d;
  z.r = hd.r;
  z.R = aug.R;
  return z;
}

PrepArgs prep_args(const HeadCore& hd, const Aug& aug, const void* H, int dtype, int T) {
  PrepArgs p{};
  p.H = H;
  p.dtype = dtype;
  p.T = p.Tpad = T;
  p.d = hd.d;
  p.A = hd.A;
  p.lda = hd.lda;
  p.r = hd.r;
  p.R = aug.R;
  p.scale = hd.scale;
  p.aug_layout = aug.layout;
  p.aug_width = aug.width;
  return p;
}

// The passes of one call.
struct Step {
  const HeadCore& hd;
  const __half *h16, *haug, *waug;
  Aug aug;
  int T, sms;
  GemmArgs g;      // pass 1's, filled
  const DistillWs* w;
  Pass one, two;   // out
  SlotPlan slots;  // out: pass 1's partials
  int cparts2 = 0, n_b2 = 0, bn2 = 0, G2 = 0;
};

constexpr const char* kNoMap = "cuTensorMapEncodeTiled failed";
constexpr const char* kNoFit = "a GEMM pass cannot be made resident on this device";
constexpr const char* kNoLaunch = "kernel launch failed";

int pair_units(const Pass& p) {
  return std::min(kMaxPairs, resident_pairs(p.kern, p.threads, p.smem));
}

// Positions as rows of both operands' maps [h, W] or [W, h], and the rank term's.
int operand_maps(const Step& s, bool aug, bool w_first, int box_a, int box_b, Pass& p,
                 const char** why) {
  const int d = s.hd.d, aw = s.aug.width, V = s.hd.V, T = s.T;
  CUtensorMap* m = p.maps;
  const int h = w_first ? 1 : 0, w = 1 - h;
  const int box_h = w_first ? box_b : box_a, box_w = w_first ? box_a : box_b;
  bool ok = make_map(&m[h], s.h16, T, d, box_h) && make_map(&m[w], s.hd.W, V, d, box_w);
  if (ok && aug)
    ok = make_map(&m[2 + h], s.haug, T, aw, box_h) && make_map(&m[2 + w], s.waug, V, aw, box_w);
  if (!ok) return *why = kNoMap, LORA_CE_ECUDA;
  if (!aug) {
    m[2] = m[0];
    m[3] = m[1];
  }
  p.n_maps = 4;
  return 0;
}

// Pass 1 of a kernel that lce_gemm_kernel makes of an epilogue.
int rows_pass(Step& s, const PassPlan& plan, bool aug, int cparts, float* p_ent, float* p_q,
              const char** why) {
  Pass& p = s.one;
  p.kern = reinterpret_cast<const void*>(plan.kern);
  p.threads = plan.threads;
  p.smem = plan.smem;
  if (int rc = operand_maps(s, aug, false, kBM, kBM, p, why)) return rc;
  const int units = pair_units(p);
  if (units < 1) return *why = kNoFit, LORA_CE_ECUDA;
  s.g.n_b = (int)(s.g.Vpad / kBN);
  p.G = (int)std::min<long long>(units, (long long)s.g.n_a * s.g.n_b);
  p.g = s.g;
  s.slots = SlotPlan{cparts, s.g.n_a, s.g.n_b, units, s.g.Tcap, s.g.p_max, s.g.p_sum, p_ent, p_q};
  return 0;
}

template <class Epi>
int sums_pass2(Step& s, const char** why) {
  const PassPlan plan = sums_plan<Epi>(s.g.kblocks);
  Pass& p = s.two;
  p.kern = reinterpret_cast<const void*>(plan.kern);
  p.threads = plan.threads;
  p.smem = plan.smem;
  if (int rc = operand_maps(s, Epi::kAug, true, kBM, kBM, p, why)) return rc;
  const int units = pair_units(p);
  if (units < 1) return *why = kNoFit, LORA_CE_ECUDA;
  p.g = s.g;
  p.g.n_a = (s.hd.V + 2 * kBM - 1) / (2 * kBM);
  p.g.n_b = s.n_b2 = (s.T + kBN - 1) / kBN;
  p.g.by_b = 1;
  s.bn2 = kBN;
  p.G = s.G2 = (int)std::min<long long>(units, (long long)p.g.n_a * p.g.n_b);
  s.cparts2 = col_parts(Epi::kWarps);
  return 0;
}

template <int kPass, int R>
int tc_pass(Step& s, const char** why) {
  const int V = s.hd.V, T = s.T, half = tc_bn(R) / 2;
  Pass& p = kPass == 1 ? s.one : s.two;
  if (int rc = operand_maps(s, true, kPass == 2, kBM, half, p, why)) return rc;
  if (!(kPass == 1 ? make_map_ld(&p.maps[4], s.w->xv, 2 * R, V, s.g.Vpad, R)
                   : make_map_ld(&p.maps[4], s.w->xt, 2 * R, T, round_up(T, kBN), R)))
    return *why = kNoMap, LORA_CE_ECUDA;
  p.n_maps = 5;
  p.g = s.g;
  p.g.stages = TcLayout::stages(s.g.kblocks, R);
  p.g.drain_gain = (float)(1.0 + acc_short(2 * tc_drain(R) * tc_bn(R) / 16, 0));
  p.kern = reinterpret_cast<const void*>(lce_gemm_tc<kPass, R, true>);
  p.threads = kThreadsT;
  p.smem = TcLayout::bytes(s.g.kblocks, p.g.stages, R);
  if (p.g.stages < 2 || p.smem > kMaxDynSmem) return *why = kNoFit, LORA_CE_ECUDA;
  const int units = pair_units(p);
  if (units < 1) return *why = kNoFit, LORA_CE_ECUDA;
  p.g.n_a = ((kPass == 1 ? T : V) + 2 * kBM - 1) / (2 * kBM);
  p.g.n_b = ((kPass == 1 ? V : T) + tc_bn(R) - 1) / tc_bn(R);
  p.G = (int)std::min<long long>(units, (long long)p.g.n_a * p.g.n_b);
  if (kPass == 1) {
    s.slots = SlotPlan{2, p.g.n_a, p.g.n_b, units, s.g.Tcap, s.g.p_max, s.g.p_sum, nullptr,
                       s.g.p_q};
  } else {
    s.n_b2 = p.g.n_b;
    s.bn2 = tc_bn(R);
    s.G2 = p.G;
    s.cparts2 = 1;
  }
  return 0;
}

template <class EL, class EG>
int sums_passes(Step& s, const char** why) {
  if (int rc = rows_pass(s, sums_plan<EL>(s.g.kblocks), EL::kAug, col_parts(EL::kWarps), nullptr,
                         s.g.p_q, why))
    return rc;
  return sums_pass2<EG>(s, why);
}
template <int R>
int tc_passes(Step& s, const char** why) {
  const int rc = tc_pass<1, R>(s, why);
  return rc ? rc : tc_pass<2, R>(s, why);
}

// Both gradient passes of kernel rank R.
int grad_passes(Step& s, int R, const char** why) {
  switch (R) {
    case 4:
      return sums_passes<EpiLse<4, false, false, true>, EpiGrad<4, false, false, true>>(s, why);
    case 8:
      return sums_passes<EpiLse<8, true, false, true>, EpiGrad<8, true, false, true>>(s, why);
    case 16: return tc_passes<16>(s, why);
    case 32: return tc_passes<32>(s, why);
    default: return tc_passes<64>(s, why);
  }
}

template <int R>
bool launch_dA(const Step& s, const DistillWs& w, cudaStream_t st) {
  cudaLaunchConfig_t lc = {};
  lc.gridDim = dim3((unsigned)((s.T + kDAChunk - 1) / kDAChunk), (unsigned)(s.hd.d / 64));
  lc.blockDim = dim3(256);
  lc.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  lc.attrs = attr;
  lc.numAttrs = 1;
  return cudaLaunchKernelEx(&lc, lh_dA<R>, s.T, s.hd.d, (const __half*)w.h16,
                            (const float*)w.dU, w.gAp) == cudaSuccess;
}

}  // namespace

namespace lce {

size_t head_score_bytes(const HeadCore& hd, int T, int top_k) {
  return score_ws(hd, T, top_k, nullptr).bytes;
}

size_t head_distill_bytes(const HeadCore& hd, int T, int, bool grads) {
  return distill_ws(hd, T, grads, nullptr).bytes;
}

int head_score_run(const HeadCore& hd, const void* H, int dtype, int T, const int32_t* tokens,
                   int top_k, float* logprob, float* entropy, int32_t* top_ids,
                   float* top_logprobs, void* ws, cudaStream_t st, const char** why) {
  Aug aug = aug_of(hd.r);
  const ScoreWs w = score_ws(hd, T, top_k, ws);
  const bool few = few_score(T, aug.R, w.sub), r4 = aug.R == 4 && !few;
  if (few) aug.layout = aug.width = 0;  // the rank term from B as it is
  const int sms = sm_count();
  const float* const Bt = !r4 ? nullptr : hd.layout ? hd.B : w.Bt;
  GemmArgs g{};
  fill_pass1(g, hd, aug, T, 1.0f);
  g.err = w.stats + kStErr;
  g.p_max = w.p_max;
  g.p_sum = w.p_sum;
  g.p_ent = w.p_ent;
  g.sub_max = w.sub_max;
  g.sub_second = w.sub_second;
  g.sub_rest = w.sub_rest;
  g.sub_arg = w.sub_arg;
  g.sub_arg2 = w.sub_arg2;
  g.n_sub = w.n_sub;
  g.sU4 = w.sU;
  g.Bt = Bt;
  // per-row kernel: a warp per position, or four where that many positions do not
  // fill the SMs (eight where there are more than 1,024 records).  V = 49152, whole
  // calls in us, four warps against one: 8 alternatives at 600 / 1,184 / 2,047 / 3,000
  // positions 90 / 127 / 176 / 246 against 106 / 127 / 176 / 231; 64 alternatives 102 /
  // 143 / 209 / 293 against 133 / 166 / 242 / 276
  ScoreArgs a{};
  a.n_sub = w.n_sub;
  a.sub = w.sub;
  a.top_k = top_k;
  a.n_pick = std::min(w.n_sub, std::max(top_k, kMinPick));
  a.cap = 2 * score_picks(a.n_pick) + top_k + 65;  // and the given token
  const bool warps = T >= sms * (top_k > 16 ? 16 : 8) && w.n_sub <= 32 * 32;
  const int tw = warps ? 1 : w.n_sub <= 8 * 128 ? 4 : 8;  // warps per position
  void (*rows)(ScoreArgs) = warps ? w.n_sub <= 24 * 32 ? lh_score_rows<1, 24> : lh_score_rows<1, 32>
                            : tw == 4 ? lh_score_rows<4, 8> : lh_score_rows<8, 32>;
  const size_t team = score_team_smem(a.n_pick, a.cap, tw);
  const size_t rows_smem =
      warps ? kScoreRows * std::max(team, (size_t)(w.n_sub + 1) * 4) : team;
  if (!allow_smem(reinterpret_cast<const void*>(rows), rows_smem))
    return *why = kNoFit, LORA_CE_ECUDA;

  PrepArgs pa = prep_args(hd, aug, H, dtype, T);
  pa.h16 = w.h16;
  pa.sU = w.sU;
  pa.haug = aug.width ? w.haug : nullptr;
  pa.hn = top_k > 0 ? w.hn : nullptr;
  pa.stats = w.stats;
  PackArgs pk{};
  pk.B = BView{hd.B, hd.V, hd.r, aug.R, hd.layout};
  pk.V = hd.V;
  pk.r = hd.r;
  pk.R = aug.R;
  pk.Vpad = g.Vpad;
  pk.Bt = r4 && !hd.layout ? w.Bt : nullptr;
  pk.waug = aug.width ? w.waug : nullptr;
  pk.aug_layout = aug.layout;
  pk.aug_width = aug.width;

  NormArgs na{};
  na.W = hd.W;
  na.V = hd.V;
  na.d = hd.d;
  na.B = pk.B;
  na.A = hd.A;
  na.lda = hd.lda;
  na.r = hd.r;
  na.out = top_k > 0 ? w.norms : nullptr;

  // all that can be refused comes before the first launch
  const PrepPlan prep = plan_prep(pa, pk, na, true, 0, !few && (pk.Bt || pk.waug), sms);
  if (!prep.ok) return *why = kNoFit, LORA_CE_ECUDA;
  if (few) {
    const int blocks = few_blocks(hd.V);
    const float lg = (float)((1.0 + kLoss32) / std::log(2.0));
    FewArgs f = few_args(hd, aug.R, T, w.h16, w.sU, lg);
    f.p_max = w.p_max;
    f.p_sum = w.p_sum;
    f.p_ent = w.p_ent;
    f.sub_max = w.sub_max;
    f.sub_second = w.sub_second;
    f.sub_rest = w.sub_rest;
    f.sub_arg = w.sub_arg;
    f.sub_arg2 = w.sub_arg2;
    f.n_sub = w.n_sub;
    const FewPlan pass = plan_few<kFewScore>(f);
    if (!pass.ok) return *why = kNoFit, LORA_CE_ECUDA;
    if (!launch_prep(prep, pa, pk, na, st) || !launch_few(pass, f, blocks, st))
      return *why = kNoLaunch, LORA_CE_ECUDA;
    a.p = SlotPlan{1, 1, blocks, blocks, f.ld, w.p_max, w.p_sum, w.p_ent, nullptr};
    a.lg = lg;
  } else {
    Step s{hd, w.h16, w.haug, w.waug, aug, T, sms, g, nullptr};
    if (int rc = rows_pass(s, score_plan(g.kblocks, w.sub, r4), aug.width != 0,
                           col_parts(EpiScore<65536, 64, false>::kWarps), w.p_ent, nullptr, why))
      return rc;
    if (!launch_prep(prep, pa, pk, na, st) || !launch_pass(s.one, st))
      return *why = kNoLaunch, LORA_CE_ECUDA;
    a.p = s.slots;
    a.lg = g.lg;
  }
  a.z = logit_args(hd, aug, T, w.h16, w.sU, w.haug, w.waug);
  a.norms = w.norms;
  a.hn = w.hn;
  a.steps = 4 * g.kmain + (g.kblocks > g.kmain ? g.n_aug : 0);
  if (Bt) a.z.B = BView{Bt, hd.V, hd.r, aug.R, 1};  // a row's ranks side by side
  a.sub_max = w.sub_max;
  a.sub_second = w.sub_second;
  a.sub_rest = w.sub_rest;
  a.sub_arg = w.sub_arg;
  a.sub_arg2 = w.sub_arg2;
  a.tokens = tokens;
  a.stats = w.stats;
  a.logprob = logprob;
  a.entropy = entropy;
  a.top_ids = top_ids;
  a.top_logprobs = top_logprobs;
  const int per = warps ? kScoreRows : 1;
  const int threads = 32 * tw * per;
  if (!launch_after(rows, (T + per - 1) / per, threads, rows_smem, st, a))
    return *why = kNoLaunch, LORA_CE_ECUDA;
  return 0;
}

template <bool kGrads>
void (*distill_rows(int tw))(DistillArgs) {
  return tw == 1   ? lh_distill_rows<kGrads, 1>
         : tw == 4 ? lh_distill_rows<kGrads, 4> : lh_distill_rows<kGrads, 8>;
}

int head_distill_run(const HeadCore& hd, const void* H, int dtype, int T, int K,
                     const int32_t* ids, const float* teacher, float tau, const float* weight,
                     float* loss, const GradOut& out, void* ws, cudaStream_t st,
                     const char** why) {
  const bool grads = out.gA != nullptr;
  Aug aug = aug_of(hd.r);
  const int R = aug.R;
  const DistillWs w = distill_ws(hd, T, grads, ws);
  const bool few = few_distill(T, R), tc = grads && R >= 16 && !few;
  if (few) aug.layout = aug.width = 0;  // the rank term from B as it is
  Step s{hd, w.h16, w.haug, w.waug, aug, T, sm_count(), GemmArgs{}, &w};
  fill_pass1(s.g, hd, aug, T, tau);
  const float* const Bt = few || !(grads || R == 4) ? nullptr : hd.layout ? hd.B : w.Bt;
  s.g.err = w.stats + kStErr;
  s.g.p_max = w.p_max;
  s.g.p_sum = w.p_sum;
  s.g.p_q = w.p_q;
  s.g.tok = w.tok;
  s.g.sU4 = w.sU;
  s.g.Bt = Bt;
  s.g.gBp = w.gBp;
  s.g.nml = w.nml;

  // weights may leave whole tiles of positions without one that counts
  const bool order = weight && !few && T > 2 * kBM;
  s.g.active = order ? w.stats + kStActive : nullptr;
  PrepArgs pa = prep_args(hd, aug, H, dtype, T);
  pa.order = order ? w.order : nullptr;
  pa.h16 = w.h16;
  pa.sU = w.sU;
  pa.haug = aug.width ? w.haug : nullptr;
  pa.stats = w.stats;
  pa.ids = ids;
  pa.teacher = teacher;
  pa.V = hd.V;
  pa.weight = weight;
  pa.K = K;
  pa.tau = tau;
  pa.wt = w.wt;
  if (grads && !tc && !few) {
    pa.tok = w.tok;
    pa.Tpad = (int)round_up(T, kBN);
  }
  PackArgs pk{};
  pk.B = BView{hd.B, hd.V, hd.r, R, hd.layout};
  pk.V = hd.V;
  pk.r = hd.r;
  pk.R = R;
  pk.Vpad = s.g.Vpad;
  pk.Bt = Bt && !hd.layout ? w.Bt : nullptr;
  pk.Bt_plain = tc;  // the rank sums' passes have xv instead
  pk.waug = aug.width ? w.waug : nullptr;
  pk.aug_layout = aug.layout;
  pk.aug_width = aug.width;
  pk.xv = tc ? w.xv : nullptr;
  pk.stats = w.stats;
  const bool pack = pk.Bt || pk.waug || pk.xv;
  const NormArgs no{};
  // all that can be refused comes before the first launch; the scale of xv needs the
  // largest |B| first
  const PrepPlan prep = plan_prep(pa, pk, no, true, tc ? 2 * s.sms : 0, pack && !tc, s.sms);
  const PrepPlan prep2 = tc ? plan_prep(pa, pk, no, false, 0, true, s.sms) : PrepPlan{};
  if (!prep.ok || (tc && !prep2.ok)) return *why = kNoFit, LORA_CE_ECUDA;
  const float few_lg = (float)((1.0 + kLoss32) / (std::log(2.0) * (double)tau));
  FewArgs f = few_args(hd, R, T, w.h16, w.sU, few_lg);
  const int v_blocks = few_blocks(hd.V);
  FewPlan forward, backward;
  if (few) {
    f.p_max = w.p_max;
    f.p_sum = w.p_sum;
    f.p_q = w.p_q;
    forward = grads ? plan_few<kFewForward>(f) : plan_few<kFewLoss>(f);
    if (grads) backward = plan_few<kFewBackward>(f);
    if (!forward.ok || !backward.ok) return *why = kNoFit, LORA_CE_ECUDA;
    s.slots = SlotPlan{1, 1, v_blocks, v_blocks, f.ld, w.p_max, w.p_sum, nullptr, w.p_q};
  } else {
    const int rc = grads ? grad_passes(s, R, why)
                         : rows_pass(s, score_plan(s.g.kblocks, 0, R == 4), aug.width != 0,
                                     col_parts(EpiScore<65536, 0, false>::kWarps), nullptr, nullptr,
                                     why);
    if (rc) return rc;
  }
  if (cudaMemsetAsync(w.stats, 0, w.zero_bytes, st) != cudaSuccess)
    return *why = "cudaMemsetAsync failed", LORA_CE_ECUDA;
  if ((order && !launch_plain(lh_order, 1, 1024, 0, st, T, K, hd.V, weight, ids, teacher, w.masks,
                              w.order, w.stats)) ||
      !launch_prep(prep, pa, pk, no, st) || (tc && !launch_prep(prep2, pa, pk, no, st)) ||
      !(few ? launch_few(forward, f, v_blocks, st) : launch_pass(s.one, st)))
    return *why = kNoLaunch, LORA_CE_ECUDA;
  DistillArgs a{};
  a.z = logit_args(hd, aug, T, w.h16, w.sU, w.haug, w.waug);
  a.z.R = R;
  a.z.B.R = R;
  if (Bt && R == 4) a.z.B = BView{Bt, hd.V, hd.r, R, 1};  // a row's ranks side by side
  a.p = s.slots;
  a.lg = few ? few_lg : s.g.lg;
  a.tau = tau;
  a.scale = hd.scale;
  a.K = K;
  a.ids = ids;
  a.teacher = teacher;
  a.order = pa.order;
  a.active = s.g.active;
  a.wt = w.wt;
  a.Bt = Bt;
  a.Bt_plain = pk.Bt && tc;
  a.stats = w.stats;
  a.loss = loss;
  a.tok = grads && !tc && !few ? w.tok : nullptr;
  a.ref = grads && few ? w.ref : nullptr;
  a.nml = tc ? w.nml : nullptr;
  a.xs = w.xs;
  a.dU = w.dU;
  a.corr = w.corr;
  // warps per position: eight while blocks of eight fit beside each other, one where
  // that many positions fill the SMs.  V = 49152, whole calls in us.  Eight / four, rank
  // 64, 64 entries, 150 and 300 positions: 217 / 238, 279 / 272; rank 4, 8 entries, 450:
  // 125 / 115.  Four / one, rank 4, 1,184 and 2,047 positions: 188 / 184, 276 / 254;
  // rank 64: 508 / 541, 741 / 727.
  const int tw = T <= 2 * s.sms ? 8 : T < 10 * s.sms ? 4 : 1;
  const int per = tw == 1 ? kRowWarps : 1;
  if (!launch_after(grads ? distill_rows<true>(tw) : distill_rows<false>(tw), (T + per - 1) / per,
                    32 * tw * per, 0, st, a))
    return *why = kNoLaunch, LORA_CE_ECUDA;
  if (!grads) return 0;
  const int a_blocks = ((out.layout ? R : hd.r) * hd.d + 255) / 256;
  if (few) {
    f.ref = w.ref;
    f.corr = w.corr;
    f.dU = w.dU;
    f.stats = w.stats;
    f.gA = out.gA;
    f.gB = out.gB;
    f.layout = out.layout;
    f.Vpad = s.g.Vpad;
    f.v_blocks = out.layout ? (int)(s.g.Vpad / kFewRows) : v_blocks;
    f.loss = loss;
    f.wt = w.wt;
    f.tail = out.tail;
    if (!launch_few(backward, f, f.v_blocks + a_blocks, st))
      return *why = kNoLaunch, LORA_CE_ECUDA;
    return 0;
  }
  if (tc) {
    const long long n = (long long)T * R;
    if (!launch_after(lh_xt, (int)std::min<long long>((n + 255) / 256, 8LL * s.sms), 256, 0, st, T,
                      R, (long long)round_up(T, kBN), (const float*)w.sU, (const float*)w.wt,
                      (const float*)w.xs, (const int*)w.stats, w.xt))
      return *why = kNoLaunch, LORA_CE_ECUDA;
  }
  if (!launch_pass(s.two, st)) return *why = kNoLaunch, LORA_CE_ECUDA;
  const bool dA_ok = R == 4    ? launch_dA<4>(s, w, st)
                     : R == 8  ? launch_dA<8>(s, w, st)
                     : R == 16 ? launch_dA<16>(s, w, st)
                     : R == 32 ? launch_dA<32>(s, w, st) : launch_dA<64>(s, w, st);
  if (!dA_ok) return *why = kNoLaunch, LORA_CE_ECUDA;
  GradArgs ga{};
  ga.T = T;
  ga.d = hd.d;
  ga.V = hd.V;
  ga.r = hd.r;
  ga.R = R;
  ga.n_chunks = (T + kDAChunk - 1) / kDAChunk;
  ga.cparts = s.cparts2;
  ga.res_rows = 2 * kBM;
  ga.n_b2 = s.n_b2;
  ga.bn2 = s.bn2;
  ga.active = s.g.active;
  ga.G2 = s.G2;
  ga.Vpad = s.g.Vpad;
  ga.gAp = w.gAp;
  ga.gBp = w.gBp;
  ga.corr = w.corr;
  ga.scaled = tc;
  ga.stats = w.stats;
  ga.gA = out.gA;
  ga.gB = out.gB;
  ga.layout = out.layout;
  ga.loss = loss;
  ga.wt = w.wt;
  ga.tail = out.tail;
  if (!launch_after(lh_grads, (int)(s.g.Vpad / kPackRows) + a_blocks, 256, 0, st, ga))
    return *why = kNoLaunch, LORA_CE_ECUDA;
  return 0;
}

int head_step_tail(const void* ws, float* tail, int* err, cudaStream_t st) {
  return launch_plain(lh_tail, 1, 1, 0, st, static_cast<const int*>(ws), tail, err) ? 0
                                                                                    : LORA_CE_ECUDA;
}

namespace {
const char* head_refuses(const HeadCore& hd, int T) {
  if (hd.d < 64 || hd.d % 64 != 0 || hd.d > 64 * kMaxHead64)
    return "dim must be a multiple of 64 in [64, 640]";
  if (hd.V < 1 || hd.V > (1 << 19)) return "vocab must be in [1, 2^19]";
  if (hd.r < 0 || hd.r > kMaxFusedRank) return "rank must be in [0, 64]";
  if (!std::isfinite(hd.scale)) return "scale must be finite";
  if (T < 1 || T > LORA_HEAD_MAX_TOKENS) return "T must be in [1, 2^20]";
  return nullptr;
}
}  // namespace

const char* head_score_refuses(const HeadCore& hd, int T, int top_k) {
  if (const char* why = head_refuses(hd, T)) return why;
  if (top_k < 0 || top_k > LORA_HEAD_MAX_TOP || top_k > hd.V)
    return "top_k must be in [0, 128] and no more than vocab";
  return nullptr;
}

const char* head_distill_refuses(const HeadCore& hd, int T, int K, bool grads, float tau) {
  if (const char* why = head_refuses(hd, T)) return why;
  if (K < 1 || K > LORA_HEAD_MAX_TOP) return "K must be in [1, 128]";
  if (grads && hd.r < 1) return "gradients need a rank of at least 1";
  if (!(tau >= 0.01f && tau <= 100.0f)) return "temperature must be in [0.01, 100]";
  return nullptr;
}

}  // namespace lce

namespace {

HeadCore core_of(const lora_head* h) {
  return HeadCore{reinterpret_cast<const __half*>(h->W), h->A, h->rank, h->B, 0,
                  h->dim, h->vocab, h->rank, h->scale};
}

// Every buffer is memory of the current device, with its alignment.
struct Buffers {
  int dev = -1;
  int rc = 0;
  void need(const void* p, uintptr_t align, const char* name) {
    if (rc) return;
    if (!p) {
      rc = hfail(LORA_CE_EINVAL, "");
      g_head_error = std::string(name) + " is null";
      return;
    }
    if (reinterpret_cast<uintptr_t>(p) % align != 0) {
      rc = hfail(LORA_CE_EINVAL, "");
      g_head_error = std::string(name) + " must be " + std::to_string(align) + "-byte aligned";
    }
  }
  // after every need(): where the memory is
  void here(const void* p, const char* name) {
    if (rc || !p) return;
    if (dev < 0 && cudaGetDevice(&dev) != cudaSuccess) {
      rc = hfail(LORA_CE_ECUDA, "no CUDA device");
      cudaGetLastError();
      return;
    }
    cudaPointerAttributes at;
    if (cudaPointerGetAttributes(&at, p) != cudaSuccess) {
      cudaGetLastError();
      at.type = cudaMemoryTypeUnregistered;
    }
    if ((at.type != cudaMemoryTypeDevice || at.device != dev) && at.type != cudaMemoryTypeManaged) {
      rc = hfail(LORA_CE_EINVAL, "");
      g_head_error = std::string(name) + " is not memory of the current device";
    }
  }
};

int check_arch() {
  static std::mutex mu;
  static std::map<int, int> major;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return hfail(LORA_CE_ECUDA, "no CUDA device");
  std::lock_guard<std::mutex> lock(mu);
  auto it = major.find(dev);
  if (it == major.end()) {
    int m = 0;
    if (cudaDeviceGetAttribute(&m, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess)
      return hfail(LORA_CE_ECUDA, "cudaDeviceGetAttribute failed");
    it = major.emplace(dev, m).first;
  }
  if (it->second != 10) return hfail(LORA_CE_ECUDA, "this library runs on sm_100 (B200) only");
  if (!encode_fn()) return hfail(LORA_CE_ECUDA, "cuTensorMapEncodeTiled unavailable");
  return 0;
}

int check_score(const lora_head* h, int T, int top_k) {
  if (!h) return hfail(LORA_CE_EINVAL, "null head");
  const char* why = head_score_refuses(core_of(h), T, top_k);
  return why ? hfail(LORA_CE_EINVAL, why) : 0;
}

int check_distill(const lora_head* h, int T, int K, bool grads, float tau) {
  if (!h) return hfail(LORA_CE_EINVAL, "null head");
  const char* why = head_distill_refuses(core_of(h), T, K, grads, tau);
  return why ? hfail(LORA_CE_EINVAL, why) : 0;
}

}  // namespace

extern "C" {

const char* lora_head_last_error(void) { return g_head_error.c_str(); }

size_t lora_head_score_workspace(const lora_head* h, int32_t T, int32_t top_k) {
  size_t bytes = 0;
  entry([&] {
    const int rc = check_score(h, T, top_k);
    if (!rc) bytes = head_score_bytes(core_of(h), T, top_k);
    return rc;
  });
  return bytes;
}

size_t lora_head_distill_workspace(const lora_head* h, int32_t T, int32_t K, int32_t grads) {
  size_t bytes = 0;
  entry([&] {
    const int rc = check_distill(h, T, K, grads != 0, 1.0f);
    if (!rc) bytes = head_distill_bytes(core_of(h), T, K, grads != 0);
    return rc;
  });
  return bytes;
}

int lora_head_score(const lora_head* h, const void* H, int32_t h_dtype, int32_t T,
                    const int32_t* tokens, int32_t top_k, float* logprob, float* entropy,
                    int32_t* top_ids, float* top_logprobs, void* ws, size_t ws_bytes,
                    void* stream) {
  return entry([&]() -> int {
    if (int rc = check_score(h, T, top_k)) return rc;
    if (h_dtype < LORA_CE_BF16 || h_dtype > LORA_CE_F32)
      return hfail(LORA_CE_EINVAL, "bad hidden-state dtype");
    if ((tokens == nullptr) != (logprob == nullptr))
      return hfail(LORA_CE_EINVAL, "tokens and logprob go together");
    if (!logprob && !entropy && top_k == 0) return hfail(LORA_CE_EINVAL, "nothing is asked for");
    Buffers b;
    struct {
      const void* p;
      uintptr_t align;
      const char* name;
      bool used;
    } all[] = {{h->W, 16, "W", true},
               {h->A, 4, "A", h->rank > 0},
               {h->B, 4, "B", h->rank > 0},
               {H, 16, "H", true},
               {tokens, 4, "tokens", tokens != nullptr},
               {logprob, 4, "logprob", logprob != nullptr},
               {entropy, 4, "entropy", entropy != nullptr},
               {top_ids, 4, "top_ids", top_k > 0},
               {top_logprobs, 4, "top_logprobs", top_k > 0},
               {ws, 256, "workspace", true}};
    for (const auto& x : all)
      if (x.used) b.need(x.p, x.align, x.name);
    if (!b.rc && ws_bytes < head_score_bytes(core_of(h), T, top_k))
      return hfail(LORA_CE_EINVAL, "workspace too small");
    for (const auto& x : all)
      if (x.used) b.here(x.p, x.name);
    if (b.rc) return b.rc;
    if (int rc = check_arch()) return rc;
    const char* why = "";
    const int rc = head_score_run(core_of(h), H, h_dtype, T, tokens, top_k, logprob, entropy,
                                  top_ids, top_logprobs, ws, static_cast<cudaStream_t>(stream), &why);
    return rc ? hfail(rc, why) : 0;
  });
}

int lora_head_distill(const lora_head* h, const void* H, int32_t h_dtype, int32_t T, int32_t K,
                      const int32_t* ids, const float* teacher, float temperature,
                      const float* weight, float* loss, float* gA, float* gB, void* ws,
                      size_t ws_bytes, void* stream) {
  return entry([&]() -> int {
    if ((gA == nullptr) != (gB == nullptr))
      return hfail(LORA_CE_EINVAL, "gA and gB go together");
    const bool grads = gA != nullptr;
    if (int rc = check_distill(h, T, K, grads, temperature)) return rc;
    if (h_dtype < LORA_CE_BF16 || h_dtype > LORA_CE_F32)
      return hfail(LORA_CE_EINVAL, "bad hidden-state dtype");
    Buffers b;
    struct {
      const void* p;
      uintptr_t align;
      const char* name;
      bool used;
    } all[] = {{h->W, 16, "W", true},
               {h->A, 4, "A", h->rank > 0},
               {h->B, 4, "B", h->rank > 0},
               {H, 16, "H", true},
               {ids, 4, "ids", true},
               {teacher, 4, "teacher", true},
               {weight, 4, "weight", weight != nullptr},
               {loss, 4, "loss", true},
               {gA, 4, "gA", grads},
               {gB, 4, "gB", grads},
               {ws, 256, "workspace", true}};
    for (const auto& x : all)
      if (x.used) b.need(x.p, x.align, x.name);
    if (!b.rc && ws_bytes < head_distill_bytes(core_of(h), T, K, grads))
      return hfail(LORA_CE_EINVAL, "workspace too small");
    for (const auto& x : all)
      if (x.used) b.here(x.p, x.name);
    if (b.rc) return b.rc;
    if (int rc = check_arch()) return rc;
    const char* why = "";
    const int rc = head_distill_run(core_of(h), H, h_dtype, T, K, ids, teacher, temperature, weight,
                                    loss, GradOut{gA, gB, 0, nullptr}, ws,
                                    static_cast<cudaStream_t>(stream), &why);
    return rc ? hfail(rc, why) : 0;
  });
}

}  // extern "C"
