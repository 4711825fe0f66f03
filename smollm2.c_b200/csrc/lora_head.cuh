// lora_head.cuh — device code of the operators on the LoRA head: token log
// probabilities with entropy and top alternatives (score), and distillation
// from a teacher's top logits (distill).  Both form
//   z[t][v] = h[t].W[v] + s (h[t].A).B[:,v],   h = f16(H)
// in the GEMM passes of lora_ce_kernels.cuh and lora_ce_tc.cuh, or, for few
// positions, in a pass of its own; this file has that, the epilogue and the
// kernels around the passes that are theirs alone.
//
// Accuracy.  tcgen05 truncates towards zero when it adds a K-step's 16
// products to the f32 accumulator, half a unit in the last place on average.
// Where a logit is large its partial sums grow about linearly over the n
// K-steps, and the mean of ulp(x) / x over a binade is 2^-23 / (2 ln 2), which
// makes the accumulator fall short by z (n + 1) 2^-26 / ln 2.  Measured against
// 64-bit sums over logits from 3 to 15: 0.79 of that at hidden sizes 64, 128
// and 576 alike (6.2e-7 z at 576, with a spread of 1.6e-7 z; an f32 product of
// a library has no shortfall and a spread of 3e-7 z).  acc_short() gives the
// measured share and the softmax's exponent factor makes it good
// (GemmArgs::lg).  That is for partial sums that grow evenly towards the logit.  Where
// channels of h cancel, the shortfall follows the partial sums, up to n 2^-24 of them,
// and no factor of z makes it good: two channels whose parts of every logit are 32 to 48
// and cancel leave log probabilities of 300 positions 2e-5 off on average and 4.5e-5 at
// most, parts of 128 to 192 9e-5 and 2e-4 (an f32 product of a library: 1e-6 and 7e-5,
// 1e-6 and 3e-4).  The order of alternatives takes them into account (logit_gaps).  Sums of many terms go in two levels (EpiLse, lce_gemm_tc).
// Gradients of 8192 positions against 64 bits, where a bias adds up and
// rounding does not: rank 4 9e-6 with neither, 6e-6 with the factor, 4e-7 with
// both; rank 64 2e-5, 1.5e-5, 4e-7 (a library's f32 products: 2e-6 to 3e-6).
// Few logits decide more than a sum: those of given tokens, of a teacher's
// entries, the largest, and alternatives whose order the pass's logits do not tell
// are computed again from the f16 operands with 64-bit sums.
#pragma once
#include "lora_ce_kernels.cuh"

namespace lce {

constexpr int kMaxTop = 128;      // largest top_k, largest teacher list
constexpr int kMinPick = 8;       // logits of a row that are computed again at least
constexpr int kPickStop = 7;      // the search ends with up to so many records beyond that,
constexpr int kPickSlack = 24;    // and takes near ties of the last up to so many
constexpr int kRowWarps = 8;      // lh_distill_rows: positions per block where each has a warp
constexpr int kMaxHead64 = 10;    // hidden size in units of 64

// Device words at the start of a workspace.
enum : int { kStErr = 0, kStBMax = 1, kStUMax = 2, kStActive = 3, kStatWords = 64 };

// B of the head: [r][V] (layout 0), or the pair-interleaved layout of a
// trainer's handle at kernel rank R (layout 1, bidx).
struct BView {
  const float* p;
  long long V;
  int r, R, layout;
  __device__ __forceinline__ float at(int j, long long v) const {
    return layout ? p[bidx(v, j, R)] : p[(long long)j * V + v];
  }
};

// ------------------------------------------------------------- pass over z
// Record k of position t: eight positions' side by side, so that an epilogue
// warp's store fills sectors and a block of eight rows reads one run.
__device__ __forceinline__ long long sub_idx(int t, int k, int n_sub) {
  return ((long long)(t >> 3) * n_sub + k) * 8 + (t & 7);
}

// The thread owns position t; columns are vocab ids (as EpiLse, without the
// rank sums).  Per column: the online max and sum(exp) in units of log2.
// kSub 0 is that alone (a loss).  Otherwise also the entropy sum and records
// from which lh_score_rows picks the alternatives:
//   kSub 64: per 64 columns the largest logit, the second largest of its 8-column
//            chunks' maxima, both with their columns, and the largest of the rest
//   kSub 8:  per 8 columns the largest, its column, the largest of the rest
//   kSub 1:  the logit
// A row's k largest logits lie in the k records with the largest maxima: were
// one outside, k records would each hold a logit that precedes it.  So 14
// bytes stand for 64 logits, and the columns of a record are computed again
// only where its rest reaches into the k largest: for random rows at k = 64,
// V = 49152 about four records in ten rows (with one logit per record only,
// and none for the second, it was 2.7 records a row).  Fewer columns per record
// where the vocabulary gives less than 4 records per alternative.
// Bound by the MMAs and their loads of W, as the training step's passes (tensor
// pipe 54% busy), not by the epilogue: without records or entropy (kSub 0) it is
// no faster, nor with the two largest of a chunk from a tree of min and max on
// logits that carry their column in the lowest bits, nor with a fifth ring stage.
// kR4: the rank term of ranks up to 4 here, in f32 from staged rows of B (as EpiLse),
// so that those ranks have f32's range, as in the training step.  As f16 pairs in a
// K-block of its own, which it filled by a quarter, the pass took as long (8,192
// positions, V = 49152, d = 576: 417 us, as pairs 420).
template <int kRing_, int kSub, bool kR4>
struct EpiScore {
  static constexpr bool kAug = !kR4;
  static constexpr bool kDepend = true;
  static constexpr int kRec = kR4 ? 4 : 0;
  static constexpr int kRing = kRing_;
  static constexpr int kRecBufs = kR4 ? 2 : 1;
  static constexpr int kWarps = 16;
  static constexpr int kCW = 8;
  static constexpr bool kTop = kSub != 0;
  int t;
  bool valid;
  float m, mL;   // reference max, m * lg
  float2 s2;     // sum of e over even / odd columns
  float2 e2s;    // sum of e * x, x the exponent in log2 units
  float S, Slo, E, Elo;  // the same over the row so far, folded every 64 columns (as EpiLse)
  float r1, r2, rest;    // kSub 64: the record so far
  int a1, a2;
  float2 sU2[kR4 ? 4 : 1];

  __device__ static const float* global_recs(const GemmArgs& g, int b) {
    return g.Bt + (long long)b * kBN * kRec;
  }
  __device__ static int limit(const GemmArgs& g) { return g.V; }

  __device__ void begin(const GemmArgs& g, int abs_row) {
    t = abs_row;
    valid = t < g.T;
    m = mL = -INFINITY;
    s2 = e2s = f2(0.f, 0.f);
    S = Slo = E = Elo = 0.f;
    r1 = r2 = rest = -INFINITY;
    a1 = a2 = 0;
    if constexpr (kR4) {
      float u[4];
      ld_vec<4>(g.sU4 + 4ll * (valid ? t : 0), u);
#pragma unroll
      for (int j = 0; j < 4; ++j) sU2[j] = f2(u[j], u[j]);
    }
  }

  // Adds the chunk's terms at reference nm = -(reference max) * lg; the first `n_in`
  // columns are the vocabulary's.
  template <bool kTail>
  __device__ __forceinline__ void sum(const float (&z)[kCW], float2 L2, float nm, int n_in) {
    const float2 nm2 = f2(nm, nm);
#pragma unroll
    for (int p = 0; p < kCW / 2; ++p) {
      float2 x2 = __ffma2_rn(f2(z[2 * p], z[2 * p + 1]), L2, nm2);
      if (kTail && kTop) {  // columns past the vocabulary: e = 0 and e * x = 0, not 0 * inf
        if (2 * p >= n_in) x2.x = -1e30f;
        if (2 * p + 1 >= n_in) x2.y = -1e30f;
      }
      const float2 e2 = f2(ex2f(x2.x), ex2f(x2.y));
      s2 = __fadd2_rn(s2, e2);
      if constexpr (kTop) e2s = __ffma2_rn(e2, x2, e2s);
    }
  }

  template <bool kTail>
  __device__ __forceinline__ void chunk(const GemmArgs& g, int v0, float (&acc)[kCW],
                                        const float* recs) {
    if constexpr (kR4) {
#pragma unroll
      for (int p = 0; p < kCW / 2; ++p) {
        float b[8];
        ld_vec<8>(recs + p * 8, b);
        float2 z2 = f2(acc[2 * p], acc[2 * p + 1]);
#pragma unroll
        for (int j = 0; j < 4; ++j) z2 = __ffma2_rn(sU2[j], f2(b[2 * j], b[2 * j + 1]), z2);
        acc[2 * p] = z2.x;
        acc[2 * p + 1] = z2.y;
      }
    }
    if (kTail) {
#pragma unroll
      for (int i = 0; i < kCW; ++i)
        if (v0 + i >= g.V) acc[i] = -INFINITY;
    }
    float cm = -INFINITY;
    if constexpr (kSub > 1) {
      float c2 = -INFINITY;
      int at = 0;
#pragma unroll
      for (int i = 0; i < kCW; ++i) {
        const float z = acc[i];
        c2 = fmaxf(c2, fminf(cm, z));
        at = z > cm ? i : at;  // the lowest column among equals
        cm = fmaxf(cm, z);
      }
      if constexpr (kSub == 8) {
        if (valid && v0 < g.V) {
          const long long o = sub_idx(t, v0 / 8, g.n_sub);
          g.sub_max[o] = cm;
          g.sub_rest[o] = c2;
          g.sub_arg[o] = (uint8_t)at;
        }
      } else {
        at += v0 & 63;
        if ((v0 & 63) == 0) {
          r1 = cm;
          a1 = at;
          r2 = -INFINITY;
          a2 = 0;
          rest = c2;
        } else {
          const bool gt = cm > r1;
          const float lo = fminf(cm, r1);
          const int lo_at = gt ? a1 : at;
          a1 = gt ? at : a1;
          r1 = fmaxf(cm, r1);
          rest = fmaxf(fmaxf(rest, c2), fminf(r2, lo));
          a2 = lo > r2 ? lo_at : a2;
          r2 = fmaxf(r2, lo);
        }
        if ((v0 & 63) == 64 - kCW && valid && v0 - (64 - kCW) < g.V) {
          const long long o = sub_idx(t, v0 / 64, g.n_sub);
          g.sub_max[o] = r1;
          g.sub_second[o] = r2;
          g.sub_rest[o] = rest;
          g.sub_arg[o] = (uint8_t)a1;
          g.sub_arg2[o] = (uint8_t)a2;
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < kCW; ++i) {
        cm = fmaxf(cm, acc[i]);
        if (kSub == 1 && valid && v0 + i < g.V) g.sub_max[sub_idx(t, v0 + i, g.n_sub)] = acc[i];
      }
    }
    if (kTail && v0 >= g.V) return;
    const float2 L2 = f2(g.lg, g.lg);
    if (cm > m + g.lazy) {  // the reference moves before the chunk is added
      // between the references as they are rounded; 0 when m = -inf
      const float to = cm * g.lg, f = ex2f(mL - to);
      if constexpr (kTop) {
        // x counts from the new reference: sum e (x - delta)
        const float delta = m == -INFINITY ? 0.f : to - mL;
        e2s = f2(f * fmaf(-delta, s2.x, e2s.x), f * fmaf(-delta, s2.y, e2s.y));
        E = f * (fmaf(-delta, S, E) + fmaf(-delta, Slo, Elo));
        Elo = 0.f;
      }
      s2 = f2(s2.x * f, s2.y * f);
      S *= f;
      Slo *= f;
      m = cm;
      mL = to;
    }
    __syncwarp();  // rejoin before the next warp-wide TMEM load
    sum<kTail>(acc, L2, -mL, g.V - v0);
    if (((v0 + kCW) & 63) == 0) fold();
  }

  __device__ __forceinline__ void fold() {
    fold_sum(s2, S, Slo);
    if constexpr (kTop) fold_sum(e2s, E, Elo);
  }

  __device__ void flush(const GemmArgs& g, int slot) {
    if (!valid) return;
    const long long o = (long long)slot * g.Tcap + t;
    g.p_max[o] = mL;
    fold();
    g.p_sum[o] = S + Slo;
    if constexpr (kTop) g.p_ent[o] = E + Elo;
  }
};

// ------------------------------------------------------------- preparation
struct PrepArgs {
  const void* H;
  int dtype, T, Tpad, d;
  const float* A;  // [d][lda], r columns used
  int lda, r, R;   // R: r rounded up to a kernel rank; 0 without an adapter
  float scale;
  __half* h16;     // [T][d]
  float* hn;       // [T] |h16|, or null
  float* sU;       // [T][R] s * U
  float* tok;      // records (tidx layout) or null
  __half* haug;    // [T][aug_width] or null
  int aug_layout, aug_width;
  // distillation: teacher lists and weights; wt[t] = weight * temperature of a
  // position that has at least one entry, else 0 (and its hidden state is read
  // as zeros, whatever it holds)
  const int32_t* ids;
  const float* teacher;
  int V;
  const float* weight;
  int K;
  float tau;
  float* wt;
  const int* order;  // position in row t of what is prepared, or null: t
  int* stats;
  __device__ __forceinline__ int source(int t) const { return order ? order[t] : t; }
};

// A teacher's entry that is there: a logit of -inf weighs nothing, as no entry does.
// (Ids past the vocabulary, NaN and +inf are: lh_distill_rows reports them.)
__device__ __forceinline__ bool is_entry(int id, float logit, int V) {
  return (id >= 0) & ((id >= V) | (logit != -INFINITY));  // (both are read at once)
}

// order: the positions that count (a weight other than 0 and an entry), then the
// others, each in ascending order; their number to stats[kStActive].  The passes run
// over the tiles that hold one that counts, a quarter of all at least: at 8,000
// positions of which 30% are a masked prompt, rank 64, the call takes 1,680 us
// instead of 2,300.
// One block: each warp takes a run of positions, 32 side by side at a time: 14 us at
// 8,000 positions (11 without the teacher's logits, which a list of -inf alone needs; 13
// then with a run of its own for each thread, its loads and stores a line each).
static __global__ void __launch_bounds__(1024) lh_order(int T, int K, int V,
                                                        const float* __restrict__ weight,
                                                        const int32_t* __restrict__ ids,
                                                        const float* __restrict__ teacher,
                                                        unsigned* __restrict__ masks,  // [T / 32]
                                                        int* __restrict__ order,
                                                        int* __restrict__ stats) {
  constexpr int kStep = 8;  // groups of 32 in flight
  constexpr unsigned kAll = 0xffffffffu;
  __shared__ int s_n[32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int groups = (T + 31) / 32, per = (groups + 31) / 32;
  const int g_lo = min(groups, w * per), g_hi = min(groups, g_lo + per);
  int n = 0;
  for (int g0 = g_lo; g0 < g_hi; g0 += kStep) {
    float wt[kStep];
    int id[kStep];
    float x[kStep];
#pragma unroll
    for (int i = 0; i < kStep; ++i) {
      const int t = 32 * (g0 + i) + lane;
      const bool in = g0 + i < g_hi && t < T;
      wt[i] = in ? weight[t] : 0.f;
      id[i] = in ? ids[(long long)t * K] : -1;
      x[i] = in ? teacher[(long long)t * K] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < kStep; ++i) {
      if (g0 + i >= g_hi) break;
      const bool first = is_entry(id[i], x[i], V);
      bool any = wt[i] != 0.f && first;
      unsigned look = __ballot_sync(kAll, wt[i] != 0.f && !first);
      for (; look; look &= look - 1) {  // the first entry is absent: seldom
        const int q = __ffs(look) - 1;
        const long long o = (long long)(32 * (g0 + i) + q) * K;
        bool some = false;
        for (int k = lane; k < K; k += 32) some |= is_entry(ids[o + k], teacher[o + k], V);
        some = __any_sync(kAll, some);
        if (lane == q) any = some;
      }
      const unsigned m = __ballot_sync(kAll, any);
      if (lane == 0) masks[g0 + i] = m;
      n += __popc(m);
    }
  }
  if (lane == 0) s_n[w] = n;
  __syncthreads();
  int before = 0, total = 0;
  for (int q = 0; q < 32; ++q) {
    before += q < w ? s_n[q] : 0;
    total += s_n[q];
  }
  int front = before, back = total + 32 * g_lo - before;
  for (int g0 = g_lo; g0 < g_hi; ++g0) {
    const unsigned m = masks[g0], below = (1u << lane) - 1u;
    const int t = 32 * g0 + lane;
    if (t < T) order[m >> lane & 1u ? front + __popc(m & below) : back + __popc(~m & below)] = t;
    front += __popc(m);
    back += 32 - __popc(m);
  }
  if (threadIdx.x == 0) stats[kStActive] = total;
}

// Elements i, i + 1 of position t.
__device__ __forceinline__ float2 load_pair(const PrepArgs& a, int t, int i) {
  const long long o = (long long)t * a.d + i;
  if (a.dtype == 0) return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(
                        reinterpret_cast<const __nv_bfloat16*>(a.H) + o));
  if (a.dtype == 1) return __half22float2(*reinterpret_cast<const __half2*>(
                        reinterpret_cast<const __half*>(a.H) + o));
  return *reinterpret_cast<const float2*>(reinterpret_cast<const float*>(a.H) + o);
}

// Elements 64 k + 2 lane, + 1 of position t for every k: all on their way at once.
__device__ __forceinline__ void load_row(const PrepArgs& a, int t, int lane,
                                         float2 (&x)[kMaxHead64]) {
  const long long o = ((long long)t * a.d >> 1) + lane;
  auto all = [&](auto* row, auto widen) {
#pragma unroll
    for (int k = 0; k < kMaxHead64; ++k)
      if (64 * k < a.d) x[k] = widen(row[o + 32 * k]);
  };
  if (a.dtype == 0)
    all(reinterpret_cast<const __nv_bfloat162*>(a.H), [](__nv_bfloat162 p) { return __bfloat1622float2(p); });
  else if (a.dtype == 1)
    all(reinterpret_cast<const __half2*>(a.H), [](__half2 p) { return __half22float2(p); });
  else
    all(reinterpret_cast<const float2*>(a.H), [](float2 p) { return p; });
}

// weight * tau of a position that counts, else 0
__device__ __forceinline__ float row_weight(const PrepArgs& a, int t, bool any) {
  const float w = a.weight ? a.weight[t] : 1.0f;
  return any && w != 0.f ? w * a.tau : 0.f;
}

// U[t][j] goes to what the passes read of it.
__device__ __forceinline__ void put_u(const PrepArgs& a, int t, int j, float u, float& umax,
                                      float wt) {
  const int R = a.R;
  const float f = a.scale * u;
  a.sU[(long long)t * R + j] = f;
  if (a.tok) a.tok[tidx(t, j, R)] = f;
  if (a.haug) {
    const __half hi = __float2half_rn(f), lo = __float2half_rn(f - __half2float(hi));
    __half* row = a.haug + (long long)t * a.aug_width;
    row[j] = hi;
    if (a.aug_layout == 1) {  // [hi | hi | lo | 0]
      row[R + j] = hi;
      row[2 * R + j] = lo;
      for (int c = 3 * R + j; c < a.aug_width; c += R) row[c] = __float2half_rn(0.f);
    } else {  // [hi | lo]
      row[R + j] = lo;
    }
  }
  const float m = fabsf(wt * f);
  if (isfinite(m)) umax = fmaxf(umax, m);
}

// The other fields of a record; all of a padding position's.
__device__ __forceinline__ void put_fields(const PrepArgs& a, int t, int from, int lane, int n) {
  for (int f = from + lane; f < tok_stride(a.R); f += n) a.tok[tidx(t, f, a.R)] = 0.f;
}

__device__ __forceinline__ void put_max(const PrepArgs& a, float umax) {
  const unsigned m = __reduce_max_sync(0xffffffffu, __float_as_uint(umax));
  if ((threadIdx.x & 31) == 0 && m)
    atomicMax(reinterpret_cast<unsigned*>(a.stats) + kStUMax, m);
}

// h16 and U = h16.A, one block per position: thread (j, slice) sums rank j over
// its slice of h.  Few positions: every A load of a thread is in flight at once
// (one warp per position, 4 loads at a time, took 40 us at rank 4 and 140 us at
// rank 16; this 6 and 9 us).
__device__ __forceinline__ void prep_row(const PrepArgs& a, int t, float* sh) {
  float* red = sh + a.d;  // [256 + 8] behind h's [d]
  const int tid = threadIdx.x, R = a.R;
  if (t >= a.T) {
    if (a.tok) put_fields(a, t, 0, tid, 256);
    return;
  }
  float wt = 0.f;
  bool active = true;
  const int from = a.source(t);
  if (a.ids) {
    const long long o = (long long)from * a.K + tid;
    const bool mine = tid < a.K && is_entry(a.ids[o], a.teacher[o], a.V);
    wt = row_weight(a, from, __syncthreads_or(mine));
    active = wt != 0.f;
    if (tid == 0) a.wt[t] = wt;
  }
  const int j = R ? tid % R : 0, sl = R ? tid / R : 0, ns = R ? 256 / R : 1;
  float av[16];
  auto fetch = [&](int i0) {
#pragma unroll
    for (int q = 0; q < 16; ++q) {
      const int i = i0 + q * ns;
      av[q] = i < a.d && j < a.r ? a.A[(long long)i * a.lda + j] : 0.f;
    }
  };
  fetch(sl);  // on its way beside h
  float hh = 0.f;
  for (int i = 2 * tid; i < a.d; i += 512) {
    const float2 x = active ? load_pair(a, from, i) : make_float2(0.f, 0.f);
    const __half2 hv = __floats2half2_rn(x.x, x.y);
    *reinterpret_cast<__half2*>(a.h16 + (long long)t * a.d + i) = hv;
    const float2 hf = __half22float2(hv);
    *reinterpret_cast<float2*>(sh + i) = hf;
    hh = fmaf(hf.x, hf.x, fmaf(hf.y, hf.y, hh));
  }
  if (a.hn) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) hh += __shfl_xor_sync(0xffffffffu, hh, off);
    if ((tid & 31) == 0) red[256 + (tid >> 5)] = hh;
  }
  __syncthreads();
  if (a.hn && tid == 0) {
    for (int q = 1; q < 8; ++q) hh += red[256 + q];
    a.hn[t] = sqrtf(hh);
  }
  if (R == 0) return;
  float u = 0.f;
  for (int i0 = sl; i0 < a.d; i0 += 16 * ns) {
    if (i0 != sl) fetch(i0);
#pragma unroll
    for (int q = 0; q < 16; ++q) {
      const int i = i0 + q * ns;
      if (i < a.d) u = fmaf(sh[i], av[q], u);
    }
  }
  red[tid] = u;
  __syncthreads();
  float umax = 0.f;
  if (tid < R) {
    u = 0.f;
    for (int q = 0; q < ns; ++q) u += red[q * R + tid];
    put_u(a, t, tid, u, umax, wt);
  }
  if (a.tok && tid < 4) put_fields(a, t, R, tid, 4);
  if (a.ids && tid < 64) put_max(a, umax);
}

// The same for kTileRows positions per block: all of their hidden states on the
// way at once (64 elements at a time with the next 64 in flight took 35 us for
// 2,047 positions, waiting), then each warp sums its eighth of the hidden size for
// every position and rank: lanes over neighbouring ranks, A straight from global
// memory 12 rows at a time, h four elements per load from shared memory, up to 32
// sums per lane.  (A through shared memory, four sums per thread, a load for each
// operand of each product and two block barriers per 64 elements: 35 us instead of
// 21 for 2,047 positions at rank 64, B packed beside them.)
constexpr int kTileRows = 16;
template <int R>
__device__ __forceinline__ void prep_tile(const PrepArgs& a, int t0, float* smem) {
  constexpr int kLanes = R >= 32 ? 32 : R > 0 ? R : 1;  // over ranks
  constexpr int kPer = R > 32 ? 2 : 1;                  // ranks per lane
  constexpr int kGroups = 32 / kLanes;                  // positions side by side
  constexpr int kPos = R > 0 ? kTileRows / kGroups : 1; // and per lane
  const int ldh = a.d + 4;
  float* hT = smem;                                     // [16][d + 4], then [8][16][R] sums
  __shared__ float swt[kTileRows];
  __shared__ int sfrom[kTileRows];
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  if (a.ids) {  // sixteen threads per position, every 16th entry each
    const int t = t0 + (tid >> 4), from = t < a.T ? a.source(t) : 0;
    bool any = false;
    if (t < a.T) {
      int id[kMaxTop / 16];
      float x[kMaxTop / 16];
#pragma unroll
      for (int q = 0; q < kMaxTop / 16; ++q) {
        const int k = (tid & 15) + 16 * q;
        const long long o = (long long)from * a.K + k;
        id[q] = k < a.K ? a.ids[o] : -1;
        x[q] = k < a.K ? a.teacher[o] : 0.f;
      }
#pragma unroll
      for (int q = 0; q < kMaxTop / 16; ++q) any |= is_entry(id[q], x[q], a.V);
    }
    const unsigned b = __ballot_sync(0xffffffffu, any) >> (lane & 16) & 0xffffu;
    if ((tid & 15) == 0) {
      const float wt = t < a.T ? row_weight(a, from, b != 0) : 0.f;
      swt[tid >> 4] = wt;
      sfrom[tid >> 4] = from;
      if (t < a.T) a.wt[t] = wt;
    }
    __syncthreads();
  }
#pragma unroll
  for (int p = 0; p < 2; ++p) {  // two rows per warp
    const int row = w + 8 * p, t = t0 + row;
    const bool in = t < a.T && (!a.ids || swt[row] != 0.f);
    const int from = !in ? 0 : a.ids ? sfrom[row] : t;
    float2 x[kMaxHead64];
#pragma unroll
    for (int k = 0; k < kMaxHead64; ++k)
      x[k] = make_float2(0.f, 0.f);
    if (in) load_row(a, from, lane, x);
    float hh = 0.f;
#pragma unroll
    for (int k = 0; k < kMaxHead64; ++k)
      if (64 * k < a.d) {
        const __half2 hv = __floats2half2_rn(x[k].x, x[k].y);
        const float2 hf = __half22float2(hv);
        if (t < a.T)
          *reinterpret_cast<__half2*>(a.h16 + (long long)t * a.d + 64 * k + 2 * lane) = hv;
        if constexpr (R > 0) *reinterpret_cast<float2*>(hT + row * ldh + 64 * k + 2 * lane) = hf;
        hh = fmaf(hf.x, hf.x, fmaf(hf.y, hf.y, hh));
      }
    if (a.hn) {
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) hh += __shfl_xor_sync(0xffffffffu, hh, off);
      if (lane == 0 && t < a.T) a.hn[t] = sqrtf(hh);
    }
  }
  if constexpr (R > 0) {
    constexpr int kRows = 12;  // of A in flight; d / 8 is a multiple of 8
    const int j = lane % kLanes, g = lane / kLanes;
    const int i_lo = a.d / 8 * w, i_hi = i_lo + a.d / 8;
    float u[kPos][kPer] = {};
    __syncthreads();
    for (int i0 = i_lo; i0 < i_hi; i0 += kRows) {
      float av[kRows][kPer];
#pragma unroll
      for (int i = 0; i < kRows; ++i)
#pragma unroll
        for (int q = 0; q < kPer; ++q)
          av[i][q] = i0 + i < i_hi && j + 32 * q < a.r
                         ? a.A[(long long)(i0 + i) * a.lda + j + 32 * q] : 0.f;
#pragma unroll
      for (int i = 0; i < kRows; i += 4) {
        if (i0 + i >= i_hi) break;
#pragma unroll
        for (int p = 0; p < kPos; ++p) {
          const float4 h = *reinterpret_cast<const float4*>(hT + (kGroups * p + g) * ldh + i0 + i);
#pragma unroll
          for (int q = 0; q < kPer; ++q)
            u[p][q] = fmaf(h.w, av[i + 3][q],
                           fmaf(h.z, av[i + 2][q],
                                fmaf(h.y, av[i + 1][q], fmaf(h.x, av[i][q], u[p][q]))));
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int p = 0; p < kPos; ++p)
#pragma unroll
      for (int q = 0; q < kPer; ++q)
        hT[(w * kTileRows + kGroups * p + g) * R + j + 32 * q] = u[p][q];
    __syncthreads();
    float umax = 0.f;
    for (int k = tid; k < kTileRows * R; k += 256) {
      const int p = k / R;
      float s = hT[k];
#pragma unroll
      for (int q = 1; q < 8; ++q) s += hT[q * kTileRows * R + k];
      if (t0 + p < a.T) put_u(a, t0 + p, k % R, s, umax, a.ids ? swt[p] : 0.f);
    }
    if (a.tok)
      for (int q = w; q < kTileRows; q += 8)
        if (t0 + q < a.Tpad) put_fields(a, t0 + q, t0 + q < a.T ? R : 0, lane, 32);
    if (a.ids) put_max(a, umax);
  }
}
__host__ __device__ inline size_t prep_tile_smem(int R, int d) {
  const size_t h = (size_t)kTileRows * (d + 4), s = (size_t)8 * kTileRows * R;
  return R == 0 ? 0 : (h > s ? h : s) * 4;
}

struct PackArgs {
  BView B;
  int V, r, R;
  long long Vpad;
  float* Bt;      // [Vpad][R], bidx layout or (Bt_plain) row by row; or null
  int Bt_plain;
  __half* waug;   // [Vpad][aug_width], or null
  int aug_layout, aug_width;
  __half* xv;     // [2R][Vpad] B^T hi / lo times 2^(exponent of stats), or null
  int* stats;
};

// Exponent e with max * 2^e in [2^to, 2^(to + 1)).
__device__ __forceinline__ int scale_exp(int max_bits, int to) {
  const float m = __int_as_float(max_bits);
  if (!(m > 0.f) || !isfinite(m)) return 0;
  return to - ilogbf(m);
}
__device__ __forceinline__ double exp2i(int e) {
  return __hiloint2double((1023 + e) << 20, 0);  // |e| < 1023
}

// The vocabulary side of the rank term for rows [v0, v0 + 64), through a tile
// [R][65] in shared memory so that both sides are read and written whole
// sectors at a time (row by row, a thread per row, it took 56 us at rank 4 and
// 370 us at rank 64 for V = 49152; this, beside the positions, 8 and 20).
constexpr int kPackRows = 64;
__device__ __forceinline__ void pack_tile(const PackArgs& a, long long v0, float* tile) {
  constexpr int ld = kPackRows + 1;
  const int R = a.R, lr = __ffs(R) - 1, tid = threadIdx.x;  // R is a power of two, 4 to 64
  const int n = R * kPackRows;                              // 256 to 4096
  // element k of the tile as [v][R] pair-interleaved: row (k >> (lr + 1)) * 2 + (k & 1)
  auto pair_row = [&](int k) { return (k >> (lr + 1) << 1) | (k & 1); };
  auto pair_col = [&](int k) { return (k & (2 * R - 1)) >> 1; };
  for (int k0 = tid; k0 < n; k0 += 8 * 256) {
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int k = k0 + 256 * e;
      const int j = a.B.layout ? pair_col(k) : k / kPackRows;
      const int i = a.B.layout ? pair_row(k) : k % kPackRows;
      x[e] = k < n && j < a.r && v0 + i < a.V ? a.B.at(j, v0 + i) : 0.f;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int k = k0 + 256 * e;
      const int j = a.B.layout ? pair_col(k) : k / kPackRows;
      const int i = a.B.layout ? pair_row(k) : k % kPackRows;
      if (k < n) tile[j * ld + i] = x[e];
    }
  }
  __syncthreads();
  if (a.Bt) {
#pragma unroll 4
    for (int k = tid; k < n; k += 256)
      a.Bt[v0 * R + k] = a.Bt_plain ? tile[(k & (R - 1)) * ld + (k >> lr)]
                                    : tile[pair_col(k) * ld + pair_row(k)];
  }
  if (a.waug) {
    const int groups = a.aug_width / 8;
    for (int k = tid; k < kPackRows * groups; k += 256) {
      const int i = k / groups, c0 = (k - i * groups) * 8;
      __align__(16) __half o[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int part = (c0 + e) >> lr, j = (c0 + e) & (R - 1);
        const bool used = part < (a.aug_layout == 1 ? 3 : 2);
        const float b = used ? tile[j * ld + i] : 0.f;
        const __half hi = __float2half_rn(b);
        o[e] = part == 1 ? __float2half_rn(b - __half2float(hi)) : hi;  // [hi | lo | hi], [hi | lo]
      }
      *reinterpret_cast<uint4*>(a.waug + (v0 + i) * a.aug_width + c0) =
          *reinterpret_cast<const uint4*>(o);
    }
  }
  if (a.xv) {
    const double up = exp2i(scale_exp(a.stats[kStBMax], 13));  // past f32 for a tiny B
#pragma unroll 2
    for (int k = tid; k < R * (kPackRows / 2); k += 256) {
      const int j = k / (kPackRows / 2), i = 2 * (k % (kPackRows / 2));
      const float x = (float)((double)tile[j * ld + i] * up);
      const float y = (float)((double)tile[j * ld + i + 1] * up);
      const __half2 hi = __floats2half2_rn(x, y);
      const float2 hf = __half22float2(hi);
      const long long o = (long long)j * a.Vpad + v0 + i;
      *reinterpret_cast<__half2*>(a.xv + o) = hi;
      *reinterpret_cast<__half2*>(a.xv + (long long)R * a.Vpad + o) =
          __floats2half2_rn(x - hf.x, y - hf.y);
    }
  }
}

// What the errors of logits are measured by (logit_gaps): the largest |W[v]| and
// |B[:, v]| of kNormBlocks runs of up to kNormRows vocab rows, spread over the vocabulary
// (all of up to 1,024), and the largest |A[:, j]|.  All of W, 57 MB, would take longer
// than the rest of a short call's preparation (one token 29 -> 42 us).
constexpr int kNormBlocks = 32, kNormRows = 32;
struct NormArgs {
  const __half* W;
  int V, d;
  BView B;
  const float* A;
  int lda, r;
  float* out;  // [kNormBlocks] W, [kNormBlocks] B, A; or null: not wanted
};
__device__ __forceinline__ void norm_block(const NormArgs& a, int blk) {
  __shared__ double red[256];
  __shared__ float redW[8];
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  int n;  // columns (of A, of B): their squares are split over threads tid % n
  double s = 0.0;
  if (blk >= kNormBlocks) {
    n = a.r > 32 ? 64 : a.r > 16 ? 32 : 16;
    const int j = tid % n;
    if (j < a.r)
#pragma unroll 16
      for (int i = tid / n; i < a.d; i += 256 / n) {
        const double x = (double)a.A[(long long)i * a.lda + j];
        s = fma(x, x, s);
      }
  } else {
    n = kNormRows;
    const int v_lo = (int)((long long)a.V * blk / kNormBlocks);
    const int v_hi = min((int)((long long)a.V * (blk + 1) / kNormBlocks), v_lo + kNormRows);
    // eight lanes per row of W, whole sectors, all of it and of B at once
    const int vw = v_lo + (tid >> 3), vb = v_lo + tid % n;
    uint4 x[kMaxHead64];
#pragma unroll
    for (int k = 0; k < kMaxHead64; ++k)
      x[k] = 64 * k < a.d && vw < v_hi
                 ? reinterpret_cast<const uint4*>(a.W + (long long)vw * a.d)[(tid & 7) + 8 * k]
                 : make_uint4(0u, 0u, 0u, 0u);
    if (vb < v_hi)
#pragma unroll 8
      for (int j = tid / n; j < a.r; j += 256 / n) {
        const double y = (double)a.B.at(j, vb);
        s = fma(y, y, s);
      }
    float q = 0.f;
#pragma unroll
    for (int k = 0; k < kMaxHead64; ++k) {
      const __half2* h = reinterpret_cast<const __half2*>(&x[k]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 y = __half22float2(h[e]);
        q = fmaf(y.x, y.x, fmaf(y.y, y.y, q));
      }
    }
    for (int off = 1; off < 8; off <<= 1) q += __shfl_xor_sync(0xffffffffu, q, off);
    q = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(q)));
    if (lane == 0) redW[w] = q;
  }
  red[tid] = s;
  __syncthreads();
  if (w != 0) return;
  double top = 0.0;
  for (int c = lane; c < n; c += 32) {
    double x = 0.0;
    for (int k = c; k < 256; k += n) x += red[k];
    top = fmax(top, x);
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, off));
  if (lane != 0) return;
  a.out[kNormBlocks + blk] = (float)sqrt(top);
  if (blk < kNormBlocks) {
    float q = redW[0];
    for (int k = 1; k < 8; ++k) q = fmaxf(q, redW[k]);
    a.out[blk] = sqrtf(q);
  }
}

// Blocks [0, norm_blocks) take norms, the next prep_blocks positions (kRank < 0: one
// each; else kTileRows at kernel rank kRank), the next max_blocks look for the largest
// finite |B| (the scale of a later launch's xv), the others pack vocab rows.
template <int kRank>
static __global__ void __launch_bounds__(256) lh_prep(PrepArgs a, PackArgs b, NormArgs n,
                                                      int norm_blocks, int prep_blocks,
                                                      int max_blocks) {
  extern __shared__ __align__(16) float smem_prep[];
  const int blk = (int)blockIdx.x - norm_blocks;
  grid_launch();  // (a kernel launched to depend waits for this one's end)
  if (blk < 0) {
    norm_block(n, blk + norm_blocks);
  } else if (blk < prep_blocks) {
    if (blk == 0 && threadIdx.x == 0 && !a.ids) a.stats[kStErr] = 0;
    if constexpr (kRank < 0) prep_row(a, blk, smem_prep);
    else prep_tile<kRank>(a, blk * kTileRows, smem_prep);
  } else if (blk < prep_blocks + max_blocks) {
    float m = 0.f;
    const long long size = b.B.layout ? b.Vpad * b.R : (long long)b.r * b.V;  // (padding is 0)
    const long long step = (long long)max_blocks * 256;
#pragma unroll 8
    for (long long k = (long long)(blk - prep_blocks) * 256 + threadIdx.x; k < size; k += step) {
      const float x = fabsf(b.B.p[k]);
      m = isfinite(x) ? fmaxf(m, x) : m;
    }
    const unsigned w = __reduce_max_sync(0xffffffffu, __float_as_uint(m));
    if ((threadIdx.x & 31) == 0 && w)
      atomicMax(reinterpret_cast<unsigned*>(b.stats) + kStBMax, w);
  } else {
    pack_tile(b, (long long)(blk - prep_blocks - max_blocks) * kPackRows,
              smem_prep);
  }
}

// Order of floats as order of unsigned words (-inf lowest, above 0).
__device__ __forceinline__ unsigned order_key(float x) {
  const unsigned u = __float_as_uint(x);
  return (u >> 31) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_float(unsigned k) {
  return __uint_as_float((k >> 31) ? (k & 0x7fffffffu) : ~k);
}

// ------------------------------------------------------------- logits again
struct LogitArgs {
  const __half* W;
  const __half* h16;
  const float* sU;  // [T][R]
  // the rank term as the passes' MMA has it (null: from sU and B)
  const __half* haug;
  const __half* waug;
  int aug_layout, aug_width;
  const float* A;   // for logit64
  int lda;
  float scale;
  BView B;
  int T, V, d, r, R;
};

// Logits of 16 vocab ids (ids[min(i, n - 1)]) of position t, by one warp: mma
// with the rows of W as A and h as the first column of B, the rank term's f16
// halves (waug, haug) behind them.  Lane c = lane % 4 takes 8 consecutive elements
// of each 32 as its share of two K-steps (any order of K will do, as long as both
// operands have it), so W is read 16 bytes at a time.
// kSum64: each 32 products are added up in a fresh accumulator, whose known loss
// (kLoss32, as acc_short) is small and made good, and go to a 64-bit sum: off by
// 5e-7 (1 + |z|) at most over 524,288 logits at hidden sizes 576 and 64, ranks
// 0, 4 and 64.  About 250 instructions for 16 logits; with every product in 64
// bits it is 1,600.  Else one f32 accumulator: to compare with a bound.
constexpr double kLoss32 = 0.79 * 1.5 / 33554432.0 * 1.4426950408889634;
template <bool kSum64, class Out>
__device__ __forceinline__ void logits16(const LogitArgs& a, int t, const int* ids, int n, int lane,
                                         Out* out, int part = 0, int parts = 1) {
  constexpr int kBatch = 6;
  const int c = lane & 3, g = lane >> 2;
  const long long v0 = ids[min(g, n - 1)], v1 = ids[min(g + 8, n - 1)];
  double z0 = 0.0, z1 = 0.0;
  float d[4] = {0.f, 0.f, 0.f, 0.f};
  auto mma = [&](unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, "
        "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  };
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  auto add = [&](uint4 p, uint4 q, uint4 x) {
    mma(p.x, q.x, p.y, q.y, x.x, x.y);
    mma(p.z, q.z, p.w, q.w, x.z, x.w);
    if constexpr (kSum64) {
      z0 += (double)d[0];
      z1 += (double)d[2];
      d[0] = d[1] = d[2] = d[3] = 0.f;
    }
  };
  {
    // six steps' rows at a time in flight: one after another, each would wait
    // for the L2
    const __half* w0 = a.W + v0 * a.d + 8 * c;
    const __half* w1 = a.W + v1 * a.d + 8 * c;
    const __half* h = a.h16 + (long long)t * a.d + 8 * c;
    const int steps = a.d / 32, k_hi = steps * (part + 1) / parts * 32;
    for (int k0 = steps * part / parts * 32; k0 < k_hi; k0 += 32 * kBatch) {
      uint4 p[kBatch], q[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        p[i] = q[i] = zero;
        if (k0 + 32 * i < k_hi) {
          p[i] = *reinterpret_cast<const uint4*>(w0 + k0 + 32 * i);
          q[i] = *reinterpret_cast<const uint4*>(w1 + k0 + 32 * i);
        }
      }
      asm volatile("" ::: "memory");  // all of them issued before the first is used
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        uint4 x = zero;
        if (g == 0 && k0 + 32 * i < k_hi) x = *reinterpret_cast<const uint4*>(h + k0 + 32 * i);
        add(p[i], q[i], x);
      }
    }
  }
  auto row16 = [&](const __half* p, bool in) {
    return in ? *reinterpret_cast<const uint4*>(p) : zero;
  };
  const bool last = part == parts - 1;  // the rank term's
  if (a.waug && last) {
    const __half* w0 = a.waug + v0 * a.aug_width + 8 * c;
    const __half* w1 = a.waug + v1 * a.aug_width + 8 * c;
    const __half* h = a.haug + (long long)t * a.aug_width + 8 * c;
    if (a.aug_layout == 1) {
#pragma unroll 2
      for (int k = 0; k < a.aug_width; k += 32) {
        const bool in = k + 8 * c < a.aug_width;
        add(row16(w0 + k, in), row16(w1 + k, in), row16(h + k, in && g == 0));
      }
    } else {  // hi . hi, lo . hi, hi . lo
#pragma unroll 2
      for (int k = 0; k < a.R; k += 32) {
        const uint4 hi0 = row16(w0 + k, true), hi1 = row16(w1 + k, true);
        const uint4 lo0 = row16(w0 + a.R + k, true), lo1 = row16(w1 + a.R + k, true);
        const uint4 x = row16(h + k, g == 0), y = row16(h + a.R + k, g == 0);
        add(hi0, hi1, x);
        add(lo0, lo1, x);
        add(hi0, hi1, y);
      }
    }
  }
  if constexpr (!kSum64) {
    z0 = d[0];
    z1 = d[2];
  }
  // lane 4 g has rows g and g + 8
  const double a0 = __shfl_sync(0xffffffffu, z0, 4 * (lane & 7));
  const double a1 = __shfl_sync(0xffffffffu, z1, 4 * (lane & 7));
  const int i = lane & 15;
  double z = i < 8 ? a0 : a1;
  if constexpr (kSum64) z = fma(z, kLoss32, z);
  if (!a.waug && a.r > 0 && last) {  // lane i % 16 takes row i, the halves of the warp every other rank
    const int v = ids[min(i, n - 1)];
    const float* su = a.sU + (long long)t * a.R;
    float s = 0.f;
#pragma unroll 8
    for (int j = lane >> 4; j < a.r; j += 2) s = fmaf(su[j], a.B.at(j, v), s);
    s += __shfl_xor_sync(0xffffffffu, s, 16);
    z += (double)s;
  }
  if (lane < 16 && i < n) out[i] = (Out)z;
}

__device__ __forceinline__ double warp_sum(double s) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
  return s;
}

// One logit by one warp with 64-bit sums throughout (products of f16 are exact in
// f32): for those whose order logits16 does not tell.  u: scale U[t], from u64.
__device__ __forceinline__ double logit64(const LogitArgs& a, int t, int v, const double* u,
                                          int lane) {
  const __half* h = a.h16 + (long long)t * a.d;
  const __half* w = a.W + (long long)v * a.d;
  double z = 0.0;
#pragma unroll
  for (int k = 0; k < kMaxHead64; ++k)
    if (64 * k < a.d) {
      const float2 x = __half22float2(*reinterpret_cast<const __half2*>(h + 64 * k + 2 * lane));
      const float2 y = __half22float2(*reinterpret_cast<const __half2*>(w + 64 * k + 2 * lane));
      z += (double)(x.x * y.x) + (double)(x.y * y.y);
    }
  for (int j = lane; j < a.r; j += 32) z = fma(u[j], (double)a.B.at(j, v), z);
  return warp_sum(z);
}

// ------------------------------------------------------------- teams
// The per-row kernels give a position to one warp, or, where positions are too
// few to fill the SMs with warps, to a block of four or eight.
template <int TW>
struct Team {
  static constexpr int kThreads = 32 * TW;
  int tid, lane, w;
  double* red;  // TW > 1: 4 x TW doubles of shared memory
  int parity = 0;
  __device__ __forceinline__ void sync() const {
    if constexpr (TW == 1) __syncwarp();
    else __syncthreads();
  }
  template <class T, class F>
  __device__ __forceinline__ T reduce(T x, F f) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) x = f(x, __shfl_xor_sync(0xffffffffu, x, off));
    if constexpr (TW > 1) {
      T* b = reinterpret_cast<T*>(red + 2 * TW * parity);
      parity ^= 1;
      if (lane == 0) b[w] = x;
      __syncthreads();
      x = b[0];
#pragma unroll
      for (int i = 1; i < TW; ++i) x = f(x, b[i]);
    }
    return x;
  }
  __device__ __forceinline__ double sum(double x) {
    return reduce(x, [](double p, double q) { return p + q; });
  }
  __device__ __forceinline__ double2 sum2(double x, double y) {
    x = warp_sum(x);
    y = warp_sum(y);
    if constexpr (TW > 1) {
      double* b = red + 2 * TW * parity;
      parity ^= 1;
      if (lane == 0) {
        b[2 * w] = x;
        b[2 * w + 1] = y;
      }
      __syncthreads();
      x = y = 0.0;
#pragma unroll
      for (int i = 0; i < TW; ++i) {
        x += b[2 * i];
        y += b[2 * i + 1];
      }
    }
    return make_double2(x, y);
  }
  __device__ __forceinline__ int count(int x) {
    x = __reduce_add_sync(0xffffffffu, x);
    if constexpr (TW > 1) {
      int* b = reinterpret_cast<int*>(red + 2 * TW * parity);
      parity ^= 1;
      if (lane == 0) b[w] = x;
      __syncthreads();
      x = 0;
#pragma unroll
      for (int i = 0; i < TW; ++i) x += b[i];
    }
    return x;
  }
  __device__ __forceinline__ float max_f(float x) {
    return reduce(x, [](float p, float q) { return fmaxf(p, q); });
  }
};

// u = scale U[t] [r] with 64-bit sums: each warp takes some of the ranks, its lanes
// neighbouring ones (A is read in whole sectors) and every n-th row of A.  A lane
// per row instead, each rank of each logit anew, took 100 us for two logits at
// rank 50.
template <int TW>
__device__ __forceinline__ void u64(const LogitArgs& a, int t, const Team<TW>& team, double* u) {
  const __half* h = a.h16 + (long long)t * a.d;
  const int per = (a.r + TW - 1) / TW;
  for (int j0 = per * team.w; j0 < min(a.r, per * (team.w + 1)); j0 += 32) {
    const int n = min(32, min(a.r, per * (team.w + 1)) - j0);
    const int span = n == 1 ? 1 : 1 << (32 - __clz(n - 1)), j = team.lane & (span - 1);
    const float* A = a.A + j0 + min(j, n - 1);
    double s = 0.0;
#pragma unroll 16
    for (int i = team.lane / span; i < a.d; i += 32 / span)
      s = fma((double)__half2float(h[i]), (double)A[(long long)i * a.lda], s);
    for (int off = span; off < 32; off <<= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    if (team.lane < n) u[j0 + j] = (double)a.scale * s;
  }
  team.sync();
}

// Where the partial sums of a position sit: pass 1 over n_b column tiles,
// 256-position blocks, tiles split over at most `units` owners.
struct SlotPlan {
  int cparts, n_a, n_b, units;
  long long ld;  // row stride of the partial arrays
  const float* p_max;
  const float* p_sum;
  const float* p_ent;
  const float* p_q;
  __device__ __forceinline__ int slots(int t) const { return slots_of(t / (2 * kBM)); }
  __device__ __forceinline__ int slots_of(int ab) const {
    // tile_owner in 32 bits: at most 4096 x 2048 tiles, 148 units (few positions:
    // 4096 of each)
    const unsigned first = (unsigned)ab * n_b, total = (unsigned)n_a * n_b;
    const unsigned G = min(total, (unsigned)units);
    const unsigned s0 = ((first + 1) * G - 1) / total, s1 = ((first + n_b) * G - 1) / total;
    return cparts * (int)(s1 - s0 + 1);
  }
};

struct RowSum {
  float M;      // reference max, log2 units (as rounded in the sums' exponents)
  double S, E;  // sum of 2^x, sum of 2^x * x, x from M
};

// A row's slots merged in a fixed order.  A thread keeps its first ones in
// registers from the maximum to the sums: a second read is a second wait.
template <bool kEnt, int TW>
__device__ __forceinline__ RowSum merge_row(const SlotPlan& p, int t, int nslot, Team<TW>& team) {
  constexpr int kKeep = TW == 1 ? 1 : 4;
  float pm[kKeep], s[kKeep], e[kKeep];
  float M = -INFINITY;
#pragma unroll
  for (int i = 0; i < kKeep; ++i) {
    const int k = team.tid + i * team.kThreads;
    const long long o = (long long)k * p.ld + t;
    pm[i] = k < nslot ? p.p_max[o] : -INFINITY;
    s[i] = k < nslot ? p.p_sum[o] : 0.f;
    e[i] = kEnt && k < nslot ? p.p_ent[o] : 0.f;
  }
#pragma unroll
  for (int i = 0; i < kKeep; ++i) M = fmaxf(M, pm[i]);
#pragma unroll 2
  for (int k = team.tid + kKeep * team.kThreads; k < nslot; k += team.kThreads)
    M = fmaxf(M, p.p_max[(long long)k * p.ld + t]);
  M = team.max_f(M);
  double S = 0.0, E = 0.0;
  auto add = [&](float m, float sum, float ent) {
    if (m == -INFINITY && sum == 0.f) return;  // a slice that saw no valid column
    const float x = m - M, f = exp2f(x);
    S += (double)(sum * f);
    if constexpr (kEnt) E += (double)(f * fmaf(x, sum, ent));
  };
#pragma unroll
  for (int i = 0; i < kKeep; ++i) add(pm[i], s[i], e[i]);
#pragma unroll 2
  for (int k = team.tid + kKeep * team.kThreads; k < nslot; k += team.kThreads) {
    const long long o = (long long)k * p.ld + t;
    add(p.p_max[o], p.p_sum[o], kEnt ? p.p_ent[o] : 0.f);
  }
  if constexpr (kEnt) {
    const double2 both = team.sum2(S, E);
    S = both.x;
    E = both.y;
  } else {
    S = team.sum(S);
  }
  return RowSum{M, S, E};
}

// logits16 of n ids to z.  A team of several warps shares a group of 16 where there
// are few: each warp takes part of the hidden size (zp: 16 TW partial sums).
template <int TW>
__device__ __forceinline__ void team_logits(const LogitArgs& a, int t, const int* ids, int n,
                                            const Team<TW>& team, double* z, double* zp) {
  const int groups = (n + 15) / 16;
  if (TW == 1 || 2 * groups > TW) {
    for (int c = 16 * team.w; c < n; c += 16 * TW)
      logits16<true>(a, t, ids + c, min(16, n - c), team.lane, z + c);
    team.sync();
  } else if (groups > 0) {
    const int parts = TW / groups, g = team.w / parts;
    if (g < groups)
      logits16<true>(a, t, ids + 16 * g, min(16, n - 16 * g), team.lane, zp + 16 * team.w,
                     team.w - g * parts, parts);
    team.sync();
    for (int c = team.tid; c < n; c += team.kThreads) {
      double s = 0.0;
      for (int q = 0; q < parts; ++q) s += zp[16 * ((c >> 4) * parts + q) + (c & 15)];
      z[c] = s;
    }
    team.sync();
  }
}

// ------------------------------------------------------------- few positions
enum FewMode { kFewScore, kFewLoss, kFewForward, kFewBackward };
struct FewArgs {
  const __half* W;
  const __half* h16;
  const float* sU;  // [T][R]
  BView B;
  int T, V, d, r, R;
  float lg;
  // forward: one slot per block
  long long ld;  // row stride of the partials
  float* p_max;
  float* p_sum;
  float* p_ent;
  float* p_q;
  // score: records of 64 columns
  float* sub_max;
  float* sub_second;
  float* sub_rest;
  uint8_t* sub_arg;
  uint8_t* sub_arg2;
  int n_sub;
  // backward
  const float2* ref;               // [T] reference max (log2), weight * tau / sum
  const unsigned long long* corr;  // [Vpad][R], row by row
  const float* dU;                 // [T][R]
  const int* stats;
  int v_blocks;  // the blocks behind them form gA
  float* gA;
  float* gB;
  int layout;
  long long Vpad;
  const float* loss;
  const float* wt;
  float* tail;
};
constexpr int kFewRows = 128;           // vocab rows per block, 16 per warp
constexpr int kFewLdZ = kFewRows + 4;   // floats per position of the logit tile
__host__ __device__ constexpr int few_ldh(int d) { return d + 32; }  // f16 per position
__host__ __device__ inline size_t few_front(int NT, int d) {
  const size_t h = (size_t)8 * NT * few_ldh(d) * 2, z = (size_t)8 * NT * kFewLdZ * 4;
  return h > z ? h : z;
}
__host__ __device__ inline size_t few_smem(int NT, int d, int R) {
  return few_front(NT, d) + (size_t)(8 * NT + kFewLdZ) * R * 4;
}

// Sum of losses and number of counted positions, by one block of 256.
__device__ __forceinline__ void put_tail(const float* loss, const float* wt, int T, float* tail) {
  __shared__ double red[256];
  __shared__ int cnt[256];
  const int tid = threadIdx.x;
  double s = 0.0;
  int c = 0;
  for (int t = tid; t < T; t += 256) {
    s += (double)loss[t];
    c += wt[t] != 0.f;
  }
  red[tid] = s;
  cnt[tid] = c;
  __syncthreads();
  for (int w = 128; w > 0; w >>= 1) {
    if (tid < w) {
      red[tid] += red[tid + w];
      cnt[tid] += cnt[tid + w];
    }
    __syncthreads();
  }
  if (tid == 0) {
    tail[0] = (float)red[0];
    tail[1] = (float)cnt[0];
  }
}

// The pass over z for up to 8 NT positions, bound by reading W once: a warp takes
// 16 vocab rows as A of mma (16 bytes per lane and row at a time, as logits16)
// and the positions as B, from shared memory; every 32 products have their own
// accumulator (kLoss32).  The rank term from B as it is, so that nothing of the
// vocabulary's side is packed.  Then the block's logits, in shared memory, give
//   score: the same partial sums and records as EpiScore<64>, one slot per block;
//   distill forward: partial sums, and with gradients those of p B^T;
//   distill backward: gB of the block's rows, whole: all positions are here, so
//   there are no partial gradients to write and join.  More blocks form gA.
// The tensor-core passes take 26 and 20 us for 1 to 256 positions (V = 49152, rank
// 4: three tiles per SM, each with an epilogue over 256 rows), and 10 more to pack
// B and to join the partial gradients.  This one: 13 us for up to 8 positions, 20 to
// 25 for 32, by when the mma and their operands' reads from shared memory, once per
// 16 vocab rows, take as long as W.
template <int NT, int kMode>
static __global__ void __launch_bounds__(256, 3) lh_few(FewArgs a) {
  constexpr int kUnroll = 6;
  constexpr unsigned kAll = 0xffffffffu;
  extern __shared__ __align__(16) uint8_t smem_few[];
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, c = lane & 3, g = lane >> 2;
  const int ldh = few_ldh(a.d);
  if (kMode == kFewBackward && (int)blockIdx.x >= a.v_blocks) {
    grid_wait();
    const int blk = (int)blockIdx.x - a.v_blocks, ra = a.layout ? a.R : a.r;
    const int k = blk * 256 + tid;
    if (k < a.d * ra) {
      const int i = k / ra, j = k - i * ra;
      float s = 0.f;
#pragma unroll 8
      for (int t = 0; t < a.T; ++t)
        s = fmaf(__half2float(a.h16[(long long)t * a.d + i]), a.dU[(long long)t * a.R + j], s);
      a.gA[k] = s;
    }
    if (a.tail && blk == 0) put_tail(a.loss, a.wt, a.T, a.tail);
    return;
  }
  __half* sh = reinterpret_cast<__half*>(smem_few);
  float* sz = reinterpret_cast<float*>(smem_few);  // over h once that is used up
  float* su = reinterpret_cast<float*>(smem_few + few_front(NT, a.d));
  float* sb = su + 8 * NT * a.R;                   // [R][kFewLdZ]
  const int v0 = (int)blockIdx.x * kFewRows;
  const __half* w0 = a.W + (long long)min(v0 + 16 * w + g, a.V - 1) * a.d + 8 * c;
  const __half* w1 = a.W + (long long)min(v0 + 16 * w + g + 8, a.V - 1) * a.d + 8 * c;
  uint4 p[kUnroll], q[kUnroll];
  auto fetch = [&](int k0) {
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      const int k = k0 + 32 * i;
      p[i] = q[i] = make_uint4(0u, 0u, 0u, 0u);
      if (k < a.d) {
        p[i] = *reinterpret_cast<const uint4*>(w0 + k);
        q[i] = *reinterpret_cast<const uint4*>(w1 + k);
      }
    }
  };
  fetch(0);  // W and B are the caller's: their reads need not wait for the kernel ahead
  {
    const int i = tid & (kFewRows - 1);
    for (int j = tid / kFewRows; j < a.R; j += 2) {
      const bool in = j < a.r && v0 + i < a.V;
      const float* src = in ? a.B.p + (a.B.layout ? bidx(v0 + i, j, a.R) : (long long)j * a.V + v0 + i)
                            : a.B.p;
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(
                       (unsigned)__cvta_generic_to_shared(sb + j * kFewLdZ + i)),
                   "l"(src), "r"(in ? 4 : 0) : "memory");
    }
  }
  grid_wait();
  if (kMode != kFewBackward) grid_launch();
  for (int t = w; t < 8 * NT; t += 8) {
    for (int i = 8 * lane; i < a.d; i += 256) {
      uint4 x = make_uint4(0u, 0u, 0u, 0u);
      if (t < a.T) x = *reinterpret_cast<const uint4*>(a.h16 + (long long)t * a.d + i);
      *reinterpret_cast<uint4*>(sh + t * ldh + i) = x;
    }
  }
  for (int k = tid; k < 8 * NT * a.R; k += 256) su[k] = k < a.T * a.R ? a.sU[k] : 0.f;
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
  float z[NT][4] = {};
  for (int k0 = 0; k0 < a.d; k0 += 32 * kUnroll) {
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      const int k = k0 + 32 * i;
      if (k < a.d) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const uint4 x = *reinterpret_cast<const uint4*>(sh + (8 * n + g) * ldh + k + 8 * c);
          float d[4];
          asm volatile(
              "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, "
              "{%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
              : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
              : "r"(p[i].x), "r"(q[i].x), "r"(p[i].y), "r"(q[i].y), "r"(x.x), "r"(x.y), "f"(0.f));
          asm volatile(
              "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, "
              "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
              : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
              : "r"(p[i].z), "r"(q[i].z), "r"(p[i].w), "r"(q[i].w), "r"(x.z), "r"(x.w));
#pragma unroll
          for (int e = 0; e < 4; ++e) z[n][e] += d[e];
        }
      }
    }
    if (k0 + 32 * kUnroll < a.d) fetch(k0 + 32 * kUnroll);
  }
  __syncthreads();
  // lane (g, c): rows g, g + 8 of positions 2 c, 2 c + 1
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      sz[(8 * n + 2 * c + (e & 1)) * kFewLdZ + 16 * w + g + 8 * (e >> 1)] = z[n][e];
  __syncthreads();
  const int vi = tid & (kFewRows - 1), t0 = tid / kFewRows;
  if (a.r > 0) {  // thread: one vocab row, every other position
    float s[4 * NT] = {};
    for (int j = 0; j < a.r; j += 4) {  // R is a multiple of 4, the rest is 0
      float b[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) b[e] = sb[(j + e) * kFewLdZ + vi];
#pragma unroll
      for (int n = 0; n < 4 * NT; ++n) {
        const float4 u = *reinterpret_cast<const float4*>(su + (2 * n + t0) * a.R + j);
        s[n] = fmaf(u.x, b[0], fmaf(u.y, b[1], fmaf(u.z, b[2], fmaf(u.w, b[3], s[n]))));
      }
    }
#pragma unroll
    for (int n = 0; n < 4 * NT; ++n) sz[(2 * n + t0) * kFewLdZ + vi] += s[n];
    __syncthreads();
  }
  if constexpr (kMode == kFewBackward) {
    // dz = p weight tau, then gB = dz^T (scale U) over all positions, less the
    // entries' part
    for (int t = w; t < 8 * NT; t += 8) {
      const float2 ref = t < a.T ? a.ref[t] : make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float& x = sz[t * kFewLdZ + lane + 32 * i];
        x = ref.y == 0.f ? 0.f : ex2f(fmaf(x, a.lg, -ref.x)) * ref.y;
      }
    }
    __syncthreads();
    const double fx = exp2i(-scale_exp(a.stats[kStUMax], 37));
    const int v = v0 + vi, T = a.T;
    for (int j = 4 * t0; j < a.R; j += 8) {
      float s[4] = {};
      unsigned long long sparse[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        sparse[e] = v < a.V ? a.corr[(long long)v * a.R + j + e] : 0ull;
#pragma unroll 4
      for (int t = 0; t < T; ++t) {
        const float x = sz[t * kFewLdZ + vi];
        const float4 u = *reinterpret_cast<const float4*>(su + t * a.R + j);
        s[0] = fmaf(x, u.x, s[0]);
        s[1] = fmaf(x, u.y, s[1]);
        s[2] = fmaf(x, u.z, s[2]);
        s[3] = fmaf(x, u.w, s[3]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = (float)((double)s[e] - (double)(long long)sparse[e] * fx);
        if (a.layout) {
          if (v < a.Vpad) a.gB[bidx(v, j + e, a.R)] = v < a.V ? x : 0.f;
        } else if (j + e < a.r && v < a.V) {
          a.gB[(long long)(j + e) * a.V + v] = x;
        }
      }
    }
  } else {
    // a warp per position: partial sums of the block's rows; score: two records
    for (int t = w; t < a.T; t += 8) {
      float x[4];
      float m = -INFINITY;
  #pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = v0 + lane + 32 * i < a.V ? sz[t * kFewLdZ + lane + 32 * i] : -INFINITY;
        m = fmaxf(m, x[i]);
      }
  #pragma unroll
      for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(kAll, m, off));
      const float mL = m * a.lg;
      float S = 0.f, E = 0.f;
  #pragma unroll
      for (int i = 0; i < 4; ++i) {
        // past the vocabulary e = 0 and e * y = 0, not 0 * inf
        const float y = v0 + lane + 32 * i < a.V ? fmaf(x[i], a.lg, -mL) : -1e30f, e = ex2f(y);
        S += e;
        if (kMode == kFewScore) E = fmaf(e, y, E);
        if (kMode == kFewForward) sz[t * kFewLdZ + lane + 32 * i] = e;
      }
  #pragma unroll
      for (int off = 16; off > 0; off >>= 1) {
        S += __shfl_xor_sync(kAll, S, off);
        if (kMode == kFewScore) E += __shfl_xor_sync(kAll, E, off);
      }
      if (lane == 0) {
        const long long o = (long long)blockIdx.x * a.ld + t;
        a.p_max[o] = mL;
        a.p_sum[o] = S;
        if (kMode == kFewScore) a.p_ent[o] = E;
      }
      if constexpr (kMode == kFewScore) {
  #pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int rec = v0 / 64 + half;
          if (rec >= a.n_sub) break;
          // the three largest, equal ones by column: columns lane and lane + 32
          unsigned k0 = order_key(x[2 * half]), k1 = order_key(x[2 * half + 1]);
          unsigned top[3];
          int at[3];
  #pragma unroll
          for (int q3 = 0; q3 < 3; ++q3) {
            top[q3] = __reduce_max_sync(kAll, max(k0, k1));
            at[q3] = (int)__reduce_min_sync(kAll, k0 == top[q3]   ? (unsigned)lane
                                                  : k1 == top[q3] ? (unsigned)lane + 32u : 64u);
            if (at[q3] == lane) k0 = 0u;
            if (at[q3] == lane + 32) k1 = 0u;
          }
          if (lane == 0) {
            const long long o = sub_idx(t, rec, a.n_sub);
            a.sub_max[o] = key_float(top[0]);
            a.sub_second[o] = key_float(top[1]);
            a.sub_rest[o] = key_float(top[2]);
            a.sub_arg[o] = (uint8_t)at[0];
            a.sub_arg2[o] = (uint8_t)at[1];
          }
        }
      }
    }
    if constexpr (kMode == kFewForward) {  // sum of e B[j] for each position and rank
      __syncthreads();
      for (int k = tid; k < a.T * a.R; k += 256) {
        const int t = k / a.R, j = k & (a.R - 1);
        const float4* x = reinterpret_cast<const float4*>(sz + t * kFewLdZ);
        const float4* b = reinterpret_cast<const float4*>(sb + j * kFewLdZ);
        float s[4] = {};
  #pragma unroll 8
        for (int i = 0; i < kFewRows / 4; ++i) {
          const float4 e = x[i], y = b[i];
          s[0] = fmaf(e.x, y.x, s[0]);
          s[1] = fmaf(e.y, y.y, s[1]);
          s[2] = fmaf(e.z, y.z, s[2]);
          s[3] = fmaf(e.w, y.w, s[3]);
        }
        a.p_q[((long long)blockIdx.x * a.ld + t) * a.R + j] = (s[0] + s[1]) + (s[2] + s[3]);
      }
    }
  }
}

// ------------------------------------------------------------- score, per row
struct ScoreArgs {
  LogitArgs z;
  const float* norms;  // NormArgs::out, PrepArgs::hn (with alternatives)
  const float* hn;
  int steps;           // the MMA steps of a logit of the pass
  SlotPlan p;
  float lg;
  int n_sub, sub, top_k;  // records, columns per record
  int n_pick;             // max(top_k, kMinPick), at most n_sub
  int cap;                // candidates that fit
  const float* sub_max;
  const float* sub_second;
  const float* sub_rest;
  const uint8_t* sub_arg;
  const uint8_t* sub_arg2;
  const int32_t* tokens;
  const int* stats;
  float* logprob;
  float* entropy;
  int32_t* top_ids;
  float* top_logprobs;
};

// Shared memory of one team: reductions and shares of logits (several warps); per
// candidate, the given token first [cap]: its logit, id, the pass's logit, that one
// made good, its rank; per picked record its number, its second and rest, its
// columns; 64 columns' ids and logits; counters.  A multiple of 16 bytes.
__host__ __device__ inline int score_picks(int n_pick) { return n_pick + kPickSlack; }
__host__ __device__ inline size_t score_team_smem(int n_pick, int cap, int warps) {
  return ((size_t)(warps == 1 ? 0 : 20 * warps) * 8 + (size_t)cap * 24 +
          (size_t)score_picks(n_pick) * 16 + 128 * 4 + 16 * 4 + 15) / 16 * 16;
}
constexpr int kScoreRows = 4;  // positions per block where each has a warp

// How far apart two logits of position t have to be for their order to be told, by a
// warp.  A sum's rounding follows its partial sums, not the logit, and these are at
// most g = |h| max |W[v]| + |s U| max |B[:, v]|, as channels that cancel show: hidden
// states whose partial sums were 50 times their logits had alternatives out of order
// when this went by the logit.
//   pass: each of its n MMA steps cuts off less than a unit in the last place of a
//         partial sum, half of one on average and that 2^-24 of the sum at most, always
//         towards zero: sums of g all along would lose n 2^-24 g more than sums near 0
//   again: logits16's sums of 32 products, at most two such losses each, come to
//         2 2^-23 g by Cauchy and Schwarz; the largest error measured is 1.8 2^-23 g
// Both have s U rounded to f32: sums of up to 80 terms with a standard deviation of
// about 2^-23 |h| |A[:, j]|, for which 8 2^-23 |h| |A[:, j]| max |B[:, v]| is taken; and
// where the rank term is of f16 pairs, what these leave out: 2^-25 of each s U[j] and
// B[j][v] and 2^-21 of their product.
struct Gaps {
  float pass, again;
};
// What a lane reads for them, and the gaps: apart, so that the reads are on their way
// beside others.
struct GapReads {
  float h, w, b, A, u;
};
__device__ __forceinline__ GapReads read_gaps(const LogitArgs& z, const float* norms,
                                              const float* hn, int t, int lane) {
  const float* su = z.sU + (long long)t * z.R;
  const float u1 = lane < z.r ? fabsf(su[lane]) : 0.f;
  const float u2 = lane + 32 < z.r ? fabsf(su[lane + 32]) : 0.f;
  return GapReads{hn[t], norms[lane], norms[kNormBlocks + lane],
                  z.r > 0 ? norms[2 * kNormBlocks] : 0.f, fmaxf(u1, u2)};
}
__device__ __forceinline__ Gaps logit_gaps(const LogitArgs& z, const GapReads& x, int steps) {
  auto most = [&](float y) {  // y >= 0
    return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(y)));
  };
  float g = x.h * most(x.w), e = 0.f;
  if (z.r > 0) {
    const float root = sqrtf((float)z.r), b = most(x.b), u = root * most(x.u);  // >= |s U|
    g = fmaf(u, b, g);
    e = 8.f * (x.h * x.A * fabsf(z.scale)) * b;
    if (z.waug) e += 0.5f * root * (u + b) + 4.f * u * b;
  }
  return Gaps{0x1p-23f * fmaf(0.5f * (float)steps, g, e), 0x1p-23f * fmaf(4.f, g, e)};
}

// Cuts a position's list of candidates [c_0, n_c) to `keep` (at least C) of them: the
// threshold rises to the C-th largest of the list, what lies below it goes, and of its
// near ties the highest ids.  For lists that overflow: a record of many large logits,
// or many such records.
struct Cut {
  int n_c;  // the new end
  float bound, above;
};
template <int TW>
__device__ __noinline__ Cut tidy_candidates(Team<TW> team, int C, int keep, int c_0, int n_c,
                                            float eps, float bound, float above, int* ids,
                                            float* approx, float* approx32, int* ranks, float* kth,
                                            int* words) {
  team.sync();
  for (int c = c_0 + team.tid; c < n_c; c += team.kThreads)
    if (approx[c] > -INFINITY) approx32[c] = approx[c];
  team.sync();
  for (int c = c_0 + team.tid; c < n_c; c += team.kThreads) {
    int rank = 0;
    for (int q = c_0; q < n_c; ++q)
      rank += approx32[q] > approx32[c] || (approx32[q] == approx32[c] && q < c);
    if (rank == C - 1) *kth = approx32[c];
  }
  team.sync();
  bound = fmaxf(bound, *kth - eps);
  above = fmaxf(above, *kth + eps);
  int n_above = 0;
  for (int c = c_0; c < n_c; ++c) n_above += approx32[c] > above;
  for (int c = c_0 + team.tid; c < n_c; c += team.kThreads) {
    bool stays = approx32[c] > above;
    if (!stays && approx32[c] >= bound) {
      int before = n_above;
      for (int q = c_0; q < n_c; ++q)
        before += approx32[q] >= bound && !(approx32[q] > above) && ids[q] < ids[c];
      stays = before < keep;
    }
    ranks[c] = stays;
  }
  team.sync();
  if (team.w == 0) {
    int n = c_0;
    for (int c0 = c_0; c0 < n_c; c0 += 32) {
      const int c = c0 + team.lane, at = min(c, n_c - 1);
      const int id = ids[at];
      const float x = approx[at], y = approx32[at];
      const unsigned b = __ballot_sync(0xffffffffu, c < n_c && ranks[at] != 0);
      if (b >> team.lane & 1u) {
        const int to = n + __popc(b & ((1u << team.lane) - 1u));
        ids[to] = id;
        approx[to] = x;
        approx32[to] = y;
      }
      n += __popc(b);
      __syncwarp();
    }
    if (team.lane == 0) words[15] = n;
  }
  team.sync();
  return Cut{words[15], bound, above};
}

// One team per position, NK records per thread.  Merge the sums; bisect for a
// threshold that n_pick to n_pick + kPickStop records reach: it is a lower bound of
// the n_pick-th largest logit; the candidates are the logits that reach it, less what
// rounding may have moved; compute again those whose order the pass's logits do not
// tell, sort, write.  The softmax's sums get the difference.  What keeps a list whole
// that overflows (tidy_candidates) costs 4 of the 106 us without being called: two turns
// over the records, and a call's registers.
// 4,096 positions, 64 alternatives: 106 us (with every candidate computed again, five
// groups of 16 rows of W a position, 25 more).  Waits for L2 and for instructions; 16
// warps an SM, with the registers that leaves, do better than 20 (115), 24 (142) or 12
// (112).
template <int TW, int NK>
static __global__ void __launch_bounds__(TW == 1 ? 32 * kScoreRows : 32 * TW, TW == 8 ? 2 : TW == 1 ? 4 : 5)
    lh_score_rows(ScoreArgs a) {
  constexpr int kTeams = TW == 1 ? kScoreRows : 1;
  constexpr int kThreads = 32 * TW;
  constexpr unsigned kAll = 0xffffffffu;
  extern __shared__ __align__(16) uint8_t smem_rows[];
  Team<TW> team;
  team.lane = threadIdx.x & 31;
  team.tid = threadIdx.x % kThreads;
  team.w = team.tid >> 5;
  const int lane = team.lane, tid = team.tid, w = team.w;
  const unsigned below = (1u << lane) - 1u;
  const int no = threadIdx.x / kThreads;
  const int t = (int)blockIdx.x * kTeams + no;
  const size_t team_bytes = score_team_smem(a.n_pick, a.cap, TW);
  const int P = score_picks(a.n_pick);
  team.red = reinterpret_cast<double*>(smem_rows + no * team_bytes);
  double* zp = team.red + 4 * TW;  // [16 TW]
  double* z64 = team.red + (TW == 1 ? 0 : 20 * TW);
  int* ids = reinterpret_cast<int*>(z64 + a.cap);
  float* approx = reinterpret_cast<float*>(ids + a.cap);
  float* approx32 = approx + a.cap;  // again, rounded
  int* ranks = reinterpret_cast<int*>(approx32 + a.cap);
  int* picked = ranks + a.cap;
  float* psecond = reinterpret_cast<float*>(picked + P);
  float* prest = psecond + P;
  int* pcol = reinterpret_cast<int*>(prest + P);
  int* col_id = pcol + P;
  float* cols = reinterpret_cast<float*>(col_id + 64);
  int* words = reinterpret_cast<int*>(cols + 64);  // [16] counts per warp

  grid_wait();
  // this thread's records: (w NK + i) 32 + lane, so that record order is warp order
  float key[NK];
  if constexpr (TW == 1) {
    // the block's rows' records are runs: through shared memory, [row][record],
    // which is the teams' after that
    float* stage = reinterpret_cast<float*>(smem_rows);
    const int ld = a.n_sub + 1, t0 = (int)blockIdx.x * kTeams;
    const float* src = a.sub_max + (long long)(t0 >> 3) * a.n_sub * 8 + (t0 & 7);
#pragma unroll 8
    for (int k = threadIdx.x; k < a.n_sub * kTeams; k += 32 * kTeams)
      stage[(k % kTeams) * ld + k / kTeams] = src[k / kTeams * 8 + k % kTeams];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      const int k = i * 32 + lane;
      key[i] = k < a.n_sub ? stage[no * ld + k] : -INFINITY;
    }
    __syncthreads();
    if (t >= a.z.T) return;
  } else {
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      const int k = (w * NK + i) * 32 + lane;
      key[i] = k < a.n_sub ? a.sub_max[sub_idx(t, k, a.n_sub)] : -INFINITY;
    }
  }
  const int tk = a.tokens ? a.tokens[t] : -1;
  GapReads gr = {};
  if (a.top_k > 0) gr = read_gaps(a.z, a.norms, a.hn, t, lane);
  const bool have_tok = tk >= 0 && tk < a.z.V;
  const RowSum rs = merge_row<true>(a.p, t, a.p.slots(t), team);
  const float nan = __int_as_float(0x7fc00000);
  // NaN or infinite logits (-inf: 0 * inf in E), or a pass that gave up
  if (!isfinite(rs.M) || !isfinite(rs.S) || !isfinite(rs.E) ||
      *reinterpret_cast<const volatile int*>(a.stats + kStErr) != 0) {
    if (tid == 0) {
      if (a.logprob) a.logprob[t] = nan;
      if (a.entropy) a.entropy[t] = nan;
    }
    for (int k = tid; k < a.top_k; k += kThreads) {
      a.top_ids[(long long)t * a.top_k + k] = -1;
      a.top_logprobs[(long long)t * a.top_k + k] = nan;
    }
    return;
  }

  const Gaps gaps = a.top_k > 0 ? logit_gaps(a.z, gr, a.steps) : Gaps{0.f, 0.f};
  // threshold `lo`: at least C records reach it, n_lo of them where that is known
  // to be few enough
  const int C = a.n_pick;
  float kmax = -INFINITY, kmin = INFINITY;
#pragma unroll
  for (int i = 0; i < NK; ++i) {
    kmax = fmaxf(kmax, key[i]);
    if (key[i] > -INFINITY) kmin = fminf(kmin, key[i]);
  }
  float hi = team.max_f(kmax), lo;
  int n_lo = a.n_sub;
  if (TW == 1 && C <= min(32, a.n_sub)) {
    // the C-th largest of the lanes' maxima: close to it from below
    int rank = 0;
#pragma unroll
    for (int q = 0; q < 32; ++q) {
      const float x = __shfl_sync(kAll, kmax, q);
      rank += x > kmax || (x == kmax && q < lane);
    }
    lo = __shfl_sync(kAll, kmax, __ffs(__ballot_sync(kAll, rank == C - 1)) - 1);
    int c = 0;
#pragma unroll
    for (int i = 0; i < NK; ++i) c += key[i] >= lo;
    n_lo = team.count(c);
  } else {
    lo = -team.max_f(-kmin);
  }
  while (n_lo > C + kPickStop && lo < hi) {
    float mid = lo + 0.5f * (hi - lo);
    if (!(mid > lo)) mid = hi;
    int c = 0;
#pragma unroll
    for (int i = 0; i < NK; ++i) c += key[i] >= mid;
    c = team.count(c);
    if (c >= C) {
      lo = mid;
      n_lo = c;
    } else if (mid == hi) {
      break;
    } else {
      hi = mid;
    }
  }
  // records that reach the threshold but for rounding; where they are more than
  // P (equal or nearly equal maxima, as of a padding row), those surely above it
  // and of the others the lowest
  const float eps = gaps.pass;
  float bound = lo - eps, above = lo + eps;
  const float first = bound;  // what a record's second had to reach
  int room = P;
  bool crowded;
  {
    int c = 0;
#pragma unroll
    for (int i = 0; i < NK; ++i) c += key[i] >= bound;
    crowded = team.count(c) > P;
    if (crowded) {
      c = 0;
#pragma unroll
      for (int i = 0; i < NK; ++i) c += key[i] > above;
      room = P - team.count(c);
    }
  }
  int n_p = 0;
  {  // this warp's picks, in record order
    int n_eq = 0;
    if constexpr (TW > 1) {
      int c = 0, e = 0;
#pragma unroll
      for (int i = 0; i < NK; ++i) {
        c += crowded ? key[i] > above : key[i] >= bound;
        e += crowded && key[i] >= bound && !(key[i] > above);
      }
      c = __reduce_add_sync(kAll, c);
      e = __reduce_add_sync(kAll, e);
      if (lane == 0) words[w] = c << 16 | e;
      team.sync();
      for (int q = 0; q < w; ++q) {
        const int eq = words[q] & 0xffff;
        n_p += (words[q] >> 16) + min(eq, max(0, room - n_eq));
        n_eq += eq;
      }
    }
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      bool take = key[i] >= bound;
      if (crowded) {
        const bool eq = take && !(key[i] > above);
        const unsigned beq = __ballot_sync(kAll, eq);
        take = take && (!eq || n_eq + __popc(beq & below) < room);
        n_eq += __popc(beq);
      }
      const unsigned bt = __ballot_sync(kAll, take);
      if (take) picked[n_p + __popc(bt & below)] = (w * NK + i) * 32 + lane;
      n_p += __popc(bt);
    }
    if constexpr (TW > 1) {
      if (w == TW - 1 && lane == 0) words[8] = n_p;
      team.sync();
      n_p = words[8];
    } else {
      __syncwarp();
    }
  }
  // (the given token comes first, then the candidates)
  const int c_0 = have_tok ? 1 : 0;
  {
    constexpr int kG = TW == 1 ? 3 : 1;  // picks' records in flight per thread
    for (int c0 = tid; c0 < n_p; c0 += kG * kThreads) {
      float m[kG], second[kG], rest[kG];
      int c1[kG], c2[kG];
#pragma unroll
      for (int i = 0; i < kG; ++i) {
        const int c = min(c0 + i * kThreads, n_p - 1);
        const long long o = sub_idx(t, picked[c], a.n_sub);
        m[i] = a.sub_max[o];
        rest[i] = a.sub > 1 ? a.sub_rest[o] : -INFINITY;
        second[i] = a.sub == 64 ? a.sub_second[o] : -INFINITY;
        c1[i] = a.sub > 1 ? a.sub_arg[o] : 0;
        c2[i] = a.sub == 64 ? a.sub_arg2[o] : 0;
      }
#pragma unroll
      for (int i = 0; i < kG; ++i) {
        const int c = c0 + i * kThreads;
        if (c >= n_p) continue;
        approx[c_0 + c] = m[i];
        ids[c_0 + c] = picked[c] * a.sub + c1[i];
        prest[c] = rest[i];
        psecond[c] = second[i];
        pcol[c] = c1[i] | c2[i] << 8;
      }
    }
  }
  if (have_tok && tid == 0) ids[0] = tk;
  team.sync();
  // seconds that reach the bound, then the columns of records whose rest does
  int n_c = c_0 + n_p;  // (up to a.cap)
  if (a.sub == 64)
    for (int c0 = 0; c0 < n_p; c0 += 32) {  // (every warp finds the same)
      const int c = c0 + lane;
      const bool two = c < n_p && psecond[c] >= bound;
      const unsigned b = __ballot_sync(kAll, two);
      if (two && w == 0) {
        const int at = n_c + __popc(b & below);
        ids[at] = picked[c] * 64 + (pcol[c] >> 8);
        approx[at] = psecond[c];
      }
      n_c += __popc(b);
    }
  // First the records whose rest lies above the threshold: their columns may come
  // before all that is known, however many ties the threshold has.  Then those whose
  // rest is a near tie of it, lowest ids first, as far as there is room.
  for (int ph = 0; ph < 2 && a.sub > 1; ++ph) {
    auto tidy = [&] {
      const Cut cut = tidy_candidates(team, C, 2 * P, c_0, n_c, eps, bound, above, ids, approx,
                                      approx32, ranks, cols, words);
      n_c = cut.n_c;
      bound = cut.bound;
      above = cut.above;
    };
    if (ph == 1 && n_c - c_0 > 2 * P) tidy();
    for (int c0 = 0; c0 < n_p; c0 += 32) {
      const float rest = c0 + lane < n_p ? prest[c0 + lane] : -INFINITY;
      unsigned more = __ballot_sync(kAll, rest >= bound && (ph == 1 || rest > above));
      for (; more && n_c < a.cap; more &= more - 1) {
        const int c = c0 + __ffs(more) - 1;
        if (ph == 0) {
          if (n_c - c_0 > 2 * P) tidy();
          if (!(prest[c] > above)) continue;  // the threshold has risen
        }
        const int v0 = picked[c] * a.sub, c1 = pcol[c] & 255, nv = min(a.sub, a.z.V - v0);
        const int c2 = a.sub == 64 && psecond[c] >= first ? pcol[c] >> 8 : -1;
        for (int q = tid; q < nv; q += kThreads) col_id[q] = v0 + q;
        team.sync();
        if (ph == 0 && tid == 0) prest[c] = -INFINITY;  // done with
        for (int q = 16 * w; q < nv; q += 16 * TW)
          logits16<false>(a.z, t, col_id + q, min(16, nv - q), lane, cols + q);
        team.sync();
        for (int q0 = 0; q0 < nv; q0 += 32) {  // (every warp finds the same)
          const int q = q0 + lane;
          const bool take = q < nv && q != c1 && q != c2 && cols[q] >= bound;
          const unsigned bt = __ballot_sync(kAll, take);
          const int at = n_c + __popc(bt & below);
          if (take && w == 0 && at < a.cap) {
            ids[at] = v0 + q;
            approx[at] = -INFINITY;  // not known: the sums keep it as it is
            approx32[at] = cols[q];
          }
          n_c = min(n_c + __popc(bt), a.cap);
        }
        team.sync();
      }
    }
  }
  // The pass's logits, made good for their known loss, tell the order of all but those
  // within gaps.pass of another.  These, the kMinPick largest (by which the softmax's sums are made good) and
  // those known only from the columns above are computed again, the others' logits
  // are the pass's; of 72 candidates of a list of 64 that is about 10, one group of
  // 16 instead of five.  All, where that is one group anyway.
  const double ln2 = 0.69314718055994531, log2e = 1.4426950408889634;
  const double back = (double)a.lg * ln2;
  team.sync();
  for (int c = c_0 + tid; c < n_c; c += kThreads)
    if (approx[c] > -INFINITY) approx32[c] = (float)((double)approx[c] * back);
  team.sync();
  constexpr int kItems = TW == 1 ? 3 : 2;
  int n_z = n_c;  // [0, n_z) are computed again
  const bool fits = n_c - c_0 <= kItems * kThreads;
  for (int b0 = c_0; b0 < n_c && (a.top_k > 0 || n_c > 16); b0 += kItems * kThreads) {
    float z[kItems], gap[kItems], was[kItems];
    int rank[kItems], close[kItems], id[kItems];
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int c = b0 + i * kThreads + tid;
      z[i] = c < n_c ? approx32[c] : INFINITY;
      gap[i] = c < n_c ? gaps.pass : -1.f;
      rank[i] = close[i] = 0;
    }
    for (int q = c_0; q < n_c; ++q) {
      const float zq = approx32[q];
#pragma unroll
      for (int i = 0; i < kItems; ++i) {
        rank[i] += zq > z[i];
        close[i] += fabsf(zq - z[i]) <= gap[i];
      }
    }
    if (!fits || n_c <= 16) {
#pragma unroll
      for (int i = 0; i < kItems; ++i) {
        const int c = b0 + i * kThreads + tid;
        if (c < n_c) ranks[c] = close[i] > 1 ? -1 : rank[i];  // (it is close to itself)
      }
      continue;
    }
    // those to be computed again to the front (one round: they all fit)
    unsigned again[kItems];
    int n_w = 0;
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int c = min(b0 + i * kThreads + tid, n_c - 1);
      was[i] = approx[c];
      id[i] = ids[c];
      again[i] = __ballot_sync(kAll, gap[i] >= 0.f && (close[i] > 1 || rank[i] < kMinPick ||
                                                       was[i] == -INFINITY));
      n_w += __popc(again[i]);
    }
    int front = c_0;
    if constexpr (TW > 1) {
      if (lane == 0) words[w] = n_w;
      __syncthreads();
      n_z = c_0;
      for (int q = 0; q < TW; ++q) {
        front += q < w ? words[q] : 0;
        n_z += words[q];
      }
    } else {
      __syncwarp();
      n_z = c_0 + n_w;
    }
    // the others behind: as many of them as stand before a candidate, less those
    // that have gone to the front
    int behind = n_z;
    if constexpr (TW > 1) {
      int mine = 0;
#pragma unroll
      for (int i = 0; i < kItems; ++i)
        mine += __popc(__ballot_sync(kAll, gap[i] >= 0.f) & ~again[i]);
      if (lane == 0) words[8 + w] = mine;
      __syncthreads();
      for (int q = 0; q < w; ++q) behind += words[8 + q];
    }
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const unsigned rest = __ballot_sync(kAll, gap[i] >= 0.f) & ~again[i];
      const bool sel = again[i] >> lane & 1;
      const int to = sel ? front + __popc(again[i] & below) : behind + __popc(rest & below);
      if (gap[i] >= 0.f) {
        ids[to] = id[i];
        approx[to] = was[i];
        approx32[to] = z[i];
        ranks[to] = close[i] > 1 ? -1 : rank[i];
      }
      front += __popc(again[i]);
      behind += __popc(rest);
    }
  }
  team.sync();
  team_logits<TW>(a.z, t, ids, n_z, team, z64, zp);
  for (int c = n_z + tid; c < n_c; c += kThreads) z64[c] = (double)approx[c] * back;
  team.sync();
  // in 64 bits throughout those that are too close to another even now
  bool any_close = false;
  for (int c = c_0 + tid; c < n_z && a.top_k > 0; c += kThreads) {
    if (ranks[c] >= 0) continue;
    int close = 0;
    for (int q = c_0; q < n_z; ++q) close += fabsf((float)(z64[q] - z64[c])) <= gaps.again;
    if (close > 1) {
      ranks[c] = -2;
      any_close = true;
    }
  }
  team.sync();
  if (team.count(any_close) > 0) {
    double* u = reinterpret_cast<double*>(col_id);  // and cols: [64]
    u64(a.z, t, team, u);
    for (int c0 = 32 * w; c0 < n_z; c0 += kThreads) {
      const int c = c0 + lane;
      unsigned near = __ballot_sync(kAll, c >= c_0 && c < n_z && ranks[min(c, n_z - 1)] == -2);
      for (; near; near &= near - 1) {
        const int q = __ffs(near) - 1;
        const double zq = logit64(a.z, t, ids[c0 + q], u, lane);
        if (lane == q) z64[c] = zq;
      }
    }
  }
  team.sync();
  // the sums with these logits as they are now
  const double Ml = (double)rs.M;
  double dS = 0.0, dE = 0.0;
  for (int c = c_0 + lane; c < n_z; c += 32) {
    if (!(approx[c] > -INFINITY)) continue;
    const double xe = z64[c] * log2e - Ml, xa = (double)approx[c] * (double)a.lg - Ml;
    // 2^xe - 2^xa = 2^xa (2^(xe - xa) - 1), without the cancellation
    const float ea = exp2f((float)xa);
    const double diff = (double)(ea * expm1f(0.69314718f * (float)(xe - xa)));
    dS += diff;
    dE += diff * xe + (double)ea * (xe - xa);
  }
  dS = warp_sum(dS);
  dE = warp_sum(dE);
  const double S = rs.S + dS, E = rs.E + dE;
  const double lnS = log(S), lse = Ml * ln2 + lnS;
  if (tid == 0) {
    if (a.logprob) a.logprob[t] = have_tok ? (float)(z64[0] - lse) : nan;
    if (a.entropy) a.entropy[t] = (float)fmax(0.0, lnS - ln2 * E / S);
  }
  for (int c = c_0 + tid; c < n_c && a.top_k > 0; c += kThreads) {
    int rank = ranks[c];
    if (rank < 0) {
      rank = 0;
      for (int q = c_0; q < n_c; ++q)
        rank += z64[q] > z64[c] || (z64[q] == z64[c] && ids[q] < ids[c]);
    }
    if (rank < a.top_k) {
      a.top_ids[(long long)t * a.top_k + rank] = ids[c];
      a.top_logprobs[(long long)t * a.top_k + rank] = (float)(z64[c] - lse);
    }
  }
}

// ------------------------------------------------------------- distill, per row
struct DistillArgs {
  LogitArgs z;
  SlotPlan p;
  float lg, tau, scale;
  int K;
  const int32_t* ids;
  const float* teacher;
  float* wt;      // in: weight * tau of rows with entries; out: 0 where none counts
  const float* Bt;  // [Vpad][R] (gradients): bidx layout, or row by row; null: z.B
  int Bt_plain;
  const int* stats;
  const int* order;   // as PrepArgs, and the number of positions that count
  const int* active;
  float* loss;
  // gradients
  float* tok;     // records of ranks 4, 8
  float2* ref;    // few positions
  float* nml;     // tensor-core rank sums: exponent offsets, factors of the rank operand
  float* xs;
  float* dU;      // [T][R]
  unsigned long long* corr;  // [Vpad][R] fixed point, row by row
};

// One team per position.  q = softmax(teacher / tau) over the entries with an
// id; loss = w tau^2 (sum q (log q - z / tau) + log sum e^(z / tau)); then,
// with kGrads, dU = s w tau (Q / S - sum q B[:, id]) and the sparse part of
// dB, sum over t of w tau q s U[t], in fixed point: 2^38 times its largest
// possible term, summed with integer atomics, so that the order in which
// positions meet an id does not change the result.
// 8,192 positions, rank 4, 8 entries: 40 us.  8,000, 70% of them counted, rank 64, 64
// entries: 147, of which 40 the atomics; the rest reads 64 rows of W, of the rank term
// and of B per position, 100 KB, from L2.
template <bool kGrads, int TW>
static __global__ void
    __launch_bounds__(32 * (TW == 1 ? kRowWarps : TW), TW == 8 ? 2 : TW == 4 ? 4 : kGrads ? 3 : 2)
    lh_distill_rows(DistillArgs a) {
  constexpr int kTeams = TW == 1 ? kRowWarps : 1, kThreads = 32 * TW;
  constexpr int kPer = (kMaxTop + kThreads - 1) / kThreads;
  __shared__ double s_red[kTeams][4 * TW];
  __shared__ int s_id[kTeams][kMaxTop];
  __shared__ float s_q[kTeams][kMaxTop];
  __shared__ double s_lq[kTeams][kMaxTop];
  __shared__ double s_z[kTeams][kMaxTop];
  __shared__ double s_Q[kTeams][kThreads > 64 ? kThreads : 64];
  Team<TW> team;
  team.lane = threadIdx.x & 31;
  team.tid = threadIdx.x % kThreads;
  team.w = team.tid >> 5;
  const int lane = team.lane, tid = team.tid, no = threadIdx.x / kThreads;
  team.red = s_red[no];
  const int t = (int)blockIdx.x * kTeams + no;
  grid_wait();
  if (t >= a.z.T) return;
  const int R = a.z.R;
  const int at = a.order ? a.order[t] : t;
  int nslot = 0;  // behind those that count the passes need not have been
  if (!a.active) {
    nslot = a.p.slots(t);
  } else if (t < *a.active) {
    SlotPlan p = a.p;
    p.n_a = active_tiles(*a.active, 2 * kBM, p.n_a, p.n_b, min(p.units, p.n_a * p.n_b));
    nslot = p.slots(t);
  }
  const float nan = __int_as_float(0x7fc00000);
  float wt = a.wt[t];
  // the teacher's distribution
  int id[kPer];
  double lq[kPer];
  double top = -INFINITY;
  int wrong = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int k = tid + i * kThreads;
    id[i] = -1;
    lq[i] = 0.0;
    if (wt != 0.f && k < a.K) {
      const int v = a.ids[(long long)at * a.K + k];
      const float x = a.teacher[(long long)at * a.K + k];
      if (v >= a.z.V || (v >= 0 && !(x < INFINITY))) wrong = 1;
      else if (v >= 0 && x > -INFINITY) {
        id[i] = v;
        lq[i] = (double)x / (double)a.tau;
        top = fmax(top, lq[i]);
      }
    }
  }
  RowSum rs = merge_row<false>(a.p, t, nslot, team);
  if (nslot == 0) rs = RowSum{0.f, 1.0, 0.0};
  wrong = team.count(wrong);
  top = team.reduce(top, [](double p, double q) { return fmax(p, q); });
  double total = 0.0;
  double e[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    e[i] = id[i] >= 0 ? exp(lq[i] - top) : 0.0;
    total += e[i];
  }
  total = team.sum(total);
  const double ltotal = wt != 0.f && !wrong ? log(total) : 0.0;
  if (wrong) wt = nan;
  const double Ml = (double)rs.M;
  const double lse = (Ml + log2(rs.S)) * 0.69314718055994531;
  const bool counts = wt != 0.f && !wrong;
  // the entries that weigh anything, in the order of the list
  int base = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const bool have = counts && e[i] > 0.0;
    const unsigned b = __ballot_sync(0xffffffffu, have);
    if constexpr (TW == 1) {
      if (have) {
        const int n = base + __popc(b & ((1u << lane) - 1u));
        s_id[no][n] = id[i];
        s_lq[no][n] = lq[i] - top - ltotal;
        s_q[no][n] = (float)(e[i] / total);
      }
      base += __popc(b);
    } else {  // kPer 1: warps 0..3 hold the list
      if (lane == 0) reinterpret_cast<int*>(s_Q[no])[team.w] = __popc(b);
      __syncthreads();
      int before = 0, n_all = 0;
      for (int q = 0; q < TW; ++q) {
        const int n = reinterpret_cast<int*>(s_Q[no])[q];
        before += q < team.w ? n : 0;
        n_all += n;
      }
      if (have) {
        const int n = before + __popc(b & ((1u << lane) - 1u));
        s_id[no][n] = id[i];
        s_lq[no][n] = lq[i] - top - ltotal;
        s_q[no][n] = (float)(e[i] / total);
      }
      base = n_all;
    }
  }
  team.sync();
  const int n = base;
  double loss = 0.0;
  team_logits<TW>(a.z, t, s_id[no], n, team, s_z[no], s_Q[no]);
  for (int k = tid; k < n; k += kThreads) {
    const double l = s_lq[no][k];
    loss += exp(l) * (l - s_z[no][k] / (double)a.tau);
  }
  loss = team.sum(loss);
  const bool gave_up = *reinterpret_cast<const volatile int*>(a.stats + kStErr) != 0;
  if (tid == 0)
    a.loss[at] = wrong || gave_up ? nan
                : counts         ? (float)((double)wt * (double)a.tau * (loss + lse)) : 0.f;
  if constexpr (kGrads) {
    const float inv = (float)(1.0 / rs.S);
    if (tid == 0) {
      a.wt[t] = wt;
      if (a.tok) {
        a.tok[tidx(t, R, R)] = -rs.M;
        a.tok[tidx(t, R + 1, R)] = wt == 0.f ? 0.f : wt * inv;
      }
      if (a.ref) a.ref[t] = make_float2(rs.M, wt == 0.f ? 0.f : wt * inv);
      if (a.nml) {
        // p = 2^(z lg + nml - 14) xs: the exponent's share of 1 / S is a whole
        // power of two and what rounding takes from nml goes into xs, so that a
        // row's p is not off by the rounding of an offset of 10 or 20
        const int ks = ilogb(rs.S);
        const double off = 14.0 - (double)ks - Ml;
        const float nml = (float)off;
        a.nml[t] = nml;
        a.xs[t] = (float)(exp2(off - (double)nml) * ldexp(1.0 / rs.S, ks));
      }
    }
    const double xb = (a.nml ? exp2i(-scale_exp(a.stats[kStBMax], 13)) : 1.0) / rs.S;
    const int fe = scale_exp(a.stats[kStUMax], 37);
    const double fx = fe > 1000 || fe < -1000 ? 0.0 : exp2i(fe);
    // threads over (rank, slice of the slots or entries)
    const int RL = R < kThreads ? R : kThreads, ns = kThreads / RL;
    const int sl = tid / RL;
    for (int j = tid % RL; j < R; j += RL) {
      double Q = 0.0;
#pragma unroll 4
      for (int k = sl; k < nslot; k += ns) {
        const long long o = (long long)k * a.p.ld + t;
        const float pm = a.p.p_max[o], pq = a.p.p_q[o * R + j];
        if (pm != -INFINITY) Q += (double)(pq * exp2f(pm - rs.M));
      }
      Q *= xb;
      const double su = (double)a.z.sU[(long long)t * R + j] * (double)wt * fx;
      const bool scatter = j < a.z.r && wt != 0.f && isfinite(su);
      const bool pairs = a.Bt ? !a.Bt_plain : a.z.B.layout != 0;
      const long long bs = a.Bt ? R : 1;
      const float* bp = a.Bt ? a.Bt + (pairs ? 0 : j) : a.z.B.p + (pairs ? 0 : (long long)j * a.z.V);
      if (!a.Bt && j >= a.z.r) bp = nullptr;
      // eight entries' rows of B at a time on the way: a load does not pass an
      // atomic, and one by one each would wait for the L2
      for (int k0 = sl; k0 < n; k0 += 8 * ns) {
        float b[8];
#pragma unroll
        for (int e8 = 0; e8 < 8; ++e8) {
          const int k = k0 + e8 * ns;
          b[e8] = 0.f;
          if (k < n && bp) {
            const int v = s_id[no][k];
            b[e8] = bp[pairs ? bidx(v, j, R) : (long long)v * bs];
          }
        }
        asm volatile("" ::: "memory");
#pragma unroll
        for (int e8 = 0; e8 < 8; ++e8) {
          const int k = k0 + e8 * ns;
          if (k >= n) continue;
          const float qk = s_q[no][k];
          Q -= (double)(qk * b[e8]);
          if (scatter)
            atomicAdd(&a.corr[(long long)s_id[no][k] * R + j],
                      (unsigned long long)__double2ll_rn(su * (double)qk));
        }
      }
      if constexpr (TW == 1) {
        for (int off = RL; off < 32; off <<= 1) Q += __shfl_xor_sync(0xffffffffu, Q, off);
      } else {  // ns slices of R (<= 64) ranks
        team.sync();
        s_Q[no][sl * R + j] = Q;
        team.sync();
        if (sl == 0)
          for (int q = 1; q < ns; ++q) Q += s_Q[no][q * R + j];
      }
      if (sl == 0)
        a.dU[(long long)t * R + j] = wt == 0.f ? 0.f : (float)((double)a.scale * (double)wt * Q);
    }
  }
}

// Pass 2's rank operand on the tensor cores: xt[j][t] = wt xs s U[t][j] 2^e as
// f16 hi / lo, e so that the largest entry is just below 2^14.  5 us for 8,000
// positions at rank 64 (2 MB read, 4 MB written).
static __global__ void lh_xt(int T, int R, long long ld, const float* __restrict__ sU,
                             const float* __restrict__ wt, const float* __restrict__ xs,
                             const int* __restrict__ stats,
                             __half* __restrict__ xt) {
  grid_wait();
  const double up = exp2i(scale_exp(stats[kStUMax], 13));
  const long long n = (long long)T * R, stride = (long long)gridDim.x * blockDim.x;
  for (long long k = (long long)blockIdx.x * blockDim.x + threadIdx.x; k < n; k += stride) {
    const int j = (int)(k / T), t = (int)(k % T);
    const float w = wt[t];
    const float x = w == 0.f ? 0.f : (float)((double)sU[(long long)t * R + j] * (double)w * (double)xs[t] * up);
    const __half hi = __float2half_rn(x);
    xt[(long long)j * ld + t] = hi;
    xt[(long long)(R + j) * ld + t] = __float2half_rn(x - __half2float(hi));
  }
}

// gAp[c][i][j] = sum over the kDAChunk positions of chunk c of h16[t][i] dU[t][j]:
// blocks of 64 hidden elements by all R ranks, 64 positions at a time through
// shared memory with the next 64 in flight.  (lce_dA_partial takes 16 ranks per
// launch: 50 us at rank 64 and 8,000 positions, this 21.)
template <int R>
static __global__ void __launch_bounds__(256) lh_dA(int T, int d, const __half* __restrict__ h16,
                                                    const float* __restrict__ dU,
                                                    float* __restrict__ gAp) {
  constexpr int JT = R >= 64 ? 4 : R == 32 ? 2 : 1;  // ranks per thread
  constexpr int TJ = R / JT;                         // threads over ranks
  constexpr int TI = 256 / TJ;                       // threads over hidden elements
  constexpr int IT = 64 / TI;                        // hidden elements per thread
  constexpr int kU = (64 * R + 255) / 256;
  __shared__ __align__(16) float sh[64][64];
  __shared__ __align__(16) float su[64][R];
  grid_wait();
  const int tid = threadIdx.x, tj = tid % TJ, ti = tid / TJ;
  const int c = (int)blockIdx.x, i0 = (int)blockIdx.y * 64;
  const int t_lo = c * kDAChunk, t_hi = min(T, t_lo + kDAChunk);
  float acc[IT][JT] = {};
  uint4 hn[2];
  float un[kU];
  auto fetch = [&](int t0) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {  // 8 f16 of row (tid + 256 q) / 8
      const int row = (tid + 256 * q) >> 3, t = t0 + row;
      hn[q] = make_uint4(0u, 0u, 0u, 0u);
      if (t < t_hi)
        hn[q] = *reinterpret_cast<const uint4*>(h16 + (long long)t * d + i0 + 8 * (tid & 7));
    }
#pragma unroll
    for (int q = 0; q < kU; ++q) {
      const int k = tid + 256 * q, t = t0 + k / R;
      un[q] = t < t_hi ? dU[(long long)t0 * R + k] : 0.f;
    }
  };
  fetch(t_lo);
  for (int t0 = t_lo; t0 < t_hi; t0 += 64) {
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const __half2* p = reinterpret_cast<const __half2*>(&hn[q]);
      float* o = &sh[(tid + 256 * q) >> 3][8 * (tid & 7)];
#pragma unroll
      for (int e = 0; e < 4; ++e) *reinterpret_cast<float2*>(o + 2 * e) = __half22float2(p[e]);
    }
#pragma unroll
    for (int q = 0; q < kU; ++q) (&su[0][0])[tid + 256 * q] = un[q];
    __syncthreads();
    if (t0 + 64 < t_hi) fetch(t0 + 64);
#pragma unroll 8
    for (int t = 0; t < 64; ++t) {
      float x[IT], y[JT];
#pragma unroll
      for (int e = 0; e < IT; ++e) x[e] = sh[t][ti * IT + e];
#pragma unroll
      for (int e = 0; e < JT; ++e) y[e] = su[t][tj * JT + e];
#pragma unroll
      for (int p = 0; p < IT; ++p)
#pragma unroll
        for (int q = 0; q < JT; ++q) acc[p][q] = fmaf(x[p], y[q], acc[p][q]);
    }
  }
#pragma unroll
  for (int p = 0; p < IT; ++p)
#pragma unroll
    for (int q = 0; q < JT; ++q)
      gAp[((long long)c * d + i0 + ti * IT + p) * R + tj * JT + q] = acc[p][q];
}

struct GradArgs {
  int T, d, V, r, R, n_chunks, cparts, res_rows, n_b2, G2;
  const int* active;  // as DistillArgs; bn2 positions per tile
  int bn2;
  long long Vpad;
  const float* gAp;                // [chunk][d][R]
  const float* gBp;                // [seg][Vpad][R] bidx
  const unsigned long long* corr;  // [Vpad][R], row by row
  int scaled;                      // gBp carries xt's 2^e
  const int* stats;
  float* gA;       // layout 0: [d][r] and [r][V]; layout 1: [d][R] and [Vpad][R] bidx
  float* gB;
  int layout;
  // layout 1: [sum of losses, counted positions] behind the gradients
  const float* loss;
  const float* wt;
  float* tail;
};

// The gradient sums in the caller's layout, every element in a fixed order.
// Blocks [0, Vpad / 64) take 64 vocab rows each, through shared memory where
// the caller's rows are ranks; the others gA; block 0 the tail too.  V = 49152: 8 us
// at rank 4 and 21 us at rank 64, where 2 partials, the 64-bit part and the result are
// 63 MB (3 TB/s); what it waits for is read at once.
static __global__ void __launch_bounds__(256) lh_grads(GradArgs a) {
  __shared__ float tile[64 * (kPackRows + 1)];
  grid_wait();
  const bool bad = *reinterpret_cast<const volatile int*>(a.stats + kStErr) != 0;
  const float nan = __int_as_float(0x7fc00000);
  const int blk = (int)blockIdx.x, tid = (int)threadIdx.x;
  const int v_blocks = (int)(a.Vpad / kPackRows);
  if (blk >= v_blocks) {
    const int ra = a.layout ? a.R : a.r;
    const long long k = (long long)(blk - v_blocks) * 256 + tid;
    if (k >= (long long)a.d * ra) return;
    const long long nA = (long long)a.d * a.R, o = k / ra * a.R + k % ra;
    double s = 0.0;
#pragma unroll 8
    for (int c = 0; c < a.n_chunks; ++c) s += (double)a.gAp[c * nA + o];
    a.gA[k] = bad ? nan : (float)s;
    return;
  }
  const double ex = a.scaled ? exp2i(-scale_exp(a.stats[kStUMax], 13)) : 1.0;
  const double fx = exp2i(-scale_exp(a.stats[kStUMax], 37));
  const long long v0 = (long long)blk * kPackRows, stride = a.Vpad * a.R;
  int slots = 0;
  if (v0 < a.V) {
    SlotPlan p{a.cparts, (a.V + a.res_rows - 1) / a.res_rows, a.n_b2, a.G2};
    if (a.active) p.n_b = active_tiles(*a.active, a.bn2, p.n_b, p.n_a, a.G2);
    slots = p.slots_of((int)v0 / a.res_rows);
  }
  constexpr int ld = kPackRows + 1;
  const int n = kPackRows * a.R, lr = __ffs(a.R) - 1;  // 256 to 4096
  const float* src = a.gBp + v0 * a.R;
  for (int k0 = tid; k0 < n; k0 += 4 * 256) {
    double s[4] = {0.0, 0.0, 0.0, 0.0};
    long long c[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int k = k0 + 256 * e, i = 2 * (k >> (lr + 1)) + (k & 1), j = (k & (2 * a.R - 1)) >> 1;
      c[e] = k < n ? (long long)a.corr[(v0 + i) * a.R + j] : 0;
    }
#pragma unroll 4
    for (int q = 0; q < slots; ++q)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (k0 + 256 * e < n) s[e] += (double)src[q * stride + k0 + 256 * e];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int k = k0 + 256 * e, i = 2 * (k >> (lr + 1)) + (k & 1), j = (k & (2 * a.R - 1)) >> 1;
      if (k < n) tile[j * ld + i] = v0 + i < a.V ? (float)(s[e] * ex - (double)c[e] * fx) : 0.f;
    }
  }
  __syncthreads();
  if (a.layout) {
    for (int k = tid; k < n; k += 256)
      a.gB[v0 * a.R + k] = bad ? nan : tile[((k & (2 * a.R - 1)) >> 1) * ld + 2 * (k >> (lr + 1)) + (k & 1)];
  } else {
    for (int k = tid; k < a.r * kPackRows; k += 256) {
      const int j = k / kPackRows, i = k % kPackRows;
      if (v0 + i < a.V) a.gB[(long long)j * a.V + v0 + i] = bad ? nan : tile[j * ld + i];
    }
  }
  if (a.tail && blk == 0) put_tail(a.loss, a.wt, a.T, a.tail);
}

// A trainer's step between its gradient sums and the optimizer: the passes' error
// goes to the handle's flag, and a step that counts no position divides by 1.
static __global__ void lh_tail(const int* stats, float* tail, int* err) {
  const int e = stats[kStErr];
  if (e != 0) atomicCAS(err, 0, e);
  if (tail[1] == 0.f) tail[1] = 1.f;
}

}  // namespace lce
