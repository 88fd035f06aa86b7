// Cross entropy of a linear head, loss_r = log sum_v exp z_rv - z_r,label with
// z = h W^T, whose logits z never reach memory, forward and backward.
//
//   forward   every tile of z is reduced where its product ends, in its
//             accumulators: per row the maximum and sum of exponentials of the
//             tile's columns, and the label's logit; a second kernel joins a
//             row's parts.
//   backward  piece by piece of the vocabulary: the piece's tiles of z once
//             more, dz = dloss (exp(z - lse) - [v = label]) stored in 16 bits
//             (the matrix cores' operand) where z would have been, and with it
//             dh += dz W (fp32, over the pieces) and dW = dz^T h.
//
// The products bound it, 2 rows hidden vocabulary operations forward and three times
// that backward, of which one third forms z again: keeping z would be the logits
// that this is to avoid.  2048 rows, hidden 2048, vocabulary 50304, bf16: forward
// 340 us, 1.24 PFLOP/s (the product alone, logits stored: 346), backward 1070 us, of
// which dz 362, dh 324 and its sum 19, dW 369.
//
// Rows whose label is ignored, and backward rows without upstream gradient,
// take no part: the others' indices are listed on the device first, the
// products gather their rows of h and end with the list, and what such rows
// hold (infinities, NaN) reaches nothing.
//
// Powers of two.  A row's dloss is split as 2^e m, 1 <= |m| < 2; dz carries m
// (in fp16 times 2^14, as exponentials down to 2^-28 then keep all digits), dh
// gets the row's 2^e back in fp32, and the rows of h that dW is formed of carry
// 2^(e - the largest e), so that gradients of any size keep their digits in
// fp16 as in bf16.  (A row's share of dW loses digits where its dloss is 2^-14
// of the largest and nothing else reaches the same row of dW.)
//
// The label's dz, p - 1, is the forward's loss: -(1 - exp(-loss)).  By way of lse,
// whose rounding is up to 2^-24 of it, 1 - p of a confident row would be that far off:
// at a logit of 100 by 5e-6, 5 % of a 1 - p of 1e-4.
//
// dz's rounding is dh's and dW's largest error (1.4 roundings with their own). It
// averages over the rows; where few take part they are listed twice, and dz is
// stored in two parts, its rounding and what that left, which the same products
// add up.
//
// No counterpart in the reference, whose head keeps the logits
// (model/flex_ops.py:1976-1981 after language_model.py:24-38).
#include <algorithm>

#include "gemm_tiles.h"

namespace eth {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// How a call's rows are listed: `count` rows take part, row r of the list
// being row rows[r] of h with label[r] (clamped); `high` is the largest exponent
// of their dloss, `alpha` dW's factor.
struct XentHead {
  int count, high;
  float alpha;
};

// over the four lanes that hold a row of the accumulators (lane % 16)
__device__ __forceinline__ float row_max(float v) {
  typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
  u32x2 p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(p.x), __uint_as_float(p.y));
  p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(p.x), __uint_as_float(p.y));
}
__device__ __forceinline__ float row_sum(float v) {
  typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
  u32x2 p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(p.x) + __uint_as_float(p.y);
  p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(p.x) + __uint_as_float(p.y);
}

// Parts of 16 rows lie together, [row / 16][part][row % 16], so a tile writes
// and the join reads whole lines.
struct XentPart {
  float m2, s;  // maximum of z log2(e), sum of 2^(z log2(e) - m2)
};

// A block of 16 rows at a time: a lane has a row's 8 to 32 columns of the wave's tile,
// their maximum, then a fused multiply-add and an exp2 each; two lane swaps join a
// row's four lanes.  No more time than storing the logits would take.
struct XentStats {
  static constexpr bool kSized = true, kGathers = true, kStarts = false, kMaps = false, kReduces = true;
  const XentHead* head;
  const int* rows;
  const int* label;
  XentPart* part;
  float* picked;
  int v0;      // the launch's first column in the vocabulary
  int part0;   // and its first part
  int parts;   // of a row, in all

  __device__ __forceinline__ void size(GemmArgs& g) const { g.M = min(g.M, head->count); }

  template <int TI, int TJ>
  __device__ __forceinline__ void reduce(f32x4_t (&acc)[TI][TJ], int row0, int col0, int M, int N) const {
    const int lane = threadIdx.x & 63, l16 = lane & 15, lg = lane >> 4;
    const int p = part0 + col0 / (TJ * 16);
    const bool edge = col0 + TJ * 16 > N;
    int at_label[TI];  // (all in flight together: a row block at a time, each waits for its own)
#pragma unroll
    for (int i = 0; i < TI; ++i) at_label[i] = label[min(row0 + i * 16 + l16, M - 1)];
#pragma unroll
    for (int i = 0; i < TI; ++i) {
      const int row = row0 + i * 16 + l16;
      const bool live = row < M;
      float z[TJ * 4];
#pragma unroll
      for (int j = 0; j < TJ; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) z[j * 4 + e] = acc[i][j][e];
      const int t = at_label[i] - v0 - col0;
      if (__ballot(live && t >= 0 && t < TJ * 16)) {
        // (one of a row's four lanes holds its label's logit; a column past N
        // is no label)
        float mine = 0.f;
#pragma unroll
        for (int j = 0; j < TJ; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (t == j * 16 + lg * 4 + e) mine = z[j * 4 + e];
        if (live && t >= 0 && t < TJ * 16 && ((t >> 2) & 3) == lg) picked[row] = mine;
      }
      if (edge) {
#pragma unroll
        for (int j = 0; j < TJ; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (col0 + j * 16 + lg * 4 + e >= N) z[j * 4 + e] = -INFINITY;
      }
      float m = z[0];
#pragma unroll
      for (int k = 1; k < TJ * 4; ++k) m = fmaxf(m, z[k]);
      const float m2 = row_max(m) * kLog2e;
      const float at = m2 == -INFINITY ? 0.f : m2;  // (columns past N alone)
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < TJ * 4; ++k) s += __builtin_amdgcn_exp2f(__builtin_fmaf(z[k], kLog2e, -at));
      s = row_sum(s);
      if (lg == 0 && live) part[((int64_t)(row >> 4) * parts + p) * 16 + l16] = XentPart{m2, s};
      __builtin_amdgcn_sched_barrier(0);  // (a row block at a time, or its values are spilled)
    }
  }
};

// (362 us for 2048 rows, hidden 2048, vocabulary 50304, where the product that
// stores z takes 346.)  dz in place of z: mult 2^(z log2 e - lse2), of the label mult
// (p - 1), zero past the vocabulary.
struct XentGrad {
  static constexpr bool kSized = true, kGathers = true, kStarts = false, kMaps = true, kReduces = false;
  const XentHead* head;
  const int* rows;
  const int* label;
  const float* lse2;
  const float* mult;
  const float* miss;  // the label's p - 1
  int v0;      // the piece's first column in the vocabulary
  int n_real;  // columns of the vocabulary in it
  int twice;   // odd rows hold what the rounding of the even ones left

  __device__ __forceinline__ void size(GemmArgs& g) const {
    g.M = min(g.M, head->count);
    g.c_bytes = g.M > 0 ? (uint32_t)(((int64_t)(g.M - 1) * g.ldc + g.N) * 2) : 0;
  }

  template <bool FP16, int TI, int TJ>
  __device__ __forceinline__ void map(f32x4_t (&acc)[TI][TJ], int row0, int col0, int M, int) const {
    const int lane = threadIdx.x & 63, l16 = lane & 15, lg = lane >> 4;
    const bool edge = col0 + TJ * 16 > n_real;
    float at[TI], f[TI], q[TI];
    int t[TI];
#pragma unroll
    for (int i = 0; i < TI; ++i) {
      const int row = min(row0 + i * 16 + l16, M - 1);  // (rows past M are not stored)
      at[i] = lse2[row];
      f[i] = mult[row];
      q[i] = miss[row];
      t[i] = label[row] - v0 - col0;
    }
#pragma unroll
    for (int i = 0; i < TI; ++i) {
#pragma unroll
      for (int j = 0; j < TJ; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          acc[i][j][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][e], kLog2e, -at[i]));
      if (__ballot(t[i] >= 0 && t[i] < TJ * 16)) {
#pragma unroll
        for (int j = 0; j < TJ; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (t[i] == j * 16 + lg * 4 + e) acc[i][j][e] = q[i];
      }
#pragma unroll
      for (int j = 0; j < TJ; ++j) acc[i][j] *= f[i];
      if (edge) {
#pragma unroll
        for (int j = 0; j < TJ; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (col0 + j * 16 + lg * 4 + e >= n_real) acc[i][j][e] = 0.f;
      }
      if (twice) {
        const bool rest = l16 & 1;
#pragma unroll
        for (int j = 0; j < TJ; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float v = acc[i][j][e], high = FP16 ? h2f_bits(f2h_bits(v)) : bf2f(f2bf(v));
            acc[i][j][e] = !rest ? v : __builtin_isfinite(high) ? v - high : 0.f;
          }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
};

// dh of a piece: the list's rows of dz.  Its 64 tiles at 2048 rows of hidden 2048 are
// a quarter of the chip, so the depth is split (324 us, 1.30 PFLOP/s); the fp32 slices
// are added to piece by piece and joined in xent_finish_kernel.
struct XentRows {
  static constexpr bool kSized = true, kGathers = false, kStarts = false, kMaps = false, kReduces = false;
  const XentHead* head;

  __device__ __forceinline__ void size(GemmArgs& g) const {
    g.M = min(g.M, head->count);
    g.a_bytes = g.M > 0 ? (uint32_t)(((int64_t)(g.M - 1) * g.lda + g.K) * 2) : 0;
    g.c_bytes = g.c_bytes && g.M > 0 ? (uint32_t)(((int64_t)(g.M - 1) * g.ldc + g.N) * 4) : 0;
  }
};

// dW of a piece: the list's rows are its depth (369 us, 1.14 PFLOP/s, of 2048 rows,
// hidden 2048, vocabulary 50304: 31 k-tiles of 64, then 206 MB stored).
struct XentDepth {
  static constexpr bool kSized = true, kGathers = false, kStarts = false, kMaps = false, kReduces = false;
  const XentHead* head;

  __device__ __forceinline__ void size(GemmArgs& g) const {
    g.K = min(g.K, head->count);
    g.alpha = head->alpha;
    // (dz has whole 16-byte units behind its last column)
    g.a_bytes = g.K > 0 ? (uint32_t)(((int64_t)(g.K - 1) * g.lda + (g.M + 7) / 8 * 8) * 2) : 0;
    g.b_bytes = g.K > 0 ? (uint32_t)(((int64_t)(g.K - 1) * g.ldb + g.N) * 2) : 0;
  }
};

// ------------------------------------------------------------- row lists --
// One workgroup lists the rows that take part, in order, 8192 a trip (2048 rows 5.3
// us, 8192 rows 7.5: a launch and its loads' latency).  Forward (dloss
// NULL): ignored rows get loss 0 here.  Backward: also each listed row's
// statistics and powers of two, and where each row went (`at`, -1: nowhere).
struct XentList {
  const int64_t* labels;
  int64_t ignore;
  int64_t n;
  int64_t vocab;
  XentHead* head;
  int* rows;
  int* label;
  float* loss;  // forward
  int* bad;
  const float* dloss;  // backward
  const float* lse;    // [2][n], the loss behind it
  int* at;
  int* exps;
  float* lse2;
  float* mult;
  float* miss;
  float* back;
  int shift;  // dz's power of two
  int twice;  // every row is listed twice (backward)
};
constexpr int kListThreads = 1024;

// e with 1 <= |v| 2^-e < 2 (0 of what is not finite)
__device__ __forceinline__ int exponent_of(float v) {
  return __builtin_isfinite(v) && v != 0.f ? ilogbf(v) : 0;
}

__global__ void __launch_bounds__(kListThreads) xent_list_kernel(XentList g) {
  constexpr int U = 8, WAVES = kListThreads / 64;  // rows of a thread a trip
  __shared__ int counts[U * WAVES], highs[WAVES];
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const bool back = g.dloss != nullptr;
  int base = 0, high = -1000;
  bool wild = false;
  for (int64_t r0 = 0; r0 < g.n; r0 += U * kListThreads) {
    int64_t t[U];
    float d[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t r = r0 + u * kListThreads + tid;
      t[u] = r < g.n ? g.labels[r] : g.ignore;
      d[u] = back && r < g.n ? g.dloss[r] : 1.f;
    }
    uint64_t on[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      on[u] = __ballot(t[u] != g.ignore && d[u] != 0.f);
      if (lane == 0) counts[u * WAVES + wid] = __popcll(on[u]);
    }
    __syncthreads();
    // rows before each wave's of each step, in every wave: two entries a lane
    static_assert(U * WAVES == 128, "two entries a lane");
    const int c0 = counts[2 * lane], c1 = counts[2 * lane + 1];
    int incl = c0 + c1;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(incl, o);
      if (lane >= o) incl += v;
    }
    const int excl = incl - c0 - c1, total = __shfl(incl, 63);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t r = r0 + u * kListThreads + tid;
      const int entry = u * WAVES + wid, lo = __shfl(excl, entry >> 1), first = __shfl(c0, entry >> 1);
      const int at = base + lo + (entry & 1 ? first : 0) + __popcll(on[u] & ((1ull << lane) - 1));
      if (r >= g.n) continue;
      if (!(on[u] >> lane & 1)) {
        if (back)
          g.at[r] = -1;
        else
          g.loss[r] = 0.f;
        continue;
      }
      wild |= t[u] < 0 || t[u] >= g.vocab;
      const int e = exponent_of(d[u]), first_at = at << g.twice;
      if (back) {
        if (__builtin_isfinite(d[u])) high = max(high, e);
        g.at[r] = first_at;
      }
      for (int to = first_at; to <= first_at + g.twice; ++to) {
        g.rows[to] = (int)r;
        g.label[to] = (int)(t[u] < 0 ? 0 : t[u] >= g.vocab ? g.vocab - 1 : t[u]);
        if (!back) continue;
        g.exps[to] = e;
        g.lse2[to] = g.lse[r];
        g.miss[to] = expm1f(-g.lse[g.n + r]);
        g.mult[to] = ldexpf(d[u], g.shift - e);
        g.back[to] = ldexpf(1.f, e - g.shift);
      }
    }
    base += total;
    __syncthreads();  // (counts are free for the next trip)
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) high = max(high, __shfl_xor(high, o));
  if (lane == 0) highs[wid] = high;
  __syncthreads();
  for (int w = 0; w < WAVES; ++w) high = max(high, highs[w]);
  if (high == -1000) high = 0;
  if (tid == 0) *g.head = XentHead{base << g.twice, high, ldexpf(1.f, high - g.shift)};
  if (wild && !back) *g.bad = 1;
}

// ------------------------------------------------------------------ join --
// A workgroup joins R rows: 1024 / R threads a row, some parts of each in flight,
// then a tree.  `lse` [2][n]: in the log2 domain, then the loss.  Latency: 4.0 us for 2048 rows of 393 parts.
// A whole 16 rows' lines lie together, but few rows of many parts are done sooner two
// a workgroup (forward, 16 / 2, us): one row of 50304 44.6 / 42.8, of 131072 35.2 /
// 30.6, 64 rows 47.7 / 46.4 and 34.5 / 31.5; 64 rows of 1000 12.0 / 12.3, 256 of 131072
// 40.5 / 41.5.
constexpr int kJoinThreads = 1024;
constexpr int64_t kFewRows = 64, kManyParts = 256;
__device__ __forceinline__ XentPart join(XentPart a, XentPart b) {
  const float m = fmaxf(a.m2, b.m2), at = m == -INFINITY ? 0.f : m;
  return XentPart{m, a.s * __builtin_amdgcn_exp2f(a.m2 - at) + b.s * __builtin_amdgcn_exp2f(b.m2 - at)};
}
template <int R>
__global__ void __launch_bounds__(kJoinThreads) xent_join_kernel(const XentHead* head, const int* rows,
                                                                 const XentPart* part, const float* picked, int parts,
                                                                 float* loss, float* lse, int64_t n_rows) {
  __shared__ XentPart red[kJoinThreads / R][R];
  const int r = threadIdx.x % R, k = threadIdx.x / R, row = blockIdx.x * R + r, n = head->count;
  if ((int)blockIdx.x * R >= n) return;
  XentPart v{-INFINITY, 0.f};
  if (row < n) {
    const XentPart* mine = part + (int64_t)(row >> 4) * parts * 16 + (row & 15);
    constexpr int STEP = kJoinThreads / R, U = R == 16 ? 8 : 4;  // parts in flight
    for (int p = k; p < parts; p += U * STEP) {
      XentPart in[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        in[u] = p + u * STEP < parts ? mine[(int64_t)(p + u * STEP) * 16] : XentPart{-INFINITY, 0.f};
#pragma unroll
      for (int u = 0; u < U; ++u) v = join(v, in[u]);
    }
  }
  red[k][r] = v;
  for (int half = kJoinThreads / R / 2; half; half >>= 1) {
    __syncthreads();
    if (k < half) red[k][r] = join(red[k][r], red[k + half][r]);
  }
  if (k == 0 && row < n) {
    const XentPart t = red[0][r];
    const float l = log2f(t.s);  // (near one the instruction alone is off by more than s is)
    // (apart from each other the large terms cancel exactly first)
    const int64_t o = rows[row];
    loss[o] = lse[n_rows + o] = kLn2 * (__builtin_fmaf(-picked[row], kLog2e, t.m2) + l);
    lse[o] = t.m2 + l;
  }
}

// ---------------------------------------------------------------- gather --
// The list's rows of h, each times its power of two: dW's second operand (5.4 us for
// 2048 rows of 2048, 10.1 for 5734 of 8192).
template <bool FP16>
__global__ void __launch_bounds__(256) xent_gather_kernel(const XentHead* head, const int* rows, const int* exps,
                                                          const uint16_t* h, int64_t ldh, uint16_t* out, int hidden) {
  const int row = blockIdx.x;
  if (row >= head->count) return;
  const uint16_t* src = h + (int64_t)rows[row] * ldh;
  const float f = ldexpf(1.f, exps[row] - head->high);
  for (int c = threadIdx.x * 8; c < hidden; c += 256 * 8) {
    const uint4 raw = *reinterpret_cast<const uint4*>(src + c);
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    uint32_t o[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint16_t lo = (uint16_t)w[k], hi = (uint16_t)(w[k] >> 16);
      o[k] = FP16 ? f2h_pair(h2f_bits(lo) * f, h2f_bits(hi) * f) : f2bf_pair(bf2f(lo) * f, bf2f(hi) * f);
    }
    *reinterpret_cast<uint4*>(out + (int64_t)row * hidden + c) = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

// dh of every row: the sum of its slices (of both of its places, where it was
// listed twice) times its power of two, rounded once; zeros where it took no part
// (2048 rows of 2048 in four slices: 19 us, 4.0 TB/s).
template <bool FP16>
__global__ void __launch_bounds__(256) xent_finish_kernel(const int* at, const float* back, const float* slices,
                                                          int n_slices, int64_t stride, int twice, uint16_t* dh,
                                                          int hidden) {
  const int64_t row = blockIdx.x;
  const int p = at[row];
  const float f = p < 0 ? 0.f : back[p];
  for (int c = threadIdx.x * 8; c < hidden; c += 256 * 8) {
    uint32_t o[4] = {0, 0, 0, 0};
    if (p >= 0) {
      float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      for (int s = 0; s < n_slices << twice; ++s) {
        const float4* src = reinterpret_cast<const float4*>(slices + (s >> twice) * stride +
                                                            (int64_t)(p + (s & twice)) * hidden + c);
        const float4 x = src[0], y = src[1];
        v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w;
        v[4] += y.x; v[5] += y.y; v[6] += y.z; v[7] += y.w;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
        o[k] = FP16 ? f2h_pair(v[2 * k] * f, v[2 * k + 1] * f) : f2bf_pair(v[2 * k] * f, v[2 * k + 1] * f);
    }
    *reinterpret_cast<uint4*>(dh + row * hidden + c) = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

// ------------------------------------------------------------------ host --
template <bool A_K, bool B_K, bool FP16, bool SHORT, class X>
static int launch_product(int tile, const GemmArgs& args, const X& x, hipStream_t s, int splits = 1) {
  const int64_t tiles = (int64_t)((args.M + tile - 1) / tile) * ((args.N + tile - 1) / tile) * splits;
  const dim3 grid((unsigned)tiles);
  GemmArgs a = args;
  a.splits = splits;
  if (tile == 256) {
    if (SHORT || a.K % 64)  // (SHORT: the depth is the device's, its last k-tile of any length)
      gemm256_m16_kernel<A_K, B_K, FP16, true, X><<<grid, 256, 0, s>>>(a, x);
    else if constexpr (!SHORT)
      gemm256_m16_kernel<A_K, B_K, FP16, false, X><<<grid, 256, 0, s>>>(a, x);
  } else if (tile == 128) {
    gemm_ring_kernel<128, A_K, B_K, FP16, X><<<grid, 256, 0, s>>>(a, x);
  } else {
    gemm_ring_kernel<64, A_K, B_K, FP16, X><<<grid, 256, 0, s>>>(a, x);
  }
  ETH_CHECK_LAUNCH("eth_linear_xent");
  return ETH_OK;
}

constexpr int64_t kMaxBytes = (1LL << 31) - 1;
// Workspace for a piece of dz, the last one apart, which may be half as long again (a
// piece is 256 columns at least).
constexpr int64_t kPieceBytes = 256LL << 20;

static int64_t up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }
static int64_t room(int64_t bytes) { return up(bytes, 256); }

// Columns of W that a launch's 32-bit offsets reach, whole 256s (check_xent: one of them
// at least).
static int64_t reach(int64_t ldw) { return std::max<int64_t>(256, kMaxBytes / 2 / ldw / 256 * 256); }

// The product [M, N] x K deep in whole rounds of 256x256 tiles and a rest along N
// in its own best tile, where the time model promises 2 %: `first` columns, then the
// others (`first` N: all in one).  Uncut / cut (us): 2048 rows of hidden 2048,
// vocabulary 50304 (1576 tiles, 6.2 rounds) forward 352 / 340, backward 1098 / 1060;
// 1001 rows of 4096, 50257, fp16: 373 / 326, 1176 / 1127.
struct XentCut {
  int64_t first;
  int tile, rest;
};
static XentCut cut_columns(int64_t M, int64_t N, int64_t K, GemmForm form) {
  XentCut c{N, plan_tile(M, N, K, true, form), 0};
  const int64_t tm = (M + 255) / 256, tn = (N + 255) / 256, n1 = tm * tn / 256 * 256 / tm * 256;
  if (c.tile != 256 || n1 <= 0 || n1 >= N) return c;
  const int rest = plan_tile(M, N - n1, K, true, form);
  if (tile_time(256, M, n1, K, 1, form) + tile_time(rest, M, N - n1, K, 1, form) <
      0.98 * tile_time(256, M, N, K, 1, form))
    c = XentCut{n1, 256, rest};
  return c;
}

struct XentForward {
  int64_t chunk;  // columns of a cut
  int64_t parts;  // of a row
  int64_t rows, label, picked, part, bytes;  // workspace offsets
};
// a wave has half a tile's columns
static int64_t parts_of(int64_t cols, int tile) { return up(cols, tile) / (tile / 2); }
static XentForward plan_forward(int64_t n, int64_t hidden, int64_t vocab, int64_t ldw) {
  XentForward p;
  p.chunk = std::min(vocab, reach(ldw));
  p.parts = 0;
  for (int64_t v = 0; v < vocab; v += p.chunk) {
    const int64_t cols = std::min(p.chunk, vocab - v);
    const XentCut c = cut_columns(n, cols, hidden, GemmForm{false, hidden % 64 != 0, 0});
    p.parts += parts_of(c.first, c.tile) + (c.rest ? parts_of(cols - c.first, c.rest) : 0);
  }
  int64_t o = room(sizeof(XentHead));
  p.rows = o, o += room(n * 4);
  p.label = o, o += room(n * 4);
  p.picked = o, o += room(n * 4);
  p.part = o, o += room(up(n, 16) * p.parts * (int64_t)sizeof(XentPart));
  p.bytes = o;
  return p;
}

// Rows up to which each is listed twice: few enough not to average dz's roundings,
// and for the products to wait for W and dW rather than for the matrix cores.
// Backward of hidden 2048, vocabulary 50304, listed once / twice (us): 1 row 216 / 222,
// 32 rows 217 / 223, 64 rows 221 / 247, 128 rows 239 / 282; of 4096, 65536: 461 / 478,
// 470 / 490, 482 / 535, 520 / 622.
constexpr int64_t kTwiceRows = 64;

struct XentBackward {
  int twice;
  int64_t n;            // rows of the list, at most
  int splits;           // of dh's depth
  int64_t k_split;
  int pieces;
  int64_t piece, last, ldz;  // columns of a piece, of the last one, of their rows
  int64_t rows, label, at, exps, lse2, mult, miss, back, gathered, dz, dh, bytes;
};
static XentBackward plan_backward(int64_t rows, int64_t hidden, int64_t vocab, int64_t ldw, bool need_dh, bool need_dw) {
  XentBackward p;
  p.twice = rows <= kTwiceRows;
  const int64_t n = p.n = rows << p.twice;
  int64_t most = std::max<int64_t>(256, kPieceBytes / (2 * n) / 256 * 256);
  const int64_t within = reach(std::max(ldw, hidden));
  most = std::min(most, within);
  // whole rounds of dW's tiles where they fit
  const int64_t tn = (hidden + 255) / 256;
  int64_t unit = 256;
  while (unit < 65536 && unit / 256 * tn % 256) unit *= 2;
  const int64_t whole = most >= unit ? most / unit * unit : most;
  // equal pieces of at most that, or whole ones and a last one of half to three halves
  int64_t many = std::max<int64_t>(1, (vocab + whole / 2 - 1) / whole);
  p.piece = std::min(up(vocab, 8), whole);
  p.last = vocab - (many - 1) * p.piece;
  if (p.last > within) {  // (what a launch's offsets do not reach is a short piece of its own)
    ++many;
    p.last -= p.piece;
  }
  p.pieces = (int)many;
  p.ldz = up(std::max(p.piece, p.last), 8);
  // dh has few tiles and a deep product: split until the chip is full
  const int64_t tiles = (n + 255) / 256 * ((hidden + 255) / 256);
  p.splits = 1;
  // (the first piece fills every slice; the last may be deeper: its splits are)
  const int64_t first = p.pieces > 1 ? p.piece : p.ldz;
  while (p.splits < 16 && tiles * p.splits * 2 <= 256 && first / (p.splits * 2) >= 512) p.splits *= 2;
  p.k_split = up((first + p.splits - 1) / p.splits, 64);
  p.splits = (int)((first + p.k_split - 1) / p.k_split);
  int64_t o = room(sizeof(XentHead));
  for (int64_t* at : {&p.rows, &p.label, &p.at, &p.exps, &p.lse2, &p.mult, &p.miss, &p.back}) *at = o, o += room(n * 4);
  p.gathered = o, o += need_dw ? room(n * hidden * 2) : 0;
  p.dz = o, o += room(n * p.ldz * 2);
  p.dh = o, o += need_dh ? room(p.splits * n * hidden * 4) : 0;
  p.bytes = o;
  return p;
}

static int check_xent(const char* name, const void* h, int64_t ldh, const void* w, int64_t ldw, const int64_t* labels,
                      const void* workspace, int64_t n, int64_t hidden, int64_t vocab, int dtype) {
  ETH_CHECK_ARG(dtype == ETH_BF16 || dtype == ETH_F16, "%s: h and W must be bf16 or fp16", name);
  // (256 columns of dz, a piece's least, stay within 32-bit offsets)
  ETH_CHECK_ARG(n > 0 && hidden > 0 && vocab > 0 && n < (1LL << 21) && vocab <= (1LL << 24) && hidden < (1LL << 20),
                "%s: bad shape: %lld rows, hidden %lld, vocabulary %lld", name, (long long)n, (long long)hidden,
                (long long)vocab);
  // (a launch takes 256 rows of W at least)
  const int64_t apart = std::min<int64_t>(vocab, 256) - 1;
  ETH_CHECK_ARG(apart == 0 || ldw <= (kMaxBytes / 2 - hidden) / apart,
                "%s: rows of W %lld elements apart: 256 of them above 2 GiB are not supported", name, (long long)ldw);
  ETH_CHECK_ARG(h && w && labels && workspace, "%s: null operand", name);
  ETH_CHECK_ARG(hidden % 8 == 0 && ldh % 8 == 0 && ldw % 8 == 0 && ldh >= hidden && ldw >= hidden,
                "%s: hidden (%lld) and row strides (%lld, %lld) must be multiples of 8", name, (long long)hidden,
                (long long)ldh, (long long)ldw);
  ETH_CHECK_ARG(((uintptr_t)h & 15) == 0 && ((uintptr_t)w & 15) == 0 && ((uintptr_t)workspace & 255) == 0,
                "%s: h and W must be 16-byte, the workspace 256-byte aligned", name);
  ETH_CHECK_ARG(((n - 1) * ldh + hidden) * 2 <= kMaxBytes, "%s: rows above 2 GiB are not supported", name);
  ETH_CHECK_ARG((n + 63) / 64 * ((vocab + 63) / 64) < (1LL << 24), "%s: %lld rows of %lld logits are too many", name,
                (long long)n, (long long)vocab);
  return ETH_OK;
}

static GemmArgs product_args(const void* A, int64_t a_elems, int64_t lda, const void* B, int64_t b_elems, int64_t ldb,
                             int64_t M, int64_t N, int64_t K) {
  GemmArgs a{};
  a.A = (const uint16_t*)A;
  a.B = (const uint16_t*)B;
  a.a_bytes = (uint32_t)(a_elems * 2);
  a.b_bytes = (uint32_t)(b_elems * 2);
  a.M = (int)M;
  a.N = (int)N;
  a.K = (int)K;
  a.lda = lda;
  a.ldb = ldb;
  a.alpha = 1.f;
  return a;
}

template <bool FP16>
static int xent_forward(const uint16_t* h, int64_t ldh, const uint16_t* w, int64_t ldw, const XentForward& p, char* ws,
                        int64_t n, int64_t hidden, int64_t vocab, hipStream_t s) {
  int part0 = 0;
  auto columns = [&](int64_t v0, int64_t cols, int tile) {
    const GemmArgs a = product_args(h, (n - 1) * ldh + hidden, ldh, w + v0 * ldw, (cols - 1) * ldw + hidden, ldw, n,
                                    cols, hidden);
    const XentStats x{(const XentHead*)ws, (const int*)(ws + p.rows), (const int*)(ws + p.label),
                      (XentPart*)(ws + p.part), (float*)(ws + p.picked), (int)v0, part0, (int)p.parts};
    part0 += (int)parts_of(cols, tile);
    return launch_product<true, true, FP16, false>(tile, a, x, s);
  };
  for (int64_t v0 = 0; v0 < vocab; v0 += p.chunk) {
    const int64_t cols = std::min(p.chunk, vocab - v0);
    const XentCut c = cut_columns(n, cols, hidden, GemmForm{false, hidden % 64 != 0, 0});
    int rc = columns(v0, c.first, c.tile);
    if (rc == ETH_OK && c.rest) rc = columns(v0 + c.first, cols - c.first, c.rest);
    if (rc != ETH_OK) return rc;
  }
  return ETH_OK;
}

template <bool FP16>
static int xent_backward(const uint16_t* h, int64_t ldh, const uint16_t* w, int64_t ldw, const XentBackward& p,
                         char* ws, int64_t n_rows, int64_t hidden, int64_t vocab, uint16_t* dh, void* dw, int dw_dtype,
                         int accumulate, hipStream_t s) {
  const int64_t n = p.n;
  const XentHead* head = (const XentHead*)ws;
  const int* rows = (const int*)(ws + p.rows);
  uint16_t* gathered = (uint16_t*)(ws + p.gathered);
  uint16_t* dz = (uint16_t*)(ws + p.dz);
  float* slices = (float*)(ws + p.dh);
  if (dw) {
    xent_gather_kernel<FP16><<<(unsigned)n, 256, 0, s>>>(head, rows, (const int*)(ws + p.exps), h, ldh, gathered,
                                                         (int)hidden);
    ETH_CHECK_LAUNCH("eth_linear_xent_bwd");
  }
  const int esz = dw_dtype == ETH_F32 ? 4 : 2;
  for (int piece = 0; piece < p.pieces; ++piece) {
    const int64_t v0 = piece * p.piece, real = piece == p.pieces - 1 ? p.last : p.piece, cols = up(real, 8);
    const uint16_t* wp = w + v0 * ldw;
    const int64_t w_elems = (real - 1) * ldw + hidden;
    int rc = ETH_OK;
    auto z_columns = [&](int64_t c0, int64_t many, int tile) {
      const int64_t there = std::min(many, real - c0);
      GemmArgs a = product_args(h, (n_rows - 1) * ldh + hidden, ldh, wp + c0 * ldw, (there - 1) * ldw + hidden, ldw, n, many,
                                hidden);
      a.C = dz + c0;
      a.ldc = p.ldz;
      a.c_dtype = FP16 ? ETH_F16 : ETH_BF16;
      a.c_vec = true;
      const XentGrad grad{head, rows, (const int*)(ws + p.label), (const float*)(ws + p.lse2),
                          (const float*)(ws + p.mult), (const float*)(ws + p.miss), (int)(v0 + c0), (int)there, p.twice};
      return launch_product<true, true, FP16, false>(tile, a, grad, s);
    };
    const XentCut zc = cut_columns(n, cols, hidden, GemmForm{false, hidden % 64 != 0, 0});
    rc = z_columns(0, zc.first, zc.tile);
    if (rc == ETH_OK && zc.rest) rc = z_columns(zc.first, cols - zc.first, zc.rest);
    if (rc != ETH_OK) return rc;
    if (dh) {
      GemmArgs d = product_args(dz, (n - 1) * p.ldz + cols, p.ldz, wp, w_elems, ldw, n, hidden, cols);
      d.C = slices;
      d.ldc = hidden;
      d.c_dtype = ETH_F32;
      d.c_vec = true;
      d.flags = v0 ? ETH_GEMM_ACCUMULATE : 0;
      const bool wide = wide_takes(n, hidden, hidden, 4, true);
      d.c_bytes = wide ? 1 : 0;
      // (the same split of the depth in every piece: some need fewer splits)
      const bool deeper = piece && cols > p.splits * p.k_split;
      d.k_split = (int)(deeper ? up((cols + p.splits - 1) / p.splits, 64) : p.k_split);
      d.c_split_stride = n * hidden;
      const int splits = (int)((cols + d.k_split - 1) / d.k_split);
      if (!wide) d.k_split = 0;
      rc = launch_product<true, false, FP16, false>(wide ? 256 : 128, d, XentRows{head}, s, wide ? splits : 1);
      if (rc != ETH_OK) return rc;
    }
    if (dw) {
      auto w_rows = [&](int64_t r0, int64_t many, int tile) {
        GemmArgs d = product_args(dz + r0, 0, p.ldz, gathered, 0, hidden, many, hidden, n);
        d.C = (char*)dw + (v0 + r0) * hidden * esz;
        d.ldc = hidden;
        d.c_dtype = dw_dtype;
        d.flags = accumulate ? ETH_GEMM_ACCUMULATE : 0;
        d.c_vec = true;
        const bool wide = wide_takes(many, hidden, hidden, esz, true);
        d.c_bytes = wide ? (uint32_t)(many * hidden * esz) : 0;
        return launch_product<false, false, FP16, true>(wide || tile != 256 ? tile : 128, d, XentDepth{head}, s);
      };
      // (the same rule with dW's rows for columns)
      const XentCut wc = cut_columns(hidden, real, n, GemmForm{esz == 4, false, 0});
      rc = w_rows(0, wc.first, wc.tile);
      if (rc == ETH_OK && wc.rest) rc = w_rows(wc.first, real - wc.first, wc.rest);
      if (rc != ETH_OK) return rc;
    }
  }
  if (dh) {
    const bool wide = wide_takes(n, hidden, hidden, 4, true);
    const int filled = wide ? p.splits : 1;
    xent_finish_kernel<FP16><<<(unsigned)n_rows, 256, 0, s>>>((const int*)(ws + p.at), (const float*)(ws + p.back), slices,
                                                         filled, n * hidden, p.twice, dh, (int)hidden);
    ETH_CHECK_LAUNCH("eth_linear_xent_bwd");
  }
  return ETH_OK;
}

}  // namespace eth

using namespace eth;

extern "C" int64_t eth_linear_xent_workspace(int64_t rows, int64_t hidden, int64_t vocab, int64_t ldw, int grads) {
  if (rows <= 0 || hidden <= 0 || vocab <= 0 || ldw < hidden) return 0;
  if (!grads) return plan_forward(rows, hidden, vocab, ldw).bytes;
  return plan_backward(rows, hidden, vocab, ldw, grads & 1, grads & 2).bytes;
}

extern "C" int eth_linear_xent_fwd(const void* h, int64_t ldh, const void* w, int64_t ldw, const int64_t* labels,
                                   int64_t ignore_index, float* loss, float* lse, void* workspace, int64_t rows,
                                   int64_t hidden, int64_t vocab, int* bad_index, int dtype, void* stream) {
  const int rc = check_xent("eth_linear_xent_fwd", h, ldh, w, ldw, labels, workspace, rows, hidden, vocab, dtype);
  if (rc != ETH_OK) return rc;
  ETH_CHECK_ARG(loss && lse && bad_index, "eth_linear_xent_fwd: null operand");
  const XentForward p = plan_forward(rows, hidden, vocab, ldw);
  char* ws = (char*)workspace;
  hipStream_t s = (hipStream_t)stream;
  XentList list{};
  list.labels = labels;
  list.ignore = ignore_index;
  list.n = rows;
  list.vocab = vocab;
  list.head = (XentHead*)ws;
  list.rows = (int*)(ws + p.rows);
  list.label = (int*)(ws + p.label);
  list.loss = loss;
  list.bad = bad_index;
  xent_list_kernel<<<1, kListThreads, 0, s>>>(list);
  ETH_CHECK_LAUNCH("eth_linear_xent_fwd");
  const int done = dtype == ETH_F16
                       ? xent_forward<true>((const uint16_t*)h, ldh, (const uint16_t*)w, ldw, p, ws, rows, hidden, vocab, s)
                       : xent_forward<false>((const uint16_t*)h, ldh, (const uint16_t*)w, ldw, p, ws, rows, hidden, vocab, s);
  if (done != ETH_OK) return done;
  const bool few = rows <= kFewRows && p.parts >= kManyParts;
  const auto join_rows = few ? xent_join_kernel<2> : xent_join_kernel<16>;
  join_rows<<<(unsigned)(few ? (rows + 1) / 2 : (rows + 15) / 16), kJoinThreads, 0, s>>>(
      (const XentHead*)ws, (const int*)(ws + p.rows), (const XentPart*)(ws + p.part), (const float*)(ws + p.picked),
      (int)p.parts, loss, lse, rows);
  ETH_CHECK_LAUNCH("eth_linear_xent_fwd");
  return ETH_OK;
}

extern "C" int eth_linear_xent_bwd(const void* h, int64_t ldh, const void* w, int64_t ldw, const int64_t* labels,
                                   int64_t ignore_index, const float* lse, const float* dloss, void* dh, void* dw,
                                   int dw_dtype, int accumulate, void* workspace, int64_t rows, int64_t hidden,
                                   int64_t vocab, int dtype, void* stream) {
  const int rc = check_xent("eth_linear_xent_bwd", h, ldh, w, ldw, labels, workspace, rows, hidden, vocab, dtype);
  if (rc != ETH_OK) return rc;
  ETH_CHECK_ARG(lse && dloss && (dh || dw), "eth_linear_xent_bwd: null operand");
  ETH_CHECK_ARG(((uintptr_t)dh & 15) == 0 && ((uintptr_t)dw & 15) == 0,
                "eth_linear_xent_bwd: dh and dW must be 16-byte aligned");
  ETH_CHECK_ARG(!dw || dw_dtype == dtype || dw_dtype == ETH_F32, "eth_linear_xent_bwd: bad dW type %d", dw_dtype);
  ETH_CHECK_ARG(!accumulate || !dw || dw_dtype == ETH_F32, "eth_linear_xent_bwd: accumulate needs fp32 dW");
  const XentBackward p = plan_backward(rows, hidden, vocab, ldw, dh != nullptr, dw != nullptr);
  char* ws = (char*)workspace;
  hipStream_t s = (hipStream_t)stream;
  XentList list{};
  list.labels = labels;
  list.ignore = ignore_index;
  list.n = rows;
  list.vocab = vocab;
  list.head = (XentHead*)ws;
  list.rows = (int*)(ws + p.rows);
  list.label = (int*)(ws + p.label);
  list.dloss = dloss;
  list.lse = lse;
  list.at = (int*)(ws + p.at);
  list.exps = (int*)(ws + p.exps);
  list.lse2 = (float*)(ws + p.lse2);
  list.mult = (float*)(ws + p.mult);
  list.miss = (float*)(ws + p.miss);
  list.back = (float*)(ws + p.back);
  list.shift = dtype == ETH_F16 ? 14 : 0;
  list.twice = p.twice;
  xent_list_kernel<<<1, kListThreads, 0, s>>>(list);
  ETH_CHECK_LAUNCH("eth_linear_xent_bwd");
  return dtype == ETH_F16 ? xent_backward<true>((const uint16_t*)h, ldh, (const uint16_t*)w, ldw, p, ws, rows, hidden,
                                                vocab, (uint16_t*)dh, dw, dw_dtype, accumulate, s)
                          : xent_backward<false>((const uint16_t*)h, ldh, (const uint16_t*)w, ldw, p, ws, rows, hidden,
                                                 vocab, (uint16_t*)dh, dw, dw_dtype, accumulate, s);
}
