// Row operators over logits [rows, V] (bf16, fp16 or fp32), beside the cross
// entropy: the log probabilities of given tokens with the row's entropy and
// its top alternatives, and the distillation loss on a teacher's top logits,
// forward and backward.
//
//   m = max z, s = sum exp(z - m), logp = (z - m) - log s, p = exp(logp)
//   token log probabilities:  logp[t], H = log s - sum e (z - m) / s, the k
//     largest logp with their ids (equal ones by the lowest id)
//     dz_j = g ([j = t] - p_j) - h p_j (logp_j + H)
//   distillation at temperature tau over the teacher's entries (id, u):
//     q = softmax(u / tau), p = softmax(z / tau)
//     loss = tau^2 sum q (log q - log p[id]),  dz_j = g tau (p_j - sum_{id = j} q)
//
// All arithmetic is fp32; the row's maximum and log s are kept apart, so that
// a large common offset of the logits costs no digits.  Rows are read once
// forward, read and written once backward: HBM bounds them (a large copy moves 5.15
// TB/s here; reads alone have reached 7.2).  Rows may start at
// any multiple of an element (odd vocabularies): vectors are loaded and stored
// with the alignment of an element, which the hardware takes.
#include <utility>

#include "common.h"

namespace eth {

// f(0) .. f(N - 1), each call's index a constant
template <class F, int... I>
__device__ __forceinline__ void each_place(std::integer_sequence<int, I...>, F f) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void each_place(F f) {
  each_place(std::make_integer_sequence<int, N>{}, f);
}

// Array length for N vectors of which every access has a constant index: the
// compiler makes one wide register, copied whole at every access, of an array of
// up to 32 words before it sees that, and takes a longer one apart.
constexpr int places_of(int n) { return n < 9 ? 9 : n; }

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLowest = -3.4028234663852886e38f;
// differences of logits are cut here before they meet a zero probability
// (0 * -inf); exp of it is 0
constexpr float kFarBelow = -1e4f;

typedef uint32_t lg_u32x4 __attribute__((ext_vector_type(4)));
typedef lg_u32x4 lg_u32x4_a2 __attribute__((aligned(2)));
typedef lg_u32x4 lg_u32x4_a4 __attribute__((aligned(4)));

// one 16-byte vector of E elements of a type
template <int DT>
struct Lg {
  static constexpr int E = 8;
  typedef uint16_t T;
  typedef lg_u32x4_a2 V;
  static __device__ __forceinline__ float one(T v) { return DT == ETH_F16 ? h2f_bits(v) : bf2f(v); }
  static __device__ __forceinline__ T round(float v) { return DT == ETH_F16 ? f2h_bits(v) : f2bf(v); }
  static __device__ __forceinline__ void unpack(const lg_u32x4& a, float (&x)[E]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[2 * j] = one((T)(a[j] & 0xffffu));
      x[2 * j + 1] = one((T)(a[j] >> 16));
    }
  }
  static __device__ __forceinline__ lg_u32x4 pack(const float (&x)[E]) {
    lg_u32x4 a;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      a[j] = DT == ETH_F16 ? f2h_pair(x[2 * j], x[2 * j + 1]) : f2bf_pair(x[2 * j], x[2 * j + 1]);
    return a;
  }
  static constexpr uint32_t kMinusInf = DT == ETH_F16 ? 0xfc00fc00u : 0xff80ff80u;
};
template <>
struct Lg<ETH_F32> {
  static constexpr int E = 4;
  typedef float T;
  typedef lg_u32x4_a4 V;
  static __device__ __forceinline__ float one(T v) { return v; }
  static __device__ __forceinline__ T round(float v) { return v; }
  static __device__ __forceinline__ void unpack(const lg_u32x4& a, float (&x)[E]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = __uint_as_float(a[j]);
  }
  static __device__ __forceinline__ lg_u32x4 pack(const float (&x)[E]) {
    lg_u32x4 a;
#pragma unroll
    for (int j = 0; j < 4; ++j) a[j] = __float_as_uint(x[j]);
    return a;
  }
  static constexpr uint32_t kMinusInf = 0xff800000u;
};

// Vectors base + threadIdx.x + i * STEP (i < NV) of the n elements at z, -inf
// past them; returns how many of the NV places hold anything for any thread of
// the workgroup, the same for all: what the passes over them visit.  Lanes past
// the row load its last whole vector instead, and only the last place is mended:
// with a choice at every place the compiler unpacks there and spills.  The
// partial vector that n % E elements end a row with is loaded one by one.
template <int DT, int NV, int STEP>
__device__ __forceinline__ int load_vecs(lg_u32x4 (&v)[places_of(NV)], const typename Lg<DT>::T* z, int base, int n) {
  constexpr int E = Lg<DT>::E;
  const int whole = n / E, rest = n - whole * E, first = base + threadIdx.x;
  const int places = min((whole + (rest > 0) - base + STEP - 1) / STEP, NV);
  const int last = max(whole - 1, 0);
  each_place<NV>([&](auto i) __attribute__((always_inline)) {
    if (i < places && whole > 0)
      v[i] = *reinterpret_cast<const typename Lg<DT>::V*>(z + (int64_t)min(first + i * STEP, last) * E);
  });
  const int end = first + (places - 1) * STEP;  // the last place's vector
  lg_u32x4 t = {Lg<DT>::kMinusInf, Lg<DT>::kMinusInf, Lg<DT>::kMinusInf, Lg<DT>::kMinusInf};
  if (end == whole && rest) {
    float x[E];
    Lg<DT>::unpack(t, x);
#pragma unroll
    for (int j = 0; j < E - 1; ++j)
      if (j < rest) x[j] = Lg<DT>::one(z[whole * E + j]);
    t = Lg<DT>::pack(x);  // (values of the type: exact)
  }
  asm volatile("" : "+v"(t));  // (whole words: not the elements it was made of)
  each_place<NV>([&](auto i) __attribute__((always_inline)) {
    if (i == places - 1 && end >= whole) v[i] = t;
  });
  return places;
}
// A vector's elements for one pass, the vector not known to be what it was:
// otherwise what was unpacked for one pass is kept for the next, and with it
// twice the registers or, spilled, much more.
template <int DT>
__device__ __forceinline__ void unpack_again(lg_u32x4& v, float (&x)[Lg<DT>::E]) {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" : "+v"(v));
  Lg<DT>::unpack(v, x);
}
// vector i of the n elements at d.  STREAM: past the caches, for gradients that
// would not stay in them (bf16 [4096, 50304] 145.8 -> 141.1 us, [4096, 32000] 95.0
// -> 90.8, fp32 [1024, 50304] 72.4 -> 69.4; but [8192, 8000] 43.6 -> 46.4).
constexpr int64_t kStreamBytes = 192LL << 20;
template <int DT, bool STREAM>
__device__ __forceinline__ void store_vec(typename Lg<DT>::T* d, int i, int n, const float (&x)[Lg<DT>::E]) {
  constexpr int E = Lg<DT>::E;
  if ((i + 1) * E <= n) {
    typename Lg<DT>::V* p = reinterpret_cast<typename Lg<DT>::V*>(d + (int64_t)i * E);
    const typename Lg<DT>::V v = Lg<DT>::pack(x);
    if constexpr (STREAM)
      __builtin_nontemporal_store(v, p);
    else
      *p = v;
  } else {
#pragma unroll
    for (int j = 0; j < E; ++j)
      if (i * E + j < n) d[i * E + j] = Lg<DT>::round(x[j]);
  }
}

__device__ __forceinline__ float exp_f(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }

// max, sum of exponentials and sum of exponentials times their difference from
// the max, of a part of a row
struct RowStat {
  float m, s, a;
};
// the same relative to a larger maximum M
__device__ __forceinline__ RowStat at_max(const RowStat& r, float M) {
  const float d = fmaxf(r.m - M, kFarBelow), f = exp_f(d);
  return RowStat{M, r.s * f, (r.a + r.s * d) * f};
}
// over the workgroup (NT threads), in every thread; `red` holds 3 * NT / 64 floats
template <int NT>
__device__ __forceinline__ RowStat block_stat(RowStat r, float* red) {
  constexpr int W = NT / 64;
  r = at_max(r, wave_max(r.m));
  r.s = wave_sum(r.s);
  r.a = wave_sum(r.a);
  if ((threadIdx.x & 63) == 0) {
    const int w = threadIdx.x >> 6;
    red[w] = r.m;
    red[W + w] = r.s;
    red[2 * W + w] = r.a;
  }
  __syncthreads();
  float M = red[0];
#pragma unroll
  for (int w = 1; w < W; ++w) M = fmaxf(M, red[w]);
  RowStat t{M, 0.f, 0.f};
#pragma unroll
  for (int w = 0; w < W; ++w) {
    const RowStat x = at_max(RowStat{red[w], red[W + w], red[2 * W + w]}, M);
    t.s += x.s;
    t.a += x.a;
  }
  return t;
}

// ---------------------------------------------------- token log probabilities --
constexpr int kLogpThreads = 512;  // of a workgroup for a long row's part
constexpr int kLogpTop = 128;   // most alternatives
constexpr int kLogpCand = 1024; // candidates that the sort takes (a multiple of 16)
constexpr int kLogpHits = 512;  // vectors with candidates
constexpr int kLogpVecs = 8;    // vectors that a thread has in flight
constexpr int kLogpTrips = 2;   // times that, at most, in a part of a row

// floats as whole numbers of the same order: -0 as +0, NaN above everything
__device__ __forceinline__ uint32_t order_of(float v) {
  const uint32_t b = __float_as_uint(v + 0.f);
  return v != v ? 0xffffffffu : (b & 0x80000000u ? ~b : b | 0x80000000u);
}
__device__ __forceinline__ float of_order(uint32_t o) {
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
// value first, then the lower index: all keys of a row differ
__device__ __forceinline__ uint64_t key_of(float v, int index) {
  return (uint64_t)order_of(v) << 32 | ~(uint32_t)index;
}
__device__ __forceinline__ int64_t index_of(uint64_t key) { return (int64_t)(uint32_t)~(uint32_t)key; }

struct LogpArgs {
  const void* z;
  int64_t ld;
  int V;
  const int64_t* tokens;
  int64_t ignore;
  float* logprob;
  float* entropy;
  float2* stats;  // max, log of the sum (-inf: no finite logit)
  float* top;     // [rows, k]
  int64_t* ids;
  int k;
  int* bad;
  int parts;          // workgroups per row
  int part;           // elements of a part (a multiple of a vector's)
  float4* part_stat;  // [rows, parts]
  uint64_t* part_key; // [rows, parts, k]
};

__device__ __forceinline__ bool logp_ignored(const LogpArgs& a, int64_t row) {
  if (a.tokens[row] != a.ignore) return false;
  for (int i = threadIdx.x; i < a.k; i += blockDim.x) {
    a.top[row * a.k + i] = -INFINITY;
    a.ids[row * a.k + i] = -1;
  }
  if (threadIdx.x == 0) {
    a.logprob[row] = 0.f;
    a.entropy[row] = 0.f;
    a.stats[row] = make_float2(0.f, -INFINITY);
  }
  return true;
}

// a row's results from its statistics (one thread)
template <int DT>
__device__ __forceinline__ void logp_row(const LogpArgs& a, int64_t row, const RowStat& r) {
  typedef typename Lg<DT>::T T;
  int64_t t = a.tokens[row];
  if (t < 0 || t >= a.V) {
    *a.bad = 1;
    t = t < 0 ? 0 : a.V - 1;
  }
  const bool none = r.s == 0.f;  // every logit is -inf
  const float ls = none ? -INFINITY : logf(r.s);
  const float z = Lg<DT>::one(reinterpret_cast<const T*>(a.z)[row * a.ld + t]);
  a.stats[row] = make_float2(r.m, ls);
  a.logprob[row] = none ? -INFINITY : (z - r.m) - ls;
  a.entropy[row] = none ? 0.f : ls - r.a / r.s;
}
__device__ __forceinline__ void logp_top(const LogpArgs& a, int64_t row, const RowStat& r, float ls, int rank,
                                         uint64_t key) {
  a.top[row * a.k + rank] = r.s == 0.f ? -INFINITY : (of_order((uint32_t)(key >> 32)) - r.m) - ls;
  a.ids[row * a.k + rank] = index_of(key);
}

// The k largest keys of the n elements at z (row indices from `first` on),
// unsorted, by every thread of a workgroup: the largest key that k keys reach,
// two bits a pass over the part.
template <int DT, int NT>
__device__ __noinline__ int logp_exact(const typename Lg<DT>::T* z, int first, int n, int k, uint64_t* cand,
                                       int* count) {
  constexpr int W = NT / 64;
  __shared__ int reach_s[3][W];
  uint64_t f = 0;
  for (int bit = 62; bit >= 0; bit -= 2) {
    int reach[3] = {0, 0, 0};
    for (int i = threadIdx.x; i < n; i += NT) {
      const uint64_t key = key_of(Lg<DT>::one(z[i]), first + i);
#pragma unroll
      for (int c = 0; c < 3; ++c) reach[c] += key >= (f | (uint64_t)(c + 1) << bit);
    }
#pragma unroll
    for (int c = 0; c < 3; ++c) {
      const int sum = (int)wave_sum((float)reach[c]);  // (below 2^24: exact)
      if ((threadIdx.x & 63) == 0) reach_s[c][threadIdx.x >> 6] = sum;
    }
    __syncthreads();
    int digit = 0;
    for (int c = 0; c < 3; ++c) {
      int total = 0;
      for (int w = 0; w < W; ++w) total += reach_s[c][w];
      digit += total >= k;
    }
    f |= (uint64_t)digit << bit;
    __syncthreads();
  }
  if (threadIdx.x == 0) *count = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += NT) {
    const uint64_t key = key_of(Lg<DT>::one(z[i]), first + i);
    if (key >= f) cand[atomicAdd(count, 1)] = key;  // (exactly k: all keys differ)
  }
  if (threadIdx.x < 16) cand[k + threadIdx.x] = 0;
  __syncthreads();
  return *count;
}

// The number of keys at `cand` that are larger than `key`, `count` of them with
// zeros behind up to a multiple of 16.
__device__ __forceinline__ int logp_rank(const uint64_t* cand, int count, uint64_t key) {
  int rank = 0;
  for (int j = 0; j < count; j += 16) {
    ulonglong2 c[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) c[u] = *reinterpret_cast<const ulonglong2*>(&cand[j + 2 * u]);
#pragma unroll
    for (int u = 0; u < 8; ++u) rank += (c[u].x > key) + (c[u].y > key);
  }
  return rank;
}

// One workgroup per part of a row, a whole row up to 512 * 16 vectors: eight
// loads in flight per thread, each logit read once.
//
// Top alternatives: every thread keeps the order (16 bits, rounded down) of
// each of its vectors' maxima.  Of 256 maxima, each of a thread or of a pair of
// them, the k-th largest is a lower bound of the row's k-th largest, and only
// about k + k^2 / 512 logits reach it: the few vectors with one are listed in LDS,
// read again an element per thread, and the candidates sorted by counting.  Where
// more reach it than the sort takes (equal logits, a row of few finite ones) or
// the row holds a NaN, the k-th key is found bit by bit: right, but 32 passes over
// the part ([2048, 50304] bf16, 20 alternatives: 48 us; of 10 allowed tokens, of equal
// logits or with a NaN in every row 3340).  HBM bounds it without alternatives
// ([4096, 50304] bf16 80 us alone, 5.2 TB/s); listing and sorting them, for which a
// workgroup has nothing else to do, adds to it (20: 92 us, 128: 108).
template <int DT, int NT, int TRIPS, bool TOP>
__global__ void __launch_bounds__(NT, 6) logp_fwd_kernel(LogpArgs a) {
  typedef typename Lg<DT>::T T;
  constexpr int E = Lg<DT>::E, NV = kLogpVecs;
  __shared__ float red[3 * NT / 64];
  __shared__ __attribute__((aligned(16))) uint64_t cand[TOP ? kLogpCand : 2];
  __shared__ __attribute__((aligned(16))) uint32_t maxima[TOP ? 256 : 4];
  __shared__ int hit[TOP ? kLogpHits : 1];
  __shared__ uint32_t floor_s;
  __shared__ int count_s, hits_s;

  const int64_t row = blockIdx.x / a.parts;
  const int part = blockIdx.x % a.parts;
  if (a.parts == 1 ? logp_ignored(a, row) : a.tokens[row] == a.ignore) return;
  const int first = part * a.part, n = min(a.V - first, a.part);
  const T* z = reinterpret_cast<const T*>(a.z) + row * a.ld + first;
  if constexpr (TOP) {
    for (int i = threadIdx.x; i < kLogpCand; i += NT) cand[i] = 0;
    if (threadIdx.x == 0) count_s = hits_s = 0;
  }

  RowStat r{kLowest, 0.f, 0.f};
  uint32_t tops[TRIPS * NV];  // orders of the vectors' maxima
  each_place<TRIPS * NV>([&](auto i) __attribute__((always_inline)) { tops[i] = 0; });
  each_place<TRIPS>([&](auto trip) __attribute__((always_inline)) {
    if (trip * NV * NT * E >= n) return;
    lg_u32x4 v[places_of(NV)];
    const int places = load_vecs<DT, NV, NT>(v, z, trip * NV * NT, n);
    float m = r.m;
    each_place<NV>([&](auto i) __attribute__((always_inline)) {
      if (i < places) {
        float x[E];
        unpack_again<DT>(v[i], x);
        float mx = x[0];
#pragma unroll
        for (int j = 1; j < E; ++j) mx = fmaxf(mx, x[j]);
        if constexpr (TOP) tops[trip * NV + i] = order_of(mx) >> 16;
        m = fmaxf(m, mx);
      }
    });
    r = trip == 0 ? RowStat{m, 0.f, 0.f} : at_max(r, m);
    each_place<NV>([&](auto i) __attribute__((always_inline)) {
      if (i < places) {
        float x[E];
        unpack_again<DT>(v[i], x);
#pragma unroll
        for (int j = 0; j < E; ++j) {
          const float d = x[j] - r.m, e = exp_f(d);
          r.s += e;
          r.a = __builtin_fmaf(e, fmaxf(d, kFarBelow), r.a);
        }
      }
    });
  });
  if constexpr (TOP) {  // (a thread of -inf alone counts as the lowest: a lower bound all the same)
    constexpr int P = NT / 256;  // threads that share a maximum
    const float pm = P == 1 ? r.m : fmaxf(r.m, __shfl_xor(r.m, 1, 64));
    if (threadIdx.x % P == 0) maxima[threadIdx.x / P] = order_of(pm) >> 16;
  }
  r = block_stat<NT>(r, red);
  if (threadIdx.x == 0) {
    if (a.parts == 1)
      logp_row<DT>(a, row, r);
    else
      a.part_stat[row * a.parts + part] = make_float4(r.m, r.s, r.a, 0.f);
  }
  if constexpr (TOP) {
    if (threadIdx.x < 64) {  // (block_stat's barrier lies behind the maxima)
      const uint4 k4 = *reinterpret_cast<const uint4*>(&maxima[threadIdx.x * 4]);
      uint32_t f = 0;
      for (int bit = 15; bit >= 0; --bit) {
        const uint32_t c = f | 1u << bit;
        const int above = __popcll(__ballot(k4.x >= c)) + __popcll(__ballot(k4.y >= c)) +
                          __popcll(__ballot(k4.z >= c)) + __popcll(__ballot(k4.w >= c));
        if (above >= a.k) f = c;
      }
      // up to the order of the lowest finite value: everything, -inf too
      if (threadIdx.x == 0) floor_s = f <= (order_of(kLowest) >> 16) ? 0 : f;
    }
    __syncthreads();
    const uint32_t floor_o = floor_s;
    uint32_t hits = 0;
    each_place<TRIPS * NV>([&](auto i) __attribute__((always_inline)) {
      hits |= tops[i] >= floor_o && (i * NT + (int)threadIdx.x) * E < n ? 1u << i : 0u;
    });
    while (hits) {
      const int slot = atomicAdd(&hits_s, 1);
      if (slot < kLogpHits) hit[slot] = (__ffs(hits) - 1) * NT + threadIdx.x;
      hits &= hits - 1;
    }
    __syncthreads();
    // one element per thread: all loads under way at once
    const int elems = min(hits_s, kLogpHits) * E;
    for (int e = threadIdx.x; e < elems; e += NT) {
      const int at = hit[e / E] * E + e % E;
      if (at >= n) continue;
      const uint64_t key = key_of(Lg<DT>::one(z[at]), first + at);
      if ((uint32_t)(key >> 48) < floor_o) continue;
      const int slot = atomicAdd(&count_s, 1);
      if (slot < kLogpCand) cand[slot] = key;
    }
    __syncthreads();
    int count = count_s;
    if (hits_s > kLogpHits || count > kLogpCand || r.s != r.s)
      count = logp_exact<DT, NT>(z, first, n, a.k, cand, &count_s);
    const float ls = logf(r.s);
    for (int i = threadIdx.x; i < count; i += NT) {
      const uint64_t key = cand[i];
      const int rank = logp_rank(cand, count, key);
      if (rank >= a.k) continue;
      if (a.parts == 1)
        logp_top(a, row, r, ls, rank, key);
      else
        a.part_key[(row * a.parts + part) * a.k + rank] = key;
    }
  }
}

// Joins the parts of a row: their statistics, and the k largest of their sorted
// keys.  k keys are at least the n-th largest of the parts' j-th keys where n * j
// >= k; the largest of these bounds over j = k, k/2, k/4, .. is taken.  Fewer than
// n parts have more than j keys above it, for every j, which leaves 1281 keys at
// the most (k = 128, 512 parts) and little more than k as a rule: they are listed
// and sorted by counting.  A search for every key in every part took, for 512 rows
// of 4 parts of 128 keys, 12.9 us where this takes 8.6, and 2017 against 47 for 64
// rows of 64 parts.  Up to a key a thread, all are listed (4 parts of 5: 5.9 us
// with the bounds, 4.3 without; of 128: 18.3 us without).
constexpr int kLogpParts = 512;  // most parts of a row
constexpr int kLogpJoined = 1296;  // (a multiple of 16)
template <int DT>
__global__ void __launch_bounds__(256) logp_join_kernel(LogpArgs a) {
  __shared__ __attribute__((aligned(16))) uint64_t cand[kLogpJoined];
  __shared__ uint64_t part_s[kLogpParts];
  __shared__ float red[3 * 256 / 64];
  __shared__ uint64_t bound_s;
  __shared__ int count_s;
  const int64_t row = blockIdx.x;
  if (logp_ignored(a, row)) return;
  const float4* ps = a.part_stat + row * a.parts;
  RowStat r{kLowest, 0.f, 0.f};
  for (int i = threadIdx.x; i < a.parts; i += 256) {
    const float4 p = ps[i];
    const float m = fmaxf(r.m, p.x);
    const RowStat x = at_max(RowStat{p.x, p.y, p.z}, m);
    r = at_max(r, m);
    r.s += x.s;
    r.a += x.a;
  }
  r = block_stat<256>(r, red);
  if (threadIdx.x == 0) logp_row<DT>(a, row, r);
  if (a.k == 0) return;
  const float ls = logf(r.s);
  const uint64_t* keys = a.part_key + row * a.parts * a.k;
  if (threadIdx.x == 0) {
    bound_s = 0;
    count_s = 0;
  }
  for (int i = threadIdx.x; i < kLogpJoined; i += 256) cand[i] = 0;
  for (int j = a.parts * a.k > 256 ? a.k : 0; j > 0; j = (j + 1) / 2) {
    const int need = (a.k + j - 1) / j;
    if (need > a.parts) break;
    for (int q = threadIdx.x; q < a.parts; q += 256) part_s[q] = keys[q * a.k + j - 1];
    __syncthreads();
    for (int q = threadIdx.x; q < a.parts; q += 256) {
      const uint64_t key = part_s[q];
      int rank = 0;
      for (int i = 0; i < a.parts; ++i) rank += part_s[i] > key;
      if (rank == need - 1 && key > bound_s) bound_s = key;  // (one thread: all keys differ)
    }
    __syncthreads();
    if (j == 1) break;
  }
  __syncthreads();
  const uint64_t bound = bound_s;
  for (int i = threadIdx.x; i < a.parts * a.k; i += 256) {
    const uint64_t key = keys[i];
    if (key < bound) continue;
    cand[min(atomicAdd(&count_s, 1), kLogpJoined - 1)] = key;
  }
  __syncthreads();
  const int count = min(count_s, kLogpJoined);
  for (int i = threadIdx.x; i < count; i += 256) {
    const int rank = logp_rank(cand, count, cand[i]);
    if (rank < a.k) logp_top(a, row, r, ls, rank, cand[i]);
  }
}

constexpr int kRowThreads = 256;
constexpr int kRowVecs = 4;  // vectors of a backward workgroup's thread

// zeros in a backward workgroup's vectors
template <int DT, bool STREAM>
__device__ __forceinline__ void zero_vecs(typename Lg<DT>::T* dz, int v0, int n) {
  float x[Lg<DT>::E] = {};
#pragma unroll
  for (int u = 0; u < kRowVecs; ++u) store_vec<DT, STREAM>(dz, v0 + u * kRowThreads + threadIdx.x, n, x);
}

// A workgroup per 1024 vectors of a row: many short ones keep HBM busier than
// one that walks the row (145 against 170 us for [4096, 50304] bf16).  A row
// without upstream gradient (and one without a finite logit) gets zeros and is
// not read.  HBM bounds it ([4096, 50304] bf16 141 us, 5.8 TB/s read and written).
template <int DT, bool STREAM>
__global__ void __launch_bounds__(kRowThreads) logp_bwd_kernel(const void* zv, int64_t ld, int V,
                                                               const int64_t* __restrict__ tokens, int64_t ignore,
                                                               const float2* __restrict__ stats,
                                                               const float* __restrict__ entropy,
                                                               const float* __restrict__ dlogprob,
                                                               const float* __restrict__ dentropy, void* dzv,
                                                               int64_t ldd, int chunks) {
  typedef typename Lg<DT>::T T;
  constexpr int E = Lg<DT>::E;
  const int64_t row = blockIdx.x / chunks;
  const int v0 = blockIdx.x % chunks * (kRowThreads * kRowVecs);
  const T* z = reinterpret_cast<const T*>(zv) + row * ld;
  T* dz = reinterpret_cast<T*>(dzv) + row * ldd;
  const int64_t token = tokens[row];
  const float2 st = stats[row];
  const bool out = token == ignore || st.y == -INFINITY;
  const int t = token < 0 ? 0 : (token >= V ? V - 1 : (int)token);
  const float g = out || !dlogprob ? 0.f : dlogprob[row], h = out || !dentropy ? 0.f : dentropy[row];
  if (g == 0.f && h == 0.f) {
    zero_vecs<DT, STREAM>(dz, v0, V);
    return;
  }
  const float H = entropy[row];
  lg_u32x4 v[places_of(kRowVecs)];
  load_vecs<DT, kRowVecs, kRowThreads>(v, z, v0, V);
  each_place<kRowVecs>([&](auto u) __attribute__((always_inline)) {
    const int i = v0 + u * kRowThreads + threadIdx.x;
    float x[E];
    Lg<DT>::unpack(v[u], x);
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const float lp = (x[j] - st.x) - st.y, p = exp_f(lp);
      const float w = g + h * (fmaxf(lp, kFarBelow) + H);
      x[j] = (i * E + j == t ? g : 0.f) - p * w;
    }
    store_vec<DT, STREAM>(dz, i, V, x);
  });
}

// ----------------------------------------------------------------- distillation --
constexpr int kDistillTop = 256;  // most teacher entries of a row
constexpr int kDistillThreads = 512;
constexpr int kDistillVecs = 8;

struct DistillArgs {
  const void* z;
  int64_t ld;
  int V;
  const int64_t* ids;  // [rows, k]; negative: no entry
  const void* teacher; // [rows, k] logits
  int teacher_dtype, k;
  float tau;
  float* loss;
  // max, log of the sum of exp((z - max) / tau); the teacher's max, and the sum
  // of exp((u - max) / tau) over its entries (0: there are none)
  float4* stats;
  int* bad;
  const float* dloss;
  void* dz;
  int64_t ldd;
  int chunks;  // backward: workgroups per row
  int parts, part;    // forward: workgroups per row, elements of each
  float2* part_stat;  // [rows, parts]: max, sum of exp((z - max) / tau)
};

// entry i of a row's teacher: its id, -1 where there is none
__device__ __forceinline__ int teacher_id(const DistillArgs& a, int64_t row, int i) {
  if (i >= a.k) return -1;
  const int64_t id = a.ids[row * a.k + i];
  if (id >= a.V) *a.bad = 1;
  return id >= 0 && id < a.V ? (int)id : -1;
}
__device__ __forceinline__ float teacher_logit(const DistillArgs& a, int64_t row, int i) {
  return load_elem(a.teacher, row * a.k + i, a.teacher_dtype);
}

// A lane's entries of a row: entry lane + 64 e of its teacher, for one wave (id),
// and the teacher's logits and the student's for them (u, zu).
constexpr int kDistillLane = kDistillTop / 64;
struct DistillEntries {
  int id[kDistillLane];
  float u[kDistillLane], zu[kDistillLane];
};
// whether the row has entries; a row without gets its results here
__device__ __forceinline__ bool distill_ids(const DistillArgs& a, int64_t row, int lane, DistillEntries& t) {
  bool any = false;
#pragma unroll
  for (int e = 0; e < kDistillLane; ++e) {
    t.id[e] = teacher_id(a, row, lane + 64 * e);
    any |= t.id[e] >= 0;
  }
  if (__any(any)) return true;
  if (threadIdx.x == 0) {  // (every part of it stores the same)
    a.loss[row] = 0.f;
    a.stats[row] = make_float4(0.f, -INFINITY, 0.f, 0.f);
  }
  return false;
}
template <int DT>
__device__ __forceinline__ void distill_logits(const DistillArgs& a, int64_t row, int lane, DistillEntries& t) {
  const typename Lg<DT>::T* z = reinterpret_cast<const typename Lg<DT>::T*>(a.z) + row * a.ld;
#pragma unroll
  for (int e = 0; e < kDistillLane; ++e) {
    t.u[e] = t.id[e] >= 0 ? teacher_logit(a, row, lane + 64 * e) : -INFINITY;
    t.zu[e] = t.id[e] >= 0 ? Lg<DT>::one(z[t.id[e]]) : 0.f;
  }
}
// a row's results from its maximum M and sum S of exp((z - M) / tau) (one wave)
__device__ __forceinline__ void distill_row(const DistillArgs& a, int64_t row, int lane, const DistillEntries& t, float M,
                                            float S) {
  const bool none = S == 0.f;  // no finite logit: no probability for any entry
  const float ls = none ? -INFINITY : logf(S);
  float um = kLowest, total = 0.f, loss = 0.f;
#pragma unroll
  for (int e = 0; e < kDistillLane; ++e) um = fmaxf(um, t.u[e]);
  um = wave_max(um);
  // (a teacher logit of NaN or +inf makes every q NaN, as the softmax does)
#pragma unroll
  for (int e = 0; e < kDistillLane; ++e) total += t.id[e] >= 0 ? exp_f((t.u[e] - um) / a.tau) : 0.f;
  total = wave_sum(total);
#pragma unroll
  for (int e = 0; e < kDistillLane; ++e) {
    const float q = t.id[e] >= 0 ? exp_f((t.u[e] - um) / a.tau) / total : 0.f;
    const float lp = none ? -INFINITY : (t.zu[e] - M) / a.tau - ls;
    if (!(q == 0.f)) loss += q * (logf(q) - lp);
  }
  loss = wave_sum(loss);
  if (lane == 0) {
    a.loss[row] = total == 0.f ? 0.f : loss * a.tau * a.tau;
    a.stats[row] = make_float4(M, ls, um, total);
  }
}

// One workgroup per row, or where rows are few and long per part of one: its
// statistics at the temperature, each thread over its own vectors, eight in
// flight.  Every wave looks the ids over (a row without entries is not read); of a
// whole row the first one weighs the entries, four a lane, while the others read,
// and joins it all behind the one barrier.  HBM bounds it ([4096, 50304] bf16, 64
// entries: 75 us alone, 5.5 TB/s; 90 behind a backward pass, whose lines are written
// back meanwhile), and for few rows the time that one workgroup takes to read its
// share.
template <int DT, int NT, bool PARTS>
__global__ void __launch_bounds__(NT) distill_fwd_kernel(DistillArgs a) {
  typedef typename Lg<DT>::T T;
  constexpr int E = Lg<DT>::E;
  __shared__ float red[2 * NT / 64];
  const int64_t row = PARTS ? blockIdx.x / a.parts : blockIdx.x;
  const int first = PARTS ? blockIdx.x % a.parts * a.part : 0, n = PARTS ? min(a.V - first, a.part) : a.V;
  const int lane = threadIdx.x & 63;
  const T* z = reinterpret_cast<const T*>(a.z) + row * a.ld + first;
  DistillEntries t;
  if (!distill_ids(a, row, lane, t)) return;
  if constexpr (!PARTS)
    if (threadIdx.x < 64) distill_logits<DT>(a, row, lane, t);
  const float c = kLog2e / a.tau;
  float m = kLowest, s = 0.f;
  const int nv = (n + E - 1) / E;
  for (int v0 = 0; v0 < nv; v0 += NT * kDistillVecs) {
    lg_u32x4 v[places_of(kDistillVecs)];
    const int places = load_vecs<DT, kDistillVecs, NT>(v, z, v0, n);
    float mx = m;
    each_place<kDistillVecs>([&](auto u) __attribute__((always_inline)) {
      if (u < places) {
        float x[E];
        unpack_again<DT>(v[u], x);
#pragma unroll
        for (int j = 0; j < E; ++j) mx = fmaxf(mx, x[j]);
      }
    });
    s *= __builtin_amdgcn_exp2f((m - mx) * c);
    m = mx;
    float trip = 0.f;  // closed by itself: a sum of V / 512 terms one after the other would lose digits
    each_place<kDistillVecs>([&](auto u) __attribute__((always_inline)) {
      if (u < places) {
        float x[E];
        unpack_again<DT>(v[u], x);
#pragma unroll
        for (int j = 0; j < E; ++j) trip += __builtin_amdgcn_exp2f((x[j] - m) * c);
      }
    });
    s += trip;
  }
  const float wm = wave_max(m);
  const float ws = wave_sum(s * __builtin_amdgcn_exp2f((m - wm) * c));
  if (lane == 0) {
    red[threadIdx.x >> 6] = wm;
    red[NT / 64 + (threadIdx.x >> 6)] = ws;
  }
  __syncthreads();
  if (threadIdx.x >= 64) return;
  float M = red[0], S = 0.f;
#pragma unroll
  for (int w = 1; w < NT / 64; ++w) M = fmaxf(M, red[w]);
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) S += red[NT / 64 + w] * __builtin_amdgcn_exp2f((red[w] - M) * c);
  if constexpr (PARTS) {
    if (lane == 0) a.part_stat[blockIdx.x] = make_float2(M, S);
  } else {
    distill_row(a, row, lane, t, M, S);
  }
}

// joins the parts of a row, one wave
template <int DT>
__global__ void __launch_bounds__(64) distill_join_kernel(DistillArgs a) {
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x;
  DistillEntries t;
  if (!distill_ids(a, row, lane, t)) return;
  distill_logits<DT>(a, row, lane, t);
  const float c = kLog2e / a.tau;
  const float2* ps = a.part_stat + row * a.parts;
  float m = kLowest, s = 0.f;
  for (int i = lane; i < a.parts; i += 64) {
    const float2 p = ps[i];
    const float mx = fmaxf(m, p.x);
    s = s * __builtin_amdgcn_exp2f((m - mx) * c) + p.y * __builtin_amdgcn_exp2f((p.x - mx) * c);
    m = mx;
  }
  const float M = wave_max(m);
  distill_row(a, row, lane, t, M, wave_sum(s * __builtin_amdgcn_exp2f((m - M) * c)));
}

// A workgroup per 1024 vectors of a row: dz = g tau p, then the entries
// among them once more with their q (an id that appears more than once by its
// first entry, with the sum).  HBM bounds it ([4096, 50304] bf16, 64 entries: 149
// us, 5.5 TB/s read and written).
template <int DT, bool STREAM>
__global__ void __launch_bounds__(kRowThreads) distill_bwd_kernel(DistillArgs a) {
  typedef typename Lg<DT>::T T;
  constexpr int E = Lg<DT>::E;
  __shared__ float q_s[kDistillTop];
  __shared__ __attribute__((aligned(16))) int id_s[kDistillTop];
  static_assert(kRowThreads == kDistillTop, "a thread per entry");
  const int64_t row = blockIdx.x / a.chunks;
  const int v0 = blockIdx.x % a.chunks * (kRowThreads * kRowVecs);
  const T* z = reinterpret_cast<const T*>(a.z) + row * a.ld;
  T* dz = reinterpret_cast<T*>(a.dz) + row * a.ldd;
  const float4 st = a.stats[row];
  const float gt = st.y == -INFINITY || st.w == 0.f ? 0.f : a.dloss[row] * a.tau;
  if (gt == 0.f) {  // (also a row without teacher entries or finite logits)
    zero_vecs<DT, STREAM>(dz, v0, a.V);
    return;
  }
  // the thread's entry, if it falls among these vectors; its loads go first,
  // so that they wait for no others
  const int mine = threadIdx.x;
  const float u = mine < a.k ? teacher_logit(a, row, mine) : 0.f;
  int id = teacher_id(a, row, mine);
  const bool here = id >= v0 * E && id < (v0 + kRowThreads * kRowVecs) * E;
  const float zu = here ? Lg<DT>::one(z[id]) : 0.f;
  lg_u32x4 v[places_of(kRowVecs)];
  load_vecs<DT, kRowVecs, kRowThreads>(v, z, v0, a.V);
  const float inv = 1.f / a.tau;
  const float q = id >= 0 ? exp_f((u - st.z) / a.tau) / st.w : 0.f;
  q_s[mine] = q;
  id_s[mine] = id;
  auto prob = [&](float x) __attribute__((always_inline)) { return exp_f((x - st.x) * inv - st.y); };
  each_place<kRowVecs>([&](auto u) __attribute__((always_inline)) {
    float x[E];
    Lg<DT>::unpack(v[u], x);
#pragma unroll
    for (int j = 0; j < E; ++j) x[j] = gt * prob(x[j]);
    store_vec<DT, STREAM>(dz, v0 + u * kRowThreads + threadIdx.x, a.V, x);
  });
  // the stores below come after those of the same places above, other waves' too
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
  __syncthreads();
  if (here) {
    int before = 0, all = 0;  // entries with this id
    for (int i = 0; i < a.k; i += 16) {  // (-1 behind the last)
      int4 x[4];
#pragma unroll
      for (int w = 0; w < 4; ++w) x[w] = *reinterpret_cast<const int4*>(&id_s[i + 4 * w]);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int y[4] = {x[w].x, x[w].y, x[w].z, x[w].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          all += y[e] == id;
          before += y[e] == id && i + 4 * w + e < mine;
        }
      }
    }
    float sum = q;
    if (all > 1) {
      sum = 0.f;
      for (int i = 0; i < a.k; ++i) sum += id_s[i] == id ? q_s[i] : 0.f;
    }
    if (before == 0) dz[id] = Lg<DT>::round(gt * (prob(zu) - sum));
  }
}

}  // namespace eth

using namespace eth;

// (far below what would leave a part of a row empty)
constexpr int64_t kMostVocab = 1LL << 24;
static_assert(kMostVocab * 4 <= (int64_t)kLogpParts * kLogpThreads * kLogpVecs * kLogpTrips * 16, "a row's parts");
static bool logits_shape(int64_t rows, int64_t V, int64_t ld) {
  return rows > 0 && V > 0 && V <= kMostVocab && ld >= V;
}
// Rows of `per` workgroups of at most `threads` threads that one launch takes:
// a grid has fewer than 2^32 threads, and more rows go in several launches.
static int64_t launch_rows(int64_t per, int threads) { return ((1LL << 32) - 1) / (per * threads); }
template <class T>
static void advance(T*& p, int64_t elements) {
  if (p) p += elements;
}
static void advance(const void*& p, int64_t elements, int dtype) {
  p = (const char*)p + elements * dtype_size(dtype);
}
static int64_t logp_parts(int64_t V, int dtype) {
  const int64_t most = (int64_t)kLogpThreads * kLogpVecs * kLogpTrips * (16 / dtype_size(dtype));
  return (V + most - 1) / most;
}

extern "C" int64_t eth_token_logprobs_workspace(int64_t rows, int64_t vocab, int top_k, int dtype) {
  if (!valid_dtype(dtype) || rows <= 0 || vocab <= 0 || vocab > kMostVocab || top_k < 0) return 0;
  const int64_t parts = logp_parts(vocab, dtype);
  return parts == 1 ? 0 : rows * parts * (int64_t)(sizeof(float4) + top_k * sizeof(uint64_t));
}

template <int DT, int NT, int TRIPS>
static void launch_logp_part(const LogpArgs& a, int grid, hipStream_t s) {
  if (a.k > 0)
    logp_fwd_kernel<DT, NT, TRIPS, true><<<grid, NT, 0, s>>>(a);
  else
    logp_fwd_kernel<DT, NT, TRIPS, false><<<grid, NT, 0, s>>>(a);
}
// Short rows in small workgroups, more of which share a compute unit: one
// closes its row while others read ([8192, 8000] bf16 with 512 -> 256 threads:
// 35 -> 27 us, with 20 alternatives 72 -> 43; [4096, 32000], two trips of 256
// against one of 512: 49.8 against 47.3 us, with 20 alternatives 56.0 against 61.7).
template <int DT>
static void launch_logp(const LogpArgs& a, int64_t rows, hipStream_t s) {
  const int grid = (int)(rows * a.parts);
  const int vecs = a.part / Lg<DT>::E;
  if (vecs <= 256 * kLogpVecs)
    launch_logp_part<DT, 256, 1>(a, grid, s);
  else if (vecs <= 512 * kLogpVecs && a.k > 0)
    logp_fwd_kernel<DT, 256, 2, true><<<grid, 256, 0, s>>>(a);
  else if (vecs <= 512 * kLogpVecs)
    logp_fwd_kernel<DT, 512, 1, false><<<grid, 512, 0, s>>>(a);
  else
    launch_logp_part<DT, kLogpThreads, kLogpTrips>(a, grid, s);
  if (a.parts > 1) logp_join_kernel<DT><<<(int)rows, 256, 0, s>>>(a);
}

extern "C" int eth_token_logprobs_fwd(const void* logits, int64_t ld, const int64_t* tokens, int64_t ignore_index,
                                      float* logprob, float* entropy, float* stats, float* top_logprobs,
                                      int64_t* top_ids, int top_k, void* workspace, int64_t rows, int64_t vocab,
                                      int* bad_index, int dtype, void* stream) {
  ETH_CHECK_ARG(valid_dtype(dtype), "eth_token_logprobs_fwd: dtype must be bf16/fp16/fp32");
  ETH_CHECK_ARG(logits_shape(rows, vocab, ld), "eth_token_logprobs_fwd: bad shape");
  ETH_CHECK_ARG(top_k >= 0 && top_k <= kLogpTop && top_k <= vocab,
                "eth_token_logprobs_fwd: top_k must be in [0, %d] and within the vocabulary (got %d)", kLogpTop, top_k);
  ETH_CHECK_ARG(logits && tokens && logprob && entropy && stats && bad_index && (top_k == 0 || (top_logprobs && top_ids)),
                "eth_token_logprobs_fwd: null pointer");
  LogpArgs a{};
  a.parts = (int)logp_parts(vocab, dtype);
  ETH_CHECK_ARG(a.parts == 1 || (workspace && ((uintptr_t)workspace & 15) == 0),
                "eth_token_logprobs_fwd: this vocabulary needs a 16-byte aligned workspace");
  ETH_CHECK_ARG(rows * a.parts < (1LL << 31), "eth_token_logprobs_fwd: too many rows (%lld)", (long long)rows);
  ETH_CHECK_ARG(((uintptr_t)logits % dtype_size(dtype)) == 0 && ((uintptr_t)stats & 7) == 0,
                "eth_token_logprobs_fwd: misaligned pointer");
  a.z = logits;
  a.ld = ld;
  a.V = (int)vocab;
  a.tokens = tokens;
  a.ignore = ignore_index;
  a.logprob = logprob;
  a.entropy = entropy;
  a.stats = (float2*)stats;
  a.top = top_logprobs;
  a.ids = top_ids;
  a.k = top_k;
  a.bad = bad_index;
  const int64_t E = 16 / dtype_size(dtype), vecs = (vocab + E - 1) / E;
  a.part = (int)((vecs + a.parts - 1) / a.parts * E);
  a.part_stat = (float4*)workspace;
  a.part_key = (uint64_t*)(a.part_stat + rows * a.parts);
  hipStream_t s = (hipStream_t)stream;
  const int64_t most = launch_rows(a.parts, kLogpThreads);
  for (int64_t r = 0; r < rows; r += most) {
    const int64_t n = rows - r < most ? rows - r : most;
    if (dtype == ETH_BF16)
      launch_logp<ETH_BF16>(a, n, s);
    else if (dtype == ETH_F16)
      launch_logp<ETH_F16>(a, n, s);
    else
      launch_logp<ETH_F32>(a, n, s);
    ETH_CHECK_LAUNCH("eth_token_logprobs_fwd");
    advance(a.z, n * ld, dtype);
    advance(a.tokens, n);
    advance(a.logprob, n);
    advance(a.entropy, n);
    advance(a.stats, n);
    advance(a.top, n * top_k);
    advance(a.ids, n * top_k);
    advance(a.part_stat, n * a.parts);
    advance(a.part_key, n * a.parts * top_k);
  }
  return ETH_OK;
}

static int row_chunks(int64_t V, int dtype) {
  const int64_t per = (int64_t)kRowThreads * kRowVecs * (16 / dtype_size(dtype));
  return (int)((V + per - 1) / per);
}

extern "C" int eth_token_logprobs_bwd(const void* logits, int64_t ld, const int64_t* tokens, int64_t ignore_index,
                                      const float* stats, const float* entropy, const float* dlogprob,
                                      const float* dentropy, void* dlogits, int64_t ldd, int64_t rows, int64_t vocab,
                                      int dtype, void* stream) {
  ETH_CHECK_ARG(valid_dtype(dtype), "eth_token_logprobs_bwd: dtype must be bf16/fp16/fp32");
  ETH_CHECK_ARG(logits_shape(rows, vocab, ld) && ldd >= vocab, "eth_token_logprobs_bwd: bad shape");
  ETH_CHECK_ARG(logits && tokens && stats && entropy && (dlogprob || dentropy) && dlogits,
                "eth_token_logprobs_bwd: null pointer");
  ETH_CHECK_ARG(((uintptr_t)logits % dtype_size(dtype)) == 0 && ((uintptr_t)dlogits % dtype_size(dtype)) == 0 &&
                    ((uintptr_t)stats & 7) == 0,
                "eth_token_logprobs_bwd: misaligned pointer");
  const int chunks = row_chunks(vocab, dtype);
  ETH_CHECK_ARG(rows * chunks < (1LL << 31), "eth_token_logprobs_bwd: too many rows (%lld)", (long long)rows);
  hipStream_t s = (hipStream_t)stream;
  const bool stream_out = rows * vocab * dtype_size(dtype) > kStreamBytes;
  const float2* row_stats = (const float2*)stats;
  const void* dz = dlogits;
  const int64_t most = launch_rows(chunks, kRowThreads);
  for (int64_t r = 0; r < rows; r += most) {
    const int64_t n = rows - r < most ? rows - r : most;
    const int grid = (int)(n * chunks);
#define ETH_LOGP_BWD(DT)                                                                              \
  (stream_out ? logp_bwd_kernel<DT, true> : logp_bwd_kernel<DT, false>)<<<grid, kRowThreads, 0, s>>>( \
      logits, ld, (int)vocab, tokens, ignore_index, row_stats, entropy, dlogprob, dentropy,           \
      const_cast<void*>(dz), ldd, chunks)
    if (dtype == ETH_BF16)
      ETH_LOGP_BWD(ETH_BF16);
    else if (dtype == ETH_F16)
      ETH_LOGP_BWD(ETH_F16);
    else
      ETH_LOGP_BWD(ETH_F32);
#undef ETH_LOGP_BWD
    ETH_CHECK_LAUNCH("eth_token_logprobs_bwd");
    advance(logits, n * ld, dtype);
    advance(dz, n * ldd, dtype);
    advance(tokens, n);
    advance(row_stats, n);
    advance(entropy, n);
    advance(dlogprob, n);
    advance(dentropy, n);
  }
  return ETH_OK;
}

static int distill_check(const char* who, const void* logits, int64_t ld, const int64_t* ids, const void* teacher,
                         int teacher_dtype, int k, float tau, const void* stats, int64_t rows, int64_t vocab,
                         const int* bad, int dtype) {
  ETH_CHECK_ARG(valid_dtype(dtype) && valid_dtype(teacher_dtype), "%s: dtypes must be bf16/fp16/fp32", who);
  ETH_CHECK_ARG(logits_shape(rows, vocab, ld) && rows < (1LL << 31), "%s: bad shape", who);
  ETH_CHECK_ARG(k >= 1 && k <= kDistillTop, "%s: 1 to %d teacher entries a row (got %d)", who, kDistillTop, k);
  ETH_CHECK_ARG(tau >= 0x1p-20f && tau <= 0x1p20f, "%s: temperature must be positive and finite", who);
  ETH_CHECK_ARG(logits && ids && teacher && stats && bad, "%s: null pointer", who);
  ETH_CHECK_ARG(((uintptr_t)logits % dtype_size(dtype)) == 0 && ((uintptr_t)teacher % dtype_size(teacher_dtype)) == 0 &&
                    ((uintptr_t)stats & 15) == 0,
                "%s: misaligned pointer", who);
  return ETH_OK;
}
static DistillArgs distill_args(const void* logits, int64_t ld, const int64_t* ids, const void* teacher,
                                int teacher_dtype, int k, float tau, const float* stats, int64_t vocab, int* bad) {
  DistillArgs a{};
  a.z = logits;
  a.ld = ld;
  a.V = (int)vocab;
  a.ids = ids;
  a.teacher = teacher;
  a.teacher_dtype = teacher_dtype;
  a.k = k;
  a.tau = tau;
  a.stats = (float4*)stats;
  a.bad = bad;
  return a;
}

// Parts that a row's forward is cut into: rows of four trips of a workgroup and
// more, into four parts and more, up to the two workgroups a compute unit that many
// rows fill by themselves ([4, 262144] fp16 20.4 us in one part each, 5.3 + 3.2 in
// eight with the join; [64, 262144] bf16 21.9, 7.2 + 4.0; [1, 2^24] fp32 1261, 13.4 +
// 5.0; [200, 262144] in two 24.0 + 4.0, which is no gain).
static int64_t distill_parts(int64_t rows, int64_t V, int dtype) {
  const int64_t trip = (int64_t)kDistillThreads * kDistillVecs * (16 / dtype_size(dtype));
  const int64_t trips = (V + trip - 1) / trip, most = 512 / rows;
  return trips < 4 || most < 4 ? 1 : trips < most ? trips : most;
}
extern "C" int64_t eth_topk_distill_workspace(int64_t rows, int64_t vocab, int dtype) {
  if (!valid_dtype(dtype) || rows <= 0 || vocab <= 0 || vocab > kMostVocab) return 0;
  const int64_t parts = distill_parts(rows, vocab, dtype);
  return parts == 1 ? 0 : rows * parts * (int64_t)sizeof(float2);
}

// the rows behind the first n
static void distill_advance(DistillArgs& a, int64_t n, int dtype) {
  advance(a.z, n * a.ld, dtype);
  const void* dz = a.dz;
  if (dz) advance(dz, n * a.ldd, dtype);
  a.dz = const_cast<void*>(dz);
  advance(a.ids, n * a.k);
  advance(a.teacher, n * a.k, a.teacher_dtype);
  advance(a.loss, n);
  advance(a.stats, n);
  advance(a.dloss, n);
  advance(a.part_stat, n * a.parts);
}

// (256 threads for short rows as above: [8192, 8000] bf16 40 -> 27 us; [4096,
// 32000] 46.4 us with 512, 48.9 with 256)
template <int DT>
static void launch_distill_fwd(DistillArgs a, int rows, hipStream_t s) {
  if (a.parts > 1) {
    distill_fwd_kernel<DT, kDistillThreads, true><<<rows * a.parts, kDistillThreads, 0, s>>>(a);
    distill_join_kernel<DT><<<rows, 64, 0, s>>>(a);
  } else if (a.V <= 256 * kDistillVecs * Lg<DT>::E) {
    distill_fwd_kernel<DT, 256, false><<<rows, 256, 0, s>>>(a);
  } else {
    distill_fwd_kernel<DT, kDistillThreads, false><<<rows, kDistillThreads, 0, s>>>(a);
  }
}

extern "C" int eth_topk_distill_fwd(const void* logits, int64_t ld, const int64_t* teacher_ids, const void* teacher,
                                    int teacher_dtype, int k, float temperature, float* loss, float* stats,
                                    void* workspace, int64_t rows, int64_t vocab, int* bad_index, int dtype,
                                    void* stream) {
  if (int rc = distill_check("eth_topk_distill_fwd", logits, ld, teacher_ids, teacher, teacher_dtype, k, temperature,
                             stats, rows, vocab, bad_index, dtype))
    return rc;
  ETH_CHECK_ARG(loss, "eth_topk_distill_fwd: null pointer");
  DistillArgs a = distill_args(logits, ld, teacher_ids, teacher, teacher_dtype, k, temperature, stats, vocab,
                               bad_index);
  a.loss = loss;
  a.parts = (int)distill_parts(rows, vocab, dtype);
  ETH_CHECK_ARG(a.parts == 1 || (workspace && ((uintptr_t)workspace & 7) == 0),
                "eth_topk_distill_fwd: so few rows of this vocabulary need an 8-byte aligned workspace");
  const int64_t E = 16 / dtype_size(dtype), vecs = (vocab + E - 1) / E;
  a.part = (int)((vecs + a.parts - 1) / a.parts * E);
  a.part_stat = (float2*)workspace;
  hipStream_t s = (hipStream_t)stream;
  const int64_t most = launch_rows(a.parts, kDistillThreads);
  for (int64_t r = 0; r < rows; r += most) {
    const int64_t n = rows - r < most ? rows - r : most;
    if (dtype == ETH_BF16)
      launch_distill_fwd<ETH_BF16>(a, (int)n, s);
    else if (dtype == ETH_F16)
      launch_distill_fwd<ETH_F16>(a, (int)n, s);
    else
      launch_distill_fwd<ETH_F32>(a, (int)n, s);
    ETH_CHECK_LAUNCH("eth_topk_distill_fwd");
    distill_advance(a, n, dtype);
  }
  return ETH_OK;
}

extern "C" int eth_topk_distill_bwd(const void* logits, int64_t ld, const int64_t* teacher_ids, const void* teacher,
                                    int teacher_dtype, int k, float temperature, const float* stats,
                                    const float* dloss, void* dlogits, int64_t ldd, int64_t rows, int64_t vocab,
                                    int* bad_index, int dtype, void* stream) {
  if (int rc = distill_check("eth_topk_distill_bwd", logits, ld, teacher_ids, teacher, teacher_dtype, k, temperature,
                             stats, rows, vocab, bad_index, dtype))
    return rc;
  ETH_CHECK_ARG(dloss && dlogits && ((uintptr_t)dlogits % dtype_size(dtype)) == 0 && ldd >= vocab,
                "eth_topk_distill_bwd: bad gradient buffers");
  DistillArgs a = distill_args(logits, ld, teacher_ids, teacher, teacher_dtype, k, temperature, stats, vocab,
                               bad_index);
  a.dloss = dloss;
  a.dz = dlogits;
  a.ldd = ldd;
  a.chunks = row_chunks(vocab, dtype);
  ETH_CHECK_ARG(rows * a.chunks < (1LL << 31), "eth_topk_distill_bwd: too many rows (%lld)", (long long)rows);
  hipStream_t s = (hipStream_t)stream;
  const bool stream_out = rows * vocab * dtype_size(dtype) > kStreamBytes;
  const int64_t most = launch_rows(a.chunks, kRowThreads);
  for (int64_t r = 0; r < rows; r += most) {
    const int64_t n = rows - r < most ? rows - r : most;
    const int grid = (int)(n * a.chunks);
#define ETH_DISTILL_BWD(DT) \
  (stream_out ? distill_bwd_kernel<DT, true> : distill_bwd_kernel<DT, false>)<<<grid, kRowThreads, 0, s>>>(a)
    if (dtype == ETH_BF16)
      ETH_DISTILL_BWD(ETH_BF16);
    else if (dtype == ETH_F16)
      ETH_DISTILL_BWD(ETH_F16);
    else
      ETH_DISTILL_BWD(ETH_F32);
#undef ETH_DISTILL_BWD
    ETH_CHECK_LAUNCH("eth_topk_distill_bwd");
    distill_advance(a, n, dtype);
  }
  return ETH_OK;
}
