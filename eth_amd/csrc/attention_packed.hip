// Causal attention over sequences of different lengths packed into one row
// dimension, with query heads that share key and value heads, forward and
// backward, on CDNA4 matrix cores (v_mfma_f32_32x32x16_{bf16,f16}).
//
// Rows [begin, begin + len) of q [T, n, hd], k and v [T, m, hd] are one
// sequence, n = m * group; query head h reads key/value head h / group:
//   S_ij = scale q_i . k_j (j <= i in the sequence), P = softmax_j S, O = P V
//   delta_i = sum dO_i . O_i,  dV_j = sum_i P_ij dO_i
//   dS = P (dO V^T - delta),   dQ = scale dS K,  dK = scale dS^T Q
// with dK and dV summed over the queries of all heads of the group.
//
// The host lists the tiles (blocks of queries, blocks of keys, blocks of rows
// that no sequence covers) once for a batch, longest chains first; a workgroup
// takes one tile of the list and one head or group of heads.
//
// Arithmetic and layouts are those of attention.hip: S^T = K Q^T with K rows
// read in swizzled order, so that P^T stays in registers as the operand of
// O^T = V^T P^T; 64-row blocks go global->LDS by direct loads into XOR-swizzled
// images a block ahead; fp32 base-2 softmax.  P and dS are rounded to the
// inputs' type for the second product, as the matrix cores take it, and delta is
// formed of the stored output: dQ and dK are 0.0025 of their norm from 64 bits in
// bf16 (8192 rows, heads of 128): 0.0017 by the rounding of the results, 0.0017 by that
// of dS and 0.0007 by that of the output in delta (0.0016 to 0.002 in sequences of 30 rows,
// whose dQ and dK are 0.003 off).  A further product with what the rounding of dS
// leaves would bring about 0.0020, and take a quarter more time backward (16384 rows,
// 8 heads of 64 on one: 982 -> 1223 us), which buys less than one bit of a gradient
// that is rounded to 8.  In fp16 (11 bits) all of it is an eighth: 0.0003 to 0.0004
// where the rounding of the results alone is 0.0002, for gradients of any size (see
// kGradShift).
//
// The same call gives the same bits every time.  A row's bits do depend on what
// else is in the call, within these roundings: one query's scores can move the
// exponent offset of the 31 beside it in its wave (fp16: its dS that of theirs), and
// the whole batch decides which chains are cut where.
//
// What bounds it: the exponentials and the products, which share a SIMD's issue
// and the card's power (the clock falls to 1.6-1.8 GHz under them, where waiting
// costs little and instructions count).  Of all SIMDs' cycles the matrix cores
// and the VALU are busy: forward 0.53 and 0.71 at a head dim of 64, 0.51 and 0.48 at
// 128; dQ 0.61 and 0.67, 0.52 and 0.39; dK/dV 0.50 and 0.40, 0.47 and 0.30.  LDS is at
// 0.27-0.38 throughout, with bank conflicts in at most 0.012; HBM is idle.  dK/dV at
// 128 fills none of them: its waves wait 0.28 of their time for loads and at the
// barrier of every 64 queries, and nothing else is on the CU.
//
// A block's buffer resource starts at its first row and ends with its
// sequence's last element, so that rows past the sequence read zeros without a
// comparison (a neighbour's infinities never meet a zero probability), and
// offsets within it fit 32 bits whatever the tensors' size.
#include "attention_tiles.h"

namespace eth {

struct PackIn {
  const uint16_t* p;
  int64_t ss, sh;  // strides of row and head (elements); dim contiguous
};
struct PackOut {
  uint16_t* p;
  int64_t ss, sh;
};

struct PackArgs {
  PackIn q, k, v, o, dout;
  PackOut out, dq, dk, dv;
  float* lse;    // [n, T] log2-domain: m2 + log2(l)
  float* delta;  // [n, T] rowsum(dO * O)
  const eth_packed_tile_t* q_tiles;
  const eth_packed_tile_t* k_tiles;
  eth_packed_split_t q_split, k_split;
  float4* partial;  // accumulators of split tiles' pieces
  int64_t T;
  int n, m, group;
  int hp;  // query heads per workgroup (1, 2 or 4; divides group)
  int hd;  // head dim (<= the kernel's D; columns hd..D-1 are zero padding)
  float scale_log2;  // scale * log2(e)
  float scale;
};

__device__ __forceinline__ const uint16_t* row_ptr(const PackIn& t, int64_t row, int h) {
  return t.p + row * t.ss + (int64_t)h * t.sh;
}
__device__ __forceinline__ uint16_t* row_ptr(const PackOut& t, int64_t row, int h) {
  return t.p + row * t.ss + (int64_t)h * t.sh;
}

// A tile's chain of steps may be split over several workgroups (`pieces`), whose
// fp32 accumulators a second kernel joins in order: the first split.tiles
// tiles of a list, which have the longest chains, take split.pieces workgroups
// per head each, and those behind them one.
struct Piece {
  int tile, head, piece;  // tile of the list, head (or group of heads)
  int pieces;             // 1: the tile is not split
};
__device__ __forceinline__ Piece piece_of(int block, int heads, const eth_packed_split_t& sp) {
  const int head = block % heads, r = block / heads, cut = sp.tiles * sp.pieces;
  if (r >= cut) return Piece{sp.tiles + r - cut, head, 0, 1};
  return Piece{r % sp.tiles, head, r / sp.tiles, sp.pieces};
}
// steps of a piece: equal shares, of split.steps or a little less each; the
// last of a short tile's pieces may be left without any
struct Steps {
  int from, to, used;  // used: pieces that have steps
};
__device__ __forceinline__ Steps steps_of(int chain, int piece, int pieces, int steps) {
  if (pieces == 1) return Steps{0, chain, 1};
  const int want = min((chain + steps - 1) / steps, pieces), share = (chain + want - 1) / want;
  return Steps{min(piece * share, chain), min((piece + 1) * share, chain), (chain + share - 1) / share};
}
// A wave's accumulators of a piece as it holds them, whole float4 vectors side
// by side: vector i of wave w of a piece's `waves`
template <int DT>
__device__ __forceinline__ float4* partial_of(const PackArgs& a, const eth_packed_split_t& sp, int heads,
                                              const Piece& pc, int piece, int waves, int w, int lane) {
  return a.partial + ((((int64_t)pc.tile * heads + pc.head) * sp.pieces + piece) * waves + w) * (DT * 4 * 64) + lane;
}
template <int DT>
__device__ __forceinline__ void put_partial(float4* p, const a_f32x16 (&x)[DT]) {
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      p[(t * 4 + g) * 64] = make_float4(x[t][g * 4], x[t][g * 4 + 1], x[t][g * 4 + 2], x[t][g * 4 + 3]);
}
template <int DT>
__device__ __forceinline__ void add_partial(const float4* p, a_f32x16 (&x)[DT], float f) {
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const float4 u = p[(t * 4 + g) * 64];
      x[t][g * 4 + 0] += u.x * f;
      x[t][g * 4 + 1] += u.y * f;
      x[t][g * 4 + 2] += u.z * f;
      x[t][g * 4 + 3] += u.w * f;
    }
}
// fp16 gradients: P is about 1/L along L keys, and dS = P (dP - delta) is smaller or
// larger by the upstream gradient's size: rounded as they are, both leave fp16's
// normal numbers (4000 rows, gradients of 1e-4: dQ 0.0126 of its norm off, where its
// own rounding is 0.0023; with dP of 2^18 dS is infinite).  The second products take
// them times powers of two, which the results lose again: P times 2^kProbShift (the
// largest P is 1, but for scores so far out that it is not exact any more), dS times
// 2^shift, which starts above any use and falls, for the wave, where a |dS| passes
// kMostGrad.  Backward of 8192 packed rows, 16 heads of 128 on four: 281 -> 284 us;
// 16384, 8 of 64 on one: 1153 -> 1173; 16 x 512 rows, 16 heads of 64: 70 -> 73.
constexpr int kProbShift = 12;
constexpr int kGradShift = 64;
constexpr float kMostGrad = 32768.f;
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }
// dS (times 2^shift) and the sums of it so far made smaller where dS asks for it;
// returns by how much shift fell.  A lane with a value that is not finite has
// no finite sum to keep and does not count.
template <int DT>
__device__ __forceinline__ int fit_grads(a_f32x16& ds, a_f32x16 (&sum)[DT], int& shift) {
  float most = 0.f;
#pragma unroll
  for (int r = 0; r < 16; ++r) most = fmaxf(most, fabsf(ds[r]));
  if (__builtin_expect(!__any(most > kMostGrad), 1)) return 0;
  most = most < INFINITY ? most : 0.f;
  most = wave_max(most);
  if (!(most > kMostGrad)) return 0;
  const int down = (int)(__builtin_amdgcn_readfirstlane(__float_as_uint(most)) >> 23) - (127 + 9);  // to 2^9 ..
  const float f = pow2(-down);
#pragma unroll
  for (int r = 0; r < 16; ++r) ds[r] *= f;
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) sum[t][r] *= f;
  shift -= down;
  return down;
}
template <int DT>
__device__ __forceinline__ void times(a_f32x16 (&x)[DT], float f) {
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) x[t][r] *= f;
}
// 32 rows of [rows, D] 16-bit values in the wave's own `stage` (rows SL elements
// apart) to rows r0 .. of a head, those below len, in 16-byte row chunks
template <int D, int SL>
__device__ __forceinline__ void store_staged(const PackOut& out, const uint16_t* stage, int64_t begin, int r0, int len,
                                             int head, int hd, int lane) {
  constexpr int CPR = D / 8;
  wave_lds_fence();  // a wave reads back only its own rows
#pragma unroll
  for (int i = 0; i < 32 * CPR / 64; ++i) {
    const int c = i * 64 + lane, r = c / CPR, col = (c % CPR) * 8;
    if (r0 + r >= len || col >= hd) continue;
    *reinterpret_cast<uint4*>(row_ptr(out, begin + r0 + r, head) + col) =
        *reinterpret_cast<const uint4*>(stage + r * SL + col);
  }
}
// A [D, 32 rows] accumulator (lane = row), times f, rounded, by way of `stage`:
// straight from the registers a store would write 16 bytes of each of 32 rows
// (forward of 8192 packed rows, 16 heads of 128 on four: 70.6 -> 66.0 us, of 80
// sequences of 100 rows 32.4 -> 30.0)
template <int D, int SL, bool FP16>
__device__ __forceinline__ void store_rows(const PackOut& out, uint16_t* stage, const a_f32x16 (&x)[D / 32], float f,
                                           int64_t begin, int r0, int len, int head, int hd, int lane) {
  uint16_t* p = stage + (lane & 31) * SL + (lane >> 5) * 4;
#pragma unroll
  for (int t = 0; t < D / 32; ++t)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<uint2*>(p + t * 32 + g * 8) =
          make_uint2(pack2<FP16>(x[t][g * 4 + 0] * f, x[t][g * 4 + 1] * f),
                     pack2<FP16>(x[t][g * 4 + 2] * f, x[t][g * 4 + 3] * f));
  store_staged<D, SL>(out, stage, begin, r0, len, head, hd, lane);
}
// A [32 keys, D] accumulator, times f, rounded, by way of the wave's own
// `stage` (rows SL elements apart) in 16-byte row chunks: lane holds d = t*32 +
// lane%32 of keys acc_row(r, hl)
template <int D, int SL, bool FP16>
__device__ __forceinline__ void store_keys(const PackOut& out, uint16_t* stage, const a_f32x16 (&x)[D / 32], float f,
                                           int64_t begin, int k0, int len, int kvh, int hd, int lane) {
#pragma unroll
  for (int t = 0; t < D / 32; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r)
      stage[acc_row(r, lane >> 5) * SL + t * 32 + (lane & 31)] = from_f<FP16>(x[t][r] * f);
  store_staged<D, SL>(out, stage, begin, k0, len, kvh, hd, lane);
}

// Direct loads of 64-row blocks of one head of one sequence by four waves:
// unit u (16 bytes) of the image holds row u / CPR, chunk (u % CPR) ^
// img_swz(row).  Rows past the sequence and columns past the head dim read
// zeros (the latter have offsets past any range).
template <int D>
struct SeqCopy {
  static constexpr int CPR = D / 8;  // 16-byte chunks per row
  static constexpr int PW = D / 32;  // 1 KB pieces per wave
  int32_t off[PW];
  const char* base;    // the sequence's first row of head 0
  int64_t row_bytes, range;
  int w;
  __device__ __forceinline__ void init(const PackIn& t, int64_t begin, int len, int hd, int wave, int lane) {
    base = reinterpret_cast<const char*>(t.p + begin * t.ss);
    row_bytes = t.ss * 2;
    range = (int64_t)(len - 1) * row_bytes + hd * 2;
    w = wave;
#pragma unroll
    for (int j = 0; j < PW; ++j) {
      const int u = (w * PW + j) * 64 + lane;
      const int r = u / CPR, c = (u % CPR) ^ img_swz<D>(r);
      off[j] = c * 8 < hd ? (int32_t)(r * row_bytes + c * 16) : kAttnOob;
    }
  }
  // rows r0 .. r0 + 63 of the head at `head` (bytes)
  __device__ __forceinline__ void issue(uint16_t* S, int r0, int64_t head) const {
    const int64_t at = r0 * row_bytes;
    int64_t left = range - at;
    left = left < 0 ? 0 : (left > 0x7fffffff ? 0x7fffffff : left);
    const a_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base + head + at), (short)0, (int)left,
                                                          0x00020000);
#pragma unroll
    for (int j = 0; j < PW; ++j) {
      const int32_t o = off[j];
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)(S + (w * PW + j) * 512),
                                               16, o, 0, 0, 0);
    }
  }
};

// zeros into `rows` rows from `row0` on of heads h0 .. h0 + nh - 1 (a tile of
// rows that no sequence covers), by `threads` threads
__device__ __forceinline__ void zero_rows(const PackOut& t, int64_t row0, int rows, int h0, int nh, int hd,
                                          int threads) {
  const int cpr = hd / 8, per = rows * cpr;
  for (int i = threadIdx.x; i < nh * per; i += threads) {
    const int h = i / per, r = (i - h * per) / cpr, c = i % cpr;
    *reinterpret_cast<uint4*>(row_ptr(t, row0 + r, h0 + h) + c * 8) = make_uint4(0u, 0u, 0u, 0u);
  }
}

// ------------------------------------------------------------------ forward --
// Largest sum of a lane's 32 P of a block before the maximum is taken again:
// within fp16, whose P is rounded relative to its own size all the same
constexpr float kMostSum = 1024.f;

// 4 waves x 32 rows; a row is a (query, head) pair: hp heads of a group share
// the workgroup's K and V blocks, 128 / hp queries each, so that a short
// sequence wastes less of a tile and the waves' chains are of equal length.
// 16384 rows, 8 heads of 64 on one: 300 us, 0.92 PFLOP/s; 4 x 2048 rows, 16 heads of
// 128: 79.9 us, 0.86; 96 rows in three sequences 4.9 us (launches of one graph).
template <int D, bool FP16>
__global__ void __launch_bounds__(kAttnThreads, 2) packed_fwd_kernel(PackArgs a) {
  constexpr int KS = D / 16;  // k-steps over the head dim
  constexpr int DT = D / 32;  // 32-row tiles over the head dim
  constexpr int IMG = kBKV * D;  // elements of one image
  __shared__ __attribute__((aligned(16))) uint16_t K0[IMG];
  __shared__ __attribute__((aligned(16))) uint16_t K1[IMG];
  __shared__ __attribute__((aligned(16))) uint16_t V0[IMG];
  __shared__ __attribute__((aligned(16))) uint16_t V1[IMG];

  // workgroups of one key/value head a multiple of m apart: on one die for
  // m % 8 == 0, whose L2 then serves the shared rows
  const int hbs = a.n / a.hp;
  const Piece pc = piece_of(blockIdx.x, hbs, a.q_split);
  const int kvh = pc.head % a.m, h0 = kvh * a.group + pc.head / a.m * a.hp;
  const eth_packed_tile_t tile = a.q_tiles[pc.tile];
  const int64_t begin = tile.begin;
  if (tile.len < 0) {
    zero_rows(a.out, begin, -tile.len, h0, a.hp, a.hd, kAttnThreads);
    for (int i = threadIdx.x; i < a.hp * -tile.len; i += kAttnThreads)
      a.lse[(int64_t)(h0 + i / -tile.len) * a.T + begin + i % -tile.len] = -INFINITY;
    return;
  }
  const int len = tile.len, bq = kBQ / a.hp;
  const int lane = threadIdx.x & 63, hl = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // wave-uniform
  const int h = h0 + w % a.hp;
  const int q0 = tile.start + w / a.hp * 32;
  const int q = q0 + (lane & 31);
  const bool real = q < len;
  const float sl2 = a.scale_log2;

  SeqCopy<D> kc, vc;
  kc.init(a.k, begin, len, a.hd, w, lane);
  vc.init(a.v, begin, len, a.hd, w, lane);
  const int64_t kh = kvh * a.k.sh * 2, vh = kvh * a.v.sh * 2;
  const int qend = min(tile.start + bq, len);  // past the tile's last query
  const Steps st = steps_of((qend + kBKV - 1) / kBKV, pc.piece, pc.pieces, a.q_split.steps);
  const int nkv = st.to;
  if (st.from >= nkv) return;
  kc.issue(K0, st.from * kBKV, kh);
  vc.issue(V0, st.from * kBKV, vh);

  uint4 qf[KS];
  {
    const uint16_t* qp = row_ptr(a.q, begin + q, h);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = load_row16<true>(qp, real, ks * 16 + hl * 8, a.hd);
  }
  a_f32x16 o[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) o[t] = a_f32x16{};
  // exponent offset (log2 units; the running max when last taken) and sum for
  // query q; the lowest finite start keeps exp2(-inf - m) at 0 for masked keys
  float m = -3.4028234e38f, l = 0.f;

  int aoff[KS], toff[DT][2];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) aoff[ks] = img_row_off<D>(lane, ks);
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int hi = 0; hi < 2; ++hi) toff[dt][hi] = img_tr_off<D>(lane, dt, hi);
  vm_wait_all();
  __syncthreads();

  auto block = [&](int j, auto cur_c) __attribute__((always_inline)) {
    constexpr int cur = decltype(cur_c)::value;
    const int kv0 = j * kBKV;
    if (j + 1 < nkv) {  // the next block, a block ahead
      kc.issue(cur ? K0 : K1, kv0 + kBKV, kh);
      vc.issue(cur ? V0 : V1, kv0 + kBKV, vh);
    }
    if (kv0 <= q0 + 31 && q0 < len) {  // wave has at least one unmasked key in the block
      const uint16_t* ki = cur ? K1 : K0;
      const uint16_t* vi = cur ? V1 : V0;
      // S^T = K Q^T (raw scores; lane = query, registers = 32 of the keys);
      // fragment order pinned as in the equal-length kernel
      a_f32x16 sc[2];
      {
        uint4 kr[KS];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) kr[ks] = *reinterpret_cast<const uint4*>(ki + aoff[ks]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          sc[0] = mma<FP16>(kr[ks], qf[ks], ks == 0 ? a_f32x16{} : sc[0]);
          __builtin_amdgcn_sched_barrier(0);
          kr[ks] = *reinterpret_cast<const uint4*>(ki + 32 * D + aoff[ks]);
          __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) sc[1] = mma<FP16>(kr[ks], qf[ks], ks == 0 ? a_f32x16{} : sc[1]);
      }
      if (kv0 + kBKV - 1 > q0) {  // diagonal block: mask keys after the query
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (kv0 + t * 32 + swz_row(r, hl) > q) sc[t][r] = -INFINITY;
      }
      // P at the exponent offset m of the blocks before (O / l and lse do not
      // depend on it): only where a lane's sum says that m has fallen too far
      // below the scores, or that there was none yet, is the maximum taken.  The
      // VALU has the most to do here (at a head dim of 64 it was busy 0.81 of the
      // cycles with the maximum, 0.71 without): 16384 rows of 8 heads on one 299.4 -> 294.5
      // us, 24 heads on three of 3000, 100 and 5000 rows 124.8 -> 117.3, 8192 rows of
      // 16 heads of 128 81.4 -> 79.3.
      uint32_t pk[2][8];
      float rs = 0.f;
      auto probs = [&]() __attribute__((always_inline)) {
        rs = 0.f;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float p0 = fast_exp2(__builtin_fmaf(sc[t][2 * i], sl2, -m));
            const float p1 = fast_exp2(__builtin_fmaf(sc[t][2 * i + 1], sl2, -m));
            rs += p0;
            rs += p1;
            pk[t][i] = pack2<FP16>(p0, p1);
          }
      };
      probs();
      if (__any(!(rs <= kMostSum))) {
        float mx = sc[0][0];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int r = 0; r < 16; ++r) mx = fmaxf(mx, sc[t][r]);
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float mnew = fmaxf(m, mx * sl2), alpha = fast_exp2(m - mnew);
        l *= alpha;
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[t][r] *= alpha;
        m = mnew;
        probs();
      }
      l += rs;
      // O^T += V^T P^T over the 64 keys (4 k-steps of 16)
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        const int t = kk >> 1, i0 = (kk & 1) * 4;
        const uint4 pb = make_uint4(pk[t][i0], pk[t][i0 + 1], pk[t][i0 + 2], pk[t][i0 + 3]);
        const uint16_t* vp = vi + kk * 16 * D;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[dt] = mma<FP16>(img_tr(vp, toff[dt][0], toff[dt][1]), pb, o[dt]);
      }
    }
    vm_wait_all();  // the next block's rows have landed
    __syncthreads();  // this block's images free, the next block's visible
  };
  int j = st.from;
  for (; j + 1 < nkv; j += 2) {
    block(j, std::integral_constant<int, 0>{});
    block(j + 1, std::integral_constant<int, 1>{});
  }
  if (j < nkv) block(j, std::integral_constant<int, 0>{});
  l += __shfl_xor(l, 32, 64);
  if (pc.pieces > 1) {
    put_partial<DT>(partial_of<DT>(a, a.q_split, hbs, pc, pc.piece, 4, w, lane), o);
    float2* ml = reinterpret_cast<float2*>(a.partial + (int64_t)a.q_split.tiles * hbs * a.q_split.pieces * (DT * 1024));
    ml[((((int64_t)pc.tile * hbs + pc.head) * a.q_split.pieces + pc.piece) * 4 + w) * 64 + lane] = make_float2(m, l);
    return;
  }
  if (q0 >= len) return;  // rows past the sequence
  uint16_t* stage = w == 0 ? K0 : w == 1 ? K1 : w == 2 ? V0 : V1;
  store_rows<D, D + 8, FP16>(a.out, stage, o, 1.0f / l, begin, q0, len, h, a.hd, lane);
  if (hl == 0 && real) a.lse[(int64_t)h * a.T + begin + q] = m + log2f(l);
}

// joins the pieces of split query tiles, in order, a wave's rows per workgroup
template <int D, bool FP16>
__global__ void __launch_bounds__(64) packed_fwd_join_kernel(PackArgs a) {
  constexpr int DT = D / 32;
  __shared__ __attribute__((aligned(16))) uint16_t stage[32 * (D + 8)];
  const int hbs = a.n / a.hp;
  const int w = blockIdx.x % 4, r = blockIdx.x / 4;
  const Piece pc{r / hbs, r % hbs, 0, a.q_split.pieces};
  const int kvh = pc.head % a.m, h0 = kvh * a.group + pc.head / a.m * a.hp;
  const eth_packed_tile_t tile = a.q_tiles[pc.tile];
  if (tile.len < 0) return;  // (stored as zeros by the first launch)
  const int lane = threadIdx.x;
  const int h = h0 + w % a.hp, q = tile.start + w / a.hp * 32 + (lane & 31);
  const int qend = min(tile.start + kBQ / a.hp, tile.len);
  const int used = steps_of((qend + kBKV - 1) / kBKV, 0, pc.pieces, a.q_split.steps).used;
  const float2* ml = reinterpret_cast<const float2*>(a.partial + (int64_t)a.q_split.tiles * hbs * a.q_split.pieces *
                                                                     (DT * 1024)) +
                     (((int64_t)pc.tile * hbs + pc.head) * a.q_split.pieces * 4 + w) * 64 + lane;
  float m = -3.4028234e38f, l = 0.f;
  for (int i = 0; i < used; ++i) m = fmaxf(m, ml[i * 256].x);
  a_f32x16 o[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) o[t] = a_f32x16{};
  for (int i = 0; i < used; ++i) {
    const float2 x = ml[i * 256];
    const float f = fast_exp2(x.x - m);
    l += x.y * f;
    add_partial<DT>(partial_of<DT>(a, a.q_split, hbs, pc, i, 4, w, lane), o, f);
  }
  store_rows<D, D + 8, FP16>(a.out, stage, o, 1.0f / l, tile.begin, q - (lane & 31), tile.len, h, a.hd, lane);
  if (lane < 32 && q < tile.len) a.lse[(int64_t)h * a.T + tile.begin + q] = m + log2f(l);
}

// ------------------------------------------------------------ backward: dQ --
// Workgroups as in the forward.  Runs first: it also writes delta, which the
// dK/dV kernels read.  S is formed again here and there: seven products for the
// five that a single pass would take, whose dQ however would be summed by atomics
// in no fixed order.  410 us at 16384 rows, 8 heads of 64 on one; 94 us at 8192
// packed rows, 16 heads of 128 on four.
template <int D, bool FP16>
__global__ void __launch_bounds__(kAttnThreads, 2) packed_bwd_dq_kernel(PackArgs a) {
  constexpr int KS = D / 16, DT = D / 32;
  constexpr int IMG = kBKV * D;  // elements of one image
  __shared__ __attribute__((aligned(16))) uint16_t K0[IMG];
  __shared__ __attribute__((aligned(16))) uint16_t K1[IMG];
  __shared__ __attribute__((aligned(16))) uint16_t V0[IMG];
  __shared__ __attribute__((aligned(16))) uint16_t V1[IMG];

  const int hbs = a.n / a.hp;
  const Piece pc = piece_of(blockIdx.x, hbs, a.q_split);
  const int kvh = pc.head % a.m, h0 = kvh * a.group + pc.head / a.m * a.hp;
  const eth_packed_tile_t tile = a.q_tiles[pc.tile];
  const int64_t begin = tile.begin;
  if (tile.len < 0) {
    zero_rows(a.dq, begin, -tile.len, h0, a.hp, a.hd, kAttnThreads);
    return;
  }
  const int len = tile.len, bq = kBQ / a.hp;
  const int lane = threadIdx.x & 63, hl = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // wave-uniform
  const int h = h0 + w % a.hp;
  const int q0 = tile.start + w / a.hp * 32;
  const int q = q0 + (lane & 31);
  const bool real = q < len;

  SeqCopy<D> kc, vc;
  kc.init(a.k, begin, len, a.hd, w, lane);
  vc.init(a.v, begin, len, a.hd, w, lane);
  const int64_t kh = kvh * a.k.sh * 2, vh = kvh * a.v.sh * 2;
  const int qend = min(tile.start + bq, len);
  const Steps st = steps_of((qend + kBKV - 1) / kBKV, pc.piece, pc.pieces, a.q_split.steps);
  const int nkv = st.to;
  if (st.from >= nkv) return;
  kc.issue(K0, st.from * kBKV, kh);
  vc.issue(V0, st.from * kBKV, vh);

  uint4 qf[KS], of[KS];
  {
    const uint16_t* qp = row_ptr(a.q, begin + q, h);
    const uint16_t* op = row_ptr(a.dout, begin + q, h);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      qf[ks] = load_row16<true>(qp, real, ks * 16 + hl * 8, a.hd);
      of[ks] = load_row16<true>(op, real, ks * 16 + hl * 8, a.hd);
    }
  }
  const int64_t srow = (int64_t)h * a.T + begin + q;
  int shift = FP16 ? kGradShift : 0;  // of dS and of the sums of it
  float lse = real ? a.lse[srow] - (float)shift : 1e30f;
  // delta = rowsum(dO * O) for this query, from the dO fragments already in
  // registers (the two half-waves hold alternate 8-element chunks of the row)
  float del = 0.f;
  {
    const uint16_t* opp = row_ptr(a.o, begin + q, h);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const uint4 ov = load_row16<true>(opp, real, ks * 16 + hl * 8, a.hd);
      const uint32_t ow[4] = {ov.x, ov.y, ov.z, ov.w};
      const uint32_t dw[4] = {of[ks].x, of[ks].y, of[ks].z, of[ks].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        del += to_f<FP16>((uint16_t)(ow[e] & 0xffffu)) * to_f<FP16>((uint16_t)(dw[e] & 0xffffu));
        del += to_f<FP16>((uint16_t)(ow[e] >> 16)) * to_f<FP16>((uint16_t)(dw[e] >> 16));
      }
    }
    del += __shfl_xor(del, 32, 64);
    if (hl == 0 && real && pc.piece == 0) a.delta[srow] = del;
  }
  a_f32x16 dq[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) dq[t] = a_f32x16{};

  int aoff[KS], toff[DT][2];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) aoff[ks] = img_row_off<D>(lane, ks);
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int hi = 0; hi < 2; ++hi) toff[dt][hi] = img_tr_off<D>(lane, dt, hi);
  vm_wait_all();
  __syncthreads();

  auto block = [&](int j, auto cur_c) __attribute__((always_inline)) {
    constexpr int cur = decltype(cur_c)::value;
    const int kv0 = j * kBKV;
    if (j + 1 < nkv) {  // the next block, a block ahead
      kc.issue(cur ? K0 : K1, kv0 + kBKV, kh);
      vc.issue(cur ? V0 : V1, kv0 + kBKV, vh);
    }
    const uint16_t* ki = cur ? K1 : K0;
    const uint16_t* vi = cur ? V1 : V0;
    // one 32-key tile at a time: S^T = K Q^T, dP^T = V dO^T (lane = query),
    // dS^T, then dQ^T += K^T dS^T over those 32 keys
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int kt0 = kv0 + t * 32;
      if (kt0 > q0 + 31 || q0 >= len) continue;  // every key of the tile follows the wave's queries
      a_f32x16 s = a_f32x16{}, dp = a_f32x16{};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        s = mma<FP16>(*reinterpret_cast<const uint4*>(ki + t * 32 * D + aoff[ks]), qf[ks], s);
        dp = mma<FP16>(*reinterpret_cast<const uint4*>(vi + t * 32 * D + aoff[ks]), of[ks], dp);
      }
      // causal mask only on the tiles that cross the diagonal
      auto dsoft = [&](auto masked) __attribute__((always_inline)) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float p = fast_exp2(__builtin_fmaf(s[r], a.scale_log2, -lse));
          dp[r] = p * (dp[r] - del);
          // (the product: a masked key's own infinities stay out of it)
          if (decltype(masked)::value && kt0 + swz_row(r, hl) > q) dp[r] = 0.f;
        }
      };
      if (kt0 + 31 > q0)
        dsoft(std::true_type{});
      else
        dsoft(std::false_type{});
      if constexpr (FP16) lse += (float)fit_grads<DT>(dp, dq, shift);
#pragma unroll
      for (int k2 = 0; k2 < 2; ++k2) {
        const int kk = t * 2 + k2, e0 = k2 * 8;
        const uint4 sb = make_uint4(pack2<FP16>(dp[e0 + 0], dp[e0 + 1]), pack2<FP16>(dp[e0 + 2], dp[e0 + 3]),
                                    pack2<FP16>(dp[e0 + 4], dp[e0 + 5]), pack2<FP16>(dp[e0 + 6], dp[e0 + 7]));
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
          dq[dt] = mma<FP16>(img_tr(ki + kk * 16 * D, toff[dt][0], toff[dt][1]), sb, dq[dt]);
      }
    }
    vm_wait_all();  // the next block's rows have landed
    __syncthreads();  // this block's images free, the next block's visible
  };
  int j = st.from;
  for (; j + 1 < nkv; j += 2) {
    block(j, std::integral_constant<int, 0>{});
    block(j + 1, std::integral_constant<int, 1>{});
  }
  if (j < nkv) block(j, std::integral_constant<int, 0>{});
  const float unit = FP16 ? pow2(-shift) : 1.f;  // (a power of two)
  if (pc.pieces > 1) {
    if constexpr (FP16) times<DT>(dq, unit);
    put_partial<DT>(partial_of<DT>(a, a.q_split, hbs, pc, pc.piece, 4, w, lane), dq);
    return;
  }
  if (q0 >= len) return;
  uint16_t* stage = w == 0 ? K0 : w == 1 ? K1 : w == 2 ? V0 : V1;
  store_rows<D, D + 8, FP16>(a.dq, stage, dq, a.scale * unit, begin, q0, len, h, a.hd, lane);
}

// joins the pieces of split query tiles, in order, a wave's rows per workgroup
template <int D, bool FP16>
__global__ void __launch_bounds__(64) packed_dq_join_kernel(PackArgs a) {
  constexpr int DT = D / 32;
  __shared__ __attribute__((aligned(16))) uint16_t stage[32 * (D + 8)];
  const int hbs = a.n / a.hp;
  const int w = blockIdx.x % 4, r = blockIdx.x / 4;
  const Piece pc{r / hbs, r % hbs, 0, a.q_split.pieces};
  const int kvh = pc.head % a.m, h0 = kvh * a.group + pc.head / a.m * a.hp;
  const eth_packed_tile_t tile = a.q_tiles[pc.tile];
  if (tile.len < 0) return;  // (stored as zeros by the first launch)
  const int lane = threadIdx.x;
  const int h = h0 + w % a.hp, q = tile.start + w / a.hp * 32 + (lane & 31);
  const int qend = min(tile.start + kBQ / a.hp, tile.len);
  const int used = steps_of((qend + kBKV - 1) / kBKV, 0, pc.pieces, a.q_split.steps).used;
  a_f32x16 dq[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) dq[t] = a_f32x16{};
  for (int i = 0; i < used; ++i) add_partial<DT>(partial_of<DT>(a, a.q_split, hbs, pc, i, 4, w, lane), dq, 1.f);
  store_rows<D, D + 8, FP16>(a.dq, stage, dq, a.scale, tile.begin, q - (lane & 31), tile.len, h, a.hd, lane);
}

// The steps of a key tile: the 64-query blocks from the tile's first query on,
// of every query head of the group, one head after the other, so that dK and
// dV of a shared head are summed in registers in a fixed order.
struct PackStep {
  int head, block;  // query head within the group, 64-query block
  __device__ __forceinline__ void next(int first, int nq) {
    if (++block == nq) {
      block = first;
      ++head;
    }
  }
  static __device__ __forceinline__ PackStep at(int i, int first, int nq) {
    const int head = i / (nq - first);
    return PackStep{head, first + i - head * (nq - first)};
  }
};

// ------------------------------------- backward: dK, dV, head dims to 96 --
// dK and dV of 32 keys in one wave, four waves per 128 keys, one barrier per
// 64 queries (see attn_bwd_dkdv_kernel).  600 us at 16384 rows, 8 heads of 64 on
// one.  Slower here: three workgroups a compute unit, at 29 spilled registers
// (982 -> 1129 us backward); both 32-query tiles of a step in one straight line
// (982 -> 981, 254 -> 256).
template <int D, bool FP16>
__global__ void __launch_bounds__(kAttnThreads, 2) packed_bwd_dkdv_kernel(PackArgs a) {
  static_assert(D == 64 || D == 96, "wider heads run on the paired kernel");
  constexpr int KS = D / 16, DT = D / 32, CPR = D / 8;
  constexpr int IMG = kBQ2 * D;  // elements of one image
  // an array per image, so the compiler can tell the direct loads into one
  // from the fragment reads of another
  __shared__ __attribute__((aligned(16))) uint16_t Q0[IMG];
  __shared__ __attribute__((aligned(16))) uint16_t Q1[IMG];
  __shared__ __attribute__((aligned(16))) uint16_t O0[IMG];
  __shared__ __attribute__((aligned(16))) uint16_t O1[IMG];
  __shared__ __attribute__((aligned(16))) float lse_s[2][kBQ2];
  __shared__ __attribute__((aligned(16))) float del_s[2][kBQ2];

  const Piece pc = piece_of(blockIdx.x, a.m, a.k_split);
  const int kvh = pc.head;
  const eth_packed_tile_t tile = a.k_tiles[pc.tile];
  const int64_t begin = tile.begin;
  if (tile.len < 0) {
    zero_rows(a.dk, begin, -tile.len, kvh, 1, a.hd, kAttnThreads);
    zero_rows(a.dv, begin, -tile.len, kvh, 1, a.hd, kAttnThreads);
    return;
  }
  const int len = tile.len;
  const int lane = threadIdx.x & 63, hl = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // wave-uniform
  const int rt = threadIdx.x;
  const int k0 = tile.start + w * 32;
  const int key = k0 + (lane & 31);

  SeqCopy<D> qc, oc;
  qc.init(a.q, begin, len, a.hd, w, lane);
  oc.init(a.dout, begin, len, a.hd, w, lane);
  // per-query statistics: threads 0-63 lse, 64-127 delta (a row past the
  // sequence gets lse = 1e30, so P = 0); delta is negated when it is stored,
  // not here, where the use would wait for every load in flight
  const float* stats = rt < 64 ? a.lse : a.delta;
  const int si = rt & 63;
  auto stat = [&](const PackStep& st) __attribute__((always_inline)) {
    float v = rt < 64 ? 1e30f : 0.f;
    const int qi = st.block * kBQ2 + si;
    if (qi < len) v = stats[(int64_t)(kvh * a.group + st.head) * a.T + begin + qi];
    return v;
  };
  auto stat_store = [&](int p, float v) __attribute__((always_inline)) {
    if (rt < 64)
      lse_s[p][rt] = FP16 ? v - (float)kProbShift : v;
    else if (rt < 128)
      del_s[p][rt - 64] = -v;
  };
  auto issue = [&](uint16_t* qi, uint16_t* oi, const PackStep& st) __attribute__((always_inline)) {
    const int64_t h = kvh * a.group + st.head;
    qc.issue(qi, st.block * kBQ2, h * a.q.sh * 2);
    oc.issue(oi, st.block * kBQ2, h * a.dout.sh * 2);
  };
  const int first = tile.start / kBQ2, nq = (len + kBQ2 - 1) / kBQ2;
  const Steps st = steps_of((nq - first) * a.group, pc.piece, pc.pieces, a.k_split.steps);
  const int steps = st.to - st.from;
  if (steps <= 0) return;
  PackStep cur = PackStep::at(st.from, first, nq), nxt = cur;
  nxt.next(first, nq);
  float stat_n = 0.f;
  issue(Q0, O0, cur);
  if (rt < 128) stat_n = stat(cur);

  uint4 kf[KS], vf[KS];  // this lane's key: K and V rows, the B operands of S and dP
  {
    const uint16_t* kp = row_ptr(a.k, begin + key, kvh);
    const uint16_t* vp = row_ptr(a.v, begin + key, kvh);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      kf[ks] = load_row16<true>(kp, key < len, ks * 16 + hl * 8, a.hd);
      vf[ks] = load_row16<true>(vp, key < len, ks * 16 + hl * 8, a.hd);
    }
  }
  a_f32x16 dk[DT], dv[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) dk[t] = dv[t] = a_f32x16{};
  int shift = kGradShift;  // fp16: of dS and dK

  int aoff[KS], toff[DT][2];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) aoff[ks] = img_row_off<D>(lane, ks);
#pragma unroll
  for (int d2 = 0; d2 < DT; ++d2)
#pragma unroll
    for (int hi = 0; hi < 2; ++hi) toff[d2][hi] = img_tr_off<D>(lane, d2, hi);
  auto bfrag = [&](const uint16_t* img, int kk, int d2) __attribute__((always_inline)) {
    return img_tr(img + kk * 16 * D, toff[d2][0], toff[d2][1]);
  };
  vm_wait_all();
  stat_store(0, stat_n);
  __syncthreads();

  auto step = [&](int i, auto par_c) __attribute__((always_inline)) {
    constexpr int P = decltype(par_c)::value;
    const int qs0 = cur.block * kBQ2;
    const bool more = i + 1 < steps;
    if (more) {  // the next step's rows into the other images, a step ahead
      issue(P ? Q0 : Q1, P ? O0 : O1, nxt);
      if (rt < 128) stat_n = stat(nxt);
    }
    const uint16_t* qi = P ? Q1 : Q0;
    const uint16_t* oi = P ? O1 : O0;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int qt = qs0 + t * 32;
      if (qt + 31 < k0 || qt >= len || k0 >= len) continue;  // every query precedes the wave's keys, or no row at all
      a_f32x16 s = a_f32x16{}, dp;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const float4 d4 = *reinterpret_cast<const float4*>(&del_s[P][t * 32 + swz_row(4 * g, hl)]);
        dp[4 * g + 0] = d4.x;
        dp[4 * g + 1] = d4.y;
        dp[4 * g + 2] = d4.z;
        dp[4 * g + 3] = d4.w;
      }
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        s = mma<FP16>(*reinterpret_cast<const uint4*>(qi + t * 32 * D + aoff[ks]), kf[ks], s);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        dp = mma<FP16>(*reinterpret_cast<const uint4*>(oi + t * 32 * D + aoff[ks]), vf[ks], dp);
      // P; query of register r = qt + swz_row(r, hl); the causal mask only on
      // the tiles that cross the diagonal
      auto probs = [&](auto masked) __attribute__((always_inline)) {
        const int kq = key - qt - 8 * hl;  // masked when > swz_row(r, 0)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float4 l4 = *reinterpret_cast<const float4*>(&lse_s[P][t * 32 + swz_row(4 * g, hl)]);
          const float lv[4] = {l4.x, l4.y, l4.z, l4.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = 4 * g + e;
            float p = fast_exp2(__builtin_fmaf(s[r], a.scale_log2, -lv[e]));
            if (decltype(masked)::value && kq > swz_row(r, 0)) p = 0.f;
            s[r] = p;
          }
        }
      };
      if (qt < k0 + 31)
        probs(std::true_type{});
      else
        probs(std::false_type{});
#pragma unroll
      for (int k2 = 0; k2 < 2; ++k2) {
        const int kk = t * 2 + k2, e0 = k2 * 8;
        const uint4 pa = make_uint4(pack2<FP16>(s[e0 + 0], s[e0 + 1]), pack2<FP16>(s[e0 + 2], s[e0 + 3]),
                                    pack2<FP16>(s[e0 + 4], s[e0 + 5]), pack2<FP16>(s[e0 + 6], s[e0 + 7]));
#pragma unroll
        for (int d2 = 0; d2 < DT; ++d2) dv[d2] = mma<FP16>(pa, bfrag(oi, kk, d2), dv[d2]);
      }
      if constexpr (FP16) {
        const float f = pow2(shift - kProbShift);
#pragma unroll
        for (int r = 0; r < 16; ++r) dp[r] = s[r] * f * dp[r];
        fit_grads<DT>(dp, dk, shift);
      } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) dp[r] = s[r] * dp[r];
      }
#pragma unroll
      for (int k2 = 0; k2 < 2; ++k2) {
        const int kk = t * 2 + k2, e0 = k2 * 8;
        const uint4 sa = make_uint4(pack2<FP16>(dp[e0 + 0], dp[e0 + 1]), pack2<FP16>(dp[e0 + 2], dp[e0 + 3]),
                                    pack2<FP16>(dp[e0 + 4], dp[e0 + 5]), pack2<FP16>(dp[e0 + 6], dp[e0 + 7]));
#pragma unroll
        for (int d2 = 0; d2 < DT; ++d2) dk[d2] = mma<FP16>(sa, bfrag(qi, kk, d2), dk[d2]);
      }
    }
    cur = nxt;
    nxt.next(first, nq);
    vm_wait_all();  // the next step's rows and statistics have landed
    if (more) stat_store(P ^ 1, stat_n);
    __syncthreads();  // this step's images free, the next step's visible
  };
  int i = 0;
  for (; i + 1 < steps; i += 2) {
    step(i, std::integral_constant<int, 0>{});
    step(i + 1, std::integral_constant<int, 1>{});
  }
  if (i < steps) step(i, std::integral_constant<int, 0>{});

  const float dv_unit = FP16 ? pow2(-kProbShift) : 1.f, dk_unit = FP16 ? pow2(-shift) : 1.f;
  if (pc.pieces > 1) {
    if constexpr (FP16) {
      times<DT>(dv, dv_unit);
      times<DT>(dk, dk_unit);
    }
    put_partial<DT>(partial_of<DT>(a, a.k_split, a.m, pc, pc.piece, 8, w, lane), dv);
    put_partial<DT>(partial_of<DT>(a, a.k_split, a.m, pc, pc.piece, 8, 4 + w, lane), dk);
    return;
  }
  // dV by way of the dO images, dK of the Q images
  static_assert(2 * 32 * D <= IMG, "two waves' staging fits an image");
  store_keys<D, D, FP16>(a.dv, (w < 2 ? O0 : O1) + (w & 1) * 32 * D, dv, dv_unit, begin, k0, len, kvh, a.hd, lane);
  store_keys<D, D, FP16>(a.dk, (w < 2 ? Q0 : Q1) + (w & 1) * 32 * D, dk, a.scale * dk_unit, begin, k0, len, kvh, a.hd, lane);
}

// ------------------------------ backward: dK, dV paired, head dims to 128 --
// Eight waves: wave w < 4 (the dV wave) and wave w + 4 (the dK wave) own the
// same 32 keys and share a SIMD, skewed by half a step (see
// attn_bwd_dkdv_x128_kernel): in step j the dV wave computes S(j) and P(j),
// hands P (fp32) over through LDS and adds P(j)^T dO(j) into dV, while the dK
// wave first finishes step j-1 and then computes dP(j) - delta.  Three Q
// images, two dO images and two P buffers (145 KB of LDS).  165 us at 8192 packed
// rows, 16 heads of 128 on four.
template <bool FP16>
__global__ void __launch_bounds__(2 * kAttnThreads, 1) packed_bwd_dkdv_x128_kernel(PackArgs a) {
  constexpr int D = 128, KS = D / 16, DT = D / 32;
  constexpr int IMG = kBQ2 * D;  // elements of one image
  __shared__ __attribute__((aligned(16))) uint16_t Qx[3 * IMG];
  __shared__ __attribute__((aligned(16))) uint16_t O0[IMG];
  __shared__ __attribute__((aligned(16))) uint16_t O1[IMG];
  __shared__ a_u32x4 Ps[2][4][2][4][64];
  __shared__ __attribute__((aligned(16))) float lse_s[2][kBQ2];
  __shared__ __attribute__((aligned(16))) float del_s[2][kBQ2];

  const Piece pc = piece_of(blockIdx.x, a.m, a.k_split);
  const int kvh = pc.head;
  const eth_packed_tile_t tile = a.k_tiles[pc.tile];
  const int64_t begin = tile.begin;
  if (tile.len < 0) {
    zero_rows(a.dk, begin, -tile.len, kvh, 1, a.hd, 2 * kAttnThreads);
    zero_rows(a.dv, begin, -tile.len, kvh, 1, a.hd, 2 * kAttnThreads);
    return;
  }
  const int len = tile.len;
  const int lane = threadIdx.x & 63, hl = lane >> 5;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // wave-uniform
  const int w = wv & 3;
  const bool dkw = wv >= 4;  // the dK wave of its pair
  const int rt = threadIdx.x & (kAttnThreads - 1);
  const int k0 = tile.start + w * 32;
  const int key = k0 + (lane & 31);

  // B operands of the first product: K rows (S = Q K^T) in the dV wave, V
  // rows (dP = dO V^T) in the dK wave
  uint4 kf[KS];
  {
    const uint16_t* kp = row_ptr(dkw ? a.v : a.k, begin + key, kvh);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) kf[ks] = load_row16<true>(kp, key < len, ks * 16 + hl * 8, a.hd);
  }
  int shift = kGradShift;  // fp16: of dS and dK (the dK wave)
  a_f32x16 acc[DT];  // dV in the dV wave, dK in the dK wave
#pragma unroll
  for (int t = 0; t < DT; ++t) acc[t] = a_f32x16{};

  // direct loads: the dV waves move Q, the dK waves dO
  SeqCopy<D> sc;
  sc.init(dkw ? a.dout : a.q, begin, len, a.hd, w, lane);
  const int64_t head_bytes = (dkw ? a.dout.sh : a.q.sh) * 2;
  auto issue = [&](uint16_t* img, const PackStep& st) __attribute__((always_inline)) {
    sc.issue(img, st.block * kBQ2, (kvh * a.group + st.head) * head_bytes);
  };
  int aoff[KS], toff[DT][2];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) aoff[ks] = img_row_off<D>(lane, ks);
#pragma unroll
  for (int d2 = 0; d2 < DT; ++d2)
#pragma unroll
    for (int hi = 0; hi < 2; ++hi) toff[d2][hi] = img_tr_off<D>(lane, d2, hi);
  auto bfrag = [&](const uint16_t* img, int kk, int d2) __attribute__((always_inline)) {
    return img_tr(img + kk * 16 * D, toff[d2][0], toff[d2][1]);
  };
  // acc += X^T B over a step's 64 queries: X (P or dS, one 32-query tile per
  // t) as the A operand, B from the transposing reads of `img`, four B
  // fragments in flight (order pinned: the scheduler otherwise hoists every
  // read and runs out of registers).  With `pbuf` (the dK wave), tile t's X is
  // first formed as dS = P (dP - delta) from P in `pbuf`.
  auto second = [&](a_f32x16 (&x)[2], const uint16_t* img, const a_u32x4 (*pbuf)[2][4][64])
                    __attribute__((always_inline)) {
    uint4 fb[DT];
#pragma unroll
    for (int d2 = 0; d2 < DT; ++d2) fb[d2] = bfrag(img, 0, d2);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      if (pbuf) {
        const float f = pow2(shift - kProbShift);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const a_u32x4 pv = pbuf[w][t][g][lane];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            x[t][4 * g + e] = (FP16 ? __uint_as_float(pv[e]) * f : __uint_as_float(pv[e])) * x[t][4 * g + e];
        }
        if constexpr (FP16) fit_grads<DT>(x[t], acc, shift);
      }
#pragma unroll
      for (int k2 = 0; k2 < 2; ++k2) {
        const int kk = t * 2 + k2, e0 = k2 * 8;
        const uint4 pa = make_uint4(pack2<FP16>(x[t][e0 + 0], x[t][e0 + 1]), pack2<FP16>(x[t][e0 + 2], x[t][e0 + 3]),
                                    pack2<FP16>(x[t][e0 + 4], x[t][e0 + 5]), pack2<FP16>(x[t][e0 + 6], x[t][e0 + 7]));
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int d2 = 0; d2 < DT; ++d2) {
          acc[d2] = mma<FP16>(pa, fb[d2], acc[d2]);
          __builtin_amdgcn_sched_barrier(0);
          if (kk < 3) fb[d2] = bfrag(img, kk + 1, d2);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
  };
  // x = (rows of img) kf^T over the 64 queries of a step, starting at x0(t):
  // S (dV wave) or dP (dK wave), query of register r of tile t = t*32 +
  // swz_row(r, hl); a rolling window of four A fragments
  auto first_product = [&](a_f32x16 (&x)[2], const uint16_t* img, auto x0) __attribute__((always_inline)) {
    auto afrag = [&](int i) __attribute__((always_inline)) {  // fragment i = t*KS + ks
      return *reinterpret_cast<const uint4*>(img + (i / KS) * 32 * D + aoff[i % KS]);
    };
    uint4 fa[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) fa[i] = afrag(i);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int i = t * KS + ks;
        x[t] = mma<FP16>(fa[i & 3], kf[ks], ks == 0 ? x0(t) : x[t]);
        __builtin_amdgcn_sched_barrier(0);
        if (i + 4 < 2 * KS) fa[i & 3] = afrag(i + 4);
        __builtin_amdgcn_sched_barrier(0);
      }
  };

  const int first = tile.start / kBQ2, nq = (len + kBQ2 - 1) / kBQ2;
  const Steps st = steps_of((nq - first) * a.group, pc.piece, pc.pieces, a.k_split.steps);
  const int n = st.to - st.from;
  if (n <= 0) return;
  auto stat = [&](const PackStep& st) __attribute__((always_inline)) {
    float v = dkw ? 0.f : 1e30f;
    const int qi = st.block * kBQ2 + rt;
    if (qi < len) v = (dkw ? a.delta : a.lse)[(int64_t)(kvh * a.group + st.head) * a.T + begin + qi];
    return v;
  };
  // (delta is negated here: at the load, the use would wait for the step's
  // direct loads too)
  auto stat_store = [&](int p, float v) __attribute__((always_inline)) {
    if (dkw)
      del_s[p][rt] = -v;
    else
      lse_s[p][rt] = FP16 ? v - (float)kProbShift : v;
  };
  PackStep cur = PackStep::at(st.from, first, nq), nxt = cur;
  nxt.next(first, nq);
  float stat_n = 0.f;
  issue(dkw ? O0 : Qx, cur);
  if (rt < kBQ2) stat_n = stat(cur);
  vm_wait_all();
  if (rt < kBQ2) stat_store(0, stat_n);
  __syncthreads();

  a_f32x16 x[2];  // S then P (dV wave); dP - delta, then dS (dK wave)
  const bool any = k0 < len;
  bool active_prev = false;
  // step j (Q image j % 3; dO image, P buffer and statistics j % 2 = P, a
  // template constant)
  auto step = [&](int j, int qslot, auto par_c, auto role_c) __attribute__((always_inline)) {
    constexpr int P = decltype(par_c)::value;
    constexpr bool DKW = decltype(role_c)::value;  // the role, a constant here
    const int qs0 = cur.block * kBQ2;
    const int qnext = qslot == 2 ? 0 : qslot + 1, qprev = qslot == 0 ? 2 : qslot - 1;
    // the next step's rows into idle images; the dV waves issue theirs behind
    // their reads of this step's Q (one array holds the three Q images, so
    // the compiler waits for loads in flight to it before a read)
    auto next = [&]() __attribute__((always_inline)) {
      if (j + 1 < n) {
        issue(DKW ? (P ? O0 : O1) : Qx + qnext * IMG, nxt);
        if (rt < kBQ2) stat_n = stat(nxt);
      }
    };
    if constexpr (DKW) next();
    // a pair whose keys all follow every query of a step skips its work
    const bool active = any && qs0 + kBQ2 - 1 >= k0;
    // the sub-products are fenced from each other: the scheduler otherwise
    // hoists every fragment read of the next product above the current
    // one and runs out of registers
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (!DKW) {
      if (active) first_product(x, Qx + qslot * IMG, [](int) { return a_f32x16{}; });
      __builtin_amdgcn_sched_barrier(0);
      next();
      __builtin_amdgcn_sched_barrier(0);
      if (active) {
        const bool diag = qs0 < k0 + 31;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          auto probs = [&](auto masked) __attribute__((always_inline)) {
            // the causal mask: query qs0 + t*32 + swz_row(r, hl) precedes the
            // key when kq > t*32 + swz_row(r, 0) (a constant per register)
            const int kq = key - qs0 - 8 * hl;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              // lse of the 4 queries of registers 4g..4g+3 (consecutive)
              const float4 l4 = *reinterpret_cast<const float4*>(&lse_s[P][t * 32 + swz_row(4 * g, hl)]);
              const float lv[4] = {l4.x, l4.y, l4.z, l4.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int r = 4 * g + e;
                float p = fast_exp2(__builtin_fmaf(x[t][r], a.scale_log2, -lv[e]));
                if (decltype(masked)::value && kq > t * 32 + swz_row(r, 0)) p = 0.f;
                x[t][r] = p;
              }
            }
          };
          if (diag)
            probs(std::true_type{});
          else
            probs(std::false_type{});
#pragma unroll
          for (int g = 0; g < 4; ++g)
            Ps[P][w][t][g][lane] = a_u32x4{__float_as_uint(x[t][4 * g]), __float_as_uint(x[t][4 * g + 1]),
                                           __float_as_uint(x[t][4 * g + 2]), __float_as_uint(x[t][4 * g + 3])};
        }
        __builtin_amdgcn_sched_barrier(0);
        second(x, P ? O1 : O0, nullptr);
      }
    } else {
      if (active_prev)  // finish step j-1: dS = P (dP - delta), dK += dS^T Q
        second(x, Qx + qprev * IMG, Ps[P ^ 1]);
      __builtin_amdgcn_sched_barrier(0);
      if (active) {
        // dP - delta: the accumulator starts at -delta (stored negated)
        first_product(x, P ? O1 : O0, [&](int t) __attribute__((always_inline)) {
          a_f32x16 d;
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const float4 d4 = *reinterpret_cast<const float4*>(&del_s[P][t * 32 + swz_row(4 * g, hl)]);
            d[4 * g + 0] = d4.x;
            d[4 * g + 1] = d4.y;
            d[4 * g + 2] = d4.z;
            d[4 * g + 3] = d4.w;
          }
          return d;
        });
      }
    }
    active_prev = active;
    cur = nxt;
    nxt.next(first, nq);
    __builtin_amdgcn_sched_barrier(0);
    vm_wait_all();  // the next step's rows and statistics have landed
    if (j + 1 < n && rt < kBQ2) stat_store(P ^ 1, stat_n);
    __syncthreads();  // P(j) handed over; images of step j-1 free
  };
  // each role runs its own copy of the step loop (the same barriers in the
  // same order), so neither keeps the other's values alive
  auto run = [&](auto role_c) __attribute__((always_inline)) {
    int j = 0, qslot = 0;
    for (; j + 1 < n; j += 2) {
      step(j, qslot, std::integral_constant<int, 0>{}, role_c);
      qslot = qslot == 2 ? 0 : qslot + 1;
      step(j + 1, qslot, std::integral_constant<int, 1>{}, role_c);
      qslot = qslot == 2 ? 0 : qslot + 1;
    }
    if (j < n) {
      step(j, qslot, std::integral_constant<int, 0>{}, role_c);
      qslot = qslot == 2 ? 0 : qslot + 1;
    }
    // the dK waves finish the last step (its P is in buffer (n - 1) % 2)
    if (decltype(role_c)::value && active_prev) {
      const int pb = (n - 1) & 1, qlast = qslot == 0 ? 2 : qslot - 1;
      second(x, Qx + qlast * IMG, Ps[pb]);
    }
  };
  if (dkw)
    run(std::true_type{});
  else
    run(std::false_type{});
  const float unit = FP16 ? pow2(dkw ? -shift : -kProbShift) : 1.f;
  if (pc.pieces > 1) {
    if constexpr (FP16) times<DT>(acc, unit);
    put_partial<DT>(partial_of<DT>(a, a.k_split, a.m, pc, pc.piece, 8, wv, lane), acc);
    return;
  }
  // the staging rows are padded by 8 elements: 8.5 KB per wave, the dV waves'
  // in the Q images, the dK waves' in the P buffers
  constexpr int SL = D + 8;
  __syncthreads();  // every image and P buffer read
  uint16_t* stage = (dkw ? reinterpret_cast<uint16_t*>(&Ps[0][0][0][0][0]) : Qx) + w * 32 * SL;
  static_assert(4 * 32 * SL <= 3 * IMG && 4 * 32 * SL * 2 <= (int)sizeof(Ps), "staging fits");
  store_keys<D, SL, FP16>(dkw ? a.dk : a.dv, stage, acc, dkw ? a.scale * unit : unit, begin, k0, len, kvh, a.hd, lane);
}

// joins the pieces of split key tiles, in order, 32 keys per workgroup: wave 0
// dV, wave 1 dK (two waves rather than eight: the reads of 124 split tiles of
// 128 x 64 spread over four times the workgroups, 27 -> 25 us)
template <int D, bool FP16>
__global__ void __launch_bounds__(128) packed_dkdv_join_kernel(PackArgs a) {
  constexpr int DT = D / 32, SL = D + 8;
  __shared__ __attribute__((aligned(16))) uint16_t stage[2 * 32 * SL];
  const int w = blockIdx.x % 4, b = blockIdx.x / 4;
  const Piece pc{b / a.m, b % a.m, 0, a.k_split.pieces};
  const eth_packed_tile_t tile = a.k_tiles[pc.tile];
  if (tile.len < 0) return;  // (stored as zeros by the first launch)
  const int lane = threadIdx.x & 63;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int first = tile.start / kBQ2, nq = (tile.len + kBQ2 - 1) / kBQ2;
  const int used = steps_of((nq - first) * a.group, 0, pc.pieces, a.k_split.steps).used;
  a_f32x16 x[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) x[t] = a_f32x16{};
  for (int i = 0; i < used; ++i)
    add_partial<DT>(partial_of<DT>(a, a.k_split, a.m, pc, i, 8, wv * 4 + w, lane), x, 1.f);
  store_keys<D, SL, FP16>(wv == 0 ? a.dv : a.dk, stage + wv * 32 * SL, x, wv == 0 ? 1.f : a.scale, tile.begin,
                          tile.start + w * 32, tile.len, pc.head, a.hd, lane);
}

}  // namespace eth

using namespace eth;

// heads of a group per workgroup: as many of the four waves as divide it
static int heads_per_tile(int group) { return group % 4 == 0 ? 4 : group % 2 == 0 ? 2 : 1; }

extern "C" int eth_packed_attn_tile_rows(int heads, int kv_heads) {
  if (heads <= 0 || kv_heads <= 0 || heads % kv_heads) return 0;
  return kBQ / heads_per_tile(heads / kv_heads);
}

static bool good_strides(const void* p, const int64_t* st) {
  // (64 rows of a block within 31-bit offsets)
  return ((uintptr_t)p & 15) == 0 && st[0] % 8 == 0 && st[1] % 8 == 0 && st[0] >= 0 && st[1] >= 0 &&
         st[0] < (1LL << 24);
}

static bool good_split(const eth_packed_split_t& sp, int n_tiles, int heads) {
  if (sp.tiles == 0) return true;
  return sp.tiles > 0 && sp.tiles <= n_tiles && sp.pieces > 1 && sp.steps > 0 &&
         (int64_t)sp.tiles * sp.pieces * heads < (1LL << 24);
}
static int64_t grid_of(const eth_packed_split_t& sp, int n_tiles, int heads) {
  return (int64_t)heads * (n_tiles - sp.tiles + (sp.tiles ? sp.tiles * sp.pieces : 0));
}
// float4 vectors of a piece: 4 waves' accumulators of a query tile (and two
// statistics a lane, forward), 8 waves' of a key tile
static int64_t piece_vectors(const eth_packed_split_t& sp, int heads, int width, int waves) {
  return sp.tiles ? (int64_t)sp.tiles * sp.pieces * heads * waves * (width / 32 * 4 * 64) : 0;
}

static int width_of(int head_dim) { return head_dim > 96 ? 128 : head_dim > 64 ? 96 : 64; }

static int packed_check(const eth_packed_attn_desc_t* d) {
  ETH_CHECK_ARG(d, "packed attention: null descriptor");
  ETH_CHECK_ARG(d->dtype == ETH_BF16 || d->dtype == ETH_F16, "packed attention: dtype must be bf16/fp16");
  ETH_CHECK_ARG(d->head_dim >= 8 && d->head_dim <= 128 && d->head_dim % 8 == 0,
                "packed attention: head_dim must be a multiple of 8 in [8, 128] (got %d)", d->head_dim);
  ETH_CHECK_ARG(d->heads > 0 && d->kv_heads > 0 && d->heads % d->kv_heads == 0,
                "packed attention: heads (%d) must be a multiple of kv_heads (%d)", d->heads, d->kv_heads);
  ETH_CHECK_ARG(d->rows > 0 && d->rows < (1LL << 31), "packed attention: rows must be in [1, 2^31) (got %lld)",
                (long long)d->rows);
  ETH_CHECK_ARG(d->q_tiles && d->k_tiles && d->n_q_tiles > 0 && d->n_k_tiles > 0, "packed attention: no tiles");
  ETH_CHECK_ARG((int64_t)d->n_q_tiles * d->heads < (1LL << 31) && (int64_t)d->n_k_tiles * d->kv_heads < (1LL << 31),
                "packed attention: too many tiles");
  ETH_CHECK_ARG(good_split(d->q_split, d->n_q_tiles, d->heads) && good_split(d->k_split, d->n_k_tiles, d->kv_heads),
                "packed attention: bad split");
  // (a grid of 2^32 threads or more would be launched modulo 2^32, without an error)
  const int64_t g_q = grid_of(d->q_split, d->n_q_tiles, d->heads / heads_per_tile(d->heads / d->kv_heads)),
                g_k = grid_of(d->k_split, d->n_k_tiles, d->kv_heads);
  ETH_CHECK_ARG(g_q * kAttnThreads < (1LL << 32) && g_k * (d->head_dim > 96 ? 2 : 1) * kAttnThreads < (1LL << 32),
                "packed attention: too many tiles (%lld and %lld workgroups)", (long long)g_q, (long long)g_k);
  // (a positive scale keeps the order of the scores, and a product with -inf is -inf)
  ETH_CHECK_ARG(d->scale >= 0x1p-100f && d->scale <= 0x1p100f, "packed attention: scale must be positive and finite");
  return ETH_OK;
}

static PackArgs packed_args(const eth_packed_attn_desc_t* d) {
  PackArgs a{};
  a.q_tiles = d->q_tiles;
  a.k_tiles = d->k_tiles;
  a.q_split = d->q_split;
  a.k_split = d->k_split;
  a.T = d->rows;
  a.n = d->heads;
  a.m = d->kv_heads;
  a.group = a.n / a.m;
  a.hp = heads_per_tile(a.group);
  a.hd = d->head_dim;
  a.scale = d->scale;
  a.scale_log2 = a.scale * 1.4426950408889634f;
  return a;
}
static PackIn pin(const void* p, const int64_t* st) { return PackIn{(const uint16_t*)p, st[0], st[1]}; }
static PackOut pout(void* p, const int64_t* st) { return PackOut{(uint16_t*)p, st[0], st[1]}; }

extern "C" int64_t eth_packed_attn_workspace(const eth_packed_attn_desc_t* d, int backward) {
  if (packed_check(d)) return 0;
  const int width = width_of(d->head_dim), hbs = d->heads / heads_per_tile(d->heads / d->kv_heads);
  const int64_t q = piece_vectors(d->q_split, hbs, width, 4), k = piece_vectors(d->k_split, d->kv_heads, width, 8);
  // (the backward joins dQ's pieces before dK's and dV's are written)
  return (backward ? (q > k ? q : k) : q + q / (width / 32 * 4) / 2) * (int64_t)sizeof(float4);
}

template <int D, bool FP16>
static void launch_packed_fwd(const PackArgs& a, int grid, hipStream_t s) {
  packed_fwd_kernel<D, FP16><<<grid, kAttnThreads, 0, s>>>(a);
  if (a.q_split.tiles) packed_fwd_join_kernel<D, FP16><<<4 * a.q_split.tiles * (a.n / a.hp), 64, 0, s>>>(a);
}

template <int D, bool FP16>
static void launch_packed_bwd(const PackArgs& a, int g_q, int g_k, hipStream_t s) {
  packed_bwd_dq_kernel<D, FP16><<<g_q, kAttnThreads, 0, s>>>(a);  // first: it also writes delta
  if (a.q_split.tiles) packed_dq_join_kernel<D, FP16><<<4 * a.q_split.tiles * (a.n / a.hp), 64, 0, s>>>(a);
  if constexpr (D == 128)
    packed_bwd_dkdv_x128_kernel<FP16><<<g_k, 2 * kAttnThreads, 0, s>>>(a);
  else
    packed_bwd_dkdv_kernel<D, FP16><<<g_k, kAttnThreads, 0, s>>>(a);
  if (a.k_split.tiles) packed_dkdv_join_kernel<D, FP16><<<4 * a.k_split.tiles * a.m, 128, 0, s>>>(a);
}

extern "C" int eth_packed_attn_fwd(const eth_packed_attn_desc_t* d, const void* q, const void* k, const void* v,
                                   void* out, float* lse, void* workspace, void* stream) {
  if (int rc = packed_check(d)) return rc;
  ETH_CHECK_ARG(q && k && v && out && lse, "eth_packed_attn_fwd: null pointer");
  ETH_CHECK_ARG(good_strides(q, d->q_strides) && good_strides(k, d->k_strides) && good_strides(v, d->v_strides) &&
                    good_strides(out, d->o_strides),
                "eth_packed_attn_fwd: rows must be 16-byte aligned, strides non-negative and rows below 2^24 apart");
  PackArgs a = packed_args(d);
  a.q = pin(q, d->q_strides);
  a.k = pin(k, d->k_strides);
  a.v = pin(v, d->v_strides);
  a.out = pout(out, d->o_strides);
  a.lse = lse;
  ETH_CHECK_ARG(!a.q_split.tiles || (workspace && ((uintptr_t)workspace & 15) == 0),
                "eth_packed_attn_fwd: split tiles need a 16-byte aligned workspace");
  a.partial = (float4*)workspace;
  const int grid = (int)grid_of(a.q_split, d->n_q_tiles, a.n / a.hp);
  hipStream_t s = (hipStream_t)stream;
  const bool fp16 = d->dtype == ETH_F16;
#define ETH_PACKED_FWD(D)                        \
  if (fp16)                                      \
    launch_packed_fwd<D, true>(a, grid, s);      \
  else                                           \
    launch_packed_fwd<D, false>(a, grid, s);
  const int width = width_of(a.hd);
  if (width == 128) {
    ETH_PACKED_FWD(128)
  } else if (width == 96) {
    ETH_PACKED_FWD(96)
  } else {
    ETH_PACKED_FWD(64)
  }
#undef ETH_PACKED_FWD
  ETH_CHECK_LAUNCH("eth_packed_attn_fwd");
  return ETH_OK;
}

extern "C" int eth_packed_attn_bwd(const eth_packed_attn_desc_t* d, const void* q, const void* k, const void* v,
                                   const void* out, const void* dout, const float* lse, float* delta, void* dq,
                                   void* dk, void* dv, void* workspace, void* stream) {
  if (int rc = packed_check(d)) return rc;
  ETH_CHECK_ARG(q && k && v && out && dout && lse && delta && dq && dk && dv, "eth_packed_attn_bwd: null pointer");
  ETH_CHECK_ARG(good_strides(q, d->q_strides) && good_strides(k, d->k_strides) && good_strides(v, d->v_strides) &&
                    good_strides(out, d->o_strides) && good_strides(dout, d->do_strides) &&
                    good_strides(dq, d->dq_strides) && good_strides(dk, d->dk_strides) &&
                    good_strides(dv, d->dv_strides),
                "eth_packed_attn_bwd: rows must be 16-byte aligned, strides non-negative and rows below 2^24 apart");
  PackArgs a = packed_args(d);
  a.q = pin(q, d->q_strides);
  a.k = pin(k, d->k_strides);
  a.v = pin(v, d->v_strides);
  a.o = pin(out, d->o_strides);
  a.dout = pin(dout, d->do_strides);
  a.dq = pout(dq, d->dq_strides);
  a.dk = pout(dk, d->dk_strides);
  a.dv = pout(dv, d->dv_strides);
  a.lse = const_cast<float*>(lse);
  a.delta = delta;
  ETH_CHECK_ARG((!a.q_split.tiles && !a.k_split.tiles) || (workspace && ((uintptr_t)workspace & 15) == 0),
                "eth_packed_attn_bwd: split tiles need a 16-byte aligned workspace");
  a.partial = (float4*)workspace;
  const int g_q = (int)grid_of(a.q_split, d->n_q_tiles, a.n / a.hp), g_k = (int)grid_of(a.k_split, d->n_k_tiles, a.m);
  hipStream_t s = (hipStream_t)stream;
  const bool fp16 = d->dtype == ETH_F16;
#define ETH_PACKED_BWD(D)                        \
  if (fp16)                                      \
    launch_packed_bwd<D, true>(a, g_q, g_k, s);  \
  else                                           \
    launch_packed_bwd<D, false>(a, g_q, g_k, s);
  const int width = width_of(a.hd);
  if (width == 128) {
    ETH_PACKED_BWD(128)
  } else if (width == 96) {
    ETH_PACKED_BWD(96)
  } else {
    ETH_PACKED_BWD(64)
  }
#undef ETH_PACKED_BWD
  ETH_CHECK_LAUNCH("eth_packed_attn_bwd");
  return ETH_OK;
}
