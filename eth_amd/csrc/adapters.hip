// Low-rank adapters of many tasks beside a shared projection:
//
//   y = x W^T + bias + s (x A_a^T) B_a^T     a: the row's adapter, s its scale
//
// and with dy:  dx = dy W + s (dy B_a) A_a,  dA_a = sum over a's rows of
// (s dy B_a)^T x,  dB_a = sum of dy^T (s x A_a^T).
//
//   shrink    u = s x A_a^T (backward: s dy B_a) of 32-row tiles of one adapter
//             each, memory-bound on x: the waves of a workgroup share the depth,
//             fragments go from memory to the matrix cores without LDS
//   product   the shared projection's tiles (gemm_tiles.h), whose accumulators
//             start at u B_a^T (backward: u A_a) instead of zero, so y and dx
//             are written once
//   outer     dA and dB: u^T x and dy^T u over chunks of an adapter's tiles, the
//             16-bit values transposed 8 x 8 in registers, memory-bound on x and dy
//   join      an adapter's chunks added in order, rounded once
//
// u is rounded to 16 bits, the matrix cores' operand: with their own rounding dA
// and dB are 1.4 roundings from exact.  It averages over the rows; tiles of up to 16
// rows, half of whose depth in those products is free, hold there what it left.  In
// fp16 a tile's u carries a power of two that puts its largest value at 2^13 to 2^14,
// taken back in fp32 from each tile's products, so that it keeps its digits whatever
// the size of gradients and adapters, and of the tiles beside it.
//
// No counterpart in the reference, whose linear layers (mpu/layers.py:357-370,
// 452-470) have one weight for all rows.
#include <algorithm>

#include "gemm_tiles.h"

namespace eth {

constexpr int kTileRows = ETH_ADAPTER_TILE_ROWS;

// 16 bytes of 8 values, zeros past `r`'s end (offset kOob and beyond)
__device__ __forceinline__ uint4 load8(rsrc_t r, int32_t off) {
  return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
}

// ---------------------------------------------------------------- shrink --
struct ShrinkArgs {
  const eth_adapter_tile_t* tiles;
  const uint16_t* x;  // [rows][ldx], K of it
  const uint16_t* a;  // [adapters][r][K]
  int64_t ldx;
  int K, r, rp;
  uint16_t* u;       // [rows][rp]: rp the rank rounded up to 32, zeros behind it
  float* row_scale;  // [rows] (fp16)
  uint16_t* ut;      // [tile][rp][32], zeros behind the tile's rows (at 16 and on, of up to 16
                     // rows, what their rounding left); or NULL
  float* tile_scale; // [tile] (fp16)
  float* partials;   // [split][tile][32][16 RB]; NULL: the depth is in one piece
  int splits, n_tiles;
};

// A tile's u of its fp32 sums: the scale, the power of two, 16 bits, both layouts.
// sum(row, j): four ranks of a row.  `turned`, `high`: LDS that nothing reads any
// more behind the next barrier.
template <int RB, int W, bool FP16, class F>
__device__ __forceinline__ void narrow(const ShrinkArgs& g, const eth_adapter_tile_t& t, int tile, uint16_t* turned,
                                       float* high, F&& sum) {
  constexpr int CELLS = kTileRows * RB * 4, PER = (CELLS + 64 * W - 1) / (64 * W);  // of four ranks
  constexpr int TS = kTileRows + 8;
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  f32x4_t v[PER];
  float top = 0.f;
#pragma unroll
  for (int c = 0; c < PER; ++c) {
    const int cell = c * 64 * W + (int)threadIdx.x, row = cell / (RB * 4), j = cell % (RB * 4) * 4;
    if (cell >= CELLS) break;
    v[c] = sum(row, j) * t.scale;
    if (FP16)
#pragma unroll
      for (int e = 0; e < 4; ++e) top = __builtin_isfinite(v[c][e]) ? fmaxf(top, fabsf(v[c][e])) : top;
  }
  const bool both = t.rows <= kTileRows / 2;
  float down = 1.f, up = 1.f;  // what the stored u is times, and what brings it back
  if (FP16) {
    top = wave_max(top);
    if (lane == 0) high[wid] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; ++w) top = fmaxf(top, high[w]);
    if (top > 0.f) {
      const int e = max(-100, min(100, ilogbf(top) - 13));
      down = ldexpf(1.f, -e);
      up = ldexpf(1.f, e);
    }
    if (threadIdx.x == 0 && g.ut) g.tile_scale[tile] = up;
    if ((int)threadIdx.x < t.rows) g.row_scale[t.row + threadIdx.x] = up;
  }
  __syncthreads();
#pragma unroll
  for (int c = 0; c < PER; ++c) {
    const int cell = c * 64 * W + (int)threadIdx.x, row = cell / (RB * 4), j = cell % (RB * 4) * 4;
    if (cell >= CELLS) break;
    uint32_t lo, hi;
    if (FP16) {
      lo = f2h_pair(v[c][0] * down, v[c][1] * down);
      hi = f2h_pair(v[c][2] * down, v[c][3] * down);
    } else {
      lo = f2bf_pair(v[c][0], v[c][1]);
      hi = f2bf_pair(v[c][2], v[c][3]);
    }
    if (g.u && row < t.rows && j < g.rp) {
      u32x2_t o = {lo, hi};
      *reinterpret_cast<u32x2_t*>(g.u + (int64_t)(t.row + row) * g.rp + j) = o;
    }
    if (both && row >= kTileRows / 2) continue;
    const uint16_t at[4] = {(uint16_t)lo, (uint16_t)(lo >> 16), (uint16_t)hi, (uint16_t)(hi >> 16)};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      turned[(j + e) * TS + row] = at[e];
      if (!both) continue;
      const float had = FP16 ? v[c][e] * down : v[c][e], is = FP16 ? h2f_bits(at[e]) : bf2f(at[e]);
      const float left = __builtin_isfinite(is) ? had - is : 0.f;
      turned[(j + e) * TS + kTileRows / 2 + row] = FP16 ? f2h_bits(left) : f2bf(left);
    }
  }
  if (RB == 1 && g.u) {  // (rp 32: the second half of a row of 16 ranks)
    for (int c = threadIdx.x; c < kTileRows * 2; c += 64 * W)
      if (c / 2 < t.rows)
        *reinterpret_cast<uint4*>(g.u + (int64_t)(t.row + c / 2) * g.rp + 16 + c % 2 * 8) = make_uint4(0, 0, 0, 0);
  }
  if (!g.ut) return;
  __syncthreads();
  uint16_t* out = g.ut + (int64_t)tile * g.rp * kTileRows;
  for (int c = threadIdx.x; c < g.rp * 4; c += 64 * W) {
    const int j = c / 4, row = c % 4 * 8;
    const uint4 o = j < RB * 16 ? *reinterpret_cast<const uint4*>(turned + j * TS + row) : make_uint4(0, 0, 0, 0);
    *reinterpret_cast<uint4*>(out + j * kTileRows + row) = o;
  }
}

// RB: blocks of 16 ranks; W waves, each with a range of the workgroup's depth: 32
// rows alone would be 32 x r / 256 results a workgroup for a depth of thousands, so
// the depth is what is shared.  Rank 16, [8192, 2048] 14 us, [8192, 8192] 39, 3.4
// TB/s of x; rank 64, [3000, 4096] 9, where every tile reads its adapter's 512 KB.
// Neighbouring workgroups have the pieces of a tile's depth: with eight, each XCD
// reads its own piece of every adapter, which its L2 holds.
// P: tiles of a workgroup, in one pass over the depth where they are one adapter's.
template <int RB, int W, int P, bool FP16>
__global__ void __launch_bounds__(64 * W) adapter_shrink_kernel(ShrinkArgs g) {
  constexpr int RS = RB * 16 + 4;  // padded row of the partial sums
  __shared__ __attribute__((aligned(16))) float red[W][kTileRows][RS];
  __shared__ float high[W];
  const int group = blockIdx.x / g.splits, piece = blockIdx.x - group * g.splits;
  const int lane = threadIdx.x & 63, l16 = lane & 15, lg = lane >> 4;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int pieces = W * g.splits, steps = (g.K + 31) / 32, per = (steps + pieces - 1) / pieces;
  const int s0 = (piece * W + wid) * per, s1 = min(steps, s0 + per);
  // steps whose loads are in flight together, and as many ahead (two at 128 ranks: 1 us
  // more at [3000, 4096] and [8192, 4096])
  constexpr int UN = RB >= 8 ? 1 : RB >= 4 ? 2 : 4;
  const int last = P == 1 ? group + 1 : min(g.n_tiles, (group + 1) * P);
  for (int tile = group * P, many; tile < last; tile += many) {
    eth_adapter_tile_t t[P];
    rsrc_t xs[P];
    t[0] = g.tiles[tile];
    many = 1;
    if (P > 1) {
      t[P - 1] = g.tiles[min(tile + 1, last - 1)];
      if (tile + 1 < last && t[P - 1].adapter == t[0].adapter) many = 2;
    }
    const rsrc_t as = make_rsrc(g.a + (int64_t)t[0].adapter * g.r * g.K, (uint32_t)(g.r * g.K * 2));
    bool live[2 * P];  // blocks of 16 rows
    int32_t xo[2 * P], ao[RB];
    f32x4_t acc[2 * P][RB];
#pragma unroll
    for (int q = 0; q < P; ++q) {
      xs[q] = make_rsrc(g.x + (int64_t)t[q].row * g.ldx, (uint32_t)(((t[q].rows - 1) * g.ldx + g.K) * 2));
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int i = q * 2 + h, row = h * 16 + l16;
        live[i] = q < many && t[q].rows > h * 16;
        xo[i] = live[i] && row < t[q].rows ? (int32_t)((row * g.ldx + lg * 8) * 2) : kOob;
#pragma unroll
        for (int j = 0; j < RB; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      }
    }
#pragma unroll
    for (int j = 0; j < RB; ++j) ao[j] = j * 16 + l16 < g.r ? ((j * 16 + l16) * g.K + lg * 8) * 2 : kOob;
    struct Batch {
      uint4 x[UN][2 * P], a[UN][RB];
    };
    auto load = [&](Batch& f, int s) __attribute__((always_inline)) {
#pragma unroll
      for (int n = 0; n < UN; ++n) {
        // (past this wave's range, or the depth: zeros)
        const bool in = s + n < s1 && (s + n) * 32 + lg * 8 < g.K;
        const int32_t at = (s + n) * 64;
#pragma unroll
        for (int i = 0; i < 2 * P; ++i) f.x[n][i] = load8(xs[i / 2], in && xo[i] != kOob ? xo[i] + at : kOob);
#pragma unroll
        for (int j = 0; j < RB; ++j) f.a[n][j] = load8(as, in && ao[j] != kOob ? ao[j] + at : kOob);
      }
    };
    auto products = [&](const Batch& f) __attribute__((always_inline)) {
#pragma unroll
      for (int n = 0; n < UN; ++n)
#pragma unroll
        for (int i = 0; i < 2 * P; ++i)
          if (i == 0 || live[i]) {
#pragma unroll
            for (int j = 0; j < RB; ++j) acc[i][j] = mfma16<FP16>(f.a[n][j], f.x[n][i], acc[i][j]);
          }
    };
    Batch one, two;
    load(one, s0);
    for (int s = s0; s < s1; s += 2 * UN) {
      load(two, s + UN);
      products(one);
      load(one, s + 2 * UN);
      products(two);
    }
    // the waves' sums, in order
    auto sum = [&](int row, int j) __attribute__((always_inline)) {
      f32x4_t v = *reinterpret_cast<const f32x4_t*>(&red[0][row][j]);
#pragma unroll
      for (int w = 1; w < W; ++w) v += *reinterpret_cast<const f32x4_t*>(&red[w][row][j]);
      return v;
    };
#pragma unroll
    for (int q = 0; q < P; ++q) {
      if (q >= many) break;
      if (P > 1) __syncthreads();  // (the tile before is out)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < RB; ++j)
          *reinterpret_cast<f32x4_t*>(&red[wid][h * 16 + l16][j * 16 + lg * 4]) = acc[q * 2 + h][j];
      __syncthreads();
      if (g.partials) {
        float* out = g.partials + ((int64_t)piece * g.n_tiles + tile + q) * kTileRows * RB * 16;
        for (int cell = threadIdx.x; cell < kTileRows * RB * 4; cell += 64 * W) {
          const int row = cell / (RB * 4), j = cell % (RB * 4) * 4;
          *reinterpret_cast<f32x4_t*>(out + row * RB * 16 + j) = sum(row, j);
        }
      } else {
        narrow<RB, W, FP16>(g, t[q], tile + q, reinterpret_cast<uint16_t*>(&red[0][0][0]), high, sum);
      }
    }
  }
}

// The pieces of the depth joined, in order (4 to 5 us, a launch and its latency).
constexpr int kMaxSplits = 8;
template <int RB, bool FP16>
__global__ void __launch_bounds__(256) adapter_narrow_kernel(ShrinkArgs g) {
  __shared__ __attribute__((aligned(16))) uint16_t turned[RB * 16 * (kTileRows + 8)];
  __shared__ float high[4];
  const float* mine = g.partials + (int64_t)blockIdx.x * kTileRows * RB * 16;
  const int64_t stride = (int64_t)gridDim.x * kTileRows * RB * 16;
  narrow<RB, 4, FP16>(g, g.tiles[blockIdx.x], blockIdx.x, turned, high, [&](int row, int j) __attribute__((always_inline)) {
    const float* at = mine + row * RB * 16 + j;
    f32x4_t in[kMaxSplits];
#pragma unroll
    for (int s = 0; s < kMaxSplits; ++s)
      in[s] = s < g.splits ? *reinterpret_cast<const f32x4_t*>(at + s * stride) : f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 1; s < kMaxSplits; ++s) in[0] += in[s];
    return in[0];
  });
}

// --------------------------------------------------------------- product --
// The accumulators start at u e^T, e [adapters][cols][r] (forward B, backward
// A transposed): for each adapter of the wave's rows (mostly one) the product of
// all its rows, zeros in the place of the others', by fragments from memory (L2):
// r / 32 k-steps of latency ahead of the main loop, whose first loads are under way
// meanwhile.  Rank 16, [8192, 2048 -> 8192]: 217 us for the plain product's 198 (four
// rounds of tiles); rank 64, [3000, 4096 -> 4096]: 91 for 82; eight rows of eight
// adapters, rank 16, [2048 -> 6144]: 13 for 9.
struct AdapterStart {
  static constexpr bool kSized = false, kGathers = false, kStarts = true, kMaps = false, kReduces = false;
  const int* of_row;
  const uint16_t* u;
  const float* row_scale;  // (fp16; NULL else)
  const uint16_t* e;
  int r, rp;

  __device__ __forceinline__ uint4 u_frag(int row, int k, bool there) const {
    return there ? *reinterpret_cast<const uint4*>(u + (int64_t)row * rp + k) : make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ uint4 e_frag(int adapter, int col, int k, int N) const {
    return col < N && k < r ? *reinterpret_cast<const uint4*>(e + ((int64_t)adapter * N + col) * r + k)
                            : make_uint4(0, 0, 0, 0);
  }

  // The products are the kernel's own kind, on accumulators that stay where they
  // are: through the builtin the wide kernel spills 130 to 380 registers, and the
  // ring kernel's accumulators move between its products and the start's.
  template <bool FP16, bool PINNED>
  __device__ __forceinline__ static void mul(f32x4_t& c, const uint4& a, const uint4& b) {
    if constexpr (PINNED)
      mfma16_asm<FP16>(c, a, b);
    else
      mfma16_tied<FP16>(c, a, b);
  }

  // bits 15 and 31: whether one of eight values is an infinity or NaN (one more
  // carries out of an exponent of all ones)
  template <bool FP16>
  __device__ __forceinline__ static uint32_t not_finite(const uint4& v) {
    constexpr uint32_t top = FP16 ? 0x7c007c00u : 0x7f807f80u, one = FP16 ? 0x04000400u : 0x00800080u;
    return ((v.x & top) + one) | ((v.y & top) + one) | ((v.z & top) + one) | ((v.w & top) + one);
  }

  template <int TI>
  struct Early {
    int mine[TI];     // the lane's rows' adapters (-1: none, -2: a row past M)
    float scale[TI];  // (fp16)
  };
  template <int TI>
  __device__ __forceinline__ void ask(Early<TI>& r, int row0, int M) const {
#pragma unroll
    for (int i = 0; i < TI; ++i) {
      const int row = row0 + i * 16 + (threadIdx.x & 15);
      r.mine[i] = row < M ? of_row[row] : -2;
      r.scale[i] = row_scale && row < M ? row_scale[row] : 0.f;
    }
  }

  template <bool FP16, bool PINNED, int TI, int TJ>
  __device__ __forceinline__ void start(f32x4_t (&acc)[TI][TJ], const Early<TI>& early, int row0, int col0, int M,
                                        int N) const {
    const int lane = threadIdx.x & 63, l16 = lane & 15, lg = lane >> 4;
    constexpr int NONE = 0x7fffffff;
    const int(&mine)[TI] = early.mine;
    // whether all rows (but those past M) have one adapter
    const int first = __builtin_amdgcn_readfirstlane(mine[0]);
    bool same = true;
#pragma unroll
    for (int i = 0; i < TI; ++i) same &= mine[i] == first || mine[i] == -2;
    const bool one = __ballot(!same) == 0;
    // the least adapter of the wave's rows above `last` (a row of 16 lanes holds all)
    auto next = [&](int last) __attribute__((always_inline)) {
      int v = NONE;
#pragma unroll
      for (int i = 0; i < TI; ++i) v = mine[i] > last ? min(v, mine[i]) : v;
      v = min(v, __builtin_amdgcn_mov_dpp(v, 0x128, 0xf, 0xf, true));  // row_ror:8
      v = min(v, __builtin_amdgcn_mov_dpp(v, 0x124, 0xf, 0xf, true));  // row_ror:4
      v = min(v, __builtin_amdgcn_mov_dpp(v, 0x4e, 0xf, 0xf, true));   // quad_perm:[2,3,0,1]
      v = min(v, __builtin_amdgcn_mov_dpp(v, 0xb1, 0xf, 0xf, true));   // quad_perm:[1,0,3,2]
      return __builtin_amdgcn_readfirstlane(v);
    };
    // 32 ranks of an adapter at a time, the next ones' fragments under way
    struct Frags {
      uint4 e[TJ], u[TI];
      int a;
    };
    auto load = [&](Frags& f, int a, int k) __attribute__((always_inline)) {
      f.a = a;
      if (a == NONE) return;
#pragma unroll
      for (int j = 0; j < TJ; ++j) f.e[j] = e_frag(a, col0 + j * 16 + l16, k + lg * 8, N);
#pragma unroll
      for (int i = 0; i < TI; ++i) f.u[i] = u_frag(row0 + i * 16 + l16, k + lg * 8, mine[i] == a);
    };
    int a = next(-1), k = 0;
    auto step = [&]() __attribute__((always_inline)) {
      k += 32;
      if (k >= rp) {
        k = 0;
        if (a != NONE) a = next(a);
      }
    };
    auto products = [&](Frags& f) __attribute__((always_inline)) {
      if (!one) {
        // zero times another adapter's infinity or NaN is NaN: where its fragments
        // hold one, zeros take their place, and its own rows become NaN
        uint32_t wild = 0;
#pragma unroll
        for (int j = 0; j < TJ; ++j) wild |= not_finite<FP16>(f.e[j]);
        if (__ballot((wild & 0x80008000u) != 0)) {
#pragma unroll
          for (int j = 0; j < TJ; ++j) f.e[j] = make_uint4(0, 0, 0, 0);
          const uint32_t nan = FP16 ? 0x7e007e00u : 0x7fc07fc0u;
#pragma unroll
          for (int i = 0; i < TI; ++i)
            if (mine[i] == f.a) f.u[i] = make_uint4(nan, nan, nan, nan);
        }
      }
#pragma unroll
      for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int j = 0; j < TJ; ++j) mul<FP16, PINNED>(acc[i][j], f.e[j], f.u[i]);
    };
    // (small tiles, whose rows often have an adapter each, look further ahead)
    constexpr int AHEAD = TI * TJ <= 4 ? 4 : 2;
    Frags f[AHEAD];
#pragma unroll
    for (int d = 0; d < AHEAD; ++d) {
      load(f[d], a, k);
      step();
    }
    while (f[0].a != NONE) {
#pragma unroll
      for (int d = 0; d < AHEAD; ++d) {
        if (f[d].a != NONE) products(f[d]);
        load(f[d], a, k);
        step();
      }
    }
    // asm MFMAs: wait states before anything reads their accumulators
    asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7" ::: "memory");
    if (FP16) {
      // (the products by f stay behind the waits by their operands, not by their
      // place alone)
#pragma unroll
      for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int j = 0; j < TJ; ++j) {
          if constexpr (PINNED)
            asm volatile("" : "+a"(acc[i][j]));
          else
            asm volatile("" : "+v"(acc[i][j]));
        }
#pragma unroll
      for (int i = 0; i < TI; ++i) {
        const float f = mine[i] >= 0 ? early.scale[i] : 0.f;
#pragma unroll
        for (int j = 0; j < TJ; ++j) acc[i][j] *= f;
        if (PINNED) __builtin_amdgcn_sched_barrier(0);  // (a row block at a time: 26 registers spilled else)
      }
    }
  }
};

// ------------------------------------------------------------- transpose --
// rows a (low) and b (high) of column h of two packed pairs
__device__ __forceinline__ uint32_t pair_of(uint32_t a, uint32_t b, int h) {
  return __builtin_amdgcn_perm(b, a, h ? 0x07060302u : 0x05040100u);
}
__device__ __forceinline__ uint32_t word_of(const uint4& v, int w) { return w == 0 ? v.x : w == 1 ? v.y : w == 2 ? v.z : v.w; }
// column f of eight rows of eight 16-bit values
__device__ __forceinline__ uint4 column_of(const uint4 (&row)[8], int f) {
  const int w = f >> 1, h = f & 1;
  return make_uint4(pair_of(word_of(row[0], w), word_of(row[1], w), h), pair_of(word_of(row[2], w), word_of(row[3], w), h),
                    pair_of(word_of(row[4], w), word_of(row[5], w), h), pair_of(word_of(row[6], w), word_of(row[7], w), h));
}

// [adapters][rows][cols] -> [adapters][cols][rows] of the adapters that are in
// use, both multiples of 8: an 8 x 8 block a thread.  (Eight adapters of rank 64,
// 8192 + 2048 long: 8.6 us, 21 MB in and out.)
struct TurnArgs {
  const uint16_t* from;
  uint16_t* to;
  int rows, cols;
};
__global__ void __launch_bounds__(256) adapter_turn_kernel(TurnArgs a, TurnArgs b, const int* used, int a_blocks) {
  int i = blockIdx.x * 256 + threadIdx.x;
  const bool second = i >= a_blocks;
  const TurnArgs t = second ? b : a;
  if (second) i -= a_blocks;
  if (i >= t.rows / 8 * (t.cols / 8)) return;
  // neighbouring threads write side by side
  const int r0 = i % (t.rows / 8) * 8, c0 = i / (t.rows / 8) * 8;
  const int64_t base = (int64_t)used[blockIdx.y] * t.rows * t.cols;
  uint4 row[8];
#pragma unroll
  for (int k = 0; k < 8; ++k)
    row[k] = *reinterpret_cast<const uint4*>(t.from + base + (int64_t)(r0 + k) * t.cols + c0);
#pragma unroll
  for (int f = 0; f < 8; ++f)
    *reinterpret_cast<uint4*>(t.to + base + (int64_t)(c0 + f) * t.rows + r0) = column_of(row, f);
}

// ----------------------------------------------------------------- outer --
// part[chunk][r][C] = sum over the chunk's tiles of u^T q, for dA (q = x) and dB
// (q = dy) in one launch: 128 columns a workgroup, its four waves taking tiles in
// turn.  Rank 16, x [8192, 2048] and dy [8192, 8192]: 30.4 us, 5.5 TB/s; rank 64, 2000
// rows of 8192 and 2048 in a chunk for each of eight adapters: 19.8 us, 640 workgroups
// whose waves have one or two tiles: latency.
struct OuterSide {
  const uint16_t* ut;
  const float* tile_scale;  // (fp16)
  const uint16_t* q;        // [rows][ldq], C of it
  int64_t ldq;
  int C;
  float* part;
};
struct OuterArgs {
  const eth_adapter_tile_t* tiles;
  const eth_adapter_chunk_t* chunks;
  int r, rp;
  OuterSide a, b;
  int a_blocks;  // workgroups along x of side a
};

template <int RB, bool FP16>
__global__ void __launch_bounds__(256) adapter_outer_kernel(OuterArgs args) {
  __shared__ __attribute__((aligned(16))) float sum[RB * 16][128 + 4];
  const bool second = (int)blockIdx.x >= args.a_blocks;
  const OuterSide g = second ? args.b : args.a;
  const int block = second ? blockIdx.x - args.a_blocks : blockIdx.x;
  const eth_adapter_chunk_t c = args.chunks[blockIdx.y];
  const int lane = threadIdx.x & 63, l16 = lane & 15, lg = lane >> 4;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = block * 128 + l16 * 8;
  // acc[j][f]: ranks 16 j + 4 (lane / 16) + 0..3, column col + f
  f32x4_t acc[RB][8];
#pragma unroll
  for (int j = 0; j < RB; ++j)
#pragma unroll
    for (int f = 0; f < 8; ++f) acc[j][f] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  for (int k = wid; k < c.tiles; k += 4) {
    const int at = c.first + k;
    const eth_adapter_tile_t t = args.tiles[at];
    const rsrc_t qs = make_rsrc(g.q + (int64_t)t.row * g.ldq, (uint32_t)(((t.rows - 1) * g.ldq + g.C) * 2));
    uint4 row[8];
    const int r0 = t.rows <= kTileRows / 2 ? lg * 8 % (kTileRows / 2) : lg * 8;  // (16 rows: twice)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      row[i] = load8(qs, r0 + i < t.rows && col < g.C ? (int32_t)(((r0 + i) * g.ldq + col) * 2) : kOob);
    uint4 fu[RB];
    // (zeros past the tile's rp ranks: 72 to 96 ranks are 96 there and 128 here)
    const rsrc_t us = make_rsrc(g.ut + (int64_t)at * args.rp * kTileRows, (uint32_t)(args.rp * kTileRows * 2));
#pragma unroll
    for (int j = 0; j < RB; ++j) fu[j] = load8(us, ((j * 16 + l16) * kTileRows + lg * 8) * 2);
    // (fp16) a tile's products get its power of two in fp32: brought to that of other
    // tiles in u's 16 bits, small tiles beside large ones or zeros lost their digits
    const float scale = FP16 ? g.tile_scale[at] : 1.f;
    // eight rows of eight columns -> a column's eight rows
    f32x4_t had[RB];
#pragma unroll
    for (int f = 0; f < 8; ++f) {
      const uint4 fq = column_of(row, f);
      if (!FP16) {
#pragma unroll
        for (int j = 0; j < RB; ++j) acc[j][f] = mfma16<FP16>(fu[j], fq, acc[j][f]);
        continue;
      }
      f32x4_t now[RB];
#pragma unroll
      for (int j = 0; j < RB; ++j) now[j] = mfma16<FP16>(fu[j], fq, f32x4_t{0.f, 0.f, 0.f, 0.f});
      // (up to 64 ranks a column's products are under way while those of the one before
      // are added, 45.3 -> 43.1 us of rank 64's gradients; above, registers are short:
      // 179 -> 202 us)
      if (RB >= 8) {
#pragma unroll
        for (int j = 0; j < RB; ++j) acc[j][f] += now[j] * scale;
        continue;
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < RB; ++j) {
        if (f) acc[j][f - 1] += had[j] * scale;
        had[j] = now[j];
      }
    }
    if (FP16 && RB < 8) {
#pragma unroll
      for (int j = 0; j < RB; ++j) acc[j][7] += had[j] * scale;
    }
  }
  // the waves' sums, one wave after the other
  for (int w = 0; w < 4; ++w) {
    if (w == wid) {
#pragma unroll
      for (int j = 0; j < RB; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          f32x4_t* s = reinterpret_cast<f32x4_t*>(&sum[j * 16 + lg * 4 + e][l16 * 8]);
          f32x4_t lo = {acc[j][0][e], acc[j][1][e], acc[j][2][e], acc[j][3][e]};
          f32x4_t hi = {acc[j][4][e], acc[j][5][e], acc[j][6][e], acc[j][7][e]};
          if (w) {
            lo += s[0];
            hi += s[1];
          }
          s[0] = lo;
          s[1] = hi;
        }
    }
    __syncthreads();
  }
  float* out = g.part + (int64_t)blockIdx.y * args.r * g.C;
  for (int i = threadIdx.x; i < args.r * 32; i += 256) {
    const int j = i / 32, q = i % 32 * 4, at = block * 128 + q;
    if (at < g.C)
      *reinterpret_cast<f32x4_t*>(out + (int64_t)j * g.C + at) = *reinterpret_cast<const f32x4_t*>(&sum[j][q]);
  }
}

// ------------------------------------------------------------------ join --
// An adapter's gradient: its chunks added in order; zeros where it has none (4.1 us
// at rank 16 of 4 adapters of 2048 + 8192, 6.4 at rank 64 of 8).
// dA [adapters][r][K] is stored as summed, dB [adapters][N][r] turned: a thread
// has eight ranks of a column.
struct JoinSide {
  const float* part;
  int C;
  void* out;
  int fp32, accumulate, turned;
};
struct JoinArgs {
  const int* first_chunk;  // [listed + 1]
  int listed;              // adapters from there on have none
  int r, dtype;
  JoinSide a, b;
  int a_blocks;
};
__device__ __forceinline__ void put8(void* out, int64_t at, int fp32, int accumulate, int dtype, const float (&v)[8]) {
  if (fp32) {
    float4* o = reinterpret_cast<float4*>(reinterpret_cast<float*>(out) + at);
    float4 a = make_float4(v[0], v[1], v[2], v[3]), b = make_float4(v[4], v[5], v[6], v[7]);
    if (accumulate) {
      const float4 p = o[0], q = o[1];
      a.x += p.x; a.y += p.y; a.z += p.z; a.w += p.w;
      b.x += q.x; b.y += q.y; b.z += q.z; b.w += q.w;
    }
    o[0] = a;
    o[1] = b;
    return;
  }
  uint32_t w[4];
#pragma unroll
  for (int k = 0; k < 4; ++k)
    w[k] = dtype == ETH_F16 ? f2h_pair(v[2 * k], v[2 * k + 1]) : f2bf_pair(v[2 * k], v[2 * k + 1]);
  *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(out) + at) = make_uint4(w[0], w[1], w[2], w[3]);
}
__global__ void __launch_bounds__(256) adapter_join_kernel(JoinArgs args) {
  const bool second = (int)blockIdx.x >= args.a_blocks;
  const JoinSide g = second ? args.b : args.a;
  const int r = args.r, a = blockIdx.y, i = (second ? blockIdx.x - args.a_blocks : blockIdx.x) * 256 + threadIdx.x;
  if (i >= r / 8 * g.C) return;
  const int c0 = a < args.listed ? args.first_chunk[a] : 0, c1 = a < args.listed ? args.first_chunk[a + 1] : 0;
  float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  const int64_t chunk = (int64_t)r * g.C;
  if (g.turned) {
    const int j = i / g.C * 8, col = i % g.C;
    for (int c = c0; c < c1; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += g.part[c * chunk + (int64_t)(j + e) * g.C + col];
    put8(g.out, (int64_t)a * chunk + (int64_t)col * r + j, g.fp32, g.accumulate, args.dtype, v);
  } else {
    for (int c = c0; c < c1; ++c) {
      const float4* p = reinterpret_cast<const float4*>(g.part + c * chunk + (int64_t)i * 8);
      const float4 x = p[0], y = p[1];
      v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w;
      v[4] += y.x; v[5] += y.y; v[6] += y.z; v[7] += y.w;
    }
    put8(g.out, (int64_t)a * chunk + (int64_t)i * 8, g.fp32, g.accumulate, args.dtype, v);
  }
}

// ------------------------------------------------------------------ host --
static int64_t room(int64_t bytes) { return (bytes + 255) / 256 * 256; }
static int padded_rank(int64_t r) { return (int)((r + 31) / 32 * 32); }

// How the product [M, N] x K deep runs: its tile, or 256x256 tiles in several
// splits of K joined by a second kernel, by the rules of the plain products.
struct ProductPlan {
  int tile, splits;
  int64_t workspace;
};
static ProductPlan plan_product(int64_t M, int64_t N, int64_t K, int b_kcontig) {
  ProductPlan p{0, 1, 0};
  const GemmForm form = gemm_form(M, N, K, 1, b_kcontig, false);
  p.tile = plan_tile(M, N, K, wide_takes(M, N, N, 2, true), form);
  const int64_t tiles = (M + 255) / 256 * ((N + 255) / 256);
  int splits = 1;
  while (tiles <= 128 && splits < 16 && tiles * splits * 2 <= 256 && K / (splits * 2) >= 1024) splits *= 2;
  if (splits > 1 && 4 * (M + 256) * N < (1LL << 31) &&
      eth_gemm_splitk_pays(M, N, K, splits, 1, b_kcontig, ETH_BF16)) {
    p.tile = 256;
    p.splits = splits;
    p.workspace = eth_gemm_splitk_workspace(M, N, splits);
  }
  return p;
}

template <bool B_K, bool FP16, class X>
static int launch_adapted(const ProductPlan& p, GemmArgs a, const X& x, float* partials, hipStream_t s) {
  if (p.splits > 1) {
    GemmArgs d = a;
    d.C = partials;
    d.bias = nullptr;
    d.flags = 0;
    d.ldc = a.N;
    d.c_dtype = ETH_F32;
    d.c_bytes = (uint32_t)((int64_t)a.M * a.N * 4);
    d.k_split = (int)(((a.K + p.splits - 1) / p.splits + 63) / 64 * 64);
    d.c_split_stride = (int64_t)a.M * a.N;
    const int splits = (a.K + d.k_split - 1) / d.k_split;
    const int tiles = ((a.M + 255) / 256) * ((a.N + 255) / 256) * splits;
    if (a.K % 64)
      gemm256_m16_kernel<true, B_K, FP16, true, X><<<tiles, 256, 0, s>>>(d, x);
    else
      gemm256_m16_kernel<true, B_K, FP16, false, X><<<tiles, 256, 0, s>>>(d, x);
    ETH_CHECK_LAUNCH("eth_adapter_linear");
    const SplitSum sum{partials, splits, d.c_split_stride, a.C, a.ldc, a.bias, a.M, a.N, a.c_dtype, 0, 1.f};
    const int64_t quads = (int64_t)a.M * (a.N / 4);
    splitk_sum_kernel<FP16><<<(int)std::min<int64_t>((quads + 255) / 256, 2048), 256, 0, s>>>(sum);
    ETH_CHECK_LAUNCH("eth_adapter_linear");
    return ETH_OK;
  }
  const int tiles = ((a.M + p.tile - 1) / p.tile) * ((a.N + p.tile - 1) / p.tile);
  if (p.tile == 256) {
    if (a.K % 64)
      gemm256_m16_kernel<true, B_K, FP16, true, X><<<tiles, 256, 0, s>>>(a, x);
    else
      gemm256_m16_kernel<true, B_K, FP16, false, X><<<tiles, 256, 0, s>>>(a, x);
  } else if (p.tile == 128) {
    gemm_ring_kernel<128, true, B_K, FP16, X><<<tiles, 256, 0, s>>>(a, x);
  } else {
    gemm_ring_kernel<64, true, B_K, FP16, X><<<tiles, 256, 0, s>>>(a, x);
  }
  ETH_CHECK_LAUNCH("eth_adapter_linear");
  return ETH_OK;
}

// From this many tiles on, and 33 ranks, a workgroup of the shrink takes two: their
// adapter's values, which L2 hands out again for every tile, serve both.  One / two
// (us, the adapters' share of a forward call): [16384, 4096] rank 128 78 / 54, rank 64
// 48 / 36, [8192, 4096] rank 128 42 / 37, rank 64 26 / 27.  Of short segments pairs are
// often of two adapters, taken one after the other: [3000, 4096] of four of rank 64
// 14 / 21.
constexpr int kPairedTiles = 128;

// Pieces of the shrink's depth: as many as bring three workgroups a compute unit
// (one from 33 ranks on, where every workgroup reads its adapter's values anew), each
// of two trips of its waves at least; a depth of fewer than eight trips, 2048 at rank
// 16, is not worth the second launch (3 us of the host).  One workgroup / two (us, the adapters' share
// of a forward call): [16384, 4096] rank 128 54 / 65, rank 64 36 / 48, [8192, 4096] 27
// / 28, [2000, 8192] 25 / 26; below 33 ranks two / three / four: [8192, 8192] rank 16 46
// / 39 / 37, [16384, 4096] rank 16 26 / 26 / 30, rank 32 33 / 33 / 37.  Four waves a
// workgroup: with eight, whose sums meet in twice the LDS, [500, 4096] rank 64 took 12.8
// for 9.9, [2000, 2048] 13.5 for 11.3, [8192, 8192] rank 16 41 for 37 ([3000, 4096]
// rank 16 11.5 for 12.6).
constexpr int kShrinkWaves = 4;
struct ShrinkPlan {
  int blocks, splits, pairs;
  int64_t workspace;
};
static ShrinkPlan plan_shrink(int64_t K, int r, int n_tiles) {
  ShrinkPlan p{r <= 16 ? 1 : r <= 32 ? 2 : r <= 64 ? 4 : 8, 1, 0, 0};
  p.pairs = p.blocks >= 4 && n_tiles >= kPairedTiles;
  const int groups = p.pairs ? (n_tiles + 1) / 2 : n_tiles;
  const int64_t trips = K / (kShrinkWaves * 32 * (p.blocks >= 4 ? 2 : 4)), slots = p.blocks >= 4 ? 256 : 768;
  if (n_tiles && trips >= 8) p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(kMaxSplits, slots / groups), trips / 2));
  if (p.splits > 1) p.workspace = (int64_t)p.splits * n_tiles * kTileRows * p.blocks * 16 * 4;
  return p;
}
template <bool FP16>
static int launch_shrink(ShrinkArgs g, int n_tiles, float* partials, hipStream_t s) {
  const ShrinkPlan p = plan_shrink(g.K, g.r, n_tiles);
  g.partials = p.splits > 1 ? partials : nullptr;
  g.splits = p.splits;
  g.n_tiles = n_tiles;
  const unsigned grid = (unsigned)((p.pairs ? (n_tiles + 1) / 2 : n_tiles) * p.splits);
#define ETH_SHRINK(RB, P)                                                                   \
  {                                                                                         \
    adapter_shrink_kernel<RB, kShrinkWaves, P, FP16><<<grid, 64 * kShrinkWaves, 0, s>>>(g); \
    ETH_CHECK_LAUNCH("eth_adapter_linear");                                                 \
    if (p.splits > 1) adapter_narrow_kernel<RB, FP16><<<n_tiles, 256, 0, s>>>(g);           \
  }
  if (p.blocks == 1) ETH_SHRINK(1, 1)
  else if (p.blocks == 2) ETH_SHRINK(2, 1)
  else if (p.blocks == 4 && p.pairs) ETH_SHRINK(4, 2)
  else if (p.blocks == 4) ETH_SHRINK(4, 1)
  else if (p.pairs) ETH_SHRINK(8, 2)
  else ETH_SHRINK(8, 1)
#undef ETH_SHRINK
  ETH_CHECK_LAUNCH("eth_adapter_linear");
  return ETH_OK;
}

template <bool FP16>
static int launch_outer(const OuterArgs& g, int n_chunks, hipStream_t s) {
  const dim3 grid((unsigned)(g.a_blocks + (g.b.C + 127) / 128), (unsigned)n_chunks);
#define ETH_OUTER(RB) adapter_outer_kernel<RB, FP16><<<grid, 256, 0, s>>>(g)
  if (g.r <= 16) ETH_OUTER(1);
  else if (g.r <= 32) ETH_OUTER(2);
  else if (g.r <= 64) ETH_OUTER(4);
  else ETH_OUTER(8);
#undef ETH_OUTER
  ETH_CHECK_LAUNCH("eth_adapter_linear_bwd");
  return ETH_OK;
}

static int check_adapter(const char* name, const eth_adapter_desc_t* d) {
  ETH_CHECK_ARG(d, "%s: null descriptor", name);
  ETH_CHECK_ARG(d->dtype == ETH_BF16 || d->dtype == ETH_F16, "%s: dtype must be bf16 or fp16", name);
  const int64_t M = d->rows, N = d->out, K = d->in;
  ETH_CHECK_ARG(M > 0 && N > 0 && K > 0 && N % 8 == 0 && K % 8 == 0 && M < (1LL << 31) && N < (1LL << 31) &&
                    K < (1LL << 31),
                "%s: bad shape: %lld rows, %lld in, %lld out (multiples of 8)", name, (long long)M, (long long)K,
                (long long)N);
  ETH_CHECK_ARG(d->rank >= 8 && d->rank <= 128 && d->rank % 8 == 0, "%s: the rank must be a multiple of 8 up to 128 (got %d)",
                name, d->rank);
  ETH_CHECK_ARG(d->ldx >= K && d->ldw >= K && d->ldx % 8 == 0 && d->ldw % 8 == 0,
                "%s: row strides must be multiples of 8", name);
  ETH_CHECK_ARG(d->adapters > 0 && d->n_tiles >= 0 && d->n_chunks >= 0 && d->n_chunks < 65536 && d->n_used >= 0 &&
                    d->n_used <= d->n_listed && d->n_listed <= d->adapters && d->adapters < 65536 && d->n_tiles < (1 << 23) &&
                    (d->n_tiles > 0) == (d->n_chunks > 0) && (d->n_tiles > 0) == (d->n_used > 0),
                "%s: bad lists", name);
  ETH_CHECK_ARG(!d->n_tiles || (d->tiles && d->chunks && d->of_row && d->used && d->first_chunk), "%s: null list", name);
  ETH_CHECK_ARG(((M - 1) * d->ldx + K) * 2 < (1LL << 31) && ((N - 1) * d->ldw + K) * 2 < (1LL << 31) &&
                    M * N * 2 < (1LL << 31) && M * K * 2 < (1LL << 31) && (int64_t)d->rank * std::max(K, N) * 2 < (1LL << 31),
                "%s: operands above 2 GiB are not supported", name);
  return ETH_OK;
}

struct AdapterForward {
  int64_t u, row_scale, product, bytes;
  ProductPlan plan;
};
static AdapterForward plan_adapter_fwd(const eth_adapter_desc_t* d) {
  AdapterForward p;
  p.plan = plan_product(d->rows, d->out, d->in, 1);
  int64_t o = 0;
  p.u = o, o += room(d->rows * padded_rank(d->rank) * 2);
  p.row_scale = o, o += room(d->rows * 4);
  // (the shrink's partial sums, then the product's)
  p.product = o, o += room(std::max(p.plan.workspace, plan_shrink(d->in, d->rank, d->n_tiles).workspace));
  p.bytes = o;
  return p;
}
struct AdapterBackward {
  int64_t u, row_scale, ut, tile_scale, at, bt, part_a, part_b, product, bytes;
  ProductPlan plan;
};
static AdapterBackward plan_adapter_bwd(const eth_adapter_desc_t* d) {
  AdapterBackward p;
  p.plan = plan_product(d->rows, d->in, d->out, 0);
  const int rp = padded_rank(d->rank);
  int64_t o = 0;
  p.u = o, o += room(d->rows * rp * 2);
  p.row_scale = o, o += room(d->rows * 4);
  p.ut = o, o += room((int64_t)d->n_tiles * rp * kTileRows * 2);
  p.tile_scale = o, o += room((int64_t)d->n_tiles * 4);
  p.at = o, o += room((int64_t)d->adapters * d->rank * d->in * 2);
  p.bt = o, o += room((int64_t)d->adapters * d->rank * d->out * 2);
  // the shrink's partial sums, the product's, then dA's and dB's chunks: each is
  // read before the next is written
  p.product = o;
  p.part_a = o;
  p.part_b = o + room((int64_t)d->n_chunks * d->rank * d->in * 4);
  o += std::max({room(p.plan.workspace), room(plan_shrink(d->out, d->rank, d->n_tiles).workspace),
                 p.part_b - o + room((int64_t)d->n_chunks * d->rank * d->out * 4)});
  p.bytes = o;
  return p;
}

static GemmArgs adapter_product(const eth_adapter_desc_t* d, const void* A, int64_t lda, int64_t a_cols, const void* B,
                                void* C, int64_t N, const void* bias) {
  GemmArgs a{};
  a.A = (const uint16_t*)A;
  a.B = (const uint16_t*)B;
  a.a_bytes = (uint32_t)(((d->rows - 1) * lda + a_cols) * 2);
  a.b_bytes = (uint32_t)(((d->out - 1) * d->ldw + d->in) * 2);
  a.C = C;
  a.bias = (const uint16_t*)bias;
  a.M = (int)d->rows;
  a.N = (int)N;
  a.K = (int)a_cols;
  a.lda = lda;
  a.ldb = d->ldw;
  a.ldc = N;
  a.c_dtype = d->dtype;
  a.flags = bias ? ETH_GEMM_BIAS : 0;
  a.alpha = 1.f;
  a.c_vec = true;
  a.c_bytes = (uint32_t)(d->rows * N * 2);
  return a;
}

template <bool FP16>
static int adapter_forward(const eth_adapter_desc_t* d, const void* x, const void* w, const void* bias,
                           const void* lora_a, const void* lora_b, void* y, void* ut, float* tile_scale, char* ws,
                           hipStream_t s) {
  const AdapterForward p = plan_adapter_fwd(d);
  const int rp = padded_rank(d->rank);
  const GemmArgs a = adapter_product(d, x, d->ldx, d->in, w, y, d->out, bias);
  if (!d->n_tiles) return launch_adapted<true, FP16>(p.plan, a, PlainProduct{}, (float*)(ws + p.product), s);
  const ShrinkArgs g{d->tiles, (const uint16_t*)x, (const uint16_t*)lora_a, d->ldx, (int)d->in, d->rank, rp,
                     (uint16_t*)(ws + p.u), (float*)(ws + p.row_scale), (uint16_t*)ut, tile_scale, nullptr, 1, 0};
  const int rc = launch_shrink<FP16>(g, d->n_tiles, (float*)(ws + p.product), s);
  if (rc != ETH_OK) return rc;
  const AdapterStart start{d->of_row, g.u, FP16 ? g.row_scale : nullptr, (const uint16_t*)lora_b, d->rank, rp};
  return launch_adapted<true, FP16>(p.plan, a, start, (float*)(ws + p.product), s);
}

template <bool FP16>
static int adapter_backward(const eth_adapter_desc_t* d, const void* x, const void* w, const void* lora_a,
                            const void* lora_b, const void* dy, const void* ut, const float* tile_scale, void* dx,
                            const eth_adapter_grad_t* da, const eth_adapter_grad_t* db, char* ws, hipStream_t s) {
  const AdapterBackward p = plan_adapter_bwd(d);
  const int rp = padded_rank(d->rank);
  int rc = ETH_OK;
  GemmArgs a = adapter_product(d, dy, d->out, d->out, w, dx, d->in, nullptr);
  if (!d->n_tiles) {
    if (dx) rc = launch_adapted<false, FP16>(p.plan, a, PlainProduct{}, (float*)(ws + p.product), s);
    if (rc != ETH_OK) return rc;
  }
  if (d->n_tiles && (dx || da->grad)) {
    // A^T for the start of dx, B^T for u
    const TurnArgs turn_a{(const uint16_t*)lora_a, (uint16_t*)(ws + p.at), d->rank, (int)d->in};
    const TurnArgs turn_b{(const uint16_t*)lora_b, (uint16_t*)(ws + p.bt), (int)d->out, d->rank};
    const int a_blocks = dx ? d->rank / 8 * (int)(d->in / 8) : 0, b_blocks = d->rank / 8 * (int)(d->out / 8);
    adapter_turn_kernel<<<dim3((unsigned)((a_blocks + b_blocks + 255) / 256), (unsigned)d->n_used), 256, 0, s>>>(
        turn_a, turn_b, d->used, a_blocks);
    ETH_CHECK_LAUNCH("eth_adapter_linear_bwd");
    const ShrinkArgs g{d->tiles, (const uint16_t*)dy, turn_b.to, d->out, (int)d->out, d->rank, rp,
                       (uint16_t*)(dx ? ws + p.u : nullptr), (float*)(ws + p.row_scale),
                       (uint16_t*)(da->grad ? ws + p.ut : nullptr), (float*)(ws + p.tile_scale), nullptr, 1, 0};
    rc = launch_shrink<FP16>(g, d->n_tiles, (float*)(ws + p.product), s);
    if (rc != ETH_OK) return rc;
    if (dx) {
      const AdapterStart start{d->of_row, g.u, FP16 ? g.row_scale : nullptr, turn_a.to, d->rank, rp};
      rc = launch_adapted<false, FP16>(p.plan, a, start, (float*)(ws + p.product), s);
      if (rc != ETH_OK) return rc;
    }
  }
  const OuterSide none{};
  if (d->n_tiles && (da->grad || db->grad)) {
    OuterArgs g{d->tiles, d->chunks, d->rank, rp, none, none, 0};
    if (da->grad) {
      g.a = OuterSide{(const uint16_t*)(ws + p.ut), (const float*)(ws + p.tile_scale), (const uint16_t*)x, d->ldx,
                      (int)d->in, (float*)(ws + p.part_a)};
      g.a_blocks = (int)((d->in + 127) / 128);
    }
    if (db->grad)
      g.b = OuterSide{(const uint16_t*)ut, tile_scale, (const uint16_t*)dy, d->out, (int)d->out,
                      (float*)(ws + p.part_b)};
    rc = launch_outer<FP16>(g, d->n_chunks, s);
    if (rc != ETH_OK) return rc;
  }
  // (without rows, what is added to stays as it is)
  const bool join_a = da->grad && (d->n_tiles || !da->accumulate), join_b = db->grad && (d->n_tiles || !db->accumulate);
  if (join_a || join_b) {
    const int64_t a_blocks = join_a ? (d->rank / 8 * d->in + 255) / 256 : 0;
    const int64_t b_blocks = join_b ? (d->rank / 8 * d->out + 255) / 256 : 0;
    const JoinSide a{(const float*)(ws + p.part_a), (int)d->in, da->grad, da->fp32, da->accumulate, 0};
    const JoinSide b{(const float*)(ws + p.part_b), (int)d->out, db->grad, db->fp32, db->accumulate, 1};
    const JoinArgs j{d->first_chunk, d->n_tiles ? d->n_listed : 0, d->rank, d->dtype, a, b, (int)a_blocks};
    adapter_join_kernel<<<dim3((unsigned)(a_blocks + b_blocks), (unsigned)d->adapters), 256, 0, s>>>(j);
    ETH_CHECK_LAUNCH("eth_adapter_linear_bwd");
  }
  return ETH_OK;
}

}  // namespace eth

using namespace eth;

extern "C" int64_t eth_adapter_linear_workspace(const eth_adapter_desc_t* desc, int backward) {
  if (check_adapter("eth_adapter_linear_workspace", desc) != ETH_OK) return -1;
  return backward ? plan_adapter_bwd(desc).bytes : plan_adapter_fwd(desc).bytes;
}

extern "C" int eth_adapter_linear_fwd(const eth_adapter_desc_t* desc, const void* x, const void* w, const void* bias,
                                      const void* lora_a, const void* lora_b, void* y, void* ut, float* tile_scale,
                                      void* workspace, void* stream) {
  const int rc = check_adapter("eth_adapter_linear_fwd", desc);
  if (rc != ETH_OK) return rc;
  ETH_CHECK_ARG(x && w && lora_a && lora_b && y && workspace && (!ut || desc->dtype != ETH_F16 || tile_scale),
                "eth_adapter_linear_fwd: null operand");
  ETH_CHECK_ARG((((uintptr_t)x | (uintptr_t)w | (uintptr_t)lora_a | (uintptr_t)lora_b | (uintptr_t)y | (uintptr_t)ut) &
                 15u) == 0 && ((uintptr_t)workspace & 255) == 0,
                "eth_adapter_linear_fwd: operands must be 16-byte, the workspace 256-byte aligned");
  return desc->dtype == ETH_F16
             ? adapter_forward<true>(desc, x, w, bias, lora_a, lora_b, y, ut, tile_scale, (char*)workspace,
                                     (hipStream_t)stream)
             : adapter_forward<false>(desc, x, w, bias, lora_a, lora_b, y, ut, tile_scale, (char*)workspace,
                                      (hipStream_t)stream);
}

extern "C" int eth_adapter_linear_bwd(const eth_adapter_desc_t* desc, const void* x, const void* w, const void* lora_a,
                                      const void* lora_b, const void* dy, const void* ut, const float* tile_scale,
                                      void* dx, const eth_adapter_grad_t* da, const eth_adapter_grad_t* db,
                                      void* workspace, void* stream) {
  const int rc = check_adapter("eth_adapter_linear_bwd", desc);
  if (rc != ETH_OK) return rc;
  ETH_CHECK_ARG(x && w && lora_a && lora_b && dy && da && db && workspace, "eth_adapter_linear_bwd: null operand");
  ETH_CHECK_ARG(dx || da->grad || db->grad, "eth_adapter_linear_bwd: nothing to compute");
  ETH_CHECK_ARG(!db->grad || !desc->n_tiles || (ut && (desc->dtype != ETH_F16 || tile_scale)),
                "eth_adapter_linear_bwd: dB needs what the forward saved");
  ETH_CHECK_ARG((((uintptr_t)x | (uintptr_t)w | (uintptr_t)lora_a | (uintptr_t)lora_b | (uintptr_t)dy | (uintptr_t)ut |
                  (uintptr_t)dx | (uintptr_t)da->grad | (uintptr_t)db->grad) & 15u) == 0 &&
                    ((uintptr_t)workspace & 255) == 0,
                "eth_adapter_linear_bwd: operands must be 16-byte, the workspace 256-byte aligned");
  ETH_CHECK_ARG(!da->grad || da->grad != db->grad, "eth_adapter_linear_bwd: dA and dB in one place");
  for (const eth_adapter_grad_t* t : {da, db})
    ETH_CHECK_ARG(!t->accumulate || t->fp32, "eth_adapter_linear_bwd: accumulate needs an fp32 gradient");
  return desc->dtype == ETH_F16
             ? adapter_backward<true>(desc, x, w, lora_a, lora_b, dy, ut, tile_scale, dx, da, db, (char*)workspace,
                                      (hipStream_t)stream)
             : adapter_backward<false>(desc, x, w, lora_a, lora_b, dy, ut, tile_scale, dx, da, db, (char*)workspace,
                                       (hipStream_t)stream);
}
