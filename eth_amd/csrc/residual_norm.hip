// The norm behind a block, its gate, the scaled residual and the norm before
// the next block in one pass over the rows, forward and backward:
//
//   n = (x - mu1) r1 post_gamma + post_beta        the block's output, normed
//   h = residual_scale residual + gate n           the residual stream, stored in 16 bits
//   y = (h - mu2) r2 gamma + beta                  of h before that rounding
//
// (root-mean-square norms: mu = 0, r = 1 / sqrt(mean of squares + eps), no
// betas).  With D the gradient of h, from h's own consumers and through y,
//
//   D  = dh + r2 (dy gamma - mean(dy gamma) - hhat mean(dy gamma hhat))
//   dresidual = residual_scale D
//   dx = r1 (u - mean(u) - xhat mean(u xhat)),  u = D gate post_gamma
//   S1 = sum D xhat, S2 = sum D, S3 = sum dy hhat, S4 = sum dy  over the rows:
//   dpost_gamma = gate S1, dpost_beta = gate S2, dgate = post_gamma S1 +
//   post_beta S2, dgamma = S3, dbeta = S4.
//
// The backward makes h again from x and the residual, with the forward's
// operations, rather than read the rounded one: the same bytes, and h's rounding is
// in no other result (read back, it took every result's error from 1 to 1.4
// roundings, and to more where few rows or columns average it).
//
// Memory bounds it: 8 bytes an element forward (x and residual in, h and y
// out), 12 backward (x, residual, dh, dy in, dx, dresidual out).
//
// Beside the bias-dropout-add and LayerNorm of model/flex_ops.py:104-134 and
// model/fused_layer_norm.py:62-89; no counterpart in the reference.
#include "common.h"

// Only the fused multiply-adds that are written are fused, so the backward's h is
// the forward's, bit for bit.
#pragma clang fp contract(off)

namespace eth {

constexpr int kRnMaxCols = 8192;
constexpr int kRnWaves = 4;     // rows of a forward workgroup

template <bool FP16>
__device__ __forceinline__ float rn_in(uint16_t v) {
  return FP16 ? h2f_bits(v) : bf2f(v);
}
template <bool FP16>
__device__ __forceinline__ uint16_t rn_out(float v) {
  return FP16 ? f2h_bits(v) : f2bf(v);
}
typedef uint32_t rn_u32x4 __attribute__((ext_vector_type(4)));
typedef float rn_f32x4 __attribute__((ext_vector_type(4)));
template <bool FP16>
__device__ __forceinline__ float rn_at(const rn_u32x4& v, int j) {
  const uint32_t w = v[j >> 1];
  return rn_in<FP16>((uint16_t)((j & 1) ? (w >> 16) : (w & 0xffffu)));
}
// a row of cols 16-bit elements: vectors past its end, and rows that are not
// `live`, read as zeros and are not stored
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rn_row(const uint16_t* base, int64_t row, int cols, bool live) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(base + (live ? row * cols : 0)), (short)0,
                                           live ? cols * 2 : 0, 0x00020000);
}
__device__ __forceinline__ rn_u32x4 rn_load(__amdgpu_buffer_rsrc_t r, int off) {
  return __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0);
}

struct RnParams {
  const uint16_t *post_gamma, *post_beta, *gate, *gamma, *beta;  // betas NULL: rms; gate may be NULL (one)
  float scale, eps;
  int rows, cols, rms;
};

// stats [4][rows]: mu1, r1, mu2, r2

// h of an element of x and of the residual
template <bool FP16>
__device__ __forceinline__ float rn_stream(float x, float mu, float r, float gamma, float beta, float gate, float scale,
                                           float res) {
  return __builtin_fmaf(gate, __builtin_fmaf((x - mu) * r, gamma, beta), scale * res);
}

// One wave a row, NV vectors of 8 a lane, all of the row's loads in flight at once and
// nothing read twice: no barrier, sums by lane moves.  [8192, 2048] 24.5 us, 5.5 TB/s;
// [4096, 4096] 27.8, 4.8; [16384, 1024] 22.7, 5.9; [2048, 8192] 27.4, 4.9.
template <int NV, bool FP16>
__global__ void __launch_bounds__(64 * kRnWaves) rn_fwd_kernel(RnParams g, const uint16_t* __restrict__ x,
                                                               const uint16_t* __restrict__ res,
                                                               uint16_t* __restrict__ h, uint16_t* __restrict__ y,
                                                               float* __restrict__ stats) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * kRnWaves + (threadIdx.x >> 6);
  if (row >= g.rows) return;
  const int cols = g.cols;
  const bool rms = g.rms;
  const __amdgpu_buffer_rsrc_t xr = rn_row(x, row, cols, true), rr = rn_row(res, row, cols, true);
  rn_u32x4 x16[NV], r16[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) x16[i] = rn_load(xr, (i * 64 + lane) * 16);
#pragma unroll
  for (int i = 0; i < NV; ++i) r16[i] = rn_load(rr, (i * 64 + lane) * 16);
  // (columns past the row's end are zeros, and count as such in the sums)
  float v[NV][8];
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[i][j] = rn_at<FP16>(x16[i], j);
      s += v[i][j];
    }
  auto deviation = [&](float mu) __attribute__((always_inline)) {
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if ((i * 64 + lane) * 8 < cols) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float d = v[i][j] - mu;
          q = __builtin_fmaf(d, d, q);
        }
      }
    return rsqrtf(wave_sum(q) / cols + g.eps);
  };
  const float mu1 = rms ? 0.f : wave_sum(s) / cols;
  const float r1 = deviation(mu1);
  const __amdgpu_buffer_rsrc_t pg = rn_row(g.post_gamma, 0, cols, true), pb = rn_row(g.post_beta, 0, cols, !rms),
                               gt = rn_row(g.gate, 0, cols, g.gate), ho = rn_row(h, row, cols, true);
  s = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int off = (i * 64 + lane) * 16;
    const rn_u32x4 ga = rn_load(pg, off), be = rn_load(pb, off), gv = rn_load(gt, off);
    rn_u32x4 o;
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      float t[2];
#pragma unroll
      for (int k = 0; k < 2; ++k)
        t[k] = rn_stream<FP16>(v[i][j + k], mu1, r1, rn_at<FP16>(ga, j + k), rn_at<FP16>(be, j + k),
                               g.gate ? rn_at<FP16>(gv, j + k) : 1.f, g.scale, rn_at<FP16>(r16[i], j + k));
      o[j >> 1] = FP16 ? f2h_pair(t[0], t[1]) : f2bf_pair(t[0], t[1]);
#pragma unroll
      for (int k = 0; k < 2; ++k) v[i][j + k] = t[k];
    }
    __builtin_amdgcn_raw_buffer_store_b128(o, ho, off, 0, 0);
    const bool in = off < cols * 2;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[i][j] = in ? v[i][j] : 0.f;
      s += v[i][j];
    }
  }
  const float mu2 = rms ? 0.f : wave_sum(s) / cols;
  const float r2 = deviation(mu2);
  const __amdgpu_buffer_rsrc_t g2 = rn_row(g.gamma, 0, cols, true), b2 = rn_row(g.beta, 0, cols, !rms),
                               yo = rn_row(y, row, cols, true);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int off = (i * 64 + lane) * 16;
    const rn_u32x4 ga = rn_load(g2, off), be = rn_load(b2, off);
    rn_u32x4 o;
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      float t[2];
#pragma unroll
      for (int k = 0; k < 2; ++k)
        t[k] = __builtin_fmaf((v[i][j + k] - mu2) * r2, rn_at<FP16>(ga, j + k), rn_at<FP16>(be, j + k));
      o[j >> 1] = FP16 ? f2h_pair(t[0], t[1]) : f2bf_pair(t[0], t[1]);
    }
    __builtin_amdgcn_raw_buffer_store_b128(o, yo, off, 0, 0);
  }
  if (lane == 0) {
    stats[row] = mu1;
    stats[g.rows + row] = r1;
    stats[2 * (int64_t)g.rows + row] = mu2;
    stats[3 * (int64_t)g.rows + row] = r2;
  }
}

// Backward.  As in the LayerNorm backward, T waves share a row (a team), NVW
// vectors of 512 columns each; a workgroup's W / T teams walk the rows g, g + G, ...,
// the next row's loads are issued while one is computed, and column sums stay in
// registers for all of a workgroup's rows.  Both norms' row sums meet in LDS, one
// barrier each.  [8192, 2048] 42.6 us, 4.7 TB/s; [3001, 5120] 49.5, 3.7: a team of ten
// waves fills a compute unit's registers, and its two barriers a row show; the
// gradients of the parameters behind it 6.4 and 10.2 us.
template <int W, int T, int NVW, bool FP16>
__global__ void __launch_bounds__(64 * W) rn_bwd_kernel(
    RnParams p, const uint16_t* __restrict__ x, const uint16_t* __restrict__ res, const float* __restrict__ stats,
    const uint16_t* __restrict__ dh, const uint16_t* __restrict__ dy, uint16_t* __restrict__ dx,
    uint16_t* __restrict__ dres, float* __restrict__ part) {
  constexpr int TEAMS = W / T;
  const int lane = threadIdx.x & 63;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int team = wid / T, sub = wid - team * T;
  const int cols = p.cols, rows = p.rows;
  const bool rms = p.rms;
  const int voff = ((sub * NVW) * 64 + lane) * 16;
  rn_u32x4 pg16[NVW], pb16[NVW], gt16[NVW], g216[NVW];
  float acc[4][NVW][8];
  {
    const __amdgpu_buffer_rsrc_t a = rn_row(p.post_gamma, 0, cols, true), b = rn_row(p.gate, 0, cols, p.gate),
                                 c = rn_row(p.gamma, 0, cols, true), e = rn_row(p.post_beta, 0, cols, !rms);
#pragma unroll
    for (int i = 0; i < NVW; ++i) {
      pg16[i] = rn_load(a, voff + i * 1024);
      pb16[i] = rn_load(e, voff + i * 1024);
      gt16[i] = rn_load(b, voff + i * 1024);
      g216[i] = rn_load(c, voff + i * 1024);
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[q][i][j] = 0.f;
    }
  }
  const int G = gridDim.x, g = blockIdx.x;
  const int nrows = (rows - g + G - 1) / G;
  const int iters = (nrows + TEAMS - 1) / TEAMS;  // equal for every wave of the workgroup
  const float inv_n = 1.0f / cols;
  __shared__ float rsum[2][2][W][2];  // [norm][row parity]

  rn_u32x4 nx[NVW], nr[NVW], nd[NVW], ny[NVW];
  auto load_row = [&](int k) __attribute__((always_inline)) {
    const bool live = k < nrows;
    const int64_t r = g + (int64_t)k * G;
    const __amdgpu_buffer_rsrc_t xr = rn_row(x, r, cols, live), rr = rn_row(res, r, cols, live),
                                 dr = rn_row(dh, r, cols, live && dh), yr = rn_row(dy, r, cols, live && dy);
#pragma unroll
    for (int i = 0; i < NVW; ++i) {
      nx[i] = rn_load(xr, voff + i * 1024);
      nr[i] = rn_load(rr, voff + i * 1024);
    }
#pragma unroll
    for (int i = 0; i < NVW; ++i) {
      ny[i] = rn_load(yr, voff + i * 1024);
      nd[i] = rn_load(dr, voff + i * 1024);
    }
  };
  // the team's sums of (a, b), in a fixed order
  auto team_sums = [&](float& a, float& b, int norm, int it) __attribute__((always_inline)) {
    a = wave_sum(a);
    b = wave_sum(b);
    if (T > 1) {
      if (lane == 0) {
        rsum[norm][it & 1][wid][0] = a;
        rsum[norm][it & 1][wid][1] = b;
      }
      __syncthreads();
      a = b = 0.f;
#pragma unroll
      for (int t = 0; t < T; ++t) {
        a += rsum[norm][it & 1][team * T + t][0];
        b += rsum[norm][it & 1][team * T + t][1];
      }
    }
  };
  load_row(team);
  for (int it = 0; it < iters; ++it) {
    const int k = it * TEAMS + team;
    const int64_t r = g + (int64_t)k * G;
    const bool valid = k < nrows;
    rn_u32x4 cx[NVW], cr[NVW], cd[NVW], cy[NVW];
#pragma unroll
    for (int i = 0; i < NVW; ++i) {
      cx[i] = nx[i];
      cr[i] = nr[i];
      cd[i] = nd[i];
      cy[i] = ny[i];
    }
    const float mu1 = valid ? stats[r] : 0.f, r1 = valid ? stats[rows + r] : 0.f;
    const float mu2 = valid ? stats[2LL * rows + r] : 0.f, r2 = valid ? stats[3LL * rows + r] : 0.f;
    if (it + 1 < iters) load_row(k + TEAMS);
    float hhat[NVW][8];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < NVW; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float dv = rn_at<FP16>(cy[i], j);
        const float h = rn_stream<FP16>(rn_at<FP16>(cx[i], j), mu1, r1, rn_at<FP16>(pg16[i], j), rn_at<FP16>(pb16[i], j),
                                        p.gate ? rn_at<FP16>(gt16[i], j) : 1.f, p.scale, rn_at<FP16>(cr[i], j));
        const float hh = hhat[i][j] = (h - mu2) * r2;
        const float dg = dv * rn_at<FP16>(g216[i], j);
        s1 += dg;
        s2 = __builtin_fmaf(dg, hh, s2);
        acc[2][i][j] = __builtin_fmaf(dv, hh, acc[2][i][j]);
        acc[3][i][j] += dv;
      }
    team_sums(s1, s2, 0, it);
    if (rms) s1 = 0.f;
    // the packed values are converted again: kept in fp32 across the sums they
    // would not fit the registers
#pragma unroll
    for (int i = 0; i < NVW; ++i) {
      asm volatile("" : "+v"(cx[i]), "+v"(cy[i]));
      asm volatile("" : "+v"(g216[i]), "+v"(gt16[i]), "+v"(pg16[i]));
    }
    float d[NVW][8];
    float t1 = 0.f, t2 = 0.f;
#pragma unroll
    for (int i = 0; i < NVW; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float dv = rn_at<FP16>(cy[i], j);
        const float hh = hhat[i][j];
        const float through = r2 * __builtin_fmaf(-inv_n, __builtin_fmaf(hh, s2, s1), dv * rn_at<FP16>(g216[i], j));
        d[i][j] = rn_at<FP16>(cd[i], j) + through;
        const float xh = (rn_at<FP16>(cx[i], j) - mu1) * r1;
        const float u = d[i][j] * (p.gate ? rn_at<FP16>(gt16[i], j) : 1.f) * rn_at<FP16>(pg16[i], j);
        t1 += u;
        t2 = __builtin_fmaf(u, xh, t2);
      }
    if (valid) {
      // (columns past the row's end, whose hhat is not zero, meet nothing: their
      // gamma and dy are zeros, D there is of no column)
#pragma unroll
      for (int i = 0; i < NVW; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float xh = (rn_at<FP16>(cx[i], j) - mu1) * r1;
          acc[0][i][j] = __builtin_fmaf(d[i][j], xh, acc[0][i][j]);
          acc[1][i][j] += d[i][j];
        }
      if (dres) {
        const __amdgpu_buffer_rsrc_t orow = rn_row(dres, r, cols, true);
#pragma unroll
        for (int i = 0; i < NVW; ++i) {
          rn_u32x4 o;
#pragma unroll
          for (int j = 0; j < 8; j += 2)
            o[j >> 1] = FP16 ? f2h_pair(p.scale * d[i][j], p.scale * d[i][j + 1])
                             : f2bf_pair(p.scale * d[i][j], p.scale * d[i][j + 1]);
          __builtin_amdgcn_raw_buffer_store_b128(o, orow, voff + i * 1024, 0, 0);
        }
      }
    }
    team_sums(t1, t2, 1, it);
    if (rms) t1 = 0.f;
#pragma unroll
    for (int i = 0; i < NVW; ++i) {
      asm volatile("" : "+v"(cx[i]));
      asm volatile("" : "+v"(gt16[i]), "+v"(pg16[i]));
    }
    if (valid && dx) {
      const __amdgpu_buffer_rsrc_t orow = rn_row(dx, r, cols, true);
#pragma unroll
      for (int i = 0; i < NVW; ++i) {
        rn_u32x4 o;
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          float v[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float xh = (rn_at<FP16>(cx[i], j + e) - mu1) * r1;
            const float u =
                d[i][j + e] * (p.gate ? rn_at<FP16>(gt16[i], j + e) : 1.f) * rn_at<FP16>(pg16[i], j + e);
            v[e] = r1 * __builtin_fmaf(-inv_n, __builtin_fmaf(xh, t2, t1), u);
          }
          o[j >> 1] = FP16 ? f2h_pair(v[0], v[1]) : f2bf_pair(v[0], v[1]);
        }
        __builtin_amdgcn_raw_buffer_store_b128(o, orow, voff + i * 1024, 0, 0);
      }
    }
  }
  // the teams' column sums, added in a fixed order: part[g][4][cols]
  __shared__ float red[W][512];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    float* dst = part + ((int64_t)blockIdx.x * 4 + q) * cols;
#pragma unroll
    for (int i = 0; i < NVW; ++i) {
      __syncthreads();
      rn_f32x4* rw = reinterpret_cast<rn_f32x4*>(&red[wid][lane * 8]);
      rw[0] = rn_f32x4{acc[q][i][0], acc[q][i][1], acc[q][i][2], acc[q][i][3]};
      rw[1] = rn_f32x4{acc[q][i][4], acc[q][i][5], acc[q][i][6], acc[q][i][7]};
      __syncthreads();
      for (int n = threadIdx.x; n < T * 512; n += 64 * W) {
        const int k = n / 512, e = n % 512, c = (k * NVW + i) * 512 + e;  // a column of sub k's vectors
        if (c < cols) {
          float a = 0.f;
#pragma unroll
          for (int t = 0; t < TEAMS; ++t) a += red[t * T + k][e];
          dst[c] = a;
        }
      }
    }
  }
}

// The parameters' gradients of the workgroups' column sums, added in a fixed
// order: 16 columns and all four sums a workgroup, 16 threads a column quad and
// sum.
struct RnGrads {
  eth_residual_norm_grad_t post_gamma, post_beta, gate, gamma, beta;
};
__device__ __forceinline__ void rn_put(const eth_residual_norm_grad_t& t, int c, int dtype, float v) {
  if (!t.grad) return;
  if (t.fp32) {
    float* o = reinterpret_cast<float*>(t.grad) + c;
    *o = t.accumulate ? *o + v : v;
  } else {
    store_elem(t.grad, c, dtype, v);
  }
}
constexpr int kRnGradCols = 16;
__global__ void __launch_bounds__(256) rn_grads_kernel(RnParams p, const float* __restrict__ part, int groups,
                                                       RnGrads out, int dtype) {
  __shared__ rn_f32x4 red[16][4][4];
  const int quad = threadIdx.x & 3, q = (threadIdx.x >> 2) & 3, lane = threadIdx.x >> 4;
  const int c = blockIdx.x * kRnGradCols + quad * 4;
  rn_f32x4 v = {0.f, 0.f, 0.f, 0.f};
  if (c < p.cols) {
    const float* mine = part + (int64_t)q * p.cols + c;
    for (int g = lane; g < groups; g += 16 * 8) {
      rn_f32x4 in[8];
#pragma unroll
      for (int u = 0; u < 8; ++u)
        in[u] = g + u * 16 < groups ? *reinterpret_cast<const rn_f32x4*>(mine + (int64_t)(g + u * 16) * 4 * p.cols)
                                    : rn_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int u = 0; u < 8; ++u) v += in[u];
    }
  }
  red[lane][q][quad] = v;
  for (int half = 8; half; half >>= 1) {
    __syncthreads();
    if (lane < half) red[lane][q][quad] += red[lane + half][q][quad];
  }
  __syncthreads();
  const int col = blockIdx.x * kRnGradCols + (int)threadIdx.x;
  if (threadIdx.x < kRnGradCols && col < p.cols) {
    float s[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) s[k] = red[0][k][threadIdx.x >> 2][threadIdx.x & 3];
    const float gate = p.gate ? load_elem(p.gate, col, dtype) : 1.f;
    const float pg = load_elem(p.post_gamma, col, dtype), pb = p.post_beta ? load_elem(p.post_beta, col, dtype) : 0.f;
    rn_put(out.post_gamma, col, dtype, gate * s[0]);
    rn_put(out.post_beta, col, dtype, gate * s[1]);
    rn_put(out.gate, col, dtype, __builtin_fmaf(pg, s[0], pb * s[1]));
    rn_put(out.gamma, col, dtype, s[2]);
    rn_put(out.beta, col, dtype, s[3]);
  }
}

// Waves of a workgroup, waves that share a row, and vectors of 512 columns a wave
// has of it: a vector a wave and as many rows as 16 waves take, but two vectors and
// one wave for 513 to 1024 columns, which need no barrier (us, gradients of the
// parameters included, two vectors a wave / one: [16384, 1024] 42.2 / 44.6, [8192,
// 2048] 46.8 / 45.2, [4096, 4096] 49.8 / 47.1, [3001, 5120] 60.9 / 52.2).
struct RnShape {
  int waves, team, vectors;
};
inline RnShape rn_shape(int64_t cols) {
  if (cols > 512 && cols <= 1024) return {8, 1, 2};
  const int team = (int)((cols + 511) / 512);
  return {team == 1 ? 8 : 16 / team * team, team, 1};
}
// at most a workgroup a compute unit, each with a row for every team
inline int rn_groups(int64_t rows, int64_t cols) {
  const RnShape f = rn_shape(cols);
  const int64_t teams = f.waves / f.team, g = (rows + teams - 1) / teams;
  return (int)(g > 256 ? 256 : g < 1 ? 1 : g);
}

template <bool FP16>
static void launch_rn_fwd(const RnParams& p, const uint16_t* x, const uint16_t* res, uint16_t* h, uint16_t* y,
                          float* stats, hipStream_t s) {
  const unsigned grid = (unsigned)((p.rows + kRnWaves - 1) / kRnWaves);
  switch ((p.cols + 511) / 512) {
#define ETH_RN_CASE(N) \
  case N: rn_fwd_kernel<N, FP16><<<grid, 64 * kRnWaves, 0, s>>>(p, x, res, h, y, stats); break;
    ETH_RN_CASE(1) ETH_RN_CASE(2) ETH_RN_CASE(3) ETH_RN_CASE(4) ETH_RN_CASE(5) ETH_RN_CASE(6)
    ETH_RN_CASE(7) ETH_RN_CASE(8) ETH_RN_CASE(9) ETH_RN_CASE(10) ETH_RN_CASE(11) ETH_RN_CASE(12)
    ETH_RN_CASE(13) ETH_RN_CASE(14) ETH_RN_CASE(15) ETH_RN_CASE(16)
#undef ETH_RN_CASE
  }
}

template <bool FP16>
static void launch_rn_bwd(const RnParams& p, int groups, const uint16_t* x, const uint16_t* res, const float* stats,
                          const uint16_t* dh, const uint16_t* dy, uint16_t* dx, uint16_t* dres, float* part,
                          hipStream_t s) {
  const RnShape f = rn_shape(p.cols);
#define ETH_RN_BWD(W, T, N)                                                                        \
  case T * 10 + N:                                                                                 \
    rn_bwd_kernel<W, T, N, FP16><<<groups, 64 * W, 0, s>>>(p, x, res, stats, dh, dy, dx, dres, part); \
    break;
  switch (f.team * 10 + f.vectors) {
    ETH_RN_BWD(8, 1, 1) ETH_RN_BWD(8, 1, 2) ETH_RN_BWD(15, 3, 1) ETH_RN_BWD(16, 4, 1) ETH_RN_BWD(15, 5, 1)
    ETH_RN_BWD(12, 6, 1) ETH_RN_BWD(14, 7, 1) ETH_RN_BWD(16, 8, 1) ETH_RN_BWD(9, 9, 1) ETH_RN_BWD(10, 10, 1)
    ETH_RN_BWD(11, 11, 1) ETH_RN_BWD(12, 12, 1) ETH_RN_BWD(13, 13, 1) ETH_RN_BWD(14, 14, 1) ETH_RN_BWD(15, 15, 1)
    ETH_RN_BWD(16, 16, 1)
  }
#undef ETH_RN_BWD
}

static int check_rn(const char* name, const eth_residual_norm_desc_t* d) {
  ETH_CHECK_ARG(d, "%s: null descriptor", name);
  ETH_CHECK_ARG(d->dtype == ETH_BF16 || d->dtype == ETH_F16, "%s: dtype must be bf16 or fp16", name);
  // (a grid of 2^32 threads and more is taken modulo 2^32: 64 threads a row, rounded up to four rows)
  ETH_CHECK_ARG(d->rows >= 0 && d->rows <= (1LL << 26) - 4 && d->cols > 0 && d->cols <= kRnMaxCols && d->cols % 8 == 0,
                "%s: cols must be a positive multiple of 8 up to %d, rows up to 2^26 - 4 (got %lld, %lld)", name, kRnMaxCols,
                (long long)d->cols, (long long)d->rows);
  ETH_CHECK_ARG(d->post_gamma && d->gamma && (d->rms ? !d->post_beta && !d->beta : d->post_beta && d->beta),
                "%s: gammas are needed, and betas exactly where the norms are not root-mean-square", name);
  ETH_CHECK_ARG((((uintptr_t)d->post_gamma | (uintptr_t)d->post_beta | (uintptr_t)d->gate | (uintptr_t)d->gamma |
                  (uintptr_t)d->beta) & 15u) == 0, "%s: parameters must be 16-byte aligned", name);
  ETH_CHECK_ARG(d->eps >= 0.f && d->eps < 1e30f && d->residual_scale > -1e30f && d->residual_scale < 1e30f,
                "%s: eps must be finite and not negative, the residual scale finite", name);
  return ETH_OK;
}
static RnParams rn_params(const eth_residual_norm_desc_t* d) {
  return RnParams{(const uint16_t*)d->post_gamma, (const uint16_t*)d->post_beta, (const uint16_t*)d->gate,
                  (const uint16_t*)d->gamma, (const uint16_t*)d->beta, d->residual_scale, d->eps, (int)d->rows,
                  (int)d->cols, d->rms};
}

}  // namespace eth

using namespace eth;

extern "C" int eth_residual_norm_fwd(const eth_residual_norm_desc_t* desc, const void* x, const void* residual, void* h,
                                     void* y, float* stats, void* stream) {
  const int rc = check_rn("eth_residual_norm_fwd", desc);
  if (rc != ETH_OK) return rc;
  if (desc->rows == 0) return ETH_OK;
  ETH_CHECK_ARG(x && residual && h && y && stats, "eth_residual_norm_fwd: null pointer");
  ETH_CHECK_ARG((((uintptr_t)x | (uintptr_t)residual | (uintptr_t)h | (uintptr_t)y) & 15u) == 0,
                "eth_residual_norm_fwd: operands must be 16-byte aligned");
  const RnParams p = rn_params(desc);
  hipStream_t s = (hipStream_t)stream;
  if (desc->dtype == ETH_F16)
    launch_rn_fwd<true>(p, (const uint16_t*)x, (const uint16_t*)residual, (uint16_t*)h, (uint16_t*)y, stats, s);
  else
    launch_rn_fwd<false>(p, (const uint16_t*)x, (const uint16_t*)residual, (uint16_t*)h, (uint16_t*)y, stats, s);
  ETH_CHECK_LAUNCH("eth_residual_norm_fwd");
  return ETH_OK;
}

extern "C" int64_t eth_residual_norm_workspace(int64_t rows, int64_t cols) {
  return rows > 0 && cols > 0 ? (int64_t)rn_groups(rows, cols) * 4 * cols : 0;
}

extern "C" int eth_residual_norm_bwd(const eth_residual_norm_desc_t* desc, const void* x, const void* residual,
                                     const float* stats, const void* dh, const void* dy, void* dx, void* dresidual,
                                     const eth_residual_norm_grad_t* grads, float* workspace, void* stream) {
  const int rc = check_rn("eth_residual_norm_bwd", desc);
  if (rc != ETH_OK) return rc;
  if (desc->rows == 0) return ETH_OK;
  ETH_CHECK_ARG(x && residual && stats && (dh || dy) && grads && workspace, "eth_residual_norm_bwd: null pointer");
  ETH_CHECK_ARG((((uintptr_t)x | (uintptr_t)residual | (uintptr_t)dh | (uintptr_t)dy | (uintptr_t)dx | (uintptr_t)dresidual |
                  (uintptr_t)workspace) & 15u) == 0, "eth_residual_norm_bwd: operands must be 16-byte aligned");
  ETH_CHECK_ARG((desc->gate || !grads[2].grad) && (!desc->rms || (!grads[1].grad && !grads[4].grad)),
                "eth_residual_norm_bwd: a gradient of a parameter that is not there");
  for (int i = 0; i < 5; ++i) {
    ETH_CHECK_ARG(!grads[i].accumulate || grads[i].fp32, "eth_residual_norm_bwd: accumulate needs an fp32 gradient");
    ETH_CHECK_ARG((uintptr_t)grads[i].grad % (grads[i].fp32 ? 4 : 2) == 0, "eth_residual_norm_bwd: gradient alignment");
    for (int j = 0; j < i; ++j)
      ETH_CHECK_ARG(!grads[i].grad || grads[i].grad != grads[j].grad,
                    "eth_residual_norm_bwd: two parameters' gradients in one place");
  }
  const RnParams p = rn_params(desc);
  const int groups = rn_groups(desc->rows, desc->cols);
  hipStream_t s = (hipStream_t)stream;
  if (desc->dtype == ETH_F16)
    launch_rn_bwd<true>(p, groups, (const uint16_t*)x, (const uint16_t*)residual, stats, (const uint16_t*)dh,
                        (const uint16_t*)dy, (uint16_t*)dx, (uint16_t*)dresidual, workspace, s);
  else
    launch_rn_bwd<false>(p, groups, (const uint16_t*)x, (const uint16_t*)residual, stats, (const uint16_t*)dh,
                         (const uint16_t*)dy, (uint16_t*)dx, (uint16_t*)dresidual, workspace, s);
  ETH_CHECK_LAUNCH("eth_residual_norm_bwd");
  bool any = false;
  for (int i = 0; i < 5; ++i) any |= grads[i].grad != nullptr;
  if (any) {
    rn_grads_kernel<<<(unsigned)((desc->cols + kRnGradCols - 1) / kRnGradCols), 256, 0, s>>>(
        p, workspace, groups, RnGrads{grads[0], grads[1], grads[2], grads[3], grads[4]}, desc->dtype);
    ETH_CHECK_LAUNCH("eth_residual_norm_bwd gradients");
  }
  return ETH_OK;
}
