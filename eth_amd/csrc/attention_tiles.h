// Building blocks of the causal attention kernels on CDNA4 matrix cores: the
// 32x32x16 MFMA with its operand and result layouts, conversions to and from
// the 16-bit types, and 64-row blocks of a tensor as swizzled images in LDS.
#pragma once

#include <type_traits>

#include "common.h"

namespace eth {

typedef __bf16 a_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 a_f16x8 __attribute__((ext_vector_type(8)));
typedef float a_f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t a_u32x4 __attribute__((ext_vector_type(4)));

template <bool FP16>
__device__ __forceinline__ a_f32x16 mma(const uint4& a, const uint4& b, const a_f32x16& c) {
  if constexpr (FP16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(a_f16x8, a), __builtin_bit_cast(a_f16x8, b),
                                                  c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(a_bf16x8, a),
                                                   __builtin_bit_cast(a_bf16x8, b), c, 0, 0, 0);
}

template <bool FP16>
__device__ __forceinline__ float to_f(uint16_t v) {
  return FP16 ? h2f_bits(v) : bf2f(v);
}
template <bool FP16>
__device__ __forceinline__ uint16_t from_f(float v) {
  return FP16 ? f2h_bits(v) : f2bf(v);
}
template <bool FP16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (FP16)
    return f2h_pair(a, b);
  else
    return f2bf_pair(a, b);
}
__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
// s_waitcnt vmcnt(0) (expcnt, lgkmcnt unconstrained) as the builtin, so the
// compiler's own wait-count tracking knows that no vector load is pending
__device__ __forceinline__ void vm_wait_all() { __builtin_amdgcn_s_waitcnt(0x0F70); }
// Between a wave's LDS accesses of one type and its accesses of another to the
// same memory, all of them its own: its LDS operations execute in order, but
// the compiler may take float, 16-bit and 16-byte accesses to be apart and
// move one past the other.  The clobber holds them in place.
__device__ __forceinline__ void wave_lds_fence() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
// 8 fp32 -> one 16-byte MFMA operand
template <bool FP16>
__device__ __forceinline__ uint4 pack8(const float* v) {
  return make_uint4(pack2<FP16>(v[0], v[1]), pack2<FP16>(v[2], v[3]), pack2<FP16>(v[4], v[5]),
                    pack2<FP16>(v[6], v[7]));
}

__device__ __forceinline__ int swz(int r) {  // swap bits 2 and 3
  return (r & ~12) | ((r & 4) << 1) | ((r & 8) >> 1);
}
// index (within a 32-row MFMA tile) held by accumulator register r of a lane
// in half h, when the operand rows were swizzled
__device__ __forceinline__ int swz_row(int r, int h) { return (r < 8 ? 0 : 16) + h * 8 + (r & 7); }
// natural accumulator row of register r for half h
__device__ __forceinline__ int acc_row(int r, int h) { return (r >> 2) * 8 + h * 4 + (r & 3); }

constexpr int kAttnThreads = 256;
constexpr float kRescaleLog2 = 8.0f;  // forward: tolerated growth of the running max (log2 units)
constexpr int kBQ = 128;   // forward / dQ: queries per workgroup (4 waves x 32)
constexpr int kBKV = 64;   // forward / dQ: keys per step
constexpr int kBKV2 = 128; // dK/dV: keys per workgroup (4 waves x 32)
constexpr int kBQ2 = 64;   // dK/dV: queries per step
constexpr int32_t kAttnOob = (int32_t)0x80000000u;  // buffer offset past any tensor: loads read zeros
// 16 bytes of a row at column `col` of a strided tensor; with PAD, zeros
// past the sequence or the head dim (without, every row and column is real)
template <bool PAD>
__device__ __forceinline__ uint4 load_row16(const uint16_t* row, bool in_seq, int col, int hd) {
  if constexpr (PAD)
    return in_seq && col < hd ? *reinterpret_cast<const uint4*>(row + col) : make_uint4(0u, 0u, 0u, 0u);
  else
    return *reinterpret_cast<const uint4*>(row + col);
}

typedef __amdgpu_buffer_rsrc_t a_rsrc_t;
typedef short a_s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) a_s16x4 a_lds_s16x4;
typedef uint32_t a_u32x2 __attribute__((ext_vector_type(2)));
// ------------------------------------------------------- images in LDS --
// A 64-row block of a tensor lies in LDS as it is in memory, except that chunk
// c (8 columns, 16 bytes) of row r is at c ^ img_swz(r): the row reads of an
// MFMA operand (16 lanes on 16 rows, one chunk) and the transposing
// ds_read_b64_tr_b16 reads (4 rows x 64 bytes per 32 lanes) then both hit
// distinct banks, so one image serves both.  It is filled by direct
// global->LDS loads a whole block ahead: no register staging, no copy phase.
// Each image is an array of its own, so the compiler can tell the loads into
// one from the reads of another and puts no wait between them.
__device__ __forceinline__ int xsw(int r) { return ((r & 3) << 2) | ((r >> 2) & 3); }
template <int D>
__device__ __forceinline__ int img_swz(int r) {
  if constexpr (D == 128)
    return xsw(r);
  else if constexpr (D == 64)  // 128-byte rows: bit 0 of r picks the half of the banks
    return (((r >> 1) & 1) << 2) | (((r >> 3) & 1) << 1) | ((r >> 2) & 1);
  else  // 192-byte rows start 64 bytes apart in the banks: within groups of four chunks
    return (r >> 2) & 3;
}
// Row reads: row t*32 + swz(lane%32) (the swizzled order that makes the
// result's layout the operand layout of the next product), chunk 2*ks + lane/32:
// element offset of k-step ks within a 32-row tile.
template <int D>
__device__ __forceinline__ int img_row_off(int lane, int ks) {
  const int r = swz(lane & 31);
  return r * D + (((2 * ks + (lane >> 5)) ^ img_swz<D>(r)) << 3);
}
// Transposing reads: rows kk*16 + 8*(l/32) + (l%16)/4 (+4 for the second
// read, hi), columns ct*32 + 16*((l/16)%2) + 4*(l%4): element offset within
// the 16-row group kk.
template <int D>
__device__ __forceinline__ int img_tr_off(int lane, int ct, int hi) {
  const int r = 8 * (lane >> 5) + ((lane & 15) >> 2) + 4 * hi;
  const int c = 4 * ct + 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1);
  return r * D + ((c ^ img_swz<D>(r)) << 3) + (lane & 1) * 4;
}
__device__ __forceinline__ uint4 img_tr(const uint16_t* p, int lo_off, int hi_off) {
  const a_u32x2 lo = __builtin_bit_cast(a_u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((a_lds_s16x4*)(p + lo_off)));
  const a_u32x2 hi = __builtin_bit_cast(a_u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((a_lds_s16x4*)(p + hi_off)));
  return make_uint4(lo.x, lo.y, hi.x, hi.y);
}

}  // namespace eth
