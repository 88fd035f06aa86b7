// The plain products over the tiles of gemm_tiles.h: C (+)= alpha A B (+ bias)
// in one or two launches, and split-K.
#include "gemm_tiles.h"

namespace eth {

static int launch_planned(const GemmArgs& a, int a_k, int b_k, bool fp16, bool wide, GemmForm form, hipStream_t s) {
  switch (plan_tile(a.M, a.N, a.K, wide, form)) {
    case 256:
      return fp16 ? launch_256<true>(a, a_k, b_k, s) : launch_256<false>(a, a_k, b_k, s);
    case 128:
      return fp16 ? launch_ring<128, true>(a, a_k, b_k, s) : launch_ring<128, false>(a, a_k, b_k, s);
    default:
      return fp16 ? launch_ring<64, true>(a, a_k, b_k, s) : launch_ring<64, false>(a, a_k, b_k, s);
  }
}

}  // namespace eth

using namespace eth;

extern "C" int eth_gemm(const void* A, int64_t lda, int a_kcontig, const void* B, int64_t ldb,
                        int b_kcontig, void* C, int64_t ldc, int c_dtype, const void* bias,
                        int64_t M, int64_t N, int64_t K, int in_dtype, int flags, float alpha,
                        void* stream) {
  ETH_CHECK_ARG(in_dtype == ETH_BF16 || in_dtype == ETH_F16, "eth_gemm: inputs must be bf16 or fp16");
  ETH_CHECK_ARG(valid_dtype(c_dtype), "eth_gemm: bad output dtype %d", c_dtype);
  ETH_CHECK_ARG(M > 0 && N > 0 && K > 0 && M < (1LL << 31) && N < (1LL << 31) && K < (1LL << 31),
                "eth_gemm: bad shape %lld x %lld x %lld", (long long)M, (long long)N, (long long)K);
  ETH_CHECK_ARG(A && B && C, "eth_gemm: null operand");
  ETH_CHECK_ARG(K % 8 == 0, "eth_gemm: K (%lld) must be a multiple of 8", (long long)K);
  ETH_CHECK_ARG(lda % 8 == 0 && ldb % 8 == 0, "eth_gemm: lda/ldb must be multiples of 8");
  ETH_CHECK_ARG(((uintptr_t)A & 15) == 0 && ((uintptr_t)B & 15) == 0, "eth_gemm: A/B must be 16-byte aligned");
  ETH_CHECK_ARG(a_kcontig ? lda >= K : (M % 8 == 0 && lda >= M), "eth_gemm: bad A layout");
  ETH_CHECK_ARG(b_kcontig ? ldb >= K : (N % 8 == 0 && ldb >= N), "eth_gemm: bad B layout");
  ETH_CHECK_ARG(ldc >= N, "eth_gemm: ldc < N");
  ETH_CHECK_ARG(!(flags & ETH_GEMM_ACCUMULATE) || c_dtype == ETH_F32, "eth_gemm: accumulate needs fp32 C");
  ETH_CHECK_ARG(!(flags & ETH_GEMM_BIAS) || bias, "eth_gemm: bias flag without bias");
  // extents: A spans M rows of lda (K-contiguous) or K rows of lda; same for B
  const int64_t a_elems = a_kcontig ? (M - 1) * lda + K : (K - 1) * lda + M;
  const int64_t b_elems = b_kcontig ? (N - 1) * ldb + K : (K - 1) * ldb + N;
  ETH_CHECK_ARG(a_elems * 2 < (1LL << 31) && b_elems * 2 < (1LL << 31),
                "eth_gemm: operands above 2 GiB are not supported");
  GemmArgs a;
  a.A = (const uint16_t*)A;
  a.B = (const uint16_t*)B;
  a.a_bytes = (uint32_t)(a_elems * 2);
  a.b_bytes = (uint32_t)(b_elems * 2);
  a.C = C;
  a.bias = (const uint16_t*)bias;
  a.M = (int)M;
  a.N = (int)N;
  a.K = (int)K;
  a.lda = lda;
  a.ldb = ldb;
  a.ldc = ldc;
  a.c_dtype = c_dtype;
  a.flags = flags;
  a.alpha = alpha;
  hipStream_t s = (hipStream_t)stream;
  const int esz = c_dtype == ETH_F32 ? 4 : 2;
  a.c_vec = ldc % 4 == 0 && N % 4 == 0 && ((uintptr_t)C % (4 * esz)) == 0;
  a.k_split = 0;
  a.c_split_stride = 0;
  const bool wide = wide_takes(M, N, ldc, esz, a.c_vec);
  a.c_bytes = wide ? (uint32_t)(((M - 1) * ldc + N) * esz) : 0;
  const bool fp16 = in_dtype == ETH_F16;
  const GemmForm form = gemm_form(M, N, K, a_kcontig, b_kcontig, c_dtype == ETH_F32);
  const GemmCut cut = plan_cut(M, N, K, wide, form);
  if (cut.m == M && cut.n == N) return launch_planned(a, a_kcontig, b_kcontig, fp16, wide, form, s);
  // the part of whole rounds, then the rest (rows or columns of C)
  const int64_t M2 = M - cut.m, N2 = N - cut.n;
  GemmArgs r = a;
  if (M2) {
    a.M = (int)cut.m;
    a.a_bytes = (uint32_t)((a_kcontig ? (cut.m - 1) * lda + K : (K - 1) * lda + cut.m) * 2);
    a.c_bytes = (uint32_t)(((cut.m - 1) * ldc + N) * esz);
    r.M = (int)M2;
    r.A += a_kcontig ? cut.m * lda : cut.m;
    r.a_bytes = (uint32_t)((a_kcontig ? (M2 - 1) * lda + K : (K - 1) * lda + M2) * 2);
    r.C = (char*)C + cut.m * ldc * esz;
    r.c_bytes = (uint32_t)(((M2 - 1) * ldc + N) * esz);
  } else {
    a.N = (int)cut.n;
    a.b_bytes = (uint32_t)((b_kcontig ? (cut.n - 1) * ldb + K : (K - 1) * ldb + cut.n) * 2);
    a.c_bytes = (uint32_t)(((M - 1) * ldc + cut.n) * esz);
    r.N = (int)N2;
    r.B += b_kcontig ? cut.n * ldb : cut.n;
    r.b_bytes = (uint32_t)((b_kcontig ? (N2 - 1) * ldb + K : (K - 1) * ldb + N2) * 2);
    r.C = (char*)C + cut.n * esz;
    if (r.bias) r.bias += cut.n;
    r.c_bytes = (uint32_t)(((M - 1) * ldc + N2) * esz);
  }
  const int rc = launch_planned(a, a_kcontig, b_kcontig, fp16, wide, form, s);
  return rc != ETH_OK ? rc : launch_planned(r, a_kcontig, b_kcontig, fp16, wide, form, s);
}

extern "C" int eth_gemm_plan(int64_t M, int64_t N, int64_t K, int a_kcontig, int b_kcontig, int64_t ldc, int c_dtype,
                             int64_t* plan) {
  ETH_CHECK_ARG(plan, "eth_gemm_plan: null pointer");
  ETH_CHECK_ARG(valid_dtype(c_dtype), "eth_gemm_plan: bad output dtype %d", c_dtype);
  ETH_CHECK_ARG(M > 0 && N > 0 && K > 0 && M < (1LL << 31) && N < (1LL << 31) && K < (1LL << 31) && ldc >= N,
                "eth_gemm_plan: bad shape %lld x %lld x %lld", (long long)M, (long long)N, (long long)K);
  const bool wide = wide_takes(M, N, ldc, c_dtype == ETH_F32 ? 4 : 2, ldc % 4 == 0 && N % 4 == 0);
  const GemmForm form = gemm_form(M, N, K, a_kcontig, b_kcontig, c_dtype == ETH_F32);
  const GemmCut cut = plan_cut(M, N, K, wide, form);
  plan[0] = plan_tile(cut.m, cut.n, K, wide, form);
  plan[1] = cut.m;
  plan[2] = cut.n;
  const int64_t m = cut.m < M ? M - cut.m : M, n = cut.n < N ? N - cut.n : N;
  plan[3] = cut.m == M && cut.n == N ? 0 : plan_tile(m, n, K, wide, form);
  return ETH_OK;
}

extern "C" int64_t eth_gemm_splitk_workspace(int64_t M, int64_t N, int splits) {
  return splits > 0 && M > 0 && N > 0 ? (int64_t)splits * M * N * 4 : 0;
}

extern "C" int64_t eth_gemm_splitk_pays(int64_t M, int64_t N, int64_t K, int splits, int a_kcontig, int b_kcontig,
                                        int c_dtype) {
  if (M <= 0 || N <= 0 || K <= 0 || splits < 2) return 0;
  // the second kernel: a launch, and the partials (and an fp32 C) at 4.3 TB/s
  const double sum = 4.5 + 4.0 * (double)M * (double)N * (splits + (c_dtype == ETH_F32 ? 1 : 0)) / 4.3e6;
  const GemmForm form = gemm_form(M, N, K, a_kcontig, b_kcontig, c_dtype == ETH_F32);
  const double one = tile_time(plan_tile(M, N, K, true, form), M, N, K, 1, form);
  return tile_time(256, M, N, K, splits, form) + sum < one;
}

extern "C" int eth_gemm_splitk_out(const void* A, int64_t lda, int a_kcontig, const void* B, int64_t ldb,
                                   int b_kcontig, void* C, int64_t ldc, int c_dtype, const void* bias, int64_t M,
                                   int64_t N, int64_t K, int in_dtype, int flags, float alpha, int splits,
                                   float* workspace, void* stream) {
  ETH_CHECK_ARG(in_dtype == ETH_BF16 || in_dtype == ETH_F16, "eth_gemm_splitk: inputs must be bf16 or fp16");
  ETH_CHECK_ARG(valid_dtype(c_dtype), "eth_gemm_splitk: bad output dtype %d", c_dtype);
  ETH_CHECK_ARG(A && B && C && workspace, "eth_gemm_splitk: null operand");
  ETH_CHECK_ARG(splits >= 1 && splits <= 16, "eth_gemm_splitk: splits must be in [1, 16] (got %d)", splits);
  ETH_CHECK_ARG(M > 0 && N > 0 && K > 0 && M < (1LL << 31) && N < (1LL << 31) && K < (1LL << 31),
                "eth_gemm_splitk: bad shape %lld x %lld x %lld", (long long)M, (long long)N, (long long)K);
  ETH_CHECK_ARG(K % 8 == 0, "eth_gemm_splitk: K (%lld) must be a multiple of 8", (long long)K);
  const int esz = c_dtype == ETH_F32 ? 4 : 2;
  ETH_CHECK_ARG(N % 4 == 0 && ldc % 4 == 0 && ldc >= N && ((uintptr_t)C % (4 * esz)) == 0 &&
                    ((uintptr_t)workspace & 15) == 0,
                "eth_gemm_splitk: C and the workspace need aligned rows of four columns (N %% 4 == 0)");
  ETH_CHECK_ARG(lda % 8 == 0 && ldb % 8 == 0, "eth_gemm_splitk: lda/ldb must be multiples of 8");
  ETH_CHECK_ARG(((uintptr_t)A & 15) == 0 && ((uintptr_t)B & 15) == 0, "eth_gemm_splitk: A/B must be 16-byte aligned");
  ETH_CHECK_ARG(a_kcontig ? lda >= K : (M % 8 == 0 && lda >= M), "eth_gemm_splitk: bad A layout");
  ETH_CHECK_ARG(b_kcontig ? ldb >= K : (N % 8 == 0 && ldb >= N), "eth_gemm_splitk: bad B layout");
  ETH_CHECK_ARG(!(flags & ETH_GEMM_ACCUMULATE) || c_dtype == ETH_F32, "eth_gemm_splitk: accumulate needs fp32 C");
  ETH_CHECK_ARG(!(flags & ETH_GEMM_BIAS) || bias, "eth_gemm_splitk: bias flag without bias");
  const int64_t a_elems = a_kcontig ? (M - 1) * lda + K : (K - 1) * lda + M;
  const int64_t b_elems = b_kcontig ? (N - 1) * ldb + K : (K - 1) * ldb + N;
  const int64_t slice = M * N;
  ETH_CHECK_ARG(a_elems * 2 < (1LL << 31) && b_elems * 2 < (1LL << 31) && (slice + 256 * N) * 4 < (1LL << 31),
                "eth_gemm_splitk: operands above 2 GiB are not supported");
  GemmArgs a{};
  a.A = (const uint16_t*)A;
  a.B = (const uint16_t*)B;
  a.a_bytes = (uint32_t)(a_elems * 2);
  a.b_bytes = (uint32_t)(b_elems * 2);
  a.C = workspace;
  a.bias = nullptr;
  a.M = (int)M;
  a.N = (int)N;
  a.K = (int)K;
  a.lda = lda;
  a.ldb = ldb;
  a.ldc = N;
  a.c_dtype = ETH_F32;
  a.flags = 0;
  a.alpha = 1.0f;
  a.c_bytes = (uint32_t)(slice * 4);
  // whole k-tiles per split, the last split shorter; few k-tiles may leave
  // fewer splits than asked for
  a.k_split = (int)(((K + splits - 1) / splits + 63) / 64 * 64);
  splits = (int)((K + a.k_split - 1) / a.k_split);
  a.c_split_stride = slice;
  hipStream_t s = (hipStream_t)stream;
  const bool fp16 = in_dtype == ETH_F16;
  const int rc = fp16 ? launch_256<true>(a, a_kcontig, b_kcontig, s, splits)
                      : launch_256<false>(a, a_kcontig, b_kcontig, s, splits);
  if (rc != ETH_OK) return rc;
  const SplitSum sum{workspace, splits, slice, C, ldc, (flags & ETH_GEMM_BIAS) ? (const uint16_t*)bias : nullptr,
                     (int)M, (int)N, c_dtype, flags, alpha};
  const int64_t quads = M * (N / 4);
  const int grid = (int)std::min<int64_t>((quads + 255) / 256, 2048);
  if (fp16)
    splitk_sum_kernel<true><<<grid, 256, 0, s>>>(sum);
  else
    splitk_sum_kernel<false><<<grid, 256, 0, s>>>(sum);
  ETH_CHECK_LAUNCH("eth_gemm_splitk");
  return ETH_OK;
}

extern "C" int eth_gemm_splitk(const void* A, int64_t lda, int a_kcontig, const void* B, int64_t ldb, int b_kcontig,
                               float* C, int64_t ldc, int64_t M, int64_t N, int64_t K, int in_dtype, int splits,
                               int accumulate, float* workspace, void* stream) {
  ETH_CHECK_ARG(splits >= 1 && splits <= 16, "eth_gemm_splitk: splits must be in [1, 16] (got %d)", splits);
  ETH_CHECK_ARG(K % (128LL * splits) == 0, "eth_gemm_splitk: K (%lld) must be a multiple of 128 * splits",
                (long long)K);
  return eth_gemm_splitk_out(A, lda, a_kcontig, B, ldb, b_kcontig, C, ldc, ETH_F32, nullptr, M, N, K, in_dtype,
                             accumulate ? ETH_GEMM_ACCUMULATE : 0, 1.0f, splits, workspace, stream);
}
