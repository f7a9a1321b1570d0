// Products of rows and weights in 8 bits: out[m][n] = sum over blocks b of 128 columns of xs[m][b] ws[n / 128][b] sum over the block of
// x[m][c] w[n][c], for one weight or for every expert's weight and its own rows.
//
// 64 x 64 results a CTA, 4 x 4 a thread, fp32 arithmetic.
#include "common.cuh"
#include "fp8.cuh"
#include "../../include/atma_decoder.h"

namespace atma {

namespace {

constexpr int kTile = 64, kCols = 32;

__device__ __forceinline__ float wide(uint8_t v) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(v, __NV_E4M3)));
}

template <typename T>
__global__ void __launch_bounds__(256)
linear_fp8_kernel(const atma_fp8_args a) {
  __shared__ float s_x[kCols][kTile + 1], s_w[kCols][kTile + 1];
  __shared__ int s_place[3];
  const int tid = threadIdx.x;
  if (tid == 0) {                           // which group's rows, and which of them
    int tile = blockIdx.x, g = 0, lo = 0, hi = a.starts == nullptr ? a.M : 0;
    s_place[0] = -1;
    for (; g < a.groups; ++g) {
      if (a.starts != nullptr) { lo = a.starts[g]; hi = a.starts[g + 1]; }
      const int n = (hi - lo + kTile - 1) / kTile;
      if (tile < n) { s_place[0] = g; s_place[1] = lo + tile * kTile; s_place[2] = hi; break; }
      tile -= n;
    }
  }
  __syncthreads();
  if (s_place[0] < 0) return;
  const int g = s_place[0], m0 = s_place[1], m1 = s_place[2], n0 = blockIdx.y * kTile;
  const int kb = (a.K + kFp8Block - 1) / kFp8Block, width = a.N / a.parts, nb = (width + kFp8Block - 1) / kFp8Block;
  const uint8_t *x = (const uint8_t*)a.x, *w = (const uint8_t*)a.w + (int64_t)g * a.N * a.w_rs;
  const float* ws = a.w_scales + (int64_t)g * a.parts * nb * kb;
  const int ty = tid >> 4, tx = tid & 15;
  float sum[4][4] = {}, part[4][4];
  for (int c0 = 0; c0 < a.K; c0 += kCols) {
    if (c0 % kFp8Block == 0)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) part[i][j] = 0.f;
    for (int i = tid; i < kTile * kCols; i += 256) {
      const int r = i / kCols, c = i % kCols;
      s_x[c][r] = m0 + r < m1 && c0 + c < a.K ? wide(x[(int64_t)(m0 + r) * a.x_rs + c0 + c]) : 0.f;
      s_w[c][r] = n0 + r < a.N && c0 + c < a.K ? wide(w[(int64_t)(n0 + r) * a.w_rs + c0 + c]) : 0.f;
    }
    __syncthreads();
    for (int c = 0; c < kCols; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) part[i][j] = fmaf(s_x[c][ty + 16 * i], s_w[c][tx + 16 * j], part[i][j]);
    __syncthreads();
    if ((c0 + kCols) % kFp8Block == 0 || c0 + kCols >= a.K) {
      const int b = c0 / kFp8Block;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int m = m0 + ty + 16 * i;
        const float xs = m < m1 ? a.x_scales[(int64_t)b * a.xs_bs + m] : 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int n = n0 + tx + 16 * j;
          if (n < a.N) sum[i][j] = fmaf(part[i][j], xs * ws[((int64_t)(n / width) * nb + n % width / kFp8Block) * kb + b], sum[i][j]);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
      if (m < m1 && n < a.N) ((T*)a.out)[(int64_t)m * a.out_rs + n] = from_f32<T>(sum[i][j]);
    }
}

}  // namespace
}  // namespace atma

using namespace atma;

extern "C" int atma_linear_fp8(const atma_fp8_args* args, void* stream) {
  ATMA_REQUIRE(args != nullptr, "linear_fp8: null args");
  const atma_fp8_args& a = *args;
  ATMA_REQUIRE(a.dtype == ATMA_F32 || a.dtype == ATMA_BF16, "linear_fp8: unsupported dtype %d", a.dtype);
  ATMA_REQUIRE(a.M >= 0 && a.M <= (1 << 28) && a.N > 0 && a.N <= (1 << 24) && a.K > 0 && a.K <= (1 << 24), "linear_fp8: bad shape (%d, %d, %d)", a.M, a.N, a.K);
  ATMA_REQUIRE(a.groups > 0 && a.groups <= 65536 && (a.starts != nullptr || a.groups == 1), "linear_fp8: %d groups without their rows", a.groups);
  ATMA_REQUIRE((a.parts == 1 || a.parts == 2) && a.N % a.parts == 0, "linear_fp8: %d rows in %d parts", a.N, a.parts);
  if (a.M == 0) return ATMA_OK;
  auto al16 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  ATMA_REQUIRE(a.x != nullptr && a.w != nullptr && a.out != nullptr && a.x_scales != nullptr && a.w_scales != nullptr, "linear_fp8: null tensors");
  ATMA_REQUIRE(al16(a.x) && al16(a.w) && a.x_rs % 16 == 0 && a.w_rs % 16 == 0 && a.x_rs >= a.K && a.w_rs >= a.K,
               "linear_fp8: rows of x and of the weight must start on 16-byte boundaries");
  ATMA_REQUIRE(a.out_rs >= a.N && a.xs_bs >= a.M, "linear_fp8: overlapping rows");
  const dim3 grid((unsigned)(a.M / kTile + (a.groups < a.M ? a.groups : a.M)), (unsigned)((a.N + kTile - 1) / kTile));
  ATMA_REQUIRE(grid.y <= 65535, "linear_fp8: N=%d", a.N);
  cudaStream_t st = (cudaStream_t)stream;
  if (a.dtype == ATMA_F32) linear_fp8_kernel<float><<<grid, 256, 0, st>>>(a);
  else linear_fp8_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(a);
  return launch_status("linear_fp8");
}
