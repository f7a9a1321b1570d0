// Row operations around the products in 8 bits: rows to e4m3 with scales, the residual stream's norms with that output, rows copied to the
// places of their experts and the weighted sum of what comes back.  fp8.cuh says what a block's scale and values are.  Lanes share a block
// of 128 channels (a warp four each, half a warp eight), so that its largest value is a reduction among them and nothing is read twice.
//
// Norms, t = x + y, h = t / sqrt(mean t^2 + eps) (offset + w): a CTA a row, which stays in registers between the sum of squares and the
// results; scales are written block by block, a word a row, which neighbouring rows' CTAs fill up to sectors in L2.  Bound by HBM and,
// nearly as much, by instructions (85 % of the issue slots): 32768 x 2048, bf16, two norms, one of them in bf16 too 148 us, 6.4 TB/s; 229 with
// IEEE quotients and 256 threads a row.  The product with 1 / s is one more fp32 rounding behind the norm's: 48 to 60 of 67 million values lie on
// another side of a border than in 64 bits, in plain fp32 arithmetic 38 to 58; with a quotient that is rounded once 37 to 48, for 154 us.
// Rows to 8 bits: 8192 x 2048 15.5 us at 1.2 GHz, 3.2 TB/s (21 with four channels a lane).
// Sum of eight experts' results: 8192 x 8 x 2048 of fp32 91 us, 6.3 TB/s.
#include "common.cuh"
#include "early.cuh"
#include "fp8.cuh"
#include "linear_fp8.cuh"
#include "../../include/atma_decoder.h"

namespace atma {

namespace {

template <typename T, int VEC>
struct alignas(VEC * sizeof(T)) Some { T e[VEC]; };

inline bool fits(const void* p, int n) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(n - 1)) == 0; }

// Channels b * 128 + 4 * lane .. + 3 of a row of `width` (kVec), or b * 128 + lane + 32 i; what is behind its end is zero.
template <typename T, bool kVec>
__device__ __forceinline__ void load_block(const T* row, int b, int lane, int width, float (&v)[4]) {
  if constexpr (kVec) {
    const int c = b * kFp8Block + 4 * lane;
    Some<T, 4> p = {};
    if (c < width) p = *reinterpret_cast<const Some<T, 4>*>(row + c);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = c < width ? to_f32(p.e[e]) : 0.f;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int c = b * kFp8Block + lane + 32 * e;
      v[e] = c < width ? to_f32(row[c]) : 0.f;
    }
  }
}
// Stores the block's values and its scale.  kGiven: the values are an input's, see fp8.cuh.
template <bool kVec, bool kGiven>
__device__ __forceinline__ void store_block(uint8_t* row, float* scale, int b, int lane, int width, const float (&v)[4]) {
  const float s = fp8_scale(warp_max_nan(max_nan(max_nan(fabsf(v[0]), fabsf(v[1])), max_nan(fabsf(v[2]), fabsf(v[3])))));
  const float inv = fp8_inverse(s);
  if (lane == 0) *scale = s;
  if constexpr (kVec) {
    const int c = b * kFp8Block + 4 * lane;
    const uint32_t q = kGiven ? fp8_four(v, s) : fp8_four_times(v, inv);
    if (c < width) *reinterpret_cast<uint32_t*>(row + c) = q;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int c = b * kFp8Block + lane + 32 * e;
      if (c < width) row[c] = kGiven ? fp8_one(v[e], s) : fp8_one_times(v[e], inv);
    }
  }
}

// ---- rows to 8 bits ------------------------------------------------------------------------------------
constexpr int kQuantWarps = 8, kQuantBlocks = 4;            // blocks of a row that a warp has in flight

// 16 lanes a block, eight neighbouring channels a lane.
template <typename T>
__global__ void __launch_bounds__(32 * kQuantWarps)
quantize_rows_kernel(const T* x, int64_t x_rs, uint8_t* q, int64_t q_rs, float* scales, int64_t s_bs, int64_t pieces, int per_row, int width) {
  early_start();
  const int64_t piece = (int64_t)blockIdx.x * kQuantWarps + (threadIdx.x >> 5);
  if (piece >= pieces) return;
  const int lane = threadIdx.x & 31, half = lane >> 4, in = 8 * (lane & 15);
  const int64_t row = piece / per_row;
  const int b0 = (int)(piece - row * per_row) * kQuantBlocks + half;
  float v[kQuantBlocks / 2][8];
#pragma unroll
  for (int i = 0; i < kQuantBlocks / 2; ++i) {
    const int c = (b0 + 2 * i) * kFp8Block + in;
    Some<T, 4> p[2] = {};
    if (c < width) {                        // width is a multiple of 8
      if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(x + row * x_rs + c);
      } else {
        p[0] = *reinterpret_cast<const Some<T, 4>*>(x + row * x_rs + c);
        p[1] = *reinterpret_cast<const Some<T, 4>*>(x + row * x_rs + c + 4);
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[i][e] = to_f32(p[e >> 2].e[e & 3]);
  }
#pragma unroll
  for (int i = 0; i < kQuantBlocks / 2; ++i) {
    float most = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) most = max_nan(most, fabsf(v[i][e]));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
    const float s = fp8_scale(most);
    const int b = b0 + 2 * i, c = b * kFp8Block + in;
    if (c >= width) continue;
    if (in == 0) scales[b * s_bs + row] = s;
    const float lo[4] = {v[i][0], v[i][1], v[i][2], v[i][3]}, hi[4] = {v[i][4], v[i][5], v[i][6], v[i][7]};
    *reinterpret_cast<uint2*>(q + row * q_rs + c) = make_uint2(fp8_four(lo, s), fp8_four(hi, s));
  }
}

// Any width, stride and address: a warp a block.
template <typename T>
__global__ void __launch_bounds__(32 * kQuantWarps)
quantize_rows_any_kernel(const T* x, int64_t x_rs, uint8_t* q, int64_t q_rs, float* scales, int64_t s_bs, int64_t pieces, int per_row, int width) {
  early_start();
  const int64_t piece = (int64_t)blockIdx.x * kQuantWarps + (threadIdx.x >> 5);
  if (piece >= pieces) return;
  const int lane = threadIdx.x & 31;
  const int64_t row = piece / per_row;
  const int b0 = (int)(piece - row * per_row) * kQuantBlocks, blocks = (width + kFp8Block - 1) / kFp8Block;
  float v[kQuantBlocks][4];
#pragma unroll
  for (int i = 0; i < kQuantBlocks; ++i) load_block<T, false>(x + row * x_rs, b0 + i, lane, width, v[i]);
#pragma unroll
  for (int i = 0; i < kQuantBlocks; ++i)
    if (b0 + i < blocks) store_block<false, true>(q + row * q_rs, scales + (b0 + i) * s_bs + row, b0 + i, lane, width, v[i]);
}

// ---- the residual stream's norms, in 8 bits ---------------------------------------------------------------
constexpr int kNormThreads = 256;

struct NormOut {
  const void* w;
  uint8_t* q;
  float* scales;
  void* h;                                  // the same in the activation type, or null
};
struct NormArgs {
  const float* x;
  const void* y;
  float* x_out;
  NormOut out[2];
  int64_t q_rs, s_bs;
  int D;
  float eps, offset;
};

__device__ __forceinline__ float row_rms_inverse(float ss, float* s_part, const NormArgs& a) {
  ss = warp_sum(ss);
  if ((threadIdx.x & 31) == 0) s_part[threadIdx.x >> 5] = ss;
  __syncthreads();
  float tot = 0.f;
  for (int i = 0; i < (int)(blockDim.x >> 5); ++i) tot += s_part[i];
  return 1.0f / sqrtf(tot / (float)a.D + a.eps);
}

// One CTA per row; the row stays in registers between the sum of squares and the outputs.  Warp w's i-th group is block i * warps + w.
template <typename T, int NV>
__global__ void __launch_bounds__(kNormThreads)
residual_norms_fp8_kernel(const NormArgs a) {
  early_start();
  __shared__ float s_part[kNormThreads / 32];
  const int64_t row = blockIdx.x, base = row * a.D;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5, blocks = (a.D + kFp8Block - 1) / kFp8Block;
  const T* y = static_cast<const T*>(a.y);
  float v[NV][4];
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) load_block<float, true>(a.x + base, i * warps + warp, lane, a.D, v[i]);
  if (y != nullptr) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float t[4];
      load_block<T, true>(y + base, i * warps + warp, lane, a.D, t);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[i][e] += t[e];
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) ss = fmaf(v[i][e], v[i][e], ss);
  const float rs = row_rms_inverse(ss, s_part, a);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int b = i * warps + warp, c = b * kFp8Block + 4 * lane;
    if (b >= blocks) continue;                               // the whole warp
    if (a.x_out != nullptr && c < a.D) *reinterpret_cast<float4*>(a.x_out + base + c) = make_float4(v[i][0], v[i][1], v[i][2], v[i][3]);
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const NormOut& o = a.out[n];
      if (o.w == nullptr) continue;
      float f[4];
      load_block<T, true>(static_cast<const T*>(o.w), b, lane, a.D, f);
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = c < a.D ? v[i][e] * rs * (a.offset + f[e]) : 0.f;
      store_block<true, false>(o.q + row * a.q_rs, o.scales + b * a.s_bs + row, b, lane, a.D, f);
      if (o.h != nullptr && c < a.D) {
        Some<T, 4> p;
#pragma unroll
        for (int e = 0; e < 4; ++e) p.e[e] = from_f32<T>(f[e]);
        *reinterpret_cast<Some<T, 4>*>(static_cast<T*>(o.h) + base + c) = p;
      }
    }
  }
}

// Any width: the sum is taken again in the second pass.
template <typename T>
__global__ void __launch_bounds__(kNormThreads)
residual_norms_fp8_any_kernel(const NormArgs a) {
  early_start();
  __shared__ float s_part[kNormThreads / 32];
  const int64_t row = blockIdx.x, base = row * a.D;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, blocks = (a.D + kFp8Block - 1) / kFp8Block;
  const T* y = static_cast<const T*>(a.y);
  auto sum_of = [&](int b, float (&v)[4]) {
    load_block<float, false>(a.x + base, b, lane, a.D, v);
    if (y == nullptr) return;
    float t[4];
    load_block<T, false>(y + base, b, lane, a.D, t);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] += t[e];
  };
  float ss = 0.f;
  for (int b = warp; b < blocks; b += warps) {
    float v[4];
    sum_of(b, v);
#pragma unroll
    for (int e = 0; e < 4; ++e) ss = fmaf(v[e], v[e], ss);
  }
  const float rs = row_rms_inverse(ss, s_part, a);
  for (int b = warp; b < blocks; b += warps) {              // the same thread reads and writes a channel: in place is fine
    float v[4];
    sum_of(b, v);
    if (a.x_out != nullptr)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (b * kFp8Block + lane + 32 * e < a.D) a.x_out[base + b * kFp8Block + lane + 32 * e] = v[e];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const NormOut& o = a.out[n];
      if (o.w == nullptr) continue;
      float f[4];
      load_block<T, false>(static_cast<const T*>(o.w), b, lane, a.D, f);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int c = b * kFp8Block + lane + 32 * e;
        f[e] = c < a.D ? v[e] * rs * (a.offset + f[e]) : 0.f;
        if (o.h != nullptr && c < a.D) static_cast<T*>(o.h)[base + c] = from_f32<T>(f[e]);
      }
      store_block<false, false>(o.q + row * a.q_rs, o.scales + b * a.s_bs + row, b, lane, a.D, f);
    }
  }
}

// ---- rows to the places of their experts -------------------------------------------------------------------
// Row t goes to rows place[t * copies + j]; a CTA per row, 16 bytes a thread, what is behind the last whole piece byte by byte.
__global__ void __launch_bounds__(128)
scatter_rows_fp8_kernel(const uint8_t* q, int64_t q_rs, const float* scales, int64_t s_bs, const int32_t* place, int copies, uint8_t* to,
                        int64_t to_rs, float* to_scales, int64_t to_bs, int width, int blocks) {
  early_start();
  const int64_t row = blockIdx.x;
  const uint8_t* from = q + row * q_rs;
  for (int c = threadIdx.x; c < width / 16; c += 128) {
    const uint4 v = *reinterpret_cast<const uint4*>(from + 16 * c);
    for (int j = 0; j < copies; ++j) *reinterpret_cast<uint4*>(to + (int64_t)place[row * copies + j] * to_rs + 16 * c) = v;
  }
  for (int c = width / 16 * 16 + threadIdx.x; c < width; c += 128)
    for (int j = 0; j < copies; ++j) to[(int64_t)place[row * copies + j] * to_rs + c] = from[c];
  for (int i = threadIdx.x; i < blocks * copies; i += 128) {
    const int b = i / copies, j = i - b * copies;
    to_scales[b * to_bs + place[row * copies + j]] = scales[b * s_bs + row];
  }
}

// ---- the weighted sum of a token's results -------------------------------------------------------------------
// Eight results of a token at a time, all of them asked for before the first is summed: a row is 4 KB, and a token by itself is all latency.
template <typename Y, typename T, int VEC>
__global__ void __launch_bounds__(128)
combine_experts_kernel(const Y* y, const int32_t* place, const float* weights, const T* add, T* out, int copies, int D) {
  early_start();
  constexpr int kAtOnce = 8;
  const int64_t row = blockIdx.x;
  const int c = (blockIdx.y * 128 + threadIdx.x) * VEC, lane = threadIdx.x & 31;
  float v[VEC] = {};
  if (add != nullptr && c < D) {
    const Some<T, VEC> p = *reinterpret_cast<const Some<T, VEC>*>(add + row * D + c);
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = to_f32(p.e[e]);
  }
  for (int j0 = 0; j0 < copies; j0 += kAtOnce) {
    const bool mine = lane < kAtOnce && j0 + lane < copies;
    const int at = mine ? place[row * copies + j0 + lane] : 0;
    const float weight = mine ? weights[row * copies + j0 + lane] : 0.f;
    Some<Y, VEC> p[kAtOnce];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      const int64_t from = __shfl_sync(0xffffffffu, at, j);
      if (j0 + j < copies && c < D) p[j] = *reinterpret_cast<const Some<Y, VEC>*>(y + from * D + c);
    }
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      const float w = __shfl_sync(0xffffffffu, weight, j);
      if (j0 + j < copies && c < D)
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = fmaf(w, to_f32(p[j].e[e]), v[e]);
    }
  }
  if (c >= D) return;
  Some<T, VEC> p;
#pragma unroll
  for (int e = 0; e < VEC; ++e) p.e[e] = from_f32<T>(v[e]);
  *reinterpret_cast<Some<T, VEC>*>(out + row * D + c) = p;
}

template <typename Y, typename T>
void launch_combine(const void* y, const int32_t* place, const float* weights, const void* add, void* out, int rows, int copies, int D, cudaStream_t st) {
  constexpr int V = 16 / sizeof(Y);                          // 16 bytes of y a thread
  const bool vec = D % V == 0 && fits(y, 16) && fits(add, V * sizeof(T)) && fits(out, V * sizeof(T));
  const dim3 grid((unsigned)rows, (unsigned)((D + 128 * (vec ? V : 1) - 1) / (128 * (vec ? V : 1))));
  auto* kernel = vec ? combine_experts_kernel<Y, T, V> : combine_experts_kernel<Y, T, 1>;
  launch_early(0, kernel, grid, 128, 0, st, (const Y*)y, place, weights, (const T*)add, (T*)out, copies, D);
}

bool rows_ok(int64_t rows, int64_t width) { return rows >= 0 && rows <= INT32_MAX / 2 && width > 0 && width <= (1 << 24); }

}  // namespace

// See linear_fp8.cuh.
int combine_experts(const void* y, bool wide, const int32_t* place, const float* weights, const void* add, void* out, int rows, int copies, int D,
                    int dtype, cudaStream_t st) {
  ATMA_REQUIRE(dtype == ATMA_F32 || dtype == ATMA_BF16, "combine_experts: unsupported dtype %d", dtype);
  ATMA_REQUIRE(rows_ok(rows, D) && D <= 128 * 65535 && copies > 0 && copies <= 1024 && (int64_t)rows * copies <= INT32_MAX, "combine_experts: bad shape");
  if (rows == 0) return ATMA_OK;
  ATMA_REQUIRE(y != nullptr && place != nullptr && weights != nullptr && out != nullptr, "combine_experts: null tensors");
  if (dtype == ATMA_F32) launch_combine<float, float>(y, place, weights, add, out, rows, copies, D, st);
  else if (wide) launch_combine<float, __nv_bfloat16>(y, place, weights, add, out, rows, copies, D, st);
  else launch_combine<__nv_bfloat16, __nv_bfloat16>(y, place, weights, add, out, rows, copies, D, st);
  return launch_status("combine_experts");
}
}  // namespace atma

using namespace atma;

#define ATMA_FP8_DISPATCH(dt, T, ...)                                       \
  do {                                                                      \
    if ((dt) == ATMA_F32) { using T = float; __VA_ARGS__; }                 \
    else { using T = __nv_bfloat16; __VA_ARGS__; }                          \
  } while (0)

extern "C" int atma_quantize_rows(const void* x, int64_t x_rs, void* q, int64_t q_rs, float* scales, int64_t s_bs, int rows, int width,
                                  int dtype, void* stream) {
  ATMA_REQUIRE(dtype == ATMA_F32 || dtype == ATMA_BF16, "quantize_rows: unsupported dtype %d", dtype);
  ATMA_REQUIRE(rows_ok(rows, width) && x_rs >= 0 && q_rs >= width && s_bs >= rows, "quantize_rows: bad shape or strides");
  if (rows == 0) return ATMA_OK;
  ATMA_REQUIRE(x != nullptr && q != nullptr && scales != nullptr, "quantize_rows: null tensors");
  const int blocks = (width + kFp8Block - 1) / kFp8Block, per_row = (blocks + kQuantBlocks - 1) / kQuantBlocks;
  const int64_t pieces = (int64_t)rows * per_row, ctas = (pieces + kQuantWarps - 1) / kQuantWarps;
  ATMA_REQUIRE(ctas <= INT32_MAX, "quantize_rows: too many rows");
  cudaStream_t st = (cudaStream_t)stream;
  ATMA_FP8_DISPATCH(dtype, T, {
    const bool vec = width % 8 == 0 && x_rs % (16 / sizeof(T)) == 0 && q_rs % 8 == 0 && fits(x, 16) && fits(q, 8);
    auto* kernel = vec ? quantize_rows_kernel<T> : quantize_rows_any_kernel<T>;
    launch_early(0, kernel, (unsigned)ctas, 32 * kQuantWarps, 0, st, (const T*)x, x_rs, (uint8_t*)q, q_rs, scales, s_bs, pieces, per_row, width);
  });
  return launch_status("quantize_rows");
}

extern "C" int atma_residual_norms_fp8(const float* x, const void* y, float* x_out, const void* w1, void* q1, float* s1, void* h1,
                                       const void* w2, void* q2, float* s2, void* h2, int rows, int D, int64_t q_rs, int64_t s_bs,
                                       float eps, float offset, int dtype, void* stream) {
  ATMA_REQUIRE(dtype == ATMA_F32 || dtype == ATMA_BF16, "residual_norms_fp8: unsupported dtype %d", dtype);
  ATMA_REQUIRE(rows_ok(rows, D) && q_rs >= D && s_bs >= rows, "residual_norms_fp8: bad shape or strides");
  if (rows == 0) return ATMA_OK;
  ATMA_REQUIRE(x != nullptr, "residual_norms_fp8: null tensors");
  ATMA_REQUIRE((w1 == nullptr || (q1 != nullptr && s1 != nullptr)) && (w2 == nullptr || (q2 != nullptr && s2 != nullptr)),
               "residual_norms_fp8: a norm without its result");
  cudaStream_t st = (cudaStream_t)stream;
  const NormArgs a{x, y, x_out, {{w1, (uint8_t*)q1, s1, h1}, {w2, (uint8_t*)q2, s2, h2}}, q_rs, s_bs, D, eps, offset};
  const int vb = dtype == ATMA_F32 ? 16 : 8;
  const bool vec = D % 4 == 0 && D <= kNormThreads * 4 * 8 && q_rs % 4 == 0 && fits(x, 16) && fits(x_out, 16) && fits(y, vb) && fits(w1, vb) &&
                   fits(w2, vb) && fits(h1, vb) && fits(h2, vb) && fits(q1, 4) && fits(q2, 4);
  ATMA_FP8_DISPATCH(dtype, T, {
    // threads of a row: 32768 x 2048 159 us with 128, 172 with 256 and 212 with 64; wider rows than 4096 would have more than 8 groups a thread
    const int most = D <= 128 * 4 * 8 ? 128 : kNormThreads;
    const int nv = (D / 4 + most - 1) / most, threads = min(most, ((D / 4 + 31) / 32) * 32);
    if (!vec) launch_early(rows, residual_norms_fp8_any_kernel<T>, rows, kNormThreads, 0, st, a);
    else if (nv <= 1) launch_early(rows, residual_norms_fp8_kernel<T, 1>, rows, threads, 0, st, a);
    else if (nv <= 2) launch_early(rows, residual_norms_fp8_kernel<T, 2>, rows, threads, 0, st, a);
    else if (nv <= 4) launch_early(rows, residual_norms_fp8_kernel<T, 4>, rows, threads, 0, st, a);
    else launch_early(rows, residual_norms_fp8_kernel<T, 8>, rows, threads, 0, st, a);
  });
  return launch_status("residual_norms_fp8");
}

extern "C" int atma_scatter_rows_fp8(const void* q, int64_t q_rs, const float* scales, int64_t s_bs, const int32_t* place, int copies,
                                     void* to, int64_t to_rs, float* to_scales, int64_t to_bs, int rows, int width, void* stream) {
  ATMA_REQUIRE(rows_ok(rows, width) && copies > 0 && copies <= 1024 && (int64_t)rows * copies <= INT32_MAX, "scatter_rows_fp8: bad shape");
  if (rows == 0) return ATMA_OK;
  ATMA_REQUIRE(q != nullptr && scales != nullptr && place != nullptr && to != nullptr && to_scales != nullptr, "scatter_rows_fp8: null tensors");
  ATMA_REQUIRE(q_rs % 16 == 0 && to_rs % 16 == 0 && fits(q, 16) && fits(to, 16) && q_rs >= width && to_rs >= width && s_bs >= rows &&
                   to_bs >= (int64_t)rows * copies,
               "scatter_rows_fp8: rows must start on 16-byte boundaries");
  launch_early(0, scatter_rows_fp8_kernel, (unsigned)rows, 128, 0, (cudaStream_t)stream, (const uint8_t*)q, q_rs, scales, s_bs, place, copies, (uint8_t*)to,
               to_rs, to_scales, to_bs, width, (width + kFp8Block - 1) / kFp8Block);
  return launch_status("scatter_rows_fp8");
}

extern "C" int atma_combine_experts(const void* y, const int32_t* place, const float* weights, const void* add, void* out, int rows,
                                    int copies, int D, int dtype, void* stream) {
  return combine_experts(y, false, place, weights, add, out, rows, copies, D, dtype, (cudaStream_t)stream);
}
