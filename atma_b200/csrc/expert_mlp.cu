// The experts' feed-forwards in one call: rows to the places of their experts, both products, the weighted sum.
#include "common.cuh"
#include "linear_fp8.cuh"
#include "../../include/atma_decoder.h"

namespace atma {

namespace {

int64_t round_up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

struct Parts { int64_t rows, row_scales, act, act_scales, y, all; };             // offsets in the scratch memory, bytes

// Experts' results are fp32 until they are summed, however many there are, so that the type of out is the only rounding behind the products
// and a token's precision does not go by the tokens beside it.  (In bf16 a bf16 sum's error has a 2-norm of 2.3e-3 instead of 1.7e-3, for half of
// the bytes between the two kernels: 8192 tokens, 8 of 64 experts, 2048 / 1024, 682 us instead of 767.)

// Values of 128 bytes more than a row's are never needed: rows start on 16-byte boundaries, parts on 256-byte ones.
Parts parts_of(int64_t rows, int width, int ff) {
  Parts p;
  p.rows = 0;
  p.row_scales = round_up(p.rows + rows * round_up(width, 16), 256);
  p.act = round_up(p.row_scales + rows * 4 * ((width + 127) / 128), 256);
  p.act_scales = round_up(p.act + rows * round_up(ff, 16), 256);
  p.y = round_up(p.act_scales + rows * 4 * ((ff + 127) / 128), 256);
  p.all = p.y + rows * width * (int64_t)sizeof(float);
  return p;
}

}  // namespace
}  // namespace atma

using namespace atma;

extern "C" int64_t atma_expert_mlp_scratch_bytes(int tokens, int copies, int width, int ff, int dtype) {
  if (tokens <= 0 || copies <= 0 || width <= 0 || ff <= 0) return 0;
  (void)dtype;                              // results between the kernels have one type, whatever out's is
  return parts_of((int64_t)tokens * copies, width, ff).all;
}

extern "C" int atma_expert_mlp(const atma_expert_args* args, void* scratch, void* stream) {
  ATMA_REQUIRE(args != nullptr, "expert_mlp: null args");
  const atma_expert_args& a = *args;
  ATMA_REQUIRE(a.dtype == ATMA_F32 || a.dtype == ATMA_BF16, "expert_mlp: unsupported dtype %d", a.dtype);
  ATMA_REQUIRE(a.tokens >= 0 && a.copies > 0 && a.copies <= 1024 && (int64_t)a.tokens * a.copies <= (1 << 28) && a.width > 0 && a.ff > 0 && a.ff <= (1 << 23),
               "expert_mlp: bad shape");
  if (a.tokens == 0) return ATMA_OK;
  ATMA_REQUIRE(scratch != nullptr && (reinterpret_cast<uintptr_t>(scratch) & 255) == 0, "expert_mlp: scratch memory must be 256-byte aligned");
  ATMA_REQUIRE(a.place != nullptr && a.starts != nullptr && a.weights != nullptr && a.out != nullptr, "expert_mlp: null tensors");
  const int rows = a.tokens * a.copies;
  const Parts p = parts_of(rows, a.width, a.ff);
  uint8_t* s = static_cast<uint8_t*>(scratch);
  const int64_t x_rs = round_up(a.width, 16), act_rs = round_up(a.ff, 16);
  float *row_scales = reinterpret_cast<float*>(s + p.row_scales), *act_scales = reinterpret_cast<float*>(s + p.act_scales);
  int rc = atma_scatter_rows_fp8(a.x, a.x_rs, a.x_scales, a.xs_bs, a.place, a.copies, s + p.rows, x_rs, row_scales, rows, a.tokens, a.width, stream);
  if (rc != ATMA_OK) return rc;
  const atma_fp8_args up = {s + p.rows, x_rs, row_scales, rows, a.w_gate_up, a.w_gate_up_rs, a.w_gate_up_scales, s + p.act, act_rs, act_scales, rows,
                            a.starts, rows, 2 * a.ff, a.width, a.experts, 1, 0};
  rc = atma_linear_fp8(&up, stream);
  if (rc != ATMA_OK) return rc;
  const atma_fp8_args down = {s + p.act, act_rs, act_scales, rows, a.w_down, a.w_down_rs, a.w_down_scales, s + p.y, a.width, nullptr, 0,
                              a.starts, rows, a.width, a.ff, a.experts, 0, ATMA_F32};
  rc = atma_linear_fp8(&down, stream);
  if (rc != ATMA_OK) return rc;
  return combine_experts(s + p.y, true, a.place, a.weights, a.add, a.out, a.tokens, a.copies, a.width, a.dtype, (cudaStream_t)stream);
}
