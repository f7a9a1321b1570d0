// Products of rows and weights in 8 bits, out[m][n] = sum over blocks b of 128 columns of xs[m][b] ws[n / 128][b] (x[m], w[n] over b), for
// one weight or for every expert's weight and its own rows; or gelu_tanh of the first half of a weight's results times the second half,
// back in 8 bits.
//
// Every block of 128 columns has scales of its own, so that the tensor cores can only sum inside of one: its products (four of 32 columns)
// go to TMEM, and warps take them from there, times the scales, to sums in registers while the next block's products go to the other
// half of TMEM.  Sums are fp32 all along.
//
// Many rows (linear_fp8_pair_kernel): two SMs share a tile of 256 rows x 256 columns of results (cta_group::2: each holds its 128 rows of x
// and half of the weight's rows, so that a block is 32 KB a CTA for 512 clocks of products).  Eight warps a CTA keep 128 sums a thread.
//   warp 0 TMA, warps 1 and 3 products (of the first CTA, for both; 128 columns each), warp 2 scales, warps 4-11 sums and results.
// Bound by the way from a product to the next one in its place: places are half a block's (128 columns, two of each half), so that its 256
// clocks of products and the 300 that four warps take to read them, with 570 for the barriers between them, share two blocks' 1024.  8192 x 8192 x
// 4096 (1.25 GHz, what the power leaves): 232 to 242 us, 2.3 PFLOP/s, products alone 190.  With whole blocks in two places 250; with a
// release at cluster scope at every block 605; with scales loaded one block ahead by the warps themselves 13 more.  Tried and slower: 16
// warps of 64 sums (276 to 340: more waits than sums), 16 columns of TMEM at a time (248), every warp on both halves (266), the next
// block's wait and first load in front of the last sums (254), results by TMA (no gain, and see below).
// The sums' 128 registers and two loads of 32 fill what a thread has: a version that spills 20 words takes 360 us.
// Gated (65536 rows of 64 experts, 2048 x 2048) 300 us, 1.8 PFLOP/s with the gate and the rows behind the experts' ends; 1024 columns, where
// results leave after every 8 blocks, 175 us, 1.6, in bf16 and 220, 1.25, in fp32.
//
// Few rows (linear_fp8_rows_kernel): the weight's rows are the tensor core's rows, 128 a tile, and the tokens its columns, 16 to 64, so
// that a stage is all weight.  Bound by reading that: two CTAs an SM with 90 to 102 KB of copies in flight each; gated with 32 tokens 72 KB,
// as a third stage does not fit, and gated with 64 tokens one CTA an SM with 200 KB, whose two times 64 sums and products a thread take
// all 255 registers and spill 60 bytes.  128 rows of 64 experts, 2048 x 2048 gated 43 us, 6.2 TB/s; 2048 x 1024 25 us, 5.4.  Where a dense
// product has too few tiles for that, a cluster shares one: every CTA takes its part of the columns, and each then adds up what all of them
// have for some of the tokens, from their shared memory and in their order.  8192 x 2048: 4 rows 9.8 us, 64 rows 11.9 (20 with a token's words read one after another), 128 rows by the other kernel 12.6.
//
// Every mbarrier wait is bounded; on expiry the CTAs free their TMEM, return and leave a status word for the host.
#include "common.cuh"
#include "early.cuh"
#include "f32x2.cuh"
#include "fp8.cuh"
#include "gelu.cuh"
#include "linear_fp8.cuh"
#include "sm100_pair.cuh"
#include "../../include/atma_decoder.h"

namespace atma {

namespace {

using namespace sm100;

constexpr int kBM = 128, kBK = 128;                         // rows of a plane, columns (= bytes) of a stage
constexpr int kPlane = kBM * kBK;
constexpr int kMaxGroups = 512;

__device__ int g_linear_fp8_status = 0;

struct Args {
  const float *x_scales, *w_scales;
  void* out;
  float* out_scales;
  const int32_t* starts;
  int64_t xs_bs, out_rs, os_bs;
  int M, width, K, groups, nb, kb;          // width: columns of results (of one half in the gated form); nb, kb: blocks of width and of K
  bool vec, sectors;                        // rows of out start on 16-byte and on 32-byte boundaries
};

// Tiles of every group's rows, `tall` rows each: s_first[g] of them in front of group g's.  Called by a whole warp.
__device__ __forceinline__ void count_tiles(int* s_first, const Args& a, int tall) {
  const int lane = threadIdx.x & 31;
  int before = 0;
  for (int g0 = 0; g0 < a.groups; g0 += 32) {
    const int g = g0 + lane;
    int n = 0;
    if (g < a.groups) {
      const int lo = a.starts == nullptr ? 0 : min(max(a.starts[g], 0), a.M), hi = a.starts == nullptr ? a.M : min(max(a.starts[g + 1], 0), a.M);
      n = hi > lo ? (hi - lo + tall - 1) / tall : 0;
    }
    int in = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, in, o);
      if (lane >= o) in += t;
    }
    if (g < a.groups) s_first[g] = before + in - n;
    before += __shfl_sync(0xffffffffu, in, 31);
  }
  if (lane == 0) s_first[a.groups] = before;
}

struct Place { int group, m0, m1, n0; };    // rows m0 .. of group, whose rows end at m1; columns n0 ..

// Tile `tile` of the groups' n_tiles x (tiles of rows), kBeside tiles of rows beside one another (0: all of a group's).
template <int kBeside>
__device__ __forceinline__ Place place_of(int tile, const int* s_first, const Args& a, int tall, int wide, int n_tiles) {
  int lo = 0, hi = a.groups;                // the last group with s_first * n_tiles <= tile (empty ones are passed over)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (s_first[mid] * n_tiles <= tile) lo = mid; else hi = mid;
  }
  const int m_tiles = s_first[lo + 1] - s_first[lo], at = tile - s_first[lo] * n_tiles;
  const int band = kBeside == 0 ? 0 : at / (kBeside * n_tiles), in = at - band * kBeside * n_tiles;
  const int high = kBeside == 0 ? m_tiles : min(kBeside, m_tiles - band * kBeside);
  Place p;
  p.group = lo;
  const int first = a.starts == nullptr ? 0 : min(max(a.starts[lo], 0), a.M);
  p.m1 = a.starts == nullptr ? a.M : min(max(a.starts[lo + 1], 0), a.M);
  p.m0 = first + (band * kBeside + in % high) * tall;
  p.n0 = in / high * wide;
  return p;
}

// gelu_tanh(gate) * up of two values each: gate up / (1 + e^-2u), u = sqrt(2 / pi) (z + 0.044715 z^3), by the fast exponential and one
// reciprocal for both if they are of one row (kOne): a value's last bits then depend on the other one, which is nothing that a row may
// see of its neighbour.  The exponent stops at 2^63, where the product of two denominators still fits: results below that are
// off by 1e-19 of gate * up.  Else off by what gelu_tanh_16 is, 6e-6 at most.
template <bool kOne>
__device__ __forceinline__ uint64_t gelu_gate_two(uint64_t gate, uint64_t up) {
  constexpr float kLinear = -2.30220819814f, kCubic = kLinear * 0.044715f;         // -2 sqrt(2 / pi) log2(e)
  const float2 x = unpack2(mul2(fma2(mul2(gate, gate), pack2(kCubic, kCubic), pack2(kLinear, kLinear)), gate));
  float e0, e1;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e0) : "f"(fminf(x.x, 63.f)));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e1) : "f"(fminf(x.y, 63.f)));
  const float a = 1.f + e0, b = 1.f + e1;
  if constexpr (!kOne) return mul2(mul2(gate, up), pack2(__fdividef(1.f, a), __fdividef(1.f, b)));
  const float r = __fdividef(1.f, a * b);
  return mul2(mul2(gate, up), pack2(r * b, r * a));
}

// A barrier of kCount threads at which all of them learn whether one has given up: they leave their loops together.
template <int kCount>
__device__ __forceinline__ bool any_gave_up(bool mine) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "barrier.cta.red.or.pred p, 1, %2, q;\n\tselp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(any) : "r"((uint32_t)mine), "n"(kCount) : "memory");
  return any != 0;
}

// Scales come by a warp of their own, eight blocks ahead over all tiles: a load that the sums' warps ask for one block ahead is not there
// in time (a block of many rows takes 500 clocks, a load twice that).
constexpr int kAhead = 3, kTogether = 4;                   // groups of blocks, blocks of a group

__device__ __forceinline__ void copy_word(float* to, const float* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void arrive_behind_copies(uint64_t* bar) {              // of this thread
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// ---- many rows -------------------------------------------------------------------------------------------
constexpr int kStages = 5, kStageBytes = 2 * kPlane;
constexpr int kSumWarps = 8, kPairThreads = 128 + 32 * kSumWarps;
constexpr int kChunk = 32;                                  // columns of TMEM that a thread loads at a time
constexpr int kStaging = 32 * 128;                          // bytes of a warp's 32 rows x 128 bytes of results
constexpr int kPairSmem = kStages * kStageBytes + kSumWarps * kStaging + 1024;
constexpr int kBeside = 8;

__device__ __forceinline__ void fma_chunk(uint64_t* sum, uint32_t (&r)[kChunk], float scale) {
  const uint64_t s2 = pack2(scale, scale);
#pragma unroll
  for (int i = 0; i < kChunk / 2; ++i) sum[i] = fma2(pack2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])), s2, sum[i]);
}
// One lane's arrival at the pair's first CTA, without a branch: the loads in front of it were the whole warp's.  Nothing but TMEM that has been
// read (tcgen05.wait::ld) is handed over, so that it goes without a release, which waits for everything that the thread has in flight: 1400
// clocks at every block of 512.
__device__ __forceinline__ void arrive_cluster_if(bool mine, uint32_t bar) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %1, 0;\n\t@p mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];\n\t}"
               ::"r"(bar), "r"((int)mine) : "memory");
}
__device__ __forceinline__ bool mbar_wait_lean(uint64_t* bar, uint32_t parity, volatile int* abort) {
  if (__builtin_expect(__all_sync(0xffffffffu, mbar_try_wait(bar, parity)), 1)) return true;
  return mbar_wait_warp(bar, parity, abort);
}

template <typename T, bool kGated>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
linear_fp8_pair_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ Args a) {
  constexpr int kTileN = kGated ? 128 : 256;                // columns of results of a tile
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full[kStages], empty[kStages], acc_full[4], acc_empty[4];      // full and acc_empty: the first CTA's are used
  __shared__ uint32_t s_tmem;
  __shared__ volatile int s_abort_v;
  __shared__ int s_first[kMaxGroups + 1];
  __shared__ float s_most[kGated ? 2 : 1][2][kGated ? 128 : 1];
  __shared__ uint64_t sc_full[kAhead], sc_empty[kAhead];
  __shared__ float s_scale[kAhead][kTogether][kBM + 2];     // of the rows, then of the weight's two blocks
  __shared__ Place s_place[kAhead];                         // of the tile that a group's blocks belong to
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t rank;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

  early_start();
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  if (warp == 2) count_tiles(s_first, a, 2 * kBM);
  if (tid == 32) {
    for (int i = 0; i < kStages; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 2); }
    for (int i = 0; i < 4; ++i) { mbar_init(&acc_full[i], 1); mbar_init(&acc_empty[i], kSumWarps); }
    for (int i = 0; i < kAhead; ++i) { mbar_init(&sc_full[i], 33); mbar_init(&sc_empty[i], kSumWarps); }
    s_abort_v = 0;
    fence_barrier_init();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();                           // the neighbour's barriers are there
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  const int n_tiles = (a.width + kTileN - 1) / kTileN, tiles = s_first[a.groups] * n_tiles;
  volatile int* abort = &s_abort_v;

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 0) {
      if (elect_one()) {
        uint32_t n = 0;                     // blocks so far, over all tiles
        bool ok = true;
        for (int tile = pair; tile < tiles && ok; tile += pairs) {
          const Place p = place_of<kBeside>(tile, s_first, a, 2 * kBM, kTileN, n_tiles);
          const int xr = p.m0 + (int)rank * kBM;
          // 64 rows of the weight for either half of the tile's columns
          const int wr = kGated ? (2 * p.group + (int)rank) * a.width + p.n0 : p.group * a.width + p.n0 + (int)rank * 64, next = kGated ? 64 : 128;
          for (int it = 0; it < a.kb; ++it, ++n) {
            const uint32_t st = n % kStages;
            if (n >= kStages && !(ok = mbar_wait(&empty[st], (n / kStages - 1) & 1, abort))) break;
            uint8_t* to = smem + st * kStageBytes;
            if (rank == 0) mbar_arrive_expect_tx(&full[st], 2 * kStageBytes);
            const uint32_t bar = in_first(smem_u32(&full[st]));
            tma_load_pair(to, &tm_x, bar, it * kBK, xr);
            tma_load_pair(to + kPlane, &tm_w, bar, it * kBK, wr);
            tma_load_pair(to + kPlane + kPlane / 2, &tm_w, bar, it * kBK, wr + next);
          }
        }
        // whatever the others do, the CTA does not end before its copies have landed and the products that read them are done
        volatile int alone = 0;
        for (uint32_t i = n > kStages ? n - kStages : 0; i < n; ++i)
          if (!mbar_wait(&empty[i % kStages], (i / kStages) & 1, &alone)) { *abort = 1; break; }
      }
    } else if (warp == 1 || warp == 3) {    // a half of the results each
      if (rank == 0 && elect_one()) {
        constexpr uint32_t idesc = make_idesc(2 * kBM, kBM, 0, 0, 0);
        const int h = warp >> 1;
        const uint64_t first = make_sdesc_sw128(smem_u32(smem), 16, 1024);
        uint32_t n = 0;
        bool ok = true;
        for (int tile = pair; tile < tiles && ok; tile += pairs) {
          for (int it = 0; it < a.kb; ++it, ++n) {
            const uint32_t st = n % kStages, slot = 2 * (n & 1) + h;
            if (!(ok = mbar_wait(&full[st], (n / kStages) & 1, abort))) break;
            if (n >= 2 && !(ok = mbar_wait(&acc_empty[slot], (n / 2 - 1) & 1, abort))) break;
            tc_fence_after();
            const uint64_t x = first + st * (kStageBytes >> 4), w = x + ((kPlane + h * kPlane / 2) >> 4);      // descriptors count in 16 bytes
#pragma unroll
            for (int k = 0; k < kBK / 32; ++k) mma_pair_8bit(tmem + slot * kBM, x + 2 * k, w + 2 * k, idesc, k > 0);
            commit_pair(&acc_full[slot]);
            commit_pair(&empty[st]);
          }
        }
      }
    } else if (warp == 2) {
      uint32_t n = 0;
      bool ok = true;
      for (int tile = pair; tile < tiles && ok; tile += pairs) {
        const Place p = place_of<kBeside>(tile, s_first, a, 2 * kBM, kTileN, n_tiles);
        const int row0 = p.m0 + (int)rank * kBM + lane, block = p.n0 / 128;
        // the blocks of the weight's rows that meet in the tile: two neighbours, or one of either half
        const float* ws = a.w_scales + (kGated ? (int64_t)(2 * p.group + (lane & 1)) * a.nb + block
                                               : (int64_t)p.group * a.nb + min(block + (lane & 1), a.nb - 1)) * a.kb;
        for (int i0 = 0; i0 < a.kb; i0 += kTogether, ++n) {
          const uint32_t at = n % kAhead;
          if (n >= kAhead && !(ok = mbar_wait_warp(&sc_empty[at], (n / kAhead - 1) & 1, abort))) break;
          for (int it = i0; it < min(i0 + kTogether, a.kb); ++it) {
#pragma unroll
            for (int i = 0; i < kBM; i += 32) copy_word(&s_scale[at][it - i0][i + lane], a.x_scales + it * a.xs_bs + min(row0 + i, a.M - 1));
            if (lane < 2) copy_word(&s_scale[at][it - i0][kBM + lane], ws + it);
          }
          if (lane == 0) {
            s_place[at] = p;
            mbar_arrive(&sc_full[at]);
          }
          arrive_behind_copies(&sc_full[at]);
        }
      }
      asm volatile("cp.async.wait_all;" ::: "memory");      // nothing lands in a CTA that is gone
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int w = warp - 4, quarter = warp & 3, side = w >> 2;
    uint8_t* s = smem + kStages * kStageBytes + w * kStaging;
    const uint32_t acc_empty_there = in_first(smem_u32(&acc_empty[0]));
    uint32_t n = 0, g = 0, turn = 0;        // blocks and groups of scales so far
    bool ok = true;
    for (int tile = pair; tile < tiles && ok; tile += pairs, turn ^= 1) {
      Place p;
      const int c0 = 128 * side;              // gated: 64 of either half of the weight; else a block's
      uint64_t sum[64];
#pragma unroll
      for (int i = 0; i < 64; ++i) sum[i] = 0;
      for (int i0 = 0; i0 < a.kb && ok; i0 += kTogether, ++g) {
        const uint32_t sc = g % kAhead;
        if (!(ok = mbar_wait_lean(&sc_full[sc], (g / kAhead) & 1, abort))) break;
        p = s_place[sc];
        const int blocks = min(kTogether, a.kb - i0);
        for (int it = 0; it < blocks; ++it, ++n) {
          const uint32_t buf = n & 1, slot = 2 * buf + side, at = tmem + (uint32_t(32 * quarter) << 16) + slot * kBM;
          const float fx = s_scale[sc][it][32 * quarter + lane], fw = s_scale[sc][it][kBM + (kGated ? 0 : side)], fu = s_scale[sc][it][kBM + 1];
          if (!(ok = mbar_wait_lean(&acc_full[slot], (n / 2) & 1, abort))) break;
          tc_fence_after();
          uint32_t r[2][kChunk];
          tmem_ld32_nowait(at, r[0]);
          const float sw = fx * fw, su = kGated ? fx * fu : sw;
#pragma unroll
          for (int c = 0; c < 128; c += kChunk) {
            uint32_t(&now)[kChunk] = r[c / kChunk & 1];
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < kChunk; ++i) reg_fence(now[i]);
            const int next = c + kChunk;
            if (next < 128) tmem_ld32_nowait(at + next, r[next / kChunk & 1]);
            else {
              tc_fence_before();
              arrive_cluster_if(lane == 0, acc_empty_there + slot * 8);
            }
            fma_chunk(sum + c / 2, now, c >= 64 ? su : sw);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sc_empty[sc]);
      }
      const int row0 = p.m0 + (int)rank * kBM + 32 * quarter, row = row0 + lane;
      if constexpr (kGated) {               // whether it goes on is decided by all warps together, below
        const int f0 = p.n0 + 64 * side;
        float most = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) sum[i] = gelu_gate_two<true>(sum[i], sum[32 + i]);
        if (p.n0 + 128 > a.width)           // what is behind the last column is another matrix's
#pragma unroll
          for (int i = 0; i < 64; i += 2) {
            const float2 f = unpack2(sum[i / 2]);
            sum[i / 2] = pack2(f0 + i < a.width ? f.x : 0.f, f0 + i + 1 < a.width ? f.y : 0.f);
          }
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const float2 f = unpack2(sum[i]);
          most = max_nan(most, max_nan(fabsf(f.x), fabsf(f.y)));
        }
        // a block's 128 columns are two warps': its largest value through shared memory, in turns of two
        s_most[turn][side][32 * quarter + lane] = most;
        if (any_gave_up<32 * kSumWarps>(!ok || *abort)) break;
        const float scale = fp8_scale(max_nan(s_most[turn][0][32 * quarter + lane], s_most[turn][1][32 * quarter + lane]));
        const float inv = fp8_inverse(scale);
        if (row < p.m1) {
          if (side == 0) a.out_scales[(int64_t)(p.n0 / 128) * a.os_bs + row] = scale;
          uint8_t* to = static_cast<uint8_t*>(a.out) + (int64_t)row * a.out_rs + f0;
#pragma unroll
          for (int i = 0; i < 64; i += 32) {
            uint32_t q[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float2 f = unpack2(sum[(i + 4 * j) / 2]), h = unpack2(sum[(i + 4 * j) / 2 + 1]);
              const float four[4] = {f.x, f.y, h.x, h.y};
              q[j] = fp8_four_times(four, inv);
            }
            if (a.sectors && f0 + i + 32 <= a.width) {       // a whole sector in one go: 330 us with 16 bytes, 316 so (65536 x 2048 x 2048)
              asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                           ::"l"(to + i), "r"(q[0]), "r"(q[1]), "r"(q[2]), "r"(q[3]), "r"(q[4]), "r"(q[5]), "r"(q[6]), "r"(q[7]) : "memory");
            } else {
#pragma unroll
              for (int j = 0; j < 32; j += 16) {
                if (f0 + i + j + 16 <= a.width) {
                  *reinterpret_cast<uint4*>(to + i + j) = make_uint4(q[j / 4], q[j / 4 + 1], q[j / 4 + 2], q[j / 4 + 3]);
                } else {
#pragma unroll
                  for (int l = j; l < j + 16; ++l)
                    if (f0 + i + l < a.width) to[i + l] = (uint8_t)(q[l >> 2] >> 8 * (l & 3));
                }
              }
            }
          }
        }
      } else {
        if (!ok) break;
        constexpr int kCols = 128 / sizeof(T), kPer = 16 / sizeof(T);              // columns of a chunk of 128 bytes, of a piece of 16
        T* out = static_cast<T*>(a.out);
#pragma unroll
        for (int chunk = 0; chunk < 128 / kCols; ++chunk) {
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            alignas(16) T o[kPer];
#pragma unroll
            for (int j = 0; j < kPer; j += 2) {
              const float2 f = unpack2(sum[(chunk * kCols + q * kPer + j) / 2]);
              o[j] = from_f32<T>(f.x);
              o[j + 1] = from_f32<T>(f.y);
            }
            *reinterpret_cast<uint4*>(s + lane * 128 + ((q ^ (lane & 7)) << 4)) = *reinterpret_cast<const uint4*>(o);
          }
          __syncwarp();
          const int q = lane & 7, col = p.n0 + c0 + chunk * kCols + q * kPer;
          T* to = out + (int64_t)(row0 + (lane >> 3)) * a.out_rs + col;
          const bool full = a.vec && col + kPer <= a.width;
#pragma unroll
          for (int i = 0; i < 8; ++i, to += 4 * a.out_rs) {  // four rows at a time, 128 bytes each
            const int r = 4 * i + (lane >> 3);
            const uint4 v = *reinterpret_cast<const uint4*>(s + r * 128 + ((q ^ (r & 7)) << 4));
            if (row0 + r >= p.m1) continue;
            if (full) *reinterpret_cast<uint4*>(to) = v;
            else {
              const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
              for (int j = 0; j < kPer; ++j)
                if (col + j < a.width) to[j] = e[j];
            }
          }
          __syncwarp();
        }
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  cluster_sync();                           // nobody signals a CTA that is gone
  tc_fence_after();
  if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  if (tid == 0 && s_abort_v) atomicExch(&g_linear_fp8_status, 1);
}

// The place of another CTA of the cluster, and a word of it.
__device__ __forceinline__ uint32_t in_cta(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ float load_cluster(uint32_t addr) {
  float f;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(f) : "r"(addr));
  return f;
}

// The largest of every token's values over the lanes, of token `lane` (modulo N, 16 or 32) in the end: N shuffles for N tokens.
template <int N>
__device__ __forceinline__ float token_max(float (&m)[N]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = N / 2; o > 0; o >>= 1) {
    const bool upper = lane & o;
#pragma unroll
    for (int i = 0; i < o; ++i) {
      const float keep = upper ? m[i + o] : m[i], send = upper ? m[i] : m[i + o];
      m[i] = max_nan(keep, __shfl_xor_sync(0xffffffffu, send, o));
    }
  }
  if (N == 16) m[0] = max_nan(m[0], __shfl_xor_sync(0xffffffffu, m[0], 16));
  return m[0];
}

// ---- few rows --------------------------------------------------------------------------------------------
constexpr int kRowsThreads = 192;

template <int NT, bool kGated>
struct Few {
  static constexpr int kHalves = kGated ? 2 : 1;
  static constexpr int kStageBytes = kHalves * kPlane + NT * kBK;
  static constexpr int kCtas = kHalves * NT >= 128 ? 1 : 2; // of an SM: with 128 sums and as many products a thread there is one
  static constexpr int kStages = (kCtas == 1 ? 208 : 104) * 1024 / kStageBytes;
  static constexpr int kBufs = kHalves * NT >= 128 ? 2 : 4, kColumns = kBufs * kHalves * NT;
  static constexpr int kSmem = kStages * kStageBytes + 1024;
  static_assert(kColumns <= 256 && kColumns >= 32 && (kColumns & (kColumns - 1)) == 0, "two CTAs share an SM's TMEM");
  static_assert(kHalves * NT * 128 * 4 <= kStages * kStageBytes, "a cluster's sums lie where the copies were");
};

template <typename T, int NT, bool kGated>
__global__ void __launch_bounds__(kRowsThreads, Few<NT, kGated>::kCtas)
linear_fp8_rows_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ Args a) {
  using F = Few<NT, kGated>;
  constexpr int kHalves = F::kHalves;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full[F::kStages], empty[F::kStages], acc_full[F::kBufs], acc_empty[F::kBufs];
  __shared__ uint32_t s_tmem;
  __shared__ volatile int s_abort_v;
  __shared__ int s_first[kMaxGroups + 1];
  __shared__ __align__(16) float s_scale[4][2][kHalves][NT];
  __shared__ float s_most[kGated ? 4 : 1][kGated ? NT : 1];
  __shared__ __align__(8) float s_inverse[kGated ? 4 : 1][kGated ? NT : 2];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t rank, ranks;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
  const int worker = blockIdx.x / ranks, workers = gridDim.x / ranks;

  if (warp == 0) tmem_alloc(&s_tmem, F::kColumns);
  if (tid == 32) {
    for (int i = 0; i < F::kStages; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
    for (int i = 0; i < F::kBufs; ++i) { mbar_init(&acc_full[i], 1); mbar_init(&acc_empty[i], 4); }
    s_abort_v = 0;
    fence_barrier_init();
    prefetch_tensormap(&tm_x);
    prefetch_tensormap(&tm_w);
  }
  early_start();                            // nothing in front of it reads or writes what another kernel does
  if (warp == 2) count_tiles(s_first, a, NT);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  const int n_tiles = (a.width + kBM - 1) / kBM, tiles = s_first[a.groups] * n_tiles;
  // a cluster's CTAs share the columns of its one tile
  const int k0 = (int)((int64_t)a.kb * rank / ranks), k1 = (int)((int64_t)a.kb * (rank + 1) / ranks);
  volatile int* abort = &s_abort_v;

  if (warp == 0) {
    if (elect_one()) {
      uint32_t n = 0;
      bool ok = true;
      for (int tile = worker; tile < tiles && ok; tile += workers) {
        const Place p = place_of<0>(tile, s_first, a, NT, kBM, n_tiles);
        for (int it = k0; it < k1; ++it, ++n) {
          const uint32_t st = n % F::kStages;
          if (n >= F::kStages && !(ok = mbar_wait(&empty[st], (n / F::kStages - 1) & 1, abort))) break;
          uint8_t* to = smem + st * F::kStageBytes;
          mbar_arrive_expect_tx(&full[st], F::kStageBytes);
#pragma unroll
          for (int h = 0; h < kHalves; ++h)
            tma_load_4d(to + h * kPlane, &tm_w, &full[st], it * kBK, (kHalves * p.group + h) * a.width + p.n0, 0, 0);
          tma_load_4d(to + kHalves * kPlane, &tm_x, &full[st], it * kBK, p.m0, 0, 0);
        }
      }
      volatile int alone = 0;               // see above
      for (uint32_t i = n > F::kStages ? n - F::kStages : 0; i < n; ++i)
        if (!mbar_wait(&empty[i % F::kStages], (i / F::kStages) & 1, &alone)) { *abort = 1; break; }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      constexpr uint32_t idesc = make_idesc(kBM, NT, 0, 0, 0);
      uint32_t n = 0;
      bool ok = true;
      for (int tile = worker; tile < tiles && ok; tile += workers) {
        for (int it = k0; it < k1; ++it, ++n) {
          const uint32_t st = n % F::kStages, buf = n % F::kBufs;
          if (n >= F::kBufs && !(ok = mbar_wait(&acc_empty[buf], (n / F::kBufs - 1) & 1, abort))) break;
          if (!(ok = mbar_wait(&full[st], (n / F::kStages) & 1, abort))) break;
          tc_fence_after();
          const uint32_t at = smem_u32(smem + st * F::kStageBytes), d = tmem + buf * kHalves * NT;
#pragma unroll
          for (int h = 0; h < kHalves; ++h)
#pragma unroll
            for (int k = 0; k < kBK / 32; ++k)
              mma_8bit(d + h * NT, make_sdesc_sw128(at + h * kPlane + 32 * k, 16, 1024), make_sdesc_sw128(at + kHalves * kPlane + 32 * k, 16, 1024), idesc, k > 0);
          tc_commit(&empty[st]);
          tc_commit(&acc_full[buf]);
        }
      }
    }
  } else {
    const int quarter = warp & 3, feature = 32 * quarter + lane;         // of the tile's 128
    uint32_t n = 0;
    bool ok = true;
    for (int tile = worker; tile < tiles && ok; tile += workers) {
      const Place p = place_of<0>(tile, s_first, a, NT, kBM, n_tiles);
      const int rows = min(NT, p.m1 - p.m0), col = p.n0 + feature;
      const float* ws = a.w_scales + ((int64_t)kHalves * p.group * a.nb + p.n0 / 128) * a.kb;
      const float* us = ws + (kGated ? (int64_t)a.nb * a.kb : 0);
      uint64_t sum[kHalves][NT / 2];
#pragma unroll
      for (int h = 0; h < kHalves; ++h)
#pragma unroll
        for (int i = 0; i < NT / 2; ++i) sum[h][i] = 0;
      // lane l brings the scales of tokens l and l + 32, one block ahead
      constexpr int kOwn = (NT + 31) / 32;
      float fx[kOwn], fw, fu;
      auto bring = [&](int it) {
#pragma unroll
        for (int i = 0; i < kOwn; ++i) fx[i] = lane + 32 * i < rows ? a.x_scales[it * a.xs_bs + p.m0 + lane + 32 * i] : 0.f;
        fw = ws[it];
        fu = us[it];
      };
      bring(k0);
      for (int it = k0; it < k1; ++it, ++n) {
        const uint32_t buf = n % F::kBufs;
        float(&sc)[kHalves][NT] = s_scale[quarter][n & 1];
#pragma unroll
        for (int i = 0; i < kOwn; ++i)
          if (lane + 32 * i < NT) {
            sc[0][lane + 32 * i] = fx[i] * fw;
            if constexpr (kGated) sc[kHalves - 1][lane + 32 * i] = fx[i] * fu;
          }
        __syncwarp();
        if (it + 1 < k1) bring(it + 1);
        if (!(ok = mbar_wait_warp(&acc_full[buf], (n / F::kBufs) & 1, abort))) break;
        tc_fence_after();
        const uint32_t at = tmem + (uint32_t(32 * quarter) << 16) + buf * kHalves * NT;
        constexpr int kAtOnce = kHalves * NT <= 64 ? kHalves : 1;        // halves whose products a thread holds beside the sums
        uint32_t r[kAtOnce][NT];
#pragma unroll
        for (int h0 = 0; h0 < kHalves; h0 += kAtOnce) {
#pragma unroll
          for (int h = 0; h < kAtOnce; ++h)
#pragma unroll
            for (int c = 0; c < NT; c += 16) tmem_ld16_nowait(at + (h0 + h) * NT + c, &r[h][c]);
          tmem_ld_wait();
#pragma unroll
          for (int h = 0; h < kAtOnce; ++h)
#pragma unroll
            for (int c = 0; c < NT; ++c) reg_fence(r[h][c]);
          if (h0 + kAtOnce == kHalves) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[buf]);
          }
#pragma unroll
          for (int h = 0; h < kAtOnce; ++h)
#pragma unroll
            for (int c = 0; c < NT; c += 4) {
              const ulonglong2 f = *reinterpret_cast<const ulonglong2*>(&sc[h0 + h][c]);
              uint64_t(&to)[NT / 2] = sum[h0 + h];
              to[c / 2] = fma2(pack2(__uint_as_float(r[h][c]), __uint_as_float(r[h][c + 1])), f.x, to[c / 2]);
              to[c / 2 + 1] = fma2(pack2(__uint_as_float(r[h][c + 2]), __uint_as_float(r[h][c + 3])), f.y, to[c / 2 + 1]);
            }
        }
      }
      if (!kGated || ranks > 1)
        if (!ok) break;
      if (ranks > 1) {                      // what this CTA has, to where its copies were: all of them have been read
        float* part = reinterpret_cast<float*>(smem);
#pragma unroll
        for (int h = 0; h < kHalves; ++h)
#pragma unroll
          for (int c = 0; c < NT; c += 2) {
            const float2 f = unpack2(sum[h][c / 2]);
            part[(h * NT + c) * 128 + feature] = f.x;
            part[(h * NT + c + 1) * 128 + feature] = f.y;
          }
        break;                              // a cluster has one tile
      }
      if constexpr (kGated) {
        constexpr int kPart = NT < 32 ? NT : 32;             // tokens whose largest values the lanes sort out among them
#pragma unroll
        for (int i = 0; i < NT / 2; ++i) {
          const float2 f = unpack2(gelu_gate_two<false>(sum[0][i], sum[kHalves - 1][i]));
          sum[0][i] = col < a.width ? pack2(f.x, f.y) : 0;   // what is behind the last column is another matrix's
        }
#pragma unroll
        for (int t = 0; t < NT; t += kPart) {
          float most[kPart];
#pragma unroll
          for (int c = 0; c < kPart; c += 2) {
            const float2 f = unpack2(sum[0][(t + c) / 2]);
            most[c] = fabsf(f.x);
            most[c + 1] = fabsf(f.y);
          }
          const float mine = token_max<kPart>(most);
          if (lane < kPart) s_most[quarter][t + lane] = mine;
        }
        if (any_gave_up<128>(!ok || *abort)) break;
#pragma unroll
        for (int t = lane; t < NT; t += 32) {
          const float scale = fp8_scale(max_nan(max_nan(s_most[0][t], s_most[1][t]), max_nan(s_most[2][t], s_most[3][t])));
          if (quarter == 0 && t < rows) a.out_scales[(int64_t)(p.n0 / 128) * a.os_bs + p.m0 + t] = scale;
          s_inverse[quarter][t] = fp8_inverse(scale);
        }
        __syncwarp();
        if (col < a.width) {
          uint8_t* to = static_cast<uint8_t*>(a.out) + (int64_t)p.m0 * a.out_rs + col;
#pragma unroll
          for (int c = 0; c < NT; c += 2) {
            const float2 inv = *reinterpret_cast<const float2*>(&s_inverse[quarter][c]), f = unpack2(sum[0][c / 2]);
            const uint32_t q = fp8_two(f.x * inv.x, f.y * inv.y);
            if (c < rows) to[c * a.out_rs] = (uint8_t)q;
            if (c + 1 < rows) to[(c + 1) * a.out_rs] = (uint8_t)(q >> 8);
          }
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");       // s_most is read
      } else if (col < a.width) {
        T* out = static_cast<T*>(a.out) + (int64_t)p.m0 * a.out_rs + col;
#pragma unroll
        for (int c = 0; c < NT; ++c) {
          const float2 f = unpack2(sum[0][c / 2]);
          if (c < rows) out[c * a.out_rs] = from_f32<T>(c & 1 ? f.y : f.x);
        }
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  if (ranks > 1) {                          // the same for all of the cluster
    __syncthreads();
    cluster_sync();
    if (warp >= 2 && worker < tiles) {
      const Place p = place_of<0>(worker, s_first, a, NT, kBM, n_tiles);
      const int feature = 32 * (warp & 3) + lane, rows = min(NT, p.m1 - p.m0), col = p.n0 + feature;
      constexpr int kAtOnce = 4;            // tokens: their loads are under way together
      for (int c0 = rank; c0 < rows; c0 += kAtOnce * ranks) {
        float v[kAtOnce][kHalves] = {};
#pragma unroll 2
        for (uint32_t o = 0; o < ranks; ++o) {
          const uint32_t there = in_cta(smem_u32(smem) + feature * 4, o);
#pragma unroll
          for (int i = 0; i < kAtOnce; ++i)
#pragma unroll
            for (int h = 0; h < kHalves; ++h) v[i][h] += load_cluster(there + (h * NT + min(c0 + i * (int)ranks, NT - 1)) * 512);
        }
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
          const int c = c0 + i * ranks;
          if (c >= rows) break;             // the same for all
          if constexpr (kGated) {
            const float f = col < a.width ? gelu_tanh_16(v[i][0]) * v[i][kHalves - 1] : 0.f;
            const float most = warp_max_nan(fabsf(f));
            if (lane == 0) s_most[warp & 3][c] = most;
            asm volatile("bar.sync 1, 128;" ::: "memory");
            const float scale = fp8_scale(max_nan(max_nan(s_most[0][c], s_most[1][c]), max_nan(s_most[2][c], s_most[3][c])));
            if (feature == 0) a.out_scales[(int64_t)(p.n0 / 128) * a.os_bs + p.m0 + c] = scale;
            if (col < a.width) static_cast<uint8_t*>(a.out)[(int64_t)(p.m0 + c) * a.out_rs + col] = fp8_one_times(f, fp8_inverse(scale));
          } else if (col < a.width) {
            static_cast<T*>(a.out)[(int64_t)(p.m0 + c) * a.out_rs + col] = from_f32<T>(v[i][0]);
          }
        }
      }
    }
    cluster_sync();                         // nobody reads a CTA that is gone
  }
  __syncthreads();
  tc_fence_after();
  if (warp == 0) tmem_dealloc(tmem, F::kColumns);
  if (tid == 0 && s_abort_v) atomicExch(&g_linear_fp8_status, 1);
}

template <typename T, bool kGated>
int launch_pair(const CUtensorMap& x, const CUtensorMap& w, const Args& a, cudaStream_t st) {
  auto kern = linear_fp8_pair_kernel<T, kGated>;
  ATMA_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kPairSmem));
  const int64_t n_tiles = (a.width + (kGated ? 127 : 255)) / (kGated ? 128 : 256);
  const int64_t tiles = (a.M / (2 * kBM) + (a.groups < a.M ? a.groups : a.M)) * n_tiles;       // at most
  ATMA_REQUIRE(tiles < INT32_MAX / 2, "linear_fp8: too many tiles");
  const int pairs = sm_count_of_current_device() / 2;
  launch_early(0, kern, dim3(2 * (unsigned)(tiles < pairs ? tiles : pairs)), dim3(kPairThreads), kPairSmem, st, x, w, a);
  return launch_status("linear_fp8 (many rows)");
}

// Clusters of `ranks` CTAs that run at once.  With a CTA an SM fewer of them find a place than of its CTAs, since a cluster's lie in one GPC, and a
// second turn of clusters costs more than what sharing K gives (gated 1024 x 8192, 256 rows: 31.6 us by eight, 23.3 by four); that is asked
// for once per device.  With two CTAs an SM it is not so: what the query gives is 24 us with 192 rows of 2048 x 8192, CTAs alone 17.5.
template <int NT, bool kGated>
int64_t clusters_at_once(int ranks) {
  using F = Few<NT, kGated>;
  static int cached[64][4] = {};
  const int64_t guess = F::kCtas * (int64_t)sm_count_of_current_device() / ranks;
  int dev = 0, at = ranks == 2 ? 1 : ranks == 4 ? 2 : 3, n = 0;
  if (F::kCtas > 1 || ranks == 1 || cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return guess;
  if (cached[dev][at] == 0) {
    auto kern = linear_fp8_rows_kernel<float, NT, kGated>;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = ranks; attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3(ranks); c.blockDim = dim3(kRowsThreads); c.dynamicSmemBytes = F::kSmem; c.attrs = &attr; c.numAttrs = 1;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, F::kSmem) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, kern, &c) != cudaSuccess || n <= 0) {
      cudaGetLastError();
      return guess;
    }
    cached[dev][at] = n;                    // the same value from every host thread
  }
  return cached[dev][at];
}

// CTAs that share a tile's columns: as many as find a place with all tiles, four blocks each at least.
template <int NT, bool kGated>
int ranks_of(int64_t tiles, int kb) {
  int ranks = 1;
  while (ranks < 8 && 4 * 2 * ranks <= kb && tiles <= clusters_at_once<NT, kGated>(2 * ranks)) ranks *= 2;
  return ranks;
}

template <typename T, int NT, bool kGated>
int launch_rows(const CUtensorMap& x, const CUtensorMap& w, const Args& a, cudaStream_t st) {
  using F = Few<NT, kGated>;
  auto kern = linear_fp8_rows_kernel<T, NT, kGated>;
  ATMA_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, F::kSmem));
  const int64_t n_tiles = (a.width + kBM - 1) / kBM, slots = F::kCtas * (int64_t)sm_count_of_current_device();
  const int64_t tiles = (a.starts == nullptr ? (a.M + NT - 1) / NT : a.M / NT + (a.groups < a.M ? a.groups : a.M)) * n_tiles;
  ATMA_REQUIRE(tiles < INT32_MAX / 2, "linear_fp8: too many tiles");
  const int ranks = a.starts == nullptr ? ranks_of<NT, kGated>(tiles, a.kb) : 1;
  cudaLaunchAttribute attrs[2];
  attrs[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;              // see early.cuh
  attrs[1].val.programmaticStreamSerializationAllowed = 1;
  attrs[0].id = cudaLaunchAttributeClusterDimension;
  attrs[0].val.clusterDim.x = ranks; attrs[0].val.clusterDim.y = attrs[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t c = {};
  c.gridDim = dim3((unsigned)(tiles < slots / ranks ? tiles : slots / ranks) * ranks); c.blockDim = dim3(kRowsThreads);
  c.dynamicSmemBytes = F::kSmem; c.stream = st; c.attrs = attrs; c.numAttrs = 2;
  ATMA_CUDA_OK(cudaLaunchKernelEx(&c, kern, x, w, a));
  return launch_status("linear_fp8 (few rows)");
}

// Which kernel, by a group's rows if all have as many.  The pair kernel reads a weight once for 256 rows, but a pair walks all of K by itself,
// 5.6 us and 0.39 a block; few rows are bound by the weights, and share K: about 7.5 us and 0.58 a block, gated 14 and 0.7 (reading sums
// from one another and a barrier for every token's scale).  Chains of blocks of one weight are compared by that, experts' rows by what was
// measured, us, few rows / many rows:
//   8192 x 2048   64 rows 11.9 / 12.4   80 rows 13.6 / 12.4;   4096 x 4096   128 rows 13.3 / 18.3   512 rows 23.5 / 18.5;
//   2048 x 8192   256 rows 17.4 / 28.5   512 rows 26.1 / 29.2;   gated 4096 x 2048   40 rows 15.2 / 13.0;   gated 1024 x 8192   256 rows 24.1 / 29.4
//   64 experts of 2 x 1024 x 2048, the whole feed-forward   32 rows each 105 / 117   48 119 / 119   64 141 / 129   125 203 / 156;
//   its second product   48 119 / 130   64 141 / 144   96 174 / 165
template <bool kGated>
bool many_rows(const Args& a, int each) {
  if (a.starts != nullptr) return each > (kGated ? 48 : 64);
  if (each <= 32) return false;
  auto over = [](int64_t n, int64_t by) { return (n + by - 1) / by; };
  const int64_t sms = sm_count_of_current_device(), tiles = over(a.M, 64) * over(a.width, 128);
  const int64_t pair = over(over(a.M, 256) * over(a.width, kGated ? 128 : 256), sms / 2) * a.kb;
  const int ranks = ranks_of<64, kGated>(tiles, a.kb);
  const int64_t few = over(tiles * ranks, Few<64, kGated>::kCtas * sms) * over(a.kb, ranks);
  return kGated ? 10 * pair <= 18 * few + 200 : 10 * pair <= 15 * few + 50;
}

template <typename T, bool kGated>
int launch(const atma_fp8_args& f, const Args& a, cudaStream_t st) {
  const int each = (a.M + a.groups - 1) / a.groups, nt = many_rows<kGated>(a, each) ? 0 : each <= 16 ? 16 : each <= 32 ? 32 : 64;
  CUtensorMap x, w;
  int rc = make_tmap_8bit_rows(&x, f.x, a.M, f.x_rs, a.K, nt > 0 ? nt : kBM);
  if (rc == ATMA_OK) rc = make_tmap_8bit_rows(&w, f.w, (uint64_t)a.groups * f.N, f.w_rs, a.K, nt > 0 ? kBM : kBM / 2);
  if (rc != ATMA_OK) return rc;
  if (nt == 16) return launch_rows<T, 16, kGated>(x, w, a, st);
  if (nt == 32) return launch_rows<T, 32, kGated>(x, w, a, st);
  if (nt == 64) return launch_rows<T, 64, kGated>(x, w, a, st);
  return launch_pair<T, kGated>(x, w, a, st);
}

}  // namespace

int linear_fp8_status_fetch_and_clear(int* out) {
  int v = 0, zero = 0;
  ATMA_CUDA_OK(cudaMemcpyFromSymbol(&v, g_linear_fp8_status, sizeof(int)));
  if (v != 0) ATMA_CUDA_OK(cudaMemcpyToSymbol(g_linear_fp8_status, &zero, sizeof(int)));
  *out = v;
  return ATMA_OK;
}

}  // namespace atma

using namespace atma;

extern "C" int atma_linear_fp8(const atma_fp8_args* args, void* stream) {
  ATMA_REQUIRE(args != nullptr, "linear_fp8: null args");
  const atma_fp8_args& f = *args;
  ATMA_REQUIRE(f.form == 0 || f.form == 1, "linear_fp8: unknown form %d", f.form);
  ATMA_REQUIRE(f.form == 1 || f.dtype == ATMA_F32 || f.dtype == ATMA_BF16, "linear_fp8: unsupported dtype %d", f.dtype);
  ATMA_REQUIRE(f.M >= 0 && f.M <= (1 << 28) && f.N > 0 && f.N <= (1 << 24) && f.N % (f.form + 1) == 0 && f.K > 0 && f.K <= (1 << 24),
               "linear_fp8: bad shape (%d, %d, %d)", f.M, f.N, f.K);
  ATMA_REQUIRE(f.groups > 0 && f.groups <= kMaxGroups && (f.starts != nullptr || f.groups == 1) && (int64_t)f.groups * f.N <= INT32_MAX - kBM,
               "linear_fp8: %d groups of %d rows, or without their rows", f.groups, f.N);
  if (f.M == 0) return ATMA_OK;
  auto al16 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  ATMA_REQUIRE(f.x != nullptr && f.w != nullptr && f.out != nullptr && f.x_scales != nullptr && f.w_scales != nullptr, "linear_fp8: null tensors");
  ATMA_REQUIRE(al16(f.x) && al16(f.w) && f.x_rs % 16 == 0 && f.w_rs % 16 == 0 && f.x_rs >= f.K && f.w_rs >= f.K,
               "linear_fp8: rows of x and of the weight must start on 16-byte boundaries");
  const int width = f.N / (f.form + 1);
  ATMA_REQUIRE(f.out_rs >= width && f.xs_bs >= f.M, "linear_fp8: overlapping rows");
  ATMA_REQUIRE(f.form == 0 || (f.out_scales != nullptr && f.os_bs >= f.M && al16(f.out) && f.out_rs % 16 == 0),
               "linear_fp8: results in 8 bits need scales and rows that start on 16-byte boundaries");
  const Args a{f.x_scales, f.w_scales, f.out, f.out_scales, f.starts, f.xs_bs, f.out_rs, f.os_bs, f.M, width, f.K, f.groups, (width + 127) / 128,
               (f.K + 127) / 128, al16(f.out) && f.out_rs * (f.dtype == ATMA_F32 ? 4 : 2) % 16 == 0,
               (reinterpret_cast<uintptr_t>(f.out) & 31) == 0 && f.out_rs % 32 == 0};
  cudaStream_t st = (cudaStream_t)stream;
  if (f.form == 1) return launch<float, true>(f, a, st);
  return f.dtype == ATMA_F32 ? launch<float, false>(f, a, st) : launch<__nv_bfloat16, false>(f, a, st);
}
