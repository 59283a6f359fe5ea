// Matrix product with its epilogue, y = act(x W^T + b) + r, and its backward (bf16 operands, fp32 accumulation).
//
// One tcgen05 kernel serves the three products of a training step, C[M, N] = sum_k A[m, k] B[n, k] with either operand
// stored k-contiguous or with its other index contiguous (K- or MN-major tiles):
//   forward  y  = x W^T      A = x   (M, K)  k-contiguous     B = W (N, K)  k-contiguous
//   backward dx = dp W       A = dp  (M, N)  k-contiguous     B = W (N, K)  contiguous along the output
//            dW = dp^T x     A = dp  (M, N)  along the output  B = x (M, K)  along the output
//
// A persistent block computes 128 x BN tiles: one warp issues the TMA loads of 64-deep k blocks into a ring of stages,
// one warp issues the MMAs, eight warps read finished accumulators from tensor memory and run the epilogue while the
// MMAs of the next tile go on (two accumulators).  Operands that TMA cannot address (rows not 16-byte aligned) are laid
// out again first, padded, in the workspace.
#include "gdn_tiles.cuh"
#include "sm100_ptx.cuh"
#include "ssm_common.cuh"

namespace gdn {
namespace linear {

constexpr int BM = 128, BK = 64;
constexpr int EPI_WARPS = 8;                        // two per quarter of the tensor-memory lanes
constexpr int THREADS = 64 + 32 * EPI_WARPS;
constexpr int OUT_BYTES = 32 * 128;                 // a warp's output box: 32 rows x 64 columns
constexpr long long WAIT_CYCLES = 4000000000ll;     // ~2 s: a wait that runs this long gives up

__device__ int g_status = 0;

using bf16 = __nv_bfloat16;
using namespace ssm;  // packed fp32 arithmetic, vector loads and stores

struct Operand {  // a row-major matrix, `rows` rows of `cols` contiguous values
  const bf16* p;
  int64_t ld;
  int64_t rows, cols;
  int tma;  // rows start on 16-byte boundaries: a tensor map can address it
};

struct GemmP {
  Operand a, b;
  int64_t M, N, K;
  int tiles_m, tiles_n, splits, kblocks;  // k blocks of 64 in all
  // epilogue (splits == 1)
  bf16* y;
  int64_t ldy;
  bf16* pre;  // (M, N) contiguous, or NULL: x W^T + b, or with `slope` act'(x W^T + b) in fp16
  const bf16* bias;
  const bf16* res;
  int64_t ldr;
  int act, vec, slope;
  float* part;  // splits > 1: (splits, M, N) sums
  int part_tma; // N a multiple of four: TMA stores them
  // Tiles run along the shorter side first: a wave then reads few rows of the longer operand, once, and the shorter
  // operand stays in L2.
  int n_first;
  __device__ int tile_m(int t) const { return n_first ? t / tiles_n : t % tiles_m; }
  __device__ int tile_n(int t) const { return n_first ? t % tiles_n : t / tiles_m; }
};

// PAIR: two CTAs of a cluster work on one 256 x BN tile, each with half of A's rows, half of B's and half of the
// accumulator's rows; one of them issues the MMAs of both.  Half the operand bytes per multiplication come from L2 and
// shared memory.
template <int BN, bool PAIR>
struct Cfg {
  static constexpr int BROWS = PAIR ? BN / 2 : BN;  // rows of B that a CTA holds
  static constexpr int STAGE = (BM + BROWS) * BK * 2;
  static constexpr int STAGES = 196608 / STAGE;  // 4, 6, 8 for BN = 256 (6 in pairs), 128, 64
  static constexpr int COLS = BN == 64 ? 64 : BN / 2;  // columns per epilogue warp (with 64, half of the warps rest)
  static constexpr int SMEM = STAGES * STAGE + EPI_WARPS * OUT_BYTES + 1024 /* alignment */ + 256 /* barriers */;
};

// Phi(x), the normal distribution, and e^(-x^2 / 2), for two values: Phi(-|x|) = erfc(|x| / sqrt 2) / 2 by the rational
// approximation 7.1.26 of Abramowitz and Stegun (absolute error 1.5e-7 in erfc, no cancellation in the lower tail).
__device__ __forceinline__ f32x2 normal2(f32x2 x, f32x2& bell) {
  const float2 v = unpack2(x);
  const f32x2 ax = pack2(fabsf(v.x), fabsf(v.y));
  const float2 n = unpack2(fma2(ax, both(0.3275911f * 0.70710678f), both(1.f)));
  const f32x2 t = pack2(ssm::rcp(n.x), ssm::rcp(n.y));
  bell = exp2_2(mul2(mul2(x, x), both(-0.5f * ssm::LOG2E)));
  f32x2 q = fma2(t, both(0.5f * 1.061405429f), both(0.5f * -1.453152027f));
  q = fma2(t, q, both(0.5f * 1.421413741f));
  q = fma2(t, q, both(0.5f * -0.284496736f));
  q = fma2(t, q, both(0.5f * 0.254829592f));
  const f32x2 low = mul2(mul2(t, q), bell);
  const float2 l = unpack2(low), u = unpack2(fma2(low, both(-1.f), both(1.f)));
  return pack2(v.x < 0.f ? l.x : u.x, v.y < 0.f ? l.y : u.y);
}
__device__ __forceinline__ f32x2 act_fwd2(f32x2 p, int act) {
  if (act == GDN_ACT_SILU) return mul2(p, sigmoid2(p));
  if (act == GDN_ACT_GELU) {
    f32x2 bell;
    return mul2(p, normal2(p, bell));
  }
  return p;
}
// act(p), and act'(p) in `slope`.
__device__ __forceinline__ f32x2 act_both2(f32x2 p, int act, f32x2& slope) {
  slope = both(1.f);
  if (act == GDN_ACT_SILU) {
    const f32x2 g = sigmoid2(p);
    slope = mul2(g, fma2(p, fma2(g, both(-1.f), both(1.f)), both(1.f)));
    return mul2(p, g);
  }
  if (act == GDN_ACT_GELU) {
    f32x2 bell;
    const f32x2 phi = normal2(p, bell);
    slope = fma2(mul2(p, bell), both(0.39894228040143267794f), phi);
    return mul2(p, phi);
  }
  return p;
}
__device__ __forceinline__ f32x2 act_grad2(f32x2 p, int act) {
  f32x2 slope;
  act_both2(p, act, slope);
  return slope;
}
// What the backward needs of the activation is kept as act'(p) in fp16: a slope within [-0.2, 1.2] loses 2^-12 of itself, an
// eighth of what dp then loses on its way into the bf16 matrix product.  p itself in bf16 lost 2^-9 of p, which near the
// slope's zero (p = -1.28 for SiLU, -0.75 for GELU) is many times the slope.  The bytes are the same.
__device__ __forceinline__ uint32_t slope_bits(f32x2 v) {
  const float2 e = unpack2(v);
  const __half2 h = __floats2half2_rn(e.x, e.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ f32x2 slope_pair(uint32_t bits) {
  const float2 e = __half22float2(*reinterpret_cast<const __half2*>(&bits));
  return pack2(e.x, e.y);
}
// One value: the activation of v, with what the backward reads of it put at `pre` first.
__device__ __forceinline__ float act_one(float v, int act, bf16* pre, int slope) {
  f32x2 d;
  const float y = unpack2(act_both2(both(v), act, d)).x;
  if (pre && slope)
    *reinterpret_cast<__half*>(pre) = __float2half_rn(unpack2(d).x);
  else if (pre)
    *pre = __float2bfloat16_rn(v);
  return y;
}

__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(
          ptx::smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(ptx::smem_u32(bar)), "r"(c0), "r"(c1)
      : "memory");
}

// The pair's forms: a load into this CTA's memory that reports to a barrier of the pair's first CTA, the MMA over both
// CTAs' operands and accumulators, and the arrival on the same barrier of both.
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const CUtensorMap* map, uint32_t bar_cluster, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(
          ptx::smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar_cluster), "r"(c0), "r"(c1)
      : "memory");
}
__device__ __forceinline__ void mma_pair_elect(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred e, p;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "@e tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void commit_pair_elect(uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}" ::"r"(
          ptx::smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}

// One operand's part of a stage: ROWS output indices x 64 k.  k-contiguous: one box of ROWS rows; else ROWS / 64 boxes
// of 64 k rows.
template <int ROWS, bool MN, bool PAIR>
__device__ __forceinline__ void stage_tma(char* dst, const CUtensorMap* map, uint64_t* bar, uint32_t pair_bar, int idx0, int k0) {
  auto load = [&](char* to, int c0, int c1) {
    if (PAIR)
      tma_load_2d_pair(to, map, pair_bar, c0, c1);
    else
      tma_load_2d(to, map, bar, c0, c1);
  };
  if (!MN) {
    load(dst, k0, idx0);
  } else {
#pragma unroll
    for (int i = 0; i < ROWS / 64; ++i) load(dst + i * 8192, idx0 + i * 64, k0);
  }
}

// Operand descriptor of k step s (16 deep) in a stage part at shared address `base`.
template <bool MN>
__device__ __forceinline__ uint64_t step_desc(uint32_t base, int s) {
  return MN ? ptx::sdesc_sw128(base + s * 2048, 8192, 1024) : ptx::sdesc_sw128(base + s * 32, 16, 1024);
}

// A warp's 32 rows x 64 columns, written to `box` in the 128-byte-swizzled layout and stored by TMA (which clips rows
// and columns past the matrix).  The box is free again once the copy has read it.
__device__ __forceinline__ void box_ready(int lane) {
  if (lane == 0) ptx::bulk_wait_read0();
  __syncwarp();
}
__device__ __forceinline__ void box_put(char* box, int lane, int col, const f32x2 (&v)[16]) {  // 32 columns from col (0, 32)
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 e = unpack2(v[j * 4 + i]);
      const __nv_bfloat162 h = __floats2bfloat162_rn(e.x, e.y);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(box + lane * 128 + (((col / 8 + j) ^ (lane & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}
__device__ __forceinline__ void box_store(const CUtensorMap* map, const char* box, int lane, int64_t row, int64_t col) {
  ptx::fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(reinterpret_cast<uint64_t>(map)),
                 "r"(ptx::smem_u32(box)), "r"((int)col), "r"((int)row)
                 : "memory");
    ptx::bulk_commit();
  }
}

__device__ __forceinline__ void box_store3(const CUtensorMap* map, const char* box, int lane, int64_t row, int64_t col, int split) {
  ptx::fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(reinterpret_cast<uint64_t>(map)),
                 "r"(ptx::smem_u32(box)), "r"((int)col), "r"((int)row), "r"(split)
                 : "memory");
    ptx::bulk_commit();
  }
}

// The same box from and to rows that no vector takes: a row at a time, the lanes along its columns.
__device__ __forceinline__ bf16* box_at(char* box, int row, int col) {
  return reinterpret_cast<bf16*>(box + row * 128 + (((col >> 3) ^ (row & 7)) << 4)) + (col & 7);
}
// ROWS at a time: the reads of a batch go out before its writes, which the compiler must keep in order.
__device__ __noinline__ void box_copy_out(char* box, int lane, bf16* p, int64_t ld, int64_t row0, int64_t col0, int64_t M, int64_t N) {
  constexpr int ROWS = 8;
  __syncwarp();
  const int rows = (int)(M - row0 < 32 ? M - row0 : 32);
  const bool a = col0 + lane < N, b = col0 + 32 + lane < N;
  bf16* q = p + row0 * ld + col0 + lane;
#pragma unroll 1
  for (int r = 0; r < rows; r += ROWS, q += ROWS * ld) {
    bf16 v[ROWS][2];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      v[i][0] = *box_at(box, r + i, lane);
      v[i][1] = *box_at(box, r + i, lane + 32);
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      if (a && r + i < rows) q[i * ld] = v[i][0];
      if (b && r + i < rows) q[i * ld + 32] = v[i][1];
    }
  }
  __syncwarp();
}
__device__ __noinline__ void box_copy_in(char* box, int lane, const bf16* p, int64_t ld, int64_t row0, int64_t col0, int64_t M, int64_t N) {
  constexpr int ROWS = 16;
  const int rows = (int)(M - row0 < 32 ? M - row0 : 32);
  const bool a = col0 + lane < N, b = col0 + 32 + lane < N;
  const bf16* q = p + row0 * ld + col0 + lane;
#pragma unroll 1
  for (int r = 0; r < rows; r += ROWS, q += ROWS * ld) {
    bf16 v[ROWS][2];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      v[i][0] = a && r + i < rows ? q[i * ld] : __float2bfloat16_rn(0.f);
      v[i][1] = b && r + i < rows ? q[i * ld + 32] : __float2bfloat16_rn(0.f);
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      *box_at(box, r + i, lane) = v[i][0];
      *box_at(box, r + i, lane + 32) = v[i][1];
    }
  }
  __syncwarp();
}

// SLOPE: the forward of a training step, which keeps the activation's slopes.  (As a form of its own: with a choice at run time the
// bare products took 2 % longer.)
template <int BN, bool AMN, bool BMN, bool PAIR, bool SLOPE>
__global__ void __launch_bounds__(THREADS, 1)
    gemm_kernel(const __grid_constant__ CUtensorMap ma, const __grid_constant__ CUtensorMap mb, const __grid_constant__ CUtensorMap my,
                const __grid_constant__ CUtensorMap mpre, const __grid_constant__ CUtensorMap mres, const GemmP p) {
  using C = Cfg<BN, PAIR>;
  constexpr int ST = C::STAGES, A_BYTES = BM * BK * 2, B_BYTES = C::BROWS * BK * 2, CTAS = PAIR ? 2 : 1;
  extern __shared__ char raw_smem[];
  char* tiles = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(raw_smem) + 1023) & ~(uintptr_t)1023);
  char* boxes = tiles + ST * C::STAGE;
  uint64_t* full = reinterpret_cast<uint64_t*>(boxes + EPI_WARPS * OUT_BYTES);
  uint64_t* empty = full + ST;
  uint64_t* tfull = empty + ST;
  uint64_t* tempty = tfull + 2;
  uint64_t* rfull = tempty + 2;  // per epilogue warp: its residual box is in
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(rfull + EPI_WARPS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  if (tid == 0) {
    for (int i = 0; i < ST; ++i) {
      ptx::mbar_init(full + i, 1);
      ptx::mbar_init(empty + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(tfull + i, 1);
      ptx::mbar_init(tempty + i, BN == 64 ? 4 : EPI_WARPS * CTAS);
    }
    for (int i = 0; i < EPI_WARPS; ++i) ptx::mbar_init(rfull + i, 1);
    *abort_flag = 0;
    ptx::fence_mbar_init();
  }
  if (warp == 1) {
    if (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(ptx::smem_u32(tmem_slot)), "r"(2 * BN) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      ptx::tmem_alloc(tmem_slot, 2 * BN);
      ptx::tmem_relinquish();
    }
  }
  __syncthreads();
  if (PAIR) ptx::cluster_sync();  // both CTAs' barriers are ready
  ptx::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // A CTA, or a pair of them, takes every `units`-th item; row and column offsets of its half of the operands.
  const uint32_t rank = PAIR ? ptx::cluster_ctarank() : 0;
  const int unit = blockIdx.x / CTAS, units = gridDim.x / CTAS, half = rank * BM;
  const int items = p.tiles_m * p.tiles_n * p.splits;
  const int per = (p.kblocks + p.splits - 1) / p.splits;
  auto wait = [&](uint64_t* bar, uint32_t parity) { return ptx::mbar_wait_abortable(bar, parity, WAIT_CYCLES, abort_flag); };

  if (warp == 0) {
    if (lane == 0) {
      uint32_t n = 0;  // k blocks issued
      bool ok = true;
      for (int it = unit; ok && it < items; it += units) {
        const int tile = it / p.splits, sp = it % p.splits;
        const int m0 = p.tile_m(tile) * (BM * CTAS) + half, n0 = p.tile_n(tile) * BN + (PAIR ? half : 0);
        const int kb1 = min((sp + 1) * per, p.kblocks);
        for (int kb = sp * per; kb < kb1; ++kb, ++n) {
          const int s = n % ST;
          if (!wait(empty + s, ((n / ST) & 1) ^ 1)) { ok = false; break; }
          char* st = tiles + s * C::STAGE;
          if (rank == 0) ptx::mbar_arrive_expect_tx(full + s, (A_BYTES + B_BYTES) * CTAS);
          const uint32_t pair_bar = PAIR ? ptx::mapa_shared(ptx::smem_u32(full + s), 0) : 0;
          stage_tma<BM, AMN, PAIR>(st, &ma, full + s, pair_bar, m0, kb * BK);
          stage_tma<C::BROWS, BMN, PAIR>(st + A_BYTES, &mb, full + s, pair_bar, n0, kb * BK);
        }
      }
      if (ok && PAIR)  // the MMAs' arrivals on this CTA's barriers come from the other one: all of them, before it can leave
        for (uint32_t i = n > ST ? n - ST : 0; i < n; ++i) wait(empty + i % ST, (i / ST) & 1);
      if (!ok && rank == 0)  // leave no copy in flight: each outstanding stage's barrier, with a limit
        for (uint32_t i = n > ST ? n - ST : 0; i < n; ++i) ptx::mbar_wait_bounded(full + i % ST, (i / ST) & 1, WAIT_CYCLES / 8);
    }
  } else if (warp == 1 && rank == 0) {
    constexpr uint32_t idesc = ptx::idesc_bf16_f32(BM * CTAS, BN, AMN, BMN);
    uint32_t n = 0, acc = 0;
    bool ok = true;
    for (int it = unit; ok && it < items; it += units, ++acc) {
      const int sp = it % p.splits;
      const int kb0 = sp * per, kb1 = min((sp + 1) * per, p.kblocks);
      const uint32_t buf = acc & 1;
      if (PAIR ? !ptx::mbar_wait_abortable_cluster(tempty + buf, ((acc >> 1) & 1) ^ 1, WAIT_CYCLES, abort_flag)
               : !wait(tempty + buf, ((acc >> 1) & 1) ^ 1))
        break;
      ptx::tc_fence_after();
      for (int kb = kb0; kb < kb1; ++kb, ++n) {
        const int s = n % ST;
        if (!wait(full + s, (n / ST) & 1)) { ok = false; break; }
        ptx::tc_fence_after();
        const uint32_t a = ptx::smem_u32(tiles + s * C::STAGE), b = a + A_BYTES;
#pragma unroll
        for (int k = 0; k < BK / 16; ++k) {
          if (PAIR)
            mma_pair_elect(tmem + buf * BN, step_desc<AMN>(a, k), step_desc<BMN>(b, k), idesc, kb > kb0 || k > 0);
          else
            ptx::mma_f16_ss_elect(tmem + buf * BN, step_desc<AMN>(a, k), step_desc<BMN>(b, k), idesc, kb > kb0 || k > 0);
        }
        PAIR ? commit_pair_elect(empty + s) : ptx::mma_commit_elect(empty + s);
      }
      PAIR ? commit_pair_elect(tfull + buf) : ptx::mma_commit_elect(tfull + buf);
      if (!ok) ptx::mbar_wait_bounded(tfull + buf, (acc >> 1) & 1, WAIT_CYCLES / 8);  // no MMA left in flight
    }
  } else if (warp >= 2) {
    const int quarter = warp % 4;  // tensor-memory lanes this warp can read
    const int c0 = (warp - 2) / 4 * C::COLS;  // its first column of a tile
    char* box = boxes + (warp - 2) * OUT_BYTES;
    uint32_t acc = 0, fetched = 0;
    for (int it = unit; c0 < BN && it < items; it += units, ++acc) {
      const int tile = it / p.splits, sp = it % p.splits;
      const int64_t row0 = (int64_t)p.tile_m(tile) * (BM * CTAS) + half + quarter * 32, row = row0 + lane, n0 = (int64_t)p.tile_n(tile) * BN;
      const uint32_t buf = acc & 1;
      const bool in = row < p.M;
      // The residual of 64 columns: fetched into the box while the accumulator is waited for, taken into registers before
      // the box carries an output.
      uint4 res[8];
      auto fetch_res = [&](int64_t col) {
        if (!p.res || p.splits > 1 || row0 >= p.M || col >= p.N) return;
        if (!p.vec) {
          box_copy_in(box, lane, p.res, p.ldr, row0, col, p.M, p.N);
        } else if (lane == 0) {
          ptx::bulk_wait_read0();
          ptx::mbar_arrive_expect_tx(rfull + warp - 2, OUT_BYTES);
          tma_load_2d(box, &mres, rfull + warp - 2, (int)col, (int)row0);
        }
      };
      auto take_res = [&](int64_t col) {
        if (!p.res) return true;
        if (p.vec && !wait(rfull + warp - 2, fetched++ & 1)) return false;
#pragma unroll
        for (int j = 0; j < 8; ++j) res[j] = *reinterpret_cast<const uint4*>(box + lane * 128 + ((j ^ (lane & 7)) << 4));
        __syncwarp();
        return true;
      };
      auto send = [&](const CUtensorMap* map, bf16* to, int64_t ld, int64_t col) {  // the box's 64 columns
        if (p.vec)
          box_store(map, box, lane, row0, col);
        else
          box_copy_out(box, lane, to, ld, row0, col, p.M, p.N);
      };
      auto put = [&](const CUtensorMap* map, bf16* to, int64_t ld, int64_t col, const f32x2 (&v)[2][16]) {
        if (p.vec) box_ready(lane);
        box_put(box, lane, 0, v[0]);
        box_put(box, lane, 32, v[1]);
        send(map, to, ld, col);
      };
      fetch_res(n0 + c0);
      if (!wait(tfull + buf, (acc >> 1) & 1)) break;
      ptx::tc_fence_after();
#pragma unroll 1
      for (int c = c0; c < c0 + C::COLS; c += 64) {
        if (n0 + c >= p.N || row0 >= p.M) break;  // the warp's part lies outside
        const uint32_t t = tmem + (uint32_t)(quarter * 32 << 16) + buf * BN + c;
        if (p.splits > 1) {  // 32 x 32 sums at a time, staged and stored like the outputs
#pragma unroll 1
          for (int e = 0; e < 64; e += 32) {
            float v[32];
            ptx::tmem_ld32(t + e, v);
            ptx::tc_wait_ld();
            const int64_t col = n0 + c + e;
            if (p.part_tma) {
              box_ready(lane);
#pragma unroll
              for (int j = 0; j < 8; ++j)
                *reinterpret_cast<float4*>(box + lane * 128 + ((j ^ (lane & 7)) << 4)) = make_float4(v[j * 4], v[j * 4 + 1], v[j * 4 + 2], v[j * 4 + 3]);
              box_store3(&my, box, lane, row0, col, sp);
            } else if (in) {
              float* q = p.part + ((int64_t)sp * p.M + row) * p.N + col;
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (col + i < p.N) q[i] = v[i];
            }
            __syncwarp();  // the next load is warp-wide
          }
          continue;
        }
        f32x2 v[2][16];
        {
          float a[2][32];
          ptx::tmem_ld32(t, a[0]);
          ptx::tmem_ld32(t + 32, a[1]);
          ptx::tc_wait_ld();
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int i = 0; i < 16; ++i) v[e][i] = pack2(a[e][2 * i], a[e][2 * i + 1]);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int64_t col0 = n0 + c + e * 32;
          if (p.bias && p.vec) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint4 bv = col0 + j * 8 < p.N ? __ldg(reinterpret_cast<const uint4*>(p.bias + col0 + j * 8)) : make_uint4(0, 0, 0, 0);
              const bf16* q = reinterpret_cast<const bf16*>(&bv);
#pragma unroll
              for (int i = 0; i < 4; ++i) v[e][j * 4 + i] = add2(v[e][j * 4 + i], load_pair(q + 2 * i));
            }
          } else if (p.bias) {
            const float bl = col0 + lane < p.N ? to_f32(p.bias[col0 + lane]) : 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i)
              v[e][i] = add2(v[e][i], pack2(__shfl_sync(0xffffffffu, bl, 2 * i), __shfl_sync(0xffffffffu, bl, 2 * i + 1)));
          }
        }
        if (!__all_sync(0xffffffffu, take_res(n0 + c))) break;
        auto apply = [&](int act) {  // a loop per activation: choosing it per value cost 30 us of 183 at 32768 x 2816 x 1024
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int i = 0; i < 16; ++i) v[e][i] = act_fwd2(v[e][i], act);
        };
        auto apply_with_slope = [&](int act) {  // the slopes go to the box as they are formed
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              f32x2& q = v[j / 4][j % 4 * 4 + i];
              f32x2 d;
              q = act_both2(q, act, d);
              w[i] = slope_bits(d);
            }
            *reinterpret_cast<uint4*>(box + lane * 128 + ((j ^ (lane & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        };
        if constexpr (SLOPE) {
          if (p.vec) box_ready(lane);
          if (p.act == GDN_ACT_SILU)
            apply_with_slope(GDN_ACT_SILU);
          else
            apply_with_slope(GDN_ACT_GELU);
          send(&mpre, p.pre, p.N, n0 + c);
        } else {
          if (p.pre) put(&mpre, p.pre, p.N, n0 + c, v);
          if (p.act == GDN_ACT_SILU) apply(GDN_ACT_SILU);
          if (p.act == GDN_ACT_GELU) apply(GDN_ACT_GELU);
        }
        if (p.res) {
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int i = 0; i < 16; ++i) v[e][i] = add2(v[e][i], load_pair(reinterpret_cast<const bf16*>(&res[e * 4 + i / 4]) + i % 4 * 2));
        }
        put(&my, p.y, p.ldy, n0 + c, v);
        if (c + 64 < c0 + C::COLS) fetch_res(n0 + c + 64);
      }
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (PAIR)
          ptx::mbar_arrive_remote(ptx::mapa_shared(ptx::smem_u32(tempty + buf), 0));
        else
          ptx::mbar_arrive(tempty + buf);
      }
    }
    if (*abort_flag && p.res && p.vec && lane == 0)  // a residual box may still be on its way
      ptx::mbar_wait_bounded(rfull + warp - 2, fetched & 1, WAIT_CYCLES / 8);
    if (lane == 0) ptx::bulk_wait0();  // the stores have read the boxes and are done
    __syncwarp();
  }
  __syncthreads();
  if (tid == 0 && *abort_flag) atomicExch(&g_status, GDN_ERR_TIMEOUT);
  if (PAIR) {
    ptx::cluster_sync();  // neither CTA leaves while the other may still reach its barriers or accumulators
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * BN) : "memory");
  } else if (warp == 1) {
    ptx::tmem_dealloc(tmem, 2 * BN);
  }
}

// The splits' sums, in order, and the epilogue; 4 columns per thread (VEC: as vectors).
template <bool VEC>
__global__ void __launch_bounds__(256) split_epilogue_kernel(const GemmP p) {
  const int64_t cols = (p.N + 3) / 4;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= p.M * cols) return;
  const int64_t row = i / cols, col = (i - row * cols) * 4;
  if constexpr (VEC) {
    const float4* q = reinterpret_cast<const float4*>(p.part + row * p.N + col);
    float4 v = *q;
#pragma unroll 4
    for (int s = 1; s < p.splits; ++s) {
      const float4 w = q[(int64_t)s * p.M * p.N / 4];
      v.x += w.x; v.y += w.y; v.z += w.z; v.w += w.w;
    }
    f32x2 o[2] = {pack2(v.x, v.y), pack2(v.z, v.w)};
    auto put = [&](bf16* to) {
      const float2 a = unpack2(o[0]), b = unpack2(o[1]);
      const __nv_bfloat162 h[2] = {__floats2bfloat162_rn(a.x, a.y), __floats2bfloat162_rn(b.x, b.y)};
      *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(h);
    };
    auto add = [&](const bf16* from) {
      const uint2 r = *reinterpret_cast<const uint2*>(from);
      o[0] = add2(o[0], load_pair(reinterpret_cast<const bf16*>(&r)));
      o[1] = add2(o[1], load_pair(reinterpret_cast<const bf16*>(&r) + 2));
    };
    if (p.bias) add(p.bias + col);
    if (p.pre && !p.slope) put(p.pre + row * p.N + col);
    f32x2 d[2];
    o[0] = act_both2(o[0], p.act, d[0]);
    o[1] = act_both2(o[1], p.act, d[1]);
    if (p.pre && p.slope) *reinterpret_cast<uint2*>(p.pre + row * p.N + col) = make_uint2(slope_bits(d[0]), slope_bits(d[1]));
    if (p.res) add(p.res + row * p.ldr + col);
    put(p.y + row * p.ldy + col);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (col + k >= p.N) break;
      float v = 0.f;
      for (int s = 0; s < p.splits; ++s) v += p.part[((int64_t)s * p.M + row) * p.N + col + k];
      if (p.bias) v += to_f32(p.bias[col + k]);
      v = act_one(v, p.act, p.pre ? p.pre + row * p.N + col + k : nullptr, p.slope);
      if (p.res) v += to_f32(p.res[row * p.ldr + col + k]);
      p.y[row * p.ldy + col + k] = __float2bfloat16_rn(v);
    }
  }
}

// Few rows (M <= 16 MT; use_few): the weight is streamed once, straight into MMA fragments.  A block owns 8 columns of y and its
// 8 warps share the contraction; lane (g, q) reads 8 consecutive k of weight row g and of x rows g, g + 8 and the
// fragments take them in that order -- the contraction runs over the same permuted k on both sides.  The warps' sums
// are added in order in shared memory.
template <int MT, bool VEC>
__global__ void __launch_bounds__(256) few_rows_kernel(const GemmP p) {
  __shared__ float sums[8][MT * 16][8];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, q = lane % 4;
  const int64_t n0 = (int64_t)blockIdx.x * 8, n = n0 + g;
  float acc[MT][4];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[m][i] = 0.f;
  auto load8 = [&](const bf16* base, int64_t ld, int64_t r, int64_t rows, int64_t k) {
    uint4 raw = make_uint4(0, 0, 0, 0);
    if (r < rows) {
      const bf16* s = base + r * ld + k;
      if (VEC) {
        if (k < p.K) raw = *reinterpret_cast<const uint4*>(s);
      } else {
        bf16* e = reinterpret_cast<bf16*>(&raw);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (k + i < p.K) e[i] = s[i];
      }
    }
    return raw;
  };
#pragma unroll 4
  for (int64_t k = warp * 32 + q * 8; k - q * 8 < p.K; k += 256) {
    const uint4 w = load8(p.b.p, p.b.ld, n, p.N, k);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const uint4 x0 = load8(p.a.p, p.a.ld, m * 16 + g, p.M, k), x1 = load8(p.a.p, p.a.ld, m * 16 + g + 8, p.M, k);
      float(&d)[4] = acc[m];
      asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                   : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                   : "r"(x0.x), "r"(x1.x), "r"(x0.y), "r"(x1.y), "r"(w.x), "r"(w.y));
      asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                   : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                   : "r"(x0.z), "r"(x1.z), "r"(x0.w), "r"(x1.w), "r"(w.z), "r"(w.w));
    }
  }
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int i = 0; i < 4; ++i) sums[warp][m * 16 + g + i / 2 * 8][q * 2 + i % 2] = acc[m][i];
  __syncthreads();
  for (int i = threadIdx.x; i < MT * 128; i += 256) {
    const int64_t row = i / 8, col = n0 + i % 8;
    if (row >= p.M || col >= p.N) continue;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) v += sums[w][row][i % 8];
    if (p.bias) v += to_f32(p.bias[col]);
    v = act_one(v, p.act, p.pre ? p.pre + row * p.N + col : nullptr, p.slope);
    if (p.res) v += to_f32(p.res[row * p.ldr + col]);
    p.y[row * p.ldy + col] = __float2bfloat16_rn(v);
  }
}

// dp = dy act'(pre) (`slope`: pre holds act' itself, in fp16), with rows padded to a multiple of 8 values (zeros) so that TMA can address them, and the column
// sums of each block's DP_ROWS rows.
// A thread's loads of DP_BATCH rows go out together (16384 x 1024 with GELU: 21 us, 30 us where each row's store stood
// before the next row's loads).
constexpr int DP_ROWS = 64, DP_BATCH = 2;
template <bool VEC>
__global__ void __launch_bounds__(256) dp_kernel(const bf16* dy, int64_t ldd, const bf16* pre, bf16* dp, int64_t ldp, int64_t M, int64_t N,
                                                 int act, int slope, uint32_t col_blocks, float* colsum) {
  // 32 lanes x 8 columns, 8 row groups; the blocks of one group of DP_ROWS rows follow one another
  const int lane = threadIdx.x % 32, rg = threadIdx.x / 32;
  const uint32_t gr = blockIdx.x / col_blocks;
  const int64_t c0 = (int64_t)(blockIdx.x - gr * col_blocks) * 256, col = c0 + lane * 8, r0 = (int64_t)gr * DP_ROWS;
  f32x2 sum[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) sum[i] = both(0.f);
  auto load8 = [&](const bf16* row) {
    uint4 raw = make_uint4(0, 0, 0, 0);
    if (VEC) {
      if (col < N) raw = *reinterpret_cast<const uint4*>(row + col);
    } else {
      bf16* e = reinterpret_cast<bf16*>(&raw);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (col + i < N) e[i] = row[col + i];
    }
    return raw;
  };
  const int64_t r1 = min(r0 + DP_ROWS, M);
  auto walk = [&](int act, bool slope) {
    for (int64_t r = r0 + rg; r < r1; r += 8 * DP_BATCH) {
      uint4 rd[DP_BATCH], rp[DP_BATCH];
#pragma unroll
      for (int q = 0; q < DP_BATCH; ++q) {  // past the block's rows its last one again
        const int64_t u = min(r + 8 * q, r1 - 1);
        rd[q] = load8(dy + u * ldd);
        rp[q] = act != GDN_ACT_NONE ? load8(pre + u * N) : rd[q];
      }
#pragma unroll
      for (int q = 0; q < DP_BATCH; ++q) {
        if (r + 8 * q >= r1) break;
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          f32x2 d = load_pair(reinterpret_cast<const bf16*>(&rd[q]) + 2 * i);
          const uint32_t kept = reinterpret_cast<const uint32_t*>(&rp[q])[i];
          if (act != GDN_ACT_NONE) d = mul2(d, slope ? slope_pair(kept) : act_grad2(load_pair(reinterpret_cast<const bf16*>(&kept)), act));
          sum[i] = add2(sum[i], d);
          const float2 e = unpack2(d);
          const __nv_bfloat162 h = __floats2bfloat162_rn(e.x, e.y);
          w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
        if (dp && col < ldp) *reinterpret_cast<uint4*>(dp + (r + 8 * q) * ldp + col) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  };
  if (act == GDN_ACT_NONE) walk(GDN_ACT_NONE, false);
  else if (slope) walk(GDN_ACT_SILU, true);  // the same for every activation
  else if (act == GDN_ACT_SILU) walk(GDN_ACT_SILU, false);
  else walk(GDN_ACT_GELU, false);
  if (!colsum) return;
  __shared__ float part[8][256 + 8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 e = unpack2(sum[i]);
    part[rg][lane * 8 + 2 * i] = e.x;
    part[rg][lane * 8 + 2 * i + 1] = e.y;
  }
  __syncthreads();
  const int64_t c = c0 + threadIdx.x;
  if (c >= N) return;
  float a = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) a += part[i][threadIdx.x];
  colsum[gr * N + c] = a;
}

// Column sums of the partial rows, added in order: 32 columns x 8 groups of rows per block.
__global__ void __launch_bounds__(256) colsum_kernel(const float* part, int64_t rows, int64_t N, bf16* out) {
  __shared__ float s[8][32];
  const int lane = threadIdx.x % 32, g = threadIdx.x / 32;
  const int64_t i = (int64_t)blockIdx.x * 32 + lane;
  float a = 0.f;
  if (i < N) {
#pragma unroll 4
    for (int64_t r = g; r < rows; r += 8) a += part[r * N + i];
  }
  s[g][lane] = a;
  __syncthreads();
  if (g || i >= N) return;
#pragma unroll
  for (int k = 1; k < 8; ++k) a += s[k][lane];
  out[i] = __float2bfloat16_rn(a);
}

// ---- host -------------------------------------------------------------------------------------

int sm_count() {
  static std::atomic<int> cached[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 148;
  if (dev >= 0 && dev < 64) {
    const int c = cached[dev].load(std::memory_order_relaxed);
    if (c) return c;
  }
  int n = 0;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 1) return 148;
  if (dev >= 0 && dev < 64) cached[dev].store(n, std::memory_order_relaxed);
  return n;
}

bool rows16(const void* p, int64_t ld) { return ssm::aligned16(p) && ld % 8 == 0 && ld > 0; }

Operand operand(const void* p, int64_t ld, int64_t rows, int64_t cols) {
  return {static_cast<const bf16*>(p), ld, rows, cols, rows16(p, ld) ? 1 : 0};
}

// (cols, rows) map with boxes of 64 columns x box_rows rows, 128-byte swizzle, zeros outside.
bool make_map2(CUtensorMap* m, const Operand& o, int box_rows) {
  auto fn = tiles::encode_fn();
  if (!fn) return false;
  cuuint64_t dims[2] = {(cuuint64_t)o.cols, (cuuint64_t)o.rows};
  cuuint64_t strides[1] = {(cuuint64_t)o.ld * 2};
  cuuint32_t box[2] = {64, (cuuint32_t)box_rows};
  cuuint32_t es[2] = {1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<bf16*>(o.p), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// (N, M) map of an output, boxes of 64 columns x 32 rows.
bool make_out_map(CUtensorMap* m, bf16* p, int64_t ld, int64_t M, int64_t N) {
  memset(m, 0, sizeof(*m));
  return !p || make_map2(m, Operand{p, ld, M, N, 1}, 32);
}

size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

// (N, M, splits) map of the splits' sums, boxes of 32 x 32 fp32.
bool make_part_map(CUtensorMap* m, float* p, int64_t M, int64_t N, int64_t splits) {
  auto fn = tiles::encode_fn();
  if (!fn) return false;
  cuuint64_t dims[3] = {(cuuint64_t)N, (cuuint64_t)M, (cuuint64_t)splits};
  cuuint64_t strides[2] = {(cuuint64_t)N * 4, (cuuint64_t)(M * N) * 4};
  cuuint32_t box[3] = {32, 32, 1};
  cuuint32_t es[3] = {1, 1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, p, dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// CTA pairs that run at once (the same for every pair kernel: one CTA per SM), 0 where the device cannot say.
int pair_count() {
  static std::atomic<int> cached[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  const int c = cached[dev].load(std::memory_order_relaxed);
  if (c) return c - 1;
  using C = Cfg<256, true>;
  static std::atomic<unsigned long long> opted{0};
  auto k = gemm_kernel<256, false, false, true, false>;
  int n = 0;
  if (opt_in_smem(opted, {{(const void*)k, C::SMEM}})) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = C::SMEM;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = 2;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, k, &cfg) != cudaSuccess) {
      cudaGetLastError();
      n = 0;
    }
  }
  cached[dev].store(n + 1, std::memory_order_relaxed);
  return n;
}

struct Plan {
  int bn, splits, pairs;  // pairs: CTA pairs on 256 x 256 tiles
  size_t part;            // bytes
};

// Tile shape and splits of the contraction by a model of the time in SM clocks: waves of tiles, a k block taking 540, 300
// or 200 clocks with 256, 128 or 64 columns (the tensor pipe's 512 clocks, then the operands' way out of shared memory; a
// pair's 256 x 256 tile PAIR_CLOCKS) and a tile 2500 to start and drain; splits add their sums' way through memory (2 x 4
// bytes at 3400 bytes a clock) and a launch.
constexpr int PAIR_CLOCKS = 530;

Plan plan(int64_t M, int64_t N, int64_t K) {
  const int64_t sms = sm_count(), pairs = pair_count(), kb = (K + BK - 1) / BK;
  Plan best = {64, 1, 0, 0};
  double least = 1e300;
  const struct {
    int bm, bn, clocks;
    int64_t units;
  } shapes[] = {{256, 256, PAIR_CLOCKS, pairs}, {128, 256, 540, sms}, {128, 128, 300, sms}, {128, 64, 200, sms}};
  for (const auto& w : shapes) {
    if (w.units < 1) continue;
    const int64_t tiles = (M + w.bm - 1) / w.bm * ((N + w.bn - 1) / w.bn);
    for (int64_t s = 1; s <= 16; ++s) {
      if (s > 1 && (kb / s < 4 || tiles >= 4 * w.units)) break;
      const int64_t per = (kb + s - 1) / s, splits = (kb + per - 1) / per, waves = (tiles * splits + w.units - 1) / w.units;
      const double t = (double)waves * (double)(per * w.clocks + 2500) + (splits > 1 ? (double)splits * (double)(M * N) * 8 / 3400 + 6000 : 0);
      if (t < least) {
        least = t;
        best = {w.bn, (int)splits, w.bm == 256 ? (int)pairs : 0, 0};
      }
    }
  }
  if (best.splits > 1) best.part = up256((size_t)best.splits * M * N * sizeof(float));
  return best;
}

template <int BN, bool AMN, bool BMN, bool PAIR, bool SLOPE>
int launch_gemm(const GemmP& p, int pairs, cudaStream_t s) {
  using C = Cfg<BN, PAIR>;
  static std::atomic<unsigned long long> opted{0};
  auto k = gemm_kernel<BN, AMN, BMN, PAIR, SLOPE>;
  if (!opt_in_smem(opted, {{(const void*)k, C::SMEM}})) return GDN_ERR_LAUNCH;
  CUtensorMap ma, mb, my, mpre, mres;
  const bool out = p.vec && p.splits == 1;
  if (!make_map2(&ma, p.a, AMN ? BK : BM) || !make_map2(&mb, p.b, BMN ? BK : C::BROWS) || !make_out_map(&my, out ? p.y : nullptr, p.ldy, p.M, p.N) ||
      !make_out_map(&mpre, out ? p.pre : nullptr, p.N, p.M, p.N) || !make_out_map(&mres, out ? const_cast<bf16*>(p.res) : nullptr, p.ldr, p.M, p.N))
    return GDN_ERR_LAUNCH;
  if (p.part_tma && !make_part_map(&my, p.part, p.M, p.N, p.splits)) return GDN_ERR_LAUNCH;
  const int64_t items = (int64_t)p.tiles_m * p.tiles_n * p.splits;
  const int64_t units = PAIR ? pairs : sm_count();
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((items < units ? items : units) * (PAIR ? 2 : 1)));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = s;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = 2;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = PAIR ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, k, ma, mb, my, mpre, mres, p) == cudaSuccess ? ssm::launched() : GDN_ERR_LAUNCH;
}

// Bytes of an operand's aligned copy, 0 where it needs none, and the copy itself (which then stands for it).
size_t align_bytes(const Operand& o) { return o.tma ? 0 : up256((size_t)o.rows * ((o.cols + 7) / 8 * 8) * 2); }

struct Copies {
  struct {
    const bf16* src;
    int64_t ld;
    bf16* dst;
    int64_t rows, cols;
  } o[2];
};

// The operands' 16-byte pieces one after the other, one per thread; inside a row words of 4 bytes are read, shifted by one
// value where the row starts between two of them.  INDEX: an unsigned type that holds the number of pieces.
template <typename INDEX>
__global__ void __launch_bounds__(256) align_kernel(const Copies q) {
  INDEX i = (INDEX)blockIdx.x * 256 + threadIdx.x;
  const INDEX first = (INDEX)(q.o[0].rows * ((q.o[0].cols + 7) / 8));
  const bool other = i >= first;
  if (other) i -= first;
  const bf16* src = other ? q.o[1].src : q.o[0].src;
  bf16* dst = other ? q.o[1].dst : q.o[0].dst;
  const int64_t ld = other ? q.o[1].ld : q.o[0].ld, rows = other ? q.o[1].rows : q.o[0].rows, cols = other ? q.o[1].cols : q.o[0].cols;
  const INDEX pieces = (INDEX)((cols + 7) / 8);
  if (rows == 0 || i >= (INDEX)rows * pieces) return;
  const INDEX r = i / pieces;
  const int64_t c = (int64_t)(i - r * pieces) * 8;
  const bf16* s = src + (int64_t)r * ld + c;
  uint4 raw = make_uint4(0, 0, 0, 0);
  const bool odd = (uintptr_t)s & 2;
  if (!odd && c + 8 <= cols) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(s);
    raw = make_uint4(w[0], w[1], w[2], w[3]);
  } else if (odd && c > 0 && c + 9 <= cols) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(s - 1);
    const uint32_t v[5] = {w[0], w[1], w[2], w[3], w[4]};
    raw = make_uint4(__funnelshift_r(v[0], v[1], 16), __funnelshift_r(v[1], v[2], 16), __funnelshift_r(v[2], v[3], 16), __funnelshift_r(v[3], v[4], 16));
  } else {
    bf16* e = reinterpret_cast<bf16*>(&raw);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c + j < cols) e[j] = s[j];
  }
  reinterpret_cast<uint4*>(dst)[i] = raw;
}

// Those of the operands (second may be NULL) that TMA cannot address, laid out again in one launch.
int align_operands(Operand* first, Operand* second, char*& ws, cudaStream_t s) {
  Copies q = {};
  int n = 0;
  int64_t pieces = 0;
  for (Operand* o : {first, second}) {
    if (!o || o->tma) continue;
    q.o[n++] = {o->p, o->ld, reinterpret_cast<bf16*>(ws), o->rows, o->cols};
    pieces += o->rows * ((o->cols + 7) / 8);
    ws += align_bytes(*o);
    o->p = q.o[n - 1].dst;
    o->ld = (o->cols + 7) / 8 * 8;
    o->tma = 1;
  }
  if (!n) return GDN_OK;
  const int64_t g = (pieces + 255) / 256;
  if (g > 0x7fffffff) return GDN_ERR_SHAPE;
  if (pieces + 256 <= 0xffffffffll)
    align_kernel<uint32_t><<<(unsigned)g, 256, 0, s>>>(q);
  else
    align_kernel<uint64_t><<<(unsigned)g, 256, 0, s>>>(q);
  return ssm::launched();
}

template <bool AMN, bool BMN, bool SLOPE>
int launch_tiles(const GemmP& p, const Plan& pl, cudaStream_t s) {
  return pl.pairs      ? launch_gemm<256, AMN, BMN, true, SLOPE>(p, pl.pairs, s)
         : pl.bn == 256 ? launch_gemm<256, AMN, BMN, false, SLOPE>(p, 0, s)
         : pl.bn == 128 ? launch_gemm<128, AMN, BMN, false, SLOPE>(p, 0, s)
                        : launch_gemm<64, AMN, BMN, false, SLOPE>(p, 0, s);
}

// C[M, N] = sum_k A B with the epilogue of p; `ws` holds plan().part bytes.
template <bool AMN, bool BMN>
int gemm(GemmP p, void* ws, cudaStream_t s) {
  const Plan pl = plan(p.M, p.N, p.K);
  const int bm = pl.pairs ? 2 * BM : BM;
  const int64_t tm = (p.M + bm - 1) / bm, tn = (p.N + pl.bn - 1) / pl.bn;
  if (tm * tn * pl.splits > 0x7fffffff) return GDN_ERR_SHAPE;
  p.tiles_m = (int)tm;
  p.tiles_n = (int)tn;
  p.n_first = tn <= tm;
  p.splits = pl.splits;
  p.kblocks = (int)((p.K + BK - 1) / BK);
  p.part = static_cast<float*>(ws);
  p.part_tma = p.splits > 1 && p.N % 4 == 0;
  p.vec = rows16(p.y, p.ldy) && p.N % 8 == 0 && (!p.bias || ssm::aligned16(p.bias)) && (!p.res || rows16(p.res, p.ldr)) && (!p.pre || rows16(p.pre, p.N));
  int st;
  if constexpr (!AMN && !BMN)
    st = p.slope && p.splits == 1 ? launch_tiles<AMN, BMN, true>(p, pl, s) : launch_tiles<AMN, BMN, false>(p, pl, s);
  else
    st = launch_tiles<AMN, BMN, false>(p, pl, s);
  if (st != GDN_OK || p.splits == 1) return st;
  const int64_t g = (p.M * ((p.N + 3) / 4) + 255) / 256;
  if (g > 0x7fffffff) return GDN_ERR_SHAPE;
  p.vec ? split_epilogue_kernel<true><<<(unsigned)g, 256, 0, s>>>(p) : split_epilogue_kernel<false><<<(unsigned)g, 256, 0, s>>>(p);
  return ssm::launched();
}

// Vector loads of the few-rows kernel.
bool few_vec(const Operand& a, const Operand& b) { return a.tma && b.tma && a.cols % 8 == 0; }

// Where the few-rows kernel serves.  It needs one launch, no tensor maps and no workspace, which saves the host about 5 us a call,
// but each of its warps walks an eighth of the contraction (12.5 us for 4096 values at 16 rows) and every 8 columns read all of x
// again.  So the tiles take over where they save some 3 us on the device.  Few rows / tiles in us there, weights out of HBM, x in
// L2 (N x K, aligned):
//   16 rows: 1024 x 1024 3.1 / 7.2, 1024 x 2816 9.6 / 9.7, 1024 x 4096 12.7 / 10.4, 4096 x 4096 13.8 / 13.1, 256 x 8192 22.5 / 10.1,
//            12288 x 2048 15.5 / 19.1, 32768 x 1024 21.0 / 18.1, 50304 x 1024 31.1 / 27.3, 65536 x 64 13.0 / 8.9
//   32 rows: 2048 x 2048 9.8 / 11.1, 4096 x 2048 10.1 / 11.1, 8192 x 1024 11.5 / 10.0, 8192 x 2048 19.4 / 11.5, 1024 x 2560 12.1 / 8.8
//            (14.7 / 8.7 with x out of HBM too), 16384 x 512 10.9 / 8.2, 32768 x 256 13.6 / 8.8
//   64 rows: 1024 x 1024 4.9 / 7.2, 1024 x 1536 8.1 / 9.1, 768 x 2048 9.9 / 10.7, 1024 x 2048 11.5 / 11.0 (x out of HBM: 15.7 / 11.0),
//            2560 x 1024 12.1 / 7.9, 4096 x 4096 38.9 / 17.6, 8192 x 64 6.7 / 4.4, 16384 x 64 11.1 / 4.8
// Rows that no vector takes (the tiles then wait for their aligned copies, the few-rows kernel loads single values):
//   16 rows: 1001 x 2047 13.6 / 14.8, 8191 x 513 10.7 / 15.8; 32 rows: 501 x 999 10.5 / 11.0, 4095 x 1023 17.0 / 14.2,
//            1001 x 2047 21.8 / 15.5; 64 rows: 501 x 999 19.5 / 11.2, 8191 x 513 27.6 / 15.9
bool use_few(int64_t M, int64_t N, const Operand& a, const Operand& b) {
  const int64_t K = a.cols;
  const bool vec = few_vec(a, b);
  if (M <= 16) return K <= (vec ? 4608 : 2560) && N <= 32768;
  if (M <= 32) return K <= (vec ? 2048 : 1280) && N <= 16384 && N * K <= 1 << 23;
  return M <= 64 && K <= (vec ? 2048 : 640) && N <= 8192 && N * K <= 3 << 19;
}

int launch_few(const GemmP& p, cudaStream_t s) {
  const unsigned g = (unsigned)((p.N + 7) / 8);
  const bool v = few_vec(p.a, p.b);
  if (p.M <= 16)
    v ? few_rows_kernel<1, true><<<g, 256, 0, s>>>(p) : few_rows_kernel<1, false><<<g, 256, 0, s>>>(p);
  else if (p.M <= 32)
    v ? few_rows_kernel<2, true><<<g, 256, 0, s>>>(p) : few_rows_kernel<2, false><<<g, 256, 0, s>>>(p);
  else
    v ? few_rows_kernel<4, true><<<g, 256, 0, s>>>(p) : few_rows_kernel<4, false><<<g, 256, 0, s>>>(p);
  return ssm::launched();
}

int check_sizes(int64_t M, int64_t N, int64_t K, int act, int keep) {
  if (M < 0 || N < 1 || K < 1 || M > (1 << 30) || N > (1 << 30) || K > (1 << 30)) return GDN_ERR_SHAPE;
  if (act != GDN_ACT_NONE && act != GDN_ACT_SILU && act != GDN_ACT_GELU) return GDN_ERR_UNSUPPORTED;
  if (keep != GDN_LINEAR_KEEP_PRE && keep != GDN_LINEAR_KEEP_SLOPE) return GDN_ERR_UNSUPPORTED;
  return GDN_OK;
}

struct BwdPlan {
  int64_t ldp;       // row length of dp, 0 when dy itself serves
  size_t dp, colsum, x, w, part, total;  // bytes; x and w: their aligned copies
};

BwdPlan bwd_plan(const gdn_linear_bwd_args* a) {
  BwdPlan w = {};
  const bool copy = a->act != GDN_ACT_NONE || !rows16(a->dy, a->sdy);
  if (copy) {
    w.ldp = (a->N + 7) / 8 * 8;
    w.dp = up256((size_t)a->M * w.ldp * 2);
  }
  if (a->dweight) w.x = align_bytes(operand(a->x, a->sx, a->M, a->K));
  if (a->dx) w.w = align_bytes(operand(a->weight, a->sw, a->N, a->K));
  if (a->dbias) w.colsum = up256((size_t)((a->M + DP_ROWS - 1) / DP_ROWS) * a->N * 4);
  if (a->dx) w.part = plan(a->M, a->K, a->N).part;
  if (a->dweight) {
    const size_t q = plan(a->N, a->K, a->M).part;
    if (q > w.part) w.part = q;
  }
  w.total = w.dp + w.colsum + w.x + w.w + w.part;
  return w;
}

}  // namespace linear
}  // namespace gdn

using namespace gdn;
using namespace gdn::linear;

int gdn_linear_read_status(int* out, int reset) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, gdn::linear::g_status, sizeof(int)) != cudaSuccess) return GDN_ERR_LAUNCH;
  if (reset) {
    const int z = 0;
    if (cudaMemcpyToSymbol(gdn::linear::g_status, &z, sizeof(int)) != cudaSuccess) return GDN_ERR_LAUNCH;
  }
  *out = v;
  return GDN_OK;
}

extern "C" {

int gdn_linear_workspace_bytes(const gdn_linear_args* a, size_t* bytes) {
  if (!a || !bytes) return GDN_ERR_NULL;
  const int st = check_sizes(a->M, a->N, a->K, a->act, a->keep);
  if (st != GDN_OK) return st;
  const Operand x = operand(a->x, a->sx, a->M, a->K), w = operand(a->weight, a->sw, a->N, a->K);
  *bytes = a->M == 0 || use_few(a->M, a->N, x, w) ? 0 : plan(a->M, a->N, a->K).part + align_bytes(x) + align_bytes(w);
  return GDN_OK;
}

int gdn_linear_fwd(const gdn_linear_args* a, void* stream) {
  size_t need = 0;
  int st = gdn_linear_workspace_bytes(a, &need);
  if (st != GDN_OK) return st;
  if (a->M == 0) return GDN_OK;
  if (!a->x || !a->weight || !a->y) return GDN_ERR_NULL;
  if (a->sx < 0 || a->sw < 0 || a->sr < 0 || a->sy < 0) return GDN_ERR_SHAPE;
  if (need && (!a->workspace || a->workspace_bytes < need)) return GDN_ERR_WORKSPACE;
  if (need && !ssm::aligned16(a->workspace)) return GDN_ERR_ALIGN;
  if (!ssm::device_ok()) return GDN_ERR_DEVICE;
  GemmP p = {};
  p.a = operand(a->x, a->sx, a->M, a->K);
  p.b = operand(a->weight, a->sw, a->N, a->K);
  p.M = a->M; p.N = a->N; p.K = a->K;
  p.y = static_cast<bf16*>(a->y); p.ldy = a->sy; p.pre = static_cast<bf16*>(a->pre);
  p.bias = static_cast<const bf16*>(a->bias); p.res = static_cast<const bf16*>(a->residual); p.ldr = a->sr;
  p.act = a->act;
  p.slope = p.pre && a->keep == GDN_LINEAR_KEEP_SLOPE && a->act != GDN_ACT_NONE;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (use_few(p.M, p.N, p.a, p.b)) return launch_few(p, s);
  char* ws = static_cast<char*>(a->workspace);
  st = align_operands(&p.a, &p.b, ws, s);
  return st == GDN_OK ? gemm<false, false>(p, ws, s) : st;
}

int gdn_linear_bwd_workspace_bytes(const gdn_linear_bwd_args* a, size_t* bytes) {
  if (!a || !bytes) return GDN_ERR_NULL;
  const int st = check_sizes(a->M, a->N, a->K, a->act, a->keep);
  if (st != GDN_OK) return st;
  *bytes = bwd_plan(a).total;
  return GDN_OK;
}

int gdn_linear_bwd(const gdn_linear_bwd_args* a, void* stream) {
  size_t need = 0;
  int st = gdn_linear_bwd_workspace_bytes(a, &need);
  if (st != GDN_OK) return st;
  if (a->M == 0) return GDN_ERR_SHAPE;  // nothing flowed; the caller zeroes the gradients
  if (!a->dy || (a->act != GDN_ACT_NONE && !a->pre) || (a->dx && !a->weight) || (a->dweight && !a->x)) return GDN_ERR_NULL;
  if (a->sx < 0 || a->sw < 0 || a->sdy < 0) return GDN_ERR_SHAPE;
  if (need && (!a->workspace || a->workspace_bytes < need)) return GDN_ERR_WORKSPACE;
  if (need && !ssm::aligned16(a->workspace)) return GDN_ERR_ALIGN;
  if (!ssm::device_ok()) return GDN_ERR_DEVICE;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const BwdPlan w = bwd_plan(a);
  char* ws = static_cast<char*>(a->workspace);
  bf16* dp = w.ldp ? reinterpret_cast<bf16*>(ws) : nullptr;
  float* colsum = a->dbias ? reinterpret_cast<float*>(ws + w.dp) : nullptr;
  char* copies = ws + w.dp + w.colsum;
  void* part = copies + w.x + w.w;
  if (dp || colsum) {
    const int64_t gx = ((dp ? w.ldp : a->N) + 255) / 256, gy = (a->M + DP_ROWS - 1) / DP_ROWS;
    if (gx * gy > 0x7fffffff) return GDN_ERR_SHAPE;  // 2^45 values of dy: past any memory
    const unsigned g = (unsigned)(gx * gy);
    const bf16 *dy = static_cast<const bf16*>(a->dy), *pre = static_cast<const bf16*>(a->pre);
    if (a->N % 8 == 0 && rows16(dy, a->sdy) && (a->act == GDN_ACT_NONE || ssm::aligned16(pre)))
      dp_kernel<true><<<g, 256, 0, s>>>(dy, a->sdy, pre, dp, w.ldp, a->M, a->N, a->act, a->keep, (uint32_t)gx, colsum);
    else
      dp_kernel<false><<<g, 256, 0, s>>>(dy, a->sdy, pre, dp, w.ldp, a->M, a->N, a->act, a->keep, (uint32_t)gx, colsum);
    if (colsum) colsum_kernel<<<(unsigned)((a->N + 31) / 32), 256, 0, s>>>(colsum, gy, a->N, static_cast<bf16*>(a->dbias));
    st = ssm::launched();
    if (st != GDN_OK) return st;
  }
  const Operand d = dp ? operand(dp, w.ldp, a->M, a->N) : operand(a->dy, a->sdy, a->M, a->N);
  GemmP p = {};
  p.act = GDN_ACT_NONE;
  if (a->dx) {  // (M, K) = dp (M, N) W (N, K)
    p.a = d;
    p.b = operand(a->weight, a->sw, a->N, a->K);
    p.M = a->M; p.N = a->K; p.K = a->N;
    p.y = static_cast<bf16*>(a->dx); p.ldy = a->K;
    st = align_operands(&p.b, nullptr, copies, s);
    if (st == GDN_OK) st = gemm<false, true>(p, part, s);
    if (st != GDN_OK) return st;
  }
  if (a->dweight) {  // (N, K) = dp^T (N, M) x (M, K)
    p.a = d;
    p.b = operand(a->x, a->sx, a->M, a->K);
    p.M = a->N; p.N = a->K; p.K = a->M;
    p.y = static_cast<bf16*>(a->dweight); p.ldy = a->K;
    st = align_operands(&p.b, nullptr, copies, s);
    if (st == GDN_OK) st = gemm<true, true>(p, part, s);
  }
  return st;
}

}  // extern "C"
