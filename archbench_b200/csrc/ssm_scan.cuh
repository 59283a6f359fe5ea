// What the selective scan's forward and backward kernels share: parameters, the thread layout and the lane
// reductions.
//
// Layout: NL = 2, 4, 8 or 16 consecutive lanes hold one channel's states, four each; a warp
// walks 32 / NL channels through time together.  Work per token and channel (step size, gate) is done once, by the
// threads that stage the tile in shared memory; work per state is one multiply, one exponential (exp(s A) as
// 2^(s A log2 e)), one multiply and two FMAs.  Sums over a channel's states go across its NL lanes for NL tokens at a
// time, each lane keeping the sum of one token (NL - 1 shuffles for NL tokens).
#pragma once

#include "ssm_common.cuh"

namespace gdn {
namespace ssm {

constexpr int SCAN_THREADS = 128;
constexpr int SPL = 4;  // states per lane
constexpr float LOG2E = 1.44269504088896340736f;

struct ScanP {
  const void *x, *dt, *Bm, *Cm, *z, *dy;
  const float *A, *Dskip, *dt_bias, *h0, *dh_out;
  const int32_t* lengths;
  void *y, *dx, *ddt, *dz;
  float *h_out, *ckpt, *dh0;
  float* carry;  // (B, nseg, D, N): local end state of each segment, then the state that enters it
  float* ssum;   // (B, nseg, D): sum of the segment's step sizes
  float *pBC;    // backward: (D blocks, B, T, 2, N) partial sums of dB and dC
  float *pA;     // backward: (B * nseg, D, N) partial sums of dA
  float *pD;     // backward: (B * nseg, 2, D) partial sums of dDskip and ddt_bias
  int64_t sx_b, sx_t, sdt_b, sdt_t, sB_b, sB_t, sB_g, sC_b, sC_t, sC_g, sz_b, sz_t, sy_b, sy_t, sdy_b, sdy_t;
  int B, T, D, N, G;
  int softplus;
  int nseg, seg_len;  // segments of seg_len tokens (a multiple of GDN_SCAN_CKPT)
  int dblocks;        // channel blocks per group
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// v[i], i < NV, held by LANES lanes (stride STRIDE in lane index): sums over the lanes, spread so that lane l keeps
// the sums i = l * NV / LANES ..; with fewer values than lanes, every lane keeps one (equal on LANES / NV of them).
// On return v[0 .. max(NV / LANES, 1)) hold them and `first` is the index of v[0].
template <int NV, int LANES, int STRIDE>
__device__ __forceinline__ int spread_sum(float (&v)[NV], int lane) {
  int first = 0;
  int n = NV;
#pragma unroll
  for (int l = LANES / 2; l >= 1; l /= 2) {
    const int mask = l * STRIDE;
    const bool up = (lane & mask) != 0;
    if (n > 1) {
      n /= 2;
#pragma unroll
      for (int i = 0; i < NV / 2; ++i) {
        if (i < n) {
          const float keep = up ? v[i + n] : v[i], send = up ? v[i] : v[i + n];
          v[i] = keep + __shfl_xor_sync(0xffffffffu, send, mask);
        }
      }
      first += up ? n : 0;
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], mask);
    }
  }
  return first;
}

// Segments: as many as fill the device when B x channel blocks do not, each of at least MIN_SEG tokens.
struct SegPlan {
  int nseg, seg_len;
};
SegPlan scan_segments(int64_t B, int64_t T, int64_t blocks_per_row);

// Lanes per channel: 2, 4, 8 or 16 for N up to 8, 16, 32, 64.
inline int scan_lanes(int64_t N) {
  int nl = 2;
  while (nl * SPL < N) nl *= 2;
  return nl;
}
inline int scan_dblocks(int64_t D, int64_t G, int64_t N) {
  const int ch = SCAN_THREADS / scan_lanes(N);
  return (int)((D / G + ch - 1) / ch);
}

int scan_check(const gdn_scan_args* a, bool step);
ScanP scan_params(const gdn_scan_args* a);
// Local pass over every segment (forward, or reversed for the adjoint) and the combination of the segments: fills
// p.carry with the state that enters each segment, from p.h0 (p.dh_out).
int scan_launch_carry(const ScanP& p, int dtype, bool reverse, cudaStream_t s);

}  // namespace ssm
}  // namespace gdn
