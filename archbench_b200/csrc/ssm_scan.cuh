// What the selective scan's forward and backward kernels share: parameters, the thread layout and the lane
// reductions.
//
// Layout: NL = 2, 4, 8 or 16 consecutive lanes hold one channel's states, four each; a warp
// walks 32 / NL channels through time together.  Work per token and channel (step size, gate) is done once, by the
// threads that stage the tile in shared memory; work per state is one multiply, one exponential (exp(s A) as
// 2^(s A log2 e)), one multiply and two FMAs.  Sums over a channel's states go across its NL lanes for NL tokens at a
// time, each lane keeping the sum of one token (NL - 1 shuffles for NL tokens).
#pragma once

#include <type_traits>

#include "ssm_common.cuh"

namespace gdn {
namespace ssm {

constexpr int SCAN_THREADS = 128;
constexpr int SPL = 4;  // states per lane

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
  int quads;  // rows of B and C can be loaded four states at a time
  int nseg, seg_len;  // segments of seg_len tokens (a multiple of GDN_SCAN_CKPT)
  int dblocks;        // channel blocks per group
  int xgs;            // channels from one group to the next in x, dt, z and dy (padded copies have more than D / G)
  int tiled;          // the kernels on asynchronous tiles serve it (scan_align_plan)
  int pairs_out;      // rows of y (or dx, ddt, dz) take stores of channel pairs
  int ckpt_quads;     // rows of ckpt take stores of four states
};

// Two neighbouring values in one store.  (Written out by type: as one struct aligned to 2 * sizeof(T) the compiler ordered the
// backward otherwise, and the training step of 8 x 2048 x 2048 took 1,099 us for 1,068.)
template <typename T>
struct Pair;
template <>
struct __align__(4) Pair<__nv_bfloat16> {
  __nv_bfloat16 v[2];
};
template <>
struct __align__(8) Pair<float> {
  float v[2];
};
template <typename T>
__device__ __forceinline__ void store_pair(T* p, const float (&f)[2]) {
  Pair<T> r;
#pragma unroll
  for (int i = 0; i < 2; ++i) store_as(&r.v[i], f[i]);
  *reinterpret_cast<Pair<T>*>(p) = r;
}

// Four consecutive states of B or C at one token: one load where rows allow, else one by one, zeros past N.
template <typename T>
struct Quad {
  T v[4];
};
template <typename T>
__device__ __forceinline__ Quad<T> load_quad(const T* p, int n, int N, bool vec) {
  Quad<T> q;
  if (vec && n < N) {  // N is a multiple of four
    if constexpr (sizeof(T) == 4)
      *reinterpret_cast<float4*>(&q) = *reinterpret_cast<const float4*>(p + n);
    else
      *reinterpret_cast<uint2*>(&q) = *reinterpret_cast<const uint2*>(p + n);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      store_as(&q.v[i], 0.f);
      if (n + i < N) q.v[i] = p[n + i];
    }
  }
  return q;
}
template <typename T>
__device__ __forceinline__ float4 quad_f32(const Quad<T>& q, bool on) {
  return on ? make_float4(to_f32(q.v[0]), to_f32(q.v[1]), to_f32(q.v[2]), to_f32(q.v[3])) : make_float4(0.f, 0.f, 0.f, 0.f);
}

// exp(s A) with A2 = A log2 e.  The instruction's mean error is -1 to -2.5 parts in 10^8 for exponents from -1e-3 to -1;
// over the hundreds of tokens that slow states remember it adds up (dA came out 1.1e-6 low), so it is taken out of the
// exponent, at no cost.  2^EX2_MEAN itself is exactly 1: a step of size 0 still leaves the state alone.
constexpr float EX2_MEAN = 2.2e-8f;
__device__ __forceinline__ float decay(float s, float A2) { return ex2(fmaf(s, A2, EX2_MEAN)); }

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

// Rows are the last dimension of a grid, which ends at 65535: launch(q, rows) with q moved on to the next rows, as often as it
// takes.  (A first row that the kernels add cost them up to 7 % by another order of their instructions.)
template <typename F>
void for_grid_rows(const ScanP& p, int es, F launch) {
  constexpr int MOST = 65535;
  ScanP q = p;
  for (int64_t b = 0; b < p.B; b += MOST) {
    if (b) {
      auto token = [&](auto*& t, int64_t step) { if (t) t = (std::remove_reference_t<decltype(t)>)((const char*)t + MOST * step * es); };
      auto state = [&](auto*& t, int64_t step) { if (t) t += MOST * step; };
      const int64_t td = (int64_t)p.T * p.D, dn = (int64_t)p.D * p.N, sdn = p.nseg * dn, sd = (int64_t)p.nseg * p.D;
      token(q.x, p.sx_b); token(q.dt, p.sdt_b); token(q.Bm, p.sB_b); token(q.Cm, p.sC_b); token(q.z, p.sz_b); token(q.dy, p.sdy_b);
      token(q.y, p.sy_b); token(q.dx, td); token(q.ddt, td); token(q.dz, td);
      state(q.h0, dn); state(q.dh_out, dn); state(q.h_out, dn); state(q.dh0, dn); state(q.lengths, 1);
      state(q.ckpt, (p.T + GDN_SCAN_CKPT - 1) / GDN_SCAN_CKPT * dn);
      state(q.carry, sdn); state(q.ssum, sd); state(q.pA, sdn); state(q.pD, 2 * sd);
      state(q.pBC, (int64_t)p.T * p.G * 2 * p.N);  // its rows lie p.B apart still
    }
    launch(q, (unsigned)(p.B - b < MOST ? p.B - b : MOST));
  }
}

// Segments of time, each at least MIN_SEG tokens.
struct SegPlan {
  int nseg, seg_len;
};
SegPlan scan_segments(int64_t B, int64_t T, int64_t warps_per_row);

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

// Rows that 16-byte copies cannot take are first laid out again, padded, in the workspace: about 4 bytes moved per value
// against the kernels' 30 to 100 us per million values.  Tensors that are aligned stay where they are.
struct AlignPlan {
  bool tiled;           // the kernels on asynchronous tiles serve it: N a multiple of four, states on 16-byte boundaries
  bool x, dt, z, dy, B, C;
  size_t xb, bb;        // bytes of one copied channel tensor, of one copied B or C
  size_t total;
};
AlignPlan scan_align_plan(const ScanP& p, int es, bool bwd);
int scan_align(ScanP& p, const AlignPlan& a, int dtype, char* ws, cudaStream_t s);
// Local pass over every segment (forward, or reversed for the adjoint) and the combination of the segments: fills
// p.carry with the state that enters each segment, from p.h0 (p.dh_out).
int scan_launch_carry(const ScanP& p, int dtype, bool reverse, cudaStream_t s);

}  // namespace ssm
}  // namespace gdn
