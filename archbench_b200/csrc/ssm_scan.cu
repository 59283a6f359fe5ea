// Selective scan, forward: prompts (one pass, or split over time when the batch has few rows) and single tokens.
//
//   s_t = softplus(dt_t + bias), h_t = exp(s_t A) h_{t-1} + s_t x_t B_t, y_t = (C_t . h_t + D x_t) silu(z_t)
//
// Bound by the exponentials: N of them per token and channel on 16 lanes per SM and clock, against 8 bytes of HBM
// traffic (bf16).  The state stays in registers for the whole sequence.
#include "ssm_scan.cuh"

namespace gdn {
namespace ssm {

constexpr int TT = 32;  // tokens per tile

// One (row, channel block, segment) per block of 128 threads.
template <typename T, int NL>
__global__ void __launch_bounds__(SCAN_THREADS) scan_fwd_kernel(ScanP p) {
  constexpr int CH = SCAN_THREADS / NL, NP = NL * SPL, PER = TT * CH / SCAN_THREADS;
  __shared__ float2 sS[TT][CH];   // step size, step size * x
  __shared__ float sY[TT][CH + 1];
  __shared__ __align__(16) float sB[TT][NP], sC[TT][NP];
  const int tid = threadIdx.x, lane = tid % 32;
  const int grp = blockIdx.x / p.dblocks, dblk = blockIdx.x % p.dblocks;
  const int seg = blockIdx.y, b = blockIdx.z;
  const int dpg = p.D / p.G, d0 = grp * dpg + dblk * CH, nch = min(CH, dpg - dblk * CH);
  const int len = row_tokens(p.lengths, b, p.T);
  const int tbeg = seg * p.seg_len, tend = min(tbeg + p.seg_len, p.T);

  // per-state role
  const int hc = tid / NL, n0 = (tid % NL) * SPL;
  const bool live = hc < nch;
  float h[SPL], A2[SPL];
#pragma unroll
  for (int i = 0; i < SPL; ++i) {
    const bool ok = live && n0 + i < p.N;
    const int64_t at = (int64_t)(d0 + hc) * p.N + n0 + i;
    A2[i] = ok ? p.A[at] * LOG2E : 0.f;
    const float* from = p.nseg > 1 ? p.carry + ((int64_t)b * p.nseg + seg) * p.D * p.N : p.h0 ? p.h0 + (int64_t)b * p.D * p.N : nullptr;
    h[i] = ok && from ? from[at] : 0.f;
  }
  // per-token role: one channel, tokens ct0, ct0 + NL, ...
  const int cc = tid % CH, ct0 = tid / CH;
  const bool cok = cc < nch;
  const int d = d0 + (cok ? cc : 0);
  const float bias = p.dt_bias ? p.dt_bias[d] : 0.f, skip = p.Dskip ? p.Dskip[d] : 0.f;
  const T* xp = static_cast<const T*>(p.x) + b * p.sx_b + d;
  const T* dtp = static_cast<const T*>(p.dt) + b * p.sdt_b + d;
  const T* zp = p.z ? static_cast<const T*>(p.z) + b * p.sz_b + d : nullptr;
  T* yp = static_cast<T*>(p.y) + b * p.sy_b + d;
  const T* Bp = static_cast<const T*>(p.Bm) + b * p.sB_b + grp * p.sB_g;
  const T* Cp = static_cast<const T*>(p.Cm) + b * p.sC_b + grp * p.sC_g;
  const int nck = (p.T + GDN_SCAN_CKPT - 1) / GDN_SCAN_CKPT;

  for (int t0 = tbeg; t0 < tend; t0 += TT) {
    float xr[PER], zr[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int r = ct0 + i * NL, t = t0 + r;
      float s = 0.f;
      xr[i] = zr[i] = 0.f;
      if (cok && t < len && t < tend) {
        xr[i] = to_f32(xp[t * p.sx_t]);
        s = to_f32(dtp[t * p.sdt_t]) + bias;
        if (p.softplus) s = softplus(s);
        if (zp) zr[i] = to_f32(zp[t * p.sz_t]);
      }
      sS[r][cc] = make_float2(s, s * xr[i]);
    }
    for (int i = tid; i < TT * NP; i += SCAN_THREADS) {
      const int r = i / NP, n = i % NP, t = t0 + r;
      const bool ok = n < p.N && t < len && t < tend;
      sB[r][n] = ok ? to_f32(Bp[t * p.sB_t + n]) : 0.f;
      sC[r][n] = ok ? to_f32(Cp[t * p.sC_t + n]) : 0.f;
    }
    __syncthreads();
    const int rows = min(TT, tend - t0);
#pragma unroll 1
    for (int r0 = 0; r0 < TT; r0 += 16) {
      if (r0 >= rows) break;
      if (p.ckpt && live) {
#pragma unroll
        for (int i = 0; i < SPL; ++i)
          if (n0 + i < p.N)
            p.ckpt[(((int64_t)b * nck + (t0 + r0) / GDN_SCAN_CKPT) * p.D + d0 + hc) * p.N + n0 + i] = h[i];
      }
#pragma unroll
      for (int q = 0; q < 16; q += NL) {
        float acc[NL];
#pragma unroll
        for (int j = 0; j < NL; ++j) {
          const int r = r0 + q + j;
          const float2 ss = sS[r][hc];
          const float4 bv = *reinterpret_cast<const float4*>(&sB[r][n0]);
          const float4 cv = *reinterpret_cast<const float4*>(&sC[r][n0]);
          const float bb[4] = {bv.x, bv.y, bv.z, bv.w}, cq[4] = {cv.x, cv.y, cv.z, cv.w};
          float a = 0.f;
#pragma unroll
          for (int i = 0; i < SPL; ++i) {
            h[i] = fmaf(ex2(ss.x * A2[i]), h[i], ss.y * bb[i]);
            a = fmaf(cq[i], h[i], a);
          }
          acc[j] = a;
        }
        const int j = spread_sum<NL, NL, 1>(acc, lane);
        sY[r0 + q + j][hc] = acc[0];
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int r = ct0 + i * NL, t = t0 + r;
      if (!cok || t >= tend) continue;
      float y = fmaf(skip, xr[i], sY[r][cc]);
      if (zp) y *= silu(zr[i]);
      store_as(yp + t * p.sy_t, t < len ? y : 0.f);
    }
    // sS, sB and sC are rewritten only after every thread passed the barrier above; sY only after the next one
  }
  if (p.h_out && seg == p.nseg - 1 && live) {
#pragma unroll
    for (int i = 0; i < SPL; ++i)
      if (n0 + i < p.N) p.h_out[((int64_t)b * p.D + d0 + hc) * p.N + n0 + i] = h[i];
  }
}

// Local pass over one segment from a zero state: its end state and the sum of its step sizes (the segment's decay is
// exp(A sum s)).  Reversed for the adjoint: G <- exp(s_t A) (G + C_t dc_t), from the last token to the first, with
// dc = dy silu(z).
template <typename T, int NL, bool REV>
__global__ void __launch_bounds__(SCAN_THREADS) scan_carry_kernel(ScanP p) {
  constexpr int CH = SCAN_THREADS / NL, NP = NL * SPL, PER = TT * CH / SCAN_THREADS;
  __shared__ float2 sS[TT][CH];  // step size, step size * x (reversed: dc)
  __shared__ __align__(16) float sB[TT][NP];
  __shared__ float sSum[NL][CH];
  const int tid = threadIdx.x;
  const int grp = blockIdx.x / p.dblocks, dblk = blockIdx.x % p.dblocks;
  const int seg = blockIdx.y, b = blockIdx.z;
  if (seg == (REV ? 0 : p.nseg - 1)) return;  // nothing enters from here
  const int dpg = p.D / p.G, d0 = grp * dpg + dblk * CH, nch = min(CH, dpg - dblk * CH);
  const int len = row_tokens(p.lengths, b, p.T);
  const int tbeg = seg * p.seg_len, tend = min(min(tbeg + p.seg_len, p.T), len);
  const int hc = tid / NL, n0 = (tid % NL) * SPL;
  float h[SPL], A2[SPL];
#pragma unroll
  for (int i = 0; i < SPL; ++i) {
    h[i] = 0.f;
    A2[i] = hc < nch && n0 + i < p.N ? p.A[(int64_t)(d0 + hc) * p.N + n0 + i] * LOG2E : 0.f;
  }
  const int cc = tid % CH, ct0 = tid / CH;
  const bool cok = cc < nch;
  const int d = d0 + (cok ? cc : 0);
  const float bias = p.dt_bias ? p.dt_bias[d] : 0.f;
  const T* xp = static_cast<const T*>(REV ? p.dy : p.x) + b * (REV ? p.sdy_b : p.sx_b) + d;
  const int64_t sx = REV ? p.sdy_t : p.sx_t;
  const T* dtp = static_cast<const T*>(p.dt) + b * p.sdt_b + d;
  const T* zp = REV && p.z ? static_cast<const T*>(p.z) + b * p.sz_b + d : nullptr;
  const T* Bp = REV ? static_cast<const T*>(p.Cm) + b * p.sC_b + grp * p.sC_g : static_cast<const T*>(p.Bm) + b * p.sB_b + grp * p.sB_g;
  const int64_t sb = REV ? p.sC_t : p.sB_t;
  float total = 0.f;
  const int ntile = tend > tbeg ? (tend - tbeg + TT - 1) / TT : 0;
  for (int k = 0; k < ntile; ++k) {
    const int t0 = tbeg + (REV ? ntile - 1 - k : k) * TT;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int r = ct0 + i * NL, t = t0 + r;
      float s = 0.f, u = 0.f;
      if (cok && t < tend) {
        u = to_f32(xp[t * sx]);
        s = to_f32(dtp[t * p.sdt_t]) + bias;
        if (p.softplus) s = softplus(s);
        if (REV && zp) u *= silu(to_f32(zp[t * p.sz_t]));
        if (!REV) u *= s;
      }
      total += s;
      sS[r][cc] = make_float2(s, u);
    }
    for (int i = tid; i < TT * NP; i += SCAN_THREADS) {
      const int r = i / NP, n = i % NP, t = t0 + r;
      sB[r][n] = n < p.N && t < tend ? to_f32(Bp[t * sb + n]) : 0.f;
    }
    __syncthreads();
#pragma unroll 8
    for (int q = 0; q < TT; ++q) {
      const int r = REV ? TT - 1 - q : q;
      const float2 ss = sS[r][hc];
      const float4 bv = *reinterpret_cast<const float4*>(&sB[r][n0]);
      const float bb[4] = {bv.x, bv.y, bv.z, bv.w};
#pragma unroll
      for (int i = 0; i < SPL; ++i) {
        const float a = ex2(ss.x * A2[i]);
        h[i] = REV ? a * fmaf(bb[i], ss.y, h[i]) : fmaf(a, h[i], ss.y * bb[i]);
      }
    }
  }
  const int64_t row = (int64_t)b * p.nseg + seg;
#pragma unroll
  for (int i = 0; i < SPL; ++i)
    if (hc < nch && n0 + i < p.N) p.carry[(row * p.D + d0 + hc) * p.N + n0 + i] = h[i];
  sSum[ct0][cc] = total;
  __syncthreads();
  if (tid < nch) {
    float a = 0.f;
#pragma unroll
    for (int i = 0; i < NL; ++i) a += sSum[i][tid];
    p.ssum[row * p.D + d0 + tid] = a;
  }
}

// carry[seg] <- the state that enters segment seg.  One thread per (row, channel, state).
template <bool REV>
__global__ void __launch_bounds__(256) scan_combine_kernel(ScanP p) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int64_t dn = (int64_t)p.D * p.N;
  if (i >= p.B * dn) return;
  const int64_t b = i / dn, at = i % dn;
  const int d = (int)(at / p.N);
  const float A2 = p.A[at] * LOG2E;
  const float* from = REV ? p.dh_out : p.h0;
  float H = from ? from[i] : 0.f;
  const int last = REV ? 0 : p.nseg - 1;  // its local end state was not formed
#pragma unroll 4
  for (int k = 0; k < p.nseg; ++k) {
    const int seg = REV ? p.nseg - 1 - k : k;
    float* c = p.carry + (b * p.nseg + seg) * dn + at;
    if (seg != last) {
      const float e = *c;
      *c = H;
      H = fmaf(ex2(A2 * p.ssum[(b * p.nseg + seg) * p.D + d]), H, e);
    } else {
      *c = H;
    }
  }
}

// One token per row: the state is read and written once, 16 bytes per lane where N allows.
template <typename T, int NL>
__global__ void __launch_bounds__(SCAN_THREADS) scan_step_kernel(ScanP p) {
  const int64_t id = ((int64_t)blockIdx.x * SCAN_THREADS + threadIdx.x) / NL;
  const int n0 = (threadIdx.x % NL) * SPL, lane = threadIdx.x % 32;
  const bool live = id < (int64_t)p.B * p.D;
  const int b = live ? (int)(id / p.D) : 0, d = live ? (int)(id % p.D) : 0;
  const int grp = d / (p.D / p.G);
  float x = to_f32(static_cast<const T*>(p.x)[b * p.sx_b + d]);
  float s = to_f32(static_cast<const T*>(p.dt)[b * p.sdt_b + d]) + (p.dt_bias ? p.dt_bias[d] : 0.f);
  if (p.softplus) s = softplus(s);
  const T* Bp = static_cast<const T*>(p.Bm) + b * p.sB_b + grp * p.sB_g + n0;
  const T* Cp = static_cast<const T*>(p.Cm) + b * p.sC_b + grp * p.sC_g + n0;
  float* hp = p.h_out + ((int64_t)b * p.D + d) * p.N + n0;
  const float* Ap = p.A + (int64_t)d * p.N + n0;
  float y[1] = {0.f};
  if (live) {
#pragma unroll
    for (int i = 0; i < SPL; ++i) {
      if (n0 + i < p.N) {
        const float h = fmaf(ex2(s * Ap[i] * LOG2E), hp[i], s * x * to_f32(Bp[i]));
        hp[i] = h;
        y[0] = fmaf(to_f32(Cp[i]), h, y[0]);
      }
    }
  }
  spread_sum<1, NL, 1>(y, lane);
  if (live && n0 == 0) {
    float o = y[0] + (p.Dskip ? p.Dskip[d] * x : 0.f);
    if (p.z) o *= silu(to_f32(static_cast<const T*>(p.z)[b * p.sz_b + d]));
    store_as(static_cast<T*>(p.y) + b * p.sy_b + d, o);
  }
}

SegPlan scan_segments(int64_t B, int64_t T, int64_t blocks_per_row) {
  constexpr int64_t FILL = 148 * 4, MIN_SEG = 128;
  SegPlan one = {1, (int)T};
  if (B * blocks_per_row >= FILL / 2 || T < 2 * MIN_SEG) return one;
  int64_t n = (FILL * 2 + B * blocks_per_row - 1) / (B * blocks_per_row);
  if (n > T / MIN_SEG) n = T / MIN_SEG;
  if (n < 2) return one;
  const int64_t len = ((T + n - 1) / n + TT - 1) / TT * TT;
  return {(int)((T + len - 1) / len), (int)len};
}

int scan_check(const gdn_scan_args* a, bool step) {
  if (!a) return GDN_ERR_NULL;
  if (a->B < 0 || a->T < 0 || a->D < 1 || a->N < 1 || a->G < 1) return GDN_ERR_SHAPE;
  if (a->N > 64) return GDN_ERR_UNSUPPORTED;
  if (a->D % a->G || a->B > 65535 || a->T > (1 << 30) || a->D > (1 << 24)) return GDN_ERR_SHAPE;
  if (!elem_size(a->dtype)) return GDN_ERR_DTYPE;
  if (!a->A) return GDN_ERR_NULL;
  const int64_t st[] = {a->sx_b, a->sx_t, a->sdt_b, a->sdt_t, a->sB_b, a->sB_t, a->sB_g, a->sC_b, a->sC_t, a->sC_g, a->sz_b, a->sz_t, a->sy_b, a->sy_t};
  for (int64_t v : st)
    if (v < 0) return GDN_ERR_SHAPE;
  if (a->B > 0 && (step || a->T > 0) && (!a->x || !a->dt || !a->Bm || !a->Cm)) return GDN_ERR_NULL;
  if (step && a->B > 0 && (!a->y || !a->h_out)) return GDN_ERR_NULL;
  return GDN_OK;
}

ScanP scan_params(const gdn_scan_args* a) {
  ScanP p = {};
  p.x = a->x; p.dt = a->dt; p.Bm = a->Bm; p.Cm = a->Cm; p.z = a->z;
  p.A = a->A; p.Dskip = a->Dskip; p.dt_bias = a->dt_bias; p.h0 = a->h0; p.lengths = a->lengths;
  p.y = a->y; p.h_out = a->h_out; p.ckpt = a->ckpt;
  p.sx_b = a->sx_b; p.sx_t = a->sx_t; p.sdt_b = a->sdt_b; p.sdt_t = a->sdt_t; p.sB_b = a->sB_b; p.sB_t = a->sB_t; p.sB_g = a->sB_g;
  p.sC_b = a->sC_b; p.sC_t = a->sC_t; p.sC_g = a->sC_g; p.sz_b = a->sz_b; p.sz_t = a->sz_t; p.sy_b = a->sy_b; p.sy_t = a->sy_t;
  p.B = (int)a->B; p.T = (int)a->T; p.D = (int)a->D; p.N = (int)a->N; p.G = (int)a->G;
  p.softplus = a->softplus != 0;
  p.dblocks = scan_dblocks(a->D, a->G, a->N);
  const SegPlan sp = scan_segments(a->B > 0 ? a->B : 1, a->T, (int64_t)p.dblocks * a->G);
  p.nseg = sp.nseg;
  p.seg_len = sp.seg_len;
  return p;
}

template <typename T, bool REV>
void launch_carry(const ScanP& p, int nl, cudaStream_t s) {
  const dim3 g(p.dblocks * p.G, p.nseg, p.B);
  if (nl == 2) scan_carry_kernel<T, 2, REV><<<g, SCAN_THREADS, 0, s>>>(p);
  if (nl == 4) scan_carry_kernel<T, 4, REV><<<g, SCAN_THREADS, 0, s>>>(p);
  if (nl == 8) scan_carry_kernel<T, 8, REV><<<g, SCAN_THREADS, 0, s>>>(p);
  if (nl == 16) scan_carry_kernel<T, 16, REV><<<g, SCAN_THREADS, 0, s>>>(p);
}

int scan_launch_carry(const ScanP& p, int dtype, bool reverse, cudaStream_t s) {
  const int nl = scan_lanes(p.N);
  const int64_t g = ((int64_t)p.B * p.D * p.N + 255) / 256;
  if (g > 0x7fffffff) return GDN_ERR_SHAPE;
  if (reverse) {
    dtype == GDN_DTYPE_F32 ? launch_carry<float, true>(p, nl, s) : launch_carry<__nv_bfloat16, true>(p, nl, s);
    scan_combine_kernel<true><<<(unsigned)g, 256, 0, s>>>(p);
  } else {
    dtype == GDN_DTYPE_F32 ? launch_carry<float, false>(p, nl, s) : launch_carry<__nv_bfloat16, false>(p, nl, s);
    scan_combine_kernel<false><<<(unsigned)g, 256, 0, s>>>(p);
  }
  return launched();
}

template <typename T>
void launch_fwd(const ScanP& p, int nl, cudaStream_t s) {
  const dim3 g(p.dblocks * p.G, p.nseg, p.B);
  if (nl == 2) scan_fwd_kernel<T, 2><<<g, SCAN_THREADS, 0, s>>>(p);
  if (nl == 4) scan_fwd_kernel<T, 4><<<g, SCAN_THREADS, 0, s>>>(p);
  if (nl == 8) scan_fwd_kernel<T, 8><<<g, SCAN_THREADS, 0, s>>>(p);
  if (nl == 16) scan_fwd_kernel<T, 16><<<g, SCAN_THREADS, 0, s>>>(p);
}

template <typename T>
int launch_step(const ScanP& p, int nl, cudaStream_t s) {
  const int64_t g = ((int64_t)p.B * p.D * nl + SCAN_THREADS - 1) / SCAN_THREADS;
  if (g > 0x7fffffff) return GDN_ERR_SHAPE;
  if (nl == 2) scan_step_kernel<T, 2><<<(unsigned)g, SCAN_THREADS, 0, s>>>(p);
  if (nl == 4) scan_step_kernel<T, 4><<<(unsigned)g, SCAN_THREADS, 0, s>>>(p);
  if (nl == 8) scan_step_kernel<T, 8><<<(unsigned)g, SCAN_THREADS, 0, s>>>(p);
  if (nl == 16) scan_step_kernel<T, 16><<<(unsigned)g, SCAN_THREADS, 0, s>>>(p);
  return launched();
}

}  // namespace ssm
}  // namespace gdn

using namespace gdn::ssm;

extern "C" {

int gdn_scan_workspace_bytes(const gdn_scan_args* a, size_t* bytes) {
  if (!bytes) return GDN_ERR_NULL;
  int st = scan_check(a, false);
  if (st != GDN_OK) return st;
  const ScanP p = scan_params(a);
  *bytes = p.nseg > 1 ? (size_t)p.B * p.nseg * p.D * (p.N + 1) * sizeof(float) : 0;
  return GDN_OK;
}

int gdn_scan_fwd(const gdn_scan_args* a, void* stream) {
  size_t need = 0;
  int st = gdn_scan_workspace_bytes(a, &need);
  if (st != GDN_OK) return st;
  if (a->B == 0) return GDN_OK;
  if (a->T > 0 && !a->y) return GDN_ERR_NULL;
  if (need && (!a->workspace || a->workspace_bytes < need)) return GDN_ERR_WORKSPACE;
  if (!device_ok()) return GDN_ERR_DEVICE;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  ScanP p = scan_params(a);
  if (p.T == 0) {  // nothing to scan: the state passes through
    if (!p.h_out || p.h_out == p.h0) return GDN_OK;
    const size_t n = (size_t)p.B * p.D * p.N * sizeof(float);
    const cudaError_t e = p.h0 ? cudaMemcpyAsync(p.h_out, p.h0, n, cudaMemcpyDeviceToDevice, s) : cudaMemsetAsync(p.h_out, 0, n, s);
    return e == cudaSuccess ? GDN_OK : GDN_ERR_LAUNCH;
  }
  if (p.nseg > 1) {
    p.carry = static_cast<float*>(a->workspace);
    p.ssum = p.carry + (int64_t)p.B * p.nseg * p.D * p.N;
    st = scan_launch_carry(p, a->dtype, false, s);
    if (st != GDN_OK) return st;
  }
  const int nl = scan_lanes(p.N);
  a->dtype == GDN_DTYPE_F32 ? launch_fwd<float>(p, nl, s) : launch_fwd<__nv_bfloat16>(p, nl, s);
  return launched();
}

int gdn_scan_step(const gdn_scan_args* a, void* stream) {
  int st = scan_check(a, true);
  if (st != GDN_OK) return st;
  if (a->B == 0) return GDN_OK;
  if (!device_ok()) return GDN_ERR_DEVICE;
  const ScanP p = scan_params(a);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return a->dtype == GDN_DTYPE_F32 ? launch_step<float>(p, scan_lanes(p.N), s) : launch_step<__nv_bfloat16>(p, scan_lanes(p.N), s);
}

}  // extern "C"
