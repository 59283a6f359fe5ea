// Selective scan, backward.
//
//   g_t = C_t dc_t + G_t,  G_{t-1} = exp(s_t A) g_t   (dc = dy silu(z); G_{T-1} = gradient of the final state)
//   dx = s (g . B) + D dc;  ds = sum_n g exp(s A) h_{t-1} A + x (g . B);  ddt = ds sigmoid(dt + bias)
//   dB = sum_d g s x;  dC = sum_d dc h;  dA = sum_{b,t} g exp(s A) h_{t-1} s;  dD = sum dc x;  dz = dy (C.h + D x) silu'(z)
//
// The states are rebuilt from the forward's checkpoints, 16 tokens at a time, in registers; the adjoint then walks the
// tile backwards.  dB and dC are summed over a block's channels (lanes, then warps) and over the blocks by a second
// kernel, in a fixed order.
#include "ssm_scan.cuh"

namespace gdn {
namespace ssm {

constexpr int CK = GDN_SCAN_CKPT;

template <typename T, int NL>
__global__ void __launch_bounds__(SCAN_THREADS) scan_bwd_kernel(ScanP p) {
  constexpr int CH = SCAN_THREADS / NL, NP = NL * SPL, PER = CK * CH / SCAN_THREADS, WARPS = SCAN_THREADS / 32;
  __shared__ float2 sS[CK][CH];              // step size, step size * x
  __shared__ float sG[CK][CH];               // dc
  __shared__ float sP[CK][CH + 1], sX[CK][CH + 1], sT[CK][CH + 1];  // C.h, g.B, sum_n g a h_{t-1} A
  __shared__ __align__(16) float sB[CK][NP], sC[CK][NP];
  __shared__ float sR[WARPS][CK][2 * NP];    // dB, dC of each warp's channels
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int grp = blockIdx.x / p.dblocks, dblk = blockIdx.x % p.dblocks;
  const int seg = blockIdx.y, b = blockIdx.z;
  const int dpg = p.D / p.G, d0 = grp * dpg + dblk * CH, nch = min(CH, dpg - dblk * CH);
  const int len = row_tokens(p.lengths, b, p.T);
  const int tbeg = seg * p.seg_len, tend = min(tbeg + p.seg_len, p.T);
  const int hc = tid / NL, n0 = (tid % NL) * SPL;
  const bool live = hc < nch;
  const int64_t row = (int64_t)b * p.nseg + seg;
  float G[SPL], A[SPL], dA[SPL];
#pragma unroll
  for (int i = 0; i < SPL; ++i) {
    const bool ok = live && n0 + i < p.N;
    const int64_t at = (int64_t)(d0 + hc) * p.N + n0 + i;
    A[i] = ok ? p.A[at] : 0.f;
    dA[i] = 0.f;
    const float* from = p.nseg > 1 ? p.carry + row * p.D * p.N : p.dh_out ? p.dh_out + (int64_t)b * p.D * p.N : nullptr;
    G[i] = ok && from ? from[at] : 0.f;
  }
  const int cc = tid % CH, ct0 = tid / CH;
  const bool cok = cc < nch;
  const int d = d0 + (cok ? cc : 0);
  const float bias = p.dt_bias ? p.dt_bias[d] : 0.f, skip = p.Dskip ? p.Dskip[d] : 0.f;
  const T* xp = static_cast<const T*>(p.x) + b * p.sx_b + d;
  const T* dtp = static_cast<const T*>(p.dt) + b * p.sdt_b + d;
  const T* zp = p.z ? static_cast<const T*>(p.z) + b * p.sz_b + d : nullptr;
  const T* dyp = static_cast<const T*>(p.dy) + b * p.sdy_b + d;
  const T* Bp = static_cast<const T*>(p.Bm) + b * p.sB_b + grp * p.sB_g;
  const T* Cp = static_cast<const T*>(p.Cm) + b * p.sC_b + grp * p.sC_g;
  T *dxp = static_cast<T*>(p.dx), *ddtp = static_cast<T*>(p.ddt), *dzp = static_cast<T*>(p.dz);
  const int nck = (p.T + CK - 1) / CK;
  float sumD = 0.f, sumB = 0.f;

  for (int t0 = tbeg + (tend - tbeg - 1) / CK * CK; t0 >= tbeg; t0 -= CK) {
    float xr[PER], sr[PER], zr[PER], dyr[PER], sg[PER];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int r = ct0 + i * NL, t = t0 + r;
      xr[i] = sr[i] = zr[i] = dyr[i] = sg[i] = 0.f;
      float dc = 0.f;
      if (cok && t < len && t < tend) {
        xr[i] = to_f32(xp[t * p.sx_t]);
        dyr[i] = dc = to_f32(dyp[t * p.sdy_t]);
        const float v = to_f32(dtp[t * p.sdt_t]) + bias;
        sr[i] = p.softplus ? softplus(v) : v;
        sg[i] = p.softplus ? sigmoid(v) : 1.f;
        if (zp) {
          zr[i] = to_f32(zp[t * p.sz_t]);
          dc *= silu(zr[i]);
        }
      }
      sS[r][cc] = make_float2(sr[i], sr[i] * xr[i]);
      sG[r][cc] = dc;
    }
    for (int i = tid; i < CK * NP; i += SCAN_THREADS) {
      const int r = i / NP, n = i % NP, t = t0 + r;
      const bool ok = n < p.N && t < len && t < tend;
      sB[r][n] = ok ? to_f32(Bp[t * p.sB_t + n]) : 0.f;
      sC[r][n] = ok ? to_f32(Cp[t * p.sC_t + n]) : 0.f;
    }
    float h[SPL], hp[CK][SPL];
#pragma unroll
    for (int i = 0; i < SPL; ++i)
      h[i] = live && n0 + i < p.N ? p.ckpt[(((int64_t)b * nck + t0 / CK) * p.D + d0 + hc) * p.N + n0 + i] : 0.f;
    __syncthreads();
    // the tile's states, and C.h for the gate's gradient
#pragma unroll
    for (int q = 0; q < CK; q += NL) {
      float acc[NL];
#pragma unroll
      for (int j = 0; j < NL; ++j) {
        const int r = q + j;
        const float2 ss = sS[r][hc];
        const float4 bv = *reinterpret_cast<const float4*>(&sB[r][n0]);
        const float4 cv = *reinterpret_cast<const float4*>(&sC[r][n0]);
        const float bb[4] = {bv.x, bv.y, bv.z, bv.w}, cq[4] = {cv.x, cv.y, cv.z, cv.w};
        acc[j] = 0.f;
#pragma unroll
        for (int i = 0; i < SPL; ++i) {
          hp[r][i] = h[i];
          h[i] = fmaf(ex2(ss.x * (A[i] * LOG2E)), h[i], ss.y * bb[i]);
          acc[j] = fmaf(cq[i], h[i], acc[j]);
        }
      }
      if (zp) {
        const int j = spread_sum<NL, NL, 1>(acc, lane);
        sP[q + j][hc] = acc[0];
      }
    }
    // the adjoint, from the tile's last token
#pragma unroll
    for (int q = CK - NL; q >= 0; q -= NL) {
      float gb[NL], ga[NL];
#pragma unroll
      for (int j = NL - 1; j >= 0; --j) {
        const int r = q + j;
        const float2 ss = sS[r][hc];
        const float dc = sG[r][hc];
        const float4 bv = *reinterpret_cast<const float4*>(&sB[r][n0]);
        const float4 cv = *reinterpret_cast<const float4*>(&sC[r][n0]);
        const float bb[4] = {bv.x, bv.y, bv.z, bv.w}, cq[4] = {cv.x, cv.y, cv.z, cv.w};
        float v[2 * SPL];
        gb[j] = ga[j] = 0.f;
#pragma unroll
        for (int i = 0; i < SPL; ++i) {
          const float a = ex2(ss.x * (A[i] * LOG2E));
          const float g = fmaf(cq[i], dc, G[i]);
          gb[j] = fmaf(g, bb[i], gb[j]);
          v[i] = g * ss.y;
          v[SPL + i] = dc * fmaf(a, hp[r][i], ss.y * bb[i]);
          G[i] = a * g;
          const float flow = G[i] * hp[r][i];
          ga[j] = fmaf(flow, A[i], ga[j]);
          dA[i] = fmaf(flow, ss.x, dA[i]);
        }
        const int f = spread_sum<2 * SPL, 32 / NL, NL>(v, lane);
        constexpr int LEFT = 2 * SPL * NL / 32 > 1 ? 2 * SPL * NL / 32 : 1;
#pragma unroll
        for (int i = 0; i < LEFT; ++i) sR[warp][r][(f + i) / SPL * NP + n0 + (f + i) % SPL] = v[i];
      }
      int j = spread_sum<NL, NL, 1>(gb, lane);
      sX[q + j][hc] = gb[0];
      j = spread_sum<NL, NL, 1>(ga, lane);
      sT[q + j][hc] = ga[0];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int r = ct0 + i * NL, t = t0 + r;
      if (!cok || t >= tend) continue;
      const bool on = t < len;
      const float dc = sG[r][cc], gB = sX[r][cc];
      const float ddt = on ? fmaf(gB, xr[i], sT[r][cc]) * sg[i] : 0.f;
      sumD = fmaf(dc, xr[i], sumD);
      sumB += ddt;
      const int64_t at = ((int64_t)b * p.T + t) * p.D + d;
      store_as(dxp + at, on ? fmaf(sr[i], gB, skip * dc) : 0.f);
      store_as(ddtp + at, ddt);
      if (zp) store_as(dzp + at, on ? dyr[i] * fmaf(skip, xr[i], sP[r][cc]) * dsilu(zr[i]) : 0.f);
    }
    for (int i = tid; i < CK * 2 * NP; i += SCAN_THREADS) {
      const int r = i / (2 * NP), w = i % (2 * NP), n = w % NP, t = t0 + r;
      if (n >= p.N || t >= tend) continue;
      float a = 0.f;
#pragma unroll
      for (int k = 0; k < WARPS; ++k) a += sR[k][r][w];
      p.pBC[(((((int64_t)dblk * p.B + b) * p.T + t) * p.G + grp) * 2 + w / NP) * p.N + n] = a;
    }
  }
#pragma unroll
  for (int i = 0; i < SPL; ++i) {
    if (!live || n0 + i >= p.N) continue;
    const int64_t at = (int64_t)(d0 + hc) * p.N + n0 + i;
    p.pA[row * p.D * p.N + at] = dA[i];
    if (p.dh0 && seg == 0) p.dh0[(int64_t)b * p.D * p.N + at] = G[i];
  }
  // dD and ddt_bias over the threads of a channel
  __syncthreads();
  sS[ct0][cc] = make_float2(sumD, sumB);
  __syncthreads();
  if (tid < nch) {
    float a = 0.f, e = 0.f;
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      a += sS[i][tid].x;
      e += sS[i][tid].y;
    }
    p.pD[row * 2 * p.D + d0 + tid] = a;
    p.pD[(row * 2 + 1) * p.D + d0 + tid] = e;
  }
}

// dB and dC: the channel blocks' partial sums, (dblocks, B T G, 2, N) -> two (B T G, N) tensors.
template <typename T>
__global__ void __launch_bounds__(256) scan_sum_bc_kernel(const float* part, int dblocks, int64_t rows, int N, T* dB, T* dC) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x, n = rows * 2 * N;
  if (i >= n) return;
  float a = 0.f;
#pragma unroll 8
  for (int k = 0; k < dblocks; ++k) a += part[k * n + i];
  const int64_t r = i / (2 * N);
  const int w = (int)(i % (2 * N));
  store_as((w < N ? dB : dC) + r * N + w % N, a);
}

// dA (first D N entries), then dD, then ddt_bias: sums over the rows' and segments' partials.
__global__ void __launch_bounds__(256) scan_sum_params_kernel(ScanP p, float* dA, float* dD, float* dbias) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x, dn = (int64_t)p.D * p.N;
  if (i >= dn + 2 * p.D) return;
  const float* part = i < dn ? p.pA + i : p.pD + (i - dn);
  const int64_t step = i < dn ? dn : 2 * p.D;
  float a = 0.f;
#pragma unroll 8
  for (int k = 0; k < p.B * p.nseg; ++k) a += part[k * step];
  if (i < dn)
    dA[i] = a;
  else if (i < dn + p.D) {
    if (dD) dD[i - dn] = a;
  } else if (dbias) {
    dbias[i - dn - p.D] = a;
  }
}

struct BwdPlan {
  size_t carry, ssum, bc, a, d, total;  // floats
};

BwdPlan bwd_plan(const ScanP& p) {
  BwdPlan w = {};
  if (p.nseg > 1) {
    w.carry = (size_t)p.B * p.nseg * p.D * p.N;
    w.ssum = (size_t)p.B * p.nseg * p.D;
  }
  w.bc = (size_t)p.dblocks * p.B * p.T * p.G * 2 * p.N;
  w.a = (size_t)p.B * p.nseg * p.D * p.N;
  w.d = (size_t)p.B * p.nseg * p.D * 2;
  w.total = w.carry + w.ssum + w.bc + w.a + w.d;
  return w;
}

template <typename T>
int launch_bwd(const ScanP& p, const gdn_scan_bwd_args* a, cudaStream_t s) {
  const int nl = scan_lanes(p.N);
  const dim3 g(p.dblocks * p.G, p.nseg, p.B);
  if (nl == 2) scan_bwd_kernel<T, 2><<<g, SCAN_THREADS, 0, s>>>(p);
  if (nl == 4) scan_bwd_kernel<T, 4><<<g, SCAN_THREADS, 0, s>>>(p);
  if (nl == 8) scan_bwd_kernel<T, 8><<<g, SCAN_THREADS, 0, s>>>(p);
  if (nl == 16) scan_bwd_kernel<T, 16><<<g, SCAN_THREADS, 0, s>>>(p);
  int st = launched();
  if (st != GDN_OK) return st;
  const int64_t rows = (int64_t)p.B * p.T * p.G, n = rows * 2 * p.N;
  scan_sum_bc_kernel<T><<<(unsigned)((n + 255) / 256), 256, 0, s>>>(p.pBC, p.dblocks, rows, p.N, static_cast<T*>(a->dB), static_cast<T*>(a->dC));
  const int64_t m = (int64_t)p.D * (p.N + 2);
  scan_sum_params_kernel<<<(unsigned)((m + 255) / 256), 256, 0, s>>>(p, a->dA, a->dDskip, a->ddt_bias);
  return launched();
}

}  // namespace ssm
}  // namespace gdn

using namespace gdn::ssm;

extern "C" {

int gdn_scan_bwd_workspace_bytes(const gdn_scan_bwd_args* a, size_t* bytes) {
  if (!a || !bytes) return GDN_ERR_NULL;
  int st = scan_check(&a->fwd, false);
  if (st != GDN_OK) return st;
  *bytes = bwd_plan(scan_params(&a->fwd)).total * sizeof(float);
  return GDN_OK;
}

int gdn_scan_bwd(const gdn_scan_bwd_args* a, void* stream) {
  size_t need = 0;
  int st = gdn_scan_bwd_workspace_bytes(a, &need);
  if (st != GDN_OK) return st;
  const gdn_scan_args* f = &a->fwd;
  if (f->B == 0 || f->T == 0) return GDN_ERR_SHAPE;  // nothing flowed; the caller fills the gradients
  if (!a->dy || !a->dx || !a->ddt || !a->dB || !a->dC || !a->dA || !f->ckpt || (f->z && !a->dz)) return GDN_ERR_NULL;
  if (a->sdy_b < 0 || a->sdy_t < 0) return GDN_ERR_SHAPE;
  if ((int64_t)f->B * f->T * f->G * 2 * f->N > (int64_t)0x7fffffff * 256) return GDN_ERR_SHAPE;
  if (!a->fwd.workspace || a->fwd.workspace_bytes < need) return GDN_ERR_WORKSPACE;
  if (!device_ok()) return GDN_ERR_DEVICE;
  ScanP p = scan_params(f);
  p.dy = a->dy; p.sdy_b = a->sdy_b; p.sdy_t = a->sdy_t;
  p.dh_out = a->dh_out; p.dx = a->dx; p.ddt = a->ddt; p.dz = a->dz; p.dh0 = a->dh0;
  const BwdPlan w = bwd_plan(p);
  float* ws = static_cast<float*>(f->workspace);
  p.carry = ws; ws += w.carry;
  p.ssum = ws; ws += w.ssum;
  p.pBC = ws; ws += w.bc;
  p.pA = ws; ws += w.a;
  p.pD = ws;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (p.nseg > 1) {
    st = scan_launch_carry(p, f->dtype, true, s);
    if (st != GDN_OK) return st;
  }
  return f->dtype == GDN_DTYPE_F32 ? launch_bwd<float>(p, a, s) : launch_bwd<__nv_bfloat16>(p, a, s);
}

}  // extern "C"
