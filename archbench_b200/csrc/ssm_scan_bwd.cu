// Selective scan, backward.
//
//   g_t = C_t dc_t + G_t,  G_{t-1} = exp(s_t A) g_t   (dc = dy silu(z); G_{T-1} = gradient of the final state)
//   dx = s (g . B) + D dc;  ds = sum_n g exp(s A) h_{t-1} A + x (g . B);  ddt = ds sigmoid(dt + bias)
//   dB = sum_d g s x;  dC = sum_d dc h;  dA = sum_{b,t} g exp(s A) h_{t-1} s;  dD = sum dc x;  dz = dy (C.h + D x) silu'(z)
//
// The states are rebuilt from the forward's checkpoints, 16 tokens at a time, in registers; the adjoint then walks the
// tile backwards.  dB and dC are summed over a block's channels (lanes, then warps) and over the blocks by a second
// kernel, in a fixed order.
#include <algorithm>

#include "ssm_scan.cuh"

namespace gdn {
namespace ssm {

constexpr int CK = 16;  // tokens per tile (a multiple of GDN_SCAN_CKPT)

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
  const int nck = (p.T + GDN_SCAN_CKPT - 1) / GDN_SCAN_CKPT;
  float sumD = 0.f, sumB = 0.f;

  for (int t0 = tbeg + (tend - tbeg - 1) / CK * CK; t0 >= tbeg; t0 -= CK) {
    if (t0 >= len) {  // nothing here: zero gradients, the adjoint passes through
      for (int r = ct0; r < CK && t0 + r < tend; r += NL) {
        const int64_t at = ((int64_t)b * p.T + t0 + r) * p.D + d;
        if (!cok) continue;
        store_as(dxp + at, 0.f);
        store_as(ddtp + at, 0.f);
        if (zp) store_as(dzp + at, 0.f);
      }
      for (int i = tid; i < CK * 2 * NP; i += SCAN_THREADS) {
        const int t = t0 + i / (2 * NP), w = i % (2 * NP), n = w % NP;
        if (n < p.N && t < tend) p.pBC[(((((int64_t)dblk * p.B + b) * p.T + t) * p.G + grp) * 2 + w / NP) * p.N + n] = 0.f;
      }
      continue;
    }
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
      h[i] = live && n0 + i < p.N ? p.ckpt[(((int64_t)b * nck + t0 / GDN_SCAN_CKPT) * p.D + d0 + hc) * p.N + n0 + i] : 0.f;
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
          h[i] = fmaf(decay(ss.x, A[i] * LOG2E), h[i], ss.y * bb[i]);
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
          const float a = decay(ss.x, A[i] * LOG2E);
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

// The same where N is a multiple of four (rows are 16-byte aligned, or were laid out so).  A lane holds four states of two channels, a warp 64 / NL channels, a
// block four warps; tiles of 8 tokens (one checkpoint), last first, with one barrier each: a thread rebuilds the states of
// tile k (decays and states stay in registers, so each exponential is formed once), walks the adjoint back, stages tile
// k - 1 (earlier tokens) and finishes tile k + 1.
template <typename T, int NL>
struct BwdTiled {
  static constexpr int TT = 8, CH = 256 / NL, NP = NL * SPL, ES = (int)sizeof(T), RING = 4, WARPS = 4;
  static constexpr int ROW = CH * ES, BROW = NP * ES;
  static constexpr int RAW = TT * (4 * ROW + 2 * BROW);  // x, dt, z, dy, B, C of a tile
  static constexpr int S_OFF = RING * RAW, S_BYTES = TT * CH * 12;      // (s, u) of channel pairs, then dc
  static constexpr int P_OFF = S_OFF + 2 * S_BYTES, P_BYTES = TT * SCAN_THREADS * 24;  // (g.B, ds) parts, then C.h parts
  static constexpr int BC_OFF = P_OFF + 2 * P_BYTES, BC_BYTES = 2 * TT * NP * 4;
  static constexpr int R_OFF = BC_OFF + 2 * BC_BYTES, R_BYTES = WARPS * TT * 2 * NP * 4;  // dB, dC of each warp
  static constexpr int A_OFF = R_OFF + 2 * R_BYTES, A_BYTES = SCAN_THREADS * 32;  // each lane's dA
  static constexpr int SMEM = A_OFF + A_BYTES;
  static constexpr int XCH = ROW / 16, BCH = BROW / 16;
  static constexpr int CHUNKS = TT * (4 * XCH + 2 * BCH), COPIES = (CHUNKS + SCAN_THREADS - 1) / SCAN_THREADS;
};

template <typename T, int NL>
__global__ void __launch_bounds__(SCAN_THREADS, 2) scan_bwd_tiled_kernel(const ScanP p) {
  using K = BwdTiled<T, NL>;
  constexpr int TT = K::TT, CH = K::CH, NP = K::NP;
  static_assert(TT == GDN_SCAN_CKPT, "one checkpoint per tile");
  constexpr int TSTEP = SCAN_THREADS / (CH / 2), PER = TT / TSTEP > 0 ? TT / TSTEP : 1;
  constexpr int QUADS = 2 * TT * NL;                    // four-state groups of B and C
  constexpr int QI = (QUADS + SCAN_THREADS - 1) / SCAN_THREADS;
  constexpr int SHIFT4 = NL == 2 ? 2 : NL == 4 ? 1 : 0, SHIFT2 = NL == 2 ? 3 : NL == 4 ? 2 : NL == 8 ? 1 : 0;
  constexpr float LN2 = 0.69314718055994530942f;
  extern __shared__ __align__(16) char smem[];
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int grp = blockIdx.x / p.dblocks, dblk = blockIdx.x % p.dblocks;
  const int seg = blockIdx.y, b = blockIdx.z;
  const int dpg = p.D / p.G, d0 = grp * dpg + dblk * CH, nch = min(CH, dpg - dblk * CH);
  const int len = row_tokens(p.lengths, b, p.T);
  const int tbeg = seg * p.seg_len, tend = min(tbeg + p.seg_len, p.T), lim = min(tend, len);
  const int ntile = lim > tbeg ? (lim - tbeg + TT - 1) / TT : 0;
  const int64_t row = (int64_t)b * p.nseg + seg;

  const char* src[K::COPIES];
  int64_t step[K::COPIES];
  int tok[K::COPIES];
  constexpr int NONE = 1 << 29;
#pragma unroll
  for (int i = 0; i < K::COPIES; ++i) {
    int c = tid + i * SCAN_THREADS;
    tok[i] = NONE;
    src[i] = static_cast<const char*>(p.x);
    step[i] = 0;
    const void* base;
    int64_t sb, st, off;
    int r, j, bytes;
    if (c < 4 * TT * K::XCH) {
      const int which = c / (TT * K::XCH);
      r = c / K::XCH % TT; j = c % K::XCH; bytes = nch * K::ES; off = (int64_t)grp * p.xgs + dblk * CH;
      base = which == 0 ? p.x : which == 1 ? p.dt : which == 2 ? p.z : p.dy;
      sb = which == 0 ? p.sx_b : which == 1 ? p.sdt_b : which == 2 ? p.sz_b : p.sdy_b;
      st = which == 0 ? p.sx_t : which == 1 ? p.sdt_t : which == 2 ? p.sz_t : p.sdy_t;
    } else {
      c -= 4 * TT * K::XCH;
      const int which = c / (TT * K::BCH);
      r = c / K::BCH % TT; j = c % K::BCH; bytes = which < 2 ? p.N * K::ES : 0;
      base = which ? p.Cm : p.Bm;
      sb = which ? p.sC_b : p.sB_b;
      st = which ? p.sC_t : p.sB_t;
      off = grp * (which ? p.sC_g : p.sB_g);
    }
    if (base && j * 16 < bytes) {
      tok[i] = r;
      src[i] = static_cast<const char*>(base) + (b * sb + ((int64_t)tbeg + (ntile - 1) * TT + r) * st + off) * K::ES + j * 16;
      step[i] = -st * TT * K::ES;
    }
  }
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(smem));
  // Step k works on tile ntile - 1 - k.
  auto fetch = [&](int k) {
    if (k < ntile) {
#pragma unroll
      for (int i = 0; i < K::COPIES; ++i) {
        if (K::CHUNKS % SCAN_THREADS == 0 || tid + i * SCAN_THREADS < K::CHUNKS)
          copy16(ring + (k & (K::RING - 1)) * K::RAW + (tid + i * SCAN_THREADS) * 16, src[i], tbeg + (ntile - 1 - k) * TT + tok[i] < lim);
        src[i] += step[i];
      }
    }
    copies_commit();
  };

  // per-state role: channels hc, hc + 1 of the block
  const int hc = tid / NL * 2, n0 = tid % NL * SPL;
  const bool live = hc < nch && n0 < p.N;
  f32x2 G[2][2], A2[2][2];
  // dA of the lane, two halves of four states; a tile's terms are summed first, which keeps both its rounding and the
  // registers small
  ulonglong2* dA_sum = reinterpret_cast<ulonglong2*>(smem + K::A_OFF) + tid;
  const int64_t own = (int64_t)(d0 + hc) * p.N + n0;  // of channel hc; channel hc + 1 is N further
  const float* from = p.nseg > 1 ? p.carry + row * p.D * p.N : p.dh_out ? p.dh_out + (int64_t)b * p.D * p.N : nullptr;
  auto load4 = [&](const float* q, int c, f32x2 (&v)[2]) {
    const ulonglong2 r = q && live && hc + c < nch ? *reinterpret_cast<const ulonglong2*>(q + own + c * p.N) : make_ulonglong2(0, 0);
    v[0] = r.x;
    v[1] = r.y;
  };
  auto store4 = [&](float* q, int c, const f32x2 (&v)[2]) {
    if (live && hc + c < nch) *reinterpret_cast<ulonglong2*>(q + own + c * p.N) = make_ulonglong2(v[0], v[1]);
  };
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    load4(from, c, G[c]);
    load4(p.A, c, A2[c]);
#pragma unroll
    for (int i = 0; i < 2; ++i) A2[c][i] = mul2(A2[c][i], both(LOG2E));
    dA_sum[c * SCAN_THREADS] = make_ulonglong2(0, 0);
  }
  const int nck = (p.T + TT - 1) / TT;
  auto checkpoint = [&](int k, int c, f32x2 (&v)[2]) {
    load4(p.ckpt + ((int64_t)b * nck + tbeg / TT + ntile - 1 - k) * p.D * p.N, c, v);
  };

  // per-token role: channels cc, cc + 1, tokens ct0, ct0 + TSTEP, ...
  const int pair = tid % (CH / 2), cc = pair * 2, ct0 = tid / (CH / 2);
  const bool cok = cc < nch && ct0 < TT;
  const int d = d0 + (cc < nch ? cc : 0);
  const bool two = cc + 1 < nch;  // an odd group's last pair has one channel
  const f32x2 bias = p.dt_bias ? pack2(p.dt_bias[d], two ? p.dt_bias[d + 1] : 0.f) : both(0.f);
  const f32x2 skip = p.Dskip ? pack2(p.Dskip[d], two ? p.Dskip[d + 1] : 0.f) : both(0.f);
  auto put_pair = [&](T* q, const float (&v)[2]) {
    if (p.pairs_out) {
      store_pair(q, v);
    } else {
      store_as(q, v[0]);
      if (two) store_as(q + 1, v[1]);
    }
  };
  T *dxp = static_cast<T*>(p.dx), *ddtp = static_cast<T*>(p.ddt), *dzp = static_cast<T*>(p.dz);
  f32x2 sumD = both(0.f), sumB = both(0.f);

  auto raw_pair = [&](int k, int which, int r) {
    return load_pair(reinterpret_cast<const T*>(smem + (k & (K::RING - 1)) * K::RAW + (which * TT + r) * K::ROW + cc * K::ES));
  };
  auto stage = [&](int k, int i) {
    const int r = ct0 + i * TSTEP;
    if (TSTEP > TT && r >= TT) return;
    f32x2 s = add2(raw_pair(k, 1, r), bias);
    s = p.softplus ? softplus2(s) : s;
    const f32x2 z = raw_pair(k, 2, r), dy = raw_pair(k, 3, r);
    const f32x2 dc = p.z ? mul2(dy, mul2(z, sigmoid2(z))) : dy;
    const float2 uv = unpack2(mul2(s, raw_pair(k, 0, r))), sv = unpack2(s);
    const bool on = tbeg + (ntile - 1 - k) * TT + r < lim;
    char* o = smem + K::S_OFF + (k & 1) * K::S_BYTES;
    reinterpret_cast<float4*>(o)[r * (CH / 2) + pair] = on ? make_float4(sv.x, uv.x, sv.y, uv.y) : make_float4(0.f, 0.f, 0.f, 0.f);
    reinterpret_cast<f32x2*>(o + TT * CH * 8)[r * (CH / 2) + pair] = dc;  // 0 past the tokens: dy was filled with zeros
  };
  auto stage_bc = [&](int k) {
#pragma unroll
    for (int i = 0; i < QI; ++i) {
      const int q = tid + i * SCAN_THREADS;
      if (QUADS % SCAN_THREADS && q >= QUADS) break;
      const T* raw = reinterpret_cast<const T*>(smem + (k & (K::RING - 1)) * K::RAW + 4 * TT * K::ROW) + q * 4;
      reinterpret_cast<ulonglong2*>(smem + K::BC_OFF + (k & 1) * K::BC_BYTES)[q] = make_ulonglong2(load_pair(raw), load_pair(raw + 2));
    }
  };
  auto finish = [&](int k, int i) {
    const int r = ct0 + i * TSTEP, t = tbeg + (ntile - 1 - k) * TT + r;
    if (TSTEP > TT && r >= TT) return;
    const char* parts = smem + K::P_OFF + (k & 1) * K::P_BYTES;
    const ulonglong2* q4 = reinterpret_cast<const ulonglong2*>(parts) + r * SCAN_THREADS + pair * NL;
    const f32x2* q2 = reinterpret_cast<const f32x2*>(parts + TT * SCAN_THREADS * 16) + r * SCAN_THREADS + pair * NL;
    f32x2 gB = both(0.f), ds = both(0.f), core = both(0.f);
#pragma unroll
    for (int j = 0; j < NL; ++j) {  // each pair starts elsewhere, so that neighbours read different banks
      const ulonglong2 v = q4[(j + (pair >> SHIFT4)) & (NL - 1)];
      gB = add2(gB, v.x);
      ds = add2(ds, v.y);
      core = add2(core, q2[(j + (pair >> SHIFT2)) & (NL - 1)]);
    }
    const char* so = smem + K::S_OFF + (k & 1) * K::S_BYTES;
    const float4 su = reinterpret_cast<const float4*>(so)[r * (CH / 2) + pair];
    const f32x2 dc = reinterpret_cast<const f32x2*>(so + TT * CH * 8)[r * (CH / 2) + pair];
    const f32x2 x = raw_pair(k, 0, r), z = raw_pair(k, 2, r), dy = raw_pair(k, 3, r);
    const f32x2 v = add2(raw_pair(k, 1, r), bias);
    const bool on = t < lim;
    f32x2 ddt = fma2(ds, both(LN2), mul2(gB, x));
    ddt = p.softplus ? mul2(ddt, sigmoid2(v)) : ddt;
    ddt = on ? ddt : both(0.f);
    const f32x2 dx = fma2(pack2(su.x, su.z), gB, mul2(skip, dc));
    const f32x2 g = sigmoid2(z), dsilu = mul2(g, fma2(z, fma2(g, both(-1.f), both(1.f)), both(1.f)));
    const f32x2 dz = mul2(mul2(dy, fma2(skip, x, core)), dsilu);
    sumD = fma2(dc, x, sumD);
    sumB = add2(sumB, ddt);
    if (cok && t < tend) {
      const int64_t at = ((int64_t)b * p.T + t) * p.D + d;
      auto put = [&](T* q, f32x2 w) {
        const float2 e = unpack2(w);
        const float o[2] = {e.x, e.y};
        put_pair(q + at, o);
      };
      put(dxp, dx);
      put(ddtp, ddt);
      if (p.z) put(dzp, dz);
    }
  };
  auto finish_bc = [&](int k) {  // the four warps' dB and dC of tile k
    const float* red = reinterpret_cast<const float*>(smem + K::R_OFF + (k & 1) * K::R_BYTES);
    constexpr int N2 = TT * 2 * NP;
#pragma unroll
    for (int i = tid; i < N2; i += SCAN_THREADS) {
      const int r = i / (2 * NP), w = i % (2 * NP), n = w % NP, t = tbeg + (ntile - 1 - k) * TT + r;
      const float a = (red[i] + red[N2 + i]) + (red[2 * N2 + i] + red[3 * N2 + i]);
      if (n < p.N && t < tend) p.pBC[(((((int64_t)dblk * p.B + b) * p.T + t) * p.G + grp) * 2 + w / NP) * p.N + n] = a;
    }
  };

  fetch(0);
  fetch(1);
  f32x2 h0[2][2];
  if (ntile > 0) {
    checkpoint(0, 0, h0[0]);
    checkpoint(0, 1, h0[1]);
    copies_wait<1>();
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i) stage(0, i);
    stage_bc(0);
  }
#pragma unroll 1
  for (int k = 0; k < ntile; ++k) {
    copies_wait<0>();
    __syncthreads();
    fetch(k + 2);
    f32x2 h[TT + 1][2][2], a[TT][2][2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      h[0][c][0] = h0[c][0];
      h[0][c][1] = h0[c][1];
      if (k + 1 < ntile) checkpoint(k + 1, c, h0[c]);
    }
    const char* sS = smem + K::S_OFF + (k & 1) * K::S_BYTES;
    const float4* su_p = reinterpret_cast<const float4*>(sS) + hc / 2;
    const f32x2* dc_p = reinterpret_cast<const f32x2*>(sS + TT * CH * 8) + hc / 2;
    const float* sB = reinterpret_cast<const float*>(smem + K::BC_OFF + (k & 1) * K::BC_BYTES) + n0;
    // the tile's states
#pragma unroll
    for (int r = 0; r < TT; ++r) {
      const float4 su = su_p[r * (CH / 2)];
      const float4 bv = *reinterpret_cast<const float4*>(sB + r * NP);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float s = c ? su.z : su.x, u = c ? su.w : su.y;
        const float2 a0 = unpack2(A2[c][0]), a1 = unpack2(A2[c][1]);
        a[r][c][0] = pack2(decay(s, a0.x), decay(s, a0.y));
        a[r][c][1] = pack2(decay(s, a1.x), decay(s, a1.y));
        h[r + 1][c][0] = fma2(a[r][c][0], h[r][c][0], pack2(u * bv.x, u * bv.y));
        h[r + 1][c][1] = fma2(a[r][c][1], h[r][c][1], pack2(u * bv.z, u * bv.w));
      }
    }
    // finish the previous step's tile and stage the next one; items of one thread are its own in both
    if (k > 0) {
#pragma unroll
      for (int i = 0; i < PER; ++i) finish(k - 1, i);
      finish_bc(k - 1);
    }
    if (k + 1 < ntile) {
#pragma unroll
      for (int i = 0; i < PER; ++i) stage(k + 1, i);
      stage_bc(k + 1);
    }
    // the adjoint
    f32x2 dA[2][2];
    ulonglong2* p4 = reinterpret_cast<ulonglong2*>(smem + K::P_OFF + (k & 1) * K::P_BYTES) + tid;
    f32x2* p2 = reinterpret_cast<f32x2*>(smem + K::P_OFF + (k & 1) * K::P_BYTES + TT * SCAN_THREADS * 16) + tid;
    float* red = reinterpret_cast<float*>(smem + K::R_OFF + (k & 1) * K::R_BYTES) + warp * TT * 2 * NP;
    // A token's reads are issued before the stores of the token ahead of it: shared memory keeps the order of both.
    struct Token {
      float4 su;
      f32x2 dc;
      ulonglong2 bv, cv;
    };
    auto token = [&](int r) {
      return Token{su_p[r * (CH / 2)], dc_p[r * (CH / 2)], *reinterpret_cast<const ulonglong2*>(sB + r * NP),
                   *reinterpret_cast<const ulonglong2*>(sB + (TT + r) * NP)};
    };
    Token nxt = token(TT - 1);
#pragma unroll
    for (int r = TT - 1; r >= 0; --r) {
      const Token cur = nxt;
      if (r > 0) nxt = token(r - 1);
      const float4 su = cur.su;
      const float2 dc = unpack2(cur.dc);
      const ulonglong2 bv = cur.bv, cv = cur.cv;
      f32x2 dB[2], dC[2];
      float gb[2], ds[2], core[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const f32x2 dcd = both(c ? dc.y : dc.x), sd = both(c ? su.z : su.x), ud = both(c ? su.w : su.y);
        const f32x2 g0 = fma2(cv.x, dcd, G[c][0]), g1 = fma2(cv.y, dcd, G[c][1]);
        gb[c] = sum2(fma2(g1, bv.y, mul2(g0, bv.x)));
        core[c] = sum2(fma2(cv.y, h[r + 1][c][1], mul2(cv.x, h[r + 1][c][0])));
        dB[0] = c ? fma2(g0, ud, dB[0]) : mul2(g0, ud);
        dB[1] = c ? fma2(g1, ud, dB[1]) : mul2(g1, ud);
        dC[0] = c ? fma2(h[r + 1][c][0], dcd, dC[0]) : mul2(h[r + 1][c][0], dcd);
        dC[1] = c ? fma2(h[r + 1][c][1], dcd, dC[1]) : mul2(h[r + 1][c][1], dcd);
        G[c][0] = mul2(a[r][c][0], g0);
        G[c][1] = mul2(a[r][c][1], g1);
        const f32x2 f0 = mul2(G[c][0], h[r][c][0]), f1 = mul2(G[c][1], h[r][c][1]);
        ds[c] = sum2(fma2(f1, A2[c][1], mul2(f0, A2[c][0])));
        dA[c][0] = r == TT - 1 ? mul2(f0, sd) : fma2(f0, sd, dA[c][0]);
        dA[c][1] = r == TT - 1 ? mul2(f1, sd) : fma2(f1, sd, dA[c][1]);
      }
      p4[r * SCAN_THREADS] = make_ulonglong2(pack2(gb[0], gb[1]), pack2(ds[0], ds[1]));
      p2[r * SCAN_THREADS] = pack2(core[0], core[1]);
      const float2 b0 = unpack2(dB[0]), b1 = unpack2(dB[1]), c0 = unpack2(dC[0]), c1 = unpack2(dC[1]);
      float v[8] = {b0.x, b0.y, b1.x, b1.y, c0.x, c0.y, c1.x, c1.y};
      const int f = spread_sum<8, 32 / NL, NL>(v, lane);
      constexpr int LEFT = 8 * NL / 32 > 1 ? 8 * NL / 32 : 1;
#pragma unroll
      for (int i = 0; i < LEFT; ++i) red[r * 2 * NP + (f + i) / SPL * NP + n0 + (f + i) % SPL] = v[i];
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const ulonglong2 v = dA_sum[c * SCAN_THREADS];
      dA_sum[c * SCAN_THREADS] = make_ulonglong2(add2(v.x, dA[c][0]), add2(v.y, dA[c][1]));
    }
  }
  __syncthreads();
  if (ntile > 0) {
#pragma unroll
    for (int i = 0; i < PER; ++i) finish(ntile - 1, i);
    finish_bc(ntile - 1);
  }
  // past the row's tokens
  const float zero[2] = {0.f, 0.f};
  for (int t = tbeg + ntile * TT + ct0; t < tend; t += TSTEP) {  // (all token rows of threads: cok has only a tile's)
    if (cc >= nch) break;
    const int64_t at = ((int64_t)b * p.T + t) * p.D + d;
    put_pair(dxp + at, zero);
    put_pair(ddtp + at, zero);
    if (p.z) put_pair(dzp + at, zero);
  }
  for (int i = tid; i < (tend - tbeg - ntile * TT) * 2 * p.N; i += SCAN_THREADS) {
    const int64_t t = tbeg + ntile * TT + i / (2 * p.N);
    p.pBC[((((int64_t)dblk * p.B + b) * p.T + t) * p.G + grp) * 2 * p.N + i % (2 * p.N)] = 0.f;
  }
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const ulonglong2 v = dA_sum[c * SCAN_THREADS];
    const f32x2 dA[2] = {v.x, v.y};
    store4(p.pA + row * p.D * p.N, c, dA);
    if (p.dh0 && seg == 0) store4(p.dh0 + (int64_t)b * p.D * p.N, c, G[c]);
  }
  // dD and ddt_bias over the threads of a channel pair
  __syncthreads();
  ulonglong2* sums = reinterpret_cast<ulonglong2*>(smem);
  sums[ct0 * (CH / 2) + pair] = make_ulonglong2(sumD, sumB);
  __syncthreads();
  if (tid < (nch + 1) / 2) {
    f32x2 e = both(0.f), f = both(0.f);
#pragma unroll
    for (int i = 0; i < (TSTEP < TT ? TSTEP : TT); ++i) {
      const ulonglong2 v = sums[i * (CH / 2) + tid];
      e = add2(e, v.x);
      f = add2(f, v.y);
    }
    const float2 ev = unpack2(e), fv = unpack2(f);
    float *pd = p.pD + row * 2 * p.D + d0 + 2 * tid, *pb = pd + p.D;
    pd[0] = ev.x;
    pb[0] = fv.x;
    if (2 * tid + 1 < nch) {
      pd[1] = ev.y;
      pb[1] = fv.y;
    }
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
  size_t carry, ssum, bc, a, d, total;  // floats; then the aligned copies
};

BwdPlan bwd_plan(const ScanP& p) {
  BwdPlan w = {};
  auto up = [](size_t n) { return (n + 63) & ~(size_t)63; };  // every part on a 256-byte boundary
  if (p.nseg > 1) {
    w.carry = up((size_t)p.B * p.nseg * p.D * p.N);
    w.ssum = up((size_t)p.B * p.nseg * p.D);
  }
  w.bc = up((size_t)p.dblocks * p.B * p.T * p.G * 2 * p.N);
  w.a = up((size_t)p.B * p.nseg * p.D * p.N);
  w.d = up((size_t)p.B * p.nseg * p.D * 2);
  w.total = w.carry + w.ssum + w.bc + w.a + w.d;
  return w;
}

// Blocks of the tiled backward that run at once: two per SM by their registers, one where shared memory allows no more.
int64_t tiled_at_once(int es, int nl) {
  auto smem = [&](auto v) {
    using T = decltype(v);
    return nl == 2 ? BwdTiled<T, 2>::SMEM : nl == 4 ? BwdTiled<T, 4>::SMEM : nl == 8 ? BwdTiled<T, 8>::SMEM : BwdTiled<T, 16>::SMEM;
  };
  return (es == 4 ? smem(float()) : smem(__nv_bfloat16())) > 113 * 1024 ? 148 : 2 * 148;
}

// The backward's own segments of time: the blocks' whole waves decide.  In tokens of a block's work, a segment costs 16 more
// to start and end, the local pass 0.28 of everything and its launches 30.  With 2048 tokens, 2048 channels and 16 states, split
// and not: 4 rows 454 and 593 us, 6 rows 661 and 752 us, 7 rows 770 and 754 us; by the forward's segments 4 rows took 498 us.
SegPlan bwd_segments(const ScanP& p, int es) {
  const int nl = scan_lanes(p.N);
  const int64_t row = ((p.D / p.G + 256 / nl - 1) / (256 / nl)) * p.G, nb = std::max<int64_t>(p.B, 1) * row, slots = tiled_at_once(es, nl);
  SegPlan best = {1, p.T};
  int64_t least = 100 * ((nb + slots - 1) / slots) * (p.T + 16);
  for (int64_t k = 1; k <= 4; ++k) {
    const int64_t n = std::min<int64_t>(k * slots / nb, p.T / 32);
    if (n < 2 || n * n > 2 * (int64_t)p.T) continue;
    const int64_t len = ((p.T + n - 1) / n + GDN_SCAN_CKPT - 1) / GDN_SCAN_CKPT * GDN_SCAN_CKPT, segs = (p.T + len - 1) / len;
    const int64_t cost = 100 * ((nb * segs + slots - 1) / slots) * (len + 16) + 28 * p.T * nb / slots + 3000;
    if (segs > 1 && cost < least) {
      least = cost;
      best = {(int)segs, (int)len};
    }
  }
  return best;
}

ScanP bwd_params(const gdn_scan_bwd_args* a) {
  ScanP p = scan_params(&a->fwd);
  if (p.N % 4 == 0) {
    const SegPlan sp = bwd_segments(p, elem_size(a->fwd.dtype));
    p.nseg = sp.nseg;
    p.seg_len = sp.seg_len;
  }
  p.h_out = nullptr;
  p.dy = a->dy; p.sdy_b = a->sdy_b; p.sdy_t = a->sdy_t;
  p.dh_out = a->dh_out; p.dx = a->dx; p.ddt = a->ddt; p.dz = a->dz; p.dh0 = a->dh0;
  return p;
}

template <typename T, int NL>
int launch_bwd_tiled(const ScanP& p, cudaStream_t s) {
  using K = BwdTiled<T, NL>;
  static std::atomic<unsigned long long> opted{0};
  auto k = scan_bwd_tiled_kernel<T, NL>;
  if (!opt_in_smem(opted, {{(const void*)k, K::SMEM}})) return GDN_ERR_LAUNCH;
  for_grid_rows(p, sizeof(T), [&](const ScanP& q, unsigned rows) { k<<<dim3(p.dblocks * p.G, p.nseg, rows), SCAN_THREADS, K::SMEM, s>>>(q); });
  return launched();
}

template <typename T>
int launch_bwd(ScanP p, const gdn_scan_bwd_args* a, cudaStream_t s) {
  const int nl = scan_lanes(p.N);
  const bool tiled = p.tiled;
  if (tiled) p.dblocks = (int)((p.D / p.G + 256 / nl - 1) / (256 / nl));  // two channels per lane: half the blocks
  auto pair = [](const void* q) { return (uintptr_t)q % (2 * sizeof(T)) == 0; };
  p.pairs_out = (p.D / p.G) % 2 == 0 && pair(p.dx) && pair(p.ddt) && pair(p.dz);  // their rows are contiguous
  int st = GDN_OK;
  if (tiled) {
    st = nl == 2 ? launch_bwd_tiled<T, 2>(p, s) : nl == 4 ? launch_bwd_tiled<T, 4>(p, s) : nl == 8 ? launch_bwd_tiled<T, 8>(p, s) : launch_bwd_tiled<T, 16>(p, s);
  } else {
    for_grid_rows(p, sizeof(T), [&](const ScanP& q, unsigned rows) {
      const dim3 g(p.dblocks * p.G, p.nseg, rows);
      if (nl == 2) scan_bwd_kernel<T, 2><<<g, SCAN_THREADS, 0, s>>>(q);
      if (nl == 4) scan_bwd_kernel<T, 4><<<g, SCAN_THREADS, 0, s>>>(q);
      if (nl == 8) scan_bwd_kernel<T, 8><<<g, SCAN_THREADS, 0, s>>>(q);
      if (nl == 16) scan_bwd_kernel<T, 16><<<g, SCAN_THREADS, 0, s>>>(q);
    });
    st = launched();
  }
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
  const ScanP p = bwd_params(a);
  *bytes = bwd_plan(p).total * sizeof(float) + scan_align_plan(p, elem_size(a->fwd.dtype), true).total;
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
  if (!aligned16(a->fwd.workspace)) return GDN_ERR_ALIGN;
  if (!device_ok()) return GDN_ERR_DEVICE;
  ScanP p = bwd_params(a);
  const BwdPlan w = bwd_plan(p);
  float* ws = static_cast<float*>(f->workspace);
  p.carry = ws; ws += w.carry;
  p.ssum = ws; ws += w.ssum;
  p.pBC = ws; ws += w.bc;
  p.pA = ws; ws += w.a;
  p.pD = ws;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const AlignPlan al = scan_align_plan(p, elem_size(f->dtype), true);
  if (al.tiled) {
    st = scan_align(p, al, f->dtype, static_cast<char*>(f->workspace) + w.total * sizeof(float), s);
    if (st != GDN_OK) return st;
  }
  if (p.nseg > 1) {
    st = scan_launch_carry(p, f->dtype, true, s);
    if (st != GDN_OK) return st;
  }
  return f->dtype == GDN_DTYPE_F32 ? launch_bwd<float>(p, a, s) : launch_bwd<__nv_bfloat16>(p, a, s);
}

}  // extern "C"
