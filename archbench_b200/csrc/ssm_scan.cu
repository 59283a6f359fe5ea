// Selective scan, forward: prompts (one pass, or split over time when the batch has few rows) and single tokens.
//
//   s_t = softplus(dt_t + bias), h_t = exp(s_t A) h_{t-1} + s_t x_t B_t, y_t = (C_t . h_t + D x_t) silu(z_t)
//
// Bound by the exponentials: N of them per token and channel on 16 lanes per SM and clock, against 8 bytes of HBM
// traffic (bf16).  The state stays in registers for the whole sequence.
#include "ssm_scan.cuh"

namespace gdn {
namespace ssm {

constexpr int TT = 32;  // tokens per tile of the local pass; segments are whole tiles

// One (row, channel block, segment) per block of 128 threads.  Each tile is staged by the threads in their
// per-token role (a channel of some tokens): raw values of the next tile are already in registers while this one is
// computed, so no load is waited for.  In their per-state role the threads read (s, s, s x, s x) of their channel and
// the B and C of their four states, and leave their part of C . h in shared memory; the per-token role adds the parts.
template <typename T, int NL>
__global__ void __launch_bounds__(SCAN_THREADS, 4) scan_fwd_kernel(const ScanP p) {
  constexpr int TT = NL == 2 ? 16 : 32;  // tokens per tile (shared memory)
  constexpr int CH = SCAN_THREADS / NL, NP = NL * SPL;
  constexpr int TSTEP = SCAN_THREADS / CH, PER = TT / TSTEP;  // tokens covered at once, tokens per thread
  constexpr int QUADS = TT * NL / SCAN_THREADS > 0 ? TT * NL / SCAN_THREADS : 1;
  __shared__ __align__(16) float4 sS[TT][CH];
  __shared__ __align__(16) float sY[TT][SCAN_THREADS];
  __shared__ __align__(16) float sB[TT][NP], sC[TT][NP];
  const int tid = threadIdx.x;
  const int grp = blockIdx.x / p.dblocks, dblk = blockIdx.x % p.dblocks;
  const int seg = blockIdx.y, b = blockIdx.z;
  const int dpg = p.D / p.G, d0 = grp * dpg + dblk * CH, nch = min(CH, dpg - dblk * CH);
  const int len = row_tokens(p.lengths, b, p.T);
  const int tbeg = seg * p.seg_len, tend = min(tbeg + p.seg_len, p.T), lim = min(tend, len);

  // per-state role
  const int hc = tid / NL, n0 = (tid % NL) * SPL;
  const bool live = hc < nch;
  f32x2 h[2], A2[2];
  {
    float hv[SPL], av[SPL];
    const float* from = p.nseg > 1 ? p.carry + ((int64_t)b * p.nseg + seg) * p.D * p.N : p.h0 ? p.h0 + (int64_t)b * p.D * p.N : nullptr;
#pragma unroll
    for (int i = 0; i < SPL; ++i) {
      const bool ok = live && n0 + i < p.N;
      const int64_t at = (int64_t)(d0 + hc) * p.N + n0 + i;
      av[i] = ok ? p.A[at] * LOG2E : 0.f;
      hv[i] = ok && from ? from[at] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      h[i] = pack2(hv[2 * i], hv[2 * i + 1]);
      A2[i] = pack2(av[2 * i], av[2 * i + 1]);
    }
  }
  // per-token role: channel cc, tokens ct0, ct0 + TSTEP, ...
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

  T xr[PER], dr[PER], zr[PER];
  Quad<T> qb[QUADS], qc[QUADS];
  auto fetch = [&](int t0) {  // places past the row's tokens read its last one; their values are dropped
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int64_t t = min(t0 + ct0 + i * TSTEP, lim - 1);
      xr[i] = xp[t * p.sx_t];
      dr[i] = dtp[t * p.sdt_t];
      if (zp) zr[i] = zp[t * p.sz_t];
    }
#pragma unroll
    for (int i = 0; i < QUADS; ++i) {
      const int k = tid + i * SCAN_THREADS;
      if (TT * NL >= SCAN_THREADS || k < TT * NL) {
        const int64_t t = min(t0 + k / NL, lim - 1);
        qb[i] = load_quad(Bp + t * p.sB_t, k % NL * 4, p.N, p.quads);
        qc[i] = load_quad(Cp + t * p.sC_t, k % NL * 4, p.N, p.quads);
      }
    }
  };
  if (tbeg < lim) fetch(tbeg);
  int t0 = tbeg;
  for (; t0 < lim; t0 += TT) {
    float x[PER], z[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int r = ct0 + i * TSTEP;
      const bool on = t0 + r < lim;
      float s = to_f32(dr[i]) + bias;
      if (p.softplus) s = softplus(s);
      s = on ? s : 0.f;
      x[i] = to_f32(xr[i]);
      z[i] = zp ? to_f32(zr[i]) : 0.f;
      const float u = on ? s * x[i] : 0.f;
      sS[r][cc] = make_float4(s, s, u, u);
    }
#pragma unroll
    for (int i = 0; i < QUADS; ++i) {
      const int k = tid + i * SCAN_THREADS;
      if (TT * NL >= SCAN_THREADS || k < TT * NL) {
        const bool on = t0 + k / NL < lim;
        *reinterpret_cast<float4*>(&sB[k / NL][k % NL * 4]) = quad_f32(qb[i], on);
        *reinterpret_cast<float4*>(&sC[k / NL][k % NL * 4]) = quad_f32(qc[i], on);
      }
    }
    __syncthreads();
    if (t0 + TT < lim) fetch(t0 + TT);
#pragma unroll 1
    for (int r0 = 0; r0 < TT; r0 += GDN_SCAN_CKPT) {
      if (t0 + r0 >= lim) break;
      if (p.ckpt && live) {
        float* c = p.ckpt + (((int64_t)b * nck + (t0 + r0) / GDN_SCAN_CKPT) * p.D + d0 + hc) * p.N + n0;
        const float2 lo = unpack2(h[0]), hi = unpack2(h[1]);
        if (p.ckpt_quads) {
          if (n0 < p.N) *reinterpret_cast<float4*>(c) = make_float4(lo.x, lo.y, hi.x, hi.y);
        } else {
          const float hv[SPL] = {lo.x, lo.y, hi.x, hi.y};
#pragma unroll
          for (int i = 0; i < SPL; ++i)
            if (n0 + i < p.N) c[i] = hv[i];
        }
      }
#pragma unroll
      for (int q = 0; q < GDN_SCAN_CKPT; ++q) {
        const int r = r0 + q;
        const ulonglong2 su = *reinterpret_cast<const ulonglong2*>(&sS[r][hc]);
        const ulonglong2 bv = *reinterpret_cast<const ulonglong2*>(&sB[r][n0]);
        const ulonglong2 cv = *reinterpret_cast<const ulonglong2*>(&sC[r][n0]);
        h[0] = fma2(exp2_2(fma2(su.x, A2[0], both(EX2_MEAN))), h[0], mul2(su.y, bv.x));
        h[1] = fma2(exp2_2(fma2(su.x, A2[1], both(EX2_MEAN))), h[1], mul2(su.y, bv.y));
        sY[r][tid] = sum2(fma2(cv.y, h[1], mul2(cv.x, h[0])));
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int r = ct0 + i * TSTEP, t = t0 + r;
      if (!cok || t >= tend) continue;
      float y = 0.f;
      const float* part = &sY[r][cc * NL];
#pragma unroll
      for (int j = 0; j < NL; j += 2) {
        const float2 v = *reinterpret_cast<const float2*>(part + j);
        y += v.x + v.y;
      }
      y = fmaf(skip, x[i], y);
      if (zp) y *= silu(z[i]);
      store_as(yp + t * p.sy_t, t < lim ? y : 0.f);
    }
    // sS, sB and sC are rewritten only after every thread passed the barrier above; sY only after the next one
  }
  // past the row's tokens
  for (int t = t0 + ct0; t < tend; t += TSTEP)
    if (cok) store_as(yp + (int64_t)t * p.sy_t, 0.f);
  if (p.h_out && seg == p.nseg - 1 && live) {
    const float2 lo = unpack2(h[0]), hi = unpack2(h[1]);
    const float hv[SPL] = {lo.x, lo.y, hi.x, hi.y};
#pragma unroll
    for (int i = 0; i < SPL; ++i)
      if (n0 + i < p.N) p.h_out[((int64_t)b * p.D + d0 + hc) * p.N + n0 + i] = hv[i];
  }
}

// The same pass where N is a multiple of four (rows are 16-byte aligned, or were laid out so); one warp per block.  A lane holds SL states of two channels.
// What bounds it beside the exponentials is shared memory's 128 bytes a clock into registers (a broadcast saves nothing
// there), so a lane's B and C serve two channels: (s, u) of both, B and C are 48 bytes for eight states; with one
// channel per lane the recurrence alone cost 386 us at 8 x 4096 tokens, 2048 channels, 16 states.  A warp by itself needs
// no barrier, and 16 channels per block balance the 148 SMs better than 32.  Raw tiles of 8 tokens (16 take
// 4 % off 7 warps per SM and cost up to half where shared memory then holds 8 instead of 12 or more) come in by
// asynchronous copies; a thread runs the recurrence of tile k, forms the step sizes of tile k + 1 and finishes the
// outputs of tile k - 1 in one straight piece of code, so that their latencies overlap.
template <typename T, int NL, int SL>
struct Tiled {
  static constexpr int TT = 8, CH = 64 / NL, NP = NL * SL, ES = (int)sizeof(T), RING = 4;
  static constexpr int ROW = CH * ES, BROW = NP * ES;           // bytes of a token's channels, states
  static constexpr int RAW = TT * (3 * ROW + 2 * BROW);         // x, dt, z, B, C of a tile
  static constexpr int S_OFF = RING * RAW, S_BYTES = TT * CH * 8;
  static constexpr int Y_OFF = S_OFF + 2 * S_BYTES, Y_BYTES = TT * 32 * 8;
  static constexpr int BC_OFF = Y_OFF + 2 * Y_BYTES, BC_BYTES = 2 * TT * NP * 4;
  static constexpr int SMEM = BC_OFF + 2 * BC_BYTES;
  static constexpr int XCH = ROW / 16, BCH = BROW / 16;         // 16-byte chunks per row
  static constexpr int CHUNKS = TT * (3 * XCH + 2 * BCH), COPIES = (CHUNKS + 31) / 32;
};

template <typename T, int NL, int SL>
__global__ void __launch_bounds__(32) scan_fwd_tiled_kernel(const ScanP p) {
  using K = Tiled<T, NL, SL>;
  constexpr int TT = K::TT, CH = K::CH, NP = K::NP, PAIRS = SL / 2;
  constexpr int PER = TT / NL;           // (token, channel pair) items per lane
  constexpr int QUADS = TT * NP / 64;    // four-state groups of B and C per lane
  constexpr int GT = 2, GROUPS = TT / GT;  // tokens whose loads go together
  extern __shared__ __align__(16) char smem[];
  const int lane = threadIdx.x;
  const int grp = blockIdx.x / p.dblocks, dblk = blockIdx.x % p.dblocks;
  const int seg = blockIdx.y, b = blockIdx.z;
  const int dpg = p.D / p.G, d0 = grp * dpg + dblk * CH, nch = min(CH, dpg - dblk * CH);
  const int len = row_tokens(p.lengths, b, p.T);
  const int tbeg = seg * p.seg_len, tend = min(tbeg + p.seg_len, p.T), lim = min(tend, len);
  const int ntile = lim > tbeg ? (lim - tbeg + TT - 1) / TT : 0;

  // this lane's copies of a tile: destination in the ring slot, source and its step from tile to tile
  const char* src[K::COPIES];
  int64_t step[K::COPIES];
  uint32_t dst[K::COPIES];
  int tok[K::COPIES];  // token in the tile, or a large one for zeros
  constexpr int NONE = 1 << 29;
#pragma unroll
  for (int i = 0; i < K::COPIES; ++i) {
    int c = lane + i * 32;
    tok[i] = NONE;
    src[i] = static_cast<const char*>(p.x);
    step[i] = 0;
    dst[i] = c * 16;
    const void* base;
    int64_t sb, st, off;
    int r, j, bytes;
    if (c < 3 * TT * K::XCH) {
      const int which = c / (TT * K::XCH);
      r = c / K::XCH % TT; j = c % K::XCH; bytes = nch * K::ES; off = (int64_t)grp * p.xgs + dblk * CH;
      base = which == 0 ? p.x : which == 1 ? p.dt : p.z;
      sb = which == 0 ? p.sx_b : which == 1 ? p.sdt_b : p.sz_b;
      st = which == 0 ? p.sx_t : which == 1 ? p.sdt_t : p.sz_t;
    } else {
      c -= 3 * TT * K::XCH;
      const int which = c / (TT * K::BCH);
      r = c / K::BCH % TT; j = c % K::BCH; bytes = which < 2 ? p.N * K::ES : 0;
      base = which ? p.Cm : p.Bm;
      sb = which ? p.sC_b : p.sB_b;
      st = which ? p.sC_t : p.sB_t;
      off = grp * (which ? p.sC_g : p.sB_g);
    }
    if (base && j * 16 < bytes) {
      tok[i] = r;
      src[i] = static_cast<const char*>(base) + (b * sb + (tbeg + r) * st + off) * K::ES + j * 16;
      step[i] = st * TT * K::ES;
    }
  }
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(smem));
  auto fetch = [&](int k) {  // tile k into slot k % RING; an empty group past the last tile keeps the counts equal
    if (k < ntile) {
#pragma unroll
      for (int i = 0; i < K::COPIES; ++i) {
        if (K::CHUNKS % 32 == 0 || lane + i * 32 < K::CHUNKS)
          copy16(ring + (k & (K::RING - 1)) * K::RAW + dst[i], src[i], tbeg + k * TT + tok[i] < lim);
        src[i] += step[i];
      }
    }
    copies_commit();
  };

  // per-state role: channels hc, hc + 1
  const int hc = lane / NL * 2, n0 = lane % NL * SL;
  const bool live = hc < nch && n0 < p.N;
  f32x2 h[2][PAIRS];
  float A2[2][SL];
  const float* from = p.nseg > 1 ? p.carry + ((int64_t)b * p.nseg + seg) * p.D * p.N : p.h0 ? p.h0 + (int64_t)b * p.D * p.N : nullptr;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    float hv[SL];
#pragma unroll
    for (int i = 0; i < SL; ++i) {
      const bool ok = live && hc + c < nch && n0 + i < p.N;
      const int64_t at = (int64_t)(d0 + hc + c) * p.N + n0 + i;
      A2[c][i] = ok ? p.A[at] * LOG2E : 0.f;
      hv[i] = ok && from ? from[at] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) h[c][i] = pack2(hv[2 * i], hv[2 * i + 1]);
  }
  auto put_states = [&](float* to) {  // rows of N (a multiple of 4) states at channel d0
    if (!live) return;
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int i = 0; i < PAIRS; i += 2)
        if (hc + c < nch && n0 + 2 * i < p.N)
          *reinterpret_cast<ulonglong2*>(to + (int64_t)(hc + c) * p.N + n0 + 2 * i) = make_ulonglong2(h[c][i], h[c][i + 1]);
  };
  // per-token role: channels cc, cc + 1, tokens ct0, ct0 + NL, ...
  const int cc = lane % (CH / 2) * 2, ct0 = lane / (CH / 2);
  const bool cok = cc < nch;
  const int d = d0 + (cok ? cc : 0);
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
  T* yp = static_cast<T*>(p.y) + b * p.sy_b + d;
  const int nck = (p.T + GDN_SCAN_CKPT - 1) / GDN_SCAN_CKPT;

  // The three pieces of work of an item, each as loads, arithmetic and stores apart: shared memory's stores and loads
  // keep their order, so a load behind a store would wait for all that the store waits for.
  struct Stage {  // (s, u) of a channel pair at a token of tile k
    f32x2 dt, x;
  };
  auto stage_load = [&](int k, int i) {
    const char* raw = smem + (k & (K::RING - 1)) * K::RAW + (ct0 + i * NL) * K::ROW + cc * K::ES;
    return Stage{load_pair(reinterpret_cast<const T*>(raw + TT * K::ROW)), load_pair(reinterpret_cast<const T*>(raw))};
  };
  auto stage_make = [&](int k, int i, const Stage& g) {
    f32x2 s = add2(g.dt, bias);
    s = p.softplus ? softplus2(s) : s;
    const float2 uv = unpack2(mul2(s, g.x)), sv = unpack2(s);
    const bool on = tbeg + k * TT + ct0 + i * NL < lim;
    return on ? make_float4(sv.x, uv.x, sv.y, uv.y) : make_float4(0.f, 0.f, 0.f, 0.f);
  };
  auto stage_store = [&](int k, int i, const float4& v) {
    *(reinterpret_cast<float4*>(smem + K::S_OFF + (k & 1) * K::S_BYTES) + ((ct0 + i * NL) * CH + cc) / 2) = v;
  };
  auto bc_load = [&](int k, int i) {  // four states of B or C in fp32 (zeros past the tokens and the states)
    const T* raw = reinterpret_cast<const T*>(smem + (k & (K::RING - 1)) * K::RAW + 3 * TT * K::ROW) + (lane + i * 32) * 4;
    return make_ulonglong2(load_pair(raw), load_pair(raw + 2));
  };
  auto bc_store = [&](int k, int i, const ulonglong2& v) {
    *reinterpret_cast<ulonglong2*>(smem + K::BC_OFF + (k & 1) * K::BC_BYTES + (lane + i * 32) * 16) = v;
  };
  struct Finish {  // the outputs of a channel pair at a token of tile k
    f32x2 core, x, z;
  };
  auto finish_load = [&](int k, int i) {
    const int r = ct0 + i * NL;
    // the pair's parts from its NL lanes; odd lanes start with the second half, or half the banks would idle
    const char* part = smem + K::Y_OFF + (k & 1) * K::Y_BYTES + (r * 32 + cc / 2 * NL) * 8;
    f32x2 a[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const char* q = part + ((e ^ lane) & 1) * NL * 4;
      if (NL == 2) {
        a[e] = *reinterpret_cast<const f32x2*>(q);
      } else {
#pragma unroll
        for (int j = 0; j < NL / 2; j += 2) {
          const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(q + j * 8);
          a[e] = j ? add2(a[e], add2(v.x, v.y)) : add2(v.x, v.y);
        }
      }
    }
    const char* raw = smem + (k & (K::RING - 1)) * K::RAW + r * K::ROW + cc * K::ES;
    return Finish{add2(a[0], a[1]), load_pair(reinterpret_cast<const T*>(raw)), load_pair(reinterpret_cast<const T*>(raw + 2 * TT * K::ROW))};
  };
  auto finish_store = [&](int k, int i, const Finish& g) {
    const int t = tbeg + k * TT + ct0 + i * NL;
    const f32x2 gate = p.z ? mul2(g.z, sigmoid2(g.z)) : both(1.f);
    const float2 v = unpack2(mul2(fma2(skip, g.x, g.core), gate));
    const float out[2] = {t < lim ? v.x : 0.f, t < lim ? v.y : 0.f};
    if (cok && t >= tbeg && t < tend) put_pair(yp + t * p.sy_t, out);
  };
  struct Tokens {  // what GT tokens of the recurrence read
    float4 su[GT], b[GT][SL / 4];
    ulonglong2 c[GT][SL / 4];
  };
  auto tokens_load = [&](int k, int r0) {
    Tokens g;
    const float4* sS = reinterpret_cast<const float4*>(smem + K::S_OFF + (k & 1) * K::S_BYTES) + hc / 2;
    const float* sB = reinterpret_cast<const float*>(smem + K::BC_OFF + (k & 1) * K::BC_BYTES) + n0;
#pragma unroll
    for (int q = 0; q < GT; ++q) {
      g.su[q] = sS[(r0 + q) * (CH / 2)];
#pragma unroll
      for (int i = 0; i < SL / 4; ++i) {
        g.b[q][i] = *reinterpret_cast<const float4*>(sB + (r0 + q) * NP + 4 * i);
        g.c[q][i] = *reinterpret_cast<const ulonglong2*>(sB + (TT + r0 + q) * NP + 4 * i);
      }
    }
    return g;
  };

  fetch(0);
  fetch(1);
  if (ntile > 0) {
    copies_wait<1>();
    __syncwarp();
#pragma unroll
    for (int i = 0; i < PER; ++i) stage_store(0, i, stage_make(0, i, stage_load(0, i)));
#pragma unroll
    for (int i = 0; i < QUADS; ++i) bc_store(0, i, bc_load(0, i));
  }
#pragma unroll 1
  for (int k = 0; k < ntile; ++k) {
    copies_wait<0>();  // tile k + 1, issued one iteration ago
    __syncwarp();
    fetch(k + 2);
    f32x2* sY = reinterpret_cast<f32x2*>(smem + K::Y_OFF + (k & 1) * K::Y_BYTES) + lane;
    if (p.ckpt) put_states(p.ckpt + (((int64_t)b * nck + (tbeg + k * TT) / GDN_SCAN_CKPT) * p.D + d0) * p.N);
    // no branches from here on: past the last tile the staged values go unused, before the first one the stores are off
    Tokens cur = tokens_load(k, 0);
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      constexpr int SI = (PER + GROUPS - 1) / GROUPS, QI = (QUADS + GROUPS - 1) / GROUPS;
      Stage st[SI];
      Finish fi[SI];
      ulonglong2 bc[QI];
      float4 made[SI];
      const int i0 = g * PER / GROUPS, i1 = (g + 1) * PER / GROUPS, q0 = g * QUADS / GROUPS, q1 = (g + 1) * QUADS / GROUPS;
#pragma unroll
      for (int i = i0; i < i1; ++i) {
        st[i - i0] = stage_load(k + 1, i);
        fi[i - i0] = finish_load(k - 1, i);
      }
#pragma unroll
      for (int i = q0; i < q1; ++i) bc[i - q0] = bc_load(k + 1, i);
      Tokens nxt = cur;
      if (g + 1 < GROUPS) nxt = tokens_load(k, (g + 1) * GT);
      if (p.ckpt && g > 0 && g * GT % GDN_SCAN_CKPT == 0 && tbeg + k * TT + g * GT < lim)
        put_states(p.ckpt + (((int64_t)b * nck + (tbeg + k * TT + g * GT) / GDN_SCAN_CKPT) * p.D + d0) * p.N);
      f32x2 y[GT];
#pragma unroll
      for (int q = 0; q < GT; ++q) {
        const float4 su = cur.su[q];
        f32x2 y0, y1;
#pragma unroll
        for (int i = 0; i < PAIRS; i += 2) {
          const float4 bv = cur.b[q][i / 2];
          const ulonglong2 cv = cur.c[q][i / 2];
          h[0][i] = fma2(pack2(decay(su.x, A2[0][2 * i]), decay(su.x, A2[0][2 * i + 1])), h[0][i], pack2(su.y * bv.x, su.y * bv.y));
          h[1][i] = fma2(pack2(decay(su.z, A2[1][2 * i]), decay(su.z, A2[1][2 * i + 1])), h[1][i], pack2(su.w * bv.x, su.w * bv.y));
          h[0][i + 1] = fma2(pack2(decay(su.x, A2[0][2 * i + 2]), decay(su.x, A2[0][2 * i + 3])), h[0][i + 1], pack2(su.y * bv.z, su.y * bv.w));
          h[1][i + 1] = fma2(pack2(decay(su.z, A2[1][2 * i + 2]), decay(su.z, A2[1][2 * i + 3])), h[1][i + 1], pack2(su.w * bv.z, su.w * bv.w));
          y0 = fma2(cv.y, h[0][i + 1], i ? fma2(cv.x, h[0][i], y0) : mul2(cv.x, h[0][i]));
          y1 = fma2(cv.y, h[1][i + 1], i ? fma2(cv.x, h[1][i], y1) : mul2(cv.x, h[1][i]));
        }
        y[q] = pack2(sum2(y0), sum2(y1));
      }
#pragma unroll
      for (int i = i0; i < i1; ++i) made[i - i0] = stage_make(k + 1, i, st[i - i0]);
#pragma unroll
      for (int i = i0; i < i1; ++i) {
        finish_store(k - 1, i, fi[i - i0]);
        stage_store(k + 1, i, made[i - i0]);
      }
#pragma unroll
      for (int i = q0; i < q1; ++i) bc_store(k + 1, i, bc[i - q0]);
#pragma unroll
      for (int q = 0; q < GT; ++q) sY[(g * GT + q) * 32] = y[q];
      cur = nxt;
    }
  }
  __syncwarp();
  if (ntile > 0) {
#pragma unroll
    for (int i = 0; i < PER; ++i) finish_store(ntile - 1, i, finish_load(ntile - 1, i));
  }
  // past the row's tokens
  const float zero[2] = {0.f, 0.f};
  if (cok)
    for (int t = tbeg + ntile * TT + ct0; t < tend; t += NL) put_pair(yp + t * p.sy_t, zero);
  if (p.h_out && seg == p.nseg - 1) put_states(p.h_out + ((int64_t)b * p.D + d0) * p.N);
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
        const float a = decay(ss.x, A2[i]);
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

// The same where N is a multiple of four: scan_fwd_tiled_kernel without outputs.  Reversed, tiles and their tokens
// run from the last to the first.
template <typename T, int NL, int SL>
struct CarryTiled {
  static constexpr int TT = 8, CH = 64 / NL, NP = NL * SL, ES = (int)sizeof(T), RING = 4;
  static constexpr int ROW = CH * ES, BROW = NP * ES;
  static constexpr int RAW = TT * (3 * ROW + BROW);  // x, dt and B, or dy, dt, z and C
  static constexpr int S_OFF = RING * RAW, S_BYTES = TT * CH * 8;
  static constexpr int BC_OFF = S_OFF + 2 * S_BYTES, BC_BYTES = TT * NP * 4;
  static constexpr int SMEM = BC_OFF + 2 * BC_BYTES;
  static constexpr int XCH = ROW / 16, BCH = BROW / 16;
  static constexpr int CHUNKS = TT * (3 * XCH + BCH), COPIES = (CHUNKS + 31) / 32;
};

template <typename T, int NL, int SL, bool REV>
__global__ void __launch_bounds__(32) scan_carry_tiled_kernel(const ScanP p) {
  using K = CarryTiled<T, NL, SL>;
  constexpr int TT = K::TT, CH = K::CH, NP = K::NP, PAIRS = SL / 2, PER = TT / NL, QUADS = TT * NP / 4;
  constexpr int QI = (QUADS + 31) / 32;
  extern __shared__ __align__(16) char smem[];
  const int lane = threadIdx.x;
  const int grp = blockIdx.x / p.dblocks, dblk = blockIdx.x % p.dblocks;
  const int seg = blockIdx.y, b = blockIdx.z;
  if (seg == (REV ? 0 : p.nseg - 1)) return;  // nothing enters from here
  const int dpg = p.D / p.G, d0 = grp * dpg + dblk * CH, nch = min(CH, dpg - dblk * CH);
  const int len = row_tokens(p.lengths, b, p.T);
  const int tbeg = seg * p.seg_len, lim = min(min(tbeg + p.seg_len, p.T), len);
  const int ntile = lim > tbeg ? (lim - tbeg + TT - 1) / TT : 0;
  auto tile = [&](int k) { return REV ? ntile - 1 - k : k; };

  const char* src[K::COPIES];
  int64_t step[K::COPIES];
  int tok[K::COPIES];
  constexpr int NONE = 1 << 29;
#pragma unroll
  for (int i = 0; i < K::COPIES; ++i) {
    int c = lane + i * 32;
    tok[i] = NONE;
    src[i] = static_cast<const char*>(p.dt);
    step[i] = 0;
    const void* base;
    int64_t sb, st, off;
    int r, j, bytes;
    if (c < 3 * TT * K::XCH) {
      const int which = c / (TT * K::XCH);
      r = c / K::XCH % TT; j = c % K::XCH; bytes = nch * K::ES; off = (int64_t)grp * p.xgs + dblk * CH;
      base = which == 1 ? p.dt : which == 2 ? (REV ? p.z : nullptr) : REV ? p.dy : p.x;
      sb = which == 1 ? p.sdt_b : which == 2 ? p.sz_b : REV ? p.sdy_b : p.sx_b;
      st = which == 1 ? p.sdt_t : which == 2 ? p.sz_t : REV ? p.sdy_t : p.sx_t;
    } else {
      c -= 3 * TT * K::XCH;
      r = c / K::BCH; j = c % K::BCH; bytes = r < TT ? p.N * K::ES : 0;
      base = REV ? p.Cm : p.Bm;
      sb = REV ? p.sC_b : p.sB_b;
      st = REV ? p.sC_t : p.sB_t;
      off = grp * (REV ? p.sC_g : p.sB_g);
    }
    if (base && j * 16 < bytes) {
      tok[i] = r;
      src[i] = static_cast<const char*>(base) + (b * sb + ((int64_t)tbeg + tile(0) * TT + r) * st + off) * K::ES + j * 16;
      step[i] = (REV ? -st : st) * TT * K::ES;
    }
  }
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(smem));
  auto fetch = [&](int k) {
    if (k < ntile) {
#pragma unroll
      for (int i = 0; i < K::COPIES; ++i) {
        if (K::CHUNKS % 32 == 0 || lane + i * 32 < K::CHUNKS)
          copy16(ring + (k & (K::RING - 1)) * K::RAW + (lane + i * 32) * 16, src[i], tbeg + tile(k) * TT + tok[i] < lim);
        src[i] += step[i];
      }
    }
    copies_commit();
  };
  const int hc = lane / NL * 2, n0 = lane % NL * SL;
  const bool live = hc < nch && n0 < p.N;
  f32x2 h[2][PAIRS];
  float A2[2][SL];
#pragma unroll
  for (int c = 0; c < 2; ++c) {
#pragma unroll
    for (int i = 0; i < SL; ++i) A2[c][i] = live && hc + c < nch && n0 + i < p.N ? p.A[(int64_t)(d0 + hc + c) * p.N + n0 + i] * LOG2E : 0.f;
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) h[c][i] = both(0.f);
  }
  const int cc = lane % (CH / 2) * 2, ct0 = lane / (CH / 2);
  const int d = d0 + (cc < nch ? cc : 0);
  const bool two = cc + 1 < nch;  // an odd group's last pair has one channel
  const f32x2 bias = p.dt_bias ? pack2(p.dt_bias[d], two ? p.dt_bias[d + 1] : 0.f) : both(0.f);
  f32x2 total = both(0.f);
  auto stage = [&](int k, int i) {
    const int r = ct0 + i * NL;
    const char* raw = smem + (k & (K::RING - 1)) * K::RAW + r * K::ROW + cc * K::ES;
    f32x2 s = add2(load_pair(reinterpret_cast<const T*>(raw + TT * K::ROW)), bias);
    s = p.softplus ? softplus2(s) : s;
    f32x2 u = load_pair(reinterpret_cast<const T*>(raw));
    if (REV) {
      const f32x2 z = load_pair(reinterpret_cast<const T*>(raw + 2 * TT * K::ROW));
      u = p.z ? mul2(u, mul2(z, sigmoid2(z))) : u;
    } else {
      u = mul2(u, s);
    }
    const bool on = tbeg + tile(k) * TT + r < lim;
    s = on ? s : both(0.f);
    u = on ? u : both(0.f);
    total = add2(total, s);
    const float2 sv = unpack2(s), uv = unpack2(u);
    return make_float4(sv.x, uv.x, sv.y, uv.y);
  };
  auto stage_all = [&](int k) {
    float4 v[PER];
    ulonglong2 q[QI];
#pragma unroll
    for (int i = 0; i < PER; ++i) v[i] = stage(k, i);
#pragma unroll
    for (int i = 0; i < QI; ++i) {
      if (QUADS % 32 && lane + i * 32 >= QUADS) break;
      const T* raw = reinterpret_cast<const T*>(smem + (k & (K::RING - 1)) * K::RAW + 3 * TT * K::ROW) + (lane + i * 32) * 4;
      q[i] = make_ulonglong2(load_pair(raw), load_pair(raw + 2));
    }
#pragma unroll
    for (int i = 0; i < PER; ++i)
      *(reinterpret_cast<float4*>(smem + K::S_OFF + (k & 1) * K::S_BYTES) + ((ct0 + i * NL) * CH + cc) / 2) = v[i];
#pragma unroll
    for (int i = 0; i < QI; ++i) {
      if (QUADS % 32 && lane + i * 32 >= QUADS) break;
      reinterpret_cast<ulonglong2*>(smem + K::BC_OFF + (k & 1) * K::BC_BYTES)[lane + i * 32] = q[i];
    }
  };
  fetch(0);
  fetch(1);
  if (ntile > 0) {
    copies_wait<1>();
    __syncwarp();
    stage_all(0);
  }
#pragma unroll 1
  for (int k = 0; k < ntile; ++k) {
    copies_wait<0>();
    __syncwarp();
    fetch(k + 2);
    const float4* sS = reinterpret_cast<const float4*>(smem + K::S_OFF + (k & 1) * K::S_BYTES) + hc / 2;
    const float* sB = reinterpret_cast<const float*>(smem + K::BC_OFF + (k & 1) * K::BC_BYTES) + n0;
#pragma unroll
    for (int q = 0; q < TT; ++q) {  // only reads until the staging of the next tile
      const int r = REV ? TT - 1 - q : q;
      const float4 su = sS[r * (CH / 2)];
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) {
        const float2 bv = *reinterpret_cast<const float2*>(sB + r * NP + 2 * i);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float s = c ? su.z : su.x, u = c ? su.w : su.y;
          const f32x2 a = pack2(decay(s, A2[c][2 * i]), decay(s, A2[c][2 * i + 1])), w = pack2(u * bv.x, u * bv.y);
          h[c][i] = REV ? mul2(a, add2(h[c][i], w)) : fma2(a, h[c][i], w);
        }
      }
    }
    if (k + 1 < ntile) stage_all(k + 1);
  }
  const int64_t row = (int64_t)b * p.nseg + seg;
  if (live) {
    float* to = p.carry + (row * p.D + d0) * p.N;
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int i = 0; i < PAIRS; i += 2)
        if (hc + c < nch && n0 + 2 * i < p.N)
          *reinterpret_cast<ulonglong2*>(to + (int64_t)(hc + c) * p.N + n0 + 2 * i) = make_ulonglong2(h[c][i], h[c][i + 1]);
  }
  float2 sum = unpack2(total);
#pragma unroll
  for (int o = CH / 2; o < 32; o *= 2) {
    sum.x += __shfl_xor_sync(0xffffffffu, sum.x, o);
    sum.y += __shfl_xor_sync(0xffffffffu, sum.y, o);
  }
  if (ct0 == 0 && cc < nch) {
    p.ssum[row * p.D + d0 + cc] = sum.x;
    if (two) p.ssum[row * p.D + d0 + cc + 1] = sum.y;
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
  constexpr int BATCH = 8;  // segments whose values are read together
  for (int k0 = 0; k0 < p.nseg; k0 += BATCH) {
    float e[BATCH], a[BATCH];
#pragma unroll
    for (int q = 0; q < BATCH; ++q) {
      const int seg = REV ? p.nseg - 1 - (k0 + q) : k0 + q;
      const bool in = k0 + q < p.nseg && seg != last;
      e[q] = in ? p.carry[(b * p.nseg + seg) * dn + at] : 0.f;
      a[q] = in ? p.ssum[(b * p.nseg + seg) * p.D + d] : 0.f;
    }
#pragma unroll
    for (int q = 0; q < BATCH; ++q) {
      const int seg = REV ? p.nseg - 1 - (k0 + q) : k0 + q;
      if (k0 + q >= p.nseg) break;
      p.carry[(b * p.nseg + seg) * dn + at] = H;
      H = H == 0.f ? e[q] : fmaf(decay(a[q], A2), H, e[q]);  // zero times a growth past fp32 is zero
    }
  }
}

// One token per row: the state is read and written once, 16 bytes per access where N is a multiple of four.  Step size, gate
// and addresses are the same for all lanes of a channel, so a lane holds eight states (256 x 2048 channels, 16 states, four
// batches in turn: 21.0 us in blocks of 64 threads, 22.7 us of 128; 24.8 us with four or sixteen states; 33 us and more with
// several rows per thread).  Reading and writing that state in place alone takes 13.7 us.
constexpr int STEP_SL = 8, STEP_THREADS = 64;
template <typename T, int NL, bool VEC>
__global__ void __launch_bounds__(STEP_THREADS) scan_step_kernel(const ScanP p) {
  const int at = (blockIdx.x * STEP_THREADS + threadIdx.x) / NL;  // a channel of row b
  const int n0 = (threadIdx.x % NL) * STEP_SL, lane = threadIdx.x % 32;
  const bool live = at < p.D && n0 < p.N;
  const int b = blockIdx.y, d = live ? at : 0;
  const int grp = p.G == 1 ? 0 : d / (p.D / p.G);
  float* hp = p.h_out + ((int64_t)b * p.D + d) * p.N + n0;
  const float* Ap = p.A + (int64_t)d * p.N + n0;
  const T* Bp = static_cast<const T*>(p.Bm) + b * p.sB_b + grp * p.sB_g;
  const T* Cp = static_cast<const T*>(p.Cm) + b * p.sC_b + grp * p.sC_g;
  constexpr int Q = STEP_SL / 4;
  float h[Q][4], A[Q][4], y[1] = {0.f}, x = 0.f, s = 0.f, z = 0.f;
  Quad<T> qb[Q], qc[Q];
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    const bool in = live && n0 + 4 * q < p.N;
    if (VEC) {
      if (in) {
        load_vec<4>(hp + 4 * q, h[q]);
        load_vec<4>(Ap + 4 * q, A[q]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool one = live && n0 + 4 * q + i < p.N;
        h[q][i] = one ? hp[4 * q + i] : 0.f;
        A[q][i] = one ? Ap[4 * q + i] : 0.f;
      }
    }
    if (in) {
      qb[q] = load_quad(Bp, n0 + 4 * q, p.N, VEC && p.quads);
      qc[q] = load_quad(Cp, n0 + 4 * q, p.N, VEC && p.quads);
    }
  }
  if (live) {
    x = to_f32(static_cast<const T*>(p.x)[b * p.sx_b + d]);
    s = to_f32(static_cast<const T*>(p.dt)[b * p.sdt_b + d]) + (p.dt_bias ? p.dt_bias[d] : 0.f);
    if (p.z) z = to_f32(static_cast<const T*>(p.z)[b * p.sz_b + d]);
    if (p.softplus) s = softplus(s);
    const float u = s * x, s2 = s * LOG2E;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      if (n0 + 4 * q >= p.N) break;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        h[q][i] = fmaf(decay(s2, A[q][i]), h[q][i], u * to_f32(qb[q].v[i]));
        y[0] = fmaf(to_f32(qc[q].v[i]), h[q][i], y[0]);
      }
      if (VEC) {
        *reinterpret_cast<float4*>(hp + 4 * q) = make_float4(h[q][0], h[q][1], h[q][2], h[q][3]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (n0 + 4 * q + i < p.N) hp[4 * q + i] = h[q][i];
      }
    }
  }
  spread_sum<1, NL, 1>(y, lane);
  if (live && n0 == 0) {
    float o = y[0] + (p.Dskip ? p.Dskip[d] * x : 0.f);
    if (p.z) o *= silu(z);
    store_as(static_cast<T*>(p.y) + b * p.sy_b + d, o);
  }
}

// Time is split where the rows leave the SMs short of warps.  A split adds the local pass (0.6 of the scan's own work);
// a warp alone on a scheduler runs at 0.11 of the rate of a full SM (16 warps), so splitting pays below about 5 warps
// per SM, and then fills one wave (1 x 65536 tokens, 2048 channels: 128 warps unsplit, 18 segments).
SegPlan scan_segments(int64_t B, int64_t T, int64_t warps_per_row) {
  constexpr int64_t SMS = 148, MIN_SEG = 32;
  const SegPlan one = {1, (int)T};
  const int64_t warps = B * warps_per_row;
  if (warps >= SMS * 5 || T < 4 * MIN_SEG) return one;
  int64_t n = SMS * 16 / warps;
  while (n > 1 && n * n > 2 * T) --n;  // the combination walks the segments: sqrt(2 T) balances its steps and a segment's
  if (n > T / MIN_SEG) n = T / MIN_SEG;
  if (n < 2) return one;
  const int64_t len = ((T + n - 1) / n + TT - 1) / TT * TT;
  return {(int)((T + len - 1) / len), (int)len};
}

namespace {
bool rows16(const void* q, int v, int64_t a, int64_t b, int64_t c = 0) { return aligned16(q) && a % v == 0 && b % v == 0 && c % v == 0; }
size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }
}  // namespace

AlignPlan scan_align_plan(const ScanP& p, int es, bool bwd) {
  AlignPlan a = {};
  a.tiled = p.N % 4 == 0 && aligned16(p.A) && aligned16(p.h_out) && aligned16(p.ckpt) && aligned16(p.dh_out) && aligned16(p.dh0);
  if (!a.tiled) return a;
  const int v = 16 / es, dpg = p.D / p.G;
  const bool all = dpg % v != 0;  // groups would start off a 16-byte boundary
  a.x = all || !rows16(p.x, v, p.sx_b, p.sx_t);
  a.dt = all || !rows16(p.dt, v, p.sdt_b, p.sdt_t);
  a.z = p.z && (all || !rows16(p.z, v, p.sz_b, p.sz_t));
  a.dy = bwd && (all || !rows16(p.dy, v, p.sdy_b, p.sdy_t));
  a.B = p.N % v != 0 || !rows16(p.Bm, v, p.sB_b, p.sB_t, p.sB_g);
  a.C = p.N % v != 0 || !rows16(p.Cm, v, p.sC_b, p.sC_t, p.sC_g);
  const size_t tok = (size_t)p.B * p.T * p.G * es;
  a.xb = up256(tok * ((dpg + v - 1) / v * v));
  a.bb = up256(tok * ((p.N + v - 1) / v * v));
  a.total = a.xb * (a.x + a.dt + a.z + a.dy) + a.bb * (a.B + a.C);
  return a;
}

// dst (tokens, G, padded) <- src (b, t, G groups of `width` values), zeros in the padding; 16 bytes per thread.
struct AlignP {
  const void* src[6];
  void* dst[6];
  int64_t sb[6], st[6], sg[6];
  int width[6];
  int64_t tokens;
  int T, G;
};
template <typename T, typename I>  // I: 32-bit indices where they reach (divisions by 64-bit ones cost more than the copy)
__global__ void __launch_bounds__(256) scan_align_kernel(const AlignP p) {
  constexpr int V = 16 / (int)sizeof(T);
  const int k = blockIdx.y, w = p.width[k], chunks = (w + V - 1) / V;
  const I n = (I)(p.tokens * p.G * chunks), T_ = (I)p.T, G = (I)p.G;
  for (I i = (I)blockIdx.x * 256 + threadIdx.x; i < n; i += (I)gridDim.x * 256) {
    const I row = i / chunks, tok = row / G, b = tok / T_;
    const int c = (int)(i - row * chunks) * V;
    const T* src = static_cast<const T*>(p.src[k]) + b * p.sb[k] + (tok - b * T_) * p.st[k] + (row - tok * G) * p.sg[k] + c;
    uint4 raw = make_uint4(0, 0, 0, 0);
    T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (c + j < w) e[j] = src[j];
    static_cast<uint4*>(p.dst[k])[i] = raw;
  }
}

int scan_align(ScanP& p, const AlignPlan& a, int dtype, char* ws, cudaStream_t s) {
  const int es = elem_size(dtype), v = 16 / es, dpg = p.D / p.G;
  const int64_t dp = (dpg + v - 1) / v * v, np = (p.N + v - 1) / v * v;
  p.tiled = 1;
  p.xgs = dpg;
  AlignP q = {};
  int n = 0;
  auto move = [&](bool on, const void*& ptr, int64_t& sb, int64_t& st, int64_t* sg, int64_t from_g, int width, int64_t padded, size_t bytes) {
    if (!on) return;
    q.src[n] = ptr; q.dst[n] = ws; q.sb[n] = sb; q.st[n] = st; q.sg[n] = from_g; q.width[n] = width;
    ptr = ws; st = p.G * padded; sb = p.T * st;
    if (sg) *sg = padded;
    ws += bytes;
    ++n;
  };
  move(a.x, p.x, p.sx_b, p.sx_t, nullptr, dpg, dpg, dp, a.xb);
  move(a.dt, p.dt, p.sdt_b, p.sdt_t, nullptr, dpg, dpg, dp, a.xb);
  move(a.z, p.z, p.sz_b, p.sz_t, nullptr, dpg, dpg, dp, a.xb);
  move(a.dy, p.dy, p.sdy_b, p.sdy_t, nullptr, dpg, dpg, dp, a.xb);
  move(a.B, p.Bm, p.sB_b, p.sB_t, &p.sB_g, p.sB_g, p.N, np, a.bb);
  move(a.C, p.Cm, p.sC_b, p.sC_t, &p.sC_g, p.sC_g, p.N, np, a.bb);
  if (!n) return GDN_OK;
  if (dpg % v) p.xgs = (int)dp;
  q.tokens = (int64_t)p.B * p.T; q.T = p.T; q.G = p.G;
  const int64_t chunks = q.tokens * p.G * ((dpg > p.N ? dp : np) / v), g = (chunks + 255) / 256;
  const dim3 grid((unsigned)(g < 148 * 16 ? g : 148 * 16), n);
  const bool wide = chunks > (1ll << 31);
  if (dtype == GDN_DTYPE_F32)
    wide ? scan_align_kernel<float, uint64_t><<<grid, 256, 0, s>>>(q) : scan_align_kernel<float, uint32_t><<<grid, 256, 0, s>>>(q);
  else
    wide ? scan_align_kernel<__nv_bfloat16, uint64_t><<<grid, 256, 0, s>>>(q) : scan_align_kernel<__nv_bfloat16, uint32_t><<<grid, 256, 0, s>>>(q);
  return launched();
}

int scan_check(const gdn_scan_args* a, bool step) {
  if (!a) return GDN_ERR_NULL;
  if (a->B < 0 || a->T < 0 || a->D < 1 || a->N < 1 || a->G < 1) return GDN_ERR_SHAPE;
  if (a->N > 64) return GDN_ERR_UNSUPPORTED;
  if (a->D % a->G || a->B > (1 << 30) || a->T > (1 << 29) || a->D > (1 << 24)) return GDN_ERR_SHAPE;
  if ((double)a->B * (double)a->T * (double)a->D > (double)(1ll << 46)) return GDN_ERR_SHAPE;  // products stay in 64 bits
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
  const int es = elem_size(a->dtype);
  auto quad = [&](const void* q, int64_t sb, int64_t st, int64_t sg) { return (uintptr_t)q % (4 * es) == 0 && sb % 4 == 0 && st % 4 == 0 && sg % 4 == 0; };
  p.quads = a->N % 4 == 0 && quad(a->Bm, a->sB_b, a->sB_t, a->sB_g) && quad(a->Cm, a->sC_b, a->sC_t, a->sC_g);
  p.ckpt_quads = a->N % 4 == 0 && aligned16(a->ckpt);
  p.dblocks = scan_dblocks(a->D, a->G, a->N);
  const int64_t warp_channels = a->N <= 8 ? 32 : a->N <= 16 ? 16 : 8;  // of the kernels for aligned rows
  const SegPlan sp = scan_segments(a->B > 0 ? a->B : 1, a->T, (a->D / a->G + warp_channels - 1) / warp_channels * a->G);
  p.nseg = sp.nseg;
  p.seg_len = sp.seg_len;
  return p;
}

template <typename T, bool REV>
void launch_carry_plain(const ScanP& p, int nl, cudaStream_t s) {
  for_grid_rows(p, sizeof(T), [&](const ScanP& q, unsigned rows) {
    const dim3 g(p.dblocks * p.G, p.nseg, rows);
    if (nl == 2) scan_carry_kernel<T, 2, REV><<<g, SCAN_THREADS, 0, s>>>(q);
    if (nl == 4) scan_carry_kernel<T, 4, REV><<<g, SCAN_THREADS, 0, s>>>(q);
    if (nl == 8) scan_carry_kernel<T, 8, REV><<<g, SCAN_THREADS, 0, s>>>(q);
    if (nl == 16) scan_carry_kernel<T, 16, REV><<<g, SCAN_THREADS, 0, s>>>(q);
  });
}

template <typename T, int NL, int SL, bool REV>
int launch_carry_tiled(ScanP p, cudaStream_t s) {
  using K = CarryTiled<T, NL, SL>;
  static std::atomic<unsigned long long> opted{0};
  auto k = scan_carry_tiled_kernel<T, NL, SL, REV>;
  if (!opt_in_smem(opted, {{(const void*)k, K::SMEM}})) return GDN_ERR_LAUNCH;
  p.dblocks = (p.D / p.G + K::CH - 1) / K::CH;
  for_grid_rows(p, sizeof(T), [&](const ScanP& q, unsigned rows) { k<<<dim3(p.dblocks * p.G, p.nseg, rows), 32, K::SMEM, s>>>(q); });
  return launched();
}
template <typename T, bool REV>
int launch_carry(const ScanP& p, cudaStream_t s) {
  if (p.tiled)
    return p.N <= 8    ? launch_carry_tiled<T, 2, 4, REV>(p, s)
           : p.N <= 16 ? launch_carry_tiled<T, 4, 4, REV>(p, s)
           : p.N <= 32 ? launch_carry_tiled<T, 8, 4, REV>(p, s)
                       : launch_carry_tiled<T, 8, 8, REV>(p, s);
  launch_carry_plain<T, REV>(p, scan_lanes(p.N), s);
  return launched();
}

int scan_launch_carry(const ScanP& p, int dtype, bool reverse, cudaStream_t s) {
  const int64_t g = ((int64_t)p.B * p.D * p.N + 255) / 256;
  if (g > 0x7fffffff) return GDN_ERR_SHAPE;
  int st;
  if (reverse)
    st = dtype == GDN_DTYPE_F32 ? launch_carry<float, true>(p, s) : launch_carry<__nv_bfloat16, true>(p, s);
  else
    st = dtype == GDN_DTYPE_F32 ? launch_carry<float, false>(p, s) : launch_carry<__nv_bfloat16, false>(p, s);
  if (st != GDN_OK) return st;
  if (reverse)
    scan_combine_kernel<true><<<(unsigned)g, 256, 0, s>>>(p);
  else
    scan_combine_kernel<false><<<(unsigned)g, 256, 0, s>>>(p);
  return launched();
}

template <typename T, int NL, int SL>
int launch_tiled(ScanP p, cudaStream_t s) {
  using K = Tiled<T, NL, SL>;
  static std::atomic<unsigned long long> opted{0};
  auto k = scan_fwd_tiled_kernel<T, NL, SL>;
  if (!opt_in_smem(opted, {{(const void*)k, K::SMEM}})) return GDN_ERR_LAUNCH;
  p.dblocks = (p.D / p.G + K::CH - 1) / K::CH;
  for_grid_rows(p, sizeof(T), [&](const ScanP& q, unsigned rows) { k<<<dim3(p.dblocks * p.G, p.nseg, rows), 32, K::SMEM, s>>>(q); });
  return launched();
}
template <typename T>
int launch_tiled(const ScanP& p, cudaStream_t s) {
  return p.N <= 8 ? launch_tiled<T, 2, 4>(p, s) : p.N <= 16 ? launch_tiled<T, 4, 4>(p, s) : p.N <= 32 ? launch_tiled<T, 8, 4>(p, s) : launch_tiled<T, 8, 8>(p, s);
}

template <typename T>
int launch_plain(const ScanP& p, cudaStream_t s) {
  const int nl = scan_lanes(p.N);
  for_grid_rows(p, sizeof(T), [&](const ScanP& q, unsigned rows) {
    const dim3 g(p.dblocks * p.G, p.nseg, rows);
    if (nl == 2) scan_fwd_kernel<T, 2><<<g, SCAN_THREADS, 0, s>>>(q);
    if (nl == 4) scan_fwd_kernel<T, 4><<<g, SCAN_THREADS, 0, s>>>(q);
    if (nl == 8) scan_fwd_kernel<T, 8><<<g, SCAN_THREADS, 0, s>>>(q);
    if (nl == 16) scan_fwd_kernel<T, 16><<<g, SCAN_THREADS, 0, s>>>(q);
  });
  return launched();
}

template <typename T, bool VEC>
int launch_step(const ScanP& p, cudaStream_t s) {
  int nl = 1;
  while (nl * STEP_SL < p.N) nl *= 2;
  for_grid_rows(p, sizeof(T), [&](const ScanP& q, unsigned rows) {
    const dim3 g((unsigned)(((int64_t)p.D * nl + STEP_THREADS - 1) / STEP_THREADS), rows);
    if (nl == 1) scan_step_kernel<T, 1, VEC><<<g, STEP_THREADS, 0, s>>>(q);
    if (nl == 2) scan_step_kernel<T, 2, VEC><<<g, STEP_THREADS, 0, s>>>(q);
    if (nl == 4) scan_step_kernel<T, 4, VEC><<<g, STEP_THREADS, 0, s>>>(q);
    if (nl == 8) scan_step_kernel<T, 8, VEC><<<g, STEP_THREADS, 0, s>>>(q);
  });
  return launched();
}
template <typename T>
int launch_step(const ScanP& p, cudaStream_t s) {
  const bool vec = p.N % 4 == 0 && aligned16(p.h_out) && aligned16(p.A);
  return vec ? launch_step<T, true>(p, s) : launch_step<T, false>(p, s);
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
  *bytes = scan_align_plan(p, elem_size(a->dtype), false).total + (p.nseg > 1 ? (size_t)p.B * p.nseg * p.D * (p.N + 1) * sizeof(float) : 0);
  return GDN_OK;
}

int gdn_scan_fwd(const gdn_scan_args* a, void* stream) {
  size_t need = 0;
  int st = gdn_scan_workspace_bytes(a, &need);
  if (st != GDN_OK) return st;
  if (a->B == 0) return GDN_OK;
  if (a->T > 0 && !a->y) return GDN_ERR_NULL;
  if (need && (!a->workspace || a->workspace_bytes < need)) return GDN_ERR_WORKSPACE;
  if (need && !aligned16(a->workspace)) return GDN_ERR_ALIGN;
  if (!device_ok()) return GDN_ERR_DEVICE;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  ScanP p = scan_params(a);
  if (p.T == 0) {  // nothing to scan: the state passes through
    if (!p.h_out || p.h_out == p.h0) return GDN_OK;
    const size_t n = (size_t)p.B * p.D * p.N * sizeof(float);
    const cudaError_t e = p.h0 ? cudaMemcpyAsync(p.h_out, p.h0, n, cudaMemcpyDeviceToDevice, s) : cudaMemsetAsync(p.h_out, 0, n, s);
    return e == cudaSuccess ? GDN_OK : GDN_ERR_LAUNCH;
  }
  const int es = elem_size(a->dtype);
  const AlignPlan al = scan_align_plan(p, es, false);
  char* ws = static_cast<char*>(a->workspace);
  if (al.tiled) {
    st = scan_align(p, al, a->dtype, ws, s);
    if (st != GDN_OK) return st;
  }
  if (p.nseg > 1) {
    p.carry = reinterpret_cast<float*>(ws + al.total);
    p.ssum = p.carry + (int64_t)p.B * p.nseg * p.D * p.N;
    st = scan_launch_carry(p, a->dtype, false, s);
    if (st != GDN_OK) return st;
  }
  if (!al.tiled) return a->dtype == GDN_DTYPE_F32 ? launch_plain<float>(p, s) : launch_plain<__nv_bfloat16>(p, s);
  p.pairs_out = (p.D / p.G) % 2 == 0 && (uintptr_t)p.y % (2 * es) == 0 && p.sy_b % 2 == 0 && p.sy_t % 2 == 0;
  return a->dtype == GDN_DTYPE_F32 ? launch_tiled<float>(p, s) : launch_tiled<__nv_bfloat16>(p, s);
}

int gdn_scan_step(const gdn_scan_args* a, void* stream) {
  int st = scan_check(a, true);
  if (st != GDN_OK) return st;
  if (a->B == 0) return GDN_OK;
  if (!device_ok()) return GDN_ERR_DEVICE;
  const ScanP p = scan_params(a);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return a->dtype == GDN_DTYPE_F32 ? launch_step<float>(p, s) : launch_step<__nv_bfloat16>(p, s);
}

}  // extern "C"
