// Depthwise causal convolution (width 2 to 4) with bias and SiLU, channels last: forward, one-token
// step and backward.
//
//   p_t = b + sum_{w<W} k_w x_{t-W+1+w},  y_t = silu(p_t)
//   dp_t = dy_t silu'(p_t),  dx_t = sum_w k_w dp_{t+W-1-w},  dk_w = sum_{b,t} dp_t x_{t-W+1+w},  db = sum dp_t
//
// HBM-bound: x is read and y written once (backward: x, dy read, dx written).  A thread owns a vector
// of channels (one channel where rows are not aligned) and a run of consecutive tokens, and keeps the last W - 1 inputs
// in registers, so only the run's first W - 1 rows are read twice (from L2).
#include "ssm_common.cuh"

namespace {

using namespace gdn;
using namespace gdn::ssm;

constexpr int THREADS = 128;
constexpr int MAXW = 4;

struct ConvP {
  const void *x, *w, *bias, *state_in, *dy, *dstate_out;
  void *state_out, *y, *dx, *dstate_in;
  float* part;  // backward: (parts, C, W + 1) sums of dk and db
  const int32_t* lengths;
  int64_t sx_b, sx_t, sy_b, sy_t, sdy_b, sdy_t;
  int B, T, C, run, runs, act, w_dtype;  // runs of `run` tokens
};

// x_t of VEC channels from c for any t >= -(W - 1): before the row's first token it comes from the state.
template <typename T, int VEC, int W>
__device__ __forceinline__ void load_token(const ConvP& p, int b, int t, int c, float (&v)[VEC]) {
  if (t >= 0) {
    load_vec<VEC>(static_cast<const T*>(p.x) + b * p.sx_b + t * p.sx_t + c, v);
  } else if (p.state_in) {
    const T* s = static_cast<const T*>(p.state_in) + ((int64_t)b * p.C + c) * (W - 1) + (t + W - 1);
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = to_f32(s[i * (W - 1)]);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = 0.f;
  }
}

template <int VEC, int W>
__device__ __forceinline__ void load_weights(const ConvP& p, int c, float (&k)[W][VEC], float (&bias)[VEC]) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
#pragma unroll
    for (int w = 0; w < W; ++w) k[w][i] = load_param(p.w, (int64_t)(c + i) * W + w, p.w_dtype);
    bias[i] = p.bias ? load_param(p.bias, c + i, p.w_dtype) : 0.f;
  }
}

template <typename T, int VEC>
struct __align__(VEC * sizeof(T)) Vec {
  T v[VEC];
};

// Channels in pairs for the packed fp32 instructions; a single channel leaves the second half unused.
template <typename T, int VEC>
__device__ __forceinline__ void to_pairs(const Vec<T, VEC>& r, f32x2 (&o)[(VEC + 1) / 2]) {
  if constexpr (VEC == 1) {
    o[0] = pack2(to_f32(r.v[0]), 0.f);
  } else {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) o[i] = load_pair(&r.v[2 * i]);
  }
}
template <typename T, int VEC>
__device__ __forceinline__ Vec<T, VEC> from_pairs(const f32x2 (&o)[(VEC + 1) / 2]) {
  Vec<T, VEC> r;
#pragma unroll
  for (int i = 0; i < (VEC + 1) / 2; ++i) {
    const float2 e = unpack2(o[i]);
    store_as(&r.v[2 * i], e.x);
    if (2 * i + 1 < VEC) store_as(&r.v[2 * i + 1], e.y);
  }
  return r;
}
template <int VEC, int W>
__device__ __forceinline__ void load_weight_pairs(const ConvP& p, int c, f32x2 (&k)[W][(VEC + 1) / 2], f32x2 (&bias)[(VEC + 1) / 2]) {
  float kv[W][VEC], bv[VEC];
  load_weights<VEC, W>(p, c, kv, bv);
#pragma unroll
  for (int i = 0; i < (VEC + 1) / 2; ++i) {
    const int j = 2 * i + 1 < VEC ? 2 * i + 1 : 2 * i;
    bias[i] = pack2(bv[2 * i], bv[j]);
#pragma unroll
    for (int w = 0; w < W; ++w) k[w][i] = pack2(kv[w][2 * i], kv[w][j]);
  }
}

// A thread's own queue of its coming tokens, GROUPS groups of TOK tokens, filled by asynchronous copies: values on their
// way take no registers (queued in registers they cost more warps than they hide).  Only the thread itself reads its
// places, so no barrier is needed; a group is refilled one iteration after it was used.  Values of less than 4 bytes,
// which no such copy takes, are loaded a group at a time instead.
template <typename V, int STREAMS, int TOK, int GROUPS>
struct Queue {
  static constexpr bool ASYNC = sizeof(V) >= 4;
  static constexpr int BYTES = ASYNC ? GROUPS * TOK * STREAMS * THREADS * (int)sizeof(V) : 16;
  V* at;  // this thread's first place
  __device__ explicit Queue(char* smem) : at(reinterpret_cast<V*>(smem) + threadIdx.x) {}
  __device__ V* place(int g, int q, int stream) const { return at + ((g * TOK + q) * STREAMS + stream) * THREADS; }
  // Into place g: token q of a stream is at address src(q, stream).
  template <typename F>
  __device__ void fill(int g, F src) const {
#pragma unroll
    for (int q = 0; q < TOK; ++q)
#pragma unroll
      for (int s = 0; s < STREAMS; ++s)
        copy_bytes<(int)sizeof(V)>(static_cast<uint32_t>(__cvta_generic_to_shared(place(g, q, s))), src(q, s));
    copies_commit();
  }
};

// Four channels per thread keep 32 warps on an SM.  At 8 x 4096 x 2048 (bf16, width 4) 60.5 us; 67 us with batches of eight
// loads in registers and no queue.  A batch is a multiple of W - 1 tokens, so that the window turns by renaming registers:
// with four tokens of width 4 it is 64 us.  HBM's share is 41 us, the sigmoids' two operations per value on their pipe 30 us
// and the packed arithmetic 20 us; they overlap in part.
template <typename T, int VEC, int W>
__global__ void __launch_bounds__(THREADS, 8) conv_fwd_kernel(const ConvP p) {
  constexpr int HP = (VEC + 1) / 2, BATCH = W == 4 ? 3 : 4, GROUPS = 3;
  using V = Vec<T, VEC>;
  using Q = Queue<V, 1, BATCH, GROUPS>;
  __shared__ __align__(16) char smem[Q::BYTES];
  const int cvecs = p.C / VEC;
  const int64_t id = (int64_t)blockIdx.x * THREADS + threadIdx.x;
  if (id >= (int64_t)p.B * p.runs * cvecs) return;
  const int64_t br = id / cvecs;
  const int c = (int)(id - br * cvecs) * VEC;
  const int b = (int)(br / p.runs), run = (int)(br - (int64_t)b * p.runs);
  const int len = row_tokens(p.lengths, b, p.T);
  const int t0 = run * p.run, t1 = min(t0 + p.run, p.T), te = min(t1, len);
  const T* xp = static_cast<const T*>(p.x) + b * p.sx_b + c;
  T* yp = static_cast<T*>(p.y) + b * p.sy_b + c;
  f32x2 k[W][HP], bias[HP], x[W][HP];
  load_weight_pairs<VEC, W>(p, c, k, bias);
  if (t0 < te) {
#pragma unroll
    for (int w = 0; w < W - 1; ++w) {
      float v[VEC];
      load_token<T, VEC, W>(p, b, t0 - (W - 1) + w, c, v);
#pragma unroll
      for (int i = 0; i < HP; ++i) x[w][i] = pack2(v[2 * i], v[2 * i + 1 < VEC ? 2 * i + 1 : 2 * i]);
    }
  }
  const Q queue(smem);
  auto src = [&](int t) { return xp + (int64_t)min(t, te - 1) * p.sx_t; };  // past the run's end the last token again
  auto fill = [&](int g, int t) { queue.fill(g, [&](int q, int) { return src(t + q); }); };
  if (Q::ASYNC && t0 < te) {
#pragma unroll
    for (int g = 0; g < GROUPS - 1; ++g) fill(g, t0 + g * BATCH);
  }
  for (int t = t0, g = 0; t < te; t += BATCH, g = g + 1 == GROUPS ? 0 : g + 1) {
    V raw[BATCH];
    if (Q::ASYNC) {
      copies_wait<GROUPS - 2>();
#pragma unroll
      for (int q = 0; q < BATCH; ++q) raw[q] = *queue.place(g, q, 0);
      fill(g == 0 ? GROUPS - 1 : g - 1, t + (GROUPS - 1) * BATCH);
    } else {
#pragma unroll
      for (int q = 0; q < BATCH; ++q) raw[q] = *reinterpret_cast<const V*>(src(t + q));
    }
#pragma unroll
    for (int q = 0; q < BATCH; ++q) {
      f32x2 o[HP];
      to_pairs<T, VEC>(raw[q], x[W - 1]);
#pragma unroll
      for (int i = 0; i < HP; ++i) {
        f32x2 a = fma2(k[0][i], x[0][i], bias[i]);
#pragma unroll
        for (int w = 1; w < W; ++w) a = fma2(k[w][i], x[w][i], a);
        o[i] = p.act ? mul2(a, sigmoid2(a)) : a;
#pragma unroll
        for (int w = 0; w < W - 1; ++w) x[w][i] = x[w + 1][i];
      }
      if (t + q < te) *reinterpret_cast<V*>(yp + (int64_t)(t + q) * p.sy_t) = from_pairs<T, VEC>(o);
    }
  }
  f32x2 zero[HP];
#pragma unroll
  for (int i = 0; i < HP; ++i) zero[i] = both(0.f);
  for (int t = max(t0, te); t < t1; ++t) *reinterpret_cast<V*>(yp + (int64_t)t * p.sy_t) = from_pairs<T, VEC>(zero);
  if (p.state_out && run == 0) {  // the last W - 1 inputs of the row
    T* so = static_cast<T*>(p.state_out) + ((int64_t)b * p.C + c) * (W - 1);
#pragma unroll
    for (int w = 0; w < W - 1; ++w) {
      float v[VEC];
      load_token<T, VEC, W>(p, b, len - (W - 1) + w, c, v);
#pragma unroll
      for (int i = 0; i < VEC; ++i) store_as(so + i * (W - 1) + w, v[i]);
    }
  }
}

// An empty sequence: the state passes through.
template <typename T>
__global__ void conv_copy_state_kernel(const T* in, T* out, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i < n) store_as(out + i, in ? to_f32(in[i]) : 0.f);
}

// One token per row; the state moves up by one input in place.
template <typename T, int W>
__global__ void __launch_bounds__(THREADS) conv_step_kernel(ConvP p) {
  const int64_t id = (int64_t)blockIdx.x * THREADS + threadIdx.x;
  if (id >= (int64_t)p.B * p.C) return;
  const int c = (int)(id % p.C), b = (int)(id / p.C);
  float k[W][1], bias[1];
  load_weights<1, W>(p, c, k, bias);
  T* s = static_cast<T*>(p.state_out) + id * (W - 1);
  float x[W];
#pragma unroll
  for (int w = 0; w < W - 1; ++w) x[w] = to_f32(s[w]);
  x[W - 1] = to_f32(static_cast<const T*>(p.x)[b * p.sx_b + c]);
  float a = bias[0];
#pragma unroll
  for (int w = 0; w < W; ++w) a = fmaf(k[w][0], x[w], a);
#pragma unroll
  for (int w = 0; w < W - 1; ++w) store_as(s + w, x[w + 1]);
  store_as(static_cast<T*>(p.y) + b * p.sy_b + c, p.act ? silu(a) : a);
}

// Backward.  A thread walks its run and W - 1 tokens past it: dp_t is formed as soon as x_t is there, and dx_{t-W+1}
// once the W gradients dp_{t-W+1..t} that reach it are.  dk and db take the run's own tokens only; a thread's sums go to
// `part`, one row per (row, run), and conv_sum_kernel adds the rows in order.  At 8 x 2048 x 2048 (bf16, width 4) 69 us, and
// 4 us for the sums; without the queue the kernel took 10 us more.  HBM's share is 31 us.
template <typename T, int VEC, int W>
__global__ void __launch_bounds__(THREADS, 4) conv_bwd_kernel(const ConvP p) {
  constexpr int HP = (VEC + 1) / 2, BATCH = sizeof(Vec<T, VEC>) == 16 ? 2 : 4, GROUPS = 2;
  using V = Vec<T, VEC>;
  using Q = Queue<V, 2, BATCH, GROUPS>;
  __shared__ __align__(16) char smem[Q::BYTES];
  const int cvecs = p.C / VEC;
  const int64_t id = (int64_t)blockIdx.x * THREADS + threadIdx.x;
  if (id >= (int64_t)p.B * p.runs * cvecs) return;
  const int64_t br = id / cvecs;
  const int c = (int)(id - br * cvecs) * VEC;
  const int b = (int)(br / p.runs), run = (int)(br - (int64_t)b * p.runs);
  const int len = row_tokens(p.lengths, b, p.T);
  const int t0 = run * p.run, t1 = min(t0 + p.run, p.T);
  f32x2 k[W][HP], bias[HP], x[W][HP], dp[W][HP], dk[W][HP], db[HP];
  load_weight_pairs<VEC, W>(p, c, k, bias);
#pragma unroll
  for (int i = 0; i < HP; ++i) {
    db[i] = both(0.f);
#pragma unroll
    for (int w = 0; w < W; ++w) x[w][i] = dk[w][i] = dp[w][i] = both(0.f);
  }
  if (t0 < len) {
#pragma unroll
    for (int w = 0; w < W - 1; ++w) {
      float v[VEC];
      load_token<T, VEC, W>(p, b, t0 - (W - 1) + w, c, v);
#pragma unroll
      for (int i = 0; i < HP; ++i) x[w][i] = pack2(v[2 * i], v[2 * i + 1 < VEC ? 2 * i + 1 : 2 * i]);
    }
  }
  // dp[w] = dp_{t-W+1+w} once token t is in.  The first run also owns the W - 1 inputs of the state, which tokens
  // 0 .. W - 2 reach; its window starts with dp_{<0} = 0.  Other runs' first dx waits for token t0 + W - 1.
  const T* xp = static_cast<const T*>(p.x) + b * p.sx_b + c;
  const T* dyp = static_cast<const T*>(p.dy) + b * p.sdy_b + c;
  T* dxp = static_cast<T*>(p.dx) + (int64_t)b * p.T * p.C + c;
  const Q queue(smem);
  auto src = [&](int t, int stream) {  // places past the row's tokens read its last one; their values are dropped
    const int64_t u = max(min(t, len - 1), 0);
    return stream ? dyp + u * p.sdy_t : xp + u * p.sx_t;
  };
  auto fill = [&](int g, int t) { queue.fill(g, [&](int q, int s) { return src(t + q, s); }); };
  if (Q::ASYNC) {
#pragma unroll
    for (int g = 0; g < GROUPS - 1; ++g) fill(g, t0 + g * BATCH);
  }
  for (int tb = t0, g = 0; tb < t1 + W - 1; tb += BATCH, g = g + 1 == GROUPS ? 0 : g + 1) {
    V rx[BATCH], rd[BATCH];
    if (Q::ASYNC) {
      copies_wait<GROUPS - 2>();
#pragma unroll
      for (int q = 0; q < BATCH; ++q) {
        rx[q] = *queue.place(g, q, 0);
        rd[q] = *queue.place(g, q, 1);
      }
      fill(g == 0 ? GROUPS - 1 : g - 1, tb + (GROUPS - 1) * BATCH);
    } else {
#pragma unroll
      for (int q = 0; q < BATCH; ++q) {
        rx[q] = *reinterpret_cast<const V*>(src(tb + q, 0));
        rd[q] = *reinterpret_cast<const V*>(src(tb + q, 1));
      }
    }
#pragma unroll
    for (int q = 0; q < BATCH; ++q) {
      const int t = tb + q;
      const bool on = t < len, mine = t < t1 && on;
      f32x2 d[HP], o[HP];
      to_pairs<T, VEC>(rx[q], x[W - 1]);
      to_pairs<T, VEC>(rd[q], d);
#pragma unroll
      for (int i = 0; i < HP; ++i) {
        if (p.act) {
          f32x2 a = fma2(k[0][i], x[0][i], bias[i]);
#pragma unroll
          for (int w = 1; w < W; ++w) a = fma2(k[w][i], x[w][i], a);
          const f32x2 g = sigmoid2(a);
          d[i] = mul2(d[i], mul2(g, fma2(a, fma2(g, both(-1.f), both(1.f)), both(1.f))));
        }
        d[i] = on ? d[i] : both(0.f);
        const f32x2 m = mine ? d[i] : both(0.f);
        db[i] = add2(db[i], m);
#pragma unroll
        for (int w = 0; w < W; ++w) dk[w][i] = fma2(m, on ? x[w][i] : both(0.f), dk[w][i]);
#pragma unroll
        for (int w = 0; w < W - 1; ++w) {
          dp[w][i] = dp[w + 1][i];
          x[w][i] = x[w + 1][i];
        }
        dp[W - 1][i] = d[i];
        o[i] = mul2(k[W - 1][i], dp[0][i]);
#pragma unroll
        for (int w = 1; w < W; ++w) o[i] = fma2(k[W - 1 - w][i], dp[w][i], o[i]);
      }
      const int u = t - (W - 1);  // the input that is complete now
      if (u >= t1) continue;
      if (p.dstate_out && u >= len - (W - 1) && u < len && (u >= t0 || t0 == 0)) {  // state_out holds input u too
        const T* ds = static_cast<const T*>(p.dstate_out) + ((int64_t)b * p.C + c) * (W - 1) + (u - len + W - 1);
#pragma unroll
        for (int i = 0; i < HP; ++i)
          o[i] = add2(o[i], pack2(to_f32(ds[2 * i * (W - 1)]), 2 * i + 1 < VEC ? to_f32(ds[(2 * i + 1) * (W - 1)]) : 0.f));
      }
      if (u >= t0) {
        *reinterpret_cast<V*>(dxp + (int64_t)u * p.C) = from_pairs<T, VEC>(o);
      } else if (t0 == 0 && p.dstate_in) {  // u in -(W - 1) .. -1
        T* ds = static_cast<T*>(p.dstate_in) + ((int64_t)b * p.C + c) * (W - 1) + (u + W - 1);
        const V r = from_pairs<T, VEC>(o);
#pragma unroll
        for (int i = 0; i < VEC; ++i) ds[i * (W - 1)] = r.v[i];
      }
    }
  }
  // (W + 1) planes of C channels
  float* part = p.part + br * p.C * (W + 1) + c;
#pragma unroll
  for (int w = 0; w <= W; ++w)
#pragma unroll
    for (int i = 0; i < HP; ++i) {
      const float2 e = unpack2(w < W ? dk[w < W ? w : 0][i] : db[i]);
      part[(int64_t)w * p.C + 2 * i] = e.x;
      if (2 * i + 1 < VEC) part[(int64_t)w * p.C + 2 * i + 1] = e.y;
    }
}

// Column sums of the partial rows: 32 neighbouring columns and 8 groups of rows per block, added in order.
__global__ void __launch_bounds__(256) conv_sum_kernel(const float* part, int64_t rows, int C, int W, void* dw, void* db, int w_dtype) {
  __shared__ float s[8][32];
  const int lane = threadIdx.x % 32, g = threadIdx.x / 32;
  const int64_t n = (int64_t)C * (W + 1), i = (int64_t)blockIdx.x * 32 + lane;
  float a = 0.f;
  if (i < n) {
#pragma unroll 4
    for (int64_t r = g; r < rows; r += 8) a += part[r * n + i];
  }
  s[g][lane] = a;
  __syncthreads();
  if (g || i >= n) return;
#pragma unroll
  for (int k = 1; k < 8; ++k) a += s[k][lane];
  const int w = (int)(i / C), c = (int)(i % C);
  if (w < W)
    store_param(dw, (int64_t)c * W + w, w_dtype, a);
  else if (db)
    store_param(db, c, w_dtype, a);
}

int check(const gdn_conv_args* a, bool step) {
  if (!a) return GDN_ERR_NULL;
  if (a->B < 0 || a->T < 0 || a->C < 1 || a->B > (1 << 30) || a->T > (1 << 30) || a->C > (1 << 24)) return GDN_ERR_SHAPE;
  if ((double)a->B * (double)a->T * (double)a->C > (double)(1ll << 46)) return GDN_ERR_SHAPE;  // products stay in 64 bits
  if (a->width < 2 || a->width > MAXW) return GDN_ERR_UNSUPPORTED;
  if (a->act != GDN_ACT_NONE && a->act != GDN_ACT_SILU) return GDN_ERR_UNSUPPORTED;
  if (!elem_size(a->dtype) || !elem_size(a->w_dtype)) return GDN_ERR_DTYPE;
  if (!a->weight) return GDN_ERR_NULL;
  if (a->sx_b < 0 || a->sx_t < 0 || a->sy_b < 0 || a->sy_t < 0) return GDN_ERR_SHAPE;
  if (step && a->B > 0 && (!a->x || !a->y || !a->state_in)) return GDN_ERR_NULL;
  return GDN_OK;
}

// Tokens per thread in the forward, 16 to 64: as many as still leave about 768 threads of four channels per SM (a run's
// first W - 1 inputs are read twice).  Whole waves, as below, are level here (60.5 and 59.8 us).
int fwd_run(int64_t B, int64_t T, int64_t C) {
  const int64_t n = B * T * C / 4 / (148 * 768);
  return n >= 64 ? 64 : n >= 32 ? 32 : 16;
}

// In the backward, at least 16 and at most 128 in the fewest whole waves of the 512 threads an SM holds: a run also costs a
// row of sums (8 x 2048 x 2048: one wave of 114 tokens 74 us, 1.7 waves of 64 tokens 83 us, sums included).
int bwd_run(int64_t B, int64_t T, int64_t C) {
  const int64_t at_once = 148 * 512, row = (B * C + 3) / 4;  // threads of one run per row
  if (row < 1 || T < 1) return 16;
  const int64_t waves = ((T + 127) / 128 * row + at_once - 1) / at_once, runs = waves * at_once / row;
  const int64_t n = (T + runs - 1) / runs;
  return n < 16 ? 16 : (int)n;
}

ConvP params(const gdn_conv_args* a, bool bwd) {
  ConvP p = {};
  p.x = a->x; p.w = a->weight; p.bias = a->bias; p.state_in = a->state_in; p.state_out = a->state_out; p.y = a->y;
  p.lengths = a->lengths;
  p.sx_b = a->sx_b; p.sx_t = a->sx_t; p.sy_b = a->sy_b; p.sy_t = a->sy_t;
  p.B = (int)a->B; p.T = (int)a->T; p.C = (int)a->C; p.act = a->act; p.w_dtype = a->w_dtype;
  p.run = bwd ? bwd_run(a->B, a->T, a->C) : fwd_run(a->B, a->T, a->C);
  p.runs = (p.T + p.run - 1) / p.run;
  return p;
}

// Vectors of channels where every row starts on one.
bool vectors(const ConvP& p, int es, bool bwd) {
  const int v = 4;
  auto ok = [&](const void* q, int64_t sb, int64_t st) { return (uintptr_t)q % (v * es) == 0 && sb % v == 0 && st % v == 0; };
  if (p.C % v || !ok(p.x, p.sx_b, p.sx_t)) return false;
  return bwd ? ok(p.dy, p.sdy_b, p.sdy_t) && (uintptr_t)p.dx % (v * es) == 0 : ok(p.y, p.sy_b, p.sy_t);
}

int64_t blocks(int64_t n) { return (n + THREADS - 1) / THREADS; }

template <typename T, int VEC>
int launch_fwd(const ConvP& p, int width, cudaStream_t s) {
  const int64_t g = blocks((int64_t)p.B * p.runs * (p.C / VEC));
  if (g > 0x7fffffff) return GDN_ERR_SHAPE;
  if (width == 2) conv_fwd_kernel<T, VEC, 2><<<(unsigned)g, THREADS, 0, s>>>(p);
  if (width == 3) conv_fwd_kernel<T, VEC, 3><<<(unsigned)g, THREADS, 0, s>>>(p);
  if (width == 4) conv_fwd_kernel<T, VEC, 4><<<(unsigned)g, THREADS, 0, s>>>(p);
  return launched();
}

template <typename T, int VEC>
int launch_bwd(const ConvP& p, int width, cudaStream_t s) {
  const int64_t g = blocks((int64_t)p.B * p.runs * (p.C / VEC));
  if (g > 0x7fffffff) return GDN_ERR_SHAPE;
  if (width == 2) conv_bwd_kernel<T, VEC, 2><<<(unsigned)g, THREADS, 0, s>>>(p);
  if (width == 3) conv_bwd_kernel<T, VEC, 3><<<(unsigned)g, THREADS, 0, s>>>(p);
  if (width == 4) conv_bwd_kernel<T, VEC, 4><<<(unsigned)g, THREADS, 0, s>>>(p);
  return launched();
}

template <typename T>
int launch_step(const ConvP& p, int width, cudaStream_t s) {
  const int64_t g = blocks((int64_t)p.B * p.C);
  if (g > 0x7fffffff) return GDN_ERR_SHAPE;
  if (width == 2) conv_step_kernel<T, 2><<<(unsigned)g, THREADS, 0, s>>>(p);
  if (width == 3) conv_step_kernel<T, 3><<<(unsigned)g, THREADS, 0, s>>>(p);
  if (width == 4) conv_step_kernel<T, 4><<<(unsigned)g, THREADS, 0, s>>>(p);
  return launched();
}

}  // namespace

extern "C" {

int gdn_conv_fwd(const gdn_conv_args* a, void* stream) {
  int st = check(a, false);
  if (st != GDN_OK) return st;
  if (a->B == 0) return GDN_OK;
  if (a->T > 0 && (!a->x || !a->y)) return GDN_ERR_NULL;
  if (!device_ok()) return GDN_ERR_DEVICE;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const ConvP p = params(a, false);
  if (p.T == 0) {
    if (!a->state_out) return GDN_OK;
    const int64_t n = (int64_t)p.B * p.C * (a->width - 1), g = (n + 255) / 256;
    if (g > 0x7fffffff) return GDN_ERR_SHAPE;
    if (a->dtype == GDN_DTYPE_F32)
      conv_copy_state_kernel<float><<<(unsigned)g, 256, 0, s>>>((const float*)a->state_in, (float*)a->state_out, n);
    else
      conv_copy_state_kernel<__nv_bfloat16>
          <<<(unsigned)g, 256, 0, s>>>((const __nv_bfloat16*)a->state_in, (__nv_bfloat16*)a->state_out, n);
    return launched();
  }
  if (a->dtype == GDN_DTYPE_F32)
    return vectors(p, 4, false) ? launch_fwd<float, 4>(p, a->width, s) : launch_fwd<float, 1>(p, a->width, s);
  return vectors(p, 2, false) ? launch_fwd<__nv_bfloat16, 4>(p, a->width, s) : launch_fwd<__nv_bfloat16, 1>(p, a->width, s);
}

int gdn_conv_step(const gdn_conv_args* a, void* stream) {
  int st = check(a, true);
  if (st != GDN_OK) return st;
  if (a->B == 0) return GDN_OK;
  if (!device_ok()) return GDN_ERR_DEVICE;
  ConvP p = params(a, false);
  p.state_out = const_cast<void*>(a->state_in);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return a->dtype == GDN_DTYPE_F32 ? launch_step<float>(p, a->width, s) : launch_step<__nv_bfloat16>(p, a->width, s);
}

int gdn_conv_bwd_workspace_bytes(const gdn_conv_bwd_args* a, size_t* bytes) {
  if (!a || !bytes) return GDN_ERR_NULL;
  int st = check(&a->fwd, false);
  if (st != GDN_OK) return st;
  const ConvP p = params(&a->fwd, true);
  *bytes = (size_t)p.B * p.runs * p.C * (a->fwd.width + 1) * sizeof(float);
  return GDN_OK;
}

int gdn_conv_bwd(const gdn_conv_bwd_args* a, void* stream) {
  size_t need = 0;
  int st = gdn_conv_bwd_workspace_bytes(a, &need);
  if (st != GDN_OK) return st;
  const gdn_conv_args* f = &a->fwd;
  if (f->B == 0 || f->T == 0) return GDN_ERR_SHAPE;  // nothing flowed; the caller zeroes the gradients
  if (!f->x || !a->dy || !a->dx || !a->dweight || (need && !a->workspace)) return GDN_ERR_NULL;
  if (a->sdy_b < 0 || a->sdy_t < 0) return GDN_ERR_SHAPE;
  if (a->workspace_bytes < need) return GDN_ERR_WORKSPACE;
  if (!device_ok()) return GDN_ERR_DEVICE;
  ConvP p = params(f, true);
  p.dy = a->dy; p.dx = a->dx; p.dstate_out = a->dstate_out; p.dstate_in = a->dstate_in;
  p.sdy_b = a->sdy_b; p.sdy_t = a->sdy_t;
  p.part = static_cast<float*>(a->workspace);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (f->dtype == GDN_DTYPE_F32)
    st = vectors(p, 4, true) ? launch_bwd<float, 4>(p, f->width, s) : launch_bwd<float, 1>(p, f->width, s);
  else
    st = vectors(p, 2, true) ? launch_bwd<__nv_bfloat16, 4>(p, f->width, s) : launch_bwd<__nv_bfloat16, 1>(p, f->width, s);
  if (st != GDN_OK) return st;
  const int64_t n = (int64_t)p.C * (f->width + 1);
  conv_sum_kernel<<<(unsigned)((n + 31) / 32), 256, 0, s>>>(p.part, (int64_t)p.B * p.runs, p.C, f->width, a->dweight, a->dbias, f->w_dtype);
  return launched();
}

}  // extern "C"
