// Depthwise causal convolution (width 2 to 4) with bias and SiLU, channels last: forward, one-token
// step and backward.
//
//   p_t = b + sum_{w<W} k_w x_{t-W+1+w},  y_t = silu(p_t)
//   dp_t = dy_t silu'(p_t),  dx_t = sum_w k_w dp_{t+W-1-w},  dk_w = sum_{b,t} dp_t x_{t-W+1+w},  db = sum dp_t
//
// HBM-bound: x is read and y written once (backward: x, dy read, dx written).  A thread owns one 16-byte
// vector of channels (or one channel where rows are not aligned) and a run of consecutive tokens, and keeps the
// last W - 1 inputs in registers, so only the run's first W - 1 rows are read twice (from L2).
#include "ssm_common.cuh"

namespace {

using namespace gdn;
using namespace gdn::ssm;

constexpr int RUN = 16;      // tokens per thread
constexpr int THREADS = 128;
constexpr int MAXW = 4;

struct ConvP {
  const void *x, *w, *bias, *state_in, *dy, *dstate_out;
  void *state_out, *y, *dx, *dstate_in;
  float* part;  // backward: (parts, C, W + 1) sums of dk and db
  const int32_t* lengths;
  int64_t sx_b, sx_t, sy_b, sy_t, sdy_b, sdy_t;
  int B, T, C, runs, act, w_dtype;
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

template <typename T, int VEC, int W>
__global__ void __launch_bounds__(THREADS) conv_fwd_kernel(ConvP p) {
  const int cvecs = p.C / VEC;
  const int64_t id = (int64_t)blockIdx.x * THREADS + threadIdx.x;
  if (id >= (int64_t)p.B * p.runs * cvecs) return;
  const int c = (int)(id % cvecs) * VEC;
  const int run = (int)((id / cvecs) % p.runs), b = (int)(id / ((int64_t)cvecs * p.runs));
  const int len = row_tokens(p.lengths, b, p.T);
  const int t0 = run * RUN, t1 = min(t0 + RUN, p.T);
  float k[W][VEC], bias[VEC], x[W][VEC];
  load_weights<VEC, W>(p, c, k, bias);
  T* y = static_cast<T*>(p.y) + b * p.sy_b + c;
  if (t0 < len) {
#pragma unroll
    for (int w = 0; w < W - 1; ++w) load_token<T, VEC, W>(p, b, t0 - (W - 1) + w, c, x[w]);
  }
#pragma unroll 8
  for (int t = t0; t < t1; ++t) {
    float o[VEC];
    if (t < len) {
      load_vec<VEC>(static_cast<const T*>(p.x) + b * p.sx_b + t * p.sx_t + c, x[W - 1]);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        float a = bias[i];
#pragma unroll
        for (int w = 0; w < W; ++w) a = fmaf(k[w][i], x[w][i], a);
        o[i] = p.act ? silu(a) : a;
#pragma unroll
        for (int w = 0; w < W - 1; ++w) x[w][i] = x[w + 1][i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) o[i] = 0.f;
    }
    store_vec<VEC>(y + t * p.sy_t, o);
  }
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

// Backward.  A thread walks its run once more than W - 1 tokens past its end: dp_t is formed as soon as x_t is
// there, and dx_{t-W+1} once the W gradients dp_{t-W+1..t} that reach it are.  dk and db take the run's own tokens
// only.  Their sums go to `part`, one row per thread, and are added in order by conv_sum_kernel.
template <typename T, int VEC, int W>
__global__ void __launch_bounds__(THREADS) conv_bwd_kernel(ConvP p) {
  const int cvecs = p.C / VEC;
  const int64_t id = (int64_t)blockIdx.x * THREADS + threadIdx.x;
  if (id >= (int64_t)p.B * p.runs * cvecs) return;
  const int c = (int)(id % cvecs) * VEC;
  const int run = (int)((id / cvecs) % p.runs), b = (int)(id / ((int64_t)cvecs * p.runs));
  const int len = row_tokens(p.lengths, b, p.T);
  const int t0 = run * RUN, t1 = min(t0 + RUN, p.T);
  float k[W][VEC], bias[VEC], x[W][VEC], dp[W][VEC], dk[W][VEC], db[VEC];
  load_weights<VEC, W>(p, c, k, bias);
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    db[i] = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) dk[w][i] = dp[w][i] = 0.f;
  }
  // dp[w] = dp_{t-W+1+w} once token t is in.  The thread of the first run also owns the W - 1 inputs of the state,
  // which tokens 0 .. W - 2 reach: its window starts with dp_{<0} = 0.  Other runs' first dx waits for t0 + W - 1.
  if (t0 < len) {
#pragma unroll
    for (int w = 0; w < W - 1; ++w) load_token<T, VEC, W>(p, b, t0 - (W - 1) + w, c, x[w]);
  }
  const T* dyp = static_cast<const T*>(p.dy) + b * p.sdy_b + c;
  T* dxp = static_cast<T*>(p.dx) + (int64_t)b * p.T * p.C + c;
#pragma unroll 4
  for (int t = t0; t < t1 + W - 1; ++t) {
    float d[VEC];
    if (t < len) {
      load_vec<VEC>(static_cast<const T*>(p.x) + b * p.sx_b + t * p.sx_t + c, x[W - 1]);
      load_vec<VEC>(dyp + t * p.sdy_t, d);
      const bool mine = t < t1;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        if (p.act) {
          float a = bias[i];
#pragma unroll
          for (int w = 0; w < W; ++w) a = fmaf(k[w][i], x[w][i], a);
          d[i] *= dsilu(a);
        }
        if (mine) {
          db[i] += d[i];
#pragma unroll
          for (int w = 0; w < W; ++w) dk[w][i] = fmaf(d[i], x[w][i], dk[w][i]);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) d[i] = 0.f;
    }
    const int u = t - (W - 1);  // the input that is complete now
    float o[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
#pragma unroll
      for (int w = 0; w < W - 1; ++w) {
        dp[w][i] = dp[w + 1][i];
        x[w][i] = x[w + 1][i];
      }
      dp[W - 1][i] = d[i];
      float a = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) a = fmaf(k[W - 1 - w][i], dp[w][i], a);
      o[i] = a;
    }
    if (p.dstate_out && u >= len - (W - 1) && u < len && (u >= t0 || t0 == 0)) {  // state_out holds input u too
      const T* ds = static_cast<const T*>(p.dstate_out) + ((int64_t)b * p.C + c) * (W - 1) + (u - len + W - 1);
#pragma unroll
      for (int i = 0; i < VEC; ++i) o[i] += to_f32(ds[i * (W - 1)]);
    }
    if (u >= t0) {
      store_vec<VEC>(dxp + (int64_t)u * p.C, o);
    } else if (t0 == 0 && p.dstate_in) {  // u in -(W - 1) .. -1
      T* ds = static_cast<T*>(p.dstate_in) + ((int64_t)b * p.C + c) * (W - 1) + (u + W - 1);
#pragma unroll
      for (int i = 0; i < VEC; ++i) store_as(ds + i * (W - 1), o[i]);
    }
  }
  // Sums over the block's threads of one channel vector would save partial rows; one row per (b, run) is simple.
  float* part = p.part + ((int64_t)(b * p.runs + run) * p.C + c) * (W + 1);
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
#pragma unroll
    for (int w = 0; w < W; ++w) part[i * (W + 1) + w] = dk[w][i];
    part[i * (W + 1) + W] = db[i];
  }
}

// One warp per (channel, tap): its partial sums, lane-strided then across the lanes.
__global__ void conv_sum_kernel(const float* part, int64_t rows, int C, int W, void* dw, void* db, int w_dtype) {
  const int i = blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32, lane = threadIdx.x % 32;
  const int n = C * (W + 1);
  if (i >= n) return;
  float a = 0.f;
  for (int64_t r = lane; r < rows; r += 32) a += part[r * n + i];
#pragma unroll
  for (int o = 16; o; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
  if (lane) return;
  const int c = i / (W + 1), w = i % (W + 1);
  if (w < W)
    store_param(dw, (int64_t)c * W + w, w_dtype, a);
  else if (db)
    store_param(db, c, w_dtype, a);
}

int check(const gdn_conv_args* a, bool step) {
  if (!a) return GDN_ERR_NULL;
  if (a->B < 0 || a->T < 0 || a->C < 1 || a->B > (1 << 30) || a->T > (1 << 30) || a->C > (1 << 24)) return GDN_ERR_SHAPE;
  if (a->width < 2 || a->width > MAXW) return GDN_ERR_UNSUPPORTED;
  if (a->act != GDN_ACT_NONE && a->act != GDN_ACT_SILU) return GDN_ERR_UNSUPPORTED;
  if (!elem_size(a->dtype) || !elem_size(a->w_dtype)) return GDN_ERR_DTYPE;
  if (!a->weight) return GDN_ERR_NULL;
  if (a->sx_b < 0 || a->sx_t < 0 || a->sy_b < 0 || a->sy_t < 0) return GDN_ERR_SHAPE;
  if (step && a->B > 0 && (!a->x || !a->y || !a->state_in)) return GDN_ERR_NULL;
  return GDN_OK;
}

ConvP params(const gdn_conv_args* a) {
  ConvP p = {};
  p.x = a->x; p.w = a->weight; p.bias = a->bias; p.state_in = a->state_in; p.state_out = a->state_out; p.y = a->y;
  p.lengths = a->lengths;
  p.sx_b = a->sx_b; p.sx_t = a->sx_t; p.sy_b = a->sy_b; p.sy_t = a->sy_t;
  p.B = (int)a->B; p.T = (int)a->T; p.C = (int)a->C; p.act = a->act; p.w_dtype = a->w_dtype;
  p.runs = (p.T + RUN - 1) / RUN;
  return p;
}

// 16-byte vectors of channels where every row starts on one.
bool vectors(const ConvP& p, int es, bool bwd) {
  const int v = 16 / es;
  auto ok = [&](const void* q, int64_t sb, int64_t st) { return aligned16(q) && sb % v == 0 && st % v == 0; };
  if (p.C % v || !ok(p.x, p.sx_b, p.sx_t)) return false;
  return bwd ? ok(p.dy, p.sdy_b, p.sdy_t) && aligned16(p.dx) : ok(p.y, p.sy_b, p.sy_t);
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
  const ConvP p = params(a);
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
  return vectors(p, 2, false) ? launch_fwd<__nv_bfloat16, 8>(p, a->width, s) : launch_fwd<__nv_bfloat16, 1>(p, a->width, s);
}

int gdn_conv_step(const gdn_conv_args* a, void* stream) {
  int st = check(a, true);
  if (st != GDN_OK) return st;
  if (a->B == 0) return GDN_OK;
  if (!device_ok()) return GDN_ERR_DEVICE;
  ConvP p = params(a);
  p.state_out = const_cast<void*>(a->state_in);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return a->dtype == GDN_DTYPE_F32 ? launch_step<float>(p, a->width, s) : launch_step<__nv_bfloat16>(p, a->width, s);
}

int gdn_conv_bwd_workspace_bytes(const gdn_conv_bwd_args* a, size_t* bytes) {
  if (!a || !bytes) return GDN_ERR_NULL;
  int st = check(&a->fwd, false);
  if (st != GDN_OK) return st;
  const ConvP p = params(&a->fwd);
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
  ConvP p = params(f);
  p.dy = a->dy; p.dx = a->dx; p.dstate_out = a->dstate_out; p.dstate_in = a->dstate_in;
  p.sdy_b = a->sdy_b; p.sdy_t = a->sdy_t;
  p.part = static_cast<float*>(a->workspace);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (f->dtype == GDN_DTYPE_F32)
    st = vectors(p, 4, true) ? launch_bwd<float, 4>(p, f->width, s) : launch_bwd<float, 1>(p, f->width, s);
  else
    st = vectors(p, 2, true) ? launch_bwd<__nv_bfloat16, 8>(p, f->width, s) : launch_bwd<__nv_bfloat16, 1>(p, f->width, s);
  if (st != GDN_OK) return st;
  const int n = p.C * (f->width + 1);
  conv_sum_kernel<<<(n + 7) / 8, 256, 0, s>>>(p.part, (int64_t)p.B * p.runs, p.C, f->width, a->dweight, a->dbias, f->w_dtype);
  return launched();
}

}  // extern "C"
