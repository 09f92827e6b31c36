// causal_conv1d_grad.cu -- the channel-last depthwise causal conv continued from a
// carried state (single tokens, short runs), and the conv's gradients.
//
//   u[t] = bias + sum_k w[k] x[t - W + 1 + k],  out = act(u)
//   du = dy act'(u);  dx[t] = sum_k w[k] du[t + W - 1 - k];  dw[k] = sum_t du[t] x[t - W + 1 + k];  db = sum_t du
//
// The reference's conv (kernels/causal_conv1d/kernel.py:170-230) is forward only, from
// zeros.
#include "host_util.h"
#include "rowops.cuh"

namespace thm {
namespace convg {

constexpr int kMaxW = 8;

// --------------------------------------------------------------------------- step
struct StepArgs {
  const void* x;      // [B, S, D], strides xb, xt
  const void* state;  // [B, W - 1, D]: the inputs before x
  const float *w, *b;
  void *out, *state_out;
  long long xb, xt;
  int B, S, D, act;
};

// One thread per VEC channels of a sequence: the window of W - 1 inputs lives in
// registers. state_out may be state: a thread reads its channels before it writes them.
template <typename T, int VEC, int W>
__global__ void __launch_bounds__(128) conv_step(const StepArgs p) {
  const long long idx = (long long)blockIdx.x * 128 + threadIdx.x;
  const int nvec = p.D / VEC;
  if (idx >= (long long)p.B * nvec) return;
  const long long bt = idx / nvec;
  const int c = (int)(idx - bt * nvec) * VEC;
  const T* x = static_cast<const T*>(p.x) + bt * p.xb + c;
  const T* st = static_cast<const T*>(p.state) + bt * (W - 1) * p.D + c;
  T* so = static_cast<T*>(p.state_out) + bt * (W - 1) * p.D + c;
  T* out = static_cast<T*>(p.out) + bt * p.S * p.D + c;
  float win[W][VEC], w[W][VEC], b[VEC];
#pragma unroll
  for (int k = 0; k + 1 < W; ++k) load_vec<T, VEC>(st + (long long)k * p.D, win[k + 1]);
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    b[e] = p.b[c + e];
#pragma unroll
    for (int k = 0; k < W; ++k) w[k][e] = p.w[(long long)(c + e) * W + k];
  }
  for (int t = 0; t < p.S; ++t) {
#pragma unroll
    for (int k = 0; k + 1 < W; ++k)
#pragma unroll
      for (int e = 0; e < VEC; ++e) win[k][e] = win[k + 1][e];
    load_vec<T, VEC>(x + t * p.xt, win[W - 1]);
    float u[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      u[e] = b[e];
#pragma unroll
      for (int k = 0; k < W; ++k) u[e] = fmaf(w[k][e], win[k][e], u[e]);
      if (p.act) u[e] = silu_of<T>(u[e]);
    }
    store_vec<T, VEC>(out + (long long)t * p.D, u);
  }
#pragma unroll
  for (int k = 0; k + 1 < W; ++k) store_vec<T, VEC>(so + (long long)k * p.D, win[k + 1]);
}

// --------------------------------------------------------------------------- backward
struct BwdArgs {
  const void *x, *dy;
  const float *w, *b;
  void* dx;
  float* part;  // [blocks, W + 1, D]
  long long xb, xt, gb, gt;
  int S, D, act, rows;  // rows: of a warp's strip
};

constexpr int kWarps = 8;

// A block has 32 * VEC channels and kWarps strips of rows of one sequence, a strip per
// warp. A thread walks its strip and W - 1 rows past its end: du of row t needs x of
// rows t - W + 1 .. t, and dx of row t du of rows t .. t + W - 1, so windows of both stay
// in registers and every row is read once but for the halo. Rows past the strip count
// for dx only, not for dw and db.
template <typename T, int VEC, int W>
__global__ void __launch_bounds__(32 * kWarps) conv_bwd(const BwdArgs p) {
  __shared__ float fold[kWarps][32 * VEC];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = (blockIdx.x * 32 + lane) * VEC;
  const bool on = c < p.D;
  const int t0 = (blockIdx.y * kWarps + warp) * p.rows;
  const int t1 = min(t0 + p.rows, p.S);
  const T* x = static_cast<const T*>(p.x) + (long long)blockIdx.z * p.xb + c;
  const T* dy = static_cast<const T*>(p.dy) + (long long)blockIdx.z * p.gb + c;
  T* dx = static_cast<T*>(p.dx) + (long long)blockIdx.z * p.S * p.D + c;
  float w[W][VEC], dw[W][VEC], b[VEC], db[VEC], xw[W][VEC], du[W][VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    b[e] = on ? p.b[c + e] : 0.f;
    db[e] = 0.f;
#pragma unroll
    for (int k = 0; k < W; ++k) {
      w[k][e] = on ? p.w[(long long)(c + e) * W + k] : 0.f;
      dw[k][e] = du[k][e] = xw[k][e] = 0.f;
    }
  }
  if (on && t0 < t1) {
#pragma unroll
    for (int k = 1; k < W; ++k)  // rows t0 - W + k, in xw[k]
      if (t0 - W + k >= 0) load_vec<T, VEC>(x + (long long)(t0 - W + k) * p.xt, xw[k]);
    for (int t = t0; t < t1 + W - 1; ++t) {
#pragma unroll
      for (int k = 0; k + 1 < W; ++k)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          xw[k][e] = xw[k + 1][e];
          du[k][e] = du[k + 1][e];
        }
      if (t < p.S) {
        load_vec<T, VEC>(x + t * p.xt, xw[W - 1]);
        load_vec<T, VEC>(dy + t * p.gt, du[W - 1]);
        if (p.act) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            float u = b[e], f, df;
#pragma unroll
            for (int k = 0; k < W; ++k) u = fmaf(w[k][e], xw[k][e], u);
            silu_grad<T>(u, f, df);
            du[W - 1][e] *= df;
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) du[W - 1][e] = 0.f;
      }
      if (t < t1) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          db[e] += du[W - 1][e];
#pragma unroll
          for (int k = 0; k < W; ++k) dw[k][e] = fmaf(du[W - 1][e], xw[k][e], dw[k][e]);
        }
      }
      if (t - (W - 1) >= t0) {  // dx of row t - W + 1: du of rows t - W + 1 .. t are du[0 .. W - 1]
        float g[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          g[e] = 0.f;
#pragma unroll
          for (int k = 0; k < W; ++k) g[e] = fmaf(w[k][e], du[W - 1 - k][e], g[e]);
        }
        store_vec<T, VEC>(dx + (long long)(t - W + 1) * p.D, g);
      }
    }
  }
  // The strips' sums, added in the order of the rows.
  float* part = p.part + ((long long)blockIdx.z * gridDim.y + blockIdx.y) * (W + 1) * p.D;
#pragma unroll
  for (int k = 0; k <= W; ++k) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < VEC; ++e) fold[warp][lane * VEC + e] = k < W ? dw[k < W ? k : 0][e] : db[e];
    __syncthreads();
    for (int j = threadIdx.x; j < 32 * VEC; j += 32 * kWarps) {
      const int col = blockIdx.x * 32 * VEC + j;
      if (col < p.D) {
        float acc = 0.f;
#pragma unroll
        for (int s = 0; s < kWarps; ++s) acc += fold[s][j];
        part[(long long)k * p.D + col] = acc;
      }
    }
  }
}

struct StoreGrads {
  float *dw, *db;
  int D, W;
  __device__ void operator()(int c, float v) const {
    const int k = c / D, d = c - k * D;
    if (k < W)
      dw[(long long)d * W + k] = v;
    else
      db[d] = v;
  }
};

// Rows of a warp's strip.
int strip_rows(int B, int S, int D) {
  (void)B;
  (void)D;
  return S >= 1024 ? 64 : 16;
}

template <typename F>
bool with_width(int W, F f) {
  switch (W) {
    case 1: f(std::integral_constant<int, 1>()); return true;
    case 2: f(std::integral_constant<int, 2>()); return true;
    case 3: f(std::integral_constant<int, 3>()); return true;
    case 4: f(std::integral_constant<int, 4>()); return true;
    case 5: f(std::integral_constant<int, 5>()); return true;
    case 6: f(std::integral_constant<int, 6>()); return true;
    case 7: f(std::integral_constant<int, 7>()); return true;
    case 8: f(std::integral_constant<int, 8>()); return true;
  }
  return false;
}

// Channels a thread may take as one access, given what addresses and strides are multiples
// of: 4, or 1.
int vector_of(uintptr_t bits, int elem) { return (bits & (4 * elem - 1)) == 0 ? 4 : 1; }

int check_sizes(int B, int S, int D, int W, int act, int dtype) {
  if (B < 0 || S < 0 || D < 0 || W <= 0) return THM_ERR_INVALID;
  if (act != THM_ACT_NONE && act != THM_ACT_SILU) return THM_ERR_INVALID;
  if (dtype != THM_F32 && dtype != THM_BF16) return THM_ERR_INVALID;
  if (W > kMaxW) return THM_ERR_UNSUPPORTED;
  return THM_OK;
}

template <typename T>
void launch_step(const StepArgs& p, int W, int vec, cudaStream_t st) {
  const long long n = (long long)p.B * (p.D / vec);
  const unsigned blocks = (unsigned)((n + 127) / 128);
  with_width(W, [&](auto w) {
    constexpr int kW = decltype(w)::value;
    if (vec == 4)
      conv_step<T, 4, kW><<<blocks, 128, 0, st>>>(p);
    else
      conv_step<T, 1, kW><<<blocks, 128, 0, st>>>(p);
  });
}

template <typename T>
void launch_bwd(const BwdArgs& p, dim3 grid, int W, int vec, cudaStream_t st) {
  with_width(W, [&](auto w) {
    constexpr int kW = decltype(w)::value;
    if (vec == 4)
      conv_bwd<T, 4, kW><<<grid, 32 * kWarps, 0, st>>>(p);
    else
      conv_bwd<T, 1, kW><<<grid, 32 * kWarps, 0, st>>>(p);
  });
}

}  // namespace convg
}  // namespace thm

extern "C" int thm_causal_conv1d_step(const void* x, const void* state, const float* weight, const float* bias,
                                      void* out, void* state_out, long long x_bs, long long x_ts, int B, int S,
                                      int D, int W, int dtype, int activation, thm_stream_t stream) {
  using namespace thm;
  const int bad = convg::check_sizes(B, S, D, W, activation, dtype);
  if (bad != THM_OK) return bad;
  if (B == 0 || D == 0) return THM_OK;
  if (!weight || !bias || (S > 0 && (!x || !out)) || (W > 1 && (!state || !state_out))) return THM_ERR_INVALID;
  const int elem = dtype == THM_BF16 ? 2 : 4;
  const uintptr_t bits = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(state) |
                         reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(state_out) |
                         (uintptr_t)(D * elem) | (uintptr_t)(x_bs * elem) | (uintptr_t)(x_ts * elem);
  const int vec = convg::vector_of(bits, elem);
  if (((long long)B * (D / vec) + 127) / 128 > 0x7fffffffLL) return THM_ERR_UNSUPPORTED;
  const convg::StepArgs p{x, state, weight, bias, out, state_out, x_bs, x_ts, B, S, D, activation == THM_ACT_SILU};
  if (dtype == THM_BF16)
    convg::launch_step<__nv_bfloat16>(p, W, vec, reinterpret_cast<cudaStream_t>(stream));
  else
    convg::launch_step<float>(p, W, vec, reinterpret_cast<cudaStream_t>(stream));
  return check_launch();
}

// Rows of the workspace [rows, W + 1, D] that thm_causal_conv1d_bwd uses.
extern "C" int thm_causal_conv1d_bwd_parts(int B, int S, int D) {
  using namespace thm;
  if (B <= 0 || S <= 0 || D <= 0) return 0;
  const int per = convg::kWarps * convg::strip_rows(B, S, D);
  const long long n = (long long)B * ((S + per - 1) / per);
  return n > 0x7fffffffLL ? -1 : (int)n;
}

extern "C" int thm_causal_conv1d_bwd(const void* x, const float* weight, const float* bias, const void* dy, void* dx,
                                     float* dweight, float* dbias, float* workspace, long long x_bs, long long x_ts,
                                     long long dy_bs, long long dy_ts, int B, int S, int D, int W, int dtype,
                                     int activation, thm_stream_t stream) {
  using namespace thm;
  const int bad = convg::check_sizes(B, S, D, W, activation, dtype);
  if (bad != THM_OK) return bad;
  if (D == 0) return THM_OK;
  if (!weight || !bias || !dweight || !dbias) return THM_ERR_INVALID;
  const int parts = thm_causal_conv1d_bwd_parts(B, S, D);
  if (parts < 0 || B > 65535) return THM_ERR_UNSUPPORTED;
  if (parts > 0 && (!x || !dy || !dx || !workspace)) return THM_ERR_INVALID;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (parts > 0) {
    const int elem = dtype == THM_BF16 ? 2 : 4;
    const uintptr_t bits = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(dy) |
                           reinterpret_cast<uintptr_t>(dx) | (uintptr_t)(D * elem) | (uintptr_t)(x_bs * elem) |
                           (uintptr_t)(x_ts * elem) | (uintptr_t)(dy_bs * elem) | (uintptr_t)(dy_ts * elem);
    const int vec = convg::vector_of(bits, elem);
    const int rows = convg::strip_rows(B, S, D);
    const int blocks_y = parts / B;
    if (blocks_y > 65535) return THM_ERR_UNSUPPORTED;
    const dim3 grid((D + 32 * vec - 1) / (32 * vec), blocks_y, B);
    const convg::BwdArgs p{x,     dy,    weight, bias, dx, workspace, x_bs, x_ts, dy_bs, dy_ts, S, D,
                           activation == THM_ACT_SILU, rows};
    if (dtype == THM_BF16)
      convg::launch_bwd<__nv_bfloat16>(p, grid, W, vec, st);
    else
      convg::launch_bwd<float>(p, grid, W, vec, st);
    const int e = check_launch();
    if (e != THM_OK) return e;
  }
  sum_parts(workspace, parts, (W + 1) * D, convg::StoreGrads{dweight, dbias, D, W}, st);
  return check_launch();
}
