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

constexpr int kWarps = 8, kBlockRows = 4;

__device__ __forceinline__ float2 f2(float v) { return make_float2(v, v); }

// VEC channels as fp32 pairs (one channel: an empty second half).
template <typename T, int VEC>
__device__ __forceinline__ void widen(const Pack<T, VEC>& q, float2 (&f)[(VEC + 1) / 2]) {
  if constexpr (VEC == 1) {
    f[0] = make_float2(to_f32<T>(q.v[0]), 0.f);
  } else {
#pragma unroll
    for (int e = 0; e < VEC / 2; ++e) {
      if constexpr (sizeof(T) == 2) {
        const uint32_t w = reinterpret_cast<const uint32_t*>(&q)[e];
        f[e] = make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
      } else {
        f[e] = make_float2(q.v[2 * e], q.v[2 * e + 1]);
      }
    }
  }
}
template <typename T, int VEC>
__device__ __forceinline__ void store_pairs(T* p, const float2 (&f)[(VEC + 1) / 2]) {
  if constexpr (VEC == 1) {
    *p = from_f32<T>(f[0].x);
  } else {
    Pack<T, VEC> q;
#pragma unroll
    for (int e = 0; e < VEC / 2; ++e) {
      if constexpr (sizeof(T) == 2)
        reinterpret_cast<uint32_t*>(&q)[e] = pack_bf16x2(f[e].x, f[e].y);
      else
        reinterpret_cast<float2*>(&q)[e] = f[e];
    }
    *reinterpret_cast<Pack<T, VEC>*>(p) = q;
  }
}

// g silu'(u) = g s (1 + u (1 - s)), s = sigmoid(u).
template <typename T>
__device__ __forceinline__ float2 through_silu(float2 g, float2 u) {
  float2 s;
  if constexpr (sizeof(T) == 2) {
    const float2 e = __fmul2_rn(u, f2(-1.4426950408889634f));
    const float2 d = __fadd2_rn(make_float2(ex2_approx(e.x), ex2_approx(e.y)), f2(1.f));
    s = make_float2(rcp_approx(d.x), rcp_approx(d.y));
  } else {
    s = make_float2(sigmoid<T>(u.x), sigmoid<T>(u.y));
  }
  return __fmul2_rn(g, __fmul2_rn(s, __ffma2_rn(u, __ffma2_rn(s, f2(-1.f), f2(1.f)), f2(1.f))));
}

// A block has 32 * VEC channels and kWarps strips of rows of one sequence, a strip per
// warp. A lane walks its strip and W - 1 rows past its end, four rows at a time, the next four
// in flight: du of row t needs x of rows t - W + 1 .. t, and dx of row t du of rows t .. t + W - 1,
// so windows of both stay in registers and every row is read once but for the halo. Rows past
// the strip count for dx only, not for dw and db; rows past the sequence are zeros, whose du is 0.
template <typename T, int VEC, int W, bool ACT>
__global__ void __launch_bounds__(32 * kWarps, W <= 4 ? 2 : 1) conv_bwd(const BwdArgs p) {
  constexpr int NP = (VEC + 1) / 2, RB = kBlockRows;
  using Raw = Pack<T, VEC>;
  __shared__ float fold[kWarps][32 * VEC];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = (blockIdx.x * 32 + lane) * VEC;
  const bool on = c < p.D;
  const int t0 = (blockIdx.y * kWarps + warp) * p.rows;
  const int t1 = min(t0 + p.rows, p.S);
  const T* x = static_cast<const T*>(p.x) + (long long)blockIdx.z * p.xb + c;
  const T* dy = static_cast<const T*>(p.dy) + (long long)blockIdx.z * p.gb + c;
  T* dx = static_cast<T*>(p.dx) + (long long)blockIdx.z * p.S * p.D + c;
  float2 w[W][NP], dw[W][NP], b[NP], db[NP], xw[W - 1 + RB][NP], du[W - 1 + RB][NP];
#pragma unroll
  for (int e = 0; e < NP; ++e) {
    const bool two = VEC > 1;
    b[e] = on ? make_float2(p.b[c + 2 * e], two ? p.b[c + 2 * e + 1] : 0.f) : f2(0.f);
    db[e] = f2(0.f);
#pragma unroll
    for (int k = 0; k < W; ++k) {
      w[k][e] = on ? make_float2(p.w[(long long)(c + 2 * e) * W + k], two ? p.w[(long long)(c + 2 * e + 1) * W + k] : 0.f)
                   : f2(0.f);
      dw[k][e] = f2(0.f);
    }
  }
  if (on && t0 < t1) {
    const int end = min(t1 + W - 1, p.S);  // rows that there are and that count
#pragma unroll
    for (int k = 0; k + 1 < W; ++k) {  // the rows before the strip
      const int t = t0 - (W - 1) + k;
      Raw q{};
      if (t >= 0) q = *reinterpret_cast<const Raw*>(x + t * p.xt);
      widen<T, VEC>(q, xw[k]);
#pragma unroll
      for (int e = 0; e < NP; ++e) du[k][e] = f2(0.f);
    }
    Raw xr[RB], gr[RB];
    auto load = [&](int t) {
#pragma unroll
      for (int k = 0; k < RB; ++k) {
        xr[k] = gr[k] = Raw{};
        if (t + k < end) {
          xr[k] = *reinterpret_cast<const Raw*>(x + (t + k) * p.xt);
          gr[k] = *reinterpret_cast<const Raw*>(dy + (t + k) * p.gt);
        }
      }
    };
    load(t0);
    for (int t = t0; t < t1 + W - 1; t += RB) {
#pragma unroll
      for (int k = 0; k < RB; ++k) {
        widen<T, VEC>(xr[k], xw[W - 1 + k]);
        widen<T, VEC>(gr[k], du[W - 1 + k]);
      }
      load(t + RB);
      if constexpr (ACT) {
#pragma unroll
        for (int k = 0; k < RB; ++k)
#pragma unroll
          for (int e = 0; e < NP; ++e) {
            float2 u = b[e];
#pragma unroll
            for (int j = 0; j < W; ++j) u = __ffma2_rn(w[j][e], xw[k + j][e], u);
            du[W - 1 + k][e] = through_silu<T>(du[W - 1 + k][e], u);
          }
      }
      if (t < t1) {  // strips are whole blocks of rows, but for the sequence's end
#pragma unroll
        for (int k = 0; k < RB; ++k)
#pragma unroll
          for (int e = 0; e < NP; ++e) {
            db[e] = __fadd2_rn(db[e], du[W - 1 + k][e]);
#pragma unroll
            for (int j = 0; j < W; ++j) dw[j][e] = __ffma2_rn(du[W - 1 + k][e], xw[k + j][e], dw[j][e]);
          }
      }
#pragma unroll
      for (int k = 0; k < RB; ++k) {  // dx of row t + k - (W - 1)
        const int row = t + k - (W - 1);
        if (row < t0 || row >= t1) continue;
        float2 g[NP];
#pragma unroll
        for (int e = 0; e < NP; ++e) {
          g[e] = __fmul2_rn(w[0][e], du[k + W - 1][e]);
#pragma unroll
          for (int j = 1; j < W; ++j) g[e] = __ffma2_rn(w[j][e], du[k + W - 1 - j][e], g[e]);
        }
        store_pairs<T, VEC>(dx + (long long)row * p.D, g);
      }
#pragma unroll
      for (int k = 0; k + 1 < W; ++k)
#pragma unroll
        for (int e = 0; e < NP; ++e) {
          xw[k][e] = xw[k + RB][e];
          du[k][e] = du[k + RB][e];
        }
    }
  }
  // The strips' sums, added in the order of the rows.
  float* part = p.part + ((long long)blockIdx.z * gridDim.y + blockIdx.y) * (W + 1) * p.D;
#pragma unroll
  for (int k = 0; k <= W; ++k) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < NP; ++e) {
      const float2 v = k < W ? dw[k < W ? k : 0][e] : db[e];
      fold[warp][lane * VEC + 2 * e] = v.x;
      if constexpr (VEC > 1) fold[warp][lane * VEC + 2 * e + 1] = v.y;
    }
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

// Channels a lane of the backward kernel takes where vectors fit: its windows and sums of more
// than 4 taps do not fit the registers for 4.
constexpr int bwd_vec(int W) { return W <= 4 ? 4 : 2; }

template <typename T>
void launch_bwd(const BwdArgs& p, dim3 grid, int W, int vec, cudaStream_t st) {
  with_width(W, [&](auto w) {
    constexpr int kW = decltype(w)::value, kVec = bwd_vec(kW);
    auto k = vec > 1 ? (p.act ? conv_bwd<T, kVec, kW, true> : conv_bwd<T, kVec, kW, false>)
                     : (p.act ? conv_bwd<T, 1, kW, true> : conv_bwd<T, 1, kW, false>);
    k<<<grid, 32 * kWarps, 0, st>>>(p);
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
    const int vec = convg::vector_of(bits, elem) > 1 ? convg::bwd_vec(W) : 1;
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
