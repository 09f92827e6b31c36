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

THM_DEFINE_STATUS(g_status_conv_grad)

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
// registers. state_out may be state: a thread reads its channels before it writes them. Launch
// latency bounds it: 64 sequences of one token, D 2048, W 4, bf16 take 2.9 us.
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
  int S, D, rows;  // rows: of a warp's strip, a multiple of kBlockRows
};
struct BwdMaps {
  CUtensorMap x, dy;
};

constexpr int kWarps = 8, kBlockRows = 4, kCols = 64;

__device__ __forceinline__ float2 f2(float v) { return make_float2(v, v); }

// Two neighbouring channels in shared memory.
template <typename T>
__device__ __forceinline__ float2 get_pair(const uint8_t* p) {
  if constexpr (sizeof(T) == 2) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(p);
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  } else {
    return *reinterpret_cast<const float2*>(p);
  }
}
// ... and in global memory, as one access (PAIRED) or as two.
template <typename T, bool PAIRED>
__device__ __forceinline__ float2 load_pair(const T* p, bool two) {
  if constexpr (PAIRED) return get_pair<T>(reinterpret_cast<const uint8_t*>(p));
  return make_float2(to_f32<T>(p[0]), two ? to_f32<T>(p[1]) : 0.f);
}
template <typename T, bool PAIRED>
__device__ __forceinline__ void store_pair(T* p, float2 f, bool two) {
  if constexpr (PAIRED) {
    if constexpr (sizeof(T) == 2)
      *reinterpret_cast<uint32_t*>(p) = pack_bf16x2(f.x, f.y);
    else
      *reinterpret_cast<float2*>(p) = f;
  } else {
    p[0] = from_f32<T>(f.x);
    if (two) p[1] = from_f32<T>(f.y);
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

// A block has 64 channels and 8 strips of rows of one sequence, a strip per warp and two channels
// a lane. A warp walks its strip and W - 1 rows past its end: du of row t needs x of rows
// t - W + 1 .. t, and dx of row t du of rows t .. t + W - 1, so windows of both stay in registers, as
// rings that the unrolled loop indexes, and every row is read once but for the halo. Rows past
// the strip count for dx only, not for dw and db; rows past the sequence come as zeros, whose du
// is 0.
//
// The rows come by TMA, a ring's worth (fp32) or two of both tensors at a time, into stages of the
// warp's own: no block barrier, no address arithmetic, and the bytes in flight
// take no registers (loads of 4 rows ahead into registers left HBM at a third of its rate).
// Where addresses or strides are no multiples of 16 bytes (TMA false), the lanes fill their own
// slots. B8 S8192 D2048 W4 with SiLU, bf16: 151 us and 5 for the second launch, 5.2 TB/s (0.79 of a
// copy), issuing on 61 % of the cycles with the FMA pipe 53 % busy.
template <typename T, int W>
struct Bwd {
  static constexpr int kNB = (W - 1 + 2 * kBlockRows - 1) / kBlockRows;  // blocks of rows in a ring
  static constexpr int kRing = kNB * kBlockRows;
  static constexpr int kStep = sizeof(T) == 2 ? 2 * kRing : kRing;  // rows of a stage
  static constexpr int kTile = kStep * kCols * (int)sizeof(T);
  static constexpr int kStages = 2;
  static constexpr int kBytes = kWarps * kStages * 2 * kTile;
};

template <typename T, int W, bool ACT, bool TMA>
__global__ void __launch_bounds__(32 * kWarps, W <= 5 ? 3 : 2)
    conv_bwd(const __grid_constant__ BwdArgs p, const __grid_constant__ BwdMaps tm) {
  using C = Bwd<T, W>;
  constexpr int RB = kBlockRows, RING = C::kRing, STEP = C::kStep, NS = C::kStages;
  extern __shared__ __align__(128) uint8_t stages[];
  __shared__ float2 fold[kWarps][32];
  __shared__ __align__(8) uint64_t full[kWarps][NS];
  const int lane = threadIdx.x & 31, warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  const int c = blockIdx.x * kCols + 2 * lane;
  const bool on = c < p.D, two = c + 1 < p.D;
  const int t0 = (blockIdx.y * kWarps + warp) * p.rows;
  const int t1 = min(t0 + p.rows, p.S);
  uint8_t* ring = stages + warp * NS * 2 * C::kTile;
  if (lane == 0) {
    for (int k = 0; k < NS; ++k) mbar_init(&full[warp][k], 1);
    fence_mbar_init();
  }
  __syncwarp();
  const int steps = t0 < t1 ? (t1 - t0 + W - 1 + STEP - 1) / STEP : 0;
  bool ok = true;
  int asked = 0, failed = 0;
  auto ask = [&](int j) {
    if (j >= steps || !ok) return;
    asked = j + 1;
    uint64_t* bar = &full[warp][j % NS];
    uint8_t* slot = ring + (j % NS) * 2 * C::kTile;
    mbar_arrive_expect_tx(bar, 2 * C::kTile);
    tma_load_3d(slot, &tm.x, bar, blockIdx.x * kCols, t0 + j * STEP, blockIdx.z);
    tma_load_3d(slot + C::kTile, &tm.dy, bar, blockIdx.x * kCols, t0 + j * STEP, blockIdx.z);
  };
  if (TMA && lane == 0)
    for (int j = 0; j < NS; ++j) ask(j);
  float2 w[W], dw[W], b = f2(0.f), db = f2(0.f);
  if (on) b = make_float2(p.b[c], two ? p.b[c + 1] : 0.f);
#pragma unroll
  for (int k = 0; k < W; ++k) {
    w[k] = on ? make_float2(p.w[(long long)c * W + k], two ? p.w[(long long)(c + 1) * W + k] : 0.f) : f2(0.f);
    dw[k] = f2(0.f);
  }
  const T* x = static_cast<const T*>(p.x) + (long long)blockIdx.z * p.xb + c;
  const T* dy = static_cast<const T*>(p.dy) + (long long)blockIdx.z * p.gb + c;
  T* dx = static_cast<T*>(p.dx) + ((long long)blockIdx.z * p.S + t0 - (W - 1)) * p.D + c;
  float2 xw[RING], du[RING];  // row t0 + k at k % RING
#pragma unroll
  for (int k = 0; k < RING; ++k) xw[k] = du[k] = f2(0.f);
#pragma unroll
  for (int k = 1; k < W; ++k)  // the rows before the strip
    if (on && t0 < t1 && t0 - k >= 0) xw[RING - k] = load_pair<T, TMA>(x + (t0 - k) * p.xt, two);
  for (int j = 0; j < steps; ++j) {
    const int tb = t0 + j * STEP;
    uint8_t* slot = ring + (j % NS) * 2 * C::kTile + 2 * lane * (int)sizeof(T);
    if constexpr (TMA) {
      if (ok) {
        ok = mbar_wait(&full[warp][j % NS], (j / NS) & 1, &g_status_conv_grad);
        failed = j;
      }
    } else {
// Four rows at a time, loads without conditions so that all are in flight at once: rows past the
// sequence repeat its last and are then taken as zeros, a second channel that is not there repeats
// the first.
#pragma unroll
      for (int k0 = 0; k0 < STEP; k0 += RB) {
        T v[2][RB][2];
        const int next = two ? 1 : 0;
        if (on) {
#pragma unroll
          for (int k = 0; k < RB; ++k) {
            const long long t = min(tb + k0 + k, p.S - 1);
            v[0][k][0] = x[t * p.xt];
            v[0][k][1] = x[t * p.xt + next];
            v[1][k][0] = dy[t * p.gt];
            v[1][k][1] = dy[t * p.gt + next];
          }
#pragma unroll
          for (int k = 0; k < RB; ++k)
#pragma unroll
            for (int n = 0; n < 2; ++n) {
              const float2 f = make_float2(to_f32<T>(v[n][k][0]), to_f32<T>(v[n][k][1]));
              store_pair<T, true>(reinterpret_cast<T*>(slot + n * C::kTile + (k0 + k) * kCols * sizeof(T)),
                                  tb + k0 + k < p.S ? f : f2(0.f), true);
            }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < STEP / RB; ++i) {
      const int t = tb + i * RB, r0 = i * RB + RING;  // ring index of row t
      if (t >= t1 + W - 1) break;
#pragma unroll
      for (int k = 0; k < RB; ++k) {
        xw[(r0 + k) % RING] = get_pair<T>(slot + (i * RB + k) * kCols * sizeof(T));
        du[(r0 + k) % RING] = get_pair<T>(slot + C::kTile + (i * RB + k) * kCols * sizeof(T));
      }
      if constexpr (ACT) {
#pragma unroll
        for (int k = 0; k < RB; ++k) {
          float2 u = b;
#pragma unroll
          for (int l = 0; l < W; ++l) u = __ffma2_rn(w[l], xw[(r0 + k - (W - 1) + l) % RING], u);
          du[(r0 + k) % RING] = through_silu<T>(du[(r0 + k) % RING], u);
        }
      }
      if (t < t1) {  // strips are whole blocks of rows, but for the sequence's end
#pragma unroll
        for (int k = 0; k < RB; ++k) {
          const float2 g = du[(r0 + k) % RING];
          db = __fadd2_rn(db, g);
#pragma unroll
          for (int l = 0; l < W; ++l) dw[l] = __ffma2_rn(g, xw[(r0 + k - (W - 1) + l) % RING], dw[l]);
        }
      }
      float2 g[RB];  // dx of rows t + k - (W - 1)
#pragma unroll
      for (int k = 0; k < RB; ++k) {
        g[k] = __fmul2_rn(w[0], du[(r0 + k) % RING]);
#pragma unroll
        for (int l = 1; l < W; ++l) g[k] = __ffma2_rn(w[l], du[(r0 + k - l) % RING], g[k]);
      }
      const int row = t - (W - 1);
      if (on) {
        if (row >= t0 && row + RB <= t1) {
#pragma unroll
          for (int k = 0; k < RB; ++k) store_pair<T, TMA>(dx + (long long)(i * RB + k) * p.D, g[k], two);
        } else {
#pragma unroll
          for (int k = 0; k < RB; ++k)
            if (row + k >= t0 && row + k < t1) store_pair<T, TMA>(dx + (long long)(i * RB + k) * p.D, g[k], two);
        }
      }
    }
    dx += (long long)STEP * p.D;
    __syncwarp();  // the stage has been read
    if (TMA && lane == 0) ask(j + NS);
  }
  if (TMA && lane == 0)  // after a wait that ran out: once more for what is still on its way here
    for (int j = failed; !ok && j < asked; ++j) mbar_wait(&full[warp][j % NS], (j / NS) & 1, &g_status_conv_grad);
  let_dependents_launch();
  // The strips' sums, added in the order of the rows.
  float* part = p.part + ((long long)blockIdx.z * gridDim.y + blockIdx.y) * (W + 1) * p.D;
#pragma unroll
  for (int k = 0; k <= W; ++k) {
    __syncthreads();
    fold[warp][lane] = k < W ? dw[k < W ? k : 0] : db;
    __syncthreads();
    if (warp == 0 && on) {
      float2 acc = fold[0][lane];
#pragma unroll
      for (int s = 1; s < kWarps; ++s) acc = __fadd2_rn(acc, fold[s][lane]);
      part[(long long)k * p.D + c] = acc.x;
      if (two) part[(long long)k * p.D + c + 1] = acc.y;
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

// Rows of a warp's strip: blocks of a launch take about as long, so what counts is how many rounds
// of resident blocks (three an SM) there are and what one takes: the strip's rows, and about 12
// more for the halo, the first loads and the sums.
int strip_rows(int B, int S, int D) {
  const long long cols = (long long)B * ((D + kCols - 1) / kCols), slots = 3ll * sm_count();
  int best = 16;
  long long least = -1;
  for (int rows = 16; rows <= 256; rows += kBlockRows) {
    const long long blocks = cols * ((S + (long long)kWarps * rows - 1) / (kWarps * rows));
    const long long cost = (blocks + slots - 1) / slots * (rows + 12);
    if (least < 0 || cost < least) {
      least = cost;
      best = rows;
    }
  }
  return best;
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
  if (W > kMaxW || S > 1 << 30) return THM_ERR_UNSUPPORTED;
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

// x or dy [B, S, D] in boxes of `rows` x 64. A dimension of one entry may have any stride.
int encode(CUtensorMap* m, int dtype, const void* base, long long bs, long long ts, int B, int S, int D, int rows) {
  const int elem = dtype == THM_BF16 ? 2 : 4;
  const uint64_t dims[3] = {(uint64_t)D, (uint64_t)S, (uint64_t)B};
  const uint64_t ts_b = S > 1 ? (uint64_t)ts * elem : (uint64_t)(D * elem + 15) / 16 * 16;
  const uint64_t strides[2] = {ts_b, B > 1 ? (uint64_t)bs * elem : ts_b * (uint64_t)S};
  const uint32_t box[3] = {(uint32_t)kCols, (uint32_t)rows, 1};
  if (strides[0] == 0 || strides[1] == 0 || strides[0] >= (1ull << 40) || strides[1] >= (1ull << 40))
    return THM_ERR_UNSUPPORTED;
  return encode_tiled(m, dtype == THM_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3,
                      base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE);
}

template <typename T>
int launch_bwd(const BwdArgs& p, dim3 grid, int B, int W, bool act, int dtype, cudaStream_t st) {
  const int elem = sizeof(T);
  const uintptr_t bits = reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.dy) |
                         reinterpret_cast<uintptr_t>(p.dx) | (uintptr_t)(p.D * elem) |
                         (uintptr_t)((B > 1 ? p.xb | p.gb : 0) * elem) | (uintptr_t)((p.xt | p.gt) * elem);
  int status = THM_OK;
  with_width(W, [&](auto w) {
    constexpr int kW = decltype(w)::value;
    using C = Bwd<T, kW>;
    BwdMaps tm{};
    const bool tma = (bits & 15) == 0 && encode(&tm.x, dtype, p.x, p.xb, p.xt, B, p.S, p.D, C::kStep) == THM_OK &&
                     encode(&tm.dy, dtype, p.dy, p.gb, p.gt, B, p.S, p.D, C::kStep) == THM_OK;
    auto k = tma ? (act ? conv_bwd<T, kW, true, true> : conv_bwd<T, kW, false, true>)
                 : (act ? conv_bwd<T, kW, true, false> : conv_bwd<T, kW, false, false>);
    if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kBytes) != cudaSuccess) {
      cudaGetLastError();
      status = THM_ERR_CUDA;
      return;
    }
    k<<<grid, 32 * kWarps, C::kBytes, st>>>(p, tm);
  });
  return status != THM_OK ? status : check_launch();
}

}  // namespace convg
}  // namespace thm

THM_STATUS_READER(thm_internal_status_conv_grad, g_status_conv_grad)

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
    const int blocks_y = parts / B;
    if (blocks_y > 65535) return THM_ERR_UNSUPPORTED;
    const dim3 grid((D + convg::kCols - 1) / convg::kCols, blocks_y, B);
    const convg::BwdArgs p{x, dy, weight, bias, dx, workspace, x_bs, x_ts, dy_bs, dy_ts, S, D, convg::strip_rows(B, S, D)};
    const bool act = activation == THM_ACT_SILU;
    const int e = dtype == THM_BF16 ? convg::launch_bwd<__nv_bfloat16>(p, grid, B, W, act, dtype, st)
                                    : convg::launch_bwd<float>(p, grid, B, W, act, dtype, st);
    if (e != THM_OK) return e;
  }
  return sum_parts(workspace, parts, (W + 1) * D, convg::StoreGrads{dweight, dbias, D, W}, st);
}
