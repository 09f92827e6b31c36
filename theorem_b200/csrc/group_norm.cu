// group_norm.cu -- norm over groups of consecutive channels of each token, channel-last,
// with SiLU or a gate, and its gradients.
//
//   xh = (x - mu) rs  (or x rs),  rs = 1 / sqrt(mean((x - mu)^2) + eps)   per token and group
//   u  = xh w + b;    y = act(u), or u act(z) with a gate z
//
//   du = dy act'(u)  (or dy act(z), dz = dy u act'(z));   dxh = du w
//   dx = rs (dxh - mean(dxh) - xh mean(dxh xh))           (no mean(dxh) without centring)
//   dw = sum du xh, db = sum du over all tokens
//
// A group belongs to a team of threads that hold it in registers, so x is read once: the
// variance is formed from the centred values, not from a difference of sums. Teams are
// TL consecutive lanes (a power of two up to a warp), or the whole block for groups that
// a warp's registers do not hold. A thread keeps its channels from row to row: w and b are
// read once, and dw, db are summed in registers over the block's rows; each block leaves
// one row of partial sums and a second launch adds those up in a fixed order.
#include "host_util.h"
#include "rowops.cuh"

namespace thm {
namespace gnorm {

struct Args {
  const void *x, *z, *dy;
  const float *w, *b;
  void *y, *dx, *dz;
  float* part;             // backward: [blocks in y, 2, C] sums of dw and db, or null
  long long xs, zs, gs;    // row strides of x, z, dy
  long long R;
  int C, G, groups;
  int tl;                  // lanes of a team; 0: the whole block
  int gpc, rpi;            // groups and rows that a block works on at a time
  int center, act;
  float eps;
};

// Sum over the team, the same value in each of its threads.
__device__ __forceinline__ float team_sum(float v, int tl, float* sh) {
  if (tl != 0) {
    for (int o = tl >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  }
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();  // the previous sum has been read
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
  for (int k = 0; k < (int)(blockDim.x >> 5); ++k) s += sh[k];
  return s;
}

// Where a thread stands: its team's group and row offset in the block, and whether the
// team has work. Channel of vector j: c0 + j * step.
struct Place {
  int group, sub, lane, width;
  bool on;
};
__device__ __forceinline__ Place place(const Args& p) {
  Place q;
  const int team = p.tl != 0 ? threadIdx.x / p.tl : 0;
  q.width = p.tl != 0 ? p.tl : blockDim.x;
  q.lane = p.tl != 0 ? threadIdx.x % p.tl : threadIdx.x;
  q.sub = team / p.gpc;
  q.group = blockIdx.x * p.gpc + team % p.gpc;
  q.on = q.sub < p.rpi && q.group < p.groups;
  return q;
}

constexpr int max_threads(int vec) { return vec == 1 ? 1024 : vec == 2 ? 512 : 256; }

// Mean (if centred) and scale of the group in v; masked vectors hold zeros. v is centred.
template <int VEC, int NV>
__device__ __forceinline__ float normalise(float (&v)[NV][VEC], const bool (&have)[NV], const Args& p, float* sh) {
  const float inv = 1.f / (float)p.G;
  if (p.center) {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < VEC; ++e) s += v[j][e];
    const float mu = team_sum(s, p.tl, sh) * inv;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[j][e] = have[j] ? v[j][e] - mu : 0.f;
  }
  float s2 = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int e = 0; e < VEC; ++e) s2 = fmaf(v[j][e], v[j][e], s2);
  return rsqrtf(fmaf(team_sum(s2, p.tl, sh), inv, p.eps));
}

template <typename T, int VEC, int NV>
__global__ void __launch_bounds__(max_threads(VEC)) norm_fwd(const Args p) {
  __shared__ float sh[32];
  const Place q = place(p);
  int ch[NV];
  bool have[NV];
  float w[NV][VEC], b[NV][VEC];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int k = (q.lane + j * q.width) * VEC;
    have[j] = q.on && k < p.G;
    ch[j] = have[j] ? q.group * p.G + k : 0;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      w[j][e] = have[j] && p.w != nullptr ? p.w[ch[j] + e] : 1.f;
      b[j][e] = have[j] && p.b != nullptr ? p.b[ch[j] + e] : 0.f;
    }
  }
  const long long step = (long long)gridDim.y * p.rpi;
  for (long long base = (long long)blockIdx.y * p.rpi; base < p.R; base += step) {
    const long long row = base + q.sub;
    const bool rowok = row < p.R;
    float v[NV][VEC], z[NV][VEC];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[j][e] = z[j][e] = 0.f;
      if (have[j] && rowok) {
        load_vec<T, VEC>(static_cast<const T*>(p.x) + row * p.xs + ch[j], v[j]);
        if (p.z != nullptr) load_vec<T, VEC>(static_cast<const T*>(p.z) + row * p.zs + ch[j], z[j]);
      }
    }
    const float rs = normalise<VEC, NV>(v, have, p, sh);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (!(have[j] && rowok)) continue;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        float u = fmaf(v[j][e] * rs, w[j][e], b[j][e]);
        if (p.z != nullptr)
          u *= p.act ? silu_of<T>(z[j][e]) : z[j][e];
        else if (p.act)
          u = silu_of<T>(u);
        v[j][e] = u;
      }
      store_vec<T, VEC>(static_cast<T*>(p.y) + row * p.C + ch[j], v[j]);
    }
  }
}

template <typename T, int VEC, int NV>
__global__ void __launch_bounds__(max_threads(VEC)) norm_bwd(const Args p) {
  __shared__ float sh[32];
  extern __shared__ float fold[];  // [rpi][gpc * G] when a block works on several rows
  const Place q = place(p);
  const float inv = 1.f / (float)p.G;
  int ch[NV];
  bool have[NV];
  float w[NV][VEC], dw[NV][VEC], db[NV][VEC];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int k = (q.lane + j * q.width) * VEC;
    have[j] = q.on && k < p.G;
    ch[j] = have[j] ? q.group * p.G + k : 0;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      w[j][e] = have[j] && p.w != nullptr ? p.w[ch[j] + e] : 1.f;
      dw[j][e] = db[j][e] = 0.f;
    }
  }
  const long long step = (long long)gridDim.y * p.rpi;
  for (long long base = (long long)blockIdx.y * p.rpi; base < p.R; base += step) {
    const long long row = base + q.sub;
    const bool rowok = row < p.R;
    float v[NV][VEC], d[NV][VEC];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[j][e] = d[j][e] = 0.f;
      if (have[j] && rowok) {
        load_vec<T, VEC>(static_cast<const T*>(p.x) + row * p.xs + ch[j], v[j]);
        load_vec<T, VEC>(static_cast<const T*>(p.dy) + row * p.gs + ch[j], d[j]);
      }
    }
    const float rs = normalise<VEC, NV>(v, have, p, sh);
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (!(have[j] && rowok)) continue;
      float z[VEC];
      if (p.z != nullptr) load_vec<T, VEC>(static_cast<const T*>(p.z) + row * p.zs + ch[j], z);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float xh = v[j][e] * rs;
        const float u = fmaf(xh, w[j][e], p.b != nullptr ? p.b[ch[j] + e] : 0.f);
        float du = d[j][e];
        if (p.z != nullptr) {
          float f = z[e], df = 1.f;
          if (p.act) silu_grad<T>(z[e], f, df);
          z[e] = du * u * df;
          du *= f;
        } else if (p.act) {
          float f, df;
          silu_grad<T>(u, f, df);
          du *= df;
        }
        dw[j][e] = fmaf(du, xh, dw[j][e]);
        db[j][e] += du;
        const float dxh = du * w[j][e];
        s1 += dxh;
        s2 = fmaf(dxh, xh, s2);
        v[j][e] = xh;
        d[j][e] = dxh;
      }
      if (p.z != nullptr) store_vec<T, VEC>(static_cast<T*>(p.dz) + row * p.C + ch[j], z);
    }
    const float m1 = p.center ? team_sum(s1, p.tl, sh) * inv : 0.f;
    const float m2 = team_sum(s2, p.tl, sh) * inv;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (!(have[j] && rowok)) continue;
#pragma unroll
      for (int e = 0; e < VEC; ++e) d[j][e] = rs * (d[j][e] - m1 - v[j][e] * m2);
      store_vec<T, VEC>(static_cast<T*>(p.dx) + row * p.C + ch[j], d[j]);
    }
  }
  if (p.part == nullptr) return;
  // One row of dw and db sums for the block: the block's rows are added in order.
  const int span = p.gpc * p.G;
  const int first = blockIdx.x * span;
  for (int pass = 0; pass < 2; ++pass) {
    float* out = p.part + ((long long)blockIdx.y * 2 + pass) * p.C;
    if (p.rpi == 1) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (have[j])
#pragma unroll
          for (int e = 0; e < VEC; ++e) out[ch[j] + e] = pass == 0 ? dw[j][e] : db[j][e];
      continue;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (have[j])
#pragma unroll
        for (int e = 0; e < VEC; ++e) fold[q.sub * span + ch[j] - first + e] = pass == 0 ? dw[j][e] : db[j][e];
    __syncthreads();
    for (int k = threadIdx.x; k < span && first + k < p.C; k += blockDim.x) {
      float acc = 0.f;
      for (int s = 0; s < p.rpi; ++s) acc += fold[s * span + k];
      out[first + k] = acc;
    }
  }
}

struct StoreParams {
  float *dw, *db;
  int C;
  __device__ void operator()(int c, float v) const {
    if (c < C) {
      if (dw != nullptr) dw[c] = v;
    } else if (db != nullptr) {
      db[c - C] = v;
    }
  }
};

constexpr int kMaxGroup = 4096;

struct Plan {
  int vec, nv, threads;
  dim3 grid;
};

// How a call is cut up. Vectors are the widest (up to 16 bytes) that the group size, the
// row strides and the addresses allow. `blocks`: rows of blocks wanted.
Plan make_plan(Args& p, int elem, const void* const* ptrs, int nptr, int blocks_per_sm) {
  Plan q{};
  q.vec = 16 / elem;
  uintptr_t bits = (uintptr_t)(p.G * elem);
  bits |= (uintptr_t)(p.xs * elem) | (uintptr_t)(p.zs * elem) | (uintptr_t)(p.gs * elem);
  for (int k = 0; k < nptr; ++k) bits |= reinterpret_cast<uintptr_t>(ptrs[k]);
  while (q.vec > 1 && (bits & (q.vec * elem - 1)) != 0) q.vec >>= 1;
  const int nvec = (p.G + q.vec - 1) / q.vec;
  q.threads = 256;
  if (nvec <= 128) {
    p.tl = 1;
    while (p.tl < 32 && p.tl < nvec) p.tl <<= 1;
    q.nv = (nvec + p.tl - 1) / p.tl;
    q.nv = q.nv > 2 ? 4 : q.nv;
    const int teams = q.threads / p.tl;
    p.gpc = teams < p.groups ? teams : p.groups;
    p.rpi = teams / p.gpc;
  } else {
    p.tl = 0;
    p.gpc = p.rpi = 1;
    const int cap = max_threads(q.vec);
    q.nv = 1;
    while (q.nv < 4 && nvec > 256 * q.nv) q.nv <<= 1;
    q.threads = ((nvec + q.nv - 1) / q.nv + 31) / 32 * 32;
    if (q.threads > cap) q.threads = cap;
  }
  const int gx = (p.groups + p.gpc - 1) / p.gpc;
  const long long need = (p.R + p.rpi - 1) / p.rpi;
  long long want = (long long)sm_count() * blocks_per_sm / gx;
  want = want < 1 ? 1 : want;
  const long long gy = need < want ? need : want;
  q.grid = dim3(gx, (unsigned)(gy < 1 ? 1 : gy));
  return q;
}

constexpr int kFwdBlocks = 8, kBwdBlocks = 4;

template <typename T, int VEC>
void launch(const Plan& q, const Args& p, bool bwd, cudaStream_t st) {
  const size_t fold = bwd && p.part != nullptr && p.rpi > 1 ? sizeof(float) * p.rpi * p.gpc * p.G : 0;
  auto go = [&](auto nv) {
    constexpr int NV = decltype(nv)::value;
    if (bwd)
      norm_bwd<T, VEC, NV><<<q.grid, q.threads, fold, st>>>(p);
    else
      norm_fwd<T, VEC, NV><<<q.grid, q.threads, 0, st>>>(p);
  };
  if (q.nv == 1)
    go(std::integral_constant<int, 1>());
  else if (q.nv == 2)
    go(std::integral_constant<int, 2>());
  else
    go(std::integral_constant<int, 4>());
}

int dispatch(const Plan& q, const Args& p, int dtype, bool bwd, cudaStream_t st) {
  if (dtype == THM_BF16) {
    using T = __nv_bfloat16;
    if (q.vec == 8) launch<T, 8>(q, p, bwd, st);
    else if (q.vec == 4) launch<T, 4>(q, p, bwd, st);
    else if (q.vec == 2) launch<T, 2>(q, p, bwd, st);
    else launch<T, 1>(q, p, bwd, st);
  } else {
    if (q.vec == 4) launch<float, 4>(q, p, bwd, st);
    else if (q.vec == 2) launch<float, 2>(q, p, bwd, st);
    else launch<float, 1>(q, p, bwd, st);
  }
  return check_launch();
}

int check_sizes(long long R, int C, int G, int act, int dtype) {
  if (R < 0 || C < 0 || G <= 0 || C % G != 0) return THM_ERR_INVALID;
  if (act != THM_ACT_NONE && act != THM_ACT_SILU) return THM_ERR_INVALID;
  if (dtype != THM_F32 && dtype != THM_BF16) return THM_ERR_INVALID;
  if (G > kMaxGroup) return THM_ERR_UNSUPPORTED;
  return THM_OK;
}

Args make_args(long long R, int C, int G, int center, int act, float eps) {
  Args p{};
  p.R = R; p.C = C; p.G = G; p.groups = C / G;
  p.center = center != 0; p.act = act == THM_ACT_SILU; p.eps = eps;
  return p;
}

}  // namespace gnorm
}  // namespace thm

extern "C" int thm_group_norm_fwd(const void* x, const void* gate, const float* weight, const float* bias, void* y,
                                  long long x_rs, long long gate_rs, long long R, int C, int G, int center,
                                  int activation, float eps, int dtype, thm_stream_t stream) {
  using namespace thm;
  const int bad = gnorm::check_sizes(R, C, G, activation, dtype);
  if (bad != THM_OK) return bad;
  if (R == 0 || C == 0) return THM_OK;
  if (!x || !y) return THM_ERR_INVALID;
  gnorm::Args p = gnorm::make_args(R, C, G, center, activation, eps);
  p.x = x; p.z = gate; p.w = weight; p.b = bias; p.y = y;
  p.xs = x_rs; p.zs = gate != nullptr ? gate_rs : 0;
  const void* ptrs[] = {x, gate, y};
  const gnorm::Plan q = gnorm::make_plan(p, dtype == THM_BF16 ? 2 : 4, ptrs, 3, gnorm::kFwdBlocks);
  return gnorm::dispatch(q, p, dtype, false, reinterpret_cast<cudaStream_t>(stream));
}

// Rows of the workspace [rows, 2, C] that thm_group_norm_bwd may use at most.
extern "C" int thm_group_norm_bwd_parts(long long R, int C, int G) {
  (void)C;
  (void)G;
  const long long most = (long long)thm::sm_count() * thm::gnorm::kBwdBlocks;
  return (int)(R < most ? (R < 1 ? 1 : R) : most);
}

extern "C" int thm_group_norm_bwd(const void* x, const void* gate, const float* weight, const float* bias,
                                  const void* dy, void* dx, void* dgate, float* dweight, float* dbias,
                                  float* workspace, long long x_rs, long long gate_rs, long long dy_rs, long long R,
                                  int C, int G, int center, int activation, float eps, int dtype,
                                  thm_stream_t stream) {
  using namespace thm;
  const int bad = gnorm::check_sizes(R, C, G, activation, dtype);
  if (bad != THM_OK) return bad;
  if (C == 0) return THM_OK;
  const bool params = dweight != nullptr || dbias != nullptr;
  if (params && !workspace) return THM_ERR_INVALID;
  if (R > 0 && (!x || !dy || !dx || (gate != nullptr) != (dgate != nullptr))) return THM_ERR_INVALID;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  int rows = 0;
  if (R > 0) {
    gnorm::Args p = gnorm::make_args(R, C, G, center, activation, eps);
    p.x = x; p.z = gate; p.w = weight; p.b = bias; p.dy = dy; p.dx = dx; p.dz = dgate;
    p.part = params ? workspace : nullptr;
    p.xs = x_rs; p.zs = gate != nullptr ? gate_rs : 0; p.gs = dy_rs;
    const void* ptrs[] = {x, gate, dy, dx, dgate};
    const gnorm::Plan q = gnorm::make_plan(p, dtype == THM_BF16 ? 2 : 4, ptrs, 5, gnorm::kBwdBlocks);
    const int e = gnorm::dispatch(q, p, dtype, true, st);
    if (e != THM_OK) return e;
    rows = (int)q.grid.y;
  }
  if (params) {
    sum_parts(workspace, rows, 2 * C, gnorm::StoreParams{dweight, dbias, C}, st);
    return check_launch();
  }
  return THM_OK;
}
