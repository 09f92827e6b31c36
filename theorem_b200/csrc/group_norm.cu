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
  float* part;             // backward: [blocks in y, 1 or 2, C] sums of dw and db, or null
  long long xs, zs, gs;    // row strides of x, z, dy
  long long R;
  int C, G, groups;
  int tl;                  // lanes of a team; 0: the whole block
  int gpc, rpi;            // groups and rows that a block works on at a time
  int center, flags;
  float eps;
};

// Sum over the team, the same value in each of its threads.
__device__ __forceinline__ float team_sum(float v, int tl, float* sh) {
  if (tl != 0) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
      if (tl > o) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();  // the previous sum has been read
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
  for (int k = 0; k < (int)(blockDim.x >> 5); ++k) s += sh[k];
  return s;
}
// Two at a time: their steps overlap, and a block needs one exchange for both.
__device__ __forceinline__ float2 team_sum2(float2 v, int tl, float2* sh) {
  if (tl != 0) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
      if (tl > o)
        v = __fadd2_rn(v, make_float2(__shfl_xor_sync(0xffffffffu, v.x, o), __shfl_xor_sync(0xffffffffu, v.y, o)));
    return v;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    v = __fadd2_rn(v, make_float2(__shfl_xor_sync(0xffffffffu, v.x, o), __shfl_xor_sync(0xffffffffu, v.y, o)));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  float2 s = make_float2(0.f, 0.f);
  for (int k = 0; k < (int)(blockDim.x >> 5); ++k) s = __fadd2_rn(s, sh[k]);
  return s;
}

// Where a thread stands: its team's group and row offset in the block, and whether the
// team has work.
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

// Threads of a block at most: 4096 channels of single elements take 512 threads with eight each.
constexpr int max_threads(int vec, int nv) { return (vec == 1 && nv == 8) || vec == 2 ? 512 : 256; }

// What a call does besides the norm: template arguments of the kernels.
constexpr int kGate = 1, kAct = 2, kBias = 4;

__device__ __forceinline__ float2 f2(float v) { return make_float2(v, v); }

// sigmoid of a pair; bf16 outputs take the hardware exponential and reciprocal.
template <typename T>
__device__ __forceinline__ float2 sigmoid2(float2 x) {
  if constexpr (sizeof(T) == 2) {
    const float2 e = __fmul2_rn(x, f2(-1.4426950408889634f));
    const float2 d = __fadd2_rn(make_float2(ex2_approx(e.x), ex2_approx(e.y)), f2(1.f));
    return make_float2(rcp_approx(d.x), rcp_approx(d.y));
  } else {
    return make_float2(sigmoid<T>(x.x), sigmoid<T>(x.y));
  }
}

// A thread's share of a group: NV vectors of VEC channels as fp32 pairs (a single channel has
// an empty second half).
//
// EDGE: the group's borders are no multiples of a vector, but the rows' are. Its lanes then take the
// aligned vectors that cover it, two of which may hold channels of its neighbours: those are taken
// as zeros, which no sum sees, and not stored.
template <typename T, int VEC, int NV, bool EDGE>
struct Share {
  static constexpr int kPairs = (VEC * NV + 1) / 2;
  using Vec = Pack<T, VEC>;
  int c0, step;    // channel of vector j: c0 + j step
  bool have[NV];
  uint32_t valid;  // EDGE: which channels are the group's, bit j VEC + e

  __device__ __forceinline__ Share(const Args& p, const Place& q) {
    step = q.width * VEC;
    valid = 0;
    if constexpr (EDGE) {
      const int first = q.group * p.G, end = first + p.G;
      c0 = q.on ? first / VEC * VEC + q.lane * VEC : 0;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        have[j] = q.on && c0 + j * step < end;
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          if (have[j] && c0 + j * step + e >= first && c0 + j * step + e < end) valid |= 1u << (j * VEC + e);
      }
    } else {
      c0 = q.on ? q.group * p.G + q.lane * VEC : 0;
#pragma unroll
      for (int j = 0; j < NV; ++j) have[j] = q.on && (q.lane + j * q.width) * VEC < p.G;
    }
  }
  __device__ __forceinline__ bool mine(int j, int e) const { return EDGE ? (valid >> (j * VEC + e)) & 1 : have[j]; }
  // Zeros for what is not the group's (absent vectors are zeros as loaded).
  __device__ __forceinline__ void mask(float2 (&f)[kPairs]) const {
    if constexpr (EDGE) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          if (!mine(j, e)) at(f, j, e) = 0.f;
    }
  }
  // The vectors at t (channel c0 of a row); absent ones, and all where there is no row, are 0.
  __device__ __forceinline__ void load(const T* t, bool ok, Vec (&raw)[NV]) const {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      raw[j] = Vec{};
      if (have[j] && ok) raw[j] = *reinterpret_cast<const Vec*>(t + j * step);
    }
  }
  static __device__ __forceinline__ void widen(const Vec (&raw)[NV], float2 (&f)[kPairs]) {
    if constexpr (VEC == 1) {
#pragma unroll
      for (int j = 0; j < kPairs; ++j)
        f[j] = make_float2(to_f32<T>(raw[2 * j].v[0]), 2 * j + 1 < NV ? to_f32<T>(raw[2 * j + 1 < NV ? 2 * j + 1 : 0].v[0]) : 0.f);
    } else {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < VEC / 2; ++e) {
          if constexpr (sizeof(T) == 2) {
            const uint32_t w = reinterpret_cast<const uint32_t*>(&raw[j])[e];
            f[j * VEC / 2 + e] = make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
          } else {
            f[j * VEC / 2 + e] = make_float2(raw[j].v[2 * e], raw[j].v[2 * e + 1]);
          }
        }
    }
  }
  __device__ __forceinline__ void store(T* r, bool ok, const float2 (&f)[kPairs]) const {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (!(have[j] && ok)) continue;
      if constexpr (EDGE) {
        constexpr uint32_t kAll = (1u << VEC) - 1;
        if (((valid >> (j * VEC)) & kAll) != kAll) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const int k = j * VEC + e;
            if (mine(j, e)) r[j * step + e] = from_f32<T>(k & 1 ? f[k / 2].y : f[k / 2].x);
          }
          continue;
        }
      }
      if constexpr (VEC == 1) {
        r[j * step] = from_f32<T>(j & 1 ? f[j / 2].y : f[j / 2].x);
      } else {
        Vec v;
#pragma unroll
        for (int e = 0; e < VEC / 2; ++e) {
          const float2 w = f[j * VEC / 2 + e];
          if constexpr (sizeof(T) == 2)
            reinterpret_cast<uint32_t*>(&v)[e] = pack_bf16x2(w.x, w.y);
          else
            reinterpret_cast<float2*>(&v)[e] = w;
        }
        *reinterpret_cast<Vec*>(r + j * step) = v;
      }
    }
  }
  // Element e of vector j in pairs, for the parameters and their gradients.
  static __device__ __forceinline__ float& at(float2 (&f)[kPairs], int j, int e) {
    const int k = j * VEC + e;
    return k & 1 ? f[k / 2].y : f[k / 2].x;
  }
  __device__ __forceinline__ void params(const float* t, float absent, float2 (&f)[kPairs]) const {
#pragma unroll
    for (int k = 0; k < kPairs; ++k) f[k] = f2(0.f);
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < VEC; ++e) at(f, j, e) = mine(j, e) ? (t != nullptr ? t[c0 + j * step + e] : absent) : 0.f;
  }
  // Sum of a over the thread's channels.
  static __device__ __forceinline__ float sum(const float2 (&a)[kPairs]) {
    float2 s = a[0];
#pragma unroll
    for (int k = 1; k < kPairs; ++k) s = __fadd2_rn(s, a[k]);
    return s.x + s.y;
  }
  static __device__ __forceinline__ float dot(const float2 (&a)[kPairs], const float2 (&b)[kPairs]) {
    float2 s = __fmul2_rn(a[0], b[0]);
#pragma unroll
    for (int k = 1; k < kPairs; ++k) s = __ffma2_rn(a[k], b[k], s);
    return s.x + s.y;
  }
  // Take the mean off v where the group is centred (absent channels stay 0); 1 / sqrt(mean of
  // squares + eps).
  __device__ __forceinline__ float normalise(float2 (&v)[kPairs], const Args& p, float* sh) const {
    const float inv = 1.f / (float)p.G;
    if (p.center) {
      const float mu = team_sum(sum(v), p.tl, sh) * inv;
#pragma unroll
      for (int k = 0; k < kPairs; ++k) v[k] = __fadd2_rn(v[k], f2(-mu));
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          if (!mine(j, e)) at(v, j, e) = 0.f;
      if constexpr (VEC * NV == 1) v[0].y = 0.f;
    }
    return rsqrtf(fmaf(team_sum(dot(v, v), p.tl, sh), inv, p.eps));
  }
};

// The next row's loads are issued before a row is worked on, so that a row's arithmetic hides
// them. Bound by HBM: 131072 x 2048 bf16 in groups of 128 with a gate takes 260 to 265 us, 6.1 TB/s
// (0.93 of a copy), at 18 instructions per 32 elements; without packed arithmetic, the loads ahead
// and the flags as template arguments it took 30 and 366 us.
template <typename T, int VEC, int NV, bool EDGE, int FLAGS>
__global__ void __launch_bounds__(max_threads(VEC, NV)) norm_fwd(const Args p) {
  __shared__ float sh[32];
  using S = Share<T, VEC, NV, EDGE>;
  constexpr int N = S::kPairs;
  const Place q = place(p);
  const S me(p, q);
  float2 w[N], b[N];
  me.params(p.w, 1.f, w);
  me.params(p.b, 0.f, b);
  const long long step = (long long)gridDim.y * p.rpi;
  long long row = (long long)blockIdx.y * p.rpi + q.sub;
  const T *x = static_cast<const T*>(p.x) + row * p.xs + me.c0, *zp = static_cast<const T*>(p.z) + row * p.zs + me.c0;
  T* y = static_cast<T*>(p.y) + row * p.C + me.c0;
  const long long xstep = step * p.xs, zstep = step * p.zs, ystep = step * p.C;
  typename S::Vec xr[NV], zr[NV];
  me.load(x, row < p.R, xr);
  if constexpr ((FLAGS & kGate) != 0) me.load(zp, row < p.R, zr);
  for (; row - q.sub < p.R; row += step) {
    float2 v[N], z[N];
    S::widen(xr, v);
    me.mask(v);
    if constexpr ((FLAGS & kGate) != 0) S::widen(zr, z);
    const bool more = row + step < p.R;
    me.load(x += xstep, more, xr);
    if constexpr ((FLAGS & kGate) != 0) me.load(zp += zstep, more, zr);
    const float rs = me.normalise(v, p, sh);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      float2 u = __fmul2_rn(v[k], f2(rs));
      u = (FLAGS & kBias) != 0 ? __ffma2_rn(u, w[k], b[k]) : __fmul2_rn(u, w[k]);
      if constexpr ((FLAGS & kGate) != 0) {
        if constexpr ((FLAGS & kAct) != 0) u = __fmul2_rn(u, sigmoid2<T>(z[k]));
        u = __fmul2_rn(u, z[k]);
      } else if constexpr ((FLAGS & kAct) != 0) {
        u = __fmul2_rn(u, sigmoid2<T>(u));
      }
      v[k] = u;
    }
    me.store(y, row < p.R, v);
    y += ystep;
  }
}

// As above with three tensors in, two out and the parameters' sums in registers: 32768 x 2048 bf16
// in groups of 128 with a gate takes 113 us and 3 for the second launch, 5.6 TB/s (0.86 of a copy),
// issuing on 67 % of the cycles; three blocks of 80 registers an SM. Narrow groups are bound by
// their instructions: 7777 x 1960 fp32 in groups of 49 with SiLU takes 69 us (0.40 of a copy; with single
// elements 148 with two channels a lane and the flags looked up, 100 with two blocks an SM, then 76).
template <typename T, int VEC, int NV, bool EDGE, int FLAGS>
__global__ void __launch_bounds__(max_threads(VEC, NV), (VEC * NV == 8 && sizeof(T) == 2) || VEC * NV == 4 ? 3 : 1) norm_bwd(const Args p) {
  __shared__ float sh[32];
  __shared__ float2 sh2[32];
  extern __shared__ float fold[];  // [rpi][gpc * G] when a block works on several rows
  using S = Share<T, VEC, NV, EDGE>;
  constexpr int N = S::kPairs;
  const Place q = place(p);
  const S me(p, q);
  const float inv = 1.f / (float)p.G;
  float2 w[N], b[N], dw[N], db[N];
  me.params(p.w, 1.f, w);
  if constexpr ((FLAGS & kBias) != 0) me.params(p.b, 0.f, b);
#pragma unroll
  for (int k = 0; k < N; ++k) dw[k] = db[k] = f2(0.f);
  const long long step = (long long)gridDim.y * p.rpi;
  long long row = (long long)blockIdx.y * p.rpi + q.sub;
  const T *x = static_cast<const T*>(p.x) + row * p.xs + me.c0, *dy = static_cast<const T*>(p.dy) + row * p.gs + me.c0,
          *zp = static_cast<const T*>(p.z) + row * p.zs + me.c0;
  T *dx = static_cast<T*>(p.dx) + row * p.C + me.c0, *dz = static_cast<T*>(p.dz) + row * p.C + me.c0;
  const long long xstep = step * p.xs, gstep = step * p.gs, zstep = step * p.zs, ostep = step * p.C;
  typename S::Vec xr[NV], gr[NV], zr[NV];
  me.load(x, row < p.R, xr);
  me.load(dy, row < p.R, gr);
  if constexpr ((FLAGS & kGate) != 0) me.load(zp, row < p.R, zr);
  for (; row - q.sub < p.R; row += step) {
    float2 v[N], d[N], z[N];
    S::widen(xr, v);
    S::widen(gr, d);
    if constexpr ((FLAGS & kGate) != 0) S::widen(zr, z);
    me.mask(v);
    me.mask(d);
    if constexpr ((FLAGS & kGate) != 0) me.mask(z);
    const bool more = row + step < p.R;
    me.load(x += xstep, more, xr);
    me.load(dy += gstep, more, gr);
    if constexpr ((FLAGS & kGate) != 0) me.load(zp += zstep, more, zr);
    const float rs = me.normalise(v, p, sh);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      v[k] = __fmul2_rn(v[k], f2(rs));  // xh
      const float2 u = (FLAGS & kBias) != 0 ? __ffma2_rn(v[k], w[k], b[k]) : __fmul2_rn(v[k], w[k]);
      // du and, with a gate, dz = dy u act'(z); silu'(x) = s (1 + x (1 - s)).
      float2 du = d[k];
      if constexpr ((FLAGS & kGate) != 0) {
        float2 f = z[k], dz = __fmul2_rn(du, u);
        if constexpr ((FLAGS & kAct) != 0) {
          const float2 s = sigmoid2<T>(f);
          dz = __fmul2_rn(dz, __fmul2_rn(s, __ffma2_rn(f, __ffma2_rn(s, f2(-1.f), f2(1.f)), f2(1.f))));
          f = __fmul2_rn(f, s);
        }
        z[k] = dz;
        du = __fmul2_rn(du, f);
      } else if constexpr ((FLAGS & kAct) != 0) {
        const float2 s = sigmoid2<T>(u);
        du = __fmul2_rn(du, __fmul2_rn(s, __ffma2_rn(u, __ffma2_rn(s, f2(-1.f), f2(1.f)), f2(1.f))));
      }
      dw[k] = __ffma2_rn(du, v[k], dw[k]);
      if constexpr ((FLAGS & kBias) != 0) db[k] = __fadd2_rn(db[k], du);
      d[k] = __fmul2_rn(du, w[k]);  // dxh
    }
    if constexpr ((FLAGS & kGate) != 0) me.store(dz, row < p.R, z);
    if (p.center) {
      const float2 m = team_sum2(make_float2(S::sum(d), S::dot(d, v)), p.tl, sh2);
#pragma unroll
      for (int k = 0; k < N; ++k)
        d[k] = __fmul2_rn(f2(rs), __ffma2_rn(v[k], f2(-m.y * inv), __fadd2_rn(d[k], f2(-m.x * inv))));
    } else {
      const float m2 = team_sum(S::dot(d, v), p.tl, sh) * inv;
#pragma unroll
      for (int k = 0; k < N; ++k) d[k] = __fmul2_rn(f2(rs), __ffma2_rn(v[k], f2(-m2), d[k]));
    }
    me.store(dx, row < p.R, d);
    dx += ostep;
    dz += ostep;
  }
  if (p.part == nullptr) return;
  let_dependents_launch();
  // One row of dw (and db) sums for the block: the block's rows are added in order.
  const int span = p.gpc * p.G, first = blockIdx.x * span;
  const int npass = (FLAGS & kBias) != 0 ? 2 : 1;
  for (int pass = 0; pass < npass; ++pass) {
    float* out = p.part + ((long long)blockIdx.y * npass + pass) * p.C;
    if (pass == 1)
#pragma unroll
      for (int k = 0; k < N; ++k) dw[k] = db[k];
    if (p.rpi == 1) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          if (me.mine(j, e)) out[me.c0 + j * me.step + e] = S::at(dw, j, e);
      continue;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (me.mine(j, e)) fold[q.sub * span + me.c0 + j * me.step - first + e] = S::at(dw, j, e);
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
  bool edge;
  dim3 grid;
};

// How a call is cut up. Vectors are the widest (up to 16 bytes) that the group size, the
// row strides and the addresses allow.
Plan make_plan(Args& p, int elem, const void* const* ptrs, int nptr, int blocks_per_sm) {
  Plan q{};
  q.vec = 16 / elem;
  uintptr_t bits = (uintptr_t)(p.C * elem);
  bits |= (uintptr_t)(p.xs * elem) | (uintptr_t)(p.zs * elem) | (uintptr_t)(p.gs * elem);
  for (int k = 0; k < nptr; ++k) bits |= reinterpret_cast<uintptr_t>(ptrs[k]);
  int nvec = p.G / q.vec;
  if ((bits & 15) != 0 || p.G % q.vec != 0) {
    // Rows of whole vectors, groups that are not: masked borders, where they are a small part of the
    // group (7777 x 1960 fp32 in groups of 49, backward: 69 us instead of 76 with single elements;
    // 20000 x 1960 bf16 in groups of 245: 103 us)
    // and a block's registers hold its vectors.
    nvec = (p.G + 2 * q.vec - 2) / q.vec;
    q.edge = (bits & 15) == 0 && p.G >= 4 * q.vec && nvec <= 256 * (16 / q.vec);
    if (!q.edge) {
      bits |= (uintptr_t)(p.G * elem);
      q.vec = (bits & (2 * elem - 1)) == 0 ? 2 : 1;
      nvec = p.G / q.vec;
    }
  }
  // Whole 16-byte vectors: a lane has one, so that more lanes have loads in flight, and never more
  // than 16 channels, whose sums and parameters fit its registers. Narrow ones: a lane has four,
  // because their sums across lanes cost more than their loads.
  const bool wide = q.vec * elem == 16;
  const int most = wide ? 16 / q.vec : q.vec == 2 ? 4 : 8;            // vectors of a lane
  const int least = wide ? 1 : q.vec == 1 && nvec > 128 ? 8 : 4;
  if (nvec <= 32 * most) {
    p.tl = 1;
    while (p.tl < 32 && p.tl * least < nvec) p.tl <<= 1;
    q.nv = (nvec + p.tl - 1) / p.tl;
    q.nv = !wide ? least : q.nv > 2 ? 4 : q.nv;
    // Blocks of equal shares of a row's groups, and no more threads than those shares have lanes.
    const int teams = 256 / p.tl, cuts = (p.groups + teams - 1) / teams;
    p.gpc = (p.groups + cuts - 1) / cuts;
    p.rpi = teams / p.gpc;
    q.threads = (p.gpc * p.rpi * p.tl + 31) / 32 * 32;
  } else {
    p.tl = 0;
    p.gpc = p.rpi = 1;
    q.nv = wide ? 1 : most;
    while (wide && nvec > 256 * q.nv) q.nv <<= 1;
    q.threads = ((nvec + q.nv - 1) / q.nv + 31) / 32 * 32;
  }
  const int gx = (p.groups + p.gpc - 1) / p.gpc;
  const long long need = (p.R + p.rpi - 1) / p.rpi;
  // As many threads as blocks_per_sm blocks of 256 an SM; no more rows of blocks than that has
  // blocks (the workspace of the backward pass).
  const long long full = (long long)sm_count() * blocks_per_sm;
  long long want = (long long)sm_count() * (blocks_per_sm * 256 / q.threads) / gx;
  want = want < 1 ? 1 : want > full ? full : want;
  const long long gy = need < want ? need : want;
  q.grid = dim3(gx, (unsigned)(gy < 1 ? 1 : gy));
  return q;
}

constexpr int kFwdBlocks = 4, kBwdBlocks = 3;

template <typename T, int VEC, int NV, bool EDGE, int FLAGS>
void launch(const Plan& q, const Args& p, bool bwd, cudaStream_t st) {
  const size_t fold = bwd && p.part != nullptr && p.rpi > 1 ? sizeof(float) * p.rpi * p.gpc * p.G : 0;
  if (bwd)
    norm_bwd<T, VEC, NV, EDGE, FLAGS><<<q.grid, q.threads, fold, st>>>(p);
  else
    norm_fwd<T, VEC, NV, EDGE, FLAGS><<<q.grid, q.threads, 0, st>>>(p);
}

template <typename T, int VEC, int NV, bool EDGE = false>
void launch_flags(const Plan& q, const Args& p, bool bwd, cudaStream_t st) {
  switch (p.flags) {
    case 0: launch<T, VEC, NV, EDGE, 0>(q, p, bwd, st); break;
    case 1: launch<T, VEC, NV, EDGE, 1>(q, p, bwd, st); break;
    case 2: launch<T, VEC, NV, EDGE, 2>(q, p, bwd, st); break;
    case 3: launch<T, VEC, NV, EDGE, 3>(q, p, bwd, st); break;
    case 4: launch<T, VEC, NV, EDGE, 4>(q, p, bwd, st); break;
    case 5: launch<T, VEC, NV, EDGE, 5>(q, p, bwd, st); break;
    case 6: launch<T, VEC, NV, EDGE, 6>(q, p, bwd, st); break;
    default: launch<T, VEC, NV, EDGE, 7>(q, p, bwd, st); break;
  }
}

template <typename T>
int dispatch(const Plan& q, const Args& p, bool bwd, cudaStream_t st) {
  constexpr int kWide = 16 / sizeof(T);
  if (q.edge) {
    if (q.nv == 1) launch_flags<T, kWide, 1, true>(q, p, bwd, st);
    else if (q.nv == 2) launch_flags<T, kWide, 2, true>(q, p, bwd, st);
    else if constexpr (sizeof(T) == 4) launch_flags<T, kWide, 4, true>(q, p, bwd, st);
  } else if (q.vec == kWide) {
    if (q.nv == 1) launch_flags<T, kWide, 1>(q, p, bwd, st);
    else if (q.nv == 2) launch_flags<T, kWide, 2>(q, p, bwd, st);
    else if constexpr (sizeof(T) == 4) launch_flags<T, kWide, 4>(q, p, bwd, st);
  } else if (q.vec == 2) {
    launch_flags<T, 2, 4>(q, p, bwd, st);
  } else if (q.nv == 4) {
    launch_flags<T, 1, 4>(q, p, bwd, st);
  } else {
    launch_flags<T, 1, 8>(q, p, bwd, st);
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
  p.center = center != 0; p.flags = act == THM_ACT_SILU ? kAct : 0; p.eps = eps;
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
  p.flags |= (gate != nullptr ? gnorm::kGate : 0) | (bias != nullptr ? gnorm::kBias : 0);
  p.xs = x_rs; p.zs = gate != nullptr ? gate_rs : 0;
  const void* ptrs[] = {x, gate, y};
  const gnorm::Plan q = gnorm::make_plan(p, dtype == THM_BF16 ? 2 : 4, ptrs, 3, gnorm::kFwdBlocks);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return dtype == THM_BF16 ? gnorm::dispatch<__nv_bfloat16>(q, p, false, st) : gnorm::dispatch<float>(q, p, false, st);
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
  if ((params && !workspace) || (dbias != nullptr && bias == nullptr)) return THM_ERR_INVALID;
  if (R > 0 && (!x || !dy || !dx || (gate != nullptr) != (dgate != nullptr))) return THM_ERR_INVALID;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  int rows = 0;
  if (R > 0) {
    gnorm::Args p = gnorm::make_args(R, C, G, center, activation, eps);
    p.x = x; p.z = gate; p.w = weight; p.b = bias; p.dy = dy; p.dx = dx; p.dz = dgate;
    p.part = params ? workspace : nullptr;
    p.flags |= (gate != nullptr ? gnorm::kGate : 0) | (bias != nullptr ? gnorm::kBias : 0);
    p.xs = x_rs; p.zs = gate != nullptr ? gate_rs : 0; p.gs = dy_rs;
    const void* ptrs[] = {x, gate, dy, dx, dgate};
    const gnorm::Plan q = gnorm::make_plan(p, dtype == THM_BF16 ? 2 : 4, ptrs, 5, gnorm::kBwdBlocks);
    const int e = dtype == THM_BF16 ? gnorm::dispatch<__nv_bfloat16>(q, p, true, st) : gnorm::dispatch<float>(q, p, true, st);
    if (e != THM_OK) return e;
    rows = (int)q.grid.y;
  }
  if (params) {
    return sum_parts(workspace, rows, bias != nullptr ? 2 * C : C, gnorm::StoreParams{dweight, dbias, C}, st);
  }
  return THM_OK;
}
