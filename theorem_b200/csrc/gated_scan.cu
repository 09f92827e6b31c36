// gated_scan.cu -- per-channel gated linear recurrence over time, channel-last, and
// its gradients.
//
//   s = sigmoid(r_t)   L = decay s   a_t = e^-L   p = sigmoid(i_t)   m = sqrt(1 - a_t^2)
//   h_t = a_t h_{t-1} + m p x_t
//
// m keeps the state's variance that of p x whatever the decay. A token with r < -43 (-inf)
// holds the state: x and i are not used there.
//
// The gradients, with dh_t = dy_t + a_{t+1} dh_{t+1} (dfinal after the last token):
//   dx = dh m p          di = dh m x p (1 - p)
//   dL = dh (a^2/m p x - a h_{t-1})     dr = dL L (1 - s)     ddecay = sum dL s
//   dh0 = a_1 dh_1
// h_{t-1} is recomputed in fp32 from the state that entered each 64-row chunk, which the
// forward pass keeps (4 / 64 bytes an element), not read back from the rounded y.
#include <initializer_list>

#include "host_util.h"
#include "rowops.cuh"

namespace thm {
namespace gscan {

constexpr int kChunk = 64;

struct Args {
  const void *x, *r, *i, *dy;
  const float *decay, *h0, *dfinal;
  const int* cu;  // packed: nseq + 1 row offsets, else null
  void *y, *dx, *dr, *di;
  float *states, *final_state, *ddecay_part, *dh0;
  long long xb, xt, rb, rt, ib, it, gb, gt;  // strides of x, r, i, dy over batch and time
  int T, D, nseq, zero_rest;
};

// Rows of sequence n: dense batches have T rows at batch entry n, packed ones the rows
// [cu[n], cu[n+1]) of entry 0. Offsets outside [0, T] or out of order are clamped, so no
// access leaves the tensors. `slot` is the sequence's first chunk-state slot.
struct Seq {
  long long batch, slot;
  int lo, len;
};
__device__ __forceinline__ Seq sequence(const Args& p, int n) {
  Seq q;
  if (p.cu == nullptr) {
    q.batch = n;
    q.lo = 0;
    q.len = p.T;
    q.slot = (long long)n * ((p.T + kChunk - 1) / kChunk);
  } else {
    q.batch = 0;
    q.lo = min(max(p.cu[n], 0), p.T);
    q.len = min(max(p.cu[n + 1], q.lo), p.T) - q.lo;
    q.slot = q.lo / kChunk + n;
  }
  return q;
}

// The first row from t on that no packed sequence holds: those before the first and
// behind the last.
__device__ __forceinline__ long long rest_row(const Args& p, long long t) {
  return t < p.cu[0] ? t : max(t, (long long)max(p.cu[p.nseq], 0));
}

// --------------------------------------------------------------------------- channel pairs
// A lane works on two channels at a time (packed fp32x2 arithmetic): neighbours 2 l, 2 l + 1
// read as one access where addresses and strides allow it (ADJ), else l and l + 32.
template <typename T>
struct RawPair;
template <>
struct RawPair<__nv_bfloat16> {
  uint32_t v;
  static constexpr uint32_t kHold = 0xff80ff80u;  // -inf, -inf
  __device__ __forceinline__ float2 get() const {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  }
  __device__ __forceinline__ void hold() { v = kHold; }
  __device__ __forceinline__ void zero() { v = 0u; }
};
template <>
struct RawPair<float> {
  float2 v;
  __device__ __forceinline__ float2 get() const { return v; }
  __device__ __forceinline__ void hold() { v = make_float2(-INFINITY, -INFINITY); }
  __device__ __forceinline__ void zero() { v = make_float2(0.f, 0.f); }
};

template <typename T, bool ADJ>
__device__ __forceinline__ void load_pair(RawPair<T>& q, const T* p, bool on1) {
  if constexpr (ADJ) {
    q.v = *reinterpret_cast<const decltype(q.v)*>(p);
  } else if constexpr (sizeof(T) == 2) {
    const uint16_t* u = reinterpret_cast<const uint16_t*>(p);
    q.v = u[0] | (on1 ? (uint32_t)u[32] << 16 : 0u);
  } else {
    q.v = make_float2(p[0], on1 ? p[32] : 0.f);
  }
}
template <typename T, bool ADJ>
__device__ __forceinline__ void store_pair(T* p, float2 f, bool on1) {
  if constexpr (ADJ) {
    if constexpr (sizeof(T) == 2)
      *reinterpret_cast<uint32_t*>(p) = pack_bf16x2(f.x, f.y);
    else
      *reinterpret_cast<float2*>(p) = f;
  } else {
    p[0] = from_f32<T>(f.x);
    if (on1) p[32] = from_f32<T>(f.y);
  }
}

// A lane's channels: c0 (its first), whether it has one or two, and the second's offset.
template <bool ADJ>
struct Lane {
  int c0;
  bool on0, on1;
  static constexpr int kNext = ADJ ? 1 : 32;
  __device__ __forceinline__ Lane(int base, int D) {
    const int l = threadIdx.x & 31;
    c0 = base + (ADJ ? 2 * l : l);
    on0 = c0 < D;
    on1 = c0 + kNext < D;
  }
  __device__ __forceinline__ float2 load(const float* p) const {  // p at c0
    return make_float2(on0 ? p[0] : 0.f, on1 ? p[kNext] : 0.f);
  }
  __device__ __forceinline__ void store(float* p, float2 v) const {
    if (on0) p[0] = v.x;
    if (on1) p[kNext] = v.y;
  }
};

__device__ __forceinline__ float2 f2(float v) { return make_float2(v, v); }

__device__ __forceinline__ float ex2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float sqrt_approx(float x) {
  float r;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float min_nan(float a, float b) {  // NaN when either is
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Below this gate logit a token holds the state: sigmoid(r) < 2^-62 changes no fp32 state of
// the size of x by even 1e-2 of a rounding step, and x and i may hold anything.
constexpr float kHoldBelow = -43.f;
// e^-87 is the smallest decay of one token that stays a normal number.
constexpr float kMaxDecay = 87.f;

// s = sigmoid(r), p = sigmoid(i) of one channel. For bf16 inputs the two share a reciprocal,
// 1 / ((1 + e^-r)(1 + e^-i)), with both exponentials kept under 2^62 so that the product stays
// finite: the special-function unit is what this kernel would be bound by (16 lanes a clock
// and SM), and this takes three of its operations instead of four.
template <typename T>
__device__ __forceinline__ void sigmoids(float r, float i, float& s, float& p) {
  if constexpr (sizeof(T) == 2) {
    constexpr float kNegLog2e = -1.4426950408889634f;
    i = r < kHoldBelow ? 0.f : i;  // a held token's NaN must not reach s through the shared product
    const float A = 1.f + ex2_approx(min_nan(r * kNegLog2e, 62.f));
    const float B = 1.f + ex2_approx(min_nan(i * kNegLog2e, 62.f));
    const float q = rcp_approx(A * B);
    s = q * B;
    p = q * A;
  } else {
    s = 1.f / (1.f + expf(-r));
    p = 1.f / (1.f + expf(-i));
  }
}

// a = e^-L and m^2 = 1 - a^2 for 0 <= L <= 87, both to fp32 accuracy and without the
// special-function unit, whose exponential is off by up to 2^-22 always to the same side: in a
// product over a memory of hundreds of tokens that adds up. -L = k ln 2 + f; e^f - 1 is a
// polynomial fitted by reweighted least squares over |f| <= ln 2 / 2 (largest relative error
// 1.3e-8); t = a - 1 = 2^k (e^f - 1) + (2^k - 1) does not cancel, so neither does
// m^2 = -t (2 + t).
__device__ __forceinline__ void decay_pair(float2 L, float2& a, float2& m2) {
  constexpr float kMagic = 12582912.f;  // 1.5 2^23: adding it rounds to an integer in the low bits
  const float2 km = __ffma2_rn(L, f2(-1.4426950408889634f), f2(kMagic));
  const float2 k = __fadd2_rn(km, f2(-kMagic));
  const float2 scale = make_float2(__int_as_float((__float_as_int(km.x) << 23) + 0x3f800000),
                                   __int_as_float((__float_as_int(km.y) << 23) + 0x3f800000));
  const float2 nL = __fmul2_rn(L, f2(-1.f));
  const float2 f = __ffma2_rn(k, f2(-1.42860677e-6f), __ffma2_rn(k, f2(-0.693145752f), nL));
  float2 c = __ffma2_rn(f, f2(0.00138825101f), f2(0.00836658047f));
  c = __ffma2_rn(f, c, f2(0.0416672018f));
  c = __ffma2_rn(f, c, f2(0.166665432f));
  c = __ffma2_rn(f, c, f2(0.499999981f));
  const float2 q = __ffma2_rn(__fmul2_rn(f, f), c, f);
  a = __ffma2_rn(scale, q, scale);
  const float2 t = __ffma2_rn(scale, q, __fadd2_rn(scale, f2(-1.f)));
  m2 = __fmul2_rn(__fmul2_rn(t, f2(-1.f)), __fadd2_rn(t, f2(2.f)));
}

// One token of two channels: h -> a h + b. `decay` is already limited to kMaxDecay.
template <typename T>
__device__ __forceinline__ void token_pair(float2 x, float2 r, float2 i, float2 decay, float2& a, float2& b) {
  float2 s, p, m2;
  sigmoids<T>(r.x, i.x, s.x, p.x);
  sigmoids<T>(r.y, i.y, s.y, p.y);
  decay_pair(__fmul2_rn(decay, s), a, m2);
  const float2 m = make_float2(sqrt_approx(m2.x), sqrt_approx(m2.y));
  const float2 v = __fmul2_rn(__fmul2_rn(m, p), x);
  b = make_float2(r.x < kHoldBelow ? 0.f : v.x, r.y < kHoldBelow ? 0.f : v.y);
}

__device__ __forceinline__ float2 limit_decay(float2 d) {
  return make_float2(min_nan(d.x, kMaxDecay), min_nan(d.y, kMaxDecay));
}

// --------------------------------------------------------------------------- forward, few tokens
// A lane walks its two channels token by token: single-token steps and short runs, where there
// is nothing to split along time and a launch is all the latency there is.
constexpr int kDirectThreads = 64;

template <typename T, bool ADJ>
__global__ void __launch_bounds__(kDirectThreads) scan_direct(const Args p) {
  const Lane<ADJ> ln(((blockIdx.x * kDirectThreads + threadIdx.x) >> 5) * 64, p.D);
  const int n = blockIdx.y;
  if (!ln.on0) return;
  const int c = ln.c0;
  T* y = static_cast<T*>(p.y) + c;
  if (n == p.nseq) {  // rows of no sequence
    for (long long t = rest_row(p, 0); t < p.T; t = rest_row(p, t + 1)) store_pair<T, ADJ>(y + t * p.D, f2(0.f), ln.on1);
    return;
  }
  const Seq q = sequence(p, n);
  const T* x = static_cast<const T*>(p.x) + q.batch * p.xb + q.lo * p.xt + c;
  const T* r = static_cast<const T*>(p.r) + q.batch * p.rb + q.lo * p.rt + c;
  const T* i = static_cast<const T*>(p.i) + q.batch * p.ib + q.lo * p.it + c;
  y += (q.batch * p.T + q.lo) * p.D;
  const float2 decay = limit_decay(ln.load(p.decay + c));
  float2 h = p.h0 != nullptr ? ln.load(p.h0 + (long long)n * p.D + c) : f2(0.f);
  for (int k = 0; k < q.len; ++k) {
    if (p.states != nullptr && k % kChunk == 0) ln.store(p.states + (q.slot + k / kChunk) * p.D + c, h);
    RawPair<T> xv, rv, iv;
    load_pair<T, ADJ>(xv, x + k * p.xt, ln.on1);
    load_pair<T, ADJ>(rv, r + k * p.rt, ln.on1);
    load_pair<T, ADJ>(iv, i + k * p.it, ln.on1);
    float2 a, b;
    token_pair<T>(xv.get(), rv.get(), iv.get(), decay, a, b);
    h = __ffma2_rn(a, h, b);
    store_pair<T, ADJ>(y + (long long)k * p.D, h, ln.on1);
  }
  if (p.final_state != nullptr) ln.store(p.final_state + (long long)n * p.D + c, h);
}

// --------------------------------------------------------------------------- forward, many tokens
// A block takes 64 channels and tiles of 64 tokens (one chunk), 8 tokens a warp. A warp's lanes
// scan their 8 tokens from zero and leave the run's map h -> A h + S in shared memory; after one
// barrier every lane composes the maps before its own with the state that enters the tile, and
// its tokens' states are local + (product of a) x (entering state). Loads of the next tile are
// issued before the barrier.
//
// Where there are too few channels to fill the GPU, a cluster of up to 8 blocks shares a
// sequence: block k takes tiles k, k + n, ... . The blocks exchange their tiles' maps through
// distributed shared memory once a round, so the chain along time costs one cluster barrier for
// n tiles and x, r, i are still read once.
constexpr int kWarps = 8, kRows = 8;

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Store 16 bytes at the same shared-memory address in block `rank` of the cluster.
__device__ __forceinline__ void store_remote(const void* local, uint32_t rank, float4 v) {
  uint32_t addr;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(smem_u32(local)), "r"(rank));
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(v.x), "f"(v.y), "f"(v.z),
               "f"(v.w)
               : "memory");
}

// The map (A, S) of two channels, h -> A h + S.
__device__ __forceinline__ float2 apply(float4 m, float2 h) {
  return __ffma2_rn(make_float2(m.x, m.y), h, make_float2(m.z, m.w));
}

template <typename T, bool ADJ>
struct Tile {  // a lane's 8 tokens, as loaded
  RawPair<T> x[kRows], r[kRows], i[kRows];
  // Rows row0 .. row0 + 7 of a sequence of len rows; rows past its end hold the state.
  __device__ __forceinline__ void load(const T* xp, const T* rp, const T* ip, const Args& p, int row0, int len,
                                       const Lane<ADJ>& ln) {
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      if (ln.on0 && row0 + k < len) {
        load_pair<T, ADJ>(r[k], rp + (long long)(row0 + k) * p.rt, ln.on1);
        load_pair<T, ADJ>(i[k], ip + (long long)(row0 + k) * p.it, ln.on1);
        load_pair<T, ADJ>(x[k], xp + (long long)(row0 + k) * p.xt, ln.on1);
      } else {
        r[k].hold();
        i[k].zero();
        x[k].zero();
      }
    }
  }
};

template <typename T, bool ADJ>
__global__ void __launch_bounds__(32 * kWarps) scan_tiles(const Args p) {
  __shared__ float4 maps[2][kWarps][32];
  __shared__ float4 tiles[2][8][32];  // the cluster's blocks
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Lane<ADJ> ln(blockIdx.y * 64, p.D);
  const int c = ln.c0, n = blockIdx.z;
  const int nblk = cluster_size(), rank = cluster_rank();
  T* y = static_cast<T*>(p.y) + c;
  if (n == p.nseq) {  // rows of no sequence, a row per warp of the cluster
    const int w = rank * kWarps + warp;
    for (long long t = rest_row(p, 0); t < p.T; t = rest_row(p, t + 1))
      if (t % (nblk * kWarps) == w && ln.on0) store_pair<T, ADJ>(y + t * p.D, f2(0.f), ln.on1);
    return;
  }
  const Seq q = sequence(p, n);
  const T* x = static_cast<const T*>(p.x) + q.batch * p.xb + q.lo * p.xt + c;
  const T* r = static_cast<const T*>(p.r) + q.batch * p.rb + q.lo * p.rt + c;
  const T* i = static_cast<const T*>(p.i) + q.batch * p.ib + q.lo * p.it + c;
  y += (q.batch * p.T + q.lo) * p.D;
  const float2 decay = limit_decay(ln.load(p.decay + c));
  float2 carry = p.h0 != nullptr ? ln.load(p.h0 + (long long)n * p.D + c) : f2(0.f);
  const int ntiles = (q.len + kChunk - 1) / kChunk;
  const int rounds = (ntiles + nblk - 1) / nblk;
  if (nblk > 1) cluster_barrier();  // every block of the cluster runs before one writes to another
  Tile<T, ADJ> in;
  in.load(x, r, i, p, rank * kChunk + warp * kRows, q.len, ln);
  for (int round = 0; round < rounds; ++round) {
    const int tile = round * nblk + rank, row0 = tile * kChunk + warp * kRows, par = round & 1;
    float2 A[kRows], S[kRows];
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      float2 a, b;
      token_pair<T>(in.x[k].get(), in.r[k].get(), in.i[k].get(), decay, a, b);
      A[k] = k == 0 ? a : __fmul2_rn(a, A[k - 1]);
      S[k] = k == 0 ? b : __ffma2_rn(a, S[k - 1], b);
    }
    in.load(x, r, i, p, row0 + nblk * kChunk, q.len, ln);
    maps[par][warp][lane] = make_float4(A[kRows - 1].x, A[kRows - 1].y, S[kRows - 1].x, S[kRows - 1].y);
    __syncthreads();
    float2 h = carry;
    if (nblk > 1) {
      if (warp == 0) {
        float2 ta = f2(1.f), ts = f2(0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float4 m = maps[par][w][lane];
          ta = __fmul2_rn(ta, make_float2(m.x, m.y));
          ts = apply(m, ts);
        }
        for (int b = 0; b < nblk; ++b) store_remote(&tiles[par][rank][lane], b, make_float4(ta.x, ta.y, ts.x, ts.y));
      }
      cluster_barrier();
      for (int b = 0; b < nblk; ++b) {
        if (b == rank) h = carry;
        carry = apply(tiles[par][b][lane], carry);
      }
    }
    if (p.states != nullptr && warp == 0 && tile < ntiles) ln.store(p.states + (q.slot + tile) * p.D + c, h);
    float2 hin = h;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w == warp) hin = h;
      h = apply(maps[par][w][lane], h);
    }
    if (nblk == 1) carry = h;
    if (ln.on0) {
#pragma unroll
      for (int k = 0; k < kRows; ++k)
        if (row0 + k < q.len)
          store_pair<T, ADJ>(y + (long long)(row0 + k) * p.D, __ffma2_rn(A[k], hin, S[k]), ln.on1);
    }
  }
  if (p.final_state != nullptr && rank == 0 && warp == 0) ln.store(p.final_state + (long long)n * p.D + c, carry);
}

// One thread per channel, one token after another.
struct Gate {
  float s, L, a, p, m2;
};
template <typename T>
__device__ __forceinline__ Gate gate(float r, float i, float decay) {
  Gate g;
  sigmoids<T>(r, i, g.s, g.p);
  g.L = r < kHoldBelow ? 0.f : fminf(decay, kMaxDecay) * g.s;
  float2 a, m2;
  decay_pair(f2(g.L), a, m2);
  g.a = a.x;
  g.m2 = m2.x;
  return g;
}
template <typename T>
__global__ void __launch_bounds__(128) scan_bwd_direct(const Args p) {
  const int c = blockIdx.x * 128 + threadIdx.x;
  const int n = blockIdx.y;
  if (c >= p.D) return;
  T *dx = static_cast<T*>(p.dx), *dr = static_cast<T*>(p.dr), *di = static_cast<T*>(p.di);
  if (n == p.nseq) {
    for (long long t = rest_row(p, 0); t < p.T; t = rest_row(p, t + 1))
      dx[t * p.D + c] = dr[t * p.D + c] = di[t * p.D + c] = from_f32<T>(0.f);
    return;
  }
  const Seq q = sequence(p, n);
  const T* x = static_cast<const T*>(p.x) + q.batch * p.xb + c;
  const T* r = static_cast<const T*>(p.r) + q.batch * p.rb + c;
  const T* i = static_cast<const T*>(p.i) + q.batch * p.ib + c;
  const T* dy = static_cast<const T*>(p.dy) + q.batch * p.gb + c;
  const long long o = q.batch * p.T * p.D + c;
  const float decay = p.decay[c];
  float dh = p.dfinal != nullptr ? p.dfinal[(long long)n * p.D + c] : 0.f;  // a_{t+1} dh_{t+1}
  float ddecay = 0.f;
  float prev[kChunk];
  for (int ch = (q.len + kChunk - 1) / kChunk - 1; ch >= 0; --ch) {
    const int rows = min(kChunk, q.len - ch * kChunk);
    float h = p.states[(q.slot + ch) * p.D + c];
    for (int k = 0; k < rows; ++k) {
      const long long t = q.lo + ch * kChunk + k;
      prev[k] = h;
      const Gate g = gate<T>(to_f32<T>(r[t * p.rt]), to_f32<T>(i[t * p.it]), decay);
      const float b = g.L != 0.f ? sqrtf(g.m2) * g.p * to_f32<T>(x[t * p.xt]) : 0.f;
      h = fmaf(g.a, h, b);
    }
    for (int k = rows - 1; k >= 0; --k) {
      const long long t = q.lo + ch * kChunk + k;
      Gate g = gate<T>(to_f32<T>(r[t * p.rt]), to_f32<T>(i[t * p.it]), decay);
      const bool held = g.L == 0.f;
      const float xv = held ? 0.f : to_f32<T>(x[t * p.xt]);
      const float pv = held ? 0.f : g.p;
      const float im = held ? 0.f : rsqrtf(g.m2);
      const float m = g.m2 * im;
      dh += to_f32<T>(dy[t * p.gt]);
      const float dLv = dh * fmaf(g.a * g.a * im, pv * xv, -g.a * prev[k]);
      dx[o + t * p.D] = from_f32<T>(dh * m * pv);
      di[o + t * p.D] = from_f32<T>(dh * m * xv * pv * (1.f - pv));
      dr[o + t * p.D] = from_f32<T>(dLv * g.L * (1.f - g.s));
      ddecay = fmaf(dLv, g.s, ddecay);
      dh *= g.a;
    }
  }
  p.ddecay_part[(long long)n * p.D + c] = ddecay;
  if (p.dh0 != nullptr) p.dh0[(long long)n * p.D + c] = dh;
}

struct StoreColumn {
  float* out;
  __device__ void operator()(int c, float v) const { out[c] = v; }
};

// Whether two neighbouring channels can be read as one access everywhere.
bool pairs_fit(int elem, int D, std::initializer_list<const void*> ptrs, std::initializer_list<long long> strides) {
  uintptr_t bits = (uintptr_t)D;
  for (long long s : strides) bits |= (uintptr_t)s;
  bits *= elem;
  for (const void* q : ptrs) bits |= reinterpret_cast<uintptr_t>(q);
  return (bits & (2 * elem - 1)) == 0;
}

// Up to this many tokens a lane's serial walk beats the tiles.
constexpr int kDirectTokens = 16;

// Blocks that share a sequence: doubled while the grid has fewer than four blocks an SM and a
// block still has two tiles of an average sequence.
int cluster_blocks(const Args& p) {
  const long long base = (long long)p.nseq * ((p.D + 63) / 64);
  const long long tiles = ((p.cu != nullptr ? (p.T + p.nseq - 1) / p.nseq : p.T) + kChunk - 1) / kChunk;
  int n = 1;
  while (n < 8 && base * n < 4ll * sm_count() && tiles >= 4 * n) n *= 2;
  return n;
}

template <typename T, bool ADJ>
int launch_fwd(const Args& p, int seqs, cudaStream_t st) {
  if (p.T <= kDirectTokens) {
    const dim3 grid((p.D + 2 * kDirectThreads - 1) / (2 * kDirectThreads), seqs);
    scan_direct<T, ADJ><<<grid, kDirectThreads, 0, st>>>(p);
    return check_launch();
  }
  const int n = cluster_blocks(p);
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3(n, (p.D + 63) / 64, seqs);
  cfg.blockDim = dim3(32 * kWarps);
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = n;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, scan_tiles<T, ADJ>, p) != cudaSuccess) {
    cudaGetLastError();
    return THM_ERR_CUDA;
  }
  return check_launch();
}

int check_sizes(int B, int T, int D, int nseq, const int* cu, int dtype) {
  if (B < 0 || T < 0 || D < 0 || nseq < 0) return THM_ERR_INVALID;
  if (dtype != THM_F32 && dtype != THM_BF16) return THM_ERR_INVALID;
  if (cu != nullptr ? B != 1 : nseq != B) return THM_ERR_INVALID;
  if (nseq >= 65535) return THM_ERR_UNSUPPORTED;
  return THM_OK;
}

}  // namespace gscan
}  // namespace thm

extern "C" int thm_gated_scan_fwd(const void* x, const void* r, const void* i, const float* decay, const float* h0,
                                  const int* cu_seqlens, void* y, float* final_state, float* states,
                                  long long x_bs, long long x_ts, long long r_bs, long long r_ts, long long i_bs,
                                  long long i_ts, int B, int T, int D, int nseq, int zero_rest, int dtype,
                                  thm_stream_t stream) {
  using namespace thm;
  const int bad = gscan::check_sizes(B, T, D, nseq, cu_seqlens, dtype);
  if (bad != THM_OK) return bad;
  if (D == 0 || nseq == 0) return THM_OK;
  if (!decay || (T > 0 && (!x || !r || !i || !y))) return THM_ERR_INVALID;
  gscan::Args p{};
  p.x = x; p.r = r; p.i = i; p.decay = decay; p.h0 = h0; p.cu = cu_seqlens;
  p.y = y; p.final_state = final_state; p.states = states;
  p.xb = x_bs; p.xt = x_ts; p.rb = r_bs; p.rt = r_ts; p.ib = i_bs; p.it = i_ts;
  p.T = T; p.D = D; p.nseq = nseq;
  const int seqs = nseq + (cu_seqlens != nullptr && zero_rest);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int elem = dtype == THM_BF16 ? 2 : 4;
  const bool adj = gscan::pairs_fit(elem, D, {x, r, i, y}, {x_bs, x_ts, r_bs, r_ts, i_bs, i_ts});
  if (dtype == THM_BF16)
    return adj ? gscan::launch_fwd<__nv_bfloat16, true>(p, seqs, st) : gscan::launch_fwd<__nv_bfloat16, false>(p, seqs, st);
  return adj ? gscan::launch_fwd<float, true>(p, seqs, st) : gscan::launch_fwd<float, false>(p, seqs, st);
}

extern "C" int thm_gated_scan_bwd(const void* x, const void* r, const void* i, const float* decay,
                                  const float* states, const void* dy, const float* dfinal, const int* cu_seqlens,
                                  void* dx, void* dr, void* di, float* ddecay, float* dh0, float* workspace,
                                  long long x_bs, long long x_ts, long long r_bs, long long r_ts, long long i_bs,
                                  long long i_ts, long long dy_bs, long long dy_ts, int B, int T, int D, int nseq,
                                  int zero_rest, int dtype, thm_stream_t stream) {
  using namespace thm;
  const int bad = gscan::check_sizes(B, T, D, nseq, cu_seqlens, dtype);
  if (bad != THM_OK) return bad;
  if (D == 0) return THM_OK;
  if (!decay || !ddecay || (nseq > 0 && !workspace)) return THM_ERR_INVALID;
  if (nseq > 0 && T > 0 && (!x || !r || !i || !dy || !states || !dx || !dr || !di)) return THM_ERR_INVALID;
  gscan::Args p{};
  p.x = x; p.r = r; p.i = i; p.dy = dy; p.decay = decay; p.dfinal = dfinal; p.cu = cu_seqlens;
  p.states = const_cast<float*>(states);
  p.dx = dx; p.dr = dr; p.di = di; p.ddecay_part = workspace; p.dh0 = dh0;
  p.xb = x_bs; p.xt = x_ts; p.rb = r_bs; p.rt = r_ts; p.ib = i_bs; p.it = i_ts; p.gb = dy_bs; p.gt = dy_ts;
  p.T = T; p.D = D; p.nseq = nseq;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (nseq > 0) {
    const dim3 grid((D + 127) / 128, nseq + (cu_seqlens != nullptr && zero_rest));
    if (dtype == THM_BF16)
      gscan::scan_bwd_direct<__nv_bfloat16><<<grid, 128, 0, st>>>(p);
    else
      gscan::scan_bwd_direct<float><<<grid, 128, 0, st>>>(p);
    const int e = check_launch();
    if (e != THM_OK) return e;
  }
  sum_parts(workspace, nseq, D, gscan::StoreColumn{ddecay}, st);
  return check_launch();
}
