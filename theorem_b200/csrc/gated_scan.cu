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
#include <cmath>
#include <initializer_list>

#include "host_util.h"
#include "rowops.cuh"

THM_DEFINE_STATUS(g_status_scan)

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
  int T, D, nseq;
  int cols;          // runs of 64 channels of a sequence
  int first, count;  // of the launch: its first (sequence, run of channels) and how many
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
// A lane works on two neighbouring channels at a time, in packed fp32x2 arithmetic.
template <typename T>
struct RawPair;
template <>
struct RawPair<__nv_bfloat16> {
  uint32_t v;
  __device__ __forceinline__ float2 get() const {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  }
  static __device__ __forceinline__ RawPair of(float2 f) { return {pack_bf16x2(f.x, f.y)}; }
};
template <>
struct RawPair<float> {
  float2 v;
  __device__ __forceinline__ float2 get() const { return v; }
  static __device__ __forceinline__ RawPair of(float2 f) { return {f}; }
};

// The pair at p as one access (PAIRED: addresses and strides allow it) or as two.
template <typename T, bool PAIRED>
__device__ __forceinline__ RawPair<T> load_pair(const T* p, bool two) {
  if constexpr (PAIRED) {
    return *reinterpret_cast<const RawPair<T>*>(p);
  } else if constexpr (sizeof(T) == 2) {
    const uint16_t* u = reinterpret_cast<const uint16_t*>(p);
    return {u[0] | (two ? (uint32_t)u[1] << 16 : 0u)};
  } else {
    return {make_float2(p[0], two ? p[1] : 0.f)};
  }
}
template <typename T, bool PAIRED>
__device__ __forceinline__ void store_pair(T* p, float2 f, bool two) {
  if constexpr (PAIRED) {
    *reinterpret_cast<RawPair<T>*>(p) = RawPair<T>::of(f);
  } else {
    p[0] = from_f32<T>(f.x);
    if (two) p[1] = from_f32<T>(f.y);
  }
}

// A lane's channels c, c + 1, and which of them there are.
struct Lane {
  int c;
  bool on, two;
  __device__ __forceinline__ Lane(int base, int D) {
    c = base + 2 * (threadIdx.x & 31);
    on = c < D;
    two = c + 1 < D;
  }
  __device__ __forceinline__ float2 load(const float* p) const {  // p at channel 0
    return make_float2(on ? p[c] : 0.f, two ? p[c + 1] : 0.f);
  }
  __device__ __forceinline__ void store(float* p, float2 v) const {
    if (on) p[c] = v.x;
    if (two) p[c + 1] = v.y;
  }
};

__device__ __forceinline__ float2 f2(float v) { return make_float2(v, v); }

__device__ __forceinline__ float sqrt_approx(float x) {
  float r;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rsqrt_approx(float x) {
  float r;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float min_nan(float a, float b) {  // NaN when either is
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Below this gate logit a token holds the state: sigmoid(r) < 2^-62 changes no fp32 state of
// the size of x by even 1e-2 of a rounding step, and x and i may hold anything.
constexpr float kHoldBelow = -43.f;
// e^-87 is the smallest decay of one token that stays a normal number: L is limited to it.
constexpr float kMaxL = 87.f;

// A token of two channels is computed in one of two ways. PLAIN tokens have 1e-6 <= decay <= 1
// on every channel of the warp and no held token among the warp's 16 (both checked once a tile,
// which costs a bf16 minimum a row): no range reduction, no selects, a third fewer
// instructions. Others take the general way.
constexpr float kPlainDecayMin = 1e-6f, kPlainDecayMax = 1.f;

// s = sigmoid(r), p = sigmoid(i). For bf16 inputs the two share a reciprocal,
// 1 / ((1 + e^-r)(1 + e^-i)): three operations of the special-function unit, which runs at an
// eighth of the FMA rate, instead of four. Both exponentials are kept under 2^62, so the product
// is finite. A held token has s = 0, and its i (which may be NaN) is taken as 0 so that it does
// not reach s.
template <typename T, bool PLAIN>
__device__ __forceinline__ void sigmoids(float2 r, float2 i, float2& s, float2& p) {
  if constexpr (!PLAIN) i = make_float2(r.x < kHoldBelow ? 0.f : i.x, r.y < kHoldBelow ? 0.f : i.y);
  if constexpr (sizeof(T) == 2) {
    float2 nr = __fmul2_rn(r, f2(-1.4426950408889634f));
    if constexpr (!PLAIN) nr = make_float2(min_nan(nr.x, 62.5f), min_nan(nr.y, 62.5f));
    const float2 ni = __fmul2_rn(i, f2(-1.4426950408889634f));
    const float2 A = __fadd2_rn(make_float2(ex2_approx(nr.x), ex2_approx(nr.y)), f2(1.f));
    const float2 B =
        __fadd2_rn(make_float2(ex2_approx(min_nan(ni.x, 62.f)), ex2_approx(min_nan(ni.y, 62.f))), f2(1.f));
    const float2 d = __fmul2_rn(A, B);
    const float2 q = make_float2(rcp_approx(d.x), rcp_approx(d.y));
    s = __fmul2_rn(q, B);
    p = __fmul2_rn(q, A);
  } else {
    s = make_float2(sigmoid<T>(r.x), sigmoid<T>(r.y));
    p = make_float2(sigmoid<T>(i.x), sigmoid<T>(i.y));
  }
  if constexpr (!PLAIN) s = make_float2(r.x < kHoldBelow ? 0.f : s.x, r.y < kHoldBelow ? 0.f : s.y);
}

// a = e^-L and t = a - 1 from nL = -L, L >= 0 (PLAIN: L <= 1), both to fp32 accuracy and
// without the special-function unit, whose exponential is off by up to 2^-22, always to the same
// side: in a product over a memory of hundreds of tokens that adds up. e^f - 1 is a polynomial
// fitted by reweighted least squares, over -1 <= f <= 0 (largest relative error 2.7e-9) or, after
// nL = k ln 2 + f, over |f| <= ln 2 / 2 (1.3e-8). t = 2^k (e^f - 1) + (2^k - 1) does not cancel,
// and so neither does m^2 = 1 - a^2 = -t (2 + t).
template <bool PLAIN>
__device__ __forceinline__ void decay_pair(float2 nL, float2& a, float2& t) {
  if constexpr (PLAIN) {
    float2 c = __ffma2_rn(nL, f2(0.000129130927f), f2(0.00130112648f));
    c = __ffma2_rn(nL, c, f2(0.00827620872f));
    c = __ffma2_rn(nL, c, f2(0.0416474683f));
    c = __ffma2_rn(nL, c, f2(0.166663656f));
    c = __ffma2_rn(nL, c, f2(0.499999841f));
    t = __ffma2_rn(__fmul2_rn(nL, nL), c, nL);
    a = __fadd2_rn(t, f2(1.f));
  } else {
    nL = make_float2(max_nan(nL.x, -kMaxL), max_nan(nL.y, -kMaxL));
    constexpr float kMagic = 12582912.f;  // 1.5 2^23: adding it rounds to an integer in the low bits
    const float2 km = __ffma2_rn(nL, f2(1.4426950408889634f), f2(kMagic));
    const float2 k = __fadd2_rn(km, f2(-kMagic));
    const float2 scale = make_float2(__int_as_float((__float_as_int(km.x) << 23) + 0x3f800000),
                                     __int_as_float((__float_as_int(km.y) << 23) + 0x3f800000));
    const float2 f = __ffma2_rn(k, f2(-1.42860677e-6f), __ffma2_rn(k, f2(-0.693145752f), nL));
    float2 c = __ffma2_rn(f, f2(0.00138825101f), f2(0.00836658047f));
    c = __ffma2_rn(f, c, f2(0.0416672018f));
    c = __ffma2_rn(f, c, f2(0.166665432f));
    c = __ffma2_rn(f, c, f2(0.499999981f));
    const float2 q = __ffma2_rn(__fmul2_rn(f, f), c, f);
    a = __ffma2_rn(scale, q, scale);
    t = __ffma2_rn(scale, q, __fadd2_rn(scale, f2(-1.f)));
  }
}
__device__ __forceinline__ float2 m2_of(float2 t) { return __fmul2_rn(t, __ffma2_rn(t, f2(-1.f), f2(-2.f))); }

// One token of two channels: h -> a h + b. `ndecay` is -decay.
template <typename T, bool PLAIN>
__device__ __forceinline__ void token_pair(float2 x, float2 r, float2 i, float2 ndecay, float2& a, float2& b) {
  float2 s, p, t;
  sigmoids<T, PLAIN>(r, i, s, p);
  decay_pair<PLAIN>(__fmul2_rn(ndecay, s), a, t);
  const float2 m2 = m2_of(t);
  const float2 m = make_float2(sqrt_approx(m2.x), sqrt_approx(m2.y));
  b = __fmul2_rn(__fmul2_rn(m, p), x);
  if constexpr (!PLAIN) b = make_float2(s.x == 0.f ? 0.f : b.x, s.y == 0.f ? 0.f : b.y);
}

// The smaller of two pairs, elementwise; a NaN gives way to the other.
template <typename T>
__device__ __forceinline__ RawPair<T> min_pair(RawPair<T> u, RawPair<T> v) {
  if constexpr (sizeof(T) == 2) {
    const __nv_bfloat162 m =
        __hmin2(*reinterpret_cast<const __nv_bfloat162*>(&u.v), *reinterpret_cast<const __nv_bfloat162*>(&v.v));
    return {*reinterpret_cast<const uint32_t*>(&m)};
  } else {
    return {make_float2(fminf(u.v.x, v.v.x), fminf(u.v.y, v.v.y))};
  }
}
template <typename T, int N>
__device__ __forceinline__ RawPair<T> min_rows(const RawPair<T> (&r)[N]) {
  RawPair<T> m[N / 2];
#pragma unroll
  for (int k = 0; k < N / 2; ++k) m[k] = min_pair(r[k], r[k + N / 2]);
  if constexpr (N == 2)
    return m[0];
  else
    return min_rows<T, N / 2>(m);
}
template <typename T>
__device__ __forceinline__ bool any_held(RawPair<T> m) {
  const float2 f = m.get();
  return __any_sync(0xffffffffu, f.x < kHoldBelow || f.y < kHoldBelow);
}

// -decay of a lane's channels; channels that it does not have do not keep its warp from PLAIN.
__device__ __forceinline__ float2 neg_decay(const Lane& ln, const float* decay) {
  const float2 d = ln.load(decay);
  return make_float2(ln.on ? -d.x : -1.f, ln.two ? -d.y : -1.f);
}
__device__ __forceinline__ bool plain_decays(float2 nd) {
  return __all_sync(0xffffffffu, -nd.x >= kPlainDecayMin && -nd.x <= kPlainDecayMax && -nd.y >= kPlainDecayMin &&
                                     -nd.y <= kPlainDecayMax);
}

// --------------------------------------------------------------------------- forward, few tokens
// A lane walks its two channels token by token, a warp 64 channels of a sequence: single-token
// steps and short runs, where there is nothing to split along time and a launch is all the
// latency there is.
constexpr int kDirectThreads = 64;

// BATCH tokens' loads are in flight together: 4 for runs (a token 0.15 us instead of 0.35), 1 for
// fewer, in fewer registers (B256 T1: 4.5 us instead of 5.5).
template <typename T, bool PAIRED, int BATCH>
__global__ void __launch_bounds__(kDirectThreads) scan_direct(const Args p) {
  const int chain = (blockIdx.x * kDirectThreads + threadIdx.x) >> 5, n = chain / p.cols;
  const Lane ln(chain % p.cols * 64, p.D);
  if (!ln.on || chain >= p.count) return;
  T* y = static_cast<T*>(p.y) + ln.c;
  if (n == p.nseq) {  // rows of no sequence
    for (long long t = rest_row(p, 0); t < p.T; t = rest_row(p, t + 1))
      store_pair<T, PAIRED>(y + t * p.D, f2(0.f), ln.two);
    return;
  }
  const Seq q = sequence(p, n);
  const T* x = static_cast<const T*>(p.x) + q.batch * p.xb + q.lo * p.xt + ln.c;
  const T* r = static_cast<const T*>(p.r) + q.batch * p.rb + q.lo * p.rt + ln.c;
  const T* i = static_cast<const T*>(p.i) + q.batch * p.ib + q.lo * p.it + ln.c;
  y += (q.batch * p.T + q.lo) * p.D;
  const float2 ndecay = neg_decay(ln, p.decay);
  float2 h = p.h0 != nullptr ? ln.load(p.h0 + (long long)n * p.D) : f2(0.f);
  auto token = [&](int k, RawPair<T> xv, RawPair<T> rv, RawPair<T> iv) {
    if (p.states != nullptr && k % kChunk == 0) ln.store(p.states + (q.slot + k / kChunk) * p.D, h);
    float2 a, b;
    token_pair<T, false>(xv.get(), rv.get(), iv.get(), ndecay, a, b);
    h = __ffma2_rn(a, h, b);
    store_pair<T, PAIRED>(y + (long long)k * p.D, h, ln.two);
  };
  int k = 0;
  for (; BATCH > 1 && k + BATCH <= q.len; k += BATCH) {
    RawPair<T> xv[BATCH], rv[BATCH], iv[BATCH];
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      rv[u] = load_pair<T, PAIRED>(r + (k + u) * p.rt, ln.two);
      iv[u] = load_pair<T, PAIRED>(i + (k + u) * p.it, ln.two);
      xv[u] = load_pair<T, PAIRED>(x + (k + u) * p.xt, ln.two);
    }
#pragma unroll
    for (int u = 0; u < BATCH; ++u) token(k + u, xv[u], rv[u], iv[u]);
  }
  for (; k < q.len; ++k)
    token(k, load_pair<T, PAIRED>(x + k * p.xt, ln.two), load_pair<T, PAIRED>(r + k * p.rt, ln.two),
          load_pair<T, PAIRED>(i + k * p.it, ln.two));
  if (p.final_state != nullptr) ln.store(p.final_state + (long long)n * p.D, h);
}

// --------------------------------------------------------------------------- tiles
// A block takes 64 channels and tiles of 64 tokens (one chunk), 16 tokens a warp, two channels
// a lane. A lane scans its 16 tokens from zero and leaves the run's map h -> A h + S in shared
// memory; after one barrier every lane composes the maps before its own with the state that
// enters the tile, and its tokens' states are local + (product of a) x (entering state). Long
// runs a lane make the arithmetic independent work for its own latencies and the maps few: 16
// tokens beat 8 with twice the warps on an SM (forward B16 T8192 D2048 389 against 399 us, B1
// T131072 519 against 573, backward B1 T65536 469 against 535), 4 (606 us) and 32 (408 us).
//
// Tiles come by TMA, so loading costs the warps no addresses; the barrier that the maps need
// also says that a tile has been read, and its stage is refilled there. Where addresses or
// strides are no multiples of 16 bytes (TMA false), the lanes fill their own slots with plain
// loads.
//
// B16 T8192 D2048 bf16 takes 389 us, 5.5 TB/s (0.84 of a copy): between HBM, the special-function
// unit (63 % busy, four operations an element) and the latencies of 12 warps an SM.
//
// Where there are too few channels to fill the GPU, a cluster of up to 16 blocks shares a
// sequence: block k takes tiles k, k + n, ... . Each round the blocks send their tiles' maps to
// one another's shared memory, counted in by an mbarrier, so the chain along time costs one
// such exchange for n tiles, and x, r, i are still read once.
constexpr int kWarps = 4, kRows = 16, kCols = 64;
static_assert(kWarps * kRows == kChunk, "a tile is a chunk");

struct Maps {  // of x, r, i, dy, where TMA carries the tiles
  CUtensorMap in[4];
};

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

// The map (A, S) of two channels, h -> A h + S.
__device__ __forceinline__ float2 apply(float4 m, float2 h) {
  return __ffma2_rn(make_float2(m.x, m.y), h, make_float2(m.z, m.w));
}

// What the blocks of a cluster tell each other about a round: a map each, DEPTH rounds deep.
// A block that receives round j right after sending it sends round j + 2 only after it
// has all of round j + 1, which each block sends after a block barrier that follows its reads of
// round j: 2 are enough. One that receives a round behind sends round j + 2 once it has
// round j, which a block sends before it reads round j - 1: 4 rounds are in use.
template <int DEPTH>
struct Exchange {
  float4* slots;  // [DEPTH][nblk][32], behind the stages
  uint64_t* bar;
  int nblk, rank;
  bool ok;
  static constexpr int bytes(int n) { return n > 1 ? DEPTH * n * 32 * (int)sizeof(float4) : 0; }
  __device__ __forceinline__ Exchange(void* s, uint64_t* b, int n, int r)
      : slots(static_cast<float4*>(s)), bar(b), nblk(n), rank(r), ok(true) {
    if (nblk > 1) {
      if (threadIdx.x == 0) {
        for (int k = 0; k < DEPTH; ++k) mbar_init(&bar[k], 1);
        fence_mbar_init();
      }
      cluster_barrier();  // every block of the cluster runs, its barriers set up, before one sends
    }
  }
  // One warp: send this block's map of round j to every block.
  __device__ __forceinline__ void send(int j, float4 m) {
    const int lane = threadIdx.x & 31, par = j % DEPTH;
    if (lane == 0) mbar_arrive_expect_tx(&bar[par], nblk * 32 * (int)sizeof(float4));
    const uint32_t slot = smem_u32(slots + (par * nblk + rank) * 32 + lane), b = smem_u32(&bar[par]);
    for (int k = 0; k < nblk; ++k) {
      uint32_t rs, rb;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(rs) : "r"(slot), "r"(k));
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(rb) : "r"(b), "r"(k));
      asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(
                       rs),
                   "f"(m.x), "f"(m.y), "f"(m.z), "f"(m.w), "r"(rb)
                   : "memory");
    }
  }
  // All threads: the state that enters this block's tile of round j, and in `carry` the one
  // that enters the next round.
  __device__ __forceinline__ float2 receive(int j, float2& carry, unsigned* status) {
    const int lane = threadIdx.x & 31, par = j % DEPTH;
    if (ok) ok = mbar_wait(&bar[par], (j / DEPTH) & 1, status);
    float2 mine = carry;
    for (int k = 0; k < nblk; ++k) {
      if (k == rank) mine = carry;
      carry = apply(slots[(par * nblk + k) * 32 + lane], carry);
    }
    return mine;
  }
};

// The ring of stages that a block's tiles pass through: NIN input tiles a stage.
template <typename T, int NIN, int NSTAGE>
struct Ring {
  static constexpr int kTile = kChunk * kCols * (int)sizeof(T);
  static constexpr int kStage = NIN * kTile;
  static constexpr int kBytes = NSTAGE * kStage;
  uint8_t* base;
  uint64_t* full;
  int asked, failed;  // steps asked for (one thread), and the first whose wait ran out
  bool ok;

  __device__ __forceinline__ Ring(uint8_t* b, uint64_t* f) : base(b), full(f), asked(0), failed(0), ok(true) {
    if (threadIdx.x == 0) {
      for (int k = 0; k < NSTAGE; ++k) mbar_init(&full[k], 1);
      fence_mbar_init();
    }
    __syncthreads();
  }
  __device__ __forceinline__ uint8_t* slot(int j, int in) const { return base + (j % NSTAGE) * kStage + in * kTile; }
  // One thread: ask for the tiles of step j, rows from `row` of batch entry `batch`.
  __device__ __forceinline__ void ask(const CUtensorMap* in, int j, int col, int row, int batch) {
    if (!ok) return;
    asked = j + 1;
    uint64_t* bar = &full[j % NSTAGE];
    mbar_arrive_expect_tx(bar, kStage);
#pragma unroll
    for (int k = 0; k < NIN; ++k) tma_load_3d(slot(j, k), &in[k], bar, col, row, batch);
  }
  // All threads: the tiles of step j are there. After a wait that ran out no further one is
  // entered and nothing more is asked for: the kernel ends, and the device status says why.
  __device__ __forceinline__ void wait(int j, unsigned* status) {
    if (!ok) return;
    ok = mbar_wait(&full[j % NSTAGE], (j / NSTAGE) & 1, status);
    failed = j;
  }
  // The thread that asked, before it leaves: after a wait that ran out, once more for what is still
  // on its way into this block's memory.
  __device__ __forceinline__ void drain(unsigned* status) {
    for (int j = failed; !ok && j < asked; ++j) mbar_wait(&full[j % NSTAGE], (j / NSTAGE) & 1, status);
  }
};

template <typename T>
__device__ __forceinline__ RawPair<T> get_pair(const uint8_t* tile, int k) {
  return *reinterpret_cast<const RawPair<T>*>(tile + k * kCols * sizeof(T));
}
template <typename T>
__device__ __forceinline__ void put_pair(uint8_t* tile, int k, float2 f) {
  *reinterpret_cast<RawPair<T>*>(tile + k * kCols * sizeof(T)) = RawPair<T>::of(f);
}
// A lane's first `rows` rows of a tensor into its slots, without TMA. Loads without conditions, so
// that all are in flight at once: rows past the last repeat it (the caller overwrites them), and a
// second channel that is not there repeats the first.
template <typename T>
__device__ __forceinline__ void fill(uint8_t* tile, const void* t, long long first, long long stride, int rows, bool two) {
  if (rows == 0) return;
  const T* q = static_cast<const T*>(t) + first;
  const int next = two ? 1 : 0;
  T v[kRows][2];
#pragma unroll
  for (int k = 0; k < kRows; ++k) {
    const T* row = q + min(k, rows - 1) * stride;
    v[k][0] = row[0];
    v[k][1] = row[next];
  }
#pragma unroll
  for (int k = 0; k < kRows; ++k) put_pair<T>(tile, k, make_float2(to_f32<T>(v[k][0]), to_f32<T>(v[k][1])));
}

// Stages, and resident blocks an SM: for bf16 three of 153 registers a thread forward (four of 128
// were slower: 416 against 389 us), two of 240 in a chain of blocks, which keeps two tiles in
// registers, and backward; for fp32 shared memory holds two, without the room that finishing a
// round behind takes.
template <typename T, bool CHAIN>
struct Fwd {
  static constexpr int kStages = 2, kPerSm = sizeof(T) == 2 && !CHAIN ? 3 : 2;
  static constexpr bool kBehind = CHAIN && sizeof(T) == 2;  // a tile is finished a round behind
  static constexpr int kDepth = kBehind ? 4 : 2;
  using R = Ring<T, 3, kStages>;
};
template <typename T>
struct Bwd {
  static constexpr int kStages = sizeof(T) == 2 ? 3 : 1, kPerSm = 2;
  using R = Ring<T, 4, kStages>;
};

// CHAIN: blocks in clusters. A round's exchange takes as long as half a tile's arithmetic, so for
// bf16 a block scans its next tile before it receives the last one's entering state, two tiles in
// registers (B1 T131072 D2048, with 8 tokens a warp: 618 -> 578 us).
template <typename T, bool TMA, bool CHAIN>
__global__ void __launch_bounds__(32 * kWarps, Fwd<T, CHAIN>::kPerSm)
    scan_tiles(const __grid_constant__ Args p, const __grid_constant__ Maps tm) {
  constexpr bool BEHIND = Fwd<T, CHAIN>::kBehind;
  constexpr int NS = Fwd<T, CHAIN>::kStages, NM = BEHIND ? 3 : 2, DEPTH = Fwd<T, CHAIN>::kDepth;
  extern __shared__ __align__(128) uint8_t stages[];
  __shared__ __align__(16) float4 maps[NM][kWarps][32];
  __shared__ __align__(8) uint64_t full[NS], xbar[DEPTH];
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int nblk = CHAIN ? cluster_size() : 1, rank = CHAIN ? cluster_rank() : 0;
  const int chain = p.first + blockIdx.x / nblk, n = chain / p.cols, col = chain % p.cols * kCols;
  const Lane ln(col, p.D);
  T* y = static_cast<T*>(p.y) + ln.c;
  if (n == p.nseq) {  // rows of no sequence, in turn over the cluster's warps
    const int w = rank * kWarps + warp;
    for (long long t = rest_row(p, 0); t < p.T; t = rest_row(p, t + 1))
      if (t % (nblk * kWarps) == w && ln.on) store_pair<T, false>(y + t * p.D, f2(0.f), ln.two);
    return;
  }
  typename Fwd<T, CHAIN>::R ring(stages, full);
  Exchange<DEPTH> ex(stages + Fwd<T, CHAIN>::R::kBytes, xbar, nblk, rank);
  const Seq q = sequence(p, n);
  y += (q.batch * p.T + q.lo) * p.D;
  const float2 ndecay = neg_decay(ln, p.decay);
  const bool plain = plain_decays(ndecay);
  float2 carry = p.h0 != nullptr ? ln.load(p.h0 + (long long)n * p.D) : f2(0.f);
  const int ntiles = (q.len + kChunk - 1) / kChunk;
  const int rounds = (ntiles + nblk - 1) / nblk;
  auto ask = [&](int j) {
    const int tile = j * nblk + rank;
    if (tile < ntiles) ring.ask(tm.in, j, col, q.lo + tile * kChunk, (int)q.batch);
  };
  if (TMA && threadIdx.x == 0)
    for (int j = 0; j < NS; ++j) ask(j);
  const int own = (warp * kRows * kCols + 2 * lane) * (int)sizeof(T);

  // The lane's tokens of step j from zero, their maps' last one into shared memory.
  auto scan_tile = [&](int j, float2(&A)[kRows], float2(&S)[kRows]) {
    const int tile = j * nblk + rank, row0 = tile * kChunk + warp * kRows;
    const int have = min(max(q.len - row0, 0), kRows);  // rows of the lane's 16 that there are
    uint8_t *xs = ring.slot(j, 0) + own, *rs = ring.slot(j, 1) + own, *is = ring.slot(j, 2) + own;
    if constexpr (TMA) {
      if (tile < ntiles) ring.wait(j, &g_status_scan);
    } else if (ln.on) {
      const long long t = q.lo + row0;
      fill<T>(xs, p.x, q.batch * p.xb + t * p.xt + ln.c, p.xt, have, ln.two);
      fill<T>(rs, p.r, q.batch * p.rb + t * p.rt + ln.c, p.rt, have, ln.two);
      fill<T>(is, p.i, q.batch * p.ib + t * p.it + ln.c, p.it, have, ln.two);
    }
    for (int k = have; k < kRows; ++k) {  // rows past the sequence's end hold the state
      put_pair<T>(rs, k, f2(-INFINITY));
      put_pair<T>(is, k, f2(0.f));
      put_pair<T>(xs, k, f2(0.f));
    }
    if (TMA && have < kRows) fence_proxy_async_smem();  // before TMA writes there again
    RawPair<T> r[kRows];
#pragma unroll
    for (int k = 0; k < kRows; ++k) r[k] = get_pair<T>(rs, k);
    auto scan_rows = [&](auto is_plain) {
#pragma unroll
      for (int k = 0; k < kRows; ++k) {
        float2 a, b;
        token_pair<T, decltype(is_plain)::value>(get_pair<T>(xs, k).get(), r[k].get(), get_pair<T>(is, k).get(), ndecay,
                                                 a, b);
        A[k] = k == 0 ? a : __fmul2_rn(a, A[k - 1]);
        S[k] = k == 0 ? b : __ffma2_rn(a, S[k - 1], b);
      }
    };
    if (plain && !any_held(min_rows(r)))
      scan_rows(std::true_type());
    else
      scan_rows(std::false_type());
    maps[j % NM][warp][lane] = make_float4(A[kRows - 1].x, A[kRows - 1].y, S[kRows - 1].x, S[kRows - 1].y);
  };
  // The tile of step j, entered by h, the lane's run by hin: its states.
  auto emit = [&](int j, float2 h, float2 hin, const float2(&A)[kRows], const float2(&S)[kRows]) {
    const int tile = j * nblk + rank, row0 = tile * kChunk + warp * kRows;
    const int have = min(max(q.len - row0, 0), kRows);
    if (p.states != nullptr && warp == 0 && tile < ntiles) ln.store(p.states + (q.slot + tile) * p.D, h);
    if (!ln.on) return;
    T* yr = y + (long long)row0 * p.D;
    if (have == kRows) {
#pragma unroll
      for (int k = 0; k < kRows; ++k) store_pair<T, TMA>(yr + (long long)k * p.D, __ffma2_rn(A[k], hin, S[k]), ln.two);
    } else {
#pragma unroll
      for (int k = 0; k < kRows; ++k)
        if (k < have) store_pair<T, TMA>(yr + (long long)k * p.D, __ffma2_rn(A[k], hin, S[k]), ln.two);
    }
  };
  if constexpr (!CHAIN) {
    float2 A[kRows], S[kRows];
    for (int j = 0; j < rounds; ++j) {
      scan_tile(j, A, S);
      __syncthreads();
      if (TMA && threadIdx.x == 0) ask(j + NS);
      const float2 h = carry;
      float2 hin = carry;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        if (w == warp) hin = carry;
        carry = apply(maps[j % NM][w][lane], carry);
      }
      emit(j, h, hin, A, S);
    }
  } else {
    auto finish = [&](int j, const float2(&A)[kRows], const float2(&S)[kRows]) {
      const float2 h = ex.receive(j, carry, &g_status_scan);
      float2 hin = h;
      for (int w = 0; w < warp; ++w) hin = apply(maps[j % NM][w][lane], hin);
      emit(j, h, hin, A, S);
    };
    auto scan_and_send = [&](int j, float2(&A)[kRows], float2(&S)[kRows]) {
      scan_tile(j, A, S);
      __syncthreads();
      if (TMA && threadIdx.x == 0) ask(j + NS);
      if (warp == kWarps - 1) {
        float2 ta = f2(1.f), ts = f2(0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float4 m = maps[j % NM][w][lane];
          ta = __fmul2_rn(ta, make_float2(m.x, m.y));
          ts = apply(m, ts);
        }
        ex.send(j, make_float4(ta.x, ta.y, ts.x, ts.y));
      }
    };
    float2 A0[kRows], S0[kRows];
    if constexpr (BEHIND) {
      float2 A1[kRows], S1[kRows];
      for (int j = 0; j < rounds; j += 2) {
        scan_and_send(j, A0, S0);
        if (j > 0) finish(j - 1, A1, S1);
        if (j + 1 < rounds) {
          scan_and_send(j + 1, A1, S1);
          finish(j, A0, S0);
        }
      }
      if (rounds & 1)
        finish(rounds - 1, A0, S0);
      else if (rounds > 0)
        finish(rounds - 1, A1, S1);
    } else {
      for (int j = 0; j < rounds; ++j) {
        scan_and_send(j, A0, S0);
        finish(j, A0, S0);
      }
    }
  }
  if (TMA && threadIdx.x == 0) ring.drain(&g_status_scan);
  // No block leaves while another may still send to it, and final_state may be h0: every block has
  // read that by now.
  if (CHAIN) cluster_barrier();
  if (p.final_state != nullptr && rank == 0 && warp == 0) ln.store(p.final_state + (long long)n * p.D, carry);
}

// --------------------------------------------------------------------------- backward
// The same tiles from the back. A lane keeps s, p, t = a - 1 and the injected term of its 16
// tokens; two maps a warp go through shared memory, the forward one (h, from the chunk's kept
// state) and the backward one (G_t = a_t dh_t, from the tile behind). Clusters exchange the
// backward maps only: every tile's entering state is known. x and dy are read again from the
// tile after the barrier, so a stage is refilled at the next step's barrier. B8 T4096 D2048 bf16
// takes 213 us, 4.4 TB/s (0.67 of a copy): 53 instructions per 32 elements from 8 warps an SM, and
// 256 blocks on 148 SMs.
template <typename T, bool TMA>
__global__ void __launch_bounds__(32 * kWarps, Bwd<T>::kPerSm)
    scan_bwd_tiles(const __grid_constant__ Args p, const __grid_constant__ Maps tm) {
  extern __shared__ __align__(128) uint8_t stages[];
  __shared__ __align__(16) float4 maps[2][kWarps][32];
  __shared__ __align__(16) float2 back[2][kWarps][32];
  __shared__ __align__(8) uint64_t full[Bwd<T>::kStages], xbar[2];
  constexpr int NS = Bwd<T>::kStages;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int nblk = cluster_size(), rank = cluster_rank();
  const int chain = p.first + blockIdx.x / nblk, n = chain / p.cols, col = chain % p.cols * kCols;
  const Lane ln(col, p.D);
  T *dx = static_cast<T*>(p.dx) + ln.c, *dr = static_cast<T*>(p.dr) + ln.c, *di = static_cast<T*>(p.di) + ln.c;
  if (n == p.nseq) {
    const int w = rank * kWarps + warp;
    for (long long t = rest_row(p, 0); t < p.T; t = rest_row(p, t + 1))
      if (t % (nblk * kWarps) == w && ln.on) {
        store_pair<T, false>(dx + t * p.D, f2(0.f), ln.two);
        store_pair<T, false>(dr + t * p.D, f2(0.f), ln.two);
        store_pair<T, false>(di + t * p.D, f2(0.f), ln.two);
      }
    return;
  }
  typename Bwd<T>::R ring(stages, full);
  Exchange<2> ex(stages + Bwd<T>::R::kBytes, xbar, nblk, rank);
  const Seq q = sequence(p, n);
  const long long first = (q.batch * p.T + q.lo) * p.D;
  const float2 ndecay = neg_decay(ln, p.decay);
  const bool plain = plain_decays(ndecay);
  float2 carry = p.dfinal != nullptr ? ln.load(p.dfinal + (long long)n * p.D) : f2(0.f);
  float2 ddecay = f2(0.f);
  const int ntiles = (q.len + kChunk - 1) / kChunk;
  const int rounds = (ntiles + nblk - 1) / nblk;
  auto ask = [&](int j) {
    const int tile = ntiles - 1 - (j * nblk + rank);
    if (tile >= 0) ring.ask(tm.in, j, col, q.lo + tile * kChunk, (int)q.batch);
  };
  if (TMA && threadIdx.x == 0)
    for (int j = 0; j < NS; ++j) ask(j);
  const int own = (warp * kRows * kCols + 2 * lane) * (int)sizeof(T);
  for (int j = 0; j < rounds; ++j) {
    const int tile = ntiles - 1 - (j * nblk + rank), row0 = tile * kChunk + warp * kRows, par = j & 1;
    uint8_t *xs = ring.slot(j, 0) + own, *rs = ring.slot(j, 1) + own, *is = ring.slot(j, 2) + own,
            *gs = ring.slot(j, 3) + own;
    const int have = tile < 0 ? 0 : min(max(q.len - row0, 0), kRows);
    float2 h = tile >= 0 ? ln.load(p.states + (q.slot + tile) * p.D) : f2(0.f);
    if constexpr (NS == 1) {
      if (j > 0) {  // the one stage: refilled once every warp is through with it
        __syncthreads();
        if (TMA && threadIdx.x == 0) ask(j);
      }
    }
    if constexpr (TMA) {
      if (tile >= 0) ring.wait(j, &g_status_scan);
    } else if (ln.on) {
      const long long t = q.lo + row0;
      fill<T>(xs, p.x, q.batch * p.xb + t * p.xt + ln.c, p.xt, have, ln.two);
      fill<T>(rs, p.r, q.batch * p.rb + t * p.rt + ln.c, p.rt, have, ln.two);
      fill<T>(is, p.i, q.batch * p.ib + t * p.it + ln.c, p.it, have, ln.two);
      fill<T>(gs, p.dy, q.batch * p.gb + t * p.gt + ln.c, p.gt, have, ln.two);
    }
    for (int k = have; k < kRows; ++k) {
      put_pair<T>(rs, k, f2(-INFINITY));
      put_pair<T>(is, k, f2(0.f));
      put_pair<T>(xs, k, f2(0.f));
      put_pair<T>(gs, k, f2(0.f));
    }
    if (TMA && have < kRows) fence_proxy_async_smem();
    float2 t[kRows], hp[kRows], s[kRows], pi[kRows];
    float2 A = f2(1.f), S = f2(0.f), P = f2(0.f);
    RawPair<T> r[kRows];
#pragma unroll
    for (int k = 0; k < kRows; ++k) r[k] = get_pair<T>(rs, k);
    auto scan_rows = [&](auto is_plain) {
      constexpr bool kPlain = decltype(is_plain)::value;
#pragma unroll
      for (int k = 0; k < kRows; ++k) {
        float2 a;
        sigmoids<T, kPlain>(r[k].get(), get_pair<T>(is, k).get(), s[k], pi[k]);
        decay_pair<kPlain>(__fmul2_rn(ndecay, s[k]), a, t[k]);
        const float2 m2 = m2_of(t[k]);
        const float2 m = make_float2(sqrt_approx(m2.x), sqrt_approx(m2.y));
        hp[k] = __fmul2_rn(__fmul2_rn(m, pi[k]), get_pair<T>(xs, k).get());
        if constexpr (!kPlain) hp[k] = make_float2(s[k].x == 0.f ? 0.f : hp[k].x, s[k].y == 0.f ? 0.f : hp[k].y);
        A = __fmul2_rn(a, A);
        S = __ffma2_rn(a, S, hp[k]);
      }
    };
    const bool plain_tile = plain && !any_held(min_rows(r));
    if (plain_tile)
      scan_rows(std::true_type());
    else
      scan_rows(std::false_type());
#pragma unroll
    for (int k = kRows - 1; k >= 0; --k)
      P = __fmul2_rn(__fadd2_rn(t[k], f2(1.f)), __fadd2_rn(P, get_pair<T>(gs, k).get()));
    maps[par][warp][lane] = make_float4(A.x, A.y, S.x, S.y);
    back[par][warp][lane] = P;
    __syncthreads();
    if (NS > 1 && TMA && threadIdx.x == 0 && j > 0) ask(j - 1 + NS);  // step j - 1's stage is free
    float2 gin = carry;
    if (nblk == 1) {
#pragma unroll
      for (int w = kWarps - 1; w >= 0; --w) {
        if (w == warp) gin = carry;
        const float4 m = maps[par][w][lane];
        carry = __ffma2_rn(make_float2(m.x, m.y), carry, back[par][w][lane]);
      }
      for (int w = 0; w < warp; ++w) h = apply(maps[par][w][lane], h);
    } else {
      if (warp == 0) {
        float2 ta = f2(1.f), tp = f2(0.f);
#pragma unroll
        for (int w = kWarps - 1; w >= 0; --w) {
          const float4 m = maps[par][w][lane];
          ta = __fmul2_rn(ta, make_float2(m.x, m.y));
          tp = __ffma2_rn(make_float2(m.x, m.y), tp, back[par][w][lane]);
        }
        ex.send(j, make_float4(ta.x, ta.y, tp.x, tp.y));
      }
      for (int w = 0; w < warp; ++w) h = apply(maps[par][w][lane], h);
      gin = ex.receive(j, carry, &g_status_scan);
      for (int w = kWarps - 1; w > warp; --w) {
        const float4 m = maps[par][w][lane];
        gin = __ffma2_rn(make_float2(m.x, m.y), gin, back[par][w][lane]);
      }
    }
#pragma unroll
    for (int k = 0; k < kRows; ++k) {  // the state before each token
      const float2 b = hp[k];
      hp[k] = h;
      h = __ffma2_rn(__fadd2_rn(t[k], f2(1.f)), h, b);
    }
    const long long o = first + (long long)row0 * p.D;
    T *dxr = dx + o, *drr = dr + o, *dir = di + o;
    auto grad_rows = [&](auto is_plain) {
      constexpr bool kPlain = decltype(is_plain)::value;
#pragma unroll
      for (int k = kRows - 1; k >= 0; --k) {
        const float2 a = __fadd2_rn(t[k], f2(1.f)), m2 = m2_of(t[k]);
        float2 im = make_float2(rsqrt_approx(m2.x), rsqrt_approx(m2.y));
        float2 x = get_pair<T>(xs, k).get();
        if constexpr (!kPlain) {  // no gradient through m where it is 0, none at all where the token held
          im = make_float2(m2.x > 0.f ? im.x : 0.f, m2.y > 0.f ? im.y : 0.f);
          x = make_float2(s[k].x == 0.f ? 0.f : x.x, s[k].y == 0.f ? 0.f : x.y);
        }
        const float2 dh = __fadd2_rn(get_pair<T>(gs, k).get(), gin);
        gin = __fmul2_rn(a, dh);
        const float2 w = __fmul2_rn(im, pi[k]);                // p / m
        const float2 gx = __fmul2_rn(dh, __fmul2_rn(m2, w));   // dh m p
        const float2 gi = __fmul2_rn(__fmul2_rn(gx, x), __ffma2_rn(pi[k], f2(-1.f), f2(1.f)));
        // dL = a dh (a p x / m - h_{t-1})
        const float2 u = __ffma2_rn(hp[k], f2(-1.f), __fmul2_rn(__fmul2_rn(a, w), x));
        const float2 dLs = __fmul2_rn(__fmul2_rn(gin, u), s[k]);
        ddecay = __fadd2_rn(ddecay, dLs);
        const float2 gr = __fmul2_rn(__fmul2_rn(dLs, ndecay), __fadd2_rn(s[k], f2(-1.f)));
        if (ln.on && k < have) {
          store_pair<T, TMA>(dxr + (long long)k * p.D, gx, ln.two);
          store_pair<T, TMA>(drr + (long long)k * p.D, gr, ln.two);
          store_pair<T, TMA>(dir + (long long)k * p.D, gi, ln.two);
        }
      }
    };
    if (plain_tile)
      grad_rows(std::true_type());
    else
      grad_rows(std::false_type());
  }
  if (TMA && threadIdx.x == 0) ring.drain(&g_status_scan);
  if (nblk > 1) cluster_barrier();  // as in the forward kernel, of dh0 and dfinal
  let_dependents_launch();
  // ddecay over the block's warps, in order.
  __syncthreads();
  back[0][warp][lane] = ddecay;
  __syncthreads();
  if (warp == 0) {
    float2 d = f2(0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) d = __fadd2_rn(d, back[0][w][lane]);
    ln.store(p.ddecay_part + ((long long)n * nblk + rank) * p.D, d);
    if (p.dh0 != nullptr && rank == 0) ln.store(p.dh0 + (long long)n * p.D, carry);
  }
}

struct StoreColumn {
  float* out;
  __device__ void operator()(int c, float v) const { out[c] = v; }
};

// --------------------------------------------------------------------------- launches
// Whether all of these are multiples of `unit` bytes.
bool multiples(int unit, int elem, int D, std::initializer_list<const void*> ptrs,
               std::initializer_list<long long> strides) {
  uintptr_t bits = (uintptr_t)D;
  for (long long s : strides) bits |= (uintptr_t)s;
  bits *= elem;
  for (const void* q : ptrs) bits |= reinterpret_cast<uintptr_t>(q);
  return (bits & (unit - 1)) == 0;
}

// A [B, T, D] tensor in 64 x 64 boxes. A dimension of one entry may have any stride.
int encode(CUtensorMap* m, int dtype, const void* base, long long bs, long long ts, int B, int T, int D) {
  const int elem = dtype == THM_BF16 ? 2 : 4;
  const uint64_t dims[3] = {(uint64_t)D, (uint64_t)T, (uint64_t)B};
  const uint64_t ts_b = (uint64_t)(T > 1 ? ts : (long long)(D * elem + 15) / 16 * 16 / elem) * elem;
  const uint64_t bs_b = B > 1 ? (uint64_t)bs * elem : ts_b * (uint64_t)T;
  const uint64_t strides[2] = {ts_b, bs_b};
  const uint32_t box[3] = {(uint32_t)kCols, (uint32_t)kChunk, 1};
  if (ts_b == 0 || bs_b == 0 || ts_b >= (1ull << 40) || bs_b >= (1ull << 40)) return THM_ERR_UNSUPPORTED;
  return encode_tiled(m, dtype == THM_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3,
                      base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE);
}

// Up to how many tokens a lane's serial walk beats the tiles, by the sequences of 64 channels.
// Measured (us, bf16, D 2048, walk / tiles): 32 sequences 4.1 / 4.0 at 16 tokens, 256 5.3 / 5.0
// at 24, 2048 11.1 / 19.0 at 32 and 20.1 / 15.5 at 64, 8192 33 / 68 and 71 / 62.
int direct_tokens(int count) {
  const int most = 14 + count / 48;
  return most < 48 ? most : 48;
}

// Blocks that share a sequence: as many as fit the GPU at once, and no more than a sequence has
// pairs of tiles for. Measured on bf16, forward: B8 T4096 D2048 (256 sequences of channels)
// 127 us alone, 141 with two blocks each, 158 with eight; B16 T8192 446 us alone, 484 with two;
// B1 T131072 2473 us alone, 578 with eight. Packed lengths are not known here: the longest of n
// random pieces has about (1 + ln n) / n of the rows, and the rest of the work fits beside it; of
// a few pieces one may have nearly all, and more blocks than needed cost little (65537 rows in 5
// pieces backward: 902 us alone, 622, 506 and 517 with two, four, eight; other cuts with four up
// to 618; 20011 rows in 37 pieces forward fp32: 80, 86, 111, 164).
//
// Sixteen, more than every GPU has to allow, only forward in bf16, where two such blocks still fit an
// SM, and for a dozen chains at most, which find room beside each other (T44352 D272, 5 chains: 155
// us with eight, 95 with sixteen; T32768 D1024, 16 chains: 136 and 140; backward T32768 D512: 189
// and 208).
int cluster_blocks(double chains, double tokens, int slots, bool wide) {
  int n = 1;
  while (n < 8 && chains * n * 2 <= slots && tokens / kChunk >= 4 * n) n *= 2;
  if (wide && n == 8 && chains * 16 * 3 <= slots * 2 && tokens / kChunk >= 32) n = 16;
  return n;
}
int packed_blocks(int T, int cols, int nseq, int slots, bool wide) {
  const double longest = nseq <= 8 ? 1. : (1. + std::log((double)nseq)) / nseq;
  return cluster_blocks(cols / longest, T * longest, slots, wide);
}

int bwd_cluster(int T, int D, int nseq, bool packed, int dtype) {
  const int slots = sm_count() * (dtype == THM_BF16 ? Bwd<__nv_bfloat16>::kPerSm : Bwd<float>::kPerSm);
  const int cols = (D + kCols - 1) / kCols;
  return packed ? packed_blocks(T, cols, nseq, slots, false) : cluster_blocks((double)nseq * cols, T, slots, false);
}

// `count` sequences of channels from `first` on, n blocks each.
template <typename K>
int launch_tiles(K kernel, Args p, const Maps& tm, int n, int first, int count, int smem, cudaStream_t st) {
  p.first = first;
  p.count = count;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) {
    cudaGetLastError();
    return THM_ERR_CUDA;
  }
  if (n > 8 && cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) {
    cudaGetLastError();
    return THM_ERR_CUDA;
  }
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3((unsigned)(n * count));
  cfg.blockDim = dim3(32 * kWarps);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = n;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kernel, p, tm) != cudaSuccess) {
    cudaGetLastError();
    return THM_ERR_CUDA;
  }
  return check_launch();
}

template <typename T>
int run_fwd(Args p, int B, int seqs, int dtype, cudaStream_t st) {
  constexpr int elem = sizeof(T);
  const int count = seqs * p.cols;
  if (p.T <= direct_tokens(count)) {
    const unsigned grid = (unsigned)((count + kDirectThreads / 32 - 1) / (kDirectThreads / 32));
    p.count = count;
    const bool paired = multiples(2 * elem, elem, p.D, {p.x, p.r, p.i, p.y}, {p.xb, p.xt, p.rb, p.rt, p.ib, p.it});
    auto kernel = p.T < 4 ? (paired ? scan_direct<T, true, 1> : scan_direct<T, false, 1>)
                          : (paired ? scan_direct<T, true, 4> : scan_direct<T, false, 4>);
    kernel<<<grid, kDirectThreads, 0, st>>>(p);
    return check_launch();
  }
  Maps tm{};
  bool tma = multiples(16, elem, p.D, {p.x, p.r, p.i, p.y}, {B > 1 ? p.xb : 0, p.xt, B > 1 ? p.rb : 0, p.rt, B > 1 ? p.ib : 0, p.it});
  tma = tma && encode(&tm.in[0], dtype, p.x, p.xb, p.xt, B, p.T, p.D) == THM_OK &&
        encode(&tm.in[1], dtype, p.r, p.rb, p.rt, B, p.T, p.D) == THM_OK &&
        encode(&tm.in[2], dtype, p.i, p.ib, p.it, B, p.T, p.D) == THM_OK;
  static_assert(Fwd<T, false>::R::kBytes == Fwd<T, true>::R::kBytes);
  auto run = [&](int n, int first, int cnt) {
    const int smem = Fwd<T, true>::R::kBytes + Exchange<Fwd<T, true>::kDepth>::bytes(n);
    if (n > 1)
      return tma ? launch_tiles(scan_tiles<T, true, true>, p, tm, n, first, cnt, smem, st)
                 : launch_tiles(scan_tiles<T, false, true>, p, tm, n, first, cnt, smem, st);
    return tma ? launch_tiles(scan_tiles<T, true, false>, p, tm, 1, first, cnt, smem, st)
               : launch_tiles(scan_tiles<T, false, false>, p, tm, 1, first, cnt, smem, st);
  };
  const int chain_slots = sm_count() * Fwd<T, true>::kPerSm, slots = sm_count() * Fwd<T, false>::kPerSm;
  // All blocks of a launch take about as long, so a few sequences more than the GPU holds cost as
  // much as a whole round of them: what is left over whole rounds runs as chains of blocks, in a
  // launch of its own (B16 T8192 D2048 bf16, 68 of 512 left over: 446 us in one launch, 424 in two).
  const int rest = count % slots;
  if (p.cu == nullptr && count > slots && rest > 0) {
    const int n = cluster_blocks(rest, p.T, chain_slots, sizeof(T) == 2);
    if (n > 1) {
      const int e = run(1, 0, count - rest);
      return e != THM_OK ? e : run(n, count - rest, rest);
    }
  }
  return run(p.cu == nullptr ? cluster_blocks(count, p.T, chain_slots, sizeof(T) == 2)
                               : packed_blocks(p.T, p.cols, p.nseq, chain_slots, sizeof(T) == 2), 0,
             count);
}

template <typename T>
int run_bwd(const Args& p, int B, int seqs, int dtype, int n, cudaStream_t st) {
  const int count = seqs * p.cols;
  constexpr int elem = sizeof(T);
  Maps tm{};
  bool tma = multiples(16, elem, p.D, {p.x, p.r, p.i, p.dy, p.dx, p.dr, p.di},
                       {B > 1 ? p.xb : 0, p.xt, B > 1 ? p.rb : 0, p.rt, B > 1 ? p.ib : 0, p.it, B > 1 ? p.gb : 0, p.gt});
  tma = tma && p.T > 0 && encode(&tm.in[0], dtype, p.x, p.xb, p.xt, B, p.T, p.D) == THM_OK &&
        encode(&tm.in[1], dtype, p.r, p.rb, p.rt, B, p.T, p.D) == THM_OK &&
        encode(&tm.in[2], dtype, p.i, p.ib, p.it, B, p.T, p.D) == THM_OK &&
        encode(&tm.in[3], dtype, p.dy, p.gb, p.gt, B, p.T, p.D) == THM_OK;
  const int smem = Bwd<T>::R::kBytes + Exchange<2>::bytes(n);
  return tma ? launch_tiles(scan_bwd_tiles<T, true>, p, tm, n, 0, count, smem, st)
             : launch_tiles(scan_bwd_tiles<T, false>, p, tm, n, 0, count, smem, st);
}

int check_sizes(int B, int T, int D, int nseq, const int* cu, int dtype) {
  if (B < 0 || T < 0 || D < 0 || nseq < 0) return THM_ERR_INVALID;
  if (dtype != THM_F32 && dtype != THM_BF16) return THM_ERR_INVALID;
  if (cu != nullptr ? B != 1 : nseq != B) return THM_ERR_INVALID;
  if (T > 1 << 30) return THM_ERR_UNSUPPORTED;  // rows, and those of a last round, count in 31 bits
  // (sequence, 64 channels) pairs, times the blocks of a cluster, are counted in 31 bits.
  if (((long long)nseq + 1) * ((D + kCols - 1) / kCols) >= 1ll << 27) return THM_ERR_UNSUPPORTED;
  return THM_OK;
}

}  // namespace gscan
}  // namespace thm

THM_STATUS_READER(thm_internal_status_scan, g_status_scan)

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
  p.T = T; p.D = D; p.nseq = nseq; p.cols = (D + gscan::kCols - 1) / gscan::kCols;
  const int seqs = nseq + (cu_seqlens != nullptr && zero_rest);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return dtype == THM_BF16 ? gscan::run_fwd<__nv_bfloat16>(p, B, seqs, dtype, st)
                           : gscan::run_fwd<float>(p, B, seqs, dtype, st);
}

extern "C" int thm_gated_scan_bwd_parts(int T, int D, int nseq, int packed, int dtype) {
  using namespace thm;
  if (T < 0 || D <= 0 || nseq <= 0) return 0;
  return nseq * gscan::bwd_cluster(T, D, nseq, packed != 0, dtype);
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
  p.T = T; p.D = D; p.nseq = nseq; p.cols = (D + gscan::kCols - 1) / gscan::kCols;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  int parts = 0;
  if (nseq > 0) {
    const int seqs = nseq + (cu_seqlens != nullptr && zero_rest);
    const int n = gscan::bwd_cluster(T, D, nseq, cu_seqlens != nullptr, dtype);
    parts = nseq * n;
    const int e = dtype == THM_BF16 ? gscan::run_bwd<__nv_bfloat16>(p, B, seqs, dtype, n, st)
                                    : gscan::run_bwd<float>(p, B, seqs, dtype, n, st);
    if (e != THM_OK) return e;
  }
  return sum_parts(workspace, parts, D, gscan::StoreColumn{ddecay}, st);
}
