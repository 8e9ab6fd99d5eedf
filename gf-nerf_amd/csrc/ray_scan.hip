// ray_scan.hip -- the gated linear recurrence along the packed samples of each ray,
//     h_t = a_t h_{t-1} + b_t ,   h_{-1} = h0 (or 0),
// front to back or back to front, its backward pass, and its form for one sample of every ray.  f [N, G] gates, c [N, D] inputs; gate
// d / (D / G) belongs to channel d:
//     linear   a = f              b = c
//     sigmoid  a = sigmoid(f)     b = (1 - a) c
//     decay    a = exp(-f)        b = (1 - a) c        (f = optical thickness: back to front this is alpha compositing of D channels)
// Backward:  l_t = dh_t + a_{t+1} l_{t+1} (the last row's: + d_state);  dc = l (1 - a) (linear: l);  df = l (h_{t-1} - c) da/df (linear:
// l h_{t-1}), summed over the channels of a gate;  dh0 = a_first l_first.  h_{t-1} is not read back: the forward leaves the f32 state it
// had on entering every aligned block of 8 rows (1/4 of the bytes of a 16-bit h, and nothing is rounded), and the backward walks each
// block forward from there in registers before it walks it backward.
//
// A lane owns VEC channels and walks rows: of one ray where there are rays enough to fill the chip, else of one RUN of rows (several to a
// ray, or several rays to one).  Rows are taken in aligned blocks of 8, the next block requested before this one is worked on, so the
// recurrence's chain of multiply-adds runs on data that has arrived.  A run's walk starts from a state that the rows in front of it
// decide: a first reading (AGG) reduces every run to one step state -> A state + S (state -> S where a ray begins in it), run_prefix_kernel
// composes the steps in order, and the second reading writes the results.  A product of many gates leaves f32's range long before a state
// does, so A has an exponent of its own: it is zero only where a gate is, and what a walk row by row keeps -- a state, a NaN -- a step keeps.  Every sum has a fixed order: the same bits
// every run.  State and adjoint are f32.
#include "gfn_common.h"

namespace {

constexpr int kBlock = GFN_SCAN_BLOCK;  // rows a saved state covers
enum { GATE_LINEAR = 0, GATE_SIGMOID = 1, GATE_DECAY = 2 };

template <bool EXACT>
__device__ __forceinline__ float exp_of(float v) {
  if constexpr (EXACT) return expf(v);
  return __builtin_amdgcn_exp2f(v * 1.44269504088896340736f);
}

// a and 1 - a, each with its own relative accuracy (a thin sample's 1 - a is its whole contribution)
template <int GATE, bool EXACT>
__device__ __forceinline__ void gate_of(float f, float& a, float& rest) {
  if constexpr (GATE == GATE_LINEAR) {
    a = f;
    rest = 1.f;
  } else if constexpr (GATE == GATE_SIGMOID) {
    const float e = exp_of<EXACT>(-f);  // infinite from f < -88 on: a = 0, 1 - a = 1
    a = EXACT ? 1.f / (1.f + e) : __builtin_amdgcn_rcpf(1.f + e);
    rest = e > 1.f ? 1.f - a : e * a;
  } else {
    a = exp_of<EXACT>(-f);
    if constexpr (EXACT) {
      rest = -expm1f(-f);
    } else {  // f (1 - f/2 + f^2/6 - ...) below 1/4: the next term is 5e-8 of the sum
      float p = __builtin_fmaf(f, -1.f / 720.f, 1.f / 120.f);
      p = __builtin_fmaf(p, -f, 1.f / 24.f);
      p = __builtin_fmaf(p, -f, 1.f / 6.f);
      p = __builtin_fmaf(p, -f, 0.5f);
      p = __builtin_fmaf(p, -f, 1.f);
      rest = __builtin_fabsf(f) < 0.25f ? f * p : 1.f - a;
    }
  }
}

template <typename T, int VEC>
struct alignas(VEC * sizeof(T)) Vec {
  T v[VEC];
};

struct ScanArgs {
  const int32_t* offsets;
  int64_t rays, n_max;
  const void *f, *c, *dh;
  int64_t ldf, ldc, ldh, lddh, lddf, lddc;
  int d, g, reverse;
  const float *h0, *d_state;
  void *h, *df, *dc;
  float *state, *saved, *dh0;
  const float* saved_in;
  int per_gate;  // channels of a gate
  int clear;     // rows of no ray: write zeros
  // how lanes are dealt out: `lanes` to a walk, in slots of `slot` (a power of two) to a shared gate, `parts` slots of 64 where one is
  // not enough (df's sums over each go to `partial` [parts][n_max][g] then)
  int lanes, slot, parts;
  float* partial;
  int64_t run_rows, runs;  // 0: a walk is a ray; else rows of a run (a multiple of kBlock) and their number
  struct Step* agg;        // [d][runs]: AGG writes the steps; then .s is the state in front of the run
};

// What a run does to the state in front of it: A state + s, A = m 2^e with m = 0 or 1/2 <= |m| < 1 (or not finite); begins: s alone.
struct alignas(16) Step {
  float m;
  int e;
  float s;
  int begins;
};
struct Gain {  // A on its way through a run
  float m = 1.f;
  int e = 0;
  __device__ __forceinline__ void times(float a) {  // up to 8 times between normalize()
    m *= __builtin_amdgcn_frexp_mantf(a);
    e += __builtin_amdgcn_frexp_expf(a);
  }
  __device__ __forceinline__ void normalize() {  // (e stays far inside an int however long the run)
    e += __builtin_amdgcn_frexp_expf(m);
    m = __builtin_amdgcn_frexp_mantf(m);
    e = e < -(1 << 28) ? -(1 << 28) : e > 1 << 28 ? 1 << 28 : e;
  }
};
// the state behind a step from the state in front of it.  (A state of zero leaves s: gates that are not finite have met it already.)
__device__ __forceinline__ float after(const Step& q, float s) {
  if (q.begins || s == 0.f) return q.s;
  if (q.e > -100 && q.e < 100) return __builtin_fmaf(__builtin_amdgcn_ldexpf(q.m, q.e), s, q.s);
  return (q.e > 0 ? __builtin_amdgcn_ldexpf(s, q.e - 1) * (q.m + q.m) : __builtin_amdgcn_ldexpf(q.m * s, q.e)) + q.s;
}
// q1 and then q2, as one step
__device__ __forceinline__ Step both(const Step& q1, const Step& q2) {
  Gain g;
  g.m = q1.m * q2.m;
  g.e = q1.e + q2.e;
  g.normalize();
  return {g.m, g.e, after(q2, q1.s), q1.begins | q2.begins};
}

struct Place {
  int64_t walk;  // the ray or run
  int ch, gate, part;
  bool active;   // a lane of a slot that no channel fills stays for the slot's reductions, reading channel 0 of its gate
};

template <int VEC, bool SHARED>
__device__ __forceinline__ bool scan_place(const ScanArgs& a, Place& p) {
  const int64_t id = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  p.walk = id / a.lanes;
  const int at = (int)(id - p.walk * a.lanes);
  p.part = 0;
  if constexpr (SHARED) {
    const int span = a.slot * a.parts, in = at % span;
    p.gate = at / span;
    p.part = in / a.slot;
    p.active = in * VEC < a.per_gate;
    p.ch = p.gate * a.per_gate + (p.active ? in * VEC : 0);
  } else {
    p.ch = p.gate = at * VEC;
    p.active = true;
  }
  return p.walk < (a.run_rows ? a.runs : a.rays);
}

__device__ __forceinline__ int64_t clamp_row(int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : (v > hi ? hi : v); }

// The pieces of a walk: one ray, or a run's share of each ray it meets, in the order `asc` says.  Offsets are kept inside the arrays,
// whatever they hold.
struct Pieces {
  const ScanArgs& a;
  bool asc;
  int64_t lo, hi, ray;  // the run's rows (a ray: all); the ray of the next piece
  __device__ Pieces(const ScanArgs& args, int64_t walk, bool up) : a(args), asc(up) {
    if (!a.run_rows) {
      lo = 0;
      hi = a.n_max;
      ray = walk;
      return;
    }
    const int64_t r = asc ? walk : a.runs - 1 - walk;  // runs are numbered in the walk's order
    lo = r * a.run_rows;
    hi = lo + a.run_rows < a.n_max ? lo + a.run_rows : a.n_max;
    int64_t x = 0, y = a.rays;  // up: the first ray that ends behind the first row; down: the last that begins in front of the last
    while (x < y) {
      const int64_t m = (x + y) >> 1;
      if (asc ? a.offsets[m + 1] > lo : a.offsets[m] >= hi) y = m;
      else x = m + 1;
    }
    ray = asc ? x : x - 1;
  }
  // rows [s, e) of the next piece and whether its ray begins / ends (in the walk's order) there; false: no more
  __device__ bool next(int64_t& of, int64_t& s, int64_t& e, bool& begins, bool& ends) {
    for (bool passed = false;; passed = true) {
      if (ray < 0 || ray >= a.rays) return false;
      const int64_t rs = clamp_row(a.offsets[ray], 0, a.n_max), re = clamp_row(a.offsets[ray + 1], rs, a.n_max);
      if (a.run_rows && (asc ? rs >= hi : re <= lo)) return false;
      of = ray;
      s = rs > lo ? rs : lo;
      e = re < hi ? re : hi;
      begins = asc ? s == rs : e == re;
      ends = asc ? e == re : s == rs;
      if (!a.run_rows) {
        ray = a.rays;
        return true;
      }
      if (s < e || !passed) {
        ray += asc ? 1 : -1;
        if (s < e) return true;
      } else {  // a second ray without rows: there may be many
        int64_t x = asc ? ray + 1 : 0, y = asc ? a.rays : ray;
        while (x < y) {
          const int64_t m = (x + y) >> 1;
          if (asc ? a.offsets[m + 1] > rs : a.offsets[m] >= re) y = m;
          else x = m + 1;
        }
        ray = asc ? x : x - 1;
      }
    }
  }
};

// rows of no ray (behind the last ray's): -> 0
template <typename T>
__device__ __forceinline__ void clear_rows(const ScanArgs& a, T* p, int64_t ld, int width) {
  const int64_t begin = clamp_row(a.offsets[a.rays], 0, a.n_max);
  for (int64_t e = begin * width + (int64_t)blockIdx.x * blockDim.x + threadIdx.x; e < a.n_max * width; e += (int64_t)gridDim.x * blockDim.x)
    p[e / width * ld + e % width] = (T)0.f;
}

template <int BYTES>
struct BitsOf { using type = uint32_t; };
template <>
struct BitsOf<2> { using type = uint16_t; };

// One block of a piece: its rows in the walk's order are row0, row0 + dir, ...; those in [s, e) count.
template <typename T, int VEC, bool SHARED, bool BWD, bool AGG>
struct Rows {
  using F = typename BitsOf<sizeof(T) * (SHARED ? 1 : VEC)>::type;
  using C = typename BitsOf<sizeof(T) * VEC>::type;
  F f[kBlock];
  C c[kBlock], dh[BWD ? kBlock : 1];
  T fd;  // shared gates dealt out over 8 lanes or more: this lane's row's
  __device__ __forceinline__ float gate(int r, int v) const {
    if constexpr (SHARED) return (float)__builtin_bit_cast(T, f[r]);
    else return (float)__builtin_bit_cast(Vec<T, VEC>, f[r]).v[v];
  }
  __device__ __forceinline__ float in(int r, int v) const { return (float)__builtin_bit_cast(Vec<T, VEC>, c[r]).v[v]; }
  __device__ __forceinline__ float grad(int r, int v) const { return (float)__builtin_bit_cast(Vec<T, VEC>, dh[BWD ? r : 0]).v[v]; }
  template <typename R>
  static __device__ __forceinline__ void column(R (&to)[kBlock], const T* from, int64_t ld, int64_t row0, bool asc, bool whole, int64_t s, int64_t e) {
    if (whole) {
      const T* q = from + row0 * ld;
      const int64_t step = asc ? ld : -ld;
#pragma unroll
      for (int r = 0; r < kBlock; r++) to[r] = *reinterpret_cast<const R*>(q + r * step);
    } else {  // another kind of load, or the compiler joins the two ways' loads and keeps sixteen addresses for them
#pragma unroll
      for (int r = 0; r < kBlock; r++) to[r] = __builtin_nontemporal_load(reinterpret_cast<const R*>(from + clamp_row(asc ? row0 + r : row0 - r, s, e - 1) * ld));
    }
  }
  template <bool INNER>
  __device__ __forceinline__ void load(const ScanArgs& a, const T* pf, const T* pc, const T* pd, int64_t base, bool asc, int64_t s, int64_t e, int deal) {
    const int64_t row0 = base + (asc ? 0 : kBlock - 1);
    const bool whole = INNER || __all(base >= s && base + kBlock <= e);
    if (SHARED && deal >= 0) fd = pf[clamp_row(asc ? row0 + deal : row0 - deal, s, e - 1) * a.ldf];
    else column(f, pf, a.ldf, row0, asc, whole, s, e);
    if constexpr (!(BWD && AGG)) column(c, pc, a.ldc, row0, asc, whole, s, e);
    if constexpr (BWD) column(dh, pd, a.lddh, row0, asc, whole, s, e);
  }
};

constexpr int kScanThreads = 256;

// The gates of a block: each lane its own, or -- shared by 8 lanes or more -- one evaluation a lane, dealt through LDS.
template <typename T, int GATE, int VEC, bool SHARED>
struct Gates {
  float2* pool;  // kBlock entries of the slot's, or null
  int deal;
  __device__ __forceinline__ void begin(const T& fd) {
    if (SHARED && pool) {
      float x, y;
      gate_of<GATE, sizeof(T) == 4>((float)fd, x, y);
      __builtin_amdgcn_wave_barrier();
      pool[deal] = make_float2(x, y);  // lanes with the same row write the same value
      __builtin_amdgcn_wave_barrier();
    }
  }
  template <typename R>
  __device__ __forceinline__ void get(int r, const R& rows, float (&x)[VEC], float (&y)[VEC]) const {
    if (SHARED && pool) {
      const float2 q = pool[r];
#pragma unroll
      for (int v = 0; v < VEC; v++) { x[v] = q.x; y[v] = q.y; }
    } else {
#pragma unroll
      for (int v = 0; v < VEC; v++) {
        if (!SHARED || v == 0) gate_of<GATE, sizeof(T) == 4>(rows.gate(r, v), x[v], y[v]);
        else { x[v] = x[0]; y[v] = y[0]; }
      }
    }
  }
};

struct Yes { static constexpr bool value = true; };
struct No { static constexpr bool value = false; };
// Whether this block and the next are whole rows of the piece in every lane, with one more behind them.  Such blocks are worked on without
// a branch, so that a wait for the next block's rows is not one for the stores behind their requests (loads and stores are counted together,
// in order): backward of 4096 rays x 192 rows x 128 channels in bf16 255 -> 237 us, a first reading of 2 x 131072 x 64 f16 21 -> 19 us (then without the exponents).
template <typename F>
__device__ __forceinline__ bool inner(int64_t i, int64_t blocks, int64_t lo, int64_t hi, F base_of, bool active) {
  if (!__all(active && i + 2 < blocks)) return false;
  const int64_t p = base_of(i), q = base_of(i + 1);
  return __all(p >= lo && p + kBlock <= hi && q >= lo && q + kBlock <= hi);
}

// Walks along runs never meet a ray without rows: its last state is the one it starts with (its adjoint likewise).
__device__ __forceinline__ void empty_rays(const ScanArgs& a, const float* __restrict__ from, float* __restrict__ to) {
  const int lane = threadIdx.x & 63;
  const int64_t waves = (int64_t)gridDim.x * blockDim.x / 64;
  for (int64_t ray = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) / 64; ray < a.rays; ray += waves)
    if (a.offsets[ray + 1] <= a.offsets[ray])
      for (int i = lane; i < a.d; i += 64) to[ray * a.d + i] = from ? from[ray * a.d + i] : 0.f;
}

template <typename T, int GATE, int VEC, bool SHARED, bool AGG>
__global__ __launch_bounds__(kScanThreads) void scan_fwd_kernel(ScanArgs a) {
  using V = Vec<T, VEC>;
  __shared__ float2 pool[SHARED ? kScanThreads : 1];
  if (!AGG && a.clear) clear_rows(a, static_cast<T*>(a.h), a.ldh, a.d);
  if (!AGG && a.run_rows && a.state) empty_rays(a, a.h0, a.state);
  Place at;
  if (!scan_place<VEC, SHARED>(a, at)) return;
  const bool asc = !a.reverse, dealt = SHARED && a.slot >= kBlock;
  const int deal = dealt ? threadIdx.x & (kBlock - 1) : -1;
  Gates<T, GATE, VEC, SHARED> gates{dealt ? pool + (threadIdx.x & ~(a.slot - 1)) : nullptr, deal};
  const T *f = static_cast<const T*>(a.f) + at.gate, *c = static_cast<const T*>(a.c) + at.ch;
  T* h = static_cast<T*>(a.h) + at.ch;
  float s[VEC];
  Gain A[VEC];
  int begun = 0;
#pragma unroll
  for (int v = 0; v < VEC; v++) s[v] = !AGG && a.run_rows ? a.agg[(at.ch + v) * a.runs + at.walk].s : 0.f;
  Pieces pieces(a, at.walk, asc);
  int64_t ray, lo, hi;
  bool begins, ends;
  while (pieces.next(ray, lo, hi, begins, ends)) {
    if (begins) {
      begun = 1;
#pragma unroll
      for (int v = 0; v < VEC; v++) s[v] = a.h0 ? a.h0[ray * a.d + at.ch + v] : 0.f;
    }
    const int64_t b0 = lo / kBlock, blocks = hi > lo ? (hi - 1) / kBlock - b0 + 1 : 0;
    Rows<T, VEC, SHARED, false, AGG> now, next;
    auto base_of = [&](int64_t i) { return (asc ? b0 + i : b0 + blocks - 1 - i) * kBlock; };
    if (blocks) now.template load<false>(a, f, c, nullptr, base_of(0), asc, lo, hi, deal);
    auto work = [&](int64_t i, auto inner_c) {
      constexpr bool INNER = decltype(inner_c)::value;
      const int64_t base = base_of(i), row0 = base + (asc ? 0 : kBlock - 1);
      if (!AGG && a.saved && (INNER || (at.active && row0 >= lo && row0 < hi)))
#pragma unroll
        for (int v = 0; v < VEC; v++) a.saved[base / kBlock * a.d + at.ch + v] = s[v];
      if (INNER || i + 1 < blocks) next.template load<INNER>(a, f, c, nullptr, base_of(i + 1), asc, lo, hi, deal);
      gates.begin(now.fd);
      const bool whole = INNER || __all(base >= lo && base + kBlock <= hi && at.active);
      T* out = h + row0 * a.ldh;
      const int64_t step = asc ? a.ldh : -a.ldh;
#pragma unroll
      for (int r = 0; r < kBlock; r++) {
        float x[VEC], y[VEC];
        gates.get(r, now, x, y);
        V o;
        const int64_t row = asc ? row0 + r : row0 - r;
        const bool in = whole || (row >= lo && row < hi);
#pragma unroll
        for (int v = 0; v < VEC; v++) {
          const float n = __builtin_fmaf(x[v], s[v], y[v] * now.in(r, v));
          s[v] = in ? n : s[v];
          if (AGG) A[v].times(in ? x[v] : 1.f);
          o.v[v] = (T)s[v];
        }
        if (!AGG) {
          if (whole) *reinterpret_cast<V*>(out + r * step) = o;
          else if (in && at.active) *reinterpret_cast<V*>(out + r * step) = o;
        }
      }
      if (AGG)
#pragma unroll
        for (int v = 0; v < VEC; v++) A[v].normalize();
      if (INNER || i + 1 < blocks) now = next;
    };
    for (int64_t i = 0; i < blocks; i++) {
      if constexpr (AGG)  // (writing h as well it costs a wave a SIMD: 180 instead of 158 us for 4096 rays x 192 rows x 128 channels, bf16)
        for (; inner(i, blocks, lo, hi, base_of, at.active); i++) work(i, Yes{});
      work(i, No{});
    }
    if (!AGG && ends && a.state && at.active)
#pragma unroll
      for (int v = 0; v < VEC; v++) a.state[ray * a.d + at.ch + v] = s[v];
  }
  if (AGG && at.active)
#pragma unroll
    for (int v = 0; v < VEC; v++) a.agg[(at.ch + v) * a.runs + at.walk] = {A[v].m, A[v].e, s[v], begun};
}

template <typename T, int GATE, int VEC, bool SHARED, bool AGG>
__global__ __launch_bounds__(kScanThreads) void scan_bwd_kernel(ScanArgs a) {
  using V = Vec<T, VEC>;
  __shared__ float2 pool[SHARED ? kScanThreads : 1];
  if (!AGG && a.clear) {
    clear_rows(a, static_cast<T*>(a.df), a.lddf, a.g);
    clear_rows(a, static_cast<T*>(a.dc), a.lddc, a.d);
  }
  if (!AGG && a.run_rows && a.dh0) empty_rays(a, a.d_state, a.dh0);
  Place at;
  if (!scan_place<VEC, SHARED>(a, at)) return;
  const bool asc = a.reverse != 0, dealt = SHARED && a.slot >= kBlock;  // against the recurrence
  const int deal = dealt ? threadIdx.x & (kBlock - 1) : -1;
  Gates<T, GATE, VEC, SHARED> gates{dealt ? pool + (threadIdx.x & ~(a.slot - 1)) : nullptr, deal};
  const T *f = static_cast<const T*>(a.f) + at.gate, *c = static_cast<const T*>(a.c) + at.ch, *dh = static_cast<const T*>(a.dh) + at.ch;
  T *df = static_cast<T*>(a.df) + at.gate, *dc = static_cast<T*>(a.dc) + at.ch;
  float l[VEC];
  Gain A[VEC];
  int begun = 0;
#pragma unroll
  for (int v = 0; v < VEC; v++) l[v] = !AGG && a.run_rows ? a.agg[(at.ch + v) * a.runs + at.walk].s : 0.f;
  Pieces pieces(a, at.walk, asc);
  int64_t ray, lo, hi;
  bool begins, ends;
  while (pieces.next(ray, lo, hi, begins, ends)) {
    if (begins) {
      begun = 1;
#pragma unroll
      for (int v = 0; v < VEC; v++) l[v] = a.d_state ? a.d_state[ray * a.d + at.ch + v] : 0.f;
    }
    const int64_t b0 = lo / kBlock, blocks = hi > lo ? (hi - 1) / kBlock - b0 + 1 : 0;
    Rows<T, VEC, SHARED, true, AGG> now, next;
    auto base_of = [&](int64_t i) { return (asc ? b0 + i : b0 + blocks - 1 - i) * kBlock; };
    float entry[VEC];  // the state in front of the next block's rows (in the recurrence's order), requested with them
    auto enter = [&](int64_t i, auto inner_c) {
      if constexpr (!AGG) {
        const bool ray_starts = !decltype(inner_c)::value && ends && i == blocks - 1;  // the recurrence's first row of the ray is in this block
        const int64_t base = base_of(i), first = asc ? hi - 1 : lo;                       // the recurrence's first row of the piece, in its last block
        const float* from = ray_starts ? a.h0 : a.saved_in;
        const int64_t of = ray_starts ? ray : (asc ? (base + kBlock - 1 < first ? base + kBlock - 1 : first) : (base > first ? base : first)) / kBlock;
#pragma unroll
        for (int v = 0; v < VEC; v++) entry[v] = decltype(inner_c)::value || from ? from[of * a.d + at.ch + v] : 0.f;
      }
    };
    if (blocks) {
      now.template load<false>(a, f, c, dh, base_of(0), asc, lo, hi, deal);
      enter(0, No{});
    }
    auto work = [&](int64_t i, auto inner_c) {
      constexpr bool INNER = decltype(inner_c)::value;
      const int64_t base = base_of(i), row0 = base + (asc ? 0 : kBlock - 1);
      float before[AGG ? 1 : kBlock][VEC], st[VEC];
      if (!AGG)
#pragma unroll
        for (int v = 0; v < VEC; v++) st[v] = entry[v];
      if (INNER || i + 1 < blocks) {
        next.template load<INNER>(a, f, c, dh, base_of(i + 1), asc, lo, hi, deal);
        enter(i + 1, inner_c);
      }
      gates.begin(now.fd);
      const bool whole = INNER || __all(base >= lo && base + kBlock <= hi && at.active);
      float x[kBlock][VEC], y[kBlock][VEC];
#pragma unroll
      for (int r = kBlock - 1; r >= 0; r--) {  // the recurrence's order
        gates.get(r, now, x[r], y[r]);
        if (!AGG) {
          const int64_t row = asc ? row0 + r : row0 - r;
          const bool in = whole || (row >= lo && row < hi);
#pragma unroll
          for (int v = 0; v < VEC; v++) {
            before[r][v] = st[v];
            const float n = __builtin_fmaf(x[r][v], st[v], y[r][v] * now.in(r, v));
            st[v] = in ? n : st[v];
          }
        }
      }
      float sums[SHARED && !AGG ? kBlock : 1];
      T *out_c = dc + row0 * a.lddc, *out_f = df + row0 * a.lddf;
      const int64_t step_c = asc ? a.lddc : -a.lddc, step_f = asc ? a.lddf : -a.lddf;
#pragma unroll
      for (int r = 0; r < kBlock; r++) {
        const int64_t row = asc ? row0 + r : row0 - r;
        const bool in = whole || (row >= lo && row < hi);
        V oc, of;
        float sum = 0.f;
#pragma unroll
        for (int v = 0; v < VEC; v++) {
          const float lt = l[v] + now.grad(r, v), xv = x[r][v], yv = y[r][v];
          if (!AGG) {
            const float cv = now.in(r, v);
            float d;
            if constexpr (GATE == GATE_LINEAR) d = lt * before[r][v];
            else if constexpr (GATE == GATE_SIGMOID) d = lt * (before[r][v] - cv) * (xv * yv);
            else d = lt * (cv - before[r][v]) * xv;
            oc.v[v] = (T)(lt * yv);
            if constexpr (SHARED) sum += d;
            else of.v[v] = (T)d;
          }
          l[v] = in ? xv * lt : l[v];
          if (AGG) A[v].times(in ? xv : 1.f);
        }
        if (!AGG) {
          if (whole) {
            *reinterpret_cast<V*>(out_c + r * step_c) = oc;
            if constexpr (!SHARED) *reinterpret_cast<V*>(out_f + r * step_f) = of;
          } else if (in && at.active) {
            *reinterpret_cast<V*>(out_c + r * step_c) = oc;
            if constexpr (!SHARED) *reinterpret_cast<V*>(out_f + r * step_f) = of;
          }
          if constexpr (SHARED) sums[r] = at.active ? sum : 0.f;
        }
      }
      if constexpr (SHARED && !AGG) {  // a gate's lanes add their channels: halve the rows a lane holds while lanes are left, then add plainly
        int held = kBlock, first = 0;
#pragma unroll
        for (int o = 1; o < kBlock; o <<= 1) {
          if (o < a.slot) {
            held >>= 1;
            const bool up = threadIdx.x & o;
#pragma unroll
            for (int k = 0; k < kBlock / 2; k++)
              if (k < held) {
                const float send = up ? sums[k] : sums[k + held], keep = up ? sums[k + held] : sums[k];
                sums[k] = keep + __shfl_xor(send, o, 64);
              }
            first += up ? held : 0;
          }
        }
        for (int o = kBlock; o < a.slot; o <<= 1) sums[0] += __shfl_xor(sums[0], o, 64);
        const bool writer = (int)(threadIdx.x & (a.slot - 1)) < kBlock;
#pragma unroll
        for (int k = 0; k < kBlock; k++)
          if (k < held && writer) {
            const int64_t row = asc ? row0 + first + k : row0 - first - k;
            if (row >= lo && row < hi) {
              if (a.parts > 1) a.partial[((int64_t)at.part * a.n_max + row) * a.g + at.gate] = sums[k];
              else df[row * a.lddf] = (T)sums[k];
            }
          }
      }
      if (AGG)
#pragma unroll
        for (int v = 0; v < VEC; v++) A[v].normalize();
      if (INNER || i + 1 < blocks) now = next;
    };
    for (int64_t i = 0; i < blocks; i++) {
      for (; inner(i, blocks, lo, hi, base_of, at.active); i++) work(i, Yes{});
      work(i, No{});
    }
    if (!AGG && ends && a.dh0 && at.active)
#pragma unroll
      for (int v = 0; v < VEC; v++) a.dh0[ray * a.d + at.ch + v] = l[v];
  }
  if (AGG && at.active)
#pragma unroll
    for (int v = 0; v < VEC; v++) a.agg[(at.ch + v) * a.runs + at.walk] = {A[v].m, A[v].e, l[v], begun};
}

// AGG's steps -> the state in front of every run (in the walk's order).  A workgroup: one channel, 1,024 stretches of neighbouring runs, each
// composed in registers (up to kHeld runs of a stretch; more are read twice), the stretches joined by doubling within a wave and the
// waves' steps one after the other.  Latency bound: 9 us for 4,096 runs of 64 channels.  (Steps without an exponent: 5,
// and laid out as [runs][channels], four channels a workgroup, 18 -- every load then takes a part of a line, on a quarter of the CUs.)
constexpr int kHeld = 4, kPrefixWaves = 16;
__device__ __forceinline__ Step step_up(const Step& q, int by) {
  return {__shfl_up(q.m, by, 64), __shfl_up(q.e, by, 64), __shfl_up(q.s, by, 64), __shfl_up(q.begins, by, 64)};
}
__global__ __launch_bounds__(64 * kPrefixWaves) void run_prefix_kernel(Step* __restrict__ steps, int64_t runs) {
  __shared__ Step last[kPrefixWaves];
  Step* __restrict__ agg = steps + (int64_t)blockIdx.x * runs;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t per = (runs + 64 * kPrefixWaves - 1) / (64 * kPrefixWaves), lo = threadIdx.x * per, hi = lo + per < runs ? lo + per : runs;
  Step held[kHeld], q = {0.5f, 1, 0.f, 0};
#pragma unroll
  for (int i = 0; i < kHeld; i++) held[i] = lo + i < hi ? agg[lo + i] : Step{0.5f, 1, 0.f, 0};
#pragma unroll
  for (int i = 0; i < kHeld; i++)
    if (lo + i < hi) q = both(q, held[i]);
  for (int64_t i = lo + kHeld; i < hi; i++) q = both(q, agg[i]);
#pragma unroll
  for (int off = 1; off < 64; off *= 2) {  // then q is the step of the wave's stretches up to this one
    const Step q1 = step_up(q, off);
    if (lane >= off) q = both(q1, q);
  }
  if (lane == 63) last[wave] = q;
  __syncthreads();
  float front = 0.f;  // the state in front of the wave's first stretch, then of this one
  for (int w = 0; w < wave; w++) front = after(last[w], front);
  const Step q1 = step_up(q, 1);
  float s = lane ? after(q1, front) : front;
#pragma unroll
  for (int i = 0; i < kHeld; i++)
    if (lo + i < hi) {
      agg[lo + i].s = s;
      s = after(held[i], s);
    }
  for (int64_t i = lo + kHeld; i < hi; i++) {
    const Step r = agg[i];
    agg[i].s = s;
    s = after(r, s);
  }
}

// df of gates whose channels take several slots: the slots' sums in order
template <typename T>
__global__ __launch_bounds__(256) void scan_gate_sums_kernel(ScanArgs a, const float* __restrict__ partial, int parts) {
  const int64_t n = a.n_max * a.g, live_lo = (int64_t)a.offsets[0] * a.g, live_hi = (int64_t)a.offsets[a.rays] * a.g;
  for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < n; e += (int64_t)gridDim.x * 256) {
    const bool live = e >= live_lo && e < live_hi;
    if (!live && !a.clear) continue;
    float s = 0.f;
    if (live)
      for (int i = 0; i < parts; i++) s += partial[i * n + e];
    static_cast<T*>(a.df)[e / a.g * a.lddf + e % a.g] = (T)s;
  }
}

// one more row of every ray: state[r] = a state[r] + b
template <typename T, int GATE>
__global__ __launch_bounds__(256) void scan_step_kernel(ScanArgs a) {
  const int64_t n = a.rays * a.d;
  for (int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x; id < n; id += (int64_t)gridDim.x * 256) {
    const int64_t row = id / a.d;
    const int ch = (int)(id - row * a.d);
    float ga, rest;
    gate_of<GATE, sizeof(T) == 4>((float)static_cast<const T*>(a.f)[row * a.ldf + ch / a.per_gate], ga, rest);
    const float s = __builtin_fmaf(ga, a.state[id], rest * (float)static_cast<const T*>(a.c)[row * a.ldc + ch]);
    a.state[id] = s;
    static_cast<T*>(a.h)[row * a.ldh + ch] = (T)s;
  }
}

// ---- host ---------------------------------------------------------------------------------------------------------------------------
int check_scan(const char* who, int64_t rays, int64_t n_max, int d, int g, int dtype, int gate, int64_t ldf, int64_t ldc) {
  GFN_CHECK_ARG(rays >= 0 && rays < (1ll << 31) && n_max >= 0 && n_max < (1ll << 31), "%s: %lld rays, n_max %lld", who, (long long)rays, (long long)n_max);
  GFN_CHECK_ARG(d >= 1 && d <= GFN_SCAN_MAX_CHANNELS && g >= 1 && g <= d && d % g == 0, "%s: %d gates for %d channels (1..%d channels, the gates dividing them)", who, g, d,
                GFN_SCAN_MAX_CHANNELS);
  GFN_CHECK_ARG(dtype >= GFN_F32 && dtype <= GFN_F16, "%s: dtype %d", who, dtype);
  GFN_CHECK_ARG(gate >= 0 && gate <= 2, "%s: gate %d", who, gate);
  GFN_CHECK_ARG(ldf >= g && ldc >= d, "%s: a row stride is below the row's width", who);
  return GFN_OK;
}

// whether every pointer, stride and gate group leaves pairs of 16-bit channels aligned
bool two_channels(const ScanArgs& a, bool shared, bool bwd) {
  const int64_t strides = a.ldc | (bwd ? a.lddh | a.lddc : a.ldh) | (shared ? 0 : a.ldf | (bwd ? a.lddf : 0)) | (shared ? a.per_gate : a.d);
  uintptr_t at = reinterpret_cast<uintptr_t>(a.c) | (bwd ? reinterpret_cast<uintptr_t>(a.dh) | reinterpret_cast<uintptr_t>(a.dc) : reinterpret_cast<uintptr_t>(a.h));
  if (!shared) at |= reinterpret_cast<uintptr_t>(a.f) | (bwd ? reinterpret_cast<uintptr_t>(a.df) : 0);
  return strides % 2 == 0 && at % 4 == 0;
}

// Rays or runs.  A walk along a ray waits 0.13 to 0.3 us a row where rays do not fill the chip; runs read everything twice and stop at every
// ray's beginning.  One rule for every type, gate and direction, by the rays' mean length; us of a call, rays of EQUAL lengths (of spread lengths
// the longest decides a walk along rays: 512 x 512 x 128 bf16 139 instead of 82), runs / rays:
//                                     bf16 forward   bf16 backward   f32 forward   f32 backward   one gate, bf16 backward
//   16 rays x 2048 rows x 32 channels   22 / 261        24 / 284       24 / 366      26 / 380        30 / 593
//   512 x 512 x 128                     82 / 82         97 / 99       160 / 128     193 / 167        87 / 169
//   512 x 128 x 64                      27 / 22         31 / 25        33 / 30       36 / 31         37 / 46
//   1024 x 192 x 64                     43 / 35         48 / 34        60 / 44       67 / 46         48 / 65
//   1024 x 100 x 8                      36 / 18         44 / 22        42 / 23       49 / 27         58 / 38
//   512 x 1024 x 256                   299 / 219       368 / 259      551 / 314     676 / 452       293 / 344
//   4096 x 192 x 128                   232 / 130       276 / 178      443 / 247     532 / 332       227 / 156
bool use_runs(int64_t rays, int64_t n_max, int d) {
  const int64_t mean = rays > 0 ? n_max / rays : 0;
  return mean >= 96 && rays < 6 * mean && rays * d < 128 * 1024;
}

struct ScanPlan {
  int slot, parts, lanes;
  int64_t run_rows, runs;
};
ScanPlan plan_scan(int64_t rays, int64_t n_max, int d, int g, int vec) {
  ScanPlan p{1, 1, d / vec, 0, 0};
  if (g != d) {
    const int need = (d / g + vec - 1) / vec;
    while (p.slot < need && p.slot < 64) p.slot <<= 1;
    p.parts = (need + 63) / 64;
    p.lanes = g * p.slot * p.parts;
  }
  if (use_runs(rays, n_max, d)) {
    p.run_rows = n_max * p.lanes / (128 * 1024);  // two waves a SIMD (four: each reading 1 to 3 us shorter, the prefix 6 us longer)
    p.run_rows = (p.run_rows + kBlock - 1) / kBlock * kBlock;
    if (p.run_rows < 4 * kBlock) p.run_rows = 4 * kBlock;
    p.runs = (n_max + p.run_rows - 1) / p.run_rows;
  }
  return p;
}
// Two waves a SIMD with `vec` channels a lane: wider loads pay from there on (two channels / one, us, bf16 forward: 4096 rays x 192 rows x 128
// channels 154 / 170, 2 x 131072 x 64 45 / 50; below, 512 x 128 x 64 41 / 33, 4096 x 128 x 8 52 / 40).
bool enough_lanes(const ScanArgs& a, int vec) {
  const ScanPlan p = plan_scan(a.rays, a.n_max, a.d, a.g, vec);
  return (p.run_rows ? p.runs : a.rays) * p.lanes >= 128 * 1024;
}
// workspace: the runs' steps, df's sums over parts of gates
int64_t scan_workspace(int64_t rays, int64_t n_max, int d, int g) {
  int64_t runs = 0, parts = 0;
  for (int vec = 1; vec <= 2; vec++)
    if (d / (g == d ? 1 : g) % vec == 0) {
      const ScanPlan p = plan_scan(rays, n_max, d, g, vec);
      if (p.runs > runs) runs = p.runs;
      if (p.parts > parts) parts = p.parts;
    }
  return runs * d * (int64_t)sizeof(Step) + (parts > 1 ? parts * n_max * g * 4 : 0);
}

template <typename T, int GATE, int VEC, bool SHARED>
int launch_scan(ScanArgs a, bool bwd, char* ws, hipStream_t st) {
  const ScanPlan p = plan_scan(a.rays, a.n_max, a.d, a.g, VEC);
  a.slot = p.slot;
  a.parts = p.parts;
  a.lanes = p.lanes;
  a.run_rows = p.run_rows;
  a.runs = p.runs;
  a.agg = reinterpret_cast<Step*>(ws);
  a.partial = reinterpret_cast<float*>(ws + p.runs * a.d * sizeof(Step));
  const int64_t threads = (p.run_rows ? p.runs : a.rays) * p.lanes, blocks = (threads + kScanThreads - 1) / kScanThreads;
  GFN_CHECK_ARG(blocks < (1ll << 31), "gfn_ray_scan: %lld rays of %d channels are too many for one launch", (long long)a.rays, a.d);
  const unsigned grid = (unsigned)(blocks < 1 ? 1 : blocks);
  if (p.run_rows) {
    if (bwd) scan_bwd_kernel<T, GATE, VEC, SHARED, true><<<grid, kScanThreads, 0, st>>>(a);
    else scan_fwd_kernel<T, GATE, VEC, SHARED, true><<<grid, kScanThreads, 0, st>>>(a);
    GFN_CHECK_LAUNCH();
    run_prefix_kernel<<<(unsigned)a.d, 64 * kPrefixWaves, 0, st>>>(a.agg, p.runs);
    GFN_CHECK_LAUNCH();
  }
  if (bwd) scan_bwd_kernel<T, GATE, VEC, SHARED, false><<<grid, kScanThreads, 0, st>>>(a);
  else scan_fwd_kernel<T, GATE, VEC, SHARED, false><<<grid, kScanThreads, 0, st>>>(a);
  GFN_CHECK_LAUNCH();
  if (bwd && p.parts > 1 && a.n_max > 0) {
    const int64_t groups = (a.n_max * a.g + 255) / 256;
    scan_gate_sums_kernel<T><<<(unsigned)(groups < 4096 ? groups : 4096), 256, 0, st>>>(a, a.partial, p.parts);
    GFN_CHECK_LAUNCH();
  }
  return GFN_OK;
}

template <typename T, int GATE>
int dispatch_vec(const ScanArgs& a, bool bwd, char* ws, hipStream_t st) {
  const bool shared = a.g != a.d;
  if constexpr (sizeof(T) == 2) {  // two 16-bit channels a lane; f32: one is 256 bytes a wave already
    if (two_channels(a, shared, bwd) && enough_lanes(a, 2)) return shared ? launch_scan<T, GATE, 2, true>(a, bwd, ws, st) : launch_scan<T, GATE, 2, false>(a, bwd, ws, st);
  }
  return shared ? launch_scan<T, GATE, 1, true>(a, bwd, ws, st) : launch_scan<T, GATE, 1, false>(a, bwd, ws, st);
}
template <typename T>
int dispatch_gate(const ScanArgs& a, int gate, bool bwd, char* ws, hipStream_t st) {
  if (gate == GATE_LINEAR) return dispatch_vec<T, GATE_LINEAR>(a, bwd, ws, st);
  if (gate == GATE_SIGMOID) return dispatch_vec<T, GATE_SIGMOID>(a, bwd, ws, st);
  return dispatch_vec<T, GATE_DECAY>(a, bwd, ws, st);
}
int dispatch_scan(const char* who, const ScanArgs& a, int dtype, int gate, bool bwd, void* workspace, int64_t bytes, hipStream_t st) {
  const int64_t need = scan_workspace(a.rays, a.n_max, a.d, a.g);
  GFN_CHECK_ARG(bytes >= need && (need == 0 || workspace), "%s: workspace of %lld bytes, %lld needed", who, (long long)bytes, (long long)need);
  if (a.rays == 0 && !(a.clear && a.n_max > 0)) return GFN_OK;
  const int size = dtype == GFN_F32 ? 4 : 2;
  const int64_t n = a.n_max, states = a.rays * a.d, blocks = (n + kBlock - 1) / kBlock * a.d;
  if (int rc = gfn_check_apart(who,
                               {{"h", a.h, n, a.d, a.ldh, size}, {"df", a.df, n, a.g, a.lddf, size}, {"dc", a.dc, n, a.d, a.lddc, size}, gfn_flat("state", a.state, states, 4),
                                gfn_flat("saved", a.saved, blocks, 4), gfn_flat("dh0", a.dh0, states, 4), gfn_flat("the workspace", workspace, need, 1)},
                               {gfn_flat("pts_offsets", a.offsets, a.rays + 1, 4), {"f", a.f, n, a.g, a.ldf, size}, {"c", a.c, n, a.d, a.ldc, size}, {"dh", a.dh, n, a.d, a.lddh, size},
                                gfn_flat("h0", a.h0, states, 4), gfn_flat("d_state", a.d_state, states, 4), gfn_flat("saved", a.saved_in, blocks, 4)}))
    return rc;
  char* ws = static_cast<char*>(workspace);
  if (dtype == GFN_F32) return dispatch_gate<float>(a, gate, bwd, ws, st);
  if (dtype == GFN_BF16) return dispatch_gate<__bf16>(a, gate, bwd, ws, st);
  return dispatch_gate<_Float16>(a, gate, bwd, ws, st);
}

}  // namespace

extern "C" {

int64_t gfn_ray_scan_workspace(int64_t n_rays, int64_t n_max, int channels, int gates) {
  if (check_scan("gfn_ray_scan_workspace", n_rays, n_max, channels, gates, GFN_F32, 0, gates, channels)) return GFN_ERR_ARG;
  return scan_workspace(n_rays, n_max, channels, gates);
}

int gfn_ray_scan_fwd(const int32_t* pts_offsets, int64_t n_rays, const void* f, int64_t ldf, const void* c, int64_t ldc, int64_t n_max, int channels,
                     int gates, int dtype, int gate, int reverse, const float* h0, void* h, int64_t ldh, float* state, float* saved, int clear_tail,
                     void* workspace, int64_t workspace_bytes, void* stream) {
  if (int rc = check_scan("gfn_ray_scan_fwd", n_rays, n_max, channels, gates, dtype, gate, ldf, ldc)) return rc;
  GFN_CHECK_ARG(pts_offsets && (n_max == 0 || (f && c && h)), "gfn_ray_scan_fwd: null pointer");
  GFN_CHECK_ARG(ldh >= channels, "gfn_ray_scan_fwd: a row stride is below the row's width");
  ScanArgs a{};
  a.offsets = pts_offsets; a.rays = n_rays; a.n_max = n_max;
  a.f = f; a.ldf = ldf; a.c = c; a.ldc = ldc; a.h = h; a.ldh = ldh;
  a.d = channels; a.g = gates; a.per_gate = channels / gates; a.reverse = reverse != 0;
  a.h0 = h0; a.state = state; a.saved = saved;
  a.clear = clear_tail != 0;
  return dispatch_scan("gfn_ray_scan_fwd", a, dtype, gate, false, workspace, workspace_bytes, gfn_stream(stream));
}

int gfn_ray_scan_bwd(const int32_t* pts_offsets, int64_t n_rays, const void* f, int64_t ldf, const void* c, int64_t ldc, const void* dh, int64_t lddh,
                     int64_t n_max, int channels, int gates, int dtype, int gate, int reverse, const float* h0, const float* d_state, const float* saved,
                     void* df, int64_t lddf, void* dc, int64_t lddc, float* dh0, int clear_tail, void* workspace,
                     int64_t workspace_bytes, void* stream) {
  if (int rc = check_scan("gfn_ray_scan_bwd", n_rays, n_max, channels, gates, dtype, gate, ldf, ldc)) return rc;
  GFN_CHECK_ARG(pts_offsets && (n_max == 0 || (f && c && dh && saved && df && dc)), "gfn_ray_scan_bwd: null pointer");
  GFN_CHECK_ARG(lddh >= channels && lddf >= gates && lddc >= channels, "gfn_ray_scan_bwd: a row stride is below the row's width");
  ScanArgs a{};
  a.offsets = pts_offsets; a.rays = n_rays; a.n_max = n_max;
  a.f = f; a.ldf = ldf; a.c = c; a.ldc = ldc; a.dh = dh; a.lddh = lddh;
  a.d = channels; a.g = gates; a.per_gate = channels / gates; a.reverse = reverse != 0;
  a.h0 = h0; a.d_state = d_state; a.saved_in = saved;
  a.df = df; a.lddf = lddf; a.dc = dc; a.lddc = lddc; a.dh0 = dh0;
  a.clear = clear_tail != 0;
  return dispatch_scan("gfn_ray_scan_bwd", a, dtype, gate, true, workspace, workspace_bytes, gfn_stream(stream));
}

int gfn_ray_scan_step(const void* f, int64_t ldf, const void* c, int64_t ldc, int64_t n_rays, int channels, int gates, int dtype, int gate, float* state,
                      void* h, int64_t ldh, void* stream) {
  if (int rc = check_scan("gfn_ray_scan_step", n_rays, n_rays, channels, gates, dtype, gate, ldf, ldc)) return rc;
  if (n_rays == 0) return GFN_OK;
  GFN_CHECK_ARG(f && c && state && h, "gfn_ray_scan_step: null pointer");
  GFN_CHECK_ARG(ldh >= channels, "gfn_ray_scan_step: a row stride is below the row's width");
  ScanArgs a{};
  a.rays = n_rays; a.f = f; a.ldf = ldf; a.c = c; a.ldc = ldc; a.h = h; a.ldh = ldh; a.state = state;
  a.d = channels; a.g = gates; a.per_gate = channels / gates;
  // a thread reads its row's gate and its channel of c and of the state and writes state and h: what lies in the same places may be the same
  const int size = dtype == GFN_F32 ? 4 : 2;
  const gfn_rows rf{"f", f, n_rays, gates, ldf, size}, rc{"c", c, n_rays, channels, ldc, size}, rh{"h", h, n_rays, channels, ldh, size}, rs{"state", state, n_rays, channels, channels, 4};
  if (int e = gfn_check_apart("gfn_ray_scan_step", {rh, rs}, {gates == channels && gfn_same_rows(rs, rf) ? gfn_rows{} : rf})) return e;
  GFN_CHECK_ARG(gfn_same_rows(rh, rc) || !gfn_overlap(rh, rc), "gfn_ray_scan_step: h overlaps c");
  GFN_CHECK_ARG(gfn_same_rows(rs, rc) || !gfn_overlap(rs, rc), "gfn_ray_scan_step: state overlaps c");
  const int64_t blocks = (n_rays * channels + 255) / 256;
  const unsigned grid = (unsigned)(blocks < 8192 ? blocks : 8192);
  hipStream_t st = gfn_stream(stream);
#define GFN_STEP(T)                                                                     \
  if (gate == GATE_LINEAR) scan_step_kernel<T, GATE_LINEAR><<<grid, 256, 0, st>>>(a);    \
  else if (gate == GATE_SIGMOID) scan_step_kernel<T, GATE_SIGMOID><<<grid, 256, 0, st>>>(a); \
  else scan_step_kernel<T, GATE_DECAY><<<grid, 256, 0, st>>>(a)
  if (dtype == GFN_F32) { GFN_STEP(float); }
  else if (dtype == GFN_BF16) { GFN_STEP(__bf16); }
  else { GFN_STEP(_Float16); }
#undef GFN_STEP
  GFN_CHECK_LAUNCH();
  return GFN_OK;
}

}  // extern "C"
