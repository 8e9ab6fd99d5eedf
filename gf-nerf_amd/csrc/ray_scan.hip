// ray_scan.hip -- the gated linear recurrence along the packed samples of each ray,
//     h_t = a_t h_{t-1} + b_t ,   h_{-1} = h0 (or 0),
// front to back or back to front, its backward pass, and its form for one sample of every ray.  f [N, G] gates, c [N, D] inputs; gate
// d / (D / G) belongs to channel d:
//     linear   a = f              b = c
//     sigmoid  a = sigmoid(f)     b = (1 - a) c
//     decay    a = exp(-f)        b = (1 - a) c        (f = optical thickness: back to front this is alpha compositing of D channels)
// Backward:  l_t = dh_t + a_{t+1} l_{t+1} (the last row's: + d_state);  dc = l (1 - a) (linear: l);  df = l (h_{t-1} - c) da/df (linear:
// l h_{t-1}), summed over the channels of a gate;  dh0 = a_first l_first.  h_{t-1} is not read back: the forward leaves the f32 state it
// had on entering every aligned block of 16 rows (1/8 of the bytes of a 16-bit h, and nothing is rounded), and the backward walks each
// block forward from there in registers before it walks it backward.
//
// A lane owns VEC channels of one ray and walks the ray's rows; the 16 rows of a block are requested together, so the recurrence's
// chain of multiply-adds runs on data that has arrived.  State and adjoint are f32.
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
    const float e = exp_of<EXACT>(-__builtin_fabsf(f));
    const float r = EXACT ? 1.f / (1.f + e) : __builtin_amdgcn_rcpf(1.f + e);
    a = f >= 0.f ? r : e * r;
    rest = f >= 0.f ? e * r : r;
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
  int slot;      // lanes a (ray, gate) takes when gates are shared: a power of two >= the lanes it needs
  int per_gate;  // channels of a gate
};

// this thread's ray and first channel; false: nothing to do (the lanes of a slot that no channel fills stay for the reductions)
template <int VEC, bool SHARED>
__device__ __forceinline__ bool scan_place(const ScanArgs& a, int64_t& ray, int& ch, int& gate, bool& active) {
  const int64_t id = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if constexpr (SHARED) {
    const int64_t s = id / a.slot;
    ray = s / a.g;
    gate = (int)(s - ray * a.g);
    const int at = (int)(id & (a.slot - 1)) * VEC;
    ch = gate * a.per_gate + at;
    active = at < a.per_gate;
  } else {
    const int lanes = a.d / VEC;
    ray = id / lanes;
    ch = (int)(id - ray * lanes) * VEC;
    gate = ch;
    active = true;
  }
  return ray < a.rays;
}

__device__ __forceinline__ void ray_rows(const ScanArgs& a, int64_t ray, int64_t& start, int64_t& end) {  // inside the arrays, whatever the offsets say
  start = a.offsets[ray];
  end = a.offsets[ray + 1];
  start = start < 0 ? 0 : (start > a.n_max ? a.n_max : start);
  end = end < start ? start : (end > a.n_max ? a.n_max : end);
}

template <typename T, int GATE, int VEC, bool SHARED>
__global__ __launch_bounds__(256) void scan_fwd_kernel(ScanArgs a) {
  constexpr bool EXACT = sizeof(T) == 4;
  using V = Vec<T, VEC>;
  int64_t ray, start, end;
  int ch, gate;
  bool active;
  if (!scan_place<VEC, SHARED>(a, ray, ch, gate, active) || !active) return;
  ray_rows(a, ray, start, end);
  const T *f = static_cast<const T*>(a.f) + gate, *c = static_cast<const T*>(a.c) + ch;
  T* h = static_cast<T*>(a.h) + ch;
  float s[VEC];
#pragma unroll
  for (int v = 0; v < VEC; v++) s[v] = a.h0 ? a.h0[ray * a.d + ch + v] : 0.f;
  const int64_t b0 = start / kBlock, blocks = end > start ? (end - 1) / kBlock - b0 + 1 : 0;
  for (int64_t i = 0; i < blocks; i++) {
    const int64_t base = (a.reverse ? b0 + blocks - 1 - i : b0 + i) * kBlock;
    const int64_t lo = base > start ? base : start, hi = base + kBlock < end ? base + kBlock : end;
    if (a.saved && i)
#pragma unroll
      for (int v = 0; v < VEC; v++) a.saved[base / kBlock * a.d + ch + v] = s[v];
    V fr[kBlock], cr[kBlock];
#pragma unroll
    for (int r = 0; r < kBlock; r++) {
      int64_t row = base + (a.reverse ? kBlock - 1 - r : r);
      row = row < lo ? lo : (row >= hi ? hi - 1 : row);
      if constexpr (SHARED) fr[r].v[0] = f[row * a.ldf];
      else fr[r] = *reinterpret_cast<const V*>(f + row * a.ldf);
      cr[r] = *reinterpret_cast<const V*>(c + row * a.ldc);
    }
#pragma unroll
    for (int r = 0; r < kBlock; r++) {
      const int64_t row = base + (a.reverse ? kBlock - 1 - r : r);
      if (row >= lo && row < hi) {
        V out;
        float ga, rest;
#pragma unroll
        for (int v = 0; v < VEC; v++) {
          if (!SHARED || v == 0) gate_of<GATE, EXACT>((float)fr[r].v[v], ga, rest);
          s[v] = __builtin_fmaf(ga, s[v], rest * (float)cr[r].v[v]);
          out.v[v] = (T)s[v];
        }
        *reinterpret_cast<V*>(h + row * a.ldh) = out;
      }
    }
  }
  if (a.state)
#pragma unroll
    for (int v = 0; v < VEC; v++) a.state[ray * a.d + ch + v] = s[v];
}

template <typename T, int GATE, int VEC, bool SHARED>
__global__ __launch_bounds__(256) void scan_bwd_kernel(ScanArgs a) {
  constexpr bool EXACT = sizeof(T) == 4;
  using V = Vec<T, VEC>;
  int64_t ray, start = 0, end = 0;
  int ch, gate;
  bool active;
  const bool here = scan_place<VEC, SHARED>(a, ray, ch, gate, active);
  if (!SHARED && !here) return;
  if (here) ray_rows(a, ray, start, end);
  active = active && here;
  if (!here) gate = ch = 0;
  const int cl = active ? ch : 0;  // a lane without a channel reads channel 0 and counts for nothing
  const T *f = static_cast<const T*>(a.f) + gate, *c = static_cast<const T*>(a.c) + cl, *dh = static_cast<const T*>(a.dh) + cl;
  T *df = static_cast<T*>(a.df) + gate, *dc = static_cast<T*>(a.dc) + ch;
  float l[VEC], first[VEC];
#pragma unroll
  for (int v = 0; v < VEC; v++) {
    l[v] = active && a.d_state ? a.d_state[ray * a.d + ch + v] : 0.f;
    first[v] = active && a.h0 ? a.h0[ray * a.d + ch + v] : 0.f;
  }
  const int64_t b0 = start / kBlock, blocks = end > start ? (end - 1) / kBlock - b0 + 1 : 0;
  for (int64_t i = blocks - 1; i >= 0; i--) {  // the recurrence's last block first
    const int64_t base = (a.reverse ? b0 + blocks - 1 - i : b0 + i) * kBlock;
    const int64_t lo = base > start ? base : start, hi = base + kBlock < end ? base + kBlock : end;
    V fr[kBlock], cr[kBlock], dr[kBlock];
#pragma unroll
    for (int r = 0; r < kBlock; r++) {
      int64_t row = base + (a.reverse ? kBlock - 1 - r : r);
      row = row < lo ? lo : (row >= hi ? hi - 1 : row);
      if constexpr (SHARED) fr[r].v[0] = f[row * a.ldf];
      else fr[r] = *reinterpret_cast<const V*>(f + row * a.ldf);
      cr[r] = *reinterpret_cast<const V*>(c + row * a.ldc);
      dr[r] = *reinterpret_cast<const V*>(dh + row * a.lddh);
    }
    float before[kBlock][VEC], s[VEC];  // the state in front of each row
#pragma unroll
    for (int v = 0; v < VEC; v++) s[v] = i ? a.saved_in[base / kBlock * a.d + cl + v] : first[v];
#pragma unroll
    for (int r = 0; r < kBlock; r++) {
      const int64_t row = base + (a.reverse ? kBlock - 1 - r : r);
      float ga, rest;
#pragma unroll
      for (int v = 0; v < VEC; v++) {
        before[r][v] = s[v];
        if (!SHARED || v == 0) gate_of<GATE, EXACT>((float)fr[r].v[v], ga, rest);
        if (row >= lo && row < hi) s[v] = __builtin_fmaf(ga, s[v], rest * (float)cr[r].v[v]);
      }
    }
#pragma unroll
    for (int r = kBlock - 1; r >= 0; r--) {
      const int64_t row = base + (a.reverse ? kBlock - 1 - r : r);
      if (row >= lo && row < hi) {
        V oc, of;
        float ga, rest, sum = 0.f;
#pragma unroll
        for (int v = 0; v < VEC; v++) {
          if (!SHARED || v == 0) gate_of<GATE, EXACT>((float)fr[r].v[v], ga, rest);
          const float lt = l[v] + (float)dr[r].v[v], cv = (float)cr[r].v[v];
          float d;
          if constexpr (GATE == GATE_LINEAR) d = lt * before[r][v];
          else if constexpr (GATE == GATE_SIGMOID) d = lt * (before[r][v] - cv) * (ga * rest);
          else d = lt * (cv - before[r][v]) * ga;
          oc.v[v] = (T)(lt * rest);
          if constexpr (SHARED) sum += d;
          else of.v[v] = (T)d;
          l[v] = ga * lt;
        }
        if (active) *reinterpret_cast<V*>(dc + row * a.lddc) = oc;
        if constexpr (SHARED) {
          if (!active) sum = 0.f;
          for (int o = a.slot >> 1; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
          if ((threadIdx.x & (a.slot - 1)) == 0) df[row * a.lddf] = (T)sum;
        } else {
          *reinterpret_cast<V*>(df + row * a.lddf) = of;
        }
      }
    }
  }
  if (a.dh0 && active)
#pragma unroll
    for (int v = 0; v < VEC; v++) a.dh0[ray * a.d + ch + v] = l[v];
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

// rows behind the last ray's last -> 0
template <typename T>
__global__ __launch_bounds__(256) void zero_tail_kernel(const int32_t* __restrict__ offsets, int64_t rays, int64_t n_max, T* __restrict__ p, int64_t ld, int width) {
  int64_t begin = offsets[rays];
  begin = begin < 0 ? 0 : begin;
  for (int64_t e = begin * width + (int64_t)blockIdx.x * 256 + threadIdx.x; e < n_max * width; e += (int64_t)gridDim.x * 256) p[e / width * ld + e % width] = (T)0.f;
}

// ---- host ---------------------------------------------------------------------------------------------------------------------------
int check_scan(const char* who, int64_t rays, int64_t n_max, int d, int g, int dtype, int gate, int64_t ldf, int64_t ldc) {
  GFN_CHECK_ARG(rays >= 0 && rays < (1ll << 31) && n_max >= 0 && n_max < (1ll << 31), "%s: %lld rays, n_max %lld", who, (long long)rays, (long long)n_max);
  GFN_CHECK_ARG(d >= 1 && d <= GFN_SCAN_MAX_CHANNELS && g >= 1 && g <= d && d % g == 0, "%s: %d gates for %d channels (1..%d channels, the gates dividing them)", who, g, d,
                GFN_SCAN_MAX_CHANNELS);
  GFN_CHECK_ARG(d / g <= 256 || g == d, "%s: %d channels share a gate (at most 256)", who, d / g);
  GFN_CHECK_ARG(dtype >= GFN_F32 && dtype <= GFN_F16, "%s: dtype %d", who, dtype);
  GFN_CHECK_ARG(gate >= 0 && gate <= 2, "%s: gate %d", who, gate);
  GFN_CHECK_ARG(ldf >= g && ldc >= d, "%s: a row stride is below the row's width", who);
  return GFN_OK;
}

// channels a lane: as wide as every pointer, stride and gate group allows
int pick_vec(const ScanArgs& a, int size, bool shared, bool bwd) {
  const int per = shared ? a.per_gate : a.d;
  for (int vec = shared && per > 128 ? 4 : 2; vec > 1; vec >>= 1) {
    const int64_t strides = a.ldc | (bwd ? a.lddh | a.lddc : a.ldh) | (shared ? 0 : a.ldf | (bwd ? a.lddf : 0));
    uintptr_t at = reinterpret_cast<uintptr_t>(a.c) | (bwd ? reinterpret_cast<uintptr_t>(a.dh) | reinterpret_cast<uintptr_t>(a.dc) : reinterpret_cast<uintptr_t>(a.h));
    if (!shared) at |= reinterpret_cast<uintptr_t>(a.f) | (bwd ? reinterpret_cast<uintptr_t>(a.df) : 0);
    if (per % vec == 0 && strides % vec == 0 && at % ((uintptr_t)vec * size) == 0) return vec;
  }
  return 1;
}

template <typename T, int GATE, int VEC, bool SHARED>
int launch_scan(ScanArgs a, bool bwd, hipStream_t st) {
  int64_t threads;
  if (SHARED) {
    const int need = (a.per_gate + VEC - 1) / VEC;
    a.slot = 1;
    while (a.slot < need) a.slot <<= 1;
    threads = a.rays * a.g * a.slot;
  } else {
    threads = a.rays * (a.d / VEC);
  }
  const int64_t blocks = (threads + 255) / 256;
  GFN_CHECK_ARG(blocks < (1ll << 31), "gfn_ray_scan: %lld rays of %d channels are too many for one launch", (long long)a.rays, a.d);
  if (bwd) scan_bwd_kernel<T, GATE, VEC, SHARED><<<(unsigned)blocks, 256, 0, st>>>(a);
  else scan_fwd_kernel<T, GATE, VEC, SHARED><<<(unsigned)blocks, 256, 0, st>>>(a);
  GFN_CHECK_LAUNCH();
  return GFN_OK;
}

template <typename T, int GATE>
int dispatch_vec(const ScanArgs& a, bool bwd, hipStream_t st) {
  const bool shared = a.g != a.d;
  const int vec = pick_vec(a, sizeof(T), shared, bwd);
  if (!shared) return vec == 2 ? launch_scan<T, GATE, 2, false>(a, bwd, st) : launch_scan<T, GATE, 1, false>(a, bwd, st);
  GFN_CHECK_ARG((a.per_gate + vec - 1) / vec <= 64, "gfn_ray_scan: %d channels share a gate, but their rows are not aligned to %d elements (at most 64 a gate then)",
                a.per_gate, a.per_gate > 128 ? 4 : 2);
  if (vec == 4) return launch_scan<T, GATE, 4, true>(a, bwd, st);
  return vec == 2 ? launch_scan<T, GATE, 2, true>(a, bwd, st) : launch_scan<T, GATE, 1, true>(a, bwd, st);
}
template <typename T>
int dispatch_gate(const ScanArgs& a, int gate, bool bwd, hipStream_t st) {
  if (gate == GATE_LINEAR) return dispatch_vec<T, GATE_LINEAR>(a, bwd, st);
  if (gate == GATE_SIGMOID) return dispatch_vec<T, GATE_SIGMOID>(a, bwd, st);
  return dispatch_vec<T, GATE_DECAY>(a, bwd, st);
}
int dispatch_scan(const ScanArgs& a, int dtype, int gate, bool bwd, hipStream_t st) {
  if (a.rays == 0) return GFN_OK;
  if (dtype == GFN_F32) return dispatch_gate<float>(a, gate, bwd, st);
  if (dtype == GFN_BF16) return dispatch_gate<__bf16>(a, gate, bwd, st);
  return dispatch_gate<_Float16>(a, gate, bwd, st);
}

int zero_tail(const ScanArgs& a, int dtype, void* p, int64_t ld, int width, hipStream_t st) {
  if (a.n_max == 0) return GFN_OK;
  const int64_t blocks = (a.n_max * width + 2047) / 2048;
  const unsigned grid = (unsigned)(blocks < 1024 ? blocks : 1024);
  if (dtype == GFN_F32) zero_tail_kernel<float><<<grid, 256, 0, st>>>(a.offsets, a.rays, a.n_max, static_cast<float*>(p), ld, width);
  else zero_tail_kernel<_Float16><<<grid, 256, 0, st>>>(a.offsets, a.rays, a.n_max, static_cast<_Float16*>(p), ld, width);
  GFN_CHECK_LAUNCH();
  return GFN_OK;
}

}  // namespace

extern "C" {

int gfn_ray_scan_fwd(const int32_t* pts_offsets, int64_t n_rays, const void* f, int64_t ldf, const void* c, int64_t ldc, int64_t n_max, int channels,
                     int gates, int dtype, int gate, int reverse, const float* h0, void* h, int64_t ldh, float* state, float* saved, int clear_tail, void* stream) {
  if (int rc = check_scan("gfn_ray_scan_fwd", n_rays, n_max, channels, gates, dtype, gate, ldf, ldc)) return rc;
  GFN_CHECK_ARG(pts_offsets && (n_max == 0 || (f && c && h)), "gfn_ray_scan_fwd: null pointer");
  GFN_CHECK_ARG(ldh >= channels, "gfn_ray_scan_fwd: a row stride is below the row's width");
  ScanArgs a{};
  a.offsets = pts_offsets; a.rays = n_rays; a.n_max = n_max;
  a.f = f; a.ldf = ldf; a.c = c; a.ldc = ldc; a.h = h; a.ldh = ldh;
  a.d = channels; a.g = gates; a.per_gate = channels / gates; a.reverse = reverse != 0;
  a.h0 = h0; a.state = state; a.saved = saved;
  if (int rc = dispatch_scan(a, dtype, gate, false, gfn_stream(stream))) return rc;
  return clear_tail ? zero_tail(a, dtype, h, ldh, channels, gfn_stream(stream)) : GFN_OK;
}

int gfn_ray_scan_bwd(const int32_t* pts_offsets, int64_t n_rays, const void* f, int64_t ldf, const void* c, int64_t ldc, const void* dh, int64_t lddh,
                     int64_t n_max, int channels, int gates, int dtype, int gate, int reverse, const float* h0, const float* d_state, const float* saved,
                     void* df, int64_t lddf, void* dc, int64_t lddc, float* dh0, int clear_tail, void* stream) {
  if (int rc = check_scan("gfn_ray_scan_bwd", n_rays, n_max, channels, gates, dtype, gate, ldf, ldc)) return rc;
  GFN_CHECK_ARG(pts_offsets && (n_max == 0 || (f && c && dh && saved && df && dc)), "gfn_ray_scan_bwd: null pointer");
  GFN_CHECK_ARG(lddh >= channels && lddf >= gates && lddc >= channels, "gfn_ray_scan_bwd: a row stride is below the row's width");
  ScanArgs a{};
  a.offsets = pts_offsets; a.rays = n_rays; a.n_max = n_max;
  a.f = f; a.ldf = ldf; a.c = c; a.ldc = ldc; a.dh = dh; a.lddh = lddh;
  a.d = channels; a.g = gates; a.per_gate = channels / gates; a.reverse = reverse != 0;
  a.h0 = h0; a.d_state = d_state; a.saved_in = saved;
  a.df = df; a.lddf = lddf; a.dc = dc; a.lddc = lddc; a.dh0 = dh0;
  if (int rc = dispatch_scan(a, dtype, gate, true, gfn_stream(stream))) return rc;
  if (!clear_tail) return GFN_OK;
  if (int rc = zero_tail(a, dtype, df, lddf, gates, gfn_stream(stream))) return rc;
  return zero_tail(a, dtype, dc, lddc, channels, gfn_stream(stream));
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
