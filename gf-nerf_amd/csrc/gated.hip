// gated.hip -- the gated feed-forward layer  h = act(x Wg^T + bg) * (x Wu^T + bu)  and its backward pass.
//
// Forward.  Weights are the MFMA's A operand (rows = hidden features), samples its columns, so a lane owns ONE sample and, with
// the feature rows of two 16-row tiles dealt out as 32 p + 8 (i >> 2) + 4 t + (i & 3), eight CONSECUTIVE features of it for both
// projections: activation and product happen in its registers and leave as one 16-byte store (four lanes write 64 bytes of a row).
// The weights of a block of features sit in LDS for the life of the workgroup; a wave keeps the inputs of 16 G samples in
// registers and passes over the features once.  Nothing but x, the weights and h touches memory.
//
// Backward.  g and u are formed again (they are cheaper than the two N x H arrays a saved forward would read back), then
//   dg = dh u act'(g), du = dh act(g)          in registers, eight consecutive features of a sample in each lane -- which is the
//   dx = dg Wg + du Wu                         B operand of this product as it stands (contraction over the features; the A operand
//                                              is W transposed, read from the same LDS image with transposing reads);
//   [dWg; dWu] = [dg; du]^T x                  contracts over the samples: the wave's dz goes to LDS and every wave accumulates its own
//                                              rows of dW over all samples of the tile, in registers until the workgroup's last tile.
// One pass: x and dh are read once, dx is written once; each workgroup's partial dW goes to a workspace and a second launch adds the
// partials in a fixed order (no atomics: the same bits every run).  The biases' gradients are the same product against a column of ones
// and travel as column k of the partials.
// 16-bit: dz goes into both products as several operands of the type (dz_operands), not rounded to one.  bf16: three, which are dz itself;
// of 33 million values of dx in the case below 5,300 then differ from their rounded 64-bit values (f32 torch: 7,600; two operands, 17 bits:
// 80,000, and one: two in five), for 180 us instead of 141 and 115 a call.  f16: two, 22 bits, under powers of two taken from
// the |dz| themselves (power_of); 28,400 of 12.8 million values of dx at 100k x 128 -> 128 differ (f32 torch: 28,200; a power
// from |dh| alone: 79,000), for 91 instead of 84 us.
//
// What bounds them (times without a profiler, shares of the kernel's cycles from counters: matrix pipe, vector issue, LDS).
// Forward, 786k x 63 -> 128 bf16 silu: 92 us for 300 MB (a copy of that size: 55); four waves a SIMD, requests a tile ahead.  No unit is full
// (11, 43, 10 %); rows that start at any 2 bytes cost 16 % (64 columns), and what holds the rest is not known.  262k x 32 -> 128 f32 gelu:
// 65 us; products (f32's run at 1/8 of bf16's rate) take 41 % and vector instructions 44 %, one after the other for the most part.
// Backward, two waves a SIMD (W's image, x, dz and dW's accumulators fill LDS and registers), whose vector instructions, LDS reads and
// products add up rather than overlap.  524k x 63 -> 128 bf16: 180 us a call, the reduction's 7 included, for 266 MB (a copy: 49); 31, 46 and
// 48 %.  100k x 128 -> 128 f16: 91 with the reduction's 13, four rounds of tiles for 3.05 of samples; 17, 35 and 27 %.  50k x 32 -> 64 f32: 29
// + 5, two rounds for 1.5; 23, 16 and 10 %.
#include "gated_device.h"

namespace {

constexpr int kWaves = 4;

// Waits for the rows requested ahead, before this tile's last results are stored: loads and stores are counted together and in order, so a
// wait for those rows behind the stores would be a wait for the stores.
__device__ __forceinline__ void loads_done() { __builtin_amdgcn_s_waitcnt(0x0f70); }

template <int V>
struct Constant {
  static constexpr int value = V;
};
// f for the activation's own constant: the choice is made once, outside of what f does.
template <typename F>
__device__ __forceinline__ void for_act(int act, F f) {
  switch (act) {
    case GATED_SILU: return f(Constant<GATED_SILU>{});
    case GATED_GELU: return f(Constant<GATED_GELU>{});
    case GATED_RELU: return f(Constant<GATED_RELU>{});
    default: return f(Constant<GATED_SIGMOID>{});
  }
}

// row i of tile t <-> hidden feature 32 p + 8 (i >> 2) + 4 t + (i & 3); the LDS image keeps rows in tile order
__device__ __forceinline__ int image_feature(int row) { return (row & ~31) + 8 * ((row & 15) >> 2) + 4 * ((row >> 4) & 1) + (row & 3); }

// [2 matrices][HC rows][KS units + one piece]: the odd number of pieces a row keeps 16 rows' equal pieces on different banks.
template <typename T, int KS>
__device__ __forceinline__ void stage_weights(char* lds, const T* wg, const T* wu, int k, int h, int h0, int hc) {
  constexpr int PIECES = 4 * KS, ROW = PIECES * 16 + 16;
  for (int e = threadIdx.x; e < 2 * hc * PIECES; e += blockDim.x) {
    const int row = e / PIECES, c = e - row * PIECES, m = row >= hc;
    const int f = h0 + image_feature(row - m * hc);
    *reinterpret_cast<u32x4*>(lds + row * ROW + c * 16) = f < h ? row_piece(((m ? wu : wg) + (int64_t)f * k), c, k) : u32x4{0u, 0u, 0u, 0u};
  }
}
// the biases as f32, [2][hc] in the images' order (zeros without): where the accumulators start
template <typename T>
__device__ __forceinline__ void stage_bias(float* bias, const T* bg, const T* bu, int h, int h0, int hc) {
  for (int e = threadIdx.x; e < 2 * hc; e += blockDim.x) {
    const int m = e >= hc, f = h0 + image_feature(e - m * hc);
    bias[e] = bg && f < h ? (float)(m ? bu : bg)[f] : 0.f;
  }
}

// workgroups of the forward that share a CU: registers for four, or for two where the rows are long.  (A launch without the bound keeps its
// accumulators apart from the vector registers and copies them: 117 us instead of 105 for 786k x 63 -> 128 bf16.)
constexpr int fwd_per_cu(int ks) { return ks <= 2 ? 4 : 2; }

template <typename T, int KS, int G>
__global__ __launch_bounds__(64 * kWaves, fwd_per_cu(KS)) void gated_fwd_kernel(int64_t n_max, const int32_t* __restrict__ n_dev, const T* __restrict__ x, int64_t ldx,
                                                               const T* __restrict__ wg, const T* __restrict__ wu, const T* __restrict__ bg,
                                                               const T* __restrict__ bu, int k, int h, int hc, int act, T* __restrict__ out, int64_t ldo) {
  constexpr int ROW = KS * 64 + 16;
  constexpr bool EXACT = sizeof(T) == 4;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  float* bias = reinterpret_cast<float*>(lds + 2 * hc * ROW);  // [2][hc] in tile order
  const int h0 = blockIdx.y * hc;
  stage_weights<T, KS>(lds, wg, wu, k, h, h0, hc);
  stage_bias(bias, bg, bu, h, h0, hc);
  __syncthreads();
  const int64_t n = gfn_live_n(n_max, n_dev);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = lane & 15, kg = lane >> 4;
  const int pairs = ((h - h0 < hc ? h - h0 : hc) + 31) / 32;
  const char* wrow = lds + j * ROW + kg * 16;
  const int64_t stride = (int64_t)gridDim.x * kWaves * 16 * G;
  int64_t s0 = ((int64_t)blockIdx.x * kWaves + wave) * 16 * G;
  const int cut = cut_piece<T>(k);
  u32x4 xr[G][KS], next[G][KS];
  auto fetch = [&](u32x4 (&to)[G][KS], int64_t first) {
#pragma unroll
    for (int g = 0; g < G; g++) {
      const int64_t s = first + 16 * g + j;
#pragma unroll
      for (int u = 0; u < KS; u++) to[g][u] = s < n ? piece_request(x + s * ldx, 4 * u + kg, k) : u32x4{0u, 0u, 0u, 0u};
    }
  };
  if (s0 < n) fetch(next, s0);
  auto pass = [&](auto act_c) {
    for (; s0 < n; s0 += stride) {
#pragma unroll
      for (int g = 0; g < G; g++)
#pragma unroll
        for (int u = 0; u < KS; u++) {
          xr[g][u] = next[g][u];
          if (u == cut >> 2 && kg == (cut & 3)) xr[g][u] = piece_shift<T>(next[g][u], k);
        }
      if (s0 + stride < n) fetch(next, s0 + stride);  // on its way under this tile's work
      for (int p = 0; p < pairs; p++) {
        f32x4 acc[2][2][G];  // [matrix][tile]
#pragma unroll
        for (int m = 0; m < 2; m++)
#pragma unroll
          for (int t = 0; t < 2; t++) {
            const f32x4 b = *reinterpret_cast<const f32x4*>(bias + m * hc + 32 * p + 16 * t + 4 * kg);
#pragma unroll
            for (int g = 0; g < G; g++) acc[m][t][g] = b;
          }
#pragma unroll
        for (int u = 0; u < KS; u++)
#pragma unroll
          for (int m = 0; m < 2; m++)
#pragma unroll
            for (int t = 0; t < 2; t++) {
              const u32x4 w = *reinterpret_cast<const u32x4*>(wrow + (m * hc + 32 * p + 16 * t) * ROW + u * 64);
#pragma unroll
              for (int g = 0; g < G; g++) acc[m][t][g] = mma(w, xr[g][u], acc[m][t][g], (T*)nullptr);
            }
        const int f = h0 + 32 * p + 8 * kg;
#pragma unroll
        for (int g = 0; g < G; g++) {
          const int64_t s = s0 + 16 * g + j;
          float v[8];
          gated8<decltype(act_c)::value, EXACT>([&](int i) { return acc[0][i >> 2][g][i & 3]; }, [&](int i) { return acc[1][i >> 2][g][i & 3]; }, v);
          if (s < n) store_row<T, 8>(out + s * ldo + f, h - f, v);
        }
      }
    }
  };
  for_act(act, pass);
}

// ---- backward ---------------------------------------------------------------------------------------------------------------------
// The powers of two that f16 operands of dz are formed under.  A sample's dz of one pair of feature tiles have their own: the multiple of 8 that
// brings their largest into [2^7, 2^15).  Nothing overflows, two operands hold 22 bits of a number, and what f16's grid of 2^-24 cuts off is
// small beside that largest.
// dx: one column of its product is one sample, whose sums stand under the lowest power of its pairs so far (rescaled where that falls).  So a
// sample's gradient does not depend on its neighbours, and at most 2^-30 of its largest |dz| is cut off of a term.
// dW contracts over the samples of a tile, whose dz of a pair share the lowest of their powers: at most 2^-30 of the tile's largest is cut off (a
// term below 2^-8 of it loses bits that f32 would hold, one below 2^-19 of it bits that f16 would).  The sums over the tiles are rescaled
// where it moves; it never rises more than 2^64 above its lowest, so that they stay in f32.
constexpr int kTopPower = 96, kNoPower = 104;  // no dz but zeros: no power
__device__ __forceinline__ int power_of(float largest) {
  const int e = (15 - __builtin_amdgcn_frexp_expf(largest)) & ~7;  // largest < 2^frexp_exp
  return largest == 0.f ? kNoPower : e < kTopPower ? e : kTopPower;
}
__device__ __forceinline__ float pow2(int e) { return __builtin_bit_cast(float, (uint32_t)(127 + e) << 23); }
__device__ __forceinline__ void rescale(f32x4& v, int by) {
#pragma unroll
  for (int i = 0; i < 4; i++) v[i] = __builtin_amdgcn_ldexpf(v[i], by);
}
// the lowest of e over the lanes that share lane >> 4: neighbours, pairs of them, the half row and the row mirrored
template <int CTRL>
__device__ __forceinline__ int min_with(int e) {
  const int o = __builtin_amdgcn_mov_dpp(e, CTRL, 0xf, 0xf, true);
  return o < e ? o : e;
}
__device__ __forceinline__ int min_over_sixteen(int e) { return min_with<0x140>(min_with<0x141>(min_with<0x4e>(min_with<0xb1>(e)))); }
// eight f16 times 2^by, by <= 0, in two steps: 2^by itself may be below f16's range where the products are not.  (2^-48 takes everything finite
// to zero, and leaves infinities.)
__device__ __forceinline__ u32x4 times_pow2(u32x4 v, int by) {
  by = by < -48 ? -48 : by;
  const _Float16 f = (_Float16)pow2(by >> 1), g = (_Float16)pow2(by - (by >> 1));
  const f16x8 r = __builtin_bit_cast(f16x8, v) * f16x8{f, f, f, f, f, f, f, f} * f16x8{g, g, g, g, g, g, g, g};
  return __builtin_bit_cast(u32x4, r);
}
// the largest finite |z|
__device__ __forceinline__ float largest_of(const float (&z)[2][8]) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 8; i++) m = fmaxf(m, fmaxf(__builtin_fabsf(z[0][i]), __builtin_fabsf(z[1][i])));
  if (__builtin_isinf(m)) {
    m = 0.f;
#pragma unroll
    for (int i = 0; i < 16; i++) {
      const float a = __builtin_fabsf(z[i >> 3][i & 7]);
      m = a > m && !__builtin_isinf(a) ? a : m;
    }
  }
  return m;
}

// use(i, load(i)) for i = 0 .. N - 1 with the loads AHEAD of their use, in this order: a read from LDS passes under the products of the
// ones before it (left to itself, and short of registers, the compiler reads right before each use and waits every time).
template <int N, int AHEAD, typename L, typename U>
__device__ __forceinline__ void read_ahead(L load, U use) {
  u32x4 v[AHEAD + 1];
#pragma unroll
  for (int i = 0; i < (AHEAD < N ? AHEAD : N); i++) v[i] = load(i);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int i = 0; i < N; i++) {
    if (i + AHEAD < N) v[(i + AHEAD) % (AHEAD + 1)] = load(i + AHEAD);
    use(i, v[i % (AHEAD + 1)]);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// four rows r0 .. r0 + 3 (one for each lane quarter of a 16-lane group) x 16 columns come back column-major: lane i gets column
// (i & 3) of the 8-byte piece lane 4 q + (i >> 2) points at, rows q = 0 .. 3.
__device__ __forceinline__ u32x2 tr4(const char* a) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)a));
}

// waves a workgroup of the backward: eight where the weights' images leave a CU one workgroup, four where two fit and wait for their
// barriers apart from each other (us a call, eight / four: 524k x 63 -> 128 bf16 200 / 183, f16 208 / 182; 524k x 20 -> 128 bf16 126 / 115, f16
// 157 / 137; 262k x 96 -> 128 bf16 121 / 165, f16 122 / 169; 100k x 128 -> 128 bf16 88 / 102)
constexpr int bwd_waves(int ks) { return ks == 3 || ks == 4 ? 8 : 4; }

// dz as the operands of its products.  bf16: three, each the upper eight of the bits that the one before left -- 24 in all, so their sum is dz
// itself (cutting never overflows, as rounding next to the largest number does).  f16: its rounding, and the rounding of what that left.
__device__ __forceinline__ void dz_operands(float z, float, __bf16 (&e)[3]) {
  float left = z;
#pragma unroll
  for (int q = 0; q < 3; q++) {
    const uint32_t top = __builtin_bit_cast(uint32_t, left) & 0xffff0000u;
    e[q] = __builtin_bit_cast(__bf16, (uint16_t)(top >> 16));
    // an infinity leaves inf - inf: a finite number in its place, which the infinity swallows
    if (q == 0) left = __builtin_amdgcn_fmed3f(left - __builtin_bit_cast(float, top), -0x1p120f, 0x1p120f);
    else left -= __builtin_bit_cast(float, top);
  }
}
__device__ __forceinline__ void dz_operands(float z, float by, _Float16 (&e)[2]) {  // |z by| < 2^15, or not finite; by a power of two
  e[0] = (_Float16)(z * by);
  e[1] = (_Float16)__builtin_amdgcn_fmed3f(__builtin_fmaf(z, by, -(float)e[0]), -64.f, 64.f);  // as above: what a finite one leaves is at most 2^4
}
template <typename T, int OPS>
__device__ __forceinline__ void dz_operands(const float (&z)[2][8], float by, T (&part)[OPS][2][8]) {
#pragma unroll
  for (int m = 0; m < 2; m++)
#pragma unroll
    for (int i = 0; i < 8; i++) {
      T e[OPS];
      dz_operands(z[m][i], by, e);
#pragma unroll
      for (int q = 0; q < OPS; q++) part[q][m][i] = e[q];
    }
}

// bytes behind a row of dz: the rows that one read covers start on different banks (16 rows of 8-byte pieces; f32: 2 rows of 64 bytes)
constexpr int bwd_pad(int dtype) { return dtype == GFN_F32 ? 64 : 16; }
// operands dz is made of in the products, and the bytes of one pair of feature tiles' dz of a sample
constexpr int bwd_operands(int dtype) { return dtype == GFN_F32 ? 1 : dtype == GFN_BF16 ? 3 : 2; }
constexpr int bwd_ztile(int dtype) { return dtype == GFN_F32 ? 256 : 128 * bwd_operands(dtype); }
// LDS of a workgroup of the backward with room for the dz of `buffers` pairs of feature tiles
constexpr int bwd_lds(int dtype, int ks, int np, int buffers) {
  return 64 * np * (ks * 64 + 16 + 4) + 16 * bwd_waves(ks) * (ks * 64 + 16 + buffers * bwd_ztile(dtype) + bwd_pad(dtype)) + 64;
}
// Pairs of feature tiles whose dz are kept at once, all, two or one, as many as fit without costing the CU its second workgroup: dW's product
// reads x once for them, between two barriers.  (As many / one at a time: 262k x 96 -> 128 f32 862 / 969 us, f16 122 / 126;
// 100k x 48 -> 128 f32 127 / 140.  bf16, whose dz are three operands, has room for one where rows are long.)
constexpr int bwd_buffers(int dtype, int ks, int np) {
  const int room = bwd_lds(dtype, ks, np, 1) <= 80 * 1024 ? 80 * 1024 : 160 * 1024;
  return bwd_lds(dtype, ks, np, np) <= room ? np : np > 2 && bwd_lds(dtype, ks, np, 2) <= room ? 2 : 1;
}
template <typename T>
constexpr int dtype_of() { return sizeof(T) == 4 ? GFN_F32 : __is_same(T, __bf16) ? GFN_BF16 : GFN_F16; }

struct GatedBwd {
  int64_t n_max;
  const int32_t* n_dev;
  const void *x, *wg, *wu, *bg, *bu, *dh;
  int64_t ldx, lddh, lddx;
  int k, h, h0, act;
  void* dx;           // T, or null
  float* dx_sum;      // f32 [n_max][k] between the launches of several feature blocks, or null
  int dx_first, dx_last;
  float* part;        // [workgroup][64 NP][kp] f32, or null: column k is the bias's
  int kp;
};

template <typename T, int KS, int NP>
__global__ __launch_bounds__(64 * bwd_waves(KS), KS < 3 ? 2 : 1) void gated_bwd_kernel(GatedBwd a) {
  constexpr int WAVES = bwd_waves(KS);
  constexpr int E = Piece<T>::E, TPU = sizeof(T) == 4 ? 1 : 2;  // 16-column tiles a unit
  constexpr int KT = KS * TPU, ROW = KS * 64 + 16, HB = 32 * NP, NB = bwd_buffers(dtype_of<T>(), KS, NP);
  constexpr int OPS = bwd_operands(dtype_of<T>()), SAMPLES = 16 * WAVES, ZTILE = bwd_ztile(dtype_of<T>()), ZROW = NB * ZTILE + bwd_pad(dtype_of<T>());
  constexpr int FT_WAVES = WAVES / 4, KT_WAVE = (KT + FT_WAVES - 1) / FT_WAVES;  // waves that share a row tile of dW, its column tiles a wave
  constexpr bool EXACT = sizeof(T) == 4, SCALED = sizeof(T) == 2 && !__is_same(T, __bf16);
  extern __shared__ __attribute__((aligned(16))) char lds[];
  char* xs = lds + 2 * HB * ROW;        // [SAMPLES][ROW]
  char* zs = xs + SAMPLES * ROW;        // [SAMPLES][NB][dg 32 | du 32], 16-bit: the same of what their rounding left
  float* bias = reinterpret_cast<float*>(zs + SAMPLES * ZROW);  // [2][HB]
  int* lowest = reinterpret_cast<int*>(bias + 2 * HB);          // [2][WAVES]: the waves' powers
  const T *x = static_cast<const T*>(a.x), *dh = static_cast<const T*>(a.dh);
  const bool biased = a.bg != nullptr;
  const int k = a.k, h = a.h, h0 = a.h0, act = a.act;
  stage_weights<T, KS>(lds, static_cast<const T*>(a.wg), static_cast<const T*>(a.wu), k, h, h0, HB);
  stage_bias(bias, static_cast<const T*>(a.bg), static_cast<const T*>(a.bu), h, h0, HB);
  const int64_t n = gfn_live_n(a.n_max, a.n_dev);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = lane & 15, kg = lane >> 4;
  const int ft = wave & 3, kt0 = (wave >> 2) * KT_WAVE;
  f32x4 dw[NP][KT_WAVE], db = {0.f, 0.f, 0.f, 0.f};  // db: the sums of dz itself, pair p's in column p
#pragma unroll
  for (int p = 0; p < NP; p++)
#pragma unroll
    for (int t = 0; t < KT_WAVE; t++) dw[p][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  const bool sums = biased && wave < 4;  // one wave for each row tile
  int tile_power[NP], lowest_power = kTopPower;  // dw and db hold the sums of pair p times 2^tile_power[p]
#pragma unroll
  for (int p = 0; p < NP; p++) tile_power[p] = kTopPower;
  const char* wrow = lds + j * ROW + kg * 16;
  const int64_t tiles = (n + SAMPLES - 1) / SAMPLES;
  constexpr int DP = 8 / E;  // pieces of eight features
  const int width = h - h0 < HB ? h - h0 : HB;
  const int cut = cut_piece<T>(k), dh_cut = cut_piece<T>(width);
  constexpr int IN_FLIGHT = 3;  // reads from LDS ahead of the products
  constexpr bool HELD = KS < 4;   // this tile's x stays in registers as well; else the projections read it from LDS
  u32x4 xr[KS], xn[KS], dr[NP][DP], dn[NP][DP];
  auto fetch = [&](int64_t tile) {
    const int64_t s = tile * SAMPLES + wave * 16 + j;
#pragma unroll
    for (int u = 0; u < KS; u++) xn[u] = s < n ? piece_request(x + s * a.ldx, 4 * u + kg, k) : u32x4{0u, 0u, 0u, 0u};
#pragma unroll
    for (int p = 0; p < NP; p++)
#pragma unroll
      for (int q = 0; q < DP; q++)
        dn[p][q] = s < n ? piece_request(dh + s * a.lddh + h0, (32 * p + 8 * kg) / E + q, width) : u32x4{0u, 0u, 0u, 0u};
  };
  if ((int64_t)blockIdx.x < tiles) fetch(blockIdx.x);
  for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int64_t s = tile * SAMPLES + wave * 16 + j;
#pragma unroll
    for (int u = 0; u < KS; u++) {
      xr[u] = xn[u];
      if (u == cut >> 2 && kg == (cut & 3)) xr[u] = piece_shift<T>(xr[u], k);
    }
#pragma unroll
    for (int p = 0; p < NP; p++)
#pragma unroll
      for (int q = 0; q < DP; q++) {
        dr[p][q] = dn[p][q];
        if (p == dh_cut >> (DP + 1) && DP * kg + q == (dh_cut & (4 * DP - 1))) dr[p][q] = piece_shift<T>(dr[p][q], width);
      }
    __syncthreads();  // the weights are staged (first tile); the tile before has been read from xs, zs and top
#pragma unroll
    for (int u = 0; u < KS; u++) *reinterpret_cast<u32x4*>(xs + (wave * 16 + j) * ROW + u * 64 + kg * 16) = xr[u];
    if (tile + gridDim.x < tiles) fetch(tile + gridDim.x);  // on its way under this tile's work
    auto grad = [&](int p, int i) {  // dh of feature 32 p + 8 kg + i
      T t[E];
      __builtin_memcpy(t, &dr[p][i / E], 16);
      return (float)t[i % E];
    };
    // dW's rows of the pairs p0 .. p0 + NB - 1 += their dz^T x over the tile's samples, and db their sums
    auto product = [&](int p0) {
      f32x4 total[NB];  // the same in every column
#pragma unroll
      for (int i = 0; i < NB; i++) total[i] = f32x4{0.f, 0.f, 0.f, 0.f};
      if constexpr (sizeof(T) == 2) {
        // 32 samples at a time, in the order 4 kg .. + 3, 16 + 4 kg .. + 3: a read covers 16 rows, on different banks
        const char* r = zs + (4 * kg + (j >> 2)) * ZROW + (16 * ft + 4 * (j & 3)) * 2;
        const char* q = xs + (4 * kg + (j >> 2)) * ROW + 8 * (j & 3) + 32 * kt0;
        constexpr uint32_t one = __is_same(T, __bf16) ? 0x3f803f80u : 0x3c003c00u;
        constexpr int DEEP = KS < 4 ? 2 : 1;  // dz of the next 32 samples requested with the last x of these, where registers are left for it
        u32x4 av[DEEP][NB][OPS];
        auto samples = [&](int c) {
#pragma unroll
          for (int o = 0; o < NB; o++)
#pragma unroll
            for (int q = 0; q < OPS; q++) {  // dz's 16 bits, then what they left
              const char* e = r + 32 * c * ZROW + o * ZTILE + 128 * q;
              const u32x2 lo = tr4(e), hi = tr4(e + 16 * ZROW);
              av[c % DEEP][o][q] = u32x4{lo[0], lo[1], hi[0], hi[1]};
            }
        };
        read_ahead<SAMPLES / 32 * KT_WAVE, IN_FLIGHT>(
            [&](int i) {
              if (DEEP == 2 && i % KT_WAVE == 0) samples(i / KT_WAVE);
              const char* e = q + 32 * (i / KT_WAVE) * ROW + 32 * (i % KT_WAVE);
              const u32x2 lo = tr4(e), hi = tr4(e + 16 * ROW);
              return u32x4{lo[0], lo[1], hi[0], hi[1]};
            },
            [&](int i, const u32x4& b) {
              const int c = i / KT_WAVE, t = i % KT_WAVE;
              if (DEEP == 1 && t == 0) samples(c);
#pragma unroll
              for (int o = 0; o < NB; o++) {
                const u32x4(&z)[OPS] = av[c % DEEP][o];
#pragma unroll
                for (int q = OPS - 1; q >= 0; q--) {
                  if (t == 0) total[o] = mma(z[q], u32x4{one, one, one, one}, total[o], (T*)nullptr);
                  dw[p0 + o][t] = mma(z[q], b, dw[p0 + o][t], (T*)nullptr);
                }
              }
            });
      } else {
        float sum[NB];
#pragma unroll
        for (int o = 0; o < NB; o++) sum[o] = 0.f;
#pragma unroll 4
        for (int c = 0; c < SAMPLES; c += 4) {
          const char* q = xs + (c + kg) * ROW + j * 4;
          float av[NB];
#pragma unroll
          for (int o = 0; o < NB; o++) {
            av[o] = *reinterpret_cast<const float*>(zs + (c + kg) * ZROW + o * ZTILE + (16 * ft + j) * 4);
            sum[o] += av[o];
          }
#pragma unroll
          for (int t = 0; t < KT_WAVE; t++)
            if (KT % FT_WAVES == 0 || kt0 + t < KT) {
              const float b = *reinterpret_cast<const float*>(q + 64 * (kt0 + t));
#pragma unroll
              for (int o = 0; o < NB; o++) dw[p0 + o][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(av[o], b, dw[p0 + o][t], 0, 0, 0);
            }
        }
#pragma unroll
        for (int o = 0; o < NB; o++) total[o] = __builtin_amdgcn_mfma_f32_16x16x4f32(sum[o], 1.f, total[o], 0, 0, 0);
      }
#pragma unroll
      for (int o = 0; o < NB; o++)
#pragma unroll
        for (int i = 0; i < 4; i++) db[i] = j == p0 + o ? db[i] + total[o][i] : db[i];
    };
    int power = kNoPower;  // dx holds the sample's sums times 2^power
    f32x4 dx[KT];
#pragma unroll
    for (int t = 0; t < KT; t++) dx[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int p = 0; p < NP; p++) {
      f32x4 acc[2][2];
#pragma unroll
      for (int m = 0; m < 2; m++)
#pragma unroll
        for (int t = 0; t < 2; t++) acc[m][t] = *reinterpret_cast<const f32x4*>(bias + m * HB + 32 * p + 16 * t + 4 * kg);
      u32x4 xb[2];
      read_ahead<4 * KS, IN_FLIGHT>(
          [&](int i) {
            if (!HELD && i % 4 == 0) xb[i >> 2 & 1] = *reinterpret_cast<const u32x4*>(xs + (wave * 16 + j) * ROW + (i >> 2) * 64 + kg * 16);
            return *reinterpret_cast<const u32x4*>(wrow + ((i >> 1 & 1) * HB + 32 * p + 16 * (i & 1)) * ROW + (i >> 2) * 64);
          },
          [&](int i, const u32x4& w) { acc[i >> 1 & 1][i & 1] = mma(w, HELD ? xr[i >> 2] : xb[i >> 2 & 1], acc[i >> 1 & 1][i & 1], (T*)nullptr); });
      float d[8], z[2][8];
#pragma unroll
      for (int i = 0; i < 8; i++) d[i] = grad(p, i);
      for_act(act, [&](auto act_c) { gated8_grad<decltype(act_c)::value, EXACT>([&](int i) { return acc[0][i >> 2][i & 3]; }, [&](int i) { return acc[1][i >> 2][i & 3]; }, d, z[0], z[1]); });
      T part[OPS][2][8];
      int own = 0;  // the power of this sample's dz of the pair
      if constexpr (SCALED) {
        float m = largest_of(z);
        m = fmaxf(m, __shfl_xor(m, 16, 64));
        m = fmaxf(m, __shfl_xor(m, 32, 64));
        own = power_of(m);
        const int by = own < power ? own - power : 0;
        power += by;
        if (p && __any(by))
#pragma unroll
          for (int t = 0; t < KT; t++) rescale(dx[t], by);
        if (a.part) {
          const int e = min_over_sixteen(own);
          if (lane == 0) lowest[(p & 1) * WAVES + wave] = e;
        }
      }
      if constexpr (sizeof(T) == 2) dz_operands(z, pow2(own), part);
      if (a.part) {
        if (SCALED || (p && p % NB == 0)) __syncthreads();  // the pairs before have been read; the waves' powers are there
        int by = 0;
        if constexpr (SCALED) {
          int e = lowest[(p & 1) * WAVES];
#pragma unroll
          for (int w = 1; w < WAVES; w++) e = lowest[(p & 1) * WAVES + w] < e ? lowest[(p & 1) * WAVES + w] : e;
          e = __builtin_amdgcn_readfirstlane(e);
          if (e == kNoPower) e = tile_power[p];
          if (e > lowest_power + 64) e = lowest_power + 64;
          if (e < lowest_power) lowest_power = e;
          if (e != tile_power[p]) {
#pragma unroll
            for (int t = 0; t < KT_WAVE; t++) rescale(dw[p][t], e - tile_power[p]);
#pragma unroll
            for (int i = 0; i < 4; i++) db[i] = j == p ? __builtin_amdgcn_ldexpf(db[i], e - tile_power[p]) : db[i];
            tile_power[p] = e;
          }
          by = own == kNoPower ? 0 : e - own;
        }
        char* zr = zs + (wave * 16 + j) * ZROW + p % NB * ZTILE + 8 * kg * sizeof(T);
        if constexpr (sizeof(T) == 2) {
#pragma unroll
          for (int q = 0; q < OPS; q++)
#pragma unroll
            for (int m = 0; m < 2; m++) {
              u32x4 v = __builtin_bit_cast(u32x4, part[q][m]);
              if (SCALED && __any(by)) v = times_pow2(v, by);
              *reinterpret_cast<u32x4*>(zr + 128 * q + 64 * m) = v;
            }
        } else {
#pragma unroll
          for (int m = 0; m < 2; m++) __builtin_memcpy(__builtin_assume_aligned(zr + 128 * m, 16), z[m], sizeof(z[m]));
        }
      }
      if (a.dx || a.dx_sum) {  // dx[k] += sum over these 32 features
        if constexpr (SCALED)
          if (__any(own != power && own != kNoPower))
#pragma unroll
            for (int q = 0; q < OPS; q++)
#pragma unroll
              for (int m = 0; m < 2; m++) {
                const u32x4 v = times_pow2(__builtin_bit_cast(u32x4, part[q][m]), own == kNoPower ? 0 : power - own);
                __builtin_memcpy(part[q][m], &v, 16);
              }
        if constexpr (sizeof(T) == 2) {
          // features 8 kg .. + 3 are image rows 4 kg .. + 3 of tile 0, the next four those of tile 1
          const char* r = lds + (32 * p + 4 * kg + (j >> 2)) * ROW + 8 * (j & 3);
          read_ahead<2 * KT, IN_FLIGHT>(
              [&](int i) {
                const char* q = r + (i / KT) * HB * ROW + 32 * (i % KT);
                const u32x2 lo = tr4(q), hi = tr4(q + 16 * ROW);
                return u32x4{lo[0], lo[1], hi[0], hi[1]};
              },
              [&](int i, const u32x4& w) {
#pragma unroll
                for (int q = OPS - 1; q >= 0; q--) dx[i % KT] = mma(w, __builtin_bit_cast(u32x4, part[q][i / KT]), dx[i % KT], (T*)nullptr);
              });
        } else {
#pragma unroll
          for (int m = 0; m < 2; m++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
              const char* r = lds + (m * HB + 32 * p + 4 * kg + 16 * (i >> 2) + (i & 3)) * ROW;
#pragma unroll
              for (int t = 0; t < KT; t++)
                dx[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(*reinterpret_cast<const float*>(r + (16 * t + j) * 4), z[m][i], dx[t], 0, 0, 0);
            }
        }
      }
      if (a.part && p % NB == NB - 1) {
        __syncthreads();
        product(p - NB + 1);
      }
    }
    loads_done();
    if ((a.dx || a.dx_sum) && s < n) {  // lane (j, kg) holds columns 16 t + 4 kg + r of sample j
#pragma unroll
      for (int t = 0; t < KT; t++) {
        const int col = 16 * t + 4 * kg;
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = SCALED ? __builtin_amdgcn_ldexpf(dx[t][i], -power) : dx[t][i];
        if (col < k) {
          if (!a.dx_first) {
#pragma unroll
            for (int i = 0; i < 4; i++)
              if (col + i < k) v[i] += a.dx_sum[s * k + col + i];
          }
          if (a.dx_last) {
            store_row<T, 4>(static_cast<T*>(a.dx) + s * a.lddx + col, k - col, v);
          } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
              if (col + i < k) a.dx_sum[s * k + col + i] = v[i];
          }
        }
      }
    }
  }
  if (a.part) {
    const int kp = a.kp;
    float* o = a.part + (int64_t)blockIdx.x * (64 * NP * kp);
#pragma unroll
    for (int p = 0; p < NP; p++)
#pragma unroll
      for (int t = 0; t < KT_WAVE; t++) {
        const int col = 16 * (kt0 + t) + j;
        if (col < k)
#pragma unroll
          for (int r = 0; r < 4; r++) o[(64 * p + 16 * ft + 4 * kg + r) * kp + col] = SCALED ? __builtin_amdgcn_ldexpf(dw[p][t][r], -tile_power[p]) : dw[p][t][r];
      }
#pragma unroll
    for (int p = 0; p < NP; p++)
      if (sums && j == p)
#pragma unroll
        for (int r = 0; r < 4; r++) o[(64 * p + 16 * ft + 4 * kg + r) * kp + k] = SCALED ? __builtin_amdgcn_ldexpf(db[r], -tile_power[p]) : db[r];
  }
}

// dW[f][c] = sum over the workgroups of part[f's row][c], in their order: 32 columns x 32 runs of workgroups a block
template <typename T>
__global__ __launch_bounds__(1024) void gated_reduce_kernel(const float* __restrict__ part, int parts, int rows, int kp, int k, int h, int h0, int cols,
                                                            T* __restrict__ dwg, T* __restrict__ dwu, T* __restrict__ dbg, T* __restrict__ dbu) {
  __shared__ float sums[32][33];
  const int col = threadIdx.x & 31, run = threadIdx.x >> 5, row = blockIdx.y;
  const int c = blockIdx.x * 32 + col, f = h0 + (row >> 6) * 32 + (row & 31);
  const int per = (parts + 31) / 32, last = parts < (run + 1) * per ? parts : (run + 1) * per;
  float s = 0.f;
  if (c < cols && f < h) {
    const float* p = part + (int64_t)row * kp + c;
#pragma unroll 16
    for (int b = run * per; b < last; b++) s += p[(int64_t)b * rows * kp];
  }
  sums[run][col] = s;
  __syncthreads();
  if (run || c >= cols || f >= h) return;
#pragma unroll
  for (int r = 1; r < 32; r++) s += sums[r][col];
  const bool up = (row >> 5) & 1;
  if (c < k) (up ? dwu : dwg)[(int64_t)f * k + c] = (T)s;
  else (up ? dbu : dbg)[f] = (T)s;
}

// ---- host ---------------------------------------------------------------------------------------------------------------------------
constexpr int kMaxIn = 128, kMaxHidden = 1024;

int check_common(const char* who, int64_t n_max, int k, int h, int dtype, int act) {
  GFN_CHECK_ARG(n_max >= 0 && n_max < (1ll << 31), "%s: n_max=%lld", who, (long long)n_max);
  GFN_CHECK_ARG(k >= 1 && k <= kMaxIn && h >= 1 && h <= kMaxHidden, "%s: dims %dx%d unsupported (in 1..%d, hidden 1..%d)", who, k, h, kMaxIn, kMaxHidden);
  GFN_CHECK_ARG(dtype >= GFN_F32 && dtype <= GFN_F16, "%s: dtype %d", who, dtype);
  GFN_CHECK_ARG(act >= 0 && act <= 3, "%s: act %d", who, act);
  return GFN_OK;
}

template <typename K>
int allow_lds(K kernel, size_t bytes) {  // above the 64 KB a kernel may use without asking
  GFN_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
  return GFN_OK;
}

struct GatedFwd {
  const void *x, *wg, *wu, *bg, *bu;
  int64_t ldx, ldo, n_max;
  const int32_t* n_dev;
  int k, h, act;
  void* out;
};

template <typename T, int KS, int G>
int launch_fwd(const GatedFwd& a, hipStream_t st) {
  constexpr int ROW = KS * 64 + 16;
  const int hp = (a.h + 31) & ~31;
  const int64_t tiles = (a.n_max + 16 * G * kWaves - 1) / (16 * G * kWaves);
  // features a workgroup: all of them (x is read once) while there are samples enough for every CU, else blocks of 32 (63 -> 128 bf16,
  // blocks / all: 128 rows 4.3 / 7.5 us, 16384 7.3 / 9.4, 32768 11.4 / 10.2, 65536 20.5 / 14.4)
  int hc = hp < 128 ? hp : 128;
  if ((size_t)2 * hc * ROW > 80 * 1024) hc = 64;
  if (tiles < 256) hc = 32;
  const size_t bytes = (size_t)2 * hc * (ROW + 4);
  static unsigned long long seen = 0;
  if (gfn_first_call_on_device(seen))
    if (int rc = allow_lds(gated_fwd_kernel<T, KS, G>, 160 * 1024)) return rc;
  const int64_t at_once = 256 * (int64_t)(160 * 1024 / (bytes + 512) < 4 ? 160 * 1024 / (bytes + 512) : 4);
  const int64_t blocks = tiles < at_once ? tiles : at_once;
  const dim3 grid((unsigned)blocks, (unsigned)((hp + hc - 1) / hc));
  gated_fwd_kernel<T, KS, G><<<grid, 64 * kWaves, bytes, st>>>(a.n_max, a.n_dev, static_cast<const T*>(a.x), a.ldx, static_cast<const T*>(a.wg),
                                                              static_cast<const T*>(a.wu), static_cast<const T*>(a.bg), static_cast<const T*>(a.bu), a.k, a.h,
                                                              hc, a.act, static_cast<T*>(a.out), a.ldo);
  GFN_CHECK_LAUNCH();
  return GFN_OK;
}

template <typename T>
int dispatch_fwd(const GatedFwd& a, hipStream_t st) {
  const int units = (a.k + 4 * Piece<T>::E - 1) / (4 * Piece<T>::E);
  // one group of 16 samples a wave or two (each weight read once for both): us for 63 -> 128 bf16, one / two: 4096 rows 4.5 / 5.3, 16384
  // 7.4 / 7.3, 32768 13.6 / 11.4
  const bool few = a.n_max < 16384;
#define GFN_GATED(KS, G)                                                             \
  if (units <= KS) return few ? launch_fwd<T, KS, 1>(a, st) : launch_fwd<T, KS, G>(a, st)
  GFN_GATED(1, 2);
  GFN_GATED(2, 2);
  if constexpr (sizeof(T) == 4) {
    GFN_GATED(4, 2);
    GFN_GATED(8, 1);
  } else {
    GFN_GATED(3, 2);
    GFN_GATED(4, 2);
  }
#undef GFN_GATED
  return GFN_ERR_ARG;
}

// The backward's plan for (n, k, h, type): units a row, feature blocks of 32 NP, waves and workgroups.
struct BwdPlan {
  int ks, np, waves, blocks, launches, kp;
  size_t lds, part_floats;
  bool dx_sum;
};

BwdPlan plan_bwd(int64_t n, int k, int h, int dtype, bool bias) {
  BwdPlan p;
  const int e = dtype == GFN_F32 ? 4 : 8;
  p.ks = (k + 4 * e - 1) / (4 * e);
  if (p.ks > 4) p.ks = 8;  // f32 only
  p.waves = bwd_waves(p.ks);
  p.kp = (k + (bias ? 1 : 0) + 15) & ~15;
  const int most = p.ks > 4 ? 2 : 4;  // 32-feature pairs a launch: the weights and dW's accumulators fit
  const int pairs = (h + 31) / 32;
  p.np = pairs >= 3 && most == 4 ? 4 : pairs >= 2 ? 2 : 1;
  p.launches = (pairs + p.np - 1) / p.np;
  const int samples = 16 * p.waves;
  p.lds = bwd_lds(dtype, p.ks, p.np, bwd_buffers(dtype, p.ks, p.np));
  const int64_t tiles = (n + samples - 1) / samples;
  const int at_once = 256 * (p.lds <= 80 * 1024 ? 2 : 1);
  p.blocks = tiles < 1 ? 1 : (int)(tiles < at_once ? tiles : at_once);
  p.part_floats = (size_t)p.blocks * 64 * p.np * p.kp;
  p.dx_sum = p.launches > 1;
  return p;
}

template <typename T, int KS, int NP>
int launch_bwd(const GatedBwd& a, const BwdPlan& p, hipStream_t st) {
  static unsigned long long seen = 0;
  if (gfn_first_call_on_device(seen))
    if (int rc = allow_lds(gated_bwd_kernel<T, KS, NP>, 160 * 1024)) return rc;
  gated_bwd_kernel<T, KS, NP><<<p.blocks, 64 * p.waves, p.lds, st>>>(a);
  GFN_CHECK_LAUNCH();
  return GFN_OK;
}

template <typename T>
int dispatch_bwd(const GatedBwd& a, const BwdPlan& p, hipStream_t st) {
#define GFN_GATED_NP(KS, NP) \
  if (p.ks == KS && p.np == NP) return launch_bwd<T, KS, NP>(a, p, st)
#define GFN_GATED(KS)   \
  GFN_GATED_NP(KS, 1);  \
  GFN_GATED_NP(KS, 2);  \
  GFN_GATED_NP(KS, 4)
  GFN_GATED(1);
  GFN_GATED(2);
  GFN_GATED(3);
  GFN_GATED(4);
  if constexpr (sizeof(T) == 4) {
    GFN_GATED_NP(8, 1);
    GFN_GATED_NP(8, 2);
  }
#undef GFN_GATED
#undef GFN_GATED_NP
  gfn_set_error("gfn_gated_bwd: no kernel for %d units x %d", p.ks, p.np);
  return GFN_ERR_ARG;
}

template <typename T>
int gated_bwd_typed(GatedBwd a, const BwdPlan& p, void* dwg, void* dwu, void* dbg, void* dbu, hipStream_t st) {
  const int cols = a.k + (a.bg ? 1 : 0);
  for (int l = 0; l < p.launches; l++) {
    a.h0 = l * 32 * p.np;
    a.dx_first = l == 0;
    a.dx_last = l == p.launches - 1;
    if (int rc = dispatch_bwd<T>(a, p, st)) return rc;
    if (a.part) {
      gated_reduce_kernel<T><<<dim3((unsigned)((cols + 31) / 32), (unsigned)(64 * p.np)), 1024, 0, st>>>(
          a.part, p.blocks, 64 * p.np, p.kp, a.k, a.h, a.h0, cols, static_cast<T*>(dwg), static_cast<T*>(dwu), static_cast<T*>(dbg), static_cast<T*>(dbu));
      GFN_CHECK_LAUNCH();
    }
  }
  return GFN_OK;
}

}  // namespace

extern "C" {

int gfn_gated_fwd(const void* x, int64_t ldx, const void* wg, const void* wu, const void* bg, const void* bu, int64_t n_max, const int32_t* n_dev,
                  int in_dim, int hidden, int dtype, int act, void* out, int64_t ldo, void* stream) {
  if (int rc = check_common("gfn_gated_fwd", n_max, in_dim, hidden, dtype, act)) return rc;
  if (n_max == 0) return GFN_OK;
  GFN_CHECK_ARG(x && wg && wu && out, "gfn_gated_fwd: null pointer");
  GFN_CHECK_ARG(!bg == !bu, "gfn_gated_fwd: one bias without the other");
  GFN_CHECK_ARG(ldx >= in_dim && ldo >= hidden, "gfn_gated_fwd: row strides %lld / %lld below %d / %d", (long long)ldx, (long long)ldo, in_dim, hidden);
  const int size = dtype == GFN_F32 ? 4 : 2;
  const int64_t weights = (int64_t)hidden * in_dim;
  if (int rc = gfn_check_apart("gfn_gated_fwd", {{"out", out, n_max, hidden, ldo, size}},
                               {{"x", x, n_max, in_dim, ldx, size}, gfn_flat("wg", wg, weights, size), gfn_flat("wu", wu, weights, size), gfn_flat("bg", bg, hidden, size),
                                gfn_flat("bu", bu, hidden, size), gfn_flat("n_dev", n_dev, 1, 4)}))
    return rc;
  const GatedFwd a{x, wg, wu, bg, bu, ldx, ldo, n_max, n_dev, in_dim, hidden, act, out};
  hipStream_t st = gfn_stream(stream);
  if (dtype == GFN_F32) return dispatch_fwd<float>(a, st);
  if (dtype == GFN_BF16) return dispatch_fwd<__bf16>(a, st);
  return dispatch_fwd<_Float16>(a, st);
}

int64_t gfn_gated_bwd_workspace(int64_t n_max, int in_dim, int hidden, int dtype, int bias, int need_dx, int need_dw) {
  if (check_common("gfn_gated_bwd_workspace", n_max, in_dim, hidden, dtype, 0)) return GFN_ERR_ARG;
  const BwdPlan p = plan_bwd(n_max, in_dim, hidden, dtype, bias != 0);
  int64_t bytes = need_dw ? (int64_t)p.part_floats * 4 : 0;
  if (need_dx && p.dx_sum) bytes += n_max * (int64_t)in_dim * 4;
  return bytes;
}

int gfn_gated_bwd(const void* x, int64_t ldx, const void* wg, const void* wu, const void* bg, const void* bu, const void* dh, int64_t lddh, int64_t n_max,
                  const int32_t* n_dev, int in_dim, int hidden, int dtype, int act, void* dx, int64_t lddx, void* dwg, void* dwu, void* dbg, void* dbu,
                  void* workspace, int64_t workspace_bytes, void* stream) {
  if (int rc = check_common("gfn_gated_bwd", n_max, in_dim, hidden, dtype, act)) return rc;
  GFN_CHECK_ARG(wg && wu && (n_max == 0 || (x && dh)), "gfn_gated_bwd: null pointer");
  GFN_CHECK_ARG(!bg == !bu, "gfn_gated_bwd: one bias without the other");
  GFN_CHECK_ARG(!dwg == !dwu, "gfn_gated_bwd: one weight gradient without the other");
  GFN_CHECK_ARG((dbg != nullptr) == (dbu != nullptr) && (dbg != nullptr) == (dwg != nullptr && bg != nullptr), "gfn_gated_bwd: the biases' gradients go with the biases and the weights' gradients");
  GFN_CHECK_ARG(ldx >= in_dim && lddh >= hidden && (!dx || lddx >= in_dim), "gfn_gated_bwd: a row stride is below the row's width");
  if (!dx && !dwg) return GFN_OK;
  const int64_t need = gfn_gated_bwd_workspace(n_max, in_dim, hidden, dtype, bg != nullptr, dx != nullptr, dwg != nullptr);
  GFN_CHECK_ARG(workspace_bytes >= need && (need == 0 || workspace), "gfn_gated_bwd: workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)need);
  if (n_max == 0 && !dwg) return GFN_OK;
  const int size = dtype == GFN_F32 ? 4 : 2;
  const int64_t weights = (int64_t)hidden * in_dim;
  if (int rc = gfn_check_apart("gfn_gated_bwd",
                               {{"dx", dx, n_max, in_dim, lddx, size}, gfn_flat("dwg", dwg, weights, size), gfn_flat("dwu", dwu, weights, size), gfn_flat("dbg", dbg, hidden, size),
                                gfn_flat("dbu", dbu, hidden, size), gfn_flat("the workspace", workspace, need, 1)},
                               {{"x", x, n_max, in_dim, ldx, size}, {"dh", dh, n_max, hidden, lddh, size}, gfn_flat("wg", wg, weights, size), gfn_flat("wu", wu, weights, size),
                                gfn_flat("bg", bg, hidden, size), gfn_flat("bu", bu, hidden, size), gfn_flat("n_dev", n_dev, 1, 4)}))
    return rc;
  const BwdPlan p = plan_bwd(n_max, in_dim, hidden, dtype, bg != nullptr);
  GatedBwd a{};
  a.n_max = n_max; a.n_dev = n_dev;
  a.x = x; a.wg = wg; a.wu = wu; a.bg = bg; a.bu = bu; a.dh = dh;
  a.ldx = ldx; a.lddh = lddh; a.lddx = lddx;
  a.k = in_dim; a.h = hidden; a.act = act;
  a.dx = dx;
  a.kp = p.kp;
  float* ws = static_cast<float*>(workspace);
  if (dwg) {
    a.part = ws;
    ws += p.part_floats;
  }
  if (dx && p.dx_sum) a.dx_sum = ws;
  hipStream_t st = gfn_stream(stream);
  if (dtype == GFN_F32) return gated_bwd_typed<float>(a, p, dwg, dwu, dbg, dbu, st);
  if (dtype == GFN_BF16) return gated_bwd_typed<__bf16>(a, p, dwg, dwu, dbg, dbu, st);
  return gated_bwd_typed<_Float16>(a, p, dwg, dwu, dbg, dbu, st);
}

}  // extern "C"
