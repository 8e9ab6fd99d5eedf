// dropout.hip -- dropout whose mask is a function of (seed, call, row, column): Philox4x32-10 (Salmon et al., SC'11) with the counter
// (column / 8, row, call), 16 of its 128 bits for each of eight columns.  Nothing is stored; the backward pass is the same launch on dy.
// 16 bits place p on a grid of 2^-16 and the kept elements' factor is that grid point's, so the expectation is exact; 32 bits an element
// would double the generator's work (20 32 x 32 -> 64 bit multiplications, quarter rate, for four elements instead of eight) and make
// the kernel as long as the generator instead of as long as its memory traffic.
#include "gfn_common.h"

namespace {

__device__ __forceinline__ void philox(uint32_t (&c)[4], uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int r = 0; r < 10; r++) {
    const uint64_t p0 = (uint64_t)0xD2511F53u * c[0], p1 = (uint64_t)0xCD9E8D57u * c[2];
    const uint32_t n0 = (uint32_t)(p1 >> 32) ^ c[1] ^ k0, n2 = (uint32_t)(p0 >> 32) ^ c[3] ^ k1;
    c[1] = (uint32_t)p1;
    c[3] = (uint32_t)p0;
    c[0] = n0;
    c[2] = n2;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
}

// a thread: eight columns of a row.  WIDE: cols and strides are multiples of eight elements and the pointers of 16 bytes; else the same
// accesses at any address, the row's end element by element.  Memory bound: 786k x 128 in bf16 67 us, 6.0 TB/s (a large copy on the card
// 5.1 to 5.4), 90 us without WIDE; 786k x 127 146 us (element by element throughout: 227).
template <typename T, bool WIDE>
__global__ __launch_bounds__(256) void dropout_kernel(const T* x, int64_t ldx, int64_t rows, int cols, uint32_t below, float scale, uint64_t seed,
                                                      const unsigned long long* __restrict__ call_dev, T* y, int64_t ldy) {
  const unsigned long long call = *call_dev;
  const int per_row = (cols + 7) / 8;
  const int64_t n = rows * per_row;
  for (int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x; id < n; id += (int64_t)gridDim.x * 256) {
    const int64_t row = id / per_row;
    const int blk = (int)(id - row * per_row), left = cols - 8 * blk;
    uint32_t c[4] = {(uint32_t)blk, (uint32_t)row, (uint32_t)call, (uint32_t)(call >> 32)};
    const T* xp = x + row * ldx + 8 * blk;
    T* yp = y + row * ldy + 8 * blk;
    T v[8];
    if constexpr (WIDE) {
      __builtin_memcpy(v, __builtin_assume_aligned(xp, 16), sizeof(v));
    } else if (left >= 8) {
      __builtin_memcpy(v, xp, sizeof(v));
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] = i < left ? xp[i] : (T)0.f;
    }
    philox(c, (uint32_t)seed, (uint32_t)(seed >> 32));
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const uint32_t bits = (i & 1) ? c[i >> 1] >> 16 : c[i >> 1] & 0xffffu;
      v[i] = bits >= below ? (T)((float)v[i] * scale) : (T)0.f;
    }
    if constexpr (WIDE) {
      __builtin_memcpy(__builtin_assume_aligned(yp, 16), v, sizeof(v));
    } else if (left >= 8) {
      __builtin_memcpy(yp, v, sizeof(v));
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++)
        if (i < left) yp[i] = v[i];
    }
  }
}

__global__ void dropout_call_kernel(unsigned long long* __restrict__ counter, unsigned long long* __restrict__ call) { *call = atomicAdd(counter, 1ull); }

template <typename T>
int launch_dropout(const void* x, int64_t ldx, int64_t rows, int cols, uint32_t below, float scale, uint64_t seed, const uint64_t* call, void* y, int64_t ldy,
                   hipStream_t st) {
  const int64_t n = rows * ((cols + 7) / 8);
  const int64_t blocks = (n + 255) / 256;
  const unsigned grid = (unsigned)(blocks < 65536 ? blocks : 65536);
  const bool wide = ((ldx | ldy | cols) & 7) == 0 && ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) & 15) == 0;
  const auto* c = reinterpret_cast<const unsigned long long*>(call);
  if (wide) dropout_kernel<T, true><<<grid, 256, 0, st>>>(static_cast<const T*>(x), ldx, rows, cols, below, scale, seed, c, static_cast<T*>(y), ldy);
  else dropout_kernel<T, false><<<grid, 256, 0, st>>>(static_cast<const T*>(x), ldx, rows, cols, below, scale, seed, c, static_cast<T*>(y), ldy);
  GFN_CHECK_LAUNCH();
  return GFN_OK;
}

}  // namespace

extern "C" {

int gfn_dropout(const void* x, int64_t ldx, int64_t rows, int cols, int dtype, float p, uint64_t seed, const uint64_t* call, void* y, int64_t ldy, void* stream) {
  GFN_CHECK_ARG(rows >= 0 && rows < (1ll << 32) && cols >= 0, "gfn_dropout: %lld rows of %d", (long long)rows, cols);
  GFN_CHECK_ARG(p >= 0.f && p <= 1.f, "gfn_dropout: p = %g is not in [0, 1]", (double)p);
  GFN_CHECK_ARG(dtype >= GFN_F32 && dtype <= GFN_F16, "gfn_dropout: dtype %d", dtype);
  if (rows == 0 || cols == 0) return GFN_OK;
  GFN_CHECK_ARG(x && y && call, "gfn_dropout: null pointer");
  GFN_CHECK_ARG(ldx >= cols && ldy >= cols, "gfn_dropout: a row stride is below the row's width");
  const int size = dtype == GFN_F32 ? 4 : 2;
  const gfn_rows rx{"x", x, rows, cols, ldx, size}, ry{"y", y, rows, cols, ldy, size};
  GFN_CHECK_ARG(gfn_same_rows(rx, ry) || !gfn_overlap(rx, ry), "gfn_dropout: y overlaps x, and is not x");
  GFN_CHECK_ARG(!gfn_overlap(ry, gfn_flat("call", call, 1, 8)), "gfn_dropout: y overlaps call");
  const uint32_t below = (uint32_t)((double)p * 65536.0 + 0.5);
  const float scale = below < 65536u ? (float)(65536.0 / (65536u - below)) : 0.f;
  hipStream_t st = gfn_stream(stream);
  if (dtype == GFN_F32) return launch_dropout<float>(x, ldx, rows, cols, below, scale, seed, call, y, ldy, st);
  if (dtype == GFN_BF16) return launch_dropout<__bf16>(x, ldx, rows, cols, below, scale, seed, call, y, ldy, st);
  return launch_dropout<_Float16>(x, ldx, rows, cols, below, scale, seed, call, y, ldy, st);
}

int gfn_dropout_call(uint64_t* counter, uint64_t* call, void* stream) {
  GFN_CHECK_ARG(counter && call, "gfn_dropout_call: null pointer");
  GFN_CHECK_ARG(!gfn_overlap(gfn_flat("counter", counter, 1, 8), gfn_flat("call", call, 1, 8)), "gfn_dropout_call: call overlaps counter");
  dropout_call_kernel<<<1, 1, 0, gfn_stream(stream)>>>(reinterpret_cast<unsigned long long*>(counter), reinterpret_cast<unsigned long long*>(call));
  GFN_CHECK_LAUNCH();
  return GFN_OK;
}

}  // extern "C"
