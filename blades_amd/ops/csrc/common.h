// Shared device helpers for the gfx950 (CDNA4, wave64) kernels.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#define BLADES_API extern "C" __attribute__((visibility("default")))

constexpr int kWave = 64;

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  return v;
}
__device__ __forceinline__ int wave_sum_i(int v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// Block-wide sum for blockDim.x == 256 (4 waves). `red` is >= 4 floats of LDS.
__device__ __forceinline__ float block_sum_256(float v, float* red) {
  v = wave_sum(v);
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  __syncthreads();
  if (lane == 0) red[w] = v;
  __syncthreads();
  return red[0] + red[1] + red[2] + red[3];
}

// A kernel's output, past the caches' replacement where `through` (a uniform value).  What a rule for it has to weigh: the
// kernel itself does not wait for write-backs, but what reads the output next finds less of it near.
template <typename V> __device__ __forceinline__ void store_out(void* p, const V& v, bool through) {
  if constexpr (sizeof(V) % 4 == 0) {
    typedef unsigned words __attribute__((ext_vector_type(sizeof(V) / 4)));
    if (through) {
      asm volatile("");  // (before and after: keeps the compiler from making one plain store of both)
      __builtin_nontemporal_store(__builtin_bit_cast(words, v), (words*)p);
      asm volatile("");
      return;
    }
  }
  *(V*)p = v;
}

// n / d for n < 2^31 by a multiplication (Granlund and Montgomery, "Division by invariant integers")
struct Div {
  uint32_t d, m, s;
  static Div of(uint32_t d) {
    Div r{d, 0, 0};
    while ((1ull << r.s) < d) ++r.s;
    r.m = (uint32_t)(((1ull << 32) * ((1ull << r.s) - d)) / d + 1);
    return r;
  }
  __device__ __forceinline__ uint32_t over(uint32_t n) const { return (__umulhi(n, m) + n) >> s; }
};

static inline int cdiv(long a, long b) { return (int)((a + b - 1) / b); }

// Philox4x32-10 — bit-identical to ops/reference.py::_philox4x32.
struct Philox4 { uint32_t x, y, z, w; };
__host__ __device__ __forceinline__ Philox4 philox4x32_10(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3,
                                                          uint32_t k0, uint32_t k1) {
  constexpr uint32_t M0 = 0xD2511F53u, M1 = 0xCD9E8D57u, W0 = 0x9E3779B9u, W1 = 0xBB67AE85u;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = (uint64_t)c0 * M0, p1 = (uint64_t)c2 * M1;
    const uint32_t hi0 = (uint32_t)(p0 >> 32), lo0 = (uint32_t)p0;
    const uint32_t hi1 = (uint32_t)(p1 >> 32), lo1 = (uint32_t)p1;
    const uint32_t n0 = hi1 ^ c1 ^ k0, n2 = hi0 ^ c3 ^ k1;
    c0 = n0; c1 = lo1; c2 = n2; c3 = lo0;
    k0 += W0; k1 += W1;
  }
  return {c0, c1, c2, c3};
}
