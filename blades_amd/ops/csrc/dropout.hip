// Client-keyed dropout without a stored mask: y = x * m, the same kernel for the gradient (dx = gy * m).
//
// Value i of client `uid` is kept iff the 24-bit draw of word i & 3 of Philox4x32-10(counter (i >> 2, uid, tag, c3), seed)
// is >= p; m = scale for kept values, 0 for dropped ones.  A draw belongs to one element, to one channel of a sample
// (nn.Dropout2d) or to one sample (stochastic depth); i counts them in row-major (sample, channel, pixel) order, whatever
// the layout in memory, so the mask depends on (seed, client, tag, layer) alone and equals client_dropout_mult's.
// `tag` may live in device memory: a captured HIP graph then replays with the current round's.
//
// Multiplication, not selection, as the stored multipliers had it: 0 * inf stays NaN.
#include "common.h"

namespace {
constexpr int TPB = 256;

struct Half { unsigned short v; };
struct Bf16 { unsigned short v; };
__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(Bf16 v) { return __uint_as_float((unsigned)v.v << 16); }
__device__ __forceinline__ float to_f(Half v) { return (float)__builtin_bit_cast(_Float16, v.v); }
__device__ __forceinline__ void from_f(float f, float& o) { o = f; }
__device__ __forceinline__ void from_f(float f, Bf16& o) { o.v = __builtin_bit_cast(unsigned short, (__bf16)f); }
__device__ __forceinline__ void from_f(float f, Half& o) { o.v = __builtin_bit_cast(unsigned short, (_Float16)f); }
template <typename T, int VEC> struct alignas(sizeof(T) * VEC) Pack { T e[VEC]; };

struct Key {
  const long* uids;
  const long* tag;  // null: tag_value
  long tag_value;
  uint32_t c3, k0, k1, least;  // least: smallest 24-bit draw that is kept
  float scale;
};

// keep bits of the values 4q .. 4q + 3
__device__ __forceinline__ unsigned keep4(const Key& key, uint32_t q, uint32_t uid, uint32_t tag) {
  const Philox4 r = philox4x32_10(q, uid, tag, key.c3, key.k0, key.k1);
  return ((r.x >> 8) >= key.least ? 1u : 0u) | ((r.y >> 8) >= key.least ? 2u : 0u) | ((r.z >> 8) >= key.least ? 4u : 0u) |
         ((r.w >> 8) >= key.least ? 8u : 0u);
}
__device__ __forceinline__ uint32_t tag_of(const Key& key) { return (uint32_t)(key.tag ? key.tag[0] : key.tag_value); }

// ---------------------------------------------------------------------------------------------------------------
// Contiguous blocks.  Block r holds `len` values of memory starting at r * len; they belong to client r % Kc (inner) or r
// and are its elements e0 = (r / Kc) * len (inner) or 0 onwards.  A value is drawn for every `seg` elements (1: each).
template <typename T, int VEC, bool SEG>
__global__ __launch_bounds__(TPB) void drop_flat_kernel(Key key, const T* __restrict__ x, T* __restrict__ y, long nblk, int Kc,
                                                        int inner, long len, long seg) {
  typedef Pack<T, VEC> V;
  const uint32_t tag = tag_of(key);
  for (long r = blockIdx.y; r < nblk; r += gridDim.y) {
    const uint32_t uid = (uint32_t)key.uids[inner ? r % Kc : r];
    const long e0 = inner ? r / Kc * len : 0;
    const T* xb = x + r * len;
    T* yb = y + r * len;
    if (!SEG && VEC > 1) {
      // e0 and len are multiples of VEC here: a vector is one or two whole draws of four
      const long nv = len / VEC;
      for (long v = (long)blockIdx.x * TPB + threadIdx.x; v < nv; v += (long)gridDim.x * TPB) {
        V w = reinterpret_cast<const V*>(xb)[v];
        const uint32_t q = (uint32_t)((e0 + v * VEC) >> 2);
        unsigned m = keep4(key, q, uid, tag);
        if (VEC == 8) m |= keep4(key, q + 1, uid, tag) << 4;
#pragma unroll
        for (int j = 0; j < VEC; ++j) from_f(to_f(w.e[j]) * ((m >> j) & 1u ? key.scale : 0.f), w.e[j]);
        reinterpret_cast<V*>(yb)[v] = w;
      }
    } else if (!SEG) {
      // one draw of four per thread, wherever the block starts inside it
      const long q0 = e0 >> 2, nq = ((e0 + len - 1) >> 2) - q0 + 1;
      for (long q = (long)blockIdx.x * TPB + threadIdx.x; q < nq; q += (long)gridDim.x * TPB) {
        const unsigned m = keep4(key, (uint32_t)(q0 + q), uid, tag);
        const long first = (q0 + q) * 4 - e0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const long i = first + j;
          if (i >= 0 && i < len) from_f(to_f(xb[i]) * ((m >> j) & 1u ? key.scale : 0.f), yb[i]);
        }
      }
    } else {
      // one draw per vector: seg is a multiple of VEC
      const long nv = len / VEC;
      for (long v = (long)blockIdx.x * TPB + threadIdx.x; v < nv; v += (long)gridDim.x * TPB) {
        V w = reinterpret_cast<const V*>(xb)[v];
        const long i = (e0 + v * VEC) / seg;
        const float s = (keep4(key, (uint32_t)(i >> 2), uid, tag) >> (i & 3)) & 1u ? key.scale : 0.f;
#pragma unroll
        for (int j = 0; j < VEC; ++j) from_f(to_f(w.e[j]) * s, w.e[j]);
        reinterpret_cast<V*>(yb)[v] = w;
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------
// Channels-last maps.  Sample b of client k: pixel p, channel c at base(b, k) + p * pitch + c.  The draws of CT channels x
// PT pixels go to LDS first, one byte per draw of four — in the order they are counted in, pixels fastest — then the tile
// is walked in memory order, VEC channels a thread.  kind 0: value (b * C + c) * HW + p; 1: b * C + c; 2: b.
constexpr int TILE_BYTES = 8192;
template <typename T, int VEC>
__global__ __launch_bounds__(TPB) void drop_last_kernel(Key key, const T* __restrict__ x, T* __restrict__ y, int Kc, int B, int C,
                                                        int HW, int inner, int kind, int CT, int PT, int ct_n, int pt_n) {
  typedef Pack<T, VEC> V;
  __shared__ unsigned char bits[TILE_BYTES];
  const uint32_t tag = tag_of(key);
  for (long tile = blockIdx.x; tile < (long)Kc * B * ct_n * pt_n; tile += gridDim.x) {
    long blk = tile;
    const int pt = (int)(blk % pt_n); blk /= pt_n;
    const int ct = (int)(blk % ct_n); blk /= ct_n;  // blk: sample in memory order
    const int k = (int)(inner ? blk % Kc : blk / B), b = (int)(inner ? blk / Kc : blk % B);
    const uint32_t uid = (uint32_t)key.uids[k];
    const int c0 = ct * CT, cn = min(CT, C - c0), p0 = pt * PT, pn = min(PT, HW - p0);
    const long pitch = inner ? (long)Kc * C : C;
    const size_t base = inner ? ((size_t)b * HW * Kc + k) * C : ((size_t)k * B + b) * HW * C;
    const int nb = (PT + 3) / 4 + 1;  // bytes of a channel
    if (kind == 0) {
      for (int i = threadIdx.x; i < cn * nb; i += TPB) {
        const int c = i / nb, o = i - c * nb;
        const long s = ((long)b * C + c0 + c) * HW + p0;
        if (o <= ((s + pn - 1) >> 2) - (s >> 2)) bits[i] = (unsigned char)keep4(key, (uint32_t)((s >> 2) + o), uid, tag);
      }
    } else if (kind == 1) {
      const long s = (long)b * C + c0;
      for (int i = threadIdx.x; i <= ((s + cn - 1) >> 2) - (s >> 2); i += TPB)
        bits[i] = (unsigned char)keep4(key, (uint32_t)((s >> 2) + i), uid, tag);
    } else if (threadIdx.x == 0) {
      bits[0] = (unsigned char)keep4(key, (uint32_t)(b >> 2), uid, tag);
    }
    __syncthreads();
    const int nvec = cn / VEC;
    for (int i = threadIdx.x; i < nvec * pn; i += TPB) {
      const int p = i / nvec, c = (i - p * nvec) * VEC;
      const size_t o = base + (size_t)(p0 + p) * pitch + c0 + c;
      V w = *reinterpret_cast<const V*>(x + o);
  #pragma unroll
      for (int j = 0; j < VEC; ++j) {
        int at, bit;
        if (kind == 0) {
          const int s = (int)((((long)b * C + c0 + c + j) * HW + p0) & 3) + p;
          at = (c + j) * nb + (s >> 2); bit = s & 3;
        } else if (kind == 1) {
          const int s = (int)(((long)b * C + c0) & 3) + c + j;
          at = s >> 2; bit = s & 3;
        } else {
          at = 0; bit = b & 3;
        }
        from_f(to_f(w.e[j]) * ((bits[at] >> bit) & 1 ? key.scale : 0.f), w.e[j]);
      }
      *reinterpret_cast<V*>(y + o) = w;
    }
    __syncthreads();  // the next tile's draws overwrite these
  }
}

template <typename T>
int flat_t(const Key& key, const void* x, void* y, long nblk, int Kc, int inner, long len, long seg, int vec, hipStream_t st) {
  constexpr int W = 16 / sizeof(T);
  const long items = seg > 1 || vec > 1 ? len / (vec > 1 ? W : 1) : len / 4 + 2;
  long gy = nblk < 65535 ? nblk : 65535;
  long gx = (items + TPB - 1) / TPB, most = 256 * 16 / gy + 1;
  if (gx > most) gx = most;
  const dim3 grid((unsigned)gx, (unsigned)gy), block(TPB);
#define DROP(V, S)                                                                                                     \
  hipLaunchKernelGGL((drop_flat_kernel<T, V, S>), grid, block, 0, st, key, (const T*)x, (T*)y, nblk, Kc, inner, len, seg)
  if (seg > 1) { if (vec > 1) DROP(W, true); else DROP(1, true); }
  else { if (vec > 1) DROP(W, false); else DROP(1, false); }
#undef DROP
  return 0;
}

template <typename T>
int last_t(const Key& key, const void* x, void* y, int Kc, int B, int C, int HW, int inner, int kind, int vec, hipStream_t st) {
  constexpr int W = 16 / sizeof(T);
  const int CT = C < 64 ? C : 64;
  int PT = 4 * (TILE_BYTES / CT - 1);  // CT * ((PT + 3) / 4 + 1) <= TILE_BYTES
  const int most = C < 64 ? 16384 / CT : 256;
  if (PT > most) PT = most;
  if (PT > HW) PT = HW;
  const int ct_n = (C + CT - 1) / CT, pt_n = (HW + PT - 1) / PT;
  long tiles = (long)Kc * B * ct_n * pt_n;
  if (tiles > (1L << 20)) tiles = 1L << 20;
  const dim3 grid((unsigned)tiles), block(TPB);
  if (vec > 1)
    hipLaunchKernelGGL((drop_last_kernel<T, W>), grid, block, 0, st, key, (const T*)x, (T*)y, Kc, B, C, HW, inner, kind, CT, PT,
                       ct_n, pt_n);
  else
    hipLaunchKernelGGL((drop_last_kernel<T, 1>), grid, block, 0, st, key, (const T*)x, (T*)y, Kc, B, C, HW, inner, kind, CT, PT,
                       ct_n, pt_n);
  return 0;
}
}  // namespace

// dtype 0 fp32, 1 bf16, 2 fp16.  kind 0 element, 1 channel, 2 sample.  last: channels-last maps, else contiguous
// [.., C, HW].  inner: [B][Kc][C] instead of [Kc][B][C] in the leading dimensions.  vec != 0: 16-byte accesses are
// allowed (the caller checked the addresses; lengths are checked here).  least: smallest 24-bit draw that is kept.
BLADES_API int blades_client_dropout(const void* x, void* y, const long* uids, const long* tag, long tag_value, int Kc, long B,
                                     long C, long HW, int kind, int inner, int last, unsigned c3, unsigned long long seed,
                                     unsigned least, float scale, int dtype, int vec, hipStream_t st) {
  if (Kc < 1 || B < 1 || C < 1 || HW < 1 || kind < 0 || kind > 2 || dtype < 0 || dtype > 2) return 1;
  if ((double)B * C * HW > 1.7e10) return 1;  // draws of four are counted in 32 bits
  const Key key{uids, tag, tag_value, c3, (uint32_t)seed, (uint32_t)(seed >> 32), least, scale};
  const int W = dtype == 0 ? 4 : 8;
  if (last && HW > 1) {
    if (C > (1 << 30) || HW > (1 << 30) || B > (1 << 30)) return 1;
    const int v = vec && C % W == 0 ? W : 1;
    if (dtype == 0) return last_t<float>(key, x, y, Kc, (int)B, (int)C, (int)HW, inner, kind, v, st);
    if (dtype == 1) return last_t<Bf16>(key, x, y, Kc, (int)B, (int)C, (int)HW, inner, kind, v, st);
    return last_t<Half>(key, x, y, Kc, (int)B, (int)C, (int)HW, inner, kind, v, st);
  }
  const long one = C * HW, seg = kind == 0 ? 1 : kind == 1 ? HW : one;
  const long nblk = inner ? Kc * B : Kc, len = inner ? one : B * one;
  const int v = vec && (seg == 1 ? len : seg) % W == 0 && len % W == 0 ? W : 1;
  if (dtype == 0) return flat_t<float>(key, x, y, nblk, Kc, inner, len, seg, v, st);
  if (dtype == 1) return flat_t<Bf16>(key, x, y, nblk, Kc, inner, len, seg, v, st);
  return flat_t<Half>(key, x, y, nblk, Kc, inner, len, seg, v, st);
}
