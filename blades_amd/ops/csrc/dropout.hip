// Client-keyed dropout without a stored mask: y = x * m, the same kernel for the gradient (dx = gy * m).
//
// Value i of client `uid` is kept iff the 24-bit draw of word i & 3 of Philox4x32-10(counter (i >> 2, uid, tag, c3), seed)
// is >= p; m = scale for kept values, 0 for dropped ones.  A draw belongs to one element, to one channel of a sample
// (nn.Dropout2d) or to one sample (stochastic depth); i counts them in row-major (sample, channel, pixel) order, whatever
// the layout in memory, so the mask depends on (seed, client, tag, layer) alone and equals client_dropout_mult's.
// `tag` may live in device memory: a captured HIP graph then replays with the current round's.
//
// Bound by the generator (element draws: 18 64-bit products and 34 exclusive ors per draw of four) and memory alike: 32 x 64 x
// 64 x 128 fp32 22 us (134 MB, 6.0 TB/s; the bytes alone 17 at the cache's 8), and by memory where a draw is shared: 3840 x 64
// x 6 x 6 bf16 by channel 9.7 (35 MB).  Outputs are stored through the caches: what follows reads them at once.
//
// Multiplication, not selection, as the stored multipliers had it: 0 * inf stays NaN.
#include "common.h"
#include "layers_abi.h"

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
  uint32_t c3, k0, k1, least;  // least: smallest word that is kept (the smallest kept 24-bit draw, 8 zero bits below)
  float scale;
};

// keep bits of the values 4q .. 4q + 3
__device__ __forceinline__ unsigned keep4(const Key& key, uint32_t q, uint32_t uid, uint32_t tag) {
  const Philox4 r = philox4x32_10(q, uid, tag, key.c3, key.k0, key.k1);
  return (r.x >= key.least ? 1u : 0u) | (r.y >= key.least ? 2u : 0u) | (r.z >= key.least ? 4u : 0u) | (r.w >= key.least ? 8u : 0u);
}
__device__ __forceinline__ uint32_t tag_of(const Key& key) { return (uint32_t)(key.tag ? key.tag[0] : key.tag_value); }

// ---------------------------------------------------------------------------------------------------------------
// A draw for every element of contiguous blocks.  Block r holds `len` values of memory starting at r * len; they belong to
// client r % Kc (inner) or r and are its elements e0 = (r / Kc) * len (inner) or 0 onwards.  U vectors a thread are on their
// way while the draws are made; VEC 1 (a share whose length is no multiple of a vector's): one draw of four a thread,
// wherever the block starts inside it.
template <typename T, int VEC, int U>
__global__ __launch_bounds__(TPB) void drop_elem_kernel(Key key, const T* __restrict__ x, T* __restrict__ y, long nblk, int Kc,
                                                        int inner, long len) {
  typedef Pack<T, VEC> V;
  const uint32_t tag = tag_of(key);
  for (long r = blockIdx.y; r < nblk; r += gridDim.y) {
    const uint32_t uid = (uint32_t)key.uids[inner ? r % Kc : r];
    const long e0 = inner ? r / Kc * len : 0;
    const T* xb = x + r * len;
    T* yb = y + r * len;
    if (VEC > 1) {
      // e0 and len are multiples of VEC here: a vector is one or two whole draws of four
      const long nv = len / VEC;
      for (long v0 = (long)blockIdx.x * TPB * U + threadIdx.x; v0 < nv; v0 += (long)gridDim.x * TPB * U) {
        V w[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (v0 + u * TPB < nv) w[u] = reinterpret_cast<const V*>(xb)[v0 + u * TPB];
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (v0 + u * TPB < nv) {
            const uint32_t q = (uint32_t)((e0 + (v0 + u * TPB) * VEC) >> 2);
            unsigned m = keep4(key, q, uid, tag);
            if (VEC == 8) m |= keep4(key, q + 1, uid, tag) << 4;
#pragma unroll
            for (int j = 0; j < VEC; ++j) from_f(to_f(w[u].e[j]) * ((m >> j) & 1u ? key.scale : 0.f), w[u].e[j]);
            reinterpret_cast<V*>(yb)[v0 + u * TPB] = w[u];
          }
      }
    } else {
      const long q0 = e0 >> 2, nq = ((e0 + len - 1) >> 2) - q0 + 1;
      for (long q = (long)blockIdx.x * TPB + threadIdx.x; q < nq; q += (long)gridDim.x * TPB) {
        const long first = (q0 + q) * 4 - e0;
        T w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (first + j >= 0 && first + j < len) w[j] = xb[first + j];
        const unsigned m = keep4(key, (uint32_t)(q0 + q), uid, tag);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (first + j >= 0 && first + j < len) {
            from_f(to_f(w[j]) * ((m >> j) & 1u ? key.scale : 0.f), w[j]);
            yb[first + j] = w[j];
          }
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------
// A draw for every channel of a sample (kind 1) or every sample (2), shared by its pixels.  Memory is outer rows of Ct
// channels: samples of C channels, or (inner) a batch index's Kc * C; LAST: pixels first, [pixel][Ct], else [Ct][pixel].  A
// workgroup takes `ns` whole rows, or (ns = 1) `cv` vectors of a large one: its first U vectors a thread are on their way while
// the rows' draws go to LDS, a byte per channel.  (A draw by every vector's thread instead: 12.8 us against 9.7 for 3840 x 64
// x 6 x 6 bf16, the generator bound.)
constexpr int GROUP_BYTES = 16384;
struct Rows {
  long outer;                // rows
  int Kc, B, C, Ct, HW, inner, kind;
  int ns, cv, chunks, quads; // quads: C is a multiple of 4, draws come in fours
  long nv;                   // vectors of a row
  Div by_ct, by_hw, by_nv;   // by_hw: pixels in vectors
};
template <typename T, int VEC, bool LAST>
__global__ __launch_bounds__(TPB) void drop_group_kernel(Key key, Rows q, const T* __restrict__ x, T* __restrict__ y) {
  typedef Pack<T, VEC> V;
  constexpr int U = 4;
  __shared__ alignas(16) unsigned char keep[GROUP_BYTES];
  const uint32_t tag = tag_of(key);
  const long tiles = (q.outer + q.ns - 1) / q.ns * q.chunks;
  for (long tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const long t = tile / q.chunks, o0 = t * q.ns;
    const int rows = (int)(q.outer - o0 < q.ns ? q.outer - o0 : q.ns);
    const long v0 = (tile - t * q.chunks) * q.cv;
    const int items = (int)(q.ns > 1 || q.chunks == 1 ? rows * q.nv : (q.nv - v0 < q.cv ? q.nv - v0 : q.cv));
    const V* src = reinterpret_cast<const V*>(x) + o0 * q.nv + v0;
    V* dst = reinterpret_cast<V*>(y) + o0 * q.nv + v0;
    V w[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if ((int)threadIdx.x + u * TPB < items) w[u] = src[threadIdx.x + u * TPB];
    // channels of a row that these vectors touch
    const int lo = LAST ? 0 : (int)(v0 / q.by_hw.d) & ~3;
    const int hi = LAST || q.chunks == 1 ? q.Ct : min(q.Ct, (int)((v0 + items - 1) / q.by_hw.d) + 1);
    const int step = q.quads ? 4 : 1, per = (hi - lo + step - 1) / step;
    for (int i = threadIdx.x; i < rows * per; i += TPB) {
      const int r = i / per, ch = lo + (i - r * per) * step;
      const long o = o0 + r;
      const int k = (int)(q.inner ? ch / q.C : o / q.B), c = q.inner ? ch - k * q.C : ch;
      const long b = q.inner ? o : o - (long)k * q.B, e = q.kind == 2 ? b : b * q.C + c;
      unsigned m = keep4(key, (uint32_t)(e >> 2), (uint32_t)key.uids[k], tag);
      unsigned char* at = keep + r * q.Ct + ch;
      if (q.quads) {
        if (q.kind == 2) m = (m >> (e & 3)) & 1u ? 15u : 0u;
        *reinterpret_cast<unsigned*>(at) = (m & 1u) | (m & 2u) << 7 | (m & 4u) << 14 | (m & 8u) << 21;
      } else {
        *at = (unsigned char)((m >> (e & 3)) & 1u);
      }
    }
    __syncthreads();
    auto finish = [&](V v, uint32_t i) {
      const uint32_t r = q.ns > 1 ? q.by_nv.over(i) : 0u, f = i - r * (uint32_t)q.nv;  // (ns > 1: rows begin at v0 = 0)
      const unsigned char* row = keep + r * q.Ct;
      if (LAST) {
        const uint32_t g = (uint32_t)((v0 * VEC) % q.Ct) + f * VEC, ch = g - q.by_ct.over(g) * q.Ct;
#pragma unroll
        for (int j = 0; j < VEC; ++j) from_f(to_f(v.e[j]) * (row[ch + j] ? key.scale : 0.f), v.e[j]);
      } else {
        const uint32_t first = (uint32_t)(v0 % q.by_hw.d), ch = (uint32_t)(v0 / q.by_hw.d) + q.by_hw.over(first + f);
        const float s = row[ch] ? key.scale : 0.f;
#pragma unroll
        for (int j = 0; j < VEC; ++j) from_f(to_f(v.e[j]) * s, v.e[j]);
      }
      dst[i] = v;
    };
#pragma unroll
    for (int u = 0; u < U; ++u)
      if ((int)threadIdx.x + u * TPB < items) finish(w[u], threadIdx.x + u * TPB);
    for (int i = threadIdx.x + U * TPB; i < items; i += TPB) finish(src[i], i);
    __syncthreads();  // the next tile's draws overwrite these
  }
}

// The same for rows of more channels than a workgroup keeps: every vector's thread makes its own draws.  Memory is walked by
// vectors of VEC channels (LAST: [sample][pixel][client if inner][C]) or of one channel's pixels (else: [sample][C][pixel]);
// index arithmetic in I bits.
template <typename T, int VEC, bool LAST, typename I>
__global__ __launch_bounds__(TPB) void drop_wide_kernel(Key key, const T* __restrict__ x, T* __restrict__ y, int Kc, I B, I C,
                                                         I HW, int inner, int kind, I total) {
  typedef Pack<T, VEC> V;
  constexpr int U = 2;
  const uint32_t tag = tag_of(key);
  for (I i0 = (I)blockIdx.x * (TPB * U) + threadIdx.x; i0 < total; i0 += (I)gridDim.x * (TPB * U)) {
    V w[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i0 + u * TPB < total) w[u] = reinterpret_cast<const V*>(x)[i0 + u * TPB];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i0 + u * TPB < total) {
        const I f = (i0 + u * TPB) * VEC;
        I c, k, b;
        if (LAST) {
          I t = f / C;
          c = f - t * C;
          if (inner) { const I s = t / Kc; k = t - s * Kc; b = s / HW; }
          else { const I s = t / HW; k = s / B; b = s - k * B; }
        } else {
          const I t = f / HW, s = t / C;
          c = t - s * C;
          if (inner) { b = s / Kc; k = s - b * Kc; }
          else { k = s / B; b = s - k * B; }
        }
        const uint32_t uid = (uint32_t)key.uids[k];
        unsigned m;
        if (kind == 2) {
          m = (keep4(key, (uint32_t)(b >> 2), uid, tag) >> (b & 3)) & 1u ? 0xFFu : 0u;
        } else if (LAST && VEC > 1) {  // channels c .. c + VEC - 1: C and so b * C + c are multiples of VEC
          const long e = (long)b * C + c;
          m = keep4(key, (uint32_t)(e >> 2), uid, tag);
          if (VEC == 8) m |= keep4(key, (uint32_t)(e >> 2) + 1, uid, tag) << 4;
        } else {
          const long e = (long)b * C + c;
          m = (keep4(key, (uint32_t)(e >> 2), uid, tag) >> (e & 3)) & 1u ? 0xFFu : 0u;
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) from_f(to_f(w[u].e[j]) * ((m >> j) & 1u ? key.scale : 0.f), w[u].e[j]);
        reinterpret_cast<V*>(y)[i0 + u * TPB] = w[u];
      }
  }
}

// ---------------------------------------------------------------------------------------------------------------
// A draw for every element of channels-last maps: value (b * C + c) * HW + p is counted pixels first, memory runs over
// channels first.  The draws of CT channels x PT pixels go to LDS, one byte per draw of four in the order they are counted
// in, then the tile is walked in memory order, VEC channels a thread; its first U vectors are on their way meanwhile.
constexpr int TILE_BYTES = 8192;
template <typename T, int VEC>
__global__ __launch_bounds__(TPB) void drop_last_kernel(Key key, const T* __restrict__ x, T* __restrict__ y, int Kc, int B, int C,
                                                        int HW, int inner, int CT, int PT, int ct_n, int pt_n) {
  typedef Pack<T, VEC> V;
  constexpr int U = 4;
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
    const size_t base = (inner ? ((size_t)b * HW * Kc + k) * C : ((size_t)k * B + b) * HW * C) + (size_t)p0 * pitch + c0;
    const int nvec = cn / VEC, items = nvec * pn;
    V w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = threadIdx.x + u * TPB, p = i / nvec;
      if (i < items) w[u] = *reinterpret_cast<const V*>(x + base + (size_t)p * pitch + (i - p * nvec) * VEC);
    }
    const int nb = (PT + 3) / 4 + 1;  // bytes of a channel
    for (int i = threadIdx.x; i < cn * nb; i += TPB) {
      const int c = i / nb, o = i - c * nb;
      const long s = ((long)b * C + c0 + c) * HW + p0;
      if (o <= ((s + pn - 1) >> 2) - (s >> 2)) bits[i] = (unsigned char)keep4(key, (uint32_t)((s >> 2) + o), uid, tag);
    }
    __syncthreads();
    const int s0 = (int)((((long)b * C + c0) * HW + p0) & 3), sc = HW & 3;
    auto finish = [&](V v, int i) {
      const int p = i / nvec, c = (i - p * nvec) * VEC;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const int s = ((s0 + (c + j) * sc) & 3) + p;
        from_f(to_f(v.e[j]) * ((bits[(c + j) * nb + (s >> 2)] >> (s & 3)) & 1 ? key.scale : 0.f), v.e[j]);
      }
      *reinterpret_cast<V*>(y + base + (size_t)p * pitch + c) = v;
    };
#pragma unroll
    for (int u = 0; u < U; ++u)
      if ((int)threadIdx.x + u * TPB < items) finish(w[u], threadIdx.x + u * TPB);
    for (int i = threadIdx.x + U * TPB; i < items; i += TPB) {
      const int p = i / nvec;
      finish(*reinterpret_cast<const V*>(x + base + (size_t)p * pitch + (i - p * nvec) * VEC), i);
    }
    __syncthreads();  // the next tile's draws overwrite these
  }
}

template <typename T>
int elem_t(const Key& key, const void* x, void* y, long nblk, int Kc, int inner, long len, int vec, hipStream_t st) {
  constexpr int W = 16 / sizeof(T), U = 16 / W;  // 16 elements a thread and round
  const long items = vec ? (len / W + U - 1) / U : len / 4 + 2;
  const long gy = nblk < 65535 ? nblk : 65535, most = 256 * 16 / gy + 1;
  long gx = (items + TPB - 1) / TPB;
  if (gx > most) gx = most;
  const dim3 grid((unsigned)gx, (unsigned)gy), block(TPB);
  if (vec)
    hipLaunchKernelGGL((drop_elem_kernel<T, W, U>), grid, block, 0, st, key, (const T*)x, (T*)y, nblk, Kc, inner, len);
  else
    hipLaunchKernelGGL((drop_elem_kernel<T, 1, 1>), grid, block, 0, st, key, (const T*)x, (T*)y, nblk, Kc, inner, len);
  return 0;
}

template <typename T, int VEC, bool LAST>
int wide_v(const Key& key, const void* x, void* y, int Kc, long B, long C, long HW, int inner, int kind, hipStream_t st) {
  const long elems = Kc * B * C * HW, total = elems / VEC;
  long gx = (total + 2 * TPB - 1) / (2 * TPB);
  if (gx > 8192) gx = 8192;
  const dim3 grid((unsigned)gx), block(TPB);
  if (elems < (1L << 31))  // (a stride of the grid beyond the end still fits 32 bits)
    hipLaunchKernelGGL((drop_wide_kernel<T, VEC, LAST, uint32_t>), grid, block, 0, st, key, (const T*)x, (T*)y, Kc, (uint32_t)B,
                       (uint32_t)C, (uint32_t)HW, inner, kind, (uint32_t)total);
  else
    hipLaunchKernelGGL((drop_wide_kernel<T, VEC, LAST, long>), grid, block, 0, st, key, (const T*)x, (T*)y, Kc, B, C, HW, inner,
                       kind, total);
  return 0;
}

template <typename T, int VEC, bool LAST>
int group_v(const Key& key, const void* x, void* y, int Kc, long B, long C, long HW, int inner, int kind, hipStream_t st) {
  Rows q;
  q.Kc = Kc; q.B = (int)B; q.C = (int)C; q.HW = (int)HW; q.inner = inner; q.kind = kind;
  const long Ct = inner ? Kc * C : C;
  if (Ct > GROUP_BYTES || Ct * HW >= (1L << 31)) return wide_v<T, VEC, LAST>(key, x, y, Kc, B, C, HW, inner, kind, st);
  q.outer = inner ? B : Kc * B;
  q.Ct = (int)Ct;
  q.nv = Ct * HW / VEC;
  q.quads = C % 4 == 0;
  constexpr int want = TPB * 8;
  long ns = want / q.nv, most = GROUP_BYTES / Ct;
  if (ns > most) ns = most;
  if (ns > q.outer / 1024) ns = q.outer / 1024;  // (1024 workgroups first)
  q.ns = (int)(ns < 1 ? 1 : ns);
  q.cv = want;
  q.chunks = q.ns > 1 || q.nv <= want ? 1 : (int)((q.nv + want - 1) / want);
  q.by_ct = Div::of((uint32_t)Ct); q.by_hw = Div::of((uint32_t)(LAST ? HW : HW / VEC)); q.by_nv = Div::of((uint32_t)q.nv);
  long tiles = (q.outer + q.ns - 1) / q.ns * q.chunks;
  if (tiles > (1L << 20)) tiles = 1L << 20;
  hipLaunchKernelGGL((drop_group_kernel<T, VEC, LAST>), dim3((unsigned)tiles), dim3(TPB), 0, st, key, q, (const T*)x, (T*)y);
  return 0;
}

template <typename T>
int last_t(const Key& key, const void* x, void* y, int Kc, int B, int C, int HW, int inner, int vec, hipStream_t st) {
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
  if (vec)
    hipLaunchKernelGGL((drop_last_kernel<T, W>), grid, block, 0, st, key, (const T*)x, (T*)y, Kc, B, C, HW, inner, CT, PT, ct_n,
                       pt_n);
  else
    hipLaunchKernelGGL((drop_last_kernel<T, 1>), grid, block, 0, st, key, (const T*)x, (T*)y, Kc, B, C, HW, inner, CT, PT, ct_n,
                       pt_n);
  return 0;
}

template <typename T>
int dropout_t(const Key& key, const void* x, void* y, int Kc, long B, long C, long HW, int kind, int inner, int last, int vec,
              hipStream_t st) {
  constexpr int W = 16 / sizeof(T);
  if (kind == 0) {
    if (last && HW > 1) return last_t<T>(key, x, y, Kc, (int)B, (int)C, (int)HW, inner, vec && C % W == 0, st);
    const long nblk = inner ? Kc * B : Kc, len = inner ? C * HW : B * C * HW;
    return elem_t<T>(key, x, y, nblk, Kc, inner, len, vec && len % W == 0, st);
  }
  if (kind == 2 && !inner) { HW *= C; C = 1; last = 0; }  // a sample is one run of memory: one channel
  if (last) {
    if (vec && C % W == 0) return group_v<T, W, true>(key, x, y, Kc, B, C, HW, inner, kind, st);
    return group_v<T, 1, true>(key, x, y, Kc, B, C, HW, inner, kind, st);
  }
  if (vec && HW % W == 0) return group_v<T, W, false>(key, x, y, Kc, B, C, HW, inner, kind, st);
  return group_v<T, 1, false>(key, x, y, Kc, B, C, HW, inner, kind, st);
}
}  // namespace

BLADES_API long blades_client_dropout_plan_size() { return sizeof(DropPlan); }

// tag null: tag_value.
BLADES_API int blades_client_dropout(const void* x, void* y, const long* uids, const long* tag, long tag_value,
                                     const DropPlan* p, hipStream_t st) {
  if (p->Kc < 1 || p->B < 1 || p->C < 1 || p->HW < 1 || p->kind < 0 || p->kind > 2 || p->dtype < 0 || p->dtype > 2 ||
      p->least >> 24)
    return 1;
  if ((double)p->B * p->C * p->HW > 1.7e10) return 1;  // draws of four are counted in 32 bits
  // the kernels that share draws or walk tiles count samples, channels and pixels in 32 bits; drop_elem_kernel in 64
  const bool tiled = p->kind != 0 || (p->last && p->HW > 1);
  if (tiled && (p->C > (1 << 30) || p->HW > (1 << 30) || p->B > (1 << 30))) return 2;
  const Key key{uids, tag, tag_value, p->c3, (uint32_t)p->seed, (uint32_t)(p->seed >> 32), p->least << 8, p->scale};
  const int vec = (((uintptr_t)x | (uintptr_t)y) & 15) == 0;  // 16-byte accesses (the lengths permitting)
#define DROP(T) return dropout_t<T>(key, x, y, p->Kc, p->B, p->C, p->HW, p->kind, p->inner, p->last, vec, st)
  if (p->dtype == 0) DROP(float);
  if (p->dtype == 1) DROP(Bf16);
  DROP(Half);
#undef DROP
}
