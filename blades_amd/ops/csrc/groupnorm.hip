// Group normalisation with a fused residual add and activation on channels-last activations, forward and backward,
// with one affine pair for everybody or one per client and per-client affine gradients.
//
//   x [N][P][C] (P pixels of one sample, channels contiguous), G groups of D = C / G channels:
//     mu, var over a sample's P x D values of a group,  xhat = (x - mu) * rstd,  z = gamma * xhat + beta (+ res),
//     y = act(z)                                                   act: 0 none, 1 ReLU, 2 GELU (erf), 3 SiLU
//     g = gy * act'(z) (= dres),   A_c = sum_p g,   B_c = sum_p g * xhat                      per (sample, channel)
//     dx = rstd * (gamma g - mean(gamma g) - xhat * mean(gamma g xhat))                       means over the group
//     dgamma_c = sum of B_c, dbeta_c = sum of A_c over the samples of a client
//
// A workgroup takes a slab: the S = k * D channels of whole groups of one sample, all pixels, held in registers (up to
// 64 values a thread), so x is read from memory once in each direction: mean, then the squares around that mean (no
// cancellation for offset activations), then the result, all from registers.  Lane l of a pixel row owns VEC channels
// (16 bytes), so a thread keeps its channels for the whole sweep.  A sample too large for a workgroup's registers is
// cut into pixel chunks: the same kernel leaves (mean, M2) or (A, B) of its chunk, a small kernel joins them in chunk
// order, and a second sweep applies; the batch is walked in pieces that stay in the 256 MB last-level cache between the
// two sweeps.  All sums are fp32 in a fixed order (double where many partial sums meet): bitwise reproducible.
#include "common.h"

namespace {

struct Half { unsigned short v; };
struct Bf16 { unsigned short v; };

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(Bf16 v) { return __uint_as_float((unsigned)v.v << 16); }
__device__ __forceinline__ float to_f(Half v) { return (float)__builtin_bit_cast(_Float16, v.v); }
__device__ __forceinline__ void from_f(float f, float& o) { o = f; }
__device__ __forceinline__ void from_f(float f, Bf16& o) { o.v = __builtin_bit_cast(unsigned short, (__bf16)f); }
__device__ __forceinline__ void from_f(float f, Half& o) { o.v = __builtin_bit_cast(unsigned short, (_Float16)f); }

template <typename T, int VEC> struct alignas(sizeof(T) * VEC) Pack { T e[VEC]; };

// threads of a workgroup: up to 1024 of 128 registers; 512 of 256 where a thread has eight channels (twice the tables)
template <int VEC> constexpr int max_threads() { return VEC == 8 ? 512 : 1024; }
constexpr int MAX_SLAB = 2048;  // channels of a slab: the sums of the backward pass then fit 64 KB of LDS

struct Geo {
  int N, P, C, D;                    // samples of this launch, pixels, channels, channels of a group
  int first, per_client;             // number of the launch's first sample in the batch, samples of a client
  int S, nslab, L, rows;             // channels of a slab, slabs, lanes of a pixel row, pixel rows at a time
  int chunk, nchunk;                 // pixels of a chunk, chunks of a sample
  int nv, pre, tw, tw_ch, tw_gr;     // see slab_sums
  int act;
  float eps;
  long gstride, bstride;
};

__device__ __forceinline__ float act_f(float z, int act) {
  if (act == 1) return z <= 0.f ? 0.f : z;  // (a NaN stays one)
  if (act == 2) return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
  if (act == 3) return z / (1.f + expf(-z));
  return z;
}
__device__ __forceinline__ float act_slope(float z, int act) {
  if (act == 1) return z > 0.f ? 1.f : 0.f;
  if (act == 2)
    return 0.5f * (1.f + erff(z * 0.70710678118654752f)) + z * 0.39894228040143268f * expf(-0.5f * z * z);
  if (act == 3) { const float s = 1.f / (1.f + expf(-z)); return s * (1.f + z * (1.f - s)); }
  return 1.f;
}

// K sums at once over the pixels of a slab, per run of `gw` entries of a pixel row (gw = 1: per channel).
// v[k][j]: this thread's sum of its channel j; nv = 1: the thread's channels lie in one group and are added first.
// Rows of one wave meet in shuffles where L divides 64 (`pre`), the rest through LDS, by teams of `tw` lanes per run.
template <int K, int VEC>
__device__ __forceinline__ void slab_sums(float (&v)[K][VEC], int nv, int gw, int runs, int tw, const Geo& q, int l, int row,
                                          bool active, float* red, float* out) {
  const int t = threadIdx.x, nt = blockDim.x, W = q.L * nv;
  if (VEC > 1 && nv == 1) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int j = 1; j < VEC; ++j) v[k][0] += v[k][j];
    }
  }
  if (q.pre) {
    for (int o = q.L; o < 64; o <<= 1) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          if (j < nv) v[k][j] += __shfl_xor(v[k][j], o, 64);
      }
    }
  }
  const int nr = q.pre ? nt >> 6 : q.rows, rr = q.pre ? t >> 6 : row;
  if (q.pre ? (t & 63) < q.L : active) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (j < nv) red[(k * nr + rr) * W + l * nv + j] = v[k][j];
    }
  }
  __syncthreads();
  const int e0 = t & (tw - 1);
  for (int g = t / tw; g < runs * K; g += nt / tw) {  // (a team's lanes share g: they leave the loop together)
    const int k = g / runs, base = (g - k * runs) * gw;
    float a = 0.f;
    int r = e0 / gw, c = e0 - r * gw;
    const int dr = tw / gw, dc = tw - dr * gw;
    while (r < nr) {
      a += red[(k * nr + r) * W + base + c];
      r += dr; c += dc;
      if (c >= gw) { c -= gw; ++r; }
    }
    for (int o = tw >> 1; o > 0; o >>= 1) a += __shfl_xor(a, o, 64);
    if (e0 == 0) out[g] = a;
  }
  __syncthreads();
}

// which sample / slab / chunk: a sample's slabs and chunks follow each other on one XCD (workgroup ids go round the 8)
__device__ __forceinline__ bool locate(const Geo& q, int& n, int& slab, int& chunk) {
  const int per = q.nslab * q.nchunk, b = blockIdx.x >> 3;
  const int i = b / per, rest = b - i * per;
  n = i * 8 + (blockIdx.x & 7);
  chunk = rest / q.nslab;
  slab = rest - chunk * q.nslab;
  return n < q.N;
}

// PHASE 0: the whole sample is here.  1: leaves (mean, M2) of a pixel chunk.  2: applies joined statistics to a chunk.
template <typename T, int VEC, int R, int PHASE>
__global__ __launch_bounds__(max_threads<VEC>()) void gn_fwd_kernel(Geo q, const T* __restrict__ x, const T* __restrict__ res,
                                                                  const float* __restrict__ gamma,
                                                                  const float* __restrict__ beta, T* __restrict__ y,
                                                                  unsigned char* __restrict__ gate, float* __restrict__ mean,
                                                                  float* __restrict__ rstd, float2* __restrict__ part) {
  extern __shared__ float lds[];
  typedef Pack<T, VEC> V;
  int n, slab, chunk;
  if (!locate(q, n, slab, chunk)) return;
  const int l = threadIdx.x % q.L, row = threadIdx.x / q.L, Gs = q.S / q.D, G = q.C / q.D;
  const bool active = row < q.rows;
  const int p0 = chunk * q.chunk, pn = min(q.chunk, q.P - p0);
  const size_t base = ((size_t)n * q.P + p0) * q.C + (size_t)slab * q.S + (size_t)l * VEC;
  const size_t step = (size_t)q.rows * q.C;
  V xr[R];
  {
    const T* p = x + base + (size_t)row * q.C;
#pragma unroll
    for (int i = 0; i < R; ++i)
      if (active && row + i * q.rows < pn) xr[i] = *reinterpret_cast<const V*>(p + i * step);
  }
  float mu[VEC], rs[VEC];
  int gl[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) gl[j] = (l * VEC + j) / q.D;
  if (PHASE != 2) {
    float *out = lds, *out2 = lds + Gs, *red = lds + 2 * Gs;
    const float inv = 1.f / ((float)pn * (float)q.D);
    const int gw = q.nv == 1 ? q.D / VEC : q.D;
    float v[1][VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[0][j] = 0.f;
#pragma unroll
    for (int i = 0; i < R; ++i)
      if (active && row + i * q.rows < pn)
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[0][j] += to_f(xr[i].e[j]);
    slab_sums<1, VEC>(v, q.nv, gw, Gs, q.tw, q, l, row, active, red, out);
#pragma unroll
    for (int j = 0; j < VEC; ++j) { mu[j] = active ? out[gl[j]] * inv : 0.f; v[0][j] = 0.f; }
#pragma unroll
    for (int i = 0; i < R; ++i)
      if (active && row + i * q.rows < pn)
#pragma unroll
        for (int j = 0; j < VEC; ++j) { const float d = to_f(xr[i].e[j]) - mu[j]; v[0][j] = fmaf(d, d, v[0][j]); }
    slab_sums<1, VEC>(v, q.nv, gw, Gs, q.tw, q, l, row, active, red, out2);
    if (PHASE == 1) {
      for (int g = threadIdx.x; g < Gs; g += blockDim.x)
        part[((size_t)n * q.nchunk + chunk) * G + slab * Gs + g] = make_float2(out[g] * inv, out2[g]);
      return;
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) rs[j] = active ? 1.f / sqrtf(out2[gl[j]] * inv + q.eps) : 0.f;
    if (mean != nullptr)
      for (int g = threadIdx.x; g < Gs; g += blockDim.x) {
        const size_t o = (size_t)n * G + slab * Gs + g;
        mean[o] = out[g] * inv;
        rstd[o] = 1.f / sqrtf(out2[g] * inv + q.eps);
      }
  } else if (active) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const size_t o = (size_t)n * G + slab * Gs + gl[j];
      mu[j] = mean[o]; rs[j] = rstd[o];
    }
  }
  if (!active) return;
  float ga[VEC], be[VEC];
  const int client = (q.first + n) / q.per_client, c0 = slab * q.S + l * VEC;
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    ga[j] = gamma ? gamma[client * q.gstride + c0 + j] : 1.f;
    be[j] = beta ? beta[client * q.bstride + c0 + j] : 0.f;
  }
  const size_t at = base + (size_t)row * q.C;
#pragma unroll
  for (int i = 0; i < R; ++i)
    if (row + i * q.rows < pn) {
      const size_t o = at + i * step;
      float z[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) z[j] = fmaf((to_f(xr[i].e[j]) - mu[j]) * rs[j], ga[j], be[j]);
      if (res != nullptr) {
        const V rv = *reinterpret_cast<const V*>(res + o);
#pragma unroll
        for (int j = 0; j < VEC; ++j) z[j] += to_f(rv.e[j]);
      }
      if (gate != nullptr) {
        unsigned m = 0;
#pragma unroll
        for (int j = 0; j < VEC; ++j) m |= (z[j] > 0.f ? 1u : 0u) << j;
        gate[o / VEC] = (unsigned char)m;
      }
      V w;
#pragma unroll
      for (int j = 0; j < VEC; ++j) from_f(act_f(z[j], q.act), w.e[j]);
      *reinterpret_cast<V*>(y + o) = w;
    }
}

// joins the chunks' (mean, M2): one wave per (sample, group), fixed order
__global__ __launch_bounds__(256) void gn_fwd_join_kernel(const float2* __restrict__ part, int n0, int cnt, int G, int D, int P,
                                                          int chunk, int nchunk, float eps, float* __restrict__ mean,
                                                          float* __restrict__ rstd) {
  const long i = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (i >= (long)cnt * G) return;
  const long n = i / G;
  const int g = (int)(i - n * G);
  const float2* p = part + (size_t)n * nchunk * G + g;
  double s = 0.0;
  for (int k = lane; k < nchunk; k += 64) s += (double)min(chunk, P - k * chunk) * p[(size_t)k * G].x;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  const double m = s / P;
  double m2 = 0.0;
  for (int k = lane; k < nchunk; k += 64) {
    const float2 e = p[(size_t)k * G];
    const double d = (double)e.x - m;
    m2 += (double)e.y + (double)min(chunk, P - k * chunk) * D * d * d;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m2 += __shfl_xor(m2, o, 64);
  if (lane == 0) {
    const size_t o = (size_t)(n0 + n) * G + g;
    mean[o] = (float)m;
    rstd[o] = (float)(1.0 / sqrt(m2 / ((double)P * D) + (double)eps));
  }
}

// PHASE as in the forward kernel: 0 whole sample, 1 leaves (A, B) per channel of a chunk, 2 applies the joined means.
// sums: PHASE 0 / 1 out, [N][nchunk][C] (A, B).  means: PHASE 2 in, [N][G] (mean of gamma g, mean of gamma g xhat).
template <typename T, int VEC, int R, int PHASE>
__global__ __launch_bounds__(max_threads<VEC>()) void gn_bwd_kernel(Geo q, const T* __restrict__ x, const T* __restrict__ res,
                                                                  const T* __restrict__ gy, const unsigned char* __restrict__ gate,
                                                                  const float* __restrict__ gamma,
                                                                  const float* __restrict__ beta,
                                                                  const float* __restrict__ mean,
                                                                  const float* __restrict__ rstd, T* __restrict__ dx,
                                                                  T* __restrict__ dres, float2* __restrict__ sums,
                                                                  const float2* __restrict__ means) {
  extern __shared__ float lds[];
  typedef Pack<T, VEC> V;
  int n, slab, chunk;
  if (!locate(q, n, slab, chunk)) return;
  const int l = threadIdx.x % q.L, row = threadIdx.x / q.L, Gs = q.S / q.D, G = q.C / q.D;
  const bool active = row < q.rows;
  const int p0 = chunk * q.chunk, pn = min(q.chunk, q.P - p0);
  const size_t at = ((size_t)n * q.P + p0 + row) * q.C + (size_t)slab * q.S + (size_t)l * VEC;
  const size_t step = (size_t)q.rows * q.C;
  V xr[R], gr[R];
#pragma unroll
  for (int i = 0; i < R; ++i)
    if (active && row + i * q.rows < pn) {
      xr[i] = *reinterpret_cast<const V*>(x + at + i * step);
      gr[i] = *reinterpret_cast<const V*>(gy + at + i * step);
    }
  float mu[VEC], rs[VEC], ga[VEC], be[VEC];
  const int client = (q.first + n) / q.per_client, c0 = slab * q.S + l * VEC;
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    mu[j] = rs[j] = ga[j] = be[j] = 0.f;
    if (active) {
      const size_t o = (size_t)n * G + (c0 + j) / q.D;
      mu[j] = mean[o]; rs[j] = rstd[o];
      ga[j] = gamma ? gamma[client * q.gstride + c0 + j] : 1.f;
      be[j] = beta ? beta[client * q.bstride + c0 + j] : 0.f;
    }
  }
  const int act = q.act;
  // g of vector i: gy behind the activation.  The gate byte or the recomputed z decides; z takes the residual again
  // where the activation is smooth.
  auto slope = [&](int i, float (&g)[VEC]) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) g[j] = to_f(gr[i].e[j]);
    if (act == 0) return;
    if (gate != nullptr) {
      const unsigned m = gate[(at + i * step) / VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) g[j] = (m >> j) & 1u ? g[j] : 0.f;
      return;
    }
    float z[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) z[j] = fmaf((to_f(xr[i].e[j]) - mu[j]) * rs[j], ga[j], be[j]);
    if (res != nullptr) {
      const V rv = *reinterpret_cast<const V*>(res + at + i * step);
#pragma unroll
      for (int j = 0; j < VEC; ++j) z[j] += to_f(rv.e[j]);
    }
    if (act == 1) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) g[j] = z[j] > 0.f ? g[j] : 0.f;
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) g[j] *= act_slope(z[j], act);
    }
  };
  float m1[VEC], m2[VEC];
  if (PHASE != 2) {
    float v[2][VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[0][j] = v[1][j] = 0.f;
#pragma unroll
    for (int i = 0; i < R; ++i)
      if (active && row + i * q.rows < pn) {
        float g[VEC];
        slope(i, g);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          v[0][j] += g[j];
          v[1][j] = fmaf(g[j], (to_f(xr[i].e[j]) - mu[j]) * rs[j], v[1][j]);
        }
        if (sizeof(T) == 4 && PHASE == 0) {  // (fp32: g replaces gy in its registers; 16-bit types would round it)
#pragma unroll
          for (int j = 0; j < VEC; ++j) from_f(g[j], gr[i].e[j]);
        }
      }
    float *ch = lds, *gsum = lds + 2 * q.S, *red = gsum + 2 * Gs;
    slab_sums<2, VEC>(v, VEC, 1, q.S, q.tw_ch, q, l, row, active, red, ch);  // ch[0..S): A, ch[S..2S): B
    for (int c = threadIdx.x; c < q.S; c += blockDim.x)
      sums[((size_t)n * q.nchunk + chunk) * q.C + slab * q.S + c] = make_float2(ch[c], ch[q.S + c]);
    if (PHASE == 1) return;
    const int tw = q.tw_gr, e0 = threadIdx.x & (tw - 1);
    for (int g = threadIdx.x / tw; g < 2 * Gs; g += blockDim.x / tw) {
      const int k = g / Gs, cb = (g - k * Gs) * q.D;
      float a = 0.f;
      for (int e = e0; e < q.D; e += tw) {
        const float w = gamma ? gamma[client * q.gstride + slab * q.S + cb + e] : 1.f;
        a = fmaf(w, ch[k * q.S + cb + e], a);
      }
      for (int o = tw >> 1; o > 0; o >>= 1) a += __shfl_xor(a, o, 64);
      if (e0 == 0) gsum[g] = a;
    }
    __syncthreads();
    const float inv = 1.f / ((float)q.P * (float)q.D);
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const int g = (l * VEC + j) / q.D;
      m1[j] = active ? gsum[g] * inv : 0.f;
      m2[j] = active ? gsum[Gs + g] * inv : 0.f;
    }
  } else if (active) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const float2 m = means[(size_t)n * G + (c0 + j) / q.D];
      m1[j] = m.x; m2[j] = m.y;
    }
  }
  if (!active) return;
#pragma unroll
  for (int i = 0; i < R; ++i)
    if (row + i * q.rows < pn) {
      const size_t o = at + i * step;
      float g[VEC];
      if (sizeof(T) == 4 && PHASE == 0) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) g[j] = to_f(gr[i].e[j]);
      } else {
        slope(i, g);
      }
      if (dx != nullptr) {
        V w;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float xh = (to_f(xr[i].e[j]) - mu[j]) * rs[j];
          from_f(rs[j] * (fmaf(g[j], ga[j], -m1[j]) - xh * m2[j]), w.e[j]);
        }
        *reinterpret_cast<V*>(dx + o) = w;
      }
      if (dres != nullptr) {
        V w;
#pragma unroll
        for (int j = 0; j < VEC; ++j) from_f(g[j], w.e[j]);
        *reinterpret_cast<V*>(dres + o) = w;
      }
    }
}

// joins the chunks' (A, B) of one (sample, slab): channel sums for the affine gradients, group means for the second sweep
__global__ __launch_bounds__(256) void gn_bwd_join_kernel(const float2* __restrict__ part, int n0, int C, int S, int D, int P,
                                                          int nchunk, int per_client, const float* __restrict__ gamma,
                                                          long gstride, float2* __restrict__ sums, float2* __restrict__ means) {
  extern __shared__ float lds[];
  const int nslab = C / S, i = blockIdx.x / nslab, slab = blockIdx.x - i * nslab, n = n0 + i;
  for (int c = threadIdx.x; c < S; c += 256) {
    double a = 0.0, b = 0.0;
    const float2* p = part + (size_t)i * nchunk * C + slab * S + c;
    for (int k = 0; k < nchunk; ++k) { const float2 e = p[(size_t)k * C]; a += (double)e.x; b += (double)e.y; }
    sums[(size_t)n * C + slab * S + c] = make_float2((float)a, (float)b);
    const float w = gamma ? gamma[(n / per_client) * gstride + slab * S + c] : 1.f;
    lds[c] = w * (float)a; lds[S + c] = w * (float)b;
  }
  __syncthreads();
  const int Gs = S / D;
  const double inv = 1.0 / ((double)P * D);
  for (int g = threadIdx.x; g < Gs; g += 256) {
    double a = 0.0, b = 0.0;
    for (int c = g * D; c < (g + 1) * D; ++c) { a += (double)lds[c]; b += (double)lds[S + c]; }
    means[(size_t)n * (C / D) + slab * Gs + g] = make_float2((float)(a * inv), (float)(b * inv));
  }
}

// dgamma / dbeta of a client: its samples' (A, B), 16 channels a workgroup, 64 rows of threads, fixed order
constexpr int AFF_CH = 16, AFF_ROWS = 64;
__global__ __launch_bounds__(AFF_CH * AFF_ROWS) void gn_affine_kernel(const float2* __restrict__ sums, int per_client, int C,
                                                                      const float* __restrict__ coef, float* __restrict__ dg,
                                                                      float* __restrict__ db, long ld, int accumulate) {
  __shared__ double red[AFF_ROWS][AFF_CH][2];
  const int chl = threadIdx.x % AFF_CH, r0 = threadIdx.x / AFF_CH, groups = (C + AFF_CH - 1) / AFF_CH;
  const int k = blockIdx.x / groups, ch = (blockIdx.x - k * groups) * AFF_CH + chl;
  double a = 0.0, b = 0.0;
  if (ch < C)
    for (int r = r0; r < per_client; r += AFF_ROWS) {
      const float2 e = sums[((size_t)k * per_client + r) * C + ch];
      a += (double)e.x; b += (double)e.y;
    }
  red[r0][chl][0] = a; red[r0][chl][1] = b;
  for (int o = AFF_ROWS / 2; o > 0; o >>= 1) {
    __syncthreads();
    if (r0 < o) { red[r0][chl][0] += red[r0 + o][chl][0]; red[r0][chl][1] += red[r0 + o][chl][1]; }
  }
  if (r0 != 0 || ch >= C) return;
  const float s = coef ? coef[k] : 1.f;
  const float vg = s * (float)red[0][chl][1], vb = s * (float)red[0][chl][0];
  if (dg != nullptr) { float* p = dg + k * ld + ch; *p = accumulate ? *p + vg : vg; }
  if (db != nullptr) { float* p = db + k * ld + ch; *p = accumulate ? *p + vb : vb; }
}

// ---------------------------------------------------------------------------------------------------------------
inline int pow2_up(int v) { int p = 1; while (p < v) p <<= 1; return p; }

struct Plan { Geo q; int threads, R, split; size_t lds; long piece; };

// The launch of one direction (`hold`: 16-byte vectors of registers per pixel vector — 1 forward, 2 backward).
// Returns false where no slab of whole groups fits a workgroup.
bool make_plan(Plan& pl, long N, long P, int C, int G, int esize, int vec, int hold, int per_client) {
  const int D = C / G, maxt = vec == 8 ? 512 : 1024, maxr = 16 / hold;
  Geo& q = pl.q;
  q.N = (int)N; q.P = (int)P; q.C = C; q.D = D;
  q.per_client = per_client;
  // Slabs: as few as give workgroups of at most 256 threads x `maxr` vectors, but with pixel rows of at least a cache
  // line (128 bytes).  Narrower ones (down to 64 bytes) only where a sample would not fit a workgroup otherwise, and down
  // to single groups where the chip would stand half empty.  A sample that does not fit even so is split into chunks of
  // the widest slabs.
  const long want = (long)256 * maxr, most = (long)maxt * maxr;
  int widest = 0, best = 0;
  for (int ns = 1; ns <= G; ++ns) {
    if (G % ns || (C / ns) % vec || C / ns > MAX_SLAB || C / ns / vec > maxt) continue;
    if (best == 0) { widest = best = ns; continue; }
    const long row = (long)(C / ns) * esize, now = P * (C / best / vec);
    if ((now > want && row >= 128) || (now > most && row >= 64) || (now > 64 && now <= most && N * best < 512)) best = ns;
  }
  if (best == 0) return false;
  pl.split = P * (C / best / vec) > most;
  if (pl.split) best = widest;
  q.nslab = best;
  q.S = C / best;
  q.L = q.S / vec;
  const long unit = pl.split ? (long)256 * maxr : P * q.L;
  int t = (int)((unit + maxr / 2 - 1) / (maxr / 2));
  t = (t + 63) / 64 * 64;
  if (t < 64) t = 64;
  if (t < q.L) t = (q.L + 63) / 64 * 64;
  if (t > maxt) t = maxt;
  q.pre = q.L < 64 && 64 % q.L == 0;
  pl.threads = t;
  q.rows = t / q.L;
  if (pl.split) {
    q.chunk = q.rows * (maxr / 2);
    q.nchunk = (int)((P + q.chunk - 1) / q.chunk);
    pl.R = maxr / 2;
  } else {
    q.chunk = (int)P; q.nchunk = 1;
    int R = (int)((P + q.rows - 1) / q.rows);
    if (R > maxr) {  // a row count that does not divide evenly: more threads, at worst the largest workgroup
      pl.threads = t = maxt;
      q.rows = t / q.L;
      R = (int)((P + q.rows - 1) / q.rows);
      if (R > maxr) {
        pl.split = 1;
        q.chunk = q.rows * (maxr / 2);
        q.nchunk = (int)((P + q.chunk - 1) / q.chunk);
        R = maxr / 2;
      }
    }
    pl.R = pow2_up(R);
  }
  q.nv = (vec > 1 && D % vec == 0) ? 1 : vec;
  const int Gs = q.S / D, nr = q.pre ? pl.threads / 64 : q.rows;
  const int gw = q.nv == 1 ? D / vec : D;
  auto team = [](long n) { int p = pow2_up((int)(n > 64 ? 64 : n)); return p > 64 ? 64 : p; };
  q.tw = team((long)nr * gw);
  q.tw_ch = team(nr);
  q.tw_gr = team(D);
  pl.lds = hold == 1 ? (2 * (size_t)Gs + (size_t)nr * q.L * q.nv) * 4
                     : (2 * (size_t)q.S + 2 * (size_t)Gs + 2 * (size_t)nr * q.S) * 4;
  // pieces of the batch whose activations (x, or x and gy) stay in the last-level cache between the two sweeps
  const long wgs = (long)q.nslab * q.nchunk, fit = ((1L << 32) - 1) / ((long)pl.threads * wgs) / 8 * 8;
  pl.piece = N;
  if (pl.split) pl.piece = (96L << 20) / (P * C * esize * hold);
  if (pl.piece > fit) pl.piece = fit;  // a grid counts its threads in 32 bits
  if (pl.piece > N) pl.piece = N;
  if (pl.piece < 1) pl.piece = 1;
  return wgs * 8 * pl.threads < (1L << 32);
}

template <typename T, int VEC, int PHASE>
void launch_fwd(const Plan& pl, const Geo& q, const void* x, const void* res, const float* gamma, const float* beta, void* y,
                unsigned char* gate, float* mean, float* rstd, float2* part, hipStream_t st) {
  const dim3 grid((unsigned)((q.N + 7) / 8 * 8) * q.nslab * q.nchunk), block(pl.threads);
#define GN_FWD(RR)                                                                                                         \
  hipLaunchKernelGGL((gn_fwd_kernel<T, VEC, RR, PHASE>), grid, block, pl.lds, st, q, (const T*)x, (const T*)res, gamma,    \
                     beta, (T*)y, gate, mean, rstd, part)
  if constexpr (PHASE != 0) {
    GN_FWD(8);
  } else {
    switch (pl.R) {
      case 1: case 2: GN_FWD(2); break;
      case 4: GN_FWD(4); break;
      case 8: GN_FWD(8); break;
      default: GN_FWD(16); break;
    }
  }
#undef GN_FWD
}

template <typename T, int VEC, int PHASE>
void launch_bwd(const Plan& pl, const Geo& q, const void* x, const void* res, const void* gy, const unsigned char* gate,
                const float* gamma, const float* beta, const float* mean, const float* rstd, void* dx, void* dres,
                float2* sums, const float2* means, hipStream_t st) {
  const dim3 grid((unsigned)((q.N + 7) / 8 * 8) * q.nslab * q.nchunk), block(pl.threads);
#define GN_BWD(RR)                                                                                                         \
  hipLaunchKernelGGL((gn_bwd_kernel<T, VEC, RR, PHASE>), grid, block, pl.lds, st, q, (const T*)x, (const T*)res,           \
                     (const T*)gy, gate, gamma, beta, mean, rstd, (T*)dx, (T*)dres, sums, means)
  if constexpr (PHASE != 0) {
    GN_BWD(4);
  } else {
    switch (pl.R) {
      case 1: case 2: GN_BWD(2); break;
      case 4: GN_BWD(4); break;
      default: GN_BWD(8); break;
    }
  }
#undef GN_BWD
}

template <typename T, int VEC>
int forward_t(Plan& pl, const void* x, const void* res, const float* gamma, const float* beta, void* y, unsigned char* gate,
              float* mean, float* rstd, float* ws, hipStream_t st) {
  const Geo q = pl.q;
  const int G = q.C / q.D, N = q.N;
  const size_t per = (size_t)q.P * q.C;
  for (long n0 = 0; n0 < N; n0 += pl.piece) {
    Geo s = q;
    s.N = (int)(N - n0 < pl.piece ? N - n0 : pl.piece);
    s.first = (int)n0;
    const T *xp = (const T*)x + n0 * per, *rp = res ? (const T*)res + n0 * per : nullptr;
    T* yp = (T*)y + n0 * per;
    unsigned char* tp = gate ? gate + n0 * per / VEC : nullptr;
    float *mp = mean ? mean + n0 * G : nullptr, *sp = rstd ? rstd + n0 * G : nullptr;
    if (!pl.split) {
      launch_fwd<T, VEC, 0>(pl, s, xp, rp, gamma, beta, yp, tp, mp, sp, nullptr, st);
      continue;
    }
    launch_fwd<T, VEC, 1>(pl, s, xp, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, (float2*)ws, st);
    hipLaunchKernelGGL(gn_fwd_join_kernel, dim3(cdiv((long)s.N * G, 4)), dim3(256), 0, st, (const float2*)ws, (int)n0, s.N, G,
                       q.D, q.P, q.chunk, q.nchunk, q.eps, mean, rstd);
    launch_fwd<T, VEC, 2>(pl, s, xp, rp, gamma, beta, yp, tp, mp, sp, nullptr, st);
  }
  return 0;
}

template <typename T, int VEC>
int backward_t(Plan& pl, const void* x, const void* res, const void* gy, const unsigned char* gate, const float* gamma,
               const float* beta, const float* mean, const float* rstd, void* dx, void* dres, float* ws, hipStream_t st) {
  const Geo q = pl.q;
  const int G = q.C / q.D, N = q.N;
  float2* sums = (float2*)ws;  // [N][C]
  float2* means = sums + (size_t)N * q.C;  // [N][G]               (these two: split plans alone)
  float2* part = means + (size_t)N * G;    // [piece][nchunk][C]
  const size_t per = (size_t)q.P * q.C;
  for (long n0 = 0; n0 < N; n0 += pl.piece) {
    Geo s = q;
    s.N = (int)(N - n0 < pl.piece ? N - n0 : pl.piece);
    s.first = (int)n0;
    const T *xp = (const T*)x + n0 * per, *gp = (const T*)gy + n0 * per, *rp = res ? (const T*)res + n0 * per : nullptr;
    const unsigned char* tp = gate ? gate + n0 * per / VEC : nullptr;
    T *dp = dx ? (T*)dx + n0 * per : nullptr, *ep = dres ? (T*)dres + n0 * per : nullptr;
    if (!pl.split) {
      launch_bwd<T, VEC, 0>(pl, s, xp, rp, gp, tp, gamma, beta, mean + n0 * G, rstd + n0 * G, dp, ep, sums + n0 * q.C, nullptr,
                            st);
      continue;
    }
    launch_bwd<T, VEC, 1>(pl, s, xp, rp, gp, tp, gamma, beta, mean + n0 * G, rstd + n0 * G, nullptr, nullptr, part, nullptr,
                          st);
    hipLaunchKernelGGL(gn_bwd_join_kernel, dim3((unsigned)s.N * q.nslab), dim3(256), 2 * (size_t)q.S * 4, st, part, (int)n0,
                       q.C, q.S, q.D, q.P, q.nchunk, q.per_client, gamma, q.gstride, sums, means);
    if (dx != nullptr || dres != nullptr)
      launch_bwd<T, VEC, 2>(pl, s, xp, rp, gp, tp, gamma, beta, mean + n0 * G, rstd + n0 * G, dp, ep, nullptr, means + n0 * G,
                            st);
  }
  return 0;
}

bool valid(long N, long P, int C, int G, int vec, int dtype, int per_client) {
  if (N < 1 || P < 1 || C < 1 || G < 1 || C % G || per_client < 1 || N % per_client) return false;
  if (dtype < 0 || dtype > 2 || (vec != 1 && vec != (dtype == 0 ? 4 : 8)) || C % vec) return false;
  // grids and in-kernel counters are 32 bits, offsets 64
  return N < (1L << 24) && P < (1L << 30) && (double)N * P * C < 9e15;
}

}  // namespace

// dtype 0 fp32, 1 bf16, 2 fp16; vec: elements per 16 bytes, or 1 where C or an address does not allow it.
// Workspace bytes of a direction (0 forward, 1 backward); -1: not supported (a group's channels exceed a workgroup).
BLADES_API long blades_group_norm_ws(long N, long P, int C, int G, int dtype, int vec, int direction) {
  Plan pl;
  if (!valid(N, P, C, G, vec, dtype, 1)) return -1;
  if (!make_plan(pl, N, P, C, G, dtype == 0 ? 4 : 2, vec, direction ? 2 : 1, 1)) return -1;
  const long g = C / pl.q.D;
  if (direction == 0) return pl.split ? pl.piece * pl.q.nchunk * g * 8 : 0;
  return (N * C + (pl.split ? N * g + pl.piece * pl.q.nchunk * C : 0)) * 8;
}

// gamma / beta: null, one vector (stride 0) or one per client (stride in floats).  mean / rstd [N][G]: may be null where
// no backward pass follows (then not for a split plan: callers always pass them).  gate: one byte per vector, null: none.
BLADES_API int blades_group_norm_forward(const void* x, const void* res, const float* gamma, const float* beta, long N, long P,
                                         int C, int G, float eps, int act, int per_client, long gstride, long bstride, void* y,
                                         void* gate, float* mean, float* rstd, float* ws, int dtype, int vec, hipStream_t st) {
  Plan pl;
  if (!valid(N, P, C, G, vec, dtype, per_client) || act < 0 || act > 3) return 1;
  if (!make_plan(pl, N, P, C, G, dtype == 0 ? 4 : 2, vec, 1, per_client)) return 2;
  pl.q.eps = eps; pl.q.act = act; pl.q.gstride = gstride; pl.q.bstride = bstride; pl.q.first = 0;
  unsigned char* gt = (unsigned char*)gate;
#define GN_F(T, V) return forward_t<T, V>(pl, x, res, gamma, beta, y, gt, mean, rstd, ws, st)
  if (dtype == 0) { if (vec == 4) GN_F(float, 4); GN_F(float, 1); }
  if (dtype == 1) { if (vec == 8) GN_F(Bf16, 8); GN_F(Bf16, 1); }
  if (vec == 8) GN_F(Half, 8);
  GN_F(Half, 1);
#undef GN_F
}

// dx / dres may be null.  dgamma / dbeta: rows of `ld` floats per client (an update matrix's rows or a [clients][C]
// tensor), scaled by coef[client] (null: 1) and added to what is there where `accumulate`; null: not wanted.
BLADES_API int blades_group_norm_backward(const void* x, const void* res, const void* gy, const void* gate, const float* gamma,
                                          const float* beta, const float* mean, const float* rstd, long N, long P, int C,
                                          int G, int act, int per_client, long gstride, long bstride, void* dx, void* dres,
                                          const float* coef, float* dgamma, float* dbeta, long ld, int accumulate, float* ws,
                                          int dtype, int vec, hipStream_t st) {
  Plan pl;
  if (!valid(N, P, C, G, vec, dtype, per_client) || act < 0 || act > 3) return 1;
  if (!make_plan(pl, N, P, C, G, dtype == 0 ? 4 : 2, vec, 2, per_client)) return 2;
  pl.q.eps = 0.f; pl.q.act = act; pl.q.gstride = gstride; pl.q.bstride = bstride; pl.q.first = 0;
  const unsigned char* gt = (const unsigned char*)gate;
  int rc = 3;
#define GN_B(T, V) rc = backward_t<T, V>(pl, x, res, gy, gt, gamma, beta, mean, rstd, dx, dres, ws, st)
  if (dtype == 0) { if (vec == 4) GN_B(float, 4); else GN_B(float, 1); }
  else if (dtype == 1) { if (vec == 8) GN_B(Bf16, 8); else GN_B(Bf16, 1); }
  else { if (vec == 8) GN_B(Half, 8); else GN_B(Half, 1); }
#undef GN_B
  if (rc == 0 && (dgamma != nullptr || dbeta != nullptr))
    hipLaunchKernelGGL(gn_affine_kernel, dim3((unsigned)(N / per_client) * cdiv(C, AFF_CH)), dim3(AFF_CH * AFF_ROWS), 0, st,
                       (const float2*)ws, per_client, C, coef, dgamma, dbeta, ld, accumulate);
  return rc;
}
