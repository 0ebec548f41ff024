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
// (four, or one where the channel count or an address does not allow it), so a thread keeps its channels for the whole sweep.
// A sample too large for a workgroup's registers is
// cut into pixel chunks: a first sweep leaves (mean, M2) or (A, B) of each, small kernels join them in chunk order, and a
// second sweep applies, from the last sample to the first: what the first sweep read last is still in the 256 MB cache
// (walking the batch in pieces that fit it as a whole costs more in launches than it saves: 48 x 64 x 112 x 112 fp32
// forward + backward 380 us in pieces of 96 MB, 319 in 180 MB, 292 at once).  All sums are fp32 in a fixed order (double
// where many partial sums meet): bitwise reproducible.
//
// Bound by memory.  Kernel times on average over training passes (MI355X; copies run at 5.0 - 5.4 TB/s beyond the last-level
// cache, at 8 within it): 2048 x 64 x 32 x 32 fp32 forward 196 us (5.5 TB/s), backward 332 (4.9); 2048 x 128 x 16 x 16 bf16 SiLU
// 50 and 91 (5.4, 4.4); 2048 x 512 x 4 x 4 fp32 with a residual 33 and 56 (6.2, 4.9); two sweeps of 48 x 64 x 112 x 112 fp32
// GELU 28 + 49 and 53 + 74.  fp16 is slower than bf16 (2048 x 128 x 16 x 16: 70 and 187 us against 46 and 77): its conversions
// to 32 bits stay in registers, and the backward kernel's no longer fit.
#pragma once
#include "common.h"
#include "layers_abi.h"

namespace groupnorm {

struct Half { unsigned short v; };
struct Bf16 { unsigned short v; };

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(Bf16 v) { return __uint_as_float((unsigned)v.v << 16); }
__device__ __forceinline__ float to_f(Half v) { return (float)__builtin_bit_cast(_Float16, v.v); }
__device__ __forceinline__ void from_f(float f, float& o) { o = f; }
__device__ __forceinline__ void from_f(float f, Bf16& o) { o.v = __builtin_bit_cast(unsigned short, (__bf16)f); }
__device__ __forceinline__ void from_f(float f, Half& o) { o.v = __builtin_bit_cast(unsigned short, (_Float16)f); }

template <typename T, int VEC> struct alignas(sizeof(T) * VEC) Pack { T e[VEC]; };

constexpr int MAX_THREADS = 1024;  // of 128 registers
constexpr int BLOCK = 4;           // vectors a thread has in flight in the sweeps over pixel chunks
// channels of a slab with several groups, and of a single group: the backward pass's sums then fit 64 KB of LDS
constexpr int MAX_SLAB = 1024, MAX_GROUP = 2048;

struct Geo {
  int N, P, C, D;                    // samples of this launch, pixels, channels, channels of a group
  int first, per_client;             // number of the launch's first sample in the batch, samples of a client
  int S, nslab, L, rows;             // channels of a slab, slabs, lanes of a pixel row, pixel rows at a time
  int chunk, nchunk;                 // pixels of a chunk, chunks of a sample
  int through;                       // outputs past the caches (store_out)
  int back;                          // samples from the last one (the second sweep: what the first read last is still near)
  int pre, tw, tw_ch, tw_gr;         // see slab_sums
  int act;
  float eps;
  long gstride, bstride;
};

// FINE below (32-bit outputs): errors of a few half steps everywhere; otherwise of |z| or z^2 of them in the tails, far under
// the half step of a 16-bit output.
//
// 1 / (1 + e^-z): the hardware's 2^x and reciprocal, one unit in the last place each.  FINE: what the exponent's rounding
// lost, |z| half steps of the result, is made up for.  (z is clamped for that: beyond 128 the result is 0 or 1 anyway.)
template <bool FINE>
__device__ __forceinline__ float sigmoid(float z) {
  constexpr float C = -1.44269504088896f;
  if (!FINE) return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * C));
  const float v = __builtin_amdgcn_fmed3f(z, -128.f, 128.f), t = v * C;
  const float lost = fmaf(v, C, -t) + v * (float)(-1.4426950408889634074 - (double)C);
  return __builtin_amdgcn_rcpf(fmaf(__builtin_amdgcn_exp2f(t), fmaf(lost, 0.69314718055994531f, 1.f), 1.f));
}
// The normal distribution's integral; e = exp(-z^2 / 2), which the density needs as well.  Its tail is e times a polynomial in
// t = 1 / (1 + 0.3 |z|), least squares of the relative error at Chebyshev nodes (at most 1.8e-7 for every z, so that small
// values keep their digits: 1 - erf would not); a dozen instructions where the library's error function is sixty.  FINE: within
// one standard deviation 0.5 + z r(z^2), fitted alike (7.6e-10), whose rounding is a third.
template <bool FINE>
__device__ __forceinline__ float normal_cdf(float z, float e) {
  const float a = fabsf(z), t = __builtin_amdgcn_rcpf(fmaf(0.3f, a, 1.f));
  float p = 3.622337431e-02f;
  p = fmaf(p, t, -1.593545526e-01f);
  p = fmaf(p, t, 2.098195851e-01f);
  p = fmaf(p, t, -5.664497241e-02f);
  p = fmaf(p, t, 1.300049871e-01f);
  p = fmaf(p, t, 9.951351583e-02f);
  p = fmaf(p, t, 1.208121851e-01f);
  p = fmaf(p, t, 1.196258739e-01f);
  const float tail = p * t * e, far = z < 0.f ? tail : 1.f - tail;
  if (!FINE) return far;
  const float u = z * z;
  float r = -7.662608368e-06f;
  r = fmaf(r, u, 1.135074781e-04f);
  r = fmaf(r, u, -1.186348498e-03f);
  r = fmaf(r, u, 9.973330423e-03f);
  r = fmaf(r, u, -6.649035960e-02f);
  r = fmaf(r, u, 3.989422917e-01f);
  return a < 1.f ? fmaf(z, r, 0.5f) : far;
}
__device__ __forceinline__ float gauss(float z) { return __builtin_amdgcn_exp2f(z * z * -0.72134752044448f); }

// AK: kind of activation the code is made for (0 none or ReLU, 2 GELU, 3 SiLU, -1 any: `act` decides)
template <int AK, bool FINE>
__device__ __forceinline__ float act_f(float z, int act) {
  if (AK == 2 || (AK < 0 && act == 2)) return z * normal_cdf<FINE>(z, gauss(z));
  if (AK == 3 || (AK < 0 && act == 3)) return z * sigmoid<FINE>(z);
  return act == 1 && z <= 0.f ? 0.f : z;  // (a NaN stays one)
}
template <int AK, bool FINE>
__device__ __forceinline__ float act_slope(float z, int act) {  // of the smooth ones
  if (AK == 2 || (AK < 0 && act == 2)) {
    const float e = gauss(z);
    return fmaf(z * 0.39894228040143268f, e, normal_cdf<FINE>(z, e));
  }
  const float s = sigmoid<FINE>(z);
  return s * fmaf(z, 1.f - s, 1.f);
}

// a run of floats at any 4-byte address (the hardware takes 16 bytes from there at once)
template <int VEC> struct Floats { float e[VEC]; };
template <int VEC>
__device__ __forceinline__ void load_floats(const float* p, float fill, float (&v)[VEC]) {
  if (p == nullptr) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = fill;
  } else {
    const Floats<VEC> t = *reinterpret_cast<const Floats<VEC>*>(p);
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = t.e[j];
  }
}

// K sums at once over the pixels of a slab, per run of `gw` entries of a pixel row.  v[k]: this thread's NV sums, entry
// l * NV + j of its row.  Rows of one wave meet in shuffles where L divides 64 (`pre`), the rest through LDS, by teams of
// `tw` lanes per run.  out[k * runs + r] is there for all threads on return.
template <int K, int NV>
__device__ __forceinline__ void slab_sums(float (&v)[K][NV], int gw, int runs, int tw, const Geo& q, int l, int row, bool active,
                                          float* red, float* out) {
  const int t = threadIdx.x, nt = blockDim.x, W = q.L * NV;
  if (q.pre) {
    for (int o = q.L; o < 64; o <<= 1) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int j = 0; j < NV; ++j) v[k][j] += __shfl_xor(v[k][j], o, 64);
      }
    }
  }
  const int nr = q.pre ? nt >> 6 : q.rows, rr = q.pre ? t >> 6 : row;
  if (q.pre ? (t & 63) < q.L : active) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int j = 0; j < NV; ++j) red[(k * nr + rr) * W + l * NV + j] = v[k][j];
    }
  }
  __syncthreads();
  const int e0 = t & (tw - 1), dr = tw / gw, dc = tw - dr * gw, r0 = e0 / gw, c0 = e0 - r0 * gw;
  for (int g = t / tw; g < runs * K; g += nt / tw) {  // (a team's lanes share g: they leave the loop together)
    const int k = g / runs, base = (g - k * runs) * gw;
    float a = 0.f;
    int r = r0, c = c0;
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

// Which sample / slab / chunk this workgroup has (a sample's slabs and chunks follow each other on one XCD: workgroup ids
// go round the 8), and which channels this thread.  NM: groups a thread's VEC channels can lie in (1, or VEC: any).
template <int VEC, int NM>
struct Place {
  int n, slab, chunk, client, l, row, p0, pn, G, Gs, c0;
  int g[NM];  // groups of this thread's channels, within the slab
  bool here, active;
  size_t at, step;  // this thread's first vector, from pixel row to pixel row
  __device__ __forceinline__ explicit Place(const Geo& q) {
    const int per = q.nslab * q.nchunk, b = blockIdx.x >> 3, i = b / per, rest = b - i * per;
    n = i * 8 + (blockIdx.x & 7);
    here = n < q.N;
    if (q.back) n = q.N - 1 - n;
    chunk = rest / q.nslab;
    slab = rest - chunk * q.nslab;
    row = threadIdx.x / q.L;
    l = threadIdx.x - row * q.L;
    active = row < q.rows;
    G = q.C / q.D; Gs = q.S / q.D;
    client = (q.first + n) / q.per_client;
    p0 = chunk * q.chunk; pn = min(q.chunk, q.P - p0);
    c0 = slab * q.S + l * VEC;
    at = ((size_t)n * q.P + p0 + row) * q.C + c0;
    step = (size_t)q.rows * q.C;
    const int a = l * VEC / q.D;
    int d = l * VEC - a * q.D, k = a;
#pragma unroll
    for (int j = 0; j < NM; ++j) {
      g[j] = k;
      if (++d == q.D) { d = 0; ++k; }
    }
  }
};

template <typename T, int VEC, int NM>
__device__ __forceinline__ void normed(const Pack<T, VEC>& x, const float (&mu)[NM], const float (&rs)[NM], float (&xh)[VEC]) {
#pragma unroll
  for (int j = 0; j < VEC; ++j) xh[j] = (to_f(x.e[j]) - mu[NM == 1 ? 0 : j]) * rs[NM == 1 ? 0 : j];
}

// ---------------------------------------------------------------------------------------------------------------
inline int pow2_up(int v) { int p = 1; while (p < v) p <<= 1; return p; }

struct Plan { Geo q; int threads, R, split, one; size_t lds; long piece, ws; };
// both directions of a layer's shape
struct Layer { Plan fwd, bwd; int dtype, vec; };

// The launch of one direction (`hold`: vectors of registers per vector of the sample — 1 forward, 2 backward).
// Returns false where no slab of whole groups fits a workgroup.
inline bool make_plan(Plan& pl, long N, long P, int C, int G, int esize, int vec, int hold, int per_client) {
  const int D = C / G, maxt = MAX_THREADS, maxr = hold == 1 || esize == 2 ? 16 : 8;
  Geo& q = pl.q;
  q.N = (int)N; q.P = (int)P; q.C = C; q.D = D;
  q.per_client = per_client;
  q.first = 0;
  q.back = 0;
  // Outputs of up to 256 MB, the last-level cache, are stored past it.  Kernel times on average, stored past it against through
  // it: repeated alone / in a row of three with a product of equal size in front and behind.
  //   2048 x 128 x 16 x 16 bf16 (128 MB)  forward 53 : 64 / 147 : 151   backward 104 : 115 / 206 : 207
  //   2048 x 512 x 4 x 4 fp32 (64 MB)     forward 31 : 36 /  87 :  85   backward  55 :  60 / 104 : 107
  //   2048 x 64 x 32 x 32 fp32 (512 MB)   forward 212 : 193 / 577 : 547 backward 321 : 328 / 666 : 663   (hence the limit)
  q.through = N * P * C * esize <= (256L << 20);
  // Slabs: as few as give workgroups of at most 256 threads x `maxr` vectors, but with pixel rows of at least a cache
  // line (128 bytes).  Narrower ones (down to 64 bytes) only where a sample would not fit a workgroup otherwise, and down
  // to single groups where the chip would stand half empty.  A sample that does not fit even so is split into chunks of
  // the widest slabs.
  const long want = (long)256 * maxr, most = (long)maxt * maxr;
  int widest = 0, best = 0;
  for (int ns = 1; ns <= G; ++ns) {
    const int S = C / ns;
    if (G % ns || S % vec || S > (S == D ? MAX_GROUP : MAX_SLAB) || S / vec > maxt) continue;
    if (best == 0) { widest = best = ns; continue; }
    const long row = (long)S * esize, now = P * (C / best / vec);
    if ((now > want && row >= 128) || (now > most && row >= 64) || (now > 64 && now <= most && N * best < 512)) best = ns;
  }
  if (best == 0) return false;
  pl.split = P * (C / best / vec) > most;
  auto shape = [&](int ns, int t) {
    q.nslab = ns;
    q.S = C / ns;
    q.L = q.S / vec;
    t = (t + 63) / 64 * 64;
    if (t < q.L) t = (q.L + 63) / 64 * 64;
    if (t > maxt) t = maxt;
    pl.threads = t;
    q.rows = t / q.L;
  };
  if (!pl.split) {
    // as many vectors a thread as its registers hold (fewer threads share the set-up and the sums), unless that leaves
    // the chip's 256 x 16 waves idle
    int r = maxr;
    const long unit = P * (C / best / vec);
    while (r > 2 && N * best * ((unit + r - 1) / r) < 262144) r /= 2;
    shape(best, (int)((unit + r - 1) / r));
    q.chunk = (int)P; q.nchunk = 1;
    int R = (int)((P + q.rows - 1) / q.rows);
    if (R > maxr) {  // rows that do not divide the threads evenly
      shape(best, maxt);
      R = (int)((P + q.rows - 1) / q.rows);
    }
    if (R > maxr) pl.split = 1;
    pl.R = pow2_up(R);
  }
  if (pl.split) {
    // about 2048 workgroups that take at least 2 rounds of BLOCK vectors a thread
    shape(widest, 256);
    long chunks = (2048 + N * q.nslab - 1) / (N * q.nslab), least = (long)q.rows * BLOCK * 2;
    if (P / chunks < least) chunks = (P + least - 1) / least;
    q.chunk = (int)((P + chunks - 1) / chunks);
    q.nchunk = (int)((P + q.chunk - 1) / q.chunk);
    pl.R = BLOCK;
  }
  q.pre = q.L < 64 && 64 % q.L == 0;
  pl.one = D % vec == 0;
  const int Gs = q.S / D, nr = q.pre ? pl.threads / 64 : q.rows, nm = pl.one ? 1 : vec;
  const int gw = pl.one ? D / vec : D;
  auto team = [](long n) { return n >= 64 ? 64 : pow2_up((int)n); };
  q.tw = team((long)nr * gw);
  q.tw_ch = team(nr);
  q.tw_gr = team(D);
  pl.lds = hold == 1 ? (2 * (size_t)Gs + (size_t)nr * q.L * nm) * 4
                     : (3 * (size_t)q.S + 4 * (size_t)Gs + 2 * (size_t)nr * q.S) * 4;
  // a grid counts its threads in 32 bits: the sweeps', and the joins' workgroup of 256 per (sample, group)
  const long wgs = (long)q.nslab * q.nchunk, sweep = wgs * pl.threads, join = pl.split ? (long)G * 256 : 0;
  const long each = sweep > join ? sweep : join, fit = ((1L << 32) - 1) / each / 8 * 8;
  pl.piece = N < fit ? N : fit;
  return fit > 0;
}

inline bool valid(long N, long P, int C, int G, int vec, int dtype, int per_client) {
  if (N < 1 || P < 1 || C < 1 || G < 1 || C % G || per_client < 1 || N % per_client) return false;
  if (dtype < 0 || dtype > 2 || (vec != 1 && vec != 4) || C % vec) return false;
  // grids and in-kernel counters are 32 bits, offsets 64; gn_affine_kernel's grid has C / 8 workgroups of 1024 per client
  return C <= (1 << 24) && N < (1L << 24) && P < (1L << 30) && (double)N * P * C < 9e15;
}

}  // namespace groupnorm
