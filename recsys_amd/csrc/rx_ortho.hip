// Newton-Schulz orthogonalisation of weight updates (gfx950):  X = G / (|G|_F + eps), then `steps` times
//   A = X X^T,  B = b A + c A A,  X <- a X + B X          (m = min(rows, cols) rows after a transpose, n = max columns)
//
// The products take all the time: m^2 n + m^3 + 2 m^2 n operations per step, A and A A being symmetric (only tiles on and
// below the diagonal are computed, the others are their mirror images).  Small singular values grow by up to a^steps = 485,
// and so do rounding errors along them: 16-bit products would leave errors of the size of the result there, so the products
// keep fp32 accuracy.
// Operands are cut into two fp16 planes (11 + 11 significant bits: the value to 2^-22) and multiplied as high high + high low
// + low high.  What is left out is below 2^-22 of a term and differs in sign from term to term, so that the result is as near
// the exact one as fp32 products leave it, at a third of the 16-bit rate, where fp32 matrix instructions have a sixteenth.
// fp16 lacks range, but the iteration does not use it: |X|_2 <= 1 at the start and the coefficients bound it from there
// on, so each array has one power-of-two scale that takes its bound to 2^15, found on the host.
//   * Matrices that fit one workgroup's LDS take all steps in one launch (ns_split): such lists are bound by launches and latency.
//   * The others share three launches per step, whatever their number.  X, X^T, A and B live in the workspace as planes, cut
//     once in the epilogue that makes them; with X^T kept beside X all three products read both operands along the
//     contraction.
// Measured, where a large fp16 product reaches 1105 TFLOP/s: a step of 3344 x 3344, 1672 x 3344 and 836 x 1672 takes A 169, B 168
// and X 338 us (850, 762 and 850 TFLOP/s of plane products); one of 1024 x 1024 16 us a product, of 256 x 256 7 us (a launch
// is 4.5 of them); one workgroup's 64 x 128 33 us for all five steps.
#include "rx_common.h"

#include <math.h>

typedef _Float16 ns_h8 __attribute__((ext_vector_type(8)));
typedef _Float16 ns_h2 __attribute__((ext_vector_type(2)));
typedef float ns_f2 __attribute__((ext_vector_type(2)));
typedef float ns_f4 __attribute__((ext_vector_type(4)));
typedef float ns_acc __attribute__((ext_vector_type(16)));

#define NS_MAXDIM 16384
#define NS_SMALL_M 96
#define NS_SMALL_LDS (152 * 1024)
#define NS_SMALL_THREADS 512
#define NS_SMALL_JOBS 8          // tiles of A times shares of their contraction
#define NS_PARTS 256           // norm partials per matrix

// two values times a scale -> their words in the two planes
__device__ __forceinline__ void ns_cut2(float a, float b, uint32_t* w) {
  ns_f2 v = {a, b};
  const ns_h2 h = __builtin_convertvector(v, ns_h2);
  ns_f2 r = {a - (float)h.x, b - (float)h.y};
  w[0] = __builtin_bit_cast(uint32_t, h);
  w[1] = __builtin_bit_cast(uint32_t, __builtin_convertvector(r, ns_h2));
}
// Planes in memory: the 32 high halves of a group of 32 elements, then its 32 low ones: 128 bytes, one cache line.  `ld`:
// elements per row, a multiple of 32.
__device__ __forceinline__ int64_t ns_at(int64_t row, int k, int ld) { return (row * ld + (k & ~31)) * 2 + (k & 31); }
// four neighbouring values from their planes
__device__ __forceinline__ void ns_join4(const uint16_t* p, int64_t plane, float* v) {
  const uint2 hi = *reinterpret_cast<const uint2*>(p), lo = *reinterpret_cast<const uint2*>(p + plane);
  const uint32_t h[2] = {hi.x, hi.y}, l[2] = {lo.x, lo.y};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const ns_h2 a = __builtin_bit_cast(ns_h2, h[i]), b = __builtin_bit_cast(ns_h2, l[i]);
    v[2 * i] = (float)a.x + (float)b.x;
    v[2 * i + 1] = (float)a.y + (float)b.y;
  }
}

// ---------------------------------------------------------------- small matrices: one workgroup each
struct NsSmall {
  const float* g[RX_ORTHO_MAX];
  float* out[RX_ORTHO_MAX];
  float *mom[RX_ORTHO_MAX], *w[RX_ORTHO_MAX];
  float alpha[RX_ORTHO_MAX];
  int32_t rows[RX_ORTHO_MAX], cols[RX_ORTHO_MAX];
  int32_t steps, nesterov;
  float a, b, c, eps, mu;
  float sx, sa, sb;            // scales of X, A and B
  const float* scale;
};
// What is orthogonalised of a gradient value: the value itself, or with momentum (m: in the new, out the stored one)
// u = s g + mu m, m = mu m + s g.
__device__ __forceinline__ float ns_update(float g, float* m, float mu, int nesterov) {
  *m = fmaf(mu, *m, g);
  return nesterov ? fmaf(mu, *m, g) : *m;
}
// what a matrix is divided by; 1 for zeros without an eps
__device__ __forceinline__ float ns_divisor(double ss, float eps) {
  const float d = (float)(sqrt(ss) + (double)eps);
  return d == 0.f ? 1.f : d;
}
static inline int ns_up(int x, int a) { return (x + a - 1) / a * a; }
// LDS of one matrix: X as fp32 [mp][np + 4], A and B as planes [2][mp][mp + 8], and where fewer tiles of A than wavefronts
// exist, a 32 x 36 partial tile per wavefront.  (m <= 16: see ns_tiny_run.)
static size_t ns_small_lds(int rows, int cols) {
  const int m = rows < cols ? rows : cols, mp = ns_up(m, 32), np = ns_up(rows < cols ? cols : rows, 32);
  if (m <= 16) return ((size_t)m * (np + 4) + 320 * (2 + NS_SMALL_JOBS)) * 4;
  return (size_t)mp * (np + 4) * 4 + (size_t)8 * mp * (mp + 8) + (mp < 96 ? (size_t)NS_SMALL_JOBS * 32 * 36 * 4 : 0);
}
static bool ns_is_small(int rows, int cols) {
  return (rows < cols ? rows : cols) <= NS_SMALL_M && ns_small_lds(rows, cols) <= NS_SMALL_LDS;
}

// eight fp32 values -> fragments of the two planes
__device__ __forceinline__ void ns_cut8(const float* v, ns_h8* f) {
  union { uint32_t w[4]; ns_h8 h; } p[2];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t w[2];
    ns_cut2(v[2 * i], v[2 * i + 1], w);
    p[0].w[i] = w[0];
    p[1].w[i] = w[1];
  }
  f[0] = p[0].h;
  f[1] = p[1].h;
}
// one step of the contraction into three sums: a matrix instruction does not wait for the one before it
struct NsSum {
  ns_acc hh = {}, hl = {}, lh = {};
  __device__ __forceinline__ void add(const ns_h8* a, const ns_h8* b) {
    hh = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[0], b[0], hh, 0, 0, 0);
    hl = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[0], b[1], hl, 0, 0, 0);
    lh = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[1], b[0], lh, 0, 0, 0);
  }
  __device__ __forceinline__ ns_acc total() const { return hh + (hl + lh); }
};

// MB = m / 32, rounded up; rows past m hold zeros.  All arrays hold their values times their scale (X: sx, A: sa, B: sb).
// All MB^2 tiles of A and B are computed: the lower and the upper one of a pair come out the same, bit for bit, and each
// is written four rows at a time without a second, scattered image.
template <int MB>
__device__ __forceinline__ void ns_small_run(const NsSmall& a, float* X, int np) {
  constexpr int MP = MB * 32, LDP = MP + 8, PLANE = MP * LDP, TILES = MB * MB, W = NS_SMALL_THREADS / 64;
  constexpr int KS = NS_SMALL_JOBS / TILES < 1 ? 1 : NS_SMALL_JOBS / TILES;
  const int ldx = np + 4, lane = rx_lane(), wave = threadIdx.x >> 6, l31 = lane & 31, h = lane >> 5;
  uint16_t* A = reinterpret_cast<uint16_t*>(X + MP * ldx);
  uint16_t* B = A + 2 * PLANE;
  float* part = reinterpret_cast<float*>(B + 2 * PLANE);
  auto planes_row = [&](const uint16_t* p, int row, int k, ns_h8* f) {
#pragma unroll
    for (int q = 0; q < 2; ++q) f[q] = *reinterpret_cast<const ns_h8*>(p + q * PLANE + row * LDP + k);
  };
  auto x_row = [&](int row, int k, ns_h8* f) {
    const float4 lo = *reinterpret_cast<const float4*>(X + row * ldx + k), hi = *reinterpret_cast<const float4*>(X + row * ldx + k + 4);
    const float v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    ns_cut8(v, f);
  };
  auto put4 = [&](uint16_t* p, int r, int c, const float* v) {      // rows r .. r + 3 of column c
    uint32_t w0[2], w1[2];
    ns_cut2(v[0], v[1], w0);
    ns_cut2(v[2], v[3], w1);
#pragma unroll
    for (int q = 0; q < 2; ++q) *reinterpret_cast<uint2*>(p + q * PLANE + c * LDP + r) = make_uint2(w0[q], w1[q]);
  };
  const float ua = a.sa / (a.sx * a.sx), ub = a.b * a.sb / a.sa, uc = a.c * a.sb / (a.sa * a.sa), ux = 1.f / a.sb;
  const int shares = np >= 128 * KS ? KS : 1;          // a contraction of up to 8 steps is not worth the second pass
  for (int step = 0; step < a.steps; ++step) {
    // A = X X^T
    for (int job = wave; job < TILES * shares; job += W) {
      const int t = job / shares, s = job % shares, i = t / MB, j = t % MB;
      const int steps = np / 16, lo = steps * s / shares, hi = steps * (s + 1) / shares;
      NsSum sum;
      for (int k = lo; k < hi; ++k) {
        ns_h8 fi[2], fj[2];
        x_row(i * 32 + l31, k * 16 + h * 8, fi);
        if (i == j) sum.add(fi, fi);
        else {
          x_row(j * 32 + l31, k * 16 + h * 8, fj);
          sum.add(fi, fj);
        }
      }
      const ns_acc acc = sum.total();
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float v[4] = {acc[4 * q] * ua, acc[4 * q + 1] * ua, acc[4 * q + 2] * ua, acc[4 * q + 3] * ua};
        if (KS > 1 && shares > 1) *reinterpret_cast<float4*>(part + (job * 32 + l31) * 36 + 8 * q + 4 * h) = make_float4(v[0], v[1], v[2], v[3]);
        else put4(A, i * 32 + 8 * q + 4 * h, j * 32 + l31, v);
      }
    }
    __syncthreads();
    if (KS > 1 && shares > 1) {
      for (int x = threadIdx.x; x < TILES * 256; x += NS_SMALL_THREADS) {
        const int t = x >> 8, c = x & 31, r = (x >> 5 & 7) * 4;
        float v[4] = {};
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          const float4 f = *reinterpret_cast<const float4*>(part + ((t * KS + s) * 32 + c) * 36 + r);
          v[0] += f.x; v[1] += f.y; v[2] += f.z; v[3] += f.w;
        }
        put4(A, t / MB * 32 + r, t % MB * 32 + c, v);
      }
      __syncthreads();
    }
    // B = b A + c A A
    for (int t = wave; t < TILES; t += W) {
      const int i = t / MB, j = t % MB, c = j * 32 + l31;
      NsSum sum;
#pragma unroll
      for (int k = 0; k < MP / 16; ++k) {
        ns_h8 fi[2], fj[2];
        planes_row(A, i * 32 + l31, k * 16 + h * 8, fi);
        planes_row(A, c, k * 16 + h * 8, fj);
        sum.add(fi, fj);
      }
      const ns_acc acc = sum.total();
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int r = i * 32 + 8 * q + 4 * h;
        float v[4];
        ns_join4(A + c * LDP + r, PLANE, v);             // A is its own mirror image
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = fmaf(ub, v[e], uc * acc[4 * q + e]);
        put4(B, r, c, v);
      }
    }
    __syncthreads();
    // X = a X + B X: a wavefront owns 32 columns and has read all of them before it writes any
    for (int cb = wave; cb < np / 32; cb += W) {
      float* col = X + cb * 32 + l31;
      ns_h8 fx[MP / 16][2];
#pragma unroll
      for (int k = 0; k < MP / 16; ++k) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = col[(k * 16 + h * 8 + e) * ldx];
        ns_cut8(v, fx[k]);
      }
#pragma unroll 1
      for (int i = 0; i < MB; ++i) {
        NsSum sum;
#pragma unroll
        for (int k = 0; k < MP / 16; ++k) {
          ns_h8 fb[2];
          planes_row(B, i * 32 + l31, k * 16 + h * 8, fb);
          sum.add(fb, fx[k]);
        }
        const ns_acc acc = sum.total();
        float* p = col + (i * 32 + 4 * h) * ldx;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float* at = p + (8 * (e / 4) + e % 4) * ldx;
          *at = fmaf(a.a, *at, acc[e] * ux);
        }
      }
    }
    __syncthreads();
  }
}

// m <= 16: one tile on fp32 matrix instructions, whose rate does not matter here; the contraction of A is shared out
// among the wavefronts.  A [16][20] and B [16][20] behind X, the shares [waves][16][20] behind them.
__device__ __forceinline__ void ns_tiny_run(const NsSmall& a, float* X, int m, int np) {
  constexpr int W = NS_SMALL_JOBS;
  const int ldx = np + 4, lane = rx_lane(), wave = threadIdx.x >> 6, l15 = lane & 15, q = lane >> 4;
  float *A = X + m * ldx, *B = A + 320, *part = B + 320;
  const float one = 1.f / (a.sx * a.sx);
  for (int step = 0; step < a.steps; ++step) {
    if (wave < W) {
      ns_f4 acc[4] = {};
      const int quads = np / 4, lo = quads * wave / W, hi = quads * (wave + 1) / W;
      for (int k = lo; k < hi; k += 4)
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (k + u < hi) {
            const float v = l15 < m ? X[l15 * ldx + (k + u) * 4 + q] : 0.f;
            acc[u] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, v, acc[u], 0, 0, 0);
          }
#pragma unroll
      for (int e = 0; e < 4; ++e) part[wave * 320 + (q * 4 + e) * 20 + l15] = ((acc[0][e] + acc[1][e]) + (acc[2][e] + acc[3][e])) * one;
    }
    __syncthreads();
    if (threadIdx.x < 256) {
      const int at = (threadIdx.x >> 4) * 20 + (threadIdx.x & 15);
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) s += part[w * 320 + at];
      A[at] = s;
    }
    __syncthreads();
    if (wave == 0) {
      ns_f4 acc = {};
#pragma unroll
      for (int k = 0; k < 4; ++k) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(A[l15 * 20 + 4 * k + q], A[l15 * 20 + 4 * k + q], acc, 0, 0, 0);
#pragma unroll
      for (int e = 0; e < 4; ++e) B[(q * 4 + e) * 20 + l15] = fmaf(a.b, A[(q * 4 + e) * 20 + l15], a.c * acc[e]);
    }
    __syncthreads();
    for (int cb = wave; cb < np / 16; cb += NS_SMALL_THREADS / 64) {
      float* col = X + cb * 16 + l15;
      ns_f4 acc = {};
#pragma unroll
      for (int k = 0; k < 4; ++k)
        acc = __builtin_amdgcn_mfma_f32_16x16x4f32(B[l15 * 20 + 4 * k + q], 4 * k + q < m ? col[(4 * k + q) * ldx] : 0.f, acc, 0, 0, 0);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (q * 4 + e < m) col[(q * 4 + e) * ldx] = fmaf(a.a, col[(q * 4 + e) * ldx], acc[e]);
    }
    __syncthreads();
  }
}

__global__ void __launch_bounds__(NS_SMALL_THREADS) ns_small_kernel(NsSmall a) {
  extern __shared__ __align__(16) float ns_lds[];
  __shared__ double part[NS_SMALL_THREADS / 64];
  const float* g = a.g[blockIdx.x];
  float* out = a.out[blockIdx.x];
  float* mom = a.mom[blockIdx.x];
  const int rows = a.rows[blockIdx.x], cols = a.cols[blockIdx.x];
  const bool flip = rows > cols;
  const int m = flip ? cols : rows, n = flip ? rows : cols, np = (n + 31) & ~31, ldx = np + 4;
  float* X = ns_lds;
  const int lane = rx_lane(), wave = threadIdx.x >> 6;
  const float sc = a.scale ? *a.scale : 1.f;
  double ss = 0.0;
  // along G, four values of a thread on their way at once
  const int total = rows * cols, dr = NS_SMALL_THREADS / cols, dc = NS_SMALL_THREADS - dr * cols;
  {
    int r = threadIdx.x / cols, c = threadIdx.x - r * cols;
    for (int i0 = threadIdx.x; i0 < total; i0 += 4 * NS_SMALL_THREADS) {
      float v[4], mv[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = i0 + u * NS_SMALL_THREADS;
        v[u] = i < total ? g[i] : 0.f;
        mv[u] = mom && i < total ? mom[i] : 0.f;
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = i0 + u * NS_SMALL_THREADS;
        if (i < total) {
          if (mom) {
            v[u] = ns_update(v[u] * sc, &mv[u], a.mu, a.nesterov);
            mom[i] = mv[u];
          }
          ss = fma((double)v[u], (double)v[u], ss);
          X[flip ? c * ldx + r : r * ldx + c] = v[u];
        }
        r += dr;
        c += dc;
        if (c >= cols) { c -= cols; ++r; }
      }
    }
  }
  for (int i = threadIdx.x; i < m * (ldx - n); i += NS_SMALL_THREADS) X[i / (ldx - n) * ldx + n + i % (ldx - n)] = 0.f;
  if (m > 16)
    for (int i = m * ldx + threadIdx.x; i < ((m + 31) & ~31) * ldx; i += NS_SMALL_THREADS) X[i] = 0.f;
  ss = rx_wave_sum_f64(ss);
  if (lane == 0) part[wave] = ss;
  __syncthreads();
  ss = 0.0;
  for (int w = 0; w < NS_SMALL_THREADS / 64; ++w) ss += part[w];
  const float div = ns_divisor(ss, a.eps);
  for (int r = wave; r < m; r += NS_SMALL_THREADS / 64)
    for (int c = lane; c < n; c += 64) X[r * ldx + c] = X[r * ldx + c] / div * a.sx;
  __syncthreads();
  if (m <= 16) ns_tiny_run(a, X, m, np);
  else if (m <= 32) ns_small_run<1>(a, X, np);
  else if (m <= 64) ns_small_run<2>(a, X, np);
  else ns_small_run<3>(a, X, np);
  float* w = a.w[blockIdx.x];
  const float alpha = a.alpha[blockIdx.x], undo = 1.f / a.sx;
  int r = threadIdx.x / cols, c = threadIdx.x - r * cols;
  for (int i = threadIdx.x; i < total; i += NS_SMALL_THREADS) {
    const float v = X[flip ? c * ldx + r : r * ldx + c] * undo;
    if (w) w[i] = fmaf(-alpha, v, w[i]);
    else out[i] = v;
    r += dr;
    c += dc;
    if (c >= cols) { c -= cols; ++r; }
  }
}

// ---------------------------------------------------------------- large matrices: planes
struct NsMat {
  const float* g;
  float *out, *mom, *w;
  int32_t rows, cols;          // as given
  int32_t m, n, mp, np;        // working shape, and padded to the tile
  uint16_t *x[2], *xt[2];      // planes of [mp][np], [np][mp], alternating by step
  uint16_t *A, *B;             // planes of [mp][mp]
  int32_t tiles_sym, tiles_x;
  float alpha;
};
struct NsList {
  NsMat mat[RX_ORTHO_MAX];
  int32_t count, steps, tile, nesterov;
  float a, b, c, eps, mu;
  float sx, sa, sb;            // scales of the X, A and B planes
  const float* scale;
  double* parts;               // [count][NS_PARTS]
};

__global__ void __launch_bounds__(RX_BLOCK) ns_norm_kernel(NsList a) {
  const int mi = blockIdx.x / NS_PARTS, pt = blockIdx.x % NS_PARTS;
  const NsMat& t = a.mat[mi];
  const int64_t n = (int64_t)t.rows * t.cols;
  const float sc = a.scale ? *a.scale : 1.f;
  double s = 0.0;
  const int64_t stride = (int64_t)NS_PARTS * RX_BLOCK;
  for (int64_t i0 = (int64_t)pt * RX_BLOCK + threadIdx.x; i0 < n; i0 += 8 * stride) {
    float u[8], m[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {              // eight values of a thread on their way at once
      const int64_t i = i0 + k * stride;
      u[k] = i < n ? t.g[i] : 0.f;
      m[k] = t.mom && i < n ? t.mom[i] : 0.f;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int64_t i = i0 + k * stride;
      if (t.mom && i < n) {
        u[k] = ns_update(u[k] * sc, &m[k], a.mu, a.nesterov);
        t.mom[i] = m[k];
      }
      s = fma((double)u[k], (double)u[k], s);
    }
  }
  __shared__ double w[RX_BLOCK / 64];
  s = rx_wave_sum_f64(s);
  if (rx_lane() == 0) w[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) a.parts[blockIdx.x] = ((w[0] + w[1]) + w[2]) + w[3];
}

// planes of X and X^T from G, 64 x 64 at a time, padding included
__global__ void __launch_bounds__(RX_BLOCK) ns_init_kernel(NsList a) {
  __shared__ float tl[64][65];
  int mi = 0, b = blockIdx.x;
  for (; mi < a.count; ++mi) {
    const int k = (a.mat[mi].mp / 64) * (a.mat[mi].np / 64);
    if (b < k) break;
    b -= k;
  }
  if (mi == a.count) return;
  const NsMat& t = a.mat[mi];
  double ss = 0.0;
  __shared__ double wsum[RX_BLOCK / 64];
  ss = rx_wave_sum_f64(a.parts[mi * NS_PARTS + threadIdx.x]);
  if (rx_lane() == 0) wsum[threadIdx.x >> 6] = ss;
  __syncthreads();
  ss = ((wsum[0] + wsum[1]) + wsum[2]) + wsum[3];
  const float div = ns_divisor(ss, a.eps);
  const float sc = a.scale ? *a.scale : 1.f;
  const int r0 = b / (t.np / 64) * 64, c0 = b % (t.np / 64) * 64;      // of X
  const bool flip = t.rows > t.cols;
  float v[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const int i = k * RX_BLOCK + threadIdx.x, y = i / 64, x = i % 64;
    const int r = flip ? c0 + y : r0 + y, c = flip ? r0 + x : c0 + x;  // of G: rows of it are read along
    v[k] = 0.f;
    if (r < t.rows && c < t.cols) {
      const int64_t at = (int64_t)r * t.cols + c;
      v[k] = t.g[at];
      if (t.mom) v[k] = a.nesterov ? fmaf(a.mu, t.mom[at], v[k] * sc) : t.mom[at];     // the norm's pass stored the new momentum
    }
  }
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const int i = k * RX_BLOCK + threadIdx.x, y = i / 64, x = i % 64;
    if (flip) tl[x][y] = v[k] / div * a.sx;
    else tl[y][x] = v[k] / div * a.sx;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int i = k * RX_BLOCK + threadIdx.x, y = i / 16, x = i % 16 * 4;
    uint32_t w0[2], w1[2];
    ns_cut2(tl[y][x], tl[y][x + 1], w0);
    ns_cut2(tl[y][x + 2], tl[y][x + 3], w1);
#pragma unroll
    for (int p = 0; p < 2; ++p) *reinterpret_cast<uint2*>(t.x[0] + ns_at(r0 + y, c0 + x, t.np) + p * 32) = make_uint2(w0[p], w1[p]);
    ns_cut2(tl[x][y], tl[x + 1][y], w0);
    ns_cut2(tl[x + 2][y], tl[x + 3][y], w1);
#pragma unroll
    for (int p = 0; p < 2; ++p) *reinterpret_cast<uint2*>(t.xt[0] + ns_at(c0 + y, r0 + x, t.mp) + p * 32) = make_uint2(w0[p], w1[p]);
  }
}

// One T x T tile of P Q^T from the planes of P and Q: four wavefronts, (T / 2)^2 each, BK of the contraction per step.
// A step of an operand lies in LDS as SUB groups of T rows of 128 bytes, brought there from memory without passing through
// registers, 8 rows per instruction of a wavefront.  Such a load fills LDS in the order of the lanes, so rows cannot be padded
// apart; instead the 16-byte chunks of row r change places by (r / 2) % 8, which has 16 neighbouring rows meet every bank.
template <int T>
struct NsTile {
  static constexpr int NB = T / 64, SUMS = T == 64 ? 3 : 2;
  // Two steps of 32 KiB of both operands are in LDS, so that two workgroups share a CU.  Of a 3344 x 3344 product (T = 128)
  // one workgroup per CU with four such steps took 411 us where two with two took 325, steps of 16 elements 390; of lists
  // of 1024 x 1024 and less (T = 64) four steps were no faster.
  static constexpr int SUB = T == 128 ? 1 : 2, BK = 32 * SUB;
  static constexpr int OP = SUB * T * 64;                     // 16-bit elements of one operand's step
};

enum { NS_MODE_A, NS_MODE_B, NS_MODE_X };

typedef __attribute__((address_space(3))) void* ns_shared;

struct NsFeed {                // what a wavefront loads: its half of one operand's rows
  const uint16_t* src;
  int bytes;                   // of the half's rows: nothing behind them is read
  int off[2];                  // of a lane, for even and odd groups of 8 rows
  int rows8;                   // bytes from one group of 8 rows to the next
};
// 16 bytes per lane from src + lane_at + at (bytes) to 1 KiB of LDS, in the order of the lanes
__device__ __forceinline__ void ns_load_lds(const uint16_t* src, int bytes, uint16_t* to, int lane_at, int at) {
#ifdef __HIP_DEVICE_COMPILE__                                 // the host's pass does not know the type of a buffer descriptor
  const auto d = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(src), 0, bytes, 0x27000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(d, (ns_shared)to, 16, lane_at, at, 0, 0);
#endif
}
// step i -> one LDS buffer
template <int T>
__device__ __forceinline__ void ns_feed(const NsFeed& f, uint16_t* buf, int i) {
  typedef NsTile<T> Tile;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint16_t* to = buf + (wave >> 1) * Tile::OP + (wave & 1) * (T / 2) * 64;
#pragma unroll
  for (int s = 0; s < Tile::SUB; ++s)
#pragma unroll
    for (int j = 0; j < T / 16; ++j)
      ns_load_lds(f.src, f.bytes, to + s * T * 64 + j * 512, f.off[j & 1], j * f.rows8 + (i * Tile::SUB + s) * 128);
}
// acc: high high products, and the two others; of T = 64 the first in two sums.  Each addition into a sum rounds at its size:
// with all in one, matrices of 33 x 1400 came out with 2.2 times the error of fp32 products.
template <int T>
__device__ __forceinline__ void ns_step(const uint16_t* buf, const int (&at)[2][2], int wi, int wj, ns_acc (&acc)[NsTile<T>::SUMS][NsTile<T>::NB][NsTile<T>::NB]) {
  typedef NsTile<T> Tile;
  constexpr int NB = Tile::NB;
#pragma unroll
  for (int s = 0; s < Tile::SUB; ++s)
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      ns_h8 fa[NB][2], fb[NB][2];
#pragma unroll
      for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          fa[i][p] = *reinterpret_cast<const ns_h8*>(buf + (s * T + (wi * NB + i) * 32) * 64 + at[p][ks]);
          fb[i][p] = *reinterpret_cast<const ns_h8*>(buf + Tile::OP + (s * T + (wj * NB + i) * 32) * 64 + at[p][ks]);
        }
      constexpr int PA[3] = {1, 0, 0}, PB[3] = {0, 0, 1};
#pragma unroll
      for (int u = 0; u < 3; ++u)
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
          for (int j = 0; j < NB; ++j) {
            ns_acc& c = acc[u != 1 ? 0 : T == 64 ? 1 + ks : 1][i][j];
            c = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[i][PA[u]], fb[j][PB[u]], c, 0, 0, 0);
          }
    }
}

// Tile b of a product: bands of 8 tile rows, each band column by column, so that the 64 tiles an XCD works on at a time
// are about 8 x 8 and share operand rows.  FULL: all of tm x tn; otherwise the lower triangle of tm x tm.
template <bool FULL>
__device__ __forceinline__ void ns_tile(int b, int tm, int tn, int* ti, int* tj) {
  for (int r0 = 0;; r0 += 8) {
    const int rows = tm - r0 < 8 ? tm - r0 : 8;
    const int square = rows * (FULL ? tn : r0), all = square + (FULL ? 0 : rows * (rows + 1) / 2);
    if (b >= all && r0 + 8 < tm) { b -= all; continue; }
    if (b < square) {
      *ti = r0 + b % rows;
      *tj = b / rows;
      return;
    }
    b -= square;
    int i = 0;
    while (b > i) b -= ++i;
    *ti = r0 + i;
    *tj = r0 + b;
    return;
  }
}

// Workgroups are dealt to the 8 XCDs in turn.  Of a matrix's k tiles each XCD takes a run of neighbours, which share operand
// rows in its L2; the runs one longer than the others go on where those of the matrix before ended (`off`: tiles so
// far), so that every XCD has the same number of tiles, and as many of each length, to one.
__host__ __device__ __forceinline__ int ns_run_of(int k, int xcd, int off, int* first) {
  const int x = (xcd - off) & 7, rest = k & 7;
  *first = x * (k >> 3) + (x < rest ? x : rest);
  return (k >> 3) + (x < rest ? 1 : 0);
}

template <int T, int MODE>
__global__ void __launch_bounds__(RX_BLOCK, 2) ns_gemm_kernel(NsList a, int step) {
  typedef NsTile<T> Tile;
  constexpr int NB = Tile::NB;
  // two arrays: the compiler sees that loads into one and reads of the other do not meet
  __shared__ __align__(128) uint16_t b0[2 * Tile::OP], b1[2 * Tile::OP];
  int mi = 0, b = blockIdx.x / 8, off = 0;
  for (; mi < a.count; ++mi) {
    const int k = MODE == NS_MODE_X ? a.mat[mi].tiles_x : a.mat[mi].tiles_sym;
    int first;
    const int run = ns_run_of(k, blockIdx.x % 8, off, &first);
    if (b < run) { b += first; break; }
    b -= run;
    off += k;
  }
  if (mi == a.count) return;
  const NsMat& t = a.mat[mi];
  const int cur = step & 1;
  int ti, tj;
  ns_tile<MODE == NS_MODE_X>(b, t.mp / T, t.np / T, &ti, &tj);
  const uint16_t *P, *Q;
  int K, ld;
  if (MODE == NS_MODE_A) { P = Q = t.x[cur]; K = t.np; ld = t.np; }
  else if (MODE == NS_MODE_B) { P = Q = t.A; K = t.mp; ld = t.mp; }
  else { P = t.B; Q = t.xt[cur]; K = t.mp; ld = t.mp; }
  const int lane = rx_lane(), l31 = lane & 31, h = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wi = wave >> 1, wj = wave & 1;
  NsFeed feed;
  const uint16_t* mine = (wave >> 1 ? Q + (int64_t)tj * T * ld * 2 : P + (int64_t)ti * T * ld * 2) + (int64_t)(wave & 1) * (T / 2) * ld * 2;
  feed.src = mine;
  feed.bytes = (T / 2) * ld * 4;
  feed.rows8 = 32 * ld;
#pragma unroll
  for (int o = 0; o < 2; ++o) feed.off[o] = (lane >> 3) * ld * 4 + ((lane & 7) ^ (o * 4 + (lane >> 4))) * 16;
  int at[2][2];                // of a lane's fragment in a group of 32 rows, by plane and half of the 32
#pragma unroll
  for (int p = 0; p < 2; ++p)
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) at[p][ks] = l31 * 64 + (((p * 4 + ks * 2 + h) ^ (l31 >> 1 & 7)) * 8);
  ns_acc sums[Tile::SUMS][NB][NB] = {};
  const int steps = K / Tile::BK;
  ns_feed<T>(feed, b0, 0);
  // One barrier per step: behind it step i is there for everybody (each wavefront has waited for its own loads) and everybody
  // has done with step i - 1, whose buffer step i + 1 goes into.
  auto stage = [&](int i, const uint16_t* now, uint16_t* next) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (i + 1 < steps) ns_feed<T>(feed, next, i + 1);
    ns_step<T>(now, at, wi, wj, sums);
  };
  for (int i = 0; i < steps; i += 2) {
    stage(i, b0, b1);
    if (i + 1 < steps) stage(i + 1, b1, b0);
  }
  __syncthreads();
  // lane: column tj * T + .. + l31, rows 8 q + 4 h + k.  The transposed image is written from the registers, four rows
  // (8 bytes) at a time; the row-major one goes through LDS to be written 16 bytes at a time.
  const bool last = MODE == NS_MODE_X && step + 1 == a.steps;
  const bool flip = t.rows > t.cols;
  const float undo = MODE == NS_MODE_A ? 1.f / (a.sx * a.sx) : MODE == NS_MODE_B ? 1.f / (a.sa * a.sa) : 1.f / (a.sb * a.sx);
  const float scale = MODE == NS_MODE_A ? a.sa : MODE == NS_MODE_B ? a.sb : a.sx;
  uint16_t* row_major = MODE == NS_MODE_A ? t.A : MODE == NS_MODE_B ? t.B : t.x[cur ^ 1];
  uint16_t* mirror = MODE == NS_MODE_A ? t.A : MODE == NS_MODE_B ? t.B : t.xt[cur ^ 1];
  const int ldr = MODE == NS_MODE_X ? t.np : t.mp;
  uint32_t (*turn)[36] = reinterpret_cast<uint32_t (*)[36]>(b0) + wave * 32;    // 32 x 32 words per wavefront
#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const int r0 = ti * T + (wi * NB + i) * 32, c = tj * T + (wj * NB + j) * 32 + l31;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int r = r0 + 8 * q + 4 * h;
        float v[4], e[4];
        if (MODE == NS_MODE_B) ns_join4(t.A + ns_at(c, r, t.mp), 32, e);         // A is its own mirror image
        if (MODE == NS_MODE_X) ns_join4(t.xt[cur] + ns_at(c, r, t.mp), 32, e);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          v[k] = (sums[0][i][j][4 * q + k] + (T == 64 ? sums[1][i][j][4 * q + k] + sums[Tile::SUMS - 1][i][j][4 * q + k] : sums[1][i][j][4 * q + k])) * undo;
          if (MODE == NS_MODE_B) v[k] = fmaf(a.b / a.sa, e[k], a.c * v[k]);
          if (MODE == NS_MODE_X) v[k] = fmaf(a.a / a.sx, e[k], v[k]);
        }
        if (last) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (r + k < t.m && c < t.n) {
              const int64_t at = flip ? (int64_t)c * t.cols + r + k : (int64_t)(r + k) * t.cols + c;
              if (t.w) t.w[at] = fmaf(-t.alpha, v[k], t.w[at]);
              else t.out[at] = v[k];
            }
          continue;
        }
        uint32_t w0[2], w1[2];
        ns_cut2(v[0] * scale, v[1] * scale, w0);
        ns_cut2(v[2] * scale, v[3] * scale, w1);
#pragma unroll
        for (int p = 0; p < 2; ++p) *reinterpret_cast<uint2*>(mirror + ns_at(c, r, t.mp) + p * 32) = make_uint2(w0[p], w1[p]);
        if (MODE == NS_MODE_X || ti != tj) {             // a diagonal tile is its own mirror image
          const int y = 8 * q + 4 * h;
          turn[y][l31] = (w0[0] & 0xffffu) | (w0[1] << 16);
          turn[y + 1][l31] = (w0[0] >> 16) | (w0[1] & 0xffff0000u);
          turn[y + 2][l31] = (w1[0] & 0xffffu) | (w1[1] << 16);
          turn[y + 3][l31] = (w1[0] >> 16) | (w1[1] & 0xffff0000u);
        }
      }
      if (last || !(MODE == NS_MODE_X || ti != tj)) continue;
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      const int y = lane >> 1, x = (lane & 1) * 16;      // half a row per lane
      uint32_t u[16];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint4 f = *reinterpret_cast<const uint4*>(&turn[y][x + 4 * k]);
        u[4 * k] = f.x; u[4 * k + 1] = f.y; u[4 * k + 2] = f.z; u[4 * k + 3] = f.w;
      }
      uint16_t* d = row_major + ns_at(r0 + y, tj * T + (wj * NB + j) * 32 + x, ldr);
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          uint32_t o[4];
#pragma unroll
          for (int z = 0; z < 4; ++z) o[z] = __builtin_amdgcn_perm(u[8 * k + 2 * z + 1], u[8 * k + 2 * z], p ? 0x07060302u : 0x05040100u);
          *reinterpret_cast<uint4*>(d + p * 32 + 8 * k) = make_uint4(o[0], o[1], o[2], o[3]);
        }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}

// ---------------------------------------------------------------- host
struct NsArgs {                // rx_ortho_args and rx_muon_args in one form
  const float* g[RX_ORTHO_MAX];
  float *out[RX_ORTHO_MAX], *mom[RX_ORTHO_MAX], *w[RX_ORTHO_MAX];
  float alpha[RX_ORTHO_MAX];
  int32_t rows[RX_ORTHO_MAX], cols[RX_ORTHO_MAX];
  int32_t count, steps, nesterov;
  float a, b, c, eps, mu;
  float sx, sa, sb;
  const float* scale;
};

static int ns_check_eps(const char* who, float eps) {
  RX_REQUIRE(eps >= 0.f, "%s: eps=%g is negative", who, (double)eps);      // the scales count on |G|_F / (|G|_F + eps) <= 1
  return 0;
}

static int ns_check(const char* who, const int32_t* rows, const int32_t* cols, int count, int steps) {
  RX_REQUIRE(count >= 0 && count <= RX_ORTHO_MAX, "%s: %d matrices (at most %d)", who, count, RX_ORTHO_MAX);
  RX_REQUIRE(steps >= 1 && steps <= 32, "%s: steps=%d (1..32)", who, steps);
  for (int i = 0; i < count; ++i)
    RX_REQUIRE(rows[i] >= 1 && cols[i] >= 1 && rows[i] <= NS_MAXDIM && cols[i] <= NS_MAXDIM, "%s: matrix %d is %d x %d (1..%d)", who, i,
               rows[i], cols[i], NS_MAXDIM);
  return 0;
}

// Bounds of |X|_2, |A|_2 and |B|_2 over the steps, for singular values that start in [0, 1] (what the division by the norm
// guarantees): the largest |a s + b s^3 + c s^5| over [0, bound so far], from its extrema; refuses coefficients that let
// the bound grow past 16.
static int ns_bounds(const char* who, double ca, double cb, double cc, int steps, float* x, float* a, float* b) {
  double m = 1.0;
  for (int k = 0; k < steps; ++k) {
    double u[3] = {m * m, -1.0, -1.0};                   // s^2 of the candidates
    if (cc != 0.0) {
      const double d = 9.0 * cb * cb - 20.0 * ca * cc;
      if (d >= 0.0) {
        u[1] = (-3.0 * cb + sqrt(d)) / (10.0 * cc);
        u[2] = (-3.0 * cb - sqrt(d)) / (10.0 * cc);
      }
    } else if (cb != 0.0) {
      u[1] = -ca / (3.0 * cb);
    }
    double top = m;
    for (int i = 0; i < 3; ++i)
      if (u[i] > 0.0 && u[i] <= m * m) top = fmax(top, fabs(sqrt(u[i]) * (ca + u[i] * (cb + u[i] * cc))));
    RX_REQUIRE(top <= 16.0 && isfinite(ca + cb + cc), "%s: coefficients (%g, %g, %g) let singular values in [0, 1] grow past 16 in %d steps",
               who, ca, cb, cc, steps);
    if (top == m) break;
    m = top;
  }
  const double l = m * m, e = cc != 0.0 ? -cb / (2.0 * cc) : -1.0;
  double q = fabs(l * (cb + l * cc));
  if (e > 0.0 && e < l) q = fmax(q, fabs(e * (cb + e * cc)));
  *x = (float)m; *a = (float)l; *b = (float)q;
  return 0;
}
// power of two that takes a bound, with a margin for rounding, to at most 2^15
static float ns_scale_of(float bound) { return bound > 0.f ? ldexpf(1.f, 14 - ilogbf(bound * 1.1f)) : 1.f; }

// Time of a step's three products in tiles of t, in microseconds without the launches: each takes as long as its longest
// contraction on a CU of its own, and as all its tiles' contractions shared out over 256 CUs (measured per 32 elements and tile:
// with 128 0.8, and 0.8 to 1.09 where CUs have several; with 64 0.31).  Against the times of single matrices with both tiles: 2048 x 2048 841 us with 128
// and 880 with 64, 1900 x 1900 792 and 643, 1500 x 3000 959 and 678, 1024 x 1024 483 and 238.
static float ns_cost(const NsArgs& a, const bool* small, int t) {
  float longest[3] = {}, shared[3] = {};
  for (int i = 0; i < a.count; ++i) {
    if (small[i]) continue;
    const int lo = a.rows[i] < a.cols[i] ? a.rows[i] : a.cols[i], hi = a.rows[i] < a.cols[i] ? a.cols[i] : a.rows[i];
    const int tm = (lo + t - 1) / t, tn = (hi + t - 1) / t;
    const float sym = 0.5f * tm * (tm + 1), steps_m = tm * t / 32.f, steps_n = tn * t / 32.f;
    const float tiles[3] = {sym, sym, (float)tm * tn}, steps[3] = {steps_n, steps_m, steps_m};
    for (int p = 0; p < 3; ++p) {
      if (steps[p] > longest[p]) longest[p] = steps[p];
      shared[p] += tiles[p] * steps[p] / 256.f;
    }
  }
  float sum = 0.f;
  for (int p = 0; p < 3; ++p) {
    const float one = longest[p] * (t == 128 ? 0.8f : 0.31f), all = shared[p] * (t == 128 ? 0.9f : 0.31f);
    sum += one > all ? one : all;
  }
  return sum;
}

// Which matrices take a workgroup of their own; returns the tile of the others.  All that fit one do, but in a list that needs
// the large path anyway they join it while all its 64 x 64 tiles are on the chip at once: its launches take little longer for
// them (845 x 13, 63 x 257, 300 x 7, 1 x 1 and 129 x 130: 148 us with 63 x 257 there, 162 without).  Up to 16 rows stay apart
// where they fit: with so few terms fp32 products leave an error that 22-bit planes would treble.
static int ns_split(const NsArgs& a, bool* small) {
  int64_t all = 0;
  bool large = false;
  for (int i = 0; i < a.count; ++i) {
    small[i] = ns_is_small(a.rows[i], a.cols[i]);
    all += rx_cdiv(a.rows[i], 64) * rx_cdiv(a.cols[i], 64);
    large = large || !small[i];
  }
  const int tile = ns_cost(a, small, 128) < ns_cost(a, small, 64) ? 128 : 64;
  if (large && tile == 64 && all <= 512)
    for (int i = 0; i < a.count; ++i) small[i] = small[i] && (a.rows[i] < a.cols[i] ? a.rows[i] : a.cols[i]) <= 16;
  return tile;
}

static void ns_plan(const NsArgs& a, NsList* l, size_t* bytes, uint8_t* ws) {
  memset(l, 0, sizeof(*l));
  bool small[RX_ORTHO_MAX];
  l->tile = ns_split(a, small);
  int order[RX_ORTHO_MAX], k = 0;
  for (int i = 0; i < a.count; ++i)
    if (!small[i]) {
      int at = k++;
      auto cost = [&](int x) { return a.rows[x] < a.cols[x] ? a.rows[x] : a.cols[x]; };
      while (at > 0 && cost(order[at - 1]) < cost(i)) { order[at] = order[at - 1]; --at; }   // longest contractions first
      order[at] = i;
    }
  l->count = k;
  l->steps = a.steps;
  l->nesterov = a.nesterov;
  l->mu = a.mu;
  l->scale = a.scale;
  l->a = a.a; l->b = a.b; l->c = a.c; l->eps = a.eps;
  l->sx = a.sx; l->sa = a.sa; l->sb = a.sb;
  size_t at = 0;
  auto take = [&](size_t n) { uint8_t* p = ws ? ws + at : nullptr; at += rx_align_up(n, 256); return p; };
  l->parts = (double*)take(sizeof(double) * NS_PARTS * (size_t)k);
  for (int i = 0; i < k; ++i) {
    NsMat& t = l->mat[i];
    const int o = order[i];
    t.g = a.g[o]; t.out = a.out[o]; t.mom = a.mom[o]; t.w = a.w[o]; t.alpha = a.alpha[o];
    t.rows = a.rows[o]; t.cols = a.cols[o];
    t.m = t.rows < t.cols ? t.rows : t.cols;
    t.n = t.rows < t.cols ? t.cols : t.rows;
    t.mp = ns_up(t.m, l->tile); t.np = ns_up(t.n, l->tile);
    const int tm = t.mp / l->tile;
    t.tiles_sym = tm * (tm + 1) / 2;
    t.tiles_x = tm * (t.np / l->tile);
    const size_t mn = (size_t)t.mp * t.np * 4, mm = (size_t)t.mp * t.mp * 4;
    for (int q = 0; q < 2; ++q) { t.x[q] = (uint16_t*)take(mn); t.xt[q] = (uint16_t*)take(mn); }
    t.A = (uint16_t*)take(mm);
    t.B = (uint16_t*)take(mm);
  }
  *bytes = k ? at : 0;
}

template <int T>
static void ns_run(const NsList& l, hipStream_t st) {
  unsigned sym = 0, full = 0;
  for (int xcd = 0; xcd < 8; ++xcd) {
    unsigned ns = 0, nf = 0;
    int os = 0, of = 0, first;
    for (int i = 0; i < l.count; ++i) {
      ns += ns_run_of(l.mat[i].tiles_sym, xcd, os, &first);
      nf += ns_run_of(l.mat[i].tiles_x, xcd, of, &first);
      os += l.mat[i].tiles_sym;
      of += l.mat[i].tiles_x;
    }
    if (ns > sym) sym = ns;
    if (nf > full) full = nf;
  }
  sym *= 8;
  full *= 8;
  for (int s = 0; s < l.steps; ++s) {
    hipLaunchKernelGGL((ns_gemm_kernel<T, NS_MODE_A>), dim3(sym), dim3(RX_BLOCK), 0, st, l, s);
    hipLaunchKernelGGL((ns_gemm_kernel<T, NS_MODE_B>), dim3(sym), dim3(RX_BLOCK), 0, st, l, s);
    hipLaunchKernelGGL((ns_gemm_kernel<T, NS_MODE_X>), dim3(full), dim3(RX_BLOCK), 0, st, l, s);
  }
}

static int ns_go(const char* who, NsArgs& a, void* ws, size_t ws_bytes, int device, void* stream) {
  float bx, ba, bb;
  if (ns_bounds(who, a.a, a.b, a.c, a.steps, &bx, &ba, &bb)) return 1;
  a.sx = ns_scale_of(bx); a.sa = ns_scale_of(ba); a.sb = ns_scale_of(bb);
  NsList l;
  size_t need;
  ns_plan(a, &l, &need, (uint8_t*)ws);
  RX_REQUIRE(need == 0 || (ws && ws_bytes >= need && ((uintptr_t)ws & 255) == 0), "%s: workspace of %zu bytes, %zu needed", who, ws_bytes, need);
  RX_GUARD_DEVICE(device);
  hipStream_t st = (hipStream_t)stream;
  NsSmall s;
  memset(&s, 0, sizeof(s));
  s.steps = a.steps; s.nesterov = a.nesterov; s.mu = a.mu; s.scale = a.scale;
  s.a = a.a; s.b = a.b; s.c = a.c; s.eps = a.eps;
  s.sx = a.sx; s.sa = a.sa; s.sb = a.sb;
  bool small[RX_ORTHO_MAX];
  ns_split(a, small);
  int k = 0;
  size_t lds = 0;
  for (int i = 0; i < a.count; ++i)
    if (small[i]) {
      s.g[k] = a.g[i]; s.out[k] = a.out[i]; s.mom[k] = a.mom[i]; s.w[k] = a.w[i]; s.alpha[k] = a.alpha[i];
      s.rows[k] = a.rows[i]; s.cols[k] = a.cols[i];
      const size_t b = ns_small_lds(a.rows[i], a.cols[i]);
      if (b > lds) lds = b;
      ++k;
    }
  if (k) {
    if (lds > 64 * 1024) RX_HIP(hipFuncSetAttribute((const void*)ns_small_kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    hipLaunchKernelGGL(ns_small_kernel, dim3(k), dim3(NS_SMALL_THREADS), lds, st, s);
    RX_LAUNCH_CHECK();
  }
  if (l.count == 0) return 0;
  unsigned blocks = 0;
  for (int i = 0; i < l.count; ++i) blocks += (l.mat[i].mp / 64) * (l.mat[i].np / 64);
  hipLaunchKernelGGL(ns_norm_kernel, dim3(l.count * NS_PARTS), dim3(RX_BLOCK), 0, st, l);
  hipLaunchKernelGGL(ns_init_kernel, dim3(blocks), dim3(RX_BLOCK), 0, st, l);
  if (l.tile == 128) ns_run<128>(l, st);
  else ns_run<64>(l, st);
  RX_LAUNCH_CHECK();
  return 0;
}

static size_t ns_bytes(const int32_t* rows, const int32_t* cols, int count, int steps) {
  NsArgs a;
  memset(&a, 0, sizeof(a));
  a.count = count; a.steps = steps;
  memcpy(a.rows, rows, sizeof(a.rows));
  memcpy(a.cols, cols, sizeof(a.cols));
  NsList l;
  size_t bytes;
  ns_plan(a, &l, &bytes, nullptr);
  return bytes;
}

// two ranges of n and m floats share memory
static bool ns_overlap(const float* p, size_t n, const float* q, size_t m) {
  return (uintptr_t)p < (uintptr_t)(q + m) && (uintptr_t)q < (uintptr_t)(p + n);
}

extern "C" size_t rx_orthogonalize_workspace_bytes(const rx_ortho_args* a) {
  if (!a || ns_check("rx_orthogonalize", a->rows, a->cols, a->count, a->steps)) return 0;
  return ns_bytes(a->rows, a->cols, a->count, a->steps);
}

extern "C" int rx_orthogonalize(const rx_ortho_args* args, void* ws, size_t ws_bytes, int device, void* stream) {
  RX_REQUIRE(args, "rx_orthogonalize: null argument");
  if (ns_check("rx_orthogonalize", args->rows, args->cols, args->count, args->steps) || ns_check_eps("rx_orthogonalize", args->eps)) return 1;
  NsArgs a;
  memset(&a, 0, sizeof(a));
  for (int i = 0; i < args->count; ++i) {
    const size_t n = (size_t)args->rows[i] * args->cols[i];
    RX_REQUIRE(args->g[i] && args->out[i] && (((uintptr_t)args->g[i] | (uintptr_t)args->out[i]) & 3) == 0,
               "rx_orthogonalize: matrix %d: null or unaligned pointer", i);
    for (int j = 0; j < args->count; ++j) {
      const size_t m = (size_t)args->rows[j] * args->cols[j];
      RX_REQUIRE(args->g[j] && !ns_overlap(args->out[i], n, args->g[j], m), "rx_orthogonalize: output %d overlaps input %d", i, j);
      RX_REQUIRE(i == j || !ns_overlap(args->out[i], n, args->out[j], m), "rx_orthogonalize: outputs %d and %d overlap", i, j);
    }
    a.g[i] = args->g[i]; a.out[i] = args->out[i]; a.rows[i] = args->rows[i]; a.cols[i] = args->cols[i];
  }
  a.count = args->count; a.steps = args->steps;
  a.a = args->a; a.b = args->b; a.c = args->c; a.eps = args->eps;
  if (a.count == 0) return 0;
  return ns_go("rx_orthogonalize", a, ws, ws_bytes, device, stream);
}

extern "C" size_t rx_muon_step_workspace_bytes(const rx_muon_args* a) {
  if (!a || ns_check("rx_muon_step", a->rows, a->cols, a->count, a->steps)) return 0;
  return ns_bytes(a->rows, a->cols, a->count, a->steps);
}

extern "C" int rx_muon_step(const rx_muon_args* args, void* ws, size_t ws_bytes, int device, void* stream) {
  RX_REQUIRE(args, "rx_muon_step: null argument");
  if (ns_check("rx_muon_step", args->rows, args->cols, args->count, args->steps) || ns_check_eps("rx_muon_step", args->eps)) return 1;
  RX_REQUIRE(((uintptr_t)args->scale & 3) == 0, "rx_muon_step: unaligned scale");
  NsArgs a;
  memset(&a, 0, sizeof(a));
  for (int i = 0; i < args->count; ++i) {
    const size_t n = (size_t)args->rows[i] * args->cols[i];
    RX_REQUIRE(args->g[i] && args->w[i] && args->mom[i] && (((uintptr_t)args->g[i] | (uintptr_t)args->w[i] | (uintptr_t)args->mom[i]) & 3) == 0,
               "rx_muon_step: matrix %d: null or unaligned pointer", i);
    for (int j = 0; j < args->count; ++j) {
      const size_t m = (size_t)args->rows[j] * args->cols[j];
      RX_REQUIRE(args->g[j] && args->mom[j] && !ns_overlap(args->w[i], n, args->g[j], m) && !ns_overlap(args->mom[i], n, args->g[j], m) &&
                     !ns_overlap(args->w[i], n, args->mom[j], m) &&
                     (i == j || (!ns_overlap(args->w[i], n, args->w[j], m) && !ns_overlap(args->mom[i], n, args->mom[j], m))),
                 "rx_muon_step: buffers of matrices %d and %d overlap", i, j);
    }
    a.g[i] = args->g[i]; a.w[i] = args->w[i]; a.mom[i] = args->mom[i]; a.alpha[i] = args->lr[i];
    a.rows[i] = args->rows[i]; a.cols[i] = args->cols[i];
  }
  a.count = args->count; a.steps = args->steps; a.nesterov = args->nesterov != 0;
  a.a = args->a; a.b = args->b; a.c = args->c; a.eps = args->eps; a.mu = args->momentum;
  a.scale = args->scale;
  if (a.count == 0) return 0;
  return ns_go("rx_muon_step", a, ws, ws_bytes, device, stream);
}
