// Softmax over a whole item catalogue (gfx950): scores s_rv = x_r . t_v + b_v of rows x [R, D] against a table
// t [V, D], never stored.
//   forward   lse_r = log sum_v exp s_rv,  logprob_r = s_{r,y_r} - lse_r,  mean_r = sum_{v != y_r} p_rv t_v,  rest_r = sum_{v != y_r} p_rv
//   backward  dx_r = q_r t_{y_r} + c_r mean_r,   dt_v = sum_{r: y_r != v} c_r p_rv x_r + sum_{r: y_r = v} q_r x_r,
//             c_r = g_lse_r - g_r,   q_r = g_r + c_r p_{r,y_r} = g_r rest_r + g_lse_r p_{r,y_r}
// The rows' expectation does not depend on the gradient, so the forward pass takes it along (online softmax with
// the table as keys and values) and a train step costs four products of 2 R V D operations: scores and mean forward,
// scores and dt backward.  A row's target stays out of its sums and joins them at their end: on a row that is nearly sure of it the
// gradients are of the size of 1 - p_y, and so are all their errors then; g + c p_y would keep those of g.
//
// Both passes are one loop.  One side is stationary (forward: rows, backward: items): its vectors sit in registers as
// matrix operands, 32 per wavefront and block, one per lane column.  The other side streams through LDS in tiles, kept
// twice: row-major for the scores, transposed for the second product.  Scores come out of the matrix unit with the
// streaming index along a lane's registers and the stationary index across the lanes, so the softmax reference and sum
// are one number per lane, and the weights go straight back in as the other operand of the second product: its
// contraction index may run in any order, and the transposed tile is laid out in the order the registers have.
//
// fp32 operands are cut into two fp16 planes (11 + 11 significant bits: the value to 2^-22) and multiplied as high high +
// high low + low high in fp32.  What is left out is below 2^-22 of a term, and such errors differ in sign from term to
// term: sums of tens of terms come out as near the exact ones as fp32's own, whose additions round as often.  That takes
// three products at the 16-bit matrix rate, where fp32 matrix instructions run at 1/16 of it and three bf16 planes would
// take six products.  fp16 has no
// range to spare, so everything is scaled by powers of two first, which costs no accuracy: a stationary vector by its
// own largest element, a streaming tile by the tile's (both to 2^14 .. 2^15: elements down to 2^-15 of the largest keep
// all their bits, smaller ones an absolute error of 2^-39 of it), and the weights by a running reference per stationary
// vector (the softmax's own in the forward pass).  The factors fold into numbers the loop has anyway.
// bf16 operands take one plane, exactly; there the weights of the second product are rounded to bf16 as well, by up to 2^-8 of
// each and independently from term to term.  Where they meet a large term of the other sign, the rounding is made good: dx takes the sum
// of the rounded weights for rest, so that it is a sum of (t_y - t_v) under them, and the targets' shares q of the table's gradient come
// with their low part.
// Scores, references, sums, means and gradients accumulate in fp32.
// Measured under a kernel trace (the calls run about a tenth faster), where a large bf16 product reaches 1151 TFLOP/s and an fp16 one
// 1105: 2048 x 1000003 x 64 fp32 forward 1.75 ms, table gradient 1.85 (900 and 852 TFLOP/s of plane products), 8192 x 100003 x 128
// bf16 544 and 600 us (772 and 699).  Matrix unit, vector instructions (an exponential, two cuts, the sums) and LDS (a transposed copy)
// are each busy for 37 to 55 % of that time; none of them alone is the bound.  1024 x 3706 x 64 fp32: 15 and 19 us, latency.
#include "rx_common.h"

#include <type_traits>

typedef __bf16 ct_h8 __attribute__((ext_vector_type(8)));
typedef __bf16 ct_h2 __attribute__((ext_vector_type(2)));
typedef _Float16 ct_f8 __attribute__((ext_vector_type(8)));
typedef _Float16 ct_p2 __attribute__((ext_vector_type(2)));
typedef float ct_f2 __attribute__((ext_vector_type(2)));
typedef float ct_acc __attribute__((ext_vector_type(16)));

#define CT_L2E 1.44269504088896340736f
#define CT_LN2 0.69314718055994530942f
#define CT_NINF (-__builtin_inff())
#define CT_MAXD 256
#define CT_LIM 3.0e38f       // |bias * log2 e| is held inside fp32: masks of the type's lowest value stay finite
// A running reference is set so that the largest weight is 2^CT_BASE and moves when one passes 2^CT_TOP: fp16 weights stay
// below 2^16 (a weight and a target's share on top of it), bf16 ones have room.  The planes hold a weight to 2^-25, that is
// to 2^-36 of the largest beside it.
#define CT_BASE(PL) ((PL) == 2 ? 11.f : 0.f)
#define CT_TOP(PL) ((PL) == 2 ? 14.f : 24.f)
// Sums of weights are held times the tile's scale undone (at most 2^100: a tile of zeros), which 2^CT_TOP of 2^30 items would take
// out of fp32: fp32 operands' sums are held times 2^-CT_DOWN.
#define CT_DOWN(PL) ((PL) == 2 ? 20.f : 0.f)
#define CT_UNIT 9.5367431640625e-7f       // 2^-CT_DOWN(2)
#define CT_THREADS 256
#define CT_WAVES 4

struct CtRow {               // what the backward pass needs of a row
  float m2, l2s, z, sgn;     // p_rv |c_r| = 2^(s log2 e - m2 - l2s), z = m2 + l2s, sgn = sign of c_r
  float q;                   // what stands in for c p at the target
  int32_t y;                 // target or -1
  float ql2;                // log2 |q|
  int32_t pad;
};

union CtFrag { uint4 u; ct_h8 h; ct_f8 f; };

__device__ __forceinline__ uint32_t ct_pk(float a, float b) {
  ct_f2 v = {a, b};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, ct_h2));
}
__device__ __forceinline__ float ct_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float ct_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// two floats -> their words in PL planes (1: bf16, 2: fp16)
template <int PL>
__device__ __forceinline__ void ct_cut2(float a, float b, uint32_t* w) {
  if constexpr (PL == 1) {
    w[0] = ct_pk(a, b);
  } else {
    ct_f2 v = {a, b};
    w[0] = __builtin_bit_cast(uint32_t, __builtin_convertvector(v, ct_p2));
    // a - high, b - high in one mixed-precision instruction each (the compiler converts back and subtracts)
    ct_f2 r;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r.x) : "v"(w[0]), "v"(a));
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r.y) : "v"(w[0]), "v"(b));
    w[1] = __builtin_bit_cast(uint32_t, __builtin_convertvector(r, ct_p2));
  }
}
// power of two that takes a largest magnitude (its bits) to [2^14, 2^15); infinities and NaN stay what they are
__device__ __forceinline__ float ct_scale(uint32_t peak) {
  const int e = 268 - (int)(peak >> 23);
  return __uint_as_float((uint32_t)(e < 227 ? e : 227) << 23);
}
__device__ __forceinline__ float ct_inverse(float scale) { return __uint_as_float((254u << 23) - __float_as_uint(scale)); }
__device__ __forceinline__ float ct_log2(float scale) { return (float)((int)(__float_as_uint(scale) >> 23) - 127); }
__device__ __forceinline__ uint32_t ct_abs(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t ct_umax(uint32_t a, uint32_t b) { return a > b ? a : b; }
// largest of the wavefront, in every lane
__device__ __forceinline__ uint32_t ct_wave_umax(uint32_t v) {
#define CT_DPP(c) v = ct_umax(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, c, 0xf, 0xf, true))
  CT_DPP(0x111); CT_DPP(0x112); CT_DPP(0x114); CT_DPP(0x118);      // rows of 16: shifts by 1, 2, 4, 8
  CT_DPP(0x142); CT_DPP(0x143);                                   // on to the next row, on to the upper half
#undef CT_DPP
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
template <int PL>
__device__ __forceinline__ void ct_cut8(const float* v, CtFrag* f) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t w[PL];
    ct_cut2<PL>(v[2 * i], v[2 * i + 1], w);
#pragma unroll
    for (int p = 0; p < PL; ++p) reinterpret_cast<uint32_t*>(&f[p])[i] = w[p];
  }
}
// acc += A B over the planes, the smallest products first
template <int PL>
__device__ __forceinline__ ct_acc ct_mma(const CtFrag* a, const CtFrag* b, ct_acc c) {
  if constexpr (PL == 2) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[1].f, b[0].f, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[0].f, b[1].f, c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a[0].f, b[0].f, c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[0].h, b[0].h, c, 0, 0, 0);
  }
}

// ---------------------------------------------------------------- global reads
template <typename T> __device__ __forceinline__ float ct_elem(const T* p);
template <> __device__ __forceinline__ float ct_elem<float>(const float* p) { return *p; }
template <> __device__ __forceinline__ float ct_elem<uint16_t>(const uint16_t* p) { return __uint_as_float((uint32_t)*p << 16); }

// four consecutive elements as they lie in memory, at any alignment of their own type: a buffer load needs no more
template <typename T> struct CtQuad;
template <> struct CtQuad<float> { typedef float4 V; };
template <> struct CtQuad<uint16_t> { typedef uint2 V; };
__device__ __forceinline__ float4 ct_floats(const float4& q) { return q; }
__device__ __forceinline__ float4 ct_floats(const uint2& q) { return make_float4(ct_lo(q.x), ct_hi(q.x), ct_lo(q.y), ct_hi(q.y)); }

// `bytes` of memory: four elements from offset `at` on, zeros where that lies outside.  (The whole offset is in the vector
// operand: the scalar one takes no part in the bounds check.)
#define CT_MAXLD (1 << 22)       // 64 rows of four bytes apart at this distance: offsets stay below CT_OUTSIDE
#define CT_OUTSIDE (1 << 30)
struct CtBuffer {
#ifdef __HIP_DEVICE_COMPILE__                                 // the host's pass does not know the type
  __amdgpu_buffer_rsrc_t d;
  __device__ __forceinline__ CtBuffer(const void* p, int bytes) : d(__builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, bytes, 0x27000)) {}
  __device__ __forceinline__ void load(float4& v, int at) const {
    v = __builtin_bit_cast(float4, __builtin_amdgcn_raw_buffer_load_b128(d, at, 0, 0));
  }
  __device__ __forceinline__ void load(uint2& v, int at) const {
    v = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(d, at, 0, 0));
  }
#else
  __device__ CtBuffer(const void*, int) {}
  template <typename V> __device__ void load(V&, int) const {}
#endif
};

// a whole row of fewer than four elements (d = 0; zeros past it), as it would lie in memory
__device__ __forceinline__ float4 ct_short4(const float* row, int d, int D) {
  return make_float4(d < D ? row[d] : 0.f, d + 1 < D ? row[d + 1] : 0.f, d + 2 < D ? row[d + 2] : 0.f, 0.f);
}
__device__ __forceinline__ uint2 ct_short4(const uint16_t* row, int d, int D) {
  uint2 r = make_uint2(0u, 0u);
  if (d < D) r.x = row[d];
  if (d + 1 < D) r.x |= (uint32_t)row[d + 1] << 16;
  if (d + 2 < D) r.y = row[d + 2];
  return r;
}
// elements moved down by n of four, zeros behind them
__device__ __forceinline__ void ct_shift(float4& v, int n) {
  if (n & 1) v = make_float4(v.y, v.z, v.w, 0.f);
  if (n & 2) v = make_float4(v.z, v.w, 0.f, 0.f);
}
__device__ __forceinline__ void ct_shift(uint2& v, int n) {
  const uint64_t u = ((uint64_t)v.y << 32 | v.x) >> (16 * n);
  v = make_uint2((uint32_t)u, (uint32_t)(u >> 32));
}

// stationary operands of the 32 vectors from row0 on (uniform; zeros past `rows` and where `out`): lane column l & 31, element
// ks * 16 + 8 (l >> 5) + j; returns what the scores have to be multiplied with to undo the vector's scale
template <typename T, int PL, int DP>
__device__ __forceinline__ float ct_stationary(const T* base, int64_t ld, int64_t row0, int64_t rows, int D, bool out, CtFrag (*f)[PL]) {
  const int l31 = rx_lane() & 31, h = rx_lane() >> 5, step = (int)ld * (int)sizeof(T);
  const int left = rows <= row0 ? 0 : rows - row0 < 32 ? (int)(rows - row0) : 32;
  // in scalar registers for certain: a 64-bit comparison takes them out, and a descriptor elsewhere means a loop over its values
  const uint64_t at0 = (uint64_t)(base + (left ? row0 : 0) * ld);
  const T* first = (const T*)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(at0 >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)at0));
  const CtBuffer b(first, __builtin_amdgcn_readfirstlane(left ? (left - 1) * step + D * (int)sizeof(T) : 0));
  const bool mine = l31 < left && !out;
  typename CtQuad<T>::V raw[DP / 16][2];
#pragma unroll
  for (int ks = 0; ks < DP / 16; ++ks)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int d = ks * 16 + h * 8 + u * 4, at = d + 4 <= D ? d : D - 4;
      const bool on = mine && d < D;
      if (DP == 32 && D < 4) raw[ks][u] = on ? ct_short4(first + l31 * ld, d, D) : typename CtQuad<T>::V{};
      else b.load(raw[ks][u], on ? l31 * step + at * (int)sizeof(T) : CT_OUTSIDE);
    }
  if (D % 4 != 0 && D >= 4) {
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int d = ks * 16 + h * 8 + u * 4;
        ct_shift(raw[ks][u], d < D && d + 4 > D ? d + 4 - D : 0);
      }
  }
  float scale = 1.f;
  if constexpr (PL == 2) {
    uint32_t peak = 0;
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const float4 a = ct_floats(raw[ks][u]);
        peak = ct_umax(ct_umax(peak, ct_umax(ct_abs(a.x), ct_abs(a.y))), ct_umax(ct_abs(a.z), ct_abs(a.w)));
      }
    scale = ct_scale(ct_umax(peak, (uint32_t)__shfl_xor((int)peak, 32, 64)));
  }
#pragma unroll
  for (int ks = 0; ks < DP / 16; ++ks) {
    const float4 a = ct_floats(raw[ks][0]), c = ct_floats(raw[ks][1]);
    float v[8] = {a.x, a.y, a.z, a.w, c.x, c.y, c.z, c.w};
    if constexpr (PL == 2) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] *= scale;
    }
    ct_cut8<PL>(v, f[ks]);
  }
  return ct_inverse(scale);
}

// ---------------------------------------------------------------- streaming tiles
// A tile of BN vectors in LDS: rm[PL][BN][DP + 8] row-major and, with TR, tr[PL][DP][BN] transposed.  In the
// transposed copy the 16 vectors of a contraction step lie as {0-3, 8-11, 4-7, 12-15}: the order in which the two
// halves of a wavefront hold the scores.  Row-major rows are an odd multiple of 16 bytes apart, so that 16-byte reads down
// the rows meet every bank equally often; the transposed copy, written 8 bytes at a time by threads four rows apart as
// well as read down its rows, permutes the 16-byte chunks of a row instead (ct_swz).
template <int PL, int DP, int BN, bool TR, int NT>
struct CtTile {
  static constexpr int RS = DP + 8, TS = BN;
  static constexpr int RM = PL * BN * RS, TM = TR ? PL * DP * TS : 0;    // 16-bit elements
  static constexpr int BYTES = (RM + TM) * 2;
  static constexpr int BLOCKS = BN * DP / 16, PER = (BLOCKS + NT - 1) / NT;   // 4 x 4 blocks, per thread
};

// chunk of row d that holds chunk c: eight neighbouring rows, and eight rows four apart, take different banks
template <int BN>
__device__ __forceinline__ int ct_swz(int d, int c) {
  if constexpr (BN == 64) return c ^ ((((d & 3) << 1) | ((d >> 2) & 1)) ^ ((d >> 3) & 7));
  else return c ^ (((d & 2) | ((d >> 2) & 1)) ^ ((d >> 3) & 3));
}

template <typename T, int PL, int DP, int BN, bool TR, int NT>
struct CtStage {
  typedef CtTile<PL, DP, BN, TR, NT> Tile;
  typedef typename CtQuad<T>::V Quad;          // as they lie in memory, of four vectors
  Quad v[Tile::PER][4];
  // Vectors [row0, row0 + BN) of the streaming side, zeros past `rows`.  A row's last, partial four elements are read as its
  // last four and put in place by settle(): nothing here waits for what it loads.  The loads go through a buffer descriptor:
  // what lies outside is zero without a branch, and one offset per block of a thread is all the registers they need.
  __device__ __forceinline__ void load(const T* base, int64_t ld, int64_t row0, int64_t rows, int D) {
    const int left = rows - row0 < BN ? (int)(rows - row0) : BN, step = (int)ld * (int)sizeof(T);
    const CtBuffer b(base + row0 * ld, (left - 1) * step + D * (int)sizeof(T));
#pragma unroll
    for (int q = 0; q < Tile::PER; ++q) {
      const int blk = q * NT + threadIdx.x;
      const int d = blk % (DP / 4) * 4, i = blk / (DP / 4) * 4, at = d + 4 <= D ? d : D - 4;
      const bool on = d < D && (Tile::BLOCKS % NT == 0 || blk < Tile::BLOCKS);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (DP == 32 && D < 4) v[q][k] = i + k < left && on ? ct_short4(base + (row0 + i + k) * ld, d, D) : Quad{};
        else b.load(v[q][k], on ? (i + k) * step + at * (int)sizeof(T) : CT_OUTSIDE);
      }
    }
  }
  __device__ __forceinline__ void settle(int D) {
    if (D % 4 == 0 || D < 4) return;
#pragma unroll
    for (int q = 0; q < Tile::PER; ++q) {
      const int d = (q * NT + threadIdx.x) % (DP / 4) * 4, n = d < D && d + 4 > D ? d + 4 - D : 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) ct_shift(v[q][k], n);
    }
  }
  // Some vectors become zeros, whatever they hold: items that are out (bias -inf: their score is -inf all the same) in the
  // forward pass, rows without a gradient (ct_prep_kernel's marks: their weights are 0) in the backward pass.
  float bias[Tile::PER][4];
  uint32_t mark[Tile::PER];    // a byte per vector: the branch below is rarely taken, and four floats cost 180 us of 590
  __device__ __forceinline__ void load_bias(const float* b, int64_t row0, int64_t rows) {
#pragma unroll
    for (int q = 0; q < Tile::PER; ++q)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int64_t row = row0 + (q * NT + threadIdx.x) / (DP / 4) * 4 + k;
        bias[q][k] = row < rows ? b[row] : 0.f;
      }
  }
  __device__ __forceinline__ void load_marks(const uint8_t* m, int64_t row0) {     // of whole tiles, 4-byte aligned
#pragma unroll
    for (int q = 0; q < Tile::PER; ++q) {
      const int blk = q * NT + threadIdx.x;
      mark[q] = *reinterpret_cast<const uint32_t*>(m + row0 + (Tile::BLOCKS % NT == 0 || blk < Tile::BLOCKS ? blk / (DP / 4) * 4 : 0));
    }
  }
  __device__ __forceinline__ void drop_marked() {
    uint32_t any = 0;
#pragma unroll
    for (int q = 0; q < Tile::PER; ++q) any |= mark[q];
    if (!__ballot(any != 0)) return;
#pragma unroll
    for (int q = 0; q < Tile::PER; ++q)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (mark[q] >> (8 * k) & 255) v[q][k] = Quad{};
  }
  __device__ __forceinline__ void drop() {
#pragma unroll
    for (int q = 0; q < Tile::PER; ++q)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (bias[q][k] == CT_NINF) v[q][k] = Quad{};
  }
  // bits of the largest magnitude the wavefront holds
  __device__ __forceinline__ uint32_t peak() const {
    uint32_t m = 0;
#pragma unroll
    for (int q = 0; q < Tile::PER; ++q)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if constexpr (PL == 2)
          m = ct_umax(ct_umax(m, ct_umax(ct_abs(v[q][k].x), ct_abs(v[q][k].y))), ct_umax(ct_abs(v[q][k].z), ct_abs(v[q][k].w)));
    return ct_wave_umax(m);
  }
  // into LDS, times `scale`; `flip` (may be null): sign words of the tile's vectors, applied to the transposed copy
  __device__ __forceinline__ void store(uint16_t* rm, uint16_t* tr, const uint32_t* flip, float scale) {
#pragma unroll
    for (int q = 0; q < Tile::PER; ++q) {
      const int blk = q * NT + threadIdx.x;
      if (Tile::BLOCKS % NT != 0 && blk >= Tile::BLOCKS) continue;
      const int d = blk % (DP / 4) * 4, ib = blk / (DP / 4);
      uint32_t w[4][2][PL];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (PL == 2) {
          ct_cut2<PL>(v[q][k].x * scale, v[q][k].y * scale, w[k][0]);
          ct_cut2<PL>(v[q][k].z * scale, v[q][k].w * scale, w[k][1]);
        } else {
          w[k][0][0] = v[q][k].x;
          w[k][1][0] = v[q][k].y;
        }
      }
#pragma unroll
      for (int p = 0; p < PL; ++p)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          *reinterpret_cast<uint2*>(rm + (p * BN + ib * 4 + k) * Tile::RS + d) = make_uint2(w[k][0][p], w[k][1][p]);
      if constexpr (TR) {
        if (flip) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t f = flip[ib * 4 + k];
#pragma unroll
            for (int p = 0; p < PL; ++p) { w[k][0][p] ^= f; w[k][1][p] ^= f; }
          }
        }
        const int pos = (ib >> 2) * 16 + ((ib & 1) * 2 + ((ib >> 1) & 1)) * 4;
#pragma unroll
        for (int p = 0; p < PL; ++p)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t sel = (e & 1) ? 0x07060302u : 0x05040100u;     // upper or lower halves of two words
            const uint32_t a = __builtin_amdgcn_perm(w[1][e >> 1][p], w[0][e >> 1][p], sel);
            const uint32_t b = __builtin_amdgcn_perm(w[3][e >> 1][p], w[2][e >> 1][p], sel);
            *reinterpret_cast<uint2*>(tr + (p * DP + d + e) * Tile::TS + ct_swz<BN>(d + e, pos >> 3) * 8 + (pos & 4)) = make_uint2(a, b);
          }
      }
    }
  }
};

// scores of 32 streaming vectors [it * 32, + 32) of the tile against the stationary block
template <int PL, int DP, int BN>
__device__ __forceinline__ ct_acc ct_scores(const uint16_t* rm, int it, const CtFrag (*st)[PL]) {
  typedef CtTile<PL, DP, BN, true, 256> Tile;
  const int l31 = rx_lane() & 31, h = rx_lane() >> 5;
  ct_acc s = {};
#pragma unroll
  for (int ks = 0; ks < DP / 16; ++ks) {
    CtFrag a[PL];
#pragma unroll
    for (int p = 0; p < PL; ++p) a[p].u = *reinterpret_cast<const uint4*>(rm + (p * BN + it * 32 + l31) * Tile::RS + ks * 16 + h * 8);
    s = ct_mma<PL>(a, st[ks], s);
    if constexpr (DP == 256) __builtin_amdgcn_sched_barrier(0);      // registers are full: no fragments ahead of their use
  }
  return s;
}
// out[db] += transposed tile (dims db * 32 ..) x weights, w[16] in the scores' register order
template <int PL, int DP, int BN, bool SUM = false>
__device__ __forceinline__ void ct_weigh(const uint16_t* tr, int it, const float* w, ct_acc* out, float* sum = nullptr) {
  typedef CtTile<PL, DP, BN, true, 256> Tile;
  const int l31 = rx_lane() & 31, h = rx_lane() >> 5;
#pragma unroll
  for (int k2 = 0; k2 < 2; ++k2) {
    CtFrag b[PL];
    ct_cut8<PL>(w + k2 * 8, b);
    if constexpr (SUM) {                    // of the weights as they are used
      const ct_h2 one = {(__bf16)1.f, (__bf16)1.f};
      const uint32_t u[4] = {b[0].u.x, b[0].u.y, b[0].u.z, b[0].u.w};
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) s = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(ct_h2, u[i]), one, s, false);
      *sum += s;
    }
#pragma unroll
    for (int db = 0; db < DP / 32; ++db) {
      CtFrag a[PL];
#pragma unroll
      for (int p = 0; p < PL; ++p)
        a[p].u = *reinterpret_cast<const uint4*>(tr + (p * DP + db * 32 + l31) * Tile::TS + ct_swz<BN>(db * 32 + l31, it * 4 + k2 * 2 + h) * 8);
      out[db] = ct_mma<PL>(a, b, out[db]);
      if constexpr (DP == 256) __builtin_amdgcn_sched_barrier(0);
    }
  }
}

// element e of four neighbouring LDS floats: one 16-byte read for the four of them
__device__ __forceinline__ float ct_at(const float* p, int e) {
  const float4 f = *reinterpret_cast<const float4*>(p);
  return e == 0 ? f.x : e == 1 ? f.y : e == 2 ? f.z : f.w;
}
__device__ __forceinline__ float ct_bias2(float b) {      // bias in log2 units; what is finite stays finite, infinities and NaN stay what they are
  return fabsf(b) < __builtin_inff() ? fminf(fmaxf(b * CT_L2E, -CT_LIM), CT_LIM) : b;
}

// Which split and which stationary tile a workgroup takes.  Workgroups are dealt to the 8 XCDs in turn; with the splits
// dealt the same way all tiles of one split meet its part of the streaming side in one L2.
__device__ __forceinline__ void ct_place(int tiles, int n_split, int* tile, int* split) {
  const int b = blockIdx.x;
  if (n_split % 8 == 0) {
    *split = b % 8 + 8 * (b / (8 * tiles));
    *tile = b / 8 % tiles;
  } else {
    *split = b / tiles;
    *tile = b % tiles;
  }
}

// sum of 16 weights in four roundings
__device__ __forceinline__ float ct_sum16(const float* w) {
  float p[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) p[i] = w[2 * i] + w[2 * i + 1];
  return ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
}
// sum += add, with the rounding that the last such addition lost: near-equal terms would all round the same way
__device__ __forceinline__ void ct_add(float add, float* sum, float* lost) {
  add -= *lost;
  const float s = *sum + add;
  *lost = (s - *sum) - add;
  *sum = s;
}

// ---------------------------------------------------------------- forward
struct CtFwd {
  const void *x, *t;
  int64_t ld_x, ld_t, R, V;
  const float* bias;
  int D, tiles, n_split;
  int64_t per_split;           // items per split, a multiple of the tile
  const int64_t* targets;      // a row's target takes no part in what follows
  float2* part;                // [n_split][R]: reference, sum times 2^-CT_DOWN
  float* rest;                 // [n_split][R], bf16 with MEAN: the same sum, of the weights as out has them
  float* out;                  // [n_split][R][D]: sum of weight * t_v
};

// The loop has one barrier per tile: while tile i is worked on, tile i + 1 goes from registers into the other LDS buffer
// and tile i + 2 from memory into the registers; its largest magnitude is known one barrier before its scale is needed.
template <typename T, int PL, int DP, int MB, int BN, bool MEAN, bool BIAS, int NW, int OCC>
__global__ void __launch_bounds__(NW * 64, OCC) ct_fwd_kernel(CtFwd a) {
  typedef CtTile<PL, DP, BN, MEAN, NW * 64> Tile;
  extern __shared__ __align__(16) uint8_t ct_lds[];
  float* lb = reinterpret_cast<float*>(ct_lds + 2 * Tile::BYTES);           // [2][BN] bias
  uint32_t* lm = reinterpret_cast<uint32_t*>(lb + 2 * BN);                  // [2][NW] largest magnitudes
  int tile, split;
  ct_place(a.tiles, a.n_split, &tile, &split);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l31 = rx_lane() & 31, h = rx_lane() >> 5;
  const int64_t row0 = ((int64_t)tile * NW + wave) * (32 * MB);
  const int64_t v0 = split * a.per_split, v1 = v0 + a.per_split < a.V ? v0 + a.per_split : a.V;
  const int n = (int)((v1 - v0 + BN - 1) / BN);             // tiles of this split, at least one
  CtStage<T, PL, DP, BN, MEAN, NW * 64> stage;
  float nb = 0.f;
  auto fetch = [&](int i) {
    const int64_t v = v0 + (int64_t)i * BN;
    stage.load((const T*)a.t, a.ld_t, v, v1, a.D);
    if constexpr (BIAS) stage.load_bias(a.bias, v, v1);
    if (BIAS && threadIdx.x < BN) nb = v + threadIdx.x < v1 ? ct_bias2(a.bias[v + threadIdx.x]) : CT_NINF;
  };
  auto publish = [&](int i) {
    stage.settle(a.D);
    if constexpr (BIAS) stage.drop();
    if constexpr (PL == 2) {
      const uint32_t m = stage.peak();
      if (rx_lane() == 0) lm[(i & 1) * NW + wave] = m;
    }
  };
  auto put = [&](int i) -> float {                          // tile i into its buffer; returns its scale
    float scale = 1.f;
    if constexpr (PL == 2) {
      uint32_t m = 0;
#pragma unroll
      for (int w = 0; w < NW; ++w) m = ct_umax(m, lm[(i & 1) * NW + w]);
      scale = ct_scale(m);
    }
    uint16_t* rm = reinterpret_cast<uint16_t*>(ct_lds + (i & 1) * Tile::BYTES);
    stage.store(rm, rm + Tile::RM, nullptr, scale);
    if (BIAS && threadIdx.x < BN) lb[(i & 1) * BN + threadIdx.x] = nb;
    return scale;
  };
  fetch(0);
  CtFrag st[MB][DP / 16][PL];
  ct_acc o[MB][MEAN ? DP / 32 : 1] = {};
  // w = 2^((score - ref) + (kt - kr)), kt the tile's scale undone; sum: of w / 2^(kt + CT_DOWN).  Without a bias kt is part of the
  // score and kr stays 0: one operation less per score.  A bias may be a mask of 1e38, which would swallow it.
  float inv[MB], ref[MB], kr[MB], sum[MB], lost[MB];
  float rest[MB];                                          // bf16 with MEAN
  int32_t target[MB];                                      // or -1; counted from the next tile's first item
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) {
    inv[mb] = CT_L2E * ct_stationary<T, PL, DP>((const T*)a.x, a.ld_x, row0 + mb * 32, a.R, a.D, false, st[mb]);
    ref[mb] = CT_NINF;
    kr[mb] = sum[mb] = lost[mb] = rest[mb] = 0.f;
    const int64_t row = row0 + mb * 32 + l31, y = row < a.R ? a.targets[row] : -1;
    target[mb] = y >= v0 && y < v1 ? (int32_t)(y - v0) : -1;
  }
  publish(0);
  __syncthreads();
  float scale = put(0), next = 1.f;
  if (n > 1) {
    fetch(1);
    publish(1);
  }
  __syncthreads();
  for (int i = 0; i < n; ++i) {
    if (i + 1 < n) {
      next = put(i + 1);
      if (i + 2 < n) fetch(i + 2);
    }
    const uint16_t* rm = reinterpret_cast<const uint16_t*>(ct_lds + (i & 1) * Tile::BYTES);
    const uint16_t* tr = rm + Tile::RM;
    const float* bb = lb + (i & 1) * BN;
    const float kt = PL == 2 ? -ct_log2(scale) : 0.f, back = ct_inverse(scale), unit = scale * CT_UNIT;
    const int64_t left = v1 - v0 - (int64_t)i * BN;
    const int live = left < BN ? (int)left : BN;
    bool mine = false;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) mine = mine || (uint32_t)target[mb] < (uint32_t)BN;
    const bool special = live < BN || __ballot(mine) != 0;    // items past the end, or a row's target
#pragma unroll
    for (int it = 0; it < BN / 32; ++it) {
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) {
        const ct_acc s = ct_scores<PL, DP, BN>(rm, it, st[mb]);
        const float mul = PL == 2 ? inv[mb] * back : CT_L2E;
        float r0 = ref[mb] == CT_NINF ? 0.f : ref[mb];
        const float kb = PL == 2 && BIAS ? kt : 0.f;
        float w[16], mx = CT_NINF;
        // without a bias: relative to the reference at once
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          if constexpr (BIAS) w[e] = fmaf(s[e], mul, ct_at(bb + it * 32 + 8 * (e / 4) + 4 * h, e % 4));
          else w[e] = fmaf(s[e], mul, (PL == 2 ? kt : 0.f) - r0);
        }
        if (special) {
          int end = live - (it * 32 + 4 * h), at = target[mb] - (it * 32 + 4 * h);
          asm volatile("" : "+v"(end), "+v"(at));             // the comparisons are for few tiles only, and stay behind the branch
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int k = 8 * (e / 4) + e % 4;
            if (k >= end || k == at) w[e] = CT_NINF;
          }
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) mx = fmaxf(mx, w[e]);
        const float base = ref[mb] == CT_NINF ? CT_NINF : BIAS ? ref[mb] - (kb - kr[mb]) : 0.f;
        if (__ballot(mx > base + CT_TOP(PL))) {               // rare after the first tile
          const float m = fmaxf(mx, __shfl_xor(mx, 32, 64));
          if (m > base + CT_TOP(PL)) {                        // both halves of a row decide alike
            const float nk = BIAS ? kb - CT_BASE(PL) : 0.f, nr = BIAS ? m : (m + r0) - CT_BASE(PL);
            if (ref[mb] != CT_NINF) {
              const float f = __builtin_amdgcn_exp2f((ref[mb] - nr) + (kr[mb] - nk));
              sum[mb] *= f;
              lost[mb] *= f;
              rest[mb] *= f;
              if constexpr (MEAN) {
#pragma unroll
                for (int db = 0; db < DP / 32; ++db)
#pragma unroll
                  for (int e = 0; e < 16; ++e) o[mb][db][e] *= f;
              }
            }
            if constexpr (!BIAS) {
#pragma unroll
              for (int e = 0; e < 16; ++e) w[e] -= nr - r0;
            }
            ref[mb] = r0 = nr;
            kr[mb] = nk;
          }
        }
        const float dk = kb - kr[mb];
#pragma unroll
        for (int e = 0; e < 16; ++e) w[e] = __builtin_amdgcn_exp2f(!BIAS ? w[e] : PL == 2 ? (w[e] - r0) + dk : w[e] - r0);
        ct_add(PL == 2 ? ct_sum16(w) * unit : ct_sum16(w), &sum[mb], &lost[mb]);
        if constexpr (MEAN) ct_weigh<PL, DP, BN, PL == 1>(tr, it, w, o[mb], &rest[mb]);
      }
    }
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) target[mb] -= BN;
    if (i + 2 < n) publish(i);
    scale = next;
    __syncthreads();
  }
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) {
    float total = sum[mb] + __shfl_xor(sum[mb], 32, 64);
    const float others = MEAN && PL == 1 ? rest[mb] + __shfl_xor(rest[mb], 32, 64) : 0.f;
    if constexpr (PL == 2 && BIAS) {                          // back to 2^(score - ref)
      const float f = __builtin_amdgcn_exp2f(kr[mb]);
      total *= f;
      if constexpr (MEAN) {
#pragma unroll
        for (int db = 0; db < DP / 32; ++db)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[mb][db][i] *= f;
      }
    }
    const int64_t row = row0 + mb * 32 + l31;
    if (row >= a.R) continue;
    if (h == 0) a.part[(int64_t)split * a.R + row] = make_float2(ref[mb], total);
    if constexpr (MEAN) {
      if (PL == 1 && h == 0) a.rest[(int64_t)split * a.R + row] = others;
      float* out = a.out + ((int64_t)split * a.R + row) * a.D;
      const bool v4 = a.D % 4 == 0;
#pragma unroll
      for (int db = 0; db < DP / 32; ++db)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int d = db * 32 + 8 * q + 4 * h;
          if (v4 && d < a.D) *reinterpret_cast<float4*>(out + d) = make_float4(o[mb][db][4 * q], o[mb][db][4 * q + 1], o[mb][db][4 * q + 2], o[mb][db][4 * q + 3]);
          else
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (d + i < a.D) out[d + i] = o[mb][db][4 * q + i];
        }
    }
  }
}

// Joins a row's splits and its target, whose score is a plain dot product: TPR threads per row, which share out the splits as
// well as the dimensions.  A wavefront per row (64) for up to 8 splits, where 8192 rows of 4 take 21 us against 29; a
// workgroup (256) for more: 143 rows of 512 splits 50 us with the pass before it, against 170.
struct CtJoin {
  const void *x, *t;
  int64_t ld_x, ld_t, R, V;
  const float* bias;
  const int64_t* targets;
  int D, n_split;
  const float2* part;
  const float *rest, *out;
  float *logprob, *lse, *stats, *mean;
};
template <typename T>
__device__ __forceinline__ float ct_dot(const T* x, const T* t, int D) {
  float s = 0.f;
  for (int d = rx_lane(); d < D; d += 64) s = fmaf(ct_elem(x + d), ct_elem(t + d), s);
  return rx_wave_sum(s);
}
// sum or maximum over a row's threads, in every one of them
template <bool MAX, int TPR>
__device__ __forceinline__ float ct_row(float v, float* w) {
  for (int x = 32; x > 0; x >>= 1) v = MAX ? fmaxf(v, __shfl_xor(v, x, 64)) : v + __shfl_xor(v, x, 64);
  if constexpr (TPR == 64) return v;
  __syncthreads();
  if (rx_lane() == 0) w[threadIdx.x >> 6] = v;
  __syncthreads();
  return MAX ? fmaxf(fmaxf(w[0], w[1]), fmaxf(w[2], w[3])) : (w[0] + w[1]) + (w[2] + w[3]);
}
template <typename T, int TPR>
__global__ void __launch_bounds__(CT_THREADS) ct_join_kernel(CtJoin a, int32_t* err) {
  __shared__ float w[CT_WAVES], sums[CT_THREADS];
  const int64_t row = (int64_t)blockIdx.x * (CT_THREADS / TPR) + threadIdx.x / TPR;
  const int lane = rx_lane(), tid = threadIdx.x % TPR;
  if (TPR == 64 && row >= a.R) return;
  constexpr int PL = sizeof(T) == 4 ? 2 : 1;
  const int64_t y = a.targets[row];
  const bool ok = y >= 0 && y < a.V;
  const float bias = ok && a.bias ? a.bias[y] : 0.f, b2 = ct_bias2(bias);
  const float dot = ok ? ct_dot((const T*)a.x + row * a.ld_x, (const T*)a.t + y * a.ld_t, a.D) : 0.f;
  const float mine = ok && bias != CT_NINF ? fmaf(dot, CT_L2E, b2) : CT_NINF;      // the target's score, in log2 units
  float ref = CT_NINF;
  for (int q = tid; q < a.n_split; q += TPR) ref = fmaxf(ref, a.part[(int64_t)q * a.R + row].x);
  ref = ct_row<true, TPR>(ref, w);
  const float r0 = ref == CT_NINF ? 0.f : ref;
  float sum = 0.f, used = 0.f;             // of all but the target: their sum, and that of the weights as the mean has them
  for (int q = tid; q < a.n_split; q += TPR) {
    const float2 p = a.part[(int64_t)q * a.R + row];
    const float f = __builtin_amdgcn_exp2f(p.x - r0);
    sum += p.y * f;
    if (PL == 1 && a.mean) used += a.rest[(int64_t)q * a.R + row] * f;
  }
  sum = ct_row<false, TPR>(sum, w);
  used = PL == 1 && a.mean ? ct_row<false, TPR>(used, w) : sum;
  // Weight of the others and of the target relative to the larger of the two, 2^m2.  A reference holds the tile's scale undone, up to
  // 100, and the sum makes up for it: their integer parts meet first (unless the reference is too large to take them, a mask), or
  // all that follows would round at that size.
  const float up = (float)__builtin_amdgcn_frexp_expf(sum) + CT_DOWN(PL), near = r0 + up;
  const bool fits = near - r0 == up;
  const float m2 = sum == 0.f ? (mine == CT_NINF ? 0.f : mine) : fmaxf(fits ? near : r0, mine);
  const float others = sum == 0.f ? 0.f
      : fits ? __builtin_amdgcn_frexp_mantf(sum) * __builtin_amdgcn_exp2f(near - m2) : sum * __builtin_amdgcn_exp2f(r0 - m2 + CT_DOWN(PL));
  const float own = __builtin_amdgcn_exp2f(mine - m2), s = others + own;
  const bool empty = s == 0.f;
  const float l2s = empty ? 0.f : log2f(s), lse = empty ? CT_NINF : (m2 + l2s) * CT_LN2;
  const float rest = empty ? 0.f : others / s;
  if (a.mean) {
    const int wide = a.D <= 32 ? 32 : a.D <= 64 ? 64 : a.D <= 128 ? 128 : 256;
    const int dp = wide < TPR ? wide : TPR, groups = TPR / dp;      // threads along the dimensions, and along the splits
    for (int d0 = 0; d0 < a.D; d0 += dp) {
      const int d = d0 + tid % dp;
      float m = 0.f;
      if (d < a.D) {
#pragma unroll 4
        for (int q = tid / dp; q < a.n_split; q += groups)
          m = fmaf(a.out[((int64_t)q * a.R + row) * a.D + d], __builtin_amdgcn_exp2f(a.part[(int64_t)q * a.R + row].x - r0), m);
      }
      if constexpr (TPR == 64) {
        if (groups == 2) m += __shfl_xor(m, 32, 64);
      } else {
        sums[tid] = m;
        __syncthreads();
        if (tid < dp)
          for (int k = 1; k < groups; ++k) m += sums[k * dp + tid];
      }
      if (tid < dp && d < a.D) a.mean[row * a.D + d] = sum == 0.f ? 0.f : (PL == 2 ? m * CT_UNIT : m) / sum * rest;
    }
  }
  if (tid >= 64) return;
  float lp = y == -1 ? 0.f : __builtin_nanf("");
  if (ok) {
    if (empty || bias == CT_NINF) lp = CT_NINF;
    else if (fabsf(b2) == CT_LIM && fabsf(m2) < 1e38f) lp = dot + bias - lse;      // a mask of the type's lowest value
    else lp = (mine - m2 - l2s) * CT_LN2;
  }
  if (lane == 0) {
    if (!ok && y != -1 && err) atomicOr(err, RX_ERR_INDEX);
    a.logprob[row] = lp;
    a.lse[row] = lse;
    if (a.stats) {                         // -inf: no item left.  Of p_y and 1 - p_y the smaller, the second one with its sign changed.
      const float py = empty ? 0.f : own <= others ? own / s : -rest;
      reinterpret_cast<float4*>(a.stats)[row] = make_float4(empty ? CT_NINF : m2, l2s, sum == 0.f ? 0.f : used / sum * rest, py);
    }
  }
}

// ---------------------------------------------------------------- backward
struct CtPrep {
  const void* t;
  int64_t ld_t, R, V;
  const float* bias;
  const int64_t* targets;
  int D;
  const float *stats, *mean, *g, *gl;
  void* dx;
  CtRow* rows;
  uint8_t* marks;              // 1: nothing of the row reaches the table's gradient
};
// dx, and the rows as the table's pass wants them; one wavefront per row
template <typename T>
__global__ void __launch_bounds__(CT_THREADS) ct_prep_kernel(CtPrep a) {
  const int64_t row = (int64_t)blockIdx.x * CT_WAVES + (threadIdx.x >> 6);
  if (row >= a.R) return;
  const float4 st = reinterpret_cast<const float4*>(a.stats)[row];
  int64_t y = a.targets[row];
  const bool dead = st.x == CT_NINF;
  if (dead || y < 0 || y >= a.V || (a.bias && a.bias[y] == CT_NINF)) y = -1;      // nothing depends on such a target
  const float g = y >= 0 && a.g ? a.g[row] : 0.f;
  const float gl = dead || !a.gl ? 0.f : a.gl[row], c = gl - g;
  const bool none = g == 0.f && gl == 0.f;                  // such a row may hold anything
  const bool sure = __float_as_uint(st.w) >> 31;            // see the forward pass
  const float py = sure ? 1.f + st.w : st.w, rest = sure ? -st.w : 1.f - st.w;
  const float share = none || y < 0 ? 0.f : fmaf(g, rest, gl * py);
  if (rx_lane() == 0 && a.rows) {
    CtRow r;
    r.sgn = c < 0.f ? -1.f : 1.f;
    r.m2 = dead || none ? 0.f : st.x;
    r.l2s = c == 0.f ? __builtin_inff() : st.y - log2f(fabsf(c));
    r.z = r.m2 + r.l2s;
    r.q = share;
    r.y = (int32_t)y;
    r.ql2 = log2f(fabsf(share));
    r.pad = 0;
    a.rows[row] = r;
    a.marks[row] = none;
  }
  if (a.dx) {
    const float q = none || y < 0 ? 0.f : fmaf(g, st.z, gl * py);       // under the weights that the mean has
    const T* t = (const T*)a.t + (y < 0 ? 0 : y) * a.ld_t;
    for (int d = rx_lane(); d < a.D; d += 64) {
      float v = c == 0.f ? 0.f : c * a.mean[row * a.D + d];
      if (y >= 0 && !none) v = fmaf(q, ct_elem(t + d), v);
      if constexpr (sizeof(T) == 4) ((float*)a.dx)[row * a.D + d] = v;
      else ((uint16_t*)a.dx)[row * a.D + d] = (uint16_t)ct_pk(v, v);
    }
  }
}

struct CtBwd {
  const void *x, *t;
  int64_t ld_x, ld_t, R, V;
  const float* bias;
  const CtRow* rows;
  const uint8_t* marks;
  int D, tiles, n_split;
  int64_t per_split;           // rows per split, a multiple of the tile
  void* dt;                    // [V][D] in the table's type, or fp32 [n_split][V][D]
  float* db;                   // [V], or [n_split][V]
  bool partial;
};

template <typename T, int PL, int DP, int MB, int BN, bool BIAS, int NW, int OCC>
__global__ void __launch_bounds__(NW * 64, OCC) ct_bwd_kernel(CtBwd a) {
  typedef CtTile<PL, DP, BN, true, NW * 64> Tile;
  extern __shared__ __align__(16) uint8_t ct_lds[];
  float* lz0 = reinterpret_cast<float*>(ct_lds + 2 * Tile::BYTES); // [2][7][BN], see below
  uint32_t* lm = reinterpret_cast<uint32_t*>(lz0 + 14 * BN);       // [2][NW] largest magnitudes
  int tile, split;
  ct_place(a.tiles, a.n_split, &tile, &split);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = rx_lane(), l31 = lane & 31, h = lane >> 5;
  const int64_t item0 = ((int64_t)tile * NW + wave) * (32 * MB);
  const int64_t r0 = split * a.per_split, r1 = r0 + a.per_split < a.R ? r0 + a.per_split : a.R;
  const int n = (int)((r1 - r0 + BN - 1) / BN);             // tiles of this split, at least one
  CtStage<T, PL, DP, BN, true, NW * 64> stage;
  CtRow info;
  auto fetch = [&](int i) {
    const int64_t r = r0 + (int64_t)i * BN;
    stage.load((const T*)a.x, a.ld_x, r, r1, a.D);
    stage.load_marks(a.marks, r);
    if (threadIdx.x < BN) {
      if (r + threadIdx.x < r1) info = a.rows[r + threadIdx.x];
      else { info.m2 = 0.f; info.l2s = info.z = __builtin_inff(); info.sgn = 1.f; info.q = 0.f; info.ql2 = CT_NINF; info.y = -1; }
    }
  };
  auto publish = [&](int i) {      // before the barrier in front of put(i): the largest magnitude, the sign words
    stage.settle(a.D);
    stage.drop_marked();
    if constexpr (PL == 2) {
      const uint32_t m = stage.peak();
      if (lane == 0) lm[(i & 1) * NW + wave] = m;
    }
    if (threadIdx.x < BN) reinterpret_cast<uint32_t*>(lz0 + (i & 1) * 7 * BN)[5 * BN + threadIdx.x] = info.sgn < 0.f ? 0x80008000u : 0u;
  };
  auto put = [&](int i) -> float {
    float scale = 1.f;
    if constexpr (PL == 2) {
      uint32_t m = 0;
#pragma unroll
      for (int w = 0; w < NW; ++w) m = ct_umax(m, lm[(i & 1) * NW + w]);
      scale = ct_scale(m);
    }
    const float kt = PL == 2 ? -ct_log2(scale) : 0.f;
    float* lz = lz0 + (i & 1) * 7 * BN;
    if (threadIdx.x < BN) {
      float* p = lz + threadIdx.x;
      p[0] = BIAS ? info.m2 : info.z - kt;
      if (BIAS) { p[BN] = info.l2s - kt; p[2 * BN] = info.sgn * (PL == 2 ? scale * CT_UNIT : scale); }   // sign of c, with the tile's scale undone
      p[3 * BN] = info.q * info.sgn;
      p[4 * BN] = __int_as_float(info.y);
      p[6 * BN] = info.ql2 + kt;
    }
    uint16_t* rm = reinterpret_cast<uint16_t*>(ct_lds + (i & 1) * Tile::BYTES);
    stage.store(rm, rm + Tile::RM, reinterpret_cast<const uint32_t*>(lz + 5 * BN), scale);
    return scale;
  };
  fetch(0);
  CtFrag st[MB][DP / 16][PL];
  float inv[MB], b2[MB], dbias[MB], lost[MB], ref[MB];      // ref: of w = 2^(log2 (|c| p) + kt - ref); PL == 1 keeps it at 0
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) {
    const int64_t item = item0 + mb * 32 + l31;
    b2[mb] = BIAS && item < a.V ? ct_bias2(a.bias[item]) : 0.f;
    const bool out = b2[mb] == CT_NINF;                       // an item that is out may hold anything
    inv[mb] = CT_L2E * ct_stationary<T, PL, DP>((const T*)a.t, a.ld_t, item0 + mb * 32, a.V, a.D, out, st[mb]);
    dbias[mb] = lost[mb] = 0.f;
    ref[mb] = PL == 2 ? CT_NINF : 0.f;
  }
  ct_acc o[MB][DP / 32] = {};
  publish(0);
  __syncthreads();
  float scale = put(0), next = 1.f;
  if (n > 1) {
    fetch(1);
    publish(1);
  }
  __syncthreads();
  for (int i = 0; i < n; ++i) {
    if (i + 1 < n) {
      next = put(i + 1);
      if (i + 2 < n) fetch(i + 2);
    }
    const uint16_t* rm = reinterpret_cast<const uint16_t*>(ct_lds + (i & 1) * Tile::BYTES);
    const uint16_t* tr = rm + Tile::RM;
    const float* lz = lz0 + (i & 1) * 7 * BN;             // z, or m2 with a bias
    const float *ll = lz + BN, *lsg = lz + 2 * BN, *lq = lz + 3 * BN, *lql = lz + 6 * BN;
    const float* ly = lz + 4 * BN;                        // int32 targets
    const float kt = PL == 2 ? -ct_log2(scale) : 0.f, back = ct_inverse(scale);
    // rows of this tile whose target is among the wavefront's items
    const int32_t of = lane < BN ? __float_as_int(ly[lane]) : -1;
    const int64_t rel = of >= 0 ? of - item0 : -1;
    const uint64_t hits = __ballot(rel >= 0 && rel < 32 * MB);
  // bf16, 128 wide and with a bias: both halves of a tile at once spill 44 registers (1203 us against 721 at 8192 x 100k)
#pragma unroll BIAS && PL == 1 && DP == 128 ? 1 : BN / 32
    for (int it = 0; it < BN / 32; ++it) {
      const bool hit = (uint32_t)(hits >> (it * 32)) != 0;
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) {
        const ct_acc s = ct_scores<PL, DP, BN>(rm, it, st[mb]);
        const float mul = PL == 2 ? inv[mb] * back : CT_L2E;
        float w[16], mx = CT_NINF;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int k = it * 32 + 8 * (e / 4) + 4 * h;
          if constexpr (BIAS) w[e] = (fmaf(s[e], mul, b2[mb]) - ct_at(lz + k, e % 4)) - ct_at(ll + k, e % 4);
          else w[e] = fmaf(s[e], mul, -ct_at(lz + k, e % 4));
        }
        const int32_t mine = (int32_t)(item0 + mb * 32 + l31);
        if constexpr (PL == 2) {
          if (hit) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const int k = it * 32 + 8 * (e / 4) + 4 * h;
              w[e] = __float_as_int(ct_at(ly + k, e % 4)) == mine ? ct_at(lql + k, e % 4) : w[e];
            }
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) mx = fmaxf(mx, w[e]);
          if (__ballot(mx > ref[mb] + CT_TOP(PL))) {
            const float n = fmaxf(mx, __shfl_xor(mx, 32, 64));
            if (n > ref[mb] + CT_TOP(PL)) {
              if (ref[mb] != CT_NINF) {
                const float f = __builtin_amdgcn_exp2f(ref[mb] - (n - CT_BASE(PL)));
                dbias[mb] *= f;
                lost[mb] *= f;
#pragma unroll
                for (int db = 0; db < DP / 32; ++db)
#pragma unroll
                  for (int e = 0; e < 16; ++e) o[mb][db][e] *= f;
              }
              ref[mb] = n - CT_BASE(PL);
            }
          }
        }
        const float rf = ref[mb] == CT_NINF ? 0.f : ref[mb];
#pragma unroll
        for (int e = 0; e < 16; ++e) w[e] = __builtin_amdgcn_exp2f(PL == 2 ? w[e] - rf : w[e]);
        if (hit) {                // a row's own target: sgn(c) q in place of |c| p, still to meet sgn(c) x
          // two factors: q 2^(kt - ref) is below 2^CT_TOP, 2^(kt - ref) alone is out of range for a q below 2^-114 (and for 0 anything)
          const float up = PL == 2 ? __builtin_amdgcn_exp2f(fminf(0.5f * (kt - rf), 126.f)) : 1.f;
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int k = it * 32 + 8 * (e / 4) + 4 * h;
            const float share = PL == 2 ? ct_at(lq + k, e % 4) * up * up : ct_at(lq + k, e % 4);
            w[e] = __float_as_int(ct_at(ly + k, e % 4)) == mine ? share : w[e];
          }
        }
        if constexpr (BIAS) {       // a sum over all rows: 16 at a time, each sum joined with the rounding that the last join lost
          float part[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float* sg = lsg + it * 32 + 8 * q + 4 * h;
            part[q] = fmaf(w[4 * q + 1], ct_at(sg, 1), w[4 * q] * ct_at(sg, 0)) + fmaf(w[4 * q + 3], ct_at(sg, 3), w[4 * q + 2] * ct_at(sg, 2));
          }
          ct_add((part[0] + part[1]) + (part[2] + part[3]), &dbias[mb], &lost[mb]);
        }
        ct_weigh<PL, DP, BN>(tr, it, w, o[mb]);
        if (PL == 1 && hit) {     // a target's share may be as large as the whole gradient: what bf16 dropped of these weights goes in too
#pragma unroll
          for (int e = 0; e < 16; e += 2) {
            const uint32_t u = ct_pk(w[e], w[e + 1]);
            w[e] -= ct_lo(u);
            w[e + 1] -= ct_hi(u);
          }
          ct_weigh<PL, DP, BN>(tr, it, w, o[mb]);
        }
      }
    }
    if (i + 2 < n) publish(i);
    scale = next;
    __syncthreads();
  }
  if constexpr (PL == 2) {        // back from the references, in two steps: 2^ref alone may be below the smallest number
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
      const float f = ref[mb] == CT_NINF ? 1.f : __builtin_amdgcn_exp2f(0.5f * ref[mb]);
      dbias[mb] = dbias[mb] * f * f / CT_UNIT;
#pragma unroll
      for (int db = 0; db < DP / 32; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[mb][db][i] = o[mb][db][i] * f * f;
    }
  }
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) {
    const float total = dbias[mb] + __shfl_xor(dbias[mb], 32, 64);
    const int64_t item = item0 + mb * 32 + l31;
    if (item >= a.V) continue;
    const int64_t at = (a.partial ? (int64_t)split * a.V : 0) + item;
    if (BIAS && h == 0) a.db[at] = total;
    const bool v4 = a.D % 4 == 0;
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int d = db * 32 + 8 * q + 4 * h;
        const float e[4] = {o[mb][db][4 * q], o[mb][db][4 * q + 1], o[mb][db][4 * q + 2], o[mb][db][4 * q + 3]};
        if (sizeof(T) == 4 || a.partial) {
          float* p = (float*)a.dt + at * a.D + d;
          if (v4 && d < a.D) *reinterpret_cast<float4*>(p) = make_float4(e[0], e[1], e[2], e[3]);
          else
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (d + i < a.D) p[i] = e[i];
        } else {
          uint16_t* p = (uint16_t*)a.dt + at * a.D + d;
          if (v4 && d < a.D) *reinterpret_cast<uint2*>(p) = make_uint2(ct_pk(e[0], e[1]), ct_pk(e[2], e[3]));
          else
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (d + i < a.D) p[i] = (uint16_t)ct_pk(e[i], e[i]);
        }
      }
  }
}

// sums of n_split partial arrays in split order: n elements of the table gradient, nb of the bias gradient behind them
template <typename T>
__global__ void __launch_bounds__(CT_THREADS) ct_sum_kernel(const float* __restrict__ part, int64_t n, const float* __restrict__ part_b,
                                                            int64_t nb, int n_split, T* __restrict__ out, float* __restrict__ out_b) {
  for (int64_t i = (int64_t)blockIdx.x * CT_THREADS + threadIdx.x; i < n + nb; i += (int64_t)gridDim.x * CT_THREADS) {
    const bool b = i >= n;
    const float* p = b ? part_b + (i - n) : part + i;
    const int64_t step = b ? nb : n;
    float s = 0.f;
#pragma unroll 8
    for (int q = 0; q < n_split; ++q) s += p[q * step];
    if (b) out_b[i - n] = s;
    else if constexpr (sizeof(T) == 4) out[i] = s;
    else out[i] = (uint16_t)ct_pk(s, s);
  }
}

// ---------------------------------------------------------------- host
// Padded widths.  Without 96 and 192 train passes (forward + backward) over 100003 items took 370 + 417 us instead of 314 + 355 at
// 2048 x 80 fp32, 161 + 174 instead of 145 + 141 in bf16, 447 + 841 instead of 370 + 539 at 1024 x 160 fp32.
static int ct_dp(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : D <= 96 ? 96 : D <= 128 ? 128 : D <= 192 ? 192 : 256; }
// X(T, PL, DP, MB, BN, NW, OCC): the kernels there are, one per element type and padded width: MB blocks of 32 stationary vectors
// for each of NW wavefronts, tiles of BN streaming ones, OCC workgroups per CU.  MB, BN: what the registers (256 with OCC = 2) and
// the LDS of a double-buffered tile leave.  bf16 of 32 and 64 has room for two blocks: the gradient at 4096 x 100003 takes 129
// and 157 us, with one 153 and 186.  fp32 of 64 with two and OCC = 1 took 571 where one with OCC = 2 took 453.
#define CT_KERNELS(X, bf16, dp)                                                  \
  (bf16 ? dp == 32 ? X(uint16_t, 1, 32, 2, 64, 4, 2)                             \
          : dp == 64 ? X(uint16_t, 1, 64, 2, 64, 4, 2)                           \
          : dp == 96 ? X(uint16_t, 1, 96, 1, 64, 4, 2)                           \
          : dp == 128 ? X(uint16_t, 1, 128, 1, 64, 4, 2)                         \
          : dp == 192 ? X(uint16_t, 1, 192, 1, 32, 4, 1)                         \
                      : X(uint16_t, 1, 256, 1, 32, 4, 1)                         \
   : dp == 32 ? X(float, 2, 32, 1, 64, 4, 2)                                     \
   : dp == 64 ? X(float, 2, 64, 1, 64, 4, 2)                                     \
   : dp == 96 ? X(float, 2, 96, 1, 32, 4, 2)                                     \
   : dp == 128 ? X(float, 2, 128, 1, 32, 4, 2)                                   \
   : dp == 192 ? X(float, 2, 192, 1, 32, 4, 1)                                   \
               : X(float, 2, 256, 1, 32, 4, 1))

// stationary vectors per workgroup and streaming ones per tile, of the kernels in CT_KERNELS
#define CT_BM(T, PL, DP, MB, BN, NW, OCC) ((NW) * 32 * (MB))
#define CT_BN(T, PL, DP, MB, BN, NW, OCC) (BN)
#define CT_OCC(T, PL, DP, MB, BN, NW, OCC) (OCC)

struct CtPlan {
  int tiles, n_split;
  int64_t per_split;
};
// `fixed` vectors are stationary, `moving` ones stream.  The number of splits is the one with the least time by this
// estimate, in tiles of the stream: rounds of `slots` workgroups (what the chip holds at a time), each as long as its share of
// the stream and two tiles more for the stationary vectors and the result; a last round that leaves every other workgroup
// of a CU out takes 0.65 of one; a partial result on its way to memory and back costs 1/200, a pass that adds them up `join`.
// At 372 x 17389 x 240 (fp32) this takes 85 splits where four workgroups per CU were 341: 91 against 169 us.
static CtPlan ct_plan(int64_t fixed, int64_t moving, int bm, int bn, int slots, float join) {
  CtPlan p;
  p.tiles = (int)rx_cdiv(fixed, bm);
  const int64_t stream = rx_cdiv(moving, bn);
  const int64_t most = stream < 8 * slots / p.tiles + 1 ? stream : 8 * slots / p.tiles + 1;
  float best = 0.f;
  p.per_split = 0;
  for (int64_t n = 1; n <= most; n += n < 64 ? 1 : 8) {
    const int64_t per = rx_cdiv(stream, n), blocks = p.tiles * rx_cdiv(stream, per), rest = blocks % slots;
    const float rounds = (float)(blocks / slots) + (rest == 0 ? 0.f : rest > slots / 2 || slots == 256 ? 1.f : 0.65f);
    const float cost = rounds * (float)(per + 2) + (per < stream ? (float)blocks / 200.f + join : 0.f);
    if (p.per_split == 0 || cost < best) {
      best = cost;
      p.per_split = per * bn;
    }
  }
  p.n_split = (int)rx_cdiv(moving, p.per_split);
  return p;
}

static size_t ct_rest_at(const CtPlan& p, int64_t R) { return rx_align_up((size_t)p.n_split * R * sizeof(float2), 256); }
static size_t ct_out_at(const CtPlan& p, int64_t R, int bf16) { return ct_rest_at(p, R) + (bf16 ? rx_align_up((size_t)p.n_split * R * 4, 256) : 0); }

static int ct_check(const rx_catalog_args* a, const char* who) {
  RX_REQUIRE(a, "%s: null argument", who);
  RX_REQUIRE(a->R >= 0 && a->R <= (1 << 24) && a->V >= 1 && a->V <= (1ll << 30) && a->D >= 1 && a->D <= CT_MAXD,
             "%s: bad shape R=%lld V=%lld D=%d (R up to 2^24, V up to 2^30, D up to %d)", who, (long long)a->R, (long long)a->V, a->D, CT_MAXD);
  RX_REQUIRE(a->ld_x >= a->D && a->ld_t >= a->D, "%s: row strides %lld, %lld below D=%d", who, (long long)a->ld_x, (long long)a->ld_t, a->D);
  RX_REQUIRE(a->ld_x <= CT_MAXLD && a->ld_t <= CT_MAXLD, "%s: rows %lld, %lld elements apart (at most %d)", who, (long long)a->ld_x,
             (long long)a->ld_t, CT_MAXLD);
  RX_REQUIRE(a->bf16 == 0 || a->bf16 == 1, "%s: bad element type %d", who, a->bf16);
  if (a->R == 0) return 0;
  RX_REQUIRE(a->x && a->table && a->targets, "%s: null argument", who);
  const uintptr_t al = a->bf16 ? 1 : 3;
  RX_REQUIRE(((uintptr_t)a->x & al) == 0 && ((uintptr_t)a->table & al) == 0, "%s: x or table not aligned to their elements", who);
  return 0;
}
static CtPlan ct_fwd_plan(int64_t R, int64_t V, int D, int bf16) {
  const int dp = ct_dp(D);
  return ct_plan(R, V, CT_KERNELS(CT_BM, bf16, dp), CT_KERNELS(CT_BN, bf16, dp), 256 * CT_KERNELS(CT_OCC, bf16, dp), 0.f);
}
static CtPlan ct_bwd_plan(int64_t R, int64_t V, int D, int bf16, bool bias) {
  const int dp = ct_dp(D);
  // two blocks and a bias do not fit the registers of two wavefronts per SIMD: one there (ct_pick_bwd)
  const int bm = CT_KERNELS(CT_BM, bf16, dp) / (bf16 && dp == 64 && bias ? 2 : 1);
  // the narrow fp32 kernel uses few enough registers for three workgroups per CU
  const int occ = !bf16 && dp == 32 ? 3 : CT_KERNELS(CT_OCC, bf16, dp);
  return ct_plan(V, R, bm, CT_KERNELS(CT_BN, bf16, dp), 256 * occ, 0.8f);
}

extern "C" size_t rx_catalog_fwd_workspace_bytes(int64_t R, int64_t V, int32_t D, int32_t bf16, int32_t want_mean) {
  if (R <= 0 || V <= 0 || D < 1 || D > CT_MAXD) return 0;
  const CtPlan p = ct_fwd_plan(R, V, D, bf16);
  return want_mean ? ct_out_at(p, R, bf16) + (size_t)p.n_split * R * D * 4 : ct_rest_at(p, R);
}
extern "C" size_t rx_catalog_bwd_workspace_bytes(int64_t R, int64_t V, int32_t D, int32_t bf16, int32_t want_bias) {
  if (R <= 0 || V <= 0 || D < 1 || D > CT_MAXD) return 0;
  const CtPlan p = ct_bwd_plan(R, V, D, bf16, want_bias != 0);
  return rx_align_up((size_t)R * sizeof(CtRow), 256) + rx_align_up((size_t)R, 256) +
         (p.n_split > 1 ? rx_align_up((size_t)p.n_split * V * D * 4, 256) + (want_bias ? (size_t)p.n_split * V * 4 : 0) : 0);
}

template <typename K>
static int ct_allow_lds(K kernel, int bytes) {
  if (bytes > 64 * 1024) RX_HIP(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
  return 0;
}
template <typename T, int PL, int DP, int MB, int BN, int NW, int OCC, bool MEAN, bool BIAS>
static int ct_go_fwd(const CtFwd& f, hipStream_t st) {
  auto kernel = ct_fwd_kernel<T, PL, DP, MB, BN, MEAN, BIAS, NW, OCC>;
  const int lds = 2 * CtTile<PL, DP, BN, MEAN, NW * 64>::BYTES + 2 * BN * 4 + 2 * NW * 4;
  if (ct_allow_lds(kernel, lds)) return 1;
  hipLaunchKernelGGL(kernel, dim3((unsigned)(f.tiles * f.n_split)), dim3(NW * 64), lds, st, f);
  return 0;
}
template <typename T, int PL, int DP, int MB, int BN, int NW, int OCC>
static int ct_pick_fwd(const CtFwd& f, hipStream_t st) {
  if (f.out) return f.bias ? ct_go_fwd<T, PL, DP, MB, BN, NW, OCC, true, true>(f, st) : ct_go_fwd<T, PL, DP, MB, BN, NW, OCC, true, false>(f, st);
  return f.bias ? ct_go_fwd<T, PL, DP, MB, BN, NW, OCC, false, true>(f, st) : ct_go_fwd<T, PL, DP, MB, BN, NW, OCC, false, false>(f, st);
}
template <typename T, int PL, int DP, int MB, int BN, int NW, int OCC, bool BIAS>
static int ct_go_bwd(const CtBwd& f, hipStream_t st) {
  auto kernel = ct_bwd_kernel<T, PL, DP, MB, BN, BIAS, NW, OCC>;
  const int lds = 2 * CtTile<PL, DP, BN, true, NW * 64>::BYTES + 14 * BN * 4 + 2 * NW * 4;
  if (ct_allow_lds(kernel, lds)) return 1;
  hipLaunchKernelGGL(kernel, dim3((unsigned)(f.tiles * f.n_split)), dim3(NW * 64), lds, st, f);
  return 0;
}
template <typename T, int PL, int DP, int MB, int BN, int NW, int OCC>
static int ct_pick_bwd(const CtBwd& f, hipStream_t st) {
  return f.db ? ct_go_bwd<T, PL, DP, DP == 64 ? 1 : MB, BN, NW, OCC, true>(f, st) : ct_go_bwd<T, PL, DP, MB, BN, NW, OCC, false>(f, st);
}

extern "C" int rx_catalog_fwd(const rx_catalog_args* args, float* d_logprob, float* d_lse, float* d_stats, float* d_mean, void* ws,
                              size_t ws_bytes, int32_t* err_flag, int device, void* stream) {
  if (ct_check(args, "rx_catalog_fwd")) return 1;
  const rx_catalog_args a = *args;
  if (a.R == 0) return 0;
  RX_REQUIRE(d_logprob && d_lse, "rx_catalog_fwd: null output");
  RX_REQUIRE(((uintptr_t)d_stats & 15) == 0, "rx_catalog_fwd: stats must be 16-byte aligned");
  const size_t need = rx_catalog_fwd_workspace_bytes(a.R, a.V, a.D, a.bf16, d_mean != nullptr);
  RX_REQUIRE(ws && ws_bytes >= need && ((uintptr_t)ws & 15) == 0, "rx_catalog_fwd: workspace of %zu bytes, %zu needed", ws_bytes, need);
  RX_GUARD_DEVICE(device);
  const CtPlan p = ct_fwd_plan(a.R, a.V, a.D, a.bf16);
  float2* part = (float2*)ws;
  float* rest = d_mean ? (float*)((uint8_t*)ws + ct_rest_at(p, a.R)) : nullptr;
  float* out = d_mean ? (float*)((uint8_t*)ws + ct_out_at(p, a.R, a.bf16)) : nullptr;
  CtFwd f = {a.x, a.table, a.ld_x, a.ld_t, a.R, a.V, a.bias, a.D, p.tiles, p.n_split, p.per_split, a.targets, part, rest, out};
  hipStream_t st = (hipStream_t)stream;
#define CT_GO(...) ct_pick_fwd<__VA_ARGS__>(f, st)
  const int rc = CT_KERNELS(CT_GO, a.bf16, ct_dp(a.D));
#undef CT_GO
  if (rc) return rc;
  RX_LAUNCH_CHECK();
  CtJoin j = {a.x, a.table, a.ld_x, a.ld_t, a.R, a.V, a.bias, a.targets, a.D, p.n_split, part, rest, out, d_logprob, d_lse, d_stats, d_mean};
  const bool few = p.n_split <= 8;
  auto join = few ? (a.bf16 ? ct_join_kernel<uint16_t, 64> : ct_join_kernel<float, 64>)
                  : (a.bf16 ? ct_join_kernel<uint16_t, 256> : ct_join_kernel<float, 256>);
  hipLaunchKernelGGL(join, dim3((unsigned)(few ? rx_cdiv(a.R, CT_WAVES) : a.R)), dim3(CT_THREADS), 0, st, j, err_flag);
  RX_LAUNCH_CHECK();
  return 0;
}

extern "C" int rx_catalog_bwd(const rx_catalog_args* args, const float* d_stats, const float* d_mean, const float* d_g_logprob,
                              const float* d_g_lse, void* d_dx, void* d_dtable, float* d_dbias, void* ws, size_t ws_bytes, int device,
                              void* stream) {
  if (ct_check(args, "rx_catalog_bwd")) return 1;
  const rx_catalog_args a = *args;
  if (a.R == 0) return 0;
  RX_REQUIRE(d_stats && ((uintptr_t)d_stats & 15) == 0, "rx_catalog_bwd: stats missing or not 16-byte aligned");
  RX_REQUIRE(!d_dx || d_mean, "rx_catalog_bwd: the gradient of x needs the means of the forward call");
  RX_REQUIRE(!d_dbias || (a.bias && d_dtable), "rx_catalog_bwd: the bias gradient needs a bias and comes with the table's");
  RX_REQUIRE(!a.bias || !d_dtable || d_dbias, "rx_catalog_bwd: with a bias the table's gradient comes with the bias gradient");
  RX_REQUIRE(((uintptr_t)d_dtable & 15) == 0 && ((uintptr_t)d_dx & (a.bf16 ? 1 : 3)) == 0, "rx_catalog_bwd: gradient buffers not aligned");
  const bool want_t = d_dtable != nullptr;
  const size_t need = want_t ? rx_catalog_bwd_workspace_bytes(a.R, a.V, a.D, a.bf16, d_dbias != nullptr) : 0;
  RX_REQUIRE(!want_t || (ws && ws_bytes >= need && ((uintptr_t)ws & 15) == 0), "rx_catalog_bwd: workspace of %zu bytes, %zu needed",
             ws_bytes, need);
  RX_GUARD_DEVICE(device);
  hipStream_t st = (hipStream_t)stream;
  CtRow* rows = want_t ? (CtRow*)ws : nullptr;
  uint8_t* marks = want_t ? (uint8_t*)ws + rx_align_up((size_t)a.R * sizeof(CtRow), 256) : nullptr;    // rounded up to whole tiles
  CtPrep q = {a.table, a.ld_t, a.R, a.V, a.bias, a.targets, a.D, d_stats, d_mean, d_g_logprob, d_g_lse, d_dx, rows, marks};
  const dim3 grid((unsigned)rx_cdiv(a.R, CT_WAVES));
  if (a.bf16) hipLaunchKernelGGL(ct_prep_kernel<uint16_t>, grid, dim3(CT_THREADS), 0, st, q);
  else hipLaunchKernelGGL(ct_prep_kernel<float>, grid, dim3(CT_THREADS), 0, st, q);
  RX_LAUNCH_CHECK();
  if (!want_t) return 0;
  const CtPlan p = ct_bwd_plan(a.R, a.V, a.D, a.bf16, d_dbias != nullptr);
  uint8_t* w = marks + rx_align_up((size_t)a.R, 256);
  const bool partial = p.n_split > 1;
  float* pt = (float*)w;
  float* pb = (float*)(w + rx_align_up((size_t)p.n_split * a.V * a.D * 4, 256));
  CtBwd f = {a.x, a.table, a.ld_x, a.ld_t, a.R, a.V, a.bias, rows, marks, a.D, p.tiles, p.n_split, p.per_split,
             partial ? (void*)pt : d_dtable, partial ? (d_dbias ? pb : nullptr) : d_dbias, partial};
#define CT_GO(...) ct_pick_bwd<__VA_ARGS__>(f, st)
  const int rc = CT_KERNELS(CT_GO, a.bf16, ct_dp(a.D));
#undef CT_GO
  if (rc) return rc;
  RX_LAUNCH_CHECK();
  if (partial) {
    const int64_t n = a.V * a.D, nb = d_dbias ? a.V : 0;
    const dim3 g((unsigned)(rx_cdiv(n + nb, CT_THREADS) < 8192 ? rx_cdiv(n + nb, CT_THREADS) : 8192));
    if (a.bf16) hipLaunchKernelGGL(ct_sum_kernel<uint16_t>, g, dim3(CT_THREADS), 0, st, pt, n, pb, nb, p.n_split, (uint16_t*)d_dtable, d_dbias);
    else hipLaunchKernelGGL(ct_sum_kernel<float>, g, dim3(CT_THREADS), 0, st, pt, n, pb, nb, p.n_split, (float*)d_dtable, d_dbias);
    RX_LAUNCH_CHECK();
  }
  return 0;
}
