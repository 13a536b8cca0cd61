// List-wise log-probabilities (gfx950): for scores l [R, V], per row
//   lse = log sum_v exp l_v,  logprob_t = l_{y_t} - lse,  H = lse - sum_v p_v l_v,  the k largest l_v,
// and the gradient  dl_v = sum_t g_t (1[v = y_t] - p_v) + g_lse p_v - g_H p_v (log p_v + H).
//
// Both directions read every score once and are bound by that read (and the write of dl): the softmax statistics are
// online.  Each lane keeps its own running reference m (log2 units), sum s = sum 2^(l' - m) and t = sum 2^(l' - m) (l' - m)
// with l' = l log2(e); the reference moves only when a score exceeds it by 2^4, so the rescale is off the common path.
// m is a rounded number, and a score's distance from it is off by half of m's last step: no more than one up to LP_BIG, which is why
// it is never below -LP_FLOOR (a lane that sees nothing but masks sums up zeros) and why rows whose largest score lies
// beyond LP_BIG are read a second time.  What lanes, wavefronts and column splits join at the end is in score units, relative to
// the largest score itself.  All sums are fp32, whatever the scores' type.
// Alternatives: a wavefront keeps the 64 best keys (value, column) sorted across its lanes; scores that beat the k-th
// one are collected in a small LDS buffer and merged 64 at a time, so a row costs one compare per 16 bytes in the
// common case.  Keys order by value, then by the lower column, and are unique, so the result does not depend on
// how the row was split.
// Measured: 2048 x 50021 bf16, rows ending anywhere (half of all columns live): forward 30 us (3.4 TB/s), gradient 61 us (5.0 TB/s
// read and written); 1 x 1000003 fp32, 50 alternatives: 12 us and 6 for the join; 6040 x 100, 10 alternatives: 8.9 us.
#include "rx_common.h"

#define LP_SMALL 1024        // rows up to this width: one wavefront (or part of one) per row, scores in registers
#define LP_WIDE 256          // threads per split of a wide row
#define LP_TOP 64            // most alternatives per row
#define LP_SPLIT_MIN 4096    // fewest columns worth a split of their own
#define LP_SPLIT_MAX 256
#define LP_L2E 1.44269504088896340736f
#define LP_LN2 0.69314718055994530942f
#define LP_BIG 16777216.f    // |largest score| up to which l * log2(e) - m is good to one; other rows take the form (l - m) log2(e)
#define LP_FLOOR 33554432.f  // below -LP_BIG in log2 units, by more than any weight survives
#define LP_NINF (-__builtin_inff())

typedef uint32_t lp_u4 __attribute__((ext_vector_type(4)));

struct LpPart {   // one split's share of a row
  float raw;      // largest score
  float s, t;     // sums relative to it
  float pad;
};

// ---------------------------------------------------------------- element access
template <typename T> __device__ __forceinline__ float lp_elem(const T* p);
template <> __device__ __forceinline__ float lp_elem<float>(const float* p) { return *p; }
template <> __device__ __forceinline__ float lp_elem<uint16_t>(const uint16_t* p) { return __uint_as_float((uint32_t)*p << 16); }

template <typename T> struct LpVec { static constexpr int N = 16 / (int)sizeof(T); };

template <typename T>
__device__ __forceinline__ void lp_unpack(const lp_u4& q, float* v);
template <>
__device__ __forceinline__ void lp_unpack<float>(const lp_u4& q, float* v) {
  v[0] = __uint_as_float(q.x); v[1] = __uint_as_float(q.y); v[2] = __uint_as_float(q.z); v[3] = __uint_as_float(q.w);
}
template <>
__device__ __forceinline__ void lp_unpack<uint16_t>(const lp_u4& q, float* v) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

__device__ __forceinline__ uint16_t lp_to_bf16(float f) {   // round to nearest even; NaN stays NaN
  const uint32_t u = __float_as_uint(f);
  if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t)((u >> 16) | 0x40u);
  return (uint16_t)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
}
template <typename T> __device__ __forceinline__ void lp_put(T* p, float f);
template <> __device__ __forceinline__ void lp_put<float>(float* p, float f) { *p = f; }
template <> __device__ __forceinline__ void lp_put<uint16_t>(uint16_t* p, float f) { *p = lp_to_bf16(f); }

// of loaded values; fmaxf would quiet each of them first.  NaN loses against a number.
__device__ __forceinline__ float lp_max3(float a, float b, float c) {
  float d;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "v"(c));
  return d;
}
// value of lane ^ M without going through LDS: quad permutes, row mirrors and rotations, and the swaps of 16 and 32 lanes
template <int M>
__device__ __forceinline__ uint32_t lp_xor(uint32_t x) {
#define LP_DPP(v, c) (uint32_t)__builtin_amdgcn_mov_dpp((int)(v), c, 0xf, 0xf, true)
  if constexpr (M == 1) return LP_DPP(x, 0xB1);                     // quad_perm 1,0,3,2
  else if constexpr (M == 2) return LP_DPP(x, 0x4E);                // quad_perm 2,3,0,1
  else if constexpr (M == 4) return LP_DPP(LP_DPP(x, 0x141), 0x1B); // half row mirrored (^ 7), quads reversed (^ 3)
  else if constexpr (M == 8) return LP_DPP(x, 0x128);               // row rotated by 8
  else if constexpr (M == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return (rx_lane() & 16) ? r[0] : r[1];
  } else {
    const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return (rx_lane() & 32) ? r[0] : r[1];
  }
#undef LP_DPP
}
template <int M>
__device__ __forceinline__ float lp_xorf(float v) { return __uint_as_float(lp_xor<M>(__float_as_uint(v))); }
// largest / sum over G neighbouring lanes, in each of them
template <int G>
__device__ __forceinline__ float lp_max(float v) {
  if constexpr (G > 1) {
    const float o = lp_xorf<G / 2>(v);
    return lp_max<G / 2>(lp_max3(v, o, o));
  } else return v;
}
template <int G>
__device__ __forceinline__ float lp_sum(float v) {
  if constexpr (G > 1) return lp_sum<G / 2>(v + lp_xorf<G / 2>(v));
  else return v;
}
__device__ __forceinline__ float lp_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// ---------------------------------------------------------------- alternatives
// key: order-preserving image of the value above, complemented column below; larger key = better alternative
__device__ __forceinline__ uint64_t lp_key(float v, int32_t col) {
  const uint32_t u = __float_as_uint(v + 0.0f);            // -0 counts as 0
  const uint32_t o = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((uint64_t)o << 32) | (uint32_t)~col;
}
__device__ __forceinline__ float lp_key_value(uint64_t key) {
  const uint32_t o = (uint32_t)(key >> 32);
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}
// the next smaller score (of a finite one or +inf)
__device__ __forceinline__ float lp_below(float v) {
  const uint32_t u = __float_as_uint(v);
  return __uint_as_float(v > 0.f ? u - 1 : v < 0.f ? u + 1 : 0x80000001u);
}
__device__ __forceinline__ int32_t lp_key_col(uint64_t key) { return (int32_t)~(uint32_t)key; }
// key 0 is no score's key: value bits 0 would be the image of a negative NaN

template <int M>
__device__ __forceinline__ uint64_t lp_xor64(uint64_t x) {
  return ((uint64_t)lp_xor<M>((uint32_t)(x >> 32)) << 32) | lp_xor<M>((uint32_t)x);
}
// compare-exchange with lane ^ ST: lanes with `small` keep the smaller key
template <int ST>
__device__ __forceinline__ uint64_t lp_exchange(uint64_t x, bool small) {
  const uint64_t o = lp_xor64<ST>(x);
  return ((x < o) == small) ? x : o;
}
template <int SIZE, int ST>
__device__ __forceinline__ uint64_t lp_stage(uint64_t x) {
  const int lane = rx_lane();
  const bool up = SIZE == 64 || (lane & SIZE) == 0, low = (lane & ST) == 0;
  x = lp_exchange<ST>(x, up == low);
  if constexpr (ST > 1) return lp_stage<SIZE, ST / 2>(x);
  else return x;
}
// keys of the wavefront's lanes in ascending lane order (bitonic network, 21 compare-exchange steps)
__device__ __forceinline__ uint64_t lp_sort_up(uint64_t x) {
  x = lp_stage<2, 1>(x);
  x = lp_stage<4, 2>(x);
  x = lp_stage<8, 4>(x);
  x = lp_stage<16, 8>(x);
  x = lp_stage<32, 16>(x);
  return lp_stage<64, 32>(x);
}
// best 64 of `list` (descending over the lanes) and `cand` (ascending), descending
template <int ST>
__device__ __forceinline__ uint64_t lp_down(uint64_t x) {
  x = lp_exchange<ST>(x, (rx_lane() & ST) != 0);
  if constexpr (ST > 1) return lp_down<ST / 2>(x);
  else return x;
}
__device__ __forceinline__ uint64_t lp_merge(uint64_t list, uint64_t cand) {
  return lp_down<32>(list > cand ? list : cand);
}
__device__ __forceinline__ uint64_t lp_lane64(uint64_t x, int lane) {
  const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)x, lane), hi = __builtin_amdgcn_readlane((uint32_t)(x >> 32), lane);
  return ((uint64_t)hi << 32) | lo;
}

// One wavefront's list of alternatives: `list` sorted over the lanes, `buf` [128] candidates waiting in LDS.
struct LpTop {
  uint64_t list;
  uint64_t* buf;
  int cnt;
  float thr;       // score of the k-th alternative, as of the last refresh(); -inf while there are fewer
  __device__ __forceinline__ void init(uint64_t* b) { list = 0; buf = b; cnt = 0; thr = LP_NINF; }
  __device__ __forceinline__ void take(uint64_t key) { list = lp_merge(list, lp_sort_up(key)); }
  // lanes with `on` add their key; called by the whole wavefront
  __device__ __forceinline__ void push(bool on, uint64_t key) {
    const uint64_t mask = __ballot(on);
    if (!mask) return;
    if (on) buf[cnt + __popcll(mask & ((1ull << rx_lane()) - 1))] = key;
    cnt += (int)__popcll(mask);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (cnt >= 64) {
      const uint64_t a = buf[rx_lane()], b = buf[64 + rx_lane()];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      cnt -= 64;
      if (rx_lane() < cnt) buf[rx_lane()] = b;
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      take(a);
    }
  }
  __device__ __forceinline__ void flush() {
    if (!cnt) return;
    take(rx_lane() < cnt ? buf[rx_lane()] : 0);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    cnt = 0;
  }
  // The filter admits only scores above the k-th of the list.  It is refreshed between two groups of columns, never
  // inside one: all columns of the list are then lower than any column still to come, so an equal score may go.
  __device__ __forceinline__ void refresh(int k) {
    const uint64_t kth = lp_lane64(list, k - 1);
    thr = kth ? lp_key_value(kth) : LP_NINF;
  }
};

// ---------------------------------------------------------------- shared row pieces
struct LpRow {
  float ref, l2s;        // final reference (a score) and log2 of the sum of weights relative to it
  float lse, H;
  bool empty;
};

// raw: largest score; s, t relative to it
__device__ __forceinline__ LpRow lp_finish(float raw, float s, float t) {
  LpRow r;
  r.empty = raw == LP_NINF && s == s;        // nothing above -inf (and no NaN): no distribution
  r.ref = raw == LP_NINF ? 0.f : raw;
  r.l2s = log2f(s);
  r.lse = r.empty ? LP_NINF : r.ref + r.l2s * LP_LN2;
  r.H = r.empty ? 0.f : (r.l2s - t / s) * LP_LN2;
  return r;
}
// log-probability of a score, from the reference rather than from the rounded lse
__device__ __forceinline__ float lp_of(const LpRow& r, float l) {
  return l == LP_NINF || r.empty ? LP_NINF : (l - r.ref) - r.l2s * LP_LN2;
}
// what the gradient needs of a row: (reference, log2 s, 1: empty row, H).  Kept apart from lse, whose rounding would cost the
// probabilities a factor of 1 + |lse| 2^-24.
__device__ __forceinline__ void lp_write_row(const rx_logprob_args& a, const LpRow& r, int64_t row) {
  a.lse[row] = r.lse;
  a.entropy[row] = r.H;
  if (a.stats) reinterpret_cast<float4*>(a.stats)[row] = make_float4(r.ref, r.l2s, r.empty ? 1.f : 0.f, r.H);
}
__device__ __forceinline__ int32_t lp_live(const rx_logprob_args& a, int64_t row) {
  if (!a.lengths) return (int32_t)a.V;
  const int64_t n = a.lengths[row];
  return (int32_t)(n < 0 ? 0 : n > a.V ? a.V : n);
}
template <typename T>
__device__ __forceinline__ void lp_write_target(const rx_logprob_args& a, const LpRow& r, const T* l, int32_t n, int64_t row, int t, int32_t* err) {
  const int64_t y = a.targets[row * a.T + t];
  float out;
  if (y == -1) out = 0.f;                                            // no target here
  else if (!rx_row_ok(y, a.V, err)) out = __builtin_nanf("");
  else out = y < n ? lp_of(r, lp_elem(l + y)) : LP_NINF;
  a.logprob[row * a.T + t] = out;
}
__device__ __forceinline__ void lp_write_top(const rx_logprob_args& a, const LpRow& r, int64_t row, int i, uint64_t key) {
  a.top_index[row * a.k + i] = key ? (int64_t)lp_key_col(key) : -1;
  a.top_logprob[row * a.k + i] = key ? lp_of(r, lp_key_value(key)) : LP_NINF;
}

// ---------------------------------------------------------------- narrow rows: G lanes per row, PER scores per lane
template <typename T, int G, int PER, bool TOP>
__global__ void __launch_bounds__(RX_BLOCK)
lp_small_kernel(rx_logprob_args a, int32_t* err) {
  __shared__ uint64_t tops[TOP ? RX_BLOCK / 64 : 1][TOP ? 128 : 1];
  const int sub = threadIdx.x & (G - 1);
  const int64_t row = (int64_t)blockIdx.x * (RX_BLOCK / G) + threadIdx.x / G;
  if (G == 64 && row >= a.R) return;             // whole wavefronts leave
  const bool on = row < a.R;
  const T* l = (const T*)a.logits + (on ? row : 0) * a.ld;
  const int32_t n = on ? lp_live(a, row) : 0;
  float v[PER], m = LP_NINF;
#pragma unroll
  for (int q = 0; q < PER; ++q) {
    const int c = q * G + sub;
    v[q] = c < n ? lp_elem(l + c) : LP_NINF;
    m = fmaxf(m, v[q]);
  }
  m = lp_max<G>(m);
  const float ref = m == LP_NINF ? 0.f : m;
  float s = 0.f, t = 0.f;
#pragma unroll
  for (int q = 0; q < PER; ++q) {
    const float d = (v[q] - ref) * LP_L2E, e = lp_exp2(d);
    s += e;
    t = fmaf(e, fmaxf(d, -1e4f), t);             // a masked score: e = 0 times a finite number
  }
  s = lp_sum<G>(s);
  t = lp_sum<G>(t);
  const LpRow r = lp_finish(m, s, t);
  if (on && sub == 0) lp_write_row(a, r, row);
  if (on)
    for (int q = sub; q < a.T; q += G) lp_write_target<T>(a, r, l, n, row, q, err);
  if constexpr (TOP) {
    // A round takes the largest score left and its lowest column: about 15 + 3 PER instructions, against 400 for sorting
    // and merging 64 keys.
    if (a.k * (15 + 3 * PER) <= 400 * PER) {
      uint64_t mine = 0;
      for (int j = 0; j < a.k; ++j) {
        float best = v[0];
#pragma unroll
        for (int q = 1; q < PER; ++q) best = lp_max3(best, v[q], v[q]);
        best = lp_max<64>(best);
        if (!(best > LP_NINF)) break;
        int32_t col = -1;
#pragma unroll
        for (int q = 0; q < PER; ++q) {
          const uint64_t at = __ballot(v[q] == best);
          if (col < 0 && at) {
            const int ln = __builtin_ctzll(at);
            col = q * 64 + ln;
            if (rx_lane() == ln) v[q] = LP_NINF;
          }
        }
        if (rx_lane() == j) mine = lp_key(best, col);
      }
      if (sub < a.k) lp_write_top(a, r, row, sub, mine);
      return;
    }
    LpTop top;
    top.init(tops[threadIdx.x >> 6]);
#pragma unroll
    for (int q = 0; q < PER; ++q) {
      if (q * 64 < n) {                          // the row's (wavefront's) live columns
        if (q == 0) top.take(v[0] > LP_NINF ? lp_key(v[0], sub) : 0);
        else top.push(v[q] > top.thr, lp_key(v[q], q * 64 + sub));
        top.refresh(a.k);
      }
    }
    top.flush();
    if (sub < a.k) lp_write_top(a, r, row, sub, top.list);
  }
}

// ---------------------------------------------------------------- wide rows
struct LpAcc {
  float raw, m2, s, t;
  float lost;                  // what the last addition to s rounded away
  __device__ __forceinline__ void init() { raw = LP_NINF; m2 = -LP_FLOOR; clear(); }
  __device__ __forceinline__ void clear() { s = 0.f; t = 0.f; lost = 0.f; }
  __device__ __forceinline__ void rebase(float n) {          // move the reference up to n (log2 units)
    const float d = fmaxf(m2 - n, -1e4f), f = lp_exp2(d);    // clamped: f is 0 there, and its factor stays finite
    t = (t + s * d) * f;
    s *= f;
    lost *= f;
    m2 = n;
  }
  // s and t of N scores d log2 units from the reference: in four sums each, then with the rounding that the last addition to s
  // lost.  One by one, near-equal weights would all round the same way (4e-5 of the sum after 4000 of them).
  template <int N, typename F>
  __device__ __forceinline__ void join(F distance) {
    float a[4] = {}, b[4] = {};
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float d = distance(i), e = lp_exp2(d);
      a[i & 3] += e;
      b[i & 3] = fmaf(e, fmaxf(d, -1e4f), b[i & 3]);       // a masked score: e = 0 times a finite number
    }
    const float add = ((a[0] + a[1]) + (a[2] + a[3])) - lost, n = s + add;
    lost = (n - s) - add;
    s = n;
    t += (b[0] + b[1]) + (b[2] + b[3]);
  }
  template <int N>
  __device__ __forceinline__ float add(const float* v) {     // returns the largest of v
    float mx = lp_max3(v[0], v[1], v[2]);
#pragma unroll
    for (int i = 3; i + 1 < N; i += 2) mx = lp_max3(mx, v[i], v[i + 1]);
    mx = lp_max3(mx, v[N - 1], v[N - 1]);
    raw = lp_max3(raw, mx, mx);
    const float n2 = mx * LP_L2E;
    const bool grow = n2 > m2 + 4.f;
    if (__ballot(grow)) {
      if (grow) rebase(n2);
    }
    join<N>([&](int i) { return fmaf(v[i], LP_L2E, -m2); });
    return mx;
  }
  // rows beyond LP_BIG (e.g. masks of the type's lowest value with nothing else in the row): the same sums relative to
  // the known maximum
  template <int N>
  __device__ __forceinline__ void add_big(const float* v, float m) {
    join<N>([&](int i) { return (v[i] - m) * LP_L2E; });
  }
};

// Columns of a row as 16-byte vectors: `head` scores before the first 16-byte boundary, `nvec` vectors, the rest.
template <typename T>
__device__ __forceinline__ void lp_frame(const T* l, int32_t n, int32_t* head, int32_t* nvec) {
  const int32_t h = (int32_t)((16 - ((uintptr_t)l & 15)) & 15) / (int32_t)sizeof(T);
  *head = h < n ? h : n;
  *nvec = (n - *head) / LpVec<T>::N;
}

// Calls f(v[2 N], column of v[0]) over this wavefront's share of the columns [part of row], in ascending groups: every
// column of one call is lower than every column of the next.  v[N] .. are LP_NEXT(T) columns further on.  A call's
// 32 bytes per lane are loaded one call ahead.
#define LP_NEXT(T) (64 * LpVec<T>::N)
template <typename T, typename F>
__device__ __forceinline__ void lp_stream(const T* l, int32_t n, int split, int n_split, F f) {
  constexpr int N = LpVec<T>::N;
  int32_t head, nvec;
  lp_frame(l, n, &head, &nvec);
  const int lane = rx_lane(), wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const bool first = split == 0 && wave == 0;
  float v[2 * N];
  if (first && head) {
#pragma unroll
    for (int i = 0; i < 2 * N; ++i) v[i] = LP_NINF;
    if (lane < head) v[0] = lp_elem(l + lane);
    f(v, lane);
  }
  const int32_t chunk = (nvec + n_split - 1) / n_split;
  const int32_t lo = split * chunk < nvec ? split * chunk : nvec;
  const int32_t hi = lo + chunk < nvec ? lo + chunk : nvec;
  const lp_u4* p = reinterpret_cast<const lp_u4*>(l + head);
  lp_u4 q0 = {}, q1 = {};
  int32_t b = lo + wave * 128;
  if (b + lane < hi) q0 = p[b + lane];
  if (b + 64 + lane < hi) q1 = p[b + 64 + lane];
  for (; b < hi; b += waves * 128) {
    const int32_t c = b + waves * 128;
    lp_u4 n0 = {}, n1 = {};
    if (c + lane < hi) n0 = p[c + lane];
    if (c + 64 + lane < hi) n1 = p[c + 64 + lane];
    lp_unpack<T>(q0, v);
    lp_unpack<T>(q1, v + N);
    if (b + 128 > hi) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (b + lane >= hi) v[i] = LP_NINF;
        if (b + 64 + lane >= hi) v[N + i] = LP_NINF;
      }
    }
    f(v, head + (b + lane) * N);
    q0 = n0;
    q1 = n1;
  }
  const int32_t tail = head + nvec * N;
  if (first && tail < n) {
#pragma unroll
    for (int i = 0; i < 2 * N; ++i) v[i] = LP_NINF;
    if (lane < n - tail) v[0] = lp_elem(l + tail + lane);
    f(v, tail + lane);
  }
}

// s and t, relative to a reference d log2 units away from the new one (-inf and NaN: nothing of them is left, but for NaN)
__device__ __forceinline__ void lp_move(float d, float* s, float* t) {
  d = fmaxf(d, -1e4f);
  const float f = lp_exp2(d);
  *t = (*t + *s * d) * f;
  *s *= f;
}

template <typename T, bool TOP>
__global__ void __launch_bounds__(LP_WIDE)
lp_wide_kernel(rx_logprob_args a, LpPart* parts, uint64_t* lists, int n_split, int32_t* err) {
  constexpr int N = LpVec<T>::N, W = LP_WIDE / 64;
  __shared__ float top_of[W];
  __shared__ float2 sums[W];
  __shared__ uint64_t tops[TOP ? W : 1][TOP ? 128 : 1];
  const int64_t row = blockIdx.x / n_split;
  const int split = blockIdx.x % n_split;
  const int wave = threadIdx.x >> 6, lane = rx_lane();
  const T* l = (const T*)a.logits + row * a.ld;
  const int32_t n = lp_live(a, row);
  LpAcc acc;
  acc.init();
  LpTop top;
  if constexpr (TOP) top.init(tops[wave]);
  lp_stream<T>(l, n, split, n_split, [&](const float* v, int32_t col) {
    const float mx = acc.add<2 * N>(v);
    if constexpr (TOP) {
      if (__ballot(mx > top.thr)) {
        // no list yet: k lanes hold a score that large, so only scores from the k-th largest lane maximum up can be in it
        float lim = top.thr;
        if (lim == LP_NINF) {
          const uint64_t kth = lp_lane64(lp_sort_up(mx > LP_NINF ? lp_key(mx, 0) : 0), 64 - a.k);
          if (kth) lim = lp_below(lp_key_value(kth));
        }
#pragma unroll
        for (int i = 0; i < 2 * N; ++i) top.push(v[i] > lim, lp_key(v[i], col + (i < N ? i : LP_NEXT(T) + i - N)));
        top.refresh(a.k);
      }
    }
  });
  // the largest score of the workgroup is its reference, and decides, uniformly, whether the sums have to be taken again
  float raw = lp_max<64>(acc.raw);
  if (lane == 0) top_of[wave] = raw;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < W; ++w) raw = fmaxf(raw, top_of[w]);
  if (fabsf(raw) > LP_BIG && fabsf(raw) < __builtin_inff()) {
    acc.clear();
    lp_stream<T>(l, n, split, n_split, [&](const float* v, int32_t) { acc.add_big<2 * N>(v, raw); });
  } else {
    lp_move(-fmaf(raw == LP_NINF ? 0.f : raw, LP_L2E, -acc.m2), &acc.s, &acc.t);
  }
  LpPart p = {raw, lp_sum<64>(acc.s), lp_sum<64>(acc.t), 0.f};
  if (lane == 0) sums[wave] = make_float2(p.s, p.t);
  if constexpr (TOP) {
    top.flush();
    tops[wave][lane] = top.list;
  }
  __syncthreads();
  p.s = p.t = 0.f;
#pragma unroll
  for (int w = 0; w < W; ++w) { p.s += sums[w].x; p.t += sums[w].y; }
  if constexpr (TOP) {
    if (wave == 0)
      for (int w = 1; w < W; ++w) top.list = lp_merge(top.list, tops[w][63 - lane]);
  }
  if (n_split > 1) {
    if (threadIdx.x == 0) parts[blockIdx.x] = p;
    if constexpr (TOP) {
      if (wave == 0 && lane < a.k) lists[(int64_t)blockIdx.x * a.k + lane] = top.list;
    }
    return;
  }
  const LpRow r = lp_finish(p.raw, p.s, p.t);
  if (threadIdx.x == 0) lp_write_row(a, r, row);
  for (int t = threadIdx.x; t < a.T; t += LP_WIDE) lp_write_target<T>(a, r, l, n, row, t, err);
  if constexpr (TOP) {
    if (wave == 0 && lane < a.k) lp_write_top(a, r, row, lane, top.list);
  }
}

// One workgroup per row joins the splits.  The k-th largest of the lists' first keys bounds the row's k-th key from
// below (k lists have a key at least that large), which leaves about k of the n_split k candidates to be merged.
template <typename T, bool TOP>
__global__ void __launch_bounds__(RX_BLOCK)
lp_join_kernel(rx_logprob_args a, const LpPart* parts, const uint64_t* lists, int n_split, int32_t* err) {
  constexpr int W = RX_BLOCK / 64;
  __shared__ float top_of[W];
  __shared__ float2 sums[W];
  __shared__ uint64_t heads[W][64];
  __shared__ uint64_t tops[TOP ? W : 1][TOP ? 128 : 1];
  const int64_t row = blockIdx.x;
  const int wave = threadIdx.x >> 6, lane = rx_lane();
  const T* l = (const T*)a.logits + row * a.ld;
  const int32_t n = lp_live(a, row);
  LpPart p = {LP_NINF, 0.f, 0.f, 0.f};
  if ((int)threadIdx.x < n_split) p = parts[row * n_split + threadIdx.x];
  float raw = lp_max<64>(p.raw);
  if (lane == 0) top_of[wave] = raw;
  if constexpr (TOP) {
    heads[wave][lane] = lp_sort_up((int)threadIdx.x < n_split ? lists[(row * n_split + threadIdx.x) * a.k] : 0);
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < W; ++w) raw = fmaxf(raw, top_of[w]);
  lp_move((p.raw - raw) * LP_L2E, &p.s, &p.t);
  p.s = lp_sum<64>(p.s);
  p.t = lp_sum<64>(p.t);
  if (lane == 0) sums[wave] = make_float2(p.s, p.t);
  __syncthreads();
  p.s = p.t = 0.f;
#pragma unroll
  for (int w = 0; w < W; ++w) { p.s += sums[w].x; p.t += sums[w].y; }
  const LpRow r = lp_finish(raw, p.s, p.t);
  if (threadIdx.x == 0) lp_write_row(a, r, row);
  for (int t = threadIdx.x; t < a.T; t += RX_BLOCK) lp_write_target<T>(a, r, l, n, row, t, err);
  if constexpr (TOP) {
    uint64_t best = heads[0][63 - lane];
    for (int w = 1; w < W; ++w) best = lp_merge(best, heads[w][lane]);
    const uint64_t th = lp_lane64(best, a.k - 1);            // 0 while there are fewer than k lists
    LpTop top;
    top.init(tops[wave]);
    // a lane per list, which is sorted: down to the first key below the bound
    const uint64_t* mine = lists + (row * n_split + threadIdx.x) * (int64_t)a.k;
    bool more = (int)threadIdx.x < n_split;
    for (int j = 0; j < a.k && __ballot(more); ++j) {
      const uint64_t key = more ? mine[j] : 0;
      more = key != 0 && key >= th;
      top.push(more, key);
    }
    top.flush();
    tops[wave][lane] = top.list;
    __syncthreads();
    if (wave == 0) {
      for (int w = 1; w < W; ++w) top.list = lp_merge(top.list, tops[w][63 - lane]);
      if (lane < a.k) lp_write_top(a, r, row, lane, top.list);
    }
  }
}

// ---------------------------------------------------------------- gradient
// dl = p (A - g_H log p),  A = g_lse - sum_t g_t - g_H H, and the targets' own share on top.  A target that carries no
// probability (-1, a masked score, a column past the row's end) takes no part; a row with nothing left gets zeros.
struct LpGrad {
  float ref, l2s, A, gh2;      // gh2 = g_H ln 2: log p is held in log2 units
  bool dead;
  __device__ __forceinline__ float of(float l) const {
    const float d = fmaf(l - ref, LP_L2E, -l2s), p = lp_exp2(d);
    return p * fmaf(-gh2, fmaxf(d, -1e4f), A);
  }
};
template <typename T>
__device__ __forceinline__ bool lp_target_on(const rx_logprob_args& a, const T* l, int32_t n, int64_t row, int t, int64_t* y) {
  *y = a.targets[row * a.T + t];
  return *y >= 0 && *y < n && lp_elem(l + *y) != LP_NINF;
}
__device__ __forceinline__ LpGrad lp_grad_row(const rx_logprob_args& a, const float* gh, const float* gl, float gsum, int64_t row) {
  const float4 st = reinterpret_cast<const float4*>(a.stats)[row];
  LpGrad r;
  const float h = gh ? gh[row] : 0.f;
  r.ref = st.x; r.l2s = st.y;
  r.gh2 = h * LP_LN2;
  r.A = (gl ? gl[row] : 0.f) - gsum - h * st.w;
  r.dead = st.z != 0.f;
  return r;
}
// the whole gradient of target t's column: its share of the softmax and every gradient that names the column; written
// by the first target that does
template <typename T>
__device__ __forceinline__ void lp_fix_target(const rx_logprob_args& a, const LpGrad& r, const T* l, T* d, int32_t n,
                                              const float* g, int64_t row, int t, int32_t lo, int32_t hi) {
  int64_t y;
  if (r.dead || !lp_target_on(a, l, n, row, t, &y) || y < lo || y >= hi) return;
  float sum = 0.f;
  for (int u = 0; u < a.T; ++u) {
    if (a.targets[row * a.T + u] != y) continue;
    if (u < t) return;
    sum += g[row * a.T + u];
  }
  lp_put<T>(d + y, r.of(lp_elem(l + y)) + sum);
}

template <typename T, int G, int PER>
__global__ void __launch_bounds__(RX_BLOCK)
lp_bwd_small_kernel(rx_logprob_args a, const float* __restrict__ g, const float* __restrict__ gh, const float* __restrict__ gl,
                    T* __restrict__ dl, int64_t ld_d) {
  const int sub = threadIdx.x & (G - 1);
  const int64_t row = (int64_t)blockIdx.x * (RX_BLOCK / G) + threadIdx.x / G;
  if (G == 64 && row >= a.R) return;
  const bool on = row < a.R;
  const int64_t rr = on ? row : 0;
  const T* l = (const T*)a.logits + rr * a.ld;
  T* d = dl + rr * ld_d;
  const int32_t n = on ? lp_live(a, row) : 0;
  float gs = 0.f;
  if (g && on)
    for (int t = sub; t < a.T; t += G) {
      int64_t y;
      if (lp_target_on(a, l, n, row, t, &y)) gs += g[row * a.T + t];
    }
  gs = lp_sum<G>(gs);
  if (!on) return;
  const LpGrad r = lp_grad_row(a, gh, gl, gs, row);
  float v[PER];
#pragma unroll
  for (int q = 0; q < PER; ++q) {
    const int c = q * G + sub;
    v[q] = c < n && !r.dead ? r.of(lp_elem(l + c)) : 0.f;
  }
  if (g && !r.dead) {
    // every lane looks at all targets: its own columns take their gradients in ascending target order
    for (int t = 0; t < a.T; ++t) {
      int64_t y;
      if (!lp_target_on(a, l, n, row, t, &y)) continue;
      const float gt = g[row * a.T + t];
#pragma unroll
      for (int q = 0; q < PER; ++q)
        if (y == q * G + sub) v[q] += gt;
    }
  }
#pragma unroll
  for (int q = 0; q < PER; ++q)
    if (q * G + sub < a.V) lp_put<T>(d + q * G + sub, v[q]);
}

template <typename T>
__global__ void __launch_bounds__(RX_BLOCK)
lp_bwd_wide_kernel(rx_logprob_args a, const float* __restrict__ g, const float* __restrict__ gh, const float* __restrict__ gl,
                   T* __restrict__ dl, int64_t ld_d, int n_split) {
  constexpr int N = LpVec<T>::N;
  __shared__ float part[RX_BLOCK / 64];
  const int64_t row = blockIdx.x / n_split;
  const int split = blockIdx.x % n_split;
  const T* l = (const T*)a.logits + row * a.ld;
  T* d = dl + row * ld_d;
  const int32_t n = lp_live(a, row), V = (int32_t)a.V;
  float gs = 0.f;
  if (g) {
    for (int t = threadIdx.x; t < a.T; t += RX_BLOCK) {
      int64_t y;
      if (lp_target_on(a, l, n, row, t, &y)) gs += g[row * a.T + t];
    }
    gs = rx_wave_sum(gs);
    if (rx_lane() == 0) part[threadIdx.x >> 6] = gs;
    __syncthreads();
    gs = part[0] + part[1] + part[2] + part[3];
  }
  const LpGrad r = lp_grad_row(a, gh, gl, gs, row);
  // the vectors follow the stores' alignment; scores that lie differently are read one by one
  const int32_t head = min((int32_t)((16 - ((uintptr_t)d & 15)) & 15) / (int32_t)sizeof(T), V);
  const int32_t nvec = (V - head) / N;
  const bool same = ((((uintptr_t)l) ^ ((uintptr_t)d)) & 15) == 0;
  const int32_t chunk = (nvec + n_split - 1) / n_split;
  const int32_t lo = min(split * chunk, nvec), hi = min(lo + chunk, nvec);
  for (int32_t q = lo + threadIdx.x; q < hi; q += RX_BLOCK) {
    const int32_t c = head + q * N;
    float v[N];
    if (c + N <= n && !r.dead) {
      if (same) lp_unpack<T>(*reinterpret_cast<const lp_u4*>(l + c), v);
      else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = lp_elem(l + c + i);
      }
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = r.of(v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = c + i < n && !r.dead ? r.of(lp_elem(l + c + i)) : 0.f;
    }
    uint4 o;
    if constexpr (sizeof(T) == 4) {
      o = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    } else {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = (uint32_t)lp_to_bf16(v[2 * i]) | ((uint32_t)lp_to_bf16(v[2 * i + 1]) << 16);
      o = make_uint4(w[0], w[1], w[2], w[3]);
    }
    *reinterpret_cast<uint4*>(d + c) = o;
  }
  // columns outside the vectors, with the first and the last split
  const int32_t tail = head + nvec * N;
  if (split == 0 && (int)threadIdx.x < head) {
    const int c = threadIdx.x;
    lp_put<T>(d + c, c < n && !r.dead ? r.of(lp_elem(l + c)) : 0.f);
  }
  if (split == n_split - 1 && (int)threadIdx.x < V - tail) {
    const int c = tail + threadIdx.x;
    lp_put<T>(d + c, c < n && !r.dead ? r.of(lp_elem(l + c)) : 0.f);
  }
  if (!g) return;
  __syncthreads();           // the targets' columns are written again, after everything else of this split
  const int32_t c0 = split == 0 ? 0 : head + lo * N, c1 = split == n_split - 1 ? V : head + hi * N;
  for (int t = threadIdx.x; t < a.T; t += RX_BLOCK) lp_fix_target<T>(a, r, l, d, n, g, row, t, c0, c1);
}

// ---------------------------------------------------------------- host
static int lp_splits(int64_t R, int64_t V) {
  // Enough workgroups to fill the chip (4 per CU) when there are few rows, each with at least LP_SPLIT_MIN columns.
  int64_t want = rx_cdiv(1024, R > 0 ? R : 1), most = V / LP_SPLIT_MIN;
  if (want > most) want = most;
  if (want > LP_SPLIT_MAX) want = LP_SPLIT_MAX;
  return want < 1 ? 1 : (int)want;
}

static int lp_check(const rx_logprob_args* a, const char* who) {
  RX_REQUIRE(a, "%s: null argument", who);
  RX_REQUIRE(a->R >= 0 && a->V >= 1 && a->V < (1ll << 31) - 64 && a->ld >= a->V, "%s: bad shape R=%lld V=%lld ld=%lld", who,
             (long long)a->R, (long long)a->V, (long long)a->ld);
  RX_REQUIRE(a->T >= 0 && a->T <= 1024, "%s: T=%d targets per row (at most 1024)", who, a->T);
  // a launch takes fewer than 2^32 threads
  const int64_t per = a->V > LP_SMALL ? 1 : a->V <= 8 && a->k == 0 ? RX_BLOCK / 8 : RX_BLOCK / 64;
  RX_REQUIRE(a->R <= ((1ll << 24) - 1) * per / lp_splits(a->R, a->V), "%s: R=%lld rows are more than one launch takes", who, (long long)a->R);
  RX_REQUIRE(a->bf16 == 0 || a->bf16 == 1, "%s: bad element type %d", who, a->bf16);
  if (a->R == 0) return 0;
  RX_REQUIRE(a->logits && (a->T == 0 || a->targets), "%s: null argument", who);
  RX_REQUIRE(((uintptr_t)a->stats & 15) == 0, "%s: stats must be 16-byte aligned", who);
  RX_REQUIRE(((uintptr_t)a->logits & (a->bf16 ? 1 : 3)) == 0, "%s: logits are not aligned to their elements", who);
  return 0;
}

extern "C" size_t rx_logprob_workspace_bytes(int64_t R, int64_t V, int32_t k) {
  if (R <= 0 || V <= LP_SMALL || k < 0 || k > LP_TOP) return 0;
  const int n = lp_splits(R, V);
  return n > 1 ? (size_t)R * n * (sizeof(LpPart) + 8 * (size_t)k) : 0;
}

template <typename T, bool TOP>
static void lp_launch_small(const rx_logprob_args& a, int32_t* err, hipStream_t st) {
#define LP_GO(G, PER)                                                                                              \
  hipLaunchKernelGGL((lp_small_kernel<T, G, PER, TOP>), dim3((unsigned)rx_cdiv(a.R, RX_BLOCK / (G))), dim3(RX_BLOCK), 0, st, a, err)
  if constexpr (!TOP) {
    if (a.V <= 8) { LP_GO(8, 1); return; }
    if (a.V <= 32) { LP_GO(32, 1); return; }
  }
  if (a.V <= 64) LP_GO(64, 1);
  else if (a.V <= 128) LP_GO(64, 2);
  else if (a.V <= 256) LP_GO(64, 4);
  else if (a.V <= 512) LP_GO(64, 8);
  else LP_GO(64, 16);
#undef LP_GO
}

template <typename T>
static void lp_launch_fwd(const rx_logprob_args& a, void* ws, int32_t* err, hipStream_t st) {
  if (a.V <= LP_SMALL) {
    if (a.k) lp_launch_small<T, true>(a, err, st);
    else lp_launch_small<T, false>(a, err, st);
    return;
  }
  const int n = lp_splits(a.R, a.V);
  LpPart* parts = (LpPart*)ws;
  uint64_t* lists = (uint64_t*)(parts + (n > 1 ? a.R * n : 0));
  const dim3 grid((unsigned)(a.R * n)), blk(RX_BLOCK), wide(LP_WIDE);
  if (a.k) {
    hipLaunchKernelGGL((lp_wide_kernel<T, true>), grid, wide, 0, st, a, parts, lists, n, err);
    if (n > 1) hipLaunchKernelGGL((lp_join_kernel<T, true>), dim3((unsigned)a.R), blk, 0, st, a, parts, lists, n, err);
  } else {
    hipLaunchKernelGGL((lp_wide_kernel<T, false>), grid, wide, 0, st, a, parts, lists, n, err);
    if (n > 1) hipLaunchKernelGGL((lp_join_kernel<T, false>), dim3((unsigned)a.R), blk, 0, st, a, parts, lists, n, err);
  }
}

extern "C" int rx_logprob_fwd(const rx_logprob_args* args, void* ws, size_t ws_bytes, int32_t* err_flag, int device, void* stream) {
  if (lp_check(args, "rx_logprob_fwd")) return 1;
  const rx_logprob_args a = *args;
  RX_REQUIRE(a.k >= 0 && a.k <= LP_TOP, "rx_logprob_fwd: k=%d alternatives (at most %d)", a.k, LP_TOP);
  if (a.R == 0) return 0;
  RX_REQUIRE(a.lse && a.entropy && (a.T == 0 || a.logprob) && (a.k == 0 || (a.top_logprob && a.top_index)), "rx_logprob_fwd: null output");
  const size_t need = rx_logprob_workspace_bytes(a.R, a.V, a.k);
  RX_REQUIRE(need == 0 || (ws && ws_bytes >= need && ((uintptr_t)ws & 15) == 0), "rx_logprob_fwd: workspace of %zu bytes, %zu needed",
             ws_bytes, need);
  RX_GUARD_DEVICE(device);
  if (a.bf16) lp_launch_fwd<uint16_t>(a, ws, err_flag, (hipStream_t)stream);
  else lp_launch_fwd<float>(a, ws, err_flag, (hipStream_t)stream);
  RX_LAUNCH_CHECK();
  return 0;
}

template <typename T>
static void lp_launch_bwd(const rx_logprob_args& a, const float* g, const float* gh, const float* gl, T* dl, int64_t ld, hipStream_t st) {
#define LP_GO(G, PER)                                                                                                     \
  hipLaunchKernelGGL((lp_bwd_small_kernel<T, G, PER>), dim3((unsigned)rx_cdiv(a.R, RX_BLOCK / (G))), dim3(RX_BLOCK), 0, st, a, g, gh, \
                     gl, dl, ld)
  if (a.V <= 8) LP_GO(8, 1);
  else if (a.V <= 32) LP_GO(32, 1);
  else if (a.V <= 64) LP_GO(64, 1);
  else if (a.V <= 128) LP_GO(64, 2);
  else if (a.V <= 256) LP_GO(64, 4);
  else if (a.V <= 512) LP_GO(64, 8);
  else if (a.V <= LP_SMALL) LP_GO(64, 16);
  else {
    const int n = lp_splits(a.R, a.V);
    hipLaunchKernelGGL((lp_bwd_wide_kernel<T>), dim3((unsigned)(a.R * n)), dim3(RX_BLOCK), 0, st, a, g, gh, gl, dl, ld, n);
  }
#undef LP_GO
}

extern "C" int rx_logprob_bwd(const rx_logprob_args* args, const float* d_g_logprob, const float* d_g_entropy, const float* d_g_lse,
                              void* d_dlogits, int64_t ld_d, int device, void* stream) {
  if (lp_check(args, "rx_logprob_bwd")) return 1;
  const rx_logprob_args a = *args;
  RX_REQUIRE(ld_d >= a.V, "rx_logprob_bwd: row stride %lld below V=%lld", (long long)ld_d, (long long)a.V);
  if (a.R == 0) return 0;
  RX_REQUIRE(a.stats && d_dlogits && ((uintptr_t)d_dlogits & (a.bf16 ? 1 : 3)) == 0, "rx_logprob_bwd: bad gradient buffer");
  RX_GUARD_DEVICE(device);
  if (a.T == 0) d_g_logprob = nullptr;
  if (a.bf16) lp_launch_bwd<uint16_t>(a, d_g_logprob, d_g_entropy, d_g_lse, (uint16_t*)d_dlogits, ld_d, (hipStream_t)stream);
  else lp_launch_bwd<float>(a, d_g_logprob, d_g_entropy, d_g_lse, (float*)d_dlogits, ld_d, (hipStream_t)stream);
  RX_LAUNCH_CHECK();
  return 0;
}
