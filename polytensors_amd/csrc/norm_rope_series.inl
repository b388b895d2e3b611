// RMSNorm of every head of queries and keys and the rotation by position, in one pass over each.
//
// Per head row x of D elements at position pos, orders 0..K:
//   n = x (*) r,  r = (mean(x (*) x) + eps)^(-1/2)   (norm_series.inl's root series)
//   y = R(pos) (w (*) n)
// w an ordinary weight, a series or none. R turns pair j < rotary / 2 by the angle whose cosine and sine
// are table[pos][j]: (a, b) -> (a cos - b sin, b cos + a sin). The pairs are the elements j and
// j + rotary / 2 of the head, or its neighbours 2 j and 2 j + 1 where interleaved; elements from `rotary`
// on are not turned. R and w are the same for every order, so each acts on the orders singly (a series w
// by a Cauchy product).
// Rows are read by their strides from [batch, length, heads, D] (a part of a projection's output) and
// written as [batch, heads, length, D], as attention takes them.
// A negative position marks padding: its rows are zero, and so are their gradients. One past the table
// has no angle: its rows are NaN.
//
// Gradient: with g = R^T dy, h = w (*) g, u = mean(x (*) h):
//   dx = r (*) h - (r (*) r (*) r (*) u) (*) x,   dw = sum over rows of n (*) g.
//
// G lanes (a power of two, at most a wave) share a row, 256 / G rows a block. A lane holds chunks of V
// pairs, every order of them, so that a rotation needs no exchange between lanes: two V-vectors an order,
// at the two halves of the rotated part or of the head. The row sums go over the G lanes in registers.
//
// HBM bounds the forward: 4 x 2048 tokens of 16 + 16 heads of 128, bfloat16, degree 4 132 us, 5.1 TB/s (a stream over the same
// buffers 113); 2 x 2048 of 32 + 8 heads, degree 3 59 us (57); 3 x 1001 of 24 heads of 80, float32, degree 3 34 us (33).
// The gradient of the second takes 99 us and 4 for the weights' sums, 5.1 TB/s (80): its vector instructions, 78 a pair and
// order, alone are about 83 us of issue; that of the third 64 us (49), at two or three waves a SIMD.
#pragma once

#include "norm_rope_series.h"
#include "norm_series.inl"
#include "series_math.h"

namespace pt {

constexpr int kRopeThreads = 256;

// V elements at any element's address. Loads are cached: a row's two vectors an order lie in one or two cache lines, and
// neighbouring rows share them (non-temporal loads: 2 x 2048 tokens of 32 + 8 heads of 128, degree 3, bfloat16 70 us, 60 with these;
// 3 x 1001 tokens of 24 heads of 80, float32, and its gradient 52 and 80 us, 47 and 63). The output's stores are
// non-temporal where neighbouring lanes' vectors fill whole 128-byte lines (the first of these 74 us cached, 60 so), cached
// where they leave parts of lines to the next instruction (the second: 47 us non-temporal, 32 so); the gradient's rows
// follow one another in memory, and its stores are non-temporal (2 x 2048 tokens of 16 + 16 heads of 128, degree 1, float32: 82
// us cached, 69 so).
template <int BYTES>
struct RopeWords {
  typedef uint32_t type __attribute__((ext_vector_type(BYTES / 4)));
  typedef type any __attribute__((aligned(2)));
};
template <>
struct RopeWords<4> {
  typedef uint32_t type;
  typedef type any __attribute__((aligned(2)));
};
template <>
struct RopeWords<2> {
  typedef uint16_t type;
  typedef type any;
};
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> rope_load(const T* p) {
  if constexpr (V == 1) {
    Vec<T, 1> r;
    r.v[0] = *p;
    return r;
  } else {
    const typename RopeWords<sizeof(T) * V>::type w = *reinterpret_cast<const typename RopeWords<sizeof(T) * V>::any*>(p);
    return __builtin_bit_cast(Vec<T, V>, w);
  }
}
template <bool STREAM, typename T, int V>
__device__ __forceinline__ void rope_store(T* p, const Vec<T, V>& v) {
  if constexpr (V == 1) {
    *p = v.v[0];
  } else {
    using W = RopeWords<sizeof(T) * V>;
    const typename W::type w = __builtin_bit_cast(typename W::type, v);
    if constexpr (STREAM) __builtin_nontemporal_store(w, reinterpret_cast<typename W::any*>(p));
    else *reinterpret_cast<typename W::any*>(p) = w;
  }
}
// Element e (a bfloat16 vector is read by words, which a single element has not).
template <typename T, int V>
__device__ __forceinline__ typename AccOf<T>::type rope_get(const Vec<T, V>& v, int e) {
  if constexpr (V == 1) return to_acc(v.v[0]);
  else return vec_get(v, e);
}
// The vector where it is kept, else zeros: a choice of words (assigning an empty vector under a branch leaves the
// series in scratch memory).
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> rope_kept(const Vec<T, V>& v, bool keep) {
  using W = typename RopeWords<sizeof(T) * V>::type;
  const W w = __builtin_bit_cast(W, v);
  return __builtin_bit_cast(Vec<T, V>, keep ? w : W(0));
}

// Sum over the G lanes of a row (G a power of two, uniform): every lane of the row ends with the same bits.
__device__ __forceinline__ float group_sum(float x, int G) {
  if (G >= 2) x += dpp_mov<0xB1>(x);
  if (G >= 4) x += dpp_mov<0x4E>(x);
  if (G >= 8) x += dpp_mov<0x141>(x);
  if (G >= 16) x += dpp_mov<0x140>(x);
  if (G >= 32) x += __shfl_xor(x, 16, kWave);
  if (G >= 64) x += __shfl_xor(x, 32, kWave);
  return x;
}
__device__ __forceinline__ double group_sum(double x, int G) {
  for (int off = 1; off < G; off <<= 1) x += __shfl_xor(x, off, kWave);
  return x;
}

// n / d for n below 2^31 as (n m) / 2^(31 + s), s = ceil(log2 d), m = ceil(2^(31 + s) / d): m d - 2^(31 + s) < d <= 2^s, so that
// the error n (m d - 2^(31 + s)) / (d 2^(31 + s)) stays below 1 / d. (Two divisions by a variable were a fifth of a row's
// instructions.)
struct RopeDivisor {
  uint32_t d, m, shift;
};
static RopeDivisor rope_divisor(uint32_t d) {
  uint32_t s = 0;
  while ((1ull << s) < d) ++s;
  return {d, static_cast<uint32_t>(((1ull << (31 + s)) + d - 1) / d), 31 + s};
}
__device__ __forceinline__ uint32_t operator/(uint32_t n, const RopeDivisor& by) {
  return static_cast<uint32_t>((static_cast<uint64_t>(n) * by.m) >> by.shift);
}

template <typename T>
struct RopeOperand {
  CPtrs<T> x, w, g;
  MPtrs<T> y;                  // the output, or dx
  int64_t stride_b, stride_l, stride_h;
  RopeDivisor heads;
  uint32_t rows, blocks;
  int w_orders;
  bool want_dw;
  typename AccOf<T>::type* partial;   // [blocks][orders summed][D]
};

template <typename T>
struct RopeKernelArgs {
  RopeOperand<T> op[2];
  RopeDivisor length;
  int head_dim, rotary, lanes;
  bool interleaved;
  const typename AccOf<T>::type* cos;
  const typename AccOf<T>::type* sin;
  int64_t table_rows;
  const int64_t* positions;
  int64_t position_batch_stride;
  typename AccOf<T>::type eps;
};

// Where a lane's chunk of V pairs lies in a head: its two V-vectors, the table columns of their pairs, and whether the
// vectors exist (the last element of an odd head has no partner; V = 1 there). Pairs of elements half the rotated part apart take
// an element of either vector, column after column from `lo_pair`. Neighbours (V > 1) lie within a vector, V / 2 pairs each;
// the second vector is half a head away all the same, so that neighbouring lanes' vectors are side by side.
struct RopeChunk {
  int lo, hi, lo_pair, hi_pair;
  bool has_lo, has_hi;
};
template <int V>
__device__ __forceinline__ RopeChunk rope_chunk(int chunk, int head_dim, int rotary, bool interleaved) {
  RopeChunk c;
  const int pair = chunk * V;
  c.lo_pair = c.hi_pair = pair;
  c.has_lo = 2 * pair < head_dim;
  if (interleaved && V > 1) {
    c.lo = pair;
    c.hi = pair + head_dim / 2;
    c.lo_pair = c.lo / 2;
    c.hi_pair = c.hi / 2;
  } else if (interleaved) {
    c.lo = 2 * pair;
    c.hi = c.lo + 1;
  } else if (pair < rotary / 2) {
    c.lo = pair;
    c.hi = pair + rotary / 2;
  } else {
    c.lo = rotary + pair - rotary / 2;
    c.hi = c.lo + (head_dim - rotary + 1) / 2;
  }
  c.has_hi = c.has_lo && c.hi < head_dim;
  if (!c.has_lo) c.lo = c.lo_pair = c.hi_pair = 0;   // (addresses stay inside the row and the table; the values are not used)
  if (!c.has_hi) c.hi = c.lo;
  return c;
}

// A row's place: where it is read and written, and its position in the tables.
struct RopeRow {
  int64_t in, out, pos;
  bool live;
};
template <typename T>
__device__ __forceinline__ RopeRow rope_row(const RopeKernelArgs<T>& a, uint32_t row, uint32_t rows,
                                            const RopeDivisor& heads, int64_t sb, int64_t sl, int64_t sh) {
  RopeRow r;
  r.live = row < rows;
  if (!r.live) row = rows - 1;
  const uint32_t bl = row / heads, h = row - bl * heads.d, b = bl / a.length, l = bl - b * a.length.d;
  r.in = b * sb + l * sl + h * sh;
  r.out = ((static_cast<int64_t>(b) * heads.d + h) * a.length.d + l) * a.head_dim;
  r.pos = a.positions != nullptr ? a.positions[b * a.position_batch_stride + l] : static_cast<int64_t>(l);
  return r;
}

// Cosines and sines of N neighbouring pairs from `pair` on (1 and 0 behind the rotated part), NaN past the table.
template <typename A, int N>
__device__ __forceinline__ void rope_columns(const A* cos, const A* sin, int64_t table_rows, int rotary, int64_t pos, int pair,
                                             A* c, A* s) {
  const int half = rotary / 2;
  const bool inside = pos >= 0 && pos < table_rows;
  const int64_t at = inside ? pos * half : 0;
  if (inside && pair + N <= half) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      c[e] = cos[at + pair + e];
      s[e] = sin[at + pair + e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const bool turned = inside && pair + e < half;
      c[e] = turned ? cos[at + pair + e] : A(1);
      s[e] = turned ? sin[at + pair + e] : A(0);
    }
    if (pos >= table_rows) {
#pragma unroll
      for (int e = 0; e < N; ++e) c[e] = __builtin_nan("");
    }
  }
}

// Those of a chunk's pairs, in the order of RopeUnit.
template <int V, bool NEXT, typename T>
__device__ __forceinline__ void rope_angles(const RopeKernelArgs<T>& a, int64_t pos, const RopeChunk& ch,
                                            typename AccOf<T>::type (&c)[V], typename AccOf<T>::type (&s)[V]) {
  using A = typename AccOf<T>::type;
  if constexpr (V > 1 && NEXT) {
    rope_columns<A, V / 2>(a.cos, a.sin, a.table_rows, a.rotary, pos, ch.lo_pair, &c[0], &s[0]);
    rope_columns<A, V / 2>(a.cos, a.sin, a.table_rows, a.rotary, pos, ch.hi_pair, &c[V / 2], &s[V / 2]);
  } else {
    rope_columns<A, V>(a.cos, a.sin, a.table_rows, a.rotary, pos, ch.lo_pair, &c[0], &s[0]);
  }
}

// Every order of a lane's chunk in its storage type (half the registers of float values for 16-bit types): element i
// is the first vector's below V, the second's from there.
template <typename T, int K, int V>
struct RopeSeries {
  using A = typename AccOf<T>::type;
  Vec<T, V> half[2][K + 1];   // (indexed by i / V: a choice between two members puts them in scratch memory)

  __device__ __forceinline__ void read(const T* const (&p)[K + 1], int64_t at, const RopeChunk& ch) {
#pragma unroll
    for (int k = 0; k <= K; ++k) {
      half[0][k] = rope_load<T, V>(p[k] + at + ch.lo);
      half[1][k] = rope_load<T, V>(p[k] + at + ch.hi);
    }
  }
  // Zero where the lane has no element, and in rows that are not used.
  __device__ __forceinline__ void mask(const RopeChunk& ch, bool use) {
    if (use && ch.has_hi) return;
#pragma unroll
    for (int k = 0; k <= K; ++k) {
      half[0][k] = rope_kept(half[0][k], use && ch.has_lo);
      half[1][k] = rope_kept(half[1][k], false);
    }
  }
  __device__ __forceinline__ A get(int k, int i) const { return rope_get(half[i / V][k], i % V); }
  // Elements i and i + 1 of one vector (element i alone where a vector has one).
  __device__ __forceinline__ void put(int k, int i, A a, A b) {
    if constexpr (V == 1) half[i][k].v[0] = from_acc<T>(a);
    else vec_put2(half[i / V][k], i % V, a, b);
  }
  template <bool STREAM>
  __device__ __forceinline__ void write(T* const (&p)[K + 1], int64_t at, const RopeChunk& ch) const {
#pragma unroll
    for (int k = 0; k <= K; ++k) {
      if (ch.has_lo) rope_store<STREAM>(p[k] + at + ch.lo, half[0][k]);
      if (ch.has_hi) rope_store<STREAM>(p[k] + at + ch.hi, half[1][k]);
    }
  }
  // Sums of the elements of x (*) x.
  __device__ __forceinline__ void squares(A (&s)[K + 1]) const {
#pragma unroll
    for (int i = 0; i < 2 * V; ++i) {
      A c[K + 1];
#pragma unroll
      for (int k = 0; k <= K; ++k) c[k] = get(k, i);
#pragma unroll
      for (int k = 0; k <= K; ++k) s[k] += cauchy_square<A, K>(c, k);
    }
  }
};

// A chunk is worked on by units of two pairs (one where a vector has one element): the unit's elements, in the order
// that puts them back two at a time, and its pairs among them. NEXT: a pair's elements are neighbours.
template <int V, bool NEXT>
struct RopeUnit {
  static constexpr int kPairs = V == 1 ? 1 : 2, kElements = 2 * kPairs, kUnits = V / kPairs;
  static __device__ __forceinline__ constexpr int element(int unit, int i) {
    if (V == 1) return i;
    if (NEXT) return 4 * unit + i;
    return i < 2 ? 2 * unit + i : V + 2 * unit + i - 2;
  }
  static __device__ __forceinline__ constexpr int first(int pair) { return V > 1 && NEXT ? 2 * pair : pair; }
  static __device__ __forceinline__ constexpr int second(int pair) { return V > 1 && NEXT ? 2 * pair + 1 : kPairs + pair; }
};

// (a, b) -> (a c - b s, b c + a s) on the pairs of a unit, every order; BACK: by the opposite angle.
template <int K, int V, bool NEXT, bool BACK, typename A, int N>
__device__ __forceinline__ void rope_turn(A (&v)[N][K + 1], const A (&c)[V], const A (&s)[V], int unit) {
  using U = RopeUnit<V, NEXT>;
#pragma unroll
  for (int p = 0; p < U::kPairs; ++p) {
    const A co = c[unit * U::kPairs + p], si = BACK ? -s[unit * U::kPairs + p] : s[unit * U::kPairs + p];
#pragma unroll
    for (int k = 0; k <= K; ++k) {
      A &a = v[U::first(p)][k], &b = v[U::second(p)][k];
      const A x = a;
      a = x * co - b * si;
      b = b * co + x * si;
    }
  }
}

// An ordinary weight, or the constant order of a series of them, for a lane's chunk (ones without a weight).
template <typename T, int V>
struct RopeWeight {
  Vec<T, V> half[2];
  __device__ __forceinline__ void read(const T* w, int w_orders, const RopeChunk& ch) {
    if (w_orders > 0) {
      half[0] = rope_load<T, V>(w + ch.lo);
      half[1] = rope_load<T, V>(w + ch.hi);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) half[0].v[e] = from_acc<T>(typename AccOf<T>::type(1));
      half[1] = half[0];
    }
  }
  __device__ __forceinline__ typename AccOf<T>::type get(int i) const { return rope_get(half[i / V], i % V); }
};

// v <- w (*) v for element i of a chunk (the higher orders of a series weight read where they are used).
template <typename T, int K, int V>
__device__ __forceinline__ void rope_weigh(const RopeWeight<T, V>& w, const T* const (&w_p)[K + 1], int w_orders, const RopeChunk& ch,
                                           int i, typename AccOf<T>::type (&v)[K + 1]) {
  using A = typename AccOf<T>::type;
  const A w0 = w.get(i);
  if (K > 0 && w_orders > 1) {
    const int at = i < V ? ch.lo + i : ch.hi + i - V;
    A ws[K + 1];
    ws[0] = w0;
#pragma unroll
    for (int k = 1; k <= K; ++k) ws[k] = to_acc(w_p[k][at]);
#pragma unroll
    for (int k = K; k >= 0; --k) {
      A s = v[k] * w0;
#pragma unroll
      for (int j = 0; j < k; ++j) s = fma(v[j], ws[k - j], s);
      v[k] = s;
    }
  } else {
#pragma unroll
    for (int k = 0; k <= K; ++k) v[k] *= w0;
  }
}

// x (*) r of one element.
template <typename A, int K>
__device__ __forceinline__ void rope_product(const A (&x)[K + 1], const A (&r)[K + 1], A (&n)[K + 1]) {
#pragma unroll
  for (int k = 0; k <= K; ++k) {
    A v = x[k] * r[0];
#pragma unroll
    for (int j = 0; j < k; ++j) v = fma(x[j], r[k - j], v);
    n[k] = v;
  }
}

#define PT_ROPE_PICK(field) (second ? a.op[1].field : a.op[0].field)

template <typename T, int K, int V, int C, bool NEXT, bool STREAM>
__global__ __launch_bounds__(kRopeThreads) void norm_rope_series_kernel(const RopeKernelArgs<T> a) {
  using A = typename AccOf<T>::type;
  using U = RopeUnit<V, NEXT>;
  const bool second = blockIdx.x >= a.op[0].blocks;
  const uint32_t block = second ? blockIdx.x - a.op[0].blocks : blockIdx.x;
  const T* x_p[K + 1];
  const T* w_p[K + 1];
  T* y_p[K + 1];
#pragma unroll
  for (int k = 0; k <= K; ++k) {
    x_p[k] = PT_ROPE_PICK(x.p[k]);
    w_p[k] = PT_ROPE_PICK(w.p[k]);
    y_p[k] = PT_ROPE_PICK(y.p[k]);
  }
  const int G = a.lanes, lane = threadIdx.x & (G - 1), w_orders = PT_ROPE_PICK(w_orders);
  const uint32_t rows = PT_ROPE_PICK(rows);
  const RopeDivisor heads{PT_ROPE_PICK(heads.d), PT_ROPE_PICK(heads.m), PT_ROPE_PICK(heads.shift)};
  const RopeRow row = rope_row(a, block * (kRopeThreads / G) + threadIdx.x / G, rows, heads, PT_ROPE_PICK(stride_b),
                               PT_ROPE_PICK(stride_l), PT_ROPE_PICK(stride_h));
  const bool use = row.pos >= 0;
  // every load of the row before the first sum: the weight and the angles arrive while it is formed
  RopeChunk ch[C];
  RopeSeries<T, K, V> x[C];
  RopeWeight<T, V> w[C];
  A c[C][V], sn[C][V];
#pragma unroll
  for (int i = 0; i < C; ++i) {
    ch[i] = rope_chunk<V>(lane + i * G, a.head_dim, a.rotary, a.interleaved);
    x[i].read(x_p, row.in, ch[i]);
    w[i].read(w_p[0], w_orders, ch[i]);
  }
#pragma unroll
  for (int i = 0; i < C; ++i)
    rope_angles<V, NEXT>(a, row.pos, ch[i], c[i], sn[i]);
  A s[K + 1], r[K + 1];
#pragma unroll
  for (int k = 0; k <= K; ++k) s[k] = A(0);
#pragma unroll
  for (int i = 0; i < C; ++i) {
    x[i].mask(ch[i], use);
    x[i].squares(s);
  }
#pragma unroll
  for (int k = 0; k <= K; ++k) s[k] = group_sum(s[k], G);
  rsqrt_series<A, K>(s, A(1) / A(a.head_dim), a.eps, r);
#pragma unroll
  for (int i = 0; i < C; ++i) {
#pragma unroll
    for (int u = 0; u < U::kUnits; ++u) {
      A v[U::kElements][K + 1];
#pragma unroll
      for (int e = 0; e < U::kElements; ++e) {
        const int at = U::element(u, e);
        A t[K + 1];
#pragma unroll
        for (int k = 0; k <= K; ++k) t[k] = x[i].get(k, at);
        rope_product<A, K>(t, r, v[e]);
        rope_weigh<T, K, V>(w[i], w_p, w_orders, ch[i], at, v[e]);
      }
      rope_turn<K, V, NEXT, false>(v, c[i], sn[i], u);
#pragma unroll
      for (int e = 0; e < U::kElements; e += V == 1 ? 1 : 2)
#pragma unroll
        for (int k = 0; k <= K; ++k) x[i].put(k, U::element(u, e), v[e][k], v[V == 1 ? e : e + 1][k]);
    }
    x[i].mask(ch[i], use);   // padding: zero, whatever the weight is
    if (row.live) x[i].template write<STREAM>(y_p, row.out, ch[i]);
  }
}

// SUM: weight gradients are summed, of order K alone (1: an ordinary weight under the reversed cotangents
// of coefficient gradients) or of every order (2); 0: none. Then a block takes every blocks-th group of
// rows and leaves its sums as a row of `partial`, which rope_weight_reduce_kernel adds in a fixed order.
// The cotangent is turned back twice, before the sums and after them, rather than kept in the arithmetic type.
template <typename T, int K, int V, int C, bool NEXT, int SUM>
__global__ __launch_bounds__(kRopeThreads) void norm_rope_series_bwd_kernel(const RopeKernelArgs<T> a) {
  using A = typename AccOf<T>::type;
  using U = RopeUnit<V, NEXT>;
  constexpr int kSums = SUM == 0 ? 0 : SUM == 1 ? 1 : K + 1;
  const bool second = blockIdx.x >= a.op[0].blocks;
  const uint32_t block = second ? blockIdx.x - a.op[0].blocks : blockIdx.x;
  const T* x_p[K + 1];
  const T* g_p[K + 1];
  const T* w_p[K + 1];
  T* dx_p[K + 1];
#pragma unroll
  for (int k = 0; k <= K; ++k) {
    x_p[k] = PT_ROPE_PICK(x.p[k]);
    g_p[k] = PT_ROPE_PICK(g.p[k]);
    w_p[k] = PT_ROPE_PICK(w.p[k]);
    dx_p[k] = PT_ROPE_PICK(y.p[k]);
  }
  const int G = a.lanes, lane = threadIdx.x & (G - 1), w_orders = PT_ROPE_PICK(w_orders);
  const uint32_t rows = PT_ROPE_PICK(rows), per_block = kRopeThreads / G;
  const RopeDivisor heads{PT_ROPE_PICK(heads.d), PT_ROPE_PICK(heads.m), PT_ROPE_PICK(heads.shift)};
  const uint32_t blocks = PT_ROPE_PICK(blocks);
  RopeChunk ch[C];
  RopeWeight<T, V> w[C];
#pragma unroll
  for (int i = 0; i < C; ++i) {
    ch[i] = rope_chunk<V>(lane + i * G, a.head_dim, a.rotary, a.interleaved);
    w[i].read(w_p[0], w_orders, ch[i]);
  }
  A dw[kSums > 0 ? kSums : 1][C][2 * V];
  if constexpr (SUM > 0) {
#pragma unroll
    for (int q = 0; q < kSums; ++q)
#pragma unroll
      for (int i = 0; i < C; ++i)
#pragma unroll
        for (int e = 0; e < 2 * V; ++e) dw[q][i][e] = A(0);
  }
  for (uint32_t group = block; static_cast<uint64_t>(group) * per_block < rows; group += blocks) {
    const uint32_t index = group * per_block + threadIdx.x / G;
    const RopeRow row =
        rope_row(a, index, rows, heads, PT_ROPE_PICK(stride_b), PT_ROPE_PICK(stride_l), PT_ROPE_PICK(stride_h));
    const bool use = row.pos >= 0 && row.live;
    RopeSeries<T, K, V> x[C], g[C];
    A c[C][V], sn[C][V];
#pragma unroll
    for (int i = 0; i < C; ++i) {
      x[i].read(x_p, row.in, ch[i]);
      g[i].read(g_p, row.out, ch[i]);
    }
#pragma unroll
    for (int i = 0; i < C; ++i)
      rope_angles<V, NEXT>(a, row.pos, ch[i], c[i], sn[i]);
    A s[K + 1], u[K + 1], r[K + 1];
#pragma unroll
    for (int k = 0; k <= K; ++k) s[k] = u[k] = A(0);
#pragma unroll
    for (int i = 0; i < C; ++i) {
      x[i].mask(ch[i], use);
      g[i].mask(ch[i], use);
      x[i].squares(s);
    }
#pragma unroll
    for (int k = 0; k <= K; ++k) s[k] = group_sum(s[k], G);
    rsqrt_series<A, K>(s, A(1) / A(a.head_dim), a.eps, r);
#pragma unroll
    for (int k = 0; k <= K; ++k) r[k] = use ? r[k] : A(0);
    // of a unit x (*) R^T dy, which gives both sums: w (*) it summed over the row is mean(x (*) h) D, r (*) it the
    // weight's gradient
#pragma unroll
    for (int i = 0; i < C; ++i) {
#pragma unroll
      for (int t = 0; t < U::kUnits; ++t) {
        A h[U::kElements][K + 1];
#pragma unroll
        for (int e = 0; e < U::kElements; ++e)
#pragma unroll
          for (int k = 0; k <= K; ++k) h[e][k] = g[i].get(k, U::element(t, e));
        rope_turn<K, V, NEXT, true>(h, c[i], sn[i], t);
#pragma unroll
        for (int e = 0; e < U::kElements; ++e) {
          const int at = U::element(t, e);
          A v[K + 1], xg[K + 1];
#pragma unroll
          for (int k = 0; k <= K; ++k) v[k] = x[i].get(k, at);
          rope_product<A, K>(v, h[e], xg);
          if constexpr (SUM > 0) {
#pragma unroll
            for (int q = 0; q < kSums; ++q) {
              const int order = SUM == 1 ? K : q;
#pragma unroll
              for (int j = 0; j <= order; ++j) dw[q][i][at] = fma(r[j], xg[order - j], dw[q][i][at]);
            }
          }
          if (K == 0 || w_orders <= 1) {
            const A w0 = w[i].get(at);
#pragma unroll
            for (int k = 0; k <= K; ++k) u[k] = fma(w0, xg[k], u[k]);
          } else {
            rope_weigh<T, K, V>(w[i], w_p, w_orders, ch[i], at, xg);
#pragma unroll
            for (int k = 0; k <= K; ++k) u[k] += xg[k];
          }
        }
      }
    }
#pragma unroll
    for (int k = 0; k <= K; ++k) u[k] = group_sum(u[k], G) * (A(1) / A(a.head_dim));
    A r2[K + 1], r3[K + 1], c3[K + 1];
    cauchy_mul<A, K>(r, r, r2);
    cauchy_mul<A, K>(r2, r, r3);
    cauchy_mul<A, K>(r3, u, c3);
#pragma unroll
    for (int i = 0; i < C; ++i) {
#pragma unroll
      for (int t = 0; t < U::kUnits; ++t) {
        A h[U::kElements][K + 1];
#pragma unroll
        for (int e = 0; e < U::kElements; ++e)
#pragma unroll
          for (int k = 0; k <= K; ++k) h[e][k] = g[i].get(k, U::element(t, e));
        rope_turn<K, V, NEXT, true>(h, c[i], sn[i], t);
#pragma unroll
        for (int e = 0; e < U::kElements; ++e) {
          const int at = U::element(t, e);
          A v[K + 1];
          rope_product<A, K>(h[e], r, v);
          rope_weigh<T, K, V>(w[i], w_p, w_orders, ch[i], at, v);
#pragma unroll
          for (int k = 0; k <= K; ++k) {
#pragma unroll
            for (int j = 0; j <= k; ++j) v[k] = fma(-c3[j], x[i].get(k - j, at), v[k]);
            h[e][k] = v[k];
          }
        }
#pragma unroll
        for (int e = 0; e < U::kElements; e += V == 1 ? 1 : 2)
#pragma unroll
          for (int k = 0; k <= K; ++k) g[i].put(k, U::element(t, e), h[e][k], h[V == 1 ? e : e + 1][k]);
      }
      g[i].mask(ch[i], use);
      // dx is [batch, length, heads, D]: row after row
      if (row.live) g[i].template write<true>(dx_p, static_cast<int64_t>(index) * a.head_dim, ch[i]);
    }
  }
  if constexpr (SUM > 0) {   // the block's rows: those of a wave by lane exchanges, then its waves in order
    constexpr int kWaves = kRopeThreads / kWave;
    __shared__ A buf[2 * V * C][kRopeThreads];
    A* partial = PT_ROPE_PICK(partial);
    if (!PT_ROPE_PICK(want_dw)) return;
    const int wave = threadIdx.x / kWave, in_wave = threadIdx.x % kWave;
#pragma unroll
    for (int q = 0; q < kSums; ++q) {
#pragma unroll
      for (int i = 0; i < C; ++i)
#pragma unroll
        for (int e = 0; e < 2 * V; ++e) {
          A sum = dw[q][i][e];
          for (int off = G; off < kWave; off <<= 1) sum += __shfl_xor(sum, off, kWave);
          if (in_wave < G) buf[i * 2 * V + e][wave * G + in_wave] = sum;
        }
      __syncthreads();
      for (int slot = threadIdx.x; slot < G * 2 * V * C; slot += kRopeThreads) {   // (slot / G: the lane's value, slot mod G: the lane)
        const int value = slot / G, from = slot & (G - 1), i = value / (2 * V), e = value % (2 * V);
        A sum = A(0);
#pragma unroll
        for (int w = 0; w < kWaves; ++w) sum += buf[value][w * G + from];
        const RopeChunk c = rope_chunk<V>(from + i * G, a.head_dim, a.rotary, a.interleaved);
        if (e < V ? c.has_lo : c.has_hi)
          partial[(static_cast<int64_t>(block) * kSums + q) * a.head_dim + (e < V ? c.lo + e : c.hi + e - V)] = sum;
      }
      __syncthreads();
    }
  }
}

template <typename T>
struct RopeReduceArgs {
  const typename AccOf<T>::type* partial[2];
  uint32_t blocks[2];
  int orders[2];      // orders returned: 0, 1 (the last order summed) or every order
  MPtrs<T> out[2];
  int sums, head_dim;
};

// The partial rows' sum: 4 columns a block, 64 threads a column, each adding every 64th row, eight loads at a time; then
// the 64 sums in order. (16 columns a block with one load at a time: 18 us for 1024 rows, each waiting for its loads.)
template <typename T>
__global__ __launch_bounds__(kRopeThreads) void rope_weight_reduce_kernel(const RopeReduceArgs<T> a) {
  using A = typename AccOf<T>::type;
  constexpr int kColumns = 4, kStrands = kRopeThreads / kColumns, kAhead = 8;
  __shared__ A red[kStrands][kColumns];
  const bool second = blockIdx.y == 1;
  const int orders = second ? a.orders[1] : a.orders[0];
  const uint32_t blocks = second ? a.blocks[1] : a.blocks[0];
  const A* partial = second ? a.partial[1] : a.partial[0];
  const int order = blockIdx.z, column = blockIdx.x * kColumns + threadIdx.x % kColumns;
  const uint32_t strand = threadIdx.x / kColumns;
  if (order >= orders) return;
  const int from = orders == 1 ? a.sums - 1 : order;
  const int64_t step = static_cast<int64_t>(a.sums) * a.head_dim;
  A s = A(0);
  if (column < a.head_dim) {
    const A* p = partial + from * a.head_dim + column;
    for (uint32_t b = strand; b < blocks; b += kAhead * kStrands) {
      A v[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const uint32_t row = b + i * kStrands;
        v[i] = p[(row < blocks ? row : b) * step];
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) s += b + i * kStrands < blocks ? v[i] : A(0);
    }
  }
  red[strand][threadIdx.x % kColumns] = s;
  __syncthreads();
  if (threadIdx.x < kColumns && column < a.head_dim) {
    A total = A(0);
#pragma unroll
    for (int i = 0; i < kStrands; ++i) total += red[i][threadIdx.x];
    T* out = nullptr;
#pragma unroll
    for (int k = 0; k < kMaxOrders; ++k)
      if (k == order) out = second ? a.out[1].p[k] : a.out[0].p[k];
    out[column] = from_acc<T>(total);
  }
}

// Lanes a row and the kernel's arguments for chunks of V pairs, C a lane.
template <typename T>
static RopeKernelArgs<T> rope_args(const NormRopeArgs& a, int V, int C, bool backward, int sums) {
  using A = typename AccOf<T>::type;
  RopeKernelArgs<T> k{};
  const int64_t pairs = (a.head_dim + 1) / 2, chunks = (pairs + V - 1) / V;
  int lanes = 1;
  while (static_cast<int64_t>(lanes) * C < chunks) lanes *= 2;
  k.length = rope_divisor(static_cast<uint32_t>(a.length));
  k.head_dim = static_cast<int>(a.head_dim);
  k.rotary = static_cast<int>(a.rotary);
  k.lanes = lanes;
  k.interleaved = a.interleaved != 0;
  k.cos = static_cast<const A*>(a.cos);
  k.sin = static_cast<const A*>(a.sin);
  k.table_rows = a.table_rows;
  k.positions = a.positions;
  k.position_batch_stride = a.position_batch_stride;
  k.eps = static_cast<A>(a.eps);
  A* partial = static_cast<A*>(a.workspace);
  for (int o = 0; o < a.n_ops; ++o) {
    const pt_norm_rope_operand& in = a.ops[o];
    RopeOperand<T>& op = k.op[o];
    for (int i = 0; i <= a.degree; ++i) {
      op.x.p[i] = static_cast<const T*>(in.x[i]);
      if (in.weight != nullptr && i < in.weight_orders) op.w.p[i] = static_cast<const T*>(in.weight[i]);
      if (backward) op.g.p[i] = static_cast<const T*>(in.grad[i]);
      op.y.p[i] = static_cast<T*>(backward ? in.dx[i] : in.y[i]);
    }
    op.stride_b = in.stride_b;
    op.stride_l = in.stride_l;
    op.stride_h = in.stride_h;
    op.heads = rope_divisor(static_cast<uint32_t>(in.heads));
    op.rows = static_cast<uint32_t>(a.batch * a.length * in.heads);
    op.w_orders = in.weight_orders;
    op.want_dw = backward && in.dweight_orders > 0;
    const uint32_t per_block = static_cast<uint32_t>(kRopeThreads / lanes);
    op.blocks = (op.rows + per_block - 1) / per_block;
    if (sums > 0 && op.blocks > kRopeMaxPartials) op.blocks = static_cast<uint32_t>(kRopeMaxPartials);
    if (op.want_dw) {
      op.partial = partial;
      partial += norm_rope_partials(op.rows) * (a.degree + 1) * a.head_dim;
    }
  }
  return k;
}

// Whether chunks of V pairs cover a head exactly, none across the end of the rotated part's halves (V even: neighbours
// lie within a vector).
static bool rope_whole(const NormRopeArgs& a, int V) {
  return a.interleaved ? a.head_dim % (2 * V) == 0
                       : (a.rotary / 2) % V == 0 && (a.head_dim - a.rotary) % (2 * V) == 0;
}

template <typename T, int K>
static int launch_norm_rope_k(const NormRopeArgs& a) {
  // 16 bytes an access, 8 for 16-bit types: with 16 there a lane holds twice the values, and fewer waves are there at once
  // (2 x 2048 tokens of 32 + 8 heads of 128, bfloat16, degree 3: 59 us, 55 with 8 bytes; degree 4 76 and 68)
  constexpr int V = sizeof(T) == 8 ? 2 : 4;
  const bool whole = rope_whole(a, V);
  const RopeKernelArgs<T> k = rope_args<T>(a, whole ? V : 1, whole ? 1 : 2, false, 0);
  const dim3 grid(k.op[0].blocks + k.op[1].blocks);
  const int64_t line = 128 / static_cast<int64_t>(sizeof(T));   // whether the vectors of a head's parts fill whole lines
  const bool lines = a.interleaved ? a.head_dim / 2 % line == 0
                                   : a.rotary / 2 % line == 0 && (a.head_dim - a.rotary) / 2 % line == 0;
#define PT_ROPE_LAUNCH(VV, CC, NX, ST) \
  norm_rope_series_kernel<T, K, VV, CC, NX, ST><<<grid, dim3(kRopeThreads), 0, a.stream>>>(k)
  if (!whole) PT_ROPE_LAUNCH(1, 2, false, false);   // (single elements: lo and hi are a pair's in either arrangement)
  else if (a.interleaved && lines) PT_ROPE_LAUNCH(V, 1, true, true);
  else if (a.interleaved) PT_ROPE_LAUNCH(V, 1, true, false);
  else if (lines) PT_ROPE_LAUNCH(V, 1, false, true);
  else PT_ROPE_LAUNCH(V, 1, false, false);
#undef PT_ROPE_LAUNCH
  PT_LAUNCH_CHECK();
  return PT_OK;
}

// WITHOUT, WITH: whether calls without and with weight gradients come here.
template <typename T, int K, int V, int C, bool NEXT, bool WITHOUT, bool WITH>
static int launch_norm_rope_bwd_v(const NormRopeArgs& a) {
  int sum = 0;
  for (int o = 0; o < a.n_ops; ++o) {
    const int want = a.ops[o].dweight_orders;
    const int mode = want == 0 ? 0 : want == 1 ? 1 : 2;
    sum = mode > sum ? mode : sum;
  }
  const RopeKernelArgs<T> k = rope_args<T>(a, V, C, true, sum);
  const dim3 grid(k.op[0].blocks + k.op[1].blocks);
  const dim3 block(kRopeThreads);
  if constexpr (WITHOUT) {
    if (sum == 0) norm_rope_series_bwd_kernel<T, K, V, C, NEXT, 0><<<grid, block, 0, a.stream>>>(k);
  }
  if constexpr (WITH) {
    if (sum == 1) norm_rope_series_bwd_kernel<T, K, V, C, NEXT, 1><<<grid, block, 0, a.stream>>>(k);
    if (sum == 2) norm_rope_series_bwd_kernel<T, K, V, C, NEXT, 2><<<grid, block, 0, a.stream>>>(k);
  }
  PT_LAUNCH_CHECK();
  if (sum > 0) {
    RopeReduceArgs<T> r{};
    r.sums = sum == 1 ? 1 : K + 1;
    r.head_dim = static_cast<int>(a.head_dim);
    for (int o = 0; o < a.n_ops; ++o) {
      r.partial[o] = k.op[o].partial;
      r.blocks[o] = k.op[o].blocks;
      r.orders[o] = a.ops[o].dweight_orders;
      for (int i = 0; i < a.ops[o].dweight_orders; ++i) r.out[o].p[i] = static_cast<T*>(a.ops[o].dweight[i]);
    }
    rope_weight_reduce_kernel<T><<<dim3((r.head_dim + 3) / 4, a.n_ops, r.sums), dim3(kRopeThreads), 0, a.stream>>>(r);
    PT_LAUNCH_CHECK();
  }
  return PT_OK;
}

template <typename T, int K>
static int launch_norm_rope_bwd_k(const NormRopeArgs& a) {
  // x and the cotangent of every order are in registers: half the pairs a lane from degree 5 on, and in 16-bit types from
  // degree 2 on where weight gradients are summed beside them (2 x 2048 tokens of 32 + 8 heads of 128, bfloat16,
  // degree 3: 101 us without and 116 with weight gradients in fours, 113 and 109 in twos; degree 1 43 and 56, 62 and 61)
  constexpr int V = K <= 4 ? (sizeof(T) == 8 ? 2 : 4) : 2;
  constexpr bool kFewer = sizeof(T) == 2 && K >= 2 && V > 2;
  if constexpr (!(sizeof(T) == 8 && K > 4)) {
    if constexpr (kFewer) {
      bool sums = false;
      for (int o = 0; o < a.n_ops; ++o) sums = sums || a.ops[o].dweight_orders > 0;
      if (sums && rope_whole(a, 2))
        return a.interleaved ? launch_norm_rope_bwd_v<T, K, 2, 1, true, false, true>(a)
                             : launch_norm_rope_bwd_v<T, K, 2, 1, false, false, true>(a);
    }
    if (rope_whole(a, V))
      return a.interleaved ? launch_norm_rope_bwd_v<T, K, V, 1, true, true, !kFewer>(a)
                           : launch_norm_rope_bwd_v<T, K, V, 1, false, true, !kFewer>(a);
  }
  return launch_norm_rope_bwd_v<T, K, 1, 2, false, true, true>(a);
}

#define PT_ROPE_DEGREES(launch)                                                      \
  switch (a.degree) {                                                                \
    case 0: return launch<T, 0>(a);                                                  \
    case 1: return launch<T, 1>(a);                                                  \
    case 2: return launch<T, 2>(a);                                                  \
    case 3: return launch<T, 3>(a);                                                  \
    case 4: return launch<T, 4>(a);                                                  \
    case 5: return launch<T, 5>(a);                                                  \
    case 6: return launch<T, 6>(a);                                                  \
    case 7: return launch<T, 7>(a);                                                  \
    case 8: return launch<T, 8>(a);                                                  \
    default: break;                                                                  \
  }                                                                                  \
  pt_host::set_error("norm and rotation series: degree outside 0..PT_MAX_DEGREE");   \
  return PT_UNSUPPORTED

template <typename T>
int launch_norm_rope(const NormRopeArgs& a) {
  PT_ROPE_DEGREES(launch_norm_rope_k);
}

template <typename T>
int launch_norm_rope_bwd(const NormRopeArgs& a) {
  PT_ROPE_DEGREES(launch_norm_rope_bwd_k);
}

}  // namespace pt
