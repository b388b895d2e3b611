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
// at the two halves of the rotated part or side by side. The row sums go over the G lanes in registers.
#pragma once

#include "norm_rope_series.h"
#include "norm_series.inl"
#include "series_math.h"

namespace pt {

constexpr int kRopeThreads = 256;
constexpr int64_t kRopeMaxPartials = 1024;   // blocks an operand where weight gradients are summed: four a compute unit

// V elements at any element's address.
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef u32x2_t u32x2_any_t __attribute__((aligned(2)));
typedef uint32_t u32_any_t __attribute__((aligned(2)));
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> rope_load(const T* p) {
  if constexpr (V == 1) {
    Vec<T, 1> r;
    r.v[0] = *p;
    return r;
  } else if constexpr (sizeof(T) * V == 16) {
    return load_vec_nt_any<T, V>(p);
  } else if constexpr (sizeof(T) * V == 8) {
    const u32x2_t w = __builtin_nontemporal_load(reinterpret_cast<const u32x2_any_t*>(p));
    return __builtin_bit_cast(Vec<T, V>, w);
  } else {
    static_assert(sizeof(T) * V == 4, "4, 8 or 16 bytes");
    const uint32_t w = __builtin_nontemporal_load(reinterpret_cast<const u32_any_t*>(p));
    return __builtin_bit_cast(Vec<T, V>, w);
  }
}
template <typename T, int V>
__device__ __forceinline__ void rope_store(T* p, const Vec<T, V>& v) {
  if constexpr (V == 1) {
    *p = v.v[0];
  } else if constexpr (sizeof(T) * V == 16) {
    store_vec_nt_any<T, V>(p, v);
  } else if constexpr (sizeof(T) * V == 8) {
    __builtin_nontemporal_store(__builtin_bit_cast(u32x2_t, v), reinterpret_cast<u32x2_any_t*>(p));
  } else {
    __builtin_nontemporal_store(__builtin_bit_cast(uint32_t, v), reinterpret_cast<u32_any_t*>(p));
  }
}
// Element e (a bfloat16 vector is read by words, which a single element has not).
template <typename T, int V>
__device__ __forceinline__ typename AccOf<T>::type rope_get(const Vec<T, V>& v, int e) {
  if constexpr (V == 1) return to_acc(v.v[0]);
  else return vec_get(v, e);
}
template <typename T, int V>
__device__ __forceinline__ void rope_put(T* p, const typename AccOf<T>::type* f) {
  Vec<T, V> v;
  if constexpr (V == 1) {
    v.v[0] = from_acc<T>(f[0]);
  } else {
#pragma unroll
    for (int e = 0; e < V; e += 2) vec_put2(v, e, f[e], f[e + 1]);
  }
  rope_store<T, V>(p, v);
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

template <typename T>
struct RopeOperand {
  CPtrs<T> x, w, g;
  MPtrs<T> y;                  // the output, or dx
  int64_t stride_b, stride_l, stride_h;
  uint32_t heads, rows, blocks;
  int w_orders;
  bool want_dw;
  typename AccOf<T>::type* partial;   // [blocks][orders summed][D]
};

template <typename T>
struct RopeKernelArgs {
  RopeOperand<T> op[2];
  uint32_t length;
  int head_dim, rotary, lanes;
  bool interleaved;
  const typename AccOf<T>::type* cos;
  const typename AccOf<T>::type* sin;
  int64_t table_rows;
  const int64_t* positions;
  int64_t position_batch_stride;
  typename AccOf<T>::type eps;
};

// Where a lane's chunk of V pairs lies in a head: its two V-vectors, and whether the second exists
// (the last element of an odd head has no partner; V = 1 there).
struct RopeChunk {
  int lo, hi, pair;
  bool has_lo, has_hi;
};
template <int V>
__device__ __forceinline__ RopeChunk rope_chunk(int chunk, int head_dim, int rotary, bool interleaved) {
  RopeChunk c;
  c.pair = chunk * V;
  if (interleaved) {
    c.lo = 2 * c.pair;
    c.hi = c.lo + V;
  } else if (c.pair < rotary / 2) {
    c.lo = c.pair;
    c.hi = c.pair + rotary / 2;
  } else {
    c.lo = rotary + c.pair - rotary / 2;
    c.hi = c.lo + (head_dim - rotary + 1) / 2;
  }
  c.has_lo = 2 * c.pair < head_dim;
  c.has_hi = c.has_lo && c.hi < head_dim;
  if (!c.has_lo) c.lo = 0;        // (addresses stay inside the row; the values are not used)
  if (!c.has_hi) c.hi = c.lo;
  return c;
}

// A row's place: where it is read and written, and its position in the tables.
struct RopeRow {
  int64_t in, out, pos;
  bool live;
};
template <typename T>
__device__ __forceinline__ RopeRow rope_row(const RopeKernelArgs<T>& a, uint32_t row, uint32_t rows, uint32_t heads,
                                            int64_t sb, int64_t sl, int64_t sh) {
  RopeRow r;
  r.live = row < rows;
  if (!r.live) row = rows - 1;
  const uint32_t h = row % heads, bl = row / heads, l = bl % a.length, b = bl / a.length;
  r.in = b * sb + l * sl + h * sh;
  r.out = ((static_cast<int64_t>(b) * heads + h) * a.length + l) * a.head_dim;
  r.pos = a.positions != nullptr ? a.positions[b * a.position_batch_stride + l] : static_cast<int64_t>(l);
  return r;
}

// Cosines and sines of a chunk's pairs (1 and 0 behind the rotated part).
template <typename A, int V>
__device__ __forceinline__ void rope_angles(const A* cos, const A* sin, int64_t table_rows, int rotary, int64_t pos, int pair,
                                            A (&c)[V], A (&s)[V]) {
  const int half = rotary / 2;
  const bool inside = pos >= 0 && pos < table_rows;
  const int64_t at = inside ? pos * half : 0;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const bool turned = inside && pair + e < half;
    c[e] = turned ? cos[at + pair + e] : A(1);
    s[e] = turned ? sin[at + pair + e] : A(0);
  }
  if (pos >= table_rows) {
#pragma unroll
    for (int e = 0; e < V; ++e) c[e] = __builtin_nan("");
  }
}

// (a, b) -> (a c - b s, b c + a s) on the pairs of a chunk v = [lo, hi]. NEXT: a pair's elements are
// neighbours (a template argument: a branch between the two forms puts v in scratch memory).
template <typename A, int V, bool NEXT>
__device__ __forceinline__ void rope_turn(A (&v)[2 * V], const A (&c)[V], const A (&s)[V]) {
  auto turn = [](A& a, A& b, A co, A si) {
    const A x = a;
    a = x * co - b * si;
    b = b * co + x * si;
  };
#pragma unroll
  for (int e = 0; e < V; ++e) {
    if constexpr (NEXT) turn(v[2 * e], v[2 * e + 1], c[e], s[e]);
    else turn(v[e], v[V + e], c[e], s[e]);
  }
}

// The orders of a chunk in the arithmetic type (zero where the lane has none).
template <typename T, int K, int V>
__device__ __forceinline__ void rope_read(const T* const (&p)[K + 1], int64_t at, const RopeChunk& ch, bool use,
                                          typename AccOf<T>::type (&v)[K + 1][2 * V]) {
  using A = typename AccOf<T>::type;
  Vec<T, V> lo[K + 1], hi[K + 1];
#pragma unroll
  for (int k = 0; k <= K; ++k) {
    lo[k] = rope_load<T, V>(p[k] + at + ch.lo);
    hi[k] = rope_load<T, V>(p[k] + at + ch.hi);
  }
#pragma unroll
  for (int k = 0; k <= K; ++k)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      v[k][e] = use && ch.has_lo ? rope_get(lo[k], e) : A(0);
      v[k][V + e] = use && ch.has_hi ? rope_get(hi[k], e) : A(0);
    }
}

template <typename T, int K, int V>
__device__ __forceinline__ void rope_write(T* const (&p)[K + 1], int64_t at, const RopeChunk& ch,
                                           const typename AccOf<T>::type (&v)[K + 1][2 * V]) {
#pragma unroll
  for (int k = 0; k <= K; ++k) {
    if (ch.has_lo) rope_put<T, V>(p[k] + at + ch.lo, &v[k][0]);
    if (ch.has_hi) rope_put<T, V>(p[k] + at + ch.hi, &v[k][V]);
  }
}

// v <- w (*) v on a chunk (w ordinary, or a series of K + 1 orders).
template <typename T, int K, int V>
__device__ __forceinline__ void rope_weigh(const T* const (&w)[K + 1], int w_orders, const RopeChunk& ch,
                                           typename AccOf<T>::type (&v)[K + 1][2 * V]) {
  using A = typename AccOf<T>::type;
  if (w_orders == 0) return;
  if (K == 0 || w_orders == 1) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const A lo = to_acc(w[0][ch.lo + e]), hi = to_acc(w[0][ch.hi + e]);
#pragma unroll
      for (int k = 0; k <= K; ++k) {
        v[k][e] *= lo;
        v[k][V + e] *= hi;
      }
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 2 * V; ++e) {
    const int at = e < V ? ch.lo + e : ch.hi + e - V;
    A ws[K + 1];
#pragma unroll
    for (int k = 0; k <= K; ++k) ws[k] = to_acc(w[k][at]);
#pragma unroll
    for (int k = K; k >= 0; --k) {
      A s = v[k][e] * ws[0];
#pragma unroll
      for (int i = 0; i < k; ++i) s = fma(v[i][e], ws[k - i], s);
      v[k][e] = s;
    }
  }
}

// Sums of a chunk's elements of x (*) x.
template <typename A, int K, int N>
__device__ __forceinline__ void rope_square(const A (&x)[K + 1][N], A (&s)[K + 1]) {
#pragma unroll
  for (int e = 0; e < N; ++e) {
    A c[K + 1];
#pragma unroll
    for (int k = 0; k <= K; ++k) c[k] = x[k][e];
#pragma unroll
    for (int k = 0; k <= K; ++k) s[k] += cauchy_square<A, K>(c, k);
  }
}

#define PT_ROPE_PICK(field) (second ? a.op[1].field : a.op[0].field)

template <typename T, int K, int V, int C, bool NEXT>
__global__ __launch_bounds__(kRopeThreads) void norm_rope_series_kernel(const RopeKernelArgs<T> a) {
  using A = typename AccOf<T>::type;
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
  const uint32_t rows = PT_ROPE_PICK(rows), heads = PT_ROPE_PICK(heads);
  const RopeRow row = rope_row(a, block * (kRopeThreads / G) + threadIdx.x / G, rows, heads, PT_ROPE_PICK(stride_b),
                               PT_ROPE_PICK(stride_l), PT_ROPE_PICK(stride_h));
  const bool use = row.pos >= 0;
  RopeChunk ch[C];
  A x[C][K + 1][2 * V];
  A s[K + 1];
#pragma unroll
  for (int k = 0; k <= K; ++k) s[k] = A(0);
#pragma unroll
  for (int i = 0; i < C; ++i) {
    ch[i] = rope_chunk<V>(lane + i * G, a.head_dim, a.rotary, a.interleaved);
    rope_read<T, K, V>(x_p, row.in, ch[i], use, x[i]);
  }
#pragma unroll
  for (int i = 0; i < C; ++i) rope_square<A, K, 2 * V>(x[i], s);
#pragma unroll
  for (int k = 0; k <= K; ++k) s[k] = group_sum(s[k], G);
  A r[K + 1];
  rsqrt_series<A, K>(s, A(1) / A(a.head_dim), a.eps, r);
#pragma unroll
  for (int k = 0; k <= K; ++k) r[k] = use ? r[k] : A(0);
#pragma unroll
  for (int i = 0; i < C; ++i) {
#pragma unroll
    for (int e = 0; e < 2 * V; ++e)
#pragma unroll
      for (int k = K; k >= 0; --k) {
        A v = x[i][k][e] * r[0];
#pragma unroll
        for (int j = 0; j < k; ++j) v = fma(x[i][j][e], r[k - j], v);
        x[i][k][e] = v;
      }
    rope_weigh<T, K, V>(w_p, w_orders, ch[i], x[i]);
    A c[V], sn[V];
    rope_angles<A, V>(a.cos, a.sin, a.table_rows, a.rotary, row.pos, ch[i].pair, c, sn);
#pragma unroll
    for (int k = 0; k <= K; ++k) rope_turn<A, V, NEXT>(x[i][k], c, sn);
    if (!use) {   // (a weight or an angle that is no number does not reach padding)
#pragma unroll
      for (int k = 0; k <= K; ++k)
#pragma unroll
        for (int e = 0; e < 2 * V; ++e) x[i][k][e] = A(0);
    }
    if (row.live) rope_write<T, K, V>(y_p, row.out, ch[i], x[i]);
  }
}

// SUM: weight gradients are summed, of order K alone (1: an ordinary weight under the reversed cotangents
// of coefficient gradients) or of every order (2); 0: none. Then a block takes every blocks-th group of
// rows and leaves its sums as a row of `partial`, which rope_weight_reduce_kernel adds in a fixed order.
template <typename T, int K, int V, int C, bool NEXT, int SUM>
__global__ __launch_bounds__(kRopeThreads) void norm_rope_series_bwd_kernel(const RopeKernelArgs<T> a) {
  using A = typename AccOf<T>::type;
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
  const uint32_t rows = PT_ROPE_PICK(rows), heads = PT_ROPE_PICK(heads), per_block = kRopeThreads / G;
  const uint32_t blocks = PT_ROPE_PICK(blocks);
  RopeChunk ch[C];
#pragma unroll
  for (int i = 0; i < C; ++i) ch[i] = rope_chunk<V>(lane + i * G, a.head_dim, a.rotary, a.interleaved);
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
    A x[C][K + 1][2 * V], g[C][K + 1][2 * V];
    A s[K + 1], u[K + 1], r[K + 1];
#pragma unroll
    for (int k = 0; k <= K; ++k) s[k] = u[k] = A(0);
#pragma unroll
    for (int i = 0; i < C; ++i) {
      rope_read<T, K, V>(x_p, row.in, ch[i], use, x[i]);
      rope_read<T, K, V>(g_p, row.out, ch[i], use, g[i]);
    }
#pragma unroll
    for (int i = 0; i < C; ++i) rope_square<A, K, 2 * V>(x[i], s);
#pragma unroll
    for (int k = 0; k <= K; ++k) s[k] = group_sum(s[k], G);
    rsqrt_series<A, K>(s, A(1) / A(a.head_dim), a.eps, r);
#pragma unroll
    for (int k = 0; k <= K; ++k) r[k] = use ? r[k] : A(0);
#pragma unroll
    for (int i = 0; i < C; ++i) {
      A c[V], sn[V];
      rope_angles<A, V>(a.cos, a.sin, a.table_rows, a.rotary, row.pos, ch[i].pair, c, sn);
#pragma unroll
      for (int e = 0; e < V; ++e) sn[e] = -sn[e];
#pragma unroll
      for (int k = 0; k <= K; ++k) rope_turn<A, V, NEXT>(g[i][k], c, sn);
      if constexpr (SUM > 0) {
#pragma unroll
        for (int e = 0; e < 2 * V; ++e) {
          A n[K + 1];
#pragma unroll
          for (int k = 0; k <= K; ++k) {
            A v = x[i][k][e] * r[0];
#pragma unroll
            for (int j = 0; j < k; ++j) v = fma(x[i][j][e], r[k - j], v);
            n[k] = v;
          }
#pragma unroll
          for (int q = 0; q < kSums; ++q) {
            const int order = SUM == 1 ? K : q;
#pragma unroll
            for (int j = 0; j <= order; ++j) dw[q][i][e] = fma(n[j], g[i][order - j][e], dw[q][i][e]);
          }
        }
      }
      rope_weigh<T, K, V>(w_p, w_orders, ch[i], g[i]);
#pragma unroll
      for (int e = 0; e < 2 * V; ++e)
#pragma unroll
        for (int k = 0; k <= K; ++k)
#pragma unroll
          for (int j = 0; j <= k; ++j) u[k] = fma(x[i][j][e], (e < V ? ch[i].has_lo : ch[i].has_hi) ? g[i][k - j][e] : A(0), u[k]);
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
      for (int e = 0; e < 2 * V; ++e)
#pragma unroll
        for (int k = K; k >= 0; --k) {
          A v = r[0] * g[i][k][e];
#pragma unroll
          for (int j = 1; j <= k; ++j) v = fma(r[j], g[i][k - j][e], v);
#pragma unroll
          for (int j = 0; j <= k; ++j) v = fma(-c3[j], x[i][k - j][e], v);
          g[i][k][e] = use ? v : A(0);
        }
      if (row.live) {
        // dx is [batch, length, heads, D]: row after row
        const int64_t at = static_cast<int64_t>(index) * a.head_dim;
        rope_write<T, K, V>(dx_p, at, ch[i], g[i]);
      }
    }
  }
  if constexpr (SUM > 0) {
    __shared__ A buf[kRopeThreads * 2 * V * C];
    A* partial = PT_ROPE_PICK(partial);
    if (!PT_ROPE_PICK(want_dw)) return;
#pragma unroll
    for (int q = 0; q < kSums; ++q) {
#pragma unroll
      for (int i = 0; i < C; ++i)
#pragma unroll
        for (int e = 0; e < 2 * V; ++e) buf[(i * 2 * V + e) * kRopeThreads + threadIdx.x] = dw[q][i][e];
      __syncthreads();
      for (int slot = threadIdx.x; slot < G * 2 * V * C; slot += kRopeThreads) {   // (slot / G: the lane's value, slot mod G: the lane)
        A sum = A(0);
        for (uint32_t row = 0; row < per_block; ++row) sum += buf[(slot / G) * kRopeThreads + row * G + (slot & (G - 1))];
        const int i = (slot / G) / (2 * V), e = (slot / G) % (2 * V);
        const RopeChunk c = rope_chunk<V>((slot & (G - 1)) + i * G, a.head_dim, a.rotary, a.interleaved);
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
  k.length = static_cast<uint32_t>(a.length);
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
    op.heads = static_cast<uint32_t>(in.heads);
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

// Whether chunks of V pairs cover a head exactly, none across the end of the rotated part's halves.
static bool rope_whole(const NormRopeArgs& a, int V) {
  return a.interleaved ? a.head_dim % (2 * V) == 0
                       : (a.rotary / 2) % V == 0 && (a.head_dim - a.rotary) % (2 * V) == 0;
}

template <typename T, int K>
static int launch_norm_rope_k(const NormRopeArgs& a) {
  constexpr int V = VecWidth<T>::value;
  const bool whole = rope_whole(a, V);
  const RopeKernelArgs<T> k = rope_args<T>(a, whole ? V : 1, whole ? 1 : 2, false, 0);
  const dim3 grid(k.op[0].blocks + k.op[1].blocks);
  if (whole && a.interleaved)
    norm_rope_series_kernel<T, K, V, 1, true><<<grid, dim3(kRopeThreads), 0, a.stream>>>(k);
  else if (whole)
    norm_rope_series_kernel<T, K, V, 1, false><<<grid, dim3(kRopeThreads), 0, a.stream>>>(k);
  else   // (single elements: lo and hi are a pair's in either arrangement)
    norm_rope_series_kernel<T, K, 1, 2, false><<<grid, dim3(kRopeThreads), 0, a.stream>>>(k);
  PT_LAUNCH_CHECK();
  return PT_OK;
}

template <typename T, int K, int V, int C, bool NEXT>
static int launch_norm_rope_bwd_v(const NormRopeArgs& a) {
  int sum = 0;
  for (int o = 0; o < a.n_ops; ++o) {
    const int want = a.ops[o].dweight_orders;
    const int mode = want == 0 ? 0 : want == 1 ? 1 : 2;
    sum = mode > sum ? mode : sum;
  }
  const RopeKernelArgs<T> k = rope_args<T>(a, V, C, true, sum);
  const dim3 grid(k.op[0].blocks + k.op[1].blocks);
  if (sum == 0)
    norm_rope_series_bwd_kernel<T, K, V, C, NEXT, 0><<<grid, dim3(kRopeThreads), 0, a.stream>>>(k);
  else if (sum == 1)
    norm_rope_series_bwd_kernel<T, K, V, C, NEXT, 1><<<grid, dim3(kRopeThreads), 0, a.stream>>>(k);
  else
    norm_rope_series_bwd_kernel<T, K, V, C, NEXT, 2><<<grid, dim3(kRopeThreads), 0, a.stream>>>(k);
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
  // x, the cotangent and the sums of every order in registers: half of the forward's chunk, a quarter of it above degree 4
  constexpr int V = K <= 4 ? (sizeof(T) == 2 ? 4 : VecWidth<T>::value) : 2;
  if constexpr (!(sizeof(T) == 8 && K > 4)) {
    if (rope_whole(a, V))
      return a.interleaved ? launch_norm_rope_bwd_v<T, K, V, 1, true>(a) : launch_norm_rope_bwd_v<T, K, V, 1, false>(a);
  }
  return launch_norm_rope_bwd_v<T, K, 1, 2, false>(a);
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
