// Log probabilities of given tokens, the entropy and the most probable alternatives of rows of logits,
// as degree-K series, in one streaming pass a row.
//
// For a row z(t) over C classes, with m = max z_0 and the row's series shifted by (m, rho_1, .., rho_K), rho
// the mean of the row's first 64 classes (any shift common to all classes changes no probability; this
// one leaves values of the size of their spread, so that no order loses its digits to an offset):
//   E = exp(z) a class,   F_k = k E_k = sum_{j=1..k} j z_j E_{k-j}
//   S = sum E,   Q = sum E (*) z,   k Q_k = sum_c (F_k + sum_{a=1..k} F_a z_{k-a})
//   L = log S (the log series),  log p = z - L,   H = L - Q / S  (= -sum p (*) log p)
// A thread keeps m, S_0, sum F_k and W_k = sum_a sum F_a z_{k-a} (W_0 = sum E_0 z_0) of its share; a new
// maximum m' turns W_k into e^(m - m') (W_k + (m - m') sum F_k). The threads' states are joined by the
// same rule, in a fixed order.
// A class with z_0 = -inf has probability zero whatever its higher orders hold. A row without any other
// class has no distribution: its results are NaN.
//
// Alternatives are the classes of the largest z_0 (before a softcap, which keeps the order), ties by the
// lower class, NaN first. Each thread keeps the largest of its share. With 64 groups of threads, the
// `top`-th largest group maximum is a bound that at least `top` classes reach, and only threads whose
// maximum reaches it can hold such classes: their shares are read again, by the whole block, and the
// classes that reach the bound (a few more than `top`, unless the row is arranged against it) are ranked
// by counting. Too many, too few (fewer than `top` classes above -inf) or a NaN in the row: the block
// finds one class after the other in passes over the row.
//
// Few rows are cut into pieces, a block each, whose states and alternatives a second kernel joins.
//
// HBM bounds long rows: 8192 x 32000 float32 at degree 4 with 5 alternatives 803 us, 6.5 TB/s; 4096 x 32001 bfloat16 at degree
// 3 170 us, 6.2 TB/s, its gradient 419 us, 5.0 TB/s (streams over the same buffers 158 and 340). 16-bit logits of low
// degree come nearer the vector units' rate: 2048 x 128256 bfloat16, degree 1, 20 alternatives 223 us, 4.7 TB/s.
// Few rows are bound by a block's chain of loads and barriers, about 10 us, and the join's 7 (8 x 131072: 9.5 + 7.0).
#pragma once

#include <type_traits>

#include "cross_entropy_series.inl"
#include "token_log_probs_series.h"

namespace pt {

constexpr int kLpThreads = 256;
constexpr int kLpWaves = kLpThreads / kWave;
constexpr int kLpMaxTop = PT_LOG_PROBS_MAX_TOP;
constexpr int kLpMaxSplits = 64;   // one lane of a wave joins each
constexpr int kLpCandidates = 512;

// ---- the order of classes ---------------------------------------------------
// Bits that compare as the values do: NaN above everything, -0 and +0 alike; 0 is no value's.
__device__ __forceinline__ uint32_t rank_bits(float x) {
  x += 0.0f;
  const uint32_t u = __float_as_uint(x);
  if (x != x) return 0xffffffffu;
  return (u >> 31) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint64_t rank_bits(double x) {
  x += 0.0;
  const uint64_t u = static_cast<uint64_t>(__double_as_longlong(x));
  if (x != x) return ~0ull;
  return (u >> 63) ? ~u : u | (1ull << 63);
}

template <typename A>
struct TopKey {
  using U = decltype(rank_bits(A()));
  U v;          // 0: no class
  uint32_t i;   // the class
};
template <typename A>
__device__ __forceinline__ bool before(const TopKey<A>& a, const TopKey<A>& b) {
  return a.v > b.v || (a.v == b.v && a.i < b.i);
}
template <typename A>
__device__ __forceinline__ TopKey<A> no_key() {
  return {0, 0xffffffffu};
}
template <typename A>
__device__ __forceinline__ TopKey<A> shuffled(const TopKey<A>& k, int mask) {
  return {static_cast<typename TopKey<A>::U>(__shfl_xor(static_cast<unsigned long long>(k.v), mask, kWave)),
          static_cast<uint32_t>(__shfl_xor(static_cast<int>(k.i), mask, kWave))};
}

// Elements before the vectors of a row, which start at the first cache line that begins at or after p, so that a wave's
// accesses take whole lines; in rows below 16 KB, where the elements before them would cost more, at the first 16
// bytes (4096 x 32001 bfloat16, degree 3: 178 and 490 us forward and backward from the first 16 bytes, 168 and 418 from the
// first line; 16384 x 1000 float32, degree 2: 101 and 84, 108 and 87).
template <typename T>
__device__ __forceinline__ int64_t lp_head(const T* p, int64_t n) {
  const uint32_t line = n * static_cast<int64_t>(sizeof(T)) >= 16384 ? 128u : 16u;
  const int64_t head = static_cast<int64_t>((0u - static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p))) & (line - 1)) /
                       static_cast<int64_t>(sizeof(T));
  return head < n ? head : n;
}

// ---- a row's running state ----------------------------------------------------
template <typename A, int K>
struct LpState {
  A m, S[K + 1], W[K + 1];
};

template <typename A>
__device__ __forceinline__ A lp_floor() { return A(-1e4); }   // exp of it is 0 in both types

template <typename A, int K>
__device__ __forceinline__ void lp_clear(LpState<A, K>& st) {
  st.m = -__builtin_huge_val();
#pragma unroll
  for (int k = 0; k <= K; ++k) st.S[k] = st.W[k] = A(0);
}

// The state with its sums relative to M >= m. Where nothing of it is left both factors are zero: products
// with them, so that a sum that is no number stays one.
template <typename A, int K>
__device__ __forceinline__ void lp_rebase(LpState<A, K>& st, A M) {
  A delta = st.m - M;
  A f = exp_fast(delta);
  if (st.m == A(-__builtin_huge_val()) || f == A(0)) delta = f = A(0);
#pragma unroll
  for (int k = 0; k <= K; ++k) {
    st.W[k] = f * fma(delta, st.S[k], st.W[k]);
    st.S[k] *= f;
  }
  st.m = M;
}

// One class: d its series with d[0] = z_0, d[k >= 1] shifted.
template <typename A, int K>
__device__ __forceinline__ void lp_add(LpState<A, K>& st, const A (&d)[K + 1]) {
  const A q = d[0] - st.m;
  const A q0 = fmax(q, lp_floor<A>());   // (E_0 is zero below: 0 times a number, not times -inf)
  A E[K + 1], F[K + 1], jd[K + 1];
  E[0] = exp_fast(q);
  st.S[0] += E[0];
  st.W[0] = fma(E[0], q0, st.W[0]);
#pragma unroll
  for (int k = 1; k <= K; ++k) {
    jd[k] = A(k) * d[k];
    A s = A(0);
#pragma unroll
    for (int j = 1; j <= k; ++j) s = j == 1 ? jd[j] * E[k - j] : fma(jd[j], E[k - j], s);
    F[k] = s;
    E[k] = s * (A(1) / A(k));
    st.S[k] += s;
    A w = fma(s, q0, st.W[k]);
#pragma unroll
    for (int a = 1; a < k; ++a) w = fma(F[a], d[k - a], w);
    st.W[k] = w;
  }
}

template <typename A, int K>
__device__ __forceinline__ void lp_join_wave(LpState<A, K>& st) {
  lp_rebase(st, wave_max(st.m));
#pragma unroll
  for (int k = 0; k <= K; ++k) {
    st.S[k] = wave_sum(st.S[k]);
    st.W[k] = wave_sum(st.W[k]);
  }
}

template <typename T>
struct LpKernelArgs {
  using A = typename AccOf<T>::type;
  CPtrs<T> z;
  int64_t classes, row_stride, piece;
  uint32_t splits;
  const int64_t* tokens;
  int64_t ignore_index;
  A cap, inv_cap;
  int top;
  MPtrs<A> log_probs, entropy, top_log_probs, lse;
  int64_t* top_tokens;
  A* partial;                       // [row][split][3 K + 3]: m, S, W and the shift, the same in every piece
  typename TopKey<A>::U* key_bits;  // [row][split][top]
  uint32_t* key_class;
};

// The shift of the row's higher orders, by every wave alike: the mean of its first 64 classes, of the finite
// values among them.
template <typename T, int K, bool CAP>
__device__ __forceinline__ void lp_shift(const LpKernelArgs<T>& a, int64_t row, typename AccOf<T>::type (&rho)[K + 1]) {
  using A = typename AccOf<T>::type;
  const int n = a.classes < kWave ? static_cast<int>(a.classes) : kWave, lane = threadIdx.x % kWave;
  A x[K + 1];
#pragma unroll
  for (int k = CAP ? 0 : 1; k <= K; ++k) x[k] = to_acc(a.z.p[k][row * a.row_stride + (lane < n ? lane : 0)]);
  if constexpr (CAP) softcap_series<A, K>(x, a.cap, a.inv_cap);
  rho[0] = A(0);
#pragma unroll
  for (int k = 1; k <= K; ++k) {
    const A sum = wave_sum(lane < n && fabs(x[k]) < A(__builtin_huge_val()) ? x[k] : A(0)) / A(n);
    rho[k] = fabs(sum) < A(__builtin_huge_val()) ? sum : A(0);
  }
}

// Results of a row from its whole state, by the block: thread 0 the series, then a thread an alternative.
template <typename T, int K, bool CAP, bool TOP>
__device__ __forceinline__ void lp_finish(const LpKernelArgs<T>& a, int64_t row, int64_t y,
                                          const LpState<typename AccOf<T>::type, K>& st,
                                          const typename AccOf<T>::type (&rho)[K + 1],
                                          const TopKey<typename AccOf<T>::type>* best, typename AccOf<T>::type* shared) {
  using A = typename AccOf<T>::type;
  if (threadIdx.x == 0) {
    const bool valid = y >= 0 && y < a.classes;
    A zy[K + 1];
#pragma unroll
    for (int k = 0; k <= K; ++k) zy[k] = valid ? to_acc(a.z.p[k][row * a.row_stride + y]) : A(0);
    if constexpr (CAP) softcap_series<A, K>(zy, a.cap, a.inv_cap);
    A n[K + 1], L[K + 1], Q[K + 1];
    n[0] = A(1);
    const A inv = A(1) / st.S[0];
    L[0] = log_acc(st.S[0]);
    Q[0] = st.W[0] * inv;
#pragma unroll
    for (int k = 1; k <= K; ++k) {
      n[k] = st.S[k] * (A(1) / A(k)) * inv;
      A s = n[k];
#pragma unroll
      for (int i = 1; i < k; ++i) s -= (A(i) / A(k)) * L[i] * n[k - i];
      L[k] = s;
      A q = n[k] + st.W[k] * (A(1) / A(k)) * inv;
#pragma unroll
      for (int j = 1; j <= k; ++j) q -= n[j] * Q[k - j];
      Q[k] = q;
    }
    const A none = __builtin_nan("");
#pragma unroll
    for (int k = 0; k <= K; ++k) {
      const A shift = k == 0 ? st.m : rho[k];
      a.log_probs.p[k][row] = valid ? (zy[k] - shift) - L[k] : none;   // a token that is no class has no probability
      a.entropy.p[k][row] = L[k] - Q[k];
      a.lse.p[k][row] = shift + L[k];
      shared[k] = L[k];
    }
  }
  if constexpr (TOP) {
    __syncthreads();
    const int j = threadIdx.x;
    if (j < a.top) {
      const uint32_t c = best[j].i;
      A x[K + 1];
#pragma unroll
      for (int k = 0; k <= K; ++k) x[k] = to_acc(a.z.p[k][row * a.row_stride + c]);
      if constexpr (CAP) softcap_series<A, K>(x, a.cap, a.inv_cap);
      a.top_tokens[row * a.top + j] = c;
#pragma unroll
      for (int k = 0; k <= K; ++k)
        a.top_log_probs.p[k][row * a.top + j] = (x[k] - (k == 0 ? st.m : rho[k])) - shared[k];
    }
  }
}

// A row without a token: zero results, no alternatives.
template <typename T, int K, bool TOP>
__device__ __forceinline__ void lp_ignored(const LpKernelArgs<T>& a, int64_t row) {
  using A = typename AccOf<T>::type;
  if (threadIdx.x == 0) {
#pragma unroll
    for (int k = 0; k <= K; ++k) a.log_probs.p[k][row] = a.entropy.p[k][row] = a.lse.p[k][row] = A(0);
  }
  if (TOP && static_cast<int>(threadIdx.x) < a.top) {
    a.top_tokens[row * a.top + threadIdx.x] = -1;
#pragma unroll
    for (int k = 0; k <= K; ++k) a.top_log_probs.p[k][row * a.top + threadIdx.x] = A(0);
  }
}

// The first `top` of n keys, in order, into best[]: each key's place is the number of keys before it.
template <typename A>
__device__ __forceinline__ void lp_rank(const TopKey<A>* keys, int n, int top, TopKey<A>* best) {
  for (int c = threadIdx.x; c < n; c += kLpThreads) {
    const TopKey<A> key = keys[c];
    int place = 0;
    for (int j = 0; j < n; ++j) place += before(keys[j], key);
    if (place < top) best[place] = key;
  }
  __syncthreads();
}

template <typename A>
struct LpTopShared {
  TopKey<A> group[64], bound, best[kLpMaxTop], found[kLpCandidates], wave[kLpWaves];
  uint32_t threads[kLpThreads];
  int n_threads, n_found;
};

// A key that at least `top` of the threads' own reach, a little below the top-th: the top-th largest of 64
// groups' maxima (no key's where fewer groups have one). The counters are cleared.
template <typename A, typename Shared>
__device__ __forceinline__ TopKey<A> lp_bound(TopKey<A> own, int top, Shared& sh) {
#pragma unroll
  for (int mask = 1; mask <= 2; mask <<= 1) {
    const TopKey<A> o = shuffled(own, mask);
    if (before(o, own)) own = o;
  }
  if (threadIdx.x % 4 == 0) sh.group[threadIdx.x / 4] = own;
  if (threadIdx.x == 0) {
    sh.bound = no_key<A>();
    sh.n_threads = sh.n_found = 0;
  }
  __syncthreads();
  if (threadIdx.x < 64) {
    const TopKey<A> key = sh.group[threadIdx.x];
    int place = 0;
#pragma unroll 16
    for (int j = 0; j < 64; ++j) place += before(sh.group[j], key);
    if (place == top - 1 && key.v != 0) sh.bound = key;
  }
  __syncthreads();
  return sh.bound;
}

// The block's `top` first classes of z0[0 .. n), whose vectors start at `head`; classes are numbered from `first`.
template <typename T>
__device__ void lp_select(const T* z0, int64_t n, int64_t head, uint32_t first, TopKey<typename AccOf<T>::type> own, bool careful,
                          int top, LpTopShared<typename AccOf<T>::type>& sh) {
  using A = typename AccOf<T>::type;
  constexpr int V = VecWidth<T>::value;
  const int64_t nvec = (n - head) / V, around = n - nvec * V;
  const TopKey<A> bound = lp_bound(own, top, sh);
  bool done = false;
  if (bound.v != 0 && !careful) {
    if (!before(bound, own)) sh.threads[atomicAdd(&sh.n_threads, 1)] = threadIdx.x;
    __syncthreads();
    const int64_t per = (nvec + kLpThreads - 1) / kLpThreads + 1, total = sh.n_threads * per;
    auto offer = [&](A x, int64_t at) {
      const TopKey<A> key{rank_bits(x), first + static_cast<uint32_t>(at)};
      if (!before(bound, key)) {
        const int place = atomicAdd(&sh.n_found, 1);
        if (place < kLpCandidates) sh.found[place] = key;
      }
    };
    for (int64_t w = threadIdx.x; w < total; w += kLpThreads) {
      const int64_t thread = sh.threads[w / per], part = w % per, j = thread + part * kLpThreads;
      if (part == per - 1) {   // the thread's element around the vectors
        if (thread < around) {
          const int64_t at = thread < head ? thread : thread + nvec * V;
          offer(to_acc(z0[at]), at);
        }
      } else if (j < nvec) {
        const Vec<T, V> v = load_vec_nt_any<T, V>(z0 + head + j * V);
#pragma unroll
        for (int e = 0; e < V; ++e) offer(vec_get(v, e), head + j * V + e);
      }
    }
    __syncthreads();
    done = sh.n_found >= top && sh.n_found <= kLpCandidates;
  }
  if (done) {
    lp_rank(sh.found, sh.n_found, top, sh.best);
    return;
  }
  TopKey<A> last{static_cast<typename TopKey<A>::U>(~static_cast<typename TopKey<A>::U>(0)), 0};
  bool any = false;   // whether `last` is a class found
  for (int r = 0; r < top; ++r) {
    TopKey<A> key = no_key<A>();
    for (int64_t i = threadIdx.x; i < n; i += kLpThreads) {
      const TopKey<A> k{rank_bits(to_acc(z0[i])), first + static_cast<uint32_t>(i)};
      if ((!any || before(last, k)) && before(k, key)) key = k;
    }
#pragma unroll
    for (int mask = 1; mask < kWave; mask <<= 1) {
      const TopKey<A> o = shuffled(key, mask);
      if (before(o, key)) key = o;
    }
    if (threadIdx.x % kWave == 0) sh.wave[threadIdx.x / kWave] = key;
    __syncthreads();
    key = sh.wave[0];
#pragma unroll
    for (int w = 1; w < kLpWaves; ++w)
      if (before(sh.wave[w], key)) key = sh.wave[w];
    if (threadIdx.x == 0) sh.best[r] = key;
    last = key;
    any = true;
    __syncthreads();
  }
}

// Classes at z_0 = -inf: their higher orders become zero, so that what they hold does not reach the sums.
template <typename T, int K, int U>
__device__ __forceinline__ void lp_masked(Vec<T, VecWidth<T>::value> (&v)[U][K + 1]) {
  using A = typename AccOf<T>::type;
  constexpr int V = VecWidth<T>::value;
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (vec_get(v[u][0], e) == A(-__builtin_huge_val())) {
#pragma unroll
        for (int k = 1; k <= K; ++k) v[u][k].v[e] = T{};
      }
}

template <typename T, int K, bool CAP, bool TOP>
__global__ __launch_bounds__(kLpThreads) void token_log_probs_series_kernel(const LpKernelArgs<T> a) {
  using A = typename AccOf<T>::type;
  constexpr int V = VecWidth<T>::value;
  constexpr A kNegInf = -__builtin_huge_val();
  __shared__ LpState<A, K> red[kLpWaves];
  __shared__ A series[K + 1];
  const uint32_t split = blockIdx.x % a.splits;
  const int64_t row = blockIdx.x / a.splits;
  const int64_t y = a.tokens[row];
  A rho[K + 1];
  lp_shift<T, K, CAP>(a, row, rho);   // (its loads beside the token's, not after it)
  if (y == a.ignore_index) {
    if (a.splits == 1) lp_ignored<T, K, TOP>(a, row);
    return;
  }
  const int64_t c0 = split * a.piece < a.classes ? split * a.piece : a.classes;
  const int64_t n = c0 + a.piece < a.classes ? a.piece : a.classes - c0;
  const int64_t base = row * a.row_stride + c0;
  LpState<A, K> st;
  lp_clear(st);
  A raw_max = kNegInf;   // the maximum before the softcap
  A best = kNegInf;
  uint32_t best_class = 0xffffffffu;

  // A batch of vectors: the maximum first, then every class.
  auto batch = [&](auto& v, const uint32_t* at) {
    constexpr int U = std::extent_v<std::remove_reference_t<decltype(v)>>;
    A hi = CAP ? A(-1e30) : kNegInf, lo = A(0);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const A x = vec_get(v[u][0], e);
        hi = fmax(hi, x);
        if (!CAP) lo = fmin(lo, x);
      }
    if (!CAP && lo == kNegInf) lp_masked<T, K, U>(v);
    if (hi > raw_max) {
      raw_max = hi;
      lp_rebase(st, CAP ? a.cap * tanh_acc(hi * a.inv_cap) : hi);
    }
    if (raw_max == kNegInf) {   // (a share of -inf and NaN so far: the row's sum is no number then)
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (const A x = vec_get(v[u][0], e); x != x) st.S[0] = x;
      return;
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        A x[K + 1];
#pragma unroll
        for (int k = 0; k <= K; ++k) x[k] = vec_get(v[u][k], e);
        if constexpr (TOP) {
          const bool larger = x[0] > best;
          best = larger ? x[0] : best;
          best_class = larger ? at[u] + e : best_class;
        }
        if constexpr (CAP) softcap_series<A, K>(x, a.cap, a.inv_cap);
#pragma unroll
        for (int k = 1; k <= K; ++k) x[k] -= rho[k];
        lp_add(st, x);
      }
  };

  constexpr int U = 2;
  const int64_t head = lp_head(a.z.p[0] + base, n), nvec = (n - head) / V;
  int64_t j = threadIdx.x;
  for (; j + (U - 1) * kLpThreads < nvec; j += U * kLpThreads) {
    Vec<T, V> v[U][K + 1];
    uint32_t at[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      at[u] = static_cast<uint32_t>(c0 + head + (j + u * kLpThreads) * V);
#pragma unroll
      for (int k = 0; k <= K; ++k) v[u][k] = load_vec_nt_any<T, V>(a.z.p[k] + base + head + (j + u * kLpThreads) * V);
    }
    batch(v, at);
  }
  for (; j < nvec; j += kLpThreads) {
    Vec<T, V> v[1][K + 1];
    const uint32_t at[1] = {static_cast<uint32_t>(c0 + head + j * V)};
#pragma unroll
    for (int k = 0; k <= K; ++k) v[0][k] = load_vec_nt_any<T, V>(a.z.p[k] + base + head + j * V);
    batch(v, at);
  }
  for (int64_t i = threadIdx.x; i < n - nvec * V; i += kLpThreads) {   // the elements around the vectors
    const int64_t at = i < head ? i : i + nvec * V;
    A x[K + 1];
#pragma unroll
    for (int k = 0; k <= K; ++k) x[k] = to_acc(a.z.p[k][base + at]);
    if (TOP && (x[0] > best || (x[0] == best && c0 + at < best_class))) {
      best = x[0];
      best_class = static_cast<uint32_t>(c0 + at);
    }
    if (!CAP && x[0] == kNegInf) continue;
    if constexpr (CAP) softcap_series<A, K>(x, a.cap, a.inv_cap);
    if (x[0] > st.m) lp_rebase(st, x[0]);
#pragma unroll
    for (int k = 1; k <= K; ++k) x[k] -= rho[k];
    lp_add(st, x);
  }

  lp_join_wave(st);
  if (threadIdx.x % kWave == 0) red[threadIdx.x / kWave] = st;
  __syncthreads();
  A M = red[0].m;
#pragma unroll
  for (int w = 1; w < kLpWaves; ++w) M = fmax(M, red[w].m);
  lp_clear(st);
  st.m = M;
#pragma unroll
  for (int w = 0; w < kLpWaves; ++w) {
    LpState<A, K> part = red[w];
    lp_rebase(part, M);
#pragma unroll
    for (int k = 0; k <= K; ++k) {
      st.S[k] += part.S[k];
      st.W[k] += part.W[k];
    }
  }
  if constexpr (TOP) {
    __shared__ LpTopShared<A> sh;
    const TopKey<A> own = best_class == 0xffffffffu ? no_key<A>() : TopKey<A>{rank_bits(best), best_class};
    // (S_0 is no number where a logit is none, which a thread's maximum does not show)
    lp_select<T>(a.z.p[0] + base, n, head, static_cast<uint32_t>(c0), own, st.S[0] != st.S[0], a.top, sh);
    if (a.splits == 1) {
      lp_finish<T, K, CAP, true>(a, row, y, st, rho, sh.best, series);
    } else {
      const int64_t at = static_cast<int64_t>(blockIdx.x) * a.top + threadIdx.x;
      if (static_cast<int>(threadIdx.x) < a.top) {
        a.key_bits[at] = sh.best[threadIdx.x].v;
        a.key_class[at] = sh.best[threadIdx.x].i;
      }
    }
  } else if (a.splits == 1) {
    lp_finish<T, K, CAP, false>(a, row, y, st, rho, nullptr, series);
  }
  if (a.splits > 1 && threadIdx.x == 0) {
    A* out = a.partial + static_cast<int64_t>(blockIdx.x) * (3 * K + 3);
    out[0] = st.m;
#pragma unroll
    for (int k = 0; k <= K; ++k) {
      out[1 + k] = st.S[k];
      out[2 + K + k] = st.W[k];
      if (k > 0) out[2 + 2 * K + k] = rho[k];
    }
  }
}

template <typename A>
struct LpJoinShared {
  TopKey<A> group[64], bound, best[kLpMaxTop], found[kLpMaxSplits * kLpMaxTop];
  int n_threads, n_found;
};

// A row's pieces joined: a lane of every wave takes a piece's state; of the pieces' alternatives those that reach
// the bound of the threads' largest are ranked. (Ranking all 64 x 20 of 8 rows that reached the largest of the
// pieces' last ones, about half of them: 82 us.)
template <typename T, int K, bool CAP, bool TOP>
__global__ __launch_bounds__(kLpThreads) void token_log_probs_join_kernel(const LpKernelArgs<T> a) {
  using A = typename AccOf<T>::type;
  __shared__ A series[K + 1];
  const int64_t row = blockIdx.x;
  const int64_t y = a.tokens[row];
  if (y == a.ignore_index) {
    lp_ignored<T, K, TOP>(a, row);
    return;
  }
  LpState<A, K> st;
  lp_clear(st);
  A rho[K + 1];
  const uint32_t lane = threadIdx.x % kWave;
  const A* in = a.partial + (row * a.splits + (lane < a.splits ? lane : 0)) * (3 * K + 3);
  if (lane < a.splits) {
    st.m = in[0];
#pragma unroll
    for (int k = 0; k <= K; ++k) {
      st.S[k] = in[1 + k];
      st.W[k] = in[2 + K + k];
    }
  }
  rho[0] = A(0);
#pragma unroll
  for (int k = 1; k <= K; ++k) rho[k] = in[2 + 2 * K + k];
  lp_join_wave(st);
  if constexpr (TOP) {
    __shared__ LpJoinShared<A> sh;
    const auto* bits = a.key_bits + row * a.splits * a.top;
    const uint32_t* classes = a.key_class + row * a.splits * a.top;
    const int n = static_cast<int>(a.splits) * a.top;
    constexpr int kEach = kLpMaxSplits * kLpMaxTop / kLpThreads;
    TopKey<A> mine[kEach], own = no_key<A>();
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int at = threadIdx.x + i * kLpThreads;
      mine[i] = at < n ? TopKey<A>{bits[at], classes[at]} : no_key<A>();
      if (before(mine[i], own)) own = mine[i];
    }
    const TopKey<A> bound = lp_bound(own, a.top, sh);   // (none: every key is ranked)
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      if (mine[i].v != 0 && !before(bound, mine[i])) sh.found[atomicAdd(&sh.n_found, 1)] = mine[i];
    __syncthreads();
    lp_rank(sh.found, sh.n_found, a.top, sh.best);
    lp_finish<T, K, CAP, true>(a, row, y, st, rho, sh.best, series);
  } else {
    lp_finish<T, K, CAP, false>(a, row, y, st, rho, nullptr, series);
  }
}

template <typename T, int K>
static int launch_log_probs_k(const LogProbArgs& in) {
  using A = typename AccOf<T>::type;
  constexpr int V = VecWidth<T>::value;
  LpKernelArgs<T> a{};
  for (int k = 0; k <= K; ++k) {
    a.z.p[k] = static_cast<const T*>(in.z[k]);
    a.log_probs.p[k] = static_cast<A*>(in.log_probs[k]);
    a.entropy.p[k] = static_cast<A*>(in.entropy[k]);
    a.lse.p[k] = static_cast<A*>(in.lse[k]);
    if (in.top > 0) a.top_log_probs.p[k] = static_cast<A*>(in.top_log_probs[k]);
  }
  const int64_t splits = log_prob_splits(in.rows, in.classes, sizeof(T), false);
  a.classes = in.classes;
  a.row_stride = in.row_stride;
  a.splits = static_cast<uint32_t>(splits);
  a.piece = splits == 1 ? in.classes : ((in.classes + splits - 1) / splits + V - 1) / V * V;
  a.tokens = in.tokens;
  a.ignore_index = in.ignore_index;
  const bool cap = in.softcap > 0.0;
  a.cap = cap ? static_cast<A>(in.softcap) : A(1);
  a.inv_cap = A(1) / a.cap;
  a.top = in.top;
  a.top_tokens = in.top_tokens;
  if (splits > 1) {   // [key bits | partial states | key classes]
    char* w = static_cast<char*>(in.workspace);
    a.key_bits = reinterpret_cast<typename TopKey<A>::U*>(w);
    w += sizeof(A) * in.rows * splits * in.top;
    a.partial = reinterpret_cast<A*>(w);
    w += sizeof(A) * in.rows * splits * (3 * K + 3);
    a.key_class = reinterpret_cast<uint32_t*>(w);
  }
  const dim3 grid(static_cast<uint32_t>(in.rows * splits)), block(kLpThreads);
#define PT_LP_LAUNCH(CP, TP)                                                                                \
  do {                                                                                                      \
    token_log_probs_series_kernel<T, K, CP, TP><<<grid, block, 0, in.stream>>>(a);                          \
    PT_LAUNCH_CHECK();                                                                                      \
    if (splits > 1) token_log_probs_join_kernel<T, K, CP, TP><<<dim3(in.rows), block, 0, in.stream>>>(a);   \
    PT_LAUNCH_CHECK();                                                                                      \
  } while (0)
  if (in.top > 0) {
    if (cap) PT_LP_LAUNCH(true, true);
    else PT_LP_LAUNCH(false, true);
  } else {
    if (cap) PT_LP_LAUNCH(true, false);
    else PT_LP_LAUNCH(false, false);
  }
#undef PT_LP_LAUNCH
  return PT_OK;
}

// ---------------------------------------------------------------------------
// Gradient series: with l = z - lse, p = exp(l), c the sum of the row's log-probability cotangents and c_H
// the entropy's,
//   dz = -p (*) (c + c_H (*) (l + H)) + (the log-probability cotangents at their classes),
// times the softcap's derivative series. A block streams its classes once and writes dz; the classes with
// cotangents of their own are written again afterwards, each by one thread that adds all of theirs.
template <typename T>
struct LpBwdKernelArgs {
  using A = typename AccOf<T>::type;
  CPtrs<T> z;
  int64_t classes, row_stride, piece;
  uint32_t splits;
  const int64_t* tokens;
  int64_t ignore_index;
  A cap, inv_cap;
  int top;
  const int64_t* top_tokens;
  CPtrs<A> lse, entropy, cot_log_probs, cot_entropy, cot_top;   // cotangents: null for zero
  MPtrs<T> dz;
};

template <typename A, int K, bool CAP, bool ENT>
__device__ __forceinline__ void lp_bwd_class(const A (&x)[K + 1], const A (&lse)[K + 1], const A (&c)[K + 1],
                                             const A (&ch)[K + 1], A cap, A inv_cap, const A (&own)[K + 1], A (&dz)[K + 1]) {
  A l[K + 1], dt[K + 1], p[K + 1], q[K + 1];
#pragma unroll
  for (int k = 0; k <= K; ++k) l[k] = x[k];
  if constexpr (CAP) softcap_series<A, K>(l, cap, inv_cap, dt);
#pragma unroll
  for (int k = 0; k <= K; ++k) l[k] -= lse[k];
  p[0] = exp_acc(l[0]);
#pragma unroll
  for (int k = 1; k <= K; ++k) {
    A s = A(0);
#pragma unroll
    for (int j = 1; j <= k; ++j) s = j == 1 ? l[j] * p[k - j] : fma(A(j) * l[j], p[k - j], s);
    p[k] = s * (A(1) / A(k));
  }
#pragma unroll
  for (int k = 0; k <= K; ++k) q[k] = c[k];
  if constexpr (ENT) {
    l[0] = fmax(l[0], lp_floor<A>());   // (p_0 is zero below)
#pragma unroll
    for (int k = 0; k <= K; ++k)
#pragma unroll
      for (int i = 0; i <= k; ++i) q[k] = fma(ch[i], l[k - i], q[k]);
  }
#pragma unroll
  for (int k = 0; k <= K; ++k) {
    A s = own[k];
#pragma unroll
    for (int i = 0; i <= k; ++i) s = fma(-p[i], q[k - i], s);
    dz[k] = s;
  }
  if constexpr (CAP) {
    A r[K + 1];
    cauchy_mul<A, K>(dz, dt, r);
#pragma unroll
    for (int k = 0; k <= K; ++k) dz[k] = r[k];
  }
}

template <typename T, int K, bool CAP, bool ENT>
__global__ __launch_bounds__(kLpThreads) void token_log_probs_bwd_kernel(const LpBwdKernelArgs<T> a) {
  using A = typename AccOf<T>::type;
  constexpr int V = VecWidth<T>::value;
  constexpr A kNegInf = -__builtin_huge_val();
  __shared__ int64_t own_class[kLpMaxTop + 1];
  const uint32_t split = blockIdx.x % a.splits;
  const int64_t row = blockIdx.x / a.splits;
  const int64_t y = a.tokens[row];
  const int64_t c0 = split * a.piece < a.classes ? split * a.piece : a.classes;
  const int64_t n = c0 + a.piece < a.classes ? a.piece : a.classes - c0;
  const int64_t base = row * a.row_stride + c0, out = row * a.classes + c0;
  const int64_t head = lp_head(a.dz.p[0] + out, n), nvec = (n - head) / V;
  if (y == a.ignore_index) {
    const Vec<T, V> zero{};
    for (int64_t j = threadIdx.x; j < nvec; j += kLpThreads)
#pragma unroll
      for (int k = 0; k <= K; ++k) store_vec_nt_any<T, V>(a.dz.p[k] + out + head + j * V, zero);
    for (int64_t i = threadIdx.x; i < n - nvec * V; i += kLpThreads)
#pragma unroll
      for (int k = 0; k <= K; ++k) a.dz.p[k][out + (i < head ? i : i + nvec * V)] = T{};
    return;
  }
  const bool valid = y >= 0 && y < a.classes;
  A lse[K + 1], c[K + 1], ch[K + 1], none[K + 1];
#pragma unroll
  for (int k = 0; k <= K; ++k) {
    lse[k] = a.lse.p[k][row];
    // (NaN through the log probability of a token that is no class)
    c[k] = a.cot_log_probs.p[0] == nullptr ? A(0) : valid ? a.cot_log_probs.p[k][row] : A(__builtin_nan(""));
    ch[k] = ENT ? a.cot_entropy.p[k][row] : A(0);
    none[k] = A(0);
    if (a.cot_top.p[0] != nullptr)
      for (int j = 0; j < a.top; ++j) c[k] += a.cot_top.p[k][row * a.top + j];
  }
  if constexpr (ENT) {   // c + c_H (*) H
    A H[K + 1];
#pragma unroll
    for (int k = 0; k <= K; ++k) H[k] = a.entropy.p[k][row];
#pragma unroll
    for (int k = 0; k <= K; ++k)
#pragma unroll
      for (int i = 0; i <= k; ++i) c[k] = fma(ch[i], H[k - i], c[k]);
  }
  auto batch = [&](auto& v, int64_t j0) {
    constexpr int U = std::extent_v<std::remove_reference_t<decltype(v)>>;
    A lo = A(0);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < V; ++e) lo = fmin(lo, vec_get(v[u][0], e));
    if (!CAP && lo == kNegInf) lp_masked<T, K, U>(v);
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int e = 0; e < V; e += 2) {
        A r[2][K + 1];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          A x[K + 1];
#pragma unroll
          for (int k = 0; k <= K; ++k) x[k] = vec_get(v[u][k], e + h);
          lp_bwd_class<A, K, CAP, ENT>(x, lse, c, ch, a.cap, a.inv_cap, none, r[h]);
        }
#pragma unroll
        for (int k = 0; k <= K; ++k) vec_put2(v[u][k], e, r[0][k], r[1][k]);
      }
#pragma unroll
      for (int k = 0; k <= K; ++k) store_vec_nt_any<T, V>(a.dz.p[k] + out + head + (j0 + u * kLpThreads) * V, v[u][k]);
    }
  };
  auto single = [&](int64_t at, const A (&own)[K + 1]) {
    A x[K + 1], r[K + 1];
#pragma unroll
    for (int k = 0; k <= K; ++k) x[k] = to_acc(a.z.p[k][base + at]);
    if (!CAP && x[0] == kNegInf) {
#pragma unroll
      for (int k = 1; k <= K; ++k) x[k] = A(0);
    }
    lp_bwd_class<A, K, CAP, ENT>(x, lse, c, ch, a.cap, a.inv_cap, own, r);
#pragma unroll
    for (int k = 0; k <= K; ++k) a.dz.p[k][out + at] = from_acc<T>(r[k]);
  };
  constexpr int U = 2;
  int64_t j = threadIdx.x;
  for (; j + (U - 1) * kLpThreads < nvec; j += U * kLpThreads) {
    Vec<T, V> v[U][K + 1];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int k = 0; k <= K; ++k) v[u][k] = load_vec_nt_any<T, V>(a.z.p[k] + base + head + (j + u * kLpThreads) * V);
    batch(v, j);
  }
  for (; j < nvec; j += kLpThreads) {
    Vec<T, V> v[1][K + 1];
#pragma unroll
    for (int k = 0; k <= K; ++k) v[0][k] = load_vec_nt_any<T, V>(a.z.p[k] + base + head + j * V);
    batch(v, j);
  }
  for (int64_t i = threadIdx.x; i < n - nvec * V; i += kLpThreads) single(i < head ? i : i + nvec * V, none);

  const int owners = a.cot_top.p[0] != nullptr ? a.top + 1 : 1;
  const int me = threadIdx.x;
  if (me < owners) {
    const int64_t cls = me == 0 ? y : a.top_tokens[row * a.top + me - 1];
    own_class[me] = cls >= c0 && cls < c0 + n ? cls : -1;
  }
  __syncthreads();   // (and the block's stores above are done before those below)
  if (me < owners && own_class[me] >= 0) {
    bool first = true;
    for (int o = 0; o < me; ++o) first = first && own_class[o] != own_class[me];
    if (first) {
      A own[K + 1];
#pragma unroll
      for (int k = 0; k <= K; ++k) own[k] = A(0);
      for (int o = me; o < owners; ++o)
        if (own_class[o] == own_class[me]) {
#pragma unroll
          for (int k = 0; k <= K; ++k) {
            if (o == 0)
              own[k] += a.cot_log_probs.p[0] != nullptr ? a.cot_log_probs.p[k][row] : A(0);
            else
              own[k] += a.cot_top.p[k][row * a.top + o - 1];
          }
        }
      single(own_class[me] - c0, own);
    }
  }
}

template <typename T, int K>
static int launch_log_probs_bwd_k(const LogProbBwdArgs& in) {
  using A = typename AccOf<T>::type;
  constexpr int V = VecWidth<T>::value;
  LpBwdKernelArgs<T> a{};
  for (int k = 0; k <= K; ++k) {
    a.z.p[k] = static_cast<const T*>(in.z[k]);
    a.dz.p[k] = static_cast<T*>(in.dz[k]);
    a.lse.p[k] = static_cast<const A*>(in.lse[k]);
    a.entropy.p[k] = static_cast<const A*>(in.entropy[k]);
    if (in.cot_log_probs != nullptr) a.cot_log_probs.p[k] = static_cast<const A*>(in.cot_log_probs[k]);
    if (in.cot_entropy != nullptr) a.cot_entropy.p[k] = static_cast<const A*>(in.cot_entropy[k]);
    if (in.cot_top_log_probs != nullptr && in.top > 0) a.cot_top.p[k] = static_cast<const A*>(in.cot_top_log_probs[k]);
  }
  const int64_t splits = log_prob_splits(in.rows, in.classes, sizeof(T), true);
  a.classes = in.classes;
  a.row_stride = in.row_stride;
  a.splits = static_cast<uint32_t>(splits);
  a.piece = splits == 1 ? in.classes : ((in.classes + splits - 1) / splits + V - 1) / V * V;
  a.tokens = in.tokens;
  a.ignore_index = in.ignore_index;
  const bool cap = in.softcap > 0.0;
  a.cap = cap ? static_cast<A>(in.softcap) : A(1);
  a.inv_cap = A(1) / a.cap;
  a.top = in.top;
  a.top_tokens = in.top_tokens;
  const dim3 grid(static_cast<uint32_t>(in.rows * splits)), block(kLpThreads);
  if (in.cot_entropy != nullptr) {
    if (cap) token_log_probs_bwd_kernel<T, K, true, true><<<grid, block, 0, in.stream>>>(a);
    else token_log_probs_bwd_kernel<T, K, false, true><<<grid, block, 0, in.stream>>>(a);
  } else {
    if (cap) token_log_probs_bwd_kernel<T, K, true, false><<<grid, block, 0, in.stream>>>(a);
    else token_log_probs_bwd_kernel<T, K, false, false><<<grid, block, 0, in.stream>>>(a);
  }
  PT_LAUNCH_CHECK();
  return PT_OK;
}

#define PT_LP_DEGREES(launch)                                                          \
  switch (in.degree) {                                                                 \
    case 0: return launch<T, 0>(in);                                                   \
    case 1: return launch<T, 1>(in);                                                   \
    case 2: return launch<T, 2>(in);                                                   \
    case 3: return launch<T, 3>(in);                                                   \
    case 4: return launch<T, 4>(in);                                                   \
    case 5: return launch<T, 5>(in);                                                   \
    case 6: return launch<T, 6>(in);                                                   \
    case 7: return launch<T, 7>(in);                                                   \
    case 8: return launch<T, 8>(in);                                                   \
    default: break;                                                                    \
  }                                                                                    \
  pt_host::set_error("token log-prob series: degree outside 0..PT_MAX_DEGREE");        \
  return PT_UNSUPPORTED

template <typename T>
int launch_log_probs(const LogProbArgs& in) {
  PT_LP_DEGREES(launch_log_probs_k);
}

template <typename T>
int launch_log_probs_bwd(const LogProbBwdArgs& in) {
  PT_LP_DEGREES(launch_log_probs_bwd_k);
}

}  // namespace pt
