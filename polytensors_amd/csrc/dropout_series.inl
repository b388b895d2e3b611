// Dropout of a series: y_k = x_k m / (1 - p) for every order k with one 0/1 mask m, which is a function
// of the seed and the element's index alone and is never stored; the gradient is the same operation on the
// cotangent.
//
// m comes from the counter-based generator Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel
// random numbers: as easy as 1, 2, 3", SC 2011): block c = i / 4 is the ten-round encryption of the
// counter (c mod 2^32, c / 2^32, 0, 0) under the seed's two words, element i has word i mod 4, and is
// kept where that word is at least p 2^32. The index is the element's place in row-major order, so the
// mask does not depend on the launch shape, the alignment or the type.
//
// A thread takes one 16-byte vector of every order (two in float64, so that a generator block is drawn
// once) and one or two generator blocks for all of them; every load is issued before the generator's 20 wide products.
// HBM bounds it: 8192 x 4096 bfloat16 at degree 4 116 us, 5.8 TB/s (a stream over the same buffers 112); 8192 x 768
// float32 at degree 3 35 us, 5.7 TB/s (35).
#pragma once

#include "dropout_series.h"

namespace pt {

constexpr int kDropoutThreads = 256;

struct Philox {
  uint32_t w[4];
};

__device__ __forceinline__ Philox philox(uint64_t block, uint64_t seed) {
  uint32_t k0 = static_cast<uint32_t>(seed), k1 = static_cast<uint32_t>(seed >> 32);
  uint32_t c0 = static_cast<uint32_t>(block), c1 = static_cast<uint32_t>(block >> 32), c2 = 0, c3 = 0;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = static_cast<uint64_t>(c0) * 0xD2511F53u, b = static_cast<uint64_t>(c2) * 0xCD9E8D57u;
    c0 = static_cast<uint32_t>(b >> 32) ^ c1 ^ k0;
    c1 = static_cast<uint32_t>(b);
    c2 = static_cast<uint32_t>(a >> 32) ^ c3 ^ k1;
    c3 = static_cast<uint32_t>(a);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return {{c0, c1, c2, c3}};
}

// x scale rounded to the arithmetic type, then to the storage type, wherever the element lies: left alone, the
// compiler forms some float16 products with v_fma_mixlo_f16, which rounds once and differs in ties.
__device__ __forceinline__ float dropout_scaled(float x, float scale) {
  float v = x * scale;
  asm("" : "+v"(v));
  return v;
}
__device__ __forceinline__ double dropout_scaled(double x, double scale) { return x * scale; }

// all: p = 1, everything dropped (the threshold 2^32 has no 32-bit word). A dropped element is zero
// whatever it held.
template <typename T, int N>
__global__ __launch_bounds__(kDropoutThreads) void dropout_series_kernel(
    CPtrs<T> x, MPtrs<T> y, int64_t numel, uint32_t threshold, bool all, typename AccOf<T>::type scale,
    const int64_t* __restrict__ seed_ptr) {
  using A = typename AccOf<T>::type;
  constexpr int V = VecWidth<T>::value;
  constexpr int E = V < 4 ? 4 : V;   // elements a thread
  const int64_t i0 = (static_cast<int64_t>(blockIdx.x) * kDropoutThreads + threadIdx.x) * E;
  if (i0 >= numel) return;
  const uint64_t seed = static_cast<uint64_t>(*seed_ptr);
  const bool whole = i0 + E <= numel;
  Vec<T, V> a[N][E / V];
  if (whole) {
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
      for (int h = 0; h < E / V; ++h) a[k][h] = load_vec_nt_any<T, V>(x.p[k] + i0 + h * V);
  }
  bool keep[E];
#pragma unroll
  for (int b = 0; b < E / 4; ++b) {
    const Philox w = philox(static_cast<uint64_t>(i0 / 4 + b), seed);
#pragma unroll
    for (int e = 0; e < 4; ++e) keep[4 * b + e] = !all && w.w[e] >= threshold;
  }
  if (whole) {
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
      for (int h = 0; h < E / V; ++h) {
#pragma unroll
        for (int e = 0; e < V; e += 2)
          vec_put2(a[k][h], e, keep[h * V + e] ? dropout_scaled(vec_get(a[k][h], e), scale) : A(0),
                   keep[h * V + e + 1] ? dropout_scaled(vec_get(a[k][h], e + 1), scale) : A(0));
        store_vec_nt_any<T, V>(y.p[k] + i0 + h * V, a[k][h]);
      }
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (i0 + e < numel) {
#pragma unroll
        for (int k = 0; k < N; ++k)
          y.p[k][i0 + e] = from_acc<T>(keep[e] ? dropout_scaled(to_acc(x.p[k][i0 + e]), scale) : A(0));
      }
    }
  }
}

template <typename T, int N>
static int launch_dropout_n(const DropoutArgs& a, int from) {
  using A = typename AccOf<T>::type;
  constexpr int V = VecWidth<T>::value;
  constexpr int64_t E = V < 4 ? 4 : V;
  CPtrs<T> x{};
  MPtrs<T> y{};
  for (int k = 0; k < N; ++k) {
    x.p[k] = static_cast<const T*>(a.x[from + k]);
    y.p[k] = static_cast<T*>(a.y[from + k]);
  }
  const int64_t blocks = ((a.numel + E - 1) / E + kDropoutThreads - 1) / kDropoutThreads;
  PT_REQUIRE(blocks <= INT32_MAX, PT_UNSUPPORTED, "dropout series: more elements than a launch holds");
  const bool all = a.p >= 1.0;
  const uint32_t threshold = all ? 0u : static_cast<uint32_t>(a.p * 4294967296.0);
  dropout_series_kernel<T, N><<<dim3(blocks), dim3(kDropoutThreads), 0, a.stream>>>(
      x, y, a.numel, threshold, all, all ? A(0) : static_cast<A>(1.0 / (1.0 - a.p)), a.seed);
  PT_LAUNCH_CHECK();
  return PT_OK;
}

// Orders above kMaxOrders take launches of their own, which draw the same mask again.
template <typename T>
int launch_dropout(const DropoutArgs& a) {
  for (int from = 0; from < a.orders; from += kMaxOrders) {
    int status = PT_OK;
    switch (a.orders - from < kMaxOrders ? a.orders - from : kMaxOrders) {
      case 1: status = launch_dropout_n<T, 1>(a, from); break;
      case 2: status = launch_dropout_n<T, 2>(a, from); break;
      case 3: status = launch_dropout_n<T, 3>(a, from); break;
      case 4: status = launch_dropout_n<T, 4>(a, from); break;
      case 5: status = launch_dropout_n<T, 5>(a, from); break;
      case 6: status = launch_dropout_n<T, 6>(a, from); break;
      case 7: status = launch_dropout_n<T, 7>(a, from); break;
      case 8: status = launch_dropout_n<T, 8>(a, from); break;
      default: status = launch_dropout_n<T, 9>(a, from); break;
    }
    if (status != PT_OK) return status;
  }
  return PT_OK;
}

}  // namespace pt
