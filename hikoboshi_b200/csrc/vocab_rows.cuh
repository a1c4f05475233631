// Shared device code of the operators on vocabulary rows (vocab_sample.cu,
// vocab_top.cu, vocab_distill.cu).
//
// A row is V logits of one position, f32, fp16 or bf16.  A cluster of C CTAs
// (C = 1, 2, 4 or 8) holds one row in its shared memory, CTA c the slice
// [c * chunk, min(V, (c + 1) * chunk)), so every pass after the first reads
// shared memory and the row crosses HBM once.  C grows with V (a slice has to
// fit) and when there are few rows (a row is then read by more SMs).
//
// Slices are kept in the 16-byte phase of their global addresses: element i of
// the slice sits at index ph + i, so whole 16-byte vectors are copied by
// cp.async whatever the row's alignment, and every pass reads 16-byte vectors.
// The ph elements in front and those behind the slice up to the vector's end
// hold -inf, which no operator selects and whose weight is zero.
#pragma once

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <math_constants.h>
#include <stdint.h>

#include "common.cuh"

namespace hkb {
namespace vocab {

namespace cg = cooperative_groups;

constexpr int kMaxThreads = 512;
constexpr int kMaxWarps = kMaxThreads / 32;
constexpr int kMaxCluster = 8;

__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(__half x) { return __half2float(x); }
__device__ __forceinline__ float widen(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T>
__device__ __forceinline__ T narrow(float x);
template <>
__device__ __forceinline__ float narrow<float>(float x) {
  return x;
}
template <>
__device__ __forceinline__ __half narrow<__half>(float x) {
  return __float2half_rn(x);
}
template <>
__device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}

// 16 bytes of a row, as 32-bit words: 16-bit elements stay packed in pairs.
template <typename T>
struct alignas(16) Vec {
  static constexpr int kN = 16 / (int)sizeof(T);
  uint32_t w[4];

  __device__ __forceinline__ float at(int e) const;    // element e, widened
  __device__ __forceinline__ void clear(int e);        // element e = -inf
  __device__ __forceinline__ float2 pair(int i) const; // elements 2 i and 2 i + 1
  __device__ __forceinline__ void set_pair(int i, float2 y);
  __device__ __forceinline__ float largest() const;    // a NaN is less than any number
};

template <>
__device__ __forceinline__ float Vec<float>::at(int e) const {
  return __uint_as_float(w[e]);
}
template <>
__device__ __forceinline__ float Vec<__half>::at(int e) const {
  return __half2float(__ushort_as_half((unsigned short)(w[e >> 1] >> (16 * (e & 1)))));
}
template <>
__device__ __forceinline__ float Vec<__nv_bfloat16>::at(int e) const {
  return __uint_as_float(e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
}
template <>
__device__ __forceinline__ void Vec<float>::clear(int e) {
  w[e] = 0xff800000u;
}
template <>
__device__ __forceinline__ void Vec<__half>::clear(int e) {
  w[e >> 1] = e & 1 ? (w[e >> 1] & 0xffffu) | 0xfc000000u : (w[e >> 1] & 0xffff0000u) | 0xfc00u;
}
template <>
__device__ __forceinline__ void Vec<__nv_bfloat16>::clear(int e) {
  w[e >> 1] = e & 1 ? (w[e >> 1] & 0xffffu) | 0xff800000u : (w[e >> 1] & 0xffff0000u) | 0xff80u;
}
template <>
__device__ __forceinline__ float2 Vec<float>::pair(int i) const {
  return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
}
template <>
__device__ __forceinline__ float2 Vec<__half>::pair(int i) const {
  return __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
}
template <>
__device__ __forceinline__ float2 Vec<__nv_bfloat16>::pair(int i) const {
  return make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
}
template <>
__device__ __forceinline__ void Vec<float>::set_pair(int i, float2 y) {
  w[2 * i] = __float_as_uint(y.x);
  w[2 * i + 1] = __float_as_uint(y.y);
}
template <>
__device__ __forceinline__ void Vec<__half>::set_pair(int i, float2 y) {
  const __half2 h = __float22half2_rn(y);
  w[i] = *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ void Vec<__nv_bfloat16>::set_pair(int i, float2 y) {
  const __nv_bfloat162 h = __float22bfloat162_rn(y);
  w[i] = *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ float Vec<float>::largest() const {
  return fmaxf(fmaxf(at(0), at(1)), fmaxf(at(2), at(3)));
}
template <>
__device__ __forceinline__ float Vec<__half>::largest() const {
  const __half2* h = reinterpret_cast<const __half2*>(w);
  const float2 m = __half22float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
  return fmaxf(m.x, m.y);
}
template <>
__device__ __forceinline__ float Vec<__nv_bfloat16>::largest() const {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(w);
  const float2 m = __bfloat1622float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
  return fmaxf(m.x, m.y);
}

// Order-preserving key of a value: a < b <=> key(a) < key(b); -0 and +0 share
// one key.  NaN never reaches it (rows are cleaned on load).
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
constexpr uint32_t kKeyNegInf = 0x007fffffu;  // order_key(-inf)

// 2^t for t <= 0 in 64 bits by the table method (P. T. P. Tang, "Table-driven
// implementation of the exponential function in IEEE floating-point
// arithmetic", 1989): t = n + j/16 + r with |r| <= 1/32, 2^t = 2^n 2^(j/16) 2^r,
// the last by its Taylor series to the 6th power (remainder 0.0217^7 / 5040 =
// 4.5e-16).  0 below 2^-1020.  The choice of a token compares sums of such
// weights with each other; in 64 bits a sum over 2^18 tokens keeps 1e-13, so
// the token is the formula's unless the uniform lies that close to a border.
//
// The 16 table entries fill the 32 banks of shared memory once, so lanes that
// look up different entries never conflict.  11 operations on the 64-bit pipe
// with the exponent's, against 18 for a series without the table.
struct Exp2Table {
  double v[16];
  __device__ __forceinline__ void fill() {
    if (threadIdx.x < 16) v[threadIdx.x] = exp2((double)threadIdx.x / 16.0);
  }
  __device__ __forceinline__ double operator()(double t) const {
    const double shift = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to an integer
    const double tn = fma(t, 16.0, shift);
    const int n = __double2loint(tn);
    const double r = fma(__dsub_rn(tn, shift), -0.0625, t);
    double p = 1.5403530393381606e-4;          // ln(2)^6 / 6!
    p = fma(p, r, 1.3333558146428441e-3);      // ln(2)^5 / 5!
    p = fma(p, r, 9.618129107628477e-3);      // ln(2)^4 / 4!
    p = fma(p, r, 5.5504108664821576e-2);      // ln(2)^3 / 3!
    p = fma(p, r, 2.402265069591007e-1);      // ln(2)^2 / 2!
    p = fma(p, r, 6.931471805599453e-1);      // ln(2)
    p = fma(p, r, 1.0) * v[n & 15];
    const double y =
        __hiloint2double(__double2hiint(p) + ((n >> 4) << 20), __double2loint(p));
    // t > -1020, by its upper word (t is not positive)
    return (unsigned)__double2hiint(t) < 0xc08fe000u ? y : 0.0;
  }
};

// 2^x on the special-function unit (2 ulp over the range used here).
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The slice of a row that one CTA holds, and the cluster it belongs to.
template <typename T, bool kClustered>
struct RowSlice {
  static constexpr int kE = Vec<T>::kN;
  T* s;          // shared memory, 16-byte aligned
  int ph;        // first element of the slice is s[ph]
  int n;         // elements of the slice
  int nvec;      // 16-byte vectors that hold them
  int start;     // index in the row of the slice's first element
  int rank;      // CTA of the cluster
  int size;      // CTAs of the cluster
  int per_warp;  // vectors of a warp: warp w owns [w * per_warp, (w + 1) * per_warp)

  __device__ __forceinline__ void init(T* smem, const T* row, int vocab, int chunk) {
    if (kClustered) {
      rank = (int)cg::this_cluster().block_rank();
      size = (int)cg::this_cluster().num_blocks();
    } else {
      rank = 0;
      size = 1;
    }
    s = smem;
    start = min(vocab, rank * chunk);
    n = min(vocab - start, chunk);
    ph = (int)((reinterpret_cast<uintptr_t>(row + start) & 15) / sizeof(T));
    nvec = n > 0 ? (ph + n + kE - 1) / kE : 0;
    const int warps = (int)blockDim.x >> 5;
    per_warp = (nvec + warps - 1) / warps;
  }

  // Copies the slice (asynchronously where whole vectors lie inside it); the
  // caller waits with cp_async_wait_all and a barrier.
  __device__ __forceinline__ void load(const T* row) {
    const T* g = row + start - ph;  // 16-byte aligned; read only at [ph, ph + n)
    const T lowest = narrow<T>(-CUDART_INF_F);
    for (int v = threadIdx.x; v < nvec; v += blockDim.x) {
      const int e0 = v * kE;
      if (e0 >= ph && e0 + kE <= ph + n) {
        cp_async16(s + e0, g + e0, true);
      } else {
#pragma unroll
        for (int e = 0; e < kE; ++e)
          s[e0 + e] = (e0 + e >= ph && e0 + e < ph + n) ? g[e0 + e] : lowest;
      }
    }
    cp_async_commit();
  }

  // f(index in the row, value) over this warp's elements, leaving out vectors
  // with no element of at least `skip`.
  template <typename F>
  __device__ __forceinline__ void for_each_from(float skip, F f) const {
    for_each([&](int i0, const Vec<T>& x) {
      if (!(x.largest() >= skip)) return;
#pragma unroll
      for (int e = 0; e < kE; ++e) f(i0 + e, x.at(e));
    });
  }

  // f(first element index of the vector in the row, vector) over this warp's
  // vectors, in the order of their indices over the lanes.
  template <typename F>
  __device__ __forceinline__ void for_each(F f) const {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int end = min(nvec, (warp + 1) * per_warp);
    for (int v = warp * per_warp + lane; v < end; v += 32)
      f(v * kE - ph + start, reinterpret_cast<Vec<T>*>(s)[v]);
  }
  // f(x), x an array of kU vectors or of one, over this warp's vectors
  template <int kU, typename F>
  __device__ __forceinline__ void for_each_array(F f) const {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int end = min(nvec, (warp + 1) * per_warp);
    const Vec<T>* vec = reinterpret_cast<const Vec<T>*>(s);
    int v = warp * per_warp + lane;
    for (; v + (kU - 1) * 32 < end; v += kU * 32) {
      Vec<T> x[kU];
#pragma unroll
      for (int u = 0; u < kU; ++u) x[u] = vec[v + u * 32];
      f(x);
    }
    for (; v < end; v += 32) {
      Vec<T> x[1] = {vec[v]};
      f(x);
    }
  }
};

// Reductions over the CTA and its cluster by a commutative operation; every
// thread gets the result, the same bits in every CTA: the order of the
// operations is fixed.  CTAs have a power of two of warps.
constexpr int kSlotBytes = 32;
struct ReduceScratch {
  alignas(16) unsigned char warp[2][kMaxWarps * kSlotBytes];
  alignas(16) unsigned char cta[2][kMaxCluster * kSlotBytes];
};

__device__ __forceinline__ double2 operator+(double2 a, double2 b) {
  return make_double2(a.x + b.x, a.y + b.y);
}
template <typename V>
__device__ __forceinline__ V shfl_xor(V v, int o) {
  return __shfl_xor_sync(0xffffffffu, v, o);
}
template <>
__device__ __forceinline__ ulonglong2 shfl_xor(ulonglong2 v, int o) {
  return make_ulonglong2(__shfl_xor_sync(0xffffffffu, v.x, o), __shfl_xor_sync(0xffffffffu, v.y, o));
}
template <>
__device__ __forceinline__ double2 shfl_xor(double2 v, int o) {
  return make_double2(__shfl_xor_sync(0xffffffffu, v.x, o), __shfl_xor_sync(0xffffffffu, v.y, o));
}

template <bool kClustered>
struct Reducer {
  ReduceScratch* sc;
  int buf;

  __device__ __forceinline__ explicit Reducer(ReduceScratch* s) : sc(s), buf(0) {}

  template <typename V, typename Op>
  __device__ __forceinline__ V all(V v, Op op) {
    static_assert(sizeof(V) <= kSlotBytes, "a slot holds one value");
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = op(v, shfl_xor(v, o));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = (int)blockDim.x >> 5;
    V* part = reinterpret_cast<V*>(sc->warp[buf]);
    if (lane == 0) part[warp] = v;
    __syncthreads();
    // every warp joins the warps' values (their number is a power of two) in
    // the same tree
    V r = part[lane & (warps - 1)];
    for (int o = 1; o < warps; o <<= 1) r = op(r, shfl_xor(r, o));
    if (kClustered) {
      // each CTA writes its value into every CTA's slots; two buffers, so a
      // slot is written again only after the next reduction's barrier
      auto cl = cg::this_cluster();
      const int size = (int)cl.num_blocks();
      V* slots = reinterpret_cast<V*>(sc->cta[buf]);
      if ((int)threadIdx.x < size) cl.map_shared_rank(slots, threadIdx.x)[cl.block_rank()] = r;
      cl.sync();
      r = slots[0];
      for (int c = 1; c < size; ++c) r = op(r, slots[c]);
    }
    buf ^= 1;
    return r;
  }

  // Every CTA's value (uniform within it), in rank order; valid until the next
  // call.
  template <typename V>
  __device__ __forceinline__ const V* spread(V v) {
    static_assert(sizeof(V) <= kSlotBytes, "a slot holds one value");
    V* slots = reinterpret_cast<V*>(sc->cta[buf]);
    if (kClustered) {
      auto cl = cg::this_cluster();
      if (threadIdx.x < cl.num_blocks())
        cl.map_shared_rank(slots, threadIdx.x)[cl.block_rank()] = v;
      cl.sync();
    } else {
      if (threadIdx.x == 0) slots[0] = v;
      __syncthreads();
    }
    buf ^= 1;
    return slots;
  }

  template <typename V>
  __device__ __forceinline__ V sum(V v) {
    return all(v, [](V a, V b) { return a + b; });
  }
  template <typename V>
  __device__ __forceinline__ V max(V v) {
    return all(v, [](V a, V b) { return a > b ? a : b; });
  }
  template <typename V>
  __device__ __forceinline__ V min(V v) {
    return all(v, [](V a, V b) { return a < b ? a : b; });
  }
};

// Tokens of a row picked out for the CTA of rank 0 to put in order: key << 32 |
// ~index, so that the larger item is the earlier one of the row's order (value
// down, index up).
constexpr int kListCap = 2048;
struct TokenList {
  unsigned count;  // of this CTA's own items
  alignas(16) unsigned long long item[kListCap];
};
__device__ __forceinline__ unsigned long long list_item(uint32_t key, int index) {
  return ((unsigned long long)key << 32) | (uint32_t)~index;
}
__device__ __forceinline__ uint32_t item_key(unsigned long long it) { return (uint32_t)(it >> 32); }
__device__ __forceinline__ int item_index(unsigned long long it) { return (int)~(uint32_t)it; }

// Collects the row's elements for which pick(index, value) holds, none of them
// below `skip`.  Returns their number; if it is at most kListCap, rank 0's list
// holds them all, in no particular order, else the lists are of no use.
template <typename T, bool kClustered, typename F>
__device__ int collect(const RowSlice<T, kClustered>& row, Reducer<kClustered>& red,
                       TokenList& list, float skip, F pick) {
  if (threadIdx.x == 0) list.count = 0;
  __syncthreads();
  row.for_each_from(skip, [&](int i, float x) {
    if (pick(i, x)) {
      const unsigned at = atomicAdd(&list.count, 1u);
      if (at < kListCap) list.item[at] = list_item(order_key(x), i);
    }
  });
  __syncthreads();
  if (!kClustered) return (int)list.count;
  const int mine = (int)list.count;
  const int* counts = red.spread(mine);
  int total = 0, offset = 0;
  for (int c = 0; c < row.size; ++c) {
    if (c < row.rank) offset += counts[c];
    total += counts[c];
  }
  if (total > kListCap) return total;
  // rank 0's own items are in place, the other CTAs' go behind them
  if (row.rank != 0) {
    unsigned long long* out = cg::this_cluster().map_shared_rank(list.item, 0) + offset;
    for (int i = threadIdx.x; i < mine; i += blockDim.x) out[i] = list.item[i];
  }
  cg::this_cluster().sync();
  return total;
}

// Number of the first n items that are larger than `me`, as counted by every
// `group`-th thread from `part` on: each takes its share of pairs, four loads at
// a time.
__device__ __forceinline__ int count_larger(const unsigned long long* item, int n,
                                            unsigned long long me, int part, int group) {
  const ulonglong2* pair = reinterpret_cast<const ulonglong2*>(item);
  const int pairs = n / 2;
  int c = 0, j = part;
  for (; j + 3 * group < pairs; j += 4 * group) {
    const ulonglong2 a = pair[j], b = pair[j + group], d = pair[j + 2 * group],
                     e = pair[j + 3 * group];
    c += (a.x > me) + (a.y > me) + (b.x > me) + (b.y > me) + (d.x > me) + (d.y > me) +
         (e.x > me) + (e.y > me);
  }
  for (; j < pairs; j += group) c += (pair[j].x > me) + (pair[j].y > me);
  if ((n & 1) && part == 0) c += item[n - 1] > me;
  return c;
}

// Sorts n <= kListCap items downwards: bitonic, the strides below 32 in registers
// of a warp each.  All the CTA's threads call it, whole warps.
__device__ __forceinline__ void sort_down(unsigned long long* item, int n) {
  const int warps = (int)blockDim.x >> 5, warp = (int)threadIdx.x >> 5, lane = threadIdx.x & 31;
  int size = 32;
  while (size < n) size <<= 1;
  for (int i = n + (int)threadIdx.x; i < size; i += blockDim.x) item[i] = 0;
  __syncthreads();
  auto exchange = [lane](unsigned long long v, int i, int k, int j) {
    const unsigned long long o = __shfl_xor_sync(0xffffffffu, v, j);
    return (((lane & j) == 0) == ((i & k) == 0)) == (v < o) ? o : v;
  };
  for (int i = warp * 32 + lane; i < size; i += warps * 32) {
    unsigned long long v = item[i];
#pragma unroll
    for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
      for (int j = k >> 1; j > 0; j >>= 1) v = exchange(v, i, k, j);
    item[i] = v;
  }
  __syncthreads();
  for (int k = 64; k <= size; k <<= 1) {
    for (int j = k >> 1; j >= 32; j >>= 1) {
      for (int p = threadIdx.x; p < size / 2; p += blockDim.x) {
        const int i = ((p & ~(j - 1)) << 1) | (p & (j - 1)), l = i | j;
        const unsigned long long a = item[i], b = item[l];
        if ((a < b) == ((i & k) == 0)) {
          item[i] = b;
          item[l] = a;
        }
      }
      __syncthreads();
    }
    for (int i = warp * 32 + lane; i < size; i += warps * 32) {
      unsigned long long v = item[i];
#pragma unroll
      for (int j = 16; j > 0; j >>= 1) v = exchange(v, i, k, j);
      item[i] = v;
    }
    __syncthreads();
  }
}

// Of the threads' largest keys: a key, in its upper 16 bits, that at least
// `want` threads of this CTA reach; 0 if fewer threads have one.
__device__ __forceinline__ uint32_t reached_by(uint32_t key, int want) {
  uint32_t lo = 0;
  for (uint32_t bit = 0x80000000u; bit >= 0x10000u; bit >>= 1)
    if (__syncthreads_count(key >= (lo | bit)) >= want) lo |= bit;
  return lo;
}

// Inclusive prefix sums over the CTA: thread t's value becomes the sum of those
// of threads 0..t.  `scratch` holds a number per warp.
template <typename V>
__device__ __forceinline__ V block_scan(V v, V* scratch, V* total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = (int)blockDim.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  __syncthreads();  // the scratch may still be read
  if (lane == 31) scratch[warp] = v;
  __syncthreads();
  V base = V(0), all = V(0);
  for (int w = 0; w < warps; ++w) {
    if (w == warp) base = all;
    all += scratch[w];
  }
  *total = all;
  return base + v;
}

// ---- rows that are streamed -------------------------------------------------
//
// With many rows a CTA walks a whole row once for its sums and once more for
// what depends on them; the second walk finds the row in L2 as long as the rows
// of all resident CTAs fit there (two a SM of 512 threads: 78 MB with rows of
// 131,072 16-bit logits; rows of more than 400 KB go to HBM again).  That needs no
// cluster and no shared memory for the row, so several CTAs a SM cover each
// other's barriers.

template <typename T>
struct RowStream {
  static constexpr int kE = Vec<T>::kN;
  const T* g;   // 16-byte aligned: vector v is g[v * kE ..]; row element i is g[ph + i]
  int ph, end;  // the row's elements are [ph, end)
  int lo, hi;   // vectors that lie wholly in the row

  __device__ __forceinline__ RowStream(const T* row, int vocab) {
    ph = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    g = row - ph;
    end = ph + vocab;
    lo = ph > 0;
    hi = end / kE;
  }
  // A vector that lies partly in the row, -inf outside.
  __device__ __forceinline__ Vec<T> partial(int v) const {
    Vec<T> x;
#pragma unroll
    for (int i = 0; i < 4; ++i) x.w[i] = 0;
#pragma unroll
    for (int e = 0; e < kE; ++e) {
      const int i = v * kE + e;
      if (i >= ph && i < end) reinterpret_cast<T*>(x.w)[e] = g[i];
      else x.clear(e);
    }
    return x;
  }
  // f(x, v, step, whole, slot) over the CTA's threads: x an array of vectors v,
  // v + step, ..., in the slots slot, slot + 1, ... of kU that a thread's vectors
  // take in turn.  The next kU loads are in flight while f works on kU vectors; the
  // ends of the row that fill no vector come last, one vector each.  With kTeam
  // the row is a team's of that many lanes, not the CTA's.
  template <int kU, int kTeam = 0, typename F>
  __device__ __forceinline__ void walk(F f) const {
    const int threads = kTeam ? kTeam : (int)blockDim.x;
    const int tid = kTeam ? (int)threadIdx.x % (kTeam ? kTeam : 1) : (int)threadIdx.x;
    const Vec<T>* vec = reinterpret_cast<const Vec<T>*>(g);
    int v = lo + tid;
    if (v + (kU - 1) * threads < hi) {
      Vec<T> y[kU];
#pragma unroll
      for (int u = 0; u < kU; ++u) y[u] = vec[v + u * threads];
      for (; v + (kU - 1) * threads < hi; v += kU * threads) {
        Vec<T> x[kU];
#pragma unroll
        for (int u = 0; u < kU; ++u) x[u] = y[u];
        if (v + (2 * kU - 1) * threads < hi) {
#pragma unroll
          for (int u = 0; u < kU; ++u) y[u] = vec[v + (kU + u) * threads];
        }
        f(x, v, threads, true, 0);
      }
    }
#pragma unroll
    for (int u = 0; u < kU - 1; ++u)
      if (v + u * threads < hi) {
        Vec<T> x[1] = {vec[v + u * threads]};
        f(x, v + u * threads, threads, true, u);
      }
    if ((tid == 0 && lo > 0) || (tid == threads - 1 && hi >= lo && hi * kE < end)) {
      const int at = tid == 0 && lo > 0 ? 0 : hi;
      Vec<T> x[1] = {partial(at)};
      f(x, at, threads, false, kU - 1);
    }
  }
};

// The threads that share a row: the CTA, or kTeam neighbouring lanes, of which a
// warp then has several, each at its own place in the code.
template <int kTeam>
struct Team {
  unsigned mask;
  __device__ __forceinline__ explicit Team(ReduceScratch*)
      : mask((kTeam == 32 ? 0xffffffffu : (1u << (kTeam & 31)) - 1u)
             << (threadIdx.x & 31 & ~(unsigned)(kTeam - 1))) {}
  __device__ __forceinline__ int rank() const { return threadIdx.x & (kTeam - 1); }
  __device__ __forceinline__ int size() const { return kTeam; }
  __device__ __forceinline__ void sync() const { __syncwarp(mask); }
  __device__ __forceinline__ bool any(bool p) const {
    __syncwarp(mask);
    return __any_sync(mask, p);
  }
  template <typename V, typename Op>
  __device__ __forceinline__ V all(V v, Op op) const {
    static_assert(sizeof(V) % 4 == 0, "moved as words");
#pragma unroll
    for (int o = kTeam / 2; o > 0; o >>= 1) {
      unsigned w[sizeof(V) / 4];
      memcpy(w, &v, sizeof(V));
#pragma unroll
      for (unsigned& x : w) x = __shfl_xor_sync(mask, x, o);
      V y;
      memcpy(&y, w, sizeof(V));
      v = op(v, y);
    }
    __syncwarp(mask);
    return v;
  }
};
template <>
struct Team<0> {
  Reducer<false> red;
  __device__ __forceinline__ explicit Team(ReduceScratch* s) : red(s) {}
  __device__ __forceinline__ int rank() const { return threadIdx.x; }
  __device__ __forceinline__ int size() const { return blockDim.x; }
  __device__ __forceinline__ void sync() const { __syncthreads(); }
  __device__ __forceinline__ bool any(bool p) const { return __syncthreads_or(p); }
  template <typename V, typename Op>
  __device__ __forceinline__ V all(V v, Op op) {
    return red.all(v, op);
  }
};

// Running largest logit m and sum of 2^((x - m) c), 32 bits.  -inf and 0 when
// nothing above -inf was added; NaN once a NaN or +inf was.
struct SoftSum {
  float m, s;

  __device__ __forceinline__ SoftSum() : m(-INFINITY), s(0.0f) {}

  // Adds the vectors x[0..kU): one test for a new maximum, then pairs on the
  // packed 32-bit pipe.
  template <typename T, int kU>
  __device__ __forceinline__ void add(Vec<T> (&x)[kU], float c) {
    float vm = x[0].largest();
#pragma unroll
    for (int u = 1; u < kU; ++u) vm = fmaxf(vm, x[u].largest());
    if (vm > m) {
      s *= exp2_fast((m - vm) * c);
      m = vm;
    }
    const float ref = m == -INFINITY ? 0.0f : m;
    const float2 minus = make_float2(-ref, -ref), scale = make_float2(c, c);
    float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int u = 0; u < kU; ++u)
#pragma unroll
      for (int i = 0; i < Vec<T>::kN / 2; ++i) {
        const float2 t = __fmul2_rn(__fadd2_rn(x[u].pair(i), minus), scale);
        sum = __fadd2_rn(sum, make_float2(exp2_fast(t.x), exp2_fast(t.y)));
      }
    s += sum.x + sum.y;
  }
  __device__ __forceinline__ static SoftSum join(SoftSum a, SoftSum b, float c) {
    SoftSum r;
    r.m = fmaxf(a.m, b.m);
    const float fa = a.m == r.m ? 1.0f : exp2_fast((a.m - r.m) * c);
    const float fb = b.m == r.m ? 1.0f : exp2_fast((b.m - r.m) * c);
    r.s = __fadd_rn(__fmul_rn(a.s, fa), __fmul_rn(b.s, fb));
    return r;
  }
};

template <>
__device__ __forceinline__ SoftSum shfl_xor(SoftSum v, int o) {
  SoftSum r;
  r.m = __shfl_xor_sync(0xffffffffu, v.m, o);
  r.s = __shfl_xor_sync(0xffffffffu, v.s, o);
  return r;
}

// Streaming is used from more rows than four a SM, where a CTA's set-up and its
// barriers cost rows in shared memory more, and from more bytes than about two
// thirds of what the SMs' shared memory holds at once (two slices of 64 KB each).
// Measured (us), streamed and in shared memory, bf16, loss with its gradient: 150 x
// 2000: 12 and 10; 300 x 8000: 20 and 12; 600 x 100: 10 and 16; 600 x 8000: 23 and 20;
// 2000 x 2000: 16 and 29; 2000 x 8000: 29 and 39; 40 x 131072 (10.5 MB): 25 and 20; 74 x
// 131072 (19 MB): 25 and 33; 150 x 50001 (15 MB): 23 and 31.  Top 64 gains less, and
// loses where slices are full: 4000 x 8000: 68 and 57; 2000 x 1000: 18 and 25; 74 x
// 131072: 20 and 27.
inline bool use_stream(int64_t rows, int vocab, int elem_bytes) {
  return rows > 4 * 148 || rows * vocab * elem_bytes > 12000000;
}

// Threads for a CTA that streams rows: a power of two, 20 to 40 vectors a thread.  Fewer threads a row leave room for more CTAs, whose
// barriers then cover each other.  Measured (loss and gradient, us): 2000 x
// 50001 bf16 243 with 512 threads, 172 with 256; 4096 x 131072 bf16 478 and 484.
constexpr int kStreamThreads = 512;
inline int stream_threads(int vocab, int elem_bytes) {
  const int nvec = vocab / (16 / elem_bytes) + 1;
  int t = 32;
  while (t < kStreamThreads && t * 40 < nvec) t *= 2;
  return t;
}

// ---- rows of a warp -----------------------------------------------------------
//
// Rows of at most kWarpVocab tokens: a warp owns a row, lane l its tokens
// [l * kPer, (l + 1) * kPer) in registers, so that a lane's number orders
// tokens and ballots find the first of them.  kPer is odd: the lanes' walks
// over the staged row then start in different banks.
constexpr int kWarpVocab = 31 * 32;
constexpr int kWarpRows = 4;  // warps of a CTA

// A warp's passes over its tokens take their time, a CTA a row its set-up: with
// few rows of more than seven tokens a lane the CTA is mostly faster, from four
// rows a SM the warp.  Measured (us), warp and CTA, f32, top 100 logits / top-p 0.9 /
// top-k 20: 100 x 224: 14 and 10 / 12 and 12 / 10 and 10; 100 x 500: 18 and 10 / 27
// and 14 / 16 and 10; 600 x 500: 20 and 16 / 27 and 25 / 16 and 16; 600 x 900: 20 and 14
// / 27 and 37 / 16 and 16; 2000 x 900: 29 and 29 / 39 and 92 / 25 and 31; 4000 x 100: 18
// and 39 / 18 and 82 / 16 and 51.
inline bool use_warp_rows(int64_t rows, int vocab) {
  return vocab <= 7 * 32 || (vocab <= kWarpVocab && rows >= 4 * 148);
}

template <typename T, int kPer>
struct WarpRow {
  static constexpr int kE = Vec<T>::kN;
  const T* s;       // shared memory
  int ph, vocab;
  float x[kPer];    // -inf past the row and for a NaN

  __host__ __device__ static constexpr int bytes(int vocab) { return (vocab / kE + 2) * 16; }
  __device__ __forceinline__ void stage(T* smem, const T* g, int v) {
    const int lane = threadIdx.x & 31;
    vocab = v;
    ph = (int)((reinterpret_cast<uintptr_t>(g) & 15) / sizeof(T));
    s = smem;
    const T* from = g - ph;
    for (int e0 = lane * kE; e0 < ph + v; e0 += 32 * kE) {
      if (e0 >= ph && e0 + kE <= ph + v) {
        cp_async16(smem + e0, from + e0, true);
      } else {
#pragma unroll
        for (int e = 0; e < kE; ++e)
          if (e0 + e >= ph && e0 + e < ph + v) smem[e0 + e] = from[e0 + e];
      }
    }
    cp_async_commit();
  }
  // after cp_async_wait_all and a barrier
  __device__ __forceinline__ void read() {
    const int first = (threadIdx.x & 31) * kPer;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const float v = first + e < vocab ? widen(s[ph + first + e]) : -CUDART_INF_F;
      x[e] = v > -CUDART_INF_F ? v : -CUDART_INF_F;
    }
  }
  __device__ __forceinline__ float largest() const {
    float m = x[0];
#pragma unroll
    for (int e = 1; e < kPer; ++e) m = fmaxf(m, x[e]);
    return key_value(__reduce_max_sync(0xffffffffu, order_key(m)));
  }
  // tokens of the row at or above `from`
  __device__ __forceinline__ int count(float from) const {
    int n = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) n += x[e] >= from;
    return __reduce_add_sync(0xffffffffu, n);
  }
  // largest value that at least n tokens reach (n of the row's are above -inf)
  __device__ __forceinline__ float nth_largest(int n, float xmax) const {
    uint32_t lo = kKeyNegInf + 1, hi = order_key(xmax);
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo + 1) / 2;
      if (count(key_value(mid)) >= n) lo = mid;
      else hi = mid - 1;
    }
    return key_value(lo);
  }
  // this lane's part of `from`: its tokens above t and, of the row's first
  // `ties` tokens of `from` that equal t, those that are its own
  __device__ __forceinline__ unsigned head(unsigned from, float t, int ties) const {
    const int lane = threadIdx.x & 31;
    unsigned above = 0, equal = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      above |= (x[e] > t ? 1u : 0u) << e;
      equal |= (x[e] == t ? 1u : 0u) << e;
    }
    above &= from;
    equal &= from;
    int before = __popc(equal);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += y;
    }
    for (int left = ties - (before - __popc(equal)); left > 0 && equal != 0; --left) {
      above |= equal & (0u - equal);
      equal &= equal - 1;
    }
    return above;
  }
};

template <typename V>
__device__ __forceinline__ V warp_total(V v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// kernel<kPer> for the smallest of the compiled widths that holds `vocab`.
#define HKB_WARP_WIDTH(vocab, ...)        \
  do {                                    \
    if ((vocab) <= 3 * 32) {              \
      constexpr int kPer = 3;             \
      __VA_ARGS__;                        \
    } else if ((vocab) <= 7 * 32) {       \
      constexpr int kPer = 7;             \
      __VA_ARGS__;                        \
    } else if ((vocab) <= 15 * 32) {      \
      constexpr int kPer = 15;            \
      __VA_ARGS__;                        \
    } else {                              \
      constexpr int kPer = 31;            \
      __VA_ARGS__;                        \
    }                                     \
  } while (0)

// ---- short rows -------------------------------------------------------------
//
// Rows of at most kShortVocab tokens: a thread owns a row, a CTA kShortRows of
// them, staged through shared memory.  Rows that lie one after another are
// copied as they are, in 16-byte pieces; with an odd number of tokens the
// threads' walks over their rows then meet (almost) no bank conflict.  Other
// rows are staged token by token, element (row, i) at [i * kShortPitch + row]:
// 524,288 x 20 f32, top-p and min-p, 57 us; with 21 tokens 49.
constexpr int kShortVocab = 32;
constexpr int kShortRows = 128;
constexpr int kShortPitch = kShortRows + 1;

// f(row in the CTA, token, element index in the dense block of rows) over the
// CTA's `rows` rows of `width` numbers, consecutive threads on consecutive
// elements.
template <typename F>
__device__ __forceinline__ void for_each_short(int rows, int width, F f) {
  const int step_row = kShortRows / width, step_col = kShortRows % width;
  int row = (int)threadIdx.x / width, col = (int)threadIdx.x % width;
#pragma unroll 4
  for (int i = threadIdx.x; i < rows * width; i += kShortRows) {
    f(row, col, i);
    row += step_row;
    col += step_col;
    if (col >= width) {
      col -= width;
      ++row;
    }
  }
}

template <typename T>
struct ShortRows {
  T* s;
  int rows, vocab;
  int row_step, col_step;

  __host__ __device__ static constexpr int bytes(int vocab) {
    return (vocab * kShortPitch * (int)sizeof(T) + 15) / 16 * 16;
  }
  __device__ __forceinline__ static bool dense(const T* g, int64_t row_stride, int vocab) {
    return row_stride == vocab && (vocab & 1) && (reinterpret_cast<uintptr_t>(g) & 15) == 0;
  }
  // Starts the copy of the CTA's rows; the caller waits with cp_async_wait_all
  // and a barrier.
  __device__ __forceinline__ void load(T* smem, const T* g, int64_t row_stride, int n, int v) {
    s = smem;
    rows = n;
    vocab = v;
    if (dense(g, row_stride, v)) {
      row_step = v;
      col_step = 1;
      const int bytes = n * v * (int)sizeof(T);
      const char* from = reinterpret_cast<const char*>(g);
      char* to = reinterpret_cast<char*>(s);
      for (int b = 16 * (int)threadIdx.x; b + 16 <= bytes; b += 16 * kShortRows)
        cp_async16(to + b, from + b, true);
      const int whole = bytes / 16 * 16 / (int)sizeof(T);
      if (whole + (int)threadIdx.x < n * v) s[whole + threadIdx.x] = g[whole + threadIdx.x];
    } else {
      row_step = 1;
      col_step = kShortPitch;
      for_each_short(n, v, [&](int row, int col, int) {
        s[col * kShortPitch + row] = g[row * row_stride + col];
      });
    }
    cp_async_commit();
  }
  __device__ __forceinline__ T& at(int row, int i) const { return s[row * row_step + i * col_step]; }
  // Writes the rows out of shared memory.
  __device__ __forceinline__ void store(T* g, int64_t row_stride) const {
    if (col_step == 1 && dense(g, row_stride, vocab)) {
      const int bytes = rows * vocab * (int)sizeof(T);
      for (int b = 16 * (int)threadIdx.x; b + 16 <= bytes; b += 16 * kShortRows)
        __stcs(reinterpret_cast<uint4*>(reinterpret_cast<char*>(g) + b),
               *reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(s) + b));
      const int whole = bytes / 16 * 16 / (int)sizeof(T);
      if (whole + (int)threadIdx.x < rows * vocab) g[whole + threadIdx.x] = s[whole + threadIdx.x];
    } else {
      for_each_short(rows, vocab,
                     [&](int row, int col, int) { g[row * row_stride + col] = at(row, col); });
    }
  }
};

// The comparators of the network's stage (P, K) and of the stages after it.
template <int kPad, int P, int K>
__device__ __forceinline__ void merge_stages(uint32_t (&key)[kPad]) {
#pragma unroll
  for (int j = K % P; j + K < kPad; j += 2 * K)
#pragma unroll
    for (int i = 0; i < K; ++i)
      if (i + j + K < kPad && (i + j) / (2 * P) == (i + j + K) / (2 * P)) {
        const uint32_t a = key[i + j], b = key[i + j + K];
        key[i + j] = ::max(a, b);
        key[i + j + K] = ::min(a, b);
      }
  if constexpr (K > 1) merge_stages<kPad, P, K / 2>(key);
  else if constexpr (2 * P < kPad) merge_stages<kPad, 2 * P, 2 * P>(key);
}

// The order of a short row in registers: key[j] holds, in its lower 5 bits, 31
// minus the index of the j-th token of the order (value down, index up), 0 past
// the tokens above -inf.  The values' keys lose their lower 5 bits to the index,
// so the network (odd-even merge sort, K. E. Batcher 1968; two instructions a
// comparator) may leave values that agree in 27 bits in the wrong order: such
// neighbours are compared in full and swapped.  16-bit logits have no lower
// bits to lose.
template <int kPad, typename F>
__device__ __forceinline__ void sort_short(uint32_t (&key)[kPad], int vocab, bool exact, F value) {
#pragma unroll
  for (int i = 0; i < kPad; ++i) {
    const float x = i < vocab ? value(i) : -CUDART_INF_F;
    key[i] = x > -CUDART_INF_F ? (order_key(x) & ~31u) | (31 - i) : 0u;
  }
  merge_stages<kPad, 1, 1>(key);
  if (exact) return;
  bool close = false;
#pragma unroll
  for (int j = 0; j + 1 < kPad; ++j) close |= (key[j] ^ key[j + 1]) < 32u && key[j + 1] != 0;
  while (close) {
    close = false;
#pragma unroll
    for (int j = 0; j + 1 < kPad; ++j) {
      if ((key[j] ^ key[j + 1]) >= 32u || key[j + 1] == 0) continue;
      const float a = value(31 - (int)(key[j] & 31)), b = value(31 - (int)(key[j + 1] & 31));
      if (b > a || (b == a && (key[j + 1] & 31) > (key[j] & 31))) {
        const uint32_t k = key[j];
        key[j] = key[j + 1];
        key[j + 1] = k;
        close = true;
      }
    }
  }
}

// kernel<kPad> for the smallest of the compiled widths that holds `vocab`.
#define HKB_SHORT_WIDTH(vocab, ...)       \
  do {                                    \
    if ((vocab) <= 8) {                   \
      constexpr int kPad = 8;             \
      __VA_ARGS__;                        \
    } else if ((vocab) <= 16) {           \
      constexpr int kPad = 16;            \
      __VA_ARGS__;                        \
    } else if ((vocab) <= 24) {           \
      constexpr int kPad = 24;            \
      __VA_ARGS__;                        \
    } else {                              \
      constexpr int kPad = 32;            \
      __VA_ARGS__;                        \
    }                                     \
  } while (0)

}  // namespace vocab
}  // namespace hkb
