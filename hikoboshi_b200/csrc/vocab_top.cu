// The k largest logits of each vocabulary row in the order (logit down, index
// up), with the row's log-sum-exp.
#include "hkb_mpnn.h"
#include "kernels.hpp"
#include "vocab.hpp"
#include "vocab_rows.cuh"

namespace hkb {
namespace vocab {
namespace {

// Writes row r's listing: the first k of the n items of the CTA's list in order.
template <typename T>
__device__ __forceinline__ void write_listing(TokenList& list, int n, const T* g, int64_t r,
                                              const TopArgs& a, int by_count) {
  const int tid = threadIdx.x, threads = blockDim.x;
  T* values = static_cast<T*>(a.values) + r * a.k;
  int32_t* tokens = a.tokens + r * a.k;
  auto put = [&](int place, int index) {
    values[place] = g[index];
    tokens[place] = index;
  };
  if (n <= by_count) {
    // an item's place is the number of larger ones, counted by a group of
    // threads
    int group = 32;
    while (group > 1 && n * group > threads) group >>= 1;
    for (int i0 = 0; i0 < n; i0 += threads / group) {
      const int i = i0 + tid / group;
      const unsigned long long me = i < n ? list.item[i] : 0ull;
      int place = i < n ? count_larger(list.item, n, me, tid % group, group) : 0;
      for (int o = group >> 1; o > 0; o >>= 1) place += __shfl_xor_sync(0xffffffffu, place, o);
      if (i < n && tid % group == 0 && place < a.k) put(place, item_index(me));
    }
  } else {
    sort_down(list.item, n);
    for (int i = tid; i < n && i < a.k; i += threads) put(i, item_index(list.item[i]));
  }
  for (int i = n + tid; i < a.k; i += threads) {
    values[i] = narrow<T>(-CUDART_INF_F);
    tokens[i] = -1;
  }
}

// What the CTAs of a row find together: its largest logit and sum, and the least
// of the keys that enough of their threads reach.
struct RowTop {
  SoftSum soft;
  uint32_t reached;
};

}  // namespace

template <>
__device__ __forceinline__ RowTop shfl_xor(RowTop v, int o) {
  RowTop r;
  r.soft = shfl_xor(v.soft, o);
  r.reached = __shfl_xor_sync(0xffffffffu, v.reached, o);
  return r;
}

namespace {

struct TopSmem {
  ReduceScratch red;
  TokenList list;
};

// Few rows: a cluster holds a row, each CTA finds its largest logits and sum in
// one pass, one joint reduction gives the bound, rank 0 orders what reaches it.
// Bound by latency: 5 x 100003 f32, top 256: 15 us, 40 CTAs of 148 SMs.
template <typename T, bool kClustered>
__global__ void __launch_bounds__(kMaxThreads, 2) top_rows_kernel(const T* __restrict__ logits,
                                                               int64_t row_stride, int vocab,
                                                               int chunk, TopArgs a) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  __shared__ TopSmem sm;
  const int cluster = kClustered ? (int)cg::this_cluster().num_blocks() : 1;
  const int64_t r = blockIdx.x / cluster;
  RowSlice<T, kClustered> row;
  const T* g = logits + r * row_stride;
  row.init(reinterpret_cast<T*>(smem_raw), g, vocab, chunk);
  row.load(g);
  cp_async_wait_all();
  if (kClustered) cg::this_cluster().sync();  // every CTA of the row runs from here on
  else __syncthreads();
  Reducer<kClustered> red(&sm.red);

  const float c = a.c;
  RowTop mine;
  float tmax = -CUDART_INF_F;
  row.template for_each_array<2>([&](auto& x) {
    constexpr int n = sizeof(x) / sizeof(x[0]);
#pragma unroll
    for (int u = 0; u < n; ++u) tmax = fmaxf(tmax, x[u].largest());
    if (a.log_norm) mine.soft.add(x, c);
  });
  mine.soft.m = tmax;
  if (a.log_norm && mine.soft.s != mine.soft.s) {
    // a NaN or +inf among the thread's logits: again, without the NaN (with a
    // +inf the sum is not used)
    mine.soft.s = 0.0f;
    row.for_each_from(-CUDART_MAX_NORMAL_F, [&](int, float y) {
      if (y > -CUDART_INF_F) mine.soft.s += exp2_fast((y == tmax ? 0.0f : y - tmax) * c);
    });
  }
  // The k-th largest of the row is no less than the k/C-th largest of the
  // threads' own largest logits in the CTA where that is least; few more than
  // k tokens reach it.
  mine.reached = reached_by(order_key(tmax), (a.k + row.size - 1) / row.size);
  mine = red.all(mine, [c](RowTop p, RowTop q) {
    RowTop t;
    t.soft = SoftSum::join(p.soft, q.soft, c);
    t.reached = ::min(p.reached, q.reached);
    return t;
  });
  const float xmax = mine.soft.m;
  if (a.log_norm && threadIdx.x == 0 && row.rank == 0)
    a.log_norm[r] = xmax == -CUDART_INF_F || xmax == CUDART_INF_F
                        ? xmax
                        : (float)((double)xmax * a.inv_temperature + log((double)mine.soft.s));
  const uint32_t bound = mine.reached;
  const float from = bound <= kKeyNegInf ? -CUDART_MAX_NORMAL_F : key_value(bound);
  int n = collect(row, red, sm.list, from, [&](int, float x) { return x >= from; });
  if (n > kListCap) {
    // many equal logits, or a row whose large logits lie side by side: the
    // k-th largest key by bisection, and the last index taken of its tokens
    auto count = [&](float from, int last) {
      int c = 0;
      row.for_each_from(from, [&](int i, float x) { c += x > from || (x == from && i <= last); });
      return red.sum(c);
    };
    uint32_t lo = kKeyNegInf + 1, hi = order_key(xmax);
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo + 1) / 2;
      if (count(key_value(mid), 0x7fffffff) >= a.k) lo = mid;
      else hi = mid - 1;
    }
    const float t = key_value(lo);
    int i_lo = 0, i_hi = vocab - 1;
    while (i_lo < i_hi) {
      const int mid = (i_lo + i_hi) / 2;
      if (count(t, mid) >= a.k) i_hi = mid;
      else i_lo = mid + 1;
    }
    n = collect(row, red, sm.list, t, [&](int i, float x) {
      return x > t || (x == t && i <= i_lo);
    });
  }
  if (row.rank == 0) write_listing(sm.list, n, g, r, a, 2 * (int)blockDim.x);
}

// Many rows: a CTA streams a row for its maxima and sum, then again, from L2, to
// collect what reaches the bound.  Bound by instructions and exponentials (69 %
// of issue, XU 50 %): 2048 x 131072 bf16, top 64: 153 us, 3.5 TB/s; with the row in
// a cluster's shared memory it was 652.  256 threads instead of 512: 186 against
// 166; the next loads in flight during the work: 161 against 166.
struct TopStreamSmem {
  ReduceScratch red;
  TokenList list;
  int scan[kMaxWarps];
  uint32_t bound;
};

// A lower bound of the k-th largest logit from the counts of the keys' upper 12
// bits, in the list's memory; 0 if the row has fewer than k.
constexpr int kTopBins = 4096;
// Longest list that is ordered by counting larger items instead of sorting (5000 x
// 8000 bf16 with 32 threads a row, top 40: 133 us, 143 with 48; top 128: 176, 182 with
// 192).
constexpr int kByCount = 96;
static_assert(kTopBins * sizeof(int) <= kListCap * sizeof(unsigned long long), "");

template <typename T>
__device__ __forceinline__ uint32_t bound_by_counts(const RowStream<T>& row, TopStreamSmem& sm,
                                                    int k) {
  constexpr int kE = Vec<T>::kN;
  int* bins = reinterpret_cast<int*>(sm.list.item);
  const int tid = threadIdx.x, threads = blockDim.x, per = kTopBins / threads;
  for (int i = tid; i < kTopBins; i += threads) bins[i] = 0;
  if (tid == 0) sm.bound = 0;
  __syncthreads();
  row.template walk<1>([&](auto& x, int, int, bool, int) {
#pragma unroll
    for (int e = 0; e < kE; ++e) {
      const float y = x[0].at(e);
      if (y > -CUDART_INF_F) atomicAdd(&bins[order_key(y) >> 20], 1);
    }
  });
  __syncthreads();
  // thread t sums the t-th share of the bins from the top
  const int top = kTopBins - 1 - tid * per;
  int mine = 0, all;
  for (int i = 0; i < per; ++i) mine += bins[top - ((i + tid) & (per - 1))];  // in turn: banks
  int above = block_scan(mine, sm.scan, &all) - mine;
  if (above < k && above + mine >= k) {
    int bin = top;
    while (above + bins[bin] < k) above += bins[bin--];
    sm.bound = (uint32_t)bin << 20;
  }
  __syncthreads();
  return sm.bound;
}

template <typename T>
__global__ void __launch_bounds__(kStreamThreads, 2) top_stream_kernel(const T* __restrict__ logits,
                                                                    int64_t row_stride, int vocab,
                                                                    TopArgs a) {
  __shared__ TopStreamSmem sm;
  constexpr int kE = Vec<T>::kN, kU = 4;
  const int64_t r = blockIdx.x;
  const T* g = logits + r * row_stride;
  const RowStream<T> row(g, vocab);
  Reducer<false> red(&sm.red);
  const int tid = threadIdx.x, threads = blockDim.x;
  if (tid == 0) sm.list.count = 0;

  const float c = a.c;
  SoftSum soft;
  float part[kU];  // largest logit of the vectors in each slot
#pragma unroll
  for (int u = 0; u < kU; ++u) part[u] = -CUDART_INF_F;
  row.template walk<kU>([&](auto& x, int, int, bool, int slot) {
    constexpr int n = sizeof(x) / sizeof(x[0]);
#pragma unroll
    for (int u = 0; u < n; ++u) part[(slot + u) % kU] = fmaxf(part[(slot + u) % kU], x[u].largest());
    if (a.log_norm) soft.add(x, c);
  });
  const float tmax = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
  if (a.log_norm) {
    if (soft.s != soft.s) {
      // a NaN or +inf among the thread's logits: again, one at a time, without
      // the NaN (with a +inf the sum is not used)
      soft = SoftSum();
      soft.m = tmax;
      row.template walk<1>([&](auto& x, int, int, bool, int) {
#pragma unroll
        for (int e = 0; e < kE; ++e) {
          const float y = x[0].at(e);
          if (y == y && tmax > -CUDART_INF_F) soft.s += exp2_fast((y == tmax ? 0.0f : y - tmax) * c);
        }
      });
    }
    soft = red.all(soft, [c](SoftSum p, SoftSum q) { return SoftSum::join(p, q, c); });
    if (tid == 0) {
      const bool inf = soft.m == -CUDART_INF_F || soft.m == CUDART_INF_F;
      a.log_norm[r] =
          inf ? soft.m : (float)((double)soft.m * a.inv_temperature + log((double)soft.s));
    }
  }
  // a lower bound of the k-th largest logit: one that k of the threads' own
  // maxima reach, or k of the maxima of their slots
  uint32_t bound = 0;
  if (a.k <= threads / 2) {
    bound = reached_by(order_key(tmax), a.k);
  } else if (threads < kStreamThreads) {
    bound = bound_by_counts(row, sm, a.k);
  } else {
    for (uint32_t bit = 0x80000000u; bit >= 0x10000u; bit >>= 1) {
      int n = 0;
#pragma unroll
      for (int u = 0; u < kU; ++u) n += __syncthreads_count(order_key(part[u]) >= (bound | bit));
      if (n >= a.k) bound |= bit;
    }
  }
  const float from = bound <= kKeyNegInf ? -CUDART_MAX_NORMAL_F : key_value(bound);
  __syncthreads();
  row.template walk<kU>([&](auto& x, int v, int step, bool, int) {
    constexpr int n = sizeof(x) / sizeof(x[0]);
#pragma unroll
    for (int u = 0; u < n; ++u) {
      if (!(x[u].largest() >= from)) continue;
      const int i0 = (v + u * step) * kE - row.ph;
#pragma unroll
      for (int e = 0; e < kE; ++e) {
        const float y = x[u].at(e);
        if (y >= from) {
          const unsigned at = atomicAdd(&sm.list.count, 1u);
          if (at < kListCap) sm.list.item[at] = list_item(order_key(y), i0 + e);
        }
      }
    }
  });
  __syncthreads();
  int n = (int)sm.list.count;
  if (n > kListCap) {
    // many equal logits or a large k: the k-th largest key by bisection, and
    // the last index taken of its tokens
    auto count = [&](uint32_t lo, int last) {
      int m = 0;
      row.template walk<1>([&](auto& x, int v, int, bool, int) {
#pragma unroll
        for (int e = 0; e < kE; ++e) {
          const float y = x[0].at(e);
          const uint32_t k = y == y ? order_key(y) : 0u;
          m += k > lo || (k == lo && v * kE - row.ph + e <= last);
        }
      });
      return red.sum(m);
    };
    uint32_t lo = bound > kKeyNegInf ? bound : kKeyNegInf + 1, hi = 0xffffffffu;
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo) / 2 + 1;
      if (count(mid, 0x7fffffff) >= a.k) lo = mid;
      else hi = mid - 1;
    }
    int i_lo = 0, i_hi = vocab - 1;
    while (i_lo < i_hi) {
      const int mid = (i_lo + i_hi) / 2;
      if (count(lo, mid) >= a.k) i_hi = mid;
      else i_lo = mid + 1;
    }
    if (tid == 0) sm.list.count = 0;
    __syncthreads();
    row.template walk<1>([&](auto& x, int v, int, bool, int) {
#pragma unroll
      for (int e = 0; e < kE; ++e) {
        const float y = x[0].at(e);
        const uint32_t k = y == y ? order_key(y) : 0u;
        const int i = v * kE - row.ph + e;
        if (k > lo || (k == lo && i <= i_lo))
          sm.list.item[atomicAdd(&sm.list.count, 1u)] = list_item(k, i);
      }
    });
    __syncthreads();
    n = a.k;
  }
  write_listing(sm.list, n, g, r, a, kByCount);
}

// Rows of up to kWarpVocab tokens, a warp each.  A short listing takes the
// largest remaining token k times; a longer one finds the k-th largest by
// bisection of keys and puts the k tokens in order in shared memory.  Bound by
// instructions: 121,729 x 422 bf16, top 2: 103 us (330 with a CTA a row).
constexpr int kTakeOneByOne = 16;

template <typename T, int kPer>
__global__ void __launch_bounds__(32 * kWarpRows) top_warp_kernel(const T* __restrict__ logits,
                                                                  int64_t row_stride,
                                                                  int64_t n_rows, int vocab,
                                                                  int list_size, TopArgs a) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t r = (int64_t)blockIdx.x * kWarpRows + warp;
  if (r >= n_rows) return;  // warps share nothing
  const int row_bytes = WarpRow<T, kPer>::bytes(vocab);
  WarpRow<T, kPer> row;
  row.stage(reinterpret_cast<T*>(smem_raw + warp * row_bytes), logits + r * row_stride, vocab);
  cp_async_wait_all();
  __syncwarp();
  row.read();
  const float xmax = row.largest();
  if (a.log_norm) {
    const float c = a.c;
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < kPer; ++e)
      s += exp2_fast((row.x[e] == xmax ? 0.0f : row.x[e] - xmax) * c);
    const double total = warp_total((double)s);
    if (lane == 0)
      a.log_norm[r] = xmax == -CUDART_INF_F || xmax == CUDART_INF_F
                          ? xmax
                          : (float)((double)xmax * a.inv_temperature + log(total));
  }
  T* values = static_cast<T*>(a.values) + r * a.k;
  int32_t* tokens = a.tokens + r * a.k;
  int n = 0;
  if (a.k <= kTakeOneByOne) {
    for (; n < a.k; ++n) {
      float best = -CUDART_INF_F;
      int at = 0;
#pragma unroll
      for (int e = 0; e < kPer; ++e)
        if (row.x[e] > best) {
          best = row.x[e];
          at = e;
        }
      const uint32_t key = order_key(best), most = __reduce_max_sync(0xffffffffu, key);
      if (most <= kKeyNegInf) break;
      if (lane == __ffs(__ballot_sync(0xffffffffu, key == most)) - 1) {
        const int index = lane * kPer + at;
        values[n] = row.s[row.ph + index];
        tokens[n] = index;
#pragma unroll
        for (int e = 0; e < kPer; ++e)
          if (e == at) row.x[e] = -CUDART_INF_F;
      }
    }
  } else {
    unsigned keep = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) keep |= (row.x[e] > -CUDART_INF_F ? 1u : 0u) << e;
    if ((int)__reduce_add_sync(0xffffffffu, __popc(keep)) > a.k) {
      const float t = row.nth_largest(a.k, xmax);
      int above = 0;
#pragma unroll
      for (int e = 0; e < kPer; ++e) above += row.x[e] > t;
      keep = row.head(keep, t, a.k - (int)__reduce_add_sync(0xffffffffu, above));
    }
    int at = __popc(keep);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, at, o);
      if (lane >= o) at += y;
    }
    n = __shfl_sync(0xffffffffu, at, 31);
    at -= __popc(keep);
    unsigned long long* item =
        reinterpret_cast<unsigned long long*>(smem_raw + kWarpRows * row_bytes) + warp * list_size;
#pragma unroll
    for (int e = 0; e < kPer; ++e)
      if (keep >> e & 1u) item[at++] = list_item(order_key(row.x[e]), lane * kPer + e);
    int size = 32;
    while (size < n) size <<= 1;  // list_size is a power of two of at least k
    for (int i = n + lane; i < size; i += 32) item[i] = 0;
    __syncwarp();
    for (int k = 2; k <= size; k <<= 1)
      for (int j = k >> 1; j > 0; j >>= 1) {
        for (int p = lane; p < size / 2; p += 32) {
          const int i = ((p & ~(j - 1)) << 1) | (p & (j - 1)), l = i | j;
          const unsigned long long u = item[i], w = item[l];
          if ((u < w) == ((i & k) == 0)) {
            item[i] = w;
            item[l] = u;
          }
        }
        __syncwarp();
      }
    for (int i = lane; i < n; i += 32) {
      const int index = item_index(item[i]);
      values[i] = row.s[row.ph + index];
      tokens[i] = index;
    }
  }
  for (int i = n + lane; i < a.k; i += 32) {
    values[i] = narrow<T>(-CUDART_INF_F);
    tokens[i] = -1;
  }
}

// Short rows, one thread each: sorts the row in registers.  The listing goes
// through shared memory, so that it leaves coalesced.  Bound by instructions (78 %
// of issue): 786,432 x 21 f32, top 8: 47 us (18.5 us of memory traffic); taking the
// largest remaining token 8 times took 76, and 40 registers a thread for twelve
// CTAs a SM 51 instead of 57.
template <typename T, int kPad>
__global__ void __launch_bounds__(kShortRows, kPad <= 24 ? 12 : 6) top_short_kernel(const T* __restrict__ logits,
                                                               int64_t row_stride, int64_t n_rows,
                                                               int vocab, TopArgs a) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  signed char* places = reinterpret_cast<signed char*>(smem_raw + ShortRows<T>::bytes(vocab));
  const int64_t r0 = (int64_t)blockIdx.x * kShortRows;
  const int rows = (int)::min((int64_t)kShortRows, n_rows - r0), tid = threadIdx.x;
  ShortRows<T> sr;
  sr.load(reinterpret_cast<T*>(smem_raw), logits + r0 * row_stride, row_stride, rows, vocab);
  cp_async_wait_all();
  __syncthreads();
  const int listed = ::min(a.k, vocab);
  if (tid < rows) {
    auto value = [&](int i) { return widen(sr.at(tid, i)); };
    uint32_t key[kPad];
    sort_short(key, vocab, sizeof(T) == 2, value);
#pragma unroll
    for (int j = 0; j < kPad; ++j)
      if (j < listed) places[j * kShortRows + tid] = key[j] ? (signed char)(31 - (key[j] & 31)) : -1;
    if (a.log_norm) {
      const float c = a.c;
      const float xmax = key[0] ? value(31 - (int)(key[0] & 31)) : -CUDART_INF_F;
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < kPad; ++i)
        if (i < vocab) {
          const float v = value(i);
          if (v > -CUDART_INF_F) s += exp2_fast((v == xmax ? 0.0f : v - xmax) * c);
        }
      a.log_norm[r0 + tid] = xmax == -CUDART_INF_F || xmax == CUDART_INF_F
                                 ? xmax
                                 : (float)fma((double)xmax, a.inv_temperature, (double)logf(s));
    }
  }
  __syncthreads();
  T* values = static_cast<T*>(a.values) + r0 * a.k;
  int32_t* tokens = a.tokens + r0 * a.k;
  for_each_short(rows, a.k, [&](int row, int j, int i) {
    const int at = j < listed ? places[j * kShortRows + row] : -1;
    values[i] = at >= 0 ? sr.at(row, at) : narrow<T>(-CUDART_INF_F);
    tokens[i] = at;
  });
}

template <typename T>
cudaError_t launch(cudaStream_t st, const VocabRows& v, const TopArgs& a) {
  if (v.vocab <= kShortVocab) {
    const int smem = ShortRows<T>::bytes(v.vocab) + kShortRows * v.vocab;
    const unsigned blocks = (unsigned)((v.rows + kShortRows - 1) / kShortRows);
    HKB_SHORT_WIDTH(v.vocab, (top_short_kernel<T, kPad><<<blocks, kShortRows, smem, st>>>(
                                 static_cast<const T*>(v.logits), v.row_stride, v.rows, v.vocab, a)));
    return cudaGetLastError();
  }
  if (use_warp_rows(v.rows, v.vocab)) {
    // the kept items: at most k of them, and of the row
    int list_size = 0;
    if (a.k > kTakeOneByOne)
      for (list_size = 32; list_size < a.k && list_size < v.vocab;) list_size *= 2;
    const int smem = kWarpRows * (WarpRow<T, 1>::bytes(v.vocab) + list_size * 8);
    const unsigned blocks = (unsigned)((v.rows + kWarpRows - 1) / kWarpRows);
    HKB_WARP_WIDTH(v.vocab, (top_warp_kernel<T, kPer><<<blocks, 32 * kWarpRows, smem, st>>>(
                                static_cast<const T*>(v.logits), v.row_stride, v.rows, v.vocab,
                                list_size, a)));
    return cudaGetLastError();
  }
  if (use_stream(v.rows, v.vocab, (int)sizeof(T))) {
    int threads = stream_threads(v.vocab, (int)sizeof(T));
    const int vectors = v.vocab / (16 / (int)sizeof(T)) + 1;
    // Twice as many threads as tokens wanted, where the row has work for them: the
    // bound then comes from the threads' own maxima.  Else it comes from counts.
    // Measured (us), maxima and counts, bf16: 12,899 x 3,101, top 64: 160 and 229;
    // top 128: 238 and 217; top 298: 991 and 342; 5000 x 8000, top 64: 82 and 154;
    // top 128: 133 and 129; 2000 x 20000, top 128: 74 and 121; top 298: 139 and 111;
    // 571 x 70000, top 298: 66 and 84; top 700: 139 and 92.  Counting with 128 and 256
    // threads: 36,363 x 1100, top 298: 662 and 801; top 700: 1026 and 1169.
    const bool by_maxima = a.k <= 64 ? 2 * a.k <= vectors : 16 * a.k <= vectors;
    const int most = by_maxima ? kStreamThreads : 128;
    while (threads < most && threads < (by_maxima ? 2 * a.k : a.k / 2)) threads *= 2;
    top_stream_kernel<T><<<(unsigned)v.rows, threads, 0, st>>>(
        static_cast<const T*>(v.logits), v.row_stride, v.vocab, a);
    return cudaGetLastError();
  }
  const RowShape s = row_shape(v.rows, v.vocab, (int)sizeof(T));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(v.rows * s.cluster));
  cfg.blockDim = dim3((unsigned)s.threads);
  cfg.dynamicSmemBytes = s.smem;
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = (unsigned)s.cluster;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  auto kernel = s.cluster > 1 ? top_rows_kernel<T, true> : top_rows_kernel<T, false>;
  ensure_dynamic_smem((const void*)kernel, 131072 + 16);
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<const T*>(v.logits), v.row_stride, v.vocab,
                            s.chunk, a);
}

}  // namespace
}  // namespace vocab

cudaError_t launch_top_logits(cudaStream_t st, const VocabRows& v, const TopArgs& a) {
  switch (v.dtype) {
    case HKB_F32: return vocab::launch<float>(st, v, a);
    case HKB_F16: return vocab::launch<__half>(st, v, a);
    default: return vocab::launch<__nv_bfloat16>(st, v, a);
  }
}

}  // namespace hkb
