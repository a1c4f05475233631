// Sampling with temperature, top-k, top-p and min-p from given uniforms.
//
// Row x, temperature T, w_i = exp((x_i - max x) / T).  Every filter keeps the
// head of the row in the order (x down, index up): top-k its first k, top-p
// the shortest head whose mass is at least p of the top-k mass, min-p the
// tokens with w_i >= min_p.  The kept set is the shortest of the three heads.
// The token is the first, in index order, whose running kept mass exceeds
// u * (kept mass).
//
// All masses are sums of 64-bit weights added in a fixed order: whether a
// token is kept or drawn depends on values next to a border, and 32-bit sums
// over a large vocabulary would move it.
#include <algorithm>

#include "hkb_mpnn.h"
#include "kernels.hpp"
#include "vocab.hpp"
#include "vocab_rows.cuh"

namespace hkb {

RowShape row_shape(int64_t rows, int vocab, int elem_bytes) {
  const int per16 = 16 / elem_bytes;
  RowShape s{};
  // slices of at most 64 KB, and more CTAs a row while there are few rows and
  // a slice keeps 4 KB
  s.cluster = 1;
  while (s.cluster < vocab::kMaxCluster) {
    const int64_t slice = (int64_t)vocab * elem_bytes / s.cluster;
    if (slice > 65536 || (rows * s.cluster < 148 && slice > 8192))
      s.cluster *= 2;
    else
      break;
  }
  const int chunk = (vocab + s.cluster - 1) / s.cluster;
  s.chunk = (chunk + per16 - 1) / per16 * per16;
  const int vecs = s.chunk / per16 + 1;
  s.smem = (size_t)vecs * 16;
  // a power of two (the bins of the sampler are dealt out evenly), about two
  // vectors a thread
  s.threads = 32;
  while (s.threads < vocab::kMaxThreads && s.threads * 2 < vecs) s.threads *= 2;
  return s;
}

namespace vocab {
namespace {

constexpr double kLog2e = 1.4426950408889634074;
constexpr double kLn2 = 0.69314718055994530942;

__device__ __forceinline__ bool settings_valid(float T, int top_k, float top_p, float min_p,
                                               double u) {
  return T >= 0.0f && T < CUDART_INF_F && top_k >= 0 && top_p >= 0.0f && top_p <= 1.0f &&
         min_p >= 0.0f && min_p <= 1.0f && u >= 0.0 && u <= 1.0;
}

constexpr int kBins = 1024;

struct SampleSmem {
  ReduceScratch red;
  ReduceScratch block;
  double seg[kMaxWarps];
  double total;
  int found;
  Exp2Table table;
  TokenList list;
  unsigned hist[kBins];
};

// First token, in index order, whose running sum of f exceeds `share` times the
// sum over the row (`absolute`: exceeds `share`); every thread of the cluster
// gets it.  f(index, value) is a weight, or negative for a token that is not
// kept; *total_out is the sum, *kept_out the number of kept tokens.  Rounding
// may leave no sum larger than the target: then the last token with f > 0 is
// it.  -1 if there is none.
template <typename T, bool kClustered, typename F>
__device__ int locate(const RowSlice<T, kClustered>& row, Reducer<kClustered>& red, SampleSmem& sm,
                      double share, bool absolute, double* total_out, int* kept_out, F f) {
  constexpr int kE = Vec<T>::kN;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = (int)blockDim.x >> 5;
  double mine = 0.0;
  int last = -1, n = 0;
  row.for_each([&](int i0, const Vec<T>& x) {
#pragma unroll
    for (int e = 0; e < kE; ++e) {
      const double w = f(i0 + e, x.at(e));
      if (w >= 0.0) {
        mine += w;
        ++n;
        if (w > 0.0) last = i0 + e;
      }
    }
  });
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  __syncthreads();
  if (lane == 0) sm.seg[warp] = mine;
  if (threadIdx.x == 0) sm.found = -1;
  *kept_out = red.sum(n);
  // mass of this CTA, of the row, and of the CTAs before this one
  double cta = 0.0;
  for (int w = 0; w < warps; ++w) cta += sm.seg[w];
  const double* of_cta = red.spread(cta);
  double before = 0.0, total = 0.0;
  for (int c = 0; c < row.size; ++c) {
    if (c == row.rank) before = total;
    total += of_cta[c];
  }
  *total_out = total;
  const double target = absolute ? share : share * total;
  // the warp in which the running sum passes the target
  double base = before;
  int hit = -1;
  for (int w = 0; w < warps; ++w) {
    const double next = base + sm.seg[w];
    if (sm.seg[w] > 0.0 && next > target) {
      hit = w;
      break;
    }
    base = next;
  }
  const bool here = hit >= 0 && !(before > target);
  if (here && warp == hit) {
    const int begin = warp * row.per_warp, end = min(row.nvec, begin + row.per_warp);
    int token = -1, seen = -1;
    for (int v0 = begin; v0 < end && token < 0; v0 += 32) {
      const int v = v0 + lane, i0 = v * kE - row.ph + row.start;
      double w[kE], sum = 0.0;
#pragma unroll
      for (int e = 0; e < kE; ++e) {
        w[e] = v < end ? f(i0 + e, reinterpret_cast<const Vec<T>*>(row.s)[v].at(e)) : 0.0;
        w[e] = w[e] > 0.0 ? w[e] : 0.0;
        sum += w[e];
      }
      double incl = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
      }
      const unsigned pass = __ballot_sync(0xffffffffu, sum > 0.0 && base + incl > target);
      const unsigned any = __ballot_sync(0xffffffffu, sum > 0.0);
      const int pick = pass ? __ffs(pass) - 1 : (any ? 31 - __clz(any) : -1);
      if (pick >= 0) {
        double run = __shfl_up_sync(0xffffffffu, incl, 1);
        run = base + (lane == 0 ? 0.0 : run);
        int t = -1;
        bool done = false;
#pragma unroll
        for (int e = 0; e < kE; ++e) {
          run += w[e];
          if (!done && w[e] > 0.0) {
            t = i0 + e;  // the last one with weight if rounding lets none pass
            done = run > target;
          }
        }
        t = __shfl_sync(0xffffffffu, t, pick);
        seen = t;
        if (pass) token = t;
      }
      base += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (token < 0) token = seen;
    if (lane == 0) sm.found = token;
  }
  __syncthreads();
  const int found = red.max(sm.found);
  if (found >= 0) return found;
  return red.max(last);
}

// Settings of one row.
struct RowSettings {
  float temperature;
  int top_k;
  float top_p, min_p;
  double u;
};

// Weights of a row: exponents relative to the largest logit.
struct Weights {
  float xmax;
  double c2;  // log2(e) / T
  const Exp2Table* table;
  __device__ __forceinline__ float below(float x) const { return x == xmax ? 0.0f : xmax - x; }
  __device__ __forceinline__ double exponent(float x) const {
    return x == xmax ? 0.0 : ((double)x - (double)xmax) * c2;
  }
  __device__ __forceinline__ double weight(float x) const { return (*table)(exponent(x)); }
};

// finish_list for more items than threads: sorts them, twice.
__device__ __noinline__ void finish_long_list(SampleSmem& sm, int n, const Weights& wt, const RowSettings& s,
                            double need, int64_t r, const SampleArgs& a) {
  unsigned long long* item = sm.list.item;
  Reducer<false> red(&sm.block);
  sort_down(item, n);
  const int nk = s.top_k > 0 ? ::min(n, s.top_k) : n;
  const int per = (nk + (int)blockDim.x - 1) / (int)blockDim.x;
  const int i0 = ::min(nk, (int)threadIdx.x * per), i1 = ::min(nk, i0 + per);
  auto weight = [&](int i) { return wt.weight(key_value(item_key(item[i]))); };
  int n_kept = nk;
  if (s.top_p < 1.0f || s.min_p > 0.0f) {
    double mine = 0.0, total;
    for (int i = i0; i < i1; ++i) mine += weight(i);
    double run = block_scan(mine, sm.seg, &total) - mine;
    if (need < 0.0) need = (double)s.top_p * total;
    int under = 0, heavy = 0;
    for (int i = i0; i < i1; ++i) {
      const double w = weight(i);
      run += w;
      under += run < need;
      heavy += w >= (double)s.min_p;
    }
    under = red.sum(under);
    heavy = red.sum(heavy);
    if (s.top_p < 1.0f) n_kept = ::min(n_kept, under + 1);
    n_kept = ::max(1, ::min(n_kept, heavy));
  }
  // the kept items in index order: (~index, key) downwards
  __syncthreads();
  for (int i = threadIdx.x; i < n_kept; i += blockDim.x) item[i] = item[i] << 32 | item[i] >> 32;
  __syncthreads();
  sort_down(item, n_kept);
  const int per2 = (n_kept + (int)blockDim.x - 1) / (int)blockDim.x;
  const int j0 = ::min(n_kept, (int)threadIdx.x * per2), j1 = ::min(n_kept, j0 + per2);
  auto weight2 = [&](int i) { return wt.weight(key_value((uint32_t)item[i])); };
  double mine = 0.0, total;
  for (int i = j0; i < j1; ++i) mine += weight2(i);
  double run = block_scan(mine, sm.seg, &total) - mine;
  const double target = s.u * total;
  int hit = 0x7fffffff, last = -1;
  for (int i = j0; i < j1; ++i) {
    const double w = weight2(i);
    run += w;
    if (w > 0.0) {
      last = i;
      if (run > target && hit == 0x7fffffff) hit = i;
    }
  }
  hit = red.min(hit);
  last = red.max(last);
  if (threadIdx.x == 0) {
    const unsigned long long it = item[hit != 0x7fffffff ? hit : last];
    const float x = key_value((uint32_t)it);
    a.tokens[r] = (int)~(uint32_t)(it >> 32);
    a.log_probs[r] = (float)(wt.exponent(x) * kLn2 - log(total));
    a.kept[r] = n_kept;
  }
}

// Finishes a row whose kept tokens are all among the n items of this CTA's
// list: puts them in order, cuts them to the shortest head and draws.  `need`
// is the mass that ends the top-p head, or negative: top_p of the mass of the
// first top_k items.  No more items than threads: each item's place in the
// order, and its running mass in index order, is counted over all items by a
// group of threads, which takes few barriers.
__device__ void finish_list(SampleSmem& sm, int n, const Weights& wt, const RowSettings& s,
                            double need, int64_t r, const SampleArgs& a) {
  const int threads = blockDim.x, tid = threadIdx.x;
  if (n > threads) {
    finish_long_list(sm, n, wt, s, need, r, a);
    return;
  }
  Reducer<false> red(&sm.block);
  const unsigned long long* item = sm.list.item;
  unsigned long long* sorted = sm.list.item + kMaxThreads;
  double* weight = reinterpret_cast<double*>(sm.list.item + 2 * kMaxThreads);
  int group = 32;  // threads an item, a power of two
  while (group > 1 && n * group > threads) group >>= 1;
  const int i = tid / group, part = tid % group;
  const bool mine = i < n, lead = mine && part == 0;
  int place = 0;
  unsigned long long me = 0;
  if (mine) {
    me = item[i];
    for (int j = part; j < n; j += group) place += item[j] > me;
  }
  for (int o = group >> 1; o > 0; o >>= 1) place += __shfl_xor_sync(0xffffffffu, place, o);
  if (lead) {
    sorted[place] = me;
    weight[place] = wt.weight(key_value(item_key(me)));
  }
  __syncthreads();
  const int nk = s.top_k > 0 ? ::min(n, s.top_k) : n;
  const double w = tid < nk ? weight[tid] : 0.0;
  double total;
  const double run = block_scan(w, sm.seg, &total);
  if (need < 0.0) need = (double)s.top_p * total;
  int kept = nk;
  if (s.top_p < 1.0f) kept = ::min(kept, 1 + __syncthreads_count(tid < nk && run < need));
  if (s.min_p > 0.0f) kept = ::min(kept, __syncthreads_count(tid < nk && w >= (double)s.min_p));
  kept = ::max(kept, 1);
  if (tid == kept - 1) sm.total = run;
  __syncthreads();
  const double mass = sm.total, target = s.u * mass;
  double upto = 0.0, own = 0.0;
  int index = -1;
  if (mine && i < kept) {
    me = sorted[i];
    own = weight[i];
    index = item_index(me);
    for (int j = part; j < kept; j += group)
      if (item_index(sorted[j]) <= index) upto += weight[j];
  }
  for (int o = group >> 1; o > 0; o >>= 1) upto += __shfl_xor_sync(0xffffffffu, upto, o);
  int token = red.min(own > 0.0 && upto > target ? index : 0x7fffffff);
  if (token == 0x7fffffff) token = red.max(own > 0.0 ? index : -1);  // rounding, or u = 1
  if (index == token && part == 0) {
    a.tokens[r] = token;
    a.log_probs[r] = (float)(wt.exponent(key_value(item_key(me))) * kLn2 - log(mass));
    a.kept[r] = kept;
  }
}

template <typename T, bool kClustered>
__global__ void __launch_bounds__(kMaxThreads, 2) sample_rows_kernel(
    const T* __restrict__ logits, int64_t row_stride, int vocab, int chunk, SampleArgs a) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  __shared__ SampleSmem sm;
  constexpr int kE = Vec<T>::kN;
  const int cluster = kClustered ? (int)cg::this_cluster().num_blocks() : 1;
  const int64_t r = blockIdx.x / cluster;
  RowSlice<T, kClustered> row;
  const T* g = logits + r * row_stride;
  row.init(reinterpret_cast<T*>(smem_raw), g, vocab, chunk);
  row.load(g);

  RowSettings s;
  s.temperature = a.temperatures ? a.temperatures[r] : a.temperature;
  s.top_k = a.top_ks ? a.top_ks[r] : a.top_k;
  s.top_p = a.top_ps ? a.top_ps[r] : a.top_p;
  s.min_p = a.min_ps ? a.min_ps[r] : a.min_p;
  s.u = a.uniforms_f64 ? static_cast<const double*>(a.uniforms)[r]
                       : (double)static_cast<const float*>(a.uniforms)[r];
  const bool valid = settings_valid(s.temperature, s.top_k, s.top_p, s.min_p, s.u);
  const bool writer = threadIdx.x == 0 && row.rank == 0;
  for (int b = threadIdx.x; b < kBins; b += blockDim.x) sm.hist[b] = 0;
  sm.table.fill();
  cp_async_wait_all();
  if (kClustered) cg::this_cluster().sync();  // every CTA of the row runs from here on
  else __syncthreads();
  if (!valid) {
    if (writer) {
      a.tokens[r] = -1;
      a.log_probs[r] = CUDART_NAN_F;
      a.kept[r] = 0;
    }
    return;
  }
  Reducer<kClustered> red(&sm.red);

  // largest logit and its first place; NaN becomes -inf
  float tmax = -CUDART_INF_F;
  int ibest = 0x7fffffff;
  row.for_each([&](int i0, Vec<T>& x) {
#pragma unroll
    for (int e = 0; e < kE; ++e) {
      const float v = x.at(e);
      if (v != v) x.clear(e);
      if (v > tmax) {
        tmax = v;
        ibest = i0 + e;
      }
    }
  });
  const uint32_t tkey = order_key(tmax);
  // of a row with top-k: a key that ceil(k / C) threads of this CTA reach
  if (s.top_k >= vocab) s.top_k = 0;
  const bool list_k = s.top_k > 0 && s.top_k <= kListCap / 2 && s.temperature > 0.0f;
  const uint32_t reached = list_k ? reached_by(tkey, (s.top_k + row.size - 1) / row.size) : 0;
  const ulonglong2 joint = red.all(make_ulonglong2(list_item(tkey, ibest), reached),
                                   [](ulonglong2 p, ulonglong2 q) {
                                     return make_ulonglong2(p.x > q.x ? p.x : q.x,
                                                            p.y < q.y ? p.y : q.y);
                                   });
  const unsigned long long best = joint.x;
  const uint32_t kmax = item_key(best);
  if (kmax <= kKeyNegInf || s.temperature == 0.0f) {
    if (writer) {
      const bool none = kmax <= kKeyNegInf;
      a.tokens[r] = none ? -1 : item_index(best);
      a.log_probs[r] = none ? -CUDART_INF_F : 0.0f;
      a.kept[r] = none ? 0 : 1;
    }
    return;
  }
  const Weights wt{key_value(kmax), kLog2e / (double)s.temperature, &sm.table};

  // Top-k of a number that fits the list: the k-th largest of the row is no
  // less than the k/C-th largest of the threads' own largest logits in the CTA
  // where that is least, and few more than k tokens reach it.
  if (list_k) {
    const uint32_t bound = (uint32_t)joint.y;
    const float from = bound <= kKeyNegInf ? -CUDART_MAX_NORMAL_F : key_value(bound);
    const int n = collect(row, red, sm.list, [&](int, float x) { return x >= from; });
    if (n <= kListCap) {
      if (row.rank == 0) finish_list(sm, n, wt, s, -1.0, r, a);
      return;
    }
  }

  // The kept head is { (key, index) : key > t, or key == t and index <= icut },
  // further cut by min-p and by `reach`, the largest distance from the largest
  // logit that a kept token can have.
  uint32_t t = kKeyNegInf + 1;
  int icut = 0x7fffffff;
  auto in_head = [&](int i, uint32_t k) { return k > t || (k == t && i <= icut); };
  if (s.top_k > 0) {
    // largest key with at least k tokens at or above it, by bisection
    auto count = [&](uint32_t lo) {
      int c = 0;
      row.for_each([&](int, const Vec<T>& x) {
#pragma unroll
        for (int e = 0; e < kE; ++e) c += order_key(x.at(e)) >= lo;
      });
      return red.sum(c);
    };
    if (count(kKeyNegInf + 1) > s.top_k) {
      uint32_t lo = kKeyNegInf + 1, hi = kmax;
      while (lo < hi) {
        const uint32_t mid = lo + (hi - lo + 1) / 2;
        if (count(mid) >= s.top_k) lo = mid;
        else hi = mid - 1;
      }
      t = lo;
      const int above = t == 0xffffffffu ? 0 : count(t + 1);
      double ties;
      int n;
      icut = locate(row, red, sm, (double)(s.top_k - above) - 0.5, true, &ties, &n,
                    [&](int, float x) { return order_key(x) == t ? 1.0 : -1.0; });
    }
  }
  const double zmin = s.min_p > 0.0f ? log2((double)s.min_p) - 1e-3 : -CUDART_INF;
  float reach = CUDART_INF_F;
  if (zmin > -CUDART_INF) reach = (float)(-zmin / wt.c2) * 1.000001f;

  if (s.top_p < 1.0f) {
    double m = 0.0;
    row.for_each([&](int i0, const Vec<T>& x) {
#pragma unroll
      for (int e = 0; e < kE; ++e) {
        const float v = x.at(e);
        if (in_head(i0 + e, order_key(v))) m += wt.weight(v);
      }
    });
    const double mass = red.sum(m);
    const double need = (double)s.top_p * mass;
    // Tokens lighter than (1 - p) * mass / V have less than (1 - p) * mass
    // together, so the border lies above them.
    const double z0 =
        fmax(zmin, log2((1.0 - (double)s.top_p) * mass / (double)vocab) - 1e-3);
    reach = (float)(-z0 / wt.c2) * 1.000001f;
    // Count the tokens within reach in bins of equal width: a bin's weights lie
    // between those of its ends, so the counts bound the running mass from both
    // sides (1e-4 covers the 32-bit arithmetic), and the border lies in the
    // few bins that the two bounds leave.
    const float scale = (float)kBins / reach;
    auto bin_of = [&](float x) { return ::min(kBins - 1, (int)(wt.below(x) * scale)); };
    row.for_each([&](int i0, const Vec<T>& x) {
#pragma unroll
      for (int e = 0; e < kE; ++e) {
        const float v = x.at(e);
        if (wt.below(v) <= reach && in_head(i0 + e, order_key(v))) atomicAdd(&sm.hist[bin_of(v)], 1u);
      }
    });
    if (kClustered) cg::this_cluster().sync();
    else __syncthreads();
    // every CTA adds up the whole row's bins and finds the same border
    const int per = kBins / (int)blockDim.x, b0 = (int)threadIdx.x * per;
    const float width2 = (float)(wt.c2 / (double)scale);  // of a bin, in powers of two
    float low = 0.0f, high = 0.0f, all;
    int number = 0;
    auto bin_count = [&](int b) {
      if (!kClustered) return (int)sm.hist[b];
      int c = 0;
      for (int k = 0; k < row.size; ++k)
        c += (int)cg::this_cluster().map_shared_rank(sm.hist, k)[b];
      return c;
    };
    for (int b = b0; b < b0 + per; ++b) {
      const float c = (float)bin_count(b);
      low += c * exp2f(-(float)(b + 1) * width2) * 0.9999f;
      high += c * exp2f(-(float)b * width2) * 1.0001f;
      number += (int)c;
    }
    float* fscratch = reinterpret_cast<float*>(sm.seg);
    int* iscratch = reinterpret_cast<int*>(sm.seg);
    int number_all;
    float run_low = block_scan(low, fscratch, &all) - low;
    float run_high = block_scan(high, fscratch, &all) - high;
    int run_number = block_scan(number, iscratch, &number_all) - number;
    // last bin that is certainly kept, first bin that certainly ends the head
    int certain = -1, ends = kBins;
    for (int b = b0; b < b0 + per; ++b) {
      const float c = (float)bin_count(b);
      run_low += c * exp2f(-(float)(b + 1) * width2) * 0.9999f;
      run_high += c * exp2f(-(float)b * width2) * 1.0001f;
      if (run_high < (float)need * 0.9999f) certain = b;
      if (run_low >= (float)need * 1.0001f) ends = ::min(ends, b);
    }
    Reducer<false> block(&sm.block);
    certain = block.max(certain);
    ends = ::min(kBins - 1, block.min(ends));
    int upto_certain = 0, upto_ends = 0;
    for (int b = b0; b < b0 + per; ++b) {
      run_number += bin_count(b);
      if (b == certain) upto_certain = run_number;
      if (b == ends) upto_ends = run_number;
    }
    upto_certain = block.sum(upto_certain);
    upto_ends = block.sum(upto_ends);
    // (the others may still read this CTA's bins: until their next reduction)

    // temperatures at the ends of the type's range leave no finite bin width
    const bool binned = scale > 0.0f && scale < CUDART_INF_F;
    const int list_from = upto_ends <= kListCap ? -1 : certain;
    if (binned && upto_ends - (list_from < 0 ? 0 : upto_certain) <= kListCap) {
      double above = 0.0;
      if (list_from >= 0) {
        row.for_each([&](int i0, const Vec<T>& x) {
#pragma unroll
          for (int e = 0; e < kE; ++e) {
            const float v = x.at(e);
            if (wt.below(v) <= reach && in_head(i0 + e, order_key(v)) && bin_of(v) <= list_from)
              above += wt.weight(v);
          }
        });
        above = red.sum(above);
      }
      const int n = collect(row, red, sm.list, [&](int i, float x) {
        if (!(wt.below(x) <= reach) || !in_head(i, order_key(x))) return false;
        const int b = bin_of(x);
        return b > list_from && b <= ends;
      });
      if (list_from < 0) {
        if (row.rank == 0) finish_list(sm, n, wt, s, need, r, a);
        return;
      }
      // the head ends inside the list, or (cut by min-p) nowhere
      unsigned long long border = 0;
      if (row.rank == 0) {
        sort_down(sm.list.item, n);
        const int per_t = (n + (int)blockDim.x - 1) / (int)blockDim.x;
        const int i0 = ::min(n, (int)threadIdx.x * per_t), i1 = ::min(n, i0 + per_t);
        double mine = 0.0, total;
        for (int i = i0; i < i1; ++i) mine += wt.weight(key_value(item_key(sm.list.item[i])));
        double run = above + (block_scan(mine, sm.seg, &total) - mine);
        int under = 0;
        for (int i = i0; i < i1; ++i) {
          run += wt.weight(key_value(item_key(sm.list.item[i])));
          under += run < need;
        }
        under = block.sum(under);
        if (under < n) border = sm.list.item[under];
      }
      border = red.spread(border)[0];
      if (border != 0) {
        t = item_key(border);
        icut = item_index(border);
      }
    } else {
      // equal logits crowd a bin: bisect between its ends
      auto mass_from = [&](uint32_t lo) {
        double m = 0.0;
        row.for_each([&](int i0, const Vec<T>& x) {
#pragma unroll
          for (int e = 0; e < kE; ++e) {
            const float v = x.at(e);
            const uint32_t k = order_key(v);
            if (k >= lo && in_head(i0 + e, k)) m += wt.weight(v);
          }
        });
        return red.sum(m);
      };
      uint32_t lo = t, hi = kmax;
      while (lo < hi) {
        const uint32_t mid = lo + (hi - lo + 1) / 2;
        if (mass_from(mid) >= need) lo = mid;
        else hi = mid - 1;
      }
      // `lo` is the border's key: of its tokens the first `ties` are kept
      const double above = lo == kmax ? 0.0 : mass_from(lo + 1);
      const double w = wt.weight(key_value(lo));
      double ties = w > 0.0 ? ceil((need - above) / w) : 1.0;
      if (ties < 1.0) ties = 1.0;
      const uint32_t old_t = t;
      const int old_cut = icut;
      t = lo;
      icut = 0x7fffffff;
      double all_ties;
      int n;
      icut = locate(row, red, sm, ties - 0.5, true, &all_ties, &n, [&](int i, float x) {
        const uint32_t k = order_key(x);
        return k == lo && (k > old_t || i <= old_cut) ? 1.0 : -1.0;
      });
    }
  }
  double total;
  int n;
  const int token = locate(row, red, sm, s.u, false, &total, &n, [&](int i, float x) {
    if (!(wt.below(x) <= reach) || !in_head(i, order_key(x))) return -1.0;
    const double w = wt.weight(x);
    return w >= (double)s.min_p ? w : -1.0;
  });
  if (writer) {
    a.tokens[r] = token;
    a.log_probs[r] = (float)(wt.exponent(widen(g[token])) * kLn2 - log(total));
    a.kept[r] = n;
  }
}

// Short rows, one thread each: 64-bit weights in shared memory; the head is
// found by taking the largest remaining token until a filter stops it, which
// ends early on the peaked rows that filters are for.
template <typename T>
__global__ void __launch_bounds__(kShortRows) sample_short_kernel(const T* __restrict__ logits,
                                                                  int64_t row_stride, int64_t n_rows,
                                                                  int vocab, SampleArgs a) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  __shared__ Exp2Table table;
  double* w = reinterpret_cast<double*>(smem_raw) + threadIdx.x;  // [i * kShortRows]
  float* xs = reinterpret_cast<float*>(smem_raw + sizeof(double) * kShortRows * vocab);
  const int64_t r0 = (int64_t)blockIdx.x * kShortRows;
  const int rows = (int)::min((int64_t)kShortRows, n_rows - r0);
  table.fill();
  load_short(xs, logits + r0 * row_stride, row_stride, rows, vocab, true);
  __syncthreads();
  if ((int)threadIdx.x >= rows) return;
  const int64_t r = r0 + threadIdx.x;
  const float* x = xs + threadIdx.x;  // [i * kShortPitch]
  const float Tf = a.temperatures ? a.temperatures[r] : a.temperature;
  const int topk = a.top_ks ? a.top_ks[r] : a.top_k;
  const float top_p = a.top_ps ? a.top_ps[r] : a.top_p;
  const float min_p = a.min_ps ? a.min_ps[r] : a.min_p;
  const double u = a.uniforms_f64 ? static_cast<const double*>(a.uniforms)[r]
                                  : (double)static_cast<const float*>(a.uniforms)[r];
  if (!settings_valid(Tf, topk, top_p, min_p, u)) {
    a.tokens[r] = -1;
    a.log_probs[r] = CUDART_NAN_F;
    a.kept[r] = 0;
    return;
  }
  float xmax = -CUDART_INF_F;
  int best = -1, live = 0;
  for (int i = 0; i < vocab; ++i) {
    const float v = x[i * kShortPitch];
    if (v > xmax) {
      xmax = v;
      best = i;
    }
    live += v > -CUDART_INF_F;
  }
  if (best < 0 || Tf == 0.0f) {
    a.tokens[r] = best;
    a.log_probs[r] = best < 0 ? -CUDART_INF_F : 0.0f;
    a.kept[r] = best < 0 ? 0 : 1;
    return;
  }
  const double c2 = kLog2e / (double)Tf;
  double sum = 0.0;
  for (int i = 0; i < vocab; ++i) {
    const float v = x[i * kShortPitch];
    const double wi = table(v == xmax ? 0.0 : ((double)v - (double)xmax) * c2);
    w[i * kShortRows] = wi;
    sum += wi;
  }
  unsigned keep = 0;  // the kept tokens
  const bool cut_k = topk > 0 && topk < live;
  if (cut_k || top_p < 1.0f) {
    // takes tokens in the head's order while `more` says so; their mass goes to `sum`
    auto head = [&](auto more) {
      unsigned taken = 0;
      int n = 0;
      double mass = 0.0;
      while (n < live && more(n, mass)) {
        float top = -CUDART_INF_F;
        int at = 0;
        for (int i = 0; i < vocab; ++i) {
          const float v = x[i * kShortPitch];
          if (v > top && !(taken >> i & 1u)) {
            top = v;
            at = i;
          }
        }
        taken |= 1u << at;
        mass += w[at * kShortRows];
        ++n;
      }
      sum = mass;
      return taken;
    };
    if (cut_k) keep = head([&](int n, double) { return n < topk; });
    if (top_p < 1.0f) {
      const double need = (double)top_p * sum;
      keep = head([&](int n, double mass) {
        return n == 0 || (mass < need && !(cut_k && n >= topk));
      });
    }
  } else {
    for (int i = 0; i < vocab; ++i)
      if (x[i * kShortPitch] > -CUDART_INF_F) keep |= 1u << i;
  }
  double total = 0.0;
  for (int i = 0; i < vocab; ++i) {
    const double wi = w[i * kShortRows];
    if (wi < (double)min_p) keep &= ~(1u << i);
    if (keep >> i & 1u) total += wi;
  }
  const double target = u * total;
  double run = 0.0;
  int token = best;
  for (int i = 0; i < vocab && !(run > target); ++i) {
    const double wi = keep >> i & 1u ? w[i * kShortRows] : 0.0;
    run += wi;
    if (wi > 0.0) token = i;
  }
  a.tokens[r] = token;
  a.log_probs[r] = (float)log(w[token * kShortRows] / total);
  a.kept[r] = __popc(keep);
}

template <typename T>
cudaError_t launch(cudaStream_t st, const VocabRows& v, const SampleArgs& a) {
  if (v.vocab <= kShortVocab) {
    const int smem = v.vocab * (int)(sizeof(double) * kShortRows + sizeof(float) * kShortPitch);
    ensure_dynamic_smem((const void*)sample_short_kernel<T>, kShortVocab *
                        (int)(sizeof(double) * kShortRows + sizeof(float) * kShortPitch));
    const unsigned blocks = (unsigned)((v.rows + kShortRows - 1) / kShortRows);
    sample_short_kernel<T><<<blocks, kShortRows, smem, st>>>(
        static_cast<const T*>(v.logits), v.row_stride, v.rows, v.vocab, a);
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
  auto kernel = s.cluster > 1 ? sample_rows_kernel<T, true> : sample_rows_kernel<T, false>;
  ensure_dynamic_smem((const void*)kernel, 131072 + 16);
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<const T*>(v.logits), v.row_stride, v.vocab,
                            s.chunk, a);
}

}  // namespace
}  // namespace vocab

cudaError_t launch_sample_tokens(cudaStream_t st, const VocabRows& v, const SampleArgs& a) {
  switch (v.dtype) {
    case HKB_F32: return vocab::launch<float>(st, v, a);
    case HKB_F16: return vocab::launch<__half>(st, v, a);
    default: return vocab::launch<__nv_bfloat16>(st, v, a);
  }
}

}  // namespace hkb
