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
  // slices of at most 64 KB (128 KB where 8 CTAs share a row of more than 131,072
  // 32-bit logits), and more CTAs a row while there are few rows and a slice keeps
  // 4 KB
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
  // 256 or 512, about two vectors a thread (1024 is no faster for a single row:
  // the barriers take longer)
  s.threads = vecs > 2 * 256 ? 512 : 256;
  // with more rows than two CTAs a SM, slices of which four fit a SM (beside the
  // sampler's 28 KB) do better on 256 threads: 25,892 rows of 3,227 f32, top-k: 678
  // us with 512 threads, 340 with 256; larger ones do not: 256 rows of 131,072
  // bf16 (64 KB), top-p: 348 and 381
  if (rows * s.cluster > 2 * 148 && s.smem <= 28 * 1024) s.threads = 256;
  return s;
}

namespace vocab {
namespace {

constexpr double kLog2e = 1.4426950408889634074;
constexpr double kLn2 = 0.69314718055994530942;

// Settings of one row.
struct RowSettings {
  float temperature;
  int top_k;
  float top_p, min_p;
  double u;
};

__device__ __forceinline__ RowSettings row_settings(const SampleArgs& a, int64_t r) {
  RowSettings s;
  s.temperature = a.temperatures ? a.temperatures[r] : a.temperature;
  s.top_k = a.top_ks ? a.top_ks[r] : a.top_k;
  s.top_p = a.top_ps ? a.top_ps[r] : a.top_p;
  s.min_p = a.min_ps ? a.min_ps[r] : a.min_p;
  s.u = a.uniforms_f64 ? static_cast<const double*>(a.uniforms)[r]
                       : (double)static_cast<const float*>(a.uniforms)[r];
  return s;
}

__device__ __forceinline__ bool settings_valid(const RowSettings s) {
  return s.temperature >= 0.0f && s.temperature < CUDART_INF_F && s.top_k >= 0 &&
         s.top_p >= 0.0f && s.top_p <= 1.0f && s.min_p >= 0.0f && s.min_p <= 1.0f &&
         s.u >= 0.0 && s.u <= 1.0;
}

constexpr int kBins = 1024;
constexpr int kSubList = 192;  // items of a list whose order is found by counting

// Bounds of the running mass and the number of tokens up to a bin.
struct alignas(16) Bounds {
  float low, high;
  int number, pad;
};

// Mass of some tokens and the span of some others.
struct Extent {
  double mass;
  float most, least;
};

// The same of list items, with their weights' sum in multiples of 2^-52.
struct ListExtent {
  unsigned long long sum;
  float most, least;
};

}  // namespace

template <>
__device__ __forceinline__ ListExtent shfl_xor(ListExtent v, int o) {
  ListExtent r;
  r.sum = __shfl_xor_sync(0xffffffffu, v.sum, o);
  r.most = __shfl_xor_sync(0xffffffffu, v.most, o);
  r.least = __shfl_xor_sync(0xffffffffu, v.least, o);
  return r;
}
template <>
__device__ __forceinline__ Extent shfl_xor(Extent v, int o) {
  Extent r;
  r.mass = __shfl_xor_sync(0xffffffffu, v.mass, o);
  r.most = __shfl_xor_sync(0xffffffffu, v.most, o);
  r.least = __shfl_xor_sync(0xffffffffu, v.least, o);
  return r;
}

namespace {

__device__ __forceinline__ ListExtent join(Reducer<false>& red, ListExtent v) {
  return red.all(v, [](ListExtent p, ListExtent q) {
    return ListExtent{p.sum + q.sum, fmaxf(p.most, q.most), fminf(p.least, q.least)};
  });
}

struct SampleSmem {
  Bounds bounds[kMaxWarps];
  ReduceScratch red;
  ReduceScratch block;
  double seg[kMaxWarps];
  int number[kMaxWarps];
  unsigned sub_count;
  unsigned long long sub[kSubList];
  unsigned long long sub_weight[kSubList];
  double step[32];  // a warp owns at most 17 steps of 32 vectors
  double total;
  Exp2Table table;
  TokenList list;
  alignas(8) unsigned hist[kBins];
};

// First token, in index order, whose running sum of f exceeds `share` times the
// sum over the row (`absolute`: exceeds `share`).  f(index, value) is a weight,
// or negative for a token that is not kept; *total_out is the sum, *kept_out
// the number of kept tokens.  Rounding may leave no sum larger than the target:
// then the last token with f > 0 is it.  The lanes of one warp of the cluster
// get the token, all other threads -1.
template <typename T, bool kClustered, typename F>
__device__ int locate(const RowSlice<T, kClustered>& row, Reducer<kClustered>& red, SampleSmem& sm,
                      float skip, double share, bool absolute, double* total_out, int* kept_out,
                      F f) {
  constexpr int kE = Vec<T>::kN;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = (int)blockDim.x >> 5;
  double mine = 0.0;
  int n = 0;
  row.for_each_from(skip, [&](int i, float x) {
    const double w = f(i, x);
    mine += w >= 0.0 ? w : 0.0;
    n += w >= 0.0;
  });
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  n = __reduce_add_sync(0xffffffffu, n);
  __syncthreads();
  if (lane == 0) {
    sm.seg[warp] = mine;
    sm.number[warp] = n;
  }
  __syncthreads();
  // running masses of the CTA's warps, in every warp
  const double seg = lane < warps ? sm.seg[lane] : 0.0;
  n = __reduce_add_sync(0xffffffffu, lane < warps ? sm.number[lane] : 0);
  double upto = seg;
#pragma unroll
  for (int o = 1; o < kMaxWarps; o <<= 1) {
    const double y = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += y;
  }
  const double cta = __shfl_sync(0xffffffffu, upto, kMaxWarps - 1);
  const double2* of_cta = red.spread(make_double2(cta, (double)n));
  double total = 0.0, kept = 0.0;
  for (int c = 0; c < row.size; ++c) {
    total += of_cta[c].x;
    kept += of_cta[c].y;
  }
  *total_out = total;
  *kept_out = (int)kept;
  const double target = absolute ? share : share * total;
  // the CTA in which the running sum passes the target, the same for all: the
  // last with any mass if rounding lets none pass
  int owner = -1;
  double run = 0.0, before = 0.0;
  bool passed = false;
  for (int c = 0; c < row.size && !passed; ++c) {
    const double m = of_cta[c].x;
    if (m > 0.0) {
      owner = c;
      before = run;
      passed = run + m > target;
    }
    run += m;
  }
  if (owner != row.rank) return -1;
  // its warp, likewise
  unsigned pass = __ballot_sync(0xffffffffu, seg > 0.0 && before + upto > target);
  const unsigned any = __ballot_sync(0xffffffffu, seg > 0.0);
  const int hit = pass ? __ffs(pass) - 1 : 31 - __clz(any);
  before += __shfl_sync(0xffffffffu, upto, hit) - __shfl_sync(0xffffffffu, seg, hit);
  // all warps add up the 32-vector steps of that warp's vectors
  const int begin = hit * row.per_warp, end = ::min(row.nvec, begin + row.per_warp);
  const int steps = (end - begin + 31) / 32;
  double w[kE];
  auto weigh = [&](int step) {
    const int v = begin + step * 32 + lane;
    double sum = 0.0;
#pragma unroll
    for (int e = 0; e < kE; ++e) {
      w[e] = v < end ? f(v * kE - row.ph + row.start + e,
                         reinterpret_cast<const Vec<T>*>(row.s)[v].at(e))
                     : 0.0;
      w[e] = w[e] > 0.0 ? w[e] : 0.0;
      sum += w[e];
    }
    return sum;
  };
  for (int i = warp; i < steps; i += warps) {
    double sum = weigh(i);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) sm.step[i] = sum;
  }
  __syncthreads();
  if (warp != hit) return -1;
  const double mass = lane < steps ? sm.step[lane] : 0.0;
  upto = mass;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double y = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += y;
  }
  pass = __ballot_sync(0xffffffffu, mass > 0.0 && before + upto > target);
  const unsigned heavy = __ballot_sync(0xffffffffu, mass > 0.0);
  const int step = pass ? __ffs(pass) - 1 : 31 - __clz(heavy);
  before += __shfl_sync(0xffffffffu, upto, step) - __shfl_sync(0xffffffffu, mass, step);
  // its vector and element
  const double sum = weigh(step);
  upto = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double y = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += y;
  }
  pass = __ballot_sync(0xffffffffu, sum > 0.0 && before + upto > target);
  const unsigned some = __ballot_sync(0xffffffffu, sum > 0.0);
  const int at = pass ? __ffs(pass) - 1 : 31 - __clz(some);
  double at_run = before + upto - sum;
  int token = -1;
  bool done = false;
#pragma unroll
  for (int e = 0; e < kE; ++e) {
    at_run += w[e];
    if (!done && w[e] > 0.0) {
      token = (begin + step * 32 + lane) * kE - row.ph + row.start + e;
      done = at_run > target;
    }
  }
  return __shfl_sync(0xffffffffu, token, at);
}

// Weights of a row: exponents relative to the largest logit.
struct Weights {
  float xmax;  // finite
  double c2;   // log2(e) / T
  const Exp2Table* table;
  __device__ __forceinline__ double exponent(float x) const {
    return ((double)x - (double)xmax) * c2;
  }
  __device__ __forceinline__ double weight(float x) const { return (*table)(exponent(x)); }
};

// The sums of the threads before this one.
__device__ __forceinline__ Bounds scan_bounds(Bounds v, SampleSmem& sm) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = (int)blockDim.x >> 5;
  Bounds incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const float low = __shfl_up_sync(0xffffffffu, incl.low, o);
    const float high = __shfl_up_sync(0xffffffffu, incl.high, o);
    const int number = __shfl_up_sync(0xffffffffu, incl.number, o);
    if (lane >= o) {
      incl.low += low;
      incl.high += high;
      incl.number += number;
    }
  }
  Bounds before;
  before.low = __shfl_up_sync(0xffffffffu, incl.low, 1);
  before.high = __shfl_up_sync(0xffffffffu, incl.high, 1);
  before.number = __shfl_up_sync(0xffffffffu, incl.number, 1);
  before.pad = 0;
  if (lane == 0) before = Bounds{0.0f, 0.0f, 0, 0};
  if (lane == 31) sm.bounds[warp] = incl;
  __syncthreads();
  for (int w = 0; w < warp && w < warps; ++w) {
    before.low += sm.bounds[w].low;
    before.high += sm.bounds[w].high;
    before.number += sm.bounds[w].number;
  }
  return before;
}

// Bins of falling value from xhi on: the last that certainly belongs to the
// head and the first that certainly ends it, with the tokens up to their ends.
struct Bracket {
  int certain, upto_certain, end, upto_end;
};

// Where the running mass from xhi on reaches `rest`, as far as the bins'
// counts tell.  The bounds leave 1e-5 for the 32-bit arithmetic (exponents of at
// most 45: 3e-6; sums: 1e-6).  Called by all threads of the CTA.
template <typename F>
__device__ __forceinline__ Bracket bracket(SampleSmem& sm, float scale, const Weights wt,
                                           float xhi, double rest64, F bin_count) {
  constexpr int kPerThread = kBins / 256;  // CTAs have 256 threads or more
  const int per = kBins / (int)blockDim.x, b0 = (int)threadIdx.x * per;
  const float width2 = (float)(wt.c2 / (double)scale);  // of a bin, in powers of two
  const float first = (float)wt.weight(xhi), rest = (float)rest64;
  float low[kPerThread], high[kPerThread];
  int number[kPerThread];
  Bounds sum{0.0f, 0.0f, 0, 0};
#pragma unroll
  for (int k = 0; k < kPerThread; ++k) {
    number[k] = k < per ? bin_count(b0 + k) : 0;
    low[k] = (float)number[k] * first * exp2_fast(-(float)(b0 + k + 1) * width2) * 0.99999f;
    high[k] = (float)number[k] * first * exp2_fast(-(float)(b0 + k) * width2) * 1.00001f;
    sum.low += low[k];
    sum.high += high[k];
    sum.number += number[k];
  }
  Bounds run = scan_bounds(sum, sm);
  unsigned long long certain = 0, ends = ~0ull;
#pragma unroll
  for (int k = 0; k < kPerThread; ++k)
    if (k < per) {
      run.low += low[k];
      run.high += high[k];
      run.number += number[k];
      const unsigned long long v =
          ((unsigned long long)(b0 + k + 1) << 32) | (unsigned)run.number;
      if (run.high < rest * 0.999999f) certain = v;
      if (run.low >= rest * 1.000001f || b0 + k == kBins - 1) ends = ::min(ends, v);
    }
  const ulonglong2 both = Reducer<false>(&sm.block).all(
      make_ulonglong2(certain, ends), [](ulonglong2 p, ulonglong2 q) {
        return make_ulonglong2(p.x > q.x ? p.x : q.x, p.y < q.y ? p.y : q.y);
      });
  __syncthreads();  // the reduction's scratch is free again
  return {(int)(both.x >> 32) - 1, (int)(uint32_t)both.x, (int)(both.y >> 32) - 1,
          (int)(uint32_t)both.y};
}

// Sums over the list are in whole multiples of 2^-52, as the list's own order
// changes from run to run and must not change the sums: at most 2^11 weights of
// at most 1 fit 64 bits, and lose 2^-42 in all.
constexpr double kFixedOne = 4503599627370496.0;
__device__ __forceinline__ unsigned long long fixed_weight(double w) {
  return __double2ull_rn(w * kFixedOne);
}
// For the draw: a weight above zero counts at least 2^-52, so that u = 0 finds the
// first kept token of any weight; 2^-41 of the mass in all.
__device__ __forceinline__ unsigned long long drawn_weight(double w) {
  const unsigned long long f = fixed_weight(w);
  return f == 0 && w > 0.0 ? 1ull : f;
}

// Three counts of up to kListCap in one word.
__device__ __forceinline__ unsigned long long three_counts(bool a, bool b, bool c) {
  return (a ? 1ull : 0ull) | (b ? 1ull << 20 : 0ull) | (c ? 1ull << 40 : 0ull);
}
__device__ __forceinline__ int count_of(unsigned long long v, int i) {
  return (int)(v >> (20 * i) & 0xfffffu);
}

// Smallest index up to which `want` of the list's n items with that key lie.
__device__ __forceinline__ int nth_index(SampleSmem& sm, int n, uint32_t key, int want) {
  Reducer<false> red(&sm.block);
  int from = 0, to = HKB_VOCAB_MAX - 1;
  while (from < to) {
    const int step = (to - from) / 4 + 1;
    unsigned long long c = 0;
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
      const unsigned long long it = sm.list.item[i];
      const int at = item_index(it);
      if (item_key(it) == key)
        c += three_counts(at < from + step, at < from + 2 * step, at < from + 3 * step);
    }
    c = red.sum(c);
    const int k = count_of(c, 0) >= want ? 0 : count_of(c, 1) >= want ? 1 : count_of(c, 2) >= want ? 2 : 3;
    const int end = ::min(to, from + step * (k + 1) - 1);
    from = ::min(from + step * k, to);
    if (k < 3) to = end;
  }
  __syncthreads();
  return from;
}

// Of the n items of this CTA's list, in order, the one at which the running
// mass, `above` before the first, reaches `need`; 0 if none does.  The bins of
// the row's search again, now of the list's own span, leave a few items; each
// of these adds up what comes before it.
__device__ __forceinline__ unsigned long long border_in_list(SampleSmem& sm, int n,
                                                             const Weights wt, double above,
                                                             double need) {
  Reducer<false> red(&sm.block);
  const int tid = threadIdx.x, threads = blockDim.x;
  const unsigned long long* item = sm.list.item;
  auto weight = [&](float x) { return fixed_weight(wt.weight(x)); };
  const double goal = (need - above) * kFixedOne;  // for the list's own sums
  unsigned long long sum = 0;                      // of its items before xhi
  float xhi = CUDART_INF_F, xlo = -CUDART_INF_F;
  int left = n;
  for (int round = 0; left > kSubList; ++round) {
    // span of the items that are left
    ListExtent ext{0, -CUDART_INF_F, CUDART_INF_F};
    for (int i = tid; i < n; i += threads) {
      const float x = key_value(item_key(item[i]));
      if (x > xhi || x < xlo) continue;
      ext.most = fmaxf(ext.most, x);
      ext.least = fminf(ext.least, x);
    }
    ext = join(red, ext);
    xhi = ext.most;
    xlo = ext.least;
    const float scale = (float)kBins / (xhi - xlo);
    if (xlo < xhi && (!(scale > 0.0f && scale < CUDART_INF_F) || round == 16)) {
      // no width of bins tells them apart (spans near the type's smallest
      // numbers): the border's key by bisection
      auto sum_from = [&](uint32_t key) {
        unsigned long long m = 0;
        for (int i = tid; i < n; i += threads) {
          const uint32_t k = item_key(item[i]);
          if (k >= key && key_value(k) <= xhi) m += weight(key_value(k));
        }
        return red.sum(m);
      };
      uint32_t lo = order_key(xlo), hi = order_key(xhi);
      while (lo < hi) {
        const uint32_t mid = lo + (hi - lo + 1) / 2;
        if ((double)(sum + sum_from(mid)) >= goal) lo = mid;
        else hi = mid - 1;
      }
      if (key_value(lo) < xhi) sum += sum_from(lo + 1);
      xhi = xlo = key_value(lo);
    }
    if (xlo == xhi) {
      // equal logits: by their number
      const double w = (double)weight(xhi);
      const double ties = w > 0.0 ? fmax(1.0, ceil((goal - (double)sum) / w)) : 1.0;
      if (ties > (double)left) return 0;
      __syncthreads();
      return list_item(order_key(xhi), nth_index(sm, n, order_key(xhi), (int)ties));
    }
    auto bin_of = [&](float x) { return ::min(kBins - 1, (int)((xhi - x) * scale)); };
    for (int b = tid; b < kBins; b += threads) sm.hist[b] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += threads) {
      const float x = key_value(item_key(item[i]));
      if (x <= xhi && x >= xlo) atomicAdd(&sm.hist[bin_of(x)], 1u);
    }
    __syncthreads();
    const Bracket br = bracket(sm, scale, wt, xhi, (goal - (double)sum) / kFixedOne,
                               [&](int b) { return (int)sm.hist[b]; });
    ext = ListExtent{0, -CUDART_INF_F, CUDART_INF_F};
    for (int i = tid; i < n; i += threads) {
      const float x = key_value(item_key(item[i]));
      if (x > xhi || x < xlo) continue;
      const int b = bin_of(x);
      if (b <= br.certain) {
        ext.sum += weight(x);
      } else if (b <= br.end) {
        ext.most = fmaxf(ext.most, x);
        ext.least = fminf(ext.least, x);
      }
    }
    ext = join(red, ext);
    sum += ext.sum;
    left = br.upto_end - br.upto_certain;
    xhi = ext.most;
    xlo = ext.least;
  }
  // the items that are left, and the running sum at each of them
  if (tid == 0) sm.sub_count = 0;
  __syncthreads();
  for (int i = tid; i < n; i += threads) {
    const float x = key_value(item_key(item[i]));
    if (x > xhi || x < xlo) continue;
    const unsigned at = atomicAdd(&sm.sub_count, 1u);
    sm.sub[at] = item[i];
    sm.sub_weight[at] = weight(x);
  }
  __syncthreads();
  unsigned long long border = 0;
  if (tid < left) {
    const unsigned long long me = sm.sub[tid];
    unsigned long long run = sum;
#pragma unroll 4
    for (int j = 0; j < left; ++j) run += sm.sub[j] >= me ? sm.sub_weight[j] : 0ull;
    if ((double)run >= goal) border = me;
  }
  return red.max(border);
}

constexpr int kOwnItems = 8;  // kListCap items over at least 256 threads

constexpr int kBuckets = 512;
static_assert(kBuckets * sizeof(unsigned long long) <= kBins * sizeof(unsigned), "in sm.hist");

// Filters and draw for a list of more than kSubList items.  They are sorted for the
// filters; the draw goes by the masses of buckets of neighbouring indices, then by
// the items of the one bucket.  A thread has up to kOwnItems neighbouring places.
// 64 x 131072 bf16, settings per row, 24 batches: 41 to 64 us, median 55; with
// searches over the unsorted list 41 to 76, median 66; sorting by index for the
// draw 39 to 66, median 53, but 4096 x 4000 f32, top-p 0.9: 338 us instead of 272.
__device__ __forceinline__ void finish_long_list(SampleSmem& sm, int n, const Weights wt,
                                                 const RowSettings s, double need, int64_t r,
                                                 const SampleArgs& a) {
  Reducer<false> red(&sm.block);
  const int threads = blockDim.x, tid = threadIdx.x;
  unsigned long long* item = sm.list.item;
  sort_down(item, n);
  const int nk = s.top_k > 0 ? ::min(n, s.top_k) : n;
  const int per = (nk + threads - 1) / threads, first = tid * per;
  unsigned long long own[kOwnItems];  // 0: none
  double w[kOwnItems], sum = 0.0;
#pragma unroll
  for (int j = 0; j < kOwnItems; ++j) {
    own[j] = j < per && first + j < nk ? item[first + j] : 0ull;
    w[j] = own[j] != 0 ? wt.weight(key_value(item_key(own[j]))) : 0.0;
    sum += w[j];
  }
  double total;
  double run = block_scan(sum, sm.seg, &total) - sum;
  if (need < 0.0) need = (double)s.top_p * total;
  int before = 0, heavy = 0;  // places before the border, and those of enough weight
#pragma unroll
  for (int j = 0; j < kOwnItems; ++j) {
    run += w[j];
    before += own[j] != 0 && run < need;
    heavy += own[j] != 0 && w[j] >= (double)s.min_p;
  }
  int kept = nk;
  if (s.top_p < 1.0f) kept = ::min(kept, 1 + red.sum(before));
  if (s.min_p > 0.0f) kept = ::min(kept, red.sum(heavy));
  kept = ::max(kept, 1);

  unsigned long long* bucket = reinterpret_cast<unsigned long long*>(sm.hist);
  int most = 0;
#pragma unroll
  for (int j = 0; j < kOwnItems; ++j) {
    if (first + j >= kept) own[j] = 0;
    if (own[j] != 0) most = ::max(most, item_index(own[j]));
  }
  for (int i = tid; i < kBuckets; i += threads) bucket[i] = 0;
  most = red.max(most);  // and its barrier
  int shift = 0;
  while (most >> shift >= kBuckets) ++shift;
#pragma unroll
  for (int j = 0; j < kOwnItems; ++j)
    if (own[j] != 0) atomicAdd(&bucket[item_index(own[j]) >> shift], drawn_weight(w[j]));
  if (tid == 0) sm.sub_count = 0;
  __syncthreads();
  // a thread has one bucket, or two
  const int pair = kBuckets / threads - 1;
  const unsigned long long m0 = bucket[tid << pair], m1 = pair ? bucket[2 * tid + 1] : 0ull;
  unsigned long long all;
  const unsigned long long upto =
      block_scan(m0 + m1, reinterpret_cast<unsigned long long*>(sm.seg), &all) - (m0 + m1);
  const double target = s.u * (double)all;
  int at = 0x7fffffff, last = -1;
  if (m0 != 0) {
    if ((double)(upto + m0) > target) at = tid << pair;
    last = tid << pair;
  }
  if (m1 != 0) {
    if (at == 0x7fffffff && (double)(upto + m0 + m1) > target) at = 2 * tid + 1;
    last = 2 * tid + 1;
  }
  // (rounding, or u = 1, may leave none: the last with any mass, here and below)
  at = red.min(at);
  last = red.max(last);
  if (at == 0x7fffffff) at = last;
  if (at >> pair == tid) sm.sub_weight[0] = upto + (at != tid << pair ? m0 : 0ull);
#pragma unroll
  for (int j = 0; j < kOwnItems; ++j)
    if (own[j] != 0 && item_index(own[j]) >> shift == at) {
      const unsigned i = atomicAdd(&sm.sub_count, 1u);
      item[2 * i] = (unsigned)item_index(own[j]);
      item[2 * i + 1] = drawn_weight(w[j]);
    }
  __syncthreads();
  const int m = (int)sm.sub_count;  // at most 2^shift <= 512
  int token = 0x7fffffff, end = -1;
  for (int i = tid; i < m; i += threads) {
    const unsigned long long me = item[2 * i];
    if (item[2 * i + 1] == 0) continue;
    unsigned long long sums = sm.sub_weight[0];
    for (int j = 0; j < m; ++j) sums += item[2 * j] <= me ? item[2 * j + 1] : 0ull;
    if ((double)sums > target) token = ::min(token, (int)me);
    end = ::max(end, (int)me);
  }
  token = red.min(token);
  end = red.max(end);
  if (token == 0x7fffffff) token = end;
#pragma unroll
  for (int j = 0; j < kOwnItems; ++j)
    if (own[j] != 0 && item_index(own[j]) == token) {
      a.tokens[r] = token;
      a.log_probs[r] = (float)(wt.exponent(key_value(item_key(own[j]))) * kLn2 -
                               log((double)all / kFixedOne));
      a.kept[r] = kept;
    }
}

// Finishes a row whose kept tokens are all among the n items of this CTA's
// list: puts them in order, cuts them to the shortest head and draws.  `need`
// is the mass that ends the top-p head, or negative: top_p of the mass of the
// first top_k items.  Of a short list each item's place in the order, and its
// running mass in index order, is counted over all items by a group of threads,
// which takes few barriers.
__device__ __forceinline__ void finish_list(SampleSmem& sm, int n, const Weights wt, const RowSettings s,
                            double need, int64_t r, const SampleArgs& a) {
  const int threads = blockDim.x, tid = threadIdx.x;
  if (n > kSubList) {
    finish_long_list(sm, n, wt, s, need, r, a);
    return;
  }
  Reducer<false> red(&sm.block);
  const unsigned long long* item = sm.list.item;
  unsigned long long* sorted = sm.list.item + kListCap / 4;
  double* weight = reinterpret_cast<double*>(sm.list.item + kListCap / 2);
  int group = 32;  // threads an item, a power of two
  while (group > 1 && n * group > threads) group >>= 1;
  const int i = tid / group, part = tid % group;
  const bool mine = i < n, lead = mine && part == 0;
  int place = 0;
  unsigned long long me = 0;
  if (mine) {
    me = item[i];
    place = count_larger(item, n, me, part, group);
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
#pragma unroll 4
    for (int j = part; j < kept; j += group)
      upto += item_index(sorted[j]) <= index ? weight[j] : 0.0;
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

// Long rows in the shared memory of a CTA or a cluster.  Top-k of up to 1024
// collects the few tokens above a bound and lets rank 0 finish; without it the
// mass of the whole row is added up in 64 bits, the top-p border bracketed by
// bins, and the token found by the running masses of CTAs, warps and steps.
//
// Bound by latency with few rows (1 x 32768 f32, top-k: 12 us; cluster barriers
// of about 1000 cycles each; 1 x 131072 bf16, top-p: 82) and by instructions and
// latency together with more (192 x 50001 f16, unfiltered: 38 us, 61 % of issue,
// FP64 pipe 30 %, 40 % of the warps active; 1024 x 32768 f32, top-p: 393).  Top-k
// above 1024 bisects keys instead: 1024 x 32768 f32, top-k 2000: 591.  Slices of
// 64 KB let two CTAs share a SM, those of 128 KB do not; of 32 KB 64 rows of
// 131,072 bf16 took 145 us (top-p) instead of 102.
template <typename T, bool kClustered>
__global__ void __launch_bounds__(kMaxThreads, 2) sample_rows_kernel(
    const T* __restrict__ logits, int64_t row_stride, int vocab, int chunk, SampleArgs a) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  __shared__ SampleSmem sm;
  const int cluster = kClustered ? (int)cg::this_cluster().num_blocks() : 1;
  const int64_t r = blockIdx.x / cluster;
  RowSlice<T, kClustered> row;
  const T* g = logits + r * row_stride;
  row.init(reinterpret_cast<T*>(smem_raw), g, vocab, chunk);
  row.load(g);

  RowSettings s = row_settings(a, r);
  const bool valid = settings_valid(s);
  const bool writer = threadIdx.x == 0 && row.rank == 0;
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

  // Largest logit; a NaN is less than any number in this and every later
  // comparison, so it is never kept.
  float tmax = -CUDART_INF_F;
  row.template for_each_array<4>([&](auto& x) {
    constexpr int n = sizeof(x) / sizeof(x[0]);
#pragma unroll
    for (int u = 0; u < n; ++u) tmax = fmaxf(tmax, x[u].largest());
  });
  // of a row with top-k: a key that ceil(k / C) threads of this CTA reach
  if (s.top_k >= vocab) s.top_k = 0;
  const bool list_k = s.top_k > 0 && s.top_k <= kListCap / 2 && s.temperature > 0.0f;
  const uint32_t reached =
      list_k ? reached_by(order_key(tmax), (s.top_k + row.size - 1) / row.size) : 0;
  const ulonglong2 joint = red.all(make_ulonglong2(order_key(tmax), reached),
                                   [](ulonglong2 p, ulonglong2 q) {
                                     return make_ulonglong2(p.x > q.x ? p.x : q.x,
                                                            p.y < q.y ? p.y : q.y);
                                   });
  float xmax = key_value((uint32_t)joint.x);
  if (xmax == -CUDART_INF_F || s.temperature == 0.0f) {
    const bool none = xmax == -CUDART_INF_F;
    int first = 0x7fffffff;
    if (!none) {
      row.for_each_from(xmax, [&](int i, float x) {
        if (x == xmax) first = ::min(first, i);
      });
      first = red.min(first);
    }
    if (writer) {
      a.tokens[r] = none ? -1 : first;
      a.log_probs[r] = none ? -CUDART_INF_F : 0.0f;
      a.kept[r] = none ? 0 : 1;
    }
    return;
  }
  uint32_t bound = (uint32_t)joint.y;
  double c2 = kLog2e / (double)s.temperature;
  if (xmax == CUDART_INF_F) {
    // Logits of +inf share the whole mass: zeros in their places, the finite
    // ones far below and, by the factor of the exponents, without weight.
    row.for_each([&](int, Vec<T>& x) {
#pragma unroll
      for (int e = 0; e < Vec<T>::kN; ++e) {
        const float v = x.at(e);
        if (v > -CUDART_INF_F)
          reinterpret_cast<T*>(x.w)[e] = narrow<T>(v == CUDART_INF_F ? 0.0f : -60000.0f);
      }
    });
    xmax = 0.0f;
    bound = 0;
    c2 = 1e300;
    __syncthreads();
  }
  const Weights wt{xmax, c2, &sm.table};

  int listed = -1;  // tokens of rank 0's list, where it holds all that can be kept

  // Top-k of a number that fits the list: the k-th largest of the row is no
  // less than the k/C-th largest of the threads' own largest logits in the CTA
  // where that is least, and few more than k tokens reach it.
  if (list_k) {
    const float from = bound <= kKeyNegInf ? -CUDART_MAX_NORMAL_F : key_value(bound);
    const int n = collect(row, red, sm.list, from, [&](int, float x) { return x >= from; });
    if (n <= kListCap) listed = n;
  }
  double list_need = -1.0;  // top_p of the list's own mass

  // The kept head so far: x > xt, or x == xt and index <= icut.
  float xt = -CUDART_MAX_NORMAL_F;
  int icut = 0x7fffffff;
  auto in_head = [&](int i, float x) { return x >= xt && !(x == xt && i > icut); };
  if (listed < 0 && s.top_k > 0) {
    // largest value with at least k tokens at or above it, by bisection of keys
    auto count = [&](uint32_t key) {
      const float from = key_value(key);
      int c = 0;
      row.for_each_from(from, [&](int, float x) { c += x >= from; });
      return red.sum(c);
    };
    if (count(kKeyNegInf + 1) > s.top_k) {
      uint32_t lo = kKeyNegInf + 1, hi = order_key(xmax);
      while (lo < hi) {
        const uint32_t mid = lo + (hi - lo + 1) / 2;
        if (count(mid) >= s.top_k) lo = mid;
        else hi = mid - 1;
      }
      const int above = lo == order_key(xmax) ? 0 : count(lo + 1);
      xt = key_value(lo);
      double ties;
      int n;
      icut = red.max(locate(row, red, sm, xt, (double)(s.top_k - above) - 0.5, true, &ties, &n,
                            [&](int, float x) { return x == xt ? 1.0 : -1.0; }));
    }
  }
  // Distance from the largest logit within which kept tokens lie.
  const double zmin = s.min_p > 0.0f ? log2((double)s.min_p) - 1e-3 : -CUDART_INF;
  float reach = s.min_p > 0.0f ? (float)(-zmin / wt.c2) * 1.000001f : CUDART_INF_F;

  if (listed < 0 && s.top_p < 1.0f) {
    double m = 0.0;
    row.for_each_from(xt, [&](int i, float x) {
      const double w = wt.weight(x);
      m += in_head(i, x) ? w : 0.0;
    });
    const double mass = red.sum(m);
    const double need = (double)s.top_p * mass;
    // Tokens lighter than (1 - p) * mass / V have less than (1 - p) * mass
    // together, so the border lies above them.
    const double z0 =
        fmax(zmin, log2((1.0 - (double)s.top_p) * mass / (double)vocab) - 1e-3);
    reach = (float)(-z0 / wt.c2) * 1.000001f;
    // The border lies between xhi and xlo, `above` is the mass of the head
    // before xhi.  The tokens between are counted in bins of equal width: a
    // bin's weights lie between those of its ends, so the counts bound the
    // running mass from both sides, and the border lies in the few bins that
    // the two bounds leave.  They are put in
    // order, or divided again while they are too many for the list.
    float xhi = xmax, xlo = fmaxf(xt, xmax - reach * 1.00001f);
    double above = 0.0;
    bool found = false;
    for (int round = 0; round < 8 && !found && listed < 0 && xlo < xhi; ++round) {
      const float scale = (float)kBins / (xhi - xlo);
      // temperatures at the ends of the type's range leave no finite bin width
      if (!(scale > 0.0f && scale < CUDART_INF_F)) break;
      auto within = [&](int i, float x) { return x >= xlo && x <= xhi && in_head(i, x); };
      auto bin_of = [&](float x) { return ::min(kBins - 1, (int)((xhi - x) * scale)); };
      for (int b = threadIdx.x; b < kBins; b += blockDim.x) sm.hist[b] = 0;
      __syncthreads();
      row.for_each_from(xlo, [&](int i, float x) {
        if (within(i, x)) atomicAdd(&sm.hist[bin_of(x)], 1u);
      });
      if (kClustered) cg::this_cluster().sync();
      else __syncthreads();
      // every CTA adds up the whole row's bins and finds the same border
      const Bracket br = bracket(
          sm, scale, wt, xhi, need - above, [&](int b) {
            if (!kClustered) return (int)sm.hist[b];
            int c = 0;
            for (int k = 0; k < row.size; ++k)
              c += (int)cg::this_cluster().map_shared_rank(sm.hist, k)[b];
            return c;
          });
      if (round == 0 && br.upto_end <= kListCap) {
        const int n = collect(row, red, sm.list, xlo, [&](int i, float x) {
          return within(i, x) && bin_of(x) <= br.end;
        });
        listed = n;
        list_need = need;
        break;
      }
      // the mass before the uncertain bins, and the tokens in them or their span
      const bool fits = br.upto_end - br.upto_certain <= kListCap;
      Extent ext{0.0, -CUDART_INF_F, CUDART_INF_F};
      const int n = collect(row, red, sm.list, xlo, [&](int i, float x) {
        const bool in = within(i, x);
        const int b = in ? bin_of(x) : kBins;
        const double w = wt.weight(x);
        ext.mass += b <= br.certain ? w : 0.0;
        const bool open = b > br.certain && b <= br.end;
        ext.most = open ? fmaxf(ext.most, x) : ext.most;
        ext.least = open ? fminf(ext.least, x) : ext.least;
        return open && fits;
      });
      ext = red.all(ext, [](Extent p, Extent q) {
        return Extent{p.mass + q.mass, fmaxf(p.most, q.most), fminf(p.least, q.least)};
      });
      above += ext.mass;
      if (fits) {
        // the head ends inside the list, or (cut by min-p) nowhere
        unsigned long long border = 0;
        if (row.rank == 0) border = border_in_list(sm, n, wt, above, need);
        border = red.spread(border)[0];
        if (border != 0) {
          xt = key_value(item_key(border));
          icut = item_index(border);
        }
        found = true;
      }
      xhi = ext.most;
      xlo = ext.least;
    }
    if (!found && listed < 0) {
      if (xlo < xhi) {
        // by bisection of keys; only for temperatures without a bin width
        auto mass_from = [&](uint32_t key) {
          const float from = key_value(key);
          double v = 0.0;
          row.for_each_from(from, [&](int i, float x) {
            if (x >= from && in_head(i, x)) v += wt.weight(x);
          });
          return red.sum(v);
        };
        uint32_t lo = order_key(xlo), hi = order_key(xhi);
        while (lo < hi) {
          const uint32_t mid = lo + (hi - lo + 1) / 2;
          if (mass_from(mid) >= need) lo = mid;
          else hi = mid - 1;
        }
        xhi = key_value(lo);
        above = lo == order_key(xmax) ? 0.0 : mass_from(lo + 1);
      }
      // the head ends among the tokens that equal xhi: the first `ties` are kept
      const double w = wt.weight(xhi);
      double ties = w > 0.0 ? ceil((need - above) / w) : 1.0;
      if (ties < 1.0) ties = 1.0;
      double all_ties;
      int n;
      icut = red.max(locate(row, red, sm, xhi, ties - 0.5, true, &all_ties, &n,
                            [&](int i, float x) { return x == xhi && in_head(i, x) ? 1.0 : -1.0; }));
      xt = xhi;
    }
  }
  if (listed >= 0) {
    if (row.rank == 0) finish_list(sm, listed, wt, s, list_need, r, a);
    return;
  }
  // draw among the kept tokens of the whole row
  const float skip = fmaxf(xt, xmax - reach * 1.00001f);
  double total;
  int n;
  const int token = locate(row, red, sm, skip, s.u, false, &total, &n, [&](int i, float x) {
    const double w = wt.weight(x);
    return in_head(i, x) && w >= (double)s.min_p ? w : -1.0;
  });
  if (token >= 0 && (threadIdx.x & 31) == 0) {
    const float x = fminf(widen(g[token]), xmax);
    a.tokens[r] = token;
    a.log_probs[r] = (float)(wt.exponent(x) * kLn2 - log(total));
    a.kept[r] = n;
  }
}

// Rows of up to kWarpVocab tokens, a warp each.  As for the short rows below,
// the head is found with 32-bit weights, by bisection of the logits' keys, and
// again with 64-bit ones where a comparison with the border is too close (or
// where equal logits share the border: their number needs the exact masses).
// Bound by instructions: 415,936 x 143 f32, settings per row (nine in ten with a
// top-p below 1), 1.16 ms (9.5 ms with a CTA a row, whose barriers and set-up such
// rows do not repay); top-p 0.9 1.09, unfiltered 0.40.
template <typename T, int kPer>
__global__ void __launch_bounds__(32 * kWarpRows) sample_warp_kernel(
    const T* __restrict__ logits, int64_t row_stride, int64_t n_rows, int vocab, SampleArgs a) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  __shared__ Exp2Table table;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t r = (int64_t)blockIdx.x * kWarpRows + warp;
  WarpRow<T, kPer> row;
  RowSettings s{};
  if (r < n_rows) {
    row.stage(reinterpret_cast<T*>(smem_raw + warp * WarpRow<T, kPer>::bytes(vocab)),
              logits + r * row_stride, vocab);
    s = row_settings(a, r);
  }
  table.fill();
  cp_async_wait_all();
  __syncthreads();
  if (r >= n_rows) return;
  if (!settings_valid(s)) {
    if (lane == 0) {
      a.tokens[r] = -1;
      a.log_probs[r] = CUDART_NAN_F;
      a.kept[r] = 0;
    }
    return;
  }
  row.read();
  const float xmax = row.largest();
  if (xmax == -CUDART_INF_F || s.temperature == 0.0f) {
    int first = -1;
#pragma unroll
    for (int e = kPer - 1; e >= 0; --e)
      if (row.x[e] == xmax) first = lane * kPer + e;
    const bool none = xmax == -CUDART_INF_F;
    const unsigned has = __ballot_sync(0xffffffffu, first >= 0);
    if (lane == (none ? 0 : __ffs(has) - 1)) {
      a.tokens[r] = none ? -1 : first;
      a.log_probs[r] = none ? -CUDART_INF_F : 0.0f;
      a.kept[r] = none ? 0 : 1;
    }
    return;
  }
  const double c2 = kLog2e / (double)s.temperature;
  auto exponent = [&](float x) { return x == xmax ? 0.0 : ((double)x - (double)xmax) * c2; };
  unsigned keep = 0;
#pragma unroll
  for (int e = 0; e < kPer; ++e) keep |= (row.x[e] > -CUDART_INF_F ? 1u : 0u) << e;
  if (s.top_k > 0 && s.top_k < (int)__reduce_add_sync(0xffffffffu, __popc(keep))) {
    const float t = row.nth_largest(s.top_k, xmax);
    int above = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) above += row.x[e] > t;
    above = __reduce_add_sync(0xffffffffu, above);
    keep = row.head(keep, t, s.top_k - above);
  }
  if (s.top_p < 1.0f) {
    const float c = (float)c2;
    float w[kPer], sum = 0.0f;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const float x = row.x[e];
      w[e] = keep >> e & 1u ? exp2_fast((x == xmax ? 0.0f : x - xmax) * c) : 0.0f;
      sum += w[e];
    }
    sum = warp_total(sum);
    const float need = s.top_p * sum, slack = 4e-6f * sum;
    uint32_t lo = kKeyNegInf + 1, hi = order_key(xmax);
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo + 1) / 2;
      const float from = key_value(mid);
      float m = 0.0f;
#pragma unroll
      for (int e = 0; e < kPer; ++e) m += row.x[e] >= from ? w[e] : 0.0f;
      if (warp_total(m) >= need) lo = mid;
      else hi = mid - 1;
    }
    float t = key_value(lo), at = 0.0f, over = 0.0f;
    int ties = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      at += row.x[e] >= t ? w[e] : 0.0f;
      over += row.x[e] > t ? w[e] : 0.0f;
      ties += row.x[e] == t && (keep >> e & 1u);
    }
    at = warp_total(at);
    over = warp_total(over);
    ties = __reduce_add_sync(0xffffffffu, ties);
    // 32 bits see nothing where differences of logits overflow them (the largest
    // temperatures) or their scale does (below 4.24e-39: 0 * inf is NaN)
    const bool blind = s.temperature > 1e30f || c == CUDART_INF_F;
    if (blind || ties > 1 || !(at - need > slack && need - over > slack)) {
      // In 64 bits: from the largest value that 32 bits cannot rule out (or the
      // row's largest) down, value by value, until the mass is reached or no
      // smaller value is left.
      float from = xmax;
      if (!blind) {
        lo = order_key(t);
        hi = order_key(xmax);
        while (lo < hi) {
          const uint32_t mid = lo + (hi - lo + 1) / 2;
          const float at_least = key_value(mid);
          float m = 0.0f;
#pragma unroll
          for (int e = 0; e < kPer; ++e) m += row.x[e] >= at_least ? w[e] : 0.0f;
          if (warp_total(m) >= need - slack) lo = mid;
          else hi = mid - 1;
        }
        from = key_value(lo);
      }
      double mass = 0.0, above = 0.0;
#pragma unroll 1
      for (unsigned b = keep; b != 0; b &= b - 1) {
        const float x = widen(row.s[row.ph + lane * kPer + __ffs(b) - 1]);
        const double v = table(exponent(x));
        mass += v;
        above += x > from ? v : 0.0;
      }
      mass = warp_total(mass);
      above = warp_total(above);
      const double border = (double)s.top_p * mass;
      for (t = from;;) {
        float next = -CUDART_INF_F;
        ties = 0;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
          const bool in = keep >> e & 1u;
          ties += in && row.x[e] == t;
          next = in && row.x[e] < t ? fmaxf(next, row.x[e]) : next;
        }
        ties = __reduce_add_sync(0xffffffffu, ties);
        next = key_value(__reduce_max_sync(0xffffffffu, order_key(next)));
        const double each = table(exponent(t));
        const double upto = above + (double)ties * each;
        if (upto >= border || next == -CUDART_INF_F) {
          const double n = each > 0.0 ? ceil((border - above) / each) : 1.0;
          ties = (int)fmin(fmax(n, 1.0), (double)ties);
          break;
        }
        above = upto;
        t = next;
      }
    }
    keep = row.head(keep, t, ties);
  }
  // the kept mass; with min-p, of those heavy enough
  double mine = 0.0;
#pragma unroll
  for (int e = 0; e < kPer; ++e)
    if (keep >> e & 1u) {
      const double w = table(exponent(row.x[e]));
      if (w >= (double)s.min_p) mine += w;
      else keep &= ~(1u << e);
    }
  const int kept = __reduce_add_sync(0xffffffffu, __popc(keep));
  double upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double y = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += y;
  }
  const double total = __shfl_sync(0xffffffffu, upto, 31), target = s.u * total;
  // the lane in which the running mass passes the target (rounding, or u = 1,
  // may leave none: the last with any mass), then its token, a lane for each
  const unsigned pass = __ballot_sync(0xffffffffu, mine > 0.0 && upto > target);
  const unsigned any = __ballot_sync(0xffffffffu, mine > 0.0);
  const int hit = pass ? __ffs(pass) - 1 : 31 - __clz(any);
  const double before = __shfl_sync(0xffffffffu, upto - mine, hit);
  const unsigned bits = __shfl_sync(0xffffffffu, keep, hit);
  const int token = hit * kPer + lane;
  float x = -CUDART_INF_F;
  double w = 0.0;
  if (lane < kPer && (bits >> lane & 1u)) {
    x = widen(row.s[row.ph + token]);
    w = table(exponent(x));
  }
  double run = w;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double y = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += y;
  }
  const unsigned over = __ballot_sync(0xffffffffu, w > 0.0 && before + run > target);
  const unsigned some = __ballot_sync(0xffffffffu, w > 0.0);
  if (lane == (over ? __ffs(over) - 1 : 31 - __clz(some))) {
    a.tokens[r] = token;
    a.log_probs[r] = (float)(exponent(x) * kLn2 - log(total));
    a.kept[r] = kept;
  }
}

// Short rows, one thread each.  The head is found with 32-bit weights, whose
// sums are off by less than 2e-6 of the mass (2 ulp of the function, three
// roundings of an exponent, 31 of the sum); a row where a comparison with a
// border is closer than twice that repeats it with 64-bit weights.  The kept
// tokens' mass and the draw are in 64 bits, so their number sets the time on
// the 64-bit pipe, not V.
//
// 524,288 x 21 f32, top-p and min-p: 47 us (8 us of memory traffic), 65 % of the
// issue rate; taking the largest remaining token until the filters stop took 75.
template <typename T, int kPad>
__global__ void __launch_bounds__(kShortRows) sample_short_kernel(const T* __restrict__ logits,
                                                                  int64_t row_stride, int64_t n_rows,
                                                                  int vocab, SampleArgs a) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  __shared__ Exp2Table table;
  double* weight = reinterpret_cast<double*>(smem_raw) + threadIdx.x;  // [i * kShortRows]
  const int64_t r0 = (int64_t)blockIdx.x * kShortRows, r = r0 + threadIdx.x;
  const int rows = (int)::min((int64_t)kShortRows, n_rows - r0), tid = threadIdx.x;
  ShortRows<T> sr;
  sr.load(reinterpret_cast<T*>(smem_raw + sizeof(double) * kShortRows * vocab),
          logits + r0 * row_stride, row_stride, rows, vocab);
  table.fill();
  RowSettings s{};
  if (tid < rows) s = row_settings(a, r);
  cp_async_wait_all();
  __syncthreads();
  if (tid >= rows) return;
  if (!settings_valid(s)) {
    a.tokens[r] = -1;
    a.log_probs[r] = CUDART_NAN_F;
    a.kept[r] = 0;
    return;
  }
  auto value = [&](int i) { return widen(sr.at(tid, i)); };
  float xmax = -CUDART_INF_F;
  int best = -1;
  unsigned live = 0;  // tokens above -inf
#pragma unroll
  for (int i = 0; i < kPad; ++i)
    if (i < vocab) {
      const float v = value(i);
      if (v > xmax) {
        xmax = v;
        best = i;
      }
      live |= (v > -CUDART_INF_F ? 1u : 0u) << i;
    }
  if (best < 0 || s.temperature == 0.0f) {
    a.tokens[r] = best;
    a.log_probs[r] = best < 0 ? -CUDART_INF_F : 0.0f;
    a.kept[r] = best < 0 ? 0 : 1;
    return;
  }
  const double c2 = kLog2e / (double)s.temperature;
  auto exponent = [&](float x) { return x == xmax ? 0.0 : ((double)x - (double)xmax) * c2; };
  unsigned keep = live;
  const bool cut_k = s.top_k > 0 && s.top_k < __popc(live);
  if (cut_k || s.top_p < 1.0f) {
    uint32_t key[kPad];
    sort_short(key, vocab, sizeof(T) == 2, value);
    const int nk = cut_k ? s.top_k : __popc(live);
    const float c = (float)c2;
    // 32-bit weights, in the places of the 64-bit ones
    auto light = [&](int i) -> float& {
      return *reinterpret_cast<float*>(weight + i * kShortRows);
    };
    float sum = 0.0f;
    if (s.top_p < 1.0f) {
#pragma unroll
      for (int i = 0; i < kPad; ++i)
        if (i < vocab) {
          const float x = value(i);
          const float w = x > -CUDART_INF_F ? exp2_fast((x == xmax ? 0.0f : x - xmax) * c) : 0.0f;
          light(i) = w;
          sum += w;
        }
    }
    if (cut_k) {
      keep = 0;
      sum = 0.0f;
#pragma unroll
      for (int j = 0; j < kPad; ++j) {
        if (j >= nk) break;
        const int i = 31 - (int)(key[j] & 31);
        keep |= 1u << i;
        if (s.top_p < 1.0f) sum += light(i);
      }
    }
    if (s.top_p < 1.0f) {
      const float need = s.top_p * sum, slack = 4e-6f * sum;
      unsigned head = 0;
      float run = 0.0f;
      // 32-bit differences of logits may overflow, or their scale
      bool close = s.temperature > 1e30f || c == CUDART_INF_F;
#pragma unroll
      for (int j = 0; j < kPad; ++j) {
        if (j >= nk || (j > 0 && !(run < need))) break;
        const int i = 31 - (int)(key[j] & 31);
        head |= 1u << i;
        run += light(i);
        close |= fabsf(run - need) < slack;
      }
      if (close) {
        // in 64 bits, over the order in shared memory
        signed char* order = reinterpret_cast<signed char*>(weight);
        double mass = 0.0;
#pragma unroll
        for (int j = 0; j < kPad; ++j)
          if (j < vocab) order[j / 8 * kShortRows * 8 + j % 8] = (signed char)(31 - (key[j] & 31));
        for (int j = 0; j < nk; ++j)
          mass += table(exponent(value(order[j / 8 * kShortRows * 8 + j % 8])));
        const double border = (double)s.top_p * mass;
        double upto = 0.0;
        head = 0;
        for (int j = 0; j < nk && (j == 0 || upto < border); ++j) {
          const int i = order[j / 8 * kShortRows * 8 + j % 8];
          head |= 1u << i;
          upto += table(exponent(value(i)));
        }
      }
      keep = head;
    }
  }
  // the kept tokens' mass in index order; with min-p, of those heavy enough
  double total = 0.0;
  for (unsigned m = keep; m != 0; m &= m - 1) {
    const int i = __ffs(m) - 1;
    const double w = table(exponent(value(i)));
    weight[i * kShortRows] = w;
    if (w >= (double)s.min_p) total += w;
    else keep &= ~(1u << i);
  }
  const double target = s.u * total;
  double run = 0.0;
  int token = best;
  for (unsigned m = keep; m != 0 && !(run > target); m &= m - 1) {
    const int i = __ffs(m) - 1;
    const double w = weight[i * kShortRows];
    run += w;
    if (w > 0.0) token = i;
  }
  a.tokens[r] = token;
  a.log_probs[r] = (float)(exponent(value(token)) * kLn2 - log(total));
  a.kept[r] = __popc(keep);
}

template <typename T>
cudaError_t launch(cudaStream_t st, const VocabRows& v, const SampleArgs& a) {
  if (v.vocab <= kShortVocab) {
    const int smem = ShortRows<T>::bytes(v.vocab) + (int)sizeof(double) * kShortRows * v.vocab;
    const unsigned blocks = (unsigned)((v.rows + kShortRows - 1) / kShortRows);
    HKB_SHORT_WIDTH(v.vocab, {
      ensure_dynamic_smem((const void*)sample_short_kernel<T, kPad>,
                          ShortRows<T>::bytes(kPad) + (int)sizeof(double) * kShortRows * kPad);
      sample_short_kernel<T, kPad><<<blocks, kShortRows, smem, st>>>(
          static_cast<const T*>(v.logits), v.row_stride, v.rows, v.vocab, a);
    });
    return cudaGetLastError();
  }
  if (use_warp_rows(v.rows, v.vocab)) {
    const int smem = kWarpRows * WarpRow<T, 1>::bytes(v.vocab);
    const unsigned blocks = (unsigned)((v.rows + kWarpRows - 1) / kWarpRows);
    HKB_WARP_WIDTH(v.vocab, (sample_warp_kernel<T, kPer><<<blocks, 32 * kWarpRows, smem, st>>>(
                                static_cast<const T*>(v.logits), v.row_stride, v.rows, v.vocab, a)));
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
