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
  s.threads = std::min(vocab::kMaxThreads, std::max(32, (vecs / 2 + 31) / 32 * 32));
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

struct SampleSmem {
  ReduceScratch red;
  double seg[kMaxWarps];
  int found;
};

// First token, in index order, whose running sum of f exceeds `target`, over
// the whole row; every thread of the cluster gets it.  f(index, value) >= 0.
// Rounding may leave the sum at the end no larger than the target: then the
// last token with f > 0 is it.  -1 if there is none.
template <typename T, bool kClustered, typename F>
__device__ int locate(const RowSlice<T, kClustered>& row, Reducer<kClustered>& red, SampleSmem& sm,
                      double share, bool absolute, double* total_out, F f) {
  constexpr int kE = Vec<T>::kN;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = (int)blockDim.x >> 5;
  double mine = 0.0;
  int last = -1;
  row.for_each([&](int i0, const Vec<T>& x) {
#pragma unroll
    for (int e = 0; e < kE; ++e) {
      const double w = f(i0 + e, widen(x.v[e]));
      mine += w;
      if (w > 0.0) last = i0 + e;
    }
  });
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  __syncthreads();
  if (lane == 0) sm.seg[warp] = mine;
  if (threadIdx.x == 0) sm.found = -1;
  __syncthreads();
  // mass of this CTA, of the row, and of the CTAs before this one
  double cta = 0.0;
  for (int w = 0; w < warps; ++w) cta += sm.seg[w];
  double before = 0.0, total = cta;
  if (kClustered) {
    // one reduction per CTA's value: the sums below run in rank order
    total = 0.0;
    for (int c = 0; c < row.size; ++c) {
      const double v = red.max(c == row.rank ? cta : 0.0);
      if (c < row.rank) before += v;
      total += v;
    }
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
        w[e] = v < end ? f(i0 + e, widen(reinterpret_cast<const Vec<T>*>(row.s)[v].v[e])) : 0.0;
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
  // at most one CTA found it; the largest also serves the fallback
  const int found = red.max(sm.found);
  if (found >= 0) return found;
  return red.max(last);
}

template <typename T, bool kClustered>
__global__ void __launch_bounds__(kMaxThreads) sample_rows_kernel(
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

  const float Tf = a.temperatures ? a.temperatures[r] : a.temperature;
  const int topk = a.top_ks ? a.top_ks[r] : a.top_k;
  const float top_p = a.top_ps ? a.top_ps[r] : a.top_p;
  const float min_p = a.min_ps ? a.min_ps[r] : a.min_p;
  const double u = a.uniforms_f64 ? static_cast<const double*>(a.uniforms)[r]
                                  : (double)static_cast<const float*>(a.uniforms)[r];
  const bool valid = settings_valid(Tf, topk, top_p, min_p, u);
  const bool writer = threadIdx.x == 0 && row.rank == 0;
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
  uint32_t kbest = 0;
  int ibest = 0x7fffffff;
  row.for_each([&](int i0, Vec<T>& x) {
    bool nan = false;
#pragma unroll
    for (int e = 0; e < kE; ++e) {
      const float v = widen(x.v[e]);
      if (v != v) {
        x.v[e] = narrow<T>(-CUDART_INF_F);
        nan = true;
        continue;
      }
      const uint32_t k = order_key(v);
      if (k > kbest) {
        kbest = k;
        ibest = i0 + e;
      }
    }
    (void)nan;
  });
  const unsigned long long best = red.max(((unsigned long long)kbest << 32) | (uint32_t)~ibest);
  const uint32_t kmax = (uint32_t)(best >> 32);
  if (kmax <= kKeyNegInf || Tf == 0.0f) {
    if (writer) {
      const bool none = kmax <= kKeyNegInf;
      a.tokens[r] = none ? -1 : (int)~(uint32_t)best;
      a.log_probs[r] = none ? -CUDART_INF_F : 0.0f;
      a.kept[r] = none ? 0 : 1;
    }
    return;
  }
  const float xmax = key_value(kmax);
  const double c2 = kLog2e / (double)Tf;
  auto exponent = [&](float x) { return x == xmax ? 0.0 : ((double)x - (double)xmax) * c2; };

  // The kept head is { (key, index) : key > t, or key == t and index <= icut }.
  uint32_t t = kKeyNegInf + 1;
  int icut = 0x7fffffff;
  auto in_head = [&](int i, uint32_t k) { return k > t || (k == t && i <= icut); };

  if (topk > 0 && topk < vocab) {
    // largest key with at least k tokens at or above it
    auto count = [&](uint32_t lo) {
      int c = 0;
      row.for_each([&](int, const Vec<T>& x) {
#pragma unroll
        for (int e = 0; e < kE; ++e) c += order_key(widen(x.v[e])) >= lo;
      });
      return red.sum(c);
    };
    if (count(kKeyNegInf + 1) > topk) {
      uint32_t lo = kKeyNegInf + 1, hi = kmax;
      while (lo < hi) {
        const uint32_t mid = lo + (hi - lo + 1) / 2;
        if (count(mid) >= topk) lo = mid;
        else hi = mid - 1;
      }
      t = lo;
      const int above = t == 0xffffffffu ? 0 : count(t + 1);
      double ties;
      icut = locate(row, red, sm, (double)(topk - above) - 0.5, true, &ties,
                    [&](int, float x) { return order_key(x) == t ? 1.0 : 0.0; });
    }
  }
  if (top_p < 1.0f) {
    auto mass = [&](uint32_t lo) {
      double m = 0.0;
      row.for_each([&](int i0, const Vec<T>& x) {
#pragma unroll
        for (int e = 0; e < kE; ++e) {
          const float v = widen(x.v[e]);
          const uint32_t k = order_key(v);
          if (k >= lo && in_head(i0 + e, k)) m += exp2_neg(exponent(v));
        }
      });
      return red.sum(m);
    };
    const double need = (double)top_p * mass(t);
    uint32_t lo = t, hi = kmax;
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo + 1) / 2;
      if (mass(mid) >= need) lo = mid;
      else hi = mid - 1;
    }
    // `lo` is the border's key: of its tokens the first m are kept
    const double above = lo == kmax ? 0.0 : mass(lo + 1);
    const double w = exp2_neg(exponent(key_value(lo)));
    double m = w > 0.0 ? ceil((need - above) / w) : 1.0;
    if (m < 1.0) m = 1.0;
    const uint32_t old_t = t;
    const int old_cut = icut;
    t = lo;
    icut = 0x7fffffff;
    double ties;
    icut = locate(row, red, sm, m - 0.5, true, &ties, [&](int i, float x) {
      const uint32_t k = order_key(x);
      return k == lo && (k > old_t || i <= old_cut) ? 1.0 : 0.0;
    });
  }
  double total;
  int n = 0;
  const int token = locate(row, red, sm, u, false, &total, [&](int i, float x) {
    const uint32_t k = order_key(x);
    if (!in_head(i, k)) return 0.0;
    const double w = exp2_neg(exponent(x));
    return w >= (double)min_p ? w : 0.0;
  });
  row.for_each([&](int i0, const Vec<T>& x) {
#pragma unroll
    for (int e = 0; e < kE; ++e) {
      const float v = widen(x.v[e]);
      n += in_head(i0 + e, order_key(v)) &&
           (min_p == 0.0f || exp2_neg(exponent(v)) >= (double)min_p);
    }
  });
  n = red.sum(n);
  if (writer) {
    const float x = widen(g[token]);
    a.tokens[r] = token;
    a.log_probs[r] = (float)(exponent(x) * kLn2 - log(total));
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
  double* w = reinterpret_cast<double*>(smem_raw) + threadIdx.x;  // [i * kShortRows]
  float* xs = reinterpret_cast<float*>(smem_raw + sizeof(double) * kShortRows * vocab);
  const int64_t r0 = (int64_t)blockIdx.x * kShortRows;
  const int rows = (int)::min((int64_t)kShortRows, n_rows - r0);
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
    const double wi = exp2_neg(v == xmax ? 0.0 : ((double)v - (double)xmax) * c2);
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
