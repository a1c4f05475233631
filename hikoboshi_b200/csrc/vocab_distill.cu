// Divergence of student rows from a teacher's listed logits, and its gradient.
//
// With M the row's largest logit, S = sum exp((x_i - M) / tau) and the
// teacher's masses q_k (in 64 bits, K of them), the loss needs S, the K listed
// logits and, where the unlisted tokens form a class, their own sum.  That sum
// is taken over the row with the listed entries replaced by -inf, not as a
// difference of sums: a student that puts almost everything on the list would
// lose it to cancellation.  The gradient is e_i G for every unlisted token,
// with e_i recomputed from the row in shared memory and one factor G per row,
// and is set entry by entry on the list.
#include <type_traits>

#include "hkb_mpnn.h"
#include "kernels.hpp"
#include "vocab.hpp"
#include "vocab_rows.cuh"

namespace hkb {
namespace vocab {
namespace {

constexpr double kLog2e = 1.4426950408889634074;

// The loss carries temperature^2 and the listed gradient temperature, while the
// divergence itself falls with them: an error of the row's sum of weights, up to
// 2e-7 with 32-bit exponentials, comes out as temperature^2 times that.  At 16
// that is 5e-5 of a loss of about one, at 100 a thousandth, at 1e4 nothing is
// left.  Above kWideTemperature the weights and their sums are therefore 64-bit
// (kWide): off by temperature^2 * 1e-14 at most, 1e-6 at the largest temperature
// that is accepted.  What that costs (us, loss and gradient, 32 and 64 bits):
// 524,288 x 21 f32 53 and 87; 100,000 x 100 bf16 49 and 78; 48 x 1009 f16 11 and 12;
// 2000 x 50001 bf16 103 and 287; 4096 x 131072 bf16 488 and 1139.
constexpr double kWideTemperature = 16.0;

template <int kBytes>
struct BitsOf;
template <>
struct BitsOf<4> {
  using type = uint32_t;
};
template <>
struct BitsOf<2> {
  using type = uint16_t;
};

__device__ __forceinline__ float load_value(const void* p, int dtype, int64_t i) {
  if (dtype == HKB_F32) return static_cast<const float*>(p)[i];
  if (dtype == HKB_F16) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

// Whether an entry makes its row NaN: a token outside the vocabulary, or a value
// that is NaN or +inf (one of -inf is no entry).  Tested before the masses are
// taken: with an infinite log-norm or value they would be 0 or inf, and the row's
// loss a number that stands for nothing.
__device__ __forceinline__ bool bad_entry(int token, float v, int vocab) {
  return token >= vocab || !(v < CUDART_INF_F);
}
// Likewise the log-norm of a row with entries.
__device__ __forceinline__ bool bad_norm(const float* log_norm, int64_t r) {
  return log_norm != nullptr && !(fabsf(log_norm[r]) < CUDART_INF_F);
}

// What a row's loss and gradient need beside the row.
struct RowFactors {
  float base;     // of the body's exponents
  double F;       // gradient of an unlisted token: exp2((x - base) c) * F * Q
  double each, Q; // gradient on the list: Q each exp((x - xmax) / tau) - Q q
  double total;   // of the row's weights, relative to its largest logit
  double mass;    // the teacher's
  double rest_q;  // of it, the unlisted tokens' where they are a class
};

// The body's largest logit and sum (relative to it), the row's largest logit
// and, where the unlisted tokens are a class of their own (the body), the sum of
// the listed ones relative to it; q_sum is the listed masses' sum: 1, or NaN,
// without the class.
__device__ __forceinline__ RowFactors row_factors(bool tail, float bmax, double body, float xmax,
                                                  double listed, double q_sum, double inv_tau,
                                                  double temperature, float weight) {
  RowFactors f;
  const double lift = bmax == xmax           ? 1.0
                      : bmax == -CUDART_INF_F ? 0.0
                                              : exp(((double)bmax - (double)xmax) * inv_tau);
  f.total = body * lift + listed;
  f.rest_q = tail && bmax != -CUDART_INF_F ? fmax(0.0, 1.0 - q_sum) : 0.0;
  f.mass = q_sum + f.rest_q;
  const double each = f.mass / f.total;
  f.base = bmax == -CUDART_INF_F ? 0.0f : bmax;
  f.F = each * lift - (f.rest_q > 0.0 ? f.rest_q / body : 0.0);
  f.each = each;
  f.Q = (double)weight * temperature;
  return f;
}

__device__ __forceinline__ double listed_gradient(double Q, double each, double e, double q) {
  return __dmul_rn(__dmul_rn(Q, each), e) - __dmul_rn(Q, q);
}

// What a backward pass needs of a row's forward pass.
enum StatFlags { kStatBad = 1, kStatEmpty = 2, kStatTwice = 4 };
__device__ __forceinline__ void write_stats(double* stats, int64_t r, const RowFactors& f,
                                            double q_scale, float xmax, float from, int flags) {
  double* s = stats + r * HKB_DISTILL_STATS;
  s[0] = f.F;
  s[1] = f.each;
  s[2] = q_scale;
  s[3] = __hiloint2double(__float_as_int(f.base), __float_as_int(xmax));
  s[4] = __hiloint2double(__float_as_int(from), flags);
}

// dot = sum q (log q - (x - xmax) / tau).  Everything is relative to the row's
// largest logit, so logits of any size leave the loss its digits.
__device__ __forceinline__ float row_loss(const RowFactors& f, double dot, float bmax, float xmax,
                                          double body, double inv_tau, double temperature) {
  double l = dot + f.mass * log(f.total);
  if (f.rest_q > 0.0)
    l += f.rest_q * (log(f.rest_q / body) - ((double)bmax - (double)xmax) * inv_tau);
  return (float)(temperature * temperature * l);
}

// exp((x - ref) / tau) in 64 bits for x <= ref, c2 = log2(e) / tau; NaN for a NaN
// and for x = ref = +-inf.
__device__ __forceinline__ double wide_weight(float x, float ref, double c2,
                                              const Exp2Table& table) {
  const double t = ((double)x - (double)ref) * c2;
  return t <= 0.0 ? table(t) : t;
}

// SoftSum in 64 bits.
struct WideSum {
  float m;
  double s;

  __device__ __forceinline__ WideSum() : m(-INFINITY), s(0.0) {}

  template <typename T, int kU>
  __device__ __forceinline__ void add(Vec<T> (&x)[kU], double c2, const Exp2Table& table) {
    float vm = x[0].largest();
#pragma unroll
    for (int u = 1; u < kU; ++u) vm = fmaxf(vm, x[u].largest());
    if (vm > m) {
      s *= table(((double)m - (double)vm) * c2);
      m = vm;
    }
    const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int u = 0; u < kU; ++u)
#pragma unroll
      for (int e = 0; e < Vec<T>::kN; ++e) s += wide_weight(x[u].at(e), ref, c2, table);
  }
  __device__ __forceinline__ static WideSum join(WideSum a, WideSum b, double c2) {
    WideSum r;
    r.m = fmaxf(a.m, b.m);
    const double fa = a.m == r.m ? 1.0 : exp2(((double)a.m - (double)r.m) * c2);
    const double fb = b.m == r.m ? 1.0 : exp2(((double)b.m - (double)r.m) * c2);
    r.s = __dadd_rn(__dmul_rn(a.s, fa), __dmul_rn(b.s, fb));
    return r;
  }
};

struct DistillSmem {
  ReduceScratch cluster;
  ReduceScratch block;
  Exp2Table table;
};

// Listing of a row in shared memory, behind the slice's buffer.
struct Listing {
  double* q;   // teacher's mass
  float* x;    // student's logit, where this CTA owns the entry
  int* token;  // -1: no entry
  int* own;    // 1: the token is this CTA's and the entry stands for it; -1: another does
};

// Writes one value over the row's slice of the gradient.
template <typename T, bool kClustered>
__device__ void fill_slice(const RowSlice<T, kClustered>& row, T* grad, float value) {
  for (int i = threadIdx.x; i < row.n; i += blockDim.x) grad[row.start + i] = narrow<T>(value);
}

// Few rows, in the shared memory of a CTA or a cluster: bound by latency (48 x
// 1009 f16: 10 us).
template <typename T, bool kClustered, bool kWide>
__global__ void __launch_bounds__(kMaxThreads, 2) distill_rows_kernel(
    const T* logits, int64_t row_stride, int vocab, int chunk, int slice_bytes, DistillArgs a) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  __shared__ DistillSmem sm;
  using Bits = typename BitsOf<sizeof(T)>::type;
  constexpr int kE = Vec<T>::kN;
  const int cluster = kClustered ? (int)cg::this_cluster().num_blocks() : 1;
  const int64_t r = blockIdx.x / cluster;
  RowSlice<T, kClustered> row;
  const T* g = logits + r * row_stride;
  row.init(reinterpret_cast<T*>(smem_raw), g, vocab, chunk);
  row.load(g);
  Listing ls;
  ls.q = reinterpret_cast<double*>(smem_raw + slice_bytes);
  ls.x = reinterpret_cast<float*>(ls.q + a.k);
  ls.token = reinterpret_cast<int*>(ls.x + a.k);
  ls.own = ls.token + a.k;

  sm.table.fill();
  // the teacher's masses, while the row is on its way
  const bool tail = a.log_norm != nullptr;
  const double inv_tau = a.inv_temperature;
  Reducer<false> block(&sm.block);
  float amax = -CUDART_INF_F;
  bool any = false, bad = false;
  for (int k = threadIdx.x; k < a.k; k += blockDim.x) {
    const float v = load_value(a.values, a.teacher_dtype, r * a.k + k);
    int token = a.tokens[r * a.k + k];
    if (token < 0 || v == -CUDART_INF_F) token = -1;
    bad |= token >= 0 && bad_entry(token, v, vocab);
    any |= token >= 0;
    if (token >= 0) amax = fmaxf(amax, v);
    ls.token[k] = token;
    ls.x[k] = v;
  }
  const bool row_any = __syncthreads_or(any);
  const bool row_bad = __syncthreads_or(bad) || (row_any && bad_norm(a.log_norm, r));
  cp_async_wait_all();
  if (kClustered) cg::this_cluster().sync();
  else __syncthreads();
  T* grad = a.grad ? static_cast<T*>(a.grad) + r * a.grad_row_stride : nullptr;
  const bool writer = threadIdx.x == 0 && row.rank == 0;
  if (row_bad || !row_any) {
    const float v = row_bad ? CUDART_NAN_F : 0.0f;
    const bool zero_weight =
        a.row_weights != nullptr && a.row_weights[r * a.row_weight_stride] == 0.0f;
    if (writer && a.loss) a.loss[r] = v;
    if (writer && a.stats)
      write_stats(a.stats, r, RowFactors{}, 0.0, 0.0f, 0.0f, row_bad ? kStatBad : kStatEmpty);
    if (grad) fill_slice(row, grad, zero_weight ? 0.0f : v);
    return;
  }
  // masses: exp(a / tau - norm), or relative to the largest until their sum is known
  if (!tail) amax = block.max(amax);
  const double from = tail ? 0.0 : (double)amax, norm = tail ? (double)a.log_norm[r] : 0.0;
  double q_sum = 0.0, dot = 0.0;  // sum q; over the entries in this slice sum q log q
  float listed_max = -CUDART_INF_F;
  for (int k = threadIdx.x; k < a.k; k += blockDim.x) {
    const int token = ls.token[k];
    double q = 0.0;
    int own = 0;
    if (token >= 0) {
      const double log_q = ((double)ls.x[k] - from) * inv_tau - norm, t = log_q * kLog2e;
      q = t <= 0.0 ? sm.table(t) : exp2(t);
      q_sum += q;
      const int at = token - row.start;
      if (at >= 0 && at < row.n) {
        const float x = widen(row.s[row.ph + at]);
        ls.x[k] = x;
        listed_max = fmaxf(listed_max, x);
        if (q != 0.0) dot += q * log_q;
        own = 1;
      }
    }
    ls.q[k] = q;
    ls.own[k] = own;
  }
  q_sum = block.sum(q_sum);  // of all entries, in every CTA
  // One entry stands for a token that is listed more than once: each writes
  // its number in the token's place, the one that is found there stays.  Then
  // the place gets -inf (unlisted class) or its logit back.
  __syncthreads();
  for (int k = threadIdx.x; k < a.k; k += blockDim.x)
    if (ls.own[k])
      reinterpret_cast<Bits*>(row.s)[row.ph + ls.token[k] - row.start] = (Bits)k;
  __syncthreads();
  bool twice = false;
  for (int k = threadIdx.x; k < a.k; k += blockDim.x)
    if (ls.own[k] && reinterpret_cast<Bits*>(row.s)[row.ph + ls.token[k] - row.start] != (Bits)k) {
      ls.own[k] = -1;
      twice = true;
    }
  const bool row_twice = __syncthreads_or(twice);
  if (row_twice)
    // the first of a token's entries stands for it, so that sums over the
    // entries do not change from run to run
    for (int k = threadIdx.x; k < a.k; k += blockDim.x) {
      if (ls.own[k] == 0) continue;
      int first = 0;
      while (ls.token[first] != ls.token[k]) ++first;
      ls.own[k] = first == k ? 1 : -1;
    }
  for (int k = threadIdx.x; k < a.k; k += blockDim.x)
    if (ls.own[k] > 0)
      row.s[row.ph + ls.token[k] - row.start] = narrow<T>(tail ? -CUDART_INF_F : ls.x[k]);
  __syncthreads();

  Reducer<kClustered> red(&sm.cluster);
  float bmax = -CUDART_INF_F;
  row.for_each([&](int, const Vec<T>& x) {
#pragma unroll
    for (int e = 0; e < kE; ++e) bmax = fmaxf(bmax, x.at(e));
  });
  bmax = red.max(bmax);           // of the body: all tokens, or the unlisted ones
  listed_max = red.max(listed_max);
  const float xmax = fmaxf(bmax, listed_max);
  const float base = bmax == -CUDART_INF_F ? 0.0f : bmax;
  const float c = a.c;
  std::conditional_t<kWide, double, float> s = 0;
  row.for_each([&](int, const Vec<T>& x) {
#pragma unroll
    for (int e = 0; e < kE; ++e) {
      if constexpr (kWide) s += wide_weight(x.at(e), base, kLog2e * inv_tau, sm.table);
      else s += exp2_fast((x.at(e) - base) * c);
    }
  });
  double listed = 0.0;  // sum over listed tokens exp((x - xmax) / tau)
  for (int k = threadIdx.x; k < a.k; k += blockDim.x) {
    if (ls.own[k] == 0) continue;
    const double z = ((double)ls.x[k] - (double)xmax) * inv_tau, q = ls.q[k];
    // a mass that underflows counts nothing, also on a masked token
    if (q != 0.0) dot -= q * z;
    if (tail && ls.own[k] > 0) listed += exp(z);
  }
  const double body = red.sum((double)s);
  const double2 sums = red.sum(make_double2(listed, dot));
  listed = sums.x;
  dot = sums.y;
  const double sum_q = q_sum, q_scale = tail ? 1.0 : 1.0 / sum_q;
  q_sum *= q_scale;
  if (!tail) dot = dot * q_scale - log(sum_q);
  const float weight = a.row_weights ? a.row_weights[r * a.row_weight_stride] : 1.0f;
  const RowFactors f =
      row_factors(tail, bmax, body, xmax, listed, q_sum, inv_tau, a.temperature, weight);
  if (writer && a.loss) a.loss[r] = row_loss(f, dot, bmax, xmax, body, inv_tau, a.temperature);
  if (a.stats) {
    const bool twice_at_all = red.max((int)row_twice);  // in any CTA's slice
    if (writer)
      write_stats(a.stats, r, f, q_scale, xmax, tail ? 0.0f : amax, twice_at_all ? kStatTwice : 0);
  }
  if (grad == nullptr) return;
  if (weight == 0.0f) {
    fill_slice(row, grad, 0.0f);
    return;
  }
  const float G = (float)(f.Q * f.F);
  T* gs = grad + row.start - row.ph;  // element e0 of the slice's vectors goes to gs[e0]
  const bool same_phase = (reinterpret_cast<uintptr_t>(gs) & 15) == 0;
  row.for_each([&](int i0, const Vec<T>& x) {
    Vec<T> y;
#pragma unroll
    for (int i = 0; i < kE / 2; ++i) {
      const float2 p = x.pair(i);
      y.set_pair(i, make_float2(exp2_fast((p.x - base) * c) * G, exp2_fast((p.y - base) * c) * G));
    }
    const int e0 = i0 - row.start + row.ph;
    if (same_phase && e0 >= row.ph && e0 + kE <= row.ph + row.n) {
      *reinterpret_cast<Vec<T>*>(gs + e0) = y;
    } else {
#pragma unroll
      for (int e = 0; e < kE; ++e)
        if (e0 + e >= row.ph && e0 + e < row.ph + row.n) gs[e0 + e] = reinterpret_cast<const T*>(y.w)[e];
    }
  });
  __syncthreads();
  for (int k = threadIdx.x; k < a.k; k += blockDim.x) {
    if (ls.own[k] <= 0) continue;
    double q = ls.q[k];
    if (row_twice) {
      q = 0.0;
      for (int j = 0; j < a.k; ++j)
        if (ls.token[j] == ls.token[k]) q += ls.q[j];
    }
    const double e = exp(((double)ls.x[k] - (double)xmax) * inv_tau);
    grad[ls.token[k]] = narrow<T>((float)listed_gradient(f.Q, f.each, e, q * q_scale));
  }
}


// A row's sum and its largest listed logit.
template <typename Sum>
struct RowSum {
  Sum soft;
  float lmax;
};

// Sums over a row's entries: masses, q (log q - (x - xmax) / tau), and
// exp((x - xmax) / tau) of the listed tokens where they are left out of the
// row's sum; whether a token is listed twice rides along.
struct EntrySums {
  double q, dot, listed;
  int twice;
};

}  // namespace

template <>
__device__ __forceinline__ WideSum shfl_xor(WideSum v, int o) {
  WideSum r;
  r.m = __shfl_xor_sync(0xffffffffu, v.m, o);
  r.s = __shfl_xor_sync(0xffffffffu, v.s, o);
  return r;
}
template <>
__device__ __forceinline__ RowSum<SoftSum> shfl_xor(RowSum<SoftSum> v, int o) {
  v.soft = shfl_xor(v.soft, o);
  v.lmax = __shfl_xor_sync(0xffffffffu, v.lmax, o);
  return v;
}
template <>
__device__ __forceinline__ RowSum<WideSum> shfl_xor(RowSum<WideSum> v, int o) {
  v.soft = shfl_xor(v.soft, o);
  v.lmax = __shfl_xor_sync(0xffffffffu, v.lmax, o);
  return v;
}
template <>
__device__ __forceinline__ EntrySums shfl_xor(EntrySums v, int o) {
  EntrySums r;
  r.q = __shfl_xor_sync(0xffffffffu, v.q, o);
  r.dot = __shfl_xor_sync(0xffffffffu, v.dot, o);
  r.listed = __shfl_xor_sync(0xffffffffu, v.listed, o);
  r.twice = __shfl_xor_sync(0xffffffffu, v.twice, o);
  return r;
}

namespace {

// Of the entries of one token the first stands for it.
__device__ __forceinline__ void own_first(const Listing& ls, int k_all, int tid,
                                          int threads) {
  for (int k = tid; k < k_all; k += threads) {
    if (ls.token[k] < 0) continue;
    int first = 0;
    while (ls.token[first] != ls.token[k]) ++first;
    ls.own[k] = first == k;
  }
}

constexpr int kTeamThreads = 128;  // of a CTA whose rows are its teams'

template <int kTeam>
struct StreamSmem {
  ReduceScratch red;
  Exp2Table table;
  struct {
    RowFactors f;
    EntrySums sums;
  } row[kTeam ? kTeamThreads / (kTeam ? kTeam : 1) : 1];
};

// Many rows: a CTA, or a team of lanes, streams a row for its sum, then again for
// the gradient.  The
// listed tokens are marked in a bit map in the phase of the row's vectors, a
// vector's marks in one byte or half a byte, so that the first pass leaves them
// out where the unlisted ones form a class; the entry that sets a mark stands
// for its token.  The entries' own work comes between the two passes.
//
// 4096 x 131072 bf16, loss and gradient: 503 us, 4.3 TB/s, DRAM 73 % and XU 54 %
// busy (1072 with the row in a cluster's shared memory); 1024 x 32768 f32, loss: 33
// us, 4.1 TB/s.
template <typename T, int kTeam, bool kWide>
__global__ void __launch_bounds__(kTeam ? kTeamThreads : kStreamThreads, kTeam ? 8 : 2)
    distill_stream_kernel(const T* logits, int64_t row_stride, int64_t n_rows, int vocab,
                          int row_bytes, DistillArgs a) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  __shared__ StreamSmem<kTeam> sm;
  constexpr int kE = Vec<T>::kN, kU = 4;
  Team<kTeam> team(&sm.red);
  const int tid = team.rank(), threads = team.size();
  const int own_row = kTeam ? (int)threadIdx.x / (kTeam ? kTeam : 1) : 0;
  auto& mine = sm.row[own_row];
  const int64_t r = kTeam ? (int64_t)blockIdx.x * (kTeamThreads / (kTeam ? kTeam : 1)) + own_row
                          : (int64_t)blockIdx.x;
  sm.table.fill();
  if (kTeam) {
    __syncthreads();
    if (r >= n_rows) return;
  }
  const T* g = logits + r * row_stride;
  const RowStream<T> row(g, vocab);
  Listing ls;  // q holds masses up to the factor q_scale
  ls.q = reinterpret_cast<double*>(smem_raw + own_row * row_bytes);
  ls.x = reinterpret_cast<float*>(ls.q + a.k);
  ls.token = reinterpret_cast<int*>(ls.x + a.k);
  ls.own = ls.token + a.k;
  uint32_t* marks = reinterpret_cast<uint32_t*>(ls.own + a.k);

  const bool tail = a.log_norm != nullptr;
  T* grad = a.grad ? static_cast<T*>(a.grad) + r * a.grad_row_stride : nullptr;
  const float weight = a.row_weights ? a.row_weights[r * a.row_weight_stride] : 1.0f;
  const bool marked = tail || grad != nullptr || a.stats != nullptr;
  if (marked)
    for (int w = tid; w < (row.end + 31) / 32; w += threads) marks[w] = 0;
  unsigned flags = 0;  // 1: an entry, 2: a bad one
  float amax = -CUDART_INF_F;
  for (int k = tid; k < a.k; k += threads) {
    const float v = load_value(a.values, a.teacher_dtype, r * a.k + k);
    int token = a.tokens[r * a.k + k];
    if (token < 0 || v == -CUDART_INF_F) token = -1;
    if (token >= 0) {
      flags |= bad_entry(token, v, vocab) ? 2u : 1u;
      amax = fmaxf(amax, v);
    }
    ls.token[k] = token;
    ls.x[k] = v;
  }
  const unsigned long long head =
      team.all(((unsigned long long)order_key(amax) << 32) | flags,
              [](unsigned long long p, unsigned long long q) {
                return (p > q ? p : q) | (p & 3) | (q & 3);
              });
  const bool row_any = head & 1, row_bad = head & 2 || (row_any && bad_norm(a.log_norm, r));
  if (row_bad || !row_any) {
    const float v = row_bad ? CUDART_NAN_F : 0.0f;
    if (tid == 0 && a.loss) a.loss[r] = v;
    if (tid == 0 && a.stats)
      write_stats(a.stats, r, RowFactors{}, 0.0, 0.0f, 0.0f, row_bad ? kStatBad : kStatEmpty);
    if (grad)
      for (int i = tid; i < vocab; i += threads) grad[i] = narrow<T>(weight == 0.0f ? 0.0f : v);
    return;
  }
  amax = key_value((uint32_t)(head >> 32));
  EntrySums sums{0.0, 0.0, 0.0, 0};
  bool twice_here = false;
  if (marked) {
    for (int k = tid; k < a.k; k += threads) {
      const int token = ls.token[k];
      if (token < 0) continue;
      const int bit = token + row.ph;
      const int own = !(atomicOr(&marks[bit >> 5], 1u << (bit & 31)) >> (bit & 31) & 1u);
      twice_here |= !own;
      ls.own[k] = own;
    }
    sums.twice = twice_here;
    // The marks are read in the first pass.  Of a token's entries any may stand
    // for it where only its gradient is written; in a sum it is the first, so
    // that the sum does not change from run to run.
    if (tail && team.any(twice_here)) own_first(ls, a.k, tid, threads);
  }

  const double inv_tau = a.inv_temperature;
  const float c = a.c;
  using Sum = std::conditional_t<kWide, WideSum, SoftSum>;
  Sum soft;
  row.template walk<kU, kTeam>([&](auto& x, int v, int step, bool, int) {
    if (tail) {
      constexpr int n = sizeof(x) / sizeof(x[0]);
#pragma unroll
      for (int u = 0; u < n; ++u) {
        const int e0 = (v + u * step) * kE;
        const uint32_t m = marks[e0 >> 5] >> (e0 & 31) & ((1u << kE) - 1u);
        if (m)
#pragma unroll
          for (int e = 0; e < kE; ++e)
            if (m >> e & 1u) x[u].clear(e);
      }
    }
    if constexpr (kWide) soft.add(x, kLog2e * inv_tau, sm.table);
    else soft.add(x, c);
  });

  RowSum<Sum> sum{soft, -CUDART_INF_F};
  for (int k = tid; k < a.k; k += threads) {
    if (ls.token[k] < 0) continue;
    const float x = widen(g[ls.token[k]]);
    ls.q[k] = (double)x;
    sum.lmax = fmaxf(sum.lmax, x);
  }
  sum = team.all(sum, [c, inv_tau](RowSum<Sum> p, RowSum<Sum> q) {
    RowSum<Sum> t;
    if constexpr (kWide) t.soft = Sum::join(p.soft, q.soft, kLog2e * inv_tau);
    else t.soft = Sum::join(p.soft, q.soft, c);
    t.lmax = fmaxf(p.lmax, q.lmax);
    return t;
  });
  const float bmax = sum.soft.m, xmax = fmaxf(bmax, sum.lmax);
  const double body = (double)sum.soft.s;
  // masses: exp(a / tau - norm), or relative to the largest until their sum is known
  const double from = tail ? 0.0 : (double)amax, norm = tail ? (double)a.log_norm[r] : 0.0;
  for (int k = tid; k < a.k; k += threads) {
    if (ls.token[k] < 0) continue;
    const double log_q = ((double)ls.x[k] - from) * inv_tau - norm, t = log_q * kLog2e;
    const double q = t <= 0.0 ? sm.table(t) : exp2(t);
    const double z = (ls.q[k] - (double)xmax) * inv_tau;
    sums.q += q;
    // a mass that underflows counts nothing, also on a masked token
    if (q != 0.0) sums.dot += q * (log_q - z);
    if (tail && ls.own[k]) sums.listed += exp(z);
    ls.x[k] = (float)ls.q[k];
    ls.q[k] = q;
  }
  sums = team.all(sums, [](EntrySums p, EntrySums q) {
    return EntrySums{p.q + q.q, p.dot + q.dot, p.listed + q.listed, p.twice | q.twice};
  });
  const double q_scale = tail ? 1.0 : 1.0 / sums.q;
  const RowFactors f = row_factors(tail, bmax, body, xmax, sums.listed, sums.q * q_scale, inv_tau,
                                   a.temperature, weight);
  if (tid == 0) {
    // what the list and the loss need waits in shared memory
    mine.f = f;
    mine.sums = sums;
    if (a.stats)
      write_stats(a.stats, r, f, q_scale, xmax, tail ? 0.0f : amax, sums.twice ? kStatTwice : 0);
  }
  auto write_loss = [&] {
    const double dot = tail ? sums.dot : sums.dot * q_scale - log(sums.q);
    a.loss[r] = row_loss(f, dot, bmax, xmax, body, inv_tau, a.temperature);
  };
  if (grad == nullptr || weight == 0.0f) {
    if (tid == 0 && a.loss) write_loss();
    if (grad)
      for (int i = tid; i < vocab; i += threads) grad[i] = narrow<T>(0.0f);
    return;
  }
  T* gv = grad - row.ph;  // vector v of the row goes to gv[v * kE ..]
  const bool same_phase = (reinterpret_cast<uintptr_t>(gv) & 15) == 0;
  const float2 minus = make_float2(-f.base, -f.base), scale = make_float2(c, c),
               G = make_float2((float)(f.Q * f.F), (float)(f.Q * f.F));
  row.template walk<kU, kTeam>([&](auto& x, int v, int step, bool whole, int) {
    constexpr int n = sizeof(x) / sizeof(x[0]);
#pragma unroll
    for (int u = 0; u < n; ++u) {
      const int e0 = (v + u * step) * kE;
      Vec<T> y;
#pragma unroll
      for (int i = 0; i < kE / 2; ++i) {
        const float2 t = __fmul2_rn(__fadd2_rn(x[u].pair(i), minus), scale);
        y.set_pair(i, __fmul2_rn(make_float2(exp2_fast(t.x), exp2_fast(t.y)), G));
      }
      if (same_phase && whole) {
        __stcs(reinterpret_cast<uint4*>(gv + e0), *reinterpret_cast<const uint4*>(&y));
      } else {
#pragma unroll
        for (int e = 0; e < kE; ++e)
          if (e0 + e >= row.ph && e0 + e < row.end) gv[e0 + e] = reinterpret_cast<const T*>(y.w)[e];
      }
    }
  });
  team.sync();
  const bool twice = mine.sums.twice;
  const double sum_q = mine.sums.q, scale_q = tail ? 1.0 : 1.0 / sum_q;
  for (int k = tid; k < a.k; k += threads) {
    if (ls.token[k] < 0 || !ls.own[k]) continue;
    double q = ls.q[k];
    if (twice) {
      q = 0.0;
      for (int j = 0; j < a.k; ++j)
        if (ls.token[j] == ls.token[k]) q += ls.q[j];
    }
    const double e = exp(((double)ls.x[k] - (double)xmax) * inv_tau);
    grad[ls.token[k]] = narrow<T>((float)listed_gradient(mine.f.Q, mine.f.each, e, q * scale_q));
  }
  // the last warp has fewest entries to see to
  if (tid == threads - 1 && a.loss) {
    const double dot = tail ? mine.sums.dot : mine.sums.dot * scale_q - log(sum_q);
    a.loss[r] = row_loss(mine.f, dot, bmax, xmax, body, inv_tau, a.temperature);
  }
}

// The gradient from a forward pass's statistics: a row is read once, in parts of
// a CTA each.  The same formulas as above, to the bit.  Bound by memory: 2000 x
// 50001 bf16: 74 us, 5.4 TB/s; reading the rows twice, without statistics, 100.
template <typename T>
__global__ void __launch_bounds__(256, 4) distill_backward_kernel(const T* logits,
                                                                  int64_t row_stride, int vocab,
                                                                  int parts, int part_vectors,
                                                                  DistillArgs a) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  __shared__ Exp2Table table;
  constexpr int kE = Vec<T>::kN, kU = 4;
  const int64_t r = blockIdx.x / (unsigned)parts;
  const int part = (int)(blockIdx.x % (unsigned)parts);
  const int tid = threadIdx.x, threads = blockDim.x;
  const T* g = logits + r * row_stride;
  const RowStream<T> row(g, vocab);
  T* gv = static_cast<T*>(a.grad) + r * a.grad_row_stride - row.ph;
  // this CTA's whole vectors, and its elements with the row's ends
  const int v0 = ::min(row.hi, row.lo + part * part_vectors);
  const int v1 = part == parts - 1 ? ::max(v0, row.hi) : ::min(row.hi, v0 + part_vectors);
  const int e_first = part == 0 ? row.ph : v0 * kE;
  const int e_last = part == parts - 1 ? row.end : v1 * kE;  // one behind
  Listing ls;
  ls.q = reinterpret_cast<double*>(smem_raw);
  ls.x = reinterpret_cast<float*>(ls.q + a.k);
  ls.token = reinterpret_cast<int*>(ls.x + a.k);
  table.fill();

  const double* st = a.stats + r * HKB_DISTILL_STATS;
  const double F = st[0], each = st[1], q_scale = st[2];
  const float base = __int_as_float(__double2hiint(st[3])), xmax = __int_as_float(__double2loint(st[3]));
  const float amax = __int_as_float(__double2hiint(st[4]));
  const int flags = __double2loint(st[4]);
  const float weight = a.row_weights ? a.row_weights[r * a.row_weight_stride] : 1.0f;
  if ((flags & (kStatBad | kStatEmpty)) || weight == 0.0f) {
    const T v = narrow<T>((flags & kStatBad) && weight != 0.0f ? CUDART_NAN_F : 0.0f);
    for (int e = e_first + tid; e < e_last; e += threads) gv[e] = v;
    return;
  }
  const bool tail = a.log_norm != nullptr;
  const double inv_tau = a.inv_temperature;
  const double from = tail ? 0.0 : (double)amax, norm = tail ? (double)a.log_norm[r] : 0.0;
  __syncthreads();  // the table
  for (int k = tid; k < a.k; k += threads) {
    const float v = load_value(a.values, a.teacher_dtype, r * a.k + k);
    int token = a.tokens[r * a.k + k];
    if (token < 0 || token >= vocab || v == -CUDART_INF_F) token = -1;
    const int e = token + row.ph;
    const bool here = token >= 0 && e >= e_first && e < e_last;
    ls.token[k] = here ? token : -1;
    if (here) {
      const double t = (((double)v - from) * inv_tau - norm) * kLog2e;
      ls.q[k] = t <= 0.0 ? table(t) : exp2(t);
      ls.x[k] = widen(g[token]);
    }
  }
  __syncthreads();  // read before the gradient may take the logits' place
  const double Q = (double)weight * a.temperature;
  const float c = a.c, Gf = (float)(Q * F);
  const float2 minus = make_float2(-base, -base), scale = make_float2(c, c), G = make_float2(Gf, Gf);
  const bool same_phase = (reinterpret_cast<uintptr_t>(gv) & 15) == 0;
  auto put = [&](const Vec<T>& x, int v, bool whole) {
    Vec<T> y;
#pragma unroll
    for (int i = 0; i < kE / 2; ++i) {
      const float2 t = __fmul2_rn(__fadd2_rn(x.pair(i), minus), scale);
      y.set_pair(i, __fmul2_rn(make_float2(exp2_fast(t.x), exp2_fast(t.y)), G));
    }
    const int e0 = v * kE;
    if (same_phase && whole) {
      __stcs(reinterpret_cast<uint4*>(gv + e0), *reinterpret_cast<const uint4*>(&y));
    } else {
#pragma unroll
      for (int e = 0; e < kE; ++e)
        if (e0 + e >= row.ph && e0 + e < row.end) gv[e0 + e] = reinterpret_cast<const T*>(y.w)[e];
    }
  };
  const Vec<T>* vec = reinterpret_cast<const Vec<T>*>(row.g);
  int v = v0 + tid;
  for (; v + (kU - 1) * threads < v1; v += kU * threads) {
    Vec<T> x[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) x[u] = vec[v + u * threads];
#pragma unroll
    for (int u = 0; u < kU; ++u) put(x[u], v + u * threads, true);
  }
  for (; v < v1; v += threads) put(vec[v], v, true);
  if (tid == 0 && part == 0 && row.lo > 0) put(row.partial(0), 0, false);
  if (tid == threads - 1 && part == parts - 1 && row.hi >= row.lo && row.hi * kE < row.end)
    put(row.partial(row.hi), row.hi, false);
  __syncthreads();
  for (int k = tid; k < a.k; k += threads) {
    if (ls.token[k] < 0) continue;
    double q = ls.q[k];
    if (flags & kStatTwice) {
      q = 0.0;
      for (int j = 0; j < a.k; ++j)
        if (ls.token[j] == ls.token[k]) q += ls.q[j];
    }
    const double e = exp(((double)ls.x[k] - (double)xmax) * inv_tau);
    gv[row.ph + ls.token[k]] = narrow<T>((float)listed_gradient(Q, each, e, q * q_scale));
  }
}

// f(value, token) over the entries of row r, in order; rows of 32-bit values in
// multiples of four entries are read 16 bytes at a time.
template <typename F>
__device__ __forceinline__ void for_each_entry(const DistillArgs& a, int64_t r, F f) {
  const int64_t at = r * a.k;
  if (a.teacher_dtype == HKB_F32 && (a.k & 3) == 0 &&
      ((reinterpret_cast<uintptr_t>(a.values) | reinterpret_cast<uintptr_t>(a.tokens)) & 15) == 0) {
    const float4* v = reinterpret_cast<const float4*>(static_cast<const float*>(a.values) + at);
    const int4* t = reinterpret_cast<const int4*>(a.tokens + at);
    for (int k = 0; k < a.k / 4; ++k) {
      const float4 x = v[k];
      const int4 y = t[k];
      f(x.x, y.x);
      f(x.y, y.y);
      f(x.z, y.z);
      f(x.w, y.w);
    }
  } else {
    for (int k = 0; k < a.k; ++k)
      f(load_value(a.values, a.teacher_dtype, at + k), a.tokens[at + k]);
  }
}

// Short rows, one thread each.  The masses of a row's tokens are added up in
// shared memory, so a token listed twice needs no special case; the weights stay
// in registers between the sum and the gradient, which replaces the row's copy and
// leaves as the row came.  Up to kWideTemperature a token's mass and the listed
// gradient are 32-bit (a few roundings of 2^-24 of temperature * mass; the loss
// has the masses in 64 bits): half the shared memory and registers.  Bound by
// instructions (73 % of issue, FP64 16 %): 524,288 x 21 f32, 8 entries: 49 us (20
// us of memory traffic); with 64-bit exponentials for the student too it was 120.
template <typename T, int kPad, bool kWide>
__global__ void __launch_bounds__(kShortRows, kWide ? 3 : kPad <= 24 ? 8 : 5) distill_short_kernel(const T* logits,
                                                                   int64_t row_stride,
                                                                   int64_t n_rows, int vocab,
                                                                   DistillArgs a) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  __shared__ Exp2Table table;
  const int tid = threadIdx.x;
  using S = std::conditional_t<kWide, double, float>;
  S* qs = reinterpret_cast<S*>(smem_raw + ShortRows<T>::bytes(vocab)) + tid;
  const int64_t r0 = (int64_t)blockIdx.x * kShortRows, r = r0 + tid;
  const int rows = (int)::min((int64_t)kShortRows, n_rows - r0);
  ShortRows<T> sr;
  sr.load(reinterpret_cast<T*>(smem_raw), logits + r0 * row_stride, row_stride, rows, vocab);
  table.fill();
  const bool tail = a.log_norm != nullptr;
  const double inv_tau = a.inv_temperature;
  unsigned listed = 0;
  bool bad = false;
  float amax = -CUDART_INF_F;
  if (tid < rows)
    for_each_entry(a, r, [&](float v, int token) {
      if (token < 0 || v == -CUDART_INF_F) return;
      bad |= bad_entry(token, v, vocab);
      listed |= token < vocab ? 1u << token : 0u;
      amax = fmaxf(amax, v);
    });
  if (tid < rows && listed != 0) bad |= bad_norm(a.log_norm, r);
  cp_async_wait_all();
  __syncthreads();
  if (tid < rows) {
    auto value = [&](int i) { return widen(sr.at(tid, i)); };
    const float weight = a.row_weights ? a.row_weights[r * a.row_weight_stride] : 1.0f;
    if (bad || listed == 0) {
      const float v = bad ? CUDART_NAN_F : 0.0f;
      if (a.loss) a.loss[r] = v;
      if (a.grad)
        for (int i = 0; i < vocab; ++i) sr.at(tid, i) = narrow<T>(weight == 0.0f ? 0.0f : v);
    } else {
      // the body is the whole row, or its unlisted tokens
      const unsigned body = tail ? ~listed : ~0u;
      float bmax = -CUDART_INF_F, lmax = -CUDART_INF_F;
#pragma unroll
      for (int i = 0; i < kPad; ++i)
        if (i < vocab) {
          const float v = value(i);
          if (body >> i & 1u) bmax = fmaxf(bmax, v);
          else lmax = fmaxf(lmax, v);
          qs[i * kShortPitch] = 0;
        }
      const float xmax = fmaxf(bmax, lmax);
      // masses exp(a / tau - norm), or relative to the largest until their sum
      // is known, and sum q (log q - (x - xmax) / tau)
      const double norm = tail ? (double)a.log_norm[r] : 0.0, from = tail ? 0.0 : (double)amax;
      double q_sum = 0.0, dot = 0.0;
      for_each_entry(a, r, [&](float v, int token) {
        if (token < 0 || v == -CUDART_INF_F) return;
        const double log_q = ((double)v - from) * inv_tau - norm;
        const double t = log_q * kLog2e;
        const double q = t <= 0.0 ? table(t) : exp2(t);
        q_sum += q;
        // a mass that underflows counts nothing, also on a masked token
        if (q != 0.0) dot += q * (log_q - ((double)value(token) - (double)xmax) * inv_tau);
        qs[token * kShortPitch] += (S)q;
      });
      double q_scale = 1.0;
      if (!tail) {
        q_scale = 1.0 / q_sum;
        dot = dot * q_scale - log(q_sum);
        q_sum *= q_scale;
      }
      const float base = bmax == -CUDART_INF_F ? 0.0f : bmax;
      const float c = a.c;
      auto weight_of = [&](float x, float ref) -> S {
        if constexpr (kWide) return wide_weight(x, ref, kLog2e * inv_tau, table);
        else return exp2_fast((x - ref) * c);
      };
      S e[kPad], sum = 0, rest = 0;  // of the body and, relative to xmax, of the list
#pragma unroll
      for (int i = 0; i < kPad; ++i) {
        e[i] = 0;
        if (i < vocab) {
          const bool in_body = body >> i & 1u;
          e[i] = weight_of(value(i), in_body ? base : xmax);
          if (in_body) sum += e[i];
          else rest += e[i];
        }
      }
      const S lift = bmax == -CUDART_INF_F ? (S)0
                     : bmax == xmax        ? (S)1
                                           : weight_of(bmax, xmax);
      const double total = fma((double)sum, (double)lift, (double)rest);
      double rest_q = 0.0;
      if (tail && bmax != -CUDART_INF_F) rest_q = fmax(0.0, 1.0 - q_sum);
      const double mass = q_sum + rest_q;
      const double share = rest_q > 0.0 ? rest_q / (double)sum : 0.0;
      if (a.loss) {
        double l = dot + mass * log(total);
        if (rest_q > 0.0) l += rest_q * (log(share) - ((double)bmax - (double)xmax) * inv_tau);
        a.loss[r] = (float)(a.temperature * a.temperature * l);
      }
      if (a.grad) {
        const double wt = (double)weight * a.temperature;
        const double each = mass / total;
        // gradient: e G off the list, e P - q Q on it (the body's e G where
        // listed tokens are part of the body: lift is 1 then)
        const S G = (S)(wt * (each * (double)lift - share));
        const S P = (S)(wt * each), Q = (S)(wt * q_scale);
#pragma unroll
        for (int i = 0; i < kPad; ++i)
          if (i < vocab) {
            const S y = listed >> i & 1u ? e[i] * P - qs[i * kShortPitch] * Q : e[i] * G;
            sr.at(tid, i) = narrow<T>(weight == 0.0f ? 0.0f : (float)y);
          }
      }
    }
  }
  if (a.grad == nullptr) return;
  __syncthreads();
  sr.store(static_cast<T*>(a.grad) + r0 * a.grad_row_stride, a.grad_row_stride);
}

// A row of a few hundred tokens costs a warp some 1400 instructions, most of them
// the same for any V: the reductions, the masses' sums and logarithms.  Teams of 4
// or 8 lanes share them, when there are rows for two CTAs a SM.  More entries
// than four (sixteen) a lane take it back; a lane adds at most 128 weights.  Measured
// (us), loss and gradient, bf16, a CTA, 4 and 8 lanes a row: 100,000 x 40, 10
// entries: 184, 41 and 63; 40 entries: 213, 84 and 86; 100,000 x 400, 10: 209, 78 and
// 98; 40: 246, 139 and 127; 120: 369 and 305 with 8; 10,000 x 400, 10: 29, 20 and 18;
// 2400 x 400, 10: 12, 16 and 14.
template <int kTeam>
bool use_team(const VocabRows& v, int k) {
  return v.vocab <= (kTeam == 4 ? 512 : 31 * 32) && k <= (kTeam == 4 ? 16 : 128) &&
         v.rows >= 2 * 148 * (kTeamThreads / kTeam);
}
template <typename T, int kTeam, bool kWide>
cudaError_t launch_teams(cudaStream_t st, const VocabRows& v, const DistillArgs& a, int row_bytes) {
  constexpr int kTeams = kTeamThreads / kTeam;
  distill_stream_kernel<T, kTeam, kWide>
      <<<(unsigned)((v.rows + kTeams - 1) / kTeams), kTeamThreads, row_bytes * kTeams, st>>>(
          static_cast<const T*>(v.logits), v.row_stride, v.rows, v.vocab, row_bytes, a);
  return cudaGetLastError();
}

template <typename T, bool kWide>
cudaError_t launch_as(cudaStream_t st, const VocabRows& v, const DistillArgs& a) {
  if (v.vocab <= kShortVocab) {
    constexpr int kMass = kWide ? sizeof(double) : sizeof(float);
    const int smem = ShortRows<T>::bytes(v.vocab) + kMass * kShortPitch * v.vocab;
    const unsigned blocks = (unsigned)((v.rows + kShortRows - 1) / kShortRows);
    HKB_SHORT_WIDTH(v.vocab, {
      if (kWide)  // 49 KB at 32 tokens of 32 bits
        ensure_dynamic_smem((const void*)distill_short_kernel<T, kPad, kWide>,
                            ShortRows<T>::bytes(kPad) + kMass * kShortPitch * kPad);
      distill_short_kernel<T, kPad, kWide><<<blocks, kShortRows, smem, st>>>(
          static_cast<const T*>(v.logits), v.row_stride, v.rows, v.vocab, a);
    });
    return cudaGetLastError();
  }
  if (use_stream(v.rows, v.vocab, (int)sizeof(T))) {
    // bits of a row in its vectors' phase, in whole words
    const int words = (v.vocab + 16 / (int)sizeof(T) - 1 + 31) / 32;
    const int bytes = (a.k * 20 + words * 4 + 7) / 8 * 8;
    if (use_team<4>(v, a.k)) return launch_teams<T, 4, kWide>(st, v, a, bytes);
    if (use_team<8>(v, a.k)) return launch_teams<T, 8, kWide>(st, v, a, bytes);
    ensure_dynamic_smem((const void*)distill_stream_kernel<T, 0, kWide>,
                        HKB_LISTING_MAX * 20 + HKB_VOCAB_MAX / 8 + 8);
    distill_stream_kernel<T, 0, kWide>
        <<<(unsigned)v.rows, stream_threads(v.vocab, (int)sizeof(T)), bytes, st>>>(
            static_cast<const T*>(v.logits), v.row_stride, v.rows, v.vocab, 0, a);
    return cudaGetLastError();
  }
  const RowShape s = row_shape(v.rows, v.vocab, (int)sizeof(T));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(v.rows * s.cluster));
  cfg.blockDim = dim3((unsigned)s.threads);
  cfg.dynamicSmemBytes = s.smem + (size_t)a.k * 20;
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = (unsigned)s.cluster;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  auto kernel =
      s.cluster > 1 ? distill_rows_kernel<T, true, kWide> : distill_rows_kernel<T, false, kWide>;
  ensure_dynamic_smem((const void*)kernel, 131072 + 16 + HKB_LISTING_MAX * 20);
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<const T*>(v.logits), v.row_stride, v.vocab,
                            s.chunk, (int)s.smem, a);
}

template <typename T>
cudaError_t launch(cudaStream_t st, const VocabRows& v, const DistillArgs& a) {
  return a.temperature > kWideTemperature ? launch_as<T, true>(st, v, a)
                                          : launch_as<T, false>(st, v, a);
}

template <typename T>
cudaError_t launch_backward(cudaStream_t st, const VocabRows& v, const DistillArgs& a) {
  // a short row's thread has the whole row at hand: nothing to save
  if (v.vocab <= kShortVocab) return launch<T>(st, v, a);
  // parts of up to 16 vectors a thread; of as few as two while that gives no
  // four CTAs a SM
  const int nvec = v.vocab / (16 / (int)sizeof(T)) + 1;
  int threads = 256, per = 16;
  while (threads > 32 && threads * 4 > nvec) threads /= 2;
  while (per > 2 && v.rows * ((nvec + threads * per - 1) / (threads * per)) < 4 * 148) per /= 2;
  const int part = threads * per, parts = (nvec + part - 1) / part;
  const int smem = a.k * 16;
  distill_backward_kernel<T><<<(unsigned)(v.rows * parts), threads, smem, st>>>(
      static_cast<const T*>(v.logits), v.row_stride, v.vocab, parts, part, a);
  return cudaGetLastError();
}

}  // namespace
}  // namespace vocab

cudaError_t launch_distill_backward(cudaStream_t st, const VocabRows& v, const DistillArgs& a) {
  switch (v.dtype) {
    case HKB_F32: return vocab::launch_backward<float>(st, v, a);
    case HKB_F16: return vocab::launch_backward<__half>(st, v, a);
    default: return vocab::launch_backward<__nv_bfloat16>(st, v, a);
  }
}

cudaError_t launch_distill(cudaStream_t st, const VocabRows& v, const DistillArgs& a) {
  switch (v.dtype) {
    case HKB_F32: return vocab::launch<float>(st, v, a);
    case HKB_F16: return vocab::launch<__half>(st, v, a);
    default: return vocab::launch<__nv_bfloat16>(st, v, a);
  }
}

}  // namespace hkb
