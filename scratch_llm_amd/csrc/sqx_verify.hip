// Verification of drafted tokens against the target model's logits, from given random numbers (speculative sampling), and
// the sampling of the token that follows.
//
// With p_t = softmax(logits_t / temperature) and q_t the draft's probabilities, draft t is accepted while
// u_t q_t(x_t) < p_t(x_t). After the first rejection the token is drawn from max(p - q, 0) of that row, after none from p
// of the row behind the drafts: the least i whose cumulative weight exceeds r times the total, so the kept tokens are
// distributed as the target's own. Temperature 0: accept while x_t is the row's argmax, then take the argmax.
//
// What the pick is made from is double: it falls between two neighbours of a cumulative sum over a whole vocabulary, and in
// fp32 about one pick in a hundred would depend on the order of the sums. That takes a dozen double operations an element
// (below), for one row per sequence. The other rows are only compared with u: their sums are of fp32 exponentials, good to
// 2^-18 (31 additions of at most 2^-24 each, exponentials to 2^-23, arguments to 2^-23 of the 17 powers of two that count),
// which moves a few decisions in a million at the worst. With every row in double, 64 x (5 + 1) x 128256 bf16 logits took 38 us, twice their reading.
//
// Three launches (two at temperature 0): statistics of every slice of every row; the double sums of every slice of the one
// row per sequence that is drawn from; the pick. The decision is a few operations on the slices' statistics, so every
// workgroup of the second repeats it instead of waiting for one. The second does not know that row's total Z yet, only
// its estimate 1 / inv: with e the exponentials and P the elements where e inv > q, its slices sum e, (e inv - q) over P
// and e over P, and the third, which has Z, adds (1 / Z - inv) times the last. P misses only elements within 2^-18 of a tie.
//
// Those 64 rows, with fp32 draft probabilities, a call 47 us: 22 us (4.4 TB/s of logits), 17 us (49 MB, the verdict's chain of loads and the
// double exponentials) and 8 us (a chain of loads); 1 x (4 + 1) x 32000 fp32 logits: 3, 6 and 7 us. The last two in one
// launch, a workgroup a sequence walking its whole row, took 14 us there but 48 for the 64 rows.
#include <type_traits>

#include "sqx_common.h"

namespace sqx {

constexpr int kSlice = 8192;                // elements of a workgroup's slice
constexpr int kPer = 8;                     // consecutive elements of a thread, a pass
constexpr int kPass = 256 * kPer;           // elements of a pass
constexpr int kPasses = kSlice / kPass;
constexpr int kMaxDrafts = 63;              // a lane each, and one for the row behind them

struct VerifyArgs {
  const void* logits;  // [B, T + 1, V]
  const int* draft;    // [B, T]
  const int* counts;   // NULL: T drafts in every row
  const void* probs;   // [B, T, V], or NULL: each draft was certain
  const float *u, *r;
  int T, V, S;
  double k;   // 64 log2(e) / temperature
  float k32;  // log2(e) / temperature
  double* sums;  // [B, T + 1, S]
  double* rest;  // [3, B, S]: of the row drawn from, the sums above
  double* verdict;  // [B, 3]: accepted, then of the row behind them the maximum and 1 / sum as estimated
  float* maxs;   // [B, T + 1, S]
  int* args;     // [B, T + 1, S], temperature 0
  int *n_acc, *tokens;
};

// 2^(y / 64) for y <= 0: y = n + f with n the nearest integer and |f| <= 1/2; 2^(n / 64) from a table of 64 powers (64 lanes
// reading 8-byte entries at random meet few bank conflicts) and an exponent, e^(f ln 2 / 64) from its Taylor polynomial with
// the fourth power replaced by its Chebyshev economization over |x| <= h = ln 2 / 128: x^4 ~ h^2 x^2 - h^4 / 8, which
// leaves an error of h^4 / 192 = 5e-12. A probability of 5e-12 moved anywhere in a vocabulary of 128256 changes a pick with a chance of about 1e-6 at the
// worst; the order of the double sums has a millionth of that.
constexpr double kLn2_64 = 0.693147180559945309417 / 64.0;
constexpr double kH2 = (kLn2_64 / 2) * (kLn2_64 / 2);
__device__ inline double exp2_64th(double y, const double* pow64) {
  y = fmax(y, -64000.0);  // 2^-1000: nothing next to a sum that holds a 1. Drops a NaN: callers look for those in fp32
  const double t = y + 0x1.8p52;  // the nearest integer in the low bits of the mantissa
  const int n = __double2loint(t);
  const double f = y - (t - 0x1.8p52);
  double p = fma(f, kLn2_64 * kLn2_64 * kLn2_64 / 6.0, kLn2_64 * kLn2_64 * (0.5 + kH2 / 24.0));
  p = fma(p, f, kLn2_64);
  p = fma(p, f, 1.0 - kH2 * kH2 / 192.0);
  const double w = pow64[n & 63];  // in [1, 2): the exponent n >> 6 is added to its bits
  return p * __hiloint2double(__double2hiint(w) + ((n & ~63) << 14), __double2loint(w));
}
static __device__ const double kPow64[64] = {  // 2^(i / 64)
    1.0, 1.0108892860517005, 1.0218971486541166, 1.0330248790212284,
    1.0442737824274138, 1.0556451783605572, 1.0671404006768237, 1.0787607977571199,
    1.0905077326652577, 1.102382583307841, 1.1143867425958924, 1.1265216186082418,
    1.1387886347566916, 1.1511892299529827, 1.1637248587775775, 1.1763969916502812,
    1.189207115002721, 1.202156731452703, 1.215247359980469, 1.22848053610687,
    1.241857812073484, 1.255380757024691, 1.2690509571917332, 1.2828700160787783,
    1.2968395546510096, 1.3109612115247644, 1.3252366431597413, 1.339667524053303,
    1.3542555469368927, 1.3690024229745905, 1.383909881963832, 1.3989796725383112,
    1.4142135623730951, 1.42961333839197, 1.4451808069770467, 1.460917794180647,
    1.4768261459394993, 1.4929077282912648, 1.5091644275934228, 1.5255981507445384,
    1.5422108254079407, 1.559004400237837, 1.5759808451078865, 1.593142151342267,
    1.6104903319492543, 1.6280274218573478, 1.645755478153965, 1.6636765803267364,
    1.681792830507429, 1.7001063537185235, 1.718619298122478, 1.7373338352737062,
    1.7562521603732995, 1.7753764925265212, 1.7947090750031072, 1.8142521755003989,
    1.8340080864093424, 1.8539791250833855, 1.8741676341103, 1.8945759815869656,
    1.9152065613971474, 1.9360617934922943, 1.9571441241754002, 1.978456026387951,
};
__device__ inline void fill_pow64(double* pow64) {
  if (threadIdx.x < 64) pow64[threadIdx.x] = kPow64[threadIdx.x];
}

// Elements base .. base + 7 of a row of V as fp32; past the end `fill`. Without VEC one by one: 64 rows of 5 drafts over 50257
// tokens take 49 us a call, over 50264 32.
template <int DT, bool VEC>
__device__ inline void load_row8(const void* p, int64_t row0, int base, int V, float fill, float (&v)[kPer]) {
  if constexpr (VEC) {
    const int64_t at = row0 + min(base, V - kPer);
    if constexpr (DT == SQX_DTYPE_F32) {
      const f32x4_t* q = reinterpret_cast<const f32x4_t*>(static_cast<const float*>(p) + at);
      const f32x4_t a = q[0], b = q[1];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] = a[e];
        v[4 + e] = b[e];
      }
    } else {
      const u32x4_t a = *reinterpret_cast<const u32x4_t*>(static_cast<const uint16_t*>(p) + at);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t w = a[e];
        v[2 * e] = DT == SQX_DTYPE_BF16 ? bf16_lo(w) : f16_bits_to_f32(static_cast<uint16_t>(w));
        v[2 * e + 1] = DT == SQX_DTYPE_BF16 ? bf16_hi(w) : f16_bits_to_f32(static_cast<uint16_t>(w >> 16));
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < kPer; ++e) v[e] = load_as_f32(p, DT, row0 + min(base + e, V - 1));
  }
  if (base + kPer > V) {
#pragma unroll
    for (int e = 0; e < kPer; ++e) v[e] = base + e < V ? v[e] : fill;
  }
}

__device__ inline double wave_sum_f64(double v) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o, 64);
  return v;
}
// The sums over the workgroup, in every thread.
template <int N>
__device__ inline void block_sums_f64(double (&v)[N], double (&red)[N][4]) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = wave_sum_f64(v[i]);
  if ((threadIdx.x & 63) == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) red[i][threadIdx.x >> 6] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = (red[i][0] + red[i][1]) + (red[i][2] + red[i][3]);
}

// Slice s of row (b, t): its maximum and the sum of 2^(k32 (x - maximum)); temperature 0: the maximum's first index
// (NaN counts as the maximum).
template <int DT, bool VEC, bool GREEDY>
__global__ __launch_bounds__(256) void verify_stats_kernel(const VerifyArgs a) {
  __shared__ double red[1][4];
  __shared__ float redm[4];
  __shared__ int redi[4];
  const int s = blockIdx.x, row = blockIdx.y, b = row / (a.T + 1), t = row % (a.T + 1);
  const int count = a.counts != nullptr ? min(max(a.counts[b], 0), a.T) : a.T;
  if (t > count) return;
  const int64_t row0 = static_cast<int64_t>(row) * a.V;
  const int at = s * kSlice + threadIdx.x * kPer;
  float v[kPasses][kPer];
#pragma unroll
  for (int p = 0; p < kPasses; ++p) load_row8<DT, VEC>(a.logits, row0, at + p * kPass, a.V, -INFINITY, v[p]);
  const int64_t out = static_cast<int64_t>(row) * a.S + s;
  if constexpr (GREEDY) {
    float best = -INFINITY;
    int arg = 0x7fffffff;
#pragma unroll
    for (int p = 0; p < kPasses; ++p)
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const int i = at + p * kPass + e;
        const bool nan = v[p][e] != v[p][e], bn = best != best;
        if (i < a.V && !bn && (nan || v[p][e] > best || arg == 0x7fffffff)) {
          best = v[p][e];
          arg = i;
        }
      }
    auto join = [&](float ob, int oa) {
      const bool on = ob != ob, bn = best != best;
      const bool take = oa != 0x7fffffff &&
                        (arg == 0x7fffffff || (on && !bn) || (on == bn && ((on || ob == best) ? oa < arg : ob > best)));
      if (take) {
        best = ob;
        arg = oa;
      }
    };
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const float ob = __shfl_xor(best, o, 64);
      const int oa = __shfl_xor(arg, o, 64);
      join(ob, oa);
    }
    if ((threadIdx.x & 63) == 0) {
      redm[threadIdx.x >> 6] = best;
      redi[threadIdx.x >> 6] = arg;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < 4; ++w) join(redm[w], redi[w]);
      a.maxs[out] = best;
      a.args[out] = arg;
    }
  } else {
    float m = -INFINITY;  // the maximum that keeps a NaN
#pragma unroll
    for (int p = 0; p < kPasses; ++p)
#pragma unroll
      for (int e = 0; e < kPer; ++e) m = __builtin_elementwise_maximum(m, v[p][e]);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) m = __builtin_elementwise_maximum(m, __shfl_xor(m, o, 64));
    if ((threadIdx.x & 63) == 0) redm[threadIdx.x >> 6] = m;
    __syncthreads();
    m = __builtin_elementwise_maximum(__builtin_elementwise_maximum(redm[0], redm[1]),
                                      __builtin_elementwise_maximum(redm[2], redm[3]));
    double sum[1] = {0.0};
    if (m > -INFINITY && m < INFINITY) {  // the same in every thread
      float mine = 0.0f;
#pragma unroll
      for (int p = 0; p < kPasses; ++p)
#pragma unroll
        for (int e = 0; e < kPer; ++e) mine += __builtin_amdgcn_exp2f((v[p][e] - m) * a.k32);
      sum[0] = static_cast<double>(mine);
      block_sums_f64(sum, red);
    }
    if (threadIdx.x == 0) {
      a.maxs[out] = m;  // NaN or infinite: the row is no distribution; -infinite: the slice is all masked
      a.sums[out] = sum[0];
    }
  }
}

// e^((x - m) / temperature) / sum; 0 for a masked x. The difference comes before the factor: x k - m k, fused or not, would
// leave the rounding of m k at x = m, which is many powers of two for an m of 1e20.
__device__ inline double prob(float x, double m, double k, double inv, const double* pow64) {
  const double e = exp2_64th((static_cast<double>(x) - m) * k, pow64) * inv;
  return x == -INFINITY ? 0.0 : e;
}

struct Verdict {
  int n, count;   // accepted, drafted
  int x;          // the draft of row n, where n < count
  double m, inv;  // of row n: its maximum and 1 / sum; inv is NaN where the row has no distribution
};

// Decides on the drafts of row b: thread (t, part) joins every fourth slice of row t, lane by lane of a quad. The same in every
// wave; up to 16 rows at a time (a wave holds 16 quads), so that the loads of a row's slices run side by side.
template <int DT>
__device__ inline Verdict decide(const VerifyArgs& a, int b, int pdt, const double* pow64) {
  const int lane = threadIdx.x & 63, part = lane & 3;
  Verdict r;
  r.count = a.counts != nullptr ? min(max(a.counts[b], 0), a.T) : a.T;
  for (int t0 = 0;; t0 += 16) {
    const int t = t0 + (lane >> 2);
    const bool mine = t <= r.count;
    const int64_t row = static_cast<int64_t>(b) * (a.T + 1) + t, prow = static_cast<int64_t>(b) * a.T + t;
    const int64_t at = row * a.S;
    int x = -1;
    float lx = 0.0f;
    double qx = 1.0, ux = 0.0;
    if (mine && t < r.count) {
      x = a.draft[prow];
      ux = static_cast<double>(a.u[prow]);
      if (x >= 0 && x < a.V) {
        lx = load_as_f32(a.logits, DT, row * a.V + x);
        if (a.probs != nullptr) qx = static_cast<double>(load_as_f32(a.probs, pdt, prow * a.V + x));
      }
    }
    float mx = -INFINITY;
    if (mine) {
#pragma unroll 4
      for (int s = part; s < a.S; s += 4) mx = __builtin_elementwise_maximum(mx, a.maxs[at + s]);
    }
    mx = __builtin_elementwise_maximum(mx, __shfl_xor(mx, 1, 64));
    mx = __builtin_elementwise_maximum(mx, __shfl_xor(mx, 2, 64));
    const bool fine = mx > -INFINITY && mx < INFINITY;
    const double m = fine ? static_cast<double>(mx) : 0.0;
    double z = 0.0;
    if (mine && fine) {
#pragma unroll 4
      for (int s = part; s < a.S; s += 4) {
        const float ms = a.maxs[at + s];
        z += prob(ms, m, a.k, 1.0, pow64) * a.sums[at + s];
      }
    }
    z += __shfl_xor(z, 1, 64);
    z += __shfl_xor(z, 2, 64);
    const double inv = fine ? 1.0 / z : __builtin_nan("");
    const bool good = mine && t < r.count && x >= 0 && x < a.V && ux * qx < prob(lx, m, a.k, inv, pow64);
    const uint64_t bad = ~__ballot(good || t >= r.count) & 0x1111111111111111ull;
    const int stop = bad != 0 ? t0 + (static_cast<int>(__builtin_ctzll(bad)) >> 2) : r.count;
    if (stop < t0 + 16 || r.count < t0 + 16) {
      r.n = min(stop, r.count);
      r.x = __shfl(x, (r.n - t0) * 4, 64);
      r.m = __shfl(m, (r.n - t0) * 4, 64);
      r.inv = __shfl(inv, (r.n - t0) * 4, 64);
      return r;
    }
  }
}

// Of elements base .. base + 7 of the row drawn from: e, and in w the weight by the estimated total, which is zero outside P.
template <int DT, bool VEC>
__device__ inline void weights8(const VerifyArgs& a, const Verdict& v, int b, int base, int pdt, bool residual, int x,
                                const double* pow64, double (&ex)[kPer], double (&w)[kPer]) {
  const int64_t row0 = (static_cast<int64_t>(b) * (a.T + 1) + v.n) * a.V;
  float l[kPer], q[kPer];
  load_row8<DT, VEC>(a.logits, row0, base, a.V, -INFINITY, l);
#pragma unroll
  for (int e = 0; e < kPer; ++e) q[e] = 0.0f;
  if (residual && a.probs != nullptr) {
    const int64_t p0 = (static_cast<int64_t>(b) * a.T + v.n) * a.V;
    if (pdt == SQX_DTYPE_F32) load_row8<SQX_DTYPE_F32, VEC>(a.probs, p0, base, a.V, 0.0f, q);
    else if (pdt == SQX_DTYPE_BF16) load_row8<SQX_DTYPE_BF16, VEC>(a.probs, p0, base, a.V, 0.0f, q);
    else load_row8<SQX_DTYPE_F16, VEC>(a.probs, p0, base, a.V, 0.0f, q);
  }
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    ex[e] = prob(l[e], v.m, a.k, 1.0, pow64);
    const double p = ex[e] * v.inv;
    const double qe = residual && a.probs == nullptr ? (base + e == x ? 1.0 : 0.0) : static_cast<double>(q[e]);
    w[e] = residual ? (p > qe ? p - qe : 0.0) : p;
  }
}

template <int DT, bool VEC>
__global__ __launch_bounds__(256) void verify_rest_kernel(const VerifyArgs a, int pdt) {
  __shared__ double pow64[64], red[3][4];
  fill_pow64(pow64);
  __syncthreads();
  const int s = blockIdx.x, b = blockIdx.y;
  const Verdict v = decide<DT>(a, b, pdt, pow64);
  if (s == 0 && threadIdx.x == 0) {
    a.verdict[3 * b] = v.n;
    a.verdict[3 * b + 1] = v.m;
    a.verdict[3 * b + 2] = v.inv;
  }
  const bool residual = v.n < v.count;
  const int x = v.x;
  double sum[3] = {0.0, 0.0, 0.0};
#pragma unroll 2
  for (int p = 0; p < kPasses; ++p) {
    double ex[kPer], w[kPer];
    weights8<DT, VEC>(a, v, b, s * kSlice + p * kPass + threadIdx.x * kPer, pdt, residual, x, pow64, ex, w);
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      sum[0] += ex[e];
      sum[1] += w[e];
      sum[2] += w[e] > 0.0 ? ex[e] : 0.0;
    }
  }
  block_sums_f64(sum, red);
  if (threadIdx.x < 3) {
    const int64_t each = static_cast<int64_t>(gridDim.y) * a.S;
    a.rest[threadIdx.x * each + static_cast<int64_t>(b) * a.S + s] = threadIdx.x == 0 ? sum[0] : threadIdx.x == 1 ? sum[1] : sum[2];
  }
}

// The pick, by one workgroup of a thread per eight elements of a slice: the slice in which the cumulative sum passes the
// threshold (every wave finds it from the slices' sums, a lane each), then the element in it.
constexpr int kPickThreads = kSlice / kPer, kPickWaves = kPickThreads / 64;
template <int DT, bool VEC>
__global__ __launch_bounds__(kPickThreads) void verify_pick_kernel(const VerifyArgs a, int pdt) {
  __shared__ double pow64[64], wsum[kPickWaves];
  __shared__ int found, last;
  const int b = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  fill_pow64(pow64);
  if (threadIdx.x == 0) {
    found = 0x7fffffff;
    last = -1;
  }
  const double* const rest = a.rest + static_cast<int64_t>(b) * a.S;
  const int64_t each = static_cast<int64_t>(gridDim.x) * a.S;
  double first[3];  // of slice `lane`, on their way beside the verdict
#pragma unroll
  for (int i = 0; i < 3; ++i) first[i] = lane < a.S ? rest[i * each + lane] : 0.0;
  Verdict v;
  v.count = a.counts != nullptr ? min(max(a.counts[b], 0), a.T) : a.T;
  v.n = static_cast<int>(a.verdict[3 * b]);
  v.m = a.verdict[3 * b + 1];
  v.inv = a.verdict[3 * b + 2];
  const double r = static_cast<double>(a.r[b]);
  const int drafted = lane < a.T ? a.draft[static_cast<int64_t>(b) * a.T + lane] : -1;
  const int x = __shfl(drafted, v.n, 64);
  __syncthreads();
  bool residual = v.n < v.count;
  auto sums = [&](int i, int s) -> double { return s >= a.S ? 0.0 : s < 64 ? first[i] : rest[i * each + s]; };
  double all = 0.0;
  for (int s = lane; s < a.S; s += 64) all += sums(0, s);
  all = wave_sum_f64(all);
  const double inv = v.inv == v.inv ? 1.0 / all : v.inv, more = inv - v.inv;
  auto slice_sum = [&](int s) -> double { return residual ? fmax(sums(1, s) + sums(2, s) * more, 0.0) : sums(0, s) * inv; };
  auto sum_all = [&]() {
    double mine = 0.0;
    for (int s = lane; s < a.S; s += 64) mine += slice_sum(s);
    return wave_sum_f64(mine);
  };
  auto scan = [&](double w) {  // inclusive, over the wave
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double u = __shfl_up(w, o, 64);
      if (lane >= o) w += u;
    }
    return w;
  };
  double total = sum_all();
  if (residual && v.inv == v.inv && total <= 0.0) {  // p nowhere above q: drawn from p
    residual = false;
    total = sum_all();
  }
  if (total > 0.0) {  // false for a row without a distribution
    const double theta = r * total;
    int hit = -1, fallback = 0;
    double before = 0.0;
    for (int s0 = 0; s0 < a.S && hit < 0; s0 += 64) {
      const double w = slice_sum(s0 + lane), cum = before + scan(w);
      const uint64_t over = __ballot(w > 0.0 && cum > theta), some = __ballot(w > 0.0);
      if (some != 0) fallback = s0 + 63 - __builtin_clzll(some);
      if (over != 0) {
        const int first = __builtin_ctzll(over);
        hit = s0 + first;
        before = __shfl(cum - w, first, 64);
      } else {
        before = __shfl(cum, 63, 64);
      }
    }
    const bool none = hit < 0;  // r next to 1 and a rounding: the last token that has a weight
    if (none) hit = fallback;
    const int at = hit * kSlice + threadIdx.x * kPer;
    double ex[kPer], w[kPer], mine = 0.0;
    weights8<DT, VEC>(a, v, b, at, pdt, residual, x, pow64, ex, w);
    int first = 0x7fffffff, end = -1;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      if (w[e] > 0.0) end = at + e;  // by the sums' own rule, so that a slice that has a sum has a last one
      w[e] = w[e] > 0.0 ? fmax(w[e] + ex[e] * more, 0.0) : 0.0;
      mine += w[e];
    }
    const double inc = scan(mine);
    if (lane == 63) wsum[wave] = inc;
    __syncthreads();
    double c = before;
#pragma unroll
    for (int i = 0; i < kPickWaves; ++i)
      if (i < wave) c += wsum[i];
    c += inc - mine;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      c += w[e];
      if (first == 0x7fffffff && w[e] > 0.0 && c > theta) first = at + e;
    }
    // the wave's first and last, which lie in its first and last lane that has one; of whole numbers: any order of the waves
    const uint64_t firsts = __ballot(!none && first != 0x7fffffff), ends = __ballot(end >= 0);
    if (firsts != 0 && lane == static_cast<int>(__builtin_ctzll(firsts))) atomicMin(&found, first);
    if (ends != 0 && lane == 63 - static_cast<int>(__builtin_clzll(ends))) atomicMax(&last, end);
    __syncthreads();
  }
  if (threadIdx.x == 0) a.n_acc[b] = v.n;
  if (static_cast<int>(threadIdx.x) <= a.T) {
    const int t = threadIdx.x;
    const int pick = found != 0x7fffffff ? found : last;
    a.tokens[static_cast<int64_t>(b) * (a.T + 1) + t] = t < v.n ? drafted : t == v.n ? pick : -1;  // t is the lane
  }
}

__global__ __launch_bounds__(64) void verify_greedy_kernel(const VerifyArgs a) {
  const int b = blockIdx.x, lane = threadIdx.x;
  const int count = a.counts != nullptr ? min(max(a.counts[b], 0), a.T) : a.T;
  int arg = 0x7fffffff;
  float best = -INFINITY;
  bool good = false;
  if (lane <= count) {
    const int64_t at = (static_cast<int64_t>(b) * (a.T + 1) + lane) * a.S;
    for (int s = 0; s < a.S; ++s) {  // slices are in order: a later one has to be above
      const float ob = a.maxs[at + s];
      if (arg == 0x7fffffff || (best == best && (ob != ob || ob > best))) {
        best = ob;
        arg = a.args[at + s];
      }
    }
    good = lane < count && a.draft[static_cast<int64_t>(b) * a.T + lane] == arg;
  }
  const uint64_t bad = ~__ballot(good);
  const int n = min(static_cast<int>(__builtin_ctzll(bad | (uint64_t(1) << 63))), count);
  const int pick = __shfl(arg, n, 64);
  if (lane == 0) a.n_acc[b] = n;
  if (lane <= a.T)
    a.tokens[static_cast<int64_t>(b) * (a.T + 1) + lane] = lane < n ? a.draft[static_cast<int64_t>(b) * a.T + lane] : lane == n ? pick : -1;
}

}  // namespace sqx

using namespace sqx;

extern "C" int64_t sqx_verify_draft_workspace_bytes(int64_t B, int64_t T, int64_t V) {
  if (B <= 0 || T < 0 || V <= 0) return 0;
  const int64_t S = ceil_div(V, kSlice);
  return B * (T + 1) * S * 16 + B * (3 * S + 3) * 8;
}

extern "C" int sqx_verify_draft(const void* logits, int dtype, const int* draft, const int* counts, const void* probs,
                                int probs_dtype, const float* u, const float* r, double temperature, int64_t B, int64_t T,
                                int64_t V, int* n_accepted, int* tokens, void* ws, int64_t ws_bytes, sqx_stream_t stream) {
  const char* fn = "sqx_verify_draft";
  SQX_REQUIRE(dtype == SQX_DTYPE_F32 || dtype == SQX_DTYPE_BF16 || dtype == SQX_DTYPE_F16, SQX_E_ARG,
              "%s: logits must be F32, BF16 or F16", fn);
  SQX_REQUIRE(probs == nullptr || probs_dtype == SQX_DTYPE_F32 || probs_dtype == SQX_DTYPE_BF16 || probs_dtype == SQX_DTYPE_F16,
              SQX_E_ARG, "%s: probs must be F32, BF16 or F16", fn);
  SQX_REQUIRE(B >= 0 && T >= 0 && T <= kMaxDrafts && B * (T + 1) < 65536, SQX_E_ARG,
              "%s: bad shape (B=%lld, T=%lld up to %d, B (T + 1) below 65536)", fn, (long long)B, (long long)T, kMaxDrafts);
  SQX_REQUIRE(V >= 1 && V < (int64_t(1) << 30), SQX_E_ARG, "%s: V=%lld", fn, (long long)V);
  SQX_REQUIRE(temperature == 0.0 || (temperature >= 1e-4 && temperature <= 1e4), SQX_E_ARG,
              "%s: temperature must be 0 or within 1e-4 .. 1e4", fn);
  if (B == 0) return SQX_OK;
  const bool greedy = temperature == 0.0;
  SQX_REQUIRE(logits && n_accepted && tokens && ws && (T == 0 || draft) && (greedy || (r && (T == 0 || u))), SQX_E_ARG,
              "%s: null pointer", fn);
  const int64_t need = sqx_verify_draft_workspace_bytes(B, T, V);
  SQX_REQUIRE(ws_bytes >= need, SQX_E_SPACE, "%s: workspace of %lld bytes, %lld needed", fn, (long long)ws_bytes,
              (long long)need);
  SQX_REQUIRE(reinterpret_cast<uintptr_t>(ws) % 8 == 0, SQX_E_ARG, "%s: workspace must be 8-byte aligned", fn);
  VerifyArgs a{};
  a.logits = logits; a.draft = draft; a.counts = counts; a.probs = probs; a.u = u; a.r = r;
  a.T = static_cast<int>(T); a.V = static_cast<int>(V); a.S = static_cast<int>(ceil_div(V, kSlice));
  a.k = greedy ? 0.0 : 64.0 * 1.4426950408889634074 / temperature;
  a.k32 = static_cast<float>(a.k / 64.0);
  const int64_t rows = B * (T + 1) * a.S;
  a.sums = static_cast<double*>(ws);
  a.rest = a.sums + rows;
  a.verdict = a.rest + 3 * B * a.S;
  a.maxs = reinterpret_cast<float*>(a.verdict + 3 * B);
  a.args = reinterpret_cast<int*>(a.maxs + rows);
  a.n_acc = n_accepted; a.tokens = tokens;
  auto aligned = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  const bool vec = V % 8 == 0 && aligned(logits) && aligned(probs);
  const hipStream_t s = as_stream(stream);
  const dim3 all(static_cast<unsigned>(a.S), static_cast<unsigned>(B * (T + 1)));
  const dim3 one(static_cast<unsigned>(a.S), static_cast<unsigned>(B)), seqs(static_cast<unsigned>(B));
  auto go = [&](auto dt, auto vv) {
    constexpr int DT = decltype(dt)::value;
    constexpr bool VEC = decltype(vv)::value;
    if (greedy) {
      hipLaunchKernelGGL((verify_stats_kernel<DT, VEC, true>), all, dim3(256), 0, s, a);
      hipLaunchKernelGGL(verify_greedy_kernel, seqs, dim3(64), 0, s, a);
      return;
    }
    hipLaunchKernelGGL((verify_stats_kernel<DT, VEC, false>), all, dim3(256), 0, s, a);
    hipLaunchKernelGGL((verify_rest_kernel<DT, VEC>), one, dim3(256), 0, s, a, probs_dtype);
    hipLaunchKernelGGL((verify_pick_kernel<DT, VEC>), seqs, dim3(kPickThreads), 0, s, a, probs_dtype);
  };
  auto with_vec = [&](auto dt) {
    if (vec) go(dt, std::true_type{});
    else go(dt, std::false_type{});
  };
  if (dtype == SQX_DTYPE_F32) with_vec(std::integral_constant<int, SQX_DTYPE_F32>{});
  else if (dtype == SQX_DTYPE_BF16) with_vec(std::integral_constant<int, SQX_DTYPE_BF16>{});
  else with_vec(std::integral_constant<int, SQX_DTYPE_F16>{});
  SQX_LAUNCH_CHECK(fn);
  return SQX_OK;
}
