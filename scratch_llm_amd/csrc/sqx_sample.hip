// The next token of every row from its logits and one given random number: temperature, top-k, top-p, min-p.
//
// With l_i the logits, m their maximum and w_i = exp((l_i - m) / T), tokens stand in the order of their logits, equal ones by
// their id. Each limit keeps a run from the front: top-k the first k; top-p, of these, those with less than p of these's
// weight before them; min-p those with w_i >= min_p. So what is kept is one run, and its end ("the cut") is one place in the
// order, a pair (logit, id) packed in 64 bits. The draw is the least id for which the kept weight up to it exceeds u times all.
//
// No sort of the vocabulary: two launches.
//  1. Workgroup (slice, row) reads its 8192 logits once, keeps them in registers and leaves a histogram of 1024 bins over the
//     distance from the maximum, 1/32 of the temperature wide: a count and a weight of each bin. Bins lie on a grid that
//     does not depend on the row (floor(32 l / T)), so slices with different maxima are joined by a shift and a factor,
//     and the row's maximum need not be known first. Weights are added as whole numbers of 2^-48 of the slice's largest one:
//     atomics in any order give the same sum.
//  2. One workgroup a row joins the histograms and finds the bin that each limit ends in. The tokens of these bins, a few
//     hundred as a rule, are collected and sorted, which gives the cut exactly; slices' weights before the cut come from
//     the histograms, and one slice is read again for the draw itself. Where more than 4096 tokens lie in these bins
//     (equal logits, a row that is nearly flat) the cut is found digit by digit over the row.
//
// A token 32 T or further behind the maximum (the bins' end lies within 1/32 before that) has less than 2^-45 of its weight and is
// never drawn; u itself has 24 bits.
//
// Weights are double, from a table of 64 powers and a Taylor polynomial of degree 5 (x^6 / 720 < 4e-17): the decisions fall
// between neighbours of sums over a vocabulary, which fp32 would move in one row of a hundred.
#include <type_traits>

#include "sqx_common.h"
#include "sqx_pow64.h"

namespace sqx {

constexpr int kSampleSlice = 8192;
constexpr int kBins = 1024;
constexpr int kPerT = 32;          // bins per unit of (m - l) / T
constexpr int kCap = 4096;         // tokens that are sorted
constexpr int kMaxSlices = 128;    // 2^20 tokens
constexpr int kHistThreads = 512, kPickThreads = 1024;
constexpr double kFix = 0x1p48;

struct SampleArgs {
  const void* logits;  // [B, V]
  const float* u;
  const float *temp_t, *p_t, *minp_t;  // per row, or NULL: the numbers below
  const int* k_t;
  double temp, p, minp;
  int k, V, S;
  float* smax;                // [B, S]
  int* sarg;                  // [B, S]
  unsigned long long* mass;   // [B, S, kBins]
  unsigned* count;            // [B, S, kBins]
  int* out;
};

// 2^(y / 64), y <= 0.
__device__ inline double pow2_64th(double y, const double* pow64) {
  y = fmax(y, -64000.0);
  const double t = y + 0x1.8p52;
  const int n = __double2loint(t);
  const double x = (y - (t - 0x1.8p52)) * (0.693147180559945309417 / 64.0);
  double q = fma(x, 1.0 / 120.0, 1.0 / 24.0);
  q = fma(q, x, 1.0 / 6.0);
  q = fma(q, x, 0.5);
  q = fma(q, x, 1.0);
  q = fma(q, x, 1.0);
  const double w = pow64[n & 63];
  return q * __hiloint2double(__double2hiint(w) + ((n & ~63) << 14), __double2loint(w));
}

// The whole number nearest to w 2^48, 0 <= w <= 1.
__device__ inline unsigned long long to_fix(double w) {
  return __builtin_bit_cast(unsigned long long, fma(w, kFix, 0x1p52)) & 0xfffffffffffffull;
}

// A row's temperature: greedy (0) where it is not above 0, else within 1e-4 .. 1e4.
__device__ inline double row_temp(const SampleArgs& a, int b) {
  const double t = a.temp_t != nullptr ? static_cast<double>(a.temp_t[b]) : a.temp;
  return t > 0.0 ? fmin(fmax(t, 1e-4), 1e4) : 0.0;
}

template <int DT>
struct Loads8 {  // eight elements, at any multiple of an element
  static constexpr int kBytes = DT == SQX_DTYPE_F32 ? 4 : 2;
  struct __attribute__((packed, aligned(kBytes))) Raw { uint32_t w[2 * kBytes]; };
  __device__ static inline void load(const void* p, int64_t row0, int at, int V, float (&v)[8]) {
    if (at + 8 <= V) {
      const Raw r = *reinterpret_cast<const Raw*>(static_cast<const char*>(p) + (row0 + at) * kBytes);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if constexpr (DT == SQX_DTYPE_F32) {
          const uint32_t w = r.w[e];
          v[e] = __builtin_bit_cast(float, w);
        } else {
          const uint32_t w = r.w[e >> 1];
          const uint16_t h = static_cast<uint16_t>(e & 1 ? w >> 16 : w);
          v[e] = DT == SQX_DTYPE_BF16 ? bf16_bits_to_f32(h) : f16_bits_to_f32(h);
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = at + e < V ? load_as_f32(p, DT, row0 + at + e) : -INFINITY;
    }
  }
};

// Whether (ov, oi) comes before (cv, ci) as a greedy pick: the first maximum, a NaN counts as one.
__device__ inline bool greedy_takes(float ov, int oi, float cv, int ci) {
  const bool on = ov != ov, cn = cv != cv;
  if (on || cn) return on && (!cn || oi < ci);
  return ov > cv || (ov == cv && oi < ci);
}

template <int DT>
__global__ __launch_bounds__(kHistThreads) void sample_hist_kernel(const SampleArgs a) {
  constexpr int W = kHistThreads / 64, G = kSampleSlice / (8 * kHistThreads);
  __shared__ double pow64[64];
  __shared__ unsigned long long mass[kBins];
  __shared__ unsigned count[kBins];
  __shared__ float redv[W];
  __shared__ int redi[W];
  const int s = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const int base = s * kSampleSlice + 8 * tid;
  float v[G][8];
#pragma unroll
  for (int g = 0; g < G; ++g) Loads8<DT>::load(a.logits, static_cast<int64_t>(b) * a.V, base + g * 8 * kHistThreads, a.V, v[g]);
  fill_pow64(pow64);
#pragma unroll
  for (int i = tid; i < kBins; i += kHistThreads) {
    mass[i] = 0;
    count[i] = 0;
  }
  float best = -INFINITY;
  int arg = 0x7fffffff;
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int i = base + g * 8 * kHistThreads + e;
      if (i < a.V && greedy_takes(v[g][e], i, best, arg)) {
        best = v[g][e];
        arg = i;
      }
    }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const float ov = __shfl_xor(best, o, 64);
    const int oi = __shfl_xor(arg, o, 64);
    if (greedy_takes(ov, oi, best, arg)) {
      best = ov;
      arg = oi;
    }
  }
  if ((tid & 63) == 0) {
    redv[tid >> 6] = best;
    redi[tid >> 6] = arg;
  }
  __syncthreads();
  best = redv[0];
  arg = redi[0];
#pragma unroll
  for (int w = 1; w < W; ++w)
    if (greedy_takes(redv[w], redi[w], best, arg)) {
      best = redv[w];
      arg = redi[w];
    }
  const int64_t at = static_cast<int64_t>(b) * a.S + s;
  if (tid == 0) {
    a.smax[at] = best;
    a.sarg[at] = arg;
  }
  const double T = row_temp(a, b);
  if (T == 0.0 || !(best < INFINITY)) return;  // greedy, or no distribution: no bin is read
  const double inv = kPerT / T, k = 64.0 * 1.4426950408889634074 / T, m = static_cast<double>(best), top = floor(m * inv);
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int i = base + g * 8 * kHistThreads + e;
      const double l = static_cast<double>(v[g][e]);
      const double d = top - floor(l * inv);
      if (i < a.V && d < kBins) {  // false of a NaN: a masked token of a slice that is all masked
        const int bin = static_cast<int>(d);
        atomicAdd(&count[bin], 1u);
        atomicAdd(&mass[bin], to_fix(pow2_64th((l - m) * k, pow64)));
      }
    }
  __syncthreads();
  for (int i = tid; i < kBins; i += kHistThreads) {
    a.mass[at * kBins + i] = mass[i];
    a.count[at * kBins + i] = count[i];
  }
}

// Inclusive sums over the workgroup of kPickThreads threads, of a double and of an int.
__device__ inline double pick_scan(double x, double* red, double& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  if (lane == 63) red[wave] = x;
  __syncthreads();
  double before = 0.0;
  total = 0.0;
#pragma unroll
  for (int w = 0; w < kPickThreads / 64; ++w) {
    const double r = red[w];
    if (w == wave) before = total;
    total += r;
  }
  __syncthreads();
  return before + x;
}
__device__ inline int pick_scan(int x, int* red, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  if (lane == 63) red[wave] = x;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kPickThreads / 64; ++w) {
    const int r = red[w];
    if (w == wave) before = total;
    total += r;
  }
  __syncthreads();
  return before + x;
}

// A token's place in the order: the larger the earlier. Zeros of either sign are equal.
__device__ inline unsigned long long place(float l, int i) {
  uint32_t u = __builtin_bit_cast(uint32_t, l);
  u = l == 0.0f ? 0u : u;
  const uint32_t key = u ^ (u >> 31 ? 0xffffffffu : 0x80000000u);
  return (static_cast<unsigned long long>(key) << 32) | (0xffffffffu - static_cast<uint32_t>(i));
}
__device__ inline float place_logit(unsigned long long q) {
  const uint32_t key = static_cast<uint32_t>(q >> 32);
  return __builtin_bit_cast(float, key ^ (key >> 31 ? 0x80000000u : 0xffffffffu));
}

// A row's bins and weights.
struct RowBins {
  double inv, k, m, top;
  const double* pow64;
  __device__ int bin(double l) const {  // kBins: none
    const double d = top - floor(l * inv);
    return d < kBins ? static_cast<int>(d) : kBins;
  }
  __device__ double weight(float l) const {
    const double w = pow2_64th((static_cast<double>(l) - m) * k, pow64);
    return l == -INFINITY ? 0.0 : w;
  }
  // Weights of tokens from bin c on are at most 2^-lift(c): they are added as whole numbers of 2^-48 2^-lift.
  __device__ static int lift(int c) { return static_cast<int>((max(c, 1) - 1) * (1.4426950408889634 / kPerT)); }
};

template <int DT>
__global__ __launch_bounds__(kPickThreads) void sample_pick_kernel(const SampleArgs a) {
  __shared__ double pow64[64];
  __shared__ double redd[kPickThreads / 64], weight_to[kBins], slice_w[kMaxSlices], scale[kMaxSlices];
  __shared__ int redi[kPickThreads / 64], shift[kMaxSlices];
  __shared__ float smax[kMaxSlices];
  __shared__ unsigned long long slice_fix[kMaxSlices];
  __shared__ unsigned long long list[kCap];
  __shared__ double before[kCap + 1];  // weight of the list's tokens before each; the digits' counts and weights where it is not sorted
  __shared__ int found, at_k, rank_k, in_k, at_p0, at_p1, pos_k, pos_p, pos_m, n_p, n_m, end_p, end_m, pick, last;
  __shared__ double z0, z1;
  __shared__ unsigned long long digit_place, dropped;
  __shared__ double digit_left;
  __shared__ int digit_rank;
  const int b = blockIdx.x, tid = threadIdx.x, S = a.S;
  const int64_t at = static_cast<int64_t>(b) * S, row0 = static_cast<int64_t>(b) * a.V;
  if (tid < S) smax[tid] = a.smax[at + tid];
  if (tid < kMaxSlices) slice_fix[tid] = 0;
  fill_pow64(pow64);
  if (tid == 0) {
    found = at_k = at_p0 = at_p1 = pos_k = pos_p = pos_m = n_p = n_m = rank_k = in_k = 0;
    end_p = pick = 0x7fffffff;
    end_m = 0x7fffffff;
    last = -1;
    dropped = 0;
  }
  __syncthreads();
  float m = smax[0];
  int ms = 0;
  for (int s = 1; s < S; ++s)
    if (greedy_takes(smax[s], s, m, ms)) {
      m = smax[s];
      ms = s;
    }
  const double T = row_temp(a, b);
  if (T == 0.0 || !(m < INFINITY) || m == -INFINITY) {  // a NaN is not below infinity
    if (tid == 0) a.out[b] = T == 0.0 ? a.sarg[at + ms] : -1;
    return;
  }
  RowBins r;
  r.inv = kPerT / T;
  r.k = 64.0 * 1.4426950408889634074 / T;
  r.m = static_cast<double>(m);
  r.top = floor(r.m * r.inv);
  r.pow64 = pow64;
  const int want_k = a.k_t != nullptr ? a.k_t[b] : a.k;
  const double p = a.p_t != nullptr ? static_cast<double>(a.p_t[b]) : a.p;
  const double minp_in = a.minp_t != nullptr ? static_cast<double>(a.minp_t[b]) : a.minp, minp = minp_in > 0.0 ? fmin(minp_in, 1.0) : 0.0;

  // ---- the row's histogram: thread i is bin i
  if (tid < S) {
    shift[tid] = r.bin(static_cast<double>(smax[tid]));
    scale[tid] = smax[tid] == -INFINITY ? 0.0 : r.weight(smax[tid]) * (1.0 / kFix);
  }
  __syncthreads();
  int c = 0;
  double w = 0.0;
  for (int s = 0; s < S; ++s) {
    const int64_t h = (at + s) * kBins;
    const int from = tid - shift[s];
    if (from >= 0) {
      c += a.count[h + from];
      w = fma(static_cast<double>(a.mass[h + from]), scale[s], w);
    }
  }
  int all;
  double total;
  const int to = pick_scan(c, redi, all);
  weight_to[tid] = pick_scan(w, redd, total);
  __syncthreads();
  const double w_before = tid > 0 ? weight_to[tid - 1] : 0.0;
  const bool by_k = want_k >= 1 && want_k < all, by_p = p < 1.0, by_m = minp > 0.0;

  // ---- the bins that the limits end in
  if (by_k && to - c < want_k && want_k <= to) {
    at_k = tid;
    rank_k = want_k - (to - c);
    in_k = c;
    z0 = rank_k == c ? weight_to[tid] : w_before;  // of the first k: exactly, or between these
    z1 = weight_to[tid];
  }
  __syncthreads();
  const double zlo = by_k ? z0 : total, zhi = by_k ? z1 : total;
  if (by_p && c > 0) {
    if (w_before < p * zlo) atomicMax(&at_p0, tid);
    if (w_before < p * zhi) atomicMax(&at_p1, tid);
  }
  __syncthreads();
  const int p0 = at_p0, p1 = max(at_p1, at_p0);
  const double edge = r.m + T * log(minp), slack = 1e-9 * (fabs(edge) + T);
  const int m0 = by_m ? r.bin(edge + slack) : kBins, m1 = by_m ? r.bin(edge - slack) : kBins;
  // The cut of top-p lies within the first k: the k-th token is looked for where top-p is off, or its weight matters.
  const bool use_k = by_k && !(by_p && rank_k == in_k);
  const bool use_m = m0 < kBins && m0 <= (by_p ? p1 : by_k ? at_k : kBins);
  auto wanted = [&](int bin) { return (use_k && bin == at_k) || (by_p && bin >= p0 && bin <= p1) || (use_m && bin >= m0 && bin <= m1); };
  const bool mine = wanted(tid);
  int n;
  const int pos = pick_scan(mine ? c : 0, redi, n) - (mine ? c : 0);
  if (use_k && tid == at_k) pos_k = pos;
  if (by_p && tid >= p0 && tid <= p1) {
    if (tid == p0) pos_p = pos;
    atomicAdd(&n_p, c);
  }
  if (use_m && tid >= m0 && tid <= m1) {
    if (tid == m0) pos_m = pos;
    atomicAdd(&n_m, c);
  }
  __syncthreads();

  // Every token of the row, 8 a thread a pass, the next pass on its way.
  auto walk = [&](auto&& each) __attribute__((always_inline)) {
    float x[8], y[8];
    Loads8<DT>::load(a.logits, row0, 8 * tid, a.V, x);
    for (int s = 0; s < S; ++s) {
      const int i0 = s * kSampleSlice + 8 * tid;
      if (s + 1 < S) Loads8<DT>::load(a.logits, row0, i0 + kSampleSlice, a.V, y);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (i0 + e < a.V) each(x[e], i0 + e, s);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = y[e];
    }
  };

  unsigned long long cut = 0;  // kept of bin cut_bin: places from here on
  int cut_bin = kBins;         // bins before it are kept whole
  auto cut_at = [&](unsigned long long q, int bin) {  // the earliest cut counts
    if (bin < cut_bin || (bin == cut_bin && q > cut)) {
      cut = q;
      cut_bin = bin;
    }
  };
  if (n > 0 && n <= kCap) {
    // ---- collected and sorted
    walk([&](float l, int i, int) {
      if (wanted(r.bin(static_cast<double>(l)))) list[min(atomicAdd(&found, 1), kCap - 1)] = place(l, i);
    });
    int size = 64;
    while (size < n) size <<= 1;
    __syncthreads();
    for (int i = tid; i < size; i += kPickThreads)
      if (i >= n) list[i] = 0;
    __syncthreads();
    for (int len = 2; len <= size; len <<= 1)
      for (int half = len >> 1; half > 0; half >>= 1) {
        for (int i = tid; i < size / 2; i += kPickThreads) {
          const int lo = 2 * i - (i & (half - 1)), hi = lo + half;
          const unsigned long long x = list[lo], y = list[hi];
          if ((x < y) == ((lo & len) == 0)) {
            list[lo] = y;
            list[hi] = x;
          }
        }
        __syncthreads();
      }
    constexpr int E = kCap / kPickThreads;
    double e[E], mine_w = 0.0;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const int i = E * tid + j;
      e[j] = i < n ? r.weight(place_logit(list[i])) : 0.0;
      mine_w += e[j];
    }
    double all_w;
    double run = pick_scan(mine_w, redd, all_w) - mine_w;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      before[E * tid + j] = run;
      run += e[j];
    }
    if (tid == kPickThreads - 1) before[kCap] = run;
    __syncthreads();
    double z = total;
    if (by_k) z = use_k ? (at_k > 0 ? weight_to[at_k - 1] : 0.0) + (before[pos_k + rank_k] - before[pos_k]) : zhi;
    if (by_p) {  // the last token with less than p z before it
      const double left = p * z - (p0 > 0 ? weight_to[p0 - 1] : 0.0) + before[pos_p];
      for (int i = tid; i < n_p; i += kPickThreads)
        if (i > 0 && !(before[pos_p + i] < left)) atomicMin(&end_p, i - 1);
    }
    if (use_m) {  // the first token below min_p
      for (int i = tid; i < n_m; i += kPickThreads)
        if (r.weight(place_logit(list[pos_m + i])) < minp) atomicMin(&end_m, i);
    }
    __syncthreads();
    auto cut_here = [&](int i, int more) { cut_at(list[i] + more, r.bin(static_cast<double>(place_logit(list[i])))); };
    if (use_k) cut_here(pos_k + rank_k - 1, 0);
    if (by_p) cut_here(pos_p + min(end_p, n_p - 1), 0);
    if (use_m && n_m > 0) {
      if (end_m < n_m) cut_here(pos_m + end_m, 1);
      else cut_here(pos_m + n_m - 1, 0);
    }
  } else if (n > kCap) {
    // ---- digit by digit
    unsigned long long* const digit_w = reinterpret_cast<unsigned long long*>(before);
    unsigned* const digit_c = reinterpret_cast<unsigned*>(before + 256);
    // The place of the last token of bins b0 .. b1 that is kept: of the first `rank`, or of those with less than `left` before
    // them, both counted from bin b0.
    auto select = [&](int b0, int b1, bool by_rank, int rank, double left) {
      const double unit = ldexp(1.0, r.lift(b0) + 42);  // 2^20 tokens of at most 1 / unit 2^42 fit 64 bits
      if (tid == 0) {
        digit_place = 0;
        digit_rank = rank;
        digit_left = left * unit;
      }
      for (int sh = 56; sh >= 0; sh -= 8) {
        if (tid < 256) {
          digit_w[tid] = 0;
          digit_c[tid] = 0;
        }
        __syncthreads();
        const unsigned long long so_far = digit_place;
        walk([&](float l, int i, int) {
          const int bin = r.bin(static_cast<double>(l));
          const unsigned long long q = place(l, i);
          if (bin < b0 || bin > b1 || (sh < 56 && (q ^ so_far) >> (sh + 8) != 0)) return;
          const int d = static_cast<int>(q >> sh) & 255;
          const unsigned long long f = static_cast<unsigned long long>(fma(r.weight(l), unit, 0.5));
          const unsigned long long same = __ballot(d == __builtin_amdgcn_readfirstlane(d));
          if (same == __ballot(true)) {  // equal logits: one addition for the wave's tokens, not one after the other
            unsigned long long sum = 0;
            for (unsigned long long left_lanes = same; left_lanes != 0; left_lanes &= left_lanes - 1) {
              const int lane = __ffsll(left_lanes) - 1;
              const unsigned lo = __builtin_amdgcn_readlane(static_cast<unsigned>(f), lane);
              const unsigned hi = __builtin_amdgcn_readlane(static_cast<unsigned>(f >> 32), lane);
              sum += (static_cast<unsigned long long>(hi) << 32) | lo;
            }
            if ((threadIdx.x & 63) == __ffsll(same) - 1) {
              atomicAdd(&digit_c[d], static_cast<unsigned>(__popcll(same)));
              atomicAdd(&digit_w[d], sum);
            }
          } else {
            atomicAdd(&digit_c[d], 1u);
            atomicAdd(&digit_w[d], f);
          }
        });
        __syncthreads();
        if (tid == 0) {
          int chosen = -1, rank_at = 0;
          double left_at = 0.0, w_run = 0.0;
          int c_run = 0;
          for (int d = 255; d >= 0; --d) {
            if (digit_c[d] == 0) continue;
            if (chosen < 0 || (by_rank ? c_run < digit_rank : w_run < digit_left)) {
              chosen = d;
              rank_at = digit_rank - c_run;
              left_at = digit_left - w_run;
            }
            c_run += digit_c[d];
            w_run += static_cast<double>(digit_w[d]);
          }
          digit_place |= static_cast<unsigned long long>(max(chosen, 0)) << sh;
          digit_rank = rank_at;
          digit_left = left_at;
        }
        __syncthreads();
      }
      const unsigned long long q = digit_place;
      __syncthreads();
      return q;
    };
    // The weight of bin b0's tokens up to place q, in units of the row's largest.
    auto weight_up_to = [&](int b0, unsigned long long q) {
      double sum = 0.0, all_w;
      walk([&](float l, int i, int) {
        if (r.bin(static_cast<double>(l)) == b0 && place(l, i) >= q) sum += r.weight(l);
      });
      pick_scan(sum, redd, all_w);
      return all_w;
    };
    double z = total;
    if (use_k) {
      const unsigned long long q = select(at_k, at_k, true, rank_k, 0.0);
      cut_at(q, at_k);
      if (by_p) z = (at_k > 0 ? weight_to[at_k - 1] : 0.0) + weight_up_to(at_k, q);
    } else if (by_k) {
      z = zhi;
    }
    if (by_p) {
      const unsigned long long q = select(p0, p1, false, 0, p * z - (p0 > 0 ? weight_to[p0 - 1] : 0.0));
      cut_at(q, r.bin(static_cast<double>(place_logit(q))));
    }
    if (use_m) {
      walk([&](float l, int i, int) {
        const int bin = r.bin(static_cast<double>(l));
        if (bin >= m0 && bin <= m1 && r.weight(l) < minp) atomicMax(&dropped, place(l, i));
      });
      __syncthreads();
      if (dropped != 0) cut_at(dropped + 1, r.bin(static_cast<double>(place_logit(dropped))));
      else cut_at(~0ull, m1 + 1);
    }
  }
  if (use_m && n_m == 0) cut_at(~0ull, m0);  // no token near the limit

  // ---- the weight that each slice keeps: whole bins, and the tokens of the cut's bin
  const double unit = ldexp(kFix / 64, r.lift(cut_bin)), back = 1.0 / unit;  // 8192 tokens of at most 2^42 fit 64 bits
  if (cut_bin < kBins) {
    auto add = [&](float l, unsigned long long q, int s) {
      if (q >= cut && r.bin(static_cast<double>(l)) == cut_bin)
        atomicAdd(&slice_fix[s], static_cast<unsigned long long>(fma(r.weight(l), unit, 0.5)));
    };
    if (n <= kCap) {
      for (int i = tid; i < n; i += kPickThreads)
        add(place_logit(list[i]), list[i], static_cast<int>((0xffffffffu - static_cast<uint32_t>(list[i])) / kSampleSlice));
    } else {
      walk([&](float l, int i, int s) { add(l, place(l, i), s); });
    }
    __syncthreads();
  }
  for (int s = tid >> 6; s < S; s += kPickThreads / 64) {
    double sum = 0.0;
    for (int i = tid & 63; i < kBins && i + shift[s] < min(cut_bin, kBins); i += 64)
      sum = fma(static_cast<double>(a.mass[(at + s) * kBins + i]), scale[s], sum);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o, 64);
    if ((tid & 63) == 0) slice_w[s] = fma(static_cast<double>(slice_fix[s]), back, sum);
  }
  __syncthreads();

  // ---- the draw: its slice, then its token
  double kept = 0.0;
  for (int s = 0; s < S; ++s) kept += slice_w[s];
  const double target = static_cast<double>(a.u[b]) * kept;
  int chosen = -1;
  double skipped = 0.0, run = 0.0;
  for (int s = 0; s < S; ++s) {
    if (slice_w[s] > 0.0 && (chosen < 0 || !(run > target))) {  // the first that passes the target, else the last with weight
      chosen = s;
      skipped = run;
    }
    run += slice_w[s];
  }
  chosen = max(chosen, 0);
  float x[8];
  const int i0 = chosen * kSampleSlice + 8 * tid;
  Loads8<DT>::load(a.logits, row0, i0, a.V, x);
  double e[8], sum = 0.0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int bin = r.bin(static_cast<double>(x[j]));
    const bool in = i0 + j < a.V && bin < kBins && (bin < cut_bin || (bin == cut_bin && place(x[j], i0 + j) >= cut));
    e[j] = in ? r.weight(x[j]) : 0.0;
    sum += e[j];
  }
  double all_w;
  double upto = skipped + pick_scan(sum, redd, all_w) - sum;
  int first = 0x7fffffff, end = -1;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    upto += e[j];
    if (e[j] > 0.0) {
      end = i0 + j;
      if (upto > target) first = min(first, i0 + j);
    }
  }
  if (first != 0x7fffffff) atomicMin(&pick, first);
  if (end >= 0) atomicMax(&last, end);
  __syncthreads();
  if (tid == 0) a.out[b] = pick != 0x7fffffff ? pick : last;
}

}  // namespace sqx

using namespace sqx;

extern "C" int64_t sqx_sample_workspace_bytes(int64_t B, int64_t V) {
  if (B <= 0 || V <= 0) return 0;
  const int64_t S = ceil_div(V, kSampleSlice);
  return B * S * (kBins * 12 + 8) + 16;
}

extern "C" int sqx_sample(const void* logits, int dtype, const float* u, const float* temperature_t, double temperature,
                          const int* top_k_t, int64_t top_k, const float* top_p_t, double top_p, const float* min_p_t, double min_p,
                          int64_t B, int64_t V, int* tokens, void* ws, int64_t ws_bytes, sqx_stream_t stream) {
  const char* fn = "sqx_sample";
  SQX_REQUIRE(dtype == SQX_DTYPE_F32 || dtype == SQX_DTYPE_BF16 || dtype == SQX_DTYPE_F16, SQX_E_ARG,
              "%s: logits must be F32, BF16 or F16", fn);
  SQX_REQUIRE(B >= 0 && B < 65536 && V >= 1 && V <= (int64_t(1) << 20), SQX_E_ARG,
              "%s: B=%lld rows (below 65536) of V=%lld tokens (1 to 2^20)", fn, (long long)B, (long long)V);
  SQX_REQUIRE(temperature_t || temperature == 0.0 || (temperature >= 1e-4 && temperature <= 1e4), SQX_E_ARG,
              "%s: temperature must be 0 or within 1e-4 .. 1e4", fn);
  SQX_REQUIRE(top_k_t || top_k >= 0, SQX_E_ARG, "%s: top_k must not be negative", fn);
  SQX_REQUIRE(top_p_t || (top_p > 0.0 && top_p <= 1.0), SQX_E_ARG, "%s: top_p must be above 0 and at most 1", fn);
  SQX_REQUIRE(min_p_t || (min_p >= 0.0 && min_p <= 1.0), SQX_E_ARG, "%s: min_p must be within 0 .. 1", fn);
  if (B == 0) return SQX_OK;
  SQX_REQUIRE(logits && u && tokens, SQX_E_ARG, "%s: null pointer", fn);
  SQX_REQUIRE(reinterpret_cast<uintptr_t>(logits) % (dtype == SQX_DTYPE_F32 ? 4 : 2) == 0, SQX_E_ARG, "%s: misaligned logits", fn);
  const int64_t S = ceil_div(V, kSampleSlice), need = sqx_sample_workspace_bytes(B, V);
  SQX_REQUIRE(ws != nullptr && ws_bytes >= need && reinterpret_cast<uintptr_t>(ws) % 16 == 0, SQX_E_SPACE,
              "%s: %lld bytes of 16-byte aligned workspace needed, %lld given", fn, (long long)need, (long long)ws_bytes);
  SampleArgs a{};
  a.logits = logits; a.u = u;
  a.temp_t = temperature_t; a.p_t = top_p_t; a.minp_t = min_p_t; a.k_t = top_k_t;
  a.temp = temperature; a.p = top_p; a.minp = min_p;
  a.k = static_cast<int>(std::min<int64_t>(top_k, 0x7fffffff)); a.V = static_cast<int>(V); a.S = static_cast<int>(S);
  a.mass = static_cast<unsigned long long*>(ws);
  a.count = reinterpret_cast<unsigned*>(a.mass + B * S * kBins);
  a.smax = reinterpret_cast<float*>(a.count + B * S * kBins);
  a.sarg = reinterpret_cast<int*>(a.smax + B * S);
  a.out = tokens;
  const dim3 grid(static_cast<unsigned>(S), static_cast<unsigned>(B));
  const hipStream_t s = as_stream(stream);
  auto go = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    hipLaunchKernelGGL((sample_hist_kernel<DT>), grid, dim3(kHistThreads), 0, s, a);
    hipLaunchKernelGGL((sample_pick_kernel<DT>), dim3(static_cast<unsigned>(B)), dim3(kPickThreads), 0, s, a);
  };
  if (dtype == SQX_DTYPE_F32) go(std::integral_constant<int, SQX_DTYPE_F32>{});
  else if (dtype == SQX_DTYPE_BF16) go(std::integral_constant<int, SQX_DTYPE_BF16>{});
  else go(std::integral_constant<int, SQX_DTYPE_F16>{});
  SQX_LAUNCH_CHECK(fn);
  return SQX_OK;
}
