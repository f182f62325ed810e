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
//     and the row's maximum need not be known first. Weights are added as whole numbers, of a unit that falls along the bins, so
//     that atomics in any order give the same sum and every weight counts to 2^-49 of itself.
//  2. One workgroup a row joins the histograms and finds the bin that each limit ends in. The tokens of these bins, a few
//     hundred as a rule, are collected and sorted, which gives the cut exactly; slices' weights before the cut come from
//     the histograms, and one slice is read again for the draw itself. Where more than 4096 tokens lie in these bins
//     (equal logits, a row that is nearly flat) the cut is found digit by digit over the row.
//
// A token 32 T or further behind the maximum (the bins' end lies within 1/32 before that) has less than 2^-45 of its weight and is
// never drawn; u itself has 24 bits.
//
// us of the two launches: 1 row of 32000 in fp32 with top-k 6.3 + 10.9, latency: four dependent rounds in each. 64 rows of 128256 in
// bf16 with top-p 22.2 + 40.9: the first is bound by its atomics in LDS and its exponentials in double, one of each a token; in the
// second a row's workgroup, of some 28 us alone, spends 3 on its maximum, 3 on joining the histograms, 8 on collecting, 5 on sorting
// some 100 tokens (15 for 1000) and 6 on the draw; the longest row counts. 201 rows of 50257 in fp32 with all limits 23.4 + 34.0.
// The falling unit costs 1.6 of the 22.2: with one unit of 2^-48 a slice of a heavy token and faint ones was up to 0.3 in 100 of these off.
// The way digit by digit takes 64 such rows 0.47 ms (top-k) to 0.64 and 0.84 ms (top-p; 128256 tokens at T = 20, and all equal), and
// 0.88 ms for bf16 logits around 40, whose steps of 1/4 put some 5000 tokens into the bin where top-p 0.95 ends (56 us around 0): it
// reads the row for each of seven digits, and most of its time goes to atomics on few addresses.
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
constexpr int kFew = 1024;         // up to this k all tokens that may stay are collected, and slices leave no weights
constexpr int kMaxSlices = 128;    // 2^20 tokens
constexpr int kHistThreads = 512, kPickThreads = 1024;
constexpr double kFix = 0x1p50;

// Weights of bin c are between 0.46 and 1.001 times 2^-lift: as whole numbers of 2^-50 2^-lift they are good to 2^-49 of themselves,
// and 8192 of them add up below 2^64.
__host__ __device__ constexpr int bin_lift20(int c) { return (c - 1) * 47274; }  // 2^20 (c - 1) log2 e / kPerT
__host__ __device__ constexpr int bin_lift(int c) { return bin_lift20(c) >> 20; }
constexpr int kMostLift = bin_lift(kBins - 1);

struct SampleArgs {
  const void* logits;  // [B, V]
  const float* u;
  const float *temp_t, *p_t, *minp_t;  // per row, or NULL: the numbers below
  const int* k_t;
  double temp, p, minp;
  int k, V, S;
  float* smax;                // [B, S]
  int* sarg;                  // [B, S]
  double* mass;               // [B, S, kBins], of the slice's maximum's weight, summed from bin 0 on
  unsigned* count;            // [B, S, kBins], likewise
  int* out;
};

// 2^(y / 64 + floor(lift20 / 2^20)), y <= 0.
__device__ inline double pow2_64th(double y, const double* pow64, int lift20 = 0) {
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
  return q * __hiloint2double(__double2hiint(w) + ((n & ~63) << 14) + (lift20 & ~0xfffff), __double2loint(w));  // to its exponent
}

// The whole number nearest to w 2^50, 0 <= w < 2.
__device__ inline unsigned long long to_fix(double w) {
  return __builtin_bit_cast(unsigned long long, fma(w, kFix, 0x1p52)) & 0xfffffffffffffull;
}

// A row's temperature: greedy (0) where it is not above 0, else within 1e-4 .. 1e4.
__device__ inline double row_temp(const SampleArgs& a, int b) {
  const double t = a.temp_t != nullptr ? static_cast<double>(a.temp_t[b]) : a.temp;
  return t > 0.0 ? fmin(fmax(t, 1e-4), 1e4) : 0.0;
}

__device__ inline int row_k(const SampleArgs& a, int b) { return a.k_t != nullptr ? a.k_t[b] : a.k; }

// Eight elements of a row of V in one load, at any multiple of an element: those from `at` on, or the row's last eight where it ends
// within them. Element e is number first(at, V) + e, a thread's own if has(at, V, e).
template <int DT>
struct Loads8 {
  static constexpr int kBytes = DT == SQX_DTYPE_F32 ? 4 : 2;
  struct __attribute__((packed, aligned(kBytes))) Raw { uint32_t w[2 * kBytes]; };
  __device__ static inline int first(int at, int V) { return min(at, V - 8); }  // V >= 8
  __device__ static inline bool has(int at, int V, int e) { return first(at, V) + e >= at; }
  __device__ static inline Raw raw(const void* p, int64_t row0, int at, int V) {
    return *reinterpret_cast<const Raw*>(static_cast<const char*>(p) + (row0 + first(at, V)) * kBytes);
  }
  __device__ static inline void floats(const Raw& r, float (&v)[8]) {
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
  }
  __device__ static inline void load(const void* p, int64_t row0, int at, int V, float (&v)[8]) { floats(raw(p, row0, at, V), v); }
};

// Whether (ov, oi) comes before (cv, ci) as a greedy pick: the first maximum, a NaN counts as one.
__device__ inline bool greedy_takes(float ov, int oi, float cv, int ci) {
  const bool on = ov != ov, cn = cv != cv;
  if (on || cn) return on && (!cn || oi < ci);
  return ov > cv || (ov == cv && oi < ci);
}

// Sums over a wave's lanes up to each one's own, by moves between lanes' registers: within rows of 16, then a row's last lane to the
// next row (of rows 1 and 3), then lane 31 to the upper half. (As shuffles, through LDS, 0.7 us more of 22.)
template <int CTRL, int ROWS, typename N>
__device__ inline void add_moved(N& x) {
  constexpr int W = sizeof(N) / 4;
  uint32_t w[W];
  __builtin_memcpy(w, &x, sizeof(N));
#pragma unroll
  for (int i = 0; i < W; ++i) w[i] = __builtin_amdgcn_update_dpp(0u, w[i], CTRL, ROWS, 0xf, false);  // 0 where no lane sends
  N y;
  __builtin_memcpy(&y, w, sizeof(N));
  x += y;
}
template <typename N>
__device__ inline void wave_sums(N& x) {
  add_moved<0x111, 0xf>(x);  // row_shr:1, 2, 4, 8
  add_moved<0x112, 0xf>(x);
  add_moved<0x114, 0xf>(x);
  add_moved<0x118, 0xf>(x);
  add_moved<0x142, 0xa>(x);  // row_bcast:15
  add_moved<0x143, 0xc>(x);  // row_bcast:31
}

// 8192 tokens a workgroup: 16 a thread stay in registers between the maximum and the bins, and a row of 128256 leaves 16 histograms
// to be joined.
template <int DT>
__global__ __launch_bounds__(kHistThreads) void sample_hist_kernel(const SampleArgs a) {
  constexpr int W = kHistThreads / 64, G = kSampleSlice / (8 * kHistThreads);
  __shared__ double pow64[64];
  __shared__ unsigned long long mass[kBins];
  __shared__ unsigned count[kBins];
  __shared__ float redv[W];
  __shared__ int redi[W];
  __shared__ unsigned __int128 redm[W];
  __shared__ unsigned redc[W];
  static_assert(kBins == 2 * kHistThreads, "two bins a thread");
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
      const int i = Loads8<DT>::first(base + g * 8 * kHistThreads, a.V) + e;
      if (Loads8<DT>::has(base + g * 8 * kHistThreads, a.V, e) && greedy_takes(v[g][e], i, best, arg)) {
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
  const int want_k = row_k(a, b);
  const bool few = want_k >= 1 && want_k <= kFew;
  const double inv = kPerT / T, k = 64.0 * 1.4426950408889634074 / T, m = static_cast<double>(best), top = floor(m * inv);
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const double l = static_cast<double>(v[g][e]);
      const double d = top - floor(l * inv);
      if (Loads8<DT>::has(base + g * 8 * kHistThreads, a.V, e) && d < kBins) {  // false of a NaN: a masked token of a slice that is all masked
        const int bin = static_cast<int>(d);
        if (want_k >= 1) atomicAdd(&count[bin], 1u);
        if (!few) atomicAdd(&mass[bin], to_fix(pow2_64th((l - m) * k, pow64, __mul24(bin - 1, 47274))));
      }
    }
  __syncthreads();
  // sums from bin 0 on: two bins a thread, then over the workgroup. Weights are whole numbers of 2^-50 2^-kMostLift, below 2^110:
  // exact, and so no sum is less than the one before it, rounded to double too
  using u128 = unsigned __int128;
  const int lane = tid & 63, wave = tid >> 6;
  const bool counts = want_k >= 1;  // as `few` of the whole workgroup
  auto of = [&](int bin) { return static_cast<u128>(mass[bin]) << (kMostLift - bin_lift(bin)); };
  const u128 m0 = of(2 * tid), m1 = m0 + of(2 * tid + 1);
  const unsigned c0 = count[2 * tid], c1 = c0 + count[2 * tid + 1];
  u128 ms = m1;
  unsigned cs = c1;
  if (!few) {
    wave_sums(ms);
    if (lane == 63) redm[wave] = ms;
  }
  if (counts) {
    wave_sums(cs);
    if (lane == 63) redc[wave] = cs;
  }
  __syncthreads();
  if (!few) {
    ms -= m1;
#pragma unroll
    for (int w = 0; w < W; ++w) ms += w < wave ? redm[w] : u128{0};
    auto weight = [](u128 x) {
      const double hi = static_cast<double>(static_cast<unsigned long long>(x >> 64));
      return fma(hi, 0x1p64, static_cast<double>(static_cast<unsigned long long>(x))) * (1.0 / kFix) * ldexp(1.0, -kMostLift);
    };
    double2 mo;
    mo.x = weight(ms + m0);
    mo.y = weight(ms + m1);
    reinterpret_cast<double2*>(a.mass + at * kBins)[tid] = mo;
  }
  if (counts) {
    cs -= c1;
#pragma unroll
    for (int w = 0; w < W; ++w) cs += w < wave ? redc[w] : 0u;
    uint2 co;
    co.x = cs + c0;
    co.y = cs + c1;
    reinterpret_cast<uint2*>(a.count + at * kBins)[tid] = co;
  }
}

// Inclusive sums over the workgroup of kPickThreads threads.
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
// The largest, or the least, of the workgroup's values where `is`, into *to; values ascend with the lanes. One atomic a wave.
__device__ inline void raise(int* to, bool is, int value) {
  const unsigned long long b = __ballot(is);
  if (b != 0 && (threadIdx.x & 63) == 63 - __clzll(b)) atomicMax(to, value);
}
__device__ inline void lower(int* to, bool is, int value) {
  const unsigned long long b = __ballot(is);
  if (b != 0 && (threadIdx.x & 63) == __ffsll(b) - 1) atomicMin(to, value);
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

typedef __attribute__((address_space(3))) unsigned long long* lds_u64_t;
// The value of lane ^ X, by moves between lanes' registers.
template <int X>
__device__ inline uint32_t lane_xor(uint32_t v) {
  if constexpr (X == 1) return __builtin_amdgcn_mov_dpp(v, 0xb1, 0xf, 0xf, true);  // within four: 1 0 3 2
  if constexpr (X == 2) return __builtin_amdgcn_mov_dpp(v, 0x4e, 0xf, 0xf, true);  // 2 3 0 1
  if constexpr (X == 4) return __builtin_amdgcn_mov_dpp(__builtin_amdgcn_mov_dpp(v, 0x141, 0xf, 0xf, true), 0x1b, 0xf, 0xf, true);  // eight reversed, fours reversed
  if constexpr (X == 8) return __builtin_amdgcn_mov_dpp(v, 0x128, 0xf, 0xf, true);  // sixteen turned by eight
  if constexpr (X == 16) {
    const auto h = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    const uint32_t h0 = h[0], h1 = h[1];
    return threadIdx.x & 16 ? h0 : h1;
  }
  const auto h = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  const uint32_t h0 = h[0], h1 = h[1];
  return threadIdx.x & 32 ? h0 : h1;
}
// Bitonic steps over 64 E elements of a wave, element E lane + e in x[e]: all of them unrolled, as the instructions of loops over
// strides would take several times those of the steps. `len` is the length of the runs that are made.
template <int STRIDE, int E>
__device__ inline void sort_step(unsigned long long (&x)[E], int len) {
  auto keep = [](unsigned long long mine, unsigned long long other, bool larger) { return (mine > other) == larger ? mine : other; };
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const bool down = ((E * threadIdx.x + e) & len) == 0;
    if constexpr (STRIDE < E) {
      if ((e & STRIDE) == 0) {
        const unsigned long long p = x[e], q = x[e | STRIDE];
        x[e] = keep(p, q, down);
        x[e | STRIDE] = keep(q, p, !down);
      }
    } else {
      constexpr int X = STRIDE / E;
      const unsigned long long y = (static_cast<unsigned long long>(lane_xor<X>(static_cast<uint32_t>(x[e] >> 32))) << 32) |
                                   lane_xor<X>(static_cast<uint32_t>(x[e]));
      x[e] = keep(x[e], y, ((threadIdx.x & X) == 0) == down);
    }
  }
}
template <int LEN, int E>
__device__ inline void sort_merge(unsigned long long (&x)[E], int len) {  // strides LEN / 2 .. 1
  if constexpr (LEN > 1) {
    sort_step<LEN / 2>(x, len);
    sort_merge<LEN / 2>(x, len);
  }
}
template <int LEN, int E>
__device__ inline void sort_wave(unsigned long long (&x)[E]) {  // runs of 2, 4 .. LEN
  if constexpr (LEN > 2) sort_wave<LEN / 2>(x);
  sort_merge<LEN>(x, LEN);
}
// Sorts list[0 .. n), n <= E kPickThreads, the largest first. Only strides of 64 E and more cross LDS behind barriers, and only
// waves that hold some of the n (or are merged with such) take part.
template <int E>
__device__ inline void sort_places(lds_u64_t list, int n) {
  constexpr int W = 64 * E;
  const int tid = threadIdx.x, i0 = E * tid;
  unsigned long long x[E];
#pragma unroll
  for (int e = 0; e < E; ++e) x[e] = i0 + e < n ? list[i0 + e] : 0ull;
  if ((i0 & ~(W - 1)) < n) sort_wave<W>(x);
  for (int len = 2 * W; len < 2 * n; len <<= 1) {  // up to the power of two that holds n
    const bool in = (i0 & ~(len - 1)) < n;
    for (int half = len >> 1; half >= W; half >>= 1) {
      __syncthreads();
      if (in) {
#pragma unroll
        for (int e = 0; e < E; ++e) list[i0 + e] = x[e];
      }
      __syncthreads();
      if (in) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const unsigned long long y = list[(i0 + e) ^ half];
          const bool down = ((i0 + e) & len) == 0, low = (i0 & half) == 0;
          x[e] = (x[e] > y) == (low == down) ? x[e] : y;
        }
      }
    }
    if (in) sort_merge<W>(x, len);
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < E; ++e) list[i0 + e] = x[e];
  __syncthreads();
}
__device__ inline void sort_list(lds_u64_t list, int n) {
  __syncthreads();
  if (n <= kPickThreads) sort_places<1>(list, n);
  else if (n <= 2 * kPickThreads) sort_places<2>(list, n);
  else sort_places<kCap / kPickThreads>(list, n);
}

// A row's bins and weights.
struct RowBins {
  double inv, k, m, top;
  const double* pow64;
  __device__ int bin(double l) const {  // kBins: none. A number above the maximum (a limit's margin) counts as the maximum
    const double d = top - floor(l * inv);
    return d < kBins ? static_cast<int>(fmax(d, 0.0)) : kBins;
  }
  // The least logit of bins up to b: the float next to the bin's end, or a neighbour of it.
  __device__ float least(int b) const {
    if (b < 0) return INFINITY;
    float f = static_cast<float>((top - b) / inv);
    if (f != f) f = -INFINITY;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float lower = nextafterf(f, -INFINITY);
      if (bin(static_cast<double>(lower)) <= b) f = lower;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (bin(static_cast<double>(f)) > b) f = nextafterf(f, INFINITY);
    return f;
  }
  __device__ double weight(float l) const {
    const double w = pow2_64th((static_cast<double>(l) - m) * k, pow64);
    return l == -INFINITY ? 0.0 : w;
  }
};

// One workgroup a row.
template <int DT>
__global__ __launch_bounds__(kPickThreads) void sample_pick_kernel(const SampleArgs a) {
  constexpr int kAhead = DT == SQX_DTYPE_F32 ? 4 : 8, kWaves = kPickThreads / 64, E = kCap / kPickThreads;
  __shared__ double pow64[64];
  __shared__ double redd[kWaves], weight_to[kBins], slice_w[kMaxSlices], scale[kMaxSlices];
  __shared__ int shift[kMaxSlices], count_to[kBins];
  __shared__ float smax[kMaxSlices];
  __shared__ unsigned long long slice_fix[kMaxSlices];
  __shared__ unsigned long long list[kCap];
  __shared__ double before[kCap + 1];  // weight of the list's tokens before each; where there is no list, of a digit's tokens
  __shared__ int found, at_k, at_p0, at_p1, begin[3], end[3], cut_p, cut_m, pick, last, digit_rank;
  __shared__ unsigned long long digit_place, digit_left, dropped;
  const int b = blockIdx.x, tid = threadIdx.x, S = a.S;
  const int64_t at = static_cast<int64_t>(b) * S, row0 = static_cast<int64_t>(b) * a.V;
  // the row's first slices are on their way while the histograms are joined
  typename Loads8<DT>::Raw ahead[kAhead];
#pragma unroll
  for (int j = 0; j < kAhead; ++j) ahead[j] = Loads8<DT>::raw(a.logits, row0, j * kSampleSlice + 8 * tid, a.V);
  if (tid < S) smax[tid] = a.smax[at + tid];
  if (tid < kMaxSlices) slice_fix[tid] = 0;
  fill_pow64(pow64);
  if (tid == 0) {
    found = at_k = at_p0 = at_p1 = 0;
    pick = cut_p = cut_m = 0x7fffffff;
    last = -1;
    dropped = 0;
#pragma unroll
    for (int i = 0; i < 3; ++i) begin[i] = end[i] = 0x7fffffff;
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
  const int want_k = row_k(a, b);
  const double p = a.p_t != nullptr ? static_cast<double>(a.p_t[b]) : a.p, u = static_cast<double>(a.u[b]);
  const double minp_in = a.minp_t != nullptr ? static_cast<double>(a.minp_t[b]) : a.minp, minp = minp_in > 0.0 ? fmin(minp_in, 1.0) : 0.0;
  const bool few = want_k >= 1 && want_k <= kFew, by_p = p < 1.0, by_m = minp > 0.0;

  // ---- the row's histogram: thread i is bin i
  if (tid < S) {
    shift[tid] = r.bin(static_cast<double>(smax[tid]));
    scale[tid] = smax[tid] == -INFINITY ? 0.0 : r.weight(smax[tid]);
  }
  __syncthreads();
  int to = 0;
  double w_to = 0.0;
  auto join = [&](auto counts, auto weights) {
#pragma unroll 8
    for (int s = 0; s < S; ++s) {  // sums of monotone terms in one order: monotone
      const int from = tid - shift[s];
      const int64_t h = (at + s) * kBins + max(from, 0);
      if constexpr (decltype(counts)::value) {
        const unsigned cs = a.count[h];
        to += from >= 0 ? cs : 0u;
      }
      if constexpr (decltype(weights)::value) {
        const double ws = a.mass[h];
        w_to = fma(from >= 0 ? ws : 0.0, scale[s], w_to);
      }
    }
  };
  if (few) join(std::true_type{}, std::false_type{});
  else if (want_k >= 1) join(std::true_type{}, std::true_type{});
  else join(std::false_type{}, std::true_type{});
  weight_to[tid] = w_to;
  count_to[tid] = to;
  __syncthreads();
  const int all = count_to[kBins - 1];
  const bool by_k = want_k >= 1 && want_k < all;

  // ---- the bins that the limits end in
  if (by_k && (tid > 0 ? count_to[tid - 1] : 0) < want_k && want_k <= to) at_k = tid;
  __syncthreads();
  const int rank_k = by_k ? want_k - (at_k > 0 ? count_to[at_k - 1] : 0) : 0;  // of bin at_k the first so many
  const bool whole_k = by_k && want_k == count_to[at_k];
  const double total = weight_to[kBins - 1];
  // the weight of the first k: exactly, or between these
  const double zlo = !by_k ? total : whole_k ? weight_to[at_k] : at_k > 0 ? weight_to[at_k - 1] : 0.0, zhi = by_k ? weight_to[at_k] : total;
  const double edge = r.m + T * log(by_m ? minp : 1.0), slack = 1e-9 * (fabs(edge) + T);
  const int m0 = by_m ? r.bin(edge + slack) : kBins, m1 = by_m ? r.bin(edge - slack) : kBins;
  if (!few && by_p) {
    const double w_before = tid > 0 ? weight_to[tid - 1] : 0.0;
    const bool some = w_to > w_before;
    raise(&at_p0, some && w_before < p * zlo, tid);
    raise(&at_p1, some && w_before < p * zhi, tid);
  }
  __syncthreads();
  const int p0 = at_p0, p1 = max(at_p1, at_p0);
  // Tokens to collect: with a small k all that may stay; else those of the bins in which a limit ends. The cut of top-p lies
  // within the first k: the k-th token is looked for where top-p is off, or where the weight of the first k needs it.
  const bool use_k = few || (by_k && !(by_p && whole_k));
  const bool use_p = !few && by_p, use_m = !few && m0 < kBins && m0 <= (by_p ? p1 : by_k ? at_k : kBins);
  float from[3], below[3];  // of logits, [from, below)
  {
    // lane i of a wave finds one of their ends
    float x = 0.0f;
    const int lane = tid & 63;
    if (lane < 6) {
      const int i = lane >> 1, b0 = i == 0 ? (few ? 0 : at_k) : i == 1 ? p0 : m0, b1 = i == 0 ? (by_k ? at_k : kBins - 1) : i == 1 ? p1 : m1;
      x = r.least(lane & 1 ? b0 - 1 : min(b1, kBins - 1));
    }
    const bool used[3] = {use_k, use_p, use_m};
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const float lo = __shfl(x, 2 * i, 64), hi = __shfl(x, 2 * i + 1, 64);
      from[i] = used[i] ? lo : INFINITY;
      below[i] = used[i] ? hi : -INFINITY;
    }
  }
  const float lowest = fminf(from[0], fminf(from[1], from[2])), highest = fmaxf(below[0], fmaxf(below[1], below[2]));
  const bool limited = use_k || use_p || use_m, several = use_k + use_p + use_m > 1;

  if (limited) {
    // ---- every token of the row, 8 a thread a pass, kAhead passes loaded together
    auto look = [&](const typename Loads8<DT>::Raw& x, int at8) __attribute__((always_inline)) {
      float v[8];
      Loads8<DT>::floats(x, v);
      unsigned hits = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) hits |= static_cast<unsigned>((v[e] >= lowest) & (v[e] < highest)) << e;
      const int i0 = Loads8<DT>::first(at8, a.V);
      if (i0 != at8) {  // of the last eight what no other thread has
#pragma unroll
        for (int e = 0; e < 8; ++e) hits &= Loads8<DT>::has(at8, a.V, e) ? ~0u : ~(1u << e);
      }
      if (__ballot(hits != 0) == 0) return;
      unsigned in = hits;
      if (several) {
        in = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float l = v[e];
          const bool i0 = (l >= from[0]) & (l < below[0]), i1 = (l >= from[1]) & (l < below[1]), i2 = (l >= from[2]) & (l < below[2]);
          in |= static_cast<unsigned>(i0 | i1 | i2) << e;
        }
        in &= hits;
      }
      if (in == 0) return;
      int zero;  // to the compiler any number: it would add a wave's lanes up one by one before a single atomic
      asm volatile("v_mov_b32 %0, 0" : "=v"(zero));
      int to_place = atomicAdd(&found + zero, __popc(in));  // whichever lane comes first: the list is sorted
      while (in != 0) {
        const int e = __ffs(in) - 1;
        in &= in - 1;
        float l = v[0];
#pragma unroll
        for (int j = 1; j < 8; ++j) l = j == e ? v[j] : l;
        if (to_place < kCap) list[to_place] = place(l, i0 + e);
        ++to_place;
      }
    };
    for (int s0 = 0; s0 < S; s0 += kAhead) {
#pragma unroll
      for (int j = 0; j < kAhead; ++j)
        if (s0 + j < S) look(ahead[j], (s0 + j) * kSampleSlice + 8 * tid);
      if (s0 + kAhead < S) {
#pragma unroll
        for (int j = 0; j < kAhead; ++j) ahead[j] = Loads8<DT>::raw(a.logits, row0, (s0 + kAhead + j) * kSampleSlice + 8 * tid, a.V);
      }
    }
    __syncthreads();
  }
  const int n = found;

  if (few && n <= 64) {
    // ---- all that may stay in the first wave's lanes: no further barrier (1 row of 32000, top-k 40: 11.1 us of the kernel, 15.2
    // with the way below)
    if (tid >= 64) return;
    unsigned long long x[1] = {tid < n ? list[tid] : 0ull};
    sort_wave<64>(x);
    const double w = tid < n ? r.weight(place_logit(x[0])) : 0.0;
    double run = w;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double y = __shfl_up(run, o, 64);
      run += tid >= o ? y : 0.0;
    }
    const int first_k = min(want_k, n);
    const double left = p * __shfl(run, first_k - 1, 64);
    const double ahead_of = __shfl_up(run, 1, 64);
    const unsigned long long ends = __ballot(tid > 0 && tid < first_k && ((by_p && !(ahead_of < left)) || w < minp));
    const int stay = min(first_k, ends != 0 ? __ffsll(ends) - 1 : 64);
    // the kept weight of ids up to a lane's, in one order for all lanes
    const uint32_t id = 0xffffffffu - static_cast<uint32_t>(x[0]);
    double upto = 0.0, kept = 0.0;
    for (int i = 0; i < stay; ++i) {
      const double wi = __shfl(w, i, 64);
      upto += static_cast<uint32_t>(__shfl(static_cast<int>(id), i, 64)) <= id ? wi : 0.0;
      kept += wi;
    }
    const bool in = tid < stay;
    uint32_t least = in && upto > u * kept ? id : 0xffffffffu, most = in ? id : 0u;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      least = min(least, static_cast<uint32_t>(__shfl_xor(static_cast<int>(least), o, 64)));
      most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), o, 64)));
    }
    if (tid == 0) a.out[b] = static_cast<int>(least != 0xffffffffu ? least : most);
    return;
  }

  unsigned long long cut = 0;  // kept of bin cut_bin: places from here on
  int cut_bin = kBins;         // bins before it are kept whole
  auto cut_at = [&](unsigned long long q, int bin) {  // the earliest cut counts
    if (bin < cut_bin || (bin == cut_bin && q > cut)) {
      cut = q;
      cut_bin = bin;
    }
  };
  bool walked = false;  // slices' weights are summed token by token
  double e[E];
  if (limited && n <= kCap) {  // the list sorted, its tokens' weights and their sums
    sort_list((lds_u64_t)list, n);
    double mine = 0.0, whole;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const int i = E * tid + j;
      e[j] = 0.0;
      if (i < n) e[j] = r.weight(place_logit(list[i]));
      mine += e[j];
    }
    double run = pick_scan(mine, redd, whole) - mine;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      before[E * tid + j] = run;
      run += e[j];
    }
    if (tid == kPickThreads - 1) before[kCap] = run;
    __syncthreads();
  }

  if (few && n <= kCap) {
    // ---- all that may stay is in the list: the cut is a length, and the draw is among its tokens, by id
    const int first_k = min(want_k, n);
    const double left = p * before[first_k];
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const int i = E * tid + j;
      if (i < first_k && i > 0) {
        lower(&cut_p, by_p && !(before[i] < left), i);
        lower(&cut_m, e[j] < minp, i);
      }
    }
    __syncthreads();
    const int stay = min(first_k, min(cut_p, cut_m));
    unsigned long long mine[E];
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const int i = E * tid + j;
      mine[j] = i < stay ? (list[i] << 32) | static_cast<unsigned>(i) : 0ull;  // the low word of a place falls as the id grows
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < E; ++j) {
      before[E * tid + j] = e[j];
      list[E * tid + j] = mine[j];
    }
    sort_list((lds_u64_t)list, stay);
    double sum = 0.0, kept;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const int i = E * tid + j;
      e[j] = i < stay ? before[static_cast<uint32_t>(list[i])] : 0.0;
      sum += e[j];
    }
    double upto = pick_scan(sum, redd, kept) - sum;
    int first = 0x7fffffff;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      upto += e[j];
      if (E * tid + j < stay && upto > u * kept) first = min(first, E * tid + j);
    }
    lower(&pick, first != 0x7fffffff, first);
    __syncthreads();
    if (tid == 0) a.out[b] = static_cast<int>(0xffffffffu - static_cast<uint32_t>(list[min(pick, stay - 1)] >> 32));
    return;
  }
  if (limited && n <= kCap) {
    // ---- the tokens of the bins that the limits end in
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const int i = E * tid + j;
      if (i >= n) continue;
      const float l = place_logit(list[i]);
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        lower(&begin[k], l < below[k], i);
        lower(&end[k], l < from[k], i);
      }
    }
    __syncthreads();
    auto bound = [&](int x) { return min(x, n); };
    const int k0 = bound(begin[0]), q0 = bound(begin[1]), q1 = bound(end[1]), e0 = bound(begin[2]), e1 = bound(end[2]);
    double z = total;
    if (by_k) z = use_k ? (at_k > 0 ? weight_to[at_k - 1] : 0.0) + (before[min(k0 + rank_k, n)] - before[k0]) : zhi;
    if (use_p) {  // the first token with p z before it
      const double left = p * z - (p0 > 0 ? weight_to[p0 - 1] : 0.0) + before[q0];
      for (int i = q0 + tid; i < q1; i += kPickThreads) lower(&cut_p, i > q0 && !(before[i] < left), i);
    }
    if (use_m) {  // the first token below min_p
      for (int i = e0 + tid; i < e1; i += kPickThreads) lower(&cut_m, r.weight(place_logit(list[i])) < minp, i);
    }
    __syncthreads();
    auto bin_at = [&](int i) { return r.bin(static_cast<double>(place_logit(list[i]))); };
    auto keep_to = [&](int i) { cut_at(list[i], bin_at(i)); };  // the i-th token is the last that stays
    if (use_k) keep_to(min(k0 + rank_k, n) - 1);
    if (use_p && q1 > q0) keep_to(min(cut_p, q1) - 1);
    if (use_m) {
      if (e1 == e0) cut_at(~0ull, m0);  // no token near the limit
      else if (cut_m < e1) cut_at(list[cut_m] + 1, bin_at(cut_m));
      else keep_to(e1 - 1);
    }
  } else if (limited) {
    // ---- too many for the list: the cut digit by digit
    unsigned long long* const digit_w = reinterpret_cast<unsigned long long*>(before);
    unsigned* const digit_c = reinterpret_cast<unsigned*>(before + 256);
    auto walk = [&](auto&& each, auto&& slice_done) {
      for (int s = 0; s < S; ++s) {
        const int i0 = s * kSampleSlice + 8 * tid;
        float v[8];
        Loads8<DT>::load(a.logits, row0, i0, a.V, v);
#pragma unroll 1
        for (int j = 0; j < 8; ++j)
          if (Loads8<DT>::has(i0, a.V, j)) {
            float l = v[0];
#pragma unroll
            for (int k = 1; k < 8; ++k) l = k == j ? v[k] : l;
            if (l > -INFINITY) each(l, place(l, Loads8<DT>::first(i0, a.V) + j));
          }
        slice_done(s);
      }
    };
    auto go_on = [](int) {};
    // The place of the last token that is kept: of the first `rank`, or, among those of places from `cut` on, whose weight is z, of
    // those with less than `left` before them. Their weights are whole numbers of 2^-62 of a power of two above z, so that sums in
    // any order are equal and below 2^63; 2^17 equal ones are off by 2^-45 of z together, where a sum of doubles may be by 2^-36.
    auto select = [&](bool by_rank, int rank, double z, double left) {
      int above = 0;
      if (!by_rank) frexp(z, &above);
      const double unit = ldexp(1.0, 62 - above);
      if (tid == 0) {
        digit_place = 0;
        digit_rank = rank;
        digit_left = by_rank ? 0ull : static_cast<unsigned long long>(ceil(fmax(left * unit, 0.0)));
      }
      for (int sh = 56; sh >= 0; sh -= sh == 32 ? 16 : 8) {  // ids have 20 bits: the highest of the low word's bytes is 255
        if (tid < 256) {
          digit_w[tid] = 0;
          digit_c[tid] = 0;
        }
        __syncthreads();
        const unsigned long long so_far = digit_place;
        walk([&](float l, unsigned long long q) {
          if ((sh < 56 && (q ^ so_far) >> (sh + 8) != 0) || (!by_rank && q < cut)) return;
          const int d = static_cast<int>(q >> sh) & 255;
          const unsigned long long f = by_rank ? 0ull : static_cast<unsigned long long>(fma(r.weight(l), unit, 0.5));
          // equal logits: one addition for the wave's tokens, not one after the other
          const unsigned long long here = __ballot(true);
          const unsigned long long f0 = (static_cast<unsigned long long>(__builtin_amdgcn_readfirstlane(static_cast<unsigned>(f >> 32))) << 32) |
                                        __builtin_amdgcn_readfirstlane(static_cast<unsigned>(f));
          if (__ballot(d == __builtin_amdgcn_readfirstlane(d) && f == f0) == here) {
            if ((threadIdx.x & 63) == __ffsll(here) - 1) {
              atomicAdd(&digit_c[d], static_cast<unsigned>(__popcll(here)));
              if (!by_rank) atomicAdd(&digit_w[d], f * __popcll(here));
            }
          } else {
            atomicAdd(&digit_c[d], 1u);
            if (!by_rank) atomicAdd(&digit_w[d], f);
          }
        }, go_on);
        __syncthreads();
        if (tid == 0) {
          int chosen = -1, rank_at = 0, c_run = 0;
          unsigned long long left_at = 0, w_run = 0;
          for (int d = 255; d >= 0; --d) {
            if (digit_c[d] == 0) continue;
            if (chosen < 0 || (by_rank ? c_run < digit_rank : w_run < digit_left)) {
              chosen = d;
              rank_at = digit_rank - c_run;
              left_at = digit_left - w_run;
            }
            c_run += digit_c[d];
            w_run += digit_w[d];
          }
          digit_place |= static_cast<unsigned long long>(max(chosen, 0)) << sh;
          if (sh == 32) digit_place |= 0xff000000ull;
          digit_rank = rank_at;
          digit_left = left_at;
        }
        __syncthreads();
      }
      const unsigned long long q = digit_place;
      __syncthreads();
      return q;
    };
    if (by_k) cut = select(true, want_k, 0.0, 0.0);
    if (by_p) {
      double mine = 0.0, z;
      walk([&](float l, unsigned long long q) { mine += q >= cut && r.bin(static_cast<double>(l)) < kBins ? r.weight(l) : 0.0; }, go_on);
      pick_scan(mine, redd, z);
      cut = max(cut, select(false, 0, z, p * z));
    }
    if (by_m) {
      walk([&](float l, unsigned long long q) {
        if (r.weight(l) < minp) atomicMax(&dropped, q);
      }, go_on);
      __syncthreads();
      cut = max(cut, dropped + 1);
    }
    double mine = 0.0;
    walk([&](float l, unsigned long long q) { mine += q >= cut && r.bin(static_cast<double>(l)) < kBins ? r.weight(l) : 0.0; },
         [&](int s) {
           double whole;
           pick_scan(mine, redd, whole);
           if (tid == 0) slice_w[s] = whole;
           mine = 0.0;
         });
    walked = true;
  }

  // ---- the weight that each slice keeps: whole bins, and the tokens of the cut's bin
  const double unit = ldexp(kFix, bin_lift(cut_bin));
  if (!walked && cut_bin < kBins) {
    for (int i = tid; i < n; i += kPickThreads) {
      const unsigned long long q = list[i];
      const float l = place_logit(q);
      if (q >= cut && r.bin(static_cast<double>(l)) == cut_bin)
        atomicAdd(&slice_fix[(0xffffffffu - static_cast<uint32_t>(q)) / kSampleSlice], static_cast<unsigned long long>(fma(r.weight(l), unit, 0.5)));
    }
    __syncthreads();
  }
  if (tid < S && !walked) {
    const int upto = min(cut_bin, kBins) - 1 - shift[tid];
    const double whole = upto >= 0 ? a.mass[(at + tid) * kBins + upto] * scale[tid] : 0.0;
    slice_w[tid] = fma(static_cast<double>(slice_fix[tid]), 1.0 / unit, whole);
  }
  __syncthreads();

  // ---- the draw: its slice, then its token
  double kept = 0.0;
  for (int s = 0; s < S; ++s) kept += slice_w[s];
  const double target = u * kept;
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
  const int at8 = chosen * kSampleSlice + 8 * tid, i0 = Loads8<DT>::first(at8, a.V);
  Loads8<DT>::load(a.logits, row0, at8, a.V, x);
  // bins as floats: tokens from `any` on have one, those from `all_from` on one before the cut's
  const float any = r.least(kBins - 1);
  const float all_from = walked ? (cut >> 32 == 0 ? any : INFINITY) : r.least(min(cut_bin, kBins) - 1);  // a cut behind all is none
  const float cut_l = place_logit(cut);  // of no cut a NaN
  const uint32_t cut_i = 0xffffffffu - static_cast<uint32_t>(cut);
  const bool has_cut = walked || cut_bin < kBins;
  double d[8], sum = 0.0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const bool above = has_cut & ((x[j] > cut_l) | ((x[j] == cut_l) & (static_cast<uint32_t>(i0 + j) <= cut_i)));
    const bool in = Loads8<DT>::has(at8, a.V, j) & (x[j] >= any) & ((x[j] >= all_from) | above);
    d[j] = in ? r.weight(x[j]) : 0.0;
    sum += d[j];
  }
  double all_w;
  double upto = skipped + pick_scan(sum, redd, all_w) - sum;
  int first = 0x7fffffff, least = -1;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    upto += d[j];
    if (d[j] > 0.0) {
      least = i0 + j;
      if (upto > target) first = min(first, i0 + j);
    }
  }
  lower(&pick, first != 0x7fffffff, first);
  raise(&last, least >= 0, least);
  __syncthreads();
  if (tid == 0) a.out[b] = pick != 0x7fffffff ? pick : last;
}

// Fewer than eight tokens: a thread a row.
__global__ __launch_bounds__(256) void sample_short_kernel(const SampleArgs a, int dtype, int B) {
  const int b = blockIdx.x * 256 + threadIdx.x;
  if (b >= B) return;
  const int64_t row0 = static_cast<int64_t>(b) * a.V;
  float l[7];
  float best = -INFINITY;
  int arg = 0x7fffffff;
#pragma unroll
  for (int i = 0; i < 7; ++i) {
    l[i] = i < a.V ? load_as_f32(a.logits, dtype, row0 + i) : -INFINITY;
    if (i < a.V && greedy_takes(l[i], i, best, arg)) {
      best = l[i];
      arg = i;
    }
  }
  const double T = row_temp(a, b);
  if (T == 0.0 || !(best < INFINITY) || best == -INFINITY) {
    a.out[b] = T == 0.0 ? arg : -1;
    return;
  }
  const int k = row_k(a, b);
  const double p = a.p_t != nullptr ? static_cast<double>(a.p_t[b]) : a.p, u = static_cast<double>(a.u[b]);
  const double minp = a.minp_t != nullptr ? static_cast<double>(a.minp_t[b]) : a.minp;
  double w[7], z = 0.0;
  int rank[7];
#pragma unroll
  for (int i = 0; i < 7; ++i) {
    const double d = (static_cast<double>(l[i]) - static_cast<double>(best)) / T;
    w[i] = i < a.V && d > -32.0 ? exp(d) : 0.0;
    rank[i] = 0;
#pragma unroll
    for (int j = 0; j < 7; ++j) rank[i] += l[j] > l[i] || (l[j] == l[i] && j < i);
    if (k >= 1 && rank[i] >= k) w[i] = 0.0;
    z += w[i];
  }
  double kept = 0.0, v[7];
#pragma unroll
  for (int i = 0; i < 7; ++i) {
    double before = 0.0;
#pragma unroll
    for (int j = 0; j < 7; ++j) before += rank[j] < rank[i] ? w[j] : 0.0;
    v[i] = (p < 1.0 && rank[i] > 0 && !(before < p * z)) || (minp > 0.0 && w[i] < fmin(minp, 1.0)) ? 0.0 : w[i];
    kept += v[i];
  }
  double upto = 0.0;
  int pick = -1, last = 0;
#pragma unroll
  for (int i = 0; i < 7; ++i) {
    upto += v[i];
    if (v[i] > 0.0) {
      last = i;
      if (pick < 0 && upto > u * kept) pick = i;
    }
  }
  a.out[b] = pick < 0 ? last : pick;
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
  a.mass = static_cast<double*>(ws);
  a.count = reinterpret_cast<unsigned*>(a.mass + B * S * kBins);
  a.smax = reinterpret_cast<float*>(a.count + B * S * kBins);
  a.sarg = reinterpret_cast<int*>(a.smax + B * S);
  a.out = tokens;
  const dim3 grid(static_cast<unsigned>(S), static_cast<unsigned>(B));
  const hipStream_t s = as_stream(stream);
  if (V < 8) {
    hipLaunchKernelGGL(sample_short_kernel, dim3(static_cast<unsigned>(ceil_div(B, 256))), dim3(256), 0, s, a, dtype, static_cast<int>(B));
    SQX_LAUNCH_CHECK(fn);
    return SQX_OK;
  }
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
