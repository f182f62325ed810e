// Attention of a row's new tokens over the block-scaled 8-bit KV cache (layout: sqx_kvblock.h): one decoded token, a few
// drafted ones, a chunk of a prompt. Token t of row b stands at position starts[b] + t and attends the keys at and
// before it; the G query heads of a kv head share its keys, so (token, head) pairs are the rows of one product.
//
// Per 64 keys a wave computes S^T = K Q^T and O^T += V^T P^T with v_mfma_f32_16x16x32_f16. Codes of either format are
// exact in fp16. Queries are exact too: bf16 rows are first brought to a maximum just below 2^15 by a power of two, which
// fp16's 11 bits hold down to 2^-31 of the row's maximum.
//  - Which key is which row of a score tile is free to choose: row p of tile t is key 16 (p / 4) + 4 t + p % 4. Lane (g, r)
//    (g = lane / 16) then gets the scores of the 16 keys 16 g .. 16 g + 15 of query row r over the four tiles, which is
//    the order in which it must hold P for the second product: the probabilities never leave their lane.
//  - Values are stored [D, block], so a lane's part of V^T is 16 consecutive bytes, the same 16 keys.
//  - A page holds at least 16 tokens, so a lane's 16 keys share one key scale and one value scale. With x the raw
//    product, u = x (ks scale log2 e) + log2 vs; with m a maximum of u, p = 2^(u - m + 7), O sums p c and the softmax's
//    denominator sums p / vs. Probabilities thus carry their value scale, and the largest terms of the output are near
//    2^7 whatever the scales. m follows the running maximum only where that has grown by more than 8: p stays below
//    2^15, and a prompt rescales O in a few of its first steps only. fp16 rounds p by 2^-11 of itself, or by 2^-25
//    (2^-32 of the largest) where it is subnormal, which the matrix unit keeps. Sums, m and the denominator are fp32.
#include "sqx_kvblock.h"

namespace sqx {

struct KvAttnArgs {
  const uint16_t* q;
  int64_t q_sb, q_st, q_sh;
  const uint8_t *kc, *vc;
  const float *ks, *vs;
  const int *table, *starts, *counts;
  uint16_t* out;  // [B, T, H, D]
  float *po, *pml;
  int T, H, Hkv, G, width, pages, block, shift, nsplit;
  float qscale;  // scale * log2(e)
};

constexpr int kStepKeys = 64;
constexpr int kAttnWaves = 4;
constexpr float kPOffset = 7.0f;      // p of the maximum that m stands for
constexpr float kPGrowth = 8.0f;      // m stays while the maximum is within this: p is below 2^15
constexpr float kTinyScale = 1e-30f;  // stands in for a scale of zero (a page never written)

// Four codes of a dword as fp16 pairs (elements 0, 1 and 2, 3), exact.
template <bool E4M3>
__device__ inline void codes_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (E4M3) {
    lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
    hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true));
  } else {
    // byte c + 128 under the exponent of 1024 is the fp16 number 1024 + c + 128
    const uint32_t u = w ^ 0x80808080u;
    const uint32_t a = __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u), b = __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u);
    const f16x2_t off = {static_cast<_Float16>(-1152.0f), static_cast<_Float16>(-1152.0f)};
    lo = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2_t, a) + off);
    hi = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2_t, b) + off);
  }
}

// Eight codes as an MFMA operand.
template <bool E4M3>
__device__ inline u32x4_t codes8(uint32_t w0, uint32_t w1) {
  uint32_t a, b, c, d;
  codes_to_f16<E4M3>(w0, a, b);
  codes_to_f16<E4M3>(w1, c, d);
  return u32x4_t{a, b, c, d};
}

// Bytes of w that are E4M3 NaNs, as 0x80 in their place.
__device__ inline uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// The maximum over the four lane groups, in all of them: two exchanges in registers.
__device__ inline float groups_max(float x) {
  uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto h = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const uint32_t h0 = h[0], h1 = h[1];  // through scalars: hipcc's bit_cast of a vector element reads element 0
  x = __builtin_elementwise_maximum(__builtin_bit_cast(float, h0), __builtin_bit_cast(float, h1));
  u = __builtin_bit_cast(uint32_t, x);
  const auto q = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t q0 = q[0], q1 = q[1];
  return __builtin_elementwise_maximum(__builtin_bit_cast(float, q0), __builtin_bit_cast(float, q1));
}

// One 64-key step of the softmax for R tiles of 16 query rows: lane (g, r) holds the raw scores of keys 16 g + 4 t + j of
// row r in sc[.][t][j], of which those from behind[.] on are not attended (MASKED); f and lvs bring them to u, ivs is
// 1 / vs. Updates m, l and O^T's columns, leaves p as the operands pf. A NaN score makes its row's l NaN: m takes no part.
template <int R, int VD, bool MASKED>
__device__ inline void softmax_step(f32x4_t (&sc)[R][4], const int (&behind)[R], const float (&f)[R], float lvs, float ivs,
                                    float (&m)[R], float (&l)[R], f32x4_t (&o)[R][VD], u32x4_t (&pf)[R][2]) {
  float mx[R];
  bool grow = false;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    if constexpr (MASKED) {
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) sc[i][t][j] = 4 * t + j >= behind[i] ? -INFINITY : sc[i][t][j];
    }
    mx[i] = sc[i][0][0];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j) mx[i] = __builtin_elementwise_maximum(mx[i], sc[i][t][j]);
    mx[i] = fmaf(mx[i], f[i], lvs);  // f > 0: the maximum of u
    if constexpr (MASKED) mx[i] = behind[i] <= 0 ? -INFINITY : mx[i];  // a page that no key is attended on: any scale
    mx[i] = groups_max(mx[i]);
    grow = grow || mx[i] > m[i] + kPGrowth;
  }
  if (__ballot(grow) != 0) {  // wave-uniform; also from -infinity
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const float mn = fmaxf(m[i], mx[i]);  // not a NaN
      const float al = m[i] == mn ? 1.0f : __builtin_amdgcn_exp2f(m[i] - mn);
      l[i] *= al;
#pragma unroll
      for (int c = 0; c < VD; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][c][j] *= al;
      m[i] = mn;
    }
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const float base = lvs - (m[i] == -INFINITY ? 0.0f : m[i]) + kPOffset;
    float p[16], sum = 0.0f;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float& e = p[4 * t + j];
        e = __builtin_amdgcn_exp2f(fmaf(sc[i][t][j], f[i], base));
        if constexpr (MASKED) e = 4 * t + j >= behind[i] ? 0.0f : e;  // whatever its page's scales are
        sum += e;  // in fp32, not of the rounded p: a p too small for fp16 may be a large p / vs
      }
#pragma unroll
    for (int e = 0; e < 8; ++e) pf[i][e >> 2][e & 3] = ActF16::pack_rne(p[2 * e], p[2 * e + 1]);
    if constexpr (MASKED) l[i] = sum == 0.0f ? l[i] : fmaf(sum, ivs, l[i]);
    else l[i] = fmaf(sum, ivs, l[i]);
  }
}

// 1.0 for the lane's keys below `behind`, 0 from there on, in the order of softmax_step's pf.
__device__ inline void attended(int behind, u32x4_t (&am)[2]) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
    am[i >> 2][i & 3] = (2 * i < behind ? 0x3c00u : 0u) | (2 * i + 1 < behind ? 0x3c000000u : 0u);
}

// The 8 N dims of query row `src` that a lane holds, 8 each from column `at(k)`, as fp16, and the factor that brings a raw
// score to u. bf16 rows are scaled by a power of two; the lanes of a row, LANES apart, share it.
template <int N, bool BF16, int LANES, typename F>
__device__ inline float load_query_at(const uint16_t* src, bool ok, float qscale, u32x4_t (&qf)[N], const F& at) {
#pragma unroll
  for (int k = 0; k < N; ++k) {
    qf[k] = u32x4_t{0u, 0u, 0u, 0u};
    if (ok) qf[k] = *reinterpret_cast<const u32x4_t*>(src + at(k));
  }
  if constexpr (!BF16) return qscale;
  float most = 0.0f;
#pragma unroll
  for (int k = 0; k < N; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t w = qf[k][e];
      most = fmaxf(most, fmaxf(fabsf(bf16_lo(w)), fabsf(bf16_hi(w))));
    }
#pragma unroll
  for (int x = LANES; x < 64; x <<= 1) most = fmaxf(most, __shfl_xor(most, x, 64));
  float up = 1.0f;
  if (most > 0.0f && most <= 3.402823466e38f) {
    int e;
    frexpf(most, &e);
    up = ldexpf(1.0f, 15 - max(e, -100));
  }
#pragma unroll
  for (int k = 0; k < N; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t w = qf[k][e];
      qf[k][e] = ActF16::pack_rne(bf16_lo(w) * up, bf16_hi(w) * up);
    }
  return qscale * (1.0f / up);
}
template <int KD, bool BF16>  // lane (g, r) of four groups: 64 i + 16 g + 8 half ..
__device__ inline float load_query(const uint16_t* src, bool ok, int g, float qscale, u32x4_t (&qf)[2 * KD]) {
  return load_query_at<2 * KD, BF16, 16>(src, ok, qscale, qf, [&](int k) { return 64 * (k >> 1) + 16 * g + 8 * (k & 1); });
}
template <int KD, bool BF16>  // lane (hi, r) of two: 32 i + 16 hi + 8 half ..
__device__ inline float load_query32(const uint16_t* src, bool ok, int hi, float qscale, u32x4_t (&qf)[2 * KD]) {
  return load_query_at<2 * KD, BF16, 32>(src, ok, qscale, qf, [&](int k) { return 32 * (k >> 1) + 16 * hi + 8 * (k & 1); });
}

// The rows and keys of a tile of `span` rows from row0: token `last` is its last one below the count, keys below `keys` are
// attended by some row of it, keys up to `first` by every row. A token past the table attends what the table has.
struct KvSpan {
  int count, start, most, first, keys;
  __device__ int position(int t) const {  // without the sum's overflow
    return static_cast<int>(min(static_cast<int64_t>(start) + t, static_cast<int64_t>(most) - 1));
  }
};
__device__ inline bool kv_span(const KvAttnArgs& a, int b, int row0, int span, KvSpan& s) {
  s.count = a.counts != nullptr ? min(max(a.counts[b], 0), a.T) : a.T;
  if (row0 / a.G >= s.count) return false;  // rows from the count on are left as they are
  s.start = a.starts[b];
  s.most = a.width * a.block;  // below 2^30
  s.keys = max(s.position(min((row0 + span - 1) / a.G, s.count - 1)) + 1, 0);
  s.first = s.position(row0 / a.G);
  return true;
}

// Eight (D / 16) output dims of a joined row: to the workspace as they are, or divided and rounded to the output.
template <int D, bool BF16, int DT>
__device__ inline void put_row(const KvAttnArgs& a, int b, int h, int split, int row, int jd, float M, float sum,
                               const float (&acc)[DT]) {
  const int rows = a.T * a.G;
  if (a.nsplit > 1) {
    const int64_t at = ((static_cast<int64_t>(b) * a.Hkv + h) * a.nsplit + split) * rows + row;
    if (jd == 0) {
      a.pml[2 * at] = M;
      a.pml[2 * at + 1] = sum;
    }
#pragma unroll
    for (int d = 0; d < DT; d += 4)
      *reinterpret_cast<f32x4_t*>(a.po + at * D + jd + d) = f32x4_t{acc[d], acc[d + 1], acc[d + 2], acc[d + 3]};
    return;
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;  // no key: zeros
  uint16_t* dst = a.out + ((static_cast<int64_t>(b) * a.T + row / a.G) * a.H + h * a.G + row % a.G) * D + jd;
#pragma unroll
  for (int d = 0; d < DT; d += 4) {
    const uint32_t w0 = BF16 ? ActBF16::pack_rne(acc[d] * inv, acc[d + 1] * inv) : ActF16::pack_rne(acc[d] * inv, acc[d + 1] * inv);
    const uint32_t w1 = BF16 ? ActBF16::pack_rne(acc[d + 2] * inv, acc[d + 3] * inv) : ActF16::pack_rne(acc[d + 2] * inv, acc[d + 3] * inv);
    *reinterpret_cast<u32x2v_t*>(dst + d) = u32x2v_t{w0, w1};
  }
}

__device__ inline float scale_or_tiny(float s) { return fmaxf(s, kTinyScale) + (s - s); }  // a NaN or infinity gives NaN

// Workgroup (h, s * tiles + tile, b): kv head h, the 16 R (token, head) rows of a tile, part s of nsplit of its keys. For few
// rows, where reading the cache once is the bound: the four waves take alternate 64-key steps straight from memory into
// registers and share nothing until the end. A step's keys are loaded while the step before is worked on.
//
// Measured with 32 heads over 8 kv heads of 128: one token in 64 rows of up to 8192 keys 151 us a call, 5.2 TB/s; in 3 rows of
// 800000 keys 836 us, 5.8 TB/s; over 2048 keys 7 us, the latency of two steps a wave and the join through LDS. Five tokens in
// 16 rows of E4M3 80 us a call where one row of 16000 keys stands beside others of half, 3.8 TB/s; int8 74. E4M3 with R = 2 and
// heads of 128 spills 36 to 41 registers, which the NaNs' put-back below holds whether it runs or not. Cutting all rows' steps
// laid end to end into equal parts, so that the workgroups end together, took 74 us in the kernel where this order took 73.
template <int D, int R, bool E4M3, bool BF16>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void kv_attn_kernel(const KvAttnArgs a) {
  constexpr int KD = D / 64;  // 16-byte pieces of a key per lane
  constexpr int VD = D / 16;  // 16-dim tiles of the output
  const int h = blockIdx.x, b = blockIdx.z;
  const int rows = a.T * a.G;
  const int tiles = (rows + 16 * R - 1) / (16 * R);
  const int tile = blockIdx.y % tiles, split = blockIdx.y / tiles;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int g = lane >> 4, r = lane & 15;
  const int row0 = tile * 16 * R;
  KvSpan sp;
  if (!kv_span(a, b, row0, 16 * R, sp)) return;
  const int L = sp.keys;
  const int steps = (L + kStepKeys - 1) / kStepKeys;
  const int s0 = static_cast<int>(static_cast<int64_t>(steps) * split / a.nsplit);
  const int s1 = static_cast<int>(static_cast<int64_t>(steps) * (split + 1) / a.nsplit);

  const int64_t pstride = static_cast<int64_t>(a.Hkv) * a.block * D;
  const uint8_t* const kb = a.kc + static_cast<int64_t>(h) * a.block * D;
  const uint8_t* const vb = a.vc + static_cast<int64_t>(h) * a.block * D;
  const int* const trow = a.table + static_cast<int64_t>(b) * a.width;
  const int gk = (lane >> 2) & 3;  // the 16-key group of the lane's key rows; of its scores and values it is g
  auto page_of = [&](int key) { return trow[min(key, L - 1) >> a.shift]; };  // L >= 1 where this is called
  auto sane = [&](int p) { return p >= 0 && p < a.pages ? p : 0; };
  u32x4_t kr[4][KD], vr[VD];
  float ks = 0.0f, vs = 0.0f;
  auto load_k = [&](int k0, int pk, int pv) {
    const int slot = ((k0 + 16 * gk) & (a.block - 1)) + (lane & 3);
    const uint8_t* p = kb + sane(pk) * pstride + slot * D + 16 * g;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < KD; ++i) kr[t][i] = *reinterpret_cast<const u32x4_t*>(p + 4 * t * D + 64 * i);
    const int64_t at = static_cast<int64_t>(sane(pv)) * a.Hkv + h;
    ks = a.ks[at];
    vs = a.vs[at];
    if (pv < 0 || pv >= a.pages) ks = __builtin_nanf("");  // no such page: whoever attends it gets NaN
  };
  int step = s0 + wave;
  int pk = 0, pv = 0, pk2 = 0, pv2 = 0;
  if (step < s1) {
    pk = page_of(step * kStepKeys + 16 * gk);
    pv = page_of(step * kStepKeys + 16 * g);
    pk2 = page_of((step + kAttnWaves) * kStepKeys + 16 * gk);
    pv2 = page_of((step + kAttnWaves) * kStepKeys + 16 * g);
    load_k(step * kStepKeys, pk, pv);
  }

  u32x4_t qf[R][2 * KD];
  float qs[R];
  int pos[R];
  f32x4_t o[R][VD];
  float m[R], l[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int row = row0 + 16 * i + r;
    const int t = row / a.G;
    const bool ok = row < rows && t < sp.count;
    pos[i] = ok ? sp.position(t) : -1;
    qs[i] = load_query<KD, BF16>(a.q + b * a.q_sb + (ok ? t * a.q_st + (h * a.G + row % a.G) * a.q_sh : 0), ok, g, a.qscale, qf[i]);
    m[i] = -INFINITY;
    l[i] = 0.0f;
#pragma unroll
    for (int c = 0; c < VD; ++c) o[i][c] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  }

  auto work = [&](auto is_masked) __attribute__((always_inline)) {
    constexpr bool masked = decltype(is_masked)::value;
    const int k0 = step * kStepKeys;
    {
      const uint8_t* p = vb + sane(pv) * pstride + r * a.block + ((k0 + 16 * g) & (a.block - 1));
#pragma unroll
      for (int c = 0; c < VD; ++c) vr[c] = *reinterpret_cast<const u32x4_t*>(p + 16 * c * a.block);
    }
    f32x4_t sc[R][4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int i = 0; i < R; ++i) sc[i][t] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < KD; ++k) {
        const u32x4_t w = kr[t][k];
        const u32x4_t k0f = codes8<E4M3>(w[0], w[1]), k1f = codes8<E4M3>(w[2], w[3]);
#pragma unroll
        for (int i = 0; i < R; ++i) {
          sc[i][t] = ActF16::mfma(k0f, qf[i][2 * k], sc[i][t]);
          sc[i][t] = ActF16::mfma(k1f, qf[i][2 * k + 1], sc[i][t]);
        }
      }
    }
    const float kscale = scale_or_tiny(ks), vscale = scale_or_tiny(vs);
    const float lvs = __log2f(vscale), ivs = 1.0f / vscale;
    // the next step's keys, and the pages of the one after it
    pv = pv2;
    load_k(k0 + kAttnWaves * kStepKeys, pk2, pv2);
    pk2 = page_of(k0 + 2 * kAttnWaves * kStepKeys + 16 * gk);
    pv2 = page_of(k0 + 2 * kAttnWaves * kStepKeys + 16 * g);

    u32x4_t pf[R][2];
    int behind[R];
    float f[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      behind[i] = pos[i] + 1 - (k0 + 16 * g);
      f[i] = qs[i] * kscale;
    }
    softmax_step<R, VD, masked>(sc, behind, f, lvs, ivs, m, l, o, pf);
    // E4M3 values may be NaN where some row must not see them (a later token, a slot never written), and 0 NaN is NaN: in
    // masked steps NaN codes are taken out, and put back where a product of their indicator with that of the keys attended
    // is not zero (p itself may round to zero).
    if constexpr (E4M3 && masked) {
      {
        uint32_t bad = 0;
#pragma unroll
        for (int c = 0; c < VD; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t w = vr[c][e];
            bad |= nan_bytes(w);
          }
        if (__ballot(bad != 0) != 0) {  // wave-uniform
#pragma unroll
          for (int c = 0; c < VD; ++c) {
            u32x4_t one;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t w = vr[c][e], nb = nan_bytes(w) >> 7;
              one[e] = nb * 0x38u;  // 1.0
              vr[c][e] = w & ~(nb * 0xffu);
            }
#pragma unroll
            for (int i = 0; i < R; ++i) {
              u32x4_t am[2];
              attended(behind[i], am);
              f32x4_t hit{0.0f, 0.0f, 0.0f, 0.0f};
              hit = ActF16::mfma(codes8<true>(one[0], one[1]), am[0], hit);
              hit = ActF16::mfma(codes8<true>(one[2], one[3]), am[1], hit);
#pragma unroll
              for (int j = 0; j < 4; ++j)
                if (hit[j] > 0.0f) o[i][c][j] = __builtin_nanf("");
            }
          }
        }
      }
    }
#pragma unroll
    for (int c = 0; c < VD; ++c) {
      const u32x4_t w = vr[c];
      const u32x4_t v0 = codes8<E4M3>(w[0], w[1]), v1 = codes8<E4M3>(w[2], w[3]);
#pragma unroll
      for (int i = 0; i < R; ++i) {
        o[i][c] = ActF16::mfma(v0, pf[i][0], o[i][c]);
        o[i][c] = ActF16::mfma(v1, pf[i][1], o[i][c]);
      }
    }
  };
  // steps whose keys every row attends, then those that some row does not
  const int whole = min(max((sp.first + 1) / kStepKeys, 0), s1);
  for (; step < whole; step += kAttnWaves) work(std::false_type{});
  for (; step < s1; step += kAttnWaves) work(std::true_type{});

  // the waves' parts join through LDS, one 16-row tile at a time
  __shared__ float sm[kAttnWaves][16], sl[kAttnWaves][16];
  __shared__ __attribute__((aligned(16))) float so[kAttnWaves][16][D + 4];
  constexpr int DT = D / 16;  // dims per thread: 16 threads a row
  const int jr = threadIdx.x >> 4, jd = (threadIdx.x & 15) * DT;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    float ls = l[i];
    ls += __shfl_xor(ls, 16, 64);
    ls += __shfl_xor(ls, 32, 64);
    if (i > 0) __syncthreads();
    if (g == 0) {
      sm[wave][r] = m[i];
      sl[wave][r] = ls;
    }
#pragma unroll
    for (int c = 0; c < VD; ++c) *reinterpret_cast<f32x4_t*>(&so[wave][r][16 * c + 4 * g]) = o[i][c];
    __syncthreads();
    const int row = row0 + 16 * i + jr;
    if (row < rows && row / a.G < sp.count) {
      float M = sm[0][jr];
#pragma unroll
      for (int w = 1; w < kAttnWaves; ++w) M = fmaxf(M, sm[w][jr]);
      float sum = 0.0f, acc[DT];
#pragma unroll
      for (int d = 0; d < DT; ++d) acc[d] = 0.0f;
#pragma unroll
      for (int w = 0; w < kAttnWaves; ++w) {
        const float wt = attn_chunk_weight(sm[w][jr], M);
        sum = fmaf(sl[w][jr], wt, sum);
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[d] = fmaf(so[w][jr][jd + d], wt, acc[d]);
      }
      put_row<D, BF16, DT>(a, b, h, split, row, jd, M, sum, acc);
    }
  }
}

typedef float f32x16_t __attribute__((__vector_size__(16 * sizeof(float))));

__device__ inline f32x16_t mfma32(u32x4_t a, u32x4_t b, f32x16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}

// Orders a block of N operand reads from LDS with an MFMA each: kLead reads ahead of the first use, then one per MFMA. Left
// to itself the compiler waits for every read right before its use.
template <int N>
__device__ inline void reads_ahead() {
  constexpr int kLead = 4;
  __builtin_amdgcn_sched_group_barrier(0x100, kLead, 0);  // LDS reads
#pragma unroll
  for (int i = 0; i < N - kLead; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // MFMAs
    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
  }
  __builtin_amdgcn_sched_group_barrier(0x008, kLead, 0);
}

// f16 pairs with NaNs replaced by zero; `one` gets 1.0 in their place.
__device__ inline uint32_t drop_nan16(uint32_t w, uint32_t& one) {
  const uint32_t lo = (w & 0x7fffu) > 0x7c00u ? 0xffffu : 0u, hi = (w & 0x7fff0000u) > 0x7c000000u ? 0xffff0000u : 0u;
  one = (lo | hi) & 0x3c003c00u;
  return w & ~(lo | hi);
}

// softmax_step for 32 query rows and N tiles of 32 keys: lane (hi, r), hi = lane / 32, holds the scores of the 16 keys
// 32 t + 16 hi + e of row r in sc[t][e], attended below behind - 32 t. One m and l a lane.
template <int N, int VD, bool MASKED>
__device__ inline void softmax_step32(f32x16_t (&sc)[N], int behind, float qs, const float (&ks)[N], const float (&lvs)[N],
                                      const float (&ivs)[N], float& m, float& l, f32x16_t (&o)[VD], u32x4_t (&pf)[N][2]) {
  float mx = -INFINITY;
#pragma unroll
  for (int t = 0; t < N; ++t) {
    if constexpr (MASKED) {
#pragma unroll
      for (int e = 0; e < 16; ++e) sc[t][e] = 32 * t + e >= behind ? -INFINITY : sc[t][e];
    }
    float mi = sc[t][0];
#pragma unroll
    for (int e = 1; e < 16; ++e) mi = __builtin_elementwise_maximum(mi, sc[t][e]);
    mi = fmaf(mi, qs * ks[t], lvs[t]);
    if constexpr (MASKED) mi = behind <= 32 * t ? -INFINITY : mi;
    mx = __builtin_elementwise_maximum(mx, mi);
  }
  {
    const uint32_t u = __builtin_bit_cast(uint32_t, mx);
    const auto h = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t h0 = h[0], h1 = h[1];
    mx = __builtin_elementwise_maximum(__builtin_bit_cast(float, h0), __builtin_bit_cast(float, h1));
  }
  if (__ballot(mx > m + kPGrowth) != 0) {  // wave-uniform; also from -infinity
    const float mn = fmaxf(m, mx);         // not a NaN
    const float al = m == mn ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
    l *= al;
#pragma unroll
    for (int c = 0; c < VD; ++c)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[c][e] *= al;
    m = mn;
  }
#pragma unroll
  for (int t = 0; t < N; ++t) {
    const float f = qs * ks[t], base = lvs[t] - (m == -INFINITY ? 0.0f : m) + kPOffset;
    float p[16], sum = 0.0f;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      p[e] = __builtin_amdgcn_exp2f(fmaf(sc[t][e], f, base));
      if constexpr (MASKED) p[e] = 32 * t + e >= behind ? 0.0f : p[e];  // whatever its page's scales are
      sum += p[e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) pf[t][e >> 2][e & 3] = ActF16::pack_rne(p[2 * e], p[2 * e + 1]);
    if constexpr (MASKED) l = sum == 0.0f ? l : fmaf(sum, ivs[t], l);
    else l = fmaf(sum, ivs[t], l);
  }
}

// For many rows (prompts), where the matrix and vector units are the bound: workgroup (h, s * tiles + tile, b) takes 256
// rows, 32 in each of eight waves (heads of 256: 128 rows, four waves with twice the registers), and all waves work on
// the same keys. A 64-key piece of the cache is read once, turned to fp16 once (its conversion would cost a wave of its
// own two thirds of its softmax) and kept in LDS as the operands that the lanes want, so writes and reads are consecutive.
// Two tiles in LDS and one in registers: while a tile is worked on, the next is converted behind one barrier a tile and the
// one after it is on its way.
//
// The products are v_mfma_f32_32x32x16_f16, with the row order of the direct kernel carried over: row p of a 32-key tile is
// key 16 ((p / 4) % 2) + 4 (p / 8) + p % 4, so that lane (hi, r) gets the scores of 16 hi .. 16 hi + 15.
//
// 2 rows, 2048 tokens of 32 heads (8 kv heads) and up to 6000 keys: 247 us, 908 TFLOP/s (E4M3, whose forms all spill, 19 to 128
// registers: 259); 4 even rows of as many tokens run at 1005, a library product of 8192^3 in fp16 at 1101. Bound by the vector and the matrix unit together: on this card two waves
// of a SIMD overlap little of them (an MFMA of 16 cycles hides two vector instructions; 16x16x32 with four vector
// instructions and an exponential takes 33.7 ns for two waves where the parts take 16.3, 10.2 and 7.6, the 32x32x16 form
// 27.9). So vector instructions are what counts. Two groups of waves half a tile apart (one in its products while the other
// is in its softmax), and products and softmax of neighbouring tiles in one stream, took as long as this plain order (290
// and 298 us against 287, before the 32x32x16 form); turning the order of the second half of the workgroups, so that the
// shortest share a CU with the longest, 309 against 278 under the profiler; 128 rows in four waves 366 against 338.
//
// BIG: pages of 64 tokens or more, so a 64-key piece lies in one. Its page and scales are the same for all lanes and addresses
// are scalar; the per-lane form costs 70 vector instructions a tile, a fifth of all: 270 and 261 us with pages of 16 and 32
// tokens where 64 take 247.
constexpr int tile_waves(int d) { return d == 256 ? 4 : 8; }
constexpr int tile_rows(int d) { return 32 * tile_waves(d); }
template <int D, bool E4M3, bool BF16, bool BIG>
__global__ __launch_bounds__(64 * tile_waves(D), D == 256 ? 1 : 2) void kv_attn_tile_kernel(const KvAttnArgs a) {
  constexpr int kWaves = tile_waves(D), kTileRows = tile_rows(D);
  constexpr int KD = D / 32, VD = D / 32;        // 32-dim pieces of a key; of the output
  constexpr int NS = D == 64 ? 2 : 1;            // 64-key pieces of a tile
  constexpr int U = 2 * KD * NS / kWaves;        // 16-byte units of keys, and of values, per thread
  constexpr int kTileKeys = 64 * NS, NT = 2 * NS;  // 32-key tiles
  // operands of a tile: keys [32-key tile][i][2][lane], values [32-key tile][c][2][lane], 16 bytes each
  __shared__ u32x4_t lk[2][NT * KD * 2 * 64], lv[2][NT * VD * 2 * 64];
  __shared__ float lf[2][2 * NT], lg[2][2 * NT], li[2][2 * NT];  // per 16 keys: key scale, log2 and inverse of the value scale
  __shared__ int lnan[3];  // tile i holds a NaN value: slot i % 3, cleared while tile i - 2 is worked on
  const int h = blockIdx.x, b = blockIdx.z;
  const int rows = a.T * a.G;
  const int tiles = (rows + kTileRows - 1) / kTileRows;
  const int tile = tiles - 1 - blockIdx.y % tiles, split = blockIdx.y / tiles;  // the longest first
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hi = lane >> 5, r = lane & 31;
  const int row0 = tile * kTileRows;
  KvSpan sp;
  if (!kv_span(a, b, row0, kTileRows, sp)) return;
  const int L = sp.keys;
  const int steps = (L + kTileKeys - 1) / kTileKeys;
  const int s0 = static_cast<int>(static_cast<int64_t>(steps) * split / a.nsplit);
  const int s1 = static_cast<int>(static_cast<int64_t>(steps) * (split + 1) / a.nsplit);

  // loads: a thread's unit w is piece (t, i) of the keys and (t, c) of the values for its lane, t the 32-key tile
  const int64_t pstride = static_cast<int64_t>(a.Hkv) * a.block * D;
  const uint8_t* const kb = a.kc + static_cast<int64_t>(h) * a.block * D;
  const uint8_t* const vb = a.vc + static_cast<int64_t>(h) * a.block * D;
  const int* const trow = a.table + static_cast<int64_t>(b) * a.width;
  constexpr int kWavesPerTile = kWaves / NT;  // waves that load one 32-key tile
  const int lt = wave / kWavesPerTile, pw = wave % kWavesPerTile;
  const int gk = (r >> 2) & 1;  // the 16-key half of the lane's key row; of its scores and values it is hi
  auto sane = [&](int p) { return p >= 0 && p < a.pages ? p : 0; };
  // scalar loads: the table and the scales are constant while the kernel runs
  auto constant = [](const auto* p) { return (const __attribute__((address_space(4))) std::decay_t<decltype(*p)>*)(uintptr_t)p; };
  auto page_of = [&](int key) {
    if constexpr (BIG) return constant(trow)[min(key, L - 1) >> a.shift];
    else return trow[min(key, L - 1) >> a.shift];
  };
  u32x4_t kreg[U], vreg[U];
  float ks = 0.0f, vs = 0.0f;
  int pk = 0, pv = 0;
  const uint32_t klane = ((BIG ? 16 * gk : 0) + 4 * (r >> 3) + (r & 3)) * D + 16 * hi;
  const uint32_t vlane = r * a.block + (BIG ? 16 * hi : 0);
  auto load_pages = [&](int step) {
    const int k0 = step * kTileKeys + 32 * lt;
    pk = page_of(k0 + (BIG ? 0 : 16 * gk));
    pv = BIG ? pk : page_of(k0 + 16 * hi);
  };
  auto load_tile = [&](int step) {  // past the end: the last page again, not used
    const int k0 = step * kTileKeys + 32 * lt;
    const uint8_t* p = kb + sane(pk) * pstride + ((k0 + (BIG ? 0 : 16 * gk)) & (a.block - 1)) * D;
    const uint8_t* q = vb + sane(pv) * pstride + ((k0 + (BIG ? 0 : 16 * hi)) & (a.block - 1));
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int w = pw + kWavesPerTile * u;  // i of the keys, c of the values
      kreg[u] = *reinterpret_cast<const u32x4_t*>(p + 32 * w + klane);
      vreg[u] = *reinterpret_cast<const u32x4_t*>(q + 32 * w * a.block + vlane);
    }
    if (pw == 0) {
      const int64_t at = static_cast<int64_t>(sane(pv)) * a.Hkv + h;
      ks = BIG ? constant(a.ks)[at] : a.ks[at];
      vs = BIG ? constant(a.vs)[at] : a.vs[at];
      if (pv < 0 || pv >= a.pages) ks = __builtin_nanf("");
    }
  };
  auto store_tile = [&](int to) {
    const int buf = to & 1;
    [[maybe_unused]] const int slot = to % 3;
    uint32_t bad = 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int w = pw + kWavesPerTile * u;
      const u32x4_t k = kreg[u], v = vreg[u];
      u32x4_t* dk = &lk[buf][((lt * KD + w) * 2) * 64 + lane];
      u32x4_t* dv = &lv[buf][((lt * VD + w) * 2) * 64 + lane];
      dk[0] = codes8<E4M3>(k[0], k[1]);
      dk[64] = codes8<E4M3>(k[2], k[3]);
      dv[0] = codes8<E4M3>(v[0], v[1]);
      dv[64] = codes8<E4M3>(v[2], v[3]);
      if constexpr (E4M3) bad |= nan_bytes(v[0]) | nan_bytes(v[1]) | nan_bytes(v[2]) | nan_bytes(v[3]);
    }
    if (pw == 0 && r == 0) {
      const float vscale = scale_or_tiny(vs);
      lf[buf][2 * lt + hi] = scale_or_tiny(ks);
      lg[buf][2 * lt + hi] = __log2f(vscale);
      li[buf][2 * lt + hi] = 1.0f / vscale;
    }
    if constexpr (E4M3) {
      if (bad != 0) lnan[slot] = 1;
    }
  };

  if (s0 < s1) {
    load_pages(s0);
    load_tile(s0);
    load_pages(s0 + 1);
  }
  u32x4_t qf[2 * KD];
  const int wrow = row0 + 32 * wave, row = wrow + r, rt = row / a.G;
  const bool ok = row < rows && rt < sp.count;
  const int pos = ok ? sp.position(rt) : -1;
  const float qs = load_query32<KD, BF16>(a.q + b * a.q_sb + (ok ? rt * a.q_st + (h * a.G + row % a.G) * a.q_sh : 0), ok, hi, a.qscale, qf);
  float m = -INFINITY, l = 0.0f;
  f32x16_t o[VD];
#pragma unroll
  for (int c = 0; c < VD; ++c)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[c][e] = 0.0f;
  int last = -1;  // the wave's last position
  {
    const int end = min(min(wrow + 32, rows), sp.count * a.G);  // rows of the wave below the count
    if (end > wrow) last = sp.position((end - 1) / a.G);
  }
  const int first = sp.position(wrow / a.G);

  if (threadIdx.x < 3) lnan[threadIdx.x] = 0;
  __syncthreads();
  if (s0 < s1) {
    store_tile(s0);
    load_tile(s0 + 1);
    load_pages(s0 + 2);
  }
  auto work = [&](int step, auto masked) __attribute__((always_inline)) {
    constexpr bool M = decltype(masked)::value;
    const int buf = step & 1, k0 = step * kTileKeys;
    f32x16_t sc[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) sc[t][e] = 0.0f;
    const u32x4_t* const kt = &lk[buf][lane];
#pragma unroll
    for (int k = 0; k < 2 * KD; ++k)
#pragma unroll
      for (int t = 0; t < NT; ++t) sc[t] = mfma32(kt[(t * 2 * KD + k) * 64], qf[k], sc[t]);
    reads_ahead<2 * KD * NT>();
    float kscale[NT], lvs[NT], ivs[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      kscale[t] = lf[buf][2 * t + hi];
      lvs[t] = lg[buf][2 * t + hi];
      ivs[t] = li[buf][2 * t + hi];
    }
    u32x4_t pf[NT][2];
    const int behind = pos + 1 - (k0 + 16 * hi);
    softmax_step32<NT, VD, M>(sc, behind, qs, kscale, lvs, ivs, m, l, o, pf);
    const u32x4_t* const vt = &lv[buf][lane];
    if (E4M3 && M && lnan[step % 3] != 0) {  // as in the direct kernel
#pragma unroll
      for (int c = 0; c < VD; ++c)
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          u32x4_t one[2], w[2], am[2];
          attended(behind - 32 * t, am);
          f32x16_t hit;
#pragma unroll
          for (int e = 0; e < 16; ++e) hit[e] = 0.0f;
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            w[y] = vt[((t * VD + c) * 2 + y) * 64];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t q = w[y][e];
              uint32_t z;
              w[y][e] = drop_nan16(q, z);
              one[y][e] = z;
            }
            hit = mfma32(one[y], am[y], hit);
            o[c] = mfma32(w[y], pf[t][y], o[c]);
          }
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (hit[e] > 0.0f) o[c][e] = __builtin_nanf("");
        }
      return;
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int y = 0; y < 2; ++y)
#pragma unroll
        for (int c = 0; c < VD; ++c) o[c] = mfma32(vt[((t * VD + c) * 2 + y) * 64], pf[t][y], o[c]);
    reads_ahead<2 * VD * NT>();
  };
  // tile `step` is in LDS behind this, the other buffer is free and takes the next one
  auto next = [&](int step) __attribute__((always_inline)) {
    __syncthreads();
    if constexpr (E4M3) {
      if (threadIdx.x == 0) lnan[(step + 2) % 3] = 0;  // read by nobody since this barrier, set after the next
    }
    store_tile(step + 1);  // past the end: not used
    load_tile(step + 2);
    load_pages(step + 3);
  };
  // tiles that every row of the wave attends whole, tiles that some row does not, tiles past its last position
  const int whole = min(max((first + 1) / kTileKeys, s0), s1);
  const int some = max(whole, last < 0 ? s0 : min(max(last / kTileKeys + 1, s0), s1));
  int step = s0;
  for (; step < whole; ++step) {
    next(step);
    work(step, std::false_type{});
  }
  for (; step < some; ++step) {
    next(step);
    work(step, std::true_type{});
  }
  for (; step < s1; ++step) next(step);

  // each wave has its rows whole: lane (hi, r) holds dims 32 c + 8 e + 4 hi + j of row r
  float ls = l;
  ls += __shfl_xor(ls, 32, 64);
  if (ok) {
#pragma unroll
    for (int c = 0; c < VD; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float acc[4] = {o[c][4 * e], o[c][4 * e + 1], o[c][4 * e + 2], o[c][4 * e + 3]};
        put_row<D, BF16, 4>(a, b, h, split, row, 32 * c + 8 * e + 4 * hi, m, ls, acc);
      }
  }
}

// Joins the nsplit parts of every (token, head) row. Bound by the latency of its loads, so PG threads share a part's place of
// 16 bytes in the row: each takes every PG-th part, the first ones on their way while the maxima are compared. 96 rows of 21
// parts take 4.4 us (12.5 with a wave a row), 32 of 8 parts 2.7; up to 4 parts, PG = 2 and more rows a workgroup: 2560 rows
// of 4 parts 4.2 us, 5.5 with PG = 8 and 8 parts.
template <int D, bool BF16, int PG>
__global__ __launch_bounds__(256) void kv_attn_join_kernel(const KvAttnArgs a, int64_t total) {
  constexpr int C = D / 4, kRows = 256 / (PG * C), kAhead = 4;
  __shared__ float rm[kRows][PG], rl[kRows][PG];
  __shared__ f32x4_t ro[kRows][PG][C];
  const int rr = threadIdx.x / (PG * C), p = threadIdx.x / C % PG, c = threadIdx.x % C;
  const int64_t id = std::min<int64_t>(static_cast<int64_t>(blockIdx.x) * kRows + rr, total - 1);  // the last row again
  const int rows = a.T * a.G, n = a.nsplit;
  const int row = static_cast<int>(id % rows);
  const int64_t bh = id / rows;
  const int b = static_cast<int>(bh / a.Hkv), h = static_cast<int>(bh % a.Hkv);
  const int count = a.counts != nullptr ? min(max(a.counts[b], 0), a.T) : a.T;
  const bool live = row / a.G < count;  // no part has been written of the others
  const int mine = live ? n : 0;
  auto at = [&](int s) { return (bh * n + s) * rows + row; };
  f32x4_t x[kAhead];
  float m[kAhead], l[kAhead];
#pragma unroll
  for (int u = 0; u < kAhead; ++u) {
    x[u] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    m[u] = -INFINITY;
    l[u] = 0.0f;
    if (p + PG * u < mine) {
      x[u] = *reinterpret_cast<const f32x4_t*>(a.po + at(p + PG * u) * D + 4 * c);
      m[u] = a.pml[2 * at(p + PG * u)];
      l[u] = a.pml[2 * at(p + PG * u) + 1];
    }
  }
  float M = -INFINITY;
#pragma unroll
  for (int u = 0; u < kAhead; ++u) M = fmaxf(M, m[u]);
  for (int s = p + PG * kAhead; s < mine; s += PG) M = fmaxf(M, a.pml[2 * at(s)]);
  if (c == 0) rm[rr][p] = M;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PG; ++i) M = fmaxf(M, rm[rr][i]);
  float sum = 0.0f;
  f32x4_t acc{0.0f, 0.0f, 0.0f, 0.0f};
  auto add = [&](float ms, float ls, f32x4_t v) {
    const float wt = attn_chunk_weight(ms, M);
    sum = fmaf(ls, wt, sum);
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = fmaf(v[e], wt, acc[e]);
  };
#pragma unroll
  for (int u = 0; u < kAhead; ++u)
    if (p + PG * u < mine) add(m[u], l[u], x[u]);
#pragma unroll 4
  for (int s = p + PG * kAhead; s < mine; s += PG)
    add(a.pml[2 * at(s)], a.pml[2 * at(s) + 1], *reinterpret_cast<const f32x4_t*>(a.po + at(s) * D + 4 * c));
  ro[rr][p][c] = acc;
  if (c == 0) rl[rr][p] = sum;
  __syncthreads();
  if (p != 0 || !live || static_cast<int64_t>(blockIdx.x) * kRows + rr >= total) return;
  sum = 0.0f;
  acc = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < PG; ++i) {
    sum += rl[rr][i];
    const f32x4_t v = ro[rr][i][c];
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] += v[e];
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  uint16_t* dst = a.out + ((static_cast<int64_t>(b) * a.T + row / a.G) * a.H + h * a.G + row % a.G) * D + 4 * c;
  const float o0 = acc[0] * inv, o1 = acc[1] * inv, o2 = acc[2] * inv, o3 = acc[3] * inv;
  *reinterpret_cast<u32x2v_t*>(dst) = BF16 ? u32x2v_t{ActBF16::pack_rne(o0, o1), ActBF16::pack_rne(o2, o3)}
                                           : u32x2v_t{ActF16::pack_rne(o0, o1), ActF16::pack_rne(o2, o3)};
}

// How a call is laid out: 16-row tiles of a workgroup of the direct kernel (0: the tile kernel), tiles of rows, and
// the parts that its keys are cut into. The host knows the table's width, not what the rows hold: one token over 2048 keys
// takes 9.6 us behind a table of 2048 tokens and 11.5 behind one of 32768 to 524288, 16 rows of it 22.5 behind any.
struct KvAttnPlan {
  int R, tiles, splits;
};
inline KvAttnPlan kv_attn_plan(int64_t B, int64_t rows, int64_t Hkv, int64_t hd, int64_t keys) {
  KvAttnPlan p;
  const int64_t steps = ceil_div(keys, kStepKeys);
  // The direct kernel reads the cache once for every 16 R rows, the tile kernel for every 256 (128 with heads of 256) and keeps
  // its matrix unit busier. us, direct (R = 2) and tile, heads of 128, 8 kv heads, int8, in 8 rows of 16000 keys and 1 of 2000:
  //   64 rows 65, 127 and 12, 17; 128 rows 112, 136 and 14, 19; 192 rows 185, 151 and 19, 21
  // heads of 256, direct (R = 1) and tile: 64 rows 199, 203 and 16, 26; 68 rows 354, 204 and 24, 26.
  // With R = 2 it needs registers that heads of 256 do not have (E4M3, 36 rows: 232 against 195, 20 against 14); smaller heads
  // are better off with R = 1 while a call has at most 4096 steps, two for each of 512 x 4 waves, R = 2 and R = 1:
  //   1 row of 2000 keys: 20 rows 11.4, 9.5, 64 rows 12.4, 10.4; of 16000 keys: 32 rows 20.1, 17.8, 64 rows 21.1, 22.7
  //   8 rows of 16000 keys: 20 rows 51, 57, 36 rows 61, 99
  const bool one = hd == 256 || rows <= 16 || (rows <= 64 && B * Hkv * ceil_div(rows, 16) * steps <= 4096);
  p.R = rows > (hd == 256 ? 64 : 128) ? 0 : one ? 1 : 2;
  const int64_t span = p.R == 0 ? tile_rows(static_cast<int>(hd)) : 16 * p.R;
  p.tiles = static_cast<int>(std::min<int64_t>(ceil_div(rows, span), 1 << 30));
  const int64_t groups = B * Hkv * p.tiles;
  // Two workgroups of the direct kernel a CU (twice as many: 28 -> 39 us for 2 rows of 60000 keys and 16 heads over one), one
  // of the tile kernel (two: 30 -> 43 us for 128 rows over 16000 keys); no further round for a few.
  const int64_t want = std::max<int64_t>(1, (p.R == 0 ? 256 : 512) / groups);
  p.splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(want, ceil_div(steps, kAttnWaves))));
  return p;
}

}  // namespace sqx

using namespace sqx;

extern "C" int64_t sqx_kvblock_attention_workspace_bytes(int64_t B, int64_t T, int64_t H, int64_t Hkv, int64_t hd,
                                                         int64_t block, int64_t width) {
  if (B <= 0 || T <= 0 || Hkv <= 0 || H <= 0 || H % Hkv != 0 || !(hd == 64 || hd == 128 || hd == 256) ||
      !kv_block_ok(block) || width <= 0)
    return 0;
  const int64_t rows = T * (H / Hkv);
  const int ns = kv_attn_plan(B, rows, Hkv, hd, width * block).splits;
  return ns == 1 ? 0 : B * Hkv * ns * rows * (hd + 2) * 4;
}

extern "C" int sqx_kvblock_attention(const void* q, int dtype, int64_t q_sb, int64_t q_st, int64_t q_sh, int fmt,
                                     const void* k_codes, const void* v_codes, const float* k_scale,
                                     const float* v_scale, const int* table, const int* starts, const int* counts,
                                     int64_t B, int64_t T, int64_t H, int64_t Hkv, int64_t hd, int64_t block,
                                     int64_t pages, int64_t width, float scale, void* out, void* ws, int64_t ws_bytes,
                                     sqx_stream_t stream) {
  const char* fn = "sqx_kvblock_attention";
  KV_SHAPE(fn);
  SQX_REQUIRE(dtype != SQX_DTYPE_F32, SQX_E_ARG, "%s: queries must be BF16 or F16", fn);
  SQX_REQUIRE(H >= 1 && H % Hkv == 0 && H <= 8192, SQX_E_ARG, "%s: H=%lld must be a multiple of Hkv=%lld, up to 8192", fn,
              (long long)H, (long long)Hkv);
  SQX_REQUIRE(scale > 0.0f && scale <= 1.0e30f, SQX_E_ARG, "%s: scale must be positive and at most 1e30", fn);
  SQX_REQUIRE(q_sb >= 0 && q_st >= 0 && q_sh >= 0 && (q_sb | q_st | q_sh) % 8 == 0, SQX_E_ARG,
              "%s: strides must be multiples of 8 elements", fn);
  if (B == 0 || T == 0) return SQX_OK;
  SQX_REQUIRE(q && k_codes && v_codes && k_scale && v_scale && table && starts && out, SQX_E_ARG, "%s: null pointer", fn);
  SQX_REQUIRE(al16(q) && al16(k_codes) && al16(v_codes) && al16(out), SQX_E_ARG,
              "%s: q, codes and out must be 16-byte aligned", fn);
  const int64_t G = H / Hkv, rows = T * G;
  SQX_REQUIRE(rows < (int64_t(1) << 28), SQX_E_ARG, "%s: %lld tokens of %lld heads per kv head", fn, (long long)T, (long long)G);
  const KvAttnPlan plan = kv_attn_plan(B, rows, Hkv, hd, width * block);
  const int64_t tiles = plan.tiles;
  const int ns = plan.splits;
  const int64_t need = sqx_kvblock_attention_workspace_bytes(B, T, H, Hkv, hd, block, width);
  SQX_REQUIRE(need == 0 || (ws != nullptr && ws_bytes >= need && al16(ws)), SQX_E_SPACE,
              "%s: %lld bytes of 16-byte aligned workspace needed, %lld given", fn, (long long)need, (long long)ws_bytes);
  SQX_REQUIRE(tiles * ns < 65536, SQX_E_ARG, "%s: T=%lld tokens are too many for one call", fn, (long long)T);
  KvAttnArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.q_sb = q_sb; a.q_st = q_st; a.q_sh = q_sh;
  a.kc = static_cast<const uint8_t*>(k_codes); a.vc = static_cast<const uint8_t*>(v_codes);
  a.ks = k_scale; a.vs = v_scale;
  a.table = table; a.starts = starts; a.counts = counts;
  a.out = static_cast<uint16_t*>(out);
  a.po = static_cast<float*>(ws);
  a.pml = ns > 1 ? a.po + B * Hkv * ns * rows * hd : nullptr;
  a.T = static_cast<int>(T); a.H = static_cast<int>(H); a.Hkv = static_cast<int>(Hkv); a.G = static_cast<int>(G);
  a.width = static_cast<int>(width); a.pages = static_cast<int>(pages); a.block = static_cast<int>(block);
  a.shift = kv_shift(block); a.nsplit = ns;
  a.qscale = static_cast<float>(static_cast<double>(scale) * 1.4426950408889634);
  const dim3 grid(static_cast<unsigned>(Hkv), static_cast<unsigned>(tiles * ns), static_cast<unsigned>(B));
  const hipStream_t s = as_stream(stream);
  with_head(hd, [&](auto dd) {
    constexpr int D = decltype(dd)::value;
    auto go = [&](auto e4, auto bf) {
      constexpr bool E = decltype(e4)::value, BF = decltype(bf)::value;
      if (plan.R == 1) hipLaunchKernelGGL((kv_attn_kernel<D, 1, E, BF>), grid, dim3(256), 0, s, a);
      else if (plan.R == 2) {
        if constexpr (D < 256) hipLaunchKernelGGL((kv_attn_kernel<D, 2, E, BF>), grid, dim3(256), 0, s, a);
      } else if (block >= kStepKeys) hipLaunchKernelGGL((kv_attn_tile_kernel<D, E, BF, true>), grid, dim3(64 * tile_waves(D)), 0, s, a);
      else hipLaunchKernelGGL((kv_attn_tile_kernel<D, E, BF, false>), grid, dim3(64 * tile_waves(D)), 0, s, a);
    };
    auto with_type = [&](auto e4) {
      if (dtype == SQX_DTYPE_BF16) go(e4, std::true_type{});
      else go(e4, std::false_type{});
    };
    if (fmt == SQX_KV_E4M3) with_type(std::true_type{});
    else with_type(std::false_type{});
  });
  SQX_LAUNCH_CHECK(fn);
  if (ns > 1) {
    const int64_t total = B * Hkv * rows;
    with_head(hd, [&](auto dd) {
      constexpr int D = decltype(dd)::value;
      auto go = [&](auto bf, auto pg) {
        constexpr int PG = decltype(pg)::value;
        const dim3 jg(static_cast<unsigned>(ceil_div(total, 1024 / (PG * D))));
        hipLaunchKernelGGL((kv_attn_join_kernel<D, decltype(bf)::value, PG>), jg, dim3(256), 0, s, a, total);
      };
      auto with_parts = [&](auto bf) {
        if (ns > 4) go(bf, std::integral_constant<int, D == 256 ? 4 : 8>{});
        else go(bf, std::integral_constant<int, 2>{});
      };
      if (dtype == SQX_DTYPE_BF16) with_parts(std::true_type{});
      else with_parts(std::false_type{});
    });
    SQX_LAUNCH_CHECK(fn);
  }
  return SQX_OK;
}
