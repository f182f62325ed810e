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
//    product, u = x (ks scale log2 e) + log2 vs; the running maximum is that of u, p = 2^(u - max + 15), O sums p c and
//    the softmax's denominator sums p / vs. Probabilities thus carry their value scale, and the largest term of the
//    output is near 2^15 whatever the scales: fp16 keeps 11 bits of every p down to 2^-29 of it. Sums, maxima and the
//    denominator are fp32.
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

typedef _Float16 f16x4_t __attribute__((__vector_size__(4 * sizeof(_Float16))));

constexpr int kStepKeys = 64;
constexpr int kAttnWaves = 4;
constexpr float kPOffset = 15.0f;     // p reaches 2^15
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

// Workgroup (h, s * tiles + tile, b): kv head h, the 16 R (token, head) rows of a tile, part s of nsplit of its keys.
// The four waves take alternate 64-key steps.
template <int D, int R, bool E4M3, bool BF16>
__global__ __launch_bounds__(256) void kv_attn_kernel(const KvAttnArgs a) {
  constexpr int KD = D / 64;  // 16-byte pieces of a key per lane
  constexpr int VD = D / 16;  // 16-dim tiles of the output
  const int h = blockIdx.x, b = blockIdx.z;
  const int rows = a.T * a.G;
  const int tiles = (rows + 16 * R - 1) / (16 * R);
  const int tile = blockIdx.y % tiles, split = blockIdx.y / tiles;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int g = lane >> 4, r = lane & 15;
  const int count = a.counts != nullptr ? min(max(a.counts[b], 0), a.T) : a.T;
  const int row0 = tile * 16 * R;
  if (row0 / a.G >= count) return;  // rows from the count on are left as they are
  const int start = a.starts[b];
  const int last = min((row0 + 16 * R - 1) / a.G, count - 1);  // last token of the tile
  // keys below L are attended by some row of the tile; keys up to `first` by every row
  const int64_t end = static_cast<int64_t>(start) + last + 1;
  const int L = static_cast<int>(end < 0 ? 0 : (end < static_cast<int64_t>(a.width) * a.block ? end : static_cast<int64_t>(a.width) * a.block));
  const int first = start + row0 / a.G;
  const int steps = (L + kStepKeys - 1) / kStepKeys;
  const int s0 = static_cast<int>(static_cast<int64_t>(steps) * split / a.nsplit);
  const int s1 = static_cast<int>(static_cast<int64_t>(steps) * (split + 1) / a.nsplit);

  // queries: dims 64 i + 16 g + 8 half .. of row r, scaled by a power of two
  u32x4_t qf[R][2 * KD];
  float qs[R];
  int pos[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int row = row0 + 16 * i + r;
    const int t = row / a.G;
    const bool ok = row < rows && t < count;
    pos[i] = ok ? start + t : -1;
    const uint16_t* src = a.q + b * a.q_sb + (ok ? t * a.q_st + (h * a.G + row % a.G) * a.q_sh : 0);
#pragma unroll
    for (int k = 0; k < 2 * KD; ++k) {
      qf[i][k] = u32x4_t{0u, 0u, 0u, 0u};
      if (ok) qf[i][k] = *reinterpret_cast<const u32x4_t*>(src + 64 * (k >> 1) + 16 * g + 8 * (k & 1));
    }
    qs[i] = a.qscale;
    if constexpr (BF16) {
      float most = 0.0f;
#pragma unroll
      for (int k = 0; k < 2 * KD; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t w = qf[i][k][e];
          most = fmaxf(most, fmaxf(fabsf(bf16_lo(w)), fabsf(bf16_hi(w))));
        }
      most = fmaxf(most, __shfl_xor(most, 16, 64));
      most = fmaxf(most, __shfl_xor(most, 32, 64));
      int e = 0;
      if (most > 0.0f && most <= 3.402823466e38f) {
        frexpf(most, &e);
        e = max(e, -100);
      }
      const float up = most > 0.0f && most <= 3.402823466e38f ? ldexpf(1.0f, 15 - e) : 1.0f;
      qs[i] = a.qscale * (1.0f / up);
#pragma unroll
      for (int k = 0; k < 2 * KD; ++k)
#pragma unroll
        for (int e2 = 0; e2 < 4; ++e2) {
          const uint32_t w = qf[i][k][e2];
          qf[i][k][e2] = ActF16::pack_rne(bf16_lo(w) * up, bf16_hi(w) * up);
        }
    }
  }

  f32x4_t o[R][VD];
  float m[R], l[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.0f;
#pragma unroll
    for (int c = 0; c < VD; ++c) o[i][c] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  }

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
    const int64_t sp = static_cast<int64_t>(sane(pv)) * a.Hkv + h;
    ks = a.ks[sp];
    vs = a.vs[sp];
    if (pv < 0 || pv >= a.pages) ks = __builtin_nanf("");  // no such page: whoever attends it gets NaN
  };

  int step = s0 + wave;
  if (step < s1) {
    int pk = page_of(step * kStepKeys + 16 * gk), pv = page_of(step * kStepKeys + 16 * g);
    load_k(step * kStepKeys, pk, pv);
    int pk2 = page_of((step + kAttnWaves) * kStepKeys + 16 * gk), pv2 = page_of((step + kAttnWaves) * kStepKeys + 16 * g);
    for (; step < s1; step += kAttnWaves) {
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
      const float kscale = fmaxf(ks, kTinyScale) + (ks - ks);  // a NaN stays one
      const float vscale = fmaxf(vs, kTinyScale) + (vs - vs);
      const float lvs = __log2f(vscale), ivs = 1.0f / vscale;
      // the next step's keys, and the pages of the one after it
      pv = pv2;
      load_k(k0 + kAttnWaves * kStepKeys, pk2, pv2);
      pk2 = page_of(k0 + 2 * kAttnWaves * kStepKeys + 16 * gk);
      pv2 = page_of(k0 + 2 * kAttnWaves * kStepKeys + 16 * g);

      const bool masked = k0 + kStepKeys - 1 > first;  // wave-uniform
      u32x4_t pf[R][2];
#pragma unroll
      for (int i = 0; i < R; ++i) {
        if (masked) {
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (k0 + 16 * g + 4 * t + j > pos[i]) sc[i][t][j] = -INFINITY;
        }
        const float f = qs[i] * kscale;
        float mx = sc[i][0][0];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j) mx = fmaxf(mx, sc[i][t][j]);
        mx = fmaf(mx, f, lvs);  // f > 0: the maximum of u
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float mn = fmaxf(m[i], mx);
        if (__ballot(mn > m[i]) != 0) {  // wave-uniform
          const float al = m[i] == mn ? 1.0f : __builtin_amdgcn_exp2f(m[i] - mn);
          l[i] *= al;
#pragma unroll
          for (int c = 0; c < VD; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[i][c][j] *= al;
          m[i] = mn;
        }
        const float base = lvs - (mn == -INFINITY ? 0.0f : mn) + kPOffset;
        float p[16], sum = 0.0f;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            p[4 * t + j] = __builtin_amdgcn_exp2f(fmaf(sc[i][t][j], f, base));
            if (masked) p[4 * t + j] = sc[i][t][j] == -INFINITY ? 0.0f : p[4 * t + j];  // whatever its page's scales are
            sum += p[4 * t + j];
          }
        l[i] = sum == 0.0f ? l[i] : fmaf(sum, ivs, l[i]);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          pf[i][t >> 1][2 * (t & 1)] = ActF16::pack_rne(p[4 * t], p[4 * t + 1]);
          pf[i][t >> 1][2 * (t & 1) + 1] = ActF16::pack_rne(p[4 * t + 2], p[4 * t + 3]);
        }
      }
      // E4M3 values may be NaN where some row must not see them (a later token, a slot never written), and 0 NaN is
      // NaN: in masked steps NaN codes are taken out and put back through a product of their indicator.
      bool any_nan = false;
      if constexpr (E4M3) {
        if (masked) {
          uint32_t bad = 0;
#pragma unroll
          for (int c = 0; c < VD; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t w = vr[c][e];
              bad |= nan_bytes(w);
            }
          any_nan = __ballot(bad != 0) != 0;
        }
      }
#pragma unroll
      for (int c = 0; c < VD; ++c) {
        u32x4_t w = vr[c];
        if constexpr (E4M3) {
          if (any_nan) {  // wave-uniform
            u32x4_t one;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t x = w[e], nb = nan_bytes(x);
              one[e] = (nb >> 7) * 0x38u;  // 1.0
              w[e] = x & ~((nb >> 7) * 0xffu);
            }
#pragma unroll
            for (int i = 0; i < R; ++i) {
              f32x4_t hit{0.0f, 0.0f, 0.0f, 0.0f};
              hit = ActF16::mfma(codes8<true>(one[0], one[1]), pf[i][0], hit);
              hit = ActF16::mfma(codes8<true>(one[2], one[3]), pf[i][1], hit);
#pragma unroll
              for (int j = 0; j < 4; ++j)
                if (hit[j] > 0.0f) o[i][c][j] = __builtin_nanf("");
            }
          }
        }
        const u32x4_t v0 = codes8<E4M3>(w[0], w[1]), v1 = codes8<E4M3>(w[2], w[3]);
#pragma unroll
        for (int i = 0; i < R; ++i) {
          o[i][c] = ActF16::mfma(v0, pf[i][0], o[i][c]);
          o[i][c] = ActF16::mfma(v1, pf[i][1], o[i][c]);
        }
      }
    }
  }

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
    const int t = row / a.G;
    if (row < rows && t < count) {
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
      if (a.nsplit > 1) {
        const int64_t at = ((static_cast<int64_t>(b) * a.Hkv + h) * a.nsplit + split) * rows + row;
        if (jd == 0) {
          a.pml[2 * at] = M;
          a.pml[2 * at + 1] = sum;
        }
#pragma unroll
        for (int d = 0; d < DT; d += 4)
          *reinterpret_cast<f32x4_t*>(a.po + at * D + jd + d) = f32x4_t{acc[d], acc[d + 1], acc[d + 2], acc[d + 3]};
      } else {
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;  // no key: zeros
        uint32_t w[DT / 2];
#pragma unroll
        for (int d = 0; d < DT; d += 2)
          w[d / 2] = BF16 ? ActBF16::pack_rne(acc[d] * inv, acc[d + 1] * inv) : ActF16::pack_rne(acc[d] * inv, acc[d + 1] * inv);
        uint16_t* dst = a.out + ((static_cast<int64_t>(b) * a.T + t) * a.H + h * a.G + row % a.G) * D + jd;
#pragma unroll
        for (int d = 0; d < DT / 2; d += 2) *reinterpret_cast<u32x2v_t*>(dst + 2 * d) = u32x2v_t{w[d], w[d + 1]};
      }
    }
  }
}

// Joins the nsplit parts of every (token, head) row: one wave per row.
template <int D, bool BF16>
__global__ __launch_bounds__(256) void kv_attn_join_kernel(const KvAttnArgs a, int64_t total) {
  constexpr int E = D / 64;
  const int64_t id = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (id >= total) return;
  const int lane = threadIdx.x & 63;
  const int rows = a.T * a.G;
  const int row = static_cast<int>(id % rows);
  const int64_t bh = id / rows;
  const int b = static_cast<int>(bh / a.Hkv), h = static_cast<int>(bh % a.Hkv);
  const int t = row / a.G;
  const int count = a.counts != nullptr ? min(max(a.counts[b], 0), a.T) : a.T;
  if (t >= count) return;
  float M = -INFINITY;
  for (int s = 0; s < a.nsplit; ++s) M = fmaxf(M, a.pml[2 * ((bh * a.nsplit + s) * rows + row)]);
  float sum = 0.0f, acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.0f;
  for (int s = 0; s < a.nsplit; ++s) {
    const int64_t at = (bh * a.nsplit + s) * rows + row;
    const float wt = attn_chunk_weight(a.pml[2 * at], M);
    sum = fmaf(a.pml[2 * at + 1], wt, sum);
    const float* src = a.po + at * D + E * lane;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = fmaf(src[e], wt, acc[e]);
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  uint16_t* dst = a.out + ((static_cast<int64_t>(b) * a.T + t) * a.H + h * a.G + row % a.G) * D + E * lane;
#pragma unroll
  for (int e = 0; e < E; ++e) dst[e] = BF16 ? f32_to_bf16_bits(acc[e] * inv) : f32_to_f16_bits(acc[e] * inv);
}

// 16-row tiles of a workgroup, and the parts that its keys are cut into.
inline int kv_attn_tiles(int64_t rows, int64_t hd) { return rows <= 16 ? 1 : (rows <= 32 || hd == 256) ? 2 : 4; }
inline int kv_attn_splits(int64_t B, int64_t rows, int64_t Hkv, int64_t hd, int64_t keys) {
  const int64_t groups = B * Hkv * ceil_div(rows, 16 * kv_attn_tiles(rows, hd));
  const int64_t steps = ceil_div(keys, kStepKeys);
  const int64_t want = ceil_div(512, groups);
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({want, ceil_div(steps, kAttnWaves), 64})));
}

}  // namespace sqx

using namespace sqx;

extern "C" int64_t sqx_kvblock_attention_workspace_bytes(int64_t B, int64_t T, int64_t H, int64_t Hkv, int64_t hd,
                                                         int64_t block, int64_t width) {
  if (B <= 0 || T <= 0 || Hkv <= 0 || H <= 0 || H % Hkv != 0 || !(hd == 64 || hd == 128 || hd == 256) ||
      !kv_block_ok(block) || width <= 0)
    return 0;
  const int64_t rows = T * (H / Hkv);
  const int ns = kv_attn_splits(B, rows, Hkv, hd, width * block);
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
  SQX_REQUIRE(scale > 0.0f && scale <= 3.0e38f, SQX_E_ARG, "%s: scale must be positive and finite", fn);
  SQX_REQUIRE(q_sb >= 0 && q_st >= 0 && q_sh >= 0 && (q_sb | q_st | q_sh) % 8 == 0, SQX_E_ARG,
              "%s: strides must be multiples of 8 elements", fn);
  if (B == 0 || T == 0) return SQX_OK;
  SQX_REQUIRE(q && k_codes && v_codes && k_scale && v_scale && table && starts && out, SQX_E_ARG, "%s: null pointer", fn);
  SQX_REQUIRE(al16(q) && al16(k_codes) && al16(v_codes) && al16(out), SQX_E_ARG,
              "%s: q, codes and out must be 16-byte aligned", fn);
  const int64_t G = H / Hkv, rows = T * G;
  SQX_REQUIRE(rows < (int64_t(1) << 28), SQX_E_ARG, "%s: %lld tokens of %lld heads per kv head", fn, (long long)T, (long long)G);
  const int R = kv_attn_tiles(rows, hd);
  const int64_t tiles = ceil_div(rows, 16 * R);
  const int ns = kv_attn_splits(B, rows, Hkv, hd, width * block);
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
  auto go = [&](auto dd, auto rr) {
    constexpr int D = decltype(dd)::value, RR = decltype(rr)::value;
    const bool bf = dtype == SQX_DTYPE_BF16;
    if (fmt == SQX_KV_E4M3) {
      if (bf) hipLaunchKernelGGL((kv_attn_kernel<D, RR, true, true>), grid, dim3(256), 0, s, a);
      else hipLaunchKernelGGL((kv_attn_kernel<D, RR, true, false>), grid, dim3(256), 0, s, a);
    } else {
      if (bf) hipLaunchKernelGGL((kv_attn_kernel<D, RR, false, true>), grid, dim3(256), 0, s, a);
      else hipLaunchKernelGGL((kv_attn_kernel<D, RR, false, false>), grid, dim3(256), 0, s, a);
    }
  };
  with_head(hd, [&](auto dd) {
    if (R == 1) go(dd, std::integral_constant<int, 1>{});
    else if (R == 2) go(dd, std::integral_constant<int, 2>{});
    else if constexpr (decltype(dd)::value != 256) go(dd, std::integral_constant<int, 4>{});
  });
  SQX_LAUNCH_CHECK(fn);
  if (ns > 1) {
    const int64_t total = B * Hkv * rows;
    const dim3 jg(static_cast<unsigned>(ceil_div(total, 4)));
    with_head(hd, [&](auto dd) {
      constexpr int D = decltype(dd)::value;
      if (dtype == SQX_DTYPE_BF16) hipLaunchKernelGGL((kv_attn_join_kernel<D, true>), jg, dim3(256), 0, s, a, total);
      else hipLaunchKernelGGL((kv_attn_join_kernel<D, false>), jg, dim3(256), 0, s, a, total);
    });
    SQX_LAUNCH_CHECK(fn);
  }
  return SQX_OK;
}
