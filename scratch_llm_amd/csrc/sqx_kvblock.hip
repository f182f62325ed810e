// The block-scaled 8-bit KV cache: writing new tokens (quantized as they are written, rotary positions included) and
// reading values back. Layout and code formats: sqx_kvblock.h.
//
// A block's scale. A block whose first token is part of the write takes s = max(a, 1e-12), a = fl(amax fl(1 / qmax)) over the
// tokens written, qmax 127 or 448. A block that already holds tokens keeps its scale, doubled k times, the least k with
// a <= s 2^k, and its codes become rne(c 2^-k). With growth in powers of two every later rescale at least
// doubles the step, so what the rescales add to a token's error is at most s/2 (1 + 1/2 + 1/4 + ...) < s of the final
// scale, however often the block grows; growing to each token's own amax would add s/2 at every token.
// amax is taken over finite magnitudes: infinities saturate to the largest code, a NaN is a NaN in E4M3 and 0 in int8.
#include "sqx_kvblock.h"

namespace sqx {

struct KvWriteArgs {
  const void *k, *v, *q;  // q: NULL where none is rotated
  void* q_out;
  int64_t k_sb, k_st, k_sh, v_sb, v_st, v_sh, q_sb, q_st, q_sh;  // strides in elements: row, token, head
  uint8_t *kc, *vc;
  float *ks, *vs;
  const int *table, *starts, *counts;  // counts: NULL means T everywhere
  const float *cos_t, *sin_t;          // NULL: nothing is rotated
  int rope_rows, rot, inter;
  int T, H, Hkv, width, pages, block, shift;
};

constexpr int kQHeads = 4;  // query heads per workgroup of the rotary part, all taken by a thread at once

// The rotation of the rows x[0 .. NP) of one 8-column group. In halves the other half of a pair lies in the lane half8
// further on or back, of the same token.
template <int DT>
__device__ inline void rotate_lane(Row8<DT>& x, int c, int rot, bool inter, const Angles8& g) {
  if (inter) {
    if (8 * c < rot) rotate_pairs<DT>(x, g);
    return;
  }
  const int half8 = rot / 16, lane = threadIdx.x & 63;
  const bool second = c >= half8;
  const int from = 8 * c < rot ? (second ? lane - half8 : lane + half8) : lane;
  Row8<DT> o;
#pragma unroll
  for (int i = 0; i < Row8<DT>::kWords; ++i) o.w[i] = __shfl(static_cast<int>(x.w[i]), from, 64);
  if (8 * c >= rot) return;
  if (second) {
    rotate_halves<DT>(o, x, g);
  } else {
    rotate_halves<DT>(x, o, g);
  }
}

// Workgroup (j, y, b): block j of the blocks that row b's tokens touch. y < Hkv: the keys of head y; then the values;
// then groups of kQHeads query heads, whose rotation needs no block. A block's scale needs all of its new tokens before the
// first code, so a workgroup holds a block of one head in registers and reads it once.
//
// Bound by HBM for prompts: 12977 tokens in 8 rows, 32 query and 8 kv heads of 128, bf16 to int8: 80 us, 3.7 TB/s (the least of
// 27 passes 70, of the form with eight heads a workgroup 81). Two thirds of that are queries, which need no block: their
// four rounds of load, rotate and store wait for one another. One token in each of 8 rows takes 5.8 us: a launch and a
// chain of table, scale and old codes, behind which the rows and angles are loaded.
//
// A thread holds 8 columns of NP tokens: of a whole block, tokens NP tl .. NP tl + NP - 1, so that four codes of a value
// column are one dword of the transposed tile; of at most 256 / C tokens (NP = 1), token tl of the write. Slots outside
// the write read its nearest token, so that all loads are issued together, and are not stored.
template <int DT, int D, bool E4M3, int NP>
__global__ __launch_bounds__(256) void kv_write_kernel(const KvWriteArgs a) {
  using Code = KvCode<E4M3>;
  constexpr int C = D / 8;                            // 8-column groups of a token
  constexpr int TP = 256 / C;                         // tokens held by the workgroup, per NP
  constexpr int kPitch = (NP == 1 ? 128 : NP * TP) + 16;  // LDS pitch of a value column
  __shared__ float red[4];
  __shared__ __attribute__((aligned(16))) uint8_t tile[D * kPitch];
  const int j = blockIdx.x, y = blockIdx.y, b = blockIdx.z;
  const int start = a.starts[b];
  const int off = start & (a.block - 1);
  const int tid = threadIdx.x, c = tid % C, tl = tid / C;
  auto angles = [&](Angles8& g, int t) {
    const int64_t p = static_cast<int64_t>(start) + t;
    const int64_t at = static_cast<int64_t>(p < 0 ? 0 : (p < a.rope_rows ? p : a.rope_rows - 1)) * (a.rot / 2);
    g.load(c, a.rot, a.inter, a.cos_t + at, a.sin_t + at);
  };

  if (y >= 2 * a.Hkv) {  // query heads: every token of the row, whatever its count
    const int h0 = (y - 2 * a.Hkv) * kQHeads;
    const int ta = max(0, j * a.block - off), tb = min(a.T, (j + 1) * a.block - off);
    for (int t = ta + tl; t < tb; t += TP) {
      Angles8 g;
      angles(g, t);
      Row8<DT> x[kQHeads];
      const int64_t row = b * a.q_sb + t * a.q_st + 8 * c;
#pragma unroll
      for (int e = 0; e < kQHeads; ++e) x[e].load(a.q, row + min(h0 + e, a.H - 1) * a.q_sh);
#pragma unroll
      for (int e = 0; e < kQHeads; ++e) {
        rotate_lane<DT>(x[e], c, a.rot, a.inter, g);
        if (h0 + e < a.H) x[e].store(a.q_out, ((static_cast<int64_t>(b) * a.T + t) * a.H + h0 + e) * D + 8 * c);
      }
    }
    return;
  }

  if (start < 0) return;
  const int count = a.counts != nullptr ? min(max(a.counts[b], 0), a.T) : a.T;
  const int lo = j == 0 ? off : 0, hi = min(a.block, off + count - j * a.block);
  const int blk = (start >> a.shift) + j;
  if (hi <= lo || blk >= a.width) return;
  const int page = a.table[static_cast<int64_t>(b) * a.width + blk];
  if (page < 0 || page >= a.pages) return;  // no such page: the tokens are not stored
  const bool is_v = y >= a.Hkv;
  const int h = is_v ? y - a.Hkv : y;
  const int64_t ph = static_cast<int64_t>(page) * a.Hkv + h;
  float* const sp = (is_v ? a.vs : a.ks) + ph;
  uint8_t* const codes = (is_v ? a.vc : a.kc) + ph * a.block * D;
  const float had = lo > 0 ? fmaxf(*sp, kKvMinScale) : 0.0f;

  const int slot0 = NP == 1 ? lo + tl : NP * tl;
  Row8<DT> x[NP];
  {
    const void* const src = is_v ? a.v : a.k;
    const int64_t row = (is_v ? b * a.v_sb + h * a.v_sh : b * a.k_sb + h * a.k_sh) + 8 * c;
    const int64_t st = is_v ? a.v_st : a.k_st;
#pragma unroll
    for (int p = 0; p < NP; ++p) x[p].load(src, row + (min(max(slot0 + p, lo), hi - 1) - off + j * a.block) * st);
  }
  if (!is_v && a.cos_t != nullptr) {
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      Angles8 g;
      angles(g, min(max(slot0 + p, lo), hi - 1) - off + j * a.block);
      rotate_lane<DT>(x[p], c, a.rot, a.inter, g);
    }
  }
  float most = 0.0f, top = 0.0f;  // largest finite magnitude; largest of all, NaN where there is one
#pragma unroll
  for (int p = 0; p < NP; ++p)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float m = fabsf(x[p].get(e));
      top = __builtin_elementwise_maximum(top, m);
    }
  most = top;
  if (!(top <= 3.402823466e38f)) {
    most = 0.0f;
#pragma unroll
    for (int p = 0; p < NP; ++p)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float m = fabsf(x[p].get(e));
        most = fmaxf(most, m <= 3.402823466e38f ? m : 0.0f);
      }
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) most = fmaxf(most, __shfl_xor(most, o, 64));
  if ((tid & 63) == 0) red[tid >> 6] = most;
  __syncthreads();
  most = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  float s = fmaxf(most * Code::kInvMax, kKvMinScale);
  float down = 1.0f;  // 2^-k
  if (lo > 0) {
    int en, eh;
    const float mn = frexpf(s, &en), mh = frexpf(had, &eh);
    const int k = max(en - eh + (mn > mh ? 1 : 0), 0);
    s = ldexpf(had, k);
    down = ldexpf(1.0f, -k);
  }
  if (tid == 0) *sp = s;
  const SharedDiv sd = shared_div(s);
  const bool quick = sd.ok && __ballot(!fast_div(sd, top)) == 0;  // wave-uniform
  auto encode4 = [&](float v0, float v1, float v2, float v3) -> uint32_t {
    if (quick) return Code::encode4(sd, v0, v1, v2, v3);
    return Code::encode(sd, v0) | (Code::encode(sd, v1) << 8) | (Code::encode(sd, v2) << 16) | (Code::encode(sd, v3) << 24);
  };

  if (!is_v) {
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const int slot = slot0 + p;
      const u32x2v_t w = {encode4(x[p].get(0), x[p].get(1), x[p].get(2), x[p].get(3)),
                          encode4(x[p].get(4), x[p].get(5), x[p].get(6), x[p].get(7))};
      if (slot >= lo && slot < hi) *reinterpret_cast<u32x2v_t*>(codes + slot * D + 8 * c) = w;
    }
    if (down != 1.0f) {
      for (int i = tid; i < lo * (D / 4); i += 256) {
        uint32_t* w = reinterpret_cast<uint32_t*>(codes) + i;
        *w = Code::shrink4(*w, down);
      }
    }
    return;
  }
  // values: transposed through LDS, then 16 tokens of a column at a time, merged with the codes that stay. Column d lies at
  // row (d % 8) C + d / 8: the lanes of a wave write rows kPitch apart, which spreads them over the banks.
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    uint8_t* const t = tile + (e * C + c) * kPitch;
    if constexpr (NP >= 4) {
#pragma unroll
      for (int p = 0; p < NP; p += 4)
        *reinterpret_cast<uint32_t*>(t + slot0 + p) = encode4(x[p].get(e), x[p + 1].get(e), x[p + 2].get(e), x[p + 3].get(e));
    } else if constexpr (NP == 2) {
      *reinterpret_cast<uint16_t*>(t + slot0) = static_cast<uint16_t>(encode4(x[0].get(e), x[1].get(e), 0.0f, 0.0f));
    } else if (e % 4 == 0) {
      const uint32_t w = encode4(x[0].get(e), x[0].get(e + 1), x[0].get(e + 2), x[0].get(e + 3));
      if (slot0 < hi) {
#pragma unroll
        for (int q = 0; q < 4; ++q) t[q * C * kPitch + slot0] = static_cast<uint8_t>(w >> (8 * q));
      }
    }
  }
  __syncthreads();
  const int sh = a.shift - 4;  // 16-token pieces of a column: 1 << sh
  for (int i = tid; i < D << sh; i += 256) {
    const int d = i >> sh, s0 = (i & ((1 << sh) - 1)) * 16;
    if (s0 >= hi || (s0 + 16 <= lo && down == 1.0f)) continue;
    u32x4_t* g = reinterpret_cast<u32x4_t*>(codes + d * a.block + s0);
    const u32x4_t n = *reinterpret_cast<const u32x4_t*>(tile + ((d & 7) * C + (d >> 3)) * kPitch + s0);
    u32x4_t w;
    if (s0 >= lo && s0 + 16 <= hi) {
      w = n;
    } else {
      w = *g;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        uint32_t r = w[q];
        const uint32_t nw = n[q];
        const int s4 = s0 + 4 * q;
        const uint32_t less = down != 1.0f && s4 < lo ? Code::shrink4(r, down) : r;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t byte = 0xffu << (8 * e);
          if (s4 + e < lo) r = (r & ~byte) | (less & byte);
          else if (s4 + e < hi) r = (r & ~byte) | (nw & byte);
        }
        w[q] = r;
      }
    }
    *g = w;
  }
}

// Values of positions starts[b] .. + tokens - 1 of every row: fp32(code) * scale, rounded once; zeros from counts[b] on,
// outside the table and where it names no page. 12977 tokens as bf16: 20 us, 3.9 TB/s, values through LDS.
template <int DT, int D, bool E4M3>
__global__ __launch_bounds__(256) void kv_read_kernel(const uint8_t* __restrict__ kc, const uint8_t* __restrict__ vc,
                                                      const float* __restrict__ ks, const float* __restrict__ vs,
                                                      const int* __restrict__ table, const int* __restrict__ starts,
                                                      const int* __restrict__ counts, int T, int Hkv, int width,
                                                      int pages, int block, int shift, void* k_out, void* v_out) {
  using Code = KvCode<E4M3>;
  constexpr int C = D / 8, TP = 256 / C, kPitch = 128 + 16;
  __shared__ __attribute__((aligned(16))) uint8_t tile[D * kPitch];
  const int j = blockIdx.x, y = blockIdx.y, b = blockIdx.z;
  const bool is_v = y >= Hkv;
  const int h = is_v ? y - Hkv : y;
  const int start = starts[b], off = start & (block - 1);
  const int count = counts != nullptr ? min(max(counts[b], 0), T) : T;
  const int lo = j == 0 ? off : 0, hi = min(block, off + T - j * block);
  const int tid = threadIdx.x, c = tid % C, tl = tid / C;
  if (hi <= lo) return;
  const int64_t blk = (static_cast<int64_t>(start) >> shift) + j;
  int page = -1;
  if (start >= 0 && blk < width) page = table[static_cast<int64_t>(b) * width + blk];
  const bool some = page >= 0 && page < pages;
  const int64_t ph = some ? static_cast<int64_t>(page) * Hkv + h : 0;
  const float s = some ? (is_v ? vs : ks)[ph] : 0.0f;
  const uint8_t* codes = (is_v ? vc : kc) + ph * block * D;
  void* const out = is_v ? v_out : k_out;
  const int64_t row0 = static_cast<int64_t>(b) * T + (static_cast<int64_t>(j) * block - off);  // of slot 0
  // eight codes of a token's columns 8 c .. as values, to its row of the output
  auto put = [&](int slot, uint32_t w0, uint32_t w1) {
    const bool have = some && slot - off + j * block < count;
    Row8<DT> r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = i < 2 ? w0 : w1;
      const float lo_v = Code::decode((w >> (16 * (i & 1))) & 0xffu) * s, hi_v = Code::decode((w >> (16 * (i & 1) + 8)) & 0xffu) * s;
      r.set_pair(i, have ? lo_v : 0.0f, have ? hi_v : 0.0f);
    }
    r.store(out, ((row0 + slot) * Hkv + h) * D + 8 * c);
  };
  if (!is_v || !some) {
#pragma unroll 4
    for (int slot = lo + tl; slot < hi; slot += TP) {
      u32x2v_t w = {0u, 0u};
      if (some) w = *reinterpret_cast<const u32x2v_t*>(codes + slot * D + 8 * c);
      put(slot, w[0], w[1]);
    }
    return;
  }
  // values: through LDS as in the write, four tokens of eight columns at a time
  const int sh = shift - 4;
#pragma unroll 4
  for (int i = tid; i < D << sh; i += 256) {
    const int d = i >> sh, s0 = (i & ((1 << sh) - 1)) * 16;
    *reinterpret_cast<u32x4_t*>(tile + ((d & 7) * C + (d >> 3)) * kPitch + s0) = *reinterpret_cast<const u32x4_t*>(codes + d * block + s0);
  }
  __syncthreads();
  for (int g = tl; g < block / 4; g += TP) {
    if (4 * g + 4 <= lo || 4 * g >= hi) continue;
    uint32_t w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = *reinterpret_cast<const uint32_t*>(tile + (e * C + c) * kPitch + 4 * g);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (4 * g + q < lo || 4 * g + q >= hi) continue;
      const uint32_t sel = 0x0c0c0400u + 0x0101u * q;  // byte q of each of two dwords
      const uint32_t a = __builtin_amdgcn_perm(w[1], w[0], sel) | (__builtin_amdgcn_perm(w[3], w[2], sel) << 16);
      const uint32_t z = __builtin_amdgcn_perm(w[5], w[4], sel) | (__builtin_amdgcn_perm(w[7], w[6], sel) << 16);
      put(4 * g + q, a, z);
    }
  }
}

// The open block of a row is the one that its next token, at position starts[b], goes into behind earlier ones. Workgroup
// (i, b, l): piece i of row b's open block of layer l, between the cache and `saved` [L, B, 2, Hkv * block * D] (keys, then
// values), scales behind it [L, B, 2, Hkv]. Nothing where the row has no such block or rows[b] is zero. Bound by HBM: the
// blocks of 64 tokens of 32 layers (8 kv heads of 128) of 64 rows, 268 MB each way, take 107 us, 5.0 TB/s; of 8 rows 11 us.
constexpr int kOpenUnits = 4;  // 16-byte units of a thread, loaded before the first is stored
template <bool BACK>
__global__ __launch_bounds__(256) void kv_open_kernel(u32x4_t* __restrict__ kc, u32x4_t* __restrict__ vc, float* __restrict__ ks,
                                                      float* __restrict__ vs, const int* __restrict__ table,
                                                      const int* __restrict__ starts, const int* __restrict__ rows, int Hkv,
                                                      int width, int pages, int block, int shift, int units,
                                                      u32x4_t* __restrict__ saved, float* __restrict__ saved_scale) {
  const int b = blockIdx.y, l = blockIdx.z, tid = threadIdx.x;
  const int start = starts[b], blk = start >> shift;
  if (start < 0 || (start & (block - 1)) == 0 || blk >= width || (rows != nullptr && rows[b] == 0)) return;
  const int page = table[static_cast<int64_t>(b) * width + blk];
  if (page < 0 || page >= pages) return;
  const int64_t at = static_cast<int64_t>(l) * pages + page, to = (static_cast<int64_t>(l) * gridDim.y + b) * 2;
  u32x4_t w[kOpenUnits];
  u32x4_t* src[kOpenUnits];
  u32x4_t* dst[kOpenUnits];
#pragma unroll
  for (int u = 0; u < kOpenUnits; ++u) {
    const int i = min((blockIdx.x * kOpenUnits + u) * 256 + tid, 2 * units - 1);  // past the end: the last unit again
    u32x4_t* const c = i < units ? kc + at * units + i : vc + at * units + i - units;
    u32x4_t* const s = saved + to * units + i;
    src[u] = BACK ? s : c;
    dst[u] = BACK ? c : s;
    w[u] = *src[u];
  }
#pragma unroll
  for (int u = 0; u < kOpenUnits; ++u) *dst[u] = w[u];
  if (blockIdx.x != 0) return;
  for (int h = tid; h < 2 * Hkv; h += 256) {
    float* const c = h < Hkv ? ks + at * Hkv + h : vs + at * Hkv + h - Hkv;
    float* const s = saved_scale + to * Hkv + h;
    if (BACK) *c = *s;
    else *s = *c;
  }
}

}  // namespace sqx

using namespace sqx;

extern "C" int sqx_kvblock_write(const void* k, const void* v, int dtype, int64_t k_sb, int64_t k_st, int64_t k_sh,
                                 int64_t v_sb, int64_t v_st, int64_t v_sh, const void* q, int64_t q_sb, int64_t q_st,
                                 int64_t q_sh, void* q_out, const float* cos_t, const float* sin_t, int64_t rope_rows,
                                 int64_t rot, int interleaved, int fmt, void* k_codes, void* v_codes, float* k_scale,
                                 float* v_scale, const int* table, const int* starts, const int* counts, int64_t B,
                                 int64_t T, int64_t H, int64_t Hkv, int64_t hd, int64_t block, int64_t pages,
                                 int64_t width, sqx_stream_t stream) {
  const char* fn = "sqx_kvblock_write";
  KV_SHAPE(fn);
  SQX_REQUIRE((cos_t == nullptr) == (sin_t == nullptr), SQX_E_ARG, "%s: give both tables or neither", fn);
  SQX_REQUIRE(q == nullptr || cos_t != nullptr, SQX_E_ARG, "%s: queries are only rotated here: give the tables", fn);
  SQX_REQUIRE((q == nullptr) == (q_out == nullptr), SQX_E_ARG, "%s: q and q_out go together", fn);
  SQX_REQUIRE(q == nullptr || (H >= 1 && H <= 8192), SQX_E_ARG, "%s: H=%lld (1 to 8192)", fn, (long long)H);
  SQX_REQUIRE(cos_t == nullptr || (rot >= 16 && rot % 16 == 0 && rot <= hd && rope_rows >= 1 &&
                                   rope_rows < (int64_t(1) << 31)),
              SQX_E_ARG, "%s: rot=%lld must be a multiple of 16 up to head_dim, and the table not empty", fn, (long long)rot);
  SQX_REQUIRE(k_sb >= 0 && k_st >= 0 && k_sh >= 0 && v_sb >= 0 && v_st >= 0 && v_sh >= 0 && q_sb >= 0 && q_st >= 0 &&
                  q_sh >= 0,
              SQX_E_ARG, "%s: negative stride", fn);
  SQX_REQUIRE((k_sb | k_st | k_sh | v_sb | v_st | v_sh | q_sb | q_st | q_sh) % 8 == 0, SQX_E_ARG,
              "%s: strides must be multiples of 8 elements", fn);
  if (B == 0 || T == 0) return SQX_OK;
  SQX_REQUIRE(k && v && k_codes && v_codes && k_scale && v_scale && table && starts, SQX_E_ARG, "%s: null pointer", fn);
  SQX_REQUIRE(al16(k) && al16(v) && al16(q) && al16(q_out) && al16(k_codes) && al16(v_codes) && al16(cos_t) && al16(sin_t),
              SQX_E_ARG, "%s: rows, codes and tables must be 16-byte aligned", fn);
  KvWriteArgs a{};
  a.k = k; a.v = v; a.q = q; a.q_out = q_out;
  a.k_sb = k_sb; a.k_st = k_st; a.k_sh = k_sh;
  a.v_sb = v_sb; a.v_st = v_st; a.v_sh = v_sh;
  a.q_sb = q_sb; a.q_st = q_st; a.q_sh = q_sh;
  a.kc = static_cast<uint8_t*>(k_codes); a.vc = static_cast<uint8_t*>(v_codes);
  a.ks = k_scale; a.vs = v_scale;
  a.table = table; a.starts = starts; a.counts = counts;
  a.cos_t = cos_t; a.sin_t = sin_t;
  a.rope_rows = static_cast<int>(cos_t ? rope_rows : 1); a.rot = static_cast<int>(cos_t ? rot : 0); a.inter = interleaved;
  a.T = static_cast<int>(T); a.H = static_cast<int>(H); a.Hkv = static_cast<int>(Hkv); a.width = static_cast<int>(width);
  a.pages = static_cast<int>(pages); a.block = static_cast<int>(block);
  a.shift = kv_shift(block);
  const dim3 grid(static_cast<unsigned>((T + 2 * block - 2) / block),
                  static_cast<unsigned>(2 * Hkv + (q ? ceil_div(H, kQHeads) : 0)), static_cast<unsigned>(B));
  with_dtype(dtype, [&](auto dt) {
    with_head(hd, [&](auto dd) {
      constexpr int DT = decltype(dt)::value, D = decltype(dd)::value, TP = 2048 / D;
      auto go = [&](auto np) {
        constexpr int NP = decltype(np)::value;
        if (fmt == SQX_KV_E4M3)
          hipLaunchKernelGGL((kv_write_kernel<DT, D, true, NP>), grid, dim3(256), 0, as_stream(stream), a);
        else
          hipLaunchKernelGGL((kv_write_kernel<DT, D, false, NP>), grid, dim3(256), 0, as_stream(stream), a);
      };
      // tokens per thread: one where those of a block fit the workgroup once, else a block's
      const int64_t np = std::min(T, block) <= TP ? 1 : block / TP;
      if (np == 1) go(std::integral_constant<int, 1>{});
      else if (np == 2) go(std::integral_constant<int, 2>{});
      else if (np == 4) go(std::integral_constant<int, 4>{});
      else if constexpr (D > 64) {
        if (np == 8) go(std::integral_constant<int, 8>{});
        else if constexpr (D > 128) go(std::integral_constant<int, 16>{});
      }
    });
  });
  SQX_LAUNCH_CHECK(fn);
  return SQX_OK;
}

extern "C" int sqx_kvblock_read(int fmt, const void* k_codes, const void* v_codes, const float* k_scale,
                                const float* v_scale, const int* table, const int* starts, const int* counts, int64_t B,
                                int64_t T, int64_t Hkv, int64_t hd, int64_t block, int64_t pages, int64_t width,
                                int dtype, void* k_out, void* v_out, sqx_stream_t stream) {
  const char* fn = "sqx_kvblock_read";
  KV_SHAPE(fn);
  if (B == 0 || T == 0) return SQX_OK;
  SQX_REQUIRE(k_codes && v_codes && k_scale && v_scale && table && starts && k_out && v_out, SQX_E_ARG, "%s: null pointer",
              fn);
  SQX_REQUIRE(al16(k_codes) && al16(v_codes) && al16(k_out) && al16(v_out), SQX_E_ARG,
              "%s: codes and outputs must be 16-byte aligned", fn);
  const int shift = kv_shift(block);
  const dim3 grid(static_cast<unsigned>((T + 2 * block - 2) / block), static_cast<unsigned>(2 * Hkv),
                  static_cast<unsigned>(B));
  with_dtype(dtype, [&](auto dt) {
    with_head(hd, [&](auto dd) {
      auto go = [&](auto e4) {
        hipLaunchKernelGGL((kv_read_kernel<decltype(dt)::value, decltype(dd)::value, decltype(e4)::value>), grid, dim3(256), 0,
                           as_stream(stream), static_cast<const uint8_t*>(k_codes), static_cast<const uint8_t*>(v_codes),
                           k_scale, v_scale, table, starts, counts, static_cast<int>(T), static_cast<int>(Hkv),
                           static_cast<int>(width), static_cast<int>(pages), static_cast<int>(block), shift, k_out, v_out);
      };
      if (fmt == SQX_KV_E4M3) go(std::true_type{});
      else go(std::false_type{});
    });
  });
  SQX_LAUNCH_CHECK(fn);
  return SQX_OK;
}

extern "C" int64_t sqx_kvblock_open_bytes(int64_t L, int64_t B, int64_t Hkv, int64_t hd, int64_t block) {
  if (L <= 0 || B <= 0 || Hkv <= 0 || !(hd == 64 || hd == 128 || hd == 256) || !kv_block_ok(block)) return 0;
  return L * B * 2 * Hkv * (block * hd + 4);
}

extern "C" int sqx_kvblock_open(int back, void* k_codes, void* v_codes, float* k_scale, float* v_scale, const int* table,
                                const int* starts, const int* rows, int64_t L, int64_t B, int64_t Hkv, int64_t hd,
                                int64_t block, int64_t pages, int64_t width, void* saved, int64_t saved_bytes,
                                sqx_stream_t stream) {
  const char* fn = "sqx_kvblock_open";
  const int fmt = SQX_KV_INT8, dtype = SQX_DTYPE_F32;
  const int64_t T = 1;
  KV_SHAPE(fn);
  SQX_REQUIRE(L >= 0 && L < 65536, SQX_E_ARG, "%s: L=%lld layers (below 65536)", fn, (long long)L);
  if (L == 0 || B == 0) return SQX_OK;
  SQX_REQUIRE(k_codes && v_codes && k_scale && v_scale && table && starts && saved, SQX_E_ARG, "%s: null pointer", fn);
  SQX_REQUIRE(al16(k_codes) && al16(v_codes) && al16(saved), SQX_E_ARG, "%s: codes and saved must be 16-byte aligned", fn);
  const int64_t need = sqx_kvblock_open_bytes(L, B, Hkv, hd, block);
  SQX_REQUIRE(saved_bytes >= need, SQX_E_SPACE, "%s: %lld bytes needed for the saved blocks, %lld given", fn, (long long)need,
              (long long)saved_bytes);
  const int64_t units = Hkv * block * hd / 16;
  float* const scales = reinterpret_cast<float*>(static_cast<char*>(saved) + L * B * 2 * units * 16);
  const dim3 grid(static_cast<unsigned>(ceil_div(2 * units, 256 * kOpenUnits)), static_cast<unsigned>(B), static_cast<unsigned>(L));
  auto go = [&](auto bk) {
    hipLaunchKernelGGL((kv_open_kernel<decltype(bk)::value>), grid, dim3(256), 0, as_stream(stream), static_cast<u32x4_t*>(k_codes),
                       static_cast<u32x4_t*>(v_codes), k_scale, v_scale, table, starts, rows, static_cast<int>(Hkv),
                       static_cast<int>(width), static_cast<int>(pages), static_cast<int>(block), kv_shift(block),
                       static_cast<int>(units), static_cast<u32x4_t*>(saved), scales);
  };
  if (back != 0) go(std::true_type{});
  else go(std::false_type{});
  SQX_LAUNCH_CHECK(fn);
  return SQX_OK;
}
