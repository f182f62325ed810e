// Shared pieces of the block-scaled 8-bit KV cache kernels (sqx_kvblock.hip, sqx_kvattn.hip): element types, the two
// code formats, rotary pairs.
//
// A layer's cache is paged. Page p holds `block` tokens (16, 32, 64 or 128) of every kv head: key codes
// [page, Hkv, block, D], value codes [page, Hkv, D, block] (the value product contracts over tokens, and a lane's matrix
// operand is then 16 consecutive bytes), one fp32 scale per page and head for the keys and one for the values. A code c
// stands for c * scale: int8 in [-127, 127], or E4M3.
#pragma once

#include <type_traits>

#include "sqx_common.h"
#include "sqx_quant.h"

namespace sqx {

constexpr float kKvMinScale = 1e-12f;  // a block of zeros

// Eight consecutive elements of a row in registers: packed pairs for the 16-bit types.
template <int DT>
struct Row8 {
  static constexpr int kWords = DT == SQX_DTYPE_F32 ? 8 : 4;
  uint32_t w[kWords];

  __device__ inline float get(int e) const {
    if constexpr (DT == SQX_DTYPE_F32) return __builtin_bit_cast(float, w[e]);
    else if constexpr (DT == SQX_DTYPE_BF16) return (e & 1) ? bf16_hi(w[e >> 1]) : bf16_lo(w[e >> 1]);
    else return f16_bits_to_f32(static_cast<uint16_t>((e & 1) ? w[e >> 1] >> 16 : w[e >> 1]));
  }
  __device__ inline void set_pair(int pair, float lo, float hi) {  // elements 2 pair, 2 pair + 1, each rounded once
    if constexpr (DT == SQX_DTYPE_F32) {
      w[2 * pair] = __builtin_bit_cast(uint32_t, lo);
      w[2 * pair + 1] = __builtin_bit_cast(uint32_t, hi);
    } else if constexpr (DT == SQX_DTYPE_BF16) {
      w[pair] = ActBF16::pack_rne(lo, hi);
    } else {
      w[pair] = ActF16::pack_rne(lo, hi);
    }
  }
  __device__ inline void load(const void* base, int64_t elem) {  // elem a multiple of 8, base 16-byte aligned
    const u32x4_t* p = reinterpret_cast<const u32x4_t*>(static_cast<const char*>(base) + elem * (kWords / 2));
#pragma unroll
    for (int i = 0; i < kWords / 4; ++i) {
      const u32x4_t a = p[i];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[4 * i + j] = a[j];
    }
  }
  __device__ inline void store(void* base, int64_t elem) const {
    u32x4_t* p = reinterpret_cast<u32x4_t*>(static_cast<char*>(base) + elem * (kWords / 2));
#pragma unroll
    for (int i = 0; i < kWords / 4; ++i) p[i] = u32x4_t{w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]};
  }
};

// One rotary pair. Contraction is off: each product and each sum rounds to fp32 on its own, as separate elementwise
// operations do, so the stored keys do not depend on which kernel rotated them.
__device__ inline void rope_pair(float a, float b, float c, float s, float& ya, float& yb) {
#pragma clang fp contract(off)
  const float ac = a * c, bs = b * s, as = a * s, bc = b * c;
  ya = ac - bs;
  yb = as + bc;
}

// The angles of the 8 columns from column 8 c of a head whose first `rot` columns are rotated (rot % 16 == 0): interleaved
// pairs 2i, 2i + 1 take four of them, halves (pairs i, i + rot / 2) eight. cos_r, sin_r: the position's table row.
struct Angles8 {
  float c[8], s[8];
  __device__ inline void load(int col8, int rot, bool inter, const float* cos_r, const float* sin_r) {
    if (8 * col8 >= rot) return;
    const int at = inter ? 4 * col8 : 8 * (col8 < rot / 16 ? col8 : col8 - rot / 16);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (h == 1 && inter) break;
      const f32x4_t a = *reinterpret_cast<const f32x4_t*>(cos_r + at + 4 * h);
      const f32x4_t b = *reinterpret_cast<const f32x4_t*>(sin_r + at + 4 * h);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        c[4 * h + j] = a[j];
        s[4 * h + j] = b[j];
      }
    }
  }
};
template <int DT>
__device__ inline void rotate_pairs(Row8<DT>& x, const Angles8& g) {  // interleaved
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float ya, yb;
    rope_pair(x.get(2 * i), x.get(2 * i + 1), g.c[i], g.s[i], ya, yb);
    x.set_pair(i, ya, yb);
  }
}
template <int DT>
__device__ inline void rotate_halves(Row8<DT>& a, Row8<DT>& b, const Angles8& g) {  // a of the first half, b of the second
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float ya[2], yb[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) rope_pair(a.get(2 * i + e), b.get(2 * i + e), g.c[2 * i + e], g.s[2 * i + e], ya[e], yb[e]);
    a.set_pair(i, ya[0], ya[1]);
    b.set_pair(i, yb[0], yb[1]);
  }
}

// Codes.
template <bool E4M3>
struct KvCode {
  static constexpr float kInvMax = 1.0f / (E4M3 ? 448.0f : 127.0f);  // the largest code may be passed by an ulp: it clamps
  __device__ static inline uint32_t encode(const SharedDiv& d, float v) {
    const float y = div_by(d, v);
    if constexpr (E4M3) return e4m3_encode_sat(y);
    const float r = y != y ? 0.0f : fminf(fmaxf(rintf(y), -127.0f), 127.0f);  // int8 has no NaN: it stores zero
    return static_cast<uint32_t>(static_cast<int>(r)) & 0xffu;
  }
  // Four codes where every value is finite and the shared division's fast form holds: the same bits as encode. The sum with
  // 1.5 2^23 rounds to the nearest even integer and leaves it, as two's complement, in the low byte.
  __device__ static inline uint32_t encode4(const SharedDiv& d, float v0, float v1, float v2, float v3) {
    const float v[4] = {v0, v1, v2, v3};
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = __builtin_amdgcn_fmed3f(quick_div(d, v[i]), E4M3 ? -448.0f : -127.0f, E4M3 ? 448.0f : 127.0f);
    if constexpr (E4M3) {
      int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
      return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true));
    }
    uint32_t t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = __builtin_bit_cast(uint32_t, y[i] + 12582912.0f);
    const uint32_t lo = __builtin_amdgcn_perm(t[1], t[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(t[3], t[2], 0x04000c0cu);
    return lo | hi;
  }
  __device__ static inline float decode(uint32_t byte) {
    if constexpr (E4M3) {
      const f32x2_t p = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(byte), false);
      return p[0];
    }
    return static_cast<float>(static_cast<int>(static_cast<int8_t>(byte)));
  }
  // c * down for a power of two `down` <= 1, rounded to nearest even
  __device__ static inline uint32_t shrink(uint32_t byte, float down) {
    if constexpr (E4M3) {
      if ((byte & 0x7fu) == 0x7fu) return byte;
      return e4m3_encode_sat(decode(byte) * down);
    }
    return static_cast<uint32_t>(static_cast<int>(rintf(decode(byte) * down))) & 0xffu;
  }
  __device__ static inline uint32_t shrink4(uint32_t w, float down) {
    uint32_t r = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) r |= shrink((w >> (8 * i)) & 0xffu, down) << (8 * i);
    return r;
  }
};

// ---------------------------------------------------------------- host side ----
inline bool kv_block_ok(int64_t block) { return block == 16 || block == 32 || block == 64 || block == 128; }
inline int kv_shift(int64_t block) { return block == 16 ? 4 : block == 32 ? 5 : block == 64 ? 6 : 7; }
inline bool al16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

template <typename F>
void with_dtype(int dtype, const F& f) {
  if (dtype == SQX_DTYPE_F32) f(std::integral_constant<int, SQX_DTYPE_F32>{});
  else if (dtype == SQX_DTYPE_BF16) f(std::integral_constant<int, SQX_DTYPE_BF16>{});
  else f(std::integral_constant<int, SQX_DTYPE_F16>{});
}
template <typename F>
void with_head(int64_t d, const F& f) {
  if (d == 64) f(std::integral_constant<int, 64>{});
  else if (d == 128) f(std::integral_constant<int, 128>{});
  else f(std::integral_constant<int, 256>{});
}

}  // namespace sqx

// What every entry point of the cache checks of its sizes.
#define KV_SHAPE(fn)                                                                                                     \
  SQX_REQUIRE(dtype == SQX_DTYPE_F32 || dtype == SQX_DTYPE_BF16 || dtype == SQX_DTYPE_F16, SQX_E_ARG,                    \
              "%s: keys and values must be F32, BF16 or F16", fn);                                                       \
  SQX_REQUIRE(fmt == SQX_KV_INT8 || fmt == SQX_KV_E4M3, SQX_E_ARG, "%s: unknown code format %d", fn, fmt);               \
  SQX_REQUIRE(kv_block_ok(block), SQX_E_ARG, "%s: block=%lld (16, 32, 64 or 128 tokens)", fn, (long long)block);         \
  SQX_REQUIRE(hd == 64 || hd == 128 || hd == 256, SQX_E_ARG, "%s: head_dim=%lld (64, 128 or 256)", fn, (long long)hd);   \
  SQX_REQUIRE(B >= 0 && B < 65536 && T >= 0 && T < (int64_t(1) << 24) && Hkv >= 1 && Hkv <= 1024, SQX_E_ARG,             \
              "%s: bad shape (B=%lld below 65536, T=%lld below 2^24, Hkv=%lld up to 1024)", fn, (long long)B,            \
              (long long)T, (long long)Hkv);                                                                             \
  SQX_REQUIRE(pages >= 1 && pages < (int64_t(1) << 31) && width >= 1 && width * block < (int64_t(1) << 30), SQX_E_ARG,   \
              "%s: pages=%lld and a table of %lld blocks (at least 1; positions below 2^30)", fn, (long long)pages,      \
              (long long)width)
