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
      w[pair] = static_cast<uint32_t>(f32_to_bf16_bits(lo)) | (static_cast<uint32_t>(f32_to_bf16_bits(hi)) << 16);
    } else {
      w[pair] = static_cast<uint32_t>(f32_to_f16_bits(lo)) | (static_cast<uint32_t>(f32_to_f16_bits(hi)) << 16);
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

// Rotates the 8 elements at column 8 c of a row whose first `rot` columns are rotated (rot % 16 == 0), in the
// interleaved layout (pairs 2i, 2i + 1) or in halves (pairs i, i + rot / 2; `load_other` fetches the 8 elements of
// the other half). cos_r, sin_r: the position's table row.
template <int DT, typename F>
__device__ inline void rope_row8(Row8<DT>& x, int c, int rot, bool inter, const float* cos_r, const float* sin_r,
                                 const F& load_other) {
  if (8 * c >= rot) return;
  if (inter) {
    const f32x4_t cs = *reinterpret_cast<const f32x4_t*>(cos_r + 4 * c);
    const f32x4_t sn = *reinterpret_cast<const f32x4_t*>(sin_r + 4 * c);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float ya, yb;
      rope_pair(x.get(2 * i), x.get(2 * i + 1), cs[i], sn[i], ya, yb);
      x.set_pair(i, ya, yb);
    }
    return;
  }
  const int half8 = rot / 16;  // 8-element groups per half
  const bool second = c >= half8;
  const int cc = second ? c - half8 : c;
  const Row8<DT> o = load_other(second ? cc : cc + half8);
  float cs[8], sn[8];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const f32x4_t a = *reinterpret_cast<const f32x4_t*>(cos_r + 8 * cc + 4 * h);
    const f32x4_t b = *reinterpret_cast<const f32x4_t*>(sin_r + 8 * cc + 4 * h);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      cs[4 * h + j] = a[j];
      sn[4 * h + j] = b[j];
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float y[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int k = 2 * i + e;
      float ya, yb;
      rope_pair(second ? o.get(k) : x.get(k), second ? x.get(k) : o.get(k), cs[k], sn[k], ya, yb);
      y[e] = second ? yb : ya;
    }
    x.set_pair(i, y[0], y[1]);
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
