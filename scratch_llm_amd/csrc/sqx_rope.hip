// Rotary positions of rows of heads, on their own: interleaved pairs or halves, all of a head's columns or the first
// `rot`, any table. The cache write (sqx_kvblock.hip) applies the same pairs to the keys and queries of a step.
//
// y_a = x_a cos - x_b sin, y_b = x_a sin + x_b cos, in fp32 with every product and sum rounded on its own, rounded once
// to x's type. Three flops per element against two memory passes over it: bound by HBM for prompts (8191 tokens of 40 heads
// of 128 columns in fp16, half of them rotated: 28 us, 6.1 TB/s, of which the 84 MB written partly end in the last cache; a
// call among others 31 us, 5.5 TB/s), by the launch for a few tokens (one: 2.2 us). Rounding pairs by the packed conversions
// instead of one by one was worth 31 -> 27 us.
#include "sqx_kvblock.h"

namespace sqx {

// Eight columns of kRopeHeads heads of a row of heads: with halves the thread at a column of the first half takes both groups
// of its pairs (rows may be rotated in place), and those of the second half are idle. All loads come before the first use.
constexpr int kRopeHeads = 4;
template <int DT>
__device__ inline void rope_columns(const void* x, int64_t row, int64_t sh, void* out, int64_t orow, int64_t oh, int h0,
                                    int hs, int heads, int c, int rot, bool inter, const Angles8& ang) {
  const int half8 = inter ? 0 : rot / 16;
  if (c >= half8 && c < 2 * half8) return;
  Row8<DT> a[kRopeHeads], b[kRopeHeads];
#pragma unroll
  for (int i = 0; i < kRopeHeads; ++i) {
    const int h = h0 + i * hs;
    if (h >= heads) break;
    a[i].load(x, row + h * sh + 8 * c);
    if (c < half8) b[i].load(x, row + h * sh + 8 * (c + half8));
  }
#pragma unroll
  for (int i = 0; i < kRopeHeads; ++i) {
    const int h = h0 + i * hs;
    if (h >= heads) break;
    if (c < half8) rotate_halves<DT>(a[i], b[i], ang);
    else if (inter && 8 * c < rot) rotate_pairs<DT>(a[i], ang);
    a[i].store(out, orow + h * oh + 8 * c);
    if (c < half8) b[i].store(out, orow + h * oh + 8 * (c + half8));
  }
}

// One workgroup per token: a thread owns a group of 8 columns (its part of the table row is read once) and walks the heads,
// 256 / (d / 8) heads apart, four at a time.
template <int DT>
__global__ __launch_bounds__(256) void rope_kernel(const void* x, int64_t sn, int64_t sh, const int* __restrict__ pos,
                                                   const float* __restrict__ cos_t, const float* __restrict__ sin_t,
                                                   int rows, int heads, int d8, int rot, int inter, void* out,
                                                   int64_t on, int64_t oh) {
  const int64_t n = blockIdx.x;
  const int c = threadIdx.x % d8, h0 = threadIdx.x / d8, hs = 256 / d8;
  if (h0 >= hs) return;
  const int p = min(max(pos[n], 0), rows - 1);
  Angles8 ang;
  ang.load(c, rot, inter, cos_t + static_cast<int64_t>(p) * (rot / 2), sin_t + static_cast<int64_t>(p) * (rot / 2));
  for (int h = h0; h < heads; h += kRopeHeads * hs)
    rope_columns<DT>(x, n * sn, sh, out, n * on, oh, h, hs, heads, c, rot, inter, ang);
}

// Any even rot and any alignment: a thread per pair (or per column past the rotated ones), two bytes a load: 91 us where the
// form above takes 29 (8191 tokens of 40 heads of 128, 40 and 48 columns rotated).
template <int DT>
__global__ __launch_bounds__(256) void rope_pairs_kernel(const void* x, int64_t sn, int64_t sh,
                                                         const int* __restrict__ pos, const float* __restrict__ cos_t,
                                                         const float* __restrict__ sin_t, int rows, int heads, int d,
                                                         int rot, int inter, void* out, int64_t on, int64_t oh) {
  const int64_t n = blockIdx.x;
  const int units = rot / 2 + (d - rot);
  const int p = min(max(pos[n], 0), rows - 1);
  using T = std::conditional_t<DT == SQX_DTYPE_F32, float, uint16_t>;
  const T* xs = static_cast<const T*>(x);
  T* os = static_cast<T*>(out);
  auto put = [&](int64_t at, float v) {
    if constexpr (DT == SQX_DTYPE_F32) os[at] = v;
    else os[at] = DT == SQX_DTYPE_BF16 ? f32_to_bf16_bits(v) : f32_to_f16_bits(v);
  };
  for (int i = threadIdx.x; i < heads * units; i += 256) {
    const int h = i / units, u = i - h * units;
    const int64_t row = n * sn + h * sh, orow = n * on + h * oh;
    if (u >= rot / 2) {
      os[orow + u + rot / 2] = xs[row + u + rot / 2];
      continue;
    }
    const int ia = inter ? 2 * u : u, ib = inter ? 2 * u + 1 : u + rot / 2;
    float ya, yb;
    rope_pair(load_as_f32(x, DT, row + ia), load_as_f32(x, DT, row + ib), cos_t[static_cast<int64_t>(p) * (rot / 2) + u],
              sin_t[static_cast<int64_t>(p) * (rot / 2) + u], ya, yb);
    put(orow + ia, ya);
    put(orow + ib, yb);
  }
}

}  // namespace sqx

using namespace sqx;

extern "C" int sqx_rope(const void* x, int dtype, int64_t n, int64_t heads, int64_t d, int64_t x_stride_n,
                        int64_t x_stride_h, const int* positions, const float* cos_t, const float* sin_t,
                        int64_t table_rows, int64_t rot, int interleaved, void* out, int64_t out_stride_n,
                        int64_t out_stride_h, sqx_stream_t stream) {
  const char* fn = "sqx_rope";
  SQX_REQUIRE(dtype == SQX_DTYPE_F32 || dtype == SQX_DTYPE_BF16 || dtype == SQX_DTYPE_F16, SQX_E_ARG,
              "%s: x must be F32, BF16 or F16", fn);
  SQX_REQUIRE(n >= 0 && n < (int64_t(1) << 24) && heads >= 1 && heads <= 65536 && d >= 1 && d <= 2048, SQX_E_ARG,
              "%s: bad shape (n=%lld below 2^24, heads=%lld up to 65536, d=%lld up to 2048)", fn, (long long)n, (long long)heads,
              (long long)d);
  SQX_REQUIRE(rot >= 2 && rot % 2 == 0 && rot <= d, SQX_E_ARG, "%s: rot=%lld must be even and within 2 .. d=%lld", fn,
              (long long)rot, (long long)d);
  SQX_REQUIRE(table_rows >= 1 && table_rows < (int64_t(1) << 31), SQX_E_ARG, "%s: empty table", fn);
  SQX_REQUIRE(x_stride_n >= 0 && x_stride_h >= 0 && out_stride_n >= 0 && out_stride_h >= 0, SQX_E_ARG,
              "%s: negative stride", fn);
  if (n == 0) return SQX_OK;
  SQX_REQUIRE(x && positions && cos_t && sin_t && out, SQX_E_ARG, "%s: null pointer", fn);
  const int64_t es = dtype == SQX_DTYPE_F32 ? 4 : 2;
  SQX_REQUIRE(reinterpret_cast<uintptr_t>(x) % es == 0 && reinterpret_cast<uintptr_t>(out) % es == 0, SQX_E_ARG,
              "%s: x and out must be aligned to their element", fn);
  const bool vec = d % 8 == 0 && d <= 2048 && rot % 16 == 0 && (reinterpret_cast<uintptr_t>(x) % 16 == 0) &&
                   (reinterpret_cast<uintptr_t>(out) % 16 == 0) && (reinterpret_cast<uintptr_t>(cos_t) % 16 == 0) &&
                   (reinterpret_cast<uintptr_t>(sin_t) % 16 == 0) && x_stride_n % 8 == 0 && x_stride_h % 8 == 0 &&
                   out_stride_n % 8 == 0 && out_stride_h % 8 == 0;
  const dim3 grid(static_cast<unsigned>(n));
  auto go = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    if (vec)
      hipLaunchKernelGGL((rope_kernel<DT>), grid, dim3(256), 0, as_stream(stream), x, x_stride_n, x_stride_h, positions,
                         cos_t, sin_t, static_cast<int>(table_rows), static_cast<int>(heads), static_cast<int>(d / 8),
                         static_cast<int>(rot), interleaved, out, out_stride_n, out_stride_h);
    else
      hipLaunchKernelGGL((rope_pairs_kernel<DT>), grid, dim3(256), 0, as_stream(stream), x, x_stride_n, x_stride_h,
                         positions, cos_t, sin_t, static_cast<int>(table_rows), static_cast<int>(heads),
                         static_cast<int>(d), static_cast<int>(rot), interleaved, out, out_stride_n, out_stride_h);
  };
  if (dtype == SQX_DTYPE_F32) go(std::integral_constant<int, SQX_DTYPE_F32>{});
  else if (dtype == SQX_DTYPE_BF16) go(std::integral_constant<int, SQX_DTYPE_BF16>{});
  else go(std::integral_constant<int, SQX_DTYPE_F16>{});
  SQX_LAUNCH_CHECK(fn);
  return SQX_OK;
}
