// Entry points of the attention over the block-scaled 8-bit KV cache (kernels and their figures: sqx_kvattn.h).
#include "sqx_kvattn.h"

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
