// Attention over the block-scaled 8-bit KV cache of a batch whose rows share the first pages of their contexts (several answers
// to a prompt, one system prompt for all): the shared keys are read once for all rows of a group, each row's own keys for itself.
//
// Softmax over the union of two sets of keys needs of each only its maximum m, its sum l and its weighted values o, so the two
// are computed apart and joined: (m, l, o) of every part weighs in with 2^(m - max). A group of n rows brings n T G query rows to
// one product over the shared keys, where each row alone would bring T G: up to some hundred times the work per byte read.
//
// The plan says which rows make a group and how many whole blocks all of them name alike; it is made on the device from the
// table itself, and holds until the rows or their shared entries change. It also lists the workgroups of the shared part: a
// group's query rows in tiles, its keys in as many parts as its share of the work is of the chip's workgroups.
//
// Launches: the large groups' shared part (the prompt kernel: 256 query rows a workgroup, keys turned to fp16 once in LDS); the
// small groups' and every row's own keys in one (the direct kernel, 32 rows, straight from memory); the join.
//
// us a call in a graph, beside the attention that reads all keys for each row (32 heads over 8 of 128, int8 unless stated): 8 rows
// behind 2000 keys 13 (13); 64 behind 8192 33 (106); 32 behind 8192 26 (59); 128 behind 8192 55 (189); 256 behind 4096 73 (201); 16
// behind 32768 28 (101); 2 groups of 32 behind 16384 50 (186); 6 of 16 behind some 15000, E4M3, 78 (251); 24 pairs behind 4000 47
// (59). Few rows are bound by launches and dependent loads, the others by the products over the shared keys, whose conversion
// from 8 bits is repeated for every 32 query rows, and by the rows' own keys, from HBM.
#include "sqx_kvattn.h"

namespace sqx {

constexpr int kPlanThreads = 1024;
constexpr int kPlanRows = 4096;      // rows of a batch
// The prompt kernel takes groups of so many query rows, and of so many products of these with shared keys: its prologue and the 133
// KB that each of its workgroups leaves to be joined have to pay. us a call, direct and prompt kernel, 8 kv heads of 128, int8, at half
// the products, at the border and at twice as many:
//   512 rows x 8192 keys 51, 56; 16384 75, 72; 32768 122, 110
//   1024 x 4096 57, 66; 8192 86, 84; 16384 132, 120 (E4M3: 8192 83, 84; 16384 126, 120; heads of 64: 49, 57; 78, 75)
//   2048 x 2048 85, 94; 4096 111, 112; 8192 160, 149
// Heads of 256 gain more (4 kv heads: 512 x 16384 125, 90). The rule does not look at the kv heads: one alone at 1024 x 8192 24, 38.
constexpr int kTileFrom = 512;
constexpr int64_t kTileWork = int64_t(1) << 23;
constexpr int kDirectGroups = 512, kTileGroups = 256;
constexpr int kPartSteps = 40;

// Query rows of a row (T G) up to which the direct kernel takes it; from there on it reads its keys once for many rows by itself.
constexpr int own_most(int64_t d) { return d == 256 ? 64 : 128; }
constexpr int direct_rows(int d) { return d == 256 ? 16 : 32; }

// A plan's arrays. What a workgroup or a row needs stands together, to be had in one load.
struct KvItem {  // a workgroup of the shared part
  int lead;         // a row that names the shared blocks; -1: no item
  int first, M;     // the group's first row in `order`, its query rows per kv head
  int keys;         // shared keys
  int tile, part, parts, pad;
  int64_t at;       // of the group's first partial result
  int64_t pad2;
};
struct KvRow {  // a row of the batch
  int shared, parts, M, member;  // shared keys (0: none), the parts they come in, the group's query rows, the row's place among its rows
  int64_t at;
  int64_t pad;
};
struct KvGroup {
  int lead, first, rows, keys, parts, M, item, pad;
  int64_t at;
};

struct KvSharedPlan {
  int *order, *lead, *same, *member;  // the last three between the plan's two kernels
  KvRow* rows;
  KvItem *direct, *tile;
};

struct KvPlanSizes {
  int64_t B, TG, wd, wt, direct, tile, partials, bytes;
};
inline KvPlanSizes kv_plan_sizes(int64_t B, int64_t T, int64_t H, int64_t Hkv, int64_t hd) {
  KvPlanSizes s{};
  s.B = B;
  s.TG = T * (H / Hkv);
  if (s.TG > own_most(hd)) {  // the plain kernels: nothing to plan
    s.bytes = 16;
    return s;
  }
  const int64_t span = direct_rows(static_cast<int>(hd)), tspan = tile_rows(static_cast<int>(hd));
  s.wd = std::max<int64_t>(1, kDirectGroups / Hkv);
  s.wt = std::max<int64_t>(1, kTileGroups / Hkv);
  // sum over groups of tiles x parts, parts at most 1 or the group's share of the workgroups
  s.direct = ceil_div(B * s.TG, span) + B / 2 + s.wd;
  s.tile = B * s.TG >= kTileFrom ? ceil_div(B * s.TG, tspan) + B / 2 + s.wt : 0;
  s.partials = B * s.TG + s.wd * span + (s.tile ? s.wt * tspan : 0);
  const int64_t r4 = (B + 3) / 4 * 4;
  s.bytes = 4 * r4 * 4 + B * static_cast<int64_t>(sizeof(KvRow)) + (s.direct + s.tile) * static_cast<int64_t>(sizeof(KvItem));
  return s;
}
inline KvSharedPlan kv_plan_at(void* p, const KvPlanSizes& s) {
  KvSharedPlan a{};
  char* w = static_cast<char*>(p);
  auto take = [&](int64_t bytes) {
    char* const at = w;
    w += bytes;
    return at;
  };
  const int64_t r4 = (s.B + 3) / 4 * 4;
  for (int** x : {&a.order, &a.lead, &a.same, &a.member}) *x = reinterpret_cast<int*>(take(4 * r4));
  a.rows = reinterpret_cast<KvRow*>(take(s.B * sizeof(KvRow)));
  a.direct = reinterpret_cast<KvItem*>(take(s.direct * sizeof(KvItem)));
  a.tile = reinterpret_cast<KvItem*>(take(s.tile * sizeof(KvItem)));
  return a;
}

// Workgroup b: the first row with row b's leader, how many such rows stand before b, and how many whole blocks before row b's
// start name the same pages in both. Rows that are too short to share anything (emptied ones) belong to no group: they would leave
// the others nothing.
__global__ __launch_bounds__(256) void shared_match_kernel(const int* table, const int* starts, const int* leaders, int B, int width,
                                                           int shift, int unit, KvSharedPlan p) {
  __shared__ int first, differ, rank;
  const int b = blockIdx.x, lead = starts[b] >= unit ? leaders[b] : -1;
  if (threadIdx.x == 0) {
    first = b;
    differ = 0x7fffffff;
    rank = 0;
  }
  __syncthreads();
  if (lead >= 0) {
    int mine = 0, least = 0x7fffffff;
    for (int c = threadIdx.x; c < b; c += 256)
      if (leaders[c] == lead && starts[c] >= unit) {
        least = min(least, c);
        ++mine;
      }
    if (mine != 0) {
      atomicMin(&first, least);
      atomicAdd(&rank, mine);
    }
  }
  __syncthreads();
  const int f = first;
  const int most = lead < 0 ? 0 : min(max(starts[b], 0) >> shift, width);
  const int* const mine = table + static_cast<int64_t>(b) * width;
  const int* const other = table + static_cast<int64_t>(f) * width;
  for (int j0 = 0; j0 < most; j0 += 1024) {
    int at = 0x7fffffff;
#pragma unroll
    for (int k = 3; k >= 0; --k) {
      const int j = j0 + 256 * k + threadIdx.x;
      if (j < most && (mine[j] != other[j] || mine[j] < 0)) at = j;
    }
    if (at != 0x7fffffff) atomicMin(&differ, at);
    __syncthreads();
    const bool done = differ != 0x7fffffff;
    __syncthreads();
    if (done) break;
  }
  if (threadIdx.x == 0) {
    p.same[b] = min(differ, most);
    p.lead[b] = lead < 0 ? -1 : f;
    p.member[b] = rank;
  }
}

struct PlanArgs {
  KvSharedPlan p;
  int B, TG, shift, block, span, tspan;
  int unit;    // shared keys come in multiples of so many: whole steps of either kernel
  int wd, wt, direct, tile;  // workgroups per kv head to aim at, and at most
};

// The sum of `x` over the threads before this one, and of all.
template <typename N>
__device__ inline N plan_scan(N x, N* red, N& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  N s = x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const N y = __shfl_up(s, o, 64);
    if (lane >= o) s += y;
  }
  if (lane == 63) red[wave] = s;
  __syncthreads();
  N before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / 64; ++w) {
    if (w == wave) before = total;
    total += red[w];
  }
  __syncthreads();
  return before + s - x;
}

// One workgroup: groups, their order, their items. Chains of sums over the rows and groups, 8 to 9 us for 8 to 96 rows; a plan serves
// all layers and the steps until the rows change.
__global__ __launch_bounds__(kPlanThreads) void shared_plan_kernel(const PlanArgs a) {
  constexpr int E = kPlanRows / kPlanThreads;
  __shared__ int lead[kPlanRows], many[kPlanRows], blocks[kPlanRows], id[kPlanRows];
  __shared__ int64_t red[kPlanThreads / 64];
  __shared__ KvGroup group[kPlanRows / 2];
  const int tid = threadIdx.x;
  for (int b = tid; b < a.B; b += kPlanThreads) {
    lead[b] = a.p.lead[b];
    many[b] = 0;
    blocks[b] = 0x7fffffff;
  }
  __syncthreads();
  for (int b = tid; b < a.B; b += kPlanThreads)
    if (lead[b] >= 0) {
      atomicAdd(&many[lead[b]], 1);
      atomicMin(&blocks[lead[b]], a.p.same[b]);
    }
  __syncthreads();
  // groups in the order of their first rows: E consecutive rows a thread; rows of groups in the high word, groups in the low
  int64_t n = 0, sum;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int b = E * tid + e;
    const bool is = b < a.B && lead[b] == b && many[b] >= 2 && blocks[b] << a.shift >= a.unit;
    if (b < a.B) id[b] = is ? 0 : -1;
    n += is ? (static_cast<int64_t>(many[b]) << 32) + 1 : 0;
  }
  n = plan_scan(n, red, sum);
  const int groups = static_cast<int>(sum);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int b = E * tid + e;
    if (b < a.B && id[b] == 0) {
      const int g = static_cast<int>(n);
      id[b] = g;
      group[g] = KvGroup{b, static_cast<int>(n >> 32), many[b], (blocks[b] << a.shift) & -a.unit, 1, many[b] * a.TG, 0, 0, 0};
      n += (static_cast<int64_t>(many[b]) << 32) + 1;
    }
  }
  __syncthreads();
  // parts: a group's keys in as many as its share of its kernel's workgroups
  constexpr int F = kPlanRows / 2 / kPlanThreads;  // consecutive groups a thread
  auto big = [&](const KvGroup& x) { return x.M >= kTileFrom && static_cast<int64_t>(x.M) * x.keys >= kTileWork; };
  auto tiles_of = [&](const KvGroup& x) { return big(x) ? (x.M + a.tspan - 1) / a.tspan : (x.M + a.span - 1) / a.span; };
  auto steps_of = [&](const KvGroup& x) { return (x.keys + kStepKeys - 1) / kStepKeys; };
  int64_t cost[2] = {0, 0}, all[2] = {0, 0};
#pragma unroll
  for (int f = 0; f < F; ++f) {
    const int i = F * tid + f;
    if (i < groups) cost[big(group[i])] += static_cast<int64_t>(tiles_of(group[i])) * steps_of(group[i]);
  }
  plan_scan(cost[0], red, all[0]);
  if (a.tile > 0) plan_scan(cost[1], red, all[1]);  // uniform
  // The direct kernel's workgroups: one a CU, two where each then still has kPartSteps steps. 64 rows over 8192 keys, a call: 41.8
  // us with 512, 37.0 with 256; 16 rows over 32768 37, 30; 6 groups of 16 rows over 9000 to 15000 84, 94.
  const int64_t wd = max(static_cast<int64_t>(a.wd / 2), min(static_cast<int64_t>(a.wd), all[0] / kPartSteps));
  int64_t items = 0, partials = 0, total;  // items of the prompt kernel in the high word
#pragma unroll
  for (int f = 0; f < F; ++f) {
    const int i = F * tid + f;
    if (i < groups) {
      KvGroup& x = group[i];
      const int steps = steps_of(x);
      // a part has a step for each of the direct kernel's waves, or two tiles of the prompt kernel's
      const int64_t share = (big(x) ? a.wt : wd) * steps / all[big(x)];
      x.parts = static_cast<int>(max(static_cast<int64_t>(1), min(share, static_cast<int64_t>(big(x) ? (steps + 1) / 2 : (steps + 3) / 4))));
      items += static_cast<int64_t>(tiles_of(x) * x.parts) << (big(x) ? 32 : 0);
      partials += static_cast<int64_t>(x.M) * x.parts;
    }
  }
  int64_t first = plan_scan(items, red, total), every;
  partials = plan_scan(partials, red, every);
#pragma unroll
  for (int f = 0; f < F; ++f) {
    const int i = F * tid + f;
    if (i < groups) {
      KvGroup& x = group[i];
      x.at = partials;
      x.item = static_cast<int>(big(x) ? first >> 32 : first);
      partials += static_cast<int64_t>(x.M) * x.parts;
      first += static_cast<int64_t>(tiles_of(x) * x.parts) << (big(x) ? 32 : 0);
    }
  }
  __syncthreads();
  for (int b = tid; b < a.B; b += kPlanThreads) {
    const int l = lead[b], to = l >= 0 ? id[l] : -1, member = a.p.member[b];
    KvRow row{0, 0, 0, 0, 0, 0};
    if (to >= 0) {
      const KvGroup& x = group[to];
      a.p.order[x.first + member] = b;
      row = KvRow{x.keys, x.parts, x.M, member, x.at, 0};
    }
    a.p.rows[b] = row;
  }
  for (int i = tid >> 6; i < groups; i += kPlanThreads / 64) {
    const KvGroup x = group[i];
    const int tiles = tiles_of(x);
    KvItem* const to = (big(x) ? a.p.tile : a.p.direct) + x.item;
    for (int j = tid & 63; j < tiles * x.parts; j += 64) to[j] = KvItem{x.lead, x.first, x.M, x.keys, j % tiles, j / tiles, x.parts, 0, x.at, 0};
  }
  const KvItem none{-1, 0, 0, 0, 0, 0, 0, 0, 0, 0};
  for (int i = static_cast<int>(total & 0xffffffff) + tid; i < a.direct; i += kPlanThreads) a.p.direct[i] = none;
  for (int i = static_cast<int>(total >> 32) + tid; i < a.tile; i += kPlanThreads) a.p.tile[i] = none;
}

struct KvSharedArgs {
  KvAttnArgs a;
  KvSharedPlan p;
  float *so, *sml;     // partial results of the shared part: [Hkv, partials, D] and (m, l)
  int64_t partials;
  int B, direct, own_tiles;  // own_tiles: of a row's own keys
};

// Shared keys of row b: none where its start has fallen behind them since the plan was made.
__device__ inline int shared_keys(int shared, int start) { return shared > 0 && start >= shared ? shared : 0; }

template <int D, int DT>
__device__ inline void put_part(float* po, float* pml, int64_t at, int jd, float M, float sum, const float (&acc)[DT]) {
  if (jd == 0) {
    pml[2 * at] = M;
    pml[2 * at + 1] = sum;
  }
#pragma unroll
  for (int d = 0; d < DT; d += 4)
    *reinterpret_cast<f32x4_t*>(po + at * D + jd + d) = f32x4_t{acc[d], acc[d + 1], acc[d + 2], acc[d + 3]};
}

// The query rows of a group over a part of its shared keys. Every row attends all of them, and they are whole steps: so the loops
// have no masks, which for E4M3 hold 40 registers.
struct KvGroupRows {
  static constexpr bool kWhole = true;
  const KvSharedArgs& x;
  KvItem g;
  const int* trow;
  int h, row0, TG;
  int base, L, s0, s1, first;
  __device__ KvGroupRows(const KvSharedArgs& args, const KvItem& item, int span, int keys) : x(args), g(item) {
    h = blockIdx.x;
    row0 = item.tile * span;
    TG = x.a.T * x.a.G;
    base = 0;
    L = g.keys;
    first = L - 1;
    const int steps = (L + keys - 1) / keys;
    s0 = static_cast<int>(static_cast<int64_t>(steps) * g.part / g.parts);
    s1 = static_cast<int>(static_cast<int64_t>(steps) * (g.part + 1) / g.parts);
    trow = x.a.table + static_cast<int64_t>(g.lead) * x.a.width;
  }
  __device__ bool row(int i, int& pos, const uint16_t*& src) const {
    const int row = row0 + i;
    pos = -1;
    src = x.a.q;
    if (row >= g.M) return false;
    const int m = row / TG, rest = row - m * TG, t = rest / x.a.G, head = rest - t * x.a.G;
    const int b = x.p.order[g.first + m];
    const int count = x.a.counts != nullptr ? min(max(x.a.counts[b], 0), x.a.T) : x.a.T;
    if (t >= count) return false;
    pos = L - 1;
    src = x.a.q + b * x.a.q_sb + t * x.a.q_st + (h * x.a.G + head) * x.a.q_sh;
    return true;
  }
  __device__ bool live(int i) const { return row0 + i < g.M; }
  __device__ void span(int i, int, int& first_, int& last_) const {
    first_ = L - 1;
    last_ = row0 + i < g.M ? L - 1 : -1;
  }
  template <int D, bool BF16, int DT>
  __device__ void put(int i, int jd, float M, float sum, const float (&acc)[DT]) const {
    put_part<D>(x.so, x.sml, h * x.partials + g.at + static_cast<int64_t>(g.part) * g.M + row0 + i, jd, M, sum, acc);
  }
};

// Parts that a row's own keys are cut into: up to nsplit, with a step for every wave.
__device__ inline int own_parts(int steps, int nsplit) { return min(nsplit, max(1, (steps + kAttnWaves - 1) / kAttnWaves)); }

// A row's queries over the keys behind the shared ones.
struct KvTailRows {
  static constexpr bool kWhole = false;
  const KvSharedArgs& x;
  KvSpan sp;
  const int* trow;
  int b, h, part, row0, rows;
  int base, L, s0, s1, first;
  __device__ KvTailRows(const KvSharedArgs& args) : x(args) {}
  __device__ bool begin(int item, int span) {
    const KvAttnArgs& a = x.a;
    h = blockIdx.x;
    rows = a.T * a.G;
    const int per = x.own_tiles * a.nsplit;
    b = item / per;
    const int rest = item - b * per;
    part = rest / x.own_tiles;
    row0 = (rest - part * x.own_tiles) * span;
    if (!kv_span(a, b, row0, span, sp)) return false;
    base = shared_keys(x.p.rows[b].shared, sp.start);
    L = sp.keys;
    first = sp.first;
    const int steps = (max(L - base, 0) + kStepKeys - 1) / kStepKeys, parts = own_parts(steps, a.nsplit);
    if (part >= parts) return false;
    s0 = static_cast<int>(static_cast<int64_t>(steps) * part / parts);
    s1 = static_cast<int>(static_cast<int64_t>(steps) * (part + 1) / parts);
    trow = a.table + static_cast<int64_t>(b) * a.width;
    return true;
  }
  __device__ bool row(int i, int& pos, const uint16_t*& src) const {
    const KvAttnArgs& a = x.a;
    const int row = row0 + i, t = row / a.G;
    const bool ok = row < rows && t < sp.count;
    pos = ok ? sp.position(t) : -1;
    src = a.q + b * a.q_sb + (ok ? t * a.q_st + (h * a.G + row % a.G) * a.q_sh : 0);
    return ok;
  }
  __device__ bool live(int i) const { return row0 + i < rows && (row0 + i) / x.a.G < sp.count; }
  template <int D, bool BF16, int DT>
  __device__ void put(int i, int jd, float M, float sum, const float (&acc)[DT]) const {
    put_part<D>(x.a.po, x.a.pml, ((static_cast<int64_t>(b) * x.a.Hkv + h) * x.a.nsplit + part) * rows + row0 + i, jd, M, sum, acc);
  }
};

// Workgroups (h, i): the items of the small groups and the rows' own keys.
template <int D, int R, bool E4M3, bool BF16>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void kv_shared_direct_kernel(const KvSharedArgs x) {
  __shared__ float sm[kAttnWaves][16], sl[kAttnWaves][16];
  __shared__ __attribute__((aligned(16))) float so[kAttnWaves][16][D + 4];
  constexpr int RG = direct_rows(D) / 16;
  // The shared part first: with one such workgroup a CU, rows of their own fill the other places. (In turn, one and one, the shared
  // part's would lie on every other CU: 43.7 us where this order takes 34.6.)
  const int i = blockIdx.y;
  if (i < x.direct) {
    const KvItem item = x.p.direct[i];
    if (item.lead < 0) return;
    const KvGroupRows rows(x, item, 16 * RG, kStepKeys);
    kv_attn_body<D, RG, E4M3, BF16>(x.a, rows, sm, sl, so);
  } else {
    KvTailRows rows(x);
    if (rows.begin(i - x.direct, 16 * R)) kv_attn_body<D, R, E4M3, BF16>(x.a, rows, sm, sl, so);
  }
}

template <int D, bool E4M3, bool BF16, bool BIG>
__global__ __launch_bounds__(64 * tile_waves(D), D == 256 ? 1 : 2) void kv_shared_tile_kernel(const KvSharedArgs x) {
  const int i = blockIdx.y;
  const KvItem item = x.p.tile[i];
  if (item.lead < 0) return;
  const KvGroupRows rows(x, item, tile_rows(D), 64 * tile_steps(D));
  kv_attn_tile_body<D, E4M3, BF16, BIG>(x.a, rows);
}

// Joins the parts of every (token, head) row: those of its own keys, then those of the shared ones. As kv_attn_join_kernel.
template <int D, bool BF16, int PG>
__global__ __launch_bounds__(256) void kv_shared_join_kernel(const KvSharedArgs x, int span, int64_t total) {
  constexpr int C = D / 4, kRows = 256 / (PG * C), kAhead = 4;
  __shared__ float rm[kRows][PG], rl[kRows][PG];
  __shared__ f32x4_t ro[kRows][PG][C];
  const KvAttnArgs& a = x.a;
  const int rr = threadIdx.x / (PG * C), p = threadIdx.x / C % PG, c = threadIdx.x % C;
  const int64_t id = std::min<int64_t>(static_cast<int64_t>(blockIdx.x) * kRows + rr, total - 1);  // the last row again
  const int rows = a.T * a.G;
  const int row = static_cast<int>(id % rows);
  const int64_t bh = id / rows;
  const int b = static_cast<int>(bh / a.Hkv), h = static_cast<int>(bh % a.Hkv);
  const KvRow info = x.p.rows[b];
  KvSpan sp;
  const bool live = kv_span(a, b, row / span * span, span, sp) && row / a.G < sp.count;
  int own = 0, mine = 0;
  const float *so = x.so, *sml = x.sml;
  int64_t shared_at = 0, M = 0;
  if (live) {
    const int base = shared_keys(info.shared, sp.start);
    own = mine = own_parts((max(sp.keys - base, 0) + kStepKeys - 1) / kStepKeys, a.nsplit);
    if (base > 0) {
      M = info.M;
      shared_at = h * x.partials + info.at + info.member * rows + row;
      mine += info.parts;
    }
  }
  auto part = [&](int s, const float*& po, const float*& pml) {
    if (s < own) {
      const int64_t at = (bh * a.nsplit + s) * rows + row;
      po = a.po + at * D + 4 * c;
      pml = a.pml + 2 * at;
    } else {
      const int64_t at = shared_at + (s - own) * M;
      po = so + at * D + 4 * c;
      pml = sml + 2 * at;
    }
  };
  f32x4_t v[kAhead];
  float m[kAhead], l[kAhead];
#pragma unroll
  for (int u = 0; u < kAhead; ++u) {
    v[u] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    m[u] = -INFINITY;
    l[u] = 0.0f;
    if (p + PG * u < mine) {
      const float *po, *pml;
      part(p + PG * u, po, pml);
      v[u] = *reinterpret_cast<const f32x4_t*>(po);
      m[u] = pml[0];
      l[u] = pml[1];
    }
  }
  float most = -INFINITY;
#pragma unroll
  for (int u = 0; u < kAhead; ++u) most = fmaxf(most, m[u]);
  for (int s = p + PG * kAhead; s < mine; s += PG) {
    const float *po, *pml;
    part(s, po, pml);
    most = fmaxf(most, pml[0]);
  }
  if (c == 0) rm[rr][p] = most;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PG; ++i) most = fmaxf(most, rm[rr][i]);
  float sum = 0.0f;
  f32x4_t acc{0.0f, 0.0f, 0.0f, 0.0f};
  auto add = [&](float ms, float ls, f32x4_t w) {
    const float wt = attn_chunk_weight(ms, most);
    sum = fmaf(ls, wt, sum);
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = fmaf(w[e], wt, acc[e]);
  };
#pragma unroll
  for (int u = 0; u < kAhead; ++u)
    if (p + PG * u < mine) add(m[u], l[u], v[u]);
#pragma unroll 4
  for (int s = p + PG * kAhead; s < mine; s += PG) {
    const float *po, *pml;
    part(s, po, pml);
    add(pml[0], pml[1], *reinterpret_cast<const f32x4_t*>(po));
  }
  ro[rr][p][c] = acc;
  if (c == 0) rl[rr][p] = sum;
  __syncthreads();
  if (p != 0 || !live || static_cast<int64_t>(blockIdx.x) * kRows + rr >= total) return;
  sum = 0.0f;
  acc = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < PG; ++i) {
    sum += rl[rr][i];
    const f32x4_t w = ro[rr][i][c];
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] += w[e];
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;  // no key: zeros
  uint16_t* dst = a.out + ((static_cast<int64_t>(b) * a.T + row / a.G) * a.H + h * a.G + row % a.G) * D + 4 * c;
  const float o0 = acc[0] * inv, o1 = acc[1] * inv, o2 = acc[2] * inv, o3 = acc[3] * inv;
  *reinterpret_cast<u32x2v_t*>(dst) = BF16 ? u32x2v_t{ActBF16::pack_rne(o0, o1), ActBF16::pack_rne(o2, o3)}
                                           : u32x2v_t{ActF16::pack_rne(o0, o1), ActF16::pack_rne(o2, o3)};
}

}  // namespace sqx

using namespace sqx;

#define KV_SHARED_SHAPE(fn)                                                                                                     \
  SQX_REQUIRE(kv_block_ok(block) && (hd == 64 || hd == 128 || hd == 256), SQX_E_ARG,                                            \
              "%s: block=%lld (16, 32, 64 or 128 tokens), head_dim=%lld (64, 128 or 256)", fn, (long long)block, (long long)hd); \
  SQX_REQUIRE(B >= 1 && B <= kPlanRows, SQX_E_ARG, "%s: B=%lld rows (1 to %d)", fn, (long long)B, kPlanRows);                   \
  SQX_REQUIRE(T >= 1 && T < (int64_t(1) << 20) && Hkv >= 1 && Hkv <= 1024 && H >= 1 && H % Hkv == 0 && H <= 8192, SQX_E_ARG,     \
              "%s: bad shape (T=%lld from 1 and below 2^20, H=%lld up to 8192 and a multiple of Hkv=%lld, up to 1024)", fn,       \
              (long long)T, (long long)H, (long long)Hkv);                                                                     \
  SQX_REQUIRE(width >= 1 && width * block < (int64_t(1) << 30), SQX_E_ARG, "%s: a table of %lld blocks (at least 1; positions below 2^30)", \
              fn, (long long)width)

static bool kv_shared_ok(int64_t B, int64_t T, int64_t H, int64_t Hkv, int64_t hd, int64_t block, int64_t width) {
  return B >= 1 && B <= kPlanRows && T >= 1 && T < (int64_t(1) << 20) && Hkv >= 1 && H >= 1 && H % Hkv == 0 && kv_block_ok(block) &&
         (hd == 64 || hd == 128 || hd == 256) && width >= 1;
}

extern "C" int64_t sqx_kvshared_plan_bytes(int64_t B, int64_t T, int64_t H, int64_t Hkv, int64_t hd) {
  return kv_shared_ok(B, T, H, Hkv, hd, 16, 1) ? kv_plan_sizes(B, T, H, Hkv, hd).bytes : 0;
}

extern "C" int sqx_kvshared_plan(const int* table, const int* starts, const int* leaders, int64_t B, int64_t T, int64_t H, int64_t Hkv,
                                 int64_t hd, int64_t block, int64_t width, void* plan, int64_t plan_bytes, sqx_stream_t stream) {
  const char* fn = "sqx_kvshared_plan";
  KV_SHARED_SHAPE(fn);
  SQX_REQUIRE(table && starts && leaders, SQX_E_ARG, "%s: null pointer", fn);
  const KvPlanSizes z = kv_plan_sizes(B, T, H, Hkv, hd);
  SQX_REQUIRE(plan != nullptr && plan_bytes >= z.bytes && al16(plan), SQX_E_SPACE, "%s: %lld bytes of 16-byte aligned plan needed, %lld given",
              fn, (long long)z.bytes, (long long)plan_bytes);
  if (z.TG > own_most(hd)) return SQX_OK;
  PlanArgs a{};
  a.p = kv_plan_at(plan, z);
  a.B = static_cast<int>(B); a.TG = static_cast<int>(z.TG); a.shift = kv_shift(block); a.block = static_cast<int>(block);
  a.unit = kStepKeys * tile_steps(static_cast<int>(hd));
  a.span = direct_rows(static_cast<int>(hd)); a.tspan = tile_rows(static_cast<int>(hd));
  a.wd = static_cast<int>(z.wd); a.wt = static_cast<int>(z.wt); a.direct = static_cast<int>(z.direct); a.tile = static_cast<int>(z.tile);
  hipLaunchKernelGGL(shared_match_kernel, dim3(static_cast<unsigned>(B)), dim3(256), 0, as_stream(stream), table, starts, leaders, a.B,
                     static_cast<int>(width), a.shift, a.unit, a.p);
  hipLaunchKernelGGL(shared_plan_kernel, dim3(1), dim3(kPlanThreads), 0, as_stream(stream), a);
  SQX_LAUNCH_CHECK(fn);
  return SQX_OK;
}

extern "C" int64_t sqx_kvshared_attention_workspace_bytes(int64_t B, int64_t T, int64_t H, int64_t Hkv, int64_t hd, int64_t block,
                                                          int64_t width) {
  if (!kv_shared_ok(B, T, H, Hkv, hd, block, width)) return 0;
  const int64_t rows = T * (H / Hkv);
  if (rows > own_most(hd)) return sqx_kvblock_attention_workspace_bytes(B, T, H, Hkv, hd, block, width);
  const int64_t own = B * Hkv * kv_attn_plan(B, rows, Hkv, hd, width * block).splits * rows;
  return (own + Hkv * kv_plan_sizes(B, T, H, Hkv, hd).partials) * (hd + 2) * 4;
}

extern "C" int sqx_kvshared_attention(const void* q, int dtype, int64_t q_sb, int64_t q_st, int64_t q_sh, int fmt, const void* k_codes,
                                      const void* v_codes, const float* k_scale, const float* v_scale, const int* table,
                                      const int* starts, const int* counts, int64_t B, int64_t T, int64_t H, int64_t Hkv, int64_t hd,
                                      int64_t block, int64_t pages, int64_t width, float scale, const void* plan, int64_t plan_bytes,
                                      void* out, void* ws, int64_t ws_bytes, sqx_stream_t stream) {
  const char* fn = "sqx_kvshared_attention";
  KV_SHAPE(fn);
  KV_SHARED_SHAPE(fn);
  SQX_REQUIRE(dtype != SQX_DTYPE_F32, SQX_E_ARG, "%s: queries must be BF16 or F16", fn);
  SQX_REQUIRE(scale > 0.0f && scale <= 1.0e30f, SQX_E_ARG, "%s: scale must be positive and at most 1e30", fn);
  SQX_REQUIRE(q_sb >= 0 && q_st >= 0 && q_sh >= 0 && (q_sb | q_st | q_sh) % 8 == 0, SQX_E_ARG,
              "%s: strides must be multiples of 8 elements", fn);
  SQX_REQUIRE(q && k_codes && v_codes && k_scale && v_scale && table && starts && out, SQX_E_ARG, "%s: null pointer", fn);
  SQX_REQUIRE(al16(q) && al16(k_codes) && al16(v_codes) && al16(out), SQX_E_ARG, "%s: q, codes and out must be 16-byte aligned", fn);
  const KvPlanSizes z = kv_plan_sizes(B, T, H, Hkv, hd);
  SQX_REQUIRE(plan != nullptr && plan_bytes >= z.bytes && al16(plan), SQX_E_SPACE, "%s: %lld bytes of 16-byte aligned plan needed, %lld given",
              fn, (long long)z.bytes, (long long)plan_bytes);
  const int64_t need = sqx_kvshared_attention_workspace_bytes(B, T, H, Hkv, hd, block, width);
  SQX_REQUIRE(need == 0 || (ws != nullptr && ws_bytes >= need && al16(ws)), SQX_E_SPACE,
              "%s: %lld bytes of 16-byte aligned workspace needed, %lld given", fn, (long long)need, (long long)ws_bytes);
  const int64_t G = H / Hkv, rows = T * G;
  // A chunk of a prompt reads its keys once for all its rows already.
  if (rows > own_most(hd))
    return sqx_kvblock_attention(q, dtype, q_sb, q_st, q_sh, fmt, k_codes, v_codes, k_scale, v_scale, table, starts, counts, B, T, H, Hkv,
                                 hd, block, pages, width, scale, out, ws, ws_bytes, stream);
  const KvAttnPlan own = kv_attn_plan(B, rows, Hkv, hd, width * block);
  const int ns = own.splits;
  KvSharedArgs x{};
  KvAttnArgs& a = x.a;
  a.q = static_cast<const uint16_t*>(q);
  a.q_sb = q_sb; a.q_st = q_st; a.q_sh = q_sh;
  a.kc = static_cast<const uint8_t*>(k_codes); a.vc = static_cast<const uint8_t*>(v_codes);
  a.ks = k_scale; a.vs = v_scale;
  a.table = table; a.starts = starts; a.counts = counts;
  a.out = static_cast<uint16_t*>(out);
  const int64_t parts = B * Hkv * ns * rows, shared = Hkv * z.partials;
  a.po = static_cast<float*>(ws);
  x.so = a.po + parts * hd;
  a.pml = x.so + shared * hd;
  x.sml = a.pml + 2 * parts;
  a.T = static_cast<int>(T); a.H = static_cast<int>(H); a.Hkv = static_cast<int>(Hkv); a.G = static_cast<int>(G);
  a.width = static_cast<int>(width); a.pages = static_cast<int>(pages); a.block = static_cast<int>(block);
  a.shift = kv_shift(block); a.nsplit = ns;
  a.qscale = static_cast<float>(static_cast<double>(scale) * 1.4426950408889634);
  x.p = kv_plan_at(const_cast<void*>(plan), z);
  x.partials = z.partials;
  x.B = static_cast<int>(B); x.direct = static_cast<int>(z.direct); x.own_tiles = own.tiles;
  const int64_t items = z.direct + B * own.tiles * ns;
  SQX_REQUIRE(items < 65536 && z.tile < 65536, SQX_E_ARG, "%s: %lld rows of %lld tokens are too many for one call", fn, (long long)B, (long long)T);
  const hipStream_t s = as_stream(stream);
  const unsigned heads = static_cast<unsigned>(Hkv);
  with_head(hd, [&](auto dd) {
    constexpr int D = decltype(dd)::value;
    auto go = [&](auto e4, auto bf) {
      constexpr bool E = decltype(e4)::value, BF = decltype(bf)::value;
      if (z.tile > 0 && B * rows * width * block >= kTileWork) {  // else no group is that large; a wide table alone gives no items
        const dim3 grid(heads, static_cast<unsigned>(z.tile));
        if (block >= kStepKeys) hipLaunchKernelGGL((kv_shared_tile_kernel<D, E, BF, true>), grid, dim3(64 * tile_waves(D)), 0, s, x);
        else hipLaunchKernelGGL((kv_shared_tile_kernel<D, E, BF, false>), grid, dim3(64 * tile_waves(D)), 0, s, x);
      }
      const dim3 grid(heads, static_cast<unsigned>(items));
      if (own.R == 1) hipLaunchKernelGGL((kv_shared_direct_kernel<D, 1, E, BF>), grid, dim3(256), 0, s, x);
      else if constexpr (D < 256) hipLaunchKernelGGL((kv_shared_direct_kernel<D, 2, E, BF>), grid, dim3(256), 0, s, x);
      const int64_t total = B * Hkv * rows;
      auto join = [&](auto pg) {
        constexpr int PG = decltype(pg)::value;
        hipLaunchKernelGGL((kv_shared_join_kernel<D, BF, PG>), dim3(static_cast<unsigned>(ceil_div(total, 1024 / (PG * D)))), dim3(256), 0, s, x,
                           16 * own.R, total);
      };
      if (total <= 1024) join(std::integral_constant<int, D == 256 ? 4 : 8>{});
      else join(std::integral_constant<int, 2>{});
    };
    auto with_type = [&](auto e4) {
      if (dtype == SQX_DTYPE_BF16) go(e4, std::true_type{});
      else go(e4, std::false_type{});
    };
    if (fmt == SQX_KV_E4M3) with_type(std::true_type{});
    else with_type(std::false_type{});
  });
  SQX_LAUNCH_CHECK(fn);
  return SQX_OK;
}
