// Pages of the block-scaled KV cache (layout: sqx_kvblock.h; here with all layers of a model one behind the other): who holds
// them, and their copies. refs[p] counts the table entries that name page p; a page with none is free.
//
// All bookkeeping is whole numbers on the device, so a call can be captured in a graph and waits for nothing on the host.
// Counts change by atomic additions only where their order cannot show, and a free page is always the lowest one, so equal
// calls give equal tables. A call that hands out pages does all of it or, where the pool is too small, nothing.
//
// Two kinds of launches: small ones over tables and counts, bound by the latency of a launch and of two or three dependent
// loads each, and one that copies the pages, bound by HBM. us of the kernels: fork of 8 rows (7 pages of 4 layers copied) 5.4
// and 5.5; of 64 rows of beams (260 MB read and written) 7.4 to 8.4 and 54 to 60, 4.3 to 4.8 TB/s; release and reservation for 96 rows 3.2 and
// 8.9, 8.9 for the 46 MB copied; a pool of 1100 pages of 32 layers, 128 KiB each, compacted (2.1 GB) 434, 4.9 TB/s, with 5
// before it for each of the counts, their sums and the plan.
//
// Rows are looked at by many workgroups, but pages are dealt out by one: the place of a page in the list of free ones depends on
// all before it, and one workgroup that reads 64 KiB of counts a step is through a pool of 16384 pages in one.
#include "sqx_kvblock.h"

namespace sqx {

constexpr int kPlan = 1024;      // threads of a workgroup that scans the pool alone
constexpr int kScan = 16;        // pages of a thread, a pass over the pool
constexpr int kCopyUnits = 1024;  // 16-byte units of a workgroup's piece, four a thread in flight
constexpr int kCopyGroups = 2048;
// What one workgroup plans: eight entries of the tables a thread in a fork; at most sixteen in a reservation, which looks at few.
constexpr int kSmallRows = kPlan, kSmallEntries = 8192, kSmallPages = 8192, kSmallReserve = 16384;

struct KvPool {
  uint8_t *kc, *vc;  // [L, pages, unit16 * 16 bytes]
  float *ks, *vs;    // [L, pages, Hkv]
  int L, Hkv, pages;
  int units;  // 16-byte units of a page's keys, and of its values
};

struct int4a { int v[4]; };  // four ints at any multiple of four bytes

// The exclusive sum of one int a thread over a workgroup of 64 W threads, and the total; `red` holds W ints.
template <int W>
__device__ inline int block_scan(int x, int* red, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int s = x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(s, o, 64);
    if (lane >= o) s += y;
  }
  if (lane == 63) red[wave] = s;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    const int r = red[w];
    before += w < wave ? r : 0;
    total += r;
  }
  __syncthreads();  // red may be written again
  return before + s - x;
}

// Copies pages src[i] -> dst[i], i < n, in all layers. A workgroup's piece is kCopyUnits units of one page, or several small
// pages; pieces are dealt out in a loop, since the count is known on the device only. Pairs that name no page, or the same one
// twice, are left out. Stores that pass the caches by leave these to the loads: 500 MB (read and written) of pages of 64 KiB in
// 99 us, 5.3 TB/s, where plain stores take 115; 2 GiB in 437 and 448; pages of 2 KiB, 250 MB, in 39 and 57. Loads that pass them by
// too take 112, 434 and 61; twice as many workgroups change nothing.
__device__ inline void copy_pages(const KvPool& p, const int* src, const int* dst, uint32_t n, uint32_t group, uint32_t groups) {
  const uint32_t units = p.units, per = max(kCopyUnits / units, 1u);      // per: jobs (pair, layer, keys or values) of a piece
  const uint32_t pieces = (units + kCopyUnits - 1) / kCopyUnits;          // of a job
  const uint32_t jobs = n * p.L * 2, work = pieces > 1 ? jobs * pieces : (jobs + per - 1) / per;  // below 2^31
  for (uint32_t w = group; w < work; w += groups) {
    const uint32_t job0 = pieces > 1 ? w / pieces : w * per, unit0 = pieces > 1 ? (w - job0 * pieces) * kCopyUnits : 0;
    u32x4_t x[4];
    u32x4_t* to[4];
    const float* sc_from[4];
    float* sc_to[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t e = threadIdx.x + 256 * k;
      const uint32_t j = pieces > 1 ? 0 : e / units, unit = unit0 + e - j * units, job = job0 + j;
      to[k] = nullptr;
      sc_to[k] = nullptr;
      if (j >= per || job >= jobs || unit >= units) continue;
      const uint32_t pair = job / (2 * p.L), rest = job - pair * (2 * p.L);
      const int s = src[pair], d = dst[pair];
      if (s < 0 || s >= p.pages || d < 0 || d >= p.pages || s == d) continue;
      u32x4_t* const base = reinterpret_cast<u32x4_t*>(rest & 1 ? p.vc : p.kc);
      const int64_t at = static_cast<int64_t>(rest >> 1) * p.pages;
      x[k] = base[(at + s) * units + unit];
      to[k] = base + (at + d) * units + unit;
      if (unit < static_cast<uint32_t>(p.Hkv)) {  // a page has more units than heads
        float* const sc = rest & 1 ? p.vs : p.ks;
        sc_from[k] = sc + (at + s) * p.Hkv + unit;
        sc_to[k] = sc + (at + d) * p.Hkv + unit;
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (to[k] != nullptr) __builtin_nontemporal_store(x[k], to[k]);
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (sc_to[k] != nullptr) *sc_to[k] = *sc_from[k];
  }
}

__global__ __launch_bounds__(256) void kv_copy_kernel(const KvPool p, const int* src, const int* dst, const int* count, int most) {
  copy_pages(p, src, dst, static_cast<uint32_t>(count != nullptr ? *count : most), blockIdx.x, gridDim.x);
}

// The lowest free pages of counts[0 .. pages), ascending, into list[0 .. want); returns how many there are, up to want. A
// workgroup of kPlan threads, all of which call it.
__device__ inline int free_pages(const int* counts, int pages, int want, int* list, int* red) {
  int found = 0;
  for (int64_t base = 0; base < pages && found < want; base += kPlan * kScan) {
    const int64_t mine = base + threadIdx.x * kScan;
    int4a c[kScan / 4];
    int n = 0;
    uint32_t is = 0;
    if (mine + kScan <= pages) {
#pragma unroll
      for (int i = 0; i < kScan / 4; ++i) c[i] = *reinterpret_cast<const int4a*>(counts + mine + 4 * i);
#pragma unroll
      for (int i = 0; i < kScan; ++i) is |= (c[i / 4].v[i % 4] == 0 ? 1u : 0u) << i;
    } else {
      for (int i = 0; i < kScan; ++i)
        if (mine + i < pages && counts[mine + i] == 0) is |= 1u << i;
    }
    n = __popc(is);
    int total;
    int at = found + block_scan<kPlan / 64>(n, red, total);
    while (is != 0 && at < want) {
      const int i = __ffs(is) - 1;
      is &= is - 1;
      list[at++] = static_cast<int>(mine) + i;
    }
    found += total;
  }
  return min(found, want);
}

// ------------------------------------------------------------------------------------------------ fork
struct ForkArgs {
  const int* parents;
  int *table, *lengths, *refs;
  // workspace: the tables as they will be, what a row's open block is copied from (-1: not), the copies and their number
  int *table2, *lengths2, *refs2, *need, *src, *dst, *free, *count;
  int* ok;
  int B, width, pages, block, shift;
};

__global__ __launch_bounds__(256) void fork_begin_kernel(const ForkArgs a) {
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < a.pages; i += static_cast<int64_t>(gridDim.x) * 256)
    a.refs2[i] = a.refs[i];
}

// Workgroup (chunk, b): 256 entries of row b's new table, and the counts that they change. The open block of a parent that does
// not go on from itself stays with the first row that goes on from it.
__global__ __launch_bounds__(256) void fork_rows_kernel(const ForkArgs a) {
  const int b = blockIdx.y, j = blockIdx.x * 256 + threadIdx.x;
  const int p = a.parents[b];
  const int64_t row = static_cast<int64_t>(b) * a.width;
  auto page = [&](int64_t at) {
    const int x = a.table[at];
    return x >= 0 && x < a.pages ? x : -1;
  };
  if (p == b) {
    if (blockIdx.x == 0 && threadIdx.x == 0) {
      a.need[b] = -1;
      a.lengths2[b] = a.lengths[b];
    }
    if (j < a.width) a.table2[row + j] = a.table[row + j];
    return;
  }
  const bool none = p < 0 || p >= a.B;
  const int most = a.width << a.shift;  // below 2^30
  const int len = none ? 0 : min(max(a.lengths[p], 0), most);
  const int blocks = (len + a.block - 1) >> a.shift, open = (len & (a.block - 1)) != 0 ? blocks - 1 : -1;
  bool keeps = false;
  if (open >= 0 && a.parents[p] != p) {  // uniform over the workgroup
    bool before = false;
    for (int c = threadIdx.x; c < b; c += 256) before |= a.parents[c] == p;
    keeps = __syncthreads_or(before) == 0;
  }
  const int64_t from = static_cast<int64_t>(none ? 0 : p) * a.width;
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    a.need[b] = open >= 0 && !keeps ? page(from + open) : -1;
    a.lengths2[b] = len;
  }
  if (j >= a.width) return;
  const int had = page(row + j), now = j < blocks && (j != open || keeps) ? page(from + j) : -1;
  a.table2[row + j] = now;  // of a copied block until its page is known
  if (had != now) {
    if (had >= 0) atomicAdd(a.refs2 + had, -1);
    if (now >= 0) atomicAdd(a.refs2 + now, 1);
  }
}

// One workgroup: a page for every copy, in the order of the rows.
__global__ __launch_bounds__(kPlan) void fork_assign_kernel(const ForkArgs a) {
  __shared__ int red[kPlan / 64];
  int n = 0;
  for (int b0 = 0; b0 < a.B; b0 += kPlan) {
    const int b = b0 + threadIdx.x, s = b < a.B ? a.need[b] : -1;
    int total;
    const int at = n + block_scan<kPlan / 64>(s >= 0, red, total);
    if (s >= 0) {
      a.src[at] = s;
      a.dst[at] = b;  // the row, until it has a page
    }
    n += total;
  }
  const int found = free_pages(a.refs2, a.pages, n, a.free, red);
  __syncthreads();  // src, dst and free are read by other threads than those that wrote them
  const bool ok = found == n;
  if (ok) {
    for (int i = threadIdx.x; i < n; i += kPlan) {
      const int b = a.dst[i], page = a.free[i];
      a.table2[static_cast<int64_t>(b) * a.width + ((a.lengths2[b] - 1) >> a.shift)] = page;
      a.refs2[page] = 1;
      a.dst[i] = page;
    }
  }
  if (threadIdx.x == 0) {
    *a.count = ok ? n : 0;
    *a.ok = ok ? 1 : 0;
  }
}

// The three kernels above in one workgroup, the counts in LDS: for up to kSmallRows rows, kSmallEntries entries and kSmallPages pages.
// 8 rows, 392 entries: 5.2 us, and the call 16.6 where the three take 1.9, 3.3 and 4.2, and it 23.0; 64 rows, 1536 entries: 7.4,
// 66.5 for 4.7, 4.6, 5.2 and 70.0.

__global__ __launch_bounds__(kPlan) void fork_small_kernel(const ForkArgs a) {
  __shared__ int refs[kSmallPages], free[kSmallRows], red[kPlan / 64];
  __shared__ int parent[kSmallRows], taker[kSmallRows];  // taker: the first row that goes on from this one
  __shared__ int4a todo[kSmallRows];                     // parent (-1: the row stays), blocks, the block without a page of the parent's
  const int b = threadIdx.x;
  const int p = b < a.B ? a.parents[b] : -1;
  parent[b] = p;
  taker[b] = 0x7fffffff;
  for (int i = b; i < a.pages; i += kPlan) refs[i] = a.refs[i];
  __syncthreads();
  const bool other = b < a.B && p != b, none = p < 0 || p >= a.B;
  if (other && !none) atomicMin(&taker[p], b);
  __syncthreads();
  auto page = [&](int64_t at) {
    const int x = a.table[at];
    return x >= 0 && x < a.pages ? x : -1;
  };
  int need = -1;
  if (b < a.B) {
    const int len = !other ? a.lengths[b] : none ? 0 : min(max(a.lengths[p], 0), a.width << a.shift);
    int4a x{{-1, 0, -1, 0}};
    if (other) {
      const int blocks = (len + a.block - 1) >> a.shift;
      const int open = (len & (a.block - 1)) != 0 && (parent[p] == p || taker[p] != b) ? blocks - 1 : -1;
      need = open >= 0 ? page(static_cast<int64_t>(p) * a.width + open) : -1;
      x = int4a{{none ? 0 : p, blocks, open, 0}};
    }
    a.lengths2[b] = len;
    todo[b] = x;
  }
  __syncthreads();
#pragma unroll 4
  for (int i = b; i < a.B * a.width; i += kPlan) {
    const int r = i / a.width, j = i - r * a.width;
    const int4a x = todo[r];
    const int was = a.table[i];
    int now = was;
    if (x.v[0] >= 0) {
      const int had = was >= 0 && was < a.pages ? was : -1;
      now = j < x.v[1] && j != x.v[2] ? page(x.v[0] * a.width + j) : -1;
      if (had != now) {
        if (had >= 0) atomicAdd(&refs[had], -1);
        if (now >= 0) atomicAdd(&refs[now], 1);
      }
    }
    a.table2[i] = now;
  }
  int n;
  const int at = block_scan<kPlan / 64>(need >= 0, red, n);  // has a barrier: counts and tables are there behind it
  const bool ok = free_pages(refs, a.pages, n, free, red) == n;
  __syncthreads();
  if (ok) {
    if (need >= 0) {
      const int to = free[at];
      a.src[at] = need;
      a.dst[at] = to;
      a.table2[b * a.width + todo[b].v[2]] = to;
      refs[to] = 1;
    }
    __syncthreads();
    for (int i = b; i < a.pages; i += kPlan) a.refs2[i] = refs[i];
  }
  if (b == 0) {
    *a.count = ok ? n : 0;
    *a.ok = ok ? 1 : 0;
  }
}

// Takes the new tables over and copies.
__global__ __launch_bounds__(256) void fork_end_kernel(const ForkArgs a, const KvPool p) {
  if (*a.ok == 0) return;
  const int64_t step = static_cast<int64_t>(gridDim.x) * 256, at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  for (int64_t i = at; i < static_cast<int64_t>(a.B) * a.width; i += step) a.table[i] = a.table2[i];
  for (int64_t i = at; i < a.pages; i += step) a.refs[i] = a.refs2[i];
  for (int64_t i = at; i < a.B; i += step) a.lengths[i] = a.lengths2[i];
  copy_pages(p, a.src, a.dst, *a.count, blockIdx.x, gridDim.x);
}

// ------------------------------------------------------------------------------------------------ reserve
struct ReserveArgs {
  int* table;
  const int *starts, *counts;
  int* refs;
  uint8_t* kind;  // [B, width]: 0 the block stays as it is, 1 it gets a page, 2 it gets a copy of its page
  int *per, *first, *free, *src, *dst, *count;  // per row, its first page's place; the pages handed out; the copies, their number
  int* ok;
  int B, width, pages, block, shift, most;  // most: pages that a call can hand out
};

// The blocks [lo, hi) of row b that its next tokens lie in.
__device__ inline void touched(const ReserveArgs& a, int b, int& lo, int& hi) {
  const int s = a.starts[b];
  const int64_t end = min(static_cast<int64_t>(s) + max(a.counts[b], 0), static_cast<int64_t>(a.width) << a.shift);
  const bool some = s >= 0 && end > s;
  lo = some ? s >> a.shift : 0;
  hi = some ? static_cast<int>((end + a.block - 1) >> a.shift) : 0;
}

__global__ __launch_bounds__(256) void reserve_count_kernel(const ReserveArgs a) {
  __shared__ int red[4];
  const int b = blockIdx.x;
  int lo, hi, n = 0;
  touched(a, b, lo, hi);
  for (int j = lo + threadIdx.x; j < hi; j += 256) {
    const int64_t at = static_cast<int64_t>(b) * a.width + j;
    const int page = a.table[at];
    const bool has = page >= 0 && page < a.pages;
    const int kind = !has ? 1 : a.refs[page] > 1 ? 2 : 0;
    a.kind[at] = static_cast<uint8_t>(kind);
    n += kind != 0;
  }
  int total;
  block_scan<4>(n, red, total);
  if (threadIdx.x == 0) a.per[b] = total;
}

__global__ __launch_bounds__(kPlan) void reserve_assign_kernel(const ReserveArgs a) {
  __shared__ int red[kPlan / 64];
  int64_t n = 0;
  for (int b0 = 0; b0 < a.B; b0 += kPlan) {
    const int b = b0 + threadIdx.x, c = b < a.B ? a.per[b] : 0;
    int total;
    const int before = block_scan<kPlan / 64>(c, red, total);
    if (b < a.B) a.first[b] = static_cast<int>(min(n + before, static_cast<int64_t>(a.most)));
    n += total;
  }
  const bool fits = n <= a.most;  // uniform
  const int found = fits ? free_pages(a.refs, a.pages, static_cast<int>(n), a.free, red) : 0;
  if (threadIdx.x == 0) {
    *a.count = 0;
    *a.ok = fits && found == n ? 1 : 0;
  }
}

__global__ __launch_bounds__(256) void reserve_rows_kernel(const ReserveArgs a) {
  __shared__ int red[4];
  if (*a.ok == 0) return;
  const int b = blockIdx.x;
  int lo, hi;
  touched(a, b, lo, hi);
  int next = a.first[b];
  for (int j0 = lo; j0 < hi; j0 += 256) {
    const int j = j0 + threadIdx.x;
    const int64_t at = static_cast<int64_t>(b) * a.width + j;
    const int kind = j < hi ? a.kind[at] : 0;
    int total;
    const int i = next + block_scan<4>(kind != 0, red, total);
    if (kind != 0) {
      const int page = a.free[i];
      if (kind == 2) {
        const int had = a.table[at];
        atomicAdd(a.refs + had, -1);
        const int c = atomicAdd(a.count, 1);  // the copies' order does not show
        a.src[c] = had;
        a.dst[c] = page;
      }
      a.table[at] = page;
      a.refs[page] = 1;
    }
    next += total;
  }
}

// The three kernels above in one workgroup, for up to kSmallRows rows and kSmallReserve entries: the blocks that tokens lie in stand
// one behind the other, row after row, a thread for each, kPlan at a time. 96 rows, some 600 blocks: 8.4 us where the three take 3.5,
// 4.4 and 4.0 and two more launches; with the entries dealt out to the threads in equal runs, looked at or not, 13.8.
__global__ __launch_bounds__(kPlan) void reserve_small_kernel(const ReserveArgs a) {
  __shared__ int begin[kSmallRows], from[kSmallRows], red[kPlan / 64], copies;  // begin: blocks of the rows before
  const int tid = threadIdx.x;
  int lo = 0, hi = 0, blocks;
  if (tid < a.B) touched(a, tid, lo, hi);
  if (tid == 0) copies = 0;
  begin[tid] = block_scan<kPlan / 64>(hi - lo, red, blocks);
  from[tid] = lo;
  __syncthreads();
  auto entry = [&](int t) {
    int r = 0;  // the last row that begins at t or before it: it holds t, as rows of no blocks begin where the next does
#pragma unroll
    for (int step = kSmallRows / 2; step > 0; step >>= 1) r += begin[r + step] <= t ? step : 0;
    return r * a.width + from[r] + t - begin[r];
  };
  int n = 0;
  uint32_t fresh = 0, copied = 0;  // bit k: of block kPlan k + tid
  for (int k = 0; k * kPlan < blocks; ++k) {
    const int t = k * kPlan + tid;
    int kind = 0;
    if (t < blocks) {
      const int page = a.table[entry(t)];
      kind = page < 0 || page >= a.pages ? 1 : a.refs[page] > 1 ? 2 : 0;
      fresh |= (kind == 1 ? 1u : 0u) << k;
      copied |= (kind == 2 ? 1u : 0u) << k;
    }
    n += __syncthreads_count(kind != 0);
  }
  const bool ok = n <= a.most && free_pages(a.refs, a.pages, n, a.free, red) == n;
  __syncthreads();  // the free pages are read by other threads than those that wrote them
  if (ok) {
    int next = 0;
    for (int k = 0; k * kPlan < blocks; ++k) {
      int total;
      const int rank = next + block_scan<kPlan / 64>((fresh | copied) >> k & 1u, red, total);
      next += total;
      if (((fresh | copied) >> k & 1u) == 0) continue;
      const int i = entry(k * kPlan + tid), page = a.free[rank];
      if ((copied >> k) & 1u) {
        const int had = a.table[i], c = atomicAdd(&copies, 1);  // the copies' order does not show
        atomicAdd(a.refs + had, -1);
        a.src[c] = had;
        a.dst[c] = page;
      }
      a.table[i] = page;
      a.refs[page] = 1;
    }
  }
  __syncthreads();
  if (tid == 0) {
    *a.count = copies;
    *a.ok = ok ? 1 : 0;
  }
}

// ------------------------------------------------------------------------------------------------ free
__global__ __launch_bounds__(256) void free_rows_kernel(const int* keep, int* table, int* lengths, int* refs, int width, int pages,
                                                        int block, int shift) {
  const int b = blockIdx.y;
  const int k = max(keep[b], 0);
  const int j = blockIdx.x * 256 + threadIdx.x;
  if (j == 0) lengths[b] = min(lengths[b], k);
  if (j >= width || j < (k >> shift) + ((k & (block - 1)) != 0)) return;
  const int64_t at = static_cast<int64_t>(b) * width + j;
  const int page = table[at];
  if (page >= 0 && page < pages) atomicAdd(refs + page, -1);
  table[at] = -1;
}

// ------------------------------------------------------------------------------------------------ compact
constexpr int kTile = kPlan * 4;  // pages of a workgroup that counts

struct CompactArgs {
  int *table, *refs, *moved, *live;
  int *tiles;      // pages in use of every tile, then those before it
  int *src, *dst;  // [pages / 2 + 1]
  int* count;
  int pages, ntiles;
  int64_t entries;
};

// Bits of the four pages from `at` that are in use.
__device__ inline uint32_t used4(const int* refs, int64_t at, int pages) {
  uint32_t is = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (at + i < pages && refs[at + i] > 0) is |= 1u << i;
  return is;
}

__global__ __launch_bounds__(kPlan) void compact_count_kernel(const CompactArgs a) {
  __shared__ int red[kPlan / 64];
  const uint32_t is = used4(a.refs, static_cast<int64_t>(blockIdx.x) * kTile + 4 * threadIdx.x, a.pages);
  int total;
  block_scan<kPlan / 64>(__popc(is), red, total);
  if (threadIdx.x == 0) a.tiles[blockIdx.x] = total;
}

__global__ __launch_bounds__(kPlan) void compact_scan_kernel(const CompactArgs a) {
  __shared__ int red[kPlan / 64];
  int n = 0;
  for (int t0 = 0; t0 < a.ntiles; t0 += kPlan) {
    const int t = t0 + threadIdx.x, c = t < a.ntiles ? a.tiles[t] : 0;
    int total;
    const int before = block_scan<kPlan / 64>(c, red, total);
    if (t < a.ntiles) a.tiles[t] = n + before;
    n += total;
  }
  if (threadIdx.x == 0) *a.live = n;
}

// Page p in use, the r-th of these: it stays if p < live, else it is the (r - r_live)-th that moves, r_live those in use below
// `live`. A free page p < live is the (p - r)-th hole; there are as many holes as pages that move.
__global__ __launch_bounds__(kPlan) void compact_plan_kernel(const CompactArgs a) {
  __shared__ int red[kPlan / 64];
  const int live = *a.live;
  int stay;
  {  // pages in use below `live`: those before its tile, and in it
    const int t = live / kTile;
    const int64_t at = static_cast<int64_t>(t) * kTile + 4 * threadIdx.x;
    uint32_t is = used4(a.refs, at, live);
    block_scan<kPlan / 64>(__popc(is), red, stay);
    stay += t < a.ntiles ? a.tiles[t] : live;
  }
  const int64_t at = static_cast<int64_t>(blockIdx.x) * kTile + 4 * threadIdx.x;
  const uint32_t is = used4(a.refs, at, a.pages);
  int total;
  int r = a.tiles[blockIdx.x] + block_scan<kPlan / 64>(__popc(is), red, total);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int p = static_cast<int>(at) + i;
    if (at + i >= a.pages) break;
    const bool used = (is >> i) & 1u;
    a.moved[p] = used ? p : -1;  // of a page that moves until its place is known
    if (used && p >= live) a.src[r - stay] = p;
    if (!used && p < live) a.dst[p - r] = p;
    r += used;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.count = live - stay;
}

__global__ __launch_bounds__(256) void compact_move_kernel(const CompactArgs a, const KvPool p) {
  const int n = *a.count;
  const int64_t step = static_cast<int64_t>(gridDim.x) * 256;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += step) {
    const int s = a.src[i], d = a.dst[i];
    a.moved[s] = d;
    a.refs[d] = a.refs[s];
    a.refs[s] = 0;
  }
  copy_pages(p, a.src, a.dst, n, blockIdx.x, gridDim.x);
}

__global__ __launch_bounds__(256) void compact_table_kernel(const CompactArgs a) {
  const int64_t step = static_cast<int64_t>(gridDim.x) * 256;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < a.entries; i += step) {
    const int page = a.table[i];
    if (page >= 0 && page < a.pages) a.table[i] = a.moved[page];
  }
}

// ------------------------------------------------------------------------------------------------ host
inline int64_t up4(int64_t n) { return (n + 3) / 4 * 4; }
inline int64_t reserve_most(int64_t B, int64_t width, int64_t pages) { return std::min(B * width, pages); }
inline unsigned blocks_for(int64_t n) { return static_cast<unsigned>(std::min<int64_t>(std::max<int64_t>(ceil_div(n, 256), 1), kCopyGroups)); }

// Workgroups of a launch that copies up to `most` pages.
inline unsigned copy_groups(const KvPool& p, int64_t most) {
  const int64_t units = 2 * most * p.L * p.units;  // below 2^31 pieces
  return static_cast<unsigned>(std::min<int64_t>(std::max<int64_t>(ceil_div(units, kCopyUnits), 1), kCopyGroups));
}

}  // namespace sqx

using namespace sqx;

// What every entry point checks of a pool of pages.
#define KV_POOL(fn)                                                                                                             \
  SQX_REQUIRE(L >= 1 && L < 65536 && Hkv >= 1 && Hkv <= 1024 && (hd == 64 || hd == 128 || hd == 256) && kv_block_ok(block),     \
              SQX_E_ARG, "%s: L=%lld layers (below 65536), Hkv=%lld (up to 1024), hd=%lld (64, 128 or 256), block=%lld (16, 32, 64 or 128)", \
              fn, (long long)L, (long long)Hkv, (long long)hd, (long long)block);                                              \
  SQX_REQUIRE(pages >= 1 && pages < (int64_t(1) << 31) - kTile, SQX_E_ARG, "%s: pages=%lld", fn, (long long)pages)
#define KV_POOL_POINTERS(fn)                                                                                                    \
  SQX_REQUIRE(k_codes && v_codes && k_scale && v_scale, SQX_E_ARG, "%s: null pointer", fn);                                     \
  SQX_REQUIRE(al16(k_codes) && al16(v_codes), SQX_E_ARG, "%s: codes must be 16-byte aligned", fn);                              \
  const KvPool pool{static_cast<uint8_t*>(k_codes), static_cast<uint8_t*>(v_codes), k_scale, v_scale, static_cast<int>(L),      \
                    static_cast<int>(Hkv), static_cast<int>(pages), static_cast<int>(Hkv * block * hd / 16)}
// A copy of up to n pages counts its pieces in 32 bits.
#define KV_POOL_PIECES(fn, n)                                                                                                   \
  SQX_REQUIRE(2 * L * ceil_div(pool.units, kCopyUnits) < (int64_t(1) << 31) / std::max<int64_t>(n, 1), SQX_E_ARG,                \
              "%s: %lld pages of %lld layers are too many for one call", fn, (long long)(n), (long long)L)
#define KV_TABLE(fn)                                                                                                            \
  SQX_REQUIRE(kv_block_ok(block), SQX_E_ARG, "%s: block=%lld (16, 32, 64 or 128 tokens)", fn, (long long)block);                \
  SQX_REQUIRE(B >= 0 && B < 65536 && width >= 1 && width * block < (int64_t(1) << 30) && pages >= 1 &&                          \
                  pages < (int64_t(1) << 31) - kTile,                                                                           \
              SQX_E_ARG, "%s: B=%lld rows (below 65536) of %lld blocks (at least 1; positions below 2^30), pages=%lld", fn,     \
              (long long)B, (long long)width, (long long)pages)
#define KV_SPACE(fn, need)                                                                                                      \
  SQX_REQUIRE(ws != nullptr && ws_bytes >= (need) && al16(ws), SQX_E_SPACE,                                                     \
              "%s: %lld bytes of 16-byte aligned workspace needed, %lld given", fn, (long long)(need), (long long)ws_bytes)

extern "C" int sqx_kvpages_copy(const int* src, const int* dst, int64_t n, void* k_codes, void* v_codes, float* k_scale,
                                float* v_scale, int64_t L, int64_t Hkv, int64_t hd, int64_t block, int64_t pages,
                                sqx_stream_t stream) {
  const char* fn = "sqx_kvpages_copy";
  KV_POOL(fn);
  SQX_REQUIRE(n >= 0 && n < (int64_t(1) << 31), SQX_E_ARG, "%s: n=%lld", fn, (long long)n);
  if (n == 0) return SQX_OK;
  SQX_REQUIRE(src && dst, SQX_E_ARG, "%s: null pointer", fn);
  KV_POOL_POINTERS(fn);
  KV_POOL_PIECES(fn, n);
  hipLaunchKernelGGL(kv_copy_kernel, dim3(copy_groups(pool, n)), dim3(256), 0, as_stream(stream), pool, src, dst,
                     static_cast<const int*>(nullptr), static_cast<int>(n));
  SQX_LAUNCH_CHECK(fn);
  return SQX_OK;
}

extern "C" int64_t sqx_kvpages_fork_workspace_bytes(int64_t B, int64_t width, int64_t pages) {
  if (B <= 0 || width <= 0 || pages <= 0) return 0;
  return 4 * (up4(B * width) + up4(pages) + 5 * up4(B) + 4);
}

extern "C" int sqx_kvpages_fork(const int* parents, void* k_codes, void* v_codes, float* k_scale, float* v_scale, int* table,
                                int* lengths, int* refs, int64_t L, int64_t B, int64_t Hkv, int64_t hd, int64_t block,
                                int64_t pages, int64_t width, int* ok, void* ws, int64_t ws_bytes, sqx_stream_t stream) {
  const char* fn = "sqx_kvpages_fork";
  KV_POOL(fn);
  KV_TABLE(fn);
  SQX_REQUIRE(B >= 1, SQX_E_ARG, "%s: no rows", fn);
  SQX_REQUIRE(parents && table && lengths && refs && ok, SQX_E_ARG, "%s: null pointer", fn);
  KV_POOL_POINTERS(fn);
  KV_POOL_PIECES(fn, B);
  KV_SPACE(fn, sqx_kvpages_fork_workspace_bytes(B, width, pages));
  int* w = static_cast<int*>(ws);
  auto take = [&](int64_t n) {
    int* const at = w;
    w += up4(n);
    return at;
  };
  ForkArgs a{};
  a.parents = parents; a.table = table; a.lengths = lengths; a.refs = refs; a.ok = ok;
  a.table2 = take(B * width); a.refs2 = take(pages);
  a.lengths2 = take(B); a.need = take(B); a.src = take(B); a.dst = take(B); a.free = take(B); a.count = take(1);
  a.B = static_cast<int>(B); a.width = static_cast<int>(width); a.pages = static_cast<int>(pages);
  a.block = static_cast<int>(block); a.shift = kv_shift(block);
  const hipStream_t s = as_stream(stream);
  if (B <= kSmallRows && B * width <= kSmallEntries && pages <= kSmallPages) {
    hipLaunchKernelGGL(fork_small_kernel, dim3(1), dim3(kPlan), 0, s, a);
  } else {
    hipLaunchKernelGGL(fork_begin_kernel, dim3(blocks_for(pages)), dim3(256), 0, s, a);
    hipLaunchKernelGGL(fork_rows_kernel, dim3(static_cast<unsigned>(ceil_div(width, 256)), static_cast<unsigned>(B)), dim3(256), 0, s, a);
    hipLaunchKernelGGL(fork_assign_kernel, dim3(1), dim3(kPlan), 0, s, a);
  }
  hipLaunchKernelGGL(fork_end_kernel, dim3(std::max(copy_groups(pool, B), blocks_for(std::max(B * width, pages)))), dim3(256), 0, s, a, pool);
  SQX_LAUNCH_CHECK(fn);
  return SQX_OK;
}

extern "C" int64_t sqx_kvpages_reserve_workspace_bytes(int64_t B, int64_t width, int64_t pages) {
  if (B <= 0 || width <= 0 || pages <= 0) return 0;
  return 4 * (up4(ceil_div(B * width, 4)) + 2 * up4(B) + 3 * up4(reserve_most(B, width, pages)) + 4);
}

extern "C" int sqx_kvpages_reserve(void* k_codes, void* v_codes, float* k_scale, float* v_scale, int* table, const int* starts,
                                   const int* counts, int* refs, int64_t L, int64_t B, int64_t Hkv, int64_t hd, int64_t block,
                                   int64_t pages, int64_t width, int* ok, void* ws, int64_t ws_bytes, sqx_stream_t stream) {
  const char* fn = "sqx_kvpages_reserve";
  KV_POOL(fn);
  KV_TABLE(fn);
  SQX_REQUIRE(B >= 1, SQX_E_ARG, "%s: no rows", fn);
  SQX_REQUIRE(table && starts && counts && refs && ok, SQX_E_ARG, "%s: null pointer", fn);
  KV_POOL_POINTERS(fn);
  KV_POOL_PIECES(fn, reserve_most(B, width, pages));
  KV_SPACE(fn, sqx_kvpages_reserve_workspace_bytes(B, width, pages));
  const int64_t most = reserve_most(B, width, pages);
  int* w = static_cast<int*>(ws);
  auto take = [&](int64_t n) {
    int* const at = w;
    w += up4(n);
    return at;
  };
  ReserveArgs a{};
  a.table = table; a.starts = starts; a.counts = counts; a.refs = refs; a.ok = ok;
  a.kind = reinterpret_cast<uint8_t*>(take(ceil_div(B * width, 4)));
  a.per = take(B); a.first = take(B); a.free = take(most); a.src = take(most); a.dst = take(most); a.count = take(1);
  a.B = static_cast<int>(B); a.width = static_cast<int>(width); a.pages = static_cast<int>(pages);
  a.block = static_cast<int>(block); a.shift = kv_shift(block); a.most = static_cast<int>(most);
  const hipStream_t s = as_stream(stream);
  if (B <= kSmallRows && B * width <= kSmallReserve) {
    hipLaunchKernelGGL(reserve_small_kernel, dim3(1), dim3(kPlan), 0, s, a);
  } else {
    hipLaunchKernelGGL(reserve_count_kernel, dim3(static_cast<unsigned>(B)), dim3(256), 0, s, a);
    hipLaunchKernelGGL(reserve_assign_kernel, dim3(1), dim3(kPlan), 0, s, a);
    hipLaunchKernelGGL(reserve_rows_kernel, dim3(static_cast<unsigned>(B)), dim3(256), 0, s, a);
  }
  hipLaunchKernelGGL(kv_copy_kernel, dim3(copy_groups(pool, most)), dim3(256), 0, s, pool, a.src, a.dst, a.count,
                     static_cast<int>(most));
  SQX_LAUNCH_CHECK(fn);
  return SQX_OK;
}

extern "C" int sqx_kvpages_free(const int* keep, int* table, int* lengths, int* refs, int64_t B, int64_t block, int64_t pages,
                                int64_t width, sqx_stream_t stream) {
  const char* fn = "sqx_kvpages_free";
  KV_TABLE(fn);
  if (B == 0) return SQX_OK;
  SQX_REQUIRE(keep && table && lengths && refs, SQX_E_ARG, "%s: null pointer", fn);
  hipLaunchKernelGGL(free_rows_kernel, dim3(static_cast<unsigned>(ceil_div(width, 256)), static_cast<unsigned>(B)), dim3(256), 0,
                     as_stream(stream), keep, table, lengths, refs, static_cast<int>(width), static_cast<int>(pages),
                     static_cast<int>(block), kv_shift(block));
  SQX_LAUNCH_CHECK(fn);
  return SQX_OK;
}

extern "C" int64_t sqx_kvpages_compact_workspace_bytes(int64_t pages) {
  return pages <= 0 ? 0 : 4 * (up4(ceil_div(pages, kTile)) + 2 * up4(pages / 2 + 1) + 4);
}

extern "C" int sqx_kvpages_compact(void* k_codes, void* v_codes, float* k_scale, float* v_scale, int* table, int* refs, int64_t L,
                                   int64_t B, int64_t Hkv, int64_t hd, int64_t block, int64_t pages, int64_t width, int* live,
                                   int* moved, void* ws, int64_t ws_bytes, sqx_stream_t stream) {
  const char* fn = "sqx_kvpages_compact";
  KV_POOL(fn);
  KV_TABLE(fn);
  SQX_REQUIRE((table || B == 0) && refs && live && moved, SQX_E_ARG, "%s: null pointer", fn);
  KV_POOL_POINTERS(fn);
  KV_POOL_PIECES(fn, pages / 2 + 1);
  KV_SPACE(fn, sqx_kvpages_compact_workspace_bytes(pages));
  int* w = static_cast<int*>(ws);
  auto take = [&](int64_t n) {
    int* const at = w;
    w += up4(n);
    return at;
  };
  CompactArgs a{};
  a.table = table; a.refs = refs; a.moved = moved; a.live = live;
  a.pages = static_cast<int>(pages); a.ntiles = static_cast<int>(ceil_div(pages, kTile)); a.entries = B * width;
  a.tiles = take(a.ntiles); a.src = take(pages / 2 + 1); a.dst = take(pages / 2 + 1); a.count = take(1);
  const hipStream_t s = as_stream(stream);
  const dim3 tiles(static_cast<unsigned>(a.ntiles));
  hipLaunchKernelGGL(compact_count_kernel, tiles, dim3(kPlan), 0, s, a);
  hipLaunchKernelGGL(compact_scan_kernel, dim3(1), dim3(kPlan), 0, s, a);
  hipLaunchKernelGGL(compact_plan_kernel, tiles, dim3(kPlan), 0, s, a);
  hipLaunchKernelGGL(compact_move_kernel, dim3(copy_groups(pool, pages / 2 + 1)), dim3(256), 0, s, a, pool);
  if (a.entries > 0) hipLaunchKernelGGL(compact_table_kernel, dim3(blocks_for(a.entries)), dim3(256), 0, s, a);
  SQX_LAUNCH_CHECK(fn);
  return SQX_OK;
}
