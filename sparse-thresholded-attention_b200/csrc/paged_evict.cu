// Eviction from a paged cache by accumulated attention weight.
//
// Per (sequence, kv head) the min(len, budget) slots to keep are the forced ones (first n_global,
// last n_local) and the heaviest others, ties to the lowest slot.  Two launches:
//
// Selection, one CTA per (sequence, kv head), or a cluster of up to 8 where the slots exceed 16384
// per CTA; each CTA holds a contiguous slice.  The weights become order-preserving integer keys in
// shared memory; the key of the last kept slot is found by radix selection (11 + 11 + 10 bits):
// every CTA counts its slice, reads all CTAs' counts (distributed shared memory) and finds the
// digit, one cluster barrier per digit; then each CTA writes its kept slots in order.  It reads 4
// bytes per slot (and leaves the pages' places) and is bound by latency: 12 us for 128 heads of up to
// 8192 slots (a CTA each), 20 us for 32 heads of 65536 (clusters of four: 6 us until the keys are
// there, 2.4 us per digit, 4 us for the order).  Weights are read four at a time where pages and strides allow it (one at a
// time: 13.5 us for the 128 heads), and the keys lie in shared memory as long as a slice fits (in
// global memory: 22 us for the 32 heads).
//
// Copy of the kept rows of K, V and weights into the new pages, 8 or 16 rows per warp wherever
// they come from, set up while the selection runs (programmatic launch).  Source and destination pages
// are disjoint, so rows move independently: a new page that holds rows of the cache, or that another
// entry of the new table names too, is found by the places that the selection leaves, and its rows
// are dropped and reported.  Bound by HBM: rows are read and written once (16
// sequences cut to 2048 keys of 8 kv heads, f32, d = 128: 71 us behind the selection, 427 MB at 6.0 TB/s; 4
// sequences cut to 8192 keys, bf16: 48 us, 270 MB at 5.6 TB/s).
#include <cooperative_groups.h>

#include "paged.cuh"

namespace cg = cooperative_groups;

namespace sta {

namespace {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 2048;
// Slots of a CTA that call for a larger cluster where that makes kFewCtas CTAs at most, so that the
// clusters run at once (a CTA takes an SM): 8 heads of 16384 slots take 12.5 us in clusters of 2 and
// 15 with a CTA each, but 16 heads of 65536 slots 38 us in clusters of 8 and 18.5 in clusters of 4,
// 32 heads 57 and 20 us (46 with a CTA each).  Otherwise only twice the slots call for it.
constexpr int kSlice = 8192;
constexpr int kFewCtas = 64;
constexpr int kCopy = 256;             // threads of the copy
constexpr int kItems = 8;              // consecutive slots of a thread in the compaction
constexpr int kChunk = kThreads * kItems;
constexpr int kSliceSmem = 20 * 1024;  // slots of a slice whose keys fit shared memory (80 KB)

struct EvP {
  PagedView c;
  int64_t budget, n_global, n_local;
  const int32_t* table_out;
  int64_t tos;
  uint32_t cap_out;
  int32_t* kept;
  int32_t* lens_out;
  int rows;           // rows of a warp in the copy: 8 or 16
  int quads;          // weights of four neighbouring slots may be loaded at once
  uint32_t* keys;     // (B, Hkv, cap rounded up to 4) where a slice exceeds shared memory, else null
  int2* from;         // (n_pages,) places in the table, and in the new one
  int2* to;
  int* err;
};

struct __align__(16) SmemE {
  uint32_t hist[3][kBins];  // of each digit (others may still read the one before)
  uint32_t scan[2][kWarps];
  uint32_t digit[3], rest[3];  // the digits found and how many of their slots are kept
  __align__(16) uint32_t counts[4];  // slots of the slice above the last kept key, and equal to it
};

// larger weight, larger key; NaN below everything, forced slots above everything
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0u;
  const uint32_t b = __float_as_uint(w == 0.f ? 0.f : w);  // -0 and +0 are equal
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

__device__ __forceinline__ uint32_t warp_incl_sum(uint32_t x) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  return x;
}

// (every warp sums the warps' totals for itself; calls in a row take two buffers in turn)
__device__ __forceinline__ uint32_t block_excl_sum(uint32_t x, uint32_t* sh, uint32_t& total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const uint32_t inc = warp_incl_sum(x);
  if (lane == 31) sh[w] = inc;
  __syncthreads();
  const uint32_t sums = warp_incl_sum(lane < kWarps ? sh[lane] : 0u);
  const uint32_t base = __shfl_sync(0xffffffffu, sums, w == 0 ? 0 : w - 1);
  total = __shfl_sync(0xffffffffu, sums, 31);
  return (w == 0 ? 0u : base) + inc - x;
}

// four words of CTA q's shared memory
__device__ __forceinline__ uint4 far_words(const uint32_t* mine, int q) {
  uint32_t a;
  uint4 x;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(mine)), "r"(q));
  asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(a));
  return x;
}

__global__ void __launch_bounds__(kThreads) paged_evict_select_kernel(const EvP p) {
  extern __shared__ __align__(16) uint32_t s_keys[];
  __shared__ SmemE sm;
  cg::cluster_group cluster = cg::this_cluster();
  grid_wait();
  grid_dependents();
  const int rank = blockIdx.x, CL = gridDim.x;  // the cluster is the grid's first dimension
  const int h = blockIdx.y, b = blockIdx.z;
  const int tid = threadIdx.x, lane = tid & 31;
  const int len = paged_len(p.c, b);
  const int n = (int)min((int64_t)len, p.budget);
  int32_t* kept = p.kept + ((int64_t)b * p.c.Hkv + h) * p.budget;
  if (rank == 0 && h == 0 && tid == 0) p.lens_out[b] = n;
  for (int64_t r = n + (int64_t)rank * kThreads + tid; r < p.budget; r += (int64_t)CL * kThreads) kept[r] = -1;
  const int per = ((len + CL - 1) / CL + 3) & ~3;
  const int lo = min(rank * per, len), cnt = min(per, len - lo);  // this CTA's slots
  // the places of the sequence's pages, old and new, left by all its CTAs; a thread's first entries
  // are asked for here and left once the keys have been asked for
  const int32_t* table = p.c.table + b * p.c.ts;
  const int32_t* table_out = p.table_out + b * p.tos;
  const uint32_t t0 = (uint32_t)(h * CL + rank) * kThreads + tid, steps = (uint32_t)p.c.Hkv * CL * kThreads;
  const uint32_t olds = entries_of(p.c, len), news = entries_of(p.c, n);
  const int32_t old0 = t0 < olds ? __ldg(table + t0) : -1, new0 = t0 < news ? __ldg(table_out + t0) : -1;
  auto leave = [&]() {
    leave_place(p.from, p.c.n_pages, old0, b, t0);
    leave_place(p.to, p.c.n_pages, new0, b, t0);
    if (olds - min(olds, t0) > steps) leave_places(p.from, p.c.n_pages, table, b, olds, t0 + steps, steps);
    if (news - min(news, t0) > steps) leave_places(p.to, p.c.n_pages, table_out, b, news, t0 + steps, steps);
  };
  if (len <= p.budget) {  // (the same for all CTAs of the cluster)
    for (int i = tid; i < cnt; i += kThreads) kept[lo + i] = lo + i;
    leave();
    return;
  }
  uint32_t* keys = p.keys ? p.keys + ((int64_t)b * p.c.Hkv + h) * ((p.c.cap + 3) & ~3u) + lo : s_keys;

  // ---- keys, and the count of their first digits; the loads of a thread are asked for together
  for (int i = tid; i < 3 * kBins; i += kThreads) sm.hist[0][i] = 0u;
  if (tid < 4) sm.counts[tid] = 0u;
  __syncthreads();
  auto take_key = [&](int i, float w) {  // of slot lo + i
    const int j = lo + i;
    const uint32_t key = j < p.n_global || j >= len - p.n_local ? 0xffffffffu : weight_key(w);
    if (i < cnt) atomicAdd(&sm.hist[0][~(key >> 21) & (kBins - 1)], 1u);
    return key;
  };
  constexpr int U = 4;
  const float* weights = p.c.w + h * p.c.wsh;
  const float nan = __int_as_float(0x7fffffff);  // of a bad page: the smallest
  const int step = p.quads ? 4 : 1;  // quads: four neighbouring slots share a page and a 16-byte load
  for (int i0 = tid * step; i0 < cnt; i0 += U * kThreads * step) {
    int32_t entry[U];
    uint32_t slot[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t j = (uint32_t)lo + (uint32_t)(i0 + u * kThreads * step), t = j / p.c.page;
      slot[u] = j - t * p.c.page;
      entry[u] = i0 + u * kThreads * step < cnt ? __ldg(table + t) : 0;
    }
    float4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * kThreads * step;
      const bool ok = entry[u] >= 0 && entry[u] < p.c.n_pages;
      const float* src = weights + entry[u] * p.c.wsp + slot[u];
      w[u] = make_float4(nan, nan, nan, nan);
      if (i < cnt && ok) {
        if (p.quads) w[u] = *reinterpret_cast<const float4*>(src);
        else w[u].x = *src;
      }
      if (!ok) atomicCAS(p.err, 0, kErrPageEvict);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * kThreads * step;
      if (i >= cnt) break;
      if (p.quads)  // (a slice has room for a multiple of four)
        *reinterpret_cast<uint4*>(keys + i) = make_uint4(take_key(i, w[u].x), take_key(i + 1, w[u].y),
                                                         take_key(i + 2, w[u].z), take_key(i + 3, w[u].w));
      else
        keys[i] = take_key(i, w[u].x);
    }
  }

  leave();

  // ---- the n-th largest key of all slices, and how many of its equals are kept
  uint32_t prefix = 0u, mask = 0u, need = (uint32_t)n;
  uint32_t above = 0u, equal = 0u;  // this slice's slots above the key (this thread's bins), and equal
#pragma unroll 1
  for (int round = 0; round < 3; ++round) {
    const int bits = round < 2 ? 11 : 10, shift = round == 0 ? 21 : (round == 1 ? 10 : 0);
    uint32_t* hist = sm.hist[round];
    if (round > 0) {
      for (int i = tid * 4; i < cnt; i += kThreads * 4) {
        const uint4 four = *reinterpret_cast<const uint4*>(keys + i);
        const uint32_t key[4] = {four.x, four.y, four.z, four.w};
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (i + k < cnt && (key[k] & mask) == prefix)
            atomicAdd(&hist[~(key[k] >> shift) & ((1u << bits) - 1u)], 1u);
      }
    }
    cluster.sync();
    // this thread's four bins (bin i counts digit bins - 1 - i) of all slices
    uint32_t c[4] = {0u, 0u, 0u, 0u};
    if (tid * 4 < (1 << bits)) {
      uint4 x[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) x[q] = q < CL ? far_words(hist + tid * 4, q) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        c[0] += x[q].x;
        c[1] += x[q].y;
        c[2] += x[q].z;
        c[3] += x[q].w;
      }
    }
    const uint32_t sum = c[0] + c[1] + c[2] + c[3];
    uint32_t all;
    uint32_t before = block_excl_sum(sum, sm.scan[0], all);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (before < need && before + c[i] >= need) {
        sm.digit[round] = (uint32_t)((1 << bits) - 1 - tid * 4 - i);
        sm.rest[round] = need - before;
      }
      before += c[i];
    }
    __syncthreads();
    const uint32_t bin = ((1u << bits) - 1u) - sm.digit[round];
    if (tid * 4 < (1 << bits)) {
      const uint4 mine = *reinterpret_cast<const uint4*>(hist + tid * 4);
      above += (tid * 4u < bin ? mine.x : 0u) + (tid * 4u + 1u < bin ? mine.y : 0u) +
               (tid * 4u + 2u < bin ? mine.z : 0u) + (tid * 4u + 3u < bin ? mine.w : 0u);
    }
    equal = hist[bin];  // (of the last round)
    prefix |= sm.digit[round] << shift;
    mask |= ((1u << bits) - 1u) << shift;
    need = sm.rest[round];
  }

  // ---- where this slice's kept slots go
  above = __reduce_add_sync(0xffffffffu, above);
  if (lane == 0) atomicAdd(&sm.counts[0], above);
  if (tid == 0) sm.counts[1] = equal;
  cluster.sync();
  // lane q: slots of slice q above and equal; the equals go to the slices in order
  uint4 c = lane < CL ? far_words(sm.counts, lane) : make_uint4(0u, 0u, 0u, 0u);
  cluster.barrier_arrive();  // (waited for at the end: no CTA goes while another may read its counts)
  uint32_t eq = c.y;
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, eq, o);
    if (lane >= o) eq += y;
  }
  const uint32_t eq_before = eq - c.y, take = eq_before >= need ? 0u : min(c.y, need - eq_before);
  const uint32_t holds = c.x + take;  // kept slots of slice q
  uint32_t upto = holds;
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += y;
  }
  const int base = (int)__shfl_sync(0xffffffffu, upto - holds, rank);
  const uint32_t ties = __shfl_sync(0xffffffffu, take, rank);

  // ---- the kept slots in order
  uint32_t done_above = 0, done_equal = 0;
  for (int i0 = 0; i0 < cnt; i0 += kChunk) {
    const int i = i0 + tid * kItems;
    uint32_t key[kItems], x = 0;
#pragma unroll
    for (int k = 0; k < kItems; k += 4) {
      const uint4 four = i + k < cnt ? *reinterpret_cast<const uint4*>(keys + i + k) : make_uint4(0u, 0u, 0u, 0u);
      key[k] = four.x; key[k + 1] = four.y; key[k + 2] = four.z; key[k + 3] = four.w;
    }
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      if (i + k < cnt) x += key[k] > prefix ? 1u : (key[k] == prefix ? 1u << 16 : 0u);
    }
    uint32_t all;
    const uint32_t at = block_excl_sum(x, sm.scan[i0 / kChunk & 1], all);
    uint32_t a = done_above + (at & 0xffffu), e = done_equal + (at >> 16);
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      if (i + k >= cnt) break;
      const bool tie = key[k] == prefix;
      if (key[k] > prefix || (tie && e < ties)) kept[base + a + min(e, ties)] = lo + i + k;
      a += key[k] > prefix;
      e += tie;
    }
    done_above += all & 0xffffu;
    done_equal += all >> 16;
  }
  cluster.barrier_wait();
}

template <int CH>
__global__ void __launch_bounds__(kCopy, 4) paged_evict_copy_kernel(const EvP p) {
  const int lane = threadIdx.x & 31, h = blockIdx.y, b = blockIdx.z;
  const int n = (int)min((int64_t)paged_len(p.c, b), p.budget);
  const int r0 = (int)(blockIdx.x * (kCopy / 32) + threadIdx.x / 32) * p.rows, r = r0 + lane;
  const int end = min(n, r0 + p.rows);
  int64_t kd = 0, vd = 0, wd = -1, pd = -1;
  uint32_t to = 0;
  if (r < end) {
    to = (uint32_t)r / p.c.page;
    const uint32_t ds = (uint32_t)r - to * p.c.page;
    pd = (uint32_t)r < p.cap_out ? paged_page(p.c, p.table_out, p.tos, b, to) : -1;
    if (pd >= 0) {
      kd = pd * p.c.ksp + h * p.c.ksh + ds * p.c.ksn;
      vd = pd * p.c.vsp + h * p.c.vsh + ds * p.c.vsn;
      wd = pd * p.c.wsp + h * p.c.wsh + ds;
    }
  }
  grid_wait();
  if (r0 >= n) return;
  int64_t ks = -1, vs = 0;
  if (r < end) {
    // the row's slot and the places at its new page, then what they name: two chains of loads side by side
    const int2 none = make_int2(-1, -1);
    const int2 old = pd >= 0 ? p.from[pd] : none, own = pd >= 0 ? p.to[pd] : none;
    const uint32_t j = (uint32_t)p.kept[((int64_t)b * p.c.Hkv + h) * p.budget + r];
    const uint32_t t = j / p.c.page, slot = j - t * p.c.page;
    const bool named = old.x >= 0 && old.x < p.c.B && (uint32_t)old.y < p.c.width;
    const int len = named ? paged_len(p.c, old.x) : 0;
    const int32_t entry = named ? __ldg(p.c.table + old.x * p.c.ts + old.y) : -1;
    const int64_t pg = paged_page(p.c, p.c.table, p.c.ts, b, t);
    const bool used = entry == pd && (uint32_t)old.y < entries_of(p.c, len);
    if (pg < 0 || wd < 0) {
      atomicCAS(p.err, 0, kErrPageEvict);
    } else if (used || !is_place(own, b, to)) {
      atomicCAS(p.err, 0, kErrPageTwice);
    } else {
      ks = pg * p.c.ksp + h * p.c.ksh + slot * p.c.ksn;
      vs = pg * p.c.vsp + h * p.c.vsh + slot * p.c.vsn;
      p.c.w[wd] = p.c.w[pg * p.c.wsp + h * p.c.wsh + slot];
    }
  }
  move_rows<CH, true>(p.c.k, p.c.v, p.c.k, p.c.v, ks, vs, kd, vd, end - r0, 0);
}

int check(const sta_paged_cache* c, const sta_paged_evict_args* a) {
  int rc = paged_check(c);
  if (rc == STA_OK) rc = paged_check_rows_written(c);
  if (rc != STA_OK) return rc;
  if (!a || (c->batch > 0 && (!a->table_out || !a->kept || !a->lens_out)))
    return fail(STA_ERR_ARG, "sta_paged_evict: null pointer");
  if (!c->weights) return fail(STA_ERR_ARG, "sta_paged_evict: the cache has no weights");
  if (a->budget <= 0 || a->budget > ((int64_t)1 << 31) - 65)
    return fail(STA_ERR_ARG, "sta_paged_evict: bad budget");
  if (a->n_global < 0 || a->n_local < 0 || a->n_global > a->budget ||
      a->n_local > a->budget - a->n_global)
    return fail(STA_ERR_ARG, "sta_paged_evict: n_global + n_local must not exceed the budget");
  if (a->table_out_width <= 0) return fail(STA_ERR_ARG, "sta_paged_evict: empty table_out");
  const int64_t cap = c->table_width * c->page_size;
  const int64_t most = cap < a->budget ? cap : a->budget;  // rows that a sequence can keep
  if (a->table_out_width < (most + c->page_size - 1) / c->page_size)
    return fail(STA_ERR_ARG, "sta_paged_evict: table_out has no room for the budget");
  if (a->lens_out < c->lens + c->batch && c->lens < a->lens_out + c->batch)
    return fail(STA_ERR_ARG, "sta_paged_evict: lens_out overlaps lens");
  if (c->batch > 65535) return fail(STA_ERR_UNSUPPORTED, "sta_paged_evict: too many sequences");
  return STA_OK;
}

int cluster_size(const sta_paged_cache* c) {
  const int64_t cap = c->table_width * c->page_size;
  const int64_t segs = c->batch * c->n_kv_heads;
  int cl = 1;
  while (cl < 8 && (cap / cl > 2 * kSlice || (cap / cl > kSlice && 2 * cl * segs <= kFewCtas))) cl *= 2;
  return cl;
}

size_t places_bytes(const sta_paged_cache* c) { return (2 * (size_t)c->n_pages * sizeof(int2) + 255) & ~size_t(255); }

bool keys_in_smem(const sta_paged_cache* c) {
  const int64_t cap = c->table_width * c->page_size;
  return (cap + cluster_size(c) - 1) / cluster_size(c) + 3 <= kSliceSmem;
}

cudaError_t launch_select(const EvP& p, int cl, cudaStream_t st) {
  static bool ready[64];
  const cudaError_t e = allow_smem(paged_evict_select_kernel, kSliceSmem * 4, ready);
  if (e != cudaSuccess) return e;
  const size_t bytes = p.keys ? 0 : ((size_t)(p.c.cap + cl - 1) / cl + 3) * 4;
  return launch_behind(paged_evict_select_kernel, dim3((unsigned)cl, (unsigned)p.c.Hkv, (unsigned)p.c.B), kThreads,
                       p, st, bytes, cl > 1 ? (unsigned)cl : 0u);
}

}  // namespace

size_t paged_evict_workspace_bytes(const sta_paged_cache* c, const sta_paged_evict_args* a) {
  if (check(c, a) != STA_OK) return 0;
  const size_t keys = (size_t)(c->batch * c->n_kv_heads) * ((c->table_width * c->page_size + 3) & ~(int64_t)3) * 4;
  return places_bytes(c) + (keys_in_smem(c) ? 0 : keys) + 256;
}

int paged_evict(const sta_paged_cache* c, const sta_paged_evict_args* a, void* ws, size_t ws_len,
                cudaStream_t st) {
  const int rc = check(c, a);
  if (rc != STA_OK) return rc;
  if (c->batch == 0) return STA_OK;
  if (!ws || ws_len < paged_evict_workspace_bytes(c, a))
    return fail(STA_ERR_WORKSPACE, "sta_paged_evict: workspace too small");
  EvP p;
  p.c = paged_view(c);
  p.budget = a->budget; p.n_global = a->n_global; p.n_local = a->n_local;
  p.table_out = a->table_out;
  p.tos = a->table_out_stride;
  const int64_t cap_out = a->table_out_width * c->page_size;
  p.cap_out = (uint32_t)(cap_out < a->budget ? cap_out : a->budget);
  p.kept = a->kept;
  p.lens_out = a->lens_out;
  uint8_t* w = static_cast<uint8_t*>(ws);
  w += (256 - reinterpret_cast<uintptr_t>(w) % 256) % 256;
  p.from = reinterpret_cast<int2*>(w);
  p.to = p.from + c->n_pages;
  p.keys = keys_in_smem(c) ? nullptr : reinterpret_cast<uint32_t*>(w + places_bytes(c));
  p.quads = p.c.page % 4 == 0 && (reinterpret_cast<uintptr_t>(p.c.w) & 15) == 0 && p.c.wsp % 4 == 0 && p.c.wsh % 4 == 0;
  p.err = page_error_word();
  if (!p.err) return fail(STA_ERR_CUDA, "sta_paged_evict: no device");
  const int ch = c->d * (c->dtype == STA_DTYPE_F32 ? 4 : 2) / 16;
  const int64_t most = p.c.cap < a->budget ? p.c.cap : a->budget;
  // 16 rows of a warp even out ragged sequences (16 of them as above: 71 us, with 32 rows 74; equal
  // ones 48 and 47 us), 8 where that is what it takes to give 16 warps to every SM (1024 rows of 8
  // kv heads: the copy adds 3.5 us, with 32 rows 7.5)
  p.rows = 16;
  while (p.rows > 8 && most * p.c.Hkv * p.c.B < (int64_t)p.rows * 16 * 148) p.rows /= 2;
  const int64_t per = (int64_t)p.rows * (kCopy / 32);
  const dim3 grid((unsigned)((most + per - 1) / per), (unsigned)p.c.Hkv, (unsigned)p.c.B);
  cudaError_t e = launch_select(p, cluster_size(c), st);
  if (e == cudaSuccess)
    e = ch == 8 ? launch_behind(paged_evict_copy_kernel<8>, grid, kCopy, p, st)
                : (ch == 16 ? launch_behind(paged_evict_copy_kernel<16>, grid, kCopy, p, st)
                            : launch_behind(paged_evict_copy_kernel<32>, grid, kCopy, p, st));
  return e == cudaSuccess ? STA_OK : fail(STA_ERR_CUDA, cudaGetErrorString(e));
}

}  // namespace sta
