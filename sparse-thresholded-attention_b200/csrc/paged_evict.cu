// Eviction from a paged cache by accumulated attention weight.
//
// Per (sequence, kv head) the min(len, budget) slots to keep are the forced ones (first n_global,
// last n_local) and the heaviest others, ties to the lowest slot.  One cluster of up to 8 CTAs
// does all of it for one (sequence, kv head); each CTA holds a contiguous slice of the slots:
//   1. the weights become order-preserving integer keys in shared memory;
//   2. the key of the last kept slot is found by radix selection (11 + 11 + 10 bits): every CTA
//      counts its slice, then reads all CTAs' counts (distributed shared memory) and finds the
//      digit, so that no CTA waits for a result of another beyond one cluster barrier per digit;
//   3. each CTA compacts its slice, and copies the rows of K, V and weights that it keeps into the
//      new pages.  Source and destination pages are disjoint: rows move independently.
// The kept rows (read and written once) bound it: the selection reads 4 bytes per slot.
#include <cooperative_groups.h>

#include "paged.cuh"

namespace cg = cooperative_groups;

namespace sta {

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 2048;
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
  uint32_t* keys;     // (B, Hkv, cap) where a slice exceeds shared memory, else null
  int* err;
};

struct Counts {
  int above, equal;
};

struct SmemE {
  uint32_t hist[3][kBins];  // of each digit (others may still read the one before)
  uint32_t scan[kWarps];
  uint32_t digit, rest;  // the digit found and how many of its slots are kept
  Counts counts;
};

// larger weight, larger key; NaN below everything, forced slots above everything
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0u;
  const uint32_t b = __float_as_uint(w == 0.f ? 0.f : w);  // -0 and +0 are equal
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

__device__ __forceinline__ uint32_t block_excl_sum(uint32_t x, uint32_t* sh, uint32_t& total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  uint32_t inc = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += y;
  }
  if (lane == 31) sh[w] = inc;
  __syncthreads();
  uint32_t base = 0, all = 0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    const uint32_t y = sh[i];
    if (i < w) base += y;
    all += y;
  }
  __syncthreads();
  total = all;
  return base + inc - x;
}

// 32 kept rows of a warp: lane l has slot j (its rank r = r0 + l); `n` of them are rows.  A row's K
// and V are LPU lanes' 16-byte chunks; four of a lane's loads are in flight.
template <int CH>
__device__ __forceinline__ void copy_rows(const EvP& p, int b, int h, int j, int r, int n) {
  constexpr int LPU = 2 * CH < 32 ? 2 * CH : 32, PER = 32 / LPU, PASS = 2 * CH / LPU, U = 4 / PASS;
  const int lane = threadIdx.x & 31;
  int64_t ks = -1, vs = 0, kd = 0, vd = 0;
  if (lane < n) {
    const uint32_t t = (uint32_t)j / p.c.page, to = (uint32_t)r / p.c.page;
    const int64_t pg = paged_page(p.c, p.c.table, p.c.ts, b, t);
    const int64_t pd = (uint32_t)r < p.cap_out ? paged_page(p.c, p.table_out, p.tos, b, to) : -1;
    if (pg < 0 || pd < 0) {
      atomicCAS(p.err, 0, kErrPageEvict);
    } else {
      const int64_t slot = (uint32_t)j - t * p.c.page, ds = (uint32_t)r - to * p.c.page;
      ks = pg * p.c.ksp + h * p.c.ksh + slot * p.c.ksn;
      vs = pg * p.c.vsp + h * p.c.vsh + slot * p.c.vsn;
      kd = pd * p.c.ksp + h * p.c.ksh + ds * p.c.ksn;
      vd = pd * p.c.vsp + h * p.c.vsh + ds * p.c.vsn;
      p.c.w[pd * p.c.wsp + h * p.c.wsh + ds] = p.c.w[pg * p.c.wsp + h * p.c.wsh + slot];
    }
  }
  const int sub = lane / LPU, ch = lane % CH;
  const bool is_v = PASS == 1 && (lane / CH) % 2 == 1;
#pragma unroll 1
  for (int i0 = 0; i0 < n; i0 += U * PER) {
    uint4 x[U][PASS];
    char* to[U][PASS];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * PER + sub;
      const int64_t a = __shfl_sync(0xffffffffu, ks, i & 31), c = __shfl_sync(0xffffffffu, kd, i & 31);
      const int64_t d = __shfl_sync(0xffffffffu, vs, i & 31), e = __shfl_sync(0xffffffffu, vd, i & 31);
#pragma unroll
      for (int q = 0; q < PASS; ++q) {
        const bool v = PASS == 1 ? is_v : q == 1;
        to[u][q] = i < n && a >= 0 ? (v ? p.c.v + e : p.c.k + c) + ch * 16 : nullptr;
        if (to[u][q]) x[u][q] = __ldcs(reinterpret_cast<const uint4*>((v ? p.c.v + d : p.c.k + a) + ch * 16));
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int q = 0; q < PASS; ++q)
        if (to[u][q]) *reinterpret_cast<uint4*>(to[u][q]) = x[u][q];
  }
}

template <int CH>
__global__ void __launch_bounds__(kThreads, 2) paged_evict_kernel(const EvP p) {
  extern __shared__ uint32_t s_keys[];
  __shared__ SmemE sm;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = blockIdx.x, CL = gridDim.x;  // the cluster is the grid's first dimension
  const int h = blockIdx.y, b = blockIdx.z;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int len = paged_len(p.c, b);
  const int n = (int)min((int64_t)len, p.budget);
  int32_t* kept = p.kept + ((int64_t)b * p.c.Hkv + h) * p.budget;
  if (rank == 0 && h == 0 && tid == 0) p.lens_out[b] = n;
  for (int64_t r = n + (int64_t)rank * kThreads + tid; r < p.budget; r += (int64_t)CL * kThreads) kept[r] = -1;
  const int per = (len + CL - 1) / CL;
  const int lo = min(rank * per, len), cnt = min(per, len - lo);  // this CTA's slots
  if (len <= p.budget) {  // (the same for all CTAs of the cluster)
    for (int i0 = warp * 32; i0 < cnt; i0 += kThreads) {
      const int j = lo + i0 + lane;
      if (i0 + lane < cnt) kept[j] = j;
      copy_rows<CH>(p, b, h, j, j, min(32, cnt - i0));
    }
    return;
  }
  uint32_t* keys = p.keys ? p.keys + ((int64_t)b * p.c.Hkv + h) * p.c.cap + lo : s_keys;

  // ---- keys
  for (int i = tid; i < 3 * kBins; i += kThreads) sm.hist[0][i] = 0u;
#pragma unroll 4
  for (int i = tid; i < cnt; i += kThreads) {
    const int j = lo + i;
    const uint32_t t = (uint32_t)j / p.c.page;
    const int64_t pg = paged_page(p.c, p.c.table, p.c.ts, b, t);
    uint32_t key = 0u;
    if (pg < 0) atomicCAS(p.err, 0, kErrPageEvict);
    else key = weight_key(p.c.w[pg * p.c.wsp + h * p.c.wsh + ((uint32_t)j - t * p.c.page)]);
    if (j < p.n_global || j >= len - p.n_local) key = 0xffffffffu;
    keys[i] = key;
  }
  __syncthreads();

  // ---- the n-th largest key of all slices, and how many of its equals are kept
  uint32_t prefix = 0u, mask = 0u, need = (uint32_t)n;
#pragma unroll 1
  for (int round = 0; round < 3; ++round) {
    const int bits = round < 2 ? 11 : 10, shift = round == 0 ? 21 : (round == 1 ? 10 : 0);
    uint32_t* hist = sm.hist[round];
    for (int i = tid; i < cnt; i += kThreads) {
      const uint32_t key = keys[i];
      if ((key & mask) == prefix) atomicAdd(&hist[(key >> shift) & ((1u << bits) - 1u)], 1u);
    }
    cluster.sync();
    // this thread's bins of all slices, largest digit first
    constexpr int PB = kBins / kThreads;
    uint32_t c[PB], sum = 0;
#pragma unroll
    for (int i = 0; i < PB; ++i) c[i] = 0u;
    const int top = (1 << bits) - 1 - tid * PB;  // digits top, top - 1, ..
    if (top >= 0)
      for (int q = 0; q < CL; ++q) {
        const uint32_t* far = CL == 1 ? hist : cluster.map_shared_rank(hist, q);
#pragma unroll
        for (int i = 0; i < PB; ++i) c[i] += far[top - i];
      }
#pragma unroll
    for (int i = 0; i < PB; ++i) sum += c[i];
    uint32_t all;
    uint32_t before = block_excl_sum(sum, sm.scan, all);
#pragma unroll
    for (int i = 0; i < PB; ++i) {
      if (before < need && before + c[i] >= need) {
        sm.digit = (uint32_t)(top - i);
        sm.rest = need - before;
      }
      before += c[i];
    }
    __syncthreads();
    prefix |= sm.digit << shift;
    mask |= ((1u << bits) - 1u) << shift;
    need = sm.rest;
    __syncthreads();
  }

  // ---- where this slice's kept slots go
  uint32_t above = 0, equal = 0;
  for (int i = tid; i < cnt; i += kThreads) {
    above += keys[i] > prefix;
    equal += keys[i] == prefix;
  }
  uint32_t all_above, all_equal;
  block_excl_sum(above, sm.scan, all_above);
  block_excl_sum(equal, sm.scan, all_equal);
  if (tid == 0) sm.counts = {(int)all_above, (int)all_equal};
  cluster.sync();
  int base = 0, ties = (int)need;  // rank of the first kept slot, equals left for this slice and those behind
  for (int q = 0; q < rank; ++q) {
    const Counts c = *cluster.map_shared_rank(&sm.counts, q);
    const int take = min(c.equal, ties);
    base += c.above + take;
    ties -= take;
  }
  ties = min(ties, (int)all_equal);
  cluster.sync();  // no CTA ends while another may read its counts

  // ---- compaction in slot order, in place: entry i of the list never lies behind the keys read
  const int mine = (int)all_above + ties;
  uint32_t done_above = 0, done_equal = 0;
  for (int i0 = 0; i0 < cnt; i0 += kChunk) {
    const int i = i0 + tid * kItems;
    uint32_t key[kItems], x = 0;
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      key[k] = i + k < cnt ? keys[i + k] : 0u;
      if (i + k < cnt) x += key[k] > prefix ? 1u : (key[k] == prefix ? 1u << 16 : 0u);
    }
    uint32_t all;
    const uint32_t at = block_excl_sum(x, sm.scan, all);  // (ends behind a barrier: all keys are read)
    uint32_t a = done_above + (at & 0xffffu), e = done_equal + (at >> 16);
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      if (i + k >= cnt) break;
      const bool tie = key[k] == prefix;
      if (key[k] > prefix || (tie && e < (uint32_t)ties)) keys[a + min(e, (uint32_t)ties)] = (uint32_t)(lo + i + k);
      a += key[k] > prefix;
      e += tie;
    }
    done_above += all & 0xffffu;
    done_equal += all >> 16;
    __syncthreads();
  }

  // ---- rows
  for (int i0 = warp * 32; i0 < mine; i0 += kThreads) {
    const bool in = i0 + lane < mine;
    const int j = in ? (int)keys[i0 + lane] : 0, r = base + i0 + lane;
    if (in) kept[r] = j;
    copy_rows<CH>(p, b, h, j, r, min(32, mine - i0));
  }
}

int check(const sta_paged_cache* c, const sta_paged_evict_args* a) {
  const int rc = paged_check(c);
  if (rc != STA_OK) return rc;
  if (!a || !a->table_out || !a->kept || !a->lens_out)
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

// CTAs of a cluster: enough to fill the GPU (two CTAs per SM) and to hold the keys in shared
// memory, but slices of 128 slots at least.
int cluster_size(const sta_paged_cache* c) {
  const int64_t cap = c->table_width * c->page_size, segs = c->batch * c->n_kv_heads;
  int cl = 1;
  while (cl < 8 && cap / cl >= 256 && (segs * cl < 296 || cap / cl > kSliceSmem)) cl *= 2;
  return cl;
}

bool keys_in_smem(const sta_paged_cache* c) {
  const int64_t cap = c->table_width * c->page_size;
  return (cap + cluster_size(c) - 1) / cluster_size(c) <= kSliceSmem;
}

template <int CH>
cudaError_t launch(const EvP& p, int cl, int64_t cap, cudaStream_t st) {
  const int bytes = p.keys ? 0 : (int)(((cap + cl - 1) / cl) * 4);
  static bool ready[64];
  const cudaError_t e = allow_smem(paged_evict_kernel<CH>, kSliceSmem * 4, ready);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)cl, (unsigned)p.c.Hkv, (unsigned)p.c.B);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = (size_t)bytes;
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)cl;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, paged_evict_kernel<CH>, p);
}

}  // namespace

size_t paged_evict_workspace_bytes(const sta_paged_cache* c, const sta_paged_evict_args* a) {
  if (check(c, a) != STA_OK) return 0;
  const size_t keys = (size_t)(c->batch * c->n_kv_heads) * (c->table_width * c->page_size) * 4;
  return (keys_in_smem(c) ? 0 : keys) + 256;
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
  p.keys = keys_in_smem(c) ? nullptr
                           : reinterpret_cast<uint32_t*>(w + (256 - reinterpret_cast<uintptr_t>(w) % 256) % 256);
  p.err = device_error_word();
  if (!p.err) return fail(STA_ERR_CUDA, "sta_paged_evict: no device");
  const int ch = c->d * (c->dtype == STA_DTYPE_F32 ? 4 : 2) / 16, cl = cluster_size(c);
  const cudaError_t e = ch == 8 ? launch<8>(p, cl, p.c.cap, st)
                                : (ch == 16 ? launch<16>(p, cl, p.c.cap, st) : launch<32>(p, cl, p.c.cap, st));
  return e == cudaSuccess ? STA_OK : fail(STA_ERR_CUDA, cudaGetErrorString(e));
}

}  // namespace sta
