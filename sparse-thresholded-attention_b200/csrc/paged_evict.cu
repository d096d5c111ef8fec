// Eviction from a paged cache by accumulated attention weight.
//
// Per (sequence, kv head): the min(len, budget) slots to keep are the forced ones (first
// n_global, last n_local) and the heaviest others, ties to the lowest slot -- an order statistic
// over order-preserving integer keys, found by radix selection (4 rounds of 8 bits), then a
// compaction in slot order.  A second launch copies the kept rows of K, V and weights into the
// new pages; source and destination pages are disjoint, so rows move independently of each other.
#include "paged.cuh"

namespace sta {

namespace {

constexpr int kSel = 1024;
constexpr int kCopy = 256;
constexpr int kIter = 4;

struct EvP {
  PagedView c;
  int64_t budget, n_global, n_local;
  const int32_t* table_out;
  int64_t tos;
  uint32_t cap_out;
  int32_t* kept;
  int32_t* lens_out;
  uint32_t* keys;  // (B, Hkv, cap) order-preserving keys
  int* err;
};

// larger weight, larger key; NaN below everything, forced slots above everything
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0u;
  const uint32_t b = __float_as_uint(w == 0.f ? 0.f : w);  // -0 and +0 are equal
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

__device__ __forceinline__ int block_excl_sum(int x, int* sh, int& total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int inc = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += y;
  }
  if (lane == 31) sh[w] = inc;
  __syncthreads();
  int base = 0, all = 0;
  for (int i = 0; i < kSel / 32; ++i) {
    if (i < w) base += sh[i];
    all += sh[i];
  }
  __syncthreads();
  total = all;
  return base + inc - x;
}

__global__ void __launch_bounds__(kSel) paged_evict_select_kernel(const EvP p) {
  __shared__ uint32_t hist[256];
  __shared__ int sh[kSel / 32];
  __shared__ uint32_t s_prefix;
  __shared__ int s_k;
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const int len = paged_len(p.c, b);
  const int n = (int)min((int64_t)len, p.budget);
  int32_t* kept = p.kept + ((int64_t)b * p.c.Hkv + h) * p.budget;
  if (h == 0 && tid == 0) p.lens_out[b] = n;
  for (int64_t r = n + tid; r < p.budget; r += kSel) kept[r] = -1;
  if (len <= p.budget) {
    for (int r = tid; r < n; r += kSel) kept[r] = r;
    return;
  }
  uint32_t* keys = p.keys + ((int64_t)b * p.c.Hkv + h) * p.c.cap;
  for (int j = tid; j < len; j += kSel) {
    uint32_t key;
    if (j < p.n_global || j >= len - p.n_local) {
      key = 0xffffffffu;
    } else {
      const uint32_t t = (uint32_t)j / p.c.page;
      const int64_t pg = paged_page(p.c, p.c.table, p.c.ts, b, t);
      if (pg < 0) atomicCAS(p.err, 0, kErrPageEvict);
      key = pg < 0 ? 0u : weight_key(p.c.w[pg * p.c.wsp + h * p.c.wsh + ((uint32_t)j - t * p.c.page)]);
    }
    keys[j] = key;
  }
  // the n-th largest key and how many of its equals are kept
  if (tid == 0) {
    s_prefix = 0u;
    s_k = n;
  }
  uint32_t mask = 0u;
  for (int round = 0; round < 4; ++round) {
    const int shift = 24 - 8 * round;
    if (tid < 256) hist[tid] = 0u;
    __syncthreads();
    const uint32_t prefix = s_prefix;
    for (int j = tid; j < len; j += kSel) {
      const uint32_t key = keys[j];
      if ((key & mask) == prefix) atomicAdd(&hist[(key >> shift) & 255u], 1u);
    }
    __syncthreads();
    if (tid == 0) {
      int kk = s_k, d = 255;
      for (; d > 0; --d) {
        if ((int)hist[d] >= kk) break;
        kk -= (int)hist[d];
      }
      s_k = kk;
      s_prefix = prefix | ((uint32_t)d << shift);
    }
    __syncthreads();
    mask |= 255u << shift;
  }
  const uint32_t cut = s_prefix;
  const int equals = s_k;
  int carry = 0, tie_carry = 0;
  for (int j0 = 0; j0 < len; j0 += kSel) {
    const int j = j0 + tid;
    const uint32_t key = j < len ? keys[j] : 0u;
    const int tie = j < len && key == cut;
    int ties, all;
    const int tr = block_excl_sum(tie, sh, ties);
    const int keep = j < len && (key > cut || (tie && tie_carry + tr < equals));
    const int r = carry + block_excl_sum(keep, sh, all);
    if (keep) kept[r] = j;
    carry += all;
    tie_carry += ties;
  }
}

// One unit: the K and V row of one kept slot; 16-byte chunks, all loads before the stores.
template <int CH>
__global__ void __launch_bounds__(kCopy) paged_evict_copy_kernel(const EvP p) {
  constexpr int UNITS = kCopy / (2 * CH);
  const int tid = threadIdx.x;
  const int ch = tid % CH, is_v = (tid / CH) & 1, sub = tid / (2 * CH);
  const int h = blockIdx.y, b = blockIdx.z;
  const int n = (int)min((int64_t)paged_len(p.c, b), p.budget);
  const int r0 = (int)blockIdx.x * (UNITS * kIter) + sub;
  if (r0 >= n) return;
  const int32_t* kept = p.kept + ((int64_t)b * p.c.Hkv + h) * p.budget;
  uint4 x[kIter];
  float w[kIter];
  char* dst[kIter];
  float* wdst[kIter];
#pragma unroll
  for (int i = 0; i < kIter; ++i) {
    const int r = r0 + i * UNITS;
    dst[i] = nullptr;
    wdst[i] = nullptr;
    if (r >= n) continue;
    const uint32_t j = (uint32_t)kept[r];
    const uint32_t t = j / p.c.page, to = (uint32_t)r / p.c.page;
    const int64_t pg = paged_page(p.c, p.c.table, p.c.ts, b, t);
    const int64_t pd = (uint32_t)r < p.cap_out ? paged_page(p.c, p.table_out, p.tos, b, to) : -1;
    if (pg < 0 || pd < 0) {
      if (ch == 0) atomicCAS(p.err, 0, kErrPageEvict);
      continue;
    }
    const uint32_t slot = j - t * p.c.page, ds = (uint32_t)r - to * p.c.page;
    const char* s = is_v ? p.c.v + pg * p.c.vsp + h * p.c.vsh + slot * p.c.vsn
                         : p.c.k + pg * p.c.ksp + h * p.c.ksh + slot * p.c.ksn;
    dst[i] = (is_v ? p.c.v + pd * p.c.vsp + h * p.c.vsh + ds * p.c.vsn
                   : p.c.k + pd * p.c.ksp + h * p.c.ksh + ds * p.c.ksn) + ch * 16;
    x[i] = *reinterpret_cast<const uint4*>(s + ch * 16);
    if (is_v && ch == 0) {
      wdst[i] = p.c.w + pd * p.c.wsp + h * p.c.wsh + ds;
      w[i] = p.c.w[pg * p.c.wsp + h * p.c.wsh + slot];
    }
  }
#pragma unroll
  for (int i = 0; i < kIter; ++i) {
    if (dst[i]) *reinterpret_cast<uint4*>(dst[i]) = x[i];
    if (wdst[i]) *wdst[i] = w[i];
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

}  // namespace

size_t paged_evict_workspace_bytes(const sta_paged_cache* c, const sta_paged_evict_args* a) {
  if (check(c, a) != STA_OK) return 0;
  return (size_t)(c->batch * c->n_kv_heads) * (c->table_width * c->page_size) * 4 + 256;
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
  p.keys = reinterpret_cast<uint32_t*>(w + (256 - reinterpret_cast<uintptr_t>(w) % 256) % 256);
  p.err = device_error_word();
  if (!p.err) return fail(STA_ERR_CUDA, "sta_paged_evict: no device");
  paged_evict_select_kernel<<<dim3((unsigned)p.c.Hkv, (unsigned)p.c.B), kSel, 0, st>>>(p);
  const int ch = c->d * (c->dtype == STA_DTYPE_F32 ? 4 : 2) / 16;
  const int64_t per = (int64_t)kCopy / (2 * ch) * kIter;
  const int64_t most = p.c.cap < a->budget ? p.c.cap : a->budget;
  const dim3 grid((unsigned)((most + per - 1) / per), (unsigned)p.c.Hkv, (unsigned)p.c.B);
  if (ch == 8) paged_evict_copy_kernel<8><<<grid, kCopy, 0, st>>>(p);
  else if (ch == 16) paged_evict_copy_kernel<16><<<grid, kCopy, 0, st>>>(p);
  else paged_evict_copy_kernel<32><<<grid, kCopy, 0, st>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? STA_OK : fail(STA_ERR_CUDA, cudaGetErrorString(e));
}

}  // namespace sta
