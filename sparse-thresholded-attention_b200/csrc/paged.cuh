// The paged key-value cache on the device: slot -> page lookup and the argument checks that the
// append, decode and evict kernels share.
#pragma once

#include "common.cuh"
#include "sta_internal.h"

namespace sta {

enum : int { kErrPageAppend = 201, kErrPageDecode = 202, kErrPageEvict = 203, kErrPageTwice = 204 };

struct PagedView {
  char* k;
  char* v;
  int64_t ksp, ksh, ksn, vsp, vsh, vsn;  // bytes
  float* w;
  int64_t wsp, wsh;                      // elements
  const int32_t* table;
  int64_t ts;
  const int32_t* lens;
  int64_t n_pages;
  uint32_t page, width, cap;             // page size, entries of a table row, slots it can name
  int B, Hkv;
};

inline PagedView paged_view(const sta_paged_cache* c) {
  const int64_t es = c->dtype == STA_DTYPE_F32 ? 4 : 2;
  PagedView v;
  v.k = static_cast<char*>(c->k);
  v.v = static_cast<char*>(c->v);
  v.ksp = c->k_stride_p * es; v.ksh = c->k_stride_h * es; v.ksn = c->k_stride_n * es;
  v.vsp = c->v_stride_p * es; v.vsh = c->v_stride_h * es; v.vsn = c->v_stride_n * es;
  v.w = c->weights; v.wsp = c->weights_stride_p; v.wsh = c->weights_stride_h;
  v.table = c->table; v.ts = c->table_stride;
  v.lens = c->lens;
  v.n_pages = c->n_pages;
  v.page = (uint32_t)c->page_size;
  v.width = (uint32_t)c->table_width;
  v.cap = (uint32_t)(c->table_width * c->page_size);
  v.B = (int)c->batch;
  v.Hkv = (int)c->n_kv_heads;
  return v;
}

__device__ __forceinline__ int paged_len(const PagedView& c, int b) {
  const int n = c.lens[b];  // (an append may store the new length in place: not a read-only load)
  return n < 0 ? 0 : ((uint32_t)n > c.cap ? (int)c.cap : n);
}

// page number in entry t of sequence b's table row, -1 where it lies outside the pool
__device__ __forceinline__ int64_t paged_page(const PagedView& c, const int32_t* table, int64_t ts,
                                              int b, uint32_t t) {
  const int64_t pg = __ldg(table + b * ts + t);
  return pg >= 0 && pg < c.n_pages ? pg : -1;
}

// Where a page stands in a table: (sequence, entry).  Finding pages that stand there twice takes an
// array of one place per page that nobody clears: every entry in use leaves its place at its page,
// a later kernel looks whether its own is still there.  Of two entries that name one page exactly
// one finds its own.  Whether a page is in use at all shows in the table entry that its place names
// (where nobody left one, any place that an earlier call's scratch names is checked the same way).
__device__ __forceinline__ void leave_place(int2* places, int64_t n_pages, int32_t pg, int b, uint32_t t) {
  if (pg >= 0 && pg < n_pages) places[pg] = make_int2(b, (int)t);
}
__device__ __forceinline__ void leave_places(int2* places, int64_t n_pages, const int32_t* row, int b,
                                             uint32_t entries, uint32_t first, uint32_t step) {
  for (uint32_t t = first; t < entries; t += step) leave_place(places, n_pages, __ldg(row + t), b, t);
}
__device__ __forceinline__ uint32_t entries_of(const PagedView& c, int len) {
  return len > 0 ? (uint32_t)(len - 1) / c.page + 1 : 0u;
}
__device__ __forceinline__ bool is_place(int2 x, int b, uint32_t t) { return x.x == b && x.y == (int)t; }

// Moves up to 32 rows of K and V by one warp: lane l has row l's byte offsets (ks < 0: no row), `n`
// rows in all.  Neighbouring lanes hold the 16-byte chunks (CH of a row) of K, then of V; four
// loads of a lane are in flight before the first store.  VEC: sources lie on 16-byte boundaries;
// otherwise they are read by elements of `es` bytes.
template <int CH, bool VEC>
__device__ __forceinline__ void move_rows(const char* ksrc, const char* vsrc, char* kdst, char* vdst,
                                          int64_t ks, int64_t vs, int64_t kd, int64_t vd, int n, int es) {
  constexpr int LPU = 2 * CH < 32 ? 2 * CH : 32;  // lanes of a row
  constexpr int PER = 32 / LPU, PASS = 2 * CH / LPU, U = 4 / PASS;
  const int lane = threadIdx.x & 31, sub = lane / LPU, ch = lane % CH;
  const bool is_v = PASS == 1 && (lane / CH) % 2 == 1;
#pragma unroll 1
  for (int i0 = 0; i0 < n; i0 += U * PER) {
    uint4 x[U][PASS];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * PER + sub;
      const int64_t a = __shfl_sync(0xffffffffu, ks, i & 31), c = __shfl_sync(0xffffffffu, vs, i & 31);
#pragma unroll
      for (int q = 0; q < PASS; ++q) {
        const bool v = PASS == 1 ? is_v : q == 1;
        const char* s = (v ? vsrc + c : ksrc + a) + ch * 16;
        if (i >= n || a < 0) continue;
        if (VEC) {
          x[u][q] = __ldcs(reinterpret_cast<const uint4*>(s));
        } else if (es == 4) {
          const uint32_t* e = reinterpret_cast<const uint32_t*>(s);
          x[u][q] = make_uint4(e[0], e[1], e[2], e[3]);
        } else {
          const uint16_t* e = reinterpret_cast<const uint16_t*>(s);
          x[u][q] = make_uint4(e[0] | (uint32_t)e[1] << 16, e[2] | (uint32_t)e[3] << 16,
                               e[4] | (uint32_t)e[5] << 16, e[6] | (uint32_t)e[7] << 16);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * PER + sub;
      const int64_t a = __shfl_sync(0xffffffffu, kd, i & 31), c = __shfl_sync(0xffffffffu, vd, i & 31);
      const int64_t from = __shfl_sync(0xffffffffu, ks, i & 31);  // (by all lanes, rows or not)
      const bool in = i < n && from >= 0;
#pragma unroll
      for (int q = 0; q < PASS; ++q) {
        const bool v = PASS == 1 ? is_v : q == 1;
        if (in) *reinterpret_cast<uint4*>((v ? vdst + c : kdst + a) + ch * 16) = x[u][q];
      }
    }
  }
}

// Programmatic launches: every kernel of the paged cache may be set up while the one ahead of it in
// the stream runs.  grid_wait: what the kernel ahead, and all before it, wrote is there from here
// on; every block passes it.  grid_dependents: the next kernel may be set up.  The first kernel of
// a call waits before it lets the next one start, so that the later kernels of the call may read
// what the call was given (not what their predecessor writes) ahead of their own wait.
__device__ __forceinline__ void grid_dependents() { asm volatile("griddepcontrol.launch_dependents;"); }
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Launches a kernel that may begin before the one ahead of it in the stream has ended (it waits
// for that kernel's results itself), so that its launch does not add to the call.
template <typename K, typename P>
inline cudaError_t launch_behind(K kernel, dim3 grid, int threads, const P& p, cudaStream_t st,
                                 size_t smem = 0, unsigned cluster = 0) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

// Lets a kernel have `bytes` of dynamic shared memory; asked for once per device (`ready`).
template <typename K>
inline cudaError_t allow_smem(K kernel, int bytes, bool (&ready)[64]) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || (dev < 64 && ready[dev])) return e;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev < 64) ready[dev] = true;
  return e;
}

inline int paged_check(const sta_paged_cache* c) {
  if (!c || !c->k || !c->v || (c->batch != 0 && (!c->table || !c->lens)))
    return fail(STA_ERR_ARG, "sta_paged: null pointer");
  if (c->d != 64 && c->d != 128) return fail(STA_ERR_UNSUPPORTED, "sta_paged: d must be 64 or 128");
  if (c->dtype != STA_DTYPE_F32 && c->dtype != STA_DTYPE_BF16)
    return fail(STA_ERR_UNSUPPORTED, "sta_paged: dtype must be f32 or bf16");
  if (c->n_pages <= 0 || c->n_kv_heads <= 0 || c->batch < 0 || c->table_width <= 0)
    return fail(STA_ERR_ARG, "sta_paged: bad sizes");
  if (c->page_size < 1 || c->page_size > 65536)
    return fail(STA_ERR_UNSUPPORTED, "sta_paged: page_size must lie in 1 .. 65536");
  if (c->table_width >= ((int64_t)1 << 31) || c->table_width * c->page_size > ((int64_t)1 << 31) - 65)
    return fail(STA_ERR_UNSUPPORTED, "sta_paged: table_width * page_size must stay below 2^31 - 64");
  if (c->n_kv_heads > 65535 || c->batch > ((int64_t)1 << 24))
    return fail(STA_ERR_UNSUPPORTED, "sta_paged: too many kv heads / sequences");
  const int64_t es = c->dtype == STA_DTYPE_F32 ? 4 : 2;
  const int64_t strides[6] = {c->k_stride_p, c->k_stride_h, c->k_stride_n,
                              c->v_stride_p, c->v_stride_h, c->v_stride_n};
  for (int64_t s : strides)
    if (s < 0 || s * es % 16)
      return fail(STA_ERR_ARG, "sta_paged: K / V strides must be non-negative multiples of 16 bytes");
  if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15u)
    return fail(STA_ERR_ARG, "sta_paged: K / V must start on a 16-byte boundary");
  return STA_OK;
}

// Tensors that a call writes: a stride of zero (heads or pages broadcast) would send the rows of
// several slots to one place.
inline int paged_check_weights_written(const sta_paged_cache* c) {
  if ((c->n_pages > 1 && c->weights_stride_p == 0) || (c->n_kv_heads > 1 && c->weights_stride_h == 0))
    return fail(STA_ERR_ARG, "sta_paged: weights are written, their strides must not be zero");
  return STA_OK;
}

inline int paged_check_rows_written(const sta_paged_cache* c) {
  if ((c->n_pages > 1 && (c->k_stride_p == 0 || c->v_stride_p == 0)) ||
      (c->n_kv_heads > 1 && (c->k_stride_h == 0 || c->v_stride_h == 0)) ||
      (c->page_size > 1 && (c->k_stride_n == 0 || c->v_stride_n == 0)))
    return fail(STA_ERR_ARG, "sta_paged: K / V are written, their strides must not be zero");
  return c->weights ? paged_check_weights_written(c) : STA_OK;
}

}  // namespace sta
