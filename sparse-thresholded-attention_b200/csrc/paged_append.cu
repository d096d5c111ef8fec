// Rows of new tokens into the pages of their sequences.
//
// A pure copy: every row is read once and written once (2 * d * element size bytes each for K
// and V), so HBM bounds it for prompts and launch latency for single tokens.  A warp takes 8 or 32
// (token, kv head) rows, kv heads of a token next to each other (the order in which a projection
// leaves them): each lane looks up one row's page, then the warp moves the rows.  Sources that
// are not 16-byte aligned take element loads (prompts of 52 000 tokens, 8 kv heads, bf16: 108 us
// where 16-byte loads took 75).
//
// Measured: two prompts, 52 000 tokens in all, 8 kv heads of d = 128, bf16: 71 us, 424 MB moved at
// 6.0 TB/s; one token of each of 64 sequences: 4 us on the device, 8 us a call from Python.
#include <initializer_list>

#include "paged.cuh"

namespace sta {

namespace {

constexpr int kThreads = 256;
// (token, kv head) rows of a warp, of a block.  Eight keep many small blocks in flight, which evens
// out ragged prompts (d = 128, bf16 prompts as above: 71 us, with 32 rows 75); rows of
// 128 bytes are too little work for that (d = 64: 49 us with 16, 40 with 32).
constexpr int warp_rows(int ch) { return ch == 8 ? 32 : 8; }
constexpr int block_rows(int ch) { return kThreads / 32 * warp_rows(ch); }

struct AppP {
  PagedView c;
  const char* k;
  const char* v;
  int64_t ksb, ksh, ksn, vsb, vsh, vsn;  // bytes
  uint32_t n;
  const int32_t* counts;
  int32_t* lens_out;
  int store_lens;  // the first block of a sequence stores its new length
  int es;
  int* err;
};

__device__ __forceinline__ int new_len(const AppP& p, int b, int len, int& cnt) {
  cnt = (int)p.n;
  if (p.counts) cnt = min(max(p.counts[b], 0), (int)p.n);  // (may be overwritten: not a read-only load)
  return (uint32_t)len + (uint32_t)cnt > p.c.cap ? (int)p.c.cap : len + cnt;
}

// CH: 16-byte chunks of a row (8, 16 or 32)
template <int CH, bool VEC>
__global__ void __launch_bounds__(kThreads, 4) paged_append_kernel(const AppP p) {
  constexpr int ROWS = warp_rows(CH);
  const int tid = threadIdx.x, lane = tid & 31;
  grid_wait();
  grid_dependents();
  for (int b = blockIdx.y; b < p.c.B; b += gridDim.y) {
    const int len = paged_len(p.c, b);
    int cnt;
    const int total = new_len(p, b, len, cnt);
    const int64_t units = (int64_t)cnt * p.c.Hkv, u0 = (int64_t)blockIdx.x * block_rows(CH) + (tid >> 5) * ROWS;
    const int64_t u = u0 + lane;
    if (u0 < units) {
      int64_t ks = -1, vs = 0, kd = 0, vd = 0;
      if (u < units && lane < ROWS) {
        const uint32_t r = (units >> 32) == 0 ? (uint32_t)u / (uint32_t)p.c.Hkv : (uint32_t)(u / p.c.Hkv);
        const uint32_t h = (uint32_t)(u - (int64_t)r * p.c.Hkv), j = (uint32_t)len + r, t = j / p.c.page;
        const int64_t pg = j < p.c.cap ? paged_page(p.c, p.c.table, p.c.ts, b, t) : -1;
        if (pg < 0) {
          atomicCAS(p.err, 0, kErrPageAppend);
        } else {
          const uint32_t slot = j - t * p.c.page;
          ks = h * p.ksh + r * p.ksn;
          vs = h * p.vsh + r * p.vsn;
          kd = pg * p.c.ksp + h * p.c.ksh + slot * p.c.ksn;
          vd = pg * p.c.vsp + h * p.c.vsh + slot * p.c.vsn;
          if (p.c.w) p.c.w[pg * p.c.wsp + h * p.c.wsh + slot] = 0.f;
        }
      }
      move_rows<CH, VEC>(p.k + b * p.ksb, p.v + b * p.vsb, p.c.k, p.c.v, ks, vs, kd, vd,
                         (int)min((int64_t)ROWS, units - u0), p.es);
    }
    if (p.store_lens && blockIdx.x == 0) {
      __syncthreads();  // lens_out may be lens or counts: every thread of the (then only) block has read them
      if (tid == 0) p.lens_out[b] = total;
    }
  }
}

__global__ void __launch_bounds__(kThreads) paged_lens_kernel(const AppP p) {
  const int b = blockIdx.x * kThreads + threadIdx.x;
  grid_wait();
  if (b >= p.c.B) return;
  int cnt;
  p.lens_out[b] = new_len(p, b, paged_len(p.c, b), cnt);
}

template <int CH>
cudaError_t launch(const AppP& p, bool vec, dim3 grid, cudaStream_t st) {
  return vec ? launch_behind(paged_append_kernel<CH, true>, grid, kThreads, p, st)
             : launch_behind(paged_append_kernel<CH, false>, grid, kThreads, p, st);
}

}  // namespace

int paged_append(const sta_paged_cache* c, const sta_paged_append_args* a, cudaStream_t st) {
  int rc = paged_check(c);
  if (rc == STA_OK) rc = paged_check_rows_written(c);
  if (rc != STA_OK) return rc;
  if (!a || (c->batch > 0 && !a->lens_out)) return fail(STA_ERR_ARG, "sta_paged_append: null pointer");
  if (a->n < 0 || a->n > ((int64_t)1 << 31) - 65) return fail(STA_ERR_ARG, "sta_paged_append: bad n");
  for (int64_t x : {a->k_stride_h, a->k_stride_n, a->v_stride_h, a->v_stride_n})
    if (x < 0) return fail(STA_ERR_ARG, "sta_paged_append: negative stride");
  if (a->n > 0 && c->batch > 0 && (!a->k || !a->v)) return fail(STA_ERR_ARG, "sta_paged_append: null pointer");
  if (a->lens_out != c->lens && a->lens_out < c->lens + c->batch && c->lens < a->lens_out + c->batch)
    return fail(STA_ERR_ARG, "sta_paged_append: lens_out overlaps lens without being it");
  if (a->counts && a->lens_out != a->counts && a->lens_out < a->counts + c->batch && a->counts < a->lens_out + c->batch)
    return fail(STA_ERR_ARG, "sta_paged_append: lens_out overlaps counts without being it");
  if (c->batch == 0) return STA_OK;
  AppP p;
  p.c = paged_view(c);
  p.es = c->dtype == STA_DTYPE_F32 ? 4 : 2;
  p.k = static_cast<const char*>(a->k);
  p.v = static_cast<const char*>(a->v);
  p.ksb = a->k_stride_b * p.es; p.ksh = a->k_stride_h * p.es; p.ksn = a->k_stride_n * p.es;
  p.vsb = a->v_stride_b * p.es; p.vsh = a->v_stride_h * p.es; p.vsn = a->v_stride_n * p.es;
  p.n = (uint32_t)a->n;
  p.counts = a->counts;
  p.lens_out = a->lens_out;
  p.err = page_error_word();
  if (!p.err) return fail(STA_ERR_CUDA, "sta_paged_append: no device");
  const bool vec = ((reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v) | p.ksb |
                     p.ksh | p.ksn | p.vsb | p.vsh | p.vsn) & 15) == 0;
  const int ch = c->d * p.es / 16;
  const int64_t gx = (a->n * c->n_kv_heads + block_rows(ch) - 1) / block_rows(ch);
  if (gx > ((int64_t)1 << 31) - 1) return fail(STA_ERR_UNSUPPORTED, "sta_paged_append: too many rows");
  const dim3 grid((unsigned)(gx > 0 ? gx : 1), (unsigned)(c->batch < 65535 ? c->batch : 65535));
  // a length or count that is overwritten in place is read by one block only, or the lengths are
  // stored by a second launch
  p.store_lens = (a->lens_out != c->lens && a->lens_out != a->counts) || grid.x == 1;
  cudaError_t e = ch == 8 ? launch<8>(p, vec, grid, st)
                          : (ch == 16 ? launch<16>(p, vec, grid, st) : launch<32>(p, vec, grid, st));
  if (e == cudaSuccess && !p.store_lens)
    e = launch_behind(paged_lens_kernel, dim3((unsigned)((c->batch + kThreads - 1) / kThreads)), kThreads, p, st);
  return e == cudaSuccess ? STA_OK : fail(STA_ERR_CUDA, cudaGetErrorString(e));
}

}  // namespace sta
