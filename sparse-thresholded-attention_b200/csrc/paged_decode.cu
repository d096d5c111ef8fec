// Dense attention of one new token per sequence over a paged cache of raw keys.
//
//   s_j = scale * (R(p_i) q) . (R(p_j) k_j)     p = softmax(s)     out = sum_j p_j v_j
//
// Split over the length: the 64-key tiles of all (sequence, kv head, q-head group) segments form
// one list, cut into equal shares for a fixed number of CTAs, so that ragged batches and single
// long sequences load the whole GPU alike without the host knowing a length.  A CTA walks its
// share with an online softmax per segment; a segment that lies inside one share is finished
// there, others leave (max, sum, unnormalised output) partials that a second launch joins.
//
// Rotation: within a tile p_j = p_0 + t * pos_scale with t = 0 .. 63, and only differences of
// positions matter, so keys are rotated by the tile-local t * pos_scale (one 64 x d/2 table for
// the whole call) and the query once per tile by p_i - p_0 (64-bit angles).  Dual Chunk
// Attention positions fit the same scheme: a tile lies in one chunk, whose relation to the
// query's chunk sets p_i.
//
// Each key and value row is read from HBM once.  The bf16 kernel comes to 5 TB/s and is bound by the
// instructions it issues per key and, for short sequences, by its fixed part (there).  The f32 kernel
// here is bound by its shared memory reads and a barrier per tile: 65536 keys of 8 kv heads, d = 128,
// take 110 us with one q head each (537 MB, 4.9 TB/s), 132 us with four, 166 us with eight.
#include <float.h>
#include <stdlib.h>

#include <type_traits>

#include "paged_decode.cuh"

namespace sta {

namespace {

// Sums of NV values (a power of two up to 32) over the warp: lane l returns the sum of value
// l / (32 / NV).  Each round halves the values a lane carries, so NV = 32 takes 31 shuffles.
template <int NV>
__device__ __forceinline__ float warp_reduce(float (&v)[NV]) {
  const int lane = threadIdx.x & 31;
  int n = NV;
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) {
    if (n > 1) {
      n >>= 1;
      const bool hi = lane & o;
#pragma unroll
      for (int i = 0; i < NV / 2; ++i) {
        if (i >= n) break;
        const float send = hi ? v[i] : v[i + n];
        const float mine = hi ? v[i + n] : v[i];
        v[i] = mine + __shfl_xor_sync(0xffffffffu, send, o);
      }
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
    }
  }
  return v[0];
}

// The f32 kernel: CUDA cores, so that scores keep full fp32 products (a warp has 4 or 8 keys of a
// tile; a lane holds D / 32 dims and reduces its partial dots with the other lanes').
template <int D, int GT>
struct F32 {
  // one CTA per SM at d = 128 (its ring takes 192 KB), of 16 warps (8 where 8 heads' accumulators
  // need the registers: 16 warps spill and take 204 us instead of 165 at 65536 keys of 8 kv heads);
  // two CTAs of 8 warps at d = 64
  static constexpr int THREADS = D == 128 && GT < 8 ? 512 : 256, WARPS = THREADS / 32;
  static constexpr int KEYS = kTile / WARPS;  // keys of a tile per warp
};

template <int D, int GT>
struct Smem {
  static constexpr int STAGES = 3, NWF = F32<D, GT>::WARPS, KPW = F32<D, GT>::KEYS;
  static constexpr int CH = D / 4;   // 16-byte chunks of a row
  uint4 kv[STAGES][2][kTile * CH];   // K rows, V rows (also the flush's scratch)
  float q[2][GT][D];                 // rotated, scaled queries of this tile and the next
  float p[NWF][KPW][GT];  // a warp's probabilities
  float m[NWF][GT], l[NWF][GT];
  int64_t koff[2][kTile], voff[2][kTile];
};

template <int D, int GT>
__global__ void __launch_bounds__(F32<D, GT>::THREADS) paged_decode_f32_kernel(const PDecP p) {
  using S = Smem<D, GT>;
  constexpr int NTH = F32<D, GT>::THREADS, NWF = F32<D, GT>::WARPS, KPW = F32<D, GT>::KEYS;
  constexpr int HALF = D / 2, CH = S::CH, ST = S::STAGES;
  constexpr int FP = HALF / 32;               // frequencies of a lane
  constexpr int KB = KPW * GT > 32 ? 32 / GT : KPW, NV = KB * GT;  // keys of one reduction
  constexpr int LPV = 32 / NV;                // lanes that hold the same value
  constexpr int QH = GT * HALF / NTH > 0 ? GT * HALF / NTH : 1;  // q pairs of a thread
  extern __shared__ __align__(128) unsigned char smem_raw[];
  S& sm = *reinterpret_cast<S*>(smem_raw);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  grid_wait();
  grid_dependents();
  int64_t me;
  const Share share = find_share<false>(p, first_len(p.c), me);
  const int count = share.count;
  if (count == 0) return;
  Place cur = share.at;
  Place qa = cur, oa = cur;  // where queries and row offsets stand
  int q_it = 0, l_it = 0, o_it = 0;

  // ---- row offsets of a tile (threads 0 .. 63), -1: no row, -2: a page outside the pool.  The
  // table entry is asked for in lookup() and used in offsets(), a tile's work later.
  int32_t entry = -1;
  auto lookup = [&]() {
    if (o_it < count && tid < kTile) {
      const int j = oa.n * kTile + tid;
      if (j < oa.len) entry = __ldg(p.c.table + oa.b * p.c.ts + (uint32_t)j / p.c.page);
    }
  };
  auto offsets = [&]() {
    if (o_it < count) {
      if (tid < kTile) {
        const int j = oa.n * kTile + tid;
        int64_t ko = -1, vo = -1;
        if (j < oa.len) {
          if (entry < 0 || entry >= p.c.n_pages) {
            ko = -2;
            atomicCAS(p.err, 0, kErrPageDecode);
          } else {
            const int64_t slot = (uint32_t)j % p.c.page, h = oa.h;
            ko = entry * p.c.ksp + h * p.c.ksh + slot * p.c.ksn;
            vo = entry * p.c.vsp + h * p.c.vsh + slot * p.c.vsn;
          }
        }
        sm.koff[o_it & 1][tid] = ko;
        sm.voff[o_it & 1][tid] = vo;
      }
      step(p, oa);
    }
    ++o_it;
  };
  // ---- copies of a tile's rows (rows without data are zero; of a bad page, K is NaN)
  auto loads = [&]() {
    if (l_it < count) {
      const int st = l_it % ST;
#pragma unroll 4
      for (int i = tid; i < kTile * CH; i += NTH) {
        const int row = i / CH, ch = i % CH;
        const int64_t ko = sm.koff[l_it & 1][row], vo = sm.voff[l_it & 1][row];
        cp_async16(&sm.kv[st][1][i], p.c.v + (vo >= 0 ? vo + ch * 16 : 0), vo >= 0 ? 16 : 0);
        if (ko == -2) {
          sm.kv[st][0][i] = make_uint4(0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u);
        } else {
          cp_async16(&sm.kv[st][0][i], p.c.k + (ko >= 0 ? ko + ch * 16 : 0), ko >= 0 ? 16 : 0);
        }
      }
    }
    asm volatile("cp.async.commit_group;\n" ::: "memory");
    ++l_it;
  };
  // ---- queries of a tile: rotated by p_i - p_0
  float q1[QH], q2[QH];
  const int qf = tid % HALF, qg = tid / HALF;  // frequency, first head (step NTH / HALF)
  auto queries = [&]() {
    if (q_it < count) {
      if (q_it == 0 || qa.n == 0) {
        const int h0 = qa.h * p.G + qa.grp * GT;
#pragma unroll
        for (int i = 0; i < QH; ++i) {
          const int g = qg + i * (NTH / HALF);
          const bool in = g < GT && qa.grp * GT + g < p.G;
          const float* src = static_cast<const float*>(p.q) + qa.b * p.qsb + (h0 + g) * p.qsh;
          q1[i] = in ? (src[qf]) * p.qscale : 0.f;
          q2[i] = in ? (src[qf + HALF]) * p.qscale : 0.f;
        }
      }
      float c, s;
      turn(query_offset(p, qa.len, qa.n), __ldg(p.inv_freq + qf), c, s);
#pragma unroll
      for (int i = 0; i < QH; ++i) {
        const int g = qg + i * (NTH / HALF);
        if (g < GT) {
          sm.q[q_it & 1][g][qf] = q1[i] * c - q2[i] * s;
          sm.q[q_it & 1][g][qf + HALF] = q2[i] * c + q1[i] * s;
        }
      }
      step(p, qa);
    }
    ++q_it;
  };

  for (int i = 0; i < ST - 1; ++i) {
    lookup();
    offsets();
    __syncthreads();
    loads();
  }
  lookup();
  offsets();
  queries();
  float2 rot[KPW][FP];  // cos / sin of the warp's key offsets at the lane's frequencies
#pragma unroll
  for (int t = 0; t < KPW; ++t)
#pragma unroll
    for (int e = 0; e < FP; ++e)
      turn((double)(warp * KPW + t) * p.pos_scale, __ldg(p.inv_freq + lane * FP + e), rot[t][e].x,
           rot[t][e].y);

  float acc[GT][2 * FP];
  float mx = -INFINITY, sum = 0.f;  // of head (lane / LPV) % GT, replicated over its lanes
#pragma unroll
  for (int g = 0; g < GT; ++g)
#pragma unroll
    for (int e = 0; e < 2 * FP; ++e) acc[g][e] = 0.f;

  for (int it = 0; it < count; ++it) {
    asm volatile("cp.async.wait_group %0;\n" ::"n"(ST - 2) : "memory");
    __syncthreads();
    loads();
    lookup();
    const int st = it % ST;
    const float* ks = reinterpret_cast<const float*>(sm.kv[st][0]);
    const float* vs = reinterpret_cast<const float*>(sm.kv[st][1]);
    float qr[GT][2 * FP];
#pragma unroll
    for (int g = 0; g < GT; ++g)
#pragma unroll
      for (int e = 0; e < FP; ++e) {
        qr[g][e] = sm.q[it & 1][g][lane * FP + e];
        qr[g][FP + e] = sm.q[it & 1][g][HALF + lane * FP + e];
      }
    const int valid = cur.len - cur.n * kTile;  // keys of this tile
    float* sc = p.scores
        ? p.scores + ((((int64_t)cur.b * p.c.Hkv * p.NG + cur.h * p.NG + cur.grp) * p.cap_tiles + cur.n) * p.SG) * kTile
        : nullptr;
#pragma unroll
    for (int kb = 0; kb < KPW / KB; ++kb) {
      const int key0 = warp * KPW + kb * KB;
      float v[NV];
#pragma unroll
      for (int kk = 0; kk < KB; ++kk) {
        const int t = key0 + kk;
        float r1[FP], r2[FP];
#pragma unroll
        for (int e = 0; e < FP; ++e) {
          const float x1 = (ks[t * D + lane * FP + e]);
          const float x2 = (ks[t * D + HALF + lane * FP + e]);
          const float2 cs = rot[kb * KB + kk][e];
          r1[e] = x1 * cs.x - x2 * cs.y;
          r2[e] = x2 * cs.x + x1 * cs.y;
        }
#pragma unroll
        for (int g = 0; g < GT; ++g) {
          float d = 0.f;
#pragma unroll
          for (int e = 0; e < FP; ++e) d = fmaf(qr[g][FP + e], r2[e], fmaf(qr[g][e], r1[e], d));
          v[kk * GT + g] = d;
        }
      }
      float s = warp_reduce<NV>(v);
      const int idx = lane / LPV, kk = idx / GT, g = idx % GT;
      if (key0 + kk >= valid) s = -INFINITY;
      if (sc && g < p.SG && (LPV == 1 || lane % LPV == 0)) sc[g * kTile + key0 + kk] = s;
      float mb = s;
#pragma unroll
      for (int o = GT * LPV; o < 32; o <<= 1) mb = fmaxf(mb, __shfl_xor_sync(0xffffffffu, mb, o));
      const float mn = fmaxf(mx, mb), ms = mn == -INFINITY ? 0.f : mn;
      const float a = exp2f(mx - ms), e = exp2f(s - ms);
      float se = e;
#pragma unroll
      for (int o = GT * LPV; o < 32; o <<= 1) se += __shfl_xor_sync(0xffffffffu, se, o);
      sum = sum * a + se;
      mx = mn;
      if (LPV == 1 || lane % LPV == 0) sm.p[warp][kk][g] = e;
#pragma unroll
      for (int gg = 0; gg < GT; ++gg) {
        const float ag = __shfl_sync(0xffffffffu, a, gg * LPV);
#pragma unroll
        for (int x = 0; x < 2 * FP; ++x) acc[gg][x] *= ag;
      }
      __syncwarp();
#pragma unroll
      for (int k2 = 0; k2 < KB; ++k2) {
        const int t = key0 + k2;
        float vv[2 * FP];
#pragma unroll
        for (int x = 0; x < FP; ++x) {
          vv[x] = (vs[t * D + lane * FP + x]);
          vv[FP + x] = (vs[t * D + HALF + lane * FP + x]);
        }
#pragma unroll
        for (int gg = 0; gg < GT; ++gg) {
          const float pr = sm.p[warp][k2][gg];
#pragma unroll
          for (int x = 0; x < 2 * FP; ++x) acc[gg][x] = fmaf(pr, vv[x], acc[gg][x]);
        }
      }
      __syncwarp();
    }
    const bool seg_end = cur.n == cur.units - 1;
    if (seg_end || it == count - 1) {
      // the warps' partial results of this segment, joined and stored
      float* part_acc = reinterpret_cast<float*>(sm.kv[st][0]);  // [warp][head][d]
      __syncthreads();
      const int idx = lane / LPV;
      if (idx < GT && lane % LPV == 0) {
        sm.m[warp][idx] = mx;
        sm.l[warp][idx] = sum;
      }
#pragma unroll
      for (int g = 0; g < GT; ++g)
#pragma unroll
        for (int x = 0; x < FP; ++x) {
          part_acc[(warp * GT + g) * D + lane * FP + x] = acc[g][x];
          part_acc[(warp * GT + g) * D + HALF + lane * FP + x] = acc[g][FP + x];
        }
      __syncthreads();
      const bool started = cur.n <= it;  // the segment's first tile lies in this share
      const bool whole = seg_end && started;
      const int slot = 2 * blockIdx.x + (started ? 1 : 0);
      const int h0 = cur.h * p.G + cur.grp * GT;
      for (int i = tid; i < GT * D; i += NTH) {
        const int g = i / D, d = i % D;
        if (cur.grp * GT + g >= p.G) continue;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < NWF; ++w) M = fmaxf(M, sm.m[w][g]);
        const float ms = M == -INFINITY ? 0.f : M;
        float L = 0.f, o = 0.f;
#pragma unroll
        for (int w = 0; w < NWF; ++w) {
          const float f = exp2f(sm.m[w][g] - ms);
          L += sm.l[w][g] * f;
          o += part_acc[(w * GT + g) * D + d] * f;
        }
        if (whole) {
          store_out(static_cast<float*>(p.out) + ((int64_t)cur.b * p.H + h0 + g) * D + d, o / L);
          if (d == 0) p.ml[(int64_t)cur.b * p.H + h0 + g] = make_float2(ms, 1.f / L);
        } else {
          p.part[((int64_t)slot * GT + g) * D + d] = o;
          if (d == 0) p.part_ml[(int64_t)slot * GT + g] = make_float2(M, L);
        }
      }
#pragma unroll
      for (int g = 0; g < GT; ++g)
#pragma unroll
        for (int x = 0; x < 2 * FP; ++x) acc[g][x] = 0.f;
      mx = -INFINITY;
      sum = 0.f;
    }
    offsets();
    queries();
    step(p, cur);
  }
}

constexpr int kUpd = 256;       // threads of the weights update, four keys each

// The shares [w0, w1] that cut a segment; one share (w0 == w1) has finished it.  Of the others, w0
// holds its first unit and left partial 2 w0 + 1; share w behind it left partial 2 w.
struct Cut {
  int64_t w0, w1;
};

// the share of unit t: share_begin(w) <= t < share_begin(w + 1), decided without a division
__device__ __forceinline__ int64_t share_of(int64_t total, int64_t t, int64_t W) {
  int64_t w = (int64_t)((double)t * (double)W / (double)total);
  while (total * (w + 1) < (t + 1) * W) ++w;
  while (total * w >= (t + 1) * W) --w;
  return w;
}

__device__ __forceinline__ Cut cut_of(const PDecP& p, int b, int hg, int units) {
  int64_t before;
  const int64_t total = scan_lengths(p, b, &before), W = n_shares(p, total);
  const int64_t s0 = before + (int64_t)hg * units;
  return {share_of(total, s0, W), share_of(total, s0 + units - 1, W)};
}

__device__ __forceinline__ int64_t slot_of(const Cut& c, int64_t w) { return 2 * w + (w == c.w0 ? 1 : 0); }

// One block per (sequence, q head) joins the partials of the shares that cut its segment: each of
// NW warps joins every NW-th, four of them in flight, then the warps' results are joined.  Empty
// sequences give zeros.
template <int D, typename TV, int NW>
__global__ void __launch_bounds__(NW * 32) paged_join_kernel(const PDecP p) {
  constexpr int V = D / 32, U = 4;
  __shared__ float s_o[NW][D];
  __shared__ float2 s_ml[NW];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  grid_dependents();
  const int b = blockIdx.x / p.H, h = blockIdx.x % p.H;
  const int g0 = h % p.G, hg = h / p.G * p.NG + g0 / p.GT, g = g0 % p.GT;
  const int units = n_units(p, paged_len(p.c, b));
  TV* out = static_cast<TV*>(p.out) + (int64_t)blockIdx.x * D;
  if (units == 0) {
    grid_wait();
    if (tid < D) store_out(out + tid, 0.f);
    return;
  }
  const Cut c = cut_of(p, b, hg, units);
  // (scratch of this call, which the first kernel's wait has handed over)
  if (p.places)
    leave_places(p.places, p.c.n_pages, p.c.table + b * p.c.ts, b, entries_of(p.c, paged_len(p.c, b)),
                 (uint32_t)(h * NW * 32 + tid), (uint32_t)(p.H * NW * 32));
  grid_wait();
  if (c.w0 == c.w1) return;
  float M = -INFINITY, L = 0.f, o[V];
#pragma unroll
  for (int i = 0; i < V; ++i) o[i] = 0.f;
  // a warp looks at 32 partials at a time and loads those that are not empty, up to U at once
  for (int64_t w = c.w0 + warp; w <= c.w1; w += NW * 32) {
    const int64_t mine = w + (int64_t)lane * NW;
    float2 my = make_float2(-INFINITY, 0.f);
    if (mine <= c.w1) my = p.part_ml[slot_of(c, mine) * p.GT + g];
    uint32_t full = __ballot_sync(0xffffffffu, my.y != 0.f);
    while (full) {
      float x[U][V];
      float2 ml[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int src = full ? __ffs(full) - 1 : -1;
        full &= full - 1u;
        ml[u].x = __shfl_sync(0xffffffffu, my.x, src & 31);
        ml[u].y = __shfl_sync(0xffffffffu, my.y, src & 31);
        if (src < 0) ml[u] = make_float2(-INFINITY, 0.f);
        const float* part = p.part + (slot_of(c, w + (int64_t)(src < 0 ? 0 : src) * NW) * p.GT + g) * D + lane * V;
#pragma unroll
        for (int i = 0; i < V; ++i) x[u][i] = 0.f;
        if (src < 0) continue;
        if (V == 4) {
          const float4 y = *reinterpret_cast<const float4*>(part);
          x[u][0] = y.x; x[u][1] = y.y; x[u][V - 2] = y.z; x[u][V - 1] = y.w;
        } else {
          const float2 y = *reinterpret_cast<const float2*>(part);
          x[u][0] = y.x; x[u][V - 1] = y.y;
        }
      }
      float mn = M;
#pragma unroll
      for (int u = 0; u < U; ++u) mn = fmaxf(mn, ml[u].x);
      const float ms = mn == -INFINITY ? 0.f : mn, a = exp2f(M - ms);
      L *= a;
#pragma unroll
      for (int i = 0; i < V; ++i) o[i] *= a;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float f = exp2f(ml[u].x - ms);
        L = fmaf(ml[u].y, f, L);
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = fmaf(x[u][i], f, o[i]);
      }
      M = mn;
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) s_o[warp][lane * V + i] = o[i];
  if (lane == 0) s_ml[warp] = make_float2(M, L);
  __syncthreads();
  if (tid < D) {  // (NW >= 4: there are that many threads)
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < NW; ++i) m = fmaxf(m, s_ml[i].x);
    const float ms = m == -INFINITY ? 0.f : m;
    float x = 0.f, l = 0.f;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      const float f = exp2f(s_ml[i].x - ms);
      l = fmaf(s_ml[i].y, f, l);
      x = fmaf(s_o[i][tid], f, x);
    }
    store_out(out + tid, x / l);
    if (tid == 0) p.ml[blockIdx.x] = make_float2(ms, 1.f / l);
  }
}

// weights_out[j] = weights[j] + sum_g exp2(s_gj - M_g) / L_g, 1024 keys of a (sequence, kv head)
// per block.  QUADS: a thread's four neighbouring keys share a page and 16-byte accesses (page size
// and strides multiples of four); otherwise each key is looked up.  Bound by the scores that it
// reads, which the kernel before it left in L2: 7.4 us for 32 ragged sequences up to 8192 keys (key by
// key two more).  A page that stands in the table twice would be read and written by several blocks
// at once: one of its entries updates it, the others are dropped and reported (0.7 us).
template <bool QUADS>
__global__ void __launch_bounds__(kUpd) paged_weights_kernel(const PDecP p) {
  const int64_t chunks = (p.c.cap + kUpd * 4 - 1) / (kUpd * 4), seg = div_fast(blockIdx.x, chunks);
  const int b = (int)div_fast(seg, p.c.Hkv), h = (int)(seg - (int64_t)b * p.c.Hkv);
  const int len = paged_len(p.c, b);
  const int j = ((int)(blockIdx.x - seg * chunks) * kUpd + (int)threadIdx.x) * 4;  // this thread's first key
  if (j >= len) {
    grid_wait();  // no block of a chain of programmatic launches ends before the kernel ahead has
    return;
  }
  constexpr int N = QUADS ? 1 : 4;
  int64_t to[N], pg[N];
  uint32_t t[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    to[i] = pg[i] = -1;
    t[i] = 0;
    if (j + i >= len) continue;
    t[i] = (uint32_t)(j + i) / p.c.page;
    pg[i] = paged_page(p.c, p.c.table, p.c.ts, b, t[i]);
    if (pg[i] >= 0) to[i] = pg[i] * p.c.wsp + h * p.c.wsh + ((uint32_t)(j + i) - t[i] * p.c.page);
  }
  float4 w = make_float4(0.f, 0.f, 0.f, 0.f);
  if (QUADS) {
    if (to[0] >= 0) w = *reinterpret_cast<const float4*>(p.c.w + to[0]);
  } else {
    if (to[0] >= 0) w.x = p.c.w[to[0]];
    if (to[QUADS ? 0 : 1] >= 0) w.y = p.c.w[to[QUADS ? 0 : 1]];
    if (to[QUADS ? 0 : 2] >= 0) w.z = p.c.w[to[QUADS ? 0 : 2]];
    if (to[QUADS ? 0 : 3] >= 0) w.w = p.c.w[to[QUADS ? 0 : 3]];
  }
  grid_wait();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (to[i] >= 0 && !is_place(p.places[pg[i]], b, t[i])) {
      to[i] = -1;
      atomicCAS(p.err, 0, kErrPageTwice);
    }
  }
  const float2* ml = p.ml + (int64_t)b * p.H + h * p.G;
  const float* sc = p.scores + (((int64_t)b * p.c.Hkv + h) * p.NG * p.cap_tiles + j / kTile) * p.SG * kTile + j % kTile;
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int grp = 0; grp < p.NG; ++grp, sc += p.cap_tiles * p.SG * kTile) {
    const int heads = min(p.GT, p.G - grp * p.GT);
#pragma unroll 4
    for (int g = 0; g < heads; ++g) {
      const float2 x = ml[grp * p.GT + g];
      const float4 s = *reinterpret_cast<const float4*>(sc + g * kTile);
      sum.x = fmaf(exp2f(s.x - x.x), x.y, sum.x);
      sum.y = fmaf(exp2f(s.y - x.x), x.y, sum.y);
      sum.z = fmaf(exp2f(s.z - x.x), x.y, sum.z);
      sum.w = fmaf(exp2f(s.w - x.x), x.y, sum.w);
    }
  }
  w.x += sum.x;
  w.y += sum.y;
  w.z += sum.z;
  w.w += sum.w;
  if (QUADS && j + 4 <= len) {
    if (to[0] >= 0) *reinterpret_cast<float4*>(p.w_out + to[0]) = w;
    return;
  }
  const float x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t at = QUADS ? (to[0] >= 0 && j + i < len ? to[0] + i : -1) : to[QUADS ? 0 : i];
    if (at >= 0) p.w_out[at] = x[i];
  }
}

struct PLayout {
  size_t part, part_ml, ml, scores, places, total;
  int GT, NG, W, unit;
  int64_t cap_tiles;
};

inline size_t al(size_t x) { return (x + 255) & ~size_t(255); }

int sm_count() {
  static int n[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (!n[dev]) {
    int v = 0;
    if (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
    n[dev] = v;
  }
  return n[dev];
}

PLayout layout(const sta_paged_cache* c, const sta_paged_decode_args* a) {
  PLayout L{};
  const int64_t G = a->n_heads / c->n_kv_heads;
  const bool f32 = c->dtype == STA_DTYPE_F32;
  // q heads that one pass over a kv head's keys serves: f32 by registers (padded to 1, 2, 4 or 8),
  // bf16 by the 8 columns of a tensor-core product, one or two of them (two where one is enough:
  // 126 us for 94 at 131072 keys of 8 kv heads)
  if (f32) L.GT = G > 4 ? 8 : (G > 2 ? 4 : (int)G);
  else L.GT = G > 8 ? 16 : 8;
  L.NG = (int)((G + L.GT - 1) / L.GT);
  L.cap_tiles = (c->table_width * c->page_size + kTile - 1) / kTile;
  L.unit = f32 ? kUnitF32 : kUnitBf16;
  const int64_t units = (c->table_width * c->page_size + (1 << L.unit) - 1) >> L.unit;
  const int64_t most = c->batch * c->n_kv_heads * L.NG * units;
  const int64_t w = (f32 ? (c->d == 128 ? 1 : 2) : paged_decode_bf16_shares(c->d, L.GT)) * (int64_t)sm_count();
  L.W = (int)(most < w ? most : w);
  size_t o = 0;
  auto take = [&](size_t bytes) {
    const size_t r = o;
    o += al(bytes);
    return r;
  };
  L.part = take((size_t)2 * L.W * L.GT * c->d * 4);
  L.part_ml = take((size_t)2 * L.W * L.GT * 8);
  L.ml = take((size_t)c->batch * a->n_heads * 8);
  L.scores = a->weights_out ? take((size_t)(c->batch * c->n_kv_heads * L.NG) * L.cap_tiles * (G < L.GT ? G : L.GT) * kTile * 4) : 0;
  L.places = a->weights_out ? take((size_t)c->n_pages * sizeof(int2)) : 0;
  L.total = o + 256;
  return L;
}

// Whether two arrays laid out like the weights, `delta` elements apart, have a place in common:
// delta = a * stride_p + b * stride_h + r with |a|, |b|, |r| less than the sizes.
bool share_places(const sta_paged_cache* c, int64_t delta) {
  const int64_t sp = c->weights_stride_p, sh = c->weights_stride_h;
  if (llabs(delta) > (c->n_pages - 1) * sp + (c->n_kv_heads - 1) * sh + c->page_size - 1) return false;
  for (int64_t b = 1 - c->n_kv_heads; b < c->n_kv_heads; ++b) {
    const int64_t rest = delta - b * sh, a0 = sp > 0 ? rest / sp : 0;  // (one of the three: |r| < stride_p)
    for (int64_t a = a0 - 1; a <= a0 + 1; ++a)
      if (llabs(a) < c->n_pages && llabs(rest - a * sp) < c->page_size) return true;
  }
  return false;
}

int check(const sta_paged_cache* c, const sta_paged_decode_args* a) {
  int rc = paged_check(c);
  if (rc != STA_OK) return rc;
  if (!a || (c->batch > 0 && (!a->q || !a->out)) || !a->inv_freq)
    return fail(STA_ERR_ARG, "sta_paged_decode: null pointer");
  if (reinterpret_cast<uintptr_t>(a->out) & 15u)
    return fail(STA_ERR_ARG, "sta_paged_decode: out must start on a 16-byte boundary");
  if (a->n_heads <= 0 || a->n_heads % c->n_kv_heads)
    return fail(STA_ERR_ARG, "sta_paged_decode: n_heads must be a multiple of n_kv_heads");
  if (a->chunk_size < 0 || (a->chunk_size > 0 && (a->local_window <= 0 || a->chunk_size <= a->local_window)))
    return fail(STA_ERR_ARG, "sta_paged_decode: bad chunk_size / local_window");
  if (a->chunk_size > 0 && (a->chunk_size - a->local_window) % kTile)
    return fail(STA_ERR_UNSUPPORTED, "sta_paged_decode: chunk_size - local_window must be a multiple of 64");
  if (a->chunk_size > 0 && a->pos_scale != 1.0)
    return fail(STA_ERR_ARG, "sta_paged_decode: Dual Chunk Attention positions take pos_scale 1");
  if (a->weights_out && !c->weights)
    return fail(STA_ERR_ARG, "sta_paged_decode: weights_out needs a cache with weights");
  if (a->weights_out && (rc = paged_check_weights_written(c)) != STA_OK) return rc;
  if (a->weights_out && a->weights_out != c->weights &&
      share_places(c, (int64_t)(reinterpret_cast<intptr_t>(a->weights_out) - reinterpret_cast<intptr_t>(c->weights)) / 4))
    return fail(STA_ERR_ARG, "sta_paged_decode: weights_out overlaps the weights without being them");
  if (a->weights_out && c->batch * c->n_kv_heads * (c->table_width * c->page_size / 1024 + 1) > ((int64_t)1 << 30))
    return fail(STA_ERR_UNSUPPORTED, "sta_paged_decode: too many slots for one update of the weights");
  if (c->batch * a->n_heads > ((int64_t)1 << 30))
    return fail(STA_ERR_UNSUPPORTED, "sta_paged_decode: too many heads");
  return STA_OK;
}

template <int D, int GT>
int launch_f32(const PDecP& p, cudaStream_t st) {
  constexpr int bytes = (int)sizeof(Smem<D, GT>);
  static bool ready[64];
  const cudaError_t e = allow_smem(paged_decode_f32_kernel<D, GT>, bytes, ready);
  if (e != cudaSuccess) return fail(STA_ERR_CUDA, cudaGetErrorString(e));
  const cudaError_t r = launch_behind(paged_decode_f32_kernel<D, GT>, dim3((unsigned)p.W), F32<D, GT>::THREADS, p, st, bytes);
  return r == cudaSuccess ? STA_OK : fail(STA_ERR_CUDA, cudaGetErrorString(r));
}

template <int D>
int launch_f32(const PDecP& p, cudaStream_t st) {
  if (p.GT == 1) return launch_f32<D, 1>(p, st);
  if (p.GT == 2) return launch_f32<D, 2>(p, st);
  if (p.GT == 4) return launch_f32<D, 4>(p, st);
  return launch_f32<D, 8>(p, st);
}

template <int D, typename TV>
cudaError_t launch_join(const PDecP& p, cudaStream_t st) {
  const dim3 grid((unsigned)((int64_t)p.c.B * p.H));
  // partials of a segment, where all sequences are alike: 16 warps join them for a few long
  // sequences (8 segments of 32768 keys: the join adds 3.5 us, 6.6 with 4 warps), 4 where there are
  // many segments and few partials of each (256 segments: 3.5 us, 12 with 16 warps)
  const int64_t each = p.W / ((int64_t)p.c.B * p.c.Hkv * p.NG);
  return each > 32 ? launch_behind(paged_join_kernel<D, TV, 16>, grid, 512, p, st)
                   : launch_behind(paged_join_kernel<D, TV, 4>, grid, 128, p, st);
}

template <typename TV>
cudaError_t launch_finish(const PDecP& p, int d, cudaStream_t st) {
  cudaError_t e = d == 128 ? launch_join<128, TV>(p, st) : launch_join<64, TV>(p, st);
  if (e == cudaSuccess && p.scores) {
    const int64_t chunks = (p.c.cap + kUpd * 4 - 1) / (kUpd * 4);
    const dim3 grid((unsigned)(p.c.B * p.c.Hkv * chunks));
    const bool quads = p.c.page % 4 == 0 && p.c.wsp % 4 == 0 && p.c.wsh % 4 == 0 &&
                       ((reinterpret_cast<uintptr_t>(p.c.w) | reinterpret_cast<uintptr_t>(p.w_out)) & 15) == 0;
    e = quads ? launch_behind(paged_weights_kernel<true>, grid, kUpd, p, st)
              : launch_behind(paged_weights_kernel<false>, grid, kUpd, p, st);
  }
  return e;
}

}  // namespace

size_t paged_decode_workspace_bytes(const sta_paged_cache* c, const sta_paged_decode_args* a) {
  if (check(c, a) != STA_OK) return 0;
  return layout(c, a).total;
}

int paged_decode(const sta_paged_cache* c, const sta_paged_decode_args* a, void* ws, size_t ws_len,
                 cudaStream_t st) {
  int rc = check(c, a);
  if (rc != STA_OK) return rc;
  if (c->batch == 0) return STA_OK;
  const PLayout L = layout(c, a);
  if (!ws || ws_len < L.total) return fail(STA_ERR_WORKSPACE, "sta_paged_decode: workspace too small");
  const bool f32 = c->dtype == STA_DTYPE_F32;
  uint8_t* w = static_cast<uint8_t*>(ws);
  w += (256 - reinterpret_cast<uintptr_t>(w) % 256) % 256;
  PDecP p;
  p.c = paged_view(c);
  p.q = a->q; p.qsb = a->q_stride_b; p.qsh = a->q_stride_h;
  p.q_words = (reinterpret_cast<uintptr_t>(a->q) & 3) == 0 && a->q_stride_b % 2 == 0 && a->q_stride_h % 2 == 0;
  p.out = a->out;
  p.H = (int)a->n_heads;
  p.G = (int)(a->n_heads / c->n_kv_heads);
  p.NG = L.NG;
  p.GT = L.GT;
  p.SG = p.G < L.GT ? p.G : L.GT;
  p.unit = L.unit;
  p.W = L.W;
  p.min_log = f32 ? 0 : 1;
  p.sms = sm_count();
  p.merge = p.W > 16 * c->batch * c->n_kv_heads * L.NG;
  p.k16 = 16 * p.c.ksn;
  p.v16 = 16 * p.c.vsn;
  p.inv_freq = a->inv_freq;
  p.pos_scale = a->pos_scale;
  p.qscale = (float)((double)a->sm_scale * a->rope_scale * a->rope_scale * 1.4426950408889634);
  p.L = a->chunk_size > 0 ? a->chunk_size - a->local_window : 0;
  p.s = a->chunk_size;
  p.part = reinterpret_cast<float*>(w + L.part);
  p.part_ml = reinterpret_cast<float2*>(w + L.part_ml);
  p.ml = reinterpret_cast<float2*>(w + L.ml);
  p.scores = a->weights_out ? reinterpret_cast<float*>(w + L.scores) : nullptr;
  p.places = a->weights_out ? reinterpret_cast<int2*>(w + L.places) : nullptr;
  p.cap_tiles = L.cap_tiles;
  p.w_out = a->weights_out;
  p.err = page_error_word();
  if (!p.err) return fail(STA_ERR_CUDA, "sta_paged_decode: no device");
  if (f32) rc = c->d == 128 ? launch_f32<128>(p, st) : launch_f32<64>(p, st);
  else rc = launch_paged_decode_bf16(p, c->d, st);
  if (rc != STA_OK) return rc;
  const cudaError_t e = f32 ? launch_finish<float>(p, c->d, st) : launch_finish<__nv_bfloat16>(p, c->d, st);
  return e == cudaSuccess ? STA_OK : fail(STA_ERR_CUDA, cudaGetErrorString(e));
}

}  // namespace sta
