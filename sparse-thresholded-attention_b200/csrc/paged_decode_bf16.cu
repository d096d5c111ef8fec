// Decode over a paged bf16 cache on the tensor cores (schedule and rotation: paged_decode.cuh).
//
// One new token has few q heads per kv head, so the products are (16 keys) x (d) x (8 or 16
// heads): warp-level m16n8k16 with the keys as rows wastes nothing up to 8 heads, where a
// 128-row tcgen05 tile would spend 15 of 16 rows on padding.  Per 16 keys a warp forms
//   S^T (16 keys x heads) = K (rotated) . Q^T     A = K rows, B = the tile's rotated queries
//   O^T (d x heads)      += V^T . P^T             A = V^T, B = P transposed in registers (movmatrix)
// Rotated keys, queries and probabilities are fp32 values carried as hi + lo bf16 pieces (four
// products for S, two for P.V: V is exact), which leaves errors of 2^-15 (keys, whose hi piece is
// cut instead of rounded) and 2^-16; running max, sums and accumulators are fp32.  For the output
// that is far below its own rounding to bf16 (2^-8).  The fp32 weights show it: a weight comes from a
// score that is off by up to 3 * 2^-16 |q| |k| scale (4096 keys, d = 128, scores over a range of 8:
// 4e-6 in norm where the f32 kernel is at 1.6e-7; over 25: 1.3e-5 and 5.4e-7).
//
// Every warp walks a share of its own and needs no barrier: its rows come by cp.async (16-byte
// chunks, swizzled by row) into a ring of its own, two units of K and one of V, so that some 7 KB
// per warp (d = 128) are in flight all the time; 12 warps per SM hide each other's latencies.  The
// cos / sin of the 64 key offsets of a tile lie in shared memory in the order the lanes read them,
// the queries of a tile in registers as B fragments.
//
// Measured with 4 q heads per kv head, d = 128, the join included: 131072 keys of 8 kv heads 98 us
// (537 MB of cache, 5.5 TB/s; 92 in short bursts, in a row the card is at its power limit and the SM
// clock falls from 1965 to 1690 MHz), 65536 keys 54, 32768 keys 35, 8192 keys 19 us.  Each further
// byte comes at 7 TB/s (6.0 beyond 65536 keys in a row); 13 to 17 us are fixed: the start (lengths,
// page table, first rows: a chain of loads), uneven ends and the join.  An SM issues in 53 % of its
// cycles and the tensor pipe is active in 25 %: what the loop waits for is its own arithmetic.
#include "mma_frag.cuh"
#include "paged_decode.cuh"

namespace sta {

namespace {

// tiles after which the running angle of the query is formed anew: it drifts by 2^-24 per tile
constexpr int kRenew = 32;

template <int D, int NT>
struct Cfg {
  // warps of a CTA and CTAs of an SM by registers: 168 a thread for <128, 1> and <64, 2>, 255 for
  // <128, 2>, 128 for <64, 1>
  static constexpr int NW = D == 128 ? (NT == 1 ? 12 : 8) : (NT == 1 ? 8 : 12);
  static constexpr int CTAS = D == 64 && NT == 1 ? 2 : 1;
};

template <int D, int NT>
struct SmemB {
  static constexpr int NW = Cfg<D, NT>::NW;
  uint4 k[NW][2][16 * D / 8];             // K rows of two units
  uint4 v[NW][16 * D / 8];                // V rows of one
  float4 rot[4][D / 32][4][32];           // (cos, cos, sin, sin) of two dims: unit, k step, register, lane
  float4 ang[NW][D / 4];                  // (cos, cos, sin, sin) of the query's angle, two dims, times the scale
  uint4 q[NW][NT][D / 32][32];            // a lane's raw queries of a k step: dims 0, 8, d/2, d/2 + 8 on, two each
  float2 turns[16][D / 2];                // cos / sin of turns by 0 .. 7 and by 0, 8 .. 56 positions
  float inv_freq[D / 2];
  float2 end_ml[NW][8 * NT];              // the partials that the shares end with: max and sum,
  int4 end[NW];                           // sequence (-1: none), kv head, group, first unit included
  int4 seg[NW][4];                        // segments entered by the loads: sequence, kv head, group, length
};

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// C = A (16x16 bf16, row) * B (16x8 bf16, col)
__device__ __forceinline__ void mma_bf16_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                               uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

// two fp32 values in a register pair, and the packed arithmetic on them
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pair(float a, float b) {
  f32x2 d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ void unpair(f32x2 d, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(d));
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ f32x2 widen(uint32_t x) {  // two bf16
  return pair(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
}
// hi: the upper halves of the fp32 words (truncation: one byte permute), lo: the rest, rounded
__device__ __forceinline__ void split_cut(f32x2 x, f32x2 minus_one, uint32_t& hi, uint32_t& lo) {
  float a, b;
  unpair(x, a, b);
  const uint32_t ua = __float_as_uint(a), ub = __float_as_uint(b);
  hi = __byte_perm(ua, ub, 0x7632);
  const f32x2 rest = fma2(pair(__uint_as_float(ua & 0xffff0000u), __uint_as_float(ub & 0xffff0000u)),
                          minus_one, x);
  unpair(rest, a, b);
  lo = pack_bf16(a, b);
}

// both pieces rounded
__device__ __forceinline__ void split_round(f32x2 x, f32x2 minus_one, uint32_t& hi, uint32_t& lo) {
  float a, b;
  unpair(x, a, b);
  hi = pack_bf16(a, b);
  unpair(fma2(widen(hi), minus_one, x), a, b);
  lo = pack_bf16(a, b);
}

// Where the 16 keys of a unit lie: entry of the page table and slot in that page (of this lane's
// row where the page size is no multiple of 16).
struct Rows {
  int32_t entry;
  uint32_t slot, t;
  bool fresh;  // another page than the unit before
};

// How a unit's 16 rows lie: anywhere; in one page (its size is a multiple of 16); in one page,
// one behind the other.
enum RowMode { kAnyRows, kPageRows, kDenseRows };

template <int D, int NT, RowMode MODE>
__global__ void __launch_bounds__(Cfg<D, NT>::NW * 32, Cfg<D, NT>::CTAS)
    paged_decode_bf16_kernel(const PDecP p) {
  using S = SmemB<D, NT>;
  constexpr int HALF = D / 2, CH = D / 8, NW = Cfg<D, NT>::NW, NH = D / 32, MT = D / 16, GT = 8 * NT;
  constexpr int FPL = D / 64;      // frequencies of a lane in the angles
  constexpr int RPI = 32 / CH;     // rows that one copy of the warp covers
  constexpr bool P16 = MODE != kAnyRows;
  extern __shared__ __align__(128) unsigned char smem_raw[];
  S& sm = *reinterpret_cast<S*>(smem_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int fr = lane >> 2, fc = lane & 3;

  grid_wait();
  grid_dependents();
  // The start is a chain of loads (lengths, page table, rows) that nothing may stand ahead of: what
  // can be computed meanwhile comes once the rows have been asked for.
  static_assert(NW * 32 % HALF == 0, "a thread's turns share one frequency");
  const float my_freq = __ldg(p.inv_freq + threadIdx.x % HALF);
  int64_t me;  // this warp's share: a CTA has neighbouring ones, all CTAs as many
  const Share share = find_share(p, first_len(p.c), me);
  const int count = share.count;
  Place nx = share.at;              // the unit whose K rows are loaded next
  Rows rows{-1, 0, 0, true};
  int segs = 0, k_it = 0;           // segments entered, units whose K rows are loaded
  int n = nx.n;                     // the unit in hand, of its segment

  // ---- page lookup of unit nx
  auto lookup = [&](bool first) {
    if (first || nx.n == 0) {
      if (lane == 0) sm.seg[warp][segs & 3] = make_int4(nx.b, nx.h, nx.grp, nx.len);
      ++segs;
    }
    if (P16) {
      rows.fresh = true;
      if (first || nx.n == 0) {
        const uint32_t j = (uint32_t)nx.n * 16;
        rows.t = j / p.c.page;
        rows.slot = j - rows.t * p.c.page;
      } else {
        rows.slot += 16;
        rows.fresh = rows.slot == p.c.page;
        if (rows.fresh) {
          rows.slot = 0;
          ++rows.t;
        }
      }
      if (rows.fresh) rows.entry = __ldg(p.c.table + nx.b * p.c.ts + rows.t);
    } else {
      const uint32_t j = (uint32_t)nx.n * 16 + (lane & 15);
      const uint32_t t = j / p.c.page;
      rows.slot = j - t * p.c.page;
      rows.entry = j < (uint32_t)nx.len ? __ldg(p.c.table + nx.b * p.c.ts + t) : -1;
    }
  };
  // ---- copies.  Rows without data are zero; of a bad page, K is NaN.
  const int lch = lane % CH, lrow = lane / CH;
  const uint32_t ring_k = smem_u32(sm.k[warp][0]), ring_v = smem_u32(sm.v[warp]);
  uint32_t dst0[8 / RPI];  // this lane's chunk of the first 8 rows, chunks swizzled by row
#pragma unroll
  for (int i = 0; i < 8 / RPI; ++i) {
    const int row = lrow + RPI * i;
    dst0[i] = (uint32_t)(row * (D * 2) + ((lch ^ row) << 4));
  }
  const char *kbase = p.c.k, *vbase = p.c.v, *vnext = p.c.v;  // P16: this lane's first row
  int64_t koff = 0, vonext = 0;            // otherwise: of row (lane & 15); -1: no row, -2: bad page
  int left = 0, vleft = 0;                 // keys of the unit from its first on; 0: a bad page
  auto copy = [&](uint32_t ring, const char* base, const char* pool, int64_t off, int64_t stride, int rest) {
    uint32_t to[8 / RPI];
#pragma unroll
    for (int i = 0; i < 8 / RPI; ++i) to[i] = ring + dst0[i];
    if (P16 && rest >= 16) {
#pragma unroll
      for (int i = 0; i < 16 / RPI; ++i)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n"
                     ::"r"(to[i % (8 / RPI)] + i / (8 / RPI) * (8 * D * 2)),
                       "l"(base + i * RPI * (MODE == kDenseRows ? D * 2 : stride)) : "memory");
    } else {
#pragma unroll
      for (int i = 0; i < 16 / RPI; ++i) {
        const uint32_t dst = to[i % (8 / RPI)] + i / (8 / RPI) * (8 * D * 2);
        const char* src = base + i * RPI * stride;
        bool in = lrow + RPI * i < rest;
        if (!P16) {
          const int64_t o = __shfl_sync(0xffffffffu, off, lrow + RPI * i);
          in = o >= 0;
          src = pool + (o + lch * 16);
        }
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n"
                     ::"r"(dst), "l"(in ? src : pool), "r"(in ? 16 : 0) : "memory");
      }
    }
  };
  auto load_k = [&]() {  // unit nx; its V rows follow one unit later
    if (k_it < count) {
      bool bad = false;
      if (P16) {
        if (rows.fresh) {
          const bool ok = rows.entry >= 0 && rows.entry < p.c.n_pages;
          const int64_t pg = ok ? rows.entry : 0;
          kbase = p.c.k + (lrow + rows.slot) * p.c.ksn + lch * 16 + nx.h * p.c.ksh + pg * p.c.ksp;
          vbase = p.c.v + (lrow + rows.slot) * p.c.vsn + lch * 16 + nx.h * p.c.vsh + pg * p.c.vsp;
          left = ok ? 16 : 0;
        } else {
          kbase += p.k16;
          vbase += p.v16;
        }
        bad = left == 0;
        vnext = vbase;
        vleft = bad ? 0 : nx.len - nx.n * 16;
        copy(ring_k + (k_it & 1) * (D * 32), kbase, p.c.k, 0, p.c.ksn, vleft);
      } else {
        const bool in = nx.n * 16 + (lane & 15) < nx.len;
        const bool ok = rows.entry >= 0 && rows.entry < p.c.n_pages;
        koff = in && ok ? rows.entry * p.c.ksp + nx.h * p.c.ksh + rows.slot * p.c.ksn : -1;
        vonext = in && ok ? rows.entry * p.c.vsp + nx.h * p.c.vsh + rows.slot * p.c.vsn : -1;
        bad = __any_sync(0xffffffffu, in && !ok);
        copy(ring_k + (k_it & 1) * (D * 32), p.c.k, p.c.k, koff, 0, 16);
      }
      if (bad) {  // the whole unit: every output of the sequence is NaN
        // a lane waits for its own copies only: without the barrier another lane's zeros could still
        // land on the NaN stored here
        asm volatile("cp.async.wait_all;\n" ::: "memory");
        __syncwarp();
        if (lane == 0) atomicCAS(p.err, 0, kErrPageDecode);
        for (int i = lane; i < 16 * CH; i += 32)
          sm.k[warp][k_it & 1][i] = make_uint4(0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u);
      }
      if (k_it + 1 < count) {
        step(p, nx);
        lookup(false);
      }
    }
    asm volatile("cp.async.commit_group;\n" ::: "memory");
    ++k_it;
  };
  auto load_v = [&](int it, const char* base, int64_t off, int rest) {
    if (it < count) copy(ring_v, base, p.c.v, off, p.c.vsn, rest);
    asm volatile("cp.async.commit_group;\n" ::: "memory");
  };

  // ---- a segment's raw queries, as the lanes rotate them: asked for, then stored
  uint32_t raw[NT][NH][4];
  auto ask_queries = [&](const int4& at) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int g = at.z * GT + nt * 8 + fr;
      const uint16_t* src = static_cast<const uint16_t*>(p.q) + at.x * p.qsb + (at.y * p.G + g) * p.qsh + fc * 2;
#pragma unroll
      for (int ks = 0; ks < NH; ++ks)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int d = ks * 16 + (i & 1) * 8 + (i >> 1) * HALF;
          raw[nt][ks][i] = 0u;
          if (g < p.G)
            raw[nt][ks][i] = p.q_words ? *reinterpret_cast<const uint32_t*>(src + d)
                                       : src[d] | (uint32_t)src[d + 1] << 16;
        }
    }
  };
  auto keep_queries = [&]() {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int ks = 0; ks < NH; ++ks)
        sm.q[warp][nt][ks][lane] = make_uint4(raw[nt][ks][0], raw[nt][ks][1], raw[nt][ks][2], raw[nt][ks][3]);
  };
  const char* vcur = p.c.v;   // the V rows that follow next
  int64_t vocur = 0;
  int vlcur = 0;
  if (count > 0) {
    lookup(true);
    ask_queries(make_int4(share.at.b, share.at.h, share.at.grp, 0));
    load_k();
    vcur = vnext; vocur = vonext; vlcur = vleft;
    load_v(0, vcur, vocur, vlcur);
    load_k();
    vcur = vnext; vocur = vonext; vlcur = vleft;
    keep_queries();
  }
  // ---- cos / sin of the key offsets t * pos_scale, t = 0 .. 63, by all warps: t = 8 i + j as the
  // product of the turns by 8 i and by j (16 sincos per frequency instead of 64)
  for (int i = threadIdx.x; i < 16 * HALF; i += NW * 32) {
    const int f = i % HALF, t = i / HALF;
    turn((double)(t < 8 ? t : (t - 8) * 8) * p.pos_scale, my_freq, sm.turns[t][f].x, sm.turns[t][f].y);
  }
  if (threadIdx.x < HALF) sm.inv_freq[threadIdx.x] = my_freq;
  __syncthreads();
  for (int i = threadIdx.x; i < 4 * NH * 4 * 32; i += NW * 32) {
    const int l = i & 31, r = (i >> 5) & 3, ks = (i >> 7) % NH, u = i / (128 * NH);
    const int f = ks * 16 + (l & 3) * 2 + (r >> 1) * 8;
    const float4 a = *reinterpret_cast<const float4*>(&sm.turns[l >> 2][f]);
    const float4 b = *reinterpret_cast<const float4*>(&sm.turns[8 + 2 * u + (r & 1)][f]);
    sm.rot[u][ks][r][l] = make_float4(a.x * b.x - a.y * b.y, a.z * b.z - a.w * b.w,
                                      a.x * b.y + a.y * b.x, a.z * b.w + a.w * b.z);
  }
  if (lane == 0) sm.end[warp].x = -1;
  __syncthreads();

  // ---- the query's angle at a tile, this lane's frequencies; it moves by a constant from tile to
  // tile of a segment (of a chunk)
  float ac[FPL], as[FPL], dc[FPL], ds[FPL];
#pragma unroll
  for (int e = 0; e < FPL; ++e) {
    turn(-(double)kTile * p.pos_scale, sm.inv_freq[lane * FPL + e], dc[e], ds[e]);
    ac[e] = as[e] = 0.f;
  }
  uint32_t qb[NT][2 * NH][4];      // B fragments of a k step: hi b0, hi b1, lo b0, lo b1
  const f32x2 minus_one = pair(-1.f, -1.f);

  float acc[NT][MT][4];
  float mx[NT][2], mref[NT][2], sum[NT][2];  // of heads 8 nt + 2 fc + {0, 1}; sums of this lane's keys
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int x = 0; x < 4; ++x) acc[nt][mt][x] = 0.f;
    mx[nt][0] = mx[nt][1] = -INFINITY;
    mref[nt][0] = mref[nt][1] = sum[nt][0] = sum[nt][1] = 0.f;
  }
  // ldmatrix lane addresses of a unit's first chunks; chunk c lies c * 16 bytes on, by exclusive or
  const uint32_t k_lane = ring_k + (lane & 15) * (D * 2) + (((lane >> 4) ^ (lane & 7)) << 4);
  const uint32_t v_lane = ring_v + ((lane & 7) + ((lane >> 4) << 3)) * (D * 2) +
                          ((((lane >> 3) & 1) ^ (lane & 7)) << 4);

  int seg = -1, len = 0;           // the segment in hand and its length
  bool fresh_seg = true;
#pragma unroll 1
  for (int it = 0; it < count; ++it) {
    if (fresh_seg) {
      ++seg;
      len = sm.seg[warp][seg & 3].w;
    }
    // ---- queries, once per tile
    if (it == 0 || (n & 3) == 0) {
      const int4 at = sm.seg[warp][seg & 3];
      const int tile = n >> 2;
      if (it == 0 || tile % kRenew == 0 || (p.L > 0 && tile * kTile % p.L == 0)) {
        const double x = query_offset(p, len, tile);
#pragma unroll
        for (int e = 0; e < FPL; ++e) turn(x, sm.inv_freq[lane * FPL + e], ac[e], as[e]);
      } else {
#pragma unroll
        for (int e = 0; e < FPL; ++e) {
          const float c = ac[e] * dc[e] - as[e] * ds[e];
          as[e] = as[e] * dc[e] + ac[e] * ds[e];
          ac[e] = c;
        }
      }
      if (fresh_seg && it > 0) {
        ask_queries(at);
        keep_queries();
      }
#pragma unroll
      for (int e = 0; e < FPL; ++e) {
        float* x = reinterpret_cast<float*>(&sm.ang[warp][(lane * FPL + e) / 2]) + ((lane * FPL + e) & 1);
        x[0] = ac[e] * p.qscale;
        x[2] = as[e] * p.qscale;
      }
      __syncwarp();
#pragma unroll
      for (int ks = 0; ks < NH; ++ks)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const uint4 raw = sm.q[warp][nt][ks][lane];
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            const float4 cs = sm.ang[warp][ks * 8 + b * 4 + fc];
            const f32x2 c = pair(cs.x, cs.y), s = pair(cs.z, cs.w);
            const f32x2 x1 = widen(b == 0 ? raw.x : raw.y), x2 = widen(b == 0 ? raw.z : raw.w);
            split_round(fma2(mul2(x2, s), minus_one, mul2(x1, c)), minus_one, qb[nt][ks][b], qb[nt][ks][2 + b]);
            split_round(fma2(x1, s, mul2(x2, c)), minus_one, qb[nt][ks + NH][b], qb[nt][ks + NH][2 + b]);
          }
        }
      __syncwarp();
    }
    // ---- S^T
    asm volatile("cp.async.wait_group 2;\n" ::: "memory");
    __syncwarp();
    float sc[NT][2][4];
    const float4* rot = &sm.rot[n & 3][0][0][lane];
    const uint32_t kb = k_lane + (it & 1) * (D * 32);
#pragma unroll
    for (int ks = 0; ks < NH; ++ks) {
      uint32_t a[4], b[4], ah[4], al[4], bh[4], bl[4];
      ldsm_x4(kb ^ (ks * 32), a[0], a[1], a[2], a[3]);
      ldsm_x4(kb ^ (ks * 32 + D), b[0], b[1], b[2], b[3]);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const f32x2 x1 = widen(a[r]), x2 = widen(b[r]);
        const float4 cs = rot[(ks * 4 + r) * 32];
        const f32x2 c = pair(cs.x, cs.y), s = pair(cs.z, cs.w);
        split_cut(fma2(mul2(x2, s), minus_one, mul2(x1, c)), minus_one, ah[r], al[r]);
        split_cut(fma2(x1, s, mul2(x2, c)), minus_one, bh[r], bl[r]);
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const uint32_t(&qa)[4] = qb[nt][ks];
        const uint32_t(&qc)[4] = qb[nt][ks + NH];
        if (ks == 0) {
          mma_bf16_first(sc[nt][0], ah, qa[0], qa[1]);
          mma_bf16_first(sc[nt][1], ah, qa[2], qa[3]);
        } else {
          mma_bf16(sc[nt][0], ah, qa[0], qa[1]);
          mma_bf16(sc[nt][1], ah, qa[2], qa[3]);
        }
        mma_bf16(sc[nt][0], al, qa[0], qa[1]);
        mma_bf16(sc[nt][1], al, qa[2], qa[3]);
        mma_bf16(sc[nt][0], bh, qc[0], qc[1]);
        mma_bf16(sc[nt][1], bh, qc[2], qc[3]);
        mma_bf16(sc[nt][0], bl, qc[0], qc[1]);
        mma_bf16(sc[nt][1], bl, qc[2], qc[3]);
      }
    }
    // ---- the K rows of the unit after the next, into the place just read
    __syncwarp();
    load_k();
    // ---- online softmax over the 16 keys
    uint32_t ph[NT][2], pl[NT][2];
    bool grow = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int x = 0; x < 4; ++x)
        sc[nt][0][x] += sc[nt][1][x];
    if (n * 16 + 16 > len) {
      const int rest = len - n * 16 - fr;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int x = 0; x < 4; ++x)
          if ((x < 2 ? 0 : 8) >= rest) sc[nt][0][x] = -INFINITY;
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) grow |= fmaxf(sc[nt][0][c], sc[nt][0][c + 2]) > mx[nt][c];
    if (__any_sync(0xffffffffu, grow)) {  // rare after the first units of a segment
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float m = fmaxf(sc[nt][0][c], sc[nt][0][c + 2]);
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
          m = fmaxf(mx[nt][c], m);
          const float to = m == -INFINITY ? 0.f : m, f = ex2(mx[nt][c] - to);
          mx[nt][c] = m;
          mref[nt][c] = to;
          sum[nt][c] *= f;
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            acc[nt][mt][c] *= f;
            acc[nt][mt][c + 2] *= f;
          }
        }
    }
    if (p.scores) {
      const int4 at = sm.seg[warp][seg & 3];
      float* out = p.scores + ((((int64_t)at.x * p.c.Hkv + at.y) * p.NG + at.z) * p.cap_tiles + (n >> 2)) *
                                  p.SG * kTile + (n & 3) * 16 + fr;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int g = nt * 8 + fc * 2 + (x & 1);
          if (at.z * GT + g < p.G) out[g * kTile + (x >> 1) * 8] = sc[nt][0][x];
        }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float e[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        e[x] = ex2(sc[nt][0][x] - mref[nt][x & 1]);
        sum[nt][x & 1] += e[x];
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        uint32_t hi, lo;
        split_round(pair(e[2 * r], e[2 * r + 1]), minus_one, hi, lo);
        ph[nt][r] = transpose8x8(hi);
        pl[nt][r] = transpose8x8(lo);
      }
    }
    // ---- O^T += V^T . P^T
    asm volatile("cp.async.wait_group 1;\n" ::: "memory");
    __syncwarp();
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      uint32_t a[4];
      ldsm_x4_t(v_lane ^ (mt * 32), a[0], a[1], a[2], a[3]);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        mma_bf16(acc[nt][mt], a, ph[nt][0], ph[nt][1]);
        mma_bf16(acc[nt][mt], a, pl[nt][0], pl[nt][1]);
      }
    }
    __syncwarp();
    load_v(it + 1, vcur, vocur, vlcur);
    vcur = vnext;
    vocur = vonext;
    vlcur = vleft;
    fresh_seg = n * 16 + 16 >= len;
    if (fresh_seg || it + 1 == count) {
      // the share's part of this segment: the result itself, or a partial
      const int4 at = sm.seg[warp][seg & 3];
      const bool started = n <= it;  // the segment's first unit lies in this share
      const bool whole = fresh_seg && started;
      // what is left open at the share's end is joined with the neighbours' below; it waits in the
      // ring, which is free by then
      const bool last = share.merge && it + 1 == count;
      const int64_t slot = 2 * me + (started ? 1 : 0);
      float* part = last ? reinterpret_cast<float*>(sm.k[warp][0]) : p.part + slot * GT * D;
      if (last && !whole && lane == 0) sm.end[warp] = make_int4(at.x, at.y, at.z, started ? 1 : 0);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float l = sum[nt][c];
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
          const int g = nt * 8 + fc * 2 + c;
          if (at.z * GT + g < p.G) {
            const int64_t head = (int64_t)at.x * p.H + at.y * p.G + at.z * GT + g;
            if (whole) {
              __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.out) + head * D + fr;
              const float f = 1.f / l;
#pragma unroll
              for (int mt = 0; mt < MT; ++mt) {
                out[mt * 16] = __float2bfloat16_rn(acc[nt][mt][c] * f);
                out[mt * 16 + 8] = __float2bfloat16_rn(acc[nt][mt][c + 2] * f);
              }
              if (fr == 0) p.ml[head] = make_float2(mref[nt][c], f);
            } else {
              float* to = part + g * D + fr;
#pragma unroll
              for (int mt = 0; mt < MT; ++mt) {
                to[mt * 16] = acc[nt][mt][c];
                to[mt * 16 + 8] = acc[nt][mt][c + 2];
              }
              if (fr == 0) {
                if (last) sm.end_ml[warp][g] = make_float2(mx[nt][c], l);
                else p.part_ml[slot * GT + g] = make_float2(mx[nt][c], l);
              }
            }
          }
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) acc[nt][mt][c] = acc[nt][mt][c + 2] = 0.f;
          mx[nt][c] = -INFINITY;
          mref[nt][c] = sum[nt][c] = 0.f;
        }
    }
    n = fresh_seg ? 0 : n + 1;
  }

  // ---- the open ends of neighbouring shares that lie in one segment become one partial, that of
  // the first; the others' are marked as empty
  if (!share.merge) return;
  __syncthreads();
#pragma unroll 1
  for (int w0 = 0; w0 < NW;) {
    const int4 at = sm.end[w0];
    int w1 = w0 + 1;
    if (at.x >= 0) {
      while (w1 < NW && sm.end[w1].x == at.x && sm.end[w1].y == at.y && sm.end[w1].z == at.z) ++w1;
      const int64_t slot = 2 * (me - warp + w0) + at.w;
      const int heads = min(GT, p.G - at.z * GT);
      for (int i = threadIdx.x; i < heads * D; i += NW * 32) {
        const int g = i / D;
        float M = -INFINITY, L = 0.f, o = 0.f;
        for (int w = w0; w < w1; ++w) M = fmaxf(M, sm.end_ml[w][g].x);
        const float ms = M == -INFINITY ? 0.f : M;
        for (int w = w0; w < w1; ++w) {
          const float2 ml = sm.end_ml[w][g];
          const float f = ex2(ml.x - ms);
          L = fmaf(ml.y, f, L);
          o = fmaf(reinterpret_cast<const float*>(sm.k[w][0])[i], f, o);
        }
        p.part[slot * GT * D + i] = o;
        if (i % D == 0) p.part_ml[slot * GT + g] = make_float2(M, L);
      }
      for (int i = threadIdx.x; i < (w1 - w0 - 1) * GT; i += NW * 32)
        p.part_ml[2 * (me - warp + w0 + 1) * GT + i / GT * 2 * GT + i % GT] = make_float2(-INFINITY, 0.f);
    }
    w0 = w1;
  }
}

template <int D, int NT, RowMode MODE>
int launch(const PDecP& p, cudaStream_t st) {
  constexpr int bytes = (int)sizeof(SmemB<D, NT>), NW = Cfg<D, NT>::NW;
  static bool ready[64];
  const cudaError_t e = allow_smem(paged_decode_bf16_kernel<D, NT, MODE>, bytes, ready);
  if (e != cudaSuccess) return fail(STA_ERR_CUDA, cudaGetErrorString(e));
  // shares go to the CTAs in turn, so few shares spread over the SMs
  const int grid = p.W < p.sms * Cfg<D, NT>::CTAS ? p.W : p.sms * Cfg<D, NT>::CTAS;
  // a CTA joins its shares' open ends where it has more than three shares, so that it has some to
  // join, and segments are cut into many (16 on average): then the join gets shorter by more than
  // the barrier at the end costs (one sequence of 32768 keys, 8 kv heads: 35.0 us, without 36.3;
  // 32 ragged sequences up to 8192, 7 shares each: 91.6 us with, 89.6 without)
  PDecP q = p;
  q.merge = p.merge ? 3 * grid + 1 : 1 << 30;
  const cudaError_t r = launch_behind(paged_decode_bf16_kernel<D, NT, MODE>, dim3((unsigned)grid), NW * 32, q, st, bytes);
  return r == cudaSuccess ? STA_OK : fail(STA_ERR_CUDA, cudaGetErrorString(r));
}

template <int D, int NT>
int launch(const PDecP& p, cudaStream_t st) {
  // rows found one by one cost more (32768 keys of 8 kv heads, d = 128: 38.7 us, in one page of dense
  // rows 35.1); the stride of dense rows folds into the copies' addresses (as a variable 36.3 us)
  if (p.c.page % 16 != 0) return launch<D, NT, kAnyRows>(p, st);
  if (p.c.ksn == 2 * D && p.c.vsn == 2 * D) return launch<D, NT, kDenseRows>(p, st);
  return launch<D, NT, kPageRows>(p, st);
}

}  // namespace

int paged_decode_bf16_shares(int d, int GT) {
  if (d == 128) return GT == 8 ? Cfg<128, 1>::NW * Cfg<128, 1>::CTAS : Cfg<128, 2>::NW * Cfg<128, 2>::CTAS;
  return GT == 8 ? Cfg<64, 1>::NW * Cfg<64, 1>::CTAS : Cfg<64, 2>::NW * Cfg<64, 2>::CTAS;
}

int launch_paged_decode_bf16(const PDecP& p, int d, cudaStream_t st) {
  if (d == 128) return p.GT == 8 ? launch<128, 1>(p, st) : launch<128, 2>(p, st);
  return p.GT == 8 ? launch<64, 1>(p, st) : launch<64, 2>(p, st);
}

}  // namespace sta
