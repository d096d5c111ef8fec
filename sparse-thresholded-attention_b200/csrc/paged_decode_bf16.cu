// Decode over a paged bf16 cache on the tensor cores (schedule and rotation: paged_decode.cuh).
//
// One new token has few q heads per kv head, so the products are (64 keys) x (d) x (8 or 16
// heads): warp-level m16n8k16 with the keys as rows wastes nothing up to 8 heads, where a
// 128-row tcgen05 tile would spend 15 of 16 rows on padding.  A warp owns 16 keys of each tile:
//   S^T (16 keys x heads) = K (rotated) . Q^T     A = K rows (ldmatrix), B = the tile's queries
//   O^T (d x heads)      += V^T . P^T             A = V^T (ldmatrix.trans), B = P transposed in
//                                                 registers (movmatrix)
// Rotated keys, queries and probabilities are fp32 values carried as hi + lo bf16 pieces (four
// products for S, two for P.V: V is exact), which leaves errors of 2^-15 (keys, whose hi piece is
// cut instead of rounded) and 2^-16, far below the output's own rounding; running max, sums and
// accumulators are fp32.
//
// The rows of two to four tiles are in flight per CTA (cp.async, 16-byte chunks swizzled by row); a
// thread's cos / sin of the tile-local key offsets stay in registers for the whole call.
#include "mma_frag.cuh"
#include "paged_decode.cuh"

namespace sta {

namespace {

// A tile as its producer describes it.
struct TileInfo {
  uint32_t b;  // sequence, and kFull / kFresh / kStart
  int hg, n, len;
};
constexpr uint32_t kFull = 1u << 31;   // 64 keys, every page inside the pool
constexpr uint32_t kFresh = 1u << 30;  // the query's angle does not follow from the tile before
constexpr uint32_t kStart = 1u << 29;  // another segment than the tile before
constexpr uint32_t kSeq = kStart - 1;
// tiles after which the running angle is formed anew: it drifts by 2^-24 per tile
constexpr int kRenew = 32;

template <int D, int NT>
struct SmemB {
  static constexpr int ST = D == 128 && NT == 1 ? 3 : 5;  // two CTAs per SM, one for <128, 2>
  static constexpr int KS = D / 16;          // k steps of the score product
  static constexpr int RING = ST + 2;
  uint4 kv[ST][2][kTile * D / 8];            // K rows, V rows (also the flush's scratch)
  uint4 q[2][NT][KS][32];                    // B fragments (hi b0, hi b1, lo b0, lo b1)
  longlong2 off[2][kTile];                   // byte offsets of the K and V rows (of 8 rows each)
  TileInfo info[RING];
  float m[kDecWarps][8 * NT], l[kDecWarps][8 * NT];
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

// ROWS: rows that share one page lookup (8 where the page size is a multiple of 8, else 1).
template <int D, int NT, int ROWS>
__global__ void __launch_bounds__(kDecThreads) paged_decode_bf16_kernel(const PDecP p) {
  using S = SmemB<D, NT>;
  constexpr int HALF = D / 2, CH = D / 8, ST = S::ST, KS = S::KS, MT = D / 16, GT = 8 * NT;
  constexpr int RPP = kDecThreads / CH;            // rows that one pass of the CTA copies
  constexpr int HP = HALF / 2;                     // frequency pairs
  constexpr int QH = GT * HP / kDecThreads;        // heads of a thread in the query rotation
  extern __shared__ __align__(128) unsigned char smem_raw[];
  S& sm = *reinterpret_cast<S*>(smem_raw);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t total = scan_lengths<kDecThreads>(p, 0, nullptr);
  const int64_t t0 = total * blockIdx.x / gridDim.x, t1 = total * (blockIdx.x + 1) / gridDim.x;
  if (t0 >= t1) return;
  const int count = (int)(t1 - t0);
  Place oa = find_tile<kDecThreads>(p, t0);  // where the producer stands
  int q_it = 0, l_it = 0, o_it = 0;

  // ---- page lookups of a tile, by one warp at a time (the warps take turns).  The table entry is
  // read in lookup() and used in publish(), after the products of the tile in between.
  constexpr int LK = kTile / ROWS / 32 > 0 ? kTile / ROWS / 32 : 1;  // lookups of a lane
  int32_t entry[LK];
  auto lookup = [&]() {
    if (o_it < count && warp == (o_it & 3)) {
#pragma unroll
      for (int i = 0; i < LK; ++i) {
        const int r = (lane + 32 * i) * ROWS, j = oa.n * kTile + r;
        entry[i] = -1;
        if (r < kTile && j < oa.len) entry[i] = __ldg(p.c.table + oa.b * p.c.ts + (uint32_t)j / p.c.page);
      }
    }
  };
  auto publish = [&]() {
    if (o_it < count) {
      if (warp == (o_it & 3)) {
        bool good = true;
#pragma unroll
        for (int i = 0; i < LK; ++i) {
          const int r = (lane + 32 * i) * ROWS;
          const uint32_t j = (uint32_t)(oa.n * kTile + r);
          if (r < kTile) {
            longlong2 o = make_longlong2(-1, -1);  // no row
            if (j < (uint32_t)oa.len) {
              if (entry[i] < 0 || entry[i] >= p.c.n_pages) {
                o.x = -2;  // a page outside the pool
                good = false;
                atomicCAS(p.err, 0, kErrPageDecode);
              } else {
                const int64_t slot = j % p.c.page, h = oa.hg / p.NG;
                o = make_longlong2(entry[i] * p.c.ksp + h * p.c.ksh + slot * p.c.ksn,
                                   entry[i] * p.c.vsp + h * p.c.vsh + slot * p.c.vsn);
              }
            }
            sm.off[o_it & 1][r / ROWS] = o;
          }
        }
        good = __all_sync(0xffffffffu, good);
        if (lane == 0) {
          TileInfo t;
          t.b = (uint32_t)oa.b;
          if (good && oa.len - oa.n * kTile >= kTile) t.b |= kFull;
          if (oa.n == 0 || o_it == 0) t.b |= kStart;
          if (oa.n % kRenew == 0 || o_it == 0 || (p.L > 0 && oa.n * kTile % p.L == 0)) t.b |= kFresh;
          t.hg = oa.hg;
          t.n = oa.n;
          t.len = oa.len;
          sm.info[o_it % S::RING] = t;
        }
      }
      step(p, oa);
    }
    ++o_it;
  };
  // ---- copies of a tile's rows (rows without data are zero; of a bad page, K is NaN)
  const int lch = tid % CH, lrow = tid / CH;
  const int ldst = lrow * CH + (lch ^ (lrow & 7));  // 16-byte chunk in the stage, first pass
  const int64_t kthr = (lrow % ROWS) * p.c.ksn + lch * 16, vthr = (lrow % ROWS) * p.c.vsn + lch * 16;
  auto loads = [&]() {
    if (l_it < count) {
      uint4* ks = sm.kv[l_it % ST][0];
      uint4* vs = sm.kv[l_it % ST][1];
      const TileInfo t = sm.info[l_it % S::RING];
      if (t.b & kFull) {
#pragma unroll
        for (int i = 0; i < kTile / RPP; ++i) {
          const longlong2 o = sm.off[l_it & 1][(lrow + i * RPP) / ROWS];
          cp_async16(ks + ldst + i * RPP * CH, p.c.k + (o.x + kthr), 16);
          cp_async16(vs + ldst + i * RPP * CH, p.c.v + (o.y + vthr), 16);
        }
      } else {
        const int valid = t.len - t.n * kTile;
        for (int i = 0; i < kTile / RPP; ++i) {
          const int row = lrow + i * RPP, dst = ldst + i * RPP * CH;
          const longlong2 o = sm.off[l_it & 1][row / ROWS];
          const bool in = row < valid && o.x >= 0;
          cp_async16(vs + dst, p.c.v + (in ? o.y + vthr : 0), in ? 16 : 0);
          if (row < valid && o.x == -2) {
            ks[dst] = make_uint4(0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u);
          } else {
            cp_async16(ks + dst, p.c.k + (in ? o.x + kthr : 0), in ? 16 : 0);
          }
        }
      }
    }
    asm volatile("cp.async.commit_group;\n" ::: "memory");
    ++l_it;
  };
  // ---- queries of a tile: rotated by p_i - p_0, stored as B fragments.  From tile to tile of a
  // segment the angle moves by a constant step.
  const int qf = 2 * (tid % HP), qg = tid / HP;  // frequencies qf, qf + 1; heads qg + i * (128 / HP)
  float q1[QH][2], q2[QH][2], qc[2], qs[2], dc[2], ds[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    turn(-(double)kTile * (p.L > 0 ? 1.0 : p.pos_scale), __ldg(p.inv_freq + qf + e), dc[e], ds[e]);
    qc[e] = 1.f;
    qs[e] = 0.f;
  }
  auto queries = [&]() {
    if (q_it < count) {
      const TileInfo t = sm.info[q_it % S::RING];
      if (t.b & kStart) {
        const int gbase = (t.hg % p.NG) * GT, h0 = (t.hg / p.NG) * p.G + gbase;
#pragma unroll
        for (int i = 0; i < QH; ++i) {
          const int g = qg + i * (kDecThreads / HP);
          const bool in = gbase + g < p.G;
          const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(p.q) +
                                     (int64_t)(t.b & kSeq) * p.qsb + (h0 + g) * p.qsh + qf;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            q1[i][e] = in ? __bfloat162float(src[e]) * p.qscale : 0.f;
            q2[i][e] = in ? __bfloat162float(src[e + HALF]) * p.qscale : 0.f;
          }
        }
      }
      if (t.b & kFresh) {
        const double at = query_offset(p, t.len, t.n);
        turn(at, __ldg(p.inv_freq + qf), qc[0], qs[0]);
        turn(at, __ldg(p.inv_freq + qf + 1), qc[1], qs[1]);
      } else {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float c = qc[e] * dc[e] - qs[e] * ds[e];
          qs[e] = qs[e] * dc[e] + qc[e] * ds[e];
          qc[e] = c;
        }
      }
      const int ks = qf / 16, reg = (qf % 16) / 8, fc = (qf % 8) / 2;
#pragma unroll
      for (int i = 0; i < QH; ++i) {
        const int g = qg + i * (kDecThreads / HP);
        float r1[2], r2[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          r1[e] = q1[i][e] * qc[e] - q2[i][e] * qs[e];
          r2[e] = q2[i][e] * qc[e] + q1[i][e] * qs[e];
        }
        uint32_t hi, lo;
        pack_split(r1[0], r1[1], hi, lo);
        uint32_t* d = reinterpret_cast<uint32_t*>(&sm.q[q_it & 1][g / 8][ks][(g % 8) * 4 + fc]);
        d[reg] = hi;
        d[2 + reg] = lo;
        pack_split(r2[0], r2[1], hi, lo);
        d += KS / 2 * 32 * 4;
        d[reg] = hi;
        d[2 + reg] = lo;
      }
    }
    ++q_it;
  };

#pragma unroll
  for (int i = 0; i < ST - 1; ++i) {
    lookup();
    publish();
    __syncthreads();
    loads();
  }
  lookup();
  publish();
  queries();
  // cos / sin of this thread's key offsets, in the order of its A fragment's elements
  const int fr = lane >> 2, fc = lane & 3;
  f32x2 rc[KS / 2][4], rs[KS / 2][4], rn[KS / 2][4];  // cos, sin, -sin
  const f32x2 minus_one = pair(-1.f, -1.f);
#pragma unroll
  for (int ks = 0; ks < KS / 2; ++ks)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int t = warp * 16 + fr + (r & 1) * 8, f = ks * 16 + fc * 2 + (r >> 1) * 8;
      const double at = (double)t * (p.L > 0 ? 1.0 : p.pos_scale);
      float c[2], s[2];
      turn(at, __ldg(p.inv_freq + f), c[0], s[0]);
      turn(at, __ldg(p.inv_freq + f + 1), c[1], s[1]);
      rc[ks][r] = pair(c[0], c[1]);
      rs[ks][r] = pair(s[0], s[1]);
      rn[ks][r] = pair(-s[0], -s[1]);
    }

  float acc[NT][MT][4];
  float mx[NT][2], mref[NT][2], sum[NT][2];  // of heads 8 nt + 2 fc + {0, 1}; sums of this thread's keys
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int x = 0; x < 4; ++x) acc[nt][mt][x] = 0.f;
    mx[nt][0] = mx[nt][1] = -INFINITY;
    mref[nt][0] = mref[nt][1] = sum[nt][0] = sum[nt][1] = 0.f;
  }
  // ldmatrix lane addresses inside a stage (bytes)
  const uint32_t k_row = (uint32_t)(warp * 16 + (lane & 15)) * (D * 2), sw = lane & 7;
  const uint32_t v_row = (uint32_t)(warp * 16 + (lane & 7) + ((lane >> 4) << 3)) * (D * 2);

  for (int it = 0; it < count; ++it) {
    asm volatile("cp.async.wait_group %0;\n" ::"n"(ST - 2) : "memory");
    __syncthreads();
    loads();
    lookup();
    const TileInfo cur = sm.info[it % S::RING];
    const int cur_b = (int)(cur.b & kSeq);
    const uint32_t kb = smem_u32(sm.kv[it % ST][0]), vb = smem_u32(sm.kv[it % ST][1]);
    // ---- S^T
    float sc[NT][4][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int x = 0; x < 4; ++x) sc[nt][i][x] = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS / 2; ++ks) {
      uint32_t a[4], b[4], ah[4], al[4], bh[4], bl[4];
      const uint32_t ch = 2 * ks + (lane >> 4);
      ldsm_x4(kb + k_row + ((ch ^ sw) << 4), a[0], a[1], a[2], a[3]);
      ldsm_x4(kb + k_row + (((ch + CH / 2) ^ sw) << 4), b[0], b[1], b[2], b[3]);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const f32x2 x1 = widen(a[r]), x2 = widen(b[r]);
        split_cut(fma2(x2, rn[ks][r], mul2(x1, rc[ks][r])), minus_one, ah[r], al[r]);
        split_cut(fma2(x1, rs[ks][r], mul2(x2, rc[ks][r])), minus_one, bh[r], bl[r]);
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const uint4 qa4 = sm.q[it & 1][nt][ks][lane], qb4 = sm.q[it & 1][nt][ks + KS / 2][lane];
        mma_bf16(sc[nt][0], ah, qa4.x, qa4.y);
        mma_bf16(sc[nt][1], ah, qa4.z, qa4.w);
        mma_bf16(sc[nt][2], al, qa4.x, qa4.y);
        mma_bf16(sc[nt][3], al, qa4.z, qa4.w);
        mma_bf16(sc[nt][0], bh, qb4.x, qb4.y);
        mma_bf16(sc[nt][1], bh, qb4.z, qb4.w);
        mma_bf16(sc[nt][2], bl, qb4.x, qb4.y);
        mma_bf16(sc[nt][3], bl, qb4.z, qb4.w);
      }
    }
    // ---- online softmax over this warp's 16 keys (rows fr and fr + 8 of the fragment)
    uint32_t ph[NT][2], pl[NT][2];
    bool grow = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int x = 0; x < 4; ++x)
        sc[nt][0][x] = sc[nt][0][x] + ((sc[nt][1][x] + sc[nt][2][x]) + sc[nt][3][x]);
    if (!(cur.b & kFull)) {
      const int left = cur.len - cur.n * kTile - warp * 16 - fr;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int x = 0; x < 4; ++x)
          if ((x < 2 ? 0 : 8) >= left) sc[nt][0][x] = -INFINITY;
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) grow |= fmaxf(sc[nt][0][c], sc[nt][0][c + 2]) > mx[nt][c];
    if (__any_sync(0xffffffffu, grow)) {  // rare after the first tiles of a segment
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
      float* out = p.scores +
          (((int64_t)cur_b * p.c.Hkv * p.NG + cur.hg) * p.cap_tiles + cur.n) * GT * kTile + warp * 16 + fr;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int g = nt * 8 + fc * 2 + (x & 1);
          if ((cur.hg % p.NG) * GT + g < p.G) out[g * kTile + (x >> 1) * 8] = sc[nt][0][x];
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
        pack_split(e[2 * r], e[2 * r + 1], hi, lo);
        ph[nt][r] = transpose8x8(hi);
        pl[nt][r] = transpose8x8(lo);
      }
    }
    // ---- O^T += V^T . P^T
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      uint32_t a[4];
      const uint32_t ch = 2 * mt + ((lane >> 3) & 1);
      ldsm_x4_t(vb + v_row + ((ch ^ sw) << 4), a[0], a[1], a[2], a[3]);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        mma_bf16(acc[nt][mt], a, ph[nt][0], ph[nt][1]);
        mma_bf16(acc[nt][mt], a, pl[nt][0], pl[nt][1]);
      }
    }
    const bool seg_end = cur.n == n_tiles(cur.len) - 1;
    if (seg_end || it == count - 1) {
      // the warps' partial results of this segment, joined (in the stage just used) and stored
      float* part_acc = reinterpret_cast<float*>(sm.kv[it % ST][0]);  // [warp][head][d]
      __syncthreads();
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float l = sum[nt][c];
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
          const int g = nt * 8 + fc * 2 + c;
          if (fr == 0) {
            sm.m[warp][g] = mx[nt][c];
            sm.l[warp][g] = l;
          }
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            part_acc[(warp * GT + g) * D + mt * 16 + fr] = acc[nt][mt][c];
            part_acc[(warp * GT + g) * D + mt * 16 + fr + 8] = acc[nt][mt][c + 2];
            acc[nt][mt][c] = acc[nt][mt][c + 2] = 0.f;
          }
          mx[nt][c] = -INFINITY;
          mref[nt][c] = sum[nt][c] = 0.f;
        }
      __syncthreads();
      const bool started = cur.n <= it;  // the segment's first tile lies in this share
      const bool whole = seg_end && started;
      const int slot = 2 * blockIdx.x + (started ? 1 : 0);
      const int gbase = (cur.hg % p.NG) * GT, h0 = (cur.hg / p.NG) * p.G + gbase;
      const int heads = min(GT, p.G - gbase);
      for (int i = tid; i < heads * D; i += kDecThreads) {
        const int g = i / D, d = i % D;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < kDecWarps; ++w) M = fmaxf(M, sm.m[w][g]);
        const float ms = M == -INFINITY ? 0.f : M;
        float L = 0.f, o = 0.f;
#pragma unroll
        for (int w = 0; w < kDecWarps; ++w) {
          const float f = exp2f(sm.m[w][g] - ms);
          L += sm.l[w][g] * f;
          o += part_acc[(w * GT + g) * D + d] * f;
        }
        if (whole) {
          store_out(static_cast<__nv_bfloat16*>(p.out) + ((int64_t)cur_b * p.H + h0 + g) * D + d, o / L);
          if (d == 0) p.ml[(int64_t)cur_b * p.H + h0 + g] = make_float2(ms, 1.f / L);
        } else {
          p.part[((int64_t)slot * GT + g) * D + d] = o;
          if (d == 0) p.part_ml[(int64_t)slot * GT + g] = make_float2(M, L);
        }
      }
    }
    publish();
    queries();
  }
}

template <int D, int NT, int ROWS>
int launch(const PDecP& p, int W, cudaStream_t st) {
  constexpr int bytes = (int)sizeof(SmemB<D, NT>);
  const cudaError_t e = cudaFuncSetAttribute(paged_decode_bf16_kernel<D, NT, ROWS>,
                                             cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return fail(STA_ERR_CUDA, cudaGetErrorString(e));
  paged_decode_bf16_kernel<D, NT, ROWS><<<W, kDecThreads, bytes, st>>>(p);
  return STA_OK;
}

template <int D, int NT>
int launch(const PDecP& p, int W, cudaStream_t st) {
  return p.c.page % 8 == 0 ? launch<D, NT, 8>(p, W, st) : launch<D, NT, 1>(p, W, st);
}

}  // namespace

int paged_decode_bf16_ctas(int d, int GT) { return d == 128 && GT == 16 ? 1 : 2; }

int launch_paged_decode_bf16(const PDecP& p, int d, int W, cudaStream_t st) {
  if (d == 128) return p.GT == 8 ? launch<128, 1>(p, W, st) : launch<128, 2>(p, W, st);
  return p.GT == 8 ? launch<64, 1>(p, W, st) : launch<64, 2>(p, W, st);
}

}  // namespace sta
