// Decode over a paged bf16 cache on the tensor cores (schedule and rotation: paged_decode.cuh).
//
// One new token has few q heads per kv head, so the products are (64 keys) x (d) x (8 or 16
// heads): warp-level m16n8k16 with the keys as rows wastes nothing up to 8 heads, where a
// 128-row tcgen05 tile would spend 15 of 16 rows on padding.  A warp owns 16 keys of each tile:
//   S^T (16 keys x heads) = K (rotated) . Q^T     A = K rows (ldmatrix), B = the tile's queries
//   O^T (d x heads)      += V^T . P^T             A = V^T (ldmatrix.trans), B = P transposed in
//                                                 registers (movmatrix)
// Rotated keys, queries and probabilities are fp32 values carried as hi + lo bf16 pieces (three
// products for S, two for P.V: V is exact), which leaves errors near 2^-16, far below the output's
// own rounding; running max, sums and accumulators are fp32.
//
// The rows of two to four tiles are in flight per CTA (cp.async, 16-byte chunks swizzled by row); a
// thread's cos / sin of the tile-local key offsets stay in registers for the whole call.
#include "mma_frag.cuh"
#include "paged_decode.cuh"

namespace sta {

namespace {

template <int D, int NT>
struct SmemB {
  static constexpr int ST = D == 128 && NT == 1 ? 3 : 5;  // two CTAs per SM, one for <128, 2>
  static constexpr int KS = D / 16;          // k steps of the score product
  uint4 kv[ST][2][kTile * D / 8];            // K rows, V rows (also the flush's scratch)
  uint4 q[2][NT][KS][32];                    // B fragments (hi b0, hi b1, lo b0, lo b1)
  longlong2 off[2][kTile];                   // byte offsets of the K and V row
  float m[kDecWarps][8 * NT], l[kDecWarps][8 * NT];
};

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

template <int D, int NT>
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
  Place cur = find_tile<kDecThreads>(p, t0);
  Place qa = cur, oa = cur;  // where queries and row offsets stand
  int q_it = 0, l_it = 0, o_it = 0;

  // ---- row offsets of a tile (threads 0 .. 63), -1: no row, -2: a page outside the pool
  auto offsets = [&]() {
    if (o_it < count) {
      if (tid < kTile) {
        const int j = oa.n * kTile + tid;
        longlong2 o = make_longlong2(-1, -1);
        if (j < oa.len) {
          const uint32_t t = (uint32_t)j / p.c.page;
          const int64_t pg = paged_page(p.c, p.c.table, p.c.ts, oa.b, t);
          if (pg < 0) {
            o.x = -2;
            atomicCAS(p.err, 0, kErrPageDecode);
          } else {
            const int64_t slot = (uint32_t)j - t * p.c.page, h = oa.hg / p.NG;
            o = make_longlong2(pg * p.c.ksp + h * p.c.ksh + slot * p.c.ksn,
                               pg * p.c.vsp + h * p.c.vsh + slot * p.c.vsn);
          }
        }
        sm.off[o_it & 1][tid] = o;
      }
      step(p, oa);
    }
    ++o_it;
  };
  // ---- copies of a tile's rows (rows without data are zero; of a bad page, K is NaN)
  const int lch = tid % CH, lrow = tid / CH;
  const int ldst = lrow * CH + (lch ^ (lrow & 7));  // 16-byte chunk in the stage, first pass
  auto loads = [&]() {
    if (l_it < count) {
      uint4* ks = sm.kv[l_it % ST][0];
      uint4* vs = sm.kv[l_it % ST][1];
#pragma unroll
      for (int i = 0; i < kTile / RPP; ++i) {
        const longlong2 o = sm.off[l_it & 1][lrow + i * RPP];
        const int dst = ldst + i * RPP * CH;
        cp_async16(vs + dst, p.c.v + (o.y >= 0 ? o.y + lch * 16 : 0), o.y >= 0 ? 16 : 0);
        if (o.x == -2) {
          ks[dst] = make_uint4(0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u);
        } else {
          cp_async16(ks + dst, p.c.k + (o.x >= 0 ? o.x + lch * 16 : 0), o.x >= 0 ? 16 : 0);
        }
      }
    }
    asm volatile("cp.async.commit_group;\n" ::: "memory");
    ++l_it;
  };
  // ---- queries of a tile: rotated by p_i - p_0, stored as B fragments
  const int qf = 2 * (tid % HP), qg = tid / HP;  // frequencies qf, qf + 1; heads qg + i * (128 / HP)
  float q1[QH][2], q2[QH][2];
  auto queries = [&]() {
    if (q_it < count) {
      if (q_it == 0 || qa.n == 0) {
        const int gbase = (qa.hg % p.NG) * GT, h0 = (qa.hg / p.NG) * p.G + gbase;
#pragma unroll
        for (int i = 0; i < QH; ++i) {
          const int g = qg + i * (kDecThreads / HP);
          const bool in = gbase + g < p.G;
          const __nv_bfloat16* src =
              static_cast<const __nv_bfloat16*>(p.q) + qa.b * p.qsb + (h0 + g) * p.qsh + qf;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            q1[i][e] = in ? __bfloat162float(src[e]) * p.qscale : 0.f;
            q2[i][e] = in ? __bfloat162float(src[e + HALF]) * p.qscale : 0.f;
          }
        }
      }
      const double at = query_offset(p, qa);
      float c[2], s[2];
      turn(at, __ldg(p.inv_freq + qf), c[0], s[0]);
      turn(at, __ldg(p.inv_freq + qf + 1), c[1], s[1]);
      const int ks = qf / 16, reg = (qf % 16) / 8, fc = (qf % 8) / 2;
#pragma unroll
      for (int i = 0; i < QH; ++i) {
        const int g = qg + i * (kDecThreads / HP);
        float r1[2], r2[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          r1[e] = q1[i][e] * c[e] - q2[i][e] * s[e];
          r2[e] = q2[i][e] * c[e] + q1[i][e] * s[e];
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
      step(p, qa);
    }
    ++q_it;
  };

#pragma unroll
  for (int i = 0; i < ST - 1; ++i) {
    offsets();
    __syncthreads();
    loads();
  }
  offsets();
  queries();
  // cos / sin of this thread's key offsets, in the order of its A fragment's elements
  const int fr = lane >> 2, fc = lane & 3;
  float rc[KS / 2][4][2], rs[KS / 2][4][2];
#pragma unroll
  for (int ks = 0; ks < KS / 2; ++ks)
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int t = warp * 16 + fr + (r & 1) * 8, f = ks * 16 + fc * 2 + (r >> 1) * 8 + e;
        turn((double)t * p.pos_scale, __ldg(p.inv_freq + f), rc[ks][r][e], rs[ks][r][e]);
      }

  float acc[NT][MT][4];
  float mx[NT][2], sum[NT][2];  // of heads 8 nt + 2 fc + {0, 1}; sums of this thread's keys only
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int x = 0; x < 4; ++x) acc[nt][mt][x] = 0.f;
    mx[nt][0] = mx[nt][1] = -INFINITY;
    sum[nt][0] = sum[nt][1] = 0.f;
  }
  // ldmatrix lane addresses inside a stage (bytes)
  const uint32_t k_row = (uint32_t)(warp * 16 + (lane & 15)) * (D * 2), k_sw = lane & 7;
  const uint32_t v_row = (uint32_t)(warp * 16 + (lane & 7) + ((lane >> 4) << 3)) * (D * 2);

  for (int it = 0; it < count; ++it) {
    asm volatile("cp.async.wait_group %0;\n" ::"n"(ST - 2) : "memory");
    __syncthreads();
    loads();
    const uint32_t kb = smem_u32(sm.kv[it % ST][0]), vb = smem_u32(sm.kv[it % ST][1]);
    // ---- S^T
    float sc[NT][3][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 3; ++i)
#pragma unroll
        for (int x = 0; x < 4; ++x) sc[nt][i][x] = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS / 2; ++ks) {
      uint32_t a[4], b[4], ah[4], al[4], bh[4], bl[4];
      const uint32_t ch = 2 * ks + (lane >> 4);
      ldsm_x4(kb + k_row + ((ch ^ k_sw) << 4), a[0], a[1], a[2], a[3]);
      ldsm_x4(kb + k_row + (((ch + CH / 2) ^ k_sw) << 4), b[0], b[1], b[2], b[3]);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float r1[2], r2[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float x1 = __uint_as_float(e ? a[r] & 0xffff0000u : a[r] << 16);
          const float x2 = __uint_as_float(e ? b[r] & 0xffff0000u : b[r] << 16);
          r1[e] = x1 * rc[ks][r][e] - x2 * rs[ks][r][e];
          r2[e] = x2 * rc[ks][r][e] + x1 * rs[ks][r][e];
        }
        pack_split(r1[0], r1[1], ah[r], al[r]);
        pack_split(r2[0], r2[1], bh[r], bl[r]);
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const uint4 qa4 = sm.q[it & 1][nt][ks][lane], qb4 = sm.q[it & 1][nt][ks + KS / 2][lane];
        mma_bf16(sc[nt][0], ah, qa4.x, qa4.y);
        mma_bf16(sc[nt][1], ah, qa4.z, qa4.w);
        mma_bf16(sc[nt][2], al, qa4.x, qa4.y);
        mma_bf16(sc[nt][0], bh, qb4.x, qb4.y);
        mma_bf16(sc[nt][1], bh, qb4.z, qb4.w);
        mma_bf16(sc[nt][2], bl, qb4.x, qb4.y);
      }
    }
    // ---- online softmax over this warp's 16 keys
    const int key = cur.n * kTile + warp * 16 + fr;  // rows fr and fr + 8 of the fragment
    const bool in0 = key < cur.len, in1 = key + 8 < cur.len;
    uint32_t ph[NT][2], pl[NT][2];
    float mn[NT][2];
    bool grow = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float s = sc[nt][0][x] + (sc[nt][1][x] + sc[nt][2][x]);
        sc[nt][0][x] = (x < 2 ? in0 : in1) ? s : -INFINITY;
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float m = fmaxf(sc[nt][0][c], sc[nt][0][c + 2]);
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        mn[nt][c] = fmaxf(mx[nt][c], m);
        grow |= mn[nt][c] > mx[nt][c];
      }
    }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float f = exp2f(mx[nt][c] - (mn[nt][c] == -INFINITY ? 0.f : mn[nt][c]));
          sum[nt][c] *= f;
          mx[nt][c] = mn[nt][c];
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            acc[nt][mt][c] *= f;
            acc[nt][mt][c + 2] *= f;
          }
        }
    }
    if (p.scores) {
      float* out = p.scores +
          (((int64_t)cur.b * p.c.Hkv * p.NG + cur.hg) * p.cap_tiles + cur.n) * GT * kTile + warp * 16 + fr;
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
        e[x] = exp2f(sc[nt][0][x] - (mx[nt][x & 1] == -INFINITY ? 0.f : mx[nt][x & 1]));
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
      ldsm_x4_t(vb + v_row + ((ch ^ k_sw) << 4), a[0], a[1], a[2], a[3]);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        mma_bf16(acc[nt][mt], a, ph[nt][0], ph[nt][1]);
        mma_bf16(acc[nt][mt], a, pl[nt][0], pl[nt][1]);
      }
    }
    const bool seg_end = cur.n == cur.tiles - 1;
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
          sum[nt][c] = 0.f;
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
          store_out(static_cast<__nv_bfloat16*>(p.out) + ((int64_t)cur.b * p.H + h0 + g) * D + d, o / L);
          if (d == 0) {
            float* ml = p.ml + ((int64_t)cur.b * p.H + h0 + g) * 2;
            ml[0] = ms;
            ml[1] = 1.f / L;
          }
        } else {
          float* part = p.part + ((int64_t)slot * GT + g) * (D + 2);
          part[d] = o;
          if (d == 0) {
            part[D] = M;
            part[D + 1] = L;
          }
        }
      }
    }
    offsets();
    queries();
    step(p, cur);
  }
}

template <int D, int NT>
int launch(const PDecP& p, int W, cudaStream_t st) {
  constexpr int bytes = (int)sizeof(SmemB<D, NT>);
  const cudaError_t e = cudaFuncSetAttribute(paged_decode_bf16_kernel<D, NT>,
                                             cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return fail(STA_ERR_CUDA, cudaGetErrorString(e));
  paged_decode_bf16_kernel<D, NT><<<W, kDecThreads, bytes, st>>>(p);
  return STA_OK;
}

}  // namespace

int paged_decode_bf16_ctas(int d, int GT) { return d == 128 && GT == 16 ? 1 : 2; }

int launch_paged_decode_bf16(const PDecP& p, int d, int W, cudaStream_t st) {
  if (d == 128) return p.GT == 8 ? launch<128, 1>(p, W, st) : launch<128, 2>(p, W, st);
  return p.GT == 8 ? launch<64, 1>(p, W, st) : launch<64, 2>(p, W, st);
}

}  // namespace sta
