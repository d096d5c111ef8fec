// What the decode kernels of the paged cache share: the list of tiles and a CTA's place in it, the
// rotation of a tile's query, and the parameters.
#pragma once

#include "paged.cuh"

namespace sta {

constexpr int kTile = 64;      // keys per tile
constexpr int kDecThreads = 128;  // 4 warps, 16 keys of a tile each
constexpr int kDecWarps = kDecThreads / 32;

struct PDecP {
  PagedView c;
  const void* q;
  int64_t qsb, qsh;  // elements
  void* out;
  int H, G, NG, GT;  // q heads, per kv head, groups of GT of them
  const float* inv_freq;
  double pos_scale;
  float qscale;      // sm_scale * rope_scale^2 * log2(e): scores are in units of log2
  int L, s;          // Dual Chunk Attention: chunk length and chunk size, L = 0 for plain positions
  float* part;       // (2 * W, GT, D): unnormalised outputs of cut segments
  float2* part_ml;   // (2 * W, GT): their max and sum
  float2* ml;        // (B, H): max and 1 / sum of segments that one share holds
  float* scores;     // (B, Hkv * NG, capacity tiles, GT, 64) or null
  int64_t cap_tiles;
  float* w_out;
  int* err;
};

__device__ __forceinline__ int n_tiles(int len) { return (len + kTile - 1) / kTile; }

// A CTA's place in the list of tiles.
struct Place {
  int b, hg, n, tiles, len;
};

__device__ __forceinline__ void seek_sequence(const PagedView& c, Place& a) {
  a.tiles = 0;
  while (a.b < c.B) {
    a.len = paged_len(c, a.b);
    a.tiles = n_tiles(a.len);
    if (a.tiles > 0) return;
    ++a.b;
  }
}

__device__ __forceinline__ void step(const PDecP& p, Place& a) {
  if (++a.n < a.tiles) return;
  a.n = 0;
  if (++a.hg < p.c.Hkv * p.NG) return;
  a.hg = 0;
  ++a.b;
  seek_sequence(p.c, a);
}

// Number of tiles of all segments (block-wide, NT threads), and with `find` >= 0 the place of
// tile `find`; `before` receives the tiles of the sequences before sequence `until`.
template <int NT>
__device__ __forceinline__ int64_t scan_lengths(const PDecP& p, int until, int64_t* before) {
  __shared__ int64_t s_all[NT / 32], s_bef[NT / 32];
  const int tid = threadIdx.x;
  int64_t all = 0, bef = 0;
  for (int b = tid; b < p.c.B; b += NT) {
    const int t = n_tiles(paged_len(p.c, b));
    all += t;
    if (b < until) bef += t;
  }
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) {
    all += __shfl_xor_sync(0xffffffffu, all, o);
    bef += __shfl_xor_sync(0xffffffffu, bef, o);
  }
  if ((tid & 31) == 0) {
    s_all[tid >> 5] = all;
    s_bef[tid >> 5] = bef;
  }
  __syncthreads();
  all = bef = 0;
#pragma unroll
  for (int i = 0; i < NT / 32; ++i) {
    all += s_all[i];
    bef += s_bef[i];
  }
  __syncthreads();
  const int64_t hg = (int64_t)p.c.Hkv * p.NG;
  if (before) *before = bef * hg;
  return all * hg;
}

template <int NT>
__device__ __forceinline__ Place find_tile(const PDecP& p, int64_t t) {
  __shared__ int s_b, s_hit;
  __shared__ int64_t s_rest, s_sum[NT / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t hg = (int64_t)p.c.Hkv * p.NG;
  int64_t base = 0;
  Place a{};
  if (tid == 0) s_hit = 0;
  __syncthreads();
  for (int b0 = 0; b0 < p.c.B; b0 += NT) {
    const int b = b0 + tid;
    const int64_t mine = b < p.c.B ? (int64_t)n_tiles(paged_len(p.c, b)) * hg : 0;
    int64_t inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    if (lane == 31) s_sum[warp] = inc;
    __syncthreads();
    int64_t off = base, tot = 0;
#pragma unroll
    for (int i = 0; i < NT / 32; ++i) {
      if (i < warp) off += s_sum[i];
      tot += s_sum[i];
    }
    const int64_t lo = off + inc - mine;
    if (mine > 0 && t >= lo && t < lo + mine) {
      s_b = b;
      s_rest = t - lo;
      s_hit = 1;
    }
    __syncthreads();
    if (s_hit) break;
    base += tot;
  }
  a.b = s_b;
  a.len = paged_len(p.c, a.b);
  a.tiles = n_tiles(a.len);
  a.hg = (int)(s_rest / a.tiles);
  a.n = (int)(s_rest - (int64_t)a.hg * a.tiles);
  return a;
}

// cos / sin of pos * inv_freq: the angle in turns is formed and reduced in 64 bits
__device__ __forceinline__ void turn(double pos, float inv_freq, float& c, float& s) {
  const double x = pos * ((double)inv_freq * 0.15915494309189533577);  // 1 / (2 pi)
  sincospif((float)(2.0 * (x - rint(x))), &s, &c);
}

// p_i - p_0 of a tile (position of the query minus that of the tile's first key)
__device__ __forceinline__ double query_offset(const PDecP& p, int len, int n) {
  const int i = len - 1, j0 = n * kTile;
  if (p.L == 0) return (double)i * p.pos_scale - (double)j0 * p.pos_scale;
  const int away = i / p.L - j0 / p.L, in = i % p.L;
  const int qp = away == 0 ? in : (away == 1 ? min(p.L + in, p.s) : min(2 * p.L - 1, p.s));
  return (double)(qp - j0 % p.L);
}

__device__ __forceinline__ void store_out(float* o, float x) { *o = x; }
__device__ __forceinline__ void store_out(__nv_bfloat16* o, float x) { *o = __float2bfloat16_rn(x); }

// Decode kernel for bf16 caches (tensor cores): CTAs that fit one SM, and the launch of W CTAs.
int paged_decode_bf16_ctas(int d, int GT);
int launch_paged_decode_bf16(const PDecP& p, int d, int W, cudaStream_t st);

}  // namespace sta
