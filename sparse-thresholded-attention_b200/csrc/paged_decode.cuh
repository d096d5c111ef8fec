// What the decode kernels of the paged cache share: the list of units (runs of keys) and a share's
// place in it, the angles of the rotation, and the parameters.
#pragma once

#include "paged.cuh"

namespace sta {

constexpr int kTile = 64;  // keys whose query is rotated once; block of the scores buffer

struct PDecP {
  PagedView c;
  const void* q;
  int64_t qsb, qsh;  // elements
  int q_words;       // 16-bit queries start on 4-byte boundaries
  void* out;
  int H, G, NG, GT;  // q heads, per kv head, groups of GT of them
  int SG;            // heads of a group that are there: min(G, GT)
  int unit;          // log2 of the keys of a unit of work
  int W, min_log;    // shares at most, log2 of the units of a share at least
  int sms;
  int merge;         // bf16: whether a CTA may join its shares' partials; shares from which on it does
  int64_t k16, v16;  // bytes of 16 rows
  const float* inv_freq;
  double pos_scale;
  float qscale;      // sm_scale * rope_scale^2 * log2(e): scores are in units of log2
  int L, s;          // Dual Chunk Attention: chunk length and chunk size, L = 0 for plain positions
  float* part;       // (2 * W, GT, D): unnormalised outputs of cut segments
  float2* part_ml;   // (2 * W, GT): their max and sum
  float2* ml;        // (B, H): max and 1 / sum of segments that one share holds
  float* scores;     // (B, Hkv * NG, capacity tiles, SG, 64) or null
  int64_t cap_tiles;
  float* w_out;
  int2* places;      // (n_pages,) with the weights: which table entry adds to a page's
  int* err;
};

__device__ __forceinline__ int n_units(const PDecP& p, int len) {
  return (int)(((uint32_t)len + (1u << p.unit) - 1u) >> p.unit);
}

// Units of all segments (sequence, kv head, q-head group), summed by a warp; `before` receives
// those of the sequences before `until`.
__device__ __forceinline__ int64_t scan_lengths(const PDecP& p, int until, int64_t* before) {
  int64_t all = 0, bef = 0;
  for (int b = threadIdx.x & 31; b < p.c.B; b += 32) {
    const int t = n_units(p, paged_len(p.c, b));
    all += t;
    if (b < until) bef += t;
  }
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) {
    all += __shfl_xor_sync(0xffffffffu, all, o);
    if (before) bef += __shfl_xor_sync(0xffffffffu, bef, o);
  }
  const int64_t hg = (int64_t)p.c.Hkv * p.NG;
  if (before) *before = bef * hg;
  return all * hg;
}

// Shares that the units are cut into: share w holds the units from share_begin(w) = total w / W
// (rounded down) to share_begin(w + 1).
__device__ __forceinline__ int64_t n_shares(const PDecP& p, int64_t total) {
  const int64_t w = (total + (1 << p.min_log) - 1) >> p.min_log;
  return w < p.W ? w : p.W;
}

// x / y for x >= 0, y > 0; 64-bit divisions are long, and seldom needed
__device__ __forceinline__ int64_t div_fast(int64_t x, int64_t y) {
  return ((x | y) >> 32) == 0 ? (int64_t)((uint32_t)x / (uint32_t)y) : x / y;
}
__device__ __forceinline__ int64_t share_begin(int64_t total, int64_t w, int64_t W) {
  return div_fast(total * w, W);
}

// A place in the list of units.
struct Place {
  int b, h, grp, n, units, len;  // sequence, kv head, q-head group, unit of the segment
};

__device__ __forceinline__ void seek_sequence(const PDecP& p, Place& a) {
  a.units = 0;
  while (a.b < p.c.B) {
    a.len = paged_len(p.c, a.b);
    a.units = n_units(p, a.len);
    if (a.units > 0) return;
    ++a.b;
  }
}

__device__ __forceinline__ void step(const PDecP& p, Place& a) {
  if (++a.n < a.units) return;
  a.n = 0;
  if (++a.grp < p.NG) return;
  a.grp = 0;
  if (++a.h < p.c.Hkv) return;
  a.h = 0;
  ++a.b;
  seek_sequence(p, a);
}

// What the share of this warp holds: `count` units from the place `at` on (count 0: nothing).  The
// shares are dealt to the CTAs in runs of (nearly) equal length; `me` receives the warp's (of a
// CTA that is a share by itself: every warp's is the CTA's).  `len` is the length of sequence
// `lane` (0 beyond the batch).
struct Share {
  int count;
  bool merge;  // the CTA joins its shares' partials (else the join takes them all)
  Place at;
};

template <bool WARP_SHARES = true>
__device__ __forceinline__ Share find_share(const PDecP& p, int len, int64_t& me) {
  const int lane = threadIdx.x & 31;
  const int64_t hg = (int64_t)p.c.Hkv * p.NG;
  int64_t mine = n_units(p, len) * hg, inc = mine;  // of the first 32 sequences
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += y;
  }
  int64_t base = 0, total = __shfl_sync(0xffffffffu, inc, 31);
  const int64_t head = total;
  if (p.c.B > 32) {
    int64_t more = 0;
    for (int b = 32 + lane; b < p.c.B; b += 32) more += n_units(p, paged_len(p.c, b));
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) more += __shfl_xor_sync(0xffffffffu, more, o);
    total += more * hg;
  }
  const int64_t shares = n_shares(p, total);
  Share s{};
  s.merge = shares >= p.merge;
  int64_t end = shares;
  me = blockIdx.x;
  if (WARP_SHARES) {
    me = share_begin(shares, blockIdx.x, gridDim.x) + (threadIdx.x >> 5);
    end = share_begin(shares, blockIdx.x + 1, gridDim.x);
  }
  if (me >= end) return s;
  const int64_t t = share_begin(total, me, shares);
  s.count = (int)(share_begin(total, me + 1, shares) - t);
  int b0 = 0;
  while (t >= base + (b0 == 0 ? head : __shfl_sync(0xffffffffu, inc, 31))) {  // (t < total: ends)
    base += b0 == 0 ? head : __shfl_sync(0xffffffffu, inc, 31);
    b0 += 32;
    len = b0 + lane < p.c.B ? paged_len(p.c, b0 + lane) : 0;
    inc = mine = n_units(p, len) * hg;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
  }
  const int src = __ffs(__ballot_sync(0xffffffffu, t < base + inc)) - 1;
  const int64_t rest = t - base - __shfl_sync(0xffffffffu, inc - mine, src);
  s.at.b = b0 + src;
  s.at.len = __shfl_sync(0xffffffffu, len, src);
  s.at.units = n_units(p, s.at.len);
  const int g = (int)div_fast(rest, s.at.units);
  s.at.n = (int)(rest - (int64_t)g * s.at.units);
  s.at.h = p.NG == 1 ? g : g / p.NG;
  s.at.grp = g - s.at.h * p.NG;
  return s;
}

__device__ __forceinline__ int first_len(const PagedView& c) {
  const int lane = threadIdx.x & 31;
  return lane < c.B ? paged_len(c, lane) : 0;
}

// cos / sin of pos * inv_freq: the angle in turns is formed and reduced in 64 bits
__device__ __forceinline__ void turn(double pos, float inv_freq, float& c, float& s) {
  const double x = pos * ((double)inv_freq * 0.15915494309189533577);  // 1 / (2 pi)
  sincospif((float)(2.0 * (x - rint(x))), &s, &c);
}

// p_i - p_0 of a tile (position of the query minus that of the tile's first key)
__device__ __forceinline__ double query_offset(const PDecP& p, int len, int tile) {
  const int i = len - 1, j0 = tile * kTile;
  if (p.L == 0) return (double)i * p.pos_scale - (double)j0 * p.pos_scale;
  const int away = i / p.L - j0 / p.L, in = i % p.L;
  const int qp = away == 0 ? in : (away == 1 ? min(p.L + in, p.s) : min(2 * p.L - 1, p.s));
  return (double)(qp - j0 % p.L);
}

__device__ __forceinline__ void store_out(float* o, float x) { *o = x; }
__device__ __forceinline__ void store_out(__nv_bfloat16* o, float x) { *o = __float2bfloat16_rn(x); }

// Decode kernel for bf16 caches (tensor cores): shares per SM that it runs, keys of a unit
// (log2), and the launch for p.W shares.
int paged_decode_bf16_shares(int d, int GT);
constexpr int kUnitBf16 = 4, kUnitF32 = 6;
int launch_paged_decode_bf16(const PDecP& p, int d, cudaStream_t st);

}  // namespace sta
