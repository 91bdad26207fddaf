// lbk_adapter.hip — low-rank adapters of many requests beside a shared projection, out = y + s B (A x) with each
// token's own A, B and s, with the backward (gfx950, bf16 or fp16 MFMA, fp32 sums), and the entry points of
// include/lbk.h.
//
// Tokens are sorted by adapter once for all projections (the plan) and taken in tiles of up to 64 tokens of one adapter:
//   shrink  t = A x of a tile, K in shares, fp32 partial sums          expand  out = y + B t', t' = s (sum of t's shares)
//   grad    dA = dt'^T x, dB = dy^T t' over an adapter's tiles         with dt' = s B^T dy by shrink, dx = A^T dt' by expand
// t' and dt' enter the second products as three bf16 each, which hold all 24 bits of an fp32 mantissa (8 bits at a time, cut
// off and not rounded): fp32 sums as the first products', at three matrix instructions where these calls wait for memory.
// fp16 operands beside them are two bf16, which is exact; of the six products the last, below 2^-24 of the whole, is left out.
#include "lbk.h"
#include "lbk_device.h"
#include "lbk_internal.h"

#include <algorithm>

namespace lbk {
namespace {

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));

constexpr int TILE = 64;             // tokens of a tile: four subtiles of a matrix instruction's 16
constexpr int MAX_ADAPTERS = 4096, MAX_RANK = 256;

// ------------------------------------------------------------------ the plan
// int32 words: seg [n + 2] (first place of each bin; bin n holds the tokens without an adapter), tstart [n + 2] (first
// tile), tiles [max_tiles] of {adapter or -1, first place, tokens, bins with tokens before}, perm [N] (place -> token).
struct Tile {
  int32_t adapter, first, count, ord;
};

__host__ __device__ inline int64_t max_tiles(int64_t N, int n) { return N / TILE + (N < n + 1 ? N : n + 1); }
inline int64_t plan_words(int64_t N, int n) { return 2 * ((int64_t)n + 2 + ((n & 1) ? 1 : 0)) + 4 * max_tiles(N, n) + N + 4; }

struct Plan {
  const int32_t *seg, *tstart, *perm;
  const Tile* tiles;
};
__host__ __device__ inline Plan plan_view(const int32_t* p, int64_t N, int n) {
  const int64_t w = ((int64_t)n + 2 + 1) & ~(int64_t)1;        // even: the tiles lie on 16 bytes
  const int32_t* tiles = p + 2 * w;
  return {p, p + w, tiles + 4 * max_tiles(N, n), reinterpret_cast<const Tile*>(tiles)};
}

// A tile as a kernel may use it, whatever buffer was passed for the plan; adapter -1: none
__device__ __forceinline__ Tile tile_at(const Plan& p, int64_t k, int64_t N, int n) {
  Tile t = p.tiles[k];
  t.adapter = t.adapter < 0 || t.adapter > n || t.count < 1 ? -1 : t.adapter;
  t.first = min((uint32_t)t.first, (uint32_t)(N - 1));
  t.count = min(t.count, min(TILE, (int)(N - t.first)));
  return t;
}
__device__ __forceinline__ int64_t row_at(const Plan& p, int place, int64_t N) { return min((uint32_t)p.perm[place], (uint32_t)(N - 1)); }

// A stable counting sort by one workgroup, once for all projections of a batch (16384 tokens: 19 us, 64: 5.6).  Each wave
// counts a run of tokens of its own, the counts are added up bin by
// bin and wave by wave, and each wave goes over its run again: a token's place is its bin's and wave's first one plus
// the same bin's tokens before it, those of the wave's 64 found by comparing the bins' bits.
template <typename I>
__global__ __launch_bounds__(1024) void plan_kernel(const I* __restrict__ ids, int64_t N, int n, int waves, int32_t* __restrict__ plan) {
  extern __shared__ int32_t lds[];
  int32_t* cnt = lds;                        // [waves][n + 1]
  int32_t* ts = lds + waves * (n + 1);       // [n + 2] tiles before a bin
  __shared__ int32_t wsum[3][16];
  const int tid = threadIdx.x, T = blockDim.x, lane = tid & 63, w = uniform(tid >> 6), nw = T >> 6;
  const Plan pv = plan_view(plan, N, n);
  int32_t *seg = const_cast<int32_t*>(pv.seg), *tstart = const_cast<int32_t*>(pv.tstart), *perm = const_cast<int32_t*>(pv.perm);
  Tile* tiles = const_cast<Tile*>(pv.tiles);
  for (int k = tid; k < waves * (n + 1); k += T) cnt[k] = 0;
  const int64_t run = ((N + waves - 1) / waves + 63) / 64 * 64, r0 = w * run, r1 = min(r0 + run, N);
  int bits = 1;
  while (n >> bits) ++bits;
  // the lanes whose token has this lane's bin (-1: no token): the first of them counts for all, as 64 additions to one
  // counter would follow each other
  auto alike = [&](int b) {
    uint64_t same = __ballot(b >= 0);
    for (int k = 0; k < bits; ++k) {
      const uint64_t m = __ballot(b >= 0 && (b >> k & 1));
      same &= (b >> k & 1) ? m : ~m;
    }
    return same;
  };
  constexpr int AHEAD = 8;                   // turns of 64 tokens whose ids are loaded together
  auto load = [&](int64_t t0, int (&b)[AHEAD]) {
    I v[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) v[k] = t0 + 64 * k + lane < r1 ? ids[t0 + 64 * k + lane] : (I)0;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) b[k] = t0 + 64 * k + lane >= r1 ? -1 : v[k] >= 0 && v[k] < n ? (int)v[k] : n;
  };
  int kept[AHEAD];                           // the run's first ones, for the second time too
  if (w < waves) load(r0, kept);
  __syncthreads();
  if (w < waves)
    for (int64_t t0 = r0; t0 < r1; t0 += 64 * AHEAD) {
      int b[AHEAD];
      if (t0 > r0) load(t0, b);
      else
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) b[k] = kept[k];
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        if (!__ballot(b[k] >= 0)) break;
        const uint64_t same = alike(b[k]);
        if (b[k] >= 0 && !(same & (((uint64_t)1 << lane) - 1))) cnt[w * (n + 1) + b[k]] += __popcll(same);
        // a counter's next addition may be another lane's
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
      }
    }
  __syncthreads();
  // tokens, tiles and bins before each bin: every thread has a run of bins
  const int per = (n + 1 + T - 1) / T, b0 = min(tid * per, n + 1), b1 = min(b0 + per, n + 1);
  int s[3] = {0, 0, 0};
  for (int b = b0; b < b1; ++b) {
    int c = 0;
    for (int k = 0; k < waves; ++k) c += cnt[k * (n + 1) + b];
    s[0] += c, s[1] += (c + TILE - 1) / TILE, s[2] += c > 0;
  }
  int pre[3];
  for (int k = 0; k < 3; ++k) {
    int v = s[k];
    for (int o = 1; o < 64; o <<= 1) {
      const int u = __shfl_up(v, o, 64);
      if (lane >= o) v += u;
    }
    pre[k] = v - s[k];
    if (lane == 63) wsum[k][w] = v;
  }
  __syncthreads();
  for (int k = 0; k < 3; ++k)
    for (int j = 0; j < w; ++j) pre[k] += wsum[k][j];
  int total = 0;
  for (int j = 0; j < nw; ++j) total += wsum[1][j];
  for (int b = b0; b < b1; ++b) {
    seg[b] = pre[0];
    tstart[b] = ts[b] = pre[1];
    int c = 0;
    for (int k = 0; k < waves; ++k) {
      int32_t& v = cnt[k * (n + 1) + b];
      const int t = v;
      v = pre[0] + c;                        // this wave's first place in the bin
      c += t;
    }
    // the bin's first tile here, the others below
    if (c) tiles[pre[1]] = {b, pre[0], min(c, TILE), pre[2]};
    pre[0] += c, pre[1] += (c + TILE - 1) / TILE, pre[2] += c > 0;
  }
  if (tid == 0) seg[n + 1] = (int32_t)N, tstart[n + 1] = ts[n + 1] = total;
  __threadfence_block();
  __syncthreads();
  for (int t = tid; t < (int)max_tiles(N, n); t += T) {
    if (t >= total) {
      tiles[t] = {-1, 0, 0, 0};
      continue;
    }
    int lo = 0, hi = n;                      // the last bin that begins at or before t and is not empty
    while (lo < hi) {
      const int m = (lo + hi + 1) >> 1;
      if (ts[m] <= t) lo = m;
      else hi = m - 1;
    }
    if (t == ts[lo]) continue;
    const Tile f = tiles[ts[lo]];
    const int first = f.first + TILE * (t - ts[lo]);
    tiles[t] = {lo, first, min(TILE, seg[lo + 1] - first), f.ord};
  }
  if (w >= waves) return;
  for (int64_t t0 = r0; t0 < r1; t0 += 64 * AHEAD) {
    int bins[AHEAD];
    if (t0 > r0) load(t0, bins);
    else
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) bins[k] = kept[k];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int b = bins[j];
      const bool there = b >= 0;
      if (!__ballot(there)) break;
      const uint64_t same = alike(b);
      const int before = __popcll(same & (((uint64_t)1 << lane) - 1));
      const int at = there ? cnt[w * (n + 1) + b] : 0;
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");     // the wave has read before its leaders write
      __builtin_amdgcn_wave_barrier();
      if (there && before == 0) cnt[w * (n + 1) + b] = at + __popcll(same);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      if (there) perm[at + before] = (int32_t)(t0 + 64 * j + lane);
    }
  }
}

// ------------------------------------------------------------------ values
template <bool H>
__device__ __forceinline__ f32x4 mfma16(const u32x4& a, const u32x4& b, const f32x4& c) {
  if constexpr (H) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  else return mfma_bf16(a, b, c);
}
template <bool H> __device__ __forceinline__ float half_lo(uint32_t w) {
  if constexpr (H) return (float)__builtin_bit_cast(f16x2_t, w)[0];
  else return bf_lo(w);
}
template <bool H> __device__ __forceinline__ float half_hi(uint32_t w) {
  if constexpr (H) return (float)__builtin_bit_cast(f16x2_t, w)[1];
  else return bf_hi(w);
}
template <bool H> __device__ __forceinline__ uint32_t pack2h(float lo, float hi) {
  if constexpr (H) {
    const f16x2_t v = {(_Float16)lo, (_Float16)hi};
    return __builtin_bit_cast(uint32_t, v);
  } else {
    return pack2_bf16(lo, hi);
  }
}

// v = its upper 16 bits + a rest, whose upper 16 bits and what is left of it are bf16 again, exactly.  Where nothing is left (of
// an Inf too) the part is 2^-60 of the whole, which no fp32 sum beside the whole sees: a part of 0 times an Inf would be NaN
// where the whole times the Inf is one (from |v| = 2^-73 on; parts of smaller values end as 0).  All parts have the whole's
// sign, a NaN's are NaN.
__device__ __forceinline__ float upper(float v) { return __uint_as_float(__float_as_uint(v) & 0xffff0000u); }
__device__ __forceinline__ float faint(float v) { return v * 0x1p-60f; }
__device__ __forceinline__ float rest(float v, float whole) {
  const float r = v - upper(v);
  return fabsf(r) > 0.0f ? r : faint(whole);
}
__device__ __forceinline__ uint32_t upper2(float lo, float hi) {
  return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
}
// eight fp16 values as two bf16 each, exactly
__device__ __forceinline__ void split_f16(const u32x4& v, u32x4& hi, u32x4& lo) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float a = half_lo<true>(v[k]), b = half_hi<true>(v[k]);
    hi[k] = upper2(a, b);
    lo[k] = upper2(rest(a, a), rest(b, b));
  }
}

// ------------------------------------------------------------------ shrink
// part[share][tile][slot][rank] = sum over a share of K of W[a][rank][k] x[token][k], W [n, r, K].  Memory-bound: x once
// (long prompts: 134 MB of 16384 x 4096 in 28 us) or W once (a token an adapter).  A workgroup takes a tile and a share of
// K, its waves 64 K at a time in turn (a line of each row); a lane's operands are 16 bytes of a row, from memory to the
// matrix instruction.  A tile's shares lie in consecutive workgroups, so that all of a row is in work at a time (16384 x 1024:
// 15.5 -> 13.3 us).
struct Shrink {
  const uint16_t *x, *w;
  int64_t ldx, N, tiles;
  int n, r, K, shares, rs;      // rs: ranks rounded up to 4
  const int32_t* plan;
  float* part;
};

template <bool H, int RT>
__global__ __launch_bounds__(256) void shrink_kernel(Shrink p) {
  extern __shared__ f32x4 red[];              // [wave][RT * 4][64]
  const Plan plan = plan_view(p.plan, p.N, p.n);
  const unsigned tile = blockIdx.x / p.shares, share = blockIdx.x - tile * p.shares;
  const Tile t = tile_at(plan, tile, p.N, p.n);
  if ((unsigned)t.adapter >= (unsigned)p.n) return;
  const int lane = threadIdx.x & 63, w = uniform(threadIdx.x >> 6), i = lane & 15, q = lane >> 4;
  const int subs = (t.count + 15) >> 4, r0 = blockIdx.y * 64;
  const uint16_t* xr[4];
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    xr[s] = p.x + row_at(plan, t.first + min(16 * s + i, t.count - 1), p.N) * p.ldx + 8 * q;
  }
  const uint16_t* wr[RT];
#pragma unroll
  for (int k = 0; k < RT; ++k) wr[k] = p.w + ((int64_t)t.adapter * p.r + min(r0 + 16 * k + i, p.r - 1)) * p.K + 8 * q;
  const int units = (p.K + 63) / 64, u0 = (int)((int64_t)units * share / p.shares), u1 = (int)((int64_t)units * (share + 1) / p.shares);
  f32x4 acc[RT][4] = {};
  const u32x4 none = {0, 0, 0, 0};
  struct Unit {
    u32x4 x[2][4], w[2][RT];
  };
  auto fetch = [&](int u, Unit& v) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = 64 * u + 32 * h;
      const bool in = k + 8 * q < p.K;
#pragma unroll
      for (int j = 0; j < RT; ++j) v.w[h][j] = in ? *reinterpret_cast<const u32x4*>(wr[j] + k) : none;
#pragma unroll
      for (int s = 0; s < 4; ++s)
        if (s < subs) v.x[h][s] = in ? *reinterpret_cast<const u32x4*>(xr[s] + k) : none;
    }
  };
  // two units' operands in two sets of registers: a set is loaded again as soon as it is used up
  auto turn = [&](int u, Unit& v) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int s = 0; s < 4; ++s)
        if (s < subs)
#pragma unroll
          for (int j = 0; j < RT; ++j) acc[j][s] = mfma16<H>(v.w[h][j], v.x[h][s], acc[j][s]);
    if (u + 8 < u1) fetch(u + 8, v);
  };
  Unit v0, v1;
  if (u0 + w < u1) fetch(u0 + w, v0);
  if (u0 + w + 4 < u1) fetch(u0 + w + 4, v1);
  for (int u = u0 + w; u < u1; u += 8) {
    turn(u, v0);
    if (u + 4 < u1) turn(u + 4, v1);
  }
#pragma unroll
  for (int j = 0; j < RT; ++j)
#pragma unroll
    for (int s = 0; s < 4; ++s)
      if (s < subs) red[(w * RT * 4 + j * 4 + s) * 64 + lane] = acc[j][s];
  __syncthreads();
  // entry (j, s) of a lane (i, q): token 16 s + i, ranks 16 j + 4 q .. + 3
  for (int e = w; e < RT * 4; e += 4) {
    const int j = e >> 2, s = e & 3, slot = 16 * s + i, rank = r0 + 16 * j + 4 * q;
    if (slot >= t.count || rank >= p.rs) continue;
    f32x4 v = red[e * 64 + lane];
#pragma unroll
    for (int k = 1; k < 4; ++k) v += red[(k * RT * 4 + e) * 64 + lane];
    *reinterpret_cast<f32x4*>(p.part + (((int64_t)share * p.tiles + tile) * TILE + slot) * p.rs + rank) = v;
  }
}

// ------------------------------------------------------------------ expand
// out[token][f] = y[token][f] + sum over ranks of W[a][f][rank] t'[token][rank], W [n, F, r] with rows of ldw.
// Memory-bound by y and out (16384 tokens, 1024 / 4096, rank 16: 268 MB in 53 us), or by W (64 tokens, an adapter each,
// 4096 / 14336: 27 MB in 10 us).  A workgroup takes a tile and a share of F: it adds up t's shares, splits t' into LDS in
// the order of the matrix instruction's operand (`planes`: and for grad, ranks first), and its waves share the features.
// The 32 features of two products are dealt so that a lane ends with 8 consecutive ones of a token.
struct Expand {
  const uint16_t *w, *y;        // y NULL: out is the product alone
  uint16_t* out;
  int64_t ldy, ldo, N, tiles;
  int n, r, F, ldw, shares, chunks, rs;
  bool few;
  const int32_t* plan;
  const float *part, *scales;
  uint16_t* planes;             // [tile][three parts][ranks to 16][64 slots], or NULL
};

// the operand of a lane: ranks k .. k + 7 of a row, those from r on zero.  RV: ranks that lie aligned together
template <int RV>
__device__ __forceinline__ u32x4 rank8(const uint16_t* row, int k, int r) {
  if constexpr (RV == 8) {
    return k < r ? *reinterpret_cast<const u32x4*>(row + k) : u32x4{0, 0, 0, 0};
  } else if constexpr (RV == 4) {
    const u32x2 z = {0, 0}, a = k < r ? *reinterpret_cast<const u32x2*>(row + k) : z, b = k + 4 < r ? *reinterpret_cast<const u32x2*>(row + k + 4) : z;
    return u32x4{a[0], a[1], b[0], b[1]};
  } else {
    uint32_t e[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) e[j] = row[min(k + j, r - 1)];
    u32x4 v;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = (k + 2 * j < r ? e[2 * j] : 0u) | (k + 2 * j + 1 < r ? e[2 * j + 1] << 16 : 0u);
    return v;
  }
}

// Ranks up to 16 take two matrix instructions, two parts of t' side by side in the first's K and the third in the second's;
// more go 32 at a time, the parts one after the other.
enum { R16, R32, R64, RMORE };
// places of a step's second and third parts behind its first
template <int RK> constexpr int second = RK == R16 ? 32 : 256;
template <int RK> constexpr int third = RK == R16 ? 256 : 512;

// over lanes l, l + 16, l + 32 and l + 48
__device__ __forceinline__ float rows_sum(float x) {
  auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(s[0]) + __uint_as_float(s[1]);
  s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}

// t' of a tile, its shares summed and scaled, split into LDS: [step of 32 ranks][part][subtile][lane] (R16: [two parts, the
// third][subtile][lane]); slots without a token hold anything, as they stay in their columns of the products.  A thread has 4 ranks of a
// token, the threads beside it the next ones (a token's 8 ranks each were 32 bytes of every row at a time: expand of 4099
// tokens, 2048 / 8192, rank 64 43.9 -> 42.9 us).  FEW: lanes 16 apart take every fourth share each.
template <int RK, bool FEW>
__device__ __forceinline__ void split_t(const Expand& p, const Tile& t, unsigned tile, u32x4* tf) {
  constexpr int QB = RK == R16 ? 2 : 3;      // fours of a step's ranks: 4 (two halves of a K), 8
  const int lane = threadIdx.x & 63, w = uniform(threadIdx.x >> 6);
  const float scale = p.scales ? p.scales[t.adapter] : 1.0f;
  const int64_t share = p.tiles * TILE * p.rs;
  const int items = (RK == R16 ? 1 : (p.r + 31) / 32) * 4 << (QB + 4);
  u32x2* out = reinterpret_cast<u32x2*>(tf);
  constexpr int AT = FEW ? 2 : 4, BY = FEW ? 4 : 1, PASS = FEW ? 64 : 256;
#pragma unroll 2
  for (int k0 = 0; k0 < items; k0 += PASS) {
    const int item = k0 + (FEW ? 16 * w + (lane & 15) : (int)threadIdx.x);
    const int four = item & ((1 << QB) - 1), l = item >> QB & 15, s = item >> (QB + 4) & 3, step = item >> (QB + 6);
    const int slot = 16 * s + l, rank = 32 * step + 4 * four;
    f32x4 f = {0, 0, 0, 0};
    if (slot < t.count && rank < p.r) {
      const float* at = p.part + ((int64_t)tile * TILE + slot) * p.rs + rank;
      for (int k = FEW ? lane >> 4 : 0; k < p.shares; k += AT * BY) {       // the last shares are read again for nothing
        f32x4 v[AT];
#pragma unroll
        for (int j = 0; j < AT; ++j) v[j] = *reinterpret_cast<const f32x4*>(at + min(k + j * BY, p.shares - 1) * share);
#pragma unroll
        for (int j = 0; j < AT; ++j)
          if (k + j * BY < p.shares) f += v[j];
      }
    }
    if (16 * s >= t.count) continue;         // the same for all lanes of a wave
    float r[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (FEW) f[e] = rows_sum(f[e]);
      f[e] = rank + e < p.r ? f[e] * scale : 0.0f;
      r[e] = rest(f[e], f[e]);
    }
    if (FEW && lane >= 16) continue;
    const int at = RK == R16 ? s * 64 + 16 * (four >> 1) + l : (step * 12 + s) * 64 + 16 * (four >> 1) + l;
    u32x2* const to = out + 2 * at + (four & 1);
    to[0] = u32x2{upper2(f[0], f[1]), upper2(f[2], f[3])};
    to[2 * second<RK>] = u32x2{upper2(r[0], r[1]), upper2(r[2], r[3])};
    to[2 * third<RK>] = u32x2{upper2(rest(r[0], f[0]), rest(r[1], f[1])), upper2(rest(r[2], f[2]), rest(r[3], f[3]))};
    if constexpr (RK == R16) to[2 * (third<RK> + 32)] = u32x2{upper2(faint(f[0]), faint(f[1])), upper2(faint(f[2]), faint(f[3]))};
  }
}

// t' from LDS for grad: ranks first, slots without a token zero
template <int RK>
__device__ __forceinline__ void put_planes(const Expand& p, const Tile& t, unsigned tile, const u32x4* tf) {
  const int slot = threadIdx.x & 63, w = uniform(threadIdx.x >> 6), s = slot >> 4, l = slot & 15, r16 = (p.r + 15) & ~15;
  const u32x4 none = {0, 0, 0, 0};
  for (int g = w; 8 * g < r16; g += 4) {
    const int at = RK == R16 ? s * 64 + 16 * g + l : ((g >> 2) * 12 + s) * 64 + 16 * (g & 3) + l;
    const u32x4 part[3] = {slot < t.count ? tf[at] : none, slot < t.count ? tf[at + second<RK>] : none, slot < t.count ? tf[at + third<RK>] : none};
    uint16_t* pl = p.planes + ((int64_t)tile * 3 * r16 + 8 * g) * TILE + slot;
#pragma unroll
    for (int k = 0; k < 3; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) pl[(k * r16 + e) * TILE] = (uint16_t)(part[k][e >> 1] >> (16 * (e & 1)));
  }
}

// t' of a subtile and step as the matrix instructions take it (R16: two of them)
template <int RK> struct Parts { u32x4 v[RK == R16 ? 2 : 3]; };
template <int RK>
__device__ __forceinline__ Parts<RK> parts_of(const u32x4* tf, int step, int sub, int lane) {
  const u32x4* at = tf + (step * 12 + sub) * 64 + lane;
  if constexpr (RK == R16) return {{at[0], at[third<RK>]}};
  else return {{at[0], at[second<RK>], at[third<RK>]}};
}

// 32 features of 16 tokens, ranks of one step: the product added to acc[0 .. 1]
template <bool H, int RK>
__device__ __forceinline__ void add_step(const u32x4 (&w)[2], const Parts<RK>& t, f32x4 (&acc)[2]) {
  constexpr int P = RK == R16 ? 2 : 3;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    u32x4 wv = w[j], wl;
    if constexpr (H) split_f16(w[j], wv, wl);
#pragma unroll
    for (int k = 0; k < P; ++k) acc[j] = mfma_bf16(wv, t.v[k], acc[j]);
    if constexpr (H) {
#pragma unroll
      for (int k = 0; k + 1 < P; ++k) acc[j] = mfma_bf16(wl, t.v[k], acc[j]);
    }
  }
}
template <bool H>
__device__ __forceinline__ u32x4 plus(const u32x4& y, const f32x4 (&acc)[2]) {
  u32x4 o;
#pragma unroll
  for (int c = 0; c < 4; ++c)
    o[c] = pack2h<H>(half_lo<H>(y[c]) + acc[c >> 1][2 * (c & 1)], half_hi<H>(y[c]) + acc[c >> 1][2 * (c & 1) + 1]);
  return o;
}
// the row of W that row i of the j-th matrix instruction of 32 features takes: two of them leave a lane 8 consecutive ones
__device__ __forceinline__ int feature(int i, int j) { return 8 * (i >> 2) + 4 * j + (i & 3); }

// Tiles that mostly have up to 16 tokens: bound by W, of which a wave has 64 features in work and 64 in flight, from memory
// to the matrix instruction; further subtiles one after the other
template <bool H, int RV, int RK>
__device__ __forceinline__ void expand_few(const Expand& p, const Plan& plan, const Tile& t, unsigned tile, unsigned chunk, u32x4* tf) {
  constexpr bool ONE = RK == R16;
  constexpr int STEPS = RK == R64 ? 2 : 1;   // of 32 ranks, loaded ahead (RMORE: none)
  const bool bare = t.adapter == p.n;        // tokens without an adapter
  const int lane = threadIdx.x & 63, w = uniform(threadIdx.x >> 6), i = lane & 15, q = lane >> 4;
  const int units = (p.F + 63) / 64, u0 = (int)((int64_t)units * chunk / p.chunks) + w, u1 = (int)((int64_t)units * (chunk + 1) / p.chunks);
  const uint16_t* wa = p.w + (int64_t)t.adapter * p.F * p.ldw;
  auto weights = [&](int f0, int step, u32x4 (&v)[2]) {
#pragma unroll
    for (int j = 0; j < 2; ++j) v[j] = rank8<RV>(wa + (int64_t)min(f0 + feature(i, j), p.F - 1) * p.ldw, ONE ? 8 * (q & 1) : 32 * step + 8 * q, p.r);
  };
  struct Unit {
    u32x4 y[2], w[2][STEPS][2];
  };
  int64_t row = 0;
  auto fetch_w = [&](int u, Unit& g) {
    if (bare || RK == RMORE) return;
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int st = 0; st < STEPS; ++st) weights(64 * u + 32 * e, st, g.w[e][st]);
  };
  auto fetch_y = [&](int u, Unit& g) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int fl = 64 * u + 32 * e + 8 * q;
      g.y[e] = p.y && fl < p.F ? *reinterpret_cast<const u32x4*>(p.y + row * p.ldy + fl) : u32x4{0, 0, 0, 0};
    }
  };
  Unit v0, v1;                               // a set is loaded again as soon as it is used up
  if (u0 < u1) fetch_w(u0, v0);              // they need no more than the tile
  if (u0 + 4 < u1) fetch_w(u0 + 4, v1);
  row = row_at(plan, t.first + min(i, t.count - 1), p.N);
  if (u0 < u1) fetch_y(u0, v0);
  if (u0 + 4 < u1) fetch_y(u0 + 4, v1);
  if (!bare) {
    split_t<RK, true>(p, t, tile, tf);
    __syncthreads();
    if (p.planes && chunk == 0) put_planes<RK>(p, t, tile, tf);
  }
  int sub = 0;
  Parts<RK> t16;
  auto turn = [&](int u, Unit& v) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      f32x4 acc[2] = {};
      if (!bare) {
        if constexpr (ONE) {
          add_step<H, RK>(v.w[e][0], t16, acc);
        } else if constexpr (RK == RMORE) {
          for (int st = 0; st < (p.r + 31) / 32; ++st) {
            u32x4 w2[2];
            weights(64 * u + 32 * e, st, w2);
            add_step<H, RK>(w2, parts_of<RK>(tf, st, sub, lane), acc);
          }
        } else {
#pragma unroll
          for (int st = 0; st < STEPS; ++st) add_step<H, RK>(v.w[e][st], parts_of<RK>(tf, st, sub, lane), acc);
        }
      }
      const int fl = 64 * u + 32 * e + 8 * q;
      if (16 * sub + i < t.count && fl < p.F) *reinterpret_cast<u32x4*>(p.out + row * p.ldo + fl) = bare ? v.y[e] : plus<H>(v.y[e], acc);
    }
    if (u + 8 < u1) fetch_w(u + 8, v), fetch_y(u + 8, v);
  };
  for (;;) {
    if (ONE && !bare) t16 = parts_of<RK>(tf, 0, sub, lane);
    for (int u = u0; u < u1; u += 8) {
      turn(u, v0);
      if (u + 4 < u1) turn(u + 4, v1);
    }
    if (16 * ++sub >= t.count) return;
    row = row_at(plan, t.first + min(16 * sub + i, t.count - 1), p.N);
    if (u0 < u1) fetch_w(u0, v0), fetch_y(u0, v0);
    if (u0 + 4 < u1) fetch_w(u0 + 4, v1), fetch_y(u0 + 4, v1);
  }
}

// A lane has 8 features of its token in each of two groups of 32 (x, y): lanes of the upper eight tokens of 16 give theirs
// of the first group for the lower eight's of the second.  Then x holds whole 128-byte lines of the lower tokens' rows
// across the wave, y of the upper ones', where x and y before held halves of 16 rows' lines; the same again undoes it.
__device__ __forceinline__ void trade(u32x4& x, u32x4& y, bool upper) {
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const uint32_t give = upper ? x[c] : y[c];
    const uint32_t got = __builtin_amdgcn_update_dpp(0, give, 0x128, 0xf, 0xf, true);      // from the lane 8 on in its 16
    x[c] = upper ? got : x[c];
    y[c] = upper ? y[c] : got;
  }
}

// Larger tiles: bound by y and out.  A wave takes 128 features, whose part of W it holds in registers for all subtiles, one
// subtile after the other: the four waves of a workgroup work on 1 KB of 16 rows at a time.  What counts is how much of a
// row is in work together: 16384 tokens, 1024 / 4096, rank 16, took 85 us with 64 bytes of 64 rows a wave, 62 with 256 bytes
// of 16 rows and a subtile a wave, 59 with W through LDS and whole lines a load, 55 so, and 53 with loads that no path leaves out; rank 64
// (4099 tokens, 2048 / 8192) 64, 81, 50 and 42, rank 16 there 42 and 35 (with loads left out for subtiles that are not there).
template <bool H, int RV, int RK, bool Y>
__device__ __forceinline__ void expand_many(const Expand& p, const Plan& plan, const Tile& t, unsigned tile, unsigned chunk, u32x4* tf) {
  constexpr bool ONE = RK == R16;
  constexpr int STEPS = RK == R64 || RK == RMORE ? 2 : 1;      // of 32 ranks, held at a time
  // Loads end in their order, and one that some path leaves out counts as ended, so that the others are waited for with
  // those behind them.  Up to 32 ranks, all loads are made and all four subtiles taken, whether there or not.  More ranks leave
  // too few registers for that, and there a subtile that is not there costs more.
  constexpr bool ALL = STEPS == 1;
  const int lane = threadIdx.x & 63, w = uniform(threadIdx.x >> 6), i = lane & 15, q = lane >> 4;
  const int subs = (t.count + 15) >> 4;
  const int units = (p.F + 127) / 128, u0 = (int)((int64_t)units * chunk / p.chunks) + w, u1 = (int)((int64_t)units * (chunk + 1) / p.chunks);
  const uint16_t* wa = p.w + (int64_t)t.adapter * p.F * p.ldw;
  u32x4 wv[4][STEPS][2];
  auto fetch_w = [&](int u, int rb) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int st = 0; st < STEPS; ++st)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          wv[e][st][j] = rank8<RV>(wa + (int64_t)min(128 * u + 32 * e + feature(i, j), p.F - 1) * p.ldw, ONE ? 8 * (q & 1) : 64 * rb + 32 * st + 8 * q, p.r);
  };
  if (RK != RMORE && u0 < u1) fetch_w(u0, 0);                  // it needs no more than the tile
  // y and out by whole lines: of tokens i % 8 and 8 + i % 8 of a subtile, features 64 g + 32 (i / 8) + 8 q on
  const bool upper = i >= 8;
  int32_t row[4][2];
#pragma unroll
  for (int s = 0; s < 4; ++s)
#pragma unroll
    for (int e = 0; e < 2; ++e) row[s][e] = (int32_t)row_at(plan, t.first + min(16 * s + 8 * e + (i & 7), t.count - 1), p.N);
  auto column = [&](int u, int g) { return 128 * u + 64 * g + 32 * (i >> 3) + 8 * q; };
  auto fetch_y = [&](int u, int s, u32x4 (&y)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int fl = column(u, e >> 1);
      if (Y && (ALL || (s < subs && fl < p.F))) y[e] = *reinterpret_cast<const u32x4*>(p.y + row[s][e & 1] * p.ldy + min(fl, p.F - 8));
      else y[e] = u32x4{0, 0, 0, 0};
    }
  };
  u32x4 y0[4], y1[4];                                          // subtiles in turn, loaded again as soon as they are used up
  if (u0 < u1) fetch_y(u0, 0, y0), fetch_y(u0, 1, y1);
  split_t<RK, false>(p, t, tile, tf);
  __syncthreads();
  if (p.planes && chunk == 0) put_planes<RK>(p, t, tile, tf);
  auto turn = [&](int u, int s, u32x4 (&y)[4]) {
    const bool here = ALL || s < subs, more = ALL || u + 4 < u1;
    const int next = ALL ? min(u + 4, units - 1) : u + 4;
    f32x4 acc[4][2] = {};
    if (here) {
      const int blocks = RK == RMORE ? (p.r + 63) / 64 : 1;
      for (int rb = 0; rb < blocks; ++rb) {
        if (RK == RMORE) fetch_w(u, rb);
#pragma unroll
        for (int st = 0; st < STEPS; ++st) {
          const int step = 2 * rb + st;
          if (RK == RMORE && 32 * step >= p.r) break;
          const Parts<RK> parts = parts_of<RK>(tf, step, s, lane);
#pragma unroll
          for (int e = 0; e < 4; ++e) add_step<H, RK>(wv[e][st], parts, acc[e]);
        }
      }
    }
    // ahead of the stores: they would have to end before it is there (rank 64: 43.3 -> 42.1 us)
    if (s == 3 && more && RK != RMORE) fetch_w(next, 0);
    u32x4 o[4] = {y[0], y[1], y[2], y[3]};
    if (here)
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        trade(o[2 * g], o[2 * g + 1], upper);
        o[2 * g] = plus<H>(o[2 * g], acc[2 * g]);
        o[2 * g + 1] = plus<H>(o[2 * g + 1], acc[2 * g + 1]);
        trade(o[2 * g], o[2 * g + 1], upper);
      }
    if (ALL) fetch_y(s < 2 ? u : next, s ^ 2, y);
    if (here)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int fl = column(u, e >> 1);
        if (16 * s + 8 * (e & 1) + (i & 7) < t.count && fl < p.F) *reinterpret_cast<u32x4*>(p.out + row[s][e & 1] * p.ldo + fl) = o[e];
      }
    if (!ALL && (s < 2 || more)) fetch_y(s < 2 ? u : next, s ^ 2, y);
  };
  for (int u = u0; u < u1; u += 4) {
    turn(u, 0, y0);
    turn(u, 1, y1);
    turn(u, 2, y0);
    turn(u, 3, y1);
  }
}

// Tokens without an adapter: out = y (or zero)
__device__ __forceinline__ void copy_rows(const Expand& p, const Plan& plan, const Tile& t, unsigned chunk) {
  const int lane = threadIdx.x & 63, w = uniform(threadIdx.x >> 6);
  const int units = (p.F + 511) / 512, u0 = (int)((int64_t)units * chunk / p.chunks), u1 = (int)((int64_t)units * (chunk + 1) / p.chunks);
  const int f0 = 512 * u0 + 8 * lane, f1 = min(512 * u1, p.F);
  for (int s = 4 * w; s < t.count; s += 16) {      // four rows in flight
    int64_t row[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) row[j] = row_at(plan, t.first + min(s + j, t.count - 1), p.N);
    for (int f = f0; f < f1; f += 512) {
      u32x4 v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = p.y ? *reinterpret_cast<const u32x4*>(p.y + row[j] * p.ldy + f) : u32x4{0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (s + j < t.count) *reinterpret_cast<u32x4*>(p.out + row[j] * p.ldo + f) = v[j];
    }
  }
}

// (registers for two waves a SIMD where tiles are large: held to three, the kernel is slower, 57 against 44 us at rank 64 and 63
// against 56 at rank 16, as more rows are open in memory at a time)
template <bool H, int RV, int RK, bool FEW>
__global__ __launch_bounds__(256, FEW || RK == R64 ? 1 : 2) void expand_kernel(Expand p) {
  extern __shared__ u32x4 tf[];
  const Plan plan = plan_view(p.plan, p.N, p.n);
  // a tile's shares of F in consecutive workgroups: at any time all of a row's stretch is in work, not one share of all
  // rows, whose stride would put it on part of the memory channels; and a power of two of them, so that an XCD meets
  // its own features of an adapter again and again
  const unsigned tile = blockIdx.x / p.chunks, chunk = blockIdx.x - tile * p.chunks;
  const Tile t = tile_at(plan, tile, p.N, p.n);
  if (t.adapter < 0) return;
  if (t.adapter == p.n && p.y == p.out) return;
  if constexpr (FEW) expand_few<H, RV, RK>(p, plan, t, tile, chunk, tf);
  else if (t.adapter == p.n) copy_rows(p, plan, t, chunk);
  else if (p.y) expand_many<H, RV, RK, true>(p, plan, t, tile, chunk, tf);
  else expand_many<H, RV, RK, false>(p, plan, t, tile, chunk, tf);
}

// ------------------------------------------------------------------ grad
// part[piece][rank][f] = sum over the tokens of a piece of P[token][rank] Q[token][f], P from planes, Q = x or dy.
// Memory-bound by Q (dA and dB of 16384 tokens, 1024 / 4096, rank 16: 168 MB in 34 us; 53 while three of four workgroups
// of the grid had nothing to do).  Registers are held to four waves a SIMD at ranks up to 16 (whole training step 159 us, at
// three 166) and two above 32 (rank 64: 275 us, at one 308), and left to the compiler between (rank 32: 194 us, held to
// three 200).  A workgroup takes `turn` tiles in a row, its waves 64 features each; a wave's 32 tokens
// lie in an LDS slice of its own and are read transposed.  Where the adapter changes on the way, a piece ends: piece number =
// tile / turn + the adapter's number among those with tokens, which grows with either.
struct Grad {
  const uint16_t* q[2];
  const uint16_t* planes[2];
  float* part[2];
  int64_t ldq[2], N, tiles;
  int F[2], turn[2];
  int64_t first;               // workgroups of dA, ahead of those of dB
  int n, r, rblocks;
  const int32_t* plan;
};

constexpr int QROW = 72;             // elements of a token's row in LDS: 64 and 16 bytes, which moves the rows over the banks

template <bool H, int RT>
__global__ __launch_bounds__(256, RT == 1 ? 4 : RT == 2 ? 1 : 2) void grad_kernel(Grad p) {
  __shared__ __attribute__((aligned(16))) uint16_t slices[4][(H ? 2 : 1) * 32 * QROW];
  const int z = blockIdx.x >= p.first, F = p.F[z], fb = (F + 255) / 256;
  const unsigned id = blockIdx.x - (z ? (unsigned)p.first : 0), run = id / fb;
  const int r0 = blockIdx.y * 64;
  const int lane = threadIdx.x & 63, w = uniform(threadIdx.x >> 6), i = lane & 15, q = lane >> 4;
  const int f0 = ((id - run * fb) * 4 + w) * 64, r16 = (p.r + 15) & ~15;
  const int64_t t0 = (int64_t)run * p.turn[z], t1 = min(t0 + p.turn[z], p.tiles);
  if (f0 >= F || t0 >= t1) return;
  const Plan plan = plan_view(p.plan, p.N, p.n);
  uint16_t* slice = slices[w];
  const int fl = f0 + 8 * (lane & 7);

  // The steps of 32 tokens.  Two of them have their rows and planes in registers, in sets that are loaded again as soon as
  // they are used up, and the places of the rows behind these are there already.
  struct Step {
    int64_t tile;
    Tile t;
    int half;
    bool ok;
  };
  auto open = [&](int64_t tile) {
    Step s;
    s.tile = tile, s.half = 0;
    s.ok = tile < t1;
    if (s.ok) {
      s.t = tile_at(plan, tile, p.N, p.n);
      s.ok = (unsigned)s.t.adapter < (unsigned)p.n;      // else tokens without an adapter, or no tile: nothing behind them
    }
    return s;
  };
  auto after = [&](const Step& s) {
    if (!s.ok) return s;
    if (32 * (s.half + 1) < s.t.count) {
      Step n = s;
      ++n.half;
      return n;
    }
    return open(s.tile + 1);
  };
  auto places = [&](const Step& s, int32_t (&row)[4]) {
    if (s.ok)
#pragma unroll
      for (int j = 0; j < 4; ++j) row[j] = plan.perm[s.t.first + min(32 * s.half + 8 * j + (lane >> 3), s.t.count - 1)];
  };
  struct Set {
    u32x4 v[4], a[RT][3];
  };
  auto rows = [&](const Step& s, const int32_t (&row)[4], Set& g) {
    if (s.ok)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool there = 32 * s.half + 8 * j + (lane >> 3) < s.t.count && fl < F;
        g.v[j] = there ? *reinterpret_cast<const u32x4*>(p.q[z] + (int64_t)min((uint32_t)row[j], (uint32_t)(p.N - 1)) * p.ldq[z] + fl)
                       : u32x4{0, 0, 0, 0};
      }
  };
  auto factors = [&](const Step& s, Set& g) {
    if (!s.ok) return;
    const uint16_t* pl = p.planes[z] + (s.tile * 3 * r16 + r0 + i) * TILE + 32 * s.half + 8 * q;
#pragma unroll
    for (int j = 0; j < RT; ++j)
#pragma unroll
      for (int h = 0; h < 3; ++h)
        g.a[j][h] = r0 + 16 * j < r16 ? *reinterpret_cast<const u32x4*>(pl + (16 * j + h * r16) * TILE) : u32x4{0, 0, 0, 0};
  };

  f32x4 acc[RT][4] = {};
  auto flush = [&](const Step& s) {
    const int ord = min((uint32_t)s.t.ord, (uint32_t)min(p.N, (int64_t)p.n) - 1);
    float* out = p.part[z] + (s.tile / p.turn[z] + ord) * p.r * F;
#pragma unroll
    for (int j = 0; j < RT; ++j)
#pragma unroll
      for (int ft = 0; ft < 4; ++ft) {
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const int rank = r0 + 16 * j + 4 * q + v, f = f0 + 16 * ft + i;
          if (rank < p.r && f < F) out[(int64_t)rank * F + f] = acc[j][ft][v];
        }
        acc[j][ft] = f32x4{0, 0, 0, 0};
      }
  };
  Step now = open(t0), next = after(now), third = after(next);
  int32_t row[4];
  Set g0, g1;
  places(now, row);
  rows(now, row, g0);
  factors(now, g0);
  places(next, row);
  rows(next, row, g1);
  factors(next, g1);
  places(third, row);
  auto turn = [&](Set& g) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint16_t* at = slice + (8 * j + (lane >> 3)) * QROW + 8 * (lane & 7);
      if constexpr (H) {
        u32x4 hi, lo;
        split_f16(g.v[j], hi, lo);
        *reinterpret_cast<u32x4*>(at) = hi;
        *reinterpret_cast<u32x4*>(at + 32 * QROW) = lo;
      } else {
        *reinterpret_cast<u32x4*>(at) = g.v[j];
      }
    }
    rows(third, row, g);
    const Step fourth = after(third);
    places(fourth, row);
#pragma unroll
    for (int ft = 0; ft < 4; ++ft) {
      const u32x4 b = tr_frag(slice, QROW, 0, 16 * ft, lane);
      u32x4 bl;
      if constexpr (H) bl = tr_frag(slice + 32 * QROW, QROW, 0, 16 * ft, lane);
#pragma unroll
      for (int j = 0; j < RT; ++j) {
#pragma unroll
        for (int h = 0; h < 3; ++h) acc[j][ft] = mfma_bf16(g.a[j][h], b, acc[j][ft]);
        if constexpr (H) acc[j][ft] = mfma_bf16(g.a[j][1], bl, mfma_bf16(g.a[j][0], bl, acc[j][ft]));
      }
    }
    factors(third, g);
    if (!next.ok || next.t.adapter != now.t.adapter) flush(now);
    now = next, next = third, third = fourth;
  };
  while (now.ok) {
    turn(g0);
    if (now.ok) turn(g1);
  }
}

// The pieces of every adapter in their order, rounded: dA [n, r, F] (z even), dB [n, F, r] (z odd); adapters without
// tokens get zeros.  A workgroup takes 64 features and 16 ranks, a thread 4 features of a rank, with eight pieces' loads in
// flight (one piece at a time: 91 us instead of 7 at 16384 tokens, 1024 / 4096, rank 16); dB turns through LDS.
struct GradSum {
  const float* part[2];
  uint16_t* out[2];
  int F[2], turn[2];
  int64_t N;
  int n, r, h;
  const int32_t* plan;
};

__global__ __launch_bounds__(256) void grad_sum_kernel(GradSum p) {
  __shared__ uint16_t s[64][18];
  const int z = blockIdx.z & 1, F = p.F[z], a = blockIdx.y, f0 = blockIdx.x * 64, r0 = (blockIdx.z >> 1) * 16;
  if (!p.out[z] || f0 >= F) return;
  const int k = threadIdx.x >> 4, rank = r0 + k, f = f0 + 4 * (threadIdx.x & 15);
  const Plan plan = plan_view(p.plan, p.N, p.n);
  const int tiles = (int)max_tiles(p.N, p.n), ta = max(plan.tstart[a], 0), tb = min(plan.tstart[a + 1], tiles);      // as tile_at
  f32x4 v = {0, 0, 0, 0};
  if (tb > ta && rank < p.r && f < F) {
    const int ord = min((uint32_t)plan.tiles[ta].ord, (uint32_t)min(p.N, (int64_t)p.n) - 1), s0 = ta / p.turn[z] + ord, pieces = (tb - 1) / p.turn[z] + ord - s0 + 1;
    const float* at = p.part[z] + ((int64_t)s0 * p.r + rank) * F + f;
    const int64_t piece = (int64_t)p.r * F;
    for (int j0 = 0; j0 < pieces; j0 += 8) {
      f32x4 u[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) u[j] = *reinterpret_cast<const f32x4*>(at + min(j0 + j, pieces - 1) * piece);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j0 + j < pieces) v += u[j];
    }
  }
  const uint32_t lo = p.h ? pack2h<true>(v[0], v[1]) : pack2h<false>(v[0], v[1]), hi = p.h ? pack2h<true>(v[2], v[3]) : pack2h<false>(v[2], v[3]);
  if (z == 0) {
    if (rank < p.r && f < F) *reinterpret_cast<u32x2*>(p.out[0] + ((int64_t)a * p.r + rank) * F + f) = u32x2{lo, hi};
    return;
  }
  const int c = 4 * (threadIdx.x & 15);
  s[c][k] = (uint16_t)lo, s[c + 1][k] = (uint16_t)(lo >> 16), s[c + 2][k] = (uint16_t)hi, s[c + 3][k] = (uint16_t)(hi >> 16);
  __syncthreads();
  const int ranks = min(16, p.r - r0);
  uint16_t* out = p.out[1] + ((int64_t)a * F + f0) * p.r + r0;
  for (int e = threadIdx.x; e < min(64, F - f0) * ranks; e += 256) out[(int64_t)(e / ranks) * p.r + e % ranks] = s[e / ranks][e % ranks];
}

// dst [n][cols][ld] = the transposes of src [n][rows][cols], rows to ld zero; two of them in one launch (z: 2 n).  A thread's
// 16 loads are all in flight before the first is used (4 adapters of rank 16, 1024 / 4096: 10 -> 4 us, which is latency).
struct Transpose {
  const uint16_t* src[2];
  uint16_t* dst[2];
  int rows[2], cols[2], ld[2], n;
};

__global__ __launch_bounds__(256) void transpose_kernel(Transpose p) {
  __shared__ uint16_t s[64][66];
  const int which = blockIdx.z >= p.n, rows = p.rows[which], cols = p.cols[which], ld = p.ld[which];
  const int64_t a = blockIdx.z - which * p.n;
  const int tc = (cols + 63) / 64, tr = (ld + 63) / 64;
  if ((int)blockIdx.x >= tc * tr) return;
  const int c0 = (blockIdx.x % tc) * 64, r0 = (blockIdx.x / tc) * 64, x = threadIdx.x & 63, y = threadIdx.x >> 6;
  const uint16_t* src = p.src[which];
  uint16_t* dst = p.dst[which];
  uint16_t v[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) v[k] = src[(a * rows + min(r0 + 4 * k + y, rows - 1)) * cols + min(c0 + x, cols - 1)];
#pragma unroll
  for (int k = 0; k < 16; ++k) s[4 * k + y][x] = r0 + 4 * k + y < rows && c0 + x < cols ? v[k] : (uint16_t)0;
  __syncthreads();
  for (int k = y; k < 64; k += 4)
    if (c0 + k < cols && r0 + x < ld) dst[(a * cols + c0 + k) * ld + r0 + x] = s[x][k];
}

// ------------------------------------------------------------------ launches
inline hipStream_t S(void* s) { return reinterpret_cast<hipStream_t>(s); }
inline int launched() { return hipGetLastError() == hipSuccess ? LBK_OK : LBK_ERR_LAUNCH; }
inline bool a16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }

// Whether tiles have few tokens: on average up to 16, were every adapter (and none) to occur.  64 tokens of 128 adapters,
// 4096 -> 14336, rank 16: expand 10 us this way, 15 the other; 16384 tokens of 4, 1024 -> 4096: 85 and 55.
bool few_of(int64_t N, int n) { return N <= 16 * (int64_t)(n + 1); }

// Shares of K of a shrink, up to four workgroups on a CU and at least 512 K each: every workgroup of expand adds a tile's shares
// up (dy of 16384 x 4096, 260 tiles: 2 shares 40 us and 12.8 in expand, 4 shares 35.5 and 13.7, 6 shares 36.7 and 15.1).
int shares_of(int64_t tiles, int K) {
  const int64_t s = (1024 + tiles - 1) / tiles, most = (K + 511) / 512;
  return (int)std::max<int64_t>(1, std::min(s, most));
}
// Shares of F of an expand: a power of two, up to about 1100 workgroups, a unit of features for every wave at least
int chunks_of(int64_t tiles, int F, bool few) {
  int64_t c = 1;
  while (2 * c * tiles <= 1100 && c < 64) c *= 2;
  const int unit = few ? 256 : 512;
  return (int)std::max<int64_t>(1, std::min<int64_t>(c, (F + unit - 1) / unit));
}
size_t part_bytes(int64_t tiles, int K, int r) { return align256((size_t)shares_of(tiles, K) * tiles * TILE * ((r + 3) & ~3) * 4); }
size_t plane_bytes(int64_t tiles, int r) { return align256((size_t)tiles * 3 * ((r + 15) & ~15) * TILE * 2); }

// tiles of a workgroup of grad, and its pieces
int turn_of(int64_t tiles, int F) {
  const int64_t fb = (F + 255) / 256;
  return (int)std::max<int64_t>(1, tiles * fb / 512);
}
int64_t pieces_of(int64_t tiles, int64_t N, int n, int turn) { return (tiles + turn - 1) / turn + std::min<int64_t>(N, n); }

int launch_shrink(bool h, const Shrink& p, hipStream_t st) {
  const int rb = (p.r + 63) / 64, rt = std::min((p.r + 15) / 16, 4);
  const dim3 grid((unsigned)(p.tiles * p.shares), rb);
  auto go = [&](auto* k, int RT) {
    k<<<grid, 256, RT * 16384, st>>>(p);
    return launched();
  };
  if (rt == 1) return h ? go(shrink_kernel<true, 1>, 1) : go(shrink_kernel<false, 1>, 1);
  if (rt == 2) return h ? go(shrink_kernel<true, 2>, 2) : go(shrink_kernel<false, 2>, 2);
  return h ? go(shrink_kernel<true, 4>, 4) : go(shrink_kernel<false, 4>, 4);
}

template <bool H, int RV, int RK, bool FEW>
int launch_expand_f(const Expand& p, hipStream_t st) {
  static std::atomic<uint64_t> limit{0};
  const int lds = (RK == R16 ? 512 : (p.r + 31) / 32 * 768) * 16;      // t': at most 96 KB
  const auto k = expand_kernel<H, RV, RK, FEW>;
  if (lds > 65536 && set_lds_limit_once(reinterpret_cast<const void*>(k), MAX_RANK / 32 * 768 * 16, limit)) return LBK_ERR_LAUNCH;
  k<<<(unsigned)(p.tiles * p.chunks), 256, lds, st>>>(p);
  return launched();
}
template <bool H, int RV, int RK>
int launch_expand_t(const Expand& p, hipStream_t st) {
  return p.few ? launch_expand_f<H, RV, RK, true>(p, st) : launch_expand_f<H, RV, RK, false>(p, st);
}
template <bool H>
int launch_expand_h(const Expand& p, hipStream_t st) {
  const int rv = p.ldw % 8 == 0 ? 8 : p.ldw % 4 == 0 ? 4 : 1;
  if (p.r <= 16) return rv == 8 ? launch_expand_t<H, 8, R16>(p, st) : rv == 4 ? launch_expand_t<H, 4, R16>(p, st) : launch_expand_t<H, 1, R16>(p, st);
  if (rv == 8 && p.r <= 32) return launch_expand_t<H, 8, R32>(p, st);
  if (rv == 8 && p.r <= 64) return launch_expand_t<H, 8, R64>(p, st);
  return rv == 8 ? launch_expand_t<H, 8, RMORE>(p, st) : rv == 4 ? launch_expand_t<H, 4, RMORE>(p, st) : launch_expand_t<H, 1, RMORE>(p, st);
}
int launch_expand(bool h, const Expand& p, hipStream_t st) { return h ? launch_expand_h<true>(p, st) : launch_expand_h<false>(p, st); }

int check_adapter(const lbk_adapter* d) {
  if (!d) return LBK_ERR_NULL;
  if ((d->type != LBK_BF16 && d->type != LBK_FP16) || d->N < 0) return LBK_ERR_ARG;
  if (d->n < 1 || d->rank < 1 || d->in_features < 8 || d->out_features < 8 || d->in_features % 8 || d->out_features % 8) return LBK_ERR_SHAPE;
  if (d->n > MAX_ADAPTERS || d->rank > MAX_RANK || d->N > (1 << 30) || d->in_features > (1 << 21) || d->out_features > (1 << 21))
    return LBK_ERR_TOO_LARGE;
  // a launch takes fewer than 2^32 threads; so many tiles are not split into shares
  if (max_tiles(d->N, d->n) > (int64_t)UINT32_MAX / 256) return LBK_ERR_TOO_LARGE;
  return LBK_OK;
}

}  // namespace
}  // namespace lbk

using namespace lbk;

extern "C" {

size_t lbk_adapter_plan_bytes(int64_t N, int32_t n_adapters) {
  if (N < 0 || N > (1 << 30) || n_adapters < 1 || n_adapters > MAX_ADAPTERS) return 0;
  return (size_t)plan_words(N, n_adapters) * 4;
}

int lbk_adapter_plan(const void* ids, int32_t id_bytes, int64_t N, int32_t n_adapters, void* plan, size_t plan_bytes, void* stream) {
  if ((id_bytes != 4 && id_bytes != 8) || N < 0) return LBK_ERR_ARG;
  if (n_adapters < 1) return LBK_ERR_SHAPE;
  if (N > (1 << 30) || n_adapters > MAX_ADAPTERS) return LBK_ERR_TOO_LARGE;
  if ((N > 0 && !ids) || !plan) return LBK_ERR_NULL;
  if (!a16(plan) || (reinterpret_cast<uintptr_t>(ids) & (id_bytes - 1))) return LBK_ERR_ALIGN;
  if (plan_bytes < lbk_adapter_plan_bytes(N, n_adapters)) return LBK_ERR_WORKSPACE;
  // waves that count: as many as have 64 tokens and as 44 KB of counters hold
  const int bins = n_adapters + 1;
  const int waves = (int)std::max<int64_t>(1, std::min<int64_t>({16, 11264 / bins, (N + 63) / 64}));
  const int lds = (waves * bins + bins + 1) * 4;
  const int threads = waves <= 4 && bins <= 1024 ? 256 : 1024;
  if (id_bytes == 4) plan_kernel<int32_t><<<1, threads, lds, S(stream)>>>(static_cast<const int32_t*>(ids), N, n_adapters, waves, static_cast<int32_t*>(plan));
  else plan_kernel<int64_t><<<1, threads, lds, S(stream)>>>(static_cast<const int64_t*>(ids), N, n_adapters, waves, static_cast<int32_t*>(plan));
  return launched();
}

size_t lbk_adapter_planes_bytes(const lbk_adapter* d) {
  return check_adapter(d) || d->N == 0 ? 0 : plane_bytes(max_tiles(d->N, d->n), d->rank);
}

size_t lbk_adapter_add_workspace_bytes(const lbk_adapter* d) {
  return check_adapter(d) || d->N == 0 ? 0 : part_bytes(max_tiles(d->N, d->n), d->in_features, d->rank);
}

int lbk_adapter_add(const lbk_adapter* d, const void* x, int64_t ldx, const void* y, int64_t ldy, void* out, int64_t ldo,
                    void* planes, void* workspace, size_t workspace_bytes, void* stream) {
  if (int st = check_adapter(d)) return st;
  if (ldx < d->in_features || ldy < d->out_features || ldo < d->out_features) return LBK_ERR_ARG;
  if (d->N == 0) return LBK_OK;
  if (!d->a || !d->b || !d->plan || !x || !y || !out) return LBK_ERR_NULL;
  for (const void* p : {d->a, d->b, (const void*)d->plan, x, y, (const void*)out, (const void*)planes, (const void*)workspace})
    if (!a16(p)) return LBK_ERR_ALIGN;
  if (ldx % 8 || ldy % 8 || ldo % 8 || (reinterpret_cast<uintptr_t>(d->scales) & 3)) return LBK_ERR_ALIGN;
  if (out == y && ldo != ldy && d->N > 1) return LBK_ERR_ARG;      // rows of out would lie over other rows of y
  if (!workspace || workspace_bytes < lbk_adapter_add_workspace_bytes(d)) return LBK_ERR_WORKSPACE;
  const bool h = d->type == LBK_FP16;
  const int64_t tiles = max_tiles(d->N, d->n);
  const int rs = (d->rank + 3) & ~3, shares = shares_of(tiles, d->in_features);
  const Shrink s{static_cast<const uint16_t*>(x), static_cast<const uint16_t*>(d->a), ldx, d->N, tiles, d->n, d->rank, d->in_features, shares, rs,
                 d->plan, static_cast<float*>(workspace)};
  if (int st = launch_shrink(h, s, S(stream))) return st;
  const Expand e{static_cast<const uint16_t*>(d->b), static_cast<const uint16_t*>(y), static_cast<uint16_t*>(out), ldy, ldo, d->N, tiles, d->n,
                 d->rank, d->out_features, d->rank, shares, chunks_of(tiles, d->out_features, few_of(d->N, d->n)), rs, few_of(d->N, d->n),
                 d->plan, static_cast<const float*>(workspace),
                 d->scales, static_cast<uint16_t*>(planes)};
  return launch_expand(h, e, S(stream));
}

// shares of dy's shrink, planes of dt', the transposes of B and A, the pieces of dA and dB: what the wanted gradients need
struct BwdParts {
  size_t part, planes, bt, at, pa, pb, all;
};
static BwdParts bwd_parts(const lbk_adapter* d, bool dx, bool da, bool db) {
  const int64_t tiles = max_tiles(d->N, d->n);
  BwdParts p{};
  if (dx || da) p.part = part_bytes(tiles, d->out_features, d->rank);
  if (dx || da) p.bt = align256((size_t)d->n * d->rank * d->out_features * 2);
  if (da) p.planes = plane_bytes(tiles, d->rank);
  if (dx) p.at = align256((size_t)d->n * ((d->rank + 7) & ~7) * d->in_features * 2);
  auto pieces = [&](int F) { return align256((size_t)pieces_of(tiles, d->N, d->n, turn_of(tiles, F)) * d->rank * F * 4); };
  if (da) p.pa = pieces(d->in_features);
  if (db) p.pb = pieces(d->out_features);
  p.all = p.part + p.planes + p.bt + p.at + p.pa + p.pb;
  return p;
}

size_t lbk_adapter_bwd_workspace_bytes_for(const lbk_adapter* d, int dx, int da, int db) {
  return check_adapter(d) || d->N == 0 ? 0 : bwd_parts(d, dx, da, db).all;
}
size_t lbk_adapter_bwd_workspace_bytes(const lbk_adapter* d) { return lbk_adapter_bwd_workspace_bytes_for(d, 1, 1, 1); }

int lbk_adapter_bwd(const lbk_adapter* d, const void* x, int64_t ldx, const void* dout, int64_t ldo, const void* planes, void* dx,
                    void* da, void* db, void* workspace, size_t workspace_bytes, void* stream) {
  if (int st = check_adapter(d)) return st;
  if (ldx < d->in_features || ldo < d->out_features) return LBK_ERR_ARG;
  if (!d->plan) return LBK_ERR_NULL;
  const bool some = d->N > 0;
  if (some && (!d->a || !d->b || !dout || (da && !x) || (db && !planes))) return LBK_ERR_NULL;
  for (const void* p : {d->a, d->b, (const void*)d->plan, x, dout, planes, (const void*)dx, (const void*)da, (const void*)db, (const void*)workspace})
    if (!a16(p)) return LBK_ERR_ALIGN;
  if (ldx % 8 || ldo % 8 || (reinterpret_cast<uintptr_t>(d->scales) & 3)) return LBK_ERR_ALIGN;
  BwdParts sz{};
  if (some) sz = bwd_parts(d, dx, da, db);
  if (sz.all && (!workspace || workspace_bytes < sz.all)) return LBK_ERR_WORKSPACE;
  const bool h = d->type == LBK_FP16;
  const int64_t tiles = max_tiles(d->N, d->n);
  const int in = d->in_features, out = d->out_features, r = d->rank, rs = (r + 3) & ~3, r8 = (r + 7) & ~7;
  hipStream_t st = S(stream);
  char* at = static_cast<char*>(workspace);
  auto take = [&](size_t b) {
    char* p = at;
    at += b;
    return p;
  };
  float* part = reinterpret_cast<float*>(take(sz.part));
  uint16_t* dplanes = reinterpret_cast<uint16_t*>(take(sz.planes));
  uint16_t* bt = reinterpret_cast<uint16_t*>(take(sz.bt));
  uint16_t* att = reinterpret_cast<uint16_t*>(take(sz.at));
  float* pa = reinterpret_cast<float*>(take(sz.pa));
  float* pb = reinterpret_cast<float*>(take(sz.pb));
  if (some && (dx || da)) {
    Transpose tp{};
    tp.src[0] = static_cast<const uint16_t*>(d->b), tp.dst[0] = bt, tp.rows[0] = out, tp.cols[0] = r, tp.ld[0] = out;
    tp.src[1] = static_cast<const uint16_t*>(d->a), tp.dst[1] = att, tp.rows[1] = r, tp.cols[1] = in, tp.ld[1] = r8, tp.n = d->n;
    const int most = std::max((out + 63) / 64, dx ? (in + 63) / 64 : 0) * ((r8 + 63) / 64);
    transpose_kernel<<<dim3(most, 1, dx ? 2 * d->n : d->n), 256, 0, st>>>(tp);
    if (int e = launched()) return e;
    const int shares = shares_of(tiles, out);
    const Shrink s{static_cast<const uint16_t*>(dout), bt, ldo, d->N, tiles, d->n, r, out, shares, rs, d->plan, part};
    if (int e = launch_shrink(h, s, st)) return e;
    const Expand e{att, nullptr, static_cast<uint16_t*>(dx), in, in, d->N, tiles, d->n, r, dx ? in : 0, r8, shares,
                   dx ? chunks_of(tiles, in, few_of(d->N, d->n)) : 1, rs, few_of(d->N, d->n), d->plan, part, d->scales, da ? dplanes : nullptr};
    if (int k = launch_expand(h, e, st)) return k;
  }
  if (!da && !db) return LBK_OK;
  Grad g{};
  g.q[0] = static_cast<const uint16_t*>(x), g.q[1] = static_cast<const uint16_t*>(dout);
  g.planes[0] = dplanes, g.planes[1] = static_cast<const uint16_t*>(planes);
  g.part[0] = pa, g.part[1] = pb, g.ldq[0] = ldx, g.ldq[1] = ldo;
  g.N = d->N, g.tiles = tiles, g.n = d->n, g.r = r, g.rblocks = (r + 63) / 64, g.plan = d->plan;
  g.F[0] = da ? in : 0, g.F[1] = db ? out : 0;
  g.turn[0] = some ? turn_of(tiles, in) : 1, g.turn[1] = some ? turn_of(tiles, out) : 1;
  if (some) {
    int64_t blocks[2];
    for (int z = 0; z < 2; ++z) blocks[z] = (int64_t)((g.F[z] + 255) / 256) * ((tiles + g.turn[z] - 1) / g.turn[z]);
    g.first = blocks[0];
    const dim3 grid((unsigned)(blocks[0] + blocks[1]), g.rblocks);
    const int rt = std::min((r + 15) / 16, 4);
    auto go = [&](auto* k) {
      k<<<grid, 256, 0, st>>>(g);
      return launched();
    };
    if (int e = rt == 1 ? (h ? go(grad_kernel<true, 1>) : go(grad_kernel<false, 1>))
                : rt == 2 ? (h ? go(grad_kernel<true, 2>) : go(grad_kernel<false, 2>))
                          : (h ? go(grad_kernel<true, 4>) : go(grad_kernel<false, 4>)))
      return e;
  }
  GradSum m{};
  m.part[0] = pa, m.part[1] = pb, m.out[0] = static_cast<uint16_t*>(da), m.out[1] = static_cast<uint16_t*>(db);
  m.F[0] = in, m.F[1] = out, m.turn[0] = g.turn[0], m.turn[1] = g.turn[1], m.N = d->N, m.n = d->n, m.r = r, m.h = h, m.plan = d->plan;
  const int most = (std::max(da ? in : 0, db ? out : 0) + 63) / 64;
  grad_sum_kernel<<<dim3(most, d->n, 2 * ((r + 15) / 16)), 256, 0, st>>>(m);
  return launched();
}

}  // extern "C"
