// lbk_seam.hip — dropout from a counter-based generator, and the seam between two applications of a block: the
// branch's norm, dropout, gate and scale, the residual sum and the norm ahead of the next application, with their
// backward (gfx950), and their entry points of include/lbk.h.
//
//   z  = y rs(y) w_post            rs(v) = 1 / sqrt(mean(v^2) + eps)
//   h' = h + alpha gate drop(z)
//   n  = h' rs(h') w_pre
//
// All arithmetic is fp32; h', n and the gradients are rounded once, to their own types.
#include "lbk.h"
#include "lbk_device.h"
#include "lbk_internal.h"

#include <math.h>

namespace lbk {
namespace {

typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
// rows of any length start at any element: 16-byte loads and stores that need no more than an element's alignment
typedef u32x4 u32x4_2 __attribute__((aligned(2)));
typedef f32x4 f32x4_4 __attribute__((aligned(4)));

// ------------------------------------------------------------------ the generator
// 16 bits for each of 8 consecutive columns of a row: Philox4x32 (Salmon, Moraes, Dror and Shaw, "Parallel random
// numbers: as easy as 1, 2, 3", 2011) with the 7 rounds that the paper finds free of statistical defects, key =
// seed, counter = (column / 8, row, stream).  A drop probability is then a multiple of 2^-16; words of 32 bits an
// element would take twice the generator's arithmetic, which at 14 wide multiplications a block is what bounds a
// dropout of 16-bit values next to memory.
struct Random {
  const int64_t* seed_dev;      // read by the kernel where it is given, so that a replayed graph follows it
  int64_t seed;
  uint32_t stream, cut;         // an element is dropped where its 16 bits are below cut
  float keep;                   // 65536 / (65536 - cut)
};

__device__ __forceinline__ u32x4 random8(uint64_t key, uint32_t group, uint64_t row, uint32_t stream) {
  uint32_t k0 = (uint32_t)key, k1 = (uint32_t)(key >> 32);
  uint32_t c0 = group, c1 = (uint32_t)row, c2 = (uint32_t)(row >> 32), c3 = stream;
#pragma unroll
  for (int r = 0; r < 7; ++r) {
    const uint64_t p0 = (uint64_t)c0 * 0xD2511F53u, p1 = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)p1;
    c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)p0;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return u32x4{c0, c1, c2, c3};
}

// A dropped element is 0 whatever it held.
__device__ __forceinline__ void drop8(float (&f)[8], const u32x4& w, uint32_t cut, float keep) {
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    const uint32_t u = (q & 1) ? w[q >> 1] >> 16 : w[q >> 1] & 0xffffu;
    f[q] = u >= cut ? f[q] * keep : 0.0f;
  }
}

// ------------------------------------------------------------------ eight consecutive elements, n of them there
template <int T> struct Elem { typedef uint16_t type; };
template <> struct Elem<LBK_FP32> { typedef float type; };

template <int T>
__device__ __forceinline__ float to_f(typename Elem<T>::type v) {
  if constexpr (T == LBK_FP32) return v;
  else if constexpr (T == LBK_BF16) return bf2f(v);
  else return (float)__builtin_bit_cast(_Float16, v);
}
template <int T>
__device__ __forceinline__ typename Elem<T>::type from_f(float f) {
  if constexpr (T == LBK_FP32) return f;
  else if constexpr (T == LBK_BF16) return f2bf(f);
  else return __builtin_bit_cast(uint16_t, (_Float16)f);
}

// A lane's 8 columns of a row of d, the last of them perhaps behind the row's end.  Such a lane loads the row's last 8
// and moves them to their places after the wait: with loads one by one under a condition the waves that hold a row's end
// wait for every array in turn (4097 x 1001, backward: 31.2 -> 28.1 us).
struct Cols {
  int col, n, from, shift;      // first column, columns there (< 8 or negative: the end), column loaded from, places to move by
  bool tail;                    // of any lane of the wave
  __device__ __forceinline__ Cols() {}
  __device__ __forceinline__ Cols(int c, int d) : col(c), n(d - c) {
    from = min(c, max(d - 8, 0));
    shift = d >= 8 && n > 0 && n < 8 ? 8 - n : 0;
    tail = __any(n < 8);
  }
};

// as loaded, so that a load can be in flight while something else is worked on
template <int T> struct Raw8 { u32x4 v[T == LBK_FP32 ? 2 : 1]; };

// SMALL: d may be less than 8 (one lane holds the row).  Off: of a column's offset in bytes.  Where all lanes share the base and
// rows are short, 32 bits make that one register of an address in a lane; a row of 2^30 fp32 columns or more needs 64.
template <int T, bool SMALL = false, class Off = uint32_t>
__device__ __forceinline__ void fetch8(const void* base, int64_t row, int d, const Cols& c, Raw8<T>& r) {
  const auto* p = static_cast<const typename Elem<T>::type*>(base) + row * d;
  if (!SMALL || d >= 8) {
    const auto* q = reinterpret_cast<const u32x4_2*>(reinterpret_cast<const char*>(p) + (Off)c.from * (Off)sizeof(*p));
    r.v[0] = q[0];
    if constexpr (T == LBK_FP32) r.v[1] = q[1];
    return;
  }
  uint32_t e[8];
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    if constexpr (T == LBK_FP32) e[q] = __float_as_uint(p[min(q, d - 1)]);
    else e[q] = p[min(q, d - 1)];
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    if constexpr (T == LBK_FP32) r.v[0][q] = e[q], r.v[1][q] = e[4 + q];
    else r.v[0][q] = e[2 * q] | e[2 * q + 1] << 16;
  }
}
template <int K>
__device__ __forceinline__ void move_down(float (&f)[8], int shift) {
  const uint32_t by = shift & K ? ~0u : 0u;
#pragma unroll
  for (int q = 0; q + K < 8; ++q) f[q] = __uint_as_float((__float_as_uint(f[q + K]) & by) | (__float_as_uint(f[q]) & ~by));
}
// ODD: a row's last columns may be fewer than 8; else a lane has all of its columns or none
template <int T, bool ODD = true>
__device__ __forceinline__ void unpack8(const Raw8<T>& r, const Cols& c, float (&f)[8]) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    if constexpr (T == LBK_FP32) f[q] = __uint_as_float(r.v[0][q]), f[4 + q] = __uint_as_float(r.v[1][q]);
    else f[2 * q] = to_f<T>((uint16_t)r.v[0][q]), f[2 * q + 1] = to_f<T>((uint16_t)(r.v[0][q] >> 16));
  }
  if (c.tail) {
    if constexpr (ODD) {
      move_down<4>(f, c.shift);
      move_down<2>(f, c.shift);
      move_down<1>(f, c.shift);
    }
#pragma unroll
    for (int q = 0; q < 8; ++q) f[q] = (ODD ? q < c.n : c.n > 0) ? f[q] : 0.0f;
  }
}
template <int T, bool ODD = true>
__device__ __forceinline__ void load8(const void* base, int64_t row, int d, const Cols& c, float (&f)[8]) {
  Raw8<T> r;
  fetch8<T>(base, row, d, c, r);
  unpack8<T, ODD>(r, c, f);
}

__device__ __forceinline__ uint32_t pack2_f16(float lo, float hi) {
  const f16x2_t v = {(_Float16)lo, (_Float16)hi};
  return __builtin_bit_cast(uint32_t, v);
}

template <int T, bool ODD = true, class Off = uint32_t>
__device__ __forceinline__ void store8(void* base, int64_t row, int d, const Cols& c, const float (&f)[8]) {
  auto* b = static_cast<typename Elem<T>::type*>(base) + row * d;
  auto* p = reinterpret_cast<decltype(b)>(reinterpret_cast<char*>(b) + (Off)c.col * (Off)sizeof(*b));
  if (c.n >= 8) {
    if constexpr (T == LBK_FP32) {
      *reinterpret_cast<f32x4_4*>(p) = f32x4{f[0], f[1], f[2], f[3]};
      *reinterpret_cast<f32x4_4*>(p + 4) = f32x4{f[4], f[5], f[6], f[7]};
    } else {
      u32x4 v;
#pragma unroll
      for (int q = 0; q < 4; ++q)
        v[q] = T == LBK_BF16 ? pack2_bf16(f[2 * q], f[2 * q + 1]) : pack2_f16(f[2 * q], f[2 * q + 1]);
      *reinterpret_cast<u32x4_2*>(p) = v;
    }
  } else if constexpr (ODD) {
#pragma unroll
    for (int q = 0; q < 7; ++q)
      if (q < c.n) p[q] = from_f<T>(f[q]);
  }
}

// of a type known at run time only (the gate's)
template <bool ODD>
__device__ __forceinline__ void load8_any(int type, const void* base, int64_t row, int d, const Cols& c, float (&f)[8]) {
  if (type == LBK_FP32) load8<LBK_FP32, ODD>(base, row, d, c, f);
  else if (type == LBK_BF16) load8<LBK_BF16, ODD>(base, row, d, c, f);
  else load8<LBK_FP16, ODD>(base, row, d, c, f);
}
template <bool ODD>
__device__ __forceinline__ void store8_any(int type, void* base, int64_t row, int d, const Cols& c, const float (&f)[8]) {
  if (type == LBK_FP32) store8<LBK_FP32, ODD>(base, row, d, c, f);
  else if (type == LBK_BF16) store8<LBK_BF16, ODD>(base, row, d, c, f);
  else store8<LBK_FP16, ODD>(base, row, d, c, f);
}

// ------------------------------------------------------------------ dropout
struct DropArgs {
  const void* x;
  void* y;
  int64_t N, ldx;
  int F, G;                     // G: groups of 8 columns in a row
  uint32_t magic, shift;        // n / G = n magic >> shift for n < 2^31
  Random r;
};

constexpr int DROP_GROUPS = 4;  // of a thread, all loaded ahead (16384 x 1024 bf16: 67 MB in 13 us)

template <int T, bool SMALL>
__global__ __launch_bounds__(256) void dropout_kernel(DropArgs a) {
  const uint64_t key = (uint64_t)(a.r.seed_dev ? *a.r.seed_dev : a.r.seed);
  const int64_t first = (int64_t)blockIdx.x * (256 * DROP_GROUPS), row0 = first / a.G;
  const uint32_t g0 = (uint32_t)(first - row0 * a.G) + threadIdx.x;
  Raw8<T> raw[DROP_GROUPS];
  Cols c[DROP_GROUPS];
  int64_t row[DROP_GROUPS];
#pragma unroll
  for (int k = 0; k < DROP_GROUPS; ++k) {
    const uint32_t off = g0 + 256 * k, dr = (uint32_t)((uint64_t)off * a.magic >> a.shift);
    row[k] = row0 + dr;
    c[k] = Cols(8 * (int)(off - dr * a.G), a.F);
    const bool there = row[k] < a.N;
    if (!there) c[k].n = 0;
    const char* from = static_cast<const char*>(a.x) + (there ? row[k] : 0) * a.ldx * sizeof(typename Elem<T>::type);
    fetch8<T, SMALL, uint64_t>(from, 0, a.F, c[k], raw[k]);
  }
#pragma unroll
  for (int k = 0; k < DROP_GROUPS; ++k) {
    float f[8];
    unpack8<T>(raw[k], c[k], f);
    drop8(f, random8(key, (uint32_t)c[k].col >> 3, row[k], a.r.stream), a.r.cut, a.r.keep);
    store8<T, true, uint64_t>(a.y, row[k], a.F, c[k], f);
  }
}

// ------------------------------------------------------------------ rows
template <int CTRL>
__device__ __forceinline__ float lane_dpp(float x) {
  return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), CTRL, 0xf, 0xf, true));
}
struct Add { static __device__ __forceinline__ float of(float a, float b) { return a + b; } };
struct Max { static __device__ __forceinline__ float of(float a, float b) { return fmaxf(a, b); } };

// over the 64 lanes, the result in every lane: neighbours, pairs, quads and halves of 16 by DPP, then the rows of 16
// and the halves of the wave against each other
template <class Op>
__device__ __forceinline__ float wave_reduce(float x) {
  x = Op::of(x, lane_dpp<0xB1>(x));
  x = Op::of(x, lane_dpp<0x4E>(x));
  x = Op::of(x, lane_dpp<0x141>(x));
  x = Op::of(x, lane_dpp<0x140>(x));
  auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = Op::of(__uint_as_float(s[0]), __uint_as_float(s[1]));
  s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return Op::of(__uint_as_float(s[0]), __uint_as_float(s[1]));
}

// A row belongs to NW waves of a workgroup, `first` and those behind it; a lane's E vectors of 8 columns lie 512 NW
// apart.
struct RowSum {
  float (*buf)[16];
  int NW, first, wave, turn;
  template <class Op>
  __device__ __forceinline__ float over(float x) {
    x = wave_reduce<Op>(x);
    if (NW == 1) return x;
    turn ^= 1;                        // two buffers: a wave that is a reduction ahead writes the other
    if ((threadIdx.x & 63) == 0) buf[turn][wave] = x;
    __syncthreads();
    float v = buf[turn][first];
    for (int k = 1; k < NW; ++k) v = Op::of(v, buf[turn][first + k]);
    return v;
  }
};

// rs of a row.  Squares pass fp32 from 1.8e19 on and lose bits below 1e-19 (which shows where eps is as small), and bf16 and fp32
// rows may hold such values: their squares are summed again of values scaled by a power of two.  (The condition is the
// same in all waves of the row.)
template <int E>
__device__ __forceinline__ float row_rs(const float (&v)[E][8], int d, float eps, RowSum& rows) {
  float ss = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e)
#pragma unroll
    for (int q = 0; q < 8; ++q) ss += v[e][q] * v[e][q];
  ss = rows.over<Add>(ss);
  float rs = 1.0f / sqrtf(ss / (float)d + eps);
  if (ss > 3.0e38f || (ss < 0x1p-90f && eps < 0x1p-90f)) {
    float top = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
      for (int q = 0; q < 8; ++q) top = fmaxf(top, fabsf(v[e][q]));
    top = rows.over<Max>(top);
    if (top > 0.0f && top <= 3.4028235e38f) {
      const float s = ss > 1.0f ? 0x1p-80f : 0x1p80f;   // d <= 2^14: the sum lies between 2^-48 and 2^110, or 2^-138 and 2^84
      ss = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e)
#pragma unroll
        for (int q = 0; q < 8; ++q) ss += v[e][q] * s * (v[e][q] * s);
      ss = rows.over<Add>(ss);
      rs = s / sqrtf(ss / (float)d + eps * s * s);
    }
  }
  return rs;
}

struct SeamArgs {
  int64_t N;
  int d, NW;
  const void *h, *y;
  const float *post, *pre;
  const void* gate;
  int gate_type;
  int64_t gate_rows, per;       // rows of the gate, and rows of h that share one
  float alpha, eps;
  Random r;
  void *h_out, *n_out;
  float *rs_post, *rs_pre;
  // backward
  const void *dh_out, *dn;
  void *dh, *dy;
  float* part;                  // [vectors][blocks][d]
  void* d_gate;
  int64_t W, blocks, bpg;       // rows of a worker, workgroups, workgroups of a gate row (0: gate rows lie in workers)
};

// Memory-bound: the row is read once and stays in registers through both norms (16384 x 1024, fp32 state, bf16 branch: 201
// MB in 38 us, 42 with dropout; a lone row of 4096: 3.4 us).
template <int TH, int TY, int E, bool DROP, bool ODD>
__global__ __launch_bounds__(512) void seam_fwd_kernel(SeamArgs a) {
  __shared__ float buf[2][16];
  const int lane = threadIdx.x & 63, wv = uniform(threadIdx.x >> 6);
  const int worker = a.NW == 1 ? wv : 0, w = a.NW == 1 ? 0 : wv, R = a.NW == 1 ? (int)(blockDim.x >> 6) : 1;
  RowSum rows{buf, a.NW, 0, w, 0};
  const int64_t row = (int64_t)blockIdx.x * R + worker;
  if (row >= a.N) return;           // one worker a workgroup where there are barriers
  float h[E][8], y[E][8];
  Cols c[E];
  {
    Raw8<TY> ry[E];
    Raw8<TH> rh[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      c[e] = Cols(8 * ((e * a.NW + w) * 64 + lane), a.d);
      fetch8<TY>(a.y, row, a.d, c[e], ry[e]);
      fetch8<TH>(a.h, row, a.d, c[e], rh[e]);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) unpack8<TY, ODD>(ry[e], c[e], y[e]), unpack8<TH, ODD>(rh[e], c[e], h[e]);
  }
  if (a.post) {
    const float rs = row_rs<E>(y, a.d, a.eps, rows);
    if (a.rs_post && lane == 0 && w == 0) a.rs_post[row] = rs;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      float p[8];
      load8<LBK_FP32, ODD>(a.post, 0, a.d, c[e], p);
#pragma unroll
      for (int q = 0; q < 8; ++q) y[e][q] = y[e][q] * rs * p[q];
    }
  }
  const uint64_t key = DROP ? (uint64_t)(a.r.seed_dev ? *a.r.seed_dev : a.r.seed) : 0;
  const int64_t grow = a.gate ? (a.gate_rows == 1 ? 0 : (int64_t)((uint32_t)row / (uint32_t)a.per)) : 0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if constexpr (DROP) drop8(y[e], random8(key, (uint32_t)c[e].col >> 3, row, a.r.stream), a.r.cut, a.r.keep);
    if (a.gate) {
      float g[8];
      load8_any<ODD>(a.gate_type, a.gate, grow, a.d, c[e], g);
#pragma unroll
      for (int q = 0; q < 8; ++q) y[e][q] *= g[q];
    }
#pragma unroll
    for (int q = 0; q < 8; ++q) h[e][q] += a.alpha * y[e][q];
    store8<TH, ODD>(a.h_out, row, a.d, c[e], h[e]);
  }
  if (a.pre) {
    const float rs = row_rs<E>(h, a.d, a.eps, rows);
    if (a.rs_pre && lane == 0 && w == 0) a.rs_pre[row] = rs;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      float p[8];
      load8<LBK_FP32, ODD>(a.pre, 0, a.d, c[e], p);
#pragma unroll
      for (int q = 0; q < 8; ++q) h[e][q] = h[e][q] * rs * p[q];
      store8<TY, ODD>(a.n_out, row, a.d, c[e], h[e]);
    }
  }
}

// The backward of a row.  h' is made again from h and y, in fp32: what was stored of it is rounded.  With
// q = w_pre dn, x2 = h' rs(h'), x1 = y rs(y):
//   t  = dh' + rs(h') (q - x2 mean(q x2)) = dh          d_pre  = sum of dn x2
//   s  = alpha gate t, dropped as z was                 d_gate = sum of alpha t drop(z), d_post = sum of s x1
//   dy = rs(y) (v - x1 mean(v x1)),  v = w_post s
// A workgroup takes consecutive rows, a worker (NW waves) W of these, and keeps the columns' sums in registers; the next
// row's loads are in flight while a row is worked on.  Sums go to `part`, one row a workgroup, and are added in a fixed
// order by seam_sum_kernel: no atomics.  A gate's rows either lie in one worker each (bpg = 0: written at once) or take bpg
// workgroups each.  Memory-bound: 302 MB of 16384 x 1024 (fp32 state, bf16 branch) in 61 to 65 us by the card with dropout,
// which is the copy's rate (FULL; with post, pre and gate loaded in every row, which waits for the next row's loads too, 75).
template <int TH, int TY, int E, bool DROP, bool ODD, bool FULL>
__global__ __launch_bounds__(512) void seam_bwd_kernel(SeamArgs a) {
  __shared__ float buf[2][16];
  extern __shared__ __attribute__((aligned(16))) float shared[];    // [workers][d]; FULL: and ahead of it post, pre, gate, 512 NW each
  const bool with_dn = FULL || a.dn, with_dh = FULL || a.dh_out, with_post = FULL || a.post;
  const int lane = threadIdx.x & 63, wv = uniform(threadIdx.x >> 6), R = (int)(blockDim.x >> 6) / a.NW;
  const int worker = uniform(wv / a.NW), w = wv - worker * a.NW;
  RowSum rows{buf, a.NW, worker * a.NW, wv, 0};
  int64_t r0, end;
  if (a.bpg) {                      // workgroups of one gate row
    const int64_t g = blockIdx.x / a.bpg, c = blockIdx.x - g * a.bpg;
    r0 = g * a.per + (c * R + worker) * a.W;
    end = min(r0 + a.W, (g + 1) * a.per);
  } else {
    r0 = ((int64_t)blockIdx.x * R + worker) * a.W;
    end = min(r0 + a.W, a.N);
  }
  const uint64_t key = DROP ? (uint64_t)(a.r.seed_dev ? *a.r.seed_dev : a.r.seed) : 0;
  float s_pre[E][8] = {}, s_post[E][8] = {}, s_gate[E][8] = {};
  Cols c[E];
#pragma unroll
  for (int e = 0; e < E; ++e) c[e] = Cols(8 * ((e * a.NW + w) * 64 + lane), a.d);
  int64_t grow = a.gate && a.gate_rows > 1 && r0 < a.N ? r0 / a.per : 0, gend = (grow + 1) * a.per;
  Raw8<TH> rt[E], rh[E];
  Raw8<TY> ry[E], rv[E];
  float next1 = 1.0f, next2 = 1.0f;
  // y and dn for the next row are loaded once this row's are unpacked, dh and h once the first sum has taken h's place.
  // Loads end in their order, so nothing else is loaded in between: what all rows share lies in LDS (FULL), and a load that
  // some path left out would count as one that has ended (behind the last row it is loaded again).
  auto fetch_y = [&](int64_t row) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      fetch8<TY>(a.y, row, a.d, c[e], ry[e]);
      if (with_dn) fetch8<TY>(a.dn, row, a.d, c[e], rv[e]);
    }
    if (with_post) next1 = a.rs_post[row];
    if (with_dn) next2 = a.rs_pre[row];
  };
  auto fetch_h = [&](int64_t row) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (with_dn) fetch8<TH>(a.h, row, a.d, c[e], rh[e]);
      if (with_dh) fetch8<TH>(a.dh_out, row, a.d, c[e], rt[e]);
    }
  };
  // computed here, before the registers that it was computed from are loaded again
  auto settle = [](float (&f)[8]) {
#pragma unroll
    for (int q = 0; q < 8; ++q) asm volatile("" : "+v"(f[q]));
  };
  if (r0 < end) fetch_y(r0), fetch_h(r0);
  if constexpr (FULL) {
    static_assert(E == 1);
    const int P = 512 * a.NW;
    const float* from[2] = {a.post, a.pre};
    for (int k = threadIdx.x; k < P; k += blockDim.x) {
#pragma unroll
      for (int j = 0; j < 2; ++j) shared[j * P + k] = k < a.d ? from[j][k] : 0.0f;
    }
    if (threadIdx.x < P / 8) {
      const Cols o(8 * threadIdx.x, a.d);
      float g[8];
      if (a.gate) load8_any<ODD>(a.gate_type, a.gate, a.bpg ? blockIdx.x / a.bpg : 0, a.d, o, g);
#pragma unroll
      for (int q = 0; q < 8; ++q) shared[2 * P + o.col + q] = a.gate ? g[q] : 1.0f;
    }
    __syncthreads();
  }
  auto param = [&](int k, const void* from, int e, float (&f)[8]) {
    if constexpr (FULL) {
      const f32x4* p = reinterpret_cast<const f32x4*>(shared + k * 512 * a.NW + c[0].col);
      const f32x4 lo = p[0], hi = p[1];
#pragma unroll
      for (int q = 0; q < 4; ++q) f[q] = lo[q], f[4 + q] = hi[q];
    } else {
      load8<LBK_FP32, ODD>(from, 0, a.d, c[e], f);
    }
  };
  // All workers make W turns, for the barriers of a row of many waves; one past its rows' end only takes part in these.
  for (int64_t row = r0; row < r0 + a.W; ++row) {
    if (row >= end) {
      if (a.NW == 1) break;
      if (with_dn) rows.over<Add>(0.f);
      if (with_post) rows.over<Add>(0.f);
      continue;
    }
    if (a.gate && row >= gend) ++grow, gend += a.per;
    const float rs1 = next1, rs2 = next2;
    float t[E][8], y[E][8], z[E][8], g[E][8];
    u32x4 rnd[E];
    float x[E][8], v[E][8];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      unpack8<TY, ODD>(ry[e], c[e], y[e]);
      unpack8<TY, ODD>(rv[e], c[e], v[e]);
#pragma unroll
      for (int q = 0; q < 8; ++q) y[e][q] *= rs1;             // x1
      settle(y[e]), settle(v[e]);
    }
    const int64_t next = min(row + 1, end - 1);
    fetch_y(next);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (FULL) param(2, nullptr, e, g[e]);
      else if (a.gate) load8_any<ODD>(a.gate_type, a.gate, grow, a.d, c[e], g[e]);
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        z[e][q] = y[e][q];
        if (!FULL && !a.gate) g[e][q] = 1.0f;
      }
      if (with_post) {
        float p[8];
        param(0, a.post, e, p);
#pragma unroll
        for (int q = 0; q < 8; ++q) z[e][q] *= p[q];
      }
      if constexpr (DROP) {
        rnd[e] = random8(key, (uint32_t)c[e].col >> 3, row, a.r.stream);
        drop8(z[e], rnd[e], a.r.cut, a.r.keep);
      }
    }
    float dot = 0.f;
    if (with_dn) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        float p[8];
        param(1, a.pre, e, p);
        unpack8<TH, ODD>(rh[e], c[e], x[e]);
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          x[e][q] = (x[e][q] + a.alpha * (z[e][q] * g[e][q])) * rs2;
          s_pre[e][q] += v[e][q] * x[e][q];
          v[e][q] *= p[q];
          dot += v[e][q] * x[e][q];
        }
      }
      dot = rows.over<Add>(dot) / (float)a.d;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      unpack8<TH, ODD>(rt[e], c[e], t[e]);
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        if (!with_dh) t[e][q] = 0.f;
        if (with_dn) t[e][q] += rs2 * (v[e][q] - x[e][q] * dot);
      }
      settle(t[e]);
    }
    fetch_h(next);
    dot = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (FULL || a.dh) store8<TH, ODD>(a.dh, row, a.d, c[e], t[e]);
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        t[e][q] *= a.alpha;
        s_gate[e][q] += t[e][q] * z[e][q];
        t[e][q] *= g[e][q];
      }
      if constexpr (DROP) drop8(t[e], rnd[e], a.r.cut, a.r.keep);
      if (with_post) {
        float p[8];
        param(0, a.post, e, p);
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          s_post[e][q] += t[e][q] * y[e][q];
          t[e][q] *= p[q];
          dot += t[e][q] * y[e][q];
        }
      }
    }
    if (with_post) {
      dot = rows.over<Add>(dot) / (float)a.d;
#pragma unroll
      for (int e = 0; e < E; ++e)
#pragma unroll
        for (int q = 0; q < 8; ++q) t[e][q] = rs1 * (t[e][q] - y[e][q] * dot);
    }
    if (FULL || a.dy)
#pragma unroll
      for (int e = 0; e < E; ++e) store8<TY, ODD>(a.dy, row, a.d, c[e], t[e]);
    if (!FULL && a.d_gate && a.bpg == 0 && row + 1 == gend) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        store8_any<ODD>(a.gate_type, a.d_gate, grow, a.d, c[e], s_gate[e]);
#pragma unroll
        for (int q = 0; q < 8; ++q) s_gate[e][q] = 0.f;
      }
    }
  }
  float* sums = shared + (FULL ? 3 * 512 * a.NW : 0);
  if (!a.part) return;
  // the workers' sums in their order, one vector after the other through LDS
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    if (k == 2 && (!a.d_gate || a.bpg == 0)) break;
    float* dst = a.part + (k * a.blocks + blockIdx.x) * a.d;
    if (R == 1) {
#pragma unroll
      for (int e = 0; e < E; ++e) store8<LBK_FP32, ODD>(dst, 0, a.d, c[e], k == 0 ? s_pre[e] : k == 1 ? s_post[e] : s_gate[e]);
      continue;
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
      for (int q = 0; q < 8; ++q)
        if (q < c[e].n) sums[worker * a.d + c[e].col + q] = k == 0 ? s_pre[e][q] : k == 1 ? s_post[e][q] : s_gate[e][q];
    __syncthreads();
    for (int c = threadIdx.x; c < a.d; c += blockDim.x) {
      float v = sums[c];
      for (int j = 1; j < R; ++j) v += sums[j * a.d + c];
      dst[c] = v;
    }
  }
}

// d_pre, d_post (jobs 0 and 1) and the gate's rows (2 ..): sums of `part` over a job's workgroups
struct SumArgs {
  const float* part;
  int64_t blocks, bpg;
  int d, gate_type, chunks;         // chunks: workgroups of a job
  float *d_pre, *d_post;
  void* d_gate;
};

// A workgroup sums 64 columns, 4 a lane, in 64 slices of the rows: 16-byte loads, eight of a thread in flight (2-byte
// aligned as everywhere, for odd d).
__global__ __launch_bounds__(1024) void seam_sum_kernel(SumArgs a) {
  __shared__ f32x4 sums[64][16];
  const int64_t job = blockIdx.x / a.chunks;
  const int lane = threadIdx.x & 15, slice = threadIdx.x >> 4, c0 = (int)(blockIdx.x - job * a.chunks) * 64, c = c0 + 4 * lane;
  const int64_t first = job < 2 ? job * a.blocks : 2 * a.blocks + (job - 2) * a.bpg, count = job < 2 ? a.blocks : a.bpg;
  const bool wanted = job == 0 ? a.d_pre != nullptr : job == 1 ? a.d_post != nullptr : true;
  if (!wanted) return;
  f32x4 v = {0, 0, 0, 0};
  const float* p = a.part + first * a.d + c;
  if (c + 4 <= a.d) {
#pragma unroll 8
    for (int64_t b = slice; b < count; b += 64) v += *reinterpret_cast<const f32x4_4*>(p + b * a.d);
  } else if (c < a.d) {
    for (int64_t b = slice; b < count; b += 64)
      for (int q = 0; q < a.d - c; ++q) v[q] += p[b * a.d + q];
  }
  sums[slice][lane] = v;
  __syncthreads();
  if (threadIdx.x >= 64 || c0 + (int)threadIdx.x >= a.d) return;
  const int col = c0 + threadIdx.x;
  float t = 0.f;
#pragma unroll 16
  for (int k = 0; k < 64; ++k) t += sums[k][threadIdx.x >> 2][threadIdx.x & 3];
  if (job == 0) a.d_pre[col] = t;
  else if (job == 1) a.d_post[col] = t;
  else {
    const int64_t at = (job - 2) * a.d + col;
    if (a.gate_type == LBK_FP32) static_cast<float*>(a.d_gate)[at] = t;
    else static_cast<uint16_t*>(a.d_gate)[at] = a.gate_type == LBK_BF16 ? from_f<LBK_BF16>(t) : from_f<LBK_FP16>(t);
  }
}

// ------------------------------------------------------------------ launches
inline hipStream_t S(void* s) { return reinterpret_cast<hipStream_t>(s); }
inline int launched() { return hipGetLastError() == hipSuccess ? LBK_OK : LBK_ERR_LAUNCH; }
// a launch takes fewer than 2^32 threads
inline bool too_many(int64_t blocks, int threads) { return blocks > (int64_t)UINT32_MAX / threads; }
inline bool elem_aligned(const void* p, int type) { return (reinterpret_cast<uintptr_t>(p) & (type == LBK_FP32 ? 3u : 1u)) == 0; }

bool random_of(double p, const int64_t* seed_dev, int64_t seed, uint32_t stream, Random& r) {
  if (!(p >= 0.0 && p <= 1.0)) return false;
  r.seed_dev = seed_dev, r.seed = seed, r.stream = stream;
  r.cut = (uint32_t)floor(p * 65536.0 + 0.5);
  r.keep = (float)(65536.0 / (65536.0 - r.cut));     // unused at cut = 65536
  return true;
}

// Vectors of 8 a lane (E) and waves a row: one vector up to the 8 waves of a workgroup.  Two in half as many waves spare
// the barriers of a row of 1024 and measure the same forward (41.9 and 42.4 us at 16384 x 1024 with dropout, 78.8 and 79.0
// backward), but a lone row of 4096 takes 4.0 us instead of 3.4, and the backward has no registers left.
struct RowPlan {
  int E, NW;
};
RowPlan row_plan(int d) {
  int NW = 1;
  const int E = d <= 4096 ? 1 : 2;
  while (NW * 512 * E < d) NW *= 2;
  return {E, NW};
}

// rows of a worker and workgroups of the backward
struct BwdPlan {
  RowPlan row;
  int R;
  int64_t W, blocks, bpg;
};
BwdPlan bwd_plan(int64_t N, int d, bool gate, int64_t gate_rows) {
  BwdPlan p;
  p.row = row_plan(d);
  // workgroups of eight waves, one on a CU (backward and sums of 16384 x 1024: 64.9 us, of 4097 x 1001 in fp16 25.5; four
  // waves, two on a CU: 64.0 and 28.5, three: 65.9 and 29.3; eight waves, two on a CU: 68.5 and 34.5)
  p.R = 8 / p.row.NW;
  const int64_t most = 256, W = (N + most * p.R - 1) / (most * p.R);
  const int64_t per = gate ? N / gate_rows : N;
  p.W = W;
  if (!gate) {
    p.bpg = 0;
    p.blocks = (N + W * p.R - 1) / (W * p.R);
  } else if (per >= W * p.R) {
    p.bpg = (per + W * p.R - 1) / (W * p.R);
    p.blocks = p.bpg * gate_rows;
  } else {
    p.W = W > per ? W / per * per : per;
    p.bpg = 0;
    p.blocks = (N + p.W * p.R - 1) / (p.W * p.R);
  }
  return p;
}

constexpr int MAX_D = 8192;

int check_seam(const lbk_seam* s, SeamArgs& a) {
  if (!s) return LBK_ERR_NULL;
  const bool types = (s->state_type == s->type || s->state_type == LBK_FP32) && s->type >= LBK_BF16 && s->type <= LBK_FP32;
  if (!types || s->N < 0 || !(s->eps >= 0.0f) || !random_of(s->p, s->seed_dev, s->seed, s->stream_id, a.r)) return LBK_ERR_ARG;
  if (s->d < 8) return LBK_ERR_SHAPE;
  if (s->d > MAX_D || s->N > 0x7fffffff) return LBK_ERR_TOO_LARGE;
  if (s->gate) {
    if (s->gate_type < LBK_BF16 || s->gate_type > LBK_FP32) return LBK_ERR_ARG;
    if (s->gate_rows <= 0 || s->N % s->gate_rows) return LBK_ERR_SHAPE;
    if (!elem_aligned(s->gate, s->gate_type)) return LBK_ERR_ALIGN;
  }
  if (!elem_aligned(s->post_scale, LBK_FP32) || !elem_aligned(s->pre_scale, LBK_FP32)) return LBK_ERR_ALIGN;
  a.N = s->N, a.d = s->d;
  a.post = s->post_scale, a.pre = s->pre_scale;
  a.gate = s->gate, a.gate_type = s->gate_type;
  a.gate_rows = s->gate ? s->gate_rows : 1, a.per = a.N / a.gate_rows;
  a.alpha = s->residual_scale, a.eps = s->eps;
  return LBK_OK;
}

template <int TH, int TY, int E, bool ODD, bool BWD>
int launch_seam_e(const SeamArgs& a, int64_t blocks, int threads, int lds, hipStream_t st) {
  auto go = [&](auto* k, int more = 0) {
    k<<<(unsigned)blocks, threads, lds + more, st>>>(a);
    return launched();
  };
  if constexpr (BWD && E == 1) {
    // a training step's call, all operands of its rows there and a workgroup's rows under one gate
    if (a.dn && a.dh_out && a.post && a.dh && a.dy && (!a.gate || a.bpg))
      return a.r.cut ? go(seam_bwd_kernel<TH, TY, E, true, ODD, true>, 3 * 2048 * a.NW)
                     : go(seam_bwd_kernel<TH, TY, E, false, ODD, true>, 3 * 2048 * a.NW);
  }
  if constexpr (BWD) return a.r.cut ? go(seam_bwd_kernel<TH, TY, E, true, ODD, false>) : go(seam_bwd_kernel<TH, TY, E, false, ODD, false>);
  else return a.r.cut ? go(seam_fwd_kernel<TH, TY, E, true, ODD>) : go(seam_fwd_kernel<TH, TY, E, false, ODD>);
}
template <int TH, int TY, bool BWD>
int launch_seam_t(const SeamArgs& a, int E, int64_t blocks, int threads, int lds, hipStream_t st) {
  if (a.d % 8) {
    return E == 1 ? launch_seam_e<TH, TY, 1, true, BWD>(a, blocks, threads, lds, st)
                  : launch_seam_e<TH, TY, 2, true, BWD>(a, blocks, threads, lds, st);
  }
  return E == 1 ? launch_seam_e<TH, TY, 1, false, BWD>(a, blocks, threads, lds, st)
                : launch_seam_e<TH, TY, 2, false, BWD>(a, blocks, threads, lds, st);
}
template <bool BWD>
int launch_seam(int state, int type, const SeamArgs& a, int E, int64_t blocks, int threads, int lds, hipStream_t st) {
  if (state == LBK_FP32) {
    if (type == LBK_BF16) return launch_seam_t<LBK_FP32, LBK_BF16, BWD>(a, E, blocks, threads, lds, st);
    if (type == LBK_FP16) return launch_seam_t<LBK_FP32, LBK_FP16, BWD>(a, E, blocks, threads, lds, st);
    return launch_seam_t<LBK_FP32, LBK_FP32, BWD>(a, E, blocks, threads, lds, st);
  }
  if (type == LBK_BF16) return launch_seam_t<LBK_BF16, LBK_BF16, BWD>(a, E, blocks, threads, lds, st);
  return launch_seam_t<LBK_FP16, LBK_FP16, BWD>(a, E, blocks, threads, lds, st);
}

}  // namespace
}  // namespace lbk

using namespace lbk;

extern "C" {

int lbk_dropout(const void* x, int32_t dtype, int64_t N, int32_t F, int64_t ldx, double p, const int64_t* seed_dev,
                int64_t seed, uint32_t stream_id, void* y, void* stream) {
  DropArgs a{};
  if (dtype < LBK_BF16 || dtype > LBK_FP32 || N < 0 || ldx < F || !random_of(p, seed_dev, seed, stream_id, a.r)) return LBK_ERR_ARG;
  if (F <= 0) return LBK_ERR_SHAPE;
  if (N == 0) return LBK_OK;
  if (!x || !y) return LBK_ERR_NULL;
  if (x == y && ldx != F && N > 1) return LBK_ERR_ARG;      // rows of y would lie over other rows of x
  if (!elem_aligned(x, dtype) || !elem_aligned(y, dtype)) return LBK_ERR_ALIGN;
  const int64_t G = ((int64_t)F + 7) / 8;
  if (N > INT64_MAX / 64 / ldx || N > ((int64_t)0x7fffffff * 256) / G) return LBK_ERR_TOO_LARGE;
  a.x = x, a.y = y, a.N = N, a.ldx = ldx, a.F = F, a.G = (int)G;
  uint32_t s = 0;
  while (((int64_t)1 << s) < G) ++s;
  a.shift = 31 + s;
  a.magic = (uint32_t)((((uint64_t)1 << a.shift) + G - 1) / G);
  const int64_t blocks = (N * G + 256 * DROP_GROUPS - 1) / (256 * DROP_GROUPS);
  if (too_many(blocks, 256)) return LBK_ERR_TOO_LARGE;
  auto go = [&](auto* k) {
    k<<<(unsigned)blocks, 256, 0, S(stream)>>>(a);
    return launched();
  };
  if (dtype == LBK_BF16) return F < 8 ? go(dropout_kernel<LBK_BF16, true>) : go(dropout_kernel<LBK_BF16, false>);
  if (dtype == LBK_FP16) return F < 8 ? go(dropout_kernel<LBK_FP16, true>) : go(dropout_kernel<LBK_FP16, false>);
  return F < 8 ? go(dropout_kernel<LBK_FP32, true>) : go(dropout_kernel<LBK_FP32, false>);
}

int lbk_residual_norm_fwd(const lbk_seam* s, const void* h, const void* y, void* h_out, void* n_out, float* rs_post,
                          float* rs_pre, void* stream) {
  SeamArgs a{};
  if (int st = check_seam(s, a)) return st;
  if (a.N == 0) return LBK_OK;
  if (!h || !y || !h_out || (a.pre && !n_out)) return LBK_ERR_NULL;
  if (!elem_aligned(h, s->state_type) || !elem_aligned(h_out, s->state_type) || !elem_aligned(y, s->type) ||
      !elem_aligned(n_out, s->type) || !elem_aligned(rs_post, LBK_FP32) || !elem_aligned(rs_pre, LBK_FP32))
    return LBK_ERR_ALIGN;
  a.h = h, a.y = y, a.h_out = h_out, a.n_out = n_out, a.rs_post = rs_post, a.rs_pre = rs_pre;
  const RowPlan p = row_plan(a.d);
  a.NW = p.NW;
  const int R = p.NW == 1 ? 4 : 1;
  if (too_many((a.N + R - 1) / R, 64 * p.NW * R)) return LBK_ERR_TOO_LARGE;
  return launch_seam<false>(s->state_type, s->type, a, p.E, (a.N + R - 1) / R, 64 * p.NW * R, 0, S(stream));
}

size_t lbk_residual_norm_bwd_workspace_bytes(const lbk_seam* s) {
  SeamArgs a{};
  if (check_seam(s, a)) return 0;
  if (a.N == 0) return 0;
  const BwdPlan p = bwd_plan(a.N, a.d, a.gate != nullptr, a.gate_rows);
  return ((size_t)3 * p.blocks * a.d * 4 + 255) & ~(size_t)255;
}

int lbk_residual_norm_bwd(const lbk_seam* s, const void* h, const void* y, const float* rs_post, const float* rs_pre,
                          const void* dh_out, const void* dn, void* dh, void* dy, float* d_post, void* d_gate, float* d_pre,
                          void* workspace, size_t workspace_bytes, void* stream) {
  SeamArgs a{};
  if (int st = check_seam(s, a)) return st;
  if ((dn && !a.pre) || (d_pre && !a.pre) || (d_post && !a.post) || (d_gate && !a.gate)) return LBK_ERR_ARG;
  if (a.N > 0 && (!y || (dn && (!h || !rs_pre)) || (a.post && !rs_post))) return LBK_ERR_NULL;
  if (!elem_aligned(y, s->type) || !elem_aligned(h, s->state_type) || !elem_aligned(dh_out, s->state_type) ||
      !elem_aligned(dn, s->type) || !elem_aligned(dh, s->state_type) || !elem_aligned(dy, s->type) ||
      !elem_aligned(d_gate, s->gate_type) || !elem_aligned(d_post, LBK_FP32) || !elem_aligned(d_pre, LBK_FP32) ||
      !elem_aligned(rs_post, LBK_FP32) || !elem_aligned(rs_pre, LBK_FP32) || !elem_aligned(workspace, LBK_FP32))
    return LBK_ERR_ALIGN;
  const bool vectors = d_post || d_gate || d_pre;
  const size_t need = vectors ? lbk_residual_norm_bwd_workspace_bytes(s) : 0;
  if (need && (!workspace || workspace_bytes < need)) return LBK_ERR_WORKSPACE;
  BwdPlan p{};
  if (a.N > 0) {
    p = bwd_plan(a.N, a.d, a.gate != nullptr, a.gate_rows);
    a.NW = p.row.NW, a.W = p.W, a.blocks = p.blocks, a.bpg = p.bpg;
    a.h = h, a.y = y, a.rs_post = const_cast<float*>(rs_post), a.rs_pre = const_cast<float*>(rs_pre);
    a.dh_out = dh_out, a.dn = dn, a.dh = dh, a.dy = dy, a.d_gate = d_gate;
    a.part = vectors ? static_cast<float*>(workspace) : nullptr;
    const int lds = p.R > 1 ? p.R * a.d * 4 : 0;      // at most 16 KB
    if (int st = launch_seam<true>(s->state_type, s->type, a, p.row.E, p.blocks, 64 * p.row.NW * p.R, lds, S(stream))) return st;
  }
  if (!vectors) return LBK_OK;
  SumArgs m{static_cast<float*>(workspace), p.blocks, p.bpg, a.d, a.gate_type, (a.d + 63) / 64, d_pre, d_post, d_gate};
  // a gate without rows has no gradients to write, but for the one row that stands for none
  const int64_t jobs = 2 + (d_gate && (p.bpg || a.N == 0) ? a.gate_rows : 0);
  if (too_many(jobs * m.chunks, 1024)) return LBK_ERR_TOO_LARGE;
  seam_sum_kernel<<<(unsigned)(jobs * m.chunks), 1024, 0, S(stream)>>>(m);
  return launched();
}

}  // extern "C"
