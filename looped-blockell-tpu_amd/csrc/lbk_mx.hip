// lbk_mx.hip — microscaled 4-bit floating point: quantisation, Block-ELL products and the SwiGLU FFN
// on such weights, and their entry points of include/lbk.h.
//
// Format (OCP MXFP4): groups of 32 consecutive input features share a power of two.
//   scale byte b = clamp(floor(log2 max|x|) - 2 + 127, 0, 254), value 2^(b - 127); 255 (NaN) where
//   the group holds an Inf or a NaN;
//   code: sign and one of 0, .5, 1, 1.5, 2, 3, 4, 6, the nearest to x / 2^(b - 127), ties to the even
//   code, beyond 6 to 6; two codes a byte, the even index low.
// A lane of the scaled MFMAs holds 32 consecutive K codes (16 bytes) of one row and their scale byte,
// so an operand register is a piece of a row as it lies in memory, and a group may come from any
// Block-ELL slot: one 32x32x64 MFMA takes two B = 32 slots or one B = 64 slot.
//   A (32 x 64): lane l holds row l % 32, k = 32 (l / 32) .. + 31;  B the same for column l % 32
//   C (32 x 32): lane l holds column l % 32, rows (v % 4) + 8 (v / 4) + 4 (l / 32), v = 0 .. 15
// Weights are A and tokens B, so a lane ends with 16 outputs of one token and its partner l ^ 32 with
// the other 16: a group of 32 outputs is requantised with one exchange.
#include "lbk.h"
#include "lbk_device.h"
#include "lbk_internal.h"

#include <initializer_list>
#include <type_traits>

namespace lbk {

typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));

// fp4 x fp4; sa, sb: the scale bytes in bits 0 .. 7
__device__ __forceinline__ f32x16 mfma_fp4(const u32x4& a, const u32x4& b, const f32x16& c, uint32_t sa, uint32_t sb) {
  const i32x8_t A = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
  const i32x8_t Bm = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(A, Bm, c, 4, 4, 0, (int)sa, 0, (int)sb);
}

// the scale byte of a group from the bits of its largest magnitude (integer order is float order, and
// a NaN's bits are above an Inf's)
__device__ __forceinline__ uint32_t mx_scale(uint32_t absbits) {
  const int e = (int)(absbits >> 23);
  return e == 255 ? 255u : (uint32_t)max(e - 2, 0);
}
// 2^(b - 127) for b = 0 .. 254 (2^-127 is subnormal)
__device__ __forceinline__ float mx_pow2(uint32_t b) { return __uint_as_float(b ? b << 23 : 0x00400000u); }
// The conversion rounds to the nearest even code and saturates (checked on gfx950, subnormal scales
// included); an Inf scale stands in for 255, whose codes nobody reads as numbers.
__device__ __forceinline__ uint32_t mx_code8(const float (&f)[8], float s) {
  uint32_t r = 0;
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, f[0], f[1], s, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, f[2], f[3], s, 1);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, f[4], f[5], s, 2);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, f[6], f[7], s, 3);
  return r;
}
__device__ __forceinline__ uint32_t absbits(float f) { return __float_as_uint(f) & 0x7fffffffu; }

// ------------------------------------------------------------------ element types
template <int DT> struct Elem;                       // 0 bf16, 1 fp16, 2 fp32
template <> struct Elem<LBK_BF16> {
  using T = uint16_t;
  static __device__ __forceinline__ float get(T v) { return bf2f(v); }
  static __device__ __forceinline__ T put(float f) { return f2bf(f); }
};
template <> struct Elem<LBK_FP16> {
  using T = uint16_t;
  static __device__ __forceinline__ float get(T v) { return (float)__builtin_bit_cast(_Float16, v); }
  static __device__ __forceinline__ T put(float f) { return __builtin_bit_cast(uint16_t, (_Float16)f); }
};
template <> struct Elem<LBK_FP32> {
  using T = float;
  static __device__ __forceinline__ float get(T v) { return v; }
  static __device__ __forceinline__ T put(float f) { return f; }
};

// 8 consecutive elements at a 16-byte aligned address
template <int DT>
__device__ __forceinline__ void load8(const typename Elem<DT>::T* p, float (&f)[8]) {
  if constexpr (DT == LBK_FP32) {
    const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = a[i], f[4 + i] = b[i];
  } else {
    const u32x4 w = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = Elem<DT>::get((uint16_t)(w[i] & 0xffffu));
      f[2 * i + 1] = Elem<DT>::get((uint16_t)(w[i] >> 16));
    }
  }
}

// ------------------------------------------------------------------ rows
// Four lanes a group, 8 features each: 16-byte loads, 4-byte stores, the largest magnitude through
// two exchanges.  HBM-bound: 2 + 17/32 bytes a bf16 element.
template <int DT>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const typename Elem<DT>::T* __restrict__ x, int64_t ldx,
                                                          int64_t n8, int F, uint8_t* __restrict__ codes,
                                                          uint8_t* __restrict__ scales) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;      // this lane's run of 8 elements
  if (i >= n8) return;                                            // n8 is a multiple of 4: groups stay whole
  const int64_t f8 = F >> 3, row = i / f8;
  float f[8];
  load8<DT>(x + row * ldx + (i - row * f8) * 8, f);
  uint32_t m = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) m = max(m, absbits(f[k]));
  m = max(m, (uint32_t)__shfl_xor((int)m, 1));
  m = max(m, (uint32_t)__shfl_xor((int)m, 2));
  const uint32_t b = mx_scale(m);
  reinterpret_cast<uint32_t*>(codes)[i] = mx_code8(f, mx_pow2(b));
  if ((i & 3) == 0) scales[i >> 2] = (uint8_t)b;
}

template <int DT>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(const uint8_t* __restrict__ codes,
                                                            const uint8_t* __restrict__ scales, int64_t n8,
                                                            typename Elem<DT>::T* __restrict__ out) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n8) return;
  const uint32_t w = reinterpret_cast<const uint32_t*>(codes)[i], b = scales[i >> 2];
  const float s = mx_pow2(b);
  float f[8];
  {
    const f32x2_t p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0);
    const f32x2_t p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1);
    const f32x2_t p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 2);
    const f32x2_t p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 3);
    f[0] = p0[0], f[1] = p0[1], f[2] = p1[0], f[3] = p1[1], f[4] = p2[0], f[5] = p2[1], f[6] = p3[0], f[7] = p3[1];
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) f[k] = b == 255 ? __uint_as_float(0x7fc00000u) : f[k] * s;
  typename Elem<DT>::T o[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) o[k] = Elem<DT>::put(f[k]);
  u32x4* p = reinterpret_cast<u32x4*>(out + i * 8);
  const u32x4* q = reinterpret_cast<const u32x4*>(o);
#pragma unroll
  for (int k = 0; k < (int)sizeof(o) / 16; ++k) p[k] = q[k];
}

// ------------------------------------------------------------------ tiles
// values [tile][B_in][B_out] -> codes [tile][B_out][B_in / 2], scales [tile][B_out][B_in / 32]: a thread
// takes the 32 inputs of one output; consecutive threads read consecutive outputs.
template <int DT>
__global__ __launch_bounds__(256) void mx_quantize_tiles_kernel(const typename Elem<DT>::T* __restrict__ v, int64_t n,
                                                                int B, uint8_t* __restrict__ codes,
                                                                uint8_t* __restrict__ scales) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;      // (tile, input group, output)
  if (i >= n) return;
  const int G = B / 32;
  const int64_t tg = i / B, tile = tg / G;
  const int j = (int)(i - tg * B), g = (int)(tg - tile * G);
  const typename Elem<DT>::T* p = v + (tile * B + 32 * g) * B + j;
  float f[4][8];
  uint32_t m = 0;
#pragma unroll
  for (int q = 0; q < 4; ++q)
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      f[q][k] = Elem<DT>::get(p[(int64_t)(8 * q + k) * B]);
      m = max(m, absbits(f[q][k]));
    }
  const uint32_t b = mx_scale(m);
  const float s = mx_pow2(b);
  u32x4 w;
#pragma unroll
  for (int q = 0; q < 4; ++q) w[q] = mx_code8(f[q], s);
  const int64_t at = (tile * B + j) * G + g;
  reinterpret_cast<u32x4*>(codes)[at] = w;
  scales[at] = (uint8_t)b;
}

template <int DT>
__global__ __launch_bounds__(256) void mx_dequantize_tiles_kernel(const uint8_t* __restrict__ codes,
                                                                  const uint8_t* __restrict__ scales, int64_t n, int B,
                                                                  typename Elem<DT>::T* __restrict__ v) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const int G = B / 32;
  const int64_t tg = i / B, tile = tg / G;
  const int j = (int)(i - tg * B), g = (int)(tg - tile * G);
  const int64_t at = (tile * B + j) * G + g;
  const u32x4 w = reinterpret_cast<const u32x4*>(codes)[at];
  const uint32_t b = scales[at];
  const float s = b == 255 ? __uint_as_float(0x7fc00000u) : mx_pow2(b);
  typename Elem<DT>::T* p = v + (tile * B + 32 * g) * B + j;
#pragma unroll
  for (int k = 0; k < 32; ++k) {
    const uint32_t c = (w[k >> 3] >> (4 * (k & 7))) & 15u, mag = c & 7u;
    float f = mag < 2 ? 0.5f * (float)mag : (float)((2 + (mag & 1)) << (mag >> 1)) * 0.25f;
    f = (c & 8u) ? -f : f;
    p[(int64_t)k * B] = Elem<DT>::put(f * s);
  }
}

// ------------------------------------------------------------------ token panels
// The quantised tokens that the panel products read: blocks of TB = 32 MT tokens, each [group][token] codes
// of 16 bytes, then [group][token % 32][token / 32] scale bytes, both padded to 1 KB: a workgroup copies a
// block to LDS as it lies, 32 lanes read consecutive 16-byte pieces there, and one read gives the scale
// bytes of a lane's MT tokens.  Tokens behind the last one hold whatever was there: they reach no output.
struct Panel {
  int64_t codes, bytes;      // bytes of a block's codes, and of the block
};
__host__ __device__ inline Panel panel_of(int G, int TB) {
  const int64_t c = ((int64_t)G * TB * 16 + 1023) & ~(int64_t)1023;
  return {c, c + (((int64_t)G * TB + 1023) & ~(int64_t)1023)};
}

// x [N, F] bf16 -> panel blocks.  A wave takes 16 tokens and two groups (a 128-byte line of each token):
// four lanes a token and group, 8 features each.
__global__ __launch_bounds__(256) void mx_quantize_panel_kernel(const uint16_t* __restrict__ x, int64_t N, int F, int TB,
                                                                uint8_t* __restrict__ panels) {
  const int lane = threadIdx.x & 63, G = F >> 5, pairs = (G + 1) >> 1;
  const int64_t wv = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t n = wv / pairs * 16 + (lane >> 2);
  const int g0 = (int)(wv % pairs) * 2, part = lane & 3;
  if (n >= N) return;                                             // four lanes of a token leave together
  const Panel P = panel_of(G, TB);
  uint8_t* blk = panels + n / TB * P.bytes;
  const int tt = (int)(n % TB), MT = TB / 32;
  float f[2][8];
#pragma unroll
  for (int k = 0; k < 2; ++k)
    if (g0 + k < G) load8<LBK_BF16>(x + n * F + (g0 + k) * 32 + part * 8, f[k]);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if (g0 + k >= G) break;
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = max(m, absbits(f[k][e]));
    m = max(m, (uint32_t)__shfl_xor((int)m, 1));
    m = max(m, (uint32_t)__shfl_xor((int)m, 2));
    const uint32_t b = mx_scale(m);
    const int64_t at = (int64_t)(g0 + k) * TB;
    *reinterpret_cast<uint32_t*>(blk + (at + tt) * 16 + part * 4) = mx_code8(f[k], mx_pow2(b));
    if (part == 0) blk[P.codes + at + (tt & 31) * MT + (tt >> 5)] = (uint8_t)b;
  }
}

// ------------------------------------------------------------------ products
// Gate/up epilogue: this lane's 16 values of a group of 32 hidden features of one token (features
// (v % 4) + 8 (v / 4) + 4 half; the partner lane l ^ 32 has the others) -> codes and scale.  The group's
// maximum and code halves cross by one exchange each; each lane stores 8 of the 16 code bytes.
__device__ __forceinline__ void mx_store_group(const float (&h)[16], int half, uint8_t* hc, uint8_t* hs, bool live) {
  // positive values are largest as signed integers, negative ones as unsigned (NaNs above all, either way):
  // half an instruction a value each, where masking the sign off took a whole one
  int mp = 0;
  uint32_t mn = 0;
#pragma unroll
  for (int v = 0; v < 16; ++v) {
    mp = max(mp, __float_as_int(h[v]));
    mn = max(mn, __float_as_uint(h[v]));
  }
  uint32_t m = max((uint32_t)mp, mn & 0x7fffffffu);
  m = max(m, (uint32_t)__shfl_xor((int)m, 32));
  const uint32_t b = mx_scale(m);
  const float s = mx_pow2(b);
  uint32_t c[4];                            // features 8 q + 4 half .. + 3, in the low 16 bits
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint32_t r = 0;
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, h[4 * q], h[4 * q + 1], s, 0);
    c[q] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, h[4 * q + 2], h[4 * q + 3], s, 1) & 0xffffu;
  }
  const uint32_t mine01 = c[0] | c[1] << 16, mine23 = c[2] | c[3] << 16;
  const uint32_t got = (uint32_t)__shfl_xor((int)(half ? mine01 : mine23), 32);   // the half that this lane stores
  const uint32_t lo = half ? got : mine01, hi = half ? mine23 : got;              // from lanes l % 32 and + 32
  if (live) {
    *reinterpret_cast<u32x2*>(hc + 8 * half) =
        u32x2{__builtin_amdgcn_perm(hi, lo, 0x05040100u), __builtin_amdgcn_perm(hi, lo, 0x07060302u)};
    if (half == 0) *hs = (uint8_t)b;
  }
}

// ------------------------------------------------------------------ products on token panels
struct MxPanelArgs {
  const uint8_t* x;                         // panels of 32 MT tokens, or
  const uint16_t* xb;                       // (not NULL) bf16 rows [N, F], quantised by the workgroup
  int64_t N;
  int F, slices;
  lbk_bell_mx w0, w1;
  const float* b0; const float* b1;
  const uint16_t* resid;
  uint16_t* y;                              // MODE 0
  uint8_t* h; int TBh;                      // MODE 1: panels of TBh tokens
};

// A workgroup of NW waves holds 32 MT tokens in LDS and one of `slices` shares of the 32-row output tiles; a
// wave takes every NW-th tile of the share.  The (tile, weight, slot pair) positions of a wave form one stream:
// their codes (16 bytes a lane), scale and column are loaded D positions ahead, always all three, so that the
// compiler's load counters stay exact across tiles.  A dead slot, and the second half of an odd row's last
// pair, multiplies zeros with unit scales.
// MODE 1 (16384 tokens, 1024 -> 4096 at 0.25: 59 us) issues 30 us of vector instructions on every SIMD, counted at
// four clocks each, and its exponentials and reciprocals, at a quarter of that rate, take 10 more; the matrix unit
// is busy for 7 of them.  What the remaining time waits for is not measured.  Its 12 waves (three a SIMD) hold 64
// accumulators each.
// FROM: where a workgroup's tokens are: 0 a panel copied to LDS, 1 bf16 rows that it quantises into LDS itself,
// 2 the panel in global memory (too wide for LDS: 32 lanes read 512 consecutive bytes there too).
template <int B, int MODE, int MT, int NW, bool BIAS, int FROM>
__global__ __launch_bounds__(NW * 64, NW / 4) void mx_panel_kernel(MxPanelArgs a) {
  constexpr int TB = 32 * MT, D = 2;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, w = uniform(tid >> 6), half = lane >> 5, i = lane & 31;
  const int G = a.F >> 5, C = a.F / B;
  const Panel P = panel_of(G, TB);
  const int64_t tb = blockIdx.x / a.slices;
  const int sl = (int)(blockIdx.x % a.slices);
  const int tiles = a.w0.R * (B / 32);
  const int mEnd = (int)((int64_t)tiles * (sl + 1) / a.slices), m0 = (int)((int64_t)tiles * sl / a.slices) + w;

  typedef __attribute__((address_space(3))) unsigned char lds_byte;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_byte*)smem;
  if constexpr (FROM == 1) {
    // 16 tokens and two groups (a 128-byte line of each token) a wave and turn, four lanes a group
    const int tl = lane >> 2, part = lane & 3, pairs = (G + 1) >> 1;
#pragma unroll 2
    for (int v = w; v < 2 * MT * pairs; v += NW) {
      const int tt = v % (2 * MT) * 16 + tl, g0 = v / (2 * MT) * 2;
      const int64_t n = min(tb * TB + tt, a.N - 1);
      const uint16_t* row = a.xb + n * a.F + part * 8;
      float f[2][8];
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (g0 + k < G) load8<LBK_BF16>(row + (g0 + k) * 32, f[k]);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        if (g0 + k >= G) break;
        uint32_t m = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) m = max(m, absbits(f[k][e]));
        m = max(m, (uint32_t)__shfl_xor((int)m, 1));
        m = max(m, (uint32_t)__shfl_xor((int)m, 2));
        const uint32_t b = mx_scale(m);
        const int at = (g0 + k) * TB;
        *reinterpret_cast<uint32_t*>(smem + (at + tt) * 16 + part * 4) = mx_code8(f[k], mx_pow2(b));
        if (part == 0) smem[P.codes + at + (tt & 31) * MT + (tt >> 5)] = (uint8_t)b;
      }
    }
  } else if constexpr (FROM == 0) {
    const uint8_t* src = a.x + tb * P.bytes + lane * 16;
    for (int p = w; p < (int)(P.bytes >> 10); p += NW) lds_fetch16(src + (int64_t)p * 1024, lds0 + (uint32_t)p * 1024);
  }

  // a position is QP instructions' slots (STEP each)
  constexpr int STEP = 64 / B, QP = 2;     // (the scales' and columns' passing on is for two)
  const int P0 = (a.w0.K + STEP * QP - 1) / (STEP * QP), P1 = MODE == 1 ? (a.w1.K + STEP * QP - 1) / (STEP * QP) : 0;
  // loading position, D ahead of the computing one: the row's codes, scales and columns, and this lane's place
  // in a slot's tile; a tile on is NW * 32 / B block rows on
  struct Row {
    const uint8_t *c, *s;
    const int32_t* i;
  };
  int lm = min(m0, mEnd - 1), lup = 0, lj = 0;
  auto row_of = [&](const lbk_bell_mx& wt) {
    const int64_t base = (int64_t)(lm * 32 / B) * wt.K;
    return Row{wt.codes + base * (B * B / 2), wt.scales + base * (B * B / 32), wt.col_idx + base};
  };
  Row r0 = row_of(a.w0), r1 = MODE == 1 ? row_of(a.w1) : Row{};
  const uint32_t place = (uint32_t)(lm * 32 % B + i) * (B / 32) + (B == 64 ? half : 0);
  // Every load takes its turn of 16 cycles of the CU's address unit, whatever its size, so one fetches the
  // position's scales (two bytes a lane: B = 32 the four slots' 128 bytes as they lie, B = 64 both input halves
  // of the tile's 32 rows of two slots) and one its columns (even lanes those of the first instruction, odd ones
  // of the second); the lanes pass them on in compute.
  u32x4 wr[D][QP];
  uint32_t sr[D];
  int cr[D];
  const int odd = lane & 1;
  const uint32_t splace = B == 32 ? 2 * lane : (uint32_t)(lm * 32 % B + i) * 2;
  auto load = [&](int d) {
    const Row& r = MODE == 1 && lup ? r1 : r0;
    const int K = MODE == 1 && lup ? a.w1.K : a.w0.K;
#pragma unroll
    for (int p = 0; p < QP; ++p) {
      const uint32_t slot = (uint32_t)min(B == 32 ? 2 * (lj * QP + p) + half : lj * QP + p, K - 1);
      wr[d][p] = reinterpret_cast<const u32x4*>(r.c)[slot * (B * (B / 32)) + place];
    }
    const uint32_t sat = B == 32 ? min((uint32_t)lj * 128 + splace, (uint32_t)K * 32 - 2)
                                 : (uint32_t)min(lj * QP + half, K - 1) * 128 + splace;
    sr[d] = *reinterpret_cast<const uint16_t*>(r.s + sat);
    cr[d] = r.i[min(B == 32 ? lj * 4 + 2 * odd + half : lj * QP + odd, K - 1)];
    if (++lj == (MODE == 1 && lup ? P1 : P0)) {
      lj = 0;
      if (MODE == 1 && !lup) {
        lup = 1;
      } else {
        lup = 0;
        if (lm + NW < mEnd) {                    // behind the last tile: its loads again, for nobody
          lm += NW;
          r0 = row_of(a.w0);
          if constexpr (MODE == 1) r1 = row_of(a.w1);
        }
      }
    }
  };
#pragma unroll
  for (int d = 0; d < D; ++d) load(d);
  // the panel is in LDS
  if constexpr (FROM == 1) asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  if constexpr (FROM == 0) asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((QP + 2) * D) : "memory");
  if (m0 >= mEnd) return;

  f32x16 acc[MODE + 1][MT] = {};
  const unsigned char* const xc = FROM == 2 ? a.x + tb * P.bytes : smem;
  const unsigned char* const xs = xc + P.codes;
  int cm = m0, cup = 0, cj = 0;
  auto compute = [&](int d, f32x16 (&c)[MT], int K, bool first) {
    u32x4 wv[QP], xv[QP][MT];
    uint32_t sa[QP], sb[QP];
    int g[QP];
    bool live[QP], whole = true;
    const int other = __builtin_amdgcn_mov_dpp(cr[d], 0xb1, 0xf, 0xf, true);      // the neighbouring lane's
    const int col[QP] = {odd ? other : cr[d], odd ? cr[d] : other};
#pragma unroll
    for (int p = 0; p < QP; ++p) {
      live[p] = (B == 64 ? cj * QP + p : 2 * (cj * QP + p) + half) < K && (uint32_t)col[p] < (uint32_t)C;
      whole &= live[p];
      g[p] = B == 32 ? col[p] : 2 * col[p] + half;
      wv[p] = wr[d][p];
      const int from = B == 32 ? (2 * p + half) * 16 + (i >> 1) : 32 * p + i;
      sa[p] = (uint32_t)__builtin_amdgcn_ds_bpermute(from * 4, (int)sr[d]) >> (B == 32 ? 8 * odd : 8 * half);
    }
    const bool dead = __ballot(whole) != ~0ull;
    if (dead) {
#pragma unroll
      for (int p = 0; p < QP; ++p)
        if (!live[p]) g[p] = 0, wv[p] = u32x4{0, 0, 0, 0}, sa[p] = 127u;
    }
#pragma unroll
    for (int p = 0; p < QP; ++p) {
      if constexpr (MT == 2) sb[p] = reinterpret_cast<const uint16_t*>(xs)[g[p] * 32 + i];
      else sb[p] = xs[g[p] * 32 + i];
#pragma unroll
      for (int t = 0; t < MT; ++t) xv[p][t] = reinterpret_cast<const u32x4*>(xc)[g[p] * TB + 32 * t + i];
    }
    if (dead) {
#pragma unroll
      for (int p = 0; p < QP; ++p)
        if (!live[p]) sb[p] = 0x7f7fu;
    }
#pragma unroll
    for (int p = 0; p < QP; ++p) {
      const i32x8_t A = {(int)wv[p][0], (int)wv[p][1], (int)wv[p][2], (int)wv[p][3], 0, 0, 0, 0};
      auto mm = [&](int t, auto sel) {
        const i32x8_t Bm = {(int)xv[p][t][0], (int)xv[p][t][1], (int)xv[p][t][2], (int)xv[p][t][3], 0, 0, 0, 0};
        if (first && p == 0) c[t] = f32x16{};
        c[t] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(A, Bm, c[t], 4, 4, 0, (int)sa[p], decltype(sel)::value, (int)sb[p]);
      };
      mm(0, std::integral_constant<int, 0>{});
      if constexpr (MT == 2) mm(1, std::integral_constant<int, 1>{});
    }
  };
  // a tile's biases, one a lane (lanes 32 .. 63: up's), loaded with its first position and passed on from there
  float bias = 0.0f;
  auto load_bias = [&]() {
    const float* b = MODE == 1 && half ? a.b1 : a.b0;
    bias = b ? b[cm * 32 + i] : 0.0f;
  };
  auto bias_at = [&](int q, int from) {
    return __int_as_float(__builtin_amdgcn_ds_bpermute((from + (q & 3) + 8 * (q >> 2) + 4 * half) * 4, __float_as_int(bias)));
  };
  auto store = [&]() {
    const int o0 = cm * 32;
    if constexpr (MODE == 1) {
      const int Gh = a.w0.R * (B / 32);
      const Panel Ph = panel_of(Gh, a.TBh);
      const int MTh = a.TBh / 32;
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        float v[16];
#pragma unroll
        for (int q = 0; q < 16; ++q) {
          const float g = acc[0][t][q], u = acc[MODE][t][q];
          v[q] = BIAS ? silu_f(g + bias_at(q, 0)) * (u + bias_at(q, 32)) : silu_f(g) * u;
        }
        const int64_t tile = tb * MT + t;                       // of 32 tokens; TBh is 32 or 64
        const int sub = (int)tile & (MTh - 1);
        uint8_t* blk = a.h + (tile >> (MTh - 1)) * Ph.bytes;
        mx_store_group(v, half, blk + (cm * a.TBh + sub * 32 + i) * 16, blk + Ph.codes + cm * a.TBh + i * MTh + sub,
                       tile * 32 + i < a.N);
      }
    } else {
      const int64_t ld = (int64_t)a.w0.R * B;
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        const int64_t n = tb * TB + 32 * t + i;
#pragma unroll
        for (int q = 0; q < 4; q += 2) {
          // 4 features of each of q and q + 1 -> 8 consecutive ones: half 0 takes those of q, half 1 of q + 1
          float f[8];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(acc[0][t][4 * q + e]),
                                                             __float_as_uint(acc[0][t][4 * q + 4 + e]), false, false);
            f[e] = __uint_as_float(sw[0]);
            f[4 + e] = __uint_as_float(sw[1]);
          }
          const int o = o0 + 8 * (q + half);
          if constexpr (BIAS) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              f[e] += __int_as_float(__builtin_amdgcn_ds_bpermute((8 * (q + half) + e) * 4, __float_as_int(bias)));
          }
          if (n < a.N) {
            if (a.resid) {
              float r[8];
              load_bf16x<8>(a.resid + n * ld + o, r);
#pragma unroll
              for (int e = 0; e < 8; ++e) f[e] += r[e];
            }
            store_bf16x<8>(a.y + n * ld + o, f);
          }
        }
      }
    }
  };
  for (;;) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      // a tile's first products add to the constant 0 of the instruction, in code of their own
      if (MODE == 1 && cup) {
        if (cj == 0) compute(d, acc[MODE], a.w1.K, true);
        else compute(d, acc[MODE], a.w1.K, false);
      } else {
        if (cj == 0) {
          if constexpr (BIAS) load_bias();
          compute(d, acc[0], a.w0.K, true);
        } else {
          compute(d, acc[0], a.w0.K, false);
        }
      }
      load(d);
      if (++cj == (MODE == 1 && cup ? P1 : P0)) {
        cj = 0;
        if (MODE == 1 && !cup) cup = 1;
        else {
          store();
          cup = 0;
          cm += NW;
          if (cm >= mEnd) return;
        }
      }
    }
  }
}

// Whether the codes and scales of 32 tokens are too wide for LDS, and the tokens of a panel block.  (Tokens of
// 8192 features read from global memory, 64 at a time, instead of 32 in LDS: 54 -> 51 us at 2048 tokens of
// 4096 / 8192, but 26 -> 31 at 512 and 48 -> 57 with the four times shorter rows of 2048 / 8192.)
inline bool mx_wide(int F) { return F > 9600; }
inline int mx_block_tokens(int F) { return mx_wide(F) || panel_of(F / 32, 64).bytes <= 160 * 1024 ? 64 : 32; }

// Waves of a workgroup, and the shares of the output tiles: the fewest rounds of 256 workgroups times tiles a
// wave, a workgroup's start counted as one tile
template <int MODE>
constexpr int mx_panel_waves(int MT) { return MODE == 1 && MT == 2 ? 12 : 16; }     // registers of two accumulators
template <int MODE>
int mx_panel_slices(int64_t N, int TB, int tiles) {
  const int NW = mx_panel_waves<MODE>(TB / 32);
  const int64_t nb = (N + TB - 1) / TB;
  int best = 1;
  int64_t least = INT64_MAX;
  for (int sl = 1; sl <= 32 && sl * NW <= tiles + NW - 1; ++sl) {
    const int64_t cost = (nb * sl + 255) / 256 * ((tiles + sl * NW - 1) / (sl * NW) + 1);
    if (cost < least) least = cost, best = sl;
  }
  return best;
}

// Whether a product's panels times shares are more workgroups than a launch takes (its threads are a 32-bit
// number).  Hidden features between 4800 and 9600 leave 32 tokens a panel, which passes it below the limit on tokens.
template <int MODE>
bool mx_panel_too_large(int64_t N, int F, const lbk_bell_mx& w) {
  const int TB = mx_block_tokens(F);
  return (N + TB - 1) / TB * mx_panel_slices<MODE>(N, TB, w.R * (w.B / 32)) > 0x3fffff;
}

template <int B, int MODE, int MT, bool BIAS, int FROM>
int launch_mx_panel_t(MxPanelArgs a, hipStream_t st) {
  constexpr int NW = mx_panel_waves<MODE>(MT);
  auto* k = mx_panel_kernel<B, MODE, MT, NW, BIAS, FROM>;
  const int64_t lds = FROM == 2 ? 0 : panel_of(a.F / 32, 32 * MT).bytes, nb = (a.N + 32 * MT - 1) / (32 * MT);
  a.slices = mx_panel_slices<MODE>(a.N, 32 * MT, a.w0.R * (B / 32));
  static std::atomic<uint64_t> done{0};
  if (lds > 65536 && set_lds_limit_once(reinterpret_cast<const void*>(k), 160 * 1024, done) != 0) return -1;
  k<<<(unsigned)(nb * a.slices), NW * 64, lds, st>>>(a);
  return hipGetLastError() == hipSuccess ? 0 : -1;
}
template <int MODE, bool BIAS, int FROM>
int launch_mx_panel_b(int TB, const MxPanelArgs& a, hipStream_t st) {
  const bool b32 = a.w0.B == 32;
  if (TB == 64) return b32 ? launch_mx_panel_t<32, MODE, 2, BIAS, FROM>(a, st) : launch_mx_panel_t<64, MODE, 2, BIAS, FROM>(a, st);
  if constexpr (FROM != 2)
    return b32 ? launch_mx_panel_t<32, MODE, 1, BIAS, FROM>(a, st) : launch_mx_panel_t<64, MODE, 1, BIAS, FROM>(a, st);
  return -1;
}
// a.x or a.xb given
template <int MODE>
int launch_mx_panel(int TB, const MxPanelArgs& a, hipStream_t st) {
  const bool bias = a.b0 || (MODE == 1 && a.b1);
  if (mx_wide(a.F)) return bias ? launch_mx_panel_b<MODE, true, 2>(TB, a, st) : launch_mx_panel_b<MODE, false, 2>(TB, a, st);
  if (a.xb) return bias ? launch_mx_panel_b<MODE, true, 1>(TB, a, st) : launch_mx_panel_b<MODE, false, 1>(TB, a, st);
  return bias ? launch_mx_panel_b<MODE, true, 0>(TB, a, st) : launch_mx_panel_b<MODE, false, 0>(TB, a, st);
}

int launch_quantize_panel(const uint16_t* x, int64_t N, int F, int TB, uint8_t* panels, hipStream_t st) {
  const int64_t waves = (N + 15) / 16 * ((F / 32 + 1) / 2);      // < 2^26 (too_many)
  mx_quantize_panel_kernel<<<(unsigned)((waves + 3) / 4), 256, 0, st>>>(x, N, F, TB, panels);
  return hipGetLastError() == hipSuccess ? 0 : -1;
}

// ------------------------------------------------------------------ few tokens
// A workgroup of 8 waves makes one 32-row output tile of 32 tokens: the slots are dealt to the waves (MODE 1:
// gate's to waves 0 .. 3, up's to 4 .. 7) and their sums joined through LDS in a fixed order.  The weights are
// read once, two positions on their way per wave where tokens come as bf16 rows, quantised where they are used
// (one launch less, and a row of the slot's columns is 64 bytes a lane), four where they come as panels of 32 (XQ:
// the hidden state).  Latency-bound at these sizes: 16 tokens, 4096 / 14336 at 0.1, 9 MB of weights.
template <int B, int MODE, bool XQ>
__global__ __launch_bounds__(512, 4) void mx_decode_kernel(MxPanelArgs a, const uint16_t* __restrict__ x) {
  constexpr int U = XQ ? 4 : 2, STEP = 64 / B, DEAL = MODE == 1 ? 4 : 8;
  __shared__ f32x4 part[8][4][64];
  __shared__ uint32_t top[4][64];
  const int tid = threadIdx.x, lane = tid & 63, w = uniform(tid >> 6), half = lane >> 5, i = lane & 31;
  const int64_t n = (int64_t)blockIdx.y * 32 + i;
  const int C = a.F / B, o0 = blockIdx.x * 32, r = o0 / B, j = o0 % B + i;
  const bool up = MODE == 1 && w >= 4;
  const lbk_bell_mx& wt = up ? a.w1 : a.w0;
  const int K = wt.K, P = (K + STEP - 1) / STEP;
  const Panel Px = panel_of(a.F >> 5, 32);
  const uint8_t* panel = a.x + blockIdx.y * Px.bytes;
  f32x16 acc = {};
  for (int p0 = w & (DEAL - 1); p0 < P; p0 += DEAL * U) {
    u32x4 wv[U], xv[U][XQ ? 1 : 4];
    uint32_t sa[U], sb[U];
    int col[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int pos = p0 + u * DEAL;
      if (pos >= P) break;
      const int slot = B == 32 ? 2 * pos + half : pos;
      const int64_t idx = (int64_t)r * K + min(slot, K - 1), at = (idx * B + j) * (B / 32) + (B == 64 ? half : 0);
      wv[u] = reinterpret_cast<const u32x4*>(wt.codes)[at];
      sa[u] = wt.scales[at];
      col[u] = slot < K ? wt.col_idx[idx] : -1;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (p0 + u * DEAL >= P) break;
      const bool live = (uint32_t)col[u] < (uint32_t)C;
      const int g = live ? (B == 32 ? col[u] : 2 * col[u] + half) : 0;
      if (!live) wv[u] = u32x4{0, 0, 0, 0}, sa[u] = 127;
      if constexpr (XQ) {
        xv[u][0] = reinterpret_cast<const u32x4*>(panel)[g * 32 + i];
        sb[u] = live ? panel[Px.codes + g * 32 + i] : 127u;
      } else {
        const u32x4* src = reinterpret_cast<const u32x4*>(x + n * a.F + g * 32);
#pragma unroll
        for (int k = 0; k < 4; ++k) xv[u][k] = live && n < a.N ? src[k] : u32x4{0, 0, 0, 0};
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (p0 + u * DEAL >= P) break;
      u32x4 b;
      if constexpr (XQ) {
        b = xv[u][0];
      } else {
        // the largest magnitude over packed pairs: as 16-bit integers in the upper and the lower halves
        uint32_t hi = 0, lo = 0;
        float f[4][8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          unpack8_bf16(xv[u][k], f[k]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            hi = max(hi, xv[u][k][e] & 0x7fffffffu);
            lo = max(lo, xv[u][k][e] << 16 & 0x7fffffffu);
          }
        }
        sb[u] = mx_scale(max(hi, lo));
        const float s = mx_pow2(sb[u]);
#pragma unroll
        for (int k = 0; k < 4; ++k) b[k] = mx_code8(f[k], s);
      }
      acc = mfma_fp4(wv[u], b, acc, sa[u], sb[u]);
    }
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) part[w][q][lane] = f32x4{acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]};
  __syncthreads();
  // wave q < 4: features 8 q + 4 half .. + 3 of the tile
  const int q = w & 3, o = o0 + 8 * q + 4 * half;
  float f[4] = {}, v[4] = {};
  if (w < 4) {
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      const f32x4 t = part[s][q][lane];
#pragma unroll
      for (int e = 0; e < 4; ++e) (MODE == 1 && s >= 4 ? v : f)[e] += t[e];
    }
  }
  if constexpr (MODE == 1) {
    uint32_t m = 0;
    if (w < 4) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f[e] = silu_f(f[e] + (a.b0 ? a.b0[o + e] : 0.0f)) * (v[e] + (a.b1 ? a.b1[o + e] : 0.0f));
        m = max(m, absbits(f[e]));
      }
      top[q][lane] = max(m, (uint32_t)__shfl_xor((int)m, 32));
    }
    __syncthreads();
    if (w < 4 && n < a.N) {
      m = max(max(top[0][lane], top[1][lane]), max(top[2][lane], top[3][lane]));
      const uint32_t b = mx_scale(m);
      const float s = mx_pow2(b);
      uint32_t c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, f[0], f[1], s, 0);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[2], f[3], s, 1);
      const Panel Ph = panel_of(a.w0.R * (B / 32), 32);
      uint8_t* blk = a.h + blockIdx.y * Ph.bytes;
      const int at = blockIdx.x * 32 + i;
      *reinterpret_cast<uint16_t*>(blk + at * 16 + 4 * q + 2 * half) = (uint16_t)c;
      if (q == 0 && half == 0) blk[Ph.codes + at] = (uint8_t)b;
    }
  } else {
    if (w >= 4 || n >= a.N) return;
    const int64_t at = n * ((int64_t)a.w0.R * B) + o;
    if (a.b0) {
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] += a.b0[o + e];
    }
    if (a.resid) {
      float t[4];
      load_bf16x<4>(a.resid + at, t);
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] += t[e];
    }
    store_bf16x<4>(a.y + at, f);
  }
}

// x: bf16 rows, or NULL for a.x's panels
template <int MODE>
int launch_mx_decode(const MxPanelArgs& a0, const uint16_t* x0, hipStream_t st) {
  const int64_t blocks = (a0.N + 31) / 32, O = (int64_t)a0.w0.R * a0.w0.B;
  for (int64_t b0 = 0; b0 < blocks; b0 += 65535) {                // grid.y's limit
    MxPanelArgs a = a0;
    const int64_t n0 = b0 * 32;
    a.N = a0.N - n0 < 65535 * 32 ? a0.N - n0 : 65535 * 32;
    const uint16_t* x = x0 ? x0 + n0 * a.F : nullptr;
    if (a.x) a.x += b0 * panel_of(a.F / 32, 32).bytes;
    if (a.h) a.h += b0 * panel_of((int)(O / 32), 32).bytes;
    if (a.resid) a.resid += n0 * O;
    if (a.y) a.y += n0 * O;
    const dim3 grid((unsigned)(O / 32), (unsigned)((a.N + 31) / 32));
    if (a.w0.B == 32) {
      if (x) mx_decode_kernel<32, MODE, false><<<grid, 512, 0, st>>>(a, x);
      else mx_decode_kernel<32, MODE, true><<<grid, 512, 0, st>>>(a, x);
    } else {
      if (x) mx_decode_kernel<64, MODE, false><<<grid, 512, 0, st>>>(a, x);
      else mx_decode_kernel<64, MODE, true><<<grid, 512, 0, st>>>(a, x);
    }
  }
  return hipGetLastError() == hipSuccess ? 0 : -1;
}

}  // namespace lbk

using namespace lbk;

namespace {

inline bool a16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline hipStream_t S(void* s) { return reinterpret_cast<hipStream_t>(s); }
constexpr int64_t kMaxThreads = 0xffffff00;     // of one launch
constexpr int64_t kMaxTokens = (int64_t)1 << 27;  // the products' launches, 32 tokens a workgroup
constexpr int32_t kMaxFeatures = 1 << 24;         // and slots of a row: places in a panel and in a row are 32-bit
// of a product's input: the quantising launch takes 1024 elements a wave
bool too_many(int64_t N, int32_t F) { return N > kMaxTokens || N > ((int64_t)1 << 35) / F; }

int check_mx(const lbk_bell_mx* w) {
  if (!w) return LBK_ERR_NULL;
  if (w->B != 32 && w->B != 64) return LBK_ERR_TILE;
  if (w->R < 0 || w->K < 0) return LBK_ERR_SHAPE;
  if ((int64_t)w->R * w->B > kMaxFeatures || w->K > kMaxFeatures) return LBK_ERR_TOO_LARGE;
  if ((int64_t)w->R * w->K > 0 && (!w->codes || !w->scales || !w->col_idx)) return LBK_ERR_NULL;
  if (w->codes && !a16(w->codes)) return LBK_ERR_ALIGN;
  if (w->scales && (reinterpret_cast<uintptr_t>(w->scales) & 1u)) return LBK_ERR_ALIGN;
  return LBK_OK;
}

template <template <int> class L, typename... A>
int by_dtype(int dtype, A... a) {
  if (dtype == LBK_BF16) return L<LBK_BF16>::go(a...);
  if (dtype == LBK_FP16) return L<LBK_FP16>::go(a...);
  return L<LBK_FP32>::go(a...);
}
int launched() { return hipGetLastError() == hipSuccess ? LBK_OK : LBK_ERR_LAUNCH; }

template <int DT> struct QuantizeRows {
  static int go(const void* x, int64_t ldx, int64_t n8, int F, uint8_t* c, uint8_t* s, hipStream_t st) {
    mx_quantize_kernel<DT><<<(unsigned)((n8 + 255) / 256), 256, 0, st>>>((const typename Elem<DT>::T*)x, ldx, n8, F, c, s);
    return launched();
  }
};
template <int DT> struct DequantizeRows {
  static int go(const uint8_t* c, const uint8_t* s, int64_t n8, void* out, hipStream_t st) {
    mx_dequantize_kernel<DT><<<(unsigned)((n8 + 255) / 256), 256, 0, st>>>(c, s, n8, (typename Elem<DT>::T*)out);
    return launched();
  }
};
template <int DT> struct QuantizeTiles {
  static int go(const void* v, int64_t n, int B, uint8_t* c, uint8_t* s, hipStream_t st) {
    mx_quantize_tiles_kernel<DT><<<(unsigned)((n + 255) / 256), 256, 0, st>>>((const typename Elem<DT>::T*)v, n, B, c, s);
    return launched();
  }
};
template <int DT> struct DequantizeTiles {
  static int go(const uint8_t* c, const uint8_t* s, int64_t n, int B, void* v, hipStream_t st) {
    mx_dequantize_tiles_kernel<DT><<<(unsigned)((n + 255) / 256), 256, 0, st>>>(c, s, n, B, (typename Elem<DT>::T*)v);
    return launched();
  }
};

int check_rows(int32_t dtype, int64_t N, int32_t F) {
  if (dtype < LBK_BF16 || dtype > LBK_FP32 || N < 0) return LBK_ERR_ARG;
  if (F <= 0 || F % 32) return LBK_ERR_SHAPE;
  return N > kMaxThreads / (F / 8) ? LBK_ERR_TOO_LARGE : LBK_OK;
}
int check_tiles(int32_t dtype, int32_t R, int32_t K, int32_t B) {
  if (dtype < LBK_BF16 || dtype > LBK_FP32) return LBK_ERR_ARG;
  if (B != 32 && B != 64) return LBK_ERR_TILE;
  if (R < 0 || K < 0) return LBK_ERR_SHAPE;
  return (int64_t)R * K > kMaxThreads / (B * (B / 32)) ? LBK_ERR_TOO_LARGE : LBK_OK;
}

int check_ffn_mx(const lbk_bell_mx* gate, const lbk_bell_mx* up, const lbk_bell_mx* down, int32_t d_model) {
  for (const lbk_bell_mx* w : {gate, up, down})
    if (int st = check_mx(w)) return st;
  if (gate->B != up->B || gate->B != down->B) return LBK_ERR_TILE;
  if (gate->R != up->R || gate->R <= 0 || d_model <= 0 || d_model % gate->B) return LBK_ERR_SHAPE;
  return (int64_t)down->R * down->B == d_model ? LBK_OK : LBK_ERR_SHAPE;
}

// Shares of the output tiles up to which each quantises its tokens itself: one share spares the quantising
// launch (16384 tokens, 1024 -> 4096: 80 -> 70 us), three redo its work too often (4099 tokens, 2048 / 8192:
// 89 -> 93 us)
constexpr int kFillSlices = 2;
template <int MODE>
bool fills(int64_t N, int F, const lbk_bell_mx* w) {
  return !mx_wide(F) && mx_panel_slices<MODE>(N, mx_block_tokens(F), w->R * (w->B / 32)) <= kFillSlices;
}

// Tokens up to which mx_decode_kernel takes them.  FFN in us, so / on panels: 4096 / 14336 at 0.1 64 tokens 15 / 35,
// 128 tokens 22 / 36, 256 tokens 38 / 38; 4096 / 16384 at 0.125 256 tokens 55 / 47; 1024 / 4096 at 1.0 256 tokens
// 26 / 42.  It also takes weights without slots, at any number.
constexpr int64_t kDecode = 128;
bool decodes(int64_t N, std::initializer_list<const lbk_bell_mx*> ws) {
  bool empty = false;
  for (const lbk_bell_mx* w : ws) empty |= w->K == 0;
  return N <= kDecode || empty;
}

size_t panels_bytes(int64_t N, int64_t F, int TB) { return (size_t)((N + TB - 1) / TB * panel_of((int)(F / 32), TB).bytes); }

}  // namespace

extern "C" {

int lbk_mx_quantize(const void* x, int32_t dtype, int64_t N, int32_t F, int64_t ldx, uint8_t* codes, uint8_t* scales,
                    void* stream) {
  if (int st = check_rows(dtype, N, F)) return st;
  if (ldx < F) return LBK_ERR_ARG;
  if (N == 0) return LBK_OK;
  if (!x || !codes || !scales) return LBK_ERR_NULL;
  if (!a16(x) || !a16(codes) || ldx % (dtype == LBK_FP32 ? 4 : 8)) return LBK_ERR_ALIGN;
  return by_dtype<QuantizeRows>(dtype, x, ldx, N * (F / 8), (int)F, codes, scales, S(stream));
}

int lbk_mx_dequantize(const uint8_t* codes, const uint8_t* scales, int64_t N, int32_t F, int32_t dtype, void* out,
                      void* stream) {
  if (int st = check_rows(dtype, N, F)) return st;
  if (N == 0) return LBK_OK;
  if (!codes || !scales || !out) return LBK_ERR_NULL;
  if (!a16(codes) || !a16(out)) return LBK_ERR_ALIGN;
  return by_dtype<DequantizeRows>(dtype, codes, scales, N * (F / 8), out, S(stream));
}

int lbk_mx_quantize_tiles(const void* values, int32_t dtype, int32_t R, int32_t K, int32_t B, uint8_t* codes,
                          uint8_t* scales, void* stream) {
  if (int st = check_tiles(dtype, R, K, B)) return st;
  const int64_t n = (int64_t)R * K * B * (B / 32);
  if (n == 0) return LBK_OK;
  if (!values || !codes || !scales) return LBK_ERR_NULL;
  if (!a16(codes)) return LBK_ERR_ALIGN;
  return by_dtype<QuantizeTiles>(dtype, values, n, (int)B, codes, scales, S(stream));
}

int lbk_mx_dequantize_tiles(const uint8_t* codes, const uint8_t* scales, int32_t R, int32_t K, int32_t B,
                            int32_t dtype, void* values, void* stream) {
  if (int st = check_tiles(dtype, R, K, B)) return st;
  const int64_t n = (int64_t)R * K * B * (B / 32);
  if (n == 0) return LBK_OK;
  if (!codes || !scales || !values) return LBK_ERR_NULL;
  if (!a16(codes)) return LBK_ERR_ALIGN;
  return by_dtype<DequantizeTiles>(dtype, codes, scales, n, (int)B, values, S(stream));
}

size_t lbk_mx_matmul_workspace_bytes(int64_t N, int32_t in_features, const lbk_bell_mx* w) {
  if (!w || N <= 0 || in_features <= 0 || check_mx(w) || decodes(N, {w}) || fills<0>(N, in_features, w)) return 0;
  return panels_bytes(N, in_features, mx_block_tokens(in_features));
}

int lbk_mx_matmul_bf16(const uint16_t* x, int64_t N, int32_t in_features, const lbk_bell_mx* w, const float* bias,
                       uint16_t* y, void* workspace, size_t workspace_bytes, void* stream) {
  if (int st = check_mx(w)) return st;
  if (N < 0) return LBK_ERR_ARG;
  if (in_features <= 0 || in_features % w->B) return LBK_ERR_SHAPE;
  if (in_features > kMaxFeatures) return LBK_ERR_TOO_LARGE;
  if (N == 0 || w->R == 0) return LBK_OK;
  if (!x || !y) return LBK_ERR_NULL;
  if (!a16(x) || !a16(y) || !a16(workspace)) return LBK_ERR_ALIGN;
  if (too_many(N, in_features)) return LBK_ERR_TOO_LARGE;
  const size_t need = lbk_mx_matmul_workspace_bytes(N, in_features, w);
  if (need && (!workspace || workspace_bytes < need)) return LBK_ERR_WORKSPACE;
  if (!decodes(N, {w}) && mx_panel_too_large<0>(N, in_features, *w)) return LBK_ERR_TOO_LARGE;
  MxPanelArgs a{};
  a.N = N; a.F = in_features; a.w0 = *w; a.b0 = bias; a.y = y;
  int err;
  if (decodes(N, {w})) {
    err = launch_mx_decode<0>(a, x, S(stream));
  } else {
    const int TB = mx_block_tokens(in_features);
    a.x = static_cast<uint8_t*>(workspace);
    if (fills<0>(N, in_features, w)) a.xb = x;
    else if (launch_quantize_panel(x, N, in_features, TB, static_cast<uint8_t*>(workspace), S(stream))) return LBK_ERR_LAUNCH;
    err = launch_mx_panel<0>(TB, a, S(stream));
  }
  return err == 0 ? LBK_OK : LBK_ERR_LAUNCH;
}

size_t lbk_mx_swiglu_workspace_bytes(int64_t N, int32_t d_model, const lbk_bell_mx* gate, const lbk_bell_mx* up,
                                     const lbk_bell_mx* down) {
  if (N <= 0 || check_ffn_mx(gate, up, down, d_model)) return 0;
  const int d_ff = gate->R * gate->B;
  if (decodes(N, {gate, up, down})) return panels_bytes(N, d_ff, 32);
  return (fills<1>(N, d_model, gate) ? 0 : panels_bytes(N, d_model, mx_block_tokens(d_model))) +
         panels_bytes(N, d_ff, mx_block_tokens(d_ff));
}

int lbk_mx_swiglu_fwd_bf16(const uint16_t* x, int64_t N, int32_t d_model, const lbk_bell_mx* gate,
                           const lbk_bell_mx* up, const lbk_bell_mx* down, const float* b_gate, const float* b_up,
                           const float* b_down, int add_residual, uint16_t* out, void* workspace,
                           size_t workspace_bytes, void* stream) {
  if (int st = check_ffn_mx(gate, up, down, d_model)) return st;
  if (N < 0) return LBK_ERR_ARG;
  if (N == 0) return LBK_OK;
  if (!x || !out) return LBK_ERR_NULL;
  if (!a16(x) || !a16(out) || !a16(workspace)) return LBK_ERR_ALIGN;
  if (too_many(N, d_model)) return LBK_ERR_TOO_LARGE;
  const size_t need = lbk_mx_swiglu_workspace_bytes(N, d_model, gate, up, down);
  if (!workspace || workspace_bytes < need) return LBK_ERR_WORKSPACE;
  const int d_ff = gate->R * gate->B;
  if (!decodes(N, {gate, up, down}) && (mx_panel_too_large<1>(N, d_model, *gate) || mx_panel_too_large<0>(N, d_ff, *down)))
    return LBK_ERR_TOO_LARGE;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  MxPanelArgs g{}, d{};
  g.N = d.N = N; g.F = d_model; d.F = d_ff;
  g.w0 = *gate; g.w1 = *up; g.b0 = b_gate; g.b1 = b_up;
  d.w0 = *down; d.b0 = b_down; d.resid = add_residual ? x : nullptr; d.y = out;
  if (decodes(N, {gate, up, down})) {
    g.h = ws; d.x = ws;
    if (launch_mx_decode<1>(g, x, S(stream)) != 0) return LBK_ERR_LAUNCH;
    return launch_mx_decode<0>(d, nullptr, S(stream)) == 0 ? LBK_OK : LBK_ERR_LAUNCH;
  }
  const int TBx = mx_block_tokens(d_model), TBh = mx_block_tokens(d_ff);
  if (fills<1>(N, d_model, gate)) {
    g.xb = x;
  } else {
    if (launch_quantize_panel(x, N, d_model, TBx, ws, S(stream)) != 0) return LBK_ERR_LAUNCH;
    g.x = ws;
    ws += panels_bytes(N, d_model, TBx);
  }
  g.h = ws; g.TBh = TBh; d.x = ws;
  if (launch_mx_panel<1>(TBx, g, S(stream)) != 0) return LBK_ERR_LAUNCH;
  return launch_mx_panel<0>(TBh, d, S(stream)) == 0 ? LBK_OK : LBK_ERR_LAUNCH;
}

}  // extern "C"
