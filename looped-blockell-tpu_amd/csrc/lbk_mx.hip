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

namespace lbk {

typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
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

// ------------------------------------------------------------------ products
struct MxArgs {
  const uint8_t* xc; const uint8_t* xs;     // quantised tokens [N, F / 2], [N, F / 32]
  int64_t N;
  int F;                                    // input features
  lbk_bell_mx w0, w1;                       // the product's weight, or gate and up
  const float* b0; const float* b1;
  const uint16_t* resid;                    // MODE 0, optional [N, R B]
  uint16_t* y;                              // MODE 0: [N, R B]
  uint8_t* hc; uint8_t* hs;                 // MODE 1: quantised silu(gate) * up
};

// Gate/up epilogue: this lane's 16 values of a group of 32 hidden features of one token (features
// (v % 4) + 8 (v / 4) + 4 half; the partner lane l ^ 32 has the others) -> codes and scale.  The group's
// maximum and code halves cross by one exchange each; each lane stores 8 of the 16 code bytes.
__device__ __forceinline__ void mx_store_group(const float (&h)[16], int half, uint8_t* hc, uint8_t* hs, bool live) {
  uint32_t m = 0;
#pragma unroll
  for (int v = 0; v < 16; ++v) m = max(m, absbits(h[v]));
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

// MODE 0: y = Q(x) W (+ bias) (+ resid).  MODE 1: quantised silu(gate + b0) * (up + b1).
// The general kernel: four waves of 32 tokens share 32 outputs; every operand comes from global memory
// (L1 and L2).  Any N, K and F.
template <int B, int MODE>
__global__ __launch_bounds__(256) void mx_rowblock_kernel(MxArgs a) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, i = lane & 31;
  const int64_t n = ((int64_t)blockIdx.y * 4 + wave) * 32 + i;
  if (((int64_t)blockIdx.y * 4 + wave) * 32 >= a.N) return;
  const int64_t nc = n < a.N ? n : a.N - 1;
  const uint8_t* xc = a.xc + nc * (a.F >> 1);
  const uint8_t* xs = a.xs + nc * (a.F >> 5);
  const int o0 = blockIdx.x * 32, r = o0 / B, j = o0 % B + i, C = a.F / B;

  auto product = [&](const lbk_bell_mx& w) {
    f32x16 acc = {};
    constexpr int STEP = 64 / B;            // slots of one MFMA
    for (int k = 0; k < w.K; k += STEP) {
      const int slot = B == 32 ? k + half : k;
      const int col = slot < w.K ? w.col_idx[(int64_t)r * w.K + slot] : -1;
      const bool live = col >= 0 && col < C;
      u32x4 wa = {}, xb = {};
      uint32_t sa = 127, sb = 127;          // a dead slot multiplies zeros
      if (live) {
        const int64_t at = (((int64_t)r * w.K + slot) * B + j) * (B / 32) + (B == 64 ? half : 0);
        const int g = B == 32 ? col : 2 * col + half;
        wa = reinterpret_cast<const u32x4*>(w.codes)[at];
        sa = w.scales[at];
        xb = reinterpret_cast<const u32x4*>(xc)[g];
        sb = xs[g];
      }
      acc = mfma_fp4(wa, xb, acc, sa, sb);
    }
    return acc;
  };

  const f32x16 p0 = product(a.w0);
  float v[16];
  if constexpr (MODE == 1) {
    const f32x16 p1 = product(a.w1);
#pragma unroll
    for (int q = 0; q < 16; ++q) {
      const int o = o0 + (q & 3) + 8 * (q >> 2) + 4 * half;
      const float g = p0[q] + (a.b0 ? a.b0[o] : 0.0f), u = p1[q] + (a.b1 ? a.b1[o] : 0.0f);
      v[q] = silu_f(g) * u;
    }
    const int64_t grp = nc * ((int64_t)a.w0.R * B / 32) + blockIdx.x;
    mx_store_group(v, half, a.hc + grp * 16, a.hs + grp, n < a.N);
  } else {
    if (n >= a.N) return;
    const int64_t ld = (int64_t)a.w0.R * B;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int o = o0 + 8 * q + 4 * half;
      float f[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = p0[4 * q + e] + (a.b0 ? a.b0[o + e] : 0.0f);
      if (a.resid) {
        float t[4];
        load_bf16x<4>(a.resid + n * ld + o, t);
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] += t[e];
      }
      store_bf16x<4>(a.y + n * ld + o, f);
    }
  }
}

template <int MODE>
int launch_mx_rowblock(const MxArgs& a, hipStream_t st) {
  const int B = a.w0.B;
  const int64_t blocks = (a.N + 127) / 128;
  for (int64_t b0 = 0; b0 < blocks; b0 += 65535) {                // grid.y's limit
    MxArgs p = a;
    const int64_t n0 = b0 * 128, F = a.F, O = (int64_t)a.w0.R * B;
    p.N = a.N - n0 < 65535 * 128 ? a.N - n0 : 65535 * 128;
    p.xc += n0 * (F >> 1);
    p.xs += n0 * (F >> 5);
    if (p.resid) p.resid += n0 * O;
    if (p.y) p.y += n0 * O;
    if (p.hc) p.hc += n0 * (O / 2), p.hs += n0 * (O / 32);
    const dim3 grid((unsigned)(O / 32), (unsigned)((p.N + 127) / 128));
    if (B == 32) mx_rowblock_kernel<32, MODE><<<grid, 256, 0, st>>>(p);
    else mx_rowblock_kernel<64, MODE><<<grid, 256, 0, st>>>(p);
  }
  return hipGetLastError() == hipSuccess ? 0 : -1;
}

}  // namespace lbk

using namespace lbk;

namespace {

inline bool a16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline hipStream_t S(void* s) { return reinterpret_cast<hipStream_t>(s); }
inline size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }
constexpr int64_t kMaxThreads = 0xffffff00;     // of one launch

int check_mx(const lbk_bell_mx* w) {
  if (!w) return LBK_ERR_NULL;
  if (w->B != 32 && w->B != 64) return LBK_ERR_TILE;
  if (w->R < 0 || w->K < 0) return LBK_ERR_SHAPE;
  if ((int64_t)w->R * w->B > 0x7fffffff) return LBK_ERR_SHAPE;
  if ((int64_t)w->R * w->K > 0 && (!w->codes || !w->scales || !w->col_idx)) return LBK_ERR_NULL;
  if (w->codes && !a16(w->codes)) return LBK_ERR_ALIGN;
  return LBK_OK;
}

// codes and scales of [N, F] in a workspace
struct Quantised {
  uint8_t* c;
  uint8_t* s;
};
size_t quantised_bytes(int64_t N, int64_t F) { return align256((size_t)N * F / 2) + align256((size_t)N * F / 32); }
Quantised quantised_at(void* p, int64_t N, int64_t F) {
  uint8_t* c = static_cast<uint8_t*>(p);
  return {c, c + align256((size_t)N * F / 2)};
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
  if (N > 0 && (N * (int64_t)F) / F != N) return LBK_ERR_TOO_LARGE;
  return N * (int64_t)F / 8 > kMaxThreads ? LBK_ERR_TOO_LARGE : LBK_OK;
}
int check_tiles(int32_t dtype, int32_t R, int32_t K, int32_t B) {
  if (dtype < LBK_BF16 || dtype > LBK_FP32) return LBK_ERR_ARG;
  if (B != 32 && B != 64) return LBK_ERR_TILE;
  return R < 0 || K < 0 ? LBK_ERR_SHAPE : LBK_OK;
}

int check_ffn_mx(const lbk_bell_mx* gate, const lbk_bell_mx* up, const lbk_bell_mx* down, int32_t d_model) {
  for (const lbk_bell_mx* w : {gate, up, down})
    if (int st = check_mx(w)) return st;
  if (gate->B != up->B || gate->B != down->B) return LBK_ERR_TILE;
  if (gate->R != up->R || gate->R <= 0 || d_model <= 0 || d_model % gate->B) return LBK_ERR_SHAPE;
  return (int64_t)down->R * down->B == d_model ? LBK_OK : LBK_ERR_SHAPE;
}

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
  if (n > kMaxThreads) return LBK_ERR_TOO_LARGE;
  if (!values || !codes || !scales) return LBK_ERR_NULL;
  if (!a16(codes)) return LBK_ERR_ALIGN;
  return by_dtype<QuantizeTiles>(dtype, values, n, (int)B, codes, scales, S(stream));
}

int lbk_mx_dequantize_tiles(const uint8_t* codes, const uint8_t* scales, int32_t R, int32_t K, int32_t B,
                            int32_t dtype, void* values, void* stream) {
  if (int st = check_tiles(dtype, R, K, B)) return st;
  const int64_t n = (int64_t)R * K * B * (B / 32);
  if (n == 0) return LBK_OK;
  if (n > kMaxThreads) return LBK_ERR_TOO_LARGE;
  if (!codes || !scales || !values) return LBK_ERR_NULL;
  if (!a16(codes)) return LBK_ERR_ALIGN;
  return by_dtype<DequantizeTiles>(dtype, codes, scales, n, (int)B, values, S(stream));
}

size_t lbk_mx_matmul_workspace_bytes(int64_t N, int32_t in_features, const lbk_bell_mx* w) {
  if (!w || N <= 0 || in_features <= 0) return 0;
  return quantised_bytes(N, in_features);
}

int lbk_mx_matmul_bf16(const uint16_t* x, int64_t N, int32_t in_features, const lbk_bell_mx* w, const float* bias,
                       uint16_t* y, void* workspace, size_t workspace_bytes, void* stream) {
  if (int st = check_mx(w)) return st;
  if (N < 0) return LBK_ERR_ARG;
  if (in_features <= 0 || in_features % w->B) return LBK_ERR_SHAPE;
  if (N == 0 || w->R == 0) return LBK_OK;
  if (!x || !y) return LBK_ERR_NULL;
  if (!a16(x) || !a16(y) || !a16(workspace)) return LBK_ERR_ALIGN;
  const size_t need = lbk_mx_matmul_workspace_bytes(N, in_features, w);
  if (need && (!workspace || workspace_bytes < need)) return LBK_ERR_WORKSPACE;
  const Quantised q = quantised_at(workspace, N, in_features);
  if (int st = lbk_mx_quantize(x, LBK_BF16, N, in_features, in_features, q.c, q.s, stream)) return st;
  MxArgs a{};
  a.xc = q.c; a.xs = q.s; a.N = N; a.F = in_features; a.w0 = *w; a.b0 = bias; a.y = y;
  return launch_mx_rowblock<0>(a, S(stream)) == 0 ? LBK_OK : LBK_ERR_LAUNCH;
}

size_t lbk_mx_swiglu_workspace_bytes(int64_t N, int32_t d_model, const lbk_bell_mx* gate, const lbk_bell_mx* up,
                                     const lbk_bell_mx* down) {
  if (!gate || !up || !down || N <= 0 || d_model <= 0) return 0;
  return quantised_bytes(N, d_model) + quantised_bytes(N, (int64_t)gate->R * gate->B);
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
  const size_t need = lbk_mx_swiglu_workspace_bytes(N, d_model, gate, up, down);
  if (!workspace || workspace_bytes < need) return LBK_ERR_WORKSPACE;
  const int64_t d_ff = (int64_t)gate->R * gate->B;
  const Quantised q = quantised_at(workspace, N, d_model);
  const Quantised h = quantised_at(static_cast<uint8_t*>(workspace) + quantised_bytes(N, d_model), N, d_ff);
  if (int st = lbk_mx_quantize(x, LBK_BF16, N, d_model, d_model, q.c, q.s, stream)) return st;
  MxArgs g{};
  g.xc = q.c; g.xs = q.s; g.N = N; g.F = d_model; g.w0 = *gate; g.w1 = *up; g.b0 = b_gate; g.b1 = b_up;
  g.hc = h.c; g.hs = h.s;
  if (launch_mx_rowblock<1>(g, S(stream)) != 0) return LBK_ERR_LAUNCH;
  MxArgs d{};
  d.xc = h.c; d.xs = h.s; d.N = N; d.F = (int)d_ff; d.w0 = *down; d.b0 = b_down; d.y = out;
  d.resid = add_residual ? x : nullptr;
  return launch_mx_rowblock<0>(d, S(stream)) == 0 ? LBK_OK : LBK_ERR_LAUNCH;
}

}  // extern "C"
