// lbk_gated.hip — the dense gated FFN, out = (act(x Wg^T) * (x Wu^T)) Wd^T (+ x), with its backward
// (gfx950, bf16 or fp16 MFMA, fp32 sums), and its entry points of include/lbk.h.
//
// Weights are dense Linear weights [out, in].  Six matrix products, all on one tiled kernel:
//   forward   g, u = x Wg^T, x Wu^T with h = act(g) u in the epilogue;  out = h Wd^T (+ x)
//   backward  dh = dy Wd with dg = dh u act'(g), du = dh act(g) in the epilogue;
//             dx = dg Wg + du Wu (+ dy) as one product over both;  dWg = dg^T x, dWu = du^T x, dWd = dy^T h
// g, u, h, dg and du are rounded to the inputs' type between the products (they are the matrix
// instructions' operands, and g and u are kept for the backward); sums are fp32.
#include "lbk.h"
#include "lbk_device.h"
#include "lbk_internal.h"

namespace lbk {
namespace {

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef short i16x4_g __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) i16x4_g lds_i16x4_g;
typedef __attribute__((address_space(3))) unsigned char lds_byte;

template <bool H> struct Half;             // H: fp16, else bf16
template <> struct Half<false> {
  static __device__ __forceinline__ f32x4 mfma(const u32x4& a, const u32x4& b, const f32x4& c) { return mfma_bf16(a, b, c); }
  static __device__ __forceinline__ uint32_t pack2(float lo, float hi) { return pack2_bf16(lo, hi); }
  static __device__ __forceinline__ float lo(uint32_t w) { return bf_lo(w); }
  static __device__ __forceinline__ float hi(uint32_t w) { return bf_hi(w); }
};
template <> struct Half<true> {
  static __device__ __forceinline__ f32x4 mfma(const u32x4& a, const u32x4& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    const f16x2_t v = {(_Float16)lo, (_Float16)hi};
    return __builtin_bit_cast(uint32_t, v);
  }
  static __device__ __forceinline__ float lo(uint32_t w) { return (float)__builtin_bit_cast(f16x2_t, w)[0]; }
  static __device__ __forceinline__ float hi(uint32_t w) { return (float)__builtin_bit_cast(f16x2_t, w)[1]; }
};

// four consecutive values
template <bool H>
__device__ __forceinline__ void load4h(const uint16_t* p, float (&f)[4]) {
  const u32x2 w = *reinterpret_cast<const u32x2*>(p);
  f[0] = Half<H>::lo(w[0]), f[1] = Half<H>::hi(w[0]), f[2] = Half<H>::lo(w[1]), f[3] = Half<H>::hi(w[1]);
}
template <bool H>
__device__ __forceinline__ void store4h(uint16_t* p, const float (&f)[4]) {
  *reinterpret_cast<u32x2*>(p) = u32x2{Half<H>::pack2(f[0], f[1]), Half<H>::pack2(f[2], f[3])};
}

// sixteen zero bytes that out-of-range pieces of a tile are loaded from
__device__ const u32x4 zero16 = {0, 0, 0, 0};

// act and act' at z
__device__ __forceinline__ float act_f(float z, int act) { return act == LBK_GELU ? gelu_f(z) : silu_f(z); }
__device__ __forceinline__ void act_both(float z, int act, float& a, float& d) {
  if (act == LBK_GELU) {
    a = gelu_f(z);
    d = gelu_grad_f(z);
  } else {
    const float s = __builtin_amdgcn_rcpf(1.0f + __expf(-z));
    a = z * s;
    d = s + a * (1.0f - s);
  }
}

// ------------------------------------------------------------------ the tiled product
// D[n][m] = sum_k A(m, k) B(n, k) over one or two (A, B) pairs, in fp32; rows m of A are the features
// that lie consecutive in D.  An operand is stored [rows][K] (KC: K consecutive) or [K][rows] (MC).
//   EPI_STORE  D (+ resid) rounded to the type       EPI_PART  fp32 partial sums of a share of K
//   EPI_GATE   A holds two weights; h = act(g) u, and g, u if asked
//   EPI_GRAD   D = dh; from g and u: dg = dh u act'(g), du = dh act(g)
enum { EPI_STORE = 0, EPI_PART = 1, EPI_GATE = 2, EPI_GRAD = 3 };

struct Gemm {
  const uint16_t* A[2];
  const uint16_t* B[2];
  int64_t lda, ldb;          // row strides (elements) of the stored matrices
  int64_t M, N, K;           // K of one pair
  int pairs;                 // K runs over pairs * K
  int splits;                // shares of K (EPI_PART)
  int act;
  uint16_t* d0; uint16_t* d1; uint16_t* d2;   // STORE: D | GATE: h, g, u | GRAD: dg, du
  const uint16_t* s0; const uint16_t* s1;     // STORE: resid | GRAD: g, u
  float* part;
  int64_t ldd;
};

constexpr int BK = 64;

// A tile lies in LDS as 16-byte chunks, [row][chunk], the chunk's place XORed with a function of the
// row so that the lanes of a read phase fall on all banks (the direct loads write 1 KB of consecutive
// places; each lane fetches the chunk that belongs at its place):
//   KC: rows of 8 chunks.  A 16-row fragment takes rows 16 (i / 4) + 4 t + i % 4 of 64, so that a lane of
//       four fragments ends with 16 consecutive features; eight lanes of a phase, eight f.
//   MC: K rows of ROWS / 8 chunks, read transposed; 32 lanes of a phase read 32 bytes of 8 rows.
__device__ __forceinline__ int f_kc(int row) { return (row & 3) | (((row >> 4) & 1) << 2); }
__device__ __forceinline__ int f_mc(int k) { return 2 * ((k & 3) | (((k >> 3) & 1) << 2)); }

template <bool H, bool AMC, bool BMC, int EPI, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__((BM / WM) * (BN / WN) * 64) void gemm_kernel(Gemm p) {
  constexpr int WAVES = (BM / WM) * (BN / WN), MW = BM / WM;
  constexpr int MT = WM / 16, NT = WN / 16;
  constexpr int ABYTES = BM * BK * 2, BBYTES = BN * BK * 2, STAGE = ABYTES + BBYTES;
  constexpr int APW = ABYTES / 1024 / WAVES, BPW = BBYTES / 1024 / WAVES;
  static_assert(ABYTES % (1024 * WAVES) == 0 && BBYTES % (1024 * WAVES) == 0, "whole loads per wave");
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, w = uniform(tid >> 6);
  const int i = lane & 15, q = lane >> 4;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_byte*)smem;

  constexpr int FM = EPI == EPI_GATE ? BM / 2 : BM;       // features of a tile (of each weight)
  const int64_t mt = (p.M + FM - 1) / FM, nt = (p.N + BN - 1) / BN;
  // workgroup -> tile: workgroups are dealt to the 8 XCDs round robin; each XCD takes a run of the
  // tiles (features fastest), so that its L2 keeps the B rows of a run
  const int64_t tiles = mt * nt * p.splits;
  const int64_t per = (tiles + 7) / 8;
  const int64_t id = (int64_t)(blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if ((int64_t)(blockIdx.x >> 3) >= per || id >= tiles) return;
  const int64_t m0 = (id % mt) * FM, n0 = (id / mt % nt) * BN;
  const int split = (int)(id / (mt * nt));

  // K in tiles of BK; tile t belongs to pair t / kt
  const int kt = (int)((p.K + BK - 1) / BK), all = kt * p.pairs;
  const int t0 = (int)((int64_t)all * split / p.splits), t1 = (int)((int64_t)all * (split + 1) / p.splits);

  // the 1 KB loads of one operand tile; R: rows of the tile, `which`: whether the row is in range, and where
  auto stage = [&](int t, uint32_t base) {
    const int pr = t >= kt ? 1 : 0;
    const int64_t k0 = (int64_t)(t - pr * kt) * BK;
#pragma unroll
    for (int c = 0; c < APW + BPW; ++c) {
      const bool isA = c < APW;
      const int piece = isA ? w * APW + c : w * BPW + (c - APW);
      const int L = piece * 64 + lane;                     // 16-byte place in the operand's tile
      const uint32_t at = base + (isA ? 0 : ABYTES) + (uint32_t)piece * 1024;
      const uint16_t* src;
      if (isA ? AMC : BMC) {
        const int CH = (isA ? BM : BN) / 8, kr = L / CH, ch = (L % CH) ^ f_mc(kr);
        const int64_t k = k0 + kr, r = (isA ? m0 : n0) + ch * 8;
        const uint16_t* X = isA ? p.A[pr] : p.B[pr];
        src = k < p.K && r < (isA ? p.M : p.N) ? X + k * (isA ? p.lda : p.ldb) + r : (const uint16_t*)&zero16;
      } else {
        const int row = L / 8, ch = (L % 8) ^ f_kc(row);
        const int64_t k = k0 + ch * 8;
        const uint16_t* X = isA ? p.A[EPI == EPI_GATE ? (row >> 6) & 1 : pr] : p.B[pr];
        const int64_t r = isA ? (EPI == EPI_GATE ? m0 + (row >> 7) * 64 + (row & 63) : m0 + row) : n0 + row;
        src = k < p.K && r < (isA ? p.M : p.N) ? X + r * (isA ? p.lda : p.ldb) + k : (const uint16_t*)&zero16;
      }
      lds_load16(src, at);
    }
  };

  f32x4 acc[MT][NT];
#pragma unroll
  for (int a = 0; a < MT; ++a)
#pragma unroll
    for (int b = 0; b < NT; ++b) acc[a][b] = f32x4{0.f, 0.f, 0.f, 0.f};

  const int wm = (w % MW) * WM, wn = (w / MW) * WN;
  // fragment t of a 64-row span at row `r0` of an operand's tile, K step ks
  auto frag_kc = [&](const unsigned char* s, int r0, int t, int ks) {
    const int row = r0 + (t >> 2) * 64 + 16 * (i >> 2) + 4 * (t & 3) + (i & 3);
    return *reinterpret_cast<const u32x4*>(s + row * 128 + (((ks * 4 + q) ^ f_kc(row)) << 4));
  };
  auto frag_mc = [&](const unsigned char* s, int r0, int t, int ks, int rows) {
    const int k = ks * 32 + 8 * q + (i >> 2);
    const int ch = (r0 + 16 * t) / 8 + ((i & 3) >> 1);
    const unsigned char* a = s + (k * (rows / 8) + (ch ^ f_mc(k))) * 16 + (i & 1) * 8;
    const unsigned char* b = s + ((k + 4) * (rows / 8) + (ch ^ f_mc(k + 4))) * 16 + (i & 1) * 8;
    const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_g*)(lds_byte*)a));
    const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_g*)(lds_byte*)b));
    return u32x4{lo[0], lo[1], hi[0], hi[1]};
  };
  // B rows of a KC operand in their own order: column i of fragment t is row 16 t + i
  auto frag_b = [&](const unsigned char* s, int t, int ks) {
    const int row = wn + 16 * t + i;
    return *reinterpret_cast<const u32x4*>(s + row * 128 + (((ks * 4 + q) ^ f_kc(row)) << 4));
  };

  if (t0 < t1) stage(t0, lds0);
  for (int t = t0; t < t1; ++t) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    const uint32_t cur = (uint32_t)((t - t0) & 1) * STAGE;
    if (t + 1 < t1) stage(t + 1, lds0 + (STAGE - cur));
    const unsigned char* sa = smem + cur;
    const unsigned char* sb = sa + ABYTES;
#pragma unroll
    for (int ks = 0; ks < BK / 32; ++ks) {
      u32x4 fb[NT];
#pragma unroll
      for (int b = 0; b < NT; ++b) fb[b] = BMC ? frag_mc(sb, wn, b, ks, BN) : frag_b(sb, b, ks);
#pragma unroll
      for (int a = 0; a < MT; ++a) {
        const u32x4 fa = AMC ? frag_mc(sa, wm, a, ks, BM) : frag_kc(sa, wm, a, ks);
#pragma unroll
        for (int b = 0; b < NT; ++b) acc[a][b] = Half<H>::mfma(fa, fb[b], acc[a][b]);
      }
    }
  }

  // lane (i, q) of acc[a][b]: column n = n0 + wn + 16 b + i; features from wm + 64 (a / 4) + 16 q + 4 (a % 4)
  // (KC) or wm + 16 a + 4 q (MC), four consecutive
#pragma unroll
  for (int b = 0; b < NT; ++b) {
    const int64_t n = n0 + wn + 16 * b + i;
    if (n >= p.N) continue;
    if constexpr (EPI == EPI_GATE) {
#pragma unroll
      for (int a = 0; a < MT / 2; ++a) {
        const int64_t f = m0 + wm / 2 + (a >> 2) * 64 + 16 * q + 4 * (a & 3);
        if (f >= p.M) continue;
        const f32x4 &g = acc[(a >> 2) * 8 + (a & 3)][b], &u = acc[(a >> 2) * 8 + 4 + (a & 3)][b];
        float h[4], gv[4], uv[4];
#pragma unroll
        for (int v = 0; v < 4; ++v) gv[v] = g[v], uv[v] = u[v], h[v] = act_f(g[v], p.act) * u[v];
        store4h<H>(p.d0 + n * p.ldd + f, h);
        if (p.d1) {
          store4h<H>(p.d1 + n * p.ldd + f, gv);
          store4h<H>(p.d2 + n * p.ldd + f, uv);
        }
      }
    } else {
#pragma unroll
      for (int a = 0; a < MT; ++a) {
        const int64_t f = m0 + wm + (AMC ? 16 * a + 4 * q : (a >> 2) * 64 + 16 * q + 4 * (a & 3));
        if (f >= p.M) continue;
        const int64_t at = n * p.ldd + f;
        float v[4] = {acc[a][b][0], acc[a][b][1], acc[a][b][2], acc[a][b][3]};
        if constexpr (EPI == EPI_PART) {
          *reinterpret_cast<f32x4*>(p.part + (int64_t)split * p.N * p.ldd + at) = acc[a][b];
        } else if constexpr (EPI == EPI_STORE) {
          if (p.s0) {
            float r[4];
            load4h<H>(p.s0 + at, r);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] += r[e];
          }
          store4h<H>(p.d0 + at, v);
        } else {
          float g[4], u[4], dg[4], du[4];
          load4h<H>(p.s0 + at, g);
          load4h<H>(p.s1 + at, u);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float ac, de;
            act_both(g[e], p.act, ac, de);
            dg[e] = v[e] * u[e] * de;
            du[e] = v[e] * ac;
          }
          store4h<H>(p.d0 + at, dg);
          store4h<H>(p.d1 + at, du);
        }
      }
    }
  }
}

template <bool H, bool AMC, bool BMC, int EPI, int BM, int BN, int WM, int WN>
int launch_tile(const Gemm& p, hipStream_t st) {
  constexpr int FM = EPI == EPI_GATE ? BM / 2 : BM;
  const int64_t tiles = (p.M + FM - 1) / FM * ((p.N + BN - 1) / BN) * p.splits;
  if (tiles == 0) return LBK_OK;
  const int64_t blocks = (tiles + 7) / 8 * 8;
  if (blocks > 0x3fffff) return LBK_ERR_TOO_LARGE;
  constexpr int lds = 2 * (BM + BN) * BK * 2;
  auto* k = gemm_kernel<H, AMC, BMC, EPI, BM, BN, WM, WN>;
  static std::atomic<uint64_t> done{0};
  if (lds > 65536 && set_lds_limit_once(reinterpret_cast<const void*>(k), lds, done) != 0) return LBK_ERR_LAUNCH;
  k<<<(unsigned)blocks, (BM / WM) * (BN / WN) * 64, lds, st>>>(p);
  return hipGetLastError() == hipSuccess ? LBK_OK : LBK_ERR_LAUNCH;
}

template <bool H, bool AMC, bool BMC, int EPI>
int launch_gemm(const Gemm& p, hipStream_t st) {
  if constexpr (EPI == EPI_GATE) return launch_tile<H, AMC, BMC, EPI, 128, 128, 128, 32>(p, st);
  else return launch_tile<H, AMC, BMC, EPI, 128, 128, 64, 64>(p, st);
}

Gemm operands(const void* A, int64_t lda, const void* B, int64_t ldb, int64_t M, int64_t N, int64_t K) {
  Gemm p{};
  p.A[0] = p.A[1] = static_cast<const uint16_t*>(A);
  p.B[0] = p.B[1] = static_cast<const uint16_t*>(B);
  p.lda = lda, p.ldb = ldb, p.M = M, p.N = N, p.K = K;
  p.pairs = p.splits = 1;
  return p;
}

struct GatedArgs {
  int64_t N, D, F;
  int act;
  const void *wg, *wu, *wd;
};

template <bool H>
int gated_fwd(const GatedArgs& a, const void* x, int residual, void* out, void* h, void* g, void* u, hipStream_t st) {
  Gemm p = operands(a.wg, a.D, x, a.D, a.F, a.N, a.D);
  p.A[1] = static_cast<const uint16_t*>(a.wu);
  p.act = a.act, p.ldd = a.F;
  p.d0 = static_cast<uint16_t*>(h), p.d1 = static_cast<uint16_t*>(g), p.d2 = static_cast<uint16_t*>(u);
  if (int s = launch_gemm<H, false, false, EPI_GATE>(p, st)) return s;
  Gemm d = operands(a.wd, a.F, h, a.F, a.D, a.N, a.F);
  d.ldd = a.D, d.d0 = static_cast<uint16_t*>(out), d.s0 = residual ? static_cast<const uint16_t*>(x) : nullptr;
  return launch_gemm<H, false, false, EPI_STORE>(d, st);
}

template <bool H>
int gated_bwd(const GatedArgs& a, const void* dy, const void* x, const void* g, const void* u, const void* h, int residual,
              void* dx, void* dwg, void* dwu, void* dwd, void* dg, void* du, hipStream_t st) {
  if (dx || dwg || dwu) {
    Gemm p = operands(a.wd, a.F, dy, a.D, a.F, a.N, a.D);
    p.act = a.act, p.ldd = a.F;
    p.d0 = static_cast<uint16_t*>(dg), p.d1 = static_cast<uint16_t*>(du);
    p.s0 = static_cast<const uint16_t*>(g), p.s1 = static_cast<const uint16_t*>(u);
    if (int s = launch_gemm<H, true, false, EPI_GRAD>(p, st)) return s;
  }
  if (dx) {
    Gemm p = operands(a.wg, a.D, dg, a.F, a.D, a.N, a.F);
    p.A[1] = static_cast<const uint16_t*>(a.wu), p.B[1] = static_cast<const uint16_t*>(du), p.pairs = 2;
    p.ldd = a.D, p.d0 = static_cast<uint16_t*>(dx), p.s0 = residual ? static_cast<const uint16_t*>(dy) : nullptr;
    if (int s = launch_gemm<H, true, false, EPI_STORE>(p, st)) return s;
  }
  const void* gr[2] = {dg, du};
  void* dw[2] = {dwg, dwu};
  for (int k = 0; k < 2; ++k)
    if (dw[k]) {
      Gemm p = operands(x, a.D, gr[k], a.F, a.D, a.F, a.N);
      p.ldd = a.D, p.d0 = static_cast<uint16_t*>(dw[k]);
      if (int s = launch_gemm<H, true, true, EPI_STORE>(p, st)) return s;
    }
  if (dwd) {
    Gemm p = operands(h, a.F, dy, a.D, a.F, a.D, a.N);
    p.ldd = a.F, p.d0 = static_cast<uint16_t*>(dwd);
    if (int s = launch_gemm<H, true, true, EPI_STORE>(p, st)) return s;
  }
  return LBK_OK;
}

inline bool a16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline hipStream_t S(void* s) { return reinterpret_cast<hipStream_t>(s); }
inline size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }

int check_gated(int32_t dtype, int32_t act, int64_t N, int32_t D, int32_t F) {
  if ((dtype != LBK_BF16 && dtype != LBK_FP16) || (act != LBK_SILU && act != LBK_GELU) || N < 0) return LBK_ERR_ARG;
  if (D <= 0 || F <= 0 || D % 8 || F % 8) return LBK_ERR_SHAPE;
  return N > ((int64_t)1 << 31) ? LBK_ERR_TOO_LARGE : LBK_OK;
}

}  // namespace
}  // namespace lbk

using namespace lbk;

extern "C" {

size_t lbk_gated_fwd_workspace_bytes(int64_t N, int32_t d_model, int32_t d_ff, int want_intermediates) {
  if (N <= 0 || d_model <= 0 || d_ff <= 0) return 0;
  return want_intermediates ? 0 : align256((size_t)N * d_ff * 2);
}

int lbk_gated_fwd(int32_t dtype, int32_t act, const void* x, int64_t N, int32_t d_model, int32_t d_ff,
                  const void* w_gate, const void* w_up, const void* w_down, int add_residual, void* out, void* h_out,
                  void* gate_pre_out, void* up_out, void* workspace, size_t workspace_bytes, void* stream) {
  if (int st = check_gated(dtype, act, N, d_model, d_ff)) return st;
  if (N == 0) return LBK_OK;
  if (!x || !w_gate || !w_up || !w_down || !out) return LBK_ERR_NULL;
  const bool inter = h_out || gate_pre_out || up_out;
  if (inter && (!h_out || !gate_pre_out || !up_out)) return LBK_ERR_NULL;
  for (const void* p : {x, w_gate, w_up, w_down, (const void*)out, (const void*)h_out, (const void*)gate_pre_out,
                        (const void*)up_out, (const void*)workspace})
    if (!a16(p)) return LBK_ERR_ALIGN;
  const size_t need = lbk_gated_fwd_workspace_bytes(N, d_model, d_ff, inter);
  if (need && (!workspace || workspace_bytes < need)) return LBK_ERR_WORKSPACE;
  const GatedArgs a{N, d_model, d_ff, act, w_gate, w_up, w_down};
  void* h = inter ? h_out : workspace;
  return dtype == LBK_FP16 ? gated_fwd<true>(a, x, add_residual, out, h, gate_pre_out, up_out, S(stream))
                           : gated_fwd<false>(a, x, add_residual, out, h, gate_pre_out, up_out, S(stream));
}

size_t lbk_gated_bwd_workspace_bytes(int64_t N, int32_t d_model, int32_t d_ff) {
  if (N <= 0 || d_model <= 0 || d_ff <= 0) return 0;
  return 2 * align256((size_t)N * d_ff * 2);
}

int lbk_gated_bwd(int32_t dtype, int32_t act, const void* grad_out, const void* x, const void* gate_pre,
                  const void* up_out, const void* h, int64_t N, int32_t d_model, int32_t d_ff, const void* w_gate,
                  const void* w_up, const void* w_down, int add_residual, void* dx, void* dw_gate, void* dw_up,
                  void* dw_down, void* workspace, size_t workspace_bytes, void* stream) {
  if (int st = check_gated(dtype, act, N, d_model, d_ff)) return st;
  if (!w_gate || !w_up || !w_down) return LBK_ERR_NULL;
  if (N > 0 && (!grad_out || !x || !gate_pre || !up_out || !h)) return LBK_ERR_NULL;
  for (const void* p : {grad_out, x, gate_pre, up_out, h, w_gate, w_up, w_down, (const void*)dx, (const void*)dw_gate,
                        (const void*)dw_up, (const void*)dw_down, (const void*)workspace})
    if (!a16(p)) return LBK_ERR_ALIGN;
  const size_t need = lbk_gated_bwd_workspace_bytes(N, d_model, d_ff);
  if (need && (!workspace || workspace_bytes < need)) return LBK_ERR_WORKSPACE;
  const GatedArgs a{N, d_model, d_ff, act, w_gate, w_up, w_down};
  void* dg = workspace;
  void* du = static_cast<char*>(workspace) + align256((size_t)N * d_ff * 2);
  return dtype == LBK_FP16
             ? gated_bwd<true>(a, grad_out, x, gate_pre, up_out, h, add_residual, dx, dw_gate, dw_up, dw_down, dg, du, S(stream))
             : gated_bwd<false>(a, grad_out, x, gate_pre, up_out, h, add_residual, dx, dw_gate, dw_up, dw_down, dg, du, S(stream));
}

}  // extern "C"
