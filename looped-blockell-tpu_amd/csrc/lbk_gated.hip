// lbk_gated.hip — the dense gated FFN, out = (act(x Wg^T) * (x Wu^T)) Wd^T (+ x), with its backward
// (gfx950, bf16 or fp16 MFMA, fp32 sums), and its entry points of include/lbk.h.
//
// Weights are dense Linear weights [out, in].  Six matrix products, all on one tiled kernel:
//   forward   g, u = x Wg^T, x Wu^T with h = act(g) u in the epilogue, and for the backward the factors
//             cg = u act'(g), cu = act(g);  out = h Wd^T (+ x)
//   backward  dh = dy Wd with dg = dh cg, du = dh cu in the epilogue;
//             dx = dg Wg + du Wu (+ dy) as one product over both;  dWg = dg^T x, dWu = du^T x, dWd = dy^T h
// h, dg and du are rounded to the inputs' type between the products: they are the matrix instructions' operands.
// cg and cu, which the forward makes from fp32 values, are kept in 24 bits.  In place of g and u they spare the
// backward's epilogue the activation.  Sums are fp32.
#include "lbk.h"
#include "lbk_device.h"
#include "lbk_gated_plan.h"
#include "lbk_internal.h"

#include <algorithm>
#include <type_traits>

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

// eight consecutive values
template <bool H>
__device__ __forceinline__ void unpack8h(const u32x4& w, float (&f)[8]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) f[2 * k] = Half<H>::lo(w[k]), f[2 * k + 1] = Half<H>::hi(w[k]);
}
template <bool H>
__device__ __forceinline__ void store4h(uint16_t* p, const float (&f)[4]) {
  *reinterpret_cast<u32x2*>(p) = u32x2{Half<H>::pack2(f[0], f[1]), Half<H>::pack2(f[2], f[3])};
}
template <bool H>
__device__ __forceinline__ void store8h(uint16_t* p, const float (&f)[8]) {
  *reinterpret_cast<u32x4*>(p) =
      u32x4{Half<H>::pack2(f[0], f[1]), Half<H>::pack2(f[2], f[3]), Half<H>::pack2(f[4], f[5]), Half<H>::pack2(f[6], f[7])};
}

// The factors that the forward keeps: fp32 rounded to 24 bits (sign, 8 bits of exponent, 15 of mantissa), the
// upper 2 bytes of all in one plane and the third bytes, `third` bytes on, in another.  In 16 bits they left the
// gradients 1.7 times as far off as the rounding of the results alone does, so 1.4 times (what is left is dg's and
// du's); a training step of 16384 tokens, 1024 / 4096, costs 4 % more by it, one of 4096 tokens 11 %.  One
// plane of 3-byte groups (24 bytes a lane) was much worse: 1560 against 1265 us.
// A factor is read by the backward only, and its larger plane goes past the caches, which keep h for the next
// product (1286 -> 1265 us; the third bytes lose by it: 1265 -> 1286, and so do dg and du, which the next products
// read).
__device__ __forceinline__ void store_factor8(uint8_t* p, int64_t third, const float (&f)[8]) {
  uint32_t b[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) b[k] = __float_as_uint(f[k]) + 0x80u;
  u32x4 hi;
  uint32_t t[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    hi[k] = __builtin_amdgcn_perm(b[2 * k + 1], b[2 * k], 0x07060302u);
    t[k] = __builtin_amdgcn_perm(b[2 * k + 1], b[2 * k], 0x0c0c0501u);
  }
  __builtin_nontemporal_store(hi, reinterpret_cast<u32x4*>(p));
  *reinterpret_cast<u32x2*>(p + third) = u32x2{t[0] | t[1] << 16, t[2] | t[3] << 16};
}
__device__ __forceinline__ void store_factor4(uint8_t* p, int64_t third, const float (&f)[4]) {
  uint32_t b[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) b[k] = __float_as_uint(f[k]) + 0x80u;
  *reinterpret_cast<u32x2*>(p) =
      u32x2{__builtin_amdgcn_perm(b[1], b[0], 0x07060302u), __builtin_amdgcn_perm(b[3], b[2], 0x07060302u)};
  *reinterpret_cast<uint32_t*>(p + third) =
      __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0501u) | __builtin_amdgcn_perm(b[3], b[2], 0x0c0c0501u) << 16;
}
struct Factor8 {
  u32x4 hi;
  u32x2 lo;
};
__device__ __forceinline__ Factor8 load_factor8(const uint8_t* p, int64_t third) {
  return {*reinterpret_cast<const u32x4*>(p), *reinterpret_cast<const u32x2*>(p + third)};
}
__device__ __forceinline__ void unpack_factor8(const Factor8& v, float (&f)[8]) {
  const u32x4& hi = v.hi;
  const u32x2& lo = v.lo;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t j = 2 * (k & 1), l = lo[k >> 1];      // zero, the third byte, the upper half
    f[2 * k] = __uint_as_float(__builtin_amdgcn_perm(hi[k], l, 0x0504000cu | j << 8));
    f[2 * k + 1] = __uint_as_float(__builtin_amdgcn_perm(hi[k], l, 0x0706000cu | (j + 1) << 8));
  }
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
//   EPI_GATE   A holds two weights; h = act(g) u, and cg, cu if asked
//   EPI_GRAD   D = dh; dg = dh cg, du = dh cu
// (the enumeration, BK and the choice of tiles: lbk_gated_plan.h)
struct Gemm {
  const uint16_t* A[2];
  const uint16_t* B[2];
  int64_t lda, ldb;          // row strides (elements) of the stored matrices
  int64_t M, N, K;           // K of one pair
  int pairs;                 // K runs over pairs * K
  int parts;                 // 2: two products of one A, with B[0] and B[1], results d0 and d1 (or both in part)
  int splits;                // shares of K (EPI_PART)
  int act;
  uint16_t* d0; uint16_t* d1;                 // STORE: D of each part | GATE: h | GRAD: dg, du
  uint8_t* c0; uint8_t* c1;                   // GATE (or NULL), GRAD: cg, cu
  const uint16_t* s0;                         // STORE: resid, or NULL
  float* part;
  int64_t ldd;
};

constexpr int KS = 32;       // K of a matrix instruction

// The 32 K of a step of an operand lie in LDS as 16-byte chunks whose place is XORed with a function of the row, so
// that the lanes of a read phase fall on all banks (the direct loads write 1 KB of consecutive places; each
// lane fetches the chunk that belongs at its place):
//   KC: [row][4 chunks], fragment t is rows 16 t + i.  A read phase is lanes 0 .. 3, 12 .. 15 and 20 .. 27 (or
//       the others) of a half-wave: rows of all four (row / 4) % 4, two each of two neighbouring chunks.
//   MC: [k][ROWS / 8 chunks], read transposed; 32 lanes of a phase read 32 bytes of 8 K rows.
__device__ __forceinline__ int f_kc(int row) { return -(row >> 2) & 3; }
__device__ __forceinline__ int f_mc(int k) { return 2 * ((k & 3) | (((k >> 3) & 1) << 2)); }

// The matrix row that row i of A's fragment t holds.  A lane (i, q) of the products' results holds rows 4 q ..
// + 3 of each fragment.  KC: with this order two fragments give 8 consecutive features, and the four q of a
// column 32; EPI_GATE: fragments 0 and 1 of four are gate's, 2 and 3 the same features of up.
template <bool GATE>
__device__ __forceinline__ int a_row(int t, int i) {
  return (GATE ? t >> 2 : t >> 1) * 32 + 8 * (i >> 2) + 4 * (t & 1) + (i & 3);
}

// MC fragments hold rows in their own order: fragments a and a + 1 of lane q = 0 .. 3 become 8 consecutive
// features, those of fragment a + (q & 1) from 8 (q / 2) on, by exchanging neighbouring rows of 16 lanes
__device__ __forceinline__ void pair_rows(const f32x4& x, const f32x4& y, float (&f)[8]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x[e]), __float_as_uint(y[e]), false, false);
    f[e] = __uint_as_float(s[0]);
    f[4 + e] = __uint_as_float(s[1]);
  }
}

// Output tiles of TILE x TILE, waves of TILE / 2 x 64.  Two K stages in LDS, of two steps each; a step's
// fragments are read while the step before is multiplied.  Workgroups are persistent, and the K stages of
// their output tiles form one stream of loads: the next output tile's are in flight during the epilogue.
// TAIL: K is no multiple of 64.
template <bool H, bool AMC, bool BMC, int EPI, int TILE, bool TAIL>
__global__ __launch_bounds__(TILE * 2, 2) void gemm_kernel(Gemm p) {
  constexpr int BM = TILE, BN = TILE, WAVES = TILE / 32;
  constexpr int WM = BM / 2, WN = 64, MT = WM / 16, NT = WN / 16;
  constexpr int ABYTES = BM * KS * 2, STEP = ABYTES + BN * KS * 2, STAGE = 2 * STEP;
  constexpr int PA = ABYTES / 1024 / WAVES, PB = PA, PIECES = PA + PB;             // 1 KB loads of a wave and step
  constexpr bool GATE = EPI == EPI_GATE;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, w = uniform(tid >> 6);
  const int i = lane & 15, q = lane >> 4;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_byte*)smem;

  constexpr int FM = GATE ? BM / 2 : BM;                        // features of a tile
  const int mt = (int)((p.M + FM - 1) / FM), nt1 = (int)((p.N + BN - 1) / BN), nt = nt1 * p.parts;
  const int tiles = mt * nt * p.splits;                         // < 2^30 (launch_tile)
  // workgroups are dealt to the 8 XCDs round robin; an XCD takes a run of the tiles, which go eight
  // columns at a time, so that the tiles in work on it share operand rows in its L2.  The eight runs begin at
  // different features of their columns, or all in work at a time would lie in one stretch of the results' rows,
  // whose stride puts it on part of the memory channels (a training step of 16384 tokens, 1024 / 4096: 1265 ->
  // 1210 us; of 8192, 2048 / 8192: 2150 -> 2055).
  const int per = (tiles + 7) / 8, xcd = (int)(blockIdx.x & 7), stride = (int)(gridDim.x >> 3);
  const int last = min((xcd + 1) * per, tiles);
  int id = xcd * per + (int)(blockIdx.x >> 3);
  if (id >= last) return;

  const int kt = (int)((p.K + BK - 1) / BK), all = kt * p.pairs;
  struct Where {
    int m0, n0, part, split, t0, t1;
  };
  auto where = [&](int idx) {
    Where v;
    v.split = idx / (mt * nt);
    const int r = idx - v.split * (mt * nt), ng = r / (mt * 8), rr = r - ng * mt * 8;
    const int wide = min(8, nt - ng * 8);
    const int turn = mt >= 8 ? (idx - rr) / per * (mt / 8) : 0;       // one for the whole group of columns
    v.m0 = uniform((rr / wide + turn) % mt * FM);
    const int c = ng * 8 + rr % wide;
    v.part = uniform(c >= nt1 ? 1 : 0);
    v.n0 = uniform((c - v.part * nt1) * BN);
    v.t0 = uniform((int)((int64_t)all * v.split / p.splits));
    v.t1 = uniform((int)((int64_t)all * (v.split + 1) / p.splits));
    return v;
  };

  // byte offsets of this lane's chunks from an output tile's first row (KC) or column (MC); rows behind the
  // matrix read its last row, and reach no output
  uint32_t aoff[PA], boff[PB];
  auto offsets = [&](const Where& v) {
    const int r4 = lane >> 2, ch = (lane & 3) ^ f_kc(lane >> 2);
#pragma unroll
    for (int c = 0; c < PA; ++c) {
      const int piece = w * PA + c;
      if constexpr (AMC) {
        const int kr = (piece * 64 + lane) / (BM / 8), r = ((lane % (BM / 8)) ^ f_mc(kr)) * 8;
        aoff[c] = (uint32_t)((kr * p.lda + min(r, (int)(p.M - 8 - v.m0))) * 2);
      } else {
        aoff[c] = (uint32_t)((min(a_row<GATE>(piece, r4), (int)(p.M - 1 - v.m0)) * p.lda + ch * 8) * 2);
      }
    }
#pragma unroll
    for (int c = 0; c < PB; ++c) {
      const int piece = w * PB + c;
      if constexpr (BMC) {
        const int kr = (piece * 64 + lane) / (BN / 8), r = ((lane % (BN / 8)) ^ f_mc(kr)) * 8;
        boff[c] = (uint32_t)((kr * p.ldb + min(r, (int)(p.N - 8 - v.n0))) * 2);
      } else {
        boff[c] = (uint32_t)((min(piece * 16 + r4, (int)(p.N - 1 - v.n0)) * p.ldb + ch * 8) * 2);
      }
    }
  };
  // the stream of loads: K stage lt of output tile lv; its bases, and how much of K is left there
  Where lv = where(id);
  int lid = id, lt = lv.t0, left = 0;
  const char *sa0 = nullptr, *sa1 = nullptr, *sb0 = nullptr;
  auto ptr = [](const uint16_t* b, int64_t elems) {
    const uint64_t v = reinterpret_cast<uint64_t>(b + elems);
    return reinterpret_cast<const char*>((uint64_t)(uint32_t)uniform((int)(uint32_t)v) |
                                         (uint64_t)(uint32_t)uniform((int)(uint32_t)(v >> 32)) << 32);
  };
  const int64_t da = AMC ? BK * 2 * p.lda : BK * 2, db = BMC ? BK * 2 * p.ldb : BK * 2;
  auto source = [&]() {
    const int pr = lt >= kt ? 1 : 0;
    const int64_t k0 = (int64_t)(lt - pr * kt) * BK;
    const int64_t ao = AMC ? k0 * p.lda + lv.m0 : lv.m0 * p.lda + k0, bo = BMC ? k0 * p.ldb + lv.n0 : lv.n0 * p.ldb + k0;
    sa0 = ptr(GATE || !pr ? p.A[0] : p.A[1], ao);
    if constexpr (GATE) sa1 = ptr(p.A[1], ao);
    sb0 = ptr(pr | lv.part ? p.B[1] : p.B[0], bo);
    left = (int)(p.K - k0);
    asm volatile("s_nop 4" : "+s"(sa0), "+s"(sa1), "+s"(sb0));      // wait states from readfirstlane to a load's base
  };
  auto advance = [&]() {                // behind the stream's end its last K stage is loaded again, for nobody
    ++lt;
    if (lt == lv.t1 || lt == kt) {
      if (lt == lv.t1) {
        if (lid + stride < last) {
          lid += stride;
          lv = where(lid);
          offsets(lv);
          lt = lv.t0;
        } else {
          --lt;
        }
      }
      source();
    } else {
      sa0 += da;
      sa1 += da;
      sb0 += db;
      left -= BK;
    }
  };
  // load c (0 .. 2 PIECES - 1) of the K stage at `base`: both steps' chunks of a row one after the other
  const int64_t ha = AMC ? KS * 2 * p.lda : KS * 2, hb = BMC ? KS * 2 * p.ldb : KS * 2;
  auto load = [&](uint32_t base, int c) {
    const int ks = c & 1, cp = c >> 1;
    const bool isA = cp < PA;
    const int cc = isA ? cp : cp - PA, piece = isA ? w * PA + cc : w * PB + cc;
    const uint32_t at = base + ks * STEP + (isA ? 0 : ABYTES) + (uint32_t)piece * 1024, off = isA ? aoff[cc] : boff[cc];
    // EPI_GATE: a load is a fragment's 16 rows, all of one weight
    const char* b = (!isA ? sb0 : GATE && (piece & 2) ? sa1 : sa0) + (ks ? (isA ? ha : hb) : 0);
    if constexpr (TAIL) {
      const int R = isA ? BM : BN;
      const int k = ks * KS + ((isA ? AMC : BMC) ? (piece * 64 + lane) / (R / 8) : ((lane & 3) ^ f_kc(lane >> 2)) * 8);
      lds_fetch16(k < left ? b + off : reinterpret_cast<const char*>(&zero16), at);
    } else {
      lds_fetch16(b, off, at);
    }
  };

  const int wm = (w & 1) * WM, wn = (w >> 1) * WN;
  // fragment addresses in a step: KC one (fragments are immediates), MC one a fragment
  uint32_t ra[AMC ? MT : 1], rb[BMC ? NT : 1];
#pragma unroll
  for (int t = 0; t < (AMC ? MT : 1); ++t)
    ra[t] = AMC ? (uint32_t)((8 * q + (i >> 2)) * (BM * 2) +
                             (((wm + 16 * t) / 8 + ((i & 3) >> 1)) ^ f_mc(8 * q + (i >> 2))) * 16 + (i & 1) * 8)
                : (uint32_t)((wm + i) * 64 + ((q ^ f_kc(i)) << 4));
#pragma unroll
  for (int t = 0; t < (BMC ? NT : 1); ++t)
    rb[t] = (uint32_t)ABYTES +
            (BMC ? (uint32_t)((8 * q + (i >> 2)) * (BN * 2) +
                              (((wn + 16 * t) / 8 + ((i & 3) >> 1)) ^ f_mc(8 * q + (i >> 2))) * 16 + (i & 1) * 8)
                 : (uint32_t)((wn + i) * 64 + ((q ^ f_kc(i)) << 4)));
  auto tr = [&](const unsigned char* s, int row) {
    const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_g*)(lds_byte*)s));
    const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_g*)(lds_byte*)(s + 4 * row)));
    return u32x4{lo[0], lo[1], hi[0], hi[1]};
  };
  auto frag_a = [&](const unsigned char* s, int t) {
    if constexpr (AMC) return tr(s + ra[t], BM * 2);
    else return *reinterpret_cast<const u32x4*>(s + ra[0] + t * 1024);
  };
  auto frag_b = [&](const unsigned char* s, int t) {
    if constexpr (BMC) return tr(s + rb[t], BN * 2);
    else return *reinterpret_cast<const u32x4*>(s + rb[0] + t * 1024);
  };

  offsets(lv);
  source();
#pragma unroll
  for (int st = 0; st < 2; ++st) {
#pragma unroll
    for (int c = 0; c < 2 * PIECES; ++c) load(lds0 + st * STAGE, c);
    advance();
  }
  f32x4 acc[MT][NT];
  auto clear = [&]() {
#pragma unroll
    for (int a = 0; a < MT; ++a)
#pragma unroll
      for (int b = 0; b < NT; ++b) acc[a][b] = f32x4{0.f, 0.f, 0.f, 0.f};
  };
  clear();
  u32x4 fa[2][MT], fb[2][NT];
  asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(2 * PIECES) : "memory");
#pragma unroll
  for (int b = 0; b < NT; ++b) fb[0][b] = frag_b(smem, b);
#pragma unroll
  for (int a = 0; a < MT; ++a) fa[0][a] = frag_a(smem, a);
  // a step's products, the next step's fragments read beside the first of them; the order is pinned, or the
  // compiler gathers the reads behind the products and waits for them
  auto step = [&](auto set, const unsigned char* next, auto&& beside) {
    constexpr int c = decltype(set)::value, n = 1 - c;
#pragma unroll
    for (int a = 0; a < MT; ++a) {
      beside(a);
      if (a < NT) fb[n][a] = frag_b(next, a);
      if (2 * a < MT) {
        fa[n][2 * a] = frag_a(next, 2 * a);
        fa[n][2 * a + 1] = frag_a(next, 2 * a + 1);
      }
#pragma unroll
      for (int b = 0; b < NT; ++b) acc[a][b] = Half<H>::mfma(fa[c][a], fb[c][b], acc[a][b]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  Where done = where(id);
  uint32_t cur = 0;                     // the stage in work
  for (int t = done.t0;;) {
    step(std::integral_constant<int, 0>{}, smem + cur + STEP, [](int) {});
    // the stage is read, and the next one has landed, for every wave
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    step(std::integral_constant<int, 1>{}, smem + (STAGE - cur), [&](int a) {
#pragma unroll
      for (int c = 0; c < 2 * PIECES / MT; ++c) load(lds0 + cur, a * (2 * PIECES / MT) + c);
    });
    cur = STAGE - cur;
    advance();
    if (++t < done.t1) continue;

    // column n of lane (i, q), features f .. f + 7 of two fragments (EPI_GATE: of two of each weight)
    const int64_t f0 = done.m0 + (GATE ? wm / 2 : wm) + (AMC ? 16 * (q & 1) + 8 * (q >> 1) : 8 * q);
#pragma unroll
    for (int b = 0; b < NT; ++b) {
      __builtin_amdgcn_sched_barrier(0);      // or the columns' loads are gathered, and registers spill
      const int64_t n = done.n0 + wn + 16 * b + i;
      const bool in_n = n < p.N;
      if constexpr (GATE) {
        if (!in_n) continue;
#pragma unroll
        for (int a = 0; a < MT; a += 4) {
          const int64_t f = f0 + a * 8, at = n * p.ldd + f, third = 2 * p.N * p.ldd - at;
          if (f >= p.M) continue;
          float h[8], cg[8], cu[8];
          if (p.c0) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float g = acc[a + (e >> 2)][b][e & 3], u = acc[a + 2 + (e >> 2)][b][e & 3];
              float d;
              act_both(g, p.act, cu[e], d);
              h[e] = cu[e] * u;
              cg[e] = u * d;
            }
            store_factor8(p.c0 + 2 * at, third, cg);
            store_factor8(p.c1 + 2 * at, third, cu);
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              h[e] = act_f(acc[a + (e >> 2)][b][e & 3], p.act) * acc[a + 2 + (e >> 2)][b][e & 3];
          }
          store8h<H>(p.d0 + at, h);
        }
      } else {
        constexpr int AHEAD = EPI == EPI_GRAD ? 2 : 1;
        Factor8 r0[AHEAD], r1[AHEAD];
#pragma unroll
        for (int a = 0; a < MT; a += 2) {
          // the factors of two groups together, ahead of the stores that loads wait behind (16384 x 4096, K 1024: 303 ->
          // 281 us; of four, with spilled registers, 343)
          if (EPI == EPI_GRAD && a / 2 % AHEAD == 0) {
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) {
              const int64_t at = min(n, p.N - 1) * p.ldd + min(f0 + (a + 2 * k) * 16, p.M - 8), third = 2 * p.N * p.ldd - at;
              r0[k] = load_factor8(p.c0 + 2 * at, third);
              r1[k] = load_factor8(p.c1 + 2 * at, third);
            }
          }
          float x[8];
          if constexpr (AMC) {
            pair_rows(acc[a][b], acc[a + 1][b], x);       // all lanes take part
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = acc[a + (e >> 2)][b][e & 3];
          }
          const int64_t f = f0 + a * 16, at = n * p.ldd + f;
          if (!in_n || f >= p.M) continue;
          if constexpr (EPI == EPI_PART) {
            float* d = p.part + (int64_t)(done.split * p.parts + done.part) * p.N * p.ldd + at;
            *reinterpret_cast<f32x4*>(d) = f32x4{x[0], x[1], x[2], x[3]};
            *reinterpret_cast<f32x4*>(d + 4) = f32x4{x[4], x[5], x[6], x[7]};
          } else if constexpr (EPI == EPI_STORE) {
            if (p.s0) {
              float r[8];
              unpack8h<H>(*reinterpret_cast<const u32x4*>(p.s0 + at), r);
#pragma unroll
              for (int e = 0; e < 8; ++e) x[e] += r[e];
            }
            store8h<H>((done.part ? p.d1 : p.d0) + at, x);
          } else {
            float dg[8], du[8];
            unpack_factor8(r0[a / 2 % AHEAD], dg);
            unpack_factor8(r1[a / 2 % AHEAD], du);
#pragma unroll
            for (int e = 0; e < 8; ++e) dg[e] *= x[e], du[e] *= x[e];
            store8h<H>(p.d0 + at, dg);
            store8h<H>(p.d1 + at, du);
          }
        }
      }
    }
    id += stride;
    if (id >= last) break;
    done = where(id);
    t = done.t0;
    clear();
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");      // the loads behind the stream's end
}

// gradients of no tokens: the tiled product needs a K of 1 and more
__global__ __launch_bounds__(256) void zero_kernel(u32x4* __restrict__ p, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) p[i] = u32x4{0, 0, 0, 0};
}

// ------------------------------------------------------------------ few tokens
// D of up to 16 NT columns (tokens) where A is KC: the weights are streamed once.  A workgroup makes 16
// features (GATE: of both weights), its waves take K in turns of 64 (128 bytes of a row), U turns on their way;
// the waves' sums meet in LDS and are added in their order.
// EIGHT (up to 8 columns): 8 features, rows and columns 8 .. 15 of the matrix instructions taking the next 64 K
// of the same features and tokens, so that twice the workgroups stream with whole loads.
// HBM-bound: 1 token, 2048 / 8192, 100 MB of weights: 143 us on the tiled kernel, 25 so.
template <bool H, bool GATE, int NT, int NW, bool EIGHT>
__global__ __launch_bounds__(NW * 64) void skinny_kernel(Gemm p) {
  constexpr int MATS = GATE ? 2 : 1, ROWS = EIGHT ? 8 : 16, TURN = EIGHT ? 128 : 64;
  constexpr int U = NT == 1 ? 4 : 2;
  static_assert(!EIGHT || NT == 1, "one tile");
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  f32x4* part = reinterpret_cast<f32x4*>(smem);                 // [NW][MATS][NT][64]
  const int tid = threadIdx.x, lane = tid & 63, w = uniform(tid >> 6), i = lane & 15, q = lane >> 4;
  const int ii = EIGHT ? i & 7 : i, k0 = 16 * q + (EIGHT ? (i >> 3) * 64 : 0);
  const int64_t f0 = (int64_t)blockIdx.x * ROWS;
  const int S = (int)((p.K + TURN - 1) / TURN);
  const uint16_t *wp[MATS], *xp[NT];
#pragma unroll
  for (int m = 0; m < MATS; ++m) wp[m] = p.A[m] + min(f0 + ii, p.M - 1) * p.lda + k0;
#pragma unroll
  for (int b = 0; b < NT; ++b) xp[b] = p.B[0] + min((int64_t)(16 * b + ii), p.N - 1) * p.ldb + k0;
  f32x4 acc[MATS][NT] = {};
  for (int s0 = w; s0 < S; s0 += NW * U) {
    u32x4 wv[U][MATS][2], xv[U][NT][2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = s0 + u * NW;
      if (s >= S) break;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const bool in = (int64_t)s * TURN + k0 + 8 * c < p.K;   // K is a multiple of 8
        const int64_t at = (int64_t)s * TURN + 8 * c;
#pragma unroll
        for (int m = 0; m < MATS; ++m)
          wv[u][m][c] = in ? *reinterpret_cast<const u32x4*>(wp[m] + at) : u32x4{0, 0, 0, 0};
#pragma unroll
        for (int b = 0; b < NT; ++b) xv[u][b][c] = in ? *reinterpret_cast<const u32x4*>(xp[b] + at) : u32x4{0, 0, 0, 0};
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s0 + u * NW >= S) break;
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int m = 0; m < MATS; ++m)
#pragma unroll
          for (int b = 0; b < NT; ++b) acc[m][b] = Half<H>::mfma(wv[u][m][c], xv[u][b][c], acc[m][b]);
    }
  }
  auto slot = [&](int wave, int m, int b) { return ((wave * MATS + m) * NT + b) * 64 + lane; };
#pragma unroll
  for (int m = 0; m < MATS; ++m)
#pragma unroll
    for (int b = 0; b < NT; ++b) part[slot(w, m, b)] = acc[m][b];
  __syncthreads();
  if (w >= NT) return;
  // wave w: columns 16 w + i, features f .. f + 3
  if (EIGHT && (i >= 8 || q >= 2)) return;
  const int64_t n = 16 * w + i, f = f0 + 4 * q, at = n * p.ldd + f;
  f32x4 v[MATS] = {};
#pragma unroll
  for (int s = 0; s < NW; ++s)
#pragma unroll
    for (int m = 0; m < MATS; ++m) {
      v[m] += part[slot(s, m, w)];
      if constexpr (EIGHT) v[m] += part[slot(s, m, w) + 8 + 32];      // rows and columns 8 further on
    }
  if (n >= p.N || f >= p.M) return;
  float x[4] = {v[0][0], v[0][1], v[0][2], v[0][3]};
  if constexpr (GATE) {
    float cg[4], cu[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float d;
      act_both(x[e], p.act, cu[e], d);
      cg[e] = v[1][e] * d;
      x[e] = cu[e] * v[1][e];
    }
    if (p.c0) {
      store_factor4(p.c0 + 2 * at, 2 * p.N * p.ldd - at, cg);
      store_factor4(p.c1 + 2 * at, 2 * p.N * p.ldd - at, cu);
    }
  } else if (p.s0) {
    const u32x2 t = *reinterpret_cast<const u32x2*>(p.s0 + at);
    x[0] += Half<H>::lo(t[0]), x[1] += Half<H>::hi(t[0]), x[2] += Half<H>::lo(t[1]), x[3] += Half<H>::hi(t[1]);
  }
  store4h<H>(p.d0 + at, x);
}

template <bool H, bool GATE, int NT, int NW, bool EIGHT = false>
int launch_skinny_t(const Gemm& p, hipStream_t st) {
  constexpr int lds = NW * (GATE ? 2 : 1) * NT * 64 * 16, rows = EIGHT ? 8 : 16;
  static_assert(lds <= 65536, "within the default limit");
  skinny_kernel<H, GATE, NT, NW, EIGHT><<<(unsigned)((p.M + rows - 1) / rows), NW * 64, lds, st>>>(p);
  return hipGetLastError() == hipSuccess ? LBK_OK : LBK_ERR_LAUNCH;
}
template <bool H, bool GATE>
int launch_skinny(const Gemm& p, hipStream_t st) {
  const bool few = p.M < 256 * 16;          // fewer workgroups of 16 features than CUs
  if (p.N <= 8 && few) return launch_skinny_t<H, GATE, 1, 16, true>(p, st);
  if (p.N <= 16) return few ? launch_skinny_t<H, GATE, 1, 16>(p, st) : launch_skinny_t<H, GATE, 1, 8>(p, st);
  return few ? launch_skinny_t<H, GATE, 2, 16>(p, st) : launch_skinny_t<H, GATE, 2, 8>(p, st);
}

// The partial products of the shares of K, summed in their order, + resid, rounded; `total` elements of each
// of `parts` results.  HBM-bound (or the memory-side cache's).
template <bool H>
__global__ __launch_bounds__(256) void reduce_kernel(const float* __restrict__ part, int splits, int parts, int64_t total,
                                                     const uint16_t* __restrict__ resid, uint16_t* __restrict__ d0,
                                                     uint16_t* __restrict__ d1) {
  const int64_t all = total * parts, step = (int64_t)gridDim.x * 256 * 8;
  for (int64_t e0 = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8; e0 < all; e0 += step) {
    float x[8] = {};
    for (int s = 0; s < splits; ++s) {
      const f32x4 *p = reinterpret_cast<const f32x4*>(part + s * all + e0), v = p[0], u = p[1];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] += v[e], x[4 + e] += u[e];
    }
    const bool second = e0 >= total;
    const int64_t at = second ? e0 - total : e0;
    if (resid) {
      float r[8];
      unpack8h<H>(*reinterpret_cast<const u32x4*>(resid + at), r);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] += r[e];
    }
    store8h<H>((second ? d1 : d0) + at, x);
  }
}

size_t part_bytes(int64_t M, int64_t N, int64_t K, int parts) {
  const Plan p = plan(M, N, K, parts, EPI_PART, true);
  return p.splits > 1 ? (size_t)M * N * parts * p.splits * 4 : 0;
}

// of the forward's second product
size_t down_part_bytes(int64_t N, int64_t D, int64_t F) { return skinny(N, D, F) ? 0 : part_bytes(D, N, F, 1); }

template <bool H, bool AMC, bool BMC, int EPI, int TILE, bool TAIL>
int launch_tile(const Gemm& p, hipStream_t st) {
  constexpr int FM = EPI == EPI_GATE ? TILE / 2 : TILE;
  const int64_t tiles = (p.M + FM - 1) / FM * ((p.N + TILE - 1) / TILE) * p.parts * p.splits;
  if (tiles == 0) return LBK_OK;
  // every share of K holds a K stage: the kernel's stream of loads counts on it
  if (p.K < 1 || p.splits > (p.K + BK - 1) / BK * p.pairs) return LBK_ERR_ARG;
  if (tiles > 0x3fffffff) return LBK_ERR_TOO_LARGE;
  // workgroups that run at once, all XCDs alike
  const int64_t most = TILE == 256 ? 256 : 512, blocks = tiles >= most ? most : (tiles + 7) / 8 * 8;
  constexpr int lds = 2 * 2 * TILE * BK * 2;
  auto* k = gemm_kernel<H, AMC, BMC, EPI, TILE, TAIL>;
  static std::atomic<uint64_t> done{0};
  if (lds > 65536 && set_lds_limit_once(reinterpret_cast<const void*>(k), lds, done) != 0) return LBK_ERR_LAUNCH;
  k<<<(unsigned)blocks, TILE * 2, lds, st>>>(p);
  return hipGetLastError() == hipSuccess ? LBK_OK : LBK_ERR_LAUNCH;
}

template <bool H, bool AMC, bool BMC, int EPI>
int launch_gemm(const Gemm& p, int tile, hipStream_t st) {
  if (p.K % BK) return tile == 256 ? launch_tile<H, AMC, BMC, EPI, 256, true>(p, st) : launch_tile<H, AMC, BMC, EPI, 128, true>(p, st);
  return tile == 256 ? launch_tile<H, AMC, BMC, EPI, 256, false>(p, st) : launch_tile<H, AMC, BMC, EPI, 128, false>(p, st);
}

// EPI_STORE, whole or in shares of K by way of `part`
template <bool H, bool AMC, bool BMC>
int store_gemm(Gemm p, float* part, hipStream_t st) {
  const Plan pl = plan(p.M, p.N, p.K * p.pairs, p.parts, EPI_PART, part != nullptr);
  if (pl.splits == 1) return launch_gemm<H, AMC, BMC, EPI_STORE>(p, pl.tile, st);
  p.splits = pl.splits;
  p.part = part;
  if (int s = launch_gemm<H, AMC, BMC, EPI_PART>(p, pl.tile, st)) return s;
  const int64_t total = p.N * p.ldd, threads = (total * p.parts / 8 + 255) / 256;
  reduce_kernel<H><<<(unsigned)(threads < 2048 ? threads : 2048), 256, 0, st>>>(part, pl.splits, p.parts, total, p.s0, p.d0, p.d1);
  return hipGetLastError() == hipSuccess ? LBK_OK : LBK_ERR_LAUNCH;
}

Gemm operands(const void* A, int64_t lda, const void* B, int64_t ldb, int64_t M, int64_t N, int64_t K) {
  Gemm p{};
  p.A[0] = p.A[1] = static_cast<const uint16_t*>(A);
  p.B[0] = p.B[1] = static_cast<const uint16_t*>(B);
  p.lda = lda, p.ldb = ldb, p.M = M, p.N = N, p.K = K;
  p.pairs = p.parts = p.splits = 1;
  return p;
}

struct GatedArgs {
  int64_t N, D, F;
  int act;
  const void *wg, *wu, *wd;
};

template <bool H>
int gated_fwd(const GatedArgs& a, const void* x, int residual, void* out, void* h, uint8_t* cg, uint8_t* cu, float* part,
              hipStream_t st) {
  Gemm p = operands(a.wg, a.D, x, a.D, a.F, a.N, a.D);
  p.A[1] = static_cast<const uint16_t*>(a.wu);
  p.act = a.act, p.ldd = a.F;
  p.d0 = static_cast<uint16_t*>(h), p.c0 = cg, p.c1 = cu;
  if (int s = skinny(a.N, a.D, a.F) ? launch_skinny<H, true>(p, st)
                             : launch_gemm<H, false, false, EPI_GATE>(p, plan(p.M, p.N, p.K, 1, EPI_GATE, false).tile, st))
    return s;
  Gemm d = operands(a.wd, a.F, h, a.F, a.D, a.N, a.F);
  d.ldd = a.D, d.d0 = static_cast<uint16_t*>(out), d.s0 = residual ? static_cast<const uint16_t*>(x) : nullptr;
  return skinny(a.N, a.D, a.F) ? launch_skinny<H, false>(d, st) : store_gemm<H, false, false>(d, part, st);
}

template <bool H>
int gated_bwd(const GatedArgs& a, const void* dy, const void* x, const uint8_t* cg, const uint8_t* cu, const void* h, int residual,
              void* dx, void* dwg, void* dwu, void* dwd, void* dg, void* du, float* part, hipStream_t st) {
  if (a.N == 0) {
    for (void* d : {dwg, dwu, dwd})
      if (d) zero_kernel<<<256, 256, 0, st>>>(static_cast<u32x4*>(d), a.D * a.F / 8);
    return hipGetLastError() == hipSuccess ? LBK_OK : LBK_ERR_LAUNCH;
  }
  if (dx || dwg || dwu) {
    Gemm p = operands(a.wd, a.F, dy, a.D, a.F, a.N, a.D);
    p.ldd = a.F;
    p.d0 = static_cast<uint16_t*>(dg), p.d1 = static_cast<uint16_t*>(du);
    p.c0 = const_cast<uint8_t*>(cg), p.c1 = const_cast<uint8_t*>(cu);      // read
    if (int s = launch_gemm<H, true, false, EPI_GRAD>(p, plan(p.M, p.N, p.K, 1, EPI_GRAD, false).tile, st)) return s;
  }
  if (dx) {
    Gemm p = operands(a.wg, a.D, dg, a.F, a.D, a.N, a.F);
    p.A[1] = static_cast<const uint16_t*>(a.wu), p.B[1] = static_cast<const uint16_t*>(du), p.pairs = 2;
    p.ldd = a.D, p.d0 = static_cast<uint16_t*>(dx), p.s0 = residual ? static_cast<const uint16_t*>(dy) : nullptr;
    if (int s = store_gemm<H, true, false>(p, part, st)) return s;
  }
  if (dwg || dwu) {
    // one launch for both, which share x, where both are wanted
    Gemm p = operands(x, a.D, dwg ? dg : du, a.F, a.D, a.F, a.N);
    p.ldd = a.D, p.d0 = static_cast<uint16_t*>(dwg ? dwg : dwu), p.parts = dwg && dwu ? 2 : 1;
    p.B[1] = static_cast<const uint16_t*>(du), p.d1 = static_cast<uint16_t*>(dwu);
    if (int s = store_gemm<H, true, true>(p, part, st)) return s;
  }
  if (dwd) {
    Gemm p = operands(h, a.F, dy, a.D, a.F, a.D, a.N);
    p.ldd = a.F, p.d0 = static_cast<uint16_t*>(dwd);
    if (int s = store_gemm<H, true, true>(p, part, st)) return s;
  }
  return LBK_OK;
}

inline bool a16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline hipStream_t S(void* s) { return reinterpret_cast<hipStream_t>(s); }
inline size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }

int check_gated(int32_t dtype, int32_t act, int64_t N, int32_t D, int32_t F) {
  if ((dtype != LBK_BF16 && dtype != LBK_FP16) || (act != LBK_SILU && act != LBK_GELU) || N < 0) return LBK_ERR_ARG;
  if (D <= 0 || F <= 0 || D % 8 || F % 8) return LBK_ERR_SHAPE;
  // row and column numbers are 32-bit, and so are the byte offsets within a tile's rows
  return N > 0x7ffffe00 || D > (1 << 22) || F > (1 << 22) ? LBK_ERR_TOO_LARGE : LBK_OK;
}

}  // namespace
}  // namespace lbk

using namespace lbk;

extern "C" {

size_t lbk_gated_fwd_workspace_bytes(int64_t N, int32_t d_model, int32_t d_ff, int want_intermediates) {
  if (N <= 0 || d_model <= 0 || d_ff <= 0) return 0;
  return (want_intermediates ? 0 : align256((size_t)N * d_ff * 2)) + down_part_bytes(N, d_model, d_ff);
}

int lbk_gated_fwd(int32_t dtype, int32_t act, const void* x, int64_t N, int32_t d_model, int32_t d_ff,
                  const void* w_gate, const void* w_up, const void* w_down, int add_residual, void* out, void* h_out,
                  uint8_t* gate_factor_out, uint8_t* up_factor_out, void* workspace, size_t workspace_bytes, void* stream) {
  if (int st = check_gated(dtype, act, N, d_model, d_ff)) return st;
  if (N == 0) return LBK_OK;
  if (!x || !w_gate || !w_up || !w_down || !out) return LBK_ERR_NULL;
  const bool inter = h_out || gate_factor_out || up_factor_out;
  if (inter && (!h_out || !gate_factor_out || !up_factor_out)) return LBK_ERR_NULL;
  for (const void* p : {x, w_gate, w_up, w_down, (const void*)out, (const void*)h_out, (const void*)gate_factor_out,
                        (const void*)up_factor_out, (const void*)workspace})
    if (!a16(p)) return LBK_ERR_ALIGN;
  const size_t need = lbk_gated_fwd_workspace_bytes(N, d_model, d_ff, inter);
  if (need && (!workspace || workspace_bytes < need)) return LBK_ERR_WORKSPACE;
  const GatedArgs a{N, d_model, d_ff, act, w_gate, w_up, w_down};
  void* h = inter ? h_out : workspace;
  float* part = down_part_bytes(N, d_model, d_ff)
                    ? reinterpret_cast<float*>(static_cast<char*>(workspace) + (inter ? 0 : align256((size_t)N * d_ff * 2)))
                    : nullptr;
  return dtype == LBK_FP16 ? gated_fwd<true>(a, x, add_residual, out, h, gate_factor_out, up_factor_out, part, S(stream))
                           : gated_fwd<false>(a, x, add_residual, out, h, gate_factor_out, up_factor_out, part, S(stream));
}

size_t lbk_gated_bwd_workspace_bytes(int64_t N, int32_t d_model, int32_t d_ff) {
  if (N <= 0 || d_model <= 0 || d_ff <= 0) return 0;
  const size_t parts[] = {part_bytes(d_model, N, 2 * (int64_t)d_ff, 1), part_bytes(d_model, d_ff, N, 2),
                          part_bytes(d_model, d_ff, N, 1), part_bytes(d_ff, d_model, N, 1)};
  return 2 * align256((size_t)N * d_ff * 2) + *std::max_element(parts, parts + 4);
}

int lbk_gated_bwd(int32_t dtype, const void* grad_out, const void* x, const uint8_t* gate_factor,
                  const uint8_t* up_factor, const void* h, int64_t N, int32_t d_model, int32_t d_ff, const void* w_gate,
                  const void* w_up, const void* w_down, int add_residual, void* dx, void* dw_gate, void* dw_up,
                  void* dw_down, void* workspace, size_t workspace_bytes, void* stream) {
  if (int st = check_gated(dtype, LBK_SILU, N, d_model, d_ff)) return st;
  if (!w_gate || !w_up || !w_down) return LBK_ERR_NULL;
  if (N > 0 && (!grad_out || !x || !gate_factor || !up_factor || !h)) return LBK_ERR_NULL;
  for (const void* p : {grad_out, x, (const void*)gate_factor, (const void*)up_factor, h, w_gate, w_up, w_down, (const void*)dx, (const void*)dw_gate,
                        (const void*)dw_up, (const void*)dw_down, (const void*)workspace})
    if (!a16(p)) return LBK_ERR_ALIGN;
  const size_t need = lbk_gated_bwd_workspace_bytes(N, d_model, d_ff);
  if (need && (!workspace || workspace_bytes < need)) return LBK_ERR_WORKSPACE;
  const GatedArgs a{N, d_model, d_ff, LBK_SILU, w_gate, w_up, w_down};
  void* dg = workspace;
  void* du = static_cast<char*>(workspace) + align256((size_t)N * d_ff * 2);
  float* part = reinterpret_cast<float*>(static_cast<char*>(du) + align256((size_t)N * d_ff * 2));
  return dtype == LBK_FP16
             ? gated_bwd<true>(a, grad_out, x, gate_factor, up_factor, h, add_residual, dx, dw_gate, dw_up, dw_down, dg, du, part, S(stream))
             : gated_bwd<false>(a, grad_out, x, gate_factor, up_factor, h, add_residual, dx, dw_gate, dw_up, dw_down, dg, du, part, S(stream));
}

}  // extern "C"
