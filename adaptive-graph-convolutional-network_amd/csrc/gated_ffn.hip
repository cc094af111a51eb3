// Gated feed-forward block over node rows (beside DenseMol, models/layers/dense_layer.py:33-50, one product without a gate):
//     G = X Wg, U = X Wu, A = act(G) (.) U, Y = A Wd            X [M, Fin], Wg, Wu [Fin, H], Wd [H, Fout]
//     dA = dY Wd^T;  dG = dA (.) U (.) act'(G);  dU = dA (.) act(G)
//     dX = dG Wg^T + dU Wu^T;  dWg = X^T dG;  dWu = X^T dU;  dWd = A^T dY
// Bound by the matrix pipe (18 M F H operations a training pass), for few rows by the weights' bytes.  Everything is one tiled
// product kernel on v_mfma_f32_16x16x32_bf16 with fp32 accumulators:
//   * Both projections share one pass over X: a workgroup's tile holds the same columns of Wg and Wu, so that the gate and its
//     partner meet in one lane's registers and the epilogue writes A (and, for a backward, P = U act'(G) and Q = act(G)).  dA never
//     reaches memory either: its epilogue reads P and Q and writes dG = dA P and dU = dA Q.  dX is one product over 2 H, dWg and
//     dWu share X's tiles.
//   * fp32 operands are split exactly into three bf16 pieces (bf16_split.h), and a product is the sum of six piece products (the
//     dropped ones are below 2^-24).  Much work: planes of pieces in memory, a stage holds the three of both operands, and every
//     fragment read serves two products.  Few rows or little work: fp32 in memory and LDS, split in registers.
//   * Tiles go from memory to LDS directly (buffer_load .. lds, 16 bytes per lane), in two or three stages.  An operand whose rows
//     run along k is read back with ds_read_b128, one whose rows run across k (weights in X W, both operands in X^T dG) with the
//     transposing ds_read_b64_tr_b16: nothing is transposed in memory.  The 16-byte chunks of a tile row are permuted (xor with
//     row bits) so that the lanes of a read hit different banks; the permutation is in the GLOBAL addresses, the LDS image being
//     linear.  Rows, columns and k beyond the operand read as zeros (the buffer's own bound).
//   * The accumulators leave through LDS, so that a lane gets eight neighbouring columns of one row: wide loads and stores, and
//     one small loop of epilogue code instead of one copy per fragment.
//   * Few tiles for the chip: the k loop is cut into splits whose fp32 tiles a second kernel adds in order (no atomics) and
//     puts through the same epilogue.
//   * One to four rows are bound by the weights' bytes: kernels of their own on the vector unit (ffn_rows_kernel).
//   * Features of at most 128, forward only: both products in one kernel, A stays in registers (ffn_fused_kernel).
// Roundings of bf16 calls: A, dG, dU are stored in bf16 for the products that read them (the matrix pipe takes bf16; calls with few
// elements of A keep a second piece); P and Q, which are only multiplied element by element, keep 24 bits (sign, exponent, 15
// bits of the mantissa: in bf16 they would add as much error to every gradient as dG's own rounding); sums, activations and their slopes are fp32.
#include <hip/hip_bf16.h>
#include <hip/hip_runtime.h>

#include <algorithm>

#include "bf16_split.h"
#include "gate_math.h"
#include "sgc_kernels.h"

namespace agcn {
namespace {
typedef uint32_t u32x4u __attribute__((ext_vector_type(4), aligned(4)));   // at the alignment of an element: unaligned access mode
typedef uint32_t u32x4h __attribute__((ext_vector_type(4), aligned(2)));
#define AGCN_LDS __attribute__((address_space(3)))

enum { EPI_GATED = 0, EPI_STORE = 1, EPI_DH = 2 };

// How operands lie in memory: bf16 matrices, three bf16 planes of an fp32 one, or fp32 matrices that are split on the way to the
// matrix pipe (few rows or little work: no launch for the planes, and a third of the bytes that they cost)
// (OP_WORDS: OP_FP32 whose rows do not start at 16 bytes or end in whole chunks; it is loaded into LDS four bytes a lane)
enum { OP_BF16 = 1, OP_FP32 = 2, OP_PLANES = 3, OP_WORDS = 4 };

struct Seg { const void *a, *b, *b2; };

struct GemmArgs {
  Seg seg[4];                        // the k loop runs over one to four products of the same sizes
  int32_t nseg;
  int32_t M, N, K;                   // N: columns of one B matrix (two B matrices: of each)
  int32_t lda, ldb;
  int64_t a_plane, b_plane;          // elements between the planes of pieces
  int32_t ktiles, tiles_m, tiles_n, splits;
  float* part;                       // splits > 1: [split][B matrix][M][ldp] fp32
  int32_t ldp;
  // epilogue
  int32_t act, f32, op, words;       // words: OP_FP32 as OP_WORDS
  int32_t two;                       // A, dG, dU in two bf16 pieces
  int32_t ldh;                       // leading dimension of P, Q, A, dG, dU
  int64_t plane;                     // elements between the planes of A, dG, dU
  void *out, *out2;                  // EPI_STORE: [M, ldo]
  int32_t ldo;
  void *p, *q;                       // U act'(G) and act(G): f32, or 24 bits: [M, ldh] upper sixteen, then [M, ldh] lower eight
  void *hid, *dg, *du;               // as the products read them (OP_*)
};

__device__ __forceinline__ uint32_t pk_bf(float a, float b) {
  return __builtin_bit_cast(uint32_t, (bf16x2){(__bf16)a, (__bf16)b});
}

// act(g) and act'(g).  The slopes are formed from e^-|g| (no 1 - s where s is near 1).  F32: within a few 2^-24 (gate_math.h; with
// gates() below 115 -> 93 us for a 32768 x 128 x 512 forward that called the library and branched for every value).  bf16 calls,
// whose results are rounded to eight bits: the hardware's exp2 and reciprocal as they are (a few 2^-24, and |g| 2^-23 from the exponent's rounding), and for the normal
// distribution function the five-term fit of Abramowitz and Stegun, 7.1.26 (1.4e-7; relative to the tail 3e-5 at g = -2.8,
// beyond which the library function takes over).
template <int ACT, bool F32>
__device__ __forceinline__ void gate(float g, float& a, float& da) {
  if constexpr (ACT == AGCN_ACT_RELU) {
    a = g > 0.f ? g : 0.f;
    da = g > 0.f ? 1.f : 0.f;
    if (g != g) a = da = g;
  } else if constexpr (ACT == AGCN_ACT_GELU && F32) {
    const float c = 0.5f * erfcf(-0.70710678f * g);
    a = g * c;
    da = fmaf(g, 0.39894228f * expf(-0.5f * g * g), c);
  } else if constexpr (ACT == AGCN_ACT_GELU) {
    const float x = 0.70710678f * fabsf(g), t = __builtin_amdgcn_rcpf(fmaf(0.3275911f, x, 1.f));
    const float e = __builtin_amdgcn_exp2f(-0.72134752f * g * g);       // e^(-g^2 / 2)
    float q = fmaf(fmaf(fmaf(fmaf(1.061405429f, t, -1.453152027f), t, 1.421413741f), t, -0.284496736f), t, 0.254829592f) * t * e;
    if (g < -2.828427f) q = erfcf(x);
    const float c = g < 0.f ? 0.5f * q : fmaf(-0.5f, q, 1.f);
    a = g * c;
    da = fmaf(g, 0.39894228f * e, c);
  } else {
    float e, d;
    if constexpr (F32) {
      e = exp_neg(fabsf(g));
      d = recip_1p(e);
    } else {
      e = __builtin_amdgcn_exp2f(-1.44269504f * fabsf(g));
      d = __builtin_amdgcn_rcpf(1.f + e);
    }
    const float s = g >= 0.f ? d : e * d, ns = g >= 0.f ? e * d : d;    // sigmoid(g), sigmoid(-g)
    if constexpr (ACT == AGCN_ACT_SIGMOID) {
      a = s;
      da = s * ns;
    } else {
      a = g * s;
      da = s * fmaf(g, ns, 1.f);
    }
  }
}
// the same for N values: one branch for all, so that their chains run side by side
template <bool F32, int N>
__device__ __forceinline__ void gates(int act, const float (&g)[N], float (&a)[N], float (&da)[N]) {
  if (act == AGCN_ACT_SILU) {
#pragma unroll
    for (int i = 0; i < N; ++i) gate<AGCN_ACT_SILU, F32>(g[i], a[i], da[i]);
  } else if (act == AGCN_ACT_GELU) {
#pragma unroll
    for (int i = 0; i < N; ++i) gate<AGCN_ACT_GELU, F32>(g[i], a[i], da[i]);
  } else if (act == AGCN_ACT_SIGMOID) {
#pragma unroll
    for (int i = 0; i < N; ++i) gate<AGCN_ACT_SIGMOID, F32>(g[i], a[i], da[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) gate<AGCN_ACT_RELU, F32>(g[i], a[i], da[i]);
  }
}

// ---- eight neighbouring values of a row -----------------------------------------------------------------------------
struct F8 { float v[8]; };

// the library's own matrices: rows at multiples of eight elements
__device__ __forceinline__ void store8_f32(float* p, const F8& x) {
  *reinterpret_cast<f32x4*>(p) = (f32x4){x.v[0], x.v[1], x.v[2], x.v[3]};
  *reinterpret_cast<f32x4*>(p + 4) = (f32x4){x.v[4], x.v[5], x.v[6], x.v[7]};
}
__device__ __forceinline__ F8 load8_f32(const float* p) {
  const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
  return {{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
}
__device__ __forceinline__ u32x4 bf8(const F8& x) {
  return (u32x4){pk_bf(x.v[0], x.v[1]), pk_bf(x.v[2], x.v[3]), pk_bf(x.v[4], x.v[5]), pk_bf(x.v[6], x.v[7])};
}
// What the backward's epilogue reads: P and Q.  fp32 calls: as they are.  bf16 calls: 24 bits of each value, rounded to nearest (ties
// away; a carry out of the largest finite value gives infinity), the upper sixteen and the lower eight in planes of their own;
// bytes are moved with v_perm.  (A NaN stays one: those of a bf16 call have nothing in the low bits that the rounding could carry
// out of.)
template <bool F32> struct Kept8;
template <> struct Kept8<true> { f32x4 a, b; };
template <> struct Kept8<false> { u32x4 hi; u32x2 lo; };
__device__ __forceinline__ uint8_t* low_plane(const GemmArgs& g, const void* p) {
  return reinterpret_cast<uint8_t*>(const_cast<uint16_t*>(static_cast<const uint16_t*>(p)) + (int64_t)g.M * g.ldh);
}
template <bool F32>
__device__ __forceinline__ void store8_kept(const GemmArgs& g, void* p, int64_t at, const F8& x) {
  if constexpr (F32) {
    store8_f32(static_cast<float*>(p) + at, x);
  } else {
    uint32_t r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = __float_as_uint(x.v[i]) + 0x80u;
    u32x4 hi;
    u32x2 lo;
#pragma unroll
    for (int i = 0; i < 4; ++i) hi[i] = __builtin_amdgcn_perm(r[2 * i + 1], r[2 * i], 0x07060302u);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      lo[i] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(r[4 * i + 3], r[4 * i + 2], 0x0c0c0501u),
                                    __builtin_amdgcn_perm(r[4 * i + 1], r[4 * i], 0x0c0c0501u), 0x05040100u);
    *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(p) + at) = hi;
    *reinterpret_cast<u32x2*>(low_plane(g, p) + at) = lo;
  }
}
template <bool F32>
__device__ __forceinline__ void store_kept(void* p, int64_t plane, int64_t at, float x) {
  if constexpr (F32) {
    static_cast<float*>(p)[at] = x;
  } else {
    const uint32_t r = __float_as_uint(x) + 0x80u;
    static_cast<uint16_t*>(p)[at] = (uint16_t)(r >> 16);
    reinterpret_cast<uint8_t*>(static_cast<uint16_t*>(p) + plane)[at] = (uint8_t)(r >> 8);
  }
}
template <bool F32>
__device__ __forceinline__ void fetch8_kept(const GemmArgs& g, const void* p, int64_t at, Kept8<F32>& k) {
  if constexpr (F32) {
    const float* q = static_cast<const float*>(p) + at;
    k.a = *reinterpret_cast<const f32x4*>(q);
    k.b = *reinterpret_cast<const f32x4*>(q + 4);
  } else {
    k.hi = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p) + at);
    k.lo = *reinterpret_cast<const u32x2*>(low_plane(g, p) + at);
  }
}
template <bool F32>
__device__ __forceinline__ F8 kept8(const Kept8<F32>& k) {
  F8 x;
  if constexpr (F32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) { x.v[i] = k.a[i]; x.v[4 + i] = k.b[i]; }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      x.v[i] = __uint_as_float(__builtin_amdgcn_perm(k.hi[i >> 1], k.lo[i >> 2], (i & 1 ? 0x07060000u : 0x05040000u) | (uint32_t)(i & 3) << 8 | 0x0cu));
  }
  return x;
}
// what bf16 leaves of x (nothing, where the leading piece is infinite: the products would make NaN of inf - inf)
__device__ __forceinline__ float rest_of(float x, float lead) { return fabsf(lead) < __builtin_inff() ? x - lead : 0.f; }
// eight values of a matrix that a later product reads
template <bool F32>
__device__ __forceinline__ void store8_operand(const GemmArgs& g, void* dst, int64_t at, const F8& x) {
  uint16_t* p = static_cast<uint16_t*>(dst);
  if constexpr (!F32) {
    const u32x4 h = bf8(x);
    *reinterpret_cast<u32x4*>(p + at) = h;
    if (g.two) {
      F8 rest;
#pragma unroll
      for (int i = 0; i < 8; ++i) rest.v[i] = rest_of(x.v[i], __uint_as_float(i & 1 ? h[i >> 1] & 0xffff0000u : h[i >> 1] << 16));
      *reinterpret_cast<u32x4*>(p + g.plane + at) = bf8(rest);
    }
  } else if (g.op == OP_FP32) {
    store8_f32(static_cast<float*>(dst) + at, x);
  } else {
    u32x4 h, m, l;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t a, b, c;
      split3(x.v[2 * i], x.v[2 * i + 1], a, b, c);
      h[i] = a; m[i] = b; l[i] = c;
    }
    *reinterpret_cast<u32x4*>(p + at) = h;
    *reinterpret_cast<u32x4*>(p + g.plane + at) = m;
    *reinterpret_cast<u32x4*>(p + 2 * g.plane + at) = l;
  }
}
// a caller's matrix: any alignment, any tail
template <bool F32>
__device__ __forceinline__ void store8_out(const GemmArgs& g, void* p, int64_t row, int n, const F8& x) {
  const int64_t at = row * g.ldo + n;
  if constexpr (F32) {
    float* o = static_cast<float*>(p) + at;
    if (n + 8 <= g.N) {
#pragma unroll
      for (int k = 0; k < 8; k += 4)
        *reinterpret_cast<u32x4u*>(o + k) = (u32x4u){__float_as_uint(x.v[k]), __float_as_uint(x.v[k + 1]), __float_as_uint(x.v[k + 2]), __float_as_uint(x.v[k + 3])};
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) if (n + i < g.N) o[i] = x.v[i];
    }
  } else {
    uint16_t* o = static_cast<uint16_t*>(p) + at;
    const u32x4 b = bf8(x);
    if (n + 8 <= g.N) {
      *reinterpret_cast<u32x4h*>(o) = (u32x4h){b.x, b.y, b.z, b.w};
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) if (n + i < g.N) o[i] = (uint16_t)(b[i >> 1] >> (16 * (i & 1)));
    }
  }
}

// What becomes of columns n .. n + 7 of row m (v1: of the second B matrix; P, Q: fetched by the caller)
template <int EPI, int NB, bool F32>
__device__ __forceinline__ void epilogue(const GemmArgs& g, int m, int n, const F8& v0, const F8& v1, const Kept8<F32>& P, const Kept8<F32>& Q) {
  if (EPI == EPI_STORE) {
    if (n >= g.N) return;
    store8_out<F32>(g, g.out, m, n, v0);
    if (NB == 2) store8_out<F32>(g, g.out2, m, n, v1);
    return;
  }
  // (the library's own matrices are padded to eights: the columns behind H get the zeros that the products read there)
  if (n >= g.ldh) return;
  const int64_t at = (int64_t)m * g.ldh + n;
  if (EPI == EPI_GATED) {
    F8 hv, pv, qv;
    float a[8], da[8];
    gates<F32, 8>(g.act, v0.v, a, da);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      qv.v[i] = n + i < g.N ? a[i] : 0.f;
      hv.v[i] = n + i < g.N ? a[i] * v1.v[i] : 0.f;
      pv.v[i] = n + i < g.N ? da[i] * v1.v[i] : 0.f;
    }
    if (g.p) {
      store8_kept<F32>(g, g.p, at, pv);
      store8_kept<F32>(g, g.q, at, qv);
    }
    store8_operand<F32>(g, g.hid, at, hv);
  } else {
    const F8 pv = kept8<F32>(P), qv = kept8<F32>(Q);
    F8 dg, du;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      dg.v[i] = v0.v[i] * pv.v[i];
      du.v[i] = v0.v[i] * qv.v[i];
    }
    store8_operand<F32>(g, g.dg, at, dg);
    store8_operand<F32>(g, g.du, at, du);
  }
}

#ifdef __HIP_DEVICE_COMPILE__      // (address spaces and builtins that the host pass does not know)
// The tiles of one operand in a stage: NMAT matrices of PL planes, each ROWS rows of the operand (m or n) by BK, ES bytes an element.
// T (transposed): the operand's matrix is [k][rows].  Every wave issues kSlots loads of 64 x LB bytes.
// INTER (transposed bf16): a fragment's lanes q = lane / 16 hold k = 4 q .. 4 q + 3 and 16 + 4 q .. 16 + 4 q + 3 of its 32 (as the
// accumulators of two neighbouring fragments lie), in place of 8 q .. 8 q + 7.
template <int ROWS, bool T, int BK, int PL, int ES, int LB, int NMAT, int WAVES, bool INTER = false>
struct Tiles {
  static constexpr int kEpc = 16 / ES;                         // elements of a chunk
  static constexpr int kRowBytes = (T ? ROWS : BK) * ES, kRowChunks = kRowBytes / 16;
  static constexpr int kBytes = ROWS * BK * ES;                // of one tile
  static constexpr int kPerTile = kBytes / (64 * LB);          // loads of a wave for one tile
  static constexpr int kSlots = kPerTile * PL * NMAT / WAVES;
  static_assert(kPerTile * PL * NMAT % WAVES == 0 && kBytes % (64 * LB) == 0, "whole loads per wave");
  int voff[kSlots], kl[kSlots];

  // Which chunk of row r lies where (an xor).  Rows along k: sixteen rows of one chunk in different 16-byte columns of the 256-byte
  // bank line.  Rows across k, bf16: the four rows that sixteen lanes read, and the set eight rows on, in different 32-byte
  // columns; fp32: the rows that the four sixteens of lanes read, eight apart, in different 64-byte columns.
  static __device__ __forceinline__ int perm(int r) {
    if (!T) return kRowBytes == 128 ? (r >> 1) & 7 : (r >> 2) & 3;
    if (ES == 4) return ((r >> 3) & 3) << 2 & (kRowChunks - 1);
    constexpr int hb = INTER ? 2 : 3;
    if (kRowChunks >= 16) return ((r & 3) | ((r >> hb) & 1) << 2) << 1;
    if (kRowChunks == 8) return (((r >> 1) & 1) | ((r >> hb) & 1) << 1) << 1;
    return ((r >> 3) & 1) << 1;
  }
  __device__ __forceinline__ void init(int row0, int rows, int ld, int wave, int lane) {
#pragma unroll
    for (int i = 0; i < kSlots; ++i) {
      const int byte = (((wave * kSlots + i) % kPerTile) * 64 + lane) * LB, ci = byte >> 4, tr = ci / kRowChunks;
      const int e = ((ci % kRowChunks) ^ perm(tr)) * kEpc + (byte & 15) / ES;      // place in the tile's row
      const int r = T ? e : tr, k = T ? tr : e;
      voff[i] = (T ? k * ld + r : r * ld + k) * ES;
      kl[i] = row0 + r < rows ? k : 0x7fffffff;
    }
  }
  // k tile kt of the operand at p0 / p1, its row (T: column) row0 on, into LDS; `left`: k that remain there
  __device__ __forceinline__ void load(const void* p0, const void* p1, int row0, int64_t plane, int ld, int kt, int left, AGCN_LDS char* dst, int wave) const {
    const int64_t at = (T ? (int64_t)kt * BK * ld + row0 : (int64_t)row0 * ld + (int64_t)kt * BK) * ES;
#pragma unroll
    for (int i = 0; i < kSlots; ++i) {
      const int t = wave * kSlots + i, tile = t / kPerTile;    // tile: matrix * PL + plane
      const char* base = static_cast<const char*>(NMAT == 2 && tile >= PL ? p1 : p0) + (PL == 1 ? 0 : (tile % PL) * plane * ES) + at;
      const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), 0, 0x7fffffff, 0x00020000);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (AGCN_LDS void*)(dst + t * (64 * LB)), LB, kl[i] < left ? voff[i] : (int)0x80000000, 0, 0, 0);
    }
  }
  // Fragment f, k step kk (32 k) of tile `tile`: sixteen rows, lane (r = lane & 15, q = lane / 16) gets k = 8 q .. 8 q + 7 of row r.
  // T: the lane's place in each of the FR fragments is worked out once and hidden from the compiler: through the chain of additions
  // that it would build otherwise it does not see which array a transposing read reads, and waits for all loads in flight.
  template <int FR>
  struct Reader {
    int at[T ? FR : 1], lane, row0;
    __device__ __forceinline__ Reader(int row, int lane_) : lane(lane_), row0(row) {
      const int l = lane & 15, q = lane >> 4, k = ES == 4 ? q * 8 : q * (INTER ? 4 : 8) + (l >> 2);
#pragma unroll
      for (int f = 0; f < (T ? FR : 0); ++f) {
        // (fp32: a column's 32 bits; bf16: where the transposing read wants this lane to point, four columns of one k)
        const int col = row + f * 16 + (ES == 4 ? l : (l & 3) * 4), chunk = (col / kEpc) ^ perm(k);
        at[f] = k * kRowBytes + chunk * 16 + col % kEpc * ES;
        asm volatile("" : "+v"(at[f]));
      }
    }
    // bf16 elements
    __device__ __forceinline__ u32x4 operator()(const AGCN_LDS char* s, int tile, int f, int kk) const {
      if (!T) {
        const int l = lane & 15, q = lane >> 4;
        return *reinterpret_cast<const AGCN_LDS u32x4*>(s + tile * kBytes + (row0 + f * 16 + l) * kRowBytes + (((kk * 4 + q) ^ perm(l)) << 4));
      } else {
        const AGCN_LDS char* p = s + at[f] + (tile * BK + kk * 32) * kRowBytes;
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((AGCN_LDS s16x4*)p);
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((AGCN_LDS s16x4*)(p + (INTER ? 16 : 4) * kRowBytes));
        const u32x2 a = __builtin_bit_cast(u32x2, lo), b = __builtin_bit_cast(u32x2, hi);
        return (u32x4){a.x, a.y, b.x, b.y};
      }
    }
    // fp32 elements, as their three pieces (BK == 32: one k step)
    __device__ __forceinline__ Pieces pieces(const AGCN_LDS char* s, int tile, int f) const {
      f32x4 lo, hi;
      if (!T) {
        const int l = lane & 15, q = lane >> 4;
        const AGCN_LDS char* p = s + tile * kBytes + (row0 + f * 16 + l) * kRowBytes;
        lo = *reinterpret_cast<const AGCN_LDS f32x4*>(p + (((q * 2) ^ perm(l)) << 4));
        hi = *reinterpret_cast<const AGCN_LDS f32x4*>(p + (((q * 2 + 1) ^ perm(l)) << 4));
      } else {
        const AGCN_LDS char* p = s + at[f] + tile * kBytes;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          lo[i] = *reinterpret_cast<const AGCN_LDS float*>(p + i * kRowBytes);
          hi[i] = *reinterpret_cast<const AGCN_LDS float*>(p + (4 + i) * kRowBytes);
        }
      }
      return split3x8(lo, hi);
    }
  };
};
#endif

// BM x (NB x BN) tile by WGM x WGN waves, operands as OP says, S (2, 3) stages; AT / BT: the operand's matrix has k along its rows
template <int OP, int BM, int BN, int WGM, int WGN, bool AT, bool BT, int NB, int EPI, int S>
__global__ __launch_bounds__(64 * WGM * WGN) void ffn_gemm_kernel(GemmArgs g) {
#ifdef __HIP_DEVICE_COMPILE__
  constexpr int WAVES = WGM * WGN, FM = BM / WGM / 16, FN = BN / WGN / 16, BK = OP == OP_BF16 ? 64 : 32;
  constexpr bool WHOLE = OP == OP_FP32 || OP == OP_WORDS;      // fp32 operands, split here
  constexpr int PL = OP == OP_PLANES ? 3 : 1, ES = WHOLE ? 4 : 2, P = OP == OP_BF16 ? 1 : 3, LB = OP == OP_WORDS ? 4 : 16;      // planes; bytes of an element; pieces; bytes of a load
  constexpr bool F32 = OP != OP_BF16;
  typedef Tiles<BM, AT, BK, PL, ES, LB, 1, WAVES> TA;
  typedef Tiles<BN, BT, BK, PL, ES, LB, NB, WAVES> TB;
  constexpr int SA = PL * TA::kBytes, SB = NB * PL * TB::kBytes;
  // (arrays of their own for every stage and operand: the compiler then sees that the loads into one do not touch the reads of
  // another; it would wait for all loads in flight otherwise)
  __shared__ __attribute__((aligned(1024))) char sa0[SA], sa1[SA], sa2[S > 2 ? SA : 16];
  __shared__ __attribute__((aligned(1024))) char sb0[SB], sb1[SB], sb2[S > 2 ? SB : 16];
  AGCN_LDS char *const a0 = (AGCN_LDS char*)sa0, *const a1 = (AGCN_LDS char*)sa1, *const a2 = (AGCN_LDS char*)sa2;
  AGCN_LDS char *const b0 = (AGCN_LDS char*)sb0, *const b1 = (AGCN_LDS char*)sb1, *const b2 = (AGCN_LDS char*)sb2;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WGN, wn = wave - wm * WGN;

  // workgroup -> tile: workgroups go round the eight dies; a die gets a run of neighbouring tiles (its L2 holds their operands),
  // and within a run four tile rows are walked together
  const int total = g.tiles_m * g.tiles_n * g.splits, run = (total + 7) >> 3;
  const int id = (blockIdx.x & 7) * run + (blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= run || id >= total) return;
  const int tile = id / g.splits, split = id - tile * g.splits;
  const int per = 4 * g.tiles_n, grp = tile / per, first = grp * 4;
  const int rows_in = g.tiles_m - first < 4 ? g.tiles_m - first : 4;
  const int in = tile - grp * per, tm = first + in % rows_in, tn = in / rows_in;
  const int m0 = tm * BM, n0 = tn * BN;

  TA ta;
  TB tb;
  ta.init(m0, g.M, g.lda, wave, lane);
  tb.init(n0, g.N, g.ldb, wave, lane);

  const int iters = g.nseg * g.ktiles;
  const int it0 = (int)((int64_t)iters * split / g.splits), it1 = (int)((int64_t)iters * (split + 1) / g.splits);
  int lit = it0, seg = it0 / g.ktiles, kt = it0 - seg * g.ktiles;      // the next k tile to load
  // (three stages: past the last one the loads still run, on nothing, so that the count of loads in flight stays what the
  // waits below expect.  Two stages: no load, and the branch keeps the scheduler from spreading the loads over the products, which
  // costs it more registers than there are)
  auto load = [&](AGCN_LDS char* a, AGCN_LDS char* b) {
    const Seg s = g.seg[seg < 4 ? seg : 3];
    const int left = lit < it1 ? g.K - kt * BK : 0;
    ta.load(s.a, nullptr, m0, g.a_plane, g.lda, kt, left, a, wave);
    tb.load(s.b, s.b2, n0, g.b_plane, g.ldb, kt, left, b, wave);
    ++lit;
    if (++kt == g.ktiles) { kt = 0; ++seg; }
  };
  f32x4 acc[NB][FM][FN];
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) acc[b][i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
  const typename TA::template Reader<FM> ra(wm * FM * 16, lane);
  const typename TB::template Reader<FN> rb(wn * FN * 16, lane);
  auto compute = [&](const AGCN_LDS char* a, const AGCN_LDS char* b) {
#pragma unroll
    for (int kk = 0; kk < BK / 32; ++kk) {
      u32x4 fa[P][FM], fb[P][NB][FN];
      if constexpr (WHOLE) {
#pragma unroll
        for (int i = 0; i < FM; ++i) {
          const Pieces x = ra.pieces(a, 0, i);
          fa[0][i] = x.h; fa[1][i] = x.m; fa[2][i] = x.l;
        }
#pragma unroll
        for (int c = 0; c < NB; ++c)
#pragma unroll
          for (int j = 0; j < FN; ++j) {
            const Pieces x = rb.pieces(b, c, j);
            fb[0][c][j] = x.h; fb[1][c][j] = x.m; fb[2][c][j] = x.l;
          }
      } else {
#pragma unroll
        for (int p = 0; p < P; ++p) {
#pragma unroll
          for (int i = 0; i < FM; ++i) fa[p][i] = ra(a, p, i, kk);
#pragma unroll
          for (int c = 0; c < NB; ++c)
#pragma unroll
            for (int j = 0; j < FN; ++j) fb[p][c][j] = rb(b, c * P + p, j, kk);
        }
      }
      // (B as the first operand: a lane then holds four neighbouring COLUMNS of one row of the result.  Pieces: small terms first)
      constexpr int NP = P == 1 ? 1 : 6;
      constexpr int pa[6] = {P - 1, 0, P == 1 ? 0 : 1, P == 1 ? 0 : 1, 0, 0}, pb[6] = {0, P - 1, P == 1 ? 0 : 1, 0, P == 1 ? 0 : 1, 0};
#pragma unroll
      for (int t = 0; t < NP; ++t)
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
          for (int c = 0; c < NB; ++c)
#pragma unroll
            for (int j = 0; j < FN; ++j) acc[c][i][j] = mfma_bf(fb[pb[t]][c][j], fa[pa[t]][i], acc[c][i][j]);
    }
  };
  // a stage is there when every wave's own loads of it are (vmcnt counts the later stages' loads that may still fly) and all
  // waves have said so; the same barrier says that the stage about to be overwritten has been read
  auto ready = [] {
    constexpr int fly = (S - 2) * (TA::kSlots + TB::kSlots);
    // (not __syncthreads(), whose fence waits for every load in flight; and the builtin, not text, so that the compiler's own
    // account of the loads in flight sees the wait)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((fly & 15) | 7 << 4 | (fly >> 4) << 14);       // vmcnt(fly) lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  load(a0, b0);
  if (S > 2) load(a1, b1);
  int it = it0;
  if constexpr (S == 2) {
    // (ifs, not breaks: one way out of the loop, or the accumulators are copied at each)
    for (; it < it1; it += 2) {
      ready();
      if (it + 1 < it1) load(a1, b1);
      compute(a0, b0);
      if (it + 1 < it1) {
        ready();
        if (it + 2 < it1) load(a0, b0);
        compute(a1, b1);
      }
    }
  } else {
    // (whole turns without branches, in which the compiler can count the loads in flight; then what is left)
    for (; it + 3 <= it1; it += 3) {
      ready();
      load(a2, b2);
      compute(a0, b0);
      ready();
      load(a0, b0);
      compute(a1, b1);
      ready();
      load(a1, b1);
      compute(a2, b2);
    }
    if (it < it1) {
      ready();
      load(a2, b2);
      compute(a0, b0);
      if (it + 1 < it1) {
        ready();
        compute(a1, b1);
      }
    }
  }
  // Through LDS: a wave's fragments of PR rows at a time, [row][B matrix][column] with the 16-byte chunks permuted by the row
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  constexpr int CH = NB * FN * 4, REGION = (SA < SB ? SA : SB) / (WAVES / 4);      // a quarter of the waves in each array of two stages
  constexpr int FIT = REGION / (CH * 16) / 16, PF = FIT >= FM ? FM : (FIT >= FM / 2 ? FM / 2 : FM / 4), PR = PF * 16;      // fragments, rows per pass
  static_assert(PF >= 1 && PF <= FIT && FM % PF == 0 && WAVES % 4 == 0, "the epilogue's rows have to fit the wave's part of the stages");
  AGCN_LDS char* reg = (wave & 2 ? (wave & 1 ? b1 : b0) : (wave & 1 ? a1 : a0)) + (wave >> 2) * REGION;
  const int n_wave = n0 + wn * FN * 16;
#pragma unroll
  for (int ps = 0; ps < FM / PF; ++ps) {
    const int mr = lane & 15, q = lane >> 4;
#pragma unroll
    for (int i = 0; i < PF; ++i)
#pragma unroll
      for (int c = 0; c < NB; ++c)
#pragma unroll
        for (int j = 0; j < FN; ++j)
          *reinterpret_cast<AGCN_LDS f32x4*>(reg + (i * 16 + mr) * (CH * 16) + ((((c * FN + j) * 4 + q) ^ (mr & (CH - 1))) << 4)) = acc[c][ps * PF + i][j];
    // (one wave's own rows: the wait is for its own writes)
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    constexpr int LPR = FN * 2, RPI = 64 / LPR;       // lanes per row, eight columns each; rows at a time
    // (dA's epilogue: the reads of P and Q of UN turns fly together; one turn's at a time left the matrix pipe waiting for memory, 36
    // us a tile of 8192 x 8192)
    constexpr int UN = EPI == EPI_DH ? (PR / RPI < 4 ? PR / RPI : 4) : 1;
    const int c8 = lane % LPR, n = n_wave + c8 * 8;
#pragma unroll 1
    for (int r0 = 0; r0 < PR; r0 += RPI * UN) {
      Kept8<F32> kp[UN], kq[UN];
      if (EPI == EPI_DH && g.splits == 1) {
#pragma unroll
        for (int u = 0; u < UN; ++u) {
          const int m = m0 + wm * FM * 16 + ps * PR + r0 + u * RPI + lane / LPR;
          if (m < g.M && n < g.ldh) {
            fetch8_kept<F32>(g, g.p, (int64_t)m * g.ldh + n, kp[u]);
            fetch8_kept<F32>(g, g.q, (int64_t)m * g.ldh + n, kq[u]);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < UN; ++u) {
        const int r = r0 + u * RPI + lane / LPR, m = m0 + wm * FM * 16 + ps * PR + r;
        F8 v[NB];
#pragma unroll
        for (int c = 0; c < NB; ++c) {
          const int ch = (c * FN * 4 + c8 * 2), x = r & 15 & (CH - 1);
          const f32x4 lo = *reinterpret_cast<const AGCN_LDS f32x4*>(reg + r * (CH * 16) + ((ch ^ x) << 4));
          const f32x4 hi = *reinterpret_cast<const AGCN_LDS f32x4*>(reg + r * (CH * 16) + (((ch + 1) ^ x) << 4));
          v[c] = {{lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w}};
        }
        if (m < g.M) {
          if (g.splits > 1) {
            if (n < g.ldp) {
              float* p = g.part + ((int64_t)split * NB * g.M + m) * g.ldp + n;
              store8_f32(p, v[0]);
              if (NB == 2) store8_f32(p + (int64_t)g.M * g.ldp, v[NB - 1]);
            }
          } else {
            epilogue<EPI, NB, F32>(g, m, n, v[0], v[NB - 1], kp[u], kq[u]);
          }
        }
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
#endif
}

// Adds the splits' tiles in order and puts the sums through the epilogue.  A workgroup takes 32 times eight columns; eight lanes
// share the splits of each (a single lane would wait for one load after another), and their sums are added in lane order.
template <int NB, int EPI, bool F32>
__global__ __launch_bounds__(256) void ffn_reduce_kernel(GemmArgs g) {
  __shared__ float sums[8][32][NB * 8 + 1];
  const int64_t per = g.ldp >> 3, e = (int64_t)blockIdx.x * 32 + (threadIdx.x & 31);
  const int sl = threadIdx.x >> 5, ev = threadIdx.x & 31;
  const bool live = e < per * g.M;
  const int m = live ? (int)(e / per) : 0, n = live ? (int)(e - (int64_t)m * per) * 8 : 0;
  float v[NB * 8];
#pragma unroll
  for (int i = 0; i < NB * 8; ++i) v[i] = 0.f;
  if (live) {
#pragma unroll 4
    for (int s = sl; s < g.splits; s += 8)
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const F8 x = load8_f32(g.part + (((int64_t)s * NB + b) * g.M + m) * g.ldp + n);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[b * 8 + i] += x.v[i];
      }
  }
#pragma unroll
  for (int i = 0; i < NB * 8; ++i) sums[sl][ev][i] = v[i];
  __syncthreads();
  if (sl || !live) return;
  F8 o[NB];
#pragma unroll
  for (int i = 0; i < NB * 8; ++i) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) s += sums[k][ev][i];
    o[i >> 3].v[i & 7] = s;
  }
  Kept8<F32> kp, kq;
  if (EPI == EPI_DH) {
    fetch8_kept<F32>(g, g.p, (int64_t)m * g.ldh + n, kp);
    fetch8_kept<F32>(g, g.q, (int64_t)m * g.ldh + n, kq);
  }
  epilogue<EPI, NB, F32>(g, m, n, o[0], o[NB - 1], kp, kq);
}

// ---- both products in one kernel: forwards that keep nothing, features of at most 128 -----------------------------------------------------------
struct FusedArgs {
  GemmArgs g;                        // seg[0]: X, Wg, Wu with lda, ldb, b_plane; M, N = H, act, out, ldo, part, ldp, splits
  const void* wd;
  int64_t d_plane;
  int32_t ldd, Fin, Fout;
};

// A wave owns 16 rows: their X stays in its registers (as the pieces that the matrix pipe takes), Y's accumulators too, and H is walked
// in chunks of 32 columns: G and U of the chunk, the gate, and at once the chunk's 32 k of Y.  The gate's results already lie as the
// next product's operand wants them but for the order of k, and Wd is read in that order: A needs neither memory nor LDS.  The
// chunk's weights (three matrices, 144 KB of LDS for two stages of fp32 pieces at 128 features) are all that is loaded.
// A chunk's gate is worked out among the next chunk's first products: the vector unit's work (as much as the matrix pipe's) is
// hidden there (93 -> 75 us; two dependent products in a row in place of four accumulators in turn: 74 -> 70 us).  32768 x 128 x 512
// fp32: the call 108 us as two products (80 + 31: the first has four k stages between filling and emptying its tiles, and A's planes
// are 100 MB each way), 70 here, the kernel 74 on a profile's average: 1.05 PFLOP/s of bf16 products; bound by the matrix pipe and what is
// left of the vector unit.
// bf16 calls give A to the second product in two pieces (851 x 16 x 5656, one piece: 1.5 times the error of an unrounded A; 32768 x 64 x 256
// 12.8 -> 14.7 us, as two products 21.5).
template <int P, int D, int WV, int ACT>
__global__ __launch_bounds__(64 * WV) void ffn_fused_kernel(FusedArgs f) {
#ifdef __HIP_DEVICE_COMPILE__
  constexpr bool F32 = P == 3;
  constexpr int KK = D / 32, FO = D / 16, MID = P == 3 ? 1 : 0, LOW = P - 1;
  typedef Tiles<32, true, D, P, 2, 16, 2, WV> TW;
  typedef Tiles<D, true, 32, P, 2, 16, 1, WV, true> TD;
  __shared__ __attribute__((aligned(1024))) char sw0[2 * P * TW::kBytes], sw1[2 * P * TW::kBytes], sd0[P * TD::kBytes], sd1[P * TD::kBytes];
  AGCN_LDS char *const w0 = (AGCN_LDS char*)sw0, *const w1 = (AGCN_LDS char*)sw1, *const d0 = (AGCN_LDS char*)sd0, *const d1 = (AGCN_LDS char*)sd1;
  const GemmArgs& g = f.g;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, q = lane >> 4;
  const int split = blockIdx.x % g.splits, m = (int)(blockIdx.x / g.splits) * (16 * WV) + wave * 16 + r;
  const int chunks = (g.N + 31) >> 5;
  const int c0 = (int)((int64_t)chunks * split / g.splits), c1 = (int)((int64_t)chunks * (split + 1) / g.splits);
  TW tw;
  TD td;
  td.init(0, f.Fout, f.ldd, wave, lane);
  auto load_w = [&](int c, AGCN_LDS char* w) {
    tw.init(c * 32, g.N, g.ldb, wave, lane);
    tw.load(g.seg[0].b, g.seg[0].b2, c * 32, g.b_plane, g.ldb, 0, f.Fin, w, wave);
  };
  auto load_d = [&](int c, AGCN_LDS char* d) { td.load(f.wd, nullptr, 0, f.d_plane, f.ldd, c, g.N - c * 32, d, wave); };
  load_w(c0, w0);

  u32x4 xa[P][KK];
#pragma unroll
  for (int kk = 0; kk < KK; ++kk) {
    const int k = kk * 32 + q * 8, left = m < g.M ? f.Fin - k : 0;
    const int64_t at = (int64_t)m * g.lda + k;
    if constexpr (F32) {
      const float* x = static_cast<const float*>(g.seg[0].a) + at;
      f32x4 lo = {0.f, 0.f, 0.f, 0.f}, hi = lo;
      if (left >= 8) {
        const u32x4u a = *reinterpret_cast<const u32x4u*>(x), b = *reinterpret_cast<const u32x4u*>(x + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) { lo[e] = __uint_as_float(a[e]); hi[e] = __uint_as_float(b[e]); }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (e < left) lo[e] = x[e];
          if (4 + e < left) hi[e] = x[4 + e];
        }
      }
      const Pieces s = split3x8(lo, hi);
      xa[0][kk] = s.h; xa[MID][kk] = s.m; xa[LOW][kk] = s.l;
    } else {
      const uint16_t* x = static_cast<const uint16_t*>(g.seg[0].a) + at;
      u32x4 v = {0, 0, 0, 0};
      if (left >= 8) {
        const u32x4h a = *reinterpret_cast<const u32x4h*>(x);
        v = (u32x4){a.x, a.y, a.z, a.w};
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) if (e < left) v[e >> 1] |= (uint32_t)x[e] << (16 * (e & 1));
      }
      xa[0][kk] = v;
    }
  }
  f32x4 y[FO];
#pragma unroll
  for (int j = 0; j < FO; ++j) y[j] = (f32x4){0.f, 0.f, 0.f, 0.f};
  const typename TW::template Reader<2> rw(0, lane);
  const typename TD::template Reader<FO> rd(0, lane);
  // (pieces: small terms first)
  constexpr int NP = P == 1 ? 1 : 6;
  constexpr int pa[6] = {LOW, 0, MID, MID, 0, 0}, pb[6] = {0, LOW, MID, 0, MID, 0};
  struct Chunk { f32x4 v[2][2]; };                          // G and U: 16 columns, 16 columns
  auto first = [&](const AGCN_LDS char* w, Chunk& gu) {
#pragma unroll
    for (int b = 0; b < 2; ++b) gu.v[b][0] = gu.v[b][1] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      u32x4 fb[P][2][2];
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int j = 0; j < 2; ++j) fb[p][b][j] = rw(w, b * P + p, j, kk);
#pragma unroll
      for (int t = 0; t < NP; ++t)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int j = 0; j < 2; ++j) gu.v[b][j] = mfma_bf(fb[pb[t]][b][j], xa[pa[t]][kk], gu.v[b][j]);
    }
  };
  struct Gated { u32x4 fa[F32 ? 3 : 2]; };                  // A's pieces (bf16 calls: two, so that it is rounded nowhere that shows)
  auto gated = [&](const Chunk& gu, Gated& o) {
    f32x4 A[2];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float a, slope;
      gate<ACT, F32>(gu.v[0][e >> 2][e & 3], a, slope);
      A[e >> 2][e & 3] = a * gu.v[1][e >> 2][e & 3];
    }
    if constexpr (F32) {
      const Pieces s = split3x8(A[0], A[1]);
      o.fa[0] = s.h; o.fa[MID] = s.m; o.fa[LOW] = s.l;
    } else {
      const u32x4 h = {pk_bf(A[0][0], A[0][1]), pk_bf(A[0][2], A[0][3]), pk_bf(A[1][0], A[1][1]), pk_bf(A[1][2], A[1][3])};
      o.fa[0] = h;
#pragma unroll
      for (int e = 0; e < 8; ++e) A[e >> 2][e & 3] = rest_of(A[e >> 2][e & 3], __uint_as_float(e & 1 ? h[e >> 1] & 0xffff0000u : h[e >> 1] << 16));
      o.fa[1] = (u32x4){pk_bf(A[0][0], A[0][1]), pk_bf(A[0][2], A[0][3]), pk_bf(A[1][0], A[1][1]), pk_bf(A[1][2], A[1][3])};
    }
  };
  auto second = [&](const AGCN_LDS char* d, const Gated& o) {
#pragma unroll
    for (int j0 = 0; j0 < FO; j0 += 4) {                    // (four accumulators in turn: one product waits for its last)
      u32x4 fd[P][4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int p = 0; p < P; ++p) fd[p][j] = rd(d, p, j0 + j, 0);
      if constexpr (!F32) {
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j0 + j] = mfma_bf(fd[0][j], o.fa[1], y[j0 + j]);
      }
#pragma unroll
      for (int t = 0; t < NP; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j0 + j] = mfma_bf(fd[pb[t]][j], o.fa[pa[t]], y[j0 + j]);
    }
  };
  // (a stage is there when every wave's loads of it are and all have said so; by then the other stage has been read)
  auto ready = [] {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(7 << 4);                     // vmcnt(0) lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  auto both = [&](const AGCN_LDS char* w, Chunk& next, const AGCN_LDS char* d, const Chunk& gu) {
    Gated o;
    first(w, next);
    gated(gu, o);
    second(d, o);
  };
  Chunk ga, gb;
  ready();
  load_d(c0, d0);
  if (c0 + 1 < c1) load_w(c0 + 1, w1);
  first(w0, ga);
  int c = c0;
  for (; c + 2 < c1; c += 2) {
    ready();
    load_d(c + 1, d1);
    load_w(c + 2, w0);
    both(w1, gb, d0, ga);
    ready();
    load_d(c + 2, d0);
    if (c + 3 < c1) load_w(c + 3, w1);
    both(w0, ga, d1, gb);
  }
  ready();
  Gated o;
  if (c + 1 < c1) {
    load_d(c + 1, d1);
    both(w1, gb, d0, ga);
    ready();
    gated(gb, o);
    second(d1, o);
  } else {
    gated(ga, o);
    second(d0, o);
  }
#pragma unroll
  for (int j = 0; j < FO; ++j) {
    const int n = j * 16 + q * 4;
    if (m >= g.M || n >= f.Fout) continue;
    const f32x4 v = y[j];
    if (g.splits > 1) {
      *reinterpret_cast<f32x4*>(g.part + ((int64_t)split * g.M + m) * g.ldp + n) = v;
    } else if constexpr (F32) {
      float* o = static_cast<float*>(g.out) + (int64_t)m * g.ldo + n;
      if (n + 4 <= f.Fout) {
        *reinterpret_cast<u32x4u*>(o) = (u32x4u){__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) if (n + e < f.Fout) o[e] = v[e];
      }
    } else {
      __bf16* o = static_cast<__bf16*>(g.out) + (int64_t)m * g.ldo + n;
#pragma unroll
      for (int e = 0; e < 4; ++e) if (n + e < f.Fout) o[e] = (__bf16)v[e];
    }
  }
#endif
}

// Few rows (single tokens while serving): bound by the weights' bytes, nothing else is worth waiting for.  A workgroup takes a strip of
// 128 bytes of the weights' columns, eight lanes a row, eight rows in flight per lane; products and sums in fp32 on the vector unit.
// The lanes' sums meet by halving exchanges in the wave, then in LDS.  The first product's workgroups take one projection each and
// leave fp32 sums (of a part of k each, where the strips alone do not fill the chip); the second product's lanes add the
// parts, apply the gate to the eight k they need (one per lane, handed round by shuffles), and multiply: no launch in between, and A is
// rounded nowhere.
template <typename T> struct Cols;
template <> struct Cols<float> {
  static constexpr int n = 4;
  static __device__ __forceinline__ u32x4 load(const float* p, int left) {
    if (left >= 4) { const u32x4u v = *reinterpret_cast<const u32x4u*>(p); return (u32x4){v.x, v.y, v.z, v.w}; }
    u32x4 v = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 3; ++i) if (i < left) v[i] = __float_as_uint(p[i]);
    return v;
  }
  static __device__ __forceinline__ float at(const u32x4& v, int i) { return __uint_as_float(v[i]); }
};
template <> struct Cols<uint16_t> {
  static constexpr int n = 8;
  static __device__ __forceinline__ u32x4 load(const uint16_t* p, int left) {
    if (left >= 8) { const u32x4h v = *reinterpret_cast<const u32x4h*>(p); return (u32x4){v.x, v.y, v.z, v.w}; }
    u32x4 v = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 7; ++i) if (i < left) v[i >> 1] |= (uint32_t)p[i] << (16 * (i & 1));
    return v;
  }
  static __device__ __forceinline__ float at(const u32x4& v, int i) { return __uint_as_float(i & 1 ? v[i >> 1] & 0xffff0000u : v[i >> 1] << 16); }
};

// Sums of N values over the lanes whose numbers differ in the bits from M down to LX: a lane gives away half of its values at every
// step and adds what it gets to the other half (`first`: which are left to it); with one value left, both lanes add.
template <int N, int M, int LX>
constexpr int halved() { if constexpr (M < LX) return N; else return halved<(N > 1 ? N / 2 : 1), M / 2, LX>(); }
template <int N, int M, int LX>
__device__ __forceinline__ void halve(float* v, int lane, int& first, bool& mine) {
  if constexpr (M >= LX) {
    const bool up = lane & M;
    if constexpr (N > 1) {
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        const float keep = up ? v[i + N / 2] : v[i], give = up ? v[i] : v[i + N / 2];
        v[i] = keep + __shfl_xor(give, M);
      }
      first += up ? N / 2 : 0;
    } else {
      v[0] += __shfl_xor(v[0], M);
      mine = mine && !up;
    }
    halve<(N > 1 ? N / 2 : 1), M / 2, LX>(v, lane, first, mine);
  }
}

struct FewArgs {
  const void *x, *w[2];              // GATE: w[0] alone
  const float* sums;                 // GATE: the first product's, [split][G, U][M][ld_sums]
  float* part;                       // [split][matrix][M][ldp]
  void* out;                         // GATE, one split: [M, N]
  void *p, *q, *hid;                 // GATE, training: [M, ld of the sums], as the matrix pipe's path leaves them
  int32_t M, N, K, ldx, ldw, ld_sums, ldp, act, strips, splits, in_splits, two;
};
constexpr int kFewLanes = 8;         // of a weight row

template <typename TW, int R, bool GATE>
__global__ __launch_bounds__(512) void ffn_rows_kernel(FewArgs g) {
  typedef Cols<TW> CW;
  constexpr bool F32 = sizeof(TW) == 4;
  constexpr int LX = kFewLanes, N0 = R * CW::n, COLS = LX * CW::n, GROUPS = 512 / LX, MATS = GATE ? 1 : 2;
  __shared__ float sums[8][LX * N0];
  const int total = g.strips * MATS * g.splits, run = (total + 7) >> 3;
  const int id = (blockIdx.x & 7) * run + (blockIdx.x >> 3);        // neighbouring strips on one die
  if ((int)(blockIdx.x >> 3) >= run || id >= total) return;
  const int sm = id / g.strips, split = sm / MATS, n_wg = (id - sm * g.strips) * COLS;
  const int lane = threadIdx.x & 63, lx = threadIdx.x % LX, n = n_wg + lx * CW::n;
  const TW* x = static_cast<const TW*>(g.x);
  const TW* w = static_cast<const TW*>(g.w[sm % MATS]);
  float acc[R][CW::n];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int i = 0; i < CW::n; ++i) acc[r][i] = 0.f;
  const int blocks = (g.K + 7) >> 3;
  const int b1 = (int)((int64_t)blocks * (split + 1) / g.splits);
  for (int b = (int)((int64_t)blocks * split / g.splits) + threadIdx.x / LX; b < b1; b += GROUPS) {
    const int k = b * 8;
    u32x4 wv[8];
    if (k + 8 <= g.K && n + CW::n <= g.N) {                         // (loads without branches: they all fly together)
#pragma unroll
      for (int i = 0; i < 8; ++i) wv[i] = CW::load(w + (int64_t)(k + i) * g.ldw + n, CW::n);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) wv[i] = CW::load(w + (int64_t)(k + i) * g.ldw + n, k + i < g.K ? g.N - n : 0);
    }
    if constexpr (GATE) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float a = 0.f, da = 0.f, U = 0.f;
        if (k + lx < g.K && r < g.M) {
          float G = 0.f;
          for (int q = 0; q < g.in_splits; ++q) {
            const float* p = g.sums + ((int64_t)q * 2 * g.M + r) * g.ld_sums + k + lx;
            G += p[0];
            U += p[(int64_t)g.M * g.ld_sums];
          }
          const float one[1] = {G};
          float oa[1], oda[1];
          gates<F32, 1>(g.act, one, oa, oda);
          a = oa[0]; da = oda[0];
        }
        if (g.p && n_wg == 0 && r < g.M) {                          // (pads included: zeros)
          const int64_t at = (int64_t)r * g.ld_sums + k + lx;
          store_kept<F32>(g.p, (int64_t)g.M * g.ld_sums, at, da * U);
          store_kept<F32>(g.q, (int64_t)g.M * g.ld_sums, at, a);
          if (F32) static_cast<float*>(g.hid)[at] = a * U;
          else {
            const __bf16 h = (__bf16)(a * U);
            static_cast<__bf16*>(g.hid)[at] = h;
            if (g.two) static_cast<__bf16*>(g.hid)[(int64_t)g.M * g.ld_sums + at] = (__bf16)rest_of(a * U, (float)h);
          }
        }
        a *= U;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float ai = __shfl(a, (lane & ~(LX - 1)) + i);
#pragma unroll
          for (int e = 0; e < CW::n; ++e) acc[r][e] = fmaf(ai, CW::at(wv[i], e), acc[r][e]);
        }
      }
    } else {
      u32x4 xv[R][8 / CW::n];
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < 8 / CW::n; ++i) xv[r][i] = CW::load(x + (int64_t)(r < g.M ? r : 0) * g.ldx + k + i * CW::n, g.K - k - i * CW::n);
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int e = 0; e < CW::n; ++e)
#pragma unroll
          for (int r = 0; r < R; ++r) acc[r][e] = fmaf(CW::at(xv[r][i / CW::n], i % CW::n), CW::at(wv[i], e), acc[r][e]);
    }
  }
  float v[N0];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int e = 0; e < CW::n; ++e) v[r * CW::n + e] = acc[r][e];
  int first = 0;
  bool mine = true;
  constexpr int have = halved<N0, 32, LX>();
  halve<N0, 32, LX>(v, lane, first, mine);
  if (mine) {
#pragma unroll
    for (int i = 0; i < have; ++i) sums[threadIdx.x >> 6][lx * N0 + first + i] = v[i];
  }
  __syncthreads();
  // a thread: one column of one row
  for (int j = threadIdx.x; j < R * COLS; j += 512) {
    const int m = j / COLS, c = j % COLS, at = c / CW::n * N0 + m * CW::n + c % CW::n;
    if (m >= g.M || n_wg + c >= g.N) continue;
    float s = sums[0][at];
#pragma unroll
    for (int q = 1; q < 8; ++q) s += sums[q][at];
    if (!GATE || g.splits > 1) g.part[((int64_t)sm * g.M + m) * g.ldp + n_wg + c] = s;
    else if (F32) static_cast<float*>(g.out)[(int64_t)m * g.N + n_wg + c] = s;
    else static_cast<__bf16*>(g.out)[(int64_t)m * g.N + n_wg + c] = (__bf16)s;
  }
}

// Operand images: bf16 matrices whose rows do not start at 16 bytes or end at eights, padded with zeros; fp32 ones as three planes of
// bf16 pieces.  One launch for all matrices of a call; a thread makes eight columns.
struct Image { const void* src; void* dst; int64_t rows, plane, chunk0; int32_t cols, ld_src, ld_dst, f32; };
struct ImageArgs { Image im[4]; int32_t n; int64_t chunks; };
__global__ __launch_bounds__(256) void ffn_image_kernel(ImageArgs a) {
  for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < a.chunks; e += (int64_t)gridDim.x * 256) {
    int k = 0;
    while (k + 1 < a.n && a.im[k + 1].chunk0 <= e) ++k;
    const Image& im = a.im[k];
    const int64_t at = e - im.chunk0, per = im.ld_dst >> 3, r = at / per;
    const int c = (int)(at - r * per) * 8;
    uint16_t* dst = static_cast<uint16_t*>(im.dst) + r * im.ld_dst + c;
    if (im.f32) {
      const float* p = static_cast<const float*>(im.src) + r * im.ld_src + c;
      float v[8];
      if (c + 8 <= im.cols) {
        const u32x4u lo = *reinterpret_cast<const u32x4u*>(p), hi = *reinterpret_cast<const u32x4u*>(p + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[i] = __uint_as_float(lo[i]); v[4 + i] = __uint_as_float(hi[i]); }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c + i < im.cols ? p[i] : 0.f;
      }
      u32x4 h, m, l;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t x, y, z;
        split3(v[2 * i], v[2 * i + 1], x, y, z);
        h[i] = x; m[i] = y; l[i] = z;
      }
      *reinterpret_cast<u32x4*>(dst) = h;
      *reinterpret_cast<u32x4*>(dst + im.plane) = m;
      *reinterpret_cast<u32x4*>(dst + 2 * im.plane) = l;
    } else {
      const uint16_t* p = static_cast<const uint16_t*>(im.src) + r * im.ld_src + c;
      u32x4 v;
      if (c + 8 <= im.cols) {
        v = *reinterpret_cast<const u32x4h*>(p);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          v[i] = (c + 2 * i < im.cols ? (uint32_t)p[2 * i] : 0u) | (c + 2 * i + 1 < im.cols ? (uint32_t)p[2 * i + 1] << 16 : 0u);
      }
      *reinterpret_cast<u32x4*>(dst) = v;
    }
  }
}

__global__ __launch_bounds__(256) void ffn_zero_kernel(void* p, int64_t bytes) {
  for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < bytes >> 1; e += (int64_t)gridDim.x * 256) static_cast<uint16_t*>(p)[e] = 0;
}

// ---- host side ---------------------------------------------------------------------------------------------------
inline int pad8(int v) { return (v + 7) & ~7; }
inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// A matrix as the products read it: its own memory, or an image of it
struct Mat { const void* p; int32_t ld; int64_t plane; bool chunks; };      // chunks: rows at 16 bytes, of whole 16-byte chunks

struct Carve {
  char* base;
  size_t off;
  void* take(size_t bytes) {
    void* r = base ? base + off : nullptr;
    off += align256(bytes);
    return r;
  }
};

// How an fp32 call lays its operands out, by its sizes alone (the backward has to come to the same answer).  Measured, planes / as
// they are, forward: 16 rows through 2048 x 8192 188 / 77 us, 256 rows 292 / 226, 400 rows 329 / 379 (training pass: 128 rows 487 / 404, 200
// rows 595 / 654); 5000 rows through 128 x 512 39 / 38, 10000 rows 54 / 60; 700 rows through 1024 x 1024 62 / 66.
int op_of(const AgcnFfnDesc& d) {
  if (d.dtype == AGCN_DTYPE_BF16) return OP_BF16;
  return d.rows <= (d.training ? 160 : 320) || d.rows * (int64_t)d.H * (d.Fin + d.Fout) <= (int64_t)640 << 20 ? OP_FP32 : OP_PLANES;
}
// bf16 calls whose A has few elements: A, dG and dU go on in two bf16 pieces.  Errors of a training pass's results, relative to rounding
// them alone: two pieces 1.00 at every size; one piece 1.40 to 1.48 (a rounding of A, dG or dU is as much as one of the result), more where
// few roundings make up a result or a tensor has few elements (6 rows through 1617 x 270 1.56, 18 through 64 x 64 1.60, 4000 through
// 8 x 8 1.92).  The limit weighs that against time, a captured training pass with one piece / two: 64 x 64 x 256 24.1 / 26.8 us, 6 x 1617 x
// 270 39.4 / 42.1, 1000 x 16 x 16 26.4 / 28.5; beyond the limit 260 x 64 x 256 27.2 / 33.4, 300 x 75 x 200 30.6 / 37.3, 16 x 2048 x 8192
// 91.5 / 99.5, and where the matrix pipe is the bound fifteen products of M F H in place of nine.
bool two_pieces(const AgcnFfnDesc& d) { return d.dtype == AGCN_DTYPE_BF16 && d.rows * d.H <= 16384; }
bool whole_chunks(const AgcnFfnDesc& d, const void* p, int cols, int ld) {
  const int epc = d.dtype == AGCN_DTYPE_BF16 ? 8 : 4;
  return cols % epc == 0 && ld % epc == 0 && ((uintptr_t)p & 15) == 0;
}
// read in place: whole fp32 matrices always, bf16 ones in whole chunks
bool direct(const AgcnFfnDesc& d, const void* p, int cols, int ld) {
  return op_of(d) == OP_FP32 || (op_of(d) == OP_BF16 && whole_chunks(d, p, cols, ld));
}

// Which forwards the few-row kernels serve.  Measured with them / on the matrix pipe, 1 row and 4 rows: 2048 x 8192 bf16 29.5 / 36.3 us and
// 35.5 / 36.1, 2000 x 8001 bf16 (no images of the weights) 30 / 59 and 36 / 58, 2048 x 8192 f32 50 / 79 and 56 / 71, 1024 x 4096 f32 20.5 / 30
// and 20.5 / 31, 128 x 512 17.5 / 17.5 us; 8 rows 43 / 36, 54 / 59, 70 / 72.
bool few_rows(const AgcnFfnDesc& d) { return d.rows <= 4; }

// Which forwards the fused kernel serves: those that keep nothing (written from its registers, P, Q and A leave in pieces of 16 bytes: 100000
// x 64 x 4096 bf16 training forward 2250 us, 970 as two products).  Measured as two products / fused, in a captured graph: 4608 x 64 x 256
// f32 19 / 15 us, bf16 11 / 10; 5 x 64 x 256 f32 15 / 10; 1000 x 64 x 4096 38 / 25; 5 x 64 x 4096 13 / 16; up to 128 features 4608 x 512 f32 35 / 30,
// bf16 15.8 / 16.1; 10000 x 512 f32 53 / 40; 32768 x 128 45 / 26; but 1000 x 1000 f32 24 / 27, 4608 x 128 17 / 23 (a chunk of 128 features
// takes a workgroup 3 us, whatever its neighbours do).
bool wide(const AgcnFfnDesc& d) { return d.Fin > 64 || d.Fout > 64; }
bool fused(const AgcnFfnDesc& d) {
  if (d.training || few_rows(d) || d.Fin > 128 || d.Fout > 128) return false;
  return !wide(d) || d.rows * d.H >= 1 << 21;
}

// What the forward leaves for the backward.  The images are there only where a matrix cannot be read as it is; room is kept for
// them whenever the SIZES alone would not rule them out (an address can be odd).
struct Reserve { void *x, *wg, *wu, *wd, *hid, *p, *q; };
size_t carve_reserve(const AgcnFfnDesc& d, void* mem, Reserve* r) {
  Carve c{static_cast<char*>(mem), 0};
  const int op = op_of(d), Hp = pad8(d.H), Fp = pad8(d.Fin), Op = pad8(d.Fout);
  const size_t image = op == OP_BF16 ? 2 : op == OP_FP32 ? 0 : 6, e = two_pieces(d) || op == OP_FP32 ? 4 : image, kept = d.dtype == AGCN_DTYPE_F32 ? 4 : 3;
  const bool served = !d.training && few_rows(d), one = fused(d);        // (neither reads images nor A; fp32 planes lie in the workspace)
  const size_t weights = served || (one && d.dtype == AGCN_DTYPE_F32) ? 0 : image;
  r->x = c.take(served || one ? 0 : image * d.rows * Fp);
  r->wg = c.take(weights * d.Fin * Hp);
  r->wu = c.take(weights * d.Fin * Hp);
  r->wd = c.take(weights * d.H * Op);
  r->hid = c.take(served || one ? 0 : e * d.rows * Hp);
  r->p = d.training ? c.take(kept * d.rows * Hp) : nullptr;
  r->q = d.training ? c.take(kept * d.rows * Hp) : nullptr;
  return c.off;
}

// Tile of a product, its splits, and the kernel's stages: 0 large (256 x 256; three planes: 256 x 128), 1 middle (128 x 128; 128 x 64),
// 2 small (64 x 64; two B matrices: 64 of each; fp32: 32 of each).
struct Config { int kind, bm, bn, splits; };      // bn: columns of one B matrix
Config tile_of(int kind, int op, int nb, int splits) {
  if (kind == 0) return {0, 256, (op == OP_BF16 ? 256 : 128) / nb, splits};
  if (kind == 1) return {1, 128, (op == OP_BF16 ? 128 : 64) / nb, splits};
  return {2, 64, op == OP_BF16 ? 64 : 64 / nb, splits};
}
// The choice: the least time by a model of the chip's 256 CUs.  per_it[w - 1]: a k stage with w workgroups on the CU (the large tile's
// 8 waves fill it; two middle or two to three small ones share it), fixed: a tile's first loads and its epilogue -- microseconds,
// measured on 5003 x 1001 x 2731 (bf16) and 32768 x 128 x 512 (fp32, its training pass) with every kind in turn: e.g. X^T dG, 344 middle tiles of 79
// stages 84 us, 172 large ones in two splits 82 + 17, small ones 105; A^T dY, 176 middle tiles 70 us, in two splits 54 + 9.
// Splits cost their fp32 tiles' way to memory and back (4 MB a microsecond; half that through the gates' epilogues).
Config choose(int64_t M, int64_t N, int nb, int op, int64_t iters, bool gates) {
  struct Cost { float per_it[3], fixed; int at_once, most; };
  static const Cost kBf16[3] = {{{2.0f, 0.f, 0.f}, 8.f, 1, 4}, {{0.82f, 1.08f, 0.f}, 6.f, 2, 8}, {{0.45f, 0.65f, 0.86f}, 4.f, 3, 64}};
  static const Cost kF32[3] = {{{2.8f, 0.f, 0.f}, 8.f, 1, 4}, {{1.0f, 1.6f, 0.f}, 5.f, 2, 8}, {{0.6f, 0.9f, 0.f}, 4.f, 2, 64}};
  static const Cost kWhole = {{0.6f, 0.8f, 1.0f}, 4.f, 3, 64};
  Config best = tile_of(2, op, nb, 1);
  float least = 1e30f;
  for (int kind = op == OP_FP32 ? 2 : 0; kind < 3; ++kind) {              // (fp32 operands: the small tile alone)
    const Cost& k = op == OP_BF16 ? kBf16[kind] : op == OP_FP32 ? kWhole : kF32[kind];
    const int at_once = kind == 2 && nb == 2 && op == OP_BF16 ? 2 : k.at_once;            // (the LDS of two B matrices: two workgroups)
    const Config c = tile_of(kind, op, nb, 1);
    const int64_t tiles = std::max<int64_t>(1, cdiv(M, c.bm) * cdiv(N, c.bn));     // (size queries come here with no rows, too)
    for (int s = 1; s <= k.most && s <= std::max<int64_t>(1, iters / 2); s += s < 8 ? 1 : 4) {
      const int64_t per_cu = cdiv(tiles * s, 256), its = cdiv(iters, s);
      const int rest = (int)(per_cu % at_once);
      float t = (float)(per_cu / at_once) * (its * k.per_it[at_once - 1] + k.fixed);
      if (rest) t += its * k.per_it[rest - 1] + k.fixed;
      if (s > 1) t += 4.f + (float)s * nb * M * N * 8.f / (gates ? 2e6f : 4e6f);
      if (t < least) {
        least = t;
        best = tile_of(kind, op, nb, s);
      }
    }
  }
  return best;
}

size_t part_bytes(const Config& c, int64_t M, int64_t N, int nb) {
  return c.splits > 1 ? (size_t)c.splits * nb * M * ((N + 7) & ~7ll) * sizeof(float) : 0;
}
int64_t ktiles_of(const AgcnFfnDesc& d, int64_t K) { return cdiv(K, d.dtype == AGCN_DTYPE_F32 ? 32 : 64); }

template <int OP, int BM, int BN, int WGM, int WGN, bool AT, bool BT, int NB, int EPI, int S>
void launch_tile(const GemmArgs& g, hipStream_t s) {
  const int64_t total = (int64_t)g.tiles_m * g.tiles_n * g.splits;
  hipLaunchKernelGGL((ffn_gemm_kernel<OP, BM, BN, WGM, WGN, AT, BT, NB, EPI, S>), dim3((unsigned)(cdiv(total, 8) * 8)), dim3(64 * WGM * WGN), 0, s, g);
}

template <bool AT, bool BT, int NB, int EPI>
void product(GemmArgs& g, void* part, hipStream_t s) {
  g.ktiles = (int)cdiv(g.K, g.f32 ? 32 : 64);
  const int n_all = EPI == EPI_STORE ? g.N : g.ldh;         // columns that the epilogue has to reach
  const Config c = choose(g.M, n_all, NB, g.op, (int64_t)g.nseg * g.ktiles, EPI != EPI_STORE);
  g.tiles_m = (int)cdiv(g.M, c.bm); g.tiles_n = (int)cdiv(n_all, c.bn); g.splits = c.splits;
  g.part = static_cast<float*>(part); g.ldp = (n_all + 7) & ~7;
  if (g.op == OP_BF16) {
    if (c.kind == 0) launch_tile<OP_BF16, 256, 256 / NB, 2, 4, AT, BT, NB, EPI, 2>(g, s);
    else if (c.kind == 1) launch_tile<OP_BF16, 128, 128 / NB, 2, 2, AT, BT, NB, EPI, 2>(g, s);
    else launch_tile<OP_BF16, 64, 64, 2, 2, AT, BT, NB, EPI, 3>(g, s);
  } else if (g.op == OP_PLANES) {
    if (c.kind == 0) launch_tile<OP_PLANES, 256, 128 / NB, 4, 2, AT, BT, NB, EPI, 2>(g, s);
    else if (c.kind == 1) launch_tile<OP_PLANES, 128, 64 / NB, 2, 2, AT, BT, NB, EPI, 2>(g, s);
    else launch_tile<OP_PLANES, 64, 64 / NB, 2, 2, AT, BT, NB, EPI, 3>(g, s);
  } else {
    if (g.words) launch_tile<OP_WORDS, 64, 64 / NB, 2, 2, AT, BT, NB, EPI, 3>(g, s);
    else launch_tile<OP_FP32, 64, 64 / NB, 2, 2, AT, BT, NB, EPI, 3>(g, s);
  }
  const dim3 rg((unsigned)cdiv((int64_t)g.M * (g.ldp / 8), 32));
  if (g.splits > 1 && !g.f32) hipLaunchKernelGGL((ffn_reduce_kernel<NB, EPI, false>), rg, dim3(256), 0, s, g);
  else if (g.splits > 1) hipLaunchKernelGGL((ffn_reduce_kernel<NB, EPI, true>), rg, dim3(256), 0, s, g);
}

// The few-row products: strips of 128 bytes, and k cut until 256 workgroups are there (a workgroup has 512 k in flight; 512 of them: 2048
// x 8192 bf16 30 -> 31.5 us).  The second product's parts cost a launch that adds them: from 2048 k on (1 row through 512 x 2048 17.6 us
// whole, 20.7 in parts; 2 rows through 1024 x 4096 24.8 whole, 21.5 in parts).
struct Few { int strips, splits; size_t part; int ldp; };
Few few_of(const AgcnFfnDesc& d, int64_t N, int64_t K, int mats) {
  Few c;
  c.strips = (int)cdiv(N, kFewLanes * (d.dtype == AGCN_DTYPE_F32 ? 4 : 8));
  c.splits = (int)std::max<int64_t>(1, std::min<int64_t>(16, std::min(cdiv(256, c.strips * mats), K / 512)));
  if (mats == 1 && K <= 2048) c.splits = 1;
  c.ldp = pad8((int)N);
  c.part = mats == 2 || c.splits > 1 ? align256((size_t)c.splits * mats * d.rows * c.ldp * sizeof(float)) : 0;
  return c;
}
template <typename TW, bool GATE>
void few_launch(const FewArgs& g, hipStream_t s) {
  const dim3 grid((unsigned)(cdiv((int64_t)g.strips * g.splits * (GATE ? 1 : 2), 8) * 8)), block(512);
  if (g.M == 1) hipLaunchKernelGGL((ffn_rows_kernel<TW, 1, GATE>), grid, block, 0, s, g);
  else if (g.M == 2) hipLaunchKernelGGL((ffn_rows_kernel<TW, 2, GATE>), grid, block, 0, s, g);
  else hipLaunchKernelGGL((ffn_rows_kernel<TW, 4, GATE>), grid, block, 0, s, g);
}
void few_forward(const AgcnFfnDesc& d, const void* X, const void* Wg, const void* Wu, const void* Wd, void* Y, const Reserve& r, void* workspace, hipStream_t s) {
  const Few a = few_of(d, d.H, d.Fin, 2), b = few_of(d, d.Fout, d.H, 1);
  const bool f32 = d.dtype == AGCN_DTYPE_F32;
  float *sums = static_cast<float*>(workspace), *part = reinterpret_cast<float*>(static_cast<char*>(workspace) + a.part);
  const FewArgs up = {X, {Wg, Wu}, nullptr, sums, nullptr, nullptr, nullptr, nullptr, (int)d.rows, d.H, d.Fin, d.ldx, d.H, 0, a.ldp, d.activation, a.strips, a.splits, 0, 0};
  const FewArgs down = {nullptr, {Wd, nullptr}, sums, part, Y, r.p, r.q, r.hid, (int)d.rows, d.Fout, d.H, 0, d.Fout, a.ldp, b.ldp, d.activation, b.strips, b.splits, a.splits, two_pieces(d)};
  if (f32) few_launch<float, false>(up, s), few_launch<float, true>(down, s);
  else few_launch<uint16_t, false>(up, s), few_launch<uint16_t, true>(down, s);
  if (b.splits == 1) return;
  GemmArgs g;
  std::memset(&g, 0, sizeof(g));
  g.part = part; g.ldp = b.ldp; g.splits = b.splits; g.M = (int)d.rows; g.N = g.ldo = d.Fout; g.out = Y;
  const dim3 grid((unsigned)cdiv((int64_t)g.M * (g.ldp / 8), 32));
  if (f32) hipLaunchKernelGGL((ffn_reduce_kernel<1, EPI_STORE, true>), grid, dim3(256), 0, s, g);
  else hipLaunchKernelGGL((ffn_reduce_kernel<1, EPI_STORE, false>), grid, dim3(256), 0, s, g);
}

// the operands of a product: one or two pairs of matrices
void operands(GemmArgs* g, const Mat& a, const Mat& b, const Mat* b2) {
  g->seg[g->nseg++] = {a.p, b.p, b2 ? b2->p : nullptr};
  g->a_plane = a.plane; g->b_plane = b.plane;
  g->lda = a.ld; g->ldb = b.ld;
  g->words |= !a.chunks || !b.chunks || (b2 && !b2->chunks);
}

// the lower pieces of A, dG, dU: products of their own, added first
Mat rest(const GemmArgs& g, const Mat& m) { return {static_cast<const uint16_t*>(m.p) + g.plane, m.ld, 0, true}; }

int check_ffn(const AgcnFfnDesc* d, const char* who) {
  if (!d) return fail(AGCN_EINVAL, "%s: null descriptor", who);
  if (d->rows < 0 || d->rows > 0x7fffffff - 256) return fail(AGCN_EINVAL, "%s: rows must be in 0..2^31-257 (%lld)", who, (long long)d->rows);
  for (int v : {d->Fin, d->H, d->Fout})
    if (v < 1 || v > 65536) return fail(AGCN_EINVAL, "%s: Fin, H and Fout must be in 1..65536 (%d, %d, %d)", who, d->Fin, d->H, d->Fout);
  if (d->dtype != AGCN_DTYPE_F32 && d->dtype != AGCN_DTYPE_BF16) return fail(AGCN_EINVAL, "%s: f32 or bf16", who);
  if (d->activation != AGCN_ACT_RELU && d->activation != AGCN_ACT_SIGMOID && d->activation != AGCN_ACT_SILU && d->activation != AGCN_ACT_GELU)
    return fail(AGCN_EINVAL, "%s: the gate's activation is relu, sigmoid, silu or gelu", who);
  if (d->ldx < d->Fin || d->ldx > (1 << 20)) return fail(AGCN_EINVAL, "%s: ldx must be in Fin..2^20", who);
  return AGCN_OK;
}

// which operands are read in place; both projections or neither: they have one leading dimension
struct InPlace {
  bool x, w, wd;
  InPlace(const AgcnFfnDesc& d, const void* X, const void* Wg, const void* Wu, const void* Wd)
      : x(direct(d, X, d.Fin, d.ldx)), w(direct(d, Wg, d.H, d.H) && direct(d, Wu, d.H, d.H)), wd(direct(d, Wd, d.Fout, d.Fout)) {}
};

struct ImageList {
  ImageArgs a;
  ImageList() { std::memset(&a, 0, sizeof(a)); }
  Mat add(const AgcnFfnDesc& d, const void* src, int64_t rows, int cols, int ld, void* dst, bool in_place) {
    if (in_place) return {src, ld, 0, whole_chunks(d, src, cols, ld)};
    return image(op_of(d), src, rows, cols, ld, dst);
  }
  Mat image(int op, const void* src, int64_t rows, int cols, int ld, void* dst) {
    const int lp = pad8(cols);
    Image& im = a.im[a.n++];
    im = {src, dst, rows, rows * lp, a.chunks, cols, ld, lp, op == OP_PLANES};
    a.chunks += rows * (lp >> 3);
    return {dst, lp, op == OP_PLANES ? im.plane : 0, true};
  }
  void launch(hipStream_t s) const {
    if (a.chunks) hipLaunchKernelGGL(ffn_image_kernel, dim3((unsigned)std::min<int64_t>(cdiv(a.chunks, 256), 1 << 20)), dim3(256), 0, s, a);
  }
};
// the same matrix in the backward, whose image the forward has left
Mat same(const AgcnFfnDesc& d, const void* src, int64_t rows, int cols, int ld, const void* img, bool in_place) {
  if (in_place) return {src, ld, 0, whole_chunks(d, src, cols, ld)};
  return {img, pad8(cols), op_of(d) == OP_PLANES ? rows * pad8(cols) : 0, true};
}

GemmArgs base_args(const AgcnFfnDesc& d) {
  GemmArgs g;
  std::memset(&g, 0, sizeof(g));
  g.act = d.activation; g.f32 = d.dtype == AGCN_DTYPE_F32; g.op = op_of(d); g.two = two_pieces(d);
  g.ldh = pad8(d.H); g.plane = (int64_t)d.rows * g.ldh;
  return g;
}

int pieces_of(const AgcnFfnDesc& d) { return two_pieces(d) ? 2 : 1; }
size_t product_part(const AgcnFfnDesc& d, int64_t M, int64_t N, int nb, int64_t K, int nseg, bool gates) {
  return part_bytes(choose(M, N, nb, op_of(d), nseg * ktiles_of(d, K), gates), M, N, nb);
}
// The fused kernel: workgroups, splits of H, and the weights' planes.  The splits by a model like choose()'s: a chunk takes a workgroup
// t_chunk on a CU of its own (microseconds, measured), workgroups that share a CU overlap (not those of fp32 pieces of 128 features: they
// fill its LDS), and parts cost a launch and their way to memory and back: 10000 x 64 x 256 fp32 18.4 us whole, 22.7 in two
// parts; 10000 x 64 x 4096 193 whole, 107 in three.
struct Fused { int waves, blocks, splits, ldp; size_t planes, part; };
Fused fused_of(const AgcnFfnDesc& d) {
  const bool f32 = d.dtype == AGCN_DTYPE_F32;
  Fused c;
  c.waves = f32 && wide(d) ? 8 : 4;
  c.blocks = (int)cdiv(std::max<int64_t>(1, d.rows), 16 * c.waves);
  c.splits = 1;
  const float t_chunk = f32 ? (wide(d) ? 3.2f : 1.5f) : (wide(d) ? 1.0f : 0.6f);
  const int64_t chunks = cdiv(d.H, 32);
  float least = 1e30f;
  for (int s = 1; s <= 32 && s <= chunks; ++s) {
    const int64_t per_cu = cdiv((int64_t)c.blocks * s, 256);
    float t = cdiv(chunks, s) * t_chunk * (per_cu == 1 || c.waves == 8 ? per_cu : 0.7f * per_cu);
    if (s > 1) t += 3.5f + (float)s * d.rows * pad8(d.Fout) * 2e-6f;
    if (t < least) {
      least = t;
      c.splits = s;
    }
  }
  c.ldp = pad8(d.Fout);
  c.planes = f32 ? align256((size_t)6 * (2 * (size_t)d.Fin * pad8(d.H) + (size_t)d.H * pad8(d.Fout))) : 0;
  c.part = c.splits > 1 ? align256((size_t)c.splits * d.rows * c.ldp * sizeof(float)) : 0;
  return c;
}
template <int P, int D, int WV>
void fused_launch(const FusedArgs& f, const Fused& c, hipStream_t s) {
  const dim3 grid((unsigned)((int64_t)c.blocks * c.splits)), block(64 * WV);
  if (f.g.act == AGCN_ACT_SILU) hipLaunchKernelGGL((ffn_fused_kernel<P, D, WV, AGCN_ACT_SILU>), grid, block, 0, s, f);
  else if (f.g.act == AGCN_ACT_GELU) hipLaunchKernelGGL((ffn_fused_kernel<P, D, WV, AGCN_ACT_GELU>), grid, block, 0, s, f);
  else if (f.g.act == AGCN_ACT_SIGMOID) hipLaunchKernelGGL((ffn_fused_kernel<P, D, WV, AGCN_ACT_SIGMOID>), grid, block, 0, s, f);
  else hipLaunchKernelGGL((ffn_fused_kernel<P, D, WV, AGCN_ACT_RELU>), grid, block, 0, s, f);
}
void fused_forward(const AgcnFfnDesc& d, const void* X, const Mat& wg, const Mat& wu, const Mat& wd, void* Y, float* part, hipStream_t s) {
  const Fused c = fused_of(d);
  FusedArgs f;
  std::memset(&f, 0, sizeof(f));
  GemmArgs& g = f.g;
  g = base_args(d);
  g.seg[0] = {X, wg.p, wu.p};
  g.lda = d.ldx; g.ldb = wg.ld; g.b_plane = wg.plane;
  g.M = (int)d.rows; g.N = d.H;
  g.out = Y; g.ldo = d.Fout; g.part = part; g.ldp = c.ldp; g.splits = c.splits;
  f.wd = wd.p; f.d_plane = wd.plane; f.ldd = wd.ld; f.Fin = d.Fin; f.Fout = d.Fout;
  if (g.f32) wide(d) ? fused_launch<3, 128, 8>(f, c, s) : fused_launch<3, 64, 4>(f, c, s);
  else wide(d) ? fused_launch<1, 128, 4>(f, c, s) : fused_launch<1, 64, 4>(f, c, s);
  if (c.splits == 1) return;
  GemmArgs q = g;
  q.N = d.Fout;
  const dim3 grid((unsigned)cdiv((int64_t)q.M * (q.ldp / 8), 32));
  if (g.f32) hipLaunchKernelGGL((ffn_reduce_kernel<1, EPI_STORE, true>), grid, dim3(256), 0, s, q);
  else hipLaunchKernelGGL((ffn_reduce_kernel<1, EPI_STORE, false>), grid, dim3(256), 0, s, q);
}

size_t forward_part(const AgcnFfnDesc& d) {
  if (fused(d)) return fused_of(d).planes + fused_of(d).part;
  if (few_rows(d)) return few_of(d, d.H, d.Fin, 2).part + few_of(d, d.Fout, d.H, 1).part;
  return std::max(product_part(d, d.rows, pad8(d.H), 2, d.Fin, 1, true), product_part(d, d.rows, d.Fout, 1, d.H, pieces_of(d), false));
}
struct BackWs { void *dy, *dg, *du, *part; };
size_t carve_backward(const AgcnFfnDesc& d, void* mem, BackWs* w) {
  const int op = op_of(d), Hp = pad8(d.H), pc = pieces_of(d);
  const size_t image = op == OP_BF16 ? 2 : op == OP_FP32 ? 0 : 6, e = two_pieces(d) || op == OP_FP32 ? 4 : image;
  Carve c{static_cast<char*>(mem), 0};
  w->dy = c.take(image * d.rows * pad8(d.Fout));
  w->dg = c.take(e * d.rows * Hp);
  w->du = c.take(e * d.rows * Hp);
  w->part = c.take(std::max(std::max(product_part(d, d.rows, Hp, 1, d.Fout, 1, true), product_part(d, d.rows, d.Fin, 1, d.H, 2 * pc, false)),
                            std::max(product_part(d, d.Fin, d.H, 2, d.rows, pc, false), product_part(d, d.H, d.Fout, 1, d.rows, pc, false))));
  return c.off;
}
// A launch holds fewer than 2^32 threads.  The most that one of the call's own takes: of a product and of the sums of its parts.
int64_t product_threads(const AgcnFfnDesc& d, int64_t M, int64_t N, int nb, int64_t K, int nseg, bool gates) {
  const Config c = choose(M, N, nb, op_of(d), nseg * ktiles_of(d, K), gates);
  const int64_t tiles = cdiv(M, c.bm) * cdiv(N, c.bn) * c.splits;
  return std::max(cdiv(tiles, 8) * 8 * (c.kind == 0 ? 512 : 256), c.splits > 1 ? cdiv(M * (pad8((int)N) / 8), 32) * 256 : 0);
}
int check_threads(const AgcnFfnDesc& d, bool back, const char* who) {
  const int64_t widest = std::max(std::max(d.Fin, d.H), d.Fout);
  if (d.rows * (widest + 64) < (int64_t)1 << 26) return AGCN_OK;         // (2^15 of the smallest tiles, 256 threads each, in 64 parts: 2^29)
  const int pc = pieces_of(d), Hp = pad8(d.H);
  int64_t most = 0;
  if (back) {
    most = std::max(std::max(product_threads(d, d.rows, Hp, 1, d.Fout, 1, true), product_threads(d, d.rows, d.Fin, 1, d.H, 2 * pc, false)),
                    std::max(product_threads(d, d.Fin, d.H, 2, d.rows, pc, false), product_threads(d, d.H, d.Fout, 1, d.rows, pc, false)));
  } else if (fused(d)) {
    const Fused c = fused_of(d);
    most = std::max((int64_t)c.blocks * c.splits * 64 * c.waves, c.splits > 1 ? cdiv(d.rows * (c.ldp / 8), 32) * 256 : 0);
  } else if (!few_rows(d)) {
    most = std::max(product_threads(d, d.rows, Hp, 2, d.Fin, 1, true), product_threads(d, d.rows, d.Fout, 1, d.H, pc, false));
  }
  if (most > 0xffffffffll) return fail(AGCN_EINVAL, "%s: %lld rows at these widths are more than one launch holds", who, (long long)d.rows);
  return AGCN_OK;
}
void zero(void* p, int64_t bytes, hipStream_t s) {
  hipLaunchKernelGGL(ffn_zero_kernel, dim3((unsigned)std::min<int64_t>(cdiv(bytes / 2, 256), 1 << 16)), dim3(256), 0, s, p, bytes);
}
}  // namespace
}  // namespace agcn

using namespace agcn;

extern "C" size_t agcn_gated_ffn_reserve_bytes(const AgcnFfnDesc* desc) {
  if (check_ffn(desc, "agcn_gated_ffn_reserve_bytes") != AGCN_OK) return 0;
  Reserve r;
  return std::max<size_t>(256, carve_reserve(*desc, nullptr, &r));
}

extern "C" size_t agcn_gated_ffn_forward_workspace_bytes(const AgcnFfnDesc* desc) {
  if (check_ffn(desc, "agcn_gated_ffn_forward_workspace_bytes") != AGCN_OK) return 0;
  return std::max<size_t>(256, align256(forward_part(*desc)));
}

extern "C" size_t agcn_gated_ffn_backward_workspace_bytes(const AgcnFfnDesc* desc) {
  if (check_ffn(desc, "agcn_gated_ffn_backward_workspace_bytes") != AGCN_OK) return 0;
  BackWs w;
  return std::max<size_t>(256, carve_backward(*desc, nullptr, &w));
}

extern "C" int agcn_gated_ffn_forward(const AgcnFfnDesc* desc, const void* X, const void* Wg, const void* Wu, const void* Wd, void* Y,
                                      void* reserve, size_t reserve_bytes, void* workspace, size_t workspace_bytes, void* hip_stream) {
  const char* who = "agcn_gated_ffn_forward";
  int rc = check_ffn(desc, who);
  if (rc != AGCN_OK) return rc;
  const AgcnFfnDesc& d = *desc;
  if (d.rows == 0) return AGCN_OK;
  if ((rc = check_threads(d, false, who)) != AGCN_OK) return rc;
  if (!X || !Wg || !Wu || !Wd || !Y) return fail(AGCN_EINVAL, "%s: null tensor", who);
  Reserve r;
  const size_t need = carve_reserve(d, reserve, &r), wneed = forward_part(d);
  if (!reserve || ((uintptr_t)reserve & 255) || reserve_bytes < need)
    return fail(AGCN_ENOSPACE, "%s: reserve too small or not at 256 bytes (%zu < %zu)", who, reserve_bytes, need);
  if (wneed && (!workspace || ((uintptr_t)workspace & 255) || workspace_bytes < wneed))
    return fail(AGCN_ENOSPACE, "%s: workspace too small or not at 256 bytes (%zu < %zu)", who, workspace_bytes, wneed);
  hipStream_t s = static_cast<hipStream_t>(hip_stream);
  ImageList list;
  const InPlace in(d, X, Wg, Wu, Wd);
  if (fused(d)) {
    const Fused c = fused_of(d);
    Mat w[3];
    if (c.planes) {
      char* at = static_cast<char*>(workspace);
      const size_t one = (size_t)6 * d.Fin * pad8(d.H);
      w[0] = list.image(OP_PLANES, Wg, d.Fin, d.H, d.H, at);
      w[1] = list.image(OP_PLANES, Wu, d.Fin, d.H, d.H, at + one);
      w[2] = list.image(OP_PLANES, Wd, d.H, d.Fout, d.Fout, at + 2 * one);
    } else {
      w[0] = list.add(d, Wg, d.Fin, d.H, d.H, r.wg, in.w);
      w[1] = list.add(d, Wu, d.Fin, d.H, d.H, r.wu, in.w);
      w[2] = list.add(d, Wd, d.H, d.Fout, d.Fout, r.wd, in.wd);
    }
    list.launch(s);
    fused_forward(d, X, w[0], w[1], w[2], Y, reinterpret_cast<float*>(static_cast<char*>(workspace) + c.planes), s);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail(AGCN_EDEVICE, "%s: %s", who, hipGetErrorString(e));
    return AGCN_OK;
  }
  const Mat x = list.add(d, X, d.rows, d.Fin, d.ldx, r.x, in.x), wg = list.add(d, Wg, d.Fin, d.H, d.H, r.wg, in.w),
            wu = list.add(d, Wu, d.Fin, d.H, d.H, r.wu, in.w), wd = list.add(d, Wd, d.H, d.Fout, d.Fout, r.wd, in.wd);
  if (few_rows(d)) {
    if (d.training) list.launch(s);                           // (the backward reads them)
    few_forward(d, X, Wg, Wu, Wd, Y, r, workspace, s);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail(AGCN_EDEVICE, "%s: %s", who, hipGetErrorString(e));
    return AGCN_OK;
  }
  list.launch(s);
  GemmArgs g = base_args(d);
  operands(&g, x, wg, &wu);
  g.M = (int)d.rows; g.N = d.H; g.K = d.Fin;
  g.p = r.p; g.q = r.q; g.hid = r.hid;
  product<false, true, 2, EPI_GATED>(g, workspace, s);
  const Mat hid = {r.hid, g.ldh, g.op == OP_PLANES ? g.plane : 0, true};
  GemmArgs q = base_args(d);
  if (q.two) operands(&q, rest(q, hid), wd, nullptr);
  operands(&q, hid, wd, nullptr);
  q.M = (int)d.rows; q.N = d.Fout; q.K = d.H;
  q.out = Y; q.ldo = d.Fout;
  product<false, true, 1, EPI_STORE>(q, workspace, s);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(AGCN_EDEVICE, "%s: %s", who, hipGetErrorString(e));
  return AGCN_OK;
}

extern "C" int agcn_gated_ffn_backward(const AgcnFfnDesc* desc, const void* X, const void* Wg, const void* Wu, const void* Wd,
                                       const void* dY, void* dX, void* dWg, void* dWu, void* dWd, const void* reserve,
                                       size_t reserve_bytes, void* workspace, size_t workspace_bytes, void* hip_stream) {
  const char* who = "agcn_gated_ffn_backward";
  int rc = check_ffn(desc, who);
  if (rc != AGCN_OK) return rc;
  const AgcnFfnDesc& d = *desc;
  if (!d.training) return fail(AGCN_EINVAL, "%s: the forward was not a training one (nothing was kept)", who);
  if ((dWg != nullptr) != (dWu != nullptr)) return fail(AGCN_EINVAL, "%s: dWg and dWu go together", who);
  hipStream_t s = static_cast<hipStream_t>(hip_stream);
  const int64_t esz = d.dtype == AGCN_DTYPE_F32 ? 4 : 2;
  if (d.rows == 0) {                          // no rows: the weights' gradients are sums of nothing
    if (dWg) { zero(dWg, esz * d.Fin * d.H, s); zero(dWu, esz * d.Fin * d.H, s); }
    if (dWd) zero(dWd, esz * d.H * d.Fout, s);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail(AGCN_EDEVICE, "%s: %s", who, hipGetErrorString(e));
    return AGCN_OK;
  }
  if ((rc = check_threads(d, true, who)) != AGCN_OK) return rc;
  if (!X || !Wg || !Wu || !Wd || !dY) return fail(AGCN_EINVAL, "%s: null tensor", who);
  Reserve r;
  BackWs w;
  const size_t need = carve_reserve(d, const_cast<void*>(reserve), &r), wneed = carve_backward(d, workspace, &w);
  if (!reserve || ((uintptr_t)reserve & 255) || reserve_bytes < need)
    return fail(AGCN_ENOSPACE, "%s: reserve too small or not at 256 bytes (%zu < %zu)", who, reserve_bytes, need);
  if (!workspace || ((uintptr_t)workspace & 255) || workspace_bytes < wneed)
    return fail(AGCN_ENOSPACE, "%s: workspace too small or not at 256 bytes (%zu < %zu)", who, workspace_bytes, wneed);
  const InPlace in(d, X, Wg, Wu, Wd);
  const Mat x = same(d, X, d.rows, d.Fin, d.ldx, r.x, in.x), wg = same(d, Wg, d.Fin, d.H, d.H, r.wg, in.w),
            wu = same(d, Wu, d.Fin, d.H, d.H, r.wu, in.w), wd = same(d, Wd, d.H, d.Fout, d.Fout, r.wd, in.wd);
  ImageList list;
  const Mat dy = list.add(d, dY, d.rows, d.Fout, d.Fout, w.dy, direct(d, dY, d.Fout, d.Fout));
  list.launch(s);
  GemmArgs base = base_args(d);
  const int64_t pl = base.op == OP_PLANES ? base.plane : 0;
  const Mat hid = {r.hid, base.ldh, pl, true}, dg = {w.dg, base.ldh, pl, true}, du = {w.du, base.ldh, pl, true};
  if (dX || dWg) {
    GemmArgs g = base;                        // dA = dY Wd^T, and from it dG and dU
    operands(&g, dy, wd, nullptr);
    g.M = (int)d.rows; g.N = d.H; g.K = d.Fout;
    g.p = r.p; g.q = r.q; g.dg = w.dg; g.du = w.du;
    product<false, false, 1, EPI_DH>(g, w.part, s);
  }
  if (dX) {
    GemmArgs g = base;
    if (g.two) operands(&g, rest(g, dg), wg, nullptr), operands(&g, rest(g, du), wu, nullptr);
    operands(&g, dg, wg, nullptr);
    operands(&g, du, wu, nullptr);
    g.M = (int)d.rows; g.N = d.Fin; g.K = d.H;
    g.out = dX; g.ldo = d.Fin;
    product<false, false, 1, EPI_STORE>(g, w.part, s);
  }
  if (dWg) {
    GemmArgs g = base;
    const Mat du_rest = rest(g, du);
    if (g.two) operands(&g, x, rest(g, dg), &du_rest);
    operands(&g, x, dg, &du);
    g.M = d.Fin; g.N = d.H; g.K = (int)d.rows;
    g.out = dWg; g.out2 = dWu; g.ldo = d.H;
    product<true, true, 2, EPI_STORE>(g, w.part, s);
  }
  if (dWd) {
    GemmArgs g = base;
    if (g.two) operands(&g, rest(g, hid), dy, nullptr);
    operands(&g, hid, dy, nullptr);
    g.M = d.H; g.N = d.Fout; g.K = (int)d.rows;
    g.out = dWd; g.ldo = d.Fout;
    product<true, true, 1, EPI_STORE>(g, w.part, s);
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(AGCN_EDEVICE, "%s: %s", who, hipGetErrorString(e));
  return AGCN_OK;
}
