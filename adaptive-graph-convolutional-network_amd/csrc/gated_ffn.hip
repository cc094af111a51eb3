// Gated feed-forward block over node rows (beside DenseMol, models/layers/dense_layer.py:33-50, one product without a gate):
//     G = X Wg, U = X Wu, A = act(G) (.) U, Y = A Wd            X [M, Fin], Wg, Wu [Fin, H], Wd [H, Fout]
//     dA = dY Wd^T;  dG = dA (.) U (.) act'(G);  dU = dA (.) act(G)
//     dX = dG Wg^T + dU Wu^T;  dWg = X^T dG;  dWu = X^T dU;  dWd = A^T dY
// Bound by the matrix pipe (18 M F H operations a training pass), for few rows by the weights' bytes.  Everything is one tiled
// product kernel on v_mfma_f32_16x16x32_bf16 with fp32 accumulators:
//   * Both projections share one pass over X: a workgroup's tile holds the same columns of Wg and Wu, so that the gate and its
//     partner meet in one lane's registers and the epilogue writes A (and, for a backward, G and U).  dA never reaches memory
//     either: its epilogue reads G and U and writes dG and dU.  dX is one product over 2 H, dWg and dWu share X's tiles.
//   * fp32 operands are split exactly into three bf16 pieces (bf16_split.h); a product is then the sum of six piece products
//     (the dropped ones are below 2^-24), which the kernel runs as six SEGMENTS of one long k loop, small terms first.
//   * Tiles go from memory to LDS directly (buffer_load .. lds, 16 bytes per lane), two stages.  An operand whose rows run along k
//     is read back with ds_read_b128, one whose rows run across k (weights in X W, both operands in X^T dG) with the transposing
//     ds_read_b64_tr_b16: nothing is transposed in memory.  The 16-byte chunks of a tile row are permuted (xor with row bits) so
//     that the lanes of a read hit different banks; the permutation is in the GLOBAL addresses, the LDS image being linear.
//     Rows, columns and k beyond the operand read as zeros (the buffer's own bound).
//   * Few tiles for the chip: the k loop is cut into splits whose fp32 tiles a second kernel adds in order (no atomics) and
//     puts through the same epilogue.
// Roundings of bf16 calls: G, U, A, dG, dU are stored in bf16 for the products that read them (the matrix pipe takes bf16); sums,
// activations and their slopes are fp32.
#include <hip/hip_bf16.h>
#include <hip/hip_runtime.h>

#include <algorithm>

#include "bf16_split.h"
#include "sgc_kernels.h"

namespace agcn {
namespace {
typedef uint32_t u32x4u __attribute__((ext_vector_type(4), aligned(4)));   // at the alignment of an element: unaligned access mode
typedef uint32_t u32x4h __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2h __attribute__((ext_vector_type(2), aligned(2)));
#define AGCN_LDS __attribute__((address_space(3)))

constexpr int BK = 64;               // k of a stage
constexpr int kMaxSeg = 12;

enum { EPI_GATED = 0, EPI_STORE = 1, EPI_DH = 2 };

struct Seg { const uint16_t *a, *b, *b2; };

struct GemmArgs {
  Seg seg[kMaxSeg];
  int32_t nseg;
  int32_t M, N, K;                   // N: columns of one B matrix (two B matrices: of each)
  int32_t lda, ldb;
  int32_t ktiles, tiles_m, tiles_n, splits;
  float* part;                       // splits > 1: [split][B matrix][M][ldp] fp32
  int32_t ldp;
  // epilogue
  int32_t act, f32, planes;
  int32_t ldh;                       // leading dimension of G, U, A, dG, dU
  int64_t plane;                     // elements between the planes of A, dG, dU
  void *out, *out2;                  // EPI_STORE: [M, ldo]
  int32_t ldo;
  void *g, *u;                       // f32 or bf16
  uint16_t *hid, *dg, *du;           // bf16 pieces
};

__device__ __forceinline__ uint32_t pk_bf(float a, float b) {
  return __builtin_bit_cast(uint32_t, (bf16x2){(__bf16)a, (__bf16)b});
}

// act(g) and act'(g).  The slopes are formed from e^-|g| (no 1 - s where s is near 1).
__device__ __forceinline__ void gate_of(int act, float g, float& a, float& da) {
  if (act == AGCN_ACT_RELU) {
    a = g > 0.f ? g : 0.f;
    da = g > 0.f ? 1.f : 0.f;
    if (g != g) a = da = g;
  } else if (act == AGCN_ACT_GELU) {
    const float c = 0.5f * erfcf(-0.70710678f * g);
    a = g * c;
    da = fmaf(g, 0.39894228f * expf(-0.5f * g * g), c);
  } else {
    const float e = expf(-fabsf(g)), d = 1.f / (1.f + e);
    const float s = g >= 0.f ? d : e * d, ns = g >= 0.f ? e * d : d;    // sigmoid(g), sigmoid(-g)
    if (act == AGCN_ACT_SIGMOID) {
      a = s;
      da = s * ns;
    } else {
      a = g * s;
      da = s * fmaf(g, ns, 1.f);
    }
  }
}

__device__ __forceinline__ f32x4 load4(const void* p, int64_t at, bool f32) {       // 16- / 8-byte aligned rows of the library's own
  if (f32) return *reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + at);
  const u32x2 v = *reinterpret_cast<const u32x2*>(static_cast<const uint16_t*>(p) + at);
  return (f32x4){__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16), __uint_as_float(v.y & 0xffff0000u)};
}
__device__ __forceinline__ void store4(void* p, int64_t at, bool f32, f32x4 v) {
  if (f32) *reinterpret_cast<f32x4*>(static_cast<float*>(p) + at) = v;
  else *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(p) + at) = (u32x2){pk_bf(v.x, v.y), pk_bf(v.z, v.w)};
}
// the bf16 pieces of four values (planes == 1: the rounded value itself)
__device__ __forceinline__ void store_pieces(uint16_t* p, int64_t at, int planes, int64_t plane, f32x4 v) {
  if (planes == 1) {
    *reinterpret_cast<u32x2*>(p + at) = (u32x2){pk_bf(v.x, v.y), pk_bf(v.z, v.w)};
  } else {
    uint32_t h[2], m[2], l[2];
    split3(v.x, v.y, h[0], m[0], l[0]);
    split3(v.z, v.w, h[1], m[1], l[1]);
    *reinterpret_cast<u32x2*>(p + at) = (u32x2){h[0], h[1]};
    *reinterpret_cast<u32x2*>(p + plane + at) = (u32x2){m[0], m[1]};
    *reinterpret_cast<u32x2*>(p + 2 * plane + at) = (u32x2){l[0], l[1]};
  }
}
// four results of a caller's matrix: any alignment, any tail
__device__ __forceinline__ void store_out(void* p, int64_t row, int ld, int n, int N, bool f32, f32x4 v) {
  const int64_t at = row * ld + n;
  if (f32) {
    float* o = static_cast<float*>(p) + at;
    if (n + 4 <= N) {
      *reinterpret_cast<u32x4u*>(o) = (u32x4u){__float_as_uint(v.x), __float_as_uint(v.y), __float_as_uint(v.z), __float_as_uint(v.w)};
    } else {
      for (int i = 0; i < 4; ++i) if (n + i < N) o[i] = v[i];
    }
  } else {
    uint16_t* o = static_cast<uint16_t*>(p) + at;
    const uint32_t a = pk_bf(v.x, v.y), b = pk_bf(v.z, v.w);
    if (n + 4 <= N) {
      *reinterpret_cast<u32x2h*>(o) = (u32x2h){a, b};
    } else {
      if (n < N) o[0] = (uint16_t)a;
      if (n + 1 < N) o[1] = (uint16_t)(a >> 16);
      if (n + 2 < N) o[2] = (uint16_t)b;
    }
  }
}

// What becomes of four neighbouring columns n .. n + 3 of row m (v1: of the second B matrix)
template <int EPI, int NB>
__device__ __forceinline__ void epilogue(const GemmArgs& g, int m, int n, f32x4 v0, f32x4 v1) {
  const bool f32 = g.f32 != 0;
  if (EPI == EPI_STORE) {
    if (n >= g.N) return;
    store_out(g.out, m, g.ldo, n, g.N, f32, v0);
    if (NB == 2) store_out(g.out2, m, g.ldo, n, g.N, f32, v1);
    return;
  }
  // (the library's own matrices are padded to eights: the columns behind H get the zeros that the products read there)
  if (n >= g.ldh) return;
  const int64_t at = (int64_t)m * g.ldh + n;
  if (EPI == EPI_GATED) {
    f32x4 hv;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float a, da;
      gate_of(g.act, v0[i], a, da);
      hv[i] = n + i < g.N ? a * v1[i] : 0.f;
    }
    if (g.g) {
      store4(g.g, at, f32, v0);
      store4(g.u, at, f32, v1);
    }
    store_pieces(g.hid, at, g.planes, g.plane, hv);
  } else {
    const f32x4 gv = load4(g.g, at, f32), uv = load4(g.u, at, f32);
    f32x4 dg, du;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float a, da;
      gate_of(g.act, gv[i], a, da);
      dg[i] = n + i < g.N ? v0[i] * uv[i] * da : 0.f;
      du[i] = n + i < g.N ? v0[i] * a : 0.f;
    }
    store_pieces(g.dg, at, g.planes, g.plane, dg);
    store_pieces(g.du, at, g.planes, g.plane, du);
  }
}

#ifdef __HIP_DEVICE_COMPILE__      // (address spaces and builtins that the host pass does not know)
// One operand's tile of a stage: ROWS rows of the operand (m or n) by BK.  T (transposed): the operand's matrix is [k][rows].
template <int ROWS, bool T, int THREADS>
struct Tile {
  static constexpr int kSlots = ROWS * BK / 8 / THREADS;       // 16-byte chunks per thread
  static constexpr int kChunks = ROWS / 8;                     // T: chunks per k row
  static_assert(ROWS * BK / 8 % THREADS == 0, "whole chunks per thread");
  int voff[kSlots], kl[kSlots];

  // permutation of the chunks of k row k (T): flips 32-byte halves, so that the four k rows that sixteen lanes read, and the two
  // sets eight rows apart, lie in different banks
  static __device__ __forceinline__ int perm(int k) { return (((k & 3) | ((k >> 3) & 1) << 2) << 1) & (kChunks - 1); }

  __device__ __forceinline__ void init(int row0, int rows, int ld, int wave, int lane) {
#pragma unroll
    for (int i = 0; i < kSlots; ++i) {
      const int ci = (wave * kSlots + i) * 64 + lane;
      int r, k;
      if (T) {
        k = ci / kChunks;
        r = ((ci % kChunks) ^ perm(k)) * 8;
        voff[i] = (k * ld + r) * 2;
      } else {
        r = ci >> 3;
        k = ((ci & 7) ^ (r & 7)) * 8;
        voff[i] = (r * ld + k) * 2;
      }
      kl[i] = row0 + r < rows ? k : 0x7fffffff;
    }
  }
  // k tile kt of the operand at p (its row / column row0 already added) into LDS
  __device__ __forceinline__ void load(const uint16_t* p, int ld, int kt, int K, AGCN_LDS char* dst, int wave) const {
    const uint16_t* base = p + (T ? (int64_t)kt * BK * ld : (int64_t)kt * BK);
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(base), 0, 0x7fffffff, 0x00020000);
    const int left = K - kt * BK;
#pragma unroll
    for (int i = 0; i < kSlots; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (AGCN_LDS void*)(dst + (wave * kSlots + i) * 1024), 16,
                                               kl[i] < left ? voff[i] : (int)0x80000000, 0, 0, 0);
  }
};

// fragment f (16 rows from row r0 + 16 f) of k step kk (32 k): lane (r = lane & 15, q = lane / 16) gets k = 8 q .. 8 q + 7 of row r
template <int ROWS, bool T>
__device__ __forceinline__ u32x4 fragment(const AGCN_LDS char* s, int row, int kk, int lane) {
  const int l = lane & 15, q = lane >> 4;
  if (!T) {
    const int off = (row + l) * (BK * 2) + (((kk * 4 + q) ^ (l & 7)) << 4);
    return *reinterpret_cast<const AGCN_LDS u32x4*>(s + off);
  } else {
    const int k = kk * 32 + q * 8 + (l >> 2);
    const int chunk = ((row >> 3) + ((l & 3) >> 1)) ^ Tile<ROWS, true, 256>::perm(q * 8 + (l >> 2));
    const AGCN_LDS char* p = s + k * (ROWS * 2) + chunk * 16 + (l & 1) * 8;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((AGCN_LDS s16x4*)p);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((AGCN_LDS s16x4*)(p + 4 * ROWS * 2));
    const u32x2 a = __builtin_bit_cast(u32x2, lo), b = __builtin_bit_cast(u32x2, hi);
    return (u32x4){a.x, a.y, b.x, b.y};
  }
}

#endif

// BM x (NB x BN) tile by WGM x WGN waves; AT / BT: the operand's matrix has k along its rows
template <int BM, int BN, int WGM, int WGN, bool AT, bool BT, int NB, int EPI>
__global__ __launch_bounds__(64 * WGM * WGN) void ffn_gemm_kernel(GemmArgs g) {
#ifdef __HIP_DEVICE_COMPILE__
  constexpr int THREADS = 64 * WGM * WGN, FM = BM / WGM / 16, FN = BN / WGN / 16;
  constexpr int SA = BM * BK * 2, SB = BN * BK * 2;
  __shared__ __attribute__((aligned(1024))) char sA0[SA];
  __shared__ __attribute__((aligned(1024))) char sA1[SA];
  __shared__ __attribute__((aligned(1024))) char sB0[NB * SB];
  __shared__ __attribute__((aligned(1024))) char sB1[NB * SB];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WGN, wn = wave - wm * WGN;

  // workgroup -> tile: workgroups go round the eight dies; a die gets a run of neighbouring tiles (its L2 holds their operands),
  // and within a run four tile rows are walked together
  const int tiles = g.tiles_m * g.tiles_n, total = tiles * g.splits, run = (total + 7) >> 3;
  const int id = (blockIdx.x & 7) * run + (blockIdx.x >> 3);
  if (id >= total) return;
  const int tile = id / g.splits, split = id - tile * g.splits;
  const int per = 4 * g.tiles_n, grp = tile / per, first = grp * 4;
  const int rows_in = g.tiles_m - first < 4 ? g.tiles_m - first : 4;
  const int in = tile - grp * per, tm = first + in % rows_in, tn = in / rows_in;
  const int m0 = tm * BM, n0 = tn * BN;

  Tile<BM, AT, THREADS> ta;
  Tile<BN, BT, THREADS> tb;
  ta.init(m0, g.M, g.lda, wave, lane);
  tb.init(n0, g.N, g.ldb, wave, lane);
  const int64_t a_at = AT ? m0 : (int64_t)m0 * g.lda, b_at = BT ? n0 : (int64_t)n0 * g.ldb;

  const int iters = g.nseg * g.ktiles;
  const int it0 = (int)((int64_t)iters * split / g.splits), it1 = (int)((int64_t)iters * (split + 1) / g.splits);
  int seg = it0 / g.ktiles, kt = it0 - seg * g.ktiles;
  auto load = [&](AGCN_LDS char* a, AGCN_LDS char* b) {
    const Seg s = g.seg[seg];
    ta.load(s.a + a_at, g.lda, kt, g.K, a, wave);
    tb.load(s.b + b_at, g.ldb, kt, g.K, b, wave);
    if (NB == 2) tb.load(s.b2 + b_at, g.ldb, kt, g.K, b + SB, wave);
    if (++kt == g.ktiles) { kt = 0; ++seg; }
  };
  f32x4 acc[NB][FM][FN];
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) acc[b][i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
  auto compute = [&](const AGCN_LDS char* a, const AGCN_LDS char* b) {
#pragma unroll
    for (int kk = 0; kk < BK / 32; ++kk) {
      u32x4 fa[FM], fb[NB][FN];
#pragma unroll
      for (int i = 0; i < FM; ++i) fa[i] = fragment<BM, AT>(a, wm * FM * 16 + i * 16, kk, lane);
#pragma unroll
      for (int c = 0; c < NB; ++c)
#pragma unroll
        for (int j = 0; j < FN; ++j) fb[c][j] = fragment<BN, BT>(b + c * SB, wn * FN * 16 + j * 16, kk, lane);
      // (B as the first operand: a lane then holds four neighbouring COLUMNS of one row of the result)
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int c = 0; c < NB; ++c)
#pragma unroll
          for (int j = 0; j < FN; ++j) acc[c][i][j] = mfma_bf(fb[c][j], fa[i], acc[c][i][j]);
    }
  };
  // a stage is there when every wave's own transfers are (vmcnt) and all waves have said so
  auto ready = [] {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  };
  AGCN_LDS char *a0 = (AGCN_LDS char*)sA0, *a1 = (AGCN_LDS char*)sA1, *b0 = (AGCN_LDS char*)sB0, *b1 = (AGCN_LDS char*)sB1;
  int it = it0;
  if (it < it1) load(a0, b0);
  while (it < it1) {
    ready();
    if (it + 1 < it1) load(a1, b1);
    compute(a0, b0);
    if (++it >= it1) break;
    ready();
    if (it + 1 < it1) load(a0, b0);
    compute(a1, b1);
    ++it;
  }
  const int mr = lane & 15, nq = (lane >> 4) * 4;
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int m = m0 + (wm * FM + i) * 16 + mr;
    __builtin_amdgcn_sched_barrier(0);       // (the reads of G and U of one row of fragments in flight at a time: registers)
    if (m >= g.M) continue;
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int n = n0 + (wn * FN + j) * 16 + nq;
      if (g.splits > 1) {
        if (n < g.ldp) {
          float* p = g.part + (((int64_t)split * NB) * g.M + m) * g.ldp + n;
          *reinterpret_cast<f32x4*>(p) = acc[0][i][j];
          if (NB == 2) *reinterpret_cast<f32x4*>(p + (int64_t)g.M * g.ldp) = acc[NB - 1][i][j];
        }
      } else {
        epilogue<EPI, NB>(g, m, n, acc[0][i][j], acc[NB - 1][i][j]);
      }
    }
  }
#endif
}

// adds the splits' tiles in order and puts the sums through the epilogue; a thread takes four columns
template <int NB, int EPI>
__global__ __launch_bounds__(256) void ffn_reduce_kernel(GemmArgs g) {
  const int64_t per = g.ldp >> 2, e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= per * g.M) return;
  const int m = (int)(e / per), n = (int)(e - (int64_t)m * per) * 4;
  f32x4 v[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
  for (int s = 0; s < g.splits; ++s)
#pragma unroll
    for (int b = 0; b < NB; ++b)
      v[b] += *reinterpret_cast<const f32x4*>(g.part + (((int64_t)s * NB + b) * g.M + m) * g.ldp + n);
  epilogue<EPI, NB>(g, m, n, v[0], v[NB - 1]);
}

// Operand images: bf16 matrices whose rows do not start at 16 bytes or end at eights, padded with zeros; fp32 ones as three planes of
// bf16 pieces.  One launch for all matrices of a call; a thread makes eight columns.
struct Image { const void* src; uint16_t* dst; int64_t rows, plane, chunk0; int32_t cols, ld_src, ld_dst, f32; };
struct ImageArgs { Image im[4]; int32_t n; int64_t chunks; };
__global__ __launch_bounds__(256) void ffn_image_kernel(ImageArgs a) {
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= a.chunks) return;
  int k = 0;
  while (k + 1 < a.n && a.im[k + 1].chunk0 <= e) ++k;
  const Image& im = a.im[k];
  const int64_t at = e - im.chunk0, per = im.ld_dst >> 3, r = at / per;
  const int c = (int)(at - r * per) * 8;
  uint16_t* dst = im.dst + r * im.ld_dst + c;
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

__global__ __launch_bounds__(256) void ffn_zero_kernel(void* p, int64_t bytes) {
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e < bytes >> 1) static_cast<uint16_t*>(p)[e] = 0;
}

// ---- host side ---------------------------------------------------------------------------------------------------
inline int pad8(int v) { return (v + 7) & ~7; }
inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// A matrix as the products read it: its own memory where that is bf16 with rows at 16 bytes, an image otherwise
struct Mat { const uint16_t* p; int32_t ld; int64_t plane; };

struct Carve {
  char* base;
  size_t off;
  void* take(size_t bytes) {
    void* r = base ? base + off : nullptr;
    off += align256(bytes);
    return r;
  }
};

bool direct(const AgcnFfnDesc& d, const void* p, int cols, int ld) {
  return d.dtype == AGCN_DTYPE_BF16 && cols % 8 == 0 && ld % 8 == 0 && ((uintptr_t)p & 15) == 0;
}

// What the forward leaves for the backward.  The images are there only where a matrix cannot be read as it is; room is kept for
// them whenever the SIZES alone would not rule them out (an address can be odd).
struct Reserve { uint16_t *x, *wg, *wu, *wd, *hid; void *g, *u; };
size_t carve_reserve(const AgcnFfnDesc& d, void* mem, Reserve* r) {
  Carve c{static_cast<char*>(mem), 0};
  const int P = d.dtype == AGCN_DTYPE_F32 ? 3 : 1, Hp = pad8(d.H), Fp = pad8(d.Fin), Op = pad8(d.Fout);
  const size_t e = d.dtype == AGCN_DTYPE_F32 ? 4 : 2;
  r->x = static_cast<uint16_t*>(c.take((size_t)P * d.rows * Fp * 2));
  r->wg = static_cast<uint16_t*>(c.take((size_t)P * d.Fin * Hp * 2));
  r->wu = static_cast<uint16_t*>(c.take((size_t)P * d.Fin * Hp * 2));
  r->wd = static_cast<uint16_t*>(c.take((size_t)P * d.H * Op * 2));
  r->hid = static_cast<uint16_t*>(c.take((size_t)P * d.rows * Hp * 2));
  r->g = d.training ? c.take(e * d.rows * Hp) : nullptr;
  r->u = d.training ? c.take(e * d.rows * Hp) : nullptr;
  return c.off;
}

struct Config { int bm, bn, splits; };      // bn: columns of one B matrix

// Tile and splits for an [M, N] result over `iters` k stages with nb B matrices.
Config choose(int64_t M, int64_t N, int nb, int64_t iters) {
  const int bns = 256 / nb;
  if (cdiv(M, 256) * cdiv(N, bns) >= 192) return {256, bns, 1};
  if (cdiv(M, 128) * cdiv(N, 128 / nb) >= 256) return {128, 128 / nb, 1};
  const int64_t tiles = std::max<int64_t>(1, cdiv(M, 64) * cdiv(N, 64));    // (size queries come here with no rows, too)
  int64_t s = 1;
  if (tiles < 512) s = std::min(cdiv(1024, tiles), std::max<int64_t>(1, iters / 4));
  return {64, 64, (int)s};
}

size_t part_bytes(const Config& c, int64_t M, int64_t N, int nb) {
  return c.splits > 1 ? (size_t)c.splits * nb * M * ((N + 3) & ~3ll) * sizeof(float) : 0;
}

// segments of a product of two piece matrices, small terms first
int add_segments(GemmArgs* g, int at, const Mat& a, const Mat& b, const Mat* b2) {
  static const int ia[6] = {2, 0, 1, 1, 0, 0}, ib[6] = {0, 2, 1, 0, 1, 0};
  const int n = a.plane ? 6 : 1;
  for (int i = 0; i < n; ++i) {
    const int x = n == 1 ? 0 : ia[i], y = n == 1 ? 0 : ib[i];
    g->seg[at + i] = {a.p + x * a.plane, b.p + y * b.plane, b2 ? b2->p + y * b2->plane : nullptr};
  }
  return at + n;
}

template <int BM, int BN, int WGM, int WGN, bool AT, bool BT, int NB, int EPI>
void launch_tile(const GemmArgs& g, hipStream_t s) {
  const int64_t total = (int64_t)g.tiles_m * g.tiles_n * g.splits;
  hipLaunchKernelGGL((ffn_gemm_kernel<BM, BN, WGM, WGN, AT, BT, NB, EPI>), dim3((unsigned)(cdiv(total, 8) * 8)), dim3(64 * WGM * WGN), 0, s, g);
}

template <bool AT, bool BT, int NB, int EPI>
void product(GemmArgs& g, void* part, hipStream_t s) {
  g.ktiles = (int)cdiv(g.K, BK);
  const int n_all = EPI == EPI_STORE ? g.N : g.ldh;         // columns that the epilogue has to reach
  const Config c = choose(g.M, n_all, NB, (int64_t)g.nseg * g.ktiles);
  g.tiles_m = (int)cdiv(g.M, c.bm); g.tiles_n = (int)cdiv(n_all, c.bn); g.splits = c.splits;
  g.part = static_cast<float*>(part); g.ldp = (n_all + 3) & ~3;
  if (c.bm == 256) launch_tile<256, 256 / NB, 2, 4, AT, BT, NB, EPI>(g, s);
  else if (c.bm == 128) launch_tile<128, 128 / NB, 2, 2, AT, BT, NB, EPI>(g, s);
  else launch_tile<64, 64, 2, 2, AT, BT, NB, EPI>(g, s);
  if (g.splits > 1)
    hipLaunchKernelGGL((ffn_reduce_kernel<NB, EPI>), dim3((unsigned)cdiv((int64_t)g.M * (g.ldp / 4), 256)), dim3(256), 0, s, g);
}

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

struct ImageList {
  ImageArgs a;
  ImageList() { std::memset(&a, 0, sizeof(a)); }
  Mat add(const AgcnFfnDesc& d, const void* src, int64_t rows, int cols, int ld, uint16_t* dst) {
    if (direct(d, src, cols, ld)) return {static_cast<const uint16_t*>(src), ld, 0};
    const bool f32 = d.dtype == AGCN_DTYPE_F32;
    const int lp = pad8(cols);
    Image& im = a.im[a.n++];
    im = {src, dst, rows, rows * lp, a.chunks, cols, ld, lp, f32 ? 1 : 0};
    a.chunks += rows * (lp >> 3);
    return {dst, lp, f32 ? im.plane : 0};
  }
  void launch(hipStream_t s) const {
    if (a.chunks) hipLaunchKernelGGL(ffn_image_kernel, dim3((unsigned)cdiv(a.chunks, 256)), dim3(256), 0, s, a);
  }
};
// the same matrix in the backward, whose image the forward has left
Mat same(const AgcnFfnDesc& d, const void* src, int64_t rows, int cols, int ld, uint16_t* img) {
  if (direct(d, src, cols, ld)) return {static_cast<const uint16_t*>(src), ld, 0};
  return {img, pad8(cols), d.dtype == AGCN_DTYPE_F32 ? rows * pad8(cols) : 0};
}

GemmArgs base_args(const AgcnFfnDesc& d) {
  GemmArgs g;
  std::memset(&g, 0, sizeof(g));
  g.act = d.activation; g.f32 = d.dtype == AGCN_DTYPE_F32; g.planes = g.f32 ? 3 : 1;
  g.ldh = pad8(d.H); g.plane = (int64_t)d.rows * g.ldh;
  return g;
}
int nsegs(const AgcnFfnDesc& d) { return d.dtype == AGCN_DTYPE_F32 ? 6 : 1; }

size_t forward_part(const AgcnFfnDesc& d) {
  const int ns = nsegs(d), Hp = pad8(d.H);
  return std::max(part_bytes(choose(d.rows, Hp, 2, ns * cdiv(d.Fin, BK)), d.rows, Hp, 2),
                  part_bytes(choose(d.rows, d.Fout, 1, ns * cdiv(d.H, BK)), d.rows, d.Fout, 1));
}
struct BackWs { uint16_t *dy, *dg, *du; void* part; };
size_t carve_backward(const AgcnFfnDesc& d, void* mem, BackWs* w) {
  const int ns = nsegs(d), P = ns == 6 ? 3 : 1, Hp = pad8(d.H);
  Carve c{static_cast<char*>(mem), 0};
  w->dy = static_cast<uint16_t*>(c.take((size_t)P * d.rows * pad8(d.Fout) * 2));
  w->dg = static_cast<uint16_t*>(c.take((size_t)P * d.rows * Hp * 2));
  w->du = static_cast<uint16_t*>(c.take((size_t)P * d.rows * Hp * 2));
  const size_t part = std::max(std::max(part_bytes(choose(d.rows, Hp, 1, ns * cdiv(d.Fout, BK)), d.rows, Hp, 1),
                                        part_bytes(choose(d.rows, d.Fin, 1, 2 * ns * cdiv(d.H, BK)), d.rows, d.Fin, 1)),
                               std::max(part_bytes(choose(d.Fin, d.H, 2, ns * cdiv(d.rows, BK)), d.Fin, d.H, 2),
                                        part_bytes(choose(d.H, d.Fout, 1, ns * cdiv(d.rows, BK)), d.H, d.Fout, 1)));
  w->part = c.take(part);
  return c.off;
}
void zero(void* p, int64_t bytes, hipStream_t s) {
  hipLaunchKernelGGL(ffn_zero_kernel, dim3((unsigned)cdiv(bytes / 2, 256)), dim3(256), 0, s, p, bytes);
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
  if (!X || !Wg || !Wu || !Wd || !Y) return fail(AGCN_EINVAL, "%s: null tensor", who);
  Reserve r;
  const size_t need = carve_reserve(d, reserve, &r), wneed = forward_part(d);
  if (!reserve || ((uintptr_t)reserve & 255) || reserve_bytes < need)
    return fail(AGCN_ENOSPACE, "%s: reserve too small or not at 256 bytes (%zu < %zu)", who, reserve_bytes, need);
  if (wneed && (!workspace || ((uintptr_t)workspace & 255) || workspace_bytes < wneed))
    return fail(AGCN_ENOSPACE, "%s: workspace too small or not at 256 bytes (%zu < %zu)", who, workspace_bytes, wneed);
  hipStream_t s = static_cast<hipStream_t>(hip_stream);
  ImageList list;
  const Mat x = list.add(d, X, d.rows, d.Fin, d.ldx, r.x), wg = list.add(d, Wg, d.Fin, d.H, d.H, r.wg);
  // (read in place or as an image, both projections have one leading dimension: in place only if H is a multiple of eight)
  const Mat wu = list.add(d, Wu, d.Fin, d.H, d.H, r.wu);
  const Mat wd = list.add(d, Wd, d.H, d.Fout, d.Fout, r.wd);
  list.launch(s);
  GemmArgs g = base_args(d);
  g.nseg = add_segments(&g, 0, x, wg, &wu);
  g.M = (int)d.rows; g.N = d.H; g.K = d.Fin; g.lda = x.ld; g.ldb = wg.ld;
  g.g = r.g; g.u = r.u; g.hid = r.hid;
  product<false, true, 2, EPI_GATED>(g, workspace, s);
  const Mat hid = {r.hid, g.ldh, g.f32 ? g.plane : 0};
  GemmArgs q = base_args(d);
  q.nseg = add_segments(&q, 0, hid, wd, nullptr);
  q.M = (int)d.rows; q.N = d.Fout; q.K = d.H; q.lda = hid.ld; q.ldb = wd.ld;
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
  if (!X || !Wg || !Wu || !Wd || !dY) return fail(AGCN_EINVAL, "%s: null tensor", who);
  Reserve r;
  BackWs w;
  const size_t need = carve_reserve(d, const_cast<void*>(reserve), &r), wneed = carve_backward(d, workspace, &w);
  if (!reserve || ((uintptr_t)reserve & 255) || reserve_bytes < need)
    return fail(AGCN_ENOSPACE, "%s: reserve too small or not at 256 bytes (%zu < %zu)", who, reserve_bytes, need);
  if (!workspace || ((uintptr_t)workspace & 255) || workspace_bytes < wneed)
    return fail(AGCN_ENOSPACE, "%s: workspace too small or not at 256 bytes (%zu < %zu)", who, workspace_bytes, wneed);
  const Mat x = same(d, X, d.rows, d.Fin, d.ldx, r.x), wg = same(d, Wg, d.Fin, d.H, d.H, r.wg), wu = same(d, Wu, d.Fin, d.H, d.H, r.wu),
            wd = same(d, Wd, d.H, d.Fout, d.Fout, r.wd);
  ImageList list;
  const Mat dy = list.add(d, dY, d.rows, d.Fout, d.Fout, w.dy);
  list.launch(s);
  GemmArgs base = base_args(d);
  const int64_t pl = base.f32 ? base.plane : 0;
  const Mat hid = {r.hid, base.ldh, pl}, dg = {w.dg, base.ldh, pl}, du = {w.du, base.ldh, pl};
  if (dX || dWg) {
    GemmArgs g = base;                        // dA = dY Wd^T, and from it dG and dU
    g.nseg = add_segments(&g, 0, dy, wd, nullptr);
    g.M = (int)d.rows; g.N = d.H; g.K = d.Fout; g.lda = dy.ld; g.ldb = wd.ld;
    g.g = r.g; g.u = r.u; g.dg = w.dg; g.du = w.du;
    product<false, false, 1, EPI_DH>(g, w.part, s);
  }
  if (dX) {
    GemmArgs g = base;
    g.nseg = add_segments(&g, add_segments(&g, 0, dg, wg, nullptr), du, wu, nullptr);
    g.M = (int)d.rows; g.N = d.Fin; g.K = d.H; g.lda = dg.ld; g.ldb = wg.ld;
    g.out = dX; g.ldo = d.Fin;
    product<false, false, 1, EPI_STORE>(g, w.part, s);
  }
  if (dWg) {
    GemmArgs g = base;
    g.nseg = add_segments(&g, 0, x, dg, &du);
    g.M = d.Fin; g.N = d.H; g.K = (int)d.rows; g.lda = x.ld; g.ldb = dg.ld;
    g.out = dWg; g.out2 = dWu; g.ldo = d.H;
    product<true, true, 2, EPI_STORE>(g, w.part, s);
  }
  if (dWd) {
    GemmArgs g = base;
    g.nseg = add_segments(&g, 0, hid, dy, nullptr);
    g.M = d.H; g.N = d.Fout; g.K = (int)d.rows; g.lda = hid.ld; g.ldb = dy.ld;
    g.out = dWd; g.ldo = d.Fout;
    product<true, true, 1, EPI_STORE>(g, w.part, s);
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(AGCN_EDEVICE, "%s: %s", who, hipGetErrorString(e));
  return AGCN_OK;
}
