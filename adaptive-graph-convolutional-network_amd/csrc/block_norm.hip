// The frame of a residual block in one pass over the rows: the norm behind the block, its gate and residual scale, the residual
// sum, and the norm in front of the next block (beside BlockEnd, models/layers/blockend.py:67-86, whose sum has neither):
//     u = N(z; w, b)          N: rms  v / sqrt(mean v^2 + eps) * w   |   layer  (v - mean v) / sqrt(var v + eps) * w + b
//     y = x + s (.) a(g) (.) u
//     h = N(y; w', b')
// Backward, with D = dy + N'(dh; y):
//     dx = D;  dg = D s u a'(g);  dz = N'(D s a(g); z);  N'(d; v) = r (d w - vh mean(d w vh) [- mean(d w)]),  vh = (v [- mean]) r
//     with q1 = sum D a zh and q2 = sum D a over the rows:  dw = s q1, db = s q2, ds = w q1 + b q2;
//     dw' = sum dh yh, db' = sum dh;  a gate per graph:  dg = a'(g) s (w sum D zh + b sum D) over the graph's rows.
// Bound by memory: every operand is read once and every result written once (the row stays in registers between the two norms
// and through all reductions).  L lanes share a row (eight consecutive elements per lane, so that a lane keeps the parameters and
// the column sums of ITS columns in registers over all rows it meets); few elements per lane and many waves, which hide the
// memory's latency where a row after another would not.  Sums, means and column sums are fp32 (a column sum's partials, one per
// workgroup, are added in a fixed order: no atomics); rounding happens where a result is stored, and h is taken from the unrounded
// y.  Pad rows give zeros and take part in no sum.
// Measured, forward / backward, a profile's averages: 32916 x 4096 bf16 203 / 381 us (1074 MB: 5.3 TB/s; 1611 MB: 4.2 TB/s, registers
// leave half of the forward's waves); 19202 x 1001, fp32 rows, bf16 z and a gate per element 68 / 121 us (4.0 and 3.5 TB/s: rows at odd
// addresses, sigmoids); 4071 x 256 fp32 with a gate per graph 8.6 / 23 us in three launches.
// Wide rows spill.  The backwards of 1025 to 4096 features without gate and means spill 14 registers (60 bytes a lane) to the rows
// fetched ahead, which pays all the same; fp32-row gated layer norms of 2049 to 4096 2 to 4; from 4097 on the layer norms' backwards
// 20 to 65, beyond 8192, with two vectors a lane, every kernel 4 to 326.  134 M elements, forward / backward in TB/s: 4096 features bf16 rms
// 4.8 / 4.4, layer 4.0 / 3.2, fp32 gated layer 5.0 / 5.0; 8192 4.7 / 4.3, 3.8 / 3.6, 5.2 / 3.8; 16384 4.9 / 2.7, 2.9 / 1.4, 3.3 / 1.9;
// rows of odd widths beyond 4096 (5001) 2.2 / 1.9, 1.9 / 1.8, 3.3 / 2.5.
#include <hip/hip_bf16.h>
#include <hip/hip_runtime.h>

#include <algorithm>

#include "agcn_device.h"
#include "gate_math.h"
#include "sgc_kernels.h"

namespace agcn {
namespace {
constexpr int V = 8;                    // elements per vector

struct NormArgs {
  AgcnNormDesc d;
  // plan (nullable: no pad rows, no graphs)
  const int32_t *n, *row_off, *row_graph;
  int32_t B, graph_log2;                // per-graph gates: log2 of the rows of a graph that one workgroup adds up
  const void *z, *x, *gate, *dy, *dh;
  const float *scale, *w, *b, *w2, *b2;
  void *y, *h, *dz, *dx, *dgate;
  float* stats;                         // [rows][4]: mean z, 1 / deviation of z, mean y, 1 / deviation of y
  float* part;                          // [units][4][F]; with a gate per graph the first B become the graphs' own
  int32_t units, pads;                  // partial sums
};

typedef uint32_t u4f __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u4h __attribute__((ext_vector_type(4), aligned(2)));

// eight elements, columns c .. c + 7 of a row of F (0 beyond), as floats.  Vectors are read at the alignment of an element: the
// target runs in unaligned access mode, and odd widths start every row elsewhere.
// In two halves: the memory's bits first (so that a row's can be in flight while the row before it is worked on), then floats.
template <typename T> struct Raw;
template <> struct Raw<float> { u4f a, b; };
template <> struct Raw<__hip_bfloat16> { u4h a; };
__device__ __forceinline__ void fetch8(const float* p, int c, int F, Raw<float>& r) {
  if (c + V <= F) {
    r.a = *reinterpret_cast<const u4f*>(p + c);
    r.b = *reinterpret_cast<const u4f*>(p + c + 4);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      r.a[i] = c + i < F ? __float_as_uint(p[c + i]) : 0u;
      r.b[i] = c + 4 + i < F ? __float_as_uint(p[c + 4 + i]) : 0u;
    }
  }
}
__device__ __forceinline__ void fetch8(const __hip_bfloat16* p_, int c, int F, Raw<__hip_bfloat16>& r) {
  const uint16_t* p = reinterpret_cast<const uint16_t*>(p_);
  if (c + V <= F) {
    r.a = *reinterpret_cast<const u4h*>(p + c);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      r.a[i] = (c + 2 * i < F ? (uint32_t)p[c + 2 * i] : 0u) | (c + 2 * i + 1 < F ? (uint32_t)p[c + 2 * i + 1] << 16 : 0u);
  }
}
__device__ __forceinline__ void unpack8(const Raw<float>& r, float* v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) { v[i] = __uint_as_float(r.a[i]); v[4 + i] = __uint_as_float(r.b[i]); }
}
__device__ __forceinline__ void unpack8(const Raw<__hip_bfloat16>& r, float* v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(r.a[i] << 16); v[2 * i + 1] = __uint_as_float(r.a[i] & 0xffff0000u); }
}
__device__ __forceinline__ void clear8(Raw<float>& r) { r.a = (u4f)(0u); r.b = (u4f)(0u); }
__device__ __forceinline__ void clear8(Raw<__hip_bfloat16>& r) { r.a = (u4h)(0u); }

__device__ __forceinline__ void load8(const float* p, int c, int F, float* v) {
  Raw<float> r;
  fetch8(p, c, F, r);
  unpack8(r, v);
}

__device__ __forceinline__ void store8(float* p, int c, int F, const float* v) {
  if (c + V <= F) {
    u4f a, b;
#pragma unroll
    for (int i = 0; i < 4; ++i) { a[i] = __float_as_uint(v[i]); b[i] = __float_as_uint(v[4 + i]); }
    *reinterpret_cast<u4f*>(p + c) = a;
    *reinterpret_cast<u4f*>(p + c + 4) = b;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) if (c + i < F) p[c + i] = v[i];
  }
}
__device__ __forceinline__ uint32_t pk_bf(float a, float b) {
  typedef __bf16 b2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, (b2){(__bf16)a, (__bf16)b});
}
__device__ __forceinline__ void store8(__hip_bfloat16* p_, int c, int F, const float* v) {
  uint16_t* p = reinterpret_cast<uint16_t*>(p_);
  if (c + V <= F) {
    u4h a;
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = pk_bf(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<u4h*>(p + c) = a;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) if (c + i < F) p[c + i] = (uint16_t)pk_bf(v[i], 0.f);
  }
}

// The gate's activation and its slope, which is formed from e^-|g| (1 - a^2 and a (1 - a) lose their digits where the activation is flat).
// tanh below 1/4: its series (1 - e^-2|g| loses digits there; the first term left out is 2^-26 of the sum).
__device__ __forceinline__ float series_tanh(float g) {
  const float t = g * g;
  return fmaf(g * t, fmaf(t, fmaf(t, fmaf(t, 0.021869489f, -0.053968254f), 0.13333333f), -0.33333333f), g);
}
// N gates: one branch on the activation for all.  (Against the library's functions, called for each value where it was needed: 19202 x 1001
// with sigmoids forward 71 -> 66, backward 134 -> 120 us.)
template <int N>
__device__ __forceinline__ void gates(int act, const float (&g)[N], float (&a)[N], float (&slope)[N]) {
  if (act == AGCN_ACT_SIGMOID) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float e = exp_neg(fabsf(g[i])), d = recip_1p(e);
      a[i] = g[i] >= 0.f ? d : e * d;
      slope[i] = e * d * d;
    }
  } else if (act == AGCN_ACT_TANH) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float e = exp_neg(2.f * fabsf(g[i])), d = recip_1p(e);
      a[i] = fabsf(g[i]) < 0.25f ? series_tanh(g[i]) : copysignf((1.f - e) * d, g[i]);
      slope[i] = 4.f * e * d * d;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      a[i] = g[i];
      slope[i] = 1.f;
    }
  }
}

// Sums of N values over the L lanes of a row; every lane gets them.  L > 64: over the row's waves through `red`
// (two areas used in turn, so that one barrier per call is enough).
template <int L, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float* red, int& turn) {
#pragma unroll
  for (int o = (L < 64 ? L : 64) >> 1; o; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor(v[i], o);
  if (L > 64) {
    constexpr int W = L > 64 ? L / 64 : 1;
    float* r = red + turn * 32;
    turn ^= 1;
    const int wave = threadIdx.x >> 6, first = wave / W * W;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) r[wave * 2 + i] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) s += r[(first + w) * 2 + i];
      v[i] = s;
    }
  }
}

template <int L> constexpr int threads_of() { return L < 256 ? 256 : L; }

// Normalises the row in place: v -> vh; returns mean and 1 / deviation.  Two passes over the registers: the sum of squares is
// taken around the mean, not as a difference of two large sums.
template <int L, int NV, bool LAYER>
__device__ __forceinline__ void normalise(float (&v)[NV][V], const NormArgs& a, int lane, float& mean, float& r, float* red, int& turn) {
  const float inv = 1.f / (float)a.d.F;
  mean = 0.f;
  if (LAYER) {
    float s[1] = {0.f};
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) s[0] += v[k][i];          // (columns beyond F hold 0)
    row_sums<L, 1>(s, red, turn);
    mean = s[0] * inv;
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) v[k][i] = (k * L + lane) * V + i < a.d.F ? v[k][i] - mean : 0.f;
  }
  float q[1] = {0.f};
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) q[0] = fmaf(v[k][i], v[k][i], q[0]);
  row_sums<L, 1>(q, red, turn);
  r = 1.f / sqrtf(fmaf(q[0], inv, a.d.eps));
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) v[k][i] *= r;
}

// eight parameters, or `none` where there are none
__device__ __forceinline__ void load_param(const float* p, int c, int F, float none, float* v) {
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = none;
  if (p) load8(p, c, F, v);
}

__device__ __forceinline__ bool is_pad(const NormArgs& a, int64_t row) {
  if (!a.pads) return false;
  const int g = a.row_graph[row];
  return (int)row - a.row_off[g] >= a.n[g];
}

// A gate per graph: the strips of S = 2^graph_log2 rows that the graphs are cut into, each from its first row on.  Place g: the first
// strip of graph g.  Place B + e: the graph that holds row (e + 1) S - 1, its strip e - row_off / S + 1 (of those there are, or one
// behind the graph's end: nothing).  That gives every further strip a place of its own -- a graph of n rows has at most as many as there
// are such rows in it --, needs one load, and rows / S + B places, however the rows are spread over the graphs.
__device__ __forceinline__ int strip_place(const NormArgs& a, int g, int strip) {
  return strip ? a.B + (a.row_off[g] >> a.graph_log2) + strip - 1 : g;
}
__device__ __forceinline__ int strip_at(const NormArgs& a, int place, int& g) {
  g = place;
  if (place < a.B) return 0;
  const int e = place - a.B;
  g = a.row_graph[((e + 1) << a.graph_log2) - 1];
  return e - (a.row_off[g] >> a.graph_log2) + 1;
}

template <typename TX, typename TZ, int L, int NV, bool LAYER>
__global__ __launch_bounds__(threads_of<L>()) void norm_forward_kernel(NormArgs a) {
  constexpr int R = threads_of<L>() / L;                    // rows side by side
  __shared__ float red[64];
  const int lane = threadIdx.x % L, F = a.d.F;
  int turn = 0;
  // s w, s b, w', b': y = x + a(g) (zh sw + sb)
  float sw[NV][V], sb[LAYER ? NV : 1][V], w2[NV][V], b2[LAYER ? NV : 1][V];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (k * L + lane) * V;
    float s[V];
    load_param(a.scale, c, F, 1.f, s);
    load_param(a.w, c, F, 1.f, sw[k]);
    load_param(a.w2, c, F, 1.f, w2[k]);
    if (LAYER) {
      load_param(a.b, c, F, 0.f, sb[k]);
      load_param(a.b2, c, F, 0.f, b2[k]);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      sw[k][i] *= s[i];
      if (LAYER) sb[k][i] *= s[i];
    }
  }
  const int64_t step = (int64_t)gridDim.x * R;
  Raw<TX> nx[NV];
  Raw<TZ> nz[NV], ng[NV];
  bool nlive, nuse;
  auto fetch = [&](int64_t row) {
    nlive = row < a.d.rows;
    nuse = nlive && !is_pad(a, row);
    const int64_t grow = a.d.gate == AGCN_GATE_GRAPH ? (nlive ? a.row_graph[row] : 0) : row;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * L + lane) * V;
      clear8(nx[k]); clear8(nz[k]); clear8(ng[k]);
      if (nuse) {
        fetch8(static_cast<const TX*>(a.x) + row * a.d.ldx, c, F, nx[k]);
        if (a.z) fetch8(static_cast<const TZ*>(a.z) + row * a.d.ldz, c, F, nz[k]);
        if (a.gate) fetch8(static_cast<const TZ*>(a.gate) + grow * a.d.ldg, c, F, ng[k]);
      }
    }
  };
  fetch((int64_t)blockIdx.x * R + threadIdx.x / L);
  // (the loop runs on the workgroup's first row: all its lanes meet at the barriers of row_sums)
  for (int64_t r0 = (int64_t)blockIdx.x * R; r0 < a.d.rows; r0 += step) {
    const int64_t row = r0 + threadIdx.x / L;
    const bool live = nlive, use = nuse;
    float y[NV][V], zz[NV][V], g[NV][V];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      unpack8(nx[k], y[k]);
      unpack8(nz[k], zz[k]);
      unpack8(ng[k], g[k]);
    }
    fetch(row + step);
    float mz = 0.f, rz = 1.f, my = 0.f, ry = 1.f;
    if (a.z) {
      if (a.w) normalise<L, NV, LAYER>(zz, a, lane, mz, rz, red, turn);
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = (k * L + lane) * V;
        float slope[V];
        if (a.gate) {
          const float (&gk)[V] = g[k];
          float act[V];
          gates<V>(a.d.gate_activation, gk, act, slope);
#pragma unroll
          for (int i = 0; i < V; ++i) g[k][i] = act[i];
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float ga = a.gate ? g[k][i] : 1.f;
          const float u = LAYER ? fmaf(zz[k][i], sw[k][i], sb[k][i]) : zz[k][i] * sw[k][i];
          y[k][i] = c + i < F && use ? fmaf(ga, u, y[k][i]) : 0.f;
        }
        if (live) store8(static_cast<TX*>(a.y) + row * F, c, F, y[k]);
      }
    }
    if (a.h) {
      normalise<L, NV, LAYER>(y, a, lane, my, ry, red, turn);
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = (k * L + lane) * V;
        float o[V];
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = !use ? 0.f : (LAYER ? fmaf(y[k][i], w2[k][i], b2[k][i]) : y[k][i] * w2[k][i]);
        if (live) store8(static_cast<TZ*>(a.h) + row * F, c, F, o);
      }
    }
    if (a.stats && live && lane == 0) *reinterpret_cast<f32x4*>(a.stats + row * 4) = (f32x4){mz, rz, my, ry};
  }
}

// One workgroup walks a strip of rows (no gate per graph: rows block, block + grid, ..; with one: up to 2^graph_log2 rows of one
// graph) and leaves the partial sums of its columns: q1, q2 (per graph: sum D zh, sum D), q3 = sum dh yh, q4 = sum dh (q2 and q4
// for the biases of layer norms alone).
// y is formed again from x, z and the gate, which have to be read anyway (x in y's place): the stored y may be rounded to
// bf16, and a row whose features differ by less than that rounding would get a wrong yh.
// AHEAD: the next row's operands are fetched while a row is worked on.  It pays where it costs few registers (bf16 rows, no gate, no
// means: 32916 x 4096 463 -> 395 us on average, although 14 registers are spilled for it); with more it costs more than it gives.
template <typename TX, typename TZ, int L, int NV, bool LAYER, bool GATED>
__global__ __launch_bounds__(threads_of<L>(), LAYER || GATED ? 3 : 4) void norm_backward_kernel(NormArgs a) {
  constexpr bool AHEAD = !LAYER && !GATED && NV == 1 && sizeof(TX) == 2;
  constexpr int T = threads_of<L>(), R = T / L, NL = LAYER ? NV : 1;
  __shared__ float red[64];
  __shared__ float cols[R > 1 ? T * V : 1];
  const int lane = threadIdx.x % L, rl = threadIdx.x / L, F = a.d.F;
  int turn = 0;
  const float inv = 1.f / (float)F;
  const bool per_graph = GATED && a.d.gate == AGCN_GATE_GRAPH;
  int64_t row_begin, row_end, step;
  if (per_graph) {
    int g;
    const int strip = strip_at(a, blockIdx.x, g), r1 = a.row_off[g + 1];   // pad rows too: their gradients are written (0)
    row_begin = a.row_off[g] + ((int64_t)strip << a.graph_log2);
    if (row_begin >= r1) return;
    row_end = row_begin + (1 << a.graph_log2);
    if (row_end > r1) row_end = r1;
    step = R;
  } else {
    row_begin = (int64_t)blockIdx.x * R;
    row_end = a.d.rows;
    step = (int64_t)gridDim.x * R;
  }
  float q1[NV][V], q2[NL][V], q3[NV][V], q4[NL][V];
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      q1[k][i] = 0.f; q3[k][i] = 0.f;
      if (LAYER) { q2[k][i] = 0.f; q4[k][i] = 0.f; }
    }
  Raw<TX> nx[NV], ny[NV];
  Raw<TZ> nz[NV], ng[NV], nh[NV];
  f32x4 nst;
  bool nlive, nuse;
  auto fetch = [&](int64_t row) {
    nlive = row < row_end;
    nuse = nlive && !is_pad(a, row);
    nst = (f32x4){0.f, 1.f, 0.f, 1.f};
    if (nuse) nst = *reinterpret_cast<const f32x4*>(a.stats + row * 4);
    const int64_t grow = per_graph ? (nlive ? a.row_graph[row] : 0) : row;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * L + lane) * V;
      clear8(nx[k]); clear8(ny[k]); clear8(nz[k]); clear8(ng[k]); clear8(nh[k]);
      if (nuse) {
        fetch8(static_cast<const TX*>(a.x) + row * a.d.ldx, c, F, nx[k]);
        if (a.z) fetch8(static_cast<const TZ*>(a.z) + row * a.d.ldz, c, F, nz[k]);
        if (GATED) fetch8(static_cast<const TZ*>(a.gate) + grow * a.d.ldg, c, F, ng[k]);
        if (a.dy) fetch8(static_cast<const TX*>(a.dy) + row * F, c, F, ny[k]);
        if (a.dh) fetch8(static_cast<const TZ*>(a.dh) + row * F, c, F, nh[k]);
      }
    }
  };
  if (AHEAD) fetch(row_begin + rl);
  for (int64_t r0 = row_begin; r0 < row_end; r0 += step) {
    const int64_t row = r0 + rl;
    if (!AHEAD) fetch(row);
    const bool live = nlive, use = nuse;
    const f32x4 st = nst;
    // D: the gradient of y (dx); e: dh, then times w'; yh: y, then normalised; zh; g: the gate's activation, its slope
    float D[NV][V], e[NV][V], yh[NV][V], zh[NV][V], g[NV][V], slope[NV][V];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      unpack8(nx[k], yh[k]);
      unpack8(nz[k], zh[k]);
      if (GATED) {
        float before[V];
        unpack8(ng[k], before);
        gates<V>(a.d.gate_activation, before, g[k], slope[k]);
      }
      unpack8(ny[k], D[k]);
      unpack8(nh[k], e[k]);
    }
    if (AHEAD) fetch(row + step);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * L + lane) * V;
      if (a.z) {
        float s[V], w[V], b[V];
        load_param(a.scale, c, F, 1.f, s);
        load_param(a.w, c, F, 1.f, w);
        if (LAYER) load_param(a.b, c, F, 0.f, b);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          zh[k][i] = c + i < F && use ? (LAYER ? zh[k][i] - st.x : zh[k][i]) * st.y : 0.f;   // (no post norm: mean 0, deviation 1)
          const float ga = GATED ? g[k][i] : 1.f;
          const float sw = s[i] * w[i], u = LAYER ? fmaf(zh[k][i], sw, s[i] * b[i]) : zh[k][i] * sw;
          yh[k][i] = fmaf(ga, u, yh[k][i]);
        }
      }
    }
    if (a.dh) {
      float m[2] = {0.f, 0.f};
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = (k * L + lane) * V;
        float w2[V];
        load8(a.w2, c, F, w2);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          yh[k][i] = c + i < F && use ? (LAYER ? yh[k][i] - st.z : yh[k][i]) * st.w : 0.f;
          q3[k][i] = fmaf(e[k][i], yh[k][i], q3[k][i]);
          if (LAYER) q4[k][i] += e[k][i];
          e[k][i] *= w2[i];
          m[0] = fmaf(e[k][i], yh[k][i], m[0]);
          if (LAYER) m[1] += e[k][i];
        }
      }
      row_sums<L, LAYER ? 2 : 1>(reinterpret_cast<float(&)[LAYER ? 2 : 1]>(m), red, turn);
      const float m0 = m[0] * inv, m1 = LAYER ? m[1] * inv : 0.f;
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) D[k][i] = fmaf(st.w, e[k][i] - fmaf(yh[k][i], m0, m1), D[k][i]);
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * L + lane) * V;
#pragma unroll
      for (int i = 0; i < V; ++i) D[k][i] = c + i < F && use ? D[k][i] : 0.f;
      if (live) store8(static_cast<TX*>(a.dx) + row * F, c, F, D[k]);
    }
    if (a.z) {
      float m[2] = {0.f, 0.f};
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = (k * L + lane) * V;
        float s[V], w[V], b[V], dg[V];
        load_param(a.scale, c, F, 1.f, s);
        load_param(a.w, c, F, 1.f, w);
        if (LAYER) load_param(a.b, c, F, 0.f, b);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float ga = GATED ? g[k][i] : 1.f;
          const float Dq = per_graph ? D[k][i] : D[k][i] * ga;
          q1[k][i] = fmaf(Dq, zh[k][i], q1[k][i]);
          if (LAYER) q2[k][i] += Dq;
          const float u = LAYER ? fmaf(zh[k][i], w[i], b[i]) : zh[k][i] * w[i];
          dg[i] = GATED ? D[k][i] * s[i] * u * slope[k][i] : 0.f;
          D[k][i] *= s[i] * ga * w[i];                                 // gradient of zh
          m[0] = fmaf(D[k][i], zh[k][i], m[0]);
          if (LAYER) m[1] += D[k][i];
        }
        if (GATED && a.d.gate == AGCN_GATE_ROW && live) store8(static_cast<TZ*>(a.dgate) + row * F, c, F, dg);
      }
      float m0 = 0.f, m1 = 0.f;
      if (a.w) {
        row_sums<L, LAYER ? 2 : 1>(reinterpret_cast<float(&)[LAYER ? 2 : 1]>(m), red, turn);
        m0 = m[0] * inv;
        m1 = LAYER ? m[1] * inv : 0.f;
      }
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = (k * L + lane) * V;
        float o[V];
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = st.y * (D[k][i] - fmaf(zh[k][i], m0, m1));
        if (live) store8(static_cast<TZ*>(a.dz) + row * F, c, F, o);
      }
    }
  }
  // partial column sums of the workgroup: the R row lanes of a column through LDS, in order
  float* part = a.part + (int64_t)blockIdx.x * 4 * F;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if ((j < 2 && !a.z) || (j >= 2 && !a.dh) || (!LAYER && (j & 1))) continue;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const float* q = j == 0 ? q1[k] : j == 1 ? q2[LAYER ? k : 0] : j == 2 ? q3[k] : q4[LAYER ? k : 0];
      if (R > 1) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < V; ++i) cols[(rl * L + lane) * V + i] = q[i];
        __syncthreads();
        for (int e = threadIdx.x; e < L * V; e += T) {
          float sum = 0.f;
          for (int r = 0; r < R; ++r) sum += cols[r * L * V + e];
          if (k * L * V + e < F) part[(int64_t)j * F + k * L * V + e] = sum;
        }
      } else {
        store8(part + (int64_t)j * F, (k * L + lane) * V, F, q);
      }
    }
  }
}

struct ReduceArgs {
  NormArgs a;
  float *dscale, *dw, *db, *dw2, *db2;
};

// Adds the partial column sums (sixteen columns per workgroup, 64 row lanes that add theirs in order, then the lanes' sums in
// order) and forms the parameters' gradients.
template <bool Z, bool H, bool TWO>
__device__ __forceinline__ void add_parts(const float* t, int u0, int units, int64_t step, int F, float (&q)[4]) {
#pragma unroll 4
  for (int u = u0; u < units; u += 64) {       // (no branch inside: the loads of four turns fly together)
    const float* x = t + u * step;
    if (Z) q[0] += x[0];
    if (Z && TWO) q[1] += x[F];
    if (H) q[2] += x[2 * F];
    if (H && TWO) q[3] += x[3 * F];
  }
}
__global__ __launch_bounds__(1024) void norm_params_kernel(ReduceArgs p) {
  __shared__ float s[4][64][17];
  const NormArgs& a = p.a;
  const int F = a.d.F, cl = threadIdx.x & 15, rl = threadIdx.x >> 4, c = blockIdx.x * 16 + cl;
  const bool two = a.d.norm == AGCN_NORM_LAYER;
  float q[4] = {0.f, 0.f, 0.f, 0.f};
  if (c < F) {
    const int64_t step = (int64_t)4 * F;
    const float* t = a.part + c;
    if (a.z && a.dh && two) add_parts<true, true, true>(t, rl, a.units, step, F, q);
    else if (a.z && a.dh) add_parts<true, true, false>(t, rl, a.units, step, F, q);
    else if (a.z && two) add_parts<true, false, true>(t, rl, a.units, step, F, q);
    else if (a.z) add_parts<true, false, false>(t, rl, a.units, step, F, q);
    else if (a.dh && two) add_parts<false, true, true>(t, rl, a.units, step, F, q);
    else if (a.dh) add_parts<false, true, false>(t, rl, a.units, step, F, q);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) s[j][rl][cl] = q[j];
  __syncthreads();
  // one wave per sum: four lanes of a column add sixteen rows each
  if (threadIdx.x >= 256) return;
  const int j = threadIdx.x >> 6, part = (threadIdx.x >> 4) & 3;
  float v = 0.f;
#pragma unroll
  for (int r = 0; r < 16; ++r) v += s[j][part * 16 + r][cl];
  v += __shfl_xor(v, 16);
  v += __shfl_xor(v, 32);
  __syncthreads();
  if (part == 0) s[j][0][cl] = v;
  __syncthreads();
  if (threadIdx.x >= 16 || c >= F) return;
#pragma unroll
  for (int k = 0; k < 4; ++k) q[k] = s[k][0][cl];
  const float sc = a.scale ? a.scale[c] : 1.f, w = a.w ? a.w[c] : 1.f, b = a.b ? a.b[c] : 0.f;
  if (p.dscale) p.dscale[c] = fmaf(w, q[0], b * q[1]);
  if (p.dw) p.dw[c] = sc * q[0];
  if (p.db) p.db[c] = sc * q[1];
  if (p.dw2) p.dw2[c] = q[2];
  if (p.db2) p.db2[c] = q[3];
}

// A gate per graph: dg[graph] = a'(g) s (w sum D zh + b sum D), one thread per graph and column; and the graph's sums for the
// parameters (those over z times a(g)), left in the place of its first strip.
__global__ __launch_bounds__(64) void norm_graph_gate_kernel(NormArgs a) {
  const int F = a.d.F, g = blockIdx.x, c = blockIdx.y * 64 + threadIdx.x;
  if (c >= F) return;
  const int n = (int)(((int64_t)a.row_off[g + 1] - a.row_off[g] + (1 << a.graph_log2) - 1) >> a.graph_log2);
  const bool two = a.d.norm == AGCN_NORM_LAYER;
  float q[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int sp = 0; sp < n; ++sp) {
    const float* t = a.part + (int64_t)strip_place(a, g, sp) * 4 * F + c;
    q[0] += t[0];
    if (two) q[1] += t[F];
    if (a.dh) {
      q[2] += t[2 * (int64_t)F];
      if (two) q[3] += t[3 * (int64_t)F];
    }
  }
  const bool bf = a.d.z_dtype == AGCN_DTYPE_BF16;
  const int64_t at = (int64_t)g * a.d.ldg + c;
  const float gv = bf ? __uint_as_float((uint32_t)reinterpret_cast<const uint16_t*>(a.gate)[at] << 16) : static_cast<const float*>(a.gate)[at];
  float one[1] = {gv}, act[1], slope[1];
  gates<1>(a.d.gate_activation, one, act, slope);
  const float ga = act[0], da = slope[0];
  const float sc = a.scale ? a.scale[c] : 1.f, w = a.w ? a.w[c] : 1.f, b = a.b ? a.b[c] : 0.f;
  const float o = da * sc * fmaf(w, q[0], b * q[1]);
  if (bf) reinterpret_cast<uint16_t*>(a.dgate)[(int64_t)g * F + c] = (uint16_t)pk_bf(o, 0.f);
  else static_cast<float*>(a.dgate)[(int64_t)g * F + c] = o;
  float* sums = a.part + (int64_t)g * 4 * F + c;
  sums[0] = ga * q[0];
  if (two) sums[F] = ga * q[1];
  if (a.dh) {
    sums[2 * (int64_t)F] = q[2];
    if (two) sums[3 * (int64_t)F] = q[3];
  }
}

// ---- host side ---------------------------------------------------------------------------------------------------

// lanes per row and vectors per lane for a width: the fewest lanes that hold the row in one vector each (two beyond 8192)
struct Shape { int L, NV; };
Shape shape_for(int F) {
  const int vecs = (F + V - 1) / V;
  for (int L = 16; L <= 1024; L *= 2)
    if (vecs <= L) return {L, 1};
  return {1024, 2};
}

template <typename TX, typename TZ, int L, int NV>
void launch_one(bool back, const NormArgs& a, int grid, hipStream_t s) {
  const dim3 g(grid), t(threads_of<L>());
  const bool layer = a.d.norm == AGCN_NORM_LAYER;
  if (!back) {
    if (layer) hipLaunchKernelGGL((norm_forward_kernel<TX, TZ, L, NV, true>), g, t, 0, s, a);
    else hipLaunchKernelGGL((norm_forward_kernel<TX, TZ, L, NV, false>), g, t, 0, s, a);
  } else if (a.gate) {
    if (layer) hipLaunchKernelGGL((norm_backward_kernel<TX, TZ, L, NV, true, true>), g, t, 0, s, a);
    else hipLaunchKernelGGL((norm_backward_kernel<TX, TZ, L, NV, false, true>), g, t, 0, s, a);
  } else {
    if (layer) hipLaunchKernelGGL((norm_backward_kernel<TX, TZ, L, NV, true, false>), g, t, 0, s, a);
    else hipLaunchKernelGGL((norm_backward_kernel<TX, TZ, L, NV, false, false>), g, t, 0, s, a);
  }
}
template <typename TX, typename TZ>
void launch_shape(bool back, const NormArgs& a, Shape sh, int grid, hipStream_t s) {
  if (sh.NV == 2) launch_one<TX, TZ, 1024, 2>(back, a, grid, s);
  else if (sh.L == 16) launch_one<TX, TZ, 16, 1>(back, a, grid, s);
  else if (sh.L == 32) launch_one<TX, TZ, 32, 1>(back, a, grid, s);
  else if (sh.L == 64) launch_one<TX, TZ, 64, 1>(back, a, grid, s);
  else if (sh.L == 128) launch_one<TX, TZ, 128, 1>(back, a, grid, s);
  else if (sh.L == 256) launch_one<TX, TZ, 256, 1>(back, a, grid, s);
  else if (sh.L == 512) launch_one<TX, TZ, 512, 1>(back, a, grid, s);
  else launch_one<TX, TZ, 1024, 1>(back, a, grid, s);
}
void launch(bool back, const NormArgs& a, Shape sh, int grid, hipStream_t s) {
  if (a.d.x_dtype == AGCN_DTYPE_F32 && a.d.z_dtype == AGCN_DTYPE_F32) launch_shape<float, float>(back, a, sh, grid, s);
  else if (a.d.x_dtype == AGCN_DTYPE_F32) launch_shape<float, __hip_bfloat16>(back, a, sh, grid, s);
  else launch_shape<__hip_bfloat16, __hip_bfloat16>(back, a, sh, grid, s);
}

int rows_at_once(Shape sh) { return sh.L < 256 ? 256 / sh.L : 1; }
int threads_for(Shape sh) { return sh.L < 256 ? 256 : sh.L; }
// places for the partial sums of all graphs (a gate per graph)
int64_t graph_units(const NormArgs& a) { return (a.d.rows >> a.graph_log2) + a.B; }
// workgroups that walk the rows: as many as the rows ask for, up to what the chip holds (2048 threads per CU forward, 1024 backward)
int row_grid(const AgcnNormDesc& d, Shape sh, bool back) {
  const int64_t want = (d.rows + rows_at_once(sh) - 1) / rows_at_once(sh), cap = (int64_t)256 * (back ? 1024 : 2048) / threads_for(sh);
  return (int)std::max<int64_t>(1, std::min(want, cap));
}

int check_norm(const AgcnNormDesc* d, const void* plan_host, const void* plan_dev, NormArgs* a, const char* who) {
  std::memset(a, 0, sizeof(*a));
  if (!d) return fail(AGCN_EINVAL, "%s: null descriptor", who);
  a->d = *d;
  if (d->rows < 0 || d->rows > 0x7fffffff || d->F < 1 || d->F > 16384)
    return fail(AGCN_EINVAL, "%s: rows must be in 0..2^31-1 and F in 1..16384 (%lld, %d)", who, (long long)d->rows, d->F);
  if (d->norm != AGCN_NORM_RMS && d->norm != AGCN_NORM_LAYER) return fail(AGCN_EINVAL, "%s: unknown norm %d", who, d->norm);
  if (!(d->eps > 0.f)) return fail(AGCN_EINVAL, "%s: eps must be positive", who);
  if (d->gate < AGCN_GATE_NONE || d->gate > AGCN_GATE_GRAPH) return fail(AGCN_EINVAL, "%s: unknown gate %d", who, d->gate);
  if (d->gate_activation != AGCN_ACT_LINEAR && d->gate_activation != AGCN_ACT_TANH && d->gate_activation != AGCN_ACT_SIGMOID)
    return fail(AGCN_EINVAL, "%s: the gate's activation is linear, tanh or sigmoid", who);
  const bool xf = d->x_dtype == AGCN_DTYPE_F32, zf = d->z_dtype == AGCN_DTYPE_F32;
  if ((!xf && d->x_dtype != AGCN_DTYPE_BF16) || (!zf && d->z_dtype != AGCN_DTYPE_BF16) || (!xf && zf))
    return fail(AGCN_EINVAL, "%s: types are f32 / f32, bf16 / bf16, or an f32 residual with a bf16 block", who);
  if (plan_host) {
    PlanView host, dev;
    int rc = plan_view(plan_host, plan_host, &host);
    if (rc != AGCN_OK) return rc;
    if (!plan_dev) return fail(AGCN_EINVAL, "%s: null device plan", who);
    plan_view(plan_host, plan_dev, &dev);
    if (host.info.rows != d->rows) return fail(AGCN_EINVAL, "%s: %lld rows, but the plan has %d", who, (long long)d->rows, host.info.rows);
    a->n = dev.n; a->row_off = dev.row_off; a->row_graph = dev.row_graph;
    a->B = host.info.B;
    a->pads = host.info.rows != host.info.N1;
    if (d->gate == AGCN_GATE_GRAPH) {
      // rows of a graph per workgroup: few enough for a thousand workgroups, up to 64 (each leaves four sums per column)
      const Shape sh = shape_for(d->F);
      for (int r = rows_at_once(sh); r > 1; r >>= 1) ++a->graph_log2;
      while (a->graph_log2 < 6 && (d->rows >> a->graph_log2) > 1024) ++a->graph_log2;
      if (graph_units(*a) > 0xffffffffll / threads_for(sh))
        return fail(AGCN_EINVAL, "%s: %d graphs are more than one launch holds", who, host.info.B);
    }
  } else if (d->gate == AGCN_GATE_GRAPH) {
    return fail(AGCN_EINVAL, "%s: a gate per graph needs a plan", who);
  }
  return AGCN_OK;
}

int check_inputs(NormArgs* a, const AgcnNormInputs* in, const char* who) {
  const AgcnNormDesc& d = a->d;
  if (!in || !in->x) return fail(AGCN_EINVAL, "%s: null tensor", who);
  if (!in->z && (in->gate || in->scale || in->post_weight || in->post_bias))
    return fail(AGCN_EINVAL, "%s: gate, scale and post norm need a block output z", who);
  if (!in->z && !in->pre_weight) return fail(AGCN_EINVAL, "%s: neither a block output z nor a pre norm: nothing to compute", who);
  if ((in->post_bias && !in->post_weight) || (in->pre_bias && !in->pre_weight)) return fail(AGCN_EINVAL, "%s: a bias without its weight", who);
  if (d.norm == AGCN_NORM_RMS && (in->post_bias || in->pre_bias)) return fail(AGCN_EINVAL, "%s: the rms norm has no bias", who);
  if ((d.gate != AGCN_GATE_NONE) != (in->gate != nullptr)) return fail(AGCN_EINVAL, "%s: gate tensor and gate kind do not agree", who);
  if (d.ldx < d.F || (in->z && d.ldz < d.F) || (in->gate && d.ldg < d.F)) return fail(AGCN_EINVAL, "%s: a leading dimension is smaller than F", who);
  a->z = in->z; a->x = in->x; a->gate = in->gate; a->scale = in->scale;
  a->w = in->post_weight; a->b = in->post_bias; a->w2 = in->pre_weight; a->b2 = in->pre_bias;
  return AGCN_OK;
}

int back_units(const NormArgs& a) {
  return a.d.gate == AGCN_GATE_GRAPH ? (int)graph_units(a) : row_grid(a.d, shape_for(a.d.F), true);
}
}  // namespace
}  // namespace agcn

using namespace agcn;

extern "C" int agcn_norm_gate_residual_forward(const AgcnNormDesc* desc, const void* plan_host, const void* plan_dev,
                                               const AgcnNormInputs* in, void* y, void* h, float* stats, void* hip_stream) {
  const char* who = "agcn_norm_gate_residual_forward";
  NormArgs a;
  int rc = check_norm(desc, plan_host, plan_dev, &a, who);
  if (rc != AGCN_OK) return rc;
  if ((rc = check_inputs(&a, in, who)) != AGCN_OK) return rc;
  if ((a.z != nullptr) != (y != nullptr) || (a.w2 != nullptr) != (h != nullptr))
    return fail(AGCN_EINVAL, "%s: y goes with z, h with the pre norm", who);
  if (a.d.rows == 0) return AGCN_OK;
  a.y = y; a.h = h; a.stats = stats;
  hipStream_t s = static_cast<hipStream_t>(hip_stream);
  const Shape sh = shape_for(a.d.F);
  launch(false, a, sh, row_grid(a.d, sh, false), s);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(AGCN_EDEVICE, "%s: %s", who, hipGetErrorString(e));
  return AGCN_OK;
}

extern "C" size_t agcn_norm_gate_residual_backward_workspace_bytes(const AgcnNormDesc* desc, const void* plan_host) {
  NormArgs a;
  if (check_norm(desc, plan_host, plan_host, &a, "agcn_norm_gate_residual_backward_workspace_bytes") != AGCN_OK) return 0;
  return align256((size_t)back_units(a) * 4 * a.d.F * sizeof(float));
}

extern "C" int agcn_norm_gate_residual_backward(const AgcnNormDesc* desc, const void* plan_host, const void* plan_dev,
                                                const AgcnNormInputs* in, const float* stats, const void* dy, const void* dh,
                                                const AgcnNormGrads* grads, void* workspace,
                                                size_t workspace_bytes, void* hip_stream) {
  const char* who = "agcn_norm_gate_residual_backward";
  NormArgs a;
  int rc = check_norm(desc, plan_host, plan_dev, &a, who);
  if (rc != AGCN_OK) return rc;
  if ((rc = check_inputs(&a, in, who)) != AGCN_OK) return rc;
  if (!grads || !grads->dx || !stats || (a.z && !grads->dz)) return fail(AGCN_EINVAL, "%s: null tensor", who);
  if ((grads->dgate != nullptr) != (a.gate != nullptr) || (grads->dscale && !a.scale) || (grads->dpost_weight && !a.w) ||
      (grads->dpost_bias && !a.b) || (grads->dpre_weight && !a.w2) || (grads->dpre_bias && !a.b2) || (dy && !a.z) || (dh && !a.w2))
    return fail(AGCN_EINVAL, "%s: gradients do not agree with the inputs", who);
  a.units = back_units(a);
  const size_t need = (size_t)a.units * 4 * a.d.F * sizeof(float);
  if (!workspace || workspace_bytes < need) return fail(AGCN_ENOSPACE, "%s: workspace too small (%zu < %zu)", who, workspace_bytes, need);
  a.stats = const_cast<float*>(stats); a.dy = dy; a.dh = dh;
  a.dz = grads->dz; a.dx = grads->dx; a.dgate = grads->dgate; a.part = static_cast<float*>(workspace);
  hipStream_t s = static_cast<hipStream_t>(hip_stream);
  // (no rows: the one workgroup of the grid leaves zero sums, and the parameters' gradients come out zero)
  launch(true, a, shape_for(a.d.F), a.units, s);
  ReduceArgs p;
  std::memset(&p, 0, sizeof(p));
  p.a = a;
  p.dscale = grads->dscale; p.dw = grads->dpost_weight; p.db = grads->dpost_bias;
  p.dw2 = grads->dpre_weight; p.db2 = grads->dpre_bias;
  if (a.d.gate == AGCN_GATE_GRAPH) {
    hipLaunchKernelGGL(norm_graph_gate_kernel, dim3(a.B, (a.d.F + 63) / 64), dim3(64), 0, s, a);
    p.a.units = a.B;
  }
  if (p.dscale || p.dw || p.db || p.dw2 || p.db2)
    hipLaunchKernelGGL(norm_params_kernel, dim3((a.d.F + 15) / 16), dim3(1024), 0, s, p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(AGCN_EDEVICE, "%s: %s", who, hipGetErrorString(e));
  return AGCN_OK;
}
