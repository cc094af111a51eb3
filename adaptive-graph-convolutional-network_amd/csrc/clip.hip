// Global norm of many gradient tensors, and clipping by it (no counterpart in the reference's step, which clips per
// Laplacian only; the semantics are those of its framework's clip-by-global-norm):
//     n = sqrt(sum_t sum_i x_ti^2),   out_ti = x_ti * c / max(n, c);   n, in fp32, not finite -> every output is NaN.
// Two passes over the data, bound by memory: 3 transfers per element (read, read, write), of which the second read comes from
// the caches as far as they reach.  The tensors are cut into chunks; a workgroup sums one chunk in 64 bits (a square of any fp32
// value is finite there: neither a large nor a tiny gradient changes the answer's accuracy) and leaves one partial sum.  The
// second pass walks the chunks BACKWARDS, so that it begins with what the first pass left in the 256 MB memory-side cache.
// No atomics: the partial sums are added in a fixed order.
// Measured: 571 M bf16 gradients in 96 tensors (1143 MB) 667 us, on a profile's average sums 216 us (5.3 TB/s) and scaling 425 us (5.4
// TB/s); a large copy on this card reaches 4.9.  331 tensors of both types, 99 MB: 60 us on the GPU, 226 us with the host's table of
// tensors; 31 tensors 35 us.
#include <hip/hip_bf16.h>
#include <hip/hip_runtime.h>

#include <algorithm>
#include <vector>

#include "agcn_device.h"
#include "sgc_kernels.h"

namespace agcn {
namespace {
constexpr int kMaxT = 120;        // tensors per launch: the table travels in the kernel arguments (under 4 KB)
constexpr int kDirect = 1024;     // up to so many partial sums every workgroup of the second pass adds them itself

struct ClipTable {
  const void* in[kMaxT];
  void* out[kMaxT];
  int64_t numel[kMaxT];
  int32_t chunk0[kMaxT + 1];      // first chunk of the tensor, counted over this launch
  uint8_t bf16[kMaxT];
};
struct ClipArgs {
  ClipTable t;
  int32_t n, chunk_log2;          // tensors; log2 of a chunk's BYTES
  int32_t base, total;            // first chunk of this launch over all launches; all chunks
  float clip;
  double* part;                   // [total] partial sums; [total]: their sum
  float* norm;
};
static_assert(sizeof(ClipArgs) <= 4064, "the tensor table has to fit the kernel argument segment");

// 16 bytes at the alignment of an element: one global_load_dwordx4 (the target runs in unaligned access mode)
typedef uint32_t u32x4a __attribute__((ext_vector_type(4), aligned(2)));
__device__ __forceinline__ float bf_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
__device__ __forceinline__ uint32_t pack_bf(float a, float b) {
  typedef __bf16 b2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, (b2){(__bf16)a, (__bf16)b});
}

__device__ __forceinline__ int find_tensor(const ClipArgs& a, int chunk) {
  int lo = 0, hi = a.n - 1;                                // last tensor whose first chunk is <= chunk
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.t.chunk0[mid] <= chunk) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// sum over the workgroup (256 threads) of a double, the same value and order in every thread
__device__ __forceinline__ double block_sum_d(double v, double* red) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  const int w = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) red[w] = v;
  __syncthreads();
  double s = 0.0;
  for (int i = 0; i < (int)(blockDim.x >> 6); ++i) s += red[i];
  return s;
}

__device__ __forceinline__ void add_sq(const u32x4a& v, bool bf, double& s0, double& s1) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (bf) {
      const double x = (double)bf_lo(v[i]), y = (double)bf_hi(v[i]);
      s0 = fma(x, x, s0); s1 = fma(y, y, s1);
    } else {
      const double x = (double)__uint_as_float(v[i]);
      if (i & 1) s1 = fma(x, x, s1); else s0 = fma(x, x, s0);
    }
  }
}

__global__ __launch_bounds__(256) void clip_sumsq_kernel(ClipArgs a) {
  __shared__ double red[4];
  const int chunk = blockIdx.x, t = find_tensor(a, chunk), tid = threadIdx.x;
  const bool bf = a.t.bf16[t] != 0;
  const int64_t bytes = a.t.numel[t] << (bf ? 1 : 2);
  const int64_t b0 = (int64_t)(chunk - a.t.chunk0[t]) << a.chunk_log2;
  const int64_t left = bytes - b0;
  const int len = (int)(left < (1 << a.chunk_log2) ? left : (1 << a.chunk_log2));
  const char* p = static_cast<const char*>(a.t.in[t]) + b0;
  double s0 = 0.0, s1 = 0.0;
  const int full = len >> 4;                               // 16-byte pieces
  int i = tid;
  for (; i + 768 < full; i += 1024) {                      // four loads in flight
    u32x4a v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = *reinterpret_cast<const u32x4a*>(p + ((int64_t)(i + 256 * k) << 4));
#pragma unroll
    for (int k = 0; k < 4; ++k) add_sq(v[k], bf, s0, s1);
  }
  for (; i < full; i += 256) add_sq(*reinterpret_cast<const u32x4a*>(p + ((int64_t)i << 4)), bf, s0, s1);
  const int rest0 = full << 4, esz = bf ? 2 : 4;
  if (rest0 + tid * esz < len) {                           // the tensor's last elements (fewer than eight)
    double x;
    if (bf) x = (double)__uint_as_float((uint32_t)reinterpret_cast<const uint16_t*>(p + rest0)[tid] << 16);
    else x = (double)reinterpret_cast<const float*>(p + rest0)[tid];
    s0 = fma(x, x, s0);
  }
  const double s = block_sum_d(s0 + s1, red);
  if (tid == 0) a.part[a.base + chunk] = s;
}

__device__ __forceinline__ double sum_parts(const double* part, int n, double* red) {
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += blockDim.x) s += part[i];
  return block_sum_d(s, red);
}

// more partial sums than every workgroup of the second pass should add for itself, or no second pass at all
__global__ __launch_bounds__(1024) void clip_total_kernel(double* part, int total, float* norm) {
  __shared__ double red[16];
  const double s = sum_parts(part, total, red);
  if (threadIdx.x == 0) {
    part[total] = s;
    norm[0] = (float)sqrt(s);
  }
}

__device__ __forceinline__ float times(float x, double f) { return (float)((double)x * f); }
__device__ __forceinline__ u32x4a scaled(u32x4a v, bool bf, float k, bool tiny, double f) {
  if (tiny) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = bf ? pack_bf(times(bf_lo(v[i]), f), times(bf_hi(v[i]), f)) : __float_as_uint(times(__uint_as_float(v[i]), f));
    return v;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = bf ? pack_bf(bf_lo(v[i]) * k, bf_hi(v[i]) * k) : __float_as_uint(__uint_as_float(v[i]) * k);
  return v;
}

__global__ __launch_bounds__(256) void clip_scale_kernel(ClipArgs a) {
  __shared__ double red[4];
  const int chunk = (int)(gridDim.x - 1 - blockIdx.x), t = find_tensor(a, chunk), tid = threadIdx.x;
  double s;
  if (a.total <= kDirect) {
    s = sum_parts(a.part, a.total, red);
    if (a.base + chunk == 0 && tid == 0) a.norm[0] = (float)sqrt(s);
  } else {
    s = a.part[a.total];
  }
  const double n = sqrt(s), c = (double)a.clip;
  // Finite or not is asked of the norm as it is handed back, in fp32: a caller that skips a step by it and the results agree.  (A
  // NaN or infinite sum fails both comparisons.)
  const bool finite = (float)n < INFINITY;
  const double f = finite ? (n <= c ? 1.0 : c / n) : NAN;
  const float k = (float)f;
  // a factor below fp32's normal numbers has lost digits: those products are taken in 64 bits
  const bool tiny = f < (double)__FLT_MIN__;
  const void* in = a.t.in[t];
  void* out = a.t.out[t];
  if (k == 1.f && in == out) return;
  const bool bf = a.t.bf16[t] != 0;
  const int64_t bytes = a.t.numel[t] << (bf ? 1 : 2);
  const int64_t b0 = (int64_t)(chunk - a.t.chunk0[t]) << a.chunk_log2;
  const int64_t left = bytes - b0;
  const int len = (int)(left < (1 << a.chunk_log2) ? left : (1 << a.chunk_log2));
  const char* p = static_cast<const char*>(in) + b0;
  char* q = static_cast<char*>(out) + b0;
  const int full = len >> 4;
  int i = tid;
  for (; i + 768 < full; i += 1024) {
    u32x4a v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const u32x4a*>(p + ((int64_t)(i + 256 * j) << 4));
#pragma unroll
    for (int j = 0; j < 4; ++j) *reinterpret_cast<u32x4a*>(q + ((int64_t)(i + 256 * j) << 4)) = scaled(v[j], bf, k, tiny, f);
  }
  for (; i < full; i += 256)
    *reinterpret_cast<u32x4a*>(q + ((int64_t)i << 4)) = scaled(*reinterpret_cast<const u32x4a*>(p + ((int64_t)i << 4)), bf, k, tiny, f);
  const int rest0 = full << 4, esz = bf ? 2 : 4;
  if (rest0 + tid * esz < len) {
    if (bf) {
      const uint16_t x = reinterpret_cast<const uint16_t*>(p + rest0)[tid];
      const float v = __uint_as_float((uint32_t)x << 16);
      reinterpret_cast<uint16_t*>(q + rest0)[tid] = (uint16_t)pack_bf(tiny ? times(v, f) : v * k, 0.f);
    } else {
      const float v = reinterpret_cast<const float*>(p + rest0)[tid];
      reinterpret_cast<float*>(q + rest0)[tid] = tiny ? times(v, f) : v * k;
    }
  }
}

// log2 of a chunk's bytes: 4 KB (one workgroup reads it with one load per thread) while that leaves no more than four chunks
// per CU, up to 64 KB (16 loads per thread)
int chunk_log2_for(int64_t bytes) {
  int l = 12;
  while (l < 16 && (bytes >> l) > 1024) ++l;
  return l;
}
inline int64_t tensor_bytes(int64_t numel, int32_t dtype) { return numel << (dtype == AGCN_DTYPE_BF16 ? 1 : 2); }

// chunks of all tensors; negative: bad table
int64_t count_chunks(int32_t n, const int64_t* numel, const int32_t* dtype, int* log2_out) {
  int64_t bytes = 0;
  for (int32_t i = 0; i < n; ++i) {
    if (numel[i] < 0 || numel[i] > ((int64_t)1 << 46) || (dtype[i] != AGCN_DTYPE_F32 && dtype[i] != AGCN_DTYPE_BF16)) return -1;
    bytes += tensor_bytes(numel[i], dtype[i]);
  }
  const int l = chunk_log2_for(bytes);
  int64_t chunks = 0;
  for (int32_t i = 0; i < n; ++i) chunks += (tensor_bytes(numel[i], dtype[i]) + ((int64_t)1 << l) - 1) >> l;
  *log2_out = l;
  return chunks;
}

struct Span { uintptr_t a, b; int32_t i; };
}  // namespace
}  // namespace agcn

using namespace agcn;

extern "C" size_t agcn_clip_workspace_bytes(int32_t n_tensors, const int64_t* numel, const int32_t* dtype) {
  int l = 0;
  const int64_t chunks = n_tensors >= 1 && numel && dtype ? count_chunks(n_tensors, numel, dtype, &l) : -1;
  if (chunks < 0 || chunks > 0x7ffffff0) {
    fail(AGCN_EINVAL, "agcn_clip_workspace_bytes: bad tensor table (at least one tensor, sizes >= 0, f32 or bf16)");
    return 0;
  }
  return align256((size_t)(chunks + 1) * sizeof(double));
}

extern "C" int agcn_clip_by_global_norm(int32_t n_tensors, const void* const* in, void* const* out, const int64_t* numel,
                                        const int32_t* dtype, float clip_norm, float* norm, void* workspace,
                                        size_t workspace_bytes, void* hip_stream) {
  const char* who = "agcn_clip_by_global_norm";
  if (n_tensors < 1 || !in || !numel || !dtype || !norm) return fail(AGCN_EINVAL, "%s: no tensors or a null table", who);
  if (out && !(clip_norm > 0.f)) return fail(AGCN_EINVAL, "%s: clip_norm must be positive", who);
  int l = 0;
  const int64_t chunks = count_chunks(n_tensors, numel, dtype, &l);
  if (chunks < 0 || chunks > 0x7ffffff0) return fail(AGCN_EINVAL, "%s: bad tensor table (sizes >= 0, f32 or bf16)", who);
  for (int32_t i = 0; i < n_tensors; ++i) {
    const uintptr_t mask = dtype[i] == AGCN_DTYPE_BF16 ? 1 : 3;
    if (numel[i] && (!in[i] || (out && !out[i]))) return fail(AGCN_EINVAL, "%s: tensor %d is null", who, i);
    if (((uintptr_t)in[i] & mask) || (out && ((uintptr_t)out[i] & mask))) return fail(AGCN_EINVAL, "%s: tensor %d is not aligned to its type", who, i);
  }
  if (!workspace || ((uintptr_t)workspace & 7) || workspace_bytes < (size_t)(chunks + 1) * sizeof(double))
    return fail(AGCN_ENOSPACE, "%s: workspace too small (%zu < %zu)", who, workspace_bytes, (size_t)(chunks + 1) * sizeof(double));
  if (out) {
    // an output may be its own input (in place) and nothing else: two tensors over the same memory would be scaled twice, and a
    // tensor read after another's output was written over it would give a mixture
    try {
      std::vector<Span> w;
      w.reserve(n_tensors);
      for (int32_t i = 0; i < n_tensors; ++i)
        if (numel[i]) w.push_back({(uintptr_t)out[i], (uintptr_t)out[i] + (uintptr_t)tensor_bytes(numel[i], dtype[i]), i});
      std::sort(w.begin(), w.end(), [](const Span& p, const Span& q) { return p.a < q.a; });
      for (size_t k = 1; k < w.size(); ++k)
        if (w[k].a < w[k - 1].b) return fail(AGCN_EINVAL, "%s: outputs %d and %d overlap", who, w[k - 1].i, w[k].i);
      for (int32_t i = 0; i < n_tensors; ++i) {
        if (!numel[i]) continue;
        const uintptr_t a = (uintptr_t)in[i], b = a + (uintptr_t)tensor_bytes(numel[i], dtype[i]);
        // first output that ends behind a
        auto it = std::upper_bound(w.begin(), w.end(), a, [](uintptr_t v, const Span& s) { return v < s.b; });
        for (; it != w.end() && it->a < b; ++it)
          if (it->i != i || in[i] != out[i]) return fail(AGCN_EINVAL, "%s: input %d overlaps output %d", who, i, it->i);
      }
    } catch (...) {
      return fail(AGCN_EINVAL, "%s: out of host memory", who);
    }
  }
  hipStream_t s = static_cast<hipStream_t>(hip_stream);
  double* part = static_cast<double*>(workspace);
  ClipArgs a;
  for (int pass = 0; pass < (out ? 2 : 1); ++pass) {
    // (the second pass takes the launches, too, from the last to the first)
    std::memset(&a, 0, sizeof(a));
    a.chunk_log2 = l; a.total = (int32_t)chunks; a.clip = clip_norm; a.part = part; a.norm = norm;
    int32_t i = pass ? n_tensors - 1 : 0, done = 0;
    const int32_t step = pass ? -1 : 1;
    while (i >= 0 && i < n_tensors) {
      int32_t take[kMaxT], k = 0;
      for (; i >= 0 && i < n_tensors && k < kMaxT; i += step)
        if (numel[i]) take[k++] = i;
      if (!k) break;
      if (pass) std::reverse(take, take + k);
      int32_t c = 0;
      for (int32_t j = 0; j < k; ++j) {
        const int32_t q = take[j];
        a.t.in[j] = in[q]; a.t.out[j] = out ? out[q] : nullptr; a.t.numel[j] = numel[q];
        a.t.bf16[j] = dtype[q] == AGCN_DTYPE_BF16; a.t.chunk0[j] = c;
        c += (int32_t)((tensor_bytes(numel[q], dtype[q]) + ((int64_t)1 << l) - 1) >> l);
      }
      a.t.chunk0[k] = c; a.n = k;
      done += c;
      a.base = pass ? (int32_t)chunks - done : done - c;
      if (pass) hipLaunchKernelGGL(clip_scale_kernel, dim3(c), dim3(256), 0, s, a);
      else hipLaunchKernelGGL(clip_sumsq_kernel, dim3(c), dim3(256), 0, s, a);
    }
    // (no chunks at all: the norm of empty tensors is 0)
    if (pass == 0 && (!out || chunks > kDirect || chunks == 0))
      hipLaunchKernelGGL(clip_total_kernel, dim3(1), dim3(1024), 0, s, part, (int)chunks, norm);
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(AGCN_EDEVICE, "%s: %s", who, hipGetErrorString(e));
  return AGCN_OK;
}
