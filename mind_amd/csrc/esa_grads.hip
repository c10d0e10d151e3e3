// The norm over the values of many tensors together, and the tensors scaled
// by the factor that clips it.
//
//   n = sqrt(sum over all tensors of x^2)  (or the largest |x|),
//   x' = x min(1, max_norm / (n + 1e-6)).
//
// Memory bounds both passes on large models and launches on small ones: the
// tensors' pointers and sizes travel in the kernel arguments, kTable tensors a
// launch, so that no table is copied to the device or kept between calls, and
// a block takes 8,192 values of one tensor.  Loads are 16 bytes a lane at any
// element alignment (gradients in a flat buffer begin anywhere; global memory
// instructions take unaligned addresses).  Squares are summed in fp64, which
// costs nothing beside the loads and neither overflows nor loses the small
// gradients beside large ones; every sum has a fixed order.
#include <algorithm>

#include "esa_common.h"
#include "esa_profile.h"
#include "../../include/esa_hip.h"

namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 8192;    // values a block takes
constexpr int kTable = 112;     // tensors a launch: 3.4 KB of kernel arguments

struct Table {
  const void* in[kTable];
  void* out[kTable];
  long long count[kTable];
  unsigned first[kTable + 1];   // the tensors' first chunks; the last entry is the launch's chunks
  unsigned char in_f32[kTable], out_f32[kTable];
  int n;
};

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef __bf16 bf16x8u __attribute__((ext_vector_type(8), aligned(2)));

// The tensor that holds chunk b: first[i] <= b < first[i + 1] (block-uniform; tensors without values have no chunk).
DEVI int tensor_of(const Table& t, unsigned b) {
  int lo = 0, hi = t.n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.first[mid] <= b) lo = mid; else hi = mid;
  }
  return lo;
}

struct Eight { float v[8]; };
DEVI Eight load8(const float* p) {
  const f32x4u a = reinterpret_cast<const f32x4u*>(p)[0], b = reinterpret_cast<const f32x4u*>(p)[1];
  return Eight{{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]}};
}
DEVI Eight load8(const bf16* p) {
  const bf16x8u a = *reinterpret_cast<const bf16x8u*>(p);
  Eight r;
#pragma unroll
  for (int e = 0; e < 8; ++e) r.v[e] = (float)a[e];
  return r;
}
DEVI void store8(float* p, const Eight& x) {
  f32x4u a, b;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    a[e] = x.v[e];
    b[e] = x.v[4 + e];
  }
  reinterpret_cast<f32x4u*>(p)[0] = a;
  reinterpret_cast<f32x4u*>(p)[1] = b;
}
DEVI void store8(bf16* p, const Eight& x) {   // the clipped value's one rounding
  bf16x8u a;
#pragma unroll
  for (int e = 0; e < 8; ++e) a[e] = (bf16)x.v[e];
  *reinterpret_cast<bf16x8u*>(p) = a;
}

// Calls use(i, values) for the thread's runs of 8 of the chunk's n values and one(i, value) for the rest.
template <typename T, class Use, class One>
DEVI void chunk_values(const T* p, int n, Use use, One one) {
  const int whole = n & ~7;
  if (n == kChunk) {   // four loads in flight
#pragma unroll
    for (int j = 0; j < kChunk / (8 * kThreads); ++j) {
      const int i = 8 * (threadIdx.x + j * kThreads);
      use(i, load8(p + i));
    }
    return;
  }
  for (int i = 8 * threadIdx.x; i < whole; i += 8 * kThreads) use(i, load8(p + i));
  if (whole + (int)threadIdx.x < n) one(whole + threadIdx.x, (float)p[whole + threadIdx.x]);
}

// A running sum of squares or largest magnitude, a NaN staying one.
template <bool MAX>
struct Norm {
  double v = 0.0;
  DEVI void add(float x) {
    if (MAX) join((double)fabsf(x));
    else v = fma((double)x, (double)x, v);
  }
  DEVI void join(double o) {
    if (MAX) v = v != v ? v : !(o <= v) ? o : v;
    else v += o;
  }
};

template <bool MAX>
DEVI double block_join(Norm<MAX> x, double* s) {   // lane 0 of wave 0 has the result
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) x.join(__shfl_down(x.v, o));
  const int waves = blockDim.x / 64, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (lane == 0) s[wave] = x.v;
  __syncthreads();
  if (threadIdx.x == 0)
    for (int w = 1; w < waves; ++w) x.join(s[w]);
  return x.v;
}

template <bool MAX>
__global__ __launch_bounds__(kThreads) void grad_norm_kernel(const Table t, double* __restrict__ part) {
  __shared__ double s[kThreads / 64];
  const int i = tensor_of(t, blockIdx.x);
  const long long at = (long long)(blockIdx.x - t.first[i]) * kChunk;
  const int n = (int)min((long long)kChunk, t.count[i] - at);
  Norm<MAX> sum;
  auto use = [&](int, const Eight& x) {
#pragma unroll
    for (int e = 0; e < 8; ++e) sum.add(x.v[e]);
  };
  auto one = [&](int, float x) { sum.add(x); };
  if (t.in_f32[i]) chunk_values(static_cast<const float*>(t.in[i]) + at, n, use, one);
  else chunk_values(static_cast<const bf16*>(t.in[i]) + at, n, use, one);
  const double v = block_join(sum, s);
  if (threadIdx.x == 0) part[blockIdx.x] = v;
}

template <bool MAX>
__global__ __launch_bounds__(1024) void grad_norm_join_kernel(const double* __restrict__ part, long long n, float* __restrict__ norm) {
  __shared__ double s[16];
  Norm<MAX> sum;
#pragma unroll 4
  for (long long i = threadIdx.x; i < n; i += 1024) sum.join(part[i]);
  const double v = block_join(sum, s);
  if (threadIdx.x == 0) *norm = (float)(MAX ? v : sqrt(v));
}

template <typename TI, typename TO>
DEVI void clip_chunk(const void* in, void* out, long long at, int n, float factor) {
  TO* o = static_cast<TO*>(out) + at;
  chunk_values(
      static_cast<const TI*>(in) + at, n,
      [&](int i, Eight x) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x.v[e] *= factor;
        store8(o + i, x);
      },
      [&](int i, float x) { o[i] = (TO)(x * factor); });
}

__global__ __launch_bounds__(kThreads) void grad_clip_kernel(const Table t, float max_norm, const float* __restrict__ norm) {
  const int i = tensor_of(t, blockIdx.x);
  const long long at = (long long)(blockIdx.x - t.first[i]) * kChunk;
  const int n = (int)min((long long)kChunk, t.count[i] - at);
  const float f = max_norm / (*norm + 1e-6f), factor = f > 1.f ? 1.f : f;   // a NaN stays one
  if (t.in_f32[i]) clip_chunk<float, float>(t.in[i], t.out[i], at, n, factor);
  else if (t.out_f32[i]) clip_chunk<bf16, float>(t.in[i], t.out[i], at, n, factor);
  else clip_chunk<bf16, bf16>(t.in[i], t.out[i], at, n, factor);
}

long long chunks_of(long long count) { return (count + kChunk - 1) / kChunk; }

int check(int n, const void* const* in, const long long* counts, const int* dtypes) {
  if (n < 0) return ESA_ERR_SHAPE;
  if (n && (!in || !counts || !dtypes)) return ESA_ERR_NULL;
  for (int i = 0; i < n; ++i) {
    if (counts[i] < 0 || counts[i] > 1LL << 40) return ESA_ERR_SHAPE;
    if (dtypes[i] != ESA_F32 && dtypes[i] != ESA_BF16) return ESA_ERR_DTYPE;
    if (!counts[i]) continue;
    if (!in[i]) return ESA_ERR_NULL;
    if (reinterpret_cast<uintptr_t>(in[i]) % (dtypes[i] == ESA_F32 ? 4 : 2)) return ESA_ERR_ALIGN;
  }
  return ESA_OK;
}

// Calls go(table, chunks) for runs of at most kTable tensors with values and 2^30 chunks.
template <class Go>
int tables(int n, const void* const* in, void* const* out, const long long* counts, const int* in_dtypes, const int* out_dtypes,
           Go go) {
  Table t;
  t.n = 0;
  unsigned chunks = 0;
  auto flush = [&]() {
    if (!t.n) return (int)ESA_OK;
    t.first[t.n] = chunks;
    const int rc = go(t, chunks);
    t.n = 0;
    chunks = 0;
    return rc;
  };
  for (int i = 0; i < n; ++i) {
    if (!counts[i]) continue;
    if (t.n == kTable || chunks + chunks_of(counts[i]) > 1LL << 30)
      if (const int rc = flush()) return rc;
    t.in[t.n] = in[i];
    t.out[t.n] = out ? out[i] : nullptr;
    t.count[t.n] = counts[i];
    t.first[t.n] = chunks;
    t.in_f32[t.n] = in_dtypes[i] == ESA_F32;
    t.out_f32[t.n] = out_dtypes && out_dtypes[i] == ESA_F32;
    chunks += (unsigned)chunks_of(counts[i]);
    ++t.n;
  }
  return flush();
}

}  // namespace

extern "C" {

int esa_grad_norm_workspace_size(int n, const long long* counts, size_t* bytes) {
  if (!bytes || (n > 0 && !counts)) return ESA_ERR_NULL;
  if (n < 0) return ESA_ERR_SHAPE;
  long long chunks = 0;
  for (int i = 0; i < n; ++i) {
    if (counts[i] < 0 || counts[i] > 1LL << 40) return ESA_ERR_SHAPE;
    chunks += chunks_of(counts[i]);
  }
  *bytes = (size_t)chunks * sizeof(double);
  return ESA_OK;
}

int esa_grad_norm(int n, const void* const* in, const long long* counts, const int* dtypes, int infinity, float* norm,
                  void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check(n, in, counts, dtypes);
  if (rc) return rc;
  if (!norm) return ESA_ERR_NULL;
  size_t need = 0;
  if ((rc = esa_grad_norm_workspace_size(n, counts, &need))) return rc;
  if (need && !workspace) return ESA_ERR_NULL;
  if (reinterpret_cast<uintptr_t>(workspace) % 8 || reinterpret_cast<uintptr_t>(norm) % 4) return ESA_ERR_ALIGN;
  if (workspace_bytes < need) return ESA_ERR_WORKSPACE;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  double* part = static_cast<double*>(workspace);
  long long done = 0;
  rc = tables(n, in, nullptr, counts, dtypes, nullptr, [&](const Table& t, unsigned chunks) {
    ESA_TIMED(esa_profile::kGradNorm, st,
              if (infinity) hipLaunchKernelGGL((grad_norm_kernel<true>), dim3(chunks), dim3(kThreads), 0, st, t, part + done);
              else hipLaunchKernelGGL((grad_norm_kernel<false>), dim3(chunks), dim3(kThreads), 0, st, t, part + done));
    done += chunks;
    ESA_LAUNCH_CHECK();
    return (int)ESA_OK;
  });
  if (rc) return rc;
  ESA_TIMED(esa_profile::kGradNorm, st,
            if (infinity) hipLaunchKernelGGL((grad_norm_join_kernel<true>), dim3(1), dim3(1024), 0, st, part, done, norm);
            else hipLaunchKernelGGL((grad_norm_join_kernel<false>), dim3(1), dim3(1024), 0, st, part, done, norm));
  ESA_LAUNCH_CHECK();
  return ESA_OK;
}

int esa_grad_clip(int n, const void* const* in, void* const* out, const long long* counts, const int* in_dtypes,
                  const int* out_dtypes, float max_norm, const float* norm, void* stream) {
  int rc = check(n, in, counts, in_dtypes);
  if (rc) return rc;
  if (n && (!out || !out_dtypes)) return ESA_ERR_NULL;
  for (int i = 0; i < n; ++i) {
    if (out_dtypes[i] != in_dtypes[i] && out_dtypes[i] != ESA_F32) return ESA_ERR_DTYPE;
    if (!counts[i]) continue;
    if (!out[i]) return ESA_ERR_NULL;
    if (reinterpret_cast<uintptr_t>(out[i]) % (out_dtypes[i] == ESA_F32 ? 4 : 2)) return ESA_ERR_ALIGN;
  }
  if (!norm) return ESA_ERR_NULL;
  if (!(max_norm >= 0.f)) return ESA_ERR_SHAPE;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  return tables(n, in, out, counts, in_dtypes, out_dtypes, [&](const Table& t, unsigned chunks) {
    ESA_TIMED(esa_profile::kGradClip, st,
              hipLaunchKernelGGL(grad_clip_kernel, dim3(chunks), dim3(kThreads), 0, st, t, max_norm, norm));
    ESA_LAUNCH_CHECK();
    return (int)ESA_OK;
  });
}

}  // extern "C"
