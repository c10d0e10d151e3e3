// The norm over the values of many tensors together, and the tensors scaled
// by the factor that clips it.
//
//   n = sqrt(sum over all tensors of x^2)  (or the largest |x|),
//   x' = x min(1, max_norm / (n + 1e-6)).
//
// Memory bounds both passes on large models and launches on small ones.  The
// tensors' pointers and sizes travel in the kernel arguments of the norm's
// launches, kTable tensors a launch, so that no table is copied to the device
// or kept between calls; a block takes 8,192 values of one tensor and notes
// in the workspace where they lie, so that the clipping is one launch
// whatever the number of tensors (768 bf16 gradients of 37 million values
// into fp32: five launches of the norm, 6.5 us each, and one of 35 us).
// Loads are 16 bytes a lane at any element alignment (gradients in a flat
// buffer begin anywhere; global memory instructions take unaligned
// addresses).  Squares are summed in fp64, which costs nothing beside the
// loads and neither overflows nor loses the small gradients beside large
// ones; every sum has a fixed order.
#include <algorithm>

#include "esa_common.h"
#include "esa_profile.h"
#include "../../include/esa_hip.h"

namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 8192;    // values a block takes
constexpr int kTable = 160;     // tensors a launch: 3.9 KB of kernel arguments
// Up to so many sums the clipping's blocks join them by themselves, a launch less.  Norm and clipping of 4, 200, 480
// and 1,000 chunks took 5.1, 8.1, 10.6 and 17.6 us, with the join's launch 6.6, 9.4, 11.7 and 17.5 (in a graph).
constexpr int kOwnJoin = 512;
constexpr int kInF32 = 1, kOutF32 = 2;

struct Table {
  const void* in[kTable];
  void* out[kTable];
  unsigned count[kTable];       // values of the tensor, or of a part of it
  unsigned first[kTable];       // the tensors' first chunks, their kinds in the low two bits
  int n;
};

// Where the values of a chunk lie.
struct Chunk {
  const void* in;
  void* out;
  int n, kind;
};

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef __bf16 bf16x8u __attribute__((ext_vector_type(8), aligned(2)));

// Chunk b of the launch (block-uniform): of the last tensor that begins at or before it.
DEVI Chunk chunk_of(const Table& t, unsigned b) {
  int lo = 0, hi = t.n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.first[mid] >> 2 <= b) lo = mid; else hi = mid;
  }
  const unsigned at = (b - (t.first[lo] >> 2)) * kChunk;
  Chunk c;
  c.kind = t.first[lo] & 3;
  c.n = (int)min((unsigned)kChunk, t.count[lo] - at);
  c.in = static_cast<const char*>(t.in[lo]) + (size_t)at * (c.kind & kInF32 ? 4 : 2);
  c.out = t.out[lo] ? static_cast<char*>(t.out[lo]) + (size_t)at * (c.kind & kOutF32 ? 4 : 2) : nullptr;
  return c;
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
__global__ __launch_bounds__(kThreads) void grad_norm_kernel(const Table t, double* __restrict__ part,
                                                             Chunk* __restrict__ chunks) {
  __shared__ double s[kThreads / 64];
  const Chunk c = chunk_of(t, blockIdx.x);
  Norm<MAX> sum;
  auto use = [&](int, const Eight& x) {
#pragma unroll
    for (int e = 0; e < 8; ++e) sum.add(x.v[e]);
  };
  auto one = [&](int, float x) { sum.add(x); };
  if (c.kind & kInF32) chunk_values(static_cast<const float*>(c.in), c.n, use, one);
  else chunk_values(static_cast<const bf16*>(c.in), c.n, use, one);
  const double v = block_join(sum, s);
  if (threadIdx.x == 0) {
    part[blockIdx.x] = v;
    if (chunks) chunks[blockIdx.x] = c;
  }
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
DEVI void clip_chunk(const Chunk& c, float factor) {
  TO* o = static_cast<TO*>(c.out);
  chunk_values(
      static_cast<const TI*>(c.in), c.n,
      [&](int i, Eight x) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x.v[e] *= factor;
        store8(o + i, x);
      },
      [&](int i, float x) { o[i] = (TO)(x * factor); });
}

// JOINS: no join launch went before; every block joins the `parts` sums by itself, and the first notes the norm.
template <bool JOINS, bool MAX>
__global__ __launch_bounds__(kThreads) void grad_clip_kernel(const Chunk* __restrict__ chunks, float max_norm,
                                                             float* __restrict__ norm, const double* __restrict__ part, int parts) {
  __shared__ double s[kThreads / 64];
  __shared__ float joined;
  const Chunk c = chunks[blockIdx.x];
  float n;
  if (JOINS) {
    Norm<MAX> sum;
#pragma unroll 4
    for (int i = threadIdx.x; i < parts; i += kThreads) sum.join(part[i]);
    const double v = block_join(sum, s);
    if (threadIdx.x == 0) {
      joined = (float)(MAX ? v : sqrt(v));
      if (blockIdx.x == 0) *norm = joined;
    }
    __syncthreads();
    n = joined;
  } else {
    n = *norm;
  }
  const float f = max_norm / (n + 1e-6f), factor = f > 1.f ? 1.f : f;   // a NaN stays one
  if (c.kind & kInF32) clip_chunk<float, float>(c, factor);
  else if (c.kind & kOutF32) clip_chunk<bf16, float>(c, factor);
  else clip_chunk<bf16, bf16>(c, factor);
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

size_t up256(size_t x) { return (x + 255) & ~size_t(255); }
long long all_chunks(int n, const long long* counts) {
  long long chunks = 0;
  for (int i = 0; i < n; ++i) chunks += chunks_of(counts[i]);
  return chunks;
}

// The norm's launches, and where `out` is given the chunks' places.
template <bool MAX>
int norm_launches(int n, const void* const* in, void* const* out, const long long* counts, const int* in_dtypes,
                  const int* out_dtypes, float* norm, double* part, Chunk* chunks, hipStream_t st) {
  constexpr unsigned kPart = 1u << 30;      // values of an entry: longer tensors take several
  constexpr unsigned kMostChunks = 1u << 28;
  Table t;
  t.n = 0;
  unsigned here = 0;
  long long done = 0;
  auto flush = [&]() {
    if (!t.n) return (int)ESA_OK;
    ESA_TIMED(esa_profile::kGradNorm, st,
              hipLaunchKernelGGL((grad_norm_kernel<MAX>), dim3(here), dim3(kThreads), 0, st, t, part + done,
                                 out ? chunks + done : nullptr));
    ESA_LAUNCH_CHECK();
    done += here;
    t.n = 0;
    here = 0;
    return (int)ESA_OK;
  };
  for (int i = 0; i < n; ++i) {
    const int size_in = in_dtypes[i] == ESA_F32 ? 4 : 2, size_out = out && out_dtypes[i] == ESA_F32 ? 4 : 2;
    for (long long at = 0; at < counts[i]; at += kPart) {
      const unsigned count = (unsigned)std::min<long long>(kPart, counts[i] - at);
      if (t.n == kTable || here > kMostChunks - kPart / kChunk)
        if (const int rc = flush()) return rc;
      t.in[t.n] = static_cast<const char*>(in[i]) + at * size_in;
      t.out[t.n] = out ? static_cast<char*>(out[i]) + at * size_out : nullptr;
      t.count[t.n] = count;
      t.first[t.n] = here << 2 | (in_dtypes[i] == ESA_F32 ? kInF32 : 0) | (out && out_dtypes[i] == ESA_F32 ? kOutF32 : 0);
      here += (unsigned)chunks_of(count);
      ++t.n;
    }
  }
  if (const int rc = flush()) return rc;
  if (out && done > 0 && done <= kOwnJoin) return ESA_OK;   // the clipping joins
  ESA_TIMED(esa_profile::kGradNorm, st,
            hipLaunchKernelGGL((grad_norm_join_kernel<MAX>), dim3(1), dim3(1024), 0, st, part, done, norm));
  ESA_LAUNCH_CHECK();
  return ESA_OK;
}

}  // namespace

extern "C" {

int esa_grad_workspace_size(int n, const long long* counts, int clip, size_t* bytes) {
  if (!bytes || (n > 0 && !counts)) return ESA_ERR_NULL;
  if (n < 0) return ESA_ERR_SHAPE;
  for (int i = 0; i < n; ++i)
    if (counts[i] < 0 || counts[i] > 1LL << 40) return ESA_ERR_SHAPE;
  const size_t chunks = (size_t)all_chunks(n, counts);
  if (clip && chunks >= (size_t)1 << 31) return ESA_ERR_SHAPE;   // one launch's blocks
  *bytes = up256(chunks * sizeof(double)) + (clip ? chunks * sizeof(Chunk) : 0);
  return ESA_OK;
}

int esa_grad_norm(int n, const void* const* in, const long long* counts, const int* dtypes, int infinity, float* norm,
                  void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check(n, in, counts, dtypes);
  if (rc) return rc;
  if (!norm) return ESA_ERR_NULL;
  size_t need = 0;
  if ((rc = esa_grad_workspace_size(n, counts, 0, &need))) return rc;
  if (need && !workspace) return ESA_ERR_NULL;
  if (reinterpret_cast<uintptr_t>(workspace) % 8 || reinterpret_cast<uintptr_t>(norm) % 4) return ESA_ERR_ALIGN;
  if (workspace_bytes < need) return ESA_ERR_WORKSPACE;
  auto go = infinity ? norm_launches<true> : norm_launches<false>;
  return go(n, in, nullptr, counts, dtypes, nullptr, norm, static_cast<double*>(workspace), nullptr,
            reinterpret_cast<hipStream_t>(stream));
}

int esa_grad_clip(int n, const void* const* in, void* const* out, const long long* counts, const int* in_dtypes,
                  const int* out_dtypes, int infinity, float max_norm, float* norm, void* workspace, size_t workspace_bytes,
                  void* stream) {
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
  size_t need = 0;
  if ((rc = esa_grad_workspace_size(n, counts, 1, &need))) return rc;
  if (need && !workspace) return ESA_ERR_NULL;
  if (reinterpret_cast<uintptr_t>(workspace) % 8 || reinterpret_cast<uintptr_t>(norm) % 4) return ESA_ERR_ALIGN;
  if (workspace_bytes < need) return ESA_ERR_WORKSPACE;
  const unsigned total = (unsigned)all_chunks(n, counts);
  Chunk* chunks = reinterpret_cast<Chunk*>(static_cast<char*>(workspace) + up256(total * sizeof(double)));
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  auto go = infinity ? norm_launches<true> : norm_launches<false>;
  if ((rc = go(n, in, out, counts, in_dtypes, out_dtypes, norm, static_cast<double*>(workspace), chunks, st))) return rc;
  if (!total) return ESA_OK;
  const double* part = static_cast<const double*>(workspace);
  auto kernel = total > kOwnJoin ? grad_clip_kernel<false, false> : infinity ? grad_clip_kernel<true, true> : grad_clip_kernel<true, false>;
  ESA_TIMED(esa_profile::kGradClip, st,
            hipLaunchKernelGGL(kernel, dim3(total), dim3(kThreads), 0, st, chunks, max_norm, norm, part, (int)total));
  ESA_LAUNCH_CHECK();
  return ESA_OK;
}

}  // extern "C"
