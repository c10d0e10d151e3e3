// RMS norm of every query and key head row with the rotation of positions in
// the same pass, forward and backward.
//
//   r = 1 / sqrt(mean(x^2) + eps),  y = x r w;  the first `rotary` dims of y in
//   pairs (i, i + rotary / 2), or (2i, 2i + 1) interleaved, turned by the angle
//   position * frequency[i]:  (a, b) -> (a cos - b sin, a sin + b cos).
// Backward: g turned back, then  dx = r (w g - x r mean(x r w g)),
//   dw = sum over rows of g x r.
//
// Memory bounds it: a row is read and written once (backward: x and g read, dx
// written).  A lane holds 8 dims of a row (HD / 8 lanes a row), so that the
// row's loads are 16 bytes a lane and consecutive; four rows are in flight per
// lane.  A block takes runs of tokens with all their heads, queries and keys
// both: the token's angles are worked out once, in 64 bits (position *
// frequency in turns; 32 would lose the angle of far positions) and its cosines
// and sines wait in LDS.  A pair's other half of the half-split order is
// fetched from the lane that holds it, four dims at a time.
//
// 129,850 tokens, 32 query and 32 key heads of 16 in bf16: forward 95 to 98 us
// for 400 MB as counted at memory, backward 163 to 168 for 533 MB; 8 and 8 heads of 64
// in fp32 (43,670 tokens): 67 to 69 us for 269 MB, 106 for 359; a copy reaches
// 4.7 TB/s.  A call of one graph is one launch of 7 us, most of it the latency of
// the 64-bit angles.
#include <algorithm>

#include "esa_common.h"
#include "esa_profile.h"
#include "../../include/esa_hip.h"

namespace {

constexpr int kThreads = 256;
constexpr int kRows = 4;            // rows in flight per lane
constexpr int kMaxTokens = 16;      // tokens of a run
constexpr int kMaxBlocks = 2048;    // of the backward: rows of weight partials

enum Rotation { kNone, kHalves, kPairs };

struct NormArgs {
  const void* x[2]; long token_stride[2], head_stride[2];   // queries, keys; strides in elements
  const void* g[2];                                         // backward: gradients of y, [T][H][HD]
  void* y[2];                                               // forward y, backward dx, [T][H][HD]
  const float* w[2];                                        // null: ones
  int heads[2];
  const void* positions; int wide_positions;                // int32, or int64
  const double* frequencies; int half;                      // half: pairs of a row
  float eps;
  int total, run;                                           // tokens, tokens of a run
  uint32_t magic;                                           // ceil(2^32 / (heads[0] + heads[1]))
  float* part;                                              // backward: [blocks][2][HD]
};

struct Row8 { float v[8]; };

DEVI Row8 load_row8(const float* p) {
  Row8 r;
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  r.v[0] = a.x; r.v[1] = a.y; r.v[2] = a.z; r.v[3] = a.w;
  r.v[4] = b.x; r.v[5] = b.y; r.v[6] = b.z; r.v[7] = b.w;
  return r;
}
DEVI Row8 load_row8(const bf16* p) {
  Row8 r;
  const bf16x8 a = *reinterpret_cast<const bf16x8*>(p);
#pragma unroll
  for (int e = 0; e < 8; ++e) r.v[e] = (float)a[e];
  return r;
}
DEVI void store_row8(float* p, const Row8& r) {
  reinterpret_cast<float4*>(p)[0] = make_float4(r.v[0], r.v[1], r.v[2], r.v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(r.v[4], r.v[5], r.v[6], r.v[7]);
}
DEVI void store_row8(bf16* p, const Row8& r) {   // the one rounding of a bf16 call
  bf16x8 a;
#pragma unroll
  for (int e = 0; e < 8; ++e) a[e] = (bf16)r.v[e];
  *reinterpret_cast<bf16x8*>(p) = a;
}

// The sum over a row's lanes, the same on each (three lanes: in their order).
template <int LANES>
DEVI float row_sum(float x, int lane) {
  if constexpr (LANES == 3) {
    const int first = lane - lane % 3;
    return __shfl(x, first) + __shfl(x, first + 1) + __shfl(x, first + 2);
  } else {
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1) x += __shfl_xor(x, o);
    return x;
  }
}

// The lane's 8 dims turned by the token's angles (BACK: by their negatives).
template <int ROT, bool BACK>
DEVI void turn(Row8& y, const float2* cs, int part, int lane, int half) {
  if constexpr (ROT == kPairs) {
    if (4 * part >= half) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 t = cs[4 * part + i];
      const float a = y.v[2 * i], b = y.v[2 * i + 1], s = BACK ? -t.y : t.y;
      y.v[2 * i] = a * t.x - b * s;
      y.v[2 * i + 1] = a * s + b * t.x;
    }
  } else if constexpr (ROT == kHalves) {
    // four dims a quarter-row step: quarter 2 part + u, its partner h4 further on (first half) or back (second)
    const int h4 = half / 4, odd = h4 & 1;
    float other[2][4];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int q = 2 * part + u, p = q < h4 ? q + h4 : q < 2 * h4 ? q - h4 : q;
      const int from = lane - part + (p >> 1);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        // a lane in the rotated part gives the quarter that its taker asks for
        const float same = y.v[4 * u + e], across = y.v[4 - 4 * u + e];
        other[u][e] = __shfl(odd ? across : same, from);
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int q = 2 * part + u;
      const bool in = q < 2 * h4;
      const float2* t = cs + (in ? 4 * (q < h4 ? q : q - h4) : 0);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 cos_sin = t[e];
        const float s = (q < h4) != BACK ? -cos_sin.y : cos_sin.y;
        const float x = y.v[4 * u + e] * cos_sin.x + other[u][e] * s;
        y.v[4 * u + e] = in ? x : y.v[4 * u + e];
      }
    }
  }
}

// The run's cosines and sines: cs[token][pair].
DEVI void angles(const NormArgs& a, int t0, int tokens, float2* cs, int tid) {
  for (int i = tid; i < tokens * a.half; i += kThreads) {
    const int t = i / a.half, j = i - t * a.half;
    const double pos = a.wide_positions ? (double)static_cast<const int64_t*>(a.positions)[t0 + t]
                                        : (double)static_cast<const int*>(a.positions)[t0 + t];
    double turns = pos * a.frequencies[j] * 0.15915494309189533577;   // 1 / (2 pi)
    turns -= rint(turns);
    float s, c;
    sincospif((float)(2.0 * turns), &s, &c);
    cs[i] = make_float2(c, s);
  }
}

// One kernel for both directions: a lane's rows of a run, four at a time.
template <typename T, int HD, int ROT, bool BACK>
__global__ __launch_bounds__(kThreads) void qk_norm_kernel(const NormArgs a) {
  constexpr int LANES = HD / 8, PER_WAVE = 64 / LANES, GROUPS = 4 * PER_WAVE;   // rows a block takes side by side
  __shared__ __align__(16) float2 cs[ROT == kNone ? 1 : kMaxTokens * 32];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int group = wave * PER_WAVE + lane / LANES, part = lane % LANES;
  const bool spare = lane >= PER_WAVE * LANES;   // head dim 24: lane 63
  const int per = a.heads[0] + a.heads[1];
  float w[2][8], dw[2][8];
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      w[n][e] = a.w[n] ? a.w[n][8 * part + e] : 1.f;
      dw[n][e] = 0.f;
    }
  for (int t0 = blockIdx.x * a.run; t0 < a.total; t0 += gridDim.x * a.run) {   // block-uniform
    const int tokens = min(a.run, a.total - t0), rows = spare ? 0 : tokens * per;
    if constexpr (ROT != kNone) {
      __syncthreads();   // the last run's rows are done
      angles(a, t0, tokens, cs, tid);
      __syncthreads();
    }
    for (int r0 = group; r0 < rows; r0 += kRows * GROUPS) {
      Row8 x[kRows], g[kRows];
      int tok[kRows], head[kRows], n[kRows];
#pragma unroll
      for (int u = 0; u < kRows; ++u) {
        const int r = r0 + u * GROUPS;
        tok[u] = per == 1 ? min(r, rows - 1) : (int)__umulhi((uint32_t)min(r, rows - 1), a.magic);
        head[u] = min(r, rows - 1) - tok[u] * per;
        n[u] = head[u] >= a.heads[0];
        head[u] -= n[u] ? a.heads[0] : 0;
        x[u] = load_row8(static_cast<const T*>(n[u] ? a.x[1] : a.x[0]) +
                         (long)(t0 + tok[u]) * (n[u] ? a.token_stride[1] : a.token_stride[0]) +
                         (long)head[u] * (n[u] ? a.head_stride[1] : a.head_stride[0]) + 8 * part);
        if constexpr (BACK)
          g[u] = load_row8(static_cast<const T*>(n[u] ? a.g[1] : a.g[0]) +
                           ((size_t)(t0 + tok[u]) * (n[u] ? a.heads[1] : a.heads[0]) + head[u]) * HD + 8 * part);
      }
#pragma unroll
      for (int u = 0; u < kRows; ++u) {
        const bool in = r0 + u * GROUPS < rows;
        float sq = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) sq = fmaf(x[u].v[e], x[u].v[e], sq);
        const float rs = 1.f / sqrtf(row_sum<LANES>(sq, lane) * (1.f / HD) + a.eps);
        Row8 out;
        const float2* c = ROT == kNone ? cs : cs + tok[u] * a.half;
        if constexpr (BACK) {
          turn<ROT, true>(g[u], c, part, lane, a.half);
          float m = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float unit = x[u].v[e] * rs, wg = (n[u] ? w[1][e] : w[0][e]) * g[u].v[e];
            m = fmaf(unit, wg, m);
            const float p = in ? g[u].v[e] * unit : 0.f;
            dw[0][e] += n[u] ? 0.f : p;
            dw[1][e] += n[u] ? p : 0.f;
            x[u].v[e] = unit;
            out.v[e] = wg;
          }
          m = row_sum<LANES>(m, lane) * (1.f / HD);
#pragma unroll
          for (int e = 0; e < 8; ++e) out.v[e] = rs * (out.v[e] - x[u].v[e] * m);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) out.v[e] = x[u].v[e] * rs * (n[u] ? w[1][e] : w[0][e]);
          turn<ROT, false>(out, c, part, lane, a.half);
        }
        if (in)
          store_row8(static_cast<T*>(n[u] ? a.y[1] : a.y[0]) +
                         ((size_t)(t0 + tok[u]) * (n[u] ? a.heads[1] : a.heads[0]) + head[u]) * HD + 8 * part,
                     out);
      }
    }
  }
  if constexpr (BACK) {   // the block's weight gradients, its groups in order
    if (!a.part) return;
    __shared__ float sum[2 * HD][GROUPS + 1];
    if (!spare)
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[n * HD + 8 * part + e][group] = dw[n][e];
    __syncthreads();
    if (tid < 2 * HD) {
      float s = 0.f;
      for (int i = 0; i < GROUPS; ++i) s += sum[tid][i];
      a.part[(size_t)blockIdx.x * 2 * HD + tid] = s;
    }
  }
}

// dw[n][d] = the sum of part[block][n][d]: 32 columns a block, its 32 rows of threads one after another.  A thread's
// loads go out eight at a time: one by one the launch took 22 us for 2,048 blocks.
__global__ __launch_bounds__(1024) void qk_norm_reduce_kernel(const float* __restrict__ part, int blocks, int hd,
                                                              float* __restrict__ dwq, float* __restrict__ dwk) {
  __shared__ float s[32][33];
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5, c = blockIdx.x * 32 + x, cols = 2 * hd;
  float sum = 0.f;
  for (int i0 = y; i0 < blocks; i0 += 8 * 32) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = i0 + 32 * j < blocks && c < cols ? part[(size_t)(i0 + 32 * j) * cols + c] : 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) sum += v[j];
  }
  s[y][x] = sum;
  __syncthreads();
  if (y || c >= cols) return;
#pragma unroll
  for (int i = 1; i < 32; ++i) sum += s[i][x];
  float* out = c < hd ? dwq : dwk;
  if (out) out[c < hd ? c : c - hd] = sum;
}

// Tokens of a run: all of a block's rows in flight at once or more, as long as the chip has its blocks.
int run_of(int total) { return std::max(1, std::min(kMaxTokens, total / 2048)); }
int blocks_of(int total, bool back) {
  const int runs = (total + run_of(total) - 1) / run_of(total);
  return back ? std::min(runs, kMaxBlocks) : runs;
}

template <typename T, int HD, bool BACK>
void launch_rot(int rot, dim3 grid, hipStream_t st, const NormArgs& a) {
  if (rot == kNone) hipLaunchKernelGGL((qk_norm_kernel<T, HD, kNone, BACK>), grid, dim3(kThreads), 0, st, a);
  else if (rot == kHalves) hipLaunchKernelGGL((qk_norm_kernel<T, HD, kHalves, BACK>), grid, dim3(kThreads), 0, st, a);
  else hipLaunchKernelGGL((qk_norm_kernel<T, HD, kPairs, BACK>), grid, dim3(kThreads), 0, st, a);
}
template <typename T, bool BACK>
void launch_hd(int hd, int rot, dim3 grid, hipStream_t st, const NormArgs& a) {
  if (hd == 16) launch_rot<T, 16, BACK>(rot, grid, st, a);
  else if (hd == 24) launch_rot<T, 24, BACK>(rot, grid, st, a);
  else if (hd == 32) launch_rot<T, 32, BACK>(rot, grid, st, a);
  else launch_rot<T, 64, BACK>(rot, grid, st, a);
}
template <bool BACK>
int launch(int dtype, int hd, int rot, hipStream_t st, const NormArgs& a) {
  const dim3 grid((unsigned)blocks_of(a.total, BACK));
  ESA_TIMED(BACK ? esa_profile::kQkNormBwd : esa_profile::kQkNormFwd, st,
            if (dtype == ESA_F32) launch_hd<float, BACK>(hd, rot, grid, st, a); else launch_hd<bf16, BACK>(hd, rot, grid, st, a));
  ESA_LAUNCH_CHECK();
  return ESA_OK;
}

bool off_boundary(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

int set_up(int total, int head_dim, int dtype, const long long* strides, int heads_q, int heads_k, const void* q, const void* k,
           const float* wq, const float* wk, const void* positions, int positions_bytes, const double* frequencies,
           int rotary_dim, float eps, NormArgs& a) {
  if (head_dim != 16 && head_dim != 24 && head_dim != 32 && head_dim != 64) return ESA_ERR_HEAD_DIM;
  if (dtype != ESA_F32 && dtype != ESA_BF16) return ESA_ERR_DTYPE;
  // a run's rows index in 16 bits for the division by `magic`
  if (total < 0 || total > INT32_MAX - kMaxTokens * kMaxBlocks || heads_q < 1 || heads_k < 0 ||
      heads_q > 2048 || heads_k > 2048 || !(eps >= 0.f))
    return ESA_ERR_SHAPE;
  if (rotary_dim < 0 || rotary_dim > head_dim || rotary_dim % 8) return ESA_ERR_SHAPE;
  if (rotary_dim && positions_bytes != 4 && positions_bytes != 8) return ESA_ERR_DTYPE;
  if (!strides) return ESA_ERR_NULL;
  if (total == 0) return ESA_OK;
  if (!q || (heads_k && !k) || (rotary_dim && (!positions || !frequencies))) return ESA_ERR_NULL;
  const int size = dtype == ESA_F32 ? 4 : 2;
  for (int i = 0; i < (heads_k ? 4 : 2); ++i)
    if (strides[i] * size % 16) return ESA_ERR_ALIGN;
  if (off_boundary(q) || off_boundary(k)) return ESA_ERR_ALIGN;
  a.x[0] = q; a.x[1] = k;
  for (int n = 0; n < 2; ++n) {
    a.token_stride[n] = n && !heads_k ? 0 : (long)strides[2 * n];
    a.head_stride[n] = n && !heads_k ? 0 : (long)strides[2 * n + 1];
  }
  a.w[0] = wq; a.w[1] = wk;
  a.heads[0] = heads_q; a.heads[1] = heads_k;
  a.positions = positions; a.wide_positions = positions_bytes == 8;
  a.frequencies = frequencies; a.half = rotary_dim / 2;
  a.eps = eps;
  a.total = total; a.run = run_of(total);
  const uint64_t per = (uint64_t)heads_q + heads_k;
  a.magic = (uint32_t)((((uint64_t)1 << 32) + per - 1) / per);   // a single row per token divides by nothing
  return ESA_OK;
}

}  // namespace

extern "C" {

int esa_qk_norm_fwd(const void* q, const void* k, const long long* strides, int total, int heads_q, int heads_k, int head_dim,
                    int dtype, const float* wq, const float* wk, const void* positions, int positions_bytes,
                    const double* frequencies, int rotary_dim, int interleaved, float eps, void* q_out, void* k_out,
                    void* stream) {
  NormArgs a{};
  const int rc = set_up(total, head_dim, dtype, strides, heads_q, heads_k, q, k, wq, wk, positions, positions_bytes,
                        frequencies, rotary_dim, eps, a);
  if (rc || total == 0) return rc;
  if (!q_out || (heads_k && !k_out)) return ESA_ERR_NULL;
  if (off_boundary(q_out) || off_boundary(k_out)) return ESA_ERR_ALIGN;
  a.y[0] = q_out; a.y[1] = k_out;
  return launch<false>(dtype, head_dim, rotary_dim == 0 ? kNone : interleaved ? kPairs : kHalves,
                       reinterpret_cast<hipStream_t>(stream), a);
}

int esa_qk_norm_bwd_workspace_size(int total, int head_dim, size_t* bytes) {
  if (!bytes) return ESA_ERR_NULL;
  if (head_dim != 16 && head_dim != 24 && head_dim != 32 && head_dim != 64) return ESA_ERR_HEAD_DIM;
  if (total < 0) return ESA_ERR_SHAPE;
  *bytes = (size_t)blocks_of(total, true) * 2 * head_dim * sizeof(float);
  return ESA_OK;
}

int esa_qk_norm_bwd(const void* gq, const void* gk, const void* q, const void* k, const long long* strides, int total,
                    int heads_q, int heads_k, int head_dim, int dtype, const float* wq, const float* wk,
                    const void* positions, int positions_bytes, const double* frequencies, int rotary_dim, int interleaved,
                    float eps, void* dq, void* dk, float* dwq, float* dwk, void* workspace, size_t workspace_bytes,
                    void* stream) {
  NormArgs a{};
  const int rc = set_up(total, head_dim, dtype, strides, heads_q, heads_k, q, k, wq, wk, positions, positions_bytes,
                        frequencies, rotary_dim, eps, a);
  if (rc) return rc;
  const bool weights = dwq || dwk;
  size_t need = 0;
  esa_qk_norm_bwd_workspace_size(total, head_dim, &need);
  if (total > 0) {
    if (!gq || !dq || (heads_k && (!gk || !dk)) || (weights && !workspace)) return ESA_ERR_NULL;
    if (off_boundary(gq) || off_boundary(gk) || off_boundary(dq) || off_boundary(dk) ||
        (weights && reinterpret_cast<uintptr_t>(workspace) % alignof(float)))
      return ESA_ERR_ALIGN;
    if (weights && workspace_bytes < need) return ESA_ERR_WORKSPACE;
  }
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (total > 0) {
    a.g[0] = gq; a.g[1] = gk;
    a.y[0] = dq; a.y[1] = dk;
    a.part = weights ? static_cast<float*>(workspace) : nullptr;
    const int bad = launch<true>(dtype, head_dim, rotary_dim == 0 ? kNone : interleaved ? kPairs : kHalves, st, a);
    if (bad) return bad;
  }
  if (weights) {
    ESA_TIMED(esa_profile::kColumnSum, st,
              hipLaunchKernelGGL(qk_norm_reduce_kernel, dim3((2 * head_dim + 31) / 32), dim3(1024), 0, st,
                                 static_cast<const float*>(workspace), total > 0 ? blocks_of(total, true) : 0, head_dim, dwq,
                                 dwk));
    ESA_LAUNCH_CHECK();
  }
  return ESA_OK;
}

}  // extern "C"
