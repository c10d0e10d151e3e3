// Entry points of the varlen attention with a learned bias by relative
// position: argument checks, the workspace, the last sum of the table's
// gradient.  The passes are the unmasked kernels' own (esa_attn_dense.hip and
// esa_attn_wide.hip for bf16, esa_attn.hip for fp32); esa_rel_bias.h has the
// bias.
#include <algorithm>

#include "esa_rel_bias.h"
#include "esa_profile.h"
#include "../../include/esa_hip.h"

namespace {

// dtable[b][h] = the sum of part[group][h][b] over the call's groups.  A block
// takes 32 columns of part; its 32 rows of threads sum every 32nd group each
// and are then added in order.
constexpr int kReduceCols = 32, kReduceRows = 32;
__global__ __launch_bounds__(kReduceCols* kReduceRows) void rel_reduce_kernel(const float* __restrict__ part,
                                                                              const int* __restrict__ count, int heads,
                                                                              int buckets, float* __restrict__ dtable) {
  __shared__ float s[kReduceRows][kReduceCols + 1];
  const int x = threadIdx.x % kReduceCols, y = threadIdx.x / kReduceCols;
  const int cols = heads * buckets, c = blockIdx.x * kReduceCols + x, n = *count;
  float sum = 0.f;
  for (int i0 = y; i0 < n; i0 += 8 * kReduceRows) {   // eight loads in flight
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int i = i0 + kReduceRows * j;
      v[j] = i < n && c < cols ? part[(size_t)i * cols + c] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) sum += v[j];
  }
  s[y][x] = sum;
  __syncthreads();
  if (y || c >= cols) return;
#pragma unroll
  for (int i = 1; i < kReduceRows; ++i) sum += s[i][x];
  dtable[(size_t)(c % buckets) * heads + c / buckets] = sum;
}

size_t up256(size_t x) { return (x + 255) & ~size_t(255); }
int tiles32(int x) { return (x + kTile - 1) / kTile; }
// At most ceil(T / tok) + (non-empty segments) groups, one more where they begin at even tokens.
size_t groups_most(int total, int batch, int tok = kGroupTok) {
  return (size_t)(total + tok - 1) / tok + (size_t)std::min(batch, total) + 1;
}

// Tokens of a group of the fp32 kernels.  A block walks its segment's partners alone, so with few blocks the walk of the
// longest segment is the time, and groups of 64, half the work for a block, take less of it; with many blocks a group of
// 128 feeds twice the products from each staged row.  A forward, and a step with its gradients, by blocks of 128 (8 heads;
// us with groups of 128 -> 64): head dim 16, 184 blocks 31, 105 -> 22, 72; 616: 49, 176 -> 41, 149; 1,872: 87, 328 -> 84,
// 316; 2,992 (32 proteins): 455, 1725 -> 458, 1765.  Head dim 64: 184: 58, 234 -> 40, 154; 376: 77, 274 -> 59, 230; 568
// (8 proteins): 264, 1072 -> 271, 1094; 1,872: 224, 1083 -> 244, 1066.
int group_tokens(int batch, int total_q, int total_k, int heads, int head_dim, int dtype) {
  if (dtype != ESA_F32) return kGroupTok;
  const size_t few = head_dim == 64 ? 512 : 2048;
  return groups_most(std::max(total_q, total_k), batch) * heads <= few ? kFewTok : kGroupTok;
}

// The bf16 forward of few queries (at most 32 a segment on average) over many keys (512 and more): with a block per
// segment and head at most kSplitMaxSegments blocks walk all of a segment's keys, one of their waves at work.  Cut so
// that about 2,048 blocks have `keys` each, 16 protein graphs (20,364 keys, 16 heads of 32), three queries each, take
// 14 us and 7 to join them instead of 31.
int split_keys(int batch, int total_q, int total_k, int heads, int dtype, bool backward) {
  if (backward || dtype != ESA_BF16 || total_q == 0 || total_q > (long long)kSplitRows * batch || batch > kSplitMaxSegments ||
      (long long)batch * heads >= 2048 || total_k < 512LL * batch)
    return 0;
  const long long want = (long long)total_k * heads / 2048;
  return (int)std::max(128LL, (want + 127) / 128 * 128);
}
// A segment's groups: of 32 queries, or of `keys` keys.
size_t split_most(int batch, int total_q, int total_k, int keys) {
  return (size_t)(total_q + kSplitRows - 1) / kSplitRows + (size_t)(total_k + keys - 1) / keys + 2 * (size_t)batch;
}

struct Layout { size_t counts, plan_q, plan_k, shift_q, shift_k, first_q, segment_q, line, top, ranges, knorm, rows, part, where, acc, ml, total; };
Layout layout(int batch, int total_q, int total_k, int heads, int head_dim, int buckets, int reach, int dtype, bool backward) {
  Layout w{};
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t at = off;
    off += up256(bytes);
    return at;
  };
  const int stride = 2 * (reach + kRelPad) + 1;
  const int split = split_keys(batch, total_q, total_k, heads, dtype, backward);
  const int tok = group_tokens(batch, total_q, total_k, heads, head_dim, dtype);
  const size_t gk = groups_most(total_k, batch, tok);
  const size_t gq = split ? split_most(batch, total_q, total_k, split) : groups_most(total_q, batch, tok);
  w.counts = take(8);
  w.plan_q = take(gq * sizeof(int4));
  w.shift_q = take(gq * sizeof(int));
  w.line = take((size_t)heads * stride * sizeof(float));
  w.top = take(heads * sizeof(float));
  w.ranges = take(buckets * sizeof(int2));
  if (backward) {
    w.plan_k = take(gk * sizeof(int4));
    w.shift_k = take(gk * sizeof(int));
    w.first_q = take((size_t)batch * sizeof(int));
    w.segment_q = take(gq * sizeof(int));
    w.rows = take((size_t)heads * tiles32(total_q) * kTile * sizeof(float2));
    w.part = take(gq * heads * buckets * sizeof(float));
  } else if (dtype == ESA_BF16) {
    if (!split) w.knorm = take((size_t)heads * tiles32(total_k) * sizeof(float));
    if (split) {
      const size_t rows = gq * kWaves * heads * kSplitRows;
      w.where = take((size_t)total_q * sizeof(int4));
      w.acc = take(rows * head_dim * sizeof(float));
      w.ml = take(rows * sizeof(float2));
    }
  }
  w.total = off;
  return w;
}

int check(int batch, int total_q, int total_k, int heads, int head_dim, int dtype, int buckets, const int* starts,
          int side) {
  if (head_dim != 16 && head_dim != 24 && head_dim != 32 && head_dim != 64) return ESA_ERR_HEAD_DIM;
  if (dtype != ESA_BF16 && dtype != ESA_F32) return ESA_ERR_DTYPE;
  // token offsets and distances (a query offset of up to 2^30 among them) stay within 32 bits
  if (batch < 1 || heads < 1 || total_q < 0 || total_k < 0 || total_q >= 1 << 28 || total_k >= 1 << 28) return ESA_ERR_SHAPE;
  if ((groups_most(std::max(total_q, total_k), batch) + 1) * (size_t)heads >= (size_t)1 << 31) return ESA_ERR_SHAPE;
  if (!starts) return ESA_ERR_NULL;
  if (buckets < 1 || buckets > kRelMaxBuckets || side < 1 || side > kRelMaxBuckets / 2 ||
      (side != buckets && 2 * side != buckets))
    return ESA_ERR_SHAPE;
  if (starts[0] != 0 || starts[side - 1] > kRelMaxReach) return ESA_ERR_SHAPE;
  for (int i = 1; i < side; ++i)
    if (starts[i] < starts[i - 1]) return ESA_ERR_SHAPE;
  return ESA_OK;
}

bool off_boundary(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

// From 1 on: distance 0 is in neither constant end of the line.
int reach_of(const int* starts, int side) { return std::max(1, starts[side - 1]); }

void fill(const Layout& w, char* ws, const void* table, int table_dtype, int buckets, const int* starts, int side,
          const int* q_start, const DenseAttnCall& c, int dtype, bool backward, RelPass& r, RelPrep& p) {
  auto at = [&](size_t off) { return ws + off; };
  RelBias& b = r.bias;
  b.reach = reach_of(starts, side);
  b.stride = 2 * (b.reach + kRelPad) + 1;
  b.buckets = buckets;
  b.far_lo = side - 1;
  b.far_hi = buckets == side ? 0 : buckets - 1;
  p.line = reinterpret_cast<float*>(at(w.line)); p.top = reinterpret_cast<float*>(at(w.top));
  p.ranges = reinterpret_cast<int2*>(at(w.ranges));
  b.line = p.line; b.top = p.top; b.ranges = p.ranges;
  b.part = backward ? reinterpret_cast<float*>(at(w.part)) : nullptr;
  r.plan_q = reinterpret_cast<int4*>(at(w.plan_q));
  r.shift_q = reinterpret_cast<int*>(at(w.shift_q));
  r.count_q = reinterpret_cast<int*>(at(w.counts));
  r.count_k = r.count_q + 1;
  r.tq_pad = tiles32(c.total_q) * kTile;
  if (backward) {
    r.plan_k = reinterpret_cast<int4*>(at(w.plan_k));
    r.shift_k = reinterpret_cast<int*>(at(w.shift_k));
    r.first_q = reinterpret_cast<int*>(at(w.first_q));
    r.bias.segment = r.segment_q = reinterpret_cast<int*>(at(w.segment_q));
    r.bias.first = r.first_q;
    r.bias.cu = c.cu_q;
    r.rows = reinterpret_cast<float2*>(at(w.rows));
  } else if (dtype == ESA_BF16) {
    if ((r.split.keys = split_keys(c.nseg, c.total_q, c.total_k, c.heads, dtype, false))) {
      r.split.most = (int)split_most(c.nseg, c.total_q, c.total_k, r.split.keys);
      r.split.where = reinterpret_cast<int4*>(at(w.where));
      r.split.acc = reinterpret_cast<float*>(at(w.acc));
      r.split.ml = reinterpret_cast<float2*>(at(w.ml));
    } else {
      r.knorm = reinterpret_cast<float*>(at(w.knorm));
      r.tk_tiles = tiles32(c.total_k);
    }
  }
  p.cu_q = c.cu_q; p.cu_k = c.cu_k; p.q_start = q_start; p.nseg = c.nseg;
  p.total_q = c.total_q; p.total_k = c.total_k; p.heads = c.heads;
  p.row16 = c.heads * c.head_dim * (dtype == ESA_F32 ? 4 : 2) / 16;
  p.table = table; p.table_dtype = table_dtype;
  std::copy(starts, starts + side, p.starts);
  p.side = side; p.two_sided = side != buckets;
  p.zero_q = static_cast<uint4*>(backward ? c.dq : c.out);
  p.zero_k = static_cast<uint4*>(c.dk); p.zero_v = static_cast<uint4*>(c.dv);
  p.lse = backward ? nullptr : c.lse;
  p.backward = backward;
  p.gtok_q = p.gtok_k = r.group_tok = r.bias.tok = group_tokens(c.nseg, c.total_q, c.total_k, c.heads, c.head_dim, dtype);
  p.key_pairs = backward && c.dropout && dtype == ESA_BF16;   // the bf16 dK/dV pass shares its hashes by key pairs
}

}  // namespace

extern "C" {

int esa_rel_attn_workspace_size(int batch, int total_q, int total_k, int heads, int head_dim, int dtype, int num_buckets,
                                const int* bucket_starts, int num_starts, int backward, size_t* bytes) {
  if (!bytes) return ESA_ERR_NULL;
  const int rc = check(batch, total_q, total_k, heads, head_dim, dtype, num_buckets, bucket_starts, num_starts);
  if (rc) return rc;
  *bytes = layout(batch, total_q, total_k, heads, head_dim, num_buckets, reach_of(bucket_starts, num_starts), dtype,
                  backward != 0)
               .total;
  return ESA_OK;
}

int esa_rel_attn_fwd(const void* q, const void* k, const void* v, const void* table, int table_dtype, int num_buckets,
                     const int* bucket_starts, int num_starts, const int* q_start, const int* cu_seqlens_q,
                     const int* cu_seqlens_k, int batch, int total_q, int total_k, int heads, int head_dim, int dtype,
                     float softmax_scale, float dropout_p, unsigned long long dropout_seed, void* out, void* out_low,
                     float* softmax_lse, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check(batch, total_q, total_k, heads, head_dim, dtype, num_buckets, bucket_starts, num_starts);
  if (rc) return rc;
  if (table_dtype != ESA_BF16 && table_dtype != ESA_F32) return ESA_ERR_DTYPE;
  if (!(dropout_p >= 0.f && dropout_p < 1.f)) return ESA_ERR_DROPOUT;
  if (!(softmax_scale > 0.f && softmax_scale <= 3.0e38f)) return ESA_ERR_SHAPE;
  if (total_q == 0) return ESA_OK;
  if (!table || !cu_seqlens_q || !cu_seqlens_k || !workspace || !q || !out || !softmax_lse || (total_k > 0 && (!k || !v)))
    return ESA_ERR_NULL;
  if (off_boundary(q) || off_boundary(k) || off_boundary(v) || off_boundary(out) || off_boundary(out_low) ||
      off_boundary(workspace))
    return ESA_ERR_ALIGN;
  const Layout w = layout(batch, total_q, total_k, heads, head_dim, num_buckets, reach_of(bucket_starts, num_starts), dtype, false);
  if (workspace_bytes < w.total) return ESA_ERR_WORKSPACE;
  DenseAttnCall c{};
  c.q = q; c.k = k; c.v = v; c.cu_q = cu_seqlens_q; c.cu_k = cu_seqlens_k; c.nseg = batch;
  c.total_q = total_q; c.total_k = total_k; c.heads = heads; c.head_dim = head_dim; c.scale = softmax_scale;
  c.out = out; c.out_low = out_low; c.lse = softmax_lse;
  c.drop = make_dropout(dropout_p, dropout_seed, heads); c.dropout = dropout_p > 0.f;
  RelPass r{};
  RelPrep p{};
  fill(w, static_cast<char*>(workspace), table, table_dtype, num_buckets, bucket_starts, num_starts, q_start, c, dtype, false, r,
       p);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  return dtype == ESA_BF16 ? dense_rel_fwd(c, r, p, st) : f32_rel_fwd(c, r, p, st);
}

int esa_rel_attn_bwd(const void* dout, const void* q, const void* k, const void* v, const void* out, const void* out_low,
                     const float* softmax_lse, const void* table, int table_dtype, int num_buckets,
                     const int* bucket_starts, int num_starts, const int* q_start, const int* cu_seqlens_q,
                     const int* cu_seqlens_k, int batch, int total_q, int total_k, int heads, int head_dim, int dtype,
                     float softmax_scale, float dropout_p, unsigned long long dropout_seed, void* dq, void* dk, void* dv,
                     float* dtable, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check(batch, total_q, total_k, heads, head_dim, dtype, num_buckets, bucket_starts, num_starts);
  if (rc) return rc;
  if (table_dtype != ESA_BF16 && table_dtype != ESA_F32) return ESA_ERR_DTYPE;
  if (!(dropout_p >= 0.f && dropout_p < 1.f)) return ESA_ERR_DROPOUT;
  if (!(softmax_scale > 0.f && softmax_scale <= 3.0e38f)) return ESA_ERR_SHAPE;
  if (!table || !dtable || !cu_seqlens_q || !cu_seqlens_k || !workspace ||
      (total_q > 0 && (!dout || !q || !out || !softmax_lse || !dq)) || (total_k > 0 && (!k || !v || !dk || !dv)))
    return ESA_ERR_NULL;
  if (off_boundary(dout) || off_boundary(q) || off_boundary(k) || off_boundary(v) || off_boundary(out) ||
      off_boundary(out_low) || off_boundary(dq) || off_boundary(dk) || off_boundary(dv) || off_boundary(workspace))
    return ESA_ERR_ALIGN;
  const Layout w = layout(batch, total_q, total_k, heads, head_dim, num_buckets, reach_of(bucket_starts, num_starts), dtype, true);
  if (workspace_bytes < w.total) return ESA_ERR_WORKSPACE;
  DenseAttnCall c{};
  c.q = q; c.k = k; c.v = v; c.cu_q = cu_seqlens_q; c.cu_k = cu_seqlens_k; c.nseg = batch;
  c.total_q = total_q; c.total_k = total_k; c.heads = heads; c.head_dim = head_dim; c.scale = softmax_scale;
  c.out_in = out; c.out_low_in = out_low; c.dout = dout; c.lse_in = softmax_lse; c.dq = dq; c.dk = dk; c.dv = dv;
  c.drop = make_dropout(dropout_p, dropout_seed, heads); c.dropout = dropout_p > 0.f;
  RelPass r{};
  RelPrep p{};
  fill(w, static_cast<char*>(workspace), table, table_dtype, num_buckets, bucket_starts, num_starts, q_start, c, dtype, true, r, p);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  rc = dtype == ESA_BF16 ? dense_rel_bwd(c, r, p, st) : f32_rel_bwd(c, r, p, st);
  if (rc) return rc;
  ESA_TIMED(esa_profile::kColumnSum, st,
            hipLaunchKernelGGL(rel_reduce_kernel, dim3((unsigned)((heads * num_buckets + kReduceCols - 1) / kReduceCols)),
                               dim3(kReduceCols * kReduceRows), 0, st, r.bias.part, r.count_q, heads, num_buckets, dtable));
  ESA_LAUNCH_CHECK();
  return ESA_OK;
}

}  // extern "C"
