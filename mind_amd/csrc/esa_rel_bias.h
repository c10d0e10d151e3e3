// The learned bias by relative position inside the unmasked attention kernels
// (esa_rel_attn_fwd / _bwd): scores get table[bucket(d)][head], d = key
// position - query position in their segment.
//
// The preparation pass writes the table out by distance: per head a line of
// bias * log2(e) at entry d + reach + kRelPad.  From `reach` (the distance at
// which a side's last bucket begins) on the bias is constant, so only tiles
// that cross |d| < reach differ within themselves.  Scores take the line's
// entries (from LDS, one per score) as their matrix product's seed or in the
// exponent's FMA.  The bf16 forward and dQ pass give the other tiles their one
// value (it moves the forward's reference point: no operation per score); the
// others read it from the line's pads.
//
// The table's gradient sums dS over the pairs of a bucket, in a fixed order
// and without atomics.  In the dQ pass a wave's dS of a stage (64 keys by its
// 32 or 16 queries) lies in its lanes as rows (keys) of columns (queries).
// Swaps between lane halves and quarters turn it into rows of 64 lanes in
// which lane C holds distance  row - C + constant,  so a diagonal is summed by
// one shift of the running sum by a lane and one addition per row.  What runs
// out at lane 0 comes from a second chain that turns round instead (their
// difference).  The sums by distance go to the wave's line in LDS, where no
// other wave writes; a block folds its lines into buckets, and a last launch
// sums the blocks.  (By ds_add_f32, one per score, into a ring of distances per
// wave, about 160 cycles an instruction, the dQ pass took 6.2 ms instead of 2.0
// at 129,850 tokens, 32 heads of 16.)
//
// Vector instructions bound it: at those sizes forward, dQ and dK/dV take 0.94,
// 1.53 and 1.58 ms at best (0.81, 1.12 and 1.36 without a bias), their vector
// pipes busy 62, 78 and 70 % of the time and their matrix pipes 32, 24 and
// 27 %; one exponential a score is 31, 19 and 18 %.  A near stage of dQ spends 96
// instructions on the diagonals beside some 210 on its two tiles.
//
// bf16 calls round P and dS to bf16 where they are operands of the products over
// keys and queries, as the kernels without a bias do: gradients 2.4 to 2.5e-3 of
// their norm off, 1.7e-3 of it their own last rounding.  Sums of dS and the row
// statistics are of unrounded values.  (P V with P's residue in a second product
// made the output and the table's gradient exact to their last rounding and dq
// 2.46 instead of 2.50e-3, for 1.61 ms instead of 0.94.)
#pragma once
#include <hip/hip_runtime.h>

#include "esa_attn_dense.h"
#include "esa_attn_tiles.h"

constexpr int kRelPad = 96;          // a stage of 64 keys and 32 queries may reach 95 past |d| = reach
constexpr int kRelMaxReach = 768;    // the waves' lines of the widest dQ kernel still fit LDS
constexpr int kRelMaxBuckets = 256;
constexpr float kRelLargest = 1.0e4f;   // finite biases beyond it count as it: exp leaves nothing of such a difference

struct RelBias {
  const float* line;        // [heads][stride]
  const float* top;         // [heads] the largest |bias| log2(e) that is finite
  const int2* ranges;       // [buckets] entries [x, y) of the line
  int reach, stride;        // stride = 2 (reach + kRelPad) + 1
  int buckets, far_lo, far_hi;   // the buckets of d <= -reach and d >= reach
  float* part;              // dQ pass: [groups][heads][buckets], the groups in their tokens' order
  const int* segment;       // dQ pass: a listed group's segment,
  const int* first;         // that segment's first place in that order
  const int* cu;            // and its first token;
  int tok;                  // tokens of a group
};

// Few queries over many keys (bf16 forward): a group is 32 queries of one
// segment and `keys` of its keys, one block and head each; the block's four
// waves take every fourth tile of 32 keys for the same queries, and each leaves
// its unnormalised output, maximum and sum.  One more launch joins them.
struct RelSplit {
  int keys;        // keys of a group, a multiple of 128; 0: not split
  int most;        // groups at most
  int4* where;     // [total_q]: a query's first group, how many it has, its row in them (no groups: in no segment)
  float* acc;      // [groups][4][heads][32][head_dim]
  float2* ml;      // [groups][4][heads][32] maximum (powers of two) and sum
};
constexpr int kSplitRows = 32;
constexpr int kSplitMaxSegments = 2048;
// Groups of a segment: its keys are cut where its queries fit one group.
DEVI int2 split_groups(int queries, int keys, int per) {
  const int ng = (queries + kSplitRows - 1) / kSplitRows;
  return make_int2(ng, ng == 1 ? max(1, (keys + per - 1) / per) : 1);
}

// What a call's attention passes read besides its tensors.
struct RelPass {
  RelBias bias;
  int4* plan_q; int4* plan_k;       // groups of 128 or 64 tokens (seg_plan_block); plan_k backward only
  int* count_q; int* count_k;
  int* shift_q; int* shift_k;       // per group: d = key token - query token - shift
  int* first_q; int* segment_q;     // backward: RelBias's first and segment
  float* knorm; int tk_tiles;       // bf16 forward: max |k| per (head, 32-key tile)
  float2* rows; int tq_pad;         // backward: row statistics [heads][tq_pad]
  RelSplit split;                   // bf16 forward of few queries
  int group_tok;   // fp32: tokens of a group
};

// The preparation: plans, bias lines and the rows of tokens in no segment.
struct RelPrep {
  const int* cu_q; const int* cu_k; const int* q_start; int nseg;   // q_start null: every segment's queries begin at 0
  int total_q, total_k, heads, row16;                               // row16: 16-byte chunks of a token's row
  const void* table; int table_dtype;                               // [buckets][heads]
  int starts[kRelMaxBuckets / 2]; int side; bool two_sided;         // distances at which a side's buckets begin
  float* line; float* top; int2* ranges;
  uint4* zero_q; uint4* zero_k; uint4* zero_v; float* lse;          // out or dq; dk, dv; forward: lse
  bool backward, key_pairs;
  int gtok_q, gtok_k;                                               // tokens of a group of queries, of keys
};
constexpr int kRelClearBlocks = 16;
inline int rel_prep_blocks(const RelPrep& p) { return 1 + (p.backward ? 2 : 0) + p.heads + kRelClearBlocks; }

// esa_attn_dense.hip (bf16: its own kernels at head dim 16 without dropout, else the next file's), esa_attn_wide.hip,
// esa_attn.hip (fp32).
int dense_rel_fwd(const DenseAttnCall& c, const RelPass& r, RelPrep p, hipStream_t st);
int dense_rel_bwd(const DenseAttnCall& c, const RelPass& r, RelPrep p, hipStream_t st);
int wide_rel_fwd(const DenseAttnCall& c, const RelPass& r, const RelPrep& p, hipStream_t st);
int wide_rel_bwd(const DenseAttnCall& c, const RelPass& r, const RelPrep& p, hipStream_t st);
int f32_rel_fwd(const DenseAttnCall& c, const RelPass& r, const RelPrep& p, hipStream_t st);
int f32_rel_bwd(const DenseAttnCall& c, const RelPass& r, const RelPrep& p, hipStream_t st);

namespace {

extern __shared__ __align__(16) float sRel[];   // the head's bias line; the dQ pass's sums behind it

// LDS floats of the dQ pass: the bias line, then for each wave a line of sums, then the far sums of every wave.
inline size_t rel_dq_floats(int stride, int waves) { return (size_t)stride * (1 + waves) + 2 * waves; }

// Entry of distance 0 at key k0 and query q0 (both first of their tiles).
DEVI int rel_base(const RelBias& r, int k0, int q0, int shift) { return k0 - q0 - shift + r.reach + kRelPad; }
// Whether keys k0 .. k0 + nk - 1 and queries q0 .. q0 + nq - 1 (base = rel_base) have a distance inside (-reach, reach);
// if not, `far_hi` says on which side.
DEVI bool rel_near(const RelBias& r, int base, int nk, int nq, bool& far_hi) {
  far_hi = base - (nq - 1) >= 2 * r.reach + kRelPad;
  return !far_hi && base + nk - 1 > kRelPad;
}

// The base moved to where the same nk by nq tile's entries lie in the line: a tile beyond its ends reads their one value
// from its pads (nk + nq - 2 entries lie within 96).  A tile then needs no case of its own where only scores are wanted.
DEVI int rel_within(const RelBias& r, int base, int nk, int nq) { return min(max(base, nq - 1), r.stride - nk); }

constexpr int kRelMaxStride = 2 * (kRelMaxReach + kRelPad) + 1;
// All of a thread's loads first: one wait for them in a block's start, not one an entry.
template <int THREADS>
DEVI void rel_load_line(float* dst, const RelBias& r, int head, int tid) {
  constexpr int N = (kRelMaxStride + THREADS - 1) / THREADS;
  float x[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int i = tid + j * THREADS;
    x[j] = i < r.stride ? r.line[(size_t)head * r.stride + i] : 0.f;
  }
#pragma unroll
  for (int j = 0; j < N; ++j)
    if (tid + j * THREADS < r.stride) dst[tid + j * THREADS] = x[j];
}

// x of the next lane (lane 63: zero, or lane 0's).
DEVI float lane_up(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x130, 0xf, 0xf, true));
}
DEVI float lane_round(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x134, 0xf, 0xf, true));
}
// a = (a's lanes 0 .. 31, b's lanes 0 .. 31), b = (a's lanes 32 .. 63, b's lanes 32 .. 63).
DEVI void swap_halves(float& a, float& b) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  a = __uint_as_float(r[0]);
  b = __uint_as_float(r[1]);
}
// Quarters of 16 lanes: a = (a0, b0, a2, b2), b = (a1, b1, a3, b3).
DEVI void swap_quarters(float& a, float& b) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  a = __uint_as_float(r[0]);
  b = __uint_as_float(r[1]);
}

// One wave's sums of dS by distance.
struct RelSums {
  float* line;    // [stride], this wave's
  float lo, hi;   // this lane's sums past -reach and reach
  DEVI RelSums(float* lds, int stride, int wave) : line(lds + (size_t)stride * (1 + wave)), lo(0.f), hi(0.f) {}
  DEVI void clear(int stride, int lane) {
    for (int i = lane; i < stride; i += 64) line[i] = 0.f;
  }
  // Adds v[row] of lane C to entry top + row - C, for two blocks of 16 rows: four chains side by side, as a shifted
  // operand must be two instructions old.
  DEVI void diagonals(const float (&v0)[16], int top0, const float (&v1)[16], int top1, int lane) {
    float a0 = v0[15], z0 = v0[15], a1 = v1[15], z1 = v1[15];
#pragma unroll
    for (int r = 14; r >= 0; --r) {
      a0 = lane_up(a0) + v0[r];
      a1 = lane_up(a1) + v1[r];
      z0 = lane_round(z0) + v0[r];
      z1 = lane_round(z1) + v1[r];
    }
    line[top0 - lane] += a0;
    if (lane > 48) line[top0 - lane + 64] += z0 - a0;
    line[top1 - lane] += a1;
    if (lane > 48) line[top1 - lane + 64] += z1 - a1;
  }
  // Two 32 x 32 tiles of a stage (keys 16 (r / 8) + 8 (lane / 32) + r % 8 and 32 more, queries lane % 32).
  DEVI void stage32(float (&t0)[16], float (&t1)[16], int base, int lane) {
    float v[2][16];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      swap_halves(t1[r], t0[r]);   // the second tile's keys are 32 further: its queries' lanes come first
      v[r >> 3][r & 7] = t1[r];
      v[r >> 3][8 + (r & 7)] = t0[r];
    }
    diagonals(v[0], base + 32, v[1], base + 48, lane);
  }
  // Four 16 x 16 blocks t[i][r]: keys 16 i + 4 (lane / 16) + r, queries lane % 16.
  static DEVI void rows16(const f32x4 (&t)[4], float (&v)[16]) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float w0 = t[3][r], w1 = t[2][r], w2 = t[1][r], w3 = t[0][r];   // lane quarter i is to hold block 3 - i
      swap_halves(w0, w2);
      swap_halves(w1, w3);
      swap_quarters(w0, w1);
      swap_quarters(w2, w3);
      v[r] = w0;
      v[4 + r] = w1;
      v[8 + r] = w2;
      v[12 + r] = w3;
    }
  }
  // The wave's B query blocks of 16 (B 1 or 2) by the stage's four key blocks.
  template <int B>
  DEVI void stage16(const f32x4 (&t)[B][4], int base, int lane) {
    float v[2][16];
    rows16(t[0], v[0]);
    if constexpr (B == 2) rows16(t[1], v[1]);
    else
#pragma unroll
      for (int r = 0; r < 16; ++r) v[1][r] = 0.f;
    diagonals(v[0], base + 48, v[1], base + 32, lane);
  }
};

// The block's dS sums by bucket: every thread of the block, after its waves' last stage.  lds: as rel_dq_floats.
// Eight lanes a bucket: the outer ones hold a hundred distances and more.
template <int THREADS>
DEVI void rel_fold(float* lds, const RelSums& own, const RelBias& r, float* part, int wave, int lane, int tid) {
  constexpr int waves = THREADS / 64;
  float lo = own.lo, hi = own.hi;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    lo += __shfl_xor(lo, o);
    hi += __shfl_xor(hi, o);
  }
  float* far = lds + (size_t)r.stride * (1 + waves);
  if (lane == 0) {
    far[2 * wave] = lo;
    far[2 * wave + 1] = hi;
  }
  __syncthreads();
  float* first = lds + r.stride;
  for (int i = tid; i < r.stride; i += THREADS) {
    float x = first[i];
#pragma unroll
    for (int w = 1; w < waves; ++w) x += first[w * r.stride + i];
    first[i] = x;
  }
  __syncthreads();
  for (int b = tid >> 3; b < r.buckets; b += THREADS / 8) {
    const int2 range = r.ranges[b];
    float x = 0.f;
#pragma unroll 4
    for (int i = range.x + (tid & 7); i < range.y; i += 8) x += first[i];
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) x += __shfl_xor(x, o);
    if (tid & 7) continue;
#pragma unroll
    for (int w = 0; w < waves; ++w) x += (b == r.far_lo ? far[2 * w] : 0.f) + (b == r.far_hi ? far[2 * w + 1] : 0.f);
    part[b] = x;
  }
}

// The bucket of distance d: the last one of its side that begins at or before it.
DEVI int rel_bucket(const RelPrep& p, int d) {
  const int far = p.two_sided ? abs(d) : max(-d, 0);
  int lo = 0, hi = p.side;   // starts[0] = 0 <= far
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (p.starts[mid] <= far) lo = mid; else hi = mid;
  }
  return lo + (p.two_sided && d > 0 ? p.side : 0);
}

// Exclusive sums over 256 threads.
DEVI int before_me(int x, int tid) {
  __shared__ int waves[4];
  int sum = x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(sum, o);
    if ((tid & 63) >= o) sum += y;
  }
  if ((tid & 63) == 63) waves[tid >> 6] = sum;
  __syncthreads();
  for (int w = 0; w < tid >> 6; ++w) sum += waves[w];
  return sum - x;
}

// The groups of a split forward (at most kSplitMaxSegments segments), in order.
template <class ShiftOf>
DEVI void split_plan_block(const RelPrep& p, const RelPass& r, int tid, ShiftOf shift_of) {
  constexpr int PER = kSplitMaxSegments / 256;
  __shared__ int first[kSplitMaxSegments + 1];
  __shared__ int all;
  int loc[PER], sum = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int s = tid * PER + i;
    loc[i] = sum;
    if (s < p.nseg) {
      const int2 n = split_groups(max(p.cu_q[s + 1] - p.cu_q[s], 0), p.cu_k[s + 1] - p.cu_k[s], r.split.keys);
      sum += n.x * n.y;
    }
  }
  const int base = before_me(sum, tid);
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int s = tid * PER + i;
    first[s] = base + loc[i];
  }
  if (tid == 255) {
    all = first[kSplitMaxSegments] = base + sum;
    *r.count_q = base + sum;
  }
  __syncthreads();
  for (int e = tid; e < all; e += 256) {
    int lo = 0, hi = p.nseg;   // the last segment that begins at or before e: it is not empty
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (first[mid] <= e) lo = mid; else hi = mid;
    }
    const int qb = p.cu_q[lo], qe = p.cu_q[lo + 1], kb = p.cu_k[lo], ke = max(p.cu_k[lo + 1], kb);
    const int2 n = split_groups(qe - qb, ke - kb, r.split.keys);
    const int g = (e - first[lo]) / n.y, c = (e - first[lo]) % n.y, q0 = qb + g * kSplitRows;
    const int k0 = n.y == 1 ? kb : kb + c * r.split.keys;
    r.plan_q[e] = make_int4(q0, min(q0 + kSplitRows, qe), k0, n.y == 1 ? ke : min(k0 + r.split.keys, ke));
    r.shift_q[e] = shift_of(lo);
    if (c == 0)
      for (int t = q0; t < min(q0 + kSplitRows, qe); ++t) r.split.where[t] = make_int4(e, n.y, t - q0, 0);
  }
}

// first[s] = groups of the segments before s.  The plan lists groups of equal work in any order; the table's partial sums
// are added in this one.
DEVI void seg_first_block(const int* cu, int nseg, int gtok, int* first, int tid) {
  const int per = (nseg + 255) / 256, s0 = min(tid * per, nseg), s1 = min(s0 + per, nseg);
  auto groups = [&](int s) { return max(cu[s + 1] - cu[s] + gtok - 1, 0) / gtok; };
  int sum = 0;
  for (int s = s0; s < s1; ++s) sum += groups(s);
  int at = before_me(sum, tid);
  for (int s = s0; s < s1; ++s) {
    first[s] = at;
    at += groups(s);
  }
}
// The place of listed group `item`, which begins at token x.
DEVI int rel_place(const RelBias& r, int item, int x) {
  const int s = r.segment[item];
  return r.first[s] + (x - r.cu[s]) / r.tok;
}

// Block b of the preparation's rel_prep_blocks (256 threads).
DEVI void rel_prep_block(const RelPrep& p, const RelPass& r, int b, int tid) {
  auto shift_of = [&](int s) {
    const int start = p.q_start ? min(max(p.q_start[s], -(1 << 30)), 1 << 30) : 0;
    return p.cu_k[s] - p.cu_q[s] + start;
  };
  if (b == 0 && r.split.keys) {
    split_plan_block(p, r, tid, shift_of);
    return;
  }
  if (b == 0) {
    seg_plan_block(p.cu_q, p.cu_k, p.nseg, p.gtok_q, r.plan_q, r.count_q, tid, false, [&](int i, int s, int) {
      r.shift_q[i] = shift_of(s);
      if (p.backward) r.segment_q[i] = s;
    });
    return;
  }
  b -= 1;
  if (p.backward) {
    if (b == 0) {
      seg_plan_block(p.cu_k, p.cu_q, p.nseg, p.gtok_k, r.plan_k, r.count_k, tid, p.key_pairs,
                     [&](int i, int s, int) { r.shift_k[i] = shift_of(s); });
      return;
    }
    if (b == 1) {
      seg_first_block(p.cu_q, p.nseg, p.gtok_q, r.first_q, tid);
      return;
    }
    b -= 2;
  }
  if (b < p.heads) {   // one head's line
    __shared__ float most[4];
    auto entry = [&](int bucket) {
      const size_t i = (size_t)bucket * p.heads + b;
      return p.table_dtype == 0 ? static_cast<const float*>(p.table)[i] : (float)static_cast<const bf16*>(p.table)[i];
    };
    float top = 0.f;
    for (int x = tid; x < r.bias.buckets; x += 256) {
      const float v = entry(x);
      top = v == -INFINITY ? top : !(fabsf(v) <= kRelLargest) && v == v ? fmaxf(top, kRelLargest) : v == v ? fmaxf(top, fabsf(v)) : INFINITY;
    }
    top = wave_max(top);
    if ((tid & 63) == 0) most[tid >> 6] = top;
    __syncthreads();
    if (tid == 0) p.top[b] = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])) * kLog2e;
    for (int i = tid; i < r.bias.stride; i += 256) {
      const float v = entry(rel_bucket(p, i - r.bias.reach - kRelPad));
      // -inf leaves its pairs out; a NaN stays one
      const float x = v == -INFINITY || v != v ? v : fminf(fmaxf(v, -kRelLargest), kRelLargest);
      p.line[(size_t)b * r.bias.stride + i] = x * kLog2e;
    }
    if (b == 0)
      for (int x = tid; x < r.bias.buckets; x += 256) {   // entries of each bucket, the line's ends included
        const bool up = p.two_sided && x >= p.side;
        const int j = up ? x - p.side : x, zero = r.bias.reach + kRelPad;
        const int lo = p.starts[j], hi = j + 1 < p.side ? p.starts[j + 1] : INT_MAX;   // distances [lo, hi)
        int2 e;
        if (up) e = make_int2(zero + max(lo, 1), hi == INT_MAX ? r.bias.stride : zero + max(hi, 1));
        else e = make_int2(hi == INT_MAX ? 0 : zero - hi + 1, p.two_sided || j > 0 ? zero - lo + 1 : r.bias.stride);
        p.ranges[x] = e;
      }
    return;
  }
  b -= p.heads;
  // rows of tokens in no segment: zeros, and an lse of -inf
  auto clear = [&](uint4* rows, const int* cu, int total) {
    if (!rows) return;
    const size_t first = (size_t)min(max(cu[0], 0), total) * p.row16;
    const size_t from = (size_t)min(max(cu[p.nseg], 0), total) * p.row16, to = (size_t)total * p.row16;
    for (size_t i = (size_t)b * 256 + tid; i < first; i += (size_t)kRelClearBlocks * 256) rows[i] = make_uint4(0, 0, 0, 0);
    for (size_t i = from + (size_t)b * 256 + tid; i < to; i += (size_t)kRelClearBlocks * 256)
      rows[i] = make_uint4(0, 0, 0, 0);
  };
  clear(p.zero_q, p.cu_q, p.total_q);
  clear(p.zero_k, p.cu_k, p.total_k);
  clear(p.zero_v, p.cu_k, p.total_k);
  const int first = min(max(p.cu_q[0], 0), p.total_q), from = min(max(p.cu_q[p.nseg], 0), p.total_q);
  auto each = [&](auto use) {
    for (int t = b * 256 + tid; t < first; t += kRelClearBlocks * 256) use(t);
    for (int t = from + b * 256 + tid; t < p.total_q; t += kRelClearBlocks * 256) use(t);
  };
  if (r.split.keys) each([&](int t) { r.split.where[t] = make_int4(0, 0, 0, 0); });
  if (p.lse)
    for (int h = 0; h < p.heads; ++h) each([&](int t) { p.lse[(size_t)h * p.total_q + t] = -INFINITY; });
}

}  // namespace
