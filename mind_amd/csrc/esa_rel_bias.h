// The learned bias by relative position inside the unmasked attention kernels
// (esa_rel_attn_fwd / _bwd): scores get table[bucket(d)][head], d = key
// position - query position in their segment.
//
// The preparation pass writes the table out by distance: per head a line of
// bias * log2(e) at entry d + reach + kRelPad.  From `reach` (the distance at
// which a side's last bucket begins) on the bias is constant, so only tiles
// that cross |d| < reach read the line (from LDS, one entry per score); every
// other tile has one value, which the exponent's FMA takes for free.
//
// The table's gradient sums dS over the pairs of a bucket, in a fixed order
// and without global atomics: in the dQ pass each wave adds its dS by distance
// to a ring of 128 LDS entries per lane group (lanes of a group own different
// queries, so the lanes of one instruction never meet in an entry, and a
// wave's LDS operations execute in order); once a stage is done, the 64
// distances that no later key of the wave's 32 queries can reach go to the
// wave's line.  A block folds its lines into buckets, and a last launch sums
// the blocks.
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
  float* part;              // dQ pass: [groups][heads][buckets]
};

// What a call's attention passes read besides its tensors.
struct RelPass {
  RelBias bias;
  int4* plan_q; int4* plan_k;       // groups of 128 tokens (seg_plan_block); plan_k backward only
  int* count_q; int* count_k;
  int* shift_q; int* shift_k;       // per group: d = key token - query token - shift
  float* knorm; int tk_tiles;       // bf16 forward: max |k| per (head, 32-key tile)
  float2* rows; int tq_pad;         // backward: row statistics [heads][tq_pad]
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
};
constexpr int kRelClearBlocks = 16;
inline int rel_prep_blocks(const RelPrep& p) { return 1 + (p.backward ? 1 : 0) + p.heads + kRelClearBlocks; }

// esa_attn_wide.hip (bf16) and esa_attn.hip (fp32).
int wide_rel_fwd(const DenseAttnCall& c, const RelPass& r, const RelPrep& p, hipStream_t st);
int wide_rel_bwd(const DenseAttnCall& c, const RelPass& r, const RelPrep& p, hipStream_t st);
int f32_rel_fwd(const DenseAttnCall& c, const RelPass& r, const RelPrep& p, hipStream_t st);
int f32_rel_bwd(const DenseAttnCall& c, const RelPass& r, const RelPrep& p, hipStream_t st);

namespace {

extern __shared__ __align__(16) float sRel[];   // the head's bias line; the dQ pass's sums behind it

constexpr int kRelRing = 128;

// LDS floats of the dQ pass: the bias line, then per wave a ring for each lane group and a line of sums, then the far
// sums of every wave.
inline size_t rel_dq_floats(int stride, int waves, int groups) {
  return (size_t)stride + (size_t)waves * (groups * kRelRing + stride) + 2 * waves;
}

// Entry of distance 0 at key k0 and query q0 (both first of their tiles).
DEVI int rel_base(const RelBias& r, int k0, int q0, int shift) { return k0 - q0 - shift + r.reach + kRelPad; }
// Whether keys k0 .. k0 + nk - 1 and queries q0 .. q0 + nq - 1 (base = rel_base) have a distance inside (-reach, reach);
// if not, `far_hi` says on which side.
DEVI bool rel_near(const RelBias& r, int base, int nk, int nq, bool& far_hi) {
  far_hi = base - (nq - 1) >= 2 * r.reach + kRelPad;
  return !far_hi && base + nk - 1 > kRelPad;
}

DEVI void rel_load_line(float* dst, const RelBias& r, int head, int tid, int threads) {
  for (int i = tid; i < r.stride; i += threads) dst[i] = r.line[(size_t)head * r.stride + i];
}

// One wave's sums of dS by distance.
template <int GROUPS>
struct RelSums {
  float* ring;    // [GROUPS][kRelRing]
  float* line;    // [stride]
  float* mine;    // this lane group's ring
  int done;       // entries below are in the line (negative: none was added)
  float lo, hi;   // this lane's sums past -reach and reach
  DEVI RelSums(float* lds, int stride, int waves, int wave, int group)
      : ring(lds + stride + (size_t)wave * (GROUPS * kRelRing + stride)), line(ring + GROUPS * kRelRing),
        mine(ring + group * kRelRing), done(-1), lo(0.f), hi(0.f) {}
  DEVI void clear(int stride, int lane) {   // ring and line are one run
    for (int i = lane; i < GROUPS * kRelRing + stride; i += 64) ring[i] = 0.f;
  }
  DEVI void add(int entry, float x) {
    __hip_atomic_fetch_add(&mine[entry & (kRelRing - 1)], x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WAVEFRONT);
  }
  DEVI void flush(int first, int stride, int lane) {    // entries first .. first + 63
    const int s = (first + lane) & (kRelRing - 1);
    float x = 0.f;
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      x += ring[g * kRelRing + s];
      ring[g * kRelRing + s] = 0.f;
    }
    if (first + lane < stride) line[first + lane] += x;   // past it nothing was added
  }
  // After a stage of 64 keys (base = rel_base of its first key) with a near tile: 32 queries' entries below
  // base + 64 - 31 are complete.
  DEVI void stage_done(int base, int stride, int lane) {
    flush(base - 31, stride, lane);
    done = base + 33;
  }
  DEVI void finish(int stride, int lane) {
    if (done >= 0) flush(done, stride, lane);
  }
};

// The block's dS sums by bucket: every thread of the block, after its waves' last add.  lds: as rel_dq_floats.
template <int GROUPS>
DEVI void rel_fold(float* lds, RelSums<GROUPS>& own, const RelBias& r, float* part, int waves, int wave, int lane,
                   int tid, int threads) {
  own.finish(r.stride, lane);
  float lo = own.lo, hi = own.hi;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    lo += __shfl_xor(lo, o);
    hi += __shfl_xor(hi, o);
  }
  const size_t per = (size_t)GROUPS * kRelRing + r.stride;
  float* far = lds + r.stride + waves * per;
  if (lane == 0) {
    far[2 * wave] = lo;
    far[2 * wave + 1] = hi;
  }
  __syncthreads();
  float* first = lds + r.stride + GROUPS * kRelRing;
  for (int i = tid; i < r.stride; i += threads) {
    float x = first[i];
    for (int w = 1; w < waves; ++w) x += first[w * per + i];
    first[i] = x;
  }
  __syncthreads();
  for (int b = tid; b < r.buckets; b += threads) {
    const int2 range = r.ranges[b];
    float x = 0.f;
    for (int i = range.x; i < range.y; ++i) x += first[i];
    if (b == r.far_lo)
      for (int w = 0; w < waves; ++w) x += far[2 * w];
    if (b == r.far_hi)
      for (int w = 0; w < waves; ++w) x += far[2 * w + 1];
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

// Block b of the preparation's rel_prep_blocks (256 threads).
DEVI void rel_prep_block(const RelPrep& p, const RelPass& r, int b, int tid) {
  auto shift_of = [&](int s) {
    const int start = p.q_start ? min(max(p.q_start[s], -(1 << 30)), 1 << 30) : 0;
    return p.cu_k[s] - p.cu_q[s] + start;
  };
  if (b == 0) {
    seg_plan_block(p.cu_q, p.cu_k, p.nseg, kGroupTok, r.plan_q, r.count_q, tid, false, r.shift_q, shift_of);
    return;
  }
  b -= 1;
  if (p.backward) {
    if (b == 0) {
      seg_plan_block(p.cu_k, p.cu_q, p.nseg, kGroupTok, r.plan_k, r.count_k, tid, p.key_pairs, r.shift_k, shift_of);
      return;
    }
    b -= 1;
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
    const size_t from = (size_t)min(max(cu[p.nseg], 0), total) * p.row16, to = (size_t)total * p.row16;
    for (size_t i = from + (size_t)b * 256 + tid; i < to; i += (size_t)kRelClearBlocks * 256)
      rows[i] = make_uint4(0, 0, 0, 0);
  };
  clear(p.zero_q, p.cu_q, p.total_q);
  clear(p.zero_k, p.cu_k, p.total_k);
  clear(p.zero_v, p.cu_k, p.total_k);
  if (p.lse) {
    const int from = min(max(p.cu_q[p.nseg], 0), p.total_q);
    for (int h = 0; h < p.heads; ++h)
      for (int t = from + b * 256 + tid; t < p.total_q; t += kRelClearBlocks * 256)
        p.lse[(size_t)h * p.total_q + t] = -INFINITY;
  }
}

}  // namespace
