// Work split of the tree attention, shared by its kernels (tree_attention.cu, tree_attention_tc.cu).
//
// A unit is one (sequence, cache head) and one block of its query rows (rows = the G query heads that read the cache
// head, times the nodes).  Its keys come in tiles: first the filled rows of the cache, then the drafted nodes.  All units'
// tiles, laid end to end, are cut into `groups` equal runs, one per CTA, whatever the sequences' lengths are; those are read
// on the device, so a captured call follows them.  Starting and ending a unit (its queries, its mask, its rows) takes a CTA as
// long as a few tiles, so `unit_cost` empty tiles stand behind each unit's own: without them the CTA that got the
// shortest sequences' units, nine of them beside twelve tiles elsewhere, ran three times as long as the others.
// A unit that falls into several runs leaves one partial result per run (fp32 rows, running maximum, sum), which the combine
// kernel folds in the order of the runs.
#pragma once

#include "common.cuh"

namespace lrqk {
namespace tree {

struct Params {
  const void *q, *cache_k, *cache_v, *tree_k, *tree_v;
  int64_t q_stride[3], ck_stride[3], cv_stride[3], tk_stride[3], tv_stride[3];
  const int32_t *lens;      // [batch] or null: all `capacity` rows
  const uint8_t *mask;      // [nodes][nodes] bytes per sequence, or null: node i sees nodes 0..i
  int64_t mask_stride;      // between sequences
  void *out;                // dense [batch][q_heads][nodes][head_dim]
  float *lse;               // dense [batch][q_heads][nodes] or null
  int32_t *status;          // device word that takes LRQK_ETIMEOUT
  float *part;              // partial rows: [slot][rows_per_block][head_dim], slot = (group * 2 + which) * row_blocks + block
  float2 *part_ml;          // [slot][rows_per_block]: maximum (base-2 logarithm units), sum
  float scale_log2;         // scale * log2(e)
  float per_node;           // 1 / nodes
  int32_t batch, nodes, q_heads, cache_heads, tree_heads, head_dim, capacity;
  int32_t rows;             // query rows of a unit: q_heads / cache_heads * nodes
  int32_t rows_per_block, row_blocks, groups, tile_keys, tree_tiles, unit_cost;
};

__device__ __forceinline__ int cache_len(const Params &p, int b) {
  if (!p.lens) return p.capacity;
  return min(max(p.lens[b], 0), p.capacity);      // a length outside the cache is cut to it
}
__device__ __forceinline__ int cache_tiles(const Params &p, int len) { return (len + p.tile_keys - 1) / p.tile_keys; }
__device__ __forceinline__ int unit_span(const Params &p, int ctiles) { return ctiles + p.tree_tiles + p.unit_cost; }

// The cut of `total` tiles (below 2^30, checked on the host) into runs: the first `more` runs have one tile more.
struct Cut {
  int each, more;
  __device__ __forceinline__ Cut(const Params &p, int total) : each(total / p.groups), more(total - each * p.groups) {}
  __device__ __forceinline__ int start(int g) const { return g * each + min(g, more); }
  // the run that holds tile x (every tile is in one: with each = 0 only the first `more` runs hold any)
  __device__ __forceinline__ int of(int x) const {
    const int big = more * (each + 1);
    return x < big ? x / (each + 1) : more + (x - big) / each;
  }
};

// One warp: the tiles of all sequences, of those before sequence `upto`, and of sequence `upto` itself (its own cache tiles).
struct Count { int total, before, ctiles; };
__device__ __forceinline__ Count count_tiles(const Params &p, int upto) {
  const int lane = threadIdx.x & 31;
  int s = 0, t = 0, own = 0;
  for (int b = lane; b < p.batch; b += 32) {
    const int c = cache_tiles(p, cache_len(p, b)), n = p.cache_heads * unit_span(p, c);
    t += n;
    if (b < upto) s += n;
    if (b == upto) own = c;
  }
  Count r;
  r.total = __reduce_add_sync(0xFFFFFFFFu, t);
  r.before = __reduce_add_sync(0xFFFFFFFFu, s);
  r.ctiles = __reduce_add_sync(0xFFFFFFFFu, own);
  return r;
}

// One warp: the sequence that tile x belongs to and the first tile of that sequence.
__device__ __forceinline__ void find_sequence(const Params &p, int x, int &seq, int &base) {
  const int lane = threadIdx.x & 31;
  int run = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 32) {
    const int b = b0 + lane;
    const int n = b < p.batch ? p.cache_heads * unit_span(p, cache_tiles(p, cache_len(p, b))) : 0;
    int sum = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xFFFFFFFFu, sum, o);
      if (lane >= o) sum += up;
    }
    const unsigned hit = __ballot_sync(0xFFFFFFFFu, b < p.batch && run + sum > x);
    if (hit) {
      const int l = __ffs(hit) - 1;
      seq = b0 + l;
      base = run + __shfl_sync(0xFFFFFFFFu, sum - n, l);
      return;
    }
    run += __shfl_sync(0xFFFFFFFFu, sum, 31);
  }
  seq = p.batch;
  base = run;
}

// The segments of one group's run [x0, x1): for (Walk w(...); w.valid(); w.next(p)).
struct Walk {
  int x0, end, base, unit;       // the run; first tile of the sequence, of the unit
  int b, len, ctiles, per;       // sequence, its length, cache tiles and own tiles of a unit
  int head, t0, t1;              // the segment: cache head, tiles [t0, t1) of the unit
  __device__ __forceinline__ Walk(const Params &p, int run0, int run1, int seq, int seq_base)
      : x0(run0), end(run1), base(seq_base), b(seq) {
    if (x0 >= end) { unit = end; return; }
    size(p);
    const int span = unit_span(p, ctiles);
    head = (x0 - base) / span;
    unit = base + head * span;
    t0 = x0 - unit;
    t1 = min(per, end - unit);
    if (t0 >= per) next(p);      // the run starts on empty tiles
  }
  __device__ __forceinline__ void size(const Params &p) {
    len = cache_len(p, b);
    ctiles = cache_tiles(p, len);
    per = ctiles + p.tree_tiles;
  }
  __device__ __forceinline__ bool valid() const { return unit < end; }
  __device__ __forceinline__ bool whole() const { return t0 == 0 && t1 == per; }
  __device__ __forceinline__ void next(const Params &p) {
    unit += unit_span(p, ctiles);
    if (unit >= end) return;
    if (++head == p.cache_heads) {
      head = 0;
      base = unit;
      ++b;
      size(p);
    }
    t0 = 0;
    t1 = min(per, end - unit);
  }
  // where the partial of this segment goes: to slot 0 for the unit that the run starts in, to slot 1 for the one it ends in
  __device__ __forceinline__ int64_t slot(const Params &p, int group, int block) const {
    return ((int64_t)group * 2 + (x0 >= unit ? 0 : 1)) * p.row_blocks + block;
  }
};

// row / nodes for a row of a unit, without an integer division: below 2^16 rows the product is within 2^-6 / nodes of
// (row + 1/2) / nodes, which lies half of 1 / nodes from a whole number.
__device__ __forceinline__ int group_row(const Params &p, int row) { return (int)(((float)row + 0.5f) * p.per_node); }

// Does row `row` of the unit (node row % nodes) see drafted node j of sequence b?
__device__ __forceinline__ bool sees(const Params &p, int b, int node, int j) {
  return p.mask ? p.mask[b * p.mask_stride + (int64_t)node * p.nodes + j] != 0 : j <= node;
}

int launch_tc(const Params &p, cudaStream_t stream);     // bf16: tcgen05 kernel (tree_attention_tc.cu)
void plan_tc(Params &p);

}  // namespace tree
}  // namespace lrqk
