// Choice of a token from logits: temperature, top-k, top-p, min-p and a given random number, one cluster per row.
//
//   w_i = exp((l_i - max) / T);  keep the k largest logits (equal ones: lowest index first);  of those, in descending
//   order, keep a token while the mass strictly before it is below p times their sum;  of those keep w_i >= m;  the token is
//   the first kept one, in index order, whose cumulative mass exceeds u times the kept sum.  T = 0: the first maximum.
//
// Every one of these decisions is a comparison of sums, and a sum in fp32 decides differently from one in another order as
// soon as a number falls near a border.  So weights are 45-bit whole numbers, W = round(2^44 w), from an exponential in
// double (own: Taylor to the fourth order around 128 table values of 2^x, Tang's table method): whole-number sums have no
// order, are the same for any cluster size, and agree with 64-bit floating sums to V 2^-45 of the largest weight for V tokens
// (2^-28 for 128256: equal logits, whose roundings all go one way), to about sqrt(V) 2^-46 where roundings are independent (2^-37).
//
// A row's logits are read once, into the shared memory of the cluster's CTAs (1, 2, 4 or 8: enough SMs for few rows,
// enough memory for large vocabularies).  Top-k and top-p look for the place in the descending order where a running count
// or mass crosses its target: a histogram of counts, or of the weights' three 15-bit limbs (the sums of 2^17 of them fit
// 32 bits, so shared-memory atomics stay 32-bit), over bins of distance from the maximum, merged over the cluster in
// distributed shared memory, finds the bin; its tokens, a few hundred at most, go to a list that every CTA gets and
// settles by itself, ties included.  A bin with more (equal logits by the thousand) is cut further by key, an
// order-preserving integer of a logit, and ties are counted in index order.  Where top-k leaves a few hundred tokens in
// all, the list takes them all and the first CTA does the rest.  The final choice, in index order, comes from per-warp
// sums of contiguous chunks and a second look at one chunk.
//
// Bound: the latency of the cluster barriers for few rows (each merge is two of them, 2.7 us with the reads between);
// barriers and instructions -- the double exponential, three atomics a token -- for many.  One row of 128256 bf16 logits
// with top-k 50 takes 14 us, 25 rows with top-p alone 52 us, 64 rows of 152064 fp32 logits with mixed settings 71 us (39 MB:
// 6 us of loads).
#include <cooperative_groups.h>

#include "common.cuh"

namespace lrqk {
namespace {

namespace cg = cooperative_groups;

constexpr int kSampThreads = 512, kSampWarps = 16, kSampBins = 512, kSampMaxCluster = 8;
constexpr int kFracBits = 44;                          // of a weight
constexpr int kTable = 128;                            // values of 2^(j / 128)
constexpr int kList = 512;                             // tokens of a list (a CTA may add kList / cluster size)
constexpr size_t kSampSliceBytes = 208 * 1024;         // logits of one CTA

struct SampleParams {
  const void *logits;
  int64_t row_stride;                                  // elements
  const float *u, *temperature, *top_p, *min_p;        // per row; null: the one value below
  const int32_t *top_k;
  int64_t *tokens;
  float *logprobs;                                     // or null
  float temperature1, top_p1, min_p1;
  int32_t top_k1, vocab, chunk;                        // elements of a warp
  int32_t vectors;                                     // rows start on 16 bytes
};

struct SampleShared {
  double table[kTable];
  unsigned long long merged[kSampBins], xsum[2][kSampMaxCluster], wsum[kSampWarps], total[2], pick_above, pick_in, pick_total;
  union {
    uint32_t hist[3][kSampBins];
    struct { unsigned long long entry[kList], weight[kList]; } list;   // key and inverted index; its weight (0: dropped)
  };
  float high[kSampMaxCluster], low[kSampMaxCluster], whigh[kSampWarps], wlow[kSampWarps];
  uint32_t count[kSampMaxCluster], mine, tie_index, pick_bin, index;
};

template <typename T> struct SampKey;                  // order-preserving keys and back
template <> struct SampKey<float> {
  __device__ static __forceinline__ uint32_t of(float f) { return order_key(f); }
  __device__ static __forceinline__ float value(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k); }
};
template <> struct SampKey<__nv_bfloat16> {
  __device__ static __forceinline__ uint32_t of(float f) { return order_key(f) >> 16; }
  __device__ static __forceinline__ float value(uint32_t k) { return __uint_as_float((k & 0x8000u) ? (k ^ 0x8000u) << 16 : ~k << 16); }
};

__device__ __forceinline__ void pack(float *to, const float (&f)[4]) { *reinterpret_cast<float4 *>(to) = make_float4(f[0], f[1], f[2], f[3]); }
__device__ __forceinline__ void pack(__nv_bfloat16 *to, const float (&f)[8]) {   // (the values are bf16: an exact repacking)
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = (__float_as_uint(f[2 * i]) >> 16) | (__float_as_uint(f[2 * i + 1]) & 0xFFFF0000u);
  *reinterpret_cast<uint4 *>(to) = make_uint4(w[0], w[1], w[2], w[3]);
}

struct Cut { float value; uint32_t index; };           // kept: larger logits, and equal ones up to this index

template <typename T> struct Sampler {
  static constexpr int VE = Elt<T>::kPerVec, STEP = 32 * VE;
  const SampleParams &p;
  SampleShared &sm;
  T *vals;
  cg::cluster_group cluster;
  int rank, csize, warp, lane, flip;
  float top, dust;                                     // the row's maximum; logits up to here weigh nothing
  double per_log;                                      // 128 log2(e) / T

  __device__ Sampler(const SampleParams &params, SampleShared &shared, T *values)
      : p(params), sm(shared), vals(values), cluster(cg::this_cluster()), rank((int)cluster.block_rank()),
        csize((int)cluster.num_blocks()), warp(threadIdx.x >> 5), lane(threadIdx.x & 31), flip(0) {}

  __device__ __forceinline__ uint32_t index_of(int at) const { return (uint32_t)(rank * kSampWarps * p.chunk + at); }

  // every value of this warp's chunk replaced
  template <typename F> __device__ __forceinline__ void each_store(F fn) const {
    for (int i = lane; i < p.chunk; i += 32) vals[warp * p.chunk + i] = Elt<T>::from_float(fn(Elt<T>::to_float(vals[warp * p.chunk + i])));
  }

  // fn(values, place of the first in the slice) for this warp's chunk: four neighbours at a time
  template <typename F> __device__ __forceinline__ void each4(F fn) const {
    const int base = warp * p.chunk;
    for (int s = 0; s < p.chunk; s += STEP) {
      const int at = base + s + lane * VE;
      float f[VE];
      Elt<T>::unpack(ld16(vals + at), f);
#pragma unroll
      for (int j = 0; j < VE; j += 4) fn(f + j, at + j);
    }
  }

  // fn(value, place in the slice) for this warp's chunk, a lane's VE neighbours at a time
  template <typename F> __device__ __forceinline__ void each(F fn) const {
    const int base = warp * p.chunk;
    for (int s = 0; s < p.chunk; s += STEP) {
      const int at = base + s + lane * VE;
      float f[VE];
      Elt<T>::unpack(ld16(vals + at), f);
#pragma unroll
      for (int j = 0; j < VE; ++j) fn(f[j], at + j);
    }
  }

  __device__ __forceinline__ bool candidate(float f) const { return f > -INFINITY; }

  // round(2^44 exp((f - top) / T)), f <= top
  __device__ __forceinline__ unsigned long long weight(float f) const {
    const double y = ((double)f - (double)top) * per_log; // 128ths of an octave, above -6100 where it counts
    const double magic = 6755399441055744.0;              // 1.5 * 2^52: the sum's low bits are the nearest whole number
    const double n = y + magic;
    const int k = __double2loint(n);
    const double r = y - (n - magic);                     // |r ln(2) / 128| < 0.0028: the series' next term is below 2^-49
    const double e = fma(r, fma(r, fma(r, fma(r, 3.583032305400251e-11, 2.6466421444330967e-08), 1.4662262387640423e-05), 0.0054152123481245725), 1.0) * sm.table[k & (kTable - 1)];
    const double scaled = __hiloint2double(__double2hiint(e) + (((k >> 7) + kFracBits) << 20), __double2loint(e));
    const double whole = scaled + 4503599627370496.0;     // 2^52
    const unsigned long long w = ((unsigned long long)(uint32_t)(__double2hiint(whole) - 0x43300000) << 32) | (uint32_t)__double2loint(whole);
    return f > dust ? w : 0ull;                           // (no branch: neighbours' chains of double operations overlap)
  }

  __device__ __forceinline__ bool inside(const Cut &c, float f, int at) const {
    return f > c.value || (f == c.value && index_of(at) <= c.index);
  }

  __device__ __forceinline__ unsigned long long entry(float f, int at) const {
    return ((unsigned long long)SampKey<T>::of(f) << 32) | (0xFFFFFFFFu - index_of(at));   // descending: larger key, lower index
  }

  // Merge the histograms of the cluster and find the bin in which the running sum from bin 0 reaches target_of(total).
  // MASS: three limbs; else counts in hist[0].
  template <bool MASS, typename F> __device__ void pick(F target_of) {
    cluster.sync();
    {
      // a thread per bin of this CTA's share and source; the sources of a bin are neighbouring lanes
      const int bin = rank * (kSampBins / csize) + threadIdx.x / csize, from = threadIdx.x % csize;
      const uint32_t *h = cluster.map_shared_rank(&sm.hist[0][0], from);
      unsigned long long v = h[bin];
      if (MASS) v += ((unsigned long long)h[kSampBins + bin] << 15) + ((unsigned long long)h[2 * kSampBins + bin] << 30);
      for (int o = 1; o < csize; o <<= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
      cluster.map_shared_rank(sm.merged, from)[bin] = v;
    }
    cluster.sync();
    if (warp == 0) {
      constexpr int PER = kSampBins / 32;
      unsigned long long mine = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) mine += sm.merged[lane * PER + i];
      unsigned long long sum = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long up = __shfl_up_sync(0xFFFFFFFFu, sum, o);
        if (lane >= o) sum += up;
      }
      const unsigned long long total = __shfl_sync(0xFFFFFFFFu, sum, 31), target = target_of(total);
      const unsigned hit = __ballot_sync(0xFFFFFFFFu, sum >= target);
      const int owner = hit ? __ffs(hit) - 1 : 31;
      if (lane == owner) {
        unsigned long long above = sum - mine;
        int i = 0;
        while (i < PER - 1 && above + sm.merged[lane * PER + i] < target) above += sm.merged[lane * PER + i++];
        sm.pick_bin = lane * PER + i;
        sm.pick_above = above;
        sm.pick_in = sm.merged[lane * PER + i];
        sm.pick_total = total;
      }
    }
    __syncthreads();
  }

  template <bool MASS> __device__ __forceinline__ void add(uint32_t bin, unsigned long long w) {
    if (MASS) {
      const uint32_t l0 = (uint32_t)w & 0x7FFFu, l1 = (uint32_t)(w >> 15) & 0x7FFFu, l2 = (uint32_t)(w >> 30);
      if (l0) atomicAdd(&sm.hist[0][bin], l0);
      if (l1) atomicAdd(&sm.hist[1][bin], l1);
      if (l2) atomicAdd(&sm.hist[2][bin], l2);
    } else {
      atomicAdd(&sm.hist[0][bin], 1u);
    }
  }

  __device__ __forceinline__ void clear() {
    __syncthreads();
    for (int i = threadIdx.x; i < 3 * kSampBins; i += kSampThreads) (&sm.hist[0][0])[i] = 0u;
    __syncthreads();
  }

  // The tokens that `wanted` names, of all CTAs, into every CTA's list (in the histograms' place); their number, or -1 if
  // one CTA has more than its share of the list holds.
  template <typename F> __device__ int gather(F wanted) {
    const uint32_t share = kList / csize;
    if (threadIdx.x == 0) sm.mine = 0u;                // (the list itself is not cleared: peers may be filling it already)
    __syncthreads();
    each([&](float f, int at) {
      if (!wanted(f, at)) return;
      const uint32_t to = atomicAdd(&sm.mine, 1u);
      if (to < share) {
        const unsigned long long e = entry(f, at);
        for (int c = 0; c < csize; ++c) cluster.map_shared_rank(sm.list.entry, c)[rank * share + to] = e;
      }
    });
    __syncthreads();
    if (threadIdx.x < (unsigned)csize) cluster.map_shared_rank(sm.count, threadIdx.x)[rank] = sm.mine;
    cluster.sync();
    // closed up: thread i takes entry i of all
    int n = 0, from = -1;
    bool fits = true;
    for (int c = 0; c < csize; ++c) {
      const int m = (int)sm.count[c];
      fits = fits && m <= (int)share;
      if (from < 0 && (int)threadIdx.x < n + m) from = c * (int)share + (int)threadIdx.x - n;
      n += m;
    }
    if (!fits) {
      cluster.sync();                                  // everyone has read the counts
      return -1;
    }
    const unsigned long long e = from >= 0 ? sm.list.entry[from] : 0ull;
    __syncthreads();
    if (from >= 0) sm.list.entry[threadIdx.x] = e;
    return n;
  }

  __device__ __forceinline__ float value_of(unsigned long long e) const { return SampKey<T>::value((uint32_t)(e >> 32)); }

  // Cut the tokens inside `cut` to those from the largest down to where the count (MASS: the mass) reaches its target.
  // lowest: the smallest candidate.  Returns -1; or, for a count whose tokens all fit the list, their number, and makes no cut.
  template <bool MASS> __device__ int narrow(Cut &cut, float lowest, unsigned long long count, double share) {
    uint32_t khi = SampKey<T>::of(top), klo = SampKey<T>::of(fmaxf(MASS ? fmaxf(lowest, dust) : lowest, cut.value));
    unsigned long long target, above, in;
    // Level 0: bins by distance from the maximum.  (Halved, so that the range of any two floats is finite.)  The bin is the
    // low bits of a sum with 2^23: a conversion instruction has a quarter of the rate.  `start` is rounded with it, to half a
    // bin, alike for all logits.
    const float range = 0.5f * top - 0.5f * SampKey<T>::value(klo), per = (float)kSampBins / range;
    const float slope = -0.5f * per, start = 0.5f * top * per + 8388608.0f;
    const auto bin0 = [&](float f) { return min(kSampBins - 1, max(0, __float_as_int(fmaf(f, slope, start)) - 0x4B000000)); };
    clear();
    each4([&](const float *f, int at) {
      unsigned long long w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = MASS ? weight(f[j]) : candidate(f[j]) ? 1ull : 0ull;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (w[j] && inside(cut, f[j], at + j)) add<MASS>(bin0(f[j]), w[j]);
    });
    const auto first_target = [&](unsigned long long total) {
      if (!MASS) return min(count, total);             // fewer candidates than asked for: all of them
      const double t = ceil(share * (double)total);    // before < share * total, for whole numbers before
      return t < 1.0 ? 1ull : min(total, (unsigned long long)t);
    };
    pick<MASS>(first_target);
    const int b0 = sm.pick_bin;
    above = sm.pick_above;
    in = sm.pick_in;
    target = first_target(sm.pick_total);
    const Cut old = cut;
    if (khi != klo) {
      // keys that can lie in that bin (wider by a bin on either side, and some rounding: the test itself is bin0)
      const float slack = (fabsf(top) + 2.0f * range) * 0x1p-20f + 1e-35f, step = 2.0f * range / kSampBins;
      khi = min(khi, SampKey<T>::of(fminf(top, top - step * (float)(b0 - 1) + slack)));
      if (b0 < kSampBins - 1) klo = max(klo, SampKey<T>::of(top - step * (float)(b0 + 2) - slack));
      if (klo > khi) klo = khi;
    }
    float from = SampKey<T>::value(klo), to = SampKey<T>::value(khi);
    if (!MASS && above + in <= kList / 2) {
      const int n = gather([&](float f, int at) { return f >= from && bin0(f) <= b0; });
      if (n >= 0) return n;
    }
    const auto in_reach = [&](float f, int at) { return f >= from && f <= to && bin0(f) == b0 && inside(old, f, at); };
    for (;;) {
      // at most so many tokens are in reach: all, if each weighs no less than the smallest key
      const unsigned long long least = MASS ? weight(from) : 1ull;
      if (least && in / least <= kList / 2) {
        const int n = gather(in_reach);
        if (n >= 0) {
          settle<MASS>(cut, n, target - above);
          return -1;
        }
      }
      if (khi == klo) break;
      const int shift = max(0, 32 - __clz((int)(khi - klo)) - 9);        // 512 bins of 2^shift keys
      clear();
      each([&](float f, int at) {
        if (!in_reach(f, at)) return;
        const unsigned long long w = MASS ? weight(f) : 1ull;
        if (w) add<MASS>((khi - SampKey<T>::of(f)) >> shift, w);
      });
      pick<MASS>([&](unsigned long long) { return target - above; });
      above += sm.pick_above;
      in = sm.pick_in;
      khi -= sm.pick_bin << shift;
      klo = shift == 0 ? khi : khi - klo < (1u << shift) ? klo : khi - (1u << shift) + 1u;
      from = SampKey<T>::value(klo);
      to = SampKey<T>::value(khi);
    }
    // equal logits by the hundred: the need-th of them, in index order
    const unsigned long long each_w = MASS ? weight(to) : 1ull;
    const unsigned long long ties = each_w ? in / each_w : 0ull, need = each_w ? (target - above + each_w - 1) / each_w : 1ull;
    cut = Cut{to, to == old.value ? old.index : 0xFFFFFFFFu};
    if (need < ties) {
      locate([&](float f, int at) -> unsigned long long { return f == to && inside(old, f, at) ? 1ull : 0ull; },
             [&](unsigned long long) { return need - 1; },
             [&](uint32_t index, float, unsigned long long) {
               for (int c = 0; c < csize; ++c) *cluster.map_shared_rank(&sm.tie_index, c) = index;
             });
      cluster.sync();
      cut.index = sm.tie_index;
    }
    return -1;
  }

  // The list's n tokens settle the cut: the one at which their count (MASS: mass), in descending order, reaches `target`.
  template <bool MASS> __device__ void settle(Cut &cut, int n, unsigned long long target) {
    const int i = threadIdx.x;
    const unsigned long long e = i < n ? sm.list.entry[i] : 0ull, w = i < n ? (MASS ? weight(value_of(e)) : 1ull) : 0ull;
    if (MASS && i < n) sm.list.weight[i] = w;
    __syncthreads();
    if (i < n) {
      unsigned long long before = 0;
      for (int j = 0; j < n; ++j)
        if (sm.list.entry[j] > e) before += MASS ? sm.list.weight[j] : 1ull;
      if (before < target && before + w >= target) { sm.pick_above = e; }
    }
    __syncthreads();
    cut = Cut{value_of(sm.pick_above), 0xFFFFFFFFu - (uint32_t)sm.pick_above};
    __syncthreads();
  }

  __device__ __forceinline__ unsigned long long block_sum(unsigned long long v, int slot) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    if (lane == 0) sm.wsum[warp] = v;
    __syncthreads();
    if (warp == 0) {
      unsigned long long t = lane < kSampWarps ? sm.wsum[lane] : 0ull;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xFFFFFFFFu, t, o);
      if (lane == 0) sm.total[slot] = t;
    }
    __syncthreads();
    return sm.total[slot];
  }

  // Few tokens are left and the list holds them all (n): top-k, top-p, min-p and the choice, in one CTA.
  template <typename G, typename F> __device__ void finish(int n, unsigned long long k, double share, bool nucleus, unsigned long long floor_w, G target_of, F found) {
    const int i = threadIdx.x;
    const unsigned long long e = i < n ? sm.list.entry[i] : 0ull, w = i < n ? weight(value_of(e)) : 0ull;
    if (i < n) sm.list.weight[i] = w;
    __syncthreads();
    unsigned long long before = 0;                     // mass of the larger ones
    uint32_t rank_of = 0;
    if (i < n)
      for (int j = 0; j < n; ++j)
        if (sm.list.entry[j] > e) { before += sm.list.weight[j]; ++rank_of; }
    const bool in_k = i < n && rank_of < k;
    const unsigned long long total = block_sum(in_k ? w : 0ull, 0);
    const double t = ceil(share * (double)total);
    const unsigned long long target = t < 1.0 ? 1ull : min(total, (unsigned long long)t);
    const unsigned long long kept = in_k && (!nucleus || before < target) && w >= floor_w ? w : 0ull;
    __syncthreads();
    if (i < n) sm.list.weight[i] = kept;
    const unsigned long long sum = block_sum(kept, 1), chosen = target_of(sum);
    if (kept) {
      unsigned long long mass = 0;                     // of the kept ones of lower index (larger inverted index)
      for (int j = 0; j < n; ++j)
        if ((uint32_t)sm.list.entry[j] > (uint32_t)e) mass += sm.list.weight[j];
      if (mass <= chosen && mass + kept > chosen) found(0xFFFFFFFFu - (uint32_t)e, value_of(e), sum);
    }
  }

  // The first token, in index order, at which the cumulative weight exceeds target_of(total): found(index, value, total)
  // is called by one thread of the cluster.
  template <typename W, typename G, typename F> __device__ void locate(W weigh, G target_of, F found) {
    unsigned long long mine = 0;
    each4([&](const float *f, int at) {
      unsigned long long w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = weigh(f[j], at + j);
      mine += (w[0] + w[1]) + (w[2] + w[3]);
    });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xFFFFFFFFu, mine, o);
    if (lane == 0) sm.wsum[warp] = mine;
    __syncthreads();
    unsigned long long before_warp = 0, here = 0;
    for (int i = 0; i < kSampWarps; ++i) {
      const unsigned long long v = sm.wsum[i];
      if (i < warp) before_warp += v;
      here += v;
    }
    if (threadIdx.x < (unsigned)csize) *cluster.map_shared_rank(&sm.xsum[flip][rank], threadIdx.x) = here;
    cluster.sync();
    unsigned long long total = 0;
    for (int c = 0; c < csize; ++c) {
      const unsigned long long v = sm.xsum[flip][c];
      if (c < rank) before_warp += v;
      total += v;
    }
    flip ^= 1;
    const unsigned long long target = target_of(total);
    if (target < before_warp || target - before_warp >= mine) return;   // another warp's (the sums are exact: one warp's)
    unsigned long long run = before_warp;
    const int base = warp * p.chunk;
    for (int s = 0; s < p.chunk; s += STEP) {
      const int at = base + s + lane * VE;
      float f[VE];
      Elt<T>::unpack(ld16(vals + at), f);
      unsigned long long w[VE], sum = 0;
#pragma unroll
      for (int j = 0; j < VE; ++j) { w[j] = weigh(f[j], at + j); sum += w[j]; }
      unsigned long long upto = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long up = __shfl_up_sync(0xFFFFFFFFu, upto, o);
        if (lane >= o) upto += up;
      }
      const unsigned hit = __ballot_sync(0xFFFFFFFFu, run + upto > target);
      if (hit) {
        if (lane == __ffs(hit) - 1) {
          unsigned long long c = run + upto - sum;
#pragma unroll
          for (int j = 0; j < VE; ++j) {
            if (c <= target && c + w[j] > target) found(index_of(at + j), f[j], total);
            c += w[j];
          }
        }
        __syncwarp();
        break;
      }
      run += __shfl_sync(0xFFFFFFFFu, upto, 31);
    }
  }
};

template <typename T>
__global__ void __launch_bounds__(kSampThreads, 2) sample_kernel(const __grid_constant__ SampleParams p) {
  pdl_launch_dependents();
  extern __shared__ __align__(16) unsigned char smem_raw[];
  __shared__ SampleShared sm;
  Sampler<T> s(p, sm, reinterpret_cast<T *>(smem_raw));
  const int row = blockIdx.x / s.csize;
  constexpr int VE = Sampler<T>::VE, STEP = Sampler<T>::STEP;
  if (threadIdx.x < kTable) sm.table[threadIdx.x] = exp2((double)threadIdx.x * (1.0 / kTable));
  pdl_wait();

  // ---- the row's slice into shared memory; NaN counts as -inf, and so does what lies behind the vocabulary -----------
  const T *src = static_cast<const T *>(p.logits) + (int64_t)row * p.row_stride;
  const int base = s.warp * p.chunk;
  float high = -INFINITY, low = INFINITY;              // of the logits above -inf
  const auto note = [&](float &f) {
    f = fmaxf(f, -INFINITY);                           // (fmaxf drops a NaN)
    high = fmaxf(high, f);
    low = fminf(low, f > -INFINITY ? f : INFINITY);
  };
  if (p.vectors) {
#pragma unroll 4
    for (int i = 0; i < p.chunk; i += STEP) {
      const int at = base + i + s.lane * VE;
      const uint32_t index = s.index_of(at);
      float f[VE];
      if (index + VE <= (uint32_t)p.vocab) {
        Elt<T>::unpack(ld_stream16(src + index), f);
      } else {
#pragma unroll
        for (int j = 0; j < VE; ++j) f[j] = index + j < (uint32_t)p.vocab ? Elt<T>::to_float(src[index + j]) : -INFINITY;
      }
#pragma unroll
      for (int j = 0; j < VE; ++j) note(f[j]);
      pack(s.vals + at, f);
    }
  } else {
#pragma unroll 4
    for (int i = 0; i < p.chunk; i += 32) {
      const int at = base + i + s.lane;
      const uint32_t index = s.index_of(at);
      float f = index < (uint32_t)p.vocab ? Elt<T>::to_float(src[index]) : -INFINITY;
      note(f);
      s.vals[at] = Elt<T>::from_float(f);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    high = fmaxf(high, __shfl_xor_sync(0xFFFFFFFFu, high, o));
    low = fminf(low, __shfl_xor_sync(0xFFFFFFFFu, low, o));
  }
  if (s.lane == 0) { sm.whigh[s.warp] = high; sm.wlow[s.warp] = low; }
  if (threadIdx.x == 0) sm.index = 0xFFFFFFFFu;
  s.cluster.sync();                                    // every CTA of the cluster runs: its shared memory can be written
  if (s.warp == 0) {
    high = sm.whigh[s.lane & (kSampWarps - 1)];
    low = sm.wlow[s.lane & (kSampWarps - 1)];
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) {
      high = fmaxf(high, __shfl_xor_sync(0xFFFFFFFFu, high, o));
      low = fminf(low, __shfl_xor_sync(0xFFFFFFFFu, low, o));
    }
    if (s.lane < s.csize) {
      *s.cluster.map_shared_rank(&sm.high[s.rank], s.lane) = high;
      *s.cluster.map_shared_rank(&sm.low[s.rank], s.lane) = low;
    }
  }
  s.cluster.sync();
  high = sm.high[0];
  low = sm.low[0];
  for (int c = 1; c < s.csize; ++c) { high = fmaxf(high, sm.high[c]); low = fminf(low, sm.low[c]); }
  s.top = high;

  const float t = p.temperature ? p.temperature[row] : p.temperature1;
  const bool first = s.rank == 0 && threadIdx.x == 0;
  if (high == -INFINITY) {                             // nothing but -inf and NaN: no token
    if (first) { p.tokens[row] = -1; if (p.logprobs) p.logprobs[row] = NAN; }
  } else if (!(t > 0.0f)) {                            // the first maximum
    s.each([&](float f, int at) { if (f == high) atomicMin(s.cluster.map_shared_rank(&sm.index, 0), s.index_of(at)); });
    s.cluster.sync();
    if (first) { p.tokens[row] = sm.index; if (p.logprobs) p.logprobs[row] = 0.0f; }
  } else {
    s.per_log = 184.6649652337873 / (double)t;         // 128 log2(e) / T
    s.dust = __fsub_rd(high, 33.0f * t);               // 33 T below the maximum a weight rounds to nothing (2^-47)
    if (high == INFINITY) {                            // the infinite logits share the mass: as if they were 0, the rest nothing
      s.each_store([](float f) { return f == INFINITY ? 0.0f : -INFINITY; });
      __syncthreads();
      s.top = high = low = 0.0f;
      s.dust = -1.0f;
    }
    const int k = p.top_k ? p.top_k[row] : p.top_k1;
    const float q = p.top_p ? p.top_p[row] : p.top_p1, m = p.min_p ? p.min_p[row] : p.min_p1, u = p.u[row];
    const unsigned long long floor_w = m > 0.0f ? (unsigned long long)__double2ull_rn(fmin((double)m, 1.0) * 17592186044416.0) : 0ull;
    const auto target_of = [&](unsigned long long total) {
      const double x = floor((double)u * (double)total);
      return x > 0.0 ? min(total - 1, (unsigned long long)x) : 0ull;
    };
    const auto found = [&](uint32_t index, float f, unsigned long long total) {
      p.tokens[row] = index;
      const double y = ((double)f - (double)high) / (double)t;
      if (p.logprobs) p.logprobs[row] = (float)(y - log((double)total * 0x1p-44));
    };
    Cut cut{-INFINITY, 0u};                            // all
    int n = -1;
    if (k > 0 && k < p.vocab) n = s.template narrow<false>(cut, low, (unsigned long long)k, 0.0);
    if (n >= 0) {
      if (s.rank == 0) s.finish(n, (unsigned long long)k, (double)q, q < 1.0f, floor_w, target_of, found);
    } else {
      if (q < 1.0f) s.template narrow<true>(cut, low, 0ull, (double)q);
      s.locate(
          [&](float f, int at) -> unsigned long long {
            const unsigned long long w = s.weight(f);
            return w >= floor_w && s.inside(cut, f, at) ? w : 0ull;
          },
          target_of, found);
    }
  }
  s.cluster.sync();                                    // no CTA leaves while a peer may still write to it
}

template <typename T> int launch_sample(SampleParams &p, int rows, cudaStream_t stream) {
  // As many CTAs a row as two an SM can hold, for the passes over its slice are what takes the time: 25 rows of 128256 bf16
  // logits take 51 us with 8 and 72 with 4, 64 rows of 152064 fp32 logits 71 with 8 and 81 with 4.  Fewer for many rows, as
  // long as a slice fits.
  constexpr int step = 32 * Elt<T>::kPerVec * kSampWarps;       // a slice is a whole number of these
  int csize = 1;
  const auto slice = [&](int c) { return ceil_div64(ceil_div64(p.vocab, c), step) * step; };
  while (csize < kSampMaxCluster && (slice(csize) * (int64_t)sizeof(T) > (int64_t)kSampSliceBytes ||
                                     (rows * csize <= 2 * kNumSMs && slice(csize) > step)))
    csize *= 2;
  if (slice(csize) * (int64_t)sizeof(T) > (int64_t)kSampSliceBytes) return LRQK_EUNSUPPORTED;
  p.chunk = (int)(slice(csize) / kSampWarps);
  const size_t smem = (size_t)slice(csize) * sizeof(T);
  static SmemOptIn opt_in;
  LRQK_CUDA_TRY(opt_in.ensure(sample_kernel<T>, kSampSliceBytes));
  LRQK_CUDA_TRY(launch_dependent(sample_kernel<T>, dim3((unsigned)(rows * csize)), dim3(kSampThreads), smem, stream, csize, p));
  return LRQK_OK;
}

}  // namespace
}  // namespace lrqk

extern "C" int lrqk_sample_tokens(const lrqk_sample_args *a, lrqk_stream_t stream) {
  using namespace lrqk;
  const int rc = check_device();
  if (rc != LRQK_OK) return rc;
  if (!a || a->rows < 0 || a->vocab <= 0) return LRQK_EINVAL;
  if (a->dtype != LRQK_F32 && a->dtype != LRQK_BF16) return LRQK_EUNSUPPORTED;
  if (a->rows == 0) return LRQK_OK;
  if (!a->logits || !a->u || !a->tokens) return LRQK_EINVAL;
  if (a->row_stride < 0 || a->vocab >= (1 << 20) || a->rows > (1 << 24)) return LRQK_EUNSUPPORTED;
  SampleParams p;
  p.logits = a->logits; p.row_stride = a->row_stride; p.u = a->u;
  p.temperature = a->temperature; p.top_p = a->top_p; p.min_p = a->min_p; p.top_k = a->top_k;
  p.temperature1 = a->temperature_all; p.top_p1 = a->top_p_all; p.min_p1 = a->min_p_all; p.top_k1 = a->top_k_all;
  p.tokens = a->tokens; p.logprobs = a->logprobs;
  p.vocab = a->vocab;
  p.vectors = ((reinterpret_cast<uintptr_t>(a->logits) | (uintptr_t)(a->row_stride * (int64_t)elt_size(a->dtype))) & 15) == 0;
  LRQK_DISPATCH_DTYPE(a->dtype, T, return launch_sample<T>(p, a->rows, as_stream(stream)));
}
