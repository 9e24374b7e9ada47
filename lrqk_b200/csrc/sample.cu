// Choice of a token from logits: temperature, top-k, top-p, min-p and a given random number, one cluster per row.
//
//   w_i = exp((l_i - max) / T);  keep the k largest logits (equal ones: lowest index first);  of those, in descending
//   order, keep a token while the mass strictly before it is below p times their sum;  of those keep w_i >= m;  the token is
//   the first kept one, in index order, whose cumulative mass exceeds u times the kept sum.  T = 0: the first maximum.
//
// Every one of these decisions is a comparison of sums, and a sum in fp32 decides differently from one in another order as
// soon as a number falls near a border.  So weights are 45-bit whole numbers, W = round(2^44 w), from an exponential in
// double (own: Taylor to the fifth order around 64 table values of 2^x, Tang's table method): whole-number sums have no
// order, are the same for any cluster size, and agree with 64-bit floating sums to 2^-34 of the mass.
//
// A row's logits are read once, into the shared memory of the cluster's CTAs (1, 2, 4 or 8: enough SMs for few rows,
// enough memory for large vocabularies).  Top-k and top-p look for the key (an order-preserving integer of a logit) at
// which a running count or mass crosses its target: histograms of counts or of the weights' three 15-bit limbs (the
// sums of 2^17 of them fit 32 bits, so shared-memory atomics stay 32-bit), merged over the cluster in distributed shared
// memory; the first level bins by distance from the maximum, which spreads the crowded exponents, the next ones by key
// until one key is left.  Positions in index order (ties at a border, the final choice) come from per-warp sums of
// contiguous chunks and a second look at one chunk.
//
// Bound: latency of the cluster barriers for few rows; fp64 and shared-memory atomics for many.
#include <cooperative_groups.h>

#include "common.cuh"

namespace lrqk {
namespace {

namespace cg = cooperative_groups;

constexpr int kSampThreads = 1024, kSampWarps = 32, kSampBins = 512, kSampMaxCluster = 8;
constexpr int kFracBits = 44;                          // of a weight
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
  double table[64];
  unsigned long long merged[kSampBins], best[kSampMaxCluster], xsum[2][kSampMaxCluster], wsum[kSampWarps], pick_above, pick_in, pick_total;
  uint32_t hist[3][kSampBins], low[kSampMaxCluster], wlow[kSampWarps], tie_index, pick_bin;
};

template <typename T> struct SampKey;                  // order-preserving keys and back
template <> struct SampKey<float> {
  static constexpr uint32_t kTop = 0xFFFFFFFFu;
  __device__ static __forceinline__ uint32_t of(float f) { return order_key(f); }
  __device__ static __forceinline__ float value(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k); }
};
template <> struct SampKey<__nv_bfloat16> {
  static constexpr uint32_t kTop = 0xFFFFu;
  __device__ static __forceinline__ uint32_t of(float f) { return order_key(f) >> 16; }
  __device__ static __forceinline__ float value(uint32_t k) { return __uint_as_float((k & 0x8000u) ? (k ^ 0x8000u) << 16 : ~k << 16); }
};

struct Cut { uint32_t key, index; };                   // kept: larger keys, and this key up to this index

template <typename T> struct Sampler {
  static constexpr int VE = Elt<T>::kPerVec, STEP = 32 * VE;
  const SampleParams &p;
  SampleShared &sm;
  T *vals;
  cg::cluster_group cluster;
  int rank, csize, warp, lane, flip;
  float top;                                           // the row's maximum
  double top_d, c64;                                   // 64 log2(e) / T

  __device__ Sampler(const SampleParams &params, SampleShared &shared, T *values)
      : p(params), sm(shared), vals(values), cluster(cg::this_cluster()), rank((int)cluster.block_rank()),
        csize((int)cluster.num_blocks()), warp(threadIdx.x >> 5), lane(threadIdx.x & 31), flip(0) {}

  __device__ __forceinline__ uint32_t index_of(int at) const { return (uint32_t)(rank * kSampWarps * p.chunk + at); }

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

  // a logit that can carry mass: with a maximum of +inf only the infinite ones do
  __device__ __forceinline__ bool candidate(float f) const { return f > -INFINITY && (top < INFINITY || f == top); }

  // round(2^44 exp((f - top) / T)), f <= top
  __device__ __forceinline__ unsigned long long weight(float f) const {
    if (f == top) return 1ull << kFracBits;
    const double y = ((double)f - top_d) * c64;        // 64ths of an octave
    if (!(y > -64.0 * (kFracBits + 1))) return 0ull;
    const double magic = 6755399441055744.0;           // 1.5 * 2^52: the sum's low bits are the nearest whole number
    const double n = y + magic;
    const int k = (int)(unsigned)__double_as_longlong(n);
    const double z = (y - (n - magic)) * 0.010830424696249145;   // ln(2) / 64; |z| < 0.0055, next term of the series below 2^-54
    const double e = fma(z, fma(z, fma(z, fma(z, fma(z, 1.0 / 120.0, 1.0 / 24.0), 1.0 / 6.0), 0.5), 1.0), 1.0) * sm.table[k & 63];
    const double scaled = __longlong_as_double(__double_as_longlong(e) + ((long long)((k >> 6) + kFracBits) << 52));
    return (unsigned long long)(__double_as_longlong(scaled + 4503599627370496.0) - __double_as_longlong(4503599627370496.0));
  }

  __device__ __forceinline__ bool inside(const Cut &c, float f, int at) const {
    const uint32_t k = SampKey<T>::of(f);
    return k > c.key || (k == c.key && index_of(at) <= c.index);
  }

  // Merge the histograms of the cluster and find the bin in which the running sum from bin 0 reaches `target`
  // (target 0: `target_of` makes it from the total).  MASS: three limbs; else counts in hist[0].
  template <bool MASS, typename F> __device__ void pick(F target_of) {
    cluster.sync();
    for (int i = threadIdx.x; i < kSampBins / csize; i += kSampThreads) {
      const int bin = rank * (kSampBins / csize) + i;
      unsigned long long s = 0;
      for (int c = 0; c < csize; ++c) {
        const uint32_t *h = cluster.map_shared_rank(&sm.hist[0][0], c);
        s += h[bin];
        if (MASS) s += ((unsigned long long)h[kSampBins + bin] << 15) + ((unsigned long long)h[2 * kSampBins + bin] << 30);
      }
      for (int c = 0; c < csize; ++c) cluster.map_shared_rank(sm.merged, c)[bin] = s;
    }
    cluster.sync();
    if (warp == 0) {
      constexpr int PER = kSampBins / 32;
      unsigned long long mine = 0;
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
    for (int i = threadIdx.x; i < 3 * kSampBins; i += kSampThreads) (&sm.hist[0][0])[i] = 0u;
    __syncthreads();
  }

  // Cut the tokens inside `cut` to those from the largest down to where the count (MASS: the mass) reaches its target.
  // lowest: key of the smallest candidate.
  template <bool MASS> __device__ void narrow(Cut &cut, uint32_t lowest, unsigned long long count, double share) {
    uint32_t khi = SampKey<T>::of(top), klo = max(lowest, cut.key);
    unsigned long long target = count, above = 0, in = 0;
    // level 0: bins by distance from the maximum.  (Halved, so that the range of any two floats is finite.)
    const float half_top = 0.5f * top, range = half_top - 0.5f * SampKey<T>::value(klo);
    const float per = (float)kSampBins / range;
    const auto bin0 = [&](float f) { return f == top ? 0 : min(kSampBins - 1, max(0, (int)((half_top - 0.5f * f) * per))); };
    clear();
    each([&](float f, int at) {
      if (candidate(f) && inside(cut, f, at)) {
        const unsigned long long w = MASS ? weight(f) : 1ull;
        if (w) add<MASS>(bin0(f), w);
      }
    });
    const auto first_target = [&](unsigned long long total) {
      if (!MASS) return min(count, total);               // fewer candidates than asked for: all of them
      const double t = ceil(share * (double)total);    // before < share * total, for whole numbers before
      return t < 1.0 ? 1ull : min(total, (unsigned long long)t);
    };
    pick<MASS>(first_target);
    const int b0 = sm.pick_bin;
    above = sm.pick_above;
    in = sm.pick_in;
    target = first_target(sm.pick_total);
    if (khi != klo) {
      // keys that can lie in that bin (a little wider: the test itself is bin0)
      const float slack = (fabsf(top) + 2.0f * range) * 0x1p-20f + 1e-37f, step = 2.0f * range / kSampBins;
      khi = min(khi, SampKey<T>::of(fminf(top, top - step * (float)b0 + slack)));
      if (b0 < kSampBins - 1) klo = max(klo, SampKey<T>::of(top - step * (float)(b0 + 1) - slack));
      if (klo > khi) klo = khi;
    }
    while (khi != klo) {
      const int shift = max(0, 32 - __clz((int)(khi - klo)) - 9);        // 512 bins of 2^shift keys
      clear();
      each([&](float f, int at) {
        if (!candidate(f) || bin0(f) != b0) return;
        const uint32_t k = SampKey<T>::of(f);
        if (k > khi || k < klo || !inside(cut, f, at)) return;
        const unsigned long long w = MASS ? weight(f) : 1ull;
        if (w) add<MASS>((khi - k) >> shift, w);
      });
      pick<MASS>([&](unsigned long long) { return target - above; });
      above += sm.pick_above;
      in = sm.pick_in;
      khi -= sm.pick_bin << shift;
      klo = shift == 0 || khi - klo < (1u << shift) ? (shift == 0 ? khi : klo) : khi - (1u << shift) + 1u;
      __syncthreads();
    }
    const unsigned long long each_w = MASS ? weight(SampKey<T>::value(khi)) : 1ull;
    const unsigned long long ties = each_w ? in / each_w : 0ull, need = each_w ? (target - above + each_w - 1) / each_w : 1ull;
    Cut got{khi, khi == cut.key ? cut.index : 0xFFFFFFFFu};
    if (need < ties) {
      // the need-th of the equal keys, in index order
      const Cut old = cut;
      locate([&](float f, int at) -> unsigned long long { return SampKey<T>::of(f) == khi && candidate(f) && inside(old, f, at) ? 1ull : 0ull; },
             [&](unsigned long long) { return need - 1; },
             [&](uint32_t index, float, unsigned long long) {
               for (int c = 0; c < csize; ++c) *cluster.map_shared_rank(&sm.tie_index, c) = index;
             });
      cluster.sync();
      got.index = sm.tie_index;
    }
    cut = got;
  }

  // The first token, in index order, at which the cumulative weight exceeds target_of(total): found(index, value, total)
  // is called by one thread of the cluster.
  template <typename W, typename G, typename F> __device__ void locate(W weigh, G target_of, F found) {
    unsigned long long mine = 0;
    each([&](float f, int at) { mine += weigh(f, at); });
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
__global__ void __launch_bounds__(kSampThreads, 1) sample_kernel(const __grid_constant__ SampleParams p) {
  pdl_launch_dependents();
  extern __shared__ __align__(16) unsigned char smem_raw[];
  __shared__ SampleShared sm;
  Sampler<T> s(p, sm, reinterpret_cast<T *>(smem_raw));
  const int row = blockIdx.x / s.csize;
  constexpr int VE = Sampler<T>::VE, STEP = Sampler<T>::STEP;
  if (threadIdx.x < 64) sm.table[threadIdx.x] = exp2((double)threadIdx.x * (1.0 / 64.0));
  pdl_wait();

  // ---- the row's slice into shared memory; NaN counts as -inf, and so does what lies behind the vocabulary -----------
  const T *src = static_cast<const T *>(p.logits) + (int64_t)row * p.row_stride;
  const int base = s.warp * p.chunk;
  unsigned long long best = 0;
  uint32_t low = SampKey<T>::kTop;
  const auto note = [&](float f, uint32_t index) {
    if (f > -INFINITY) {
      const uint32_t k = SampKey<T>::of(f);
      best = max(best, ((unsigned long long)k << 32) | (0xFFFFFFFFu - index));
      low = min(low, k);
    }
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
      for (int j = 0; j < VE; ++j) {
        if (f[j] != f[j]) f[j] = -INFINITY;
        s.vals[at + j] = Elt<T>::from_float(f[j]);
        note(f[j], index + j);
      }
    }
  } else {
#pragma unroll 4
    for (int i = 0; i < p.chunk; i += 32) {
      const int at = base + i + s.lane;
      const uint32_t index = s.index_of(at);
      float f = index < (uint32_t)p.vocab ? Elt<T>::to_float(src[index]) : -INFINITY;
      if (f != f) f = -INFINITY;
      s.vals[at] = Elt<T>::from_float(f);
      note(f, index);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    best = max(best, __shfl_xor_sync(0xFFFFFFFFu, best, o));
    low = min(low, __shfl_xor_sync(0xFFFFFFFFu, low, o));
  }
  if (s.lane == 0) { sm.wsum[s.warp] = best; sm.wlow[s.warp] = low; }
  s.cluster.sync();                                    // every CTA of the cluster runs: its shared memory can be written
  best = sm.wsum[s.lane];
  low = sm.wlow[s.lane];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    best = max(best, __shfl_xor_sync(0xFFFFFFFFu, best, o));
    low = min(low, __shfl_xor_sync(0xFFFFFFFFu, low, o));
  }
  if (threadIdx.x < (unsigned)s.csize) {
    *s.cluster.map_shared_rank(&sm.best[s.rank], threadIdx.x) = best;
    *s.cluster.map_shared_rank(&sm.low[s.rank], threadIdx.x) = low;
  }
  s.cluster.sync();
  for (int c = 0; c < s.csize; ++c) { best = max(best, sm.best[c]); low = min(low, sm.low[c]); }

  const float t = p.temperature ? p.temperature[row] : p.temperature1;
  const bool first = s.rank == 0 && threadIdx.x == 0;
  if (best == 0) {                                     // nothing but -inf and NaN: no token
    if (first) { p.tokens[row] = -1; if (p.logprobs) p.logprobs[row] = NAN; }
  } else if (!(t > 0.0f)) {
    if (first) { p.tokens[row] = 0xFFFFFFFFu - (uint32_t)best; if (p.logprobs) p.logprobs[row] = 0.0f; }
  } else {
    s.top = SampKey<T>::value((uint32_t)(best >> 32));
    s.top_d = (double)s.top;
    s.c64 = 92.33248261893193 / (double)t;             // 64 log2(e) / T
    if (s.top == INFINITY) low = (uint32_t)(best >> 32);
    const int k = p.top_k ? p.top_k[row] : p.top_k1;
    const float q = p.top_p ? p.top_p[row] : p.top_p1, m = p.min_p ? p.min_p[row] : p.min_p1, u = p.u[row];
    Cut cut{0u, 0xFFFFFFFFu};
    if (k > 0 && k < p.vocab) s.template narrow<false>(cut, low, (unsigned long long)k, 0.0);
    if (q < 1.0f) s.template narrow<true>(cut, low, 0ull, (double)q);
    const unsigned long long floor_w = m > 0.0f ? (unsigned long long)__double2ull_rn(fmin((double)m, 1.0) * 17592186044416.0) : 0ull;
    s.locate(
        [&](float f, int at) -> unsigned long long {
          if (!s.candidate(f) || !s.inside(cut, f, at)) return 0ull;
          const unsigned long long w = s.weight(f);
          return w >= floor_w ? w : 0ull;
        },
        [&](unsigned long long total) {
          const double x = floor((double)u * (double)total);
          return x > 0.0 ? min(total - 1, (unsigned long long)x) : 0ull;
        },
        [&](uint32_t index, float f, unsigned long long total) {
          p.tokens[row] = index;
          const double y = f == s.top ? 0.0 : ((double)f - s.top_d) / (double)t;
          if (p.logprobs) p.logprobs[row] = (float)(y - log((double)total * 0x1p-44));
        });
  }
  s.cluster.sync();                                    // no CTA leaves while a peer may still write to it
}

template <typename T> int launch_sample(SampleParams &p, int rows, cudaStream_t stream) {
  // Few rows: 8 CTAs each, for latency; more: fewer, as long as a slice fits.  (One row of 128256 bf16 logits, top-k 50 and
  // top-p 0.9, by cluster size: see the note at the launch.)
  constexpr int step = 32 * Elt<T>::kPerVec * kSampWarps;       // a slice is a whole number of these
  int csize = 1;
  const auto slice = [&](int c) { return ceil_div64(ceil_div64(p.vocab, c), step) * step; };
  while (csize < kSampMaxCluster && (slice(csize) * (int64_t)sizeof(T) > (int64_t)kSampSliceBytes ||
                                     (rows * csize * 2 <= kNumSMs && slice(csize) > step)))
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
