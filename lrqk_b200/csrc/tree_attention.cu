// Attention of a tree of drafted tokens over a cache:  out_i = sum_j softmax_j(scale q_i . k_j) v_j  with j over the
// filled rows of the cache and the drafted nodes that node i sees.
//
// This file: the entry points, the fp32 kernel and the combine kernel.  (bf16 runs on the tensor cores,
// tree_attention_tc.cu.)  One pass over the keys with a running maximum and sum; scores, weights and sums in fp32.
//
// The fp32 kernel keeps to fp32 multiply-adds (tf32 would cost three digits), packed two to an instruction.  A CTA holds 64
// query rows and walks 32-key tiles: scores from 4 x 2 register tiles, weights through shared memory, 4 rows x head_dim/16
// columns of the result in registers, the next tile's keys and values on their way in registers meanwhile.  75 KiB of
// shared memory: two CTAs an SM (64-key tiles took 115 KiB, one CTA and twice the time).  33 nodes of 8 heads over 4096 rows
// of 2 cache heads: 38 us for 0.5 GFLOP.  Bound: waits for the shared-memory reads of the register tiles (the schedulers
// issue in a third of the cycles) and the few tiles a CTA gets there.
#include "tree_plan.cuh"

namespace lrqk {
namespace tree {
namespace {

constexpr int kRows = 64, kKeys = 32, kThreads = 256;

// Two fp32 multiply-adds in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  unsigned long long d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(*reinterpret_cast<unsigned long long *>(&a)), "l"(*reinterpret_cast<unsigned long long *>(&b)),
      "l"(*reinterpret_cast<unsigned long long *>(&c)));
  return *reinterpret_cast<float2 *>(&d);
}

template <int D> struct SimtShared {
  float q[kRows][D], k[kKeys][D + 4], v[kKeys][D], w[kRows][kKeys + 4];
};

template <int D>
__global__ void __launch_bounds__(kThreads, 2) tree_simt_kernel(const __grid_constant__ Params p) {
  pdl_launch_dependents();
  pdl_wait();
  extern __shared__ __align__(16) unsigned char smem_raw[];
  SimtShared<D> &sm = *reinterpret_cast<SimtShared<D> *>(smem_raw);
  using T = float;
  constexpr int VE = Elt<T>::kPerVec, DC = D / 64;      // columns of a thread: DC runs of four
  const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
  const int group = blockIdx.x / p.row_blocks, block = blockIdx.x % p.row_blocks;
  const Cut cut(p, count_tiles(p, 0).total);
  const int x0 = cut.start(group), x1 = cut.start(group + 1);
  int seq = 0, base = 0;
  if (x0 < x1) find_sequence(p, x0, seq, base);
  const int row0 = block * kRows, n_rows = min(kRows, p.rows - row0), per_head = p.q_heads / p.cache_heads;
  const bool works = ty * 4 < n_rows;                   // rows of this thread exist

  for (Walk w(p, x0, x1, seq, base); w.valid(); w.next(p)) {
    __syncthreads();
    for (int i = tid; i < kRows * (D / VE); i += kThreads) {
      const int r = i / (D / VE), c = i % (D / VE) * VE;
      float f[VE] = {};
      if (r < n_rows) {
        const int g = group_row(p, row0 + r), t = row0 + r - g * p.nodes;
        Elt<T>::unpack(ld16(static_cast<const T *>(p.q) + w.b * p.q_stride[0] + (int64_t)(w.head * per_head + g) * p.q_stride[1] + t * p.q_stride[2] + c), f);
      }
#pragma unroll
      for (int j = 0; j < VE; ++j) sm.q[r][c + j] = f[j];
    }
    float top[4], sum[4];
    float2 acc[4][2 * DC];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      top[i] = -INFINITY;
      sum[i] = 0.0f;
#pragma unroll
      for (int c = 0; c < 2 * DC; ++c) acc[i][c] = make_float2(0.0f, 0.0f);
    }
    const int tree_head = w.head / (p.cache_heads / p.tree_heads);
    // a tile's keys and values, into registers (rows behind the filled ones are never read: they may hold anything)
    constexpr int kLoads = kKeys * (D / VE) / kThreads;
    float4 nk[kLoads], nv[kLoads];
    const auto fetch = [&](int tile) {
      const bool drafted = tile >= w.ctiles;
      const int first = (drafted ? tile - w.ctiles : tile) * kKeys;
      const int n_keys = min(kKeys, (drafted ? p.nodes : w.len) - first);
      const T *gk = drafted ? static_cast<const T *>(p.tree_k) + w.b * p.tk_stride[0] + tree_head * p.tk_stride[1]
                            : static_cast<const T *>(p.cache_k) + w.b * p.ck_stride[0] + w.head * p.ck_stride[1];
      const T *gv = drafted ? static_cast<const T *>(p.tree_v) + w.b * p.tv_stride[0] + tree_head * p.tv_stride[1]
                            : static_cast<const T *>(p.cache_v) + w.b * p.cv_stride[0] + w.head * p.cv_stride[1];
      const int64_t sk = drafted ? p.tk_stride[2] : p.ck_stride[2], sv = drafted ? p.tv_stride[2] : p.cv_stride[2];
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int r = (tid + i * kThreads) / (D / VE), c = (tid + i * kThreads) % (D / VE) * VE;
        nk[i] = nv[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (r < n_keys) {
          nk[i] = *reinterpret_cast<const float4 *>(gk + (int64_t)(first + r) * sk + c);
          nv[i] = *reinterpret_cast<const float4 *>(gv + (int64_t)(first + r) * sv + c);
        }
      }
    };
    fetch(w.t0);
    for (int tile = w.t0; tile < w.t1; ++tile) {
      const bool drafted = tile >= w.ctiles;
      const int first = (drafted ? tile - w.ctiles : tile) * kKeys;
      const int n_keys = min(kKeys, (drafted ? p.nodes : w.len) - first);
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int r = (tid + i * kThreads) / (D / VE), c = (tid + i * kThreads) % (D / VE) * VE;
        *reinterpret_cast<float4 *>(&sm.k[r][c]) = nk[i];
        *reinterpret_cast<float4 *>(&sm.v[r][c]) = nv[i];
      }
      __syncthreads();
      if (tile + 1 < w.t1) fetch(tile + 1);
      if (works) {                                      // whole half-warps: a row's 16 threads stay together
        float2 s2[4][2] = {};                           // sums over even and odd columns
#pragma unroll 4
        for (int c = 0; c < D; c += 4) {
          float4 a[4], b[2];
#pragma unroll
          for (int i = 0; i < 4; ++i) a[i] = *reinterpret_cast<const float4 *>(&sm.q[ty * 4 + i][c]);
#pragma unroll
          for (int j = 0; j < 2; ++j) b[j] = *reinterpret_cast<const float4 *>(&sm.k[tx + 16 * j][c]);
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
              s2[i][j] = fma2(make_float2(a[i].x, a[i].y), make_float2(b[j].x, b[j].y),
                              fma2(make_float2(a[i].z, a[i].w), make_float2(b[j].z, b[j].w), s2[i][j]));
        }
        const unsigned half = (tid & 16) ? 0xFFFF0000u : 0x0000FFFFu;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = row0 + ty * 4 + i, node = r - group_row(p, r) * p.nodes;
          float m = top[i], s[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int key = tx + 16 * j;
            const bool seen = key < n_keys && r < p.rows && (!drafted || sees(p, w.b, node, first + key));
            s[j] = seen ? (s2[i][j].x + s2[i][j].y) * p.scale_log2 : -INFINITY;
            m = fmaxf(m, s[j]);
          }
#pragma unroll
          for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(half, m, o));
          const float at = m == -INFINITY ? 0.0f : m, fade = exp2f(top[i] - at);   // a row that has seen nothing yet fades nothing
          top[i] = m;
          float add = 0.0f;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float e = exp2f(s[j] - at);
            sm.w[ty * 4 + i][tx + 16 * j] = e;
            add += e;
          }
#pragma unroll
          for (int o = 8; o > 0; o >>= 1) add += __shfl_xor_sync(half, add, o);
          sum[i] = sum[i] * fade + add;
#pragma unroll
          for (int c = 0; c < 2 * DC; ++c) acc[i][c] = make_float2(acc[i][c].x * fade, acc[i][c].y * fade);
        }
        __syncwarp(half);
        // (rows of the tile behind the filled ones are zeros, their weights too)
#pragma unroll 2
        for (int key = 0; key < kKeys; key += 4) {
          float4 e4[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) e4[i] = *reinterpret_cast<const float4 *>(&sm.w[ty * 4 + i][key]);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            float4 v[DC];
#pragma unroll
            for (int c = 0; c < DC; ++c) v[c] = *reinterpret_cast<const float4 *>(&sm.v[key + k][tx * 4 + 64 * c]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float e = k == 0 ? e4[i].x : k == 1 ? e4[i].y : k == 2 ? e4[i].z : e4[i].w;
              if (drafted && e == 0.0f) continue;       // a node that the row does not see adds nothing, whatever it holds
#pragma unroll
              for (int c = 0; c < DC; ++c) {
                acc[i][2 * c] = fma2(make_float2(e, e), make_float2(v[c].x, v[c].y), acc[i][2 * c]);
                acc[i][2 * c + 1] = fma2(make_float2(e, e), make_float2(v[c].z, v[c].w), acc[i][2 * c + 1]);
              }
            }
          }
        }
      }
    }
    if (!works) continue;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = row0 + ty * 4 + i;
      if (r >= p.rows) continue;
      if (w.whole()) {
        const int g = group_row(p, r), t = r - g * p.nodes;
        const int64_t at = ((int64_t)w.b * p.q_heads + w.head * per_head + g) * p.nodes + t;
        const float inv = sum[i] == 0.0f ? 0.0f : 1.0f / sum[i];
        T *dst = static_cast<T *>(p.out) + at * D;
#pragma unroll
        for (int c = 0; c < DC; ++c)
          *reinterpret_cast<float4 *>(dst + tx * 4 + 64 * c) = make_float4(acc[i][2 * c].x * inv, acc[i][2 * c].y * inv, acc[i][2 * c + 1].x * inv, acc[i][2 * c + 1].y * inv);
        if (p.lse && tx == 0) p.lse[at] = sum[i] == 0.0f ? -INFINITY : (top[i] + log2f(sum[i])) * 0.6931471805599453f;
      } else {
        const int64_t at = w.slot(p, group, block) * p.rows_per_block + (r - row0);
#pragma unroll
        for (int c = 0; c < DC; ++c)
          *reinterpret_cast<float4 *>(p.part + at * D + tx * 4 + 64 * c) = make_float4(acc[i][2 * c].x, acc[i][2 * c].y, acc[i][2 * c + 1].x, acc[i][2 * c + 1].y);
        if (tx == 0) p.part_ml[at] = make_float2(top[i], sum[i]);
      }
    }
  }
}

// One to eight warps (WARPS) per query row of a unit that was cut: each folds every WARPS-th of the row's partials, in the order
// of the runs, the first folds theirs.
template <typename T, int D, int WARPS>
__global__ void __launch_bounds__(256) tree_combine_kernel(const __grid_constant__ Params p) {
  constexpr int E = D / 32;                             // columns of a lane
  __shared__ float rows[8][D], row_top[8], row_sum[8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = warp % WARPS;
  const int row = blockIdx.x * (8 / WARPS) + warp / WARPS;   // (batch * q_heads * nodes is below 2^31)
  const bool exists = row < p.batch * p.q_heads * p.nodes;
  const int t = row % p.nodes, h = row / p.nodes % p.q_heads, b = row / p.nodes / p.q_heads;
  const int32_t broken = *reinterpret_cast<volatile int32_t *>(p.status);
  const Count n = count_tiles(p, b);
  T *dst = static_cast<T *>(p.out) + (int64_t)row * D + lane * E;
  const int per_head = p.q_heads / p.cache_heads, head = h / per_head;
  const int u0 = n.before + head * unit_span(p, n.ctiles), u1 = u0 + n.ctiles + p.tree_tiles;
  const Cut cut(p, n.total);
  const int g0 = exists ? cut.of(u0) : 0, g1 = exists ? cut.of(u1 - 1) : 0;
  const bool folds = exists && !broken && g0 != g1;     // (a unit that one run holds is written already)
  float top = -INFINITY, sum = 0.0f, acc[E] = {};
  if (folds) {
    const int r = (h - head * per_head) * p.nodes + t, block = r / p.rows_per_block, at = r % p.rows_per_block;
    for (int first = g0 + part; first <= g1; first += 32 * WARPS) {
      // a lane holds one run's maximum and sum (every run from the first to the last holds tiles of the unit)
      const int g = first + lane * WARPS;
      int64_t slot = 0;
      float2 ml = make_float2(-INFINITY, 0.0f);
      if (g <= g1) {
        slot = (((int64_t)g * 2 + (cut.start(g) >= u0 ? 0 : 1)) * p.row_blocks + block) * p.rows_per_block + at;
        ml = p.part_ml[slot];
      }
      float m = ml.x;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
      m = fmaxf(m, top);
      const float ref = m == -INFINITY ? 0.0f : m, fade = exp2f(top - ref), weight = exp2f(ml.x - ref);
      top = m;
      sum *= fade;
#pragma unroll
      for (int c = 0; c < E; ++c) acc[c] *= fade;
      const int runs = min(32, (g1 - first) / WARPS + 1);
      for (int i = 0; i < runs; i += 8) {               // eight runs' loads in flight
        float got[8][E], wi[8], si[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          wi[k] = __shfl_sync(0xFFFFFFFFu, weight, (i + k) & 31);
          si[k] = __shfl_sync(0xFFFFFFFFu, ml.y, (i + k) & 31);
          const int64_t at_k = __shfl_sync(0xFFFFFFFFu, slot, (i + k) & 31);
          if (i + k >= runs) si[k] = 0.0f;
          const float *src = p.part + at_k * D + lane * E;
#pragma unroll
          for (int c = 0; c < E; ++c) got[k][c] = si[k] != 0.0f ? src[c] : 0.0f;
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          if (si[k] == 0.0f) continue;                  // nothing seen there
          sum = fmaf(wi[k], si[k], sum);
#pragma unroll
          for (int c = 0; c < E; ++c) acc[c] = fmaf(wi[k], got[k][c], acc[c]);
        }
      }
    }
  }
  if (WARPS > 1) {
#pragma unroll
    for (int c = 0; c < E; ++c) rows[warp][lane * E + c] = acc[c];
    if (lane == 0) { row_top[warp] = top; row_sum[warp] = sum; }
    __syncthreads();
    if (part != 0) return;
    float m = top;
    for (int k = 1; k < WARPS; ++k) m = fmaxf(m, row_top[warp + k]);
    const float ref = m == -INFINITY ? 0.0f : m;
    sum = 0.0f;
#pragma unroll
    for (int c = 0; c < E; ++c) acc[c] = 0.0f;
    for (int k = 0; k < WARPS; ++k) {
      if (row_sum[warp + k] == 0.0f) continue;
      const float wk = exp2f(row_top[warp + k] - ref);
      sum = fmaf(wk, row_sum[warp + k], sum);
#pragma unroll
      for (int c = 0; c < E; ++c) acc[c] = fmaf(wk, rows[warp + k][lane * E + c], acc[c]);
    }
    top = m;
  }
  if (part != 0 || !exists) return;
  if (broken != 0) {                                    // a wait ran out: no row can be trusted
    for (int c = 0; c < E; ++c) dst[c] = Elt<T>::from_float(NAN);
    if (p.lse && lane == 0) p.lse[row] = NAN;
    return;
  }
  if (!folds) return;
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
  for (int c = 0; c < E; ++c) dst[c] = Elt<T>::from_float(acc[c] * inv);
  if (p.lse && lane == 0) p.lse[row] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
}

template <int D> int launch_simt(const Params &p, cudaStream_t stream) {
  static SmemOptIn opt_in;
  auto kern = tree_simt_kernel<D>;
  LRQK_CUDA_TRY(opt_in.ensure(kern, sizeof(SimtShared<D>)));
  LRQK_CUDA_TRY(launch_dependent(kern, dim3((unsigned)(p.groups * p.row_blocks)), dim3(kThreads), sizeof(SimtShared<D>), stream, 0, p));
  return LRQK_OK;
}

template <typename T, int D, int WARPS> int combine_with(const Params &p, cudaStream_t stream) {
  const int64_t rows = (int64_t)p.batch * p.q_heads * p.nodes;
  // A plain launch: as a dependent one its CTAs sat beside the last products and the pair took 2 us longer.
  tree_combine_kernel<T, D, WARPS><<<(unsigned)ceil_div64(rows, 8 / WARPS), 256, 0, stream>>>(p);
  LRQK_LAUNCH_CHECK();
  return LRQK_OK;
}

template <typename T, int D> int launch_combine(const Params &p, cudaStream_t stream) {
  // at most so many runs share a unit (where all units are alike): eight to a warp, whose loads it has in flight at once
  const int64_t units = (int64_t)p.batch * p.cache_heads, runs = p.groups / units + 2;
  if (runs <= 8) return combine_with<T, D, 1>(p, stream);
  if (runs <= 16) return combine_with<T, D, 2>(p, stream);
  if (runs <= 32) return combine_with<T, D, 4>(p, stream);
  return combine_with<T, D, 8>(p, stream);
}

// The split of these arguments (no device work).
int plan(const lrqk_tree_args *a, Params &p) {
  if (!a) return LRQK_EINVAL;
  if (a->dtype != LRQK_F32 && a->dtype != LRQK_BF16) return LRQK_EUNSUPPORTED;
  if (a->batch <= 0 || a->nodes <= 0 || a->q_heads <= 0 || a->cache_heads <= 0 || a->tree_heads <= 0 || a->capacity < 0) return LRQK_EINVAL;
  if (a->q_heads % a->cache_heads != 0 || a->cache_heads % a->tree_heads != 0) return LRQK_EINVAL;
  if (a->head_dim != 64 && a->head_dim != 128) return LRQK_EUNSUPPORTED;
  if (a->nodes > 256 || a->capacity >= (1ll << 31) - 256) return LRQK_EUNSUPPORTED;
  if ((int64_t)a->batch * a->q_heads * a->nodes >= (1ll << 31)) return LRQK_EUNSUPPORTED;
  p.batch = a->batch; p.nodes = a->nodes; p.q_heads = a->q_heads; p.cache_heads = a->cache_heads; p.tree_heads = a->tree_heads;
  p.head_dim = a->head_dim; p.capacity = (int32_t)a->capacity;
  p.rows = a->q_heads / a->cache_heads * a->nodes;
  p.per_node = 1.0f / (float)a->nodes;
  if ((int64_t)a->q_heads / a->cache_heads * a->nodes > 1 << 16) return LRQK_EUNSUPPORTED;
  // The row blocks of a unit walk the same keys at the same time, so those come from HBM once.
  if (a->dtype == LRQK_BF16) {
    plan_tc(p);
  } else {
    p.rows_per_block = kRows;
    p.tile_keys = kKeys;
    p.unit_cost = 1;
    p.row_blocks = (p.rows + p.rows_per_block - 1) / p.rows_per_block;
    p.groups = 2 * kNumSMs / p.row_blocks;   // two CTAs an SM
    if (p.groups < 1) return LRQK_EUNSUPPORTED;
  }
  p.tree_tiles = (p.nodes + p.tile_keys - 1) / p.tile_keys;
  if ((int64_t)p.batch * p.cache_heads * (ceil_div64(p.capacity, p.tile_keys) + p.tree_tiles + p.unit_cost) >= 1 << 30) return LRQK_EUNSUPPORTED;
  return LRQK_OK;
}

size_t workspace_bytes(const Params &p) {
  const size_t rows = (size_t)p.groups * 2 * p.row_blocks * p.rows_per_block;
  return rows * p.head_dim * sizeof(float) + rows * sizeof(float2) + sizeof(int32_t);   // partials; a status word
}

}  // namespace
}  // namespace tree
}  // namespace lrqk

extern "C" {

size_t lrqk_tree_attention_workspace_bytes(const lrqk_tree_args *a) {
  lrqk::tree::Params p = {};
  return lrqk::tree::plan(a, p) == LRQK_OK ? lrqk::tree::workspace_bytes(p) : 0;
}

int lrqk_tree_attention(const lrqk_tree_args *a, void *workspace, lrqk_stream_t stream) {
  using namespace lrqk;
  int rc = check_device();
  if (rc != LRQK_OK) return rc;
  tree::Params p = {};
  rc = tree::plan(a, p);
  if (rc != LRQK_OK) return rc;
  if (!a->q || !a->tree_k || !a->tree_v || !a->out || !workspace) return LRQK_EINVAL;
  if (a->capacity > 0 && (!a->cache_k || !a->cache_v)) return LRQK_EINVAL;
  if (!(a->scale > 0.0f) || a->scale > 3.0e38f) return LRQK_EINVAL;
  // 16-byte rows: what the kernels' loads need
  uintptr_t low = reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->tree_k) | reinterpret_cast<uintptr_t>(a->tree_v) |
                  reinterpret_cast<uintptr_t>(a->out) | reinterpret_cast<uintptr_t>(workspace);
  if (a->capacity > 0) low |= reinterpret_cast<uintptr_t>(a->cache_k) | reinterpret_cast<uintptr_t>(a->cache_v);
  // (a dimension with one entry has no stride that matters)
  const struct { const int64_t *from; int64_t *to; int32_t heads; int64_t rows; } tensors[5] = {
      {a->q_stride, p.q_stride, a->q_heads, a->nodes}, {a->cache_k_stride, p.ck_stride, a->cache_heads, a->capacity},
      {a->cache_v_stride, p.cv_stride, a->cache_heads, a->capacity}, {a->tree_k_stride, p.tk_stride, a->tree_heads, a->nodes},
      {a->tree_v_stride, p.tv_stride, a->tree_heads, a->nodes}};
  for (const auto &t : tensors) {
    if (t.rows == 0) continue;
    t.to[0] = a->batch > 1 ? t.from[0] : 0;
    t.to[1] = t.heads > 1 ? t.from[1] : 0;
    t.to[2] = t.rows > 1 ? t.from[2] : 0;
    if (t.to[0] < 0 || t.to[1] < 0 || t.to[2] < 0) return LRQK_EINVAL;
    if (t.rows > 1 && t.to[2] == 0) return LRQK_EINVAL;   // (a tensor copy cannot repeat one row)
    low |= (uintptr_t)((t.to[0] | t.to[1] | t.to[2]) * (int64_t)elt_size(a->dtype));
  }
  if (low & 15 || (reinterpret_cast<uintptr_t>(a->out) | reinterpret_cast<uintptr_t>(workspace)) & 31) return LRQK_EUNSUPPORTED;
  p.q = a->q; p.cache_k = a->cache_k; p.cache_v = a->cache_v; p.tree_k = a->tree_k; p.tree_v = a->tree_v;
  p.lens = a->cache_lens; p.mask = a->mask; p.mask_stride = a->mask_stride;
  p.out = a->out; p.lse = a->lse; p.status = a->status;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  p.part = static_cast<float *>(workspace);
  p.part_ml = reinterpret_cast<float2 *>(p.part + (size_t)p.groups * 2 * p.row_blocks * p.rows_per_block * p.head_dim);
  const cudaStream_t s = as_stream(stream);
  if (!p.status) {   // the call's own word: the combine kernel has to know of a wait that ran out, whoever else looks
    p.status = reinterpret_cast<int32_t *>(static_cast<unsigned char *>(workspace) + tree::workspace_bytes(p) - sizeof(int32_t));
    LRQK_CUDA_TRY(cudaMemsetAsync(p.status, 0, sizeof(int32_t), s));
  }
  if (a->dtype == LRQK_BF16) rc = tree::launch_tc(p, s);
  else rc = a->head_dim == 64 ? tree::launch_simt<64>(p, s) : tree::launch_simt<128>(p, s);
  if (rc != LRQK_OK) return rc;
  LRQK_DISPATCH_DTYPE(a->dtype, T, return a->head_dim == 64 ? tree::launch_combine<T, 64>(p, s) : tree::launch_combine<T, 128>(p, s));
}

}  // extern "C"
