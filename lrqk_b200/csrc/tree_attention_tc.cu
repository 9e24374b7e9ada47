// Tree attention on the tensor cores: bf16, head_dim 64 or 128.  (Formula, split and partials: tree_attention.cu,
// tree_plan.cuh.)
//
// A CTA walks its run of 128-key tiles with one or two blocks of 128 query rows (MT).  Per tile and row block
//     S = Q K^T   tcgen05.mma M128 N128, K from a TMA tile (K-major), S in TMEM
//     P = 2^(S c - m)   four warps, a thread per row: no exchange between lanes for the maximum and the sum
//     O += P V    tcgen05.mma with P read from TMEM and V from its TMA tile (N = head_dim, MN-major), O in TMEM
// P enters the product as TWO bf16 parts, high and low, over the columns of S that it replaces: rounding it to one bf16
// would add as much error as the final rounding of the result; the second product hides behind the loads.
// The running maximum moves only when a row's maximum has grown by more than 2^8 (then O is read, scaled and written
// back by the row's thread); weights then stay below 2^8 and sums keep fp32's full precision.
//
// Warp 0 issues the copies (a ring of K and V tiles, 128-byte swizzle), warp 1 owns TMEM and issues the MMAs, warps 2.. are
// four softmax warps per row block.  With one row block S is double-buffered, with two they alternate: while one
// block's weights are formed, the other's products run.
//
// V rows behind a length may hold anything, and 0 * NaN is NaN: the softmax warps clear them in shared memory before the
// product.  In a drafted tile, values of V out of range are replaced by zeros and their nodes noted; a row that sees such
// a node takes the values themselves afterwards, the others never meet them.
//
// Every wait is bounded: one that runs out raises the status word, the roles stop issuing, TMEM is freed, and the combine
// kernel hands out NaN rows.
#include "tc_common.cuh"
#include "tree_plan.cuh"

namespace lrqk {
namespace tree {
namespace {

using namespace tc;

constexpr int kTileKeys = 128, kBlockRows = 128;
constexpr float kGrow = 8.0f;     // octaves a maximum may grow before O is rescaled

template <int D, int MT> struct Shape {
  static constexpr int kTileBytes = kTileKeys * D * 2;
  static constexpr int kHalfBytes = kTileKeys * 128;                 // 64 columns of a tile
  static constexpr int kQBytes = MT * kBlockRows * D * 2;
  static constexpr int kStages = (208 * 1024 - kQBytes) / kTileBytes > 8 ? 8 : (208 * 1024 - kQBytes) / kTileBytes;
  static constexpr int kThreads = 64 + 128 * MT;
  static constexpr int kBufs = MT == 1 ? 2 : 1;                      // S buffers of a row block
  static constexpr int kOCol = 256;                                  // S: columns 0..255, O: 256 + 128 * block
  static constexpr size_t kSmem = kQBytes + (size_t)kStages * kTileBytes + 1024;
};

struct Barriers {
  uint64_t full[8], empty[8], s_full[2], p_ready[2], o_done[2], q_full;
  uint32_t tmem, give_up, odd[2][4];        // odd: drafted rows of V with values out of range, 128 bits for each drafted tile
  int64_t x0, x1, base;
  int32_t seq;
};

__device__ __forceinline__ void tma_tile(const CUtensorMap *map, void *dst, uint64_t *bar, int c0, int row, int head, int seq) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
               ::"r"(saddr(dst)), "l"(map), "r"(saddr(bar)), "r"(c0), "r"(row), "r"(head), "r"(seq) : "memory");
}

// D[tmem] (+)= A[tmem, 16-bit pairs in 32-bit columns] * B[shared]
__device__ __forceinline__ void umma_bf16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(tmem_d), "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}

// 32 columns of this warp's lanes; the wait names the registers, so that no use can move ahead of it
__device__ __forceinline__ void load32(uint32_t taddr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      "\n\ttcgen05.wait::ld.sync.aligned;"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
        "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
        "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
        "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(taddr) : "memory");
}
__device__ __forceinline__ void store32(uint32_t taddr, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};"
      ::"r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
        "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]),
        "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]),
        "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31]),
        "r"(taddr) : "memory");
}
__device__ __forceinline__ void store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}

struct Maps { CUtensorMap ck, cv, tk, tv; };
struct Coord { int32_t ck_head, ck_seq, cv_head, cv_seq, tk_head, tk_seq, tv_head, tv_seq; };   // 0 where a dimension is broadcast

template <int D, int MT>
__global__ void __launch_bounds__(Shape<D, MT>::kThreads, 1)
tree_tc_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Params p, const __grid_constant__ Coord co) {
  using S = Shape<D, MT>;
  constexpr int HALVES = D / 64;
  pdl_launch_dependents();
  extern __shared__ unsigned char smem_raw[];
  __shared__ Barriers bar;
  unsigned char *stages = smem_raw + ((1024u - (saddr(smem_raw) & 1023u)) & 1023u);
  unsigned char *qs = stages + (size_t)S::kStages * S::kTileBytes;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int group = blockIdx.x / p.row_blocks, block = blockIdx.x % p.row_blocks;
  const int row0 = block * p.rows_per_block, n_rows = min(p.rows_per_block, p.rows - row0);

  if (tid == 0) {
    for (int i = 0; i < S::kStages; ++i) { mbar_init(&bar.full[i], 1); mbar_init(&bar.empty[i], 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(&bar.s_full[i], 1); mbar_init(&bar.p_ready[i], 128); mbar_init(&bar.o_done[i], 1); }
    mbar_init(&bar.q_full, 128 * MT);
    bar.give_up = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (tid < 8) bar.odd[tid >> 2][tid & 3] = 0;
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(saddr(&bar.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  pdl_wait();
  if (warp == 0) {
    int64_t before, total;
    count_tiles(p, 0, before, total);
    const int64_t x0 = group_start(p, total, group), x1 = group_start(p, total, group + 1);
    int seq = 0;
    int64_t base = 0;
    if (x0 < x1) find_sequence(p, x0, seq, base);
    if (lane == 0) { bar.x0 = x0; bar.x1 = x1; bar.base = base; bar.seq = seq; }
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = bar.tmem;
  volatile uint32_t *give_up = &bar.give_up;
  const auto quit = [&]() {
    *give_up = 1;
    if (p.status) atomicExch(p.status, (int32_t)LRQK_ETIMEOUT);
  };
  const int per_head = p.q_heads / p.cache_heads, share = p.cache_heads / p.tree_heads;
  Walk w(p, bar.x0, bar.x1, bar.seq, bar.base);

  if (warp == 0) {
    // ---- copies: K and V of every tile, in turn ------------------------------------------------------------------------
    if (lane == 0) {
      int i = 0;
      for (; w.valid() && !*give_up; w.next(p)) {
        const int tree_head = w.head / share;
        for (int t = w.t0; t < w.t1 && !*give_up; ++t) {
          const bool drafted = t >= w.ctiles;
          const int row = (drafted ? t - w.ctiles : t) * kTileKeys;
          for (int v = 0; v < 2; ++v, ++i) {
            const int s = i % S::kStages;
            if (i >= S::kStages && !wait_bounded(&bar.empty[s], (i / S::kStages - 1) & 1)) { quit(); break; }
            const CUtensorMap *m = drafted ? (v ? &maps.tv : &maps.tk) : (v ? &maps.cv : &maps.ck);
            const int head = drafted ? tree_head * (v ? co.tv_head : co.tk_head) : w.head * (v ? co.cv_head : co.ck_head);
            const int seq = w.b * (drafted ? (v ? co.tv_seq : co.tk_seq) : (v ? co.cv_seq : co.ck_seq));
            unsigned char *dst = stages + (size_t)s * S::kTileBytes;
            mbar_expect_tx(&bar.full[s], S::kTileBytes);
#pragma unroll
            for (int h = 0; h < HALVES; ++h) tma_tile(m, dst + h * S::kHalfBytes, &bar.full[s], h * 64, row, head, seq);
          }
        }
      }
    }
  } else if (warp == 1) {
    // ---- products ------------------------------------------------------------------------------------------------------
    if (lane == 0) {
      constexpr uint32_t kIdescS = umma_idesc_bf16_k(128, kTileKeys);
      constexpr uint32_t kIdescO = umma_idesc_bf16_k(128, D) | (1u << 16);       // B (the values) MN-major
      const uint32_t q_base = saddr(qs), stage_base = saddr(stages);
      const auto scores = [&](int i, int m, int buf) {
        const uint32_t kb = stage_base + (uint32_t)(i % S::kStages) * S::kTileBytes, qb = q_base + m * (kBlockRows * D * 2);
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          const uint32_t off = (ks >> 2) * S::kHalfBytes + (ks & 3) * 32;
          umma_bf16(tmem + buf * 128, umma_desc_k_sw128(qb + off, 1024), umma_desc_k_sw128(kb + off, 1024), kIdescS, ks > 0);
        }
        umma_commit(&bar.s_full[buf]);
      };
      const auto values = [&](int i, int m, int buf, bool fresh) {
        const uint32_t vb = stage_base + (uint32_t)(i % S::kStages) * S::kTileBytes;
#pragma unroll
        for (int ks = 0; ks < kTileKeys / 16; ++ks) {
          const uint64_t desc = umma_desc_mn_sw128(vb + ks * 2048, S::kHalfBytes, 1024);
          const uint32_t a = tmem + buf * 128 + (ks >> 1) * 32 + (ks & 1) * 8;   // high parts; low parts 16 columns on
          umma_bf16_ts(tmem + S::kOCol + m * 128, a, desc, kIdescO, !(fresh && ks == 0));
          umma_bf16_ts(tmem + S::kOCol + m * 128, a + 16, desc, kIdescO, 1);
        }
        umma_commit(&bar.o_done[m]);
      };
      const auto arrived = [&](int i) {
        if (wait_bounded(&bar.full[i % S::kStages], (i / S::kStages) & 1)) { fence_after(); return true; }
        quit();
        return false;
      };
      int i = 0, cnt = 0, seg = 0;         // ring index of the next tile's K, tiles done, segments done
      for (; w.valid() && !*give_up; w.next(p), ++seg) {
        const int n = w.t1 - w.t0;
        if (!wait_bounded(&bar.q_full, seg & 1)) { quit(); break; }
        fence_after();
        if (!arrived(i)) break;
        if constexpr (MT == 1) {
          scores(i, 0, cnt & 1);
          umma_commit(&bar.empty[i % S::kStages]);
          for (int t = 0; t < n; ++t, ++cnt, i += 2) {
            if (t + 1 < n) {
              if (!arrived(i + 2)) break;
              scores(i + 2, 0, (cnt + 1) & 1);
              umma_commit(&bar.empty[(i + 2) % S::kStages]);
            }
            if (!arrived(i + 1)) break;
            if (!wait_bounded(&bar.p_ready[cnt & 1], (cnt >> 1) & 1)) { quit(); break; }
            fence_after();
            values(i + 1, 0, cnt & 1, t == 0);
            umma_commit(&bar.empty[(i + 1) % S::kStages]);
          }
        } else {
          scores(i, 0, 0);
          scores(i, 1, 1);
          umma_commit(&bar.empty[i % S::kStages]);
          for (int t = 0; t < n; ++t, ++cnt, i += 2) {
            if (!arrived(i + 1)) break;
            bool ok = true;
#pragma unroll
            for (int m = 0; m < 2; ++m) {
              if (!wait_bounded(&bar.p_ready[m], cnt & 1)) { quit(); ok = false; break; }
              fence_after();
              values(i + 1, m, m, t == 0);
              if (m == 1) umma_commit(&bar.empty[(i + 1) % S::kStages]);
              if (t + 1 < n) {
                if (m == 0 && !arrived(i + 2)) { ok = false; break; }
                scores(i + 2, m, m);
                if (m == 1) umma_commit(&bar.empty[(i + 2) % S::kStages]);
              }
            }
            if (!ok) break;
          }
        }
      }
    }
  } else {
    // ---- softmax: a thread per query row ---------------------------------------------------------------------------------
    const int m = (warp - 2) >> 2;                       // row block of this warp
    const int quarter = warp & 3, r_in = quarter * 32 + lane, row = m * kBlockRows + r_in;   // TMEM lanes 32 * (warp % 4)..
    const uint32_t lane_base = tmem + ((uint32_t)(quarter * 32) << 16), o_base = lane_base + S::kOCol + m * 128;
    const int at_row = row0 + row, g = at_row / p.nodes, node = at_row % p.nodes;            // query head in the group, node
    const bool real = row < n_rows, warp_real = m * kBlockRows + quarter * 32 < n_rows;
    int cnt = 0, i = 0;
    for (; w.valid() && !*give_up; w.next(p)) {
      // the block's queries, into the K-major swizzled operand (rows that do not exist: zeros)
      {
        const __nv_bfloat16 *q = static_cast<const __nv_bfloat16 *>(p.q) + w.b * p.q_stride[0] + (int64_t)(w.head * per_head) * p.q_stride[1];
        unsigned char *dst = qs + m * (kBlockRows * D * 2);
        const int t128 = quarter * 32 + lane;
        for (int e = t128; e < kBlockRows * (D / 8); e += 128) {
          const int r = e / (D / 8), c = e % (D / 8), ar = row0 + m * kBlockRows + r;
          uint4 v = make_uint4(0, 0, 0, 0);
          if (m * kBlockRows + r < n_rows) v = ld16(q + (int64_t)(ar / p.nodes) * p.q_stride[1] + (int64_t)(ar % p.nodes) * p.q_stride[2] + c * 8);
          *reinterpret_cast<uint4 *>(dst + (c >> 3) * (kBlockRows * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = v;
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        mbar_arrive(&bar.q_full);
      }
      // which nodes of the segment's first drafted tile this row sees
      uint32_t seen[4] = {0, 0, 0, 0};
      int seen_tile = -1;
      const auto look = [&](int dt) {
        seen_tile = dt;
        const int first = dt * kTileKeys, n = min(kTileKeys, p.nodes - first);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t bits = 0;
          if (real)
            for (int j = 0; j < 32 && c * 32 + j < n; ++j) bits |= (sees(p, w.b, node, first + c * 32 + j) ? 1u : 0u) << j;
          seen[c] = bits;
        }
      };
      if (w.t1 > w.ctiles) look(max(w.t0 - w.ctiles, 0));
      float top = -INFINITY, sum = 0.0f;                 // maximum in use, in octaves; sum of weights
      for (int t = w.t0; t < w.t1; ++t, ++cnt, i += 2) {
        const int buf = MT == 1 ? (cnt & 1) : m;
        const uint32_t s_base = lane_base + buf * 128;
        const bool drafted = t >= w.ctiles;
        const int dt = t - w.ctiles, n_keys = min(kTileKeys, drafted ? p.nodes - dt * kTileKeys : w.len - t * kTileKeys);
        if (drafted && dt != seen_tile) look(dt);
        if (!wait_bounded(&bar.s_full[buf], MT == 1 ? (cnt >> 1) & 1 : cnt & 1)) { quit(); break; }
        fence_after();
        bool waited = t == w.t0;                         // for the products of the tile before
        if (warp_real) {
          const bool all = !drafted && n_keys == kTileKeys;
          uint32_t v[32];
          float big = -INFINITY;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            load32(s_base + c * 32, v);
            if (all) {
#pragma unroll
              for (int j = 0; j < 32; ++j) big = fmaxf(big, __uint_as_float(v[j]));
            } else {
              const uint32_t bits = drafted ? seen[c] : (n_keys >= c * 32 + 32 ? 0xFFFFFFFFu : n_keys > c * 32 ? (1u << (n_keys - c * 32)) - 1u : 0u);
#pragma unroll
              for (int j = 0; j < 32; ++j) big = fmaxf(big, (bits >> j) & 1u ? __uint_as_float(v[j]) : -INFINITY);
            }
          }
          const float now = big * p.scale_log2;
          const bool move = now > top + kGrow || (top == -INFINITY && now > -INFINITY);
          if (__any_sync(0xFFFFFFFFu, move)) {
            const float fade = move ? exp2_fast(top - now) : 1.0f;
            if (move) { sum *= fade; top = now; }
            if (!waited) {
              if (!wait_bounded(&bar.o_done[m], (cnt - 1) & 1)) { quit(); break; }
              fence_after();
              waited = true;
#pragma unroll
              for (int c = 0; c < D; c += 32) {
                load32(o_base + c, v);
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) * fade);
                store32(o_base + c, v);
              }
            }
          }
          const float minus = top == -INFINITY ? 0.0f : -top;
          float add0 = 0.0f, add1 = 0.0f;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            load32(s_base + c * 32, v);
            const uint32_t bits = all ? 0xFFFFFFFFu : drafted ? seen[c] : (n_keys >= c * 32 + 32 ? 0xFFFFFFFFu : n_keys > c * 32 ? (1u << (n_keys - c * 32)) - 1u : 0u);
            uint32_t o[32];
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
              float a = exp2_fast(fmaf(__uint_as_float(v[j]), p.scale_log2, minus)), b = exp2_fast(fmaf(__uint_as_float(v[j + 1]), p.scale_log2, minus));
              if (!all) {
                a = (bits >> j) & 1u ? a : 0.0f;
                b = (bits >> (j + 1)) & 1u ? b : 0.0f;
              }
              add0 += a;
              add1 += b;
              const uint32_t hi = pack_bf16(a, b);
              o[j >> 1] = hi;
              o[16 + (j >> 1)] = pack_bf16(a - __uint_as_float(hi << 16), b - __uint_as_float(hi & 0xFFFF0000u));
            }
            store32(s_base + c * 32, o);
          }
          sum += add0 + add1;
        }
        // values that must not meet the product: rows of the cache behind the length, drafted rows out of range
        if (m == 0 && (drafted || n_keys < kTileKeys)) {
          const int vi = (i + 1) % S::kStages;
          unsigned char *vt = stages + (size_t)vi * S::kTileBytes;
          if (!wait_bounded(&bar.full[vi], ((i + 1) / S::kStages) & 1)) { quit(); break; }
          const bool behind = r_in >= n_keys;
          bool odd = false;
          for (int c = 0; c < D / 8; ++c) {
            uint4 *at = reinterpret_cast<uint4 *>(vt + (c >> 3) * S::kHalfBytes + r_in * 128 + (((c + lane) & 7) << 4));
            if (behind) {
              *at = make_uint4(0, 0, 0, 0);
            } else if (drafted) {
              const uint4 x = *at;
              uint32_t y[4] = {x.x, x.y, x.z, x.w};
              bool here = false;
#pragma unroll
              for (int e = 0; e < 4; ++e) {              // exponent of all ones: infinite or not a number
                if ((y[e] & 0x7F80u) == 0x7F80u) { y[e] &= 0xFFFF0000u; here = true; }
                if ((y[e] & 0x7F800000u) == 0x7F800000u) { y[e] &= 0x0000FFFFu; here = true; }
              }
              if (here) *at = make_uint4(y[0], y[1], y[2], y[3]);
              odd |= here;
            }
          }
          if (drafted) {
            const uint32_t word = __ballot_sync(0xFFFFFFFFu, odd);
            if (lane == 0) bar.odd[dt & 1][quarter] = word;
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        if (!waited && !wait_bounded(&bar.o_done[m], (cnt - 1) & 1)) { quit(); break; }
        store_wait();
        fence_before();
        mbar_arrive(&bar.p_ready[buf]);
      }
      if (*give_up) break;
      if (!wait_bounded(&bar.o_done[m], (cnt - 1) & 1)) { quit(); break; }
      fence_after();
      // ---- the segment's rows: finished, or a partial ------------------------------------------------------------------
      if (warp_real) {
        const bool whole = w.whole();
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        const int64_t at = ((int64_t)w.b * p.q_heads + w.head * per_head + g) * p.nodes + node;
        const int64_t slot = w.slot(p, group, block) * p.rows_per_block + row;
        uint32_t any_odd = 0;
        if (w.t1 > w.ctiles)
          for (int c = 0; c < 8; ++c) any_odd |= *reinterpret_cast<volatile uint32_t *>(&bar.odd[c >> 2][c & 3]);
#pragma unroll
        for (int c = 0; c < D; c += 32) {
          uint32_t v[32];
          load32(o_base + c, v);
          if (any_odd && real) {
            // values out of range of the nodes this row sees, in the tiles of this segment
            for (int dt = max(w.t0 - w.ctiles, 0); dt < w.t1 - w.ctiles; ++dt)
              for (int j = dt * kTileKeys; j < min(p.nodes, (dt + 1) * kTileKeys); ++j) {
                if (!((*reinterpret_cast<volatile uint32_t *>(&bar.odd[dt & 1][(j & 127) >> 5]) >> (j & 31)) & 1u) || !sees(p, w.b, node, j)) continue;
                const __nv_bfloat16 *src = static_cast<const __nv_bfloat16 *>(p.tree_v) + w.b * p.tv_stride[0] + (w.head / share) * p.tv_stride[1] + j * p.tv_stride[2] + c;
                for (int e = 0; e < 32; ++e) {
                  const float x = __bfloat162float(src[e]);
                  if (!(fabsf(x) < INFINITY)) v[e] = __float_as_uint(__uint_as_float(v[e]) + x);
                }
              }
          }
          if (real) {
            if (whole) {
              uint4 *dst = reinterpret_cast<uint4 *>(static_cast<__nv_bfloat16 *>(p.out) + at * D + c);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                uint32_t o[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) o[k] = pack_bf16(__uint_as_float(v[8 * e + 2 * k]) * inv, __uint_as_float(v[8 * e + 2 * k + 1]) * inv);
                dst[e] = make_uint4(o[0], o[1], o[2], o[3]);
              }
            } else {
              uint4 *dst = reinterpret_cast<uint4 *>(p.part + slot * D + c);
#pragma unroll
              for (int e = 0; e < 8; ++e) dst[e] = make_uint4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
            }
          }
        }
        if (real) {
          if (!whole) p.part_ml[slot] = make_float2(top, sum);
          else if (p.lse) p.lse[at] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
        }
      }
      fence_before();
    }
  }
  fence_before();
  __syncthreads();
  if (warp == 1) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

// A [batch, heads, rows, D] tensor of the given strides; a box is 64 columns by kTileKeys rows of one head.
int make_map(CUtensorMap *map, const void *base, int D, int64_t rows, int64_t heads, int64_t batch, const int64_t (&stride)[3], int32_t &head_mul, int32_t &seq_mul) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) { note_error_text("cuTensorMapEncodeTiled is not available from the driver"); return LRQK_ELAUNCH; }
  head_mul = stride[1] != 0;      // a broadcast dimension has one entry
  seq_mul = stride[0] != 0;
  const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)rows, (cuuint64_t)(head_mul ? heads : 1), (cuuint64_t)(seq_mul ? batch : 1)};
  const cuuint64_t row = stride[2] != 0 ? (cuuint64_t)stride[2] * 2 : (cuuint64_t)D * 2;
  const cuuint64_t strides[3] = {row, head_mul ? (cuuint64_t)stride[1] * 2 : row, seq_mul ? (cuuint64_t)stride[0] * 2 : row};
  const cuuint32_t box[4] = {64, kTileKeys, 1, 1}, step[4] = {1, 1, 1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void *>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) { note_error_text("cuTensorMapEncodeTiled failed for a cache or drafted tensor"); return LRQK_ELAUNCH; }
  return LRQK_OK;
}

template <int D, int MT> int launch(const Params &p, cudaStream_t stream) {
  using S = Shape<D, MT>;
  Maps maps;
  Coord co;
  int rc = make_map(&maps.tk, p.tree_k, D, p.nodes, p.tree_heads, p.batch, p.tk_stride, co.tk_head, co.tk_seq);
  if (rc == LRQK_OK) rc = make_map(&maps.tv, p.tree_v, D, p.nodes, p.tree_heads, p.batch, p.tv_stride, co.tv_head, co.tv_seq);
  if (rc == LRQK_OK && p.capacity > 0) {
    rc = make_map(&maps.ck, p.cache_k, D, p.capacity, p.cache_heads, p.batch, p.ck_stride, co.ck_head, co.ck_seq);
    if (rc == LRQK_OK) rc = make_map(&maps.cv, p.cache_v, D, p.capacity, p.cache_heads, p.batch, p.cv_stride, co.cv_head, co.cv_seq);
  } else {                        // an empty cache has no tiles
    maps.ck = maps.tk;
    maps.cv = maps.tv;
    co.ck_head = co.cv_head = co.ck_seq = co.cv_seq = 0;
  }
  if (rc != LRQK_OK) return rc;
  auto kern = tree_tc_kernel<D, MT>;
  static SmemOptIn opt_in;
  LRQK_CUDA_TRY(opt_in.ensure(kern, S::kSmem));
  LRQK_CUDA_TRY(launch_dependent(kern, dim3((unsigned)(p.groups * p.row_blocks)), dim3(S::kThreads), S::kSmem, stream, 0, maps, p, co));
  return LRQK_OK;
}

}  // namespace

// One block of 128 rows where the rows of a cache head fit it, two of them above; one CTA an SM.
bool plan_tc(Params &p) {
  p.rows_per_block = p.rows <= kBlockRows ? kBlockRows : 2 * kBlockRows;
  p.tile_keys = kTileKeys;
  p.row_blocks = (p.rows + p.rows_per_block - 1) / p.rows_per_block;
  p.groups = kNumSMs / p.row_blocks;
  return p.groups >= 1;
}

int launch_tc(const Params &p, cudaStream_t stream) {
  if (p.rows_per_block == kBlockRows) return p.head_dim == 64 ? launch<64, 1>(p, stream) : launch<128, 1>(p, stream);
  return p.head_dim == 64 ? launch<64, 2>(p, stream) : launch<128, 2>(p, stream);
}

}  // namespace tree
}  // namespace lrqk
