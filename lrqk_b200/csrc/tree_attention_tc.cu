// Tree attention on the tensor cores: bf16, head_dim 64 or 128.  (Formula, split and partials: tree_attention.cu,
// tree_plan.cuh.)
//
// A CTA walks its run of 128-key tiles with one block of 128 query rows.  Per tile
//     S = Q K^T   tcgen05.mma M128, K from a TMA tile (K-major), S in TMEM
//     P = 2^(S c - m)   a thread per row, 64 keys at a time, in the place of their scores
//     O += P V    tcgen05.mma with P read from TMEM and V from its TMA tile (N = head_dim, MN-major), O in TMEM, per 64 keys
// Two chains of softmax warps work side by side on alternate tiles of the same rows, each with an S buffer, an O, a maximum and
// a sum of its own, joined at a segment's end; the scores run a tile ahead.  P enters the product as TWO bf16 parts, high and
// low: one bf16 would add as much error as the final rounding of the result, and under one row block the extra product hides
// behind the loads (three products of 512 cycles in the 2800 that HBM needs for a tile).
// More rows than a block: the blocks' CTAs walk the same tiles at the same time, each loading them for itself, so that HBM
// reads them once and L2 hands them out.  (One CTA with two blocks and P as one bf16 took 254 us where this takes 318, for 64
// nodes over two full contexts; but then a row lost accuracy, half a step of bf16 in each weight, as soon as other nodes made
// the call larger.  The same with P in two parts: 331 us, six products of 512 cycles a tile.)
// The running maximum moves only when a row's maximum has grown by more than 2^8 (then O is read, scaled and written
// back by the row's thread); weights then stay below 2^8 and sums keep fp32's full precision.
//
// Warp 0 issues the copies (a ring of K and V tiles, 128-byte swizzle), warp 1 owns TMEM and issues the products, warps
// 2..9 form the weights, 32 rows a warp.  (Two threads per row, a half of each tile's keys each, had to hand the maximum from
// one to the other: 190 instead of 187 us for 32 nodes.  One chain: 163 instead of 159 us with 1 node, 200 instead of 187 with
// 32.)
//
// What bounds it, over two full contexts of 119157 rows and 8 cache heads (979 MB, 149.5 us at 6.55 TB/s), 4 query heads a
// cache head: 164 us with 1 node, 169 with 8, 176 with 16 and 192 with 32: HBM, and with more rows the products and exponentials
// beside it.  64 nodes, two row blocks: 318 to 324 us, and 380 in continuous operation, where the power cap takes the clock
// from 1965 to 1380 MHz: 65 % of the cycles with a product under way (1536 of 2400 a tile and block), 43 % of the exponential
// unit's, the rest the hand-over between a chain's products and its weights.
//
// At 168 registers a thread (320 threads) the kernel spills 172 bytes and loads 260 again for head_dim 128, about 14 loads
// from local memory a tile and warp.
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
constexpr int kOCol = 256;        // TMEM columns: S 0..255, O 256 + 128 * chain

template <int D> struct Shape {
  static constexpr int kTileBytes = kTileKeys * D * 2;
  static constexpr int kHalfBytes = kTileKeys * 128;                 // 64 columns of a tile
  static constexpr int kQBytes = kBlockRows * D * 2;
  static constexpr int kStages = (208 * 1024 - kQBytes) / kTileBytes > 8 ? 8 : (208 * 1024 - kQBytes) / kTileBytes;
  static constexpr int kThreads = 64 + 256;
  static constexpr size_t kSmem = kQBytes + (size_t)kStages * kTileBytes + 1024;
};

struct Barriers {
  uint64_t full[8], empty[8], q_full;
  uint64_t s_full[2], p_ready[2][2], o_done[2][2];   // [chain][half of the keys]
  uint64_t joined[4];                       // both chains' maximum and sum of 32 rows are in `ml`
  // ... [segment's parity][chain][row].  One buffer a parity: a warp whose chain has no tile of the next segment waits for
  // nothing before it writes that segment's, while its partner may still be about to read this one's; two segments on,
  // the `joined` between them has passed, which the partner signals behind its read.
  float2 ml[2][2][kBlockRows];
  uint32_t tmem, give_up, odd[2][4];        // odd: drafted rows of V with values out of range, 128 bits for each drafted tile
  int32_t x0, x1, base, seq;
};

// Bounded wait for a phase, suspended for up to 20 us a look: spinning on plain looks, the product warp alone issued 900
// instructions a step and slowed the two softmax warps beside it by half.
constexpr uint32_t kLooks = 1u << 17;       // a few seconds
__device__ __forceinline__ bool await(uint64_t *bar, uint32_t parity) {
  const uint32_t a = saddr(bar);
  for (uint32_t i = 0; i < kLooks; ++i) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done) : "r"(a), "r"(parity), "r"(20000u) : "memory");
    if (done) return true;
  }
  return false;
}

__device__ __forceinline__ void tma_tile(const CUtensorMap *map, void *dst, uint64_t *bar, int c0, int row, int head, int seq) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
               ::"r"(saddr(dst)), "l"(map), "r"(saddr(bar)), "r"(c0), "r"(row), "r"(head), "r"(seq) : "memory");
}

__device__ __forceinline__ uint32_t elect_one() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one;
}
// Products issued by the lane whose `leader` is 1; all lanes of the warp come along.
// D[tmem] (+)= A[shared] * B[shared]
__device__ __forceinline__ void umma_ss(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(leader) : "memory");
}
// D[tmem] (+)= A[tmem, 16-bit pairs in 32-bit columns] * B[shared]
__device__ __forceinline__ void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(tmem_d), "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(leader) : "memory");
}
__device__ __forceinline__ void commit(uint64_t *bar, uint32_t leader) {
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
               "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(saddr(bar)), "r"(leader) : "memory");
}

// 32 columns of this warp's lanes.  The registers are defined once pin() has followed the wait.
__device__ __forceinline__ void load32_async(uint32_t taddr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
        "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
        "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
        "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(taddr) : "memory");
}
__device__ __forceinline__ void load_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// An empty statement behind the wait that names the registers, so that no use can move ahead of it.
__device__ __forceinline__ void pin(uint32_t (&v)[32]) {
  asm volatile("" : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]),
                    "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]));
  asm volatile("" : "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]),
                    "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31]));
}
__device__ __forceinline__ void load32(uint32_t taddr, uint32_t (&v)[32]) {
  load32_async(taddr, v);
  load_wait();
  pin(v);
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
__device__ __forceinline__ void store8(uint32_t taddr, const uint32_t (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};"
               ::"r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(taddr) : "memory");
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

// Eight columns of O times a row's factor.
__device__ __forceinline__ void scale8(uint32_t taddr, float f) {
  uint32_t v[8];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n\ttcgen05.wait::ld.sync.aligned;"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]) : "r"(taddr) : "memory");
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) * f);
  store8(taddr, v);
}

// Pairs of fp32 in one register pair: one instruction for two multiply-adds.
__device__ __forceinline__ uint64_t pair(uint32_t a, uint32_t b) { return ((uint64_t)b << 32) | a; }
__device__ __forceinline__ uint64_t pair(float a, float b) { return pair(__float_as_uint(a), __float_as_uint(b)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float low_of(uint64_t a) { return __uint_as_float((uint32_t)a); }
__device__ __forceinline__ float high_of(uint64_t a) { return __uint_as_float((uint32_t)(a >> 32)); }
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Weights of 32 keys of a row, 2^(s c - m), in the place of their scores; adds to the sums.
__device__ __forceinline__ void weigh(uint32_t (&s)[32], uint64_t c2, uint64_t minus2, uint64_t &sum2) {
#pragma unroll
  for (int j = 0; j < 32; j += 2) {
    const uint64_t x = fma2(pair(s[j], s[j + 1]), c2, minus2);
    const float a = exp2_fast(low_of(x)), b = exp2_fast(high_of(x));
    sum2 = add2(sum2, pair(a, b));
    s[j] = __float_as_uint(a);
    s[j + 1] = __float_as_uint(b);
  }
}
// ... as bf16: high parts into 16 columns, low parts into the next 16
__device__ __forceinline__ void store_two_parts(const uint32_t (&w)[32], uint32_t taddr) {
  const uint64_t less = pair(-1.0f, -1.0f);
  uint32_t o[32];
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    o[j] = pack_bf16(__uint_as_float(w[2 * j]), __uint_as_float(w[2 * j + 1]));
    const uint64_t rest = fma2(pair(o[j] << 16, o[j] & 0xFFFF0000u), less, pair(w[2 * j], w[2 * j + 1]));
    o[16 + j] = pack_bf16(low_of(rest), high_of(rest));
  }
  store32(taddr, o);
}
__device__ __forceinline__ float max32(const uint32_t (&s)[32]) {
  float part[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int j = 0; j < 32; j += 8)
#pragma unroll
    for (int k = 0; k < 4; ++k) part[k] = max3(part[k], __uint_as_float(s[j + 2 * k]), __uint_as_float(s[j + 2 * k + 1]));
  return fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
}

// Scores of keys that the row does not see: minus infinity.
__device__ __forceinline__ void hide(uint32_t (&s)[32], uint32_t seen) {
#pragma unroll
  for (int j = 0; j < 32; ++j) s[j] = (seen >> j) & 1u ? s[j] : 0xFF800000u;
}

// 32 bytes of a row (a thread's own row: whole sectors, half the instructions of 16-byte stores)
__device__ __forceinline__ void st32(void *dst, const uint32_t *v) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
               ::"l"(dst), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}

struct Maps { CUtensorMap ck, cv, tk, tv; };
struct Coord { int32_t ck_head, ck_seq, cv_head, cv_seq, tk_head, tk_seq, tv_head, tv_seq; };   // 0 where a dimension is broadcast

template <int D>
__global__ void __launch_bounds__(Shape<D>::kThreads, 1)
tree_tc_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Params p, const __grid_constant__ Coord co) {
  using S = Shape<D>;
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
    for (int i = 0; i < 2; ++i) mbar_init(&bar.s_full[i], 1);
    for (int i = 0; i < 4; ++i) { mbar_init(&bar.p_ready[i >> 1][i & 1], 4); mbar_init(&bar.o_done[i >> 1][i & 1], 1); mbar_init(&bar.joined[i], 2); }
    mbar_init(&bar.q_full, 8);
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
    const Cut cut(p, count_tiles(p, 0).total);
    const int x0 = cut.start(group), x1 = cut.start(group + 1);
    int seq = 0, base = 0;
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
    atomicExch(p.status, (int32_t)LRQK_ETIMEOUT);
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
            if (i >= S::kStages && !await(&bar.empty[s], (i / S::kStages - 1) & 1)) { quit(); break; }
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
    // ---- products: the whole warp walks along, so that descriptors stay in uniform registers; one lane issues ----------------
    constexpr uint32_t kIdescS = umma_idesc_bf16_k(128, kTileKeys);
    constexpr uint32_t kIdescO = umma_idesc_bf16_k(128, D) | (1u << 16);       // B (the values) MN-major
    const uint32_t leader = elect_one();
    const uint64_t q_desc = umma_desc_k_sw128(saddr(qs), 1024), k_desc = umma_desc_k_sw128(saddr(stages), 1024);
    const uint64_t v_desc = umma_desc_mn_sw128(saddr(stages), S::kHalfBytes, 1024);
    const auto ready = [&](uint64_t *b, uint32_t parity) {
      if (__all_sync(0xFFFFFFFFu, await(b, parity))) { fence_after(); return true; }
      quit();
      return false;
    };
    // (Addresses in descriptors count 16 bytes.)  `i`: ring index of the tile; x: its scores' buffer.
    const auto scores = [&](int i, int x) {
      const uint64_t kd = k_desc + (uint64_t)(((i % S::kStages) * S::kTileBytes) >> 4);
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        const uint64_t off = ((ks >> 2) * S::kHalfBytes + (ks & 3) * 32) >> 4;
        umma_ss(tmem + x * 128, q_desc + off, kd + off, kIdescS, ks > 0, leader);
      }
      commit(&bar.s_full[x], leader);
    };
    // the product of one half of a tile's keys with the values, as soon as its weights are there
    const auto values = [&](int i, int x, int half, uint32_t parity, bool fresh) {
      const uint32_t d = tmem + kOCol + x * 128, a = tmem + x * 128 + half * 64;
      if (!ready(&bar.p_ready[x][half], parity)) return false;
      const uint64_t vd = v_desc + (uint64_t)(((i % S::kStages) * S::kTileBytes + half * 64 * 128) >> 4);
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        const uint32_t at = a + (ks >> 1) * 32 + (ks & 1) * 8;   // per 32 keys: 16 columns of high parts, 16 of low parts
        umma_ts(d, at, vd + ks * (2048 >> 4), kIdescO, !(fresh && half == 0 && ks == 0), leader);
        umma_ts(d, at + 16, vd + ks * (2048 >> 4), kIdescO, 1, leader);
      }
      commit(&bar.o_done[x][half], leader);
      return true;
    };
    const auto arrived = [&](int i) { return ready(&bar.full[i % S::kStages], (i / S::kStages) & 1); };
    const auto release = [&](int i) { commit(&bar.empty[i % S::kStages], leader); };
    int i = 0, cnt = 0, seg = 0;           // ring index of the tile's K, tiles done, segments done
    for (; w.valid() && !*give_up; w.next(p), ++seg) {
      const int n = w.t1 - w.t0;
      bool ok = ready(&bar.q_full, seg & 1) && arrived(i);
      if (!ok) break;
      scores(i, cnt & 1);
      release(i);
      for (int t = 0; t < n; ++t, ++cnt, i += 2) {
        if (t + 1 < n) {
          if (!(ok = arrived(i + 2))) break;
          scores(i + 2, (cnt + 1) & 1);
          release(i + 2);
        }
        const uint32_t parity = (cnt >> 1) & 1;
        if (!(ok = arrived(i + 1) && values(i + 1, cnt & 1, 0, parity, t < 2) && values(i + 1, cnt & 1, 1, parity, t < 2))) break;
        release(i + 1);
      }
      if (!ok) break;
    }
  } else {
    // ---- weights: a thread per query row -------------------------------------------------------------------------------------
    const int chain = (warp - 2) >> 2, quarter = warp & 3, row = quarter * 32 + lane;        // TMEM lanes 32 * (warp % 4)..
    const uint32_t lane_base = tmem + ((uint32_t)(quarter * 32) << 16), o_base = lane_base + kOCol + chain * 128;
    const int g = group_row(p, row0 + row), node = row0 + row - g * p.nodes;                // query head in the group, node
    const bool real = row < n_rows, warp_real = quarter * 32 < n_rows;
    int cnt = 0, i0 = 0, seg = 0;                        // tiles done, ring index of the segment's first K, segments done
    const auto signal = [&](uint64_t *b) {               // one arrival for the warp, behind all of its lanes' writes
      __syncwarp();
      if (lane == 0) mbar_arrive(b);
    };
    for (; w.valid() && !*give_up; w.next(p), ++seg) {
      // the block's queries, for the K-major swizzled operand (rows that do not exist: zeros); all loads in flight at once
      constexpr int kLoaders = 256, kLoads = kBlockRows * (D / 8) / kLoaders;
      const int first = chain * 128 + quarter * 32 + lane;
      uint4 qv[kLoads];
      {
        const __nv_bfloat16 *q = static_cast<const __nv_bfloat16 *>(p.q) + w.b * p.q_stride[0] + (int64_t)(w.head * per_head) * p.q_stride[1];
#pragma unroll
        for (int k = 0; k < kLoads; ++k) {
          const int e = first + k * kLoaders, r = e / (D / 8), c = e % (D / 8);
          const int gr = group_row(p, row0 + r);
          qv[k] = make_uint4(0, 0, 0, 0);
          if (r < n_rows) qv[k] = ld16(q + gr * p.q_stride[1] + (int64_t)(row0 + r - gr * p.nodes) * p.q_stride[2] + c * 8);
        }
      }
      // which nodes of a drafted step this row sees
      uint32_t seen[4] = {0, 0, 0, 0};
      int seen_at = -1;
      const auto look = [&](int at) {                    // a row of the mask at a time, a lane per node: coalesced, no exchange
        seen_at = at;
        const uint8_t *mask = p.mask ? p.mask + w.b * p.mask_stride : nullptr;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int first = at + c * 32, j = first + lane;
          seen[c] = 0;
          if (first >= p.nodes) continue;
          if (!mask) {
            const int n = node - first;                  // nodes up to its own
            seen[c] = n >= 31 ? 0xFFFFFFFFu : n >= 0 ? (2u << n) - 1u : 0u;
            continue;
          }
#pragma unroll 16
          for (int r = 0; r < 32; ++r) {
            const int other = __shfl_sync(0xFFFFFFFFu, node, r);
            const bool yes = j < p.nodes && mask[(int64_t)other * p.nodes + j] != 0;
            const uint32_t word = __ballot_sync(0xFFFFFFFFu, yes);
            if (lane == r) seen[c] = word;
          }
        }
      };
      if (warp_real && w.t1 > w.ctiles) look(max(w.t0 - w.ctiles, 0) * kTileKeys);   // ahead of its use
      {
#pragma unroll
        for (int k = 0; k < kLoads; ++k) {
          const int e = first + k * kLoaders, r = e / (D / 8), c = e % (D / 8);
          *reinterpret_cast<uint4 *>(qs + (c >> 3) * (kBlockRows * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = qv[k];
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        signal(&bar.q_full);
      }
      float top = -INFINITY, sum = 0.0f;                 // maximum in use, in octaves; sum of this thread's weights
      const int n_tiles = w.t1 - w.t0, plain = w.len / kTileKeys - w.t0;   // the first `plain` tiles are seen whole
      for (int st = 0; st < n_tiles; ++st, ++cnt) {
        if ((cnt & 1) != chain) continue;                // the other chain's tile
        const uint32_t parity = (cnt >> 1) & 1;
        if (!await(&bar.s_full[chain], parity)) { quit(); break; }
        const bool masked = st >= plain;
        int n_keys = kTileKeys, dt = -1;                 // filled keys of the tile; drafted tile
        if (masked) {
          dt = w.t0 + st - w.ctiles;
          n_keys = min(kTileKeys, dt >= 0 ? p.nodes - dt * kTileKeys : w.len - (w.t0 + st) * kTileKeys);
          if (warp_real && dt >= 0 && dt * kTileKeys != seen_at) look(dt * kTileKeys);
        }
        const bool drafted = dt >= 0;
        // values that must not meet the product: rows of the cache behind the length, drafted rows out of range
        if (masked) {
          // (the scores are there once every warp has left the segment before, whose marks in `odd` these replace)
          const int i = i0 + 2 * st;
          const int vi = (i + 1) % S::kStages;
          unsigned char *vt = stages + (size_t)vi * S::kTileBytes;
          if (!await(&bar.full[vi], ((i + 1) / S::kStages) & 1)) { quit(); break; }
          // this thread's row of the tile, 16 bytes at a time (in an order that keeps the banks apart)
          const auto piece = [&](int c) { return reinterpret_cast<uint4 *>(vt + (c >> 3) * S::kHalfBytes + row * 128 + (((c + lane) & 7) << 4)); };
          bool odd = false;
          if (row >= n_keys) {                           // (as a key of the tile)
#pragma unroll
            for (int c = 0; c < D / 8; ++c) *piece(c) = make_uint4(0, 0, 0, 0);
          } else if (drafted) {
            uint32_t most = 0;                           // largest magnitude, as two 16-bit patterns
#pragma unroll
            for (int c = 0; c < D / 8; ++c) {
              const uint4 y = *piece(c);
              most = __vmaxu2(__vmaxu2(most, y.x & 0x7FFF7FFFu), y.y & 0x7FFF7FFFu);
              most = __vmaxu2(__vmaxu2(most, y.z & 0x7FFF7FFFu), y.w & 0x7FFF7FFFu);
            }
            odd = (most & 0xFFFFu) >= 0x7F80u || (most >> 16) >= 0x7F80u;   // exponent of all ones: infinite or not a number
            if (odd) {
#pragma unroll 1
              for (int c = 0; c < D / 8; ++c) {
                const uint4 y4 = *piece(c);
                uint32_t y[4] = {y4.x, y4.y, y4.z, y4.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  if ((y[e] & 0x7F80u) == 0x7F80u) y[e] &= 0xFFFF0000u;
                  if ((y[e] & 0x7F800000u) == 0x7F800000u) y[e] &= 0x0000FFFFu;
                }
                *piece(c) = make_uint4(y[0], y[1], y[2], y[3]);
              }
            }
          }
          if (drafted) {
            const uint32_t word = __ballot_sync(0xFFFFFFFFu, odd);
            if (lane == 0) bar.odd[dt & 1][quarter] = word;
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        bool ok = true;
#pragma unroll
        for (int half = 0; half < 2 && ok; ++half) {
          fence_after();
          const uint32_t s_base = lane_base + chain * 128 + half * 64;
          if (warp_real) {
            uint32_t v[32], u[32];
            load32_async(s_base, v);
            load32_async(s_base + 32, u);
            load_wait();
            pin(v);
            pin(u);
            if (masked) {
              const int n = n_keys - half * 64;          // filled keys of this half
              hide(v, drafted ? seen[2 * half] : n >= 32 ? 0xFFFFFFFFu : n > 0 ? (1u << n) - 1u : 0u);
              hide(u, drafted ? seen[2 * half + 1] : n >= 64 ? 0xFFFFFFFFu : n > 32 ? (1u << (n - 32)) - 1u : 0u);
            }
            const float now = fmaxf(max32(v), max32(u)) * p.scale_log2;
            const bool move = now > top + kGrow || (top == -INFINITY && now > -INFINITY);
            if (__any_sync(0xFFFFFFFFu, move)) {
              const float use = move ? now : top, fade = move ? exp2_fast(top - use) : 1.0f;
              if (half == 1 || st >= 2) {
                // O holds the chain's products up to the half before: that one has to be in it
                if (!(ok = await(&bar.o_done[chain][half ^ 1], half == 1 ? parity : parity ^ 1))) break;
                fence_after();
#pragma unroll 1
                for (int c = 0; c < D; c += 8) scale8(o_base + c, fade);
              }
              sum *= fade;
              top = use;
            }
            const uint64_t c2 = pair(p.scale_log2, p.scale_log2), minus2 = top == -INFINITY ? 0 : pair(-top, -top);
            uint64_t sum2 = 0;
            weigh(v, c2, minus2, sum2);
            weigh(u, c2, minus2, sum2);
            store_two_parts(v, s_base);
            store_two_parts(u, s_base + 32);
            sum += low_of(sum2) + high_of(sum2);
          }
          store_wait();
          fence_before();
          signal(&bar.p_ready[chain][half]);
        }
        if (!ok) { quit(); break; }
      }
      i0 += 2 * n_tiles;
      if (*give_up) break;
      // (a segment of one tile leaves the chain that had none without an O)
      const bool last_mine = ((cnt - 1) & 1) == chain, mine = last_mine || n_tiles > 1;
      if (mine) {
        const int last = last_mine ? cnt - 1 : cnt - 2;
        if (!await(&bar.o_done[chain][1], (last >> 1) & 1)) { quit(); break; }
        fence_after();
      }
      // each chain's O and statistics for the other's warp of the same rows
      bar.ml[seg & 1][chain][row] = make_float2(top, sum);
      fence_before();
      signal(&bar.joined[quarter]);
      if (!await(&bar.joined[quarter], seg & 1)) { quit(); break; }
      fence_after();
      // ---- the segment's rows: finished, or a partial -------------------------------------------------------------------------
      if (warp_real) {
        const float2 other = bar.ml[seg & 1][chain ^ 1][row];
        const float both = fmaxf(top, other.x);
        const float fade = top == both ? 1.0f : exp2_fast(top - both), other_fade = other.x == both ? 1.0f : exp2_fast(other.x - both);
        sum = sum * fade + other.y * other_fade;
        top = both;
        const bool others = n_tiles > 1 || !mine;
        constexpr int kCols = D / 2;                     // columns of a thread: a row's two chains share them
        const int c0 = chain * kCols;
        const bool whole = w.whole();
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        const int64_t at = ((int64_t)w.b * p.q_heads + w.head * per_head + g) * p.nodes + node;
        const int64_t slot = w.slot(p, group, block) * p.rows_per_block + row;
        uint32_t any_odd = 0;
        if (w.t1 > w.ctiles)
          for (int c = 0; c < 8; ++c) any_odd |= *reinterpret_cast<volatile uint32_t *>(&bar.odd[c >> 2][c & 3]);
#pragma unroll
        for (int cc = 0; cc < kCols; cc += 32) {
          const int c = c0 + cc;
          uint32_t v[32];
          if (mine) load32(o_base + c, v);
          uint32_t u[32];
          if (others) load32(lane_base + kOCol + (chain ^ 1) * 128 + c, u);
#pragma unroll
          for (int e = 0; e < 32; ++e)
            v[e] = __float_as_uint((mine ? __uint_as_float(v[e]) * fade : 0.0f) + (others ? __uint_as_float(u[e]) * other_fade : 0.0f));
          if (any_odd && real) {
            // values out of range of the nodes this row sees, in the tiles of this segment
            for (int dt = max(w.t0 - w.ctiles, 0); dt < w.t1 - w.ctiles; ++dt)
              for (int j = dt * kTileKeys; j < min(p.nodes, (dt + 1) * kTileKeys); ++j) {
                if (!((*reinterpret_cast<volatile uint32_t *>(&bar.odd[dt & 1][(j & 127) >> 5]) >> (j & 31)) & 1u) || !sees(p, w.b, node, j)) continue;
                const __nv_bfloat16 *src = static_cast<const __nv_bfloat16 *>(p.tree_v) + w.b * p.tv_stride[0] + (w.head / share) * p.tv_stride[1] + j * p.tv_stride[2] + c;
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                  const float x = __bfloat162float(src[e]);
                  if (!(fabsf(x) < INFINITY)) v[e] = __float_as_uint(__uint_as_float(v[e]) + x);
                }
              }
          }
          if (real) {
            if (whole) {
              __nv_bfloat16 *dst = static_cast<__nv_bfloat16 *>(p.out) + at * D + c;
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                uint32_t o[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) o[k] = pack_bf16(__uint_as_float(v[16 * e + 2 * k]) * inv, __uint_as_float(v[16 * e + 2 * k + 1]) * inv);
                st32(dst + 16 * e, o);
              }
            } else {
              float *dst = p.part + slot * D + c;
#pragma unroll
              for (int e = 0; e < 4; ++e) st32(dst + 8 * e, v + 8 * e);
            }
          }
        }
        if (real && chain == 0) {
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

template <int D> int launch(const Params &p, cudaStream_t stream) {
  using S = Shape<D>;
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
  auto kern = tree_tc_kernel<D>;
  static SmemOptIn opt_in;
  LRQK_CUDA_TRY(opt_in.ensure(kern, S::kSmem));
  LRQK_CUDA_TRY(launch_dependent(kern, dim3((unsigned)(p.groups * p.row_blocks)), dim3(S::kThreads), S::kSmem, stream, 0, maps, p, co));
  return LRQK_OK;
}

}  // namespace

// Blocks of 128 rows; one CTA an SM, more than that only where there are more blocks than SMs.
void plan_tc(Params &p) {
  p.rows_per_block = kBlockRows;
  p.tile_keys = kTileKeys;
  p.unit_cost = 4;
  p.row_blocks = (p.rows + p.rows_per_block - 1) / p.rows_per_block;
  p.groups = p.row_blocks < kNumSMs ? kNumSMs / p.row_blocks : 1;
}

int launch_tc(const Params &p, cudaStream_t stream) {
  return p.head_dim == 64 ? launch<64>(p, stream) : launch<128>(p, stream);
}

}  // namespace tree
}  // namespace lrqk
