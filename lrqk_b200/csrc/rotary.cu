// Rotary positions of q and k, forward and adjoint, for prompts, single tokens and drafted trees.
//
//   pair (a, b), angle t = position * w:   a' = f (a cos t - b sin t),  b' = f (b cos t + a sin t)
//
// with (a, b) = (x[i], x[i + part/2]) (half layout) or (x[2i], x[2i+1]) (interleaved); elements from `part` on are
// copied.  The adjoint (gradient) turns by -t.  All arithmetic is fp32, rounded once on the way out.
//
// Angles: a far position loses its angle in fp32 (t = 131072 rad is known to 2^-7 rad there).  Only t modulo a turn
// matters, so a frequency is held in TURNS per position as a 64-bit binary fraction, F = 2^64 (w / 2 pi modulo 1), and
// position * F modulo 2^64 -- one wrapping integer product, right for negative positions too -- is the angle's
// fraction of a turn.  What is lost is lost in forming w / 2 pi in a double (a rounded constant, a rounded product): an
// error of |position| ((w / 2 pi) 2^-52 + 2^-65) turns, 2^-37 of a turn at position 131072 for w = 1 and less for slower
// pairs, where fp32 results resolve 2^-24.
//
// Bound: HBM.  q and k are read once and written once; the angles come from registers, not from cos/sin tables.  A
// thread owns one 16-byte run of pairs of one token, computes its cosines and sines once and applies them to a run
// of heads, four heads' loads in flight at a time; with few tokens the heads are dealt over more threads instead.
// Measured: 65536 tokens of 32 + 8 bf16 heads of 128, 1.34 GB in 219 us (6.1 TB/s, 94 % of a copy); one token of four
// sequences 2.4 us; the adjoint of 2 x 1537 tokens of 28 + 4 fp32 heads 14.9 us (its 101 MB partly from L2).
#include "common.cuh"

namespace lrqk {
namespace {

constexpr int kRotThreads = 256;
constexpr int kRotUnroll = 4;   // heads whose loads a thread has in flight

struct RotaryParams {
  const void *src[2];          // q, k
  void *dst[2];                // contiguous [batch][heads][length][head_dim]
  int64_t stride[2][3];        // batch, head, token strides of the sources, in elements
  int32_t heads[2];
  const void *positions;
  int64_t pos_stride;          // between sequences (0: shared), in elements
  const double *freq;
  float factor, sign;
  int32_t pos64, batch, length, head_dim, part, slots, rot_slots, heads_per_thread;
  int64_t total;               // batch * length * slots
};

template <typename T, int V> struct Run;   // V consecutive elements
template <> struct Run<__nv_bfloat16, 8> {
  uint4 v;
  __device__ __forceinline__ void load(const __nv_bfloat16 *p) { v = ld_stream16(p); }
  __device__ __forceinline__ void store(__nv_bfloat16 *p) const { st16(p, v); }
  __device__ __forceinline__ void get(float (&f)[8]) const { Elt<__nv_bfloat16>::unpack(v, f); }
  __device__ __forceinline__ void set(const float (&f)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t *>(&h);
    }
    v = make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <> struct Run<float, 4> {
  uint4 v;
  __device__ __forceinline__ void load(const float *p) { v = ld_stream16(p); }
  __device__ __forceinline__ void store(float *p) const { st16(p, v); }
  __device__ __forceinline__ void get(float (&f)[4]) const { Elt<float>::unpack(v, f); }
  __device__ __forceinline__ void set(const float (&f)[4]) {
    v = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};
template <typename T> struct Run<T, 2> {   // any alignment: two elements one by one
  T a, b;
  __device__ __forceinline__ void load(const T *p) { a = p[0]; b = p[1]; }
  __device__ __forceinline__ void store(T *p) const { p[0] = a; p[1] = b; }
  __device__ __forceinline__ void get(float (&f)[2]) const { f[0] = Elt<T>::to_float(a); f[1] = Elt<T>::to_float(b); }
  __device__ __forceinline__ void set(const float (&f)[2]) { a = Elt<T>::from_float(f[0]); b = Elt<T>::from_float(f[1]); }
};
template <typename T> struct Run<T, 1> {
  T a;
  __device__ __forceinline__ void load(const T *p) { a = p[0]; }
  __device__ __forceinline__ void store(T *p) const { p[0] = a; }
  __device__ __forceinline__ void get(float (&f)[1]) const { f[0] = Elt<T>::to_float(a); }
  __device__ __forceinline__ void set(const float (&f)[1]) { a = Elt<T>::from_float(f[0]); }
};

// cosine and sine (times the factor) of pair i at a position
__device__ __forceinline__ void wheel(const RotaryParams &p, int64_t pos, int i, float &c, float &s) {
  double turns = p.freq[i] * 0.15915494309189533577;   // 1 / (2 pi)
  turns -= floor(turns);
  const uint64_t per_position = __double2ull_rn(turns * 18446744073709551616.0);   // saturates where turns rounds to 1
  const float part_of_turn = __ll2float_rn((int64_t)((uint64_t)pos * per_position)) * 5.421010862427522e-20f;  // 2^-64
  sincospif(2.0f * part_of_turn, &s, &c);
  c *= p.factor;
  s *= p.factor * p.sign;
}

// V: elements of a run.  Half layout: a slot is a run of V pairs, two runs of elements.  Interleaved: a slot is one run
// of V elements, V / 2 pairs.  Slots from rot_slots on copy one run of the unrotated tail.
template <typename T, int V, bool INTERLEAVED>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(const __grid_constant__ RotaryParams p) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int PAIRS = INTERLEAVED ? V / 2 : V;
  const int64_t id = (int64_t)blockIdx.x * kRotThreads + threadIdx.x;
  if (id >= p.total) return;
  const int64_t token = id / p.slots;                  // b * length + l
  const int slot = (int)(id - token * p.slots);
  const int b = (int)(token / p.length), l = (int)(token - (int64_t)b * p.length);
  const int h0 = blockIdx.y * p.heads_per_thread, h1 = min(h0 + p.heads_per_thread, p.heads[0] + p.heads[1]);
  const bool rotate = slot < p.rot_slots;
  const int at = rotate ? slot * V : p.part + (slot - p.rot_slots) * V;
  float c[PAIRS], s[PAIRS];
  if (rotate) {
    const int64_t pi = b * p.pos_stride + l;
    const int64_t pos = p.pos64 ? static_cast<const int64_t *>(p.positions)[pi] : (int64_t)static_cast<const int32_t *>(p.positions)[pi];
    const int first = INTERLEAVED ? at / 2 : at;
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) wheel(p, pos, first + i, c[i], s[i]);
  }
  const int half = p.part >> 1;
  for (int h = h0; h < h1; h += kRotUnroll) {
    Run<T, V> x[kRotUnroll], y[kRotUnroll];
#pragma unroll
    for (int j = 0; j < kRotUnroll; ++j) {
      const int hh = h + j;
      if (hh < h1) {
        const int w = hh >= p.heads[0], hl = hh - (w ? p.heads[0] : 0);
        const T *src = static_cast<const T *>(p.src[w]) + b * p.stride[w][0] + hl * p.stride[w][1] + l * p.stride[w][2] + at;
        x[j].load(src);
        if (!INTERLEAVED && rotate) y[j].load(src + half);
      }
    }
#pragma unroll
    for (int j = 0; j < kRotUnroll; ++j) {
      const int hh = h + j;
      if (hh < h1) {
        const int w = hh >= p.heads[0], hl = hh - (w ? p.heads[0] : 0);
        T *dst = static_cast<T *>(p.dst[w]) + (((int64_t)b * p.heads[w] + hl) * p.length + l) * p.head_dim + at;
        if (rotate) {
          float f[V], g[V];
          x[j].get(f);
          if constexpr (INTERLEAVED) {
#pragma unroll
            for (int i = 0; i < PAIRS; ++i) {
              g[2 * i] = f[2 * i] * c[i] - f[2 * i + 1] * s[i];
              g[2 * i + 1] = f[2 * i + 1] * c[i] + f[2 * i] * s[i];
            }
            x[j].set(g);
          } else {
            y[j].get(g);
#pragma unroll
            for (int i = 0; i < PAIRS; ++i) {
              const float u = f[i] * c[i] - g[i] * s[i], v = g[i] * c[i] + f[i] * s[i];
              f[i] = u;
              g[i] = v;
            }
            x[j].set(f);
            y[j].set(g);
            y[j].store(dst + half);
          }
        }
        x[j].store(dst);
      }
    }
  }
}

template <typename T, int V, bool INTERLEAVED> int launch(RotaryParams &p, cudaStream_t stream) {
  p.rot_slots = INTERLEAVED ? p.part / V : p.part / 2 / V;
  p.slots = p.rot_slots + (p.head_dim - p.part) / V;
  p.total = (int64_t)p.batch * p.length * p.slots;
  const int heads = p.heads[0] + p.heads[1];
  // Enough threads to fill the GPU first (a token's cosines are then computed by several of them), then as many heads
  // to a thread as there are.  One head to a thread for a single token, all heads from a few hundred tokens on.
  const int64_t want = (int64_t)kNumSMs * 1536;
  int chunks = (int)(p.total >= want ? 1 : ceil_div64(want, p.total));
  if (chunks > heads) chunks = heads;
  p.heads_per_thread = (heads + chunks - 1) / chunks;
  chunks = (heads + p.heads_per_thread - 1) / p.heads_per_thread;
  const int64_t blocks = ceil_div64(p.total, kRotThreads);
  if (blocks >= (1ll << 31) || chunks > 65535) return LRQK_EUNSUPPORTED;
  LRQK_CUDA_TRY(launch_dependent(rotary_kernel<T, V, INTERLEAVED>, dim3((unsigned)blocks, (unsigned)chunks), dim3(kRotThreads), 0,
                                 stream, 0, p));
  return LRQK_OK;
}

template <typename T> int dispatch(RotaryParams &p, bool interleaved, bool aligned, cudaStream_t stream) {
  constexpr int VE = Elt<T>::kPerVec;
  // 16-byte runs where every row, the two halves and the tail start on 16 bytes; element by element otherwise
  const bool wide = aligned && p.head_dim % VE == 0 && p.part % VE == 0 && (interleaved || (p.part / 2) % VE == 0);
  if (interleaved) return wide ? launch<T, VE, true>(p, stream) : launch<T, 2, true>(p, stream);
  return wide ? launch<T, VE, false>(p, stream) : launch<T, 1, false>(p, stream);
}

}  // namespace
}  // namespace lrqk

extern "C" int lrqk_rotary(const lrqk_rotary_args *a, lrqk_stream_t stream) {
  using namespace lrqk;
  const int rc = check_device();
  if (rc != LRQK_OK) return rc;
  if (!a || !a->q || !a->q_out || !a->positions || !a->inv_freq) return LRQK_EINVAL;
  if (a->batch < 0 || a->length < 0 || a->q_heads <= 0 || a->k_heads < 0 || a->head_dim <= 0) return LRQK_EINVAL;
  if (a->k_heads > 0 && (!a->k || !a->k_out)) return LRQK_EINVAL;
  if (a->rotary_dim <= 0 || a->rotary_dim % 2 != 0 || a->rotary_dim > a->head_dim) return LRQK_EINVAL;
  if (a->dtype != LRQK_F32 && a->dtype != LRQK_BF16) return LRQK_EUNSUPPORTED;
  if (a->head_dim > 1024 || (a->interleaved && a->head_dim % 2 != 0)) return LRQK_EUNSUPPORTED;
  if ((int64_t)a->q_heads + a->k_heads >= (1ll << 31)) return LRQK_EUNSUPPORTED;
  if (a->batch == 0 || a->length == 0) return LRQK_OK;
  RotaryParams p;
  p.src[0] = a->q; p.src[1] = a->k;
  p.dst[0] = a->q_out; p.dst[1] = a->k_out;
  p.heads[0] = a->q_heads; p.heads[1] = a->k_heads;
  uintptr_t low = reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->q_out);
  if (a->k_heads) low |= reinterpret_cast<uintptr_t>(a->k) | reinterpret_cast<uintptr_t>(a->k_out);
  for (int i = 0; i < 3; ++i) {
    const int32_t n[2][3] = {{a->batch, a->q_heads, a->length}, {a->batch, a->k_heads, a->length}};
    p.stride[0][i] = n[0][i] > 1 ? a->q_stride[i] : 0;   // (a dimension with one entry has no stride that matters)
    p.stride[1][i] = n[1][i] > 1 && a->k_heads ? a->k_stride[i] : 0;
    low |= (uintptr_t)((p.stride[0][i] | p.stride[1][i]) * (int64_t)elt_size(a->dtype));
  }
  p.positions = a->positions; p.pos_stride = a->position_stride; p.pos64 = a->positions_are_64bit;
  p.freq = a->inv_freq; p.factor = a->factor; p.sign = a->adjoint ? -1.0f : 1.0f;
  p.batch = a->batch; p.length = a->length; p.head_dim = a->head_dim; p.part = a->rotary_dim;
  LRQK_DISPATCH_DTYPE(a->dtype, T, return dispatch<T>(p, a->interleaved != 0, (low & 15) == 0, as_stream(stream)));
}
