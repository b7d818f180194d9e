// Attention of a tree of drafted tokens over a cache (one token is the plain decode step), on tensor cores.
//
// Row t of sequence b (t < T) sees the cache's keys 0 .. len_b - 1 and, of the tree's own keys at len_b + j, those with
// mask[b][t][j]; out = softmax(scale q K^T) V, zeros where a row sees nothing. Caches hold bf16, f16, or 8-bit codes with one
// f32 scale per (head, position).
//
// The T * G rows that share a kv head (G query heads) are one block of rows, so that a key or value is fetched once for all of
// them. Work on a (sequence, kv head) is split over the keys: over the warps of a block and over the blocks of a cluster,
// each with a running (maximum, sum, output) of its own; the states meet in a fixed order, in shared memory.
//   S = Q K^T  mma.sync. The order of the head's dimensions inside the product is free, so 8-bit keys are read 16 bytes per lane
//              as they lie; the key's scale multiplies the score. q8 keys enter whole-number products (m16n8k32) unconverted,
//              others become f16 in a register (m16n8k16).
//   O += P V   the accumulators of S are the A operand of P. 8-bit values are read 16 bytes of one key per lane, and two keys'
//              bytes are interleaved on the way to f16; the value's scale goes into P. 2-byte values come by ldmatrix.trans.
// Precision. Operands are f16 (bf16 for bf16 caches); what does not fit goes as two or three terms (an f32 query: 22 or 24
// bits). A row of Q enters times a power of two that brings its largest element to 2^8 .. 2^9 (f16 has five bits of
// exponent) or, for whole-number products, as 24-bit numbers. An mma truncates where it adds to its accumulator, always toward zero,
// so a tile's P V starts from zero and joins the running output by rounded adds.
// P has two terms (22 bits; over bf16 caches 16, and three terms for f32 queries), but one of 11 bits for bf16 queries over f16 and
// 8-bit caches: a weight is off by 2^-11 of itself at most and by about 2e-4 in the mean, independently of the others, which moves a
// result by about as much of its size; its own rounding to bf16 moves it by 1.7e-3. (4 x 64 rows at 8192 over e4m3: error against 64
// bits 1.67e-3, with a plain f32 computation 1.66e-3. With two terms 85.7 us instead of 67.6, 8 x 2 rows at 8192 68.3 instead of 49.4.)
// Over 8-bit caches P takes the values' scales, relative to the largest of those that its row has seen so far: f16 ends at 2^-24, so
// what is below 2^-38 (f32 queries) or 2^-30 (others) of the largest value that a row sees is lost, however small that value's own
// weight is.
// This header: up to sixteen rows. 8 x 1 rows of 64 heads at 32768 over q8 98 us, 465 MB at 73 % of the copy bandwidth; what bounds it
// is the latency of instructions at eight warps per SM (217 registers). 1 x 5 rows of 16 heads at 600, bf16: 10.4 us. The forms for
// nine to sixteen rows over e4m3 keep registers in local memory (156 to 356 bytes are loaded back): 8 x 2 rows of 64 heads at 8192,
// f16, 68.5 us, over q8 52.3.
#pragma once

#include <algorithm>
#include <type_traits>

#include "clusters.cuh"
#include "common.cuh"
#include "kv_codes.cuh"
#include "ring.cuh"

namespace dyn {

enum { TREE_BF16 = 0, TREE_F16 = 1, TREE_Q8 = 2, TREE_E4M3 = 3 };

struct TreeArgs {
  const void* q;            // [batch][rows][heads][d]
  void* out;                // the same, dense
  const uint8_t *k, *v;     // [batch][kv head][cap][d]
  const float *ks, *vs;     // [batch][kv head][cap]; NULL for 2-byte caches
  const int64_t* lengths;   // [batch] keys in front of the tree; below zero: the sequence is passed over
  const uint8_t* mask;      // [batch][rows][rows]; NULL: each row sees the tree's keys up to its own
  int64_t qs[3];            // elements between batch entries, rows, heads
  int64_t kst[3], vst[3];   // bytes between batch entries, heads, keys
  int64_t kss[2], vss[2];   // floats between batch entries, heads
  int64_t ms[2];            // bytes between batch entries, rows
  int64_t batch, cap;
  int rows, heads, kv_heads, group, d, splits;
  float scale;
};

int tree_attention_bf16(const TreeArgs& a, int q_type, cudaStream_t s);
int tree_attention_f16(const TreeArgs& a, int q_type, cudaStream_t s);
int tree_attention_q8(const TreeArgs& a, int q_type, cudaStream_t s);
int tree_attention_e4m3(const TreeArgs& a, int q_type, cudaStream_t s);

namespace tree {

constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool live) {
  const int n = live ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src, bool live) {
  const int n = live ? 4 : 0;
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) { return __byte_perm(a, b, sel); }

// Operand type of the products: f16, or bf16 for bf16 caches.
template <bool BF>
struct Op {
  // x and y keep what the packed pair left of them
  __device__ static __forceinline__ uint32_t take(float& x, float& y) {
    if (BF) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
      x -= __low2float(h), y -= __high2float(h);
      return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __half2 h = __floats2half2_rn(x, y);
    x -= __low2float(h), y -= __high2float(h);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  __device__ static __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (BF)
      asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
          : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
          : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
      asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
          : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
          : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ uint4 lds16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint2 lds8(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}
__device__ __forceinline__ float lds4(uint32_t addr) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}

// Two e4m3 codes as an f16 pair.
__device__ __forceinline__ uint32_t e4m3_pair(uint32_t codes) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((unsigned short)codes));
  return r;
}
// Four codes of one word as two f16 pairs, in order (q8: whole numbers).
template <bool E4M3>
__device__ __forceinline__ void widen(uint32_t w, uint32_t* lo, uint32_t* hi) {
  if (E4M3) {
    *lo = e4m3_pair(w), *hi = e4m3_pair(w >> 16);
  } else {
    w ^= 0x80808080u;
    *lo = kv_q8_to_half2(prmt(w, 0x64646464u, 0x4140)), *hi = kv_q8_to_half2(prmt(w, 0x64646464u, 0x4342));
  }
}
// Entry i (0 .. 3) of two words, interleaved: (x_i, y_i) as an f16 pair; r[i].
template <bool E4M3>
__device__ __forceinline__ void widen_pairs(uint32_t x, uint32_t y, uint32_t (&r)[4]) {
  uint32_t lo = prmt(x, y, 0x5140), hi = prmt(x, y, 0x7362);
  if (E4M3) {
    r[0] = e4m3_pair(lo), r[1] = e4m3_pair(lo >> 16), r[2] = e4m3_pair(hi), r[3] = e4m3_pair(hi >> 16);
  } else {
    lo ^= 0x80808080u, hi ^= 0x80808080u;
    r[0] = kv_q8_to_half2(prmt(lo, 0x64646464u, 0x4140)), r[1] = kv_q8_to_half2(prmt(lo, 0x64646464u, 0x4342));
    r[2] = kv_q8_to_half2(prmt(hi, 0x64646464u, 0x4140)), r[3] = kv_q8_to_half2(prmt(hi, 0x64646464u, 0x4342));
  }
}
// Bytes that are e4m3's NaN become zeros; says whether there were any.
__device__ __forceinline__ bool without_nan(uint32_t& w) {
  const uint32_t some = (((w & 0x7f7f7f7fu) ^ 0x7f7f7f7fu) + 0x7f7f7f7fu) & 0x80808080u;
  const uint32_t none = some ^ 0x80808080u;
  w &= ~((none >> 7) * 0xffu);
  return none != 0;
}
// 2-byte entries that are not finite become zeros; says whether there were any.
template <bool BF>
__device__ __forceinline__ bool without_odd(uint32_t& w) {
  const uint32_t odd = BF ? ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u : ((w & 0x7c007c00u) + 0x04000400u) & 0x80008000u;
  w &= ~((odd >> 15) * 0xffffu);
  return odd != 0;
}
__device__ __forceinline__ void mma_s8(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// (x, y) += (u, v), two sums per instruction
__device__ __forceinline__ void add2(float& x, float& y, float u, float v) {
  asm("{\n\t.reg .b64 o, w;\n\tmov.b64 o, {%0, %1};\n\tmov.b64 w, {%2, %3};\n\tadd.rn.f32x2 o, o, w;\n\tmov.b64 {%0, %1}, o;\n\t}"
      : "+f"(x), "+f"(y)
      : "f"(u), "f"(v));
}

// CT: cache; TQ: type of q and out; D: head dimensions, d filled up with zeros. HALF: up to eight rows, an operand's leading terms in
// rows 0 .. 7 of a 16-row tile and its second ones in rows 8 .. 15, so that one mma takes both and a thread has scores and outputs
// of one row instead of two; else sixteen rows. Every warp of a block takes tiles of keys of its own.
template <int CT, typename TQ, int D_, bool HALF_>
struct Cfg {
  static constexpr bool HALF = HALF_;
  static constexpr int D = D_, WK = 4, H = HALF ? 1 : 2;                 // warps of a block; rows of a thread
  static constexpr bool BF = CT == TREE_BF16, WIDE = CT == TREE_BF16 || CT == TREE_F16, E4M3 = CT == TREE_E4M3;
  static constexpr int ES = WIDE ? 2 : 1;
  static constexpr bool QF = std::is_same<TQ, float>::value, QB = std::is_same<TQ, __nv_bfloat16>::value;
  // q8 keys are operands as they are, of whole-number products; Q is three signed bytes of its row's largest element
  static constexpr bool I8 = CT == TREE_Q8;
  static constexpr int QT = I8 ? 3 : BF ? (QB ? 1 : QF ? 3 : 2) : (QF ? 2 : 1);   // terms of Q
  static constexpr int PT = BF ? (QF ? 3 : 2) : (QB ? 1 : 2);            // terms of P
  static constexpr int NQ = HALF ? (QT + 1) / 2 : QT, NP = HALF ? (PT + 1) / 2 : PT;   // operands of Q and P
  static constexpr int RB = 8 * H;                                       // rows of a block
  static constexpr int THREADS = 32 * WK;
  static constexpr int KT = WIDE ? 16 : 32;                              // keys of a tile
  static constexpr int STAGES = 3;
  static constexpr int BLOCKS = HALF ? 2 : 1;                            // of an SM, as far as registers go
  static constexpr int TILE = KT * D * ES;
  static constexpr int STAGE = 2 * TILE + (WIDE ? 0 : 2 * KT * 4);
  static constexpr int RING = STAGE * STAGES * WK;
  static constexpr int QS = I8 ? D / 32 : D / 16;                        // steps of the products over the dimensions
  // a row's reference maximum may lie this far below its maximum (in powers of two): outputs are rescaled less often. f32 results
  // keep the weights' bits instead
  static constexpr float SLACK = QF ? 0.f : 8.f;
  static constexpr int PEXP = QF ? 13 : 5;                               // f16 weights enter times 2^PEXP
  static constexpr int STATE = WK * RB * (D + 2) * 4;                    // (output, maximum, sum) of every warp
  static constexpr int SMEM = RING > STATE ? RING : STATE;
};

template <typename C>
__device__ __forceinline__ uint32_t k_chunk(int key, int chunk) {  // byte offset of a 16-byte chunk of a key's row in a tile
  constexpr int PER = C::D * C::ES / 16;
  if (C::WIDE) return (uint32_t)(key * PER + (chunk ^ (key & 7 & (PER - 1)))) * 16;
  return (uint32_t)(key * PER + (PER == 8 ? chunk ^ ((key & 1) << 2) : chunk)) * 16;
}
template <typename C>
__device__ __forceinline__ uint32_t v_chunk(int key, int chunk) {
  constexpr int PER = C::D * C::ES / 16;
  return (uint32_t)(key * PER + (chunk ^ (key & 7 & (PER - 1)))) * 16;
}

__device__ __forceinline__ bool sees(const TreeArgs& a, int64_t b, int row, int64_t j) {
  if (j < 0) return true;
  if (j >= a.rows) return false;
  return a.mask ? a.mask[b * a.ms[0] + row * a.ms[1] + j] != 0 : j <= row;
}

// Bit e: whether a row sees key key0 + e, of N <= 32. Sixteen bytes of the mask are asked for at once.
template <int N>
__device__ __forceinline__ uint32_t seen_of(const TreeArgs& a, int64_t b, int row, int64_t key0, int64_t keys, int64_t len) {
  const int64_t j0 = key0 - len;
  uint32_t bits = 0;
  if (!a.mask) {
#pragma unroll
    for (int e = 0; e < N; e++)
      if (key0 + e < keys && j0 + e <= row) bits |= 1u << e;
    return bits;
  }
  const uint8_t* const of = a.mask + b * a.ms[0] + row * a.ms[1];
#pragma unroll
  for (int e0 = 0; e0 < N; e0 += 16) {
    uint8_t m[16];
#pragma unroll
    for (int e = 0; e < 16; e++) {
      const int64_t j = j0 + e0 + e;
      m[e] = j < 0 ? 1 : 0;
      if (e0 + e < N && j >= 0 && j < a.rows) m[e] = of[j];
    }
#pragma unroll
    for (int e = 0; e < 16; e++)
      if (e0 + e < N && key0 + e0 + e < keys && m[e]) bits |= 1u << (e0 + e);
  }
  return bits;
}

// What a row's output is multiplied with, from the sum of its weights. Without weights it is zero where the row sees no key, and not a
// number where all its scores are minus infinity. LANES neighbours hold the same row and look for a key together.
template <int LANES>
__device__ __forceinline__ float over_sum(const TreeArgs& a, int64_t b, int row, int64_t len, int64_t keys, float sum) {
  if (sum != 0.f) return 1.f / sum;
  bool some = len > 0;
  if (!some) {
    const int lane = threadIdx.x & 31;
#pragma unroll 1
    for (int64_t key = lane % LANES; key < keys; key += LANES) some = some || sees(a, b, row, key - len);
    some = __any_sync(LANES == 32 ? 0xffffffffu : ((1u << LANES % 32) - 1) << (lane & ~(LANES - 1)), some);
  }
  return some ? __uint_as_float(0x7fc00000u) : 0.f;
}

template <int CT, typename TQ, int D, bool HALF>
__global__ void __launch_bounds__(Cfg<CT, TQ, D, HALF>::THREADS, Cfg<CT, TQ, D, HALF>::BLOCKS) tree_attention_kernel(const __grid_constant__ TreeArgs a) {
  using C = Cfg<CT, TQ, D, HALF>;
  using O = Op<C::BF>;
  constexpr int KT = C::KT, NT = D / 8, KS = D / 16, NK = KT / 8, WK = C::WK, H = C::H, NE = 2 * H;  // NE: a thread's entries of an n8 tile
  extern __shared__ __align__(128) uint8_t tree_shared[];
  __shared__ bool odd_query[C::RB];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  const int split = (int)blockIdx.x % a.splits;
  const int64_t pair = blockIdx.x / a.splits;
  const int64_t b = pair / a.kv_heads;
  const int kvh = (int)(pair - b * a.kv_heads);
  const int total_rows = a.rows * a.group;  // at most C::RB

  int64_t len = a.lengths[b];
  int64_t keys = 0;
  if (len >= 0) {
    len = len < a.cap ? len : a.cap;
    keys = len + a.rows < a.cap ? len + a.rows : a.cap;
  }
  const uint8_t* kb = a.k + b * a.kst[0] + kvh * a.kst[1];
  const uint8_t* vb = a.v + b * a.vst[0] + kvh * a.vst[1];
  const float* ksb = C::WIDE ? nullptr : a.ks + b * a.kss[0] + kvh * a.kss[1];
  const float* vsb = C::WIDE ? nullptr : a.vs + b * a.vss[0] + kvh * a.vss[1];

  // ---- tiles: a warp takes every (splits * WK)-th one ----
  const int tiles = (int)((keys + KT - 1) / KT);
  const int first = split * WK + warp, step = a.splits * WK;
  const uint32_t ring = smem_u32(tree_shared) + (uint32_t)(warp * C::STAGES * C::STAGE);
  constexpr int PER = D * C::ES / 16, ROWS = 32 / PER, COPIES = KT / ROWS;  // a thread's copies lie ROWS keys apart
  const int my_key = lane / PER, my_chunk = lane % PER;
  const bool my_dims = my_chunk < a.d * C::ES / 16;
  const uint8_t* const kp = kb + my_key * a.kst[2] + my_chunk * 16;
  const uint8_t* const vp = vb + my_key * a.vst[2] + my_chunk * 16;
  auto fetch = [&](int tile, int stage) {
    if (tile < tiles) {
      const uint32_t at = ring + (uint32_t)(stage * C::STAGE);
      const int64_t key0 = (int64_t)tile * KT;
      const uint8_t *ks = kp + key0 * a.kst[2], *vs = vp + key0 * a.vst[2];
      if (key0 + KT <= keys) {
#pragma unroll
        for (int i = 0; i < COPIES; i++) {
          cp16(at + k_chunk<C>(my_key + i * ROWS, my_chunk), my_dims ? ks : kb, my_dims);
          cp16(at + C::TILE + v_chunk<C>(my_key + i * ROWS, my_chunk), my_dims ? vs : vb, my_dims);
          ks += ROWS * a.kst[2], vs += ROWS * a.vst[2];
        }
      } else {
#pragma unroll 1
        for (int i = 0; i < COPIES; i++) {
          const bool live = my_dims && key0 + my_key + i * ROWS < keys;
          cp16(at + k_chunk<C>(my_key + i * ROWS, my_chunk), live ? ks + i * ROWS * a.kst[2] : kb, live);
          cp16(at + C::TILE + v_chunk<C>(my_key + i * ROWS, my_chunk), live ? vs + i * ROWS * a.vst[2] : vb, live);
        }
      }
      if (!C::WIDE) {
#pragma unroll
        for (int u = lane; u < 2 * KT; u += 32) {  // the keys' scales, then the values'
          const int64_t kk = key0 + (u & (KT - 1));
          const float* const of = u < KT ? ksb : vsb;
          cp4(at + 2 * C::TILE + u * 4, kk < keys ? of + kk : of, kk < keys);
        }
      }
    }
    cp_commit();
  };
  auto begin = [&] {
#pragma unroll
    for (int i = 0; i < C::STAGES - 1; i++) fetch(first + i * step, i);
  };
  begin();

  // ---- Q: this warp's rows, in the order in which keys' dimensions come out ----
  // element e (0 .. 3) of k16 step s at lane quarter t: 2-byte keys 16 s + 2 t + {0, 1, 8, 9}; 8-bit keys lie 16 bytes per lane
  uint32_t qf[C::NQ][C::QS][4];
  float mult[H];  // what a row's scores are multiplied with: log2(e) * scale / the row's factor
  {
    float x[H][KS][4];
#pragma unroll
    for (int h = 0; h < H; h++) {
      const int r = g + 8 * h;
      const bool live = r < total_rows;
      const int tr = live ? r / a.group : 0, gh = live ? r - tr * a.group : 0;
      const TQ* src = static_cast<const TQ*>(a.q) + b * a.qs[0] + tr * a.qs[1] + (int64_t)(kvh * a.group + gh) * a.qs[2];
      float most = 0.f, odd = 0.f;
#pragma unroll
      for (int s = 0; s < KS; s++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int dim = C::WIDE ? 16 * s + 2 * t + (e & 1) + 8 * (e >> 1) : s / 4 * 64 + t * 16 + s % 4 * 4 + e;
          x[h][s][e] = live && dim < a.d ? kv_float(src[dim]) : 0.f;
          most = fmaxf(most, fabsf(x[h][s][e]));
          odd = fmaf(x[h][s][e], 0.f, odd);
        }
      float mul = 1.f, inv = 1.f;
      if (!C::BF) {
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        if (C::I8) {
          // the largest element to 127 * 2^16: three signed bytes. A row that is not finite gets scores that are not numbers
          odd += __shfl_xor_sync(0xffffffffu, odd, 1);
          odd += __shfl_xor_sync(0xffffffffu, odd, 2);
          most = fminf(fmaxf(most, 1e-31f), 3.402823466e38f);  // (f32's largest)
          mul = odd == 0.f ? 127.f * 65536.f / most : 0.f, inv = odd == 0.f ? most / (127.f * 65536.f) : __uint_as_float(0x7fc00000u);
        } else {
          // the row's largest element to 2^8 .. 2^9; zeros, infinities and extremes of f32 keep a bounded factor
          int ex = (int)((__float_as_uint(most) >> 23) & 0xff);
          ex = ex < 20 ? 20 : ex > 250 ? 250 : ex;
          mul = __uint_as_float((uint32_t)(262 - ex) << 23), inv = __uint_as_float((uint32_t)(ex - 8) << 23);
        }
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
          for (int e = 0; e < 4; e++) x[h][s][e] *= mul;
      }
      mult[h] = a.scale * LOG2E * inv;
    }
    auto keep = [&](int n, int s, const uint32_t (&f)[4]) {
#pragma unroll
      for (int i = 0; i < 4; i++) qf[n][s][i] = f[i];
    };
    if (C::I8) {
#pragma unroll
      for (int s = 0; s < C::QS; s++) {
        uint32_t term[3][H][2] = {};  // [leading to last][row][step of four dimensions]
#pragma unroll
        for (int h = 0; h < H; h++)
#pragma unroll
          for (int w = 0; w < 2; w++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const int v = __float2int_rn(x[h][(2 * s + w) % KS][e]);
              const int low = (int)(signed char)v, above = (v - low) >> 8, mid = (int)(signed char)above, top = (above - mid) >> 8;
              term[0][h][w] |= (uint32_t)(top & 0xff) << (8 * e), term[1][h][w] |= (uint32_t)(mid & 0xff) << (8 * e);
              term[2][h][w] |= (uint32_t)(low & 0xff) << (8 * e);
            }
        if (C::HALF) {
          keep(0, s, {term[0][0][0], term[1][0][0], term[0][0][1], term[1][0][1]});
          keep(1 % C::NQ, s, {term[2][0][0], 0u, term[2][0][1], 0u});
        } else {
#pragma unroll
          for (int n = 0; n < 3; n++) keep(n % C::NQ, s, {term[n][0][0], term[n][H - 1][0], term[n][0][1], term[n][H - 1][1]});
        }
      }
    } else {
#pragma unroll
      for (int s = 0; s < KS; s++)
#pragma unroll
        for (int n = 0; n < C::NQ; n++) {
          uint32_t f[4] = {};
          f[0] = O::take(x[0][s][0], x[0][s][1]), f[2] = O::take(x[0][s][2], x[0][s][3]);
          if (!C::HALF || 2 * n + 1 < C::QT) f[1] = O::take(x[H - 1][s][0], x[H - 1][s][1]), f[3] = O::take(x[H - 1][s][2], x[H - 1][s][3]);
          keep(n, s % C::QS, f);
        }
    }
  }

  // ---- the running state ----
  float out[NT][NE], top[H], sum[H];
  int vex[H];  // 8-bit: exponent that the scales of the values a row sees are taken relative to; `out` is in units of 2^(vex - 127 - PEXP)
  // Values that are not finite: weight 0, or a weight's zero second term, times one is not a number. Where a result is not finite
  // the keys are gone through once more, with such entries left out of the products and added one by one. (Codes of q8 are finite.)
  constexpr bool ODD = CT != TREE_Q8;
  for (bool careful = false;; careful = true) {
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int e = 0; e < NE; e++) out[n][e] = 0.f;
#pragma unroll
    for (int h = 0; h < H; h++) top[h] = -INFINITY, sum[h] = 0.f, vex[h] = 30;
    int stage = 0;
    for (int tile = first; tile < tiles; tile += step) {
      cp_wait<C::STAGES - 2>();
      __syncwarp();
      {
        int ahead = stage + C::STAGES - 1;
        if (ahead >= C::STAGES) ahead -= C::STAGES;
        fetch(tile + (C::STAGES - 1) * step, ahead);
      }
      const uint32_t kt = ring + (uint32_t)(stage * C::STAGE), vt = kt + C::TILE, st = vt + C::TILE;
      if (++stage == C::STAGES) stage = 0;

      // S
      float sc[NK][NE];
      if constexpr (C::I8) {
        int acc[3][NK][4] = {};  // leading, second (not HALF: HALF has both in one), last terms
        uint4 raw[NK][D / 64];
#pragma unroll
        for (int j = 0; j < NK; j++)
#pragma unroll
          for (int h = 0; h < D / 64; h++) raw[j][h] = lds16(kt + k_chunk<C>(j * 8 + g, h * 4 + t));
#pragma unroll
        for (int s = 0; s < C::QS; s++)
#pragma unroll
          for (int n = 0; n < C::NQ; n++) {
#pragma unroll
            for (int j = 0; j < NK; j++) {
              const uint4 w = raw[j][s / 2];
              mma_s8(acc[n][j], qf[n][s], s & 1 ? w.z : w.x, s & 1 ? w.w : w.y);
            }
          }
#pragma unroll
        for (int j = 0; j < NK; j++)
#pragma unroll
          for (int e = 0; e < NE; e++) {
            const int lead = acc[0][j][e], mid = C::HALF ? acc[0][j][(e + 2) & 3] : acc[1][j][e], low = acc[C::NQ - 1][j][e];
            sc[j][e] = fmaf((float)lead, 65536.f, (float)(mid * 256 + low));
          }
      } else {
        float acc[NK][4] = {};
#pragma unroll
        for (int s = 0; s < KS; s++) {
          uint32_t kf[NK][2];
          if (C::WIDE) {
#pragma unroll
            for (int j = 0; j < NK; j += 2) {
              uint32_t r[4];
              const int key = j * 8 + (lane & 7) + ((lane >> 4) << 3);
              ldsm4(r, kt + k_chunk<C>(key, 2 * s + ((lane >> 3) & 1)));
              kf[j][0] = r[0], kf[j][1] = r[1], kf[j + 1][0] = r[2], kf[j + 1][1] = r[3];
            }
          } else {
#pragma unroll
            for (int j = 0; j < NK; j++) {
              uint32_t w;
              asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(kt + k_chunk<C>(j * 8 + g, s / 4 * 4 + t) + s % 4 * 4));
              widen<C::E4M3>(w, &kf[j][0], &kf[j][1]);
            }
          }
#pragma unroll
            for (int n = C::NQ - 1; n >= 0; n--) {
#pragma unroll
              for (int j = 0; j < NK; j++) O::mma(acc[j], qf[n][s % C::QS], kf[j][0], kf[j][1]);
            }
        }
#pragma unroll
          for (int j = 0; j < NK; j++)
#pragma unroll
            for (int e = 0; e < NE; e++) sc[j][e] = C::HALF ? acc[j][e] + acc[j][e + 4 - NE] : acc[j][e];
      }

      // An infinite key entry against a term of the query that is zero, or of the other sign, is no score. Such scores are
      // computed once more, entry by entry (in units that do not matter: what comes of an infinity is none or infinite).
      if constexpr (C::WIDE) {
        bool lost = false;
        if (careful) {
#pragma unroll
          for (int h = 0; h < H; h++)
            if (g + 8 * h < total_rows && !odd_query[g + 8 * h]) {
#pragma unroll
              for (int j = 0; j < NK; j++) lost = lost || !(fabsf(sc[j][2 * h]) <= INFINITY && fabsf(sc[j][2 * h + 1]) <= INFINITY);
            }
        }
        if (lost) {
#pragma unroll
          for (int h = 0; h < H; h++) {
            const int r = min(g + 8 * h, total_rows - 1), tr = r / a.group, gh = r - tr * a.group;
            if (odd_query[r]) continue;
            const TQ* const of = static_cast<const TQ*>(a.q) + b * a.qs[0] + tr * a.qs[1] + (int64_t)(kvh * a.group + gh) * a.qs[2];
#pragma unroll
            for (int j = 0; j < NK; j++)
#pragma unroll
              for (int e = 0; e < 2; e++)
                if (!(fabsf(sc[j][2 * h + e]) <= INFINITY)) {
                  float s = 0.f;
#pragma unroll 1
                  for (int dim = 0; dim < a.d && s == s; dim++) {
                    unsigned short bits;
                    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(bits) : "r"(kt + k_chunk<C>(j * 8 + 2 * t + e, dim / 8) + (uint32_t)(dim % 8 * 2)));
                    s = fmaf(kv_float(of[dim]), C::BF ? __bfloat162float(__ushort_as_bfloat16(bits)) : __half2float(__ushort_as_half(bits)), s);
                  }
                  sc[j][2 * h + e] = s;
                }
          }
        }
      }

      // scores in powers of two, masked
      const int64_t key0 = (int64_t)tile * KT;
      float vscale[C::WIDE ? 1 : NK][2];
      int ex[H];  // 8-bit: exponent of the largest scale of the values that a row sees
      if (!C::WIDE) {
        float most = 0.f;
#pragma unroll
        for (int j = 0; j < NK; j++)
#pragma unroll
          for (int e = 0; e < 2; e++) {
            vscale[C::WIDE ? 0 : j][e] = lds4(st + (uint32_t)(KT + j * 8 + 2 * t + e) * 4);
            most = fmaxf(most, vscale[C::WIDE ? 0 : j][e]);
            const float kscale = lds4(st + (uint32_t)(j * 8 + 2 * t + e) * 4);
#pragma unroll
              for (int h = 0; h < H; h++) sc[j][2 * h + e] *= kscale;
          }
        ex[0] = ex[H - 1] = (int)(__reduce_max_sync(0xffffffffu, __float_as_uint(most)) >> 23);
      }
      const bool tail = key0 + KT > len;
      uint32_t vis[H];
#pragma unroll
        for (int h = 0; h < H; h++) vis[h] = 0xffffffffu;
      if (tail) {
#pragma unroll
          for (int h = 0; h < H; h++) {
            const int r = g + 8 * h;
            const int tr = r < total_rows ? r / a.group : 0;
            uint32_t bits = 0;
#pragma unroll
            for (int i = 0; i < 2 * NK; i++) {
              const int64_t key = key0 + (i >> 1) * 8 + 2 * t + (i & 1);
              if (key < keys && sees(a, b, tr, key - len)) bits |= 1u << i;
            }
            vis[h] = bits;
            if (!C::WIDE) {
              // a scale that the row does not see would push its weights out of f16's range
              float most = 0.f;
#pragma unroll
              for (int i = 0; i < 2 * NK; i++) most = fmaxf(most, bits >> i & 1 ? vscale[C::WIDE ? 0 : i >> 1][i & 1] : 0.f);
              most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
              ex[h] = (int)(__float_as_uint(fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2))) >> 23);
            }
          }
      }
      float decay[H];  // what a row's `out` is multiplied with
      bool change = false;
#pragma unroll
        for (int h = 0; h < H; h++) {
          decay[h] = 1.f;
          if (!C::WIDE) {
            const int e = min(max(ex[h], 30), 254);
            if (e > vex[h]) decay[h] = ex2((float)(vex[h] - e)), vex[h] = e, change = true;
          }
        }
#pragma unroll
        for (int h = 0; h < H; h++) {
          // the maximum in powers of two; a score and its reference go through one fma, so that the score is not rounded before
          // the difference. Masked entries are -infinity by a choice, not by a product with a factor that may be zero
          float best = -INFINITY;
#pragma unroll
          for (int j = 0; j < NK; j++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
              const float s = sc[j][2 * h + e] * mult[h];
              best = fmaxf(best, !tail || vis[h] >> (2 * j + e) & 1 ? s : -INFINITY);
            }
          best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 1));
          best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 2));
          if (best > top[h] + C::SLACK || top[h] == -INFINITY) {
            if (best > -INFINITY) decay[h] *= ex2(top[h] - best), change = true;
            sum[h] *= ex2(top[h] - (best == -INFINITY ? 0.f : best));
            top[h] = best;
          }
          const float base = top[h] == -INFINITY ? 0.f : top[h];
          float part = 0.f;
#pragma unroll
          for (int j = 0; j < NK; j++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
              float p = ex2(fmaf(sc[j][2 * h + e], mult[h], -base));
              if (tail && !(vis[h] >> (2 * j + e) & 1)) p = 0.f;
              sc[j][2 * h + e] = p;
              part += p;
            }
          sum[h] += part;
        }
      if (__any_sync(0xffffffffu, change)) {
#pragma unroll
          for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < NE; e++) out[n][e] *= decay[e >> 1];
      }
      // weights as operands
      uint32_t pf[C::NP][NK / 2][4];
#pragma unroll
        for (int j = 0; j < NK; j++) {
          float w[NE];
#pragma unroll
          for (int e = 0; e < NE; e++) {
            const float pmul = C::BF ? 1.f : C::WIDE ? (float)(1 << C::PEXP) : __uint_as_float((uint32_t)(254 + C::PEXP - vex[e >> 1]) << 23);
            w[e] = sc[j][e] * pmul;
            if (!C::WIDE) {
              w[e] *= vscale[C::WIDE ? 0 : j][e & 1];
              if (tail && !(vis[e >> 1] >> (2 * j + (e & 1)) & 1)) w[e] = 0.f;  // the scale of a key that is not seen
            }
          }
#pragma unroll
          for (int n = 0; n < C::NP; n++) {
            pf[n][j / 2][(j & 1) * 2] = O::take(w[0], w[1]);
            pf[n][j / 2][(j & 1) * 2 + 1] = !C::HALF || 2 * n + 1 < C::PT ? O::take(w[NE - 2], w[NE - 1]) : 0u;
          }
        }
      bool odd = false;
      if (ODD && careful) {
        for (int u = lane; u < KT * PER; u += 32) {
          const uint4 w = lds16(vt + (uint32_t)u * 16);
          uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int i = 0; i < 4; i++) odd |= C::WIDE ? without_odd<C::BF>(x[i]) : without_nan(x[i]);
        }
        odd = __any_sync(0xffffffffu, odd);
      }
      // O += P V: products of the tile start from zero
      auto fold = [&](int n, const float (&u)[4]) {
#pragma unroll
        for (int e = 0; e < 4; e += 2) add2(out[n][e % NE], out[n][e % NE + 1], u[e], u[e + 1]);
      };
      if (C::WIDE) {
#pragma unroll
        for (int nb = 0; nb < NT / 2; nb++) {
          float u[2][4] = {};
#pragma unroll
          for (int kk = 0; kk < NK / 2; kk++) {
            uint32_t r[4];
            const int key = kk * 16 + (lane & 15);
            ldsm4t(r, vt + v_chunk<C>(key, 2 * nb + (lane >> 4)));
            if (odd) {
#pragma unroll
              for (int i = 0; i < 4; i++) without_odd<C::BF>(r[i]);
            }
#pragma unroll
              for (int n = C::NP - 1; n >= 0; n--) {
                O::mma(u[0], pf[n][kk], r[0], r[1]);
                O::mma(u[1], pf[n][kk], r[2], r[3]);
              }
          }
#pragma unroll
            for (int i = 0; i < 2; i++) fold(2 * nb + i, u[i]);
        }
      } else {
        // lane g has D / 8 consecutive dimensions of a key: n8 tile i is dimension g * D / 8 + i
        constexpr int WORDS = D / 32;  // words of a key per lane
        uint32_t x[NK / 2][4][WORDS];
#pragma unroll
        for (int kk = 0; kk < NK / 2; kk++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const int key = kk * 16 + 2 * t + (i & 1) + 8 * (i >> 1);
            if (WORDS == 4) {
              const uint4 w = lds16(vt + v_chunk<C>(key, g));
              x[kk][i][0] = w.x, x[kk][i][1] = w.y, x[kk][i][2 % WORDS] = w.z, x[kk][i][3 % WORDS] = w.w;
            } else {
              const uint2 w = lds8(vt + v_chunk<C>(key, g / 2) + (uint32_t)(g % 2 * 8));
              x[kk][i][0] = w.x, x[kk][i][1] = w.y;
            }
            if (ODD && odd) {
#pragma unroll
              for (int w = 0; w < WORDS; w++) without_nan(x[kk][i][w]);
            }
          }
#pragma unroll
        for (int w = 0; w < WORDS; w++) {
          float u[4][4] = {};
#pragma unroll
          for (int kk = 0; kk < NK / 2; kk++) {
            uint32_t r0[4], r1[4];
            widen_pairs<C::E4M3>(x[kk][0][w], x[kk][1][w], r0);
            widen_pairs<C::E4M3>(x[kk][2][w], x[kk][3][w], r1);
#pragma unroll
              for (int n = C::NP - 1; n >= 0; n--)
#pragma unroll
                for (int i = 0; i < 4; i++) O::mma(u[i], pf[n][kk], r0[i], r1[i]);
          }
#pragma unroll
            for (int i = 0; i < 4; i++) fold(w * 4 + i, u[i]);
        }
      }
      if (ODD && odd) {
        // the entries left out, to the rows that see their keys
#pragma unroll 1
        for (int key = 0; key < KT; key++) {
          const int j = key / 8, from = (lane & ~3) + (key & 7) / 2;
#pragma unroll
            for (int h = 0; h < H; h++) {
              // which of the two columns is a matter of the key: picked without indexing registers
              float p = 0.f;
              uint32_t seen = 0;
#pragma unroll
              for (int jj = 0; jj < NK; jj++)
                if (jj == j) p = key & 1 ? sc[jj][2 * h + 1] : sc[jj][2 * h], seen = vis[h] >> (2 * jj + (key & 1)) & 1;
              p = __shfl_sync(0xffffffffu, p, from), seen = __shfl_sync(0xffffffffu, seen, from);
#pragma unroll
              for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                  const int dim = C::WIDE ? n * 8 + 2 * t + e : (2 * t + e) * (D / 8) + n;
                  const uint32_t at = vt + v_chunk<C>(key, dim * C::ES / 16) + (uint32_t)(dim * C::ES % 16);
                  float val = 0.f;
                  if (C::WIDE) {
                    unsigned short bits;
                    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(bits) : "r"(at));
                    if ((bits & (C::BF ? 0x7f80u : 0x7c00u)) == (C::BF ? 0x7f80u : 0x7c00u))
                      val = C::BF ? __bfloat162float(__ushort_as_bfloat16(bits)) : __half2float(__ushort_as_half(bits));
                  } else {
                    uint32_t bits;
                    asm volatile("ld.shared.u8 %0, [%1];" : "=r"(bits) : "r"(at));
                    if ((bits & 0x7fu) == 0x7fu) val = __uint_as_float(0x7fc00000u);
                  }
                  if (seen && val != 0.f) out[n][2 * h + e] += p * val;
                }
            }
        }
      }
    }
    cp_wait<0>();
    if (!ODD || careful) break;
    bool finite = true;
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int e = 0; e < NE; e++) finite = finite && fabsf(out[n][e]) < INFINITY;
    if (!__syncthreads_or(!finite)) break;
    if (C::WIDE) {  // rows whose query is not finite are what they are
      for (int r = warp; r < total_rows; r += WK) {
        const int tr = r / a.group, gh = r - tr * a.group;
        const TQ* const of = static_cast<const TQ*>(a.q) + b * a.qs[0] + tr * a.qs[1] + (int64_t)(kvh * a.group + gh) * a.qs[2];
        bool odd = false;
        for (int dim = lane; dim < a.d; dim += 32) odd = odd || !(fabsf(kv_float(of[dim])) < INFINITY);
        odd = __any_sync(0xffffffffu, odd);
        if (lane == 0) odd_query[r] = odd;
      }
      __syncthreads();
    }
    begin();
  }
  // out in its own units again
  float unit[H];
#pragma unroll
    for (int h = 0; h < H; h++) unit[h] = C::BF ? 1.f : C::WIDE ? 1.f / (float)(1 << C::PEXP) : __uint_as_float((uint32_t)(vex[h] - C::PEXP) << 23);
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int e = 0; e < NE; e++) out[n][e] *= unit[e >> 1];
#pragma unroll
    for (int h = 0; h < H; h++) {
      sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
      sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);
    }
  __syncthreads();  // the ring becomes the states' place

  // ---- states of the warps, then of the cluster's blocks ----
  float* so = reinterpret_cast<float*>(tree_shared);          // [WK][RB][D]
  float* sm = so + WK * C::RB * D;                             // [WK][RB] (maximum, sum)
#pragma unroll
    for (int h = 0; h < H; h++) {
      const int r = g + 8 * h;
      float* to = so + (warp * C::RB + r) * D;
      if (C::WIDE) {
#pragma unroll
        for (int n = 0; n < NT; n++) *reinterpret_cast<float2*>(to + n * 8 + 2 * t) = make_float2(out[n][2 * h], out[n][2 * h + 1]);
      } else {
#pragma unroll
        for (int e = 0; e < 2; e++)
#pragma unroll
          for (int n = 0; n < NT; n += 4)
            *reinterpret_cast<float4*>(to + (2 * t + e) * (D / 8) + n) =
                make_float4(out[n][2 * h + e], out[n + 1][2 * h + e], out[n + 2][2 * h + e], out[n + 3][2 * h + e]);
      }
      if (t == 0) sm[(warp * C::RB + r) * 2] = top[h], sm[(warp * C::RB + r) * 2 + 1] = sum[h];
    }
  __syncthreads();
  // group states into the first one: a thread takes four dimensions of a row
  if (WK > 1) {
    float best[1];
    for (int i = threadIdx.x; i < total_rows * (D / 4); i += C::THREADS) {
      const int r = i / (D / 4), c = i % (D / 4) * 4;
      best[0] = -INFINITY;
#pragma unroll
      for (int w = 0; w < WK; w++) best[0] = fmaxf(best[0], sm[(w * C::RB + r) * 2]);
      const float base = best[0] == -INFINITY ? 0.f : best[0];
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < WK; w++) {
        const float f = ex2(sm[(w * C::RB + r) * 2] - base);
        const float4 x = *reinterpret_cast<const float4*>(so + (w * C::RB + r) * D + c);
        o.x += f * x.x, o.y += f * x.y, o.z += f * x.z, o.w += f * x.w;
      }
      *reinterpret_cast<float4*>(so + r * D + c) = o;
    }
    __syncthreads();
    for (int r = threadIdx.x; r < total_rows; r += C::THREADS) {
      float m = -INFINITY, l = 0.f;
#pragma unroll
      for (int w = 0; w < WK; w++) m = fmaxf(m, sm[(w * C::RB + r) * 2]);
#pragma unroll
      for (int w = 0; w < WK; w++) l += sm[(w * C::RB + r) * 2 + 1] * ex2(sm[(w * C::RB + r) * 2] - (m == -INFINITY ? 0.f : m));
      sm[r * 2] = m, sm[r * 2 + 1] = l;
    }
  }
  if (a.splits > 1)
    asm volatile("barrier.cluster.arrive;\n\tbarrier.cluster.wait;" ::: "memory");
  else
    __syncthreads();
  // a block of the cluster takes every splits-th piece of four dimensions
  const uint32_t so_at = smem_u32(so), sm_at = smem_u32(sm);
  for (int i = split * C::THREADS + threadIdx.x; i < total_rows * (D / 4); i += a.splits * C::THREADS) {
    const int r = i / (D / 4), c = i % (D / 4) * 4;
    float m = -INFINITY, l = 0.f;
    float o[4] = {};
    for (int p = 0; p < a.splits; p++) {
      uint32_t at_m, at_o;
      float pm, pl, x[4];
      asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at_m) : "r"(sm_at + (uint32_t)r * 8), "r"(p));
      asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at_o) : "r"(so_at + (uint32_t)(r * D + c) * 4), "r"(p));
      asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(pm), "=f"(pl) : "r"(at_m) : "memory");
      asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]) : "r"(at_o) : "memory");
      const float next = fmaxf(m, pm), base = next == -INFINITY ? 0.f : next;
      const float fa = ex2(m - base), fb = ex2(pm - base);
      l = l * fa + pl * fb;
#pragma unroll
      for (int e = 0; e < 4; e++) o[e] = o[e] * fa + x[e] * fb;
      m = next;
    }
    const int tr = r / a.group, gh = r - tr * a.group;
    TQ* to = static_cast<TQ*>(a.out) + ((b * a.rows + tr) * a.heads + (int64_t)kvh * a.group + gh) * a.d + c;
    const float inv = over_sum<D / 4>(a, b, tr, len, keys, l);
    if (c < a.d) {
#pragma unroll
      for (int e = 0; e < 4; e++) kv_store(o[e] * inv, to + e);
    }
  }
  if (a.splits > 1) asm volatile("barrier.cluster.arrive;\n\tbarrier.cluster.wait;" ::: "memory");  // others read this block's states
}

template <int CT, typename TQ, int D, bool HALF>
int run(TreeArgs a, cudaStream_t s) {
  using C = Cfg<CT, TQ, D, HALF>;
  auto kernel = tree_attention_kernel<CT, TQ, D, HALF>;
  if (ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), C::SMEM)) return 1;
  const int64_t pairs = a.batch * a.kv_heads;
  // blocks of a cluster: as many as leave all clusters running at once, at least a tile for each warp at full capacity
  const int splits = blocks_per_cluster<tree_attention_kernel<CT, TQ, D, HALF>, C::THREADS, C::SMEM>(pairs, a.cap / (C::WK * C::KT));
  a.splits = splits;
  DYN_CHECK(pairs * splits <= 0x7fffffff, "tree_attention: too many sequences for one call");
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(pairs * splits)), cfg.blockDim = dim3(C::THREADS);
  cfg.dynamicSmemBytes = C::SMEM, cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)splits, attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr, cfg.numAttrs = 1;
  DYN_CUDA(cudaLaunchKernelEx(&cfg, kernel, a));
  count_launch();
  return 0;
}

}  // namespace tree
}  // namespace dyn
