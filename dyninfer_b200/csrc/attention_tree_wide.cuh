// Tree attention of many rows (attention_tree.cuh states the operator) on the 5th-generation tensor cores.
//
// One block = 128 rows (tokens x query heads of one kv head), the 128 lanes of tensor memory, and a share of the keys in tiles of
// 64; the blocks of a cluster take the tiles in turn and merge their states through shared memory. Roles:
//   two streams of four softmax warps, a thread per row: they take a block's tiles in turn, each with a running (maximum, sum, output) of
//                     its own, so that the latencies and the exponentials of the one run beside the products of the other. A thread turns
//                     S into P (terms side by side, in place of S) and adds U = P V to its row's f32 sums.
//   4 filling warps   bring keys and values into shared memory as swizzled 16-bit tiles: 2-byte caches by asynchronous copies
//                     straight to their places, 8-bit ones by way of a ring of raw tiles, converted on the way.
//   an issuing warp per stream. Q (up to three terms) lies in tensor memory, beside S and U of the streams; an f32 query over a bf16
//                     cache has three terms of Q and P, whose columns leave room for one stream only.
// Scores, references, slack, terms and units are those of attention_tree.cuh. Where a result is not finite (weight 0 times
// an infinity in a key that a row does not see), such rows are computed once more one by one, without tensor cores.
// All waits are bounded; one that runs out leaves a code in the device's error word.
// 4 x 64 rows of 32 heads at 8192 over e4m3, bf16: 68 us, 27 % of the measured bf16 rate; 8 x 13 at 2048 over q8, f32 (two terms of Q and P): 40.
// A stream's tile takes 3800 (bf16) to 5000 cycles (f32): maximum 750, weights 1500, the wait for U 700 to 1000 and its fold 330 with
// f32; issue and latency bound it, the tensor pipe is a quarter busy.
#pragma once

#include <atomic>

#include "attention_tree.cuh"
#include "umma.cuh"

namespace dyn {
namespace tree {

constexpr int W_ROWS = 128, W_KEYS = 64, W_FILL = 128;
constexpr int W_BOX = W_KEYS * 128;  // bytes of 64 keys x 64 two-byte dimensions

template <int CT, typename TQ, int D_>
struct Wide {
  static constexpr int D = D_;
  static constexpr bool BF = CT == TREE_BF16, WIDE = CT == TREE_BF16 || CT == TREE_F16, E4M3 = CT == TREE_E4M3;
  static constexpr bool QF = std::is_same<TQ, float>::value, QB = std::is_same<TQ, __nv_bfloat16>::value;
  static constexpr int QT = BF ? (QB ? 1 : QF ? 3 : 2) : (QF ? 2 : 1), PT = BF ? (QF ? 3 : 2) : (QB ? 1 : 2);
  static constexpr float SLACK = QF ? 0.f : 8.f;
  static constexpr int PEXP = QF ? 13 : 5;
  static constexpr int NS = PT == 3 ? 1 : 2;   // streams
  // whole warpgroups, because registers are dealt out per group: the softmax threads of the streams, fillers, issuing warps
  static constexpr int SOFTMAX = NS * W_ROWS, THREADS = SOFTMAX + W_FILL + 128;
  // 512 threads start with 128 registers each, 384 with 168
  static constexpr int START = NS == 2 ? 128 : 168, MANY = NS == 2 ? (QB ? 168 : 200) : 232, FEW = NS == 2 ? (QB ? 88 : 56) : 136;
  static_assert(SOFTMAX * MANY + (THREADS - SOFTMAX) * FEW <= THREADS * START, "the groups' shares come out of the launch's registers");
  // bf16 results leave the output in tensor memory, where the products add it up: an accumulation is off by 2^-24 of the sum, toward zero,
  // which 2^-9 does not see before some ten thousand tiles; rows whose reference moves are rescaled there. With f16 operands (one
  // term of P) there is room for P beside S, and the next tile's S is made under the present one's exponentials.
  static constexpr bool STAYS = QB, BESIDE = STAYS && PT == 1;
  // tiles with keys that not every row sees in a loop of their own: 4 x 64 rows at 8192 over e4m3 67.7 us, in one loop 72.0. Results that are
  // folded have more code, of which two copies cost short contexts more (2 x 8 at 500 over q8, f32: 20.4, in one loop 19.2)
  static constexpr bool APART = STAYS && !WIDE;
  // tensor memory columns
  static constexpr int S_COLS = PT == 3 ? 96 : 64, P_COL = BESIDE ? 64 : 0, U_AT = BESIDE ? 96 : S_COLS;  // a stream: S, P, U
  static constexpr int STREAM = U_AT + D_, Q_COL = NS * STREAM;
  static_assert(Q_COL + QT * (D_ / 2) <= 512, "tensor memory has 512 columns");
  // products' descriptors: kind::f16, f32 accumulator, M = 128, N at bit 17; bf16 operands; B contiguous along N
  static constexpr uint32_t ID = (1u << 4) | (8u << 24) | (BF ? (1u << 7) | (1u << 10) : 0u);
  static constexpr uint32_t ID_S = ID | (64u >> 3 << 17), ID_U = ID | ((uint32_t)D_ >> 3 << 17) | (1u << 16);
  // shared memory: tiles (keys, then values), the values' and keys' scales, raw tiles
  static constexpr int TILE = 2 * D * W_KEYS * 2, TILES = WIDE ? 5 : 4;
  static constexpr int RAW = WIDE ? 0 : 2 * D * W_KEYS + 2 * W_KEYS * 4, RAWS = 3;
  static constexpr int PITCH = D + 4;  // floats of a row's final state
  static constexpr int BODY = TILE * TILES + RAW * RAWS;
  static_assert(NS * W_ROWS * PITCH * 4 <= BODY, "the final states take the tiles' place");
  // A block waits for its columns of tensor memory and then for its cluster, so no two blocks of that kind may share an SM: this
  // much shared memory leaves no room for another one of this kernel, nor for one of the other kernels that do both (77 KB and more)
  static constexpr int SMEM = BODY + 1024 > 152 * 1024 ? BODY + 1024 : 152 * 1024;
  static_assert(SMEM + 1024 + 78 * 1024 > 228 * 1024 && SMEM <= 220 * 1024, "see above");
};

// B operand contiguous along N, 128-byte swizzle: a 128-byte row per K element with 64 elements of N; the next 64 a box further
__device__ __forceinline__ uint64_t wide_desc_mn(uint32_t at) {
  return (uint64_t)((at >> 4) & 0x3fff) | ((uint64_t)(W_BOX >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void wide_st8(uint32_t addr, const uint32_t (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}
// (x, y) * (u, v), (x, y) * (u, u) - (v, v): two per instruction
__device__ __forceinline__ void mul2(float& x, float& y, float u, float v) {
  asm("{\n\t.reg .b64 o, w;\n\tmov.b64 o, {%0, %1};\n\tmov.b64 w, {%2, %3};\n\tmul.rn.f32x2 o, o, w;\n\tmov.b64 {%0, %1}, o;\n\t}"
      : "+f"(x), "+f"(y)
      : "f"(u), "f"(v));
}
__device__ __forceinline__ void fms2(float& x, float& y, float u, float v) {
  asm("{\n\t.reg .b64 o, w, z;\n\tmov.b64 o, {%0, %1};\n\tmov.b64 w, {%2, %2};\n\tmov.b64 z, {%3, %3};\n\tfma.rn.f32x2 o, o, w, z;\n\tmov.b64 {%0, %1}, o;\n\t}"
      : "+f"(x), "+f"(y)
      : "f"(u), "f"(-v));
}
__device__ __forceinline__ uint32_t box_chunk(int key, int chunk) {  // a 16-byte chunk (8 dimensions) of a key in a tile
  return (uint32_t)((chunk >> 3) * W_BOX + key * 128 + (((chunk & 7) ^ (key & 7)) << 4));
}

template <int CT>
__device__ __forceinline__ float cached(const uint8_t* row, const float* scale, int dim) {  // one entry as a number
  if (CT == TREE_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(row)[dim]);
  if (CT == TREE_F16) return __half2float(reinterpret_cast<const __half*>(row)[dim]);
  if (CT == TREE_Q8) return (float)(int)(signed char)row[dim] * *scale;
  return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)row[dim], __NV_E4M3))) * *scale;
}

template <int CT, typename TQ, int D>
__global__ void __launch_bounds__(Wide<CT, TQ, D>::THREADS, 1) tree_attention_wide_kernel(const __grid_constant__ TreeArgs a, int* error) {
  using C = Wide<CT, TQ, D>;
  using O = Op<C::BF>;
  extern __shared__ uint8_t wide_shared[];
  __shared__ uint64_t kv_full[C::TILES], kv_free[C::TILES], q_full, s_full[C::NS], s_free[C::NS], p_full[C::NS], u_full[C::NS];
  __shared__ uint32_t tmem_base_s;
  __shared__ int s_abort;
  __shared__ __align__(16) float kscale[C::WIDE ? 1 : C::TILES][W_KEYS], vscale[C::WIDE ? 1 : C::TILES][W_KEYS];  // read by fours
  __shared__ int vexp[C::TILES][4];                           // exponents of the tile's largest value scale, of four filling warps
  __shared__ float s_mult[W_ROWS];                            // what a row's scores are multiplied with
  __shared__ __align__(16) float s_state[C::NS][W_ROWS][2];   // (maximum, sum), read by twos
  uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(wide_shared) + 1023) & ~uintptr_t(1023));
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const int split = (int)blockIdx.x % a.splits;
  const int64_t pair = blockIdx.x / a.splits;
  const int64_t b = pair / a.kv_heads;
  const int kvh = (int)(pair - b * a.kv_heads);
  const int row0 = blockIdx.y * W_ROWS, live_rows = min(W_ROWS, a.rows * a.group - row0);
  const int live_warps = (live_rows + 31) / 32;  // of a stream

  int64_t len = a.lengths[b], keys = 0;
  if (len >= 0) {
    len = len < a.cap ? len : a.cap;
    keys = len + a.rows < a.cap ? len + a.rows : a.cap;
  }
  const uint8_t* const kb = a.k + b * a.kst[0] + kvh * a.kst[1];
  const uint8_t* const vb = a.v + b * a.vst[0] + kvh * a.vst[1];
  const float* const ksb = C::WIDE ? nullptr : a.ks + b * a.kss[0] + kvh * a.kss[1];
  const float* const vsb = C::WIDE ? nullptr : a.vs + b * a.vss[0] + kvh * a.vss[1];
  const int tiles = (int)((keys + W_KEYS - 1) / W_KEYS);
  const int mine = split < tiles ? (tiles - split + a.splits - 1) / a.splits : 0;

  if (tid == 0) {
    s_abort = 0;
    for (int i = 0; i < C::TILES; i++) mbar_init(kv_full + i, W_FILL), mbar_init(kv_free + i, 1);
    for (int i = 0; i < C::NS; i++) mbar_init(s_full + i, 1), mbar_init(s_free + i, live_warps), mbar_init(p_full + i, live_warps), mbar_init(u_full + i, 1);
    mbar_init(&q_full, C::NS == 2 && live_rows <= 64 ? 2 * live_warps : live_warps);
    mbar_fence_init();
  }
  constexpr int ISSUING = (C::SOFTMAX + W_FILL) / 32;  // the first issuing warp
  if (warp == ISSUING) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_s)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base_s;
  auto wait = [&](uint64_t* bar, unsigned parity, int code) {
    if (!mbar_wait_bounded(bar, parity, TG_SPINS, &s_abort) && !s_abort) s_abort = code;
  };

  float* const so = reinterpret_cast<float*>(smem);  // the final states, in the tiles' place
  if (warp < C::SOFTMAX / 32) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::MANY));
    // up to 64 rows stand in the lanes a second time, for the second stream, so that its warps are on the other half of the SM
    const bool twice = C::NS == 2 && live_rows <= 64;
    const int stream = warp / 4, row = ((warp & 3) * 32 + lane) - (twice ? 64 * stream : 0);
    const bool holds = (row & ~31) >= 0 && (row & ~31) < live_rows, working = holds && mine;
    const uint32_t tlane = (uint32_t)((warp & 3) * 32) << 16;
    const int row_index = row0 + max(0, min(row, live_rows - 1)), tr = row_index / a.group, gh = row_index - tr * a.group;
    const TQ* const query = static_cast<const TQ*>(a.q) + b * a.qs[0] + tr * a.qs[1] + (int64_t)(kvh * a.group + gh) * a.qs[2];
    if (working && (stream == 0 || twice)) {
      // ---- Q into tensor memory ----
      float x[D];
      constexpr int N = 16 / sizeof(TQ);
      // 16 bytes at a time where the rows are aligned (whole pieces are in or out: d is a multiple of 16 dimensions)
      if (((reinterpret_cast<uintptr_t>(a.q) | (a.qs[0] | a.qs[1] | a.qs[2]) * sizeof(TQ)) & 15) == 0) {
#pragma unroll
        for (int d = 0; d < D; d += N) {
          uint4 w = make_uint4(0, 0, 0, 0);
          if (d < a.d) w = *reinterpret_cast<const uint4*>(query + d);
          const TQ* const e = reinterpret_cast<const TQ*>(&w);
#pragma unroll
          for (int j = 0; j < N; j++) x[d + j] = kv_float(e[j]);
        }
      } else {
#pragma unroll
        for (int d = 0; d < D; d++) x[d] = d < a.d ? kv_float(query[d]) : 0.f;
      }
      float mul = 1.f, inv = 1.f;
      if (!C::BF) {
        float most = 0.f;
#pragma unroll
        for (int d = 0; d < D; d++) most = fmaxf(most, fabsf(x[d]));
        int ex = (int)((__float_as_uint(most) >> 23) & 0xff);
        ex = ex < 20 ? 20 : ex > 250 ? 250 : ex;
        mul = __uint_as_float((uint32_t)(262 - ex) << 23), inv = __uint_as_float((uint32_t)(ex - 8) << 23);
      }
      s_mult[row] = fmaxf(a.scale * LOG2E * inv, 1.2e-38f);  // above zero: -infinity stays itself
      __syncwarp();
#pragma unroll
      for (int s = 0; s < D / 16; s++) {
#pragma unroll
        for (int e = 0; e < 16; e++) x[16 * s + e] *= mul;
#pragma unroll
        for (int n = 0; n < C::QT; n++) {
          uint32_t f[8];
#pragma unroll
          for (int e = 0; e < 8; e++) f[e] = O::take(x[16 * s + 2 * e], x[16 * s + 2 * e + 1]);
          wide_st8(tmem + tlane + C::Q_COL + n * (D / 2) + s * 8, f);
        }
      }
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full);
    }
    // ---- softmax ----
    float out[D], top = -INFINITY, sum = 0.f, mult = 0.f;
    int vex = 30;  // 8-bit: exponent that the scales of the values that the row sees are taken relative to; `out` is in units of 2^(vex - 127 - PEXP)
#pragma unroll
    for (int d = 0; d < D; d++) out[d] = 0.f;
    if (working) {
      wait(&q_full, 0, 9);
      mult = s_mult[row];
    }
    const uint32_t s_at = tmem + tlane + (uint32_t)(stream * C::STREAM), p_at = s_at + C::P_COL, u_at = s_at + C::U_AT;
    auto add_up = [&] {  // U
#pragma unroll
      for (int c = 0; c < D / 16; c += 2) {
        uint32_t u[2][16];
        tmem_ld16(u_at + 16u * c, u[0]);
        tmem_ld16(u_at + 16u * c + 16u, u[1]);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
        for (int e = 0; e < 32; e += 2)
          add2(out[16 * c + e], out[16 * c + e + 1], __uint_as_float(u[e >> 4][e & 15]), __uint_as_float(u[e >> 4][(e & 15) + 1]));
      }
    };
    int buf = stream;
    unsigned phase = 0, parity = 0;
    // tile i; `tail`: with keys that not every row sees
    auto take = [&](int i, int64_t key0, auto tail) {
      uint32_t vis[2] = {0xffffffffu, 0xffffffffu};
      // 8-bit: exponent of the largest scale of the values that the row sees. A scale that it does not see would push its weights out of f16's range
      int seen_ex = 30;
      if (tail) {
#pragma unroll
        for (int h = 0; h < 2; h++) vis[h] = seen_of<32>(a, b, tr, key0 + 32 * h, keys, len);
        if (!C::WIDE) {
          wait(kv_full + buf, phase, 2);
          float most = 0.f;
#pragma unroll(C::APART ? W_KEYS / 4 : 2)
          for (int e = 0; e < W_KEYS; e += 4) {
            const float4 v4 = *reinterpret_cast<const float4*>(&vscale[C::WIDE ? 0 : buf][e]);
            const uint32_t of4 = (e < 32 ? vis[0] : vis[1]) >> (e & 31);
            most = fmaxf(fmaxf(most, of4 & 1 ? v4.x : 0.f), fmaxf(of4 & 2 ? v4.y : 0.f, fmaxf(of4 & 4 ? v4.z : 0.f, of4 & 8 ? v4.w : 0.f)));
          }
          seen_ex = min(max((int)(__float_as_uint(most) >> 23), 30), 254);
        }
      }
      if (!C::WIDE) wait(kv_full + buf, phase, 2);  // for the scales
      wait(s_full + stream, parity, 1);
      __syncwarp();
      tc_fence_after();
      float decay = 1.f;
      if (!C::WIDE) {
        int ex = max(vexp[buf][2], vexp[buf][3]);
        if (tail) ex = seen_ex;
        if (ex > vex) decay = ex2((float)(vex - ex)), vex = ex;
      }
      const float pmul = C::BF ? 1.f : C::WIDE ? (float)(1 << C::PEXP) : __uint_as_float((uint32_t)(254 + C::PEXP - vex) << 23);
      // half of a tile's scores, in the row's units; -infinity for keys that are not seen
      auto half = [&](int h, float (&x)[32]) {
        uint32_t raw[2][16];
        tmem_ld16(s_at + 32u * h, raw[0]);
        tmem_ld16(s_at + 32u * h + 16u, raw[1]);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
        for (int e = 0; e < 32; e++) x[e] = __uint_as_float(raw[e >> 4][e & 15]);
        if (!C::WIDE) {
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            const float4 k4 = *reinterpret_cast<const float4*>(&kscale[C::WIDE ? 0 : buf][32 * h + e]);
            mul2(x[e], x[e + 1], k4.x, k4.y);
            mul2(x[e + 2], x[e + 3], k4.z, k4.w);
          }
        }
        if (tail) {
#pragma unroll
          for (int e = 0; e < 32; e++)
            if (!(vis[h] >> e & 1)) x[e] = -INFINITY;
        }
      };
      float s0 = 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;
      // half of a tile's weights into their place as operands
      auto weights = [&](int h, float* x, float base) {
#pragma unroll
        for (int c = 0; c < 2; c++) {
          float* const w = x + 16 * c;
#pragma unroll
          for (int e = 0; e < 16; e += 2) {
            fms2(w[e], w[e + 1], mult, base);
            w[e] = ex2(w[e]), w[e + 1] = ex2(w[e + 1]);
            if (e & 2) add2(s2, s3, w[e], w[e + 1]);
            else add2(s0, s1, w[e], w[e + 1]);
          }
#pragma unroll
          for (int e = 0; e < 16; e += 4) {
            if (C::WIDE) {
              if (!C::BF) mul2(w[e], w[e + 1], pmul, pmul), mul2(w[e + 2], w[e + 3], pmul, pmul);
            } else {
              float4 v4 = *reinterpret_cast<const float4*>(&vscale[C::WIDE ? 0 : buf][32 * h + 16 * c + e]);
              mul2(v4.x, v4.y, pmul, pmul);
              mul2(v4.z, v4.w, pmul, pmul);
              mul2(w[e], w[e + 1], v4.x, v4.y);
              mul2(w[e + 2], w[e + 3], v4.z, v4.w);
            }
          }
          if (!C::WIDE && tail) {  // the scale of a key that is not seen may be anything
#pragma unroll
            for (int e = 0; e < 16; e++)
              if (!(vis[h] >> (16 * c + e) & 1)) w[e] = 0.f;
          }
#pragma unroll
          for (int n = 0; n < C::PT; n++) {
            uint32_t f[8];
#pragma unroll
            for (int e = 0; e < 8; e++) f[e] = O::take(w[2 * e], w[2 * e + 1]);
            wide_st8(C::BESIDE ? p_at + 16u * h + 8u * c : s_at + (n < 2 ? 32u * h + 16u * c + 8u * n : 64u + 16u * h + 8u * c), f);
          }
        }
      };
      float best = -INFINITY;
      auto reference = [&] {  // what the row's scores are taken relative to
        best *= mult;         // which is above zero
        if (best > top + C::SLACK || top == -INFINITY) {
          const float f = ex2(top - (best == -INFINITY ? 0.f : best));
          decay *= f, sum *= f, top = best;
        }
        return top == -INFINITY ? 0.f : top;
      };
      if constexpr (C::STAYS) {
        float x[64];
        half(0, reinterpret_cast<float(&)[32]>(x[0]));
        half(1, reinterpret_cast<float(&)[32]>(x[32]));
        if (C::BESIDE) {  // S may be overwritten
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(s_free + stream);
        }
        float m[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
        for (int e = 4; e < 64; e++) m[e & 3] = fmaxf(m[e & 3], x[e]);
        best = fmaxf(best, fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])));
        const float base = reference();
        const bool moved = __any_sync(0xffffffffu, decay != 1.f);
        if (i > stream && (C::BESIDE || moved)) {  // the products before are done with P and U
          wait(u_full + stream, parity ^ 1u, 3);
          __syncwarp();
          tc_fence_after();
          if (moved) {
#pragma unroll 1
            for (int c = 0; c < D; c += 16) {
              uint32_t u[16];
              tmem_ld16(u_at + c, u);
              asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
              for (int e = 0; e < 16; e++) u[e] = __float_as_uint(__uint_as_float(u[e]) * decay);
              tmem_st16(u_at + c, u);
            }
          }
        }
        weights(0, x, base);
        weights(1, x + 32, base);
        sum += (s0 + s1) + (s2 + s3);
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full + stream);
      } else {
#pragma unroll
        for (int h = 0; h < 2; h++) {
          float x[32];
          half(h, x);
          float m0 = x[0], m1 = x[1];
#pragma unroll
          for (int e = 2; e < 32; e += 2) m0 = fmaxf(m0, x[e]), m1 = fmaxf(m1, x[e + 1]);
          best = fmaxf(best, fmaxf(m0, m1));
        }
        const float base = reference();
        if (__any_sync(0xffffffffu, decay != 1.f)) {
#pragma unroll
          for (int d = 0; d < D; d += 2) mul2(out[d], out[d + 1], decay, decay);
        }
#pragma unroll
        for (int h = 0; h < 2; h++) {
          float x[32];
          half(h, x);
          weights(h, x, base);
        }
        sum += (s0 + s1) + (s2 + s3);
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full + stream);
        wait(u_full + stream, parity, 3);
        __syncwarp();
        tc_fence_after();
        add_up();
        tc_fence_before();
      }
      parity ^= 1u;
      buf += C::NS;
      if (buf >= C::TILES) buf -= C::TILES, phase ^= 1u;
    };
    int i = stream;
    auto first_key = [&] { return ((int64_t)split + (int64_t)i * a.splits) * W_KEYS; };
    if constexpr (C::APART) {
#pragma unroll 1
      for (; i < mine && working && first_key() + W_KEYS <= len; i += C::NS) take(i, first_key(), std::false_type{});
#pragma unroll 1
      for (; i < mine && working; i += C::NS) take(i, first_key(), std::true_type{});
    } else {
#pragma unroll 1
      for (; i < mine && working; i += C::NS) take(i, first_key(), first_key() + W_KEYS > len);
    }
    if (C::STAYS && working && stream < mine) {
      wait(u_full + stream, parity ^ 1u, 3);
      __syncwarp();
      tc_fence_after();
      add_up();
    }
    bool fine = true;
    const float unit = C::BF ? 1.f : C::WIDE ? 1.f / (float)(1 << C::PEXP) : __uint_as_float((uint32_t)(vex - C::PEXP) << 23);
#pragma unroll
    for (int d = 0; d < D; d++) {
      out[d] *= unit;
      fine = fine && fabsf(out[d]) < INFINITY;
    }
    fine = fine || row < 0 || row >= live_rows;
    __syncwarp();
    __syncthreads();  // all tiles have been read
    if (working && !fine) {
      // ---- one by one: this thread's row over this stream's keys ----
      top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int d = 0; d < D; d++) out[d] = 0.f;
#pragma unroll 1
      for (int i = stream; i < mine; i += C::NS) {
        const int64_t key0 = ((int64_t)split + (int64_t)i * a.splits) * W_KEYS;
#pragma unroll 1
        for (int e = 0; e < W_KEYS && key0 + e < keys; e++) {
          if (!sees(a, b, tr, key0 + e - len)) continue;
          const uint8_t *const k = kb + (key0 + e) * a.kst[2], *const v = vb + (key0 + e) * a.vst[2];
          float s = 0.f;
#pragma unroll 4
          for (int d = 0; d < a.d; d++) s = fmaf(kv_float(query[d]), cached<CT>(k, ksb + key0 + e, d), s);
          s *= a.scale * LOG2E;
          if (!(s <= top)) {  // the maximum moves (or the score is not a number)
            const float f = s > -INFINITY ? ex2(top - s) : 1.f;
            sum *= f;
#pragma unroll
            for (int d = 0; d < D; d++) out[d] *= f;
            top = fmaxf(top, s);
          }
          const float p = ex2(s - (top == -INFINITY ? 0.f : top));
          sum += p;
#pragma unroll
          for (int d = 0; d < D; d++)
            if (d < a.d) out[d] = fmaf(p, cached<CT>(v, vsb + key0 + e, d), out[d]);
        }
      }
    }
    if (s_abort) {  // products still under way land before their memory is used again
      const long long t0 = clock64();
      while (clock64() - t0 < (1LL << 22)) {
      }
    }
    __syncwarp();
    if (holds) {
      float* const to = so + (stream * W_ROWS + row) * C::PITCH;
#pragma unroll
      for (int d = 0; d < D; d += 4) *reinterpret_cast<float4*>(to + d) = make_float4(out[d], out[d + 1], out[d + 2], out[d + 3]);
      s_state[stream][row][0] = top, s_state[stream][row][1] = sum;
    }
    __syncwarp();
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::FEW));
  } else if (warp < ISSUING) {
    // ---- filling ----
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::FEW));
    const int ft = tid - C::SOFTMAX, fw = ft / 32;
    constexpr int PER = C::WIDE ? D / 8 : D / 16;  // 16-byte pieces of a cached row
    constexpr int COPIES = W_KEYS * PER / W_FILL, ROWS = W_FILL / PER;
    // 8-bit: eight lanes have four pieces of two keys, whose places in a tile are in different banks
    const int key_l = C::WIDE || D == 64 ? ft / PER : ft / 16 * 2 + (ft >> 2 & 1), piece = C::WIDE || D == 64 ? ft % PER : (ft & 3) + (ft >> 1 & 4);
    const bool my_dims = piece * 16 < a.d * (C::WIDE ? 2 : 1);
    // this thread's pieces of a tile lie ROWS keys apart, in the cache and in shared memory
    const uint32_t to0 = C::WIDE ? box_chunk(key_l, piece) : (uint32_t)(key_l * D + (D == 128 ? piece ^ (key_l & 1) << 2 : piece) * 16);
    constexpr uint32_t TO_STEP = C::WIDE ? ROWS * 128 : ROWS * D, TO_VALUES = C::WIDE ? C::TILE / 2 : D * W_KEYS;
    const uint32_t tiles_at = smem_u32(smem), raw_at = tiles_at + (uint32_t)(C::TILES * C::TILE);
    const uint8_t *k_from = kb + ((int64_t)split * W_KEYS + key_l) * a.kst[2] + piece * 16, *v_from = vb + ((int64_t)split * W_KEYS + key_l) * a.vst[2] + piece * 16;
    const int64_t k_tile = (int64_t)a.splits * W_KEYS * a.kst[2], v_tile = (int64_t)a.splits * W_KEYS * a.vst[2];
    const int64_t k_step = ROWS * a.kst[2], v_step = ROWS * a.vst[2];
    uint32_t copy_at = C::WIDE ? tiles_at : raw_at;  // of the next tile that is asked for
    int copy_place = 0;
    auto copy = [&](int i) {  // tile i of this block's, in order: into its place, or into the raw ring
      if (i < mine) {
        const int64_t key0 = ((int64_t)split + (int64_t)i * a.splits) * W_KEYS;
        if (key0 + W_KEYS <= keys) {
#pragma unroll
          for (int j = 0; j < COPIES; j++) {
            cp16(copy_at + to0 + j * TO_STEP, my_dims ? k_from + j * k_step : kb, my_dims);
            cp16(copy_at + TO_VALUES + to0 + j * TO_STEP, my_dims ? v_from + j * v_step : vb, my_dims);
          }
        } else {
#pragma unroll 1
          for (int j = 0; j < COPIES; j++) {
            const bool live = my_dims && key0 + key_l + j * ROWS < keys;
            cp16(copy_at + to0 + j * TO_STEP, live ? k_from + j * k_step : kb, live);
            cp16(copy_at + TO_VALUES + to0 + j * TO_STEP, live ? v_from + j * v_step : vb, live);
          }
        }
        if (!C::WIDE) {
          const int64_t kk = key0 + (ft & (W_KEYS - 1));
          const float* const of = ft < W_KEYS ? ksb : vsb;
          cp4(copy_at + 2 * D * W_KEYS + ft * 4, kk < keys ? of + kk : of, kk < keys);
        }
        k_from += k_tile, v_from += v_tile;
        copy_at += C::WIDE ? C::TILE : C::RAW;
        if (++copy_place == (C::WIDE ? C::TILES : C::RAWS)) copy_place = 0, copy_at = C::WIDE ? tiles_at : raw_at;
      }
      cp_commit();
    };
    constexpr int AHEAD = C::WIDE ? C::TILES - 2 : C::RAWS - 1;  // copies under way
    // a place is free when the products of the tile before in it are done
    auto free_place = [&](int i) {
      if (i >= C::TILES && i < mine) wait(kv_free + i % C::TILES, ((i / C::TILES) - 1) & 1, 4);
    };
    for (int i = 0; i < AHEAD; i++) copy(i);
#pragma unroll 1
    for (int i = 0; i < mine; i++) {
      if (C::WIDE) {
        cp_wait<AHEAD - 1>();
      } else {
        cp_wait<AHEAD - 1>();
        asm volatile("bar.sync 5, %0;" ::"n"(W_FILL) : "memory");  // everybody's copies are there, and the oldest raw tile is done with
        copy(i + AHEAD);
        free_place(i);
        const int to = i % C::TILES;
        const uint32_t raw = raw_at + (uint32_t)(i % C::RAWS * C::RAW);
        // dimensions 16 piece .. of this thread's keys: two pieces of eight, the same places in every eighth row
        uint8_t* const tile = smem + to * C::TILE;
        const uint32_t at0 = box_chunk(key_l, 2 * piece), at1 = box_chunk(key_l, 2 * piece + 1);
#pragma unroll
        for (int kv = 0; kv < 2; kv++) {
          uint4 w[COPIES];
#pragma unroll
          for (int j = 0; j < COPIES; j++) w[j] = lds16(raw + kv * TO_VALUES + to0 + j * TO_STEP);
#pragma unroll
          for (int j = 0; j < COPIES; j++) {
            uint4 f[2];
            widen<C::E4M3>(w[j].x, &f[0].x, &f[0].y), widen<C::E4M3>(w[j].y, &f[0].z, &f[0].w);
            widen<C::E4M3>(w[j].z, &f[1].x, &f[1].y), widen<C::E4M3>(w[j].w, &f[1].z, &f[1].w);
            *reinterpret_cast<uint4*>(tile + kv * (C::TILE / 2) + at0 + j * ROWS * 128) = f[0];
            *reinterpret_cast<uint4*>(tile + kv * (C::TILE / 2) + at1 + j * ROWS * 128) = f[1];
          }
        }
        const float scale = lds4(raw + 2 * D * W_KEYS + ft * 4);
        if (ft < W_KEYS) kscale[C::WIDE ? 0 : to][ft] = scale;
        else vscale[C::WIDE ? 0 : to][ft - W_KEYS] = scale;
        int ex = (int)(__reduce_max_sync(0xffffffffu, scale > 0.f ? __float_as_uint(scale) : 0u) >> 23);  // NaN compares false
        ex = min(max(ex, 30), 254);
        if (lane == 0) vexp[to][fw] = fw < 2 ? 30 : ex;
      }
      fence_async_smem();
      mbar_arrive(kv_full + i % C::TILES);
      if (C::WIDE) {
        // behind the arrival: the products of the tile that is waited for may come after this one's scores
        free_place(i + AHEAD);
        copy(i + AHEAD);
      }
    }
    cp_wait<0>();
    __syncthreads();
  } else {
    // ---- issuing ----
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::FEW));
    // the reductions only bring what every lane has into uniform registers, where the products' operands come from
    const int stream = warp - ISSUING, n_tiles = (int)__reduce_max_sync(0xffffffffu, (unsigned)mine);
    const uint32_t tm = __reduce_max_sync(0xffffffffu, tmem), at = __reduce_max_sync(0xffffffffu, smem_u32(smem));
    const uint32_t s_col = tm + (uint32_t)(stream * C::STREAM), p_col = s_col + C::P_COL, u_col = s_col + C::U_AT;
    const uint64_t k_desc = umma_desc(at), v_desc = wide_desc_mn(at + C::TILE / 2);
    int buf = stream, k_buf = stream;  // of the values and of the keys that come next
    unsigned k_phase = 0, parity = 0;
    auto scores = [&] {
      wait(kv_full + k_buf, k_phase, 5);
      tc_fence_after();
      const uint64_t k = k_desc + (uint64_t)(k_buf * (C::TILE >> 4));
      if (elect_one()) {
#pragma unroll
        for (int n = C::QT - 1; n >= 0; n--)  // the small terms first
#pragma unroll
          for (int s = 0; s < D / 16; s++)
            umma_f16_ts(s_col, tm + C::Q_COL + n * (D / 2) + 8u * s, k + (uint64_t)((s >> 2) * (W_BOX >> 4) + 2 * (s & 3)), C::ID_S,
                        n == C::QT - 1 && s == 0 ? 0u : 1u);
        umma_commit(s_full + stream);
      }
      __syncwarp();
      k_buf += C::NS;
      if (k_buf >= C::TILES) k_buf -= C::TILES, k_phase ^= 1u;
    };
    if (stream < C::NS && stream < n_tiles) {
      wait(&q_full, 0, 6);
      scores();
#pragma unroll 1
      for (int i = stream; i < n_tiles; i += C::NS) {
        if (C::BESIDE && i + C::NS < n_tiles) {
          wait(s_free + stream, parity, 8);
          scores();
        }
        wait(p_full + stream, parity, 7);  // (the U before has been read as well)
        tc_fence_after();
        const uint64_t v = v_desc + (uint64_t)(buf * (C::TILE >> 4));
        if (elect_one()) {
#pragma unroll
          for (int n = C::PT - 1; n >= 0; n--)
#pragma unroll
            for (int s = 0; s < W_KEYS / 16; s++)
              umma_f16_ts(u_col, C::BESIDE ? p_col + 8u * s : s_col + (n < 2 ? 16u * s + 8u * n : 64u + 8u * s), v + (uint64_t)(s * (2048 >> 4)), C::ID_U,
                          n == C::PT - 1 && s == 0 ? (C::STAYS && i > stream ? 1u : 0u) : 1u);
          umma_commit(u_full + stream);
          umma_commit(kv_free + buf);
        }
        __syncwarp();
        buf += C::NS;
        if (buf >= C::TILES) buf -= C::TILES;
        if (!C::BESIDE && i + C::NS < n_tiles) {
          wait(u_full + stream, parity, 8);  // P has been read
          scores();
        }
        parity ^= 1u;
      }
    }
    __syncthreads();
  }
  if (a.splits > 1)
    asm volatile("barrier.cluster.arrive;\n\tbarrier.cluster.wait;" ::: "memory");
  else
    __syncthreads();
  const uint32_t so_at = smem_u32(so), state_at = smem_u32(&s_state[0][0][0]);
  for (int i = split * C::THREADS + tid; i < live_rows * (D / 4); i += a.splits * C::THREADS) {
    const int r = i / (D / 4), c = i % (D / 4) * 4;
    float m = -INFINITY, l = 0.f, o[4] = {};
    for (int p = 0; p < a.splits; p++) {
#pragma unroll
      for (int st = 0; st < C::NS; st++) {
        uint32_t at_m, at_o;
        float pm, pl, x[4];
        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at_m) : "r"(state_at + (uint32_t)(st * W_ROWS + r) * 8), "r"(p));
        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at_o) : "r"(so_at + (uint32_t)((st * W_ROWS + r) * C::PITCH + c) * 4), "r"(p));
        asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(pm), "=f"(pl) : "r"(at_m) : "memory");
        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]) : "r"(at_o) : "memory");
        const float next = fmaxf(m, pm), base = next == -INFINITY ? 0.f : next;
        const float fa = ex2(m - base), fb = ex2(pm - base);
        l = l * fa + pl * fb;
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] = o[e] * fa + x[e] * fb;
        m = next;
      }
    }
    const int t2 = (row0 + r) / a.group, g2 = row0 + r - t2 * a.group;
    TQ* to = static_cast<TQ*>(a.out) + ((b * a.rows + t2) * a.heads + (int64_t)kvh * a.group + g2) * a.d + c;
    const float over = over_sum<D / 4>(a, b, t2, len, keys, l);
    if (c < a.d) {
#pragma unroll
      for (int e = 0; e < 4; e++) kv_store(o[e] * over, to + e);
    }
  }
  __syncwarp();
  if (a.splits > 1)
    asm volatile("barrier.cluster.arrive;\n\tbarrier.cluster.wait;" ::: "memory");  // others read this block's states
  tc_fence_after();
  if (warp == ISSUING) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  if (tid == 0 && s_abort) report_wait_expired(error, DEV_ERR_ATTENTION_PIPE);
}

template <int CT, typename TQ, int D>
int run_wide(TreeArgs a, cudaStream_t s) {
  using C = Wide<CT, TQ, D>;
  auto kernel = tree_attention_wide_kernel<CT, TQ, D>;
  if (ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), C::SMEM)) return 1;
  int* const error = device_error_word();
  if (!error) return 1;
  // the shares above come out of what the compiler gave the launch: with fewer registers a warp would wait for more without end
  static std::atomic<int> launch_regs{0};
  if (!launch_regs) {
    cudaFuncAttributes attr;
    DYN_CUDA(cudaFuncGetAttributes(&attr, kernel));
    launch_regs = attr.numRegs;
  }
  DYN_CHECK(launch_regs >= C::START, "tree_attention: built with %d registers a thread", launch_regs.load());
  const int64_t pairs = a.batch * a.kv_heads;
  const int64_t row_blocks = ((int64_t)a.rows * a.group + W_ROWS - 1) / W_ROWS;
  // blocks of a cluster: as many as leave all clusters running at once (a block takes an SM), at least two tiles each at full
  // capacity, four for more than eight blocks
  const int64_t most = std::max(a.cap / (4 * W_KEYS), std::min<int64_t>(8, a.cap / (2 * W_KEYS)));
  const int splits = blocks_per_cluster<tree_attention_wide_kernel<CT, TQ, D>, C::THREADS, C::SMEM>(pairs * row_blocks, most);
  a.splits = splits;
  DYN_CHECK(pairs * splits <= 0x7fffffff && row_blocks <= 65535, "tree_attention: too many sequences or rows for one call");
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(pairs * splits), (unsigned)row_blocks), cfg.blockDim = dim3(C::THREADS);
  cfg.dynamicSmemBytes = C::SMEM, cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)splits, attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr, cfg.numAttrs = 1;
  DYN_CUDA(cudaLaunchKernelEx(&cfg, kernel, a, error));
  count_launch();
  return 0;
}

template <int CT, typename TQ, int D>
int by_rows(const TreeArgs& a, cudaStream_t s) {
  // us with 8 kv heads of 128, 4 query heads each; 16 rows in run / run_wide: q8 keys with f32 queries, 1 sequence of 500 13.3 / 14.7, of
  // 4000 17.7 / 22.9, of 32000 52 / 81, 8 of 500 19.1 / 15.7, 8 of 4000 35.0 / 56.1; bf16 for both 11.9 / 10.2, 16.2 / 16.1, 50.8 / 50.4, 13.6 / 11.2,
  // 34.1 / 34.1, which is not worth the slower way of rows that are not finite. 20 rows in two tiles of sixteen per warp were slower
  // than run_wide everywhere (8 of 4000: 63.8 / 56.9, bf16 50.7 / 34.1)
  const int64_t rows = (int64_t)a.rows * a.group;
  if (rows <= 8) return run<CT, TQ, D, true>(a, s);
  if (rows <= 16) return run<CT, TQ, D, false>(a, s);
  return run_wide<CT, TQ, D>(a, s);
}

template <int CT>
int by_type(const TreeArgs& a, int q_type, cudaStream_t s) {
  if (a.d <= 64) {
    if (q_type == E_F32) return by_rows<CT, float, 64>(a, s);
    if (q_type == E_F16) return by_rows<CT, __half, 64>(a, s);
    return by_rows<CT, __nv_bfloat16, 64>(a, s);
  }
  if (q_type == E_F32) return by_rows<CT, float, 128>(a, s);
  if (q_type == E_F16) return by_rows<CT, __half, 128>(a, s);
  return by_rows<CT, __nv_bfloat16, 128>(a, s);
}

}  // namespace tree
}  // namespace dyn
