// Rotary positions of a block of rows: any position per row, the half or the interleaved layout, part of the head, any table
// of frequencies (scaled ones among them), f32 / f16 / bf16.
//
//   pair (a, b) = (x[i], x[i + r/2]) (half) or (x[2i], x[2i+1]) (interleaved), i < r/2, angle = position * f_i:
//   a' = m (a cos - b sin),  b' = m (b cos + a sin);  elements from r on are copied.
//
// Angles. f32 loses them far out (position 200000 at f = 1: 0.008 rad). An angle matters modulo one turn only, so the host
// turns f / 2 pi into a 64-bit fixed-point fraction of a turn, rounded; position * fraction in wrapping 64-bit integers is their
// exact product modulo one turn, one integer multiplication and one rounding to f32. What is off is the fraction: by 2^-65 for its
// rounding, and by f 2^-65 for the two roundings of f / 2 pi to 64 bits, so an angle by at most position * (1 + f) 2^-65 turns.
// That is below f32's own rounding of it up to positions of 2^39. Signed, in half turns, it is sincospif's argument.
//
// What bounds it is memory: every element comes and goes once. A block takes one row or a few; its threads compute the row's
// cosines and sines once, into shared memory, while the first head's elements are on their way, and then stay with their
// pairs over all heads, with 16-byte accesses where strides and layout allow. 5003 rows of 72 f32 heads: 62.9 us, 90 % of the copy
// bandwidth; 2048 of 40 bf16 heads 10.4 us (62 %), where blocks starting and ending count.
#include <math.h>

#include <algorithm>

#include "common.cuh"

namespace dyn {

namespace {

struct RotaryTable {
  uint64_t turn[ROTARY_MAX_DIM / 2];  // f_i / 2 pi modulo one, times 2^64
};

struct RotaryArgs {
  const void* x;
  void* y;
  const int64_t* positions;
  int64_t rows;  // of one batch entry
  int64_t total; // rows of all
  int64_t xs[3], ys[3];  // elements between batch entries, rows, heads
  int heads, rot, d, copy, pairs;
  float magnitude;
};

template <typename T, int N>
struct alignas(N * sizeof(T)) Vec {
  T v[N];
};

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void from_f(float x, float* y) { *y = x; }
__device__ __forceinline__ void from_f(float x, __half* y) { *y = __float2half_rn(x); }
__device__ __forceinline__ void from_f(float x, __nv_bfloat16* y) { *y = __float2bfloat16_rn(x); }

// 2048 rows of 40 bf16 heads: 64 threads 9.3 us, 128 10.4, 256 14.4, 512 15.9; 5003 rows of 72 f32 heads: 70.8, 62.9, 64.2, 68.9
constexpr int ROTARY_THREADS = 128;

// Spelled out, so that every form of the kernel rounds alike.
__device__ __forceinline__ float2 turn(float a, float b, float2 cs) {
  return make_float2(__fmaf_rn(a, cs.x, -__fmul_rn(b, cs.y)), __fmaf_rn(b, cs.x, __fmul_rn(a, cs.y)));
}

// threadIdx: x = unit inside the head (rotated units first, then copied ones), y = head, z = row of the block.
// A rotated unit is N elements of either half, or N interleaved elements (N = 1: one pair of single elements).
template <typename T, int N, bool INTER>
__global__ void __launch_bounds__(ROTARY_MAX_DIM) rotary_kernel(const __grid_constant__ RotaryArgs a,
                                                                const __grid_constant__ RotaryTable table) {
  constexpr bool SPLIT = !INTER || N == 1;  // the pair's elements come by two accesses
  constexpr int PAIRS = SPLIT ? N : N / 2;
  extern __shared__ float2 turned[];        // [rows of the block][pairs] (cos, sin)
  const int64_t row = (int64_t)blockIdx.x * blockDim.z + threadIdx.z;
  const bool live = row < a.total;
  const int64_t batch = live ? row / a.rows : 0, in_batch = live ? row - batch * a.rows : 0;
  const T* x = static_cast<const T*>(a.x) + batch * a.xs[0] + in_batch * a.xs[1];
  T* y = static_cast<T*>(a.y) + batch * a.ys[0] + in_batch * a.ys[1];
  const int u = threadIdx.x, units = a.pairs / PAIRS;
  const bool rotated = u < units;
  const int first = rotated ? (SPLIT && INTER ? 2 * u : u * N) : a.rot + (u - units) * N;
  const int second = INTER ? first + 1 : first + a.pairs;  // SPLIT only
  typedef Vec<T, N> V;
  V va{}, vb{};
  int h = threadIdx.y;
  if (live && h < a.heads) {
    va = *reinterpret_cast<const V*>(x + h * a.xs[2] + first);
    if (SPLIT && rotated) vb = *reinterpret_cast<const V*>(x + h * a.xs[2] + second);
  }
  const int threads = blockDim.x * blockDim.y * blockDim.z;
  for (int i = (threadIdx.z * blockDim.y + threadIdx.y) * blockDim.x + threadIdx.x; i < a.pairs * (int)blockDim.z; i += threads) {
    const int z = i / a.pairs, p = i - z * a.pairs;
    const int64_t r = (int64_t)blockIdx.x * blockDim.z + z;
    if (r < a.total) {
      const int64_t angle = (int64_t)((uint64_t)a.positions[r] * table.turn[p]);
      float s, c;
      sincospif((float)angle * 0x1p-63f, &s, &c);
      turned[i] = make_float2(c * a.magnitude, s * a.magnitude);
    }
  }
  __syncthreads();
  if (!live) return;
  float2 cs[PAIRS];
  if (rotated) {
#pragma unroll
    for (int i = 0; i < PAIRS; i++) cs[i] = turned[threadIdx.z * a.pairs + u * PAIRS + i];
  }
  for (; h < a.heads; h += blockDim.y) {
    V ca = va, cb = vb;
    const int next = h + blockDim.y;
    if (next < a.heads) {
      va = *reinterpret_cast<const V*>(x + next * a.xs[2] + first);
      if (SPLIT && rotated) vb = *reinterpret_cast<const V*>(x + next * a.xs[2] + second);
    }
    T* to = y + h * a.ys[2];
    if (!rotated) {
      *reinterpret_cast<V*>(to + first) = ca;
    } else if (SPLIT) {
#pragma unroll
      for (int i = 0; i < PAIRS; i++) {
        const float2 r = turn(to_f(ca.v[i]), to_f(cb.v[i]), cs[i]);
        from_f(r.x, &ca.v[i]);
        from_f(r.y, &cb.v[i]);
      }
      *reinterpret_cast<V*>(to + first) = ca;
      *reinterpret_cast<V*>(to + second) = cb;
    } else {
#pragma unroll
      for (int i = 0; i < PAIRS; i++) {
        const float2 r = turn(to_f(ca.v[2 * i]), to_f(ca.v[(2 * i + 1) % N]), cs[i]);
        from_f(r.x, &ca.v[2 * i]);
        from_f(r.y, &ca.v[(2 * i + 1) % N]);
      }
      *reinterpret_cast<V*>(to + first) = ca;
    }
  }
}

template <typename T, int N, bool INTER>
int rotary_run(const RotaryArgs& a, const RotaryTable& table, cudaStream_t s) {
  const int per = INTER && N > 1 ? N / 2 : N;
  const int ux = a.pairs / per + (a.copy ? (a.d - a.rot) / N : 0);
  // (single elements of a large head may be more units than that: never more than the head has dimensions)
  const int hy = std::max(1, std::min(ROTARY_THREADS / ux, a.heads));
  const int rz = std::max(1, std::min(ROTARY_THREADS / (ux * hy), 64));
  const int64_t blocks = (a.total + rz - 1) / rz;
  DYN_CHECK(blocks <= 0x7fffffff, "rotary: %lld rows are too many for one call", (long long)a.total);
  rotary_kernel<T, N, INTER><<<(unsigned)blocks, dim3(ux, hy, rz), (size_t)rz * a.pairs * sizeof(float2), s>>>(a, table);
  count_launch();
  DYN_CUDA(cudaGetLastError());
  return 0;
}

template <typename T, int N>
int rotary_layout(const RotaryArgs& a, const RotaryTable& table, bool inter, cudaStream_t s) {
  return inter ? rotary_run<T, N, true>(a, table, s) : rotary_run<T, N, false>(a, table, s);
}

template <typename T>
int rotary_type(const RotaryArgs& a, const RotaryTable& table, bool inter, cudaStream_t s) {
  // 16-byte accesses where every unit starts on 16 bytes: 2048 rows of 40 bf16 heads take 9 us, with single elements 16 to 17
  constexpr int N = 16 / sizeof(T);
  const uintptr_t base = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.y);
  int64_t sizes = a.d | a.rot | (inter ? 0 : a.pairs);
  for (int i = 0; i < 3; i++) sizes |= a.xs[i] | a.ys[i];
  if ((base & 15) == 0 && sizes % N == 0) return rotary_layout<T, N>(a, table, inter, s);
  return rotary_layout<T, 1>(a, table, inter, s);
}

}  // namespace

int launch_rotary(const void* x, int type, int64_t batch, int64_t rows, int64_t heads, int64_t d, const int64_t* x_strides,
                  const int64_t* positions, const double* frequencies, int64_t rot, bool interleaved, double magnitude, void* y,
                  const int64_t* y_strides, cudaStream_t s) {
  if (batch * rows * heads == 0) return 0;
  RotaryTable table{};
  for (int64_t i = 0; i < rot / 2; i++) {
    long double turns = (long double)frequencies[i] * 0.15915494309189533576888376337251436L;  // one over 2 pi
    turns -= fabsl(turns) < 4e18L ? (long double)(int64_t)turns : floorl(turns);
    if (turns < 0) turns += 1;
    const long double fraction = rintl(turns * 18446744073709551616.0L);
    table.turn[i] = fraction < 18446744073709551616.0L ? (uint64_t)fraction : 0;  // a whole turn is none
  }
  RotaryArgs a{};
  a.x = x, a.y = y, a.positions = positions, a.rows = rows, a.total = batch * rows;
  bool same = x == y;
  for (int i = 0; i < 3; i++) a.xs[i] = x_strides[i], a.ys[i] = y_strides[i], same = same && x_strides[i] == y_strides[i];
  a.heads = (int)heads, a.rot = (int)rot, a.d = (int)d, a.pairs = (int)(rot / 2), a.copy = !same && rot < d;
  a.magnitude = (float)magnitude;
  if (type == E_F32) return rotary_type<float>(a, table, interleaved, s);
  if (type == E_F16) return rotary_type<__half>(a, table, interleaved, s);
  return rotary_type<__nv_bfloat16>(a, table, interleaved, s);
}

}  // namespace dyn
