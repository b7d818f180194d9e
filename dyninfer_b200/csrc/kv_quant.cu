// An 8-bit key/value cache: rows are quantised as they are written, and read back as values.
//
// A row is the d entries of one (slot, kv head, position), with one f32 scale. A scale per row lets attention use the codes as
// they are: the keys' scales multiply finished scores, the values' scales the softmax weights.
//   q8    code = round to even of x * inv, inv = f32(127 / top), scale = f32(top / 127), top the row's largest magnitude. The
//         product is rounded once, to a whole number, by an fma with 1.5 * 2^23: no second rounding moves a code over a half.
//   e4m3  scale = the least power of two with top / scale <= 448, code = e4m3(x / scale): exact but for the format's own
//         rounding; a scale with a fraction would gain no precision in a floating format.
// A row whose top is below 2^-100 becomes zeros with scale 0 (1 / top would leave f32's range). A row with an infinity or NaN
// gets a NaN scale over zero codes: it reads back as NaN, and no product ever meets a code that is not finite.
//
// Memory bounds both directions. A thread holds sixteen entries of a key row and of the value row beside it; a row's threads
// (d / 16 rounded up to a power of two) share its maximum by shuffles, and everything is touched once, 16 bytes at a time. What is
// read is asked for before anything is computed. 8 x 2048 x 8 rows of 128 bf16 entries: written 17.4 us (e4m3) and 18.9 (q8), 88 and 81 % of
// the copy bandwidth, read 21 (73 %); with eight entries per thread 25, 28 and 24.
#include <algorithm>

#include "kv_codes.cuh"

namespace dyn {

namespace {

constexpr int KV_THREADS = 128;

struct KvRowArgs {
  const void* x[2];       // write: keys, values [batch][row][head][d]; unused when reading
  void* y[2];             // read: the same
  int64_t xs[2][3];       // elements between batch entries, rows, heads
  uint8_t* codes[2];      // [slot][head][cap][d]
  int64_t cs[2][3];       // bytes between slots, heads, rows
  float* scales[2];       // [slot][head][cap]
  int64_t ss[2][2];       // floats between slots, heads
  const int64_t* starts;  // [batch]
  const int64_t* counts;  // [batch] or NULL
  int64_t batch, rows, cap;
  int heads, units;          // units of sixteen entries per row
};

template <typename T, bool WIDE>
__device__ __forceinline__ void load16(const T* p, float (&v)[16]) {
  if (WIDE) {
    uint4 raw[sizeof(T)];
#pragma unroll
    for (int i = 0; i < (int)sizeof(T); i++) raw[i] = reinterpret_cast<const uint4*>(p)[i];
    const T* e = reinterpret_cast<const T*>(raw);
#pragma unroll
    for (int i = 0; i < 16; i++) v[i] = kv_float(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 16; i++) v[i] = kv_float(p[i]);
  }
}

// Whether a row of a batch entry has a place in the cache.
__device__ __forceinline__ bool in_cache(const KvRowArgs& a, int64_t batch, int row, int64_t start) {
  // a start far outside must not wrap around into the cache
  return start > -a.cap - a.rows && start < a.cap && start + row >= 0 && start + row < a.cap && (!a.counts || row < a.counts[batch]);
}

template <typename T, bool E4M3, bool WIDE, int P>
__global__ void __launch_bounds__(KV_THREADS) kv_write_kernel(const __grid_constant__ KvRowArgs a) {
  const int lane = threadIdx.x & (P - 1);
  const unsigned pair = blockIdx.x * (KV_THREADS / P) + threadIdx.x / P;  // row and head; the head runs fastest
  const int row = (int)(pair / (unsigned)a.heads), head = (int)(pair - (unsigned)row * (unsigned)a.heads);
  const bool here = pair < (unsigned)(a.rows * a.heads) && lane < a.units;
  for (int64_t batch = blockIdx.y; batch < a.batch; batch += gridDim.y) {
    const int64_t start = a.starts[batch], at = start + row;
    float v[2][16] = {};
#pragma unroll
    for (int w = 0; w < 2; w++)
      if (here)
        load16<T, WIDE>(static_cast<const T*>(a.x[w]) + batch * a.xs[w][0] + row * a.xs[w][1] + head * a.xs[w][2] + lane * 16, v[w]);
    const bool mine = here && in_cache(a, batch, row, start);
#pragma unroll
    for (int w = 0; w < 2; w++) {
      uint32_t top = 0;  // magnitudes compare as integers; infinities and NaN come out on top
#pragma unroll
      for (int e = 0; e < 16; e++) top = max(top, __float_as_uint(v[w][e]) & 0x7fffffffu);
#pragma unroll
      for (int o = P / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      float scale, inv;
      kv_scale<E4M3>(top, &scale, &inv);
      if (mine) {
        const uint2 lo = kv_encode8<E4M3>(reinterpret_cast<float(&)[8]>(v[w][0]), inv);
        const uint2 hi = kv_encode8<E4M3>(reinterpret_cast<float(&)[8]>(v[w][8]), inv);
        *reinterpret_cast<uint4*>(a.codes[w] + batch * a.cs[w][0] + head * a.cs[w][1] + at * a.cs[w][2] + lane * 16) =
            make_uint4(lo.x, lo.y, hi.x, hi.y);
        if (lane == 0) a.scales[w][batch * a.ss[w][0] + head * a.ss[w][1] + at] = scale;
      }
    }
  }
}

template <typename T, bool E4M3, bool WIDE, int P>
__global__ void __launch_bounds__(KV_THREADS) kv_read_kernel(const __grid_constant__ KvRowArgs a) {
  const int lane = threadIdx.x & (P - 1);
  const unsigned pair = blockIdx.x * (KV_THREADS / P) + threadIdx.x / P;
  const int row = (int)(pair / (unsigned)a.heads), head = (int)(pair - (unsigned)row * (unsigned)a.heads);
  if (lane >= a.units || pair >= (unsigned)(a.rows * a.heads)) return;
  for (int64_t batch = blockIdx.y; batch < a.batch; batch += gridDim.y) {
    const int64_t start = a.starts[batch], at = start + row;
    const bool live = in_cache(a, batch, row, start);
    uint4 raw[2] = {};
    float scale[2] = {};
#pragma unroll
    for (int w = 0; w < 2; w++)
      if (live) {
        raw[w] = *reinterpret_cast<const uint4*>(a.codes[w] + batch * a.cs[w][0] + head * a.cs[w][1] + at * a.cs[w][2] + lane * 16);
        scale[w] = a.scales[w][batch * a.ss[w][0] + head * a.ss[w][1] + at];
      }
#pragma unroll
    for (int w = 0; w < 2; w++) {
      float v[16];
      kv_decode8<E4M3>(make_uint2(raw[w].x, raw[w].y), scale[w], reinterpret_cast<float(&)[8]>(v[0]));
      kv_decode8<E4M3>(make_uint2(raw[w].z, raw[w].w), scale[w], reinterpret_cast<float(&)[8]>(v[8]));
      T* to = static_cast<T*>(a.y[w]) + batch * a.xs[w][0] + row * a.xs[w][1] + head * a.xs[w][2] + lane * 16;
      uint4 packed[sizeof(T)];
      T* e = reinterpret_cast<T*>(packed);
#pragma unroll
      for (int j = 0; j < 16; j++) kv_store(live ? v[j] : 0.f, e + j);
      if (WIDE) {
#pragma unroll
        for (int j = 0; j < (int)sizeof(T); j++) reinterpret_cast<uint4*>(to)[j] = packed[j];
      } else {
#pragma unroll
        for (int j = 0; j < 16; j++) to[j] = e[j];
      }
    }
  }
}

template <typename T, bool E4M3, bool WIDE, int P>
int kv_run(const KvRowArgs& a, bool write, cudaStream_t s) {
  const int64_t blocks = (a.rows * a.heads + KV_THREADS / P - 1) / (KV_THREADS / P);
  const dim3 grid((unsigned)blocks, (unsigned)std::min<int64_t>(a.batch, 65535));
  if (write)
    kv_write_kernel<T, E4M3, WIDE, P><<<grid, KV_THREADS, 0, s>>>(a);
  else
    kv_read_kernel<T, E4M3, WIDE, P><<<grid, KV_THREADS, 0, s>>>(a);
  count_launch();
  DYN_CUDA(cudaGetLastError());
  return 0;
}

template <typename T, bool E4M3, bool WIDE>
int kv_lanes(const KvRowArgs& a, bool write, cudaStream_t s) {
  if (a.units <= 2) return kv_run<T, E4M3, WIDE, 2>(a, write, s);
  if (a.units <= 4) return kv_run<T, E4M3, WIDE, 4>(a, write, s);
  if (a.units <= 8) return kv_run<T, E4M3, WIDE, 8>(a, write, s);
  return kv_run<T, E4M3, WIDE, 16>(a, write, s);
}

template <typename T>
int kv_type(const KvRowArgs& a, bool e4m3, bool write, cudaStream_t s) {
  uintptr_t low = 0;
  for (int w = 0; w < 2; w++) {
    low |= reinterpret_cast<uintptr_t>(write ? a.x[w] : a.y[w]);
    for (int i = 0; i < 3; i++) low |= (uintptr_t)a.xs[w][i] * sizeof(T);
  }
  const bool wide = (low & 15) == 0;
  if (e4m3) return wide ? kv_lanes<T, true, true>(a, write, s) : kv_lanes<T, true, false>(a, write, s);
  return wide ? kv_lanes<T, false, true>(a, write, s) : kv_lanes<T, false, false>(a, write, s);
}

}  // namespace

int launch_kv_rows(const KvRows& r, bool write, cudaStream_t s) {
  KvRowArgs a{};
  a.batch = r.batch, a.rows = r.rows, a.cap = r.cap, a.heads = (int)r.heads, a.units = (int)(r.d / 16);
  a.starts = r.starts, a.counts = r.counts;
  if (a.batch * a.rows * a.heads == 0) return 0;
  for (int w = 0; w < 2; w++) {
    a.x[w] = r.x[w], a.y[w] = r.x[w];
    a.codes[w] = static_cast<uint8_t*>(r.codes[w]), a.scales[w] = r.scales[w];
    for (int i = 0; i < 3; i++) a.xs[w][i] = r.x_strides[w * 3 + i], a.cs[w][i] = r.code_strides[w * 3 + i];
    for (int i = 0; i < 2; i++) a.ss[w][i] = r.scale_strides[w * 2 + i];
  }
  if (r.type == E_F32) return kv_type<float>(a, r.e4m3, write, s);
  if (r.type == E_F16) return kv_type<__half>(a, r.e4m3, write, s);
  return kv_type<__nv_bfloat16>(a, r.e4m3, write, s);
}

}  // namespace dyn
