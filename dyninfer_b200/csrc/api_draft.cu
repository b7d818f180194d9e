// extern "C" surface of the operators of speculative decoding: rotary positions, the 8-bit cache, attention of drafted trees and
// their verification. Arguments are checked here, on the host, before any launch.
#include <math.h>

#include <atomic>

#include "attention_tree.cuh"
#include "common.cuh"

namespace dyn {
namespace {

int have_device() {
  static std::atomic<bool> seen{false};  // a device that was there stays
  if (seen.load(std::memory_order_relaxed)) return 0;
  int n = 0;
  const cudaError_t e = cudaGetDeviceCount(&n);
  DYN_CHECK(e == cudaSuccess && n > 0, "no usable CUDA device (%s); this target has no CPU fallback",
            e == cudaSuccess ? "device count is 0" : cudaGetErrorString(e));
  seen.store(true, std::memory_order_relaxed);
  return 0;
}
bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }
bool plain_type(int t) { return t == E_F32 || t == E_F16 || t == E_BF16; }
size_t type_bytes(int t) { return t == E_F32 ? 4 : 2; }
// Counts whose products stay far inside 64 bits
bool sane(int64_t n) { return n >= 0 && n <= (1ll << 31) - 1; }

// Strides with those of dimensions of one entry as zero: nothing is stepped along there, whatever they say.
template <int N>
struct Steps {
  int64_t v[N];
  bool repeats = false;  // a dimension of several entries without a step: what is written there would meet
  Steps(const int64_t* of, const int64_t* extents, int dims) {
    for (int i = 0; i < N; i++) {
      v[i] = of && extents[i % dims] > 1 ? of[i] : 0;
      repeats = repeats || (extents[i % dims] > 1 && v[i] == 0);
    }
  }
};

int kv_rows(const char* what, const void* k, const void* v, int type, const int64_t* x_strides, void* k_cache, void* v_cache,
            int kv_type, const int64_t* cache_strides, float* k_scale, float* v_scale, const int64_t* scale_strides,
            const int64_t* starts, const int64_t* counts, int64_t batch, int64_t rows, int64_t heads, int64_t d, int64_t cap,
            bool write, void* stream) {
  DYN_CHECK(plain_type(type), "%s: type %d unsupported (f32, f16 or bf16)", what, type);
  DYN_CHECK(kv_type == DYNINFER_KV_Q8 || kv_type == DYNINFER_KV_E4M3, "%s: cache type %d is not an 8-bit one", what, kv_type);
  DYN_CHECK(sane(batch) && sane(rows) && heads > 0 && heads <= 65536 && cap > 0 && sane(cap) && rows * heads <= (1ll << 30), "%s: bad shape", what);
  DYN_CHECK(d > 0 && d % 16 == 0 && d <= 256, "%s: head dim %lld unsupported (a multiple of 16 up to 256)", what, (long long)d);
  if (batch == 0 || rows == 0) return 0;
  DYN_CHECK(k && v && k_cache && v_cache && k_scale && v_scale && starts && x_strides && cache_strides && scale_strides,
            "%s: NULL pointer", what);
  DYN_CHECK(aligned(k, type_bytes(type)) && aligned(v, type_bytes(type)) && aligned(k_scale, 4) && aligned(v_scale, 4) &&
                aligned(starts, 8) && aligned(counts, 8),
            "%s: a pointer is not aligned to its type", what);
  const int64_t of_x[3] = {batch, rows, heads}, of_cache[3] = {batch, heads, cap};
  const Steps<6> x_steps(x_strides, of_x, 3), cache_steps(cache_strides, of_cache, 3);
  const Steps<4> scale_steps(scale_strides, of_cache, 2);
  bool even = aligned(k_cache, 16) && aligned(v_cache, 16);
  for (int64_t step : cache_steps.v) even = even && step % 16 == 0;
  DYN_CHECK(even, "%s: caches and their strides must be multiples of 16 bytes", what);
  DYN_CHECK(!write || !(cache_steps.repeats || scale_steps.repeats), "%s: a cache dimension has stride 0, rows would be written over one another", what);
  DYN_CHECK(write || !x_steps.repeats, "%s: an output dimension has stride 0", what);
  if (have_device()) return 1;
  KvRows r{};
  // read-only when writing; the struct serves both directions
  r.x[0] = const_cast<void*>(k), r.x[1] = const_cast<void*>(v), r.x_strides = x_steps.v;
  r.codes[0] = k_cache, r.codes[1] = v_cache, r.code_strides = cache_steps.v;
  r.scales[0] = k_scale, r.scales[1] = v_scale, r.scale_strides = scale_steps.v;
  r.starts = starts, r.counts = counts, r.batch = batch, r.rows = rows, r.heads = heads, r.d = d, r.cap = cap;
  r.type = type, r.e4m3 = kv_type == DYNINFER_KV_E4M3;
  return launch_kv_rows(r, write, (cudaStream_t)stream);
}

}  // namespace
}  // namespace dyn

using namespace dyn;

extern "C" {

int dyninfer_cuda_rotary(const void* x_dev, int type, const int64_t* x_strides, const int64_t* positions_dev,
                         const double* frequencies, int64_t rotary_dim, int interleaved, double magnitude, int64_t batch,
                         int64_t rows, int64_t heads, int64_t d, void* y_dev, const int64_t* y_strides, void* stream) {
  DYN_CHECK(plain_type(type), "rotary: type %d unsupported (f32, f16 or bf16)", type);
  DYN_CHECK(sane(batch) && sane(rows) && heads >= 0 && heads <= 65536 && batch * rows <= (1ll << 40), "rotary: bad shape");
  DYN_CHECK(d > 0 && d <= ROTARY_MAX_DIM && rotary_dim > 0 && rotary_dim % 2 == 0 && rotary_dim <= d,
            "rotary: %lld of %lld dimensions (an even number, at most the head's, which has up to %d)", (long long)rotary_dim,
            (long long)d, ROTARY_MAX_DIM);
  DYN_CHECK(isfinite(magnitude), "rotary: the magnitude is not finite");
  if (batch == 0 || rows == 0 || heads == 0) return 0;
  DYN_CHECK(x_dev && y_dev && x_strides && y_strides && positions_dev && frequencies, "rotary: NULL pointer");
  DYN_CHECK(aligned(x_dev, type_bytes(type)) && aligned(y_dev, type_bytes(type)) && aligned(positions_dev, 8),
            "rotary: a pointer is not aligned to its type");
  for (int64_t i = 0; i < rotary_dim / 2; i++) DYN_CHECK(isfinite(frequencies[i]), "rotary: frequency %lld is not finite", (long long)i);
  const int64_t extents[3] = {batch, rows, heads};
  const Steps<3> x_steps(x_strides, extents, 3), y_steps(y_strides, extents, 3);
  DYN_CHECK(!y_steps.repeats, "rotary: an output dimension has stride 0");
  if (have_device()) return 1;
  return launch_rotary(x_dev, type, batch, rows, heads, d, x_steps.v, positions_dev, frequencies, rotary_dim, interleaved != 0,
                       magnitude, y_dev, y_steps.v, (cudaStream_t)stream);
}

int dyninfer_cuda_kv_write(const void* k_dev, const void* v_dev, int type, const int64_t* x_strides, void* k_cache_dev,
                           void* v_cache_dev, int kv_type, const int64_t* cache_strides, float* k_scale_dev, float* v_scale_dev,
                           const int64_t* scale_strides, const int64_t* starts_dev, const int64_t* counts_dev, int64_t batch,
                           int64_t rows, int64_t kv_heads, int64_t d, int64_t kv_cap, void* stream) {
  return kv_rows("kv_write", k_dev, v_dev, type, x_strides, k_cache_dev, v_cache_dev, kv_type, cache_strides, k_scale_dev, v_scale_dev,
                 scale_strides, starts_dev, counts_dev, batch, rows, kv_heads, d, kv_cap, true, stream);
}

int dyninfer_cuda_kv_read(void* k_dev, void* v_dev, int type, const int64_t* x_strides, const void* k_cache_dev,
                          const void* v_cache_dev, int kv_type, const int64_t* cache_strides, const float* k_scale_dev,
                          const float* v_scale_dev, const int64_t* scale_strides, const int64_t* starts_dev, int64_t batch,
                          int64_t rows, int64_t kv_heads, int64_t d, int64_t kv_cap, void* stream) {
  return kv_rows("kv_read", k_dev, v_dev, type, x_strides, const_cast<void*>(k_cache_dev), const_cast<void*>(v_cache_dev), kv_type,
                 cache_strides, const_cast<float*>(k_scale_dev), const_cast<float*>(v_scale_dev), scale_strides, starts_dev, nullptr,
                 batch, rows, kv_heads, d, kv_cap, false, stream);
}

int dyninfer_cuda_tree_attention(const void* q_dev, int q_type, const int64_t* q_strides, const void* k_cache_dev,
                                 const void* v_cache_dev, int kv_type, const int64_t* cache_strides, const float* k_scale_dev,
                                 const float* v_scale_dev, const int64_t* scale_strides, const int64_t* lengths_dev,
                                 const uint8_t* mask_dev, const int64_t* mask_strides, int64_t batch, int64_t rows, int64_t heads,
                                 int64_t kv_heads, int64_t d, int64_t kv_cap, float scale, void* ctx_dev, void* stream) {
  const bool wide = kv_type == E_BF16 || kv_type == E_F16;
  DYN_CHECK(plain_type(q_type), "tree_attention: query type %d unsupported (f32, f16 or bf16)", q_type);
  DYN_CHECK(wide || kv_type == DYNINFER_KV_Q8 || kv_type == DYNINFER_KV_E4M3,
            "tree_attention: cache type %d unsupported (f16, bf16, q8 or e4m3)", kv_type);
  DYN_CHECK(sane(batch) && rows >= 0 && rows <= 65536 && heads > 0 && kv_heads > 0 && kv_cap > 0 && sane(kv_cap),
            "tree_attention: bad shape");
  DYN_CHECK(heads <= 65536 && rows * heads <= (1ll << 30) && heads % kv_heads == 0, "tree_attention: heads %lld not a multiple of kv heads %lld (or too many)",
            (long long)heads, (long long)kv_heads);
  DYN_CHECK(d > 0 && d % 16 == 0 && d <= 128, "tree_attention: head dim %lld unsupported (a multiple of 16 up to 128)", (long long)d);
  DYN_CHECK(isfinite(scale) && scale > 0, "tree_attention: the scale must be above zero and finite");
  if (batch == 0 || rows == 0) return 0;
  DYN_CHECK(q_dev && q_strides && k_cache_dev && v_cache_dev && cache_strides && lengths_dev && ctx_dev, "tree_attention: NULL pointer");
  DYN_CHECK(wide || (k_scale_dev && v_scale_dev && scale_strides), "tree_attention: an 8-bit cache needs its scales");
  DYN_CHECK(!mask_dev || mask_strides, "tree_attention: a mask needs its strides");
  DYN_CHECK(aligned(q_dev, type_bytes(q_type)) && aligned(lengths_dev, 8) && aligned(k_scale_dev, 4) && aligned(v_scale_dev, 4),
            "tree_attention: a pointer is not aligned to its type");
  const int64_t size = wide ? 2 : 1;
  const int64_t of_q[3] = {batch, rows, heads}, of_cache[3] = {batch, kv_heads, kv_cap};
  const Steps<3> q_steps(q_strides, of_q, 3);
  const Steps<6> cache_steps(cache_strides, of_cache, 3);
  const Steps<4> scale_steps(scale_strides, of_cache, 2);
  const Steps<2> mask_steps(mask_strides, of_q, 2);
  bool even = aligned(k_cache_dev, 16) && aligned(v_cache_dev, 16) && aligned(ctx_dev, 16);
  for (int64_t step : cache_steps.v) even = even && step * size % 16 == 0;
  DYN_CHECK(even, "tree_attention: caches, their strides and the output must be multiples of 16 bytes");
  // the word that waits report to is allocated here, so that no row count does it first inside a capture
  if (have_device() || !device_error_word()) return 1;
  TreeArgs a{};
  a.q = q_dev, a.out = ctx_dev, a.k = static_cast<const uint8_t*>(k_cache_dev), a.v = static_cast<const uint8_t*>(v_cache_dev);
  a.lengths = lengths_dev, a.mask = mask_dev;
  for (int i = 0; i < 3; i++) a.qs[i] = q_steps.v[i], a.kst[i] = cache_steps.v[i] * size, a.vst[i] = cache_steps.v[3 + i] * size;
  if (!wide) {
    a.ks = k_scale_dev, a.vs = v_scale_dev;
    for (int i = 0; i < 2; i++) a.kss[i] = scale_steps.v[i], a.vss[i] = scale_steps.v[2 + i];
  }
  a.ms[0] = mask_steps.v[0], a.ms[1] = mask_steps.v[1];
  a.batch = batch, a.cap = kv_cap, a.rows = (int)rows, a.heads = (int)heads, a.kv_heads = (int)kv_heads;
  a.group = (int)(heads / kv_heads), a.d = (int)d, a.scale = scale;
  const cudaStream_t s = (cudaStream_t)stream;
  if (kv_type == E_BF16) return tree_attention_bf16(a, q_type, s);
  if (kv_type == E_F16) return tree_attention_f16(a, q_type, s);
  return kv_type == DYNINFER_KV_Q8 ? tree_attention_q8(a, q_type, s) : tree_attention_e4m3(a, q_type, s);
}

int dyninfer_cuda_verify_draft(const int64_t* tokens_dev, const int64_t* parents_dev, int64_t parents_stride, const void* target_dev,
                               const int64_t* target_strides, const void* draft_dev, const int64_t* draft_strides, int type,
                               const float* uniforms_dev, int64_t batch, int64_t nodes, int64_t vocab, int64_t* accepted_dev,
                               int64_t* path_dev, int64_t* next_dev, void* stream) {
  DYN_CHECK(plain_type(type), "verify_draft: type %d unsupported (f32, f16 or bf16)", type);
  DYN_CHECK(sane(batch) && nodes >= 1 && nodes <= 1024 && vocab >= 1 && sane(vocab),
            "verify_draft: bad shape (1 to 1024 nodes, the text's last token among them)");
  if (batch == 0) return 0;
  DYN_CHECK(tokens_dev && parents_dev && target_dev && target_strides && uniforms_dev && accepted_dev && path_dev && next_dev,
            "verify_draft: NULL pointer");
  DYN_CHECK(!draft_dev || draft_strides, "verify_draft: the draft's probabilities need their strides");
  DYN_CHECK(aligned(tokens_dev, 8) && aligned(parents_dev, 8) && aligned(accepted_dev, 8) && aligned(path_dev, 8) && aligned(next_dev, 8) &&
                aligned(uniforms_dev, 4) && aligned(target_dev, type_bytes(type)) && aligned(draft_dev, type_bytes(type)),
            "verify_draft: a pointer is not aligned to its type");
  if (have_device()) return 1;
  return launch_verify_draft(tokens_dev, parents_dev, parents_stride, target_dev, target_strides, draft_dev, draft_strides, type,
                             uniforms_dev, batch, nodes, vocab, accepted_dev, path_dev, next_dev, (cudaStream_t)stream);
}

}  // extern "C"
