// Verification of a tree of drafted tokens against the target's probabilities, with given random numbers.
//
// Node 0 is the last token of the text; every other node stands behind its parent, and the target's row i is the distribution of
// the token behind node i. From node 0 on, the children c of the node reached are tried in order: with r_0 = p (the target's row
// of the node), Z_0 = 1,
//   c is taken    if u_c q(c) Z_m < r_m(c)                      (q: the draft's row of the node; 1 without a draft)
//   if refused    r_{m+1} = max(r_m / Z_m - q, 0), Z_{m+1} = sum of it;   without a draft r_{m+1} = r_m with c's entry gone and
//                 Z_{m+1} = Z_m - r_m(c).
// The last token is drawn from what is left at the node where no child was taken: the first v with r(0) + .. + r(v) above
// u_0 times the sum. Where nothing is left, from the target's row itself; where that has no finite positive sum, it is -1.
// Every sum is in 64 bits: a border between two of 150000 entries is a matter of 1e-9, and the answer is a whole number.
//
// Whether a child is taken depends on single entries, which are fetched for all nodes at once; what costs is one pass over a
// row of target (and draft) per refusal, about 1.2 MB for 150000 entries, so memory and latency bound it. A cluster of up to 16
// blocks takes a sequence, every warp a run of entries; the warps' sums meet through shared memory, in one order everywhere, so
// that all blocks walk the tree alike without asking one another. The sums are also what the draw searches: the block
// whose warp had the border in its run looks through that run once more, out of the caches.
#include <algorithm>

#include "clusters.cuh"
#include "common.cuh"
#include "ring.cuh"

// On the device, 151936 entries: a chain of 5 nodes 10.4 us (f32, drawn), 64 trees of 21 (bf16, not drawn) 21 us, 32 trees of 13 (f32, drawn,
// one to four passes each) 29 us. A pass is bound by latency and by the conversions to 64 bits, which an SM does sixteen of per cycle.
namespace dyn {

namespace {

// blocks of 256 against 512: 32 drawn trees 29.9 and 32.9 us, 64 trees 21.8 and 21.0
constexpr int VD_THREADS = 256, VD_WARPS = VD_THREADS / 32;
constexpr int VD_NODE = 5 * 8 + 3 * 4;  // bytes of shared memory of a node

struct VdArgs {
  const int64_t *tokens, *parents;  // [batch][nodes]
  int64_t parents_stride;           // 0: one tree for all
  const void *target, *draft;       // [batch][nodes][vocab]; draft may be NULL
  int64_t ts[2], ds[2];             // elements between batch entries and nodes
  const float* uniforms;            // [batch][nodes]
  int64_t *accepted, *path, *next;  // [batch], [batch][nodes], [batch]
  int nodes, blocks;                // blocks of a cluster
  int64_t vocab, run;               // entries of a warp
};

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive;\n\tbarrier.cluster.wait;" ::: "memory");
}
__device__ __forceinline__ double peer_f64(const double* p, int rank) {
  uint32_t at;
  double v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(at) : "memory");
  return v;
}

__device__ __forceinline__ double vd_value(float x) { return x; }
__device__ __forceinline__ double vd_value(__half x) { return __half2float(x); }
__device__ __forceinline__ double vd_value(__nv_bfloat16 x) { return __bfloat162float(x); }

// What is left of entry v (p and q: the rows' entries) after m refusals at the node, with `inv[j]` one over the sum behind the
// j-th (0 where nothing was left) and the tokens that are `gone`.
template <bool DRAFT>
__device__ __forceinline__ double left_of(double p, double q, int64_t v, int m, const double* inv, const int64_t* gone) {
  if (DRAFT) {
#pragma unroll 1
    for (int j = 0; j < m; j++) {
      p = (j ? p * inv[j] : p) - q;
      p = p < 0. ? 0. : p;  // NaN stays NaN
    }
  } else {
#pragma unroll 1
    for (int j = 0; j < m; j++)
      if (gone[j] == v) p = 0.;
  }
  return p;
}

template <typename T, bool DRAFT>
__global__ void __launch_bounds__(VD_THREADS, 4) verify_draft_kernel(const __grid_constant__ VdArgs a) {
  extern __shared__ double vd_shared[];
  double* p_of = vd_shared;                 // [nodes] target's entry of the node's token in its parent's row
  double* q_of = p_of + a.nodes;            // [nodes] the draft's
  double* inv = q_of + a.nodes;             // [nodes] 1 / Z_m at the present node
  int64_t* token = reinterpret_cast<int64_t*>(inv + a.nodes);
  int64_t* gone = token + a.nodes;          // tokens refused at the present node
  float* uniform = reinterpret_cast<float*>(gone + a.nodes);
  int* parent = reinterpret_cast<int*>(uniform + a.nodes);
  int* path = parent + a.nodes;
  __shared__ double own[2][VD_WARPS], all[16 * VD_WARPS], part[VD_WARPS];
  __shared__ long long s_found, s_last;
  __shared__ int s_node, s_m, s_i, s_count;  // where the walk stands
  __shared__ double s_z;

  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, n = a.nodes;
  const int rank = (int)blockIdx.x % a.blocks;
  const int64_t b = blockIdx.x / a.blocks;
  const T* target = static_cast<const T*>(a.target) + b * a.ts[0];
  const T* draft = static_cast<const T*>(a.draft) + (DRAFT ? b * a.ds[0] : 0);
  for (int i = tid; i < n; i += VD_THREADS) {
    const int64_t up = a.parents[b * a.parents_stride + i], t = a.tokens[b * n + i];
    const bool known = i > 0 && up >= 0 && up < i && t >= 0 && t < a.vocab;
    parent[i] = i > 0 && up >= 0 && up < i ? (int)up : -1;
    token[i] = t;
    uniform[i] = a.uniforms[b * n + i];
    p_of[i] = known ? vd_value(target[up * a.ts[1] + t]) : 0.;
    q_of[i] = known ? (DRAFT ? vd_value(draft[up * a.ds[1] + t]) : 1.) : 0.;
  }
  if (tid == 0) s_node = 0, s_m = 0, s_i = 1, s_count = 0, s_z = 1., path[0] = 0;
  __syncthreads();

  const int64_t lo = min(a.vocab, ((int64_t)rank * VD_WARPS + warp) * a.run), hi = min(a.vocab, lo + a.run);
  const int runs = a.blocks * VD_WARPS;
  const int per_lane = (runs + 31) / 32, from_run = min(runs, lane * per_lane), to_run = min(runs, from_run + per_lane);
  auto place = [&](int i) { return i % per_lane * 32 + i / per_lane; };  // in all[]: a lane's neighbours beside it
  int round = 0;
  double mine = 0., upto = 0., total = 0.;  // of this lane's runs, of those up to them, of all
  constexpr int N = 16 / sizeof(T), LOADS = DRAFT ? 16 / N : 4;
  struct alignas(16) Piece {
    T v[N];
  };
  // N entries' r after m refusals of drawn children
  auto all_left = [&](const T* pv, const T* qv, int m, double* r) {
#pragma unroll
    for (int e = 0; e < N; e++) r[e] = vd_value(pv[e]);
    for (int j = 0; j < m; j++) {
      const double by = j ? inv[j] : 1.;
#pragma unroll
      for (int e = 0; e < N; e++) {
        r[e] = r[e] * by - vd_value(qv[e]);
        r[e] = r[e] < 0. ? 0. : r[e];  // NaN stays NaN
      }
    }
  };
  // all[] = every warp's sum of what is left at `node` after m refusals, total = their sum: the same in all warps of all blocks
  auto sum_up = [&](int node, int m) {
    const T* p = target + (int64_t)node * a.ts[1];
    const T* q = DRAFT ? draft + (int64_t)node * a.ds[1] : nullptr;
    double sum = 0.;
    // 16 bytes at a time from the boundary below the run's first entry on; what lies outside the run, and q where it is not
    // aligned as p is, by single entries
    const int64_t base = lo - (int64_t)(reinterpret_cast<uintptr_t>(p + lo) % 16 / sizeof(T));
    bool touched = false;  // without a draft: one of the refused tokens is this warp's
    for (int j = 0; !DRAFT && j < m; j++) touched = touched || (gone[j] >= lo && gone[j] < hi);
    const bool alike = !DRAFT || (reinterpret_cast<uintptr_t>(p) - reinterpret_cast<uintptr_t>(q)) % 16 == 0;
    for (int64_t v0 = base + lane * N; v0 < hi; v0 += 32 * N * LOADS) {
      Piece pe[LOADS] = {}, qe[LOADS] = {};
#pragma unroll
      for (int j = 0; j < LOADS; j++) {
        const int64_t v = v0 + j * 32 * N;
        if (v >= lo && v + N <= hi) {
          pe[j] = *reinterpret_cast<const Piece*>(p + v);
          if (DRAFT && m && alike) qe[j] = *reinterpret_cast<const Piece*>(q + v);
        } else {
#pragma unroll
          for (int e = 0; e < N; e++)
            if (v + e >= lo && v + e < hi) {
              pe[j].v[e] = p[v + e];
              if (DRAFT && m && alike) qe[j].v[e] = q[v + e];
            }
        }
        if (DRAFT && m && !alike) {
#pragma unroll
          for (int e = 0; e < N; e++)
            if (v + e >= lo && v + e < hi) qe[j].v[e] = q[v + e];
        }
      }
#pragma unroll
      for (int j = 0; j < LOADS; j++) {
        if (!DRAFT && touched) {
          for (int g = 0; g < m; g++) {
            const int64_t at = gone[g] - (v0 + j * 32 * N);
#pragma unroll
            for (int e = 0; e < N; e++)
              if (at == e) pe[j].v[e] = T(0.f);
          }
        }
        double r[N];
        all_left(pe[j].v, qe[j].v, DRAFT ? m : 0, r);
#pragma unroll
        for (int e = 0; e < N; e++) sum += r[e];
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    // buffers alternate: one is written again behind a barrier that all its readers have passed
    if (lane == 0) own[round & 1][warp] = sum;
    cluster_sync();
    if (tid < runs) all[place(tid)] = peer_f64(&own[round & 1][tid % VD_WARPS], tid / VD_WARPS);
    round++;
    __syncthreads();
    // every warp adds them up for itself, a lane consecutive ones
    mine = 0.;
    for (int i = from_run; i < to_run; i++) mine += all[place(i)];
    upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double below = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += below;
    }
    total = __shfl_sync(0xffffffffu, upto, 31);
    if (m && tid == 0) inv[m] = total > 0. ? 1. / total : 0., s_z = total;
    __syncthreads();
  };
  for (int have_node = -1, have_m = -1;;) {
    if (warp == 0) {
      // on along the tree: to its end, or to a refusal whose sum has to be known first. 32 nodes at a time are looked through
      // for children of the one reached; all lanes try the same child
      int node = s_node, m = s_m, i = s_i, count = s_count;
      double z = s_z;
      for (bool stop = false; i < n && !stop;) {
        const int at = (i & ~31) + lane;
        const uint32_t children = __ballot_sync(0xffffffffu, at >= i && at < n && parent[at] == node);
        if (!children) {
          i = (i & ~31) + 32;
          continue;
        }
        const int c = (i & ~31) + __ffs(children) - 1;
        i = c + 1;
        const double r = left_of<DRAFT>(p_of[c], q_of[c], token[c], m, inv, gone);
        if ((double)uniform[c] * q_of[c] * z < r) {
          node = c, m = 0, z = 1., count++;
          if (lane == 0) path[count] = c;
        } else if (DRAFT) {
          m++, stop = true;
        } else {
          if (lane == 0) gone[m] = token[c];
          __syncwarp();
          m++, z -= r;
        }
      }
      if (lane == 0) s_node = node, s_m = m, s_i = i, s_count = count, s_z = z;
    }
    __syncthreads();
    if (s_node != have_node || s_m != have_m) sum_up(s_node, s_m);
    have_node = s_node, have_m = s_m;
    if (s_i >= n) break;
    __syncthreads();  // before the first warp goes on
  }
  const int node = s_node;
  int m = s_m;
  if (m && total == 0.) sum_up(node, m = 0);
  const double border = (double)uniform[0] * total;
  // the first run that reaches beyond the border, else the last one with anything in it
  int owner;
  double before_owner;
  {
    double before = upto - mine, before_last = 0., before_found = 0.;
    int last = -1, found = runs;
    for (int i = from_run; i < to_run; i++) {
      const double r = all[place(i)];
      if (r > 0.) {
        last = i, before_last = before;
        if (found == runs && before + r > border) found = i, before_found = before;
      }
      before += r;
    }
    const int first = __reduce_min_sync(0xffffffffu, found), final = __reduce_max_sync(0xffffffffu, last);
    owner = first < runs ? first : final;
    before_owner = __shfl_sync(0xffffffffu, first < runs ? before_found : before_last, max(0, owner) / per_lane);
  }
  if (rank == 0) {
    for (int i = tid; i < n; i += VD_THREADS) a.path[b * n + i] = i <= s_count ? path[i] : -1;
    if (tid == 0) a.accepted[b] = s_count;
  }
  const bool fine = total > 0. && total < __longlong_as_double(0x7ff0000000000000ll);
  if (!fine || owner < 0) {
    if (rank == 0 && tid == 0) a.next[b] = -1;
  } else if (owner / VD_WARPS == rank) {
    // the run's entries once more, over all warps of its block; a lane takes consecutive ones
    const T* p = target + (int64_t)node * a.ts[1];
    const T* q = DRAFT ? draft + (int64_t)node * a.ds[1] : nullptr;
    const int64_t begin = min(a.vocab, (int64_t)owner * a.run), end = min(a.vocab, begin + a.run);
    const int64_t per = (end - begin + VD_THREADS - 1) / VD_THREADS, from = min(end, begin + tid * per), to = min(end, from + per);
    auto entries = [&](int64_t v, double* r) {  // of v .. v + N - 1, zero from `to` on
      T pv[N] = {}, qv[N] = {};
#pragma unroll
      for (int e = 0; e < N; e++)
        if (v + e < to) {
          pv[e] = p[v + e];
          if (DRAFT && m) qv[e] = q[v + e];
        }
      for (int g = 0; !DRAFT && g < m; g++) {
#pragma unroll
        for (int e = 0; e < N; e++)
          if (gone[g] - v == e) pv[e] = T(0.f);
      }
      all_left(pv, qv, DRAFT ? m : 0, r);
    };
    double sum = 0., r[N];
    for (int64_t v = from; v < to; v += N) {
      entries(v, r);
#pragma unroll
      for (int e = 0; e < N; e++) sum += r[e];
    }
    double below_me = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double below = __shfl_up_sync(0xffffffffu, below_me, o);
      if (lane >= o) below_me += below;
    }
    if (lane == 31) part[warp] = below_me;
    if (tid == 0) s_found = a.vocab, s_last = -1;
    __syncthreads();
    double run = before_owner + (below_me - sum);
    for (int w = 0; w < warp; w++) run += part[w];
    long long found = a.vocab, last = -1;
    for (int64_t v = from; v < to; v += N) {
      if (per > N) entries(v, r);  // else they are at hand
#pragma unroll
      for (int e = 0; e < N; e++) {
        run += r[e];
        if (r[e] > 0.) {
          last = v + e;
          if (run > border && found == a.vocab) found = v + e;
        }
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      found = min(found, __shfl_xor_sync(0xffffffffu, found, o));
      last = max(last, __shfl_xor_sync(0xffffffffu, last, o));
    }
    if (lane == 0) atomicMin(&s_found, found), atomicMax(&s_last, last);
    __syncthreads();
    if (tid == 0) a.next[b] = s_found < a.vocab ? s_found : s_last;  // rounding may leave the border beyond the last sum
  }
  cluster_sync();  // no block leaves while another reads its sums
}

template <typename T, bool DRAFT>
int vd_run(VdArgs a, int64_t batch, cudaStream_t s) {
  auto kernel = verify_draft_kernel<T, DRAFT>;
  // blocks of a sequence: as many as leave all sequences running at once (up to four blocks per SM), no run of fewer than 128
  // entries. 32 drawn chains of 5 nodes (152000 entries): 14 blocks, of which 35 clusters fit, 15.5 us; 16, of which 31 do, 21.4. 48 bf16
  // trees of 21: 10 blocks 14.5, 8 17.8
  constexpr int FEW = 64 * VD_NODE, MANY = 1024 * VD_NODE;
  const int smem = a.nodes * VD_NODE;
  if (ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), smem <= FEW ? FEW : MANY)) return 1;
  const int64_t most = a.vocab / (VD_WARPS * 128);
  const int blocks = smem <= FEW ? blocks_per_cluster<verify_draft_kernel<T, DRAFT>, VD_THREADS, FEW>(batch, most)
                                 : blocks_per_cluster<verify_draft_kernel<T, DRAFT>, VD_THREADS, MANY>(batch, most);
  a.blocks = blocks;
  a.run = ((a.vocab + blocks * VD_WARPS - 1) / (blocks * VD_WARPS) + 31) / 32 * 32;
  DYN_CHECK(batch * blocks <= 0x7fffffff, "verify_draft: %lld sequences are too many for one call", (long long)batch);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(batch * blocks)), cfg.blockDim = dim3(VD_THREADS), cfg.dynamicSmemBytes = (size_t)smem, cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)blocks, attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr, cfg.numAttrs = 1;
  DYN_CUDA(cudaLaunchKernelEx(&cfg, kernel, a));
  count_launch();
  return 0;
}

template <typename T>
int vd_type(const VdArgs& a, int64_t batch, cudaStream_t s) {
  return a.draft ? vd_run<T, true>(a, batch, s) : vd_run<T, false>(a, batch, s);
}

}  // namespace

int launch_verify_draft(const int64_t* tokens, const int64_t* parents, int64_t parents_stride, const void* target,
                        const int64_t* target_strides, const void* draft, const int64_t* draft_strides, int type,
                        const float* uniforms, int64_t batch, int64_t nodes, int64_t vocab, int64_t* accepted, int64_t* path,
                        int64_t* next, cudaStream_t s) {
  if (batch == 0) return 0;
  VdArgs a{};
  a.tokens = tokens, a.parents = parents, a.parents_stride = parents_stride, a.target = target, a.draft = draft;
  a.ts[0] = target_strides[0], a.ts[1] = target_strides[1];
  if (draft) a.ds[0] = draft_strides[0], a.ds[1] = draft_strides[1];
  a.uniforms = uniforms, a.accepted = accepted, a.path = path, a.next = next, a.nodes = (int)nodes, a.vocab = vocab;
  if (type == E_F32) return vd_type<float>(a, batch, s);
  if (type == E_F16) return vd_type<__half>(a, batch, s);
  return vd_type<__nv_bfloat16>(a, batch, s);
}

}  // namespace dyn
