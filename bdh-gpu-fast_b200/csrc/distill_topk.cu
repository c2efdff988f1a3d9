// Distillation from the log probabilities that a teacher kept for its top tokens, and its
// gradient. With the student's z = x / temperature and p = softmax(z), and a row's list of K
// (token, teacher value) slots:
//
//   q_j   : tail = 0: softmax of the list's values; tail = 1: exp(value_j), and the class "every
//           other token" with r = max(0, 1 - sum_j q_j) against s = sum of p over unlisted tokens
//   loss  = w [ sum_j q_j (ln q_j - ln p[token_j]) + r (ln r - ln s) ]
//   dx_i  = w/temperature [ p_i (sum_j q_j + r) - r (p_i / s) [i unlisted] - sum_j q_j [i = token_j] ]
//
// A slot with token < 0 is empty; a repeated token's masses add; a row of weight 0 is not read.
// The unlisted tokens are summed by themselves, so that s keeps its digits when the list holds
// nearly everything. A row's slice is copied to shared memory (cp.async), the listed tokens are
// struck out there (-inf), the rest is summed from it and, in the same call, turned into the
// gradient from it, so that the logits cross HBM once. A warp takes a short row; else a CTA, or a
// cluster whose CTAs hold a slice each and exchange their sums through distributed shared memory.
// The backward from stored statistics has nothing to sum and streams.
#include <algorithm>
#include <string>

#include "bdh_sm100.h"
#include "internal.h"
#include "logits.cuh"
#include "tma_host.h"

namespace bdh {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kPiece = 16384;             // elements of a row per CTA of the streaming backward
constexpr int kSliceBytes = 48 * 1024;    // of a row per CTA, while the cluster may grow
static_assert(kThreads >= kTopMax, "one thread per slot");

template <int G>
__device__ __forceinline__ void group_sync() {
  if (G == 32) __syncwarp();
  else __syncthreads();
}

// A row's list in shared memory, K entries each (rounded up to a warp).
struct List {
  int* index;    // -1: empty slot; V: a token past the vocabulary
  float* lnq;
  float* q;
  float* z;      // the student's logit
  float* mass;   // q summed over the slots of the same token; below 0: not the token's first slot
};
struct GroupShared {
  SoftState part[kMaxCluster];
  SoftState warp_part[kWarps];
  SoftState top;       // softmax state of the listed tokens
  float total, r;      // mass of the list, of the class beside it
};

__host__ __device__ constexpr int list_room(int K) { return (K + 31) / 32 * 32; }
__host__ __device__ constexpr size_t list_smem(int K) {
  return sizeof(GroupShared) + 5 * sizeof(float) * static_cast<size_t>(list_room(K));
}
static_assert(sizeof(GroupShared) % 4 == 0, "lists follow");
__host__ __device__ constexpr size_t group_smem(int K, size_t slice_bytes) {
  return ((list_smem(K) + 15) & ~size_t(15)) + ((slice_bytes + 15) & ~size_t(15));
}
__device__ __forceinline__ List list_at(uint8_t* base, int K) {
  float* p = reinterpret_cast<float*>(base + sizeof(GroupShared));
  const int n = list_room(K);
  return {reinterpret_cast<int*>(p), p + n, p + 2 * n, p + 3 * n, p + 4 * n};
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, d));
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

// The row's list: q, its mass and the other class's, the student's logits of the listed tokens and
// their softmax state. Ends in a barrier of the group.
template <typename T, int G>
__device__ __forceinline__ void load_list(const DistillTopkArgs& a, const T* x, int64_t o, int64_t i,
                                          int tid, float c, GroupShared& sh, const List& l) {
  const int K = static_cast<int>(a.K), V = static_cast<int>(a.V);
  for (int j = tid; j < K; j += G) {
    const int64_t at = a.index[o * a.i_strides[0] + i * a.i_strides[1] + j * a.i_strides[2]];
    const float t = a.teacher[o * a.t_strides[0] + i * a.t_strides[1] + j * a.t_strides[2]];
    l.index[j] = at < 0 ? -1 : at < V ? static_cast<int>(at) : V;
    l.lnq[j] = at < 0 ? neg_inf() : t;
    l.z[j] = at >= 0 && at < V ? logit_at<T>(x, at) : neg_inf();
  }
  group_sync<G>();
  if (tid < 32) {
    float m = neg_inf();
    for (int j = tid; j < K; j += 32) m = max_nan(m, l.lnq[j]);
    m = warp_max(m);
    float shift = 0.0f;
    if (!a.tail && m != neg_inf()) {
      float s = 0.0f;
      for (int j = tid; j < K; j += 32) s += expf(l.lnq[j] - m);
      shift = m + logf(warp_sum(s));
    }
    float total = 0.0f;
    bool bad = false;
    for (int j = tid; j < K; j += 32) {
      const float v = l.lnq[j] - shift, q = expf(v);
      l.lnq[j] = v;
      l.q[j] = q;
      total += q;
      bad |= l.index[j] == V;
    }
    total = warp_sum(total);
    __syncwarp();
    // the masses of a repeated token go to its first slot
    SoftState top = soft_empty();
    int distinct = 0;
    for (int j = tid; j < K; j += 32) {
      const int at = l.index[j];
      float mass = at >= 0 ? 0.0f : -1.0f;
      if (at >= 0)
        for (int k = 0; k < K; ++k)
          if (l.index[k] == at) {
            if (k < j) {
              mass = -1.0f;
              break;
            }
            mass += l.q[k];
          }
      l.mass[j] = mass;
      if (!(mass < 0.0f)) {
        soft_add(top, l.z[j], c);
        ++distinct;
      }
    }
    top = soft_warp(top, c);
    distinct = __reduce_add_sync(0xffffffffu, distinct);
    bad = __any_sync(0xffffffffu, bad);
    if (tid == 0) {
      sh.top = top;
      sh.total = bad ? quiet_nan() : total;  // a token past the vocabulary: NaN throughout
      // where every token is listed there is no other class
      sh.r = a.tail && distinct < V ? max_nan(0.0f, 1.0f - total) : 0.0f;
    }
  }
  group_sync<G>();
}

// What the gradient needs of a row: dx_i = 2^(c (x_i - m) + shift) coef for unlisted tokens.
struct RowGradient {
  float m, shift, coef;        // unlisted: with a tail relative to their own sum s, however small
  float top_m, top_shift;      // listed: p = 2^(c (z - top_m) + top_shift)
  float scale, total;          // listed: scale (p total - mass)
  bool none;                   // no logit above -inf in the row
};
__device__ __forceinline__ RowGradient row_gradient(const DistillTopkArgs& a, const GroupShared& sh,
                                                    float m, float ln_s, float rest_m, float ln_rest,
                                                    float scale) {
  const float inv_t = 1.0f / a.temperature;
  RowGradient g;
  g.none = m == neg_inf();
  g.scale = scale * inv_t;
  g.total = sh.total + sh.r;
  g.top_m = m;
  g.top_shift = -ln_s * kLog2e;
  g.m = m;
  g.shift = g.top_shift;
  g.coef = g.scale * g.total;
  if (a.tail) {
    // p_i (total - r / s) = (p_i / s) (total s - r); nothing is unlisted and above -inf: all zeros
    const float s = expf((rest_m - m) * inv_t + ln_rest - ln_s);
    const bool empty = rest_m == neg_inf();
    g.m = empty ? 0.0f : rest_m;
    g.shift = empty ? neg_inf() : -ln_rest * kLog2e;
    g.coef = empty ? 0.0f : g.scale * (g.total * s - sh.r);
    if (g.total != g.total) g.coef = g.total;
  }
  return g;
}
// The gradient of the listed tokens of [from, to), over what the unlisted ones' formula left there.
template <typename T, int G>
__device__ __forceinline__ void write_listed(const RowGradient& g, const List& l, int K, int V, T* d,
                                             int from, int to, int tid, float c) {
  for (int j = tid; j < K; j += G) {
    const int at = l.index[j];
    if (at < from || at >= to || at >= V || l.mass[j] < 0.0f) continue;
    const float p = ex2(fmaf(l.z[j] - g.top_m, c, g.top_shift));
    logit_put(d, at, g.scale * (p * g.total - l.mass[j]));
  }
}

template <typename T>
__device__ __forceinline__ float row_weight(const DistillTopkArgs& a, int64_t o, int64_t i) {
  return a.weight.p != nullptr ? a.weight.p[o * a.weight.strides[0] + i * a.weight.strides[1]] : 1.0f;
}
struct NoSingle {
  __device__ __forceinline__ float operator()(float) const { return 0.0f; }
};
struct NoPair {
  __device__ __forceinline__ void operator()(float, float, float& a, float& b) const { a = b = 0.0f; }
};

template <typename T, int G>
__global__ void __launch_bounds__(kThreads) distill_topk_kernel(DistillTopkArgs a, int C,
                                                                size_t slice_bytes) {
  extern __shared__ __align__(16) uint8_t smem[];
  constexpr int kV = kVec<T>;
  const int tid = threadIdx.x % G, group = threadIdx.x / G;
  const int V = static_cast<int>(a.V), K = static_cast<int>(a.K);
  const uint32_t rank = G > 32 && C > 1 ? cta_rank() : 0;
  const int64_t row = G == 32 ? static_cast<int64_t>(blockIdx.x) * (kThreads / G) + group
                              : static_cast<int64_t>(blockIdx.x) / C;
  if (row >= a.outer * a.inner) return;  // whole warps of the warp form
  const int64_t o = static_cast<uint32_t>(row) / static_cast<uint32_t>(a.inner), i = row - o * a.inner;
  const T* x = static_cast<const T*>(a.logits) + o * a.l_strides[0] + i * a.l_strides[1];
  T* d = a.dlogits != nullptr
             ? static_cast<T*>(a.dlogits) + o * a.d_strides[0] + i * a.d_strides[1]
             : nullptr;

  // This CTA's slice: vectors [v0, v1) between the row's 16-byte boundaries, the row's head with
  // the first slice and its tail with the last; elements [from, to).
  const RowSpan span = row_span(x, V);
  const int per = (span.vecs + C - 1) / C;
  const int v0 = min(static_cast<int>(rank) * per, span.vecs), v1 = min(v0 + per, span.vecs);
  const int head = rank == 0 ? span.head : 0, tail = rank == C - 1 ? span.tail : 0;
  const int from = span.head + v0 * kV - head, to = span.head + v1 * kV + tail;
  const int n = to - from;

  const float w = row_weight<T>(a, o, i);
  if (w == 0.0f) {  // the whole cluster
    if (d != nullptr) map_row<T, G>(x + from, d + from, n, tid, true, NoSingle(), NoPair());
    if (tid == 0 && rank == 0) a.loss[row] = 0.0f;
    return;
  }
  if (G > 32 && C > 1) cluster_arrive();  // shared memory may be written once all CTAs have started

  uint8_t* base = smem + group * group_smem(K, slice_bytes);
  GroupShared& sh = *reinterpret_cast<GroupShared*>(base);
  const List l = list_at(base, K);
  T* buf = reinterpret_cast<T*>(base + ((list_smem(K) + 15) & ~size_t(15)));
  T* held = buf + (kV - head) % kV;  // held[e] is element from + e; vectors keep their alignment
  const uint4* vec = reinterpret_cast<const uint4*>(x + span.head) + v0;
  uint4* hvec = reinterpret_cast<uint4*>(held + head);
  const int vecs = v1 - v0;
  for (int v = tid; v < vecs; v += G)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(hvec + v)), "l"(vec + v)
                 : "memory");
  for (int e = tid; e < head + tail; e += G) {
    const int at = e < head ? e : n - tail + (e - head);
    held[at] = x[from + at];
  }
  const float inv_t = 1.0f / a.temperature, c = kLog2e * inv_t;
  load_list<T, G>(a, x, o, i, tid, c, sh, l);
  asm volatile("cp.async.wait_all;" ::: "memory");
  group_sync<G>();
  for (int j = tid; j < K; j += G) {
    const int at = l.index[j];
    if (at >= from && at < to) logit_put(held, at - from, neg_inf());
  }
  group_sync<G>();

  SoftState rest = soft_empty();
  for (int e = tid; e < head + tail; e += G)
    soft_add(rest, logit_at<T>(held, e < head ? e : n - tail + (e - head)), c);
  for (int b = 0; b < vecs; b += G * kUnroll) {
    float xs[kUnroll * kV];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int v = b + u * G + tid;
      float part[kV];
      unpack(v < vecs ? hvec[v] : void_vec<T>(), part);
#pragma unroll
      for (int e = 0; e < kV; ++e) xs[u * kV + e] = part[e];
    }
    float m = xs[0];
#pragma unroll
    for (int e = 1; e < kUnroll * kV; ++e) m = max_nan(m, xs[e]);
    if (!(m <= rest.m)) soft_raise(rest, max_nan(m, rest.m), c);
    if (rest.m != neg_inf()) soft_sum<false>(rest, xs, c);
  }
  rest = soft_warp(rest, c);
  if (G > 32) {
    if ((threadIdx.x & 31) == 0) sh.warp_part[threadIdx.x >> 5] = rest;
    __syncthreads();
    rest = sh.warp_part[0];
#pragma unroll
    for (int k = 1; k < kWarps; ++k) rest = soft_merge(rest, sh.warp_part[k], c);
    if (C > 1) {
      cluster_wait();
      if (tid < C) {
        const uint32_t at = peer_smem(&sh.part[rank], tid);
        peer_store(at, rest.m);
        peer_store(at + 4, rest.s);
      }
      cluster_arrive();
      cluster_wait();
      rest = {sh.part[0].m, sh.part[0].s, 0.0f};
      for (int k = 1; k < C; ++k) rest = soft_merge(rest, {sh.part[k].m, sh.part[k].s, 0.0f}, c);
    }
  }
  rest.a = 0.0f;
  const SoftState all = soft_merge(rest, {sh.top.m, sh.top.s, 0.0f}, c);
  const bool none = all.m == neg_inf(), rest_none = rest.m == neg_inf();
  const float ln_s = none ? neg_inf() : logf(all.s);
  const float ln_rest = rest_none ? neg_inf() : logf(rest.s);

  if (rank == 0 && tid < 32) {
    float loss = 0.0f;
    for (int j = tid; j < K; j += 32) {
      const float q = l.q[j], z = l.z[j];
      const float lp = none || z == neg_inf() ? neg_inf() : (z - all.m) * inv_t - ln_s;
      if (!(q <= 0.0f)) loss = fmaf(q, l.lnq[j] - lp, loss);
    }
    loss = warp_sum(loss);
    if (tid == 0) {
      if (sh.r > 0.0f) {
        const float ls = rest_none ? neg_inf() : (rest.m - all.m) * inv_t + ln_rest - ln_s;
        loss = fmaf(sh.r, logf(sh.r) - ls, loss);
      }
      a.loss[row] = sh.total != sh.total ? quiet_nan() : w * loss;
      if (a.stats != nullptr) {
        a.stats[4 * row] = all.m;
        a.stats[4 * row + 1] = ln_s;
        a.stats[4 * row + 2] = rest.m;
        a.stats[4 * row + 3] = ln_rest;
      }
    }
  }
  if (d == nullptr) return;

  const RowGradient g = row_gradient(a, sh, all.m, ln_s, rest.m, ln_rest, w);
  auto dense = [&](float v) { return ex2(fmaf(v - g.m, c, g.shift)) * g.coef; };
  const F2 nm2 = f2(-g.m, -g.m), c2 = f2(c, c), shift2 = f2(g.shift, g.shift), coef2 = f2(g.coef, g.coef);
  auto pair = [&](float x0, float x1, float& d0, float& d1) {
    float y0, y1;
    f2_split(f2_fma(f2_add(f2(x0, x1), nm2), c2, shift2), y0, y1);
    f2_split(f2_mul(f2(ex2(y0), ex2(y1)), coef2), d0, d1);
  };
  T* out = d + from + head;
  if ((reinterpret_cast<uintptr_t>(out) & 15u) == 0) {
    for (int e = tid; e < head + tail; e += G) {
      const int at = e < head ? e : n - tail + (e - head);
      logit_put(d, from + at, g.none ? 0.0f : dense(logit_at<T>(held, at)));
    }
    for (int v = tid; v < vecs; v += G) {
      float xs[kV], ds[kV];
      unpack(hvec[v], xs);
#pragma unroll
      for (int e = 0; e < kV; e += 2) pair(xs[e], xs[e + 1], ds[e], ds[e + 1]);
      if (g.none) {
#pragma unroll
        for (int e = 0; e < kV; ++e) ds[e] = 0.0f;
      }
      store_vec(out + static_cast<int64_t>(v) * kV, ds);
    }
  } else {  // x and d lie differently in their vectors
    for (int e = tid; e < n; e += G)
      logit_put(d, from + e, g.none ? 0.0f : dense(logit_at<T>(held, e)));
  }
  if (g.none) return;
  group_sync<G>();
  write_listed<T, G>(g, l, K, V, d, from, to, tid, c);
}

template <typename T, int G>
__global__ void __launch_bounds__(kThreads) distill_topk_bwd_kernel(DistillTopkArgs a, int pieces,
                                                                    int piece) {
  extern __shared__ __align__(16) uint8_t smem[];
  const int tid = threadIdx.x % G, group = threadIdx.x / G;
  const int V = static_cast<int>(a.V), K = static_cast<int>(a.K);
  const uint32_t unit = blockIdx.x * (kThreads / G) + group;
  const int64_t row = unit / static_cast<uint32_t>(pieces);
  if (row >= a.outer * a.inner) return;  // whole warps of the warp form
  const int64_t o = static_cast<uint32_t>(row) / static_cast<uint32_t>(a.inner), i = row - o * a.inner;
  const int from = static_cast<int>(unit - static_cast<uint32_t>(row) * pieces) * piece;
  const int n = min(piece, V - from);
  const T* x = static_cast<const T*>(a.logits) + o * a.l_strides[0] + i * a.l_strides[1];
  T* d = static_cast<T*>(a.dlogits) + o * a.d_strides[0] + i * a.d_strides[1];
  const float w = row_weight<T>(a, o, i);
  if (w == 0.0f) {
    map_row<T, G>(x + from, d + from, n, tid, true, NoSingle(), NoPair());
    return;
  }
  uint8_t* base = smem + group * group_smem(K, 0);
  GroupShared& sh = *reinterpret_cast<GroupShared*>(base);
  const List l = list_at(base, K);
  const float c = kLog2e / a.temperature;
  load_list<T, G>(a, x, o, i, tid, c, sh, l);
  const float* st = a.stats + 4 * row;
  const float up = a.g_loss.p[o * a.g_loss.strides[0] + i * a.g_loss.strides[1]];
  const RowGradient g = row_gradient(a, sh, st[0], st[1], st[2], st[3], w * up);
  auto dense = [&](float v) { return ex2(fmaf(v - g.m, c, g.shift)) * g.coef; };
  const F2 nm2 = f2(-g.m, -g.m), c2 = f2(c, c), shift2 = f2(g.shift, g.shift), coef2 = f2(g.coef, g.coef);
  auto pair = [&](float x0, float x1, float& d0, float& d1) {
    float y0, y1;
    f2_split(f2_fma(f2_add(f2(x0, x1), nm2), c2, shift2), y0, y1);
    f2_split(f2_mul(f2(ex2(y0), ex2(y1)), coef2), d0, d1);
  };
  map_row<T, G>(x + from, d + from, n, tid, g.none, dense, pair);
  if (g.none) return;
  group_sync<G>();
  write_listed<T, G>(g, l, K, V, d, from, from + n, tid, c);
}

int launch_check(const char* what, cudaError_t e) {
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) {
    set_error(std::string(what) + ": " + cudaGetErrorString(e));
    return BDH_ERR_CUDA;
  }
  return BDH_OK;
}

template <typename T, int G>
int launch_forward(const DistillTopkArgs& a, int cluster, cudaStream_t stream) {
  const int64_t rows = a.outer * a.inner;
  constexpr int kGroups = kThreads / G;
  // a slice's vectors, and one more for the row's head and one for its tail
  const size_t slice = (static_cast<size_t>((a.V / kVec<T> + cluster - 1) / cluster) + 2) * 16;
  const size_t smem = kGroups * group_smem(static_cast<int>(a.K), slice);
  auto* kern = distill_topk_kernel<T, G>;
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               static_cast<int>(smem));
    if (e != cudaSuccess) return launch_check("distill_topk shared memory", e);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(G == 32 ? (rows + kGroups - 1) / kGroups : rows * cluster));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 1 : 0;
  return launch_check("distill_topk launch", cudaLaunchKernelEx(&cfg, kern, a, cluster, slice));
}

template <typename T>
int forward_by_size(const DistillTopkArgs& a, cudaStream_t stream) {
  if (a.V <= 1024) return launch_forward<T, 32>(a, 1, stream);
  int dev = 0;
  cudaGetDevice(&dev);
  const int64_t rows = a.outer * a.inner, bytes = a.V * static_cast<int64_t>(sizeof(T));
  int cluster = 1;
  while (cluster < kMaxCluster &&
         (bytes > static_cast<int64_t>(cluster) * kSliceBytes ||
          (rows * cluster < 4 * sm_count(dev) && bytes >= cluster * int64_t(32768))))
    cluster *= 2;
  if (rows * cluster >= int64_t(1) << 31) {
    set_error("distill_topk: too many rows for this vocabulary");
    return BDH_ERR_INVALID;
  }
  return launch_forward<T, kThreads>(a, cluster, stream);
}

template <typename T>
int backward_by_size(const DistillTopkArgs& a, cudaStream_t stream) {
  const int64_t rows = a.outer * a.inner;
  const size_t lists = group_smem(static_cast<int>(a.K), 0);
  if (a.V <= 1024) {
    const unsigned grid = static_cast<unsigned>((rows + kWarps - 1) / kWarps);
    distill_topk_bwd_kernel<T, 32><<<grid, kThreads, kWarps * lists, stream>>>(a, 1, static_cast<int>(a.V));
  } else {
    const int64_t pieces = (a.V + kPiece - 1) / kPiece;
    if (rows * pieces >= int64_t(1) << 31) {
      set_error("distill_topk_bwd: too many rows for this vocabulary");
      return BDH_ERR_INVALID;
    }
    distill_topk_bwd_kernel<T, kThreads><<<static_cast<unsigned>(rows * pieces), kThreads, lists, stream>>>(
        a, static_cast<int>(pieces), kPiece);
  }
  return launch_check("distill_topk_bwd launch", cudaSuccess);
}

}  // namespace

int launch_distill_topk(const DistillTopkArgs& a, cudaStream_t stream) {
  if (a.outer * a.inner == 0) return BDH_OK;
  return a.dtype == BDH_DTYPE_F32 ? forward_by_size<float>(a, stream)
                                  : forward_by_size<uint16_t>(a, stream);
}

int launch_distill_topk_bwd(const DistillTopkArgs& a, cudaStream_t stream) {
  if (a.outer * a.inner == 0) return BDH_OK;
  return a.dtype == BDH_DTYPE_F32 ? backward_by_size<float>(a, stream)
                                  : backward_by_size<uint16_t>(a, stream);
}

}  // namespace bdh
