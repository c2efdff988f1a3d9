// Log probabilities of given tokens with entropy and top alternatives, and their gradient:
//
//   z = x / temperature, lse = ln sum_i exp(z_i), logprob = z[token] - lse,
//   entropy = - sum_i p_i ln p_i, and the K largest logits' (z_i - lse, i)
//   dx_i = 1/temperature [ p_i (g_lse - g_logprob - sum_j g_top_j - g_entropy (ln p_i + entropy))
//                          + [i = token] g_logprob + sum_j [i = top_j] g_top_j ]
//
// The forward reads a row once. A group of threads (8 to 32 lanes for a short row, a warp for many rows
// of a middling length, else a CTA of 128 or 256 threads, or a cluster of up to 8 with a slice of the row
// each) keeps a softmax state per thread and joins them at the end, through distributed shared memory in a
// cluster. For the top list it keeps the maximum of every batch of vectors that a thread reads (a cell);
// the K-th largest of the threads' own maxima bounds the K-th largest logit from below, so that only cells
// above it are looked at again, a few cache lines, and the few candidates are put in order by counting.
//
// What bounds it (times here and beside the constants: the kernels alone, from a CUDA graph): without a
// list, memory, with the exponentials close behind. 4096 rows of 131072 in bf16 take 162 us, 6.6 TB/s; the
// exponential's unit is then busy 76% of the time and 0.67 of the issue slots are used (7.2 instructions an
// element; run for seconds, at the clocks that the power limit leaves, 186). With a list the issue slots
// (0.75 used): 2048 rows of 65536 with K = 64 take 67 us, 4.0 TB/s, of which the search after the stream is
// 13, half of it the second look at the cells above the bound. A single row of 131072 with K = 20 takes 8.3
// us (with K = 128 13), the latencies of some ten steps that wait for one another (0.16 of the issue slots of
// its 8 CTAs). The backward reads and writes at 6.2 to 6.6 TB/s: 81 us for 1024 rows of 131072 in bf16.
// Through a list it is further off, since every thread adds a row's K upstream gradients and every entry
// looks for itself among the others: 16384 rows of 256 in bf16 4.7 us without, with K = 16 11.3, with
// K = 64 65; 2048 rows of 65536 83, with K = 64 125.
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
// Longest list that a warp bounds by its lanes' largest, one each; longer ones by each element of a short
// row, by 4 items a lane of a middling one. By lanes and otherwise, bf16: 1200 rows of 256 with K = 16 5.0
// and 5.3 us, 16384 rows of 1000 with K = 4 29 and 48, with K = 16 33 and 50, with K = 20 36 and 51; 8192 rows
// of 4096 with K = 4 20.7 and 21.2, with K = 16 24.7 and 24.0, with K = 20 27.3 and 25.7.
constexpr int kWarpTop = 16;
// Steps that bring the bound close where the list is more than a quarter of the items that it is searched
// among: with 24 of 32 lanes' largest above it 45 of 256 elements are, with 16 of them 22. 16384 rows of
// 256 with K = 16, a warp each: 18.9 us, 21 without; with K = 5 16 and 15.5. 8192 rows of 4096 with
// K = 128 (of 256 items): 135 us, 156 without.
__host__ __device__ constexpr int close_steps(int K, int items) { return 4 * K > items ? 10 : 0; }
// A warp takes a row of up to this size where there are this many rows for every SM: no thread waits for
// another warp, and the loads of 32 rows are in flight on an SM. 8192 rows in bf16, by warps against by
// CTAs: 4096 long 13 and 38 us (with K = 20 26 and 73), 16384 long 47 and 63 us (63 and 103), 32768 long
// 97 and 99 (158 and 140). 592 rows, 4 an SM: 4096 long 4.1 and 4.7 us (8.6 and 7.8), 8192 long 5.4 and
// 4.9 (11 and 8).
constexpr int kWarpRowBytes = 32 * 1024, kWarpRows = 8;
// Longest list of a warp's or a half CTA's row (half of their items). 8192 rows of 4096 with K = 64: 61 us by
// warps, 94 by CTAs; with K = 100 by a warp 1550 us, its items no longer bound it.
constexpr int kWarpList = 64;
// Rows of up to this size that are not split are read by CTAs of 128 threads: more rows' loads, joins and
// searches pass at a time. 8192 rows in bf16 by 128 and by 256 threads: 20000 long 60 and 76 us (with
// K = 20 93 and 123), 50021 long 129 and 141 (168 and 189), 65536 long 167 and 170 (203 and 210); 2048 rows
// of 100003 74 and 72 us (91 and 86). (By 64 threads 20000 long 59, with K = 32 89 and 96 by 128; 50021
// long 132, with K = 32 228 and 172.)
constexpr int kHalfBytes = 112 * 1024;
// Cells are batches of vectors, or single vectors in a warp's row whose batches would be fewer than four
// for every entry of the list. 8192 rows in bf16, by batches and by vectors: 1500 long with K = 4 15.7 and
// 16.9 us, with K = 32 34 and 25; 1025 long with K = 32 229 (more candidates than there is room for) and
// 22. In a CTA's longer rows the stream pays more than the search saves: 2048 rows of 65536 66 and 83 us.
// What a warp's bound is searched among, of a lane: its cells' largest in so many groups. (8192 rows of
// 2048 with K = 32: 24.5 us, with every cell by itself 28.)
constexpr int kLaneItems = 4;
// Cells per thread; longer rows put more batches into a cell. With up to 24, 48 and 96 cells: 300 rows of
// 500000 in fp32 with K = 20 120, 120 and 159 us (96: two CTAs an SM), in bf16 with K = 64 83,
// 100 and 100; 300 rows of 1000000 in bf16 with K = 20 146, 146 and 162; one row of 4000000 in fp32 46, 47
// and 52.
constexpr int kMaxCells = 48;
constexpr int kMaxCluster = 8;
// A row by itself is split over a cluster in slices of at least 16 KB, but not one of 32 KB or less, which
// a CTA has read before a cluster has met: one row of 16384 in bf16 3.3 us whole and 3.5 split, of 65536
// 4.8 whole, 3.7 split, of 131072 8.2 and 4.1.
constexpr int kUnsplitBytes = 32 * 1024, kSliceBytes = 16 * 1024;

// Threads' maxima that may lie above the bound besides the K wanted: the search for it ends early. With
// K / 8 + 2, K / 4 + 4 and K / 2 + 8: 16384 rows of 256 in bf16 with K = 5 12.8, 11.6 and 12.3 us, with K = 16
// 14.8, 15.7 and 19.3; 8192 rows of 4096 with K = 20 27.1, 25.7 and 28.9; 2048 rows of 65536 with K = 64 67.0,
// 67.3 and 69.5, with K = 8 61.0, 60.2 and 60.8; a row of 131072 in fp32 with K = 20 8.3, 8.5 and 8.7.
__host__ __device__ constexpr int top_slack(int K) { return K / 4 + 4; }
// Room for candidates: every element of the vectors that hold the maxima (a row of equal values),
// and of the row's ends.
template <typename T>
constexpr int candidate_room(int K) {
  return (K + top_slack(K)) * kVec<T> + 16;
}

// A key that at least K of a group's items are at or above, and as a rule few more, by bisection:
// first over the values' keys, [lo, hi] holding all of them, then, where more items share the value
// found than may be taken, over the index up to which they count. from(v): items with value key >= v;
// tied(v, i): items with value key v and an index up to i. The first `close` steps are taken even where
// there are few more than K.
template <typename From, typename Tied>
__device__ __forceinline__ uint64_t list_bound(int K, uint32_t lo, uint32_t hi, int V, int close,
                                               From from, Tied tied) {
  const int most = K + top_slack(K);
  int n = 0x7fffffff;
  ++hi;  // at least K items from lo, fewer than K from hi
  while (hi - lo > 1 && n > (--close >= 0 ? K : most)) {
    const uint32_t mid = lo + (hi - lo) / 2;
    const int now = from(mid);
    if (now >= K) {
      lo = mid;
      n = now;
    } else {
      hi = mid;
    }
  }
  uint32_t last = 0xffffffffu;
  if (n > most) {
    const int above = from(lo + 1);
    uint32_t left = 0, right = static_cast<uint32_t>(V);
    n = 0x7fffffff;
    while (left < right && n > most - above) {
      const uint32_t mid = left + (right - left) / 2;
      const int now = tied(lo, mid);
      if (now >= K - above) {
        right = mid;
        n = now;
      } else {
        left = mid + 1;
      }
    }
    last = right;
  }
  return (static_cast<uint64_t>(lo) << 32) | (0xffffffffu - last);
}

struct ForwardPlan {
  int cells, cell_shift;  // per thread, and log2 of the vectors in a cell: one, or some batches
  int cluster;
};

__device__ __forceinline__ uint64_t warp_max_key(uint64_t k) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const uint64_t other = __shfl_xor_sync(0xffffffffu, k, o);
    k = other > k ? other : k;
  }
  return k;
}

// A given token's logit, asked for before the row is read so that the two loads' latencies pass
// under it.
struct Token {
  bool given, left_out;  // a token inside the vocabulary; the index that counts as none
  float z;
};
template <typename T>
__device__ __forceinline__ Token load_token(const TokenLogprobsArgs& a, const T* x, int64_t o, int64_t i) {
  Token t = {false, false, 0.0f};
  const int64_t at = a.tokens[o * a.t_strides[0] + i * a.t_strides[1]];
  t.left_out = at == a.ignore_index;
  t.given = !t.left_out && at >= 0 && at < a.V;
  if (t.given) t.z = logit_at<T>(x, at);
  return t;
}

// The row's figures from its softmax state (one thread); returns ln of the sum.
__device__ __forceinline__ float ln_sum(const SoftState& st) {
  return st.m == neg_inf() ? neg_inf() : logf(st.s);  // -inf: nothing above -inf in the row
}
__device__ __forceinline__ float logprob_of(float z, const SoftState& st, float ln_s, float inv_t) {
  return st.m == neg_inf() ? neg_inf() : (z - st.m) * inv_t - ln_s;
}
__device__ __forceinline__ void write_figures(const TokenLogprobsArgs& a, int64_t row, const SoftState& st,
                                              float ln_s, float inv_t, const Token& t) {
  const bool none = st.m == neg_inf();
  if (a.lse != nullptr) a.lse[row] = none ? neg_inf() : fmaf(st.m, inv_t, ln_s);
  if (a.entropy != nullptr) a.entropy[row] = none ? 0.0f : ln_s - kLn2 * st.a / st.s;
  if (a.stats != nullptr) {  // (at any float: a caller's own allocation)
    a.stats[2 * row] = st.m;
    a.stats[2 * row + 1] = ln_s;
  }
  if (a.tokens != nullptr)
    a.logprob[row] = t.left_out ? 0.0f : t.given ? logprob_of(t.z, st, ln_s, inv_t) : quiet_nan();
}

// ------------------------------------------------------------------ lanes for a short row
// Rows of at most kShort elements stay in registers: L lanes hold E elements each of a row, and one or
// two of its unaligned ends; the maximum first, then the sums. With few lanes a row the shuffles and
// the row's own figures serve several rows at once (a byte model's 256: 4 rows a warp; 16352 such rows
// in bf16 take 4.1 us, 7.0 with a warp each). 2 us are the launch; the rest is the row's latencies.
constexpr int kShort = 1024;

template <typename T, int L, int E>
struct ShortRow {
  static constexpr int kV = kVec<T>, kVecs = E / kV, kEnds = L < 16 ? 2 : 1, kN = E + kEnds;
  RowSpan span;
  int end[kEnds];  // elements of the row's ends, or -1
  float x[kN];     // the vectors', then the ends'; -inf where there is none
  __device__ __forceinline__ int index(int u, int e, int lane) const {
    return span.head + (u * L + lane) * kV + e;
  }
  __device__ __forceinline__ bool has(int u, int lane) const { return u * L + lane < span.vecs; }
  __device__ __forceinline__ void place(const T* p, int V, int lane) {
    span = row_span(p, V);
    if (kEnds == 2) {
      end[0] = lane < span.head ? lane : -1;
      end[kEnds - 1] = lane < span.tail ? V - span.tail + lane : -1;
    } else {
      end[0] = lane < span.head ? lane : lane - span.head < span.tail ? V - span.tail + lane - span.head : -1;
    }
  }
  __device__ __forceinline__ void load(const T* p, int lane) {
    const uint4* vec = reinterpret_cast<const uint4*>(p + span.head);
    uint4 w[kVecs];
#pragma unroll
    for (int u = 0; u < kVecs; ++u) w[u] = has(u, lane) ? __ldg(vec + u * L + lane) : void_vec<T>();
#pragma unroll
    for (int i = 0; i < kEnds; ++i) x[E + i] = end[i] >= 0 ? logit_at<T>(p, end[i]) : neg_inf();
#pragma unroll
    for (int u = 0; u < kVecs; ++u) {
      float part[kV];
      unpack(w[u], part);
#pragma unroll
      for (int e = 0; e < kV; ++e) x[u * kV + e] = part[e];
    }
  }
};

template <typename T, int L, int E>
__global__ void __launch_bounds__(kThreads) token_logprobs_short_kernel(TokenLogprobsArgs a, FastDiv inner) {
  const int lane = threadIdx.x % L;
  const int rows = static_cast<int>(a.outer * a.inner);
  int row = static_cast<int>(blockIdx.x * (kThreads / L) + threadIdx.x / L);
  const bool live = row < rows;
  if (!__any_sync(0xffffffffu, live)) return;
  if (!live) row = rows - 1;  // (the warp's other rows need these lanes)
  int o, i;
  inner.divmod(row, o, i);
  const T* x = static_cast<const T*>(a.logits) + o * a.l_strides[0] + i * a.l_strides[1];
  ShortRow<T, L, E> r;
  r.place(x, static_cast<int>(a.V), lane);
  Token tok = {false, true, 0.0f};
  if (lane == 0 && a.tokens != nullptr) tok = load_token(a, x, o, i);
  r.load(x, lane);
  const SoftState st = soft_of_lanes<true, L>(r.x, a.c);
  if (lane == 0 && live) write_figures(a, row, st, ln_sum(st), a.inv_t, tok);
}

// With a list, a warp for a row: the elements' keys. Lists up to kWarpTop are bounded by the lanes'
// largest keys, where enough lanes have any and that leaves no more candidates than there is room for;
// longer ones by the elements' own. (16384 rows of 100 with K = 12, which 13 to 16 lanes hold: 22 us by the
// elements, 31 by the lanes; 200 with K = 16 20 by the lanes.)
constexpr int kShortRoom = kTopMax + top_slack(kTopMax) + 1;

template <typename T, int E>
__global__ void __launch_bounds__(kThreads) token_list_short_kernel(TokenLogprobsArgs a, FastDiv inner) {
  using Row = ShortRow<T, 32, E>;
  constexpr int kV = Row::kV, kVecs = Row::kVecs;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kWarps + warp;
  if (row >= a.outer * a.inner) return;
  int o, i;
  inner.divmod(static_cast<int>(row), o, i);
  const int V = static_cast<int>(a.V);
  const T* x = static_cast<const T*>(a.logits) + o * a.l_strides[0] + i * a.l_strides[1];
  Row r;
  r.place(x, V, lane);
  Token tok = {false, true, 0.0f};
  if (lane == 0 && a.tokens != nullptr) tok = load_token(a, x, o, i);
  r.load(x, lane);
  const float inv_t = a.inv_t;
  const SoftState st = soft_of_lanes<true, 32>(r.x, a.c);
  const float ln_s = ln_sum(st);
  if (lane == 0) write_figures(a, row, st, ln_s, inv_t, tok);

  __shared__ uint64_t room[kWarps][kShortRoom];
  __shared__ int found[kWarps];
  uint64_t* cand = room[warp];
  const int K = static_cast<int>(a.K);
  auto index_of = [&](int u, int e) { return r.index(u, e, lane); };
  const int edge = r.end[0];
  uint32_t keys[E], own = 0, own_at = 0xffffffffu;
  const uint32_t edge_key = edge >= 0 ? value_key(r.x[E]) : 0u;
#pragma unroll
  for (int u = 0; u < kVecs; ++u)
#pragma unroll
    for (int e = 0; e < kV; ++e) {
      const uint32_t k = r.has(u, lane) ? value_key(r.x[u * kV + e]) : 0u;
      keys[u * kV + e] = k;
      if (k > own) {
        own = k;
        own_at = index_of(u, e);
      }
    }
  if (edge_key > own) {
    own = edge_key;
    own_at = edge;
  }
  const uint32_t hi = __reduce_max_sync(0xffffffffu, own);
  uint64_t bound = 0;
  bool by_element = true;
  if (K <= kWarpTop && 2 * __popc(__ballot_sync(0xffffffffu, own != 0)) >= 3 * K) {
    const uint32_t lo = __reduce_min_sync(0xffffffffu, own != 0 ? own : 0xffffffffu);
    bound = list_bound(
        K, lo, hi, V, close_steps(K, 32),
        [&](uint32_t v) { return __popc(__ballot_sync(0xffffffffu, own >= v)); },
        [&](uint32_t v, uint32_t at) { return __popc(__ballot_sync(0xffffffffu, own == v && own_at <= at)); });
    by_element = false;
  }
  uint32_t least = 0, last = 0;  // the bound's value, and of elements with it the last index
  auto above = [&](uint32_t k, int at) {
    return k > least || (k == least && static_cast<uint32_t>(at) <= last);  // (an empty place's key is 0)
  };
  auto count = [&](auto in) {
    int n = in(edge_key, edge) ? 1 : 0;
#pragma unroll
    for (int u = 0; u < kVecs; ++u)
#pragma unroll
      for (int e = 0; e < kV; ++e) n += in(keys[u * kV + e], index_of(u, e)) ? 1 : 0;
    return static_cast<int>(__reduce_add_sync(0xffffffffu, n));
  };
  uint32_t bits = 0;  // this lane's candidates in its vectors
  bool at_edge = false;
  int n = kShortRoom + 1;  // the row's candidates
  auto mark = [&] {
    least = static_cast<uint32_t>(bound >> 32);
    last = key_index(bound);
    bits = 0;
#pragma unroll
    for (int u = 0; u < kVecs; ++u)
#pragma unroll
      for (int e = 0; e < kV; ++e) bits |= above(keys[u * kV + e], index_of(u, e)) ? 1u << (u * kV + e) : 0u;
    at_edge = above(edge_key, edge);
    n = __reduce_add_sync(0xffffffffu, __popc(bits) + (at_edge ? 1 : 0));
  };
  if (!by_element) mark();
  if (n > kShortRoom) {
    bound = list_bound(
        K, 1u, hi, V, 0, [&](uint32_t v) { return count([&](uint32_t k, int) { return k >= v; }); },
        [&](uint32_t v, uint32_t at) {
          return count([&](uint32_t k, int j) { return k == v && static_cast<uint32_t>(j) <= at; });
        });
    mark();
  }
  if (lane == 0) found[warp] = 0;
  __syncwarp();
  if (bits != 0 || at_edge) {
    int to = atomicAdd(&found[warp], __popc(bits) + (at_edge ? 1 : 0));
    if (at_edge) cand[to++] = top_key(r.x[E], edge);
    for (; bits != 0; bits &= bits - 1) {
      const int q = __ffs(bits) - 1, at = index_of(q / kV, q % kV);
      cand[to++] = top_key(logit_at<T>(x, at), at);  // (from L1: registers have no index)
    }
  }
  __syncwarp();
  for (int j = lane; j < n; j += 32) {
    const uint64_t mine = cand[j];
    int place = 0;
    for (int q = 0; q < n; ++q) place += cand[q] > mine ? 1 : 0;
    if (place < K) {
      a.top_index[row * K + place] = key_index(mine);
      a.top_logprob[row * K + place] =
          logprob_of(key_value(static_cast<uint32_t>(mine >> 32)), st, ln_s, inv_t);
    }
  }
}

// Over each L neighbouring lanes (all lanes take part).
template <int L, typename F>
__device__ __forceinline__ uint32_t lanes_reduce(uint32_t v, F f) {
#pragma unroll
  for (int d = L / 2; d > 0; d >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, d));
  return v;
}
template <int L>
__device__ __forceinline__ int lanes_sum(int v) {
  auto sum = [](uint32_t x, uint32_t y) { return x + y; };
  return static_cast<int>(lanes_reduce<L>(static_cast<uint32_t>(v), sum));
}

// The lanes' values below this one.
template <int L>
__device__ __forceinline__ int lanes_before(int v, int lane) {
  int to = v;
#pragma unroll
  for (int d = 1; d < L; d *= 2) {
    const int before = __shfl_up_sync(0xffffffffu, to, d, L);
    if (lane >= d) to += before;
  }
  return to - v;
}

// Many short rows with a short list: L lanes a row, as without a list. The bound is searched among the
// largest of every four of a lane's elements, for the warp's rows in step; what is not below it goes to
// the row's places in shared memory, where counting puts it in order. Bound by its instructions and by
// how few warps there are to hide their latencies (74 registers: 3 CTAs an SM): with K = 16 16384 rows take
// 593 instructions each, at 0.65 of the issue slots, in 512 CTAs of which 444 run at a time. 16384 rows
// of 256 in bf16: K = 1 10.8 us, K = 5 11.6, K = 16 15.7; with a warp a row 15.4, 16.0 and 19.1; but 1200
// rows with K = 5 5.8 against 4.4 (K = 16: 8.1 and 5.1), and where a list is more than a sixteenth of the
// row, so that the bound lets much of it through, 25 against 22 (16384 rows of 100 with K = 16).
constexpr int kLanesRoom = 64;
constexpr int kLanesRows = 32;  // for every SM

template <typename T, int L, int E>
__global__ void __launch_bounds__(kThreads, 3) token_list_lanes_kernel(TokenLogprobsArgs a, FastDiv inner) {
  using Row = ShortRow<T, L, E>;
  constexpr int kV = Row::kV, kVecs = Row::kVecs, kEnds = Row::kEnds, kCells = E / 4;
  static_assert(E <= 32 && kV % 4 == 0, "a bit for each of a lane's elements; a cell is of one vector");
  __shared__ uint64_t room[kThreads / L][kLanesRoom];
  const int lane = threadIdx.x % L;
  const int rows = static_cast<int>(a.outer * a.inner);
  int row32 = static_cast<int>(blockIdx.x * (kThreads / L) + threadIdx.x / L);
  const bool live = row32 < rows;
  if (!__any_sync(0xffffffffu, live)) return;
  if (!live) row32 = rows - 1;  // (the warp's other rows need these lanes)
  int o, i;
  inner.divmod(row32, o, i);
  const int64_t row = row32;
  const int V = static_cast<int>(a.V), K = static_cast<int>(a.K), most = K + top_slack(K);
  const T* x = static_cast<const T*>(a.logits) + o * a.l_strides[0] + i * a.l_strides[1];
  Row r;
  r.place(x, V, lane);
  Token tok = {false, true, 0.0f};
  if (lane == 0 && a.tokens != nullptr) tok = load_token(a, x, o, i);
  r.load(x, lane);
  const float inv_t = a.inv_t;
  const SoftState st = soft_of_lanes<true, L>(r.x, a.c);
  const float ln_s = ln_sum(st);
  if (lane == 0 && live) write_figures(a, row, st, ln_s, inv_t, tok);

  auto high = [](uint32_t p, uint32_t q) { return max(p, q); };
  uint32_t cells[kCells + 1], lo = 0xffffffffu, hi = 0;
  int some = 0;
  cells[kCells] = 0;
#pragma unroll
  for (int e = 0; e < kEnds; ++e)
    if (r.end[e] >= 0) cells[kCells] = max(cells[kCells], value_key(r.x[E + e]));
#pragma unroll
  for (int q = 0; q < kCells; ++q) {
    const float m = max_nan(max_nan(r.x[4 * q], r.x[4 * q + 1], r.x[4 * q + 2]), r.x[4 * q + 3]);
    cells[q] = r.has(4 * q / kV, lane) ? value_key(m) : 0u;
  }
#pragma unroll
  for (int q = 0; q <= kCells; ++q) {
    if (cells[q] != 0) lo = min(lo, cells[q]);
    hi = max(hi, cells[q]);
    some += cells[q] != 0 ? 1 : 0;
  }
  lo = lanes_reduce<L>(lo, [](uint32_t p, uint32_t q) { return min(p, q); });
  hi = lanes_reduce<L>(hi, high);
  some = lanes_sum<L>(some);
  const uint32_t top = hi++;
  for (int n = some;;) {
    const bool go = some >= K && hi - lo > 1 && n > most;
    if (!__any_sync(0xffffffffu, go)) break;
    const uint32_t mid = lo + (hi - lo) / 2;
    int now = 0;
#pragma unroll
    for (int q = 0; q <= kCells; ++q) now += cells[q] >= mid ? 1 : 0;
    now = lanes_sum<L>(now);
    if (!go) continue;
    if (now >= K) {
      lo = mid;
      n = now;
    } else {
      hi = mid;
    }
  }
  if (some < K) lo = 1;  // fewer cells than entries: every element

  uint32_t there = 0;  // this lane's elements
#pragma unroll
  for (int u = 0; u < kVecs; ++u)
    if (r.has(u, lane)) there |= ((1u << kV) - 1) << (u * kV);
  uint32_t bits = 0, ends = 0;  // the candidates among them; nothing at or above the bound is left out
  const float least = key_value(lo);
#pragma unroll
  for (int e = 0; e < E; ++e) bits |= !(r.x[e] < least) ? 1u << e : 0u;
  bits &= there;
#pragma unroll
  for (int e = 0; e < kEnds; ++e) ends |= r.end[e] >= 0 && !(r.x[E + e] < least) ? 1u << e : 0u;
  int held = __popc(bits) + __popc(ends), n = lanes_sum<L>(held);
  uint64_t* cand = room[threadIdx.x / L];
  const bool wide = n > kLanesRoom;
  if (__any_sync(0xffffffffu, wide)) {
    // Equal values, or large ones close together: the bound among the elements themselves, by value and
    // where needed by index.
    auto each = [&](auto f) {
#pragma unroll 1
      for (int at = lane; at < V; at += L) f(value_key(logit_at<T>(x, at)), at);
    };
    auto count = [&](auto in) {
      int now = 0;
      each([&](uint32_t k, int at) { now += in(k, at) ? 1 : 0; });
      return lanes_sum<L>(now);
    };
    int from = V, right = V;
    hi = wide ? top + 1 : hi;
    for (;;) {
      const bool go = wide && hi - lo > 1 && from > kLanesRoom;
      if (!__any_sync(0xffffffffu, go)) break;
      const uint32_t mid = lo + (hi - lo) / 2;
      const int now = count([&](uint32_t k, int) { return k >= mid; });
      if (!go) continue;
      if (now >= K) {
        lo = mid;
        from = now;
      } else {
        hi = mid;
      }
    }
    const int above = count([&](uint32_t k, int) { return k > lo; });
    for (int left = 0, tied = V;;) {
      const bool go = wide && from > kLanesRoom && left < right && above + tied > kLanesRoom;
      if (!__any_sync(0xffffffffu, go)) break;
      const int mid = left + (right - left) / 2;
      const int now = count([&](uint32_t k, int at) { return k == lo && at <= mid; });
      if (!go) continue;
      if (now >= K - above) {
        right = mid;
        tied = now;
      } else {
        left = mid + 1;
      }
    }
    if (wide) held = 0;
    const uint64_t bound = (static_cast<uint64_t>(lo) << 32) | (0xffffffffu - static_cast<uint32_t>(right));
    auto above_it = [&](uint32_t k, int at) {
      return wide && ((static_cast<uint64_t>(k) << 32) | (0xffffffffu - static_cast<uint32_t>(at))) >= bound;
    };
    each([&](uint32_t k, int at) { held += above_it(k, at) ? 1 : 0; });
    n = lanes_sum<L>(held);
    int to = lanes_before<L>(held, lane);
    each([&](uint32_t k, int at) {
      if (above_it(k, at))
        cand[to++] = (static_cast<uint64_t>(k) << 32) | (0xffffffffu - static_cast<uint32_t>(at));
    });
  }
  int to = lanes_before<L>(held, lane);
  if (!wide) {
#pragma unroll
    for (int e = 0; e < kEnds; ++e)
      if (ends >> e & 1) cand[to++] = top_key(logit_at<T>(x, r.end[e]), r.end[e]);
    for (; bits != 0; bits &= bits - 1) {  // (from L1: registers have no index)
      const int e = __ffs(bits) - 1, at = r.index(e / kV, e % kV, lane);
      cand[to++] = top_key(logit_at<T>(x, at), at);
    }
  }
  __syncwarp();
  for (int j = lane; j < n; j += L) {
    const uint64_t mine = cand[j];
    int place = 0;
    for (int q = 0; q < n; ++q) place += cand[q] > mine ? 1 : 0;
    if (place < K && live) {
      a.top_index[row * K + place] = key_index(mine);
      a.top_logprob[row * K + place] =
          logprob_of(key_value(static_cast<uint32_t>(mine >> 32)), st, ln_s, inv_t);
    }
  }
}

// ------------------------------------------- a warp, a CTA or a cluster for longer rows
// Shared memory of one group of G threads; with a list its cells, candidates, lists and queue follow.
struct GroupShared {
  SoftState part[kMaxCluster];  // of the cluster's CTAs, in the first
  SoftState warp_part[kWarps];
  uint64_t best[kWarps];
  uint64_t bound;
  int found, queued, close, kept;
  float m, ln_s;                // the row's
};
// The list's bound is searched among the threads' largest cells; in a warp's row among kLaneItems of a
// lane, and for a list of up to kWarpTop among the lanes' largest.
template <int G>
constexpr int bound_items = G == 32 ? 32 * kLaneItems : G;
// Candidates and queue; the items' indices, which are needed before them, take their place.
template <typename T, int G>
__host__ __device__ constexpr size_t candidate_smem(int K, int cluster) {
  size_t n = static_cast<size_t>(candidate_room<T>(K)) * (sizeof(uint64_t) + sizeof(int));
  const size_t at = bound_items<G> * sizeof(int);
  const size_t all = static_cast<size_t>(cluster) * K * sizeof(uint64_t);  // what the slices' lists leave
  if (n < at) n = at;
  if (n < all) n = all;
  return (n + 7) & ~size_t(7);
}
constexpr size_t kGroupShared = (sizeof(GroupShared) + 7) & ~size_t(7);
template <typename T, int G>
__host__ __device__ constexpr size_t group_smem(int K, int cells, int cluster) {
  size_t n = kGroupShared;
  if (K > 0)
    n += candidate_smem<T, G>(K, cluster) + static_cast<size_t>(cluster) * K * sizeof(uint64_t) +
         sizeof(int) * (static_cast<size_t>(cells + 1) * G + (G == 32 ? 0 : G));
  return (n + 15) & ~size_t(15);
}
template <int G>
__device__ __forceinline__ void group_sync() {
  if (G <= 32) __syncwarp();
  else __syncthreads();
}

// The K largest of n > K different keys, none below lo, and at most top_slack(K) more (one warp); how many.
// Counting places takes n^2 comparisons, so it is worth the steps where there are many: 8192 rows of 1025
// with K = 128, where nearly every element is a candidate, 220 us, 1270 without.
__device__ __forceinline__ int keep_largest(const uint64_t* keys, int n, int K, uint64_t lo, uint64_t* out,
                                            int lane) {
  uint64_t hi = 0;
  for (int k = lane; k < n; k += 32) hi = max(hi, keys[k]);
  hi = warp_max_key(hi) + 1;
  int above = n;
  while (hi - lo > 1 && above > K + top_slack(K)) {
    const uint64_t mid = lo + (hi - lo) / 2;
    int now = 0;
    for (int k = lane; k < n; k += 32) now += keys[k] >= mid ? 1 : 0;
    now = __reduce_add_sync(0xffffffffu, now);
    if (now >= K) {
      lo = mid;
      above = now;
    } else {
      hi = mid;
    }
  }
  int kept = 0;
  for (int from = 0; from < n; from += 32) {
    const uint64_t mine = from + lane < n ? keys[from + lane] : 0;
    const bool in = mine >= lo && from + lane < n;
    const uint32_t who = __ballot_sync(0xffffffffu, in);
    if (in) out[kept + __popc(who & ((1u << lane) - 1))] = mine;
    kept += __popc(who);
  }
  return kept;
}

// f(key, its place) for n different keys, by counting those above each: more than a warp's are shared
// out to two or four threads each while the CTA has them.
template <int G, typename F>
__device__ __forceinline__ void rank_by_counting(const uint64_t* keys, int n, int tid, F f) {
  if (G > 32 && n > 32 && 2 * n <= G) {
    const int split = 4 * n <= G ? 4 : 2, part = tid & (split - 1), k = tid / split;
    if ((tid & ~31) / split >= n) return;  // whole warps
    const uint64_t mine = keys[min(k, n - 1)];
    int place = 0;
    for (int q = part; q < n; q += split) place += keys[q] > mine ? 1 : 0;
    place += __shfl_xor_sync(0xffffffffu, place, 1);
    if (split > 2) place += __shfl_xor_sync(0xffffffffu, place, 2);
    if (part == 0 && k < n) f(mine, place);
    return;
  }
  for (int k = tid; k < n; k += G) {
    const uint64_t mine = keys[k];
    int place = 0;
    for (int q = 0; q < n; ++q) place += keys[q] > mine ? 1 : 0;
    f(mine, place);
  }
}

template <int G>
constexpr int cta_threads = G == 32 ? kThreads : G;  // groups of a warp share a CTA

// Threads of an SM: 1024; with a list 1280, 48 registers each: while some search, others read (2048 rows
// of 65536 with K = 64: 74 us with 1024, 69 with 1280).
template <typename T, int G, bool TOP>
__global__ void __launch_bounds__(cta_threads<G>, (TOP && G > 32 ? 1280 : 1024) / cta_threads<G>)
    token_logprobs_kernel(TokenLogprobsArgs a, ForwardPlan plan, FastDiv inner) {
  extern __shared__ __align__(16) uint8_t smem[];
  constexpr int kV = kVec<T>, U = kUnroll;
  const int K = static_cast<int>(a.K), V = static_cast<int>(a.V);
  const int C = G == 32 ? 1 : plan.cluster;
  const uint32_t rank = C > 1 ? cta_rank() : 0;
  const int tid = threadIdx.x % G, group = threadIdx.x / G;
  const uint32_t row32 =
      G == 32 ? blockIdx.x * (cta_threads<G> / G) + group : blockIdx.x / static_cast<uint32_t>(C);
  const int64_t row = row32;
  if (row >= a.outer * a.inner) return;  // whole warps of the warp form
  if (C > 1) cluster_arrive();  // every CTA's shared memory may be written once all have started
  int o, i;
  inner.divmod(static_cast<int>(row32), o, i);
  const T* x = static_cast<const T*>(a.logits) + o * a.l_strides[0] + i * a.l_strides[1];
  const float inv_t = a.inv_t, c = a.c, slack = kBaseSlack / c;

  uint8_t* base = smem + group * group_smem<T, G>(K, plan.cells, C);
  GroupShared& sh = *reinterpret_cast<GroupShared*>(base);
  uint64_t* cand = reinterpret_cast<uint64_t*>(base + kGroupShared);
  int* queue = reinterpret_cast<int*>(cand + candidate_room<T>(K));  // cells to look at again
  uint32_t* item_at = reinterpret_cast<uint32_t*>(cand);  // where a value's first element is
  uint64_t* lists = reinterpret_cast<uint64_t*>(base + kGroupShared + candidate_smem<T, G>(K, C));
  uint32_t* cells = reinterpret_cast<uint32_t*>(lists + C * K);  // [cell][thread]: largest value key
  uint32_t* items = cells + (plan.cells + 1) * G;                // threads' largest (not for a warp)

  // This CTA's slice of the vectors; the row's head goes with the first slice, its tail with the last.
  const RowSpan span = row_span(x, V);
  const uint4* vec = reinterpret_cast<const uint4*>(x + span.head);
  const int per = (span.vecs + C - 1) / C;
  const int v0 = min(static_cast<int>(rank) * per, span.vecs), v1 = min(v0 + per, span.vecs);
  uint4 first[U];
  load_batch<T, G>(first, vec, v0, v1, tid);
  Token tok = {false, true, 0.0f};
  // One warp (the second of a CTA, while the first is at the list's bound) has the row's figures.
  const bool figurer = G == 32 || (threadIdx.x >> 5) == 1;
  if (figurer && (threadIdx.x & 31) == 0 && rank == 0 && a.tokens != nullptr) tok = load_token(a, x, o, i);
  int edge = -1;  // this thread's element of the row's ends
  if (rank == 0 && tid < span.head) edge = tid;
  if (rank == C - 1 && tid >= 8 && tid - 8 < span.tail) edge = V - span.tail + tid - 8;
  const float edge_x = edge >= 0 ? logit_at<T>(x, edge) : neg_inf();
  const int cell_vecs = 1 << plan.cell_shift;
  SoftSums<true> sums;

  int cell = 0, in_cell = 0;          // TOP: cells written, vectors in the open one
  uint32_t own = 0;                   // largest key of the thread
  float cell_max = neg_inf();
  auto put_cell = [&](float largest, bool any) {
    const uint32_t k = any ? value_key(largest) : 0u;
    cells[cell++ * G + tid] = k;
    own = max(own, k);
  };
  stream<T, G>(first, vec, v0, v1, tid, [&](const uint4 (&w)[U], int b, auto fill, auto refill) {
    float largest;
    if (TOP && cell_vecs == 1) {
      largest = neg_inf();
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint4 one[1] = {w[u]};
        const float m = max_of(one, T());
        if (b + u * G < v1) put_cell(m, b + u * G + tid < v1);
        largest = max_nan(largest, m);
      }
    } else {
      largest = max_of(w, T());
      if (TOP) {
        cell_max = max_nan(cell_max, largest);
        in_cell += U;
        if (in_cell == cell_vecs || b + G * U >= v1) {
          put_cell(cell_max, b + (U - in_cell) * G + tid < v1);
          in_cell = 0;
          cell_max = neg_inf();
        }
      }
    }
    sums.template add<T>(w, largest, c, slack, a.least, fill, refill);
  });
  SoftState st = sums.wide ? soft_slowly<T, G>(vec, v0, v1, tid, c) : sums.state(c);
  if (edge >= 0) soft_add(st, edge_x, c);
  st = soft_join(st, c);
  if (G > 32 && (threadIdx.x & 31) == 0) sh.warp_part[threadIdx.x >> 5] = st;

  auto figures = [&](const SoftState& row_st) {
    const float ln_s = ln_sum(row_st);
    if ((threadIdx.x & 31) == 0) {
      sh.m = row_st.m;
      sh.ln_s = ln_s;
      write_figures(a, row, row_st, ln_s, inv_t, tok);
    }
  };
  auto join_warps = [&] {
    if (!figurer) return;
    if (G > 32) st = soft_join((threadIdx.x & 31) < G / 32 ? sh.warp_part[threadIdx.x & 31] : soft_empty(), c);
    if (C == 1) figures(st);
  };
  if (!TOP) {
    group_sync<G>();
    join_warps();
  } else {
    const uint32_t edge_key = edge >= 0 ? value_key(edge_x) : 0u;
    cells[cell * G + tid] = edge_key;  // the last cell: the row's ends
    own = max(own, edge_key);
    if (G > 32) items[tid] = own;
    if (tid == 0) sh.found = sh.queued = sh.kept = 0;
    group_sync<G>();
    join_warps();
    constexpr int kItems = G == 32 ? kLaneItems : G / 32;  // per lane of the searching warp
    const bool few = G == 32 && K <= kWarpTop;
    const int most = K + top_slack(K);
    // First by value (one warp): at least K items at or above lo, as a rule not many more.
    if (tid < 32) {
      uint32_t mine[kItems], lo = 0xffffffffu, hi = 0;
      int some = 0;
#pragma unroll
      for (int n = 0; n < kItems; ++n) mine[n] = G > 32 ? items[n * 32 + tid] : few && n == 0 ? own : 0u;
      if (G == 32 && !few)
        for (int q = 0; q <= cell; q += kItems)
#pragma unroll
          for (int n = 0; n < kItems; ++n)
            if (q + n <= cell) mine[n] = max(mine[n], cells[(q + n) * 32 + tid]);
#pragma unroll
      for (int n = 0; n < kItems; ++n) {
        if (mine[n] != 0) lo = min(lo, mine[n]);
        hi = max(hi, mine[n]);
        some += mine[n] != 0 ? 1 : 0;
      }
      lo = __reduce_min_sync(0xffffffffu, lo);
      hi = __reduce_max_sync(0xffffffffu, hi);
      some = __reduce_add_sync(0xffffffffu, some);
      auto from = [&](uint32_t v) {
        if (few) return __popc(__ballot_sync(0xffffffffu, mine[0] >= v));
        int n = 0;
#pragma unroll
        for (int k = 0; k < kItems; ++k) n += mine[k] >= v ? 1 : 0;
        return static_cast<int>(__reduce_add_sync(0xffffffffu, n));
      };
      uint64_t bound = 0;  // fewer than K items: every element is a candidate
      if (some >= K) {
        int n = some, close = close_steps(K, few ? 32 : bound_items<G>);
        ++hi;
        while (hi - lo > 1 && n > (--close >= 0 ? K : most)) {
          const uint32_t mid = lo + (hi - lo) / 2;
          const int now = from(mid);
          if (now >= K) {
            lo = mid;
            n = now;
          } else {
            hi = mid;
          }
        }
        // the low word: how many items may still be dropped by index, where too many share lo
        bound = (static_cast<uint64_t>(lo) << 32) | (n > most ? static_cast<uint32_t>(from(lo + 1)) + 1u : 0u);
      }
      if (tid == 0) sh.bound = bound;
    }
    group_sync<G>();
    uint64_t bound = sh.bound;
    const uint32_t lo = static_cast<uint32_t>(bound >> 32);
    uint32_t last = 0xffffffffu;  // of elements with value lo, those up to this index
    auto first_at = [&](int q) {  // the first element with value lo of this thread's cell q
      if (q == cell) return static_cast<uint32_t>(edge);
      for (int n = 0; n < cell_vecs; ++n) {
        const int v = v0 + (q * cell_vecs + n) * G + tid;
        if (v >= v1) break;
        float part[kV];
        unpack(__ldg(vec + v), part);
#pragma unroll
        for (int e = 0; e < kV; ++e)
          if (value_key(part[e]) == lo) return static_cast<uint32_t>(span.head + v * kV + e);
      }
      return 0xffffffffu;
    };
    if (static_cast<uint32_t>(bound) != 0) {
      // Then, where too many items share the value, by the index of its first element in each.
      const int above = static_cast<int>(static_cast<uint32_t>(bound)) - 1;
      const int groups = G == 32 && !few ? kLaneItems : 1;
      for (int n = 0; n < groups; ++n) {
        uint32_t at = 0xffffffffu;
        if (own >= lo)
          for (int q = n; q <= cell; q += groups)
            if (cells[q * G + tid] == lo) at = min(at, first_at(q));
        item_at[n * G + tid] = at;
      }
      group_sync<G>();
      if (tid < 32) {
        const int n_items = groups * G;
        uint32_t left = 0, right = static_cast<uint32_t>(V);
        int n = n_items;
        while (left < right && n > most - above) {
          const uint32_t mid = left + (right - left) / 2;
          int now = 0;
          for (int k = tid; k < n_items; k += 32) now += item_at[k] <= mid ? 1 : 0;
          now = __reduce_add_sync(0xffffffffu, now);
          if (now >= K - above) {
            right = mid;
            n = now;
          } else {
            left = mid + 1;
          }
        }
        if (tid == 0) sh.bound = right;
      }
      group_sync<G>();
      last = static_cast<uint32_t>(sh.bound);  // item_at is done with: candidates may come
      bound = (static_cast<uint64_t>(lo) << 32) | (0xffffffffu - last);
    }
    const int room = candidate_room<T>(K);
    auto offer = [&](float v, int at) {
      const uint64_t k = top_key(v, at);
      if (k >= bound) {
        const int n = atomicAdd(&sh.found, 1);
        if (n < room) cand[n] = k;
      }
    };
    if (edge >= 0) offer(edge_x, edge);
    if (own >= lo)
      for (int q = 0; q < cell; ++q) {
        const uint32_t k = cells[q * G + tid];
        const int v = v0 + q * cell_vecs * G + tid;
        if (k < lo || v >= v1 || (k == lo && static_cast<uint32_t>(span.head + v * kV) > last)) continue;
        const int n = atomicAdd(&sh.queued, 1);
        if (n < room) queue[n] = v;
      }
    group_sync<G>();
    // All threads on the queued cells' vectors, one each, so that their loads are under way together.
    // What is not below the bound's value (NaN is not) is looked at by its key.
    const int queued = sh.queued;
    const float least = key_value(lo);
    if (queued <= room)
      for (int n = tid; n < queued * cell_vecs; n += G) {
        const int v = queue[n >> plan.cell_shift] + (n & (cell_vecs - 1)) * G;
        if (v >= v1) continue;
        float part[kV];
        unpack(__ldg(vec + v), part);
        uint32_t some = 0;
#pragma unroll
        for (int e = 0; e < kV; ++e) some |= !(part[e] < least) ? 1u << e : 0u;
        for (; some != 0; some &= some - 1) {
          const int at = span.head + v * kV + __ffs(some) - 1;
          offer(logit_at<T>(x, at), at);  // (from L1: registers have no index)
        }
      }
    uint64_t* list = lists + rank * K;  // this slice's K largest in order
    for (int k = tid; k < K; k += G) list[k] = 0;
    group_sync<G>();
    const int found = queued <= room ? sh.found : room + 1;
    if (found <= room) {
      int n = found;
      const uint64_t* keys = cand;
      if (found > 2 * K + 32) {  // many more than wanted: one warp looks for a bound among them
        uint64_t* few_keys = reinterpret_cast<uint64_t*>(queue);  // (done with, and room for K + slack)
        if (tid < 32) {
          const int kept = keep_largest(cand, found, K, bound, few_keys, tid);
          if (tid == 0) sh.close = kept;
        }
        group_sync<G>();
        n = sh.close;
        keys = few_keys;
      }
      rank_by_counting<G>(keys, n, tid, [&](uint64_t mine, int place) {
        if (place < K) list[place] = mine;
      });
    } else {
      // More elements above the bound than there is room for: large values that keep to few
      // cells. K rounds of "the largest below the last one" over the slice.
      uint64_t before = ~0ull;
      for (int k = 0; k < K; ++k) {
        uint64_t best = 0;
        auto look = [&](float v, int at) {
          const uint64_t q = top_key(v, at);
          if (q < before && q > best) best = q;
        };
        if (edge >= 0) look(edge_x, edge);
        for (int v = v0 + tid; v < v1; v += G) {
          float part[kV];
          unpack(__ldg(vec + v), part);
#pragma unroll
          for (int e = 0; e < kV; ++e) look(part[e], span.head + v * kV + e);
        }
        best = warp_max_key(best);
        if (G > 32) {
          __syncthreads();
          if ((threadIdx.x & 31) == 0) sh.best[threadIdx.x >> 5] = best;
          __syncthreads();
          for (int w = 0; w < G / 32; ++w) best = sh.best[w] > best ? sh.best[w] : best;
        }
        if (tid == 0) list[k] = best;
        before = best;
      }
    }
    group_sync<G>();
  }

  if (C > 1) {
    cluster_wait();
    if (figurer && (threadIdx.x & 31) == 0) {
      const uint32_t to = peer_smem(&sh.part[rank], 0);
      peer_store(to, st.m);
      peer_store(to + 4, st.s);
      peer_store(to + 8, st.a);
    }
    if (TOP && rank != 0)
      for (int k = tid; k < K; k += G) peer_store(peer_smem(lists + rank * K + k, 0), lists[rank * K + k]);
    cluster_arrive();
    cluster_wait();
    if (rank != 0) return;
    if (figurer) figures(soft_join((threadIdx.x & 31) < C ? sh.part[threadIdx.x & 31] : soft_empty(), c));
  }

  if (TOP) {
    const uint64_t* sorted = lists;
    int n_sorted = K;
    if (C > 1) {
      // Of the slices' lists, what is not below the largest of their last entries nor below the least of
      // their K/C-th (at least K are not): few more than K (by the last entries alone a row of 131072 with
      // K = 128 kept some 900 and took 45 us, not 13). A slice shorter than K has zeros at its list's end.
      const int share = (K + C - 1) / C;
      uint64_t floor = 1, least = ~0ull;
      for (int r = 0; r < C; ++r) {
        floor = max(floor, lists[r * K + K - 1]);
        least = min(least, lists[r * K + share - 1]);
      }
      floor = max(floor, least);
      for (int n = tid; n < C * K; n += G) {
        const uint64_t mine = lists[n];
        if (mine < floor) continue;
        cand[atomicAdd(&sh.kept, 1)] = mine;  // (room for C K: candidate_smem)
      }
      __syncthreads();
      sorted = cand;
      n_sorted = sh.kept;
    }
    const SoftState row_st = {sh.m, 0.0f, 0.0f};
    const float ln_s = sh.ln_s;
    for (int n = tid; n < n_sorted; n += G) {
      const uint64_t mine = sorted[n];
      int place = n;
      if (C > 1) {
        place = 0;
        for (int q = 0; q < n_sorted; ++q) place += cand[q] > mine ? 1 : 0;
      }
      if (place < K) {
        a.top_index[row * K + place] = key_index(mine);
        a.top_logprob[row * K + place] =
            logprob_of(key_value(static_cast<uint32_t>(mine >> 32)), row_st, ln_s, inv_t);
      }
    }
  }
}

// The gradient writes as many bytes as it reads and needs nothing of a row but its two statistics, so
// a row is cut into pieces of kPiece elements for the CTAs. The token and the list get their own terms in
// the CTA whose piece they lie in: the element is computed again with its term added, so that it is
// rounded once. 1024 rows of 131072 in bf16: 82 us, with pieces of 8192 91 and of 32768 85 us (in fp32
// 163, 158 and 168).
constexpr int kPiece = 16384;
// Many rows of up to this size are a warp's each (8192 rows in bf16, by warps against by CTAs: 2048 long
// 12.5 and 28.7 us, 4096 long 26 and 37, 8192 long 47 and 50; 1184 rows of 8192 9.1 and 8.0), short ones
// of fewer lanes (16384 rows of 256: 5.1 us by 8 lanes, 8.9 by warps).
constexpr int kWarpGradBytes = 8 * 1024;

struct GradShared {
  int index[kTopMax + 1];
  float add[kTopMax + 1];
};

template <typename T, int G>
__global__ void __launch_bounds__(kThreads) token_logprobs_bwd_kernel(TokenLogprobsBwdArgs a,
                                                                      FastDiv pieces, int piece,
                                                                      FastDiv inner) {
  extern __shared__ __align__(16) uint8_t smem[];
  const int tid = threadIdx.x % G, group = threadIdx.x / G;
  GradShared& sh = *(reinterpret_cast<GradShared*>(smem) + group);  // with a list only
  int row32, nth, o, i;
  pieces.divmod(static_cast<int>(blockIdx.x * (kThreads / G) + group), row32, nth);
  const int64_t row = row32;
  if (row >= a.f.outer * a.f.inner) return;  // whole warps of the warp form
  inner.divmod(row32, o, i);
  const int V = static_cast<int>(a.f.V), K = a.g_top != nullptr ? static_cast<int>(a.f.K) : 0;
  const int from = nth * piece, n = min(piece, V - from);
  const T* x = static_cast<const T*>(a.f.logits) + o * a.f.l_strides[0] + i * a.f.l_strides[1];
  T* d = static_cast<T*>(a.dlogits) + o * a.d_strides[0] + i * a.d_strides[1];
  const float inv_t = a.f.inv_t, c = a.f.c;
  const float m = a.f.stats[2 * row], ln_s = a.f.stats[2 * row + 1];
  const bool none = m == neg_inf();
  auto up = [&](const RowGrad& g) {
    return g.p != nullptr ? g.p[o * g.strides[0] + i * g.strides[1]] : 0.0f;
  };
  float g_tok = a.f.tokens != nullptr ? up(a.g_logprob) : 0.0f;
  const float g_ent = up(a.g_entropy);
  const float ent = a.g_entropy.p != nullptr ? a.f.entropy[row] : 0.0f;
  float sum = up(a.g_lse);
  int tok = -1;
  if (a.g_logprob.p != nullptr && a.f.tokens != nullptr) {
    const int64_t t = a.f.tokens[o * a.f.t_strides[0] + i * a.f.t_strides[1]];
    if (t == a.f.ignore_index) g_tok = 0.0f;
    else if (t >= 0 && t < V) tok = static_cast<int>(t);
    else sum = quiet_nan();  // no such token: its log probability is NaN, and so is this
  }
  sum -= g_tok;
  if (K > 0) {
    for (int k = tid; k <= K; k += G) {
      sh.index[k] = k == 0 ? tok : static_cast<int>(a.f.top_index[row * K + k - 1]);
      sh.add[k] = k == 0 ? g_tok : a.g_top[row * K + k - 1];
    }
    group_sync<G>();
    for (int k = 1; k <= K; ++k) sum -= sh.add[k];
  }
  // p (sum - g_entropy (ln p + entropy)) / temperature
  const RowMap dense(c, none ? 0.0f : m, none ? 0.0f : ln_s * kLog2e, (sum - g_ent * ent) * inv_t,
                     -g_ent * kLn2 * inv_t);
  map_row<T, G>(x + from, d + from, n, tid, none, dense);
  if (none) return;
  if (K == 0) {
    if (tok < from || tok >= from + n) return;
    group_sync<G>();
    if (tid == 0) logit_put(d, tok, fmaf(g_tok, inv_t, row_map<G>(dense, logit_at<T>(x, tok))));
    return;
  }
  group_sync<G>();
  for (int k = tid; k <= K; k += G) {
    const int at = sh.index[k];
    bool mine = at >= from && at < from + n;
    float add = sh.add[k];
    for (int j = 0; mine && j <= K; ++j)
      if (j != k && sh.index[j] == at) {  // the token is in the list too: once, with both terms
        mine = j > k;
        add += sh.add[j];
      }
    if (mine) logit_put(d, at, fmaf(add, inv_t, row_map<G>(dense, logit_at<T>(x, at))));
  }
}

int sm_count_here() {
  int dev = 0;
  cudaGetDevice(&dev);
  return sm_count(dev);
}

template <typename T, int G>
int launch_forward(const TokenLogprobsArgs& a, int cluster, cudaStream_t stream) {
  const int64_t rows = a.outer * a.inner;
  ForwardPlan plan;
  plan.cluster = cluster;
  // vectors that a thread reads of its slice
  const int64_t mine = std::max<int64_t>(1, ((a.V / kVec<T> + cluster - 1) / cluster + G - 1) / G);
  const int64_t batches = (mine + kUnroll - 1) / kUnroll;
  plan.cell_shift = 0;
  if (G != 32 || 32 * batches >= 4 * a.K)
    for (plan.cell_shift = 2; (batches * kUnroll) >> plan.cell_shift > kMaxCells;) ++plan.cell_shift;
  static_assert(kUnroll == 4, "a cell is some batches");
  plan.cells = static_cast<int>((mine + (int64_t(1) << plan.cell_shift) - 1) >> plan.cell_shift);
  constexpr int kGroups = cta_threads<G> / G;
  const size_t smem = kGroups * group_smem<T, G>(static_cast<int>(a.K), plan.cells, cluster);
  auto* kern = a.K > 0 ? token_logprobs_kernel<T, G, true> : token_logprobs_kernel<T, G, false>;
  if (int rc = allow_shared_memory("token_logprobs shared memory", reinterpret_cast<const void*>(kern), smem))
    return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(G == 32 ? (rows + kGroups - 1) / kGroups : rows * cluster));
  cfg.blockDim = dim3(cta_threads<G>);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 1 : 0;
  return cuda_status("token_logprobs launch",
                     cudaLaunchKernelEx(&cfg, kern, a, plan, FastDiv(static_cast<uint32_t>(a.inner))));
}

template <typename T, int L, int E>
int launch_short(const TokenLogprobsArgs& a, const FastDiv& inner, cudaStream_t stream) {
  const int64_t rows = a.outer * a.inner;
  const bool lanes = L < 32 && a.K > 0 && a.K <= kWarpTop && 16 * a.K <= a.V &&
                     rows >= kLanesRows * sm_count_here();
  const int per = a.K == 0 || lanes ? kThreads / L : kWarps;
  const unsigned grid = static_cast<unsigned>((rows + per - 1) / per);
  if (a.K == 0) token_logprobs_short_kernel<T, L, E><<<grid, kThreads, 0, stream>>>(a, inner);
  else if (lanes) token_list_lanes_kernel<T, L < 32 ? L : 16, E><<<grid, kThreads, 0, stream>>>(a, inner);
  else token_list_short_kernel<T, L * E / 32><<<grid, kThreads, 0, stream>>>(a, inner);
  return cuda_status("token_logprobs launch");
}

template <typename T>
int forward_by_size(const TokenLogprobsArgs& a, cudaStream_t stream) {
  const int64_t rows = a.outer * a.inner, bytes = a.V * static_cast<int64_t>(sizeof(T));
  const FastDiv inner(static_cast<uint32_t>(a.inner));
  if (a.V <= 256) return launch_short<T, 8, 32>(a, inner, stream);
  if (a.V <= 512) return launch_short<T, 16, 32>(a, inner, stream);
  if (a.V <= kShort) return launch_short<T, 32, 32>(a, inner, stream);
  // Many rows of a middling length: a warp each.
  if (bytes <= kWarpRowBytes && a.K <= kWarpList && rows >= kWarpRows * sm_count_here())
    return launch_forward<T, 32>(a, 1, stream);
  // Few rows: split each in two while that leaves at most three CTAs for every SM. 296 rows of 131072 in
  // bf16: 13.4 us whole, 14.2 in two; 200: 13.3 whole, 11.5 in two; 64: 8.6 whole, 6.6 in four, 7.0 in eight.
  int cluster = 1;
  if (bytes > kUnsplitBytes)
    while (cluster < kMaxCluster && 2 * rows * cluster <= 3 * sm_count_here() &&
           bytes >= 2 * cluster * kSliceBytes)
      cluster *= 2;
  if (cluster == 1 && bytes <= kHalfBytes && a.K <= kWarpList)
    return launch_forward<T, kThreads / 2>(a, 1, stream);
  return launch_forward<T, kThreads>(a, cluster, stream);
}

template <typename T, int G>
int launch_backward(const TokenLogprobsBwdArgs& a, int64_t pieces, int piece, cudaStream_t stream) {
  constexpr int kGroups = kThreads / G;
  const int64_t grid = (a.f.outer * a.f.inner * pieces + kGroups - 1) / kGroups;
  if (grid * kGroups >= int64_t(1) << 31) {
    set_error("token_logprobs_bwd: too many rows for this vocabulary");
    return BDH_ERR_INVALID;
  }
  const size_t lists = a.g_top != nullptr && a.f.K > 0 ? kGroups * sizeof(GradShared) : 0;
  token_logprobs_bwd_kernel<T, G><<<static_cast<unsigned>(grid), kThreads, lists, stream>>>(
      a, FastDiv(static_cast<uint32_t>(pieces)), piece, FastDiv(static_cast<uint32_t>(a.f.inner)));
  return cuda_status("token_logprobs_bwd launch");
}

template <typename T>
int backward_by_size(const TokenLogprobsBwdArgs& a, cudaStream_t stream) {
  const int64_t rows = a.f.outer * a.f.inner, V = a.f.V, bytes = V * static_cast<int64_t>(sizeof(T));
  if (V <= 256) return launch_backward<T, 8>(a, 1, 256, stream);
  if (V <= 512) return launch_backward<T, 16>(a, 1, 512, stream);
  if (V <= kShort) return launch_backward<T, 32>(a, 1, kShort, stream);
  if (bytes <= kWarpGradBytes && rows >= kWarpRows * sm_count_here())
    return launch_backward<T, 32>(a, 1, static_cast<int>(V), stream);
  return launch_backward<T, kThreads>(a, (V + kPiece - 1) / kPiece, kPiece, stream);
}

}  // namespace

int launch_token_logprobs(const TokenLogprobsArgs& a, cudaStream_t stream) {
  if (a.outer * a.inner == 0) return BDH_OK;
  return a.dtype == BDH_DTYPE_F32 ? forward_by_size<float>(a, stream)
                                  : forward_by_size<uint16_t>(a, stream);
}

int launch_token_logprobs_bwd(const TokenLogprobsBwdArgs& a, cudaStream_t stream) {
  if (a.f.outer * a.f.inner == 0) return BDH_OK;
  return a.f.dtype == BDH_DTYPE_F32 ? backward_by_size<float>(a, stream)
                                    : backward_by_size<uint16_t>(a, stream);
}

}  // namespace bdh
