// Routing to experts and back: the router's choice and its gradient, the slots in the order of their experts, and the
// weighted sum of the experts' rows with its gradients. All of it is bound by the bytes it reads and writes or, for a
// few tokens, by latency; scores and sums are float32.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cooperative_groups.h>

#include "common.cuh"

namespace cg = cooperative_groups;
using namespace mxq;

namespace {

constexpr unsigned kAll = 0xffffffffu;
constexpr int kMostExperts = 1024, kMostChosen = 32;
constexpr float kEps = 1e-20f;

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v = __fadd_rn(v, __shfl_xor_sync(kAll, v, d));
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v = fmaxf(v, __shfl_xor_sync(kAll, v, d));
  return v;
}

// An order-preserving key of a choice value; 0 (below every other) for -Inf and NaN, which are never chosen, and where
// `live` is false; -0 as +0.
__device__ __forceinline__ uint32_t key_of(float f) {
  const uint32_t b = __float_as_uint(__fadd_rn(f, 0.0f));
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ uint32_t key_if(bool live, float f) { return live && f > -INFINITY ? key_of(f) : 0u; }
constexpr float kLowest = -3.402823466e38f;
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}
// the key of a group's two largest, whose sum may pass the type's lowest value: that is still a group to choose
__device__ __forceinline__ uint32_t key_of_pair(uint32_t best, uint32_t second) {
  return key_if(true, fmaxf(__fadd_rn(value_of(best), value_of(second)), kLowest));
}
__device__ __forceinline__ float sigmoid(float x) { return __frcp_rn(__fadd_rn(1.0f, expf(-x))); }
__device__ __forceinline__ bool is_nan(float x) { return x != x; }

struct RouteArgs {
  int64_t stride;
  int T, E, k, sigmoid, groups, keep, top2, renormalize;
  int vec, vec_bias;           // every lane's values are whole 16-byte pieces of the row (the biases), and there
  float scale;
};

// V neighbouring values of a row: 16-byte loads where the row allows them
template <typename IN, int V>
__device__ __forceinline__ void load_row(const IN* row, int e0, int E, bool vec, float (&l)[V]) {
  constexpr int N = 16 / sizeof(IN);
  if (V >= N && vec) {
#pragma unroll
    for (int i = 0; i < V / N; i++) {
      const uint4 q = __ldg(reinterpret_cast<const uint4*>(row + e0) + i);
      const IN* p = reinterpret_cast<const IN*>(&q);
#pragma unroll
      for (int j = 0; j < N; j++) l[(V >= N ? i * N + j : 0)] = to_float<IN>(p[j]);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < V; i++) l[i] = e0 + i < E ? to_float<IN>(row[e0 + i]) : -INFINITY;
}

// Two largest of two pairs
__device__ __forceinline__ void merge2(uint32_t& a, uint32_t& b, uint32_t c, uint32_t d) {
  b = max(min(a, c), max(b, d));
  a = max(a, c);
}

// A warp per token, V neighbouring experts per lane (lane V on), so that the lowest lane holds the lowest experts and a
// tie is the first lane of a ballot. The k largest are taken one after the other: the lanes' best by one warp
// reduction, and only the lane that had it finds which of its own it was. The chosen scores are made again from the
// logits at the end, by lane j for the j-th. Groups whose runs are whole lanes, a power of two of them (every usual
// shape), are ranked by shuffles, all at once; others one by one.
//
// A group's two largest are summed as scores, with a bias or without one (logits order the experts as their scores do, but not
// sums of two), and a masked expert counts there with the score 0 that its logit of -Inf has: taking an expert out cannot
// raise its group. A group with nobody left to choose is not kept.
//
// Bound by issue (about 1000 instructions a token): 8192 tokens of 256 experts (float32, bias, 8 groups, k = 8) take
// 12.6 us (11.9 without a bias), their 9.4 MB 1.4 us at the copy's rate; 16 tokens of 128 experts 3.7 us.
template <typename IN, int V>
__global__ void __launch_bounds__(128) k_route(const IN* __restrict__ logits, const float* __restrict__ bias,
                                               float* __restrict__ weights, int* __restrict__ experts, RouteArgs a) {
  const int lane = threadIdx.x & 31, e0 = lane * V;
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (t >= a.T) return;
  float l[V];
  load_row<IN, V>(logits + t * a.stride, e0, a.E, a.vec, l);
  bool bad = false;
  float top = -INFINITY, sum = 1.0f;
#pragma unroll
  for (int i = 0; i < V; i++) {
    bad |= is_nan(l[i]);
    top = fmaxf(top, l[i]);
  }
  bad = __any_sync(kAll, bad);
  uint32_t key[V], rank[V];                            // what orders the experts; the groups
  auto by_score = [&](int i, float s, float b) {
    const float v = __fadd_rn(s, b);
    rank[i] = key_of(fmaxf(v, kLowest));
    key[i] = !bias ? key_if(true, l[i]) : l[i] > -INFINITY && v > -INFINITY ? rank[i] : 0u;
  };
  if (!a.sigmoid) {
    top = warp_max(top);
    bad |= top == INFINITY;                            // Inf / Inf: no scores
    sum = 0.0f;
    float s[V];
#pragma unroll
    for (int i = 0; i < V; i++) {
      s[i] = l[i] > -INFINITY ? expf(__fsub_rn(l[i], top)) : 0.0f;
      sum = __fadd_rn(sum, s[i]);
    }
    sum = warp_sum(sum);
    if (bias) {
      float b[V];
      load_row<float, V>(bias, e0, a.E, a.vec_bias, b);
#pragma unroll
      for (int i = 0; i < V; i++) by_score(i, __fdiv_rn(s[i], sum), b[i]);
    } else if (a.top2) {
#pragma unroll
      for (int i = 0; i < V; i++) by_score(i, __fdiv_rn(s[i], sum), 0.0f);
    }
  } else if (bias) {
    float b[V];
    load_row<float, V>(bias, e0, a.E, a.vec_bias, b);
#pragma unroll
    for (int i = 0; i < V; i++) by_score(i, sigmoid(l[i]), b[i]);
  } else if (a.top2) {
#pragma unroll
    for (int i = 0; i < V; i++) by_score(i, sigmoid(l[i]), 0.0f);
  }
  if (!bias && !a.top2) {
#pragma unroll
    for (int i = 0; i < V; i++) key[i] = key_if(true, l[i]);
  }
  if (!a.top2) {
#pragma unroll
    for (int i = 0; i < V; i++) rank[i] = key[i];
  }
  if (a.groups > 1) {
    const int run = a.E / a.groups, width = run / V;
    if (run % V == 0 && (width & (width - 1)) == 0) {
      uint32_t best = 0u, second = 0u, any = 0u;
#pragma unroll
      for (int i = 0; i < V; i++) {
        merge2(best, second, rank[i], 0u);
        any |= key[i];
      }
      for (int d = 1; d < width; d <<= 1)
        merge2(best, second, __shfl_xor_sync(kAll, best, d), __shfl_xor_sync(kAll, second, d));
      const int g = lane / width;
      if (a.top2) {
        if (second) best = key_of_pair(best, second);
        const unsigned alive = __ballot_sync(kAll, any != 0u);
        if (!(alive >> (g * width & 31) & (0xffffffffu >> (32 - width)))) best = 0u;
      }
      int ahead = 0;                                   // groups that come before this lane's
      for (int o = 0; o < a.groups; o++) {
        const uint32_t v = __shfl_sync(kAll, best, o * width);
        ahead += v > best || (v == best && o < g);
      }
      if (ahead >= a.keep) {
#pragma unroll
        for (int i = 0; i < V; i++) key[i] = 0u;
      }
    } else {
      uint32_t mine = 0u;                              // lane g: the key of group g's value
      for (int g = 0; g < a.groups; g++) {
        uint32_t best = 0u, second = 0u, any = 0u;
#pragma unroll
        for (int i = 0; i < V; i++) {
          const bool in = e0 + i >= g * run && e0 + i < (g + 1) * run;
          merge2(best, second, in ? rank[i] : 0u, 0u);
          any |= in ? key[i] : 0u;
        }
        for (int d = 1; d < 32; d <<= 1)
          merge2(best, second, __shfl_xor_sync(kAll, best, d), __shfl_xor_sync(kAll, second, d));
        if (a.top2 && second) best = key_of_pair(best, second);
        if (lane == g) mine = best;
        if (!__any_sync(kAll, any != 0u) && lane == g) mine = 0u;
      }
      unsigned kept = 0u;
      for (int j = 0; j < a.keep; j++) {
        const uint32_t m = __reduce_max_sync(kAll, mine);
        if (!m) break;
        const int g = __ffs(__ballot_sync(kAll, mine == m)) - 1;
        kept |= 1u << g;
        if (lane == g) mine = 0u;
      }
#pragma unroll
      for (int i = 0; i < V; i++)
        if (e0 + i < a.E && !(kept >> ((e0 + i) / run) & 1u)) key[i] = 0u;
    }
  }
  auto largest = [&] {
    uint32_t m = key[0];
#pragma unroll
    for (int i = 1; i < V; i++) m = max(m, key[i]);
    return m;
  };
  uint32_t best = largest();
  int chosen = -1;                                     // lane j: the j-th choice
  for (int j = 0; j < a.k; j++) {
    const uint32_t m = __reduce_max_sync(kAll, best);
    if (!m) break;
    const int win = __ffs(__ballot_sync(kAll, best == m)) - 1;
    int e = 0;
    if (lane == win) {                                 // its first value that is m goes
      bool found = false;
#pragma unroll
      for (int i = 0; i < V; i++) {
        const bool here = key[i] == m && !found;
        found |= here;
        if (here) {
          e = e0 + i;
          key[i] = 0u;
        }
      }
      best = largest();
    }
    e = __shfl_sync(kAll, e, win);
    if (lane == j) chosen = e;
  }
  float w = 0.0f;
  if (chosen >= 0) {
    const float x = to_float<IN>(logits[t * a.stride + chosen]);
    w = a.sigmoid ? sigmoid(x) : __fdiv_rn(expf(__fsub_rn(x, top)), sum);
  }
  if (a.renormalize) w = __fdiv_rn(w, __fadd_rn(warp_sum(w), kEps));
  w = bad ? __uint_as_float(0x7fc00000u) : __fmul_rn(w, a.scale);
  if (lane < a.k) {
    weights[t * a.k + lane] = w;
    experts[t * a.k + lane] = chosen;
  }
}

// A warp per token. Lane j holds choice j: g = grad scale, ds = (g - sum g s / S) / S when renormalized; softmax:
// dl = p (ds - sum ds p), ds 0 where not chosen; sigmoid: dl = ds s (1 - s) at the chosen. The probabilities are made
// again from the logits: reading k floats and E logits a token, writing E. 8191 tokens of 64 experts (bf16): 4.2 us,
// two of them the launch.
template <typename IN, int V>
__global__ void __launch_bounds__(128) k_route_backward(const float* __restrict__ grad, const IN* __restrict__ logits,
                                                        const int* __restrict__ experts, IN* __restrict__ out, RouteArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (t >= a.T) return;
  const int e = lane < a.k ? experts[t * a.k + lane] : -1;
  const bool live = e >= 0 && e < a.E;
  const float le = live ? to_float<IN>(logits[t * a.stride + e]) : 0.0f;
  float l[V], top = -INFINITY, sum = 0.0f;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < V; i++) {
    const int x = i * 32 + lane;
    l[i] = x < a.E ? to_float<IN>(logits[t * a.stride + x]) : -INFINITY;
    bad |= is_nan(l[i]);
    top = fmaxf(top, l[i]);
  }
  bad = __any_sync(kAll, bad);
  float s;
  if (a.sigmoid) {
    s = live ? sigmoid(le) : 0.0f;
  } else {
    top = warp_max(top);
    bad |= top == INFINITY;
#pragma unroll
    for (int i = 0; i < V; i++) {
      l[i] = l[i] == -INFINITY ? 0.0f : expf(__fsub_rn(l[i], top));
      sum = __fadd_rn(sum, l[i]);
    }
    sum = warp_sum(sum);
    s = live ? __fdiv_rn(expf(__fsub_rn(le, top)), sum) : 0.0f;
  }
  float ds = live ? __fmul_rn(grad[t * a.k + lane], a.scale) : 0.0f;
  if (a.renormalize) {
    const float total = __fadd_rn(warp_sum(s), kEps), dot = warp_sum(__fmul_rn(ds, s));
    ds = live ? __fdiv_rn(__fsub_rn(ds, __fdiv_rn(dot, total)), total) : 0.0f;
  }
  const float nan = __uint_as_float(0x7fc00000u);
  IN* row = out + t * a.E;
  float d;
  if (a.sigmoid) {
    d = __fmul_rn(__fmul_rn(ds, s), __fsub_rn(1.0f, s));
#pragma unroll
    for (int i = 0; i < V; i++) {
      const int x = i * 32 + lane;
      if (x < a.E) row[x] = from_float<IN>(bad ? nan : 0.0f);
    }
  } else {
    const float dot = warp_sum(__fmul_rn(ds, s));
    d = __fmul_rn(s, __fsub_rn(ds, dot));
    const float f = sum > 0.0f ? __fdiv_rn(-dot, sum) : 0.0f;
#pragma unroll
    for (int i = 0; i < V; i++) {
      const int x = i * 32 + lane;
      if (x < a.E) row[x] = from_float<IN>(bad ? nan : __fmul_rn(l[i], f));
    }
  }
  __syncwarp();                                        // the chosen experts' values over the others
  if (live && !bad) row[e] = from_float<IN>(d);
}

// ----------------------------------------------------------------------------------------------- dispatch
// A stable counting sort. The slots are cut into a contiguous run per warp; each warp counts its run by expert in
// shared memory, the counts are added up over the warps, the CTAs and the experts, and each warp then walks its run
// again, 32 slots at a time in order, giving each slot the next place of its expert.
//
// The CTAs' counts meet in one of two ways. Up to kOneLaunch slots one cluster does it all and reads them through
// distributed shared memory: one launch, no workspace (128 slots of 128 experts 4.7 us; 65536 slots of 256 experts
// 12.7, against 15.3 in two launches). More slots go over the whole GPU, with a first launch that writes each CTA's
// counts to the workspace: on eight SMs the scattered stores of `order` take the time (131072 slots: 23.5 us in one
// cluster, 18.6 in two launches; 524288: 89 and 21).
constexpr int kDispatchWarps = 16;
constexpr int64_t kOneLaunch = 98304;

// slots per warp's run: whole groups of 32
__host__ __device__ __forceinline__ int64_t run_of(int64_t S, int64_t ctas) {
  const int64_t runs = ctas * kDispatchWarps;
  return ((S + runs - 1) / runs + 31) / 32 * 32;
}

__global__ void __launch_bounds__(kDispatchWarps * 32) k_dispatch_count(const int* __restrict__ ids, int64_t S, int E,
                                                                        int* __restrict__ counts) {
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  extern __shared__ int sm[];
  for (int i = threadIdx.x; i < E; i += blockDim.x) sm[i] = 0;
  __syncthreads();
  const int64_t chunk = run_of(S, gridDim.x) * kDispatchWarps;
  const int64_t begin = min(S, blockIdx.x * chunk), end = min(S, begin + chunk);
#pragma unroll 4
  for (int64_t i = begin + threadIdx.x; i < end; i += blockDim.x) {
    const int e = ids[i];
    if (e >= 0 && e < E) atomicAdd(sm + e, 1);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < E; i += blockDim.x) counts[blockIdx.x * (int64_t)E + i] = sm[i];
}

// GRID: the grid's CTAs, their counts in `counts`; else one cluster
template <bool GRID>
__global__ void __launch_bounds__(kDispatchWarps * 32) k_dispatch(const int* __restrict__ ids, int64_t S, int E,
                                                                  const int* __restrict__ counts, int* __restrict__ offsets,
                                                                  int* __restrict__ order, int* __restrict__ where) {
  extern __shared__ int sm[];
  int* count = sm;                                     // [warp][E]: counts, then the next place of each expert
  int* total = sm + kDispatchWarps * E;                // [E] this CTA's
  int* start = total + E;                              // [E] the first place of this CTA's
  int* sums = start + E;                               // [32] of the scan over experts
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = GRID ? (int)gridDim.x : (int)cluster.num_blocks(), rank = GRID ? (int)blockIdx.x : (int)cluster.block_rank();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < kDispatchWarps * E; i += blockDim.x) count[i] = 0;
  __syncthreads();
  const int64_t run = run_of(S, ctas);
  const int64_t begin = min(S, (rank * (int64_t)kDispatchWarps + warp) * run), end = min(S, begin + run);
  if (GRID) asm volatile("griddepcontrol.wait;\n" ::: "memory");
  int* mine = count + warp * E;
  // the run's first 512 slots stay in registers for the second walk
  constexpr int kHeld = 16;
  int held[kHeld];
#pragma unroll
  for (int h = 0; h < kHeld; h++) held[h] = begin + h * 32 + lane < end ? ids[begin + h * 32 + lane] : -1;
#pragma unroll
  for (int h = 0; h < kHeld; h++)
    if (held[h] >= 0 && held[h] < E) atomicAdd(mine + held[h], 1);
#pragma unroll 4
  for (int64_t i = begin + kHeld * 32 + lane; i < end; i += 32) {
    const int e = ids[i];
    if (e >= 0 && e < E) atomicAdd(mine + e, 1);
  }
  __syncthreads();
  // two experts per thread (E <= 1024), kStep apart so that neighbouring threads read neighbouring counts
  constexpr int kPer = kMostExperts / (kDispatchWarps * 32), kStep = kDispatchWarps * 32;
#pragma unroll
  for (int p = 0; p < kPer; p++) {
    const int e = p * kStep + threadIdx.x;
    if (e >= E) continue;
    int own = 0;
#pragma unroll
    for (int w = 0; w < kDispatchWarps; w++) {
      const int c = count[w * E + e];
      count[w * E + e] = own;
      own += c;
    }
    total[e] = own;
  }
  if (!GRID) cluster.sync();
  int live = 0;
#pragma unroll
  for (int p = 0; p < kPer; p++) {                     // the experts in order: kStep of them, then the next kStep
    const int e = p * kStep + threadIdx.x;
    int all = 0, before = 0;
    if (e < E) {
      if (GRID) {
        for (int c0 = 0; c0 < ctas; c0 += 32) {        // 32 loads under way
          int v[32];
#pragma unroll
          for (int c = 0; c < 32; c++) v[c] = c0 + c < ctas ? __ldg(counts + (c0 + c) * (int64_t)E + e) : 0;
#pragma unroll
          for (int c = 0; c < 32; c++) {
            before += c0 + c < rank ? v[c] : 0;
            all += v[c];
          }
        }
      } else {
        for (int c = 0; c < ctas; c++) {
          const int v = cluster.map_shared_rank(total, c)[e];
          if (c < rank) before += v;
          all += v;
        }
      }
    }
    int scan = all;                                    // over the threads: lanes, then the warps' sums
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(kAll, scan, d);
      if (lane >= d) scan += up;
    }
    __syncthreads();
    if (lane == 31) sums[warp] = scan;
    __syncthreads();
    int head = live;
#pragma unroll
    for (int w = 0; w < kDispatchWarps; w++) {
      const int v = sums[w];
      if (w < warp) head += v;
      live += v;
    }
    if (e < E) {
      if (rank == 0) offsets[e] = head + scan - all;
      start[e] = head + scan - all + before;
    }
  }
  if (rank == 0 && threadIdx.x == 0) offsets[E] = live;
  for (int64_t i = live + rank * (int64_t)blockDim.x + threadIdx.x; i < S; i += (int64_t)ctas * blockDim.x)
    order[i] = -1;
  __syncthreads();
  const int bits = 32 - __clz(E - 1);                  // 0 for one expert
  auto place32 = [&](int64_t i, int x) {
    if (x < 0 || x >= E) x = -1;
    // the lanes with this lane's expert: a ballot per bit (a match instruction takes longer)
    unsigned same = __ballot_sync(kAll, x >= 0);
    for (int bit = 0; bit < bits; bit++) {
      const bool mine_set = x >> bit & 1;
      const unsigned set = __ballot_sync(kAll, mine_set);
      same &= mine_set ? set : ~set;
    }
    const int place = x >= 0 ? start[x] + mine[x] + __popc(same & ((1u << lane) - 1u)) : -1;
    __syncwarp();
    if (x >= 0 && lane == __ffs(same) - 1) mine[x] += __popc(same);
    __syncwarp();
    if (i < end) {
      where[i] = place;
      if (place >= 0) order[place] = (int)i;
    }
  };
#pragma unroll
  for (int h = 0; h < kHeld; h++)
    if (begin + h * 32 < end) place32(begin + h * 32 + lane, held[h]);
  for (int64_t b = begin + kHeld * 32; b < end; b += 32) place32(b + lane, b + lane < end ? ids[b + lane] : -1);
  if (!GRID) cluster.sync();                           // the totals are read before their CTA leaves
}

// ------------------------------------------------------------------------------------------------ combine
template <typename T>
struct Vec {                                           // 16 bytes of T
  static constexpr int N = 16 / sizeof(T);
  uint4 raw;
  __device__ __forceinline__ void get(float (&v)[N]) const {
    const T* p = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = to_float<T>(p[i]);
  }
  __device__ __forceinline__ void set(const float (&v)[N]) {
    T* p = reinterpret_cast<T*>(&raw);
#pragma unroll
    for (int i = 0; i < N; i++) p[i] = from_float<T>(v[i]);
  }
};
// N values at column c of a row: one 16-byte access, or (VEC false) those within the row one by one
template <typename T, bool VEC>
__device__ __forceinline__ Vec<T> load_vec(const T* row, int64_t c, int64_t n) {
  Vec<T> v;
  if (VEC) {
    v.raw = __ldg(reinterpret_cast<const uint4*>(row + c));
  } else {
    T* p = reinterpret_cast<T*>(&v.raw);
#pragma unroll
    for (int i = 0; i < Vec<T>::N; i++) p[i] = c + i < n ? row[c + i] : from_float<T>(0.0f);
  }
  return v;
}
template <typename T, bool VEC>
__device__ __forceinline__ void store_vec(T* row, int64_t c, int64_t n, const Vec<T>& v) {
  if (VEC) {
    *reinterpret_cast<uint4*>(row + c) = v.raw;
  } else {
    const T* p = reinterpret_cast<const T*>(&v.raw);
#pragma unroll
    for (int i = 0; i < Vec<T>::N; i++)
      if (c + i < n) row[c + i] = p[i];
  }
}

// A CTA per token and stretch of columns, 16 bytes of y per thread; four of the experts' rows are on their way at
// once. Bound by the bytes: 4096 tokens, k = 8, 4096 columns (bf16) 47 us, 6.4 TB/s; 24 tokens of 2048 columns 2.6
// us, a launch.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) k_combine(const T* __restrict__ z, const float* __restrict__ weights,
                                                 const int* __restrict__ where, const T* __restrict__ residual,
                                                 int64_t residual_stride, T* __restrict__ y, int k, int64_t n, int64_t rows) {
  constexpr int N = Vec<T>::N;
  const int64_t t = blockIdx.x, c = ((int64_t)blockIdx.y * blockDim.x + threadIdx.x) * N;
  if (c >= n) return;
  float acc[N], v[N];
#pragma unroll
  for (int i = 0; i < N; i++) acc[i] = 0.0f;
  for (int j0 = 0; j0 < k; j0 += 4) {
    Vec<T> r[4];
    float w[4];
    int at[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      at[j] = -1;
      w[j] = 0.0f;
      if (j0 + j < k) {
        at[j] = where[t * k + j0 + j];
        w[j] = weights[t * k + j0 + j];
      }
      if (at[j] >= 0 && at[j] < rows) r[j] = load_vec<T, VEC>(z + at[j] * n, c, n);
      else r[j].raw = make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int j = 0; j < 4; j++) {
      if (j0 + j >= k) break;
      r[j].get(v);
#pragma unroll
      for (int i = 0; i < N; i++) acc[i] = __fmaf_rn(w[j], v[i], acc[i]);
    }
  }
  if (residual) {
    load_vec<T, VEC>(residual + t * residual_stride, c, n).get(v);
#pragma unroll
    for (int i = 0; i < N; i++) acc[i] = __fadd_rn(acc[i], v[i]);
  }
  Vec<T> o;
  o.set(acc);
  store_vec<T, VEC>(y + t * n, c, n, o);
}

// A CTA per token. J experts' rows (all of them up to 8) at a time: dy's piece is read once for them, their pieces of
// z are on their way together, and a thread's share of the dot products stays in registers and is added up over the
// CTA in a fixed order. Bound by the bytes: 4096 tokens, k = 6, 2048 columns (bf16) 36.7 us, 6.0 TB/s (49 us with two
// CTAs per SM; 65 with the tail's look at `order` one load after the other).
template <typename T, bool VEC, int J>
__global__ void __launch_bounds__(256, 3) k_combine_backward(const T* __restrict__ dy, int64_t dy_stride, const T* __restrict__ z,
                                                          const float* __restrict__ weights, const int* __restrict__ where,
                                                          const int* __restrict__ order, T* __restrict__ dz,
                                                          float* __restrict__ dw, int k, int64_t n, int rows) {
  constexpr int N = Vec<T>::N;
  __shared__ float part[8][J];
  const int64_t t = blockIdx.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  bool hole = false;                                   // a place without a slot among this CTA's k
  for (int j = threadIdx.x; j < k; j += blockDim.x) hole |= order[t * k + j] < 0;
  for (int j0 = 0; j0 < k; j0 += J) {
    int at[J];
    float w[J], dot[J];
#pragma unroll
    for (int j = 0; j < J; j++) {
      const bool in = j0 + j < k;
      at[j] = in ? __ldg(where + t * k + j0 + j) : -1;
      if (at[j] >= rows) at[j] = -1;
      w[j] = in ? __ldg(weights + t * k + j0 + j) : 0.0f;
      dot[j] = 0.0f;
    }
    for (int64_t c = threadIdx.x * N; c < n; c += blockDim.x * N) {
      float g[N], v[N], o[N];
      const Vec<T> mine = load_vec<T, VEC>(dy + t * dy_stride, c, n);
      Vec<T> r[J];
#pragma unroll
      for (int j = 0; j < J; j++) {
        r[j].raw = make_uint4(0, 0, 0, 0);
        if (at[j] >= 0) r[j] = load_vec<T, VEC>(z + at[j] * n, c, n);
      }
      mine.get(g);
#pragma unroll
      for (int j = 0; j < J; j++) {
        r[j].get(v);
#pragma unroll
        for (int i = 0; i < N; i++) {
          if (at[j] >= 0) dot[j] = __fmaf_rn(g[i], v[i], dot[j]);
          o[i] = __fmul_rn(w[j], g[i]);
        }
        Vec<T> q;
        q.set(o);
        if (at[j] >= 0) store_vec<T, VEC>(dz + at[j] * n, c, n, q);
      }
    }
#pragma unroll
    for (int j = 0; j < J; j++) {
      const float d = warp_sum(dot[j]);
      if (lane == 0) part[warp][j] = d;
    }
    __syncthreads();
    if (threadIdx.x < J && j0 + threadIdx.x < k) {
      float d = 0.0f;
      for (int i = 0; i < warps; i++) d = __fadd_rn(d, part[i][threadIdx.x]);
      dw[t * k + j0 + threadIdx.x] = d;
    }
    if (j0 + J < k) __syncthreads();
  }
  if (!__syncthreads_or(hole)) return;
  for (int j = 0; j < k; j++) {                        // the rows that no slot has
    if (order[t * k + j] >= 0) continue;
    Vec<T> zero;
    zero.raw = make_uint4(0, 0, 0, 0);
    for (int64_t c = threadIdx.x * N; c < n; c += blockDim.x * N) store_vec<T, VEC>(dz + (t * k + j) * n, c, n, zero);
  }
}

// --------------------------------------------------------------------------------------------------- host
bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

int check_route(const char* who, int64_t T, int64_t E, int64_t k, const mxq_route_spec* s, RouteArgs& a) {
  MXQ_REQUIRE(s != nullptr, MXQ_ERR_VALUE, "%s: no spec", who);
  MXQ_REQUIRE(T >= 0 && T < (1ll << 30) && E >= 1 && E <= kMostExperts, MXQ_ERR_VALUE, "%s: %lld tokens, %lld experts (at most %d)",
              who, (long long)T, (long long)E, kMostExperts);
  MXQ_REQUIRE(k >= 1 && k <= E && k <= kMostChosen, MXQ_ERR_VALUE, "%s: k must be in [1, min(experts, %d)], got %lld", who, kMostChosen,
              (long long)k);
  MXQ_REQUIRE(s->score == MXQ_SCORE_SOFTMAX || s->score == MXQ_SCORE_SIGMOID, MXQ_ERR_VALUE, "%s: score %d", who, s->score);
  MXQ_REQUIRE(s->groups >= 1 && s->groups <= 32 && E % s->groups == 0 && s->keep >= 1 && s->keep <= s->groups, MXQ_ERR_VALUE,
              "%s: %d of %d groups of %lld experts", who, s->keep, s->groups, (long long)E);
  a.T = (int)T;
  a.E = (int)E;
  a.k = (int)k;
  a.sigmoid = s->score == MXQ_SCORE_SIGMOID;
  a.groups = s->groups;
  a.keep = s->keep;
  a.top2 = s->top2 && s->groups > 1;
  a.renormalize = s->renormalize;
  a.scale = s->scale;
  return MXQ_OK;
}

template <typename F>
int by_type(const char* who, int32_t type, F f) {
  switch (type) {
    case MXQ_OUT_F32: return f(float{});
    case MXQ_OUT_BF16: return f(__nv_bfloat16{});
    case MXQ_OUT_F16: return f(__half{});
    default: return set_error(MXQ_ERR_VALUE, "%s: type %d", who, type);
  }
}
template <typename IN>
int row_vec(const void* logits, int64_t stride, int E, int v) {
  constexpr int N = 16 / sizeof(IN);
  return v % N == 0 && E == 32 * v && stride % N == 0 && aligned16(logits);
}
template <int N>
struct Int { static constexpr int value = N; };
template <typename F>
void by_width(int E, F f) {
  if (E <= 32) f(Int<1>{});
  else if (E <= 64) f(Int<2>{});
  else if (E <= 128) f(Int<4>{});
  else if (E <= 256) f(Int<8>{});
  else if (E <= 512) f(Int<16>{});
  else f(Int<32>{});
}

}  // namespace

extern "C" int mxq_route(const void* logits, int32_t type, int64_t stride, const float* bias, float* weights, int32_t* experts,
                         int64_t T, int64_t E, int64_t k, const mxq_route_spec* spec, void* stream) {
  RouteArgs a;
  if (int rc = check_route("route", T, E, k, spec, a)) return rc;
  a.stride = stride;
  if (T == 0) return MXQ_OK;
  return by_type("route", type, [&](auto zero) {
    using IN = decltype(zero);
    by_width(a.E, [&](auto v) {
      a.vec = row_vec<IN>(logits, stride, a.E, decltype(v)::value);
      a.vec_bias = row_vec<float>(bias, 0, a.E, decltype(v)::value);
      k_route<IN, decltype(v)::value><<<(unsigned)((T + 3) / 4), 128, 0, as_stream(stream)>>>(static_cast<const IN*>(logits), bias, weights,
                                                                                          experts, a);
    });
    return MXQ_LAUNCH_CHECK("route");
  });
}

extern "C" int mxq_route_backward(const float* grad, const void* logits, int32_t type, int64_t stride, const int32_t* experts,
                                  void* grad_logits, int64_t T, int64_t E, int64_t k, const mxq_route_spec* spec, void* stream) {
  RouteArgs a;
  if (int rc = check_route("route_backward", T, E, k, spec, a)) return rc;
  a.stride = stride;
  if (T == 0) return MXQ_OK;
  return by_type("route_backward", type, [&](auto zero) {
    using IN = decltype(zero);
    by_width(a.E, [&](auto v) {
      k_route_backward<IN, decltype(v)::value><<<(unsigned)((T + 3) / 4), 128, 0, as_stream(stream)>>>(
          grad, static_cast<const IN*>(logits), experts, static_cast<IN*>(grad_logits), a);
    });
    return MXQ_LAUNCH_CHECK("route_backward");
  });
}

static int dispatch_ctas(int64_t slots) {              // of the two-launch form: 512 slots each at least
  const int64_t want = slots / 512;
  return (int)(want < sm_count() ? want : sm_count());
}

extern "C" int64_t mxq_dispatch_workspace(int64_t slots, int64_t experts) {
  if (slots < 0 || experts < 1) return -1;
  return slots > kOneLaunch ? (int64_t)dispatch_ctas(slots) * experts * 4 : 0;
}

extern "C" int mxq_dispatch(const int32_t* experts_of, int64_t slots, int64_t experts, int32_t* offsets, int32_t* order,
                            int32_t* where, void* workspace, int64_t workspace_bytes, void* stream) {
  MXQ_REQUIRE(slots >= 0 && slots < (1ll << 30) && experts >= 1 && experts <= kMostExperts, MXQ_ERR_VALUE,
              "dispatch: %lld slots, %lld experts (at most %d)", (long long)slots, (long long)experts, kMostExperts);
  const int64_t need = mxq_dispatch_workspace(slots, experts);
  MXQ_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need && reinterpret_cast<uintptr_t>(workspace) % 4 == 0),
              MXQ_ERR_VALUE, "dispatch: needs a workspace of %lld bytes", (long long)need);
  cudaStream_t st = as_stream(stream);
  const int smem = (int)((kDispatchWarps + 2) * experts + 32) * 4, most = ((kDispatchWarps + 2) * kMostExperts + 32) * 4;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kDispatchWarps * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  cfg.attrs = at;
  cfg.numAttrs = 1;
  if (need) {
    int* counts = static_cast<int*>(workspace);
    const int ctas = dispatch_ctas(slots);
    k_dispatch_count<<<ctas, kDispatchWarps * 32, (size_t)experts * 4, st>>>(experts_of, slots, (int)experts, counts);
    if (int rc = MXQ_LAUNCH_CHECK("dispatch")) return rc;
    if (int rc = allow_smem((const void*)k_dispatch<true>, most)) return rc;
    cfg.gridDim = dim3(ctas);
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    return check_cuda(cudaLaunchKernelEx(&cfg, k_dispatch<true>, experts_of, slots, (int)experts, (const int*)counts, offsets, order, where),
                      "dispatch");
  }
  if (int rc = allow_smem((const void*)k_dispatch<false>, most)) return rc;
  // a CTA walks 2048 slots in four steps per warp; a cluster (at most 8 CTAs) shares more
  int ctas = 1;
  while (ctas < 8 && slots > 2048ll * ctas) ctas *= 2;
  cfg.gridDim = dim3(ctas);
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = ctas;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, k_dispatch<false>, experts_of, slots, (int)experts, (const int*)nullptr, offsets, order, where),
                    "dispatch");
}

static int check_combine(const char* who, int64_t T, int64_t k, int64_t N) {
  MXQ_REQUIRE(T >= 0 && k >= 1 && N >= 0 && T * k < (1ll << 31), MXQ_ERR_VALUE, "%s: T %lld, k %lld, N %lld", who, (long long)T, (long long)k,
              (long long)N);
  return MXQ_OK;
}

extern "C" int mxq_combine(const void* z, int32_t type, const float* weights, const int32_t* where, const void* residual,
                           int64_t residual_stride, void* y, int64_t T, int64_t k, int64_t N, void* stream) {
  if (int rc = check_combine("combine", T, k, N)) return rc;
  if (T == 0 || N == 0) return MXQ_OK;
  return by_type("combine", type, [&](auto zero) {
    using X = decltype(zero);
    constexpr int V = Vec<X>::N;
    const bool vec = N % V == 0 && aligned16(z) && aligned16(y) && (!residual || (aligned16(residual) && residual_stride % V == 0));
    const int64_t threads = (N + V - 1) / V;
    const int block = threads > 128 ? 256 : threads > 64 ? 128 : 64;
    const dim3 grid((unsigned)T, (unsigned)((threads + block - 1) / block));
    auto f = vec ? k_combine<X, true> : k_combine<X, false>;
    f<<<grid, block, 0, as_stream(stream)>>>(static_cast<const X*>(z), weights, where, static_cast<const X*>(residual), residual_stride,
                                             static_cast<X*>(y), (int)k, N, T * k);
    return MXQ_LAUNCH_CHECK("combine");
  });
}

extern "C" int mxq_combine_backward(const void* dy, int64_t dy_stride, const void* z, int32_t type, const float* weights,
                                    const int32_t* where, const int32_t* order, void* dz, float* dw, int64_t T, int64_t k, int64_t N,
                                    void* stream) {
  if (int rc = check_combine("combine_backward", T, k, N)) return rc;
  if (T == 0) return MXQ_OK;
  return by_type("combine_backward", type, [&](auto zero) {
    using X = decltype(zero);
    constexpr int V = Vec<X>::N;
    const bool vec = N % V == 0 && aligned16(z) && aligned16(dz) && aligned16(dy) && dy_stride % V == 0;
    const int64_t threads = (N + V - 1) / V;
    const int block = threads > 128 ? 256 : threads > 64 ? 128 : 64;
    auto go = [&](auto width) {
      constexpr int J = decltype(width)::value;
      auto f = vec ? k_combine_backward<X, true, J> : k_combine_backward<X, false, J>;
      f<<<(unsigned)T, block, 0, as_stream(stream)>>>(static_cast<const X*>(dy), dy_stride, static_cast<const X*>(z), weights, where, order,
                                                      static_cast<X*>(dz), dw, (int)k, N, (int)(T * k));
    };
    switch (k) {
      case 1: go(Int<1>{}); break;
      case 2: go(Int<2>{}); break;
      case 3: case 4: go(Int<4>{}); break;
      case 5: case 6: go(Int<6>{}); break;
      default: go(Int<8>{});
    }
    return MXQ_LAUNCH_CHECK("combine_backward");
  });
}
