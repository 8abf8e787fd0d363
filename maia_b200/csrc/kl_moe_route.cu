// Mixture-of-experts routing: the k experts of every token, their weights, the experts' counts and
// the balance loss, and the gradient of the logits (kl_moe_route, kl_moe_route_grad).
//
// p = softmax(l) over a token's E logits; the k largest l are chosen (ties: the lower index);
// w_j = p_{e_j}, or p_{e_j} / sum_i p_{e_i}. With c_e the number of slots that name e and N the
// routed tokens, the loss is E sum_e (c_e / (k N)) (1/N sum_t p_te). The counts have no gradient:
// with a_e = dL E c_e / (k N^2) and D = sum_j dw_j w_j,
//   dl_te = p_te (a_e - sum_e' p_te' a_e' - [w = p] D) + [e = e_j] w_j (dw_j - [w normalised] D).
//
// Both kernels read a row once and keep it in registers, 8 experts to a lane. What bounds them is not
// the memory but the instructions: at 256 bf16 logits a token, HBM would allow about 100 a token. So a lane sorts its
// eight keys once (19 exchanges), after which each of the k rounds takes one warp-wide maximum and a shift in the lane that
// held it (two sorted keys a lane, enough for four tokens of ten, and a second search for the rest: 69 us instead
// of 62).
// Measured, 131072 tokens of 256 bf16 experts, k = 8: routing and its sums 61 us (361 instructions a token, half of
// them on the integer pipe, which is full), gradient 44 us (280 a token). One token of 64 fp32 experts: 3.3 us. Above 512
// experts fp32 keys and values do not fit the registers (300 bytes a thread spill): 32768 x 1024 112 and 77 us.

#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <string>

#include <kl/arch/griddep.hpp>
#include <kl_gemm.h>

#include "kl_experts.cuh"
#include "kl_internal.cuh"
#include "kl_vec.cuh"

namespace cg = cooperative_groups;

namespace kl::capi {
namespace {

constexpr int kRouteThreads = 512;
constexpr int kRouteWarps = kRouteThreads / 32;

// Ordering keys: larger key = earlier choice. The value's bits in an order-preserving form sit above
// 1023 - e, so one integer maximum gives the largest value and, among equals, the lowest expert.
// 16-bit logits leave the low 12 bits of their fp32 form zero, so key and index share 32 bits. Adding 0
// makes both zeros +0 and every NaN the positive one, which orders above everything; keys up to
// kClosed are -inf, which is never chosen.
template <class T>
struct RouteKey {
  using type = uint32_t;
  static constexpr type kClosed = 0x007FFFFFu;
  static __device__ __forceinline__ type make(uint32_t ordered, int e) {
    return (ordered & 0xFFFFF000u) | uint32_t(kMaxExperts - 1 - e);
  }
  static __device__ __forceinline__ float value(type k) {
    if (k >= 0xFFFFF000u) return NAN;
    return __uint_as_float(k & 0x80000000u ? (k & 0x7FFFF000u) : ~(k | 0xFFFu));
  }
};
template <>
struct RouteKey<float> {
  using type = uint64_t;
  static constexpr type kClosed = 0x007FFFFFFFFFFFFFull;
  static __device__ __forceinline__ type make(uint32_t ordered, int e) {
    return (uint64_t(ordered) << 32) | uint32_t(kMaxExperts - 1 - e);
  }
  static __device__ __forceinline__ float value(type k) {
    const uint32_t o = uint32_t(k >> 32);
    if (o == 0xFFFFFFFFu) return NAN;
    return __uint_as_float(o & 0x80000000u ? o & 0x7FFFFFFFu : ~o);
  }
};
__device__ __forceinline__ uint32_t ordered_bits(float v) {
  const uint32_t u = __float_as_uint(v + 0.0f);
  return u ^ (uint32_t(int32_t(u) >> 31) | 0x80000000u);
}
template <class K>
__device__ __forceinline__ int key_expert(K k) {
  return kMaxExperts - 1 - int(uint32_t(k) & (kMaxExperts - 1));
}

// Eight keys, largest first, by a sorting network of 19 exchanges.
template <class K>
__device__ __forceinline__ void sort8(K (&s)[8]) {
  auto swap = [&](int i, int j) {
    const K hi = s[i] > s[j] ? s[i] : s[j];
    s[j] = s[i] > s[j] ? s[j] : s[i];
    s[i] = hi;
  };
  swap(0, 1); swap(2, 3); swap(4, 5); swap(6, 7);
  swap(0, 2); swap(1, 3); swap(4, 6); swap(5, 7);
  swap(1, 2); swap(5, 6); swap(0, 4); swap(3, 7);
  swap(1, 5); swap(2, 6);
  swap(1, 4); swap(3, 6);
  swap(2, 4); swap(3, 5);
  swap(3, 4);
}

// L lanes share a token; lane i holds experts (v L + i) 8 + 0..7 for v < NV.
template <int L>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o /= 2) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}
// The larger, or NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
template <int L>
__device__ __forceinline__ float group_max_nan(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o /= 2) v = max_nan(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
  return v;
}
template <int L, class K>
__device__ __forceinline__ K group_key_max(K k) {
  if constexpr (L == 32 && sizeof(K) == 4) {
    return __reduce_max_sync(0xFFFFFFFFu, k);
  } else {
#pragma unroll
    for (int o = L / 2; o > 0; o /= 2) {
      const K other = __shfl_xor_sync(0xFFFFFFFFu, k, o);
      k = other > k ? other : k;
    }
    return k;
  }
}

// A row's logits as they lie: whole 16-byte vectors where `vec` (aligned rows, E a multiple of 8), else
// element by element; -inf outside the row, and for a row that is not `live`.
template <class T, int NV>
struct Row {
  uint4 u[NV * 8 / kPerVec<T>];
};
template <class T>
__device__ __forceinline__ T minus_infinity() { return from_f32<T>(-INFINITY); }
template <class T, int L, int NV>
__device__ __forceinline__ void load_row(const T* row, int lane, int experts, bool vec, bool live, Row<T, NV>& r) {
  constexpr int kVecs = 8 / kPerVec<T>;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e0 = (i * L + lane) * 8;
    if (vec && live && e0 < experts) {
#pragma unroll
      for (int j = 0; j < kVecs; ++j) r.u[i * kVecs + j] = reinterpret_cast<const uint4*>(row + e0)[j];
    } else {
      T v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = live && e0 + j < experts ? row[e0 + j] : minus_infinity<T>();
      memcpy(&r.u[i * kVecs], v, sizeof(v));
    }
  }
}
template <class T, int NV>
__device__ __forceinline__ void values(Row<T, NV> const& r, float (&v)[8 * NV]) {
#pragma unroll
  for (int i = 0; i < NV * 8 / kPerVec<T>; ++i) unpack<T>(r.u[i], v + i * kPerVec<T>);
}

// exp(x) for x <= 0 as one product and one ex2: off by |x| + 4 times 2^-24, relative, and 0 below 2^-126. For a row's sum
// and what adds up over tokens, where the large probabilities count and have small |x|. The k weights, which a user
// sees one by one, take expf (131072 tokens of 256 experts: 63.9 us instead of 63.2).
__device__ __forceinline__ float exp_neg(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * 1.44269504f));
  return y;
}

struct RouteArgs {
  const void* logits;
  long long ld;
  int tokens, experts, k;
  int renormalize;
  const uint8_t* valid;
  int* ids;
  float* weights;
  int* counts;
  int* routed;
  float* loss;
  // Partial sums of block b: share[b E + e], count[b E + e], routed_part[b]. Unused by one block.
  float* share_part;
  int* count_part;
  int* routed_part;
  int vec;
};

// The loss from the finished counts and probability sums: every thread brings its experts' terms
// (sum over e of c_e s_e); the division by k N^2 comes last.
__device__ __forceinline__ float block_total(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o /= 2) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = v;
  __syncthreads();
  float t = 0.0f;
  for (int w = 0; w < int(blockDim.x) / 32; ++w) t += red[w];
  __syncthreads();
  return t;
}
__device__ __forceinline__ float loss_of(float total, int experts, int k, int routed) {
  return routed > 0 ? float(experts) * (total / (float(k) * float(routed))) / float(routed) : 0.0f;
}

// KMAX: the most rounds, 8 or 32; the lists shrink as the rounds left do, which at 8 rounds saves 4 us of 67 (131072
// tokens of 256 experts).
template <class T, int L, int NV, int KMAX>
__global__ void __launch_bounds__(kRouteThreads, NV == 1 ? 2 : 1) route_kernel(const RouteArgs a) {
  using Key = RouteKey<T>;
  using K = typename Key::type;
  constexpr int kGroups = 32 / L;  // tokens of a warp
  constexpr int kWidth = L * 8 * NV;
  constexpr int kPicks = L * 8 < KMAX ? L * 8 : KMAX;  // k is at most the number of experts
  constexpr int kHeld = (kPicks + L - 1) / L;          // picks of a lane: j = h L + lane
  extern __shared__ float share[];                             // [kRouteWarps][kWidth]
  __shared__ int count[kWidth];
  __shared__ float red[32];
  __shared__ int routed_here;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % L, group = threadIdx.x % 32 / L;
  for (int e = threadIdx.x; e < a.experts; e += kRouteThreads) count[e] = 0;
  if (threadIdx.x == 0) routed_here = 0;
  __syncthreads();
  griddep_wait();
  griddep_launch_dependents();
  const T* logits = static_cast<const T*>(a.logits);
  float acc[8 * NV];
#pragma unroll
  for (int i = 0; i < 8 * NV; ++i) acc[i] = 0.0f;
  const long long step = (long long)gridDim.x * kRouteWarps * kGroups;
  auto is_live = [&](long long t) { return t < a.tokens && (a.valid == nullptr || a.valid[t] != 0); };
  int routed = 0;
  long long t = (long long)(blockIdx.x * kRouteWarps + warp) * kGroups + group;
  Row<T, NV> next;
  load_row<T, L, NV>(logits + (t < a.tokens ? t : 0) * a.ld, lane, a.experts, a.vec, is_live(t), next);
  // Whole warps leave the loop together: the shuffles take every lane.
  for (; t - group < a.tokens; t += step) {
    float v[8 * NV];
    values<T, NV>(next, v);
    if (t - group + step < a.tokens)
      load_row<T, L, NV>(logits + (t + step < a.tokens ? t + step : 0) * a.ld, lane, a.experts, a.vec, is_live(t + step), next);
    // The k largest keys, one after another: the largest head of all lanes, taken off its lane's list.
    K pick[kHeld] = {};
    K first = 0;
    K key[NV][8];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int j = 0; j < 8; ++j) key[i][j] = Key::make(ordered_bits(v[8 * i + j]), (i * L + lane) * 8 + j);
      sort8(key[i]);
    }
#pragma unroll
    for (int j = 0; j < kPicks; ++j) {
      if (j >= a.k) break;
      K best = key[0][0];
#pragma unroll
      for (int i = 1; i < NV; ++i) best = key[i][0] > best ? key[i][0] : best;
      best = group_key_max<L>(best);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (key[i][0] == best) {
#pragma unroll
          for (int x = 0; x < 7; ++x)
            if (x < kPicks - 1 - j) key[i][x] = key[i][x + 1];
          if (7 < kPicks - 1 - j) key[i][7] = K(0);
        }
      }
      if (lane == j % L) pick[j / L] = best;
      if (j == 0) first = best;
    }
    const bool any = first > Key::kClosed;
    const float top = Key::value(first);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 8 * NV; ++i) {
      v[i] = exp_neg(v[i] - top);
      sum += v[i];
    }
    sum = group_sum<L>(sum);
    float inv = 1.0f / sum;
    if (any) {
#pragma unroll
      for (int i = 0; i < 8 * NV; ++i) acc[i] = fmaf(v[i], inv, acc[i]);
      routed += lane == 0;
    }
    float w[kHeld], part = 0.0f;
#pragma unroll
    for (int h = 0; h < kHeld; ++h) {
      w[h] = h * L + lane < a.k && pick[h] > Key::kClosed ? expf(Key::value(pick[h]) - top) : 0.0f;
      part += w[h];
    }
    if (a.renormalize) inv = 1.0f / group_sum<L>(part);
    if (t < a.tokens) {
#pragma unroll
      for (int h = 0; h < kHeld; ++h) {
        const int j = h * L + lane;
        if (j >= a.k) break;
        const bool open = pick[h] > Key::kClosed;
        const int e = open ? key_expert(pick[h]) : -1;
        a.ids[t * a.k + j] = e;
        a.weights[t * a.k + j] = open ? w[h] * inv : 0.0f;
        if (open) atomicAdd(&count[e], 1);
      }
    }
  }
  // Block sums in a fixed order: the groups of a warp by shuffles, the warps one after another.
#pragma unroll
  for (int i = 0; i < 8 * NV; ++i) {
#pragma unroll
    for (int o = L; o < 32; o *= 2) acc[i] += __shfl_xor_sync(0xFFFFFFFFu, acc[i], o);
    if (group == 0) share[warp * kWidth + (i / 8 * L + lane) * 8 + i % 8] = acc[i];
  }
  if (routed) atomicAdd(&routed_here, routed);
  __syncthreads();
  float terms = 0.0f;
  for (int e = threadIdx.x; e < a.experts; e += kRouteThreads) {
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < kRouteWarps; ++w) s += share[w * kWidth + e];
    if (gridDim.x == 1) {
      a.counts[e] = count[e];
      terms += s * float(count[e]);
    } else {
      a.share_part[(long long)blockIdx.x * a.experts + e] = s;
      a.count_part[(long long)blockIdx.x * a.experts + e] = count[e];
    }
  }
  if (gridDim.x == 1) {
    const float total = block_total(terms, red);
    if (threadIdx.x == 0) {
      *a.routed = routed_here;
      *a.loss = loss_of(total, a.experts, a.k, routed_here);
    }
  } else if (threadIdx.x == 0) {
    a.routed_part[blockIdx.x] = routed_here;
  }
}

// The blocks' partial sums by one cluster, in a fixed order: a thread takes every so-manieth block of
// one expert; the threads of an expert meet in shared memory, the cluster's blocks in rank order. A latency:
// 12 us by itself with cold caches for 296 blocks of 256 experts, part of it hidden behind the routing kernel's end.
constexpr int kFinishBlocks = 8;
constexpr int kFinishThreads = 1024;
__global__ void __launch_bounds__(kFinishThreads) route_finish_kernel(const RouteArgs a, int blocks) {
  __shared__ float share[kFinishThreads];
  __shared__ int count[kFinishThreads];
  __shared__ float term_sum;
  __shared__ float red[32];
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = int(cluster.block_rank());
  griddep_wait();
  griddep_launch_dependents();
  const int rows = kFinishThreads / a.experts, row = threadIdx.x / a.experts, e = threadIdx.x % a.experts;  // experts <= 1024
  float s = 0.0f;
  int c = 0;
  if (row < rows)
#pragma unroll 4
    for (int b = rank * rows + row; b < blocks; b += kFinishBlocks * rows) {
      s += a.share_part[(long long)b * a.experts + e];
      c += a.count_part[(long long)b * a.experts + e];
    }
  share[threadIdx.x] = s;
  count[threadIdx.x] = c;
  __syncthreads();
  if (row == 0) {
    for (int r = 1; r < rows; ++r) {
      s += share[r * a.experts + e];
      c += count[r * a.experts + e];
    }
    share[e] = s;
    count[e] = c;
  }
  cluster.sync();
  // Block `rank` ends the experts rank, rank + 8, ...
  float terms = 0.0f;
  const int mine = rank + kFinishBlocks * threadIdx.x;
  if (mine < a.experts) {
    s = 0.0f;
    c = 0;
    for (int r = 0; r < kFinishBlocks; ++r) {
      s += cluster.map_shared_rank(share, r)[mine];
      c += cluster.map_shared_rank(count, r)[mine];
    }
    a.counts[mine] = c;
    terms = s * float(c);
  }
  const float total = block_total(terms, red);
  if (threadIdx.x == 0) term_sum = total;
  cluster.sync();
  if (rank == 0 && threadIdx.x < 32) {
    int n = 0;
    for (int b = threadIdx.x; b < blocks; b += 32) n += a.routed_part[b];
    n = __reduce_add_sync(0xFFFFFFFFu, n);
    float all = 0.0f;
    for (int r = 0; r < kFinishBlocks; ++r) all += *cluster.map_shared_rank(&term_sum, r);
    if (threadIdx.x == 0) {
      *a.routed = n;
      *a.loss = loss_of(all, a.experts, a.k, n);
    }
  }
  cluster.sync();  // no block leaves while another may still read its sums
}

struct RouteGradArgs {
  const void* logits;
  long long ld;
  int tokens, experts, k;
  int renormalize;
  const uint8_t* valid;
  const int* ids;
  const float* weights;
  const int* counts;
  const int* routed;
  const float* dweights;
  const float* dloss;
  void* dlogits;
  long long ldd;
  int vec;
};

// One pass: the softmax again, two sums over the lanes, the chosen experts' own terms by way of shared memory. 45 us at
// 131072 x 256 bf16 (3.3 TB/s; 22.7 us at the copy rate); bound by its 280 instructions a token, the exchanges among
// them.
constexpr int kGradThreads = 256;
constexpr int kGradWarps = kGradThreads / 32;
template <class T, int L, int NV>
__global__ void __launch_bounds__(kGradThreads, NV == 1 && L >= 8 ? 4 : 2) route_grad_kernel(const RouteGradArgs a) {
  constexpr int kGroups = 32 / L;
  constexpr int kWidth = L * 8 * NV;
  // The chosen experts' own terms, else 0. A lane's eight lie in two vectors, each beside its neighbours' own.
  __shared__ float4 spot[kGradWarps * kGroups][kWidth / 4];
  auto place = [](int e) { return ((e / (8 * L) * 2 + e % 8 / 4) * L + e / 8 % L) * 4 + e % 4; };
  const int warp = threadIdx.x / 32, lane = threadIdx.x % L, group = threadIdx.x % 32 / L;
  for (int i = threadIdx.x; i < kGradWarps * kGroups * kWidth; i += kGradThreads) reinterpret_cast<float*>(spot)[i] = 0.0f;
  griddep_wait();
  griddep_launch_dependents();
  const float n = float(*a.routed > 0 ? *a.routed : 1);
  const float dloss = a.dloss != nullptr ? *a.dloss : 0.0f;
  float push[8 * NV];  // a_e of this lane's experts
#pragma unroll
  for (int i = 0; i < 8 * NV; ++i) {
    const int e = (i / 8 * L + lane) * 8 + i % 8;
    push[i] = e < a.experts ? dloss * float(a.experts) * (float(a.counts[e]) / (float(a.k) * n)) / n : 0.0f;
  }
  __syncthreads();
  const T* logits = static_cast<const T*>(a.logits);
  T* out = static_cast<T*>(a.dlogits);
  float4* mine = spot[warp * kGroups + group];
  float* mine_at = reinterpret_cast<float*>(mine);
  const long long step = (long long)gridDim.x * kGradWarps * kGroups;
  auto is_live = [&](long long t) { return t < a.tokens && (a.valid == nullptr || a.valid[t] != 0); };
  // Lane j of a token has slot j (of more than L slots, also j + L, ...).
  constexpr int kHeld = ((L * 8 < kMaxTopK ? L * 8 : kMaxTopK) + L - 1) / L;
  struct Slot {
    int e;  // -1: nothing to add
    float w, dw;
  };
  Slot slots[kHeld];
  Row<T, NV> next;
  auto load = [&](long long t) {
    const bool live = is_live(t);
    load_row<T, L, NV>(logits + (t < a.tokens ? t : 0) * a.ld, lane, a.experts, a.vec, live, next);
#pragma unroll
    for (int h = 0; h < kHeld; ++h) {
      const int j = h * L + lane;
      slots[h] = {-1, 0.0f, 0.0f};
      if (live && a.dweights != nullptr && j < a.k) slots[h] = {a.ids[t * a.k + j], a.weights[t * a.k + j], a.dweights[t * a.k + j]};
    }
  };
  long long t = (long long)(blockIdx.x * kGradWarps + warp) * kGroups + group;
  load(t);
  for (; t - group < a.tokens; t += step) {
    float v[8 * NV];
    values<T, NV>(next, v);
    int e_of[kHeld];
    float pull_of[kHeld], w_of[kHeld], pull = 0.0f;
#pragma unroll
    for (int h = 0; h < kHeld; ++h) {
      e_of[h] = slots[h].e < a.experts ? slots[h].e : -1;
      w_of[h] = slots[h].w;
      pull_of[h] = e_of[h] >= 0 ? slots[h].w * slots[h].dw : 0.0f;
      pull += pull_of[h];
    }
    if (t - group + step < a.tokens) load(t + step);
    float top = v[0];
#pragma unroll
    for (int i = 1; i < 8 * NV; ++i) top = max_nan(top, v[i]);
    top = group_max_nan<L>(top);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 8 * NV; ++i) {
      v[i] = exp_neg(v[i] - top);
      sum += v[i];
    }
    sum = group_sum<L>(sum);
    // A row of -inf alone is not routed: zeros, whatever dloss and dweights hold.
    const bool any = top != -INFINITY;
    const float inv = 1.0f / sum;
    float level = 0.0f;
#pragma unroll
    for (int i = 0; i < 8 * NV; ++i) {
      v[i] *= inv;
      level = fmaf(v[i], push[i], level);
    }
    float base;
    if (a.renormalize) {
      pull = group_sum<L>(pull);
      base = group_sum<L>(level);
    } else {
      base = group_sum<L>(level + pull);
      pull = 0.0f;
    }
#pragma unroll
    for (int h = 0; h < kHeld; ++h)
      if (e_of[h] >= 0) mine_at[place(e_of[h])] = fmaf(-w_of[h], pull, pull_of[h]);
    __syncwarp();
    if (t < a.tokens) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int e0 = (i * L + lane) * 8;
        const float4 s0 = mine[i * 2 * L + lane], s1 = mine[(i * 2 + 1) * L + lane];
        float g[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) g[j] = any ? fmaf(v[8 * i + j], push[8 * i + j] - base, g[j]) : 0.0f;
        if (e0 >= a.experts) continue;
        if (a.vec) {
          uint4* p = reinterpret_cast<uint4*>(out + t * a.ldd + e0);
#pragma unroll
          for (int j = 0; j < 8 / kPerVec<T>; ++j) p[j] = pack<T>(g + j * kPerVec<T>);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (e0 + j < a.experts) out[t * a.ldd + e0 + j] = from_f32<T>(g[j]);
        }
      }
    }
    __syncwarp();
#pragma unroll
    for (int h = 0; h < kHeld; ++h)
      if (e_of[h] >= 0) mine_at[place(e_of[h])] = 0.0f;
    __syncwarp();
  }
}

// Lanes of a token: enough for 8 experts each, at most a warp; wider rows take more vectors a lane.
template <class F>
void by_width(int experts, F&& f) {
  if (experts <= 8) f(std::integral_constant<int, 1>{}, std::integral_constant<int, 1>{});
  else if (experts <= 16) f(std::integral_constant<int, 2>{}, std::integral_constant<int, 1>{});
  else if (experts <= 32) f(std::integral_constant<int, 4>{}, std::integral_constant<int, 1>{});
  else if (experts <= 64) f(std::integral_constant<int, 8>{}, std::integral_constant<int, 1>{});
  else if (experts <= 128) f(std::integral_constant<int, 16>{}, std::integral_constant<int, 1>{});
  else if (experts <= 256) f(std::integral_constant<int, 32>{}, std::integral_constant<int, 1>{});
  else if (experts <= 512) f(std::integral_constant<int, 32>{}, std::integral_constant<int, 2>{});
  else f(std::integral_constant<int, 32>{}, std::integral_constant<int, 4>{});
}

template <class F>
void by_type(int32_t type, F&& f) {
  if (type == KL_F32) f(float{});
  else if (type == KL_F16) f(__half{});
  else f(__nv_bfloat16{});
}

int lanes_of(int experts) {
  int lanes = 1;
  while (lanes < 32 && lanes * 8 < experts) lanes *= 2;
  return lanes;
}

// Blocks of the routing kernel: one, and no second kernel, where its warps take at most 256 tokens in at most four
// turns, else up to the two that every SM of a 148-SM B200 holds. One block against many, k = 8: 64 tokens of 256
// experts 6.6 and 7.5 us, 128 tokens 11.2 and 7.5; 256 tokens of 64 experts 7.4 and 7.7, 1024 tokens 23.7 and 7.4;
// 512 tokens of 8 experts 7.2 and 7.2, 2048 tokens 19.9 and 12.0.
int route_blocks(int64_t tokens, int experts) {
  const int64_t turn = kRouteWarps * (32 / lanes_of(experts));  // tokens of one block at a time
  if (tokens <= 4 * turn && tokens <= 256) return 1;
  const int64_t blocks = (tokens + turn - 1) / turn;
  return int(blocks < 296 ? blocks : 296);
}

kl_status check_route(char const* who, int64_t tokens, int64_t experts, int64_t k, int32_t type, int64_t ld) {
  if (tokens < 0 || tokens > INT32_MAX / kMaxTopK) return fail(KL_ERR_INVALID_ARGUMENT, std::string(who) + ": tokens must be in [0, 2^26)");
  if (experts < 1 || experts > kMaxExperts)
    return fail(KL_ERR_NOT_SUPPORTED, std::string(who) + ": experts must be in [1, 1024]");
  if (k < 1 || k > kMaxTopK || k > experts)
    return fail(KL_ERR_INVALID_ARGUMENT, std::string(who) + ": k must be in [1, min(experts, 32)]");
  if (type != KL_BF16 && type != KL_F16 && type != KL_F32)
    return fail(KL_ERR_NOT_SUPPORTED, std::string(who) + ": logits must be bf16, f16 or f32");
  if (ld < experts) return fail(KL_ERR_INVALID_ARGUMENT, std::string(who) + ": row pitch below the number of experts");
  return KL_OK;
}

bool vector_rows(const void* p, int64_t ld, int64_t experts, int32_t type) {
  const int64_t size = type == KL_F32 ? 4 : 2;
  return aligned16(p) && ld * size % 16 == 0 && experts % 8 == 0;
}

}  // namespace
}  // namespace kl::capi

extern "C" kl_status kl_moe_route_workspace_size(int64_t tokens, int64_t experts, size_t* bytes) {
  using namespace kl::capi;
  if (bytes == nullptr) return fail(KL_ERR_INVALID_ARGUMENT, "kl_moe_route_workspace_size: null pointer");
  kl_status s = check_route("kl_moe_route_workspace_size", tokens, experts, 1, KL_F32, experts);
  if (s != KL_OK) return s;
  const int blocks = route_blocks(tokens, int(experts));
  *bytes = blocks == 1 ? 0 : size_t(blocks) * (2 * size_t(experts) + 1) * 4;
  return KL_OK;
}

extern "C" kl_status kl_moe_route(const kl_moe_route_desc* d, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace kl::capi;
  if (d == nullptr) return fail(KL_ERR_INVALID_ARGUMENT, "kl_moe_route: null descriptor");
  kl_status s = check_route("kl_moe_route", d->tokens, d->experts, d->k, d->logits_type, d->ld_logits);
  if (s != KL_OK) return s;
  if (d->counts == nullptr || d->routed == nullptr || d->loss == nullptr ||
      (d->tokens > 0 && (d->logits == nullptr || d->ids == nullptr || d->weights == nullptr)))
    return fail(KL_ERR_INVALID_ARGUMENT, "kl_moe_route: null pointer");
  if (!aligned(d->logits, d->logits_type == KL_F32 ? 4 : 2))
    return fail(KL_ERR_INVALID_ARGUMENT, "kl_moe_route: logits must be aligned to their elements");
  if (!words_aligned({d->ids, d->weights, d->counts, d->routed, d->loss}))
    return fail(KL_ERR_INVALID_ARGUMENT, "kl_moe_route: ids, weights, counts, routed and loss must be 4-byte aligned");
  const int blocks = route_blocks(d->tokens, int(d->experts));
  size_t need = 0;
  kl_moe_route_workspace_size(d->tokens, d->experts, &need);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 4 != 0))
    return fail(KL_ERR_INVALID_ARGUMENT, "kl_moe_route: needs a 4-byte aligned workspace of " + std::to_string(need) + " bytes");
  RouteArgs a = {};
  a.logits = d->logits;
  a.ld = d->ld_logits;
  a.tokens = int(d->tokens);
  a.experts = int(d->experts);
  a.k = int(d->k);
  a.renormalize = d->renormalize;
  a.valid = d->valid;
  a.ids = d->ids;
  a.weights = d->weights;
  a.counts = d->counts;
  a.routed = d->routed;
  a.loss = d->loss;
  a.share_part = static_cast<float*>(workspace);
  a.count_part = reinterpret_cast<int*>(a.share_part + size_t(blocks) * d->experts);
  a.routed_part = a.count_part + size_t(blocks) * d->experts;
  a.vec = vector_rows(d->logits, d->ld_logits, d->experts, d->logits_type);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaSuccess;
  by_type(d->logits_type, [&](auto t) {
    by_width(a.experts, [&](auto l, auto nv) {
      void* args[] = {&a};
      using T = decltype(t);
      void const* kernel = a.k <= 8 ? reinterpret_cast<void const*>(&route_kernel<T, l(), nv(), 8>)
                                    : reinterpret_cast<void const*>(&route_kernel<T, l(), nv(), kMaxTopK>);
      e = launch_dependent(st, blocks, kRouteThreads, size_t(kRouteWarps) * l() * 8 * nv() * sizeof(float), 1, kernel, args);
    });
  });
  if (e == cudaSuccess && blocks > 1) {
    int b = blocks;
    void* args[] = {&a, &b};
    e = launch_dependent(st, kFinishBlocks, kFinishThreads, 0, kFinishBlocks, reinterpret_cast<void const*>(&route_finish_kernel), args);
  }
  return e == cudaSuccess ? KL_OK : cuda_fail(e, "kl_moe_route launch");
}

extern "C" kl_status kl_moe_route_grad(const kl_moe_route_desc* d, const float* dweights, const float* dloss,
                                       void* dlogits, int64_t ld_dlogits, void* stream) {
  using namespace kl::capi;
  if (d == nullptr) return fail(KL_ERR_INVALID_ARGUMENT, "kl_moe_route_grad: null descriptor");
  kl_status s = check_route("kl_moe_route_grad", d->tokens, d->experts, d->k, d->logits_type, d->ld_logits);
  if (s != KL_OK) return s;
  if (ld_dlogits < d->experts) return fail(KL_ERR_INVALID_ARGUMENT, "kl_moe_route_grad: row pitch below the number of experts");
  if (d->tokens == 0) return KL_OK;
  if (d->logits == nullptr || d->ids == nullptr || d->weights == nullptr || d->counts == nullptr || d->routed == nullptr ||
      dlogits == nullptr)
    return fail(KL_ERR_INVALID_ARGUMENT, "kl_moe_route_grad: null pointer");
  if (!aligned(d->logits, d->logits_type == KL_F32 ? 4 : 2) || !aligned(dlogits, d->logits_type == KL_F32 ? 4 : 2))
    return fail(KL_ERR_INVALID_ARGUMENT, "kl_moe_route_grad: logits and their gradient must be aligned to their elements");
  if (!words_aligned({d->ids, d->weights, d->counts, d->routed, dweights, dloss}))
    return fail(KL_ERR_INVALID_ARGUMENT, "kl_moe_route_grad: ids, weights, counts, routed, dweights and dloss must be 4-byte aligned");
  RouteGradArgs a = {};
  a.logits = d->logits;
  a.ld = d->ld_logits;
  a.tokens = int(d->tokens);
  a.experts = int(d->experts);
  a.k = int(d->k);
  a.renormalize = d->renormalize;
  a.valid = d->valid;
  a.ids = d->ids;
  a.weights = d->weights;
  a.counts = d->counts;
  a.routed = d->routed;
  a.dweights = dweights;
  a.dloss = dloss;
  a.dlogits = dlogits;
  a.ldd = ld_dlogits;
  a.vec = vector_rows(d->logits, d->ld_logits, d->experts, d->logits_type) &&
          vector_rows(dlogits, ld_dlogits, d->experts, d->logits_type);
  const int64_t turn = kGradWarps * (32 / lanes_of(a.experts));
  const int64_t want = (d->tokens + turn - 1) / turn;
  const int blocks = int(want < 592 ? want : 592);
  cudaError_t e = cudaSuccess;
  by_type(d->logits_type, [&](auto t) {
    by_width(a.experts, [&](auto l, auto nv) {
      void* args[] = {&a};
      e = launch_dependent(static_cast<cudaStream_t>(stream), blocks, kGradThreads, 0, 1,
                 reinterpret_cast<void const*>(&route_grad_kernel<decltype(t), l(), nv()>), args);
    });
  });
  return e == cudaSuccess ? KL_OK : cuda_fail(e, "kl_moe_route_grad launch");
}
