// From a router's expert ids to the m-grouped GEMM's row layout and back: kl_moe_plan (counting
// sort of the slots by expert, each expert padded to whole blocks), kl_moe_dispatch (copy every
// token's row to its experts), kl_moe_combine (weighted sum of the experts' rows) and
// kl_moe_combine_grad.
//
// The last three move rows and are bound by memory. Measured on 8192 tokens, 4 experts each, rows of 4096 bf16:
// dispatch 83.6 us (5.6 TB/s; 72.5 us at the copy rate), combine 56.4 (5.4 TB/s), its gradient 112.0 (5.7 TB/s). The
// plan is a latency: 5.2 us for 662 slots, 10.3 for 32768 (64 experts); one cluster takes all sizes, 131072 slots 35 us, 2^20 240
// (256 experts: 42 and 281).

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

constexpr int kPlanThreads = 1024;
constexpr int kPlanWarps = kPlanThreads / 32;
constexpr int kPlanBlocks = 8;  // of the cluster, where one does not do

struct PlanArgs {
  const int* ids;
  long long total;  // slots
  int experts;
  int block;
  long long m;      // rows of the layout
  int* rows;        // [total]
  int* slots;       // [m]
  int* blocks;      // [m / 128]
  long long warp_span;  // consecutive slots of a warp, a multiple of 32
};

// Inclusive sum over the block's 1024 threads.
__device__ __forceinline__ int block_scan(int v, int* red) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const int u = __shfl_up_sync(0xFFFFFFFFu, v, o);
    if (lane >= o) v += u;
  }
  if (lane == 31) red[warp] = v;
  __syncthreads();
  if (warp == 0) {
    int w = red[lane];
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int u = __shfl_up_sync(0xFFFFFFFFu, w, o);
      if (lane >= o) w += u;
    }
    red[lane] = w;
  }
  __syncthreads();
  return warp > 0 ? v + red[warp - 1] : v;
}

// One cluster sorts all slots. Every warp counts the experts of its own run of consecutive slots;
// sums over the warps, then (through distributed shared memory) over the blocks, give each (warp,
// expert) the row of its first slot; a second walk over the same slots hands the rows out. Slots of
// one expert keep their order, and nothing depends on the timing of atomics.
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const PlanArgs a) {
  extern __shared__ int hist[];  // [kPlanWarps][experts]
  __shared__ int block_count[kMaxExperts], starts[kMaxExperts], counts[kMaxExperts];
  __shared__ int red[32];
  cg::cluster_group cluster = cg::this_cluster();
  griddep_wait();
  griddep_launch_dependents();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int rank = int(cluster.block_rank()), ranks = int(cluster.num_blocks());
  for (int i = threadIdx.x; i < kPlanWarps * a.experts; i += kPlanThreads) hist[i] = 0;
  __syncthreads();
  int* mine = hist + warp * a.experts;
  const long long begin = ((long long)rank * kPlanWarps + warp) * a.warp_span;
  const long long end = begin + a.warp_span < a.total ? begin + a.warp_span : a.total;
  auto expert_at = [&](long long s) {
    const int e = s < end ? a.ids[s] : -1;
    return e >= 0 && e < a.experts ? e : -1;
  };
  // The first kKept turns' ids stay in registers for the second walk; they load together.
  constexpr int kKept = 8;
  int kept[kKept];
#pragma unroll
  for (int i = 0; i < kKept; ++i) kept[i] = expert_at(begin + i * 32 + lane);
  auto count = [&](int e) {
    const unsigned same = __match_any_sync(0xFFFFFFFFu, e);
    if (e >= 0 && lane == __ffs(same) - 1) mine[e] += __popc(same);
    __syncwarp();
  };
#pragma unroll
  for (int i = 0; i < kKept; ++i)
    if (begin + i * 32 < end) count(kept[i]);
  for (long long s = begin + kKept * 32; s < end; s += 32) count(expert_at(s + lane));
  __syncthreads();
  const int e = threadIdx.x;
  if (e < a.experts) {
    int run = 0, c[kPlanWarps];
#pragma unroll
    for (int w = 0; w < kPlanWarps; ++w) c[w] = hist[w * a.experts + e];
#pragma unroll
    for (int w = 0; w < kPlanWarps; ++w) {
      hist[w * a.experts + e] = run;
      run += c[w];
    }
    block_count[e] = run;
  }
  cluster.sync();
  int before = 0, all = 0;
  if (e < a.experts) {
    int c[kPlanBlocks];
#pragma unroll
    for (int r = 0; r < kPlanBlocks; ++r) c[r] = r < ranks ? cluster.map_shared_rank(block_count, r)[e] : 0;
#pragma unroll
    for (int r = 0; r < kPlanBlocks; ++r) {
      before += r < rank ? c[r] : 0;
      all += c[r];
    }
  }
  const int room = (all + a.block - 1) / a.block * a.block;
  const int stop = block_scan(room, red);
  const int start = stop - room;
  if (e < a.experts)
    for (int w = 0; w < kPlanWarps; ++w) hist[w * a.experts + e] += start + before;
  // The padding behind each expert's rows, its blocks (a warp an expert), and the blocks that nobody has.
  if (e < a.experts) {
    starts[e] = start;
    counts[e] = all;
  }
  __syncthreads();
  for (int x = rank * kPlanWarps + warp; x < a.experts; x += ranks * kPlanWarps) {
    const int s0 = starts[x], n = counts[x], s1 = s0 + (n + a.block - 1) / a.block * a.block;
    for (int r = s0 + n + lane; r < s1; r += 32) a.slots[r] = -1;
    for (int b = s0 / 128 + lane; b < s1 / 128; b += 32) a.blocks[b] = x;
  }
  const long long used = red[31];
  for (long long r = used + rank * kPlanThreads + threadIdx.x; r < a.m; r += ranks * kPlanThreads) {
    a.slots[r] = -1;
    if (r % 128 == 0) a.blocks[r / 128] = -1;
  }
  auto hand_out = [&](long long s, int x) {
    const unsigned same = __match_any_sync(0xFFFFFFFFu, x);
    int row = -1;
    if (x >= 0) row = mine[x] + __popc(same & ((1u << lane) - 1));
    __syncwarp();
    if (x >= 0 && lane == __ffs(same) - 1) mine[x] += __popc(same);
    __syncwarp();
    if (s + lane < end) a.rows[s + lane] = row;
    if (row >= 0) a.slots[row] = int(s + lane);
  };
#pragma unroll
  for (int i = 0; i < kKept; ++i)
    if (begin + i * 32 < end) hand_out(begin + i * 32, kept[i]);
  for (long long s = begin + kKept * 32; s < end; s += 32) hand_out(s, expert_at(s + lane));
  cluster.sync();  // no block leaves while another may still read its counts
}

constexpr int kRowThreads = 256;

struct RowArgs {
  const void* src;      // dispatch: x [tokens]; combine: y [m]; combine_grad: y [m]
  long long ld_src;     // row pitches in bytes
  void* dst;            // dispatch: a [m]; combine: out [tokens]; combine_grad: dy [m] or NULL
  long long ld_dst;
  const void* dout;     // combine_grad: [tokens]
  long long ld_dout;
  const int* rows;      // [tokens, k], NULL = slot order
  const int* slots;     // [m], NULL = slot order
  const float* weights; // [tokens, k], NULL = 1
  float* dweights;      // combine_grad: [tokens, k] or NULL
  long long tokens, m;
  int k;
  long long width;      // accesses of a row
};

// The widest access of 16, 8, 4, 2 or 1 bytes that a call's rows allow, and how many of them, kRowThreads apart, a thread
// takes at a time: narrow ones leave the same bytes on their way. 8192 rows of 4095 bf16, 4 experts each: dispatch 103.5 us
// (one at a time 134), combine 82.9 (163), gradient 148.8 (210).
template <int Bytes>
using Access = std::conditional_t<Bytes == 16, uint4, std::conditional_t<Bytes == 8, uint2, std::conditional_t<Bytes == 4, uint32_t,
               std::conditional_t<Bytes == 2, uint16_t, uint8_t>>>>;
template <int Bytes>
constexpr int kPieces = Bytes >= 2 ? 16 / Bytes : 8;

// Rows of the layout that hold no slot become zeros: each part takes 32 rows, whose slots a warp looks up
// at once; a warp writes a row.
constexpr int kPadRows = 32;
template <class V>
__device__ __forceinline__ void zero_padding(const RowArgs& a, long long part) {
  const int lane = threadIdx.x % 32;
  const long long r0 = part * kPadRows, r = r0 + lane;
  const unsigned empty = __ballot_sync(0xFFFFFFFFu, r < a.m && a.slots[r] < 0);
  const long long bytes = a.width * (long long)sizeof(V);
  for (int i = threadIdx.x / 32; i < kPadRows; i += kRowThreads / 32) {
    if ((empty >> i & 1) == 0) continue;
    char* dst = static_cast<char*>(a.dst) + (r0 + i) * a.ld_dst;
    // Whole 16 bytes between the row's ends.
    const long long off = -reinterpret_cast<uintptr_t>(dst) & 15, head = off < bytes ? off : bytes;
    const long long body = (bytes - head) / 16, tail = head + body * 16;
    for (long long c = lane; c < body; c += 32) reinterpret_cast<uint4*>(dst + head)[c] = uint4{};
    if constexpr (sizeof(V) < 16) {  // less than 16 bytes each
      const long long c = lane * sizeof(V);
      if (c < head) *reinterpret_cast<V*>(dst + c) = V{};
      if (tail + c < bytes) *reinterpret_cast<V*>(dst + tail + c) = V{};
    }
  }
}

// A copy knows no element type. A token's row is read once and written to each of its experts.
template <int Bytes>
__global__ void __launch_bounds__(kRowThreads) dispatch_kernel(const RowArgs a) {
  using V = Access<Bytes>;
  constexpr int kAtOnce = kPieces<Bytes> > 2 ? kPieces<Bytes> : 2;  // 16 bytes: a row of 8 KB is one turn of the block
  griddep_wait();
  griddep_launch_dependents();
  if (blockIdx.x >= a.tokens) return zero_padding<V>(a, blockIdx.x - a.tokens);
  __shared__ int row[kMaxTopK];
  const long long t = blockIdx.x;
  const V* src = reinterpret_cast<const V*>(static_cast<const char*>(a.src) + t * a.ld_src);
  if (threadIdx.x < a.k) row[threadIdx.x] = a.rows[t * a.k + threadIdx.x];
  __syncthreads();
  for (long long c = threadIdx.x; c < a.width; c += kAtOnce * kRowThreads) {
    V v[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) v[i] = c + i * kRowThreads < a.width ? src[c + i * kRowThreads] : V{};
    for (int j = 0; j < a.k; ++j) {
      const long long r = row[j];
      if (r < 0 || r >= a.m) continue;
      V* dst = reinterpret_cast<V*>(static_cast<char*>(a.dst) + r * a.ld_dst);
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i)
        if (c + i * kRowThreads < a.width) dst[c + i * kRowThreads] = v[i];
    }
  }
}

// Cells of a row: accesses of so many bytes, elements of T.
template <class T, int Bytes>
struct Cells {
  static constexpr int n = Bytes / int(sizeof(T));
  using type = Access<Bytes>;
  static __device__ __forceinline__ void get(const type* p, float* v) {
    if constexpr (Bytes == 16) {
      unpack<T>(*p, v);
    } else {
      T e[n];
      memcpy(e, p, sizeof(e));
#pragma unroll
      for (int i = 0; i < n; ++i) v[i] = to_f32(e[i]);
    }
  }
  static __device__ __forceinline__ void put(type* p, const float* v) {
    if constexpr (Bytes == 16) {
      *p = pack<T>(v);
    } else {
      T e[n];
#pragma unroll
      for (int i = 0; i < n; ++i) e[i] = from_f32<T>(v[i]);
      type u;
      memcpy(&u, e, sizeof(u));
      *p = u;
    }
  }
};

__device__ __forceinline__ long long row_of(const RowArgs& a, long long slot) {
  const long long r = a.rows != nullptr ? a.rows[slot] : slot;
  return r >= 0 && r < a.m ? r : -1;
}

// A thread has its cells of a token's row and takes its slots four at a time, all their loads before the first sum.
template <class T, int Bytes>
__global__ void __launch_bounds__(kRowThreads) combine_kernel(const RowArgs a) {
  using C = Cells<T, Bytes>;
  using V = typename C::type;
  constexpr int kCells = kPieces<Bytes>;
  griddep_wait();
  griddep_launch_dependents();
  const long long t = blockIdx.x;
  const long long c = (long long)blockIdx.y * kRowThreads * kCells + threadIdx.x;
  if (c >= a.width) return;
  float sum[kCells][C::n] = {};
#pragma unroll 4
  for (int j = 0; j < a.k; ++j) {
    const long long r = row_of(a, t * a.k + j);
    if (r < 0) continue;
    const float w = a.weights != nullptr ? a.weights[t * a.k + j] : 1.0f;
    const V* src = reinterpret_cast<const V*>(static_cast<const char*>(a.src) + r * a.ld_src) + c;
    V y[kCells];
#pragma unroll
    for (int x = 0; x < kCells; ++x) y[x] = c + x * kRowThreads < a.width ? src[x * kRowThreads] : V{};
#pragma unroll
    for (int x = 0; x < kCells; ++x) {
      float v[C::n];
      C::get(&y[x], v);
#pragma unroll
      for (int i = 0; i < C::n; ++i) sum[x][i] += w * v[i];
    }
  }
  V* dst = reinterpret_cast<V*>(static_cast<char*>(a.dst) + t * a.ld_dst) + c;
#pragma unroll
  for (int x = 0; x < kCells; ++x)
    if (c + x * kRowThreads < a.width) C::put(dst + x * kRowThreads, sum[x]);
}

// dy and dw of one token: its dout is read once for kAtOnce slots at a time, each slot's y once. The slots' rows
// are looked up before the loop, and a turn's loads go out together.
constexpr int kAtOnce = 4;
template <class T, int Bytes>
__global__ void __launch_bounds__(kRowThreads) combine_grad_kernel(const RowArgs a) {
  using C = Cells<T, Bytes>;
  using V = typename C::type;
  constexpr int kCells = kPieces<Bytes>;
  __shared__ float red[kAtOnce][kRowThreads / 32];
  __shared__ long long row[kMaxTopK];
  __shared__ float weight[kMaxTopK];
  __shared__ bool writes[kMaxTopK];
  griddep_wait();
  griddep_launch_dependents();
  if (blockIdx.x >= a.tokens) return zero_padding<V>(a, blockIdx.x - a.tokens);
  const long long t = blockIdx.x;
  if (threadIdx.x < a.k) {
    const long long s = t * a.k + threadIdx.x, r = row_of(a, s);
    row[threadIdx.x] = r;
    weight[threadIdx.x] = a.weights != nullptr ? a.weights[s] : 1.0f;
    // A row's gradient, where it is wanted, is written by its own slot alone.
    writes[threadIdx.x] = r >= 0 && a.dst != nullptr && (a.slots == nullptr || a.slots[r] == s);
  }
  __syncthreads();
  const V* dout = reinterpret_cast<const V*>(static_cast<const char*>(a.dout) + t * a.ld_dout);
  for (int j0 = 0; j0 < a.k; j0 += kAtOnce) {
    float dot[kAtOnce] = {};
    for (long long c = threadIdx.x; c < a.width; c += kRowThreads * kCells) {
      V y[kAtOnce][kCells], d[kCells];
#pragma unroll
      for (int z = 0; z < kCells; ++z) d[z] = c + z * kRowThreads < a.width ? dout[c + z * kRowThreads] : V{};
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const bool reads = a.dweights != nullptr && j0 + i < a.k && row[j0 + i] >= 0;
        const V* src = reinterpret_cast<const V*>(static_cast<const char*>(a.src) + (reads ? row[j0 + i] : 0) * a.ld_src) + c;
#pragma unroll
        for (int z = 0; z < kCells; ++z) y[i][z] = reads && c + z * kRowThreads < a.width ? src[z * kRowThreads] : V{};
      }
      float g[kCells][C::n];
#pragma unroll
      for (int z = 0; z < kCells; ++z) C::get(&d[z], g[z]);
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        if (j0 + i >= a.k || row[j0 + i] < 0) continue;
        const float w = weight[j0 + i];
        V* dst = reinterpret_cast<V*>(static_cast<char*>(a.dst) + row[j0 + i] * a.ld_dst) + c;
#pragma unroll
        for (int z = 0; z < kCells; ++z) {
          float v[C::n];
          C::get(&y[i][z], v);
#pragma unroll
          for (int x = 0; x < C::n; ++x) dot[i] += g[z][x] * v[x];
          if (!writes[j0 + i] || c + z * kRowThreads >= a.width) continue;
#pragma unroll
          for (int x = 0; x < C::n; ++x) v[x] = w * g[z][x];
          C::put(dst + z * kRowThreads, v);
        }
      }
    }
    if (a.dweights == nullptr) continue;
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
#pragma unroll
      for (int o = 16; o > 0; o /= 2) dot[i] += __shfl_xor_sync(0xFFFFFFFFu, dot[i], o);
      if (threadIdx.x % 32 == 0) red[i][threadIdx.x / 32] = dot[i];
    }
    __syncthreads();
    if (threadIdx.x < kAtOnce && j0 + int(threadIdx.x) < a.k) {
      float s = 0.0f;
      for (int w = 0; w < kRowThreads / 32; ++w) s += red[threadIdx.x][w];
      a.dweights[t * a.k + j0 + threadIdx.x] = s;
    }
    __syncthreads();
  }
}

// Bytes that every one of the values is a multiple of: 16, 8, 4, 2 or 1.
int common_granule(std::initializer_list<uint64_t> values) {
  uint64_t all = 16;
  for (uint64_t v : values) all |= v;
  return int(all & (~all + 1));
}

int type_bytes(int32_t t) { return t == KL_F32 ? 4 : t == KL_BF16 || t == KL_F16 ? 2 : 0; }

kl_status check_rows(char const* who, int64_t tokens, int64_t k, int64_t m, int64_t width) {
  if (tokens < 0 || k < 1 || k > kMaxTopK || m < 0 || width < 0)
    return fail(KL_ERR_INVALID_ARGUMENT, std::string(who) + ": extents must not be negative, k in [1, 32]");
  if (tokens > INT32_MAX || m > INT32_MAX || tokens * k > INT32_MAX || tokens + (m + kPadRows - 1) / kPadRows > INT32_MAX)
    return fail(KL_ERR_INVALID_ARGUMENT, std::string(who) + ": more than 2^31 - 1 rows");
  return KL_OK;
}

}  // namespace
}  // namespace kl::capi

extern "C" int64_t kl_moe_rows(int64_t slots, int64_t experts, int32_t block) {
  if (slots < 0 || experts < 1 || (block != 128 && block != 256)) return -1;
  const int64_t holders = slots < experts ? slots : experts;
  return (slots + holders * (block - 1)) / block * block;
}

extern "C" kl_status kl_moe_plan(const int32_t* ids, int64_t tokens, int64_t k, int64_t experts, int32_t block, int64_t m,
                                 int32_t* rows, int32_t* slots, int32_t* m_block_group, void* stream) {
  using namespace kl::capi;
  kl_status s = check_rows("kl_moe_plan", tokens, k, m, 0);
  if (s != KL_OK) return s;
  if (experts < 1 || experts > kMaxExperts) return fail(KL_ERR_NOT_SUPPORTED, "kl_moe_plan: experts must be in [1, 1024]");
  if (block != 128 && block != 256) return fail(KL_ERR_INVALID_ARGUMENT, "kl_moe_plan: block must be 128 or 256");
  if (m % block != 0 || m < kl_moe_rows(tokens * k, experts, block))
    return fail(KL_ERR_INVALID_ARGUMENT, "kl_moe_plan: m must be a multiple of block, at least kl_moe_rows(tokens * k, experts, block)");
  if (m == 0) return KL_OK;
  if ((tokens > 0 && (ids == nullptr || rows == nullptr)) || slots == nullptr || m_block_group == nullptr)
    return fail(KL_ERR_INVALID_ARGUMENT, "kl_moe_plan: null pointer");
  if (!words_aligned({ids, rows, slots, m_block_group}))
    return fail(KL_ERR_INVALID_ARGUMENT, "kl_moe_plan: ids, rows, slots and m_block_group must be 4-byte aligned");
  PlanArgs a = {};
  a.ids = ids;
  a.total = tokens * k;
  a.experts = int(experts);
  a.block = block;
  a.m = m;
  a.rows = rows;
  a.slots = slots;
  a.blocks = m_block_group;
  // One block while a warp has one turn of 32 slots. One block against a cluster, 64 experts: 1024 slots 7.5 and
  // 7.7 us, 4096 slots 12.7 and 7.9, 8192 slots 19.5 and 7.8.
  const int cluster = a.total <= 32 * kPlanWarps ? 1 : kPlanBlocks;
  const long long warps = (long long)cluster * kPlanWarps;
  a.warp_span = (a.total + warps * 32 - 1) / (warps * 32) * 32;
  const size_t smem = size_t(kPlanWarps) * size_t(experts) * sizeof(int);
  void* args[] = {&a};
  cudaError_t e = launch_dependent(static_cast<cudaStream_t>(stream), dim3(unsigned(cluster)), kPlanThreads, smem, cluster,
             reinterpret_cast<void const*>(&plan_kernel), args);
  return e == cudaSuccess ? KL_OK : cuda_fail(e, "kl_moe_plan launch");
}

extern "C" kl_status kl_moe_dispatch(const void* x, int64_t ldx_bytes, int64_t tokens, int64_t row_bytes, int64_t k,
                                     const int32_t* rows, const int32_t* slots, int64_t m, void* a_out, int64_t lda_bytes,
                                     void* stream) {
  using namespace kl::capi;
  kl_status s = check_rows("kl_moe_dispatch", tokens, k, m, row_bytes);
  if (s != KL_OK) return s;
  if (m == 0 || row_bytes == 0) return KL_OK;
  if ((tokens > 0 && (x == nullptr || rows == nullptr)) || slots == nullptr || a_out == nullptr)
    return fail(KL_ERR_INVALID_ARGUMENT, "kl_moe_dispatch: null pointer");
  if (!words_aligned({rows, slots})) return fail(KL_ERR_INVALID_ARGUMENT, "kl_moe_dispatch: rows and slots must be 4-byte aligned");
  if (ldx_bytes < row_bytes || lda_bytes < row_bytes)
    return fail(KL_ERR_INVALID_ARGUMENT, "kl_moe_dispatch: row pitch below the row's bytes");
  RowArgs a = {};
  a.src = x;
  a.ld_src = ldx_bytes;
  a.dst = a_out;
  a.ld_dst = lda_bytes;
  a.rows = rows;
  a.slots = slots;
  a.tokens = tokens;
  a.m = m;
  a.k = int(k);
  const int g = common_granule({reinterpret_cast<uintptr_t>(x), reinterpret_cast<uintptr_t>(a_out), uint64_t(ldx_bytes),
                                uint64_t(lda_bytes), uint64_t(row_bytes)});
  a.width = row_bytes / g;
  void const* kernel = g == 16  ? reinterpret_cast<void const*>(&dispatch_kernel<16>)
                       : g == 8 ? reinterpret_cast<void const*>(&dispatch_kernel<8>)
                       : g == 4 ? reinterpret_cast<void const*>(&dispatch_kernel<4>)
                       : g == 2 ? reinterpret_cast<void const*>(&dispatch_kernel<2>)
                                : reinterpret_cast<void const*>(&dispatch_kernel<1>);
  void* args[] = {&a};
  cudaError_t e = launch_dependent(static_cast<cudaStream_t>(stream), dim3(unsigned(tokens + (m + kPadRows - 1) / kPadRows)),
                         kRowThreads, 0, 1, kernel, args);
  return e == cudaSuccess ? KL_OK : cuda_fail(e, "kl_moe_dispatch launch");
}

namespace kl::capi {
namespace {

// f(element, bytes of an access): at least an element's, whatever the granule of the rows' bytes allows.
template <class F>
void by_cells(int32_t type, int granule, F&& f) {
  auto by_bytes = [&](auto t) {
    if (granule >= 16) f(t, std::integral_constant<int, 16>{});
    else if (granule == 8) f(t, std::integral_constant<int, 8>{});
    else if (granule == 4 || sizeof(t) == 4) f(t, std::integral_constant<int, 4>{});
    else if constexpr (sizeof(t) == 2) f(t, std::integral_constant<int, 2>{});
  };
  if (type == KL_F32) by_bytes(float{});
  else if (type == KL_F16) by_bytes(__half{});
  else by_bytes(__nv_bfloat16{});
}

}  // namespace
}  // namespace kl::capi

extern "C" kl_status kl_moe_combine(const void* y, int32_t type, int64_t ldy, int64_t m, const int32_t* rows,
                                    const float* weights, int64_t tokens, int64_t k, int64_t width, void* out, int64_t ldo,
                                    void* stream) {
  using namespace kl::capi;
  kl_status s = check_rows("kl_moe_combine", tokens, k, m, width);
  if (s != KL_OK) return s;
  const int size = type_bytes(type);
  if (size == 0) return fail(KL_ERR_NOT_SUPPORTED, "kl_moe_combine: rows must be bf16, f16 or f32");
  if (tokens == 0 || width == 0) return KL_OK;
  if (ldy < width || ldo < width) return fail(KL_ERR_INVALID_ARGUMENT, "kl_moe_combine: row pitch below the width");
  if (rows == nullptr && m != tokens * k)
    return fail(KL_ERR_INVALID_ARGUMENT, "kl_moe_combine: without rows, y has tokens * k rows");
  if (out == nullptr || (m > 0 && y == nullptr)) return fail(KL_ERR_INVALID_ARGUMENT, "kl_moe_combine: null pointer");
  if (!aligned(y, size) || !aligned(out, size))
    return fail(KL_ERR_INVALID_ARGUMENT, "kl_moe_combine: y and out must be aligned to their elements");
  if (!words_aligned({rows, weights})) return fail(KL_ERR_INVALID_ARGUMENT, "kl_moe_combine: rows and weights must be 4-byte aligned");
  RowArgs a = {};
  a.src = y;
  a.ld_src = ldy * size;
  a.dst = out;
  a.ld_dst = ldo * size;
  a.rows = rows;
  a.weights = weights;
  a.tokens = tokens;
  a.m = m;
  a.k = int(k);
  const int g = common_granule({reinterpret_cast<uintptr_t>(y), reinterpret_cast<uintptr_t>(out), uint64_t(a.ld_src),
                                uint64_t(a.ld_dst), uint64_t(width * size)});
  a.width = width * size / g;
  const int64_t per_block = kRowThreads * (16 / g);  // accesses of a block: 4 KB
  const int64_t parts = (a.width + per_block - 1) / per_block;
  if (parts > 65535) return fail(KL_ERR_INVALID_ARGUMENT, "kl_moe_combine: rows too wide");
  cudaError_t e = cudaSuccess;
  by_cells(type, g, [&](auto t, auto v) {
    void* args[] = {&a};
    e = launch_dependent(static_cast<cudaStream_t>(stream), dim3(unsigned(tokens), unsigned(parts)), kRowThreads, 0, 1,
               reinterpret_cast<void const*>(&combine_kernel<decltype(t), decltype(v)::value>), args);
  });
  return e == cudaSuccess ? KL_OK : cuda_fail(e, "kl_moe_combine launch");
}

extern "C" kl_status kl_moe_combine_grad(const void* dout, int64_t ld_dout, const void* y, int32_t type, int64_t ldy, int64_t m,
                                         const int32_t* rows, const int32_t* slots, const float* weights, int64_t tokens,
                                         int64_t k, int64_t width, void* dy, int64_t ld_dy, float* dweights, void* stream) {
  using namespace kl::capi;
  kl_status s = check_rows("kl_moe_combine_grad", tokens, k, m, width);
  if (s != KL_OK) return s;
  const int size = type_bytes(type);
  if (size == 0) return fail(KL_ERR_NOT_SUPPORTED, "kl_moe_combine_grad: rows must be bf16, f16 or f32");
  if ((rows == nullptr) != (slots == nullptr))
    return fail(KL_ERR_INVALID_ARGUMENT, "kl_moe_combine_grad: rows and slots come together");
  if (rows == nullptr && m != tokens * k)
    return fail(KL_ERR_INVALID_ARGUMENT, "kl_moe_combine_grad: without rows, y has tokens * k rows");
  if (ldy < width || ld_dout < width || (dy != nullptr && ld_dy < width))
    return fail(KL_ERR_INVALID_ARGUMENT, "kl_moe_combine_grad: row pitch below the width");
  if (tokens == 0 && (m == 0 || dy == nullptr)) return KL_OK;
  if ((tokens > 0 && width > 0 && dout == nullptr) ||
      (m > 0 && width > 0 && ((dy == nullptr && dweights == nullptr) || (dweights != nullptr && y == nullptr))))
    return fail(KL_ERR_INVALID_ARGUMENT, "kl_moe_combine_grad: null pointer");
  if (!aligned(dout, size) || !aligned(y, size) || !aligned(dy, size))
    return fail(KL_ERR_INVALID_ARGUMENT, "kl_moe_combine_grad: dout, y and dy must be aligned to their elements");
  if (!words_aligned({rows, slots, weights, dweights}))
    return fail(KL_ERR_INVALID_ARGUMENT, "kl_moe_combine_grad: rows, slots, weights and dweights must be 4-byte aligned");
  RowArgs a = {};
  a.src = y;
  a.ld_src = ldy * size;
  a.dst = dy;
  a.ld_dst = ld_dy * size;
  a.dout = dout;
  a.ld_dout = ld_dout * size;
  a.rows = rows;
  a.slots = slots;
  a.weights = weights;
  a.dweights = dweights;
  a.tokens = tokens;
  a.m = m;
  a.k = int(k);
  const int g = common_granule({reinterpret_cast<uintptr_t>(y), reinterpret_cast<uintptr_t>(dy), reinterpret_cast<uintptr_t>(dout),
                                uint64_t(a.ld_src), uint64_t(a.ld_dst), uint64_t(a.ld_dout), uint64_t(width * size)});
  a.width = width * size / g;
  const int64_t pad_parts = slots != nullptr && dy != nullptr ? (m + kPadRows - 1) / kPadRows : 0;
  cudaError_t e = cudaSuccess;
  by_cells(type, g, [&](auto t, auto v) {
    void* args[] = {&a};
    e = launch_dependent(static_cast<cudaStream_t>(stream), dim3(unsigned(tokens + pad_parts)), kRowThreads, 0, 1,
               reinterpret_cast<void const*>(&combine_grad_kernel<decltype(t), decltype(v)::value>), args);
  });
  return e == cudaSuccess ? KL_OK : cuda_fail(e, "kl_moe_combine_grad launch");
}
