// Products with 4-bit weights and group scales for few tokens (kl_gemv_int4):
//   out[t, n] = sum_g s[n, g] sum_{i in g} (q[n, i] - z[n, g]) x[t, i],
// with one matrix, or one per expert and the expert of every (token, slot) in `ids`.
//
// The weights' bytes should bound it, so a code may cost little: at 6.5 TB/s an SM gets 46 codes a cycle and has 128
// lanes' instructions for them.
//
// One and two tokens. As unsigned bytes eight codes cost three instructions (two masks and a shift), so the products are
// integer ones (mma.sync.m16n8k32, u8 x s8 -> s32): every block first writes x as fixed-point numbers X = round(x 2^e),
// |X| <= 2^30, one e for 128 K-elements of a token, in four signed digits of 8 bits, x = 2^-e (d_0 + 256 d_1 + ...) + r.
// The sums of a scale group are exact: P_c = sum q d_c, and P_c - z D_c, D_c = sum d_c, takes the zero point off without
// cancellation. Only then come fp32 and the scales: sum over the 128s of 2^-e sum_g s 256^c (P_c - z D_c).
// A rest r is left where an element lies far below the largest of its 128 (2^-22 of it in bf16; in f16 only beside one of
// 64 and more). It may be all that counts, where the large one meets a code equal to its zero point, so 128s with a rest
// are marked, and r, which x's type holds exactly, is multiplied as below and added. One of 28000 128s of normal bf16
// values has a rest, one of 1000 of gated ones; three digits would leave one in 120 and 7 of them, in f16 15 and 1.7.
// 28672 x 8192, one token: 24.3 us for normal and for gated values, 125 with a rest in every 128.
//
// More tokens, 8 or 16 at a time. Four digits of 8 tokens would be four products and a longer sum, so here the
// codes become q - z in x's type, exactly (eleven instructions for eight codes in bf16, nine in f16), and the products are
// x's own (mma.sync.m16n8k16, sums in fp32); a group's sum is scaled once. Three digits took 44 us for 8 tokens of
// 28672 x 8192 and 83 for 16; this takes 42 and 60.
//
// Layout: a block per SM, 16 warps, each with its own ring of TMA loads (units of 16 rows x 512
// codes, two boxes of 128 bytes a row), refilled as soon as a slot has been read, so that no warp waits for another
// while the weights stream. ldmatrix hands a lane eight codes of a row at a time. Where x for all of K
// would crowd out the ring, a cluster of 2, 4 or 8 blocks splits K and adds up through distributed
// shared memory.
//
// Measured, bf16, groups of 128: 28672 x 8192 with one token 24.3 us (5.0 TB/s; 6.9 while it streams, 6 us before the first
// unit and 2 after the last), 2 tokens 25.7, 8 tokens 42, 16 tokens 60 (instruction issue, four warps a scheduler); groups
// of 32 with zero points, one token 38 (a scale, a zero point and a sum every 32 codes); 4096 x 4096, one token 6.8.

#include <cooperative_groups.h>
#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <exception>
#include <string>

#include <kl/arch/cluster.hpp>
#include <kl/arch/griddep.hpp>
#include <kl/arch/mbarrier.hpp>
#include <kl/arch/tma.hpp>
#include <kl/gemm/gemm.hpp>
#include <kl_gemm.h>

#include "kl_experts.cuh"
#include "kl_internal.cuh"
#include "kl_vec.cuh"

namespace cg = cooperative_groups;

namespace kl::capi {
namespace {

constexpr int kWarps = 16;
constexpr int kThreads = 32 * kWarps;
constexpr int kRows = 16;              // weight rows of a tile
constexpr int kBoxBytes = kRows * 128;
constexpr int kMaxSlots = 4096;        // (token, expert) pairs of a call with ids
constexpr int kMaxK = 65536;
constexpr int kSmemLimit = 226 * 1024; // dynamic; 227 KB less the static arrays

struct Int4Args {
  CUtensorMap map;  // q as bytes [experts, n, k / 2]
  const void* x;
  long long ldx;
  const void* scales;
  int lds;
  long long stride_s;
  const uint8_t* zeros;
  int ldz;
  long long stride_z;
  const int* ids;
  int experts, slots, x_div;  // slots: rows of out; x row = slot / x_div
  void* out;
  long long ldo;
  int n, k, group;
  int f32_scales, f32_out;
  int tiles;  // 16-row tiles of one matrix
  int depth;  // slots of a warp's ring
  uint32_t x_at, sums, powers, rests, pieces, block, records, bars, lists;  // offsets in shared memory
  int wide_scales;                                      // a lane's scales and zero points come by one load
  int group_span, last_group;                           // 128-element runs of a group (groups of 128 and more); index of the last
  int* status;
  unsigned long long timeout_ns;
};

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

// d = a b (+ d, unless `first`, a constant where it is called)
__device__ __forceinline__ void mma_u8s8(int (&d)[4], const uint32_t (&a)[4], uint2 b, bool first) {
  if (first)
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y), "r"(0));
  else
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y));
}

template <class T>
__device__ __forceinline__ void mma_16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, bool first) {
  constexpr bool kBf16 = std::is_same_v<T, __nv_bfloat16>;
#define KL_MMA(TYPE)                                                                                                  \
  if (first)                                                                                                          \
    asm("mma.sync.aligned.m16n8k16.row.col.f32." TYPE "." TYPE                                                        \
        ".f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"                                    \
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])                                                              \
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));                                   \
  else                                                                                                                \
    asm("mma.sync.aligned.m16n8k16.row.col.f32." TYPE "." TYPE                                                        \
        ".f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"                                        \
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])                                                              \
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1))
  if constexpr (kBf16) {
    KL_MMA("bf16");
  } else {
    KL_MMA("f16");
  }
#undef KL_MMA
}

// Zero point z (z2: with 16 bits a value) as the unpacking below takes it off, and codes - z of a word's eight codes,
// exactly, in pairs (0, 4), (1, 5), (2, 6), (3, 7). A code's bits below those of 128 (bf16) or 1024 (f16) make 128 + q
// or 1024 + q; f16 has room for 1024 + 16 q too, which spares shifts.
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t mask, uint32_t bits) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(a), "r"(mask), "r"(bits));
  return r;
}
__device__ __forceinline__ uint32_t fma_bf16(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
__device__ __forceinline__ uint32_t fma_f16(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
template <class T>
__device__ __forceinline__ uint32_t pack_two(float v) {
  const T b = from_f32<T>(v);
  uint16_t u;
  memcpy(&u, &b, 2);
  return u * 0x10001u;
}
// A constant that stays in its register: else the compiler makes it anew for every use, at an instruction each.
__device__ __forceinline__ uint32_t held(uint32_t v) {
  uint32_t r;
  asm volatile("mov.b32 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
template <class T>
struct Codes;
template <>
struct Codes<__nv_bfloat16> {
  uint32_t mask = held(0x000F000Fu), bits = held(0x43004300u), one = held(0x3F803F80u);
  struct Zero {
    uint32_t z;  // -(128 + z)
  };
  __device__ __forceinline__ Zero zero(uint32_t z2) const { return {0xC300C300u | z2}; }
  __device__ __forceinline__ void minus(uint32_t w, Zero z, uint32_t (&r)[4]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = fma_bf16(and_or(w >> 4 * i, mask, bits), one, z.z);
  }
};
template <>
struct Codes<__half> {
  uint32_t mask = held(0x000F000Fu), mask16 = held(0x00F000F0u), bits = held(0x64006400u), one = held(0x3C003C00u),
           sixteenth = held(0x2C002C00u);
  struct Zero {
    uint32_t z, z16;  // -(1024 + z), -(64 + z)
  };
  __device__ __forceinline__ Zero zero(uint32_t z2) const { return {0xE400E400u | z2, fma_f16(0xE400E400u | z2, one, 0x63806380u)}; }
  __device__ __forceinline__ void minus(uint32_t w, Zero z, uint32_t (&r)[4]) const {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t v = w >> 8 * i;
      r[2 * i] = fma_f16(and_or(v, mask, bits), one, z.z);
      r[2 * i + 1] = fma_f16(and_or(v, mask16, bits), sixteenth, z.z16);
    }
  }
};

// 32 codes - z of rows g and g + 8 as the A operands of two products in x's type.
template <class T, bool kZeros>
struct CodesOf32 {
  // bf16 has 128 + z for z up to 127; what is above goes into a product of its own.
  static constexpr uint32_t kMaxZ = std::is_same_v<T, __nv_bfloat16> ? 127 : 255;
  uint32_t low[4], high[4];
  uint32_t z[2];
  bool more = false;
  __device__ __forceinline__ CodesOf32(Codes<T> const& codes, uint32_t w0, uint32_t w1, const uint32_t (&zero)[2]) : z{zero[0], zero[1]} {
    const auto z0 = codes.zero(kZeros ? min(z[0], kMaxZ) * 0x10001u : 0x00080008u);
    const auto z1 = codes.zero(kZeros ? min(z[1], kMaxZ) * 0x10001u : 0x00080008u);
    uint32_t f0[4], f1[4];
    codes.minus(w0, z0, f0);
    codes.minus(w1, z1, f1);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      low[2 * i] = f0[i];
      low[2 * i + 1] = f1[i];
      high[2 * i] = f0[2 + i];
      high[2 * i + 1] = f1[2 + i];
    }
    if (kZeros && kMaxZ < 255) more = __any_sync(0xFFFFFFFFu, max(z[0], z[1]) > kMaxZ);
  }
  // dot = or += the products with eight tokens' 32 elements of x.
  __device__ __forceinline__ void times(float (&dot)[4], uint4 x, bool first) const {
    mma_16<T>(dot, low, x.x, x.y, first);
    mma_16<T>(dot, high, x.z, x.w, false);
    if (more) {
      uint32_t rest[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) rest[r] = pack_two<T>(-float(max(z[r], kMaxZ) - kMaxZ));
      const uint32_t fr[4] = {rest[0], rest[1], rest[0], rest[1]};
      mma_16<T>(dot, fr, x.x, x.y, false);
      mma_16<T>(dot, fr, x.z, x.w, false);
    }
  }
};

// With ids: the experts that some slot names, each with its slots, in shared memory.
struct Lists {
  int* base;        // [experts + 1]: token passes before an active expert
  uint16_t* act;    // [experts]: its number
  uint16_t* start;  // [experts + 1]: its first entry of `list`
  uint16_t* list;   // [slots]
  static __host__ __device__ size_t bytes(int experts, int slots) {
    return (size_t(experts) + 1) * 4 + (size_t(experts) + 1) * 4 + size_t(slots) * 2;
  }
};

// Counts the slots of every expert, packs the active ones and files the slots in their order: every block builds the
// lists for itself, and all have to cut an expert's slots into the same passes.
template <int TOK>
__device__ void build_lists(const Int4Args& a, Lists const& l, int* hist, int* active_out) {
  __shared__ unsigned long long warp_sum[kWarps];
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  for (int e = tid; e < a.experts; e += kThreads) hist[e] = 0;
  __syncthreads();
  for (int s = tid; s < a.slots; s += kThreads) {
    const int e = a.ids[s];
    if (e >= 0 && e < a.experts) atomicAdd(&hist[e], 1);
  }
  __syncthreads();
  // Exclusive sums over the experts, two to a thread: active experts (bits 0-15), slots (16-31), passes (32-).
  unsigned long long mine = 0, own[2];
  int count[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int e = 2 * tid + i;
    count[i] = e < a.experts ? hist[e] : 0;
    own[i] = count[i] == 0 ? 0
                           : 1ull | (unsigned long long)count[i] << 16 |
                                 (unsigned long long)((count[i] + TOK - 1) / TOK) << 32;
    mine += own[i];
  }
  unsigned long long sum = mine;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const unsigned long long u = __shfl_up_sync(0xFFFFFFFFu, sum, o);
    if (lane >= o) sum += u;
  }
  if (lane == 31) warp_sum[warp] = sum;
  __syncthreads();
  unsigned long long before = sum - mine, total = 0;
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += warp_sum[w];
    total += warp_sum[w];
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int e = 2 * tid + i;
    if (count[i] > 0) {
      const int at = int(before & 0xFFFF), first = int(before >> 16 & 0xFFFF);
      l.act[at] = uint16_t(e);
      l.start[at] = uint16_t(first);
      l.base[at] = int(before >> 32);
      hist[e] = first;
    }
    before += own[i];
  }
  const int active = int(total & 0xFFFF);
  if (tid == 0) {
    l.start[active] = uint16_t(total >> 16 & 0xFFFF);
    l.base[active] = int(total >> 32);
  }
  __syncthreads();
  if (warp == 0)
    for (int s0 = 0; s0 < a.slots; s0 += 32) {
      const int s = s0 + lane;
      int e = s < a.slots ? a.ids[s] : -1;
      if (e < 0 || e >= a.experts) e = -1;
      const unsigned same = __match_any_sync(0xFFFFFFFFu, e);
      if (e >= 0) l.list[hist[e] + __popc(same & ((1u << lane) - 1))] = uint16_t(s);
      __syncwarp();
      if (e >= 0 && lane == __ffs(same) - 1) hist[e] += __popc(same);
      __syncwarp();
    }
  __syncthreads();
  *active_out = active;
}

// TOK: tokens of a pass, 1, 2, 8 or 16. Up to two go by the integer products: four digits of two tokens fill one
// 8-column tile, digit c of token i in column 2 c + i, and the digits meet by shuffles. 8 and 16 would take four and eight
// tiles; with them the codes are turned into x's type and each 8 tokens are one tile.
template <int TOK>
constexpr bool kDigits = TOK <= 2;

// Codes of a unit's row: two boxes' worth; with 16 tokens, whose x and sums leave the ring less room, one (16 tokens of
// 28672 x 8192: 80 us with two boxes, 60 with one; 8 tokens 42.6 and 43.5).
template <int TOK>
constexpr int kUnitK = TOK <= 8 ? 512 : 256;
template <int TOK>
constexpr int kUnitBytes = kRows * kUnitK<TOK> / 2;

// x in shared memory, by 32 K-elements. Digits: a row of 32 bytes for each column that is used, and 16 bytes between, so
// that the lanes that write them meet other banks (without, 4096 x 4096 with one token 6.9 us instead of 6.8); sums D of a scale
// group, an int a column; powers 2^-e of 128 elements, times 256^c, a float a column; rests, a byte a token and 128
// elements: not 0 where some r is not. Else: 64 bytes a token, every eight
// elements in the order of the codes' pairs.
template <int TOK>
constexpr int kXRow = kDigits<TOK> ? TOK * 128 + 16 : TOK * 64;  // bytes of 32 K-elements
template <int TOK>
constexpr int kSumBytes = kDigits<TOK> ? 32 : 0;  // of a group
template <int TOK>
constexpr int kPowerBytes = kDigits<TOK> ? 32 : 0;  // of 128 K-elements
template <int TOK>
constexpr int kRestBytes = kDigits<TOK> ? 8 : 0;  // of a unit
template <int NG, int TOK>
constexpr int kXBytes = kUnitK<TOK> / 32 * kXRow<TOK> + NG * kSumBytes<TOK> + kUnitK<TOK> / 128 * kPowerBytes<TOK> + kRestBytes<TOK>;  // of a unit

constexpr int kPieces = 2;  // tiles that a warp's run of units can touch
template <int TOK>
constexpr int kPiece = TOK * kRows;  // floats of a tile's sums

// A stretch: a warp's share of one tile, consecutive units of K. Its record lies with the ring slot of its first
// unit.
struct __align__(16) Stretch {
  int row0, kb, units, flags;  // kb: of this block's K
  int batch_row0, count, pass, expert;
};
constexpr int kEnd = 1;     // the last of the warp's run in the batch
constexpr int kSecond = 2;  // the run's second
constexpr int kNone = 4;    // the warp has no unit in this batch: a slot without loads

// Shared memory, in order: rings, x with its sums and powers, pieces, the block's sums, stretch records, barriers,
// lists.
template <int NG, int TOK>
size_t lay_out(Int4Args& a, int depth, int units, int cluster) {
  a.depth = depth;
  size_t at = size_t(kWarps) * depth * kUnitBytes<TOK>;
  auto take = [&](uint32_t& offset, size_t bytes) {
    offset = uint32_t(at);
    at += bytes;
  };
  take(a.x_at, size_t(units) * (kUnitK<TOK> / 32) * kXRow<TOK>);
  take(a.sums, size_t(units) * NG * kSumBytes<TOK>);
  take(a.powers, size_t(units) * (kUnitK<TOK> / 128) * kPowerBytes<TOK>);
  take(a.rests, (size_t(units) * kRestBytes<TOK> + 15) / 16 * 16);
  take(a.pieces, size_t(kWarps) * kPieces * kPiece<TOK> * 4);
  take(a.block, cluster > 1 ? size_t(2) * kWarps * kPiece<TOK> * 4 : 0);
  take(a.records, size_t(kWarps) * depth * sizeof(Stretch));
  take(a.bars, size_t(kWarps) * depth * 8);
  take(a.lists, a.ids != nullptr ? Lists::bytes(a.experts, a.slots) : 0);
  return at + 1024;  // the base is rounded up to 1024
}

// NG: scale groups of a unit (a group of more than 128 counts for every 128).
template <class T, int NG, int TOK, bool kZeros>
__global__ void __launch_bounds__(kThreads, 1) gemv_int4_kernel(const __grid_constant__ Int4Args a) {
  constexpr int kPerGroup = kUnitK<TOK> / 32 / NG;  // 32-code chunks of a group
  constexpr int kHeld = NG >= 4 ? NG / 4 : 1;       // scales that a lane holds of each of its rows
  constexpr int kHalves = kUnitK<TOK> / 256;
  constexpr uint32_t kNibbles = 0x0F0F0F0Fu;
  extern __shared__ uint8_t dynamic[];
  uint8_t* smem = dynamic + (1024 - smem_addr(dynamic) % 1024) % 1024;  // still known to be shared memory
  cg::cluster_group cluster = cg::this_cluster();
  const int split = int(cluster.block_rank()), splits = int(cluster.num_blocks());
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  const int depth = a.depth;
  const uint32_t bar0 = smem_addr(smem + a.bars) + warp * depth * 8;
  const uint32_t ring0 = smem_addr(smem) + warp * depth * kUnitBytes<TOK>;
  Stretch* records = reinterpret_cast<Stretch*>(smem + a.records) + warp * depth;
  float* pieces = reinterpret_cast<float*>(smem + a.pieces);
  if (lane == 0) {
    for (int i = 0; i < depth; ++i) mbarrier_init(bar0 + 8 * i, 1);
    fence_barrier_init();
    if (warp == 0) tma_prefetch_map(&a.map);
  }
  Lists l;
  l.base = reinterpret_cast<int*>(smem + a.lists);
  l.act = reinterpret_cast<uint16_t*>(l.base + a.experts + 1);
  l.start = l.act + a.experts;
  l.list = l.start + a.experts + 1;
  // Nothing of global memory is touched before the kernels before this one are done; for one matrix the
  // schedule is worked out in their shadow.
  int passes = (a.slots + TOK - 1) / TOK, active = 0;
  if (a.ids != nullptr) {
    griddep_wait();
    build_lists<TOK>(a, l, reinterpret_cast<int*>(smem + a.x_at), &active);
    passes = l.base[active];
  }
  // The tokens and the matrix of a pass.
  struct Pass {
    int expert, first, count;
  };
  auto pass_of = [&](int pass) {
    Pass p;
    if (a.ids == nullptr) {
      p.expert = 0;
      p.first = pass * TOK;
      p.count = a.slots - p.first;
    } else {
      int lo = 0, hi = active;  // the last active expert whose base is not above `pass`
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (l.base[mid] <= pass) lo = mid;
        else hi = mid;
      }
      p.expert = l.act[lo];
      p.first = l.start[lo] + (pass - l.base[lo]) * TOK;
      p.count = l.start[lo + 1] - p.first;
    }
    if (p.count > TOK) p.count = TOK;
    return p;
  };
  auto slot_of = [&](int i) { return a.ids == nullptr ? i : int(l.list[i]); };
  auto row_of = [&](Pass const& p, int token) {  // of x
    return static_cast<const T*>(a.x) + (long long)(a.x_div == 1 ? slot_of(p.first + token) : slot_of(p.first + token) / a.x_div) * a.ldx;
  };

  // This block's share of K, in units, and its cluster's tiles of all passes' tiles: the `remaining` ones from
  // tile `first` of pass `pass`. They go in batches of up to 16 of one pass. A batch's units (tile, 512 or 256 codes of this
  // block's K) are dealt to the warps in even, consecutive runs, so a run touches at most two tiles:
  // count kbs w / 16 units lie before warp w's, which begin in tile count w / 16.
  const int kb_all = (a.k + kUnitK<TOK> - 1) / kUnitK<TOK>;
  const int kb0 = kb_all * split / splits, kbs = kb_all * (split + 1) / splits - kb0;
  const uint32_t clusters = gridDim.x / splits, c0 = blockIdx.x / splits, all = uint32_t(passes) * a.tiles;
  const uint32_t share = all / clusters, extra = all % clusters, begin0 = c0 * share + min(c0, extra);
  int remaining = int(share + (c0 < extra)), pass = int(begin0 / a.tiles), first = int(begin0 - pass * a.tiles);
  int count = 0, run_left = 0, tile = 0, kb = 0, expert = -1, left = 0;  // run_left: units of the run behind the stretch
  int load_x = 0, load_y = 0;
  bool failed = false;

  // Begins the warp's next stretch in ring slot `at`.
  const int scale_bytes = a.f32_scales ? 4 : 2;
  auto begin_stretch = [&](int at) {
    Stretch s;
    s.flags = 0;
    if (run_left > 0) {
      kb = 0;
      ++tile;
      left = run_left;
      s.flags = kSecond;
    } else {  // the next batch
      first += count;
      remaining -= count;
      const bool turn = first == a.tiles;
      if (turn) {
        first = 0;
        ++pass;
      }
      if (turn || expert < 0) {
        // x of a pass is on its way to L2 before the weights' queue to memory fills: loads behind it take
        // microseconds.
        const Pass p = pass_of(pass);
        expert = p.expert;
        // A token has 16 / TOK warps.
        constexpr int kTokenWarps = TOK < kWarps ? kWarps / TOK : 1;
        const int token = warp / kTokenWarps;
        if (token < p.count) {
          const char* x = reinterpret_cast<const char*>(row_of(p, token) + kb0 * kUnitK<TOK>);
          const int bytes = min(a.k - kb0 * kUnitK<TOK>, kbs * kUnitK<TOK>) * 2;
          for (int i = (warp % kTokenWarps * 32 + lane) * 128; i < bytes; i += kTokenWarps * 32 * 128)
            asm volatile("prefetch.global.L2 [%0];" ::"l"(x + i));
        }
      }
      count = min(kWarps, min(a.tiles - first, remaining));
      const int begin = count * kbs * warp / kWarps;
      run_left = count * kbs * (warp + 1) / kWarps - begin;
      tile = count * warp / kWarps;
      kb = begin - tile * kbs;
      left = min(run_left, kbs - kb);
      if (run_left > 0) {  // likewise the scales and zero points, a row of two tiles to a lane
        const int row = min((first + tile) * kRows + lane, a.n - 1), g0 = kb0 * NG / a.group_span;
        const int groups = min((kb0 + kbs) * NG / a.group_span, a.last_group + 1) - g0;
        const char* x = static_cast<const char*>(a.scales) + (expert * a.stride_s + (long long)row * a.lds + g0) * scale_bytes;
        for (int i = 0; i < groups * scale_bytes; i += 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(x + i));
        if (kZeros) {
          const uint8_t* z = a.zeros + expert * a.stride_z + (long long)row * a.ldz + g0;
          for (int i = 0; i < groups; i += 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(z + i));
        }
      } else {
        s.flags = kNone;
      }
    }
    run_left -= left;
    if (run_left == 0) s.flags |= kEnd;
    load_x = (kb0 + kb) * (kUnitK<TOK> / 2);
    load_y = (first + tile) * kRows;
    s.row0 = load_y;
    s.kb = kb;
    s.units = left;
    s.batch_row0 = first * kRows;
    s.count = count;
    s.pass = pass;
    s.expert = expert;
    if (lane == 0) records[at] = s;
  };
  // Fills ring slot `at` with the warp's next unit.
  auto produce = [&](int at) {
    const uint32_t bar = bar0 + 8 * at, to = ring0 + at * kUnitBytes<TOK>;
    if (left == 0) {
      begin_stretch(at);
      if (left == 0) {  // nothing to load: the slot's barrier goes on to its next phase all the same
        if (lane == 0) mbarrier_arrive(bar);
        return;
      }
    }
    --left;
    if (lane == 0) {
      if (failed) {
        mbarrier_arrive(bar);
      } else {
        mbarrier_arrive_expect_tx(bar, kUnitBytes<TOK>);
#pragma unroll
        for (int i = 0; i < kHalves; ++i)  // zeros behind K
          tma_load_3d(to + i * kBoxBytes, &a.map, bar, load_x + i * 128, load_y, expert);
      }
    }
    load_x += kUnitK<TOK> / 2;
  };

  // x of a pass into shared memory: a warp takes 256 K-elements of a token at a time, a lane 8 of them, and loads
  // the next piece before it works on one.
  int x_token = 0, x_half = 0;  // of the piece that is loaded; halves of a unit: kbs * kHalves a token
  uint4 x_piece = make_uint4(0, 0, 0, 0);
  auto fetch = [&](Pass const& p) {
    while (x_half >= kbs * kHalves) {
      x_half -= kbs * kHalves;
      ++x_token;
    }
    const int k = (kb0 * kHalves + x_half) * 256 + lane * 8;
    if (x_token < p.count)
      x_piece = k < a.k ? *reinterpret_cast<const uint4*>(row_of(p, x_token) + k) : make_uint4(0, 0, 0, 0);
  };
  auto begin_x = [&](Pass const& p) {
    x_token = 0;
    x_half = warp;
    fetch(p);
  };
  bool marked = false;  // a 128 that this warp wrote has a rest; after the pass's barrier, one of the block's
  auto convert = [&](Pass const& p) {
    marked = false;
    constexpr int kLanes = kUnitK<TOK> / NG / 8;  // lanes of a scale group
#pragma unroll 1
    while (x_token < p.count) {
      const int token = x_token, half = x_half;
      const uint4 u = x_piece;
      x_half += kWarps;
      fetch(p);
      uint8_t* to = smem + a.x_at + (half * 8 + lane / 4) * kXRow<TOK>;
      if constexpr (!kDigits<TOK>) {
        *reinterpret_cast<uint4*>(to + token * 64 + lane % 4 * 16) =
            make_uint4(__byte_perm(u.x, u.z, 0x5410), __byte_perm(u.x, u.z, 0x7632), __byte_perm(u.y, u.w, 0x5410), __byte_perm(u.y, u.w, 0x7632));
        continue;
      }
      // The largest |x|: both types order like their bits, with NaN above infinity.
      uint32_t m = __vmaxu2(__vmaxu2(u.x & 0x7FFF7FFFu, u.y & 0x7FFF7FFFu), __vmaxu2(u.z & 0x7FFF7FFFu, u.w & 0x7FFF7FFFu));
#pragma unroll
      for (int o = 8; o > 0; o /= 2) m = __vmaxu2(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
      const uint16_t top16 = uint16_t(max(m & 0xFFFFu, m >> 16));
      T top_t;
      memcpy(&top_t, &top16, 2);
      const float top = to_f32(top_t);
      const bool bad = !(top < INFINITY);  // an infinity or a NaN makes the token's results NaN
      // Largest |X| in [2^29, 2^30]; below 2^-97 the steps stay at 2^-126.
      const int e = min(29 + 127 - int(__float_as_uint(top) >> 23), 126);
      const float up = bad ? 0.0f : __int_as_float((e + 127) << 23), down = __int_as_float((127 - e) << 23);
      float v[8];
      unpack<T>(u, v);
      // Adding 0x80 to each byte and flipping its top bit leaves X's digits, each in [-128, 127], in four bytes. Of an
      // element whose last place is 2^-e or more nothing is left (f16 has none below 2^-24); 2 bits - 1 orders the others by
      // size, with zeros behind them.
      constexpr bool kBf16 = std::is_same_v<T, __nv_bfloat16>;
      const uint32_t whole = bad || (!kBf16 && e >= 24) ? 0 : (uint32_t(127 + (kBf16 ? 7 : 10) - e) << 24) - 1;
      uint32_t y[8], least = 0xFFFFFFFFu;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        least = min(least, 2 * __float_as_uint(v[j]) - 1);
        y[j] = (uint32_t(__float2int_rn((bad ? 0.0f : v[j]) * up)) + 0x80808080u) ^ 0x80808080u;
      }
      const unsigned rests = __ballot_sync(0xFFFFFFFFu, least < whole);
      marked |= rests != 0;
      // By digit, the even elements (low nibbles) before the odd ones, as the masks leave the codes.
      uint2 d[4];
#pragma unroll
      for (int odd = 0; odd < 2; ++odd) {
        const uint32_t a01 = __byte_perm(y[odd], y[odd + 2], 0x5140), b01 = __byte_perm(y[odd + 4], y[odd + 6], 0x5140);
        const uint32_t a23 = __byte_perm(y[odd], y[odd + 2], 0x7362), b23 = __byte_perm(y[odd + 4], y[odd + 6], 0x7362);
        (odd ? d[0].y : d[0].x) = __byte_perm(a01, b01, 0x5410);
        (odd ? d[1].y : d[1].x) = __byte_perm(a01, b01, 0x7632);
        (odd ? d[2].y : d[2].x) = __byte_perm(a23, b23, 0x5410);
        (odd ? d[3].y : d[3].x) = __byte_perm(a23, b23, 0x7632);
      }
      int sum[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) sum[c] = __dp4a(int(d[c].x), 0x01010101, __dp4a(int(d[c].y), 0x01010101, 0));
      int low = sum[0] + sum[1] * 65536, high = sum[2] + sum[3] * 65536;
#pragma unroll
      for (int o = kLanes / 2; o > 0; o /= 2) {
        low += __shfl_xor_sync(0xFFFFFFFFu, low, o);
        high += __shfl_xor_sync(0xFFFFFFFFu, high, o);
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) *reinterpret_cast<uint2*>(to + (c * TOK + token) * 32 + lane % 4 * 8) = d[c];
      const int s0 = int(int16_t(low)), s1 = (low - s0) >> 16, s2 = int(int16_t(high)), s3 = (high - s2) >> 16;
      if (lane % kLanes == 0) {
        int* f = reinterpret_cast<int*>(smem + a.sums + (half * (32 / kLanes) + lane / kLanes) * kSumBytes<TOK>) + token;
        f[0] = s0;
        f[2] = s1;
        f[4] = s2;
        f[6] = s3;
      }
      if (lane % 16 == 0) {
        const float step = bad ? NAN : down;
        float* f = reinterpret_cast<float*>(smem + a.powers + (half * 2 + lane / 16) * kPowerBytes<TOK>) + token;
        f[0] = step;
        f[2] = step * 256.0f;
        f[4] = step * 65536.0f;
        f[6] = step * 16777216.0f;
        smem[a.rests + (half * 2 + lane / 16) * 2 + token] = (rests >> (lane & 16) & 0xFFFFu) != 0;
      }
    }
  };

  // A unit's scales and zero points, loaded one unit ahead: lane t of a row's four holds kHeld groups from t kHeld.
  // Rows behind the matrix and groups behind K read the last ones: the first are not stored, the second multiply
  // zeros. Where the layout allows, a lane's groups come by one load (one token of 28672 x 8192 with zero points, groups
  // of 32: 38.2 us, else 47.7; groups of 64: 31.7 and 34.4).
  struct __align__(16) Scales {
    uint32_t s[2][kHeld];  // as loaded: nothing waits for them before the unit that uses them
    uint32_t z[2][kHeld];
  };
  const char* s_row[2] = {};
  const uint8_t* z_row[2] = {};
  int s_kb = 0;  // the unit whose scales are loaded next
  Scales raw = {};
  auto aim_scales = [&](Stretch const& s) {
    s_kb = kb0 + s.kb;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = min(s.row0 + r * 8 + g, a.n - 1);
      s_row[r] = static_cast<const char*>(a.scales) + (s.expert * a.stride_s + (long long)row * a.lds) * scale_bytes;
      if (kZeros) z_row[r] = a.zeros + s.expert * a.stride_z + (long long)row * a.ldz;
    }
  };
  auto load_scales = [&] {
    if (kHeld > 1 && a.wide_scales) {
      const int gi = min(s_kb * NG + t * kHeld, a.last_group + 1 - kHeld);
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        if constexpr (kHeld == 4) {
          if (a.f32_scales) *reinterpret_cast<uint4*>(raw.s[r]) = *reinterpret_cast<const uint4*>(s_row[r] + 4 * gi);
          else *reinterpret_cast<uint2*>(raw.s[r]) = *reinterpret_cast<const uint2*>(s_row[r] + 2 * gi);
          if (kZeros) raw.z[r][0] = *reinterpret_cast<const uint32_t*>(z_row[r] + gi);
        } else {
          if (a.f32_scales) *reinterpret_cast<uint2*>(raw.s[r]) = *reinterpret_cast<const uint2*>(s_row[r] + 4 * gi);
          else raw.s[r][0] = *reinterpret_cast<const uint32_t*>(s_row[r] + 2 * gi);
          if (kZeros) raw.z[r][0] = *reinterpret_cast<const uint16_t*>(z_row[r] + gi);
        }
      }
    } else {
#pragma unroll
      for (int h = 0; h < kHeld; ++h) {
        int gi = s_kb * NG + t * kHeld + h;
        if (kPerGroup == 4 && a.group_span != 1) gi /= a.group_span;
        gi = min(gi, a.last_group);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          if (a.f32_scales) raw.s[r][h] = reinterpret_cast<const uint32_t*>(s_row[r])[gi];
          else raw.s[r][h] = reinterpret_cast<const uint16_t*>(s_row[r])[gi];
          if (kZeros) raw.z[r][h] = z_row[r][gi];
        }
      }
    }
    ++s_kb;
  };
  auto scale_of = [&](uint32_t bits) {
    if (a.f32_scales) return __uint_as_float(bits);
    const uint16_t b16 = uint16_t(bits);
    T v;
    memcpy(&v, &b16, 2);
    return to_f32(v);
  };
  auto store = [&](int slot, int n, float v) {
    const long long o = (long long)slot * a.ldo + n;
    if (a.f32_out) static_cast<float*>(a.out)[o] = v;
    else static_cast<T*>(a.out)[o] = from_f32<T>(v);
  };

  constexpr int kSets = TOK <= 8 ? 1 : TOK / 8;  // of up to 8 tokens
  // Where a lane reads: its ldmatrix rows in a box (swizzled by 16 bytes), its column's digits (of one token, the unused
  // columns read their neighbours') or its token's elements.
  const uint32_t in_box = lane % 16 * 128 + ((lane / 16 ^ (lane & 7)) * 16);
  const int x_lane = !kDigits<TOK> ? lane * 16 : t * 8 + (TOK == 2 ? g * 32 : g / 2 * 32);
  // A batch's sums of the cluster's blocks, a tile to a block in turn. They are gathered a batch later, when the
  // others' have long arrived; two buffers: by then every block has left the one that is written next.
  Stretch gathers = {};
  Pass gathers_pass = {};
  int flip = 0;
  auto gather = [&] {
    cluster_wait();
    const float* mine = reinterpret_cast<const float*>(smem + a.block) + flip * kWarps * kPiece<TOK>;
    for (int i = threadIdx.x; split + i / kPiece<TOK> * splits < gathers.count; i += kThreads) {
      const int m = split + i / kPiece<TOK> * splits, o = i % kPiece<TOK>, token = o / kRows, n = gathers.batch_row0 + m * kRows + o % kRows;
      if (token >= gathers_pass.count || n >= a.n) continue;
      float v = 0.0f;
      for (int r = 0; r < splits; ++r) v += cluster.map_shared_rank(mine, r)[m * kPiece<TOK> + o];
      store(slot_of(gathers_pass.first + token), n, v);
    }
    __syncwarp();
  };
  const Codes<T> codes;
  float acc[kSets][4] = {};
  Pass p = {};
  Stretch u = {};
  int in = 0, out = 0, issued = 0, done = 0;  // ring slots to fill next and of unit `done`; units
  int now_left = 0, at_pass = -1;             // units left of the stretch at hand
  uint32_t parity = 0;
  const uint8_t *xd = smem, *xs = smem, *xp = smem;
  int k_at = 0;
  // The rests of a unit's marked 128s, in the form for more tokens: column i is token i, so the sums join digit 0's.
  auto add_rests = [&](uint32_t base, const float (&s_now)[2][kHeld], const uint32_t (&z_now)[2], uint2 marks) {
    const Codes<T> codes;
#pragma unroll 1
    for (int quarter = 0; quarter < 4; ++quarter) {
      if (((quarter < 2 ? marks.x : marks.y) >> quarter % 2 * 16 & 0xFFFFu) == 0) continue;
      const float down = *reinterpret_cast<const float*>(xp - t * 8 + quarter * kPowerBytes<TOK> + g % TOK * 4);
      const float up = __uint_as_float(0x7F000000u - __float_as_uint(down));
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        const int k = k_at + quarter * 128 + c * 32 + t * 8, group = quarter * (NG / 4) + c / kPerGroup;
        uint4 q = make_uint4(0, 0, 0, 0);
        if (g < p.count && k < a.k) {
          float v[8];
          unpack<T>(*reinterpret_cast<const uint4*>(row_of(p, g) + k), v);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = fmaf(-float(__float2int_rn(v[j] * up)), down, v[j]);
          q = pack<T>(v);
        }
        q = make_uint4(__byte_perm(q.x, q.z, 0x5410), __byte_perm(q.x, q.z, 0x7632), __byte_perm(q.y, q.w, 0x5410), __byte_perm(q.y, q.w, 0x7632));
        uint32_t w[4];
        ldmatrix_x4(w, (base + quarter / 2 * kBoxBytes) ^ (quarter % 2 * 64 + c / 2 * 32));
        float sc[2], dot[4];
        uint32_t z[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int from = (lane & 28) | group / kHeld;
          float s = s_now[r][0];
#pragma unroll
          for (int h = 1; h < kHeld; ++h) s = group % kHeld == h ? s_now[r][h] : s;
          sc[r] = __shfl_sync(0xFFFFFFFFu, s, from);
          z[r] = kZeros ? __shfl_sync(0xFFFFFFFFu, z_now[r], from) >> 8 * (group % kHeld) & 0xFF : 8;
        }
        CodesOf32<T, kZeros>(codes, c % 2 ? w[2] : w[0], c % 2 ? w[3] : w[1], z).times(dot, q, true);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[0][i] = fmaf(sc[i / 2], dot[i], acc[0][i]);
      }
    }
  };
  if (a.ids == nullptr) griddep_wait();
  griddep_launch_dependents();
  if (remaining > 0) {  // x first: what the start waits for goes before the weights
    p = pass_of(pass);
    begin_x(p);
  }
#pragma unroll 1
  while (true) {
    // At first one unit a warp: what the start waits for does not queue behind a whole ring of weights.
    while ((left > 0 || run_left > 0 || remaining > count) && issued - done < (at_pass < 0 ? 1 : depth)) {
      produce(in);
      in = in + 1 == depth ? 0 : in + 1;
      ++issued;
    }
    if (done == issued) break;
    if (now_left == 0) {
      __syncwarp();
      u = records[out];
      if (u.pass != at_pass) {  // every warp has a record of every batch, so all come here together
        const bool start = at_pass < 0;
        at_pass = u.pass;
        if (start) {
          aim_scales(u);
          load_scales();
        } else {
          p = pass_of(at_pass);
          begin_x(p);
          __syncthreads();
        }
        convert(p);
        if constexpr (kDigits<TOK>) marked = __syncthreads_or(marked);
        else __syncthreads();
        if (start) continue;  // to fill the ring
      }
      now_left = max(u.units, 1);
      k_at = (kb0 + u.kb) * kUnitK<TOK>;
      xd = smem + a.x_at + u.kb * (kUnitK<TOK> / 32) * kXRow<TOK> + x_lane;
      xs = smem + a.sums + u.kb * NG * kSumBytes<TOK> + t * 8;
      xp = smem + a.powers + u.kb * (kUnitK<TOK> / 128) * kPowerBytes<TOK> + t * 8;
#pragma unroll
      for (int set = 0; set < kSets; ++set) acc[set][0] = acc[set][1] = acc[set][2] = acc[set][3] = 0.0f;
    }
    float s_now[2][kHeld];
    uint32_t z_now[2];  // a byte a group
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      if (kHeld > 1 && a.wide_scales) {
#pragma unroll
        for (int h = 0; h < kHeld; ++h) s_now[r][h] = scale_of(a.f32_scales ? raw.s[r][h] : raw.s[r][h / 2] >> 16 * (h % 2) & 0xFFFFu);
        z_now[r] = raw.z[r][0];
      } else {
        z_now[r] = 0;
#pragma unroll
        for (int h = 0; h < kHeld; ++h) {
          s_now[r][h] = scale_of(raw.s[r][h]);
          z_now[r] |= raw.z[r][h] << 8 * h;
        }
      }
    }
    if (now_left > 1) {
      load_scales();
    } else if (done + 1 < issued) {
      __syncwarp();
      aim_scales(records[out + 1 == depth ? 0 : out + 1]);
      load_scales();
    }
    if ((u.flags & kNone) == 0) {
      if (!failed) failed = __any_sync(0xFFFFFFFFu, !mbarrier_wait(bar0 + 8 * out, parity, a.timeout_ns));
      if (!failed) {
        const uint32_t base = ring0 + out * kUnitBytes<TOK> + in_box;
        const bool whole = kHalves == 1 || k_at + 256 < a.k;
#pragma unroll
        for (int quarter = 0; quarter < kUnitK<TOK> / 128; ++quarter) {  // 128 codes
          if (quarter == 2 && !whole) break;
          constexpr int kGroups = 4 / kPerGroup;  // of a quarter
          int part[4];                            // of a group
          float sum[4] = {};                      // of the quarter
          float dot[kSets][4];                    // of a group
          float sc[2];
          uint32_t z[2] = {8, 8}, z_four[2];
#pragma unroll
          for (int pair = 0; pair < 2; ++pair) {
            // Matrices: rows 0-7 and 8-15 of chunk 2 pair, then of chunk 2 pair + 1.
            uint32_t w[4];
            ldmatrix_x4(w, (base + quarter / 2 * kBoxBytes) ^ (quarter % 2 * 64 + pair * 32));
#pragma unroll
            for (int cc = 0; cc < 2; ++cc) {
              const int c = pair * 2 + cc, gj = c / kPerGroup;
              const bool begins = c % kPerGroup == 0, ends = c % kPerGroup == kPerGroup - 1;
              const uint8_t* xc = xd + (quarter * 4 + c) * kXRow<TOK>;
              if (begins) {
                const int from = (lane & 28) | (quarter * kGroups + gj) / kHeld, held = (quarter * kGroups + gj) % kHeld;
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                  sc[r] = __shfl_sync(0xFFFFFFFFu, s_now[r][held], from);
                  if (kZeros && held == 0) z_four[r] = __shfl_sync(0xFFFFFFFFu, z_now[r], from);
                  if (kZeros) z[r] = z_four[r] >> 8 * held & 0xFF;
                }
              }
              if constexpr (kDigits<TOK>) {
                const uint32_t f[4] = {w[2 * cc] & kNibbles, w[2 * cc + 1] & kNibbles, (w[2 * cc] >> 4) & kNibbles,
                                       (w[2 * cc + 1] >> 4) & kNibbles};
                mma_u8s8(part, f, *reinterpret_cast<const uint2*>(xc), begins);
                if (!ends) continue;
                const int2 q = *reinterpret_cast<const int2*>(xs + (quarter * kGroups + gj) * kSumBytes<TOK>);
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[i] = fmaf(sc[i / 2], float(part[i] - int(z[i / 2]) * (i % 2 ? q.y : q.x)), sum[i]);
              } else {
                const CodesOf32<T, kZeros> f(codes, w[2 * cc], w[2 * cc + 1], z);
#pragma unroll
                for (int set = 0; set < kSets; ++set) {
                  if (set > 0 && p.count <= 8) continue;
                  f.times(dot[set], *reinterpret_cast<const uint4*>(xc + set * 512), begins);
                  if (!ends) continue;
#pragma unroll
                  for (int i = 0; i < 4; ++i) acc[set][i] = fmaf(sc[i / 2], dot[set][i], acc[set][i]);
                }
              }
            }
          }
          if constexpr (kDigits<TOK>) {
            const float2 q = *reinterpret_cast<const float2*>(xp + quarter * kPowerBytes<TOK>);
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[0][i] = fmaf(i % 2 ? q.y : q.x, sum[i], acc[0][i]);
          }
        }
        if constexpr (kDigits<TOK>) {
          if (marked) {
            uint2 rests = *reinterpret_cast<const uint2*>(smem + a.rests + (k_at / kUnitK<TOK> - kb0) * kRestBytes<TOK>);
            if (p.count == 1) rests = make_uint2(rests.x & 0x00FF00FFu, rests.y & 0x00FF00FFu);
            if (rests.x | rests.y) add_rests(base, s_now, z_now, rests);
          }
        }
        xd += kUnitK<TOK> / 32 * kXRow<TOK>;
        xs += NG * kSumBytes<TOK>;
        xp += kUnitK<TOK> / 128 * kPowerBytes<TOK>;
        k_at += kUnitK<TOK>;
        __syncwarp();  // the slot is read
      }
    }
    if (--now_left == 0) {
      // The stretch ends. In a full batch a tile is a warp's own, all of this block's K; else the warps leave their
      // parts, [token][row], and add them up in their order along K: warp w's run is [count kbs w / 16,
      // count kbs (w + 1) / 16), tile m's units [m kbs, (m + 1) kbs).
      const bool full = u.count == kWarps;
      auto spread = [&](auto&& f) {  // f(cell, sum) for this lane's cells of the tile
        if constexpr (kDigits<TOK>) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float v = acc[0][i];  // digits 0 and 1, 2 and 3, then the two sums
            v += __shfl_xor_sync(0xFFFFFFFFu, v, 1);
            v += __shfl_xor_sync(0xFFFFFFFFu, v, 2);
            if (t == 0 && i % 2 < TOK) f(i % 2 * kRows + i / 2 * 8 + g, v);
          }
        } else {
#pragma unroll
          for (int set = 0; set < kSets; ++set)
#pragma unroll
            for (int i = 0; i < 4; ++i) f((set * 8 + 2 * t + i % 2) * kRows + i / 2 * 8 + g, acc[set][i]);
        }
      };
      if (!full && (u.flags & kNone) == 0) {
        float* to = pieces + (warp * kPieces + ((u.flags & kSecond) != 0)) * kPiece<TOK>;
        spread([&](int o, float v) { to[o] = v; });
      }
      if ((u.flags & kEnd) != 0) {
        auto put = [&](int m, int o, float v) {
          const int token = o / kRows, n = u.batch_row0 + m * kRows + o % kRows;
          if (token < p.count && n < a.n) store(slot_of(p.first + token), n, v);
        };
        if (splits > 1) {
          __syncwarp();
          if (gathers.count > 0) gather();
          gathers = u;
          gathers_pass = p;
          flip ^= 1;
        }
        float* mine = reinterpret_cast<float*>(smem + a.block) + flip * kWarps * kPiece<TOK>;
        if (full) {
          if (splits > 1) spread([&](int o, float v) { mine[warp * kPiece<TOK> + o] = v; });
          else spread([&](int o, float v) { put(warp, o, v); });
        } else {
          __syncthreads();
          for (int i = threadIdx.x; i < u.count * kPiece<TOK>; i += kThreads) {
            const int m = i / kPiece<TOK>, o = i % kPiece<TOK>;
            float sum = 0.0f;
            for (int w = m * kWarps / u.count; w < kWarps; ++w) {
              const int lo = u.count * kbs * w / kWarps, hi = u.count * kbs * (w + 1) / kWarps;
              if (lo >= (m + 1) * kbs) break;
              if (lo >= hi || hi <= m * kbs) continue;  // no units, or none of this tile
              sum += pieces[(w * kPieces + (lo >= m * kbs ? 0 : 1)) * kPiece<TOK> + o];  // 1: the run began in the tile before
            }
            if (splits > 1) mine[i] = sum;
            else put(m, o, sum);
          }
          __syncthreads();
        }
        __syncwarp();
        if (splits > 1) cluster_arrive();
      }
    }
    ++done;
    out = out + 1 == depth ? 0 : out + 1;
    if (out == 0) parity ^= 1;
  }
  if (splits > 1) {
    if (gathers.count > 0) gather();
    cluster_sync();  // no block leaves while another may still read its sums
  }
  if (failed) {
    // The loads still under way end, or are given up on, before the block leaves.
    if (lane == 0) atomicOr(a.status, kl::gemm::kStatusProducerTimeout);
    for (int i = 0; i < depth; ++i) mbarrier_wait(bar0 + 8 * i, i < out ? parity : parity ^ 1, a.timeout_ns);
  }
  // Rows of slots without an expert.
  if (a.ids != nullptr && l.start[active] < a.slots)
    for (int s = blockIdx.x; s < a.slots; s += gridDim.x) {
      const int e = a.ids[s];
      if (e >= 0 && e < a.experts) continue;
      for (int n = threadIdx.x; n < a.n; n += kThreads) store(s, n, 0.0f);
    }
}

struct Fit {
  int cluster, depth;
  size_t bytes;
  Int4Args args;  // with the layout
};

// The smallest cluster whose blocks keep x in 80 KB beside a ring of two slots a warp, else 8, and the ring that the
// rest holds (at most 8 slots a warp). depth 0: does not fit. With x in 40 KB 16 tokens of 28672 x 8192 take 71.6 us
// instead of 60.3 (a cluster's sums cost more than a deeper ring gains), 13 tokens of 10007 x 4128 21.8 instead of 20.4.
template <int NG, int TOK>
Fit fit(Int4Args const& a) {
  const int kb = (a.k + kUnitK<TOK> - 1) / kUnitK<TOK>;
  Fit f = {1, 0, 0, {}};
  for (;; f.cluster *= 2) {
    const int units = (kb + f.cluster - 1) / f.cluster;
    Int4Args b = a;
    for (int depth = 2; depth <= 8; ++depth) {
      const size_t bytes = lay_out<NG, TOK>(b, depth, units, f.cluster);
      if (bytes > size_t(kSmemLimit)) break;
      f.depth = depth;
      f.bytes = bytes;
      f.args = b;
    }
    if (f.cluster == 8 || (f.depth >= 2 && size_t(units) * kXBytes<NG, TOK> <= 80 * 1024)) return f;
    f.depth = 0;
  }
}

template <class T, int NG, int TOK, bool kZeros>
kl_status launch(Fit const& f, int device, cudaStream_t stream) {
  Int4Args a = f.args;
  auto* kernel = gemv_int4_kernel<T, NG, TOK, kZeros>;
  static std::atomic<int> resident[64][4];  // by device: clusters of 1, 2, 4, 8 that fit at once
  const int which = f.cluster == 1 ? 0 : f.cluster == 2 ? 1 : f.cluster == 4 ? 2 : 3;
  constexpr uint64_t kHeld = NG >= 4 ? NG / 4 : 1;  // as in the kernel
  const uint64_t scale_bytes = a.f32_scales ? 4 : 2;
  a.wide_scales = (a.last_group + 1) % kHeld == 0 && a.lds % kHeld == 0 && a.stride_s % kHeld == 0 &&
                  reinterpret_cast<uintptr_t>(a.scales) % (kHeld * scale_bytes) == 0 &&
                  (!kZeros || (a.ldz % kHeld == 0 && a.stride_z % kHeld == 0 && reinterpret_cast<uintptr_t>(a.zeros) % kHeld == 0));
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = f.bytes;
  cfg.stream = stream;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(f.cluster);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  int most = resident[device][which].load(std::memory_order_acquire);
  if (most == 0) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimit);
    if (e != cudaSuccess) return cuda_fail(e, "kl_gemv_int4 shared memory");
    cfg.gridDim = dim3(unsigned(f.cluster), 1, 1);
    cfg.dynamicSmemBytes = kSmemLimit;
    cfg.numAttrs = 1;
    e = cudaOccupancyMaxActiveClusters(&most, kernel, &cfg);
    if (e != cudaSuccess) return cuda_fail(e, "kl_gemv_int4 occupancy");
    if (most <= 0) return fail(KL_ERR_CUDA, "kl_gemv_int4: no room for a block");
    resident[device][which].store(most, std::memory_order_release);
    cfg.dynamicSmemBytes = f.bytes;
  }
  const long long passes = a.ids != nullptr ? a.slots : (a.slots + TOK - 1) / TOK;
  const long long work = passes * a.tiles;
  if (work > INT32_MAX / 2) return fail(KL_ERR_NOT_SUPPORTED, "kl_gemv_int4: too many rows of out");
  cfg.gridDim = dim3(unsigned((work < most ? work : most) * f.cluster), 1, 1);
  cfg.numAttrs = 2;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
  return e == cudaSuccess ? KL_OK : cuda_fail(e, "kl_gemv_int4 launch");
}

// Tokens of a pass by what a matrix meets (with ids: on average), fewer where x would not fit: 16 above K = 22528, 8 above
// 28672, a little less with long lists. 28672 x 8192: 2 tokens 26 us, in the form for 8 42; 4 tokens 42, in two passes of 2
// 47; 16 tokens 60, in two passes of 8 85. 8192 rows, 16 tokens: K = 22528 52, 24576 71 (two passes of 8), 32768 200
// (eight of 2). 16 tokens x 4 of 64, 4096 x 1536, groups of 32: 53 us with even ids, 51 where one expert has every token.
template <class T, int GROUP, bool kZeros>
kl_status by_tokens(Int4Args& a, int device, cudaStream_t stream) {
  const int tokens = a.ids != nullptr ? (a.slots + a.experts - 1) / a.experts : a.slots;
  if (tokens > 8)
    if (const Fit f = fit<kUnitK<16> / GROUP, 16>(a); f.depth >= 2) return launch<T, kUnitK<16> / GROUP, 16, kZeros>(f, device, stream);
  if (tokens > 2)
    if (const Fit f = fit<kUnitK<8> / GROUP, 8>(a); f.depth >= 2) return launch<T, kUnitK<8> / GROUP, 8, kZeros>(f, device, stream);
  if (a.slots > 1)
    if (const Fit f = fit<kUnitK<2> / GROUP, 2>(a); f.depth >= 2) return launch<T, kUnitK<2> / GROUP, 2, kZeros>(f, device, stream);
  const Fit f = fit<kUnitK<1> / GROUP, 1>(a);
  if (f.depth < 2) return fail(KL_ERR_NOT_SUPPORTED, "kl_gemv_int4: k does not fit");
  return launch<T, kUnitK<1> / GROUP, 1, kZeros>(f, device, stream);
}

template <class T, bool kZeros>
kl_status by_group(Int4Args& a, int device, cudaStream_t stream) {
  if (a.group == 32) return by_tokens<T, 32, kZeros>(a, device, stream);
  if (a.group == 64) return by_tokens<T, 64, kZeros>(a, device, stream);
  return by_tokens<T, 128, kZeros>(a, device, stream);
}

template <class T>
kl_status by_zeros(Int4Args& a, int device, cudaStream_t stream) {
  return a.zeros != nullptr ? by_group<T, true>(a, device, stream) : by_group<T, false>(a, device, stream);
}

// The group as the kernel counts it, in 32 bits: one that is longer than a row is the row, in whole 128s.
int64_t group_within(kl_int4_desc const& d) {
  const int64_t row = d.k > 128 ? (d.k + 127) / 128 * 128 : 128;
  return d.group < row ? d.group : row;
}

kl_status run(kl_int4_desc const& d, int64_t slots, cudaStream_t stream) {
  const bool by_expert = d.ids != nullptr;
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  if (device < 0 || device >= 64) return fail(KL_ERR_NOT_SUPPORTED, "device index above 63");
  Int4Args a = {};
  const int64_t matrices = by_expert ? d.experts : 1;
  const int64_t shape[3] = {matrices, d.n, d.k / 2};
  const int64_t stride[3] = {matrices > 1 ? d.stride_q : d.n * d.ldq, d.ldq, 1};
  kl::TmaOptions opt;
  opt.l2_promotion = CU_TENSOR_MAP_L2_PROMOTION_L2_256B;
  kl::detail::encode_tma_map(&a.map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, CU_TENSOR_MAP_SWIZZLE_128B, 128, kRows, d.q, 3,
                             shape, stride, opt);
  a.x = d.x;
  a.ldx = d.ldx;
  a.scales = d.scales;
  a.lds = int(d.ld_scales);
  a.stride_s = matrices > 1 ? d.stride_scales : 0;
  a.zeros = d.zeros;
  a.ldz = int(d.ld_zeros);
  a.stride_z = matrices > 1 ? d.stride_zeros : 0;
  a.ids = d.ids;
  a.experts = int(matrices);
  a.slots = int(slots);
  a.x_div = by_expert && !d.x_per_slot ? int(d.topk) : 1;
  a.out = d.out;
  a.ldo = d.ldo;
  a.n = int(d.n);
  a.k = int(d.k);
  a.group = int(group_within(d));
  a.f32_scales = d.scale_type == KL_F32;
  a.f32_out = d.out_type == KL_F32;
  a.tiles = (a.n + kRows - 1) / kRows;
  a.group_span = a.group >= 128 ? a.group / 128 : 1;
  a.last_group = (a.k + a.group - 1) / a.group - 1;
  a.timeout_ns = wait_timeout_ns();
  kl_status s = device_status_ptr(&a.status);
  if (s != KL_OK) return s;
  return d.x_type == KL_BF16 ? by_zeros<__nv_bfloat16>(a, device, stream) : by_zeros<__half>(a, device, stream);
}

}  // namespace
}  // namespace kl::capi
extern "C" kl_status kl_gemv_int4(const kl_int4_desc* d, void* stream) {
  using namespace kl::capi;
  auto bad = [](char const* what) { return fail(KL_ERR_INVALID_ARGUMENT, std::string("kl_gemv_int4: ") + what); };
  if (d == nullptr) return bad("null descriptor");
  if (d->tokens < 0 || d->n < 0 || d->k < 0) return bad("negative extent");
  const bool by_expert = d->ids != nullptr;
  if (by_expert && (d->topk < 1 || d->experts < 1)) return bad("ids need topk >= 1 and experts >= 1");
  const int64_t topk = by_expert ? d->topk : 1;
  if (d->tokens > INT32_MAX / 64 || d->n > INT32_MAX / 2 || d->k > INT32_MAX / 2 || topk > kMaxSlots) return bad("extent too large");
  const int64_t slots = d->tokens * topk;
  if (by_expert && (slots > kMaxSlots || d->experts > kMaxExperts))
    return fail(KL_ERR_NOT_SUPPORTED, "kl_gemv_int4: at most 4096 (token, expert) pairs and 1024 experts a call (more tokens: in calls of some of them)");
  if (d->x_type != KL_BF16 && d->x_type != KL_F16) return fail(KL_ERR_NOT_SUPPORTED, "kl_gemv_int4: x must be bf16 or f16");
  if (d->scale_type != d->x_type && d->scale_type != KL_F32)
    return fail(KL_ERR_NOT_SUPPORTED, "kl_gemv_int4: scales must have x's type or f32");
  if (d->out_type != d->x_type && d->out_type != KL_F32)
    return fail(KL_ERR_NOT_SUPPORTED, "kl_gemv_int4: out must have x's type or f32");
  if (d->group != 32 && d->group != 64 && (d->group < 128 || d->group % 128 != 0))
    return bad("group must be 32, 64 or a multiple of 128");
  if (d->k % 32 != 0) return bad("k must be a multiple of 32");
  if (d->k > kMaxK) return fail(KL_ERR_NOT_SUPPORTED, "kl_gemv_int4: k up to 65536");
  if (slots == 0 || d->n == 0) return KL_OK;
  const int64_t group = group_within(*d), groups = (d->k + group - 1) / group;
  if (d->ldo < d->n || d->ldx < d->k || d->ldq < d->k / 2 || d->ld_scales < groups || (d->zeros != nullptr && d->ld_zeros < groups))
    return bad("row pitch below the row's extent");
  if (d->ld_scales > INT32_MAX / 4 || d->ld_zeros > INT32_MAX) return bad("row pitch too large");
  if (d->out == nullptr || (d->k > 0 && (d->x == nullptr || d->q == nullptr || d->scales == nullptr))) return bad("null pointer");
  if (d->k > 0 && (!aligned16(d->x) || !aligned16(d->q) || d->ldx % 8 != 0 || d->ldq % 16 != 0))
    return bad("x and q must be 16-byte aligned with row pitches that are multiples of 16 bytes");
  if (!aligned(d->scales, d->scale_type == KL_F32 ? 4 : 2) || !aligned(d->out, d->out_type == KL_F32 ? 4 : 2) || !aligned(d->ids, 4))
    return bad("scales, out and ids must be aligned to their elements");
  if (by_expert && d->experts > 1 && (d->stride_q % 16 != 0 || d->stride_q <= 0 || d->stride_scales < 0 || d->stride_zeros < 0))
    return bad("expert strides must not be negative, stride_q a positive multiple of 16 bytes");
  if (d->k == 0) {  // a sum of nothing
    const size_t size = d->out_type == KL_F32 ? 4 : 2;
    cudaError_t e = cudaMemset2DAsync(d->out, size_t(d->ldo) * size, 0, size_t(d->n) * size, size_t(slots), static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? KL_OK : cuda_fail(e, "kl_gemv_int4 memset");
  }
  try {
    return run(*d, slots, static_cast<cudaStream_t>(stream));
  } catch (std::exception const& e) {
    return bad(e.what());
  }
}
