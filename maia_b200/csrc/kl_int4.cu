// Products with 4-bit weights and group scales for few tokens (kl_gemv_int4):
//   out[t, n] = sum_g s[n, g] sum_{i in g} (q[n, i] - z[n, g]) x[t, i],
// with one matrix, or one per expert and the expert of every (token, slot) in `ids`.
//
// The weights' bytes bound it: each is read once for up to 8 kTiles tokens. mma.sync.m16n8k16 takes
// 16 weight rows as its A operand straight from registers and 8 tokens as its B, so up to 8 tokens
// cost what one does. The codes become bf16 / f16 exactly: OR-ing a code into the mantissa of 128
// (bf16) or 1024 (f16) gives 128 + q or 1024 + q, and subtracting 128 + z or 1024 + z leaves q - z
// without rounding. Products are summed in fp32, group by group, and each group's sum is multiplied
// by its scale in fp32.

#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <string>

#include <kl/arch/griddep.hpp>
#include <kl_gemm.h>

#include "kl_internal.cuh"
#include "kl_vec.cuh"

namespace cg = cooperative_groups;

namespace kl::capi {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kRows = 16;         // weight rows of a block
constexpr int kChunk = 128;       // K-elements a warp takes at a time
constexpr int kMaxSlots = 8192;   // (token, expert) pairs of a call with ids

struct Int4Args {
  const void* x;
  long long ldx;
  const uint8_t* q;
  long long ldq, stride_q;  // bytes
  const void* scales;
  long long lds, stride_s;
  const uint8_t* zeros;
  long long ldz, stride_z;
  const int* ids;
  int experts, slots, x_div;  // slots: rows of out; x row = slot / x_div
  void* out;
  long long ldo;
  int n, k, group;
  int f32_scales, f32_out;
  int by_slot;  // block row y of the grid: the y-th slot, if its expert's first; else expert y
};

template <class T>
struct Codes;

// Four registers of two weights each from eight codes: register c holds codes c (low) and c + 4.
template <>
struct Codes<__nv_bfloat16> {
  static __device__ __forceinline__ uint32_t offset(int z) {  // 128 + z, twice
    return 0x43004300u | uint32_t(z) * 0x00010001u;
  }
  static __device__ __forceinline__ void expand(uint32_t w, uint32_t off, uint32_t (&r)[4]) {
    const __nv_bfloat162 o = *reinterpret_cast<const __nv_bfloat162*>(&off);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      uint32_t u = ((w >> (4 * c)) & 0x000F000Fu) | 0x43004300u;
      const __nv_bfloat162 v = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&u), o);
      r[c] = *reinterpret_cast<const uint32_t*>(&v);
    }
  }
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

template <>
struct Codes<__half> {
  static __device__ __forceinline__ uint32_t offset(int z) {  // 1024 + z, twice
    return 0x64006400u | uint32_t(z) * 0x00010001u;
  }
  static __device__ __forceinline__ void expand(uint32_t w, uint32_t off, uint32_t (&r)[4]) {
    const __half2 o = *reinterpret_cast<const __half2*>(&off);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      uint32_t u = ((w >> (4 * c)) & 0x000F000Fu) | 0x64006400u;
      const __half2 v = __hsub2(*reinterpret_cast<__half2*>(&u), o);
      r[c] = *reinterpret_cast<const uint32_t*>(&v);
    }
  }
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

// kWords consecutive 32-bit words of a lane belong to one scale group: 4 (groups of 128 and
// multiples), 2 (64) or 1 (32). In a chunk of 128 K-elements, lane t of a row's four holds
// K = 8 kWords (4 h + t) .. + 8 kWords for h = 0 .. 4 / kWords - 1: the four lanes of a row read
// neighbouring words of one group, and x is read at the same K. The order of K inside an MMA is free
// as long as both operands use it.
template <int kWords>
__device__ __forceinline__ void load_words(const uint8_t* p, bool ok, uint32_t* w) {
  if constexpr (kWords == 4) {
    const uint4 u = ok ? __ldg(reinterpret_cast<const uint4*>(p)) : make_uint4(0, 0, 0, 0);
    w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
  } else if constexpr (kWords == 2) {
    const uint2 u = ok ? __ldg(reinterpret_cast<const uint2*>(p)) : make_uint2(0, 0);
    w[0] = u.x; w[1] = u.y;
  } else {
    w[0] = ok ? __ldg(reinterpret_cast<const uint32_t*>(p)) : 0u;
  }
}

template <class T, int kWords, int kTiles>
__global__ void __launch_bounds__(kThreads) gemv_int4_kernel(const Int4Args a) {
  constexpr int kHops = 4 / kWords;
  constexpr int kTok = 8 * kTiles;
  __shared__ float red[kWarps][kRows * kTok];
  extern __shared__ int list[];  // with ids: the slots of this block's expert
  __shared__ int list_size;
  cg::cluster_group cluster = cg::this_cluster();
  griddep_wait();
  griddep_launch_dependents();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  const int n0 = (blockIdx.x / cluster.num_blocks()) * kRows;
  const int split = int(cluster.block_rank()), splits = int(cluster.num_blocks());
  int expert = 0, first = 0, count = 0;
  if (a.ids == nullptr) {
    first = blockIdx.y * kTok;
    count = a.slots - first < kTok ? a.slots - first : kTok;
  } else {
    // Every block of a cluster reads the same ids and so takes the same way.
    auto id_at = [&](int s) {
      const int e = a.ids[s];
      return e >= 0 && e < a.experts ? e : a.experts;  // a.experts: no expert
    };
    expert = a.by_slot ? id_at(blockIdx.y) : int(blockIdx.y);
    if (warp == 0) {
      int found = 0;
      for (int s0 = 0; s0 < a.slots; s0 += 32) {
        const int s = s0 + lane;
        const bool mine = s < a.slots && id_at(s) == expert;
        const unsigned who = __ballot_sync(0xFFFFFFFFu, mine);
        if (mine) list[found + __popc(who & ((1u << lane) - 1))] = s;
        found += __popc(who);
      }
      if (lane == 0) list_size = found;
    }
    __syncthreads();
    count = list_size;
    if (count == 0 || (a.by_slot && list[0] != int(blockIdx.y))) return;
  }
  const long long row_a = n0 + g < a.n ? n0 + g : a.n - 1, row_b = n0 + g + 8 < a.n ? n0 + g + 8 : a.n - 1;
  const bool any = a.ids == nullptr || expert < a.experts;
  const uint8_t* q = a.q + (any ? expert : 0) * a.stride_q;
  const long long s_off = (any ? expert : 0) * a.stride_s;
  const uint8_t* z = a.zeros != nullptr ? a.zeros + (any ? expert : 0) * a.stride_z : nullptr;
  auto scale_at = [&](long long row, int gi) {
    const long long i = s_off + row * a.lds + gi;
    return a.f32_scales ? static_cast<const float*>(a.scales)[i] : to_f32(static_cast<const T*>(a.scales)[i]);
  };
  const int chunks = (a.k + kChunk - 1) / kChunk;
  for (int base = 0; base < count; base += kTok) {
    const int here = count - base < kTok ? count - base : kTok;
    const T* xp[kTiles];
    bool live[kTiles];
#pragma unroll
    for (int j = 0; j < kTiles; ++j) {
      live[j] = j * 8 + g < here;
      const int slot = !live[j] ? 0 : a.ids == nullptr ? first + j * 8 + g : list[base + j * 8 + g];
      xp[j] = static_cast<const T*>(a.x) + (long long)(slot / a.x_div) * a.ldx;
    }
    float acc[kTiles][4] = {};
    if (any) {
      for (int c = split * kWarps + warp; c < chunks; c += splits * kWarps) {
#pragma unroll
        for (int h = 0; h < kHops; ++h) {
          const int k0 = c * kChunk + 8 * kWords * (4 * h + t);
          const bool ok = k0 < a.k;  // K is a multiple of 32 = the most that a lane holds
          const int kg = c * kChunk + 32 * kWords * h;  // where the row's four lanes begin
          if (kg >= a.k) break;
          const int gi = kg / a.group;
          uint32_t wa[kWords], wb[kWords];
          load_words<kWords>(q + row_a * a.ldq + k0 / 2, ok, wa);
          load_words<kWords>(q + row_b * a.ldq + k0 / 2, ok, wb);
          const uint32_t off_a = Codes<T>::offset(z != nullptr ? z[row_a * a.ldz + gi] : 8);
          const uint32_t off_b = Codes<T>::offset(z != nullptr ? z[row_b * a.ldz + gi] : 8);
          const float sa = scale_at(row_a, gi), sb = scale_at(row_b, gi);
          float part[kTiles][4] = {};
#pragma unroll
          for (int i = 0; i < kWords; ++i) {
            uint32_t ra[4], rb[4];
            Codes<T>::expand(wa[i], off_a, ra);
            Codes<T>::expand(wb[i], off_b, rb);
            const uint32_t a0[4] = {ra[0], rb[0], ra[1], rb[1]}, a1[4] = {ra[2], rb[2], ra[3], rb[3]};
#pragma unroll
            for (int j = 0; j < kTiles; ++j) {
              if (kTiles > 1 && j * 8 >= here) break;
              uint4 u = make_uint4(0, 0, 0, 0);
              if (live[j] && ok) u = __ldg(reinterpret_cast<const uint4*>(xp[j] + k0 + 8 * i));
              Codes<T>::mma(part[j], a0, __byte_perm(u.x, u.z, 0x5410), __byte_perm(u.x, u.z, 0x7632));
              Codes<T>::mma(part[j], a1, __byte_perm(u.y, u.w, 0x5410), __byte_perm(u.y, u.w, 0x7632));
            }
          }
#pragma unroll
          for (int j = 0; j < kTiles; ++j) {
            acc[j][0] += sa * part[j][0];
            acc[j][1] += sa * part[j][1];
            acc[j][2] += sb * part[j][2];
            acc[j][3] += sb * part[j][3];
          }
        }
      }
    }
    // The warps' sums, then the cluster's blocks' sums, each in a fixed order.
#pragma unroll
    for (int j = 0; j < kTiles; ++j) {
      float* r = red[warp] + (j * 8 + 2 * t) * kRows + g;  // [token][row]
      r[0] = acc[j][0];
      r[kRows] = acc[j][1];
      r[8] = acc[j][2];
      r[kRows + 8] = acc[j][3];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kRows * kTok; i += kThreads) {
      float s = red[0][i];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) s += red[w][i];
      red[0][i] = s;
    }
    if (splits > 1) cluster.sync();
    else __syncthreads();
    if (split == 0) {
      for (int i = threadIdx.x; i < kRows * here; i += kThreads) {
        float s = red[0][i];
        for (int r = 1; r < splits; ++r) s += cluster.map_shared_rank(&red[0][0], r)[i];
        const int n = n0 + i % kRows, tok = i / kRows;
        if (n >= a.n) continue;
        const long long o = (long long)(a.ids == nullptr ? first + tok : list[base + tok]) * a.ldo + n;
        if (a.f32_out) static_cast<float*>(a.out)[o] = s;
        else static_cast<T*>(a.out)[o] = from_f32<T>(s);
      }
    }
    if (splits > 1) cluster.sync();
    else __syncthreads();
  }
}

template <class T, int kWords, int kTiles>
cudaError_t launch(Int4Args const& a, cudaStream_t stream) {
  const int tiles = (a.n + kRows - 1) / kRows;
  const int chunks = (a.k + kChunk - 1) / kChunk;
  const long long rows_y = a.ids == nullptr ? (a.slots + 8 * kTiles - 1) / (8 * kTiles) : a.by_slot ? a.slots : a.experts + 1;
  // K is split over the blocks of a cluster while there are too few blocks to fill the SMs and every
  // warp still has a chunk.
  int splits = 1;
  while (splits < 8 && (long long)tiles * rows_y * splits < 4 * 148 && chunks >= 2 * splits * kWarps) splits *= 2;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  cfg.gridDim = dim3(unsigned(tiles * splits), unsigned(rows_y), 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = a.ids != nullptr ? size_t(a.slots) * 4 : 0;
  cfg.stream = stream;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = unsigned(splits);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  auto* kernel = gemv_int4_kernel<T, kWords, kTiles>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSlots * 4);
  if (e != cudaSuccess) return e;
  return cudaLaunchKernelEx(&cfg, kernel, a);
}

template <class T, int kWords>
cudaError_t by_tiles(Int4Args const& a, cudaStream_t stream) {
  if (a.ids != nullptr) return a.slots <= 8 ? launch<T, kWords, 1>(a, stream) : launch<T, kWords, 2>(a, stream);
  if (a.slots <= 8) return launch<T, kWords, 1>(a, stream);
  if (a.slots <= 16) return launch<T, kWords, 2>(a, stream);
  return launch<T, kWords, 4>(a, stream);
}

template <class T>
cudaError_t by_group(Int4Args const& a, cudaStream_t stream) {
  if (a.group == 32) return by_tiles<T, 1>(a, stream);
  if (a.group == 64) return by_tiles<T, 2>(a, stream);
  return by_tiles<T, 4>(a, stream);
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
  if (by_expert && (slots > kMaxSlots || d->experts > 65534))
    return fail(KL_ERR_NOT_SUPPORTED, "kl_gemv_int4: at most 8192 (token, expert) pairs and 65534 experts (more tokens: kl_moe_plan and the m-grouped GEMM)");
  if (!by_expert && slots > 65535 * 8) return fail(KL_ERR_NOT_SUPPORTED, "kl_gemv_int4: at most 524280 tokens");
  if (d->x_type != KL_BF16 && d->x_type != KL_F16) return fail(KL_ERR_NOT_SUPPORTED, "kl_gemv_int4: x must be bf16 or f16");
  if (d->scale_type != d->x_type && d->scale_type != KL_F32)
    return fail(KL_ERR_NOT_SUPPORTED, "kl_gemv_int4: scales must have x's type or f32");
  if (d->out_type != d->x_type && d->out_type != KL_F32)
    return fail(KL_ERR_NOT_SUPPORTED, "kl_gemv_int4: out must have x's type or f32");
  if (d->group != 32 && d->group != 64 && (d->group < 128 || d->group % 128 != 0))
    return bad("group must be 32, 64 or a multiple of 128");
  if (d->k % 32 != 0) return bad("k must be a multiple of 32");
  if (slots == 0 || d->n == 0) return KL_OK;
  const int64_t groups = (d->k + d->group - 1) / d->group;
  if (d->ldo < d->n || d->ldx < d->k || d->ldq < d->k / 2 || d->ld_scales < groups || (d->zeros != nullptr && d->ld_zeros < groups))
    return bad("row pitch below the row's extent");
  if (d->out == nullptr || (d->k > 0 && (d->x == nullptr || d->q == nullptr || d->scales == nullptr))) return bad("null pointer");
  if (d->k > 0 && (!aligned16(d->x) || !aligned16(d->q) || d->ldx % 8 != 0 || d->ldq % 16 != 0))
    return bad("x and q must be 16-byte aligned with row pitches that are multiples of 16 bytes");
  if (by_expert && d->experts > 1 && (d->stride_q % 16 != 0 || d->stride_q < 0 || d->stride_scales < 0 || d->stride_zeros < 0))
    return bad("expert strides must not be negative, stride_q a multiple of 16 bytes");
  Int4Args a = {};
  a.x = d->x;
  a.ldx = d->ldx;
  a.q = static_cast<const uint8_t*>(d->q);
  a.ldq = d->ldq;
  a.stride_q = d->stride_q;
  a.scales = d->scales;
  a.lds = d->ld_scales;
  a.stride_s = d->stride_scales;
  a.zeros = d->zeros;
  a.ldz = d->ld_zeros;
  a.stride_z = d->stride_zeros;
  a.ids = d->ids;
  a.experts = by_expert ? int(d->experts) : 1;
  a.slots = int(slots);
  a.x_div = by_expert && !d->x_per_slot ? int(topk) : 1;
  a.out = d->out;
  a.ldo = d->ldo;
  a.n = int(d->n);
  a.k = int(d->k);
  a.group = int(d->group);
  a.f32_scales = d->scale_type == KL_F32;
  a.f32_out = d->out_type == KL_F32;
  a.by_slot = by_expert && slots <= d->experts;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = d->x_type == KL_BF16 ? by_group<__nv_bfloat16>(a, s) : by_group<__half>(a, s);
  return e == cudaSuccess ? KL_OK : cuda_fail(e, "kl_gemv_int4 launch");
}
