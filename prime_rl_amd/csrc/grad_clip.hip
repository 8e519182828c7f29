// grad_clip.hip — the gradient norm of many tensors, by group, and clipping: norm_g = sqrt(sum of squares of group g), out = grad * min(1, max_norm / (norm_g + 1e-6)).
//
// A model's adapters are thousands of small tensors: one launch per tensor costs more than reading them.  A table on the device cuts all of them into chunks,
// and three launches do the whole list: squares of each chunk, sums by group, scaling.  All of it is bound by HBM (and, on few small tensors, by the launches): 241 M f32 values of
// 2016 tensors into another buffer take 148 us for the squares (6.5 TB/s), 5 for the sums and 314 for the scaling (6.1 TB/s).
//
// Squares and sums are 64-bit: a float's square overflows 32 bits from 1.8e19 and vanishes below 1e-23, and a sum over 10^9 terms loses digits.  The card does a
// 64-bit multiply-add on each element at several times the rate at which memory delivers them.  Chunks are added in a fixed order: the same gradients give the same norm.
#include "common.hip.h"

namespace pm {
namespace gclip {

typedef __attribute__((address_space(1))) unsigned char global_byte;
struct Chunk {  // one row of the table: int64 [4]; global addresses: the compiler would take others for any kind of memory
  const global_byte* src;
  global_byte* dst;  // null: nothing is written
  int64_t n;
  int64_t flags;  // bit 0: src is bf16, bit 1: dst is bf16, bit 2: src is read past the caches, bit 3: dst is written past them, bits 8 and up: group
};

typedef float f32x4v __attribute__((ext_vector_type(4)));
// outputs start anywhere in a flat buffer: the card takes wide stores at any element (961 MB of 2016 tensors: 545 -> 468 us against one store for each element)
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(2)));
typedef __attribute__((address_space(1))) f32x4_any global_f32x4_any;
typedef __attribute__((address_space(1))) u32x2_any global_u32x2_any;
constexpr int kLoads = 8;  // 16-byte loads of a thread that are in flight together

template <typename T>
using global = __attribute__((address_space(1))) T;

template <bool BF16>
__device__ __forceinline__ float one(const global_byte* p, int64_t i) {
  if constexpr (BF16) return bf16_to_f32(((const global<bf16_t>*)p)[i]);
  else return ((const global<float>*)p)[i];
}
// elements before the first 16-byte boundary
template <bool BF16>
__device__ __forceinline__ int64_t head_of(const global_byte* p, int64_t n) {
  const int64_t h = (int64_t)((16 - ((uintptr_t)p & 15)) & 15) / (BF16 ? 2 : 4);
  return h < n ? h : n;
}

template <bool STREAM, typename T>
__device__ __forceinline__ T load_of(const global<T>* p) {
  if constexpr (STREAM) return __builtin_nontemporal_load(p);
  else return *p;
}

template <bool BF16, bool STREAM>
__device__ __forceinline__ double chunk_squares(const Chunk& c) {
  constexpr int V = BF16 ? 8 : 4;
  const int64_t head = head_of<BF16>(c.src, c.n), vecs = (c.n - head) / V;
  const global<u32x4>* body = (const global<u32x4>*)(c.src + head * (BF16 ? 2 : 4));
  double sum[4] = {0.0, 0.0, 0.0, 0.0};
  auto add = [&](const u32x4& v) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if constexpr (BF16) {
        const double lo = bf16lo(v[q]), hi = bf16hi(v[q]);
        sum[q] = fma(lo, lo, sum[q]);
        sum[q] = fma(hi, hi, sum[q]);
      } else {
        const double x = __uint_as_float(v[q]);
        sum[q] = fma(x, x, sum[q]);
      }
    }
  };
  int64_t i = threadIdx.x;
  for (; i + (kLoads - 1) * 256 < vecs; i += kLoads * 256) {
    u32x4 v[kLoads];
#pragma unroll
    for (int k = 0; k < kLoads; ++k) v[k] = load_of<STREAM, u32x4>(body + i + k * 256);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int k = 0; k < kLoads; ++k) add(v[k]);
  }
  for (; i < vecs; i += 256) add(load_of<STREAM, u32x4>(body + i));
  const int64_t tail = head + vecs * V;
  if (threadIdx.x < head) {
    const double x = one<BF16>(c.src, threadIdx.x);
    sum[0] = fma(x, x, sum[0]);
  }
  if (tail + threadIdx.x < c.n) {
    const double x = one<BF16>(c.src, tail + threadIdx.x);
    sum[1] = fma(x, x, sum[1]);
  }
  return (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

template <int WAVES = 4>
__device__ __forceinline__ double block_sum_f64(double v, double* smem) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  if ((threadIdx.x & 63) == 0) smem[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) s += smem[w];
  return s;
}

__global__ __launch_bounds__(256) void squares_kernel(const Chunk* __restrict__ chunks, double* __restrict__ partials) {
  __shared__ double smem[4];
  const Chunk c = chunks[blockIdx.x];
  double s;
  if (c.flags & 4) s = c.flags & 1 ? chunk_squares<true, true>(c) : chunk_squares<false, true>(c);
  else s = c.flags & 1 ? chunk_squares<true, false>(c) : chunk_squares<false, false>(c);
  s = block_sum_f64(s, smem);
  if (threadIdx.x == 0) partials[blockIdx.x] = s;
}

__device__ __forceinline__ float limit_of(int g, float max_norm, const float* max_norms) { return max_norms ? max_norms[g] : max_norm; }
// as torch's clip_grad_norm_ has it: a norm that is not a number leaves none
__device__ __forceinline__ float coef_of(float norm, float limit) {
  const float c = limit > 0.f ? limit / (norm + 1e-6f) : 1.0f;
  return c > 1.0f ? 1.0f : c;
}
// the sum of the partials [lo, hi)
template <int WAVES>
__device__ __forceinline__ double group_sum(const double* __restrict__ partials, int lo, int hi, double* smem) {
  double s[8] = {};
  for (int i = lo + threadIdx.x; i < hi; i += 8 * WAVES * 64)
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (i + k * WAVES * 64 < hi) s[k] += partials[i + k * WAVES * 64];
  return block_sum_f64<WAVES>(((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7])), smem);
}

// group g's partials are [offsets[g], offsets[g + 1]) (offsets null: one each)
__global__ __launch_bounds__(1024) void coef_kernel(const double* __restrict__ partials, const int32_t* __restrict__ offsets, float max_norm, const float* __restrict__ max_norms,
                                                   double* __restrict__ sumsq, float* __restrict__ norms, float* __restrict__ coefs) {
  __shared__ double smem[16];
  const int g = blockIdx.x;
  const double s = group_sum<16>(partials, offsets ? offsets[g] : g, offsets ? offsets[g + 1] : g + 1, smem);
  if (threadIdx.x) return;
  if (sumsq) sumsq[g] = s;
  if (!norms) return;
  norms[g] = (float)sqrt(s);
  coefs[g] = coef_of(norms[g], limit_of(g, max_norm, max_norms));
}

// Four elements a thread and turn: 16-byte stores in one stretch (32 bits), and one access at a time, which writes faster than a group of loads before a group of stores
// (200 M values f32 -> f32: 5.6 TB/s against 5.3).  Past the caches (where flags say so) both ways: 6.3 TB/s, and squares read 6.7 against 5.8.
template <bool SRC_BF16, bool DST_BF16, bool READ_PAST, bool WRITE_PAST>
__device__ __forceinline__ void scale_chunk(const Chunk& c, float coef) {
  auto put = [&](int64_t i, float x) {
    if constexpr (DST_BF16) ((global<bf16_t>*)c.dst)[i] = f32_to_bf16(x);
    else ((global<float>*)c.dst)[i] = x;
  };
  constexpr int kAlign = SRC_BF16 ? 8 : 16;
  int64_t head = (int64_t)((kAlign - ((uintptr_t)c.src & (kAlign - 1))) & (kAlign - 1)) / (SRC_BF16 ? 2 : 4);
  head = head < c.n ? head : c.n;
  const int64_t vecs = (c.n - head) / 4, tail = head + vecs * 4;
  const global_byte* body = c.src + head * (SRC_BF16 ? 2 : 4);
  global_byte* to = c.dst + head * (DST_BF16 ? 2 : 4);
  for (int64_t i = threadIdx.x; i < vecs; i += 256) {
    f32x4v x;
    if constexpr (SRC_BF16) {
      const u32x2 v = load_of<READ_PAST, u32x2>((const global<u32x2>*)body + i);
      x = f32x4v{bf16lo(v.x), bf16hi(v.x), bf16lo(v.y), bf16hi(v.y)};
    } else {
      x = load_of<READ_PAST, f32x4v>((const global<f32x4v>*)body + i);
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) x[q] *= coef;
    if constexpr (DST_BF16) {
      const u32x2_any v = {pack_bf16_hw(x[0], x[1]), pack_bf16_hw(x[2], x[3])};
      if constexpr (WRITE_PAST) __builtin_nontemporal_store(v, ((global_u32x2_any*)to) + i);
      else ((global_u32x2_any*)to)[i] = v;
    } else {
      if constexpr (WRITE_PAST) __builtin_nontemporal_store((f32x4_any)x, ((global_f32x4_any*)to) + i);
      else ((global_f32x4_any*)to)[i] = x;
    }
  }
  if (threadIdx.x < head) put(threadIdx.x, one<SRC_BF16>(c.src, threadIdx.x) * coef);
  if (tail + threadIdx.x < c.n) put(tail + threadIdx.x, one<SRC_BF16>(c.src, tail + threadIdx.x) * coef);
}

template <bool READ_PAST, bool WRITE_PAST>
__device__ __forceinline__ void scale_any(const Chunk& c, float coef) {
  if (!c.dst || (coef == 1.0f && c.dst == c.src)) return;  // in place, nothing to clip: every value times one is itself
  switch (c.flags & 3) {
    case 0: scale_chunk<false, false, READ_PAST, WRITE_PAST>(c, coef); break;
    case 1: scale_chunk<true, false, READ_PAST, WRITE_PAST>(c, coef); break;
    case 2: scale_chunk<false, true, READ_PAST, WRITE_PAST>(c, coef); break;
    default: scale_chunk<true, true, READ_PAST, WRITE_PAST>(c, coef); break;
  }
}
// The last pieces come first: they were read last and are still in the caches.
__global__ __launch_bounds__(256) void scale_kernel(const Chunk* __restrict__ pieces, const float* __restrict__ coefs) {
  const Chunk c = pieces[gridDim.x - 1 - blockIdx.x];
  const float coef = coefs[c.flags >> 8];
  if (c.flags & 4) scale_any<true, true>(c, coef);
  else if (c.flags & 8) scale_any<false, true>(c, coef);
  else scale_any<false, false>(c, coef);
}
// The same where groups are of few chunks: every workgroup adds up its group's partials itself, which takes less than a launch for it would.  The first workgroups write the
// groups' norms and factors.
__global__ __launch_bounds__(256) void coef_scale_kernel(const Chunk* __restrict__ pieces, int n_groups, const double* __restrict__ partials, const int32_t* __restrict__ offsets,
                                                         float max_norm, const float* __restrict__ max_norms, double* __restrict__ sumsq, float* __restrict__ norms,
                                                         float* __restrict__ coefs) {
  __shared__ double smem[2][4];
  const Chunk c = pieces[blockIdx.x];
  const int own = (int)(c.flags >> 8);
  const float coef = coef_of((float)sqrt(group_sum<4>(partials, offsets[own], offsets[own + 1], smem[0])), limit_of(own, max_norm, max_norms));
  for (int g = blockIdx.x; g < n_groups; g += gridDim.x) {
    __syncthreads();
    const double s = group_sum<4>(partials, offsets[g], offsets[g + 1], smem[1]);
    if (threadIdx.x == 0) {
      if (sumsq) sumsq[g] = s;
      norms[g] = (float)sqrt(s);
      coefs[g] = coef_of(norms[g], limit_of(g, max_norm, max_norms));
    }
  }
  scale_any<false, false>(c, coef);  // few pieces fit the caches
}

}  // namespace gclip
}  // namespace pm

using namespace pm;

extern "C" int pm_grad_clip(const int64_t* chunks, int64_t n_chunks, const int32_t* group_offsets, int32_t n_groups, const int64_t* pieces, int64_t n_pieces, const double* sumsq_in,
                            float max_norm, const float* max_norms, double* partials, double* sumsq_out, float* norms, float* coefs, void* stream) {
  constexpr int64_t kLaunch = (int64_t)1 << 23;  // workgroups of a launch, which holds less than 2^32 threads
  PM_REQUIRE(n_chunks >= 0 && n_chunks < kLaunch && n_pieces >= 0 && n_pieces <= INT32_MAX && n_groups >= 1 && n_groups <= 1 << 20, PM_ERR_INVALID_ARG, "pm_grad_clip: %lld chunks, %lld pieces, %d groups",
             (long long)n_chunks, (long long)n_pieces, n_groups);
  PM_REQUIRE(group_offsets && (n_chunks == 0 || chunks) && (n_pieces == 0 || pieces) && (sumsq_in || n_chunks == 0 || partials), PM_ERR_INVALID_ARG, "pm_grad_clip: null pointer");
  PM_REQUIRE((norms != nullptr) == (coefs != nullptr) && (norms || (sumsq_out && n_pieces == 0)), PM_ERR_INVALID_ARG, "pm_grad_clip: norms and coefs go together, scaling needs them");
  hipStream_t st = as_stream(stream);
  const gclip::Chunk* table = reinterpret_cast<const gclip::Chunk*>(chunks);
  const gclip::Chunk* scaled = reinterpret_cast<const gclip::Chunk*>(pieces);
  if (n_chunks > 0 && !sumsq_in) {
    hipLaunchKernelGGL(gclip::squares_kernel, dim3((unsigned)n_chunks), dim3(256), 0, st, table, partials);
    PM_CHECK_LAUNCH("pm_grad_clip");
  }
  if (n_pieces > 0 && n_pieces <= 2048 && n_chunks <= 2048 && !sumsq_in) {
    hipLaunchKernelGGL(gclip::coef_scale_kernel, dim3((unsigned)n_pieces), dim3(256), 0, st, scaled, n_groups, partials, group_offsets, max_norm, max_norms, sumsq_out, norms, coefs);
    PM_CHECK_LAUNCH("pm_grad_clip");
    return PM_OK;
  }
  hipLaunchKernelGGL(gclip::coef_kernel, dim3(n_groups), dim3(1024), 0, st, sumsq_in ? sumsq_in : partials, sumsq_in ? nullptr : group_offsets, max_norm, max_norms, sumsq_out, norms, coefs);
  PM_CHECK_LAUNCH("pm_grad_clip");
  for (int64_t end = n_pieces; end > 0; end -= kLaunch) {
    const int64_t count = end < kLaunch ? end : kLaunch;
    hipLaunchKernelGGL(gclip::scale_kernel, dim3((unsigned)count), dim3(256), 0, st, scaled + (end - count), coefs);
    PM_CHECK_LAUNCH("pm_grad_clip");
  }
  return PM_OK;
}
