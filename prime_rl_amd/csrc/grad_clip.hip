// grad_clip.hip — the gradient norm of many tensors, by group, and clipping: norm_g = sqrt(sum of squares of group g), out = grad * min(1, max_norm / (norm_g + 1e-6)).
//
// A model's adapters are thousands of small tensors: one launch per tensor costs more than reading them.  A table on the device cuts all of them into chunks,
// and three launches do the whole list: squares of each chunk, sums by group, scaling.  All of it is bound by HBM (and, on few small tensors, by the launches).
//
// Squares and sums are 64-bit: a float's square overflows 32 bits from 1.8e19 and vanishes below 1e-23, and a sum over 10^9 terms loses digits.  The card does a
// 64-bit multiply-add on each element at several times the rate at which memory delivers them.  Chunks are added in a fixed order: the same gradients give the same norm.
#include "common.hip.h"

namespace pm {
namespace gclip {

struct Chunk {  // one row of the table: int64 [4]
  const unsigned char* src;
  unsigned char* dst;  // null: nothing is written
  int64_t n;
  int64_t flags;  // bit 0: src is bf16, bit 1: dst is bf16, bits 8 and up: group
};

typedef float f32x4v __attribute__((ext_vector_type(4)));

template <bool BF16>
__device__ __forceinline__ float one(const unsigned char* p, int64_t i) {
  if constexpr (BF16) return bf16_to_f32(reinterpret_cast<const bf16_t*>(p)[i]);
  else return reinterpret_cast<const float*>(p)[i];
}
// elements before the first 16-byte boundary
template <bool BF16>
__device__ __forceinline__ int64_t head_of(const unsigned char* p, int64_t n) {
  const int64_t h = (int64_t)((16 - ((uintptr_t)p & 15)) & 15) / (BF16 ? 2 : 4);
  return h < n ? h : n;
}

template <bool BF16>
__device__ __forceinline__ double chunk_squares(const Chunk& c) {
  constexpr int V = BF16 ? 8 : 4;
  const int64_t head = head_of<BF16>(c.src, c.n), vecs = (c.n - head) / V;
  const u32x4* body = reinterpret_cast<const u32x4*>(c.src + head * (BF16 ? 2 : 4));
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
  for (; i + 3 * 256 < vecs; i += 4 * 256) {
    const u32x4 a = body[i], b = body[i + 256], d = body[i + 512], e = body[i + 768];
    add(a), add(b), add(d), add(e);
  }
  for (; i < vecs; i += 256) add(body[i]);
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

__device__ __forceinline__ double block_sum_f64(double v, double* smem) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  if ((threadIdx.x & 63) == 0) smem[threadIdx.x >> 6] = v;
  __syncthreads();
  return (smem[0] + smem[1]) + (smem[2] + smem[3]);
}

__global__ __launch_bounds__(256) void squares_kernel(const Chunk* __restrict__ chunks, double* __restrict__ partials) {
  __shared__ double smem[4];
  const Chunk c = chunks[blockIdx.x];
  const double s = block_sum_f64(c.flags & 1 ? chunk_squares<true>(c) : chunk_squares<false>(c), smem);
  if (threadIdx.x == 0) partials[blockIdx.x] = s;
}

__device__ __forceinline__ float limit_of(int g, float max_norm, const float* max_norms) { return max_norms ? max_norms[g] : max_norm; }
// as torch's clip_grad_norm_ has it: a norm that is not a number leaves none
__device__ __forceinline__ float coef_of(float norm, float limit) {
  const float c = limit > 0.f ? limit / (norm + 1e-6f) : 1.0f;
  return c > 1.0f ? 1.0f : c;
}
// the sum of group g's partials, [lo, hi), in one order wherever it is taken
__device__ __forceinline__ double group_sum(const double* __restrict__ partials, int lo, int hi, double* smem) {
  double s = 0.0;
  for (int i = lo + threadIdx.x; i < hi; i += 256) s += partials[i];
  return block_sum_f64(s, smem);
}

// group g's partials are [offsets[g], offsets[g + 1]) (offsets null: one each)
__global__ __launch_bounds__(256) void coef_kernel(const double* __restrict__ partials, const int32_t* __restrict__ offsets, float max_norm, const float* __restrict__ max_norms,
                                                   double* __restrict__ sumsq, float* __restrict__ norms, float* __restrict__ coefs) {
  __shared__ double smem[4];
  const int g = blockIdx.x;
  const double s = group_sum(partials, offsets ? offsets[g] : g, offsets ? offsets[g + 1] : g + 1, smem);
  if (threadIdx.x) return;
  if (sumsq) sumsq[g] = s;
  if (!norms) return;
  norms[g] = (float)sqrt(s);
  coefs[g] = coef_of(norms[g], limit_of(g, max_norm, max_norms));
}

template <bool SRC_BF16, bool DST_BF16>
__device__ __forceinline__ void scale_chunk(const Chunk& c, float coef) {
  constexpr int V = SRC_BF16 ? 8 : 4;
  auto put = [&](int64_t i, float x) {
    if constexpr (DST_BF16) reinterpret_cast<bf16_t*>(c.dst)[i] = f32_to_bf16(x);
    else reinterpret_cast<float*>(c.dst)[i] = x;
  };
  const int64_t head = head_of<SRC_BF16>(c.src, c.n), vecs = (c.n - head) / V, tail = head + vecs * V;
  const u32x4* body = reinterpret_cast<const u32x4*>(c.src + head * (SRC_BF16 ? 2 : 4));
  unsigned char* to = c.dst + head * (DST_BF16 ? 2 : 4);
  const bool aligned = ((uintptr_t)to & 15) == 0;
  auto store = [&](int64_t i, const u32x4& v) {
    float x[V];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if constexpr (SRC_BF16) {
        x[2 * q] = bf16lo(v[q]) * coef;
        x[2 * q + 1] = bf16hi(v[q]) * coef;
      } else {
        x[q] = __uint_as_float(v[q]) * coef;
      }
    }
    if (!aligned) {
#pragma unroll
      for (int q = 0; q < V; ++q) put(head + i * V + q, x[q]);
    } else if constexpr (DST_BF16) {
      uint32_t o[V / 2];
#pragma unroll
      for (int q = 0; q < V / 2; ++q) o[q] = pack_bf16_hw(x[2 * q], x[2 * q + 1]);
      if constexpr (V == 8) reinterpret_cast<u32x4*>(to)[i] = u32x4{o[0], o[1], o[2], o[3]};
      else reinterpret_cast<u32x2*>(to)[i] = u32x2{o[0], o[1]};
    } else {
#pragma unroll
      for (int q = 0; q < V / 4; ++q) reinterpret_cast<f32x4v*>(to)[i * (V / 4) + q] = f32x4v{x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]};
    }
  };
  int64_t i = threadIdx.x;
  for (; i + 3 * 256 < vecs; i += 4 * 256) {
    const u32x4 a = body[i], b = body[i + 256], d = body[i + 512], e = body[i + 768];
    store(i, a), store(i + 256, b), store(i + 512, d), store(i + 768, e);
  }
  for (; i < vecs; i += 256) store(i, body[i]);
  if (threadIdx.x < head) put(threadIdx.x, one<SRC_BF16>(c.src, threadIdx.x) * coef);
  if (tail + threadIdx.x < c.n) put(tail + threadIdx.x, one<SRC_BF16>(c.src, tail + threadIdx.x) * coef);
}

__device__ __forceinline__ void scale_any(const Chunk& c, float coef) {
  if (!c.dst || (coef == 1.0f && c.dst == c.src)) return;  // in place, nothing to clip: every value times one is itself
  switch (c.flags & 3) {
    case 0: scale_chunk<false, false>(c, coef); break;
    case 1: scale_chunk<true, false>(c, coef); break;
    case 2: scale_chunk<false, true>(c, coef); break;
    default: scale_chunk<true, true>(c, coef); break;
  }
}
// the last chunks first: they were read last and are still in the caches
__global__ __launch_bounds__(256) void scale_kernel(const Chunk* __restrict__ chunks, const float* __restrict__ coefs) {
  const Chunk c = chunks[gridDim.x - 1 - blockIdx.x];
  scale_any(c, coefs[c.flags >> 8]);
}
// The same where groups are of few chunks: every workgroup adds up its group's partials itself, which takes less than a launch for it would.  The first workgroups write the
// groups' norms and factors.
__global__ __launch_bounds__(256) void coef_scale_kernel(const Chunk* __restrict__ chunks, int n_groups, const double* __restrict__ partials, const int32_t* __restrict__ offsets,
                                                         float max_norm, const float* __restrict__ max_norms, double* __restrict__ sumsq, float* __restrict__ norms,
                                                         float* __restrict__ coefs) {
  __shared__ double smem[2][4];
  const Chunk c = chunks[blockIdx.x];
  const int own = (int)(c.flags >> 8);
  const float coef = coef_of((float)sqrt(group_sum(partials, offsets[own], offsets[own + 1], smem[0])), limit_of(own, max_norm, max_norms));
  for (int g = blockIdx.x; g < n_groups; g += gridDim.x) {
    __syncthreads();
    const double s = group_sum(partials, offsets[g], offsets[g + 1], smem[1]);
    if (threadIdx.x == 0) {
      if (sumsq) sumsq[g] = s;
      norms[g] = (float)sqrt(s);
      coefs[g] = coef_of(norms[g], limit_of(g, max_norm, max_norms));
    }
  }
  scale_any(c, coef);
}

}  // namespace gclip
}  // namespace pm

using namespace pm;

extern "C" int pm_grad_clip(const int64_t* chunks, int64_t n_chunks, const int32_t* group_offsets, int32_t n_groups, const double* sumsq_in, float max_norm, const float* max_norms,
                            double* partials, double* sumsq_out, float* norms, float* coefs, int32_t scale, void* stream) {
  PM_REQUIRE(n_chunks >= 0 && n_chunks <= INT32_MAX && n_groups >= 1, PM_ERR_INVALID_ARG, "pm_grad_clip: %lld chunks, %d groups", (long long)n_chunks, n_groups);
  PM_REQUIRE(group_offsets && (n_chunks == 0 || chunks) && (sumsq_in || n_chunks == 0 || partials), PM_ERR_INVALID_ARG, "pm_grad_clip: null pointer");
  PM_REQUIRE((norms != nullptr) == (coefs != nullptr) && (norms || (sumsq_out && !scale)), PM_ERR_INVALID_ARG, "pm_grad_clip: norms and coefs go together, scaling needs them");
  hipStream_t st = as_stream(stream);
  const gclip::Chunk* table = reinterpret_cast<const gclip::Chunk*>(chunks);
  if (n_chunks > 0 && !sumsq_in) {
    hipLaunchKernelGGL(gclip::squares_kernel, dim3((unsigned)n_chunks), dim3(256), 0, st, table, partials);
    PM_CHECK_LAUNCH("pm_grad_clip");
  }
  if (scale && !sumsq_in && n_chunks > 0 && n_chunks <= 1024) {
    hipLaunchKernelGGL(gclip::coef_scale_kernel, dim3((unsigned)n_chunks), dim3(256), 0, st, table, n_groups, partials, group_offsets, max_norm, max_norms, sumsq_out, norms, coefs);
    PM_CHECK_LAUNCH("pm_grad_clip");
    return PM_OK;
  }
  hipLaunchKernelGGL(gclip::coef_kernel, dim3(n_groups), dim3(256), 0, st, sumsq_in ? sumsq_in : partials, sumsq_in ? nullptr : group_offsets, max_norm, max_norms, sumsq_out, norms, coefs);
  PM_CHECK_LAUNCH("pm_grad_clip");
  if (scale && n_chunks > 0) {
    hipLaunchKernelGGL(gclip::scale_kernel, dim3((unsigned)n_chunks), dim3(256), 0, st, table, coefs);
    PM_CHECK_LAUNCH("pm_grad_clip");
  }
  return PM_OK;
}
