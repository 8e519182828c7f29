// lora.hip — the low-rank updates of many runs' adapters beside a shared projection: forward, backward, and an adapter merged into its projection.
//
// Rows (tokens) sorted by adapter: adapter a owns the positions [offsets[a], offsets[a+1]); position p is row row_ids[p] of the row tensors (row p itself
// without row_ids), so packed runs need no permutation and requests in arrival order need no copy.  With s = scales[a], A = a[a] [r, in], B = b[a] [r, out],
// both rank-major (the factors' long axis is contiguous), every step is one of three products:
//   shrink   z[p, :]  = s * x[row(p), :] . A^T            the long axis is contracted: both operands are K-contiguous, fragments straight from global memory
//   expand   y[row, :] = base[row, :] + z[p, :] . B         the short axis (rank) is contracted; the factor tile is read transposed out of LDS
//   outer    dW[r, c]  = sum_p z[p, r] * t[row(p), c]       the rows are contracted: both operands are read transposed out of LDS (ds_read_b64_tr_b16)
//   forward  = shrink(x, A), expand(base, z, B);   backward: dz = shrink(dy, B), dx = expand(base_dx, dz, A), dB = outer(z, dy), dA = outer(dz, x)
//   merge    = expand(W, s B^T, A) with the rows of W in the place of tokens.
//
// All of it is bound by HBM traffic of the row tensors (2 r operations per 2-byte element, far under the MFMA rate), so each kernel makes one pass over its row
// tensor with 16-byte accesses, and the matrix cores are there to keep the arithmetic out of the way.  From rank 64 on the LDS has as much to do as the memory.  Measured, in the
// kernels' own time, the least of twelve launches (medians of the long ones are up to 25 % above it; a large copy moves 5.7 TB/s, a read past the caches 6.7):
//   shrink  16 384 x 4096 rank 16 23 us = 5.8 TB/s, 32 768 x 12288 rank 64 143 us = 5.6;   expand  16 384 x 6144 rank 16 66 us = 6.1, 32 768 x 4096 rank 64 107 us = 5.0
//   outer   16 384 x 4096 rank 16 27 us = 5.0, with dz 16 384 x 6144 47 us = 4.6 (dz's parts among it), 32 768 x (12288 + 4096) rank 64 217 us = 4.9
//
// Numerics: z and dz are f32 in memory.  Where they feed the matrix cores they are split into bf16 terms that add up to the f32 value: two terms (16 bits)
// in expand, whose result is rounded to bf16 (8 bits) anyway, three terms (24 bits: all of it) in outer, whose results are f32 gradients.  Everything else in
// the products is bf16 by type and every sum is f32, in a fixed order (no atomics: the same inputs give the same bits).
#include "common.hip.h"
#include <type_traits>

namespace pm {
namespace lora {

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8_t;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef short v4i16_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4i16_t* lds_v4i16_ptr;
typedef __attribute__((address_space(3))) void* lds_void_ptr;
typedef __attribute__((address_space(1))) void* glb_void_ptr;

constexpr int kMaxRank = 128;
constexpr int64_t kMaxRows = (int64_t)1 << 28;
constexpr int kExpandRows = 64;  // positions of one adapter per expand tile
constexpr int kOuterCols = 512;  // columns of an outer workgroup

__device__ __forceinline__ f32x4 mfma(const u32x4& a, const u32x4& b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
__device__ __forceinline__ u32x2 tr_read(const unsigned char* p) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16_ptr)p));
}

// The leading bf16 terms of 4 values, which are replaced by what they leave.  An infinite term leaves nothing (not inf - inf).
__device__ __forceinline__ u32x2 take_terms(f32x4& v) {
  const u32x2 t = {pack_bf16_hw(v[0], v[1]), pack_bf16_hw(v[2], v[3])};
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const float lead = q & 1 ? bf16hi(t[q >> 1]) : bf16lo(t[q >> 1]);
    v[q] = __builtin_isfinite(lead) ? v[q] - lead : 0.f;
  }
  return t;
}
__device__ __forceinline__ u32x2 to_bf16(const f32x4& v) { return u32x2{pack_bf16_hw(v[0], v[1]), pack_bf16_hw(v[2], v[3])}; }

// Tile `t` of `rows` positions each -> its adapter and positions [p0, p1).  A tile never straddles two adapters.  Positions outside every adapter (behind the last
// offset, before the first) come after all adapters' tiles as adapter -1.  Offsets are clamped into [0, n] and never run backwards, so no table makes an access out of range.
__device__ __forceinline__ bool locate(const int32_t* __restrict__ offsets, int n_adapters, int n, int rows, int t, int lane, int& adapter, int& p0, int& p1) {
  int base = 0;
  for (int e0 = 0; e0 < n_adapters + 2; e0 += 64) {
    const int e = e0 + lane;
    int lo = 0, hi = 0;
    if (e < n_adapters) {
      lo = min(max(offsets[e], 0), n);
      hi = min(max(offsets[e + 1], lo), n);
    } else if (e == n_adapters) {
      lo = min(max(offsets[n_adapters], 0), n);
      hi = n;
    } else if (e == n_adapters + 1) {
      hi = min(max(offsets[0], 0), n);
    }
    const int tiles = (hi - lo + rows - 1) / rows;
    int incl = tiles;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int up = __shfl_up(incl, o, 64);
      if (lane >= o) incl += up;
    }
    const unsigned long long hit = __ballot(base + incl > t);
    if (hit) {
      const int src = __ffsll((long long)hit) - 1;
      const int first = base + __builtin_amdgcn_readlane(incl, src) - __builtin_amdgcn_readlane(tiles, src);
      adapter = e0 + src < n_adapters ? e0 + src : -1;
      p0 = __builtin_amdgcn_readlane(lo, src) + (t - first) * rows;
      p1 = min(p0 + rows, __builtin_amdgcn_readlane(hi, src));
      return true;
    }
    base += __builtin_amdgcn_readlane(incl, 63);
  }
  return false;
}
// Tiles that any offsets of n positions can need.
static inline int64_t max_tiles(int64_t n, int64_t n_adapters, int64_t rows) {
  const int64_t t = n / rows + n_adapters + 2;
  return t < n ? t : n;
}

// rows of the positions p[0 .. N): the ids are asked for together
template <int N>
__device__ __forceinline__ void rows_of(const int32_t* __restrict__ row_ids, const int (&p)[N], int n, int (&row)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) row[i] = p[i];
  if (row_ids) {
#pragma unroll
    for (int i = 0; i < N; ++i) row[i] = row_ids[p[i]];
#pragma unroll
    for (int i = 0; i < N; ++i) row[i] = min(max(row[i], 0), n - 1);
  }
}

constexpr int kMostParts = 8;
// z of 4 ranks: the sum of the long axis' parts, four of them in flight
__device__ __forceinline__ f32x4 sum_parts(const float* __restrict__ at, int64_t stride, int parts) {
  f32x4 sum = *reinterpret_cast<const f32x4*>(at);
#pragma unroll 1
  for (int q = 1; q < parts; q += 4) {
    f32x4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const f32x4*>(at + min(q + i, parts - 1) * stride);
#pragma unroll
    for (int i = 0; i < 4; ++i) sum += q + i < parts ? v[i] : f32x4{0.f, 0.f, 0.f, 0.f};
  }
  return sum;
}

// ---------------------------------------------------------------------------------------------------------------------
// shrink: z[part][p][r] = scale * sum over the part's columns of t[row(p)][k] * w[adapter][r][k].
// Chunks of columns of a tile's rows and of the factor come into LDS by DMA (global_load_lds: no registers, and one instruction takes whole stretches of a
// row), a ring of mostly three deep, so that two are in flight while the matrix cores work on one.  16-byte slots of a row are permuted by its row number: the 16 rows
// of a fragment read lie in different banks.  The factor's chunk is read once for each tile (from L2), which bounds how small a tile may be.
// What is the same for a wave (its number, the tile) is held as a scalar (readfirstlane, readlane): the waits' switch and the pieces' conditions cost no lanes.
// All tiles run at once and walk the columns together.  Each begins at a chunk of its own: in step they would ask for the same columns of every row, which lie on few
// of the memory channels (reading 32 768 x 4096 this way: 63 us in step, 46 with the turn; a linear read takes 44).
__device__ __forceinline__ void keep_order() { asm volatile("" ::: "memory"); }  // of the memory accesses before and after: what is counted below
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
// at most n DMA instructions of this wave outstanding
__device__ __forceinline__ void wait_dma(int n) {
  switch (n) {
#define PM_CASE(N) case N: asm volatile("s_waitcnt vmcnt(" #N ")" ::: "memory"); break;
    PM_CASE(1) PM_CASE(2) PM_CASE(3) PM_CASE(4) PM_CASE(5) PM_CASE(6) PM_CASE(7) PM_CASE(8) PM_CASE(9) PM_CASE(10)
    PM_CASE(11) PM_CASE(12) PM_CASE(13) PM_CASE(14) PM_CASE(15) PM_CASE(16) PM_CASE(17) PM_CASE(18) PM_CASE(19) PM_CASE(20)
    PM_CASE(21) PM_CASE(22) PM_CASE(23) PM_CASE(24) PM_CASE(25) PM_CASE(26) PM_CASE(27) PM_CASE(28) PM_CASE(29) PM_CASE(30)
    PM_CASE(31) PM_CASE(32) PM_CASE(33) PM_CASE(34) PM_CASE(35) PM_CASE(36) PM_CASE(37) PM_CASE(38) PM_CASE(39) PM_CASE(40)
#undef PM_CASE
    default: asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); break;
  }
}
constexpr int kStream = 2;  // cache policy of an access: do not keep
template <int POLICY>
__device__ __forceinline__ void dma16(const bf16_t* from, unsigned char* to) { __builtin_amdgcn_global_load_lds((glb_void_ptr)from, (lds_void_ptr)to, 16, 0, POLICY); }

// The ring: chunk i of `count` is chunk turn + i of the part's full ones (round and round), the last, shorter one stays last and comes through registers.
// NT + NW instructions of each of WAVES waves fill a chunk: instruction i of t (i < nt) takes tp[i] to to + i * kStep, of w to `wofs` behind that.
template <int KC, int WAVES, int NT, int NW>
struct Ring {
  static constexpr int kStep = WAVES * 1024;
  const bf16_t* tp[NT];  // this lane's 16 bytes of chunk 0
  const bf16_t* wp[NW];
  int tcol[NT], wcol[NW], nt, wofs, c0, full, turn, d;
  bool stream;
  __device__ __forceinline__ void fetch(int c, unsigned char* to, int lane) const {
    if (c < full) {
      const int k = (c0 + (c + turn < full ? c + turn : c + turn - full)) * KC;
      if (stream) {
#pragma unroll
        for (int i = 0; i < NT; ++i)
          if (i < nt) dma16<kStream>(tp[i] + k, to + i * kStep);
      } else {
#pragma unroll
        for (int i = 0; i < NT; ++i)
          if (i < nt) dma16<0>(tp[i] + k, to + i * kStep);
      }
#pragma unroll
      for (int i = 0; i < NW; ++i) dma16<0>(wp[i] + k, to + wofs + i * kStep);
    } else {  // columns past the end are zeros
      const int k = (c0 + c) * KC;
#pragma unroll
      for (int i = 0; i < NT; ++i)
        if (i < nt) *reinterpret_cast<u32x4*>(to + i * kStep + lane * 16) = k + tcol[i] < d ? *reinterpret_cast<const u32x4*>(tp[i] + k) : u32x4{0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < NW; ++i) *reinterpret_cast<u32x4*>(to + wofs + i * kStep + lane * 16) = k + wcol[i] < d ? *reinterpret_cast<const u32x4*>(wp[i] + k) : u32x4{0, 0, 0, 0};
    }
  }
};

// One instruction fills 1 KiB: kPer rows of KC columns.  Instruction i of wave v is piece WAVES i + v.
template <int KC, int WAVES, int NT, int NW>
__device__ __forceinline__ void ring_setup(Ring<KC, WAVES, NT, NW>& ring, const bf16_t* t, int64_t ldt, const bf16_t* w, const int32_t* row_ids, int n, int adapter, int rank, int d, int p0,
                                           int p1, int nt, int rows_lds, int wave, int lane, bool stream) {
  constexpr int kSlots = KC / 8, kPer = 64 / kSlots, kMask = kSlots < 16 ? kSlots - 1 : 15;
  const int sub = lane / kSlots, slot = lane % kSlots;
  int pos[NT], row[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) {  // positions past the tile's end repeat its first row and are not stored
    const int p = p0 + (i * WAVES + wave) * kPer + sub;
    pos[i] = p < p1 ? p : p0;
  }
  rows_of(row_ids, pos, n, row);
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    ring.tcol[i] = (slot ^ (((i * WAVES + wave) * kPer + sub) & kMask)) * 8;
    ring.tp[i] = t + (int64_t)row[i] * ldt + ring.tcol[i];
  }
#pragma unroll
  for (int i = 0; i < NW; ++i) {  // factor rows past the rank repeat the first; what they give is not stored
    const int r = (i * WAVES + wave) * kPer + sub;
    ring.wcol[i] = (slot ^ (r & kMask)) * 8;
    ring.wp[i] = w + ((int64_t)adapter * rank + (r < rank ? r : 0)) * d + ring.wcol[i];
  }
  ring.nt = nt;
  ring.stream = stream;
  ring.wofs = rows_lds * KC * 2;
  ring.d = d;
}

// lane -> z of position lr of 16, ranks 4 lq .. 4 lq + 3
__device__ __forceinline__ void store_z(float* zp, f32x4 v, int p, int p1, int r, int rank, int rp, float scale) {
#pragma unroll
  for (int q = 0; q < 4; ++q) v[q] = r + q < rank ? v[q] * scale : 0.f;
  if (p < p1 && r < rp) *reinterpret_cast<f32x4*>(zp + (int64_t)p * rp + r) = v;
}

// rank <= 16: 32 positions, chunks of 256 columns; the four waves take 64 columns of a chunk each and add their results up through LDS.
constexpr int kNarrowRows = 32, kNarrowChunk = 256, kRing = 3;
__global__ __launch_bounds__(256, 2) void shrink_narrow_kernel(const bf16_t* __restrict__ t, int64_t ldt, const bf16_t* __restrict__ w, const float* __restrict__ scales,
                                                               const int32_t* __restrict__ offsets, const int32_t* __restrict__ row_ids, int n, int n_adapters, int d, int rank,
                                                               int parts, int chunks_per_part, int stream, float* __restrict__ z) {
  constexpr int kRowBytes = kNarrowChunk * 2, kBytes = (kNarrowRows + 16) * kRowBytes;
  __shared__ __attribute__((aligned(1024))) unsigned char lds[kRing * kBytes];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lr = lane & 15, lq = lane >> 4;
  const int part = blockIdx.x % parts, row_tile = blockIdx.x / parts;
  int adapter, p0, p1;
  if (!locate(offsets, n_adapters, n, kNarrowRows, row_tile, lane, adapter, p0, p1) || adapter < 0) return;
  constexpr int NT = kNarrowRows * kRowBytes / 4096, NW = 16 * kRowBytes / 4096;
  Ring<kNarrowChunk, 4, NT, NW> ring;
  ring_setup(ring, t, ldt, w, row_ids, n, adapter, rank, d, p0, p1, NT, kNarrowRows, wave, lane, stream != 0);
  const int c0 = part * chunks_per_part, count = min(chunks_per_part, (d + kNarrowChunk - 1) / kNarrowChunk - c0);
  ring.c0 = c0;
  ring.full = min(count, d / kNarrowChunk - c0);
  ring.turn = ring.full > 0 ? row_tile % ring.full : 0;
  f32x4 acc[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
  unsigned char* mine = lds + wave * 1024;
  for (int c = 0; c < kRing - 1 && c < count; ++c) ring.fetch(c, mine + c * kBytes, lane);
  for (int c = 0, buf = 0; c < count; ++c) {
    // chunk c has landed once at most the next one's are outstanding; where that one came without DMA, or is none, wait for all
    wait_dma(c + 1 < ring.full ? NT + NW : 0);
    lds_barrier();  // chunk c is there for every wave, and every wave is done with chunk c - 1, whose buffer is filled next
    if (c + kRing - 1 < count) ring.fetch(c + kRing - 1, mine + (buf + kRing - 1 < kRing ? buf + kRing - 1 : buf - 1) * kBytes, lane);
    const unsigned char* at = lds + buf * kBytes;
#pragma unroll
    for (int k = 0; k < kNarrowChunk / 128; ++k) {
      const int off = lr * kRowBytes + (((wave * (kNarrowChunk / 128) + k) * 4 + lq) ^ lr) * 16;
      const u32x4 wf = *reinterpret_cast<const u32x4*>(at + kNarrowRows * kRowBytes + off);
#pragma unroll
      for (int i = 0; i < 2; ++i) acc[i] = mfma(wf, *reinterpret_cast<const u32x4*>(at + i * 16 * kRowBytes + off), acc[i]);
    }
    buf = buf + 1 < kRing ? buf + 1 : 0;
  }
  lds_barrier();
  f32x4* red = reinterpret_cast<f32x4*>(lds);
  if (wave > 0)
#pragma unroll
    for (int i = 0; i < 2; ++i) red[((wave - 1) * 2 + i) * 64 + lane] = acc[i];
  lds_barrier();
  if (wave > 0) return;
  const float scale = scales[adapter];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
#pragma unroll
    for (int q = 0; q < 3; ++q) acc[i] += red[(q * 2 + i) * 64 + lane];
    store_z(z + (int64_t)part * n * 16, acc[i], p0 + i * 16 + lr, p1, lq * 4, rank, 16, scale);
  }
}

// rank > 16: `rows` positions (a multiple of 4 up to 192, chosen on the host), chunks of 128 columns, a ring as deep as the LDS takes (2 to 4); of the eight waves four take
// every fourth 16 positions and the first half of a chunk, four the second half, and their results are added up through LDS (two waves on a SIMD wait for LDS in turn).
constexpr int kWideRows = 192, kWideChunk = 128;
template <int RT>
__global__ __launch_bounds__(512) void shrink_wide_kernel(const bf16_t* __restrict__ t, int64_t ldt, const bf16_t* __restrict__ w, const float* __restrict__ scales,
                                                          const int32_t* __restrict__ offsets, const int32_t* __restrict__ row_ids, int n, int n_adapters, int d, int rank, int rp,
                                                          int rows, int depth, int parts, int chunks_per_part, int stream, float* __restrict__ z) {
  constexpr int kRowBytes = kWideChunk * 2, NW = RT / 2;
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lr = lane & 15, lq = lane >> 4;
  const int part = blockIdx.x % parts, row_tile = blockIdx.x / parts;
  int adapter, p0, p1;
  if (!locate(offsets, n_adapters, n, rows, row_tile, lane, adapter, p0, p1) || adapter < 0) return;
  const int nt = (p1 - p0 + 31 - 4 * wave) >> 5;  // instructions of this wave that bring rows, four each; every eighth is its own
  const int held = (rows + 15) & ~15, own = wave & 3, half = wave >> 2;
  Ring<kWideChunk, 8, kWideRows / 32, NW> ring;
  ring_setup(ring, t, ldt, w, row_ids, n, adapter, rank, d, p0, p1, nt, held, wave, lane, stream != 0);
  const int c0 = part * chunks_per_part, count = min(chunks_per_part, (d + kWideChunk - 1) / kWideChunk - c0);
  ring.c0 = c0;
  ring.full = min(count, d / kWideChunk - c0);
  ring.turn = ring.full > 0 ? (int)(blockIdx.x / 32 * 8 + blockIdx.x % 8) % ring.full : 0;
  f32x4 acc[3][RT];
#pragma unroll
  for (int i = 0; i < 3; ++i)
#pragma unroll
    for (int j = 0; j < RT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int bytes = (held + RT * 16) * kRowBytes, newer = (depth - 2) * (nt + NW);
  unsigned char* mine = lds + wave * 1024;
  for (int c = 0; c < depth - 1 && c < count; ++c) ring.fetch(c, mine + c * bytes, lane);
  for (int c = 0, buf = 0; c < count; ++c) {
    wait_dma(c + depth - 2 < ring.full ? newer : 0);
    lds_barrier();
    if (c + depth - 1 < count) ring.fetch(c + depth - 1, mine + (buf > 0 ? buf - 1 : depth - 1) * bytes, lane);
    const unsigned char* at = lds + buf * bytes;
#pragma unroll
    for (int k = 0; k < kWideChunk / 64; ++k) {
      const int off = lr * kRowBytes + ((((half * 2 + k) * 4 + lq) ^ lr) << 4);
      u32x4 wf[RT];
#pragma unroll
      for (int j = 0; j < RT; ++j) wf[j] = *reinterpret_cast<const u32x4*>(at + (held + j * 16) * kRowBytes + off);
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        const int group = i * 4 + own;
        if (group * 16 >= p1 - p0) break;
        const u32x4 tf = *reinterpret_cast<const u32x4*>(at + group * 16 * kRowBytes + off);
#pragma unroll
        for (int j = 0; j < RT; ++j) acc[i][j] = mfma(wf[j], tf, acc[i][j]);
      }
    }
    buf = buf + 1 < depth ? buf + 1 : 0;
  }
  lds_barrier();
  f32x4* red = reinterpret_cast<f32x4*>(lds) + own * 3 * RT * 64;
  if (half)
#pragma unroll
    for (int i = 0; i < 3; ++i)
#pragma unroll
      for (int j = 0; j < RT; ++j) red[(i * RT + j) * 64 + lane] = acc[i][j];
  lds_barrier();
  if (half) return;
  const float scale = scales[adapter];
#pragma unroll
  for (int i = 0; i < 3; ++i)
#pragma unroll
    for (int j = 0; j < RT; ++j)
      store_z(z + (int64_t)part * n * rp, acc[i][j] + red[(i * RT + j) * 64 + lane], p0 + (i * 4 + own) * 16 + lr, p1, j * 16 + lq * 4, rank, rp, scale);
}

// join: grad[adapter][r][c] (+)= the adapter's partials of outer, added in the order of its positions; zero for an adapter without rows.  A block of 256 threads takes 1024 elements.
struct Join {
  const float *part0, *part1;  // of grad_b and grad_a
  float *grad0, *grad1;
  int64_t elems0, elems1;  // of an adapter
  const int32_t* offsets;
  int n, range0, range1, accumulate, per_adapter;  // per_adapter: blocks
};
__device__ __forceinline__ void join(const Join& j, int block) {
  const int g = block / j.per_adapter;
  const int lo = min(max(j.offsets[g], 0), j.n), hi = min(max(j.offsets[g + 1], lo), j.n);
  const int64_t at = ((int64_t)(block % j.per_adapter) * 256 + threadIdx.x) * 4;
  if (at >= j.elems0 + j.elems1) return;
  const bool second = at >= j.elems0;
  const int64_t e = second ? at - j.elems0 : at, elems = second ? j.elems1 : j.elems0;
  const int range = second ? j.range1 : j.range0;
  const float* part = (second ? j.part1 : j.part0) + e;
  float* grad = (second ? j.grad1 : j.grad0) + (int64_t)g * elems + e;
  f32x4 v = j.accumulate ? *reinterpret_cast<const f32x4*>(grad) : f32x4{0.f, 0.f, 0.f, 0.f};
  if (lo < hi) {
    const int last = (hi - 1) / range;
    for (int split = lo / range; split <= last; split += 8) {  // eight at a time in flight
      f32x4 p[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) p[q] = split + q <= last ? *reinterpret_cast<const f32x4*>(part + (int64_t)(split + q + g) * elems) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int q = 0; q < 8; ++q) v += p[q];
    }
  }
  *reinterpret_cast<f32x4*>(grad) = v;
}

// ---------------------------------------------------------------------------------------------------------------------
// expand: out[row][c] = bf16(base[row][c] + sum_r z[p][r] * w[adapter][r][c]).
// Rank <= 64: a workgroup takes 64 positions x 256 columns.  The factor tile [r][256] and z's two bf16 terms go through LDS into fragments; the factor is read transposed
// (ds_read_b64_tr_b16), as the matrix cores' A operand, so that a lane ends up with 8 consecutive columns of one position.  At rank <= 16 both terms of z fit the
// 32-deep contraction of one instruction (its two halves read the same 16 factor rows).
// base is asked for before anything waits.  It and out move row by row (512 bytes of a row and more in one instruction), and the products, 32 positions at a time, come through
// LDS into that order, over the factor tile's place: accesses in the fragments' own order (16 rows x 64 bytes) reach 4.5 TB/s where these reach 5.5 (copies of 16 384 x 6144).
// Column tiles run fastest, so that workgroups that run together cover whole rows (5.5 TB/s against 4.2 with row tiles fastest).
// The backward's last launch is expand with join's blocks behind its own: they fill its end, and the host launches one kernel less.
// Without base the sum starts from zero; rows of no adapter get the base as it is.  kMerge: positions are the rows of a weight, z[p][r] = scale * zb[r][p] (bf16).
enum Expand { kForward, kBackward, kMerge };
template <int RT>
struct ExpandShape {
  static constexpr int kCols = 256;
  static constexpr int kZStride = RT * 32 + (RT == 4 ? 16 : 32);  // bytes of a row of z's terms (rank 64: three workgroups still fit a CU's LDS)
  static constexpr int kStride = kCols * 2 + 32;  // bytes; a row shift of 32 bytes spreads the 8 rows that a transposed read takes at once over all banks
  static constexpr int kSumStride = kCols * 4 + 32;
  static constexpr int kSteps = RT == 1 ? 1 : RT / 2;  // 32-deep contraction steps over the rank
  static constexpr int kTerms = RT == 1 ? 1 : 2;       // bf16 terms that are operands of their own
  static constexpr int kBlocks = kCols / 128;          // 32-column blocks of a wave
  static constexpr int kLanes = kCols / 8;             // lanes that move one row
  static constexpr int kMoves = kCols / 64;            // accesses of a lane for 32 positions
  static constexpr int kZAt = RT * 16 * kStride, kIn = kZAt + 2 * kExpandRows * kZStride, kSums = 32 * kSumStride;
  static constexpr int kLds = kIn > kSums ? kIn : kSums;
};

template <int RT, Expand KIND>
__global__ __launch_bounds__(256, 2) void expand_kernel(const float* __restrict__ z, int parts, float* __restrict__ z_out, const bf16_t* __restrict__ zb, float merge_scale,
                                                        const bf16_t* __restrict__ w, const int32_t* __restrict__ offsets, const int32_t* __restrict__ row_ids, int n,
                                                        int n_adapters, int d, int rank, int rp, const bf16_t* base, int64_t ldb, bf16_t* out, int64_t ldo, int in_place, int stream, unsigned own, Join j) {
  constexpr bool MERGE = KIND == kMerge;
  if constexpr (KIND == kBackward) {
    if (blockIdx.x >= own) {
      join(j, blockIdx.x - own);
      return;
    }
  }
  using S = ExpandShape<RT>;
  __shared__ __attribute__((aligned(16))) unsigned char lds[S::kLds];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lr = lane & 15, lq = lane >> 4;
  const int col_tiles = (d + S::kCols - 1) / S::kCols, row_tile = blockIdx.x / col_tiles, col_tile = blockIdx.x % col_tiles;
  int adapter = 0, p0 = row_tile * kExpandRows, p1 = min(p0 + kExpandRows, n);
  if constexpr (!MERGE) {
    if (!locate(offsets, n_adapters, n, kExpandRows, row_tile, lane, adapter, p0, p1)) return;
    if (adapter < 0 && in_place) return;
  }
  const int c0 = col_tile * S::kCols;
  // the factor tile, rows past the rank and columns past the end as zeros
  constexpr int kPieces = RT * 16 * S::kLanes / 256;
  u32x4 stage[kPieces];
  if (adapter >= 0) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int piece = i * 256 + tid, r = piece / S::kLanes, c = c0 + piece % S::kLanes * 8;
      stage[i] = r < rank && c < d ? *reinterpret_cast<const u32x4*>(w + ((int64_t)adapter * rank + r) * d + c) : u32x4{0, 0, 0, 0};
    }
  }
  // base: move m of half h covers positions 32 h + (m * 4 + wave) * 64 / kLanes + lane / kLanes
  const int mrow = lane / S::kLanes, mcol = lane % S::kLanes * 8, c = c0 + mcol;
  int pos[2 * S::kMoves], row[2 * S::kMoves];
#pragma unroll
  for (int i = 0; i < 2 * S::kMoves; ++i) {
    const int p = p0 + i / S::kMoves * 32 + (i % S::kMoves * 4 + wave) * (64 / S::kLanes) + mrow;
    pos[i] = p < p1 ? p : p0;
  }
  u32x4 bv[2 * S::kMoves];
  auto load_base = [&]() {
    rows_of(row_ids, pos, n, row);
    auto load = [&](auto streams) {
#pragma unroll
      for (int i = 0; i < 2 * S::kMoves; ++i) {
        bv[i] = u32x4{0, 0, 0, 0};
        if (base && c < d && (i < S::kMoves || p1 - p0 > 32)) {
          const u32x4* from = reinterpret_cast<const u32x4*>(base + (int64_t)row[i] * ldb + c);
          if constexpr (decltype(streams)::value) bv[i] = __builtin_nontemporal_load(from);
          else bv[i] = *from;
        }
      }
    };
    if (stream) load(std::true_type{});
    else load(std::false_type{});
  };
  if (parts > 1) load_base();  // adding z's parts up waits for them: the base is asked for first
  // z, split into its two bf16 terms on the way to LDS
  constexpr int kZb = (RT * 2 + 3) / 4;
  f32x4 zv[MERGE ? 1 : RT];  // thread -> 4 ranks of one position, RT times
  u32x4 zbv[kZb];            // merge: 8 positions of one rank
  if constexpr (MERGE) {
#pragma unroll
    for (int i = 0; i < kZb; ++i) {
      const int piece = i * 256 + tid, r = piece >> 3, p = p0 + (piece & 7) * 8;
      zbv[i] = r < rank && p < p1 ? *reinterpret_cast<const u32x4*>(zb + (int64_t)r * n + p) : u32x4{0, 0, 0, 0};
    }
  } else if (adapter >= 0) {
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const int piece = i * 256 + tid, p = p0 + piece / (RT * 4), r = piece % (RT * 4) * 4;
      zv[i] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (p < p1 && r < rp) {
        zv[i] = sum_parts(z + (int64_t)p * rp + r, (int64_t)n * rp, parts);
        if (z_out && col_tile == 0) *reinterpret_cast<f32x4*>(z_out + (int64_t)p * rp + r) = zv[i];
      }
    }
  }
  if (parts <= 1) load_base();
  auto store = [&](int i, const u32x4& v) {
    const int p = p0 + i / S::kMoves * 32 + (i % S::kMoves * 4 + wave) * (64 / S::kLanes) + mrow;
    if (c < d && p < p1) *reinterpret_cast<u32x4*>(out + (int64_t)row[i] * ldo + c) = v;
  };
  if (adapter < 0) {  // rows of no adapter
#pragma unroll
    for (int i = 0; i < 2 * S::kMoves; ++i) store(i, bv[i]);
    return;
  }
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const int piece = i * 256 + tid;
    *reinterpret_cast<u32x4*>(lds + piece / S::kLanes * S::kStride + piece % S::kLanes * 16) = stage[i];
  }
  unsigned char* const lz = lds + S::kZAt;
  constexpr int kTerm = kExpandRows * S::kZStride;
  if constexpr (MERGE) {
#pragma unroll
    for (int i = 0; i < kZb; ++i) {
      const int piece = i * 256 + tid, r = piece >> 3;
      if (r >= RT * 16) break;
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const float v = merge_scale * (q & 1 ? bf16hi(zbv[i][q >> 1]) : bf16lo(zbv[i][q >> 1]));
        f32x4 one = {v, 0.f, 0.f, 0.f};
        const int off = ((piece & 7) * 8 + q) * S::kZStride + r * 2;
        *reinterpret_cast<bf16_t*>(lz + off) = (bf16_t)take_terms(one).x;
        *reinterpret_cast<bf16_t*>(lz + kTerm + off) = f32_to_bf16(one[0]);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const int piece = i * 256 + tid, off = piece / (RT * 4) * S::kZStride + piece % (RT * 4) * 8;
      *reinterpret_cast<u32x2*>(lz + off) = take_terms(zv[i]);
      *reinterpret_cast<u32x2*>(lz + kTerm + off) = to_bf16(zv[i]);
    }
  }
  lds_barrier();
  u32x4 zf[4][S::kSteps][S::kTerms];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int k = 0; k < S::kSteps; ++k) {
      const int off = (i * 16 + lr) * S::kZStride + k * 64 + lq * 8;
      u32x2 v[2][2];
#pragma unroll
      for (int term = 0; term < 2; ++term)
#pragma unroll
        for (int h = 0; h < (RT == 1 ? 1 : 2); ++h) v[term][h] = *reinterpret_cast<const u32x2*>(lz + term * kTerm + off + h * 32);
      if constexpr (RT == 1) {
        zf[i][k][0] = u32x4{v[0][0].x, v[0][0].y, v[1][0].x, v[1][0].y};
      } else {
#pragma unroll
        for (int term = 0; term < 2; ++term) zf[i][k][term < S::kTerms ? term : 0] = u32x4{v[term][0].x, v[term][0].y, v[term][1].x, v[term][1].y};
      }
    }
  // lane (lr, lq) asks for factor row 4 lq + lr / 4 (and 16 more) at columns 8 (lr % 4) + 4 h: lane lr receives column 8 (lr / 4) + 4 h + lr % 4, so the two
  // products h = 0, 1 leave columns 8 lq .. 8 lq + 7 of position lr in one lane
  u32x4 wf[S::kBlocks][S::kSteps][2];
#pragma unroll
  for (int b = 0; b < S::kBlocks; ++b)
#pragma unroll
    for (int k = 0; k < S::kSteps; ++k)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const unsigned char* q = lds + (k * 32 + lq * 4 + (lr >> 2)) * S::kStride + (wave * S::kBlocks + b) * 64 + (lr & 3) * 16 + h * 8;
        const u32x2 lo = tr_read(q), hi = RT == 1 ? lo : tr_read(q + 16 * S::kStride);
        wf[b][k][h] = u32x4{lo.x, lo.y, hi.x, hi.y};
      }
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    if (half && p1 - p0 <= 32) break;
    lds_barrier();  // the fragments, or the last half's sums, have been read
#pragma unroll
    for (int b = 0; b < S::kBlocks; ++b)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        f32x4 acc[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int k = 0; k < S::kSteps; ++k)
#pragma unroll
          for (int term = S::kTerms - 1; term >= 0; --term)  // the small term first
#pragma unroll
            for (int h = 0; h < 2; ++h) acc[h] = mfma(wf[b][k][h], zf[half * 2 + i][k][term], acc[h]);
        f32x4* to = reinterpret_cast<f32x4*>(lds + (i * 16 + lr) * S::kSumStride + ((wave * S::kBlocks + b) * 32 + lq * 8) * 4);
        to[0] = acc[0];
        to[1] = acc[1];
      }
    lds_barrier();
#pragma unroll
    for (int m = 0; m < S::kMoves; ++m) {
      const f32x4* from = reinterpret_cast<const f32x4*>(lds + ((m * 4 + wave) * (64 / S::kLanes) + mrow) * S::kSumStride + mcol * 4);
      const f32x4 sum[2] = {from[0], from[1]};
      const u32x4 v = bv[half * S::kMoves + m];
      u32x4 o;
#pragma unroll
      for (int q = 0; q < 4; ++q) o[q] = pack_bf16_hw(bf16lo(v[q]) + sum[q >> 1][(q & 1) * 2], bf16hi(v[q]) + sum[q >> 1][(q & 1) * 2 + 1]);
      store(half * S::kMoves + m, o);
    }
  }
}

// The same for rank > 64.  There the LDS bounds it, and z's fragments are most of what goes through it: a wave keeps those of 32 positions in registers, straight from memory, and
// takes the factor's tiles of 128 columns one after the other, which the four waves of a workgroup share.  Tiles come by DMA, one ahead; base and out move in the fragments' order.
// 16 384 x 6144 at rank 128: 128 us against 216 in the way of smaller ranks (a copy takes 75); at rank 64 that way is the faster one (32 768 x 4096: 107 us; this way took 164).
constexpr int kDeepRows = 128, kDeepCols = 128;
// the transposed fragments of 64 ranks at 8 columns (two halves of 4): rows of 256 bytes, [2 k][2 halves][16 rows, 16 more].  One block with its own wait: the compiler would wait for
// the tile in flight before such a read.
__device__ __forceinline__ void tr_read_deep(uint32_t a, u32x2 (&v)[8]) {
  asm volatile(
      "ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %8 offset:4096\n\tds_read_b64_tr_b16 %2, %8 offset:8\n\tds_read_b64_tr_b16 %3, %8 offset:4104\n\t"
      "ds_read_b64_tr_b16 %4, %8 offset:8192\n\tds_read_b64_tr_b16 %5, %8 offset:12288\n\tds_read_b64_tr_b16 %6, %8 offset:8200\n\tds_read_b64_tr_b16 %7, %8 offset:12296\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]), "=&v"(v[7])
      : "v"(a)
      : "memory");
}
template <int RT, Expand KIND>
__global__ __launch_bounds__(256, 2) void expand_deep_kernel(const float* __restrict__ z, int parts, float* __restrict__ z_out, const bf16_t* __restrict__ zb, float merge_scale,
                                                             const bf16_t* __restrict__ w, const int32_t* __restrict__ offsets, const int32_t* __restrict__ row_ids, int n,
                                                             int n_adapters, int d, int rank, int rp, const bf16_t* base, int64_t ldb, bf16_t* out, int64_t ldo, int in_place,
                                                             int steps, unsigned own, Join j) {
  if constexpr (KIND == kBackward) {
    if (blockIdx.x >= own) {
      join(j, blockIdx.x - own);
      return;
    }
  }
  constexpr int kRowBytes = kDeepCols * 2, kTile = RT * 16 * kRowBytes, kDma = kTile / 4096, kSteps = RT / 2;
  __shared__ __attribute__((aligned(1024))) unsigned char lds[2 * kTile];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lr = lane & 15, lq = lane >> 4;
  const int all = (d + kDeepCols - 1) / kDeepCols, groups = (all + steps - 1) / steps, row_tile = blockIdx.x / groups, group = blockIdx.x % groups;
  int adapter = 0, p0 = row_tile * kDeepRows, p1 = min(p0 + kDeepRows, n);
  if constexpr (KIND != kMerge) {
    if (!locate(offsets, n_adapters, n, kDeepRows, row_tile, lane, adapter, p0, p1)) return;
    if (adapter < 0 && in_place) return;
  }
  const int first = group * steps, last = min(first + steps, all);
  int pos[2], row[2];
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    const int p = p0 + wave * 32 + g * 16 + lr;
    pos[g] = p < p1 ? p : p0;
  }
  rows_of(row_ids, pos, n, row);
  const bool in[2] = {p0 + wave * 32 + lr < p1, p0 + wave * 32 + 16 + lr < p1};
  if (adapter < 0) {  // rows of no adapter
    for (int c = first * kDeepCols + lq * 8; c < min(last * kDeepCols, d); c += 32)
#pragma unroll
      for (int g = 0; g < 2; ++g)
        if (in[g]) *reinterpret_cast<u32x4*>(out + (int64_t)row[g] * ldo + c) = base ? *reinterpret_cast<const u32x4*>(base + (int64_t)row[g] * ldb + c) : u32x4{0, 0, 0, 0};
    return;
  }
  // a DMA instruction brings 4 rows of 256 bytes; slot pairs of row r are permuted by r % 8.  Rows past the rank repeat the first (z is zero there), columns past the end are not stored.
  const __amdgpu_buffer_rsrc_t factor = __builtin_amdgcn_make_buffer_rsrc(const_cast<bf16_t*>(w + (int64_t)adapter * rank * d), 0, rank * d * 2, 0x00020000);
  auto fetch = [&](int step, unsigned char* to) {
#pragma unroll
    for (int i = 0; i < kDma; ++i) {
      const int r = (i * 4 + wave) * 4 + lq, c = step * kDeepCols + (lr ^ ((r & 7) << 1)) * 8;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(factor, (lds_void_ptr)(to + (i * 4 + wave) * 1024), 16, ((r < rank ? r : 0) * d + (c < d ? c : 0)) * 2, 0, 0, 0);
    }
  };
  fetch(first, lds);
  u32x4 zf[2][kSteps][2];  // two bf16 terms of ranks 32 k + 4 lq .. and 16 more
#pragma unroll
  for (int g = 0; g < 2; ++g)
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      u32x2 term[2][2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = k * 32 + h * 16 + lq * 4;
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
        if constexpr (KIND == kMerge) {
#pragma unroll
          for (int q = 0; q < 4; ++q) v[q] = r + q < rank && in[g] ? merge_scale * bf16_to_f32(zb[(int64_t)(r + q) * n + pos[g]]) : 0.f;
        } else if (r < rp && in[g]) {
          v = sum_parts(z + (int64_t)pos[g] * rp + r, (int64_t)n * rp, parts);
          if (z_out && group == 0) *reinterpret_cast<f32x4*>(z_out + (int64_t)pos[g] * rp + r) = v;
        }
        term[0][h] = take_terms(v);
        term[1][h] = to_bf16(v);
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) zf[g][k][t] = u32x4{term[t][0].x, term[t][0].y, term[t][1].x, term[t][1].y};
    }
  for (int step = first; step < last; ++step) {
    const uint32_t at = (uint32_t)(uintptr_t)(lds_void_ptr)lds + (step - first & 1) * kTile;
    if (step == first) wait_dma(0);  // (the others have been waited for below)
    lds_barrier();  // this tile is there for every wave, and every wave is done with the other one
    if (step + 1 < last) fetch(step + 1, lds + (step + 1 - first & 1) * kTile);
    u32x4 bv[kDeepCols / 32][2];
#pragma unroll
    for (int b = 0; b < kDeepCols / 32; ++b)
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const int c = step * kDeepCols + b * 32 + lq * 8;
        bv[b][g] = base && c < d && in[g] ? *reinterpret_cast<const u32x4*>(base + (int64_t)row[g] * ldb + c) : u32x4{0, 0, 0, 0};
      }
#pragma unroll
    for (int b = 0; b < kDeepCols / 32; ++b) {
      f32x4 acc[2][2] = {};
      const int r = lq * 4 + (lr >> 2), slot = b * 4 + (lr & 3);
      const uint32_t q = at + r * kRowBytes + (((slot >> 1) ^ (r & 7)) << 5) + (slot & 1) * 16;
#pragma unroll
      for (int k = 0; k < kSteps; k += 2) {
        u32x2 v[8];
        tr_read_deep(q + k * 32 * kRowBytes, v);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int t = 1; t >= 0; --t)
#pragma unroll
            for (int g = 0; g < 2; ++g) acc[g][i & 1] = mfma(u32x4{v[2 * i].x, v[2 * i].y, v[2 * i + 1].x, v[2 * i + 1].y}, zf[g][k + i / 2][t], acc[g][i & 1]);
      }
      if (b == 0) wait_dma(0);  // the next tile and the base, before the first store
      const int c = step * kDeepCols + b * 32 + lq * 8;
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        u32x4 o;
#pragma unroll
        for (int q = 0; q < 4; ++q) o[q] = pack_bf16_hw(bf16lo(bv[b][g][q]) + acc[g][q >> 1][(q & 1) * 2], bf16hi(bv[b][g][q]) + acc[g][q >> 1][(q & 1) * 2 + 1]);
        if (c < d && in[g]) *reinterpret_cast<u32x4*>(out + (int64_t)row[g] * ldo + c) = o;
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// shrink and expand in one launch, for few rows (a token or a few for each adapter) and rank <= 64, where launches are what counts: the forward, and the backward's dz and grad_x.
// A workgroup takes up to 16 positions of one adapter and 32 BLOCKS columns of out for each of its eight waves.  It contracts the whole of d_in itself (a wave takes every eighth
// 64 columns, fragments straight from global memory), though all workgroups of the tile do the same: the factor comes from L2 faster than a second launch would start.  Its share of
// the other factor and the base are asked for before that, and each lane adds the waves' results up in the layout that the second product takes.
constexpr int kFewWaves = 8;
template <int RT, int BLOCKS>
__global__ __launch_bounds__(kFewWaves * 64) void few_rows_kernel(const bf16_t* __restrict__ x, int64_t ldx, const bf16_t* __restrict__ a, const bf16_t* __restrict__ b,
                                                                  const float* __restrict__ scales, const int32_t* __restrict__ offsets, const int32_t* __restrict__ row_ids, int n,
                                                                  int n_adapters, int d_in, int d_out, int rank, int rp, const bf16_t* base, int64_t ldb, bf16_t* out, int64_t ldo,
                                                                  int in_place, int groups, float* __restrict__ z) {
  constexpr int W = kFewWaves, U = RT == 1 ? 4 : 2, kSteps = (RT + 1) / 2;
  constexpr int kStride = BLOCKS * 64 + 32;  // bytes of a rank's columns in LDS; the shift as in expand
  __shared__ __attribute__((aligned(16))) f32x4 red[W][RT][64];
  __shared__ __attribute__((aligned(16))) unsigned char lb[W][RT * 16 * kStride];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lr = lane & 15, lq = lane >> 4;
  const int group = blockIdx.x % groups;
  int adapter, p0, p1;
  if (!locate(offsets, n_adapters, n, 16, blockIdx.x / groups, lane, adapter, p0, p1) || (adapter < 0 && in_place)) return;
  const int pos[1] = {p0 + lr < p1 ? p0 + lr : p0};
  int row[1];
  rows_of(row_ids, pos, n, row);
  const int c0 = (group * W + wave) * 32 * BLOCKS;
  u32x4 bv[BLOCKS];
#pragma unroll
  for (int i = 0; i < BLOCKS; ++i) {
    const int c = c0 + i * 32 + lq * 8;
    bv[i] = base && c < d_out ? *reinterpret_cast<const u32x4*>(base + (int64_t)row[0] * ldb + c) : u32x4{0, 0, 0, 0};
  }
  if (adapter < 0) {  // rows of no adapter
#pragma unroll
    for (int i = 0; i < BLOCKS; ++i)
      if (c0 + i * 32 + lq * 8 < d_out && p0 + lr < p1) *reinterpret_cast<u32x4*>(out + (int64_t)row[0] * ldo + c0 + i * 32 + lq * 8) = bv[i];
    return;
  }
  u32x4 stage[RT * BLOCKS];  // this wave's columns of the other factor, ranks past the last as zeros
#pragma unroll
  for (int i = 0; i < RT * BLOCKS; ++i) {
    const int piece = i * 64 + lane, r = piece / (BLOCKS * 4), c = c0 + piece % (BLOCKS * 4) * 8;
    stage[i] = r < rank && c < d_out ? *reinterpret_cast<const u32x4*>(b + ((int64_t)adapter * rank + r) * d_out + c) : u32x4{0, 0, 0, 0};
  }
  const float scale = scales[adapter];
  const bf16_t* xp = x + (int64_t)row[0] * ldx + lq * 8;
  const bf16_t* ap[RT];
#pragma unroll
  for (int j = 0; j < RT; ++j)  // ranks past the last repeat the first; what they give is not used
    ap[j] = a + ((int64_t)adapter * rank + (j * 16 + lr < rank ? j * 16 + lr : 0)) * d_in + lq * 8;
  f32x4 acc[RT];
#pragma unroll
  for (int j = 0; j < RT; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int full = d_in >> 6;
  int s = wave;
  for (; s + W * (U - 1) < full; s += W * U) {
    u32x4 xf[U][2], af[U][2][RT];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        xf[u][h] = *reinterpret_cast<const u32x4*>(xp + (s + W * u) * 64 + h * 32);
#pragma unroll
        for (int j = 0; j < RT; ++j) af[u][h][j] = *reinterpret_cast<const u32x4*>(ap[j] + (s + W * u) * 64 + h * 32);
      }
    __builtin_amdgcn_sched_barrier(0);  // all of them in flight
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < RT; ++j) acc[j] = mfma(af[u][h][j], xf[u][h], acc[j]);
  }
  for (; s * 64 < d_in; s += W) {  // what is left, columns past the end as zeros on both sides
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = s * 64 + h * 32;
      const bool in = k + lq * 8 < d_in;
      const u32x4 xf = in ? *reinterpret_cast<const u32x4*>(xp + k) : u32x4{0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < RT; ++j) acc[j] = mfma(in ? *reinterpret_cast<const u32x4*>(ap[j] + k) : u32x4{0, 0, 0, 0}, xf, acc[j]);
    }
  }
#pragma unroll
  for (int j = 0; j < RT; ++j) red[wave][j][lane] = acc[j];  // position lr, ranks 16 j + 4 lq .. 4 lq + 3
#pragma unroll
  for (int i = 0; i < RT * BLOCKS; ++i) {
    const int piece = i * 64 + lane;
    *reinterpret_cast<u32x4*>(lb[wave] + piece / (BLOCKS * 4) * kStride + piece % (BLOCKS * 4) * 16) = stage[i];
  }
  lds_barrier();
  u32x2 term[2][RT];
#pragma unroll
  for (int j = 0; j < RT; ++j) {
    f32x4 v = red[0][j][lane];
#pragma unroll
    for (int w = 1; w < W; ++w) v += red[w][j][lane];
    const int r = j * 16 + lq * 4;
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] = r + q < rank ? v[q] * scale : 0.f;
    if (group == 0 && wave == 0 && p0 + lr < p1 && r < rp) *reinterpret_cast<f32x4*>(z + (int64_t)(p0 + lr) * rp + r) = v;
    term[0][j] = take_terms(v);
    term[1][j] = to_bf16(v);
  }
#pragma unroll
  for (int i = 0; i < BLOCKS; ++i) {
    f32x4 sum[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int k = 0; k < kSteps; ++k)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const unsigned char* at = lb[wave] + (k * 32 + lq * 4 + (lr >> 2)) * kStride + i * 64 + (lr & 3) * 16 + h * 8;  // column 8 (lr / 4) + 4 h + lr % 4 of the block
        const u32x2 lo = tr_read(at);
        if constexpr (RT == 1) {  // both terms in one instruction
          sum[h] = mfma(u32x4{lo.x, lo.y, lo.x, lo.y}, u32x4{term[0][0].x, term[0][0].y, term[1][0].x, term[1][0].y}, sum[h]);
        } else {
          const u32x2 hi = tr_read(at + 16 * kStride);
#pragma unroll
          for (int t = 1; t >= 0; --t)
            sum[h] = mfma(u32x4{lo.x, lo.y, hi.x, hi.y}, u32x4{term[t][2 * k].x, term[t][2 * k].y, term[t][2 * k + 1].x, term[t][2 * k + 1].y}, sum[h]);
        }
      }
    u32x4 o;
#pragma unroll
    for (int q = 0; q < 4; ++q) o[q] = pack_bf16_hw(bf16lo(bv[i][q]) + sum[q >> 1][(q & 1) * 2], bf16hi(bv[i][q]) + sum[q >> 1][(q & 1) * 2 + 1]);
    const int c = c0 + i * 32 + lq * 8;
    if (c < d_out && p0 + lr < p1) *reinterpret_cast<u32x4*>(out + (int64_t)row[0] * ldo + c) = o;
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// outer: dW[adapter][r][c] = sum over the adapter's positions of z[p][r] * t[row(p)][c].
// Both products of the backward (dB from z and dy, dA from dz and x) are one launch.  A workgroup takes 512 columns and one of equal ranges of positions, whatever
// adapters these belong to: the ranges are cut so that all workgroups run in one round, one on each CU, with the same work each.  At the end of an adapter's positions
// (or of the range) the sum goes to a partial: range s and adapter g meet at most once, and s + g is a number of their own for every pair that meets.
// The positions are the contraction, so both operands are read transposed (ds_read_b64_tr_b16).  Stages of 32 positions go through LDS: t by DMA, a ring of three deep
// (16-byte slot pairs permuted by the row's number, so that the 8 rows of half a transposed read lie in different banks), z through registers, where it is split into
// three bf16 planes.  A wave takes 64 columns and all ranks.
// Bound at rank 16 by memory, less the 4 us until a workgroup's first stage is there; at rank 64 by the LDS and the matrix cores too, of which z's three terms take two thirds (with rows that
// lie in the caches 32 768 x 12288 takes 173 us, without 190).
// DZ (rank <= 16, many rows): the same pass over dy also gives dz, so that dy is read once: the tile's 512 columns are contracted with the factor's (from registers), the
// waves' results are added up through LDS while the next stage runs, and dz comes in one part for each column tile (6 % of the bytes of dy, written and read once).
struct OuterSide {
  const float* z;      // [parts][n][rp]
  int parts;
  const bf16_t* t;     // [*, ldt]
  int64_t ldt;
  int d;
  float* part;         // [ranges + adapters][rank][d]
  int range;           // positions of a workgroup
  const bf16_t* w;     // DZ: the factor and scales of dz
  const float* scales;
  float* dz;           // DZ: [column tiles][n][16]
};
constexpr int kOuterStage = 32, kOuterRing = 3, kOuterIds = 1024;  // kOuterIds: row ids held in LDS at a time

// the transposed fragments of four 16-column blocks (addresses a[0 .. 3]) of a [32][512] tile: rows 4 lq + .., then 16 more.  One block with its own wait: the compiler would
// wait for every DMA in flight before a transposed read through its builtin.
__device__ __forceinline__ void tr_read_tile(const uint32_t (&a)[4], u32x2 (&v)[8]) {
  asm volatile(
      "ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %8 offset:16384\n\t"
      "ds_read_b64_tr_b16 %2, %9\n\tds_read_b64_tr_b16 %3, %9 offset:16384\n\t"
      "ds_read_b64_tr_b16 %4, %10\n\tds_read_b64_tr_b16 %5, %10 offset:16384\n\t"
      "ds_read_b64_tr_b16 %6, %11\n\tds_read_b64_tr_b16 %7, %11 offset:16384\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]), "=&v"(v[7])
      : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3])
      : "memory");
}

// 16 bytes at each of a[0], a[1] and 16 rows on, likewise
__device__ __forceinline__ void read_tile(const uint32_t (&a)[2], u32x4 (&v)[4]) {
  asm volatile("ds_read_b128 %0, %4\n\tds_read_b128 %1, %5\n\tds_read_b128 %2, %4 offset:16384\n\tds_read_b128 %3, %5 offset:16384\n\ts_waitcnt lgkmcnt(0)"
               : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3])
               : "v"(a[0]), "v"(a[1])
               : "memory");
}

template <int RT, bool DZ, int POLICY>
__global__ __launch_bounds__(512) void outer_kernel(OuterSide s0, OuterSide s1, int tiles0, int tiles01, const int32_t* __restrict__ offsets, const int32_t* __restrict__ row_ids, int n,
                                                    int n_adapters, int rank, int rp) {
  static_assert(!DZ || RT == 1, "dz beside dB: one 16-row block of ranks");
  constexpr int SP = kOuterStage, kRowBytes = kOuterCols * 2, kBuf = SP * kRowBytes;
  constexpr int kZs = RT == 1 ? 32 : RT * 32 + 32;  // 32 bytes of shift per row keep transposed reads off each other's banks
  constexpr int kZp = (SP * RT * 4 + 511) / 512;    // 4-rank pieces of z per thread and stage
  constexpr int kDma = SP / 8;                      // instructions of a wave and stage: one row each
  __shared__ __attribute__((aligned(1024))) unsigned char lt[kOuterRing * kBuf];
  __shared__ __attribute__((aligned(16))) unsigned char lz[2][3][SP * kZs];
  __shared__ int li[kOuterIds];
  __shared__ __attribute__((aligned(16))) float lp[DZ ? 2 : 1][DZ ? 8 * SP * 16 : 4];  // dz of a stage, from each wave
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lr = lane & 15, lq = lane >> 4;
  // an XCD (workgroups go round the eight of them) takes neighbouring ranges with all their columns: whole rows, and a range's z once
  const int xcd = blockIdx.x & 7, block = xcd * (int)(gridDim.x >> 3) + min(xcd, (int)(gridDim.x & 7)) + (int)(blockIdx.x >> 3);
  const int split = block / tiles01, col_tile = block % tiles01;
  const bool second = col_tile >= tiles0;
  const OuterSide s = second ? s1 : s0;
  const int c0 = (second ? col_tile - tiles0 : col_tile) * kOuterCols;
  const int begin = split * s.range, end = min(begin + s.range, n);
  // the first adapter whose positions reach past `begin`; lane i holds the offsets of adapter e0 + i
  int g = n_adapters, e0 = 0, from = 0, upto = 0;
  auto look = [&]() { from = offsets[min(e0 + lane, n_adapters)], upto = offsets[min(e0 + lane + 1, n_adapters)]; };
  for (; e0 < n_adapters; e0 += 64) {
    look();
    const unsigned long long hit = __ballot(e0 + lane < n_adapters && upto > begin);
    if (hit) {
      g = e0 + __ffsll((long long)hit) - 1;
      break;
    }
  }
  uint32_t ta[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = lq * 4 + (lr >> 2);
    ta[i] = (uint32_t)(uintptr_t)(lds_void_ptr)lt + row * kRowBytes + (((wave * 4 + i) ^ (row & 7)) << 5) + (lr & 3) * 8;
  }
  int lo = g < n_adapters ? min(max(__builtin_amdgcn_readlane(from, g - e0), begin), end) : end;
  for (; g < n_adapters && lo < end; ++g) {
    if (g - e0 == 64) e0 = g, look();
    const int hi = min(max(__builtin_amdgcn_readlane(upto, g - e0), lo), end);
    if (hi == lo) continue;
    f32x4 acc[4][RT];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < RT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    u32x4 wf[2];
    float scale = 0.f;
    const int wcol = c0 + wave * 64 + lq * 8;
    for (int first = lo, last; first < hi; first = last) {
      last = row_ids ? min(first + kOuterIds, hi) : hi;
      const int stages = (last - first + SP - 1) / SP, full = (last - first) / SP;
      lds_barrier();  // the buffers are free
      if (row_ids) {
        for (int i = tid; i < last - first; i += 512) li[i] = min(max(row_ids[first + i], 0), n - 1);
        lds_barrier();
      }
      // wave w brings rows w, w + 8, ..; slot pairs of row r are permuted by r % 8 = w; columns past the end repeat column 0 and are not stored
      const int src = (lane ^ (wave << 1)) * 8, col = c0 + src < s.d ? c0 + src : 0;
      auto fetch = [&](int st, bool whole) {
        unsigned char* to = lt + st % kOuterRing * kBuf + wave * kRowBytes;
#pragma unroll
        for (int i = 0; i < kDma; ++i) {
          const int p = st * SP + i * 8 + wave;
          if (whole || first + p < last) {
            const int row = row_ids ? __builtin_amdgcn_readfirstlane(li[p]) : first + p;
            // a buffer access: the compiler cannot count past global accesses that write LDS, and would wait for all of them with each z
            const __amdgpu_buffer_rsrc_t from = __builtin_amdgcn_make_buffer_rsrc(const_cast<bf16_t*>(s.t + (int64_t)row * s.ldt), 0, s.d * 2, 0x00020000);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (lds_void_ptr)(to + i * 8 * kRowBytes), 16, col * 2, 0, 0, POLICY);
          } else {  // positions behind the last are zeros on both sides
            *reinterpret_cast<u32x4*>(to + i * 8 * kRowBytes + lane * 16) = u32x4{0, 0, 0, 0};
          }
        }
      };
      auto load_z = [&](int st, f32x4 (&zv)[kZp], int parts) {
#pragma unroll
        for (int i = 0; i < kZp; ++i) {
          const int piece = (i * 512 + tid) % (SP * RT * 4), p = min(first + st * SP + piece / (RT * 4), last - 1), r = min(piece % (RT * 4) * 4, rp - 4);
          zv[i] = sum_parts(s.z + (int64_t)p * rp + r, (int64_t)n * rp, parts);
        }
      };
      auto split_z = [&](int st, f32x4 (&zv)[kZp]) {
#pragma unroll
        for (int i = 0; i < kZp; ++i) {
          const int piece = i * 512 + tid, q = piece / (RT * 4), r = piece % (RT * 4) * 4;
          f32x4 v = first + st * SP + q < last && r < rp ? zv[i] : f32x4{0.f, 0.f, 0.f, 0.f};
          if (piece >= SP * RT * 4) break;
#pragma unroll
          for (int term = 0; term < 3; ++term) *reinterpret_cast<u32x2*>(&lz[st & 1][term][q * kZs + r * 2]) = take_terms(v);
        }
      };
      auto multiply = [&](int st) {
        uint32_t a[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = ta[i] + st % kOuterRing * kBuf;
        u32x2 tv[8];
        tr_read_tile(a, tv);
        // z's fragments are asked for two ahead (the schedule says so: left to itself it waits for each; rank 128 16 384 rows 4096 -> 12288 396 -> 371 us, rank 16 4096 -> 6144 86 -> 84)
        const int zrow = (lq * 4 + (lr >> 2)) * kZs + (lr & 3) * 8;
        constexpr int kAhead = 2, kFragments = RT * 3;
        u32x2 zl[kAhead + 1], zh[kAhead + 1];
        auto ask = [&](int i) {  // fragment i: ranks of block i / 3, term 2 - i % 3
          const unsigned char* q = &lz[st & 1][2 - i % 3][zrow + i / 3 * 32];
          zl[i % (kAhead + 1)] = tr_read(q), zh[i % (kAhead + 1)] = tr_read(q + 16 * kZs);
        };
#pragma unroll
        for (int i = 0; i < kAhead && i < kFragments; ++i) ask(i);
#pragma unroll
        for (int i = 0; i < kFragments; ++i) {
          if (i + kAhead < kFragments) ask(i + kAhead);
          const u32x2 l = zl[i % (kAhead + 1)], h = zh[i % (kAhead + 1)];
          const u32x4 zf = {l.x, l.y, h.x, h.y};
#pragma unroll
          for (int c = 0; c < 4; ++c) acc[c][i / 3] = mfma(u32x4{tv[2 * c].x, tv[2 * c].y, tv[2 * c + 1].x, tv[2 * c + 1].y}, zf, acc[c][i / 3]);
        }
        __builtin_amdgcn_sched_group_barrier(0x100, 2 * (kAhead + 1), 0);
#pragma unroll
        for (int i = 0; i < kFragments; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x8, 4, 0);
          __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        }
      };
      // this wave's 64 columns of dz, 32 positions x 16 ranks; and a value of the last stage's dz from all waves for each thread
      auto contract = [&](int st) {
        const uint32_t at = (uint32_t)(uintptr_t)(lds_void_ptr)lt + st % kOuterRing * kBuf + lr * kRowBytes + (((wave * 8 + lq) ^ ((lr & 7) << 1)) << 4);
        const uint32_t a[2] = {at, at ^ 64};
        u32x4 v[4];
        read_tile(a, v);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int k = 0; k < 2; ++k) sum = mfma(wf[k], wcol + k * 32 < s.d ? v[2 * i + k] : u32x4{0, 0, 0, 0}, sum);
          *reinterpret_cast<f32x4*>(&lp[st & 1][(wave * SP + i * 16 + lr) * 16 + lq * 4]) = sum;
        }
      };
      auto store_dz = [&](int st, bool whole) {
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) sum += lp[st & 1][w * SP * 16 + tid];
        const int p = first + st * SP + (tid >> 4);
        if (whole || p < last) s.dz[((int64_t)col_tile * n + p) * 16 + (tid & 15)] = (tid & 15) < rank ? sum * scale : 0.f;
      };
      if constexpr (DZ) {
        if (first == lo) {
          scale = s.scales[g];
#pragma unroll
          for (int k = 0; k < 2; ++k)
            wf[k] = lr < rank && wcol + k * 32 < s.d ? *reinterpret_cast<const u32x4*>(s.w + ((int64_t)g * rank + lr) * s.d + wcol + k * 32) : u32x4{0, 0, 0, 0};
        }
      }
      // stage st: t comes two stages ahead, z three (it is split one stage ahead)
      f32x4 z0[kZp], za[kZp], zb[kZp];
      int st = 0;
      auto stage = [&](auto steady, f32x4 (&next)[kZp]) {  // `next` holds z of stage st + 1, and gets that of st + 3
        if constexpr (decltype(steady)::value) {
          wait_dma(kDma + kZp + (DZ ? 1 : 0));  // younger than t of this stage: t of the next, z of the one after it, a store of dz
          lds_barrier();
          split_z(st + 1, next);
          if constexpr (DZ)
            if (st > 0) store_dz(st - 1, true);
          fetch(st + 2, true);
          keep_order();
          load_z(st + 3, next, 1);
        } else {
          wait_dma(0);
          lds_barrier();
          if (st + 1 < stages) split_z(st + 1, next);
          if constexpr (DZ)
            if (st > 0) store_dz(st - 1, false);
          if (st + 2 < stages) fetch(st + 2, st + 2 < full);
          if (st + 3 < stages) load_z(st + 3, next, s.parts);
        }
        multiply(st);
        if constexpr (DZ) contract(st);
        ++st;
      };
      // z and t are asked for in the order in which the loop goes on, every time: the compiler takes the least it sees on any way into the loop for the number of accesses younger than a
      // z that it waits for, and would drain everything in every second stage
      if (s.parts == 1 && full > 3) {
        load_z(0, z0, 1);
        keep_order();
        fetch(0, true);
        keep_order();
        load_z(1, zb, 1);
        keep_order();
        fetch(1, true);
        keep_order();
        load_z(2, za, 1);
        split_z(0, z0);
        do {
          stage(std::true_type{}, zb);
          stage(std::true_type{}, za);
        } while (st + 3 < full);
      } else {
        load_z(0, z0, s.parts);
        fetch(0, full > 0);
        load_z(min(1, stages - 1), zb, s.parts);
        if (stages > 1) fetch(1, full > 1);
        load_z(min(2, stages - 1), za, s.parts);
        split_z(0, z0);
      }
      while (st < stages) {
        stage(std::false_type{}, zb);
        if (st < stages) stage(std::false_type{}, za);
      }
      if constexpr (DZ) {
        lds_barrier();
        store_dz(stages - 1, false);
      }
    }
    float* part = s.part + (int64_t)(split + g) * rank * s.d;
#pragma unroll
    for (int j = 0; j < RT; ++j) {
      const int r = j * 16 + lr;
      if (r >= rank) continue;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = c0 + wave * 64 + i * 16 + lq * 4;
        if (c < s.d) *reinterpret_cast<f32x4*>(part + (int64_t)r * s.d + c) = acc[i][j];
      }
    }
    lo = hi;
  }
}

// The same for few rows, where the stages' latency is all there is: a workgroup takes 128 columns and 16 ranks of one adapter, in f32 arithmetic, and writes the gradient itself.  z's rows
// lie in LDS (32 instructions for each position); its waves (four, or one where adapters have few rows each) take eight rows of t in turn, asked for together, and
// their sums are added up through LDS.  64 rows 4096 -> 4096 rank 16, all of the backward in a graph: of one adapter 19.0 us against outer's 22.0 (with one wave 28), of 64 14.8 against 29.1
// (with four waves 21.5); 100 rows of four adapters 16.4 against 23.5, of one 22.4 against 20.3.
constexpr int kFewOuterRows = 128;
struct FewSide {
  const float* z;  // [parts][n][rp]
  int parts;
  const bf16_t* t;
  int64_t ldt;
  int d;
  float* grad;  // [adapters][rank][d]
};
template <int W>
__global__ __launch_bounds__(W * 64) void outer_few_kernel(FewSide s0, FewSide s1, int tiles0, int tiles01, const int32_t* __restrict__ offsets, const int32_t* __restrict__ row_ids, int n,
                                                       int rank, int rp, int accumulate) {
  __shared__ __attribute__((aligned(16))) f32x4 lz[kFewOuterRows][4];
  __shared__ float red[W > 1 ? W - 1 : 1][W > 1 ? 32 : 1][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = blockIdx.y, rank0 = (int)(blockIdx.x / tiles01) * 16, tile = blockIdx.x % tiles01;
  const FewSide s = tile >= tiles0 ? s1 : s0;
  const int c = (tile >= tiles0 ? tile - tiles0 : tile) * 128 + lane * 2;
  const int lo = min(max(offsets[g], 0), n), hi = min(max(offsets[g + 1], lo), n);
  float* const grad = s.grad + ((int64_t)g * rank + rank0) * s.d + c;
  const int ranks = min(16, rank - rank0);
  if (lo == hi) {
    if (!accumulate && c < s.d)
      for (int r = wave; r < ranks; r += W) *reinterpret_cast<float2*>(grad + (int64_t)r * s.d) = float2{0.f, 0.f};
    return;
  }
  for (int i = threadIdx.x; i < (hi - lo) * 4; i += W * 64) lz[i >> 2][i & 3] = sum_parts(s.z + (int64_t)(lo + (i >> 2)) * rp + rank0 + (i & 3) * 4, (int64_t)n * rp, s.parts);
  lds_barrier();
  float acc[16][2];
#pragma unroll
  for (int r = 0; r < 16; ++r) acc[r][0] = acc[r][1] = 0.f;
  const bf16_t* const t = s.t + (c < s.d ? c : 0);
  for (int p = lo + wave * 8; p < hi; p += W * 8) {
    int pos[8], row[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) pos[i] = min(p + i, hi - 1);
    rows_of(row_ids, pos, n, row);
    uint32_t v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = *reinterpret_cast<const uint32_t*>(t + (int64_t)row[i] * s.ldt);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (p + i >= hi) break;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x4 z = lz[p - lo + i][q];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          acc[q * 4 + r][0] = fmaf(z[r], bf16lo(v[i]), acc[q * 4 + r][0]);
          acc[q * 4 + r][1] = fmaf(z[r], bf16hi(v[i]), acc[q * 4 + r][1]);
        }
      }
    }
  }
  if constexpr (W > 1) {
    const int sums = min((hi - lo - 1) >> 3, W - 1);  // waves behind the first that had rows
    if (wave && wave <= sums)
#pragma unroll
      for (int r = 0; r < 32; ++r) red[wave - 1][r][lane] = acc[r >> 1][r & 1];
    lds_barrier();
    if (wave) return;
    for (int w = 0; w < sums; ++w)
#pragma unroll
      for (int r = 0; r < 32; ++r) acc[r >> 1][r & 1] += red[w][r][lane];
  }
  if (c < s.d) {
#pragma unroll
    for (int r = 0; r < 16; ++r)
      if (r < ranks) {
        float2* to = reinterpret_cast<float2*>(grad + (int64_t)r * s.d);
        const float2 old = accumulate ? *to : float2{0.f, 0.f};
        *to = float2{old.x + acc[r][0], old.y + acc[r][1]};
      }
  }
}

// z or dz of 4 ranks: its parts, added in their order (dz may be the first part)
__global__ __launch_bounds__(256) void sum_z_kernel(const float* parts, int count, int64_t elems, float* dz) {
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (at >= elems) return;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  for (int c = 0; c < count; c += 8) {
    f32x4 p[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) p[q] = c + q < count ? *reinterpret_cast<const f32x4*>(parts + (c + q) * elems + at) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int q = 0; q < 8; ++q) v += p[q];
  }
  *reinterpret_cast<f32x4*>(dz + at) = v;
}

__global__ __launch_bounds__(256) void join_kernel(Join j) { join(j, blockIdx.x); }

// ---------------------------------------------------------------------------------------------------------------------
// host side
static inline int rank_tiles(int rank) { return rank <= 16 ? 1 : rank <= 32 ? 2 : rank <= 64 ? 4 : 8; }
static inline int padded_rank(int rank) { return (rank + 15) / 16 * 16; }
constexpr int kLdsBytes = 160 * 1024;  // of a CU
// Row tensors of this many elements are read past the caches (which then keep the factors, z and what is to come): shrink and outer from 24 Mi (forward 16 384 rows 4096 -> 4096 rank
// 16 88 -> 77 us, 32 768 rows 12288 -> 4096 rank 64 287 -> 257; 4096 rows of 4096, read again while they are cached: +3 %), expand's base, which a product may have left there, from 80 Mi (forward
// 16 384 rows 4096 -> 6144 105 -> 98 us, 4096 rows 34 -> 36).
// A weight on its way to another buffer has not been touched before, and streams from 24 Mi as well (12288 x 4096: 40 -> 38 us).
constexpr int64_t kStreamRows = (int64_t)24 << 20, kStreamBase = (int64_t)80 << 20;
// Parts of z are added up by a launch of their own where the column tiles of expand (24 MB) or of outer (2 MB: its stages go on without a pause only over one part) would read more than this
// of them again and again: rank 64, 4096 rows 4096 -> 4096 forward 44 -> 35 us, backward 82 -> 68; rank 16, 1000 rows (8 and 4 MB) forward 15.6 and 18.3, backward 29 -> 27; rank 8, 777 rows
// 1024 -> 2048 (0.4 MB) the same on the card, and the host takes 2.6 us more.
static inline bool sum_first(int64_t n, int rank, int parts, int64_t expand_cols, int64_t outer_cols) {
  const int64_t bytes = n * padded_rank(rank) * 4 * parts;
  return parts > 1 && (bytes * cdiv(expand_cols, 256) > (int64_t)24 << 20 || bytes * cdiv(outer_cols, 512) > (int64_t)2 << 20);
}
static void launch_sum_z(const float* from, int parts, int64_t n, int rank, float* z, hipStream_t stream) {
  const int64_t elems = n * padded_rank(rank);
  hipLaunchKernelGGL(sum_z_kernel, dim3((unsigned)cdiv(elems, 1024)), dim3(256), 0, stream, from, parts, elems, z);
}
static inline int streamed(int64_t n, int64_t d) { return n * d >= kStreamRows ? 1 : 0; }
struct ShrinkPlan {
  int rows, depth, parts, chunks_per_part;
  int64_t tiles;
};
// Narrow: 32 positions a tile; where the tiles are fewer than the 512 workgroups that run at once, the long axis is cut into parts of at least two chunks.  Workgroups that
// all run at once end at very different times (16 384 x 12288: the first at 68, the last at 105 us), so long rows of up to two rounds are cut into parts of 12 chunks and more, which later
// workgroups take where there is room: the forward from 12288 to 4096 columns 158 -> 146 us at 16 384 rows, 91 -> 75 at 8192 (shorter parts or more rounds: no gain).
// Wide: a tile's rows and the parts are chosen together to make the busiest CU's work least: rounds of 256 workgroups (257 tiles of 128 rows take 1.5 times as long as 256) times
// what one moves (its rows and the factor, 256 bytes each in a chunk, and a start as long as 160 of these), and the parts of z, which are written and read again.
static inline ShrinkPlan shrink_plan(int64_t n, int n_adapters, int d, int rank) {
  ShrinkPlan p;
  const bool narrow = rank <= 16;
  const int factor = rank_tiles(rank) * 16, chunks = (int)cdiv(d, narrow ? kNarrowChunk : kWideChunk), most = chunks / 2 < kMostParts ? (chunks / 2 > 1 ? chunks / 2 : 1) : kMostParts;
  auto parts_of = [&](int64_t tiles, int at_once) { return tiles * most <= at_once ? most : tiles < at_once ? (int)(at_once / tiles) : 1; };
  if (narrow) {
    p.rows = kNarrowRows, p.depth = kRing, p.tiles = max_tiles(n, n_adapters, p.rows);
    p.parts = parts_of(p.tiles > 0 ? p.tiles : 1, 512);
    if (p.tiles > 0 && p.tiles <= 1024) {
      const int even = chunks / 12 < 2200 / (int)p.tiles ? chunks / 12 : 2200 / (int)p.tiles;
      p.parts = even > kMostParts ? kMostParts : even > p.parts ? even : p.parts;
    }
  } else {
    double least = 0.0;
    p.rows = 0;
    for (int rows = 16; rows <= kWideRows; rows += rows < 64 ? 16 : 4) {
      const uint32_t worst = ((uint32_t)n + (uint32_t)n_adapters * (uint32_t)(rows - 1)) / (uint32_t)rows, tiles = worst < n ? worst : (uint32_t)n;  // with rows, at most
      const int parts = parts_of(tiles > 0 ? tiles : 1, 256);
      const double cost = (double)((tiles * parts + 255) / 256) * ((rows + factor) * ((chunks + parts - 1) / parts) + 160.0) + (parts > 1 ? tiles * parts * rows * factor / (256.0 * 32.0) : 0.0);
      if (p.rows == 0 || cost <= least) least = cost, p.rows = rows, p.parts = parts;
    }
    const int fit = kLdsBytes / (((p.rows + 15) / 16 * 16 + factor) * kWideChunk * 2);
    p.depth = fit >= 6 ? 3 : fit > 4 ? 4 : fit;
    p.tiles = max_tiles(n, n_adapters, p.rows);
  }
  p.chunks_per_part = (chunks + p.parts - 1) / p.parts;
  return p;
}

// Ranges of positions in outer.  One workgroup fits a CU: what a launch takes goes with its rounds of 256, times what a workgroup moves, in rows of 512 columns
// (1 KiB): its positions, and for each adapter among them a partial (written, and read by the join: 4 rank) and the wait for the first stage (as long as about 96 rows).
static inline int outer_range(int64_t n, int n_adapters, int col_tiles, int rank) {
  double least = 0.0;
  int best = n > 0 ? (int)n : 1;
  for (int rounds = 1; rounds <= 8; ++rounds) {
    int splits = 256 * rounds / col_tiles;  // as many as fill the rounds
    if (splits < 1 && rounds > 1) continue;
    splits = splits < 1 ? 1 : splits > n ? (int)n : splits;
    const int range = splits > 0 ? (int)cdiv(n, splits) : 1, used = range > 0 ? (int)cdiv(n, range) : 1;
    const double cost = (double)((used * col_tiles + 255) / 256) * ((range < 32 ? 32 : range) + (4.0 * rank + 96.0) * (1.0 + (double)n_adapters / (used > 0 ? used : 1)));
    if (rounds == 1 || cost < least) least = cost, best = range > 0 ? range : 1;
  }
  return best;
}

// Few rows: column blocks of a wave (1 or 4) where both products run in one launch, 0 where they take one each.  All workgroups have to run at once, and what each reads of the first
// factor must not be much: the card takes about as long either way (in a graph: 1 row 4096 -> 4096 rank 16 7.9 us against 8.8, 64 rows of 32 adapters 9.0 against 9.9, 64 of one, where the
// card alone is slower this way, 10.9 against 10.4, 32 rows 2048 -> 8192 rank 20 7.7 against 10.2; but 1 row of 12288 columns rank 16 16.8 against 9.1, of 4096 rank 64 19.6 against 12.0), the host less (11.5 us a call
// against 16.3).
static inline int few_rows(int64_t n, int n_adapters, int64_t d_in, int64_t d_out, int rank) {
  if (n > 64 || rank > 64 || rank_tiles(rank) * 16 * d_in > 96 << 10) return 0;
  const int64_t tiles = max_tiles(n, n_adapters, 16);
  return tiles * cdiv(d_out, 32 * kFewWaves) <= 256 ? 1 : rank <= 32 && tiles * cdiv(d_out, 128 * kFewWaves) <= 256 ? 4 : 0;
}
static void launch_few_rows(int blocks, const void* x, int64_t ldx, const void* a, const void* b, const float* scales, const int32_t* offsets, const int32_t* row_ids, int64_t n,
                            int n_adapters, int64_t d_in, int64_t d_out, int rank, const void* base, int64_t ldb, void* out, int64_t ldo, float* z, hipStream_t stream) {
  const int groups = (int)cdiv(d_out, 32 * kFewWaves * blocks);
  auto kernel = rank <= 16 ? (blocks == 1 ? few_rows_kernel<1, 1> : few_rows_kernel<1, 4>) : rank <= 32 ? (blocks == 1 ? few_rows_kernel<2, 1> : few_rows_kernel<2, 4>) : few_rows_kernel<4, 1>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)(max_tiles(n, n_adapters, 16) * groups)), dim3(kFewWaves * 64), 0, stream, (const bf16_t*)x, ldx, (const bf16_t*)a, (const bf16_t*)b, scales,
                     offsets, row_ids, (int)n, n_adapters, (int)d_in, (int)d_out, rank, padded_rank(rank), (const bf16_t*)base, ldb, (bf16_t*)out, ldo, base == out ? 1 : 0, groups, z);
}

template <int RT>
static void launch_shrink(const ShrinkPlan& plan, const void* t, int64_t ldt, const void* w, const float* scales, const int32_t* offsets, const int32_t* row_ids, int64_t n,
                          int n_adapters, int d, int rank, float* z, hipStream_t stream) {
  const dim3 grid((unsigned)(plan.tiles * plan.parts));
  if constexpr (RT == 1)
    hipLaunchKernelGGL(shrink_narrow_kernel, grid, dim3(256), 0, stream, (const bf16_t*)t, ldt, (const bf16_t*)w, scales, offsets, row_ids, (int)n, n_adapters, d, rank, plan.parts,
                       plan.chunks_per_part, streamed(n, d), z);
  else {
    static bool attr_done[64] = {};  // per device: more than 64 KiB of LDS has to be asked for
    int dev = 0;
    (void)hipGetDevice(&dev);
    if (!attr_done[dev & 63]) {
      (void)hipFuncSetAttribute((const void*)shrink_wide_kernel<RT>, hipFuncAttributeMaxDynamicSharedMemorySize, kLdsBytes);
      attr_done[dev & 63] = true;
    }
    const int ring = plan.depth * ((plan.rows + 15) / 16 * 16 + RT * 16) * kWideChunk * 2, sums = 12 * RT * 1024;
    hipLaunchKernelGGL((shrink_wide_kernel<RT>), grid, dim3(512), ring > sums ? ring : sums, stream, (const bf16_t*)t, ldt, (const bf16_t*)w, scales, offsets,
                       row_ids, (int)n, n_adapters, d, rank, padded_rank(rank), plan.rows, plan.depth, plan.parts, plan.chunks_per_part, streamed(n, d), z);
  }
}
template <int RT, Expand KIND>
static void launch_expand(const float* z, int parts, float* z_out, const void* zb, float merge_scale, const void* w, const int32_t* offsets, const int32_t* row_ids, int64_t n,
                          int n_adapters, int d, int rank, const void* base, int64_t ldb, void* out, int64_t ldo, const Join& join, unsigned join_blocks, hipStream_t stream) {
  if constexpr (RT > 4) {
    const int64_t tiles = KIND == kMerge ? cdiv(n, kDeepRows) : max_tiles(n, n_adapters, kDeepRows);
    const int all = (int)cdiv(d, kDeepCols);
    // tiles of columns of a workgroup: the fewest rounds of 512, each as long as the tiles and one more for z (a weight of 6144 x 4096: 42 us, with one tile each 62)
    int steps = 1;
    double least = 0.0;
    for (int k = 1; k <= all && k <= 64; ++k) {
      const double cost = (double)cdiv(tiles * cdiv(all, k), 512) * (k + 1.0);
      if (k == 1 || cost < least) least = cost, steps = k;
    }
    const unsigned grid = (unsigned)(tiles * cdiv(all, steps));
    hipLaunchKernelGGL((expand_deep_kernel<RT, KIND>), dim3(grid + join_blocks), dim3(256), 0, stream, z, parts, z_out, (const bf16_t*)zb, merge_scale, (const bf16_t*)w, offsets, row_ids,
                       (int)n, n_adapters, d, rank, padded_rank(rank), (const bf16_t*)base, ldb, (bf16_t*)out, ldo, base == out ? 1 : 0, steps, grid, join);
  } else {
    const int64_t tiles = KIND == kMerge ? cdiv(n, kExpandRows) : max_tiles(n, n_adapters, kExpandRows);
    const unsigned grid = (unsigned)(tiles * cdiv(d, ExpandShape<RT>::kCols));
    hipLaunchKernelGGL((expand_kernel<RT, KIND>), dim3(grid + join_blocks), dim3(256), 0, stream, z, parts, z_out, (const bf16_t*)zb, merge_scale, (const bf16_t*)w, offsets, row_ids,
                       (int)n, n_adapters, d, rank, padded_rank(rank), (const bf16_t*)base, ldb, (bf16_t*)out, ldo, base == out ? 1 : 0,
                       n * d >= (KIND == kMerge && base != out ? kStreamRows : kStreamBase) ? 1 : 0, grid, join);
  }
}
template <int RT, bool DZ>
static void launch_outer(const OuterSide& s0, const OuterSide& s1, int tiles0, int tiles01, unsigned splits, int stream, const int32_t* offsets, const int32_t* row_ids, int64_t n,
                         int n_adapters, int rank, hipStream_t hip_stream) {
  const dim3 grid(splits * tiles01);
  if (stream)
    hipLaunchKernelGGL((outer_kernel<RT, DZ, kStream>), grid, dim3(512), 0, hip_stream, s0, s1, tiles0, tiles01, offsets, row_ids, (int)n, n_adapters, rank, padded_rank(rank));
  else
    hipLaunchKernelGGL((outer_kernel<RT, DZ, 0>), grid, dim3(512), 0, hip_stream, s0, s1, tiles0, tiles01, offsets, row_ids, (int)n, n_adapters, rank, padded_rank(rank));
}
#define PM_BY_RANK(rank, CALL)          \
  switch (::pm::lora::rank_tiles(rank)) { \
    case 1: { constexpr int RT = 1; CALL; } break; \
    case 2: { constexpr int RT = 2; CALL; } break; \
    case 4: { constexpr int RT = 4; CALL; } break; \
    default: { constexpr int RT = 8; CALL; } break; \
  }

static int check_shape(const char* who, int64_t n, int64_t n_adapters, int64_t d_in, int64_t d_out, int64_t rank) {
  PM_REQUIRE(n >= 0 && n <= kMaxRows, PM_ERR_INVALID_ARG, "%s: n_rows %lld (at most %lld)", who, (long long)n, (long long)kMaxRows);
  PM_REQUIRE(n_adapters >= 1 && n_adapters <= 65535, PM_ERR_INVALID_ARG, "%s: n_adapters %lld (1 .. 65535)", who, (long long)n_adapters);
  PM_REQUIRE(rank >= 1 && rank <= kMaxRank, PM_ERR_UNSUPPORTED, "%s: rank %lld (1 .. %d)", who, (long long)rank, kMaxRank);
  PM_REQUIRE(d_in >= 8 && d_in % 8 == 0 && d_in <= (1 << 22) && d_out >= 8 && d_out % 8 == 0 && d_out <= (1 << 22), PM_ERR_UNSUPPORTED,
             "%s: d_in %lld, d_out %lld (multiples of 8, at most 2^22)", who, (long long)d_in, (long long)d_out);
  return PM_OK;
}
// a launch holds less than 2^32 threads; expand's (and join's behind it) is the largest
static int check_launch(const char* who, int64_t tiles, int64_t d, int rank, int64_t join_elems) {
  const int64_t cols = rank <= 64 ? 256 : 128;
  PM_REQUIRE((tiles * cdiv(d, cols) + join_elems / 1024) * 256 <= UINT32_MAX, PM_ERR_UNSUPPORTED, "%s: too many rows and columns for one call: %lld tiles of %d rows by %lld columns", who,
             (long long)tiles, kExpandRows, (long long)d);
  return PM_OK;
}
static int check_rows(const char* who, const char* name, const void* p, int64_t ld, int64_t d) {
  PM_REQUIRE(p, PM_ERR_INVALID_ARG, "%s: null pointer (%s)", who, name);
  PM_REQUIRE(((uintptr_t)p & 15) == 0 && ld % 8 == 0 && ld >= d, PM_ERR_INVALID_ARG, "%s: %s rows must start 16-byte aligned, %lld elements apart or more (stride %lld)", who, name,
             (long long)d, (long long)ld);
  return PM_OK;
}

// whether two row tensors lie apart as a whole
static bool apart(const void* p, int64_t ldp, int64_t dp, const void* q, int64_t ldq, int64_t dq, int64_t n) {
  const uintptr_t a = (uintptr_t)p, b = (uintptr_t)q;
  return a + ((n - 1) * ldp + dp) * 2 <= b || b + ((n - 1) * ldq + dq) * 2 <= a;
}

}  // namespace lora
}  // namespace pm

using namespace pm;
using namespace pm::lora;

#define PM_TRY(call)              \
  do {                            \
    const int _rc = (call);       \
    if (_rc != PM_OK) return _rc; \
  } while (0)

extern "C" int64_t pm_lora_z_columns(int32_t rank) { return rank >= 1 && rank <= kMaxRank ? padded_rank(rank) : 0; }

extern "C" int64_t pm_lora_fwd_workspace_bytes(int64_t n_rows, int32_t n_adapters, int64_t d_in, int64_t d_out, int32_t rank) {
  if (n_rows <= 0 || rank < 1 || rank > kMaxRank || few_rows(n_rows, n_adapters, d_in, d_out, rank)) return 0;
  const int parts = shrink_plan(n_rows, n_adapters, (int)d_in, rank).parts;
  return parts > 1 ? (int64_t)parts * n_rows * padded_rank(rank) * 4 : 0;
}

extern "C" int pm_lora_fwd(const void* x, int64_t ldx, const void* a, const void* b, const float* scales, const int32_t* offsets, const int32_t* row_ids, int64_t n_rows,
                           int32_t n_adapters, int64_t d_in, int64_t d_out, int32_t rank, const void* base, int64_t ldbase, void* out, int64_t ldout, float* z, void* workspace,
                           int64_t workspace_bytes, void* stream) {
  PM_TRY(check_shape("pm_lora_fwd", n_rows, n_adapters, d_in, d_out, rank));
  if (n_rows == 0) return PM_OK;
  PM_TRY(check_launch("pm_lora_fwd", max_tiles(n_rows, n_adapters, kExpandRows), d_out, rank, 0));
  PM_REQUIRE(a && b && scales && offsets && z, PM_ERR_INVALID_ARG, "pm_lora_fwd: null pointer");
  PM_TRY(check_rows("pm_lora_fwd", "x", x, ldx, d_in));
  PM_TRY(check_rows("pm_lora_fwd", "out", out, ldout, d_out));
  if (base) PM_TRY(check_rows("pm_lora_fwd", "base", base, ldbase, d_out));
  PM_REQUIRE(base != out || ldbase == ldout, PM_ERR_INVALID_ARG, "pm_lora_fwd: base and out are the same rows with different strides");
  PM_REQUIRE((((uintptr_t)a | (uintptr_t)b | (uintptr_t)z) & 15) == 0, PM_ERR_INVALID_ARG, "pm_lora_fwd: a, b and z must be 16-byte aligned");
  const int blocks = few_rows(n_rows, n_adapters, d_in, d_out, rank);
  ShrinkPlan plan = shrink_plan(n_rows, n_adapters, (int)d_in, rank);
  if (blocks) plan.parts = 1, plan.chunks_per_part = (int)cdiv(d_in, rank <= 16 ? kNarrowChunk : kWideChunk);
  const int parts = plan.parts;
  const int64_t need = pm_lora_fwd_workspace_bytes(n_rows, n_adapters, d_in, d_out, rank);
  PM_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0), PM_ERR_WORKSPACE, "pm_lora_fwd: workspace of %lld bytes, %lld needed",
             (long long)workspace_bytes, (long long)need);
  hipStream_t st = as_stream(stream);
  if (blocks && apart(out, ldout, d_out, x, ldx, d_in, n_rows)) {  // every workgroup reads x to the end
    launch_few_rows(blocks, x, ldx, a, b, scales, offsets, row_ids, n_rows, n_adapters, d_in, d_out, rank, base, ldbase, out, ldout, z, st);
    PM_CHECK_LAUNCH("pm_lora_fwd");
    return PM_OK;
  }
  float* zs = parts > 1 ? (float*)workspace : z;
  PM_BY_RANK(rank, (launch_shrink<RT>(plan, x, ldx, a, scales, offsets, row_ids, n_rows, n_adapters, (int)d_in, rank, zs, st)));
  PM_CHECK_LAUNCH("pm_lora_fwd");
  const bool sum = sum_first(n_rows, rank, parts, d_out, 0);
  if (sum) {
    launch_sum_z(zs, parts, n_rows, rank, z, st);
    PM_CHECK_LAUNCH("pm_lora_fwd");
  }
  PM_BY_RANK(rank, (launch_expand<RT, kForward>(sum ? z : zs, sum ? 1 : parts, parts > 1 && !sum ? z : nullptr, nullptr, 0.f, b, offsets, row_ids, n_rows, n_adapters, (int)d_out, rank, base, ldbase, out, ldout, Join{}, 0, st)));
  PM_CHECK_LAUNCH("pm_lora_fwd");
  return PM_OK;
}

namespace {
// dz beside dB in one pass over grad_out pays from about 32 Mi elements of it (rank 16, all of the backward, two passes against one: 4096 rows 4096 -> 4096 48 and 51 us, 8192 rows 76 and
// 74, 4096 rows 4096 -> 12288 76 and 67, 16 384 rows 212 and 171, 32 768 rows 389 and 317).
constexpr int64_t kFusedElements = (int64_t)32 << 20;
static inline int64_t few_tiles(int64_t d_in, int64_t d_out, int rank) { return (cdiv(d_out, 128) + cdiv(d_in, 128)) * (padded_rank(rank) / 16); }
struct BwdPlan {
  bool fused, few;  // few: outer_few
  ShrinkPlan shrink;
  int tiles0, tiles1, range0, range1;
  int64_t dz_bytes, dz_parts_bytes, part0_bytes, part1_bytes;
};
BwdPlan bwd_plan(int64_t n, int n_adapters, int64_t d_in, int64_t d_out, int rank, bool factors) {
  BwdPlan p;
  const int rp = padded_rank(rank);
  p.tiles0 = (int)cdiv(d_out, kOuterCols), p.tiles1 = (int)cdiv(d_in, kOuterCols);
  p.fused = factors && rank <= 16 && n * d_out >= kFusedElements;
  p.shrink = shrink_plan(n, n_adapters, (int)d_out, rank);
  if (p.fused) p.shrink.parts = 1;
  p.few = !p.fused && n <= (n_adapters > 1 ? kFewOuterRows : kFewOuterRows / 2) && few_tiles(d_in, d_out, rank) * n_adapters <= 1 << 20;
  p.range0 = outer_range(n, n_adapters, p.fused ? p.tiles0 : p.tiles0 + p.tiles1, rank);
  p.range1 = p.fused ? outer_range(n, n_adapters, p.tiles1, rank) : p.range0;
  p.dz_bytes = (int64_t)p.shrink.parts * n * rp * 4;
  p.dz_parts_bytes = p.fused ? (int64_t)p.tiles0 * n * rp * 4 : 0;
  p.part0_bytes = factors && !p.few ? (cdiv(n, p.range0) + n_adapters) * rank * d_out * 4 : 0;
  p.part1_bytes = factors && !p.few ? (cdiv(n, p.range1) + n_adapters) * rank * d_in * 4 : 0;
  return p;
}
}  // namespace

extern "C" int64_t pm_lora_bwd_workspace_bytes(int64_t n_rows, int32_t n_adapters, int64_t d_in, int64_t d_out, int32_t rank, int32_t factors) {
  if (n_rows <= 0 || rank < 1 || rank > kMaxRank) return 0;
  const BwdPlan p = bwd_plan(n_rows, n_adapters, d_in, d_out, rank, factors != 0);
  return p.dz_bytes + p.dz_parts_bytes + p.part0_bytes + p.part1_bytes;
}

extern "C" int pm_lora_bwd(const void* grad_out, int64_t ldg, const void* x, int64_t ldx, const float* z, const void* a, const void* b, const float* scales, const int32_t* offsets,
                           const int32_t* row_ids, int64_t n_rows, int32_t n_adapters, int64_t d_in, int64_t d_out, int32_t rank, const void* base, int64_t ldbase, void* grad_x,
                           int64_t ldgx, float* grad_a, float* grad_b, int32_t accumulate, void* workspace, int64_t workspace_bytes, void* stream) {
  PM_TRY(check_shape("pm_lora_bwd", n_rows, n_adapters, d_in, d_out, rank));
  PM_TRY(check_launch("pm_lora_bwd", max_tiles(n_rows, n_adapters, kExpandRows), d_in, rank, n_adapters * (rank * (d_in + d_out) + 1024)));
  PM_REQUIRE((grad_a != nullptr) == (grad_b != nullptr), PM_ERR_INVALID_ARG, "pm_lora_bwd: grad_a and grad_b go together");
  PM_REQUIRE((((uintptr_t)a | (uintptr_t)b | (uintptr_t)z | (uintptr_t)grad_a | (uintptr_t)grad_b) & 15) == 0, PM_ERR_INVALID_ARG,
             "pm_lora_bwd: a, b, z, grad_a and grad_b must be 16-byte aligned");
  PM_REQUIRE(offsets, PM_ERR_INVALID_ARG, "pm_lora_bwd: null pointer");
  if (!grad_x && !grad_a) return PM_OK;  // nothing is wanted
  hipStream_t st = as_stream(stream);
  unsigned char* ws = (unsigned char*)workspace;
  BwdPlan p{};
  p.range0 = p.range1 = 1;
  float *dz = (float*)ws, *dz_parts = nullptr, *part0 = nullptr, *part1 = nullptr;
  int blocks = 0, dz_count = 1;  // of few_rows; parts of dz
  if (n_rows > 0) {
    PM_REQUIRE(a && b && scales, PM_ERR_INVALID_ARG, "pm_lora_bwd: null pointer");
    PM_TRY(check_rows("pm_lora_bwd", "grad_out", grad_out, ldg, d_out));
    if (grad_x) PM_TRY(check_rows("pm_lora_bwd", "grad_x", grad_x, ldgx, d_in));
    if (base) PM_TRY(check_rows("pm_lora_bwd", "base", base, ldbase, d_in));
    PM_REQUIRE(!grad_x || base != grad_x || ldbase == ldgx, PM_ERR_INVALID_ARG, "pm_lora_bwd: base and grad_x are the same rows with different strides");
    if (grad_a) {
      PM_REQUIRE(z, PM_ERR_INVALID_ARG, "pm_lora_bwd: null pointer (z)");
      PM_TRY(check_rows("pm_lora_bwd", "x", x, ldx, d_in));
    }
    p = bwd_plan(n_rows, n_adapters, d_in, d_out, rank, grad_a != nullptr);
    const int64_t need = p.dz_bytes + p.dz_parts_bytes + p.part0_bytes + p.part1_bytes;
    PM_REQUIRE(ws && workspace_bytes >= need && ((uintptr_t)ws & 15) == 0, PM_ERR_WORKSPACE, "pm_lora_bwd: workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
               (long long)need);
    dz_parts = (float*)(ws + p.dz_bytes);
    part0 = (float*)(ws + p.dz_bytes + p.dz_parts_bytes);
    part1 = (float*)(ws + p.dz_bytes + p.dz_parts_bytes + p.part0_bytes);
    // outer reads x and grad_out after grad_x here
    if (grad_x && apart(grad_x, ldgx, d_in, grad_out, ldg, d_out, n_rows) && (!grad_a || apart(grad_x, ldgx, d_in, x, ldx, d_in, n_rows)))
      blocks = few_rows(n_rows, n_adapters, d_out, d_in, rank);
    const bool sum = !blocks && sum_first(n_rows, rank, p.shrink.parts, grad_x ? d_in : 0, grad_a && !p.few ? d_in : 0);
    dz_count = blocks || sum ? 1 : p.shrink.parts;
    const OuterSide s0{z, 1, (const bf16_t*)grad_out, ldg, (int)d_out, part0, p.range0, (const bf16_t*)b, scales, dz_parts};
    const OuterSide s1{dz, dz_count, (const bf16_t*)x, ldx, (int)d_in, part1, p.range1, nullptr, nullptr, nullptr};
    const unsigned splits0 = (unsigned)cdiv(n_rows, p.range0), splits1 = (unsigned)cdiv(n_rows, p.range1);
    if (p.fused) {
      launch_outer<1, true>(s0, s0, p.tiles0, p.tiles0, splits0, streamed(n_rows, d_out), offsets, row_ids, n_rows, n_adapters, rank, st);
      PM_CHECK_LAUNCH("pm_lora_bwd");
      launch_sum_z(dz_parts, p.tiles0, n_rows, rank, dz, st);
      PM_CHECK_LAUNCH("pm_lora_bwd");
      launch_outer<1, false>(s1, s1, p.tiles1, p.tiles1, splits1, streamed(n_rows, d_in), offsets, row_ids, n_rows, n_adapters, rank, st);
      PM_CHECK_LAUNCH("pm_lora_bwd");
    } else {
      if (blocks) {
        launch_few_rows(blocks, grad_out, ldg, b, a, scales, offsets, row_ids, n_rows, n_adapters, d_out, d_in, rank, base, ldbase, grad_x, ldgx, dz, st);
      } else {
        PM_BY_RANK(rank, (launch_shrink<RT>(p.shrink, grad_out, ldg, b, scales, offsets, row_ids, n_rows, n_adapters, (int)d_out, rank, dz, st)));
      }
      PM_CHECK_LAUNCH("pm_lora_bwd");
      if (sum) {
        launch_sum_z(dz, p.shrink.parts, n_rows, rank, dz, st);
        PM_CHECK_LAUNCH("pm_lora_bwd");
      }
      if (grad_a && p.few) {
        const int t0 = (int)cdiv(d_out, 128), t01 = t0 + (int)cdiv(d_in, 128);
        const FewSide f0{z, 1, (const bf16_t*)grad_out, ldg, (int)d_out, grad_b}, f1{dz, dz_count, (const bf16_t*)x, ldx, (int)d_in, grad_a};
        const bool many = n_rows > 8 * n_adapters;
        hipLaunchKernelGGL((many ? outer_few_kernel<4> : outer_few_kernel<1>), dim3((unsigned)few_tiles(d_in, d_out, rank), n_adapters), dim3(many ? 256 : 64), 0, st, f0, f1, t0, t01, offsets, row_ids, (int)n_rows, rank,
                           padded_rank(rank), accumulate);
        PM_CHECK_LAUNCH("pm_lora_bwd");
      } else if (grad_a) {
        PM_BY_RANK(rank, (launch_outer<RT, false>(s0, s1, p.tiles0, p.tiles0 + p.tiles1, splits0, streamed(n_rows, (d_in + d_out) / 2), offsets, row_ids, n_rows, n_adapters, rank, st)));
        PM_CHECK_LAUNCH("pm_lora_bwd");
      }
    }
  }
  Join join{};
  unsigned join_blocks = 0;
  if (grad_a && !p.few) {
    join = Join{part0, part1, grad_b, grad_a, rank * d_out, rank * d_in, offsets, (int)n_rows, p.range0, p.range1, accumulate, (int)cdiv(rank * (d_in + d_out) / 4, 256)};
    join_blocks = (unsigned)join.per_adapter * n_adapters;
  }
  if (n_rows > 0 && grad_x && !blocks) {
    PM_BY_RANK(rank, (launch_expand<RT, kBackward>(dz, dz_count, nullptr, nullptr, 0.f, a, offsets, row_ids, n_rows, n_adapters, (int)d_in, rank, base, ldbase, grad_x, ldgx, join,
                                                   join_blocks, st)));
    PM_CHECK_LAUNCH("pm_lora_bwd");
  } else if (join_blocks) {
    hipLaunchKernelGGL(join_kernel, dim3(join_blocks), dim3(256), 0, st, join);
    PM_CHECK_LAUNCH("pm_lora_bwd");
  }
  return PM_OK;
}

extern "C" int pm_lora_merge(const void* weight, int64_t ldw, const void* a, const void* b, float scale, int64_t d_in, int64_t d_out, int32_t rank, void* out, int64_t ldo,
                             void* stream) {
  PM_TRY(check_shape("pm_lora_merge", d_out, 1, d_in, d_out, rank));
  PM_TRY(check_launch("pm_lora_merge", cdiv(d_out, kExpandRows), d_in, rank, 0));
  PM_REQUIRE(a && b, PM_ERR_INVALID_ARG, "pm_lora_merge: null pointer");
  PM_REQUIRE((((uintptr_t)a | (uintptr_t)b) & 15) == 0, PM_ERR_INVALID_ARG, "pm_lora_merge: a and b must be 16-byte aligned");
  PM_TRY(check_rows("pm_lora_merge", "weight", weight, ldw, d_in));
  PM_TRY(check_rows("pm_lora_merge", "out", out, ldo, d_in));
  PM_BY_RANK(rank, (launch_expand<RT, kMerge>(nullptr, 0, nullptr, b, scale, a, nullptr, nullptr, d_out, 1, (int)d_in, rank, weight, ldw, out, ldo, Join{}, 0, as_stream(stream))));
  PM_CHECK_LAUNCH("pm_lora_merge");
  return PM_OK;
}
