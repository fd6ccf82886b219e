// MXFP4 experts: quantisation, read-back and the two expert products with
// both operands in microscaled 4-bit floating point.
//
// Format.  Blocks of 32 consecutive elements of a row share the scale 2^e,
// e = clamp(floor(log2 max|x|) - 2, -127, 127), stored as the byte e + 127;
// an element is x / 2^e rounded to the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6
// (ties to the even code, saturating at 6) with a sign bit, two codes per byte,
// the first element in the low half.  A block that holds an infinity or a NaN
// has the byte 255 (NaN) and reads back as NaN.  Scale bytes are stored in the
// tiles the tensor core's scale copy reads: 128 rows x 4 blocks = 512 bytes,
// row r, block b of the tile at (r % 32) * 16 + (r / 32) * 4 + b; a matrix is
// [row tiles][block tiles][512], zero past its rows and blocks.  Rows grouped
// in segments (one per expert) start a row tile at every segment.
//
// x / 2^e is exact in fp32 (a power of two), so quantising is one rounding,
// and a stored value is exact in bf16; the products accumulate in fp32.
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"
#include "tmap.h"

namespace mirai {
namespace mx {

constexpr int kMaxSegs = 1024;
constexpr int kBlockRows = 128;  // rows of a scale tile

__host__ __device__ inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// ----------------------------------------------------------------------------
// quantisation

// Scale byte of a block from the largest |x| as fp32 bits (integer order is
// magnitude order, NaN above infinity): e + 127 = exponent field - 2.
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax_bits) {
  const uint32_t field = amax_bits >> 23;
  return field == 255u ? 255u : (field > 2u ? field - 2u : 0u);
}
__device__ __forceinline__ float inv_scale(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }

// Eight values already divided by their scale -> eight codes (first in the low bits).
__device__ __forceinline__ uint32_t e2m1x8(const float (&v)[8]) {
  uint32_t r;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}

template <typename T> struct Raw8 { uint4 a; };  // eight 16-bit values
template <> struct Raw8<float> { uint4 a, b; };

template <typename T> __device__ __forceinline__ void load8(const T* p, Raw8<T>& r) {
  r.a = __ldg(reinterpret_cast<const uint4*>(p));
  if constexpr (sizeof(T) == 4) r.b = __ldg(reinterpret_cast<const uint4*>(p) + 1);
}
template <typename T> __device__ __forceinline__ void zero8(Raw8<T>& r) {
  r.a = make_uint4(0, 0, 0, 0);
  if constexpr (sizeof(T) == 4) r.b = r.a;
}
__device__ __forceinline__ void unpack8(const Raw8<__nv_bfloat16>& r, float (&v)[8]) {
  const uint32_t w[4] = {r.a.x, r.a.y, r.a.z, r.a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) v[2 * i] = bf16_lo(w[i]), v[2 * i + 1] = bf16_hi(w[i]);
}
__device__ __forceinline__ void unpack8(const Raw8<__half>& r, float (&v)[8]) {
  const uint32_t w[4] = {r.a.x, r.a.y, r.a.z, r.a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    v[2 * i] = f.x, v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void unpack8(const Raw8<float>& r, float (&v)[8]) {
  v[0] = __uint_as_float(r.a.x), v[1] = __uint_as_float(r.a.y), v[2] = __uint_as_float(r.a.z);
  v[3] = __uint_as_float(r.a.w), v[4] = __uint_as_float(r.b.x), v[5] = __uint_as_float(r.b.y);
  v[6] = __uint_as_float(r.b.z), v[7] = __uint_as_float(r.b.w);
}

// Rows [begin, begin + rows) of segment g.  Ends outside [0, S] or below the
// segment's beginning are recorded and clamped, so no row index leaves [0, S).
__device__ __forceinline__ int segment_rows(const int32_t* __restrict__ offsets, int g, int64_t S, int& begin,
                                            int site) {
  const int64_t end = offsets[g];
  const int64_t beg = g > 0 ? offsets[g - 1] : 0;
  if (end < beg || end > S || beg < 0) device_fail(MIRAI_ERR_DEVICE_BOUNDS, site);
  const int64_t b = beg < 0 ? 0 : (beg > S ? S : beg);
  const int64_t e = end < b ? b : (end > S ? S : end);
  begin = (int)b;
  return (int)(e - b);
}

struct RowBlock {
  int64_t row0;  // first row of the block
  int rows;      // its rows (1..128), 0: no such block
};

// Row block `blk` of rows in segments (each starts a new block): every thread
// of a 256-thread CTA takes four segments, the CTA scans their block counts.
__device__ __forceinline__ RowBlock find_block(const int32_t* __restrict__ offsets, int nseg, int64_t S, int blk) {
  __shared__ int warp_sum[8];
  __shared__ RowBlock found;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int begin[4], rows[4], sum = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int g = threadIdx.x * 4 + i;
    begin[i] = rows[i] = 0;
    if (g < nseg) rows[i] = segment_rows(offsets, g, S, begin[i], 700);
    sum += (rows[i] + kBlockRows - 1) / kBlockRows;
  }
  int incl = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) warp_sum[warp] = incl;
  if (threadIdx.x == 0) found = RowBlock{0, 0};
  __syncthreads();
  int base = incl - sum;
  for (int w = 0; w < warp; ++w) base += warp_sum[w];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int n = (rows[i] + kBlockRows - 1) / kBlockRows;
    if (blk >= base && blk < base + n) {
      const int r = (blk - base) * kBlockRows;
      found = RowBlock{(int64_t)begin[i] + r, min(kBlockRows, rows[i] - r)};
    }
    base += n;
  }
  __syncthreads();
  return found;
}

// A CTA quantises kStrip rows of one row block, a warp one row at a time: a
// lane holds 8 elements, four lanes a block (two shuffles for its maximum),
// a step of the warp 256 elements (512 bytes of bf16 in, 128 bytes of codes
// out), kAhead steps loaded before the first is used.
constexpr int kStrip = 32;
constexpr int kAhead = 4;

template <typename T, bool ROWS>
__global__ void __launch_bounds__(256) quantize_kernel(const T* __restrict__ x, int64_t x_rows,
                                                       const int64_t* __restrict__ row_index,
                                                       const int32_t* __restrict__ offsets, int nseg, int64_t S,
                                                       int K, int kt, uint8_t* __restrict__ packed,
                                                       uint8_t* __restrict__ scale) {
  const int strip = blockIdx.x % (kBlockRows / kStrip);
  const int blk = blockIdx.x / (kBlockRows / kStrip);
  RowBlock b;
  if constexpr (ROWS) {
    b = find_block(offsets, nseg, S, blk);
  } else {  // nseg matrices of S rows
    const int per = (int)ceil_div(S, kBlockRows);
    const int r = (blk % per) * kBlockRows;
    b = RowBlock{(int64_t)(blk / per) * S + r, (int)min((int64_t)kBlockRows, S - r)};
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint8_t* tiles = scale + (int64_t)blk * kt * 512;
  for (int r = strip * kStrip + warp; r < min(b.rows, (strip + 1) * kStrip); r += 8) {
    const int64_t dst = b.row0 + r;
    int64_t src = dst;
    bool ok = true;
    if (ROWS && row_index) {
      src = row_index[dst];
      ok = src >= 0 && src < x_rows;
      if (!ok && lane == 0) device_fail(MIRAI_ERR_DEVICE_BOUNDS, 701);
    }
    const T* row = x + src * K;
    for (int k0 = lane * 8; k0 - lane * 8 < K; k0 += 256 * kAhead) {
      Raw8<T> raw[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (ok && k0 + i * 256 < K) load8(row + k0 + i * 256, raw[i]);
        else zero8(raw[i]);
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int k = k0 + i * 256;
        if (k - lane * 8 >= K) break;  // warp-uniform
        float v[8];
        unpack8(raw[i], v);
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
        m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
        const uint32_t byte = scale_byte(m);
        const float inv = inv_scale(byte == 255u ? 254u : byte);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] *= inv;
        const uint32_t codes = byte == 255u ? 0u : e2m1x8(v);
        if (k < K) *reinterpret_cast<uint32_t*>(packed + (dst * K + k) / 2) = codes;
        // four blocks make one word of the row's scales (blocks past K stay zero)
        uint32_t w = k < K ? byte << (8 * ((lane >> 2) & 3)) : 0u;
        w |= __shfl_xor_sync(0xffffffffu, w, 4);
        w |= __shfl_xor_sync(0xffffffffu, w, 8);
        const int kw = k / 128;
        if ((lane & 15) == 0 && kw < kt)
          *reinterpret_cast<uint32_t*>(tiles + (int64_t)kw * 512 + (r & 31) * 16 + (r >> 5) * 4) = w;
      }
    }
  }
}

// ----------------------------------------------------------------------------
// read-back: the same split, 8 codes of a row per lane and step

__device__ __forceinline__ void decode8(uint32_t codes, float scale, float (&v)[8]) {
  uint32_t h[4];
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(codes));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
    v[2 * i] = f.x * scale, v[2 * i + 1] = f.y * scale;
  }
}
__device__ __forceinline__ float scale_value(uint32_t byte) {
  return byte == 255u ? __uint_as_float(0x7fffffffu) : __uint_as_float(byte ? byte << 23 : 1u << 22);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                                            pack_bf16x2(v[6], v[7]));
}
__device__ __forceinline__ void store8(__half* p, const float (&v)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}

template <typename T>
__global__ void __launch_bounds__(256) dequantize_kernel(const uint8_t* __restrict__ packed,
                                                         const uint8_t* __restrict__ scale, int64_t out, int K,
                                                         int kt, T* __restrict__ dst) {
  const int strip = blockIdx.x % (kBlockRows / kStrip);
  const int blk = blockIdx.x / (kBlockRows / kStrip);
  const int per = (int)ceil_div(out, kBlockRows);
  const int r0 = (blk % per) * kBlockRows;
  const int64_t row0 = (int64_t)(blk / per) * out + r0;
  const int rows = (int)min((int64_t)kBlockRows, out - r0);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint8_t* tiles = scale + (int64_t)blk * kt * 512;
  for (int r = strip * kStrip + warp; r < min(rows, (strip + 1) * kStrip); r += 8) {
    const int64_t row = row0 + r;
    const uint8_t* srow = tiles + (r & 31) * 16 + (r >> 5) * 4;
    for (int k0 = lane * 8; k0 < K; k0 += 256 * kAhead) {
      uint32_t codes[kAhead];
      uint32_t byte[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int k = k0 + i * 256;
        if (k < K) {
          codes[i] = __ldg(reinterpret_cast<const uint32_t*>(packed + (row * K + k) / 2));
          byte[i] = __ldg(srow + (int64_t)(k / 128) * 512 + (k / 32) % 4);
        }
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int k = k0 + i * 256;
        if (k >= K) break;
        float v[8];
        decode8(codes[i], scale_value(byte[i]), v);
        store8(dst + row * K + k, v);
      }
    }
  }
}

// ----------------------------------------------------------------------------
// The expert products on the tensor cores (tcgen05.mma kind::mxf4).
//
//   GATEUP  h = silu(g) * u, g = x W1^T, u = x W3^T   (rounded once, from fp32)
//   DOWN    y = h W2^T (+ a LoRA adapter's rank block, one bf16 k-block)
//
// A tile is 256 rows of one segment x 256 accumulator columns (128 channels of
// gate beside the same 128 of up, or 256 output columns), on a CTA pair
// (cta_group::2, M = 256): each SM stages its own 128 rows of A and half of B.
// A stage is 256 elements of K: 128-byte rows of codes (128-byte swizzle, one
// TMA box per operand) and the scale tiles of both operands (two 512-byte
// tiles per 128 rows), which tcgen05.cp puts into TMEM right before the
// stage's four K = 64 MMAs.  Every SM holds the scales of all 256 columns.
//
// TMEM: two 256-column accumulators plus the scales do not fit 512 columns, so
// the accumulators overlap by 64 columns (0..255 and 192..447): the epilogue
// reads the shared 64 first and then lets the next tile's MMAs start.
//
// Warps: 0 TMA producer, 1 MMA issuer (the leader CTA's), 4..11 epilogue (two
// per TMEM lane quarter).
enum Mode { GATEUP = 0, DOWN = 1 };

constexpr int BM = 128;
constexpr int TILE_M = 2 * BM;
constexpr int TN = 256;
constexpr int BKE = 256;  // elements of K per stage
constexpr int STAGES = 5;
constexpr uint32_t A_BYTES = BM * 128;
constexpr uint32_t B_BYTES = (TN / 2) * 128;
constexpr uint32_t SFA_BYTES = 1024;      // two K tiles of this CTA's 128 rows
constexpr uint32_t SFB_BYTES = 2 * 1024;  // two K tiles of both 128-column halves
constexpr uint32_t STAGE_BYTES = A_BYTES + B_BYTES + SFA_BYTES + SFB_BYTES;
constexpr int EPI_WARPS = 8;
constexpr int EPI_FIRST = 4;
constexpr int THREADS = 32 * (EPI_FIRST + EPI_WARPS);
constexpr int BOXES = 2;                 // staging boxes per epilogue warp
constexpr uint32_t BOX_BYTES = 32 * 64;  // 32 rows x 32 bf16
constexpr uint32_t ACC_STEP = 192;       // second accumulator's first column
constexpr uint32_t SF_COL = 448;         // scale columns: two slots of 32 (8 for A, 16 for B)
constexpr uint32_t TMEM_COLS = 512;

struct Params {
  const int32_t* offsets;  // [segs] inclusive row ends
  int segs;                // row segments; segment g multiplies expert g % experts
  int experts;
  int64_t S;
  int K, N;                // reduction length; output columns (I or H)
  int n_tiles;
  int w_blocks;            // row tiles of one expert's scales
  int has_ext;
  __nv_bfloat16* out;      // h [S, I] or y [S, H]; GATEUP: may be null when hq is wanted alone
  __nv_bfloat16* gate_up;  // GATEUP: optional [S, 2I]
  uint8_t* hq;             // GATEUP: optional packed h [S, I/2] ...
  uint8_t* hscale;         // ... and its scale tiles
  int64_t h_blocks;        // row tiles of hscale
  int h_kt;
};

struct alignas(16) Smem {
  uint64_t full[STAGES];
  uint64_t empty[STAGES];
  uint64_t tfull[2];
  uint64_t tover;
  uint32_t tmem_base;
  int abort_flag;
  int warp_sum[32];
  int row_start[kMaxSegs + 1];
  int tile_prefix[kMaxSegs + 1];
  int blk_prefix[kMaxSegs + 1];
};

constexpr size_t smem_bytes() {
  return 1024 + (size_t)STAGES * STAGE_BYTES + (size_t)EPI_WARPS * BOXES * BOX_BYTES + sizeof(Smem);
}
static_assert(smem_bytes() <= 232448, "shared memory budget exceeded");

// Instruction descriptor of kind::mxf4: E2M1 operands, both K-major, UE8M0
// scales; sf_id (0 or 2) picks the two scale bytes of the K = 64 step.
__device__ __forceinline__ constexpr uint32_t idesc_mxf4(int M, int N, uint32_t sf_id) {
  return (sf_id << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | (1u << 23) | ((uint32_t)(M >> 4) << 24) |
         (sf_id << 29);
}

__device__ __forceinline__ void umma_mxf4_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa,
                                               uint32_t sfb, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
      : "memory");
}

// One 512-byte scale tile (32 rows of 16 bytes) into 4 TMEM columns, copied to
// all four lane quarters, in both CTAs of the pair.
__device__ __forceinline__ void scale_copy_pair(uint32_t tmem, uint32_t smem_addr) {
  uint64_t d = 0;
  d |= (uint64_t)((smem_addr & 0x3FFFF) >> 4);
  d |= (uint64_t)(128 >> 4) << 32;  // 8-row groups 128 bytes apart
  d |= (uint64_t)1 << 46;           // sm_100 descriptor, no swizzle
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(d) : "memory");
}

__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

// Segment table shared by every role: first rows, and exclusive prefixes of the
// 256-row tiles and of the 128-row scale blocks.  All threads take part.
__device__ __forceinline__ void build_segments(Smem& sm, const int32_t* offsets, int segs, int64_t S, int site) {
  for (int g = threadIdx.x; g < segs; g += THREADS) {
    int begin;
    const int rows = segment_rows(offsets, g, S, begin, site);
    sm.row_start[g] = begin;
    sm.blk_prefix[g] = rows;  // until the scan below
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int tiles = 0, blocks = 0, end = 0;
    for (int g0 = 0; g0 < segs; g0 += 32) {
      const int g = g0 + lane;
      const int rows = g < segs ? sm.blk_prefix[g] : 0;
      const int t = (rows + TILE_M - 1) / TILE_M, b = (rows + BM - 1) / BM;
      int ti = t, bi = b;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int tv = __shfl_up_sync(0xffffffffu, ti, o), bv = __shfl_up_sync(0xffffffffu, bi, o);
        if (lane >= o) ti += tv, bi += bv;
      }
      if (g < segs) {
        sm.tile_prefix[g] = tiles + ti - t;
        sm.blk_prefix[g] = blocks + bi - b;
        end = sm.row_start[g] + rows;
        if (g == segs - 1) sm.row_start[segs] = end;
      }
      tiles += __shfl_sync(0xffffffffu, ti, 31);
      blocks += __shfl_sync(0xffffffffu, bi, 31);
    }
    if (lane == 0) sm.tile_prefix[segs] = tiles, sm.blk_prefix[segs] = blocks;
  }
}

struct Tile {
  int seg, m, n;
};
__device__ __forceinline__ Tile decode_tile(const Smem& sm, int t, int segs, int n_tiles) {
  const int mt = t / n_tiles;
  int lo = 0, hi = segs;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (sm.tile_prefix[mid] <= mt) lo = mid;
    else hi = mid;
  }
  return Tile{lo, mt - sm.tile_prefix[lo], t - mt * n_tiles};
}

template <int MODE>
__global__ void __launch_bounds__(THREADS, 1)
    product_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_sa,
                   const __grid_constant__ CUtensorMap tmap_b0, const __grid_constant__ CUtensorMap tmap_b1,
                   const __grid_constant__ CUtensorMap tmap_sb0, const __grid_constant__ CUtensorMap tmap_sb1,
                   const __grid_constant__ CUtensorMap tmap_xa, const __grid_constant__ CUtensorMap tmap_xb,
                   const __grid_constant__ CUtensorMap tmap_o0, const __grid_constant__ CUtensorMap tmap_o1,
                   const __grid_constant__ CUtensorMap tmap_o2, const Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = base;
  uint8_t* sB = sA + STAGES * A_BYTES;
  uint8_t* sBox = sB + STAGES * B_BYTES;  // 1024-byte aligned like the operands
  uint8_t* sSA = sBox + EPI_WARPS * BOXES * BOX_BYTES;
  uint8_t* sSB = sSA + STAGES * SFA_BYTES;
  Smem& sm = *reinterpret_cast<Smem*>(sSB + STAGES * SFB_BYTES);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int unit = (int)(blockIdx.x >> 1), num_units = (int)(gridDim.x >> 1);
  const uint32_t full_leader0 = mapa_shared(smem_u32(&sm.full[0]), 0);
  const uint32_t tover_leader = mapa_shared(smem_u32(&sm.tover), 0);

  build_segments(sm, p.offsets, p.segs, p.S, 710 + MODE);
  if (warp == 1) {
    if (lane == 0) {
      for (int s = 0; s < STAGES; ++s) {
        mbar_init(&sm.full[s], 1);
        mbar_init(&sm.empty[s], 1);
      }
      mbar_init(&sm.tfull[0], 1);
      mbar_init(&sm.tfull[1], 1);
      mbar_init(&sm.tover, 2 * EPI_WARPS);
      sm.abort_flag = 0;
      fence_mbar_init();
    }
    __syncwarp();
    tmem_alloc_pair(&sm.tmem_base, TMEM_COLS);
    tmem_relinquish_pair();
  }
  if (warp == 2 && lane == 0) {
    prefetch_tmap(&tmap_a);
    prefetch_tmap(&tmap_sa);
    prefetch_tmap(&tmap_b0);
    prefetch_tmap(&tmap_sb0);
    if (MODE == GATEUP) {
      prefetch_tmap(&tmap_b1);
      prefetch_tmap(&tmap_sb1);
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  tc_fence_after();

  const uint32_t tmem = sm.tmem_base;
  const int total_tiles = sm.tile_prefix[p.segs] * p.n_tiles;
  const int num_kb = (p.K + BKE - 1) / BKE;
  const int total_kb = num_kb + p.has_ext;
  volatile int* abort_flag = &sm.abort_flag;

  if (warp == 0 && lane == 0) {
    // ======================= TMA producer =======================
    int stage = 0;
    uint32_t phase = 0;
    for (int t = unit; t < total_tiles && !*abort_flag; t += num_units) {
      const Tile tile = decode_tile(sm, t, p.segs, p.n_tiles);
      const int e = tile.seg % p.experts;
      const int row = sm.row_start[tile.seg] + tile.m * TILE_M + (int)rank * BM;
      const int ablk = sm.blk_prefix[tile.seg] + tile.m * 2 + (int)rank;
      // B rows of this CTA, and the row tiles of both halves' scales
      const CUtensorMap* mb = MODE == GATEUP && rank ? &tmap_b1 : &tmap_b0;
      const int brow = e * p.N + (MODE == GATEUP ? tile.n * BM : tile.n * TN + (int)rank * BM);
      const int bblk = e * p.w_blocks + (MODE == GATEUP ? tile.n : 2 * tile.n);
      for (int kb = 0; kb < total_kb; ++kb) {
        if (!mbar_wait(&sm.empty[stage], phase ^ 1, 70)) {
          *abort_flag = 1;
          break;
        }
        const uint32_t full = full_leader0 + 8u * stage;
        const bool ext = kb == num_kb;
        // the leader's own barrier carries the bytes of both CTAs
        if (leader) mbar_arrive_expect_tx(&sm.full[stage], 2 * (ext ? A_BYTES + B_BYTES : STAGE_BYTES));
        if (ext) {
          tma_load_2d_pair(sA + stage * A_BYTES, &tmap_xa, 0, row, full);
          tma_load_2d_pair(sB + stage * B_BYTES, &tmap_xb, 0, brow, full);
        } else {
          tma_load_2d_pair(sA + stage * A_BYTES, &tmap_a, kb * 128, row, full);
          tma_load_2d_pair(sB + stage * B_BYTES, mb, kb * 128, brow, full);
          tma_load_2d_pair(sSA + stage * SFA_BYTES, &tmap_sa, kb * 256, ablk, full);
          tma_load_2d_pair(sSB + stage * SFB_BYTES, &tmap_sb0, kb * 256, bblk, full);
          tma_load_2d_pair(sSB + stage * SFB_BYTES + 1024, MODE == GATEUP ? &tmap_sb1 : &tmap_sb0, kb * 256,
                           MODE == GATEUP ? bblk : bblk + 1, full);
        }
        if (++stage == STAGES) stage = 0, phase ^= 1;
      }
    }
    // no commit of the leader may reach this CTA after it has exited
    for (int i = 0; i < STAGES; ++i) {
      if (!mbar_wait(&sm.empty[stage], phase ^ 1, 71)) break;
      if (++stage == STAGES) stage = 0, phase ^= 1;
    }
  } else if (warp == 1 && lane == 0 && leader) {
    // ======================= MMA issuer =======================
    constexpr uint32_t id_ext = make_idesc_bf16(TILE_M, TN);
    int stage = 0, it = 0;
    uint32_t phase = 0, slot = 0;
    for (int t = unit; t < total_tiles && !*abort_flag; t += num_units, ++it) {
      // the epilogue has read the columns this accumulator shares with the
      // previous tile's (and with it all of the tile before that one)
      if (it > 0 && !mbar_wait(&sm.tover, (it - 1) & 1, 72)) {
        *abort_flag = 1;
        break;
      }
      tc_fence_after();
      const uint32_t d = tmem + (it & 1) * ACC_STEP;
      bool ok = true;
      for (int kb = 0; kb < total_kb; ++kb) {
        if (!mbar_wait(&sm.full[stage], phase, 73)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t a = smem_u32(sA + stage * A_BYTES), b = smem_u32(sB + stage * B_BYTES);
        if (kb == num_kb) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_bf16_pair(d, make_sdesc_sw128(a + k * 32, 16, 1024), make_sdesc_sw128(b + k * 32, 16, 1024), id_ext, 1u);
        } else {
          const uint32_t sf = tmem + SF_COL + slot * 32;
          slot ^= 1;
          const uint32_t sa = smem_u32(sSA + stage * SFA_BYTES), sb = smem_u32(sSB + stage * SFB_BYTES);
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            scale_copy_pair(sf + 4 * w, sa + 512 * w);
            scale_copy_pair(sf + 8 + 8 * w, sb + 512 * w);
            scale_copy_pair(sf + 8 + 8 * w + 4, sb + 1024 + 512 * w);
          }
          const int steps = min(4, (p.K - kb * BKE + 63) / 64);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (k < steps)
              umma_mxf4_pair(d, make_sdesc_sw128(a + k * 32, 16, 1024), make_sdesc_sw128(b + k * 32, 16, 1024),
                             idesc_mxf4(TILE_M, TN, (k & 1) * 2), sf + 4 * (k >> 1), sf + 8 + 8 * (k >> 1),
                             (kb | k) != 0 ? 1u : 0u);
          }
        }
        umma_commit_pair(&sm.empty[stage], 0x3);
        if (++stage == STAGES) stage = 0, phase ^= 1;
      }
      if (!ok) {
        *abort_flag = 1;
        break;
      }
      umma_commit_pair(&sm.tfull[it & 1], 0x3);
    }
  } else if (warp >= EPI_FIRST) {
    // ======================= epilogue =======================
    const int q = warp & 3;                     // TMEM lane quarter
    const int part = (warp - EPI_FIRST) / 4;    // which half of the 32-column chunks
    uint8_t* my_boxes = sBox + (warp - EPI_FIRST) * BOXES * BOX_BYTES;
    int box_i = 0;
    auto stage_store = [&](const CUtensorMap* map, int col, int64_t row0, const uint32_t (&w)[16]) {
      uint8_t* box = my_boxes + box_i * BOX_BYTES;
      if (lane == 0) bulk_wait_group_read<BOXES - 1>();
      __syncwarp();
      const uint32_t addr = smem_u32(box) + (uint32_t)lane * 64u;
      const uint32_t sw = (uint32_t)(lane >> 1) & 3u;  // 64-byte swizzle
#pragma unroll
      for (int v = 0; v < 4; ++v)
        sts128(addr + (((uint32_t)v ^ sw) << 4), w[4 * v], w[4 * v + 1], w[4 * v + 2], w[4 * v + 3]);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        tma_store_2d(map, box, col, (int)row0);
        bulk_commit_group();
      }
      box_i = box_i + 1 == BOXES ? 0 : box_i + 1;
    };
    auto row_store = [&](__nv_bfloat16* dst, const uint32_t (&w)[16]) {
#pragma unroll
      for (int v = 0; v < 4; ++v)
        reinterpret_cast<uint4*>(dst)[v] = make_uint4(w[4 * v], w[4 * v + 1], w[4 * v + 2], w[4 * v + 3]);
    };
    int it = 0;
    for (int t = unit; t < total_tiles && !*abort_flag; t += num_units, ++it) {
      const Tile tile = decode_tile(sm, t, p.segs, p.n_tiles);
      const int begin = sm.row_start[tile.seg];
      // a segment ends where its tiles say (bad offsets may leave gaps between segments)
      const int end = sm.row_start[tile.seg + 1];
      const int local = tile.m * TILE_M + (int)rank * BM + q * 32 + lane;
      const bool valid = begin + local < end;
      const int64_t row = (int64_t)begin + local;
      const bool boxed = __all_sync(0xffffffffu, valid);
      const int64_t row0 = __shfl_sync(0xffffffffu, row, 0);
      if (!mbar_wait(&sm.tfull[it & 1], (it >> 1) & 1, 74)) {
        *abort_flag = 1;
        break;
      }
      tc_fence_after();
      const uint32_t acc = tmem + (it & 1) * ACC_STEP + ((uint32_t)(q * 32) << 16);
      auto release = [&]() {  // the shared columns have been read
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(tover_leader);
      };
      if constexpr (MODE == GATEUP) {
        // shared columns: up channels 64..127 of the first accumulator, gate
        // channels 0..63 of the second
#pragma unroll 1
        for (int i = 0; i < 2; ++i) {
          const int c = part + (((it & 1) ^ i) ? 0 : 2);
          uint32_t g[32], u[32];
          tmem_ld_32x32b_x32(acc + c * 32, g);
          tmem_ld_32x32b_x32(acc + BM + c * 32, u);
          tmem_ld_wait();
          if (i == 0) release();
          const int col = tile.n * BM + c * 32;
          if (col >= p.N) continue;  // warp-uniform
          uint32_t w[16];
          if (p.gate_up) {
            const int64_t ld2 = 2 * (int64_t)p.N;
#pragma unroll
            for (int j = 0; j < 16; ++j) w[j] = pack_bf16x2(__uint_as_float(g[2 * j]), __uint_as_float(g[2 * j + 1]));
            if (boxed) stage_store(&tmap_o1, col, row0, w);
            else if (valid) row_store(p.gate_up + row * ld2 + col, w);
#pragma unroll
            for (int j = 0; j < 16; ++j) w[j] = pack_bf16x2(__uint_as_float(u[2 * j]), __uint_as_float(u[2 * j + 1]));
            if (boxed) stage_store(&tmap_o2, col, row0, w);
            else if (valid) row_store(p.gate_up + row * ld2 + p.N + col, w);
          }
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            float h[2];
#pragma unroll
            for (int s = 0; s < 2; ++s) {
              const float gv = __uint_as_float(g[2 * j + s]);
              h[s] = __fdividef(gv, 1.f + __expf(-gv)) * __uint_as_float(u[2 * j + s]);
            }
            w[j] = pack_bf16x2(h[0], h[1]);
          }
          if (p.out) {
            if (boxed) stage_store(&tmap_o0, col, row0, w);
            else if (valid) row_store(p.out + row * p.N + col, w);
          }
          if (p.hq && valid) {
            // this lane's 32 channels are one block of the quantised h
            uint32_t m = 0;
#pragma unroll
            for (int j = 0; j < 16; ++j)
              m = max(m, max((w[j] << 16) & 0x7fffffffu, w[j] & 0x7fff0000u));
            const uint32_t byte = scale_byte(m);
            const float inv = inv_scale(byte == 255u ? 254u : byte);
            uint32_t codes[4];
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              float f[8];
#pragma unroll
              for (int j = 0; j < 4; ++j) f[2 * j] = bf16_lo(w[4 * v + j]) * inv, f[2 * j + 1] = bf16_hi(w[4 * v + j]) * inv;
              codes[v] = byte == 255u ? 0u : e2m1x8(f);
            }
            *reinterpret_cast<uint4*>(p.hq + (row * p.N + col) / 2) = make_uint4(codes[0], codes[1], codes[2], codes[3]);
            const int64_t blk = sm.blk_prefix[tile.seg] + tile.m * 2 + (int)rank;
            if (blk < p.h_blocks) {
              uint8_t* word = p.hscale + (blk * p.h_kt + tile.n) * 512 + lane * 16 + q * 4;
              word[c] = (uint8_t)byte;
              if (col + 32 == p.N)  // blocks past the row's end are zero bytes
                for (int z = c + 1; z < 4; ++z) word[z] = 0;
            }
          }
        }
      } else {
        // shared columns: chunks 6, 7 of the first accumulator, 0, 1 of the second
        const int first = (it & 1) ? part : 6 + part;
#pragma unroll 1
        for (int i = 0; i < 4; ++i) {
          const int c = i == 0 ? first : ((it & 1) ? 2 : 0) + part * 3 + i - 1;
          uint32_t v[32];
          tmem_ld_32x32b_x32(acc + c * 32, v);
          tmem_ld_wait();
          if (i == 0) release();
          const int col = tile.n * TN + c * 32;
          if (col >= p.N) continue;  // warp-uniform
          uint32_t w[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) w[j] = pack_bf16x2(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1]));
          if (boxed) stage_store(&tmap_o0, col, row0, w);
          else if (valid) row_store(p.out + row * p.N + col, w);
        }
      }
    }
    if (lane == 0) bulk_wait_group_all();
    __syncwarp();
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, TMEM_COLS);
  }
}

// ----------------------------------------------------------------------------
// host side

static bool misaligned(const void* p, unsigned a = 16) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) != 0; }

// Most row tiles `rows` rows in `segs` segments can take.
static int64_t max_blocks(int64_t rows, int64_t segs) { return rows / kBlockRows + (segs < rows ? segs : rows); }

static int scale_map(CUtensorMap& m, const uint8_t* scale, int64_t blocks, int kt) {
  return make_tmap_2d(&m, CU_TENSOR_MAP_DATA_TYPE_UINT32, 4, scale, (uint64_t)kt * 128, (uint64_t)blocks,
                      (uint64_t)kt * 512, 256, 1, CU_TENSOR_MAP_SWIZZLE_NONE);
}
static int code_map(CUtensorMap& m, const uint8_t* packed, int64_t rows, int K) {
  return make_tmap_2d(&m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, packed, (uint64_t)K / 2, (uint64_t)rows, (uint64_t)K / 2,
                      128, BM, CU_TENSOR_MAP_SWIZZLE_128B);
}
static int out_map(CUtensorMap& m, void* out, int64_t rows, int N, int64_t ld) {
  return make_tmap_2d(&m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, out, (uint64_t)N, (uint64_t)rows, (uint64_t)ld * 2, 32,
                      32, CU_TENSOR_MAP_SWIZZLE_64B);
}

// CTA pairs of the kernel that fit the current device at once (per device; 0 = an error was set).
constexpr int kMaxDevices = 64;
template <int MODE> static int resident_pairs(const char* name) {
  static std::atomic<int> cached[kMaxDevices];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) {
    set_error(MIRAI_ERR_CUDA, "%s: no current device", name);
    return 0;
  }
  int n = cached[dev].load(std::memory_order_acquire);
  if (n > 0) return n;
  auto kern = product_kernel<MODE>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_bytes());
  if (e != cudaSuccess) {
    set_error(MIRAI_ERR_CUDA, "%s: cudaFuncSetAttribute: %s", name, cudaGetErrorString(e));
    return 0;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(THREADS, 1, 1);
  cfg.dynamicSmemBytes = smem_bytes();
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const int sms = sm_count();
  cfg.gridDim = dim3((unsigned)(sms & ~1), 1, 1);
  if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n <= 0) {
    cudaGetLastError();
    n = sms / 2;
  }
  cached[dev].store(n, std::memory_order_release);
  return n;
}

struct Operand {
  const uint8_t* packed;
  const uint8_t* scale;
};

template <int MODE>
static int product(const char* name, const Operand& a, const int32_t* offsets, int32_t nsrc, int32_t experts, int64_t S,
                   int32_t K, int32_t N, const mirai_mxfp4_weight* w0, const mirai_mxfp4_weight* w1, const void* rank_a,
                   const void* rank_b, void* out, void* gate_up, uint8_t* hq, uint8_t* hscale, mirai_stream_t stream) {
  if (nsrc <= 0 || experts <= 0 || (int64_t)nsrc * experts > kMaxSegs)
    return set_error(MIRAI_ERR_INVALID_ARG, "%s: %d sources x %d experts outside 1..%d segments", name, nsrc, experts,
                     kMaxSegs);
  if (S < 0 || K <= 0 || N <= 0)
    return set_error(MIRAI_ERR_INVALID_ARG, "%s: bad sizes (S=%lld, K=%d, N=%d)", name, (long long)S, K, N);
  if (K % 32 || N % 32)
    return set_error(MIRAI_ERR_UNSUPPORTED, "%s: needs K %% 32 == 0 and N %% 32 == 0 (K=%d, N=%d)", name, K, N);
  if (S >= ((int64_t)1 << 31) - TILE_M || (int64_t)experts * N >= (int64_t)1 << 31)
    return set_error(MIRAI_ERR_UNSUPPORTED, "%s: more than 2^31 routed rows or weight rows", name);
  if (S == 0) return MIRAI_OK;
  if (!a.packed || !a.scale || !offsets || !w0 || !w0->packed || !w0->scale || (w1 && (!w1->packed || !w1->scale)))
    return set_error(MIRAI_ERR_INVALID_ARG, "%s: null operand", name);
  if ((!out && !hq) || (hq && !hscale) || (!rank_a != !rank_b))
    return set_error(MIRAI_ERR_INVALID_ARG, "%s: null output, scale or rank-block pointer", name);
  if (misaligned(out) || misaligned(gate_up) || misaligned(hq))
    return set_error(MIRAI_ERR_INVALID_ARG, "%s: output not 16-byte aligned", name);
  const int kt = (int)ceil_div(K, 128);
  const int64_t segs = (int64_t)nsrc * experts;
  Params p = {};
  p.offsets = offsets;
  p.segs = (int)segs;
  p.experts = experts;
  p.S = S;
  p.K = K;
  p.N = N;
  p.n_tiles = (int)ceil_div(N, MODE == GATEUP ? BM : TN);
  p.w_blocks = (int)ceil_div(N, kBlockRows);
  p.has_ext = rank_a != nullptr;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.gate_up = static_cast<__nv_bfloat16*>(gate_up);
  p.hq = hq;
  p.hscale = hscale;
  p.h_blocks = max_blocks(S, segs);
  p.h_kt = (int)ceil_div(N, 128);
  CUtensorMap ta, tsa, tb0, tb1, tsb0, tsb1, txa, txb, to0, to1, to2;
  int rc = code_map(ta, a.packed, S, K);
  if (!rc) rc = scale_map(tsa, a.scale, p.h_blocks, kt);
  if (!rc) rc = code_map(tb0, w0->packed, (int64_t)experts * N, K);
  if (!rc) rc = scale_map(tsb0, w0->scale, (int64_t)experts * p.w_blocks, kt);
  if (!rc) rc = w1 ? code_map(tb1, w1->packed, (int64_t)experts * N, K) : (tb1 = tb0, MIRAI_OK);
  if (!rc) rc = w1 ? scale_map(tsb1, w1->scale, (int64_t)experts * p.w_blocks, kt) : (tsb1 = tsb0, MIRAI_OK);
  // maps that a call does not use are copies of another
  txa = ta;
  txb = tb0;
  if (!rc && rank_a) {
    rc = make_tmap_2d(&txa, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, rank_a, 64, (uint64_t)S, 128, 64, BM,
                      CU_TENSOR_MAP_SWIZZLE_128B);
    if (!rc)
      rc = make_tmap_2d(&txb, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, rank_b, 64, (uint64_t)experts * N, 128, 64, BM,
                        CU_TENSOR_MAP_SWIZZLE_128B);
  }
  if (!rc) rc = out ? out_map(to0, out, S, N, N) : (to0 = ta, MIRAI_OK);
  to1 = to2 = to0;
  if (!rc && gate_up) {
    rc = out_map(to1, gate_up, S, N, 2 * (int64_t)N);
    if (!rc) rc = out_map(to2, static_cast<__nv_bfloat16*>(gate_up) + N, S, N, 2 * (int64_t)N);
  }
  if (rc) return rc;
  const int pairs = resident_pairs<MODE>(name);
  if (!pairs) return MIRAI_ERR_CUDA;
  const int limit = gemm_sm_limit();
  const int sms = (limit > 0 && limit < sm_count()) ? limit : sm_count();
  int64_t units = (S / TILE_M + (segs < S ? segs : S)) * p.n_tiles;
  if (units > pairs) units = pairs;
  if (units > sms / 2) units = sms / 2 > 0 ? sms / 2 : 1;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(THREADS, 1, 1);
  cfg.gridDim = dim3((unsigned)(2 * units), 1, 1);
  cfg.dynamicSmemBytes = smem_bytes();
  cfg.stream = reinterpret_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, product_kernel<MODE>, ta, tsa, tb0, tb1, tsb0, tsb1, txa, txb, to0, to1,
                                           to2, p);
  if (e != cudaSuccess) return set_error(MIRAI_ERR_CUDA, "%s: launch failed: %s", name, cudaGetErrorString(e));
  return check_launch(name);
}

// Grid of the quantise / read-back kernels, or -1 (with the error set).
static int64_t strips(const char* name, int64_t blocks) {
  const int64_t g = blocks * (kBlockRows / kStrip);
  if (g > INT32_MAX) {
    set_error(MIRAI_ERR_UNSUPPORTED, "%s: too many rows for one call", name);
    return -1;
  }
  return g;
}

static int matrix_problem(const char* name, int32_t experts, int64_t out, int64_t in) {
  if (experts <= 0 || out <= 0 || in <= 0) return set_error(MIRAI_ERR_INVALID_ARG, "%s: bad sizes", name);
  if (in % 32) return set_error(MIRAI_ERR_UNSUPPORTED, "%s: in_features %lld %% 32 != 0", name, (long long)in);
  if (in > (1 << 24) || out > INT32_MAX / 2)
    return set_error(MIRAI_ERR_UNSUPPORTED, "%s: rows of at most 2^24 elements, 2^30 rows", name);
  return MIRAI_OK;
}

}  // namespace mx
}  // namespace mirai

using namespace mirai;

extern "C" {

size_t mirai_mxfp4_scale_bytes(int32_t num_experts, int64_t out_features, int64_t in_features) {
  if (num_experts <= 0 || out_features <= 0 || in_features <= 0) return 0;
  return (size_t)num_experts * mx::ceil_div(out_features, 128) * mx::ceil_div(in_features, 128) * 512;
}

size_t mirai_mxfp4_rows_scale_bytes(int64_t num_rows, int32_t num_segments, int32_t width) {
  if (num_rows <= 0 || num_segments <= 0 || width <= 0) return 0;
  return (size_t)mx::max_blocks(num_rows, num_segments) * mx::ceil_div(width, 128) * 512;
}

int mirai_mxfp4_quantize(const void* weight, int32_t dtype, int32_t num_experts, int64_t out_features,
                         int64_t in_features, uint8_t* packed, uint8_t* scale, mirai_stream_t stream) {
  if (int rc = mx::matrix_problem("mxfp4_quantize", num_experts, out_features, in_features)) return rc;
  if (!weight || !packed || !scale || mx::misaligned(weight) || mx::misaligned(packed) || mx::misaligned(scale))
    return set_error(MIRAI_ERR_INVALID_ARG, "mxfp4_quantize: null or misaligned pointer");
  const int64_t grid = mx::strips("mxfp4_quantize", num_experts * mx::ceil_div(out_features, mx::kBlockRows));
  if (grid < 0) return MIRAI_ERR_UNSUPPORTED;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int K = (int)in_features, kt = (int)mx::ceil_div(K, 128);
  auto go = [&](auto* w) {
    mx::quantize_kernel<std::remove_const_t<std::remove_pointer_t<decltype(w)>>, false>
        <<<(unsigned)grid, 256, 0, s>>>(w, 0, nullptr, nullptr, num_experts, out_features, K, kt, packed, scale);
  };
  if (dtype == MIRAI_DTYPE_BF16) go(static_cast<const __nv_bfloat16*>(weight));
  else if (dtype == MIRAI_DTYPE_F32) go(static_cast<const float*>(weight));
  else if (dtype == MIRAI_DTYPE_F16) go(static_cast<const __half*>(weight));
  else return set_error(MIRAI_ERR_INVALID_ARG, "mxfp4_quantize: unknown dtype %d", dtype);
  return check_launch("mxfp4_quantize");
}

int mirai_mxfp4_dequantize(const uint8_t* packed, const uint8_t* scale, int32_t num_experts, int64_t out_features,
                           int64_t in_features, void* out, int32_t dtype, mirai_stream_t stream) {
  if (int rc = mx::matrix_problem("mxfp4_dequantize", num_experts, out_features, in_features)) return rc;
  if (!out || !packed || !scale || mx::misaligned(out) || mx::misaligned(packed) || mx::misaligned(scale))
    return set_error(MIRAI_ERR_INVALID_ARG, "mxfp4_dequantize: null or misaligned pointer");
  const int64_t grid = mx::strips("mxfp4_dequantize", num_experts * mx::ceil_div(out_features, mx::kBlockRows));
  if (grid < 0) return MIRAI_ERR_UNSUPPORTED;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int K = (int)in_features, kt = (int)mx::ceil_div(K, 128);
  auto go = [&](auto* o) {
    mx::dequantize_kernel<<<(unsigned)grid, 256, 0, s>>>(packed, scale, out_features, K, kt, o);
  };
  if (dtype == MIRAI_DTYPE_BF16) go(static_cast<__nv_bfloat16*>(out));
  else if (dtype == MIRAI_DTYPE_F32) go(static_cast<float*>(out));
  else if (dtype == MIRAI_DTYPE_F16) go(static_cast<__half*>(out));
  else return set_error(MIRAI_ERR_INVALID_ARG, "mxfp4_dequantize: unknown dtype %d", dtype);
  return check_launch("mxfp4_dequantize");
}

int mirai_mxfp4_quantize_rows(const void* x, int64_t x_rows, const int64_t* row_index, const int32_t* offsets,
                              int32_t num_segments, int64_t num_rows, int32_t width, uint8_t* packed, uint8_t* scale,
                              mirai_stream_t stream) {
  if (num_segments <= 0 || num_segments > mx::kMaxSegs || num_rows < 0 || x_rows < 0 || width <= 0)
    return set_error(MIRAI_ERR_INVALID_ARG, "mxfp4_quantize_rows: bad sizes (%d segments, 1..%d)", num_segments,
                     mx::kMaxSegs);
  if (width % 32 || width > (1 << 24))
    return set_error(MIRAI_ERR_UNSUPPORTED, "mxfp4_quantize_rows: width %d is not a multiple of 32 up to 2^24", width);
  if (num_rows >= ((int64_t)1 << 31) - mx::TILE_M)
    return set_error(MIRAI_ERR_UNSUPPORTED, "mxfp4_quantize_rows: more than 2^31 rows");
  if (num_rows == 0) return MIRAI_OK;
  if (!row_index && x_rows < num_rows)
    return set_error(MIRAI_ERR_INVALID_ARG, "mxfp4_quantize_rows: %lld input rows for %lld rows", (long long)x_rows,
                     (long long)num_rows);
  if (!x || !offsets || !packed || !scale || mx::misaligned(x) || mx::misaligned(packed) || mx::misaligned(scale))
    return set_error(MIRAI_ERR_INVALID_ARG, "mxfp4_quantize_rows: null or misaligned pointer");
  const int64_t grid = mx::strips("mxfp4_quantize_rows", mx::max_blocks(num_rows, num_segments));
  if (grid < 0) return MIRAI_ERR_UNSUPPORTED;
  mx::quantize_kernel<__nv_bfloat16, true><<<(unsigned)grid, 256, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
      static_cast<const __nv_bfloat16*>(x), x_rows, row_index, offsets, num_segments, num_rows, width,
      (int)mx::ceil_div(width, 128), packed, scale);
  return check_launch("mxfp4_quantize_rows");
}

int mirai_moe_gateup_swiglu_mxfp4(const uint8_t* x_packed, const uint8_t* x_scale, const int32_t* offsets,
                                  int32_t num_sources, int32_t num_experts, int64_t num_rows, int32_t hidden,
                                  int32_t inter, const mirai_mxfp4_weight* w1, const mirai_mxfp4_weight* w3, void* h,
                                  void* gate_up, uint8_t* h_packed, uint8_t* h_scale, mirai_stream_t stream) {
  if (!w3) return set_error(MIRAI_ERR_INVALID_ARG, "gateup_swiglu_mxfp4: null operand");
  return mx::product<mx::GATEUP>("gateup_swiglu_mxfp4", {x_packed, x_scale}, offsets, num_sources, num_experts, num_rows,
                                 hidden, inter, w1, w3, nullptr, nullptr, h, gate_up, h_packed, h_scale, stream);
}

int mirai_moe_down_mxfp4(const uint8_t* h_packed, const uint8_t* h_scale, const int32_t* offsets, int32_t num_sources,
                         int32_t num_experts, int64_t num_rows, int32_t inter, int32_t hidden,
                         const mirai_mxfp4_weight* w2, const void* rank_a, const void* rank_b, void* y,
                         mirai_stream_t stream) {
  return mx::product<mx::DOWN>("down_mxfp4", {h_packed, h_scale}, offsets, num_sources, num_experts, num_rows, inter,
                               hidden, w2, nullptr, rank_a, rank_b, y, nullptr, nullptr, nullptr, stream);
}

}  // extern "C"
