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

// Sixteen values of a row as they lie in memory, by 32-byte loads.
template <typename T> struct Raw16 { uint32_t w[sizeof(T) * 4]; };

__device__ __forceinline__ void ldg256(const void* p, uint32_t* w) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
               : "l"(p));
}
__device__ __forceinline__ void stg256(void* p, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
               "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}
template <typename T> __device__ __forceinline__ void load16(const T* p, Raw16<T>& r) {
  ldg256(p, r.w);
  if constexpr (sizeof(T) == 4) ldg256(p + 8, r.w + 8);
}

// Largest |x| of the sixteen as fp32 bits, by integer maxima (two 16-bit ones per word).
__device__ __forceinline__ uint32_t amax16(const Raw16<__nv_bfloat16>& r) {
  uint32_t m = r.w[0] & 0x7fff7fffu;
#pragma unroll
  for (int i = 1; i < 8; ++i) m = __vmaxu2(m, r.w[i] & 0x7fff7fffu);
  return max(m & 0x7fff0000u, m << 16);
}
__device__ __forceinline__ uint32_t amax16(const Raw16<__half>& r) {
  uint32_t m = r.w[0] & 0x7fff7fffu;
#pragma unroll
  for (int i = 1; i < 8; ++i) m = __vmaxu2(m, r.w[i] & 0x7fff7fffu);
  const uint32_t top = max(m >> 16, m & 0xffffu);
  return __float_as_uint(__half2float(__ushort_as_half((unsigned short)top)));
}
__device__ __forceinline__ uint32_t amax16(const Raw16<float>& r) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) m = max(m, r.w[i] & 0x7fffffffu);
  return m;
}
// Eight of them (half h), as floats.
__device__ __forceinline__ void unpack8(const Raw16<__nv_bfloat16>& r, int h, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[2 * i] = bf16_lo(r.w[4 * h + i]), v[2 * i + 1] = bf16_hi(r.w[4 * h + i]);
}
__device__ __forceinline__ void unpack8(const Raw16<__half>& r, int h, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r.w[4 * h + i]));
    v[2 * i] = f.x, v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void unpack8(const Raw16<float>& r, int h, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r.w[8 * h + i]);
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
// lane holds 16 elements (one 32-byte load of 16-bit values), two lanes a block (one
// shuffle for its maximum), a step of the warp 512 elements, kAhead steps
// loaded before the first is used.  Eight elements per lane and four lanes per block
// needed half as many instructions again, which bound it.
constexpr int kStrip = 32;
constexpr int kAhead = 2;
constexpr int kStep = 512;
constexpr int kAheadBack = 4;  // read-back

template <typename T, bool ROWS>
__global__ void __launch_bounds__(256) quantize_kernel(const T* __restrict__ x, int64_t x_rows,
                                                       const int64_t* __restrict__ row_index,
                                                       const int32_t* __restrict__ offsets, int nseg, int64_t S,
                                                       int K, int kt, uint8_t* __restrict__ packed,
                                                       uint8_t* __restrict__ scale) {
  const int strip = blockIdx.x % (kBlockRows / kStrip);
  const int blk = blockIdx.x / (kBlockRows / kStrip);
  // a product launched behind this kernel may set itself up while the last blocks run (it waits for
  // their results with griddepcontrol.wait)
  if (ROWS) asm volatile("griddepcontrol.launch_dependents;");
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
  // a matrix's scale tiles are written whole: zero bytes past its last row
  const int last = ROWS ? b.rows : kBlockRows;
  for (int r = strip * kStrip + warp; r < min(last, (strip + 1) * kStrip); r += 8) {
    if (!ROWS && r >= b.rows) {
      for (int kw = lane; kw < kt; kw += 32)
        *reinterpret_cast<uint32_t*>(tiles + (int64_t)kw * 512 + (r & 31) * 16 + (r >> 5) * 4) = 0u;
      continue;
    }
    const int64_t dst = b.row0 + r;
    int64_t src = dst;
    bool ok = true;
    if (ROWS && row_index) {
      src = row_index[dst];
      ok = src >= 0 && src < x_rows;
      if (!ok && lane == 0) device_fail(MIRAI_ERR_DEVICE_BOUNDS, 701);
    }
    const T* row = x + src * K;
    for (int base = 0; base < K; base += kStep * kAhead) {
      Raw16<T> raw[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int k = base + i * kStep + lane * 16;
        if (ok && k < K) load16(row + k, raw[i]);
        else raw[i] = Raw16<T>{};
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int k = base + i * kStep + lane * 16;
        if (base + i * kStep >= K) break;  // warp-uniform
        uint32_t m = amax16(raw[i]);
        m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
        const uint32_t byte = scale_byte(m);
        const float inv = inv_scale(byte == 255u ? 254u : byte);
        uint32_t codes[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float v[8];
          unpack8(raw[i], h, v);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] *= inv;
          codes[h] = byte == 255u ? 0u : e2m1x8(v);
        }
        if (k < K) *reinterpret_cast<uint2*>(packed + (dst * K + k) / 2) = make_uint2(codes[0], codes[1]);
        // four blocks make one word of the row's scales (blocks past K stay zero)
        uint32_t w = k < K ? byte << (8 * ((lane >> 1) & 3)) : 0u;
        w |= __shfl_xor_sync(0xffffffffu, w, 2);
        w |= __shfl_xor_sync(0xffffffffu, w, 4);
        const int kw = k / 128;
        if ((lane & 7) == 0 && kw < kt)
          *reinterpret_cast<uint32_t*>(tiles + (int64_t)kw * 512 + (r & 31) * 16 + (r >> 5) * 4) = w;
      }
    }
  }
}

// ----------------------------------------------------------------------------
// read-back: the same split, 16 codes of a row per lane and step

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
// Eight values into a's words of the output type.
__device__ __forceinline__ void pack8(__nv_bfloat16, const float (&v)[8], uint32_t* w) {
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
}
__device__ __forceinline__ void pack8(__half, const float (&v)[8], uint32_t* w) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
}
__device__ __forceinline__ void pack8(float, const float (&v)[8], uint32_t* w) {
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(v[i]);
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
    for (int base = lane * 16; base < K; base += kStep * kAheadBack) {
      uint2 codes[kAheadBack];
      uint32_t byte[kAheadBack];
#pragma unroll
      for (int i = 0; i < kAheadBack; ++i) {
        const int k = base + i * kStep;
        if (k < K) {
          codes[i] = __ldg(reinterpret_cast<const uint2*>(packed + (row * K + k) / 2));
          byte[i] = __ldg(srow + (int64_t)(k / 128) * 512 + (k / 32) % 4);
        }
      }
#pragma unroll
      for (int i = 0; i < kAheadBack; ++i) {
        const int k = base + i * kStep;
        if (k >= K) break;
        const float sc = scale_value(byte[i]);
        uint32_t w[sizeof(T) * 4];
        float v[8];
        decode8(codes[i].x, sc, v);
        pack8(T(), v, w);
        decode8(codes[i].y, sc, v);
        pack8(T(), v, w + sizeof(T) * 2);
        stg256(dst + row * K + k, w);
        if constexpr (sizeof(T) == 4) stg256(dst + row * K + k + 8, w + 8);
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
// A k-block is 256 elements of K: 128-byte rows of codes (128-byte swizzle, one
// TMA box per operand) and the scale tiles of both operands.
//
// What bounds it: at the fp4 rate a pair's 256 x 256 tile takes 512 cycles per
// k-block, in which streaming both operands would move 32 KB to each SM, more
// than L2 delivers (loads alone took 127 us of the 32768-token layer's gate/up,
// the MMAs 91).  So a pair keeps the A rows of a row tile in shared memory
// (up to 8 k-blocks, K <= 2048; longer rows are streamed) and walks over a run of
// column tiles, streaming B.  The scales go to TMEM by tcgen05.st from four
// warps instead of tcgen05.cp, whose copies occupy the tensor pipe (49 us of
// the same product).
//
// TMEM: one 256-column accumulator and eight 32-column slots of scales (8 columns
// for A, 16 for B, one slot per B stage).  The epilogue warps read the whole
// accumulator at once, release it, and finish from registers while the next
// tile's MMAs run.
//
// Warps: 0 TMA producer of codes, 1 MMA issuer (the leader CTA's), 2 TMA producer of
// scales, 3 unit scheduler, 4..7 scales to TMEM, 8..15 epilogue (two per TMEM lane
// quarter).
enum Mode { GATEUP = 0, DOWN = 1 };

constexpr int BM = 128;
constexpr int TILE_M = 2 * BM;
constexpr int TN = 256;
constexpr int BKE = 256;           // elements of K per k-block
constexpr int A_BUFS = 8;          // most k-blocks of A in shared memory
constexpr int B_STAGES = 8;        // most stages of B (and TMEM scale slots)
constexpr int U_RING = 4;          // decoded units ahead of their use
constexpr uint32_t A_BYTES = BM * 128;
constexpr uint32_t B_BYTES = (TN / 2) * 128;
constexpr uint32_t SF_BYTES = 3 * 1024;  // two K tiles of this CTA's 128 rows and of both 128-column halves
constexpr int SF_FIRST = 4, EPI_FIRST = 8, EPI_WARPS = 8;
constexpr int THREADS = 32 * (EPI_FIRST + EPI_WARPS);
constexpr uint32_t BOX_BYTES = 32 * 64;  // an epilogue warp's staging box: 32 rows x 32 bf16
constexpr uint32_t SF_COL = 256;         // first scale column
constexpr uint32_t TMEM_COLS = 512;
constexpr size_t kSmemLimit = 232448;
// Registers: launched at 128 per thread (512 threads), then 56 for the producer and
// scale warpgroups and 200 for the two of the epilogue: 256 * 56 + 256 * 200 = 512 * 128.
constexpr int LAUNCH_REGS = 128, REG_LOW = 56, REG_EPI = 200;
static_assert(256 * REG_LOW + 256 * REG_EPI <= THREADS * LAUNCH_REGS, "the split must fit the launch allocation");

struct Params {
  const int32_t* offsets;  // [segs] inclusive row ends
  int segs;                // row segments; segment g multiplies expert g % experts
  int experts;
  int64_t S;
  int K, N;                // reduction length; output columns (I or H)
  int n_tiles;
  int w_blocks;            // row tiles of one expert's scales
  int has_ext;
  int a_bufs, b_stages;    // ring sizes
  int resident;            // 1: a row tile's A stays for the unit's whole run
  __nv_bfloat16* out;      // h [S, I] or y [S, H]; GATEUP: may be null when hq is wanted alone
  void* gate_up;           // GATEUP: optional [S, 2I] ...
  int gate_up_f32;         // ... in bf16, or fp32
  uint8_t* hq;             // GATEUP: optional packed h [S, I/2] ...
  uint8_t* hscale;         // ... and its scale tiles
  int64_t h_blocks;        // row tiles of hscale
  int h_kt;
};

struct alignas(16) Smem {
  uint64_t a_full[A_BUFS];      // leader: both CTAs' bytes
  uint64_t a_empty[A_BUFS];
  uint64_t b_full[B_STAGES];    // leader: both CTAs' bytes and scale warps
  uint64_t b_empty[B_STAGES];
  uint64_t sf_full[B_STAGES];   // this CTA's scale bytes
  uint64_t u_full[U_RING];
  uint64_t u_empty[U_RING];
  uint64_t tfull;
  uint64_t tempty;              // leader: both CTAs' epilogue warps
  uint32_t tmem_base;
  int abort_flag;
  int4 units[U_RING][2];        // decoded units: {row, end, expert, scale block}, {n0, n1, more, -}
  // followed by row_start, tile_prefix, blk_prefix [segs + 1]
};
struct Table {  // the segment table behind Smem
  int* row_start;
  int* tile_prefix;  // 256-row tiles before a segment
  int* blk_prefix;   // 128-row scale blocks before it
};
__host__ __device__ inline size_t table_bytes(int segs) { return ((size_t)3 * (segs + 1) * sizeof(int) + 15) / 16 * 16; }
__device__ __forceinline__ Table table_of(Smem& sm, int segs) {
  int* t = reinterpret_cast<int*>(&sm + 1);
  return Table{t, t + segs + 1, t + 2 * (segs + 1)};
}
inline size_t smem_bytes(int a_bufs, int b_stages, int segs) {
  return 1024 + (size_t)a_bufs * A_BYTES + (size_t)b_stages * (B_BYTES + SF_BYTES) +
         EPI_WARPS * BOX_BYTES + sizeof(Smem) + table_bytes(segs);
}

// Instruction descriptor of kind::mxf4: E2M1 operands, both K-major, UE8M0
// scales; sf_id (0 or 2) picks the two scale bytes of the K = 64 step.
__device__ __forceinline__ constexpr uint32_t idesc_mxf4(int M, int N, uint32_t sf_id) {
  return (sf_id << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | (1u << 23) | ((uint32_t)(M >> 4) << 24) |
         (sf_id << 29);
}

// Shared-memory descriptors are built from their low words (address / 16, the only
// part that changes) to keep the issuing thread's instructions few: it shares its
// scheduler with epilogue warps, and every instruction between two MMAs is a gap.
constexpr uint32_t DESC_HI = (1024u >> 4) | (1u << 14) | (2u << 29);  // 8-row groups 1 KB apart, sm_100, 128-byte swizzle
__device__ __forceinline__ uint32_t desc_lo(uint32_t smem_addr) { return ((smem_addr & 0x3FFFF) >> 4) | (1u << 16); }

__device__ __forceinline__ void umma_mxf4_pair(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t sfa,
                                               uint32_t sfb, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
      "mov.b64 da, {%1, %7};\n\t"
      "mov.b64 db, {%2, %7};\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], da, db, %3, [%4], [%5], p;\n\t}" ::"r"(d),
      "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate), "r"(DESC_HI)
      : "memory");
}

// Eight columns of this warp's 32 TMEM lanes.
__device__ __forceinline__ void tmem_st_x8(uint32_t taddr, uint4 a, uint4 b) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(a.x),
               "r"(a.y), "r"(a.z), "r"(a.w), "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w)
               : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

// An odd number of blocks (K % 64 == 32): the last K = 64 step reads one block past the row, whose codes
// are zeros (TMA fill).  Its scale must not be the NaN byte, which a key's padding may hold: the words' byte
// is cleared.  `blocks`: those of the last k-block; four per word, two words (K tiles) per row.
struct PadMask {
  uint32_t keep0, keep1;
};
__device__ __forceinline__ PadMask pad_mask(int blocks) {
  const uint32_t m = ~(0xffu << (8 * (blocks & 3)));
  return PadMask{blocks < 4 ? m : ~0u, blocks < 4 ? ~0u : m};
}
__device__ __forceinline__ void keep_bytes(uint4& v, uint32_t m) { v.x &= m, v.y &= m, v.z &= m, v.w &= m; }

// Bring a box of a tensor map into L2.
__device__ __forceinline__ void tma_prefetch_2d(const CUtensorMap* map, int x, int y) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(reinterpret_cast<uint64_t>(map)),
               "r"(x), "r"(y)
               : "memory");
}

// True in one lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}

// g / (1 + 2^(-g log2 e)) in four instructions: the flushing approximations (2^-22
// relative) drop the subnormal handling of expf and a division, which doubled the
// gate/up epilogue's instructions.  g below -88 gives -0.
__device__ __forceinline__ float silu(float g) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  return g * r;
}

template <int N> __device__ __forceinline__ void regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// Segment table shared by every role: first rows, and exclusive prefixes of the
// 256-row tiles and of the 128-row scale blocks.  All threads take part.
__device__ __forceinline__ void build_segments(const Table& tb, const int32_t* offsets, int segs, int64_t S, int site) {
  for (int g = threadIdx.x; g < segs; g += THREADS) {
    int begin;
    const int rows = segment_rows(offsets, g, S, begin, site);
    tb.row_start[g] = begin;
    tb.blk_prefix[g] = rows;  // until the scan below
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int tiles = 0, blocks = 0;
    for (int g0 = 0; g0 < segs; g0 += 32) {
      const int g = g0 + lane;
      const int rows = g < segs ? tb.blk_prefix[g] : 0;
      const int t = (rows + TILE_M - 1) / TILE_M, b = (rows + BM - 1) / BM;
      int ti = t, bi = b;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int tv = __shfl_up_sync(0xffffffffu, ti, o), bv = __shfl_up_sync(0xffffffffu, bi, o);
        if (lane >= o) ti += tv, bi += bv;
      }
      if (g < segs) {
        tb.tile_prefix[g] = tiles + ti - t;
        tb.blk_prefix[g] = blocks + bi - b;
        if (g == segs - 1) tb.row_start[segs] = tb.row_start[g] + rows;
      }
      tiles += __shfl_sync(0xffffffffu, ti, 31);
      blocks += __shfl_sync(0xffffffffu, bi, 31);
    }
    if (lane == 0) tb.tile_prefix[segs] = tiles, tb.blk_prefix[segs] = blocks;
  }
}

// mbar_wait by a whole warp, with one answer: its lanes go on, or give up, together, so that the
// warp-wide instructions behind it (tcgen05.ld / .st, shuffles) and a slot that lane 0 frees
// for all of them never meet a part of the warp.
__device__ __forceinline__ bool mbar_wait_warp(uint64_t* bar, uint32_t parity, int where) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, where));
}

struct Ring {  // position in a ring of buffers
  int i = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next(int size) {
    if (++i == size) i = 0, phase ^= 1;
  }
};

// A unit of work: a row tile and a run of column tiles.  As many row tiles as fill every
// pair equally often are walked whole; the rest are cut into runs, as long as they
// keep the pairs that end last short, so that all pairs end together (whole row tiles
// alone leave a third of the pairs idle for a quarter of the 32768-token layer).  Runs
// are the outer index: the pairs at work together share experts' B tiles in L2.
// One warp decodes units ahead of their use into a ring of shared memory: decoding in
// every role cost 2 us at each change of unit.
struct Unit {
  int row, end;  // first row of the pair's tile, end of its segment
  int expert;
  int blk;       // first of the tile's two scale blocks
  int n0, n1;
};
struct Schedule {
  int whole;  // units of a whole row tile
  int rest;   // row tiles cut into runs
  int run;    // column tiles of a run
  int units;
};
// By a whole warp: each lane weighs some lengths, a tile counting its B stream and a unit half a
// tile more for its A.  Streamed A (not resident) makes every tile a unit.
__device__ __forceinline__ Schedule make_schedule(int tiles, int pairs, const Params& p) {
  Schedule s;
  s.whole = p.resident ? tiles / pairs * pairs : 0;
  s.rest = tiles - s.whole;
  uint32_t best = 0xffffffffu;
  for (int r = (threadIdx.x & 31) + 1; r <= (p.resident ? p.n_tiles : 1); r += 32) {
    const int64_t rounds = ((int64_t)s.rest * ((p.n_tiles + r - 1) / r) + pairs - 1) / pairs;
    const uint32_t cost = (uint32_t)min((int64_t)0x3fffff, rounds * (2 * r + 1));
    best = min(best, cost << 10 | (uint32_t)min(r, 1023));  // the shortest run of the cheapest
  }
  s.run = (int)(__reduce_min_sync(0xffffffffu, best) & 1023u);
  s.units = s.whole + s.rest * ((p.n_tiles + s.run - 1) / s.run);
  return s;
}
__device__ __forceinline__ Unit decode_unit(const Table& tb, int u, const Schedule& s, const Params& p) {
  int mt = u, n0 = 0, n1 = p.n_tiles;
  if (u >= s.whole) {
    const int run = (u - s.whole) / s.rest;
    mt = s.whole + (u - s.whole) - run * s.rest;
    n0 = run * s.run;
    n1 = min(p.n_tiles, n0 + s.run);
  }
  int lo = 0, hi = p.segs;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (tb.tile_prefix[mid] <= mt) lo = mid;
    else hi = mid;
  }
  const int m = mt - tb.tile_prefix[lo];
  return Unit{tb.row_start[lo] + m * TILE_M, tb.row_start[lo + 1], lo % p.experts, tb.blk_prefix[lo] + 2 * m, n0, n1};
}
// The next unit, false after the last one (or a wait that gave up).  WARP: the whole warp
// calls it; otherwise one lane does.  The slot is freed once every caller has read it.
template <bool WARP> __device__ __forceinline__ bool next_unit(Smem& sm, Ring& r, Unit& u, int site) {
  if (!(WARP ? mbar_wait_warp(&sm.u_full[r.i], r.phase, site) : mbar_wait(&sm.u_full[r.i], r.phase, site))) {
    *(volatile int*)&sm.abort_flag = 1;
    return false;
  }
  const int4 a = sm.units[r.i][0], b = sm.units[r.i][1];
  u = Unit{a.x, a.y, a.z, a.w, b.x, b.y};
  if (WARP) __syncwarp();
  if (!WARP || (threadIdx.x & 31) == 0) mbar_arrive(&sm.u_empty[r.i]);
  r.next(U_RING);
  const bool more = b.z != 0 && !*(volatile int*)&sm.abort_flag;
  return WARP ? __all_sync(0xffffffffu, more) : more;
}

template <int MODE>
__global__ void __launch_bounds__(THREADS, 1)
    product_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_sa,
                   const __grid_constant__ CUtensorMap tmap_b0, const __grid_constant__ CUtensorMap tmap_b1,
                   const __grid_constant__ CUtensorMap tmap_sb0, const __grid_constant__ CUtensorMap tmap_sb1,
                   const __grid_constant__ CUtensorMap tmap_xa, const __grid_constant__ CUtensorMap tmap_xb,
                   const __grid_constant__ CUtensorMap tmap_o0, const __grid_constant__ CUtensorMap tmap_o1,
                   const __grid_constant__ CUtensorMap tmap_o2, const __grid_constant__ Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = base;
  uint8_t* sB = sA + p.a_bufs * A_BYTES;
  uint8_t* sBox = sB + p.b_stages * B_BYTES;
  uint8_t* sSF = sBox + EPI_WARPS * BOX_BYTES;  // per stage: A tiles, then B's two halves
  Smem& sm = *reinterpret_cast<Smem*>(sSF + p.b_stages * SF_BYTES);
  const Table tb = table_of(sm, p.segs);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;

  if (warp == 1) {
    if (lane == 0) {
      for (int i = 0; i < A_BUFS; ++i) {
        mbar_init(&sm.a_full[i], 1);
        mbar_init(&sm.a_empty[i], 1);
      }
      for (int i = 0; i < B_STAGES; ++i) {
        mbar_init(&sm.b_full[i], 1 + 2 * 4);  // the leader's producer, and the scale warps of both CTAs
        mbar_init(&sm.b_empty[i], 1);
        mbar_init(&sm.sf_full[i], 1);
      }
      for (int i = 0; i < U_RING; ++i) {
        mbar_init(&sm.u_full[i], 1);
        // two producers, four scale warps, the epilogue, and the leader's MMA issuer
        mbar_init(&sm.u_empty[i], 2 + 4 + EPI_WARPS + (leader ? 1 : 0));
      }
      mbar_init(&sm.tfull, 1);
      mbar_init(&sm.tempty, 2 * EPI_WARPS);
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
  // Nothing above touches global memory: the kernel may be launched before the one in front of it
  // in the stream has ended.  Every thread waits for that one here.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  build_segments(tb, p.offsets, p.segs, p.S, 710 + MODE);
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  tc_fence_after();

  const uint32_t tmem = sm.tmem_base;
  if (tmem != 0 && threadIdx.x == 0) device_fail(MIRAI_ERR_DEVICE_BOUNDS, 715);  // cannot be: see the MMA issuer
  const int num_kb = (p.K + BKE - 1) / BKE;
  const int total_kb = num_kb + p.has_ext;
  volatile int* abort_flag = &sm.abort_flag;

  if (warp < SF_FIRST) {
    regs_dec<REG_LOW>();
    if (warp == 3) {
      // ======================= unit scheduler =======================
      const int pairs = (int)(gridDim.x >> 1);
      const Schedule sched = make_schedule(tb.tile_prefix[p.segs], pairs, p);
      Ring r;
      for (int u = (int)(blockIdx.x >> 1); lane == 0; u += pairs) {
        const bool more = u < sched.units;
        Unit un = {};
        if (more) {
          un = decode_unit(tb, u, sched, p);
          // The pairs change row tiles at about the same time: bring the rows into L2 ahead of that
          // burst (19 MB at 148 SMs).  (Boxes that reach past the last row are left out: prefetching
          // them took 17 us of a 16-row call.)
          if (p.resident && un.row + (int)rank * BM + BM <= p.S)
            for (int kb = 0; kb < num_kb; ++kb) tma_prefetch_2d(&tmap_a, kb * 128, un.row + (int)rank * BM);
        }
        if (!mbar_wait(&sm.u_empty[r.i], r.phase ^ 1, 85)) {
          *abort_flag = 1;
          break;
        }
        sm.units[r.i][0] = make_int4(un.row, un.end, un.expert, un.blk);
        sm.units[r.i][1] = make_int4(un.n0, un.n1, more, 0);
        mbar_arrive(&sm.u_full[r.i]);
        r.next(U_RING);
        if (!more) break;
      }
    } else if (warp == 0 && lane == 0) {
      // ======================= TMA producer =======================
      const uint32_t a_full0 = mapa_shared(smem_u32(&sm.a_full[0]), 0), b_full0 = mapa_shared(smem_u32(&sm.b_full[0]), 0);
      Ring ra, rb, ru;
      Unit un;
      while (next_unit<false>(sm, ru, un, 80)) {
        const int e = un.expert, row = un.row + (int)rank * BM;
        const CUtensorMap* mb = MODE == GATEUP && rank ? &tmap_b1 : &tmap_b0;
        for (int n = un.n0; n < un.n1 && !*abort_flag; ++n) {
          const int brow = e * p.N + (MODE == GATEUP ? n * BM : n * TN + (int)rank * BM);  // B rows of this CTA
          for (int kb = 0; kb < total_kb; ++kb) {
            const bool ext = kb == num_kb;
            if (n == un.n0 || !p.resident) {
              if (!mbar_wait(&sm.a_empty[ra.i], ra.phase ^ 1, 70)) {
                *abort_flag = 1;
                break;
              }
              // the leader's own barrier carries the bytes of both CTAs
              if (leader) mbar_arrive_expect_tx(&sm.a_full[ra.i], 2 * A_BYTES);
              tma_load_2d_pair(sA + ra.i * A_BYTES, ext ? &tmap_xa : &tmap_a, ext ? 0 : kb * 128, row, a_full0 + 8u * ra.i);
              ra.next(p.a_bufs);
            }
            if (!mbar_wait(&sm.b_empty[rb.i], rb.phase ^ 1, 71)) {
              *abort_flag = 1;
              break;
            }
            if (leader) mbar_arrive_expect_tx(&sm.b_full[rb.i], 2 * B_BYTES);
            tma_load_2d_pair(sB + rb.i * B_BYTES, ext ? &tmap_xb : mb, ext ? 0 : kb * 128, brow, b_full0 + 8u * rb.i);
            rb.next(p.b_stages);
          }
        }
      }
      // no commit of the leader may reach this CTA after it has exited
      for (int i = 0; i < p.b_stages; ++i) {
        if (!mbar_wait(&sm.b_empty[rb.i], rb.phase ^ 1, 72)) break;
        rb.next(p.b_stages);
      }
      for (int i = 0; i < p.a_bufs; ++i) {
        if (!mbar_wait(&sm.a_empty[ra.i], ra.phase ^ 1, 73)) break;
        ra.next(p.a_bufs);
      }
    } else if (warp == 2 && lane == 0) {
      // ======================= TMA producer of the scales =======================
      Ring rb, ru;
      Unit un;
      while (next_unit<false>(sm, ru, un, 81)) {
        const int e = un.expert, ablk = un.blk + (int)rank;
        for (int n = un.n0; n < un.n1 && !*abort_flag; ++n) {
          // row tiles of both column halves
          const int bblk = e * p.w_blocks + (MODE == GATEUP ? n : 2 * n);
          for (int kb = 0; kb < total_kb; ++kb) {
            if (!mbar_wait(&sm.b_empty[rb.i], rb.phase ^ 1, 79)) {
              *abort_flag = 1;
              break;
            }
            uint64_t* sf = &sm.sf_full[rb.i];
            if (kb == num_kb) {
              mbar_arrive(sf);  // the rank block has no scales
            } else {
              uint8_t* dst = sSF + rb.i * SF_BYTES;
              mbar_arrive_expect_tx(sf, SF_BYTES);
              tma_load_2d(dst, &tmap_sa, kb * 256, ablk, sf);
              tma_load_2d(dst + 1024, &tmap_sb0, kb * 256, bblk, sf);
              tma_load_2d(dst + 2048, MODE == GATEUP ? &tmap_sb1 : &tmap_sb0, kb * 256, MODE == GATEUP ? bblk : bblk + 1, sf);
            }
            rb.next(p.b_stages);
          }
        }
      }
    } else if (warp == 1 && leader) {
      // ======================= MMA issuer =======================
      // The whole warp runs the loop, so that its operands stay in uniform
      // registers; one elected lane issues.
      const bool issue = elect_one();
      constexpr uint32_t id_ext = make_idesc_bf16(TILE_M, TN);
      constexpr uint32_t id0 = idesc_mxf4(TILE_M, TN, 0), id2 = idesc_mxf4(TILE_M, TN, 2);
      const uint32_t a_lo0 = desc_lo(smem_u32(sA)), b_lo0 = desc_lo(smem_u32(sB));
      const int last_steps = (p.K - (num_kb - 1) * BKE + 63) / 64;  // K = 64 steps of the last k-block
      Ring ra, rb, ru;
      Unit un;
      constexpr uint32_t acc = 0;  // all 512 columns are this CTA's: they start at 0 (checked above)
      uint32_t tiles = 0;
      bool ok = true;
      while (ok && next_unit<true>(sm, ru, un, 82)) {
        const Ring ra0 = ra;
        for (int n = un.n0; n < un.n1 && ok; ++n, ++tiles) {
          if (p.resident) ra = ra0;
          const bool first = n == un.n0 || !p.resident, last = n + 1 == un.n1 || !p.resident;
          // (the first k-block's operands are waited for before the accumulator: they come first)
          if ((first && !mbar_wait_warp(&sm.a_full[ra.i], ra.phase, 75)) ||
              !mbar_wait_warp(&sm.b_full[rb.i], rb.phase, 76) ||
              (tiles > 0 && !mbar_wait_warp(&sm.tempty, (tiles - 1) & 1, 74)))
            ok = false;
          for (int kb = 0; kb < total_kb && ok; ++kb) {
            if (kb > 0 && ((first && !mbar_wait_warp(&sm.a_full[ra.i], ra.phase, 75)) ||
                           !mbar_wait_warp(&sm.b_full[rb.i], rb.phase, 76))) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t a = a_lo0 + ra.i * (A_BYTES >> 4), b = b_lo0 + rb.i * (B_BYTES >> 4);
            const uint32_t sf = SF_COL + rb.i * 32;
            if (issue) {
              if (kb < num_kb - 1 || (kb < num_kb && last_steps == 4)) {
                umma_mxf4_pair(acc, a, b, id0, sf, sf + 8, kb != 0);
                umma_mxf4_pair(acc, a + 2, b + 2, id2, sf, sf + 8, 1);
                umma_mxf4_pair(acc, a + 4, b + 4, id0, sf + 4, sf + 16, 1);
                umma_mxf4_pair(acc, a + 6, b + 6, id2, sf + 4, sf + 16, 1);
              } else if (kb < num_kb) {
                umma_mxf4_pair(acc, a, b, id0, sf, sf + 8, kb != 0);
                if (last_steps > 1) umma_mxf4_pair(acc, a + 2, b + 2, id2, sf, sf + 8, 1);
                if (last_steps > 2) umma_mxf4_pair(acc, a + 4, b + 4, id0, sf + 4, sf + 16, 1);
              } else {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                  umma_bf16_pair(acc, ((uint64_t)DESC_HI << 32) | (a + 2 * k), ((uint64_t)DESC_HI << 32) | (b + 2 * k),
                                 id_ext, 1u);
              }
              umma_commit_pair(&sm.b_empty[rb.i], 0x3);
              if (last) umma_commit_pair(&sm.a_empty[ra.i], 0x3);
            }
            __syncwarp();
            rb.next(p.b_stages);
            ra.next(p.a_bufs);
          }
          if (ok && issue) umma_commit_pair(&sm.tfull, 0x3);
          __syncwarp();
        }
      }
      if (!ok && lane == 0) *abort_flag = 1;
    }
  } else if (warp < EPI_FIRST) {
    // ======================= scales: shared memory -> TMEM =======================
    // A scale tile is 32 lanes x 16 bytes: lane l holds rows l, l + 32, l + 64, l + 96,
    // one column each; every lane quarter gets a copy, its own warp's.
    regs_dec<REG_LOW>();
    const uint32_t quarter = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t b_full0 = mapa_shared(smem_u32(&sm.b_full[0]), 0);
    Ring rb, ru;
    Unit un;
    while (next_unit<true>(sm, ru, un, 83)) {
      const int blocks = (un.n1 - un.n0) * total_kb;
      int kb = 0;
      for (int i = 0; i < blocks; ++i) {
        if (!mbar_wait_warp(&sm.sf_full[rb.i], rb.phase, 77)) {
          *abort_flag = 1;
          break;
        }
        if (kb != num_kb) {
          tc_fence_after();  // the MMAs that read this slot have completed (the stage was refilled after them)
          const uint32_t src = smem_u32(sSF + rb.i * SF_BYTES) + lane * 16u;
          const uint32_t dst = tmem + SF_COL + rb.i * 32 + quarter;
          uint4 a0 = lds128(src), a1 = lds128(src + 512);
          uint4 l0 = lds128(src + 1024), l1 = lds128(src + 1536), h0 = lds128(src + 2048), h1 = lds128(src + 2560);
          if (kb == num_kb - 1 && p.K % 64) {
            const PadMask m = pad_mask(p.K % BKE / 32);
            keep_bytes(a0, m.keep0), keep_bytes(l0, m.keep0), keep_bytes(h0, m.keep0);
            keep_bytes(a1, m.keep1), keep_bytes(l1, m.keep1), keep_bytes(h1, m.keep1);
          }
          tmem_st_x8(dst, a0, a1);
          tmem_st_x8(dst + 8, l0, h0);    // K tile 0: both column halves
          tmem_st_x8(dst + 16, l1, h1);   // K tile 1
          tmem_st_wait();
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(b_full0 + 8u * rb.i);
        rb.next(p.b_stages);
        kb = kb + 1 == total_kb ? 0 : kb + 1;
      }
    }
  } else {
    // ======================= epilogue =======================
    regs_inc<REG_EPI>();
    const int q = warp & 3;                  // TMEM lane quarter
    const int part = (warp - EPI_FIRST) / 4;  // its half of the columns
    const uint32_t tempty_leader = mapa_shared(smem_u32(&sm.tempty), 0);
    const uint32_t acc = tmem + ((uint32_t)(q * 32) << 16);
    uint8_t* box = sBox + (warp - EPI_FIRST) * BOX_BYTES;
    const uint32_t box_row = smem_u32(box) + (uint32_t)lane * 64u;
    const uint32_t box_sw = (uint32_t)(lane >> 1) & 3u;  // 64-byte swizzle: 16-byte chunk ^= row bits 1..2
    uint32_t tiles = 0;
    Ring ru;
    Unit un;
    while (next_unit<true>(sm, ru, un, 84)) {
      const int64_t row = (int64_t)un.row + (int)rank * BM + q * 32 + lane;
      const bool valid = row < un.end;
      const bool boxed = __all_sync(0xffffffffu, valid);  // all 32 rows are the segment's
      const int row0 = (int)(row - lane);
      // 32 rows x 32 bf16 columns (16 fp32 ones): through the staging box and one TMA store, or row by row.  (A lane
      // storing its own row straight to global memory touches 32 lines per store: 33 us more on the
      // 32768-token layer's gate/up.)
      auto store = [&](const CUtensorMap* map, void* dst, int col, const uint32_t* w) {
        if (boxed) {
          if (lane == 0) bulk_wait_group_read<0>();  // the box's previous store has read it
          __syncwarp();
#pragma unroll
          for (int v = 0; v < 4; ++v)
            sts128(box_row + (((uint32_t)v ^ box_sw) << 4), w[4 * v], w[4 * v + 1], w[4 * v + 2], w[4 * v + 3]);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(map, box, col, row0);
            bulk_commit_group();
          }
        } else if (valid) {
#pragma unroll
          for (int v = 0; v < 4; ++v)
            reinterpret_cast<uint4*>(dst)[v] = make_uint4(w[4 * v], w[4 * v + 1], w[4 * v + 2], w[4 * v + 3]);
        }
      };
      bool ok = true;
      for (int n = un.n0; n < un.n1 && ok; ++n, ++tiles) {
        if (!mbar_wait_warp(&sm.tfull, tiles & 1, 78)) {
          *abort_flag = 1;
          ok = false;
          break;
        }
        __syncwarp();
        tc_fence_after();
        uint32_t v[4][32];
        // GATEUP: channels of chunks 2 part, 2 part + 1: gate in v[0], v[1], up in v[2], v[3].
        // DOWN: column chunks 4 part .. 4 part + 3.
#pragma unroll
        for (int i = 0; i < 4; ++i)
          tmem_ld_32x32b_x32(acc + (MODE == GATEUP ? (i / 2) * BM + part * 64 + (i % 2) * 32 : part * BM + i * 32), v[i]);
        tmem_ld_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(tempty_leader);
        if constexpr (MODE == GATEUP) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int c = 2 * part + i;
            const int col = n * BM + c * 32;
            if (col >= p.N) break;  // warp-uniform
            uint32_t w[16];
            if (p.gate_up && p.gate_up_f32) {
              float* dst = static_cast<float*>(p.gate_up) + row * 2 * (int64_t)p.N + col;
              store(&tmap_o1, dst, col, v[i]);
              store(&tmap_o1, dst + 16, col + 16, v[i] + 16);
              store(&tmap_o2, dst + p.N, col, v[i + 2]);
              store(&tmap_o2, dst + p.N + 16, col + 16, v[i + 2] + 16);
            } else if (p.gate_up) {
              __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(p.gate_up) + row * 2 * (int64_t)p.N + col;
#pragma unroll
              for (int j = 0; j < 16; ++j) w[j] = pack_bf16x2(__uint_as_float(v[i][2 * j]), __uint_as_float(v[i][2 * j + 1]));
              store(&tmap_o1, dst, col, w);
#pragma unroll
              for (int j = 0; j < 16; ++j)
                w[j] = pack_bf16x2(__uint_as_float(v[i + 2][2 * j]), __uint_as_float(v[i + 2][2 * j + 1]));
              store(&tmap_o2, dst + p.N, col, w);
            }
#pragma unroll
            for (int j = 0; j < 16; ++j)
              w[j] = pack_bf16x2(silu(__uint_as_float(v[i][2 * j])) * __uint_as_float(v[i + 2][2 * j]),
                                 silu(__uint_as_float(v[i][2 * j + 1])) * __uint_as_float(v[i + 2][2 * j + 1]));
            if (p.out) store(&tmap_o0, p.out + row * p.N + col, col, w);
            if (p.hq && valid) {
              // this lane's 32 channels are one block of the quantised h
              uint32_t m = 0;
#pragma unroll
              for (int j = 0; j < 16; ++j) m = max(m, max((w[j] << 16) & 0x7fffffffu, w[j] & 0x7fff0000u));
              const uint32_t byte = scale_byte(m);
              const float inv = inv_scale(byte == 255u ? 254u : byte);
              uint32_t codes[4];
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                float f[8];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                  f[2 * j] = bf16_lo(w[4 * x + j]) * inv, f[2 * j + 1] = bf16_hi(w[4 * x + j]) * inv;
                codes[x] = byte == 255u ? 0u : e2m1x8(f);
              }
              *reinterpret_cast<uint4*>(p.hq + (row * p.N + col) / 2) = make_uint4(codes[0], codes[1], codes[2], codes[3]);
              const int64_t blk = un.blk + (int)rank;
              if (blk < p.h_blocks) {
                uint8_t* word = p.hscale + (blk * p.h_kt + n) * 512 + lane * 16 + q * 4;
                word[c] = (uint8_t)byte;
                if (col + 32 == p.N)  // blocks past the row's end are zero bytes
                  for (int z = c + 1; z < 4; ++z) word[z] = 0;
              }
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int col = n * TN + part * BM + i * 32;
            if (col >= p.N) break;  // warp-uniform
            uint32_t w[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) w[j] = pack_bf16x2(__uint_as_float(v[i][2 * j]), __uint_as_float(v[i][2 * j + 1]));
            store(&tmap_o0, p.out + row * p.N + col, col, w);
          }
        }
      }
    }
    if (lane == 0) bulk_wait_group_all();  // the stores have read the box before the CTA exits
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
// The same products for few rows (a generation step): the weights are read once
// and nothing else counts, so the roles of the operands are exchanged -- 128
// channels of the weights are the MMA's M, up to 32 rows its N -- and a tile is
// one SM's: 128 channels of gate and the same 128 of up (DOWN: 128 outputs) of one
// segment.  The rows come in bf16 and are quantised here, into the swizzled operand,
// while the weights are on their way: one launch instead of two, no row buffer.
// A lane of the accumulator is a channel, a column a row, so a warp stores 64
// contiguous bytes of h per row.
//
// Warps: 0 TMA producer, 1 MMA issuer, 4..11 quantise the rows, 4..7 then move scales to
// TMEM and are the epilogue.
constexpr int FEW_ROWS = 32;    // rows of a tile
constexpr int FEW_STAGES = 6;   // most weight stages (and TMEM scale slots)
constexpr int FEW_QUANT = 8;    // quantising warps
constexpr int FEW_THREADS = 32 * (4 + FEW_QUANT);
constexpr int FEW_MAX_K = 4096;
constexpr uint32_t FEW_SF_COL = 64;
constexpr uint32_t FEW_COLS = 256;

struct FewParams {
  const __nv_bfloat16* x;  // [S, K]
  const int32_t* offsets;
  int segs, experts;
  int64_t S;
  int K, N;
  int n_tiles, w_blocks, stages;
  __nv_bfloat16* out;      // [S, N]
  void* gate_up;           // GATEUP: optional [S, 2N] in bf16, or fp32
  int gate_up_f32;
};

struct alignas(16) FewSmem {
  uint64_t full[FEW_STAGES];     // the producer (bytes of codes) and four scale warps
  uint64_t empty[FEW_STAGES];
  uint64_t sf_full[FEW_STAGES];  // bytes of scales
  uint64_t rows_ready;           // quantising warps
  uint64_t tfull, tempty;
  uint32_t tmem_base;
  int abort_flag;
  // followed by the segments' first rows and tile prefixes [segs + 1] each
};
template <int MODE> constexpr uint32_t few_stage_bytes() { return (MODE == GATEUP ? 2 : 1) * (A_BYTES + 1024); }
template <int MODE> static size_t few_smem_bytes(int stages, int K, int segs) {
  const int kbs = (K + BKE - 1) / BKE;
  return 1024 + (size_t)stages * few_stage_bytes<MODE>() + (size_t)kbs * (FEW_ROWS * 128 + 256) + sizeof(FewSmem) +
         ((size_t)2 * (segs + 1) * sizeof(int) + 15) / 16 * 16;
}

__device__ __forceinline__ void umma_mxf4(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t sfa,
                                          uint32_t sfb, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
      "mov.b64 da, {%1, %7};\n\t"
      "mov.b64 db, {%2, %7};\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], da, db, %3, [%4], [%5], p;\n\t}" ::"r"(d),
      "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate), "r"(DESC_HI)
      : "memory");
}

template <int MODE>
__global__ void __launch_bounds__(FEW_THREADS, 1)
    few_rows_kernel(const __grid_constant__ CUtensorMap tmap_w0, const __grid_constant__ CUtensorMap tmap_w1,
                    const __grid_constant__ CUtensorMap tmap_s0, const __grid_constant__ CUtensorMap tmap_s1,
                    const __grid_constant__ FewParams p) {
  constexpr int KEYS = MODE == GATEUP ? 2 : 1;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int num_kb = (p.K + BKE - 1) / BKE;
  uint8_t* sW = base;                                            // per stage: KEYS x 16 KB of codes
  uint8_t* sX = sW + p.stages * KEYS * A_BYTES;                  // per k-block: 32 rows x 128 bytes (swizzled)
  uint8_t* sSF = sX + num_kb * FEW_ROWS * 128;                   // per stage: KEYS x 1 KB of weight scales
  uint32_t* sXS = reinterpret_cast<uint32_t*>(sSF + p.stages * KEYS * 1024);  // per K tile: 32 words of row scales
  FewSmem& sm = *reinterpret_cast<FewSmem*>(reinterpret_cast<uint8_t*>(sXS) + num_kb * 256);
  int* row_start = reinterpret_cast<int*>(&sm + 1);
  int* prefix = row_start + p.segs + 1;  // (first the segments' rows, then tiles before each)

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int g = threadIdx.x; g < p.segs; g += FEW_THREADS) {
    int begin;
    prefix[g] = segment_rows(p.offsets, g, p.S, begin, 720 + MODE);
    row_start[g] = begin;
  }
  if (warp == 1) {
    if (lane == 0) {
      for (int i = 0; i < FEW_STAGES; ++i) {
        mbar_init(&sm.full[i], 1 + 4);
        mbar_init(&sm.empty[i], 1);
        mbar_init(&sm.sf_full[i], 1);
      }
      mbar_init(&sm.rows_ready, FEW_QUANT);
      mbar_init(&sm.tfull, 1);
      mbar_init(&sm.tempty, 4);
      sm.abort_flag = 0;
      fence_mbar_init();
    }
    __syncwarp();
    tmem_alloc(&sm.tmem_base, FEW_COLS);
    tmem_relinquish();
  }
  if (warp == 2 && lane == 0) {
    prefetch_tmap(&tmap_w0);
    prefetch_tmap(&tmap_s0);
    if (KEYS == 2) {
      prefetch_tmap(&tmap_w1);
      prefetch_tmap(&tmap_s1);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {  // tiles (32 rows) before each segment
    int carry = 0;
    for (int g0 = 0; g0 < p.segs; g0 += 32) {
      const int g = g0 + lane;
      const int rows = g < p.segs ? prefix[g] : 0;
      const int n = (rows + FEW_ROWS - 1) / FEW_ROWS;
      int incl = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      if (g < p.segs) {
        prefix[g] = carry + incl - n;
        if (g == p.segs - 1) row_start[p.segs] = row_start[g] + rows;
      }
      carry += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) prefix[p.segs] = carry;
  }
  __syncthreads();
  tc_fence_after();

  const uint32_t tmem = sm.tmem_base;
  const int tiles = prefix[p.segs] * p.n_tiles;
  volatile int* abort_flag = &sm.abort_flag;
  struct Tile {
    int row, rows, expert, n;
  };
  auto decode = [&](int t) {
    const int mt = t / p.n_tiles;
    int lo = 0, hi = p.segs;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (prefix[mid] <= mt) lo = mid;
      else hi = mid;
    }
    const int m = mt - prefix[lo], row = row_start[lo] + m * FEW_ROWS;
    return Tile{row, min(FEW_ROWS, row_start[lo + 1] - row), lo % p.experts, t - mt * p.n_tiles};
  };

  if (warp == 0 && lane == 0) {
    // ======================= TMA producer =======================
    Ring r;
    for (int t = (int)blockIdx.x; t < tiles && !*abort_flag; t += gridDim.x) {
      const Tile tl = decode(t);
      const int wrow = tl.expert * p.N + tl.n * BM, wblk = tl.expert * p.w_blocks + tl.n;
      for (int kb = 0; kb < num_kb; ++kb) {
        if (!mbar_wait(&sm.empty[r.i], r.phase ^ 1, 60)) {
          *abort_flag = 1;
          break;
        }
        uint8_t* w = sW + r.i * KEYS * A_BYTES;
        uint8_t* sf = sSF + r.i * KEYS * 1024;
        mbar_arrive_expect_tx(&sm.full[r.i], KEYS * A_BYTES);
        tma_load_2d(w, &tmap_w0, kb * 128, wrow, &sm.full[r.i]);
        if (KEYS == 2) tma_load_2d(w + A_BYTES, &tmap_w1, kb * 128, wrow, &sm.full[r.i]);
        mbar_arrive_expect_tx(&sm.sf_full[r.i], KEYS * 1024);
        tma_load_2d(sf, &tmap_s0, kb * 256, wblk, &sm.sf_full[r.i]);
        if (KEYS == 2) tma_load_2d(sf + 1024, &tmap_s1, kb * 256, wblk, &sm.sf_full[r.i]);
        r.next(p.stages);
      }
    }
  } else if (warp == 1) {
    // ======================= MMA issuer =======================
    const bool issue = elect_one();
    constexpr uint32_t id0 = idesc_mxf4(BM, FEW_ROWS, 0), id2 = idesc_mxf4(BM, FEW_ROWS, 2);
    const uint32_t w_lo0 = desc_lo(smem_u32(sW)), x_lo0 = desc_lo(smem_u32(sX));
    Ring r;
    uint32_t done = 0;
    bool ok = true;
    for (int t = (int)blockIdx.x; t < tiles && ok && !__any_sync(0xffffffffu, *abort_flag); t += gridDim.x, ++done) {
      if (!mbar_wait_warp(&sm.rows_ready, done & 1, 61) ||
          (done > 0 && !mbar_wait_warp(&sm.tempty, (done - 1) & 1, 62)))
        ok = false;
      for (int kb = 0; kb < num_kb && ok; ++kb) {
        if (!mbar_wait_warp(&sm.full[r.i], r.phase, 63)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t w = w_lo0 + r.i * (KEYS * A_BYTES >> 4), x = x_lo0 + kb * (FEW_ROWS * 128 >> 4);
        const uint32_t sf = tmem + FEW_SF_COL + r.i * 32;
        const int steps = min(4, (p.K - kb * BKE + 63) / 64);
        if (issue) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (k >= steps) break;
            const uint32_t id = k & 1 ? id2 : id0;
            umma_mxf4(tmem, w + 2 * k, x + 2 * k, id, sf + 4 * (k >> 1), sf + 16 + 4 * (k >> 1), (kb | k) != 0);
            if (KEYS == 2)
              umma_mxf4(tmem + FEW_ROWS, w + (A_BYTES >> 4) + 2 * k, x + 2 * k, id, sf + 8 + 4 * (k >> 1),
                        sf + 16 + 4 * (k >> 1), (kb | k) != 0);
          }
          umma_commit(&sm.empty[r.i]);
        }
        __syncwarp();
        r.next(p.stages);
      }
      if (ok && issue) umma_commit(&sm.tfull);
      __syncwarp();
    }
    if (!ok && lane == 0) *abort_flag = 1;
    // the last commits have arrived before the CTA frees its barriers and TMEM
    for (int i = 0; i < p.stages; ++i) {
      if (!mbar_wait_warp(&sm.empty[r.i], r.phase ^ 1, 64)) break;
      r.next(p.stages);
    }
  } else if (warp >= 4) {
    // ======================= rows, scales, epilogue =======================
    const int q = warp & 3;
    Ring r;
    uint32_t done = 0;
    for (int t = (int)blockIdx.x; t < tiles && !__any_sync(0xffffffffu, *abort_flag); t += gridDim.x, ++done) {
      const Tile tl = decode(t);
      // the previous tile's MMAs have read the rows
      if (done > 0 && !mbar_wait_warp(&sm.tfull, (done - 1) & 1, 65)) {
        *abort_flag = 1;
        break;
      }
      for (int i = warp - 4; i < tl.rows; i += FEW_QUANT) {
        const __nv_bfloat16* row = p.x + (int64_t)(tl.row + i) * p.K;
        for (int b = 0; b < num_kb * BKE; b += kStep * 4) {
          Raw16<__nv_bfloat16> raw[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int k = b + j * kStep + lane * 16;
            if (k < p.K) load16(row + k, raw[j]);
            else raw[j] = Raw16<__nv_bfloat16>{};
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int k = b + j * kStep + lane * 16;
            if (b + j * kStep >= num_kb * BKE) break;  // warp-uniform
            uint32_t m = amax16(raw[j]);
            m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
            const uint32_t byte = scale_byte(m);
            const float inv = inv_scale(byte == 255u ? 254u : byte);
            uint32_t codes[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float v[8];
              unpack8(raw[j], h, v);
#pragma unroll
              for (int z = 0; z < 8; ++z) v[z] *= inv;
              codes[h] = byte == 255u ? 0u : e2m1x8(v);
            }
            uint32_t w = byte << (8 * ((lane >> 1) & 3));
            w |= __shfl_xor_sync(0xffffffffu, w, 2);
            w |= __shfl_xor_sync(0xffffffffu, w, 4);
            if (k < num_kb * BKE) {  // 8 bytes of a 128-byte row, 16-byte chunks swizzled by the row
              const uint32_t chunk = (uint32_t)((k % BKE) / 32) ^ (uint32_t)(i & 7);
              *reinterpret_cast<uint2*>(sX + (k / BKE) * (FEW_ROWS * 128) + i * 128 + chunk * 16 + (lane & 1) * 8) =
                  make_uint2(codes[0], codes[1]);
              if ((lane & 7) == 0) sXS[(k / 128) * 32 + i] = w;
            }
          }
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.rows_ready);
      if (warp >= 8) continue;
      // every quantising warp's scale words are read here
      if (!mbar_wait_warp(&sm.rows_ready, done & 1, 68)) {
        *abort_flag = 1;
        break;
      }
      const uint32_t quarter = (uint32_t)(q * 32) << 16;
      bool ok = true;
      for (int kb = 0; kb < num_kb; ++kb) {
        if (!mbar_wait_warp(&sm.sf_full[r.i], r.phase, 66)) {
          *abort_flag = 1;
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t src = smem_u32(sSF + r.i * KEYS * 1024) + lane * 16u;
        const uint32_t dst = tmem + FEW_SF_COL + r.i * 32 + quarter;
        const bool pad = kb == num_kb - 1 && p.K % 64;
        const PadMask pm = pad_mask(p.K % BKE / 32);
#pragma unroll
        for (int key = 0; key < KEYS; ++key) {
          uint4 w0 = lds128(src + key * 1024), w1 = lds128(src + key * 1024 + 512);
          if (pad) keep_bytes(w0, pm.keep0), keep_bytes(w1, pm.keep1);
          tmem_st_x8(dst + 8 * key, w0, w1);
        }
        tmem_st_x8(dst + 16, make_uint4(sXS[2 * kb * 32 + lane], 0, 0, 0), make_uint4(sXS[(2 * kb + 1) * 32 + lane], 0, 0, 0));
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.full[r.i]);
        r.next(p.stages);
      }
      if (!ok) break;
      if (!mbar_wait_warp(&sm.tfull, done & 1, 67)) {
        *abort_flag = 1;
        break;
      }
      __syncwarp();
      tc_fence_after();
      uint32_t g[32], up[32];
      tmem_ld_32x32b_x32(tmem + quarter, g);
      if (KEYS == 2) tmem_ld_32x32b_x32(tmem + FEW_ROWS + quarter, up);
      tmem_ld_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.tempty);
      const int ch = tl.n * BM + q * 32 + lane;
      if (ch < p.N) {
        __nv_bfloat16* dst = p.out + (int64_t)tl.row * p.N + ch;
#pragma unroll
        for (int i = 0; i < FEW_ROWS; ++i) {
          if (i >= tl.rows) break;
          const float gv = __uint_as_float(g[i]);
          if (MODE == GATEUP) {
            const float uv = __uint_as_float(up[i]);
            dst[(int64_t)i * p.N] = __float2bfloat16_rn(silu(gv) * uv);
            if (p.gate_up && p.gate_up_f32) {
              float* gu = static_cast<float*>(p.gate_up) + (int64_t)(tl.row + i) * 2 * p.N + ch;
              gu[0] = gv;
              gu[p.N] = uv;
            } else if (p.gate_up) {
              __nv_bfloat16* gu = static_cast<__nv_bfloat16*>(p.gate_up) + (int64_t)(tl.row + i) * 2 * p.N + ch;
              gu[0] = __float2bfloat16_rn(gv);
              gu[p.N] = __float2bfloat16_rn(uv);
            }
          } else {
            dst[(int64_t)i * p.N] = __float2bfloat16_rn(gv);
          }
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, FEW_COLS);
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
static int out_map(CUtensorMap& m, void* out, int64_t rows, int N, int64_t ld, bool f32 = false) {
  if (f32)
    return make_tmap_2d(&m, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, out, (uint64_t)N, (uint64_t)rows, (uint64_t)ld * 4, 16,
                        32, CU_TENSOR_MAP_SWIZZLE_64B);
  return make_tmap_2d(&m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, out, (uint64_t)N, (uint64_t)rows, (uint64_t)ld * 2, 32,
                      32, CU_TENSOR_MAP_SWIZZLE_64B);
}

// CTA pairs of the kernel that are resident at once on the current device (0 = an
// error was set).  Shared memory allows one CTA per SM at every ring size.
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
  cudaFuncAttributes fa;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemLimit);
  if (e == cudaSuccess) e = cudaFuncGetAttributes(&fa, kern);
  if (e != cudaSuccess) {
    set_error(MIRAI_ERR_CUDA, "%s: %s", name, cudaGetErrorString(e));
    return 0;
  }
  if (fa.numRegs < LAUNCH_REGS) {
    set_error(MIRAI_ERR_UNSUPPORTED, "%s compiled with %d registers per thread; the register split needs %d", name,
              fa.numRegs, LAUNCH_REGS);
    return 0;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(THREADS, 1, 1);
  cfg.dynamicSmemBytes = kSmemLimit;
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
                   const void* rank_b, void* out, void* gate_up, int gate_up_dtype, uint8_t* hq, uint8_t* hscale,
                   mirai_stream_t stream) {
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
  if (gate_up_dtype != MIRAI_DTYPE_BF16 && gate_up_dtype != MIRAI_DTYPE_F32)
    return set_error(MIRAI_ERR_INVALID_ARG, "%s: gate/up is saved in bf16 or fp32 (dtype %d)", name, gate_up_dtype);
  const bool save_f32 = gate_up_dtype == MIRAI_DTYPE_F32;
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
  const int64_t tiles = S / TILE_M + (segs < S ? segs : S);  // at most; about S / 256 when segments are long
  if (tiles * p.n_tiles > INT32_MAX || p.n_tiles > 1023)
    return set_error(MIRAI_ERR_UNSUPPORTED, "%s: %lld row tiles x %d column tiles are too many for one call", name,
                     (long long)tiles, p.n_tiles);
  p.w_blocks = (int)ceil_div(N, kBlockRows);
  p.has_ext = rank_a != nullptr;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.gate_up = gate_up;
  p.gate_up_f32 = save_f32;
  p.hq = hq;
  p.hscale = hscale;
  p.h_blocks = max_blocks(S, segs);
  p.h_kt = (int)ceil_div(N, 128);
  CUtensorMap ta, tsa, tb0, tb1, tsb0, tsb1, txa, txb;
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
  CUtensorMap to0 = ta, to1 = ta, to2 = ta;
  if (!rc && out) rc = out_map(to0, out, S, N, N);
  if (!rc && gate_up) {
    rc = out_map(to1, gate_up, S, N, 2 * (int64_t)N, save_f32);
    if (!rc) rc = out_map(to2, static_cast<char*>(gate_up) + (size_t)N * (save_f32 ? 4 : 2), S, N, 2 * (int64_t)N, save_f32);
  }
  if (rc) return rc;
  const int pairs_fit = resident_pairs<MODE>(name);
  if (!pairs_fit) return MIRAI_ERR_CUDA;
  const int limit = gemm_sm_limit();
  int pairs = pairs_fit;
  if (limit > 0 && limit / 2 < pairs) pairs = limit / 2 > 0 ? limit / 2 : 1;
  const int total_kb = (int)ceil_div(K, BKE) + p.has_ext;
  p.resident = total_kb <= A_BUFS;
  // Rings: A whole where it fits, the rest for B.  (More A buffers, to start the next unit's rows
  // early, measured slower than the B stages they take: 125 against 113 us for the layer's down.)
  p.a_bufs = p.resident ? (total_kb < 4 ? 4 : total_kb) : 5;
  p.b_stages = B_STAGES;
  while (smem_bytes(p.a_bufs, p.b_stages, p.segs) > kSmemLimit) --p.b_stages;
  int64_t units = tiles * p.n_tiles;
  if (units > pairs) units = pairs;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(THREADS, 1, 1);
  cfg.gridDim = dim3((unsigned)(2 * units), 1, 1);
  cfg.dynamicSmemBytes = smem_bytes(p.a_bufs, p.b_stages, p.segs);
  cfg.stream = reinterpret_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, product_kernel<MODE>, ta, tsa, tb0, tb1, tsb0, tsb1, txa, txb, to0, to1,
                                           to2, p);
  if (e != cudaSuccess) return set_error(MIRAI_ERR_CUDA, "%s: launch failed: %s", name, cudaGetErrorString(e));
  return check_launch(name);
}

// Few rows in bf16 (see few_rows_kernel).
template <int MODE>
static int few_product(const char* name, const void* x, const int32_t* offsets, int32_t nsrc, int32_t experts, int64_t S,
                       int32_t K, int32_t N, const mirai_mxfp4_weight* w0, const mirai_mxfp4_weight* w1, void* out,
                       void* gate_up, int gate_up_dtype, mirai_stream_t stream) {
  if (nsrc <= 0 || experts <= 0 || (int64_t)nsrc * experts > kMaxSegs)
    return set_error(MIRAI_ERR_INVALID_ARG, "%s: %d sources x %d experts outside 1..%d segments", name, nsrc, experts,
                     kMaxSegs);
  if (S < 0 || K <= 0 || N <= 0)
    return set_error(MIRAI_ERR_INVALID_ARG, "%s: bad sizes (S=%lld, K=%d, N=%d)", name, (long long)S, K, N);
  if (K % 32 || N % 32 || K > FEW_MAX_K || S > MIRAI_MXFP4_FEW_ROWS)
    return set_error(MIRAI_ERR_UNSUPPORTED, "%s: needs K %% 32 == 0 up to %d, N %% 32 == 0 and at most %d rows (S=%lld, "
                     "K=%d, N=%d)", name, FEW_MAX_K, MIRAI_MXFP4_FEW_ROWS, (long long)S, K, N);
  if ((int64_t)experts * N >= (int64_t)1 << 31)
    return set_error(MIRAI_ERR_UNSUPPORTED, "%s: more than 2^31 weight rows", name);
  if (S == 0) return MIRAI_OK;
  if (!x || !offsets || !out || !w0 || !w0->packed || !w0->scale || (w1 && (!w1->packed || !w1->scale)))
    return set_error(MIRAI_ERR_INVALID_ARG, "%s: null operand", name);
  if (gate_up_dtype != MIRAI_DTYPE_BF16 && gate_up_dtype != MIRAI_DTYPE_F32)
    return set_error(MIRAI_ERR_INVALID_ARG, "%s: gate/up is saved in bf16 or fp32 (dtype %d)", name, gate_up_dtype);
  if (misaligned(x, 32)) return set_error(MIRAI_ERR_INVALID_ARG, "%s: rows not 32-byte aligned", name);
  if (misaligned(out, 2) || misaligned(gate_up, gate_up_dtype == MIRAI_DTYPE_F32 ? 4 : 2))
    return set_error(MIRAI_ERR_INVALID_ARG, "%s: output not aligned to its type", name);
  const int kt = (int)ceil_div(K, 128);
  FewParams p = {};
  p.x = static_cast<const __nv_bfloat16*>(x);
  p.offsets = offsets;
  p.segs = nsrc * experts;
  p.experts = experts;
  p.S = S;
  p.K = K;
  p.N = N;
  p.n_tiles = (int)ceil_div(N, BM);
  p.w_blocks = p.n_tiles;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.gate_up = gate_up;
  p.gate_up_f32 = gate_up_dtype == MIRAI_DTYPE_F32;
  p.stages = FEW_STAGES;
  while (few_smem_bytes<MODE>(p.stages, K, p.segs) > kSmemLimit) --p.stages;
  CUtensorMap t0, t1, s0, s1;
  int rc = code_map(t0, w0->packed, (int64_t)experts * N, K);
  if (!rc) rc = scale_map(s0, w0->scale, (int64_t)experts * p.w_blocks, kt);
  if (!rc) rc = w1 ? code_map(t1, w1->packed, (int64_t)experts * N, K) : (t1 = t0, MIRAI_OK);
  if (!rc) rc = w1 ? scale_map(s1, w1->scale, (int64_t)experts * p.w_blocks, kt) : (s1 = s0, MIRAI_OK);
  if (rc) return rc;
  static std::atomic<bool> ready[kMaxDevices];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices)
    return set_error(MIRAI_ERR_CUDA, "%s: no current device", name);
  if (!ready[dev].load(std::memory_order_acquire)) {
    const cudaError_t e =
        cudaFuncSetAttribute(few_rows_kernel<MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemLimit);
    if (e != cudaSuccess) return set_error(MIRAI_ERR_CUDA, "%s: %s", name, cudaGetErrorString(e));
    ready[dev].store(true, std::memory_order_release);
  }
  const int limit = gemm_sm_limit();
  int64_t grid = (S / FEW_ROWS + (p.segs < S ? p.segs : S)) * p.n_tiles;
  const int sms = (limit > 0 && limit < sm_count()) ? limit : sm_count();
  if (grid > sms) grid = sms;
  few_rows_kernel<MODE><<<(unsigned)grid, FEW_THREADS, few_smem_bytes<MODE>(p.stages, K, p.segs),
                          reinterpret_cast<cudaStream_t>(stream)>>>(t0, t1, s0, s1, p);
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
  if (!weight || !packed || !scale || mx::misaligned(weight, 32) || mx::misaligned(packed) || mx::misaligned(scale))
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
  if (!out || !packed || !scale || mx::misaligned(out, 32) || mx::misaligned(packed) || mx::misaligned(scale))
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
  if (!x || !offsets || !packed || !scale || mx::misaligned(x, 32) || mx::misaligned(packed) || mx::misaligned(scale))
    return set_error(MIRAI_ERR_INVALID_ARG, "mxfp4_quantize_rows: null or misaligned pointer");
  const int64_t grid = mx::strips("mxfp4_quantize_rows", mx::max_blocks(num_rows, num_segments));
  if (grid < 0) return MIRAI_ERR_UNSUPPORTED;
  mx::quantize_kernel<__nv_bfloat16, true><<<(unsigned)grid, 256, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
      static_cast<const __nv_bfloat16*>(x), x_rows, row_index, offsets, num_segments, num_rows, width,
      (int)mx::ceil_div(width, 128), packed, scale);
  return check_launch("mxfp4_quantize_rows");
}

int mirai_moe_gateup_swiglu_mxfp4_save(const uint8_t* x_packed, const uint8_t* x_scale, const int32_t* offsets,
                                       int32_t num_sources, int32_t num_experts, int64_t num_rows, int32_t hidden,
                                       int32_t inter, const mirai_mxfp4_weight* w1, const mirai_mxfp4_weight* w3,
                                       void* h, void* gate_up, int32_t gate_up_dtype, uint8_t* h_packed,
                                       uint8_t* h_scale, mirai_stream_t stream) {
  if (!w3) return set_error(MIRAI_ERR_INVALID_ARG, "gateup_swiglu_mxfp4: null operand");
  return mx::product<mx::GATEUP>("gateup_swiglu_mxfp4", {x_packed, x_scale}, offsets, num_sources, num_experts, num_rows,
                                 hidden, inter, w1, w3, nullptr, nullptr, h, gate_up, gate_up_dtype, h_packed, h_scale,
                                 stream);
}

int mirai_moe_gateup_swiglu_mxfp4(const uint8_t* x_packed, const uint8_t* x_scale, const int32_t* offsets,
                                  int32_t num_sources, int32_t num_experts, int64_t num_rows, int32_t hidden,
                                  int32_t inter, const mirai_mxfp4_weight* w1, const mirai_mxfp4_weight* w3, void* h,
                                  void* gate_up, uint8_t* h_packed, uint8_t* h_scale, mirai_stream_t stream) {
  return mirai_moe_gateup_swiglu_mxfp4_save(x_packed, x_scale, offsets, num_sources, num_experts, num_rows, hidden, inter,
                                            w1, w3, h, gate_up, MIRAI_DTYPE_BF16, h_packed, h_scale, stream);
}

int mirai_moe_gateup_swiglu_mxfp4_few_save(const void* x, const int32_t* offsets, int32_t num_sources,
                                           int32_t num_experts, int64_t num_rows, int32_t hidden, int32_t inter,
                                           const mirai_mxfp4_weight* w1, const mirai_mxfp4_weight* w3, void* h,
                                           void* gate_up, int32_t gate_up_dtype, mirai_stream_t stream) {
  if (!w3) return set_error(MIRAI_ERR_INVALID_ARG, "gateup_swiglu_mxfp4_few: null operand");
  return mx::few_product<mx::GATEUP>("gateup_swiglu_mxfp4_few", x, offsets, num_sources, num_experts, num_rows, hidden,
                                     inter, w1, w3, h, gate_up, gate_up_dtype, stream);
}

int mirai_moe_gateup_swiglu_mxfp4_few(const void* x, const int32_t* offsets, int32_t num_sources, int32_t num_experts,
                                      int64_t num_rows, int32_t hidden, int32_t inter, const mirai_mxfp4_weight* w1,
                                      const mirai_mxfp4_weight* w3, void* h, void* gate_up, mirai_stream_t stream) {
  return mirai_moe_gateup_swiglu_mxfp4_few_save(x, offsets, num_sources, num_experts, num_rows, hidden, inter, w1, w3, h,
                                                gate_up, MIRAI_DTYPE_BF16, stream);
}

int mirai_moe_down_mxfp4_few(const void* h, const int32_t* offsets, int32_t num_sources, int32_t num_experts,
                             int64_t num_rows, int32_t inter, int32_t hidden, const mirai_mxfp4_weight* w2, void* y,
                             mirai_stream_t stream) {
  return mx::few_product<mx::DOWN>("down_mxfp4_few", h, offsets, num_sources, num_experts, num_rows, inter, hidden, w2,
                                   nullptr, y, nullptr, MIRAI_DTYPE_BF16, stream);
}

int mirai_moe_down_mxfp4(const uint8_t* h_packed, const uint8_t* h_scale, const int32_t* offsets, int32_t num_sources,
                         int32_t num_experts, int64_t num_rows, int32_t inter, int32_t hidden,
                         const mirai_mxfp4_weight* w2, const void* rank_a, const void* rank_b, void* y,
                         mirai_stream_t stream) {
  return mx::product<mx::DOWN>("down_mxfp4", {h_packed, h_scale}, offsets, num_sources, num_experts, num_rows, inter,
                               hidden, w2, nullptr, rank_a, rank_b, y, nullptr, MIRAI_DTYPE_BF16, nullptr, nullptr,
                               stream);
}

}  // extern "C"
