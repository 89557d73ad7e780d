// ff_mxfp4.cuh — microscaled 4-bit floating point (MXFP4): quantiser, its SwiGLU variants and the
// way back.
//
// Format (the OCP microscaling specification): 32 consecutive values along the axis that a product
// sums over share one power-of-two scale s = 2^(S - 127), held as the byte S (E8M0); each value is
// an E2M1 code (sign, 2 exponent bits, 1 fraction bit: 0, .5, 1, 1.5, 2, 3, 4, 6), two to a byte,
// the earlier value in the low nibble.  With A = max |x| of the block,
//     s = 2^max(floor(log2 A) - 2, -127),   code = RNE(clamp(x / s, -6, 6)).
// floor(log2 A) is A's exponent field - 127, so S = max(field - 2, 0) and x / s is the product with
// the power of two whose exponent field is 254 - S: exact, no division.  The conversion instruction
// rounds to the nearest code (ties to even) and saturates.  A block that holds an infinity or a NaN
// gets the scale NaN (S = 255) and codes 0, so every value it stands for is NaN.
//
// Layout: codes [rows, ld bytes] with the blocks of a row in order (16 bytes each); scales in
// chunks of 512 bytes that cover 128 rows x 4 blocks, the order in which the tensor core takes
// them: byte (row % 32) * 16 + (row / 32 % 4) * 4 + block % 4 of chunk
// (row / 128) * chunks + block / 4, chunks = 2 * ceil(cols / 256).  Chunks of the padding hold
// S = 0 (a finite scale for the zero codes that a tile load fills in).
#pragma once

#include "ff_common.cuh"

namespace ff {
namespace mx {

constexpr int BLOCK = 32;
constexpr int TILE = 128;      // rows and columns of a CTA's tile: one scale chunk in either orientation
constexpr int THREADS = 256;
constexpr uint32_t kScaleNan = 255u;

__host__ __device__ __forceinline__ int64_t chunks_of(int64_t cols) { return 2 * ((cols + 255) / 256); }
__host__ __device__ __forceinline__ int64_t scale_bytes(int64_t rows, int64_t cols) {
  return ((rows + 127) / 128) * chunks_of(cols) * 512;
}
// byte offset of the scale of (row, block)
__device__ __forceinline__ int64_t scale_at(int64_t row, int64_t blk, int64_t chunks) {
  return ((row >> 7) * chunks + (blk >> 2)) * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4 + (blk & 3);
}

// S of a block from the bits of its largest |x| (fp32)
__device__ __forceinline__ uint32_t scale_code(uint32_t amax_bits) {
  const uint32_t field = amax_bits >> 23;
  return field == 255u ? kScaleNan : (field > 2u ? field - 2u : 0u);
}
// 1 / s as a float (0 for a NaN scale: the codes become 0)
__device__ __forceinline__ float inv_scale(uint32_t S) { return S == kScaleNan ? 0.f : __uint_as_float((254u - S) << 23); }
__device__ __forceinline__ float scale_value(uint32_t S) {
  return S == kScaleNan ? __uint_as_float(0x7FC00000u) : (S == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(S << 23));
}

// eight values (already divided by the scale) -> one word of codes, v[0] in the lowest nibble
__device__ __forceinline__ uint32_t codes8(const float (&v)[8]) {
  uint32_t w;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(w)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return w;
}
// one byte of codes -> two values
__device__ __forceinline__ float2 values2(uint32_t byte) {
  uint32_t h;
  asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, a;\n\t}" : "=r"(h) : "r"(byte));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// element types of the staged tile
template <int DT>
struct Pair;  // two neighbouring 16-bit values in one word
template <>
struct Pair<FF_DTYPE_BF16> {
  static __device__ __forceinline__ float lo(uint32_t w) { return __uint_as_float(w << 16); }
  static __device__ __forceinline__ float hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }
  static __device__ __forceinline__ uint32_t f32_bits(uint32_t h) { return h << 16; }
};
template <>
struct Pair<FF_DTYPE_F16> {
  static __device__ __forceinline__ float lo(uint32_t w) { return __half2float(__ushort_as_half((unsigned short)(w & 0xFFFFu))); }
  static __device__ __forceinline__ float hi(uint32_t w) { return __half2float(__ushort_as_half((unsigned short)(w >> 16))); }
  static __device__ __forceinline__ uint32_t f32_bits(uint32_t h) {
    return __float_as_uint(__half2float(__ushort_as_half((unsigned short)h)));
  }
};

// Where a tile's codes and scales go.  Column c of the staged tile is column col0 + c of the
// quantised matrix; `live_cols` of its columns exist (a multiple of BLOCK unless the matrix ends).
struct Out {
  uint8_t* q_rows;   // [rows, ldq], or null
  uint8_t* s_rows;
  int64_t ldq, chunks_r;
  uint8_t* q_cols;   // transposed: [cols, ldqt], or null
  uint8_t* s_cols;
  int64_t ldqt, chunks_c;
  float* colsum;     // [row tiles, cols] partial column sums, or null
  int64_t rows, cols;
};

// bytes of a staged row: 128 values and 16 bytes, so that eight rows start in distinct bank groups
template <int DT>
__host__ __device__ constexpr int row_bytes() {
  return TILE * (DT == FF_DTYPE_F32 ? 4 : 2) + 16;
}

// Row codes of a staged tile: thread item = one row's block of 32.  Four lanes take the blocks of
// one row, so a row's 64 code bytes leave together; the lanes of blocks 2 and 3 read their 16-byte
// pieces in another order, which keeps the eight lanes of a shared-memory phase on distinct banks.
// Blocks below `nblk` have their codes stored, blocks below `sblk` their scales.
template <int DT>
__device__ __forceinline__ void quant_rows(const uint8_t* tile, int64_t row0, int64_t col0, int64_t nblk, int64_t sblk,
                                           const Out& o) {
  const int lane = threadIdx.x & 31;
  const int64_t blk0 = col0 / BLOCK;
  const bool words = (blk0 & 3) == 0 && blk0 + 4 <= sblk;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int item = threadIdx.x + i * THREADS;
    const int r = item >> 2, b = item & 3;
    const int64_t row = row0 + r, blk = blk0 + b;
    const uint8_t* src = tile + r * row_bytes<DT>();
    uint32_t w[4];
    uint32_t S;
    if constexpr (DT == FF_DTYPE_F32) {
      float v[32];
      uint32_t amax = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float4 f = *reinterpret_cast<const float4*>(src + b * 128 + j * 16);
        v[4 * j] = f.x; v[4 * j + 1] = f.y; v[4 * j + 2] = f.z; v[4 * j + 3] = f.w;
      }
#pragma unroll
      for (int j = 0; j < 32; ++j) amax = max(amax, __float_as_uint(v[j]) & 0x7FFFFFFFu);
      S = scale_code(amax);
      const float inv = inv_scale(S);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float t[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] = S == kScaleNan ? 0.f : v[8 * k + e] * inv;
        w[k] = codes8(t);
      }
    } else {
      const int swap = b & 2;
      uint4 p[4];
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        p[j] = *reinterpret_cast<const uint4*>(src + b * 64 + ((j ^ swap) * 16));
        m = __vmaxu2(m, __vmaxu2(__vmaxu2(p[j].x & 0x7FFF7FFFu, p[j].y & 0x7FFF7FFFu),
                                 __vmaxu2(p[j].z & 0x7FFF7FFFu, p[j].w & 0x7FFF7FFFu)));
      }
      S = scale_code(Pair<DT>::f32_bits(max(m & 0xFFFFu, m >> 16)));
      const float inv = inv_scale(S);
      uint32_t c[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t q[4] = {p[j].x, p[j].y, p[j].z, p[j].w};
        float t[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          t[2 * e] = Pair<DT>::lo(q[e]) * inv;
          t[2 * e + 1] = Pair<DT>::hi(q[e]) * inv;
        }
        c[j] = S == kScaleNan ? 0u : codes8(t);
      }
      w[0] = swap ? c[2] : c[0];
      w[1] = swap ? c[3] : c[1];
      w[2] = swap ? c[0] : c[2];
      w[3] = swap ? c[1] : c[3];
    }
    if (row < o.rows && blk < nblk)
      *reinterpret_cast<uint4*>(o.q_rows + row * o.ldq + blk * 16) = make_uint4(w[0], w[1], w[2], w[3]);
    // scales: the four lanes of a row hold one word of a chunk when the tile starts on a chunk
    if (words) {
      const uint32_t s1 = __shfl_down_sync(0xffffffffu, S, 1);
      const uint32_t s2 = __shfl_down_sync(0xffffffffu, S, 2);
      const uint32_t s3 = __shfl_down_sync(0xffffffffu, S, 3);
      if ((lane & 3) == 0 && row0 < o.rows)
        *reinterpret_cast<uint32_t*>(o.s_rows + scale_at(row, blk, o.chunks_r)) = S | (s1 << 8) | (s2 << 16) | (s3 << 24);
    } else if (row0 < o.rows && blk < sblk) {
      o.s_rows[scale_at(row, blk, o.chunks_r)] = (uint8_t)S;
    }
  }
}

// Column codes (transposed): thread item = 32 rows of one column pair (16-bit tiles) or of one
// column (fp32).  The lanes read neighbouring words of each row: no bank conflict.  The scales are
// gathered in shared memory (four row blocks of a column make one word of a chunk); columns below
// `scol` have theirs stored, the tile's first `live` columns their codes.  With `colsum`
// the sums of the 128 rows of each column go out too (fp32, the blocks added in row order).
template <int DT>
__device__ __forceinline__ void quant_cols(const uint8_t* tile, int64_t row0, int64_t col0, int live, int64_t scol,
                                           const Out& o, uint8_t* s_buf /* 128 x 4 */, float* sum_buf /* 4 x 128 */) {
  constexpr int W = DT == FF_DTYPE_F32 ? 1 : 2;   // columns of an item
  constexpr int ITEMS = 4 * TILE / W / THREADS;
#pragma unroll 1
  for (int i = 0; i < ITEMS; ++i) {
    const int item = threadIdx.x + i * THREADS;
    const int wc = item % (TILE / W), rb = item / (TILE / W);
    const uint8_t* src = tile + (rb * BLOCK) * row_bytes<DT>() + wc * 4;
    uint32_t x[32];
#pragma unroll
    for (int j = 0; j < 32; ++j) x[j] = *reinterpret_cast<const uint32_t*>(src + j * row_bytes<DT>());
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      if constexpr (DT == FF_DTYPE_F32) m = max(m, x[j] & 0x7FFFFFFFu);
      else m = __vmaxu2(m, x[j] & 0x7FFF7FFFu);
    }
#pragma unroll
    for (int h = 0; h < W; ++h) {
      uint32_t bits;
      if constexpr (DT == FF_DTYPE_F32) bits = m;
      else bits = Pair<DT>::f32_bits(h ? m >> 16 : m & 0xFFFFu);
      const uint32_t S = scale_code(bits);
      const float inv = inv_scale(S);
      uint32_t w[4];
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float t[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float v;
          if constexpr (DT == FF_DTYPE_F32) v = __uint_as_float(x[8 * k + e]);
          else v = h ? Pair<DT>::hi(x[8 * k + e]) : Pair<DT>::lo(x[8 * k + e]);
          sum += v;
          t[e] = v * inv;
        }
        w[k] = S == kScaleNan ? 0u : codes8(t);
      }
      const int c = wc * W + h;
      // 16 bytes per 32 rows; row blocks past the matrix are not stored (ldqt covers whole blocks)
      if (c < live && row0 + rb * BLOCK < o.rows)
        *reinterpret_cast<uint4*>(o.q_cols + (col0 + c) * o.ldqt + (row0 / 2 + rb * 16)) =
            make_uint4(w[0], w[1], w[2], w[3]);
      s_buf[c * 4 + rb] = (uint8_t)S;
      if (o.colsum) sum_buf[rb * TILE + c] = sum;
    }
  }
  __syncthreads();
  const int c = threadIdx.x;
  if (c < TILE) {
    const int64_t col = col0 + c;
    // columns past the matrix still own scale bytes of its last chunk row (0: their values are 0)
    if (col < scol)
      *reinterpret_cast<uint32_t*>(o.s_cols + scale_at(col, row0 / BLOCK, o.chunks_c)) =
          *reinterpret_cast<const uint32_t*>(s_buf + c * 4);
    if (o.colsum && c < live && row0 < o.rows)
      o.colsum[(row0 / TILE) * o.cols + col] =
          ((sum_buf[c] + sum_buf[TILE + c]) + sum_buf[2 * TILE + c]) + sum_buf[3 * TILE + c];
  }
}

// Stage rows row0.. x columns col0.. of a row-major matrix (zeros outside it).  16-byte loads where
// base and leading dimension allow, all of a thread's loads in flight before the first store.
template <int DT>
__device__ __forceinline__ void stage_tile(uint8_t* tile, const void* x, int64_t ld, int64_t rows, int64_t cols,
                                           int64_t row0, int64_t col0, bool vec) {
  using T = typename Elem<DT>::T;
  constexpr int V = 16 / (int)sizeof(T);
  constexpr int PER_ROW = TILE / V;
  constexpr int N = TILE * PER_ROW / THREADS;
  const T* p = reinterpret_cast<const T*>(x);
  uint4 v[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int k = threadIdx.x + i * THREADS;
    const int64_t r = row0 + k / PER_ROW, c = col0 + (k % PER_ROW) * V;
    v[i] = make_uint4(0, 0, 0, 0);
    if (r < rows && c < cols) {
      if (vec && c + V <= cols) {
        v[i] = __ldg(reinterpret_cast<const uint4*>(p + r * ld + c));
      } else {
        T* e = reinterpret_cast<T*>(&v[i]);
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (c + j < cols) e[j] = p[r * ld + c + j];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int k = threadIdx.x + i * THREADS;
    *reinterpret_cast<uint4*>(tile + (k / PER_ROW) * row_bytes<DT>() + (k % PER_ROW) * 16) = v[i];
  }
}

// both orientations of a tile of the matrix o.rows x o.cols
template <int DT>
__device__ __forceinline__ void quant_tile(const uint8_t* tile, int64_t row0, int64_t col0, const Out& o, uint8_t* s_buf,
                                           float* sum_buf) {
  if (o.q_rows) quant_rows<DT>(tile, row0, col0, (o.cols + BLOCK - 1) / BLOCK, o.chunks_r * 4, o);
  if (o.q_cols)
    quant_cols<DT>(tile, row0, col0, (int)min64(TILE, max64(0, o.cols - col0)), (o.cols + 127) & ~(int64_t)127, o, s_buf,
                   sum_buf);
}

template <int DT>
__host__ __device__ constexpr int quant_smem() {
  return TILE * row_bytes<DT>() + TILE * 4 + 4 * TILE * 4;
}

// One 128 x 128 tile per CTA: read once, quantised along either axis or both from shared memory.
// Bound by HBM: 2 bytes read and 17/32 byte written per value and orientation.
template <int DT>
__global__ void __launch_bounds__(THREADS) mx_quant_kernel(const void* x, int64_t ldx, int64_t tiles_c, Out o, int vec) {
  extern __shared__ __align__(16) uint8_t smem[];
  uint8_t* s_buf = smem + TILE * row_bytes<DT>();
  float* sum_buf = reinterpret_cast<float*>(s_buf + TILE * 4);
  const int64_t row0 = (blockIdx.x / tiles_c) * TILE, col0 = (blockIdx.x % tiles_c) * TILE;
  stage_tile<DT>(smem, x, ldx, o.rows, o.cols, row0, col0, vec != 0);
  __syncthreads();
  quant_tile<DT>(smem, row0, col0, o, s_buf, sum_buf);
}

// silu and its derivative's parts in fp32: sigmoid from the exponential, exact at both ends
// (exp(-g) = inf gives 0, and 0 gives 1)
__device__ __forceinline__ float sigmoid_f32(float g) { return __fdividef(1.f, 1.f + __expf(-g)); }

// h = bf16(silu(g) * u) of the bf16 gate/up activations gu = [g | u], quantised like mx_quant_kernel;
// h itself is not written.
__global__ void __launch_bounds__(THREADS) mx_swiglu_quant_kernel(const __nv_bfloat16* gu, int64_t ld, int64_t F,
                                                                  int64_t tiles_c, Out o) {
  extern __shared__ __align__(16) uint8_t smem[];
  constexpr int DT = FF_DTYPE_BF16;
  uint8_t* s_buf = smem + TILE * row_bytes<DT>();
  float* sum_buf = reinterpret_cast<float*>(s_buf + TILE * 4);
  const int64_t row0 = (blockIdx.x / tiles_c) * TILE, col0 = (blockIdx.x % tiles_c) * TILE;
  constexpr int N = TILE * 16 / THREADS;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int k = threadIdx.x + i * THREADS;
    const int64_t r = row0 + k / 16, c = col0 + (k % 16) * 8;
    uint4 w = make_uint4(0, 0, 0, 0);
    if (r < o.rows && c < F) {  // F is a multiple of 32: whole pieces
      float g[8], u[8];
      load8<DT>(gu + r * ld + c, g);
      load8<DT>(gu + r * ld + F + c, u);
      uint32_t q[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float a = g[2 * e] * sigmoid_f32(g[2 * e]) * u[2 * e];
        const float b = g[2 * e + 1] * sigmoid_f32(g[2 * e + 1]) * u[2 * e + 1];
        q[e] = pack_bf16x2(mk2(a, b));
      }
      w = make_uint4(q[0], q[1], q[2], q[3]);
    }
    *reinterpret_cast<uint4*>(smem + (k / 16) * row_bytes<DT>() + (k % 16) * 16) = w;
  }
  __syncthreads();
  quant_tile<DT>(smem, row0, col0, o, s_buf, sum_buf);
}

// The gradient of gu from dh and gu (all bf16), quantised as the matrix [dg | du] of 2F columns
// without being written:  dg = bf16(dh * u * sig(g) * (1 + g * (1 - sig(g)))),  du = bf16(dh * g * sig(g)).
// One CTA takes the same 128 features of dg and of du.
__global__ void __launch_bounds__(THREADS) mx_swiglu_bwd_quant_kernel(const __nv_bfloat16* dh, int64_t lddh,
                                                                      const __nv_bfloat16* gu, int64_t ld, int64_t F,
                                                                      int64_t tiles_c, Out o) {
  extern __shared__ __align__(16) uint8_t smem[];
  constexpr int DT = FF_DTYPE_BF16;
  constexpr int TB = TILE * row_bytes<DT>();
  uint8_t* s_buf = smem + 2 * TB;
  const int64_t row0 = (blockIdx.x / tiles_c) * TILE, col0 = (blockIdx.x % tiles_c) * TILE;
  constexpr int N = TILE * 16 / THREADS;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int k = threadIdx.x + i * THREADS;
    const int64_t r = row0 + k / 16, c = col0 + (k % 16) * 8;
    uint4 wg = make_uint4(0, 0, 0, 0), wu = wg;
    if (r < o.rows && c < F) {
      float g[8], u[8], d[8], dg[8], du[8];
      load8<DT>(gu + r * ld + c, g);
      load8<DT>(gu + r * ld + F + c, u);
      load8<DT>(dh + r * lddh + c, d);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float s = sigmoid_f32(g[e]);
        dg[e] = d[e] * u[e] * (s * (1.f + g[e] * (1.f - s)));
        du[e] = d[e] * (g[e] * s);
      }
      wg = make_uint4(pack_bf16x2(mk2(dg[0], dg[1])), pack_bf16x2(mk2(dg[2], dg[3])), pack_bf16x2(mk2(dg[4], dg[5])),
                      pack_bf16x2(mk2(dg[6], dg[7])));
      wu = make_uint4(pack_bf16x2(mk2(du[0], du[1])), pack_bf16x2(mk2(du[2], du[3])), pack_bf16x2(mk2(du[4], du[5])),
                      pack_bf16x2(mk2(du[6], du[7])));
    }
    const int at = (k / 16) * row_bytes<DT>() + (k % 16) * 16;
    *reinterpret_cast<uint4*>(smem + at) = wg;
    *reinterpret_cast<uint4*>(smem + TB + at) = wu;
  }
  __syncthreads();
  const int live = (int)min64(TILE, F - col0);
#pragma unroll 1
  for (int half = 0; half < 2; ++half) {
    const uint8_t* tile = smem + half * TB;
    // this half's blocks end at column half * F + F: what follows is the other half's (or padding)
    const int64_t c0 = half * F + col0, end = c0 + live;
    if (o.q_rows) quant_rows<DT>(tile, row0, c0, end / BLOCK, end / BLOCK, o);
    if (o.q_cols) {
      quant_cols<DT>(tile, row0, c0, live, end == o.cols ? (end + 127) & ~(int64_t)127 : end, o, s_buf, nullptr);
      __syncthreads();
    }
  }
  // the padding chunks of the row scales
  if (o.q_rows && col0 + TILE >= F && row0 < o.rows) {
    const int64_t first = 2 * F / BLOCK, last = o.chunks_r * 4;
    const int64_t n = (last - first) * TILE;
    for (int64_t i = threadIdx.x; i < n; i += THREADS) o.s_rows[scale_at(row0 + i % TILE, first + i / TILE, o.chunks_r)] = 0;
  }
}

// Stage 2 of the column sums: the row tiles of a column added in order, one thread per column and
// segment of row tiles, then the segments in order (deterministic).
__global__ void __launch_bounds__(256) mx_colsum_kernel(const float* part, int64_t tiles, int64_t cols, float* out) {
  __shared__ float seg[8][32];
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;
  const int64_t b = tiles * w / 8, e = tiles * (w + 1) / 8;
  float s = 0.f;
  if (c < cols)
    for (int64_t t = b; t < e; ++t) s += part[t * cols + c];
  seg[w][lane] = s;
  __syncthreads();
  if (w == 0 && c < cols) {
    float t = seg[0][lane];
    for (int k = 1; k < 8; ++k) t += seg[k][lane];
    out[c] = t;
  }
}

// eight values per thread: one word of codes -> 16 (or 32) bytes
template <int DT>
__global__ void __launch_bounds__(256) mx_dequant_kernel(const uint8_t* q, int64_t ldq, const uint8_t* s, int64_t chunks,
                                                         int64_t rows, int64_t cols, void* out, int64_t ldo, int vec) {
  using T = typename Elem<DT>::T;
  const int64_t per_row = (cols + 7) / 8;
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= rows * per_row) return;
  const int64_t r = i / per_row, c = (i - r * per_row) * 8;
  const uint32_t w = *reinterpret_cast<const uint32_t*>(q + r * ldq + c / 2);
  const float sv = scale_value(s[scale_at(r, c / BLOCK, chunks)]);
  float v[8];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 p = values2((w >> (8 * k)) & 0xFFu);
    v[2 * k] = p.x * sv;
    v[2 * k + 1] = p.y * sv;
  }
  T t[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    if constexpr (DT == FF_DTYPE_F32) t[k] = v[k];
    else if constexpr (DT == FF_DTYPE_BF16) t[k] = __float2bfloat16_rn(v[k]);
    else t[k] = __float2half_rn(v[k]);
  }
  T* o = reinterpret_cast<T*>(out) + r * ldo + c;
  if (vec && c + 8 <= cols) {
#pragma unroll
    for (int k = 0; k < (int)(8 * sizeof(T) / 16); ++k)
      reinterpret_cast<uint4*>(o)[k] = reinterpret_cast<const uint4*>(t)[k];
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (c + k < cols) o[k] = t[k];
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
// checks of a quantiser's outputs for a matrix rows x cols, and the kernel's view of them
inline int make_out(const char* name, int64_t rows, int64_t cols, uint8_t* q_rows, int64_t ldq, uint8_t* s_rows,
                    uint8_t* q_cols, int64_t ldqt, uint8_t* s_cols, Out* o) {
  FF_REQUIRE(rows >= 0 && cols >= 1, FF_ERR_INVALID_ARG, "%s: rows=%lld cols=%lld", name, (long long)rows, (long long)cols);
  FF_REQUIRE(rows < ((int64_t)1 << 31) && cols < ((int64_t)1 << 31), FF_ERR_UNSUPPORTED, "%s: rows=%lld cols=%lld too large",
             name, (long long)rows, (long long)cols);
  FF_REQUIRE((q_rows == nullptr) == (s_rows == nullptr) && (q_cols == nullptr) == (s_cols == nullptr), FF_ERR_INVALID_ARG,
             "%s: codes and scales of an orientation come together", name);
  if (q_rows)
    FF_REQUIRE(ldq % 16 == 0 && ldq >= (cols + 31) / 32 * 16 && aligned(q_rows, 16) && aligned(s_rows, 16), FF_ERR_INVALID_ARG,
               "%s: ldq=%lld (a multiple of 16 bytes that holds every block; 16-byte aligned outputs)", name, (long long)ldq);
  if (q_cols)
    FF_REQUIRE(ldqt % 16 == 0 && ldqt >= (rows + 31) / 32 * 16 && aligned(q_cols, 16) && aligned(s_cols, 16), FF_ERR_INVALID_ARG,
               "%s: ldqt=%lld (a multiple of 16 bytes that holds every block; 16-byte aligned outputs)", name, (long long)ldqt);
  *o = Out{q_rows, s_rows, ldq, chunks_of(cols), q_cols, s_cols, ldqt, chunks_of(rows), nullptr, rows, cols};
  return FF_OK;
}

template <typename K>
inline int allow_smem(K kernel, int bytes, bool* done, const char* name) {
  int dev = 0;
  FF_CUDA_TRY(cudaGetDevice(&dev), name);
  if (dev < 64 && done[dev]) return FF_OK;
  FF_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes), name);
  if (dev < 64) done[dev] = true;
  return FF_OK;
}

template <int DT>
inline int launch_quant(const void* x, int64_t ldx, int64_t tiles_r, int64_t tiles_c, const Out& o, cudaStream_t st) {
  static bool done[64] = {false};
  int rc = allow_smem(mx_quant_kernel<DT>, quant_smem<DT>(), done, "ff_mxfp4_quant");
  if (rc) return rc;
  const int vec = aligned(x, 16) && (ldx * dtype_size(DT)) % 16 == 0;
  mx_quant_kernel<DT><<<(unsigned)(tiles_r * tiles_c), THREADS, quant_smem<DT>(), st>>>(x, ldx, tiles_c, o, vec);
  return check_launch("ff_mxfp4_quant");
}

// tiles of the grid: the padding chunks of the scales belong to it
inline int grid_of(const char* name, const Out& o, int64_t cols, int64_t* tr, int64_t* tc) {
  *tc = o.q_rows ? chunks_of(cols) : (cols + 127) / 128;
  *tr = o.q_cols ? chunks_of(o.rows) : (o.rows + 127) / 128;
  FF_REQUIRE(*tr * *tc < ((int64_t)1 << 31), FF_ERR_UNSUPPORTED, "%s: too many tiles", name);
  return FF_OK;
}

}  // namespace mx
}  // namespace ff

extern "C" int64_t ff_mxfp4_scale_bytes(int64_t rows, int64_t cols) {
  return rows < 0 || cols < 1 ? 0 : ff::mx::scale_bytes(rows, cols);
}

extern "C" int64_t ff_mxfp4_colsum_ws_elems(int64_t rows, int64_t cols) {
  return rows < 1 || cols < 1 ? 0 : (rows + 127) / 128 * cols;
}

extern "C" int ff_mxfp4_quant(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ldx, uint8_t* q_rows,
                              int64_t ldq, uint8_t* s_rows, uint8_t* q_cols_t, int64_t ldqt, uint8_t* s_cols, float* colsum,
                              float* colsum_ws, void* stream) {
  using namespace ff::mx;
  Out o;
  int rc = make_out("ff_mxfp4_quant", rows, cols, q_rows, ldq, s_rows, q_cols_t, ldqt, s_cols, &o);
  if (rc) return rc;
  FF_REQUIRE(dtype >= FF_DTYPE_F32 && dtype <= FF_DTYPE_F16, FF_ERR_INVALID_ARG, "ff_mxfp4_quant: bad dtype %d", dtype);
  FF_REQUIRE(ldx >= cols, FF_ERR_INVALID_ARG, "ff_mxfp4_quant: ldx=%lld < cols=%lld", (long long)ldx, (long long)cols);
  FF_REQUIRE(!colsum || (q_cols_t && colsum_ws), FF_ERR_INVALID_ARG,
             "ff_mxfp4_quant: column sums come with the column codes and need a workspace");
  cudaStream_t st = ff::as_stream(stream);
  if (rows == 0) {
    if (colsum) FF_CUDA_TRY(cudaMemsetAsync(colsum, 0, (size_t)cols * 4, st), "ff_mxfp4_quant");
    return FF_OK;
  }
  if (!q_rows && !q_cols_t) return FF_OK;
  FF_REQUIRE(x, FF_ERR_INVALID_ARG, "ff_mxfp4_quant: null pointer");
  o.colsum = colsum ? colsum_ws : nullptr;
  int64_t tr, tc;
  rc = grid_of("ff_mxfp4_quant", o, cols, &tr, &tc);
  if (rc) return rc;
  rc = dtype == FF_DTYPE_F32    ? launch_quant<FF_DTYPE_F32>(x, ldx, tr, tc, o, st)
       : dtype == FF_DTYPE_BF16 ? launch_quant<FF_DTYPE_BF16>(x, ldx, tr, tc, o, st)
                                : launch_quant<FF_DTYPE_F16>(x, ldx, tr, tc, o, st);
  if (rc || !colsum) return rc;
  mx_colsum_kernel<<<(unsigned)((cols + 31) / 32), 256, 0, st>>>(colsum_ws, (rows + 127) / 128, cols, colsum);
  return ff::check_launch("ff_mxfp4_quant column sums");
}

extern "C" int ff_mxfp4_swiglu_quant(const void* gu, int64_t ldgu, int64_t rows, int64_t F, uint8_t* q_rows, int64_t ldq,
                                     uint8_t* s_rows, uint8_t* q_cols_t, int64_t ldqt, uint8_t* s_cols, void* stream) {
  using namespace ff::mx;
  Out o;
  int rc = make_out("ff_mxfp4_swiglu_quant", rows, F, q_rows, ldq, s_rows, q_cols_t, ldqt, s_cols, &o);
  if (rc) return rc;
  FF_REQUIRE(F % BLOCK == 0 && ldgu >= 2 * F && ldgu % 8 == 0 && ff::aligned(gu, 16), FF_ERR_UNSUPPORTED,
             "ff_mxfp4_swiglu_quant: F=%lld (a multiple of 32), ldgu=%lld (a multiple of 8, 16-byte aligned rows)", (long long)F,
             (long long)ldgu);
  if (rows == 0 || (!q_rows && !q_cols_t)) return FF_OK;
  FF_REQUIRE(gu, FF_ERR_INVALID_ARG, "ff_mxfp4_swiglu_quant: null pointer");
  int64_t tr, tc;
  rc = grid_of("ff_mxfp4_swiglu_quant", o, F, &tr, &tc);
  if (rc) return rc;
  static bool done[64] = {false};
  rc = allow_smem(mx_swiglu_quant_kernel, quant_smem<FF_DTYPE_BF16>(), done, "ff_mxfp4_swiglu_quant");
  if (rc) return rc;
  mx_swiglu_quant_kernel<<<(unsigned)(tr * tc), THREADS, quant_smem<FF_DTYPE_BF16>(), ff::as_stream(stream)>>>(
      static_cast<const __nv_bfloat16*>(gu), ldgu, F, tc, o);
  return ff::check_launch("ff_mxfp4_swiglu_quant");
}

extern "C" int ff_mxfp4_swiglu_bwd_quant(const void* dh, int64_t lddh, const void* gu, int64_t ldgu, int64_t rows, int64_t F,
                                         uint8_t* q_rows, int64_t ldq, uint8_t* s_rows, uint8_t* q_cols_t, int64_t ldqt,
                                         uint8_t* s_cols, void* stream) {
  using namespace ff::mx;
  Out o;
  int rc = make_out("ff_mxfp4_swiglu_bwd_quant", rows, 2 * F, q_rows, ldq, s_rows, q_cols_t, ldqt, s_cols, &o);
  if (rc) return rc;
  FF_REQUIRE(F % BLOCK == 0 && ldgu >= 2 * F && ldgu % 8 == 0 && lddh >= F && lddh % 8 == 0 && ff::aligned(gu, 16) &&
                 ff::aligned(dh, 16),
             FF_ERR_UNSUPPORTED,
             "ff_mxfp4_swiglu_bwd_quant: F=%lld (a multiple of 32), lddh=%lld, ldgu=%lld (multiples of 8, 16-byte aligned rows)",
             (long long)F, (long long)lddh, (long long)ldgu);
  if (rows == 0 || (!q_rows && !q_cols_t)) return FF_OK;
  FF_REQUIRE(gu && dh, FF_ERR_INVALID_ARG, "ff_mxfp4_swiglu_bwd_quant: null pointer");
  const int64_t tc = (F + 127) / 128, tr = q_cols_t ? chunks_of(rows) : (rows + 127) / 128;
  FF_REQUIRE(tr * tc < ((int64_t)1 << 31), FF_ERR_UNSUPPORTED, "ff_mxfp4_swiglu_bwd_quant: too many tiles");
  constexpr int smem = 2 * TILE * row_bytes<FF_DTYPE_BF16>() + TILE * 4;
  static bool done[64] = {false};
  rc = allow_smem(mx_swiglu_bwd_quant_kernel, smem, done, "ff_mxfp4_swiglu_bwd_quant");
  if (rc) return rc;
  mx_swiglu_bwd_quant_kernel<<<(unsigned)(tr * tc), THREADS, smem, ff::as_stream(stream)>>>(
      static_cast<const __nv_bfloat16*>(dh), lddh, static_cast<const __nv_bfloat16*>(gu), ldgu, F, tc, o);
  return ff::check_launch("ff_mxfp4_swiglu_bwd_quant");
}

extern "C" int ff_mxfp4_dequant(const uint8_t* q, int64_t ldq, const uint8_t* s, int64_t rows, int64_t cols, void* out,
                                int dtype, int64_t ldo, void* stream) {
  using namespace ff::mx;
  Out o;
  int rc = make_out("ff_mxfp4_dequant", rows, cols, const_cast<uint8_t*>(q), ldq, const_cast<uint8_t*>(s), nullptr, 0, nullptr, &o);
  if (rc) return rc;
  FF_REQUIRE(dtype >= FF_DTYPE_F32 && dtype <= FF_DTYPE_F16, FF_ERR_INVALID_ARG, "ff_mxfp4_dequant: bad dtype %d", dtype);
  FF_REQUIRE(ldo >= cols, FF_ERR_INVALID_ARG, "ff_mxfp4_dequant: ldo=%lld < cols=%lld", (long long)ldo, (long long)cols);
  if (rows == 0) return FF_OK;
  FF_REQUIRE(q && s && out, FF_ERR_INVALID_ARG, "ff_mxfp4_dequant: null pointer");
  const int64_t blocks = (rows * ((cols + 7) / 8) + 255) / 256;
  FF_REQUIRE(blocks < ((int64_t)1 << 31), FF_ERR_UNSUPPORTED, "ff_mxfp4_dequant: too large");
  const int vec = ff::aligned(out, 16) && (ldo * ff::dtype_size(dtype)) % 16 == 0;
  cudaStream_t st = ff::as_stream(stream);
  if (dtype == FF_DTYPE_F32)
    mx_dequant_kernel<FF_DTYPE_F32><<<(unsigned)blocks, 256, 0, st>>>(q, ldq, s, o.chunks_r, rows, cols, out, ldo, vec);
  else if (dtype == FF_DTYPE_BF16)
    mx_dequant_kernel<FF_DTYPE_BF16><<<(unsigned)blocks, 256, 0, st>>>(q, ldq, s, o.chunks_r, rows, cols, out, ldo, vec);
  else
    mx_dequant_kernel<FF_DTYPE_F16><<<(unsigned)blocks, 256, 0, st>>>(q, ldq, s, o.chunks_r, rows, cols, out, ldo, vec);
  return ff::check_launch("ff_mxfp4_dequant");
}
