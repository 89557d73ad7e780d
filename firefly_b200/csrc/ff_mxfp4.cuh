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
// (row / 128) * chunks + block / 4, chunks = 2 * ceil(cols / 256).  Blocks behind a row's last hold
// S = 0 (a finite scale for the zero codes that a tile load fills in).  The bytes of rows behind the
// matrix's last (up to the next 128) are 0 from ff_mxfp4_quant; from the SwiGLU kernels some are not
// written: they scale rows of a product that are not stored.
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

// eight values (already divided by the scale) -> one word of codes, the first in the lowest nibble
__device__ __forceinline__ uint32_t codes8(f2 p, f2 q, f2 r, f2 t) {
  uint32_t w;
  float v0, v1, v2, v3, v4, v5, v6, v7;
  un2(p, v0, v1);
  un2(q, v2, v3);
  un2(r, v4, v5);
  un2(t, v6, v7);
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(w)
      : "f"(v0), "f"(v1), "f"(v2), "f"(v3), "f"(v4), "f"(v5), "f"(v6), "f"(v7));
  return w;
}
__device__ __forceinline__ uint32_t codes8(const float (&v)[8]) {
  return codes8(mk2(v[0], v[1]), mk2(v[2], v[3]), mk2(v[4], v[5]), mk2(v[6], v[7]));
}
// one byte of codes -> two values
__device__ __forceinline__ float2 values2(uint32_t byte) {
  uint32_t h;
  asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, a;\n\t}" : "=r"(h) : "r"(byte));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// Programmatic launches: a kernel launched early is ordered after the ones before it on the stream from
// this wait on (nothing otherwise) ...
__device__ __forceinline__ void wait_for_previous_kernel() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// ... and a kernel allows the next one to start early once each of its CTAs has come here.
__device__ __forceinline__ void let_next_kernel_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// element types of the staged tile
template <int DT>
struct Pair;  // two neighbouring 16-bit values in one word
template <>
struct Pair<FF_DTYPE_BF16> {
  static __device__ __forceinline__ float lo(uint32_t w) { return __uint_as_float(w << 16); }
  static __device__ __forceinline__ float hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }
  static __device__ __forceinline__ uint32_t f32_bits(uint32_t h) { return h << 16; }
  static __device__ __forceinline__ f2 both(uint32_t w) { return unpack_bf16x2(w); }
};
template <>
struct Pair<FF_DTYPE_F16> {
  static __device__ __forceinline__ float lo(uint32_t w) { return __half2float(__ushort_as_half((unsigned short)(w & 0xFFFFu))); }
  static __device__ __forceinline__ float hi(uint32_t w) { return __half2float(__ushort_as_half((unsigned short)(w >> 16))); }
  static __device__ __forceinline__ uint32_t f32_bits(uint32_t h) {
    return __float_as_uint(__half2float(__ushort_as_half((unsigned short)h)));
  }
  static __device__ __forceinline__ f2 both(uint32_t w) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    return mk2(f.x, f.y);
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
  // the tile's own bases in 64 bits, everything per item in 32
  const int64_t blk0 = col0 / BLOCK;
  const int b = threadIdx.x & 3, r0 = threadIdx.x >> 2;
  const int live_rows = (int)min64(TILE, o.rows - row0);
  const bool put = blk0 + b < nblk, word = (blk0 & 3) == 0 && blk0 + 4 <= sblk, byte = !word && blk0 + b < sblk;
  const uint32_t ldq = (uint32_t)o.ldq;  // below 2^31: cols are
  uint8_t* q = o.q_rows + row0 * o.ldq + (blk0 + b) * 16;
  uint8_t* sc = o.s_rows + scale_at(row0, word ? blk0 : blk0 + b, o.chunks_r);
  if (live_rows <= 0) return;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = r0 + i * 64;
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
      const f2 inv = splat(inv_scale(S));
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        f2 t[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] = mul2(mk2(v[8 * k + 2 * e], v[8 * k + 2 * e + 1]), inv);
        w[k] = codes8(t[0], t[1], t[2], t[3]);
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
      const f2 inv = splat(inv_scale(S));
      uint32_t c[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        c[j] = codes8(mul2(Pair<DT>::both(p[j].x), inv), mul2(Pair<DT>::both(p[j].y), inv),
                      mul2(Pair<DT>::both(p[j].z), inv), mul2(Pair<DT>::both(p[j].w), inv));
      w[0] = swap ? c[2] : c[0];
      w[1] = swap ? c[3] : c[1];
      w[2] = swap ? c[0] : c[2];
      w[3] = swap ? c[1] : c[3];
    }
    if (S == kScaleNan) w[0] = w[1] = w[2] = w[3] = 0u;
    if (put && r < live_rows)
      *reinterpret_cast<uint4*>(q + (uint64_t)ldq * (uint32_t)r) = make_uint4(w[0], w[1], w[2], w[3]);
    // scales (row % 32 at 16 bytes, row / 32 at 4): the four lanes of a row hold one word of a chunk
    // when the tile starts on a chunk
    const int at = (r & 31) * 16 + (r >> 5) * 4;
    if (word) {
      const uint32_t s1 = S | (__shfl_down_sync(0xffffffffu, S, 1) << 8);
      const uint32_t s2 = s1 | (__shfl_down_sync(0xffffffffu, s1, 2) << 16);
      if (b == 0) *reinterpret_cast<uint32_t*>(sc + at) = s2;
    } else if (byte) {
      sc[at] = (uint8_t)S;
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
  const uint32_t ldqt = (uint32_t)o.ldqt;  // below 2^31: rows are
  uint8_t* q = o.q_cols + col0 * o.ldqt + row0 / 2;
  const int live_rb = (int)min64(4, (o.rows - row0 + BLOCK - 1) / BLOCK);  // row blocks that exist
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
      const f2 inv = splat(inv_scale(S));
      auto value = [&](int i) {
        if constexpr (DT == FF_DTYPE_F32) return __uint_as_float(x[i]);
        else return h ? Pair<DT>::hi(x[i]) : Pair<DT>::lo(x[i]);
      };
      uint32_t w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        f2 t[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] = mul2(mk2(value(8 * k + 2 * e), value(8 * k + 2 * e + 1)), inv);
        w[k] = codes8(t[0], t[1], t[2], t[3]);
      }
      if (S == kScaleNan) w[0] = w[1] = w[2] = w[3] = 0u;
      const int c = wc * W + h;
      // 16 bytes per 32 rows (ldqt covers whole blocks)
      if (c < live && rb < live_rb)
        *reinterpret_cast<uint4*>(q + (uint64_t)ldqt * (uint32_t)c + rb * 16) = make_uint4(w[0], w[1], w[2], w[3]);
      s_buf[c * 4 + rb] = (uint8_t)S;
      if (o.colsum) {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) sum += value(i);
        sum_buf[rb * TILE + c] = sum;
      }
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
// base and leading dimension allow, all of a thread's loads in flight before the first store.  Otherwise
// 16-bit values are read by a warp 32 neighbours at a time (8192 x 4095, one orientation: 35 us, against 51 with
// a piece per thread); fp32 stays with the pieces, whose loads are more in flight (53 us, against 59).
template <int DT>
__device__ __forceinline__ void stage_tile(uint8_t* tile, const void* x, int64_t ld, int64_t rows, int64_t cols,
                                           int64_t row0, int64_t col0, bool vec) {
  using T = typename Elem<DT>::T;
  if (sizeof(T) == 2 && !vec) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int live = (int)min64(TILE, rows - row0), n = (int)min64(TILE, cols - col0);
    const T* p = reinterpret_cast<const T*>(x) + row0 * ld + col0 + lane;
#pragma unroll 4
    for (int i = w; i < TILE; i += THREADS / 32) {
      T v[TILE / 32];
#pragma unroll
      for (int k = 0; k < TILE / 32; ++k) v[k] = i < live && k * 32 + lane < n ? p[i * ld + k * 32] : T(0.f);
#pragma unroll
      for (int k = 0; k < TILE / 32; ++k) reinterpret_cast<T*>(tile + i * row_bytes<DT>())[k * 32 + lane] = v[k];
    }
    return;
  }
  constexpr int V = 16 / (int)sizeof(T);
  constexpr int PER_ROW = TILE / V;
  constexpr int N = TILE * PER_ROW / THREADS;
  // a thread's pieces lie below one another, THREADS / PER_ROW rows apart
  constexpr int DR = THREADS / PER_ROW;
  const int64_t c = col0 + (threadIdx.x % PER_ROW) * V, r = row0 + threadIdx.x / PER_ROW;
  const int live = (int)min64(TILE, rows - r), n = (int)min64(V, max64(0, cols - c));
  const T* p = reinterpret_cast<const T*>(x) + r * ld + c;
  uint4 v[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = make_uint4(0, 0, 0, 0);
    if (i * DR < live && n > 0) {
      const T* q = p + (int64_t)(i * DR) * ld;
      if (vec && n == V) {
        v[i] = __ldg(reinterpret_cast<const uint4*>(q));
      } else {
        T* e = reinterpret_cast<T*>(&v[i]);
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (j < n) e[j] = q[j];
      }
    }
  }
  uint8_t* d = tile + (threadIdx.x / PER_ROW) * row_bytes<DT>() + (threadIdx.x % PER_ROW) * 16;
#pragma unroll
  for (int i = 0; i < N; ++i) *reinterpret_cast<uint4*>(d + i * DR * row_bytes<DT>()) = v[i];
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

// One 128 x 128 tile per CTA: read once, quantised along either axis or both from shared memory (fp32
// inputs, few tiles, unaligned rows).  fp32 8192 x 4096, both orientations: 49 us, 3.5 TB/s.
template <int DT>
__global__ void __launch_bounds__(THREADS, DT == FF_DTYPE_F32 ? 2 : 4) mx_quant_kernel(const void* x, int64_t ldx, int64_t tiles_c, Out o, int vec) {
  extern __shared__ __align__(16) uint8_t smem[];
  let_next_kernel_start();
  uint8_t* s_buf = smem + TILE * row_bytes<DT>();
  float* sum_buf = reinterpret_cast<float*>(s_buf + TILE * 4);
  const int64_t row0 = (blockIdx.x / tiles_c) * TILE, col0 = (blockIdx.x % tiles_c) * TILE;
  stage_tile<DT>(smem, x, ldx, o.rows, o.cols, row0, col0, vec != 0);
  __syncthreads();
  quant_tile<DT>(smem, row0, col0, o, s_buf, sum_buf);
}

// The same for 16-bit inputs whose rows are 16-byte aligned: persistent CTAs, three per SM, each with two
// tile buffers, so that the next tile arrives (cp.async) while one is quantised.
// 8192 x 4096 bf16, both orientations: 27 us with 3.8 TB/s of algorithmic bytes (30 us with one tile per CTA; a
// copy of as many bytes takes 18 us); along the rows alone 21 us.  No unit is full (14.8 instructions
// per value for both orientations, issue slots 64% and the ALU pipe 63% busy): a tile's wait, its rows and its columns
// follow one another between barriers, with 20 warps on an SM to fill the gaps.
template <int DT>
__host__ __device__ constexpr int pipe_smem() {
  return 2 * TILE * row_bytes<DT>() + TILE * 4 + 4 * TILE * 4;
}
// 16-byte pieces of a tile, zeros outside the matrix
template <int DT>
__device__ __forceinline__ void stage_async(uint32_t tile, const void* x, int64_t ld, int64_t rows, int64_t cols, int64_t row0,
                                            int64_t col0) {
  static_assert(DT != FF_DTYPE_F32, "16-bit types");
  // a thread's pieces lie below one another, 16 rows apart
  const int64_t c = col0 + (threadIdx.x % 16) * 8, r = row0 + threadIdx.x / 16;
  const int n = (int)min64(16, max64(0, (cols - c) * 2));  // bytes of a piece that exist
  const int live = (int)min64(TILE, rows - r);              // its rows, counted from the first piece's
  const uint8_t* src = static_cast<const uint8_t*>(x) + (n ? (r * ld + c) * 2 : 0);
  const int64_t step = n ? ld * 32 : 0;
  const uint32_t dst = tile + (threadIdx.x / 16) * row_bytes<DT>() + (threadIdx.x % 16) * 16;
#pragma unroll
  for (int i = 0; i < TILE * 16 / THREADS; ++i) {
    const bool on = i * 16 < live;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + i * 16 * row_bytes<DT>()),
                 "l"(on ? src + i * step : static_cast<const uint8_t*>(x)), "r"(on ? n : 0)
                 : "memory");
  }
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int DT>
__global__ void __launch_bounds__(THREADS, 3) mx_quant_pipe_kernel(const void* x, int64_t ldx, int tiles_c, int tiles, Out o) {
  extern __shared__ __align__(16) uint8_t smem[];
  let_next_kernel_start();
  constexpr int TB = TILE * row_bytes<DT>();
  uint8_t* s_buf = smem + 2 * TB;
  float* sum_buf = reinterpret_cast<float*>(s_buf + TILE * 4);
  const uint32_t base = static_cast<uint32_t>(__cvta_generic_to_shared(smem));
  int t = blockIdx.x, b = 0;
  if (t < tiles) stage_async<DT>(base, x, ldx, o.rows, o.cols, (int64_t)(t / tiles_c) * TILE, (int64_t)(t % tiles_c) * TILE);
  for (; t < tiles; t += gridDim.x, b ^= 1) {
    const int n = t + gridDim.x;
    if (n < tiles)
      stage_async<DT>(base + (b ^ 1) * TB, x, ldx, o.rows, o.cols, (int64_t)(n / tiles_c) * TILE, (int64_t)(n % tiles_c) * TILE);
    else
      asm volatile("cp.async.commit_group;" ::: "memory");
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncthreads();
    quant_tile<DT>(smem + b * TB, (int64_t)(t / tiles_c) * TILE, (int64_t)(t % tiles_c) * TILE, o, s_buf, sum_buf);
    __syncthreads();  // the buffer is filled again
  }
}

// sigmoid(g) = 1 / (1 + 2^(-g log2 e)) in fp32, on the special-function unit: exact at both ends (2^.. = inf
// gives 0, and 0 gives 1), between them off by at most 1.25 |g| 2^-24 (the rounded product and constant in the
// exponent; only the side where the value is small has all of it) and 2^-21 (both approximations and the sum):
// 2^-17 at g = -86.  What follows is rounded to bf16, half a step of which is 2^-8 of it.
__device__ __forceinline__ float ex2_rcp(float t) {
  float e, s;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(1.f + e));
  return s;
}
__device__ __forceinline__ float sigmoid_f32(float g) { return ex2_rcp(g * -1.4426950408889634f); }
__device__ __forceinline__ f2 sigmoid2(f2 g) {
  float a, b;
  un2(mul2(g, splat(-1.4426950408889634f)), a, b);
  return mk2(ex2_rcp(a), ex2_rcp(b));
}

__device__ __forceinline__ uint32_t swiglu_word(uint32_t wg, uint32_t wu) {
  const f2 g = unpack_bf16x2(wg);
  return pack_bf16x2(mul2(mul2(g, sigmoid2(g)), unpack_bf16x2(wu)));
}

// h = bf16(silu(g) * u) of the bf16 gate/up activations gu = [g | u], quantised like mx_quant_kernel;
// h itself is not written.  All 16 pieces of a thread are in flight before the first is used, three CTAs per
// SM: 8192 x 11008 97 us, 4.7 TB/s (127 us with addresses worked out per piece); 22 instructions per value, issue slots
// 62% and the ALU pipe 49% busy: the latency of a tile's loads, and its phases one after another.
__global__ void __launch_bounds__(THREADS, 3) mx_swiglu_quant_kernel(const __nv_bfloat16* gu, int64_t ld, int64_t F,
                                                                  int64_t tiles_c, Out o) {
  extern __shared__ __align__(16) uint8_t smem[];
  constexpr int DT = FF_DTYPE_BF16;
  uint8_t* s_buf = smem + TILE * row_bytes<DT>();
  float* sum_buf = reinterpret_cast<float*>(s_buf + TILE * 4);
  const int64_t row0 = (blockIdx.x / tiles_c) * TILE, col0 = (blockIdx.x % tiles_c) * TILE;
  // a thread's pieces lie below one another, 16 rows apart; F is a multiple of 32: whole pieces
  constexpr int N = TILE * 16 / THREADS;
  const int64_t c = col0 + (threadIdx.x % 16) * 8, r = row0 + threadIdx.x / 16;
  const int live = c < F ? (int)min64(TILE, o.rows - r) : 0;
  const __nv_bfloat16* pg = gu + r * ld + c;
  uint8_t* d = smem + (threadIdx.x / 16) * row_bytes<DT>() + (threadIdx.x % 16) * 16;
  uint4 wg[N], wu[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    wg[i] = wu[i] = make_uint4(0, 0, 0, 0);
    if (i * 16 < live) {
      wg[i] = __ldg(reinterpret_cast<const uint4*>(pg + i * 16 * ld));
      wu[i] = __ldg(reinterpret_cast<const uint4*>(pg + i * 16 * ld + F));
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i)  // silu(0) * 0 = 0 outside the matrix
    *reinterpret_cast<uint4*>(d + i * 16 * row_bytes<DT>()) =
        make_uint4(swiglu_word(wg[i].x, wu[i].x), swiglu_word(wg[i].y, wu[i].y), swiglu_word(wg[i].z, wu[i].z),
                   swiglu_word(wg[i].w, wu[i].w));
  __syncthreads();
  quant_tile<DT>(smem, row0, col0, o, s_buf, sum_buf);
}

__device__ __forceinline__ void swiglu_bwd_word(uint32_t wg, uint32_t wu, uint32_t wd, uint32_t& dg, uint32_t& du) {
  const f2 g = unpack_bf16x2(wg), d = unpack_bf16x2(wd), s = sigmoid2(g), one = splat(1.f);
  dg = pack_bf16x2(mul2(mul2(d, unpack_bf16x2(wu)), mul2(s, fma2(g, sub2(one, s), one))));
  du = pack_bf16x2(mul2(d, mul2(g, s)));
}

// The gradient of gu from dh and gu (all bf16), quantised as the matrix [dg | du] of 2F columns
// without being written:  dg = bf16(dh * u * sig(g) * (1 + g * (1 - sig(g)))),  du = bf16(dh * g * sig(g)).
// One CTA takes the same 128 features of dg and of du.  8192 x 11008: 171 us, 4.2 TB/s; bound like the forward
// kernel, at 38 instructions per value of dh.
__global__ void __launch_bounds__(THREADS, 2) mx_swiglu_bwd_quant_kernel(const __nv_bfloat16* dh, int64_t lddh,
                                                                      const __nv_bfloat16* gu, int64_t ld, int64_t F,
                                                                      int64_t tiles_c, Out o) {
  extern __shared__ __align__(16) uint8_t smem[];
  constexpr int DT = FF_DTYPE_BF16;
  constexpr int TB = TILE * row_bytes<DT>();
  uint8_t* s_buf = smem + 2 * TB;
  const int64_t row0 = (blockIdx.x / tiles_c) * TILE, col0 = (blockIdx.x % tiles_c) * TILE;
  constexpr int N = TILE * 16 / THREADS;
  {
    const int64_t c = col0 + (threadIdx.x % 16) * 8, r = row0 + threadIdx.x / 16;
    const int live = c < F ? (int)min64(TILE, o.rows - r) : 0;
    const __nv_bfloat16 *pg = gu + r * ld + c, *pd = dh + r * lddh + c;
    uint8_t* d = smem + (threadIdx.x / 16) * row_bytes<DT>() + (threadIdx.x % 16) * 16;
    // all 24 pieces of a thread in flight, two CTAs per SM (8192 x 11008: 172 us; four rows at a time 174 us,
    // three CTAs with four or two rows at a time 205 and 189 us)
    constexpr int G = N;
#pragma unroll
    for (int i0 = 0; i0 < N; i0 += G) {
      uint4 vg[G], vu[G], vd[G];
#pragma unroll
      for (int i = 0; i < G; ++i) {
        vg[i] = vu[i] = vd[i] = make_uint4(0, 0, 0, 0);
        if ((i0 + i) * 16 < live) {
          vg[i] = __ldg(reinterpret_cast<const uint4*>(pg + (i0 + i) * 16 * ld));
          vu[i] = __ldg(reinterpret_cast<const uint4*>(pg + (i0 + i) * 16 * ld + F));
          vd[i] = __ldg(reinterpret_cast<const uint4*>(pd + (i0 + i) * 16 * lddh));
        }
      }
#pragma unroll
      for (int i = 0; i < G; ++i) {
        uint4 wg, wu;
        swiglu_bwd_word(vg[i].x, vu[i].x, vd[i].x, wg.x, wu.x);
        swiglu_bwd_word(vg[i].y, vu[i].y, vd[i].y, wg.y, wu.y);
        swiglu_bwd_word(vg[i].z, vu[i].z, vd[i].z, wg.z, wu.z);
        swiglu_bwd_word(vg[i].w, vu[i].w, vd[i].w, wg.w, wu.w);
        *reinterpret_cast<uint4*>(d + (i0 + i) * 16 * row_bytes<DT>()) = wg;
        *reinterpret_cast<uint4*>(d + TB + (i0 + i) * 16 * row_bytes<DT>()) = wu;
      }
    }
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

// Eight values per thread and row: one word of codes -> 16 (or 32) bytes.  blockDim.x threads side by side
// in a row, four rows per thread in flight.  8192 x 4096 to bf16: 17.6 us, 4.8 TB/s; a copy of as many bytes takes
// as long.  fp32, and rows that do not start on 16 bytes, are turned through shared memory, so that a
// warp writes 32 neighbouring values at a time (8192 x 4095 bf16: 27 us, against 98).
template <int DT, bool VEC>
__global__ void __launch_bounds__(256) mx_dequant_kernel(const uint8_t* q, int64_t ldq, const uint8_t* s, int chunks, int64_t rows,
                                                         int cols, void* out, int64_t ldo) {
  using T = typename Elem<DT>::T;
  __shared__ alignas(16) T turn[VEC ? 1 : 8][256];
  const int lane = threadIdx.x & 31, c = ((int)blockIdx.x * blockDim.x + threadIdx.x) * 8, c0 = c - lane * 8;
  if ((VEC ? c : c0) >= cols) return;  // otherwise the whole warp: blockDim.x is a multiple of 32
  T* mine = turn[VEC ? 0 : (threadIdx.y * blockDim.x + threadIdx.x) >> 5];
  constexpr int R = 4;
  for (int64_t r0 = ((int64_t)blockIdx.y * blockDim.y + threadIdx.y) * R; r0 < rows; r0 += (int64_t)gridDim.y * blockDim.y * R) {
    const int live = (int)min64(R, rows - r0);
    const bool in = VEC || c < cols;
    const uint8_t* qr = q + r0 * ldq + c / 2;
    const uint8_t* sr = s + scale_at(r0, c / BLOCK, chunks);  // the next three rows' scales follow 16 bytes apart
    T* o = reinterpret_cast<T*>(out) + r0 * ldo + c;
    uint32_t w[R], S[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      w[i] = in && i < live ? __ldg(reinterpret_cast<const uint32_t*>(qr + i * ldq)) : 0u;
      S[i] = in && i < live ? __ldg(sr + i * 16) : 0u;
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      if (i >= live) break;
      alignas(16) T t[8];
      const float sv = scale_value(S[i]);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 p = values2((w[i] >> (8 * k)) & 0xFFu);
        if constexpr (DT == FF_DTYPE_F32) {
          t[2 * k] = p.x * sv;
          t[2 * k + 1] = p.y * sv;
        } else if constexpr (DT == FF_DTYPE_BF16) {
          reinterpret_cast<uint32_t*>(t)[k] = pack_bf16x2(mul2(mk2(p.x, p.y), splat(sv)));
        } else {
          t[2 * k] = __float2half_rn(p.x * sv);
          t[2 * k + 1] = __float2half_rn(p.y * sv);
        }
      }
      T* d = o + i * ldo;
      if (VEC && c <= cols - 8) {
#pragma unroll
        for (int k = 0; k < (int)(8 * sizeof(T) / 16); ++k)
          reinterpret_cast<uint4*>(d)[k] = reinterpret_cast<const uint4*>(t)[k];
      } else if (VEC) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (c + k < cols) d[k] = t[k];
      } else {
        __syncwarp();
#pragma unroll
        for (int k = 0; k < (int)(8 * sizeof(T) / 16); ++k)
          reinterpret_cast<uint4*>(mine + lane * 8)[k] = reinterpret_cast<const uint4*>(t)[k];
        __syncwarp();
        T* dw = d - lane * 8;
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (c0 + k * 32 + lane < cols) dw[k * 32 + lane] = mine[k * 32 + lane];
      }
    }
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

inline int num_sms() {
  static int cache[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (!cache[dev]) {
    int n = 0;
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    cache[dev] = n > 0 ? n : 148;
  }
  return cache[dev];
}

template <int DT>
inline int launch_quant(const void* x, int64_t ldx, int64_t tiles_r, int64_t tiles_c, const Out& o, cudaStream_t st) {
  static bool done[64] = {false};
  int rc = allow_smem(mx_quant_kernel<DT>, quant_smem<DT>(), done, "ff_mxfp4_quant");
  if (rc) return rc;
  const int vec = aligned(x, 16) && (ldx * dtype_size(DT)) % 16 == 0;
  if constexpr (DT != FF_DTYPE_F32) {
    if (vec && tiles_r * tiles_c > num_sms()) {  // fewer tiles than SMs: nothing to overlap
      static bool pdone[64] = {false};
      if ((rc = allow_smem(mx_quant_pipe_kernel<DT>, pipe_smem<DT>(), pdone, "ff_mxfp4_quant"))) return rc;
      const int64_t grid = min64(tiles_r * tiles_c, (int64_t)num_sms() * 3);
      mx_quant_pipe_kernel<DT><<<(unsigned)grid, THREADS, pipe_smem<DT>(), st>>>(x, ldx, (int)tiles_c, (int)(tiles_r * tiles_c), o);
      return check_launch("ff_mxfp4_quant");
    }
  }
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
  FF_REQUIRE(ff::aligned(x, ff::dtype_size(dtype)) && ff::aligned(colsum, 4) && ff::aligned(colsum_ws, 4), FF_ERR_INVALID_ARG,
             "ff_mxfp4_quant: x or the column sums are not aligned to their elements");
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
  FF_REQUIRE(ldo >= cols && ff::aligned(out, ff::dtype_size(dtype)), FF_ERR_INVALID_ARG,
             "ff_mxfp4_dequant: ldo=%lld < cols=%lld, or an output that is not aligned to its elements", (long long)ldo, (long long)cols);
  if (rows == 0) return FF_OK;
  FF_REQUIRE(q && s && out, FF_ERR_INVALID_ARG, "ff_mxfp4_dequant: null pointer");
  const int64_t per_row = (cols + 7) / 8;
  int bx = 32;
  while (bx < 256 && bx < per_row) bx *= 2;
  const int by = 256 / bx;
  const dim3 block(bx, by), grid((unsigned)((per_row + bx - 1) / bx), (unsigned)ff::min64(65535, (rows + by * 4 - 1) / (by * 4)));
  const bool vec = ff::aligned(out, 16) && (ldo * ff::dtype_size(dtype)) % 16 == 0;
  cudaStream_t st = ff::as_stream(stream);
  const int ch = (int)o.chunks_r, nc = (int)cols;
  // fp32: a thread's 32 bytes in a row would leave as two half-filled stores (8192 x 4096: 43 us, turned 33 us)
#define FF_DEQUANT(DT, VEC) mx_dequant_kernel<DT, VEC><<<grid, block, 0, st>>>(q, ldq, s, ch, rows, nc, out, ldo)
  if (dtype == FF_DTYPE_F32) FF_DEQUANT(FF_DTYPE_F32, false);
  else if (dtype == FF_DTYPE_BF16) vec ? FF_DEQUANT(FF_DTYPE_BF16, true) : FF_DEQUANT(FF_DTYPE_BF16, false);
  else vec ? FF_DEQUANT(FF_DTYPE_F16, true) : FF_DEQUANT(FF_DTYPE_F16, false);
#undef FF_DEQUANT
  return ff::check_launch("ff_mxfp4_dequant");
}
