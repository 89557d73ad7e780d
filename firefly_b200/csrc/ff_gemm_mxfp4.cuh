// ff_gemm_mxfp4.cuh — product of two MXFP4 operands on the 5th-generation tensor cores.
//
//   D[m, n] = sum_k A[m, k] * B[n, k] (+ bias[n])     A: M x K, B: N x K, values as ff_mxfp4.cuh holds them
//
// tcgen05.mma kind::mxf4 multiplies E2M1 codes, scales each run of 32 products by the two E8M0
// scales and accumulates in fp32 in TMEM; nothing is dequantised on the way.  64 values of K per
// instruction are 32 bytes, so a 128-byte swizzled row is 256 values of K, and the operand tiles
// and descriptors are those of the int8 kernels (ff_gemm_i8.cuh).  The scales of a k-block travel in
// the order that the tensor core wants (512-byte chunks of 128 rows x 4 blocks): TMA brings two
// chunks per 128 rows, they are spread over TMEM (lane = row % 32, word = row / 32, repeated for
// the four lane quarters), and the instruction descriptor says which two of a word's
// four bytes the current 64 values use.
//
// Two kernels:
//   mx_gemm_narrow_kernel  one CTA per 128 rows of B x up to 128 rows of A, operands swapped (B is the
//                          MMA's M side), K split over a cluster: few rows of A, a stream over B
//   mx_gemm_pair_kernel    a CTA pair per 256 x 256 tile (cta_group::2), persistent
// Either can end in the SwiGLU epilogue of a gate/up projection, whose 32 features of a row are one
// block of the format: h leaves as codes and scales and is never written in bf16.
//
// Waits are time-bounded as in ff_gemm_i8.cuh.
#pragma once

#include "ff_gemm_i8.cuh"
#include "ff_mxfp4.cuh"

namespace ff {
namespace mxg {

using namespace gemm;

constexpr int KB = 256;          // values of K per stage: 128 bytes of codes, two scale chunks
constexpr int SF_BYTES = 1024;   // scales of 128 rows x KB
constexpr int ROWS_BYTES = 128 * 128;  // codes of 128 rows x KB

struct Epi {
  void* D;
  int64_t ldd, M, N;
  const float* bias;
  int out_f32;
  int vec;        // 16-byte stores of rows allowed
  int tma_store;  // bf16 output through TMA (pair kernel)
  // SwiGLU epilogue: codes and scales of h [M, F]
  uint8_t* hq;
  uint8_t* hs;
  int64_t ldh, hchunks, F;
};

// Instruction descriptor, kind::mxf4: A and B E2M1 (1 at bits 7-9 and 10-11), K-major, E8M0 scales
// (bit 23), N >> 3 at bits 17-22, M >> 7 at bits 27-28, dense K = 64 (bit 31 = 0).
__host__ __device__ constexpr uint32_t idesc_mx(int m, int n) {
  return (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | (1u << 23) | ((uint32_t)(m >> 7) << 27);
}
// which bytes of the scale words this instruction uses: 0 or 2 (B at bits 4-5, A at bits 29-30)
__host__ __device__ constexpr uint32_t idesc_sf(uint32_t id) { return (id << 4) | (id << 29); }

// a 512-byte scale chunk: 32 rows of 16 bytes, no swizzle, groups of 8 rows 128 bytes apart
__device__ __forceinline__ uint64_t sf_desc(uint32_t saddr) {
  return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(128 >> 4) << 32) | ((uint64_t)1 << 46);
}

template <int CG>
__device__ __forceinline__ void sf_copy(uint32_t taddr, uint32_t saddr) {
  if constexpr (CG == 1)
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(sf_desc(saddr)) : "memory");
  else
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(sf_desc(saddr)) : "memory");
}

template <int CG>
__device__ __forceinline__ void mma_mx(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                       uint32_t accumulate) {
  if constexpr (CG == 1)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}

__device__ __forceinline__ float bf16_round(float v) { return __bfloat162float(__float2bfloat16_rn(v)); }

// h of one feature from the fp32 sums of its gate and up projections: the activations are bf16
__device__ __forceinline__ float swiglu_h(float g, float u) {
  g = bf16_round(g);
  u = bf16_round(u);
  return bf16_round(g * mx::sigmoid_f32(g) * u);
}

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// ---------------------------------------------------------------------------
// Few rows of A: a stream over B.  One work item is 128 rows of B (NW = 2: 128 gate rows and the same
// 128 up rows) against MP rows of A; the CTAs of a cluster take equal runs of its k-blocks.  Persistent
// clusters, one CTA per SM: the loads run on from item to item.  The fp32 partial sums meet in shared
// memory: each warp of the cluster adds its (row of A, 32 columns) pieces over the CTAs in rank order,
// so the result does not depend on timing and no workspace is needed.  Two barriers per CTA and buffer
// order the exchange: `pfull` (every CTA's partial sums are written) and `pfree` (every CTA has read
// them).  Where two buffers fit, an item's sums are added up after the next item's have been written,
// so that a CTA does not stand still for the others' arrival.  1x4096x22016: 17 us (48 MB; 15 us of it after
// the quantiser, with which it overlaps); 33x11008x4096: 13 us.  One SM's copies bring a k-block in 0.45 us
// (38 GB/s, the same with half the products or without the scale copies), so 148 SMs at work all the time would take
// 8.6 us; launch, TMEM, the first load's latency and the last exchange are about 5 us, the rest is SMs
// without an item.
// ---------------------------------------------------------------------------
__host__ __device__ constexpr int nr_stage_bytes(int mp, int nw) { return nw * (ROWS_BYTES + SF_BYTES) + mp * 128 + SF_BYTES; }
__host__ __device__ constexpr int nr_bufs(int mp, int nw) { return nw * mp <= 64 ? 2 : 1; }
__host__ __device__ constexpr int nr_part_one(int mp, int nw) { return nw * mp * 128 * 4; }
__host__ __device__ constexpr int nr_part_bytes(int mp, int nw) { return nr_bufs(mp, nw) * nr_part_one(mp, nw); }
__host__ __device__ constexpr int nr_stages(int mp, int nw) {
  return (224 * 1024 - nr_part_bytes(mp, nw)) / nr_stage_bytes(mp, nw) > 10
             ? 10
             : (224 * 1024 - nr_part_bytes(mp, nw)) / nr_stage_bytes(mp, nw);
}
constexpr int NR_THREADS = NUM_THREADS + 32;  // TMA, MMA, four epilogue warps, scale copies
__host__ __device__ constexpr int nr_smem(int mp, int nw) {
  return nr_stages(mp, nw) * nr_stage_bytes(mp, nw) + nr_part_bytes(mp, nw) + 1024 + 384;
}
__host__ __device__ constexpr int pow2_cols(int c) { return c <= 32 ? 32 : c <= 64 ? 64 : c <= 128 ? 128 : c <= 256 ? 256 : 512; }
__host__ __device__ constexpr int nr_tmem(int mp, int nw) { return pow2_cols(2 * nw * mp + nr_stages(mp, nw) * (nw + 1) * 8); }

// wait for a barrier on which other CTAs of the cluster arrive
__device__ __forceinline__ bool wait_bar_cluster(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  auto ready = [&]() {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
  };
  if (ready()) return true;
  const uint64_t t0 = globaltimer_ns(), limit = wait_limit_ns();
  while (true) {
    if (ready()) return true;
    if (*abort_flag) return false;
    if (globaltimer_ns() - t0 > limit) {
      *abort_flag = 1;
      raise_status(FF_DEVICE_TIMEOUT);
      return false;
    }
  }
}

using mx::let_next_kernel_start;
using mx::wait_for_previous_kernel;

template <int MP, int NW>
__global__ void __launch_bounds__(NR_THREADS, 1)
    mx_gemm_narrow_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmSW,
                          const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmSX, int num_kb,
                          int tiles_w, int tiles_x, Epi ep) {
  constexpr int ST = nr_stages(MP, NW), SB = nr_stage_bytes(MP, NW), TC = nr_tmem(MP, NW);
  static_assert(ST >= 2 && nr_smem(MP, NW) <= 232448, "shared memory");
  static_assert(2 * NW * MP + ST * (NW + 1) * 8 <= 512, "TMEM columns");
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t pad = (1024u - (raw & 1023u)) & 1023u;
  uint8_t* smem = smem_raw + pad;
  const uint32_t sbase = raw + pad;
  // stage: NW x 16 KB of B, MP x 128 B of A (1024-byte aligned for the swizzle), then the scales
  auto sW = [&](int s, int w) { return sbase + s * SB + w * ROWS_BYTES; };
  auto sX = [&](int s) { return sbase + s * SB + NW * ROWS_BYTES; };
  auto sSW = [&](int s, int w) { return sX(s) + MP * 128 + w * SF_BYTES; };
  auto sSX = [&](int s) { return sX(s) + MP * 128 + NW * SF_BYTES; };
  float* part = reinterpret_cast<float*>(smem + ST * SB);  // [w][row of A][128]
  const uint32_t part_addr = sbase + ST * SB;
  uint8_t* ctrl = smem + ST * SB + nr_part_bytes(MP, NW);
  const uint32_t cbase = part_addr + nr_part_bytes(MP, NW);
  auto full_bar = [&](int s) { return cbase + 8u * s; };
  auto empty_bar = [&](int s) { return cbase + 8u * (ST + s); };
  auto tfull_bar = [&](int a) { return cbase + 8u * (2 * ST + a); };
  auto tempty_bar = [&](int a) { return cbase + 8u * (2 * ST + 2 + a); };
  constexpr int PB = nr_bufs(MP, NW);
  auto pfull = [&](int b) { return cbase + 8u * (2 * ST + 4 + b); };
  auto pfree = [&](int b) { return cbase + 8u * (2 * ST + 6 + b); };
  const uint32_t drain = cbase + 8u * (2 * ST + 8);
  auto sf_ready = [&](int s) { return cbase + 8u * (2 * ST + 9 + s); };  // the stage's scales are in TMEM
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(ctrl + 8 * (3 * ST + 9));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(ctrl + 8 * (3 * ST + 9) + 4);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)blockIdx.x, csize = (int)gridDim.x;  // the cluster spans grid x
  const int kb0 = (int)((int64_t)num_kb * rank / csize), kb1 = (int)((int64_t)num_kb * (rank + 1) / csize);
  const int items = tiles_w * tiles_x, first = (int)blockIdx.y, stride = (int)gridDim.y;
  const bool direct = NW == 1 && csize == 1;  // no exchange

  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
      mbar_init(sf_ready(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tfull_bar(a), 1);
      mbar_init(tempty_bar(a), 4);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(pfull(b), 4 * csize);
      mbar_init(pfree(b), 4 * csize);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    tma_prefetch_desc(&tmW);
    tma_prefetch_desc(&tmSW);
    tma_prefetch_desc(&tmX);
    tma_prefetch_desc(&tmSX);
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(TC)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  if (csize > 1) cluster_sync_all();  // every CTA's barriers are there
  else __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  let_next_kernel_start();  // after the TMEM allocation: the next kernel's CTAs may allocate theirs now

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    if (lane == 0) {
      auto load_w = [&](int s, int it, int kb) {
        const int tw = it / tiles_x;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
          tma_load_2d(sW(s, w), &tmW, kb * 128, (int)(w * ep.F) + tw * 128, full_bar(s));
          tma_load_2d(sSW(s, w), &tmSW, kb * 256, (int)(w * (ep.F / 128)) + tw, full_bar(s));
        }
      };
      auto load_x = [&](int s, int it, int kb) {
        const int tx = it % tiles_x;
        tma_load_2d(sX(s), &tmX, kb * 128, tx * MP, full_bar(s));
        tma_load_2d(sSX(s), &tmSX, kb * 256, tx * MP / 128, full_bar(s));
      };
      // the weights of the first stages are asked for before A (the last kernel's output) is waited for
      int ahead = 0;
      if (first < items) {
        for (; ahead < ST && ahead < kb1 - kb0; ++ahead) {
          mbar_arrive_expect_tx(full_bar(ahead), SB);
          load_w(ahead, first, kb0 + ahead);
        }
      }
      wait_for_previous_kernel();
      int s = 0, n = 0;
      uint32_t phase = 0, used = 0, last = 0;
      bool ok = true;
      for (int it = first; ok && it < items; it += stride) {
        for (int kb = kb0; kb < kb1; ++kb, ++n) {
          if (n >= ahead) {
            if (!wait_bar(empty_bar(s), phase ^ 1u, abort_flag)) {
              ok = false;
              break;
            }
            mbar_arrive_expect_tx(full_bar(s), SB);
            load_w(s, it, kb);
          }
          load_x(s, it, kb);
          used |= 1u << s;
          last = (last & ~(1u << s)) | (phase << s);
          if (++s == ST) {
            s = 0;
            phase ^= 1u;
          }
        }
      }
      for (int k = 0; k < ST; ++k)
        if (used & (1u << k)) drain_bar(full_bar(k), (last >> k) & 1u);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      constexpr uint32_t idesc = idesc_mx(128, MP);
      int s = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int it = first; ok && it < items; it += stride) {
        if (!wait_bar(tempty_bar(acc), acc_phase ^ 1u, abort_flag)) break;
        tc_fence_after();
        const uint32_t d = tmem + (uint32_t)(acc * NW * MP);
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!wait_bar(sf_ready(s), phase, abort_flag)) {  // after the stage itself: the copies waited for it
            ok = false;
            break;
          }
          tc_fence_after();
          // the scales of A cover 128 rows, 32 to a column: the second half of them belongs to an odd tile of 64
          const uint32_t sf = tmem + (uint32_t)(2 * NW * MP + s * (NW + 1) * 8);
          const uint32_t sfx = sf + NW * 8 + (uint32_t)(it % tiles_x * MP % 128 / 32);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
#pragma unroll
            for (int w = 0; w < NW; ++w)
              mma_mx<1>(d + w * MP, smem_desc_k_sw128(sW(s, w) + k * 32), smem_desc_k_sw128(sX(s) + k * 32),
                        idesc | idesc_sf((k & 1) * 2), sf + w * 8 + (k >> 1) * 4, sfx + (k >> 1) * 4,
                        (kb != kb0 || k != 0) ? 1u : 0u);
          }
          tc_commit(empty_bar(s));
          if (++s == ST) {
            s = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        tc_commit(tfull_bar(acc));
        if (++acc == 2) {
          acc = 0;
          acc_phase ^= 1u;
        }
      }
      tc_commit(drain);
      drain_bar(drain, 0);
    }
    __syncwarp();
  } else if (warp == 6) {
    // ------------------------------------------------------------ scales into TMEM
    // by a warp of its own: one thread's copies and products do not overlap (4096 x 22016, one CTA: 0.5 us per
    // k-block with the copies in the MMA thread)
    if (lane == 0) {
      int s = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int it = first; ok && it < items; it += stride) {
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!wait_bar(full_bar(s), phase, abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sf = tmem + (uint32_t)(2 * NW * MP + s * (NW + 1) * 8);  // slots as many as stages
#pragma unroll
          for (int c = 0; c < 2; ++c) {
#pragma unroll
            for (int w = 0; w < NW; ++w) sf_copy<1>(sf + w * 8 + c * 4, sSW(s, w) + c * 512);
            sf_copy<1>(sf + NW * 8 + c * 4, sSX(s) + c * 512);
          }
          tc_commit(sf_ready(s));
          if (++s == ST) {
            s = 0;
            phase ^= 1u;
          }
        }
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ epilogue
    const int lg = warp & 3;
    int acc = 0;
    uint32_t acc_phase = 0;
    // adds up the sums of this CTA group's n-th item, which lie in buffer n % PB
    auto finish = [&](int n) -> bool {
      const int it = first + n * stride, b = n % PB;
      const int tw = it / tiles_x, tx = it % tiles_x;
      const int jn = (int)min64(MP, ep.M - (int64_t)tx * MP);
      if (!__all_sync(0xffffffffu, wait_bar_cluster(pfull(b), (uint32_t)(n / PB) & 1u, abort_flag))) return false;
#pragma unroll 1
      for (int p = rank * 4 + (warp - 2); p < jn * 4; p += csize * 4) {
        const int j = p >> 2, lq = p & 3;
        const uint32_t at = part_addr + (uint32_t)(b * nr_part_one(MP, NW) + (j * 128 + lq * 32 + lane) * 4);
        float v = 0.f, u = 0.f;
#pragma unroll 4
        for (int r = 0; r < csize; ++r) {
          const uint32_t a = mapa_shared(at, (uint32_t)r);
          v += ld_cluster_f32(a);
          if constexpr (NW == 2) u += ld_cluster_f32(a + MP * 128 * 4);
        }
        const int64_t m = (int64_t)tx * MP + j;
        if constexpr (NW == 1) {
          const int64_t n_ = (int64_t)tw * 128 + lq * 32 + lane;
          if (n_ < ep.N) {
            if (ep.bias) v += __ldg(ep.bias + n_);
            if (ep.out_f32) static_cast<float*>(ep.D)[m * ep.ldd + n_] = v;
            else static_cast<__nv_bfloat16*>(ep.D)[m * ep.ldd + n_] = __float2bfloat16_rn(v);
          }
        } else {
          // one block of h: 32 features, a lane each
          const float h = swiglu_h(v, u);
          const uint32_t S = mx::scale_code(__reduce_max_sync(0xffffffffu, __float_as_uint(h) & 0x7FFFFFFFu));
          const float t[8] = {h * mx::inv_scale(S), 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
          uint32_t w = S == mx::kScaleNan ? 0u : (mx::codes8(t) & 0xFu) << (4 * (lane & 7));
          w |= __shfl_xor_sync(0xffffffffu, w, 1);
          w |= __shfl_xor_sync(0xffffffffu, w, 2);
          w |= __shfl_xor_sync(0xffffffffu, w, 4);
          const int64_t blk = (int64_t)tw * 4 + lq;
          if ((lane & 7) == 0) *reinterpret_cast<uint32_t*>(ep.hq + m * ep.ldh + blk * 16 + (lane >> 3) * 4) = w;
          if (lane == 0) ep.hs[mx::scale_at(m, blk, ep.hchunks)] = (uint8_t)S;
        }
      }
      if constexpr (NW == 2) {  // the padding chunk of h's scales
        if (rank == 0 && tw == tiles_w - 1 && tx % (128 / MP) == 0 && ep.hchunks * 128 > ep.F)
          reinterpret_cast<uint32_t*>(ep.hs)[((int64_t)(tx * MP / 128) * ep.hchunks + ep.F / 128) * 128 + (threadIdx.x - 64)] = 0;
      }
      __syncwarp();
      if (lane < csize) mbar_arrive_remote(mapa_shared(pfree(b), (uint32_t)lane));
      return true;
    };
    int n = 0;
    bool ok = true;
    for (int it = first; ok && it < items; it += stride, ++n) {
      const int tw = it / tiles_x, tx = it % tiles_x;
      const int jn = (int)min64(MP, ep.M - (int64_t)tx * MP);
      if (!__all_sync(0xffffffffu, wait_bar(tfull_bar(acc), acc_phase, abort_flag))) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint32_t tb = tmem + ((uint32_t)(lg * 32) << 16) + (uint32_t)(acc * NW * MP);
      if (direct) {
        const int64_t n_ = (int64_t)tw * 128 + lg * 32 + lane;
        const float b = ep.bias && n_ < ep.N ? __ldg(ep.bias + n_) : 0.f;
#pragma unroll 1
        for (int c = 0; c < jn; c += 16) {
          uint32_t r[16];
          tmem_ld16(tb + c, r);
          tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            if (c + j < jn && n_ < ep.N) {
              const int64_t at = ((int64_t)tx * MP + c + j) * ep.ldd + n_;
              const float v = __uint_as_float(r[j]) + b;
              if (ep.out_f32) static_cast<float*>(ep.D)[at] = v;
              else static_cast<__nv_bfloat16*>(ep.D)[at] = __float2bfloat16_rn(v);
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(tempty_bar(acc));
      } else {
        // the partial sums that lay in this buffer have been read everywhere
        const int b = n % PB;
        if (!__all_sync(0xffffffffu, wait_bar_cluster(pfree(b), ((uint32_t)(n / PB) & 1u) ^ 1u, abort_flag))) {
          ok = false;
          break;
        }
        float* dst = part + b * (nr_part_one(MP, NW) / 4);
#pragma unroll 1
        for (int c = 0; c < NW * MP; c += 16) {
          if (c % MP >= jn) continue;
          uint32_t r[16];
          tmem_ld16(tb + c, r);
          tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < 16; ++j) dst[(c + j) * 128 + lg * 32 + lane] = __uint_as_float(r[j]);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(tempty_bar(acc));
        if (lane < csize) mbar_arrive_remote(mapa_shared(pfull(b), (uint32_t)lane));
        if (n >= PB - 1) ok = finish(n - (PB - 1));
      }
      if (++acc == 2) {
        acc = 0;
        acc_phase ^= 1u;
      }
    }
    if (ok && !direct && PB == 2 && n > 0) finish(n - 1);
    __syncwarp();
  }

  tc_fence_before();
  if (csize > 1) cluster_sync_all();  // no CTA leaves while another reads its partial sums or arrives on its barriers
  else __syncthreads();
  tc_fence_after();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TC) : "memory");
}

// ---------------------------------------------------------------------------
// Large products: a CTA pair per 256 x 256 tile (M = 256, cta_group::2).  Each CTA stages its own 128
// rows of A and of B and the scales of its rows of A; the scales of all 256 rows of B are needed in
// both CTAs' TMEM (each multiplies its 128 rows of A with all of them), so each CTA loads them.
//
// TMEM: the scales need columns that two 256-column accumulators do not leave.  The accumulators
// overlap by half instead ([0, 256) and [128, 384)); a tile's epilogue reads the shared columns into
// registers first and then lets the next tile's products start.  Every stage has its slot of 24
// columns (the scales of one k-block: 8 of A, 16 of B) from column 384 on, so a slot is free as soon as
// its stage is loaded again.
//
// The scale copies are issued by two warps of their own.  In one thread's order copies and products do not
// overlap (8192x4096x11008: 195 us with a k-block's six copies ahead of its products, 8 us for each of the
// six, and no gain from copying earlier; 268 us with four warps writing the scales by tcgen05.st); issued
// by another warp, with a commit and a barrier between, they do: 144 us, within 2% of the time without
// any copies.  Two copy warps with half of a stage's copies each take 1 to 3% less than one (timed in turn, L2
// cold: 22016x4096x8192 268 -> 262 us = 5.6 PFLOP/s, 8192x2048x8192 63.5 -> 61.5, 4000x12288x4096 94.2 -> 92.1;
// 8192x4096x11008 136 us = 5.4, 8192x8192x2048 78 us = 3.5).  A last wave of tiles that at most half fills the
// GPU is cut into 256 x 128 halves.  The tensor pipe is active 69% of the cycles (with one copy warp), and the SM
// clock falls to 1.64 GHz under it; K = 2048 leaves eight k-blocks per tile, over which the start of a tile (its
// accumulator's shared half has to be read) weighs.
// ---------------------------------------------------------------------------
constexpr int PR_STAGES = 5;
constexpr int PR_CODES = 2 * ROWS_BYTES;                 // 128 rows of A and of B
constexpr int PR_STAGE = PR_CODES + 3 * SF_BYTES;        // and the scales of A (128 rows) and B (256 rows)
constexpr int PR_EPI_WARPS = 8;
constexpr int PR_CP_WARPS = 2;
constexpr int PR_THREADS = 64 + 32 * (PR_EPI_WARPS + PR_CP_WARPS);  // TMA, MMA, epilogue, scale copies
constexpr int PR_ACC1 = 128, PR_SF = 384, PR_SF_COLS = 24;
static_assert(PR_SF + PR_STAGES * PR_SF_COLS <= 512, "TMEM columns");
constexpr int PR_STAGING = PR_EPI_WARPS * 2 * 2048;      // two 32 x 32 bf16 boxes per epilogue warp
constexpr int PR_SMEM = PR_STAGES * PR_STAGE + 1024 + 512 + PR_STAGING;
static_assert(PR_SMEM <= 232448, "pair kernel exceeds the shared memory of a CTA");

// 32 columns of one row (a thread) of the output; all lanes take part
__device__ __forceinline__ void pair_store(uint32_t (&r)[32], int64_t row, int64_t col0, const Epi& ep, const CUtensorMap* tmD,
                                           int lane, uint8_t* stage, uint32_t stage_addr, uint32_t& nst) {
  if (col0 >= ep.N) return;
  if (ep.bias) {
    const float bl = col0 + lane < ep.N ? __ldg(ep.bias + col0 + lane) : 0.f;
#pragma unroll
    for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) + __shfl_sync(0xffffffffu, bl, j));
  }
  if (ep.tma_store) {
    uint32_t w[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) w[j] = pack_bf16x2(mk2(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1])));
    staged_store<true>(w, tmD, (int32_t)col0, (int32_t)(row - lane), lane, stage, stage_addr, nst);
  } else {
    // turned through shared memory, so that a warp writes 32 neighbouring columns of one row at a time
    // (4000x12287x4096, bf16: 115 us, against 533 with a row per thread; 22016x4096x8192 fp32: 290 against 334)
    const int64_t row0 = row - lane;
    if (row0 >= ep.M) return;
    float* t = reinterpret_cast<float*>(stage);
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 32; ++j) t[lane * 32 + (j ^ lane)] = __uint_as_float(r[j]);
    __syncwarp();
    const int rows = col0 + lane < ep.N ? (int)min((int64_t)32, ep.M - row0) : 0;
    if (ep.out_f32) {
      float* o = static_cast<float*>(ep.D) + row0 * ep.ldd + col0 + lane;
#pragma unroll
      for (int i = 0; i < 32; ++i, o += ep.ldd)
        if (i < rows) *o = t[i * 32 + (lane ^ i)];
    } else {
      __nv_bfloat16* o = static_cast<__nv_bfloat16*>(ep.D) + row0 * ep.ldd + col0 + lane;
#pragma unroll
      for (int i = 0; i < 32; ++i, o += ep.ldd)
        if (i < rows) *o = __float2bfloat16_rn(t[i * 32 + (lane ^ i)]);
    }
  }
}

template <bool GATED>
__global__ void __launch_bounds__(PR_THREADS, 1)
    mx_gemm_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmSA,
                        const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmSB,
                        const __grid_constant__ CUtensorMap tmD, const __grid_constant__ CUtensorMap tmB2, int num_kb,
                        int tiles_m, int tiles_n, int split, Epi ep) {
  constexpr int ST = PR_STAGES;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t pad = (1024u - (raw & 1023u)) & 1023u;
  uint8_t* smem = smem_raw + pad;
  const uint32_t sbase = raw + pad;
  auto sA = [&](int s) { return sbase + s * PR_STAGE; };
  auto sB = [&](int s) { return sbase + s * PR_STAGE + ROWS_BYTES; };
  auto sSA = [&](int s) { return sbase + s * PR_STAGE + PR_CODES; };
  auto sSB = [&](int s, int half) { return sbase + s * PR_STAGE + PR_CODES + (1 + half) * SF_BYTES; };
  uint8_t* ctrl = smem + ST * PR_STAGE;
  const uint32_t cbase = sbase + ST * PR_STAGE;
  auto full_bar = [&](int s) { return cbase + 8u * s; };
  auto empty_bar = [&](int s) { return cbase + 8u * (ST + s); };
  auto tfull_bar = [&](int a) { return cbase + 8u * (2 * ST + a); };
  const uint32_t shared_bar = cbase + 8u * (2 * ST + 2);  // leader: the shared columns have been read (16 warps)
  const uint32_t drain = cbase + 8u * (2 * ST + 3);
  const uint32_t done_bar = cbase + 8u * (2 * ST + 4);
  auto sf_ready = [&](int s) { return cbase + 8u * (2 * ST + 5 + s); };  // leader: the stage's scales are in TMEM
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(ctrl + 8 * (3 * ST + 5));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(ctrl + 8 * (3 * ST + 5) + 4);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank(), peer = rank ^ 1u;
  const int total = tiles_m * tiles_n, pair = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;
  // This pair's j-th item: tile pair + j * num_pairs; with `split` the tiles of the last partial wave (at
  // most half as many as pairs) are cut into 256 x 128 halves, one per pair.  half = -1: a whole tile.
  const int full_waves = split ? total / num_pairs : 0, rest = total - full_waves * num_pairs;
  auto item = [&](int j, int& tm, int& tn, int& half) -> bool {
    int t = pair + j * num_pairs;
    half = -1;
    if (split && j >= full_waves) {
      if (j > full_waves || pair >= 2 * rest) return false;
      t = full_waves * num_pairs + (pair >> 1);
      half = pair & 1;
    }
    if (t >= total) return false;
    tile_coords(t, tiles_m, tiles_n, tm, tn);
    return true;
  };
  const uint32_t num_items = split ? (uint32_t)(full_waves + (pair < 2 * rest ? 1 : 0))
                                   : (pair < total ? (uint32_t)((total - pair + num_pairs - 1) / num_pairs) : 0u);

  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
      mbar_init(sf_ready(s), PR_CP_WARPS);
    }
    mbar_init(tfull_bar(0), 1);
    mbar_init(tfull_bar(1), 1);
    mbar_init(shared_bar, 2 * PR_EPI_WARPS);
    mbar_init(drain, 1);
    mbar_init(done_bar, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmSA);
    tma_prefetch_desc(&tmB);
    tma_prefetch_desc(&tmSB);
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  let_next_kernel_start();  // after the TMEM allocation: the next kernel's CTAs may allocate theirs now

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer (both CTAs)
    if (lane == 0) {
      wait_for_previous_kernel();
      int s = 0;
      uint32_t phase = 0;
      bool ok = true;
      int tm, tn, half;
      for (int j = 0; ok && item(j, tm, tn, half); ++j) {
        const int ra = tm * 2 + (int)rank;  // this CTA's 128 rows of A, in units of 128
        // the 128-row groups of B: both halves of the tile, or twice the one half
        const int rb0 = GATED ? tn : tn * 2 + (half > 0), rb1 = GATED ? (int)(ep.F / 128) + tn : tn * 2 + (half != 0);
        const int rb = rank ? rb1 : rb0;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!wait_bar(empty_bar(s), phase ^ 1u, abort_flag)) {
            ok = false;
            break;
          }
          const uint32_t lbar = mapa_shared(full_bar(s), 0);
          if (rank == 0) mbar_arrive_expect_tx(full_bar(s), 2 * (half < 0 ? PR_STAGE : PR_STAGE - ROWS_BYTES / 2));
          tma_load_2d_pair(sSA(s), &tmSA, kb * 256, ra, lbar);
          tma_load_2d_pair(sSB(s, 0), &tmSB, kb * 256, rb0, lbar);
          tma_load_2d_pair(sSB(s, 1), &tmSB, kb * 256, rb1, lbar);
          tma_load_2d_pair(sA(s), &tmA, kb * 128, ra * 128, lbar);
          if (half < 0) tma_load_2d_pair(sB(s), &tmB, kb * 128, rb * 128, lbar);
          else tma_load_2d_pair(sB(s), &tmB2, kb * 128, rb0 * 128 + (int)rank * 64, lbar);  // its 64 rows of the half
          if (++s == ST) {
            s = 0;
            phase ^= 1u;
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (leader only)
    if (rank == 0 && lane == 0) {
      int s = 0, acc = 0, tm_, tn_, half;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = 0; ok && item(tile, tm_, tn_, half); ++tile) {
        const uint32_t idesc = half < 0 ? idesc_mx(256, 256) : idesc_mx(256, 128);
        if (tile > 0 && !wait_bar(shared_bar, (uint32_t)(tile - 1) & 1u, abort_flag)) break;
        const uint32_t d = tmem + (uint32_t)(acc * PR_ACC1);
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!wait_bar(sf_ready(s), phase, abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sf = tmem + PR_SF + (uint32_t)(s * PR_SF_COLS);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            mma_mx<2>(d, smem_desc_k_sw128(sA(s) + k * 32), smem_desc_k_sw128(sB(s) + k * 32), idesc | idesc_sf((k & 1) * 2),
                      sf + (k >> 1) * 4, sf + 8 + (k >> 1) * 8, (kb | k) != 0);
          tc_commit_pair(empty_bar(s));
          if (++s == ST) {
            s = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        tc_commit_pair(tfull_bar(acc));
        acc ^= 1;
      }
      tc_commit(drain);
      drain_bar(drain, 0);
    }
    __syncwarp();
  } else if (warp >= 2 + PR_EPI_WARPS) {
    // ------------------------------------------------------------ scales into TMEM (leader only)
    // Each of the two warps copies half of every stage's scales.  Both wait for every phase of every stage's
    // barrier, in order, and the product of a stage waits for both, so no phase can pass either of them by.
    if (rank == 0 && lane == 0) {
      const uint32_t steps = num_items * (uint32_t)num_kb;
      const uint32_t c = (uint32_t)(warp - 2 - PR_EPI_WARPS);
      int s = 0;
      uint32_t phase = 0, g = 0;
      for (; g < steps; ++g) {
        if (!wait_bar(full_bar(s), phase, abort_flag)) break;
        tc_fence_after();
        const uint32_t sf = tmem + PR_SF + (uint32_t)(s * PR_SF_COLS);
        sf_copy<2>(sf + c * 4, sSA(s) + c * 512);
        sf_copy<2>(sf + 8 + c * 8, sSB(s, 0) + c * 512);
        sf_copy<2>(sf + 8 + c * 8 + 4, sSB(s, 1) + c * 512);
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(sf_ready(s)) : "memory");
        if (++s == ST) {
          s = 0;
          phase ^= 1u;
        }
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ epilogue (both CTAs)
    const int lg = warp & 3, eh = (warp - 2) >> 2;  // TMEM lane quarter; which of the quarter's two warps
    uint8_t* stage = ctrl + 512 + (warp - 2) * 4096;
    const uint32_t stage_addr = cbase + 512 + (uint32_t)(warp - 2) * 4096;
    uint32_t nst = 0;
    int tm, tn, half;
    const uint32_t sbar = mapa_shared(shared_bar, 0);
    for (int tile = 0; item(tile, tm, tn, half); ++tile) {
      const int acc = tile & 1;
      if (!__all_sync(0xffffffffu, wait_bar(tfull_bar(acc), (uint32_t)(tile >> 1) & 1u, abort_flag))) break;
      tc_fence_after();
      const int64_t row0 = (int64_t)(tm * 2 + (int)rank) * 128 + lg * 32, row = row0 + lane;
      const uint32_t tb = tmem + ((uint32_t)(lg * 32) << 16) + (uint32_t)(acc * PR_ACC1);
      // the columns that the accumulators share (the upper half of accumulator 0, the lower half of
      // accumulator 1) are read first: two 32-column chunks per warp, then the next tile may start
      const int sh = acc || half >= 0 ? 0 : 4;  // a half tile has no other columns (and no next tile)
      uint32_t r0[32], r1[32];
      tmem_ld32(tb + (sh + eh * 2) * 32, r0);
      tmem_ld32(tb + (sh + eh * 2 + 1) * 32, r1);
      tmem_wait_ld();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_remote(sbar);
      if constexpr (!GATED) {
        const int64_t col0 = (int64_t)tn * 256 + (half > 0 ? 128 : 0) + eh * 64;
        pair_store(r0, row, col0 + sh * 32, ep, &tmD, lane, stage, stage_addr, nst);
        pair_store(r1, row, col0 + sh * 32 + 32, ep, &tmD, lane, stage, stage_addr, nst);
#pragma unroll 1
        for (int i = 0; i < 2 && half < 0; ++i) {
          tmem_ld32(tb + ((4 - sh) + eh * 2 + i) * 32, r0);
          tmem_wait_ld();
          pair_store(r0, row, col0 + (4 - sh) * 32 + i * 32, ep, &tmD, lane, stage, stage_addr, nst);
        }
      } else {
        // gate features in the lower half, up features in the upper half: one half of each block is here
        uint32_t ro[32];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int c = eh * 2 + i;
          tmem_ld32(tb + ((4 - sh) + c) * 32, ro);
          tmem_wait_ld();
          // one block of h per thread
          float h[32];
          uint32_t m = 0;
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            const float x = __uint_as_float(i ? r1[j] : r0[j]), y = __uint_as_float(ro[j]);
            h[j] = swiglu_h(acc ? x : y, acc ? y : x);
            m = max(m, __float_as_uint(h[j]) & 0x7FFFFFFFu);
          }
          const uint32_t S = mx::scale_code(m);
          const float inv = mx::inv_scale(S);
          uint32_t w[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = h[8 * k + e] * inv;
            w[k] = S == mx::kScaleNan ? 0u : mx::codes8(v);
          }
          const int64_t blk = (int64_t)tn * 4 + c;
          if (row < ep.M) {
            *reinterpret_cast<uint4*>(ep.hq + row * ep.ldh + blk * 16) = make_uint4(w[0], w[1], w[2], w[3]);
            ep.hs[mx::scale_at(row, blk, ep.hchunks)] = (uint8_t)S;
          }
        }
        // the padding chunk of h's scales: by the last tile column
        if (eh == 0 && tn == tiles_n - 1 && ep.hchunks * 128 > ep.F && row < ((ep.M + 127) & ~(int64_t)127))
          *reinterpret_cast<uint32_t*>(ep.hs + mx::scale_at(row, ep.F / 32, ep.hchunks)) = 0u;
      }
    }
    if (nst && lane == 0) bulk_wait_all();
    __syncwarp();
  }

  tc_fence_before();
  __syncthreads();
  if (*abort_flag) spin_ns(20000);  // let any TMA load still in flight land before the CTA exits
  if (threadIdx.x == 32) {  // neither CTA frees TMEM before the other is done with the pair's allocation
    mbar_arrive_remote(mapa_shared(done_bar, peer));
    drain_bar(done_bar, 0);
  }
  __syncthreads();
  tc_fence_after();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
// scales as a matrix of 32-bit words, one row per 128 rows of the operand: boxes of 256 words
inline int make_map_sf(CUtensorMap* m, const uint8_t* s, int64_t rows, int64_t cols) {
  auto fn = encode_fn();
  if (!fn) return set_error(FF_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  const int64_t words = mx::chunks_of(cols) * 128;
  cuuint64_t dims[2] = {(cuuint64_t)words, (cuuint64_t)((rows + 127) / 128)};
  cuuint64_t strides[1] = {(cuuint64_t)(words * 4)};
  cuuint32_t box[2] = {256, 1}, estr[2] = {1, 1};
  CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<uint8_t*>(s), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(FF_ERR_CUDA, "cuTensorMapEncodeTiled (scales) failed (%d)", (int)r);
  return FF_OK;
}
// codes: [rows, K] two to a byte; boxes of 128 bytes x box_rows, zeros outside
inline int make_map_codes(CUtensorMap* m, const uint8_t* q, int64_t rows, int64_t cols, int64_t ld, int box_rows) {
  return make_map(m, reinterpret_cast<const int8_t*>(q), rows, (cols + 31) / 32 * 16, ld, box_rows);
}

struct Operand {
  const uint8_t* q;
  int64_t ld;
  const uint8_t* s;
};

// attributes of a cluster launch; `early`: the kernel may start before the one ahead of it on the stream
// has finished (it waits for it where it reads that kernel's output)
struct LaunchAttrs {
  cudaLaunchAttribute a[2];
  LaunchAttrs(cudaLaunchConfig_t& cfg, int cluster, bool early) {
    a[0].id = cudaLaunchAttributeClusterDimension;
    a[0].val.clusterDim.x = (unsigned)cluster;
    a[0].val.clusterDim.y = 1;
    a[0].val.clusterDim.z = 1;
    a[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    a[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = a;
    cfg.numAttrs = early ? 2 : 1;
  }
};

// clusters of `csize` CTAs (one per SM) that run at once, cached per device
template <int MP, int NW>
inline int narrow_clusters(int csize) {
  static int cache[64][4] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return num_sms_current() / csize / 2 + 1;
  const int lc = csize == 1 ? 0 : csize == 2 ? 1 : csize == 4 ? 2 : 3;
  if (!cache[dev][lc]) {
    static bool done[64] = {false};
    mx::allow_smem(mx_gemm_narrow_kernel<MP, NW>, nr_smem(MP, NW), done, "ff_mxfp4_gemm");  // or nothing would fit
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)csize);
    cfg.blockDim = dim3(NR_THREADS);
    cfg.dynamicSmemBytes = nr_smem(MP, NW);
    LaunchAttrs at(cfg, csize, false);
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, mx_gemm_narrow_kernel<MP, NW>, &cfg) != cudaSuccess || n < 1) {
      cudaGetLastError();
      n = max(1, num_sms_current() / csize - 1);
    }
    cache[dev][lc] = n;
  }
  return cache[dev][lc];
}

// Time of the narrow kernel in units of its k-block (0.45 us a CTA, the rate at which one SM's copies
// arrive from HBM; 0.84 us with gate and up rows), and the cluster size that gives it.  A CTA takes
// `turns` items of `kbs` k-blocks; the exchange of a turn runs beside the next turn's k-blocks, the last
// one after them.  Measured on 1 to 128 rows, 512 to 22016 x 1024 to 11008, clusters of 1 to 8: an
// exchange takes 5 + rows/16 (9/c + 1) k-blocks, e.g. 2.3 us for one row and 14 us for 128 in clusters
// of 4; clusters of 1 need none (a local one for the activation).
template <int MP, int NW>
inline double narrow_cost(const Epi& ep, int64_t K, int* csize, int* clusters) {
  const int64_t items = ((NW == 2 ? ep.F : ep.N) + 127) / 128 * ((ep.M + MP - 1) / MP), num_kb = (K + KB - 1) / KB;
  const double rows = (double)min64(ep.M, MP) / 16.0;
  double best = 1e300;
  for (int c = 1; c <= 8 && c <= num_kb; c *= 2) {
    const int n = narrow_clusters<MP, NW>(c);
    const double turns = (double)((items + n - 1) / n), kbs = (double)((num_kb + c - 1) / c);
    double x = c > 1 ? 5.0 + rows * (9.0 / c + 1.0) : (NW == 2 ? 5.0 + 2.0 * rows : 0.0);
    if (NW == 2) x *= 0.7;
    const double cost = (turns - 1) * (kbs > x ? kbs : x) + kbs + x + rows;
    if (cost < best) {
      best = cost;
      *csize = c;
      *clusters = (int)min64(items, n);
    }
  }
  return best;
}

template <int MP, int NW>
inline int launch_narrow(const Operand& a, const Operand& b, int64_t K, const Epi& ep, int64_t brows, bool early,
                         cudaStream_t st) {
  static bool done[64] = {false};
  int rc = mx::allow_smem(mx_gemm_narrow_kernel<MP, NW>, nr_smem(MP, NW), done, "ff_mxfp4_gemm");
  if (rc) return rc;
  CUtensorMap tw, tsw, tx, tsx;
  if ((rc = make_map_codes(&tw, b.q, brows, K, b.ld, 128))) return rc;
  if ((rc = make_map_sf(&tsw, b.s, brows, K))) return rc;
  if ((rc = make_map_codes(&tx, a.q, ep.M, K, a.ld, MP))) return rc;
  if ((rc = make_map_sf(&tsx, a.s, ep.M, K))) return rc;
  const int64_t tiles_w = ((NW == 2 ? ep.F : ep.N) + 127) / 128, tiles_x = (ep.M + MP - 1) / MP, items = tiles_w * tiles_x;
  FF_REQUIRE(items < ((int64_t)1 << 31), FF_ERR_UNSUPPORTED, "ff_mxfp4_gemm: too many tiles");
  const int64_t num_kb = (K + KB - 1) / KB;
  int csize, clusters;
  narrow_cost<MP, NW>(ep, K, &csize, &clusters);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)csize, (unsigned)clusters);
  cfg.blockDim = dim3(NR_THREADS);
  cfg.dynamicSmemBytes = nr_smem(MP, NW);
  cfg.stream = st;
  LaunchAttrs at(cfg, csize, early);
  FF_CUDA_TRY(cudaLaunchKernelEx(&cfg, mx_gemm_narrow_kernel<MP, NW>, tw, tsw, tx, tsx, (int)num_kb, (int)tiles_w, (int)tiles_x, ep),
              "ff_mxfp4_gemm launch");
  return check_launch("ff_mxfp4_gemm");
}

template <bool GATED>
inline int launch_pair(const Operand& a, const Operand& b, int64_t K, Epi ep, int64_t brows, int max_pairs, bool early,
                       cudaStream_t st) {
  static bool done[64] = {false};
  int rc = mx::allow_smem(mx_gemm_pair_kernel<GATED>, PR_SMEM, done, "ff_mxfp4_gemm");
  if (rc) return rc;
  CUtensorMap ta, tsa, tb, tsb, td, tb2;
  memset(&td, 0, sizeof(td));
  if ((rc = make_map_codes(&ta, a.q, ep.M, K, a.ld, 128))) return rc;
  if ((rc = make_map_sf(&tsa, a.s, ep.M, K))) return rc;
  if ((rc = make_map_codes(&tb, b.q, brows, K, b.ld, 128))) return rc;
  if ((rc = make_map_sf(&tsb, b.s, brows, K))) return rc;
  // whole 16-byte pieces only: a tile store clipped at an odd column was seen to write a zero behind it
  ep.tma_store = !GATED && !ep.out_f32 && ep.vec && ep.N % 8 == 0;
  if (ep.tma_store && (rc = make_map_out_bf16(&td, ep.D, ep.M, ep.N, ep.ldd, true))) return rc;
  const int tiles_m = (int)((ep.M + 255) / 256), tiles_n = (int)(GATED ? ep.F / 128 : (ep.N + 255) / 256);
  const int total = tiles_m * tiles_n, pairs = min(total, max_pairs), rest = total % pairs;
  const int split = !GATED && total > pairs && rest > 0 && 2 * rest <= pairs;
  tb2 = tb;
  if (split && (rc = make_map_codes(&tb2, b.q, brows, K, b.ld, 64))) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * pairs));
  cfg.blockDim = dim3(PR_THREADS);
  cfg.dynamicSmemBytes = PR_SMEM;
  cfg.stream = st;
  LaunchAttrs at(cfg, 2, early);
  FF_CUDA_TRY(cudaLaunchKernelEx(&cfg, mx_gemm_pair_kernel<GATED>, ta, tsa, tb, tsb, td, tb2, (int)((K + KB - 1) / KB),
                                 tiles_m, tiles_n, split, ep),
              "ff_mxfp4_gemm pair launch");
  return check_launch("ff_mxfp4_gemm (pair)");
}

template <int NW>
inline int launch_narrow_mp(const Operand& a, const Operand& b, int64_t K, const Epi& ep, int64_t brows, bool early,
                            cudaStream_t st) {
  if (ep.M <= 16) return launch_narrow<16, NW>(a, b, K, ep, brows, early, st);
  if (ep.M <= 32) return launch_narrow<32, NW>(a, b, K, ep, brows, early, st);
  // two 128-row accumulators and their partial sums leave no room for 128 rows of A
  if (NW == 2 || ep.M <= 64) return launch_narrow<64, NW>(a, b, K, ep, brows, early, st);
  return launch_narrow<128, 1>(a, b, K, ep, brows, early, st);
}

template <int NW>
inline double narrow_cost_mp(const Epi& ep, int64_t K) {
  int c, n;
  if (ep.M <= 16) return narrow_cost<16, NW>(ep, K, &c, &n);
  if (ep.M <= 32) return narrow_cost<32, NW>(ep, K, &c, &n);
  if (NW == 2 || ep.M <= 64) return narrow_cost<64, NW>(ep, K, &c, &n);
  return narrow_cost<128, 1>(ep, K, &c, &n);
}

// The product with whichever kernel is the faster.  Pair kernel, in the units of narrow_cost and beyond
// the narrow kernel's fixed time: 4 + 7/8 of a k-block per wave and k-block (0.385 us; 6 + 0.6 with gate and
// up rows).  Measured at both: 33 x 4096 x 11008 21 us narrow, 29 us pair; 128 x 512 x 11008 21 and 29;
// 129 x 4096 x 4096 33 and 18; 16 x 22016 x 4096 23 and 27; 64 x 22016 x 4096 27 and 27;
// 512 x 12288 x 4096 37 and 25 (each with about 6 us of an empty measurement).
template <int NW>
inline int launch_product(const Operand& a, const Operand& b, int64_t K, const Epi& ep, int64_t brows, bool early,
                          cudaStream_t st) {
  const int pairs = max_pairs_current();
  const int64_t tiles = (ep.M + 255) / 256 * (NW == 2 ? ep.F / 128 : (ep.N + 255) / 256), num_kb = (K + KB - 1) / KB;
  if (pairs > 0 && tiles < ((int64_t)1 << 31)) {
    const double waves = (double)((tiles + pairs - 1) / pairs);
    const double cost = NW == 2 ? 6.0 + 0.6 * waves * (double)num_kb : 4.0 + 0.875 * waves * (double)num_kb;
    if (ep.M > 512 || cost < narrow_cost_mp<NW>(ep, K))
      return launch_pair<NW == 2>(a, b, K, ep, brows, pairs, early, st);
  }
  return launch_narrow_mp<NW>(a, b, K, ep, brows, early, st);
}

inline int check_operand(const char* name, const char* which, const Operand& o, int64_t K) {
  FF_REQUIRE(o.q && o.s, FF_ERR_INVALID_ARG, "%s: null pointer (%s)", name, which);
  FF_REQUIRE(o.ld % 16 == 0 && o.ld >= (K + 31) / 32 * 16 && aligned(o.q, 16) && aligned(o.s, 16), FF_ERR_INVALID_ARG,
             "%s: %s needs 16-byte alignment and rows of a multiple of 16 bytes that hold every block (ld=%lld)", name, which,
             (long long)o.ld);
  return FF_OK;
}

// outputs and bias in whole elements
inline int check_out(const char* name, const void* D, int kind, const float* bias) {
  FF_REQUIRE(aligned(D, kind == FF_OUT_F32 ? 4 : 2) && aligned(bias, 4), FF_ERR_INVALID_ARG,
             "%s: an output or the bias is not aligned to its elements", name);
  return FF_OK;
}

}  // namespace mxg
}  // namespace ff

extern "C" int ff_mxfp4_gemm(const uint8_t* A, int64_t lda, const uint8_t* sA, const uint8_t* B, int64_t ldb,
                             const uint8_t* sB, const float* bias, void* D, int64_t ldd, int out_kind, int64_t M, int64_t N,
                             int64_t K, void* stream) {
  using namespace ff::mxg;
  FF_REQUIRE(M >= 0 && N >= 0 && K >= 1, FF_ERR_INVALID_ARG, "ff_mxfp4_gemm: M=%lld N=%lld K=%lld", (long long)M, (long long)N,
             (long long)K);
  FF_REQUIRE(out_kind == FF_OUT_F32 || out_kind == FF_OUT_BF16, FF_ERR_INVALID_ARG, "ff_mxfp4_gemm: bad out_kind %d", out_kind);
  if (M == 0 || N == 0) return FF_OK;
  FF_REQUIRE(D && ldd >= N, FF_ERR_INVALID_ARG, "ff_mxfp4_gemm: null output or ldd=%lld < N=%lld", (long long)ldd, (long long)N);
  FF_REQUIRE(M <= 65535 * 128 && N < ((int64_t)1 << 22) && K < ((int64_t)1 << 30), FF_ERR_UNSUPPORTED,
             "ff_mxfp4_gemm: dimension too large (M=%lld N=%lld K=%lld)", (long long)M, (long long)N, (long long)K);
  const Operand a{A, lda, sA}, b{B, ldb, sB};
  int rc;
  if ((rc = check_out("ff_mxfp4_gemm", D, out_kind, bias)) || (rc = check_operand("ff_mxfp4_gemm", "A", a, K)) || (rc = check_operand("ff_mxfp4_gemm", "B", b, K))) return rc;
  Epi ep{};
  ep.D = D;
  ep.ldd = ldd;
  ep.M = M;
  ep.N = N;
  ep.bias = bias;
  ep.out_f32 = out_kind == FF_OUT_F32;
  ep.vec = ff::aligned(D, 16) && (ldd * (ep.out_f32 ? 4 : 2)) % 16 == 0;
  return launch_product<1>(a, b, K, ep, N, false, ff::as_stream(stream));
}

extern "C" int ff_mxfp4_swiglu_gemm(const uint8_t* A, int64_t lda, const uint8_t* sA, const uint8_t* B, int64_t ldb,
                                    const uint8_t* sB, uint8_t* hq, int64_t ldh, uint8_t* hs, int64_t M, int64_t F, int64_t K,
                                    void* stream) {
  using namespace ff::mxg;
  FF_REQUIRE(M >= 0 && F >= 1 && K >= 1, FF_ERR_INVALID_ARG, "ff_mxfp4_swiglu_gemm: M=%lld F=%lld K=%lld", (long long)M,
             (long long)F, (long long)K);
  FF_REQUIRE(F % 128 == 0, FF_ERR_UNSUPPORTED, "ff_mxfp4_swiglu_gemm: F=%lld is not a multiple of 128", (long long)F);
  if (M == 0) return FF_OK;
  FF_REQUIRE(M <= 65535 * 128 && F < ((int64_t)1 << 21) && K < ((int64_t)1 << 30), FF_ERR_UNSUPPORTED,
             "ff_mxfp4_swiglu_gemm: dimension too large (M=%lld F=%lld K=%lld)", (long long)M, (long long)F, (long long)K);
  const Operand a{A, lda, sA}, b{B, ldb, sB}, h{hq, ldh, hs};
  int rc;
  if ((rc = check_operand("ff_mxfp4_swiglu_gemm", "A", a, K)) || (rc = check_operand("ff_mxfp4_swiglu_gemm", "B", b, K)) ||
      (rc = check_operand("ff_mxfp4_swiglu_gemm", "h", h, F)))
    return rc;
  Epi ep{};
  ep.M = M;
  ep.N = 2 * F;
  ep.F = F;
  ep.hq = hq;
  ep.hs = hs;
  ep.ldh = ldh;
  ep.hchunks = ff::mx::chunks_of(F);
  return launch_product<2>(a, b, K, ep, 2 * F, false, ff::as_stream(stream));
}

// Workspace of the fused calls: codes, then scales, of each intermediate matrix, 1024-byte aligned parts.
namespace ff {
namespace mxg {
inline int64_t part_bytes(int64_t rows, int64_t cols) {
  return (rows * ((cols + 31) / 32 * 16) + 1023) / 1024 * 1024 + mx::scale_bytes(rows, cols);
}
inline Operand part_at(uint8_t* ws, int64_t rows, int64_t cols) {
  const int64_t ld = (cols + 31) / 32 * 16;
  return Operand{ws, ld, ws + (rows * ld + 1023) / 1024 * 1024};
}
}  // namespace mxg
}  // namespace ff

extern "C" int64_t ff_mxfp4_linear_ws_bytes(int64_t M, int64_t K) {
  return M < 1 || K < 1 ? 0 : ff::mxg::part_bytes(M, K);
}

extern "C" int64_t ff_mxfp4_swiglu_mlp_ws_bytes(int64_t M, int64_t K, int64_t F) {
  return M < 1 || K < 1 || F < 1 ? 0 : ff::mxg::part_bytes(M, K) + ff::mxg::part_bytes(M, F);
}

extern "C" int ff_mxfp4_linear(const void* x, int dtype, int64_t ldx, const uint8_t* W, int64_t ldw, const uint8_t* sW,
                               const float* bias, void* D, int64_t ldd, int out_kind, int64_t M, int64_t N, int64_t K,
                               uint8_t* ws, int64_t ws_bytes, void* stream) {
  using namespace ff::mxg;
  FF_REQUIRE(M >= 0 && N >= 0 && K >= 1, FF_ERR_INVALID_ARG, "ff_mxfp4_linear: M=%lld N=%lld K=%lld", (long long)M, (long long)N,
             (long long)K);
  FF_REQUIRE(out_kind == FF_OUT_F32 || out_kind == FF_OUT_BF16, FF_ERR_INVALID_ARG, "ff_mxfp4_linear: bad out_kind %d", out_kind);
  if (M == 0 || N == 0) return FF_OK;
  FF_REQUIRE(D && ldd >= N, FF_ERR_INVALID_ARG, "ff_mxfp4_linear: null output or ldd=%lld < N=%lld", (long long)ldd, (long long)N);
  FF_REQUIRE(M <= 65535 * 128 && N < ((int64_t)1 << 22) && K < ((int64_t)1 << 30), FF_ERR_UNSUPPORTED,
             "ff_mxfp4_linear: dimension too large (M=%lld N=%lld K=%lld)", (long long)M, (long long)N, (long long)K);
  FF_REQUIRE(ws && ff::aligned(ws, 16) && ws_bytes >= part_bytes(M, K), FF_ERR_INVALID_ARG,
             "ff_mxfp4_linear: workspace of %lld bytes (16-byte aligned) needed, got %lld", (long long)part_bytes(M, K),
             (long long)ws_bytes);
  const Operand a = part_at(ws, M, K), b{W, ldw, sW};
  int rc;
  if ((rc = check_out("ff_mxfp4_linear", D, out_kind, bias)) || (rc = check_operand("ff_mxfp4_linear", "W", b, K))) return rc;
  rc = ff_mxfp4_quant(x, dtype, M, K, ldx, const_cast<uint8_t*>(a.q), a.ld, const_cast<uint8_t*>(a.s), nullptr, 0, nullptr, nullptr,
                      nullptr, stream);
  if (rc) return rc;
  Epi ep{};
  ep.D = D;
  ep.ldd = ldd;
  ep.M = M;
  ep.N = N;
  ep.bias = bias;
  ep.out_f32 = out_kind == FF_OUT_F32;
  ep.vec = ff::aligned(D, 16) && (ldd * (ep.out_f32 ? 4 : 2)) % 16 == 0;
  return launch_product<1>(a, b, K, ep, N, true, ff::as_stream(stream));
}

extern "C" int ff_mxfp4_swiglu_mlp(const void* x, int dtype, int64_t ldx, const uint8_t* GU, int64_t ldgu, const uint8_t* sGU,
                                   const uint8_t* W, int64_t ldw, const uint8_t* sW, void* D, int64_t ldd, int out_kind,
                                   int64_t M, int64_t K, int64_t F, int64_t N, uint8_t* ws, int64_t ws_bytes, void* stream) {
  using namespace ff::mxg;
  FF_REQUIRE(M >= 0 && N >= 0 && K >= 1 && F >= 1, FF_ERR_INVALID_ARG, "ff_mxfp4_swiglu_mlp: M=%lld K=%lld F=%lld N=%lld",
             (long long)M, (long long)K, (long long)F, (long long)N);
  FF_REQUIRE(F % 128 == 0, FF_ERR_UNSUPPORTED, "ff_mxfp4_swiglu_mlp: F=%lld is not a multiple of 128", (long long)F);
  FF_REQUIRE(out_kind == FF_OUT_F32 || out_kind == FF_OUT_BF16, FF_ERR_INVALID_ARG, "ff_mxfp4_swiglu_mlp: bad out_kind %d", out_kind);
  if (M == 0 || N == 0) return FF_OK;
  FF_REQUIRE(D && ldd >= N, FF_ERR_INVALID_ARG, "ff_mxfp4_swiglu_mlp: null output or ldd=%lld < N=%lld", (long long)ldd, (long long)N);
  FF_REQUIRE(M <= 65535 * 128 && N < ((int64_t)1 << 22) && F < ((int64_t)1 << 21) && K < ((int64_t)1 << 30), FF_ERR_UNSUPPORTED,
             "ff_mxfp4_swiglu_mlp: dimension too large (M=%lld K=%lld F=%lld N=%lld)", (long long)M, (long long)K, (long long)F,
             (long long)N);
  const int64_t need = part_bytes(M, K) + part_bytes(M, F);
  FF_REQUIRE(ws && ff::aligned(ws, 16) && ws_bytes >= need, FF_ERR_INVALID_ARG,
             "ff_mxfp4_swiglu_mlp: workspace of %lld bytes (16-byte aligned) needed, got %lld", (long long)need, (long long)ws_bytes);
  const Operand a = part_at(ws, M, K), h = part_at(ws + part_bytes(M, K), M, F), gu{GU, ldgu, sGU}, w{W, ldw, sW};
  int rc;
  if ((rc = check_out("ff_mxfp4_swiglu_mlp", D, out_kind, nullptr)) || (rc = check_operand("ff_mxfp4_swiglu_mlp", "gate_up", gu, K)) || (rc = check_operand("ff_mxfp4_swiglu_mlp", "down", w, F)))
    return rc;
  rc = ff_mxfp4_quant(x, dtype, M, K, ldx, const_cast<uint8_t*>(a.q), a.ld, const_cast<uint8_t*>(a.s), nullptr, 0, nullptr, nullptr,
                      nullptr, stream);
  if (rc) return rc;
  Epi eh{};
  eh.M = M;
  eh.N = 2 * F;
  eh.F = F;
  eh.hq = const_cast<uint8_t*>(h.q);
  eh.hs = const_cast<uint8_t*>(h.s);
  eh.ldh = h.ld;
  eh.hchunks = ff::mx::chunks_of(F);
  if ((rc = launch_product<2>(a, gu, K, eh, 2 * F, true, ff::as_stream(stream)))) return rc;
  Epi ep{};
  ep.D = D;
  ep.ldd = ldd;
  ep.M = M;
  ep.N = N;
  ep.out_f32 = out_kind == FF_OUT_F32;
  ep.vec = ff::aligned(D, 16) && (ldd * (ep.out_f32 ? 4 : 2)) % 16 == 0;
  return launch_product<1>(h, w, F, ep, N, true, ff::as_stream(stream));
}

// ---------------------------------------------------------------------------
// Training steps of the linear layer and of the gated block in one call each: the host's work of a small
// step is most of its time.  `saved` keeps what the backward call reads (transposed codes), `tmp` the rest.
// ---------------------------------------------------------------------------
namespace ff {
namespace mxg {
struct Arena {  // parts of a workspace, in order
  uint8_t* p;
  int64_t left;
  Operand take(int64_t rows, int64_t cols) {
    const Operand o = part_at(p, rows, cols);
    p += part_bytes(rows, cols);
    left -= part_bytes(rows, cols);
    return o;
  }
};
inline uint8_t* mut(const uint8_t* p) { return const_cast<uint8_t*>(p); }
// rows of x [R, C] and, with t, its columns
inline int quant_to(const void* x, int dt, int64_t R, int64_t C, int64_t ld, const Operand* r, const Operand* t, float* sums,
                    float* ws, void* stream) {
  return ff_mxfp4_quant(x, dt, R, C, ld, r ? mut(r->q) : nullptr, r ? r->ld : 0, r ? mut(r->s) : nullptr, t ? mut(t->q) : nullptr,
                        t ? t->ld : 0, t ? mut(t->s) : nullptr, sums, ws, stream);
}
// Launched early: the narrow kernel asks for B before it waits for the kernel ahead of it, so B is never
// that kernel's output (the weight is quantised first, the activations last; the backward products' B is
// saved).
inline int product(const Operand& a, const Operand& b, const float* bias, void* D, int kind, int64_t M, int64_t N, int64_t K,
                   void* stream) {
  Epi ep{};
  ep.D = D;
  ep.ldd = N;
  ep.M = M;
  ep.N = N;
  ep.bias = bias;
  ep.out_f32 = kind == FF_OUT_F32;
  ep.vec = aligned(D, 16) && (N * (ep.out_f32 ? 4 : 2)) % 16 == 0;
  return launch_product<1>(a, b, K, ep, N, true, as_stream(stream));
}
inline bool float_kind(int k) { return k == FF_OUT_F32 || k == FF_OUT_BF16; }
inline int check_dims(const char* name, int64_t M, int64_t N, int64_t K) {
  // each of them is a row count of some product
  FF_REQUIRE(M >= 1 && N >= 1 && K >= 1, FF_ERR_INVALID_ARG, "%s: M=%lld N=%lld K=%lld", name, (long long)M, (long long)N, (long long)K);
  FF_REQUIRE(M < ((int64_t)1 << 22) && N < ((int64_t)1 << 22) && K < ((int64_t)1 << 22), FF_ERR_UNSUPPORTED,
             "%s: dimension too large (M=%lld N=%lld K=%lld)", name, (long long)M, (long long)N, (long long)K);
  return FF_OK;
}
inline int check_ws(const char* name, const char* what, const void* p, int64_t have, int64_t need) {
  FF_REQUIRE(need == 0 || (p && aligned(p, 16) && have >= need), FF_ERR_INVALID_ARG,
             "%s: %s of %lld bytes (16-byte aligned) needed, got %lld", name, what, (long long)need, (long long)have);
  return FF_OK;
}
}  // namespace mxg
}  // namespace ff

extern "C" int ff_mxfp4_linear_train(const void* x, int x_dtype, int64_t ldx, const void* w, int w_dtype, int64_t ldw,
                                     const float* bias, void* y, int64_t M, int64_t N, int64_t K, int need_dx, int need_dw,
                                     uint8_t* tmp, int64_t tmp_bytes, uint8_t* saved, int64_t saved_bytes, void* stream) {
  using namespace ff::mxg;
  const char* name = "ff_mxfp4_linear_train";
  int rc;
  if ((rc = check_dims(name, M, N, K)) || (rc = check_ws(name, "tmp", tmp, tmp_bytes, part_bytes(M, K) + part_bytes(N, K))) ||
      (rc = check_ws(name, "saved", saved, saved_bytes, (need_dw ? part_bytes(K, M) : 0) + (need_dx ? part_bytes(K, N) : 0))) ||
      (rc = check_out(name, y, FF_OUT_BF16, bias)))
    return rc;
  FF_REQUIRE(y, FF_ERR_INVALID_ARG, "%s: null pointer", name);
  Arena t{tmp, tmp_bytes}, k{saved, saved_bytes};
  const Operand qx = t.take(M, K), qw = t.take(N, K);
  Operand xt{}, wt{};
  if (need_dw) xt = k.take(K, M);
  if (need_dx) wt = k.take(K, N);
  if ((rc = quant_to(w, w_dtype, N, K, ldw, &qw, need_dx ? &wt : nullptr, nullptr, nullptr, stream)) ||
      (rc = quant_to(x, x_dtype, M, K, ldx, &qx, need_dw ? &xt : nullptr, nullptr, nullptr, stream)))
    return rc;
  return product(qx, qw, bias, y, FF_OUT_BF16, M, N, K, stream);
}

extern "C" int ff_mxfp4_linear_bwd(const void* dy, int dtype, int64_t lddy, const uint8_t* saved, int64_t saved_bytes,
                                   int saved_dx, int saved_dw, void* dx, int dx_kind, void* dw, int dw_kind, float* db,
                                   int64_t M, int64_t N, int64_t K, uint8_t* tmp, int64_t tmp_bytes, void* stream) {
  using namespace ff::mxg;
  const char* name = "ff_mxfp4_linear_bwd";
  int rc;
  const bool cols = dw || db;
  const int64_t sums = db ? (ff_mxfp4_colsum_ws_elems(M, N) * 4 + 15) / 16 * 16 : 0;
  if ((rc = check_dims(name, M, N, K)) ||
      (rc = check_ws(name, "saved", saved, saved_bytes, (saved_dw ? part_bytes(K, M) : 0) + (saved_dx ? part_bytes(K, N) : 0))) ||
      (rc = check_ws(name, "tmp", tmp, tmp_bytes, (dx ? part_bytes(M, N) : 0) + (cols ? part_bytes(N, M) : 0) + sums)) ||
      (rc = check_out(name, dx, dx_kind, db)) || (rc = check_out(name, dw, dw_kind, nullptr)))
    return rc;
  FF_REQUIRE((!dx || (saved_dx && float_kind(dx_kind))) && (!dw || (saved_dw && float_kind(dw_kind))), FF_ERR_INVALID_ARG,
             "%s: a gradient whose operand was not saved, or a bad output kind", name);
  Arena k{mut(saved), saved_bytes}, t{tmp, tmp_bytes};
  Operand xt{}, wt{}, q{}, qt{};
  if (saved_dw) xt = k.take(K, M);
  if (saved_dx) wt = k.take(K, N);
  if (dx) q = t.take(M, N);
  if (cols) qt = t.take(N, M);
  if ((rc = quant_to(dy, dtype, M, N, lddy, dx ? &q : nullptr, cols ? &qt : nullptr, db, db ? reinterpret_cast<float*>(t.p) : nullptr,
                     stream)))
    return rc;
  if (dx && (rc = product(q, wt, nullptr, dx, dx_kind, M, K, N, stream))) return rc;
  if (dw && (rc = product(qt, xt, nullptr, dw, dw_kind, N, K, M, stream))) return rc;
  return FF_OK;
}

extern "C" int ff_mxfp4_swiglu_train(const void* x, int x_dtype, int64_t ldx, const void* wgu, int gu_dtype, int64_t ldgu,
                                     const void* wd, int d_dtype, int64_t ldd, void* gu, void* y, int64_t M, int64_t K,
                                     int64_t F, int64_t N, int need_dx, int need_dgu, int need_dd, uint8_t* tmp,
                                     int64_t tmp_bytes, uint8_t* saved, int64_t saved_bytes, void* stream) {
  using namespace ff::mxg;
  const char* name = "ff_mxfp4_swiglu_train";
  int rc;
  const bool back = need_dx || need_dgu;
  if ((rc = check_dims(name, M, N, K)) || (rc = check_dims(name, 2 * F, N, K)) ||
      (rc = check_ws(name, "tmp", tmp, tmp_bytes, part_bytes(M, K) + part_bytes(2 * F, K) + part_bytes(M, F) + part_bytes(N, F))) ||
      (rc = check_ws(name, "saved", saved, saved_bytes,
                     (need_dgu ? part_bytes(K, M) : 0) + (need_dx ? part_bytes(K, 2 * F) : 0) + (need_dd ? part_bytes(F, M) : 0) +
                         (back ? part_bytes(F, N) : 0))) ||
      (rc = check_out(name, y, FF_OUT_BF16, nullptr)))
    return rc;
  FF_REQUIRE(y && gu && ff::aligned(gu, 16), FF_ERR_INVALID_ARG, "%s: null pointer, or gu not 16-byte aligned", name);
  Arena t{tmp, tmp_bytes}, k{saved, saved_bytes};
  const Operand qx = t.take(M, K), qgu = t.take(2 * F, K), qh = t.take(M, F), qd = t.take(N, F);
  Operand xt{}, gut{}, ht{}, dt{};
  if (need_dgu) xt = k.take(K, M);
  if (need_dx) gut = k.take(K, 2 * F);
  if (need_dd) ht = k.take(F, M);
  if (back) dt = k.take(F, N);
  if ((rc = quant_to(wd, d_dtype, N, F, ldd, &qd, back ? &dt : nullptr, nullptr, nullptr, stream)) ||
      (rc = quant_to(wgu, gu_dtype, 2 * F, K, ldgu, &qgu, need_dx ? &gut : nullptr, nullptr, nullptr, stream)) ||
      (rc = quant_to(x, x_dtype, M, K, ldx, &qx, need_dgu ? &xt : nullptr, nullptr, nullptr, stream)) ||
      (rc = product(qx, qgu, nullptr, gu, FF_OUT_BF16, M, 2 * F, K, stream)) ||
      (rc = ff_mxfp4_swiglu_quant(gu, 2 * F, M, F, mut(qh.q), qh.ld, mut(qh.s), need_dd ? mut(ht.q) : nullptr, ht.ld,
                                  need_dd ? mut(ht.s) : nullptr, stream)))
    return rc;
  return product(qh, qd, nullptr, y, FF_OUT_BF16, M, N, F, stream);
}

extern "C" int ff_mxfp4_swiglu_bwd(const void* dy, int dtype, int64_t lddy, const void* gu, void* dh, const uint8_t* saved,
                                   int64_t saved_bytes, int need_dx, int need_dgu, int need_dd, void* dx, int dx_kind,
                                   void* dwgu, int gu_kind, void* dwd, int d_kind, int64_t M, int64_t K, int64_t F, int64_t N,
                                   uint8_t* tmp, int64_t tmp_bytes, void* stream) {
  using namespace ff::mxg;
  const char* name = "ff_mxfp4_swiglu_bwd";
  int rc;
  const bool back = need_dx || need_dgu;
  if ((rc = check_dims(name, M, N, K)) || (rc = check_dims(name, 2 * F, N, K)) ||
      (rc = check_ws(name, "saved", saved, saved_bytes,
                     (need_dgu ? part_bytes(K, M) : 0) + (need_dx ? part_bytes(K, 2 * F) : 0) + (need_dd ? part_bytes(F, M) : 0) +
                         (back ? part_bytes(F, N) : 0))) ||
      (rc = check_ws(name, "tmp", tmp, tmp_bytes,
                     (back ? part_bytes(M, N) : 0) + (need_dd ? part_bytes(N, M) : 0) + (need_dx ? part_bytes(M, 2 * F) : 0) +
                         (need_dgu ? part_bytes(2 * F, M) : 0))) ||
      (rc = check_out(name, dx, dx_kind, nullptr)) || (rc = check_out(name, dwgu, gu_kind, nullptr)) ||
      (rc = check_out(name, dwd, d_kind, nullptr)))
    return rc;
  FF_REQUIRE((!need_dx || (dx && float_kind(dx_kind))) && (!need_dgu || (dwgu && float_kind(gu_kind))) &&
                 (!need_dd || (dwd && float_kind(d_kind))) && (!back || (gu && dh && ff::aligned(gu, 16) && ff::aligned(dh, 16))),
             FF_ERR_INVALID_ARG, "%s: null pointer, bad output kind, or gu or dh not 16-byte aligned", name);
  Arena k{mut(saved), saved_bytes}, t{tmp, tmp_bytes};
  Operand xt{}, gut{}, ht{}, dt{}, q{}, qt{}, p{}, pt{};
  if (need_dgu) xt = k.take(K, M);
  if (need_dx) gut = k.take(K, 2 * F);
  if (need_dd) ht = k.take(F, M);
  if (back) dt = k.take(F, N);
  if (back) q = t.take(M, N);
  if (need_dd) qt = t.take(N, M);
  if (need_dx) p = t.take(M, 2 * F);
  if (need_dgu) pt = t.take(2 * F, M);
  if ((rc = quant_to(dy, dtype, M, N, lddy, back ? &q : nullptr, need_dd ? &qt : nullptr, nullptr, nullptr, stream))) return rc;
  if (need_dd && (rc = product(qt, ht, nullptr, dwd, d_kind, N, F, M, stream))) return rc;
  if (!back) return FF_OK;
  if ((rc = product(q, dt, nullptr, dh, FF_OUT_BF16, M, F, N, stream)) ||
      (rc = ff_mxfp4_swiglu_bwd_quant(dh, F, gu, 2 * F, M, F, need_dx ? mut(p.q) : nullptr, p.ld, need_dx ? mut(p.s) : nullptr,
                                      need_dgu ? mut(pt.q) : nullptr, pt.ld, need_dgu ? mut(pt.s) : nullptr, stream)))
    return rc;
  if (need_dx && (rc = product(p, gut, nullptr, dx, dx_kind, M, K, 2 * F, stream))) return rc;
  if (need_dgu && (rc = product(pt, xt, nullptr, dwgu, gu_kind, 2 * F, K, M, stream))) return rc;
  return FF_OK;
}
