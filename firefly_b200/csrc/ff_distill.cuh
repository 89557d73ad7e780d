// ff_distill.cuh — distillation loss from a teacher's top logits, and its gradient.
//
// Row r has student logits s_v (v < V), entries j < K of the teacher (token i_j, logit t_j; an entry
// with i_j < 0 or t_j = -inf is absent) and possibly a label y.  With temperature T:
//   p_j = exp(t_j/T) / sum over the row's entries,     or, given the teacher's own log-sum-exp,
//   p_j = exp(t_j/T - lse) with p_rest = 1 - sum p for the tokens outside the entries;
//   q_v = softmax(s/T)_v,  q_rest = sum of q_v over the tokens outside the entries
//   KD  = T^2 [ sum_j p_j (log p_j - log q_{i_j}) + p_rest (log p_rest - log q_rest) ]
//   L   = alpha KD + (1 - alpha) (logsumexp(s) - s_y)
//   dL/ds_v = alpha T (w q_v - sum_{j: i_j = v} p_j)   on the entries' tokens, w = sum p + p_rest,
//             alpha T q_v (w - p_rest / q_rest)         elsewhere (without lse: alpha T q_v),
//             + (1 - alpha) (softmax(s)_v - [v = y]).
// log q_rest and q_v / q_rest have the rest's own maximum as their reference where q_rest is below 2^-60 of the row.  Where
// the entries cover the vocabulary there is no rest term; where the student has all other tokens at -inf it is infinite,
// unless p_rest is below 1e-5, the rounding of 1 - sum p.  p_rest is not negative, so w is 1, or sum p where a rounded
// lse or a token given twice make that more than 1 or there is no rest term.
// A row whose label is ignore_index, or without labels a row without entries, counts nothing.
//
// One cluster of 1 to 8 CTAs per row, each holding its slice of the row in shared memory (bulk
// copies), so the logits are read once and the gradient is written once: the bound is HBM.  On a
// slice: the maximum; the entries' logits are gathered and their places overwritten by -inf (which
// makes the sum of the rest exact instead of 1 - sum q, and leaves each token's first entry as its
// owner, so a token that occurs twice is summed once); the sum of exp; one exchange of partial
// results between the CTAs; the gradient of all tokens, then the entries' own.  While the gradient is
// formed the next row's copies move into the parts of the slice that have been read, and a ninth warp
// works out the next row's entries.
// Maxima, sums and probabilities are fp32; the gradient is rounded once.
//
// Measured (a call's three launches): 16384 x 32000 bf16 (T = 2, labels, gradient) 438 us, its bytes 322 us at copy
// speed; 1500 x 131071 (clusters of four) 225 us, its bytes 120 us; 64 x 32000 fp32 without gradient 7 us.  Three rows at a time are
// in different phases on an SM, and neither the exponentials (half of the special-function unit's rate) nor the
// copies nor the stores bound it alone: leaving out either pass over the slice takes off about a quarter.  With
// the first version's separate phases, and exponentials of their own at both temperatures, 770 us; with 384 or
// 512 threads, or 32 KB slices, slower than with 256 and 64 KB.
#pragma once

#include "ff_gemm_i8.cuh"
#include "ff_mxfp4.cuh"

namespace ff {
namespace distill {

constexpr int THREADS = 256;  // and a warp for the teacher's entries
constexpr int WARPS = THREADS / 32;
static_assert(THREADS == 256, "bar_compute counts them");
constexpr int MAX_TOP = 4096;
constexpr int MAX_SMEM = 227 * 1024;
constexpr int COUNT_CTAS = FF_DISTILL_WS_ELEMS;
// a share below which the rest is summed relative to its own maximum: exponentials end at 2^-126, so a sum above this is
// complete to 2^-66 of itself per token
constexpr float kLittle = 8.673617379884035e-19f;  // 2^-60

struct Args {
  const void* logits;
  int64_t rows, V, ldl;
  const void* ids;
  const void* tlogits;
  const void* labels;
  const float* lse;
  int64_t ldi, ldt;
  int64_t ignore;
  int K, ids64, tdtype, labels64;
  float T, alpha;
  int mean;               // divide by the number of counted rows (`counts`)
  const int32_t* counts;  // COUNT_CTAS partial counts
  float* row_loss;        // [rows], or null
  void* grad;             // [rows, ldg], or null
  int64_t ldg;
  const float* upstream;  // null: 1; else a scalar, or one value per row
  int up_stride;
  const float* held;      // the scalar upstream whose gradient `grad` holds already, or null
  int slice;              // elements of a CTA's slice (a multiple of 128)
};

__device__ __forceinline__ int64_t load_index(const void* p, int64_t i, int is64) {
  return is64 ? __ldg(static_cast<const long long*>(p) + i) : (int64_t)__ldg(static_cast<const int*>(p) + i);
}
__device__ __forceinline__ float load_float(const void* p, int64_t i, int dt) {
  if (dt == FF_DTYPE_F32) return __ldg(static_cast<const float*>(p) + i);
  if (dt == FF_DTYPE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ float neg_inf() { return __uint_as_float(0xFF800000u); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));  // below 2^-126: 0
  return y;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <int DT>
struct Vec {  // 16 bytes of logits as packed pairs of floats
  static constexpr int N = DT == FF_DTYPE_F32 ? 4 : 8, P = N / 2;
  static __device__ __forceinline__ void get(uint4 w, f2 (&v)[P]) {
    const uint32_t q[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int k = 0; k < P; ++k) {
      if constexpr (DT == FF_DTYPE_F32) {
        v[k] = mk2(__uint_as_float(q[2 * k]), __uint_as_float(q[2 * k + 1]));
      } else if constexpr (DT == FF_DTYPE_BF16) {
        v[k] = unpack_bf16x2(q[k]);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&q[k]));
        v[k] = mk2(f.x, f.y);
      }
    }
  }
  static __device__ __forceinline__ uint4 put(const f2 (&v)[P]) {
    uint32_t q[4];
#pragma unroll
    for (int k = 0; k < P; ++k) {
      if constexpr (DT == FF_DTYPE_F32) {
        words2(v[k], q[2 * k], q[2 * k + 1]);
      } else if constexpr (DT == FF_DTYPE_BF16) {
        q[k] = pack_bf16x2(v[k]);
      } else {
        float a, b;
        un2(v[k], a, b);
        const __half2 h = __floats2half2_rn(a, b);
        q[k] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    return make_uint4(q[0], q[1], q[2], q[3]);
  }
  // running maximum of a 16-byte word, two values at a time in the type itself where it has 16 bits
  struct Max {
    float f;
    __nv_bfloat162 b;
    __half2 h;
    __device__ __forceinline__ Max() {
      f = __uint_as_float(0xFF800000u);
      b.x = b.y = __ushort_as_bfloat16(0xFF80);
      h.x = h.y = __ushort_as_half(0xFC00);
    }
    __device__ __forceinline__ void add(uint4 w) {
      if constexpr (DT == FF_DTYPE_F32) {
        f = fmaxf(f, fmaxf(fmaxf(__uint_as_float(w.x), __uint_as_float(w.y)), fmaxf(__uint_as_float(w.z), __uint_as_float(w.w))));
      } else if constexpr (DT == FF_DTYPE_BF16) {
        const __nv_bfloat162* p = reinterpret_cast<const __nv_bfloat162*>(&w);
        b = __hmax2(b, __hmax2(__hmax2(p[0], p[1]), __hmax2(p[2], p[3])));
      } else {
        const __half2* p = reinterpret_cast<const __half2*>(&w);
        h = __hmax2(h, __hmax2(__hmax2(p[0], p[1]), __hmax2(p[2], p[3])));
      }
    }
    __device__ __forceinline__ float value() const {
      if constexpr (DT == FF_DTYPE_F32) return f;
      else if constexpr (DT == FF_DTYPE_BF16) return fmaxf(__bfloat162float(b.x), __bfloat162float(b.y));
      else return fmaxf(__half2float(h.x), __half2float(h.y));
    }
  };
};
template <int DT>
__device__ __forceinline__ typename Elem<DT>::T from_f32(float v) {
  if constexpr (DT == FF_DTYPE_F32) return v;
  else if constexpr (DT == FF_DTYPE_BF16) return __float2bfloat16_rn(v);
  else return __float2half_rn(v);
}

// exp((s - m)/T) = 2^(s k - m k), k = log2(e)/T: one fused multiply-add with the rounded product m k, the same
// wherever m is the reference, so that its rounding cancels between q's numerator and denominator and in log q.
// From |m| k = 2^31 on (a slice or row of nothing but a mask of -1e10 or the type's lowest value) that rounding exceeds
// 2^6 and the product may overflow.  Two different fp32 logits lie 2^7 or more apart there in log2, so 2^(s k - m k) is 1
// for s = m and 0 below: a power of two in the place of k, with |m| k about 2^100, gives just that with exact products.
// At T = 2 and 4 (PW) the softmax at 1 is a power of this one, so its k counts (2^5 or more apart at T then).
constexpr float kLn2 = 0.6931471805599453f;
template <int PW>
struct Ref {
  float m, k;  // the reference (0 for -inf) and the true factor
  bool far;
  __device__ __forceinline__ Ref(float max_, float k_, float k_of_far) : m(max_ == neg_inf() ? 0.f : max_), k(k_) {
    far = fabsf(m) * k_of_far >= 2147483648.f;
  }
  static __device__ __forceinline__ Ref at_t(float max_, float kT, float k1) { return Ref(max_, kT, PW == 2 || PW == 4 ? k1 : kT); }
  static __device__ __forceinline__ Ref at_1(float max_, float k1) { return Ref(max_, k1, k1); }
  // factor and addend of the multiply-add
  __device__ __forceinline__ float mul() const {
    return far ? __uint_as_float(min(354u - (__float_as_uint(fabsf(m)) >> 23), 254u) << 23) : k;
  }
  __device__ __forceinline__ float add() const { return -__fmul_rn(m, mul()); }
  // one value's exponential in log2 and as (s - m)/T: the multiply-add's, and where that says no more than "far below"
  // (a masked label or entry has a finite loss), the difference
  __device__ __forceinline__ float log2_of(float s) const { return far ? (s - m) * k : fmaf(s, k, add()); }
  __device__ __forceinline__ float log_at(float s, float z) const {
    if (__builtin_expect(far || z == neg_inf(), 0)) return (s - m) * kLn2 * k;
    return z * kLn2;
  }
  __device__ __forceinline__ float log_of(float s) const { return log_at(s, log2_of(s)); }
  // log2 of the factor from sums relative to `o` to sums relative to this one: the difference of the two rounded
  // products (not contracted into one multiply-add, which would leave the rounding of m k in the sums: 2^-14 for
  // |m| / T of 1000)
  __device__ __forceinline__ float near_log2_from(const Ref& o) const { return __fsub_rn(__fmul_rn(o.m, k), __fmul_rn(m, k)); }
  __device__ __forceinline__ float log2_from(const Ref& o) const { return far || o.far ? (o.m - m) * k : near_log2_from(o); }
  __device__ __forceinline__ float log_from(const Ref& o) const {
    return far || o.far ? (o.m - m) * kLn2 * k : log2_from(o) * kLn2;
  }
};

// what a CTA tells the others about its slice
struct Part {
  float m;        // largest logit
  float sum;      // sum of exp((s - m)/T)
  float sum1;     // sum of exp(s - m)
  float rest;     // sum over the tokens outside the entries of exp((s - m)/T)
  float dot;      // sum over its entries of p (log p - (s - m)/T)
  float psum;     // sum of p over its entries
  float label;    // the label's logit where the label lies in the slice, else -inf
  float rest_m;   // what `rest` is relative to: m, or where that would leave next to nothing of it the largest logit of
                  // the rest; without any rest -inf, or 0 where tokens are there but all of them at -inf
};

// shared memory: control, then K entries of 20 bytes, then the slice
struct Ctrl {
  uint64_t bar;
  alignas(16) float red[6][WARPS];
  Part parts[2][8];
  float t_sum[2];        // of the teacher's entries (two rows in turn): the sum of p,
  int t_any[2];          // whether there is any,
  int label_in_top[2];   // whether the label's token is among them,
  int twice[2];          // whether a token of the slice occurs twice
  float label_logit;
};
__host__ __device__ constexpr int ctrl_bytes() { return (int)((sizeof(Ctrl) + 127) / 128 * 128); }
__host__ __device__ inline int entry_bytes(int K) { return (K * 20 + 127) / 128 * 128; }
__host__ __device__ inline int seen_bytes(int64_t slice) { return (int)(slice / 8 + 127) / 128 * 128; }

// How the softmax at temperature 1 is had beside the one at T (PW): 1: it is the same, or not needed;
// 2, 4: T is that, and exp(x) = exp(x / T)^T by squaring; 0: an exponential of its own.  The
// exponentials are what the kernel computes most of (the special-function unit takes 16 a cycle and SM:
// two per logit are 230 us of a 16384 x 32000 batch, four 460 us, its bytes 320 us).
template <int PW>
__device__ __forceinline__ f2 at_one(f2 x, f2 v, f2 k1, f2 nm1) {
  if constexpr (PW == 2) {
    return mul2(x, x);
  } else if constexpr (PW == 4) {
    x = mul2(x, x);
    return mul2(x, x);
  } else {
    float a, b;
    un2(fma2(v, k1, nm1), a, b);
    return mk2(ex2(a), ex2(b));
  }
}
__device__ __forceinline__ f2 ex2_2(f2 y) {
  float a, b;
  un2(y, a, b);
  return mk2(ex2(a), ex2(b));
}

// eight warps' values, in warp order
__device__ __forceinline__ float sum8(const float (&v)[WARPS]) {
  const float4 x = *reinterpret_cast<const float4*>(v), y = *reinterpret_cast<const float4*>(v + 4);
  return ((((((x.x + x.y) + x.z) + x.w) + y.x) + y.y) + y.z) + y.w;
}
__device__ __forceinline__ float max8(const float (&v)[WARPS]) {
  const float4 x = *reinterpret_cast<const float4*>(v), y = *reinterpret_cast<const float4*>(v + 4);
  return fmaxf(fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w)), fmaxf(fmaxf(y.x, y.y), fmaxf(y.z, y.w)));
}

// barrier of the compute warps (the teacher's warp takes no part)
__device__ __forceinline__ void bar_compute() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

template <int DT, int PW>
__global__ void __launch_bounds__(THREADS + 32, 3) distill_kernel(Args a) {
  using T = typename Elem<DT>::T;
  constexpr int N = Vec<DT>::N, P = Vec<DT>::P, ES = (int)sizeof(T);
  constexpr bool two = PW != 1;  // a second softmax at T = 1
  extern __shared__ __align__(128) uint8_t smem[];
  Ctrl& c = *reinterpret_cast<Ctrl*>(smem);
  // the entries, of two rows in turn: log p_j; place in this slice, -1: absent, -2: in another CTA's slice
  auto pos_of = [&](uint32_t b) { return reinterpret_cast<int*>(smem + ctrl_bytes()) + b * (uint32_t)a.K; };
  auto logp_of = [&](uint32_t b) { return reinterpret_cast<float*>(smem + ctrl_bytes()) + (2 + b) * (uint32_t)a.K; };
  float* e_s = reinterpret_cast<float*>(smem + ctrl_bytes()) + 4 * a.K;  // the student's logits of this slice's entries
  // a bit per token of the slice, all zero between rows: the teacher's warp finds repeated tokens with it
  uint32_t* seen = reinterpret_cast<uint32_t*>(smem + ctrl_bytes() + entry_bytes(a.K));
  uint8_t* data = smem + ctrl_bytes() + entry_bytes(a.K) + seen_bytes(a.slice);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int csize = (int)gridDim.x, rank = (int)blockIdx.x;  // the cluster spans grid x
  const uint32_t bar = gemm::smem_u32(&c.bar);

  if (a.held && __ldg(a.upstream) == __ldg(a.held)) return;  // every CTA of the grid alike

  if (tid == 0) {
    gemm::mbar_init(bar, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  for (int i = tid; i < a.slice / 32; i += THREADS + 32) seen[i] = 0u;
  float inv_count = 1.f;
  if (a.mean) {
    int n = 0;
    for (int i = lane; i < COUNT_CTAS; i += 32) n += __ldg(a.counts + i);
#pragma unroll
    for (int o = 16; o; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    inv_count = 1.f / (float)max(n, 1);
  }

  const float inv_t = 1.f / a.T, kT = 1.4426950408889634f * inv_t, k1 = 1.4426950408889634f;
  const int64_t v0 = (int64_t)rank * a.slice;
  const int len = (int)max64(0, min64(a.slice, a.V - v0)), bytes = len * ES;
  const uint4* w = reinterpret_cast<const uint4*>(data);

  // ---- where a row's slice lies: `mis` bytes into its first 16-byte word; the words [wb, we) are whole
  struct Geo {
    const T* src;
    int mis, head, wb, we, words;
  };
  auto geo = [&](int64_t r) {
    Geo g;
    g.src = static_cast<const T*>(a.logits) + r * a.ldl + v0;
    g.mis = (int)(reinterpret_cast<uintptr_t>(g.src) & 15u);
    g.head = min(bytes, (16 - g.mis) & 15);
    g.wb = (g.mis + g.head) / 16;
    g.we = g.wb + (bytes - g.head) / 16;
    g.words = (g.mis + bytes + 15) / 16;
    return g;
  };
  // thread 0: the copies of the words [from, to) of a row; the first call of a row (from 0) announces all
  auto issue = [&](const Geo& g, int from, int to) {
    if (from == 0) gemm::mbar_arrive_expect_tx(bar, (uint32_t)(g.we - g.wb) * 16u);
    const int b = max(from, g.wb), e = min(to, g.we);
    const uint8_t* src = reinterpret_cast<const uint8_t*>(g.src) - g.mis;
    for (int o = b; o < e; o += 1024)
      asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                       gemm::smem_u32(data) + o * 16),
                   "l"(src + (int64_t)o * 16), "r"(min(1024, e - o) * 16), "r"(bar)
                   : "memory");
  };
  // one warp: the ragged ends by plain loads, and -inf around them up to whole words
  auto edges = [&](const Geo& g) {
    T* d = reinterpret_cast<T*>(data + g.mis);
    const int nh = g.head / ES, t0 = ((g.we * 16) - g.mis) / ES;  // first element after the whole words
    if (lane < nh) d[lane] = g.src[lane];
    if (bytes > g.head && lane < len - t0) d[t0 + lane] = g.src[t0 + lane];
    if (lane < g.mis / ES) reinterpret_cast<T*>(data)[lane] = from_f32<DT>(neg_inf());
    if (lane < (g.words * 16 - g.mis - bytes) / ES) d[len + lane] = from_f32<DT>(neg_inf());
  };
  auto label_ok = [&](int64_t y) { return y >= 0 && y < a.V && y != a.ignore; };

  // ---- the teacher's warp: log p of a row's entries, their places, sum p
  auto teacher = [&](int64_t r, int64_t label, uint32_t b) {
    int* e_pos = pos_of(b);
    float* e_p = logp_of(b);
    float tm = neg_inf();
    bool bad = false, in_top = false, twice = false;
#pragma unroll 4
    for (int j = lane; j < a.K; j += 32) {
      const int64_t id = load_index(a.ids, r * a.ldi + j, a.ids64);
      const float t = load_float(a.tlogits, r * a.ldt + j, a.tdtype);
      const bool on = id >= 0 && id < a.V && t != neg_inf();
      bad |= id >= a.V;
      if (on) tm = t > tm || t != t ? t : tm;
      e_p[j] = on ? t : neg_inf();
      e_pos[j] = !on ? -1 : (id >= v0 && id < v0 + len) ? (int)(id - v0) : -2;
      in_top |= on && id == label;
    }
    const bool any = __any_sync(0xffffffffu, tm != neg_inf());
    tm = warp_max(tm);
    // a token's first entry in the slice owns it, later ones are marked; then the bits are taken back
    for (int j0 = 0; j0 < a.K; j0 += 32) {
      const int j = j0 + lane, pos = j < a.K ? e_pos[j] : -1;
      const bool first = __ffs(__match_any_sync(0xffffffffu, pos)) - 1 == lane;
      if (pos >= 0 && (!first || (atomicOr(seen + (pos >> 5), 1u << (pos & 31)) >> (pos & 31) & 1u))) {
        e_pos[j] = -3 - pos;
        twice = true;
      }
    }
    __syncwarp();
    for (int j = lane; j < a.K; j += 32)
      if (e_pos[j] >= 0) seen[e_pos[j] >> 5] = 0u;
    __syncwarp();
    float lz;
    if (a.lse) {
      tm = 0.f;
      lz = __ldg(a.lse + r);
    } else {
      float z = 0.f;
#pragma unroll 2
      for (int j = lane; j < a.K; j += 32)
        if (e_pos[j] != -1) z += expf((e_p[j] - tm) * inv_t);
      lz = logf(warp_sum(z));
    }
    float ps = 0.f;
#pragma unroll 2
    for (int j = lane; j < a.K; j += 32) {
      if (e_pos[j] == -1) continue;
      const float lp = (e_p[j] - tm) * inv_t - lz;
      e_p[j] = lp;
      ps += expf(lp);
    }
    ps = warp_sum(ps);
    in_top = __any_sync(0xffffffffu, in_top);
    twice = __any_sync(0xffffffffu, twice);
    if (bad) raise_status(FF_DEVICE_BADARG);
    if (lane == 0) {
      c.t_sum[b] = ps;
      c.t_any[b] = any;
      c.label_in_top[b] = in_top;
      c.twice[b] = twice;
    }
  };

  int64_t r = blockIdx.y;
  int64_t y = a.labels && r < a.rows ? load_index(a.labels, r, a.labels64) : 0;
  __syncthreads();
  if (csize > 1) gemm::cluster_sync_all();  // every CTA of the cluster runs before its memory is written to
  if (r < a.rows && (!a.labels || label_ok(y))) {
    if (warp == WARPS) {
      teacher(r, a.labels ? y : -1, 0);
    } else {
      const Geo g = geo(r);
      if (tid == 0) issue(g, 0, g.words);
      if (warp == 1) edges(g);
    }
  }
  __syncthreads();

  uint32_t phase = 0, par = 0, buf = 0;
  // small operands are asked for early, the loaded memory answers late: labels two rows ahead, entries
  // into L2 two rows ahead
  int64_t yn = a.labels && r + gridDim.y < a.rows ? load_index(a.labels, r + gridDim.y, a.labels64) : 0;
  auto entries_to_l2 = [&](int64_t row) {
    const int isz = a.ids64 ? 8 : 4, tsz = a.tdtype == FF_DTYPE_F32 ? 4 : 2;
    for (int j = lane * 32; j < a.K * isz; j += 1024)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(static_cast<const uint8_t*>(a.ids) + row * a.ldi * isz + j));
    for (int j = lane * 32; j < a.K * tsz; j += 1024)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(static_cast<const uint8_t*>(a.tlogits) + row * a.ldt * tsz + j));
    if (a.lse && lane == 0) asm volatile("prefetch.global.L2 [%0];" ::"l"(a.lse + row));
  };
  if (warp == WARPS && r + gridDim.y < a.rows) entries_to_l2(r + gridDim.y);
  for (; r < a.rows; buf ^= 1u) {
    // does the row count, and the next one of this cluster?  (the same answer in every thread of the cluster)
    const int64_t rn = r + gridDim.y;
    yn = a.labels && rn < a.rows ? load_index(a.labels, rn, a.labels64) : 0;
    const bool counted = !a.labels || label_ok(y);
    const bool ahead = rn < a.rows && (!a.labels || label_ok(yn));
    const int64_t label = a.labels && counted ? y : -1;
    bool live = counted;

    if (warp == WARPS) {
      if (!counted && y != a.ignore && lane == 0) raise_status(FF_DEVICE_BADARG);
      if (rn + gridDim.y < a.rows) entries_to_l2(rn + gridDim.y);
      if (ahead) teacher(rn, a.labels ? yn : -1, buf ^ 1u);
      __syncwarp();
      if (counted && csize > 1) gemm::cluster_sync_all();  // the compute warps' exchange
    } else {
      const Geo g = geo(r);
      Geo gn = geo(ahead ? rn : r);
      T* grow = a.grad ? static_cast<T*>(a.grad) + r * a.ldg + v0 : nullptr;
      T* s = reinterpret_cast<T*>(data + g.mis);  // the slice: element i is token v0 + i
      int given = 0;  // words of the next row whose copies have been issued
      bool under_way = false;
      if (counted) {
        int* e_pos = pos_of(buf);
        const float* e_p = logp_of(buf);
        // wait for the copies: past the limit the error is recorded, and the copies in flight are
        // waited for once more (bounded) so that none lands after the CTA
        if (!gemm::mbar_try_wait(bar, phase)) {
          const uint64_t t0 = globaltimer_ns(), limit = wait_limit_ns();
          while (!gemm::mbar_try_wait(bar, phase)) {
            if (globaltimer_ns() - t0 > limit) {
              raise_status(FF_DEVICE_TIMEOUT);
              gemm::drain_bar(bar, phase);
              break;
            }
          }
        }
        phase ^= 1u;

        // ---- largest logit; the entries' logits, whose places become -inf (their own values go into the
        // maximum, so it does not matter when another thread comes past)
        typename Vec<DT>::Max mx;
#pragma unroll 4
        for (int k = tid; k < g.words; k += THREADS) mx.add(w[k]);
        float m = mx.value();
        const bool twice = c.twice[buf] != 0;
        const bool here = label >= v0 && label < v0 + len;  // the label lies in this slice
        if (tid == 0 && !(here && c.label_in_top[buf])) c.label_logit = here ? Elem<DT>::to_f32(s[label - v0]) : neg_inf();
        if (twice) bar_compute();  // a place is read more than once: every read before it changes
        for (int j = tid; j < a.K; j += THREADS) {
          const int pos = e_pos[j];
          if (pos == -1 || pos == -2) continue;
          const float v = Elem<DT>::to_f32(s[pos >= 0 ? pos : -3 - pos]);
          e_s[j] = v;
          m = fmaxf(m, v);
          if (here && pos == (int)(label - v0)) c.label_logit = v;
          if (pos >= 0 && !twice) s[pos] = from_f32<DT>(neg_inf());
        }
        if (twice) {
          bar_compute();
          for (int j = tid; j < a.K; j += THREADS)
            if (e_pos[j] >= 0) s[e_pos[j]] = from_f32<DT>(neg_inf());
        }
        m = warp_max(m);
        if (lane == 0) c.red[0][warp] = m;
        bar_compute();
        m = max8(c.red[0]);
        const auto rT = Ref<PW>::at_t(m, kT, k1), r1 = Ref<PW>::at_1(m, k1);  // a slice of -inf sums to 0
        float sum = 0.f, sum1 = 0.f, rest = 0.f, dot = 0.f, psum = 0.f;
        for (int j = tid; j < a.K; j += THREADS) {
          const int pos = e_pos[j];
          if (pos == -1 || pos == -2) continue;
          const float z = rT.log2_of(e_s[j]), p = expf(e_p[j]);
          if (p > 0.f) dot += p * (e_p[j] - rT.log_at(e_s[j], z));
          else if (p != p) dot = p;
          psum += p;
          if (pos >= 0) {
            sum += ex2(z);
            if (two) sum1 += ex2(r1.log2_of(e_s[j]));
          }
        }
        // ---- sums of exp over the tokens outside the entries
        f2 acc = splat(0.f), acc1 = splat(0.f);
        {
          const f2 kT2 = splat(rT.mul()), nT2 = splat(rT.add()), k12 = splat(r1.mul()), n12 = splat(r1.add());
#pragma unroll 2
          for (int k = tid; k < g.words; k += THREADS) {
            f2 v[P];
            Vec<DT>::get(w[k], v);
#pragma unroll
            for (int e = 0; e < P; ++e) {
              const f2 x = ex2_2(fma2(v[e], kT2, nT2));
              acc = add2(acc, x);
              if (two) acc1 = add2(acc1, at_one<PW>(x, v[e], k12, n12));
            }
          }
          float p, q;
          un2(acc, p, q);
          rest = p + q;
          un2(acc1, p, q);
          sum1 += p + q;
        }
        sum += rest;
        // sums over the CTA: only those that are not zero throughout
        const bool more = warp * 32 < a.K;  // this warp has entries
        sum = warp_sum(sum);
        if (two) sum1 = warp_sum(sum1);
        if (a.lse) rest = warp_sum(rest);
        if (more) {
          dot = warp_sum(dot);
          psum = warp_sum(psum);
        }
        if (lane == 0) {
          c.red[1][warp] = sum;
          c.red[2][warp] = sum1;
          c.red[3][warp] = rest;
          c.red[4][warp] = dot;
          c.red[5][warp] = psum;
        }
        if (!grow) gemm::fence_proxy_async_smem();
        bar_compute();
        float low = m;
        rest = a.lse ? sum8(c.red[3]) : 0.f;
        if (a.lse && rest < kLittle) {  // the same in every thread of the CTA
          // The rest lies so far below m that its own exponentials are lost (or there is none): its sum once more,
          // relative to its own maximum.
          typename Vec<DT>::Max mr;
          for (int k = tid; k < g.words; k += THREADS) mr.add(w[k]);
          low = warp_max(mr.value());
          if (lane == 0) c.red[0][warp] = low;
          bar_compute();
          low = max8(c.red[0]);
          const auto rr = Ref<PW>::at_t(low, kT, k1);
          rest = 0.f;
          if (low != neg_inf()) {
            f2 ar = splat(0.f);
            for (int k = tid; k < g.words; k += THREADS) {
              f2 v[P];
              Vec<DT>::get(w[k], v);
#pragma unroll
              for (int e = 0; e < P; ++e) ar = add2(ar, ex2_2(fma2(v[e], splat(rr.mul()), splat(rr.add()))));
            }
            float p, q;
            un2(ar, p, q);
            rest = p + q;
          } else {  // how many of the slice's tokens are entries
            for (int j = tid; j < a.K; j += THREADS) rest += e_pos[j] >= 0 ? 1.f : 0.f;
          }
          rest = warp_sum(rest);
          if (lane == 0) c.red[3][warp] = rest;
          if (!grow) gemm::fence_proxy_async_smem();
          bar_compute();
          rest = sum8(c.red[3]);
          if (low == neg_inf()) {
            if (rest < (float)len) low = 0.f;  // tokens at -inf
            rest = 0.f;
          }
        }
        if (!grow && ahead) {  // the slice has been read for the last time
          if (tid == 0) issue(gn, 0, gn.words);
          under_way = true;
        }
        const Part mine = Part{m, sum8(c.red[1]), two ? sum8(c.red[2]) : 0.f, rest, sum8(c.red[4]),
                               sum8(c.red[5]), c.label_logit, low};
        Part all = mine;
        if (csize > 1) {
          if (tid < csize * 8) {  // word tid % 8 of this CTA's part to CTA tid / 8
            const uint32_t dst = gemm::mapa_shared(gemm::smem_u32(&c.parts[par][rank]) + (tid & 7) * 4, (uint32_t)(tid >> 3));
            const float word = (tid & 7) == 0 ? mine.m : (tid & 7) == 1 ? mine.sum : (tid & 7) == 2 ? mine.sum1
                               : (tid & 7) == 3 ? mine.rest : (tid & 7) == 4 ? mine.dot : (tid & 7) == 5 ? mine.psum
                               : (tid & 7) == 6 ? mine.label : mine.rest_m;
            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst), "f"(word) : "memory");
          }
          __syncwarp();
          gemm::cluster_sync_all();
          all = c.parts[par][0];
          bool odd = false;  // references that are far, or a rest with one of its own
          for (int k = 0; k < csize; ++k) {
            const float qm = c.parts[par][k].m;
            all.m = fmaxf(all.m, qm);
            odd |= Ref<PW>::at_t(qm, kT, k1).far || (PW == 0 && Ref<PW>::at_1(qm, k1).far) || (a.lse && c.parts[par][k].rest_m != qm);
          }
          const auto RT = Ref<PW>::at_t(all.m, kT, k1), R1 = Ref<PW>::at_1(all.m, k1);
          all.sum = all.sum1 = all.rest = all.dot = all.psum = 0.f;
          all.label = neg_inf();
          for (int k = 0; k < csize; ++k) {
            const Part q = c.parts[par][k];
            const bool any = q.m != neg_inf();
            auto o = Ref<PW>::at_t(q.m, kT, k1), o1 = Ref<PW>::at_1(q.m, k1);
            float d = any ? RT.near_log2_from(o) : 0.f, d1 = any ? R1.near_log2_from(o1) : 0.f, dl = d * kLn2;
            if (odd && any) {
              d = RT.log2_from(o);
              d1 = R1.log2_from(o1);
              dl = RT.log_from(o);
            }
            const float f = ex2(d);
            float rest_q = q.rest * f;
            if (odd && q.rest_m != q.m) rest_q = q.rest > 0.f ? q.rest * ex2(RT.log2_from(Ref<PW>::at_t(q.rest_m, kT, k1))) : 0.f;
            all.sum += q.sum * f;
            if (two) all.sum1 += q.sum1 * ex2(d1);
            all.rest += rest_q;
            all.dot += q.psum != 0.f || q.dot != 0.f ? q.dot - q.psum * dl : 0.f;
            all.psum += q.psum;
            all.label = fmaxf(all.label, q.label);
          }
          par ^= 1u;
        }
        const auto RT = Ref<PW>::at_t(all.m, kT, k1), R1 = Ref<PW>::at_1(all.m, k1);
        const float sum1_all = two ? all.sum1 : all.sum;
        const bool has = c.t_any[buf] != 0;
        if (!a.labels) live = has;
        float p_rest = a.lse && has ? fmaxf(1.f - c.t_sum[buf], 0.f) : 0.f;
        // ---- the rest bucket: q_rest, or where that is next to nothing its logarithm from the rest's own reference
        float q_rest = 0.f, rest_m = neg_inf(), rest_sum = 0.f;
        bool little = false;
        if (a.lse) {
          if (csize == 1 && low != m && rest > 0.f) all.rest = rest * ex2(RT.log2_from(Ref<PW>::at_t(low, kT, k1)));
          q_rest = all.rest / all.sum;
          little = q_rest < kLittle;  // (not for a NaN)
        }
        if (little) {
          bool other = low != neg_inf();  // tokens outside the entries
          rest_m = low;
          rest_sum = rest;
          if (csize > 1) {
            const Part* q = c.parts[par ^ 1u];
            rest_m = neg_inf();
            rest_sum = 0.f;
            for (int k = 0; k < csize; ++k) {
              other |= q[k].rest_m != neg_inf();
              if (q[k].rest > 0.f) rest_m = fmaxf(rest_m, q[k].rest_m);
            }
            const auto rr = Ref<PW>::at_t(rest_m, kT, k1);
            for (int k = 0; k < csize; ++k)
              if (q[k].rest > 0.f) rest_sum += q[k].rest * ex2(rr.log2_from(Ref<PW>::at_t(q[k].rest_m, kT, k1)));
          }
          // no other token: no bucket; none that the student can choose: 1 - sum p may be rounding alone
          if (!other || (rest_sum == 0.f && p_rest < 1e-5f)) p_rest = 0.f;
        }
        // ---- the loss
        if (a.row_loss && rank == 0 && tid == 0) {
          float kd = 0.f, ce = 0.f;
          if (has) {
            kd = all.dot + all.psum * logf(all.sum);
            if (p_rest > 0.f) {
              float lq = logf(q_rest);
              if (little) lq = rest_sum > 0.f ? RT.log_from(Ref<PW>::at_t(rest_m, kT, k1)) + (logf(rest_sum) - logf(all.sum)) : neg_inf();
              kd += p_rest * (logf(p_rest) - lq);
            }
            kd *= a.T * a.T;
          }
          if (label >= 0 && a.alpha != 1.f) ce = logf(sum1_all) - (two ? R1 : RT).log_of(all.label);
          a.row_loss[r] = live ? (a.alpha != 0.f ? a.alpha * kd : 0.f) + (a.alpha != 1.f ? (1.f - a.alpha) * ce : 0.f) : 0.f;
        }
        // ---- the gradient, half the slice at a time; the next row's copies follow into each
        // half as it has been read
        if (grow && live) {
          const float up = a.upstream ? __ldg(a.upstream + r * a.up_stride) * inv_count : inv_count;
          const float fk = has ? up * a.alpha * a.T : 0.f, f1 = label >= 0 ? up * (1.f - a.alpha) : 0.f;
          // log sum exp(s/T) stands in the loss with the weight sum p + p_rest (1 with a rest term)
          const float mass = a.lse && p_rest == 0.f ? c.t_sum[buf] : 1.f;
          const float gq = mass * fk / all.sum, g1 = f1 / sum1_all;  // factors of exp(..) for q and the softmax at 1
          // Outside the entries: q (1 - p_rest / q_rest).  With next to no q there, q itself is nothing beside
          // p_rest q / q_rest, and that is formed from the rest's own reference; so is then what the softmax at 1
          // takes from the same exponentials.
          const bool own = little && p_rest > 0.f && rest_sum > 0.f;
          const auto GT = own ? Ref<PW>::at_t(rest_m, kT, k1) : RT;
          const float gr = own ? -(fk * p_rest / rest_sum) : p_rest > 0.f && q_rest > 0.f ? gq * (1.f - p_rest / q_rest) : gq;
          const float g1r = !own || PW == 0 ? g1
                            : g1 * ex2(PW == 1 ? RT.log2_from(GT) : R1.log2_from(Ref<PW>::at_1(rest_m, k1)));
          const bool vec = (reinterpret_cast<uintptr_t>(grow) & 15u) == (uint32_t)g.mis;
          const f2 kT2 = splat(GT.mul()), nT2 = splat(GT.add()), k12 = splat(R1.mul()), n12 = splat(R1.add()),
                   gr2 = splat(two ? gr : gr + g1r), g12 = splat(g1r);
          const int step = (max(g.words, gn.words) + 2 * THREADS - 1) / (2 * THREADS) * THREADS;
          uint4* gw = reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(grow) - g.mis);  // word k of the slice
          auto grad_word = [&](int k) {
            f2 v[P], gv[P];
            Vec<DT>::get(w[k], v);
#pragma unroll
            for (int e = 0; e < P; ++e) {
              const f2 x = ex2_2(fma2(v[e], kT2, nT2));
              gv[e] = mul2(gr2, x);
              if (two) gv[e] = fma2(g12, at_one<PW>(x, v[e], k12, n12), gv[e]);
            }
            return Vec<DT>::put(gv);
          };
          auto edge_word = [&](int k) {  // element by element: a word that the slice does not fill, or another alignment
            const uint4 q = grad_word(k);
            const T* e = reinterpret_cast<const T*>(&q);
            const int i0 = k * N - g.mis / ES;
#pragma unroll
            for (int x = 0; x < N; ++x)
              if (i0 + x >= 0 && i0 + x < len) grow[i0 + x] = e[x];
          };
#pragma unroll 1
          for (int w0 = 0; w0 < g.words; w0 += step) {
            const int w1 = min(g.words, w0 + step);
            if (vec) {
#pragma unroll 2
              for (int k = max(w0, g.wb) + tid; k < min(w1, g.we); k += THREADS) __stcs(gw + k, grad_word(k));
              if (tid == 0 && w0 == 0 && g.wb > 0) edge_word(0);
              if (tid == 32 && w1 == g.words && g.words > g.we && (g.words > 1 || g.wb == 0)) edge_word(g.words - 1);
            } else {
#pragma unroll 1
              for (int k = w0 + tid; k < w1; k += THREADS) edge_word(k);
            }
            gemm::fence_proxy_async_smem();
            bar_compute();
            if (ahead) {
              const int to = w0 + step < g.words ? w0 + step : gn.words;
              if (tid == 0) issue(gn, given, to);
              given = to;
              under_way = true;
            }
          }
          if (g.words == 0) bar_compute();
          // the entries' and the label's own values come after the tokens' (the barrier above)
          for (int j = tid; j < a.K; j += THREADS) {
            const int pos = e_pos[j];
            if (pos < 0) continue;
            float p = expf(e_p[j]);
            if (twice) {  // the token's entries in order
              p = 0.f;
              for (int x = 0; x < a.K; ++x)
                if (e_pos[x] == pos || e_pos[x] == -3 - pos) p += expf(e_p[x]);
            }
            float gv = gq * ex2(RT.log2_of(e_s[j])) - fk * p;
            if (f1 != 0.f) gv += g1 * ex2((two ? R1 : RT).log2_of(e_s[j])) - (v0 + pos == label ? f1 : 0.f);
            grow[pos] = from_f32<DT>(gv);
          }
          if (tid == 0 && label >= v0 && label < v0 + len && !c.label_in_top[buf]) {
            const float x = ex2(GT.log2_of(c.label_logit));
            grow[label - v0] = from_f32<DT>((two ? gr * x + g1 * ex2(R1.log2_of(c.label_logit)) : (gr + g1r) * x) - f1);
          }
        }
      }
      if (!live) {
        if (a.row_loss && rank == 0 && tid == 0) a.row_loss[r] = 0.f;
        if (grow) {  // zeros: single elements up to a 16-byte boundary, then whole words
          const int h0 = min(len, (int)((16u - (reinterpret_cast<uintptr_t>(grow) & 15u)) & 15u) / ES), nw = (len - h0) / N;
          for (int k = tid; k < nw; k += THREADS) __stcs(reinterpret_cast<uint4*>(grow + h0) + k, make_uint4(0, 0, 0, 0));
          if (tid < h0) grow[tid] = from_f32<DT>(0.f);
          if (tid < len - h0 - nw * N) grow[h0 + nw * N + tid] = from_f32<DT>(0.f);
        }
      }
      if (ahead) {
        if (!under_way) {  // this row's slice is not needed any more
          gemm::fence_proxy_async_smem();
          bar_compute();
          if (tid == 0) issue(gn, 0, gn.words);
        }
        if (warp == 1) edges(gn);
      }
    }
    r = rn;
    y = yn;
    __syncthreads();  // the next row's entries and edges are there
  }
}

// rows that count, one partial count per CTA
__global__ void __launch_bounds__(256) distill_count_kernel(Args a, int32_t* counts) {
  __shared__ int tot;
  if (threadIdx.x == 0) tot = 0;
  __syncthreads();
  int n = 0;
  if (a.labels) {
    for (int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x; r < a.rows; r += (int64_t)gridDim.x * 256) {
      const int64_t y = load_index(a.labels, r, a.labels64);
      n += y >= 0 && y < a.V && y != a.ignore;
    }
  } else {  // a warp per row, until an entry is found
    const int lane = threadIdx.x & 31;
    for (int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); r < a.rows; r += (int64_t)gridDim.x * 8) {
      bool any = false;
      for (int j = lane; j - lane < a.K && !any; j += 32) {
        bool on = false;
        if (j < a.K) {
          const int64_t id = load_index(a.ids, r * a.ldi + j, a.ids64);
          on = id >= 0 && id < a.V && load_float(a.tlogits, r * a.ldt + j, a.tdtype) != neg_inf();
        }
        any = __any_sync(0xffffffffu, on);
      }
      n += any && lane == 0;
    }
  }
  if (n) atomicAdd(&tot, n);  // whole numbers: any order
  __syncthreads();
  if (threadIdx.x == 0) counts[blockIdx.x] = tot;
}

// the rows' losses added in a fixed order (fp64), divided by the number that count
__global__ void __launch_bounds__(1024) distill_finish_kernel(const float* row_loss, int64_t rows, const int32_t* counts,
                                                              float* loss, float* held) {
  __shared__ double part[32];
  double s = 0.0;
  for (int64_t r = threadIdx.x; r < rows; r += 1024) s += (double)row_loss[r];
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    double t = 0.0;
    for (int k = 0; k < 32; ++k) t += part[k];
    if (counts) {
      int n = 0;
      for (int i = 0; i < COUNT_CTAS; ++i) n += counts[i];
      t /= (double)max(n, 1);
    }
    loss[0] = (float)t;
    if (held) held[0] = 1.f;
  }
}
// the gradient is its caller's from here on: no upstream is equal to this
__global__ void distill_released_kernel(float* held) { held[0] = __uint_as_float(0x7FC00000u); }

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
// CTAs per row and elements of a slice: slices of about 70 KB leave three CTAs on an SM, whose
// copies and arithmetic overlap; with few rows the row is cut further, so that every SM has work.
inline bool plan(int64_t rows, int64_t V, int K, int es, int nsm, int* csize, int* slice, int* smem) {
  auto cut = [&](int c) { return ((V + c - 1) / c + 127) / 128 * 128; };
  const int fixed = ctrl_bytes() + entry_bytes(K) + 32;
  auto all = [&](int c) { return cut(c) * es + fixed + seen_bytes(cut(c)); };
  int c = 1;
  while (c < 8 && all(c) > 75 * 1024) c *= 2;
  while (c < 8 && rows * c * 2 <= 2 * nsm && cut(2 * c) * es >= 4096) c *= 2;
  const int64_t bytes = all(c);
  if (bytes > MAX_SMEM) return false;
  *csize = c;
  *slice = (int)cut(c);
  *smem = (int)bytes;
  return true;
}

template <int DT, int PW>
inline int launch(Args& a, cudaStream_t st, const char* name) {
  int c, smem;
  FF_REQUIRE(plan(a.rows, a.V, a.K, dtype_size(DT), gemm::num_sms_current(), &c, &a.slice, &smem), FF_ERR_UNSUPPORTED,
             "%s: a row of %lld logits with %d entries does not fit", name, (long long)a.V, a.K);
  static bool done[64] = {false};
  int rc = mx::allow_smem(distill_kernel<DT, PW>, MAX_SMEM, done, name);
  if (rc) return rc;
  // shared memory in three sizes (three, two or one CTA per SM), so that the number of clusters that
  // run at once is known: a persistent grid larger than that would take a second turn
  const int size = smem <= 75 * 1024 ? 0 : smem <= 113 * 1024 ? 1 : 2, lc = c == 1 ? 0 : c == 2 ? 1 : c == 4 ? 2 : 3;
  static const int bytes[3] = {75 * 1024, 113 * 1024, MAX_SMEM};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)c, 1);
  cfg.blockDim = dim3(THREADS + 32);
  cfg.dynamicSmemBytes = (size_t)bytes[size];
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)c;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  static int resident[64][3][4] = {};
  int dev = 0;
  FF_CUDA_TRY(cudaGetDevice(&dev), name);
  int n = dev < 64 ? resident[dev][size][lc] : 0;
  if (n == 0) {
    if (cudaOccupancyMaxActiveClusters(&n, distill_kernel<DT, PW>, &cfg) != cudaSuccess || n < 1) {
      cudaGetLastError();
      n = max(1, gemm::num_sms_current() / c);
    }
    if (dev < 64) resident[dev][size][lc] = n;
  }
  cfg.gridDim = dim3((unsigned)c, (unsigned)min64(a.rows, n));
  FF_CUDA_TRY(cudaLaunchKernelEx(&cfg, distill_kernel<DT, PW>, a), name);
  return check_launch(name);
}

template <int DT>
inline int launch_pw(Args& a, cudaStream_t st, const char* name) {
  if (a.labels == nullptr || a.T == 1.f || a.alpha == 1.f) return launch<DT, 1>(a, st, name);
  return a.T == 2.f ? launch<DT, 2>(a, st, name) : a.T == 4.f ? launch<DT, 4>(a, st, name) : launch<DT, 0>(a, st, name);
}
inline int launch_dt(Args& a, int dtype, cudaStream_t st, const char* name) {
  return dtype == FF_DTYPE_F32    ? launch_pw<FF_DTYPE_F32>(a, st, name)
         : dtype == FF_DTYPE_BF16 ? launch_pw<FF_DTYPE_BF16>(a, st, name)
                                  : launch_pw<FF_DTYPE_F16>(a, st, name);
}

inline int fill(const char* name, const FfDistillRows* in, Args* a) {
  FF_REQUIRE(in, FF_ERR_INVALID_ARG, "%s: null pointer", name);
  FF_REQUIRE(in->rows >= 0 && in->vocab >= 1 && in->top >= 1, FF_ERR_INVALID_ARG, "%s: rows=%lld vocab=%lld top=%lld", name,
             (long long)in->rows, (long long)in->vocab, (long long)in->top);
  FF_REQUIRE(in->top <= MAX_TOP, FF_ERR_UNSUPPORTED, "%s: %lld entries per row (at most %d)", name, (long long)in->top, MAX_TOP);
  FF_REQUIRE(in->rows < ((int64_t)1 << 31) && in->vocab < ((int64_t)1 << 30), FF_ERR_UNSUPPORTED, "%s: rows=%lld vocab=%lld too large",
             name, (long long)in->rows, (long long)in->vocab);
  FF_REQUIRE(in->dtype >= FF_DTYPE_F32 && in->dtype <= FF_DTYPE_F16 && in->teacher_dtype >= FF_DTYPE_F32 &&
                 in->teacher_dtype <= FF_DTYPE_F16,
             FF_ERR_INVALID_ARG, "%s: bad dtype %d or teacher dtype %d", name, in->dtype, in->teacher_dtype);
  FF_REQUIRE(in->ld_logits >= in->vocab && in->ld_ids >= in->top && in->ld_teacher >= in->top, FF_ERR_INVALID_ARG,
             "%s: bad leading dims", name);
  FF_REQUIRE(in->temperature > 0.f && in->temperature < 1e30f && in->alpha >= 0.f && in->alpha <= 1.f, FF_ERR_INVALID_ARG,
             "%s: temperature=%g (positive), alpha=%g (0 to 1)", name, in->temperature, in->alpha);
  if (in->rows > 0)
    FF_REQUIRE(in->logits && in->ids && in->teacher_logits && aligned(in->logits, dtype_size(in->dtype)) &&
                   aligned(in->ids, in->ids_64 ? 8 : 4) && aligned(in->teacher_logits, dtype_size(in->teacher_dtype)) &&
                   aligned(in->labels, in->labels_64 ? 8 : 4) && aligned(in->teacher_lse, 4),
               FF_ERR_INVALID_ARG, "%s: null or unaligned pointer", name);
  *a = Args{};
  a->logits = in->logits;
  a->rows = in->rows;
  a->V = in->vocab;
  a->ldl = in->ld_logits;
  a->ids = in->ids;
  a->tlogits = in->teacher_logits;
  a->labels = in->labels;
  a->lse = in->teacher_lse;
  a->ldi = in->ld_ids;
  a->ldt = in->ld_teacher;
  a->ignore = in->ignore_index;
  a->K = (int)in->top;
  a->ids64 = in->ids_64;
  a->tdtype = in->teacher_dtype;
  a->labels64 = in->labels_64;
  a->T = in->temperature;
  a->alpha = in->alpha;
  return FF_OK;
}

}  // namespace distill
}  // namespace ff

extern "C" int ff_distill_loss(const FfDistillRows* in, int reduction, float* row_loss, float* loss, void* grad, int64_t ldg,
                               float* held, int32_t* counts, void* stream) {
  using namespace ff::distill;
  Args a;
  int rc = fill("ff_distill_loss", in, &a);
  if (rc) return rc;
  FF_REQUIRE(reduction >= FF_REDUCE_NONE && reduction <= FF_REDUCE_SUM, FF_ERR_INVALID_ARG, "ff_distill_loss: bad reduction %d",
             reduction);
  FF_REQUIRE(!grad || (ldg >= a.V && reduction != FF_REDUCE_NONE), FF_ERR_INVALID_ARG,
             "ff_distill_loss: a gradient comes with a reduction, ldg=%lld", (long long)ldg);
  FF_REQUIRE(reduction == FF_REDUCE_NONE || loss, FF_ERR_INVALID_ARG, "ff_distill_loss: null loss");
  FF_REQUIRE(reduction != FF_REDUCE_MEAN || counts, FF_ERR_INVALID_ARG, "ff_distill_loss: the mean needs counts");
  cudaStream_t st = ff::as_stream(stream);
  if (a.rows == 0) {
    if (reduction == FF_REDUCE_MEAN) FF_CUDA_TRY(cudaMemsetAsync(counts, 0, COUNT_CTAS * 4, st), "ff_distill_loss");
    if (reduction != FF_REDUCE_NONE) FF_CUDA_TRY(cudaMemsetAsync(loss, 0, 4, st), "ff_distill_loss");
    return FF_OK;
  }
  FF_REQUIRE(row_loss && ff::aligned(row_loss, 4) && ff::aligned(loss, 4) && ff::aligned(held, 4) && ff::aligned(counts, 4) &&
                 ff::aligned(grad, ff::dtype_size(in->dtype)),
             FF_ERR_INVALID_ARG, "ff_distill_loss: null row_loss or an unaligned output");
  if (reduction == FF_REDUCE_MEAN) {
    distill_count_kernel<<<COUNT_CTAS, 256, 0, st>>>(a, counts);
    rc = ff::check_launch("ff_distill_loss count");
    if (rc) return rc;
    a.mean = 1;
    a.counts = counts;
  }
  a.row_loss = row_loss;
  a.grad = grad;
  a.ldg = ldg;
  rc = launch_dt(a, in->dtype, st, "ff_distill_loss");
  if (rc || reduction == FF_REDUCE_NONE) return rc;
  distill_finish_kernel<<<1, 1024, 0, st>>>(row_loss, a.rows, reduction == FF_REDUCE_MEAN ? counts : nullptr, loss,
                                          grad ? held : nullptr);
  return ff::check_launch("ff_distill_loss finish");
}

extern "C" int ff_distill_grad(const FfDistillRows* in, int reduction, const float* upstream, float* held,
                               int replayed, const int32_t* counts, void* grad, int64_t ldg, void* stream) {
  using namespace ff::distill;
  Args a;
  int rc = fill("ff_distill_grad", in, &a);
  if (rc) return rc;
  FF_REQUIRE(reduction >= FF_REDUCE_NONE && reduction <= FF_REDUCE_SUM, FF_ERR_INVALID_ARG, "ff_distill_grad: bad reduction %d",
             reduction);
  FF_REQUIRE(ldg >= a.V && (reduction != FF_REDUCE_MEAN || counts) && !(held && reduction == FF_REDUCE_NONE),
             FF_ERR_INVALID_ARG, "ff_distill_grad: ldg=%lld, counts with the mean, held with a scalar", (long long)ldg);
  if (a.rows == 0) return FF_OK;
  FF_REQUIRE(grad && upstream && ff::aligned(grad, ff::dtype_size(in->dtype)) && ff::aligned(upstream, 4) && ff::aligned(held, 4) &&
                 ff::aligned(counts, 4),
             FF_ERR_INVALID_ARG, "ff_distill_grad: null or unaligned pointer");
  a.mean = reduction == FF_REDUCE_MEAN;
  a.counts = counts;
  a.grad = grad;
  a.ldg = ldg;
  a.upstream = upstream;
  a.up_stride = reduction == FF_REDUCE_NONE ? 1 : 0;
  a.held = held;
  rc = launch_dt(a, in->dtype, ff::as_stream(stream), "ff_distill_grad");
  if (rc || !held || !replayed) return rc;
  distill_released_kernel<<<1, 1, 0, ff::as_stream(stream)>>>(held);
  return ff::check_launch("ff_distill_grad held");
}
