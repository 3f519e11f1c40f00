// AdamW over many tensors at once: global gradient norm, clipping, decoupled weight decay and the
// moments in 32 bits or in 8 bits with one fp32 scale per block of 256 elements.
//
//   g' = coef g,  coef = min(1, clip / (||g|| + 1e-6))
//   m  = b1 m + (1 - b1) g',  v = b2 v + (1 - b2) g'^2
//   p  = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// The tensors stay where they are: a plan in device memory lists them and cuts each one into chunks
// of 4096 elements, the work of a few small workgroups; the gradients' addresses, which autograd changes
// from step to step, travel as kernel arguments.  Everything is elementwise and bound by HBM: 28 bytes
// per fp32 parameter with 32-bit moments, 16.06 with 8-bit ones, 30 / 18.06 per 16-bit one with its
// master, and the gradient once more for the norm.  Measured (kernels alone): 343 million bf16
// parameters, 32 bits: 1.59 ms, 10.3 GB at 6.5 TB/s, norm 0.11 ms; fp32, 8 bits: 0.93-0.95 ms, 5.5 GB at 5.9
// TB/s; 14 million in 152 tensors: 60 us + 14 + 5 for the norm, 8 bits 42 + 14 + 4; 62 000 in 16
// tensors: 4.3 us.
//
// 8-bit moments: m / s_m and sqrt(v) / s_r in e4m3 with s = max over the block / 448, so that the
// largest element sits on the largest code.  The codes are rounded STOCHASTICALLY, from a hash of
// (seed, step, element): one step moves v by (1 - b2) = 0.1 % of itself, half the distance of two
// codes is up to 6 %, so rounding to nearest would never move most elements again.  The arithmetic
// up to the code is in float64, so that which of two neighbouring codes is taken does not hang on the
// rounding of an intermediate; the moments that move the parameter are the ones before rounding.
#include <math.h>

#include <algorithm>
#include <memory>
#include <new>

#include "tv_common.h"

namespace {

constexpr int AW_THREADS = 256;
constexpr int AW_CHUNK = TV_ADAMW_CHUNK;
constexpr int AW_BLOCK = TV_ADAMW_BLOCK;          // elements per scale: one wave, 4 per lane
constexpr int AW_ITS = AW_CHUNK / (4 * AW_THREADS);
constexpr int AW_GRADS = 384;                     // gradient addresses per launch (3 KB of arguments)
constexpr int AW_NORM_BLOCKS = 2048;              // partial sums per launch
constexpr int64_t AW_MAGIC = 0x74765f6164616d77;

// The plan: its head, the tensors (for the host), the chunks.  A chunk holds all that its workgroup
// needs, so that one load stands between the launch and the loads of the data.
struct Plan {
  int64_t magic, count, chunks, elements;
};
struct Tensor {
  int64_t n;
  int32_t dtype, first_chunk;
};
struct Chunk {
  void *param;                                    // of its first element
  int64_t state;                                  // that element's place in the state
  double weight_decay;
  int32_t n, dtype, tensor, index;                // elements; which tensor, which chunk of it
};
struct Control {
  int64_t step;                                   // steps taken
  double lr, beta1, beta2, eps;
  double beta1_t, beta2_t;                        // beta^step
  // of the step being taken, written by begin_kernel
  double norm, coef;
  float step_size, inv_sqrt_bc2, eps_f;
  int32_t skip;
  uint32_t ticket, unused;                        // of the workgroups of a step without begin_kernel
};
struct Grads {
  const void *g[AW_GRADS];
};

__host__ __device__ inline const Tensor *plan_tensors(const void *plan) {
  return reinterpret_cast<const Tensor *>(static_cast<const char *>(plan) + sizeof(Plan));
}
__host__ __device__ inline const Chunk *plan_chunks(const void *plan, int64_t count) {
  return reinterpret_cast<const Chunk *>(static_cast<const char *>(plan) + sizeof(Plan) +
                                         count * (int64_t)sizeof(Tensor));
}

// Every access carries the hint that nothing of it is read again soon: between two steps a forward and
// a backward pass go through the caches.  Alternating between three models, with the hint against
// without: 14 million parameters 78 us against 89 (32 bits), 57 against 65 (8 bits), 343 million
// 1.70 ms against 1.98 and 0.94 against 1.03.
// Parameters and gradients come by addresses out of memory, which the compiler takes for generic ones
// (flat accesses, which wait for LDS as well): they are global.
#define AW_GLOBAL __attribute__((address_space(1)))
template <typename T> struct Four {                // four elements, at any alignment of the type
  typedef T V __attribute__((ext_vector_type(4)));
  typedef V Any __attribute__((aligned(sizeof(T))));
};
// Four consecutive elements from i on, zeros behind n.  They are widened apart from the load: a conversion
// in the branch would wait for the load there, and the next one would start behind it.
template <typename T> __device__ __forceinline__ typename Four<T>::V load4(const T *p, int i, int n) {
  const AW_GLOBAL T *q = (const AW_GLOBAL T *)(p + i);
  if (i + 4 <= n) return __builtin_nontemporal_load((const AW_GLOBAL typename Four<T>::Any *)q);
  typename Four<T>::V x;
#pragma unroll
  for (int j = 0; j < 4; ++j) x[j] = i + j < n ? q[j] : (T)0.f;
  return x;
}
template <typename V> __device__ __forceinline__ void widen(V f, float (&x)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) x[j] = (float)f[j];
}
template <typename T>
__device__ __forceinline__ void store4(T *p, int i, int n, const float (&x)[4]) {
  AW_GLOBAL T *q = (AW_GLOBAL T *)(p + i);
  if (i + 4 <= n) {
    typedef typename Four<T>::Any Any;
    typename Four<T>::V f;
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = (T)x[j];
    __builtin_nontemporal_store(f, (AW_GLOBAL Any *)q);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i + j < n) q[j] = (T)x[j];
  }
}
// the state: 16-byte aligned segments, padded to 256 elements
typedef float F4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void load4(const float *p, int i, float (&x)[4]) {
  const F4 f = __builtin_nontemporal_load(reinterpret_cast<const F4 *>(p + i));
  x[0] = f.x; x[1] = f.y; x[2] = f.z; x[3] = f.w;
}
__device__ __forceinline__ void store4(float *p, int i, const float (&x)[4]) {
  __builtin_nontemporal_store(F4{x[0], x[1], x[2], x[3]}, reinterpret_cast<F4 *>(p + i));
}
// the master: zeros behind n, whatever 0 / 0 the formula makes of the padding (eps = 0)
__device__ __forceinline__ void store_master(float *p, int i, int n, const float (&x)[4]) {
  float y[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) y[j] = i + j < n ? x[j] : 0.f;
  store4(p, i, y);
}

// ---------------------------------------------------------------------------------------
// ||g||: float64 squares, one partial per workgroup, summed in order by begin_kernel
// ---------------------------------------------------------------------------------------
template <typename T> __device__ __forceinline__ double chunk_sumsq(const T *g, int n) {
  double acc = 0.0;
  if (n == AW_CHUNK) {                            // all loads of the chunk in flight at once
    typename Four<T>::V x[AW_ITS];                  // (without the hint: the step reads them again)
#pragma unroll
    for (int it = 0; it < AW_ITS; ++it)
      x[it] = *(const AW_GLOBAL typename Four<T>::Any *)(g + it * 4 * AW_THREADS + (int)threadIdx.x * 4);
#pragma unroll
    for (int it = 0; it < AW_ITS; ++it)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc = fma((double)(float)x[it][j], (double)(float)x[it][j], acc);
  } else {
    for (int i = (int)threadIdx.x; i < n; i += AW_THREADS) {
      const double x = (double)(float)((const AW_GLOBAL T *)g)[i];
      acc = fma(x, x, acc);
    }
  }
  return acc;
}

__global__ __launch_bounds__(AW_THREADS) void adamw_sumsq_kernel(const void *plan, int64_t count,
                                                                 int64_t chunk0, int64_t chunk1,
                                                                 int64_t tensor0, Grads grads,
                                                                 double *__restrict__ partial) {
  __shared__ double red[AW_THREADS / 64];
  const Chunk *chunks = plan_chunks(plan, count);
  double acc = 0.0;
  struct Part {
    const void *g;
    int n, dtype;
  };
  auto part_of = [&](int64_t c) -> Part {
    const Chunk ch = chunks[c];
    const char *g = (const char *)grads.g[ch.tensor - tensor0];
    if (g != nullptr) g += (int64_t)ch.index * AW_CHUNK * (ch.dtype == TV_DTYPE_F32 ? 4 : 2);
    return {g, ch.n, ch.dtype};
  };
  Part next = part_of(chunk0 + blockIdx.x);       // (the grid is not larger than the number of chunks)
  for (int64_t c = chunk0 + blockIdx.x; c < chunk1; c += gridDim.x) {
    const Part p = next;
    // the next chunk's address on its way while this one is read
    if (c + gridDim.x < chunk1) next = part_of(c + gridDim.x);
    if (p.g == nullptr) continue;
    if (p.dtype == TV_DTYPE_F32) acc += chunk_sumsq((const float *)p.g, p.n);
    else if (p.dtype == TV_DTYPE_BF16) acc += chunk_sumsq((const __bf16 *)p.g, p.n);
    else acc += chunk_sumsq((const _Float16 *)p.g, p.n);
  }
  acc = tv_wave_sum_d(acc);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = acc;
  __syncthreads();
  if (threadIdx.x == 0) {
    double s = red[0];
    for (int w = 1; w < AW_THREADS / 64; ++w) s += red[w];
    partial[blockIdx.x] = s;
  }
}

// The scalars of one step: norm and clip coefficient, the NaN decision, bias corrections.  The step
// counter and the learning rate live on the device, so a captured step counts on when it is replayed.
constexpr int AW_BEGIN_THREADS = 1024;
__global__ __launch_bounds__(AW_BEGIN_THREADS) void adamw_begin_kernel(Control *ctl, bool clipped, int64_t nblk,
                                                          const double *__restrict__ partial,
                                                          double clip, double *norm_out,
                                                          const float *guard, int guard_kind,
                                                          float *guard_copy) {
  __shared__ double red[AW_BEGIN_THREADS / 64];
  if (clipped) {
    double acc = 0.0;
    for (int64_t i = threadIdx.x; i < nblk; i += AW_BEGIN_THREADS) acc += partial[i];
    acc = tv_wave_sum_d(acc);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = acc;
    __syncthreads();
  }
  if (threadIdx.x != 0) return;
  double coef = 1.0;
  if (clipped) {
    double sum = red[0];
    for (int w = 1; w < AW_BEGIN_THREADS / 64; ++w) sum += red[w];
    const double norm = sqrt(sum);
    ctl->norm = norm;
    if (norm_out != nullptr) norm_out[0] = norm;
    // a NaN norm gives a NaN coefficient, and so NaN parameters
    coef = clip / (norm + 1e-6);
    if (coef > 1.0) coef = 1.0;
  }
  ctl->coef = coef;
  bool skip = false;
  if (guard != nullptr) {
    const float v = guard[0];
    if (guard_copy != nullptr) guard_copy[0] = v;
    skip = guard_kind == 1 ? (v != v) : (v != 0.f);
  }
  ctl->skip = skip ? 1 : 0;
  if (skip) return;
  const double b1t = ctl->beta1_t * ctl->beta1, b2t = ctl->beta2_t * ctl->beta2;
  ctl->step += 1;
  ctl->beta1_t = b1t;
  ctl->beta2_t = b2t;
  ctl->step_size = (float)(ctl->lr / (1.0 - b1t));
  ctl->inv_sqrt_bc2 = (float)(1.0 / sqrt(1.0 - b2t));
  ctl->eps_f = (float)ctl->eps;
}

// ---------------------------------------------------------------------------------------
// the update
// ---------------------------------------------------------------------------------------
struct Step {
  float keep, step_size, inv_sqrt_bc2, eps;       // keep = 1 - lr * weight_decay
  double coef, beta1, beta2, omb1, omb2;
  uint32_t key;
  uint32_t far;                                   // bits of the rms from which on a block divides, see moved8
  int it0, it1;                                   // which 4 * THREADS elements of the chunk
};

__device__ __forceinline__ float moved(float p, float m, float r, const Step &s) {
  float x = fmaf(-s.step_size, m / fmaf(r, s.inv_sqrt_bc2, s.eps), p * s.keep);
  // the fp32 value itself: the compiler would fold a conversion to fp16 into the fma, and the
  // parameter would no longer be what its master rounds to
  asm("" : "+v"(x));
  return x;
}

// the same with the reciprocal of the hardware (1 ulp): the division costs more than a code does.  It takes
// what is not normal for zero, on both sides: a block in which r / sqrt(1 - b2^t) + eps may pass 2^125 divides,
// and so does every block where eps is below 2^-126.
__device__ __forceinline__ float moved8(float p, float m, float r, const Step &s) {
  float x = fmaf(-s.step_size, m * __builtin_amdgcn_rcpf(fmaf(r, s.inv_sqrt_bc2, s.eps)), p * s.keep);
  asm("" : "+v"(x));
  return x;
}

__device__ __forceinline__ uint32_t far_from(const Step &s) {
  const float r = (0x1p125f - s.eps) / s.inv_sqrt_bc2;
  return s.eps >= 0x1p-126f && r > 0.f ? __float_as_uint(r) : 0u;
}

// 16-bit parameters are rounded copies of an fp32 master; one that is not what its master rounds to
// was written by somebody else (a checkpoint was loaded), and the master follows it
template <typename T>
__device__ __forceinline__ float master_of(float p, float w) {
  return (float)(T)w == p ? w : p;
}
template <>
__device__ __forceinline__ float master_of<float>(float p, float) { return p; }

template <int THREADS, typename T>
__device__ __forceinline__ void chunk_step32(T *p, const T *g, float *w, float *m, float *v, int n,
                                             const Step &s) {
  const float b1 = (float)s.beta1, b2 = (float)s.beta2, o1 = (float)s.omb1, o2 = (float)s.omb2;
  const float coef = (float)s.coef;
  for (int it = s.it0; it < s.it1; ++it) {
    const int i = it * 4 * THREADS + (int)threadIdx.x * 4;
    if (i >= n) break;
    float px[4], gx[4], wx[4], mx[4], vx[4];
    const auto p4 = load4(p, i, n), g4 = load4(g, i, n);
    load4(m, i, mx);
    load4(v, i, vx);
    if (sizeof(T) != 4) load4(w, i, wx);
    widen(p4, px);
    widen(g4, gx);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float gj = gx[j] * coef;
      mx[j] = fmaf(b1, mx[j], o1 * gj);
      vx[j] = fmaf(b2, vx[j], o2 * gj * gj);
      px[j] = moved(sizeof(T) == 4 ? px[j] : master_of<T>(px[j], wx[j]), mx[j], sqrtf(vx[j]), s);
    }
    store4(p, i, n, px);
    store4(m, i, mx);
    store4(v, i, vx);
    if (sizeof(T) != 4) store_master(w, i, n, px);
  }
}

__host__ __device__ inline uint32_t mix(uint32_t x) {
  // two rounds of shift and multiply by odd constants (fractional bits of sqrt 2 and sqrt 3)
  x ^= x >> 16;
  x *= 0x6a09e667u;
  x ^= x >> 15;
  x *= 0xbb67ae85u;
  return x ^ (x >> 16);
}

// e4m3 magnitude code of y = x / scale in [0, 448 (1 + 2^-23)], rounded up with the probability of what
// is left over the code below: 17 random bits (the lowest always set, so an exact value stays) are added
// to the 17 mantissa bits of the high word that e4m3 drops.  Below 2^-6 codes lie 2^-9 apart: adding 2^-6
// puts those bits at the same place.  `low` may be decided in fp32: within 2^-22 of 2^-6 both ways give
// the code of 2^-6.
__device__ __forceinline__ uint32_t code_of(double x, double inverse_scale, bool low, uint32_t random17) {
  const double z = fma(x, inverse_scale, __hiloint2double(low ? 0x3f900000 : 0, 0));
  const uint32_t base = low ? 1017u << 20 : 1016u << 20;
  const uint32_t c = ((uint32_t)__double2hiint(z) + random17 - base) >> 17;
  return c < 126u ? c : 126u;
}
__device__ __forceinline__ float scale_of(float largest) {
  const float s = largest * (1.f / 448.f);
  return s >= 0x1p-100f ? s : 0.f;                // (below that the block counts as zero)
}
__device__ __forceinline__ void decode4(uint32_t c, float (&x)[4]) {
  typedef float F2 __attribute__((ext_vector_type(2)));
  const F2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false);
  const F2 b = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
  x[0] = a[0]; x[1] = a[1]; x[2] = b[0]; x[3] = b[1];
}

constexpr uint32_t INF_BITS = 0x7f800000u;
// largest value of a wave
__device__ __forceinline__ uint32_t wave_largest(uint32_t v) {
#define AW_DPP(ctrl) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, 0xf, 0xf, false))
  AW_DPP(0x111);   // row_shr 1, 2, 4, 8: lane 15 of each row of 16 has the row's
  AW_DPP(0x112);
  AW_DPP(0x114);
  AW_DPP(0x118);
  AW_DPP(0x142);   // row_bcast 15, 31: lane 63 has the wave's
  AW_DPP(0x143);
#undef AW_DPP
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// a b + c d, each of the three rounded.  (b1 m + (1 - b1) g with b1 = 0.9 is (9 m + g) / 10: one in some
// hundred is a number of 25 bits, whose rounding to the fp32 scale hangs on the last bit of float64, so
// the order of its roundings is part of the definition.)
__device__ __forceinline__ double two_products(double a, double b, double c, double d) {
#pragma clang fp contract(off)
  const double x = a * b, y = c * d;
  return x + y;
}
// sqrt(v) for v > 0 to 2^-47 (NaN for inf): the hardware's reciprocal root (2^-24) and one Newton step, a
// third of the library's sqrt.  (That is enough for the codes; the fp32 scale, made from the largest root
// of a block, is the neighbouring number in one block of some 10 million.  A second step costs 2 % of the
// whole.)
__device__ __forceinline__ double root(double v) {
  const double q = __builtin_amdgcn_rsq(v), r = v * q;
  return fma(fma(-r, r, v), 0.5 * q, r);
}
// 1 / s to 2^-45, 0 for 0
__device__ __forceinline__ double inverse(float s) {
  if (s > 0.f && s < 1e30f) {                     // (at least 2^-100)
    const double d = (double)s, q = (double)__builtin_amdgcn_rcpf(s);
    return fma(fma(-d, q, 1.0), q, q);
  }
  return s > 0.f ? 1.0 / (double)s : 0.0;
}

template <int THREADS, typename T>
__device__ __forceinline__ void chunk_step8(T *p, const T *g, float *w, uint32_t *m8, float *ms,
                                            uint32_t *r8, float *rs, int n, int64_t element0,
                                            const Step &s) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  for (int it = s.it0; it < s.it1; ++it) {
    const int b = it * (4 * THREADS / AW_BLOCK) + wave, i = b * AW_BLOCK + lane * 4;
    if (b * AW_BLOCK >= n) break;                 // (the same for the whole wave)
    // (blocks begin at multiples of 256: the high word is the same for the whole block)
    const uint32_t key = mix(s.key + (uint32_t)((element0 + b * AW_BLOCK) >> 32));
    const uint32_t element = (uint32_t)(element0 + i);
    float px[4], gx[4], wx[4], mo[4], ro[4];
    const auto p4 = load4(p, i, n), g4 = load4(g, i, n);
    const uint32_t m4 = __builtin_nontemporal_load(m8 + i / 4), r4 = __builtin_nontemporal_load(r8 + i / 4);
    if (sizeof(T) != 4) load4(w, i, wx);
    const double sm = ms[b], sr = rs[b];
    widen(p4, px);
    widen(g4, gx);
    decode4(m4, mo);
    decode4(r4, ro);
    const double k2 = s.beta2 * (sr * sr);
    double mx[4], rx[4];
    uint32_t am = 0, ar = 0;                      // bits of the largest |m| and rms in fp32
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const double gj = (double)gx[j] * s.coef;
      mx[j] = two_products(s.beta1, mo[j] * sm, s.omb1, gj);
      // (the square of a code has 8 bits: exact in fp32.  1e-300 keeps a zero from 0 / 0: its root is zero
      // in fp32, and gradients that are not zero have squares above 1e-90)
      rx[j] = root(fma(k2, (double)(ro[j] * ro[j]), fma(s.omb2 * gj, gj, 1e-300)));
      am = max(am, __float_as_uint(fabsf((float)mx[j])));
      ar = max(ar, __float_as_uint(fabsf((float)rx[j])));
    }
    am = wave_largest(am);
    ar = wave_largest(ar);
    const bool odd = max(am, ar) >= INF_BITS;     // (the same for the whole wave)
    if (odd) {                                    // infinite or NaN moments: the scales are the others'
      am = ar = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t mb = __float_as_uint(fabsf((float)mx[j])), rb = __float_as_uint(fabsf((float)rx[j]));
        am = max(am, mb < INF_BITS ? mb : 0u);
        ar = max(ar, rb < INF_BITS ? rb : 0u);
      }
      am = wave_largest(am);
      ar = wave_largest(ar);
    }
    const float nm = scale_of(__uint_as_float(am)), nr = scale_of(__uint_as_float(ar));
    const double im = inverse(nm), ir = inverse(nr);
    // below 2^-6 of a scale; everything in a block of zeros
    const float lm = nm > 0.f ? nm * 0.015625f : INFINITY, lr = nr > 0.f ? nr * 0.015625f : INFINITY;
    if (sizeof(T) != 4) {
#pragma unroll
      for (int j = 0; j < 4; ++j) px[j] = master_of<T>(px[j], wx[j]);
    }
    // (the same for the whole wave.  Parameters in loops of their own in front of the codes: 934 us for 343 million
    // fp32 parameters; the division behind the codes on reloaded parameters 957; no division at all 926)
    if (__builtin_expect(ar >= s.far, 0)) {
#pragma unroll
      for (int j = 0; j < 4; ++j) px[j] = moved(px[j], (float)mx[j], (float)rx[j], s);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) px[j] = moved8(px[j], (float)mx[j], (float)rx[j], s);
    }
    uint32_t cm = 0, cr = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t u = mix(key ^ (element + (uint32_t)j));
      const float mf = (float)mx[j], rf = (float)rx[j];
      const uint32_t a = code_of(fabs(mx[j]), im, fabsf(mf) < lm, ((u << 1) & 0x1ffffu) | 1u);
      const uint32_t c = code_of(rx[j], ir, rf < lr, (u >> 15) | 1u);
      cm |= (a | ((__float_as_uint(mf) >> 24) & 0x80u)) << (8 * j);
      cr |= max(c, min(__float_as_uint(rf), 1u)) << (8 * j);      // a positive rms stays positive
    }
    if (__builtin_expect(odd, 0)) {               // infinite and NaN moments become NaN
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (__float_as_uint(fabsf((float)mx[j])) >= INF_BITS) cm |= 0x7fu << (8 * j);
        if (__float_as_uint(fabsf((float)rx[j])) >= INF_BITS) cr |= 0x7fu << (8 * j);
      }
    }
    store4(p, i, n, px);
    if (sizeof(T) != 4) store_master(w, i, n, px);
    __builtin_nontemporal_store(cm, m8 + i / 4);
    __builtin_nontemporal_store(cr, r8 + i / 4);
    if (lane == 0) {
      ms[b] = nm;
      rs[b] = nr;
    }
  }
}

// ALONE: without begin_kernel (no norm, no guard, few workgroups): every workgroup computes the scalars,
// and the last one to finish - all others have read the counters by then - counts the step
template <bool EIGHT, bool ALONE, int THREADS>
__global__ __launch_bounds__(THREADS) void adamw_step_kernel(
    const void *plan, int64_t count, int64_t chunk0, int lg_parts, int64_t tensor0, Grads grads, Control *ctl,
    void *moment1, void *moment2, float *scale1, float *scale2, float *master, uint32_t seed_key) {
  const Chunk ch = plan_chunks(plan, count)[chunk0 + (blockIdx.x >> lg_parts)];
  const void *g = grads.g[ch.tensor - tensor0];
  const int64_t base = (int64_t)ch.index * AW_CHUNK, at = ch.state;
  const int n = ch.n;
  Step s;
  const int part = (int)blockIdx.x & ((1 << lg_parts) - 1), its = AW_CHUNK / (4 * THREADS) >> lg_parts;
  s.it0 = part * its;
  s.it1 = s.it0 + its;
  s.keep = (float)(1.0 - ctl->lr * ch.weight_decay);
  s.beta1 = ctl->beta1;
  s.beta2 = ctl->beta2;
  s.omb1 = 1.0 - s.beta1;
  s.omb2 = 1.0 - s.beta2;
  int64_t step = ctl->step;
  double b1t = 0.0, b2t = 0.0;
  bool skip = false;
  if (ALONE) {
    step += 1;
    b1t = ctl->beta1_t * s.beta1;
    b2t = ctl->beta2_t * s.beta2;
    s.step_size = (float)(ctl->lr / (1.0 - b1t));
    s.inv_sqrt_bc2 = (float)(1.0 / sqrt(1.0 - b2t));
    s.eps = (float)ctl->eps;
    s.coef = 1.0;
  } else {
    s.step_size = ctl->step_size;
    s.inv_sqrt_bc2 = ctl->inv_sqrt_bc2;
    s.eps = ctl->eps_f;
    s.coef = ctl->coef;
    skip = ctl->skip != 0;
  }
  // (tested behind the loads above, which are in flight together.  Without a gradient the tensor stays
  // as it is)
  if (!skip && g != nullptr && s.it0 * (4 * THREADS) < n) {
    float *w = master ? master + at : nullptr;
    if (EIGHT) {
      s.key = mix(seed_key + (uint32_t)step);
      s.far = far_from(s);
      uint32_t *m8 = (uint32_t *)moment1 + at / 4, *r8 = (uint32_t *)moment2 + at / 4;
      float *ms = scale1 + at / AW_BLOCK, *rs = scale2 + at / AW_BLOCK;
      if (ch.dtype == TV_DTYPE_F32)
        chunk_step8<THREADS>((float *)ch.param, (const float *)g + base, w, m8, ms, r8, rs, n, at, s);
      else if (ch.dtype == TV_DTYPE_BF16)
        chunk_step8<THREADS>((__bf16 *)ch.param, (const __bf16 *)g + base, w, m8, ms, r8, rs, n, at, s);
      else
        chunk_step8<THREADS>((_Float16 *)ch.param, (const _Float16 *)g + base, w, m8, ms, r8, rs, n, at, s);
    } else {
      float *m = (float *)moment1 + at, *v = (float *)moment2 + at;
      if (ch.dtype == TV_DTYPE_F32)
        chunk_step32<THREADS>((float *)ch.param, (const float *)g + base, w, m, v, n, s);
      else if (ch.dtype == TV_DTYPE_BF16)
        chunk_step32<THREADS>((__bf16 *)ch.param, (const __bf16 *)g + base, w, m, v, n, s);
      else
        chunk_step32<THREADS>((_Float16 *)ch.param, (const _Float16 *)g + base, w, m, v, n, s);
    }
  }
  if (ALONE) {
    // Behind the barrier the whole workgroup has its copy of the counters, and thread 0 has used its own;
    // the last ticket so means that nobody reads them any more.  No fence to the device: nothing that
    // this workgroup has written is read in this launch (and such a fence writes the L2 back: 2 us).
    __syncthreads();
    if (threadIdx.x == 0 && __hip_atomic_fetch_add(&ctl->ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
                                gridDim.x - 1) {
      ctl->ticket = 0;
      ctl->step = step;
      ctl->beta1_t = b1t;
      ctl->beta2_t = b2t;
    }
  }
}

inline int64_t padded(int64_t n) { return tv_cdiv(n, AW_BLOCK) * AW_BLOCK; }
inline int64_t groups(int64_t count) { return tv_cdiv(count, AW_GRADS); }

}  // namespace

extern "C" int64_t tv_adamw_control_bytes(void) { return (int64_t)sizeof(Control); }

extern "C" int tv_adamw_control(int64_t step, double lr, double beta1, double beta2, double eps,
                                void *control) {
  TV_REQUIRE(control, "tv_adamw_control: null pointer");
  TV_REQUIRE(step >= 0, "tv_adamw_control: step counts from 0 (steps taken so far)");
  TV_REQUIRE(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0,
             "tv_adamw_control: the betas lie in [0, 1)");
  TV_REQUIRE(eps >= 0.0 && eps < INFINITY && lr >= 0.0 && lr < INFINITY,
             "tv_adamw_control: lr and eps are finite and not negative");
  Control c = {};
  c.step = step;
  c.lr = lr;
  c.beta1 = beta1;
  c.beta2 = beta2;
  c.eps = eps;
  // the product as the steps form it, so that a run that is taken up again has the same bits (what lies
  // below 1e-30 no longer shows in 1 - beta^step); behind 2^24 steps, 20 ms, by pow
  c.beta1_t = c.beta2_t = 1.0;
  const int64_t factors = step < (1 << 24) ? step : 1 << 24;
  for (int64_t t = 0; t < factors && (c.beta1_t > 1e-30 || c.beta2_t > 1e-30); ++t) {
    c.beta1_t *= beta1;
    c.beta2_t *= beta2;
  }
  if (step > factors) {
    c.beta1_t *= pow(beta1, (double)(step - factors));
    c.beta2_t *= pow(beta2, (double)(step - factors));
  }
  *(Control *)control = c;
  return TV_OK;
}

extern "C" int64_t tv_adamw_state_elements(int64_t count, const int64_t *sizes) {
  if (count < 1 || !sizes) return -1;
  int64_t total = 0;
  for (int64_t i = 0; i < count; ++i) {
    if (sizes[i] < 0 || sizes[i] > INT64_MAX / 16 - total) return -1;
    total += padded(sizes[i]);
  }
  return total;
}

extern "C" int64_t tv_adamw_plan_bytes(int64_t count, const int64_t *sizes) {
  if (tv_adamw_state_elements(count, sizes) < 0) return -1;
  int64_t chunks = 0;
  for (int64_t i = 0; i < count; ++i) chunks += tv_cdiv(sizes[i], AW_CHUNK);
  return (int64_t)sizeof(Plan) + count * (int64_t)sizeof(Tensor) + chunks * (int64_t)sizeof(Chunk);
}

extern "C" int tv_adamw_plan(int64_t count, const int64_t *sizes, const int *dtypes,
                             void *const *params, const double *weight_decay, void *plan,
                             int64_t plan_bytes) {
  TV_REQUIRE(count >= 1 && sizes && dtypes && params && weight_decay && plan,
             "tv_adamw_plan: bad arguments");
  const int64_t need = tv_adamw_plan_bytes(count, sizes);
  TV_REQUIRE(need >= 0, "tv_adamw_plan: a size is negative or the sizes are too large");
  TV_REQUIRE((need - (int64_t)sizeof(Plan) - count * (int64_t)sizeof(Tensor)) / (int64_t)sizeof(Chunk) < ((int64_t)1 << 32) / AW_THREADS,
             "tv_adamw_plan: more chunks of %d elements than one launch takes", AW_CHUNK);
  if (plan_bytes < need) {
    tv_set_error("tv_adamw_plan: plan of %lld bytes, %lld needed", (long long)plan_bytes, (long long)need);
    return TV_ERR_WORKSPACE;
  }
  Tensor *tensors = const_cast<Tensor *>(plan_tensors(plan));
  Chunk *chunks = const_cast<Chunk *>(plan_chunks(plan, count));
  int64_t chunk = 0, state = 0;
  for (int64_t i = 0; i < count; ++i) {
    const int width = dtypes[i] == TV_DTYPE_F32 ? 4 : 2;
    TV_REQUIRE(dtypes[i] == TV_DTYPE_F32 || dtypes[i] == TV_DTYPE_BF16 || dtypes[i] == TV_DTYPE_F16,
               "tv_adamw_plan: tensor %lld has an unknown dtype %d", (long long)i, dtypes[i]);
    TV_REQUIRE((params[i] || sizes[i] == 0) && ((uintptr_t)params[i] & (uintptr_t)(width - 1)) == 0,
               "tv_adamw_plan: tensor %lld has a null or misaligned address", (long long)i);
    TV_REQUIRE(weight_decay[i] >= 0.0 && weight_decay[i] < INFINITY,
               "tv_adamw_plan: the weight decay of tensor %lld is negative or infinite", (long long)i);
    tensors[i] = Tensor{sizes[i], dtypes[i], (int32_t)chunk};
    for (int64_t k = 0; k < tv_cdiv(sizes[i], AW_CHUNK); ++k) {
      const int64_t left = sizes[i] - k * AW_CHUNK;
      chunks[chunk++] = Chunk{(char *)params[i] + k * AW_CHUNK * width, state + k * AW_CHUNK, weight_decay[i],
                              (int32_t)(left < AW_CHUNK ? left : AW_CHUNK), dtypes[i], (int32_t)i, (int32_t)k};
    }
    state += padded(sizes[i]);
  }
  // two tensors in one place would be updated twice, at once
  struct Span {
    uintptr_t first, last;
    bool operator<(const Span &o) const { return first < o.first; }
  };
  std::unique_ptr<Span[]> spans(new (std::nothrow) Span[(size_t)count]);
  TV_REQUIRE(spans, "tv_adamw_plan: out of host memory");
  int64_t used = 0;
  for (int64_t i = 0; i < count; ++i)
    if (sizes[i] > 0)
      spans[used++] = {(uintptr_t)params[i],
                       (uintptr_t)params[i] + (uintptr_t)sizes[i] * (dtypes[i] == TV_DTYPE_F32 ? 4 : 2)};
  std::sort(spans.get(), spans.get() + used);
  for (int64_t i = 1; i < used; ++i)
    TV_REQUIRE(spans[i].first >= spans[i - 1].last, "tv_adamw_plan: two tensors overlap in memory");
  Plan head = {AW_MAGIC, count, chunk, state};
  *(Plan *)plan = head;
  return TV_OK;
}

extern "C" int64_t tv_adamw_workspace_bytes(int64_t count) {
  return groups(count < 1 ? 1 : count) * AW_NORM_BLOCKS * (int64_t)sizeof(double);
}

extern "C" int tv_adamw_step(const void *plan_host, const void *plan_device,
                             const void *const *grads, int state_bits, void *moment1, void *moment2,
                             float *scale1, float *scale2, float *master, void *control,
                             double clip_norm, double *norm_out, int64_t seed, const float *guard,
                             int guard_kind, float *guard_host, void *workspace,
                             int64_t workspace_bytes, void *stream) {
  TV_REQUIRE(plan_host && plan_device && grads && control, "tv_adamw_step: null pointer");
  const Plan *plan = (const Plan *)plan_host;
  TV_REQUIRE(plan->magic == AW_MAGIC, "tv_adamw_step: not a plan of tv_adamw_plan");
  TV_REQUIRE(state_bits == 8 || state_bits == 32, "tv_adamw_step: moments of 8 or 32 bits");
  TV_REQUIRE((moment1 && moment2) || plan->elements == 0, "tv_adamw_step: null moments");
  TV_REQUIRE(state_bits == 32 || (scale1 && scale2) || plan->elements == 0,
             "tv_adamw_step: 8-bit moments need their scales");
  TV_REQUIRE(((((uintptr_t)moment1) | (uintptr_t)moment2 | (uintptr_t)master) & 15) == 0,
             "tv_adamw_step: moments and master are 16-byte aligned");
  TV_REQUIRE(clip_norm >= 0.0, "tv_adamw_step: clip_norm is 0 (off) or positive");
  TV_REQUIRE(clip_norm > 0.0 || !norm_out, "tv_adamw_step: the norm is computed with clip_norm only");
  TV_REQUIRE(guard_kind >= 0 && guard_kind <= 2 && (guard != nullptr) == (guard_kind != 0),
             "tv_adamw_step: guard_kind 1 (NaN) or 2 (non-zero) with a guard, 0 without");
  TV_REQUIRE(!guard_host || guard, "tv_adamw_step: guard_host without a guard");
  const Tensor *tensors = plan_tensors(plan_host);
  for (int64_t i = 0; i < plan->count; ++i) {
    TV_REQUIRE(((uintptr_t)grads[i] & (tensors[i].dtype == TV_DTYPE_F32 ? 3 : 1)) == 0,
               "tv_adamw_step: the gradient of tensor %lld is misaligned", (long long)i);
    TV_REQUIRE(tensors[i].dtype == TV_DTYPE_F32 || master || tensors[i].n == 0,
               "tv_adamw_step: 16-bit parameters need a master");
  }
  const int64_t ngroups = groups(plan->count);
  if (clip_norm > 0.0) {
    TV_REQUIRE(workspace, "tv_adamw_step: null workspace");
    if (workspace_bytes < tv_adamw_workspace_bytes(plan->count)) {
      tv_set_error("tv_adamw_step: workspace too small");
      return TV_ERR_WORKSPACE;
    }
  }
  float *guard_copy = nullptr;
  if (guard_host) {
    const int rc = tv_pinned_pointer("tv_adamw_step", guard_host, &guard_copy);
    if (rc != TV_OK) return rc;
  }
  auto group_grads = [&](int64_t k, Grads &g, int64_t &chunk0, int64_t &chunk1) {
    const int64_t t0 = k * AW_GRADS, t1 = t0 + AW_GRADS < plan->count ? t0 + AW_GRADS : plan->count;
    for (int64_t i = t0; i < t1; ++i) g.g[i - t0] = grads[i];
    chunk0 = tensors[t0].first_chunk;
    chunk1 = t1 < plan->count ? tensors[t1].first_chunk : plan->chunks;
  };
  int64_t nblk = 0;
  double *partial = (double *)workspace;
  for (int64_t k = 0; clip_norm > 0.0 && k < ngroups; ++k) {
    Grads g = {};
    int64_t c0, c1;
    group_grads(k, g, c0, c1);
    if (c1 == c0) continue;
    const int64_t blocks = c1 - c0 < AW_NORM_BLOCKS ? c1 - c0 : AW_NORM_BLOCKS;
    hipLaunchKernelGGL(adamw_sumsq_kernel, dim3((unsigned)blocks), dim3(AW_THREADS), 0,
                       (hipStream_t)stream, plan_device, plan->count, c0, c1, k * AW_GRADS, g,
                       partial + nblk);
    TV_LAUNCH_CHECK("tv_adamw_step");
    nblk += blocks;
  }
  // One launch where nothing has to be known before it and few workgroups take a ticket: the tickets are
  // taken one after another, 12 ns each.  A step of 64 chunks 4.9-6.3 us against 8.7-8.9 with the launch of
  // the scalars, of 128 chunks 7.3-7.7 against 8.6-9.0, of 192 chunks the same, of 512 chunks 17 against 12-15.
  const bool alone = clip_norm == 0.0 && !guard && ngroups == 1 && plan->chunks > 0 && plan->chunks <= 128;
  if (!alone) {
    hipLaunchKernelGGL(adamw_begin_kernel, dim3(1), dim3(clip_norm > 0.0 ? AW_BEGIN_THREADS : 64), 0,
                       (hipStream_t)stream, (Control *)control, clip_norm > 0.0, nblk, partial, clip_norm,
                       norm_out, guard, guard_kind, guard_copy);
    TV_LAUNCH_CHECK("tv_adamw_step");
  }
  // A chunk is the work of 2^lg workgroups side by side.  Many small ones, which begin and end one by one,
  // stream best: with 32-bit moments 268 million fp32 parameters take 1190 us in 8 x 128 threads, 1258 in
  // 4 x 256, 1276 in 1 x 1024 (bf16: 1332, 1336, 1384).  The scalars of a workgroup weigh more with 8-bit
  // moments: 729 us in 4 x 128, 797 in 8 x 128 - up to 256 chunks the other way round, 9.9 against 9.1.
  // The one-launch step takes fewer tickets with 2 x 512: 64 chunks 5.5-6.6 us against 6.5-7.1 in 4 x 256.
  const int lg = alone ? 1 : state_bits == 32 || plan->chunks <= 256 ? 3 : 2;
  // Large models, 32 bits: 24 KB of LDS that nobody uses leave 6 such workgroups on a CU, which reads and writes
  // memory in longer runs: 537 million fp32 2401 us against 2507, bf16 2569 against 2733; 25 million 113.1
  // against 113.9 and 121 against 124, 14 million with clipping 81.4 against 77.4.  (Not for 8-bit moments, which
  // need the waves to cover their arithmetic: 878 against 723.)
  const unsigned lds = state_bits == 32 && plan->chunks > 4096 ? 24 << 10 : 0;
  constexpr int64_t launch_chunks = 1 << 21;      // (a launch has less than 2^32 threads)
  for (int64_t k = 0; k < ngroups; ++k) {
    Grads g = {};
    int64_t c0, c1;
    group_grads(k, g, c0, c1);
    for (int64_t c = c0; c < c1; c += launch_chunks) {
      auto kernel = alone ? (state_bits == 8 ? adamw_step_kernel<true, true, 512> : adamw_step_kernel<false, true, 512>)
                          : (state_bits == 8 ? adamw_step_kernel<true, false, 128> : adamw_step_kernel<false, false, 128>);
      const int64_t n = c1 - c < launch_chunks ? c1 - c : launch_chunks;
      hipLaunchKernelGGL(kernel, dim3((unsigned)(n << lg)), dim3(alone ? 512 : 128), lds, (hipStream_t)stream,
                         plan_device, plan->count, c, lg, k * AW_GRADS, g, (Control *)control, moment1, moment2,
                         scale1, scale2, master, mix((uint32_t)seed));
      TV_LAUNCH_CHECK("tv_adamw_step");
    }
  }
  return TV_OK;
}
