// Optimizer over a list of tensors: global gradient norm with its clip factor, and AdamW (Keras form: epsilon outside
// the square root, decay decoupled from the gradient) with its state in fp32 or in 8 bits.
//
//   t += 1;  alpha = lr sqrt(1 - b2^t) / (1 - b1^t)
//   g' = g gs;  m += (g' - m)(1 - b1);  v += (g'^2 - v)(1 - b2);  p -= p (lr wd);  p -= alpha m / (sqrt(v) + eps)
//
// All of it is bound by HBM: an element costs its own bytes once in and once out, the arithmetic is ~20 flop.
//   * tensors of any length and alignment in ONE launch (64 per launch: their table travels in the kernel arguments, so
//     nothing is copied to the device and a captured launch owns its table);
//   * a workgroup takes 4 096 consecutive elements of one tensor and finds the tensor with one ballot over the table;
//   * a wave takes 1 024 of them as four state blocks of 256: lanes 16q..16q+15 own block q, four loads of four
//     elements each, so the block's maximum is four DPP steps inside a row of 16 lanes and never leaves the registers.
//
// 8-bit state: a block of 256 elements shares one power of two (kept as fp32), m holds e4m3 codes, v holds e5m2 codes
// (v needs the range: it is a square).  Both are stored by STOCHASTIC rounding from a counter hash of (seed, t,
// position).  v moves by (1 - b2) = 0.1 % a step; between codes 12-25 % apart nearest rounding would never move it.  The
// recursions are linear in m and v, so rounding without a bias would keep the expected state equal to the 32-bit recursion.
// A draw has 16 bits and meets the top 16 of the 20 or 21 that a code drops: what lies under them is cut, so a stored magnitude is low by
// 0 to 2^-16 of its code's spacing in the mean, and over the 1 / (1 - b) steps that the state remembers by that many times as much.
// The spacing of v is a quarter of it at most: v settles up to 0.4 % low at b2 = 0.999 and 3.8 % at 0.9999 (measured at a constant
// gradient: 0.06 and 1.3 %), steps are longer by half of that.  The entry refuses b > 0.9999 with 8 bits: there a step's own
// movement of v sinks to what is cut.  A
// positive v never rounds to zero (the step would divide by epsilon alone); a block with an infinity or NaN gets the
// scale NaN.  Arithmetic is fp32 throughout; this file is compiled without contraction so that the stored codes do
// not depend on which products a compiler fuses.
#include "common.h"
#include <math.h>

namespace cfd {

constexpr int OPT_T = 64;         // tensors per launch: one ballot finds the tensor; 3.1 KB of kernel arguments
constexpr int OPT_BLOCK = 256;    // elements that share a scale
constexpr int OPT_CHUNK = 4096;   // elements per workgroup

// loads of four elements at element alignment (global memory takes any dword-, for bf16 any 2-byte-aligned vector)
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef __bf16 bf16x4u __attribute__((ext_vector_type(4), aligned(2)));
template <typename T> struct Vec4;
template <> struct Vec4<float> { typedef f32x4u type; };
template <> struct Vec4<bf16> { typedef bf16x4u type; };

template <typename T> __device__ __forceinline__ void load4(const T *p, int left, float (&o)[4]) {
  if (left >= 4) {
    const typename Vec4<T>::type v = *(const typename Vec4<T>::type *)p;
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] = (float)v[k];
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] = k < left ? (float)p[k] : 0.f;
  }
}
template <typename T> __device__ __forceinline__ void store4(T *p, int left, const float (&o)[4]) {
  if (left >= 4) {
    typename Vec4<T>::type v;
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = (T)o[k];   // bf16: round to nearest even
    *(typename Vec4<T>::type *)p = v;
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < left) p[k] = (T)o[k];
  }
}

__host__ __device__ __forceinline__ unsigned hash32(unsigned x) {   // a bijection; shifts and factors: C. Wellons (2018), found by search for the least avalanche bias
  x ^= x >> 16; x *= 0x7feb352du;
  x ^= x >> 15; x *= 0x846ca68bu;
  return x ^ (x >> 16);
}

__device__ __forceinline__ unsigned row16_umax(unsigned v) {
  v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, false));
  v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xf, 0xf, false));
  v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x122, 0xf, 0xf, false));
  return max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x121, 0xf, 0xf, false));
}

// ---------------------------------------------------------------------------------------------------- gradient norm
// Squares and sums in fp64: no overflow for any finite fp32 gradient and no dependence on the sum's order worth naming;
// partial sums are added in a fixed order (bitwise reproducible).
struct NormArgs {
  const void *g[OPT_T];
  int64_t n[OPT_T];
  unsigned first[OPT_T];   // first workgroup of each tensor
  int nt;
  int64_t chunk;
  double *part;
};

__device__ __forceinline__ int find_tensor(const unsigned *first, int nt, unsigned bid) {
  const int lane = threadIdx.x & 63;
  const unsigned long long m = __ballot(lane < nt && first[lane] <= bid);
  return __builtin_amdgcn_readfirstlane(__popcll(m) - 1);
}

template <int NW> __device__ __forceinline__ double block_sum(double s, double *sh) {
#pragma unroll
  for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
  __syncthreads();
  double t = 0.;
#pragma unroll
  for (int i = 0; i < NW; ++i) t += sh[i];
  return t;
}

// One read: 137 MB of bf16 (68.7 M elements) take 23.6 us, 5.8 TB/s -- part of them are still in the last-level cache.
template <typename T> __global__ __launch_bounds__(256) void grad_norm_kernel(NormArgs a) {
  const int ti = find_tensor(a.first, a.nt, blockIdx.x);
  const T *g = (const T *)a.g[ti];
  const int64_t lo = (int64_t)(blockIdx.x - a.first[ti]) * a.chunk;
  const int64_t hi = min(a.n[ti], lo + a.chunk);
  double s = 0.;
  for (int64_t e = lo + threadIdx.x * 4; e < hi; e += 1024 * 4) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {   // four independent loads in flight
      const int64_t ej = e + j * 1024;
      float o[4] = {0.f, 0.f, 0.f, 0.f};
      if (ej < hi) load4(g + ej, (int)min(hi - ej, (int64_t)4), o);
#pragma unroll
      for (int k = 0; k < 4; ++k) s = fma((double)o[k], (double)o[k], s);
    }
  }
  __shared__ double sh[4];
  s = block_sum<4>(s, sh);
  if (threadIdx.x == 0) a.part[blockIdx.x] = s;
}

__global__ __launch_bounds__(1024) void grad_norm_finish_kernel(const double *part, int n, float max_norm, float *out) {
  double s = 0.;
  for (int i = threadIdx.x; i < n; i += 1024) s += part[i];
  __shared__ double sh[16];
  s = block_sum<16>(s, sh);
  if (threadIdx.x == 0) {
    const double norm = sqrt(s);
    const bool ok = norm < INFINITY;   // false for NaN too
    out[0] = (float)norm;
    out[1] = ok ? (float)(norm > (double)max_norm ? (double)max_norm / norm : 1.) : NAN;
  }
}

// ------------------------------------------------------------------------------------------------------------ AdamW
struct AdamwHyper {   // what one step's launches share, written on the device: t may live in a captured graph
  float alpha, lr, gs;
  unsigned key;       // of this step's rounding
  int skip;
};

__global__ void adamw_begin_kernel(int *t, AdamwHyper *h, const float *lr_dev, float lr, const float *grad_scale, double b1,
                                   double b2, unsigned seed) {
  const float gs = grad_scale ? *grad_scale : 1.f;
  const bool skip = !(fabsf(gs) < INFINITY);
  if (lr_dev) lr = *lr_dev;
  const int n = *t + 1;
  if (!skip) *t = n;
  double p1 = 1., p2 = 1., q1 = b1, q2 = b2;
  for (unsigned e = (unsigned)n; e; e >>= 1) {   // b^n by squaring
    if (e & 1) { p1 *= q1; p2 *= q2; }
    q1 *= q1; q2 *= q2;
  }
  h->alpha = (float)((double)lr * sqrt(1. - p2) / (1. - p1));
  h->lr = lr;
  h->gs = gs;
  h->key = hash32(seed ^ hash32((unsigned)n));
  h->skip = skip;
}

struct AdamwArgs {
  void *p[OPT_T];
  const void *g[OPT_T];
  bf16 *copy[OPT_T];
  int64_t n[OPT_T], off[OPT_T];
  float wd[OPT_T];
  unsigned first[OPT_T];
  int nt;
  void *m, *v;
  float *ms, *vs;
  const AdamwHyper *h;
  float c1, c2, eps;   // 1 - b1, 1 - b2
};

__device__ __forceinline__ void adamw_elem(float &p, float g, float &m, float &v, const AdamwHyper &h, float c1, float c2,
                                           float eps, float lrwd) {
  g = g * h.gs;
  m = m + (g - m) * c1;
  v = v + (g * g - v) * c2;
  p = p - p * lrwd;
  // (hardware square root and reciprocal, one ulp each, subnormal v as zero: eps >= 1e-12 hides what that loses; the IEEE
  // sequences are a third of the 8-bit kernel's instructions)
  p = p - (h.alpha * m) * __builtin_amdgcn_rcpf(__builtin_amdgcn_sqrtf(v) + eps);
}

// fp32 state: one 16-byte vector per stream and thread.  HBM-bound: with fp32 tensors 16 B an element in, 12 out and 2 for a bf16 copy;
// 68.7 M elements with the copy (2.06 GB) take 390 us, 5.3 TB/s, a copy's rate.
template <typename TP, typename TG> __global__ __launch_bounds__(256) void adamw32_kernel(AdamwArgs a) {
  const int ti = find_tensor(a.first, a.nt, blockIdx.x);
  const AdamwHyper h = *a.h;
  if (h.skip) return;
  const int64_t n = a.n[ti], e0 = (int64_t)(blockIdx.x - a.first[ti]) * OPT_CHUNK;
  TP *p = (TP *)a.p[ti];
  const TG *g = (const TG *)a.g[ti];
  float *m = (float *)a.m + a.off[ti], *v = (float *)a.v + a.off[ti];
  bf16 *copy = a.copy[ti];
  const float lrwd = h.lr * a.wd[ti];
  auto four = [&](int64_t e, int left) {
    float pv[4], gv[4], mv[4], vv[4];
    load4(p + e, left, pv); load4(g + e, left, gv); load4(m + e, left, mv); load4(v + e, left, vv);
#pragma unroll
    for (int k = 0; k < 4; ++k) adamw_elem(pv[k], gv[k], mv[k], vv[k], h, a.c1, a.c2, a.eps, lrwd);
    store4(p + e, left, pv); store4(m + e, left, mv); store4(v + e, left, vv);
    if (copy) store4(copy + e, left, pv);
  };
  if (e0 + OPT_CHUNK <= n) {   // whole: no lane has a tail
#pragma unroll
    for (int j = 0; j < 4; ++j) four(e0 + j * 1024 + threadIdx.x * 4, 4);
  } else {
    for (int64_t e = e0 + threadIdx.x * 4; e < n; e += 1024) four(e, (int)min(n - e, (int64_t)4));
  }
}

// fp32 exponent field of the power of two that puts `bits` (a magnitude) at or under 1.75 * 2^top; the clamp keeps the
// scale a normal number
__device__ __forceinline__ int scale_field(unsigned bits, int top) {
  const int f = (int)((bits + 0x1fffffu) >> 23) - top;
  return f < 1 ? 1 : f;
}

// magnitude -> code: |x| / 2^e lands in the fp32 subnormals whose exponent field IS the code's (2^-shift aligns them), so
// normal and subnormal codes round the same way: add 16 random bits under the kept ones, drop the rest
template <int SHIFT, int DROP> __device__ __forceinline__ unsigned round_code(float x, int e, unsigned rnd16) {
  const unsigned z = __float_as_uint(ldexpf(fabsf(x), -(e + SHIFT)));
  return (z + (rnd16 << (DROP - 16))) >> DROP;
}

template <typename TP, typename TG, bool WHOLE> __device__ __forceinline__ void adamw8_block(const AdamwArgs &a, const AdamwHyper &h,
                                                                                               int ti, int64_t e0, int64_t n) {
  const int l = threadIdx.x & 15;
  TP *p = (TP *)a.p[ti];
  const TG *g = (const TG *)a.g[ti];
  const int64_t s0 = a.off[ti] + e0;   // position in the state (a multiple of 256)
  unsigned *mq = (unsigned *)((uint8_t *)a.m + s0), *vq = (unsigned *)((uint8_t *)a.v + s0);
  float *msp = a.ms + s0 / OPT_BLOCK, *vsp = a.vs + s0 / OPT_BLOCK;
  bf16 *copy = a.copy[ti];
  const float lrwd = h.lr * a.wd[ti];

  float pv[4][4], gv[4][4], mv[4][4], vv[4][4];
  int left[4];
  unsigned mc[4], vc[4];
  const float ms = *msp, vs = *vsp;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t e = e0 + j * 64 + l * 4;
    left[j] = WHOLE ? 4 : (int)max((int64_t)0, min(n - e, (int64_t)4));
    mc[j] = mq[j * 16 + l];            // (the state is padded to whole blocks)
    vc[j] = vq[j * 16 + l];
    load4(p + e, left[j], pv[j]);
    load4(g + e, left[j], gv[j]);
  }
  unsigned mmax = 0, vmax = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const f32x2 m01 = __builtin_amdgcn_cvt_pk_f32_fp8((int)mc[j], false), m23 = __builtin_amdgcn_cvt_pk_f32_fp8((int)mc[j], true);
    const f32x2 v01 = __builtin_amdgcn_cvt_pk_f32_bf8((int)vc[j], false), v23 = __builtin_amdgcn_cvt_pk_f32_bf8((int)vc[j], true);
    mv[j][0] = m01[0] * ms; mv[j][1] = m01[1] * ms; mv[j][2] = m23[0] * ms; mv[j][3] = m23[1] * ms;
    vv[j][0] = v01[0] * vs; vv[j][1] = v01[1] * vs; vv[j][2] = v23[0] * vs; vv[j][3] = v23[1] * vs;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      adamw_elem(pv[j][k], gv[j][k], mv[j][k], vv[j][k], h, a.c1, a.c2, a.eps, lrwd);
      mmax = max(mmax, __float_as_uint(fabsf(mv[j][k])));   // as integers: NaN is the largest of all
      vmax = max(vmax, __float_as_uint(fabsf(vv[j][k])));
    }
    store4(p + e0 + j * 64 + l * 4, left[j], pv[j]);
    if (copy) store4(copy + e0 + j * 64 + l * 4, left[j], pv[j]);
  }
  mmax = row16_umax(mmax);
  vmax = row16_umax(vmax);
  const bool mbad = mmax >= 0x7f800000u, vbad = vmax >= 0x7f800000u;
  const int mf = scale_field(mmax, 8), vf = scale_field(vmax, 15);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    unsigned mo = 0, vo = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const unsigned r = hash32((unsigned)(s0 + j * 64 + l * 4 + k) ^ h.key);
      const unsigned qm = round_code<120, 20>(mv[j][k], mf - 127, r & 0xffffu) | ((__float_as_uint(mv[j][k]) >> 24) & 0x80u);
      unsigned qv = round_code<112, 21>(vv[j][k], vf - 127, r >> 16);
      qv = max(qv, vv[j][k] > 0.f ? 1u : 0u);
      mo |= qm << (8 * k);
      vo |= qv << (8 * k);
    }
    mq[j * 16 + l] = mbad ? 0u : mo;
    vq[j * 16 + l] = vbad ? 0u : vo;
  }
  if (l == 0) {
    *msp = mbad ? NAN : __uint_as_float((unsigned)mf << 23);
    *vsp = vbad ? NAN : __uint_as_float((unsigned)vf << 23);
  }
}

// HBM-bound on large tensors: with fp32 tensors 10 B an element in, 8 out with the copy; 68.7 M elements (1.24 GB) take 226 us, 5.5 TB/s.  A
// workgroup without a ragged end takes the form without tail checks.
template <typename TP, typename TG> __global__ __launch_bounds__(256) void adamw8_kernel(AdamwArgs a) {
  const int ti = find_tensor(a.first, a.nt, blockIdx.x);
  const AdamwHyper h = *a.h;
  if (h.skip) return;
  const int64_t n = a.n[ti], w0 = (int64_t)(blockIdx.x - a.first[ti]) * OPT_CHUNK + (threadIdx.x >> 6) * 1024;
  const int64_t e0 = w0 + ((threadIdx.x & 63) >> 4) * OPT_BLOCK;
  if (w0 + 1024 <= n) adamw8_block<TP, TG, true>(a, h, ti, e0, n);
  else if (e0 < n) adamw8_block<TP, TG, false>(a, h, ti, e0, n);   // (a row of 16 lanes stays or leaves together)
}

// elements per workgroup of the norm: whole rounds of 4 096, at most ~2 048 workgroups (the last kernel adds their sums)
static int64_t norm_chunk(const int64_t *n, int count) {
  int64_t total = 0;
  for (int i = 0; i < count; ++i) total += n[i];
  const int64_t c = (total / 2048 + 4095) / 4096 * 4096;
  return c < 4096 ? 4096 : c;
}
static int64_t norm_blocks(const int64_t *n, int count, int64_t chunk) {
  int64_t b = 0;
  for (int i = 0; i < count; ++i) b += (n[i] + chunk - 1) / chunk;
  return b;
}

}  // namespace cfd

using namespace cfd;

extern "C" int64_t cfd_grad_norm_workspace_bytes(const int64_t *n, int count) {
  CFD_REQUIRE(count >= 0 && (n || !count), "bad arguments");
  for (int i = 0; i < count; ++i) CFD_REQUIRE(n[i] >= 0, "tensor %d: negative length", i);
  return 8 * (norm_blocks(n, count, norm_chunk(n, count)) + 1);
}

extern "C" int cfd_grad_norm(const void *const *g, const int64_t *n, int count, int dtype, float max_norm, void *ws, float *out,
                             void *stream) {
  CFD_REQUIRE(count >= 0 && (count == 0 || (g && n)) && ws && out, "bad arguments");
  CFD_REQUIRE(dtype == CFD_F32 || dtype == CFD_BF16, "bad dtype");
  CFD_REQUIRE(max_norm > 0.f, "max_norm must be positive");
  for (int i = 0; i < count; ++i) CFD_REQUIRE(n[i] >= 0 && (g[i] || !n[i]), "tensor %d: NULL pointer or negative length", i);
  const int64_t chunk = norm_chunk(n, count), blocks = norm_blocks(n, count, chunk);
  CFD_REQUIRE(blocks <= 0xffffff, "too many elements");
  hipStream_t st = (hipStream_t)stream;
  int64_t done = 0;
  for (int i = 0; i < count;) {
    NormArgs a;
    a.nt = 0; a.chunk = chunk; a.part = (double *)ws + done;
    unsigned grid = 0;
    for (; i < count && a.nt < OPT_T; ++i) {
      if (!n[i]) continue;
      a.g[a.nt] = g[i]; a.n[a.nt] = n[i]; a.first[a.nt] = grid;
      grid += (unsigned)((n[i] + chunk - 1) / chunk);
      ++a.nt;
    }
    if (!grid) break;
    if (dtype == CFD_BF16) hipLaunchKernelGGL(grad_norm_kernel<bf16>, dim3(grid), dim3(256), 0, st, a);
    else hipLaunchKernelGGL(grad_norm_kernel<float>, dim3(grid), dim3(256), 0, st, a);
    CFD_LAUNCH_CHECK();
    done += grid;
  }
  hipLaunchKernelGGL(grad_norm_finish_kernel, dim3(1), dim3(1024), 0, st, (const double *)ws, (int)done, max_norm, out);
  CFD_LAUNCH_CHECK();
  return CFD_OK;
}

extern "C" int cfd_adamw_step(const cfd_adamw_tensor *t, int count, const cfd_adamw_desc *d, void *m, void *v, float *m_scale,
                              float *v_scale, int *step, const float *lr_device, const float *grad_scale, void *ws,
                              void *stream) {
  CFD_REQUIRE(t && count > 0 && d && m && v && step && ws, "bad arguments");
  CFD_REQUIRE(d->state_bits == 32 || (d->state_bits == 8 && m_scale && v_scale), "state_bits must be 32, or 8 with scales");
  CFD_REQUIRE((d->p_dtype == CFD_F32 || d->p_dtype == CFD_BF16) && (d->g_dtype == CFD_F32 || d->g_dtype == CFD_BF16), "bad dtype");
  CFD_REQUIRE(d->beta1 >= 0. && d->beta1 < 1. && d->beta2 >= 0. && d->beta2 < 1. && d->eps >= 1e-12f, "beta must be in [0, 1), eps at least 1e-12");
  CFD_REQUIRE(d->state_bits == 32 || (d->beta1 <= 0.9999 && d->beta2 <= 0.9999), "beta must be at most 0.9999 with an 8-bit state");
  CFD_REQUIRE((((uintptr_t)m | (uintptr_t)v) & 15) == 0, "state must be 16-byte aligned");
  int64_t blocks = 0;
  for (int i = 0; i < count; ++i) {
    CFD_REQUIRE(t[i].n >= 0 && (!t[i].n || (t[i].p && t[i].g)), "tensor %d: NULL pointer or negative length", i);
    CFD_REQUIRE(t[i].state_offset >= 0 && t[i].state_offset % OPT_BLOCK == 0, "tensor %d: state offset must be a multiple of 256", i);
    CFD_REQUIRE(!t[i].copy || d->p_dtype == CFD_F32, "tensor %d: a bf16 copy needs an fp32 parameter", i);
    blocks += (t[i].n + OPT_CHUNK - 1) / OPT_CHUNK;
  }
  CFD_REQUIRE(blocks <= 0xffffff, "too many elements");
  hipStream_t st = (hipStream_t)stream;
  AdamwHyper *h = (AdamwHyper *)ws;
  hipLaunchKernelGGL(adamw_begin_kernel, dim3(1), dim3(1), 0, st, step, h, lr_device, d->lr, grad_scale, d->beta1, d->beta2, d->seed);
  CFD_LAUNCH_CHECK();
  for (int i = 0; i < count;) {
    AdamwArgs a;
    a.nt = 0; a.m = m; a.v = v; a.ms = m_scale; a.vs = v_scale; a.h = h;
    a.c1 = (float)(1. - d->beta1); a.c2 = (float)(1. - d->beta2); a.eps = d->eps;
    unsigned grid = 0;
    for (; i < count && a.nt < OPT_T; ++i) {
      if (!t[i].n) continue;
      const int k = a.nt++;
      a.p[k] = t[i].p; a.g[k] = t[i].g; a.copy[k] = (bf16 *)t[i].copy;
      a.n[k] = t[i].n; a.off[k] = t[i].state_offset; a.wd[k] = t[i].weight_decay; a.first[k] = grid;
      grid += (unsigned)((t[i].n + OPT_CHUNK - 1) / OPT_CHUNK);
    }
    if (!grid) break;
#define ADAMW(K, TP, TG) hipLaunchKernelGGL((K<TP, TG>), dim3(grid), dim3(256), 0, st, a)
#define ADAMW_T(K)                                                    \
    if (d->p_dtype == CFD_F32 && d->g_dtype == CFD_F32) ADAMW(K, float, float); \
    else if (d->p_dtype == CFD_F32) ADAMW(K, float, bf16);            \
    else if (d->g_dtype == CFD_F32) ADAMW(K, bf16, float);            \
    else ADAMW(K, bf16, bf16);
    if (d->state_bits == 8) { ADAMW_T(adamw8_kernel) } else { ADAMW_T(adamw32_kernel) }
#undef ADAMW_T
#undef ADAMW
    CFD_LAUNCH_CHECK();
  }
  return CFD_OK;
}
