// 4-bit microscaled storage (OCP MX: E2M1 codes, one E8M0 power of two for 32 of them) and the Dense layer on it.
//
// A matrix of R rows x K columns, blocked along K: codes [R][16 nb] bytes (nb = ceil(K / 32); the low nibble is the lower
// column), scales [R][16 ceil(nb / 16)] bytes.  Codes past K are zero, scale bytes past nb are 0 (2^-127 x 0): a
// contraction may run over whole blocks and whole 512-column groups without masks.
//
// Quantisation: e = floor(log2 max|x|) - 2, one more where max|x| > 7 * 2^e, so that no element is off by more than half
// a spacing at its block's top (the plain floor would clip a block's largest values by up to a quarter); codes round to
// nearest even.  A block with an infinity or NaN gets the scale 0xFF: the whole block reads as NaN.
#include "common.h"
#include "igemm256.h"
#include <type_traits>

namespace cfd {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef __bf16 bf16x8a2 __attribute__((ext_vector_type(8), aligned(2)));

// threads of a launch per matrix row: a 64-bit division by it would be most of a streaming kernel's instructions
struct FastDiv {
  unsigned d, c[3];
  explicit FastDiv(unsigned v) : d(v) { fastdiv_make(v, c); }
  __device__ __forceinline__ unsigned div(unsigned n) const { return (unsigned)fastdiv((int)n, c); }
};
constexpr int64_t MX_GRID = 0xffffff;   // workgroups of 256 threads, under 2^32 threads in all

static inline int64_t mx_blocks(int64_t k) { return (k + 31) / 32; }
static inline int64_t mx_scale_pitch(int64_t k) { return (mx_blocks(k) + 15) / 16 * 16; }

// eight consecutive values at element alignment; `left` of them exist, the rest read as zero
__device__ __forceinline__ void load8(const float *p, int left, float (&o)[8]) {
  if (left >= 8) {
    const f32x4a4 a = *(const f32x4a4 *)p, b = *(const f32x4a4 *)(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) { o[i] = a[i]; o[4 + i] = b[i]; }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = i < left ? p[i] : 0.f;
  }
}
__device__ __forceinline__ void load8(const bf16 *p, int left, float (&o)[8]) {
  if (left >= 8) {
    const bf16x8a2 a = *(const bf16x8a2 *)p;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = (float)a[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = i < left ? (float)p[i] : 0.f;
  }
}

// E8M0 byte of a block whose largest magnitude has these bits (NaN compares largest)
__device__ __forceinline__ unsigned mx_scale_byte(unsigned amax) {
  if (amax >= 0x7f800000u) return 255u;
  const int f = (int)((amax + 0x1fffffu) >> 23) - 2;   // mantissa over 1.75 carries into the exponent
  return f < 0 ? 0u : (unsigned)f;
}
// the hardware conversions take the scale as an fp32 power of two; a byte of 0 is the subnormal 2^-127
__device__ __forceinline__ float mx_scale_f32(unsigned byte) {
  return __uint_as_float(max(byte << 23, 0x00400000u));
}
__device__ __forceinline__ unsigned mx_code8(const float (&x)[8], unsigned byte) {
  const float s = mx_scale_f32(byte);
  unsigned c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[0], x[1], s, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[2], x[3], s, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[4], x[5], s, 2);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[6], x[7], s, 3);
  return byte == 255u ? 0u : c;
}
__device__ __forceinline__ unsigned amax8(const float (&x)[8]) {
  unsigned a = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) a = max(a, __float_as_uint(x[i]) & 0x7fffffffu);
  return a;
}
__device__ __forceinline__ unsigned quad_umax(unsigned v) {
  v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, false));   // lane ^ 1
  return max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, false));  // lane ^ 2
}

// the same for eight bf16 as they lie in memory (four words): two magnitudes a comparison, and no way through fp32
__device__ __forceinline__ unsigned pk_max_u16(unsigned a, unsigned b) {
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
__device__ __forceinline__ unsigned amax8(const i32x4 &w) {
  const unsigned m = pk_max_u16(pk_max_u16((unsigned)w[0] & 0x7fff7fffu, (unsigned)w[1] & 0x7fff7fffu),
                                pk_max_u16((unsigned)w[2] & 0x7fff7fffu, (unsigned)w[3] & 0x7fff7fffu));
  return max(m & 0xffff0000u, m << 16);
}
__device__ __forceinline__ bf16x2 two_bf16(int w) { return __builtin_bit_cast(bf16x2, w); }   // (of a copy: not of a vector's element)
__device__ __forceinline__ unsigned mx_code8(const i32x4 &w, unsigned byte) {
  const float s = mx_scale_f32(byte);
  unsigned c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, two_bf16(w[0]), s, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, two_bf16(w[1]), s, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, two_bf16(w[2]), s, 2);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, two_bf16(w[3]), s, 3);
  return byte == 255u ? 0u : c;
}
// eight values as the quantisation works on them: fp32 as numbers, bf16 as words
template <typename T> struct Eight;
template <> struct Eight<float> {
  float v[8];
  __device__ __forceinline__ void load(const float *p) {
    const f32x4a4 a = *(const f32x4a4 *)p, b = *(const f32x4a4 *)(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[4 + i] = b[i]; }
  }
  __device__ __forceinline__ void load(const float *p, int left) { load8(p, left, v); }
  __device__ __forceinline__ void to_lds(unsigned *d) const {
    *(f32x4 *)d = (f32x4){v[0], v[1], v[2], v[3]};
    *(f32x4 *)(d + 4) = (f32x4){v[4], v[5], v[6], v[7]};
  }
  __device__ __forceinline__ const float (&get() const)[8] { return v; }
};
typedef int i32x4a2 __attribute__((ext_vector_type(4), aligned(2)));
template <> struct Eight<bf16> {
  i32x4 w;
  __device__ __forceinline__ void load(const bf16 *p) { w = *(const i32x4a2 *)p; }
  __device__ __forceinline__ void load(const bf16 *p, int left) {
    if (left >= 8) { load(p); return; }
    unsigned short h[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = i < left ? ((const unsigned short *)p)[i] : (unsigned short)0;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = (int)(h[2 * i] | ((unsigned)h[2 * i + 1] << 16));
  }
  __device__ __forceinline__ void to_lds(unsigned *d) const { *(i32x4 *)d = w; }
  __device__ __forceinline__ const i32x4 &get() const { return w; }
};

// one lane stores four consecutive scale bytes from block b on (bytes of blocks that are not there are zero), and the zeros
// behind them if they are the row's last
__device__ __forceinline__ void put_scales4(uint8_t *row, int b, int nb, int pitch, unsigned bytes) {
  *(unsigned *)(row + b) = bytes;
  if (b + 4 >= nb)
    for (int i = b + 4; i < pitch; i += 4) *(unsigned *)(row + i) = 0u;
}
// the four scale bytes that a row of 16 lanes holds, one per quad
__device__ __forceinline__ unsigned row16_bytes(unsigned byte) {
  unsigned v = byte << (((threadIdx.x >> 2) & 3) * 8);
  v |= (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xf, 0xf, false);
  return v | (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, false);
}
__device__ __forceinline__ unsigned quad_bytes(unsigned byte) {   // the same over the four lanes of a quad
  unsigned v = byte << ((threadIdx.x & 3) * 8);
  v |= (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, false);
  return v | (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, false);
}

// rows only: four lanes share a block of 32 (eight columns each): 32-byte / 16-byte loads, 4-byte stores, the block's
// maximum in two DPP steps.  HBM-bound, 2 (bf16) or 4 bytes in and 0.53 out an element: 64 x 262144 bf16 (42.5 MB) take 8.8 us,
// 4.8 TB/s.  A row is walked in multiples of 128 columns, so that 16 lanes hold four whole scale bytes.
template <typename T> __global__ __launch_bounds__(256) void mx_quant_rows_kernel(const T *x, int64_t ldx, int64_t rows, int K,
                                                                                   int nb, int pitch, uint8_t *codes,
                                                                                   uint8_t *scales, FastDiv G) {
  const unsigned t = blockIdx.x * 256 + threadIdx.x;       // (the host keeps the grid under 2^32 threads)
  const int64_t row = G.div(t);
  if (row >= rows) return;                // (whole rows of 16 lanes: G is a multiple of 16)
  const int grp = (int)(t - (unsigned)row * G.d);
  Eight<T> v;
  v.load(x + row * ldx + (int64_t)grp * 8, K - grp * 8);
  const unsigned byte = mx_scale_byte(quad_umax(amax8(v.get())));
  if ((grp >> 2) < nb) *(unsigned *)(codes + row * nb * 16 + (int64_t)grp * 4) = mx_code8(v.get(), byte);
  const unsigned bytes = row16_bytes(byte);
  if ((grp & 15) == 0) put_scales4(scales + row * pitch, grp >> 2, nb, pitch, bytes);
}

// both orientations from one read: a 128 x 128 tile; rows are coded on the way in, columns from LDS, two adjacent columns and 32
// rows a thread.  LDS words are swizzled by 16 per 32 rows: the four row blocks that a quad of lanes reads lie in different banks.
// Codes leave as 64 contiguous bytes a row in both orientations.  Near a copy's rate where there are tiles for several rounds (8192 x 4096
// fp32, 170 MB: 33 us, 5.1 TB/s); one round fills and drains the chip in ~4 us beside the bytes' time (4090 x 4102, 85 MB: 22.1 us).
constexpr int QT = 128;
template <typename T> __global__ __launch_bounds__(256) void mx_quant_both_kernel(const T *x, int64_t ldx, int R, int K,
                                                                                   int nb, int pitch, uint8_t *codes,
                                                                                   uint8_t *scales, int nbt, int pitch_t,
                                                                                   uint8_t *codes_t, uint8_t *scales_t, int tx) {
  constexpr int W = QT * (int)sizeof(T) / 4;       // words of a tile row
  __shared__ __attribute__((aligned(16))) unsigned tile[QT * W];
  // runs of four neighbouring tiles go to one XCD (workgroups alternate over the eight): the parts of a cache line that they write
  // meet in one L2 (fp32 4090 x 4102: 26.6 -> 22.6 us; long runs instead set the XCDs a power of two apart: 30 -> 39 us at 4096 x 8192)
  const int nwg = gridDim.x, wg = blockIdx.x, t = wg < (nwg & ~31) ? (wg & ~31) + (wg & 7) * 4 + ((wg >> 3) & 3) : wg;
  const int r0 = t / tx * QT, c0 = t % tx * QT;
  const int tid = threadIdx.x, c = (tid & 15) * 8;
  auto put = [&](int i, const Eight<T> &v) {       // eight values of a row into LDS, coded along the row
    const int r = i * 16 + (tid >> 4);
    v.to_lds(tile + r * W + ((c * (int)sizeof(T) / 4) ^ ((r >> 5) * 16)));
    if (codes) {
      const unsigned byte = mx_scale_byte(quad_umax(amax8(v.get()))), bytes = row16_bytes(byte);
      const int b = (c0 + c) >> 5;
      if (r0 + r < R) {
        if (b < nb) *(unsigned *)(codes + (int64_t)(r0 + r) * nb * 16 + (c0 + c) / 2) = mx_code8(v.get(), byte);
        if ((tid & 15) == 0) put_scales4(scales + (int64_t)(r0 + r) * pitch, b, nb, pitch, bytes);
      }
    }
  };
  const T *src0 = x + (int64_t)(r0 + (tid >> 4)) * ldx + c0 + c;
  if (r0 + QT <= R && c0 + QT <= K) {              // a whole tile: eight loads in flight
    Eight<T> v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i].load(src0 + i * 16 * ldx);
    const int sw = tid >> 4;
    if (codes) {       // (no element is past an end: half the instructions of `put`: 4096 x 4096 bf16 15.2 -> 14.2 us)
      uint8_t *const to = codes + (int64_t)(r0 + sw) * nb * 16 + (c0 + c) / 2;
      unsigned bytes[2] = {0, 0};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i].to_lds(tile + (i * 16 + sw) * W + ((c * (int)sizeof(T) / 4) ^ ((i >> 1) * 16)));
        const unsigned byte = mx_scale_byte(quad_umax(amax8(v[i].get())));
        *(unsigned *)(to + (int64_t)i * nb * 256) = mx_code8(v[i].get(), byte);
        bytes[i >> 2] |= byte << (8 * (i & 3));
      }
      // the four lanes of a block hold its byte of eight rows: each stores two of them
      uint8_t *const sc = scales + (int64_t)(r0 + (tid & 3) * 16 + sw) * pitch + ((c0 + c) >> 5);
      sc[0] = (uint8_t)(bytes[0] >> (8 * (tid & 3)));
      sc[(int64_t)64 * pitch] = (uint8_t)(bytes[1] >> (8 * (tid & 3)));
      if (c0 + QT == K)      // the zeros behind the last block
        for (int i = nb + (tid & 1) * 4; i < pitch; i += 8) *(unsigned *)(scales + (int64_t)(r0 + (tid >> 1)) * pitch + i) = 0u;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i].to_lds(tile + (i * 16 + sw) * W + ((c * (int)sizeof(T) / 4) ^ ((i >> 1) * 16)));
    }
  } else {
    for (int i = 0; i < 8; ++i) {
      Eight<T> v;
      v.load(src0 + i * 16 * ldx, r0 + i * 16 + (tid >> 4) < R ? K - c0 - c : 0);
      put(i, v);
    }
  }
  __syncthreads();
  const int rb = tid & 3, cc = (tid >> 2) * 2, bt = (r0 >> 5) + rb;    // this thread's row block and two columns
  const unsigned *src = tile + rb * 32 * W + ((cc * (int)sizeof(T) / 4) ^ (rb * 16));
  Eight<T> v[2][4];
  unsigned am[2] = {0, 0};
#pragma unroll
  for (int g = 0; g < 4; ++g) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const unsigned *w0 = src + (g * 8 + i) * W, *w1 = w0 + W;
      if constexpr (sizeof(T) == 2) {              // two rows of two columns -> two columns of two rows
        v[0][g].w[i / 2] = (int)__builtin_amdgcn_perm(*w1, *w0, 0x05040100u);
        v[1][g].w[i / 2] = (int)__builtin_amdgcn_perm(*w1, *w0, 0x07060302u);
      } else {
        const f32x2 p0 = *(const f32x2 *)w0, p1 = *(const f32x2 *)w1;
        v[0][g].v[i] = p0[0]; v[1][g].v[i] = p0[1];
        v[0][g].v[i + 1] = p1[0]; v[1][g].v[i + 1] = p1[1];
      }
    }
    am[0] = max(am[0], amax8(v[0][g].get()));
    am[1] = max(am[1], amax8(v[1][g].get()));
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const unsigned byte = mx_scale_byte(am[k]), bytes = quad_bytes(byte);
    const int64_t col = c0 + cc + k;
    if (col >= K) continue;
    i32x4 o;
#pragma unroll
    for (int g = 0; g < 4; ++g) o[g] = (int)mx_code8(v[k][g].get(), byte);
    if (bt < nbt) *(i32x4 *)(codes_t + col * nbt * 16 + bt * 16) = o;
    if (rb == 0) put_scales4(scales_t + col * pitch_t, bt, nbt, pitch_t, bytes);
  }
}

__device__ __forceinline__ bf16x8 mx_bf16x8(unsigned c, float s) {     // eight codes times their scale
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 1);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 2), e = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 3);
  return (bf16x8){a[0], a[1], b[0], b[1], d[0], d[1], e[0], e[1]};
}
__device__ __forceinline__ float mx_scale_or_nan(unsigned byte) { return byte == 255u ? __uint_as_float(0x7fc00000u) : mx_scale_f32(byte); }

// codes -> values (exact, or an overflow to infinity at the top of the scale's range): a lane reads eight codes and writes 16 (bf16)
// or 32 (fp32) bytes.  HBM-bound: 64 x 262144 to bf16 (42.5 MB) 8.8 us, 4.8 TB/s.
template <typename T> __global__ __launch_bounds__(256) void mx_dequant_kernel(const uint8_t *codes, const uint8_t *scales,
                                                                                int64_t rows, int K, int nb, int pitch, T *y,
                                                                                int64_t ldy, FastDiv G) {
  const unsigned t = blockIdx.x * 256 + threadIdx.x;
  const int64_t row = G.div(t);
  if (row >= rows) return;
  const int grp = (int)(t - (unsigned)row * G.d), left = K - grp * 8;
  const unsigned c = *(const unsigned *)(codes + row * nb * 16 + (int64_t)grp * 4);
  const float s = mx_scale_or_nan(scales[row * pitch + (grp >> 2)]);
  T *o = y + row * ldy + (int64_t)grp * 8;
  if constexpr (sizeof(T) == 2) {
    const bf16x8 v = mx_bf16x8(c, s);
    if (left >= 8) *(bf16x8a2 *)o = v;
    else
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < left) o[i] = v[i];
  } else {
    const f32x2 p[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 0), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 1),
                        __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 2), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 3)};
    if (left >= 8) {
      *(f32x4a4 *)o = (f32x4){p[0][0] * s, p[0][1] * s, p[1][0] * s, p[1][1] * s};
      *(f32x4a4 *)(o + 4) = (f32x4){p[2][0] * s, p[2][1] * s, p[3][0] * s, p[3][1] * s};
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < left) o[i] = p[i >> 1][i & 1] * s;
    }
  }
}

// ---------------------------------------------------------------------------------------------------------- products
struct MxDense {
  const uint8_t *xc, *xs, *wc, *ws;   // 4-bit operands: activations (M rows), weights (N rows)
  const void *x;                      // or float activations
  int64_t ldx;
  const float *bias;
  void *y;
  int64_t ldy;
  float *slab;                        // [split][M][N] partial sums (split > 1)
  int M, N, K, nb, pitch;
  int split, kt_per;                  // K groups (256 or 512 columns) per split
  int mt, nt;
  int out_bf16, act;
  float slope;
  int kwaves;                         // float activations: waves of a workgroup that share a weight tile
  int xrows;                          //   and activation rows of a tile
  bool big;                           // 256 x 256 tiles
  bool pairs;                         //   bf16 output: two columns are one aligned word
};

// activation of a sum.  ReLU by comparison, not by a slope of zero: a sum of -infinity is 0 (its product with zero would be NaN), and NaN stays
__device__ __forceinline__ float mx_relu(float v) { return v < 0.f ? 0.f : v; }
__device__ __forceinline__ float mx_act(const MxDense &p, float v) {   // (without a branch between the linear kinds)
  if (p.act == CFD_ACT_SIGMOID) return 1.f / (1.f + __expf(-v));
  const float ns = act_neg_scale(p.act, p.slope), lo = p.act == CFD_ACT_RELU ? 0.f : -INFINITY;
  return v < 0.f ? fmaxf(v, lo) * ns : v;
}
__device__ __forceinline__ void mx_store(const MxDense &p, int64_t m, int n, float v) {   // one element of the output
  if (p.out_bf16) ((bf16 *)p.y)[m * p.ldy + n] = (bf16)v;
  else ((float *)p.y)[m * p.ldy + n] = v;
}
// lane's four consecutive outputs n..n+3 of row m
__device__ __forceinline__ void mx_emit(const MxDense &p, int sk, int64_t m, int n, f32x4 v) {
  if (m >= p.M || n >= p.N) return;
  if (p.split > 1) {
    float *o = p.slab + ((int64_t)sk * p.M + m) * p.N + n;
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (n + r < p.N) o[r] = v[r];
    return;
  }
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (n + r < p.N) mx_store(p, m, n + r, mx_act(p, v[r] + (p.bias ? p.bias[n + r] : 0.f)));
}

// sums of the split slabs, bias, activation, output type: 16 lanes take 64 consecutive outputs, 16 groups of lanes take the
// slabs in turn (every load of a thread in flight at once: one thread per output and a loop over 128 slabs took 31 us for
// 256 outputs) and join in LDS.  The order is fixed: same inputs, same bits.
__global__ __launch_bounds__(256) void mx_split_sum_kernel(MxDense p) {
  __shared__ f32x4 part[16][16];
  const int l = threadIdx.x & 15, g = threadIdx.x >> 4;
  const int64_t MN = (int64_t)p.M * p.N, i = (int64_t)blockIdx.x * 64 + l * 4;
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  if (i + 4 <= MN) {
#pragma unroll 8
    for (int k = g; k < p.split; k += 16) s += *(const f32x4a4 *)(p.slab + k * MN + i);
  } else {
    for (int k = g; k < p.split; k += 16)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i + e < MN) s[e] += p.slab[k * MN + i + e];
  }
  part[g][l] = s;
  __syncthreads();
  if (g >= 4) return;
  const int64_t o = (int64_t)blockIdx.x * 64 + threadIdx.x;   // one output a thread
  if (o >= MN) return;
  float v = 0.f;
#pragma unroll
  for (int k = 0; k < 16; ++k) v += part[k][threadIdx.x >> 2][threadIdx.x & 3];
  const int64_t m = o / p.N;
  const int n = (int)(o - m * p.N);
  mx_store(p, m, n, mx_act(p, v + (p.bias ? p.bias[n] : 0.f)));
}

constexpr unsigned MX_OOB = 0x80000000u;
__device__ __forceinline__ i32x4 ld16(__amdgpu_buffer_rsrc_t r, unsigned off) {
  return __builtin_amdgcn_raw_buffer_load_b128(r, (int)off, 0, 0);
}
__device__ __forceinline__ i32x8 wide(i32x4 a) { return (i32x8){a[0], a[1], a[2], a[3], 0, 0, 0, 0}; }
__device__ __forceinline__ __amdgpu_buffer_rsrc_t mx_rsrc(const uint8_t *base, int64_t row0, int rows, int64_t pitch) {
  // tile-relative: rows past the operand fall out of range and read as zero, and no offset needs more than 31 bits
  // (the size is uniform, but min() is formed in vector registers: without saying so every load goes through a loop over lanes)
  return __builtin_amdgcn_make_buffer_rsrc((void *)(base + row0 * pitch), 0, __builtin_amdgcn_readfirstlane((int)(rows * pitch)), 0x00020000);
}

// tile of a workgroup: each XCD (it has its own L2) gets a contiguous run of them; the tiles of one K slice follow each other
__device__ __forceinline__ void mx_small_tile(const MxDense &p, int &mt, int &nt, int &sk) {
  const int nwg = p.mt * p.nt * p.split, q = nwg >> 3, r = nwg & 7, xcd = blockIdx.x & 7;
  int t = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + ((int)blockIdx.x >> 3);
  mt = t % p.mt; t /= p.mt;
  nt = t % p.nt;
  sk = __builtin_amdgcn_readfirstlane(t / p.nt);
  mt = __builtin_amdgcn_readfirstlane(mt);
  nt = __builtin_amdgcn_readfirstlane(nt);
}

// LDS-DMA: lane l's 16 bytes land at dst + 16 l.  Matrix fragments come this way rather than straight into registers: their lanes
// want 16 different rows, and neighbouring lanes in different rows make a request each (77 a load instruction: 128 x 262144 x 256 took
// 30.9 us in all that way, 20.4 this way), while here neighbouring lanes take neighbouring 16 bytes.
__device__ __forceinline__ void mx_dma16(__amdgpu_buffer_rsrc_t r, unsigned voff, unsigned soff, char *dst) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void *)dst, 16, (int)voff, (int)soff, 0, 0);
}
template <int N> __device__ __forceinline__ void mx_wait() {   // until at most N vector-memory operations are in flight
  static_assert(N == 0 || N == 8 || N == 10 || N == 13 || N == 16 || N == 18, "counts that the schedules use");
  if constexpr (N == 0) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  else if constexpr (N == 8) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
  else if constexpr (N == 10) asm volatile("s_waitcnt vmcnt(10)" ::: "memory");
  else if constexpr (N == 13) asm volatile("s_waitcnt vmcnt(13)" ::: "memory");
  else if constexpr (N == 16) asm volatile("s_waitcnt vmcnt(16)" ::: "memory");
  else asm volatile("s_waitcnt vmcnt(18)" ::: "memory");
}
__device__ __forceinline__ void mx_wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// Both operands in 4 bits, small or long products (bound by reading them): a workgroup owns 64 (m) x 64 (n), its four waves take
// K groups of 512 columns in turn and join in LDS.  Every wave streams for itself, without barriers: a half group (256 columns, 8 KiB
// of each operand) in two stages, the 16 scale bytes a row of a group in two more; the next half is under way while this one
// multiplies.  16x16x128 scaled MFMA: lane = row l & 15, step s takes block 4s + (l >> 4), a lane shifts its scale byte down.
// Chunks are XOR-ed with bits 1-3 of the row (see the 256 x 256 kernel).  Codes behind the last column (the next row's) need no
// mask: their scale bytes are zero on both operands, 2^-254 is zero in fp32.  128 x 262144 x 256 (53.5 MB): 16.7 us, 3.2 TB/s; its 32 slices
// are summed in 3.9 us more.  A K of 512 columns or fewer is one group and one wave's: 64 x 256 x 262144 to bf16 (69 MB) takes 90 us.
constexpr int MXD_OPER = 64 * 128, MXD_STAGE = 2 * MXD_OPER, MXD_WAVE = 2 * MXD_STAGE + 2 * 2048, MXD_LDS = 4 * MXD_WAVE;   // 144 KiB
__global__ __launch_bounds__(256, 1) void mx_dense_kernel(MxDense p) {
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  int mt, nt, sk;
  mx_small_tile(p, mt, nt, sk);
  const int lane = threadIdx.x & 63, fr = lane & 15, fq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m0 = mt * 64, n0 = nt * 64, cp = p.nb * 16;
  const int mr = min(64, p.M - m0), nr = min(64, p.N - n0);
  const __amdgpu_buffer_rsrc_t xr = mx_rsrc(p.xc, m0, mr, cp), wr = mx_rsrc(p.wc, n0, nr, cp);
  const __amdgpu_buffer_rsrc_t xsr = mx_rsrc(p.xs, m0, mr, p.pitch), wsr = mx_rsrc(p.ws, n0, nr, p.pitch);
  char *const my = lds + wave * MXD_WAVE;
  const unsigned lrow = lane >> 3;
  auto issue = [&](int kt, int half) {            // 16 loads: 8 rows of 128 bytes each (rows past the operand read as zero)
    const unsigned at = (unsigned)kt * 256 + half * 128;
    char *dst = my + half * MXD_STAGE;
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const unsigned row = q * 8 + lrow, off = row * cp + (((lane & 7) ^ ((row >> 1) & 7)) << 4) + at;
      mx_dma16(wr, off, 0, dst + q * 1024);
      mx_dma16(xr, off, 0, dst + MXD_OPER + q * 1024);
    }
  };
  auto issue_scales = [&](int kt, int stage) {
    const unsigned off = (unsigned)(lane * p.pitch + kt * 16);
    mx_dma16(wsr, off, 0, my + 2 * MXD_STAGE + stage);
    mx_dma16(xsr, off, 0, my + 2 * MXD_STAGE + stage + 1024);
  };
  f32x4 acc[4][4] = {};
  auto multiply = [&](int half, int stage, auto next) {     // `next` starts the loads that may overwrite what has been read
    i32x4 a[4][2], b[4][2];
    int sa[4][2], sb[4][2];
    const char *src = my + half * MXD_STAGE + fr * 128, *sc = my + 2 * MXD_STAGE + stage + fr * 16 + half * 8;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int chunk = ((4 * s + fq) ^ ((fr >> 1) & 7)) << 4;
        a[i][s] = *(const i32x4 *)(src + i * 2048 + chunk);
        b[i][s] = *(const i32x4 *)(src + MXD_OPER + i * 2048 + chunk);
        sa[i][s] = *(const int *)(sc + i * 256 + s * 4);
        sb[i][s] = *(const int *)(sc + 1024 + i * 256 + s * 4);
      }
    mx_wait_lds();
    next();
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        sa[i][s] = (int)((unsigned)sa[i][s] >> (8 * fq));
        sb[i][s] = (int)((unsigned)sb[i][s] >> (8 * fq));
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide(a[i][s]), wide(b[j][s]), acc[i][j], 4, 4, 0, sa[i][s], 0, sb[j][s]);
    }
  };
  const int k1 = min((sk + 1) * p.kt_per, p.pitch / 16);
  int kt = sk * p.kt_per + wave, stage = 0;
  if (kt < k1) {
    issue_scales(kt, 0);
    issue(kt, 0);
    issue(kt, 1);
    for (; kt < k1; kt += 4) {     // (behind the slice's end the next group is loaded all the same: the counts stay, nobody reads it)
      mx_wait<16>();               // this group's scales and first half; its second half is in flight
      multiply(0, stage, [&] { issue_scales(kt + 4, stage ^ 2048); issue(kt + 4, 0); });
      mx_wait<18>();               // the second half; the next group's scales and first half are in flight
      multiply(1, stage, [&] { issue(kt + 4, 1); });
      stage ^= 2048;
    }
    mx_wait<0>();                  // (the tail loads must not land in what follows)
  }
  __syncthreads();
  f32x4 (*const part)[16][64] = (f32x4 (*)[16][64])lds;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) part[wave][i * 4 + j][lane] = acc[i][j];
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 4; ++j) {     // wave i sums weight rows i * 16 .. + 15
    f32x4 t = part[0][wave * 4 + j][lane];
#pragma unroll
    for (int w = 1; w < 4; ++w) t += part[w][wave * 4 + j][lane];
    mx_emit(p, sk, m0 + j * 16 + fr, n0 + wave * 16 + fq * 4, t);
  }
}

// Large products: 256 (n) x 256 (m) tile, four waves of 128 x 128 (one per SIMD, 256 accumulators in the accumulation
// registers).  LDS bandwidth decides the wave tile: a 256-column step of eight 128 x 64 waves reads 192 KiB and stages 64 KiB, as
// long as its MFMAs take at 128 B/clk; four 128 x 128 waves read 128 KiB.
//   * a K tile is 256 columns = 128 bytes a row (whole cache lines: 64-byte rows filled LDS a quarter slower), two stages for each
//     operand, filled by LDS-DMA that stays in flight across barriers; 16-byte chunks are XOR-ed with bits 1-3 of
//     the row: the 16 lanes that ds_read_b128 serves together (0-3, 12-15, 20-23, 24-27 and so on) then cover all banks once;
//   * 32x32x64 scaled MFMA, lane = row l & 31, K half h = l >> 5; step s of a K tile takes block 4h + s, so one 32-bit word holds a
//     lane's four scales of the K tile and the step picks the byte;
//   * scales: 16 bytes a row cover two K tiles (8 KiB, two stages, two LDS-DMA loads per wave every second K tile);
//   * a wave holds its 128 activation rows of the K tile in registers and walks its weight rows 32 at a time: 16 MFMAs, between which
//     it reads the next 32 weight rows and a part of the next K tile's activations.  Two barriers per K tile: behind the first
//     the activations' other stage is free, behind the second the weights', and each is refilled a whole K tile ahead of its use, one
//     load every four MFMAs (in bursts of eight: 3 % slower at 4096 x 4096 x 8192).
// The K range goes in groups of two K tiles; codes behind the last column need no mask: their scale bytes are zero on both
// operands, and 2^-254 is zero in fp32.  Reads past the operand are cut off by the buffer's size, which shrinks as its base advances.
// 4096 x 8192 x 4096 takes 64-67 us, 4.1-4.3 PFLOP/s; the same MFMAs on registers alone run at 6.65.
constexpr int MXT_OPER = 256 * 128, MXT_SCALE = 4 * MXT_OPER, MXT_SCALE_STAGE = 512 * 16;   // W0, W1, X0, X1, scales
constexpr int MXT_LDS = MXT_SCALE + 2 * MXT_SCALE_STAGE;   // 144 KiB

typedef float f32x16 __attribute__((ext_vector_type(16)));

// one 32x32x64 step; the scale byte is an immediate of the instruction (s is a constant after unrolling)
__device__ __forceinline__ f32x16 mx_mma(int s, i32x4 a, i32x4 b, f32x16 c, int as, int bs) {
  switch (s) {
    case 0: return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wide(a), wide(b), c, 4, 4, 0, as, 0, bs);
    case 1: return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wide(a), wide(b), c, 4, 4, 1, as, 1, bs);
    case 2: return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wide(a), wide(b), c, 4, 4, 2, as, 2, bs);
    default: return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wide(a), wide(b), c, 4, 4, 3, as, 3, bs);
  }
}
// tile of a workgroup: of the 256 that run at once each XCD (it has its own L2) gets 32 that follow each other, 8 m tiles before the next n
// tile: 8 x 4 operand panels instead of 2 x 16.  The XCDs' runs are neighbours, so what is written at a time spreads over the
// whole width of the output (one long run for each XCD sets them a power of two apart and they meet in the same memory channels:
// 8192^2 x 512 to bf16 50 -> 43 us, to fp32 80 -> 72; 8192^3 to fp32 263 -> 254; 16384 x 4096^2 to fp32 151 -> 155)
__device__ __forceinline__ void mx_tile_of(const MxDense &p, int &mt, int &nt, int &sk) {
  const int first = (int)blockIdx.x & ~255, some = min(256, p.mt * p.nt * p.split - first), q = some >> 3, r = some & 7, xcd = blockIdx.x & 7;
  int t = first + (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + (((int)blockIdx.x & 255) >> 3);
  sk = t / (p.mt * p.nt);
  t -= sk * p.mt * p.nt;
  const int g = t / (8 * p.nt), h = min(8, p.mt - g * 8), u = t - g * 8 * p.nt;
  nt = u / h;
  mt = __builtin_amdgcn_readfirstlane(g * 8 + u - nt * h);   // (uniform: said so, or buffer descriptors go through loops)
  nt = __builtin_amdgcn_readfirstlane(nt);
  sk = __builtin_amdgcn_readfirstlane(sk);
}

enum { MX_PLAIN = 0, MX_LINEAR = 1, MX_RELU = 2, MX_SIGMOID = 3 };   // epilogue: the sums; bias and none or LeakyReLU; bias and ReLU; bias and sigmoid
template <typename TO, int MODE> __global__ __launch_bounds__(256, 1) void mx_dense256_kernel(MxDense p) {
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wr = wave >> 1, wc = wave & 1;
  int mt, nt, sk;
  mx_tile_of(p, mt, nt, sk);
  const int m0 = mt * 256, n0 = nt * 256, cp = p.nb * 16;
  const int mr = min(256, p.M - m0), nr = min(256, p.N - n0);
  const int gbeg = sk * p.kt_per, groups = min(gbeg + p.kt_per, p.pitch / 16) - gbeg;   // of two K tiles = 512 columns

  // ---- staging: a wave fills 64 rows of each operand, eight loads of 8 rows; lane -> row lane / 8, source chunk swizzled
  unsigned vload[8];
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    const int row = wave * 64 + q * 8 + (lane >> 3);
    vload[q] = (unsigned)(row * cp + (((lane & 7) ^ ((row >> 1) & 7)) << 4));
  }
  struct Stream {      // one operand: base of the next K tile, bytes from there to the operand's end, K tiles not issued yet
    const uint8_t *at;
    int left, todo;
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc() const {
      return __builtin_amdgcn_make_buffer_rsrc((void *)at, 0, left, 0x00020000);
    }
    __device__ __forceinline__ void advance() {   // behind the last K tile: loads of nothing keep the counts
      --todo;
      at += 128;
      left = __builtin_amdgcn_readfirstlane(todo > 0 ? max(left - 128, 0) : 0);
    }
  };
  Stream w = {p.wc + (int64_t)n0 * cp + (int64_t)gbeg * 256, __builtin_amdgcn_readfirstlane(nr * cp - gbeg * 256), groups * 2};
  Stream x = {p.xc + (int64_t)m0 * cp + (int64_t)gbeg * 256, __builtin_amdgcn_readfirstlane(mr * cp - gbeg * 256), groups * 2};
  char *const dmaw = lds + wave * 8192;
  auto issue = [&](const Stream &o, int q, int slot) { mx_dma16(o.rsrc(), vload[q], 0, dmaw + slot * MXT_OPER + q * 1024); };
  const __amdgpu_buffer_rsrc_t wsr = mx_rsrc(p.ws, n0, nr, p.pitch), xsr = mx_rsrc(p.xs, m0, mr, p.pitch);
  const unsigned soff = (unsigned)((wave * 64 + lane) * p.pitch);
  unsigned sgrp = (unsigned)gbeg * 16;
  const unsigned sgrp_last = (unsigned)(gbeg + groups - 1) * 16;
  auto issue_scales = [&](int stage) {
    mx_dma16(wsr, soff, sgrp, lds + MXT_SCALE + stage + wave * 1024);
    mx_dma16(xsr, soff, sgrp, lds + MXT_SCALE + stage + 4096 + wave * 1024);
    if (sgrp < sgrp_last) sgrp += 16;
  };

  // ---- fragments: weight rows (i >> 1) * 128 + wr * 64 + (i & 1) * 32 + fr, activation rows wc * 128 + j * 32 + fr
  const int fr = lane & 31, fh = lane >> 5;
  const int laneoff = fr * 128 + (((fh * 4) ^ ((fr >> 1) & 7)) << 4);
  const char *wrd[4], *xrd[4];
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    wrd[s] = lds + ((wr * 64 * 128 + laneoff) ^ (s << 4));
    xrd[s] = lds + ((2 * MXT_OPER + wc * 128 * 128 + laneoff) ^ (s << 4));
  }
  // (the two scale pointers switch stages apart: activations are read one K tile ahead)
  const char *wsc = lds + MXT_SCALE + (wr * 64 + fr) * 16 + fh * 4, *xsc = lds + MXT_SCALE + (256 + wc * 128 + fr) * 16 + fh * 4;
  auto flip = [&](const char *q) { return (const char *)(lds + ((unsigned)(q - lds) ^ MXT_SCALE_STAGE)); };

  f32x16 acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
  i32x4 a[2][4], b[2][4][4];     // [parity of i][step]; [K tile parity][j][step]
  int as[2], bs[2][4];
#define MX_READ_W(I, T, S) a[(I) & 1][S] = *(const i32x4 *)(wrd[S] + (T) * MXT_OPER + ((I) >> 1) * 16384 + ((I) & 1) * 4096);
#define MX_SCALE_W(I, T) as[(I) & 1] = *(const int *)(wsc + ((I) >> 1) * 2048 + ((I) & 1) * 512 + (T) * 8);
#define MX_READ_X(J, T, S) b[T][J][S] = *(const i32x4 *)(xrd[S] + (T) * MXT_OPER + (J) * 4096);
#define MX_SCALE_X(J, T) bs[T][J] = *(const int *)(xsc + (J) * 512 + (T) * 8);
#define MX_MMA(I, T, S, J) acc[I][J] = mx_mma(S, b[T][J][S], a[(I) & 1][S], acc[I][J], bs[T][J], as[(I) & 1]);

  issue_scales(0);
#pragma unroll
  for (int q = 0; q < 8; ++q) issue(x, q, 2);
#pragma unroll
  for (int q = 0; q < 8; ++q) issue(w, q, 0);
  x.advance(); w.advance();
#pragma unroll
  for (int q = 0; q < 8; ++q) issue(x, q, 3);
  issue_scales(MXT_SCALE_STAGE);
#pragma unroll
  for (int q = 0; q < 3; ++q) issue(w, q, 1);      // (the other five in the loop)
  x.advance();
  mx_wait<13>();
  __builtin_amdgcn_s_barrier();
#pragma unroll
  for (int s = 0; s < 4; ++s) {
#pragma unroll
    for (int j = 0; j < 4; ++j) { MX_READ_X(j, 0, s) }
    MX_READ_W(0, 0, s)
    MX_SCALE_X(s, 0)
  }
  MX_SCALE_W(0, 0)

  // T: K tile of the group = stage of both operands.  x of K tile t + 1 is read from i = 1 on, w(i + 1) at i, w(0) of t + 1 at i = 3.
  int sst = 0;         // scale stage of this group (bytes)
#define MX_KTILE(T)                                                                                                 \
  {                                                                                                                 \
    _Pragma("unroll") for (int i = 0; i < 4; ++i) {                                                                 \
      _Pragma("unroll") for (int y = 0; y < 16; ++y) {                                                              \
        MX_MMA(i, T, y >> 2, y & 3)                                                                                 \
        if (i < 3) {                                                                                                \
          if (y < 4) { MX_READ_W(i + 1, T, y) }                                                                     \
          if (y == 4) { MX_SCALE_W(i + 1, T) }                                                                      \
        }                                                                                                           \
        if (i == 0 && y == 12) {              /* x of t + 1 has landed; every wave has left x of t */               \
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                                                        \
          mx_wait<(T) ? 8 : 10>();                                                                                  \
          __builtin_amdgcn_s_barrier();                                                                             \
          if constexpr ((T) == 1) xsc = flip(xsc);                                                                  \
        }                                                                                                           \
        if ((i == 1 || i == 2) && (y & 3) == 1) issue(x, (i - 1) * 4 + (y >> 2), 2 + (T));                          \
        if (i == 1 && y >= 8 && y < 12) { MX_READ_X(0, 1 - (T), y - 8) }                                            \
        if (i == 1 && y >= 12) { MX_SCALE_X(y - 12, 1 - (T)) }                                                      \
        if (i == 2 && y >= 6 && y < 14) { MX_READ_X(1 + ((y - 6) >> 2), 1 - (T), (y - 6) & 3) }                     \
        if (i == 3 && y == 2) {               /* w of t + 1 has landed; every wave has left w of t */               \
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                                                        \
          mx_wait<8>();                                                                                             \
          __builtin_amdgcn_s_barrier();                                                                             \
          if constexpr ((T) == 1) { wsc = flip(wsc); issue_scales(sst); }                                           \
        }                                                                                                           \
        if (i == 3 && y >= 3 && y < 7) { MX_READ_W(0, 1 - (T), y - 3) }                                             \
        if (i == 3 && y == 7) { MX_SCALE_W(0, 1 - (T)) }                                                            \
        if (i == 3 && (y & 3) == 1 && y > 1) issue(w, (y >> 2) - 1, T);                                             \
        if (i == 0 && (y & 1) && y < 10) issue(w, 3 + (y >> 1), 1 - (T));                                           \
        if (i == 0 && y == 10) w.advance();                                                                         \
        if (i == 3 && y >= 8 && y < 12) { MX_READ_X(3, 1 - (T), y - 8) }                                            \
        __builtin_amdgcn_sched_barrier(0);                                                                          \
      }                                                                                                             \
    }                                                                                                               \
    x.advance();                                                                                                    \
  }
  for (int g = 0; g < groups; ++g) {
    MX_KTILE(0)
    MX_KTILE(1)
    sst ^= MXT_SCALE_STAGE;
  }
#undef MX_KTILE
#undef MX_MMA
#undef MX_SCALE_X
#undef MX_READ_X
#undef MX_SCALE_W
#undef MX_READ_W
  mx_wait<0>();        // (the tail loads must not outlive the workgroup's LDS)

  // epilogue straight from the accumulators: lane = column n = fr of fragment i, rows 8q + 4 fh + r of fragment j, so a store covers
  // 32 consecutive columns of two rows.  bf16: neighbouring lanes swap halves and store two columns of one row each.  (Through
  // LDS, in whole 512-byte rows, it took 7-10 us of a tile; one wave a SIMD hides no LDS latency.)  Rows and columns that are
  // not there have offsets past the buffer's size: the stores drop them.
  TO *const y = p.split > 1 ? (TO *)p.slab + (int64_t)sk * p.M * p.N : (TO *)p.y;
  const int64_t ldy = p.split > 1 ? p.N : p.ldy;
  constexpr int ES = sizeof(TO);
  const int rowb = (int)ldy * ES, nl = wr * 64 + fr, odd = fr & 1;
  float bias[4];
  int voff[4];
  const float ns = act_neg_scale(p.act, p.slope);
  auto fin = [&](float v, float bv) {
    if constexpr (MODE == MX_PLAIN) return v;
    else if constexpr (MODE == MX_LINEAR) return apply_act_linear(v + bv, ns);
    else if constexpr (MODE == MX_RELU) return mx_relu(v + bv);
    else return 1.f / (1.f + __expf(-(v + bv)));
  };
  auto put = [&](auto pairs) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = nl + (i >> 1) * 128 + (i & 1) * 32;
      bias[i] = MODE != MX_PLAIN && p.bias && n < nr ? p.bias[n0 + n] : 0.f;
      voff[i] = n < nr ? fh * 4 * rowb + n * ES + (decltype(pairs)::value && odd ? rowb - ES : 0) : (int)MX_OOB;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int m = wc * 128 + j * 32;
      const int bytes = __builtin_amdgcn_readfirstlane(max(0, min(32, mr - m)) * rowb);
      const __amdgpu_buffer_rsrc_t yr = __builtin_amdgcn_make_buffer_rsrc((void *)(y + (int64_t)(m0 + m) * ldy + n0), 0, bytes, 0x00020000);
      int srow = 0;
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int r = 0; r < 4; r += 2) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float v0 = fin(acc[i][j][q * 4 + r], bias[i]), v1 = fin(acc[i][j][q * 4 + r + 1], bias[i]);
            if constexpr (ES == 4) {
              __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v0), yr, voff[i] + srow, 0, 0);
              __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v1), yr, voff[i] + srow + rowb, 0, 0);
            } else {
              const unsigned own = __builtin_bit_cast(unsigned, (bf16x2){(bf16)v0, (bf16)v1});
              if constexpr (decltype(pairs)::value) {    // odd lanes: {other.hi, own.hi} of the second row, even: {own.lo, other.lo}
                const unsigned other = (unsigned)__builtin_amdgcn_update_dpp(0, (int)own, 0xB1, 0xf, 0xf, false);
                __builtin_amdgcn_raw_buffer_store_b32(__builtin_amdgcn_perm(own, other, odd ? 0x07060302u : 0x01000504u), yr,
                                                      voff[i] + srow, 0, 0);
              } else {
                __builtin_amdgcn_raw_buffer_store_b16((unsigned short)own, yr, voff[i] + srow, 0, 0);
                __builtin_amdgcn_raw_buffer_store_b16((unsigned short)(own >> 16), yr, voff[i] + srow + rowb, 0, 0);
              }
            }
          }
          srow += r ? 6 * rowb : 2 * rowb;               // (rows 4..7 of eight are the other half's)
          asm volatile("" : "+s"(srow));                 // (a running sum: all the multiples of rowb at once do not fit the registers)
          __builtin_amdgcn_sched_barrier(0);
        }
    }
  };
  if constexpr (ES == 4) put(std::false_type{});
  else if (p.pairs && nr % 2 == 0) put(std::true_type{});
  else put(std::false_type{});
}

// Float activations against 4-bit weights (serving: the weights are what is read).  A workgroup's four waves own 64 weight rows
// each, or share the K groups of 64 rows (`mx_plan` chooses).  A K group is 512 columns: step s of it
// takes block 4s + (lane >> 4), the row's 16 scale bytes come with one load.  Codes become bf16 with their scale applied (exact: two significant bits) and meet
// the activations in 16x16x32 bf16 MFMAs, whose k order is the lane's block order on both operands.  The activations of a K
// group are converted once per workgroup and wait in LDS as columns of the product: up to 48 rows in bf16, or 16 in fp32, which
// are split exactly into three bf16 terms (8 + 8 + 8 bits by truncation), a column each -- fp32 accuracy, and one row costs one
// MFMA, not three.  A row's three columns are added when the waves join.  One fp32 row on 262144 x 256 (36 MB): 10.5 us, the latency of one round
// of loads on top of 3.3 TB/s; the slices' sum takes 2.6-3.9 more.
struct Split3 { bf16 t[3]; };
__device__ __forceinline__ Split3 split3(float x) {
  Split3 r;
  const unsigned u = __float_as_uint(x);
  if ((u & 0x7f800000u) == 0x7f800000u) {          // infinity, NaN: one term carries it
    r.t[0] = (bf16)x; r.t[1] = (bf16)0.f; r.t[2] = (bf16)0.f;
    return r;
  }
  const float h = __uint_as_float(u & 0xffff0000u), d = x - h;
  const float m = __uint_as_float(__float_as_uint(d) & 0xffff0000u);
  r.t[0] = (bf16)h; r.t[1] = (bf16)m; r.t[2] = (bf16)(d - m);
  return r;
}
constexpr int MXS_ROW = 1024 + 16;      // bytes of one activation row's K group in LDS: 512 bf16 and a pad
template <typename TX, int CT> __global__ __launch_bounds__(256, 2) void mx_serve_kernel(MxDense p) {   // CT: tiles of 16 columns
  constexpr int NX = sizeof(TX) == 4 ? 3 : 1;
  extern __shared__ __attribute__((aligned(1024))) char lds[];    // [K groups of a round][NX][rows], then the partial sums
  int mt, nt, sk;
  mx_small_tile(p, mt, nt, sk);
  const int lane = threadIdx.x & 63, fr = lane & 15, fq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kw = p.kwaves, wk = wave % kw, wn = wave / kw;       // K groups taken at once; this wave's group and weight rows
  const int m0 = mt * p.xrows, n0 = (nt * (4 / kw) + wn) * 64;
  const int cp = p.nb * 16, nr = max(0, min(64, p.N - n0)), rows = min(p.xrows, p.M - m0), cols = NX * p.xrows;
  const __amdgpu_buffer_rsrc_t wr = mx_rsrc(p.wc, nr ? n0 : 0, nr, cp), wsr = mx_rsrc(p.ws, nr ? n0 : 0, nr, p.pitch);
  f32x4 acc[4][CT] = {};
  const int k0 = sk * p.kt_per, k1 = min(k0 + p.kt_per, (p.nb + 15) / 16);
  const int gbytes = NX * p.xrows * MXS_ROW;
  for (int kt = k0; kt < k1; kt += kw) {
    const bool mine = kt + wk < k1;
    const int items = min(kw, k1 - kt) * p.xrows;
    // this wave's codes are on their way while the workgroup converts the activations
    i32x4 c[4][4], sc[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {        // (rows past the operand read as zero; codes behind K meet zeros)
      const unsigned r = (unsigned)(i * 16 + fr);
      sc[i] = ld16(wsr, mine ? r * p.pitch + (kt + wk) * 16 : MX_OOB);
#pragma unroll
      for (int s = 0; s < 4; ++s) c[i][s] = ld16(wr, mine ? r * cp + (kt + wk) * 256 + fq * 16 + s * 64 : MX_OOB);
    }
    if (kt > k0) __syncthreads();        // (everyone has left the last round's activations)
    for (int t = wave; t < items; t += 4) {      // 512 columns of a row, 8 a lane
      const int col = lane * 8, g = t / p.xrows, row = t - g * p.xrows, k = (kt + g) * 512 + col;
      float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (row < rows && k < p.K) load8((const TX *)p.x + (int64_t)(m0 + row) * p.ldx + k, p.K - k, v);
      bf16x8 o[NX];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if constexpr (NX == 1) o[0][e] = (bf16)v[e];
        else {
          const Split3 q = split3(v[e]);
#pragma unroll
          for (int u = 0; u < 3; ++u) o[u][e] = q.t[u];
        }
      }
#pragma unroll
      for (int u = 0; u < NX; ++u) *(bf16x8 *)(lds + g * gbytes + (u * p.xrows + row) * MXS_ROW + col * 2) = o[u];
    }
    __syncthreads();
    if (!mine) continue;      // (uniform; no weights, and zero times an infinite activation is not zero)
    const char *xl[CT];       // (lanes past the columns there are read column 0: nobody adds or stores what comes of it)
#pragma unroll
    for (int t = 0; t < CT; ++t) xl[t] = lds + wk * gbytes + (t * 16 + fr < cols ? t * 16 + fr : 0) * MXS_ROW + fq * 64;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      float sf[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) sf[i] = mx_scale_or_nan(((unsigned)sc[i][s] >> (8 * fq)) & 255u);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        bf16x8 xb[CT], wv[4];
#pragma unroll
        for (int t = 0; t < CT; ++t) xb[t] = *(const bf16x8 *)(xl[t] + s * 256 + j * 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) wv[i] = mx_bf16x8((unsigned)c[i][s][j], sf[i]);
#pragma unroll
        for (int t = 0; t < CT; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wv[i], xb[t], acc[i][t], 0, 0, 0);
      }
    }
  }
  // join: the waves of one weight tile, and the columns of one row; each of the kw waves finishes its share of the fragments
  __syncthreads();
  f32x4 *const part = (f32x4 *)lds;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int t = 0; t < CT; ++t) part[((wave * 4 + i) * CT + t) * 64 + lane] = acc[i][t];
  __syncthreads();
  for (int i = wk; i < 4; i += kw)
    for (int m = fr; m < rows; m += 16) {
      f32x4 sum = {0.f, 0.f, 0.f, 0.f};
      for (int w = 0; w < kw; ++w)
#pragma unroll
        for (int u = NX - 1; u >= 0; --u) {
          const int col = u * p.xrows + m;
          sum += part[(((wn * kw + w) * 4 + i) * CT + (col >> 4)) * 64 + (col & 15) + 16 * fq];
        }
      mx_emit(p, sk, m0 + m, n0 + i * 16 + fq * 4, sum);
    }
}

static int mx_check(int64_t m, int64_t n, int64_t k) {
  CFD_REQUIRE(m >= 0 && n >= 0 && m <= 0x7fffff00 && n <= 0x7fffff00, "rows out of range");
  CFD_REQUIRE(k > 0 && k <= (1 << 22), "columns must be in 1 .. 4194304");
  return CFD_OK;
}

static void mx_split(MxDense &p, int groups, int64_t want) {   // K slices of whole groups, about `want` of them
  if (want > groups) want = groups;
  if (want < 1) want = 1;
  p.kt_per = (int)((groups + want - 1) / want);
  p.split = (groups + p.kt_per - 1) / p.kt_per;
}
static int mx_serve_bytes(const MxDense &p, int x_kind) {   // LDS of the float-activation kernel
  const int groups = p.kt_per < p.kwaves ? p.kt_per : p.kwaves;
  const int cols = (x_kind == CFD_MX_X_BF16 ? 1 : 3) * p.xrows, x = groups * cols * MXS_ROW, sums = 16 * ((cols + 15) / 16) * 1024;
  return x > sums ? x : sums;
}
static void mx_plan(MxDense &p, int x_kind) {
  const bool serve = x_kind != CFD_MX_X_MXFP4;
  p.nb = (int)mx_blocks(p.K);
  p.pitch = (int)mx_scale_pitch(p.K);
  // 256 x 256 tiles where there are outputs enough to fill the chip without slices of K, or work enough to hide their fixed ~8 us; else
  // 64 x 64 tiles, which read each operand four times as often.  Measured (us, 256 | 64): 2048^2 x 512 12 | 17, 4000^2 x 100 17 | 51,
  // 1024^3 11 | 8, 512^2 x 8192 21 | 15, 256 x 4096^2 27 | 27, 1024^2 x 8192 32 | 37, 512 x 1024 x 65536 40 | 83, 136 x 1100 x 4000 19 | 12
  const double mn = (double)p.M * p.N;
  p.big = !serve && p.M > 128 && p.N > 128 && (mn >= 3e6 || mn * p.K >= 4e9);
  if (p.big) {
    p.nt = (p.N + 255) / 256;
    p.mt = (p.M + 255) / 256;
    const int groups = p.pitch / 16;     // one workgroup per CU; a slice has 4 groups at least
    const int64_t want = 256 / ((int64_t)p.nt * p.mt);
    mx_split(p, groups, want < groups / 4 ? want : groups / 4);
  } else if (serve) {
    const int most = x_kind == CFD_MX_X_BF16 ? 48 : 16;
    p.mt = (p.M + most - 1) / most;
    p.xrows = (p.M + p.mt - 1) / p.mt;
    // Four waves on one weight tile where the chip has room for a workgroup per tile and K group (two on each of 256 CUs: a slice is then one
    // group, all four waves convert it and one multiplies), or where few columns are cheap to convert four times as often: a wave's
    // loads of 16 rows at a time keep a CU's address unit busy, and so they spread over more CUs.  Us, four waves on a tile | four
    // tiles: 1 row fp32 256 x 2048 7.1 | 9.0, 256 x 262144 14.0 | 16.9, 28672 x 8192 27.2 | 36.0; 16 rows bf16 4096^2 11.1 | 12.3, 8192^2
    // 19.8 | 19.3, 28672 x 8192 50 | 42; 48 rows bf16 256 x 2048 13.0 | 17.8, 256 x 65536 18.9 | 21.7, 1030 x 16384 31 | 20
    const int groups = (p.nb + 15) / 16, cols = (x_kind == CFD_MX_X_BF16 ? 1 : 3) * p.xrows;
    const int64_t units = (int64_t)((p.N + 63) / 64) * p.mt * groups;
    const bool spread = units <= 512 || (cols <= 16 && units * cols <= 32768);
    // ... and no slices, whose sum is a launch of its own, where the four waves have all the groups at few columns: one fp32 row 4096 x 1024
    // 6.2 | 7.3, 1030 x 2048 6.9 | 7.4 us, and 2.7 us less of the host's time; eight bf16 rows 8192 x 1024 6.5 | 7.5, but 1030 x 2048 8.4 | 7.1
    const bool whole = spread && groups <= 4 && cols <= (groups <= 2 ? 16 : 6);
    for (p.kwaves = spread || p.N <= 64 ? 4 : p.N <= 128 ? 2 : 1;; p.kwaves /= 2) {   // (fewer where their activations exceed the LDS)
      p.nt = (p.N + 256 / p.kwaves - 1) / (256 / p.kwaves);
      mx_split(p, groups, whole ? 1 : 512 / ((int64_t)p.nt * p.mt));
      if (p.kwaves == 1 || mx_serve_bytes(p, x_kind) <= 160 * 1024) break;
    }
  } else {
    p.nt = (p.N + 63) / 64;
    p.mt = (p.M + 63) / 64;
    // one workgroup per CU; a slice has a group for each of the four waves; no slices where half the CUs have a tile (128 x 4096 x 4096:
    // 15.3 us in two slices, whose sum is a launch of its own, 10.2 in one)
    const int groups = p.pitch / 16;
    const int64_t tiles = (int64_t)p.nt * p.mt, want = tiles >= 128 ? 1 : 256 / tiles;
    mx_split(p, groups, want < groups / 4 ? want : groups / 4);
  }
}

}  // namespace cfd

using namespace cfd;

extern "C" int64_t cfd_mxfp4_scale_pitch(int64_t cols) { return mx_scale_pitch(cols); }

extern "C" int cfd_mxfp4_quantize(const void *x, int64_t ldx, int dtype, int64_t rows, int64_t cols, uint8_t *codes,
                                  uint8_t *scales, uint8_t *codes_t, uint8_t *scales_t, void *stream) {
  if (int rc = mx_check(rows, 0, cols)) return rc;
  CFD_REQUIRE(dtype == CFD_F32 || dtype == CFD_BF16, "bad dtype");
  if (rows == 0) return CFD_OK;
  CFD_REQUIRE((codes != nullptr) == (scales != nullptr) && (codes_t != nullptr) == (scales_t != nullptr) && (codes || codes_t),
              "codes come with scales, in one orientation at least");
  CFD_REQUIRE(x && ldx >= cols, "bad arguments");
  CFD_REQUIRE((((uintptr_t)codes | (uintptr_t)scales | (uintptr_t)codes_t | (uintptr_t)scales_t) & 15) == 0,
              "codes and scales must be 16-byte aligned");
  hipStream_t st = (hipStream_t)stream;
  const int nb = (int)mx_blocks(cols), pitch = (int)mx_scale_pitch(cols);
  if (!codes_t) {
    const FastDiv G((unsigned)((nb + 3) / 4 * 16));
    const int64_t blocks = (rows * G.d + 255) / 256;
    CFD_REQUIRE(blocks <= MX_GRID, "too many elements");
    if (dtype == CFD_BF16)
      hipLaunchKernelGGL(mx_quant_rows_kernel<bf16>, dim3((unsigned)blocks), dim3(256), 0, st, (const bf16 *)x, ldx, rows,
                         (int)cols, nb, pitch, codes, scales, G);
    else
      hipLaunchKernelGGL(mx_quant_rows_kernel<float>, dim3((unsigned)blocks), dim3(256), 0, st, (const float *)x, ldx, rows,
                         (int)cols, nb, pitch, codes, scales, G);
  } else {
    if (int rc = mx_check(cols, 0, rows)) return rc;   // the rows are the other orientation's columns
    const int nbt = (int)mx_blocks(rows), pitch_t = (int)mx_scale_pitch(rows);
    const int64_t tx = (cols + QT - 1) / QT, blocks = tx * ((rows + QT - 1) / QT);
    CFD_REQUIRE(blocks <= MX_GRID, "too many elements");
    const dim3 grid((unsigned)blocks);
    if (dtype == CFD_BF16)
      hipLaunchKernelGGL(mx_quant_both_kernel<bf16>, grid, dim3(256), 0, st, (const bf16 *)x, ldx, (int)rows, (int)cols, nb,
                         pitch, codes, scales, nbt, pitch_t, codes_t, scales_t, (int)tx);
    else
      hipLaunchKernelGGL(mx_quant_both_kernel<float>, grid, dim3(256), 0, st, (const float *)x, ldx, (int)rows, (int)cols, nb,
                         pitch, codes, scales, nbt, pitch_t, codes_t, scales_t, (int)tx);
  }
  CFD_LAUNCH_CHECK();
  return CFD_OK;
}

extern "C" int cfd_mxfp4_dequantize(const uint8_t *codes, const uint8_t *scales, int64_t rows, int64_t cols, void *y, int64_t ldy,
                                    int dtype, void *stream) {
  if (int rc = mx_check(rows, 0, cols)) return rc;
  CFD_REQUIRE(dtype == CFD_F32 || dtype == CFD_BF16, "bad dtype");
  if (rows == 0) return CFD_OK;
  CFD_REQUIRE(codes && scales && y && ldy >= cols, "bad arguments");
  CFD_REQUIRE((((uintptr_t)codes | (uintptr_t)scales) & 15) == 0, "codes and scales must be 16-byte aligned");
  const int nb = (int)mx_blocks(cols), pitch = (int)mx_scale_pitch(cols);
  const FastDiv G((unsigned)(nb * 4));
  const int64_t blocks = (rows * G.d + 255) / 256;
  CFD_REQUIRE(blocks <= MX_GRID, "too many elements");
  if (dtype == CFD_BF16)
    hipLaunchKernelGGL(mx_dequant_kernel<bf16>, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, codes, scales, rows,
                       (int)cols, nb, pitch, (bf16 *)y, ldy, G);
  else
    hipLaunchKernelGGL(mx_dequant_kernel<float>, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, codes, scales, rows,
                       (int)cols, nb, pitch, (float *)y, ldy, G);
  CFD_LAUNCH_CHECK();
  return CFD_OK;
}

extern "C" int64_t cfd_mxfp4_dense_workspace_bytes(int64_t m, int64_t n, int64_t k, int x_kind) {
  if (int rc = mx_check(m, n, k)) return rc;
  CFD_REQUIRE(x_kind >= CFD_MX_X_F32 && x_kind <= CFD_MX_X_MXFP4, "bad x_kind");
  if (!m || !n) return 0;
  MxDense p = {};
  p.M = (int)m; p.N = (int)n; p.K = (int)k;
  mx_plan(p, x_kind);
  return p.split > 1 ? (int64_t)p.split * m * n * 4 : 0;
}

extern "C" int cfd_mxfp4_dense_plan(int64_t m, int64_t n, int64_t k, int x_kind, int *plan) {
  if (int rc = mx_check(m, n, k)) return rc;
  CFD_REQUIRE(x_kind >= CFD_MX_X_F32 && x_kind <= CFD_MX_X_MXFP4, "bad x_kind");
  CFD_REQUIRE(plan && m && n, "bad arguments");
  MxDense p = {};
  p.M = (int)m; p.N = (int)n; p.K = (int)k;
  mx_plan(p, x_kind);
  const bool serve = x_kind != CFD_MX_X_MXFP4;
  plan[0] = p.big ? 256 : serve ? p.xrows : 64;
  plan[1] = p.split;
  plan[2] = p.kt_per;
  plan[3] = p.big ? 1 : serve ? p.kwaves : 4;
  return CFD_OK;
}

extern "C" int cfd_mxfp4_dense(const cfd_mxfp4_dense_desc *d, const void *x, const uint8_t *x_scales, const uint8_t *w_codes,
                               const uint8_t *w_scales, const float *bias, void *y, void *ws, void *stream) {
  CFD_REQUIRE(d, "NULL descriptor");
  if (int rc = mx_check(d->m, d->n, d->k)) return rc;
  CFD_REQUIRE(d->x_kind == CFD_MX_X_MXFP4 || d->x_kind == CFD_MX_X_F32 || d->x_kind == CFD_MX_X_BF16, "bad x_kind");
  CFD_REQUIRE(d->out_dtype == CFD_F32 || d->out_dtype == CFD_BF16, "bad out_dtype");
  CFD_REQUIRE(d->act >= CFD_ACT_NONE && d->act <= CFD_ACT_SIGMOID, "bad activation");
  if (!d->m || !d->n) return CFD_OK;
  const bool serve = d->x_kind != CFD_MX_X_MXFP4;
  CFD_REQUIRE(x && w_codes && w_scales && y && d->ldy >= d->n, "bad arguments");
  CFD_REQUIRE(d->ldy <= (1 << 23), "ldy must be at most 8388608");
  CFD_REQUIRE(serve ? d->ldx >= d->k : x_scales != nullptr, "bad activations");
  CFD_REQUIRE((((uintptr_t)w_codes | (uintptr_t)w_scales) & 15) == 0, "weights must be 16-byte aligned");
  CFD_REQUIRE(serve || (((uintptr_t)x | (uintptr_t)x_scales) & 15) == 0, "4-bit activations must be 16-byte aligned");
  MxDense p = {};
  p.M = (int)d->m; p.N = (int)d->n; p.K = (int)d->k;
  mx_plan(p, d->x_kind);
  p.xc = (const uint8_t *)x; p.xs = x_scales; p.x = x; p.ldx = d->ldx; p.wc = w_codes; p.ws = w_scales; p.bias = bias;
  p.y = y; p.ldy = d->ldy; p.out_bf16 = d->out_dtype == CFD_BF16; p.act = d->act; p.slope = d->leaky_slope;
  p.slab = (float *)ws;
  p.pairs = ((uintptr_t)y & 3) == 0 && d->ldy % 2 == 0;
  CFD_REQUIRE(p.split == 1 || ws, "this shape needs a workspace");
  const int64_t blocks = (int64_t)p.mt * p.nt * p.split;
  CFD_REQUIRE(blocks <= MX_GRID, "too many tiles");
  hipStream_t st = (hipStream_t)stream;
  if (p.big) {
    const bool b16 = p.out_bf16 && p.split == 1;
    const int mode = p.split > 1 || (!bias && p.act == CFD_ACT_NONE) ? MX_PLAIN : p.act == CFD_ACT_SIGMOID ? MX_SIGMOID : p.act == CFD_ACT_RELU ? MX_RELU : MX_LINEAR;
    void (*const fns[2][4])(MxDense) = {{mx_dense256_kernel<float, MX_PLAIN>, mx_dense256_kernel<float, MX_LINEAR>, mx_dense256_kernel<float, MX_RELU>,
                                         mx_dense256_kernel<float, MX_SIGMOID>},
                                        {mx_dense256_kernel<bf16, MX_PLAIN>, mx_dense256_kernel<bf16, MX_LINEAR>, mx_dense256_kernel<bf16, MX_RELU>,
                                         mx_dense256_kernel<bf16, MX_SIGMOID>}};
    void (*const fn)(MxDense) = fns[b16][mode];
    if (int rc = set_max_lds((const void *)fn, MXT_LDS)) return rc;
    hipLaunchKernelGGL(fn, dim3((unsigned)blocks), dim3(256), MXT_LDS, st, p);
  } else if (!serve) {
    if (int rc = set_max_lds((const void *)mx_dense_kernel, MXD_LDS)) return rc;
    hipLaunchKernelGGL(mx_dense_kernel, dim3((unsigned)blocks), dim3(256), MXD_LDS, st, p);
  } else {
    const bool b16 = d->x_kind == CFD_MX_X_BF16;
    const int bytes = mx_serve_bytes(p, d->x_kind);
    const int tiles = ((b16 ? 1 : 3) * p.xrows + 15) / 16;
    void (*const fns[2][3])(MxDense) = {{mx_serve_kernel<float, 1>, mx_serve_kernel<float, 2>, mx_serve_kernel<float, 3>},
                                        {mx_serve_kernel<bf16, 1>, mx_serve_kernel<bf16, 2>, mx_serve_kernel<bf16, 3>}};
    void (*const fn)(MxDense) = fns[b16][tiles - 1];
    if (int rc = set_max_lds((const void *)fn, bytes)) return rc;
    hipLaunchKernelGGL(fn, dim3((unsigned)blocks), dim3(256), bytes, st, p);
  }
  CFD_LAUNCH_CHECK();
  if (p.split > 1) {
    const int64_t b = (d->m * d->n + 63) / 64;
    CFD_REQUIRE(b <= MX_GRID, "too many outputs");
    hipLaunchKernelGGL(mx_split_sum_kernel, dim3((unsigned)b), dim3(256), 0, st, p);
    CFD_LAUNCH_CHECK();
  }
  return CFD_OK;
}
