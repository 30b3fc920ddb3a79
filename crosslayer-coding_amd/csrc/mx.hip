// Microscaled formats: rows quantised and expanded, a resident cache of activations in them, and the encoder projection
// from 4-bit weights.
//
// 32 neighbouring elements of a row form a block and share the power of two 2^(s - 127), s one byte (255: no number).
//   s      the biased exponent of the block's largest magnitude minus the largest exponent of the element type, held in
//          0 .. 254; 255 where the block holds an infinity or a NaN, which makes all of it read back as NaN
//   codes  v 2^(127 - s), rounded to nearest even and held at the largest value (the product with a power of two is exact)
//     CLT_MXFP4    sign, two bits of exponent, one of mantissa (0 0.5 1 1.5 2 3 4 6); two to a byte, the even element low
//     CLT_MXFP8    sign, four bits of exponent, three of mantissa, up to 448
//     CLT_MXINT8   two's complement in 64ths, -127/64 .. 127/64
// A row of d elements has ceil(d / 32) blocks; the last one is filled up with zeros.
#include "clt_common.h"

namespace {

constexpr int MX_THREADS = 256;
constexpr int64_t MX_MAX_WIDTH = 262144;    // elements of a row: the pieces of a workgroup's rows are told apart with 32 bits

template <int FMT> struct Mx;
template <> struct Mx<CLT_MXFP4> { static constexpr int EMAX = 2, BLOCK_BYTES = 16; };
template <> struct Mx<CLT_MXFP8> { static constexpr int EMAX = 8, BLOCK_BYTES = 32; };
template <> struct Mx<CLT_MXINT8> { static constexpr int EMAX = 0, BLOCK_BYTES = 32; };

// 2^(b - 127) for b in 0 .. 254, NaN for 255
__device__ __forceinline__ float mx_power(uint32_t b) {
  return __uint_as_float(b == 0u ? 0x00400000u : b == 255u ? 0x7FC00000u : b << 23);
}

// Eight scaled values as codes: one word of fp4, two of the others.
template <int FMT> __device__ __forceinline__ uint2 mx_encode8(const float (&v)[8]) {
  uint2 c = make_uint2(0u, 0u);
  if constexpr (FMT == CLT_MXFP4) {
    c.x = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c.x, v[0], v[1], 1.0f, 0);
    c.x = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c.x, v[2], v[3], 1.0f, 1);
    c.x = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c.x, v[4], v[5], 1.0f, 2);
    c.x = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c.x, v[6], v[7], 1.0f, 3);
  } else if constexpr (FMT == CLT_MXFP8) {
    float h[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) h[k] = __builtin_amdgcn_fmed3f(v[k], -448.0f, 448.0f);
    c.x = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(h[0], h[1], 0, false);
    c.x = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(h[2], h[3], (int)c.x, true);
    c.y = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(h[4], h[5], 0, false);
    c.y = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(h[6], h[7], (int)c.y, true);
  } else {
    uint32_t b[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) b[k] = (uint32_t)(int)rintf(__builtin_amdgcn_fmed3f(v[k] * 64.0f, -127.0f, 127.0f)) & 0xFFu;
    c.x = b[0] | (b[1] << 8) | (b[2] << 16) | (b[3] << 24);
    c.y = b[4] | (b[5] << 8) | (b[6] << 16) | (b[7] << 24);
  }
  return c;
}

typedef __attribute__((ext_vector_type(2))) float mx_f32x2_t;

// The values eight codes stand for, before the block's scale.
template <int FMT> __device__ __forceinline__ void mx_decode8(const uint2 &c, float (&v)[8]) {
  if constexpr (FMT == CLT_MXFP4) {
    const mx_f32x2_t a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c.x, 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c.x, 1.0f, 1);
    const mx_f32x2_t e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c.x, 1.0f, 2), f = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c.x, 1.0f, 3);
    v[0] = a[0]; v[1] = a[1]; v[2] = b[0]; v[3] = b[1]; v[4] = e[0]; v[5] = e[1]; v[6] = f[0]; v[7] = f[1];
  } else if constexpr (FMT == CLT_MXFP8) {
    const mx_f32x2_t a = __builtin_amdgcn_cvt_pk_f32_fp8((int)c.x, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)c.x, true);
    const mx_f32x2_t e = __builtin_amdgcn_cvt_pk_f32_fp8((int)c.y, false), f = __builtin_amdgcn_cvt_pk_f32_fp8((int)c.y, true);
    v[0] = a[0]; v[1] = a[1]; v[2] = b[0]; v[3] = b[1]; v[4] = e[0]; v[5] = e[1]; v[6] = f[0]; v[7] = f[1];
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t w = k < 4 ? c.x : c.y;
      v[k] = (float)((int)(w << (24 - 8 * (k & 3))) >> 24) * 0.015625f;
    }
  }
}

// Rows of the batch and where they lie in the store.
struct MxRows {
  const void *index;      // [n] row numbers, 32 or 64 bits (NULL: first, first + 1, ...)
  int wide;               // 64-bit row numbers
  int64_t first, rows;    // rows of the store per layer and kind
  const int32_t *owner;   // write: [rows], the last row of the batch that names a row (NULL: all are different)
};
__device__ __forceinline__ int64_t mx_row(const MxRows &r, int64_t j) {
  if (!r.index) return r.first + j;
  return r.wide ? ((const int64_t *)r.index)[j] : (int64_t)((const int32_t *)r.index)[j];
}

// A workgroup takes 256 neighbouring pieces of eight elements: row and place in it from 32-bit numbers counted from the
// group's first row.  magic = ceil(2^32 / pieces), exact for counts up to MX_MAX_WIDTH / 8 + 256.
struct MxPiece { int64_t j; uint32_t p; };
__device__ __forceinline__ MxPiece mx_piece(uint32_t pieces, uint32_t magic) {
  const uint64_t base = (uint64_t)blockIdx.x * MX_THREADS;
  const uint64_t row0 = base / pieces;
  const uint32_t at = (uint32_t)(base - row0 * pieces) + threadIdx.x;
  const uint32_t dj = pieces == 1u ? at : __umulhi(at, magic);
  return {(int64_t)(row0 + dj), at - dj * pieces};
}

// grid: x = groups of pieces, y = layer * kinds + kind.  Four lanes hold a block and agree on its scale.
template <typename T, int FMT, bool VEC>
__global__ __launch_bounds__(MX_THREADS) void k_mx_write(const T *__restrict__ src0, const T *__restrict__ src1, int64_t layer_stride,
                                                         int64_t row_stride, int kinds, int64_t n, int64_t d, uint32_t blocks,
                                                         uint32_t magic, MxRows rows, uint8_t *__restrict__ codes,
                                                         uint8_t *__restrict__ scales) {
  const MxPiece at = mx_piece(blocks * 4u, magic);
  const int64_t l = blockIdx.y / (uint32_t)kinds;
  const int kind = (int)(blockIdx.y - (uint32_t)l * (uint32_t)kinds);
  const int64_t c = (int64_t)at.p * 8;
  const bool live = at.j < n;
  float v[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = 0.0f;
  if (live) {
    const T *sp = (kind ? src1 : src0) + l * layer_stride + at.j * row_stride + c;
    if constexpr (VEC) {
      if (c < d) {                                     // d is a multiple of 8
        if constexpr (sizeof(T) == 2) {
          const uint4 w = *reinterpret_cast<const uint4 *>(sp);
          unpack_pair<T>(w.x, v[0], v[1]); unpack_pair<T>(w.y, v[2], v[3]); unpack_pair<T>(w.z, v[4], v[5]); unpack_pair<T>(w.w, v[6], v[7]);
        } else {
          const float4 a = *reinterpret_cast<const float4 *>(sp), b = *reinterpret_cast<const float4 *>(sp + 4);
          v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        }
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (c + k < d) v[k] = Elem<T>::to_f32(sp[k]);
    }
  }
  uint32_t top = 0;                                    // magnitudes in the order of their bits: NaN above infinity above all numbers
#pragma unroll
  for (int k = 0; k < 8; ++k) top = max(top, __float_as_uint(v[k]) & 0x7FFFFFFFu);
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xf, 0xf, false));   // quad_perm [1,0,3,2]
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xf, 0xf, false));   // quad_perm [2,3,0,1]
  const uint32_t expo = top >> 23;
  uint32_t s = expo <= (uint32_t)Mx<FMT>::EMAX ? 0u : expo - (uint32_t)Mx<FMT>::EMAX;
  const float up = expo == 255u ? 0.0f : mx_power(254u - s);
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = expo == 255u ? 0.0f : v[k] * up;
  if (expo == 255u) s = 255u;
  if (!live) return;
  const int64_t r = mx_row(rows, at.j);
  if (r < 0 || r >= rows.rows) return;                 // a row outside the store is not written
  if (rows.owner && rows.owner[r] != (int32_t)at.j) return;
  const uint64_t row = ((uint64_t)l * (uint32_t)kinds + (uint32_t)kind) * (uint64_t)rows.rows + (uint64_t)r;
  const uint2 code = mx_encode8<FMT>(v);
  if constexpr (FMT == CLT_MXFP4) *reinterpret_cast<uint32_t *>(codes + row * blocks * 16u + at.p * 4u) = code.x;
  else *reinterpret_cast<uint2 *>(codes + row * blocks * 32u + at.p * 8u) = code;
  if ((at.p & 3u) == 0u) scales[row * blocks + (at.p >> 2)] = (uint8_t)s;
}

// Which row of the batch a store row keeps when several name it: the last one.  Cleared, then raised.
__global__ void k_mx_claim(MxRows rows, int64_t n, int32_t *owner, int raise) {
  const int64_t j = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (j >= n) return;
  const int64_t r = mx_row(rows, j);
  if (r < 0 || r >= rows.rows) return;
  if (raise) atomicMax(&owner[r], (int32_t)j);
  else owner[r] = -1;
}

struct MxNorm {
  int mode;
  const float *mean0, *std0, *mean1, *std1;   // [L][d] per kind
  float scale;
};

template <typename OutT, int FMT, bool VEC>
__global__ __launch_bounds__(MX_THREADS) void k_mx_read(const uint8_t *__restrict__ codes, const uint8_t *__restrict__ scales, MxRows rows,
                                                        int64_t n, int64_t d, uint32_t blocks, uint32_t pieces, uint32_t magic, int kinds,
                                                        MxNorm nm, OutT *__restrict__ out0, OutT *__restrict__ out1,
                                                        int64_t out_layer_stride, int64_t out_row_stride) {
  const MxPiece at = mx_piece(pieces, magic);
  if (at.j >= n) return;
  const int64_t l = blockIdx.y / (uint32_t)kinds;
  const int kind = (int)(blockIdx.y - (uint32_t)l * (uint32_t)kinds);
  const int64_t c = (int64_t)at.p * 8;
  const int64_t r = mx_row(rows, at.j);
  float v[8];
  if (r >= 0 && r < rows.rows) {
    const uint64_t row = ((uint64_t)l * (uint32_t)kinds + (uint32_t)kind) * (uint64_t)rows.rows + (uint64_t)r;
    uint2 code = make_uint2(0u, 0u);
    if constexpr (FMT == CLT_MXFP4) code.x = *reinterpret_cast<const uint32_t *>(codes + row * blocks * 16u + at.p * 4u);
    else code = *reinterpret_cast<const uint2 *>(codes + row * blocks * 32u + at.p * 8u);
    const float s = mx_power(scales[row * blocks + (at.p >> 2)]);
    mx_decode8<FMT>(code, v);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] *= s;
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = __uint_as_float(0x7FC00000u);      // a row outside the store is not read
  }
  const float *mean = kind ? nm.mean1 : nm.mean0, *stdv = kind ? nm.std1 : nm.std0;
  if (nm.mode == CLT_DENORM_MEAN_STD && mean && stdv) {
    const float *mp = mean + l * d + c, *tp = stdv + l * d + c;
    if constexpr (VEC) {
      const float4 m0 = *reinterpret_cast<const float4 *>(mp), m1 = *reinterpret_cast<const float4 *>(mp + 4);
      const float4 s0 = *reinterpret_cast<const float4 *>(tp), s1 = *reinterpret_cast<const float4 *>(tp + 4);
      const float mm[8] = {m0.x, m0.y, m0.z, m0.w, m1.x, m1.y, m1.z, m1.w};
      const float ss[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = (v[k] - mm[k]) / ss[k];
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (c + k < d) v[k] = (v[k] - mp[k]) / tp[k];
    }
  } else if (nm.mode == CLT_DENORM_SCALE) {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] *= nm.scale;
  }
  OutT *op = (kind ? out1 : out0) + l * out_layer_stride + at.j * out_row_stride + c;
  if constexpr (VEC) {
    if constexpr (sizeof(OutT) == 2) {
      *reinterpret_cast<uint4 *>(op) = make_uint4(pack_pair<OutT>(v[0], v[1]), pack_pair<OutT>(v[2], v[3]), pack_pair<OutT>(v[4], v[5]),
                                                  pack_pair<OutT>(v[6], v[7]));
    } else {
      *reinterpret_cast<float4 *>(op) = make_float4(v[0], v[1], v[2], v[3]);
      *reinterpret_cast<float4 *>(op + 4) = make_float4(v[4], v[5], v[6], v[7]);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (c + k < d) op[k] = Elem<OutT>::from_f32(v[k]);
  }
}

// ---- the projection -----------------------------------------------------------------------------------------------
typedef __attribute__((ext_vector_type(8))) int mx_i32x8_t;
typedef __attribute__((ext_vector_type(4))) float mx_f32x4_t;

// acc += A . B^T over 128 elements of K on 16 x 16 tiles, both operands mxfp4: lane -> row lane % 16, block lane / 16 of K, its
// 16 bytes of codes and its scale byte (in the low byte of the word)
__device__ __forceinline__ void mx_mma(mx_f32x4_t &acc, const uint4 &a, uint32_t sa, const uint4 &b, uint32_t sb) {
  const mx_i32x8_t av = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0}, bv = {(int)b.x, (int)b.y, (int)b.z, (int)b.w, 0, 0, 0, 0};
  acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, acc, 4, 4, 0, (int)sa, 0, (int)sb);
}

// pre[l][m][n] = b[l][n] + sum over k of x[l][m][k] w[l][n][k].  A wavefront takes 16 NF features x 16 MT tokens, its operands
// straight from memory; rows past the end repeat the last one and store nothing, blocks past the end count as zeros.
template <typename OutT, int NF, int MT>
__global__ __launch_bounds__(256) void k_mx_project(const uint8_t *__restrict__ xc, const uint8_t *__restrict__ xs,
                                                    const uint8_t *__restrict__ wc, const uint8_t *__restrict__ wsc,
                                                    const OutT *__restrict__ bias, OutT *__restrict__ pre, int M, int N, int blocks,
                                                    int64_t bs, int64_t ps, int64_t pre_row) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l15 = lane & 15, lq = lane >> 4;
  const int64_t layer = blockIdx.z;
  const int n0 = (blockIdx.x * 4 + wave) * 16 * NF, m0 = blockIdx.y * 16 * MT;
  if (n0 >= N) return;
  int64_t wrow[NF], xrow[MT];
#pragma unroll
  for (int j = 0; j < NF; ++j) wrow[j] = (layer * N + min(n0 + j * 16 + l15, N - 1)) * blocks;
#pragma unroll
  for (int i = 0; i < MT; ++i) xrow[i] = (layer * M + min(m0 + i * 16 + l15, M - 1)) * blocks;
  mx_f32x4_t acc[MT][NF];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NF; ++j) acc[i][j] = mx_f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  for (int kb = 0; kb < blocks; kb += 4) {
    const bool in = kb + lq < blocks;
    const int k = in ? kb + lq : blocks - 1;
    uint4 a[NF], b[MT];
    uint32_t sa[NF], sb[MT];
#pragma unroll
    for (int j = 0; j < NF; ++j) { a[j] = *reinterpret_cast<const uint4 *>(wc + (wrow[j] + k) * 16); sa[j] = wsc[wrow[j] + k]; }
#pragma unroll
    for (int i = 0; i < MT; ++i) { b[i] = *reinterpret_cast<const uint4 *>(xc + (xrow[i] + k) * 16); sb[i] = xs[xrow[i] + k]; }
    if (!in) {
#pragma unroll
      for (int j = 0; j < NF; ++j) { a[j] = make_uint4(0u, 0u, 0u, 0u); sa[j] = 0u; }
#pragma unroll
      for (int i = 0; i < MT; ++i) { b[i] = make_uint4(0u, 0u, 0u, 0u); sb[i] = 0u; }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NF; ++j) mx_mma(acc[i][j], a[j], sa[j], b[i], sb[i]);
  }
  // a lane holds four neighbouring features of token lane % 16
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int m = m0 + i * 16 + l15;
    if (m >= M) continue;
#pragma unroll
    for (int j = 0; j < NF; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int n = n0 + j * 16 + lq * 4 + q;
        if (n < N) pre[layer * ps + m * pre_row + n] = Elem<OutT>::from_f32(acc[i][j][q] + (bias ? Elem<OutT>::to_f32(bias[layer * bs + n]) : 0.0f));
      }
  }
}

bool mx_format(int fmt) { return fmt == CLT_MXFP4 || fmt == CLT_MXFP8 || fmt == CLT_MXINT8; }
uint32_t mx_magic(uint32_t pieces) { return (uint32_t)((0x100000000ull + pieces - 1) / pieces); }

template <typename T, int FMT>
int launch_mx_write(const void *src0, const void *src1, int64_t layer_stride, int64_t row_stride, int64_t L, int kinds, int64_t n, int64_t d,
                    const MxRows &rows, void *codes, uint8_t *scales, hipStream_t s) {
  const uint32_t blocks = (uint32_t)clt_ceil_div(d, 32), pieces = blocks * 4;
  const int64_t groups = clt_ceil_div(n * (int64_t)pieces, MX_THREADS);
  if (groups > 2147483647LL) return CLT_ERR_RANGE;
  const bool vec = d % 8 == 0 && clt_aligned16(src0) && (kinds == 1 || clt_aligned16(src1)) && (row_stride * (int64_t)sizeof(T)) % 16 == 0 &&
                   (layer_stride * (int64_t)sizeof(T)) % 16 == 0;
  const dim3 grid((unsigned)groups, (unsigned)(L * kinds));
  if (vec)
    k_mx_write<T, FMT, true><<<grid, MX_THREADS, 0, s>>>((const T *)src0, (const T *)src1, layer_stride, row_stride, kinds, n, d, blocks,
                                                         mx_magic(pieces), rows, (uint8_t *)codes, scales);
  else
    k_mx_write<T, FMT, false><<<grid, MX_THREADS, 0, s>>>((const T *)src0, (const T *)src1, layer_stride, row_stride, kinds, n, d, blocks,
                                                          mx_magic(pieces), rows, (uint8_t *)codes, scales);
  return clt_check_launch();
}

template <typename T>
int mx_write_as(int fmt, const void *src0, const void *src1, int64_t layer_stride, int64_t row_stride, int64_t L, int kinds, int64_t n,
                int64_t d, const MxRows &rows, void *codes, uint8_t *scales, hipStream_t s) {
  if (fmt == CLT_MXFP4) return launch_mx_write<T, CLT_MXFP4>(src0, src1, layer_stride, row_stride, L, kinds, n, d, rows, codes, scales, s);
  if (fmt == CLT_MXFP8) return launch_mx_write<T, CLT_MXFP8>(src0, src1, layer_stride, row_stride, L, kinds, n, d, rows, codes, scales, s);
  return launch_mx_write<T, CLT_MXINT8>(src0, src1, layer_stride, row_stride, L, kinds, n, d, rows, codes, scales, s);
}

int mx_write(int dtype, int fmt, const void *src0, const void *src1, int64_t layer_stride, int64_t row_stride, int64_t L, int kinds,
             int64_t n, int64_t d, const MxRows &rows, void *codes, uint8_t *scales, hipStream_t s) {
  if (dtype == CLT_BF16) return mx_write_as<bf16_t>(fmt, src0, src1, layer_stride, row_stride, L, kinds, n, d, rows, codes, scales, s);
  if (dtype == CLT_F16) return mx_write_as<f16_t>(fmt, src0, src1, layer_stride, row_stride, L, kinds, n, d, rows, codes, scales, s);
  return mx_write_as<float>(fmt, src0, src1, layer_stride, row_stride, L, kinds, n, d, rows, codes, scales, s);
}

template <typename OutT, int FMT>
int launch_mx_read(const void *codes, const uint8_t *scales, const MxRows &rows, int64_t L, int kinds, int64_t n, int64_t d, const MxNorm &nm,
                   void *out0, void *out1, int64_t out_layer_stride, int64_t out_row_stride, hipStream_t s) {
  const uint32_t blocks = (uint32_t)clt_ceil_div(d, 32), pieces = (uint32_t)clt_ceil_div(d, 8);
  const int64_t groups = clt_ceil_div(n * (int64_t)pieces, MX_THREADS);
  if (groups > 2147483647LL) return CLT_ERR_RANGE;
  const bool vec = d % 8 == 0 && clt_aligned16(out0) && (kinds == 1 || clt_aligned16(out1)) &&
                   (out_row_stride * (int64_t)sizeof(OutT)) % 16 == 0 && (out_layer_stride * (int64_t)sizeof(OutT)) % 16 == 0 &&
                   clt_aligned16(nm.mean0) && clt_aligned16(nm.std0) && clt_aligned16(nm.mean1) && clt_aligned16(nm.std1);
  const dim3 grid((unsigned)groups, (unsigned)(L * kinds));
  if (vec)
    k_mx_read<OutT, FMT, true><<<grid, MX_THREADS, 0, s>>>((const uint8_t *)codes, scales, rows, n, d, blocks, pieces, mx_magic(pieces), kinds,
                                                           nm, (OutT *)out0, (OutT *)out1, out_layer_stride, out_row_stride);
  else
    k_mx_read<OutT, FMT, false><<<grid, MX_THREADS, 0, s>>>((const uint8_t *)codes, scales, rows, n, d, blocks, pieces, mx_magic(pieces), kinds,
                                                            nm, (OutT *)out0, (OutT *)out1, out_layer_stride, out_row_stride);
  return clt_check_launch();
}

template <typename OutT>
int mx_read_as(int fmt, const void *codes, const uint8_t *scales, const MxRows &rows, int64_t L, int kinds, int64_t n, int64_t d,
               const MxNorm &nm, void *out0, void *out1, int64_t out_layer_stride, int64_t out_row_stride, hipStream_t s) {
  if (fmt == CLT_MXFP4) return launch_mx_read<OutT, CLT_MXFP4>(codes, scales, rows, L, kinds, n, d, nm, out0, out1, out_layer_stride, out_row_stride, s);
  if (fmt == CLT_MXFP8) return launch_mx_read<OutT, CLT_MXFP8>(codes, scales, rows, L, kinds, n, d, nm, out0, out1, out_layer_stride, out_row_stride, s);
  return launch_mx_read<OutT, CLT_MXINT8>(codes, scales, rows, L, kinds, n, d, nm, out0, out1, out_layer_stride, out_row_stride, s);
}

int mx_read(int dtype, int fmt, const void *codes, const uint8_t *scales, const MxRows &rows, int64_t L, int kinds, int64_t n, int64_t d,
            const MxNorm &nm, void *out0, void *out1, int64_t out_layer_stride, int64_t out_row_stride, hipStream_t s) {
  if (dtype == CLT_BF16) return mx_read_as<bf16_t>(fmt, codes, scales, rows, L, kinds, n, d, nm, out0, out1, out_layer_stride, out_row_stride, s);
  if (dtype == CLT_F16) return mx_read_as<f16_t>(fmt, codes, scales, rows, L, kinds, n, d, nm, out0, out1, out_layer_stride, out_row_stride, s);
  return mx_read_as<float>(fmt, codes, scales, rows, L, kinds, n, d, nm, out0, out1, out_layer_stride, out_row_stride, s);
}

template <typename OutT>
int launch_mx_project(const uint8_t *xc, const uint8_t *xs, const uint8_t *wc, const uint8_t *wsc, const void *bias, void *pre, int64_t T,
                      int64_t d, int64_t F, int64_t L, int64_t bs, int64_t ps, int64_t pre_row, hipStream_t s) {
  const int blocks = (int)clt_ceil_div(d, 32);
#define CLT_MXP(NF, MT)                                                                                                          \
  {                                                                                                                              \
    const dim3 grid((unsigned)clt_ceil_div(F, 64 * NF), (unsigned)clt_ceil_div(T, 16 * MT), (unsigned)L);                          \
    if (grid.y > 65535u) return CLT_ERR_RANGE;                                                                                   \
    k_mx_project<OutT, NF, MT><<<grid, 256, 0, s>>>(xc, xs, wc, wsc, (const OutT *)bias, (OutT *)pre, (int)T, (int)F, blocks, bs, ps, pre_row); \
  }
  if (T <= 16) CLT_MXP(2, 1)
  else CLT_MXP(4, 4)
#undef CLT_MXP
  return clt_check_launch();
}

// sizes that every entry point asks for
int mx_sizes(int64_t L, int64_t n, int64_t d, int64_t rows) {
  if (L <= 0 || n < 0 || d <= 0 || rows < 0) return CLT_ERR_ARG;
  if (L > 32767 || d > MX_MAX_WIDTH || n > 2147483647LL || rows > (1LL << 40)) return CLT_ERR_RANGE;
  return CLT_OK;
}

}  // namespace

extern "C" int64_t clt_mx_row_bytes(int64_t d, int fmt) {
  if (d <= 0 || !mx_format(fmt)) return 0;
  return clt_ceil_div(d, 32) * (fmt == CLT_MXFP4 ? 16 : 32);
}

extern "C" int clt_mx_quantise(const void *src, int64_t n, int64_t d, int64_t row_stride, int dtype, int fmt, void *codes, uint8_t *scales,
                               void *stream) {
  if (!clt_model_dtype(dtype)) return CLT_ERR_DTYPE;
  if (!mx_format(fmt)) return CLT_ERR_ARG;
  if (const int rc = mx_sizes(1, n, d, n)) return rc;
  if (n == 0) return CLT_OK;
  if (!src || !codes || !scales || (n > 1 && row_stride < d)) return CLT_ERR_ARG;
  if (!clt_aligned16(codes)) return CLT_ERR_ALIGN;
  const MxRows rows{nullptr, 0, 0, n, nullptr};
  return mx_write(dtype, fmt, src, nullptr, 0, row_stride, 1, 1, n, d, rows, codes, scales, (hipStream_t)stream);
}

extern "C" int clt_mx_dequantise(const void *codes, const uint8_t *scales, int64_t n, int64_t d, int fmt, void *dst, int64_t row_stride,
                                 int dtype, void *stream) {
  if (!clt_model_dtype(dtype)) return CLT_ERR_DTYPE;
  if (!mx_format(fmt)) return CLT_ERR_ARG;
  if (const int rc = mx_sizes(1, n, d, n)) return rc;
  if (n == 0) return CLT_OK;
  if (!dst || !codes || !scales || (n > 1 && row_stride < d)) return CLT_ERR_ARG;
  if (!clt_aligned16(codes)) return CLT_ERR_ALIGN;
  const MxRows rows{nullptr, 0, 0, n, nullptr};
  const MxNorm nm{CLT_DENORM_NONE, nullptr, nullptr, nullptr, nullptr, 1.0f};
  return mx_read(dtype, fmt, codes, scales, rows, 1, 1, n, d, nm, dst, nullptr, 0, row_stride, (hipStream_t)stream);
}

extern "C" int clt_mx_cache_write(const void *x, const void *tgt, int64_t layer_stride, int64_t row_stride, int dtype, const void *row_index,
                                  int index_bits, int64_t first, int64_t n, int64_t d, int64_t L, int fmt, void *codes, uint8_t *scales,
                                  int64_t rows, int32_t *owner, void *stream) {
  if (!clt_model_dtype(dtype)) return CLT_ERR_DTYPE;
  if (!mx_format(fmt) || (row_index && index_bits != 32 && index_bits != 64)) return CLT_ERR_ARG;
  if (const int rc = mx_sizes(L, n, d, rows)) return rc;
  if (n == 0) return CLT_OK;
  if (!x || !tgt || !codes || !scales || row_stride < d || layer_stride < 0) return CLT_ERR_ARG;
  if (row_index ? !owner : (first < 0 || first + n > rows)) return CLT_ERR_ARG;
  if (!clt_aligned16(codes)) return CLT_ERR_ALIGN;
  const MxRows r{row_index, index_bits == 64, first, rows, row_index ? owner : nullptr};
  hipStream_t s = (hipStream_t)stream;
  if (row_index) {
    const unsigned nb = (unsigned)clt_ceil_div(n, 256);
    k_mx_claim<<<nb, 256, 0, s>>>(r, n, owner, 0);
    k_mx_claim<<<nb, 256, 0, s>>>(r, n, owner, 1);
  }
  return mx_write(dtype, fmt, x, tgt, layer_stride, row_stride, L, 2, n, d, r, codes, scales, s);
}

extern "C" int clt_mx_cache_read(const void *codes, const uint8_t *scales, int64_t rows, int fmt, const void *row_index, int index_bits,
                                 int64_t first, int64_t n, int64_t d, int64_t L, int norm_mode, const float *mean_in, const float *std_in,
                                 const float *mean_tg, const float *std_tg, double scale, void *x_out, void *tgt_out, int64_t out_row0,
                                 int64_t T, int out_dtype, void *stream) {
  if (!clt_model_dtype(out_dtype)) return CLT_ERR_DTYPE;
  if (!mx_format(fmt) || (row_index && index_bits != 32 && index_bits != 64)) return CLT_ERR_ARG;
  if (norm_mode < CLT_DENORM_NONE || norm_mode > CLT_DENORM_SCALE) return CLT_ERR_ARG;
  if (const int rc = mx_sizes(L, n, d, rows)) return rc;
  if (T < 0 || out_row0 < 0 || out_row0 + n > T) return CLT_ERR_ARG;
  if (n == 0) return CLT_OK;
  if (!codes || !scales || !x_out || !tgt_out || rows == 0) return CLT_ERR_ARG;
  if (!row_index && (first < 0 || first + n > rows)) return CLT_ERR_ARG;
  if (!clt_aligned16(codes)) return CLT_ERR_ALIGN;
  const MxRows r{row_index, index_bits == 64, first, rows, nullptr};
  const MxNorm nm{norm_mode, mean_in, std_in, mean_tg, std_tg, (float)scale};
  const int64_t e = clt_elem_bytes(out_dtype);
  return mx_read(out_dtype, fmt, codes, scales, r, L, 2, n, d, nm, (char *)x_out + out_row0 * d * e, (char *)tgt_out + out_row0 * d * e, T * d, d,
                 (hipStream_t)stream);
}

extern "C" int clt_mx_encode(const void *x_codes, const uint8_t *x_scales, const void *w_codes, const uint8_t *w_scales, const void *bias,
                             void *pre, int64_t T, int64_t d, int64_t F, int64_t L, int64_t b_layer_stride, int64_t pre_layer_stride,
                             int64_t pre_row_stride, int dtype, void *stream) {
  if (!clt_model_dtype(dtype)) return CLT_ERR_DTYPE;
  if (T < 0 || d <= 0 || F <= 0 || L <= 0) return CLT_ERR_ARG;
  if (T == 0) return CLT_OK;
  if (!x_codes || !x_scales || !w_codes || !w_scales || !pre || pre_row_stride < F || pre_layer_stride < 0) return CLT_ERR_ARG;
  if (d > MX_MAX_WIDTH || T > (1 << 20) || F > (1 << 30) || L > 65535) return CLT_ERR_RANGE;
  if (!clt_aligned16(x_codes) || !clt_aligned16(w_codes)) return CLT_ERR_ALIGN;
  hipStream_t s = (hipStream_t)stream;
  const uint8_t *xc = (const uint8_t *)x_codes, *wc = (const uint8_t *)w_codes;
  if (dtype == CLT_BF16) return launch_mx_project<bf16_t>(xc, x_scales, wc, w_scales, bias, pre, T, d, F, L, b_layer_stride, pre_layer_stride, pre_row_stride, s);
  if (dtype == CLT_F16) return launch_mx_project<f16_t>(xc, x_scales, wc, w_scales, bias, pre, T, d, F, L, b_layer_stride, pre_layer_stride, pre_row_stride, s);
  return launch_mx_project<float>(xc, x_scales, wc, w_scales, bias, pre, T, d, F, L, b_layer_stride, pre_layer_stride, pre_row_stride, s);
}
