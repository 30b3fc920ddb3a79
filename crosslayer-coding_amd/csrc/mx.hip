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
typedef __attribute__((ext_vector_type(2))) __bf16 mx_bf16x2_t;
typedef __attribute__((ext_vector_type(2))) _Float16 mx_f16x2_t;

// two floats as packed 16-bit elements, rounded to nearest even
template <typename T> __device__ __forceinline__ uint32_t mx_pack(float a, float b) {
  const mx_f32x2_t v = {a, b};
  if constexpr (IsHalf<T>::value) return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, mx_f16x2_t));
  else return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, mx_bf16x2_t));
}

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

// grid: x = groups of pieces, y = layer * kinds + kind.  Four lanes hold a block and agree on its scale.  `blocks` of a stored row: those
// behind d are zeros.
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
      *reinterpret_cast<uint4 *>(op) = make_uint4(mx_pack<OutT>(v[0], v[1]), mx_pack<OutT>(v[2], v[3]), mx_pack<OutT>(v[4], v[5]),
                                                  mx_pack<OutT>(v[6], v[7]));
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

// The same with the scale in byte ks of the word.
__device__ __forceinline__ void mx_mma2(mx_f32x4_t &acc, const uint4 &a, uint32_t sa, const uint4 &b, uint32_t sb, int ks) {
  const mx_i32x8_t av = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0}, bv = {(int)b.x, (int)b.y, (int)b.z, (int)b.w, 0, 0, 0, 0};
  if (ks == 0) acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, acc, 4, 4, 0, (int)sa, 0, (int)sb);
  else acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, acc, 4, 4, 1, (int)sa, 1, (int)sb);
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

// ---- the projection of a batch ------------------------------------------------------------------------------------
// Tiles of BM tokens x 256 features, one persistent workgroup of 8 wavefronts (4 along the tokens, 2 along the features) per CU.
// A stage is 256 elements of K: 128 bytes of codes per row - whole cache lines - and 8 of scales, brought straight into
// LDS, chunk c of row r at chunk position c ^ ((r >> 1) & 7), so that the 16 rows of a fragment read lie in all banks.  A lane
// multiplies the blocks 2 lq and 2 lq + 1 of its row (lq = lane / 16): their scales are neighbours and come in one read.
//
// A stage is four quarters of 4 MG products: all tokens of the wavefront x 32 of its features.  The x fragments stay in
// registers for the stage, each being replaced by the next stage's behind its last use; the W fragments of the next quarter are
// read under this one's products.  Two barriers: at the first, behind quarter 0, x and the first half of W have been read by
// everybody, so those loads of the stage after next (and its scales, which have three places) are asked for; at the second,
// behind quarter 2, the rest.  A load has a stage and a half to arrive.  The stages of all of a workgroup's tiles form one
// sequence: the first stages of the next tile travel during the last ones of this tile, and its stores during the next.
constexpr int TN = 256;                       // features of a tile
constexpr int TW = 8;                         // wavefronts
constexpr int TROW = 128;                     // bytes of codes per row and stage
constexpr int TBLOCKS = 8;                    // blocks per row and stage
constexpr int PARK = 2048;                    // bytes of a wavefront's piece of the output tile on its way out

// vmcnt(n), nothing asked of the other counters
constexpr int wait_vm(int n) { return (n & 15) | ((n >> 4) << 14) | 0x0F70; }

__device__ __forceinline__ uint32_t mx_lds(const void *p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void *)p;
}
// 16 or 4 bytes per lane from base + off straight into LDS, lane i at at + 16 i or 4 i.  Not counted by the compiler: the
// waits are written out.
__device__ __forceinline__ void mx_fill16(const void *base, uint32_t off, uint32_t at) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "{m0}"(at) : "memory");
}
__device__ __forceinline__ void mx_fill4(const void *base, uint32_t off, uint32_t at) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dword %0, %1" ::"v"(off), "s"(base), "{m0}"(at) : "memory");
}

struct TileArgs {
  const uint8_t *xc, *xs, *wc, *ws;           // x rows, codes and scales, hold whole stages (zeros behind the end)
  int M, N, tiles_m, tiles_n, total, per_xcd;
  int stages, xpitch, wpitch, xspitch, wspitch;   // bytes of a row of codes, of scales
  int64_t bs, ps, pre_row;
};

template <typename OutT, int MG>
__global__ __launch_bounds__(TW * 64) __attribute__((amdgpu_waves_per_eu(2, 2))) void k_mx_project_tiles(
    TileArgs a, const OutT *__restrict__ bias, OutT *__restrict__ pre) {
  constexpr int BM = 64 * MG;                              // tokens of a tile; a wavefront takes 16 MG x 128
  constexpr int SI = (BM + TN) / 32;                       // loads of the scales of 32 rows
  constexpr int FIRST = MG + 2 + 2, REST = 2;              // loads of a stage per wavefront: x, first half of W, scales; rest of W
  constexpr int LOADS = FIRST + REST;
  constexpr int STAGE = (BM + TN) * TROW, SST = (BM + TN) * TBLOCKS;
  constexpr int HF = 128 / (int)sizeof(OutT);              // features of a parked piece: rows of 128 bytes
  constexpr int STORES = MG * (128 / HF) * 2;              // stores of a whole tile, per wavefront
  constexpr int G = 2 * MG;                                // pairs of products per quarter
  static_assert(LOADS + STORES < 64, "the wait counter holds 63");
  __shared__ __attribute__((aligned(16))) unsigned char ring[2 * STAGE];
  __shared__ __attribute__((aligned(16))) unsigned char sring[3 * SST];
  __shared__ __attribute__((aligned(16))) unsigned char parked[TW * PARK];
  __shared__ __attribute__((aligned(16))) float bias_lds[TW][128];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave & 3, wn = wave >> 2, l15 = lane & 15, lq = lane >> 4;
  const uint32_t ring0 = mx_lds(ring), sring0 = mx_lds(sring);

  // Block b runs on XCD b % 8 and takes every (gridDim / 8)-th of that XCD's share of the tiles, a run of them in an order
  // that goes through 8 feature tiles for each token tile: the W tiles stay in the XCD's L2 while the tokens pass.
  struct At { int layer, m0, n0; };
  auto locate = [&](int t) {
    const int per = a.tiles_m * a.tiles_n;
    At at;
    at.layer = t / per;
    t -= at.layer * per;
    const int g = t / (8 * a.tiles_m), r = t - g * 8 * a.tiles_m;
    const int cnt = min(8, a.tiles_n - g * 8);
    const int tm = r / cnt;
    at.m0 = tm * BM;
    at.n0 = (g * 8 + r - tm * cnt) * TN;
    return at;
  };
  const int step = (int)gridDim.x >> 3;
  const int last_tile = min((((int)blockIdx.x & 7) + 1) * a.per_xcd, a.total);
  int tile = ((int)blockIdx.x & 7) * a.per_xcd + ((int)blockIdx.x >> 3);
  if (tile >= last_tile) return;

  // ---- the loader: where its next stage comes from.  A load of codes brings 8 rows, lane l row l / 8 at chunk position l % 8.
  int in_tile = tile, in_stage = 0;
  uint32_t in_buf = 0, in_sbuf = 0, xo[MG], wo[4], so[2];
  const uint8_t *in_x, *in_w, *in_s[2];
  const uint32_t chunkE = (uint32_t)((lane & 7) ^ (lane >> 4)) * 16u;      // groups of 8 rows that begin at 0 mod 16; at 8: ^ 64
  // x: rows 8 MG wave + 8 i.  W: row groups in the order of the quarters, first half 0 .. 63 and 128 .. 191, rest behind them
  auto w_row = [&](int i) { const int u = (i & 1) * 8 + wave; return (i >> 1) * 64 + (u >> 3) * 128 + (u & 7) * 8; };
  auto aim = [&]() {
    const At at = locate(in_tile);
    int la = lane;                                            // rebuilt for every tile, see the epilogue
    asm volatile("" : "+v"(la));
    const int lr = la >> 3;
    in_x = a.xc + ((int64_t)at.layer * a.M + at.m0) * a.xpitch;
    in_w = a.wc + ((int64_t)at.layer * a.N + at.n0) * a.wpitch;
    const int xl = a.M - 1 - at.m0, wl = a.N - 1 - at.n0;     // rows past the end repeat the last one
#pragma unroll
    for (int i = 0; i < MG; ++i) {
      const int r = (wave * MG + i) * 8;
      xo[i] = (uint32_t)min(r + lr, xl) * (uint32_t)a.xpitch + (chunkE ^ ((r & 8) ? 64u : 0u));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) wo[i] = (uint32_t)min(w_row(i) + lr, wl) * (uint32_t)a.wpitch;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = (wave * 2 + i) % SI * 32;
      const bool of_x = r < BM;
      in_s[i] = of_x ? a.xs + ((int64_t)at.layer * a.M + at.m0) * a.xspitch : a.ws + ((int64_t)at.layer * a.N + at.n0) * a.wspitch;
      so[i] = (uint32_t)min((of_x ? r : r - BM) + (la >> 1), of_x ? xl : wl) * (uint32_t)(of_x ? a.xspitch : a.wspitch);
    }
  };
  // W and its scales are not filled up: behind the end the last block is repeated, and x is zero there
  auto load_w = [&](int i) {
    const int r = w_row(i);
    mx_fill16(in_w, wo[i] + min((uint32_t)in_stage * TROW + (chunkE ^ ((r & 8) ? 64u : 0u)), (uint32_t)a.wpitch - 16u), ring0 + in_buf * STAGE + (uint32_t)(BM + r) * TROW);
  };
  auto load_first = [&](int i) {
    if (i < MG) mx_fill16(in_x + (int64_t)in_stage * TROW, xo[i], ring0 + in_buf * STAGE + (uint32_t)(wave * MG + i) * (8 * TROW));
    else if (i < MG + 2) load_w(i - MG);
    else {
      const int u = (wave * 2 + i - MG - 2) % SI;
      const uint32_t pitch = (uint32_t)(u * 32 < BM ? a.xspitch : a.wspitch);
      mx_fill4(in_s[i - MG - 2], so[i - MG - 2] + min((uint32_t)in_stage * 8u + (uint32_t)(lane & 1) * 4u, pitch - 4u),
               sring0 + in_sbuf * SST + (uint32_t)u * 256u);
    }
  };
  auto load_rest = [&](int i) { load_w(2 + i); };
  auto load_next = [&]() {
    in_buf ^= 1u;
    in_sbuf = in_sbuf == 2 ? 0 : in_sbuf + 1;
    ++in_stage;
  };
  auto load_from = [&]() {                                     // in front of a stage's first load
    if (in_stage != a.stages) return;
    in_stage = 0;
    if (in_tile + step < last_tile) in_tile += step;           // behind the last tile: once more, for nobody
    aim();
  };

  // ---- fragments: row l15 of each group of 16, its blocks 2 lq and 2 lq + 1
  const uint32_t xat = (uint32_t)(wm * 16 * MG + l15) * TROW, wat = (uint32_t)(BM + wn * 128 + l15) * TROW;
  const uint32_t xsat = (uint32_t)(wm * 16 * MG + l15) * TBLOCKS + lq * 2, wsat = (uint32_t)(BM + wn * 128 + l15) * TBLOCKS + lq * 2;
  const uint32_t koff[2] = {(uint32_t)((lq * 2) ^ ((l15 >> 1) & 7)) * 16u, (uint32_t)((lq * 2 + 1) ^ ((l15 >> 1) & 7)) * 16u};
  uint4 fx[MG][2], fw[2][2][2];
  uint32_t sx[MG], sw[2][2];
  auto read_x = [&](uint32_t buf, int i, int ks) { fx[i][ks] = *reinterpret_cast<const uint4 *>(ring + buf * STAGE + xat + i * 16 * TROW + koff[ks]); };
  auto read_xs = [&](uint32_t sbuf, int i) { sx[i] = *reinterpret_cast<const uint16_t *>(sring + sbuf * SST + xsat + i * 16 * TBLOCKS); };
  auto read_w = [&](uint32_t buf, int q, int j, int ks) {
    fw[q & 1][j][ks] = *reinterpret_cast<const uint4 *>(ring + buf * STAGE + wat + (q * 2 + j) * 16 * TROW + koff[ks]);
  };
  auto read_ws = [&](uint32_t sbuf, int q, int j) { sw[q & 1][j] = *reinterpret_cast<const uint16_t *>(sring + sbuf * SST + wsat + (q * 2 + j) * 16 * TBLOCKS); };
  auto meet = [&]() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
  };

  mx_f32x4_t acc[MG][8];
#pragma unroll
  for (int i = 0; i < MG; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[i][j] = mx_f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};

  // The bias of a tile, two features per lane: asked for in front of the stores of the tile before, so that its arrival does not
  // wait for them, and put into LDS behind them.
  float b0 = 0.0f, b1 = 0.0f;
  auto load_bias = [&](int t) {
    if (!bias) return;
    const At at = locate(t);
    int la = lane;
    asm volatile("" : "+v"(la));
    const OutT *bp = bias + (int64_t)at.layer * a.bs;
    const int n = at.n0 + wn * 128 + la * 2;
    b0 = Elem<OutT>::to_f32(bp[min(n, a.N - 1)]);
    b1 = Elem<OutT>::to_f32(bp[min(n + 1, a.N - 1)]);
  };
  auto keep_bias = [&]() { *reinterpret_cast<float2 *>(&bias_lds[wave][lane * 2]) = make_float2(b0, b1); };

  load_bias(tile);
  keep_bias();
  aim();
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    load_from();
#pragma unroll
    for (int i = 0; i < FIRST; ++i) load_first(i);
#pragma unroll
    for (int i = 0; i < REST; ++i) load_rest(i);
    load_next();
  }
  __builtin_amdgcn_s_waitcnt(wait_vm(LOADS));                  // the first stage
  meet();
  uint32_t buf = 0, sbuf = 0;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    read_ws(0, 0, j);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) read_w(0, 0, j, ks);
  }
#pragma unroll
  for (int i = 0; i < MG; ++i) {
    read_xs(0, i);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) read_x(0, i, ks);
  }
  // barriers still to come at which the stores of the tile before are allowed for: STORES of them, no more and no fewer, were
  // sent behind what these wait for
  int behind = 0;

  for (;;) {
    const At at = locate(tile);
#pragma clang loop unroll(disable)
    for (int k = 0; k < a.stages; ++k) {
    load_from();
    const uint32_t next = buf ^ 1u, snext = sbuf == 2 ? 0 : sbuf + 1;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (q == 1 || q == 3) {
        // What the quarters up to the next barrier read has landed: all but the last LOADS loads (and those stores); and this
        // wavefront's reads are over.  The branch is inside the statement: around a block's end the compiler moves products.
        asm volatile("s_cmp_lt_i32 %0, 1\n\ts_cbranch_scc1 .Lmxw%=\n\ts_waitcnt vmcnt(%1) lgkmcnt(0)\n\ts_branch .Lmxd%=\n"
                     ".Lmxw%=:\n\ts_waitcnt vmcnt(%2) lgkmcnt(0)\n.Lmxd%=:"
                     ::"s"(behind), "n"(LOADS + STORES), "n"(LOADS) : "scc", "memory");
        --behind;
        meet();
      }
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const int ks = g / MG, i = g % MG;
#pragma unroll
        for (int j = 0; j < 2; ++j) mx_mma2(acc[i][q * 2 + j], fw[q & 1][j][ks], sw[q & 1][j], fx[i][ks], sx[i], ks);
#pragma unroll
        for (int r = g * 4 / G; r < (g + 1) * 4 / G; ++r) {
          if (q < 3) read_w(buf, q + 1, r & 1, r >> 1);
          else read_w(next, 0, r & 1, r >> 1);
          if (r < 2) { if (q < 3) read_ws(sbuf, q + 1, r); else read_ws(snext, 0, r); }
        }
        if (q == 3) {
          read_x(next, i, ks);
          if (ks == 1) read_xs(snext, i);
        }
        if (q == 1 || q == 2) {
#pragma unroll
          for (int r = ((q - 1) * G + g) * FIRST / (2 * G); r < ((q - 1) * G + g + 1) * FIRST / (2 * G); ++r) load_first(r);
        }
        if (q == 3 && g < REST) load_rest(g);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    load_next();
    buf = next;
    sbuf = snext;
    }
    // ---- the tile goes out: a lane holds four neighbouring features of token l15 of each group of 16 tokens.  They pass
    // through LDS, so that a store is 16 bytes per lane and 128 neighbouring bytes per token.
    const int n1 = at.n0 + wn * 128;
    const bool whole = at.m0 + BM <= a.M && at.n0 + TN <= a.N;
    // addresses are rebuilt from the lane number for every tile: as loop invariants they would live across the K loop
    int le = lane;
    asm volatile("" : "+v"(le));
    const int c15 = le & 15, cq = le >> 4;
    unsigned char *park = parked + wave * PARK;
    constexpr int PE = 16 / (int)sizeof(OutT), JH = HF / 16;
    OutT *op = pre + (int64_t)at.layer * a.ps + (int64_t)(at.m0 + wm * 16 * MG + (le >> 3)) * a.pre_row + n1 + (le & 7) * PE;
    if (tile + step < last_tile) load_bias(tile + step);
#pragma unroll
    for (int h = 0; h < 128 / HF; ++h) {
      float4 bv[JH];
#pragma unroll
      for (int jj = 0; jj < JH; ++jj) bv[jj] = *reinterpret_cast<const float4 *>(&bias_lds[wave][h * HF + jj * 16 + cq * 4]);
#pragma unroll
      for (int i = 0; i < MG; ++i) {
#pragma unroll
        for (int jj = 0; jj < JH; ++jj) {
          const int j = h * JH + jj;
          const float y[4] = {acc[i][j][0] + bv[jj].x, acc[i][j][1] + bv[jj].y, acc[i][j][2] + bv[jj].z, acc[i][j][3] + bv[jj].w};
          acc[i][j] = mx_f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
          if constexpr (sizeof(OutT) == 4) {
            const int slot = (jj * 4 + cq) ^ (c15 & 7);
            *reinterpret_cast<float4 *>(park + c15 * 128 + slot * 16) = make_float4(y[0], y[1], y[2], y[3]);
          } else {
            const int slot = (jj * 2 + (cq >> 1)) ^ (c15 & 7);
            *reinterpret_cast<uint2 *>(park + c15 * 128 + slot * 16 + (cq & 1) * 8) = make_uint2(mx_pack<OutT>(y[0], y[1]), mx_pack<OutT>(y[2], y[3]));
          }
        }
        if (whole) {
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int row = u * 8 + (le >> 3);
            const uint4 v = *reinterpret_cast<const uint4 *>(park + row * 128 + (((le & 7) ^ (row & 7)) * 16));
            __builtin_memcpy(op + (int64_t)(i * 16 + u * 8) * a.pre_row + h * HF, &v, 16);
          }
        } else {
#pragma clang loop unroll(disable)
          for (int u = 0; u < 2; ++u) {
            const int row = u * 8 + (le >> 3), left = min(a.N - (n1 + h * HF + (le & 7) * PE), PE);
            const OutT *vp = reinterpret_cast<const OutT *>(park + row * 128 + (((le & 7) ^ (row & 7)) * 16));
            if (at.m0 + wm * 16 * MG + i * 16 + row < a.M)
#pragma clang loop unroll(disable)
              for (int q = 0; q < left; ++q) op[(int64_t)(i * 16 + u * 8) * a.pre_row + h * HF + q] = vp[q];
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    keep_bias();
    behind = whole ? 3 : 0;
    tile += step;
    if (tile >= last_tile) break;
  }
  __builtin_amdgcn_s_waitcnt(0);   // no load into LDS may be under way when the workgroup ends
}

// Rows of codes and scales with whole stages of K: the blocks behind the end are zeros.
__global__ __launch_bounds__(256) void k_mx_widen(const uint8_t *__restrict__ src, uint8_t *__restrict__ dst, int64_t rows, int from, int to,
                                                  int unit) {
  const int64_t n = rows * to;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / to;
    const int b = (int)(i - r * to);
    if (unit == 16) reinterpret_cast<uint4 *>(dst)[i] = b < from ? reinterpret_cast<const uint4 *>(src)[r * from + b] : make_uint4(0u, 0u, 0u, 0u);
    else dst[i] = b < from ? src[r * from + b] : (uint8_t)0;
  }
}

int launch_mx_widen(const void *src, void *dst, int64_t rows, int64_t from, int64_t to, int unit, hipStream_t s) {
  const int64_t nb = clt_ceil_div(rows * to, 256);
  k_mx_widen<<<(unsigned)(nb < 65536 ? nb : 65536), 256, 0, s>>>((const uint8_t *)src, (uint8_t *)dst, rows, (int)from, (int)to, unit);
  return clt_check_launch();
}

bool mx_format(int fmt) { return fmt == CLT_MXFP4 || fmt == CLT_MXFP8 || fmt == CLT_MXINT8; }
uint32_t mx_magic(uint32_t pieces) { return (uint32_t)((0x100000000ull + pieces - 1) / pieces); }

template <typename T, int FMT>
int launch_mx_write(const void *src0, const void *src1, int64_t layer_stride, int64_t row_stride, int64_t L, int kinds, int64_t n, int64_t d,
                    uint32_t blocks, const MxRows &rows, void *codes, uint8_t *scales, hipStream_t s) {
  const uint32_t pieces = blocks * 4;
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
                int64_t d, uint32_t blocks, const MxRows &rows, void *codes, uint8_t *scales, hipStream_t s) {
  if (fmt == CLT_MXFP4) return launch_mx_write<T, CLT_MXFP4>(src0, src1, layer_stride, row_stride, L, kinds, n, d, blocks, rows, codes, scales, s);
  if (fmt == CLT_MXFP8) return launch_mx_write<T, CLT_MXFP8>(src0, src1, layer_stride, row_stride, L, kinds, n, d, blocks, rows, codes, scales, s);
  return launch_mx_write<T, CLT_MXINT8>(src0, src1, layer_stride, row_stride, L, kinds, n, d, blocks, rows, codes, scales, s);
}

int mx_write(int dtype, int fmt, const void *src0, const void *src1, int64_t layer_stride, int64_t row_stride, int64_t L, int kinds,
             int64_t n, int64_t d, uint32_t blocks, const MxRows &rows, void *codes, uint8_t *scales, hipStream_t s) {
  if (dtype == CLT_BF16) return mx_write_as<bf16_t>(fmt, src0, src1, layer_stride, row_stride, L, kinds, n, d, blocks, rows, codes, scales, s);
  if (dtype == CLT_F16) return mx_write_as<f16_t>(fmt, src0, src1, layer_stride, row_stride, L, kinds, n, d, blocks, rows, codes, scales, s);
  return mx_write_as<float>(fmt, src0, src1, layer_stride, row_stride, L, kinds, n, d, blocks, rows, codes, scales, s);
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

// Batches that the tile kernel takes, in tokens.
constexpr int64_t MX_TILE_MIN_TOKENS = 129;

// What the projection keeps for itself: x in codes, rows of whole stages; the scales of W where its rows are no whole number of
// words.
struct MxPlan {
  int64_t blocks, padded, wsblocks;   // blocks of a row; of a row of x in whole stages; bytes of a row of W's scales
  bool tiles;
  size_t xc, xs, ws, bytes;           // offsets in the workspace
};
MxPlan mx_plan(int64_t T, int64_t d, int64_t F, int64_t L, bool quantised) {
  MxPlan p{};
  p.blocks = clt_ceil_div(d, 32);
  p.tiles = T >= MX_TILE_MIN_TOKENS;
  p.padded = p.tiles ? (p.blocks + TBLOCKS - 1) / TBLOCKS * TBLOCKS : p.blocks;
  p.wsblocks = p.tiles ? (p.blocks + 3) / 4 * 4 : p.blocks;
  const bool own_x = !quantised || p.padded != p.blocks;
  auto up = [](size_t n) { return (n + 255) & ~(size_t)255; };
  p.xs = up(own_x ? (size_t)(L * T * p.padded * 16) : 0);
  p.ws = p.xs + up(own_x ? (size_t)(L * T * p.padded) : 0);
  p.bytes = p.ws + up(p.wsblocks != p.blocks ? (size_t)(L * F * p.wsblocks) : 0);
  return p;
}

// One persistent workgroup per CU, a whole number of rounds over the 8 XCDs; 0 when the device cannot be asked.
int mx_grid(int64_t tiles) {
  int dev = 0, cus = 0;
  if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus < 8) return 0;
  const int64_t per = clt_ceil_div(tiles, 8);
  return (int)(per * 8 < cus - cus % 8 ? per * 8 : cus - cus % 8);
}

template <typename OutT>
int launch_mx_project(const MxPlan &p, const uint8_t *xc, const uint8_t *xs, const uint8_t *wc, const uint8_t *wsc, const void *bias, void *pre,
                      int64_t T, int64_t F, int64_t L, int64_t bs, int64_t ps, int64_t pre_row, hipStream_t s) {
  if (p.tiles) {
    constexpr int MG = 4;
    const int64_t tm = clt_ceil_div(T, 64 * MG), tn = clt_ceil_div(F, TN), total = tm * tn * L;
    if (total > 1073741824LL) return CLT_ERR_RANGE;
    const int grid = mx_grid(total);
    if (grid <= 0) return CLT_ERR_LAUNCH;
    TileArgs a{xc, xs, wc, wsc, (int)T, (int)F, (int)tm, (int)tn, (int)total, (int)clt_ceil_div(total, 8), (int)(p.padded / TBLOCKS),
               (int)p.padded * 16, (int)p.blocks * 16, (int)p.padded, (int)p.wsblocks, bs, ps, pre_row};
    k_mx_project_tiles<OutT, MG><<<grid, TW * 64, 0, s>>>(a, (const OutT *)bias, (OutT *)pre);
    return clt_check_launch();
  }
  const int blocks = (int)p.blocks;
#define CLT_MXP(NF, MT)                                                                                                          \
  {                                                                                                                              \
    const dim3 grid((unsigned)clt_ceil_div(F, 64 * NF), (unsigned)clt_ceil_div(T, 16 * MT), (unsigned)L);                          \
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
  return mx_write(dtype, fmt, src, nullptr, 0, row_stride, 1, 1, n, d, (uint32_t)clt_ceil_div(d, 32), rows, codes, scales, (hipStream_t)stream);
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
  return mx_write(dtype, fmt, x, tgt, layer_stride, row_stride, L, 2, n, d, (uint32_t)clt_ceil_div(d, 32), r, codes, scales, s);
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

extern "C" size_t clt_mx_encode_workspace_bytes(int64_t T, int64_t d, int64_t F, int64_t L, int x_quantised) {
  if (T <= 0 || d <= 0 || F <= 0 || L <= 0 || d > MX_MAX_WIDTH) return 0;
  return mx_plan(T, d, F, L, x_quantised != 0).bytes;
}

extern "C" int clt_mx_encode(const void *x, const uint8_t *x_scales, const void *w_codes, const uint8_t *w_scales, const void *bias, void *pre,
                             int64_t T, int64_t d, int64_t F, int64_t L, int64_t x_layer_stride, int64_t b_layer_stride,
                             int64_t pre_layer_stride, int64_t pre_row_stride, int dtype, void *workspace, size_t workspace_bytes, void *stream) {
  if (!clt_model_dtype(dtype)) return CLT_ERR_DTYPE;
  if (T < 0 || d <= 0 || F <= 0 || L <= 0) return CLT_ERR_ARG;
  if (T == 0) return CLT_OK;
  if (!x || !w_codes || !w_scales || !pre || pre_row_stride < F || pre_layer_stride < 0 || (!x_scales && x_layer_stride < 0)) return CLT_ERR_ARG;
  if (d > MX_MAX_WIDTH || T > (1 << 20) || F > (1 << 30) || L > 32767) return CLT_ERR_RANGE;
  if ((x_scales && !clt_aligned16(x)) || !clt_aligned16(w_codes)) return CLT_ERR_ALIGN;
  const MxPlan p = mx_plan(T, d, F, L, x_scales != nullptr);
  if (p.bytes > 0 && (!workspace || workspace_bytes < p.bytes)) return CLT_ERR_WORKSPACE;
  if (p.bytes > 0 && !clt_aligned16(workspace)) return CLT_ERR_ALIGN;
  // the tile kernel fetches four scales at a time
  if (p.tiles && ((p.wsblocks == p.blocks && ((uintptr_t)w_scales & 3u) != 0) || (p.padded == p.blocks && ((uintptr_t)x_scales & 3u) != 0)))
    return CLT_ERR_ALIGN;
  hipStream_t s = (hipStream_t)stream;
  uint8_t *ws = (uint8_t *)workspace;
  const uint8_t *xc = (const uint8_t *)x, *xs = x_scales, *wc = (const uint8_t *)w_codes, *wsc = w_scales;
  int rc = CLT_OK;
  if (!x_scales) {
    const MxRows rows{nullptr, 0, 0, T, nullptr};
    rc = mx_write(dtype, CLT_MXFP4, x, nullptr, x_layer_stride, d, L, 1, T, d, (uint32_t)p.padded, rows, ws + p.xc, ws + p.xs, s);
    xc = ws + p.xc;
    xs = ws + p.xs;
  } else if (p.padded != p.blocks) {
    rc = launch_mx_widen(x, ws + p.xc, L * T, p.blocks, p.padded, 16, s);
    if (rc == CLT_OK) rc = launch_mx_widen(x_scales, ws + p.xs, L * T, p.blocks, p.padded, 1, s);
    xc = ws + p.xc;
    xs = ws + p.xs;
  }
  if (rc == CLT_OK && p.wsblocks != p.blocks) {
    rc = launch_mx_widen(w_scales, ws + p.ws, L * F, p.blocks, p.wsblocks, 1, s);
    wsc = ws + p.ws;
  }
  if (rc != CLT_OK) return rc;
  if (dtype == CLT_BF16) return launch_mx_project<bf16_t>(p, xc, xs, wc, wsc, bias, pre, T, F, L, b_layer_stride, pre_layer_stride, pre_row_stride, s);
  if (dtype == CLT_F16) return launch_mx_project<f16_t>(p, xc, xs, wc, wsc, bias, pre, T, F, L, b_layer_stride, pre_layer_stride, pre_row_stride, s);
  return launch_mx_project<float>(p, xc, xs, wc, wsc, bias, pre, T, F, L, b_layer_stride, pre_layer_stride, pre_row_stride, s);
}
