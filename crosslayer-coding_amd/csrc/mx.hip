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
#include <type_traits>
#include "clt_common.h"

namespace {

constexpr int MX_THREADS = 256;
constexpr int64_t MX_MAX_GROUPS = (1 << 24) - 1;   // workgroups of 256 threads along one axis: a launch takes fewer than 2^32 threads there
constexpr int64_t MX_MAX_ROWS = 1LL << 40;  // of a store or an output, per layer: far more than memory holds, and their bytes are counted with 64 bits
constexpr int64_t MX_MAX_WIDTH = 262144;    // elements of a row: the pieces of a workgroup's rows are told apart with 32 bits

// The tiles of the projection: MX_BM tokens (four wavefronts of MX_MG groups of 16) x TN features, K in stages of TBLOCKS blocks.
constexpr int MX_MG = 4, MX_BM = 64 * MX_MG, TN = 256, TBLOCKS = 8;

// Where the scale of block b of row r of a tile lies among those of its stage.  The rows of a wavefront are `groups` groups of
// 16; a word holds a lane's bytes of two groups and both blocks, and the lanes' words are neighbours.
__host__ __device__ __forceinline__ uint32_t mx_scale_place(uint32_t r, uint32_t b, uint32_t groups) {
  const uint32_t w = r / (16 * groups), i = r / 16 % groups, lane = (b & 3) * 16 + (r & 15);
  return ((w * (groups / 2) + (i >> 1)) * 64 + lane) * 4 + (i & 1) * 2 + (b >> 2);
}

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
typedef __attribute__((ext_vector_type(4))) unsigned int mx_u32x4_t;
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

// A workgroup takes 256 neighbouring pieces: row and place in it from 32-bit numbers counted from the group's first row.
// magic = ceil(2^32 / pieces) = (2^32 + e) / pieces, e < pieces: the quotient of `at` is exact while at * e < 2^32 (pieces - at % pieces),
// which holds for at < pieces + 256 and pieces <= MX_MAX_WIDTH / 4 = 2^16 (at = pieces - 1 is the tightest).
// A thread goes on to the same piece of `rows_apart` rows further on, so that several loads are under way and what belongs to
// the column is fetched once.
struct MxPiece { int64_t j; uint32_t p; };
__device__ __forceinline__ MxPiece mx_piece(uint32_t group, uint32_t pieces, uint32_t magic) {
  const uint64_t base = (uint64_t)group * MX_THREADS;
  const uint64_t row0 = base / pieces;
  const uint32_t at = (uint32_t)(base - row0 * pieces) + threadIdx.x;
  const uint32_t dj = pieces == 1u ? at : __umulhi(at, magic);
  return {(int64_t)(row0 + dj), at - dj * pieces};
}

// Eight elements from sp on (those in front of `left` are there), as floats.
template <typename T, bool VEC> __device__ __forceinline__ void mx_load8(const T *sp, int64_t left, float *v) {
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = 0.0f;
  if constexpr (VEC) {
    if (left > 0) {                                    // whole pieces
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
      if (k < left) v[k] = Elem<T>::to_f32(sp[k]);
  }
}

// The scale byte of the block that two neighbouring lanes hold a half of each; v is scaled for it.
template <int FMT> __device__ __forceinline__ uint32_t mx_scale16(float (&v)[16]) {
  uint32_t top = 0;                                    // magnitudes in the order of their bits: NaN above infinity above all numbers
#pragma unroll
  for (int k = 0; k < 16; ++k) top = max(top, __float_as_uint(v[k]) & 0x7FFFFFFFu);
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xf, 0xf, false));   // quad_perm [1,0,3,2]
  const uint32_t expo = top >> 23;
  const uint32_t s = expo <= (uint32_t)Mx<FMT>::EMAX ? 0u : expo - (uint32_t)Mx<FMT>::EMAX;
  const float up = expo == 255u ? 0.0f : mx_power(254u - s);
#pragma unroll
  for (int k = 0; k < 16; ++k) v[k] = expo == 255u ? 0.0f : v[k] * up;
  return expo == 255u ? 255u : s;
}

// grid: x = groups of pieces, y = layer * kinds + kind.  A piece is half a block: two lanes agree on its scale.  `blocks` of a stored
// row: those behind d are zeros.  tiled: scales as the projection's tiles of MX_BM rows take them.
//
// Bound by memory: 12 x 24576 rows of 768 bf16 to mxfp4 106 us (573 MB, 5.4 TB/s; past the caches 140 us); 12 layers of 4096 x 768 bf16,
// inputs and targets, into mxfp8 49 us from memory, 28 us where the batch is still in the memory-side cache.
struct MxWrite {
  const void *src0, *src1;
  int64_t layer_stride, row_stride, n, d;
  int kinds;
  uint32_t blocks, magic;
  MxRows rows;
  uint8_t *codes, *scales;
};
template <typename T, int FMT, bool VEC, bool TILED>
__device__ __forceinline__ void mx_write_piece(const MxWrite &a, uint32_t group) {
  const int kinds = a.kinds;
  const uint32_t blocks = a.blocks;
  const MxRows &rows = a.rows;
  const MxPiece at = mx_piece(group, blocks * 2u, a.magic);
  if (at.j >= a.n) return;                               // whole pairs: a row has whole blocks
  const int64_t l = blockIdx.y / (uint32_t)kinds;
  const int kind = (int)(blockIdx.y - (uint32_t)l * (uint32_t)kinds);
  const int64_t c = (int64_t)at.p * 16;
  const T *sp = (const T *)(kind ? a.src1 : a.src0) + l * a.layer_stride + at.j * a.row_stride + c;
  float v[16];
  mx_load8<T, VEC>(sp, a.d - c, v);
  mx_load8<T, VEC>(sp + 8, a.d - c - 8, v + 8);
  const int64_t r = mx_row(rows, at.j);
  const uint32_t s = mx_scale16<FMT>(v);
  if (r < 0 || r >= rows.rows) return;                 // a row outside the store is not written
  if (rows.owner && rows.owner[r] != (int32_t)at.j) return;
  const uint64_t row = ((uint64_t)l * (uint32_t)kinds + (uint32_t)kind) * (uint64_t)rows.rows + (uint64_t)r;
  const uint2 lo = mx_encode8<FMT>(*reinterpret_cast<float (*)[8]>(v)), hi = mx_encode8<FMT>(*reinterpret_cast<float (*)[8]>(v + 8));
  if constexpr (FMT == CLT_MXFP4) *reinterpret_cast<uint2 *>(a.codes + row * blocks * 16u + at.p * 8u) = make_uint2(lo.x, hi.x);
  else *reinterpret_cast<uint4 *>(a.codes + row * blocks * 32u + at.p * 16u) = make_uint4(lo.x, lo.y, hi.x, hi.y);
  if ((at.p & 1u) == 0u) {
    const uint32_t blk = at.p >> 1;
    if constexpr (!TILED) a.scales[row * blocks + blk] = (uint8_t)s;
    else a.scales[row / MX_BM * MX_BM * blocks + (blk / 8) * (MX_BM * 8) + mx_scale_place((uint32_t)(row % MX_BM), blk % 8, MX_MG)] = (uint8_t)s;
  }
}
template <typename T, int FMT, bool VEC> __global__ __launch_bounds__(MX_THREADS) void k_mx_write(MxWrite a) {
  mx_write_piece<T, FMT, VEC, false>(a, blockIdx.x);
}

// ---- weights that may have been written -------------------------------------------------------------------------------
// Whether rows [L][n][d] still are what their fingerprint says: 64 bytes of every row, at places that go round, so that every row
// and, from d / 32 rows on (16 bits), every column is looked at.  A layer's sums are of whole numbers, in any order; its last
// workgroup compares and stores.
// state: [L][16], a 128-byte line per layer: sum, workgroups that have arrived, fingerprint.
//
// 12 x 24576 rows of 768 bf16: 19 MB in 64-byte pieces, 21 us (0.9 TB/s), of a layer's 64 workgroups; bound by the latency of six
// rounds, since each load of a lane lies behind a branch and is waited for before the next.  Eight workgroups a layer, one column a
// round: 196 us.
constexpr int WATCH_BLOCKS = 64, WATCH_ROWS = WATCH_BLOCKS * 64;
template <typename T>
__global__ __launch_bounds__(256) void k_mx_watch(const T *__restrict__ src, int64_t layer_stride, int64_t n, int64_t d,
                                                  unsigned long long *__restrict__ state, int32_t *__restrict__ changed, int store_only) {
  constexpr int PE = 16 / (int)sizeof(T);                  // elements of a lane's piece, a quarter of a row's sample
  __shared__ unsigned long long part[4];
  const int64_t l = blockIdx.y;
  const T *base = src + l * layer_stride;
  unsigned long long h = 0;
  const int runs = (int)((d + 4 * PE - 1) / (4 * PE)), step = WATCH_ROWS % runs;
  int place = (blockIdx.x * 64 + (threadIdx.x >> 2)) % runs;
#pragma unroll 6
  for (int64_t r = (int64_t)blockIdx.x * 64 + (threadIdx.x >> 2); r < n; r += WATCH_ROWS) {
    const int64_t c = (int64_t)place * (4 * PE) + (threadIdx.x & 3) * PE;
    place += step;
    if (place >= runs) place -= runs;
    uint32_t w[4] = {0u, 0u, 0u, 0u};
    if (c + PE <= d) __builtin_memcpy(w, base + r * d + c, 16);
    else {
      T e[PE] = {};
#pragma unroll
      for (int k = 0; k < PE; ++k)
        if (c + k < d) e[k] = base[r * d + c + k];
      __builtin_memcpy(w, e, 16);
    }
    unsigned long long v = ((unsigned long long)w[1] << 32 | w[0]) * 0x9E3779B97F4A7C15ull ^ (unsigned long long)(r * 4 + (threadIdx.x & 3)) * 0xC2B2AE3D27D4EB4Full;
    v = (v ^ (v >> 29)) * 0xBF58476D1CE4E5B9ull + ((unsigned long long)w[3] << 32 | w[2]);
    v = (v ^ (v >> 32)) * 0x94D049BB133111EBull;
    h += v ^ (v >> 31);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) h += __shfl_xor(h, o);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = h;
  __syncthreads();
  if (threadIdx.x != 0) return;
  unsigned long long *line = state + l * 16;
  atomicAdd(line, part[0] + part[1] + part[2] + part[3]);
  __threadfence();
  if (atomicAdd(line + 1, 1ull) != (unsigned long long)(gridDim.x - 1)) return;
  __threadfence();
  const unsigned long long now = atomicExch(line, 0ull);    // and ready for the next call
  atomicExch(line + 1, 0ull);
  changed[l] = !store_only && line[2] != now;
  line[2] = now;
}

// mxfp4 rows of the layers that `changed` names; the others cost a launch and no more: 4 us, with a workgroup for every 256 pieces,
// as a batch is written, 22 us.
constexpr int REQUANTISE_BLOCKS = 256;
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void k_mx_requantise(const T *__restrict__ src, int64_t layer_stride, int64_t n, int64_t d, int64_t blocks,
                                                       uint8_t *__restrict__ codes, uint8_t *__restrict__ scales, const int32_t *__restrict__ changed) {
  const int64_t l = blockIdx.y;
  if (changed[l] == 0) return;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n * blocks * 2; i += REQUANTISE_BLOCKS * 256) {   // pairs stay together
    const int64_t j = i / (blocks * 2), p = i - j * blocks * 2, c = p * 16;
    const T *sp = src + l * layer_stride + j * d + c;
    float v[16];
    mx_load8<T, VEC>(sp, d - c, v);
    mx_load8<T, VEC>(sp + 8, d - c - 8, v + 8);
    const uint32_t s = mx_scale16<CLT_MXFP4>(v);
    const uint2 a = mx_encode8<CLT_MXFP4>(*reinterpret_cast<float (*)[8]>(v)), b = mx_encode8<CLT_MXFP4>(*reinterpret_cast<float (*)[8]>(v + 8));
    const int64_t row = l * n + j;
    *reinterpret_cast<uint2 *>(codes + row * blocks * 16 + p * 8) = make_uint2(a.x, b.x);
    if ((p & 1) == 0) scales[row * blocks + (p >> 1)] = (uint8_t)s;
  }
}

template <typename T>
int launch_mx_refresh(const void *src, int64_t layer_stride, int64_t L, int64_t n, int64_t d, void *codes, uint8_t *scales, uint64_t *state,
                      int32_t *changed, int store_only, hipStream_t s) {
  k_mx_watch<T><<<dim3(WATCH_BLOCKS, (unsigned)L), 256, 0, s>>>((const T *)src, layer_stride, n, d, (unsigned long long *)state, changed, store_only);
  if (store_only) return clt_check_launch();
  const int64_t blocks = clt_ceil_div(d, 32);
  const dim3 grid(REQUANTISE_BLOCKS, (unsigned)L);
  if (d % 8 == 0 && clt_aligned16(src) && d * (int64_t)sizeof(T) % 16 == 0 && layer_stride * (int64_t)sizeof(T) % 16 == 0)
    k_mx_requantise<T, true><<<grid, 256, 0, s>>>((const T *)src, layer_stride, n, d, blocks, (uint8_t *)codes, scales, changed);
  else
    k_mx_requantise<T, false><<<grid, 256, 0, s>>>((const T *)src, layer_stride, n, d, blocks, (uint8_t *)codes, scales, changed);
  return clt_check_launch();
}

// Which row of the batch a store row keeps when several name it: the last one.  Cleared, then raised: two launches of 1.8 us (one
// workgroup that does both takes 6.6 us for 501 rows, from one round trip to memory to the next).
__global__ __launch_bounds__(256) void k_mx_claim(MxRows rows, int64_t n, int32_t *owner, int raise) {
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

// a / s by the reciprocal r of s, corrected once: the quotient rounded to nearest where nothing of it leaves the range of normal
// numbers.  Eight divisions a thread in the hardware's steps took longer than the bytes (12 layers of 4096 x 768 rows drawn from
// mxfp8, normalised, to bf16: 67 us, and 49 like this).
__device__ __forceinline__ float mx_quotient(float a, float s, float r) {
  const float q = a * r, better = fmaf(fmaf(-q, s, a), r, q);
  return fabsf(q) <= 0x1p126f ? better : q;
}

// A thread gives out 16 bytes of U rows: E elements from one place on.  LINES: rows of the result are whole cache lines, so that
// a wavefront's stores are too; they go past the caches, which would hold back the reads behind them.  12 x 24576 rows of 768 from
// mxfp4 to bf16: 80 us where the codes are in the memory-side cache from the pass before and 105 where they come from memory, through the
// caches 109 and 108; 16 layers of 3001 x 2048 rows drawn from mxfp4 to float32, inputs and targets: 121 us for rows that were just
// read, 210 for others, through the caches 240 and 239.  Two rows a thread: four take 131 us on the second of these, on rows just read.
template <typename OutT, int FMT, bool VEC, int U, bool LINES>
__global__ __launch_bounds__(MX_THREADS) void k_mx_read(const uint8_t *__restrict__ codes, const uint8_t *__restrict__ scales, MxRows rows,
                                                        int64_t n, int64_t rows_apart, int64_t d, uint32_t blocks, uint32_t pieces,
                                                        uint32_t magic, int kinds, MxNorm nm, OutT *__restrict__ out0,
                                                        OutT *__restrict__ out1, int64_t out_layer_stride, int64_t out_row_stride) {
  constexpr int E = VEC && sizeof(OutT) == 4 ? 4 : 8;
  const MxPiece at = mx_piece(blockIdx.x, pieces, magic);
  if (at.j >= rows_apart) return;
  const int64_t l = blockIdx.y / (uint32_t)kinds;
  const int kind = (int)(blockIdx.y - (uint32_t)l * (uint32_t)kinds);
  const int64_t c = (int64_t)at.p * E;
  const uint64_t slab = ((uint64_t)l * (uint32_t)kinds + (uint32_t)kind) * (uint64_t)rows.rows;
  uint2 code[U];
  uint32_t sb[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t j = at.j + u * rows_apart;
    const int64_t r = j < n ? mx_row(rows, j) : -1;
    code[u] = make_uint2(0u, 0u);
    sb[u] = 255u;                                      // a row outside the store is not read
    if (r >= 0 && r < rows.rows) {
      const uint64_t row = slab + (uint64_t)r;
      const uint8_t *cp = codes + row * blocks * (uint32_t)Mx<FMT>::BLOCK_BYTES + (uint64_t)(FMT == CLT_MXFP4 ? c / 2 : c);
      if constexpr (FMT == CLT_MXFP4 && E == 4) code[u].x = *reinterpret_cast<const uint16_t *>(cp);
      else if constexpr (FMT == CLT_MXFP4 || E == 4) code[u].x = *reinterpret_cast<const uint32_t *>(cp);
      else code[u] = *reinterpret_cast<const uint2 *>(cp);
      sb[u] = scales[row * blocks + (uint64_t)(c / 32)];
    }
  }
  const float *mean = kind ? nm.mean1 : nm.mean0, *stdv = kind ? nm.std1 : nm.std0;
  const bool centred = nm.mode == CLT_DENORM_MEAN_STD && mean && stdv;
  float mm[E], ss[E], rr[E];
  bool plain = true;                                   // reciprocals that keep the correction among normal numbers
  if (centred) {
    if constexpr (VEC) {                               // (of any alignment)
      __builtin_memcpy(mm, mean + l * d + c, sizeof(mm));
      __builtin_memcpy(ss, stdv + l * d + c, sizeof(ss));
    } else {
#pragma unroll
      for (int k = 0; k < E; ++k) {
        mm[k] = c + k < d ? mean[l * d + c + k] : 0.0f;
        ss[k] = c + k < d ? stdv[l * d + c + k] : 1.0f;
      }
    }
#pragma unroll
    for (int k = 0; k < E; ++k) {
      const float r = __builtin_amdgcn_rcpf(ss[k]);
      rr[k] = fmaf(fmaf(-ss[k], r, 1.0f), r, r);
      plain = plain && fabsf(ss[k]) >= 0x1p-100f && fabsf(ss[k]) <= 0x1p100f;
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t j = at.j + u * rows_apart;
    if (j >= n) break;
    float v[8];
    mx_decode8<FMT>(code[u], v);
    const float s = mx_power(sb[u]);
#pragma unroll
    for (int k = 0; k < E; ++k) v[k] *= s;
    if (centred) {
      if (plain) {
#pragma unroll
        for (int k = 0; k < E; ++k) v[k] = mx_quotient(v[k] - mm[k], ss[k], rr[k]);
      } else {
#pragma clang loop unroll(disable)
        for (int k = 0; k < E; ++k) v[k] = (v[k] - mean[l * d + min(c + k, d - 1)]) / stdv[l * d + min(c + k, d - 1)];
      }
    } else if (nm.mode == CLT_DENORM_SCALE) {
#pragma unroll
      for (int k = 0; k < E; ++k) v[k] *= nm.scale;
    }
    OutT *op = (kind ? out1 : out0) + l * out_layer_stride + j * out_row_stride + c;
    if constexpr (!VEC) {
#pragma unroll
      for (int k = 0; k < E; ++k)
        if (c + k < d) op[k] = Elem<OutT>::from_f32(v[k]);
    } else {
      mx_u32x4_t o;
      if constexpr (sizeof(OutT) == 2) o = mx_u32x4_t{mx_pack<OutT>(v[0], v[1]), mx_pack<OutT>(v[2], v[3]), mx_pack<OutT>(v[4], v[5]), mx_pack<OutT>(v[6], v[7])};
      else o = mx_u32x4_t{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
      if constexpr (LINES) __builtin_nontemporal_store(o, reinterpret_cast<mx_u32x4_t *>(op));
      else *reinterpret_cast<mx_u32x4_t *>(op) = o;
    }
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

// The same onto c, with the scales in bytes ka and kb of their words.
template <int KA, int KB> __device__ __forceinline__ mx_f32x4_t mx_mma_at(const mx_f32x4_t &c, const uint4 &a, uint32_t sa, const uint4 &b, uint32_t sb) {
  const mx_i32x8_t av = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0}, bv = {(int)b.x, (int)b.y, (int)b.z, (int)b.w, 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, 4, 4, KA, (int)sa, KB, (int)sb);
}
__device__ __forceinline__ mx_f32x4_t mx_mma2(const mx_f32x4_t &c, const uint4 &a, uint32_t sa, int ka, const uint4 &b, uint32_t sb, int kb) {
  switch (ka * 4 + kb) {                                       // known where this is unrolled; both bytes are of the same block
    case 0: return mx_mma_at<0, 0>(c, a, sa, b, sb);
    case 2: return mx_mma_at<0, 2>(c, a, sa, b, sb);
    case 5: return mx_mma_at<1, 1>(c, a, sa, b, sb);
    case 7: return mx_mma_at<1, 3>(c, a, sa, b, sb);
    case 8: return mx_mma_at<2, 0>(c, a, sa, b, sb);
    case 10: return mx_mma_at<2, 2>(c, a, sa, b, sb);
    case 13: return mx_mma_at<3, 1>(c, a, sa, b, sb);
    default: return mx_mma_at<3, 3>(c, a, sa, b, sb);
  }
}

// ---- the projection of few tokens ---------------------------------------------------------------------------------
// pre[l][m][n] = b[l][n] + sum over k of x[l][m][k] w[l][n][k].  The weights' one pass through the chip is the work: a wavefront
// takes 32 features x 16 MT tokens, W straight from memory into registers, FEW_STEPS steps of 128 elements of K ahead of the products,
// also across its features' end; a workgroup goes on to other features of its layer and keeps x, as codes, in LDS.
// SRC says where x comes from: FEW_VALUES are quantised into LDS by every workgroup, FEW_CODES copied there; FEW_WIDE rows do not
// fit and are read as they are used.  Rows past the end repeat the last one and store nothing, blocks past the end count as zeros.
constexpr int FEW_VALUES = 0, FEW_CODES = 1, FEW_WIDE = 2;
// K is filled up to whole runs of FEW_STEPS steps of 128, whose loads and products behind the end are in vain: with three nothing at
// d = 768 and 1536, an eighth at 1024 and 2048, a fifth at 640, a half at 256 and 512.  Three were chosen at d = 768;
// over other widths two are as fast or faster, but for d = 9473 .. 9600, whose rows then no longer fit into LDS (4 layers, F 4096,
// one token, d 9536: 29 us with three, 64 with two).  One token of 12 layers with 120 MB of weights in all, us with three / two steps:
// d 256 38 / 31, 512 38 / 29, 640 27 / 27, 768 26 / 24, 1024 42 / 38, 1536 32 / 31, 2048 54 / 48, 4096 36 / 35 (above 1024 x has a
// launch of its own, MX_FEW_VALUES).
constexpr int FEW_STEPS = 3, FEW_NF = 2, FEW_TN = 4 * 16 * FEW_NF;   // features of a workgroup
constexpr int FEW_LDS = 80 * 1024;                                   // two workgroups per CU at least

struct FewArgs {
  const void *x;               // values, or codes
  const uint8_t *xs, *wc, *ws;
  int64_t x_layer, bs, ps, pre_row;
  int M, N, d, blocks, vec;
};
__host__ __device__ static inline int few_blocks(int blocks) { return (blocks + 4 * FEW_STEPS - 1) / (4 * FEW_STEPS) * (4 * FEW_STEPS); }
// a row of codes in LDS: an odd number of 16-byte chunks, so that neighbouring rows begin in other banks
__host__ __device__ static inline int few_pitch(int blocks) { return few_blocks(blocks) | 1; }
static inline int few_lds(int blocks, int mt) { return 16 * mt * (few_pitch(blocks) * 16 + few_blocks(blocks)); }

template <typename OutT, int MT, int SRC>
__global__ __launch_bounds__(256, 2) void k_mx_project_few(FewArgs a, const OutT *__restrict__ bias, OutT *__restrict__ pre) {
  extern __shared__ __attribute__((aligned(16))) uint8_t few_x[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l15 = lane & 15, lq = lane >> 4;
  const int64_t layer = blockIdx.y;
  const int m0 = blockIdx.z * 16 * MT, P = few_blocks(a.blocks), pitch = few_pitch(a.blocks);
  uint8_t *few_s = few_x + 16 * MT * pitch * 16;
  if constexpr (SRC == FEW_VALUES) {
    const OutT *x = (const OutT *)a.x + layer * a.x_layer;
    for (int t = threadIdx.x; t < 16 * MT * P * 2; t += 256) {         // half blocks; both halves of one in neighbouring lanes
      const int r = t / (2 * P), h = t - r * 2 * P, c = h * 16, m = m0 + r;
      const int left = m < a.M ? a.d - c : 0;
      const OutT *sp = x + (int64_t)m * a.d + c;
      float v[16];
      if (a.vec) {
        mx_load8<OutT, true>(sp, left, v);
        mx_load8<OutT, true>(sp + 8, left - 8, v + 8);
      } else {
        mx_load8<OutT, false>(sp, left, v);
        mx_load8<OutT, false>(sp + 8, left - 8, v + 8);
      }
      const uint32_t sc = mx_scale16<CLT_MXFP4>(v);
      const uint2 lo = mx_encode8<CLT_MXFP4>(*reinterpret_cast<float (*)[8]>(v)), hi = mx_encode8<CLT_MXFP4>(*reinterpret_cast<float (*)[8]>(v + 8));
      *reinterpret_cast<uint2 *>(few_x + (r * pitch + (h >> 1)) * 16 + (h & 1) * 8) = make_uint2(lo.x, hi.x);
      if ((h & 1) == 0) few_s[r * P + (h >> 1)] = (uint8_t)sc;
    }
  }
  if constexpr (SRC == FEW_CODES) {
    for (int t = threadIdx.x; t < 16 * MT * P; t += 256) {
      const int r = t / P, b = t - r * P, m = m0 + r;
      const bool in = m < a.M && b < a.blocks;
      const int64_t at = (layer * a.M + (in ? m : 0)) * a.blocks + (in ? b : 0);
      *reinterpret_cast<uint4 *>(few_x + (r * pitch + b) * 16) = in ? ((const uint4 *)a.x)[at] : make_uint4(0u, 0u, 0u, 0u);
      few_s[t] = in ? a.xs[at] : (uint8_t)0;
    }
  }
  __syncthreads();

  struct Ahead { uint4 c[FEW_STEPS][FEW_NF]; uint32_t s[FEW_STEPS][FEW_NF]; };
  const int units = (a.N + FEW_TN - 1) / FEW_TN, chunks = P / (4 * FEW_STEPS);
  auto fetch = [&](Ahead &f, int unit, int ch) {
#pragma unroll
    for (int j = 0; j < FEW_NF; ++j) {
      const int n = min(unit * FEW_TN + (wave * FEW_NF + j) * 16 + l15, a.N - 1);
      const int64_t row = (layer * a.N + n) * a.blocks;
#pragma unroll
      for (int t = 0; t < FEW_STEPS; ++t) {
        const int b = min((ch * FEW_STEPS + t) * 4 + lq, a.blocks - 1);     // behind the end x is zero
        f.c[t][j] = *reinterpret_cast<const uint4 *>(a.wc + (row + b) * 16);
        f.s[t][j] = a.ws[row + b];
      }
    }
  };
  mx_f32x4_t acc[MT][FEW_NF];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < FEW_NF; ++j) acc[i][j] = mx_f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  auto multiply = [&](const Ahead &f, int ch) {
#pragma unroll
    for (int t = 0; t < FEW_STEPS; ++t) {
      const int b = (ch * FEW_STEPS + t) * 4 + lq;
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        uint4 xv;
        uint32_t sv;
        if constexpr (SRC == FEW_WIDE) {
          const bool in = b < a.blocks;
          const int64_t at = (layer * a.M + min(m0 + i * 16 + l15, a.M - 1)) * a.blocks + (in ? b : 0);
          xv = in ? ((const uint4 *)a.x)[at] : make_uint4(0u, 0u, 0u, 0u);
          sv = in ? a.xs[at] : 0u;
        } else {
          const int r = i * 16 + l15;
          xv = *reinterpret_cast<const uint4 *>(few_x + (r * pitch + b) * 16);
          sv = few_s[r * P + b];
        }
#pragma unroll
        for (int j = 0; j < FEW_NF; ++j) mx_mma(acc[i][j], f.c[t][j], f.s[t][j], xv, sv);
      }
    }
  };
  // a lane holds four neighbouring features of token lane % 16
  auto give = [&](int unit) {
#pragma unroll
    for (int j = 0; j < FEW_NF; ++j) {
      const int n = unit * FEW_TN + (wave * FEW_NF + j) * 16 + lq * 4;
      float bv[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) bv[q] = bias && n < a.N ? Elem<OutT>::to_f32(bias[layer * a.bs + min(n + q, a.N - 1)]) : 0.0f;
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const int m = m0 + i * 16 + l15;
        OutT *op = pre + layer * a.ps + m * a.pre_row + n;
        const float y[4] = {acc[i][j][0] + bv[0], acc[i][j][1] + bv[1], acc[i][j][2] + bv[2], acc[i][j][3] + bv[3]};
        acc[i][j] = mx_f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
        if (m >= a.M) continue;
        if (n + 4 <= a.N) {
          if constexpr (sizeof(OutT) == 4) __builtin_memcpy(op, y, 16);
          else {
            const uint32_t w[2] = {mx_pack<OutT>(y[0], y[1]), mx_pack<OutT>(y[2], y[3])};
            __builtin_memcpy(op, w, 8);
          }
        } else {
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (n + q < a.N) op[q] = Elem<OutT>::from_f32(y[q]);
        }
      }
    }
  };
  Ahead f0, f1;
  int unit = blockIdx.x, ch = 0;                        // the grid has no more workgroups per layer than units
  fetch(f0, unit, 0);
  auto turn = [&](Ahead &now, Ahead &then) {
    const bool end = ch + 1 == chunks;
    const int nunit = end ? unit + (int)gridDim.x : unit, nch = end ? 0 : ch + 1;
    if (nunit < units) fetch(then, nunit, nch);
    multiply(now, ch);
    if (end) give(unit);
    unit = nunit;
    ch = nch;
    return unit < units;
  };
  while (turn(f0, f1) && turn(f1, f0)) {}
}

// ---- the projection of a batch ------------------------------------------------------------------------------------
// Tiles of BM tokens x 256 features, one persistent workgroup of 8 wavefronts (4 along the tokens, 2 along the features) per CU.
// A stage is 256 elements of K: 128 bytes of codes per row - whole cache lines - brought straight into LDS, chunk c of row r at
// chunk position c ^ ((r >> 1) & 7): a fragment read's lanes are served in sixteens that take half their rows from one quarter of
// the wavefront and half from the next, and these places lie in all banks for the blocks lq and lq + 4 that a lane multiplies (lq =
// lane / 16; 2 lq and 2 lq + 1 met in pairs, which cost half of LDS's cycles).  Scales come as the lanes take them
// (mx_scale_place): one word holds those of two row groups and both blocks.
//
// A stage is four quarters of 4 MG products: all tokens of the wavefront x 32 of its features.  The x fragments stay in
// registers for the stage, each being replaced by the next stage's behind its last use; the W fragments of the next quarter are
// read under this one's products.  Two barriers: behind quarter 0 x and the first half of W have been read by everybody, so those
// loads of the stage after next (and its scales and biases, which have three places) are asked for; behind quarter 2 the rest.  A
// load has a stage and a half to arrive.
//
// The stages of all of a workgroup's tiles form one sequence, and so do the ends of the tiles: a quarter's accumulators are
// final behind the last stage's quarter and taken anew in the next tile's first one, which begins from the bias, and in between they
// go out, piece by piece among the products of the last three quarters and the first ones of the next tile.  A piece is 16 tokens x
// 128 bytes; it passes through LDS, so that a store is 16 bytes per lane and whole lines.  Stores are buffer stores, whose bounds drop
// the rows behind the last token: no branch parts the stream of products.  Loads and stores share a counter that runs in order,
// so the waits for loads allow for the stores sent behind them.
//
// Measured on 12 x 4096 x 768 x 24576, bf16 out (2.42 GB: 405 - 450 us for a kernel that does nothing but store these tiles):
// 590 - 600 us over the same buffers once the power limit has settled (710 in the first 20 passes), without loads 531, without stores
// 472, without both 406 (of which the products alone would be 281 at the 6.6 PFLOP/s that the power limit leaves them on random
// operands).  On 16 x 8192 x 2048 x 16384: 2140 - 2220 us (4000 TFLOP/s); 4 products of 8192^3: 960 us (4580).  Beside the stores it
// is bound by the LDS and by how its reads and the products follow each other: per 128 of K its wavefronts read 96 KB from it and
// 32 KB are put in, 1024 of its cycles at 128 bytes each, as many as the products themselves take at their full rate, and two
// wavefronts per SIMD with two barriers a stage do not hide all of one behind the other.  On operands that are all zeros, where
// power is no limit, the second takes 1818 us, of which products alone would take 1011 at the 8.7 PFLOP/s that a loop of them reaches
// on constants: some 800 us are the schedule's, 300 - 400 the power limit's.  (The first on zeros: 496 us; 4 products of
// 8192 x 4096 x 8192: 428 us instead of 546.)
// What did not help: groups of 4, 16 or 32 feature tiles in the order of the tiles (3 - 5 us slower); wavefronts' priorities
// (nothing); four wavefronts of 128 x 128 with the accumulators in the AGPRs (642 -> 701 us; nobody fills the waits).
constexpr int TW = 8;                         // wavefronts
constexpr int TROW = 128;                     // bytes of codes per row and stage
// Of a buffer store, taken where the rows of the result begin with a cache line (LINES): its parts are whole lines, and past the caches
// they go out faster (12 x 4096 x 768 x 24576: 742 -> 625 us).  Elsewhere the L2 has to put lines together (6 x 301 x 640 x 10006,
// float32: 31 us, and 69 past the caches).
constexpr int NONTEMPORAL = 2;
constexpr int PARK = 2048;                    // bytes of a wavefront's piece of the output tile on its way out

// vmcnt(n), nothing asked of the other counters
constexpr int wait_vm(int n) { return (n & 15) | ((n >> 4) << 14) | 0x0F70; }

__device__ __forceinline__ uint32_t mx_lds(const void *p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void *)p;
}
// 16 bytes per lane from base + off straight into LDS, lane i at at + 16 i.  Not counted by the compiler: the waits are written
// out.
__device__ __forceinline__ void mx_fill16(const void *base, uint32_t off, uint32_t at) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "{m0}"(at) : "memory");
}
// The same by the lanes of `mask` alone (they lie as before).
__device__ __forceinline__ void mx_fill16_low(const void *base, uint32_t off, uint32_t at, uint64_t mask) {
  uint64_t all;
  asm volatile("s_mov_b64 %0, exec\n\ts_mov_b64 exec, %4\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b64 exec, %0"
               : "=&s"(all) : "v"(off), "s"(base), "{m0}"(at), "s"(mask) : "memory");
}

// t / d for t < 2^31 by one product: m = floor(2^(31 + s) / d) + 1 with 2^(s - 1) < d <= 2^s.
struct MxDiv { uint32_t m; int s; };
static inline MxDiv mx_div(uint32_t d) {
  int s = 0;
  while (((uint64_t)1 << s) < d) ++s;
  return {s == 0 ? 0u : (uint32_t)(((uint64_t)1 << (31 + s)) / d + 1), s};
}
__device__ __forceinline__ int mx_over(int t, const MxDiv &v) { return v.s == 0 ? t : (int)(__umulhi((uint32_t)t, v.m) >> (v.s - 1)); }

struct TileArgs {
  const uint8_t *xc, *wc;                     // x rows hold whole stages (zeros behind the end)
  const uint8_t *xs, *ws;                     // [L][tiles][stages][8 rows of a tile], as the lanes take them (mx_scale_place)
  const float *bias;                          // [L][tiles_n][256], as the tiles take them
  int M, xrows, N, tiles_m, tiles_n, total, per_xcd;   // xrows: rows of x per layer that may be read, whole tiles
  int stages, xpitch, wpitch;                 // bytes of a row of codes
  int64_t ps, pre_row;
  MxDiv per_layer, per_group, last_group, per_stages;   // by tiles of a layer, of 8 feature tiles, by feature tiles of the last group, by stages
};

template <typename OutT, int MG, bool LINES>
__global__ __launch_bounds__(TW * 64) __attribute__((amdgpu_waves_per_eu(2, 2))) void k_mx_project_tiles(
    TileArgs a, OutT *__restrict__ pre) {
  constexpr int BM = 64 * MG;                              // tokens of a tile; a wavefront takes 16 MG x 128
  constexpr int FIRST = MG + 2 + 1 + 1, REST = 2;          // loads of a stage per wavefront: x, first half of W, scales, bias; rest of W
  constexpr int LOADS = FIRST + REST;
  constexpr int STAGE = (BM + TN) * TROW, SST = (BM + TN) * TBLOCKS + TN * 4;   // codes; scales and biases
  constexpr int G = 2 * MG;                                // pairs of products per quarter
  constexpr int HF = 128 / (int)sizeof(OutT);              // features of a piece
  constexpr int JH = HF / 16;                              // and in groups of 16
  constexpr int PIECES = MG * (128 / HF);                  // of a wavefront's tile
  constexpr int PQ = PIECES / 4;                           // that go out in each of four quarters,
  constexpr int LQ0 = HF / 32;                             // of which the first is this one of a tile's last stage (its features are final)
  constexpr int EQ = 2 * PQ;                               // stores in such a quarter
  static_assert(BM + TN == TW * 64 && LOADS + 6 * EQ < 64, "a wavefront brings the scales of 64 rows; the wait counter holds 63");
  __shared__ __attribute__((aligned(16))) unsigned char ring[2 * STAGE];
  __shared__ __attribute__((aligned(16))) unsigned char sring[3 * SST];
  __shared__ __attribute__((aligned(16))) unsigned char parked[TW * PARK];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave & 3, wn = wave >> 2, l15 = lane & 15, lq = lane >> 4;
  const uint32_t ring0 = mx_lds(ring), sring0 = mx_lds(sring);

  // Block b runs on XCD b % 8 and takes every (gridDim / 8)-th of that XCD's share of the tiles, a run of them in an order
  // that goes through 8 feature tiles for each token tile: the W tiles stay in the XCD's L2 while the tokens pass.
  // The last feature tile is moved back inside the matrix; what it shares with its neighbour is the same in both.
  // K is walked from a stage of the tile's own, so that the CUs that share x or W ask for different lines at any one time.  The order of
  // a result's sum so depends on its tile: the last bit of a token's float32 results on where in the batch the token lies.
  struct At { int layer, tm, m0, n0, tn, rot; };
  auto locate = [&](int t) {
    At at;
    at.layer = mx_over(t, a.per_layer);
    t -= at.layer * a.tiles_m * a.tiles_n;
    const int g = mx_over(t, a.per_group), r = t - g * 8 * a.tiles_m;
    const int cnt = min(8, a.tiles_n - g * 8);
    at.tm = cnt == 8 ? r >> 3 : mx_over(r, a.last_group);
    at.tn = g * 8 + r - at.tm * cnt;
    at.m0 = at.tm * BM;
    at.n0 = min(at.tn * TN, a.N - TN);
    const int rot = 3 * at.tm + min(at.tn, a.tiles_n - 2);     // the last tile and its neighbour share features: the same order
    at.rot = max(rot, 0);
    return at;
  };
  const int step = (int)gridDim.x >> 3;
  const int last_tile = min((((int)blockIdx.x & 7) + 1) * a.per_xcd, a.total);
  int tile = ((int)blockIdx.x & 7) * a.per_xcd + ((int)blockIdx.x >> 3);
  if (tile >= last_tile) return;

  // ---- the loader: where its next stage comes from.  A load of codes brings 8 rows, lane l row l / 8 at chunk position l % 8.
  int in_tile = tile, in_left = a.stages, in_stage = 0;
  uint32_t in_buf = 0, in_sbuf = 0;
  const uint8_t *in_x, *in_w, *in_s;
  const float *in_b;
  const uint32_t chunkE = (uint32_t)((lane & 7) ^ (lane >> 4)) * 16u;      // groups of 8 rows that begin at 0 mod 16; at 8: ^ 64
  // x: rows 8 MG wave + 8 i.  W: row groups in the order of the quarters, first half 0 .. 63 and 128 .. 191, rest behind them
  auto w_row = [&](int i) { const int u = (i & 1) * 8 + wave; return (i >> 1) * 64 + (u >> 3) * 128 + (u & 7) * 8; };
  const uint32_t xo = (uint32_t)(lane >> 3) * (uint32_t)a.xpitch + chunkE, wo = (uint32_t)(lane >> 3) * (uint32_t)a.wpitch;
  At ahead;                                                    // where the loader is
  auto aim = [&]() {
    ahead = locate(in_tile);
    const At &at = ahead;
    in_stage = at.rot - mx_over(at.rot, a.per_stages) * a.stages;
    in_x = a.xc + ((int64_t)at.layer * a.xrows + at.m0) * a.xpitch;
    in_w = a.wc + ((int64_t)at.layer * a.N + at.n0) * a.wpitch;
    // eight wavefronts, 64 rows of scales each: those of x, then those of W
    in_s = wave * 64 < BM ? a.xs + ((int64_t)at.layer * a.tiles_m + at.tm) * a.stages * (BM * TBLOCKS) + wave * 64 * TBLOCKS
                          : a.ws + ((int64_t)at.layer * a.tiles_n + at.tn) * a.stages * (TN * TBLOCKS) + (wave * 64 - BM) * TBLOCKS;
    in_b = a.bias + ((int64_t)at.layer * a.tiles_n + at.tn) * TN;
  };
  // W and its scales are not filled up: behind the end the last block is repeated, and x is zero there
  auto load_w = [&](int i) {
    const int r = w_row(i);
    mx_fill16(in_w + (uint32_t)r * (uint32_t)a.wpitch, wo + min((uint32_t)in_stage * TROW + (chunkE ^ ((r & 8) ? 64u : 0u)), (uint32_t)a.wpitch - 16u),
              ring0 + in_buf * STAGE + (uint32_t)(BM + r) * TROW);
  };
  auto load_first = [&](int i) {
    if (i < MG) {
      const int r = (wave * MG + i) * 8;
      mx_fill16(in_x + (uint32_t)r * (uint32_t)a.xpitch + (int64_t)in_stage * TROW, xo ^ ((r & 8) ? 64u : 0u), ring0 + in_buf * STAGE + (uint32_t)r * TROW);
    } else if (i < MG + 2) load_w(i - MG);
    else if (i == MG + 2)
      mx_fill16_low(in_s + (int64_t)in_stage * (wave * 64 < BM ? BM * TBLOCKS : TN * TBLOCKS), (uint32_t)lane * 16u,
                    sring0 + in_sbuf * SST + (uint32_t)(wave * 64 * TBLOCKS), 0xFFFFFFFFull);
    else
      mx_fill16_low(in_b + wave * 32, (uint32_t)lane * 16u, sring0 + in_sbuf * SST + (BM + TN) * TBLOCKS + (uint32_t)wave * 128u, 0xFFull);
  };
  auto load_rest = [&](int i) { load_w(2 + i); };
  auto load_next = [&]() {
    in_buf ^= 1u;
    in_sbuf = in_sbuf == 2 ? 0 : in_sbuf + 1;
    if (++in_stage == a.stages) in_stage = 0;
    --in_left;
  };
  auto load_from = [&]() {                                     // in front of a stage's first load
    if (in_left != 0) return;
    in_left = a.stages;
    if (in_tile + step < last_tile) in_tile += step;           // behind the last tile: once more, for nobody
    aim();
  };

  // ---- fragments: row l15 of each group of 16, its blocks lq and lq + 4
  const uint32_t xat = (uint32_t)(wm * 16 * MG + l15) * TROW, wat = (uint32_t)(BM + wn * 128 + l15) * TROW;
  const uint32_t xsat = (uint32_t)(wm * (MG / 2) * 64 + lane) * 4, wsat = (uint32_t)(BM * TBLOCKS + (wn * 4 * 64 + lane) * 4);
  const uint32_t koff[2] = {(uint32_t)(lq ^ ((l15 >> 1) & 7)) * 16u, (uint32_t)((lq + 4) ^ ((l15 >> 1) & 7)) * 16u};
  uint4 fx[MG][2], fw[2][2][2];
  uint32_t sx[MG / 2], sw[2];
  auto read_x = [&](uint32_t buf, int i, int ks) { fx[i][ks] = *reinterpret_cast<const uint4 *>(ring + buf * STAGE + xat + i * 16 * TROW + koff[ks]); };
  auto read_xs = [&](uint32_t sbuf, int i) { sx[i] = *reinterpret_cast<const uint32_t *>(sring + sbuf * SST + xsat + i * 256); };
  auto read_w = [&](uint32_t buf, int q, int j, int ks) {
    fw[q & 1][j][ks] = *reinterpret_cast<const uint4 *>(ring + buf * STAGE + wat + (q * 2 + j) * 16 * TROW + koff[ks]);
  };
  auto read_ws = [&](uint32_t sbuf, int q) { sw[q & 1] = *reinterpret_cast<const uint32_t *>(sring + sbuf * SST + wsat + q * 256); };
  auto meet = [&]() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
  };

  mx_f32x4_t acc[MG][8], bv[2];
  auto read_bias = [&](uint32_t sbuf, int q) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
      bv[j] = *reinterpret_cast<const mx_f32x4_t *>(sring + sbuf * SST + (BM + TN) * TBLOCKS + (wn * 128 + (q * 2 + j) * 16 + lq * 4) * 4);
  };

  // ---- the way out.  A lane holds four neighbouring features of token l15 of each group of 16 tokens.
  unsigned char *park = parked + wave * PARK;
  const uint32_t out_pitch = (uint32_t)a.pre_row * (uint32_t)sizeof(OutT);
  // Addresses are rebuilt from the lane number by every stage that needs them: as invariants they would live across all others.
  int la_out = lane;
  __amdgpu_buffer_rsrc_t out = __builtin_amdgcn_make_buffer_rsrc(pre, 0, 0, 0x00020000);      // no tile yet: nothing is in bounds
  auto aim_out = [&](const At &at) {
    const int rows = min(BM, a.M - at.m0);
    out = __builtin_amdgcn_make_buffer_rsrc(pre + (int64_t)at.layer * a.ps + (int64_t)at.m0 * a.pre_row + at.n0, 0,
                                            (int)((uint32_t)(rows - 1) * out_pitch + TN * (uint32_t)sizeof(OutT)), 0x00020000);
  };
  auto put = [&](int n) {
    const int i = n % MG, h = n / MG, l15 = la_out & 15, lq = la_out >> 4;
#pragma unroll
    for (int jj = 0; jj < JH; ++jj) {
      const mx_f32x4_t y = acc[i][h * JH + jj];
      if constexpr (sizeof(OutT) == 4) {
        *reinterpret_cast<mx_f32x4_t *>(park + l15 * 128 + ((jj * 4 + lq) ^ (l15 >> 1)) * 16) = y;
      } else {
        const int slot = (jj * 2 + (lq >> 1)) ^ (l15 >> 1);
        *reinterpret_cast<uint2 *>(park + l15 * 128 + slot * 16 + (lq & 1) * 8) = make_uint2(mx_pack<OutT>(y[0], y[1]), mx_pack<OutT>(y[2], y[3]));
      }
    }
  };
  typedef __attribute__((ext_vector_type(4))) unsigned int u32x4_t;
  u32x4_t v;
  auto take = [&](int u) { v = *reinterpret_cast<const u32x4_t *>(park + (u * 8 + (la_out >> 3)) * 128 + (((la_out & 7) ^ (u * 4 + (la_out >> 4))) * 16)); };
  auto send = [&](int n, int u) {
    const int i = n % MG, h = n / MG;
    const uint32_t out_at = (uint32_t)(wm * 16 * MG + (la_out >> 3)) * out_pitch + (uint32_t)(wn * 128 * (int)sizeof(OutT) + (la_out & 7) * 16);
    __builtin_amdgcn_raw_buffer_store_b128(v, out, (int)(out_at + (uint32_t)(i * 16 + u * 8) * out_pitch + (uint32_t)h * 128u), 0, LINES ? NONTEMPORAL : 0);
  };

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
  read_ws(0, 0);
#pragma unroll
  for (int r = 0; r < 4; ++r) read_w(0, 0, r & 1, r >> 1);
  read_bias(0, 0);
#pragma unroll
  for (int i = 0; i < MG; ++i) {
    read_x(0, i, 0);
    read_x(0, i, 1);
    if (i % 2 == 0) read_xs(0, i / 2);
  }

  // One stage: the first of a tile, the last, both or neither.  At the barriers, what the quarters up to the next barrier read has
  // landed: all but the last LOADS loads and the stores sent behind what is waited for - in this stage, as its kind says, and
  // in those before: `late` says that there was a tile before and that this is its first stage, or the second one.  And this
  // wavefront's reads are over.  (The waits' branch is inside the statement: behind a
  // block's end the compiler moves products.)
  auto stage = [&](auto first, auto last, int late, const At &at) {
    constexpr bool F = decltype(first)::value, E = decltype(last)::value;
    constexpr int A0 = LOADS + (F ? EQ : 0), A1 = A0 + (F ? (4 - LQ0) * EQ : (LQ0 + 1) * EQ);
    constexpr int B0 = LOADS + (F ? LQ0 * EQ : 0) + (E ? (3 - LQ0) * EQ : 0), B1 = B0 + (F ? 2 * EQ : 0);
    load_from();
    if constexpr (F || E) {
      la_out = lane;
      asm volatile("" : "+v"(la_out));
    }
    const uint32_t next = buf ^ 1u, snext = sbuf == 2 ? 0 : sbuf + 1;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (q == 1)
        asm volatile("s_cmp_lg_u32 %0, 0\n\ts_cbranch_scc1 .Lmxl%=\n\ts_waitcnt vmcnt(%1) lgkmcnt(0)\n\ts_branch .Lmxd%=\n"
                     ".Lmxl%=:\n\ts_waitcnt vmcnt(%2) lgkmcnt(0)\n.Lmxd%=:" ::"s"(late), "n"(A0), "n"(A1) : "scc", "memory");
      if (q == 3)
        asm volatile("s_cmp_lg_u32 %0, 0\n\ts_cbranch_scc1 .Lmxl%=\n\ts_waitcnt vmcnt(%1) lgkmcnt(0)\n\ts_branch .Lmxd%=\n"
                     ".Lmxl%=:\n\ts_waitcnt vmcnt(%2) lgkmcnt(0)\n.Lmxd%=:" ::"s"(late), "n"(B0), "n"(B1) : "scc", "memory");
      if (q == 1 || q == 3) meet();
      // the pieces of this quarter: of the tile before in a first stage, of this one in a last
      const bool out_f = F && q < LQ0, out_e = E && q >= LQ0;
      if (E && q == LQ0) aim_out(at);
      const int n0 = out_e ? (q - LQ0) * PQ : (4 - LQ0 + q) * PQ;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const int ks = g / MG, i = g % MG;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          mx_f32x4_t &d = acc[i][q * 2 + j];
          d = mx_mma2(F && ks == 0 ? bv[j] : d, fw[q & 1][j][ks], sw[q & 1], j * 2 + ks, fx[i][ks], sx[i / 2], (i & 1) * 2 + ks);
        }
#pragma unroll
        for (int r = g * 4 / G; r < (g + 1) * 4 / G; ++r) {
          if (q < 3) read_w(buf, q + 1, r & 1, r >> 1);
          else read_w(next, 0, r & 1, r >> 1);
        }
        if (g == 0) { if (q < 3) read_ws(sbuf, q + 1); else read_ws(snext, 0); }
        if (g == MG && ((F && q < 3) || (E && q == 3))) read_bias(q < 3 ? sbuf : snext, (q + 1) & 3);
        if (q == 3) {
          read_x(next, i, ks);
          if (ks == 1 && i % 2 == 1) read_xs(snext, i / 2);
        }
        // the loads of a quarter lie in front of the stores that the waits count as sent behind them
        if (q == 1) {
#pragma unroll
          for (int r = g * FIRST / G; r < (g + 1) * FIRST / G; ++r) load_first(r);
        }
        if (q == 3 && g < REST) load_rest(g);
        if (out_f || out_e) {
          constexpr int GP = G / PQ;                           // places of a piece
          const int e = g / GP, place = g % GP;
          if (GP >= 4) {
            if (place == 0) put(n0 + e);
            if (place == 1) take(0);
            if (place == 2) { send(n0 + e, 0); take(1); }
            if (place == 3) send(n0 + e, 1);
          } else {
            if (place == 0) { if (e > 0) send(n0 + e - 1, 1); put(n0 + e); take(0); }
            if (place == 1) { send(n0 + e, 0); take(1); if (e == PQ - 1) send(n0 + e, 1); }
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    // the products stay in this block: the compiler would move some of them behind its end, next to their next use
#pragma unroll
    for (int i = 0; i < MG; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) asm volatile("" : "+v"(acc[i][j]));
    load_next();
    buf = next;
    sbuf = snext;
  };

  const std::true_type yes;
  const std::false_type no;
  int before = 0;
  At at = ahead;                                               // there are at least two stages: the loader is still in the first tile
  for (;;) {
    stage(yes, no, before, at);
#pragma clang loop unroll(disable)
    for (int k = 1; k < a.stages - 1; ++k) stage(no, no, before & (k == 1), at);
    stage(no, yes, before & (a.stages == 2), at);
    at = ahead;                                                // by now in the next one
    before = 1;
    tile += step;
    if (tile >= last_tile) break;
  }
#pragma unroll
  for (int n = PIECES - LQ0 * PQ; n < PIECES; ++n) {
    put(n);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      take(u);
      send(n, u);
    }
  }
  __builtin_amdgcn_s_waitcnt(0);   // no load into LDS may be under way when the workgroup ends
}

// What a tile takes beside its codes: the scales of its 256 rows in the lanes' order, zeros where there is no block or no row, and the
// biases in float32.  A workgroup takes one stage of one tile: a thread fetches the eight scales of a row and puts out two words.
struct MxSide {
  const uint8_t *scales;
  uint8_t *out;
  const void *bias;
  float *bias_out;
  int rows, blocks, stages;
  int64_t bias_stride;
};
template <typename T, int GROUPS> __device__ __forceinline__ void mx_tile_side(const MxSide &a, int x, int tile0, int64_t l) {
  __shared__ uint2 held[256];
  const int stage = x % a.stages, t = x / a.stages;
  const int64_t tile = l * tile0 + t;
  // feature tiles: the last one is moved back inside the matrix
  const int r0 = GROUPS == 8 ? min(t * 256, a.rows - 256) : t * 256, r = r0 + (int)threadIdx.x, b0 = stage * TBLOCKS;
  uint2 v = make_uint2(0u, 0u);
  if (r < a.rows) {
    const uint8_t *p = a.scales + (l * a.rows + r) * a.blocks + b0;
    if (b0 + TBLOCKS <= a.blocks) __builtin_memcpy(&v, p, 8);
    else {
      for (int b = 0; b0 + b < a.blocks; ++b) (b < 4 ? v.x : v.y) |= (uint32_t)p[b] << (b % 4 * 8);
    }
  }
  held[threadIdx.x] = v;
  __syncthreads();
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int at = half * 256 + threadIdx.x, lane = at % 64, i0 = at / 64 % (GROUPS / 2) * 2, w = at / (32 * GROUPS), shift = (lane >> 4) * 8;
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint2 h = held[(w * GROUPS + i0 + i) * 16 + (lane & 15)];
      word |= ((h.x >> shift & 255u) | (h.y >> shift & 255u) << 8) << (i * 16);
    }
    *reinterpret_cast<uint32_t *>(a.out + (tile * a.stages + stage) * 2048 + at * 4) = word;
  }
  if (a.bias_out && stage == 0) a.bias_out[tile * 256 + threadIdx.x] = a.bias ? Elem<T>::to_f32(((const T *)a.bias)[l * a.bias_stride + r]) : 0.0f;
}
template <typename T, int GROUPS> __global__ __launch_bounds__(256) void k_mx_tile_side(MxSide a) {
  mx_tile_side<T, GROUPS>(a, blockIdx.x, gridDim.x / a.stages, blockIdx.y);
}
// The same for the weights beside the quantisation of x, neither of which waits for the other: 7 us for 77 tokens of 12 x 24576 x 768,
// 148 us for 8192 of 16 x 16384 x 2048 (0.72 GB); as two launches, a thread going through a tile's stages, 5.0 + 7.6 and 136 + 38 us.
template <typename T, bool VEC> __global__ __launch_bounds__(256) void k_mx_tile_inputs(MxSide a, int tiles, MxWrite x) {
  const int side = tiles * a.stages;
  if ((int)blockIdx.x < side) mx_tile_side<T, 8>(a, blockIdx.x, tiles, blockIdx.y);
  else mx_write_piece<T, CLT_MXFP4, VEC, true>(x, blockIdx.x - side);
}

// Rows of codes at another pitch, `to` blocks of 16 bytes instead of `from`, filled up with zeros; the rows of a layer `room` rows
// apart instead of `rows`.
__global__ __launch_bounds__(256) void k_mx_widen(const uint4 *__restrict__ src, uint4 *__restrict__ dst, int64_t rows, int64_t room, int from, int to) {
  const int64_t l = blockIdx.y, n = rows * to;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / to;
    const int b = (int)(i - r * to);
    dst[l * room * to + i] = b < from ? src[(l * rows + r) * from + b] : make_uint4(0u, 0u, 0u, 0u);
  }
}

int launch_mx_widen(const void *src, void *dst, int64_t L, int64_t rows, int64_t room, int64_t from, int64_t to, hipStream_t s) {
  const int64_t nb = clt_ceil_div(rows * to, 256);
  k_mx_widen<<<dim3((unsigned)(nb < 65536 ? nb : 65536), (unsigned)L), 256, 0, s>>>((const uint4 *)src, (uint4 *)dst, rows, room, (int)from, (int)to);
  return clt_check_launch();
}

bool mx_format(int fmt) { return fmt == CLT_MXFP4 || fmt == CLT_MXFP8 || fmt == CLT_MXINT8; }
// Rows a thread gives out, where that leaves threads enough for the chip: four wavefronts per SIMD.
constexpr int MX_U = 2;
constexpr int64_t MX_MANY = 4 * 1024 * 64;
uint32_t mx_magic(uint32_t pieces) { return (uint32_t)((0x100000000ull + pieces - 1) / pieces); }

template <typename T>
bool mx_write_vec(const void *src0, const void *src1, int64_t layer_stride, int64_t row_stride, int64_t d) {
  return d % 8 == 0 && clt_aligned16(src0) && clt_aligned16(src1) && row_stride * (int64_t)sizeof(T) % 16 == 0 && layer_stride * (int64_t)sizeof(T) % 16 == 0;
}

template <typename T, int FMT>
int launch_mx_write(const void *src0, const void *src1, int64_t layer_stride, int64_t row_stride, int64_t L, int kinds, int64_t n, int64_t d,
                    uint32_t blocks, const MxRows &rows, void *codes, uint8_t *scales, hipStream_t s) {
  const int64_t groups = clt_ceil_div(n * (int64_t)(blocks * 2), MX_THREADS);
  if (groups > MX_MAX_GROUPS) return CLT_ERR_RANGE;
  const dim3 grid((unsigned)groups, (unsigned)(L * kinds));
  const MxWrite a{src0, src1, layer_stride, row_stride, n, d, kinds, blocks, mx_magic(blocks * 2), rows, (uint8_t *)codes, scales};
  if (mx_write_vec<T>(src0, src1, layer_stride, row_stride, d)) k_mx_write<T, FMT, true><<<grid, MX_THREADS, 0, s>>>(a);
  else k_mx_write<T, FMT, false><<<grid, MX_THREADS, 0, s>>>(a);
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
  constexpr int E = sizeof(OutT) == 4 ? 4 : 8;
  const int64_t row_bytes = out_row_stride * (int64_t)sizeof(OutT), layer_bytes = out_layer_stride * (int64_t)sizeof(OutT);
  const bool vec = d % E == 0 && clt_aligned16(out0) && (kinds == 1 || clt_aligned16(out1)) && row_bytes % 16 == 0 && layer_bytes % 16 == 0;
  const bool lines = d * (int64_t)sizeof(OutT) % 128 == 0 && (((uintptr_t)out0 | (uintptr_t)out1) & 127u) == 0 && row_bytes % 128 == 0 && layer_bytes % 128 == 0;
  const uint32_t blocks = (uint32_t)clt_ceil_div(d, 32), pieces = (uint32_t)(vec ? d / E : clt_ceil_div(d, 8));
  const bool many = vec && L * kinds * clt_ceil_div(n, MX_U) * pieces >= MX_MANY;
  const int64_t apart = many ? clt_ceil_div(n, MX_U) : n, groups = clt_ceil_div(apart * (int64_t)pieces, MX_THREADS);
  if (groups > MX_MAX_GROUPS) return CLT_ERR_RANGE;
  const dim3 grid((unsigned)groups, (unsigned)(L * kinds));
#define CLT_MXR(VEC, U, LINES)                                                                                                             \
  k_mx_read<OutT, FMT, VEC, U, LINES><<<grid, MX_THREADS, 0, s>>>((const uint8_t *)codes, scales, rows, n, apart, d, blocks, pieces,           \
                                                                  mx_magic(pieces), kinds, nm, (OutT *)out0, (OutT *)out1, out_layer_stride, \
                                                                  out_row_stride)
  if (many && lines) CLT_MXR(true, MX_U, true);
  else if (many) CLT_MXR(true, MX_U, false);
  else if (vec) CLT_MXR(true, 1, false);
  else CLT_MXR(false, 1, false);
#undef CLT_MXR
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

// How a shape is computed.  Up to 64 tokens, as long as their rows leave room in LDS for two workgroups per CU, by the kernel for few:
// W is read once then.  Beyond by tiles, where there are whole feature tiles and rows of the result lie at whole words (buffer
// stores); else by the kernel for few in groups of tokens.  12 layers, d 768, F 24576, bf16, kernel for few against tiles, us, x
// quantised in the call: 26 against 49 at 1 token, 31 / 48 at 17, 35 / 47 at 33, 41 / 47 at 64, 63 / 49 at 77, 75 / 50 at 128, 148 / 59
// at 256; 16 layers, d 2048, F 16384: 75 / 103 at 1, 81 / 103 at 17, 98 / 105 at 64.
// Results of 16 bits with an odd F have no whole words in their rows, and go
// through the weights once per 128 tokens: 12 layers, d 768, bf16, F 24575
// against 24576: 192 / 56 us at 256 tokens, 699 / 171 at 1024, 2127 / 627 at 4096.  Rows that LDS does not hold for even 16 tokens
// (d above about 9600) go by tiles from one token on: 4 layers, F 4096, one token: 41 us at d 9216 (1.97 TB/s of weights), 63 at 9728,
// 77 at 12288 (1.40), where 32 tokens take 78.
bool mx_tiles_fit(int64_t F, const void *pre, int64_t ps, int64_t pre_row, int64_t e) {
  return ((uintptr_t)pre & 3u) == 0 && ps * e % 4 == 0 && pre_row * e % 4 == 0 && F * e % 4 == 0 && pre_row * e <= (1 << 22);
}
// groups of 16 tokens that the kernel for few takes at a time; 0: not even one fits into LDS
int mx_few_groups(int64_t T, int64_t blocks) {
  int mt = T <= 16 ? 1 : T <= 32 ? 2 : T <= 64 ? 4 : 8;
  while (mt > 0 && (blocks > 65536 || few_lds((int)blocks, mt) > FEW_LDS)) mt >>= 1;
  return mt;
}
bool mx_use_tiles(int64_t T, int64_t F, int64_t blocks) {
  const int few = mx_few_groups(T, blocks);
  return F >= TN && T > 16 * (few < 4 ? few : 4);
}

constexpr int64_t MX_FEW_VALUES = 16384;   // elements of x that every workgroup quantises for itself

// What the projection keeps for itself: x in codes, in whole tiles of rows of whole stages, its scales and those of W in the lanes'
// order, the biases of the tiles.  For the other kernels: x in codes as they are.
struct MxPlan {
  int64_t blocks, padded;             // blocks of a row; of a row of x in whole stages, two at least
  int64_t xrows, tm, tn, stages;      // rows of x per layer; tiles
  bool tiles, own_x, values;
  int few;                            // groups of 16 tokens of the kernel for few
  size_t xc, xs, ws, bias, bytes;     // offsets in the workspace
};
MxPlan mx_plan(int64_t T, int64_t d, int64_t F, int64_t L, bool quantised, bool tiles) {
  MxPlan p{};
  p.blocks = clt_ceil_div(d, 32);
  p.tiles = tiles;
  p.padded = tiles ? clt_ceil_div(p.blocks, TBLOCKS) * TBLOCKS : p.blocks;
  if (tiles && p.padded < 2 * TBLOCKS) p.padded = 2 * TBLOCKS;
  p.stages = p.padded / TBLOCKS;
  p.tm = clt_ceil_div(T, MX_BM);
  p.tn = clt_ceil_div(F, TN);
  p.xrows = tiles ? p.tm * MX_BM : T;
  // few tokens are quantised on the way into LDS, where they fit and a workgroup has not long to go at them
  p.few = tiles ? 0 : mx_few_groups(T, p.blocks);
  p.values = !tiles && !quantised && p.few > 0 && 16 * p.few * p.blocks * 32 <= MX_FEW_VALUES;
  p.own_x = tiles ? !quantised || p.padded != p.blocks || p.xrows != T : !quantised && !p.values;
  auto up = [](size_t n) { return (n + 255) & ~(size_t)255; };
  p.xs = up(p.own_x ? (size_t)(L * p.xrows * p.padded * 16) : 0);
  p.ws = p.xs + up(tiles || p.own_x ? (size_t)(L * p.xrows * p.padded) : 0);
  p.bias = p.ws + (tiles ? (size_t)(L * p.tn * TN * p.padded) : 0);
  p.bytes = p.bias + (tiles ? (size_t)(L * p.tn * TN * 4) : 0);
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
int launch_mx_project(const MxPlan &p, const void *x, const void *xc, int64_t x_layer, bool vec, const uint8_t *xs, const uint8_t *wc, const uint8_t *wsc, const void *bias,
                      uint8_t *ws, void *pre, int64_t T, int64_t d, int64_t F, int64_t L, int64_t bs, int64_t ps, int64_t pre_row, hipStream_t s) {
  if (p.tiles) {
    const int64_t total = p.tm * p.tn * L;
    if (total > 1073741824LL || p.tn * p.stages + (x ? clt_ceil_div(T * p.padded * 2, MX_THREADS) : 0) > MX_MAX_GROUPS) return CLT_ERR_RANGE;
    const int grid = mx_grid(total);
    if (grid <= 0) return CLT_ERR_LAUNCH;
    const MxSide side{wsc, ws + p.ws, bias, (float *)(ws + p.bias), (int)F, (int)p.blocks, (int)p.stages, bs};
    if (x) {                                               // values, to be quantised into the workspace
      const uint32_t pieces = (uint32_t)p.padded * 2;
      const int64_t groups = p.tn * p.stages + clt_ceil_div(T * pieces, MX_THREADS);
      const dim3 grid((unsigned)groups, (unsigned)L);
      const MxWrite w{x, nullptr, x_layer, d, T, d, 1, (uint32_t)p.padded, mx_magic(pieces), {nullptr, 0, 0, p.xrows, nullptr}, ws + p.xc, ws + p.xs};
      if (vec) k_mx_tile_inputs<OutT, true><<<grid, 256, 0, s>>>(side, (int)p.tn, w);
      else k_mx_tile_inputs<OutT, false><<<grid, 256, 0, s>>>(side, (int)p.tn, w);
    } else k_mx_tile_side<OutT, 8><<<dim3((unsigned)(p.tn * p.stages), (unsigned)L), 256, 0, s>>>(side);
    TileArgs a{(const uint8_t *)xc, wc, xs, ws + p.ws, (const float *)(ws + p.bias), (int)T, (int)p.xrows, (int)F, (int)p.tm, (int)p.tn, (int)total,
               (int)clt_ceil_div(total, 8), (int)p.stages, (int)p.padded * 16, (int)p.blocks * 16, ps, pre_row,
               mx_div((uint32_t)(p.tm * p.tn)), mx_div((uint32_t)(8 * p.tm)), mx_div((uint32_t)(p.tn % 8 ? p.tn % 8 : 8)), mx_div((uint32_t)p.stages)};
    const int64_t e = sizeof(OutT);
    if (((uintptr_t)pre & 127u) == 0 && pre_row * e % 128 == 0 && ps * e % 128 == 0)
      k_mx_project_tiles<OutT, MX_MG, true><<<grid, TW * 64, 0, s>>>(a, (OutT *)pre);
    else
      k_mx_project_tiles<OutT, MX_MG, false><<<grid, TW * 64, 0, s>>>(a, (OutT *)pre);
    return clt_check_launch();
  }
  const int mt = p.few > 0 ? p.few : 4, lds = p.few > 0 ? few_lds((int)p.blocks, mt) : 0;
  const int64_t units = clt_ceil_div(F, FEW_TN), gz = clt_ceil_div(T, 16 * mt);
  if (gz > 65535) return CLT_ERR_RANGE;
  // three workgroups per CU where they fit, so that the last ones are not long alone
  const int64_t room = clt_ceil_div(256 * (lds > 52 * 1024 ? 2 : 3), L * gz), gx = units < room ? units : room;
  const FewArgs a{xc, xs, wc, wsc, x_layer, bs, ps, pre_row, (int)T, (int)F, (int)d, (int)p.blocks, vec ? 1 : 0};
  const dim3 grid((unsigned)gx, (unsigned)L, (unsigned)gz);
#define CLT_FEW(MT, SRC)                                                                                                            \
  {                                                                                                                                \
    if (lds > 64 * 1024 && hipFuncSetAttribute((const void *)k_mx_project_few<OutT, MT, SRC>, hipFuncAttributeMaxDynamicSharedMemorySize, \
                                               lds) != hipSuccess)                                                                 \
      return CLT_ERR_LAUNCH;                                                                                                       \
    k_mx_project_few<OutT, MT, SRC><<<grid, 256, lds, s>>>(a, (const OutT *)bias, (OutT *)pre);                                     \
  }
  if (p.few == 0) CLT_FEW(4, FEW_WIDE)
  else if (p.values) {
    if (mt == 1) CLT_FEW(1, FEW_VALUES) else if (mt == 2) CLT_FEW(2, FEW_VALUES) else if (mt == 4) CLT_FEW(4, FEW_VALUES) else CLT_FEW(8, FEW_VALUES)
  } else {
    if (mt == 1) CLT_FEW(1, FEW_CODES) else if (mt == 2) CLT_FEW(2, FEW_CODES) else if (mt == 4) CLT_FEW(4, FEW_CODES) else CLT_FEW(8, FEW_CODES)
  }
#undef CLT_FEW
  return clt_check_launch();
}

// sizes that every entry point asks for
int mx_sizes(int64_t L, int64_t n, int64_t d, int64_t rows) {
  if (L <= 0 || n < 0 || d <= 0 || rows < 0) return CLT_ERR_ARG;
  if (L > 32767 || d > MX_MAX_WIDTH || n > 2147483647LL || rows > MX_MAX_ROWS) return CLT_ERR_RANGE;
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

extern "C" int clt_mx_refresh(const void *src, int64_t L, int64_t n, int64_t d, int64_t layer_stride, int dtype, void *codes, uint8_t *scales,
                              uint64_t *state, int32_t *changed, int store_only, void *stream) {
  if (!clt_model_dtype(dtype)) return CLT_ERR_DTYPE;
  if (const int rc = mx_sizes(L, n, d, n)) return rc;
  if (n == 0) return CLT_OK;
  if (!src || !codes || !scales || !state || !changed || layer_stride < 0) return CLT_ERR_ARG;
  if (!clt_aligned16(codes) || ((uintptr_t)state & 127u) != 0) return CLT_ERR_ALIGN;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == CLT_BF16) return launch_mx_refresh<bf16_t>(src, layer_stride, L, n, d, codes, scales, state, changed, store_only, s);
  if (dtype == CLT_F16) return launch_mx_refresh<f16_t>(src, layer_stride, L, n, d, codes, scales, state, changed, store_only, s);
  return launch_mx_refresh<float>(src, layer_stride, L, n, d, codes, scales, state, changed, store_only, s);
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
  if (row_index ? !owner : (first < 0 || n > rows || first > rows - n)) return CLT_ERR_ARG;
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
  if (T < 0 || out_row0 < 0 || n > T || out_row0 > T - n) return CLT_ERR_ARG;
  if (T > MX_MAX_ROWS) return CLT_ERR_RANGE;
  if (n == 0) return CLT_OK;
  if (!codes || !scales || !x_out || !tgt_out || rows == 0) return CLT_ERR_ARG;
  if (!row_index && (first < 0 || n > rows || first > rows - n)) return CLT_ERR_ARG;
  if (!clt_aligned16(codes)) return CLT_ERR_ALIGN;
  const MxRows r{row_index, index_bits == 64, first, rows, nullptr};
  const MxNorm nm{norm_mode, mean_in, std_in, mean_tg, std_tg, (float)scale};
  const int64_t e = clt_elem_bytes(out_dtype);
  return mx_read(out_dtype, fmt, codes, scales, r, L, 2, n, d, nm, (char *)x_out + out_row0 * d * e, (char *)tgt_out + out_row0 * d * e, T * d, d,
                 (hipStream_t)stream);
}

extern "C" size_t clt_mx_encode_workspace_bytes(int64_t T, int64_t d, int64_t F, int64_t L, int x_quantised) {
  if (T <= 0 || d <= 0 || F <= 0 || L <= 0 || d > MX_MAX_WIDTH) return 0;
  // enough for any address and pitch of the result
  const size_t small = mx_plan(T, d, F, L, x_quantised != 0, false).bytes;
  const size_t tiled = mx_use_tiles(T, F, clt_ceil_div(d, 32)) ? mx_plan(T, d, F, L, x_quantised != 0, true).bytes : 0;
  return tiled > small ? tiled : small;
}

extern "C" int clt_mx_encode(const void *x, const uint8_t *x_scales, const void *w_codes, const uint8_t *w_scales, const void *bias, void *pre,
                             int64_t T, int64_t d, int64_t F, int64_t L, int64_t x_layer_stride, int64_t b_layer_stride,
                             int64_t pre_layer_stride, int64_t pre_row_stride, int dtype, void *workspace, size_t workspace_bytes, void *stream) {
  if (!clt_model_dtype(dtype)) return CLT_ERR_DTYPE;
  if (T < 0 || d <= 0 || F <= 0 || L <= 0) return CLT_ERR_ARG;
  if (T == 0) return CLT_OK;
  if (!x || !w_codes || !w_scales || !pre || pre_row_stride < F || pre_layer_stride < 0 || (!x_scales && x_layer_stride < 0)) return CLT_ERR_ARG;
  if (d > MX_MAX_WIDTH || T > 16 * 65535 || F > (1 << 30) || L > 32767) return CLT_ERR_RANGE;
  if ((x_scales && !clt_aligned16(x)) || !clt_aligned16(w_codes)) return CLT_ERR_ALIGN;
  const int64_t e = clt_elem_bytes(dtype);
  const MxPlan p = mx_plan(T, d, F, L, x_scales != nullptr,
                           mx_use_tiles(T, F, clt_ceil_div(d, 32)) && mx_tiles_fit(F, pre, pre_layer_stride, pre_row_stride, e));
  const size_t need = clt_mx_encode_workspace_bytes(T, d, F, L, x_scales != nullptr);
  if (need > 0 && (!workspace || workspace_bytes < need)) return CLT_ERR_WORKSPACE;
  if (need > 0 && !clt_aligned16(workspace)) return CLT_ERR_ALIGN;
  hipStream_t s = (hipStream_t)stream;
  uint8_t *ws = (uint8_t *)workspace;
  const void *xc = x;
  const uint8_t *xs = x_scales, *wc = (const uint8_t *)w_codes;
  const bool vec = d % 8 == 0 && clt_aligned16(x) && x_layer_stride * e % 16 == 0 && d * e % 16 == 0;
  int rc = CLT_OK;
  if (!x_scales && p.own_x) {
    xc = ws + p.xc;
    xs = ws + p.xs;
    if (!p.tiles) {
      const MxRows rows{nullptr, 0, 0, p.xrows, nullptr};
      rc = mx_write(dtype, CLT_MXFP4, x, nullptr, x_layer_stride, d, L, 1, T, d, (uint32_t)p.padded, rows, ws + p.xc, ws + p.xs, s);
    }
  } else if (p.tiles) {
    if (p.own_x) {
      rc = launch_mx_widen(x, ws + p.xc, L, T, p.xrows, p.blocks, p.padded, s);
      xc = ws + p.xc;
    }
    const MxSide side{x_scales, ws + p.xs, nullptr, nullptr, (int)T, (int)p.blocks, (int)p.stages, 0};
    k_mx_tile_side<float, MX_MG><<<dim3((unsigned)(p.tm * p.stages), (unsigned)L), 256, 0, s>>>(side);
    xs = ws + p.xs;
  }
  if (rc != CLT_OK) return rc;
#define CLT_MXE(T_) \
  launch_mx_project<T_>(p, x_scales ? nullptr : x, xc, x_layer_stride, vec, xs, wc, w_scales, bias, ws, pre, T, d, F, L, b_layer_stride, pre_layer_stride, pre_row_stride, s)
  if (dtype == CLT_BF16) return CLT_MXE(bf16_t);
  if (dtype == CLT_F16) return CLT_MXE(f16_t);
  return CLT_MXE(float);
#undef CLT_MXE
}
