// skl_cvt_mx.hip - to and from MXFP4: 32 consecutive values of a row share a scale 2^s, s = max(floor(log2 of the largest
// magnitude) - 2, -126), and become E2M1 codes of x / 2^s, rounded to the nearest, ties to even, at most 6 (the OCP
// microscaling formats' rule; include/skl-gfx950.h).
//
// With b the bits of the largest magnitude, floor(log2) + 127 is b's exponent field, so the scale byte is max((b >> 23) - 2, 1):
// no logarithm and no division. A field of 255 is a NaN or an infinity. x / 2^s and the rounding are one instruction for two
// values (v_cvt_scalef32_pk_fp4_f32 / _bf16: to nearest even, saturating).
//
// All of it is bound by memory. Rows that are contiguous (or any others, value by value): four lanes hold a block, eight values of
// 16 (bf16) or 32 bytes each, and meet in two exchanges between neighbours; a lane's codes are a dword. 8192 x 8192 fp32: 66 us,
// 4.6 TB/s; 2048 x 8192 bf16 12.9. Columns (contiguous across the rows of the result): a lane holds two neighbouring rows of a block
// of 32 k, whose loads - 32, each a whole line or two per wave - are all under way together; the codes go through LDS, where 256 k of
// a row become a whole line. 4096 x 11008 bf16: 33 us, 3.5 TB/s, 2048 x 2048 6.3 (with two blocks to a wave, one after the other,
// 9.0); the order of the workgroups and four rows to a lane changed nothing. The way back, 4096 x 11008 to bf16: 18 us, 6.3 TB/s.
#include <hip/hip_runtime.h>

#include "skl_device.hpp"
#include "skl_mx.h"

namespace {

typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef unsigned short v2u16 __attribute__((ext_vector_type(2)));
// Accesses on any boundary that the elements themselves have.
typedef unsigned u1 __attribute__((aligned(1)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));
typedef u4 u4a2 __attribute__((aligned(2)));
typedef u4 u4a4 __attribute__((aligned(4)));
typedef unsigned u1a2 __attribute__((aligned(2)));
typedef unsigned u2 __attribute__((ext_vector_type(2)));
typedef u2 u2a4 __attribute__((aligned(4)));

// The scale byte for the largest magnitude's bits: 255 where a NaN or an infinity is in the block.
__device__ __forceinline__ unsigned scale_byte(unsigned largest) {
  const unsigned field = largest >> 23;
  return field == 255u ? 255u : field > 3u ? field - 2u : 1u;
}

__device__ __forceinline__ unsigned quad_max(unsigned v) {  // over the four lanes that hold a block
  unsigned o = (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true);  // lanes 1, 0, 3, 2
  v = v > o ? v : o;
  o = (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, true);  // lanes 2, 3, 0, 1
  return v > o ? v : o;
}

// Eight values of a row as a lane holds them.
struct EightF32 {
  typedef float T;
  unsigned w[8];
  __device__ __forceinline__ void load(const float *p) {
    const u4 lo = *reinterpret_cast<const u4a4 *>(p), hi = *reinterpret_cast<const u4a4 *>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = lo[i], w[4 + i] = hi[i];
  }
  __device__ __forceinline__ void set(int i, const float *p) { w[i] = __float_as_uint(*p); }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = 0;
  }
  __device__ __forceinline__ unsigned largest() const {
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const unsigned a = w[i] & 0x7FFFFFFFu;
      m = m > a ? m : a;
    }
    return m;
  }
  __device__ __forceinline__ unsigned codes(float scale) const {
    unsigned r = 0;
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, __uint_as_float(w[0]), __uint_as_float(w[1]), scale, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, __uint_as_float(w[2]), __uint_as_float(w[3]), scale, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, __uint_as_float(w[4]), __uint_as_float(w[5]), scale, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, __uint_as_float(w[6]), __uint_as_float(w[7]), scale, 3);
  }
};

__device__ __forceinline__ v2bf as_bf16(unsigned w) { return __builtin_bit_cast(v2bf, w); }
__device__ __forceinline__ unsigned max2(unsigned a, unsigned b) {  // of the two halves each
  return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(v2u16, a), __builtin_bit_cast(v2u16, b)));
}

struct EightBf16 {
  typedef uint16_t T;
  unsigned w[4];
  __device__ __forceinline__ void load(const uint16_t *p) {
    const u4 v = *reinterpret_cast<const u4a2 *>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = v[i];
  }
  __device__ __forceinline__ void set(int i, const uint16_t *p) { w[i >> 1] |= (unsigned)*p << (16 * (i & 1)); }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = 0;
  }
  __device__ __forceinline__ unsigned largest() const {
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) m = max2(m, w[i] & 0x7FFF7FFFu);
    const unsigned lo = m << 16, hi = m & 0xFFFF0000u;
    return lo > hi ? lo : hi;
  }
  __device__ __forceinline__ unsigned codes(float scale) const {
    unsigned r = 0;
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, as_bf16(w[0]), scale, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, as_bf16(w[1]), scale, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, as_bf16(w[2]), scale, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, as_bf16(w[3]), scale, 3);
  }
};

// Rows. R rounds of 64 blocks per workgroup, all loads requested before the first is used. CONTIGUOUS: cs == 1.
template <class Eight, int R, bool CONTIGUOUS>
__global__ void __launch_bounds__(256) cvt_to_mx_rows_kernel(const typename Eight::T *__restrict__ src, size_t rs, size_t cs, unsigned blocks,
                                                             unsigned all, size_t k, uint8_t *__restrict__ dst, size_t row_bytes,
                                                             uint8_t *__restrict__ scales, size_t lds) {
  Eight v[R];
  size_t row[R], p0[R];
  const unsigned first = blockIdx.x * (64u * R) + (threadIdx.x >> 2), q = threadIdx.x & 3u;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const unsigned b = first + 64u * r;
    row[r] = b / blocks;
    p0[r] = (size_t)(b - (unsigned)row[r] * blocks) * 32 + 8 * q;
    if (CONTIGUOUS && b < all && p0[r] + 8 <= k) {
      v[r].load(src + row[r] * rs + p0[r]);
    } else {
      v[r].clear();
      if (b < all)
        for (int i = 0; i < 8; ++i)
          if (p0[r] + i < k) v[r].set(i, src + row[r] * rs + (p0[r] + i) * cs);
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const unsigned b = first + 64u * r;
    const unsigned s = scale_byte(quad_max(v[r].largest()));
    const unsigned codes = s == 255u ? 0u : v[r].codes(__uint_as_float(s << 23));
    if (b >= all) continue;
    uint8_t *to = dst + row[r] * row_bytes + p0[r] / 2;
    if (p0[r] + 8 <= k) {
      *reinterpret_cast<u1 *>(to) = codes;
    } else {
      for (size_t i = 0; p0[r] + 2 * i < k; ++i) to[i] = (uint8_t)(codes >> (8 * i));
    }
    if (q == 0) scales[row[r] * lds + p0[r] / 32] = (uint8_t)s;
  }
}

// Columns: rs == 1. A workgroup takes 128 rows of the result and 256 k of each, a wave one of the eight blocks.
constexpr int kAcrossThreads = 512, kAcrossRows = 128, kAcrossK = 256, kAcrossPitch = 144;  // bytes of a row in LDS: 16 more than it holds, against bank conflicts

template <class T>
struct PairOfRows;
template <>
struct PairOfRows<uint16_t> {
  unsigned w[32];  // both rows at one k
  __device__ __forceinline__ void load(int i, const uint16_t *p, bool two) {
    if (two) w[i] = *reinterpret_cast<const u1a2 *>(p);
    else w[i] = *p;
  }
  __device__ __forceinline__ void clear(int i) { w[i] = 0; }
  __device__ __forceinline__ void largest(unsigned &m0, unsigned &m1) const {
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) m = max2(m, w[i] & 0x7FFF7FFFu);
    m0 = m << 16, m1 = m & 0xFFFF0000u;
  }
  // Eight values of row `which`, from k = 8 * at on.
  template <int WHICH>
  __device__ __forceinline__ unsigned codes(int at, float scale) const {
    constexpr unsigned pick = WHICH ? 0x07060302u : 0x05040100u;
    unsigned r = 0;
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, as_bf16(__builtin_amdgcn_perm(w[8 * at + 1], w[8 * at + 0], pick)), scale, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, as_bf16(__builtin_amdgcn_perm(w[8 * at + 3], w[8 * at + 2], pick)), scale, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, as_bf16(__builtin_amdgcn_perm(w[8 * at + 5], w[8 * at + 4], pick)), scale, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, as_bf16(__builtin_amdgcn_perm(w[8 * at + 7], w[8 * at + 6], pick)), scale, 3);
  }
};
template <>
struct PairOfRows<float> {
  u2 w[32];
  __device__ __forceinline__ void load(int i, const float *p, bool two) {
    if (two) w[i] = *reinterpret_cast<const u2a4 *>(p);
    else w[i] = u2{__float_as_uint(*p), 0u};
  }
  __device__ __forceinline__ void clear(int i) { w[i] = u2{0u, 0u}; }
  __device__ __forceinline__ void largest(unsigned &m0, unsigned &m1) const {
    m0 = m1 = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const unsigned a = w[i].x & 0x7FFFFFFFu, b = w[i].y & 0x7FFFFFFFu;
      m0 = m0 > a ? m0 : a, m1 = m1 > b ? m1 : b;
    }
  }
  template <int WHICH>
  __device__ __forceinline__ unsigned codes(int at, float scale) const {
    unsigned r = 0;
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, __uint_as_float(w[8 * at + 0][WHICH]), __uint_as_float(w[8 * at + 1][WHICH]), scale, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, __uint_as_float(w[8 * at + 2][WHICH]), __uint_as_float(w[8 * at + 3][WHICH]), scale, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, __uint_as_float(w[8 * at + 4][WHICH]), __uint_as_float(w[8 * at + 5][WHICH]), scale, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, __uint_as_float(w[8 * at + 6][WHICH]), __uint_as_float(w[8 * at + 7][WHICH]), scale, 3);
  }
};

template <class T>
__global__ void __launch_bounds__(kAcrossThreads) cvt_to_mx_columns_kernel(const T *__restrict__ src, size_t cs, size_t m, size_t k, uint8_t *__restrict__ dst,
                                                                size_t row_bytes, uint8_t *__restrict__ scales, size_t lds) {
  __shared__ __attribute__((aligned(16))) uint8_t lines[kAcrossRows * kAcrossPitch];
  __shared__ __attribute__((aligned(8))) uint8_t bytes[kAcrossRows][8];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const size_t row0 = (size_t)blockIdx.y * kAcrossRows, k0 = (size_t)blockIdx.x * kAcrossK;
  const size_t row = row0 + 2 * (size_t)lane;
  const bool one = row < m, two = row + 1 < m;
  const size_t kb = k0 + 32 * (size_t)wave;
  PairOfRows<T> v;
  const T *p = src + row;
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    if (one && kb + i < k) v.load(i, p + (kb + i) * cs, two);
    else v.clear(i);
  }
  unsigned m0, m1;
  v.largest(m0, m1);
  const unsigned s0 = scale_byte(m0), s1 = scale_byte(m1);
  const float f0 = __uint_as_float(s0 << 23), f1 = __uint_as_float(s1 << 23);
  u4 c0, c1;
#pragma unroll
  for (int at = 0; at < 4; ++at) {
    c0[at] = s0 == 255u ? 0u : v.template codes<0>(at, f0);
    c1[at] = s1 == 255u ? 0u : v.template codes<1>(at, f1);
  }
  *reinterpret_cast<u4 *>(lines + (2 * lane) * kAcrossPitch + 16 * wave) = c0;
  *reinterpret_cast<u4 *>(lines + (2 * lane + 1) * kAcrossPitch + 16 * wave) = c1;
  bytes[2 * lane][wave] = (uint8_t)s0;
  bytes[2 * lane + 1][wave] = (uint8_t)s1;
  __syncthreads();
  const size_t rows = m - row0 < (size_t)kAcrossRows ? m - row0 : (size_t)kAcrossRows;
  const size_t left = k - k0;  // values from here on
#pragma unroll
  for (int pass = 0; pass < 2; ++pass) {
    const unsigned r = 64u * pass + (threadIdx.x >> 3), piece = threadIdx.x & 7u;
    if (r >= rows || 32 * (size_t)piece >= left) continue;
    uint8_t *to = dst + (row0 + r) * row_bytes + k0 / 2 + 16 * piece;
    const uint8_t *from = lines + r * kAcrossPitch + 16 * piece;
    if (32 * (size_t)piece + 32 <= left) {
      typedef u4 u4a1 __attribute__((aligned(1)));
      *reinterpret_cast<u4a1 *>(to) = *reinterpret_cast<const u4 *>(from);
    } else {
      for (size_t i = 0; 32 * (size_t)piece + 2 * i < left; ++i) to[i] = from[i];
    }
  }
  if (left >= (size_t)kAcrossK) {
    typedef u2 u2a1 __attribute__((aligned(1)));
    if (threadIdx.x < rows) *reinterpret_cast<u2a1 *>(scales + (row0 + threadIdx.x) * lds + k0 / 32) = *reinterpret_cast<const u2 *>(bytes[threadIdx.x]);
    return;
  }
  for (unsigned at = threadIdx.x; at < kAcrossRows * 8u; at += kAcrossThreads) {
    const unsigned r = at >> 3, block = at & 7u;
    if (r < rows && 32 * (size_t)block < left) scales[(row0 + r) * lds + k0 / 32 + block] = bytes[r][block];
  }
}

// The way back: a lane reads the dword of eight codes and its block's scale.
template <class T, bool CONTIGUOUS>
__global__ void __launch_bounds__(256) cvt_from_mx_kernel(const uint8_t *__restrict__ codes, size_t row_bytes, const uint8_t *__restrict__ scales,
                                                          size_t lds, unsigned blocks, unsigned all, size_t k, T *__restrict__ dst, size_t rs, size_t cs) {
  constexpr int R = 2;
  const unsigned first = blockIdx.x * (64u * R) + (threadIdx.x >> 2), q = threadIdx.x & 3u;
  unsigned w[R], s[R];
  size_t row[R], p0[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const unsigned b = first + 64u * r;
    row[r] = b / blocks;
    p0[r] = (size_t)(b - (unsigned)row[r] * blocks) * 32 + 8 * q;
    w[r] = s[r] = 0;
    if (b >= all || p0[r] >= k) continue;
    const uint8_t *from = codes + row[r] * row_bytes + p0[r] / 2;
    if (p0[r] + 8 <= k) {
      w[r] = *reinterpret_cast<const u1 *>(from);
    } else {
      for (int i = 0; p0[r] + 2 * i < k; ++i) w[r] |= (unsigned)from[i] << (8 * i);
    }
    s[r] = scales[row[r] * lds + p0[r] / 32];
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const unsigned b = first + 64u * r;
    if (b >= all || p0[r] >= k) continue;
    // 2^(s - 127); a byte of 0 is half of what a byte of 1 is, and every value times a half is exact in fp32
    const float scale = __uint_as_float((s[r] == 0 ? 1u : s[r]) << 23);
    float v[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      typedef float v2f __attribute__((ext_vector_type(2)));
      v2f x = {0.0f, 0.0f};
      switch (i) {
        case 0: x = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[r], 1.0f, 0); break;
        case 1: x = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[r], 1.0f, 1); break;
        case 2: x = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[r], 1.0f, 2); break;
        default: x = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[r], 1.0f, 3); break;
      }
      v[2 * i] = __fmul_rn(x.x, scale), v[2 * i + 1] = __fmul_rn(x.y, scale);
    }
    if (s[r] == 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = __fmul_rn(v[i], 0.5f);
    }
    if (s[r] == 255u) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(0x7FC00000u);
    }
    T *to = dst + row[r] * rs + p0[r] * cs;
    if constexpr (sizeof(T) == 4) {
      if (CONTIGUOUS && p0[r] + 8 <= k) {
        *reinterpret_cast<u4a4 *>(to) = u4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
        *reinterpret_cast<u4a4 *>(to + 4) = u4{__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7])};
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (p0[r] + i < k) to[i * cs] = v[i];
      }
    } else {  // a value's bf16 is its upper half: nothing below it is set
      if (CONTIGUOUS && p0[r] + 8 <= k) {
        u4 o;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = __builtin_amdgcn_perm(__float_as_uint(v[2 * i + 1]), __float_as_uint(v[2 * i]), 0x07060302u);
        *reinterpret_cast<u4a2 *>(to) = o;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (p0[r] + i < k) to[i * cs] = (T)(__float_as_uint(v[i]) >> 16);
      }
    }
  }
}

// Rows in slabs whose blocks a 32-bit number counts, rows longer than that in pieces; four threads to a block, of which a launch has less than 2^32.
// f(first row, first value, values of a row here, blocks here)
constexpr size_t kMostBlocks = (size_t)1 << 29;
template <class F>
int in_slabs(size_t m, size_t k, F f) {
  for (size_t p = 0; p < k; p += kMostBlocks * 32) {
    const size_t values = k - p < kMostBlocks * 32 ? k - p : kMostBlocks * 32, blocks = (values + 31) / 32, rows = kMostBlocks / blocks;
    for (size_t i = 0; i < m; i += rows) {
      const size_t here = m - i < rows ? m - i : rows;
      const int rc = f(i, p, values, (unsigned)(here * blocks));
      if (rc != 0) return rc;
    }
  }
  return 0;
}

// Few blocks: as many workgroups as there can be, else four rounds of loads per lane.
constexpr unsigned kFewBlocks = 64u * 4u * 512u;

template <class Eight>
int launch_rows(size_t m, size_t k, const typename Eight::T *src, size_t rs, size_t cs, uint8_t *codes, size_t ld, uint8_t *scales, size_t lds) {
  return in_slabs(m, k, [&](size_t i, size_t p, size_t k, unsigned all) {
    const unsigned blocks = (unsigned)((k + 31) / 32);
    const typename Eight::T *s = src + i * rs + p * cs;
    uint8_t *c = codes + i * (ld / 2) + p / 2, *sc = scales + i * lds + p / 32;
    hipStream_t st = skl_current_stream();
    if (cs != 1) cvt_to_mx_rows_kernel<Eight, 1, false><<<skl_div_up(all, 64), 256, 0, st>>>(s, rs, cs, blocks, all, k, c, ld / 2, sc, lds);
    else if (all <= kFewBlocks) cvt_to_mx_rows_kernel<Eight, 1, true><<<skl_div_up(all, 64), 256, 0, st>>>(s, rs, cs, blocks, all, k, c, ld / 2, sc, lds);
    else cvt_to_mx_rows_kernel<Eight, 4, true><<<skl_div_up(all, 256), 256, 0, st>>>(s, rs, cs, blocks, all, k, c, ld / 2, sc, lds);
    return skl_check_launch("cvt_to_mx_rows");
  });
}

template <class T>
int launch_columns(size_t m, size_t k, const T *src, size_t cs, uint8_t *codes, size_t ld, uint8_t *scales, size_t lds) {
  constexpr size_t kMostRows = (size_t)65535 * kAcrossRows, kMostK = (size_t)1 << 30;  // of a grid: two threads to a value of k, less than 2^32
  for (size_t p = 0; p < k; p += kMostK)
    for (size_t i = 0; i < m; i += kMostRows) {
      const size_t values = k - p < kMostK ? k - p : kMostK, here = m - i < kMostRows ? m - i : kMostRows;
      cvt_to_mx_columns_kernel<T><<<dim3(skl_div_up(values, kAcrossK), skl_div_up(here, kAcrossRows)), kAcrossThreads, 0, skl_current_stream()>>>(
          src + i + p * cs, cs, here, values, codes + i * (ld / 2) + p / 2, ld / 2, scales + i * lds + p / 32, lds);
      const int rc = skl_check_launch("cvt_to_mx_columns");
      if (rc != 0) return rc;
    }
  return 0;
}

}  // namespace

extern "C" int skl_hip_launch_cvt_to_mx(int dt, size_t m, size_t k, const void *src, size_t rs, size_t cs, uint8_t *codes, size_t ld,
                                        uint8_t *scales, size_t lds) {
  const bool columns = rs == 1 && cs != 1 && m > 1;
  if (dt == SKL_DT_F32) {
    const float *s = static_cast<const float *>(src);
    return columns ? launch_columns(m, k, s, cs, codes, ld, scales, lds) : launch_rows<EightF32>(m, k, s, rs, cs, codes, ld, scales, lds);
  }
  const uint16_t *s = static_cast<const uint16_t *>(src);
  return columns ? launch_columns(m, k, s, cs, codes, ld, scales, lds) : launch_rows<EightBf16>(m, k, s, rs, cs, codes, ld, scales, lds);
}

extern "C" int skl_hip_launch_cvt_from_mx(int dt, size_t m, size_t k, const skl_mx_operand *src, void *dst, size_t rs, size_t cs) {
  return in_slabs(m, k, [&](size_t i, size_t p, size_t k, unsigned all) {
    const unsigned blocks = (unsigned)((k + 31) / 32);
    const uint8_t *c = src->codes + i * (src->ld / 2) + p / 2, *sc = src->scales + i * src->lds + p / 32;
    hipStream_t st = skl_current_stream();
    const unsigned grid = skl_div_up(all, 128);
    if (dt == SKL_DT_F32) {
      float *d = static_cast<float *>(dst) + i * rs + p * cs;
      if (cs == 1) cvt_from_mx_kernel<float, true><<<grid, 256, 0, st>>>(c, src->ld / 2, sc, src->lds, blocks, all, k, d, rs, cs);
      else cvt_from_mx_kernel<float, false><<<grid, 256, 0, st>>>(c, src->ld / 2, sc, src->lds, blocks, all, k, d, rs, cs);
    } else {
      uint16_t *d = static_cast<uint16_t *>(dst) + i * rs + p * cs;
      if (cs == 1) cvt_from_mx_kernel<uint16_t, true><<<grid, 256, 0, st>>>(c, src->ld / 2, sc, src->lds, blocks, all, k, d, rs, cs);
      else cvt_from_mx_kernel<uint16_t, false><<<grid, 256, 0, st>>>(c, src->ld / 2, sc, src->lds, blocks, all, k, d, rs, cs);
    }
    return skl_check_launch("cvt_from_mx");
  });
}
