// skl_gemm_mxf4.hip - C = alpha * A * B + beta * C of two MXFP4 operands, both contiguous in K (include/skl-gfx950.h).
//
// v_mfma_scale_f32_32x32x64_f8f6f4 with both formats FP4: lane l holds the 32 values - 16 bytes - of row (column) l % 32 and of one of
// two blocks of 32 k, and that block's scale. So a lane's operand is one block with its scale, and which blocks of K
// meet in an instruction is free as long as A's and B's lanes take the same ones. In a chunk of 256 k (a 128-byte line of a row)
// the lower half of the wave takes blocks 0 to 3, the upper half blocks 4 to 7, one per instruction: the four scales a
// lane needs of a row are then one dword, and an instruction picks its byte of it.
//
// The instruction is given B's columns as its rows and A's rows as its columns, so that a lane's sums are four neighbouring
// values of a row of C.
#include <hip/hip_runtime.h>

#include <atomic>

#include "skl_device.hpp"
#include "skl_mx.h"

namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef v4i v4i_any __attribute__((aligned(1)));
typedef v4f v4f_any __attribute__((aligned(4)));
typedef unsigned v2u __attribute__((ext_vector_type(2)));
typedef v2u v2u_any __attribute__((aligned(1)));

struct MxArgs {
  const uint8_t *a, *b;  // row i of A at a + i * a_row (bytes), column j of B at b + j * b_col
  size_t a_row, b_col;
  const uint8_t *sa, *sb;
  size_t sa_row, sb_col;
  float *c;
  size_t rsc, csc;
  unsigned m, n;
  size_t k;
  skl_scalar alpha, beta;
  unsigned tiles_n;  // tiles along n
};

constexpr int kChunkK = 256, kLine = 128;

// The slot of a row's 16-byte piece in the row's line in LDS: lanes that read the same piece of 32 rows meet in no bank.
__device__ __forceinline__ unsigned slot_of(unsigned row, unsigned piece) { return piece ^ ((row >> 1) & 7u); }

// One of a workgroup's operands on its way from memory to LDS: ROWS rows of a chunk, 16 bytes at a time.
template <int ROWS, int THREADS>
struct Stage {
  static constexpr int kEach = ROWS * 8 / THREADS, kScales = (ROWS + THREADS - 1) / THREADS;
  static_assert(ROWS * 8 % THREADS == 0);
  v4i piece[kEach];
  v2u scale[kScales];

  // Rows from `rows` on are the last one again: computed, not written. Blocks beyond K are zeros with a scale of one; `masked`: what
  // lies behind K in its last block is not part of the matrix and counts as zero.
  __device__ __forceinline__ void load(const uint8_t *first, size_t pitch, const uint8_t *scales, size_t scale_pitch, unsigned rows, size_t k, size_t k0) {
    const bool whole = k0 + kChunkK <= k;  // the same for every thread
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const unsigned at = (unsigned)i * THREADS + threadIdx.x, r = at >> 3, q = at & 7u;
      const uint8_t *p = first + (size_t)(r < rows ? r : rows - 1) * pitch + k0 / 2 + 16 * q;
      if (whole) {
        piece[i] = *reinterpret_cast<const v4i_any *>(p);
      } else {
        const size_t kp = k0 + 32 * (size_t)q;
        piece[i] = v4i{0, 0, 0, 0};
        if (kp + 32 <= k) {
          piece[i] = *reinterpret_cast<const v4i_any *>(p);
        } else if (kp < k) {
          const unsigned left = (unsigned)(k - kp);  // values, 1 to 31
          for (unsigned byte = 0; 2 * byte < left; ++byte) {
            const unsigned v = 2 * byte + 1 < left ? p[byte] : p[byte] & 15u;
            piece[i][byte >> 2] |= (int)(v << (8 * (byte & 3u)));
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kScales; ++i) {
      const unsigned r = (unsigned)i * THREADS + threadIdx.x;
      const uint8_t *p = scales + (size_t)(r < rows ? r : rows - 1) * scale_pitch + k0 / 32;
      if (whole) {
        scale[i] = *reinterpret_cast<const v2u_any *>(p);
      } else {
        scale[i] = v2u{0x7F7F7F7Fu, 0x7F7F7F7Fu};
        for (unsigned byte = 0; byte < 8; ++byte)
          if (k0 + 32 * (size_t)byte < k) {
            const unsigned shift = 8 * (byte & 3u);
            scale[i][byte >> 2] = (scale[i][byte >> 2] & ~(255u << shift)) | ((unsigned)p[byte] << shift);
          }
      }
    }
  }
  __device__ __forceinline__ void store(char *lines, char *scale_bytes) const {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const unsigned at = (unsigned)i * THREADS + threadIdx.x, r = at >> 3, q = at & 7u;
      *reinterpret_cast<v4i *>(lines + r * kLine + slot_of(r, q) * 16) = piece[i];
    }
#pragma unroll
    for (int i = 0; i < kScales; ++i) {
      const unsigned r = (unsigned)i * THREADS + threadIdx.x;
      if (ROWS % THREADS == 0 || r < ROWS) *reinterpret_cast<v2u *>(scale_bytes + r * 8) = scale[i];
    }
  }
};

template <int OPSEL>
__device__ __forceinline__ v16f multiply(v4i x, v4i y, v16f sum, int sx, int sy) {
  const v8i xv = {x.x, x.y, x.z, x.w, 0, 0, 0, 0}, yv = {y.x, y.y, y.z, y.w, 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(xv, yv, sum, 4, 4, OPSEL, sx, OPSEL, sy);
}

// A tile of WM x WN waves, each of TM x TN blocks of 32 x 32.
template <int WM, int WN, int TM, int TN>
__global__ void __launch_bounds__(WM *WN * 64) gemm_mx_kernel(MxArgs p) {
  constexpr int kThreads = WM * WN * 64, kRows = WM * TM * 32, kCols = WN * TN * 32;
  constexpr int kStageBytes = (kRows + kCols) * kLine, kScaleBytes = (kRows + kCols) * 8;
  extern __shared__ __attribute__((aligned(128))) char mx_lds[];  // two stages, then two of scales
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wm = wave / WN, wn = wave % WN, l = lane & 31, half = lane >> 5;
  const unsigned row0 = (blockIdx.x / p.tiles_n) * kRows, col0 = (blockIdx.x % p.tiles_n) * kCols;
  const unsigned rows = p.m - row0 < (unsigned)kRows ? p.m - row0 : kRows, cols = p.n - col0 < (unsigned)kCols ? p.n - col0 : kCols;
  const uint8_t *a = p.a + (size_t)row0 * p.a_row, *b = p.b + (size_t)col0 * p.b_col;
  const uint8_t *sa = p.sa + (size_t)row0 * p.sa_row, *sb = p.sb + (size_t)col0 * p.sb_col;
  v16f sum[TN][TM];
#pragma unroll
  for (int j = 0; j < TN; ++j)
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) sum[j][i][r] = 0.0f;
  Stage<kRows, kThreads> ra;
  Stage<kCols, kThreads> rb;
  const size_t chunks = (p.k + kChunkK - 1) / kChunkK;
  if (chunks != 0) {
    ra.load(a, p.a_row, sa, p.sa_row, rows, p.k, 0);
    rb.load(b, p.b_col, sb, p.sb_col, cols, p.k, 0);
  }
  for (size_t chunk = 0; chunk < chunks; ++chunk) {
    char *lines = mx_lds + (chunk & 1) * kStageBytes, *scales = mx_lds + 2 * kStageBytes + (chunk & 1) * kScaleBytes;
    ra.store(lines, scales);
    rb.store(lines + kRows * kLine, scales + kRows * 8);
    __syncthreads();  // one per chunk: who writes this stage again has seen every wave through the chunk in between
    if (chunk + 1 < chunks) {
      ra.load(a, p.a_row, sa, p.sa_row, rows, p.k, (chunk + 1) * kChunkK);
      rb.load(b, p.b_col, sb, p.sb_col, cols, p.k, (chunk + 1) * kChunkK);
    }
    const unsigned ar = (unsigned)wm * (TM * 32) + l, br = (unsigned)wn * (TN * 32) + l;
    int scale_a[TM], scale_b[TN];
#pragma unroll
    for (int i = 0; i < TM; ++i) scale_a[i] = *reinterpret_cast<const int *>(scales + (ar + 32 * i) * 8 + 4 * half);
#pragma unroll
    for (int j = 0; j < TN; ++j) scale_b[j] = *reinterpret_cast<const int *>(scales + (kRows + br + 32 * j) * 8 + 4 * half);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const unsigned q = 4u * half + s;
      v4i x[TM], y[TN];
#pragma unroll
      for (int i = 0; i < TM; ++i) x[i] = *reinterpret_cast<const v4i *>(lines + (ar + 32 * i) * kLine + slot_of(ar + 32 * i, q) * 16);
#pragma unroll
      for (int j = 0; j < TN; ++j) y[j] = *reinterpret_cast<const v4i *>(lines + (kRows + br + 32 * j) * kLine + slot_of(br + 32 * j, q) * 16);
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          if (s == 0) sum[j][i] = multiply<0>(y[j], x[i], sum[j][i], scale_b[j], scale_a[i]);
          if (s == 1) sum[j][i] = multiply<1>(y[j], x[i], sum[j][i], scale_b[j], scale_a[i]);
          if (s == 2) sum[j][i] = multiply<2>(y[j], x[i], sum[j][i], scale_b[j], scale_a[i]);
          if (s == 3) sum[j][i] = multiply<3>(y[j], x[i], sum[j][i], scale_b[j], scale_a[i]);
        }
    }
  }
  // sum[j][i][4 q + r] is row 32 i + l of the wave's part of C, column 32 j + 8 q + 4 half + r.
  const bool init = skl_beta_is_zero<float>(p.beta);
  bool read_c = !init;
  if (init) {
    bool needs = false;
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) needs |= skl_initialise_needs_c(sum[j][i][r], p.alpha, p.beta);
    read_c = __any(needs);
  }
  const bool vec = p.csc == 1 && !read_c;
#pragma unroll
  for (int j = 0; j < TN; ++j)
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const unsigned r0 = (unsigned)wm * (TM * 32) + 32 * i + l;
      if (r0 >= rows) continue;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const unsigned c0 = (unsigned)wn * (TN * 32) + 32 * j + 8 * q + 4 * half;
        float *to = p.c + (size_t)(row0 + r0) * p.rsc + (size_t)(col0 + c0) * p.csc;
        if (vec && c0 + 4 <= cols) {
          v4f v;
#pragma unroll
          for (int r = 0; r < 4; ++r) v[r] = skl_initialise_plain(sum[j][i][4 * q + r], p.alpha, p.beta);
          *reinterpret_cast<v4f_any *>(to) = v;
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (c0 + r < cols) skl_update(sum[j][i][4 * q + r], to + (size_t)r * p.csc, p.alpha, p.beta);
        }
      }
    }
}

template <int WM, int WN, int TM, int TN>
int launch_tiles(MxArgs p) {
  constexpr int kRows = WM * TM * 32, kCols = WN * TN * 32, kBytes = 2 * (kRows + kCols) * (kLine + 8);
  static std::atomic<bool> configured{false};  // racing threads set the same value
  if (!configured.load(std::memory_order_acquire)) {
    const int rc = skl_check_hip(hipFuncSetAttribute(reinterpret_cast<const void *>(gemm_mx_kernel<WM, WN, TM, TN>),
                                                     hipFuncAttributeMaxDynamicSharedMemorySize, kBytes), "gemm_mx: LDS size");
    if (rc != 0) return rc;
    configured.store(true, std::memory_order_release);
  }
  const size_t tiles_m = ((size_t)p.m + kRows - 1) / kRows, tiles_n = ((size_t)p.n + kCols - 1) / kCols;
  if (tiles_m * tiles_n > 0x7FFFFFFFu) {
    skl_hip_record_error(-2, "gemm_mx: grid too large");
    return -2;
  }
  p.tiles_n = (unsigned)tiles_n;
  gemm_mx_kernel<WM, WN, TM, TN><<<(unsigned)(tiles_m * tiles_n), WM * WN * 64, kBytes, skl_current_stream()>>>(p);
  return skl_check_launch("gemm_mx");
}

}  // namespace

extern "C" int skl_hip_launch_gemm_mx(const skl_mx_gemm *g) {
  if (g->m > 0x7FFFFFFFu || g->n > 0x7FFFFFFFu) {
    skl_hip_record_error(-2, "gemm_mx: more than 2^31 rows or columns");
    return -2;
  }
  const MxArgs p = {g->a.codes, g->b.codes, g->a.ld / 2, g->b.ld / 2, g->a.scales, g->b.scales, g->a.lds, g->b.lds, g->c, g->rsc, g->csc,
                    (unsigned)g->m, (unsigned)g->n, g->k, g->alpha, g->beta, 0};
  const auto tiles = [&](size_t r, size_t c) { return ((g->m + r - 1) / r) * ((g->n + c - 1) / c); };
  if (tiles(256, 256) >= 200) return launch_tiles<2, 4, 4, 2>(p);
  if (tiles(128, 128) >= 200) return launch_tiles<2, 2, 2, 2>(p);
  return launch_tiles<2, 2, 1, 1>(p);
}
