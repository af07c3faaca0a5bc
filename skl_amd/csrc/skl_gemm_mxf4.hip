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
#include "skl_kcstream.hpp"
#include "skl_mx.h"
#include "skl_mx_rows.hpp"
#include "../../include/skl-hip.h"

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
  unsigned tiles_m, tiles_n;
  int past_caches;  // C is stored past them
  unsigned long long *shares;  // of K: [tile][share][8][thread], two sums each
  unsigned *counters;          // one per tile, zero between launches
};

constexpr int kChunkK = 256, kLine = 128;

// The slot of a row's 16-byte piece in the row's line in LDS: lanes that read the same piece of 32 rows meet in no bank.
__device__ __forceinline__ unsigned slot_of(unsigned row, unsigned piece) { return piece ^ ((row >> 1) & 7u); }

// The ends of rows. What lies behind a row is loaded by nobody: 16 bytes (eight scales) at an end are loaded from further down and moved into place, in one load - byte by byte, each
// waited for, the last chunk took longer than all others of a short K. Shorter rows do go byte by byte.
typedef unsigned __int128 u128;
struct EndOf {  // of the 16 bytes at `at`, in a row of `bytes`: where they are loaded from
  size_t from;
  __device__ __forceinline__ EndOf(size_t bytes, size_t at) : from(at + 16 <= bytes || bytes < 16 ? at : bytes - 16) {}
};
__device__ __forceinline__ v4i load_end(const uint8_t *row, size_t bytes, EndOf e) {
  if (bytes >= 16) return *reinterpret_cast<const v4i_any *>(row + e.from);
  v4i v = {0, 0, 0, 0};
  for (unsigned b = 0; e.from + b < bytes; ++b) v[b >> 2] |= (int)((unsigned)row[e.from + b] << (8 * (b & 3u)));
  return v;
}
// The values from 2 `at` on of a row of k, zeros behind its end; v: loaded from e.
__device__ __forceinline__ v4i settle_end(v4i v, size_t k, size_t at, EndOf e) {
  const size_t over = at - e.from;
  u128 bits = over < 16 ? __builtin_bit_cast(u128, v) >> (8 * (unsigned)over) : (u128)0;
  const size_t have = 2 * at < k ? k - 2 * at : 0;  // values
  if (have < 32) bits &= ((u128)1 << (4 * (unsigned)have)) - 1;
  return __builtin_bit_cast(v4i, bits);
}
// Eight scale bytes from `at` on of a row of `bytes`; ones behind its end.
__device__ __forceinline__ v2u load_scale_end(const uint8_t *row, size_t bytes, size_t at) {
  if (bytes >= 8) return *reinterpret_cast<const v2u_any *>(row + (at + 8 <= bytes ? at : bytes - 8));
  v2u v = {0, 0};
  for (unsigned b = 0; at + b < bytes; ++b) v[b >> 2] |= (unsigned)row[at + b] << (8 * (b & 3u));
  return v;
}
__device__ __forceinline__ v2u settle_scale_end(v2u v, size_t bytes, size_t at) {
  if (at + 8 <= bytes) return v;
  const unsigned over = bytes >= 8 ? (unsigned)(at + 8 - bytes) : 0u, have = at < bytes ? (unsigned)(bytes - at) : 0u;
  const unsigned long long kept = (1ull << (8 * have)) - 1, bits = over < 8 ? __builtin_bit_cast(unsigned long long, v) >> (8 * over) : 0ull;
  return __builtin_bit_cast(v2u, (bits & kept) | (0x7F7F7F7F7F7F7F7Full & ~kept));
}

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
    const size_t bytes = (k + 1) / 2, blocks = (k + 31) / 32;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const unsigned at = (unsigned)i * THREADS + threadIdx.x, r = at >> 3, q = at & 7u;
      const uint8_t *row = first + (size_t)(r < rows ? r : rows - 1) * pitch;
      piece[i] = whole ? *reinterpret_cast<const v4i_any *>(row + k0 / 2 + 16 * q) : load_end(row, bytes, EndOf(bytes, k0 / 2 + 16 * q));
    }
#pragma unroll
    for (int i = 0; i < kScales; ++i) {
      const unsigned r = (unsigned)i * THREADS + threadIdx.x;
      scale[i] = load_scale_end(scales + (size_t)(r < rows ? r : rows - 1) * scale_pitch, blocks, k0 / 32);
    }
    if (whole) return;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const size_t at = k0 / 2 + 16 * (((unsigned)i * THREADS + threadIdx.x) & 7u);
      piece[i] = settle_end(piece[i], k, at, EndOf(bytes, at));
    }
#pragma unroll
    for (int i = 0; i < kScales; ++i) scale[i] = settle_scale_end(scale[i], blocks, k0 / 32);
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

// C of a wave: sum[j][i][4 q + r] is row 32 i + l, column 32 j + 8 q + 4 half + r of its part, which begins at (wave_row, wave_col) of the tile. Rows of a
// row-major C go out as whole rows of 32 TN columns, by way of the wave's own `space` of kRowSpace<TN> bytes in LDS: written as the sums lie, 32 bytes of
// each of 32 rows per store, 8192^2 values took 270 us.
template <int TN>
constexpr int kRowPitch = 32 * TN * 4 + 16;  // 16 bytes more, so that 16 lanes with the same columns of 16 rows meet in no bank
template <int TN>
constexpr int kRowSpace = 32 * kRowPitch<TN>;

enum { kThrough, kPast, kRead, kAny };  // stored through the caches or past them; read first; any strides. EDGE: columns that do not exist

template <int HOW, bool EDGE, int TM, int TN>
__device__ __forceinline__ void write_rows(const MxArgs &p, const v16f (&sum)[TN][TM], unsigned row0, unsigned col0, unsigned rows, unsigned cols, int lane, char *space) {
  const int l = lane & 31, half = lane >> 5;
  constexpr int kRowsAt = MxRows<TN>::kRowsAt, kPasses = MxRows<TN>::kPasses;
  const MxRows<TN> mine(p.c + (size_t)row0 * p.rsc + (size_t)col0 * p.csc, p.rsc, p.csc, (unsigned)lane);
  const unsigned at_row = mine.at_row, at_col = mine.at_col;
  const bool init = skl_beta_is_zero<float>(p.beta);
#pragma unroll
  for (int i = 0; i < TM; ++i) {
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<v4f *>(space + l * kRowPitch<TN> + (32 * j + 8 * q + 4 * half) * 4) =
            v4f{sum[j][i][4 * q], sum[j][i][4 * q + 1], sum[j][i][4 * q + 2], sum[j][i][4 * q + 3]};
    const char *const from = space + at_row * kRowPitch<TN> + at_col * 4;
    if constexpr (HOW == kAny) {
#pragma unroll 1
      for (int n = 0; n < kPasses; ++n) {
        const unsigned r = 32u * i + (unsigned)n * kRowsAt;
        const v4f v = *reinterpret_cast<const v4f *>(from + n * kRowsAt * kRowPitch<TN>);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (mine.exists(r, rows) && at_col + e < cols) skl_update(v[e], mine.row(r) + (size_t)e * p.csc, p.alpha, p.beta);
      }
    } else {
      constexpr int kBatch = kPasses < 8 ? kPasses : 8;  // old values under way together
#pragma unroll
      for (int n0 = 0; n0 < kPasses; n0 += kBatch) {
        __builtin_amdgcn_sched_barrier(0);  // not the addresses of all of them at once
        v4f old[HOW == kRead ? kBatch : 1];
        if constexpr (HOW == kRead) {
#pragma unroll
          for (int n = 0; n < kBatch; ++n) {
            const unsigned r = 32u * i + (unsigned)(n0 + n) * kRowsAt;
            const float *const there = mine.readable(r, rows);
            if (EDGE && at_col + 4 > cols) {
#pragma unroll
              for (int e = 0; e < 4; ++e) old[n][e] = at_col + e < cols ? there[e] : 0.0f;
            } else {
              old[n] = *reinterpret_cast<const v4f_any *>(there);
            }
          }
        }
#pragma unroll
        for (int n = 0; n < kBatch; ++n) {
          const unsigned r = 32u * i + (unsigned)(n0 + n) * kRowsAt;
          v4f v = *reinterpret_cast<const v4f *>(from + (n0 + n) * kRowsAt * kRowPitch<TN>);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            v[e] = HOW != kRead ? skl_initialise_plain(v[e], p.alpha, p.beta)
                   : init       ? skl_initialise_with(v[e], old[n][e], p.alpha, p.beta)
                                : skl_combine(v[e], old[n][e], p.alpha, p.beta);
          if (!mine.exists(r, rows)) continue;
          float *const to = mine.row(r);
          if (EDGE && at_col + 4 > cols) {
#pragma unroll
            for (int e = 0; e < 3; ++e)
              if (at_col + e < cols) to[e] = v[e];
            continue;
          }
          // (Assembly: the compiler makes one of two branches that differ in this alone. The store reads its data for two states more, which the compiler does not look after here.)
          if constexpr (HOW == kPast) asm volatile("global_store_dwordx4 %0, %1, off nt\ns_nop 1" ::"v"(to), "v"(v) : "memory");
          else *reinterpret_cast<v4f_any *>(to) = v;
        }
      }
    }
  }
}

// (wave_row, wave_col): where the wave's part begins in the tile that begins at (row0, col0) and has `rows` x `cols` values that exist.
template <int TM, int TN>
__device__ __forceinline__ void write_c(const MxArgs &p, const v16f (&sum)[TN][TM], unsigned row0, unsigned col0, unsigned rows, unsigned cols, unsigned wave_row, unsigned wave_col, int lane,
                                        char *space) {
  if (wave_row >= rows || wave_col >= cols) return;
  bool read_c = !skl_beta_is_zero<float>(p.beta);
  if (!read_c) {
    bool needs = false;
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) needs |= skl_initialise_needs_c(sum[j][i][r], p.alpha, p.beta);
    read_c = __any(needs);
  }
  row0 += wave_row, col0 += wave_col, rows -= wave_row, cols -= wave_col;
  // (Columns that do not exist, value by value through kAny, made 2816 x 5000 x 7168 14 us slower than 2816 x 5120 x 7168.)
  const bool edge = cols < 32u * TN;
  if (p.csc != 1) write_rows<kAny, true, TM, TN>(p, sum, row0, col0, rows, cols, lane, space);
  else if (read_c && edge) write_rows<kRead, true, TM, TN>(p, sum, row0, col0, rows, cols, lane, space);
  else if (read_c) write_rows<kRead, false, TM, TN>(p, sum, row0, col0, rows, cols, lane, space);
  else if (edge) write_rows<kThrough, true, TM, TN>(p, sum, row0, col0, rows, cols, lane, space);
  else if (p.past_caches) write_rows<kPast, false, TM, TN>(p, sum, row0, col0, rows, cols, lane, space);
  else write_rows<kThrough, false, TM, TN>(p, sum, row0, col0, rows, cols, lane, space);
}

// Any layout: 64 x 64 tiles of four waves, one block of 32 x 32 each, operands through registers. 700 x 700 x 700 6.1 us, 1500 x 1500 x 1500 14.0.
__global__ void __launch_bounds__(256) gemm_mx_kernel(MxArgs p) {
  constexpr int WM = 2, WN = 2, TM = 1, TN = 1;
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
  __syncthreads();  // the waves' rows take the stages' place
  write_c<TM, TN>(p, sum, row0, col0, rows, cols, (unsigned)wm * (TM * 32), (unsigned)wn * (TN * 32), lane, mx_lds + wave * kRowSpace<TN>);
}

// Which tile a workgroup takes. Workgroups go to the eight dies in turn, each with a cache of its own: a die gets a run of tiles, which are walked in
// groups of eight rows of tiles, column by column.
__device__ __forceinline__ void tile_of(const MxArgs &p, unsigned id, unsigned all, unsigned *tile_m, unsigned *tile_n) {
  const unsigned die = id % 8, each = all / 8, over = all % 8;
  const unsigned t = die * each + (die < over ? die : over) + id / 8;
  const unsigned group = t / (8 * p.tiles_n), in = t % (8 * p.tiles_n), first = 8 * group;
  const unsigned rows = p.tiles_m - first < 8 ? p.tiles_m - first : 8;
  *tile_m = first + in % rows;
  *tile_n = in / rows;
}

// The same tile with its operands on their way from memory to LDS without registers (buffer_load ... lds), whole lines at a time, a chunk of
// 256 k ahead. Rows begin on 4-byte boundaries.
constexpr unsigned kRange = 0x7FFFFFF0u, kOutside = 0x7FFFFFF0u;  // of a buffer descriptor; an offset that loads zeros
typedef __attribute__((address_space(3))) char lds_char;

// What a wave requests of an operand per chunk: EACH instructions of eight lines. Lane l fetches the piece that belongs into slot l % 8 of row l / 8.
template <int EACH>
struct Lines {
  const uint8_t *base;
  unsigned off[EACH];
  __device__ __forceinline__ void set(const uint8_t *first, size_t pitch, unsigned rows, unsigned row0, int lane) {
    base = first;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const unsigned r = row0 + 8u * i + (unsigned)(lane >> 3);
      off[i] = (r < rows ? r : rows - 1) * (unsigned)pitch + (((unsigned)lane & 7u) ^ ((r >> 1) & 7u)) * 16u;
    }
  }
  // `blocks`: how many whole blocks there are from this chunk on; the others are zeros.
  template <bool TAIL>
  __device__ __forceinline__ void issue(lds_char *to, size_t chunk, unsigned blocks, unsigned row0, int lane) const {
    const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc((void *)(base + chunk * kLine), 0, (int)kRange, 0x00027000);
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const unsigned r = row0 + 8u * i + (unsigned)(lane >> 3);
      const unsigned o = TAIL && (((unsigned)lane & 7u) ^ ((r >> 1) & 7u)) >= blocks ? kOutside : off[i];
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void *)(to + (row0 + 8u * i) * kLine), 16, (int)o, 0, 0, 0);
    }
  }
};

// A wave's operands of one instruction: TM blocks of rows at `x`, TN of columns at `y`, 4096 bytes apart. The wait is the block's own: the compiler
// would make every read wait for all loads to LDS under way.
#define SKL_MX_RD(name, addr, off) "ds_read_b128 %[" #name "], %[" #addr "] offset:" #off "\n"
template <int TM, int TN>
__device__ __forceinline__ void read_blocks(v4i (&x)[TM], v4i (&y)[TN], unsigned px, unsigned py) {
  if constexpr (TM == 4 && TN == 4)
    asm volatile(SKL_MX_RD(y0, py, 0) SKL_MX_RD(x0, px, 0) SKL_MX_RD(x1, px, 4096) SKL_MX_RD(x2, px, 8192) SKL_MX_RD(x3, px, 12288) SKL_MX_RD(y1, py, 4096) SKL_MX_RD(y2, py, 8192)
                     SKL_MX_RD(y3, py, 12288) "s_waitcnt lgkmcnt(0)"
                 : [x0] "=&v"(x[0]), [x1] "=&v"(x[1]), [x2] "=&v"(x[2]), [x3] "=&v"(x[3]), [y0] "=&v"(y[0]), [y1] "=&v"(y[1]), [y2] "=&v"(y[2]), [y3] "=&v"(y[3])
                 : [px] "v"(px), [py] "v"(py) : "memory");
  else if constexpr (TM == 2 && TN == 2)
    asm volatile(SKL_MX_RD(y0, py, 0) SKL_MX_RD(x0, px, 0) SKL_MX_RD(x1, px, 4096) SKL_MX_RD(y1, py, 4096) "s_waitcnt lgkmcnt(0)"
                 : [x0] "=&v"(x[0]), [x1] "=&v"(x[1]), [y0] "=&v"(y[0]), [y1] "=&v"(y[1]) : [px] "v"(px), [py] "v"(py) : "memory");
  else
    asm volatile(SKL_MX_RD(y0, py, 0) SKL_MX_RD(x0, px, 0) "s_waitcnt lgkmcnt(0)" : [x0] "=&v"(x[0]), [y0] "=&v"(y[0]) : [px] "v"(px), [py] "v"(py) : "memory");
}
// Their scales of a chunk.
template <int TM, int TN>
__device__ __forceinline__ void read_scales(int (&x)[TM], int (&y)[TN], unsigned px, unsigned py) {
#define SKL_MX_RS(name, addr, off) "ds_read_b32 %[" #name "], %[" #addr "] offset:" #off "\n"
  if constexpr (TM == 4 && TN == 4)
    asm volatile(SKL_MX_RS(y0, py, 0) SKL_MX_RS(y1, py, 1024) SKL_MX_RS(y2, py, 2048) SKL_MX_RS(y3, py, 3072) SKL_MX_RS(x0, px, 0) SKL_MX_RS(x1, px, 1024) SKL_MX_RS(x2, px, 2048)
                     SKL_MX_RS(x3, px, 3072) "s_waitcnt lgkmcnt(0)"
                 : [x0] "=&v"(x[0]), [x1] "=&v"(x[1]), [x2] "=&v"(x[2]), [x3] "=&v"(x[3]), [y0] "=&v"(y[0]), [y1] "=&v"(y[1]), [y2] "=&v"(y[2]), [y3] "=&v"(y[3])
                 : [px] "v"(px), [py] "v"(py) : "memory");
  else if constexpr (TM == 2 && TN == 2)
    asm volatile(SKL_MX_RS(y0, py, 0) SKL_MX_RS(y1, py, 1024) SKL_MX_RS(x0, px, 0) SKL_MX_RS(x1, px, 1024) "s_waitcnt lgkmcnt(0)"
                 : [x0] "=&v"(x[0]), [x1] "=&v"(x[1]), [y0] "=&v"(y[0]), [y1] "=&v"(y[1]) : [px] "v"(px), [py] "v"(py) : "memory");
  else
    asm volatile(SKL_MX_RS(y0, py, 0) SKL_MX_RS(x0, px, 0) "s_waitcnt lgkmcnt(0)" : [x0] "=&v"(x[0]), [y0] "=&v"(y[0]) : [px] "v"(px), [py] "v"(py) : "memory");
}

// What a workgroup leaves for the last one of its tile goes past its die's cache and is read past it: no fence, which would write all of that cache back.
__device__ __forceinline__ void leave(unsigned long long *to, unsigned long long v) { __hip_atomic_store(to, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ unsigned long long found(const unsigned long long *from) { return __hip_atomic_load(from, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// Small tiles, 64 x 64, one block per wave: what the others leave. Where there are few of them, K is shared (blockIdx.y): each share's sums go to
// scratch memory, and the last of a tile's workgroups adds them in the order of K.
__global__ void __launch_bounds__(256) gemm_mx_stream_kernel(MxArgs p) {
  constexpr int WM = 2, WN = 2, TM = 1, TN = 1, kWaves = WM * WN, kThreads = kWaves * 64, kRows = WM * TM * 32, kCols = WN * TN * 32;
  constexpr int kStageBytes = (kRows + kCols) * kLine, kScaleBytes = (kRows + kCols) * 8, kScales = (kRows + kCols + kThreads - 1) / kThreads;
  extern __shared__ __attribute__((aligned(1024))) char mx_lds[];  // two stages, then two of scales
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wm = wave / WN, wn = wave % WN, l = lane & 31, half = lane >> 5;
  unsigned tile_m, tile_n;
  tile_of(p, blockIdx.x, gridDim.x, &tile_m, &tile_n);
  const unsigned row0 = tile_m * kRows, col0 = tile_n * kCols;
  const unsigned rows = p.m - row0 < (unsigned)kRows ? p.m - row0 : kRows, cols = p.n - col0 < (unsigned)kCols ? p.n - col0 : kCols;
  const unsigned ring = (unsigned)(uintptr_t)(lds_char *)mx_lds;
  lds_char *stages = (lds_char *)mx_lds;
  __shared__ unsigned arrived;
  const size_t chunks = (p.k + kChunkK - 1) / kChunkK;
  const size_t c0 = chunks * blockIdx.y / gridDim.y, c1 = chunks * (blockIdx.y + 1) / gridDim.y;
  const unsigned blocks = (unsigned)(p.k / 32), part = (unsigned)(p.k % 32);  // whole blocks, values of the one behind them

  Lines<kRows / 8 / kWaves> la;
  Lines<kCols / 8 / kWaves> lb;
  const unsigned ra0 = (unsigned)wave * (kRows / kWaves), rb0 = (unsigned)wave * (kCols / kWaves);
  la.set(p.a + (size_t)row0 * p.a_row, p.a_row, rows, ra0, lane);
  lb.set(p.b + (size_t)col0 * p.b_col, p.b_col, cols, rb0, lane);
  auto request = [&](size_t chunk) {
    lds_char *to = stages + (chunk & 1) * kStageBytes;
    if ((chunk + 1) * 8 <= blocks) {
      la.template issue<false>(to, chunk, 0, ra0, lane);
      lb.template issue<false>(to + kRows * kLine, chunk, 0, rb0, lane);
    } else {
      const unsigned left = blocks - (unsigned)chunk * 8;
      la.template issue<true>(to, chunk, left, ra0, lane);
      lb.template issue<true>(to + kRows * kLine, chunk, left, rb0, lane);
    }
  };
  // The scales of a thread's rows: first A's, then B's.
  const uint8_t *scale_at[kScales];
  v2u scale[kScales];
#pragma unroll
  for (int i = 0; i < kScales; ++i) {
    const unsigned r = (unsigned)i * kThreads + threadIdx.x, c = r - kRows;
    scale_at[i] = r < (unsigned)kRows ? p.sa + (size_t)(row0 + (r < rows ? r : rows - 1)) * p.sa_row : p.sb + (size_t)(col0 + (c < cols ? c : cols - 1)) * p.sb_col;
  }
  const size_t per_row = blocks + (part != 0);
  auto load_scales = [&](size_t chunk) {
#pragma unroll
    for (int i = 0; i < kScales; ++i) {
      scale[i] = load_scale_end(scale_at[i], per_row, chunk * 8);
    }
  };
  auto keep_scales = [&](size_t chunk) {
#pragma unroll
    for (int i = 0; i < kScales; ++i) {
      scale[i] = settle_scale_end(scale[i], per_row, chunk * 8);
      const unsigned r = (unsigned)i * kThreads + threadIdx.x;
      if ((kRows + kCols) % kThreads == 0 || r < (unsigned)(kRows + kCols))
        asm volatile("ds_write_b64 %0, %1" ::"v"(ring + 2 * kStageBytes + (unsigned)(chunk & 1) * kScaleBytes + r * 8), "v"(scale[i]) : "memory");
    }
  };
  // A last block that is not whole: read and masked, written over the zeros that stand for it.
  auto keep_part = [&](size_t chunk) {
    for (unsigned r = threadIdx.x; r < (unsigned)(kRows + kCols); r += kThreads) {
      const unsigned c = r - kRows;
      const uint8_t *const row = r < (unsigned)kRows ? p.a + (size_t)(row0 + (r < rows ? r : rows - 1)) * p.a_row : p.b + (size_t)(col0 + (c < cols ? c : cols - 1)) * p.b_col;
      const size_t bytes = (p.k + 1) / 2, at = 16 * (size_t)blocks;
      const v4i v = settle_end(load_end(row, bytes, EndOf(bytes, at)), p.k, at, EndOf(bytes, at));
      asm volatile("ds_write_b128 %0, %1" ::"v"(ring + (unsigned)(chunk & 1) * kStageBytes + r * kLine + slot_of(r, blocks & 7u) * 16), "v"(v) : "memory");
    }
  };
  // What chunk `chunk` needs is in LDS once every wave has come through here.
  auto settle = [&](size_t chunk) {
    keep_scales(chunk);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (part != 0 && chunk + 1 == chunks) {
      __builtin_amdgcn_s_barrier();  // the zeros that other waves' requests wrote are there
      keep_part(chunk);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
  };

  v16f sum[TN][TM];
#pragma unroll
  for (int j = 0; j < TN; ++j)
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) sum[j][i][r] = 0.0f;
  const unsigned ar = (unsigned)wm * (TM * 32) + l, br = kRows + (unsigned)wn * (TN * 32) + l;
  const unsigned turn = ((4u * half) ^ (((unsigned)l >> 1) & 7u)) * 16u;
  const unsigned at_x = ring + ar * kLine + turn, at_y = ring + br * kLine + turn;
  const unsigned sc_x = ring + 2 * kStageBytes + ar * 8 + 4 * half, sc_y = ring + 2 * kStageBytes + br * 8 + 4 * half;
  load_scales(c0);
  request(c0);
  settle(c0);
  for (size_t chunk = c0; chunk < c1; ++chunk) {
    const bool more = chunk + 1 < c1;
    if (more) {
      load_scales(chunk + 1);
      request(chunk + 1);
    }
    const unsigned stage = (unsigned)(chunk & 1) * kStageBytes, stage_s = (unsigned)(chunk & 1) * kScaleBytes;
    int scale_a[TM], scale_b[TN];
    read_scales<TM, TN>(scale_a, scale_b, sc_x + stage_s, sc_y + stage_s);
    v4i x[4][TM], y[4][TN];
#pragma unroll
    for (int s = 0; s < 4; ++s) read_blocks<TM, TN>(x[s], y[s], (at_x + stage) ^ (16u * s), (at_y + stage) ^ (16u * s));
    sum[0][0] = multiply<0>(y[0][0], x[0][0], sum[0][0], scale_b[0], scale_a[0]);
    sum[0][0] = multiply<1>(y[1][0], x[1][0], sum[0][0], scale_b[0], scale_a[0]);
    sum[0][0] = multiply<2>(y[2][0], x[2][0], sum[0][0], scale_b[0], scale_a[0]);
    sum[0][0] = multiply<3>(y[3][0], x[3][0], sum[0][0], scale_b[0], scale_a[0]);
    if (more) settle(chunk + 1);
  }
  if (gridDim.y > 1) {
    unsigned long long *const mine = p.shares + ((size_t)blockIdx.x * gridDim.y) * (8 * 256) + threadIdx.x;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      leave(mine + ((size_t)blockIdx.y * 8 + i) * 256, ((unsigned long long)__float_as_uint(sum[0][0][2 * i + 1]) << 32) | __float_as_uint(sum[0][0][2 * i]));
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's have reached memory
    __syncthreads();
    if (threadIdx.x == 0) arrived = __hip_atomic_fetch_add(p.counters + blockIdx.x, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (arrived != gridDim.y - 1) return;
    if (threadIdx.x == 0) __hip_atomic_store(p.counters + blockIdx.x, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
    for (int i = 0; i < 16; ++i) sum[0][0][i] = 0.0f;
#pragma unroll 2
    for (unsigned share = 0; share < gridDim.y; ++share) {
      unsigned long long v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = found(mine + ((size_t)share * 8 + i) * 256);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        sum[0][0][2 * i] = __fadd_rn(sum[0][0][2 * i], __uint_as_float((unsigned)v[i]));
        sum[0][0][2 * i + 1] = __fadd_rn(sum[0][0][2 * i + 1], __uint_as_float((unsigned)(v[i] >> 32)));
      }
    }
  }
  __syncthreads();  // the waves' rows take the stages' place
  write_c<TM, TN>(p, sum, row0, col0, rows, cols, (unsigned)wm * (TM * 32), (unsigned)wn * (TN * 32), lane, mx_lds + wave * kRowSpace<TN>);
}

// ---------------------------------------------------------------------------------------------------------------------
// Large tiles: four waves, one per SIMD (128 x 128 tiles: two), of TM x TN blocks each. What takes turns on the matrix cores elsewhere - products, reads of the next
// ones' operands from LDS, requests for a later chunk - goes out in one stream here: a step of a chunk, one product of each of a wave's pairs of blocks, is one block of
// assembly, and the wait at its end is for its own reads. What the compiler cannot know of it: a sum is under way until 20 states after its last product (the loop
// is followed by as many), and M0 is written (every load to LDS of this kernel writes it itself).
// 8192 x 8192 x 8192 280 us, 3.9 PFLOP/s: products alone need 168, without the stores of C 230; the loop, 1.7 us per chunk and tile, is as fast wherever the requests go
// out and runs at 1.96 GHz. 128 x 128 tiles, two to a compute unit, 1.05 us per chunk and pair: their lines are 61 of the 64 bytes per clock that a cache gives a compute unit;
// 2048 x 4096 x 4096 25.5 us, 2.7 PFLOP/s. 256 x 128 tiles, one to a unit: 28.
// ---------------------------------------------------------------------------------------------------------------------
#define SKL_MX_MODS0 " op_sel_hi:[0,0,0] cbsz:4 blgp:4\n"
#define SKL_MX_MODS1 " op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4\n"
#define SKL_MX_MODS2 " op_sel_hi:[1,1,0] cbsz:4 blgp:4\n"
#define SKL_MX_MODS3 " op_sel:[1,1,0] op_sel_hi:[1,1,0] cbsz:4 blgp:4\n"
#define SKL_MX_MUL(c, y, x, sy, sx, S) "v_mfma_scale_f32_32x32x64_f8f6f4 %[" #c "], %[" #y "], %[" #x "], %[" #c "], %[" #sy "], %[" #sx "]" SKL_MX_MODS##S
#define SKL_MX_TO(l, at) "s_add_u32 m0, %[" #l "], " #at "\n"
#define SKL_MX_GET(o, r) "buffer_load_dwordx4 %[" #o "], %[" #r "], 0 offen lds\n"

// run<S>: c += y x^T with the scales' byte S; n, m: the operands at p and q; step 3 also reads the next chunk's scales, at u and v. oa, ob: the requests' offsets, ra, rb their
// descriptors, la, lb where in LDS the first of each goes.
template <int TM, int TN>
struct Step;
template <>
struct Step<4, 4> {
  static constexpr int kAhead = 8;  // of a chunk's requests go out under step 3, the others under step 0 of the next chunk
  template <int S>
  __device__ static __forceinline__ void run(v16f (&c)[4][4], const v4i (&x)[4], const v4i (&y)[4], const int (&sx)[4], const int (&sy)[4], v4i (&n)[4], v4i (&m)[4], unsigned p, unsigned q,
                                             const unsigned (&oa)[8], const unsigned (&ob)[8], v4i ra, v4i rb, unsigned la, unsigned lb, int (&tx)[4], int (&ty)[4], unsigned u, unsigned v) {
    if constexpr (S == 0) {
    asm volatile(
        "s_nop 1\n" SKL_MX_MUL(c00, y0, x0, sy0, sx0, 0) SKL_MX_RD(n0, p, 0) SKL_MX_RD(m0, q, 0) SKL_MX_RD(n1, p, 4096)
        SKL_MX_TO(lb, 0) SKL_MX_MUL(c01, y0, x1, sy0, sx1, 0) SKL_MX_RD(m1, q, 4096) SKL_MX_RD(n2, p, 8192) SKL_MX_RD(m2, q, 8192) SKL_MX_GET(ob0, rb)
        SKL_MX_TO(lb, 1024) SKL_MX_MUL(c02, y0, x2, sy0, sx2, 0) SKL_MX_RD(n3, p, 12288) SKL_MX_RD(m3, q, 12288) SKL_MX_GET(ob1, rb) SKL_MX_MUL(c03, y0, x3, sy0, sx3, 0)
        SKL_MX_TO(lb, 2048) SKL_MX_MUL(c10, y1, x0, sy1, sx0, 0) SKL_MX_GET(ob2, rb) SKL_MX_MUL(c11, y1, x1, sy1, sx1, 0)
        SKL_MX_TO(lb, 3072) SKL_MX_MUL(c12, y1, x2, sy1, sx2, 0) SKL_MX_GET(ob3, rb) SKL_MX_MUL(c13, y1, x3, sy1, sx3, 0)
        SKL_MX_TO(lb, 4096) SKL_MX_MUL(c20, y2, x0, sy2, sx0, 0) SKL_MX_GET(ob4, rb) SKL_MX_MUL(c21, y2, x1, sy2, sx1, 0)
        SKL_MX_TO(lb, 5120) SKL_MX_MUL(c22, y2, x2, sy2, sx2, 0) SKL_MX_GET(ob5, rb) SKL_MX_MUL(c23, y2, x3, sy2, sx3, 0)
        SKL_MX_TO(lb, 6144) SKL_MX_MUL(c30, y3, x0, sy3, sx0, 0) SKL_MX_GET(ob6, rb) SKL_MX_MUL(c31, y3, x1, sy3, sx1, 0)
        SKL_MX_TO(lb, 7168) SKL_MX_MUL(c32, y3, x2, sy3, sx2, 0) SKL_MX_GET(ob7, rb) SKL_MX_MUL(c33, y3, x3, sy3, sx3, 0) "s_waitcnt lgkmcnt(0)"
        : [c00] "+a"(c[0][0]), [c01] "+a"(c[0][1]), [c02] "+a"(c[0][2]), [c03] "+a"(c[0][3]), [c10] "+a"(c[1][0]), [c11] "+a"(c[1][1]), [c12] "+a"(c[1][2]), [c13] "+a"(c[1][3]),
          [c20] "+a"(c[2][0]), [c21] "+a"(c[2][1]), [c22] "+a"(c[2][2]), [c23] "+a"(c[2][3]), [c30] "+v"(c[3][0]), [c31] "+v"(c[3][1]), [c32] "+v"(c[3][2]), [c33] "+v"(c[3][3]),
          [n0] "=&v"(n[0]), [n1] "=&v"(n[1]), [n2] "=&v"(n[2]), [n3] "=&v"(n[3]), [m0] "=&v"(m[0]), [m1] "=&v"(m[1]), [m2] "=&v"(m[2]), [m3] "=&v"(m[3])
        : [x0] "v"(x[0]), [x1] "v"(x[1]), [x2] "v"(x[2]), [x3] "v"(x[3]), [y0] "v"(y[0]), [y1] "v"(y[1]), [y2] "v"(y[2]), [y3] "v"(y[3]),
          [sx0] "v"(sx[0]), [sx1] "v"(sx[1]), [sx2] "v"(sx[2]), [sx3] "v"(sx[3]), [sy0] "v"(sy[0]), [sy1] "v"(sy[1]), [sy2] "v"(sy[2]), [sy3] "v"(sy[3]), [p] "v"(p), [q] "v"(q),
          [ob0] "v"(ob[0]), [ob1] "v"(ob[1]), [ob2] "v"(ob[2]), [ob3] "v"(ob[3]), [ob4] "v"(ob[4]), [ob5] "v"(ob[5]), [ob6] "v"(ob[6]), [ob7] "v"(ob[7]), [rb] "s"(rb),
          [lb] "s"(lb)
        : "memory", "scc");
    } else if constexpr (S == 1) {
    asm volatile(
        "s_nop 1\n" SKL_MX_MUL(c00, y0, x0, sy0, sx0, 1) SKL_MX_RD(n0, p, 0) SKL_MX_RD(m0, q, 0) SKL_MX_RD(n1, p, 4096)
        SKL_MX_MUL(c01, y0, x1, sy0, sx1, 1) SKL_MX_RD(m1, q, 4096) SKL_MX_RD(n2, p, 8192) SKL_MX_RD(m2, q, 8192)
        SKL_MX_MUL(c02, y0, x2, sy0, sx2, 1) SKL_MX_RD(n3, p, 12288) SKL_MX_RD(m3, q, 12288) SKL_MX_MUL(c03, y0, x3, sy0, sx3, 1) SKL_MX_MUL(c10, y1, x0, sy1, sx0, 1)
        SKL_MX_MUL(c11, y1, x1, sy1, sx1, 1) SKL_MX_MUL(c12, y1, x2, sy1, sx2, 1) SKL_MX_MUL(c13, y1, x3, sy1, sx3, 1) SKL_MX_MUL(c20, y2, x0, sy2, sx0, 1)
        SKL_MX_MUL(c21, y2, x1, sy2, sx1, 1) SKL_MX_MUL(c22, y2, x2, sy2, sx2, 1) SKL_MX_MUL(c23, y2, x3, sy2, sx3, 1) SKL_MX_MUL(c30, y3, x0, sy3, sx0, 1)
        SKL_MX_MUL(c31, y3, x1, sy3, sx1, 1) SKL_MX_MUL(c32, y3, x2, sy3, sx2, 1) SKL_MX_MUL(c33, y3, x3, sy3, sx3, 1) "s_waitcnt lgkmcnt(0)"
        : [c00] "+a"(c[0][0]), [c01] "+a"(c[0][1]), [c02] "+a"(c[0][2]), [c03] "+a"(c[0][3]), [c10] "+a"(c[1][0]), [c11] "+a"(c[1][1]), [c12] "+a"(c[1][2]), [c13] "+a"(c[1][3]),
          [c20] "+a"(c[2][0]), [c21] "+a"(c[2][1]), [c22] "+a"(c[2][2]), [c23] "+a"(c[2][3]), [c30] "+v"(c[3][0]), [c31] "+v"(c[3][1]), [c32] "+v"(c[3][2]), [c33] "+v"(c[3][3]),
          [n0] "=&v"(n[0]), [n1] "=&v"(n[1]), [n2] "=&v"(n[2]), [n3] "=&v"(n[3]), [m0] "=&v"(m[0]), [m1] "=&v"(m[1]), [m2] "=&v"(m[2]), [m3] "=&v"(m[3])
        : [x0] "v"(x[0]), [x1] "v"(x[1]), [x2] "v"(x[2]), [x3] "v"(x[3]), [y0] "v"(y[0]), [y1] "v"(y[1]), [y2] "v"(y[2]), [y3] "v"(y[3]),
          [sx0] "v"(sx[0]), [sx1] "v"(sx[1]), [sx2] "v"(sx[2]), [sx3] "v"(sx[3]), [sy0] "v"(sy[0]), [sy1] "v"(sy[1]), [sy2] "v"(sy[2]), [sy3] "v"(sy[3]), [p] "v"(p), [q] "v"(q)
        : "memory");
    } else if constexpr (S == 2) {
    asm volatile(
        "s_nop 1\n" SKL_MX_MUL(c00, y0, x0, sy0, sx0, 2) SKL_MX_RD(n0, p, 0) SKL_MX_RD(m0, q, 0) SKL_MX_RD(n1, p, 4096)
        SKL_MX_MUL(c01, y0, x1, sy0, sx1, 2) SKL_MX_RD(m1, q, 4096) SKL_MX_RD(n2, p, 8192) SKL_MX_RD(m2, q, 8192)
        SKL_MX_MUL(c02, y0, x2, sy0, sx2, 2) SKL_MX_RD(n3, p, 12288) SKL_MX_RD(m3, q, 12288) SKL_MX_MUL(c03, y0, x3, sy0, sx3, 2) SKL_MX_MUL(c10, y1, x0, sy1, sx0, 2)
        SKL_MX_MUL(c11, y1, x1, sy1, sx1, 2) SKL_MX_MUL(c12, y1, x2, sy1, sx2, 2) SKL_MX_MUL(c13, y1, x3, sy1, sx3, 2) SKL_MX_MUL(c20, y2, x0, sy2, sx0, 2)
        SKL_MX_MUL(c21, y2, x1, sy2, sx1, 2) SKL_MX_MUL(c22, y2, x2, sy2, sx2, 2) SKL_MX_MUL(c23, y2, x3, sy2, sx3, 2) SKL_MX_MUL(c30, y3, x0, sy3, sx0, 2)
        SKL_MX_MUL(c31, y3, x1, sy3, sx1, 2) SKL_MX_MUL(c32, y3, x2, sy3, sx2, 2) SKL_MX_MUL(c33, y3, x3, sy3, sx3, 2) "s_waitcnt lgkmcnt(0)"
        : [c00] "+a"(c[0][0]), [c01] "+a"(c[0][1]), [c02] "+a"(c[0][2]), [c03] "+a"(c[0][3]), [c10] "+a"(c[1][0]), [c11] "+a"(c[1][1]), [c12] "+a"(c[1][2]), [c13] "+a"(c[1][3]),
          [c20] "+a"(c[2][0]), [c21] "+a"(c[2][1]), [c22] "+a"(c[2][2]), [c23] "+a"(c[2][3]), [c30] "+v"(c[3][0]), [c31] "+v"(c[3][1]), [c32] "+v"(c[3][2]), [c33] "+v"(c[3][3]),
          [n0] "=&v"(n[0]), [n1] "=&v"(n[1]), [n2] "=&v"(n[2]), [n3] "=&v"(n[3]), [m0] "=&v"(m[0]), [m1] "=&v"(m[1]), [m2] "=&v"(m[2]), [m3] "=&v"(m[3])
        : [x0] "v"(x[0]), [x1] "v"(x[1]), [x2] "v"(x[2]), [x3] "v"(x[3]), [y0] "v"(y[0]), [y1] "v"(y[1]), [y2] "v"(y[2]), [y3] "v"(y[3]),
          [sx0] "v"(sx[0]), [sx1] "v"(sx[1]), [sx2] "v"(sx[2]), [sx3] "v"(sx[3]), [sy0] "v"(sy[0]), [sy1] "v"(sy[1]), [sy2] "v"(sy[2]), [sy3] "v"(sy[3]), [p] "v"(p), [q] "v"(q)
        : "memory");
    } else if constexpr (S == 3) {
    asm volatile(
        "s_nop 1\n" SKL_MX_MUL(c00, y0, x0, sy0, sx0, 3) SKL_MX_RD(n0, p, 0) SKL_MX_RD(m0, q, 0) SKL_MX_RD(n1, p, 4096)
        SKL_MX_TO(la, 0) SKL_MX_MUL(c01, y0, x1, sy0, sx1, 3) SKL_MX_RD(m1, q, 4096) SKL_MX_RD(n2, p, 8192) SKL_MX_RD(m2, q, 8192) SKL_MX_GET(oa0, ra)
        SKL_MX_TO(la, 1024) SKL_MX_MUL(c02, y0, x2, sy0, sx2, 3) SKL_MX_RD(n3, p, 12288) SKL_MX_RD(m3, q, 12288) SKL_MX_GET(oa1, ra)
        SKL_MX_MUL(c03, y0, x3, sy0, sx3, 3) SKL_MX_RS(tx0, u, 0) SKL_MX_RS(tx1, u, 1024) SKL_MX_RS(tx2, u, 2048)
        SKL_MX_TO(la, 2048) SKL_MX_MUL(c10, y1, x0, sy1, sx0, 3) SKL_MX_RS(tx3, u, 3072) SKL_MX_RS(ty0, v, 0) SKL_MX_RS(ty1, v, 1024) SKL_MX_GET(oa2, ra)
        SKL_MX_MUL(c11, y1, x1, sy1, sx1, 3) SKL_MX_RS(ty2, v, 2048) SKL_MX_RS(ty3, v, 3072) SKL_MX_TO(la, 3072) SKL_MX_MUL(c12, y1, x2, sy1, sx2, 3) SKL_MX_GET(oa3, ra)
        SKL_MX_MUL(c13, y1, x3, sy1, sx3, 3) SKL_MX_TO(la, 4096) SKL_MX_MUL(c20, y2, x0, sy2, sx0, 3) SKL_MX_GET(oa4, ra) SKL_MX_MUL(c21, y2, x1, sy2, sx1, 3)
        SKL_MX_TO(la, 5120) SKL_MX_MUL(c22, y2, x2, sy2, sx2, 3) SKL_MX_GET(oa5, ra) SKL_MX_MUL(c23, y2, x3, sy2, sx3, 3)
        SKL_MX_TO(la, 6144) SKL_MX_MUL(c30, y3, x0, sy3, sx0, 3) SKL_MX_GET(oa6, ra) SKL_MX_MUL(c31, y3, x1, sy3, sx1, 3)
        SKL_MX_TO(la, 7168) SKL_MX_MUL(c32, y3, x2, sy3, sx2, 3) SKL_MX_GET(oa7, ra) SKL_MX_MUL(c33, y3, x3, sy3, sx3, 3) "s_waitcnt lgkmcnt(0)"
        : [c00] "+a"(c[0][0]), [c01] "+a"(c[0][1]), [c02] "+a"(c[0][2]), [c03] "+a"(c[0][3]), [c10] "+a"(c[1][0]), [c11] "+a"(c[1][1]), [c12] "+a"(c[1][2]), [c13] "+a"(c[1][3]),
          [c20] "+a"(c[2][0]), [c21] "+a"(c[2][1]), [c22] "+a"(c[2][2]), [c23] "+a"(c[2][3]), [c30] "+v"(c[3][0]), [c31] "+v"(c[3][1]), [c32] "+v"(c[3][2]), [c33] "+v"(c[3][3]),
          [n0] "=&v"(n[0]), [n1] "=&v"(n[1]), [n2] "=&v"(n[2]), [n3] "=&v"(n[3]), [m0] "=&v"(m[0]), [m1] "=&v"(m[1]), [m2] "=&v"(m[2]), [m3] "=&v"(m[3]), [tx0] "=&v"(tx[0]),
          [tx1] "=&v"(tx[1]), [tx2] "=&v"(tx[2]), [tx3] "=&v"(tx[3]), [ty0] "=&v"(ty[0]), [ty1] "=&v"(ty[1]), [ty2] "=&v"(ty[2]), [ty3] "=&v"(ty[3])
        : [x0] "v"(x[0]), [x1] "v"(x[1]), [x2] "v"(x[2]), [x3] "v"(x[3]), [y0] "v"(y[0]), [y1] "v"(y[1]), [y2] "v"(y[2]), [y3] "v"(y[3]),
          [sx0] "v"(sx[0]), [sx1] "v"(sx[1]), [sx2] "v"(sx[2]), [sx3] "v"(sx[3]), [sy0] "v"(sy[0]), [sy1] "v"(sy[1]), [sy2] "v"(sy[2]), [sy3] "v"(sy[3]), [p] "v"(p), [q] "v"(q),
          [u] "v"(u), [v] "v"(v), [oa0] "v"(oa[0]), [oa1] "v"(oa[1]), [oa2] "v"(oa[2]), [oa3] "v"(oa[3]), [oa4] "v"(oa[4]), [oa5] "v"(oa[5]), [oa6] "v"(oa[6]), [oa7] "v"(oa[7]),
          [ra] "s"(ra), [la] "s"(la)
        : "memory", "scc");
    }
  }
};
template <>
struct Step<2, 2> {
  static constexpr int kAhead = 3;  // of a chunk's requests go out under step 3, the others under steps 0 and 1 of the next chunk
  template <int S>
  __device__ static __forceinline__ void run(v16f (&c)[2][2], const v4i (&x)[2], const v4i (&y)[2], const int (&sx)[2], const int (&sy)[2], v4i (&n)[2], v4i (&m)[2], unsigned p, unsigned q,
                                             const unsigned (&oa)[4], const unsigned (&ob)[4], v4i ra, v4i rb, unsigned la, unsigned lb, int (&tx)[2], int (&ty)[2], unsigned u, unsigned v) {
    if constexpr (S == 0) {
    asm volatile(
        "s_nop 1\n" SKL_MX_TO(la, 3072) SKL_MX_MUL(c00, y0, x0, sy0, sx0, 0) SKL_MX_RD(n0, p, 0) SKL_MX_RD(m0, q, 0) SKL_MX_RD(n1, p, 4096) SKL_MX_RD(m1, q, 4096) SKL_MX_GET(oa3, ra)
        SKL_MX_TO(lb, 0) SKL_MX_MUL(c01, y0, x1, sy0, sx1, 0) SKL_MX_GET(ob0, rb) SKL_MX_TO(lb, 1024) SKL_MX_MUL(c10, y1, x0, sy1, sx0, 0) SKL_MX_GET(ob1, rb)
        SKL_MX_MUL(c11, y1, x1, sy1, sx1, 0) "s_waitcnt lgkmcnt(0)"
        : [c00] "+a"(c[0][0]), [c01] "+a"(c[0][1]), [c10] "+a"(c[1][0]), [c11] "+a"(c[1][1]), [n0] "=&v"(n[0]), [n1] "=&v"(n[1]), [m0] "=&v"(m[0]), [m1] "=&v"(m[1])
        : [x0] "v"(x[0]), [x1] "v"(x[1]), [y0] "v"(y[0]), [y1] "v"(y[1]), [sx0] "v"(sx[0]), [sx1] "v"(sx[1]), [sy0] "v"(sy[0]), [sy1] "v"(sy[1]), [p] "v"(p), [q] "v"(q),
          [oa3] "v"(oa[3]), [ra] "s"(ra), [la] "s"(la), [ob0] "v"(ob[0]), [ob1] "v"(ob[1]), [rb] "s"(rb), [lb] "s"(lb)
        : "memory", "scc");
    } else if constexpr (S == 1) {
    asm volatile(
        "s_nop 1\n" SKL_MX_TO(lb, 2048) SKL_MX_MUL(c00, y0, x0, sy0, sx0, 1) SKL_MX_RD(n0, p, 0) SKL_MX_RD(m0, q, 0) SKL_MX_RD(n1, p, 4096) SKL_MX_RD(m1, q, 4096) SKL_MX_GET(ob2, rb)
        SKL_MX_MUL(c01, y0, x1, sy0, sx1, 1) SKL_MX_TO(lb, 3072) SKL_MX_MUL(c10, y1, x0, sy1, sx0, 1) SKL_MX_GET(ob3, rb) SKL_MX_MUL(c11, y1, x1, sy1, sx1, 1)
        "s_waitcnt lgkmcnt(0)"
        : [c00] "+a"(c[0][0]), [c01] "+a"(c[0][1]), [c10] "+a"(c[1][0]), [c11] "+a"(c[1][1]), [n0] "=&v"(n[0]), [n1] "=&v"(n[1]), [m0] "=&v"(m[0]), [m1] "=&v"(m[1])
        : [x0] "v"(x[0]), [x1] "v"(x[1]), [y0] "v"(y[0]), [y1] "v"(y[1]), [sx0] "v"(sx[0]), [sx1] "v"(sx[1]), [sy0] "v"(sy[0]), [sy1] "v"(sy[1]), [p] "v"(p), [q] "v"(q),
          [ob2] "v"(ob[2]), [ob3] "v"(ob[3]), [rb] "s"(rb), [lb] "s"(lb)
        : "memory", "scc");
    } else if constexpr (S == 2) {
    asm volatile(
        "s_nop 1\n" SKL_MX_MUL(c00, y0, x0, sy0, sx0, 2) SKL_MX_RD(n0, p, 0) SKL_MX_RD(m0, q, 0) SKL_MX_RD(n1, p, 4096) SKL_MX_RD(m1, q, 4096) SKL_MX_MUL(c01, y0, x1, sy0, sx1, 2)
        SKL_MX_MUL(c10, y1, x0, sy1, sx0, 2) SKL_MX_MUL(c11, y1, x1, sy1, sx1, 2) "s_waitcnt lgkmcnt(0)"
        : [c00] "+a"(c[0][0]), [c01] "+a"(c[0][1]), [c10] "+a"(c[1][0]), [c11] "+a"(c[1][1]), [n0] "=&v"(n[0]), [n1] "=&v"(n[1]), [m0] "=&v"(m[0]), [m1] "=&v"(m[1])
        : [x0] "v"(x[0]), [x1] "v"(x[1]), [y0] "v"(y[0]), [y1] "v"(y[1]), [sx0] "v"(sx[0]), [sx1] "v"(sx[1]), [sy0] "v"(sy[0]), [sy1] "v"(sy[1]), [p] "v"(p), [q] "v"(q)
        : "memory");
    } else if constexpr (S == 3) {
    asm volatile(
        "s_nop 1\n" SKL_MX_TO(la, 0) SKL_MX_MUL(c00, y0, x0, sy0, sx0, 3) SKL_MX_RD(n0, p, 0) SKL_MX_RD(m0, q, 0) SKL_MX_RD(n1, p, 4096) SKL_MX_RD(m1, q, 4096) SKL_MX_GET(oa0, ra)
        SKL_MX_TO(la, 1024) SKL_MX_MUL(c01, y0, x1, sy0, sx1, 3) SKL_MX_RS(tx0, u, 0) SKL_MX_RS(tx1, u, 1024) SKL_MX_RS(ty0, v, 0) SKL_MX_RS(ty1, v, 1024) SKL_MX_GET(oa1, ra)
        SKL_MX_TO(la, 2048) SKL_MX_MUL(c10, y1, x0, sy1, sx0, 3) SKL_MX_GET(oa2, ra) SKL_MX_MUL(c11, y1, x1, sy1, sx1, 3) "s_waitcnt lgkmcnt(0)"
        : [c00] "+a"(c[0][0]), [c01] "+a"(c[0][1]), [c10] "+a"(c[1][0]), [c11] "+a"(c[1][1]), [n0] "=&v"(n[0]), [n1] "=&v"(n[1]), [m0] "=&v"(m[0]), [m1] "=&v"(m[1]),
          [tx0] "=&v"(tx[0]), [tx1] "=&v"(tx[1]), [ty0] "=&v"(ty[0]), [ty1] "=&v"(ty[1])
        : [x0] "v"(x[0]), [x1] "v"(x[1]), [y0] "v"(y[0]), [y1] "v"(y[1]), [sx0] "v"(sx[0]), [sx1] "v"(sx[1]), [sy0] "v"(sy[0]), [sy1] "v"(sy[1]), [p] "v"(p), [q] "v"(q),
          [u] "v"(u), [v] "v"(v), [oa0] "v"(oa[0]), [oa1] "v"(oa[1]), [oa2] "v"(oa[2]), [ra] "s"(ra), [la] "s"(la)
        : "memory", "scc");
    }
  }
};

// A request by itself.
__device__ __forceinline__ void load_line(unsigned to, unsigned off, v4i rsrc) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(to), "v"(off), "s"(rsrc) : "memory");
}
__device__ __forceinline__ v4i descriptor(const uint8_t *base) {
  return v4i{__builtin_amdgcn_readfirstlane((int)(unsigned)(uintptr_t)base), __builtin_amdgcn_readfirstlane((int)(unsigned)((uintptr_t)base >> 32) & 0xFFFF), (int)kRange, 0x00027000};
}

// Scales come 1024 k at a time, 32 bytes of a row, two lanes each: read row by row a chunk at a time they cost the address path as much as the operands do.
constexpr int kGroupBytes = 32;
template <int TM, int TN>
struct Wide {
  static constexpr int kRows = 2 * TM * 32, kCols = 2 * TN * 32;
  static constexpr int kStageBytes = (kRows + kCols) * kLine, kScaleBytes = (kRows + kCols) * kGroupBytes;
  static constexpr int kLds = 2 * (kStageBytes + kScaleBytes);
  static_assert(4 * kRowSpace<TN> <= kLds);
};

// Rows of scales begin on 4-byte boundaries and are a multiple of 16 bytes long.
template <int TM, int TN>
__global__ void __launch_bounds__(256, TM == 2 ? 2 : 1) gemm_mx_wide_kernel(MxArgs p) {
  using W = Wide<TM, TN>;
  constexpr int kRows = W::kRows, kCols = W::kCols, kStageBytes = W::kStageBytes, kScaleBytes = W::kScaleBytes;
  constexpr int kA = kRows / 32, kB = kCols / 32, kS = (kRows + kCols) / 128;  // a wave's requests per chunk, of scales per group
  extern __shared__ __attribute__((aligned(1024))) char mx_lds[];  // two stages, then two groups of scales
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wm = wave >> 1, wn = wave & 1, l = lane & 31, half = lane >> 5;
  unsigned tile_m, tile_n;
  tile_of(p, blockIdx.x, gridDim.x, &tile_m, &tile_n);
  const unsigned row0 = tile_m * kRows, col0 = tile_n * kCols;
  const unsigned rows = p.m - row0 < (unsigned)kRows ? p.m - row0 : kRows, cols = p.n - col0 < (unsigned)kCols ? p.n - col0 : kCols;
  const unsigned ring = (unsigned)(uintptr_t)(lds_char *)mx_lds, ring_s = ring + 2 * kStageBytes;
  const unsigned chunks = (unsigned)((p.k + kChunkK - 1) / kChunkK);
  const unsigned blocks = (unsigned)(p.k / 32), part = (unsigned)(p.k % 32);  // whole blocks, values of the one behind them

  // Requests: lane l of one fetches the piece that belongs into slot l % 8 of row l / 8 of its eight. Rows that do not exist are the last one again.
  const uint8_t *const a0 = p.a + (size_t)row0 * p.a_row, *const b0 = p.b + (size_t)col0 * p.b_col;
  unsigned oa[kA], ob[kB], os[kS];
  const unsigned ra0 = (unsigned)wave * (kRows / 4), rb0 = (unsigned)wave * (kCols / 4);
  const unsigned piece = ((unsigned)lane & 7u) ^ ((unsigned)lane >> 4);  // of an even request; an odd one's is turned by four
#pragma unroll
  for (int i = 0; i < kA; ++i) {
    const unsigned r = ra0 + 8u * i + (unsigned)(lane >> 3);
    oa[i] = (r < rows ? r : rows - 1) * (unsigned)p.a_row + (piece ^ (4u * (i & 1))) * 16u;
  }
#pragma unroll
  for (int i = 0; i < kB; ++i) {
    const unsigned r = rb0 + 8u * i + (unsigned)(lane >> 3);
    ob[i] = (r < cols ? r : cols - 1) * (unsigned)p.b_col + (piece ^ (4u * (i & 1))) * 16u;
  }
  v4i ra = descriptor(a0), rb = descriptor(b0);
  const auto advance = [](v4i &r, unsigned by) {  // (a matrix does not cross 2^48)
    const unsigned long long at = (((unsigned long long)(unsigned)r.y << 32) | (unsigned)r.x) + by;
    r.x = (int)(unsigned)at, r.y = (int)(unsigned)(at >> 32);
  };
  // Ahead of the requests for chunk `next`: pieces of blocks that are not there load zeros.
  const auto trim = [&](unsigned next) {
    if ((next + 1) * 8 <= blocks) return;
    const unsigned left = next * 8 < blocks ? blocks - next * 8 : 0;
#pragma unroll
    for (int i = 0; i < kA; ++i) oa[i] = (piece ^ (4u * (i & 1))) < left ? oa[i] : kOutside;
#pragma unroll
    for (int i = 0; i < kB; ++i) ob[i] = (piece ^ (4u * (i & 1))) < left ? ob[i] : kOutside;
  };
  // Scales: a wave's kS requests of 32 rows each; A's rows first, then B's. Slot s of row r holds piece s ^ (r / 8 % 2), so that the reads of 16 rows meet in no bank twice.
  const unsigned per_row = blocks + (part != 0), s_piece = ((unsigned)lane & 1u) ^ (((unsigned)lane >> 4) & 1u);
  const uint8_t *const sa0 = p.sa + (size_t)row0 * p.sa_row, *const sb0 = p.sb + (size_t)col0 * p.sb_col;
  v4i rs[kS];
#pragma unroll
  for (int i = 0; i < kS; ++i) {
    const unsigned first = ((unsigned)wave * kS + i) * 32u, r = first % kRows + ((unsigned)lane >> 1);  // 32 rows of one operand
    const bool of_a = first < (unsigned)kRows;
    const unsigned c = first - kRows + ((unsigned)lane >> 1);
    os[i] = of_a ? (r < rows ? r : rows - 1) * (unsigned)p.sa_row : (c < cols ? c : cols - 1) * (unsigned)p.sb_col;
    os[i] += s_piece * 16u;
    rs[i] = descriptor(of_a ? sa0 : sb0);
  }
  const auto request_scales = [&](unsigned group) {
    const bool there = group * kGroupBytes + s_piece * 16u < per_row;
#pragma unroll
    for (int i = 0; i < kS; ++i) {
      load_line(ring_s + (group & 1u) * kScaleBytes + ((unsigned)wave * kS + i) * 1024u, there ? os[i] : kOutside, rs[i]);
      advance(rs[i], kGroupBytes);
    }
  };
  // A last block that is not whole: read and masked, written over the zeros that stand for it.
  const auto keep_part = [&](unsigned chunk) {
    __builtin_amdgcn_s_barrier();  // the zeros that other waves' requests wrote are there
    for (unsigned r = threadIdx.x; r < (unsigned)(kRows + kCols); r += 256) {
      const unsigned c = r - kRows;
      const uint8_t *const row = r < (unsigned)kRows ? a0 + (size_t)(r < rows ? r : rows - 1) * p.a_row : b0 + (size_t)(c < cols ? c : cols - 1) * p.b_col;
      const size_t bytes = (p.k + 1) / 2, at = 16 * (size_t)blocks;
      const v4i v = settle_end(load_end(row, bytes, EndOf(bytes, at)), p.k, at, EndOf(bytes, at));
      asm volatile("ds_write_b128 %0, %1" ::"v"(ring + (chunk & 1u) * kStageBytes + r * kLine + slot_of(r, blocks & 7u) * 16), "v"(v) : "memory");
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  };

  v16f sum[TN][TM];
#pragma unroll
  for (int j = 0; j < TN; ++j)
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) sum[j][i][r] = 0.0f;
  const unsigned to_a = ring + ra0 * kLine, to_b = ring + (kRows + rb0) * kLine;
  request_scales(0);
  trim(0);
#pragma unroll
  for (int i = 0; i < kA; ++i) load_line(to_a + i * 1024, oa[i], ra);
#pragma unroll
  for (int i = 0; i < kB; ++i) load_line(to_b + i * 1024, ob[i], rb);
  advance(ra, kLine);
  advance(rb, kLine);
  trim(1);
#pragma unroll
  for (int i = 0; i < Step<TM, TN>::kAhead; ++i) load_line(to_a + kStageBytes + i * 1024, oa[i], ra);
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(Step<TM, TN>::kAhead) : "memory");
  if (part != 0 && chunks == 1) keep_part(0);
  __builtin_amdgcn_s_barrier();

  const unsigned ar = (unsigned)wm * (TM * 32) + l, br = kRows + (unsigned)wn * (TN * 32) + l;
  const unsigned turn = ((4u * half) ^ (((unsigned)l >> 1) & 7u)) * 16u, turn_s = (((unsigned)l >> 3) & 1u) * 16u;
  const unsigned at_x = ring + ar * kLine + turn, at_y = ring + br * kLine + turn;
  const unsigned sc_x = ring_s + ar * kGroupBytes + 4 * half, sc_y = ring_s + br * kGroupBytes + 4 * half;
  // Where chunk c's scales are from sc_x on: its eight bytes are those at 8 (c % 2) of piece c / 2 % 2.
  const auto scales_of = [&](unsigned c) { return ((c >> 2) & 1u) * kScaleBytes + ((((c >> 1) & 1u) * 16u) ^ turn_s) + (c & 1u) * 8u; };
  v4i x[2][TM], y[2][TN];
  int scale_x[2][TM], scale_y[2][TN];
  read_scales<TM, TN>(scale_x[0], scale_y[0], sc_x + scales_of(0), sc_y + scales_of(0));
  read_blocks<TM, TN>(x[0], y[0], at_x, at_y);

  // Chunk c is multiplied in four steps, each of which reads the next one's operands; step 3 those of chunk c + 1, and its scales. Behind step 2 the last read of the
  // chunk's stage is done, and chunk c + 1 has to be there: a wait and a barrier, and from there on requests for chunk c + 2 take the stage.
  const auto chunk_of = [&]<int E>(unsigned chunk) __attribute__((always_inline)) {
    constexpr unsigned here = E * kStageBytes, other = (E ^ 1) * kStageBytes;
    const auto step = [&]<int S>(unsigned from, unsigned to, unsigned scales) __attribute__((always_inline)) {
      Step<TM, TN>::template run<S>(sum, x[S & 1], y[S & 1], scale_x[E], scale_y[E], x[(S & 1) ^ 1], y[(S & 1) ^ 1], at_x + from, at_y + from, oa, ob, ra, rb, to_a + to, to_b + to,
                                    scale_x[E ^ 1], scale_y[E ^ 1], sc_x + scales, sc_y + scales);
    };
    // what a step reads lies 16 bytes on: its slot's low bits turned
    step.template operator()<0>(here + ((turn ^ 16u) - turn), other, 0);
    step.template operator()<1>(here + ((turn ^ 32u) - turn), other, 0);
    if ((chunk & 3u) == 0) request_scales((chunk >> 2) + 1);
    step.template operator()<2>(here + ((turn ^ 48u) - turn), other, 0);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (part != 0 && chunk + 2 == chunks) keep_part(chunk + 1);
    __builtin_amdgcn_s_barrier();
    advance(ra, kLine);
    advance(rb, kLine);
    trim(chunk + 2);
    step.template operator()<3>(other, here, scales_of(chunk + 1));  // behind the last chunk: what lies there, not used
  };
  for (unsigned chunk = 0; chunk < chunks; chunk += 2) {
    chunk_of.template operator()<0>(chunk);
    if (chunk + 1 < chunks) chunk_of.template operator()<1>(chunk + 1);
  }
  asm volatile("s_nop 15\n s_nop 15\n s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();  // the waves' rows take the stages' place
  write_c<TM, TN>(p, sum, row0, col0, rows, cols, (unsigned)wm * (TM * 32), (unsigned)wn * (TN * 32), lane, mx_lds + wave * kRowSpace<TN>);
}

// ---------------------------------------------------------------------------------------------------------------------
// Few rows of A: the stream over B of skl_kcstream.hpp, A's lines beside B's. A workgroup has 16 CG columns and all of K; its waves take units of 256 k in turn, each from a
// ring of its own, two v_mfma_scale_f32_16x16x128_f8f6f4 per pair of 16 rows and 16 columns: lane group g takes piece g, then piece 4 + g of a line, a block of 32 k
// each. The scales of all of K are put next to the ring first, eight bytes per unit and row or column, while the first units are under way.
// 16 x 11008 x 4096: 24 MB of B in 7.5 us, a launch and a latency included.
// ---------------------------------------------------------------------------------------------------------------------
constexpr int kRowsScaleSpace = 32 * 1024;
template <int RG, int CG>
struct RowsShape {
  static constexpr int kUnitBytes = 16 * kLine * (CG + RG), kLoads = 2 * (CG + RG);  // per unit and wave
  static constexpr int kSpace = 160 * 1024 - kRowsScaleSpace;
  static constexpr int kWaves = 16 * kUnitBytes <= kSpace ? 8 : 4;
  static constexpr int kFit = kSpace / (kWaves * kUnitBytes), kUnits = kFit < 4 ? kFit : 4;
  static constexpr int kRingBytes = kWaves * kUnits * kUnitBytes;
  static constexpr int kPitch = 16 * CG + 1;
  static_assert(kUnits >= 2 && (kUnits - 1) * kLoads < 63);
  static_assert(kWaves * RG * 16 * kPitch * 4 <= kRingBytes, "the sums meet in the ring's place");
};
// Scales of `k` values of a workgroup's rows and columns: in blocks of 4096.
constexpr size_t rows_scale_bytes(int rg, int cg, size_t k) { return (k + 4095) / 4096 * 2048 * (size_t)(rg + cg); }

template <int RG, int CG>
__global__ void __launch_bounds__((RowsShape<RG, CG>::kWaves * 64)) gemm_mx_rows_kernel(MxArgs p) {
  using Shape = RowsShape<RG, CG>;
  using skl_kcstream::v2i;
  constexpr int kWaves = Shape::kWaves, kCols = 16 * CG, kAll = 16 * (CG + RG), kThreads = kWaves * 64;
  extern __shared__ __attribute__((aligned(1024))) char mx_lds[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, jl = lane & 15, g = lane >> 4;
  const unsigned col0 = blockIdx.x * kCols, cols = p.n - col0 < (unsigned)kCols ? p.n - col0 : kCols;
  const unsigned units = (unsigned)((p.k + 255) / 256), steps = (units + kWaves - 1) / kWaves;
  const unsigned ring = (unsigned)(uintptr_t)(lds_char *)mx_lds, scales = ring + Shape::kRingBytes;
  // The scales of 4096 k at a time, four to a lane, two columns or rows of A to a wave and load; those of an end are loaded from further down and moved into place.
  constexpr int kEach = kAll / (2 * kWaves);
  const unsigned count = (unsigned)(p.k / 32);  // of a row: at least 4
  unsigned word[kEach];
  const auto load_scales = [&](unsigned block) {
    const unsigned d = block * 32 + (unsigned)(lane & 31), from = 4 * d + 4 <= count ? 4 * d : count - 4, over = 4 * d - from;
#pragma unroll
    for (int q = 0; q < kEach; ++q) {
      const unsigned at = (unsigned)(q * kWaves + wave) * 2u + (unsigned)(lane >> 5), r = at - kCols;
      const uint8_t *row = at < (unsigned)kCols ? p.sb + (size_t)(col0 + (at < cols ? at : cols - 1)) * p.sb_col : p.sa + (size_t)(r < p.m ? r : p.m - 1) * p.sa_row;
      typedef unsigned any __attribute__((aligned(1)));
      word[q] = 0;
      if (over < 4) word[q] = *reinterpret_cast<const any *>(row + from) >> (8 * over);
    }
  };
  const auto keep_scales = [&](unsigned block) {
    const unsigned d = block * 32 + (unsigned)(lane & 31);
#pragma unroll
    for (int q = 0; q < kEach; ++q) {
      const unsigned at = (unsigned)(q * kWaves + wave) * 2u + (unsigned)(lane >> 5);
      // (spelled out: the compiler makes a store to LDS wait for the loads into LDS under way)
      asm volatile("ds_write_b32 %0, %1" ::"v"(scales + ((d >> 1) * kAll + at) * 8 + (d & 1) * 4), "v"(word[q]) : "memory");
    }
  };
  load_scales(0);
  skl_kcstream::Requests<RG, 1> ra;
  skl_kcstream::Requests<CG, 1> rb;
  ra.template set<false>((const char *)p.a, p.a_row, p.m, (unsigned)(p.k / 2), lane);
  rb.template set<true>((const char *)p.b + (size_t)col0 * p.b_col, p.b_col, p.n - col0, (unsigned)(p.k / 2), lane);
  lds_char *mine = (lds_char *)mx_lds + wave * Shape::kUnits * Shape::kUnitBytes;
  const unsigned at0 = (unsigned)(uintptr_t)mine + (unsigned)jl * kLine + (unsigned)(g ^ (jl & 7)) * 16u;
  const auto request = [&](unsigned step) {
    lds_char *to = mine + (step % Shape::kUnits) * Shape::kUnitBytes;
    rb.template issue<2>(to, step * kWaves + (unsigned)wave);
    ra.template issue<0>(to + 2048 * CG, step * kWaves + (unsigned)wave);
  };
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (unsigned s = 0; s < (unsigned)Shape::kUnits; ++s) request(s);
  __builtin_amdgcn_sched_barrier(0);
  keep_scales(0);
  for (unsigned block = 1; block * 128 < count; ++block) {
    load_scales(block);
    keep_scales(block);
  }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  v4f acc[2][RG][CG];
#pragma unroll
  for (int rg = 0; rg < RG; ++rg)
#pragma unroll
    for (int cg = 0; cg < CG; ++cg) acc[0][rg][cg] = acc[1][rg][cg] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  for (unsigned step = 0; step < steps; ++step) {
    skl_kcstream::wait_loads<(Shape::kUnits - 1) * Shape::kLoads>();
    const unsigned at = at0 + (step % Shape::kUnits) * Shape::kUnitBytes, unit = step * kWaves + (unsigned)wave;
    v2i sb[CG], sa[RG];
    const unsigned sc = scales + ((unit < units ? unit : 0u) * kAll + (unsigned)jl) * 8;
    skl_kcstream::read_scales<CG>(sb, sc);
    skl_kcstream::read_scales<RG>(sa, sc + kCols * 8);
    v4i a[2][RG], b[2][CG];
    skl_kcstream::read_operands<CG, RG>(b[0], a[0], at, at + 2048 * CG);
    skl_kcstream::read_operands<CG, RG>(b[1], a[1], at ^ 64u, (at ^ 64u) + 2048 * CG);
    request(step + Shape::kUnits);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int cg = 0; cg < CG; ++cg) {
        const int s_b = (int)__builtin_amdgcn_ubfe((unsigned)(h ? sb[cg].y : sb[cg].x), 8u * (unsigned)g, 8u);
        const v8i bv = {b[h][cg].x, b[h][cg].y, b[h][cg].z, b[h][cg].w, 0, 0, 0, 0};
#pragma unroll
        for (int rg = 0; rg < RG; ++rg) {
          const int s_a = (int)__builtin_amdgcn_ubfe((unsigned)(h ? sa[rg].y : sa[rg].x), 8u * (unsigned)g, 8u);
          const v8i av = {a[h][rg].x, a[h][rg].y, a[h][rg].z, a[h][rg].w, 0, 0, 0, 0};
          acc[h][rg][cg] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, acc[h][rg][cg], 4, 4, 0, s_a, 0, s_b);
        }
      }
  }
  skl_kcstream::wait_loads<0>();  // the requests behind the last unit write zeros into the ring
  __syncthreads();
  float(*red)[RG * 16][Shape::kPitch] = reinterpret_cast<float(*)[RG * 16][Shape::kPitch]>(mx_lds);
#pragma unroll
  for (int rg = 0; rg < RG; ++rg)
#pragma unroll
    for (int cg = 0; cg < CG; ++cg)
#pragma unroll
      for (int r = 0; r < 4; ++r) red[wave][16 * rg + 4 * g + r][cg * 16 + jl] = __fadd_rn(acc[0][rg][cg][r], acc[1][rg][cg][r]);
  __syncthreads();
  for (unsigned at = threadIdx.x; at < p.m * kCols; at += kThreads) {
    const unsigned i = at / kCols, j = at % kCols;
    if (j >= cols) continue;
    float v = red[0][i][j];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) v = __fadd_rn(v, red[w][i][j]);
    skl_update(v, p.c + (size_t)i * p.rsc + (size_t)(col0 + j) * p.csc, p.alpha, p.beta);
  }
}

// Rows of codes or scales on other boundaries or of other lengths are copied: codes as rows of whole blocks, scales as rows of a multiple of 16 bytes, zeros
// and scales of one behind what there is. One launch for what a product needs copied.
struct PadJob {
  const uint8_t *from;
  uint8_t *to;
  size_t from_row;   // bytes
  size_t rows;       // 0: nothing to copy
  unsigned words;    // of 16 bytes in a row of the copy
  unsigned lanes_log;  // threads to a row
  unsigned bytes;    // of a row that exist; the rest are `fill`
  unsigned last_mask;  // of its last byte's bits
  unsigned fill;
};
struct PadJobs {
  PadJob job[4];
};
// 16 bytes of a row from `at` on. A row's end is loaded from further down and moved into place: a load in a branch of its own would be waited for there.
__device__ __forceinline__ unsigned word_from(const PadJob &p, unsigned at) { return p.bytes < 16 ? 0u : at + 16 <= p.bytes ? at : p.bytes - 16; }
__device__ __forceinline__ v4i load_word(const PadJob &p, const uint8_t *row, unsigned from) {
  if (p.bytes >= 16) return *reinterpret_cast<const v4i_any *>(row + from);
  v4i v = {0, 0, 0, 0};
  for (unsigned b = 0; b < p.bytes; ++b) v[b >> 2] |= (int)((unsigned)row[b] << (8 * (b & 3u)));
  return v;
}
__device__ __forceinline__ v4i padded_word(const PadJob &p, v4i v, unsigned at, unsigned from) {
  if (at + 16 < p.bytes) return v;
  typedef unsigned __int128 u128;
  const unsigned over = at - from, have = at < p.bytes ? p.bytes - at : 0u;
  u128 bits = over < 16 ? __builtin_bit_cast(u128, v) >> (8 * over) : (u128)0;
  u128 fill = (u128)(p.fill * 0x0101010101010101ull);
  fill |= fill << 64;
  const u128 kept = have >= 16 ? ~(u128)0 : ((u128)1 << (8 * have)) - 1;
  bits = (bits & kept) | (fill & ~kept);
  if (have != 0) bits &= ~((u128)(p.last_mask ^ 255u) << (8 * (have - 1)));
  return __builtin_bit_cast(v4i, bits);
}
constexpr int kPadRows = 4;  // a thread's loads under way
__global__ void __launch_bounds__(256) mx_pad_kernel(PadJobs jobs) {
  const PadJob &p = jobs.job[blockIdx.y];
  const unsigned each = 256u >> p.lanes_log, lane = threadIdx.x & ((1u << p.lanes_log) - 1u);  // rows at a time
  const size_t step = (size_t)gridDim.x * each;
  for (size_t first = (size_t)blockIdx.x * each + (threadIdx.x >> p.lanes_log); first < p.rows; first += kPadRows * step)
    for (unsigned word = lane; word < p.words; word += 1u << p.lanes_log) {
      const unsigned from = word_from(p, 16 * word);
      v4i v[kPadRows];
#pragma unroll
      for (int i = 0; i < kPadRows; ++i) {
        const size_t row = first + i * step;
        v[i] = load_word(p, p.from + (row < p.rows ? row : first) * p.from_row, from);
      }
#pragma unroll
      for (int i = 0; i < kPadRows; ++i)
        if (const size_t row = first + i * step; row < p.rows) reinterpret_cast<v4i *>(p.to)[row * p.words + word] = padded_word(p, v[i], 16 * word, from);
    }
}

// Rows that loads to LDS read: on 4-byte boundaries, a tile's offsets 31-bit numbers.
bool rows_ok(const uint8_t *first, size_t pitch) { return ((uintptr_t)first & 3) == 0 && (pitch & 3) == 0 && pitch <= ((size_t)1 << 22); }
bool on_lines(const uint8_t *first, size_t pitch) { return rows_ok(first, pitch) && ((uintptr_t)first & (kLine - 1)) == 0 && (pitch & (kLine - 1)) == 0; }
// ... and scales, 16 bytes at a time.
bool scales_ok(const uint8_t *first, size_t pitch, size_t k) { return rows_ok(first, pitch) && ((k + 31) / 32) % 16 == 0; }

size_t up(size_t v, size_t to) { return (v + to - 1) / to * to; }

int configure(const void *kernel, int bytes, std::atomic<bool> &done) {  // racing threads set the same value
  if (done.load(std::memory_order_acquire)) return 0;
  const int rc = skl_check_hip(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes), "gemm_mx: LDS size");
  if (rc == 0) done.store(true, std::memory_order_release);
  return rc;
}

size_t tiles_of(const MxArgs &p, size_t rows, size_t cols) { return (p.m + rows - 1) / rows * ((p.n + cols - 1) / cols); }

// The grid for tiles of `rows` x `cols`, or 0 with the error recorded: 256 threads to a tile, of which a launch has less than 2^32.
unsigned grid_for(MxArgs &p, unsigned rows, unsigned cols) {
  if (tiles_of(p, rows, cols) >= 1u << 24) {
    skl_hip_record_error(SKL_HIP_ERR_BAD_ARGUMENT, "gemm_mx: grid too large");
    return 0;
  }
  p.tiles_m = (p.m + rows - 1) / rows, p.tiles_n = (p.n + cols - 1) / cols;
  return p.tiles_m * p.tiles_n;
}

template <int TM, int TN>
int launch_wide(MxArgs p) {
  static std::atomic<bool> done{false};
  const int rc = configure(reinterpret_cast<const void *>(gemm_mx_wide_kernel<TM, TN>), Wide<TM, TN>::kLds, done);
  if (rc != 0) return rc;
  const unsigned grid = grid_for(p, Wide<TM, TN>::kRows, Wide<TM, TN>::kCols);
  if (grid == 0) return SKL_HIP_ERR_BAD_ARGUMENT;
  gemm_mx_wide_kernel<TM, TN><<<grid, 256, Wide<TM, TN>::kLds, skl_current_stream()>>>(p);
  return skl_check_launch("gemm_mx_wide");
}

constexpr int kSmallStages = 2 * (64 + 64) * (kLine + 8), kSmallRows = 4 * kRowSpace<1>, kSmallLds = kSmallStages > kSmallRows ? kSmallStages : kSmallRows;

// Shares of K of `tiles` small tiles: two workgroups per compute unit, each with two chunks at least.
unsigned shares_for(size_t tiles, size_t k) {
  const size_t chunks = (k + kChunkK - 1) / kChunkK, want = 512 / tiles, most = chunks / 2 < 16 ? chunks / 2 : 16;
  return (unsigned)(want < 1 || most < 1 ? 1 : want < most ? want : most);
}

int launch_small(MxArgs p) {
  const unsigned grid = grid_for(p, 64, 64);
  if (grid == 0) return SKL_HIP_ERR_BAD_ARGUMENT;
  const unsigned shares = shares_for(grid, p.k);
  if (shares > 1) {
    const int pending = skl_hip_pending_error();
    skl_hip_sequence_begin();
    p.shares = static_cast<unsigned long long *>(skl_hip_operand_scratch((size_t)grid * shares * 8 * 256 * 8));
    p.counters = p.shares ? static_cast<unsigned *>(skl_hip_zeroed_sums(grid * sizeof(unsigned))) : nullptr;
    if (p.counters) {
      gemm_mx_stream_kernel<<<dim3(grid, shares), 256, kSmallLds, skl_current_stream()>>>(p);
      skl_hip_sequence_end();
      return skl_check_launch("gemm_mx");
    }
    skl_hip_sequence_end();
    // no scratch memory: one workgroup takes all of K
    if (pending != SKL_HIP_ERR_STREAM_SLOTS) skl_hip_withdraw_error(SKL_HIP_ERR_STREAM_SLOTS);
    if (pending != SKL_HIP_ERR_WORKSPACE) skl_hip_withdraw_error(SKL_HIP_ERR_WORKSPACE);
  }
  gemm_mx_stream_kernel<<<grid, 256, kSmallLds, skl_current_stream()>>>(p);
  return skl_check_launch("gemm_mx");
}

// Any layout, through registers: what has no scratch memory for copies, and K = 0.
int launch_any(MxArgs p) {
  const unsigned grid = grid_for(p, 64, 64);
  if (grid == 0) return SKL_HIP_ERR_BAD_ARGUMENT;
  gemm_mx_kernel<<<grid, 256, kSmallLds, skl_current_stream()>>>(p);
  return skl_check_launch("gemm_mx_any");
}

template <int RG, int CG>
int launch_rows_as(const MxArgs &p) {
  using Shape = RowsShape<RG, CG>;
  static std::atomic<bool> done{false};
  const int rc = configure(reinterpret_cast<const void *>(gemm_mx_rows_kernel<RG, CG>), Shape::kRingBytes + kRowsScaleSpace, done);
  if (rc != 0) return rc;
  gemm_mx_rows_kernel<RG, CG><<<(p.n + 16 * CG - 1) / (16 * CG), Shape::kWaves * 64, Shape::kRingBytes + rows_scale_bytes(RG, CG, p.k), skl_current_stream()>>>(p);
  return skl_check_launch("gemm_mx_rows");
}

int row_groups(const MxArgs &p) { return p.m <= 16 ? 1 : p.m <= 32 ? 2 : 4; }

int launch_rows(const MxArgs &p) {
  const int cg = skl_kcstream::column_groups(p.n), rg = row_groups(p);
#define SKL_MX_ROWS(RG, CG) \
  if (rg == RG && cg == CG) return launch_rows_as<RG, CG>(p);
  SKL_MX_ROWS(1, 1) SKL_MX_ROWS(1, 2) SKL_MX_ROWS(1, 3) SKL_MX_ROWS(1, 4)
  SKL_MX_ROWS(2, 1) SKL_MX_ROWS(2, 2) SKL_MX_ROWS(2, 3) SKL_MX_ROWS(2, 4)
  SKL_MX_ROWS(4, 1) SKL_MX_ROWS(4, 2) SKL_MX_ROWS(4, 3) SKL_MX_ROWS(4, 4)
#undef SKL_MX_ROWS
  return SKL_HIP_ERR_BAD_ARGUMENT;
}

// Which kernel, by what each takes (us, for the sizes m x n x k):
//   up to 64 rows whose scales find room next to the ring go to the stream over B (16 x 11008 x 4096 7.6, small tiles that share K 12.9; 64 x 4096 x 4096 9.2 / 12.0);
//   256 x 256 tiles where there are 200 and K is long enough for their epilogue, which nothing covers (8192 x 8192 x 4096 186, 128 x 128 tiles 193, x 1024 108 / 84;
//   4096 x 4096 x 8192 72 / 80, x 2048 31.6 / 31.7; 3000 x 5000 x 7000, behind the copies, 67 / 70);
//   128 x 128 tiles where there is one per compute unit and K is not short (2048 x 4096 x 4096 25.8, 64 x 64 tiles 42, x 256 14 / 10; 2048 x 2048 x 8192 31 / 42;
//   1024 x 1024 x 4096, 64 of them, 16.9 / 11.2);
//   else 64 x 64 tiles.
// The figures are for whole rounds of tiles, one 256 x 256 or two 128 x 128 tiles to a compute unit, or for less than one round; between 257 and some 400 large tiles, whose second round
// is mostly empty, neither side was measured.
enum Kind { kWide4, kWide2, kRows, kSmall };
Kind kind_of(const MxArgs &p) {
  if (p.m <= 64 && p.k >= 256 && rows_scale_bytes(row_groups(p), skl_kcstream::column_groups(p.n), p.k) <= (size_t)kRowsScaleSpace) return kRows;
  if (p.k <= ((size_t)1 << 23)) {  // a large tile's offsets from its first row are 31-bit numbers, 255 rows of half a byte per value
    if (tiles_of(p, 256, 256) >= 200 && p.k >= 2560) return kWide4;
    if (tiles_of(p, 128, 128) >= 256 && p.k >= 1024) return kWide2;
  }
  return kSmall;
}

int launch_kind(const MxArgs &p, Kind kind) {
  switch (kind) {
    case kWide4: return launch_wide<4, 4>(p);
    case kWide2: return launch_wide<2, 2>(p);
    case kRows: return p.k % 32 == 0 ? launch_rows(p) : launch_small(p);  // (no last block that is not whole)
    default: return launch_small(p);
  }
}

int launch_slab(const skl_mx_gemm *g) {
  MxArgs p = {g->a.codes, g->b.codes, g->a.ld / 2, g->b.ld / 2, g->a.scales, g->b.scales, g->a.lds, g->b.lds, g->c, g->rsc, g->csc,
              (unsigned)g->m, (unsigned)g->n, g->k, g->alpha, g->beta, 0, 0, 0, nullptr, nullptr};
  // C through the caches or past them (us): 8192 x 8192 x 8192 314 / 292, x 256 106 / 103; 4096 x 8192 x 4096 109.6 / 112.7, x 256 40.6 / 49.8.
  p.past_caches = g->m * g->n >= ((size_t)48 << 20);
  if (p.k == 0 || p.k > ((size_t)1 << 26)) return launch_any(p);
  const Kind kind = kind_of(p);
  // Operands in rows that the kernel does not read are copied first; for large tiles also those whose rows do not begin on lines, as every request of theirs takes a line
  // more (us with and without the copy: 3000 x 5000 x 7000 81 / 88, 2048 x 4096 x 4112 38 / 41, 2048 x 2048 x 3000 26 / 26, 8192 x 8192 x 3000 176 / 210).
  const unsigned exist = (unsigned)((p.k + 1) / 2), blocks = (unsigned)((p.k + 31) / 32), mask = p.k % 2 ? 15u : 255u;
  PadJobs jobs = {};
  const uint8_t **first[4] = {&p.a, &p.b, &p.sa, &p.sb};
  size_t *pitch[4] = {&p.a_row, &p.b_col, &p.sa_row, &p.sb_col}, bytes = 0, most = 0;
  for (int i = 0; i < 4; ++i) {
    if (i < 2 ? (kind <= kWide2 ? on_lines(*first[i], *pitch[i]) : rows_ok(*first[i], *pitch[i])) : kind > kWide2 || scales_ok(*first[i], *pitch[i], p.k)) continue;
    const unsigned row = i < 2 ? (unsigned)up(blocks * 16, kLine) : (unsigned)up(blocks, 16);
    unsigned lanes_log = 0;
    while (lanes_log < 8 && (16u << lanes_log) < row) ++lanes_log;
    jobs.job[i] = {*first[i], nullptr, *pitch[i], i % 2 ? p.n : p.m, row / 16, lanes_log, i < 2 ? exist : blocks, i < 2 ? mask : 255u, i < 2 ? 0u : 127u};
    bytes += up(jobs.job[i].rows * row, 256);
    const size_t grid = (jobs.job[i].rows << lanes_log) / (256 * kPadRows) + 1;
    most = grid > most ? grid : most;
  }
  if (bytes == 0) return launch_kind(p, kind);
  // With a short K the kernel that reads anything is done before a copy would be (us, copied and not: 700 x 700 x 700 9.5 / 6.1, 100 x 300 x 2001 11.5 / 9.6, 1500 x 1500 x 1500
  // 14.9 / 14.0, 50 x 3000 x 301 9.5 / 4.9, 1 x 4096 x 1001 8.5 / 5.7; 1500 x 1500 x 2998 22.0 / 25.9, 100 x 300 x 5001 14.2 / 19.2).
  if (kind >= kRows && p.k <= 2048) return launch_any(p);
  const int pending = skl_hip_pending_error();
  skl_hip_sequence_begin();
  uint8_t *block = static_cast<uint8_t *>(skl_hip_converted_scratch(bytes));  // (apart from the block that a product's shares of K take)
  int rc;
  if (block) {
    for (int i = 0; i < 4; ++i)
      if (PadJob &j = jobs.job[i]; j.rows != 0) {
        j.to = block;
        *first[i] = block, *pitch[i] = 16 * (size_t)j.words;
        block += up(j.rows * j.words * 16, 256);
      }
    if (jobs.job[0].rows != 0 && jobs.job[1].rows != 0) p.k = (size_t)blocks * 32;  // both filled up with zeros
    mx_pad_kernel<<<dim3((unsigned)(most < 4096 ? most : 4096), 4), 256, 0, skl_current_stream()>>>(jobs);
    rc = skl_check_launch("mx_pad");
    if (rc == 0) rc = launch_kind(p, kind);
  } else {
    if (pending != SKL_HIP_ERR_STREAM_SLOTS) skl_hip_withdraw_error(SKL_HIP_ERR_STREAM_SLOTS);
    if (pending != SKL_HIP_ERR_WORKSPACE) skl_hip_withdraw_error(SKL_HIP_ERR_WORKSPACE);
    rc = launch_any(p);
  }
  skl_hip_sequence_end();
  return rc;
}

}  // namespace

// In slabs of 2^28 rows and columns, so that the tiles fit a launch also where they are mostly empty (one column, or one row).
extern "C" int skl_hip_launch_gemm_mx(const skl_mx_gemm *g) {
  constexpr size_t kMost = (size_t)1 << 28;
  for (size_t i = 0; i < g->m; i += kMost)
    for (size_t j = 0; j < g->n; j += kMost) {
      skl_mx_gemm slab = *g;
      slab.m = g->m - i < kMost ? g->m - i : kMost, slab.n = g->n - j < kMost ? g->n - j : kMost;
      if (g->k != 0) {
        slab.a.codes += i * (g->a.ld / 2), slab.a.scales += i * g->a.lds;
        slab.b.codes += j * (g->b.ld / 2), slab.b.scales += j * g->b.lds;
      }
      slab.c += i * g->rsc + j * g->csc;
      const int rc = launch_slab(&slab);
      if (rc != 0) return rc;
    }
  return 0;
}
