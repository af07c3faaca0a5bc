// skl_gemm_u4.hip - products with integer 4-bit weights that have scales for groups along k (include/skl-gfx950.h: skl_gfx950_u4_t).
//
// v_mfma_f32_16x16x32 of 16 rows of A and 16 columns of weights: lane l holds eight k of row (column) l % 16 and, of the sums, rows 4 (l / 16) .. + 3 of
// column l % 16, so that a column's scale is one value of its lanes. A product is a * (q - z), exact: q - z is made in registers as bf16 or f16. The sums of
// at most 128 k of one group are scaled and added to the result in fp32.
#include <hip/hip_runtime.h>

#include <atomic>

#include "skl_groups.hpp"
#include "../../include/skl-hip.h"

namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));

struct U4Args {
  const uint16_t *a;
  size_t rsa;
  const int32_t *offsets, *rows;
  unsigned groups, m, n, k, a_rows, group_k;
  const uint8_t *codes;
  size_t ld, expert;
  const uint16_t *scales;
  const uint8_t *zeros;
  size_t ld_scales, expert_scales;
  void *c;
  size_t rsc;
  skl_scalar alpha, beta;
};

template <typename T>
__device__ __forceinline__ v4f product(v4i a, v4i b, v4f c);
template <>
__device__ __forceinline__ v4f product<__bf16>(v4i a, v4i b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0); }
template <>
__device__ __forceinline__ v4f product<_Float16>(v4i a, v4i b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0); }

template <typename T>
constexpr bool is_bf16 = __is_same(T, __bf16);

// Any layout: a wave takes 16 columns, 16 rows at a time, 32 of k per instruction, value by value.
template <typename T, typename TC>
__global__ void __launch_bounds__(256) gemm_u4_any_kernel(U4Args p) {
  typedef T Frag __attribute__((ext_vector_type(8)));
  const unsigned lane = threadIdx.x & 63u, l = lane & 15u, part = lane >> 4, e = blockIdx.y;
  const unsigned col0 = (blockIdx.x * 4 + (threadIdx.x >> 6)) * 16;
  if (col0 >= p.n) return;
  const SklRange r = skl_group_range(p.offsets, e, p.m);
  const unsigned col = col0 + l < p.n ? col0 + l : p.n - 1;
  const size_t first_code = (size_t)e * p.expert + (size_t)col * p.ld, first_scale = (size_t)e * p.expert_scales + (size_t)col * p.ld_scales;
  const bool read_c = !skl_beta_is_zero<float>(p.beta);
  for (unsigned row0 = 0; row0 < r.rows; row0 += 16) {
    unsigned row = row0 + l < r.rows ? r.first + row0 + l : r.first;
    bool there = row0 + l < r.rows;
    if (p.rows) {
      row = (unsigned)p.rows[row];
      there = there && row < p.a_rows;
    }
    const uint16_t *const a = p.a + (size_t)(there ? row : 0u) * p.rsa;
    v4f sum = {0, 0, 0, 0}, part_sum = {0, 0, 0, 0};
    for (unsigned k0 = 0, block = 0, end = p.group_k; k0 < p.k; k0 += 32) {  // end: of the group that all 32 are in
      Frag x, w;
      const int zero = p.zeros ? (int)p.zeros[first_scale + block] : 8;
      const float scale = skl_widen(p.scales[first_scale + block], is_bf16<T>);
#pragma unroll
      for (unsigned i = 0; i < 8; ++i) {
        const unsigned at = k0 + 8 * part + i;
        const bool in = at < p.k;
        const uint16_t v = in && there ? a[at] : (uint16_t)0;
        x[i] = __builtin_bit_cast(T, v);
        const unsigned byte = in ? p.codes[(first_code + at) / 2] : 0u;
        w[i] = (T)(float)(in ? (int)((at & 1) ? byte >> 4 : byte & 15u) - zero : 0);
      }
      part_sum = product<T>(__builtin_bit_cast(v4i, x), __builtin_bit_cast(v4i, w), part_sum);
      if (k0 + 32 < p.k && (k0 + 32) % 128 != 0 && k0 + 32 != end) continue;  // a scale meets what it meets in the stream below
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[i] = __builtin_fmaf(part_sum[i], scale, sum[i]), part_sum[i] = 0.0f;
      if (k0 + 32 == end) ++block, end += p.group_k;
    }
    if (col0 + l >= p.n) continue;
    TC *const c = reinterpret_cast<TC *>(p.c) + (size_t)r.first * p.rsc + col;
#pragma unroll
    for (unsigned i = 0; i < 4; ++i) {
      const unsigned at = row0 + 4 * part + i;
      if (at >= r.rows) continue;
      TC *const to = c + (size_t)at * p.rsc;
      const bool outside = p.rows && (unsigned)p.rows[r.first + at] >= p.a_rows;  // no scale meets its zeros: 0, if it is infinite, too
      *to = skl_grouped_result(outside ? 0.0f : sum[i], to, p.alpha, p.beta, read_c);
    }
  }
}

// ---------------------------------------------------------------------------
// The stream over the codes: rows of codes and of A on 16-byte boundaries, k a multiple of 32, group_k 32, 64 or a multiple of 128 (one group of all k
// among them).
// A workgroup of four or eight waves takes 16 F columns and all of k, in chunks: a wave UNITS units of 128 k of each, half a line of each column's codes, which go
// to registers a chunk ahead. ROWS rows of A and the columns' scales go to LDS, where all waves read them; in the end the waves' sums meet there.
// ---------------------------------------------------------------------------

// Eight values q - z of a column, exact.
template <typename T>
struct Zero;
template <>
struct Zero<__bf16> {
  float z;  // -(1024 + zero point)
  __device__ __forceinline__ explicit Zero(unsigned v) : z(-1024.0f - (float)v) {}
};
template <>
struct Zero<_Float16> {
  v2h z;
  __device__ __forceinline__ explicit Zero(unsigned v) : z(__builtin_bit_cast(v2h, (0x6400u + v) * 0x10001u)) {}  // 1024 + v, twice (v < 1024)
};
// The nibbles as they lie are pairs k0 k4, k1 k5, k2 k6, k3 k7; A is put into that order on its way to LDS (arranged()). 0x6400 | q is the f16 number 1024 + q.
// (An instruction takes one scalar besides, and no literal.)
__device__ __forceinline__ unsigned pair_of(unsigned codes, int i) {
  unsigned two;
  asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(two) : "v"(codes >> (4 * i)), "s"(0x000F000Fu), "v"(0x64006400u));
  return two;
}
__device__ __forceinline__ v4i widened(unsigned codes, Zero<__bf16> z) {
  v4i w;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // The f16 halves as factors of fp32 multiply-adds: 1024 + q - (1024 + z). (By v_cvt_f32_ubyte and a subtraction 23 instructions for eight values, so 19.)
    const unsigned two = pair_of(codes, i);
    float low, high;
    asm("v_fma_mix_f32 %0, %1, 1.0, %2 op_sel_hi:[1,0,0]" : "=v"(low) : "v"(two), "v"(z.z));
    asm("v_fma_mix_f32 %0, %1, 1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(high) : "v"(two), "v"(z.z));
    typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
    w[i] = __builtin_bit_cast(int, v2bf{(__bf16)low, (__bf16)high});
  }
  return w;
}
__device__ __forceinline__ v4i widened(unsigned codes, Zero<_Float16> z) {
  v4i w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = __builtin_bit_cast(int, __builtin_bit_cast(v2h, pair_of(codes, i)) - z.z);
  return w;
}
// k0 .. k7 as k0 k4 k1 k5 k2 k6 k3 k7.
__device__ __forceinline__ v4i arranged(v4i a) {
  v4i r;
  r[0] = (int)__builtin_amdgcn_perm((unsigned)a[2], (unsigned)a[0], 0x05040100u);
  r[1] = (int)__builtin_amdgcn_perm((unsigned)a[2], (unsigned)a[0], 0x07060302u);
  r[2] = (int)__builtin_amdgcn_perm((unsigned)a[3], (unsigned)a[1], 0x05040100u);
  r[3] = (int)__builtin_amdgcn_perm((unsigned)a[3], (unsigned)a[1], 0x07060302u);
  return r;
}

// Dword i of the four quarters of a wave, transposed: quarter p's dword j becomes quarter j's dword p.
__device__ __forceinline__ v4i quarters_transposed(v4i v) {
  typedef unsigned v2u __attribute__((ext_vector_type(2)));
  const v2u a = __builtin_amdgcn_permlane32_swap((unsigned)v[0], (unsigned)v[2], false, false), b = __builtin_amdgcn_permlane32_swap((unsigned)v[1], (unsigned)v[3], false, false);
  const v2u c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false), d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
  return v4i{(int)c[0], (int)c[1], (int)d[0], (int)d[1]};
}

constexpr unsigned kUnit = 128;  // of k

// What a kernel holds. PER: groups of a unit, 4, 2 or 1; F: 16 columns each; ROWS: of A, staged in LDS for a chunk of UNITS units per wave.
template <int PER, bool ZEROS, int F, int ROWS, int UNITS, int WAVES>
struct U4Shape {
  static constexpr unsigned kWaves = WAVES, kThreads = kWaves * 64;
  static constexpr unsigned kR = (ROWS + 15) / 16, kCols = 16 * F, kChunk = kUnit * kWaves * UNITS;
  static constexpr unsigned kPitch = kChunk * 2 + 16;  // bytes of a row of A: 16 rows meet in no bank
  static constexpr unsigned kPieces = (ROWS * kChunk / 8 + kThreads - 1) / kThreads, kRowPieces = kChunk / 8;
  static constexpr unsigned kEntries = kChunk / kUnit * PER, kEach = (kCols * kEntries + kThreads - 1) / kThreads;  // scales of a column and chunk, of a thread
  static constexpr unsigned kBytesA = ROWS * kPitch, kStage = (kBytesA + (kEntries + 1) * kCols * 4 + 15) / 16 * 16;
  static constexpr unsigned kSums = kWaves * 16 * kR * (kCols + 1) * 4, kLds = 2 * kStage > kSums ? 2 * kStage : kSums;
  static_assert(kLds <= 160 * 1024);
  struct Side {  // what goes to LDS, on its way
    v4i a[kPieces];
    unsigned scale[kEach], zero[ZEROS ? kEach : 1];
  };
};

template <typename T, int PER, bool ZEROS, int F, int ROWS, int UNITS, int MIN, int WAVES>
__global__ void __launch_bounds__(WAVES * 64, MIN) gemm_u4_stream_kernel(U4Args p, int c_single) {
  using Shape = U4Shape<PER, ZEROS, F, ROWS, UNITS, WAVES>;
  constexpr unsigned kWaves = Shape::kWaves, kThreads = Shape::kThreads;
  constexpr bool kFine = PER > 1;       // groups smaller than the 128 k whose codes the quarters of a wave hold side by side
  constexpr unsigned kCols = Shape::kCols, kChunk = Shape::kChunk, kEntries = Shape::kEntries, kEach = Shape::kEach, kPitch = Shape::kPitch, kPieces = Shape::kPieces, kRowPieces = Shape::kRowPieces;
  constexpr int R = Shape::kR;
  extern __shared__ __attribute__((aligned(16))) char u4_lds_bytes[];
  const unsigned wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63u, l = lane & 15u, part = lane >> 4, e = blockIdx.y;
  const SklRange range = skl_group_range(p.offsets, e, p.m);
  if (range.rows == 0) return;
  const unsigned col0 = blockIdx.x * kCols, cols = p.n - col0 < kCols ? p.n - col0 : kCols;
  const unsigned last_group = p.k ? (p.k - 1) / p.group_k : 0, units_per_group = PER == 1 ? p.group_k / kUnit : 1;
  const uint8_t *const codes = p.codes + ((size_t)e * p.expert + (size_t)col0 * p.ld) / 2;
  unsigned code_at[F];
#pragma unroll
  for (int f = 0; f < F; ++f) code_at[f] = (16 * f + l < cols ? 16 * f + l : cols - 1) * (unsigned)(p.ld / 2);  // (ld below 2^25, see the launch)
  const size_t scale_base = (size_t)e * p.expert_scales + (size_t)col0 * p.ld_scales;
  const bool read_c = !skl_beta_is_zero<float>(p.beta);
  const unsigned limit = p.rows ? p.a_rows : p.m, chunks = (p.k + kChunk - 1) / kChunk;

  struct Codes {
    v4i v[F];
  };
  for (unsigned row0 = 0; row0 < range.rows; row0 += ROWS) {
    // Rows that do not exist are the group's first again, those that an index puts outside A its first: computed, and written nowhere or as zeros.
    const uint16_t *a[kPieces];
#pragma unroll
    for (int i = 0; i < (int)kPieces; ++i) {
      const unsigned r = row0 + (threadIdx.x + i * kThreads) / kRowPieces;
      unsigned row = range.first + (r < range.rows ? r : 0u);
      if (p.rows) row = (unsigned)p.rows[row];
      a[i] = p.a + (size_t)(row < limit ? row : 0u) * p.rsa;
    }
    // (Without branches, at whose ends what is under way would be waited for: behind k lies what lies at its end again, with zeros for A. And the offsets anew for
    // every chunk, from a number that the compiler cannot follow: it otherwise keeps all of them.)
    const auto request_codes = [&](Codes &to, unsigned c, unsigned j) __attribute__((always_inline)) {
      asm volatile("" : "+s"(c));
      const unsigned piece = ((c * UNITS + j) * kWaves + wave) * (kUnit / 2) + 16 * part, most = p.k / 2 - 16;
#pragma unroll
      for (int f = 0; f < F; ++f) to.v[f] = __builtin_nontemporal_load(reinterpret_cast<const v4i *>(codes + (code_at[f] + (piece < most ? piece : most))));
    };
    const auto request_side = [&](typename Shape::Side &to, unsigned c) __attribute__((always_inline)) {
      asm volatile("" : "+s"(c));
#pragma unroll
      for (int i = 0; i < (int)kPieces; ++i) {
        const unsigned k = c * kChunk + (threadIdx.x + i * kThreads) % kRowPieces * 8;
        to.a[i] = *reinterpret_cast<const v4i *>(a[i] + (k < p.k ? k : p.k - 8));
      }
#pragma unroll
      for (int i = 0; i < (int)kEach; ++i) {
        const unsigned at = threadIdx.x + i * kThreads, col = at / kEntries % kCols, entry = at % kEntries + c * kEntries;
        unsigned group = PER == 1 ? entry / units_per_group : entry;
        group = (col < cols ? col : cols - 1) * (unsigned)p.ld_scales + (group < last_group ? group : last_group);
        to.scale[i] = (p.scales + scale_base)[group];
        if constexpr (ZEROS) to.zero[i] = (p.zeros + scale_base)[group];
      }
    };
    const auto stage = [&](const typename Shape::Side &from, unsigned c) __attribute__((always_inline)) {
      char *const to = u4_lds_bytes + (c & 1) * Shape::kStage;
#pragma unroll
      for (int i = 0; i < (int)kPieces; ++i) {
        const unsigned at = threadIdx.x + i * kThreads;
        if (ROWS * kRowPieces % kThreads == 0 || at < ROWS * kRowPieces) *reinterpret_cast<v4i *>(to + at / kRowPieces * kPitch + at % kRowPieces * 16) = c * kChunk + at % kRowPieces * 8 < p.k ? arranged(from.a[i]) : v4i{0, 0, 0, 0};
      }
#pragma unroll
      for (int i = 0; i < (int)kEach; ++i) {  // [column][entry]: a scale with its zero point above
        const unsigned at = threadIdx.x + i * kThreads;
        if (kCols * kEntries % kThreads == 0 || at < kCols * kEntries) reinterpret_cast<unsigned *>(to + Shape::kBytesA)[at / kEntries * (kEntries + 1) + at % kEntries] =
            (kFine && at % kEntries + c * kEntries > last_group ? 0u : from.scale[i]) | (ZEROS ? from.zero[ZEROS ? i : 0] : 8u) << 16;  // (behind k no scale that is infinite, for sums that are zero)
      }
    };
    v4f sum[R][F];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int f = 0; f < F; ++f) sum[r][f] = v4f{0, 0, 0, 0};
    const auto multiply = [&](const Codes &b, unsigned c, unsigned j) __attribute__((always_inline)) {
      const char *const tile = u4_lds_bytes + (c & 1) * Shape::kStage;
      const unsigned unit = j * kWaves + wave;
      const unsigned *const entry = reinterpret_cast<const unsigned *>(tile + Shape::kBytesA) + l * (kEntries + 1) + unit * PER;
      constexpr int kOf = 4 / PER;  // instructions of a group in a unit
      v4i code[F];
      v4f acc[R][F];
#pragma unroll
      for (int f = 0; f < F; ++f) code[f] = kFine ? quarters_transposed(b.v[f]) : b.v[f];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v4i x[R];
#pragma unroll
        for (int r = 0; r < R; ++r) x[r] = *reinterpret_cast<const v4i *>(tile + ((16 * r + l) % ROWS) * kPitch + (unit * kUnit + (kFine ? 32u * i + 8 * part : 32 * part + 8u * i)) * 2);
#pragma unroll
        for (int f = 0; f < F; ++f) {
          const v4i w = widened((unsigned)code[f][i], Zero<T>(entry[16 * f * (kEntries + 1) + i / kOf] >> 16));
#pragma unroll
          for (int r = 0; r < R; ++r) acc[r][f] = product<T>(x[r], w, i % kOf == 0 ? v4f{0, 0, 0, 0} : acc[r][f]);
        }
        if ((i + 1) % kOf == 0) {
#pragma unroll
          for (int f = 0; f < F; ++f) {
            const float by = skl_widen((uint16_t)entry[16 * f * (kEntries + 1) + i / kOf], is_bf16<T>);
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
              for (int q = 0; q < 4; ++q) sum[r][f][q] = __builtin_fmaf(acc[r][f][q], by, sum[r][f][q]);
          }
        }
      }
    };
    if (row0) __syncthreads();  // the sums of the pass before have been read
    if (chunks != 0) {
      Codes held[UNITS];
      typename Shape::Side side;
      request_side(side, 0);
#pragma unroll
      for (int j = 0; j < UNITS; ++j) request_codes(held[j], 0, j);
      stage(side, 0);
      for (unsigned c = 0; c < chunks; ++c) {
        __syncthreads();  // chunk c is staged; nobody reads chunk c - 1 any more
        request_side(side, c + 1);
#pragma unroll
        for (int j = 0; j < UNITS; ++j) {
          __builtin_amdgcn_sched_barrier(0);
          if (c * kChunk + (j * kWaves + wave) * kUnit < p.k) multiply(held[j], c, j);
          __builtin_amdgcn_sched_barrier(0);
          request_codes(held[j], c + 1, j);
        }
        stage(side, c + 1);
      }
    }
    __syncthreads();
    float(*const sums)[16 * R][kCols + 1] = reinterpret_cast<float(*)[16 * R][kCols + 1]>(u4_lds_bytes);
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int f = 0; f < F; ++f)
#pragma unroll
        for (int q = 0; q < 4; ++q) sums[wave][16 * r + 4 * part + q][16 * f + l] = sum[r][f][q];
    __syncthreads();
    for (unsigned i = threadIdx.x; i < ROWS * kCols; i += kThreads) {
      const unsigned row = i / kCols, c = i % kCols;
      if (row0 + row >= range.rows || c >= cols) continue;
      float v = 0.0f;
#pragma unroll
      for (unsigned w = 0; w < kWaves; ++w) v = __fadd_rn(v, sums[w][row][c]);
      const unsigned out = range.first + row0 + row;
      if (p.rows && (unsigned)p.rows[out] >= limit) v = 0.0f;  // what was computed is A's first row's
      const size_t at = (size_t)out * p.rsc + col0 + c;
      if (c_single) {
        float *const to = reinterpret_cast<float *>(p.c) + at;
        *to = skl_grouped_result(v, to, p.alpha, p.beta, read_c);
      } else {
        T *const to = reinterpret_cast<T *>(p.c) + at;
        *to = skl_grouped_result(v, to, p.alpha, p.beta, read_c);
      }
    }
  }
}

template <typename T, int PER, bool ZEROS, int F, int ROWS, int UNITS, int MIN, int WAVES>
int launch_stream(const U4Args &p, int c_single) {
  constexpr unsigned kLds = U4Shape<PER, ZEROS, F, ROWS, UNITS, WAVES>::kLds;
  const auto kernel = gemm_u4_stream_kernel<T, PER, ZEROS, F, ROWS, UNITS, MIN, WAVES>;
  static std::atomic<unsigned long long> allowed{0};
  const int rc = skl_allow_lds(reinterpret_cast<const void *>(kernel), kLds, allowed);
  if (rc != 0) return rc;
  kernel<<<dim3(skl_div_up(p.n, 16 * F), p.groups), dim3(WAVES * 64), kLds, skl_current_stream()>>>(p, c_single);
  return skl_check_launch("gemm_u4");
}

template <typename T, int PER, bool ZEROS>
int stream_by_size(const U4Args &p, int c_single) {
  // By the rows there are for a matrix, on average where there are several: rows beyond a pass read the codes again, and what a pass has room for is computed. us, 4 / 16 / 32 rows a pass: one
  // row 9.8 (1 row) / 10.5 (4) for 4096 x 11008; 32 matrices of 2048 x 2816 with 32 rows 23.6 / 24.9 / -, 128 rows 47.9 / 34.4 / -, 256 rows 61 / 36.3 / 54.4.
  // And by the workgroups there are, each with all of k: eight waves for a column's k where they hardly fill the chip, four where more workgroups, of half the LDS, then overlap. us,
  // eight / four: one row 4096 x 11008 9.9 / 9.5, 11008 x 4096 9.5 / 12.3, 4096 x 28672 19.4 / 17.1; 48 rows for 64 of 4096 x 1408 35.4 / 27.7; 16 rows 8192 x 8192 14.8 / 20.4, 256 rows
  // for 32 of 2048 x 2816 44.5 / 36.3, 128 rows for 8 of 4096 x 4096 39.1 / 38.6; 64 rows 4096 x 11008 40.8 / 36.4, 8192 x 8192 37.4 / 46.0.
  // Fewer columns and shorter chunks a workgroup, more workgroups: F = 2 rather than 1 costs one row 4096 x 11008 1.2 us, twice the chunk 0.1 to 1.7; with 16 rows, whose operands are read for
  // all columns, F = 2 is the faster one (16 x 8192 x 8192 14.9, F = 1 17.4).
  const size_t m = p.m, groups = p.groups, runs = (size_t)skl_div_up(p.n, 16) * groups;
  if (m == 1) return runs >= 640 ? launch_stream<T, PER, ZEROS, 1, 1, 2, 4, 4>(p, c_single) : launch_stream<T, PER, ZEROS, 1, 1, 2, 6, 8>(p, c_single);
  if (m <= 4 || m <= 2 * groups) return runs >= 512 ? launch_stream<T, PER, ZEROS, 1, 4, 2, 4, 4>(p, c_single) : launch_stream<T, PER, ZEROS, 1, 4, 1, 6, 8>(p, c_single);
  if (m <= 16 * groups) return runs >= 4096 ? launch_stream<T, PER, ZEROS, 2, 16, 1, 2, 4>(p, c_single) : launch_stream<T, PER, ZEROS, 2, 16, 1, 4, 8>(p, c_single);
  return runs >= 640 ? launch_stream<T, PER, ZEROS, 2, 32, 1, 2, 4>(p, c_single) : launch_stream<T, PER, ZEROS, 2, 32, 1, 2, 8>(p, c_single);
}

template <typename T>
int launch(U4Args p, int c_single) {
  const auto aligned = [](const void *at) { return ((uintptr_t)at & 15) == 0; };
  const bool one = p.group_k >= p.k;
  if (p.k % 32 == 0 && aligned(p.a) && aligned(p.codes) && p.rsa % 8 == 0 && p.ld < (size_t(1) << 25) && p.ld_scales < (size_t(1) << 24) && p.ld % 32 == 0 && p.expert % 32 == 0 &&
      (one || p.group_k == 32 || p.group_k == 64 || p.group_k % 128 == 0)) {
    if (one || p.group_k % 128 == 0) {
      if (one) p.group_k = (p.k + kUnit - 1) / kUnit * kUnit;
      return p.zeros ? stream_by_size<T, 1, true>(p, c_single) : stream_by_size<T, 1, false>(p, c_single);
    }
    if (p.group_k == 32) return p.zeros ? stream_by_size<T, 4, true>(p, c_single) : stream_by_size<T, 4, false>(p, c_single);
    return p.zeros ? stream_by_size<T, 2, true>(p, c_single) : stream_by_size<T, 2, false>(p, c_single);
  }
  const dim3 grid(skl_div_up(p.n, 64), p.groups);
  if (c_single) gemm_u4_any_kernel<T, float><<<grid, dim3(256), 0, skl_current_stream()>>>(p);
  else gemm_u4_any_kernel<T, T><<<grid, dim3(256), 0, skl_current_stream()>>>(p);
  return skl_check_launch("gemm_u4");
}

}  // namespace

int skl_hip_launch_gemm_u4(const skl_grouped_u4 *u) {
  const skl_grouped_gemm *g = &u->g;
  U4Args p{};
  p.a = (const uint16_t *)g->a, p.rsa = g->rsa, p.offsets = g->offsets, p.rows = g->rows;
  p.groups = (unsigned)g->groups, p.m = (unsigned)g->m, p.n = (unsigned)g->n, p.k = (unsigned)g->k, p.a_rows = (unsigned)g->a_rows, p.group_k = (unsigned)u->group_k;
  p.codes = u->codes, p.ld = u->ld, p.expert = g->groups > 1 ? u->expert : 0;
  p.scales = (const uint16_t *)u->scales, p.zeros = u->zeros, p.ld_scales = u->ld_scales, p.expert_scales = g->groups > 1 ? u->expert_scales : 0;
  p.c = g->c, p.rsc = g->rsc, p.alpha = g->alpha, p.beta = g->beta;
  // Columns of a launch: beyond 2^32 threads the runtime takes what is left of the number in 32 bits.
  const size_t slab = size_t(1) << 26;
  for (size_t col = 0; col < g->n; col += slab) {
    p.n = (unsigned)(g->n - col < slab ? g->n - col : slab);
    p.codes = u->codes + col * (u->ld / 2);
    p.scales = (const uint16_t *)u->scales + col * u->ld_scales;
    p.zeros = u->zeros ? u->zeros + col * u->ld_scales : nullptr;
    p.c = (char *)g->c + col * (g->c_single ? 4 : 2);
    const int rc = g->dt == SKL_DT_BF16 ? launch<__bf16>(p, g->c_single) : launch<_Float16>(p, g->c_single);
    if (rc != 0) return rc;
  }
  return 0;
}
