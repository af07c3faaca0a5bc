// skl_grouped_ring.hpp - the streaming kernel's way (skl_gemm_mfma_impl.hpp) with products grouped by expert: operands go from memory to LDS without registers, slices
// of 64 bytes of K in a ring of four to eight stages, the next slice's reads and a later one's requests dealt out behind the products of this one. What is different: which
// rows a tile has is known on the GPU alone, an operand's rows may come through an index, C has two types.
//
// A tile is 256, 128 or 64 rows by BN columns. What whole tiles of 256 rows leave of a group goes into the smallest tile that holds it: a group of
// 300 rows costs 256 + 64, not 512.
#pragma once

#include "skl_gemm_mfma_impl.hpp"
#include "skl_groups.hpp"
#include "../../include/skl-hip.h"

namespace {

// 64 values across K: eight chunks of a k-row of 128 bytes, two of which fill the banks. 32 lanes of a tr16 read take k-rows r .. r + 3 and r + 8 .. r + 11, two chunks of each: rows of one
// parity are parted by their second and fourth bits.
template <int NS>
struct STile<2, false, 64, NS, 16> {
  static constexpr int kStages = NS, kBytes = 64 * kRingSlice, kRegion = kBytes * NS, kRowBytes = 128, kStageStep = kBytes, kGroup = NS * 512;
  __device__ static __forceinline__ int chunk(int r, int c) { return r * 128 + ((c ^ ((r & 2) | (r >> 1 & 4))) << 4); }
};

struct GroupedRingArgs {
  const char *a, *b;
  const int32_t *offsets, *rows, *rows_b;  // rows: of A
  char *c;
  size_t a_pitch, b_pitch, b_group;  // bytes: from one line of an operand to the next - rows or columns with K side by side, or steps of K -, from one group's B to the next
  size_t rsc, gsc;                   // elements
  unsigned groups, m, n, k, a_rows, b_rows;  // OVER: k is the number of rows in all
  unsigned tiles_m, tiles_n;         // OVER: of a group
  unsigned parts;                    // OVER: a group's rows are shared out over so many; more than 1: C is each part's own
  int c_single;
  skl_scalar alpha, beta;
};

// Requests of one operand, this wave's share: lines of ROWS rows or columns with K side by side (KC), a pair of slices at a time, or lines of ROWS values across K, a slice at a time. All
// through a buffer descriptor; what does not exist has an offset beyond its range, for which zeros arrive and no memory is touched.
// INDEXED (not KC): the steps of K are rows through an index. A wave's part of a slice is a few rows, whose numbers come as scalars a step ahead of the requests.
template <bool KC, int ROWS, int WAVES, int NS, bool INDEXED>
struct GroupedLoader {
  using T = STile<2, KC, ROWS, NS, 16>;
  static constexpr unsigned kRange = 0xC0000000u, kOutside = 0xE0000000u;
  static constexpr int kBlocks = (KC ? 2 : 1) * T::kBytes / 1024 / WAVES;  // KiB per wave and unit
  static_assert(kBlocks >= 1);
  static constexpr unsigned kBlockStep = KC ? T::kGroup : 1024;
  static constexpr unsigned kUnitK = KC ? 2 * kRingSlice : kRingSlice / 2;  // bytes or steps of K
  static constexpr int kLanesPerRow = KC ? 1 : T::kRowBytes / 16, kRowsPerBlock = KC ? 1 : 1024 / T::kRowBytes, kRows = kBlocks * kRowsPerBlock;
  const char *base;
  size_t k_step;
  unsigned off[kBlocks], k_lane[KC ? 2 : kBlocks], k_total, lds;
  const __attribute__((address_space(4))) char *index;  // this wave's first row's; read by scalar loads
  unsigned index_left, index_limit, index_pitch;        // index_left: rows from there on less one
  typedef int Lines __attribute__((ext_vector_type(INDEXED ? kRows : 2)));
  Lines ahead, line;  // rows of the next step's unit; offsets of this step's (vectors: arrays in here are kept in memory)

  __device__ __forceinline__ static const char *scalar(const char *p) {
    const uintptr_t at = (uintptr_t)p;
    return (const char *)(((uintptr_t)(unsigned)__builtin_amdgcn_readfirstlane((int)(at >> 32)) << 32) | (unsigned)__builtin_amdgcn_readfirstlane((int)at));
  }
  // KC: lines first .. first + count - 1, through `index` where there is one (of `limit` lines); else columns at .. of `count` from there on, steps of K `pitch` apart.
  // k: bytes (KC) or steps.
  // INDEXED: step r is row index[index_at + r] of `limit`.
  __device__ __forceinline__ void init(const char *from, size_t pitch, const int32_t *index, unsigned index_at, unsigned limit, unsigned first, unsigned count, unsigned k) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    lds = wave * kBlocks * kBlockStep;
    k_total = k;
    if constexpr (KC) {
      base = scalar(index ? from : from + (size_t)first * pitch);
      k_step = 2 * kRingSlice;
#pragma unroll
      for (int i = 0; i < kBlocks; ++i) {
        const int row = 8 * (wave * kBlocks + i) + ((lane & 31) >> 2), c = (lane & 3) ^ T::turn(row);
        const unsigned in_k = (lane >> 5) * 64 + c * 16;
        if (i < 2) k_lane[i] = in_k;  // (the blocks' turns alternate)
        unsigned line = (unsigned)row < count ? (unsigned)row : ~0u;
        if (index && line != ~0u) {
          line = (unsigned)index[index_at + line];
          if (line >= limit) line = ~0u;
        }
        off[i] = line == ~0u ? kOutside : line * (unsigned)pitch + in_k;
      }
    } else {
      base = scalar(from + (size_t)first * 2);
      k_step = ((size_t)(unsigned)__builtin_amdgcn_readfirstlane((int)((pitch * kUnitK) >> 32)) << 32) | (unsigned)__builtin_amdgcn_readfirstlane((int)(pitch * kUnitK));
#pragma unroll
      for (int i = 0; i < kBlocks; ++i) {
        const int kr = kRowsPerBlock * (wave * kBlocks + i) + lane / kLanesPerRow, mn = ((T::chunk(kr, lane % kLanesPerRow) - kr * T::kRowBytes) >> 4) * 8;
        k_lane[i] = kr;
        off[i] = (unsigned)mn < count ? (INDEXED ? 0u : (unsigned)kr * (unsigned)pitch) + (unsigned)mn * 2 : kOutside;
      }
      if constexpr (INDEXED) {
        const unsigned mine = (unsigned)wave * kRows;
        this->index = (const __attribute__((address_space(4))) char *)(uintptr_t)scalar((const char *)(index + index_at + (mine < k ? mine : k - 1)));
        index_left = mine < k ? k - 1 - mine : 0, index_limit = limit, index_pitch = (unsigned)pitch;
        k_step = 0;
      }
    }
  }
  // The rows of the part of `unit` that is this wave's; beyond the last one that one again.
  __device__ __forceinline__ Lines look_up(unsigned unit) const {
    Lines rows = 0;
    if constexpr (INDEXED) {
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const unsigned at = unit * kUnitK + r;
        rows[r] = *(const __attribute__((address_space(4))) int32_t *)(index + (at < index_left ? at : index_left) * 4u);
      }
    }
    return rows;
  }
  __device__ __forceinline__ void take(Lines rows) {  // for the requests of a step
    if constexpr (INDEXED) {
#pragma unroll
      for (int r = 0; r < kRows; ++r) line[r] = (int)((unsigned)rows[r] < index_limit ? (unsigned)rows[r] * index_pitch : kOutside);
    }
  }
  __device__ __forceinline__ unsigned left_of(unsigned unit) const { return k_total > unit * kUnitK ? k_total - unit * kUnitK : 0; }
  __device__ __forceinline__ void request(char *region, int stage, unsigned unit, unsigned left, int i) const {
    unsigned o = k_lane[KC ? i & 1 : i] < left ? off[i] : kOutside;
    if constexpr (INDEXED) {
      const unsigned lane = threadIdx.x & 63u;
      unsigned of_line = (unsigned)line[i * kRowsPerBlock];
#pragma unroll
      for (int r = 1; r < kRowsPerBlock; ++r) of_line = lane >= (unsigned)(r * kLanesPerRow) ? (unsigned)line[i * kRowsPerBlock + r] : of_line;
      o = o == kOutside || of_line == kOutside ? kOutside : o + of_line;
    }
    asm volatile("" : "+v"(o));  // (not widened to 64 bits ahead of the loop, see SLoader)
    __builtin_amdgcn_raw_ptr_buffer_load_lds(__builtin_amdgcn_make_buffer_rsrc((void *)(base + unit * k_step), 0, (int)kRange, 0x00027000),
                                             (__attribute__((address_space(3))) void *)(region + stage * T::kStageStep + lds + i * kBlockStep), 16, (int)o, 0, 0, 0);
  }
};

// C of a wave: acc[i][j] holds, in lane l, four columns from 16 j + 4 (l / 16) on of row 16 i + l % 16. A row of blocks at a time goes through the wave's own 16 x (16 NI + 4) floats of LDS, from
// where rows leave in runs of 16 bytes a lane.
template <int MI, int NI>
constexpr unsigned grouped_space() { return 16 * (16 * NI + 4) * 4; }
template <typename TC, int MI, int NI>
__device__ __forceinline__ void grouped_write(TC *c, size_t rsc, const v4f (&acc)[MI][NI], unsigned row0, unsigned col0, unsigned rows, unsigned cols, skl_scalar alpha, skl_scalar beta, char *space) {
  constexpr int W = 16 * NI, P = W + 4, E = 16 / (int)sizeof(TC);  // a lane's columns
  constexpr int kLanes = W / E, kDown = 64 / kLanes < 16 ? 64 / kLanes : 16;
  typedef TC RunC __attribute__((ext_vector_type(E), aligned(sizeof(TC))));
  const unsigned lane = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
  const bool read_c = !skl_beta_is_zero<float>(beta);
  float *const stage = reinterpret_cast<float *>(space);
  const unsigned r_lane = lane / kLanes, col = col0 + lane % kLanes * E;
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < NI; ++j) *reinterpret_cast<v4f *>(stage + (lane & 15u) * P + 16 * j + 4 * (lane >> 4)) = acc[i][j];
#pragma unroll
    for (int d = 0; d < 16; d += kDown) {
      const unsigned r = d + r_lane, row = row0 + 16 * i + r;
      if (r >= 16 || row >= rows || col >= cols) continue;
      TC *const to = c + (size_t)row * rsc + col;
      float v[E];
#pragma unroll
      for (int q = 0; q < E; q += 4) *reinterpret_cast<v4f *>(v + q) = *reinterpret_cast<const v4f *>(stage + r * P + lane % kLanes * E + q);
      if (col + E <= cols) {
        RunC old, out;
        if (read_c) old = *reinterpret_cast<const RunC *>(to);
#pragma unroll
        for (int q = 0; q < E; ++q) out[q] = (TC)(read_c ? skl_combine(v[q], (float)old[q], alpha, beta) : skl_initialise_plain(v[q], alpha, beta));
        __builtin_nontemporal_store(out, reinterpret_cast<RunC *>(to));
      } else {
#pragma unroll
        for (int q = 0; q < E; ++q)
          if (col + q < cols) to[q] = skl_grouped_result(v[q], to + q, alpha, beta, read_c);
      }
    }
  }
}

// One tile. a, b: where its lines begin (GroupedLoader::init), k in bytes where an operand has it side by side, in steps where not; c with its first row and column.
struct GroupedTile {
  const char *a, *b;
  const int32_t *index, *index_b;
  unsigned index_at, limit, limit_b, a_first, a_count, b_first, b_count, k;  // k: values
  char *c;
  unsigned rows, cols;  // of C from there on
};

template <int DT, bool A_KC, bool B_KC, int BM, int BN, int WAVES, int WAVES_N, int NS, bool A_INDEXED = false, bool B_INDEXED = false>
struct GroupedRing {
  using M = RingMma<DT, DT, false>;
  static constexpr int WAVES_M = WAVES / WAVES_N, WM = BM / WAVES_M, WN = BN / WAVES_N, MI = WM / 16, NI = WN / 16;
  using LA = GroupedLoader<A_KC, BM, WAVES, NS, A_INDEXED>;
  using LB = GroupedLoader<B_KC, BN, WAVES, NS, B_INDEXED>;
  using RA = FragReader<2, A_KC, 16, BM, NS, 16, false>;
  using RB = FragReader<2, B_KC, 16, BN, NS, 16, false>;
  static constexpr int PA = RA::kPieces, PB = RB::kPieces, kReadsB = NI * PB, kReads = kReadsB + MI * PA, kSlots = MI * NI, kReadSlots = kSlots * 3 / 4 > 0 ? kSlots * 3 / 4 : 1;
  static constexpr int kPairA = A_KC ? LA::kBlocks : 0, kPairB = B_KC ? LB::kBlocks : 0, kEachA = A_KC ? 0 : LA::kBlocks, kEachB = B_KC ? 0 : LB::kBlocks, kEach = kEachA + kEachB;
  static_assert(NS % 2 == 0);
  // Requests of a step, U its parity: pairs of slices s + NS - 1, s + NS in odd steps, whose stages the barrier in front has freed, and slice s + NS in every step.
  static constexpr int kLoads[2] = {kEach, kPairA + kPairB + kEach};
  // ... that may be under way at the barrier of slice s, where slice s + 1 has to be there: what was requested behind the last of it.
  static constexpr int in_flight(int u) {
    const int both = kLoads[0] + kLoads[1];
    int most = 63;
    if (kPairA + kPairB) {  // since step s - NS + 1, or s - NS + 2
      const int x = kLoads[1] - kPairA - kPairB + (NS / 2 - 1) * both - (u == 0 ? 0 : kLoads[1]);
      most = x < most ? x : most;
    }
    if (kEach) {  // since step s - NS + 1
      const int x = (NS / 2 - 1) * both;
      most = x < most ? x : most;
    }
    return most;
  }
  static constexpr int kInFlight[2] = {in_flight(0), in_flight(1)};
  static_assert(kInFlight[1] + kLoads[1] < 64, "vmcnt is a 6-bit counter");
  static constexpr unsigned kRegionA = STile<2, A_KC, BM, NS, 16>::kRegion, kLdsRing = kRegionA + STile<2, B_KC, BN, NS, 16>::kRegion, kLdsRows = WAVES * grouped_space<MI, NI>();
  static constexpr unsigned kLds = kLdsRing > kLdsRows ? kLdsRing : kLdsRows;

  static constexpr int first_in_slot(int q, int n, int m) { return q >= m ? n : (q * n + m - 1) / m; }
  static constexpr int first_load(int q, int n, int m) { return q >= m ? n : q * 2 * n <= m ? 0 : (2 * q * n - m + 2 * m - 1) / (2 * m); }

  __device__ __forceinline__ static void run(const GroupedRingArgs &p, const GroupedTile &t, char *smem) {
    char *const region_a = smem, *const region_b = smem + kRegionA;
    const unsigned addr_a = (unsigned)(size_t)LDS_PTR(char, smem), addr_b = addr_a + kRegionA;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / WAVES_N * WM, wn = wave % WAVES_N * WN;
    LA la;
    LB lb;
    la.init(t.a, p.a_pitch, t.index, t.index_at, t.limit, t.a_first, t.a_count, A_KC ? t.k * 2 : t.k);
    lb.init(t.b, p.b_pitch, t.index_b, t.index_at, t.limit_b, t.b_first, t.b_count, B_KC ? t.k * 2 : t.k);
    RA ra;
    RB rb;
    ra.init(wm);
    rb.init(wn);
    v4f acc[MI][NI];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) acc[i][j] = v4f{0, 0, 0, 0};
    const unsigned slices = (t.k * 2 + 2 * kRingSlice - 1) / (2 * kRingSlice) * 2, pairs = slices / 2;
    if (slices != 0) {
      const auto unit_of = [&](bool kc, unsigned unit) {
        const unsigned most = (kc ? pairs : slices) - 1;
        return unit < most ? unit : most;
      };
      // What the steps before the first would have requested, in their order (the rows of all of it looked up ahead).
      typename LA::Lines rows_a[A_INDEXED ? NS : 1];
      typename LB::Lines rows_b[B_INDEXED ? NS : 1];
      if constexpr (A_INDEXED)
#pragma unroll
        for (int u = 0; u < NS; ++u) rows_a[u] = la.look_up(unit_of(false, u));
      if constexpr (B_INDEXED)
#pragma unroll
        for (int u = 0; u < NS; ++u) rows_b[u] = lb.look_up(unit_of(false, u));
      const auto request_a = [&](unsigned unit, unsigned stage) __attribute__((always_inline)) {
        const unsigned u = unit_of(A_KC, unit);
        if constexpr (A_INDEXED) la.take(rows_a[stage]);
#pragma unroll
        for (int i = 0; i < LA::kBlocks; ++i) la.request(region_a, (int)stage, u, la.left_of(u), i);
      };
      const auto request_b = [&](unsigned unit, unsigned stage) __attribute__((always_inline)) {
        const unsigned u = unit_of(B_KC, unit);
        if constexpr (B_INDEXED) lb.take(rows_b[stage]);
#pragma unroll
        for (int i = 0; i < LB::kBlocks; ++i) lb.request(region_b, (int)stage, u, lb.left_of(u), i);
      };
#pragma unroll
      for (int step = -NS; step < 0; ++step) {
        if (A_KC && (step & 1) && step + NS - 1 >= 0) request_a((step + NS - 1) / 2, step + NS - 1);
        if (B_KC && (step & 1) && step + NS - 1 >= 0) request_b((step + NS - 1) / 2, step + NS - 1);
        if (!A_KC) request_a(step + NS, step + NS);
        if (!B_KC) request_b(step + NS, step + NS);
      }
      la.ahead = la.look_up(unit_of(false, NS)), lb.ahead = lb.look_up(unit_of(false, NS));
      wait_loads_upto<kInFlight[1] + kLoads[1]>();  // slice 0
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();

      typename RA::Piece pa[2][MI][PA];
      typename RB::Piece pb[2][NI][PB];
      const auto read_item = [&](auto rc, auto bufc, unsigned stage_a, unsigned stage_b) __attribute__((always_inline)) {
        constexpr int R = decltype(rc)::value, BUF = decltype(bufc)::value;
        if constexpr (R < kReadsB) pb[BUF][R / PB][R % PB] = rb.template read<R / PB, R % PB>(stage_b);
        else pa[BUF][(R - kReadsB) / PA][(R - kReadsB) % PA] = ra.template read<(R - kReadsB) / PA, (R - kReadsB) % PA>(stage_a);
      };
      const auto landed = [&](int buf) __attribute__((always_inline)) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
          for (int w = 0; w < PA; ++w) asm volatile("" : "+v"(pa[buf][i][w]));
#pragma unroll
        for (int j = 0; j < NI; ++j)
#pragma unroll
          for (int w = 0; w < PB; ++w) asm volatile("" : "+v"(pb[buf][j][w]));
      };
      [&]<int... Rs>(std::integer_sequence<int, Rs...>) __attribute__((always_inline)) {
        (read_item(std::integral_constant<int, Rs>{}, std::integral_constant<int, 0>{}, addr_a, addr_b), ...);
      }(std::make_integer_sequence<int, kReads>{});

      unsigned s0 = 0;
      do {
        [&]<int... Us>(std::integer_sequence<int, Us...>) __attribute__((always_inline)) {
          (
              [&](auto uc) __attribute__((always_inline)) {
                constexpr int U = decltype(uc)::value, kHere = kLoads[U];
                const unsigned s = s0 + U;
                unsigned unit_a, unit_b, next_a, next_b, left_a, left_b;
                int fill_a, fill_b;
                // The next slice is there for every wave, and everybody has read the one whose stage is refilled.
                wait_loads_upto<kInFlight[U]>();
                landed(U);
                __builtin_amdgcn_s_barrier();
                __builtin_amdgcn_sched_barrier(0);
                [&]<int... Qs>(std::integer_sequence<int, Qs...>) __attribute__((always_inline)) {
                  (
                      [&](auto qc) __attribute__((always_inline)) {
                        constexpr int Q = decltype(qc)::value, i = Q / NI, j = Q % NI;
                        M::template run<ring_sum_in_a<MI, NI, v4f>(i, j)>(join_pieces<v4i>(pa[U][i]), join_pieces<v4i>(pb[U][j]), acc[i][j]);
                        __builtin_amdgcn_sched_barrier(0);
                        if constexpr (Q == 0) {
                          const auto unit = [&](bool kc) {
                            const unsigned x = kc ? (s + NS - 1) / 2 : s + NS, most = (kc ? pairs : slices) - 1;
                            return x < most ? x : most;
                          };
                          unit_a = unit(A_KC), unit_b = unit(B_KC);
                          left_a = la.left_of(unit_a), left_b = lb.left_of(unit_b);
                          la.take(la.ahead), lb.take(lb.ahead);  // (in front of this step's reads: the compiler waits for both together)
                          la.ahead = la.look_up(unit_a + 1 < slices ? unit_a + 1 : unit_a), lb.ahead = lb.look_up(unit_b + 1 < slices ? unit_b + 1 : unit_b);
                          fill_a = (int)((s + (A_KC ? NS - 1 : NS)) % NS), fill_b = (int)((s + (B_KC ? NS - 1 : NS)) % NS);
                          next_a = addr_a + (s + 1) % NS * STile<2, A_KC, BM, NS, 16>::kStageStep, next_b = addr_b + (s + 1) % NS * STile<2, B_KC, BN, NS, 16>::kStageStep;
                        }
                        [&]<int... Rs>(std::integer_sequence<int, Rs...>) __attribute__((always_inline)) {
                          (read_item(std::integral_constant<int, first_in_slot(Q, kReads, kReadSlots) + Rs>{}, std::integral_constant<int, U ^ 1>{}, next_a, next_b), ...);
                        }(std::make_integer_sequence<int, first_in_slot(Q + 1, kReads, kReadSlots) - first_in_slot(Q, kReads, kReadSlots)>{});
                        constexpr int L = first_load(Q, kHere, kSlots), kLoadsHere = first_load(Q + 1, kHere, kSlots) - L;
#pragma unroll
                        for (int l = L; l < L + kLoadsHere; ++l) {
                          constexpr int pair_a = U ? kPairA : 0, pair_b = U ? kPairB : 0;
                          const int each = l - pair_a - pair_b;
                          if (l < pair_a) la.request(region_a, fill_a, unit_a, left_a, l);
                          else if (l < pair_a + pair_b) lb.request(region_b, fill_b, unit_b, left_b, l - pair_a);
                          else if (each < kEachA) la.request(region_a, fill_a, unit_a, left_a, each);
                          else lb.request(region_b, fill_b, unit_b, left_b, each - kEachA);
                        }
                        __builtin_amdgcn_sched_barrier(0);
                      }(std::integral_constant<int, Qs>{}),
                      ...);
                }(std::make_integer_sequence<int, kSlots>{});
              }(std::integral_constant<int, Us>{}),
              ...);
        }(std::make_integer_sequence<int, 2>{});
        asm volatile("s_nop 7");  // the last product's passes: the compiler, to which it is no matrix instruction, may copy its sums as soon as the loop is left
        s0 += 2;
      } while (s0 < slices);
      __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
      landed(0);                           // the last step's reads, of a slice that does not exist: their registers are theirs up to here
      asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
      [&]<int... Bs>(std::integer_sequence<int, Bs...>) __attribute__((always_inline)) {
        ((acc[Bs / NI][Bs % NI] = fetched<ring_sum_in_a<MI, NI, v4f>(Bs / NI, Bs % NI)>(acc[Bs / NI][Bs % NI])), ...);
      }(std::make_integer_sequence<int, MI * NI>{});
    }
    __syncthreads();  // every wave's reads of the stages and requests into them are over
    char *const space = smem + wave * grouped_space<MI, NI>();
    if (p.c_single) grouped_write<float, MI, NI>(reinterpret_cast<float *>(t.c), p.rsc, acc, wm, wn, t.rows, t.cols, p.alpha, p.beta, space);
    else if constexpr (DT == SKL_DT_BF16) grouped_write<__bf16, MI, NI>(reinterpret_cast<__bf16 *>(t.c), p.rsc, acc, wm, wn, t.rows, t.cols, p.alpha, p.beta, space);
    else grouped_write<_Float16, MI, NI>(reinterpret_cast<_Float16 *>(t.c), p.rsc, acc, wm, wn, t.rows, t.cols, p.alpha, p.beta, space);
  }
};

template <int DT, bool B_KC, int MOST, int BN, int WAVES, int NS>
struct GroupedRows {
  using Full = GroupedRing<DT, true, B_KC, MOST, BN, WAVES, MOST == 64 ? (BN / 16 < WAVES ? BN / 16 : WAVES) : 2, NS>;
  // Fewer rows: less to compute for a slice, more slices under way. (With four as well, tiles of 64 rows took 0.61 us for a slice of 32 k, those of 256 0.80.)
  using Half = GroupedRing<DT, true, B_KC, 128, BN, WAVES, WAVES / 2, MOST == 256 ? 6 : NS>;
  using Quarter = GroupedRing<DT, true, B_KC, 64, BN, WAVES, WAVES, MOST == 256 ? 8 : NS>;
  static constexpr unsigned kLds = MOST == 256 && Quarter::kLds > Full::kLds ? Quarter::kLds : Full::kLds;
  static_assert(MOST != 256 || Half::kLds <= kLds);
  static_assert(kLds <= 160 * 1024);
};

template <int DT, bool B_KC, int MOST, int BN, int WAVES, int NS>
__global__ void __launch_bounds__(WAVES * 64) gemm_grouped_rows_kernel(GroupedRingArgs p) {
  using Rows = GroupedRows<DT, B_KC, MOST, BN, WAVES, NS>;
  extern __shared__ __attribute__((aligned(128))) char grouped_smem[];
  const GroupedPlace at = grouped_place<MOST>(p.offsets, p.groups, p.m, p.tiles_n, blockIdx.x);
  if (at.none) return;
  const unsigned col0 = at.tile_n * BN;
  GroupedTile t;
  t.a = p.a, t.index = p.rows, t.index_b = nullptr, t.index_at = at.first, t.limit = p.a_rows, t.limit_b = 0, t.a_first = at.first, t.a_count = at.rows;
  t.b = p.b + (size_t)at.e * p.b_group, t.b_first = col0, t.b_count = p.n - col0, t.k = p.k;
  t.c = p.c + ((size_t)at.first * p.rsc + col0) * (p.c_single ? 4 : 2), t.rows = at.rows, t.cols = p.n - col0;
  if constexpr (MOST > 128) {
    if (at.rows > 128) Rows::Full::run(p, t, grouped_smem);
    else if (at.rows > 64) Rows::Half::run(p, t, grouped_smem);
    else Rows::Quarter::run(p, t, grouped_smem);
  } else {
    Rows::Full::run(p, t, grouped_smem);
  }
}

// The group that comes at place `place`, the longest one first, and its rows. Finding out among 64 groups takes 1 us, so that short ones are taken as they lie unless there are few.
struct GroupedTurn {
  unsigned e;
  SklRange rows;
};
template <unsigned MOST>
__device__ __forceinline__ GroupedTurn grouped_longest_first(const int32_t *offsets, unsigned groups, unsigned most, unsigned place) {
  const unsigned lane = threadIdx.x & 63u;
  const SklRange mine = lane < groups ? skl_group_range(offsets, lane, most) : SklRange{0, 0};
  unsigned ahead = 0;
#pragma unroll
  for (unsigned g = 0; g < MOST; ++g) {  // (lanes beyond the groups hold none and come last)
    const unsigned other = (unsigned)__builtin_amdgcn_readlane((int)mine.rows, (int)g);
    ahead += other > mine.rows || (other == mine.rows && g < lane);
  }
  const int owner = (int)__builtin_ctzll(__ballot(lane < groups && ahead == place));
  return {(unsigned)owner, {(unsigned)__builtin_amdgcn_readlane((int)mine.first, owner), (unsigned)__builtin_amdgcn_readlane((int)mine.rows, owner)}};
}
__device__ __forceinline__ GroupedTurn grouped_by_length(const int32_t *offsets, unsigned groups, unsigned most, unsigned place) {
  if (groups > 1 && groups <= 16) return grouped_longest_first<16>(offsets, groups, most, place);
  if (groups > 1 && groups <= 64 && most >= 512 * groups) return grouped_longest_first<64>(offsets, groups, most, place);
  SklRange r = skl_group_range(offsets, place, most);
  return {place, {(unsigned)__builtin_amdgcn_readfirstlane((int)r.first), (unsigned)__builtin_amdgcn_readfirstlane((int)r.rows)}};
}

// Sums over the groups' rows: both operands across K, tiles of BM x BN of each group's C.
template <int DT, int BM, int BN, int WAVES, int WAVES_N, bool A_INDEXED, bool B_INDEXED>
__global__ void __launch_bounds__(WAVES * 64) gemm_grouped_over_kernel(GroupedRingArgs p) {
  using Ring = GroupedRing<DT, false, false, BM, BN, WAVES, WAVES_N, 4, A_INDEXED, B_INDEXED>;
  extern __shared__ __attribute__((aligned(128))) char grouped_smem[];
  // Each die takes a run of every group's tiles - a group's length decides how long they take -, the longest group first, walked in blocks of eight rows of tiles, column by column.
  const unsigned tiles = p.tiles_m * p.tiles_n, run = (tiles + 7) / 8, die = blockIdx.x % 8, slot = blockIdx.x / 8;
  const unsigned in = die * run + slot % run;
  if (in >= tiles) return;
  unsigned e = slot / run;  // its part, too
  SklRange r;
  if (p.parts == 1) {
    const GroupedTurn turn = grouped_by_length(p.offsets, p.groups, p.k, e);
    e = turn.e, r = turn.rows;
  } else {
    r = skl_group_range(p.offsets, e / p.parts, p.k);
    const unsigned each = (r.rows + p.parts * 64 - 1) / (p.parts * 64) * 64, before = e % p.parts * each;  // whole slices but for the last one's
    r.first = (unsigned)__builtin_amdgcn_readfirstlane((int)(r.first + (before < r.rows ? before : r.rows)));
    r.rows = (unsigned)__builtin_amdgcn_readfirstlane((int)(before < r.rows ? (r.rows - before < each ? r.rows - before : each) : 0u));
  }
  const unsigned block = in / (8 * p.tiles_n), in_block = in - block * (8 * p.tiles_n), deep = p.tiles_m - 8 * block < 8 ? p.tiles_m - 8 * block : 8;
  const unsigned row0 = (8 * block + in_block % deep) * BM, col0 = in_block / deep * BN;
  GroupedTile t;
  t.index = p.rows, t.index_b = p.rows_b, t.index_at = r.first, t.limit = p.a_rows, t.limit_b = p.b_rows;
  t.a = A_INDEXED ? p.a : p.a + (size_t)r.first * p.a_pitch, t.a_first = row0, t.a_count = p.m - row0;
  t.b = B_INDEXED ? p.b : p.b + (size_t)r.first * p.b_pitch, t.b_first = col0, t.b_count = p.n - col0, t.k = r.rows;
  t.c = p.c + ((size_t)e * p.gsc + (size_t)row0 * p.rsc + col0) * (p.c_single ? 4 : 2), t.rows = p.m - row0, t.cols = p.n - col0;
  Ring::run(p, t, grouped_smem);
}

// Sums of parts, added up in their order: C_e = alpha * (part 0 + part 1 + ..) + beta * C_e.
struct GroupedJoin {
  const float *from;  // [groups][parts][m][n]
  void *c;
  size_t rsc, gsc;
  unsigned groups, m, n, parts;
  int c_single;
  skl_scalar alpha, beta;
};
template <typename TC>
__global__ void __launch_bounds__(256) gemm_grouped_join_kernel(GroupedJoin p) {
  const size_t size = (size_t)p.m * p.n;
  const bool read_c = !skl_beta_is_zero<float>(p.beta);
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < size * p.groups; i += (size_t)gridDim.x * 256) {
    const unsigned e = (unsigned)(i / size), in = (unsigned)(i % size), row = in / p.n, col = in % p.n;
    const float *const from = p.from + (size_t)e * p.parts * size + in;
    float sum = from[0];
#pragma unroll 4
    for (unsigned part = 1; part < p.parts; ++part) sum = __fadd_rn(sum, from[part * size]);
    TC *const to = reinterpret_cast<TC *>(p.c) + (size_t)e * p.gsc + (size_t)row * p.rsc + col;
    *to = skl_grouped_result(sum, to, p.alpha, p.beta, read_c);
  }
}
template <int DT>
int launch_join(const GroupedJoin &j) {
  const size_t blocks = skl_div_up((size_t)j.m * j.n * j.groups, 256);
  const dim3 grid((unsigned)(blocks < 4096 ? blocks : 4096));
  if (j.c_single) gemm_grouped_join_kernel<float><<<grid, dim3(256), 0, skl_current_stream()>>>(j);
  else if (DT == SKL_DT_BF16) gemm_grouped_join_kernel<__bf16><<<grid, dim3(256), 0, skl_current_stream()>>>(j);
  else gemm_grouped_join_kernel<_Float16><<<grid, dim3(256), 0, skl_current_stream()>>>(j);
  return skl_check_launch("gemm_grouped: join");
}

template <typename K>
int launch_ring(K kernel, std::atomic<unsigned long long> &allowed, unsigned lds, unsigned threads, const GroupedRingArgs &p, size_t blocks) {
  const int rc = skl_allow_lds(reinterpret_cast<const void *>(kernel), lds, allowed);
  if (rc != 0) return rc;
  kernel<<<dim3((unsigned)blocks), dim3(threads), lds, skl_current_stream()>>>(p);
  return skl_check_launch("gemm_grouped");
}
constexpr size_t kMostRingBlocks = size_t(1) << 22;
template <int DT, bool B_KC, int MOST, int BN, int WAVES, int NS>
int grouped_rows(const skl_grouped_gemm &g, GroupedRingArgs p) {
  const size_t lines = g.m / MOST + (g.m < g.groups ? g.m : g.groups);  // of tiles: whole ones, and one more for each group that has a row
  const size_t most = kMostRingBlocks / (lines + 16) > 0 ? kMostRingBlocks / (lines + 16) : 1, slab = most * BN;
  static std::atomic<unsigned long long> allowed{0};
  for (size_t col = 0; col < g.n; col += slab) {
    p.n = (unsigned)(g.n - col < slab ? g.n - col : slab);
    p.tiles_n = skl_div_up(p.n, BN);
    p.b = (const char *)g.b + col * g.csb * 2;
    p.c = (char *)g.c + col * (g.c_single ? 4 : 2);
    const int rc = launch_ring(gemm_grouped_rows_kernel<DT, B_KC, MOST, BN, WAVES, NS>, allowed, GroupedRows<DT, B_KC, MOST, BN, WAVES, NS>::kLds, WAVES * 64, p, (lines * p.tiles_n / 8 + 2) * 8);
    if (rc != 0) return rc;
  }
  return 0;
}
template <int DT, bool B_KC>
int grouped_rows_by_size(const skl_grouped_gemm &g, const GroupedRingArgs &p) {
  // By how many rows a group has on average and how many tiles there are: the largest tile that is mostly filled and fills the chip. us, 256 x 256 / 128 x 128 / 64 x 64: 32 groups of
  // 2816 x 2048 with 256, 512, 1024 and 3000 tokens to four of them -, 84, 78; 92, 85, 93; 107, 116, 140; 167, 200, 315; two groups of 1024 x 1024 with 2000 rows 27, 15, 13. One token to four of
  // 32 groups: 64 x 64 with eight slices of k in the ring 12.5, 64 x 128 with four 28.
  const size_t groups = g.m < g.groups ? g.m : g.groups, lines = g.m / 256 + groups / 2, lines_half = g.m / 128 + groups / 2;  // half of the last tiles of the groups are small ones
  if (g.m >= 112 * groups && lines * skl_div_up(g.n, 256) >= 160) return grouped_rows<DT, B_KC, 256, 256, 8, 4>(g, p);
  if (g.m >= 56 * groups && lines_half * skl_div_up(g.n, 128) >= 160) return grouped_rows<DT, B_KC, 128, 128, 8, 4>(g, p);
  return grouped_rows<DT, B_KC, 64, 64, 4, 8>(g, p);
}
template <int DT>
int grouped_ring(const skl_grouped_gemm &g) {
  const bool kc = g.rsb == 1;
  GroupedRingArgs p{};
  p.a = (const char *)g.a, p.offsets = g.offsets, p.rows = g.rows;
  p.a_pitch = g.rsa * 2, p.b_pitch = (kc ? g.csb : g.rsb) * 2, p.b_group = g.gsb * 2;
  p.rsc = g.rsc, p.groups = (unsigned)g.groups, p.m = (unsigned)g.m, p.k = (unsigned)g.k, p.a_rows = (unsigned)g.a_rows;
  p.c_single = g.c_single, p.alpha = g.alpha, p.beta = g.beta;
  return kc ? grouped_rows_by_size<DT, true>(g, p) : grouped_rows_by_size<DT, false>(g, p);
}

template <int DT, int BM, int BN, int WAVES, int WAVES_N, bool A_INDEXED, bool B_INDEXED>
int grouped_over(const skl_groupedk_gemm &g, GroupedRingArgs p) {
  p.tiles_m = skl_div_up(g.m, BM);
  const size_t all_n = skl_div_up(g.n, BN), left = kMostRingBlocks / p.tiles_m > 0 ? kMostRingBlocks / p.tiles_m : 1;
  const size_t slab_n = (left < all_n ? left : all_n) * BN, slab = left / all_n > 0 ? left / all_n : 1;
  static std::atomic<unsigned long long> allowed{0};
  const auto launch = [&](size_t blocks) {
    return launch_ring(gemm_grouped_over_kernel<DT, BM, BN, WAVES, WAVES_N, A_INDEXED, B_INDEXED>, allowed, GroupedRing<DT, false, false, BM, BN, WAVES, WAVES_N, 4>::kLds, WAVES * 64, p, blocks);
  };
  if (p.parts > 1) {  // (few tiles, one launch) C of every part into scratch memory, where the join finds them
    const GroupedJoin j{(const float *)p.c, g.c, g.rsc, g.gsc, (unsigned)g.groups, p.m, (unsigned)g.n, p.parts, g.c_single, g.alpha, g.beta};
    p.n = (unsigned)g.n, p.tiles_n = (unsigned)all_n, p.offsets = g.offsets, p.groups = (unsigned)g.groups;
    p.b = (const char *)g.b;
    p.rsc = g.n, p.gsc = g.m * g.n, p.c_single = 1;
    p.alpha.f = 1.0f, p.beta.fz.value = 0.0f, p.beta.fz.skip_c_read = SKL_C_UNTOUCHED;
    const int rc = launch(g.groups * p.parts * ((p.tiles_m * all_n + 7) / 8) * 8);
    return rc != 0 ? rc : launch_join<DT>(j);
  }
  for (size_t e = 0; e < g.groups; e += slab) {
    p.groups = (unsigned)(g.groups - e < slab ? g.groups - e : slab);
    p.offsets = g.offsets ? g.offsets + e : nullptr;
    for (size_t col = 0; col < g.n; col += slab_n) {
      p.n = (unsigned)(g.n - col < slab_n ? g.n - col : slab_n);
      p.tiles_n = skl_div_up(p.n, BN);
      p.b = (const char *)g.b + col * 2;
      p.c = (char *)g.c + (e * g.gsc + col) * (g.c_single ? 4 : 2);
      const int rc = launch((size_t)p.groups * (((size_t)p.tiles_m * p.tiles_n + 7) / 8) * 8);
      if (rc != 0) return rc;
    }
  }
  return 0;
}
template <int DT, int BM, int BN, int WAVES, int WAVES_N>
int grouped_over_indexed(const skl_groupedk_gemm &g, const GroupedRingArgs &p) {
  if (g.rows_a) return g.rows_b ? grouped_over<DT, BM, BN, WAVES, WAVES_N, true, true>(g, p) : grouped_over<DT, BM, BN, WAVES, WAVES_N, true, false>(g, p);
  return g.rows_b ? grouped_over<DT, BM, BN, WAVES, WAVES_N, false, true>(g, p) : grouped_over<DT, BM, BN, WAVES, WAVES_N, false, false>(g, p);
}
template <int DT>
int grouped_over_ring(const skl_groupedk_gemm &g) {
  GroupedRingArgs p{};
  p.a = (const char *)g.a, p.a_pitch = g.rsa * 2, p.b_pitch = g.rsb * 2;
  p.rows = g.rows_a, p.rows_b = g.rows_b, p.a_rows = (unsigned)g.a_rows, p.b_rows = (unsigned)g.b_rows;
  p.rsc = g.rsc, p.gsc = g.gsc, p.m = (unsigned)g.m, p.k = (unsigned)g.total;
  p.c_single = g.c_single, p.alpha = g.alpha, p.beta = g.beta;
  p.parts = 1;
  // Tiles of 256 x 256 where they fill half the chip. (Smaller ones with two workgroups to a compute unit are slower at every length, short ones among them: us, 256 x 256 / 128 x 128,
  // 64 groups of 2048 x 1408 with 96 rows on average 165 / 217.) Fewer of them share out their rows among workgroups, if there are enough, or are 128 x 128, or both; the parts meet in scratch
  // memory. us, 256 x 256 / the same with parts / 128 x 128 / the same with parts: 4 groups of 1024 x 1024 with 32768 rows 284 / 107 / 157 / 132, 2 of 1024 x 4096 with 16384 239 / 157 / - / -,
  // 2 of 512 x 256 with 32768 356 / 62 / 197 / 32, 16 of 256 x 512 with 32000 106 / 79 / 60 / 37, 3 of 1152 x 832 with 1002 21 / 29 / 11 / 23, 2 of 512 x 512 with 64 12.4 / - / 6.6 / -.
  const size_t tiles = g.groups * skl_div_up(g.m, 256) * skl_div_up(g.n, 256), each = g.total / g.groups;
  if (tiles > 128) return grouped_over_indexed<DT, 256, 256, 8, 2>(g, p);
  const size_t small = g.groups * skl_div_up(g.m, 128) * skl_div_up(g.n, 128);
  size_t parts = 256 / tiles < each / 1024 ? 256 / tiles : each / 1024;
  const bool large = tiles == 128 || (tiles >= 64 && parts >= 2);
  if (!large) parts = 512 / small < each / 256 ? 512 / small : each / 256;
  const size_t one = g.groups * g.m * g.n * 4, most = (size_t(1) << 26) / one < 64 ? (size_t(1) << 26) / one : 64;  // the workspace's 64 MiB
  if (parts > most) parts = most;
  const bool sequence = parts >= 2;
  if (sequence) {
    skl_hip_sequence_begin();
    p.c = (char *)skl_workspace(parts * one, true);
    if (p.c) p.parts = (unsigned)parts;  // no scratch memory: in one part
  }
  const int rc = large ? grouped_over_indexed<DT, 256, 256, 8, 2>(g, p) : grouped_over_indexed<DT, 128, 128, 8, 2>(g, p);
  if (sequence) skl_hip_sequence_end();
  return rc;
}

}  // namespace
