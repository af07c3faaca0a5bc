// skl_moe_mxf4.hip - a mixture-of-experts layer over MXFP4 weights for up to 64 tokens (include/skl-gfx950.h has the formulas):
// router, choice, the chosen experts' gated input product, their output product and its weighted sum.
//
// What bounds it is the stream over the chosen experts' weights, half a byte and a thirty-second per value. They are widened in
// registers to bf16 with their scale (v_cvt_scalef32_pk_bf16_fp4, exact) and multiplied by v_mfma_f32_16x16x32_bf16: products of bf16
// values, exact, summed in fp32. A lane's 16 bytes are one block of 32 k of one row of weights; which k of a chunk of 128 meet in which
// of its four instructions is free as long as both operands' lanes take the same.
// The tokens of an expert are gathered: only rows of tokens that chose it are multiplied, 16 at a time. h travels as the sum of three bf16
// values, which is all of its 24 bits: two (7.6e-6 off at most) left y 1.0e-6 off, three 3e-7, and the stream covers the third's products.
//
// Three launches, each with a workgroup per piece of work so that the stream finds every compute unit; what must follow all of a
// launch's workgroups is done by the one that arrives last (a counter that is zero between calls): the choice behind the router's
// sums, and the weighted sum over a token's experts behind the output products. Every sum has a fixed order.
#include <hip/hip_runtime.h>

#include "skl_device.hpp"
#include "skl_mx.h"
#include "../../include/skl-hip.h"

namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));

constexpr unsigned kMaxTokens = SKL_MOE_TOKENS, kMaxExperts = 1024, kMaxTop = 64;

// What the kernels hand on, in the stream's scratch memory.
struct Slot {  // an expert that some token chose
  unsigned expert, first, count, unused;  // its first place: places are numbered by expert and then by token
};
struct Routing {
  float *parts;          // [split][token][expert], the router's sums
  unsigned *active;      // how many slots there are
  Slot *slots;           // ascending by expert
  uint8_t *tokens;       // [slot][64]
  float *weight;         // [place]
  unsigned *place;       // [token][j], of its j-th choice
  uint16_t *h[3];        // [place][inter]: the terms
  float *out;            // [split][place][hidden], the output products
  unsigned *counters;    // zero between launches: the router's, then one per tile of columns of y
  unsigned router_splits, out_splits, places;
};

struct MoeArgs {
  skl_moe_problem p;
  Routing r;
};

__device__ __forceinline__ v8bf widen_f4(unsigned w, float scale) {  // eight E2M1 values, low nibble first, times their scale: exact
  const v2bf p0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0), p1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1);
  const v2bf p2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2), p3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3);
  return v8bf{p0.x, p0.y, p1.x, p1.y, p2.x, p2.y, p3.x, p3.y};
}
__device__ __forceinline__ unsigned short bf16_of(float v) { return __builtin_bit_cast(unsigned short, (__bf16)v); }  // to nearest even
__device__ __forceinline__ float of_bf16(unsigned short v) { return __uint_as_float((unsigned)v << 16); }

// What one workgroup leaves for another of the same launch goes past its die's cache and is read past it, value by value; a fence
// instead writes all of that cache back, for every workgroup (the output products of 7 tokens 147 us with fences).
__device__ __forceinline__ void leave(float *to, float v) { __hip_atomic_store(to, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ float found(const float *from) { return __hip_atomic_load(from, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// Whether this workgroup is the last of `all` to come here; what the others have left is then there to be found.
__device__ __forceinline__ bool arrives_last(unsigned *counter, unsigned all, unsigned *shared) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's stores have reached memory
  __syncthreads();
  if (threadIdx.x == 0) *shared = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  const bool last = *shared == all - 1;
  if (last && threadIdx.x == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return last;
}

// A logit as a number that orders like it: NaN lowest, the two zeros alike; 0 is none.
__device__ __forceinline__ unsigned order_of(float v) {
  if (v != v) return 1u;
  const unsigned b = __float_as_uint(v + 0.0f);
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned max_with(unsigned v) {  // of lanes that nothing comes to: v
  const unsigned o = (unsigned)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, ROWS, 0xF, false);
  return v > o ? v : o;
}
__device__ __forceinline__ unsigned wave_max(unsigned v) {
  v = max_with<0x111, 0xF>(v);  // one, two, four and eight lanes down a row of 16
  v = max_with<0x112, 0xF>(v);
  v = max_with<0x114, 0xF>(v);
  v = max_with<0x118, 0xF>(v);
  v = max_with<0x142, 0xA>(v);  // the end of a row of 16 to the next, of 32 to the upper half
  v = max_with<0x143, 0xC>(v);
  return (unsigned)__builtin_amdgcn_readlane((int)v, 63);
}

constexpr int kRouterThreads = 1024;

struct Choice {
  unsigned mask[kMaxExperts][2];  // tokens that chose an expert
  unsigned start[kMaxExperts];
  unsigned short slot[kMaxExperts];
  unsigned short chosen[kMaxTokens * kMaxTop];
  float share[kMaxTokens * kMaxTop];
  unsigned totals[kRouterThreads / 64];
};

// The choice of one token by one wave: NE logits per lane, expert 64 i + lane.
template <int NE>
__device__ __forceinline__ void choose(const MoeArgs &a, Choice &c, unsigned t, int lane) {
  const skl_moe_problem &p = a.p;
  const unsigned experts = (unsigned)p.experts, top = (unsigned)p.top_k;
  float value[NE];
  unsigned key[NE];
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    const unsigned e = 64u * i + lane;
    value[i] = 0.0f, key[i] = 0;
    if (e < experts) {
      const float *part = a.r.parts + (size_t)t * experts + e;
      const size_t step = (size_t)p.tokens * experts;
      unsigned split = 0;
#pragma unroll 1
      for (; split + 4 <= a.r.router_splits; split += 4) {  // requested together
        float v[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = found(part + (split + q) * step);
        value[i] += (v[0] + v[1]) + (v[2] + v[3]);
      }
#pragma unroll 1
      for (; split < a.r.router_splits; ++split) value[i] += found(part + split * step);
      key[i] = order_of(value[i]);
    }
  }
  float largest = 0.0f, sum = 0.0f, mine = 0.0f;
  for (unsigned j = 0; j < top; ++j) {
    unsigned best = key[0];
#pragma unroll
    for (int i = 1; i < NE; ++i) best = key[i] > best ? key[i] : best;
    best = wave_max(best);
    unsigned e = 0xFFFFFFFFu;
    float v = 0.0f;
#pragma unroll
    for (int i = 0; i < NE; ++i) {  // the lowest expert that has it
      const unsigned long long who = __ballot(key[i] == best);
      if (e == 0xFFFFFFFFu && who) {
        const int at = __builtin_ctzll(who);
        e = 64u * i + (unsigned)at;
        v = __uint_as_float((unsigned)__builtin_amdgcn_readlane((int)__float_as_uint(value[i]), at));
        if (lane == at) key[i] = 0;
      }
    }
    if (j == 0) largest = v;
    const float x = expf(v - largest);
    if (p.normalise) sum += x;
    if ((unsigned)lane == j) mine = x;
    if (lane == 0) {
      c.chosen[t * top + j] = (unsigned short)e;
      atomicOr(&c.mask[e][t >> 5], 1u << (t & 31u));
    }
  }
  if (!p.normalise) {
#pragma unroll
    for (int i = 0; i < NE; ++i)
      if (64u * i + lane < experts) sum += expf(value[i] - largest);
#pragma unroll
    for (int step = 32; step > 0; step >>= 1) sum += __shfl_xor(sum, step, 64);
  }
  if ((unsigned)lane < top) c.share[t * top + lane] = mine / sum;
}

// The router: a workgroup takes 16 experts, 16 tokens and 512 of hidden, a wave 32 of these; the last one chooses.
template <int NE>
__global__ void __launch_bounds__(kRouterThreads) moe_router_kernel(MoeArgs a) {
  __shared__ union {
    float red[kRouterThreads / 64][16][17];
    Choice c;
  } s;
  __shared__ unsigned arrived;
  const skl_moe_problem &p = a.p;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, l = lane & 15, g = lane >> 4;
  const size_t e0 = (size_t)blockIdx.x * 16, t0 = (size_t)blockIdx.y * 16, k = (size_t)blockIdx.z * 512 + 32 * (size_t)wave;
  const size_t er = e0 + l < p.experts ? e0 + l : p.experts - 1, tr = t0 + l < p.tokens ? t0 + l : p.tokens - 1;
  v4f acc = {0.0f, 0.0f, 0.0f, 0.0f};
  if (k < p.hidden)
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*reinterpret_cast<const v8bf *>(p.x + tr * p.ldx + k + 8 * g),
                                                  *reinterpret_cast<const v8bf *>(p.router + er * p.ld_router + k + 8 * g), acc, 0, 0, 0);
#pragma unroll
  for (int r = 0; r < 4; ++r) s.red[wave][4 * g + r][l] = acc[r];
  __syncthreads();
  if (threadIdx.x < 256) {
    const unsigned i = threadIdx.x >> 4, j = threadIdx.x & 15;
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < kRouterThreads / 64; ++w) v += s.red[w][i][j];
    if (t0 + i < p.tokens && e0 + j < p.experts) leave(a.r.parts + ((size_t)blockIdx.z * p.tokens + t0 + i) * p.experts + e0 + j, v);
  }
  if (!arrives_last(a.r.counters, gridDim.x * gridDim.y * gridDim.z, &arrived)) return;
  const unsigned top = (unsigned)p.top_k, tokens = (unsigned)p.tokens, e = threadIdx.x;
  s.c.mask[e][0] = s.c.mask[e][1] = 0;  // one thread per expert
  __syncthreads();
  for (unsigned t = wave; t < tokens; t += kRouterThreads / 64) choose<NE>(a, s.c, t, lane);
  __syncthreads();
  // Where each expert's tokens begin, and its slot: one scan over the experts, the count in the lower half, the slot in the upper.
  const unsigned count = __popc(s.c.mask[e][0]) + __popc(s.c.mask[e][1]), own = count | (count ? 0x10000u : 0u);
  unsigned scan = own;
#pragma unroll
  for (int step = 1; step < 64; step <<= 1) {
    const unsigned other = __shfl_up(scan, step, 64);
    if (lane >= step) scan += other;
  }
  if (lane == 63) s.c.totals[wave] = scan;
  __syncthreads();
  for (int w = 0; w < wave; ++w) scan += s.c.totals[w];
  s.c.start[e] = (scan - own) & 0xFFFFu;
  s.c.slot[e] = (unsigned short)((scan - own) >> 16);
  if (count) a.r.slots[s.c.slot[e]] = Slot{e, s.c.start[e], count, 0};
  if (e == kMaxExperts - 1) *a.r.active = scan >> 16;
  __syncthreads();
  for (unsigned at = threadIdx.x; at < tokens * top; at += kRouterThreads) {
    const unsigned t = at / top, c = s.c.chosen[at], below = (1u << (t & 31u)) - 1u;
    const unsigned before = t < 32 ? __popc(s.c.mask[c][0] & below) : __popc(s.c.mask[c][0]) + __popc(s.c.mask[c][1] & below);
    const unsigned place = s.c.start[c] + before;
    a.r.tokens[s.c.slot[c] * kMaxTokens + before] = (uint8_t)t;
    a.r.weight[place] = s.c.share[at];
    a.r.place[at] = place;
    if (p.ids) p.ids[at] = (int32_t)c;
    if (p.weights) p.weights[at] = s.c.share[at];
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// The two products. A workgroup has CG groups of 16 rows of one expert's weights - columns of the result -, RG groups of 16 of its tokens
// at a time, and a range of k, of which each of its four waves takes a quarter: chunks of 128, the next one requested before one is
// multiplied. The waves' sums meet in LDS.
// ---------------------------------------------------------------------------------------------------------------------

constexpr int kWaves = 4;

struct Row {  // of weights: this lane's
  const uint8_t *codes, *scales;
};

template <int CG, int RG, int TERMS>
struct Chunk {
  v4i w[CG];
  unsigned s[CG];
  v4i x[RG][TERMS][4];

  // Blocks from `end` on are zeros with a scale of one, and so is what they meet.
  __device__ __forceinline__ void load(const Row (&row)[CG], const uint16_t *const (&x0)[TERMS], const unsigned (&at)[RG], unsigned k, unsigned end, int g, unsigned groups) {
    const unsigned own = k + 32u * (unsigned)g;
    const bool in = own < end;
    const unsigned from = in ? own : 0u;
#pragma unroll
    for (int c = 0; c < CG; ++c) {
      const v4i v = *reinterpret_cast<const v4i *>(row[c].codes + from / 2);
      const unsigned b = row[c].scales[from / 32];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[c][j] = in ? v[j] : 0;
      s[c] = in ? b : 127u;
    }
#pragma unroll
    for (int r = 0; r < RG; ++r)
#pragma unroll
      for (int t = 0; t < TERMS; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v4i v = {0, 0, 0, 0};
          if (r == 0 || r < (int)groups) v = *reinterpret_cast<const v4i *>(x0[t] + at[r] + from + 8 * j);
#pragma unroll
          for (int i = 0; i < 4; ++i) x[r][t][j][i] = in ? v[i] : 0;
        }
  }
  __device__ __forceinline__ void multiply(v4f (&acc)[RG][CG], unsigned groups) const {
#pragma unroll
    for (int c = 0; c < CG; ++c) {
      const float scale = __uint_as_float(s[c] << 23);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const v8bf b = widen_f4((unsigned)w[c][j], scale);
#pragma unroll
        for (int r = 0; r < RG; ++r)
          if (r == 0 || r < (int)groups)
#pragma unroll
            for (int t = 0; t < TERMS; ++t) acc[r][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, x[r][t][j]), b, acc[r][c], 0, 0, 0);
      }
    }
  }
};

// The sums of k in [first, end) into red[wave][row of tokens][column].
template <int CG, int RG, int TERMS>
__device__ __forceinline__ void stream(const Row (&row)[CG], const uint16_t *const (&x)[TERMS], const unsigned (&at)[RG], unsigned first, unsigned end, int wave, int lane,
                                       unsigned groups, float (*red)[RG * 16][16 * CG + 1]) {
  const int l = lane & 15, g = lane >> 4;
  const unsigned chunks = (end - first + 127) / 128, share = (chunks + kWaves - 1) / kWaves;
  const unsigned begin = first + 128 * share * (unsigned)wave;
  unsigned stop = begin + 128 * share;
  stop = stop < end ? stop : end;
  v4f acc[RG][CG];
#pragma unroll
  for (int r = 0; r < RG; ++r)
#pragma unroll
    for (int c = 0; c < CG; ++c) acc[r][c] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  if (begin < stop) {
    Chunk<CG, RG, TERMS> one, two;
    one.load(row, x, at, begin, stop, g, groups);
    for (unsigned k = begin; k < stop; k += 256) {
      two.load(row, x, at, k + 128, stop, g, groups);
      one.multiply(acc, groups);
      one.load(row, x, at, k + 256, stop, g, groups);
      two.multiply(acc, groups);
    }
  }
#pragma unroll
  for (int r = 0; r < RG; ++r)
#pragma unroll
    for (int c = 0; c < CG; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) red[wave][16 * r + 4 * g + i][16 * c + l] = acc[r][c][i];
}

// h of 8 CG inner columns of one expert (blockIdx.y: its slot): CG / 2 groups of gate, as many of up.
template <int CG, int RG>
__global__ void __launch_bounds__(kWaves * 64) moe_in_kernel(MoeArgs a) {
  constexpr int kCols = 8 * CG;
  __shared__ float red[kWaves][RG * 16][16 * CG + 1];
  const skl_moe_problem &p = a.p;
  const unsigned slot = blockIdx.y;
  const Slot own = a.r.slots[slot];
  const unsigned active = *a.r.active;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, l = lane & 15;
  if (slot >= active) return;
  Row row[CG];
#pragma unroll
  for (int c = 0; c < CG; ++c) {
    const skl_mx_operand &op = c < CG / 2 ? p.gate : p.up;
    const size_t col = (size_t)blockIdx.x * kCols + 16 * (c % (CG / 2)) + l;
    row[c] = {op.codes + (own.expert * p.expert_in + col * op.ld) / 2, op.scales + own.expert * p.expert_in_scales + col * op.lds};
  }
  const uint16_t *const x[1] = {p.x};
  for (unsigned done = 0; done < own.count; done += RG * 16) {  // more tokens than a pass takes: the weights again
    const unsigned left = own.count - done, here = left < RG * 16 ? left : RG * 16, groups = (here + 15) / 16;
    unsigned at[RG];
#pragma unroll
    for (int r = 0; r < RG; ++r) {
      const unsigned i = 16u * r + l;
      at[r] = (unsigned)(a.r.tokens[slot * kMaxTokens + done + (i < here ? i : here - 1)] * p.ldx);
    }
    stream<CG, RG, 1>(row, x, at, 0, (unsigned)p.hidden, wave, lane, groups, red);
    __syncthreads();
    for (unsigned n = threadIdx.x; n < here * kCols; n += kWaves * 64) {
      const unsigned i = n / kCols, j = n % kCols;
      float gv = red[0][i][j], uv = red[0][i][kCols + j];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) gv += red[w][i][j], uv += red[w][i][kCols + j];
      const unsigned place = own.first + done + i;
      const float h = skl_activate(gv, p.activation) * uv * a.r.weight[place];
      const unsigned short t0 = bf16_of(h);
      const float rest = h - of_bf16(t0);
      const unsigned short t1 = bf16_of(rest);
      const size_t to = (size_t)place * p.inter + (size_t)blockIdx.x * kCols + j;
      a.r.h[0][to] = t0;
      a.r.h[1][to] = t1;
      a.r.h[2][to] = bf16_of(rest - of_bf16(t1));
    }
    __syncthreads();
  }
}

// The output products of 64 columns, one expert (blockIdx.y) and a part of its inner columns (blockIdx.z); behind the last of a tile of columns
// their sum for each token, in the order of its choices.
constexpr int kOutCols = 64;
template <int RG>
__global__ void __launch_bounds__(kWaves * 64) moe_out_kernel(MoeArgs a) {
  constexpr int CG = kOutCols / 16;
  __shared__ float red[kWaves][RG * 16][kOutCols + 1];
  __shared__ unsigned arrived;
  const skl_moe_problem &p = a.p;
  const unsigned slot = blockIdx.y, split = blockIdx.z;
  const Slot own = a.r.slots[slot];
  const unsigned active = *a.r.active;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, l = lane & 15;
  if (slot >= active) return;
  const unsigned hidden = (unsigned)p.hidden, inter = (unsigned)p.inter, col0 = blockIdx.x * kOutCols;
  const unsigned cols = hidden - col0 < kOutCols ? hidden - col0 : kOutCols;  // 32 or 64
  const unsigned part = ((inter + a.r.out_splits - 1) / a.r.out_splits + 127) / 128 * 128;
  const unsigned begin = split * part < inter ? split * part : inter, end = begin + part < inter ? begin + part : inter;
  Row row[CG];
#pragma unroll
  for (int c = 0; c < CG; ++c) {
    const unsigned j = 16u * c + l;
    const size_t col = col0 + (j < cols ? j : cols - 1);
    row[c] = {p.down.codes + (own.expert * p.expert_down + col * p.down.ld) / 2, p.down.scales + own.expert * p.expert_down_scales + col * p.down.lds};
  }
  for (unsigned done = 0; done < own.count; done += RG * 16) {
    const unsigned left = own.count - done, here = left < RG * 16 ? left : RG * 16, groups = (here + 15) / 16;
    const size_t place = own.first + done;
    const uint16_t *const x[3] = {a.r.h[0] + place * inter, a.r.h[1] + place * inter, a.r.h[2] + place * inter};
    unsigned at[RG];
#pragma unroll
    for (int r = 0; r < RG; ++r) at[r] = (16u * r + l < here ? 16u * r + l : here - 1) * inter;
    stream<CG, RG, 3>(row, x, at, begin, end, wave, lane, groups, red);
    __syncthreads();
    for (unsigned n = threadIdx.x; n < here * kOutCols; n += kWaves * 64) {
      const unsigned i = n / kOutCols, j = n % kOutCols;
      float v = red[0][i][j];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) v += red[w][i][j];
      if (j < cols) leave(a.r.out + ((size_t)split * a.r.places + place + i) * hidden + col0 + j, v);
    }
    __syncthreads();
  }
  if (!arrives_last(a.r.counters + 1 + blockIdx.x, active * a.r.out_splits, &arrived)) return;
  for (unsigned n = threadIdx.x; n < p.tokens * kOutCols; n += kWaves * 64) {
    const unsigned t = n / kOutCols, j = n % kOutCols;
    if (j >= cols) continue;
    float v = 0.0f;
    for (unsigned c = 0; c < p.top_k; ++c) {
      const float *from = a.r.out + (size_t)a.r.place[t * p.top_k + c] * hidden + col0 + j;
      for (unsigned s = 0; s < a.r.out_splits; ++s) v += found(from + (size_t)s * a.r.places * hidden);
    }
    if (p.residual) v = __fadd_rn(__fmul_rn(p.beta, p.residual[t * p.ld_residual + col0 + j]), v);
    p.y[t * p.ldy + col0 + j] = v;
  }
}

inline size_t up256(size_t v) { return (v + 255) / 256 * 256; }

// Parts of K that give the output products of `slots` experts about four workgroups per compute unit; a part keeps a chunk for each wave.
unsigned out_splits_for(const skl_moe_problem *p, unsigned slots) {
  const size_t tiles = (p->hidden + kOutCols - 1) / kOutCols * slots, most = (p->inter + 128 * kWaves - 1) / (128 * kWaves);
  const size_t want = (1024 + tiles - 1) / tiles;
  return (unsigned)(want < 1 ? 1 : want < most ? want : most);
}

// The blocks of scratch memory; with `base` null only their size is found.
size_t lay_out(const skl_moe_problem *p, char *base, Routing *r) {
  const size_t places = p->tokens * p->top_k, slots = p->experts < places ? p->experts : places;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    char *here = base ? base + at : nullptr;
    at += up256(bytes);
    return here;
  };
  r->places = (unsigned)places;
  r->router_splits = (unsigned)((p->hidden + 511) / 512);
  r->out_splits = out_splits_for(p, (unsigned)slots);
  r->parts = reinterpret_cast<float *>(take((size_t)r->router_splits * p->tokens * p->experts * 4));
  r->active = reinterpret_cast<unsigned *>(take(4));
  r->slots = reinterpret_cast<Slot *>(take(slots * sizeof(Slot)));
  r->tokens = reinterpret_cast<uint8_t *>(take(slots * kMaxTokens));
  r->weight = reinterpret_cast<float *>(take(places * 4));
  r->place = reinterpret_cast<unsigned *>(take(places * 4));
  for (uint16_t *&h : r->h) h = reinterpret_cast<uint16_t *>(take(places * p->inter * 2));
  r->out = reinterpret_cast<float *>(take((size_t)r->out_splits * places * p->hidden * 4));
  return at;
}

size_t counters_of(const skl_moe_problem *p) { return 1 + (p->hidden + kOutCols - 1) / kOutCols; }

template <int RG>
int launch_products(const MoeArgs &a, unsigned slots, hipStream_t st) {
  // 32 inner columns per workgroup where that leaves one for every compute unit twice, else 16
  const unsigned wide = (unsigned)(a.p.inter / 32);
  if (wide * slots >= 512) moe_in_kernel<4, RG><<<dim3(wide, slots), kWaves * 64, 0, st>>>(a);
  else moe_in_kernel<2, RG><<<dim3(2 * wide, slots), kWaves * 64, 0, st>>>(a);
  const int rc = skl_check_launch("moe_in");
  if (rc != 0) return rc;
  moe_out_kernel<RG><<<dim3(skl_div_up(a.p.hidden, kOutCols), slots, a.r.out_splits), kWaves * 64, 0, st>>>(a);
  return skl_check_launch("moe_out");
}

int launch_on(const skl_moe_problem *p, char *block, unsigned *counters) {
  MoeArgs a = {*p, {}};
  lay_out(p, block, &a.r);
  a.r.counters = counters;
  const unsigned slots = (unsigned)(p->experts < a.r.places ? p->experts : a.r.places);
  hipStream_t st = skl_current_stream();
  const dim3 grid(skl_div_up(p->experts, 16), skl_div_up(p->tokens, 16), a.r.router_splits);
  if (p->experts <= 64) moe_router_kernel<1><<<grid, kRouterThreads, 0, st>>>(a);
  else if (p->experts <= 128) moe_router_kernel<2><<<grid, kRouterThreads, 0, st>>>(a);
  else if (p->experts <= 256) moe_router_kernel<4><<<grid, kRouterThreads, 0, st>>>(a);
  else moe_router_kernel<16><<<grid, kRouterThreads, 0, st>>>(a);
  const int rc = skl_check_launch("moe_router");
  if (rc != 0) return rc;
  return p->tokens <= 16 ? launch_products<1>(a, slots, st) : launch_products<2>(a, slots, st);
}

}  // namespace

extern "C" int skl_hip_launch_moe(const skl_moe_problem *p) {
  Routing r;
  const size_t bytes = lay_out(p, nullptr, &r), counters = counters_of(p) * sizeof(unsigned);
  const int pending = skl_hip_pending_error();
  int rc;
  skl_hip_sequence_begin();  // the launches hand data on through the stream's scratch memory
  char *block = static_cast<char *>(skl_hip_operand_scratch(bytes));
  unsigned *zeroed = block ? static_cast<unsigned *>(skl_hip_zeroed_sums(counters)) : nullptr;
  char *own = nullptr;
  if (!block || !zeroed) {
    // a stream without scratch memory, or no room for it: a block for this call alone, released once the stream has drained
    own = static_cast<char *>(skl_hip_malloc(bytes + counters));
    if (own && skl_hip_memset(own + bytes, 0, counters) != 0) {
      skl_hip_free(own);
      own = nullptr;
    }
    block = own;
    zeroed = reinterpret_cast<unsigned *>(own + bytes);
  }
  if (block) {
    rc = launch_on(p, block, zeroed);
  } else {
    rc = SKL_HIP_ERR_WORKSPACE;
    skl_hip_withdraw_error(SKL_HIP_ERR_STREAM_SLOTS);
    skl_hip_record_error(rc, "mixture of experts: no scratch memory, y not written");
  }
  skl_hip_sequence_end();
  if (own) {
    skl_hip_synchronize();
    skl_hip_free(own);
    if (rc == 0 && pending != SKL_HIP_ERR_WORKSPACE) skl_hip_withdraw_error(SKL_HIP_ERR_WORKSPACE);
  }
  return rc;
}
