// skl_moe_mxf4.hip - a mixture-of-experts layer over MXFP4 weights for up to 64 tokens (include/skl-gfx950.h has the formulas):
// router, choice, the chosen experts' gated input product, their output product and its weighted sum.
//
// What bounds it is the stream over the chosen experts' weights, half a byte and a thirty-second per value. They are widened in
// registers to bf16 with their scale (v_cvt_scalef32_pk_bf16_fp4, exact) and multiplied by v_mfma_f32_16x16x32_bf16: products of bf16
// values, exact, summed in fp32. A lane's 16 bytes are one block of 32 k of one row of weights; which k of a chunk of 128 meet in which
// of its four instructions is free as long as both operands' lanes take the same.
// The tokens of an expert are gathered: only rows of tokens that chose it are multiplied, 16 at a time. h travels as the sum of three bf16
// values, eight of its 24 bits each (none below 2^-133, where bf16 ends): two left y 1.0e-6 off, three 3e-7, and the stream covers the third's products.
//
// Five launches: the router's sums, the choice, the two products, the weighted sum over a token's experts; but for the choice each with a workgroup per piece of work so
// that the stream finds every compute unit. Every sum has a fixed order.
#include <hip/hip_runtime.h>

#include <atomic>

#include "skl_device.hpp"
#include "skl_mx.h"
#include "../../include/skl-hip.h"

namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));
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
__device__ __forceinline__ unsigned short upper_half(float v) { return (unsigned short)(__float_as_uint(v) >> 16); }  // as a bf16 value: v cut off
__device__ __forceinline__ bool is_number(float v) { return (__float_as_uint(v) & 0x7F800000u) != 0x7F800000u; }

// A logit as a number that orders like it: NaN lowest, the two zeros alike; 0 is none.
__device__ __forceinline__ unsigned order_of(float v) {
  if (v != v) return 1u;
  const unsigned b = __float_as_uint(v + 0.0f);
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(unsigned key) { return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key); }  // the way back; of 1, a NaN
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

template <int G>
__device__ __forceinline__ unsigned max_of(unsigned v) {  // over the G lanes of a token
  if constexpr (G == 64) return wave_max(v);
  v = max_with<0x128, 0xF>(v);  // eight, four, two and one lanes round a row of 16
  v = max_with<0x124, 0xF>(v);
  v = max_with<0x122, 0xF>(v);
  return max_with<0x121, 0xF>(v);
}

// The choice of 64 / G tokens by one wave: NE logits per lane, expert G i + l. A round finds the largest that is left and the lowest expert that has it; the j-th lane keeps
// those of round j, so that exponentials, quotients and stores come once for all rounds. Tokens from `tokens` on: the last one again, not kept.
template <int G, int NE>
__device__ __forceinline__ void choose(const MoeArgs &a, Choice &c, unsigned t, unsigned l) {
  constexpr unsigned kAhead = 8;  // parts of a sum requested together
  const skl_moe_problem &p = a.p;
  const unsigned experts = (unsigned)p.experts, top = (unsigned)p.top_k, splits = a.r.router_splits, tokens = (unsigned)p.tokens;
  float value[NE];
  unsigned key[NE];
#pragma unroll
  for (int i = 0; i < NE; ++i) value[i] = 0.0f;
#pragma unroll 1
  for (unsigned split = 0; split < splits; split += kAhead) {
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      const unsigned e = G * i + l;
      float v[kAhead];
#pragma unroll
      for (unsigned q = 0; q < kAhead; ++q)
        v[q] = a.r.parts[((size_t)(split + q < splits ? split + q : splits - 1) * tokens + (t < tokens ? t : tokens - 1)) * experts + (e < experts ? e : experts - 1)];
#pragma unroll
      for (unsigned q = 0; q < kAhead; ++q)
        if (split + q < splits) value[i] += v[q];
    }
  }
#pragma unroll
  for (int i = 0; i < NE; ++i) key[i] = G * i + l < experts ? order_of(value[i]) : 0;
  unsigned my_key = 0, my_expert = 0;
  for (unsigned j = 0; j < top; ++j) {
    unsigned best = key[0], at = 0;
#pragma unroll
    for (int i = 1; i < NE; ++i)
      if (key[i] > best) best = key[i], at = i;
    const unsigned largest = max_of<G>(best);
    const unsigned e = G == 64 && NE == 1 ? (unsigned)__builtin_ctzll(__ballot(best == largest)) : ~max_of<G>(best == largest ? ~(G * at + l) : 0u);
#pragma unroll
    for (int i = 0; i < NE; ++i) key[i] = G * i + l == e ? 0u : key[i];
    if (l == j) my_key = largest, my_expert = e;
  }
  const float mine = logit_of(my_key), largest = __shfl(mine, 0, G);
  const float x = l < top ? expf(mine - largest) : 0.0f;
  float sum = x;
  if (!p.normalise) {
    sum = 0.0f;
#pragma unroll
    for (int i = 0; i < NE; ++i)
      if (G * i + l < experts) sum += expf(value[i] - largest);
  }
#pragma unroll
  for (int step = G / 2; step > 0; step >>= 1) sum += __shfl_xor(sum, step, 64);
  if (l < top && t < tokens) {
    c.share[t * top + l] = x / sum;
    c.chosen[t * top + l] = (unsigned short)my_expert;
    atomicOr(&c.mask[my_expert][t >> 5], 1u << (t & 31u));
  }
}

// The router's sums: a workgroup takes 16 experts, 16 tokens and 512 of hidden, a wave 32 of these. 3.5 us for 1 token of 32 x 2048, 4.7 for 64 of 8 x 4096: a launch and a latency.
__global__ void __launch_bounds__(kRouterThreads) moe_router_kernel(MoeArgs a) {
  __shared__ float red[kRouterThreads / 64][16][17];
  const skl_moe_problem &p = a.p;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, l = lane & 15, g = lane >> 4;
  const size_t e0 = (size_t)blockIdx.x * 16, t0 = (size_t)blockIdx.y * 16, k = (size_t)blockIdx.z * 512 + 32 * (size_t)wave;
  const size_t er = e0 + l < p.experts ? e0 + l : p.experts - 1, tr = t0 + l < p.tokens ? t0 + l : p.tokens - 1;
  v4f acc = {0.0f, 0.0f, 0.0f, 0.0f};
  if (k < p.hidden)
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*reinterpret_cast<const v8bf *>(p.x + tr * p.ldx + k + 8 * g),
                                                  *reinterpret_cast<const v8bf *>(p.router + er * p.ld_router + k + 8 * g), acc, 0, 0, 0);
#pragma unroll
  for (int r = 0; r < 4; ++r) red[wave][4 * g + r][l] = acc[r];
  __syncthreads();
  if (threadIdx.x >= 256) return;
  const unsigned i = threadIdx.x >> 4, j = threadIdx.x & 15;
  float v = 0.0f;
#pragma unroll
  for (int w = 0; w < kRouterThreads / 64; ++w) v += red[w][i][j];
  if (t0 + i < p.tokens && e0 + j < p.experts) a.r.parts[((size_t)blockIdx.z * p.tokens + t0 + i) * p.experts + e0 + j] = v;
}

// The choice: one workgroup, of a wave per token or, for many tokens and not too many experts, per four, and a thread per expert, as far as there are that many. 3.5 us for 1
// token, for 64 tokens 5.8 (4 of 20 experts) and 11 (8 of 128; 10 and 22 with a wave per token), 54 of 512, bound by what follows one another: the sums read back, top_k rounds of
// two maxima, a scan; beyond 256 experts, with 16 logits and their keys to a lane, 15 of the 128 registers that 1024 threads leave are in scratch memory besides. (Behind a counter in the router's last workgroup the layer took as long, to 2 %.)
template <int G, int NE>
__global__ void __launch_bounds__(kRouterThreads) moe_choice_kernel(MoeArgs a) {
  __shared__ Choice c;
  const skl_moe_problem &p = a.p;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const unsigned threads = blockDim.x, top = (unsigned)p.top_k, tokens = (unsigned)p.tokens, e = threadIdx.x;
  c.mask[e][0] = c.mask[e][1] = 0;  // one thread per expert
  __syncthreads();
  constexpr unsigned kEach = 64 / G;
  for (unsigned first = wave * kEach; first < tokens; first += threads / 64 * kEach) choose<G, NE>(a, c, first + lane / G, lane % G);
  __syncthreads();
  // Where each expert's tokens begin, and its slot: one scan over the experts, the count in the lower half, the slot in the upper.
  const unsigned count = __popc(c.mask[e][0]) + __popc(c.mask[e][1]), own = count | (count ? 0x10000u : 0u);
  unsigned scan = own;
#pragma unroll
  for (int step = 1; step < 64; step <<= 1) {
    const unsigned other = __shfl_up(scan, step, 64);
    if (lane >= step) scan += other;
  }
  if (lane == 63) c.totals[wave] = scan;
  __syncthreads();
  for (int w = 0; w < wave; ++w) scan += c.totals[w];
  c.start[e] = (scan - own) & 0xFFFFu;
  c.slot[e] = (unsigned short)((scan - own) >> 16);
  if (count) a.r.slots[c.slot[e]] = Slot{e, c.start[e], count, 0};
  if (e == threads - 1) *a.r.active = scan >> 16;
  __syncthreads();
  for (unsigned at = threadIdx.x; at < tokens * top; at += threads) {
    const unsigned t = at / top, chosen = c.chosen[at], below = (1u << (t & 31u)) - 1u;
    const unsigned before = t < 32 ? __popc(c.mask[chosen][0] & below) : __popc(c.mask[chosen][0]) + __popc(c.mask[chosen][1] & below);
    const unsigned place = c.start[chosen] + before;
    a.r.tokens[c.slot[chosen] * kMaxTokens + before] = (uint8_t)t;
    a.r.weight[place] = c.share[at];
    a.r.place[at] = place;
    if (p.ids) p.ids[at] = (int32_t)chosen;
    if (p.weights) p.weights[at] = c.share[at];
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// The two products. A workgroup of eight waves has 64 CG rows of one expert's weights - columns of the result - and up to 16 RG of its tokens at a time. K comes in
// chunks of 256, a line of a row of weights and four (TERMS times) of a token, from memory to LDS without registers, whole lines at a time, a few chunks ahead. Four
// pairs of waves have 16 CG rows of weights each; of a pair, each has its half of every chunk, so that a token is read from LDS four times and not eight.
// 64 tokens, 2 of 8 experts of 14336 x 4096: 113 us for h (500 MB of weights, 4.4 TB/s) and 94 to 110 for the output products (250 MB and three terms of h, of which
// each workgroup has to have all; the more, the more experts have over 16 tokens). Read straight into registers as the operands lie - 16 lines for 1024 bytes, and as many for every token's - the compute
// units' address paths bound them: 193 and 205 us. 7 tokens, 3 of 20 experts of 1440 x 2080: 16.6 and 11.4 us; 1 token, 4 of 32 of 1024 x 2048: 7.8 and 5.6, most of
// it the way to a launch's first bytes. There, with one group of 16 tokens, a wave reads a chunk's operands together (step by step, below, 17.7 and 8.4 us for h);
// weights past the caches took 20 us at 7 tokens, whose rows of 1040 bytes share lines.
// ---------------------------------------------------------------------------------------------------------------------
typedef __attribute__((address_space(3))) char lds_char;
typedef unsigned unsigned_any __attribute__((aligned(1)));
constexpr int kWaves = 8, kThreads = kWaves * 64, kChunk = 256, kLine = 128;
constexpr unsigned kRange = 0x7FFFFFF0u, kOutside = 0x7FFFFFF0u;  // of a buffer descriptor; an offset that loads zeros

template <int CG_, int RG_, int TERMS_>
struct Shape {
  static constexpr int CG = CG_, RG = RG_, TERMS = TERMS_;
  static constexpr int kAll = 64 * CG;  // rows of weights
  static constexpr int kWeightBytes = kAll * kLine, kTokenBytes = TERMS * 16 * RG * 512;  // of a chunk
  // Two rings, that of the weights the deeper one: they come from memory, the tokens from a cache. Both for two workgroups per compute unit where two chunks of each fit.
  static constexpr int kBudget = (2 * (kWeightBytes + kTokenBytes) <= 80 * 1024 ? 80 : 160) * 1024;
  static constexpr int kFit = (kBudget - 2 * kTokenBytes) / kWeightBytes, kWeightStages = kFit < 4 ? kFit : 4;
  static constexpr int kRest = (kBudget - kWeightStages * kWeightBytes) / kTokenBytes, kTokenStages = kRest < kWeightStages ? kRest : kWeightStages;
  static constexpr int kLoads = CG + RG * TERMS;  // requests of a wave per chunk
  // With rings of one depth a chunk's weights are requested before its tokens, else behind them: what may be under way when the next chunk has to be there.
  static constexpr bool kTokensFirst = kWeightStages > kTokenStages;
  static constexpr int kUnderWay = (kTokenStages - 2) * kLoads + (kTokensFirst ? CG : 0);
  static constexpr int kTokensAt = kWeightStages * kWeightBytes, kLds = kTokensAt + kTokenStages * kTokenBytes;
  static constexpr int kPitch = kAll + 1;  // of the sums, which meet in the rings' place
  static_assert(kTokenStages >= 2 && 16 * RG * kPitch * 4 <= kLds && kUnderWay + kLoads < 63);
};

// One step: acc[r][c] += x[r][t] b[c] over G groups of tokens, T terms and CG groups of columns, while the tokens' values of the next step come from `px` on into n - and,
// if that is the first of a chunk, its weights from `pw` into w. The wait is the block's own: the compiler would make every read of LDS wait for all requests under way.
#define SKL_MOE_MUL(a, x, b) "v_mfma_f32_16x16x32_bf16 %[" a "], %[" x "], %[" b "], %[" a "]\n"
#define SKL_MOE_M2(c, t) SKL_MOE_MUL("a0" #c, "x0" #t, "b" #c) SKL_MOE_MUL("a1" #c, "x1" #t, "b" #c)
#define SKL_MOE_C1(G, t) SKL_MOE_M##G(0, t)
#define SKL_MOE_C2(G, t) SKL_MOE_C1(G, t) SKL_MOE_M##G(1, t)
#define SKL_MOE_T1(C, G) SKL_MOE_C##C(G, 0)
#define SKL_MOE_T3(C, G) SKL_MOE_C##C(G, 0) SKL_MOE_C##C(G, 1) SKL_MOE_C##C(G, 2)
#define SKL_MOE_RX(r, t) "ds_read_b128 %[n" #r #t "], %[px] offset:%c[o" #r #t "]\n"
#define SKL_MOE_RX21 SKL_MOE_RX(0, 0) SKL_MOE_RX(1, 0)
#define SKL_MOE_RX23 SKL_MOE_RX21 SKL_MOE_RX(0, 1) SKL_MOE_RX(1, 1) SKL_MOE_RX(0, 2) SKL_MOE_RX(1, 2)
#define SKL_MOE_RW1 "ds_read_b128 %[w0], %[pw]\n"
#define SKL_MOE_RW2 SKL_MOE_RW1 "ds_read_b128 %[w1], %[pw] offset:2048\n"
#define SKL_MOE_A(r, c) [a##r##c] "+v"(acc[r][c])
#define SKL_MOE_A12 SKL_MOE_A(0, 0), SKL_MOE_A(1, 0)
#define SKL_MOE_A22 SKL_MOE_A12, SKL_MOE_A(0, 1), SKL_MOE_A(1, 1)
#define SKL_MOE_N(r, t) [n##r##t] "=&v"(n[r][t])
#define SKL_MOE_N21 SKL_MOE_N(0, 0), SKL_MOE_N(1, 0)
#define SKL_MOE_N23 SKL_MOE_N21, SKL_MOE_N(0, 1), SKL_MOE_N(1, 1), SKL_MOE_N(0, 2), SKL_MOE_N(1, 2)
#define SKL_MOE_X(r, t) [x##r##t] "v"(x[r][t])
#define SKL_MOE_X21 SKL_MOE_X(0, 0), SKL_MOE_X(1, 0)
#define SKL_MOE_X23 SKL_MOE_X21, SKL_MOE_X(0, 1), SKL_MOE_X(1, 1), SKL_MOE_X(0, 2), SKL_MOE_X(1, 2)
#define SKL_MOE_W(c) [w##c] "=&v"(w[c])
#define SKL_MOE_W1 SKL_MOE_W(0)
#define SKL_MOE_W2 SKL_MOE_W1, SKL_MOE_W(1)
#define SKL_MOE_B(c) [b##c] "v"(b[c])
#define SKL_MOE_B1 SKL_MOE_B(0)
#define SKL_MOE_B2 SKL_MOE_B1, SKL_MOE_B(1)
#define SKL_MOE_OFFSETS [o00] "n"(0), [o01] "n"(TERM), [o02] "n"(2 * TERM), [o10] "n"(8192), [o11] "n"(8192 + TERM), [o12] "n"(8192 + 2 * TERM)
#define SKL_MOE_STEP(C, G, T)                                                                                                                                          \
  if constexpr (CG == C && GROUPS == G && TERMS == T) {                                                                                                                \
    if constexpr (LAST)                                                                                                                                                \
      asm volatile("s_nop 1\n" SKL_MOE_RW##C SKL_MOE_RX##G##T SKL_MOE_T##T(C, G) "s_waitcnt lgkmcnt(0)"                                                                \
                   : SKL_MOE_A##C##G, SKL_MOE_N##G##T, SKL_MOE_W##C : SKL_MOE_X##G##T, SKL_MOE_B##C, SKL_MOE_OFFSETS, [px] "v"(px), [pw] "v"(pw) : "memory");          \
    else                                                                                                                                                               \
      asm volatile("s_nop 1\n" SKL_MOE_RX##G##T SKL_MOE_T##T(C, G) "s_waitcnt lgkmcnt(0)"                                                                              \
                   : SKL_MOE_A##C##G, SKL_MOE_N##G##T : SKL_MOE_X##G##T, SKL_MOE_B##C, SKL_MOE_OFFSETS, [px] "v"(px) : "memory");                                      \
  }
#define SKL_MOE_READ(C, G, T)                                                                                                                                          \
  if constexpr (CG == C && GROUPS == G && TERMS == T)                                                                                                                  \
    asm volatile(SKL_MOE_RW##C SKL_MOE_RX##G##T "s_waitcnt lgkmcnt(0)" : SKL_MOE_N##G##T, SKL_MOE_W##C : SKL_MOE_OFFSETS, [px] "v"(px), [pw] "v"(pw) : "memory");
#define SKL_MOE_EACH(F) \
  F(1, 2, 1) F(2, 2, 1) F(1, 2, 3) F(2, 2, 3)
template <int CG, int RG, int TERMS, int GROUPS, bool LAST>
__device__ __forceinline__ void step(v4f (&acc)[RG][CG], const v4i (&x)[GROUPS][TERMS], const v8bf (&b)[CG], v4i (&n)[GROUPS][TERMS], v4i (&w)[CG], unsigned px, unsigned pw) {
  constexpr int TERM = 16 * RG * 512;
  SKL_MOE_EACH(SKL_MOE_STEP)
}
template <int CG, int RG, int TERMS, int GROUPS>
__device__ __forceinline__ void read_first(v4i (&n)[GROUPS][TERMS], v4i (&w)[CG], unsigned px, unsigned pw) {
  constexpr int TERM = 16 * RG * 512;
  SKL_MOE_EACH(SKL_MOE_READ)
}

// All that a wave takes of a chunk of one group of tokens: TERMS terms TERM bytes apart, four pieces each, whose places are those at `px`.
#define SKL_MOE_P(t) \
  "ds_read_b128 %[n" #t "0], %[p0] offset:%c[o" #t "]\nds_read_b128 %[n" #t "1], %[p1] offset:%c[o" #t "]\nds_read_b128 %[n" #t "2], %[p2] offset:%c[o" #t "]\nds_read_b128 %[n" #t "3], %[p3] offset:%c[o" #t "]\n"
#define SKL_MOE_Q(t) [n##t##0] "=&v"(x[t][0]), [n##t##1] "=&v"(x[t][1]), [n##t##2] "=&v"(x[t][2]), [n##t##3] "=&v"(x[t][3])
#define SKL_MOE_P1 SKL_MOE_P(0)
#define SKL_MOE_P3 SKL_MOE_P(0) SKL_MOE_P(1) SKL_MOE_P(2)
#define SKL_MOE_Q1 SKL_MOE_Q(0)
#define SKL_MOE_Q3 SKL_MOE_Q(0), SKL_MOE_Q(1), SKL_MOE_Q(2)
#define SKL_MOE_CHUNK(C, T)                                                                                                                                     \
  if constexpr (CG == C && TERMS == T)                                                                                                                          \
    asm volatile(SKL_MOE_RW##C SKL_MOE_P##T "s_waitcnt lgkmcnt(0)" : SKL_MOE_W##C, SKL_MOE_Q##T                                                                 \
                 : [p0] "v"(px[0]), [p1] "v"(px[1]), [p2] "v"(px[2]), [p3] "v"(px[3]), [pw] "v"(pw), [o0] "n"(0), [o1] "n"(TERM), [o2] "n"(2 * TERM) : "memory");
template <int CG, int TERMS, int TERM>
__device__ __forceinline__ void read_chunk(v4i (&x)[TERMS][4], v4i (&w)[CG], const unsigned (&px)[4], unsigned pw) {
  SKL_MOE_CHUNK(1, 1) SKL_MOE_CHUNK(2, 1) SKL_MOE_CHUNK(1, 3) SKL_MOE_CHUNK(2, 3)
}

// What a wave's lanes hold of weights and tokens while they stream.
template <class S>
struct Operands {
  const uint8_t *codes;          // the first row of weights that the wave requests
  unsigned off[S::CG];           // the lane's offsets from there, requests of eight lines
  const uint8_t *scales[S::CG];  // of the rows of weights that the lane multiplies
  const uint16_t *tokens[S::TERMS];
  unsigned at[S::RG];            // the lane's offsets from there: of request i, the pieces of row 2 (RG wave + i) + lane / 32
};

// The place of a token's 16-byte piece in its row of 32: reads of 16 rows with the same pieces meet in no bank (they are served rows 0 to 3 and 12 to 15 of one lane
// group with rows 4 to 11 of the next).
__device__ __forceinline__ unsigned turn_of(unsigned row) { return (row + 12u) & 15u; }
template <class S>
__device__ __forceinline__ unsigned row_of(int i, int wave, int lane) { return 2u * ((unsigned)wave * S::RG + i) + ((unsigned)lane >> 5); }
__device__ __forceinline__ unsigned piece_of(unsigned row, int lane) { return ((unsigned)lane & 16u) | (((unsigned)lane ^ turn_of(row)) & 15u); }

// acc[r][c] of the wave's rows of weights and its halves of the chunks in [begin, stop), `total` values in a row.
template <class S, int GROUPS>
__device__ __forceinline__ void multiply(const Operands<S> &o, v4f (&acc)[S::RG][S::CG], unsigned begin, unsigned stop, unsigned total, int wave, int lane, lds_char *stages) {
  constexpr int CG = S::CG, RG = S::RG, TERMS = S::TERMS;
  const int l = lane & 15, g = lane >> 4, pair = wave & 3, half = wave >> 2;
  const unsigned per_row = total / 32, base = (unsigned)(uintptr_t)stages;
  const unsigned piece = ((unsigned)lane & 7u) ^ ((unsigned)lane >> 3);  // of a line of weights: slot s of row r holds piece s ^ (r % 8)
  const auto request_weights = [&](unsigned chunk) __attribute__((always_inline)) {
    lds_char *const to = stages + (chunk - begin) % S::kWeightStages * S::kWeightBytes;
    const unsigned byte = chunk * kLine;
    const bool in = chunk < stop && byte + piece * 16u < total / 2;
    const __amdgpu_buffer_rsrc_t w = __builtin_amdgcn_make_buffer_rsrc((void *)(o.codes + byte), 0, (int)kRange, 0x00027000);
#pragma unroll
    for (int i = 0; i < CG; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(w, (__attribute__((address_space(3))) void *)(to + (wave * CG + i) * 8 * kLine), 16, (int)(in ? o.off[i] : kOutside), 0, 0, 0);
  };
  const auto request_tokens = [&](unsigned chunk) __attribute__((always_inline)) {
    lds_char *const to = stages + S::kTokensAt + (chunk - begin) % S::kTokenStages * S::kTokenBytes;
#pragma unroll
    for (int t = 0; t < TERMS; ++t) {
      const __amdgpu_buffer_rsrc_t x = __builtin_amdgcn_make_buffer_rsrc((void *)(o.tokens[t] + chunk * kChunk), 0, (int)kRange, 0x00027000);
#pragma unroll
      for (int i = 0; i < RG; ++i) {
        const bool there = chunk < stop && chunk * kChunk + 8u * piece_of(row_of<S>(i, wave, lane), lane) < total;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(x, (__attribute__((address_space(3))) void *)(to + t * (S::kTokenBytes / TERMS) + (wave * RG + i) * 1024), 16,
                                                 (int)(there ? o.at[i] : kOutside), 0, 0, 0);
      }
    }
  };
  const auto request = [&](int chunk) __attribute__((always_inline)) {  // when chunk `chunk` has been read, counted from the first
    if constexpr (S::kTokensFirst) request_tokens(begin + (unsigned)(chunk + S::kTokenStages));
    request_weights(begin + (unsigned)(chunk + S::kWeightStages));
    if constexpr (!S::kTokensFirst) request_tokens(begin + (unsigned)(chunk + S::kTokenStages));
  };
  // A row has four scale bytes in the half of a chunk. Lane group g loads those of the g-th of four chunks to come, from further down where the row ends - past its end they
  // become zeros, like the codes. They are moved into place late: a use waits for the load.
  const auto want_of = [&](unsigned chunk) { return (chunk + (unsigned)g) * 8u + 4u * (unsigned)half; };
  const uint8_t *from[CG];
  const auto load_scales = [&](unsigned (&s)[CG], unsigned chunk) __attribute__((always_inline)) {
    const unsigned want = want_of(chunk), at = per_row < 4 ? 0u : want + 4 <= per_row ? want : per_row - 4;
#pragma unroll
    for (int c = 0; c < CG; ++c) s[c] = *(const __attribute__((address_space(1))) unsigned_any *)(from[c] + at);  // (not through a flat load, which a wait for LDS waits for)
  };
  const auto place_scales = [&](unsigned (&s)[CG], const unsigned (&v)[CG], unsigned chunk) __attribute__((always_inline)) {
    const unsigned want = want_of(chunk), over = per_row < 4 || want + 4 <= per_row ? 0u : want >= per_row ? 32u : 8u * (want + 4 - per_row);
#pragma unroll
    for (int c = 0; c < CG; ++c) s[c] = over > 31 ? 0u : v[c] >> over;
  };
  unsigned raw[CG], ahead[CG], four[CG];  // scales as they were loaded, of four chunks, of the next four
#pragma unroll
  for (int c = 0; c < CG; ++c) from[c] = o.scales[c];
  if (per_row >= 4) {
    load_scales(raw, begin);
  } else {  // a row of one chunk, which is shorter than a load; what is loaded ahead of others is not used
#pragma unroll
    for (int c = 0; c < CG; ++c) {
      raw[c] = 0;
      for (unsigned i = 0; want_of(0) + i < per_row; ++i) raw[c] |= (unsigned)o.scales[c][want_of(0) + i] << (8 * i);
      from[c] = o.codes;
    }
  }
  load_scales(ahead, begin + 4);
  const auto factors = [&](float (&f)[CG], unsigned chunk) __attribute__((always_inline)) {
#pragma unroll
    for (int c = 0; c < CG; ++c) {
      const unsigned s = (unsigned)__builtin_amdgcn_ds_bpermute((int)(4 * l + 64 * ((chunk - begin) & 3u)), (int)four[c]);  // the lane group's that has this chunk
      f[c] = __uint_as_float(__builtin_amdgcn_ubfe(s, 8u * (unsigned)g, 8u) << 23);
    }
  };
  v4i w[CG];
  const auto widen = [&](v8bf (&b)[CG], const float (&f)[CG], int j) __attribute__((always_inline)) {
#pragma unroll
    for (int c = 0; c < CG; ++c) b[c] = widen_f4((unsigned)w[c][j], f[c]);
  };
  const unsigned at_w = base + (pair * CG * 16 + l) * kLine + (unsigned)((4 * half + g) ^ (l & 7)) * 16u;
  const unsigned at_x = base + S::kTokensAt + l * 512 + 256 * half + ((4u * g) ^ turn_of(l)) * 16u;
  unsigned at = 0, stage = 0;  // where the chunk's weights and tokens are in their rings
  const auto advance = [&]() __attribute__((always_inline)) {
    at = at == (S::kWeightStages - 1) * S::kWeightBytes ? 0 : at + S::kWeightBytes;
    stage = stage == (S::kTokenStages - 1) * S::kTokenBytes ? 0 : stage + S::kTokenBytes;
  };
#pragma unroll
  for (int c = 0; c < S::kWeightStages - S::kTokenStages; ++c) request_weights(begin + (unsigned)c);
#pragma unroll
  for (int c = 0; c < S::kTokenStages - 1; ++c) request(c - S::kTokenStages);
  if constexpr (GROUPS == 1) {
    // Little to multiply: a chunk's operands are read together and waited for once. Its stages' predecessors are free behind the barrier.
#pragma unroll 1
    for (unsigned chunk = begin; chunk < stop; ++chunk) {
      __builtin_amdgcn_sched_barrier(0);
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(S::kUnderWay) : "memory");
      __builtin_amdgcn_s_barrier();
      if (((chunk - begin) & 3u) == 0) {
        if (chunk == begin) {
          place_scales(four, raw, chunk);
        } else {
          place_scales(four, ahead, chunk);
          load_scales(ahead, chunk + 4);
        }
      }
      request((int)(chunk - begin) - 1);
      __builtin_amdgcn_sched_barrier(0);
      v4i x[TERMS][4];
      const unsigned px[4] = {at_x + stage, (at_x ^ 16u) + stage, (at_x ^ 32u) + stage, (at_x ^ 48u) + stage};
      read_chunk<CG, TERMS, 16 * RG * 512>(x, w, px, at_w + at);
      float f[CG];
      factors(f, chunk);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v8bf b[CG];
        widen(b, f, j);
#pragma unroll
        for (int t = 0; t < TERMS; ++t)
#pragma unroll
          for (int c = 0; c < CG; ++c) acc[0][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, x[t][j]), b[c], acc[0][c], 0, 0, 0);
      }
      advance();
    }
  } else {
    // Four steps of 32 k (8 from each lane group's block): the products of one run while the operands of the next come from LDS.
    request(-1);
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(S::kUnderWay + S::kLoads) : "memory");
    __builtin_amdgcn_s_barrier();
    place_scales(four, raw, begin);
    v4i x0[GROUPS][TERMS], x1[GROUPS][TERMS];
    read_first<CG, RG, TERMS, GROUPS>(x0, w, at_x, at_w);
#pragma unroll 1
    for (unsigned chunk = begin; chunk < stop; ++chunk) {
      float f[CG];
      factors(f, chunk);
      v8bf b[CG];
      v4i none[CG];
      widen(b, f, 0);
      step<CG, RG, TERMS, GROUPS, false>(acc, x0, b, x1, none, (at_x ^ 16u) + stage, 0);
      widen(b, f, 1);
      step<CG, RG, TERMS, GROUPS, false>(acc, x1, b, x0, none, (at_x ^ 32u) + stage, 0);
      widen(b, f, 2);
      step<CG, RG, TERMS, GROUPS, false>(acc, x0, b, x1, none, (at_x ^ 48u) + stage, 0);
      widen(b, f, 3);
      // Every wave has read all of this chunk; the next one is there once the requests of all waves for it are. Then this one's stages are free.
      __builtin_amdgcn_sched_barrier(0);
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(S::kUnderWay) : "memory");
      __builtin_amdgcn_s_barrier();
      if (((chunk - begin) & 3u) == 3) {
        place_scales(four, ahead, chunk + 1);
        load_scales(ahead, chunk + 5);
      }
      request((int)(chunk - begin));
      __builtin_amdgcn_sched_barrier(0);
      advance();
      step<CG, RG, TERMS, GROUPS, true>(acc, x1, b, x0, w, at_x + stage, at_w + at);
    }
#pragma unroll
    for (int r = 0; r < GROUPS; ++r)
#pragma unroll
      for (int c = 0; c < CG; ++c) asm volatile("s_nop 15" : "+v"(acc[r][c]));  // the last products' results, before anything but a product reads them
  }
}

// red[row of tokens][row of weights] = their products over k in [first, end), first a multiple of 256, `total` values in all.
template <class S>
__device__ __forceinline__ void stream(const Operands<S> &o, unsigned first, unsigned end, unsigned total, int wave, int lane, unsigned groups, char *lds) {
  const int l = lane & 15, g = lane >> 4, pair = wave & 3, half = wave >> 2;
  const unsigned begin = first / kChunk, stop = (end + kChunk - 1) / kChunk;
  v4f acc[S::RG][S::CG];
#pragma unroll
  for (int r = 0; r < S::RG; ++r)
#pragma unroll
    for (int c = 0; c < S::CG; ++c) acc[r][c] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  if (begin < stop) {  // the same for every wave
    if (S::RG == 2 && groups > 1) multiply<S, S::RG>(o, acc, begin, stop, total, wave, lane, (lds_char *)lds);
    else multiply<S, 1>(o, acc, begin, stop, total, wave, lane, (lds_char *)lds);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the requests behind the last chunk write zeros into the rings
  __syncthreads();
  float(*red)[S::kPitch] = reinterpret_cast<float(*)[S::kPitch]>(lds);
#pragma unroll
  for (int turn = 0; turn < 2; ++turn) {
    if (half == turn) {
#pragma unroll
      for (int r = 0; r < S::RG; ++r)
#pragma unroll
        for (int c = 0; c < S::CG; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float &to = red[16 * r + 4 * g + i][(pair * S::CG + c) * 16 + l];
            to = turn ? to + acc[r][c][i] : acc[r][c][i];
          }
    }
    __syncthreads();
  }
}

// Rows of weights of one matrix from `row0` on, of which `rows` exist (others are the last one again: computed, not used): those that the lane requests, from `mine` on, and
// those that it multiplies, from `part` on.
template <class S>
__device__ __forceinline__ void set_codes(Operands<S> &o, const skl_mx_operand &op, size_t expert, size_t row0, int rows, int mine, int lane) {
  const int from = mine < rows ? mine : rows - 1;
  const unsigned long long at = (unsigned long long)(uintptr_t)(op.codes + (expert + (row0 + from) * op.ld) / 2);
  // spelled out as a scalar: a descriptor in vector registers costs a loop over the lanes per load
  o.codes = (const uint8_t *)(uintptr_t)(((unsigned long long)(unsigned)__builtin_amdgcn_readfirstlane((int)(at >> 32)) << 32) | (unsigned)__builtin_amdgcn_readfirstlane((int)at));
#pragma unroll
  for (int i = 0; i < S::CG; ++i) {
    const int r = mine + 8 * i + (lane >> 3);
    o.off[i] = (unsigned)((r < rows ? r : rows - 1) - from) * (unsigned)(op.ld / 2) + (((unsigned)lane & 7u) ^ ((unsigned)lane >> 3)) * 16u;
  }
}
template <class S>
__device__ __forceinline__ void set_scales(Operands<S> &o, const skl_mx_operand &op, size_t expert, size_t row0, int rows, int part, int lane) {
#pragma unroll
  for (int c = 0; c < S::CG; ++c) {
    const int r = part + 16 * c + (lane & 15);
    o.scales[c] = op.scales + expert + (row0 + (r < rows ? r : rows - 1)) * op.lds;
  }
}
// The lane's pieces of the rows of tokens that it requests: row n at of(i, n) elements from the first; rows from `count` on are not requested.
template <class S, class F>
__device__ __forceinline__ void set_tokens(Operands<S> &o, unsigned count, int wave, int lane, F of) {
#pragma unroll
  for (int i = 0; i < S::RG; ++i) {
    const unsigned row = row_of<S>(i, wave, lane);
    o.at[i] = row < count ? 2u * of(i, row) + 16u * piece_of(row, lane) : kOutside;
  }
}

__device__ __forceinline__ Slot scalar(Slot s) {
  return Slot{(unsigned)__builtin_amdgcn_readfirstlane((int)s.expert), (unsigned)__builtin_amdgcn_readfirstlane((int)s.first), (unsigned)__builtin_amdgcn_readfirstlane((int)s.count), 0};
}

// h of 32 CG inner columns of one expert (blockIdx.y: its slot): half of the rows of weights are rows of gate, half of up.
template <int CG, int RG>
__global__ void __launch_bounds__(kThreads) moe_in_kernel(MoeArgs a) {
  using S = Shape<CG, RG, 1>;
  constexpr int kCols = 32 * CG;
  extern __shared__ __attribute__((aligned(1024))) char moe_lds[];
  const skl_moe_problem &p = a.p;
  const unsigned slot = blockIdx.y;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const Slot own = scalar(a.r.slots[slot]);
  const unsigned active = *a.r.active;
  unsigned token[RG];  // of the rows that the lane requests, in the first pass: asked for with the slot, not behind it
#pragma unroll
  for (int i = 0; i < RG; ++i) token[i] = a.r.tokens[slot * kMaxTokens + row_of<S>(i, wave, lane)];
  if (slot >= active) return;
  const unsigned col0 = blockIdx.x * kCols, inter = (unsigned)p.inter, cols = inter - col0 < (unsigned)kCols ? inter - col0 : kCols;
  Operands<S> o;
  set_codes(o, wave < 4 ? p.gate : p.up, own.expert * p.expert_in, col0, (int)cols, wave % 4 * 8 * CG, lane);
  set_scales(o, wave % 4 < 2 ? p.gate : p.up, own.expert * p.expert_in_scales, col0, (int)cols, wave % 2 * 16 * CG, lane);
  o.tokens[0] = p.x;
  for (unsigned done = 0; done < own.count; done += RG * 16) {  // more tokens than a pass takes: the weights again
    const unsigned left = own.count - done, here = left < RG * 16 ? left : RG * 16;
    if (done != 0) {
#pragma unroll
      for (int i = 0; i < RG; ++i) {
        const unsigned row = row_of<S>(i, wave, lane);
        token[i] = a.r.tokens[slot * kMaxTokens + done + (row < here ? row : 0)];
      }
    }
    set_tokens(o, here, wave, lane, [&](int i, unsigned) { return token[i] * (unsigned)p.ldx; });
    stream<S>(o, 0, (unsigned)p.hidden, (unsigned)p.hidden, wave, lane, (here + 15) / 16, moe_lds);
    const float(*red)[S::kPitch] = reinterpret_cast<const float(*)[S::kPitch]>(moe_lds);
    for (unsigned n = threadIdx.x; n < here * kCols; n += kThreads) {
      const unsigned i = n / kCols, j = n % kCols;
      if (j >= cols) continue;
      const unsigned place = own.first + done + i;
      const float h = skl_activate(red[i][j], p.activation) * red[i][kCols + j] * a.r.weight[place];
      // Its bits from the top, eight to a term: none is larger than what is left, so that neither a term nor a sum of the first two is an infinity where h is none. (The nearest
      // bf16 value is, from 2^128 - 2^119 on.) An infinity or a NaN - the arithmetic's have their upper half's bits set - has no other terms.
      const unsigned short t0 = upper_half(h);
      const float rest = is_number(h) ? h - of_bf16(t0) : 0.0f;
      const unsigned short t1 = upper_half(rest);
      const size_t to = (size_t)place * p.inter + col0 + j;
      a.r.h[0][to] = t0;
      a.r.h[1][to] = t1;
      a.r.h[2][to] = bf16_of(rest - of_bf16(t1));
    }
    __syncthreads();
  }
}

// The output products of 64 CG columns, one expert and one part of K.
template <int CG, int RG>
__global__ void __launch_bounds__(kThreads) moe_out_kernel(MoeArgs a) {
  using S = Shape<CG, RG, 3>;
  constexpr int kCols = S::kAll;
  extern __shared__ __attribute__((aligned(1024))) char moe_lds[];
  const skl_moe_problem &p = a.p;
  const unsigned slot = blockIdx.y, split = blockIdx.z;
  const Slot own = scalar(a.r.slots[slot]);
  const unsigned active = *a.r.active;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (slot >= active) return;
  const unsigned hidden = (unsigned)p.hidden, inter = (unsigned)p.inter, col0 = blockIdx.x * kCols, cols = hidden - col0 < (unsigned)kCols ? hidden - col0 : kCols;
  const unsigned chunks = (inter + kChunk - 1) / kChunk;
  const unsigned begin = chunks * split / a.r.out_splits * kChunk, stop = chunks * (split + 1) / a.r.out_splits * kChunk, end = stop < inter ? stop : inter;
  Operands<S> o;
  set_codes(o, p.down, own.expert * p.expert_down, col0, (int)cols, wave * 8 * CG, lane);
  set_scales(o, p.down, own.expert * p.expert_down_scales, col0, (int)cols, wave % 4 * 16 * CG, lane);
  for (unsigned done = 0; done < own.count; done += RG * 16) {
    const unsigned left = own.count - done, here = left < RG * 16 ? left : RG * 16;
    const size_t place = own.first + done;
#pragma unroll
    for (int t = 0; t < 3; ++t) o.tokens[t] = a.r.h[t] + place * inter;
    set_tokens(o, here, wave, lane, [&](int, unsigned row) { return row * inter; });
    stream<S>(o, begin, end, inter, wave, lane, (here + 15) / 16, moe_lds);
    const float(*red)[S::kPitch] = reinterpret_cast<const float(*)[S::kPitch]>(moe_lds);
    for (unsigned n = threadIdx.x; n < here * (kCols / 2); n += kThreads) {
      const unsigned i = n / (kCols / 2), j = n % (kCols / 2) * 2;
      if (j < cols) *reinterpret_cast<v2f *>(a.r.out + ((size_t)split * a.r.places + place + i) * hidden + col0 + j) = v2f{red[i][j], red[i][j + 1]};
    }
    __syncthreads();
  }
}

// y: two columns of a token to a thread. 3.3 to 5 us, a launch and a latency. (Left to the workgroup that is the last of its columns, the sum took 2 us more at 1 token,
// 5 at 7 and 35 at 64 tokens of 128 experts, whose output products are 4 MiB.)
__global__ void __launch_bounds__(256) moe_sum_kernel(MoeArgs a) {
  const unsigned j = (blockIdx.x * 256u + threadIdx.x) * 2u;
  if (j >= a.p.hidden) return;
  const skl_moe_problem &p = a.p;
  const unsigned t = blockIdx.y, terms = (unsigned)p.top_k * a.r.out_splits;
  v2f v = {0.0f, 0.0f};
  for (unsigned q = 0; q < terms; q += 8) {  // by choice, then by part of K; requested together
    v2f part[8];
#pragma unroll
    for (unsigned i = 0; i < 8; ++i) {
      const unsigned at = q + i < terms ? q + i : terms - 1, c = at / a.r.out_splits, s = at % a.r.out_splits;
      part[i] = *reinterpret_cast<const v2f *>(a.r.out + ((size_t)s * a.r.places + a.r.place[t * p.top_k + c]) * p.hidden + j);
    }
#pragma unroll
    for (unsigned i = 0; i < 8; ++i)
      if (q + i < terms) v.x += part[i].x, v.y += part[i].y;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) p.y[t * p.ldy + j + i] = p.residual ? __fadd_rn(__fmul_rn(p.beta, p.residual[t * p.ld_residual + j + i]), v[i]) : v[i];
}

inline size_t up256(size_t v) { return (v + 255) / 256 * 256; }

// Groups of 16 rows of weights per pair of waves: two, for fewer requests of tokens, where that leaves a workgroup per compute unit.
int groups_for(size_t columns, size_t per_group, size_t slots) { return (columns + 2 * per_group - 1) / (2 * per_group) * slots >= 256 ? 2 : 1; }
int in_groups(const skl_moe_problem *p, size_t slots) { return groups_for(p->inter, 32, slots); }
int out_groups(const skl_moe_problem *p, size_t slots) { return groups_for(p->hidden, 64, slots); }

// 32 tokens of an expert at a time where many experts have more than 16; below 8 each on average, 1 in 250 has, and its weights are read twice.
int token_groups(const skl_moe_problem *p) { return p->tokens <= 16 || p->tokens * p->top_k <= 8 * p->experts ? 1 : 2; }

// Parts of K that give the output products of `slots` experts as many workgroups as run at a time, of two chunks at least: 4 tokens, 2 of 8 x 14336, 65 us without, 53 with.
unsigned out_splits_for(const skl_moe_problem *p, size_t slots) {
  const size_t cols = 64 * (size_t)out_groups(p, slots), tiles = (p->hidden + cols - 1) / cols * slots, most = (p->inter + 2 * kChunk - 1) / (2 * kChunk);
  const size_t want = ((token_groups(p) == 1 ? 512 : 256) + tiles - 1) / tiles;
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
  r->out_splits = out_splits_for(p, slots);
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

template <class S>
int launch_as(void (*kernel)(MoeArgs), const MoeArgs &a, dim3 grid, std::atomic<bool> &done, const char *what) {
  if (!done.load(std::memory_order_acquire)) {  // racing threads set the same value
    const int rc = skl_check_hip(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, S::kLds), what);
    if (rc != 0) return rc;
    done.store(true, std::memory_order_release);
  }
  kernel<<<grid, kThreads, S::kLds, skl_current_stream()>>>(a);
  return skl_check_launch(what);
}
template <int CG, int RG>
int launch_in(const MoeArgs &a, unsigned slots) {
  static std::atomic<bool> done{false};
  return launch_as<Shape<CG, RG, 1>>(moe_in_kernel<CG, RG>, a, dim3(skl_div_up(a.p.inter, 32 * CG), slots), done, "moe_in");
}
template <int CG, int RG>
int launch_out(const MoeArgs &a, unsigned slots) {
  static std::atomic<bool> done{false};
  return launch_as<Shape<CG, RG, 3>>(moe_out_kernel<CG, RG>, a, dim3(skl_div_up(a.p.hidden, 64 * CG), slots, a.r.out_splits), done, "moe_out");
}
template <int RG>
int launch_products(const MoeArgs &a, unsigned slots) {
  const int in = in_groups(&a.p, slots), out = out_groups(&a.p, slots);
  const int rc = in == 2 ? launch_in<2, RG>(a, slots) : launch_in<1, RG>(a, slots);
  if (rc != 0) return rc;
  return out == 2 ? launch_out<2, RG>(a, slots) : launch_out<1, RG>(a, slots);
}

int launch_on(const skl_moe_problem *p, char *block) {
  MoeArgs a = {*p, {}};
  lay_out(p, block, &a.r);
  const unsigned slots = (unsigned)(p->experts < a.r.places ? p->experts : a.r.places);
  hipStream_t st = skl_current_stream();
  const dim3 grid(skl_div_up(p->experts, 16), skl_div_up(p->tokens, 16), a.r.router_splits);
  moe_router_kernel<<<grid, kRouterThreads, 0, st>>>(a);
  int rc = skl_check_launch("moe_router");
  if (rc != 0) return rc;
  const bool four = p->tokens > 16 && p->top_k <= 16 && p->experts <= 128;  // tokens to a wave
  const size_t lanes = (four ? 16 : 64) * p->tokens, want = p->experts > lanes ? p->experts : lanes;
  const unsigned threads = want < kRouterThreads ? (unsigned)(want + 63) / 64 * 64 : kRouterThreads;
  if (four && p->experts <= 64) moe_choice_kernel<16, 4><<<1, threads, 0, st>>>(a);
  else if (four) moe_choice_kernel<16, 8><<<1, threads, 0, st>>>(a);
  else if (p->experts <= 64) moe_choice_kernel<64, 1><<<1, threads, 0, st>>>(a);
  else if (p->experts <= 256) moe_choice_kernel<64, 4><<<1, threads, 0, st>>>(a);
  else moe_choice_kernel<64, 16><<<1, threads, 0, st>>>(a);
  rc = skl_check_launch("moe_choice");
  if (rc != 0) return rc;
  rc = token_groups(p) == 1 ? launch_products<1>(a, slots) : launch_products<2>(a, slots);
  if (rc != 0) return rc;
  moe_sum_kernel<<<dim3(skl_div_up(p->hidden, 512), (unsigned)p->tokens), 256, 0, st>>>(a);
  return skl_check_launch("moe_sum");
}

}  // namespace

extern "C" int skl_hip_launch_moe(const skl_moe_problem *p) {
  Routing r;
  const size_t bytes = lay_out(p, nullptr, &r);
  const int pending = skl_hip_pending_error();
  int rc;
  skl_hip_sequence_begin();  // the launches hand data on through the stream's scratch memory
  char *block = static_cast<char *>(skl_hip_operand_scratch(bytes)), *own = nullptr;
  // a stream without scratch memory, or no room for it: a block for this call alone, released once the stream has drained
  if (!block) block = own = static_cast<char *>(skl_hip_malloc(bytes));
  if (block) {
    rc = launch_on(p, block);
  } else {
    rc = SKL_HIP_ERR_WORKSPACE;
    skl_hip_withdraw_error(SKL_HIP_ERR_STREAM_SLOTS);
    skl_hip_record_error(rc, "mixture of experts: no scratch memory, y not written");
  }
  skl_hip_sequence_end();
  if (own) {
    skl_hip_synchronize();
    skl_hip_free(own);
    if (rc == 0) {  // nothing is missing
      if (pending != SKL_HIP_ERR_WORKSPACE) skl_hip_withdraw_error(SKL_HIP_ERR_WORKSPACE);
      if (pending != SKL_HIP_ERR_STREAM_SLOTS) skl_hip_withdraw_error(SKL_HIP_ERR_STREAM_SLOTS);
    }
  }
  return rc;
}
