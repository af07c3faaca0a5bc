// skl_moe_mxf4.hip - a mixture-of-experts layer over MXFP4 weights for up to 64 tokens (include/skl-gfx950.h has the formulas):
// router, choice, the chosen experts' gated input product, their output product and its weighted sum.
//
// What bounds it is the stream over the chosen experts' weights, half a byte and a thirty-second per value. They are widened in
// registers to bf16 with their scale (v_cvt_scalef32_pk_bf16_fp4, exact) and multiplied by v_mfma_f32_16x16x32_bf16: products of bf16
// values, exact, summed in fp32. A lane's 16 bytes are one block of 32 k of one row of weights; which k of a chunk of 128 meet in which
// of its four instructions is free as long as both operands' lanes take the same.
// The tokens of an expert are gathered: only rows of tokens that chose it are multiplied, 16 at a time.
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
struct Routing {
  float *logits;       // [token][expert]
  unsigned *active;    // how many experts some token chose
  unsigned *expert;    // of slot s (the active ones in ascending order)
  unsigned *first;     // its first place in the lists below
  unsigned *count;     // how many tokens chose it
  unsigned *token;     // [place], by expert and then by token
  float *weight;       // [place]
  uint16_t *hi, *lo;   // [place][inter]: h as a sum of two bf16 values
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

// Logits: a workgroup of four waves takes 16 experts and 16 tokens, each wave a quarter of hidden.
__global__ void __launch_bounds__(256) moe_router_kernel(MoeArgs a) {
  __shared__ float red[4][16][17];
  const skl_moe_problem &p = a.p;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, l = lane & 15, g = lane >> 4;
  const size_t e0 = (size_t)blockIdx.x * 16, t0 = (size_t)blockIdx.y * 16;
  const size_t e = e0 + l < p.experts ? e0 + l : p.experts - 1, t = t0 + l < p.tokens ? t0 + l : p.tokens - 1;
  const uint16_t *w = p.router + e * p.ld_router + 8 * g, *x = p.x + t * p.ldx + 8 * g;
  v4f acc = {0.0f, 0.0f, 0.0f, 0.0f};
  for (size_t k = 32 * (size_t)wave; k < p.hidden; k += 128)
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*reinterpret_cast<const v8bf *>(x + k), *reinterpret_cast<const v8bf *>(w + k), acc, 0, 0, 0);
#pragma unroll
  for (int r = 0; r < 4; ++r) red[wave][4 * g + r][l] = acc[r];
  __syncthreads();
  const unsigned i = threadIdx.x >> 4, j = threadIdx.x & 15;
  if (t0 + i < p.tokens && e0 + j < p.experts)
    a.r.logits[(t0 + i) * p.experts + e0 + j] = (red[0][i][j] + red[1][i][j]) + (red[2][i][j] + red[3][i][j]);
}

// A logit as a number that orders like it: NaN lowest, the two zeros alike.
__device__ __forceinline__ unsigned order_of(float v) {
  if (v != v) return 0u;
  const unsigned b = __float_as_uint(v + 0.0f);
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}

// The choice: one workgroup; a wave per token in turn, the experts' logits over its lanes.
__global__ void __launch_bounds__(1024) moe_choose_kernel(MoeArgs a) {
  __shared__ unsigned mask[kMaxExperts][2];  // tokens that chose an expert
  __shared__ unsigned start[kMaxExperts];
  __shared__ unsigned short chosen[kMaxTokens * kMaxTop];
  __shared__ float share[kMaxTokens * kMaxTop];
  __shared__ unsigned totals[16];
  const skl_moe_problem &p = a.p;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const unsigned experts = (unsigned)p.experts, top = (unsigned)p.top_k, tokens = (unsigned)p.tokens;
  for (unsigned e = threadIdx.x; e < kMaxExperts; e += 1024) mask[e][0] = mask[e][1] = 0;
  __syncthreads();
  for (unsigned t = wave; t < tokens; t += 16) {
    const float *logits = a.r.logits + (size_t)t * experts;
    unsigned long long key[kMaxExperts / 64];  // by logit, then by the lower expert; 0: taken, or none
    float value[kMaxExperts / 64];
#pragma unroll
    for (unsigned i = 0; i < kMaxExperts / 64; ++i) {
      const unsigned e = 64 * i + lane;
      key[i] = 0, value[i] = 0.0f;
      if (e < experts) {
        value[i] = logits[e];
        key[i] = ((unsigned long long)order_of(value[i]) << 32) | (0xFFFFFFFFu - e);
      }
    }
    float largest = 0.0f, sum = 0.0f, mine = 0.0f;
    for (unsigned j = 0; j < top; ++j) {
      unsigned long long best = 0;
#pragma unroll
      for (unsigned i = 0; i < kMaxExperts / 64; ++i) best = key[i] > best ? key[i] : best;
#pragma unroll
      for (int step = 32; step > 0; step >>= 1) {
        const unsigned long long other = __shfl_xor(best, step, 64);
        best = other > best ? other : best;
      }
      const unsigned e = 0xFFFFFFFFu - (unsigned)best;
      float v = 0.0f;
#pragma unroll
      for (unsigned i = 0; i < kMaxExperts / 64; ++i)
        if (e / 64 == i) v = value[i];
      v = __shfl(v, (int)(e & 63u), 64);
#pragma unroll
      for (unsigned i = 0; i < kMaxExperts / 64; ++i)
        if (key[i] == best) key[i] = 0;
      if (j == 0) largest = v;
      const float x = expf(v - largest);
      if (p.normalise) sum += x;
      if ((unsigned)lane == j) mine = x;
      if (lane == 0) {
        chosen[t * top + j] = (unsigned short)e;
        atomicOr(&mask[e][t >> 5], 1u << (t & 31u));
      }
    }
    if (!p.normalise) {
#pragma unroll
      for (unsigned i = 0; i < kMaxExperts / 64; ++i)
        if (64 * i + lane < experts) sum += expf(value[i] - largest);
#pragma unroll
      for (int step = 32; step > 0; step >>= 1) sum += __shfl_xor(sum, step, 64);
    }
    if ((unsigned)lane < top) share[t * top + lane] = mine / sum;
  }
  __syncthreads();
  // Where each expert's tokens begin, and its slot: one scan over the experts, the count in the lower half, the slot in the upper.
  const unsigned e = threadIdx.x;
  const unsigned count = __popc(mask[e][0]) + __popc(mask[e][1]), own = count | (count ? 0x10000u : 0u);
  unsigned scan = own;
#pragma unroll
  for (int step = 1; step < 64; step <<= 1) {
    const unsigned other = __shfl_up(scan, step, 64);
    if (lane >= step) scan += other;
  }
  if (lane == 63) totals[wave] = scan;
  __syncthreads();
  for (int w = 0; w < wave; ++w) scan += totals[w];
  start[e] = (scan - own) & 0xFFFFu;
  if (count) {
    const unsigned slot = (scan - own) >> 16;
    a.r.expert[slot] = e;
    a.r.first[slot] = start[e];
    a.r.count[slot] = count;
  }
  if (e == 1023) a.r.active[0] = scan >> 16;
  __syncthreads();
  for (unsigned at = threadIdx.x; at < tokens * top; at += 1024) {
    const unsigned t = at / top, c = chosen[at], below = t & 31u;
    const unsigned before = t < 32 ? __popc(mask[c][0] & ((1u << below) - 1u)) : __popc(mask[c][0]) + __popc(mask[c][1] & ((1u << below) - 1u));
    const unsigned place = start[c] + before;
    a.r.token[place] = t;
    a.r.weight[place] = share[at];
    if (p.ids) p.ids[at] = (int32_t)c;
    if (p.weights) p.weights[at] = share[at];
  }
}

// h of 16 inner columns of one expert (blockIdx.y: its slot) for all of its tokens: four waves take chunks of 128 k in turn and meet in
// LDS. RT groups of 16 tokens at most.
template <int RT>
__global__ void __launch_bounds__(256) moe_in_kernel(MoeArgs a) {
  __shared__ float red[4][2][RT * 16][17];
  const skl_moe_problem &p = a.p;
  const unsigned slot = blockIdx.y;
  if (slot >= a.r.active[0]) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, l = lane & 15, g = lane >> 4;
  const size_t e = a.r.expert[slot], col = (size_t)blockIdx.x * 16 + l;
  const unsigned first = a.r.first[slot], count = a.r.count[slot], groups = (count + 15) / 16;
  const uint8_t *gate = p.gate.codes + (e * p.expert_in + col * p.gate.ld) / 2, *up = p.up.codes + (e * p.expert_in + col * p.up.ld) / 2;
  const uint8_t *gate_s = p.gate.scales + e * p.expert_in_scales + col * p.gate.lds, *up_s = p.up.scales + e * p.expert_in_scales + col * p.up.lds;
  const uint16_t *x[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const unsigned at = 16u * rt + l;
    x[rt] = p.x + (size_t)a.r.token[first + (at < count ? at : count - 1)] * p.ldx;
  }
  v4f acc[2][RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) acc[0][rt] = acc[1][rt] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  const v4i zero = {0, 0, 0, 0};
  for (size_t k = 128 * (size_t)wave; k < p.hidden; k += 512) {
    const size_t own = k + 32 * (size_t)g;  // the lane's block is inside or outside
    const bool in = own < p.hidden;
    const size_t kk = in ? own : 0;
    const v4i wg = *reinterpret_cast<const v4i *>(gate + kk / 2), wu = *reinterpret_cast<const v4i *>(up + kk / 2);
    const float sg = __uint_as_float((unsigned)gate_s[kk / 32] << 23), su = __uint_as_float((unsigned)up_s[kk / 32] << 23);
    v4i xv[RT][4];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        xv[rt][j] = zero;
        if (rt < (int)groups) xv[rt][j] = *reinterpret_cast<const v4i *>(x[rt] + kk + 8 * j);
        xv[rt][j] = in ? xv[rt][j] : zero;
      }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const v8bf bg = widen_f4(in ? (unsigned)wg[j] : 0u, in ? sg : 1.0f), bu = widen_f4(in ? (unsigned)wu[j] : 0u, in ? su : 1.0f);
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
        if (rt < (int)groups) {
          const v8bf av = __builtin_bit_cast(v8bf, xv[rt][j]);
          acc[0][rt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(av, bg, acc[0][rt], 0, 0, 0);
          acc[1][rt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(av, bu, acc[1][rt], 0, 0, 0);
        }
    }
  }
#pragma unroll
  for (int rt = 0; rt < RT; ++rt)
#pragma unroll
    for (int r = 0; r < 4; ++r) red[wave][0][16 * rt + 4 * g + r][l] = acc[0][rt][r], red[wave][1][16 * rt + 4 * g + r][l] = acc[1][rt][r];
  __syncthreads();
  for (unsigned at = threadIdx.x; at < count * 16; at += 256) {
    const unsigned i = at >> 4, j = at & 15;
    const float gv = (red[0][0][i][j] + red[1][0][i][j]) + (red[2][0][i][j] + red[3][0][i][j]);
    const float uv = (red[0][1][i][j] + red[1][1][i][j]) + (red[2][1][i][j] + red[3][1][i][j]);
    const float h = skl_activate(gv, p.activation) * uv * a.r.weight[first + i];
    const unsigned short hi = bf16_of(h);
    const size_t to = (size_t)(first + i) * p.inter + (size_t)blockIdx.x * 16 + j;
    a.r.hi[to] = hi;
    a.r.lo[to] = bf16_of(h - of_bf16(hi));
  }
}

// 16 columns of y for all tokens: the active experts one after another, eight waves taking chunks of 128 of an expert's inner columns in turn.
// A wave adds an expert's rows to its own sums in LDS, one row per token; the waves' sums meet at the end.
template <int RT>
__global__ void __launch_bounds__(512) moe_out_kernel(MoeArgs a) {
  __shared__ float red[8][RT * 16][17];
  const skl_moe_problem &p = a.p;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, l = lane & 15, g = lane >> 4;
  const size_t col = (size_t)blockIdx.x * 16 + l;
  const unsigned active = a.r.active[0];
  for (unsigned i = g; i < RT * 16; i += 4) red[wave][i][l] = 0.0f;
  const v4i zero = {0, 0, 0, 0};
  for (unsigned slot = 0; slot < active; ++slot) {
    const size_t e = a.r.expert[slot];
    const unsigned first = a.r.first[slot], count = a.r.count[slot], groups = (count + 15) / 16;
    const uint8_t *down = p.down.codes + (e * p.expert_down + col * p.down.ld) / 2;
    const uint8_t *scales = p.down.scales + e * p.expert_down_scales + col * p.down.lds;
    size_t at[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) at[rt] = (size_t)(first + (16u * rt + l < count ? 16u * rt + l : count - 1)) * p.inter;
    v4f acc[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) acc[rt] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    for (size_t k = 128 * (size_t)wave; k < p.inter; k += 1024) {
      const size_t own = k + 32 * (size_t)g;
      const bool in = own < p.inter;
      const size_t kk = in ? own : 0;
      const v4i w = *reinterpret_cast<const v4i *>(down + kk / 2);
      const float s = __uint_as_float((unsigned)scales[kk / 32] << 23);
      v4i hi[RT][4], lo[RT][4];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          hi[rt][j] = lo[rt][j] = zero;
          if (rt < (int)groups) {
            hi[rt][j] = *reinterpret_cast<const v4i *>(a.r.hi + at[rt] + kk + 8 * j);
            lo[rt][j] = *reinterpret_cast<const v4i *>(a.r.lo + at[rt] + kk + 8 * j);
          }
          hi[rt][j] = in ? hi[rt][j] : zero, lo[rt][j] = in ? lo[rt][j] : zero;
        }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const v8bf b = widen_f4(in ? (unsigned)w[j] : 0u, in ? s : 1.0f);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
          if (rt < (int)groups) {
            acc[rt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, hi[rt][j]), b, acc[rt], 0, 0, 0);
            acc[rt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, lo[rt][j]), b, acc[rt], 0, 0, 0);
          }
      }
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const unsigned i = 16u * rt + 4 * g + r;
        if (i < count) red[wave][a.r.token[first + i]][l] += acc[rt][r];
      }
  }
  __syncthreads();
  for (unsigned at = threadIdx.x; at < p.tokens * 16; at += 512) {
    const unsigned t = at >> 4, j = at & 15;
    float v = red[0][t][j];
#pragma unroll
    for (int w = 1; w < 8; ++w) v += red[w][t][j];
    const size_t c = (size_t)blockIdx.x * 16 + j;
    if (p.residual) v = __fadd_rn(__fmul_rn(p.beta, p.residual[t * p.ld_residual + c]), v);
    p.y[t * p.ldy + c] = v;
  }
}

inline size_t up256(size_t v) { return (v + 255) / 256 * 256; }

template <int RT>
int launch_products(const MoeArgs &a, unsigned slots, hipStream_t st) {
  moe_in_kernel<RT><<<dim3((unsigned)(a.p.inter / 16), slots), 256, 0, st>>>(a);
  int rc = skl_check_launch("moe_in");
  if (rc != 0) return rc;
  moe_out_kernel<RT><<<(unsigned)(a.p.hidden / 16), 512, 0, st>>>(a);
  return skl_check_launch("moe_out");
}

int launch_on(const skl_moe_problem *p, char *block) {
  MoeArgs a = {*p, {}};
  const size_t places = p->tokens * p->top_k;
  const unsigned slots = (unsigned)(p->experts < places ? p->experts : places);
  auto take = [&](size_t bytes) {
    char *at = block;
    block += up256(bytes);
    return at;
  };
  a.r.logits = reinterpret_cast<float *>(take(p->tokens * p->experts * 4));
  a.r.active = reinterpret_cast<unsigned *>(take(4));
  a.r.expert = reinterpret_cast<unsigned *>(take(slots * 4));
  a.r.first = reinterpret_cast<unsigned *>(take(slots * 4));
  a.r.count = reinterpret_cast<unsigned *>(take(slots * 4));
  a.r.token = reinterpret_cast<unsigned *>(take(places * 4));
  a.r.weight = reinterpret_cast<float *>(take(places * 4));
  a.r.hi = reinterpret_cast<uint16_t *>(take(places * p->inter * 2));
  a.r.lo = reinterpret_cast<uint16_t *>(take(places * p->inter * 2));
  hipStream_t st = skl_current_stream();
  moe_router_kernel<<<dim3(skl_div_up(p->experts, 16), skl_div_up(p->tokens, 16)), 256, 0, st>>>(a);
  int rc = skl_check_launch("moe_router");
  if (rc != 0) return rc;
  moe_choose_kernel<<<1, 1024, 0, st>>>(a);
  if ((rc = skl_check_launch("moe_choose")) != 0) return rc;
  return p->tokens <= 16 ? launch_products<1>(a, slots, st) : p->tokens <= 32 ? launch_products<2>(a, slots, st) : launch_products<4>(a, slots, st);
}

size_t scratch_bytes(const skl_moe_problem *p) {
  const size_t places = p->tokens * p->top_k, slots = p->experts < places ? p->experts : places;
  return up256(p->tokens * p->experts * 4) + up256(4) + 3 * up256(slots * 4) + 2 * up256(places * 4) + 2 * up256(places * p->inter * 2);
}

}  // namespace

extern "C" int skl_hip_launch_moe(const skl_moe_problem *p) {
  skl_hip_sequence_begin();  // the launches hand data on through the stream's scratch memory
  char *block = static_cast<char *>(skl_hip_operand_scratch(scratch_bytes(p)));
  int rc = SKL_HIP_ERR_WORKSPACE;
  if (block) {
    rc = launch_on(p, block);
  } else {
    skl_hip_withdraw_error(SKL_HIP_ERR_STREAM_SLOTS);
    skl_hip_record_error(rc, "mixture of experts: no scratch memory, y not written");
  }
  skl_hip_sequence_end();
  return rc;
}
