// RMSNorm of every query and key head with the position rotation in the same pass, and its backward.
//
//   n = x r,  r = rsqrt(mean(x^2) + eps) over the head's dimensions;   y = R(pos) (w o n)
// with R the rotation of b200_rope: interleaved pairs (2i, 2i + 1) turn by pos * theta^(-2i / head_dim). The weights
// (one vector for the query heads, one for the key heads) may be missing (w = 1). With g = R(pos)^T dy and a = w o g:
//   dx = r (a - n mean(a o n)),     dw = sum over tokens and heads of g o n
// r is formed again in the backward: the row is read there anyway, and a kept r would be a third array to carry.
//
// The angles: at position 10^6 an fp32 product is off by 0.06 radians, more than bf16 outputs may be. Positions are
// multiplied in fp64 with the frequency in turns, the whole turns taken off, and the rest (at most half a turn) goes to
// sincospif in fp32. A block forms its head_dim / 2 frequencies once; a lane forms four sines and cosines per token and
// uses them for all heads of its warp.
//
// Layout: a head's row of 16-byte vectors lies on the next power of two of lanes (head_dim 128: 16 lanes, two heads per
// warp at a time), so that the sums are shuffles. A warp takes a token and runs over its heads in rounds of a few warp-wide
// vectors. Bound by memory, 4 bytes per element forward, 6 backward: to keep enough of it in flight every lane copies the
// vectors of the next two rounds into places of its own in shared memory (cp.async; registers hold no more than one round).
// Measured with 16 + 4 heads of 128: 8192 tokens forward 18 us, backward 32 us and 5 for the weights' join; 65536 tokens 110 us (6.1 TB/s)
// and 180 us (5.6 TB/s).
#include <math.h>

#include "common.cuh"
#include "../../include/b200_moe.h"

namespace b200 {
namespace qkn {

constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int MAX_HEAD_DIM = 256;
// Warp-wide vectors of a round, rounds in shared memory, blocks per SM.
constexpr int BATCH = 4, STAGES = 3, FWD_BLOCKS = 3, BWD_BLOCKS = 2;
constexpr size_t ring_bytes(bool bwd) { return (size_t)WARPS * STAGES * BATCH * (bwd ? 2 : 1) * 32 * sizeof(uint4); }

struct Params {
  int tokens, q_heads, heads;  // heads = query + key heads
  int head_dim, head_vec;      // head_vec = head_dim / 8
  bool spread;                 // a token's rounds of heads go to warps of their own
  float eps, inv_dim;
  double log2_theta;
  const int *pos;
  const uint4 *wq, *wk;        // null: ones
  const uint4 *q, *k;          // [tokens][heads][head_vec]
  const uint4 *dyq, *dyk;      // backward
  uint4 *out_q, *out_k;        // y, or dx in the backward
  float *partial;              // backward with weights: [blocks][2][head_dim]
};

__device__ __forceinline__ void copy16(uint4 *dst, const uint4 *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}

__device__ __forceinline__ void turn_angles(double pos, const double *turns, float *cs, float *sn) {
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const double t = pos * turns[j];
    sincospif(2.0f * (float)(t - rint(t)), &sn[j], &cs[j]);
  }
}

// LANES: lanes that share a head (a power of two); BWD: the backward, with the weights' gradients when p.partial is not null.
// The query heads of a token come in rounds of AT_ONCE * BATCH, then the key heads. Arithmetic on pairs (2i, 2i + 1): both kernels are
// as much bound by the instructions they issue as by memory, and packed ones halve them.
template <int LANES, bool BWD>
__global__ void __launch_bounds__(THREADS, BWD ? BWD_BLOCKS : FWD_BLOCKS) qk_norm_rope_kernel(const __grid_constant__ Params p) {
  constexpr int AT_ONCE = 32 / LANES;  // heads
  constexpr int ROUND = AT_ONCE * BATCH;
  extern __shared__ uint4 s_ring[];  // [warp][stage][vector][x, dy][lane]
  __shared__ double s_turns[MAX_HEAD_DIM / 2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = lane % LANES, slot = lane / LANES;
  const bool on_row = c < p.head_vec;
  const double *turns = s_turns + (on_row ? c * 4 : 0);
  const int rounds_q = (p.q_heads + ROUND - 1) / ROUND, rounds = rounds_q + (p.heads - p.q_heads + ROUND - 1) / ROUND;
  uint64_t gq[4] = {0, 0, 0, 0}, gk[4] = {0, 0, 0, 0};  // pairs of zeros
  const uint4 ones = make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u);

  // Many tokens: a warp takes every `stride`th token and all of its rounds. Few: one round of one token.
  const uint32_t w = blockIdx.x * WARPS + warp, stride = gridDim.x * WARPS, tokens = p.tokens;  // unsigned: a sum may pass 2^31
  struct At {
    uint32_t tok;
    int rd;
  };
  const int only = p.spread ? (int)(w % (uint32_t)rounds) : 0;
  At now = {p.spread ? w / (uint32_t)rounds : w, only};
  auto next = [&](At a) {
    if (p.spread) return At{tokens, 0};
    return a.rd + 1 < rounds ? At{a.tok, a.rd + 1} : At{a.tok + stride, 0};
  };
  struct Where {
    bool is_q;
    int heads, h0;
    int64_t at;
  };
  const int step = AT_ONCE * p.head_vec;
  auto where = [&](At a) {
    Where r;
    r.is_q = a.rd < rounds_q;
    r.heads = r.is_q ? p.q_heads : p.heads - p.q_heads;
    r.h0 = (r.is_q ? a.rd : a.rd - rounds_q) * ROUND + slot;
    r.at = ((int64_t)a.tok * r.heads + r.h0) * p.head_vec + c;
    return r;
  };
  constexpr int PER_STAGE = BATCH * (BWD ? 2 : 1) * 32;
  uint4 *ring = s_ring + warp * STAGES * PER_STAGE + lane;
  auto fetch = [&](At a, int stage) {
    if (a.tok < tokens) {
      const Where r = where(a);
      const uint4 *px = (r.is_q ? p.q : p.k) + r.at, *pd = BWD ? (r.is_q ? p.dyq : p.dyk) + r.at : nullptr;
      uint4 *to = ring + stage * PER_STAGE;
#pragma unroll
      for (int b = 0; b < BATCH; b++)
        if (on_row && r.h0 + b * AT_ONCE < r.heads) {
          copy16(to + b * (BWD ? 64 : 32), px + b * step);
          if (BWD) copy16(to + b * 64 + 32, pd + b * step);
        }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  pdl_release();
  pdl_wait();
  At ahead = now;
#pragma unroll
  for (int s = 0; s < STAGES - 1; s++) {
    fetch(ahead, s);
    if (ahead.tok < tokens) ahead = next(ahead);
  }
  int pos = now.tok < tokens ? __ldg(p.pos + now.tok) : 0;
  for (int i = threadIdx.x; i < p.head_dim / 2; i += THREADS)  // while the first rounds are on their way
    s_turns[i] = exp2(-(double)(2 * i) / (double)p.head_dim * p.log2_theta) * 0.15915494309189533577;  // / (2 pi)
  __syncthreads();
  float cs[4], sn[4];
  for (int stage = 0; now.tok < tokens; now = next(now)) {
    fetch(ahead, stage == 0 ? STAGES - 1 : stage - 1);
    if (ahead.tok < tokens) ahead = next(ahead);
    const Where r = where(now);
    if (now.rd == only) {  // a new token
      turn_angles((double)pos, turns, cs, sn);
      if (!p.spread && now.tok + stride < tokens) pos = __ldg(p.pos + now.tok + stride);
    }
    const uint4 *weight = r.is_q ? p.wq : p.wk;
    const uint4 wv = weight && on_row ? __ldg(weight + c) : ones;
    const uint32_t ww[4] = {wv.x, wv.y, wv.z, wv.w};
    // y = r (keep o x + cross o x'), x' the pair the other way round; in the forward the weights lie in these coefficients
    uint64_t wt[4], keep[4], cross[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      wt[j] = widen2(ww[j]);
      keep[j] = pack2(cs[j], cs[j]);
      cross[j] = BWD ? pack2(sn[j], -sn[j]) : pack2(-sn[j], sn[j]);
      if (!BWD) {
        keep[j] = mul2(keep[j], wt[j]);
        cross[j] = mul2(cross[j], swap2(wt[j]));
      }
    }
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
    const uint4 *from = ring + stage * PER_STAGE;
    uint4 *po = (r.is_q ? p.out_q : p.out_k) + r.at;
#pragma unroll
    for (int b = 0; b < BATCH; b++) {
      if (r.h0 - slot + b * AT_ONCE >= r.heads) break;  // the same for the whole warp
      const bool on = on_row && r.h0 + b * AT_ONCE < r.heads;
      const uint4 zero = make_uint4(0, 0, 0, 0), x = on ? from[b * (BWD ? 64 : 32)] : zero;
      const uint32_t xv[4] = {x.x, x.y, x.z, x.w};
      uint64_t f[4], ss2 = 0;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        f[j] = widen2(xv[j]);
        ss2 = fma2(f[j], f[j], ss2);
      }
      float ss, odd;
      unpack2(ss2, ss, odd);
      ss += odd;
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      // the places behind the last head hold zeros: with eps = 0 their 0 * (1 / 0) would be a NaN in the weight gradients, which sum over all places
      const float rn = BWD && !on ? 0.0f : rsqrtf(fmaf(ss, p.inv_dim, p.eps));
      const uint64_t rr = pack2(rn, rn);
      uint32_t out[4];
      if (!BWD) {
#pragma unroll
        for (int j = 0; j < 4; j++) out[j] = round2(mul2(rr, fma2(keep[j], f[j], mul2(cross[j], swap2(f[j])))));
      } else {
        const uint4 dy = on ? from[b * 64 + 32] : zero;
        const uint32_t dv[4] = {dy.x, dy.y, dy.z, dy.w};
        uint64_t a[4], dot2 = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const uint64_t d = widen2(dv[j]), g = fma2(keep[j], d, mul2(cross[j], swap2(d)));
          f[j] = mul2(f[j], rr);
          if (r.is_q) gq[j] = fma2(g, f[j], gq[j]);
          else gk[j] = fma2(g, f[j], gk[j]);
          a[j] = mul2(g, wt[j]);
          dot2 = fma2(a[j], f[j], dot2);
        }
        float dot, odd2;
        unpack2(dot2, dot, odd2);
        dot += odd2;
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
        dot *= -p.inv_dim;
        const uint64_t minus = pack2(dot, dot);
#pragma unroll
        for (int j = 0; j < 4; j++) out[j] = round2(mul2(rr, fma2(f[j], minus, a[j])));
      }
      if (on) st_stream(po + b * step, make_uint4(out[0], out[1], out[2], out[3]));
    }
    stage = stage + 1 == STAGES ? 0 : stage + 1;
  }
  if constexpr (BWD) {
    if (p.partial == nullptr) return;
    // the block's share of the weight gradients: slots of a warp, then warps, each in a fixed order
    __shared__ float s_sum[WARPS][2][MAX_HEAD_DIM];
#pragma unroll
    for (int i = 0; i < 8; i++) {
      float q0, q1, k0, k1;
      unpack2(gq[i >> 1], q0, q1);
      unpack2(gk[i >> 1], k0, k1);
      float q = i & 1 ? q1 : q0, k = i & 1 ? k1 : k0;
#pragma unroll
      for (int o = LANES; o < 32; o <<= 1) {
        q += __shfl_xor_sync(0xffffffffu, q, o);
        k += __shfl_xor_sync(0xffffffffu, k, o);
      }
      if (slot == 0 && on_row) {
        s_sum[warp][0][c * 8 + i] = q;
        s_sum[warp][1][c * 8 + i] = k;
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * p.head_dim; i += THREADS) {
      const int which = i / p.head_dim, d = i - which * p.head_dim;
      float t = 0.0f;
#pragma unroll
      for (int w = 0; w < WARPS; w++) t += s_sum[w][which][d];
      p.partial[(int64_t)blockIdx.x * 2 * p.head_dim + i] = t;
    }
  }
}

// dw = (dw +) sum of the blocks' shares: a block takes 32 columns, its 32 warps every 32nd share (all asked for at once: with eight warps
// this took 7 us), then the warps' sums in order
constexpr int JOIN_WARPS = 32;
__global__ void __launch_bounds__(JOIN_WARPS * 32) qk_weight_grad_kernel(int head_dim, int blocks, const float *__restrict__ partial,
                                                                       bool accumulate, __nv_bfloat16 *dwq, __nv_bfloat16 *dwk) {
  __shared__ float part[JOIN_WARPS][32];
  pdl_release();
  pdl_wait();
  const int lane = threadIdx.x & 31, grp = threadIdx.x >> 5;
  const int i = blockIdx.x * 32 + lane;
  float s = 0.0f;
  if (i < 2 * head_dim) {
#pragma unroll 8
    for (int b = grp; b < blocks; b += JOIN_WARPS) s += partial[(int64_t)b * 2 * head_dim + i];
  }
  part[grp][lane] = s;
  __syncthreads();
  if (grp != 0 || i >= 2 * head_dim) return;
  float t = 0.0f;
#pragma unroll
  for (int g = 0; g < JOIN_WARPS; g++) t += part[g][lane];
  __nv_bfloat16 *dw = i < head_dim ? dwq : dwk;
  if (dw == nullptr) return;
  dw += i < head_dim ? i : i - head_dim;
  *dw = __float2bfloat16_rn(accumulate ? __bfloat162float(*dw) + t : t);
}

}  // namespace qkn
}  // namespace b200

using namespace b200;

namespace {

int qkn_sms() {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

int qkn_lanes(int head_dim) {
  int l = 1;
  while (l * 8 < head_dim) l *= 2;
  return l;
}

// A warp takes whole tokens as long as these alone give every SM 16 warps (backward: 4; its blocks' shares of the weight gradients have to
// be added up); below that every round of heads gets a warp, so that few tokens spread over the GPU.
int qkn_border(bool bwd, int sms) { return sms * (bwd ? 4 : 16); }
bool qkn_spread(int tokens, bool bwd, int sms) { return tokens < qkn_border(bwd, sms); }

int qkn_blocks(int tokens, int q_heads, int heads, int head_dim, bool bwd, int sms) {
  const int round = 32 / qkn_lanes(head_dim) * qkn::BATCH, rounds = (q_heads + round - 1) / round + (heads - q_heads + round - 1) / round;
  if (qkn_spread(tokens, bwd, sms)) return (int)(((int64_t)tokens * rounds + qkn::WARPS - 1) / qkn::WARPS);
  const int want = (tokens - 1) / qkn::WARPS + 1, most = sms * (bwd ? qkn::BWD_BLOCKS : qkn::FWD_BLOCKS);
  return want < most ? want : most;
}

template <int LANES, bool BWD>
int qkn_launch_lanes(const char *op, const qkn::Params &p, int blocks, cudaStream_t s) {
  static bool done[64];
  int dev = -1;
  B200_CUDA(cudaGetDevice(&dev));
  B200_REQUIRE(dev >= 0 && dev < 64, "%s: device ordinal %d is out of range", op, dev);
  constexpr size_t smem = qkn::ring_bytes(BWD);
  if (!done[dev]) {
    B200_CUDA(cudaFuncSetAttribute(qkn::qk_norm_rope_kernel<LANES, BWD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    done[dev] = true;
  }
  B200_CUDA(b200_launch_overlapped(qkn::qk_norm_rope_kernel<LANES, BWD>, dim3(blocks), dim3(qkn::THREADS), smem, s, 1, p));
  B200_CHECK_LAUNCH(op);
  return 0;
}

template <bool BWD>
int qkn_launch(const char *op, const qkn::Params &p, int blocks, cudaStream_t s) {
  switch (qkn_lanes(p.head_dim)) {
    case 1: return qkn_launch_lanes<1, BWD>(op, p, blocks, s);
    case 2: return qkn_launch_lanes<2, BWD>(op, p, blocks, s);
    case 4: return qkn_launch_lanes<4, BWD>(op, p, blocks, s);
    case 8: return qkn_launch_lanes<8, BWD>(op, p, blocks, s);
    case 16: return qkn_launch_lanes<16, BWD>(op, p, blocks, s);
    default: return qkn_launch_lanes<32, BWD>(op, p, blocks, s);
  }
}

int qkn_params(const char *op, qkn::Params *p, int dt, int num_tokens, int num_q_heads, int num_kv_heads, int head_dim, float eps, int theta,
               const int *seq_positions, const void *q_weight, const void *k_weight, const void *X_q, const void *X_k, void *out_q,
               void *out_k) {
  B200_REQUIRE(dt == B200_DT_BF16, "%s: only bf16 is implemented (datatype code %d)", op, dt);
  B200_REQUIRE(num_tokens >= 0 && num_q_heads >= 1 && num_kv_heads >= 0 && num_q_heads <= 65536 && num_kv_heads <= 65536,
               "%s: bad number of tokens or heads (%d, %d, %d)", op, num_tokens, num_q_heads, num_kv_heads);
  B200_REQUIRE(head_dim >= 8 && head_dim % 8 == 0 && head_dim <= qkn::MAX_HEAD_DIM, "%s: head_dim must be a multiple of 8, at most %d (got %d)",
               op, qkn::MAX_HEAD_DIM, head_dim);
  B200_REQUIRE(eps >= 0.0f && theta >= 1, "%s: need eps >= 0 and theta >= 1", op);
  if (num_tokens == 0) return 0;
  B200_REQUIRE(seq_positions && X_q && out_q && (num_kv_heads == 0 || (X_k && out_k)), "%s: null argument", op);
  B200_REQUIRE(b200_aligned16(q_weight) && b200_aligned16(k_weight) && b200_aligned16(X_q) && b200_aligned16(X_k) && b200_aligned16(out_q) &&
                   b200_aligned16(out_k),
               "%s: tensors must be 16-byte aligned", op);
  *p = qkn::Params{};
  p->tokens = num_tokens;
  p->q_heads = num_q_heads;
  p->heads = num_q_heads + num_kv_heads;
  p->head_dim = head_dim;
  p->head_vec = head_dim / 8;
  p->eps = eps;
  p->inv_dim = 1.0f / (float)head_dim;
  p->log2_theta = log2((double)theta);
  p->pos = seq_positions;
  p->wq = (const uint4 *)q_weight;
  p->wk = (const uint4 *)k_weight;
  p->q = (const uint4 *)X_q;
  p->k = (const uint4 *)X_k;
  p->out_q = (uint4 *)out_q;
  p->out_k = (uint4 *)out_k;
  return 0;
}

}  // namespace

extern "C" int b200_qk_norm_rope(int fwd_dt, int num_tokens, int num_q_heads, int num_kv_heads, int head_dim, float eps, int theta,
                                 const int *seq_positions, const void *q_weight, const void *k_weight, const void *X_q, const void *X_k,
                                 void *out_q, void *out_k, void *stream) {
  qkn::Params p;
  if (qkn_params("qk_norm_rope", &p, fwd_dt, num_tokens, num_q_heads, num_kv_heads, head_dim, eps, theta, seq_positions, q_weight, k_weight,
                 X_q, X_k, out_q, out_k))
    return -1;
  if (num_tokens == 0) return 0;
  const int sms = qkn_sms();
  p.spread = qkn_spread(num_tokens, false, sms);
  return qkn_launch<false>("qk_norm_rope", p, qkn_blocks(num_tokens, p.q_heads, p.heads, head_dim, false, sms), (cudaStream_t)stream);
}

extern "C" uint64_t b200_qk_norm_rope_bwd_workspace_bytes(int num_tokens, int num_q_heads, int num_kv_heads, int head_dim) {
  if (num_tokens <= 0 || num_q_heads < 1 || num_kv_heads < 0 || head_dim < 8 || head_dim % 8 || head_dim > qkn::MAX_HEAD_DIM) return 0;
  // enough for every smaller number of tokens too: the most blocks may run just below the border between the two layouts
  const int sms = qkn_sms(), border = qkn_border(true, sms), below = num_tokens < border ? num_tokens : border - 1, heads = num_q_heads + num_kv_heads;
  const int a = qkn_blocks(num_tokens, num_q_heads, heads, head_dim, true, sms),
            b = qkn_blocks(below, num_q_heads, heads, head_dim, true, sms);
  return (uint64_t)(a > b ? a : b) * 2 * head_dim * sizeof(float);
}

extern "C" int b200_qk_norm_rope_bwd(int fwd_dt, int bwd_dt, int num_tokens, int num_q_heads, int num_kv_heads, int head_dim, float eps,
                                     int theta, const int *seq_positions, const void *q_weight, const void *k_weight, const void *X_q,
                                     const void *X_k, const void *d_out_q, const void *d_out_k, void *dX_q, void *dX_k, void *dq_weight,
                                     void *dk_weight, int accumulate, uint64_t workspace_bytes, void *workspace, void *stream) {
  qkn::Params p;
  B200_REQUIRE(bwd_dt == B200_DT_BF16, "qk_norm_rope_bwd: only bf16 is implemented (datatype code %d)", bwd_dt);
  if (qkn_params("qk_norm_rope_bwd", &p, fwd_dt, num_tokens, num_q_heads, num_kv_heads, head_dim, eps, theta, seq_positions, q_weight,
                 k_weight, X_q, X_k, dX_q, dX_k))
    return -1;
  const bool want_dw = dq_weight != nullptr || dk_weight != nullptr;
  // one vector for both would be written by two threads
  const uintptr_t wa = reinterpret_cast<uintptr_t>(dq_weight), wb = reinterpret_cast<uintptr_t>(dk_weight), wn = (uintptr_t)head_dim * 2;
  B200_REQUIRE(!wa || !wb || (wa < wb ? wa + wn <= wb : wb + wn <= wa), "qk_norm_rope_bwd: dq_weight and dk_weight overlap");
  if (num_tokens == 0) {  // the sums over no tokens
    if (dq_weight && !accumulate) B200_CUDA(cudaMemsetAsync(dq_weight, 0, (size_t)head_dim * 2, (cudaStream_t)stream));
    if (dk_weight && !accumulate) B200_CUDA(cudaMemsetAsync(dk_weight, 0, (size_t)head_dim * 2, (cudaStream_t)stream));
    return 0;
  }
  B200_REQUIRE(d_out_q && (num_kv_heads == 0 || d_out_k) && b200_aligned16(d_out_q) && b200_aligned16(d_out_k),
               "qk_norm_rope_bwd: the upstream gradients must be given and 16-byte aligned");
  const int sms = qkn_sms();
  p.spread = qkn_spread(num_tokens, true, sms);
  const int blocks = qkn_blocks(num_tokens, p.q_heads, p.heads, head_dim, true, sms);
  if (want_dw) {
    const uint64_t need = (uint64_t)blocks * 2 * head_dim * sizeof(float);
    B200_REQUIRE(workspace && b200_aligned16(workspace) && workspace_bytes >= need,
                 "qk_norm_rope_bwd: the workspace holds %llu bytes, %llu are needed (b200_qk_norm_rope_bwd_workspace_bytes)",
                 (unsigned long long)workspace_bytes, (unsigned long long)need);
    p.partial = (float *)workspace;
  }
  p.dyq = (const uint4 *)d_out_q;
  p.dyk = (const uint4 *)d_out_k;
  if (qkn_launch<true>("qk_norm_rope_bwd", p, blocks, (cudaStream_t)stream)) return -1;
  if (!want_dw) return 0;
  B200_CUDA(b200_launch_overlapped(qkn::qk_weight_grad_kernel, dim3((2 * head_dim + 31) / 32), dim3(qkn::JOIN_WARPS * 32), 0, (cudaStream_t)stream, 1,
                                   head_dim, blocks, (const float *)p.partial, accumulate != 0, (__nv_bfloat16 *)dq_weight,
                                   (__nv_bfloat16 *)dk_weight));
  B200_CHECK_LAUNCH("qk_norm_rope_bwd (weights)");
  return 0;
}
