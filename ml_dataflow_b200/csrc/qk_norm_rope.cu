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
// warp at a time), so that the sums are shuffles. A warp takes one token and runs over its heads, four warp-wide vectors
// in flight. Bound by memory: 4 bytes per element forward, 6 backward.
#include <math.h>

#include "common.cuh"
#include "../../include/b200_moe.h"

namespace b200 {
namespace qkn {

constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int MAX_HEAD_DIM = 256;
constexpr int BATCH = 4;  // warp-wide vectors in flight

struct Params {
  int tokens, q_heads, heads;  // heads = query + key heads
  int head_dim, head_vec;      // head_vec = head_dim / 8
  int parts;                   // a token's heads are split over this many warps
  float eps, inv_dim;
  double log2_theta;
  const int *pos;
  const uint4 *wq, *wk;        // null: ones
  const uint4 *q, *k;          // [tokens][heads][head_vec]
  const uint4 *dyq, *dyk;      // backward
  uint4 *out_q, *out_k;        // y, or dx in the backward
  float *partial;              // backward with weights: [blocks][2][head_dim]
};

// plain loads: the output may lie over the input
__device__ __forceinline__ uint4 ld_once(const uint4 *p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}

__device__ __forceinline__ void turn_angles(double pos, const double *turns, float *cs, float *sn) {
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const double t = pos * turns[j];
    sincospif(2.0f * (float)(t - rint(t)), &sn[j], &cs[j]);
  }
}

// LANES: lanes that share a head (a power of two); BWD: the backward; the weights' gradients when p.partial is not null
template <int LANES, bool BWD>
__global__ void __launch_bounds__(THREADS) qk_norm_rope_kernel(const Params p) {
  __shared__ double s_turns[MAX_HEAD_DIM / 2];
  for (int i = threadIdx.x; i < p.head_dim / 2; i += THREADS)
    s_turns[i] = exp2(-(double)(2 * i) / (double)p.head_dim * p.log2_theta) * 0.15915494309189533577;  // / (2 pi)
  __syncthreads();
  constexpr int AT_ONCE = 32 / LANES;  // heads
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = lane % LANES, slot = lane / LANES;
  const bool on_row = c < p.head_vec;
  const int rounds = (p.heads + AT_ONCE * BATCH - 1) / (AT_ONCE * BATCH);
  const int kv_heads = p.heads - p.q_heads;
  double turns[4];
#pragma unroll
  for (int j = 0; j < 4; j++) turns[j] = on_row ? s_turns[c * 4 + j] : 0.0;
  float gq[8] = {0, 0, 0, 0, 0, 0, 0, 0}, gk[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  const uint4 ones = make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u);
  const uint4 wq = p.wq && on_row ? __ldg(p.wq + c) : ones, wk = p.wk && on_row ? __ldg(p.wk + c) : ones;
  const int64_t units = (int64_t)p.tokens * p.parts;
  for (int64_t unit = (int64_t)blockIdx.x * WARPS + warp; unit < units; unit += (int64_t)gridDim.x * WARPS) {
    const int64_t tok = unit / p.parts;
    const int part = (int)(unit - tok * p.parts);
    float cs[4], sn[4];
    bool have_angles = false;
    for (int rd = part; rd < rounds; rd += p.parts) {
      uint4 x[BATCH], dy[BATCH];
      int64_t at[BATCH];
#pragma unroll
      for (int b = 0; b < BATCH; b++) {
        const int h = (rd * BATCH + b) * AT_ONCE + slot;
        x[b] = dy[b] = make_uint4(0, 0, 0, 0);
        at[b] = h < p.q_heads ? (tok * p.q_heads + h) * p.head_vec + c : (tok * kv_heads + (h - p.q_heads)) * p.head_vec + c;
        if (on_row && h < p.heads) {
          x[b] = ld_once((h < p.q_heads ? p.q : p.k) + at[b]);
          if (BWD) dy[b] = ld_once((h < p.q_heads ? p.dyq : p.dyk) + at[b]);
        }
      }
      if (!have_angles) {  // while the loads are on their way
        turn_angles((double)__ldg(p.pos + tok), turns, cs, sn);
        have_angles = true;
      }
#pragma unroll
      for (int b = 0; b < BATCH; b++) {
        const int h = (rd * BATCH + b) * AT_ONCE + slot;
        const bool is_q = h < p.q_heads;
        float f[8], w[8];
        unpack8(x[b], f);
        unpack8(is_q ? wq : wk, w);
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) ss = fmaf(f[i], f[i], ss);
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float r = rsqrtf(fmaf(ss, p.inv_dim, p.eps));
        if (!BWD) {
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const float e = f[2 * j] * r * w[2 * j], o = f[2 * j + 1] * r * w[2 * j + 1];
            f[2 * j] = cs[j] * e - sn[j] * o;
            f[2 * j + 1] = cs[j] * o + sn[j] * e;
          }
        } else {
          float g[8], dot = 0.0f;
          unpack8(dy[b], g);
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const float e = g[2 * j], o = g[2 * j + 1];
            g[2 * j] = cs[j] * e + sn[j] * o;
            g[2 * j + 1] = cs[j] * o - sn[j] * e;
          }
#pragma unroll
          for (int i = 0; i < 8; i++) {
            f[i] *= r;
            dot = fmaf(g[i] * w[i], f[i], dot);
          }
#pragma unroll
          for (int o = LANES / 2; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
          dot *= p.inv_dim;
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const float gn = g[i] * f[i];
            if (is_q) gq[i] += gn;
            else gk[i] += gn;
            f[i] = r * (g[i] * w[i] - f[i] * dot);
          }
        }
        if (on_row && h < p.heads) st_stream((is_q ? p.out_q : p.out_k) + at[b], pack8(f));
      }
    }
  }
  if (!BWD || p.partial == nullptr) return;
  // the block's share of the weight gradients: slots of a warp, then warps, each in a fixed order
  __shared__ float s_sum[WARPS][2][MAX_HEAD_DIM];
#pragma unroll
  for (int i = 0; i < 8; i++) {
#pragma unroll
    for (int o = LANES; o < 32; o <<= 1) {
      gq[i] += __shfl_xor_sync(0xffffffffu, gq[i], o);
      gk[i] += __shfl_xor_sync(0xffffffffu, gk[i], o);
    }
    if (slot == 0 && on_row) {
      s_sum[warp][0][c * 8 + i] = gq[i];
      s_sum[warp][1][c * 8 + i] = gk[i];
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

// dw = (dw +) sum of the blocks' shares: a block takes 32 columns, its eight warps every eighth share, then the eight sums
// in warp order
__global__ void __launch_bounds__(256) qk_weight_grad_kernel(int head_dim, int blocks, const float *__restrict__ partial, bool accumulate,
                                                             __nv_bfloat16 *dwq, __nv_bfloat16 *dwk) {
  __shared__ float part[8][32];
  const int lane = threadIdx.x & 31, grp = threadIdx.x >> 5;
  const int i = blockIdx.x * 32 + lane;
  float s = 0.0f;
  if (i < 2 * head_dim) {
#pragma unroll 4
    for (int b = grp; b < blocks; b += 8) s += partial[(int64_t)b * 2 * head_dim + i];
  }
  part[grp][lane] = s;
  __syncthreads();
  if (grp != 0 || i >= 2 * head_dim) return;
  float t = 0.0f;
#pragma unroll
  for (int g = 0; g < 8; g++) t += part[g][lane];
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

// Warps per token: one, as long as the tokens alone give every SM 16 warps; else as many as there are rounds of heads, so that few
// tokens spread over the GPU.
constexpr int QKN_MANY_TOKENS = 148 * 16;
int qkn_parts(int tokens, int heads, int head_dim) {
  const int at_once = 32 / qkn_lanes(head_dim) * qkn::BATCH, rounds = (heads + at_once - 1) / at_once;
  return tokens >= QKN_MANY_TOKENS ? 1 : rounds;
}

int qkn_blocks(int tokens, int heads, int head_dim, int per_sm) {
  const int64_t units = (int64_t)tokens * qkn_parts(tokens, heads, head_dim);
  const int64_t want = (units + qkn::WARPS - 1) / qkn::WARPS, most = (int64_t)qkn_sms() * per_sm;
  return (int)(want < most ? want : most);
}
constexpr int QKN_FWD_PER_SM = 8, QKN_BWD_PER_SM = 4;

template <bool BWD>
int qkn_launch(const char *op, const qkn::Params &p, int blocks, cudaStream_t s) {
  switch (qkn_lanes(p.head_dim)) {
    case 1: qkn::qk_norm_rope_kernel<1, BWD><<<blocks, qkn::THREADS, 0, s>>>(p); break;
    case 2: qkn::qk_norm_rope_kernel<2, BWD><<<blocks, qkn::THREADS, 0, s>>>(p); break;
    case 4: qkn::qk_norm_rope_kernel<4, BWD><<<blocks, qkn::THREADS, 0, s>>>(p); break;
    case 8: qkn::qk_norm_rope_kernel<8, BWD><<<blocks, qkn::THREADS, 0, s>>>(p); break;
    case 16: qkn::qk_norm_rope_kernel<16, BWD><<<blocks, qkn::THREADS, 0, s>>>(p); break;
    default: qkn::qk_norm_rope_kernel<32, BWD><<<blocks, qkn::THREADS, 0, s>>>(p); break;
  }
  B200_CHECK_LAUNCH(op);
  return 0;
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
  p->parts = qkn_parts(num_tokens, p->heads, head_dim);
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
  return qkn_launch<false>("qk_norm_rope", p, qkn_blocks(num_tokens, p.heads, head_dim, QKN_FWD_PER_SM), (cudaStream_t)stream);
}

extern "C" uint64_t b200_qk_norm_rope_bwd_workspace_bytes(int num_tokens, int num_q_heads, int num_kv_heads, int head_dim) {
  if (num_tokens <= 0 || num_q_heads < 1 || num_kv_heads < 0 || head_dim < 8 || head_dim % 8 || head_dim > qkn::MAX_HEAD_DIM) return 0;
  // enough for every smaller number of tokens too: the most blocks may run just below the border between the two layouts
  const int below = num_tokens < QKN_MANY_TOKENS ? num_tokens : QKN_MANY_TOKENS - 1, heads = num_q_heads + num_kv_heads;
  const int a = qkn_blocks(num_tokens, heads, head_dim, QKN_BWD_PER_SM), b = qkn_blocks(below, heads, head_dim, QKN_BWD_PER_SM);
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
  if (num_tokens == 0) {  // the sums over no tokens
    if (dq_weight && !accumulate) B200_CUDA(cudaMemsetAsync(dq_weight, 0, (size_t)head_dim * 2, (cudaStream_t)stream));
    if (dk_weight && !accumulate) B200_CUDA(cudaMemsetAsync(dk_weight, 0, (size_t)head_dim * 2, (cudaStream_t)stream));
    return 0;
  }
  B200_REQUIRE(d_out_q && (num_kv_heads == 0 || d_out_k) && b200_aligned16(d_out_q) && b200_aligned16(d_out_k),
               "qk_norm_rope_bwd: the upstream gradients must be given and 16-byte aligned");
  const int blocks = qkn_blocks(num_tokens, p.heads, head_dim, QKN_BWD_PER_SM);
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
  qkn::qk_weight_grad_kernel<<<(2 * head_dim + 31) / 32, 256, 0, (cudaStream_t)stream>>>(
      head_dim, blocks, p.partial, accumulate != 0, (__nv_bfloat16 *)dq_weight, (__nv_bfloat16 *)dk_weight);
  B200_CHECK_LAUNCH("qk_norm_rope_bwd (weights)");
  return 0;
}
