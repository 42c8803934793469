// Causal attention with a sliding window and sink tokens, forward and backward, over packed variable-length sequences with
// grouped query heads. Position p of a sequence sees key j iff j <= p and (p - j < window or j < num_sinks); the last query
// of a sequence stands at its last key.
//
//   s_pj = q_p . k_j / sqrt(head_dim),  lse_p = log sum_j exp(s_pj),  o_p = sum_j exp(s_pj - lse_p) v_j
// and backwards, with P = exp(S - lse), delta_p = do_p . o_p:
//   dV = P^T dO,   dS = P o (dO V^T - delta),   dQ = dS K / sqrt(head_dim),   dK = dS^T Q / sqrt(head_dim)
//
// This file holds the entry points and the form for head sizes that have no tensor-core kernel. It runs on the fp32 units: a warp
// per (query row, head), or per (key, key/value head) for dK and dV, walks the visible rows 32 at a time - a lane per row for the
// dot products, then a lane per dimension for the sums. Only visible rows are read, so what masked rows hold never matters, and
// every sum has a fixed order: two runs give the same bits. Latency of the dependent row loads bounds it: a window of 1024 over 8192 tokens
// of 16 heads of 128 takes 62 ms forward and backward this way, 410 us on the tensor cores.
#include <math.h>

#include <algorithm>
#include <memory>
#include <new>

#include "attention_window.cuh"
#include "common.cuh"
#include "../../include/b200_moe.h"

namespace b200 {
namespace window {

constexpr int THREADS = 128, WARPS = THREADS / 32;
constexpr int MAX_HEAD_DIM = 256;
constexpr float LOG2E = 1.4426950408889634f;

struct Params {
  SeqTable seqs;
  int window, sinks, q_heads, kv_heads, head_dim, total_q;
  float scale;
  const __nv_bfloat16 *q, *k, *v, *o, *dout;
  const float *lse_in;
  float *lse, *delta;  // [q_heads][total_q]
  __nv_bfloat16 *out, *dq, *dk, *dv;
};

__device__ __forceinline__ float dot_row(const float *a, const __nv_bfloat16 *row, int head_dim) {
  float s = 0.0f;
  for (int d = 0; d < head_dim; d += 8) {
    float f[8];
    unpack8(*reinterpret_cast<const uint4 *>(row + d), f);
#pragma unroll
    for (int i = 0; i < 8; i++) s = fmaf(a[d + i], f[i], s);
  }
  return s;
}

struct Row {  // one unit of a launch: row r of a sequence's queries (or keys), head h
  int q_off, Tq, k_off, Tk, r, h;
  bool ok;
};
__device__ __forceinline__ Row row_of(const Params &p, int heads) {
  Row w;
  const int64_t unit = (int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5);
  w.ok = unit < (int64_t)p.seqs.first[p.seqs.n] * heads;
  const int row = w.ok ? (int)(unit / heads) : 0;
  w.h = w.ok ? (int)(unit % heads) : 0;
  int s = 0;
  while (row >= p.seqs.first[s + 1]) s++;
  w.q_off = p.seqs.q_off[s];
  w.Tq = p.seqs.Tq[s];
  w.k_off = p.seqs.k_off[s];
  w.Tk = p.seqs.Tk[s];
  w.r = row - p.seqs.first[s];
  return w;
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// one pass over the visible keys with the running maximum and sum
__global__ void __launch_bounds__(THREADS) rows_fwd_kernel(const __grid_constant__ Params p) {
  __shared__ float s_q[WARPS][MAX_HEAD_DIM];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, hd = p.head_dim;
  const Row w = row_of(p, p.q_heads);
  if (!w.ok) return;
  const int64_t ldq = (int64_t)p.q_heads * hd, ldk = (int64_t)p.kv_heads * hd;
  const int pos = w.r + w.Tk - w.Tq, lo = max(0, pos - p.window + 1), sinks = min(p.sinks, lo);
  const int kvh = w.h / (p.q_heads / p.kv_heads);
  const int64_t qat = (int64_t)(w.q_off + w.r) * ldq + (int64_t)w.h * hd;
  const __nv_bfloat16 *K = p.k + (int64_t)w.k_off * ldk + (int64_t)kvh * hd, *V = p.v + (int64_t)w.k_off * ldk + (int64_t)kvh * hd;
  for (int d = lane; d < hd; d += 32) s_q[warp][d] = __bfloat162float(p.q[qat + d]) * p.scale;
  __syncwarp();
  float m = -INFINITY, l = 0.0f, acc[MAX_HEAD_DIM / 32];
#pragma unroll
  for (int i = 0; i < MAX_HEAD_DIM / 32; i++) acc[i] = 0.0f;
  const int count = sinks + pos - lo + 1;  // visible keys: the sinks, then the window
  for (int base = 0; base < count; base += 32) {
    const int at = base + lane, key = at < sinks ? at : lo + at - sinks;
    const float s = at < count ? dot_row(s_q[warp], K + key * ldk, hd) : -INFINITY;
    const float nm = fmaxf(m, warp_max(s));
    // every visible score may be -inf (a query of infinities): nothing has weight then
    const float alpha = nm == -INFINITY ? 1.0f : exp2f((m - nm) * LOG2E), pr = s == -INFINITY ? 0.0f : exp2f((s - nm) * LOG2E);
    m = nm;
    l = l * alpha + warp_sum(pr);
#pragma unroll
    for (int i = 0; i < MAX_HEAD_DIM / 32; i++) acc[i] *= alpha;
    for (int j = 0; j < min(32, count - base); j++) {
      const float pj = __shfl_sync(0xffffffffu, pr, j);
      const __nv_bfloat16 *v = V + (int64_t)__shfl_sync(0xffffffffu, key, j) * ldk;
#pragma unroll
      for (int i = 0; i < MAX_HEAD_DIM / 32; i++)
        if (i * 32 + lane < hd) acc[i] = fmaf(pj, __bfloat162float(v[i * 32 + lane]), acc[i]);
    }
  }
  const float inv = 1.0f / l;
#pragma unroll
  for (int i = 0; i < MAX_HEAD_DIM / 32; i++)
    if (i * 32 + lane < hd) p.out[qat + i * 32 + lane] = __float2bfloat16_rn(acc[i] * inv);
  if (lane == 0) p.lse[(int64_t)w.h * p.total_q + w.q_off + w.r] = m + logf(l);
}

// delta and dQ of a (query row, head)
__global__ void __launch_bounds__(THREADS) rows_bwd_q_kernel(const __grid_constant__ Params p) {
  __shared__ float s_q[WARPS][MAX_HEAD_DIM], s_do[WARPS][MAX_HEAD_DIM];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, hd = p.head_dim;
  const Row w = row_of(p, p.q_heads);
  if (!w.ok) return;
  const int64_t ldq = (int64_t)p.q_heads * hd, ldk = (int64_t)p.kv_heads * hd;
  const int pos = w.r + w.Tk - w.Tq, lo = max(0, pos - p.window + 1), sinks = min(p.sinks, lo);
  const int kvh = w.h / (p.q_heads / p.kv_heads);
  const int64_t qat = (int64_t)(w.q_off + w.r) * ldq + (int64_t)w.h * hd, stat = (int64_t)w.h * p.total_q + w.q_off + w.r;
  const __nv_bfloat16 *K = p.k + (int64_t)w.k_off * ldk + (int64_t)kvh * hd, *V = p.v + (int64_t)w.k_off * ldk + (int64_t)kvh * hd;
  float delta = 0.0f;
  for (int d = lane; d < hd; d += 32) {
    s_q[warp][d] = __bfloat162float(p.q[qat + d]) * p.scale;
    s_do[warp][d] = __bfloat162float(p.dout[qat + d]);
    delta = fmaf(s_do[warp][d], __bfloat162float(p.o[qat + d]), delta);
  }
  delta = warp_sum(delta);
  if (lane == 0) p.delta[stat] = delta;
  __syncwarp();
  const float lse = p.lse_in[stat];
  float acc[MAX_HEAD_DIM / 32];
#pragma unroll
  for (int i = 0; i < MAX_HEAD_DIM / 32; i++) acc[i] = 0.0f;
  const int count = sinks + pos - lo + 1;
  for (int base = 0; base < count; base += 32) {
    const int at = base + lane, key = at < sinks ? at : lo + at - sinks;
    float ds = 0.0f;
    if (at < count) {
      const float pr = exp2f((dot_row(s_q[warp], K + key * ldk, hd) - lse) * LOG2E);
      ds = pr * (dot_row(s_do[warp], V + key * ldk, hd) - delta) * p.scale;
    }
    for (int j = 0; j < min(32, count - base); j++) {
      const float dj = __shfl_sync(0xffffffffu, ds, j);
      const __nv_bfloat16 *k = K + (int64_t)__shfl_sync(0xffffffffu, key, j) * ldk;
#pragma unroll
      for (int i = 0; i < MAX_HEAD_DIM / 32; i++)
        if (i * 32 + lane < hd) acc[i] = fmaf(dj, __bfloat162float(k[i * 32 + lane]), acc[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < MAX_HEAD_DIM / 32; i++)
    if (i * 32 + lane < hd) p.dq[qat + i * 32 + lane] = __float2bfloat16_rn(acc[i]);
}

// dK and dV of a (key, key/value head): the queries of every head of the group that see the key
__global__ void __launch_bounds__(THREADS) rows_bwd_kv_kernel(const __grid_constant__ Params p) {
  __shared__ float s_k[WARPS][MAX_HEAD_DIM], s_v[WARPS][MAX_HEAD_DIM];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, hd = p.head_dim, group = p.q_heads / p.kv_heads;
  const Row w = row_of(p, p.kv_heads);
  if (!w.ok) return;
  const int64_t ldq = (int64_t)p.q_heads * hd, ldk = (int64_t)p.kv_heads * hd;
  const int64_t kat = (int64_t)(w.k_off + w.r) * ldk + (int64_t)w.h * hd;
  for (int d = lane; d < hd; d += 32) {
    s_k[warp][d] = __bfloat162float(p.k[kat + d]) * p.scale;
    s_v[warp][d] = __bfloat162float(p.v[kat + d]);
  }
  __syncwarp();
  const int shift = w.Tk - w.Tq;
  const int first = max(0, w.r - shift), last = w.r < p.sinks ? w.Tq - 1 : (int)min((int64_t)w.Tq - 1, (int64_t)w.r + p.window - 1 - shift);
  float dk[MAX_HEAD_DIM / 32], dv[MAX_HEAD_DIM / 32];
#pragma unroll
  for (int i = 0; i < MAX_HEAD_DIM / 32; i++) dk[i] = dv[i] = 0.0f;
  for (int g = 0; g < group; g++) {
    const int h = w.h * group + g;
    for (int base = first; base <= last; base += 32) {
      const int row = base + lane;
      const int64_t qat = (int64_t)(w.q_off + min(row, last)) * ldq + (int64_t)h * hd;
      float pr = 0.0f, ds = 0.0f;
      if (row <= last) {
        const int64_t stat = (int64_t)h * p.total_q + w.q_off + row;
        pr = exp2f((dot_row(s_k[warp], p.q + qat, hd) - p.lse_in[stat]) * LOG2E);
        ds = pr * (dot_row(s_v[warp], p.dout + qat, hd) - p.delta[stat]) * p.scale;
      }
      for (int j = 0; j < min(32, last - base + 1); j++) {
        const float pj = __shfl_sync(0xffffffffu, pr, j), dj = __shfl_sync(0xffffffffu, ds, j);
        const int64_t at = __shfl_sync(0xffffffffu, qat, j);
#pragma unroll
        for (int i = 0; i < MAX_HEAD_DIM / 32; i++)
          if (i * 32 + lane < hd) {
            dk[i] = fmaf(dj, __bfloat162float(p.q[at + i * 32 + lane]), dk[i]);
            dv[i] = fmaf(pj, __bfloat162float(p.dout[at + i * 32 + lane]), dv[i]);
          }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < MAX_HEAD_DIM / 32; i++)
    if (i * 32 + lane < hd) {
      p.dk[kat + i * 32 + lane] = __float2bfloat16_rn(dk[i]);
      p.dv[kat + i * 32 + lane] = __float2bfloat16_rn(dv[i]);
    }
}

}  // namespace window
}  // namespace b200

using namespace b200;

namespace {

// Two sequences must not write the same rows. Offsets usually ascend, and one pass shows it; else the rows are sorted first.
int disjoint(const char *op, const char *what, int num_seqs, const int *off, const int *len) {
  int64_t end = 0;
  bool ascending = true;
  for (int s = 0; s < num_seqs && ascending; s++) {
    if (len[s] == 0) continue;
    ascending = off[s] >= end;
    end = (int64_t)off[s] + len[s];
  }
  if (ascending) return 0;
  std::unique_ptr<int[]> order(new (std::nothrow) int[num_seqs]);
  B200_REQUIRE(order != nullptr, "%s: no memory to sort %d sequences", op, num_seqs);
  int n = 0;
  for (int s = 0; s < num_seqs; s++)
    if (len[s] > 0) order[n++] = s;
  std::sort(order.get(), order.get() + n, [&](int a, int b) { return off[a] < off[b]; });
  for (int i = 1; i < n; i++)
    B200_REQUIRE((int64_t)off[order[i - 1]] + len[order[i - 1]] <= off[order[i]], "%s: the %s rows of sequences %d and %d overlap", op, what, order[i - 1],
                 order[i]);
  return 0;
}

// The outputs, first n_out of the tensors, must lie apart from one another and from the inputs behind them: units of a launch, and the launches
// of a backward, read rows that others have written by then.
struct Range {
  const void *at;
  uint64_t bytes;
};
int apart(const char *op, const Range *t, int n_out, int n) {
  for (int i = 0; i < n_out; i++)
    for (int j = i + 1; j < n; j++) {
      const uintptr_t a = reinterpret_cast<uintptr_t>(t[i].at), b = reinterpret_cast<uintptr_t>(t[j].at);
      B200_REQUIRE(t[i].bytes == 0 || t[j].bytes == 0 || (a < b ? a + t[i].bytes <= b : b + t[j].bytes <= a),
                   "%s: an output overlaps another tensor", op);
    }
  return 0;
}

int window_check(const char *op, int dt, int num_seqs, int total_q, int total_k, const int *q_off, const int *q_len, const int *k_off,
                 const int *k_len, int num_q_heads, int num_kv_heads, int head_dim, int window, int num_sinks) {
  B200_REQUIRE(dt == B200_DT_BF16, "%s: only bf16 is implemented (datatype code %d)", op, dt);
  B200_REQUIRE(num_seqs >= 0 && total_q >= 0 && total_k >= 0 && (num_seqs == 0 || (q_off && q_len && k_off && k_len)),
               "%s: bad sequence description", op);
  B200_REQUIRE(num_q_heads >= 1 && num_kv_heads >= 1 && num_q_heads <= 65536 && num_q_heads % num_kv_heads == 0,
               "%s: query heads must be a multiple of the key/value heads (%d, %d)", op, num_q_heads, num_kv_heads);
  B200_REQUIRE(head_dim >= 8 && head_dim % 8 == 0 && head_dim <= b200::window::MAX_HEAD_DIM, "%s: head_dim must be a multiple of 8, at most %d (got %d)",
               op, b200::window::MAX_HEAD_DIM, head_dim);
  B200_REQUIRE(window >= 1 && num_sinks >= 0, "%s: need window >= 1 and num_sinks >= 0 (got %d, %d)", op, window, num_sinks);
  for (int s = 0; s < num_seqs; s++) {
    B200_REQUIRE(q_len[s] >= 0 && k_len[s] >= q_len[s] && q_off[s] >= 0 && k_off[s] >= 0 && (int64_t)q_off[s] + q_len[s] <= total_q &&
                     (int64_t)k_off[s] + k_len[s] <= total_k,
                 "%s: sequence %d (q %d+%d of %d, k %d+%d of %d; keys >= queries)", op, s, q_off[s], q_len[s], total_q, k_off[s], k_len[s],
                 total_k);
  }
  return disjoint(op, "query", num_seqs, q_off, q_len);
}

// the form without tensor cores: a unit of a launch is a row
window::Params rows_params(const window::Call &c) {
  window::Params p{};
  p.window = c.window;
  p.sinks = c.sinks;
  p.q_heads = c.q_heads;
  p.kv_heads = c.kv_heads;
  p.head_dim = c.head_dim;
  p.total_q = c.total_q;
  p.scale = c.scale;
  p.q = c.q;
  p.k = c.k;
  p.v = c.v;
  p.o = c.o;
  p.dout = c.dout;
  p.lse_in = c.lse_in;
  p.lse = c.lse;
  p.delta = (float *)c.workspace;
  p.out = c.out;
  p.dq = c.dq;
  p.dk = c.dk;
  p.dv = c.dv;
  return p;
}

uint64_t bwd_workspace(int num_seqs, int q_heads, int kv_heads, int head_dim, int total_q, int sinks) {
  if (window::sm100_supported(head_dim)) return window::sm100_bwd_workspace(num_seqs, q_heads, kv_heads, head_dim, total_q, sinks);
  return ((uint64_t)total_q * q_heads * sizeof(float) + 255) / 256 * 256;  // delta
}

unsigned blocks_for(int64_t warps) { return (unsigned)((warps + window::WARPS - 1) / window::WARPS); }

int rows_fwd(const window::Call &c) {
  window::Params p = rows_params(c);
  for (int next = 0; next < c.num_seqs;) {
    const int64_t rows = window::next_sequences(p.seqs, &next, c, [&](int s) { return c.q_len[s]; }, [](int) { return 0; });
    if (rows == 0) continue;
    window::rows_fwd_kernel<<<blocks_for(rows * c.q_heads), window::THREADS, 0, c.stream>>>(p);
    B200_CHECK_LAUNCH("attention_window_fwd");
    count_launch();
  }
  return 0;
}

int rows_bwd(const window::Call &c) {
  window::Params p = rows_params(c);
  for (int next = 0; next < c.num_seqs;) {
    const int64_t rows = window::next_sequences(p.seqs, &next, c, [&](int s) { return c.q_len[s]; }, [](int) { return 0; });
    if (rows == 0) continue;
    window::rows_bwd_q_kernel<<<blocks_for(rows * c.q_heads), window::THREADS, 0, c.stream>>>(p);
    B200_CHECK_LAUNCH("attention_window_bwd (dQ)");
    count_launch();
  }
  for (int next = 0; next < c.num_seqs;) {
    const int64_t rows = window::next_sequences(p.seqs, &next, c, [&](int s) { return c.k_len[s]; }, [](int) { return 0; });
    if (rows == 0) continue;
    window::rows_bwd_kv_kernel<<<blocks_for(rows * c.kv_heads), window::THREADS, 0, c.stream>>>(p);
    B200_CHECK_LAUNCH("attention_window_bwd (dK, dV)");
    count_launch();
  }
  return 0;
}

void fill_call(window::Call *c, int num_seqs, int total_q, int total_k, const int *q_off, const int *q_len, const int *k_off, const int *k_len,
               int num_q_heads, int num_kv_heads, int head_dim, const void *x_q, const void *x_k, const void *x_v, int window_, int num_sinks,
               void *stream) {
  c->num_seqs = num_seqs;
  c->total_q = total_q;
  c->total_k = total_k;
  c->q_off = q_off;
  c->q_len = q_len;
  c->k_off = k_off;
  c->k_len = k_len;
  c->q_heads = num_q_heads;
  c->kv_heads = num_kv_heads;
  c->head_dim = head_dim;
  // More than all keys changes nothing, and positions plus these stay within 32 bits. (The sinks stay above what decides on the workspace.)
  c->window = window_ < total_k ? window_ : total_k;
  const int most_sinks = total_k > (1 << 20) ? total_k : 1 << 20;
  c->sinks = num_sinks < most_sinks ? num_sinks : most_sinks;
  c->scale = 1.0f / sqrtf((float)head_dim);
  c->q = (const __nv_bfloat16 *)x_q;
  c->k = (const __nv_bfloat16 *)x_k;
  c->v = (const __nv_bfloat16 *)x_v;
  c->stream = (cudaStream_t)stream;
}

}  // namespace

extern "C" uint64_t b200_attention_window_workspace_bytes(int num_seqs, int num_q_heads, int num_kv_heads, int head_dim, int max_total_q,
                                                          int num_sinks) {
  if (num_seqs <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 || max_total_q <= 0 || num_sinks < 0) return 0;
  return bwd_workspace(num_seqs, num_q_heads, num_kv_heads, head_dim, max_total_q, num_sinks);
}

extern "C" int b200_attention_window_fwd(int fwd_dt, int num_seqs, int total_q, int total_k, const int *q_seq_offsets, const int *q_seq_lens,
                                         const int *k_seq_offsets, const int *k_seq_lens, int num_q_heads, int num_kv_heads, int head_dim,
                                         const void *x_q, const void *x_k, const void *x_v, void *x_attn_out, float *softmax_lse, int window,
                                         int num_sinks, void *stream) {
  if (window_check("attention_window_fwd", fwd_dt, num_seqs, total_q, total_k, q_seq_offsets, q_seq_lens, k_seq_offsets, k_seq_lens,
                   num_q_heads, num_kv_heads, head_dim, window, num_sinks))
    return -1;
  bool any = false;
  for (int s = 0; s < num_seqs && !any; s++) any = q_seq_lens[s] > 0;
  if (!any) return 0;
  B200_REQUIRE(x_q && x_k && x_v && x_attn_out && softmax_lse, "attention_window_fwd: null tensor");
  B200_REQUIRE(b200_aligned16(x_q) && b200_aligned16(x_k) && b200_aligned16(x_v) && b200_aligned16(x_attn_out),
               "attention_window_fwd: tensors must be 16-byte aligned");
  const uint64_t nq = (uint64_t)total_q * num_q_heads, nk = (uint64_t)total_k * num_kv_heads, row = (uint64_t)head_dim * 2;
  const Range t[] = {{x_attn_out, nq * row}, {softmax_lse, nq * 4}, {x_q, nq * row}, {x_k, nk * row}, {x_v, nk * row}};
  if (apart("attention_window_fwd", t, 2, 5)) return -1;
  window::Call c{};
  fill_call(&c, num_seqs, total_q, total_k, q_seq_offsets, q_seq_lens, k_seq_offsets, k_seq_lens, num_q_heads, num_kv_heads, head_dim, x_q,
            x_k, x_v, window, num_sinks, stream);
  c.out = (__nv_bfloat16 *)x_attn_out;
  c.lse = softmax_lse;
  return window::sm100_supported(head_dim) ? window::sm100_fwd(c) : rows_fwd(c);
}

extern "C" int b200_attention_window_bwd(int bwd_dt, int num_seqs, int total_q, int total_k, const int *q_seq_offsets, const int *q_seq_lens,
                                         const int *k_seq_offsets, const int *k_seq_lens, int num_q_heads, int num_kv_heads, int head_dim,
                                         const void *x_q, const void *x_k, const void *x_v, const void *x_attn_out, const float *softmax_lse,
                                         const void *dx_out, void *dx_q, void *dx_k, void *dx_v, int window, int num_sinks,
                                         uint64_t workspaceBytes, void *workspace, void *stream) {
  if (window_check("attention_window_bwd", bwd_dt, num_seqs, total_q, total_k, q_seq_offsets, q_seq_lens, k_seq_offsets, k_seq_lens,
                   num_q_heads, num_kv_heads, head_dim, window, num_sinks))
    return -1;
  if (disjoint("attention_window_bwd", "key", num_seqs, k_seq_offsets, k_seq_lens)) return -1;
  if (num_seqs == 0 || total_k == 0) return 0;
  B200_REQUIRE(x_k && x_v && dx_k && dx_v && (total_q == 0 || (x_q && x_attn_out && softmax_lse && dx_out && dx_q)),
               "attention_window_bwd: null tensor");
  B200_REQUIRE(b200_aligned16(x_q) && b200_aligned16(x_k) && b200_aligned16(x_v) && b200_aligned16(x_attn_out) && b200_aligned16(dx_out) &&
                   b200_aligned16(dx_q) && b200_aligned16(dx_k) && b200_aligned16(dx_v),
               "attention_window_bwd: tensors must be 16-byte aligned");
  const uint64_t need = bwd_workspace(num_seqs, num_q_heads, num_kv_heads, head_dim, total_q, num_sinks);
  B200_REQUIRE(total_q == 0 || (workspace && b200_aligned16(workspace) && workspaceBytes >= need),
               "attention_window_bwd: the workspace holds %llu bytes, %llu are needed (b200_attention_window_workspace_bytes)",
               (unsigned long long)workspaceBytes, (unsigned long long)need);
  const uint64_t nq = (uint64_t)total_q * num_q_heads, nk = (uint64_t)total_k * num_kv_heads, row = (uint64_t)head_dim * 2;
  const Range t[] = {{dx_q, nq * row}, {dx_k, nk * row}, {dx_v, nk * row},       {workspace, total_q ? need : 0}, {x_q, nq * row},
                     {x_k, nk * row},  {x_v, nk * row},  {x_attn_out, nq * row}, {softmax_lse, nq * 4},           {dx_out, nq * row}};
  if (apart("attention_window_bwd", t, 4, 10)) return -1;
  window::Call c{};
  fill_call(&c, num_seqs, total_q, total_k, q_seq_offsets, q_seq_lens, k_seq_offsets, k_seq_lens, num_q_heads, num_kv_heads, head_dim, x_q,
            x_k, x_v, window, num_sinks, stream);
  c.o = (const __nv_bfloat16 *)x_attn_out;
  c.lse_in = softmax_lse;
  c.dout = (const __nv_bfloat16 *)dx_out;
  c.dq = (__nv_bfloat16 *)dx_q;
  c.dk = (__nv_bfloat16 *)dx_k;
  c.dv = (__nv_bfloat16 *)dx_v;
  c.workspace = (unsigned char *)workspace;
  return window::sm100_supported(head_dim) ? window::sm100_bwd(c) : rows_bwd(c);
}
