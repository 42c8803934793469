// Windowed attention, what its files share: one call's arguments, and the sequences of one launch.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace b200 {
namespace window {

// Work units of a launch are numbered through its sequences: those of sequence s are first[s] .. first[s + 1] - 1.
constexpr int MAX_SEQS = 48;
struct SeqTable {
  int n;
  int q_off[MAX_SEQS], Tq[MAX_SEQS], k_off[MAX_SEQS], Tk[MAX_SEQS], first[MAX_SEQS + 1];
};

// One call; its arguments have been checked.
struct Call {
  int num_seqs, total_q, total_k;
  const int *q_off, *q_len, *k_off, *k_len;  // host
  int q_heads, kv_heads, head_dim, window, sinks;
  float scale;
  const __nv_bfloat16 *q, *k, *v;
  __nv_bfloat16 *out;    // forward
  float *lse;
  const __nv_bfloat16 *o, *dout;  // backward
  const float *lse_in;
  __nv_bfloat16 *dq, *dk, *dv;
  unsigned char *workspace;
  cudaStream_t stream;
};

// Fills the table with the next sequences that have work, at most MAX_SEQS; units_of gives a sequence's number of work units, steps_of
// how long its longest one is. The sequences with the longest units come first, so that the short ones fill in behind them (a call
// over three chunks of prompts whose units see up to 19, 7 and 10 blocks: 61.6 us, in the caller's order 71.3). Returns the units in the table.
template <typename F, typename G>
int next_sequences(SeqTable &t, int *next, const Call &c, F units_of, G steps_of) {
  int index[MAX_SEQS], steps[MAX_SEQS];
  t.n = 0;
  t.first[0] = 0;
  while (*next < c.num_seqs && t.n < MAX_SEQS) {
    const int s = (*next)++;
    if (units_of(s) == 0) continue;
    const int key = steps_of(s);
    int at = t.n++;
    for (; at > 0 && steps[at - 1] < key; at--) {
      steps[at] = steps[at - 1];
      index[at] = index[at - 1];
    }
    steps[at] = key;
    index[at] = s;
  }
  for (int i = 0; i < t.n; i++) {
    const int s = index[i];
    t.q_off[i] = c.q_off[s];
    t.Tq[i] = c.q_len[s];
    t.k_off[i] = c.k_off[s];
    t.Tk[i] = c.k_len[s];
    t.first[i + 1] = t.first[i] + units_of(s);
  }
  return t.first[t.n];
}

// Clusters of `size` CTAs that the current device seats at once, asked for on first use and kept in *known; 0 where it cannot tell. A cluster lies
// within one GPC: here 15 of eight and 33 of four CTAs that fill an SM, where 148 SMs would hold 18 and 37. The kernel's shared memory has been allowed.
template <typename K>
int cluster_seats(K kernel, int threads, size_t smem, int size, int *known) {
  if (*known == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)size);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)size;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
      cudaGetLastError();
      n = 0;
    }
    *known = n > 0 ? n : -1;
  }
  return *known > 0 ? *known : 0;
}

// attention_window_sm100.cu: tensor-core kernels for head sizes 64 and 128
bool sm100_supported(int head_dim);
int sm100_fwd(const Call &c);
// attention_window_few.cu: its forward for sequences with few queries
bool is_few(const Call &c, int s);
int few_fwd(const Call &c);
uint64_t sm100_bwd_workspace(int num_seqs, int q_heads, int kv_heads, int head_dim, int total_q, int sinks);
int sm100_bwd(const Call &c);

}  // namespace window
}  // namespace b200
