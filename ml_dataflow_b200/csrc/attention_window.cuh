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

// Fills the table with the next sequences that have work, at most MAX_SEQS; units_of gives a sequence's number of work units.
// Returns the units in the table.
template <typename F>
int next_sequences(SeqTable &t, int *next, const Call &c, F units_of) {
  t.n = 0;
  t.first[0] = 0;
  while (*next < c.num_seqs && t.n < MAX_SEQS) {
    const int s = (*next)++, units = units_of(s);
    if (units == 0) continue;
    t.q_off[t.n] = c.q_off[s];
    t.Tq[t.n] = c.q_len[s];
    t.k_off[t.n] = c.k_off[s];
    t.Tk[t.n] = c.k_len[s];
    t.first[t.n + 1] = t.first[t.n] + units;
    t.n++;
  }
  return t.first[t.n];
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
