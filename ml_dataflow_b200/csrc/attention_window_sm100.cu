// Windowed attention with sinks on the tensor cores, head sizes 64 and 128.
//
// Forward. A work unit is a pair of 128-row query tiles that read the same keys: two query heads of one key/value head over
// the same rows (or, where the group is odd, two neighbouring tiles of one head); in the last round, one of them. Key blocks of 128 that no row of the pair
// sees are never touched: the unit walks the blocks that hold sinks, then those of its window. A persistent CTA (one per SM)
// takes units in turn: while one unit's last products and its output are under way, the next one's queries and keys load.
//   warp 0     TMA loads: the query tiles, and K_0, K_1, V_0, K_2, V_1, ... through a ring, in the order they are used
//   warp 1     one thread issues the tcgen05 MMAs  S_g = Q_g K^T   (fp32 accumulators in tensor memory)
//   warps 2, 3 one thread each issues  O_g += P_g V  of its tile. Three issuers, because a wait costs an issuing thread about 250
//              cycles and the tensor pipe queues less than that: with a single one that waited for all of it in turn a step of a
//              pair took 5600 cycles
//   warps 4-11 four per tile, a thread per query row: scores to registers at once - which frees the accumulator for the next
//              S, so that the tensor cores work while the exponentials are formed -, running maximum and sum,
//              P = exp2((S - m) scale log2 e) as bf16 through shared (head size 64: tensor) memory. The second tile starts when the first has formed its
//              first P: one's waits and loads then lie under the other's exponentials
// The maximum is raised, and O and the sum rescaled, only when a block's maximum exceeds it by more than 2^8.
// Rounding: scores, statistics and accumulators fp32; P to bf16 (relative to m) before it multiplies V, the tensor cores take
// no wider operand beside bf16 values; one rounding of the output.
// Rows of V that no query of the sequence sees (before its first window, past its end) are zeroed in shared memory, so that
// whatever they hold never meets the tensor cores; the scores of masked keys are dropped by a select.
//
// What bounds it, at head size 128: shared memory. A step of a pair moves 384 KB through it - 256 that four products read, 64 of P, 64 of K and V
// that arrive -, 3070 cycles at 128 bytes each; a product of 128 x 128 x 128 alone takes 727 cycles for its 64 KB. A step takes 4000. At head size
// 64 there is room for P in tensor memory, where the product takes its rows from: 9 to 11 % less time than through shared memory. At 128 it would
// have to lie over S, and the next S then waits for P V (no window: 247 -> 299 us).
// Measured with 16 query heads on 4 of 128 and 8192 tokens: window 1024 96 us (65 GFLOP of visible pairs: 670 TFLOP/s; 86 with the masked parts
// of the blocks), no window 238 us (1155 TFLOP/s; the causal kernel without windows 330 us); heads of 64: 79 and 207 us. Tried and slower: the second
// half of the scores' columns on 8 more warps that exchange maxima (127 us where this took 108), sink blocks in a form of 32 columns (their step is
// shorter, the others' longer: 103 -> 106 us).
//
// Every wait is bounded; one that runs out raises the status word that b200_attention_status reads, and the CTA leaves.
#include <cuda.h>
#include <math.h>
#include <stddef.h>

#include <algorithm>

#include "attention_sm100.cuh"
#include "attention_window.cuh"
#include "common.cuh"
#include "sm100_ptx.cuh"
#include "../../include/b200_moe.h"

namespace b200 {
namespace window {

using fa::ex2;
using fa::sts128;

constexpr int TILE = 128;     // query rows of a tile, keys of a block
constexpr int SLAB = 16384;   // 128 rows x 64 bf16, one swizzled slab
// Forward: 4 warps that load and issue, 8 that compute. A thread of these holds a row of 128 scores: the launch gives 168 registers to each
// of the three warpgroups' threads, the loading and issuing one hands 96 of them on (72 + 2 * 216 = 3 * 168).
constexpr int FWD_THREADS = 384, REGS_CONTROL = 72, REGS_SOFTMAX = 216;
static_assert(REGS_CONTROL + 2 * REGS_SOFTMAX <= 3 * 168, "a split of more registers than the launch has would wait for ever");
// Backward, dK and dV: 4 warps that load and issue, 16 for the element-wise work.
constexpr int BWD_KV_THREADS = 640;
// Backward, dQ: 4 more that prepare a unit's row statistics and write the last one's output meanwhile. The launch gives 80 registers to
// each of the six warpgroups' threads, the first two hand 16 each on (2 * 64 + 4 * 88 = 6 * 80).
constexpr int BWD_Q_THREADS = 768, REGS_BWD_Q = 88, REGS_BWD_Q_OTHER = 64;
static_assert(2 * REGS_BWD_Q_OTHER + 4 * REGS_BWD_Q <= 6 * 80, "a split of more registers than the launch has would wait for ever");
constexpr float LOG2E = 1.4426950408889634f;

enum { ST_Q_EMPTY = 51, ST_KV_EMPTY, ST_Q_FULL, ST_KV_FULL, ST_S_FREE, ST_P, ST_O_FREE, ST_S, ST_PV, ST_FIX };

// Which units a persistent CTA takes, one after the other.
// Without a schedule: c, 2 G - 1 - c, 2 G + c, ... for G CTAs; units are numbered from the longest of a sequence on, so that a CTA that took a
// long one of a round takes a short one of the next.
// The forward of several sequences: the host deals the units out, the longest first, each to the CTA with the least work so far, and writes that
// down in runs: CTAs cta .. cta + n - 1 take units unit .. unit + n - 1. (16 heads on 4 of 128: eight sequences of 1024 tokens, window 512, 68 -> 59
// us; six of 700 to 2000, no window, 94 -> 79; the three chunks of prompts 61.5 -> 59.6. One sequence has nothing to gain, and the longer walk
// costs it 2 %, hence two kernels; dQ gained nothing.) A batch of more kinds of units, or more runs, than the tables hold goes in rounds after all: 24 ragged
// sequences of up to 2000 tokens with 16 heads take 6 % (window 512) to 12 % (no window) longer than dealt out from tables of three times the size.
constexpr int MAX_RUNS = 160;
struct Schedule {
  int n;
  struct Run {
    int unit;
    unsigned short cta, n;
  } run[MAX_RUNS];
};
__device__ __forceinline__ int unit_at(int round) {
  return (round & 1) ? (round + 1) * (int)gridDim.x - 1 - (int)blockIdx.x : round * (int)gridDim.x + (int)blockIdx.x;
}
// The forward of few units on many keys: the CTAs of a cluster share one, each takes a part of its blocks (join_parts below; 512 queries on 16384
// keys, 16 heads on 4 of 128: 184 -> 79 us).
enum { WALK_ROUNDS, WALK_DEALT, WALK_SHARED };
constexpr int MAX_SHARERS = 8;
template <int WALK>
struct Walk {
  int at = 0;
  // the CTA's next unit; `units` or more: no more
  template <typename P>
  __device__ __forceinline__ int next(const P &p) {
    if constexpr (WALK == WALK_ROUNDS) {
      return unit_at(at++);
    } else if constexpr (WALK == WALK_SHARED) {
      return at++ == 0 ? (int)blockIdx.x / p.cluster : p.units;
    } else {
      while (at < p.schedule.n) {
        const Schedule::Run r = p.schedule.run[at++];
        if ((unsigned)((int)blockIdx.x - r.cta) < (unsigned)r.n) return r.unit + (int)blockIdx.x - r.cta;
      }
      return p.units;
    }
  }
};

struct FwdParams {
  CUtensorMap tmQ, tmK, tmV;  // [rows][heads * HD] bf16, boxes of 64 columns x 128 rows, 128-byte swizzle
  SeqTable seqs;
  Schedule schedule;
  __nv_bfloat16 *O;
  float *lse;  // [q_heads][total_q]
  int window, sinks, group, q_heads, total_q, pair_heads, units;
  int whole;    // units from this one on are one tile of a pair each
  int cluster;  // CTAs that share a unit
  float scale;
  int *status;
};

template <int HD>
struct FwdShape {
  static constexpr bool P_IN_TMEM = HD == 64;  // where 128 of its columns are free
  static constexpr int Q_TILE = TILE * HD * 2, P_TILE = P_IN_TMEM ? 0 : TILE * TILE * 2, KV_TILE = TILE * HD * 2;
  static constexpr int SLOTS = HD == 128 ? 3 : 6, RING = 4;
  struct Tail {
    uint64_t q_full[2], q_empty[2], k_full[RING], v_full[RING], kv_empty[SLOTS], s_full[2], s_read[2], p_ready[2], pv_done[2], o_empty[2], begun, fixed;
    uint32_t tmem_base;
    int abort_flag;
  };
  static constexpr size_t smem = 1024 + 2 * (size_t)Q_TILE + 2 * (size_t)P_TILE + SLOTS * (size_t)KV_TILE + sizeof(Tail);
  static_assert(smem <= 232448, "more shared memory than a CTA can be given");
};

// Which keys a sequence's rows see.
struct Span {
  int q_off, Tq, k_off, Tk, shift;
};
__host__ __device__ __forceinline__ Span span_of(const SeqTable &t, int s) {
  return Span{t.q_off[s], t.Tq[s], t.k_off[s], t.Tk[s], t.Tk[s] - t.Tq[s]};
}

// One tile of a unit: its head, first row (Tq or more: no such tile) and the blocks of its window (hi inclusive).
struct Tile {
  int h, row, lo, hi;
  bool exists;
  __device__ __forceinline__ bool active(int kb, int sinks) const { return exists && kb <= hi && (kb >= lo || kb * TILE < sinks); }
};
// The key blocks of a pair of tiles: blocks 0 .. n_sink - 1 hold sinks and lie before the window, then first .. first + n - n_sink - 1.
struct Unit {
  Span sp;
  Tile a, b;
  int n, n_sink, first;
  __device__ __forceinline__ int block(int i) const { return i < n_sink ? i : first + i - n_sink; }
  // the blocks of this CTA: all, or its share
  template <int WALK>
  __device__ __forceinline__ int begin(int cluster) const { return WALK == WALK_SHARED ? n * ((int)blockIdx.x % cluster) / cluster : 0; }
  template <int WALK>
  __device__ __forceinline__ int end(int cluster) const { return WALK == WALK_SHARED ? n * ((int)blockIdx.x % cluster + 1) / cluster : n; }
};
__host__ __device__ __forceinline__ Tile tile_of(const Span &sp, int window, int h, int row) {
  Tile t;
  t.h = h;
  t.row = row;
  t.lo = max(0, row + sp.shift - window + 1) / TILE;
  t.hi = (min(row + TILE, sp.Tq) - 1 + sp.shift) / TILE;
  t.exists = row < sp.Tq;
  return t;
}
__host__ __device__ __forceinline__ Unit unit_of(const FwdParams &p, int unit) {
  Unit u;
  const int half = unit < p.whole ? 0 : 1 + ((unit - p.whole) & 1);  // 1, 2: the pair's first tile, its second
  if (half) unit = p.whole + ((unit - p.whole) >> 1);
  int s = 0;
  while (unit >= p.seqs.first[s + 1]) s++;
  u.sp = span_of(p.seqs, s);
  const int rel = unit - p.seqs.first[s], tiles = (u.sp.Tq + TILE - 1) / TILE;
  if (p.pair_heads) {
    const int pairs = p.q_heads >> 1, hp = rel % pairs, row = (tiles - 1 - rel / pairs) * TILE;
    u.a = tile_of(u.sp, p.window, 2 * hp, row);
    u.b = tile_of(u.sp, p.window, 2 * hp + 1, row);
  } else {
    const int row = ((tiles + 1) / 2 - 1 - rel / p.q_heads) * 2 * TILE;
    u.a = tile_of(u.sp, p.window, rel % p.q_heads, row);
    u.b = tile_of(u.sp, p.window, rel % p.q_heads, row + TILE);
  }
  if (half) {
    if (half == 2) u.a = u.b;
    u.b.exists = false;
  }
  u.first = u.a.lo;
  u.n_sink = min((p.sinks + TILE - 1) / TILE, u.first);
  u.n = u.a.exists ? u.n_sink + (u.b.exists ? u.b.hi : u.a.hi) - u.first + 1 : 0;  // a second tile that is not there
  return u;
}

// The MMA descriptors of a tile's 16-column steps differ from its first one by a constant in the address field; formed anew from
// `addr` where they are used (the compiler would else hold those of every tile in registers for the whole kernel).
__device__ __forceinline__ uint64_t tile_desc(uint32_t addr, uint32_t lbo) {
  asm volatile("" : "+r"(addr));
  return ptx::make_smem_desc(addr, lbo, 1024);
}
__device__ __forceinline__ uint64_t desc_at(uint64_t desc, uint32_t bytes) { return desc + (bytes >> 4); }

// The keys that a row sees in 32 columns, as bits: j <= hi and (j >= lo or j < sinks), all relative to the first column.
__device__ __forceinline__ uint32_t low_bits(int n) { return n >= 32 ? 0xffffffffu : (n <= 0 ? 0u : (1u << n) - 1u); }
__device__ __forceinline__ uint32_t seen_bits(int hi, int lo, int sinks) { return low_bits(hi + 1) & (~low_bits(lo) | low_bits(sinks)); }
// every row of a tile of queries at positions pos0 .. last sees every key of the block
__device__ __forceinline__ bool all_seen(int base, int pos0, int last, int window, int sinks) {
  return base + TILE - 1 <= pos0 && (base >= last - window + 1 || base + TILE <= sinks);
}

// x[j] = 2^(x[j] c + off). (A quarter of them by a polynomial on the FMA units, to relieve the special-function units, gave 1 % or took
// 3 % in the backward and took 15 % in the forward.)
template <int N>
__device__ __forceinline__ void probabilities(uint32_t *x, float c, float off) {
  const uint64_t cc = pack2(c, c), oo = pack2(off, off);
#pragma unroll
  for (int j = 0; j < N; j += 2) {
    float a, b;
    unpack2(fma2(pack2(__uint_as_float(x[j]), __uint_as_float(x[j + 1])), cc, oo), a, b);
    x[j] = __float_as_uint(ex2(a));
    x[j + 1] = __float_as_uint(ex2(b));
  }
}
// d[j] = p[j] (d[j] - delta)
template <int N>
__device__ __forceinline__ void score_gradients(uint32_t *d, const uint32_t *p, float delta) {
  const uint64_t minus = pack2(-delta, -delta);
#pragma unroll
  for (int j = 0; j < N; j += 2) {
    float a, b;
    unpack2(mul2(pack2(__uint_as_float(p[j]), __uint_as_float(p[j + 1])), add2(pack2(__uint_as_float(d[j]), __uint_as_float(d[j + 1])), minus)), a, b);
    d[j] = __float_as_uint(a);
    d[j + 1] = __float_as_uint(b);
  }
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// 16 fp32 values times f as bf16 to 32 bytes of global memory: one full sector per thread where the address allows it
__device__ __forceinline__ void store16(__nv_bfloat16 *dst, const uint32_t *r, float f) {
  float v[16];
#pragma unroll
  for (int j = 0; j < 16; j++) v[j] = __uint_as_float(r[j]) * f;
  const uint4 lo = pack8(v), hi = pack8(v + 8);
  if ((reinterpret_cast<uintptr_t>(dst) & 31) == 0) {
    st_global_256(dst, lo, hi);
  } else {
    reinterpret_cast<uint4 *>(dst)[0] = lo;
    reinterpret_cast<uint4 *>(dst)[1] = hi;
  }
}
// N fp32 columns of this lane from tensor memory
template <int N>
__device__ __forceinline__ void load_columns(uint32_t addr, uint32_t *r) {
  if (N == 16) {
    ptx::tmem_ld16(addr, r);
  } else {
#pragma unroll
    for (int q = 0; q < N / 32; q++) ptx::tmem_ld32(addr + q * 32, r + q * 32);
  }
  ptx::tmem_ld_wait();
}
// 8 N bf16 values of a row into a 128-byte-swizzled slab, from 16-byte chunk `chunk` of the row on
template <int N>
__device__ __forceinline__ void store_packed(uint32_t row_addr, int row, int chunk, const uint32_t *v) {
#pragma unroll
  for (int q = 0; q < N; q++) sts128(row_addr + (uint32_t)(((chunk + q) ^ (row & 7)) * 16), make_uint4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]));
}
// the same from fp32
template <int N>
__device__ __forceinline__ void store_chunks(uint32_t row_addr, int row, int chunk, const uint32_t *x) {
  uint32_t v[4 * N];
#pragma unroll
  for (int j = 0; j < 4 * N; j++) v[j] = pack_bf16(__uint_as_float(x[2 * j]), __uint_as_float(x[2 * j + 1]));
  store_packed<N>(row_addr, row, chunk, v);
}

// keys of a sequence that none of its queries sees: [sinks, dead_end), and those from Tk on
__device__ __forceinline__ int dead_end(const Span &sp, int window) { return max(0, sp.shift - window + 1); }
__device__ __forceinline__ bool has_dead(const Span &sp, int kb, int window, int sinks) {
  return kb * TILE + TILE > sp.Tk || (kb * TILE < dead_end(sp, window) && kb * TILE + TILE > sinks);
}
// a warp zeroes the rows of such keys in a tile that has landed in shared memory (a row is 128 bytes of each slab)
template <int HD>
__device__ __forceinline__ void zero_dead(uint32_t tile, const Span &sp, int kb, int window, int sinks, int lane) {
  const int end = dead_end(sp, window);
  for (int r = lane; r < TILE; r += 32) {
    const int key = kb * TILE + r;
    if (key < sp.Tk && (key < sinks || key >= end)) continue;
#pragma unroll
    for (int s = 0; s < HD / 64; s++)
#pragma unroll
      for (int c = 0; c < 8; c++) sts128(tile + s * SLAB + r * 128 + c * 16, make_uint4(0, 0, 0, 0));
  }
}

// A thread's row of a shared unit (its tile, its output in tensor memory unless it saw no key here, its maximum and sum) to shared memory, all
// CTAs' rows joined in the order of their ranks. The 16-byte pieces of a row are swizzled with the row.
template <int HD>
__device__ __forceinline__ uint32_t part_at(uint32_t base, int row, int piece) {
  return base + (uint32_t)(row * HD * 4 + ((piece ^ row) & (HD / 4 - 1)) * 16);
}
template <int HD>
__device__ __forceinline__ void store_part(uint32_t base, int row, uint32_t o_addr, bool any, float m, float l) {
#pragma unroll
  for (int q = 0; q < HD / 32; q++) {
    uint32_t v[32];
    load_columns<32>(o_addr + q * 32, v);  // whole warps
#pragma unroll
    for (int j = 0; j < 8; j++)
      sts128(part_at<HD>(base, row, q * 8 + j), any ? make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]) : make_uint4(0, 0, 0, 0));
  }
  fa::sts32(base + (uint32_t)(2 * TILE * HD * 4 + row * 8), m);
  fa::sts32(base + (uint32_t)(2 * TILE * HD * 4 + row * 8 + 4), l);
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}
template <typename T>
__device__ __forceinline__ T of_cluster(uint32_t addr, uint32_t rank);
template <>
__device__ __forceinline__ float4 of_cluster<float4>(uint32_t addr, uint32_t rank) {
  float4 v;
  asm volatile("{\n.reg .b32 ra;\nmapa.shared::cluster.u32 ra, %4, %5;\nld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [ra];\n}\n"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr), "r"(rank)
               : "memory");
  return v;
}
template <>
__device__ __forceinline__ float2 of_cluster<float2>(uint32_t addr, uint32_t rank) {
  float2 v;
  asm volatile("{\n.reg .b32 ra;\nmapa.shared::cluster.u32 ra, %2, %3;\nld.shared::cluster.v2.f32 {%0, %1}, [ra];\n}\n"
               : "=f"(v.x), "=f"(v.y)
               : "r"(addr), "r"(rank)
               : "memory");
  return v;
}
// `thread` of 256; this CTA's share of the unit's rows. First every row's weights of the CTAs' parts, then its pieces, all CTAs' loads under way at
// once (one after the other they took 12 us).
template <int HD>
__device__ __forceinline__ void join_parts(const FwdParams &p, uint32_t base, int thread) {
  constexpr int PIECES = HD / 4, AT_ONCE = 256 / PIECES;
  const float c = p.scale * LOG2E;
  const Unit u = unit_of(p, (int)blockIdx.x / p.cluster);
  const int rows = 2 * TILE / p.cluster, row0 = rows * ((int)blockIdx.x % p.cluster), piece = thread % PIECES;
  const uint32_t stats = base + (uint32_t)(2 * TILE * HD * 4), weights = stats + 2 * TILE * 8;
  if (thread < rows) {
    const int at = row0 + thread, row = at & (TILE - 1);
    const Tile &x = at < TILE ? u.a : u.b;
    float2 ml[MAX_SHARERS];
#pragma unroll
    for (int k = 0; k < MAX_SHARERS; k++) ml[k] = k < p.cluster ? of_cluster<float2>(stats + at * 8, k) : make_float2(-INFINITY, 0.0f);
    float M = -INFINITY, L = 0.0f, f[MAX_SHARERS];
#pragma unroll
    for (int k = 0; k < MAX_SHARERS; k++) M = fmaxf(M, ml[k].x);
#pragma unroll
    for (int k = 0; k < MAX_SHARERS; k++) {
      f[k] = ml[k].x == -INFINITY ? 0.0f : ex2((ml[k].x - M) * c);
      L = fmaf(f[k], ml[k].y, L);
    }
    const float inv = 1.0f / L;
#pragma unroll
    for (int k = 0; k < MAX_SHARERS; k++) fa::sts32(weights + (thread * MAX_SHARERS + k) * 4, f[k] * inv);
    if (x.exists && x.row + row < u.sp.Tq) p.lse[(int64_t)x.h * p.total_q + u.sp.q_off + x.row + row] = M * p.scale + logf(L);
  }
  asm volatile("bar.sync 1, 256;" ::: "memory");
#pragma unroll 2
  for (int q = thread / PIECES; q < rows; q += AT_ONCE) {
    const int at = row0 + q, row = at & (TILE - 1);
    const Tile &x = at < TILE ? u.a : u.b;
    if (!x.exists || x.row + row >= u.sp.Tq) continue;
    float4 v[MAX_SHARERS];
#pragma unroll
    for (int k = 0; k < MAX_SHARERS; k++)
      if (k < p.cluster) v[k] = of_cluster<float4>(part_at<HD>(base, at, piece), k);
    const float4 w[2] = {fa::lds128(weights + q * MAX_SHARERS * 4), fa::lds128(weights + q * MAX_SHARERS * 4 + 16)};
    const float f[MAX_SHARERS] = {w[0].x, w[0].y, w[0].z, w[0].w, w[1].x, w[1].y, w[1].z, w[1].w};
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int k = 0; k < MAX_SHARERS; k++)
      if (k < p.cluster) {
        sum.x = fmaf(f[k], v[k].x, sum.x);
        sum.y = fmaf(f[k], v[k].y, sum.y);
        sum.z = fmaf(f[k], v[k].z, sum.z);
        sum.w = fmaf(f[k], v[k].w, sum.w);
      }
    *reinterpret_cast<uint2 *>(p.O + ((int64_t)(u.sp.q_off + x.row + row) * p.q_heads + x.h) * HD + piece * 4) =
        make_uint2(pack_bf16(sum.x, sum.y), pack_bf16(sum.z, sum.w));
  }
}

template <int HD, int WALK>
__global__ void __launch_bounds__(FWD_THREADS, 1) window_fwd_kernel(const __grid_constant__ FwdParams p) {
  using Sh = FwdShape<HD>;
  constexpr int SLOTS = Sh::SLOTS, RING = Sh::RING;
  // S_0, S_1 (128 columns each), O_0, O_1 (HD each), at head size 64 P_0, P_1 (64 each)
  constexpr uint32_t TMEM_COLS = 512, COL_O = 256, COL_P = 384;
  extern __shared__ unsigned char window_smem[];
  unsigned char *smem = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(window_smem) + 1023) & ~static_cast<uintptr_t>(1023));
  unsigned char *sQ = smem, *sP = sQ + 2 * Sh::Q_TILE, *sKV = sP + 2 * Sh::P_TILE;
  auto *st = reinterpret_cast<typename Sh::Tail *>(sKV + SLOTS * Sh::KV_TILE);
  volatile int *abort_flag = &st->abort_flag;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  auto bar = [&](uint64_t *b) { return ptx::smem_u32(b); };
  auto wait = [&](uint64_t *b, uint32_t par, int code) { return ptx::mbar_wait<false>(bar(b), par & 1u, abort_flag, p.status, code); };
  // every thread arrives for itself (one arrival per warp measured the same)
  auto arrive = [&](uint64_t *b) { ptx::mbar_arrive(bar(b)); };

  if (tid == 0) {
    for (int g = 0; g < 2; g++) {
      ptx::mbar_init(bar(&st->q_full[g]), 1);
      ptx::mbar_init(bar(&st->q_empty[g]), 1);
      ptx::mbar_init(bar(&st->s_full[g]), 1);
      ptx::mbar_init(bar(&st->s_read[g]), TILE);
      ptx::mbar_init(bar(&st->p_ready[g]), TILE);
      ptx::mbar_init(bar(&st->pv_done[g]), 1);
      ptx::mbar_init(bar(&st->o_empty[g]), TILE);
    }
    for (int s = 0; s < RING; s++) {
      ptx::mbar_init(bar(&st->k_full[s]), 1);
      ptx::mbar_init(bar(&st->v_full[s]), 1);
    }
    for (int s = 0; s < SLOTS; s++) ptx::mbar_init(bar(&st->kv_empty[s]), 2);  // V: either tile's issuer; K: twice the one
    ptx::mbar_init(bar(&st->begun), TILE);
    ptx::mbar_init(bar(&st->fixed), 1);
    st->abort_flag = 0;
    ptx::fence_barrier_init();
    ptx::fence_proxy_async_smem();
  }
  if (warp == 1) {
    ptx::tmem_alloc(ptx::smem_u32(&st->tmem_base), TMEM_COLS);
    ptx::tmem_relinquish();
  }
  if (warp == 0 && lane == 0) {
    ptx::tma_prefetch_desc(&p.tmQ);
    ptx::tma_prefetch_desc(&p.tmK);
    ptx::tma_prefetch_desc(&p.tmV);
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem_base = st->tmem_base;
  pdl_release();
  pdl_wait();
  float part_m = -INFINITY, part_l = 0.0f;  // of a shared unit

  // The ring: step t of the CTA (counted through its units) uses K at place max(0, 2 t - 1) and V at place 2 t + 2: a unit's first K
  // goes before the last unit's last V. A slot holds K and V by turns, but
  // whoever waits on a barrier must wait for every phase of it (a phase ahead, the parity is that of the last but one): K_t and V_t are announced
  // on barriers of their own, t % 4. These are free again in time: the last load that needs no slot emptied is K_3 (six slots), and later
  // ones follow an S or P V product of step t - 3, so whoever waits has seen step t - 4.
  auto k_at = [](uint32_t t) { return t == 0 ? 0u : 2 * t - 1; };
  auto v_at = [](uint32_t t) { return 2 * t + 2; };

  if (warp < 4) {
    ptx::reg_dec<REGS_CONTROL>();
    if (warp == 0) {
      // ================= loads: the whole warp walks, one lane issues =================
      uint32_t t = 0, uq[2] = {0, 0}, fixes = 0;
      bool ok = true;
      auto waitw = [&](uint64_t *b, uint32_t par, int code) { return __all_sync(0xffffffffu, wait(b, par, code)) != 0; };
      auto load = [&](const CUtensorMap *m, uint32_t n, uint64_t *landed, const Span &sp, int kvh, int kb, bool fix) {
        const uint32_t slot = n % SLOTS;
        ok = waitw(&st->kv_empty[slot], n / SLOTS + 1, ST_KV_EMPTY);
        if (!ok) return;
        const uint32_t tile = ptx::smem_u32(sKV + slot * Sh::KV_TILE), full = fix ? bar(&st->fixed) : bar(landed);
        if (lane == 0) {
          ptx::mbar_arrive_expect_tx(full, (uint32_t)Sh::KV_TILE);
          ptx::tma_load_3d(tile, m, full, 0, sp.k_off + kb * TILE, kvh * (HD / 64));
        }
        if (!fix) return;
        ok = waitw(&st->fixed, fixes++, ST_FIX);
        if (!ok) return;
        zero_dead<HD>(tile, sp, kb, p.window, p.sinks, lane);
        ptx::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(bar(landed));
      };
      // the V of the step before
      Span last_sp;
      int last_kvh = 0, last_kb = 0;
      auto load_last_v = [&]() {
        load(&p.tmV, v_at(t - 1), &st->v_full[(t - 1) % RING], last_sp, last_kvh, last_kb, has_dead(last_sp, last_kb, p.window, p.sinks));
      };
      Walk<WALK> walk;
      for (int unit = walk.next(p); ok && unit < p.units; unit = walk.next(p)) {
        const Unit u = unit_of(p, unit);
        const int kvh = u.a.h / p.group;
        const int begin = u.begin<WALK>(p.cluster), end = u.end<WALK>(p.cluster);
        for (int i = begin; ok && i < end; i++) {
          if (i == begin) {  // the last unit's S products still read its Q
#pragma unroll
            for (int g = 0; g < 2; g++) {
              const Tile &x = g ? u.b : u.a;
              if (!ok || !x.exists) continue;
              ok = waitw(&st->q_empty[g], uq[g] + 1, ST_Q_EMPTY);
              if (ok && lane == 0) {
                ptx::mbar_arrive_expect_tx(bar(&st->q_full[g]), (uint32_t)Sh::Q_TILE);
                ptx::tma_load_3d(ptx::smem_u32(sQ + g * Sh::Q_TILE), &p.tmQ, bar(&st->q_full[g]), 0, u.sp.q_off + x.row, x.h * (HD / 64));
              }
              uq[g]++;
            }
          }
          if (ok) load(&p.tmK, k_at(t), &st->k_full[t % RING], u.sp, kvh, u.block(i), false);
          if (ok && t > 0) load_last_v();
          last_sp = u.sp;
          last_kvh = kvh;
          last_kb = u.block(i);
          t++;
        }
      }
      if (ok && t > 0) load_last_v();
      __syncwarp();
    } else if (warp == 1) {
      // ================= S products =================
      if (lane == 0) {
        const uint32_t idesc = ptx::make_idesc_bf16(TILE, TILE, 0, 0);
        const uint32_t q_base = ptx::smem_u32(sQ), kv_base = ptx::smem_u32(sKV);
        uint32_t t = 0, uq[2] = {0, 0}, ts[2] = {0, 0};  // steps; units and S products of either tile
        bool ok = true;
        Walk<WALK> walk;
        for (int unit = walk.next(p); ok && unit < p.units; unit = walk.next(p)) {
          const Unit u = unit_of(p, unit);
          const int begin = u.begin<WALK>(p.cluster), end = u.end<WALK>(p.cluster);
          if (begin == end) continue;
          if (u.a.exists) ok = wait(&st->q_full[0], uq[0]++, ST_Q_FULL);
          if (ok && u.b.exists) ok = wait(&st->q_full[1], uq[1]++, ST_Q_FULL);
          for (int i = begin; ok && i < end; i++, t++) {
            const int kb = u.block(i);
            const uint32_t slot = k_at(t) % SLOTS;
            if (!(ok = wait(&st->k_full[t % RING], t / RING, ST_KV_FULL))) break;
#pragma unroll
            for (int g = 0; g < 2; g++) {
              const Tile &x = g ? u.b : u.a;
              if (!ok || !x.active(kb, p.sinks)) continue;
              if (ts[g] > 0 && !(ok = wait(&st->s_read[g], ts[g] - 1, ST_S_FREE))) continue;
              ptx::tc_fence_after();
              const uint64_t qd = tile_desc(q_base + g * Sh::Q_TILE, 0), kd = tile_desc(kv_base + slot * Sh::KV_TILE, 0);
#pragma unroll
              for (int k16 = 0; k16 < HD / 16; k16++) {
                const uint32_t off = (uint32_t)((k16 >> 2) * SLAB + (k16 & 3) * 32);
                ptx::umma_bf16(tmem_base + (uint32_t)(g * TILE), desc_at(qd, off), desc_at(kd, off), idesc, k16 > 0);
              }
              ptx::umma_commit(bar(&st->s_full[g]));
              if (kb == x.hi) ptx::umma_commit(bar(&st->q_empty[g]));
              ts[g]++;
            }
            if (!ok) break;
            ptx::umma_commit(bar(&st->kv_empty[slot]));
            ptx::mbar_arrive(bar(&st->kv_empty[slot]));
          }
        }
      }
      __syncwarp();
    } else {
      // ================= P V products of one tile =================
      if (lane == 0) {
        const int g = warp - 2;
        const uint32_t idesc = ptx::make_idesc_bf16(TILE, HD, 0, 1);  // V is read with its head dimension contiguous
        const uint32_t p_base = ptx::smem_u32(sP + g * Sh::P_TILE), kv_base = ptx::smem_u32(sKV), o_col = tmem_base + COL_O + (uint32_t)(g * HD);
        uint32_t t = 0, units = 0, tp = 0;  // steps; units and products of this tile
        bool ok = true;
        Walk<WALK> walk;
        for (int unit = walk.next(p); ok && unit < p.units; unit = walk.next(p)) {
          const Unit u = unit_of(p, unit);
          const Tile x = g ? u.b : u.a;
          bool begun = false;
          const int end = u.end<WALK>(p.cluster);
          for (int i = u.begin<WALK>(p.cluster); ok && i < end; i++, t++) {
            const uint32_t slot = v_at(t) % SLOTS;
            if (!(ok = wait(&st->v_full[t % RING], t / RING, ST_KV_FULL))) break;
            if (!x.active(u.block(i), p.sinks)) {
              ptx::mbar_arrive(bar(&st->kv_empty[slot]));
              continue;
            }
            // P of this step is in its place, the group has rescaled O if its maxima grew - and read the last unit's O
            if (!(ok = wait(&st->p_ready[g], tp, ST_P))) break;
            if (!begun && units > 0 && !(ok = wait(&st->o_empty[g], units - 1, ST_O_FREE))) break;
            ptx::tc_fence_after();
            const uint64_t pd = tile_desc(p_base, 0), vd = tile_desc(kv_base + slot * Sh::KV_TILE, SLAB);
#pragma unroll
            for (int k16 = 0; k16 < TILE / 16; k16++) {
              const uint64_t v16 = desc_at(vd, (uint32_t)(k16 * 2048));
              if constexpr (Sh::P_IN_TMEM)
                ptx::umma_bf16_ts(o_col, tmem_base + COL_P + (uint32_t)(g * 64 + k16 * 8), v16, idesc, begun || k16 > 0);
              else
                ptx::umma_bf16(o_col, desc_at(pd, (uint32_t)((k16 >> 2) * SLAB + (k16 & 3) * 32)), v16, idesc, begun || k16 > 0);
            }
            begun = true;
            ptx::umma_commit(bar(&st->pv_done[g]));
            ptx::umma_commit(bar(&st->kv_empty[slot]));
            tp++;
          }
          units += x.exists;
        }
      }
      __syncwarp();
    }
  } else {
    ptx::reg_inc<REGS_SOFTMAX>();
    // ================= softmax and output (a thread per query row) =================
    const int g = (warp - 4) >> 2, quarter = warp & 3;  // tensor-memory lanes a warp may read: 32 * (warp % 4) ...
    const int trow = quarter * 32 + lane;
    const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16);
    const uint32_t s_addr = lane_addr + (uint32_t)(g * TILE), o_addr = lane_addr + COL_O + (uint32_t)(g * HD);
    const uint32_t p_addr = ptx::smem_u32(sP + g * Sh::P_TILE + trow * 128);
    const float c = p.scale * LOG2E;
    uint32_t t = 0;  // steps of this tile so far
    if (g == 1) {
      const Unit u = unit_of(p, Walk<WALK>().next(p));
      // (of a shared unit's neighbouring tiles the first may see none of this CTA's blocks)
      const bool both = WALK != WALK_SHARED || (p.pair_heads && u.begin<WALK>(p.cluster) < u.end<WALK>(p.cluster));
      if (u.b.exists && both && !wait(&st->begun, 0, ST_P)) goto teardown;
    }
    Walk<WALK> walk;
    for (int unit = walk.next(p); unit < p.units; unit = walk.next(p)) {
      const Unit u = unit_of(p, unit);
      const Tile x = g ? u.b : u.a;
      if (!x.exists) continue;
      const int row = x.row + trow, pos = row + u.sp.shift;
      const int tile_pos = x.row + u.sp.shift, last_pos = min(tile_pos + TILE, u.sp.Tk) - 1;
      float m = -INFINITY, l = 0.0f;
      bool first = true;
      const int end = u.end<WALK>(p.cluster);
      for (int i = u.begin<WALK>(p.cluster); i < end; i++) {
        const int kb = u.block(i);
        if (!x.active(kb, p.sinks)) continue;
        if (!wait(&st->s_full[g], t, ST_S)) goto teardown;
        ptx::tc_fence_after();
        uint32_t s[TILE];
        load_columns<TILE>(s_addr, s);
        ptx::tc_fence_before();
        arrive(&st->s_read[g]);
        if (!all_seen(kb * TILE, tile_pos, last_pos, p.window, p.sinks)) {
          const int base = kb * TILE, hi = min(pos, u.sp.Tk - 1) - base, lo = pos - p.window + 1 - base, sk = p.sinks - base;
#pragma unroll
          for (int q = 0; q < 4; q++) {
            const uint32_t see = seen_bits(hi - 32 * q, lo - 32 * q, sk - 32 * q);
#pragma unroll
            for (int j = 0; j < 32; j++) s[q * 32 + j] = (see >> j) & 1u ? s[q * 32 + j] : 0xff800000u;  // -infinity
          }
        }
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int j = 0; j < TILE; j += 2) mx4[(j >> 1) & 3] = max3(mx4[(j >> 1) & 3], __uint_as_float(s[j]), __uint_as_float(s[j + 1]));
        const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
        float alpha = 1.0f;
        if (first) {
          m = mx;
        } else if ((mx - m) * c > 8.0f) {
          // a row that had seen nothing has nothing to rescale
          if (m != -INFINITY) alpha = ex2((m - mx) * c);
          m = mx;
          l *= alpha;
        }
        // a row that has seen no key yet keeps m = -inf: its probabilities are exp2(-inf) = 0 against a zero offset
        const float mc = (m == -INFINITY) ? 0.0f : m * c;
        const uint64_t cc = pack2(c, c), off = pack2(-mc, -mc);
        uint64_t sum2[2] = {0, 0};
        uint32_t pk[TILE / 2];
#pragma unroll
        for (int j = 0; j < TILE; j += 2) {
          float x0, x1;
          unpack2(fma2(pack2(__uint_as_float(s[j]), __uint_as_float(s[j + 1])), cc, off), x0, x1);
          const float e0 = ex2(x0), e1 = ex2(x1);
          sum2[(j >> 1) & 1] = add2(sum2[(j >> 1) & 1], pack2(e0, e1));
          pk[j >> 1] = pack_bf16(e0, e1);
        }
        float sa, sb;
        unpack2(add2(sum2[0], sum2[1]), sa, sb);
        l += sa + sb;
        // the step before has read P, and O is at rest
        if (t > 0 && !wait(&st->pv_done[g], t - 1, ST_PV)) goto teardown;
        if (__any_sync(0xffffffffu, alpha != 1.0f)) {  // tensor-memory accesses are warp-wide: every lane takes part
          ptx::tc_fence_after();
#pragma unroll
          for (int q = 0; q < HD / 32; q++) {
            uint32_t r[32];
            load_columns<32>(o_addr + q * 32, r);
#pragma unroll
            for (int j = 0; j < 32; j++) r[j] = __float_as_uint(__uint_as_float(r[j]) * alpha);
            ptx::tmem_st32(o_addr + q * 32, r);
          }
          ptx::tmem_st_wait();
        }
        if constexpr (Sh::P_IN_TMEM) {
          ptx::tc_fence_after();
          ptx::tmem_st32(lane_addr + COL_P + (uint32_t)(g * 64), pk);
          ptx::tmem_st32(lane_addr + COL_P + (uint32_t)(g * 64 + 32), pk + 32);
          ptx::tmem_st_wait();
        } else {
          store_packed<8>(p_addr, trow, 0, pk);
          store_packed<8>(p_addr + SLAB, trow, 0, pk + 32);
          ptx::fence_proxy_async_smem();
        }
        ptx::tc_fence_before();
        arrive(&st->p_ready[g]);
        if (g == 0 && t == 0) arrive(&st->begun);
        first = false;
        t++;
      }
      if (WALK == WALK_SHARED && t == 0) continue;
      if (!wait(&st->pv_done[g], t - 1, ST_PV)) goto teardown;
      if (WALK == WALK_SHARED) {
        part_m = m;
        part_l = l;
        continue;
      }
      ptx::tc_fence_after();
      uint32_t r[HD];
      load_columns<HD>(o_addr, r);
      ptx::tc_fence_before();
      arrive(&st->o_empty[g]);
      if (row < u.sp.Tq) {
        const float inv = 1.0f / l;
        __nv_bfloat16 *o = p.O + ((int64_t)(u.sp.q_off + row) * p.q_heads + x.h) * HD;
#pragma unroll
        for (int q = 0; q < HD / 16; q++) store16(o + q * 16, r + q * 16, inv);
        p.lse[(int64_t)x.h * p.total_q + u.sp.q_off + row] = m * p.scale + logf(l);
      }
    }
  }

teardown:
  if (*abort_flag) {
    // give copies that are still in flight time to land before shared memory is released
    const uint64_t t0 = ptx::globaltimer_ns();
    while (ptx::globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
  }
  ptx::tc_fence_before();
  __syncthreads();
  if constexpr (WALK == WALK_SHARED) {
    // Every product has been waited for and every tile that was loaded has been used: shared memory is free. (After a wait that ran out: rubbish,
    // but every thread comes by here.)
    const int thread = tid - 128;
    ptx::tc_fence_after();
    if (warp >= 4) {
      const uint32_t o_addr = tmem_base + ((uint32_t)((warp & 3) * 32) << 16) + COL_O + (uint32_t)((thread >> 7) * HD);
      store_part<HD>(ptx::smem_u32(smem), thread, o_addr, part_m != -INFINITY, part_m, part_l);
    }
    ptx::tc_fence_before();
    cluster_sync();
    if (warp >= 4) join_parts<HD>(p, ptx::smem_u32(smem), thread);
    cluster_sync();  // nobody leaves while another reads its shared memory
  }
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

// ---------------------------------------------------------------------------------------------------------------------------
// Backward, two kernels, each with its sums in a fixed order in tensor memory (no atomics: two runs give the same bits). Both put
// query rows on the tensor-memory lanes, so that a thread's log-sum-exp and delta are its own two numbers.
//
// dQ: one query tile of one head per unit, persistent CTAs. Per key block
//     S = Q K^T,  dP = dO V^T,   dS = P o (dP - delta) as bf16 through tensor memory,   dQ += dS K
// S and dP of a block are issued while the threads still work on the block before, and a unit's first products before the last
// unit's dQ is finished. delta = rowsum(dO o O) is formed here, in fp32, and written for the other kernel. Four warps of their own
// form it for the next unit and write the last one's dQ: with these in the computing threads' way a unit of ten blocks spent 10 of its 43
// thousand cycles between the blocks. dS lies in tensor memory, where the product takes its rows from, in two places by turns: through shared
// memory, which bounds this kernel, 8 % more time, though tensor memory then held an accumulator for the next unit. K is needed from S to dQ, V
// for dP only: three slots of shared memory for K, two for V.
//
// dK, dV: one block of 128 keys of one key/value head per unit; it walks the query heads of the group and the query tiles that see
// its keys, K and V stay in shared memory. Per tile
//     S = Q K^T,  dP = dO V^T,   dV += P^T dO,   dK += dS^T Q      (P and dS are read by the tensor cores with the rows as reduction)
// Blocks that hold sinks are seen by every later query: tiles behind the block's window are cut into further units that sum their
// share of the sink rows into the workspace, and a last kernel adds the shares in order. In batches too small to fill the GPU the heads of a
// group are split over units the same way (45 - 391 keys, 8 heads on one: 30 -> 13 us).
//
// Rounding: P and dS to bf16 once each (dS from the fp32 P), accumulators fp32, one rounding per output.
// delta is formed from O as the caller holds it: rounded to bf16, off by up to 2^-8 of |O|, after a sum over probabilities that were rounded too. Against
// a delta of the exact output a dS is off by up to P times 2^-8 of |dO| |O| (and of |dO| sum P |V|), which shows where a query has few keys. The
// interface does not carry the fp32 output. tests/test_gpu_attention_window_gradients.py holds dQ and dK to the exact gradient within these bounds.
// What bounds both: shared memory. A step of dK, dV moves 384 KB through it (four products of 64, P and dS, Q and dO that arrive; 3070 cycles at
// 128 bytes each) and takes 3400; one of dQ 224 KB (1800 cycles; its third product reads K only) and takes about 2500.
// Measured with 16 query heads on 4 of 128 and 8192 tokens: window 1024, 4 sinks dQ 120 us, dK and dV 175 us, join 4 us; no window 825 us
// together (830 TFLOP/s; the causal kernel without windows 1110 us).
// ---------------------------------------------------------------------------------------------------------------------------
constexpr int DS_TILE = TILE * TILE * 2;

enum { ST_BQ_Q = 61, ST_BQ_KV_EMPTY, ST_BQ_Q_FULL, ST_BQ_KV_FULL, ST_BQ_S_FREE, ST_BQ_DP_FREE, ST_BQ_DS, ST_BQ_ACC, ST_BQ_STAT, ST_BQ_S, ST_BQ_DP,
       ST_BQ_DQ, ST_BK_KV = 81, ST_BK_Q_EMPTY, ST_BK_DO_EMPTY, ST_BK_Q, ST_BK_DO, ST_BK_S_FREE, ST_BK_DP_FREE, ST_BK_P, ST_BK_DS, ST_BK_S,
       ST_BK_DP, ST_BK_DV, ST_BK_DK, ST_BK_FIX };

struct BwdParams {
  CUtensorMap tmQ, tmK, tmV, tmdO;
  SeqTable seqs;
  const __nv_bfloat16 *o, *dout;
  const float *lse;
  float *delta;  // [q_heads][total_q]
  __nv_bfloat16 *dq, *dk, *dv;
  int window, sinks, group, q_heads, kv_heads, total_q, units;
  // dK, dV: units from main_units on are shares of the sink rows; slot[s]: the first slot of sequence s in the workspace. Or, with
  // parts > 1: every block's heads are split over so many units, whose shares cover all rows
  int main_units, slot_rows, parts;
  int far[MAX_SEQS + 1], slot[MAX_SEQS];
  float *shares;  // [slots][kv_heads][slot_rows][2][head_dim]
  float scale;
  int *status;
};

template <int HD>
struct BwdQShape {
  static constexpr int Q_TILE = TILE * HD * 2, KV_TILE = TILE * HD * 2;
  static constexpr int KS = HD == 128 ? 3 : 5, VS = HD == 128 ? 2 : 3;
  static constexpr int ACCS = 128 / HD;  // accumulators
  struct Tail {
    uint64_t q_full, q_empty, k_full[KS], k_empty[KS], v_full[VS], v_empty[VS], s_full, s_read, dp_full, dp_read, ds_ready[2], dq_done[2], acc_full[ACCS],
        acc_empty[ACCS], stat_full[2], stat_empty[2], fixed;
    uint32_t tmem_base;
    int abort_flag;
    float delta[2][TILE];  // of even and odd units
  };
  static constexpr size_t smem = 1024 + 2 * (size_t)Q_TILE + (KS + VS) * (size_t)KV_TILE + sizeof(Tail);
  static_assert(smem <= 232448, "more shared memory than a CTA can be given");
};

// one tile of one head and its key blocks
struct QUnit {
  Span sp;
  Tile x;
  int n, n_sink;
  __device__ __forceinline__ int block(int i) const { return i < n_sink ? i : x.lo + i - n_sink; }
};
__device__ __forceinline__ QUnit q_unit_of(const BwdParams &p, int unit) {
  QUnit u;
  int s = 0;
  while (unit >= p.seqs.first[s + 1]) s++;
  u.sp = span_of(p.seqs, s);
  const int rel = unit - p.seqs.first[s], tiles = (u.sp.Tq + TILE - 1) / TILE;
  u.x = tile_of(u.sp, p.window, rel % p.q_heads, (tiles - 1 - rel / p.q_heads) * TILE);
  u.n_sink = min((p.sinks + TILE - 1) / TILE, u.x.lo);
  u.n = u.n_sink + u.x.hi - u.x.lo + 1;
  return u;
}

template <int HD>
__global__ void __launch_bounds__(BWD_Q_THREADS, 1) window_bwd_q_kernel(const __grid_constant__ BwdParams p) {
  using Sh = BwdQShape<HD>;
  constexpr int KS = Sh::KS, VS = Sh::VS, ACCS = Sh::ACCS;
  // dQ: an accumulator of 128 columns or two of 64; dS of even and odd steps as bf16, 64 columns each
  constexpr uint32_t TMEM_COLS = 512, COL_S = 0, COL_DP = 128, COL_DQ = 256, COL_DS = 384;
  extern __shared__ unsigned char window_smem[];
  unsigned char *smem = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(window_smem) + 1023) & ~static_cast<uintptr_t>(1023));
  unsigned char *sQ = smem, *sDO = sQ + Sh::Q_TILE, *sK = sDO + Sh::Q_TILE, *sV = sK + KS * Sh::KV_TILE;
  auto *st = reinterpret_cast<typename Sh::Tail *>(sV + VS * Sh::KV_TILE);
  volatile int *abort_flag = &st->abort_flag;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  auto bar = [&](uint64_t *b) { return ptx::smem_u32(b); };
  auto wait = [&](uint64_t *b, uint32_t par, int code) { return ptx::mbar_wait<false>(bar(b), par & 1u, abort_flag, p.status, code); };
  // every thread arrives for itself (one arrival per warp measured the same)
  auto arrive = [&](uint64_t *b) { ptx::mbar_arrive(bar(b)); };

  if (tid == 0) {
    ptx::mbar_init(bar(&st->q_full), 1);
    ptx::mbar_init(bar(&st->q_empty), 2);  // the last S and the last dP of a unit
    for (int s = 0; s < KS; s++) {
      ptx::mbar_init(bar(&st->k_full[s]), 1);
      ptx::mbar_init(bar(&st->k_empty[s]), 1);
    }
    for (int s = 0; s < VS; s++) {
      ptx::mbar_init(bar(&st->v_full[s]), 1);
      ptx::mbar_init(bar(&st->v_empty[s]), 1);
    }
    ptx::mbar_init(bar(&st->s_full), 1);
    ptx::mbar_init(bar(&st->s_read), 512);
    ptx::mbar_init(bar(&st->dp_full), 1);
    ptx::mbar_init(bar(&st->dp_read), 512);
    for (int s = 0; s < ACCS; s++) {
      ptx::mbar_init(bar(&st->acc_full[s]), 1);
      ptx::mbar_init(bar(&st->acc_empty[s]), TILE);
    }
    for (int s = 0; s < 2; s++) {
      ptx::mbar_init(bar(&st->ds_ready[s]), 512);
      ptx::mbar_init(bar(&st->dq_done[s]), 1);
      ptx::mbar_init(bar(&st->stat_full[s]), TILE);
      ptx::mbar_init(bar(&st->stat_empty[s]), 512);
    }
    ptx::mbar_init(bar(&st->fixed), 1);
    st->abort_flag = 0;
    ptx::fence_barrier_init();
    ptx::fence_proxy_async_smem();
  }
  if (warp == 1) {
    ptx::tmem_alloc(ptx::smem_u32(&st->tmem_base), TMEM_COLS);
    ptx::tmem_relinquish();
  }
  if (warp == 0 && lane == 0) {
    ptx::tma_prefetch_desc(&p.tmQ);
    ptx::tma_prefetch_desc(&p.tmK);
    ptx::tma_prefetch_desc(&p.tmV);
    ptx::tma_prefetch_desc(&p.tmdO);
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem_base = st->tmem_base;
  pdl_release();
  pdl_wait();

  if (warp < 4) {
    ptx::reg_dec<REGS_BWD_Q_OTHER>();
    if (warp == 0) {
      // ================= loads: the whole warp walks, one lane issues =================
      uint32_t t = 0, units = 0, fixes = 0;
      bool ok = true;
      auto waitw = [&](uint64_t *b, uint32_t par, int code) { return __all_sync(0xffffffffu, wait(b, par, code)) != 0; };
      for (int round = 0, unit = unit_at(0); ok && unit < p.units; unit = unit_at(++round)) {
        const QUnit u = q_unit_of(p, unit);
        const int kvh = u.x.h / p.group;
        ok = waitw(&st->q_empty, units + 1, ST_BQ_Q);
        units++;
        if (ok && lane == 0) {
          ptx::mbar_arrive_expect_tx(bar(&st->q_full), (uint32_t)(2 * Sh::Q_TILE));
          ptx::tma_load_3d(ptx::smem_u32(sQ), &p.tmQ, bar(&st->q_full), 0, u.sp.q_off + u.x.row, u.x.h * (HD / 64));
          ptx::tma_load_3d(ptx::smem_u32(sDO), &p.tmdO, bar(&st->q_full), 0, u.sp.q_off + u.x.row, u.x.h * (HD / 64));
        }
        for (int i = 0; ok && i < u.n; i++, t++) {
          const int kb = u.block(i);
          const uint32_t ks = t % KS, vs = t % VS;
          ok = waitw(&st->k_empty[ks], t / KS + 1, ST_BQ_KV_EMPTY);
          if (!ok) break;
          // K multiplies dS: rows that no query sees have to be zero there. What they make of S and dP is dropped by a select.
          const bool fix = has_dead(u.sp, kb, p.window, p.sinks);
          const uint32_t tile = ptx::smem_u32(sK + ks * Sh::KV_TILE), full = fix ? bar(&st->fixed) : bar(&st->k_full[ks]);
          if (lane == 0) {
            ptx::mbar_arrive_expect_tx(full, (uint32_t)Sh::KV_TILE);
            ptx::tma_load_3d(tile, &p.tmK, full, 0, u.sp.k_off + kb * TILE, kvh * (HD / 64));
          }
          if (fix) {
            ok = waitw(&st->fixed, fixes++, ST_FIX);
            if (!ok) break;
            zero_dead<HD>(tile, u.sp, kb, p.window, p.sinks, lane);
            ptx::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(bar(&st->k_full[ks]));
          }
          ok = waitw(&st->v_empty[vs], t / VS + 1, ST_BQ_KV_EMPTY);
          if (ok && lane == 0) {
            ptx::mbar_arrive_expect_tx(bar(&st->v_full[vs]), (uint32_t)Sh::KV_TILE);
            ptx::tma_load_3d(ptx::smem_u32(sV + vs * Sh::KV_TILE), &p.tmV, bar(&st->v_full[vs]), 0, u.sp.k_off + kb * TILE, kvh * (HD / 64));
          }
        }
      }
      __syncwarp();
    } else if (warp < 3) {
      // ================= S = Q K^T (warp 1) and dP = dO V^T (warp 2) =================
      if (lane == 0) {
        const bool is_s = warp == 1;
        const uint32_t idesc = ptx::make_idesc_bf16(TILE, TILE, 0, 0);
        const uint32_t a_base = ptx::smem_u32(is_s ? sQ : sDO), b_base = ptx::smem_u32(is_s ? sK : sV), col = tmem_base + (is_s ? COL_S : COL_DP);
        uint64_t *full = is_s ? &st->s_full : &st->dp_full, *read = is_s ? &st->s_read : &st->dp_read;
        const uint32_t slots = is_s ? KS : VS;
        uint32_t t = 0, units = 0;
        bool ok = true;
        for (int round = 0, unit = unit_at(0); ok && unit < p.units; unit = unit_at(++round)) {
          const int steps = q_unit_of(p, unit).n;
          ok = wait(&st->q_full, units++, ST_BQ_Q_FULL);
          for (int i = 0; ok && i < steps; i++, t++) {
            const uint32_t slot = t % slots;
            if (!(ok = wait(is_s ? &st->k_full[slot] : &st->v_full[slot], t / slots, ST_BQ_KV_FULL))) break;
            if (t > 0 && !(ok = wait(read, t - 1, ST_BQ_S_FREE))) break;
            ptx::tc_fence_after();
            const uint64_t ad = tile_desc(a_base, 0), bd = tile_desc(b_base + slot * Sh::KV_TILE, 0);
#pragma unroll
            for (int k16 = 0; k16 < HD / 16; k16++) {
              const uint32_t off = (uint32_t)((k16 >> 2) * SLAB + (k16 & 3) * 32);
              ptx::umma_bf16(col, desc_at(ad, off), desc_at(bd, off), idesc, k16 > 0);
            }
            ptx::umma_commit(bar(full));
            if (!is_s) ptx::umma_commit(bar(&st->v_empty[slot]));  // K is read again by the dQ product
            if (i == steps - 1) ptx::umma_commit(bar(&st->q_empty));
          }
        }
      }
      __syncwarp();
    } else {
      // ================= dQ += dS K =================
      if (lane == 0) {
        const uint32_t idesc = ptx::make_idesc_bf16(TILE, HD, 0, 1);  // K is read with its head dimension contiguous
        const uint32_t k_base = ptx::smem_u32(sK);
        uint32_t t = 0, units = 0;
        bool ok = true;
        for (int round = 0, unit = unit_at(0); ok && unit < p.units; unit = unit_at(++round), units++) {
          const int steps = q_unit_of(p, unit).n;
          const uint32_t acc = units % ACCS;
          // the unit before in this accumulator has been read out
          if (units >= ACCS) ok = wait(&st->acc_empty[acc], units / ACCS - 1, ST_BQ_ACC);
          for (int i = 0; ok && i < steps; i++, t++) {
            const uint32_t slot = t % KS;
            if (!(ok = wait(&st->ds_ready[t & 1], t / 2, ST_BQ_DS))) break;
            if (!(ok = wait(&st->k_full[slot], t / KS, ST_BQ_KV_FULL))) break;
            ptx::tc_fence_after();
            const uint64_t bd = tile_desc(k_base + slot * Sh::KV_TILE, SLAB);
#pragma unroll
            for (int k16 = 0; k16 < TILE / 16; k16++)
              ptx::umma_bf16_ts(tmem_base + COL_DQ + acc * HD, tmem_base + COL_DS + (t & 1) * 64 + k16 * 8, desc_at(bd, (uint32_t)(k16 * 2048)), idesc,
                                i > 0 || k16 > 0);
            ptx::umma_commit(bar(&st->dq_done[t & 1]));
            ptx::umma_commit(bar(&st->k_empty[slot]));
            if (i == steps - 1) ptx::umma_commit(bar(&st->acc_full[acc]));
          }
        }
      }
      __syncwarp();
    }
  } else if (warp < 8) {
    ptx::reg_dec<REGS_BWD_Q_OTHER>();
    // ================= row statistics of the next unit, output of the last one =================
    const int quarter = warp & 3, trow = quarter * 32 + lane;
    const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16);
    auto statistics = [&](int unit, uint32_t units) {
      const QUnit u = q_unit_of(p, unit);
      const uint32_t set = units & 1;
      if (units > 1 && !wait(&st->stat_empty[set], units / 2 - 1, ST_BQ_STAT)) return false;
      const int64_t row0 = u.sp.q_off + u.x.row;
      const int rows = u.sp.Tq - u.x.row;
      // delta = dO . O: HD / 8 lanes a row, this warp's 32 rows, asked for at once
      constexpr int LANES = HD / 8, AT_ONCE = 32 / LANES;
      if (trow < rows) {
        const int64_t at = ((row0 + trow) * p.q_heads + u.x.h) * HD;
#pragma unroll
        for (int q = 0; q < HD / 64; q++) {
          asm volatile("prefetch.global.L2 [%0];" ::"l"(p.dout + at + q * 64));
          asm volatile("prefetch.global.L2 [%0];" ::"l"(p.o + at + q * 64));
        }
      }
#pragma unroll 4
      for (int q = 0; q < 32; q += AT_ONCE) {
        const int r = quarter * 32 + q + lane / LANES;
        float d = 0.0f;
        if (r < rows) {
          const int64_t at = ((row0 + r) * p.q_heads + u.x.h) * LANES + lane % LANES;
          float x[8], y[8];
          unpack8(reinterpret_cast<const uint4 *>(p.dout)[at], x);
          unpack8(reinterpret_cast<const uint4 *>(p.o)[at], y);
#pragma unroll
          for (int j = 0; j < 8; j++) d = fmaf(x[j], y[j], d);
        }
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
        if (lane % LANES == 0) {
          st->delta[set][r] = d;
          if (r < rows) p.delta[(int64_t)u.x.h * p.total_q + row0 + r] = d;
        }
      }
      arrive(&st->stat_full[set]);
      return true;
    };
    uint32_t units = 0;
    int unit = unit_at(0);
    if (unit < p.units && !statistics(unit, 0)) goto teardown;
    for (int round = 0; unit < p.units; units++) {
      const int next = unit_at(++round);
      if (next < p.units && !statistics(next, units + 1)) goto teardown;
      const QUnit u = q_unit_of(p, unit);
      const int row = u.x.row + trow;
      __nv_bfloat16 *o = p.dq + ((int64_t)(u.sp.q_off + row) * p.q_heads + u.x.h) * HD;
      const uint32_t acc = units % ACCS;
      if (!wait(&st->acc_full[acc], units / ACCS, ST_BQ_DQ)) goto teardown;
      ptx::tc_fence_after();
#pragma unroll
      for (int q = 0; q < HD / 32; q++) {
        uint32_t r[32];
        load_columns<32>(lane_addr + COL_DQ + acc * HD + q * 32, r);
        if (q == HD / 32 - 1) {
          ptx::tc_fence_before();
          arrive(&st->acc_empty[acc]);
        }
        if (row < u.sp.Tq) {
          store16(o + q * 32, r, p.scale);
          store16(o + q * 32 + 16, r + 16, p.scale);
        }
      }
      unit = next;
    }
  } else {
    ptx::reg_inc<REGS_BWD_Q>();
    // ================= element-wise work: a thread per (query row, quarter of the columns) =================
    const int quarter = warp & 3, cols = (warp - 8) >> 2;  // columns 32 * cols ...
    const int trow = quarter * 32 + lane;
    const uint32_t lane_row = tmem_base + ((uint32_t)(quarter * 32) << 16), lane_addr = lane_row + cols * 32;
    const float c = p.scale * LOG2E;
    uint32_t t = 0, units = 0;
    for (int round = 0, unit = unit_at(0); unit < p.units; unit = unit_at(++round), units++) {
      const QUnit u = q_unit_of(p, unit);
      const int row = u.x.row + trow, pos = row + u.sp.shift;
      const int pos0 = u.x.row + u.sp.shift, last_pos = min(pos0 + TILE, u.sp.Tk) - 1;
      const float lse2 = row < u.sp.Tq ? p.lse[(int64_t)u.x.h * p.total_q + u.sp.q_off + row] * LOG2E : 0.0f;
      if (!wait(&st->stat_full[units & 1], units / 2, ST_BQ_STAT)) goto teardown;
      const float delta = st->delta[units & 1][trow];
      arrive(&st->stat_empty[units & 1]);
      for (int i = 0; i < u.n; i++, t++) {
        const int kb = u.block(i);
        uint32_t s[32], d[32];
        if (!wait(&st->s_full, t, ST_BQ_S)) goto teardown;
        ptx::tc_fence_after();
        load_columns<32>(lane_addr + COL_S, s);
        ptx::tc_fence_before();
        arrive(&st->s_read);
        probabilities<32>(s, c, -lse2);
        if (!wait(&st->dp_full, t, ST_BQ_DP)) goto teardown;
        ptx::tc_fence_after();
        load_columns<32>(lane_addr + COL_DP, d);
        ptx::tc_fence_before();
        arrive(&st->dp_read);
        score_gradients<32>(d, s, delta);
        if (!all_seen(kb * TILE, pos0, last_pos, p.window, p.sinks)) {
          const int base = kb * TILE + cols * 32;
          const uint32_t see = seen_bits(min(pos, u.sp.Tk - 1) - base, pos - p.window + 1 - base, p.sinks - base);
#pragma unroll
          for (int j = 0; j < 32; j++) d[j] = (see >> j) & 1u ? d[j] : 0u;
        }
        uint32_t ds[16];
#pragma unroll
        for (int j = 0; j < 16; j++) ds[j] = pack_bf16(__uint_as_float(d[2 * j]), __uint_as_float(d[2 * j + 1]));
        // the product of the step before the last has read these columns
        if (t > 1 && !wait(&st->dq_done[t & 1], t / 2 - 1, ST_BQ_DQ)) goto teardown;
        ptx::tc_fence_after();
        ptx::tmem_st16(lane_row + COL_DS + (t & 1) * 64 + cols * 16, ds);
        ptx::tmem_st_wait();
        ptx::tc_fence_before();
        arrive(&st->ds_ready[t & 1]);
      }
    }
  }

teardown:
  if (*abort_flag) {
    const uint64_t t0 = ptx::globaltimer_ns();
    while (ptx::globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

// ---- dK, dV ----------------------------------------------------------------------------------------------------------------
// The query tiles of a sequence that a block of keys walks: t0 .. t1 - 1 see it through the window; for a block with sinks tiles
// t1 .. tiles - 1 see the sinks only, and go to `chunks` further units of `chunk` tiles. (Host and device.)
struct KeyWalk {
  int t0, t1, tiles, chunk, chunks;
};
constexpr int MIN_CHUNK = 8;         // tiles of such a unit: at least this many, and as many as a block's window spans
constexpr int MAX_SPLIT_UNITS = 148;   // units that the heads of a small batch are split into: one per SM, at most so many (the workspace holds them)
constexpr int MAX_SPLIT_SINKS = 1024;  // more sinks than this fill the GPU with blocks of their own: their units walk every tile
__host__ __device__ inline KeyWalk key_walk(int Tq, int Tk, int kb, int window, int sinks, bool split = true) {
  KeyWalk w;
  const int shift = Tk - Tq;
  w.tiles = (Tq + TILE - 1) / TILE;
  const int64_t lo = (int64_t)kb * TILE - shift, hi = (int64_t)kb * TILE + TILE - 1 + window - 1 - shift;  // rows, hi inclusive
  w.t0 = lo > 0 ? (int)(lo / TILE) : 0;
  w.t1 = hi < 0 ? 0 : (hi >= Tq ? w.tiles : (int)(hi / TILE) + 1);
  if (w.t1 < w.t0) w.t1 = w.t0;
  w.chunk = window / TILE + 1 > MIN_CHUNK ? window / TILE + 1 : MIN_CHUNK;
  w.chunks = 0;
  if ((int64_t)kb * TILE < sinks) {
    if (!split || sinks > MAX_SPLIT_SINKS)
      w.t1 = w.tiles;
    else
      w.chunks = (w.tiles - w.t1 + w.chunk - 1) / w.chunk;
  }
  return w;
}
// blocks with sinks whose far tiles are split off, and the most units one of them is split into (the first block's)
__host__ __device__ inline int split_blocks(int Tk, int sinks) {
  if (sinks > MAX_SPLIT_SINKS) return 0;
  const int s = sinks < Tk ? sinks : Tk;
  return (s + TILE - 1) / TILE;
}

template <int HD>
struct BwdKShape {
  static constexpr int T_TILE = TILE * HD * 2;
  static constexpr int Q_SLOTS = HD == 128 ? 2 : 3, DO_SLOTS = HD == 128 ? 1 : 3;
  struct Tail {
    uint64_t kv_full, q_full[Q_SLOTS], q_empty[Q_SLOTS], do_full[DO_SLOTS], do_empty[DO_SLOTS], s_full, s_read, dp_full, dp_read, p_ready, ds_ready,
        dv_done, dk_done, fixed;
    uint32_t tmem_base;
    int abort_flag;
  };
  static constexpr size_t smem = 1024 + (2 + Q_SLOTS + DO_SLOTS) * (size_t)T_TILE + 2 * DS_TILE + sizeof(Tail);
  static_assert(smem <= 232448, "more shared memory than a CTA can be given");
};

template <int HD>
__global__ void __launch_bounds__(BWD_KV_THREADS, 1) window_bwd_kv_kernel(const __grid_constant__ BwdParams p) {
  using Sh = BwdKShape<HD>;
  constexpr int KSL = HD / 64, QS = Sh::Q_SLOTS, DS = Sh::DO_SLOTS;
  constexpr uint32_t TMEM_COLS = 512, COL_S = 0, COL_DP = 128, COL_DK = 256, COL_DV = 384;
  extern __shared__ unsigned char window_smem[];
  unsigned char *smem = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(window_smem) + 1023) & ~static_cast<uintptr_t>(1023));
  unsigned char *sK = smem, *sV = sK + Sh::T_TILE, *sP = sV + Sh::T_TILE, *sDS = sP + DS_TILE, *sQ = sDS + DS_TILE, *sDO = sQ + QS * Sh::T_TILE;
  auto *st = reinterpret_cast<typename Sh::Tail *>(sDO + DS * Sh::T_TILE);
  volatile int *abort_flag = &st->abort_flag;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  auto bar = [&](uint64_t *b) { return ptx::smem_u32(b); };
  auto wait = [&](uint64_t *b, uint32_t par, int code) { return ptx::mbar_wait<false>(bar(b), par & 1u, abort_flag, p.status, code); };
  // every thread arrives for itself (one arrival per warp measured the same)
  auto arrive = [&](uint64_t *b) { ptx::mbar_arrive(bar(b)); };

  if (tid == 0) {
    ptx::mbar_init(bar(&st->kv_full), 1);
    for (int s = 0; s < QS; s++) {
      ptx::mbar_init(bar(&st->q_full[s]), 1);
      ptx::mbar_init(bar(&st->q_empty[s]), 1);
    }
    for (int s = 0; s < DS; s++) {
      ptx::mbar_init(bar(&st->do_full[s]), 1);
      ptx::mbar_init(bar(&st->do_empty[s]), 2);  // dP and dV
    }
    ptx::mbar_init(bar(&st->s_full), 1);
    ptx::mbar_init(bar(&st->s_read), 512);
    ptx::mbar_init(bar(&st->dp_full), 1);
    ptx::mbar_init(bar(&st->dp_read), 512);
    ptx::mbar_init(bar(&st->p_ready), 512);
    ptx::mbar_init(bar(&st->ds_ready), 512);
    ptx::mbar_init(bar(&st->dv_done), 1);
    ptx::mbar_init(bar(&st->dk_done), 1);
    ptx::mbar_init(bar(&st->fixed), 1);
    st->abort_flag = 0;
    ptx::fence_barrier_init();
    ptx::fence_proxy_async_smem();
  }
  if (warp == 1) {
    ptx::tmem_alloc(ptx::smem_u32(&st->tmem_base), TMEM_COLS);
    ptx::tmem_relinquish();
  }
  if (warp == 0 && lane == 0) {
    ptx::tma_prefetch_desc(&p.tmQ);
    ptx::tma_prefetch_desc(&p.tmK);
    ptx::tma_prefetch_desc(&p.tmV);
    ptx::tma_prefetch_desc(&p.tmdO);
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem_base = st->tmem_base;
  pdl_release();
  pdl_wait();

  // the unit: a block of keys of one key/value head, and the query tiles it walks for every query head of the group
  const int unit = blockIdx.x / p.parts, head_part = blockIdx.x % p.parts;
  const int h0 = head_part * p.group / p.parts, heads = (head_part + 1) * p.group / p.parts - h0;  // of the group
  int s = 0, kb, kvh, t0, t1, share = -1;  // share: the slot of the workspace that takes the sink rows
  if (unit < p.main_units) {
    while (unit >= p.seqs.first[s + 1]) s++;
    const int rel = unit - p.seqs.first[s];
    kvh = rel % p.kv_heads;
    kb = rel / p.kv_heads;
  } else {
    while (unit - p.main_units >= p.far[s + 1]) s++;
    kvh = (unit - p.main_units - p.far[s]) % p.kv_heads;
    kb = 0;
  }
  const Span sp = span_of(p.seqs, s);
  const int most = key_walk(sp.Tq, sp.Tk, 0, p.window, p.sinks, p.parts == 1).chunks;
  int part = 0;
  if (unit >= p.main_units) {
    const int rel = (unit - p.main_units - p.far[s]) / p.kv_heads;  // block, then chunk
    kb = rel / most;
    part = 1 + rel % most;
  }
  {
    const KeyWalk w = key_walk(sp.Tq, sp.Tk, kb, p.window, p.sinks, p.parts == 1);
    t0 = part == 0 ? w.t0 : w.t1 + (part - 1) * w.chunk;
    t1 = part == 0 ? w.t1 : min(w.tiles, t0 + w.chunk);
    if (w.chunks > 0) share = p.slot[s] + kb * (most + 1) + part;
    if (part > w.chunks) share = -1;  // this block is split into fewer units than the first: nothing to do
  }
  if (p.parts > 1) share = blockIdx.x;
  const int share_rows = p.parts > 1 ? sp.Tk : p.sinks;  // keys below this go to the share
  const int tiles = max(0, t1 - t0), n = tiles * heads;

  if (n > 0 && warp == 0) {
    // ================= loads: the whole warp walks, one lane issues =================
    bool ok = true;
    uint32_t fixes = 0;
    auto waitw = [&](uint64_t *b, uint32_t par, int code) { return __all_sync(0xffffffffu, wait(b, par, code)) != 0; };
    if (lane == 0) {
      ptx::mbar_arrive_expect_tx(bar(&st->kv_full), (uint32_t)(2 * Sh::T_TILE));
      ptx::tma_load_3d(ptx::smem_u32(sK), &p.tmK, bar(&st->kv_full), 0, sp.k_off + kb * TILE, kvh * KSL);
      ptx::tma_load_3d(ptx::smem_u32(sV), &p.tmV, bar(&st->kv_full), 0, sp.k_off + kb * TILE, kvh * KSL);
    }
    for (int i = 0, tile_at = t0, h = kvh * p.group + h0; ok && i < n; i++) {
      const int row = tile_at * TILE;
      const bool fix = row + TILE > sp.Tq;  // rows past the sequence's end are zeroed: dO and Q multiply P and dS
#pragma unroll
      for (int which = 0; which < 2; which++) {
        const int slot = which == 0 ? i % QS : i % DS;
        uint64_t *empty = which == 0 ? &st->q_empty[slot] : &st->do_empty[slot], *full_b = which == 0 ? &st->q_full[slot] : &st->do_full[slot];
        if (!ok) continue;
        ok = waitw(empty, (uint32_t)(i / (which == 0 ? QS : DS)) + 1, which == 0 ? ST_BK_Q_EMPTY : ST_BK_DO_EMPTY);
        if (!ok) continue;
        const uint32_t tile = ptx::smem_u32((which == 0 ? sQ : sDO) + slot * Sh::T_TILE), full = fix ? bar(&st->fixed) : bar(full_b);
        if (lane == 0) {
          ptx::mbar_arrive_expect_tx(full, (uint32_t)Sh::T_TILE);
          ptx::tma_load_3d(tile, which == 0 ? &p.tmQ : &p.tmdO, full, 0, sp.q_off + row, h * KSL);
        }
        if (!fix) continue;
        ok = waitw(&st->fixed, fixes++, ST_BK_FIX);
        if (!ok) continue;
        for (int r = sp.Tq - row + lane; r < TILE; r += 32)
#pragma unroll
          for (int q = 0; q < KSL; q++)
#pragma unroll
            for (int e = 0; e < 8; e++) sts128(tile + q * SLAB + r * 128 + e * 16, make_uint4(0, 0, 0, 0));
        ptx::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(bar(full_b));
      }
      if (++tile_at == t1) {
        tile_at = t0;
        h++;
      }
    }
    __syncwarp();
  } else if (n > 0 && warp == 1) {
    // ================= S = Q K^T, dP = dO V^T =================
    if (lane == 0) {
      const uint32_t idesc = ptx::make_idesc_bf16(TILE, TILE, 0, 0);
      auto product = [&](uint32_t a, uint32_t b, uint32_t col) {
        const uint64_t ad = tile_desc(a, 0), bd = tile_desc(b, 0);
#pragma unroll
        for (int k16 = 0; k16 < HD / 16; k16++) {
          const uint32_t off = (uint32_t)((k16 >> 2) * SLAB + (k16 & 3) * 32);
          ptx::umma_bf16(tmem_base + col, desc_at(ad, off), desc_at(bd, off), idesc, k16 > 0);
        }
      };
      bool ok = wait(&st->kv_full, 0, ST_BK_KV);
      for (int i = 0; ok && i < n; i++) {
        if (!wait(&st->q_full[i % QS], (uint32_t)(i / QS), ST_BK_Q)) break;
        if (i > 0 && !wait(&st->s_read, (uint32_t)(i - 1), ST_BK_S_FREE)) break;
        ptx::tc_fence_after();
        product(ptx::smem_u32(sQ + (i % QS) * Sh::T_TILE), ptx::smem_u32(sK), COL_S);
        ptx::umma_commit(bar(&st->s_full));
        if (!wait(&st->do_full[i % DS], (uint32_t)(i / DS), ST_BK_DO)) break;
        if (i > 0 && !wait(&st->dp_read, (uint32_t)(i - 1), ST_BK_DP_FREE)) break;
        ptx::tc_fence_after();
        product(ptx::smem_u32(sDO + (i % DS) * Sh::T_TILE), ptx::smem_u32(sV), COL_DP);
        ptx::umma_commit(bar(&st->dp_full));
        ptx::umma_commit(bar(&st->do_empty[i % DS]));
      }
    }
    __syncwarp();
  } else if (n > 0 && warp < 4) {
    // ================= dV += P^T dO (warp 2), dK += dS^T Q (warp 3) =================
    if (lane == 0) {
      const bool is_v = warp == 2;
      const uint32_t idesc = ptx::make_idesc_bf16(TILE, HD, 1, 1);  // both operands with their rows as the reduction
      const uint32_t a_base = ptx::smem_u32(is_v ? sP : sDS), b_base = ptx::smem_u32(is_v ? sDO : sQ), col = tmem_base + (is_v ? COL_DV : COL_DK);
      const uint32_t slots = is_v ? DS : QS;
      for (int i = 0; i < n; i++) {
        const uint32_t slot = (uint32_t)i % slots;
        if (!wait(is_v ? &st->p_ready : &st->ds_ready, (uint32_t)i, is_v ? ST_BK_P : ST_BK_DS)) break;
        if (!wait(is_v ? &st->do_full[slot] : &st->q_full[slot], (uint32_t)i / slots, ST_BK_DO)) break;
        ptx::tc_fence_after();
        const uint64_t ad = tile_desc(a_base, SLAB), bd = tile_desc(b_base + slot * Sh::T_TILE, SLAB);
#pragma unroll
        for (int k16 = 0; k16 < TILE / 16; k16++)
          ptx::umma_bf16(col, desc_at(ad, (uint32_t)(k16 * 2048)), desc_at(bd, (uint32_t)(k16 * 2048)), idesc, i > 0 || k16 > 0);
        ptx::umma_commit(bar(is_v ? &st->dv_done : &st->dk_done));
        ptx::umma_commit(bar(is_v ? &st->do_empty[slot] : &st->q_empty[slot]));
      }
    }
    __syncwarp();
  } else if (warp >= 4) {
    // ================= element-wise work: a thread per (query row, quarter of the keys); at the end per (key, quarter of the dims) ====
    const int quarter = warp & 3, cols = (warp - 4) >> 2;
    const int trow = quarter * 32 + lane;
    const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16);
    const uint32_t slab_row = (uint32_t)((cols >> 1) * SLAB + trow * 128);
    const uint32_t p_addr = ptx::smem_u32(sP) + slab_row, ds_addr = ptx::smem_u32(sDS) + slab_row;
    const float c = p.scale * LOG2E;
    // a step's statistics are fetched while the step before computes: `ahead` is its tile, stat_at its row in the arrays
    int ahead = t0;
    int64_t stat_at = (int64_t)(kvh * p.group + h0) * p.total_q + sp.q_off + t0 * TILE + trow;
    float lse2 = 0.0f, delta = 0.0f, next_lse = 0.0f, next_delta = 0.0f;
    auto fetch = [&]() {
      if (ahead * TILE + trow < sp.Tq) {
        next_lse = p.lse[stat_at];
        next_delta = p.delta[stat_at];
      }
      stat_at += TILE;
      if (++ahead == t1) {
        ahead = t0;
        stat_at += p.total_q - tiles * TILE;
      }
    };
    if (n > 0) fetch();
    for (int i = 0, tile_at = t0; i < n; i++) {
      lse2 = next_lse * LOG2E;
      delta = next_delta;
      if (i + 1 < n) fetch();
      const int row0 = tile_at * TILE, row = row0 + trow, pos = row + sp.shift, pos0 = row0 + sp.shift;
      if (++tile_at == t1) tile_at = t0;
      uint32_t see = 0xffffffffu;
      if (row0 + TILE > sp.Tq || !all_seen(kb * TILE, pos0, pos0 + TILE - 1, p.window, p.sinks)) {
        const int base = kb * TILE + cols * 32;
        see = row < sp.Tq ? seen_bits(pos - base, pos - p.window + 1 - base, p.sinks - base) : 0u;
      }
      const bool masked = __any_sync(0xffffffffu, see != 0xffffffffu);
      uint32_t x[32], d[32];
      if (!wait(&st->s_full, (uint32_t)i, ST_BK_S)) goto teardown;
      ptx::tc_fence_after();
      load_columns<32>(lane_addr + COL_S + cols * 32, x);
      ptx::tc_fence_before();
      arrive(&st->s_read);
      probabilities<32>(x, c, -lse2);
      if (masked) {
#pragma unroll
        for (int j = 0; j < 32; j++) x[j] = (see >> j) & 1u ? x[j] : 0u;
      }
      if (i > 0 && !wait(&st->dv_done, (uint32_t)(i - 1), ST_BK_DV)) goto teardown;  // has read P
      store_chunks<4>(p_addr, trow, (cols & 1) * 4, x);
      ptx::fence_proxy_async_smem();
      ptx::tc_fence_before();
      arrive(&st->p_ready);
      if (!wait(&st->dp_full, (uint32_t)i, ST_BK_DP)) goto teardown;
      ptx::tc_fence_after();
      load_columns<32>(lane_addr + COL_DP + cols * 32, d);
      ptx::tc_fence_before();
      arrive(&st->dp_read);
      score_gradients<32>(d, x, delta);
      if (masked) {  // a masked product may be anything
#pragma unroll
        for (int j = 0; j < 32; j++) d[j] = (see >> j) & 1u ? d[j] : 0u;
      }
      if (i > 0 && !wait(&st->dk_done, (uint32_t)(i - 1), ST_BK_DK)) goto teardown;  // has read dS
      store_chunks<4>(ds_addr, trow, (cols & 1) * 4, d);
      ptx::fence_proxy_async_smem();
      ptx::tc_fence_before();
      arrive(&st->ds_ready);
    }
    if (n > 0) {
      if (!wait(&st->dk_done, (uint32_t)(n - 1), ST_BK_DK) || !wait(&st->dv_done, (uint32_t)(n - 1), ST_BK_DV)) goto teardown;
      ptx::tc_fence_after();
    }
    if (n > 0 || part == 0) {
      // the accumulators' lanes are keys
      constexpr int DIMS = HD / 4;
      const int key = kb * TILE + trow;
      const bool to_share = share >= 0 && key < share_rows;
      const int64_t slot = p.parts > 1 ? share : (int64_t)share * p.kv_heads + kvh;
      float *sh = to_share ? p.shares + (slot * p.slot_rows + trow) * 2 * HD + cols * DIMS : nullptr;
      const int64_t at = ((int64_t)(sp.k_off + key) * p.kv_heads + kvh) * HD + cols * DIMS;
#pragma unroll
      for (int which = 0; which < 2; which++) {
        uint32_t r[DIMS];
        if (n > 0) {
          load_columns<DIMS>(lane_addr + (which == 0 ? COL_DK : COL_DV) + cols * DIMS, r);
        } else {
#pragma unroll
          for (int j = 0; j < DIMS; j++) r[j] = 0u;
        }
        const float f = which == 0 ? p.scale : 1.0f;
        if (key >= sp.Tk) continue;
        if (to_share) {
#pragma unroll
          for (int q = 0; q < DIMS / 4; q++)
            reinterpret_cast<float4 *>(sh + which * HD)[q] = make_float4(__uint_as_float(r[4 * q]) * f, __uint_as_float(r[4 * q + 1]) * f,
                                                                         __uint_as_float(r[4 * q + 2]) * f, __uint_as_float(r[4 * q + 3]) * f);
        } else if (part == 0) {
#pragma unroll
          for (int q = 0; q < DIMS / 16; q++) store16((which == 0 ? p.dk : p.dv) + at + q * 16, r + q * 16, f);
        }
      }
    }
  }

teardown:
  if (*abort_flag) {
    const uint64_t t_abort = ptx::globaltimer_ns();
    while (ptx::globaltimer_ns() - t_abort < 200000ull) __nanosleep(1000);
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

// dK and dV of the sink rows: the shares of a block's units, in order. Grid: (blocks with sinks * kv heads, sequences, elements of a
// block's rows / 256); a thread per element.
__global__ void __launch_bounds__(256) window_join_kernel(const __grid_constant__ BwdParams p, int head_dim) {
  pdl_release();
  pdl_wait();
  const int s = blockIdx.y, kb = blockIdx.x / p.kv_heads, kvh = blockIdx.x % p.kv_heads;
  const Span sp = span_of(p.seqs, s);
  if (kb >= split_blocks(sp.Tk, p.sinks)) return;
  const int chunks = key_walk(sp.Tq, sp.Tk, kb, p.window, p.sinks).chunks, most = key_walk(sp.Tq, sp.Tk, 0, p.window, p.sinks).chunks;
  const int rows = min(min(p.sinks, sp.Tk) - kb * TILE, TILE), i = blockIdx.z * 256 + threadIdx.x;
  if (chunks == 0 || i >= rows * 2 * head_dim) return;
  const int64_t step = (int64_t)p.kv_heads * p.slot_rows * 2 * head_dim;
  const float *share = p.shares + ((int64_t)(p.slot[s] + kb * (most + 1)) * p.kv_heads + kvh) * p.slot_rows * 2 * head_dim + i;
  float sum = 0.0f;
#pragma unroll 8
  for (int c = 0; c <= chunks; c++) sum += share[c * step];
  const int row = i / (2 * head_dim), d = i - row * 2 * head_dim;
  const int64_t at = ((int64_t)(sp.k_off + kb * TILE + row) * p.kv_heads + kvh) * head_dim;
  if (d < head_dim)
    p.dk[at + d] = __float2bfloat16_rn(sum);
  else
    p.dv[at + d - head_dim] = __float2bfloat16_rn(sum);
}

// dK and dV of blocks whose heads were split: their shares, in order. Grid: (blocks of keys * kv heads, elements of a block / 256).
__global__ void __launch_bounds__(256) window_join_heads_kernel(const __grid_constant__ BwdParams p, int head_dim) {
  pdl_release();
  pdl_wait();
  int s = 0;
  while ((int)blockIdx.x >= p.seqs.first[s + 1]) s++;
  const Span sp = span_of(p.seqs, s);
  const int rel = blockIdx.x - p.seqs.first[s], kvh = rel % p.kv_heads, kb = rel / p.kv_heads, i = blockIdx.y * 256 + threadIdx.x;
  const int row = i / (2 * head_dim), d = i - row * 2 * head_dim, key = kb * TILE + row;
  if (key >= sp.Tk) return;
  const int64_t step = (int64_t)TILE * 2 * head_dim;
  const float *share = p.shares + (int64_t)blockIdx.x * p.parts * step + i;
  float sum = 0.0f;
#pragma unroll 8
  for (int c = 0; c < p.parts; c++) sum += share[c * step];
  const int64_t at = ((int64_t)(sp.k_off + key) * p.kv_heads + kvh) * head_dim;
  if (d < head_dim)
    p.dk[at + d] = __float2bfloat16_rn(sum);
  else
    p.dv[at + d - head_dim] = __float2bfloat16_rn(sum);
}

bool sm100_supported(int head_dim) { return head_dim == 64 || head_dim == 128; }

}  // namespace window
}  // namespace b200

using namespace b200;

namespace {

// SM count of the current device, and the kernels' shared-memory limit raised there on first use
struct Device {
  int dev, sms;
};
int current_device(Device *d) {
  B200_CUDA(cudaGetDevice(&d->dev));
  B200_REQUIRE(d->dev >= 0 && d->dev < MAX_DEVICES, "attention_window: device ordinal %d is out of range", d->dev);
  B200_CUDA(cudaDeviceGetAttribute(&d->sms, cudaDevAttrMultiProcessorCount, d->dev));
  return 0;
}
template <typename K>
int allow_smem(K kernel, size_t bytes, bool *done) {
  if (*done) return 0;
  B200_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
  *done = true;
  return 0;
}

// bf16 [rows][cols] as [cols / 64][rows][64]: one copy brings a tile of 128 rows of one head, slab by slab (128-byte swizzle, rows past
// the end read as zeros)
int tile_map(CUtensorMap *m, const void *base, int rows, uint64_t cols, int head_dim) {
  EncodeTiledFn fn = encode_fn();
  B200_REQUIRE(fn != nullptr, "attention_window: cuTensorMapEncodeTiled is not available from this driver");
  cuuint64_t dims[3] = {64, (cuuint64_t)rows, cols / 64};
  cuuint64_t strides[2] = {cols * 2, 128};
  cuuint32_t box[3] = {64, window::TILE, (cuuint32_t)head_dim / 64};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  B200_REQUIRE(r == CUDA_SUCCESS, "attention_window: cuTensorMapEncodeTiled failed with code %d", (int)r);
  return 0;
}

// Deals the units of a launch out to `ctas` CTAs; no runs where there are too many, or nothing to deal. cost(unit) in any measure; next(unit): the
// first unit behind it that may cost something else.
template <typename F, typename G>
void deal(window::Schedule *s, int sequences, int units, int ctas, F cost, G next) {
  constexpr int MAX_CLASSES = 128;
  struct Class {
    int cost, unit, n;
  } cls[MAX_CLASSES];
  struct Group {  // CTAs cta .. cta + n - 1 have the same load
    int load, cta, n;
  } grp[MAX_CLASSES + window::MAX_RUNS];
  s->n = 0;
  if (units <= ctas || sequences == 1) return;
  int classes = 0;
  for (int unit = 0; unit < units;) {
    const int end = next(unit), c = cost(unit);
    if (classes > 0 && cls[classes - 1].cost == c && cls[classes - 1].unit + cls[classes - 1].n == unit) {
      cls[classes - 1].n += end - unit;
    } else {
      if (classes == MAX_CLASSES) return;
      cls[classes++] = Class{c, unit, end - unit};
    }
    unit = end;
  }
  std::stable_sort(cls, cls + classes, [](const Class &a, const Class &b) { return a.cost > b.cost; });
  int groups = 1, runs = 0;
  grp[0] = Group{0, 0, ctas};
  for (int i = 0; i < classes; i++)
    while (cls[i].n > 0) {
      int least = 0;
      for (int g = 1; g < groups; g++)
        if (grp[g].load < grp[least].load) least = g;
      Group &from = grp[least];
      const int n = from.n < cls[i].n ? from.n : cls[i].n;
      if (runs == window::MAX_RUNS) return;
      s->run[runs++] = window::Schedule::Run{cls[i].unit, (unsigned short)from.cta, (unsigned short)n};
      cls[i].unit += n;
      cls[i].n -= n;
      const Group to = {from.load + cls[i].cost, from.cta, n};
      from.cta += n;
      from.n -= n;
      if (from.n == 0) from = to;
      else grp[groups++] = to;
    }
  s->n = runs;
}

template <int HD, int WALK>
int allow_fwd(const Device &d) {
  static bool done[MAX_DEVICES];
  return allow_smem(window::window_fwd_kernel<HD, WALK>, window::FwdShape<HD>::smem, &done[d.dev]);
}
template <int HD, int WALK>
int launch_fwd(const window::FwdParams &p, const Device &d, cudaStream_t s) {
  constexpr size_t smem = window::FwdShape<HD>::smem;
  static_assert(smem >= 1024 + 2 * window::TILE * (HD + 2 + window::MAX_SHARERS) * sizeof(float), "the parts of a shared unit");
  if (allow_fwd<HD, WALK>(d)) return -1;
  const int ctas = p.units * p.cluster;
  B200_CUDA(b200_launch_overlapped(window::window_fwd_kernel<HD, WALK>, dim3(ctas < d.sms ? ctas : d.sms), dim3(window::FWD_THREADS), smem, s,
                                   (unsigned)p.cluster, p));
  B200_CHECK_LAUNCH("attention_window_fwd");
  return 0;
}
template <int HD>
int launch_fwd(const window::FwdParams &p, const Device &d, cudaStream_t s) {
  if (p.cluster > 1) return launch_fwd<HD, window::WALK_SHARED>(p, d, s);
  return p.schedule.n > 0 ? launch_fwd<HD, window::WALK_DEALT>(p, d, s) : launch_fwd<HD, window::WALK_ROUNDS>(p, d, s);
}

template <int HD>
int launch_bwd_q(const window::BwdParams &p, const Device &d, cudaStream_t s) {
  static bool done[MAX_DEVICES];
  constexpr size_t smem = window::BwdQShape<HD>::smem;
  if (allow_smem(window::window_bwd_q_kernel<HD>, smem, &done[d.dev])) return -1;
  B200_CUDA(b200_launch_overlapped(window::window_bwd_q_kernel<HD>, dim3(p.units < d.sms ? p.units : d.sms), dim3(window::BWD_Q_THREADS), smem, s, 1, p));
  B200_CHECK_LAUNCH("attention_window_bwd (dQ)");
  return 0;
}

template <int HD>
int launch_bwd_kv(const window::BwdParams &p, const Device &d, cudaStream_t s) {
  static bool done[MAX_DEVICES];
  constexpr size_t smem = window::BwdKShape<HD>::smem;
  if (allow_smem(window::window_bwd_kv_kernel<HD>, smem, &done[d.dev])) return -1;
  B200_CUDA(b200_launch_overlapped(window::window_bwd_kv_kernel<HD>, dim3(p.units), dim3(window::BWD_KV_THREADS), smem, s, 1, p));
  B200_CHECK_LAUNCH("attention_window_bwd (dK, dV)");
  return 0;
}

uint64_t up256(uint64_t v) { return (v + 255) / 256 * 256; }

// blocks of 128 keys that a tile of queries sees, at most (of 128 queries that see a block of keys, with the queries' number)
int blocks_seen(const window::Call &c, int Tk, int rows) {
  const int64_t span = (int64_t)c.window + 2 * window::TILE + (c.sinks < Tk ? c.sinks : Tk);
  return (int)(((span < rows ? span : rows) + window::TILE - 1) / window::TILE);
}

// CTAs that share a pair, as long as all clusters have a seat at once: joining their parts takes 6 to 8 us, a block that one walks 1.4 (half a pair) or
// 1.9. Measured at head size 128, in halves and with 2, 4, 8 CTAs a pair: 9 pairs of 10 blocks 19, 23, 17, 17 us, of 16 27, 28, 20, 17; 33 pairs of 16
// 28, 30, 22, of 24 38, 37, 25; 74 pairs of 16 29, 31, of 24 40, 39, of 48 73, 61. Without a seat for every cluster: 16 pairs of 24 with 4 and with 8
// 23, 35; 34 pairs of 10, in halves and with 4, 19, 33, of 48, with 2 and with 4, 59, 67. Head size 64: the same borders.
template <int HD>
int sharers(int pairs, int blocks, int dev) {
  static int known[MAX_DEVICES][window::MAX_SHARERS + 1];
  for (int size = window::MAX_SHARERS; size > 1; size /= 2)
    if (blocks >= (size == 8 ? 16 : size == 4 ? 10 : 22) &&
        pairs <= window::cluster_seats(window::window_fwd_kernel<HD, window::WALK_SHARED>, window::FWD_THREADS, window::FwdShape<HD>::smem, size,
                                       &known[dev][size]))
      return size;
  return 1;
}

int slot_rows(int sinks) { return sinks < window::TILE ? sinks : window::TILE; }

}  // namespace

namespace b200 {
namespace window {

// delta, then the shares: those of split heads or those of the sink rows. A block's sink shares: its own and those of at most ceil(tiles / MIN_CHUNK) further units, that is
// Tq / 1024 + 3 at most.
uint64_t sm100_bwd_workspace(int num_seqs, int q_heads, int kv_heads, int head_dim, int total_q, int sinks) {
  static_assert(TILE * MIN_CHUNK == 1024, "the bound on a sequence's shares");
  uint64_t n = 0;
  if (q_heads > kv_heads) n = (uint64_t)MAX_SPLIT_UNITS * TILE * 2 * head_dim * sizeof(float);
  if (sinks > 0 && sinks <= MAX_SPLIT_SINKS) {
    const uint64_t seqs = num_seqs < MAX_SEQS ? num_seqs : MAX_SEQS;  // of one launch
    const uint64_t shares = (uint64_t)((sinks + TILE - 1) / TILE) * ((uint64_t)total_q / 1024 + 3 * seqs) * kv_heads * slot_rows(sinks) * 2 * head_dim * sizeof(float);
    if (shares > n) n = shares;
  }
  return up256((uint64_t)total_q * q_heads * sizeof(float)) + n;
}

int sm100_bwd(const Call &c) {
  BwdParams p;
  Device d;
  if (current_device(&d)) return -1;
  const uint64_t Dq = (uint64_t)c.q_heads * c.head_dim, Dk = (uint64_t)c.kv_heads * c.head_dim;
  if (c.total_q == 0) {  // no query sees any key
    for (int s = 0; s < c.num_seqs; s++) {
      B200_CUDA(cudaMemsetAsync(c.dk + (int64_t)c.k_off[s] * Dk, 0, (size_t)c.k_len[s] * Dk * 2, c.stream));
      B200_CUDA(cudaMemsetAsync(c.dv + (int64_t)c.k_off[s] * Dk, 0, (size_t)c.k_len[s] * Dk * 2, c.stream));
    }
    return 0;
  }
  if (tile_map(&p.tmQ, c.q, c.total_q, Dq, c.head_dim) || tile_map(&p.tmdO, c.dout, c.total_q, Dq, c.head_dim) ||
      tile_map(&p.tmK, c.k, c.total_k, Dk, c.head_dim) || tile_map(&p.tmV, c.v, c.total_k, Dk, c.head_dim))
    return -1;
  p.o = c.o;
  p.dout = c.dout;
  p.lse = c.lse_in;
  p.delta = (float *)c.workspace;
  p.shares = (float *)(c.workspace + up256((uint64_t)c.total_q * c.q_heads * sizeof(float)));
  p.dq = c.dq;
  p.dk = c.dk;
  p.dv = c.dv;
  p.window = c.window;
  p.sinks = c.sinks;
  p.group = c.q_heads / c.kv_heads;
  p.q_heads = c.q_heads;
  p.kv_heads = c.kv_heads;
  p.total_q = c.total_q;
  p.scale = c.scale;
  p.main_units = 0;
  p.parts = 1;
  p.status = attn_status_ptr();
  B200_REQUIRE(p.status != nullptr, "attention_window: the status word of this device is not reachable");
  for (int next = 0; next < c.num_seqs;) {
    p.units = next_sequences(p.seqs, &next, c, [&](int s) { return (c.q_len[s] + TILE - 1) / TILE * c.q_heads; },
                             [&](int s) { return blocks_seen(c, c.k_len[s], c.k_len[s]); });
    if (p.units == 0) continue;
    if (c.head_dim == 128 ? launch_bwd_q<128>(p, d, c.stream) : launch_bwd_q<64>(p, d, c.stream)) return -1;
  }
  for (int next = 0; next < c.num_seqs;) {
    p.main_units = next_sequences(p.seqs, &next, c, [&](int s) { return (c.k_len[s] + TILE - 1) / TILE * c.kv_heads; },
                                  [&](int s) { return blocks_seen(c, c.k_len[s], c.q_len[s]); });
    if (p.main_units == 0) continue;
    // as many units as there are SMs, if the heads of a group give them
    const int wanted = d.sms < MAX_SPLIT_UNITS ? d.sms : MAX_SPLIT_UNITS;
    p.parts = p.main_units < wanted ? wanted / p.main_units : 1;
    if (p.parts > p.group) p.parts = p.group;
    p.slot_rows = p.parts > 1 ? TILE : slot_rows(c.sinks);
    int slots = 0, blocks = 0;
    p.far[0] = 0;
    for (int s = 0; s < p.seqs.n; s++) {
      const int split = split_blocks(p.seqs.Tk[s], c.sinks), chunks = key_walk(p.seqs.Tq[s], p.seqs.Tk[s], 0, c.window, c.sinks).chunks;
      const bool any = split > 0 && chunks > 0 && p.parts == 1;
      p.slot[s] = slots;
      p.far[s + 1] = p.far[s] + (any ? split * chunks * c.kv_heads : 0);
      if (any) slots += split * (chunks + 1);
      if (any && split > blocks) blocks = split;
    }
    p.units = p.parts > 1 ? p.main_units * p.parts : p.main_units + p.far[p.seqs.n];
    if (c.head_dim == 128 ? launch_bwd_kv<128>(p, d, c.stream) : launch_bwd_kv<64>(p, d, c.stream)) return -1;
    if (p.parts > 1) {
      const dim3 all((unsigned)p.main_units, (unsigned)(TILE * 2 * c.head_dim / 256));
      B200_CUDA(b200_launch_overlapped(window_join_heads_kernel, all, dim3(256), 0, c.stream, 1, p, c.head_dim));
      B200_CHECK_LAUNCH("attention_window_bwd (heads)");
    }
    if (blocks == 0) continue;
    const dim3 grid((unsigned)(blocks * c.kv_heads), (unsigned)p.seqs.n, (unsigned)(p.slot_rows * 2 * c.head_dim + 255) / 256);
    B200_CUDA(b200_launch_overlapped(window_join_kernel, grid, dim3(256), 0, c.stream, 1, p, c.head_dim));
    B200_CHECK_LAUNCH("attention_window_bwd (sinks)");
  }
  return 0;
}

int sm100_fwd(const Call &c) {
  if (few_fwd(c)) return -1;
  bool tiles = false;
  for (int s = 0; s < c.num_seqs && !tiles; s++) tiles = c.q_len[s] > 0 && !is_few(c, s);
  if (!tiles) return 0;
  FwdParams p;
  Device d;
  if (current_device(&d)) return -1;
  const uint64_t Dq = (uint64_t)c.q_heads * c.head_dim, Dk = (uint64_t)c.kv_heads * c.head_dim;
  if (tile_map(&p.tmQ, c.q, c.total_q, Dq, c.head_dim) || tile_map(&p.tmK, c.k, c.total_k, Dk, c.head_dim) ||
      tile_map(&p.tmV, c.v, c.total_k, Dk, c.head_dim))
    return -1;
  p.O = c.out;
  p.lse = c.lse;
  p.window = c.window;
  p.sinks = c.sinks;
  p.group = c.q_heads / c.kv_heads;
  p.q_heads = c.q_heads;
  p.total_q = c.total_q;
  p.pair_heads = p.group % 2 == 0;
  p.scale = c.scale;
  p.status = attn_status_ptr();
  B200_REQUIRE(p.status != nullptr, "attention_window: the status word of this device is not reachable");
  for (int next = 0; next < c.num_seqs;) {
    p.units = next_sequences(
        p.seqs, &next, c,
        [&](int s) {
          const int tiles = is_few(c, s) ? 0 : (c.q_len[s] + TILE - 1) / TILE;
          return p.pair_heads ? tiles * (c.q_heads / 2) : (tiles + 1) / 2 * c.q_heads;
        },
        [&](int s) { return blocks_seen(c, c.k_len[s], c.k_len[s]); });
    if (p.units == 0) continue;
    // In the last round, pairs are given to two CTAs as long as there are CTAs without one (8192 tokens, window 1024, 512 pairs: 103 -> 97
    // us; 400 tokens of 8 heads, 16 pairs: 14 -> 11). Not where the units of a long sequence run from one block to all: the last round's are
    // its short ones, and two halves take longer than a pair (no window: 246 -> 250 us).
    const int last = p.units % d.sms, halves = last < d.sms - last ? last : d.sms - last;
    const bool ramp = p.units > d.sms && c.window > p.seqs.Tk[0] / 2;
    const int blocks = blocks_seen(c, p.seqs.Tk[0], p.seqs.Tk[0]);
    if (c.head_dim == 128 ? allow_fwd<128, WALK_SHARED>(d) : allow_fwd<64, WALK_SHARED>(d)) return -1;
    p.cluster = c.head_dim == 128 ? sharers<128>(p.units, blocks, d.dev) : sharers<64>(p.units, blocks, d.dev);
    const int split = ramp || p.cluster > 1 ? 0 : halves;
    p.whole = p.units - split;
    p.units += split;
    // in quarters of a pair's step: a single tile's step takes three, a unit's begin and end five
    deal(
        &p.schedule, p.seqs.n, p.units, d.sms,
        [&](int unit) {
          const window::Unit u = window::unit_of(p, unit);
          return u.n * (u.b.exists ? 4 : 3) + 5;
        },
        [&](int unit) {
          if (unit >= p.whole) return unit + 1;
          int s = 0;
          while (unit >= p.seqs.first[s + 1]) s++;
          const int row = p.pair_heads ? c.q_heads / 2 : c.q_heads, end = p.seqs.first[s] + ((unit - p.seqs.first[s]) / row + 1) * row;
          return end < p.whole ? end : p.whole;
        });
    if (c.head_dim == 128 ? launch_fwd<128>(p, d, c.stream) : launch_fwd<64>(p, d, c.stream)) return -1;
  }
  return 0;
}

}  // namespace window
}  // namespace b200
