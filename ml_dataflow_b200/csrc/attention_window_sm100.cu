// Windowed attention with sinks on the tensor cores, head sizes 64 and 128.
//
// Forward. A work unit is a pair of 128-row query tiles that read the same keys: two query heads of one key/value head over
// the same rows (or, where the group is odd, two neighbouring tiles of one head). Key blocks of 128 that no row of the pair
// sees are never touched: the unit walks the blocks that hold sinks, then those of its window. A persistent CTA (one per SM)
// takes units in turn: while one unit's last products and its output are under way, the next one's queries and keys load.
//   warp 0     TMA loads: the query tiles, and K_0, K_1, V_0, K_2, V_1, ... through a ring, in the order they are used
//   warp 1     one thread issues the tcgen05 MMAs  S_g = Q_g K^T  and  O_g += P_g V  (fp32 accumulators in tensor memory)
//   warps 4-11 four per tile, a thread per query row: scores to registers at once - which frees the accumulator for the next
//              S, so that the tensor cores work while the exponentials are formed -, running maximum and sum,
//              P = exp2((S - m) scale log2 e) as bf16 through shared memory
// The maximum is raised, and O and the sum rescaled, only when a block's maximum exceeds it by more than 2^8.
// Rounding: scores, statistics and accumulators fp32; P to bf16 (relative to m) before it multiplies V, the tensor cores take
// no wider operand beside bf16 values; one rounding of the output.
// Rows of V that no query of the sequence sees (before its first window, past its end) are zeroed in shared memory, so that
// whatever they hold never meets the tensor cores; the scores of masked keys are dropped by a select.
//
// Every wait is bounded; one that runs out raises the status word that b200_attention_status reads, and the CTA leaves.
#include <cuda.h>
#include <math.h>
#include <stddef.h>

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
constexpr int FWD_THREADS = 384;
// A thread of the softmax holds a row of 128 scores: the launch gives 168 registers to each of the three warpgroups' threads, the
// loading and issuing one hands 96 of them on (72 + 216 + 216 = 3 * 168).
constexpr int REGS_CONTROL = 72, REGS_SOFTMAX = 216;
static_assert(REGS_CONTROL + 2 * REGS_SOFTMAX == 3 * 168, "a split of more registers than the launch has would wait for ever");
constexpr float LOG2E = 1.4426950408889634f;

enum { ST_Q_EMPTY = 51, ST_KV_EMPTY, ST_Q_FULL, ST_KV_FULL, ST_S_FREE, ST_P, ST_O_FREE, ST_S, ST_PV, ST_FIX };

struct FwdParams {
  CUtensorMap tmQ, tmK, tmV;  // [rows][heads * HD] bf16, boxes of 64 columns x 128 rows, 128-byte swizzle
  SeqTable seqs;
  __nv_bfloat16 *O;
  float *lse;  // [q_heads][total_q]
  int window, sinks, group, q_heads, total_q, pair_heads, units;
  float scale;
  int *status;
};

template <int HD>
struct FwdShape {
  static constexpr int Q_TILE = TILE * HD * 2, P_TILE = TILE * TILE * 2, KV_TILE = TILE * HD * 2;
  static constexpr int SLOTS = HD == 128 ? 3 : 6;
  struct Tail {
    uint64_t q_full[2], q_empty[2], kv_full[SLOTS], kv_empty[SLOTS], s_full[2], s_read[2], p_ready[2], pv_done[2], o_empty[2], fixed;
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
__device__ __forceinline__ Span span_of(const SeqTable &t, int s) {
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
};
__device__ __forceinline__ Tile tile_of(const Span &sp, int window, int h, int row) {
  Tile t;
  t.h = h;
  t.row = row;
  t.lo = max(0, row + sp.shift - window + 1) / TILE;
  t.hi = (min(row + TILE, sp.Tq) - 1 + sp.shift) / TILE;
  t.exists = row < sp.Tq;
  return t;
}
__device__ __forceinline__ Unit unit_of(const FwdParams &p, int unit) {
  Unit u;
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
  u.first = u.a.lo;
  u.n_sink = min((p.sinks + TILE - 1) / TILE, u.first);
  u.n = u.n_sink + (u.b.exists ? u.b.hi : u.a.hi) - u.first + 1;
  return u;
}

// The MMA descriptors of a tile's 16-column steps differ from its first one by a constant in the address field; formed anew from
// `addr` where they are used (the compiler would else hold those of every tile in registers for the whole kernel).
__device__ __forceinline__ uint64_t tile_desc(uint32_t addr, uint32_t lbo) {
  asm volatile("" : "+r"(addr));
  return ptx::make_smem_desc(addr, lbo, 1024);
}
__device__ __forceinline__ uint64_t desc_at(uint64_t desc, uint32_t bytes) { return desc + (bytes >> 4); }

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

template <int HD>
__global__ void __launch_bounds__(FWD_THREADS, 1) window_fwd_kernel(const __grid_constant__ FwdParams p) {
  using Sh = FwdShape<HD>;
  constexpr int KSL = HD / 64, SLOTS = Sh::SLOTS;
  constexpr uint32_t TMEM_COLS = 512, COL_O = 256;  // S_0, S_1 (128 columns each), then O_0, O_1 (HD each)
  extern __shared__ unsigned char window_smem[];
  unsigned char *smem = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(window_smem) + 1023) & ~static_cast<uintptr_t>(1023));
  unsigned char *sQ = smem, *sP = sQ + 2 * Sh::Q_TILE, *sKV = sP + 2 * Sh::P_TILE;
  auto *st = reinterpret_cast<typename Sh::Tail *>(sKV + SLOTS * Sh::KV_TILE);
  volatile int *abort_flag = &st->abort_flag;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  auto bar = [&](uint64_t *b) { return ptx::smem_u32(b); };
  auto wait = [&](uint64_t *b, uint32_t par, int code) { return ptx::mbar_wait<false>(bar(b), par & 1u, abort_flag, p.status, code); };

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
    for (int s = 0; s < SLOTS; s++) {
      ptx::mbar_init(bar(&st->kv_full[s]), 1);
      ptx::mbar_init(bar(&st->kv_empty[s]), 1);
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
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem_base = st->tmem_base;

  if (warp < 4) {
    ptx::reg_dec<REGS_CONTROL>();
    if (warp == 0) {
      // ================= loads: the whole warp walks, one lane issues =================
      int n = 0;
      uint32_t uq[2] = {0, 0}, fixes = 0;
      bool ok = true;
      auto waitw = [&](uint64_t *b, uint32_t par, int code) { return __all_sync(0xffffffffu, wait(b, par, code)) != 0; };
      for (int unit = blockIdx.x; ok && unit < p.units; unit += gridDim.x) {
        const Unit u = unit_of(p, unit);
        const int kvh = u.a.h / p.group;
#pragma unroll
        for (int g = 0; g < 2; g++) {
          const Tile &x = g ? u.b : u.a;
          if (!ok || !x.exists) continue;
          ok = waitw(&st->q_empty[g], uq[g] + 1, ST_Q_EMPTY);
          if (ok && lane == 0) {
            ptx::mbar_arrive_expect_tx(bar(&st->q_full[g]), (uint32_t)Sh::Q_TILE);
            for (int s = 0; s < KSL; s++)
              ptx::tma_load_2d(ptx::smem_u32(sQ + g * Sh::Q_TILE + s * SLAB), &p.tmQ, bar(&st->q_full[g]), x.h * HD + s * 64,
                               u.sp.q_off + x.row);
          }
          uq[g]++;
        }
        auto load = [&](const CUtensorMap *m, int kb, bool fix) {
          const int slot = n % SLOTS;
          ok = waitw(&st->kv_empty[slot], (uint32_t)(n / SLOTS) + 1, ST_KV_EMPTY);
          n++;
          if (!ok) return;
          const uint32_t tile = ptx::smem_u32(sKV + slot * Sh::KV_TILE), full = fix ? bar(&st->fixed) : bar(&st->kv_full[slot]);
          if (lane == 0) {
            ptx::mbar_arrive_expect_tx(full, (uint32_t)Sh::KV_TILE);
            for (int s = 0; s < KSL; s++) ptx::tma_load_2d(tile + s * SLAB, m, full, kvh * HD + s * 64, u.sp.k_off + kb * TILE);
          }
          if (!fix) return;
          ok = waitw(&st->fixed, fixes++, ST_FIX);
          if (!ok) return;
          zero_dead<HD>(tile, u.sp, kb, p.window, p.sinks, lane);
          ptx::fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(bar(&st->kv_full[slot]));
        };
        for (int i = 0; ok && i <= u.n; i++) {
          if (i < u.n) load(&p.tmK, u.block(i), false);
          if (ok && i > 0) load(&p.tmV, u.block(i - 1), has_dead(u.sp, u.block(i - 1), p.window, p.sinks));
        }
      }
      __syncwarp();
    } else if (warp == 1) {
      // ================= MMA issue =================
      if (lane == 0) {
        const uint32_t idesc_s = ptx::make_idesc_bf16(TILE, TILE, 0, 0);
        const uint32_t idesc_pv = ptx::make_idesc_bf16(TILE, HD, 0, 1);  // V is read with its head dimension contiguous
        const uint32_t q_base = ptx::smem_u32(sQ), p_base = ptx::smem_u32(sP), kv_base = ptx::smem_u32(sKV);
        int n = 0;
        uint32_t uq[2] = {0, 0}, ts[2] = {0, 0}, tp[2] = {0, 0};  // units, S products and P V products of either tile so far
        bool ok = true;
        for (int unit = blockIdx.x; ok && unit < p.units; unit += gridDim.x) {
          const Unit u = unit_of(p, unit);
          bool begun_s[2] = {false, false}, begun_o[2] = {false, false};
          for (int i = 0; ok && i <= u.n; i++) {
            if (i < u.n) {
              const int slot = n % SLOTS, kb = u.block(i);
              if (!(ok = wait(&st->kv_full[slot], (uint32_t)(n / SLOTS), ST_KV_FULL))) break;
              n++;
#pragma unroll
              for (int g = 0; g < 2; g++) {
                const Tile &x = g ? u.b : u.a;
                if (!ok || !x.active(kb, p.sinks)) continue;
                if (!begun_s[g]) {
                  begun_s[g] = true;
                  if (!(ok = wait(&st->q_full[g], uq[g], ST_Q_FULL))) continue;
                }
                if (ts[g] > 0 && !(ok = wait(&st->s_read[g], ts[g] - 1, ST_S_FREE))) continue;
                ptx::tc_fence_after();
                const uint64_t qd = tile_desc(q_base + g * Sh::Q_TILE, 0), kd = tile_desc(kv_base + slot * Sh::KV_TILE, 0);
#pragma unroll
                for (int k16 = 0; k16 < HD / 16; k16++) {
                  const uint32_t off = (uint32_t)((k16 >> 2) * SLAB + (k16 & 3) * 32);
                  ptx::umma_bf16(tmem_base + (uint32_t)(g * TILE), desc_at(qd, off), desc_at(kd, off), idesc_s, k16 > 0);
                }
                ptx::umma_commit(bar(&st->s_full[g]));
                if (kb == x.hi) ptx::umma_commit(bar(&st->q_empty[g]));
                ts[g]++;
              }
              if (!ok) break;
              ptx::umma_commit(bar(&st->kv_empty[slot]));
            }
            if (i > 0) {
              const int slot = n % SLOTS, kb = u.block(i - 1);
              if (!(ok = wait(&st->kv_full[slot], (uint32_t)(n / SLOTS), ST_KV_FULL))) break;
              n++;
#pragma unroll
              for (int g = 0; g < 2; g++) {
                if (!ok || !(g ? u.b : u.a).active(kb, p.sinks)) continue;
                // P of this step is in shared memory, the group has rescaled O if its maxima grew - and read the last unit's O
                if (!(ok = wait(&st->p_ready[g], tp[g], ST_P))) continue;
                if (!begun_o[g] && uq[g] > 0 && !(ok = wait(&st->o_empty[g], uq[g] - 1, ST_O_FREE))) continue;
                ptx::tc_fence_after();
                const uint64_t pd = tile_desc(p_base + g * Sh::P_TILE, 0), vd = tile_desc(kv_base + slot * Sh::KV_TILE, SLAB);
#pragma unroll
                for (int k16 = 0; k16 < TILE / 16; k16++)
                  ptx::umma_bf16(tmem_base + COL_O + (uint32_t)(g * HD), desc_at(pd, (uint32_t)((k16 >> 2) * SLAB + (k16 & 3) * 32)),
                                 desc_at(vd, (uint32_t)(k16 * 2048)), idesc_pv, begun_o[g] || k16 > 0);
                begun_o[g] = true;
                ptx::umma_commit(bar(&st->pv_done[g]));
                tp[g]++;
              }
              if (!ok) break;
              ptx::umma_commit(bar(&st->kv_empty[slot]));
            }
          }
          uq[0] += u.a.exists;
          uq[1] += u.b.exists;
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
    for (int unit = blockIdx.x; unit < p.units; unit += gridDim.x) {
      const Unit u = unit_of(p, unit);
      const Tile x = g ? u.b : u.a;
      if (!x.exists) continue;
      const int row = x.row + trow, pos = row + u.sp.shift;
      const int tile_pos = x.row + u.sp.shift, last_pos = min(tile_pos + TILE, u.sp.Tk) - 1;
      const int hi = min(pos, u.sp.Tk - 1), lo = pos - p.window + 1;  // the keys this row sees, besides the sinks
      float m = -INFINITY, l = 0.0f;
      bool first = true;
      for (int i = 0; i < u.n; i++) {
        const int kb = u.block(i);
        if (!x.active(kb, p.sinks)) continue;
        if (!wait(&st->s_full[g], t, ST_S)) goto teardown;
        ptx::tc_fence_after();
        uint32_t s[TILE];
#pragma unroll
        for (int q = 0; q < 4; q++) ptx::tmem_ld32(s_addr + q * 32, s + q * 32);
        ptx::tmem_ld_wait();
        ptx::tc_fence_before();
        ptx::mbar_arrive(bar(&st->s_read[g]));
        const int base = kb * TILE;
        // every row of the tile sees every key of the block: the window reaches back from the last row to the block's start
        const bool whole = base + TILE - 1 <= tile_pos && (base >= last_pos - p.window + 1 || base + TILE <= p.sinks);
        if (!whole) {
#pragma unroll
          for (int j = 0; j < TILE; j++) {
            const int key = base + j;
            if (!(key <= hi && (key >= lo || key < p.sinks))) s[j] = 0xff800000u;  // -infinity
          }
        }
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int j = 0; j < TILE; j++) mx4[j & 3] = fmaxf(mx4[j & 3], __uint_as_float(s[j]));
        const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
        if (first) {
          m = mx;
        } else {
          const bool grow = (mx - m) * c > 8.0f;
          if (__any_sync(0xffffffffu, grow)) {  // tensor-memory accesses are warp-wide: every lane takes part
            const float m_new = grow ? mx : m;
            // 1 for the lanes that keep their offset; a row that had seen nothing has nothing to rescale
            const float alpha = (m == -INFINITY || !grow) ? 1.0f : ex2((m - m_new) * c);
            if (!wait(&st->pv_done[g], t - 1, ST_PV)) goto teardown;
            ptx::tc_fence_after();
#pragma unroll
            for (int q = 0; q < HD / 32; q++) {
              uint32_t r[32];
              ptx::tmem_ld32(o_addr + q * 32, r);
              ptx::tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 32; j++) r[j] = __float_as_uint(__uint_as_float(r[j]) * alpha);
              ptx::tmem_st32(o_addr + q * 32, r);
            }
            ptx::tmem_st_wait();
            l *= alpha;
            m = m_new;
          }
        }
        // a row that has seen no key yet keeps m = -inf: its probabilities are exp2(-inf) = 0 against a zero offset
        const float mc = (m == -INFINITY) ? 0.0f : m * c;
        float sum4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < TILE; j++) {
          const float e = ex2(fmaf(__uint_as_float(s[j]), c, -mc));
          sum4[j & 3] += e;
          s[j] = __float_as_uint(e);
        }
        l += (sum4[0] + sum4[1]) + (sum4[2] + sum4[3]);
        // the step before has read P
        if (t > 0 && !wait(&st->pv_done[g], t - 1, ST_PV)) goto teardown;
#pragma unroll
        for (int q = 0; q < 16; q++) {
          // keys 8 q .. 8 q + 7 of this row: slab q / 8, 16-byte chunk q % 8, swizzled with the row
          uint4 v;
          v.x = pack_bf16(__uint_as_float(s[q * 8 + 0]), __uint_as_float(s[q * 8 + 1]));
          v.y = pack_bf16(__uint_as_float(s[q * 8 + 2]), __uint_as_float(s[q * 8 + 3]));
          v.z = pack_bf16(__uint_as_float(s[q * 8 + 4]), __uint_as_float(s[q * 8 + 5]));
          v.w = pack_bf16(__uint_as_float(s[q * 8 + 6]), __uint_as_float(s[q * 8 + 7]));
          sts128(p_addr + (uint32_t)((q >> 3) * SLAB + (((q & 7) ^ (trow & 7)) * 16)), v);
        }
        ptx::fence_proxy_async_smem();
        ptx::tc_fence_before();
        ptx::mbar_arrive(bar(&st->p_ready[g]));
        first = false;
        t++;
      }
      if (!wait(&st->pv_done[g], t - 1, ST_PV)) goto teardown;
      ptx::tc_fence_after();
      uint32_t r[HD];
#pragma unroll
      for (int q = 0; q < HD / 32; q++) ptx::tmem_ld32(o_addr + q * 32, r + q * 32);
      ptx::tmem_ld_wait();
      ptx::tc_fence_before();
      ptx::mbar_arrive(bar(&st->o_empty[g]));
      if (row < u.sp.Tq) {
        const float inv = 1.0f / l;
        uint4 *o = reinterpret_cast<uint4 *>(p.O + ((int64_t)(u.sp.q_off + row) * p.q_heads + x.h) * HD);
#pragma unroll
        for (int q = 0; q < HD / 8; q++) {
          float v[8];
#pragma unroll
          for (int j = 0; j < 8; j++) v[j] = __uint_as_float(r[q * 8 + j]) * inv;
          o[q] = pack8(v);
        }
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
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem_base, TMEM_COLS);
  }
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

template <int HD>
int launch_fwd(window::FwdParams &p, const Device &d, cudaStream_t s) {
  static bool done[MAX_DEVICES];
  constexpr size_t smem = window::FwdShape<HD>::smem;
  if (allow_smem(window::window_fwd_kernel<HD>, smem, &done[d.dev])) return -1;
  window::window_fwd_kernel<HD><<<p.units < d.sms ? p.units : d.sms, window::FWD_THREADS, smem, s>>>(p);
  B200_CHECK_LAUNCH("attention_window_fwd");
  return 0;
}

}  // namespace

namespace b200 {
namespace window {

int sm100_fwd(const Call &c) {
  FwdParams p;
  Device d;
  if (current_device(&d)) return -1;
  const uint64_t Dq = (uint64_t)c.q_heads * c.head_dim, Dk = (uint64_t)c.kv_heads * c.head_dim;
  if (rows_map(&p.tmQ, c.q, (uint64_t)c.total_q, Dq) || rows_map(&p.tmK, c.k, (uint64_t)c.total_k, Dk) ||
      rows_map(&p.tmV, c.v, (uint64_t)c.total_k, Dk))
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
    p.units = next_sequences(p.seqs, &next, c, [&](int s) {
      const int tiles = (c.q_len[s] + TILE - 1) / TILE;
      return p.pair_heads ? tiles * (c.q_heads / 2) : (tiles + 1) / 2 * c.q_heads;
    });
    if (p.units == 0) continue;
    if (c.head_dim == 128 ? launch_fwd<128>(p, d, c.stream) : launch_fwd<64>(p, d, c.stream)) return -1;
  }
  return 0;
}

}  // namespace window
}  // namespace b200
