// Windowed attention forward for sequences with few queries (a new token or two of a long text), head sizes 64 and 128.
//
// Such a call reads every visible key and value once and computes next to nothing: memory bounds it, and, in small batches, latency. The
// query heads of a group are the rows of one 16-row tile, so K and V are read once for all of them. A unit is such a tile of one
// sequence and key/value head; its visible keys - the sinks, then the window - are numbered through and cut into blocks of 64, which the
// CTAs of a cluster take in turn. There are as many CTAs per unit (1, 2, 4 or 8) as the device seats clusters of at once (32 sequences of up
// to 4100 visible keys, 128 units: 2 CTAs each 37 us, 4 each 44 to 49; head size 128, 4100 keys: 33 units are all seated with 8, 15 us, 4 each take
// 20; 34 units are not, 23 us against 20; 71 units with 4 and with 2 28 and 35, 72 units 39 and 34); they join their partial sums through each other's shared memory, so
// that a call is one launch and needs no workspace.
//
// A CTA: 4 warps, 16 keys of a block each, three blocks of K and V in flight (cp.async, 96 KB at head size 128, two CTAs per SM). Products
// with m16n8k16 warp-level MMAs: a 128-row tcgen05 tile would be seven eighths empty and wait for tensor memory first. Online
// softmax per warp; rounding as in the tiles' kernel (P to bf16 once, everything else fp32, one rounding of the output).
// Rows of a block that no query of the unit sees are not read: their place is filled with zeros.
// Measured at 16 query heads on 4 of 128, window 4096: 128 sequences of 4100 visible keys (1.07 GB) at 6.1 TB/s; 32 of 2 to 4100 (179 MB)
// 37 us, 4.9 TB/s, where the longest sequences' CTAs run on alone.
#include <math.h>

#include "attention_sm100.cuh"
#include "attention_window.cuh"
#include "common.cuh"
#include "sm100_ptx.cuh"

namespace b200 {
namespace window {

using fa::ex2;

constexpr int FEW_THREADS = 128, FEW_WARPS = 4;
constexpr int ROWS = 16;        // query rows of a unit: tokens x heads of the group
constexpr int KEYS = 64;        // keys of a block
constexpr int STAGES = 3;
constexpr int MAX_CLUSTER = 8;
constexpr int FEW_SEQS = 192;   // sequences of a launch
constexpr float LOG2E = 1.4426950408889634f;

struct FewParams {
  int n, q_off[FEW_SEQS], Tq[FEW_SEQS], k_off[FEW_SEQS], Tk[FEW_SEQS], first[FEW_SEQS + 1];  // units through the sequences
  const __nv_bfloat16 *q, *k, *v;
  __nv_bfloat16 *o;
  float *lse;  // [q_heads][total_q]
  int window, sinks, group, q_heads, kv_heads, total_q, cluster;
  float scale;
};

__device__ __forceinline__ void cp16(uint32_t dst, const void *src, bool on) {
  const int bytes = on ? 16 : 0;  // 0: the place is filled with zeros and src is not read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t *r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_t(uint32_t addr, uint32_t *r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// D += A B: rows x 16 by 16 x 8 columns
__device__ __forceinline__ void mma16816(float *d, const uint32_t *a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float4 ld_cluster(uint32_t addr, uint32_t rank) {
  float4 v;
  asm volatile(
      "{\n"
      ".reg .b32 ra;\n"
      "mapa.shared::cluster.u32 ra, %4, %5;\n"
      "ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [ra];\n"
      "}\n"
      : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
      : "r"(addr), "r"(rank)
      : "memory");
  return v;
}
__device__ __forceinline__ float ld_cluster1(uint32_t addr, uint32_t rank) {
  float v;
  asm volatile(
      "{\n"
      ".reg .b32 ra;\n"
      "mapa.shared::cluster.u32 ra, %1, %2;\n"
      "ld.shared::cluster.f32 %0, [ra];\n"
      "}\n"
      : "=f"(v)
      : "r"(addr), "r"(rank)
      : "memory");
  return v;
}

template <int HD>
struct FewShape {
  static constexpr int ROW = HD * 2, TILE = KEYS * ROW, STAGE = 2 * TILE;  // bytes
  static constexpr int JOIN = FEW_WARPS * ROWS * HD * 4;                   // the warps' outputs, over the stages
  // the CTA's output, row maxima and sums, and the warps' maxima and sums
  static constexpr int TAIL = ROWS * HD * 4 + 2 * ROWS * 4 + FEW_WARPS * 2 * ROWS * 4;
  static constexpr size_t smem = STAGES * STAGE + TAIL;
  static_assert(JOIN <= STAGES * STAGE, "the outputs lie over the stages");
};

// weight of a partial sum taken against maximum m when the joint maximum is M (in scores; c scales them to powers of two)
__device__ __forceinline__ float weight_of(float m, float M, float c) { return m == -INFINITY ? 0.0f : ex2((m - M) * c); }

template <int HD>
__global__ void __launch_bounds__(FEW_THREADS, 2) window_few_kernel(const __grid_constant__ FewParams p) {
  using Sh = FewShape<HD>;
  constexpr int CHUNKS = HD / 8;  // 16-byte pieces of a row
  extern __shared__ __align__(128) unsigned char few_smem[];
  float *s_out = reinterpret_cast<float *>(few_smem + STAGES * Sh::STAGE), *s_m = s_out + ROWS * HD, *s_l = s_m + ROWS, *s_wm = s_l + ROWS,
        *s_wl = s_wm + FEW_WARPS * ROWS;
  const uint32_t base = ptx::smem_u32(few_smem);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q4 = lane & 3;
  const int unit = blockIdx.x / p.cluster, rank = blockIdx.x % p.cluster;
  int lo_s = 0, hi_s = p.n;  // the sequence whose units hold this one
  while (hi_s - lo_s > 1) {
    const int mid = (lo_s + hi_s) >> 1;
    if (unit >= p.first[mid]) lo_s = mid;
    else hi_s = mid;
  }
  const int s = lo_s, rel = unit - p.first[s], kvh = rel % p.kv_heads, row0 = rel / p.kv_heads * ROWS;
  const int q_off = p.q_off[s], Tq = p.Tq[s], k_off = p.k_off[s], Tk = p.Tk[s], rows = Tq * p.group;
  // row r of the unit: token (row0 + r) / group, head kvh * group + (row0 + r) % group
  const int first_pos = row0 / p.group + Tk - Tq, last_pos = (min(row0 + ROWS, rows) - 1) / p.group + Tk - Tq;
  const int lo = max(0, first_pos - p.window + 1), sinks = min(p.sinks, lo), count = sinks + last_pos - lo + 1;
  const int blocks = (count + KEYS - 1) / KEYS, mine = blocks > rank ? (blocks - rank + p.cluster - 1) / p.cluster : 0;
  auto key_of = [&](int i) { return i < sinks ? i : lo + i - sinks; };

  const int64_t ldk = (int64_t)p.kv_heads * HD;
  const __nv_bfloat16 *K = p.k + (int64_t)k_off * ldk + (int64_t)kvh * HD, *V = p.v + (int64_t)k_off * ldk + (int64_t)kvh * HD;
  // a block's rows in shared memory: 16-byte pieces, swizzled with the row so that the eight rows of a matrix fall on different banks
  auto place = [](int row, int chunk) { return (uint32_t)(row * Sh::ROW + ((chunk & ~7) | ((chunk ^ row) & 7)) * 16); };
  auto fetch = [&](int b, int stage) {
    constexpr int STEP = FEW_THREADS / CHUNKS;  // rows at a time
    const int chunk = tid % CHUNKS, r0 = tid / CHUNKS;
    const uint32_t dst = base + stage * Sh::STAGE;
#pragma unroll
    for (int r = r0; r < KEYS; r += STEP) {
      const int i = b * KEYS + r;
      const bool on = i < count;
      const int64_t at = (on ? key_of(i) : 0) * ldk + chunk * 8;
      cp16(dst + place(r, chunk), K + at, on);
      cp16(dst + Sh::TILE + place(r, chunk), V + at, on);
    }
  };
  pdl_release();
  pdl_wait();
#pragma unroll
  for (int i = 0; i < STAGES - 1; i++) {
    if (i < mine) fetch(rank + i * p.cluster, i);
    cp_commit();
  }

  // Q: this thread's elements of the A operand, rows g and g + 8
  uint32_t qa[HD / 16][4];
  int pos[2];
  bool on[2];
  int64_t at[2];
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const int r = row0 + g + 8 * h;
    on[h] = r < rows;
    const int tok = on[h] ? r / p.group : 0, head = kvh * p.group + (on[h] ? r - tok * p.group : 0);
    pos[h] = on[h] ? tok + Tk - Tq : -1;  // a row that is not there sees nothing
    at[h] = ((int64_t)(q_off + tok) * p.q_heads + head) * HD;
#pragma unroll
    for (int k = 0; k < HD / 16; k++)
#pragma unroll
      for (int e = 0; e < 2; e++)
        qa[k][h + 2 * e] = on[h] ? *reinterpret_cast<const uint32_t *>(p.q + at[h] + k * 16 + e * 8 + q4 * 2) : 0u;
  }

  const float c = p.scale * LOG2E;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
  float o[HD / 8][4];
#pragma unroll
  for (int d = 0; d < HD / 8; d++) o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0.0f;

  for (int it = 0; it < mine; it++) {
    cp_wait<STAGES - 2>();
    __syncthreads();  // this block has landed for all, and all have left the stage that is filled next
    if (it + STAGES - 1 < mine) fetch(rank + (it + STAGES - 1) * p.cluster, (it + STAGES - 1) % STAGES);
    cp_commit();
    const uint32_t sK = base + (it % STAGES) * Sh::STAGE, sV = sK + Sh::TILE;
    const int wrow = warp * 16;  // this warp's keys of the block
    float sc[2][4] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
    for (int k = 0; k < HD / 16; k++) {
      uint32_t b[4];
      ldmatrix4(sK + place(wrow + (lane >> 4) * 8 + (lane & 7), 2 * k + ((lane >> 3) & 1)), b);
      mma16816(sc[0], qa[k], b[0], b[1]);
      mma16816(sc[1], qa[k], b[2], b[3]);
    }
    // masks, and the maximum over the four threads of a row
    const int i0 = (rank + it * p.cluster) * KEYS + wrow + q4 * 2;
    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int n = 0; n < 2; n++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int i = i0 + n * 8 + (e & 1), key = key_of(i), h = e >> 1;
        const bool seen = i < count && key <= pos[h] && (key > pos[h] - p.window || key < p.sinks);
        sc[n][e] = seen ? sc[n][e] : -INFINITY;
        mx[h] = fmaxf(mx[h], sc[n][e]);
      }
    float alpha[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
      mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
      mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
      mx[h] = fmaxf(mx[h], m[h]);
      alpha[h] = m[h] == mx[h] ? 1.0f : weight_of(m[h], mx[h], c);
      m[h] = mx[h];
      l[h] *= alpha[h];
    }
    if (__any_sync(0xffffffffu, alpha[0] != 1.0f || alpha[1] != 1.0f)) {
#pragma unroll
      for (int d = 0; d < HD / 8; d++) {
        o[d][0] *= alpha[0];
        o[d][1] *= alpha[0];
        o[d][2] *= alpha[1];
        o[d][3] *= alpha[1];
      }
    }
    uint32_t pa[4];
#pragma unroll
    for (int n = 0; n < 2; n++)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        // against a maximum of -infinity nothing has been seen: exp2(-inf) = 0
        const float mc = m[h] == -INFINITY ? 0.0f : m[h] * c;
        const float e0 = ex2(fmaf(sc[n][2 * h], c, -mc)), e1 = ex2(fmaf(sc[n][2 * h + 1], c, -mc));
        l[h] += e0 + e1;
        pa[n * 2 + h] = pack_bf16(e0, e1);
      }
#pragma unroll
    for (int d = 0; d < HD / 16; d++) {
      uint32_t b[4];
      ldmatrix4_t(sV + place(wrow + ((lane >> 3) & 1) * 8 + (lane & 7), 2 * d + (lane >> 4)), b);
      mma16816(o[2 * d], pa, b[0], b[1]);
      mma16816(o[2 * d + 1], pa, b[2], b[3]);
    }
  }
  cp_wait<0>();
  __syncthreads();
  // the warps' sums, joined in warp order
  float *s_o = reinterpret_cast<float *>(few_smem);  // [warp][row][HD]
#pragma unroll
  for (int h = 0; h < 2; h++) {
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    const int r = g + 8 * h;
    if (q4 == 0) {
      s_wm[warp * ROWS + r] = m[h];
      s_wl[warp * ROWS + r] = l[h];
    }
#pragma unroll
    for (int d = 0; d < HD / 8; d++)
      *reinterpret_cast<float2 *>(s_o + (warp * ROWS + r) * HD + d * 8 + q4 * 2) = make_float2(o[d][2 * h], o[d][2 * h + 1]);
  }
  __syncthreads();
  for (int i = tid; i < ROWS * HD / 4; i += FEW_THREADS) {
    const int r = i / (HD / 4), d = i % (HD / 4) * 4;
    float M = -INFINITY, L = 0.0f;
#pragma unroll
    for (int w = 0; w < FEW_WARPS; w++) M = fmaxf(M, s_wm[w * ROWS + r]);
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < FEW_WARPS; w++) {
      const float f = weight_of(s_wm[w * ROWS + r], M, c);
      const float4 v = *reinterpret_cast<const float4 *>(s_o + (w * ROWS + r) * HD + d);
      sum.x = fmaf(f, v.x, sum.x);
      sum.y = fmaf(f, v.y, sum.y);
      sum.z = fmaf(f, v.z, sum.z);
      sum.w = fmaf(f, v.w, sum.w);
      L = fmaf(f, s_wl[w * ROWS + r], L);
    }
    *reinterpret_cast<float4 *>(s_out + r * HD + d) = sum;
    if (d == 0) {
      s_m[r] = M;
      s_l[r] = L;
    }
  }
  // the CTAs' sums, joined in the order of their ranks; each writes its share of the unit's output
  if (p.cluster > 1) ptx::cluster_sync_all();
  else __syncthreads();
  const uint32_t a_out = ptx::smem_u32(s_out), a_m = ptx::smem_u32(s_m), a_l = ptx::smem_u32(s_l);
  for (int i = rank * FEW_THREADS + tid; i < ROWS * HD / 4; i += p.cluster * FEW_THREADS) {
    const int r = i / (HD / 4), d = i % (HD / 4) * 4, rr = row0 + r;
    if (rr >= rows) continue;
    float M = -INFINITY, L = 0.0f;
    for (int k = 0; k < p.cluster; k++) M = fmaxf(M, ld_cluster1(a_m + r * 4, k));
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int k = 0; k < p.cluster; k++) {
      const float f = weight_of(ld_cluster1(a_m + r * 4, k), M, c);
      const float4 v = ld_cluster(a_out + (r * HD + d) * 4, k);
      sum.x = fmaf(f, v.x, sum.x);
      sum.y = fmaf(f, v.y, sum.y);
      sum.z = fmaf(f, v.z, sum.z);
      sum.w = fmaf(f, v.w, sum.w);
      L = fmaf(f, ld_cluster1(a_l + r * 4, k), L);
    }
    const int tok = rr / p.group, head = kvh * p.group + rr - tok * p.group;
    const float inv = 1.0f / L;
    *reinterpret_cast<uint2 *>(p.o + ((int64_t)(q_off + tok) * p.q_heads + head) * HD + d) =
        make_uint2(pack_bf16(sum.x * inv, sum.y * inv), pack_bf16(sum.z * inv, sum.w * inv));
    if (d == 0) p.lse[(int64_t)head * p.total_q + q_off + tok] = M * p.scale + logf(L);
  }
  if (p.cluster > 1) ptx::cluster_sync_all();  // nobody leaves while another reads its shared memory
}

}  // namespace window
}  // namespace b200

using namespace b200;

namespace {

template <int HD>
int launch_few(window::FewParams &p, int units, int64_t most, cudaStream_t s) {
  static bool done[MAX_DEVICES];
  static int known[MAX_DEVICES][window::MAX_CLUSTER + 1];
  int dev = -1;
  B200_CUDA(cudaGetDevice(&dev));
  B200_REQUIRE(dev >= 0 && dev < MAX_DEVICES, "attention_window: device ordinal %d is out of range", dev);
  constexpr size_t smem = window::FewShape<HD>::smem;
  if (!done[dev]) {
    B200_CUDA(cudaFuncSetAttribute(window::window_few_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    done[dev] = true;
  }
  p.cluster = 1;
  while (p.cluster < window::MAX_CLUSTER && (int64_t)p.cluster * window::KEYS < most &&
         units <= window::cluster_seats(window::window_few_kernel<HD>, window::FEW_THREADS, smem, 2 * p.cluster, &known[dev][2 * p.cluster]))
    p.cluster *= 2;
  B200_CUDA(b200_launch_overlapped(window::window_few_kernel<HD>, dim3((unsigned)(units * p.cluster)), dim3(window::FEW_THREADS), smem, s,
                                   (unsigned)p.cluster, p));
  B200_CHECK_LAUNCH("attention_window_fwd (few queries)");
  return 0;
}

}  // namespace

namespace b200 {
namespace window {

// Rows of a sequence in one group; up to two of the 16-row tiles the keys are read through this form, beyond through the 128-row tiles.
bool is_few(const Call &c, int s) { return sm100_supported(c.head_dim) && (int64_t)c.q_len[s] * (c.q_heads / c.kv_heads) <= 2 * ROWS; }

int few_fwd(const Call &c) {
  FewParams p;
  p.q = c.q;
  p.k = c.k;
  p.v = c.v;
  p.o = c.out;
  p.lse = c.lse;
  p.window = c.window;
  p.sinks = c.sinks;
  p.group = c.q_heads / c.kv_heads;
  p.q_heads = c.q_heads;
  p.kv_heads = c.kv_heads;
  p.total_q = c.total_q;
  p.scale = c.scale;
  for (int s = 0; s < c.num_seqs;) {
    int64_t most = 0;  // visible keys of a sequence, at most
    p.n = 0;
    p.first[0] = 0;
    for (; s < c.num_seqs && p.n < FEW_SEQS; s++) {
      if (c.q_len[s] == 0 || !is_few(c, s)) continue;
      p.q_off[p.n] = c.q_off[s];
      p.Tq[p.n] = c.q_len[s];
      p.k_off[p.n] = c.k_off[s];
      p.Tk[p.n] = c.k_len[s];
      p.first[p.n + 1] = p.first[p.n] + (c.q_len[s] * p.group + ROWS - 1) / ROWS * c.kv_heads;
      p.n++;
      const int64_t seen = (int64_t)c.window + c.q_len[s] + c.sinks;
      most = seen < c.k_len[s] ? (seen > most ? seen : most) : (c.k_len[s] > most ? c.k_len[s] : most);
    }
    if (p.n == 0) return 0;
    const int units = p.first[p.n];
    if (c.head_dim == 128 ? launch_few<128>(p, units, most, c.stream) : launch_few<64>(p, units, most, c.stream)) return -1;
  }
  return 0;
}

}  // namespace window
}  // namespace b200
