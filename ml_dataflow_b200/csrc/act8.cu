// SwiGLU activations held in 8 bits between the forward and the backward. x1 and x3 (the two products the SwiGLU joins)
// are the largest tensors a MoE block keeps; here each block of 32 columns of a row is held as 32 e4m3 codes and one
// power of two, 33 bytes instead of 64.
//
//   unit e   the smallest power of two with max |x| <= 448 * 2^e over the block (448 = the largest e4m3 number)
//   code     x * 2^-e rounded to nearest e4m3, ties to even: at most half a step of four significant bits off, 2^-4
//            relative for values within 2^-14 of the block's largest, 2^-10 of the unit below that
//   value    code * 2^e, exact in bf16: a power of two loses no bits, and e4m3 has fewer of them than bf16. For the same
//            reason the codes do not depend on the order or the precision of any sum: two runs hold the same bytes.
// At the largest unit, 2^120, 256 * 2^e would leave bf16: there values above 240 * 2^e are held as that.
// e is at least -124, so that the smallest step, 2^(e - 9), is still a bf16 number. An infinity or a NaN is held as NaN
// and takes no part in the maximum: the other values of its block keep their precision.
//
// All three kernels touch every byte once. A thread takes eight columns (16 bytes of bf16, 8 of codes), four neighbouring lanes
// share a scale block, and the maximum costs two shuffles; two groups of eight per thread are in flight. What bounds them besides
// memory is the number of instructions: hence arithmetic on pairs, the special-function units' reciprocal in the sigmoid (2^-22
// relative, far below the outputs' 2^-9), special values looked for once per group, and no index divisions where the columns are whole
// scale blocks. Measured at 65536 x 1408, 744 MB a call: h and the codes 126 us (5.9 TB/s), x1, x3 and h restored 117 us (6.4), the
// backward's two gradients 116 us (6.4); a plain copy reaches 6.5.
#include <cuda_fp16.h>

#include "common.cuh"
#include "../../include/b200_moe.h"

namespace b200 {
namespace act8 {

constexpr int THREADS = 256;
constexpr int UNROLL = 2;

// Where a group of eight columns lives. Rows are padded to whole scale blocks of four groups, so that the lanes of a
// block stay together; the groups past the row's end only take part in the shuffles.
struct Place {
  int64_t vec;    // index of the group in a [rows][cols / 8] array
  int64_t block;  // index of its scale in a [rows][scale blocks] array
  bool on;
};
struct Shape {
  int64_t padded;  // rows * padded groups per row
  int vecs, padded_vecs, blocks;
};
// The groups of one thread, `at` past the block's first group `base`. WHOLE: the columns are whole scale blocks, nothing is padded.
template <bool WHOLE>
struct Places {
  int64_t base, row;
  int col;
  __device__ __forceinline__ Places(const Shape &s, int64_t first) : base(first) {
    if (!WHOLE) {
      row = first / s.padded_vecs;
      col = (int)(first - row * s.padded_vecs);
    }
  }
  __device__ __forceinline__ Place operator()(const Shape &s, int at) const {
    Place p;
    if (WHOLE) {
      p.vec = base + at;
      p.block = p.vec >> 2;
      p.on = p.vec < s.padded;
    } else {
      const int c = col + at, rows = c / s.padded_vecs, cc = c - rows * s.padded_vecs;
      p.vec = (row + rows) * s.vecs + cc;
      p.block = (row + rows) * s.blocks + (cc >> 2);
      p.on = base + at < s.padded && cc < s.vecs;
    }
    return p;
  }
};

// bypasses L1; not a read-only load, because h may be written over x1 or x3
__device__ __forceinline__ uint4 ld_once(const uint4 *p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}

// exponent of the block's unit, biased by 127, from the bf16 bits of its largest finite magnitude
__device__ __forceinline__ int unit_of(uint32_t top) {
  const int e = (int)(top >> 7) - 135 + ((top & 0x7f) > 0x60);  // 448 = 1.75 * 2^8
  return max(e, -124) + 127;
}

// largest finite magnitude of eight bf16 numbers, as bf16 bits; `odd`: an infinity or NaN is among them
__device__ __forceinline__ uint32_t top_of(const uint4 &v, bool &odd) {
  const uint32_t a[4] = {v.x & 0x7fff7fffu, v.y & 0x7fff7fffu, v.z & 0x7fff7fffu, v.w & 0x7fff7fffu};
  const uint32_t m = __vmaxu2(__vmaxu2(a[0], a[1]), __vmaxu2(a[2], a[3]));
  uint32_t t = max(m & 0xffffu, m >> 16);
  odd = t >= 0x7f80u;
  if (odd) {  // take the others
    t = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint32_t lo = a[i] & 0xffffu, hi = a[i] >> 16;
      t = max(t, max(lo < 0x7f80u ? lo : 0u, hi < 0x7f80u ? hi : 0u));
    }
  }
  return t;
}

__device__ __forceinline__ uint32_t codes2(uint64_t v) {
  float lo, hi;
  unpack2(v, lo, hi);
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// the codes of one group from its pairs x; every lane of the warp takes part
__device__ __forceinline__ uint2 encode(const uint4 &v, const uint64_t *x, int &biased) {
  bool odd;
  uint32_t top = top_of(v, odd);
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
  biased = unit_of(top);
  const float inv = __int_as_float((254 - biased) << 23);  // 2^-e
  const uint64_t ii = pack2(inv, inv);
  uint64_t y[4];
#pragma unroll
  for (int i = 0; i < 4; i++) y[i] = mul2(x[i], ii);
  if (odd || biased == 120 + 127) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      float z[2];
      unpack2(y[i], z[0], z[1]);
#pragma unroll
      for (int e = 0; e < 2; e++) {
        if (fabsf(z[e]) == INFINITY) z[e] = __int_as_float(0x7fffffff);
        else if (biased == 120 + 127 && fabsf(z[e]) > 240.0f) z[e] = copysignf(240.0f, z[e]);  // NaN stays
      }
      y[i] = pack2(z[0], z[1]);
    }
  }
  return make_uint2(codes2(y[0]) | (codes2(y[1]) << 16), codes2(y[2]) | (codes2(y[3]) << 16));
}

__device__ __forceinline__ void decode(const uint2 &codes, int biased, uint64_t *x) {
  const float unit = __int_as_float(biased << 23);
  const uint64_t uu = pack2(unit, unit);
  const uint32_t w[2] = {codes.x, codes.y};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)(w[i >> 1] >> ((i & 1) * 16))));
    const float2 f = __half22float2(*reinterpret_cast<__half2 *>(&h));
    x[i] = mul2(pack2(f.x, f.y), uu);
  }
}

// of a pair: 1 / (1 + exp(-x))
__device__ __forceinline__ uint64_t sigmoid2(uint64_t x) {
  const float minus_log2e = -1.4426950408889634f;
  float a, b;
  unpack2(mul2(x, pack2(minus_log2e, minus_log2e)), a, b);
  asm("ex2.approx.f32 %0, %0;" : "+f"(a));
  asm("ex2.approx.f32 %0, %0;" : "+f"(b));
  unpack2(add2(pack2(a, b), pack2(1.0f, 1.0f)), a, b);
  asm("rcp.approx.f32 %0, %0;" : "+f"(a));
  asm("rcp.approx.f32 %0, %0;" : "+f"(b));
  return pack2(a, b);
}
__device__ __forceinline__ void widen(const uint4 &v, uint64_t *x) {
  x[0] = widen2(v.x);
  x[1] = widen2(v.y);
  x[2] = widen2(v.z);
  x[3] = widen2(v.w);
}
__device__ __forceinline__ uint4 round_all(const uint64_t *x) { return make_uint4(round2(x[0]), round2(x[1]), round2(x[2]), round2(x[3])); }
__device__ __forceinline__ void swiglu(const uint64_t *x, const uint64_t *y, uint64_t *h) {
#pragma unroll
  for (int i = 0; i < 4; i++) h[i] = mul2(mul2(x[i], sigmoid2(x[i])), y[i]);
}

// h = silu(x1) * x3 (when asked for) and the codes of x1 and x3
template <bool WHOLE>
__global__ void __launch_bounds__(THREADS) keep_kernel(Shape s, const uint4 *x1, const uint4 *x3, uint4 *out, uint2 *c1, uint8_t *e1,
                                                       uint2 *c3, uint8_t *e3) {
  pdl_release();
  pdl_wait();
  const int64_t step = (int64_t)gridDim.x * THREADS * UNROLL;
  for (int64_t base = (int64_t)blockIdx.x * THREADS * UNROLL; base < s.padded; base += step) {
    const Places<WHOLE> places(s, base);
    uint4 a[UNROLL], b[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; u++) {
      const Place p = places(s, u * THREADS + threadIdx.x);
      a[u] = b[u] = make_uint4(0, 0, 0, 0);
      if (p.on) {
        a[u] = ld_once(x1 + p.vec);
        b[u] = ld_once(x3 + p.vec);
      }
    }
#pragma unroll
    for (int u = 0; u < UNROLL; u++) {
      const Place p = places(s, u * THREADS + threadIdx.x);
      uint64_t x[4], y[4];
      int ex, ey;
      widen(a[u], x);
      widen(b[u], y);
      const uint2 cx = encode(a[u], x, ex), cy = encode(b[u], y, ey);
      if (!p.on) continue;
      c1[p.vec] = cx;
      c3[p.vec] = cy;
      if ((threadIdx.x & 3) == 0) {
        e1[p.block] = (uint8_t)ex;
        e3[p.block] = (uint8_t)ey;
      }
      if (out != nullptr) {
        swiglu(x, y, x);
        st_stream(out + p.vec, round_all(x));
      }
    }
  }
}

// the held x1 and x3 as bf16, and h again from them: each output when its pointer is not null
template <bool WHOLE>
__global__ void __launch_bounds__(THREADS) restore_kernel(Shape s, const uint2 *c1, const uint8_t *e1, const uint2 *c3, const uint8_t *e3,
                                                          uint4 *x1, uint4 *x3, uint4 *out) {
  pdl_release();
  pdl_wait();
  const int64_t step = (int64_t)gridDim.x * THREADS * UNROLL;
  for (int64_t base = (int64_t)blockIdx.x * THREADS * UNROLL; base < s.padded; base += step) {
    const Places<WHOLE> places(s, base);
    uint2 a[UNROLL], b[UNROLL];
    int ea[UNROLL], eb[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; u++) {
      const Place p = places(s, u * THREADS + threadIdx.x);
      if (p.on) {
        a[u] = c1[p.vec];
        b[u] = c3[p.vec];
        ea[u] = e1[p.block];
        eb[u] = e3[p.block];
      }
    }
#pragma unroll
    for (int u = 0; u < UNROLL; u++) {
      const Place p = places(s, u * THREADS + threadIdx.x);
      if (!p.on) continue;
      uint64_t x[4], y[4];
      decode(a[u], ea[u], x);
      decode(b[u], eb[u], y);
      if (x1 != nullptr) st_stream(x1 + p.vec, round_all(x));
      if (x3 != nullptr) st_stream(x3 + p.vec, round_all(y));
      if (out != nullptr) {
        swiglu(x, y, x);
        st_stream(out + p.vec, round_all(x));
      }
    }
  }
}

// the SwiGLU's backward on the held values: with g = sigmoid(x1)
//   dx1 = dh x3 (g + x1 g (1 - g)),   dx3 = dh x1 g,   h = x1 g x3 (when asked for; the W2 weight gradient reads it)
template <bool WHOLE>
__global__ void __launch_bounds__(THREADS) backward_kernel(Shape s, const uint2 *c1, const uint8_t *e1, const uint2 *c3, const uint8_t *e3,
                                                           const uint4 *dh, uint4 *dx1, uint4 *dx3, uint4 *out) {
  pdl_release();
  pdl_wait();
  const int64_t step = (int64_t)gridDim.x * THREADS * UNROLL;
  for (int64_t base = (int64_t)blockIdx.x * THREADS * UNROLL; base < s.padded; base += step) {
    const Places<WHOLE> places(s, base);
    uint2 a[UNROLL], b[UNROLL];
    uint4 d[UNROLL];
    int ea[UNROLL], eb[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; u++) {
      const Place p = places(s, u * THREADS + threadIdx.x);
      if (p.on) {
        a[u] = c1[p.vec];
        b[u] = c3[p.vec];
        d[u] = dh[p.vec];  // a plain load: a gradient may be written over it
        ea[u] = e1[p.block];
        eb[u] = e3[p.block];
      }
    }
#pragma unroll
    for (int u = 0; u < UNROLL; u++) {
      const Place p = places(s, u * THREADS + threadIdx.x);
      if (!p.on) continue;
      uint64_t x[4], y[4], g[4], o1[4], o3[4];
      decode(a[u], ea[u], x);
      decode(b[u], eb[u], y);
      widen(d[u], g);
      const uint64_t one = pack2(1.0f, 1.0f), minus = pack2(-1.0f, -1.0f);
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const uint64_t sg = sigmoid2(x[i]), silu = mul2(x[i], sg);
        o3[i] = mul2(g[i], silu);
        o1[i] = mul2(mul2(g[i], y[i]), fma2(silu, fma2(sg, minus, one), sg));
        x[i] = mul2(silu, y[i]);
      }
      st_stream(dx1 + p.vec, round_all(o1));
      st_stream(dx3 + p.vec, round_all(o3));
      if (out != nullptr) st_stream(out + p.vec, round_all(x));
    }
  }
}

}  // namespace act8
}  // namespace b200

using namespace b200;

// the kernel for columns that are whole scale blocks, or the other
#define ACT8_LAUNCH(kernel, ...)                                                                                                   \
  B200_CUDA(b200_launch_overlapped(s.vecs == s.padded_vecs ? act8::kernel<true> : act8::kernel<false>, dim3(act8_grid(s.padded)),   \
                                   dim3(act8::THREADS), 0, (cudaStream_t)stream, 1, s, __VA_ARGS__))

namespace {

int act8_shape(const char *op, int n_rows, int n_cols, act8::Shape *s) {
  B200_REQUIRE(n_rows >= 0 && n_cols > 0 && n_cols % 8 == 0, "%s: need n_rows >= 0 and n_cols a positive multiple of 8 (got %d x %d)", op,
               n_rows, n_cols);
  s->vecs = n_cols / 8;
  s->padded_vecs = (s->vecs + 3) / 4 * 4;
  s->blocks = s->padded_vecs / 4;
  s->padded = (int64_t)n_rows * s->padded_vecs;
  return 0;
}

int act8_codes_ok(const char *op, const void *c1, const void *e1, const void *c3, const void *e3) {
  B200_REQUIRE(c1 && e1 && c3 && e3, "%s: null codes or scales", op);
  B200_REQUIRE(((reinterpret_cast<uintptr_t>(c1) | reinterpret_cast<uintptr_t>(c3)) & 7u) == 0, "%s: the codes must be 8-byte aligned", op);
  return 0;
}

int act8_grid(int64_t units) {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const int64_t want = (units + act8::THREADS * act8::UNROLL - 1) / (act8::THREADS * act8::UNROLL), most = (int64_t)sms * 64;
  // four blocks run on an SM: at 16 times as many the last ones end together (at 8 times, 2 % more time; at one, 2 to 16 %)
  return (int)(want < most ? want : most);
}

}  // namespace

extern "C" uint64_t b200_act8_scales_bytes(int n_rows, int n_cols) {
  return n_rows > 0 && n_cols > 0 ? (uint64_t)n_rows * (uint64_t)((n_cols + 31) / 32) : 0;
}

extern "C" int b200_swiglu_act8(int fwd_dt, int n_rows, int n_cols, const void *x_w1, const void *x_w3, void *out, void *codes_w1,
                                void *scales_w1, void *codes_w3, void *scales_w3, void *stream) {
  B200_REQUIRE(fwd_dt == B200_DT_BF16, "swiglu_act8: only bf16 is implemented (datatype code %d)", fwd_dt);
  act8::Shape s;
  if (act8_shape("swiglu_act8", n_rows, n_cols, &s)) return -1;
  if (n_rows == 0) return 0;
  B200_REQUIRE(x_w1 && x_w3 && b200_aligned16(x_w1) && b200_aligned16(x_w3) && b200_aligned16(out),
               "swiglu_act8: x_w1 and x_w3 must be given, and all tensors 16-byte aligned");
  if (act8_codes_ok("swiglu_act8", codes_w1, scales_w1, codes_w3, scales_w3)) return -1;
  ACT8_LAUNCH(keep_kernel, (const uint4 *)x_w1, (const uint4 *)x_w3, (uint4 *)out, (uint2 *)codes_w1, (uint8_t *)scales_w1, (uint2 *)codes_w3,
      (uint8_t *)scales_w3);
  B200_CHECK_LAUNCH("swiglu_act8");
  return 0;
}

extern "C" int b200_swiglu_recompute_act8(int fwd_dt, int n_rows, int n_cols, const void *codes_w1, const void *scales_w1,
                                          const void *codes_w3, const void *scales_w3, void *x_w1, void *x_w3, void *out, void *stream) {
  B200_REQUIRE(fwd_dt == B200_DT_BF16, "swiglu_recompute_act8: only bf16 is implemented (datatype code %d)", fwd_dt);
  act8::Shape s;
  if (act8_shape("swiglu_recompute_act8", n_rows, n_cols, &s)) return -1;
  if (n_rows == 0) return 0;
  B200_REQUIRE((x_w1 || x_w3 || out) && b200_aligned16(x_w1) && b200_aligned16(x_w3) && b200_aligned16(out),
               "swiglu_recompute_act8: one output at least must be given, each 16-byte aligned");
  if (act8_codes_ok("swiglu_recompute_act8", codes_w1, scales_w1, codes_w3, scales_w3)) return -1;
  ACT8_LAUNCH(restore_kernel, (const uint2 *)codes_w1, (const uint8_t *)scales_w1, (const uint2 *)codes_w3, (const uint8_t *)scales_w3, (uint4 *)x_w1,
      (uint4 *)x_w3, (uint4 *)out);
  B200_CHECK_LAUNCH("swiglu_recompute_act8");
  return 0;
}

extern "C" int b200_swiglu_bwd_x_act8(int bwd_dt, int n_rows, int n_cols, const void *codes_w1, const void *scales_w1, const void *codes_w3,
                                      const void *scales_w3, const void *upstream_dX, void *dX_w1, void *dX_w3, void *out, void *stream) {
  B200_REQUIRE(bwd_dt == B200_DT_BF16, "swiglu_bwd_x_act8: only bf16 is implemented (datatype code %d)", bwd_dt);
  act8::Shape s;
  if (act8_shape("swiglu_bwd_x_act8", n_rows, n_cols, &s)) return -1;
  if (n_rows == 0) return 0;
  B200_REQUIRE(upstream_dX && dX_w1 && dX_w3 && b200_aligned16(upstream_dX) && b200_aligned16(dX_w1) && b200_aligned16(dX_w3) &&
                   b200_aligned16(out),
               "swiglu_bwd_x_act8: the upstream gradient and both gradients must be given, and all tensors 16-byte aligned");
  if (act8_codes_ok("swiglu_bwd_x_act8", codes_w1, scales_w1, codes_w3, scales_w3)) return -1;
  ACT8_LAUNCH(backward_kernel, (const uint2 *)codes_w1, (const uint8_t *)scales_w1, (const uint2 *)codes_w3, (const uint8_t *)scales_w3,
      (const uint4 *)upstream_dX, (uint4 *)dX_w1, (uint4 *)dX_w3, (uint4 *)out);
  B200_CHECK_LAUNCH("swiglu_bwd_x_act8");
  return 0;
}
