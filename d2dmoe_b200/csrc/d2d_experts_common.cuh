// What the tensor-core expert kernels share: the packed weights' layout, the hidden epilogue's
// arithmetic and the output instruction.
#pragma once
#include "d2d_umma_api.cuh"
#include "d2d_umma_ptx.cuh"

namespace d2d {
namespace umma {

constexpr int MAX_E = 128;
constexpr int NS_MAX = 8, NS2_MAX = 8;        // stages of the two rings (upper bounds)
constexpr int SMEM_TILES = 212 * 1024;        // both rings

struct Geo {
  int kc1;         // d / 64
  int w1_stage;    // W1 (and W_up) bytes per 64-deep slice
  int kc2;         // ceil(H / 64)
  int nd, nc;      // output columns per step of the second product, steps
  int ns, ns2;     // ring stages
  int a_slot;      // bytes of a stage's rows of x
  int stage;       // bytes of a stage of the first ring: a_slot, then w1_stage
  int w2_piece;    // W2 bytes of a step's 64-deep slice (one stage of the second ring)
  long long w1_bytes, bias_off, stride;   // packed layout per expert
};

// n: tokens of the call.  A list has at most n rows, so with n <= 32 (64) a tile needs only the first
// quarter (half) of its 16 KB of x: the MMA still reads 128 rows, but what stands in the other
// rows' place reaches only accumulator rows nobody reads.  A decode step of the gated form keeps
// four stages of weights in flight instead of three.
inline Geo experts_geo(int d, int H, bool glu, long long n) {
  Geo g;
  g.kc1 = d / 64;
  g.w1_stage = (glu ? 2 : 1) * H * 128;
  g.kc2 = (H + 63) / 64;
  g.nd = !glu && d % 128 == 0 ? 128 : 64;
  g.nc = d / g.nd;
  g.a_slot = n <= 32 ? SLOT / 4 : n <= 64 ? SLOT / 2 : SLOT;
  g.stage = g.a_slot + g.w1_stage;
  g.w2_piece = g.nd * 128;
  // 48 KB of W2 pieces, then as many stages of the first ring as fit, the rest for W2
  const int ns = (SMEM_TILES - 48 * 1024) / g.stage;
  g.ns = ns < NS_MAX ? ns : NS_MAX;
  const int ns2 = (SMEM_TILES - g.ns * g.stage) / g.w2_piece;
  g.ns2 = ns2 < NS2_MAX ? ns2 : NS2_MAX;
  g.w1_bytes = (long long)g.kc1 * g.w1_stage;
  g.bias_off = g.w1_bytes + (long long)g.nc * g.kc2 * g.w2_piece;
  g.stride = (g.bias_off + 512 + 1023) / 1024 * 1024;
  return g;
}

// 16 hidden columns as 8 packed bf16 pairs, with the upstream rounding points
// (T(x W1), + b1, activation, x T(x W_up)) done in packed bf16 arithmetic: one
// float->bf16x2 conversion per pair instead of one conversion per rounding point.
// ONCE: in 32 bits instead, with one rounding at the end (the weighted form, which upstream has not).
// NORM: nacc also collects the row's norm terms of the activation (before the gating
// product), 1 = magnitudes, 2 = squares.
template <int ACT, bool GLU, bool NORM, bool ONCE = false>
__device__ __forceinline__ void ep1_pairs(const uint32_t* v, const uint32_t* u, const uint32_t* bp,
                                          uint32_t* w, float& nacc, int nord) {
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    if (ONCE) {
      float f0 = activate(__uint_as_float(v[2 * q]) + __uint_as_float(bp[q] << 16), ACT);
      float f1 = activate(__uint_as_float(v[2 * q + 1]) + __uint_as_float(bp[q] & 0xffff0000u), ACT);
      if (GLU) f0 *= __uint_as_float(u[2 * q]), f1 *= __uint_as_float(u[2 * q + 1]);
      w[q] = pack_bf16x2(f0, f1);
      continue;
    }
    __nv_bfloat162 h =
        __floats2bfloat162_rn(__uint_as_float(v[2 * q]), __uint_as_float(v[2 * q + 1]));
    h = __hadd2_rn(h, *reinterpret_cast<const __nv_bfloat162*>(&bp[q]));
    if (ACT == D2D_RELU) {
      h = __hmax2_nan(h, __float2bfloat162_rn(0.f));
    } else {
      const float2 f = __bfloat1622float2(h);
      h = __floats2bfloat162_rn(activate(f.x, ACT), activate(f.y, ACT));
    }
    if (NORM) {
      const float2 f = __bfloat1622float2(h);
      nacc += nord == 1 ? fabsf(f.x) + fabsf(f.y) : fmaf(f.x, f.x, f.y * f.y);
    }
    if (GLU) {
      const __nv_bfloat162 uu =
          __floats2bfloat162_rn(__uint_as_float(u[2 * q]), __uint_as_float(u[2 * q + 1]));
      h = __hmul2_rn(h, uu);
    }
    w[q] = *reinterpret_cast<uint32_t*>(&h);
  }
}

// Row n of a packed W2 piece holds this output column of the piece: in each block of 32 the two 2-bit
// fields above the lowest bit change places, so that column 8 f + 2 l + i of the accumulator, which
// the fragment loads give to lane l of a row, is output column 8 l + 2 f + i.
__host__ __device__ __forceinline__ int out_column(int n) {
  return (n & ~30) | ((n & 6) << 2) | ((n >> 2) & 6);
}

// t >= 0: add; t < -1: store; -1: nothing (predicated, no branch)
__device__ __forceinline__ void put_row(void* p, int t, uint4 add, uint4 st) {
  asm volatile(
      "{\n\t.reg .pred a, b;\n\t"
      "setp.ge.s32 a, %1, 0;\n\t"
      "setp.lt.s32 b, %1, -1;\n\t"
      "@a red.global.add.noftz.v4.bf16x2 [%0], {%2, %3, %4, %5};\n\t"
      "@b st.global.v4.b32 [%0], {%6, %7, %8, %9};\n\t}" ::"l"(p),
      "r"(t), "r"(add.x), "r"(add.y), "r"(add.z), "r"(add.w), "r"(st.x), "r"(st.y), "r"(st.z),
      "r"(st.w)
      : "memory");
}

// t >= 0: add
__device__ __forceinline__ void add_row(void* p, int t, uint4 v) {
  asm volatile(
      "{\n\t.reg .pred a;\n\t"
      "setp.ge.s32 a, %1, 0;\n\t"
      "@a red.global.add.noftz.v4.bf16x2 [%0], {%2, %3, %4, %5};\n\t}" ::"l"(p),
      "r"(t), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
      : "memory");
}

// Eight floats in 16 bytes: 15-bit integers in units of 2^(ex - 140) / (1 - 2^-15), where 2^(ex - 127) is the largest's power
// of two: off by half a unit, 2^-14 of the largest of eight (bf16, as many bytes, would be by 2^-8 of each).  The
// last factor keeps them below 2^14 - 1/2, so that none is rounded to 2^14; they are held with 2^14 added.  The exponent lies in the upper bits of the
// eight halves.  Exponent 255, where one is not finite: the halves are the upper 15 bits of bf16.
struct Eight {
  uint32_t f[8];           // bits of floats
};
__device__ __forceinline__ uint32_t exponent8(const Eight& v) {
  float m;
  asm("{\n\t.reg .f32 a, b, c, d, e, f, g, h;\n\t"
      "abs.f32 a, %1;\n\tabs.f32 b, %2;\n\tabs.f32 c, %3;\n\tabs.f32 d, %4;\n\t"
      "abs.f32 e, %5;\n\tabs.f32 f, %6;\n\tabs.f32 g, %7;\n\tabs.f32 h, %8;\n\t"
      "max.NaN.f32 a, a, b, c;\n\tmax.NaN.f32 d, d, e, f;\n\tmax.NaN.f32 g, g, h;\n\tmax.NaN.f32 %0, a, d, g;\n\t}"
      : "=f"(m)
      : "f"(__uint_as_float(v.f[0])), "f"(__uint_as_float(v.f[1])), "f"(__uint_as_float(v.f[2])),
        "f"(__uint_as_float(v.f[3])), "f"(__uint_as_float(v.f[4])), "f"(__uint_as_float(v.f[5])),
        "f"(__uint_as_float(v.f[6])), "f"(__uint_as_float(v.f[7])));
  return __float_as_uint(m) >> 23;
}
__device__ __forceinline__ uint4 with_exponent(uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t ex) {
  const uint32_t z = ex | ex << 15, m = 0x80008000u;       // bit 2 i to 15, bit 2 i + 1 to 31
  return make_uint4((a & ~m) | (z << 15 & m), (b & ~m) | (z << 13 & m), (c & ~m) | (z << 11 & m),
                    (d & ~m) | (z << 9 & m));
}
// ex: exponent8(v), below 255
__device__ __forceinline__ uint4 encode8(const Eight& v, uint32_t ex) {
  ex = max(ex, 14u);
  const float s = __uint_as_float(((266u - ex) << 23) + 0x7ffe00u);      // 2^(139 - ex) (2 - 2^-14)
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {                              // 1.5 2^23 + 2^14: the integer is in the lower half
    uint32_t lo, hi;
    asm("{\n\t.reg .b64 x, y, z;\n\t"
        "mov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %4};\n\tmov.b64 z, {%5, %5};\n\t"
        "fma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(v.f[2 * i]), "r"(v.f[2 * i + 1]), "f"(s), "f"(12582912.f + 16384.f));
    w[i] = __byte_perm(lo, hi, 0x5410);
  }
  return with_exponent(w[0], w[1], w[2], w[3], ex);
}
// at least one is not finite
static __device__ __noinline__ uint4 encode8_special(const Eight v) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[i] = pack_bf16x2(__uint_as_float(v.f[2 * i]), __uint_as_float(v.f[2 * i + 1]));
    w[i] = w[i] >> 1 & 0x7fff7fffu;
  }
  return with_exponent(w[0], w[1], w[2], w[3], 255u);
}
__device__ __forceinline__ uint32_t exponent_of(uint4 v) {
  const uint32_t y = (v.x >> 15 & 0x00010001u) | (v.y >> 13 & 0x00040004u) | (v.z >> 11 & 0x00100010u) |
                     (v.w >> 9 & 0x00400040u);
  return (y | y >> 15) & 255u;
}
// sum += wt * the eight (pairs of floats); ex: exponent_of(v); wt: with UNIT8 multiplied in
constexpr float UNIT8 = 1.00003051850948f;                   // 1 / (1 - 2^-15)
__device__ __forceinline__ void add_decoded8(uint4 v, uint32_t ex, float wt, unsigned long long (&sum)[4]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  const float s = wt * __uint_as_float((ex - 13u) << 23);    // 2^(ex - 140)
  unsigned long long s2, c2;
  asm("mov.b64 %0, {%1, %1};" : "=l"(s2) : "f"(s));
  asm("mov.b64 %0, {%1, %1};" : "=l"(c2) : "f"(-(8388608.f + 16384.f)));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t u = w[i] & 0x7fff7fffu;
    unsigned long long x;
    asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "r"(__byte_perm(u, 0x4b00u, 0x5410)), "r"(__byte_perm(u, 0x4b00u, 0x5432)));
    asm("add.rn.f32x2 %0, %0, %1;" : "+l"(x) : "l"(c2));
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(sum[i]) : "l"(x), "l"(s2));
  }
}
__device__ __forceinline__ void add_special8(uint4 v, float wt, unsigned long long (&sum)[4]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float lo, hi;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(sum[i]));
    lo = fmaf(wt, __uint_as_float((w[i] & 0x7fffu) << 17), lo);
    hi = fmaf(wt, __uint_as_float((w[i] >> 16 & 0x7fffu) << 17), hi);
    asm("mov.b64 %0, {%1, %2};" : "=l"(sum[i]) : "f"(lo), "f"(hi));
  }
}

}  // namespace umma

// Short calls (d2d_experts_short.cu)
bool experts_short_supported(int64_t N, int d, int E, int H, bool glu, int kept);
int launch_experts_short(const void* x, const int32_t* token_idx, const int32_t* offsets,
                         const void* packed, void* out, int64_t N, int d, int E, int H, bool glu,
                         int act, int* dev_status, cudaStream_t s, DirectRows dr);

}  // namespace d2d
