// LayerNorm / RMSNorm of token rows with its backward pass.
//
// Forward, per row of d values (xh: the normalised row):
//     mean = sum(x) / d,  var = sum((x - mean)^2) / d,  rstd = 1 / sqrt(var + eps)      (RMS: mean = 0)
//     xh = (x - mean) rstd,   y = xh (gamma + gamma_offset) + beta
// Backward, with g = dy (gamma + gamma_offset):
//     dx = rstd (g - sum(g) / d - xh sum(g xh) / d)                                     (RMS: without sum(g))
//     dgamma = sum over rows of dy xh,   dbeta = sum over rows of dy
//
// Both are one pass over their rows: a row stays in the registers of its threads between its sums and
// what is written.  DRAM is the floor, and instructions come next to it, hence
//   * rows travel by cp.async into slots that only the asking thread reads, two or three rows ahead (32768 x 2048 bf16, RMS
//     backward: next row in registers 127 us, this 95);
//   * arithmetic in packed pairs and parameters that stay with the thread (scalar: 25 instructions an element; the same
//     case 95 -> 82 us, 50432 x 768 forward 42 -> 27);
//   * a thread has the same columns of every row its block takes, so the column sums of the backward pass are running sums in
//     its registers; a block writes one partial row of them at its end, and a second kernel adds the partial rows in the
//     order of the blocks.  No atomics: the same call gives the same bits.
// Of the measured copy rate (6.5 TB/s), calls one after another, the second kernel within them: forward 88 % at 50432 x 768
// (27 us), 83 % at 32768 x 2048 (50), 81 % at 40000 x 1024 fp32 (62); backward 74 % (83 us), 83 % (90) and, at 50432 x 768, 63 %
// (56 us, 43 without the column sums: 24 columns a lane and their two sums take all 128 registers, and the second kernel some 4 us).
// Rows that no vector divides go one element a load: 4099 x 1023 fp32 forward 36 %, backward 39 % (14 and 20 us).
// Statistics, both row sums and all column sums are held in 32 bits; each output is rounded once.
#include <algorithm>

#include "d2d_common.cuh"

namespace d2d {
namespace {

constexpr int MAX_THREADS = 512;
constexpr int BLOCK = 256;                 // threads of a block, unless a row takes more
constexpr int PARTIAL_BLOCKS = 296;        // partial rows of the column sums at most: two blocks per SM

struct NormShape {
  int64_t N, x_stride, dy_stride;          // strides of rows, in elements
  int d;
  int tpr;                                 // threads per row: a power of two
  int kind;
  float eps, offset;
};

// A thread's share of a row: vectors ti, ti + tpr, .. of V elements each.
template <typename T, int V>
struct Vec;
template <typename T>
struct Vec<T, 1> {
  T v;
  __device__ __forceinline__ void load(const T* p) { v = *p; }
  __device__ __forceinline__ void zero() { v = DT<T>::from_f(0.f); }
  __device__ __forceinline__ float get(int) const { return DT<T>::to_f(v); }
};
template <>
struct Vec<float, 4> {
  float4 v;
  __device__ __forceinline__ void load(const float* p) { v = *reinterpret_cast<const float4*>(p); }
  __device__ __forceinline__ void zero() { v = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ float get(int q) const { return q == 0 ? v.x : q == 1 ? v.y : q == 2 ? v.z : v.w; }
};
template <>
struct Vec<bf16, 8> {
  uint4 v;
  __device__ __forceinline__ void load(const bf16* p) { v = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void zero() { v = make_uint4(0u, 0u, 0u, 0u); }
  __device__ __forceinline__ float get(int q) const {
    const uint32_t w = (q >> 1) == 0 ? v.x : (q >> 1) == 1 ? v.y : (q >> 1) == 2 ? v.z : v.w;
    return __uint_as_float(q & 1 ? w & 0xffff0000u : w << 16);
  }
};

// a load that stays behind the wait (its pointer need not be `fresh`, which would keep it in registers)
__device__ __forceinline__ float load_in_order(const float* p) {
  float v;
  asm volatile("ld.global.f32 %0, [%1];" : "=f"(v) : "l"(p));
  return v;
}
template <int V>
__device__ __forceinline__ void store_vec(float* p, const float* f) {
  if (V == 4) *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
  else *p = f[0];
}
template <int V>
__device__ __forceinline__ void store_vec(bf16* p, const float* f) {
  if (V == 8)
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]),
                                              pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  else
    *p = __float2bfloat16_rn(f[0]);
}
// V parameters as floats, whatever their type (V > 1: from a 16-byte boundary)
template <int V>
__device__ __forceinline__ void load_params(const float* p, float* f) {
  if (V == 1) f[0] = __ldg(p);
#pragma unroll
  for (int i = 0; i < V / 4; ++i) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p) + i);
    f[4 * i] = a.x, f[4 * i + 1] = a.y, f[4 * i + 2] = a.z, f[4 * i + 3] = a.w;
  }
}
template <int V>
__device__ __forceinline__ void load_params(const bf16* p, float* f) {
  if (V == 1) {
    f[0] = __bfloat162float(*p);
  } else {
    const uint4 a = __ldg(reinterpret_cast<const uint4*>(p));
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}

// Sums of M values over the threads of each row.  Rows of more than a warp meet in shared memory, in
// one of two buffers in turn: a buffer is written again only behind the barrier after its last reads.  The barrier is
// the row slot's own.
template <int M>
__device__ __forceinline__ void row_sum(float (&v)[M], int tpr, float (*buf)[MAX_THREADS / 32][2], int& turn) {
#pragma unroll 1
  for (int o = min(tpr, 32) >> 1; o > 0; o >>= 1)
#pragma unroll
    for (int m = 0; m < M; ++m) v[m] += __shfl_xor_sync(0xffffffffu, v[m], o);
  if (tpr <= 32) return;
  const int warp = threadIdx.x >> 5, w = tpr >> 5, w0 = warp & ~(w - 1);
  if ((threadIdx.x & 31) == 0)
#pragma unroll
    for (int m = 0; m < M; ++m) buf[turn][warp][m] = v[m];
  asm volatile("bar.sync %0, %1;" ::"r"(1 + (int)threadIdx.x / tpr), "r"(tpr) : "memory");
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int m = 0; m < M; ++m) v[m] = buf[turn][w0 + (lane & (w - 1))][m];
#pragma unroll 1
  for (int o = w >> 1; o > 0; o >>= 1)
#pragma unroll
    for (int m = 0; m < M; ++m) v[m] += __shfl_xor_sync(0xffffffffu, v[m], o);
  turn ^= 1;
}

// Rows on their way.  Vectors travel by cp.async into slots that only the thread that asked for them reads: no barrier, and
// no register holds them.  Without vectors the next row waits in registers.
template <int VPT, int IN>                 // IN: inputs (x, and dy)
constexpr int ring_stages = IN * VPT <= 6 ? 4 : 2;       // (512 threads with eight vectors each: 128 KB)
template <typename T, int V, int VPT, int IN>
struct Ahead {
  static constexpr int STAGES = ring_stages<VPT, IN>;
  static constexpr bool RING = V > 1;
  Vec<T, V> next[RING ? 1 : IN][RING ? 1 : VPT];
  uint4* slots;                            // [STAGES][IN][VPT][threads]
  int stage = 0;
  __device__ __forceinline__ uint4* slot(int st, int n, int i) const {
    return slots + ((st * IN + n) * VPT + i) * (int)blockDim.x + (int)threadIdx.x;
  }
  // asks for a row (nothing where it is not there)
  __device__ __forceinline__ void fetch(int st, const T* const (&row)[IN], bool in, int ti, int tpr, int nv) {
#pragma unroll
    for (int n = 0; n < IN; ++n)
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int c = ti + i * tpr;
        if constexpr (RING) {
          if (in && c < nv)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                             (uint32_t)__cvta_generic_to_shared(slot(st, n, i))),
                         "l"(row[n] + (int64_t)c * V)
                         : "memory");
        } else {
          if (in && c < nv) next[n][i].load(row[n] + (int64_t)c * V);
          else next[n][i].zero();
        }
      }
    if constexpr (RING) asm volatile("cp.async.commit_group;" ::: "memory");
  }
  // the row asked for longest ago
  __device__ __forceinline__ void take(Vec<T, V> (&v)[IN][VPT], bool in, int ti, int tpr, int nv) {
    if constexpr (RING) asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
#pragma unroll
    for (int n = 0; n < IN; ++n)
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        if constexpr (RING) {
          v[n][i].zero();
          if (in && ti + i * tpr < nv) v[n][i].load(reinterpret_cast<const T*>(slot(stage, n, i)));
        } else {
          v[n][i] = next[n][i];
        }
      }
    stage = stage + 1 == STAGES ? 0 : stage + 1;
  }
  static constexpr int DEPTH = RING ? STAGES - 1 : 1;      // rows asked for before the first is taken
};
template <int V, int VPT, int IN>
size_t ahead_bytes(int threads) {
  return V > 1 ? (size_t)ring_stages<VPT, IN> * IN * VPT * threads * 16 : 0;
}

// 16-byte words of the backward kernel's parameters: a pair for every two elements of a row's threads
__host__ __device__ __forceinline__ int scale_words(int tpr, int elements) { return tpr * elements / 4 + 1; }

// Two floats in one instruction: add, mul and fma of pairs round each half as the scalar ones do.
using pair = unsigned long long;
__device__ __forceinline__ pair pack2(float lo, float hi) {
  pair r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 unpack2(pair v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ pair add2(pair a, pair b) {
  pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ pair mul2(pair a, pair b) {
  pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ pair fma2(pair a, pair b, pair c) {
  pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// The VPT V elements of a thread in pairs: element k is column column(k).  Without vectors a pair's halves come from
// two neighbouring turns of the row's threads.
template <int V>
__device__ __forceinline__ int column(int k, int ti, int tpr) { return (ti + k / V * tpr) * V + k % V; }
template <typename T, int V, int VPT>
__device__ __forceinline__ void to_pairs(const Vec<T, V> (&v)[VPT], pair (&x)[VPT * V / 2]) {
#pragma unroll
  for (int k = 0; k < VPT * V; k += 2)
    x[k / 2] = pack2(v[k / V].get(k % V), v[(k + 1) / V].get((k + 1) % V));
}
// zero where there is no column
template <int V, int VPT>
__device__ __forceinline__ void cut(pair (&x)[VPT * V / 2], int ti, int tpr, int nv) {
#pragma unroll
  for (int k = 0; k < VPT * V; k += 2) {
    const bool lo = ti + k / V * tpr < nv, hi = ti + (k + 1) / V * tpr < nv;
    const float2 f = unpack2(x[k / 2]);
    x[k / 2] = pack2(lo ? f.x : 0.f, hi ? f.y : 0.f);
  }
}
template <typename T, int V, int VPT>
__device__ __forceinline__ void store_pairs(T* row, const pair (&x)[VPT * V / 2], int ti, int tpr, int nv) {
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    if (ti + i * tpr >= nv) continue;
    float f[V];
#pragma unroll
    for (int q = 0; q < V; ++q) {
      const float2 u = unpack2(x[(i * V + q) / 2]);
      f[q] = (i * V + q) % 2 ? u.y : u.x;
    }
    store_vec<V>(row + column<V>(i * V, ti, tpr), f);
  }
}
template <int N>
__device__ __forceinline__ float sum_pairs(const pair (&x)[N]) {
  pair a = x[0], b = x[1 % N];
  if (N > 1) {
#pragma unroll
    for (int i = 2; i < N; i += 2) a = add2(a, x[i]);
#pragma unroll
    for (int i = 3; i < N; i += 2) b = add2(b, x[i]);
    a = add2(a, b);
  }
  const float2 f = unpack2(a);
  return f.x + f.y;
}

// V: elements of a vector (1: rows or parameters that allow no vectors); VPT: vectors of a thread
template <typename T, typename P, int V, int VPT>
__global__ void __launch_bounds__(MAX_THREADS)
norm_forward_kernel(const T* __restrict__ x, const P* __restrict__ gamma, const P* __restrict__ beta,
                    T* __restrict__ y, float* __restrict__ mean_out, float* __restrict__ rstd_out,
                    const NormShape s) {
  extern __shared__ __align__(16) uint4 ring[];
  __shared__ float buf[2][MAX_THREADS / 32][2];
  constexpr int NP = VPT * V / 2;
  grid_launch_dependents();
  grid_dependency_wait();
  fresh(gamma, beta);
  if (V == 1) fresh(x);                      // (vectors travel by cp.async, which the wait holds back)
  const int ti = threadIdx.x & (s.tpr - 1), slot = threadIdx.x / s.tpr, rows = blockDim.x / s.tpr;
  const int nv = s.d / V;
  const bool ragged = nv != s.tpr * VPT;
  const int64_t step = (int64_t)gridDim.x * rows;
  const float inv = 1.f / (float)s.d;
  using A = Ahead<T, V, VPT, 1>;
  A ahead;
  ahead.slots = ring;
  int turn = 0;
  int64_t row = (int64_t)blockIdx.x * rows + slot;
  auto fetch = [&](int st, int64_t r) {
    const T* const at[1] = {x + r * s.x_stride};
    ahead.fetch(st, at, r < s.N, ti, s.tpr, nv);
  };
#pragma unroll
  for (int i = 0; i < A::DEPTH; ++i) fetch(i, row + i * step);
  // a thread has the same columns of every row: their parameters stay in registers
  pair w[NP], b[NP];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    float f[V], g[V];
#pragma unroll
    for (int q = 0; q < V; ++q) f[q] = 1.f, g[q] = 0.f;
    const int c = column<V>(i * V, ti, s.tpr);
    if (ti + i * s.tpr < nv) {
      if (gamma) {
        load_params<V>(gamma + c, f);
#pragma unroll
        for (int q = 0; q < V; ++q) f[q] += s.offset;
      }
      if (beta) load_params<V>(beta + c, g);
    }
#pragma unroll
    for (int q = 0; q < V; ++q) {
      const int k = i * V + q;
      if (k % 2 == 0) w[k / 2] = pack2(f[q], 0.f), b[k / 2] = pack2(g[q], 0.f);
      else w[k / 2] = pack2(unpack2(w[k / 2]).x, f[q]), b[k / 2] = pack2(unpack2(b[k / 2]).x, g[q]);
    }
  }
  // (every row slot of a warp takes as many turns: shuffles are for whole warps)
  for (int64_t first = (int64_t)blockIdx.x * rows; first < s.N; first += step, row += step) {
    const bool in = row < s.N;
    pair v[NP], acc[2];
    {
      Vec<T, V> raw[1][VPT];
      ahead.take(raw, in, ti, s.tpr, nv);
      to_pairs(raw[0], v);
    }
    fetch(A::RING ? (ahead.stage + A::STAGES - 2) % A::STAGES : 0, row + A::DEPTH * step);
    float mean = 0.f;
    if (s.kind == D2D_NORM_LAYER) {
      float sum[1] = {sum_pairs(v)};
      row_sum<1>(sum, s.tpr, buf, turn);
      mean = sum[0] * inv;
      const pair m = pack2(-mean, -mean);
#pragma unroll
      for (int k = 0; k < NP; ++k) v[k] = add2(v[k], m);
      if (ragged) cut<V, VPT>(v, ti, s.tpr, nv);
    }
    acc[0] = acc[1] = 0;
#pragma unroll
    for (int k = 0; k < NP; ++k) acc[k & 1] = fma2(v[k], v[k], acc[k & 1]);
    float sq[1] = {sum_pairs(acc)};
    row_sum<1>(sq, s.tpr, buf, turn);
    const float rstd = rsqrtf(fmaf(sq[0], inv, s.eps));
    if (!in) continue;
    if (ti == 0) {
      if (mean_out) mean_out[row] = mean;
      if (rstd_out) rstd_out[row] = rstd;
    }
    const pair r = pack2(rstd, rstd);
#pragma unroll
    for (int k = 0; k < NP; ++k) v[k] = fma2(mul2(v[k], r), w[k], b[k]);
    store_pairs<T, V, VPT>(y + row * s.d, v, ti, s.tpr, nv);
  }
}

// part: [blocks][2][d] column sums of dy xh and dy, or null.  COLS: they are wanted.
template <typename T, typename P, int V, int VPT, bool COLS>
__global__ void __launch_bounds__(MAX_THREADS)
norm_backward_kernel(const T* __restrict__ dy, const T* __restrict__ x, const P* __restrict__ gamma,
                     const float* __restrict__ mean_in, const float* __restrict__ rstd_in,
                     T* __restrict__ dx, float* __restrict__ part, const NormShape s) {
  // gamma + offset in fp32 [threads' columns], then rows on their way; at the end [row slots][2][d] column sums
  extern __shared__ __align__(16) uint4 ring[];
  __shared__ float buf[2][MAX_THREADS / 32][2];
  constexpr int NP = VPT * V / 2;
  grid_launch_dependents();
  grid_dependency_wait();
  fresh(gamma);
  if (V == 1) fresh(dy, x);
  const int ti = threadIdx.x & (s.tpr - 1), slot = threadIdx.x / s.tpr, rows = blockDim.x / s.tpr;
  const int nv = s.d / V;
  const int64_t step = (int64_t)gridDim.x * rows;
  const float inv = 1.f / (float)s.d;
  using A = Ahead<T, V, VPT, 2>;
  A ahead;
  ahead.slots = ring + scale_words(s.tpr, VPT * V);
  int turn = 0;
  int64_t row = (int64_t)blockIdx.x * rows + slot;
  auto fetch = [&](int st, int64_t r) {
    const T* const at[2] = {x + r * s.x_stride, dy + r * s.dy_stride};
    ahead.fetch(st, at, r < s.N, ti, s.tpr, nv);
  };
#pragma unroll
  for (int i = 0; i < A::DEPTH; ++i) fetch(i, row + i * step);
  // [pair][thread of a row]: 8 bytes a lane
  pair* const scale = reinterpret_cast<pair*>(ring);
  for (int i = threadIdx.x; i < NP * s.tpr; i += blockDim.x) {
    const int k = 2 * (i / s.tpr), t = i & (s.tpr - 1);
    const int c0 = column<V>(k, t, s.tpr), c1 = column<V>(k + 1, t, s.tpr);
    scale[i] = pack2(gamma && c0 < s.d ? DT<P>::to_f(gamma[c0]) + s.offset : 1.f,
                     gamma && c1 < s.d ? DT<P>::to_f(gamma[c1]) + s.offset : 1.f);
  }
  pair dg[COLS ? NP : 1], db[COLS ? NP : 1];
  if (COLS)
#pragma unroll
    for (int k = 0; k < NP; ++k) dg[k] = db[k] = 0;
  float mean = row < s.N && mean_in ? load_in_order(mean_in + row) : 0.f,
        rstd = row < s.N ? load_in_order(rstd_in + row) : 0.f;
  __syncthreads();
  for (int64_t first = (int64_t)blockIdx.x * rows; first < s.N; first += step, row += step) {
    const bool in = row < s.N, more = row + step < s.N;
    pair xh[NP], g[NP], acc[2];
    {
      Vec<T, V> raw[2][VPT];
      ahead.take(raw, in, ti, s.tpr, nv);
      to_pairs(raw[0], xh);
      to_pairs(raw[1], g);
    }
    fetch(A::RING ? (ahead.stage + A::STAGES - 2) % A::STAGES : 0, row + A::DEPTH * step);
    const float mean1 = more && mean_in ? load_in_order(mean_in + row + step) : 0.f,
                rstd1 = more ? load_in_order(rstd_in + row + step) : 0.f;
    // (a row or column that is not there is zero, and so is its dy: it adds nothing)
    const pair r = pack2(rstd, rstd), m = pack2(-mean, -mean);
    acc[0] = acc[1] = 0;
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      xh[k] = mul2(add2(xh[k], m), r);
      if (COLS) {
        dg[k] = fma2(g[k], xh[k], dg[k]);
        db[k] = add2(db[k], g[k]);
      }
      g[k] = mul2(g[k], scale[k * s.tpr + ti]);
      acc[k & 1] = fma2(g[k], xh[k], acc[k & 1]);
    }
    float sums[2] = {s.kind == D2D_NORM_LAYER ? sum_pairs(g) : 0.f, sum_pairs(acc)};
    row_sum<2>(sums, s.tpr, buf, turn);
    if (in && dx) {
      const float m0 = -sums[0] * inv * rstd, m1 = -sums[1] * inv * rstd;
      const pair m02 = pack2(m0, m0), m12 = pack2(m1, m1);
#pragma unroll
      for (int k = 0; k < NP; ++k) g[k] = fma2(xh[k], m12, fma2(g[k], r, m02));
      store_pairs<T, V, VPT>(dx + row * s.d, g, ti, s.tpr, nv);
    }
    mean = mean1;
    rstd = rstd1;
  }
  if (!COLS) return;
  if (A::RING) asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();                           // (the ring is over)
  float* const cols = reinterpret_cast<float*>(ring);
  float* const mine = rows > 1 ? cols + (int64_t)slot * 2 * s.d : part + (int64_t)blockIdx.x * 2 * s.d;
#pragma unroll
  for (int k = 0; k < VPT * V; ++k) {
    const int c = column<V>(k, ti, s.tpr);
    const float2 u = unpack2(dg[COLS ? k / 2 : 0]), v = unpack2(db[COLS ? k / 2 : 0]);
    if (c < s.d) {
      mine[c] = k % 2 ? u.y : u.x;
      mine[s.d + c] = k % 2 ? v.y : v.x;
    }
  }
  if (rows > 1) {
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * s.d; c += blockDim.x) {
      float sum = 0.f;
      for (int r = 0; r < rows; ++r) sum += cols[(int64_t)r * 2 * s.d + c];
      part[(int64_t)blockIdx.x * 2 * s.d + c] = sum;
    }
  }
}

// dgamma and dbeta from the partial rows: 32 columns and as many parts of the rows per block
constexpr int COLUMN_WARPS = 32;
template <typename P>
__global__ void __launch_bounds__(32 * COLUMN_WARPS)
norm_columns_kernel(const float* __restrict__ part, int blocks, int d, P* __restrict__ dgamma,
                    P* __restrict__ dbeta) {
  __shared__ float sums[COLUMN_WARPS][32];
  grid_launch_dependents();
  grid_dependency_wait();
  fresh(part);
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float sum = 0.f;
  if (c < 2 * d)
#pragma unroll 10
    for (int b = w; b < blocks; b += COLUMN_WARPS) sum += part[(int64_t)b * 2 * d + c];
  sums[w][lane] = sum;
  __syncthreads();
  if (w != 0 || c >= 2 * d) return;
#pragma unroll
  for (int i = 1; i < COLUMN_WARPS; ++i) sum += sums[i][lane];
  P* const to = c < d ? dgamma : dbeta;
  if (to) to[c < d ? c : c - d] = DT<P>::from_f(sum);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// threads of a row so that it takes at most `most` vectors of each; 0: too long
int threads_per_row(int nv, int most) {
  int t = 1;
  while (t < MAX_THREADS && (int64_t)t * most < nv) t *= 2;
  return (int64_t)t * most < nv ? 0 : t;
}

int blocks_for(int64_t N, int rows, int sms, int per_sm) {
  const int64_t need = ceil_div64(N, rows), most = (int64_t)sms * per_sm;
  return (int)(need < most ? need : most);
}

template <typename T, typename P, int V, int VPT>
int forward_vpt(const T* x, const P* gamma, const P* beta, T* y, float* mean, float* rstd, NormShape s,
                int sms, cudaStream_t st) {
  const int threads = s.tpr > BLOCK ? s.tpr : BLOCK, rows = threads / s.tpr;
  const size_t smem = ahead_bytes<V, VPT, 1>(threads);
  const auto k = norm_forward_kernel<T, P, V, VPT>;
  const int rc = device_launch_facts((const void*)k, smem, nullptr);
  if (rc != D2D_OK) return rc;
  const int grid = blocks_for(s.N, rows, sms, (VPT * V > 16 ? 512 : 1024) / threads);      // what is resident at once
  return launch_pdl(k, dim3((unsigned)grid), dim3((unsigned)threads), smem, st, x, gamma, beta, y, mean, rstd, s);
}

template <typename T, typename P>
int forward_t(const T* x, const P* gamma, const P* beta, T* y, float* mean, float* rstd, NormShape s,
              int sms, cudaStream_t st) {
  constexpr int VW = 16 / sizeof(T);
  const bool vec = s.d % VW == 0 && (s.x_stride * (int64_t)sizeof(T)) % 16 == 0 && aligned16(x) &&
                   aligned16(y) && aligned16(gamma) && aligned16(beta);
  int nv = s.d / VW;
  if (vec) s.tpr = threads_per_row(nv, VW == 4 ? 4 : nv <= 64 ? 2 : nv <= 96 ? 3 : 4);
  if (vec && s.tpr != 0) {
    const int vpt = ceil_div(nv, s.tpr);
    return vpt <= 1   ? forward_vpt<T, P, VW, 1>(x, gamma, beta, y, mean, rstd, s, sms, st)
           : vpt <= 2 ? forward_vpt<T, P, VW, 2>(x, gamma, beta, y, mean, rstd, s, sms, st)
           : vpt <= 3 ? forward_vpt<T, P, VW, 3>(x, gamma, beta, y, mean, rstd, s, sms, st)
                      : forward_vpt<T, P, VW, 4>(x, gamma, beta, y, mean, rstd, s, sms, st);
  }
  nv = s.d;
  s.tpr = threads_per_row(nv, nv <= 128 ? 4 : 8);
  if (s.tpr == 0) s.tpr = threads_per_row(nv, 32);
  if (s.tpr == 0) return D2D_ERR_UNSUPPORTED;
  const int vpt = ceil_div(nv, s.tpr);
  return vpt <= 4   ? forward_vpt<T, P, 1, 4>(x, gamma, beta, y, mean, rstd, s, sms, st)
         : vpt <= 8 ? forward_vpt<T, P, 1, 8>(x, gamma, beta, y, mean, rstd, s, sms, st)
                    : forward_vpt<T, P, 1, 32>(x, gamma, beta, y, mean, rstd, s, sms, st);
}

template <typename T, typename P, int V, int VPT>
int backward_vpt(const T* dy, const T* x, const P* gamma, const float* mean, const float* rstd, T* dx,
                 P* dgamma, P* dbeta, float* part, NormShape s, int sms, cudaStream_t st) {
  const int threads = s.tpr > BLOCK ? s.tpr : BLOCK, rows = threads / s.tpr;
  const bool cols = dgamma || dbeta;
  const size_t in_flight = ahead_bytes<V, VPT, 2>(threads) + (size_t)scale_words(s.tpr, VPT * V) * 16;
  const size_t smem = cols && rows > 1 ? std::max(in_flight, (size_t)rows * 2 * s.d * sizeof(float)) : in_flight;
  const auto k = cols ? norm_backward_kernel<T, P, V, VPT, true> : norm_backward_kernel<T, P, V, VPT, false>;
  int rc = device_launch_facts((const void*)k, smem, nullptr);
  if (rc != D2D_OK) return rc;
  if (!cols)
    return launch_pdl(k, dim3((unsigned)blocks_for(s.N, rows, sms, 1024 / threads)), dim3((unsigned)threads), smem, st,
                      dy, x, gamma, mean, rstd, dx, part, s);
  const int grid = std::min(blocks_for(s.N, rows, sms, 512 / threads), PARTIAL_BLOCKS);
  rc = launch_pdl(k, dim3((unsigned)grid), dim3((unsigned)threads), smem, st, dy, x, gamma, mean, rstd, dx,
                  part, s);
  if (rc != D2D_OK) return rc;
  return launch_pdl(norm_columns_kernel<P>, dim3((unsigned)ceil_div(2 * s.d, 32)), dim3(32 * COLUMN_WARPS), 0, st,
                    (const float*)part, grid, s.d, dgamma, dbeta);
}

template <typename T, typename P>
int backward_t(const T* dy, const T* x, const P* gamma, const float* mean, const float* rstd, T* dx,
               P* dgamma, P* dbeta, float* part, NormShape s, int sms, cudaStream_t st) {
  constexpr int VW = 16 / sizeof(T);
  const bool vec = s.d % VW == 0 && (s.x_stride * (int64_t)sizeof(T)) % 16 == 0 &&
                   (s.dy_stride * (int64_t)sizeof(T)) % 16 == 0 && aligned16(x) && aligned16(dy) &&
                   aligned16(dx) && aligned16(gamma);
  int nv = s.d / VW;
  // (16 elements a thread, 24 where a warp then has a bf16 row of 768: column sums and a row in 128 registers)
  if (vec) s.tpr = threads_per_row(nv, VW == 4 ? 4 : nv <= 64 ? 2 : nv <= 96 ? 3 : nv <= 1024 ? 2 : 4);
  if (vec && s.tpr != 0) {
    const int vpt = ceil_div(nv, s.tpr);
    return vpt <= 1   ? backward_vpt<T, P, VW, 1>(dy, x, gamma, mean, rstd, dx, dgamma, dbeta, part, s, sms, st)
           : vpt <= 2 ? backward_vpt<T, P, VW, 2>(dy, x, gamma, mean, rstd, dx, dgamma, dbeta, part, s, sms, st)
           : vpt <= 3 && (VW == 4 || s.tpr <= BLOCK)         // (512 threads, bf16: its ring and parameters are 246 KB)
               ? backward_vpt<T, P, VW, 3>(dy, x, gamma, mean, rstd, dx, dgamma, dbeta, part, s, sms, st)
               : backward_vpt<T, P, VW, 4>(dy, x, gamma, mean, rstd, dx, dgamma, dbeta, part, s, sms, st);
  }
  nv = s.d;
  s.tpr = threads_per_row(nv, nv <= 128 ? 4 : 8);
  if (s.tpr == 0) s.tpr = threads_per_row(nv, 32);
  if (s.tpr == 0) return D2D_ERR_UNSUPPORTED;
  const int vpt = ceil_div(nv, s.tpr);
  return vpt <= 4   ? backward_vpt<T, P, 1, 4>(dy, x, gamma, mean, rstd, dx, dgamma, dbeta, part, s, sms, st)
         : vpt <= 8 ? backward_vpt<T, P, 1, 8>(dy, x, gamma, mean, rstd, dx, dgamma, dbeta, part, s, sms, st)
                    : backward_vpt<T, P, 1, 32>(dy, x, gamma, mean, rstd, dx, dgamma, dbeta, part, s, sms, st);
}

}  // namespace

size_t norm_workspace_bytes(int64_t N, int d) {
  const int64_t blocks = std::min<int64_t>(N, PARTIAL_BLOCKS);
  return (size_t)blocks * 2 * (size_t)d * sizeof(float);
}

int launch_norm_forward(const void* x, int64_t x_stride, const void* gamma, const void* beta, float eps,
                        int kind, float offset, void* y, float* mean, float* rstd, int64_t N, int d,
                        int dtype, int param_dtype, cudaStream_t st) {
  int sms = 0;
  const int rc = device_launch_facts(nullptr, 0, &sms);
  if (rc != D2D_OK) return rc;
  const NormShape s = {N, x_stride, 0, d, 0, kind, eps, offset};
  if (dtype == D2D_F32)
    return forward_t((const float*)x, (const float*)gamma, (const float*)beta, (float*)y, mean, rstd, s, sms, st);
  if (param_dtype == D2D_F32)
    return forward_t((const bf16*)x, (const float*)gamma, (const float*)beta, (bf16*)y, mean, rstd, s, sms, st);
  return forward_t((const bf16*)x, (const bf16*)gamma, (const bf16*)beta, (bf16*)y, mean, rstd, s, sms, st);
}

int launch_norm_backward(const void* dy, int64_t dy_stride, const void* x, int64_t x_stride,
                         const void* gamma, int kind, float offset, const float* mean, const float* rstd,
                         void* dx, void* dgamma, void* dbeta, int64_t N, int d, int dtype, int param_dtype,
                         void* ws, cudaStream_t st) {
  int sms = 0;
  const int rc = device_launch_facts(nullptr, 0, &sms);
  if (rc != D2D_OK) return rc;
  const NormShape s = {N, x_stride, dy_stride, d, 0, kind, 0.f, offset};
  if (N == 0) {                              // nothing to sum over
    const size_t bytes = (size_t)d * (param_dtype == D2D_F32 ? 4 : 2);
    if ((dgamma && cudaMemsetAsync(dgamma, 0, bytes, st) != cudaSuccess) ||
        (dbeta && cudaMemsetAsync(dbeta, 0, bytes, st) != cudaSuccess)) {
      cudaGetLastError();
      return D2D_ERR_LAUNCH;
    }
    return D2D_OK;
  }
  if (dtype == D2D_F32)
    return backward_t((const float*)dy, (const float*)x, (const float*)gamma, mean, rstd, (float*)dx,
                      (float*)dgamma, (float*)dbeta, (float*)ws, s, sms, st);
  if (param_dtype == D2D_F32)
    return backward_t((const bf16*)dy, (const bf16*)x, (const float*)gamma, mean, rstd, (bf16*)dx,
                      (float*)dgamma, (float*)dbeta, (float*)ws, s, sms, st);
  return backward_t((const bf16*)dy, (const bf16*)x, (const bf16*)gamma, mean, rstd, (bf16*)dx,
                    (bf16*)dgamma, (bf16*)dbeta, (float*)ws, s, sms, st);
}

}  // namespace d2d
