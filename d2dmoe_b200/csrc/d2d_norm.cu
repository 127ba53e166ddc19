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
// what is written, and what bounds them is DRAM.  The column sums of the backward pass ride along: a
// thread has the same columns of every row its block takes, so they are running sums in its registers;
// a block writes one partial row of them at its end, and a second kernel adds the partial rows in the
// order of the blocks.  No atomics: the same call gives the same bits.
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
// one of two buffers in turn: a buffer is written again only behind the barrier after its last reads.
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
  __syncthreads();
#pragma unroll
  for (int m = 0; m < M; ++m) v[m] = 0.f;
#pragma unroll 1
  for (int i = 0; i < w; ++i)
#pragma unroll
    for (int m = 0; m < M; ++m) v[m] += buf[turn][w0 + i][m];
  turn ^= 1;
}

// V: elements of a vector (1: rows or parameters that allow no vectors); VPT: vectors of a thread
template <typename T, typename P, int V, int VPT>
__global__ void __launch_bounds__(MAX_THREADS)
norm_forward_kernel(const T* __restrict__ x, const P* __restrict__ gamma, const P* __restrict__ beta,
                    T* __restrict__ y, float* __restrict__ mean_out, float* __restrict__ rstd_out,
                    const NormShape s) {
  __shared__ float buf[2][MAX_THREADS / 32][2];
  grid_launch_dependents();
  grid_dependency_wait();
  const int ti = threadIdx.x & (s.tpr - 1), slot = threadIdx.x / s.tpr, rows = blockDim.x / s.tpr;
  const int nv = s.d / V;
  const int64_t step = (int64_t)gridDim.x * rows;
  const float inv = 1.f / (float)s.d;
  Vec<T, V> v[VPT], nxt[VPT];
  int turn = 0;
  auto fetch = [&](Vec<T, V>(&to)[VPT], int64_t row) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = ti + i * s.tpr;
      if (row < s.N && c < nv) to[i].load(x + row * s.x_stride + (int64_t)c * V);
      else to[i].zero();
    }
  };
  int64_t row = (int64_t)blockIdx.x * rows + slot;
  fetch(v, row);
  // (the barrier in row_sum is for the whole block: every row slot takes as many turns)
  for (int64_t first = (int64_t)blockIdx.x * rows; first < s.N; first += step, row += step) {
    fetch(nxt, row + step);
    float mean = 0.f;
    if (s.kind == D2D_NORM_LAYER) {
      float sum[1] = {0.f};
#pragma unroll
      for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int q = 0; q < V; ++q) sum[0] += v[i].get(q);
      row_sum<1>(sum, s.tpr, buf, turn);
      mean = sum[0] * inv;
    }
    float sq[1] = {0.f};
#pragma unroll
    for (int i = 0; i < VPT; ++i)
      if (ti + i * s.tpr < nv)
#pragma unroll
        for (int q = 0; q < V; ++q) {
          const float a = v[i].get(q) - mean;
          sq[0] = fmaf(a, a, sq[0]);
        }
    row_sum<1>(sq, s.tpr, buf, turn);
    const float rstd = rsqrtf(fmaf(sq[0], inv, s.eps));
    if (row < s.N) {
      if (ti == 0) {
        if (mean_out) mean_out[row] = mean;
        if (rstd_out) rstd_out[row] = rstd;
      }
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int c = ti + i * s.tpr;
        if (c >= nv) continue;
        float w[V], b[V], o[V];
        if (gamma) load_params<V>(gamma + (int64_t)c * V, w);
        if (beta) load_params<V>(beta + (int64_t)c * V, b);
#pragma unroll
        for (int q = 0; q < V; ++q) {
          o[q] = (v[i].get(q) - mean) * rstd;
          if (gamma) o[q] *= w[q] + s.offset;
          if (beta) o[q] += b[q];
        }
        store_vec<V>(y + row * s.d + (int64_t)c * V, o);
      }
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) v[i] = nxt[i];
  }
}

// part: [blocks][2][d] column sums of dy xh and dy, or null.  COLS: they are wanted.
template <typename T, typename P, int V, int VPT, bool COLS>
__global__ void __launch_bounds__(MAX_THREADS)
norm_backward_kernel(const T* __restrict__ dy, const T* __restrict__ x, const P* __restrict__ gamma,
                     const float* __restrict__ mean_in, const float* __restrict__ rstd_in,
                     T* __restrict__ dx, float* __restrict__ part, const NormShape s) {
  extern __shared__ float cols[];            // [row slots of a block][2][d], where a block has several
  __shared__ float buf[2][MAX_THREADS / 32][2];
  grid_launch_dependents();
  grid_dependency_wait();
  const int ti = threadIdx.x & (s.tpr - 1), slot = threadIdx.x / s.tpr, rows = blockDim.x / s.tpr;
  const int nv = s.d / V;
  const int64_t step = (int64_t)gridDim.x * rows;
  const float inv = 1.f / (float)s.d;
  Vec<T, V> a[VPT], b[VPT], an[VPT], bn[VPT];
  float dg[COLS ? VPT : 1][V], db[COLS ? VPT : 1][V];
  if (COLS)
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int q = 0; q < V; ++q) dg[i][q] = db[i][q] = 0.f;
  int turn = 0;
  auto fetch = [&](Vec<T, V>(&u)[VPT], Vec<T, V>(&w)[VPT], int64_t row) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = ti + i * s.tpr;
      if (row < s.N && c < nv) {
        u[i].load(x + row * s.x_stride + (int64_t)c * V);
        w[i].load(dy + row * s.dy_stride + (int64_t)c * V);
      } else {
        u[i].zero();
        w[i].zero();
      }
    }
  };
  int64_t row = (int64_t)blockIdx.x * rows + slot;
  fetch(a, b, row);
  for (int64_t first = (int64_t)blockIdx.x * rows; first < s.N; first += step, row += step) {
    fetch(an, bn, row + step);
    const bool in = row < s.N;
    const float mean = in && mean_in ? __ldg(mean_in + row) : 0.f, rstd = in ? __ldg(rstd_in + row) : 0.f;
    float sums[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = ti + i * s.tpr;
      if (c >= nv) continue;
      float w[V];
      if (gamma) load_params<V>(gamma + (int64_t)c * V, w);
#pragma unroll
      for (int q = 0; q < V; ++q) {
        const float xh = (a[i].get(q) - mean) * rstd, g = gamma ? b[i].get(q) * (w[q] + s.offset) : b[i].get(q);
        sums[0] += g;
        sums[1] = fmaf(g, xh, sums[1]);
        if (COLS && in) {                    // (a row that is not there has no say, whatever x's first rows hold)
          dg[i][q] = fmaf(b[i].get(q), xh, dg[i][q]);
          db[i][q] += b[i].get(q);
        }
      }
    }
    row_sum<2>(sums, s.tpr, buf, turn);
    const float m0 = s.kind == D2D_NORM_LAYER ? sums[0] * inv : 0.f, m1 = sums[1] * inv;
    if (in && dx) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int c = ti + i * s.tpr;
        if (c >= nv) continue;
        float w[V], o[V];
        if (gamma) load_params<V>(gamma + (int64_t)c * V, w);
#pragma unroll
        for (int q = 0; q < V; ++q) {
          const float xh = (a[i].get(q) - mean) * rstd, g = gamma ? b[i].get(q) * (w[q] + s.offset) : b[i].get(q);
          o[q] = rstd * (g - m0 - xh * m1);
        }
        store_vec<V>(dx + row * s.d + (int64_t)c * V, o);
      }
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) a[i] = an[i], b[i] = bn[i];
  }
  if (!COLS) return;
  float* const mine = rows > 1 ? cols + (int64_t)slot * 2 * s.d : part + (int64_t)blockIdx.x * 2 * s.d;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = ti + i * s.tpr;
    if (c < nv)
#pragma unroll
      for (int q = 0; q < V; ++q) {
        mine[c * V + q] = dg[i][q];
        mine[s.d + c * V + q] = db[i][q];
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

// dgamma and dbeta from the partial rows: 32 columns and eight parts of the rows per block
template <typename P>
__global__ void __launch_bounds__(BLOCK)
norm_columns_kernel(const float* __restrict__ part, int blocks, int d, P* __restrict__ dgamma,
                    P* __restrict__ dbeta) {
  __shared__ float sums[BLOCK / 32][32];
  grid_launch_dependents();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float sum = 0.f;
  if (c < 2 * d)
#pragma unroll 8
    for (int b = w; b < blocks; b += BLOCK / 32) sum += part[(int64_t)b * 2 * d + c];
  sums[w][lane] = sum;
  __syncthreads();
  if (w != 0 || c >= 2 * d) return;
#pragma unroll
  for (int i = 1; i < BLOCK / 32; ++i) sum += sums[i][lane];
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
  const int grid = blocks_for(s.N, rows, sms, 1024 / threads);
  return launch_pdl(norm_forward_kernel<T, P, V, VPT>, dim3((unsigned)grid), dim3((unsigned)threads), 0,
                    st, x, gamma, beta, y, mean, rstd, s);
}

template <typename T, typename P>
int forward_t(const T* x, const P* gamma, const P* beta, T* y, float* mean, float* rstd, NormShape s,
              int sms, cudaStream_t st) {
  constexpr int VW = 16 / sizeof(T);
  const bool vec = s.d % VW == 0 && (s.x_stride * (int64_t)sizeof(T)) % 16 == 0 && aligned16(x) &&
                   aligned16(y) && aligned16(gamma) && aligned16(beta);
  int nv = s.d / VW;
  if (vec) s.tpr = threads_per_row(nv, nv <= 32 ? 1 : nv <= 96 ? 3 : nv <= 256 ? 2 : 4);
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
  if (!cols)
    return launch_pdl(norm_backward_kernel<T, P, V, VPT, false>,
                      dim3((unsigned)blocks_for(s.N, rows, sms, 1024 / threads)), dim3((unsigned)threads), 0,
                      st, dy, x, gamma, mean, rstd, dx, part, s);
  const size_t smem = rows > 1 ? (size_t)rows * 2 * s.d * sizeof(float) : 0;
  const auto k = norm_backward_kernel<T, P, V, VPT, true>;
  int rc = device_launch_facts((const void*)k, smem, nullptr);
  if (rc != D2D_OK) return rc;
  const int grid = std::min(blocks_for(s.N, rows, sms, 2), PARTIAL_BLOCKS);
  rc = launch_pdl(k, dim3((unsigned)grid), dim3((unsigned)threads), smem, st, dy, x, gamma, mean, rstd, dx,
                  part, s);
  if (rc != D2D_OK) return rc;
  return launch_pdl(norm_columns_kernel<P>, dim3((unsigned)ceil_div(2 * s.d, 32)), dim3(BLOCK), 0, st,
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
  if (vec) s.tpr = threads_per_row(nv, nv <= 32 ? 1 : nv <= 96 ? 3 : nv <= 1024 ? 2 : 4);
  if (vec && s.tpr != 0) {
    const int vpt = ceil_div(nv, s.tpr);
    return vpt <= 1   ? backward_vpt<T, P, VW, 1>(dy, x, gamma, mean, rstd, dx, dgamma, dbeta, part, s, sms, st)
           : vpt <= 2 ? backward_vpt<T, P, VW, 2>(dy, x, gamma, mean, rstd, dx, dgamma, dbeta, part, s, sms, st)
           : vpt <= 3 ? backward_vpt<T, P, VW, 3>(dy, x, gamma, mean, rstd, dx, dgamma, dbeta, part, s, sms, st)
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
