// Experts weighted by a routing:
//     out[t] = last_bias (+ x[t]) + sum over slots j of w[t, j] y[t, j],   y[t, j] = FFN of expert e[t, j] on x[t]
// with the slots' experts and weights as d2d_route leaves them (expert -1: no such slot).
//
// The upstream layer adds 0/1-routed outputs into one row as they come; here the sum of a token is held in 32 bits,
// taken in the order of its slots and rounded once, so a call gives the same bits every time.  Two ways:
//   lists   The pairs p = t k + j are sorted by expert (counting sort, ascending p in each list), the expert kernels
//           run over the lists and store row p of a table [N k, d], and a last pass sums each token's k rows, which
//           lie together.  The table is in T: a row is rounded once more than it would have to be, which costs as
//           much accuracy as the rounding of the tensor cores' hidden operand does (2^-9 of a row's size in
//           bf16); rows of 32 bits would double the traffic that bounds this form.
//   few     Calls of few pairs are bound by latency and by the weights' bytes: two kernels without lists, all
//           sums in 32 bits.  The first splits every pair's hidden columns and, where there are fewer such pieces than SMs,
//           the depth d over blocks; the second adds the depth's parts, applies bias, activation and weight, and takes
//           the second product over all k H hidden values of a token at once.
#include <algorithm>

#include "d2d_common.cuh"
#include "d2d_umma_api.cuh"

namespace d2d {
namespace {

constexpr int NT = 256;
constexpr int MAX_E = 256;
constexpr int64_t ONE_BLOCK_PAIRS = 4096;   // sorted by a single block of 1024 threads
constexpr int CHUNK_BLOCKS = 148;           // blocks of larger sorts, at most

// -- lists of pairs ---------------------------------------------------------------------------------
// Counting sort, stable: every block counts its chunk of the pairs (the first kernel), then, knowing everyone's counts,
// writes it: warps take contiguous parts of the chunk, 32 pairs at a time, and pairs of one expert among them
// rank by lane.
__global__ void __launch_bounds__(NT)
pairs_count_kernel(const int32_t* __restrict__ experts, int64_t P, int E, int64_t chunk,
                   int32_t* __restrict__ table) {
  __shared__ int hist[MAX_E];
  grid_launch_dependents();
  grid_dependency_wait();
  for (int e = threadIdx.x; e < E; e += NT) hist[e] = 0;
  __syncthreads();
  const int64_t p0 = blockIdx.x * chunk, p1 = min(P, p0 + chunk);
  for (int64_t p = p0 + threadIdx.x; p < p1; p += NT) {
    const int e = experts[p];
    if ((unsigned)e < (unsigned)E) atomicAdd(&hist[e], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < E; e += NT) table[(int64_t)blockIdx.x * E + e] = hist[e];
}

// one block: no table.  Shared memory: [warps][E], then 3 E + 1 words.
__global__ void __launch_bounds__(1024)
pairs_scatter_kernel(const int32_t* __restrict__ experts, int64_t P, int E, int64_t chunk,
                     const int32_t* __restrict__ table, int32_t* __restrict__ pairs,
                     int32_t* __restrict__ offsets, int* dev_status) {
  extern __shared__ int sm[];
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, warps = blockDim.x >> 5;
  int* const mine = sm + w * E;             // this warp's counts, then where its next pair of an expert goes
  int* const total = sm + warps * E;        // [E]
  int* const before = total + E;            // [E]: pairs of earlier blocks
  int* const first = before + E;            // [E + 1]
  grid_launch_dependents();
  grid_dependency_wait();
  for (int i = tid; i < warps * E + 2 * E; i += blockDim.x) sm[i] = 0;
  __syncthreads();
  const int64_t part = (chunk + warps - 1) / warps;
  const int64_t p0 = blockIdx.x * chunk + w * part, p1 = min(min(P, (blockIdx.x + 1) * chunk), p0 + part);
  for (int64_t p = p0 + lane; p < p1; p += 32) {
    const int e = experts[p];
    if ((unsigned)e < (unsigned)E) atomicAdd(&mine[e], 1);
    else if (e != -1) report(dev_status, D2D_ERR_INDEX_RANGE);
  }
  __syncthreads();
  if (table) {
    int EP = 1;
    while (EP < E) EP *= 2;
    const int e = tid & (EP - 1), parts = blockDim.x / EP;
    int all = 0, early = 0;
    if (e < E)
#pragma unroll 4
      for (int b = tid / EP; b < (int)gridDim.x; b += parts) {
        const int n = table[(int64_t)b * E + e];
        all += n;
        early += b < (int)blockIdx.x ? n : 0;
      }
    if (all) atomicAdd(&total[e], all);
    if (early) atomicAdd(&before[e], early);
  } else {
    for (int e = tid; e < E; e += blockDim.x) {
      int sum = 0;
      for (int i = 0; i < warps; ++i) sum += sm[i * E + e];
      total[e] = sum;
    }
  }
  __syncthreads();
  if (w == 0) {
    int run = 0;
    for (int e0 = 0; e0 < E; e0 += 32) {
      const int n = e0 + lane < E ? total[e0 + lane] : 0;
      int incl = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      if (e0 + lane < E) first[e0 + lane] = run + incl - n;
      run += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) first[E] = run;
  }
  __syncthreads();
  if (blockIdx.x == 0)
    for (int e = tid; e <= E; e += blockDim.x) offsets[e] = first[e];
  for (int e = tid; e < E; e += blockDim.x) {
    int run = first[e] + before[e];
    for (int i = 0; i < warps; ++i) {
      const int n = sm[i * E + e];
      sm[i * E + e] = run;
      run += n;
    }
  }
  __syncthreads();
  for (int64_t q = p0; q < p1; q += 32) {
    const int64_t p = q + lane;
    int e = p < p1 ? experts[p] : -1;
    if ((unsigned)e >= (unsigned)E) e = -1;
    const uint32_t same = __match_any_sync(0xffffffffu, e);
    int at = 0;
    if (e >= 0) at = mine[e] + __popc(same & ((1u << lane) - 1u));
    __syncwarp();
    if (e >= 0) {
      pairs[at] = (int)p;
      if ((same >> lane) == 1u) mine[e] = at + 1;      // the last of them
    }
    __syncwarp();
  }
}

// -- sum of a token's rows --------------------------------------------------------------------------------
template <typename T, int V>
__device__ __forceinline__ void load_row(const T* p, float* f) {
  if constexpr (V == 1) {
    f[0] = DT<T>::to_f(*p);
  } else if constexpr (sizeof(T) == 4) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w;
  } else {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}
template <typename T, int V>
__device__ __forceinline__ void store_row(T* p, const float* f) {
  if constexpr (V == 1) {
    *p = DT<T>::from_f(f[0]);
  } else if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
  } else {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]),
                                              pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  }
}

// y: [N k, d].  A warp has a token; its weights are in its lanes.
template <typename T, int V>
__global__ void __launch_bounds__(NT)
combine_kernel(const T* __restrict__ y, const int32_t* __restrict__ experts, const float* __restrict__ weights,
               const T* __restrict__ last_bias, const T* __restrict__ x, T* __restrict__ out, int64_t N, int d,
               int E, int k) {
  grid_launch_dependents();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, nv = d / V;
  for (int64_t t = (int64_t)blockIdx.x * (NT / 32) + (threadIdx.x >> 5); t < N; t += (int64_t)gridDim.x * (NT / 32)) {
    const int e = lane < k ? experts[t * k + lane] : -1;
    const float w = lane < k ? weights[t * k + lane] : 0.f;
    const uint32_t there = __ballot_sync(0xffffffffu, (unsigned)e < (unsigned)E);
    for (int c = lane; c < ceil_div(nv, 32) * 32; c += 32) {
      float sum[V], f[V];
#pragma unroll
      for (int i = 0; i < V; ++i) sum[i] = 0.f;
#pragma unroll 4
      for (int j = 0; j < k; ++j) {
        const float wj = __shfl_sync(0xffffffffu, w, j);
        if ((there >> j & 1u) == 0u || c >= nv) continue;
        load_row<T, V>(y + (t * k + j) * d + (int64_t)c * V, f);
#pragma unroll
        for (int i = 0; i < V; ++i) sum[i] = fmaf(wj, f[i], sum[i]);
      }
      if (c >= nv) continue;
      if (last_bias) {
        load_row<T, V>(last_bias + (int64_t)c * V, f);
#pragma unroll
        for (int i = 0; i < V; ++i) sum[i] += f[i];
      }
      if (x) {
        load_row<T, V>(x + t * d + (int64_t)c * V, f);
#pragma unroll
        for (int i = 0; i < V; ++i) sum[i] += f[i];
      }
      store_row<T, V>(out + t * d + (int64_t)c * V, sum);
    }
  }
}

// -- few pairs ---------------------------------------------------------------------------------------------
// columns of a block: four threads of 16 bytes each, or 32 of one element
template <int V>
constexpr int few_threads = V == 1 ? 32 : 4;

// V sums of each thread over the block's threads of the same columns -> the first TC V threads, in red
template <int V>
__device__ __forceinline__ float few_sum(float (&v)[V], float* red) {
  constexpr int TC = few_threads<V>;
  const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31;
#pragma unroll
  for (int o = TC; o < 32; o <<= 1)
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  __syncthreads();
  if (lane < TC)
#pragma unroll
    for (int i = 0; i < V; ++i) red[w * TC * V + lane * V + i] = v[i];
  __syncthreads();
  float sum = 0.f;
  if (tid < TC * V)
#pragma unroll
    for (int i = 0; i < NT / 32; ++i) sum += red[i * TC * V + tid];
  return sum;
}

// part[s][p][gate, up][H]: pair p's share of x W1 (and x W_up) from depth part s
template <typename T, int V, bool GLU>
__global__ void __launch_bounds__(NT)
few_hidden_kernel(const WeightedCall c, int splits, float* __restrict__ part) {
  constexpr int TC = few_threads<V>, RG = NT / TC, G = GLU ? 2 : 1;
  __shared__ float red[NT / 32 * TC * V];
  grid_launch_dependents();
  grid_dependency_wait();
  const int tid = threadIdx.x, H = c.H, d = c.d;
  const int hcs = ceil_div(H, TC * V), hc = blockIdx.x % hcs, s = blockIdx.x / hcs;
  const int64_t p = blockIdx.y, P = c.N * c.k, t = p / c.k;
  const int e = c.experts[p];
  if ((unsigned)e >= (unsigned)c.E) {
    if (e != -1 && tid == 0) report(c.dev_status, D2D_ERR_INDEX_RANGE);
    return;
  }
  const int depth = ceil_div(d, splits), d0 = s * depth, d1 = min(d, d0 + depth);
  const int col = hc * TC * V + (tid % TC) * V;
  const bool in = col < H;
  const T* const x = (const T*)c.x + t * d;
  const T* const w1 = (const T*)c.w1 + (int64_t)e * d * H + col;
  const T* const wu = GLU ? (const T*)c.w_up + (int64_t)e * d * H + col : nullptr;
  float a[V], u[V];
#pragma unroll
  for (int i = 0; i < V; ++i) a[i] = u[i] = 0.f;
  if (in)
#pragma unroll 4
    for (int r = d0 + tid / TC; r < d1; r += RG) {
      float f[V];
      const float xv = DT<T>::to_f(x[r]);
      load_row<T, V>(w1 + (int64_t)r * H, f);
#pragma unroll
      for (int i = 0; i < V; ++i) a[i] = fmaf(xv, f[i], a[i]);
      if (GLU) {
        load_row<T, V>(wu + (int64_t)r * H, f);
#pragma unroll
        for (int i = 0; i < V; ++i) u[i] = fmaf(xv, f[i], u[i]);
      }
    }
  float* const to = part + ((int64_t)s * P + p) * G * H;
  const int out = hc * TC * V + tid;
  const float sum = few_sum<V>(a, red);
  if (tid < TC * V && out < H) to[out] = sum;
  if (GLU) {
    const float up = few_sum<V>(u, red);
    if (tid < TC * V && out < H) to[H + out] = up;
  }
}

template <typename T, int V, bool GLU>
__global__ void __launch_bounds__(NT)
few_out_kernel(const WeightedCall c, int splits, const float* __restrict__ part) {
  constexpr int TC = few_threads<V>, RG = NT / TC, G = GLU ? 2 : 1;
  extern __shared__ float hs[];             // [k][H] hidden values times their weight, then [k] experts
  __shared__ float red[NT / 32 * TC * V];
  const int tid = threadIdx.x, H = c.H, d = c.d, k = c.k;
  int* const es = reinterpret_cast<int*>(hs + k * H);
  grid_launch_dependents();
  grid_dependency_wait();
  const int64_t t = blockIdx.y, P = c.N * k;
  for (int j = tid; j < k; j += NT) {
    const int e = c.experts[t * k + j];
    es[j] = (unsigned)e < (unsigned)c.E ? e : -1;
  }
  __syncthreads();
  for (int i = tid; i < k * H; i += NT) {
    const int j = i / H, h = i - j * H, e = es[j];
    float v = 0.f;
    if (e >= 0) {
      const float* q = part + (t * k + j) * G * H + h;
      float up = 0.f;
      for (int s = 0; s < splits; ++s, q += P * G * H) {
        v += q[0];
        if (GLU) up += q[H];
      }
      if (c.b1) v += DT<T>::to_f(((const T*)c.b1)[(int64_t)e * H + h]);
      v = activate(v, c.act);
      if (GLU) v *= up;
      v *= c.weights[t * k + j];
    }
    hs[i] = v;
  }
  __syncthreads();
  const int col = blockIdx.x * TC * V + (tid % TC) * V;
  float a[V];
#pragma unroll
  for (int i = 0; i < V; ++i) a[i] = 0.f;
  if (col < d) {
    int j = 0, h = tid / TC;
#pragma unroll 4
    for (int i = tid / TC; i < k * H; i += RG) {
      while (h >= H) h -= H, ++j;
      const int e = es[j];
      if (e >= 0) {
        float f[V];
        load_row<T, V>((const T*)c.w2 + ((int64_t)e * H + h) * d + col, f);
        const float hv = hs[i];
#pragma unroll
        for (int q = 0; q < V; ++q) a[q] = fmaf(hv, f[q], a[q]);
      }
      h += RG;
    }
  }
  float sum = few_sum<V>(a, red);
  const int at = blockIdx.x * TC * V + tid;
  if (tid < TC * V && at < d) {
    if (c.last_bias) sum += DT<T>::to_f(((const T*)c.last_bias)[at]);
    if (c.add_residual) sum += DT<T>::to_f(((const T*)c.x)[t * d + at]);
    ((T*)c.out)[t * d + at] = DT<T>::from_f(sum);
  }
}

// -- host ----------------------------------------------------------------------------------------------------
bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
size_t up256(size_t v) { return (v + 255) / 256 * 256; }

bool takes_few(int64_t P, int d, int H, int k) {
  return P <= 64 && (size_t)k * H * sizeof(float) <= 64 * 1024;
}
int few_splits(int64_t P, int d, int H, int V) {
  const int64_t pieces = P * ceil_div(H, (V == 1 ? 32 : 4) * V);
  return (int)std::max<int64_t>(1, std::min<int64_t>(std::min(16, d / 128), 296 / pieces));
}
constexpr int MOST_SPLITS = 16;

struct Sort {
  int64_t chunk;
  int blocks;
};
Sort sort_shape(int64_t P) {
  if (P <= ONE_BLOCK_PAIRS) return {P, 1};
  const int64_t chunk = (ceil_div64(P, CHUNK_BLOCKS) + NT - 1) / NT * NT;
  return {chunk, (int)ceil_div64(P, chunk)};
}

struct Layout {                             // of the workspace, bytes
  size_t offsets, pairs, table, rows, total;
};
Layout layout_of(int64_t P, int d, int E, int dtype) {
  Layout l;
  l.offsets = 0;
  l.pairs = up256((size_t)(E + 1) * 4);
  l.table = l.pairs + up256((size_t)P * 4);
  l.rows = l.table + up256((size_t)sort_shape(P).blocks * E * 4);
  l.total = l.rows + up256((size_t)P * d * (dtype == D2D_F32 ? 4 : 2));
  return l;
}

template <typename T, int V, bool GLU>
int few(const WeightedCall& c, float* part, cudaStream_t s) {
  const int64_t P = c.N * c.k;
  const int splits = few_splits(P, c.d, c.H, V), cols = few_threads<V> * V;
  const size_t smem = ((size_t)c.k * c.H + c.k) * sizeof(float);
  int rc = device_launch_facts((const void*)few_out_kernel<T, V, GLU>, smem, nullptr);
  if (rc != D2D_OK) return rc;
  rc = launch_pdl(few_hidden_kernel<T, V, GLU>, dim3((unsigned)(ceil_div(c.H, cols) * splits), (unsigned)P), dim3(NT),
                  0, s, c, splits, part);
  if (rc != D2D_OK) return rc;
  return launch_pdl(few_out_kernel<T, V, GLU>, dim3((unsigned)ceil_div(c.d, cols), (unsigned)c.N), dim3(NT), smem, s,
                    c, splits, (const float*)part);
}
template <typename T>
int few_t(const WeightedCall& c, float* part, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  const bool vec = c.H % V == 0 && c.d % V == 0 && al16(c.w1) && al16(c.w_up) && al16(c.w2);
  if (c.w_up) return vec ? few<T, V, true>(c, part, s) : few<T, 1, true>(c, part, s);
  return vec ? few<T, V, false>(c, part, s) : few<T, 1, false>(c, part, s);
}

template <typename T>
int combine_t(const WeightedCall& c, const void* y, int sms, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  const bool vec = c.d % V == 0 && al16(c.x) && al16(c.out) && al16(c.last_bias);
  const int64_t need = ceil_div64(c.N, NT / 32), most = (int64_t)sms * 8;
  const dim3 grid((unsigned)(need < most ? need : most));
  const auto k = vec ? combine_kernel<T, V> : combine_kernel<T, 1>;
  return launch_pdl(k, grid, dim3(NT), 0, s, (const T*)y, c.experts, c.weights, (const T*)c.last_bias,
                    c.add_residual ? (const T*)c.x : nullptr, (T*)c.out, c.N, c.d, c.E, c.k);
}

}  // namespace

size_t weighted_workspace_bytes(int64_t N, int d, int E, int H, int k, bool glu, int dtype) {
  const int64_t P = N * k;
  if (takes_few(P, d, H, k)) return up256((size_t)MOST_SPLITS * P * (glu ? 2 : 1) * H * sizeof(float));
  return layout_of(P, d, E, dtype).total;
}

bool weighted_supported(int64_t N, int d, int E, int H, int k, bool glu, bool tiles) {
  return E <= MAX_E && k <= 32 && N * k < 0x7fffffffLL &&
         (tiles || takes_few(N * k, d, H, k) || experts_simt_fits(H, glu));
}

int launch_weighted(const WeightedCall& c, void* ws, cudaStream_t s) {
  int sms = 0;
  int rc = device_launch_facts(nullptr, 0, &sms);
  if (rc != D2D_OK) return rc;
  const int64_t P = c.N * c.k;
  if (takes_few(P, c.d, c.H, c.k))
    return c.dtype == D2D_F32 ? few_t<float>(c, (float*)ws, s) : few_t<bf16>(c, (float*)ws, s);
  const Layout l = layout_of(P, c.d, c.E, c.dtype);
  uint8_t* const base = (uint8_t*)ws;
  int32_t* const offsets = (int32_t*)(base + l.offsets);
  int32_t* const pairs = (int32_t*)(base + l.pairs);
  int32_t* const table = (int32_t*)(base + l.table);
  void* const rows = base + l.rows;
  const Sort st = sort_shape(P);
  const int threads = st.blocks == 1 ? 1024 : NT;
  if (st.blocks > 1) {
    rc = launch_pdl(pairs_count_kernel, dim3((unsigned)st.blocks), dim3(NT), 0, s, c.experts, P, c.E, st.chunk, table);
    if (rc != D2D_OK) return rc;
  }
  const size_t smem = ((size_t)(threads / 32) * c.E + 3 * (size_t)c.E + 1) * sizeof(int);
  rc = launch_pdl(pairs_scatter_kernel, dim3((unsigned)st.blocks), dim3((unsigned)threads), smem, s, c.experts, P, c.E,
                  st.chunk, st.blocks > 1 ? (const int32_t*)table : nullptr, pairs, offsets, c.dev_status);
  if (rc != D2D_OK) return rc;
  rc = c.packed ? launch_experts_umma_pairs(c.x, pairs, offsets, c.packed, rows, c.N, c.d, c.E, c.H, c.k,
                                            c.w_up != nullptr, c.act, c.dev_status, s)
                : launch_experts_simt_pairs(c.x, pairs, offsets, c.w1, c.b1, c.w_up, c.w2, rows, c.N, c.d, c.E, c.H,
                                            c.k, c.act, c.dtype, c.dev_status, s);
  if (rc != D2D_OK) return rc;
  return c.dtype == D2D_F32 ? combine_t<float>(c, rows, sms, s) : combine_t<bf16>(c, rows, sms, s);
}

}  // namespace d2d
