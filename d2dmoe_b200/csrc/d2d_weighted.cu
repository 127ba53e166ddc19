// Experts weighted by a routing:
//     out[t] = last_bias (+ x[t]) + sum over slots j of w[t, j] y[t, j],   y[t, j] = FFN of expert e[t, j] on x[t]
// with the slots' experts and weights as d2d_route leaves them (expert -1: no such slot).
//
// The upstream layer adds 0/1-routed outputs into one row as they come; here the sum of a token is held in 32 bits,
// taken in the order of its slots and rounded once, so a call gives the same bits every time.  Two ways:
//   lists   The pairs p = t k + j are sorted by expert (counting sort, ascending p in each list), the expert kernels
//           run over the lists and store row p of a table [N k, d], and a last pass sums each token's k rows, which
//           lie together.  That table is what bounds this form: it is written and read once (50432 tokens x 4 x 768:
//           310 MB each way next to 155 MB of x and out).  The tensor-core kernel's rows are 16 bits an
//           element, in a format of its own (encode8) that is off by 2^-14 of the largest of eight where bf16 would be by 2^-8 of each
//           (error of a gated call against 64 bits 2.4e-3 instead of 2.8e-3 of the 2-norm, 1.7e-3 of it the result's own
//           rounding); the fp32 and the general-shape kernel's are fp32.  50432 x 768, 4 of 24 experts: sort 11, experts 112, sum 78 us,
//           each by itself; the call 223.
//   few     Calls of few pairs are bound by latency and by the weights' bytes: two kernels without lists, all
//           sums in 32 bits.  Blocks share out a pair's hidden columns in the first, a token's columns in the second;
//           where those are fewer than the SMs take, clusters split the depth, or the slots, and meet in distributed
//           shared memory.
#include <cooperative_groups.h>

#include <algorithm>

#include "d2d_experts_common.cuh"

namespace d2d {
namespace {

constexpr int NT = 256;
constexpr int MAX_E = 256;

// -- lists of pairs ---------------------------------------------------------------------------------
// Counting sort, stable: every block counts its chunk of the pairs (the first kernel), then, knowing everyone's counts,
// writes it: warps take contiguous parts of the chunk, and pairs of one expert among 32 neighbours rank by lane.  A
// thread's R pairs are loaded at once and stay in registers; calls of one chunk need the second kernel only.
// The table of counts: [blocks][EP], EP = E up to a multiple of 8, 16 bits each (a chunk has 4096 pairs at most).
template <int R>
__device__ __forceinline__ void load_pairs(const int32_t* __restrict__ experts, int64_t p0, int64_t P, int E, int lane,
                                           int (&e)[R], int* dev_status) {
#pragma unroll
  for (int i = 0; i < R; ++i) e[i] = p0 + 32 * i + lane < P ? experts[p0 + 32 * i + lane] : -1;
#pragma unroll
  for (int i = 0; i < R; ++i)
    if ((unsigned)e[i] >= (unsigned)E) {
      if (e[i] != -1) report(dev_status, D2D_ERR_INDEX_RANGE);
      e[i] = -1;
    }
}

template <int R>
__global__ void __launch_bounds__(NT)
pairs_count_kernel(const int32_t* __restrict__ experts, int64_t P, int E, int EP, uint16_t* __restrict__ table) {
  __shared__ int hist[MAX_E];
  grid_launch_dependents();
  grid_dependency_wait();
  fresh(experts);
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int e[R];
  load_pairs<R>(experts, ((int64_t)blockIdx.x * (NT / 32) + w) * 32 * R, P, E, lane, e, nullptr);
  for (int i = threadIdx.x; i < EP; i += NT) hist[i] = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < R; ++i)
    if (e[i] >= 0) atomicAdd(&hist[e[i]], 1);
  __syncthreads();
  for (int i = threadIdx.x; i < EP; i += NT) table[(int64_t)blockIdx.x * EP + i] = (uint16_t)hist[i];
}

// table null: one block
template <int R>
__global__ void __launch_bounds__(NT)
pairs_scatter_kernel(const int32_t* __restrict__ experts, int64_t P, int E, int EP, const uint16_t* __restrict__ table,
                     int32_t* __restrict__ pairs, int32_t* __restrict__ offsets, int* dev_status) {
  constexpr int WARPS = NT / 32;
  __shared__ int count[WARPS][MAX_E];       // a warp's pairs of each expert, then where its next one goes
  __shared__ int total[MAX_E], before[MAX_E], first[MAX_E + 1];
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  grid_launch_dependents();
  for (int i = tid; i < MAX_E; i += NT) {
    total[i] = before[i] = 0;
#pragma unroll
    for (int v = 0; v < WARPS; ++v) count[v][i] = 0;
  }
  grid_dependency_wait();
  fresh(experts, table);
  const int64_t p0 = ((int64_t)blockIdx.x * WARPS + w) * 32 * R;
  int e[R];
  load_pairs<R>(experts, p0, P, E, lane, e, dev_status);
  __syncthreads();
  if (table) {                              // eight experts a thread, as many rows at once as there are threads
    const int per = EP / 8, g = tid % per, rows = NT / per;
    int all[8], early[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) all[i] = early[i] = 0;
    if (tid < rows * per)
#pragma unroll 4
      for (int b = tid / per; b < (int)gridDim.x; b += rows) {
        const uint4 v = *reinterpret_cast<const uint4*>(table + (int64_t)b * EP + 8 * g);
        const uint32_t x[4] = {v.x, v.y, v.z, v.w};
        const bool mine = b < (int)blockIdx.x;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int n = (int)(i & 1 ? x[i / 2] >> 16 : x[i / 2] & 0xffffu);
          all[i] += n;
          early[i] += mine ? n : 0;
        }
      }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (all[i]) atomicAdd(&total[8 * g + i], all[i]);
      if (early[i]) atomicAdd(&before[8 * g + i], early[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < R; ++i)
    if (e[i] >= 0) atomicAdd(&count[w][e[i]], 1);
  __syncthreads();
  if (!table) {
    for (int i = tid; i < E; i += NT) {
      int sum = 0;
#pragma unroll
      for (int v = 0; v < WARPS; ++v) sum += count[v][i];
      total[i] = sum;
    }
    __syncthreads();
  }
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
    for (int i = tid; i <= E; i += NT) offsets[i] = first[i];
  for (int i = tid; i < E; i += NT) {
    int run = first[i] + before[i];
#pragma unroll
    for (int v = 0; v < WARPS; ++v) {
      const int n = count[v][i];
      count[v][i] = run;
      run += n;
    }
  }
  __syncthreads();
  int* const mine = count[w];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const uint32_t same = __match_any_sync(0xffffffffu, e[i]);
    int at = 0;
    if (e[i] >= 0) at = mine[e[i]] + __popc(same & ((1u << lane) - 1u));
    __syncwarp();
    if (e[i] >= 0) {
      pairs[at] = (int)(p0 + 32 * i + lane);
      if ((same >> lane) == 1u) mine[e[i]] = at + 1;      // the last of them
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
template <int V>
__device__ __forceinline__ void load_plain(const float* p, float* f) {
  if constexpr (V == 1) f[0] = *p;
#pragma unroll
  for (int i = 0; i < V / 4; ++i) {
    const float4 a = *(reinterpret_cast<const float4*>(p) + i);
    f[4 * i] = a.x, f[4 * i + 1] = a.y, f[4 * i + 2] = a.z, f[4 * i + 3] = a.w;
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

// The sum's weights of four slots: zero, and no row, where there is no expert.  fours: 16-byte loads
struct Slots {
  float w[4];
  bool there[4];
};
__device__ __forceinline__ Slots load_slots(const int32_t* e, const float* w, int left, int E, bool fours) {
  int4 e4;
  float4 w4;
  if (fours) {
    e4 = *reinterpret_cast<const int4*>(e);
    w4 = *reinterpret_cast<const float4*>(w);
  } else {
    e4 = make_int4(e[0], left > 1 ? e[1] : -1, left > 2 ? e[2] : -1, left > 3 ? e[3] : -1);
    w4 = make_float4(w[0], left > 1 ? w[1] : 0.f, left > 2 ? w[2] : 0.f, left > 3 ? w[3] : 0.f);
  }
  Slots s;
  const int ee[4] = {e4.x, e4.y, e4.z, e4.w};
  const float ww[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    s.there[u] = (unsigned)ee[u] < (unsigned)E;
    s.w[u] = s.there[u] ? ww[u] : 0.f;
  }
  return s;
}
__device__ __forceinline__ bool by_fours(const int32_t* e, const float* w, int k) {
  return k % 4 == 0 && ((reinterpret_cast<uintptr_t>(e) | reinterpret_cast<uintptr_t>(w)) & 15) == 0;
}

// y: [N k, d] fp32.  A thread has V columns of a token; a block takes a few tokens.  per_row: ceil(2^32 / (d / V)), for
// quotients of numbers below 2 NT (where a token has more columns than that, it is the block's only one)
template <typename T, int V>
__global__ void __launch_bounds__(NT)
combine_kernel(const float* __restrict__ y, const int32_t* __restrict__ experts, const float* __restrict__ weights,
               const T* __restrict__ last_bias, const T* __restrict__ x, T* __restrict__ out, int64_t N, int d,
               int E, int k, int tokens, uint32_t per_row) {
  grid_launch_dependents();
  grid_dependency_wait();
  fresh(y, experts, weights, last_bias, x);
  const int nv = d / V;
  const int64_t t0 = (int64_t)blockIdx.x * tokens;
  const int items = (int)min((int64_t)tokens, N - t0) * nv;
  const bool fours = by_fours(experts, weights, k);
  for (int i = threadIdx.x; i < items; i += NT) {
    const int dt = tokens == 1 ? 0 : nv == 1 ? i : (int)__umulhi((uint32_t)i, per_row), c = (i - dt * nv) * V;
    const int64_t t = t0 + dt;
    const float* row = y + t * k * d + c;
    float sum[V], f[V];
#pragma unroll
    for (int q = 0; q < V; ++q) sum[q] = 0.f;
    // (four rows' loads at a time, asked for before the first is used)
    for (int j = 0; j < k; j += 4) {
      const Slots s = load_slots(experts + t * k + j, weights + t * k + j, k - j, E, fours);
      float v[4][V];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
#pragma unroll
        for (int q = 0; q < V; ++q) v[u][q] = 0.f;
        if (s.there[u]) load_plain<V>(row, v[u]);
        row += d;
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int q = 0; q < V; ++q) sum[q] = fmaf(s.w[u], v[u][q], sum[q]);
    }
    if (last_bias) {
      load_row<T, V>(last_bias + c, f);
#pragma unroll
      for (int q = 0; q < V; ++q) sum[q] += f[q];
    }
    if (x) {
      load_row<T, V>(x + t * d + c, f);
#pragma unroll
      for (int q = 0; q < V; ++q) sum[q] += f[q];
    }
    store_row<T, V>(out + t * d + c, sum);
  }
}

// y: [N k, d] in pieces of encode8, which bound this kernel: 310 of 464 MB at 50432 tokens x 4 x 768, 78 us.  A thread has two
// pieces of a token, half a row apart, and goes through the tokens with the grid; the four rows (and x) of its next turn
// travel by cp.async into slots of its own.  (One piece a thread: 94 us, half of it instructions; loads into registers: 101.
// Blocks of 128 threads and 3 or 4 turns ahead, so fewer warps: 84, 104.)
constexpr int COMBINE_NT = 256, COMBINE_STAGES = 2, COMBINE_ROWS = 5;
constexpr size_t COMBINE_SMEM = (size_t)COMBINE_STAGES * COMBINE_ROWS * 2 * COMBINE_NT * 16;
constexpr int COMBINE_BLOCKS = (int)(220 * 1024 / COMBINE_SMEM);       // of an SM
__global__ void __launch_bounds__(COMBINE_NT, COMBINE_BLOCKS)
combine_coded_kernel(const uint16_t* __restrict__ y, const int32_t* __restrict__ experts,
                     const float* __restrict__ weights, const bf16* __restrict__ last_bias, const bf16* __restrict__ x,
                     bf16* __restrict__ out, int64_t N, int d, int E, int k) {
  extern __shared__ __align__(16) uint4 ring[];      // [stage][row][piece][thread]
  grid_launch_dependents();
  grid_dependency_wait();
  fresh(y, experts, weights, last_bias, x);
  constexpr int NT = COMBINE_NT, ROW = 2 * NT;                // uint4 of a row of a stage
  const int nv = d / 16, groups = (k + 3) / 4;
  const bool fours = by_fours(experts, weights, k);
  const int64_t stride = (int64_t)gridDim.x * NT;
  const int dt = (int)(stride / nv), dc = (int)(stride - (int64_t)dt * nv);
  const int64_t first = (int64_t)blockIdx.x * NT + threadIdx.x, t0 = first / nv;
  // A turn: four slots (group g) of token t, columns 16 c ..; what moves with it are pointers.
  struct At {
    int64_t t;
    int c, g;
  };
  At now = {t0, (int)(first - t0 * nv), 0}, ask = now;
  const uint16_t* ask_y = y + t0 * k * d + 8 * ask.c;
  const bf16* ask_x = x ? x + t0 * d + 8 * ask.c : nullptr;
  bf16* to = out + t0 * d + 8 * now.c;
  const int32_t* e = experts + t0 * k;
  const float* w = weights + t0 * k;
  const int64_t dy = (int64_t)dt * k * d + 8 * dc - (int64_t)(groups - 1) * 4 * d;
  const int64_t wrap_y = (int64_t)k * d - d / 2, dx = (int64_t)dt * d + 8 * dc;
  const int ds = dt * k - (groups - 1) * 4;
  uint32_t fill = (uint32_t)__cvta_generic_to_shared(ring + threadIdx.x);
  const uint32_t end = fill + COMBINE_STAGES * COMBINE_ROWS * ROW * 16;
  auto fetch = [&]() {
    if (ask.t < N) {
      const int left = k - 4 * ask.g;
      const uint16_t* row = ask_y;
#pragma unroll
      for (int u = 0; u < 4; ++u, row += d)
        if (u < left)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n\tcp.async.cg.shared.global [%0 + %2], [%3], 16;" ::"r"(
                           fill + u * ROW * 16),
                       "l"(row), "n"(NT * 16), "l"(row + d / 2)
                       : "memory");
      if (x && left <= 4)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n\tcp.async.cg.shared.global [%0 + %2], [%3], 16;" ::"r"(
                         fill + 4 * ROW * 16),
                     "l"(ask_x), "n"(NT * 16), "l"(ask_x + d / 2)
                     : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    fill += COMBINE_ROWS * ROW * 16;
    if (fill >= end) fill -= COMBINE_STAGES * COMBINE_ROWS * ROW * 16;
    if (++ask.g < groups) {
      ask_y += 4 * (int64_t)d;
      return;
    }
    ask.g = 0;
    ask.t += dt;
    ask.c += dc;
    ask_y += dy;
    ask_x += dx;
    if (ask.c >= nv) ask.c -= nv, ++ask.t, ask_y += wrap_y, ask_x += d / 2;
  };
#pragma unroll
  for (int i = 0; i < COMBINE_STAGES - 1; ++i) fetch();
  Slots s = {};
  if (now.t < N) s = load_slots(e, w, k, E, fours);
  const uint4* at = ring + threadIdx.x;
  unsigned long long sum[2][4];
  while (now.t < N) {
    At next = now;
    if (++next.g < groups) {
      e += 4, w += 4;
    } else {
      next.g = 0;
      next.t += dt;
      next.c += dc;
      e += ds, w += ds;
      if (next.c >= nv) next.c -= nv, ++next.t, e += k, w += k;
    }
    Slots s1 = s;                            // the next turn's, asked for now
    if (next.t < N) s1 = load_slots(e, w, k - 4 * next.g, E, fours);
    asm volatile("cp.async.wait_group %0;" ::"n"(COMBINE_STAGES - 2) : "memory");
    uint4 raw[4][2], xr[2];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
#pragma unroll
      for (int u = 0; u < 4; ++u) raw[u][p] = at[u * ROW + p * NT];
      xr[p] = at[4 * ROW + p * NT];
    }
    at += COMBINE_ROWS * ROW;
    if (at >= ring + COMBINE_STAGES * COMBINE_ROWS * ROW) at -= COMBINE_STAGES * COMBINE_ROWS * ROW;
    fetch();
    uint32_t ex[4][2], most = 0u;
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int p = 0; p < 2; ++p) {          // (no expert, no slot: whatever lay there, as finite numbers, times zero)
        ex[u][p] = s.there[u] ? umma::exponent_of(raw[u][p]) : 14u;
        most = max(most, ex[u][p]);
      }
    if (now.g == 0)
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[0][i] = sum[1][i] = 0;
    if (most < 255u) {
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int p = 0; p < 2; ++p) umma::add_decoded8(raw[u][p], ex[u][p], s.w[u] * umma::UNIT8, sum[p]);
    } else {
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          if (ex[u][p] < 255u) umma::add_decoded8(raw[u][p], ex[u][p], s.w[u] * umma::UNIT8, sum[p]);
          else umma::add_special8(raw[u][p], s.w[u], sum[p]);
        }
    }
    if (next.g == 0) {
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        float f[8], b[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) asm("mov.b64 {%0, %1}, %2;" : "=f"(f[2 * i]), "=f"(f[2 * i + 1]) : "l"(sum[p][i]));
        if (last_bias) {
          load_row<bf16, 8>(last_bias + 8 * now.c + p * (d / 2), b);
#pragma unroll
          for (int q = 0; q < 8; ++q) f[q] += b[q];
        }
        if (x) {
          const uint32_t v[4] = {xr[p].x, xr[p].y, xr[p].z, xr[p].w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            f[2 * i] += __uint_as_float(v[i] << 16);
            f[2 * i + 1] += __uint_as_float(v[i] & 0xffff0000u);
          }
        }
        store_row<bf16, 8>(to + p * (d / 2), f);
      }
      to += dx;
      if (next.t > now.t + dt) to += d / 2;
    }
    now = next;
    s = s1;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// -- few pairs ---------------------------------------------------------------------------------------------
// TC threads side by side have V columns each of a block.  Sixteen of 16 bytes where the rows are that long: whole
// 256-byte pieces of a row of the weights (64-byte pieces of W2's 4 KB rows took 14.5 us for one token, 4 MB).
// V sums of each thread over the block's threads of the same columns -> the first TC V threads, in red
template <int V, int TC>
__device__ __forceinline__ float few_sum(float (&v)[V], float* red) {
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

// hidden[p][H]: pair p's hidden values times its weight.  A cluster has TC V of them, its CTAs share the depth and meet in
// distributed shared memory: blockIdx.x = (hidden columns, CTA of the cluster).
template <typename T, int V, int TC, bool GLU>
__global__ void __launch_bounds__(NT)
few_hidden_kernel(WeightedCall c, float* __restrict__ hidden) {
  constexpr int RG = NT / TC;
  __shared__ float red[NT / 32 * TC * V];
  __shared__ float sums[2][TC * V];
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  grid_dependency_wait();
  grid_launch_dependents();                 // behind the wait: the next kernel relies on it
  fresh(c.x, c.experts, c.weights, c.w1, c.b1, c.w_up);
  const int tid = threadIdx.x, H = c.H, d = c.d;
  const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int64_t p = blockIdx.y, t = p / c.k;
  const int e = c.experts[p];
  if ((unsigned)e >= (unsigned)c.E) {       // (all of a cluster)
    if (e != -1 && tid == 0) report(c.dev_status, D2D_ERR_INDEX_RANGE);
    return;
  }
  const int depth = ceil_div(d, ctas), d0 = rank * depth, d1 = min(d, d0 + depth);
  const int col0 = blockIdx.x / ctas * TC * V, col = col0 + (tid % TC) * V;
  const T* const x = (const T*)c.x + t * d;
  const T* const w1 = (const T*)c.w1 + (int64_t)e * d * H + col;
  const T* const wu = GLU ? (const T*)c.w_up + (int64_t)e * d * H + col : nullptr;
  float a[V], u[V];
#pragma unroll
  for (int i = 0; i < V; ++i) a[i] = u[i] = 0.f;
  if (col < H)
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
  float sum = few_sum<V, TC>(a, red), up = GLU ? few_sum<V, TC>(u, red) : 1.f;
  if (ctas > 1) {
    if (tid < TC * V) sums[0][tid] = sum, sums[1][tid] = up;
    cluster.sync();
    if (rank == 0 && tid < TC * V) {
#pragma unroll
      for (int r = 1; r < 8; ++r)
        if (r < ctas) {
          const float* const s = cluster.map_shared_rank(&sums[0][0], r);
          sum += s[tid];
          if (GLU) up += s[TC * V + tid];
        }
    }
  }
  const int h = col0 + tid;
  if (rank == 0 && tid < TC * V && h < H) {
    if (c.b1) sum += DT<T>::to_f(((const T*)c.b1)[(int64_t)e * H + h]);
    hidden[p * H + h] = activate(sum, c.act) * up * c.weights[p];
  }
  if (ctas > 1) cluster.sync();             // the others' sums are read until here
}

// A cluster has TC V columns of a token, a CTA of it `share` slots: blockIdx.x = (columns, CTA of the cluster).
// It starts when every block of the first kernel is past its own wait, so what came before that one is there: experts and W2
// are read ahead of the wait for the hidden values, and the first rows' latency goes by meanwhile.
template <typename T, int V>
struct Raw {
  uint4 v;
  __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void get(float* f) const { load_row<T, V>(reinterpret_cast<const T*>(&v), f); }
};
template <typename T>
struct Raw<T, 1> {
  T v;
  __device__ __forceinline__ void load(const T* p) { v = *p; }
  __device__ __forceinline__ void get(float* f) const { f[0] = DT<T>::to_f(v); }
};
template <typename T, int V, int TC>
__global__ void __launch_bounds__(NT)
few_out_kernel(WeightedCall c, int share, const float* __restrict__ hidden) {
  constexpr int RG = NT / TC, PRE = 8;
  extern __shared__ float hs[];             // [share][H] hidden values, then [share] experts
  __shared__ float red[NT / 32 * TC * V];
  __shared__ float sums[TC * V];
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, H = c.H, d = c.d, k = c.k;
  const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int j0 = rank * share, js = max(0, min(share, k - j0));          // my slots
  int* const es = reinterpret_cast<int*>(hs + share * H);
  grid_launch_dependents();
  const int64_t t = blockIdx.y;
  for (int j = tid; j < js; j += NT) {
    const int e = c.experts[t * k + j0 + j];
    es[j] = (unsigned)e < (unsigned)c.E ? e : -1;
  }
  __syncthreads();
  const int col0 = blockIdx.x / ctas * TC * V, col = col0 + (tid % TC) * V, rows = col < d ? js * H : 0;
  // row r of my slots: hidden column h of slot j
  Raw<T, V> pre[PRE];
  int j = 0, h = tid / TC;
#pragma unroll
  for (int i = 0; i < PRE; ++i) {
    while (h >= H) h -= H, ++j;
    if (tid / TC + i * RG < rows && es[j] >= 0) pre[i].load((const T*)c.w2 + ((int64_t)es[j] * H + h) * d + col);
    h += RG;
  }
  grid_dependency_wait();
  fresh(c.x, c.last_bias, hidden);
  for (int i = tid; i < js * H; i += NT) {
    const bool there = es[i / H] >= 0;
    hs[i] = there ? hidden[(t * k + j0) * H + i] : 0.f;
  }
  __syncthreads();
  float a[V], f[V];
#pragma unroll
  for (int i = 0; i < V; ++i) a[i] = 0.f;
  j = 0, h = tid / TC;
#pragma unroll
  for (int i = 0; i < PRE; ++i) {
    while (h >= H) h -= H, ++j;
    const int r = tid / TC + i * RG;
    if (r < rows && es[j] >= 0) {
      pre[i].get(f);
#pragma unroll
      for (int q = 0; q < V; ++q) a[q] = fmaf(hs[r], f[q], a[q]);
    }
    h += RG;
  }
  while (h >= H) h -= H, ++j;
  for (; j < js && col < d; ++j, h -= H) {
    const int e = es[j];
    if (e < 0) {
      if (h < H) h += (H - h + RG - 1) / RG * RG;
      continue;
    }
    const T* const w2 = (const T*)c.w2 + (int64_t)e * H * d + col;
#pragma unroll 4
    for (; h < H; h += RG) {
      load_row<T, V>(w2 + (int64_t)h * d, f);
      const float hv = hs[j * H + h];
#pragma unroll
      for (int q = 0; q < V; ++q) a[q] = fmaf(hv, f[q], a[q]);
    }
  }
  float sum = few_sum<V, TC>(a, red);
  if (ctas > 1) {
    if (tid < TC * V) sums[tid] = sum;
    cluster.sync();
    if (rank == 0 && tid < TC * V) {
#pragma unroll
      for (int r = 1; r < 8; ++r)
        if (r < ctas) sum += cluster.map_shared_rank(sums, r)[tid];
    }
  }
  const int at = col0 + tid;
  if (rank == 0 && tid < TC * V && at < d) {
    if (c.last_bias) sum += DT<T>::to_f(((const T*)c.last_bias)[at]);
    if (c.add_residual) sum += DT<T>::to_f(((const T*)c.x)[t * d + at]);
    ((T*)c.out)[t * d + at] = DT<T>::from_f(sum);
  }
  if (ctas > 1) cluster.sync();             // the others' sums are read until here
}

// -- host ----------------------------------------------------------------------------------------------------
bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
size_t up256(size_t v) { return (v + 255) / 256 * 256; }

// The first form reads its expert for every pair, out of L2 where all of them fit; lists read each expert once or twice, but
// have three more kernels and wait for a first tile.  Few / lists, us: 2048 x 128 gated, 128 experts (1.6 MB each) 16
// tokens x 8 34 / 58, 37 tokens 59 / 60, 48 tokens 84 / 61; 768 x 128, 24 experts (393 KB) 48 tokens x 4 14 / 17, 64 tokens
// 16.5 / 16.6, 96 tokens 20 / 16.5; 768 x 32 (98 KB) 197 tokens x 4 15 / 21.  fp32, whose lists take the longer the larger an expert
// is: 768 x 128 (786 KB) 96 tokens x 4 31 / 35, 128 tokens 40 / 33; 768 x 32 (197 KB) 197 tokens x 4 25 / 29, 256 tokens 31 / 29;
// 1024 x 512 (4.2 MB) 64 tokens x 2 53 / 75, 128 tokens 96 / 73.  Where lists mean the general-shape kernel the line is that of
// fp32 768 x 128 (256 tokens x 4 74 / 128, 400 tokens 111 / 119), for shapes whose own lines lie on either side of it: bf16
// 130 x 20 682 tokens x 3 25 / 32; bf16 1000 x 100, whose 100 no 16-byte vector divides, 128 tokens x 4 100 / 123, 256 tokens 188 / 168,
// 512 tokens 366 / 171; 1001 x 100 256 tokens 188 / 285, 512 tokens 366 / 304; gated 768 x 128 fp32 256 tokens x 4 96 / 188, 512
// tokens 182 / 204, bf16 without packed weights 512 tokens 117 / 225; gated 2048 x 128 fp32 64 tokens x 8 192 / 554.
bool takes_few(int64_t P, int d, int E, int H, int k, bool glu, int dtype, bool tiles) {
  const int64_t expert = (int64_t)(glu ? 3 : 2) * d * H * (dtype == D2D_F32 ? 4 : 2);
  const bool fp32 = dtype == D2D_F32 && !glu && experts_fp32_pairs_supported(d, E, H);
  const int64_t most = tiles  ? std::max<int64_t>(100 << 20, expert * E * 9 / 4)
                       : fp32 ? (200LL << 20) + 140 * expert
                              : 1100LL << 20;
  return P <= 2048 && P * expert <= most && (size_t)k * H * sizeof(float) <= 64 * 1024;
}

// Pairs of a thread in the sort: 4 up to 256 blocks of 1024 pairs, 16 beyond (fewer rows of counts for every block to add up;
// past a million pairs they grow again).
struct Sort {
  int per_thread, blocks, EP;
};
Sort sort_shape(int64_t P, int E) {
  Sort s;
  s.per_thread = P <= 256 * 4 * NT ? 4 : 16;
  s.blocks = (int)ceil_div64(P, (int64_t)s.per_thread * NT);
  s.EP = (E + 7) / 8 * 8;
  return s;
}

struct Layout {                             // of the workspace, bytes
  size_t offsets, pairs, table, rows, total;
};
// tiles: the tensor-core kernel's rows
Layout layout_of(int64_t P, int d, int E, bool tiles) {
  const Sort s = sort_shape(P, E);
  Layout l;
  l.offsets = 0;
  l.pairs = up256((size_t)(E + 1) * 4);
  l.table = l.pairs + up256((size_t)P * 4);
  l.rows = l.table + up256((size_t)s.blocks * s.EP * 2);
  l.total = l.rows + up256((size_t)P * d * (tiles ? 2 : 4));
  return l;
}

template <typename T, int V, int TC, bool GLU>
int few_hidden(const WeightedCall& c, float* hidden, cudaStream_t s) {
  // CTAs of a cluster: 128 rows of the depth each at least, unless there are blocks enough
  const int64_t P = c.N * c.k;
  const int pieces = ceil_div(c.H, TC * V);
  int ctas = 1;
  while (ctas < 8 && 256 * ctas <= c.d && 2 * ctas * pieces * P <= 592) ctas *= 2;
  return launch_pdl_cluster(ctas, few_hidden_kernel<T, V, TC, GLU>, dim3((unsigned)(pieces * ctas), (unsigned)P), dim3(NT), 0,
                            s, c, hidden);
}
template <typename T, int V, int TC>
int few_out(const WeightedCall& c, const float* hidden, cudaStream_t s) {
  // CTAs of a cluster: a slot each, unless there are blocks enough
  const int pieces = ceil_div(c.d, TC * V);
  int ctas = 1;
  while (ctas < 8 && 2 * ctas <= c.k && 2 * ctas * pieces * c.N <= 592) ctas *= 2;
  const int share = ceil_div(c.k, ctas);
  const size_t smem = ((size_t)share * c.H + share) * sizeof(float);
  const auto k = few_out_kernel<T, V, TC>;
  const int rc = device_launch_facts((const void*)k, smem, nullptr);
  if (rc != D2D_OK) return rc;
  return launch_pdl_cluster(ctas, k, dim3((unsigned)(pieces * ctas), (unsigned)c.N), dim3(NT), smem, s, c, share, hidden);
}
template <typename T, int V>
int few(const WeightedCall& c, float* hidden, cudaStream_t s) {
  constexpr int WIDE = V == 1 ? 32 : 16, NARROW = V == 1 ? 32 : 4;
  const int rc = c.w_up ? few_hidden<T, V, NARROW, true>(c, hidden, s) : few_hidden<T, V, NARROW, false>(c, hidden, s);
  if (rc != D2D_OK) return rc;
  return c.d >= 4 * WIDE * V ? few_out<T, V, WIDE>(c, hidden, s) : few_out<T, V, NARROW>(c, hidden, s);
}
template <typename T>
int few_t(const WeightedCall& c, float* hidden, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  const bool vec = c.H % V == 0 && c.d % V == 0 && al16(c.w1) && al16(c.w_up) && al16(c.w2);
  return vec ? few<T, V>(c, hidden, s) : few<T, 1>(c, hidden, s);
}

template <typename T, int V>
int combine_v(const WeightedCall& c, const void* y, cudaStream_t s) {
  const int nv = c.d / V, tokens = std::max(1, 2 * NT / nv);
  return launch_pdl(combine_kernel<T, V>, dim3((unsigned)ceil_div64(c.N, tokens)), dim3(NT), 0, s, (const float*)y,
                    c.experts, c.weights, (const T*)c.last_bias, c.add_residual ? (const T*)c.x : nullptr, (T*)c.out, c.N,
                    c.d, c.E, c.k, tokens, (uint32_t)((0x100000000ULL + nv - 1) / nv));
}
template <typename T>
int combine_t(const WeightedCall& c, const void* y, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  const bool vec = c.d % V == 0 && al16(c.x) && al16(c.out) && al16(c.last_bias);
  return vec ? combine_v<T, V>(c, y, s) : combine_v<T, 1>(c, y, s);
}
int combine_coded(const WeightedCall& c, const void* y, int sms, cudaStream_t s) {
  const int rc = device_launch_facts((const void*)combine_coded_kernel, COMBINE_SMEM, nullptr);
  if (rc != D2D_OK) return rc;
  const int64_t need = ceil_div64(c.N * (c.d / 16), COMBINE_NT);
  return launch_pdl(combine_coded_kernel, dim3((unsigned)std::min<int64_t>(need, COMBINE_BLOCKS * sms)), dim3(COMBINE_NT),
                    COMBINE_SMEM, s,
                    (const uint16_t*)y, c.experts, c.weights, (const bf16*)c.last_bias,
                    c.add_residual ? (const bf16*)c.x : nullptr, (bf16*)c.out, c.N, c.d, c.E, c.k);
}

}  // namespace

size_t weighted_workspace_bytes(int64_t N, int d, int E, int H, int k, bool glu, int dtype, bool tiles) {
  const int64_t P = N * k;
  if (takes_few(P, d, E, H, k, glu, dtype, tiles)) return up256((size_t)P * H * sizeof(float));
  return layout_of(P, d, E, tiles).total;
}

bool weighted_supported(int64_t N, int d, int E, int H, int k, bool glu, int dtype, bool tiles) {
  return E <= MAX_E && k <= 32 && N * k < 0x7fffffffLL &&
         (tiles || takes_few(N * k, d, E, H, k, glu, dtype, tiles) || experts_simt_fits(H, glu));
}

int launch_weighted(const WeightedCall& c, void* ws, cudaStream_t s) {
  int sms = 0;
  int rc = device_launch_facts(nullptr, 0, &sms);
  if (rc != D2D_OK) return rc;
  const int64_t P = c.N * c.k;
  if (takes_few(P, c.d, c.E, c.H, c.k, c.w_up != nullptr, c.dtype, c.packed != nullptr))
    return c.dtype == D2D_F32 ? few_t<float>(c, (float*)ws, s) : few_t<bf16>(c, (float*)ws, s);
  const Layout l = layout_of(P, c.d, c.E, c.packed != nullptr);
  uint8_t* const base = (uint8_t*)ws;
  int32_t* const offsets = (int32_t*)(base + l.offsets);
  int32_t* const pairs = (int32_t*)(base + l.pairs);
  uint16_t* const table = (uint16_t*)(base + l.table);
  void* const rows = base + l.rows;
  const Sort st = sort_shape(P, c.E);
  const dim3 grid((unsigned)st.blocks);
  if (st.blocks > 1) {
    rc = launch_pdl(st.per_thread == 4 ? pairs_count_kernel<4> : pairs_count_kernel<16>, grid, dim3(NT), 0, s, c.experts,
                    P, c.E, st.EP, table);
    if (rc != D2D_OK) return rc;
  }
  rc = launch_pdl(st.per_thread == 4 ? pairs_scatter_kernel<4> : pairs_scatter_kernel<16>, grid, dim3(NT), 0, s,
                  c.experts, P, c.E, st.EP, st.blocks > 1 ? (const uint16_t*)table : nullptr, pairs, offsets,
                  c.dev_status);
  if (rc != D2D_OK) return rc;
  if (c.packed) {
    rc = launch_experts_umma_pairs(c.x, pairs, offsets, c.packed, rows, c.N, c.d, c.E, c.H, c.k, c.w_up != nullptr,
                                   c.act, c.dev_status, s);
    return rc != D2D_OK ? rc : combine_coded(c, rows, sms, s);
  }
  rc = launch_experts_simt_pairs(c.x, pairs, offsets, c.w1, c.b1, c.w_up, c.w2, rows, c.N, c.d, c.E, c.H, c.k, c.act,
                                 c.dtype, c.dev_status, s);
  if (rc != D2D_OK) return rc;
  return c.dtype == D2D_F32 ? combine_t<float>(c, rows, s) : combine_t<bf16>(c, rows, s);
}

}  // namespace d2d
