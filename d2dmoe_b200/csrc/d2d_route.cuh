// Token-choice routing: scores of the router's logits, the choice of k experts per token, their
// weights; and the gradient of the weights with respect to the logits.
//
//     s = softmax(l) or sigmoid(l)
//     c = s + bias            what the choice goes by (without a bias: l itself, whose order is s's)
//     with groups: the experts are cut into equal groups; a group counts as much as the sum of its two best c (s
//     without a bias), and only experts of the top_groups best ones can be chosen
//     e_1 .. e_k = the k best c, ties to the lowest index
//     w_j = scale * s_{e_j}, or scale * s_{e_j} / sum_i s_{e_i}
// A logit of -inf takes an expert out of the choice (so does a c of -inf); slots that no expert is left for have
// expert -1 and weight 0.  A NaN or +inf among a token's logits or c leaves it without a choice: experts -1,
// weights NaN.
//
// The choice is made as 64 bits make it.  What bounds it is instructions, not bytes: 131072 x 128 bf16 logits take 19.5 us, 6.4 at
// the copy rate, with 58 % of the issue slots busy and the minima and maxima waiting for their pipe.  So it is made on
// 32-bit keys that hold the order in their upper bits and the index in the lower ones:
//   * L lanes have a token; each sorts its keys in batches of KP with a network (Batcher's odd-even merge sort: a
//     minimum and a maximum per exchange) and merges them into a list of its KP best; log2 L butterfly merges
//     make that the token's list in every lane.
//   * The upper bits are less than the number itself.  Where two neighbours of the list, or its last one and the
//     best that is not in it, are nearer than the keys and the arithmetic before them can tell, the
//     whole warp makes that token's choice again in 64 bits.  bf16 logits without a bias fit into the
//     upper bits and never need it.
// Scores for the choice may therefore come from the fast exponential, and so do weights that are a share of its sum
// over all experts (2 ulp); renormalised and sigmoid weights come from the accurate one.
#pragma once
#include <algorithm>

#include "d2d_common.cuh"

namespace d2d {
namespace {

constexpr int NT = 128;                    // threads of a block
constexpr int WARPS = NT / 32;
static_assert(ROUTE_MAX_E <= 1024 && ROUTE_MAX_K <= 32 && ROUTE_MAX_GROUPS <= 32, "lanes, bits and magic numbers below");
constexpr float MAX_FINITE = 3.402823466e38f;

struct RouteArgs {
  const void* logits;
  const float* bias;
  int32_t* experts;
  float* weights;
  uint32_t* mask_bits;                     // optional
  void* dense;                             // optional: [N, E] weights in T
  int64_t N;
  int E, k, groups, top_groups;
  bool softmax, renormalise;
  float scale;
  int room;                                // shared memory of a warp, bytes
  bool bias_vectors;                       // the bias allows 16-byte loads
  uint32_t group_magic;                    // e group_magic >> 22 = e / (E / groups) for e < 1024
};

__device__ __forceinline__ bool unusable(float v) { return !(v <= MAX_FINITE); }      // NaN, +inf

__device__ __forceinline__ float sigmoidf(float l) { return 1.f / (1.f + expf(-l)); }
// sigmoid(l) e^-m for m <= 0 and the largest l of those whose quotients are wanted, or 0: as large as they are, none underflows
__device__ __forceinline__ float scaled_sigmoid(float l, float m) {
  return (l < 0.f ? expf(l - m) : 1.f) / (1.f + expf(-fabsf(l)));
}

constexpr float LOG2E = 1.44269504088896340736f;
__device__ __forceinline__ float exp2_fast(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float reciprocal_fast(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// e^(l - m): 2 ulp and |l - m| half ulps off
__device__ __forceinline__ float softmax_term(float l, float m) { return exp2_fast((l - m) * LOG2E); }

// -- what a choice gives: lane q of the L that have token t holds slots q, q + L, .. (e < 0: none) --------------
// (the shuffles are for whole warps: a token that is not there, or made again, goes along with write = false)
template <typename T, int L, int R>
__device__ __forceinline__ void put_choice(const RouteArgs& a, int64_t t, int q, const int (&e)[R], bool bad,
                                           float m, float denom, bool write = true) {
  const T* row = reinterpret_cast<const T*>(a.logits) + t * a.E;
  float l[R], w[R], mx = -INFINITY;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    l[r] = e[r] >= 0 ? DT<T>::to_f(row[e[r]]) : -INFINITY;
    mx = fmaxf(mx, l[r]);
  }
  if (a.renormalise) {
#pragma unroll
    for (int o = 1; o < L; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  }
  float sum = 0.f;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    w[r] = e[r] < 0         ? 0.f
           : !a.renormalise ? (a.softmax ? softmax_term(l[r], m) / denom : sigmoidf(l[r]))
           : a.softmax      ? expf(l[r] - mx)
                            : scaled_sigmoid(l[r], fminf(mx, 0.f));
    sum += w[r];
  }
  if (a.renormalise) {
#pragma unroll
    for (int o = 1; o < L; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int j = q + L * r;
    if (a.renormalise && e[r] >= 0) w[r] /= sum;
    w[r] = bad ? __int_as_float(0x7fc00000) : w[r] * a.scale;
    if (write && j < a.k) {
      a.experts[t * a.k + j] = e[r];
      a.weights[t * a.k + j] = w[r];
    }
  }
  if (a.dense) {
    T* to = reinterpret_cast<T*>(a.dense) + t * a.E;
    if (write)
      for (int i = q; i < a.E; i += L) to[i] = DT<T>::from_f(0.f);
    __syncwarp();
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (write && e[r] >= 0) to[e[r]] = DT<T>::from_f(w[r]);
  }
}

// -- one token by a whole warp, in 64 bits ------------------------------------------------------------------------
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// c: room for E numbers of this warp
template <typename T>
__device__ __noinline__ void route_exact(const RouteArgs a, int64_t t, double* c, int lane) {
  const T* row = reinterpret_cast<const T*>(a.logits) + t * a.E;
  const double none = -INFINITY;
  const int E = a.E;
  const bool scored = a.bias != nullptr || a.groups > 1 || (a.softmax && !a.renormalise);
  float m = -INFINITY;
  bool bad = false;
  for (int e = lane; e < E; e += 32) {
    const float l = DT<T>::to_f(row[e]);
    bad |= unusable(l) || (a.bias && unusable(a.bias[e]));
    m = fmaxf(m, l);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  bad = __any_sync(0xffffffffu, bad);
  const bool empty = bad || m == -INFINITY;
  double total = 1.0;
  float denom = 1.f;                       // of the weights: of their own exponentials
  if (scored && a.softmax && !empty) {
    total = 0.0;
    denom = 0.f;
    for (int e = lane; e < E; e += 32) {
      const float l = DT<T>::to_f(row[e]);
      total += exp((double)l - (double)m);
      denom += softmax_term(l, m);
    }
    total = warp_sum(total);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) denom += __shfl_xor_sync(0xffffffffu, denom, o);
  }
  __syncwarp();
  for (int e = lane; e < E; e += 32) {
    const float l = DT<T>::to_f(row[e]);
    double v = none;
    if (!empty && l > -INFINITY) {
      if (a.bias || a.groups > 1) {
        v = a.softmax ? exp((double)l - (double)m) / total : 1.0 / (1.0 + exp(-(double)l));
        if (a.bias) v += (double)a.bias[e];
      } else {
        v = l;
      }
    }
    c[e] = v;
  }
  __syncwarp();
  if (a.groups > 1) {
    const int size = E / a.groups;
    double best = none, second = none;
    if (lane < a.groups)
      for (int i = 0; i < size; ++i) {
        const double v = c[lane * size + i];
        if (v > best) second = best, best = v;
        else if (v > second) second = v;
      }
    // (a group of one, or with one that can be chosen, counts as that one)
    const double v = second > none ? best + second : best;
    int before = 0;
    for (int g = 0; g < a.groups; ++g) {
      const double u = __shfl_sync(0xffffffffu, v, g);
      before += u > v || (u == v && g < lane);
    }
    const uint32_t kept = __ballot_sync(0xffffffffu, lane < a.groups && before < a.top_groups);
    __syncwarp();
    for (int e = lane; e < E; e += 32) {
      if (!(kept >> (e / size) & 1u)) c[e] = none;
      else if (!a.bias && c[e] > none) c[e] = DT<T>::to_f(row[e]);      // in the order of the logits
    }
    __syncwarp();
  }
  int mine[1] = {-1};
  for (int j = 0; j < a.k; ++j) {
    double best = none;
    int at = 0x7fffffff;
    for (int e = lane; e < E; e += 32)
      if (c[e] > best) best = c[e], at = e;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const double v = __shfl_xor_sync(0xffffffffu, best, o);
      const int e = __shfl_xor_sync(0xffffffffu, at, o);
      if (v > best || (v == best && e < at)) best = v, at = e;
    }
    if (at == 0x7fffffff) break;           // nothing is left
    if (lane == j) mine[0] = at;
    if ((at & 31) == lane) c[at] = none;
    __syncwarp();
  }
  if (a.mask_bits)
    for (int w = 0; w < (E + 31) / 32; ++w) {
      const uint32_t bits = mine[0] >= 0 && (mine[0] >> 5) == w ? 1u << (mine[0] & 31) : 0u;
      const uint32_t all = __reduce_or_sync(0xffffffffu, bits);
      if (lane == 0) a.mask_bits[t * ((E + 31) / 32) + w] = all;
    }
  put_choice<T, 32, 1>(a, t, lane, mine, bad, m, denom);
  __syncwarp();
}

template <typename T>
__global__ void __launch_bounds__(NT) route_exact_kernel(RouteArgs a) {
  extern __shared__ __align__(16) double scratch[];
  grid_launch_dependents();
  grid_dependency_wait();
  fresh(a.logits, a.bias);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int64_t t = (int64_t)blockIdx.x * WARPS + warp; t < a.N; t += (int64_t)gridDim.x * WARPS)
    route_exact<T>(a, t, scratch + (size_t)warp * a.E, lane);
}

// -- sorted lists of keys, the largest first --------------------------------------------------------------------------
__device__ __forceinline__ void exchange(uint32_t& hi, uint32_t& lo) {
  const uint32_t x = max(hi, lo);
  lo = min(hi, lo);
  hi = x;
}
template <int K>
__device__ __forceinline__ void sort_keys(uint32_t* v) {
#pragma unroll
  for (int p = 1; p < K; p *= 2)
#pragma unroll
    for (int s = p; s >= 1; s /= 2)
#pragma unroll
      for (int j = s % p; j + s < K; j += 2 * s)
#pragma unroll
        for (int i = 0; i < s; ++i)
          if (i + j + s < K && (i + j) / (2 * p) == (i + j + s) / (2 * p)) exchange(v[i + j], v[i + j + s]);
}
// list = the K best of list and other (both sorted)
template <int K>
__device__ __forceinline__ void merge_keys(uint32_t (&list)[K], const uint32_t* other) {
#pragma unroll
  for (int i = 0; i < K; ++i) list[i] = max(list[i], other[K - 1 - i]);
#pragma unroll
  for (int s = K / 2; s >= 1; s /= 2)
#pragma unroll
    for (int i = 0; i < K; ++i)
      if ((i & s) == 0) exchange(list[i], list[i + s]);
}

// -- a lane's share of a row ----------------------------------------------------------------------------------------------
// EL logits: vectors q, q + L, .. of V each.  bf16 vectors stay packed pairs.
template <typename T, int V, int L, int EL>
struct Row {
  static constexpr bool PACKED = sizeof(T) == 2 && V == 8;
  static constexpr int WORDS = PACKED ? EL / 2 : EL;
  uint32_t w[WORDS];
  __device__ __forceinline__ static int expert(int i, int q) { return (i / V * L + q) * V + i % V; }
  __device__ __forceinline__ void load(const T* row, int E, int q, bool in) {
#pragma unroll
    for (int v = 0; v < EL / V; ++v) {
      const int e = (v * L + q) * V;
      const bool there = in && e < E;
      if constexpr (PACKED) {
        const uint4 x = there ? *reinterpret_cast<const uint4*>(row + e)
                              : make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u);      // -inf
        w[4 * v] = x.x, w[4 * v + 1] = x.y, w[4 * v + 2] = x.z, w[4 * v + 3] = x.w;
      } else if constexpr (V == 4) {
        const uint4 x = there ? *reinterpret_cast<const uint4*>(row + e)
                              : make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u);
        w[4 * v] = x.x, w[4 * v + 1] = x.y, w[4 * v + 2] = x.z, w[4 * v + 3] = x.w;
      } else {
        w[v] = there ? __float_as_uint(DT<T>::to_f(row[e])) : 0xff800000u;
      }
    }
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (PACKED) return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    else return __uint_as_float(w[i]);
  }
  // the largest, NaN if there is one
  __device__ __forceinline__ float largest() const {
    if constexpr (PACKED) {
      uint32_t m = w[0];
#pragma unroll
      for (int i = 1; i < WORDS; ++i) asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(m) : "r"(m), "r"(w[i]));
      return max_nan(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u));
    } else {
      float m = __uint_as_float(w[0]);
#pragma unroll
      for (int i = 1; i < WORDS; ++i) m = max_nan(m, __uint_as_float(w[i]));
      return m;
    }
  }
  // Keys in the order of the logits: ordered logit, its `low` bits replaced by those of ~expert.  -inf (and what is not
  // there) is below NO_KEY.  Adding +0 makes one of both zeros, which are equal.
  __device__ __forceinline__ void keys(uint32_t* key, uint32_t low, int q) const {
    if constexpr (PACKED) {
#pragma unroll
      for (int i = 0; i < WORDS; ++i) {
        uint32_t l, sign;                                                    // of each half, all over it
        asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(l) : "r"(w[i]), "r"(0u));
        asm("prmt.b32 %0, %1, 0, 0xbb99;" : "=r"(sign) : "r"(l));
        const uint32_t o = l ^ (sign | 0x80008000u);
        const uint32_t e = ~(uint32_t)expert(2 * i, q);                      // (2 i + 1: one less)
        key[2 * i] = o << 16 | (e & low);
        key[2 * i + 1] = (o & 0xffff0000u) | ((e - 1u) & low);
      }
    } else {
#pragma unroll
      for (int i = 0; i < EL; ++i) {
        const uint32_t e = (uint32_t)expert(i, q), l = __float_as_uint(__fadd_rn(__uint_as_float(w[i]), 0.f));
        const uint32_t o = l ^ (0x80000000u | (uint32_t)((int32_t)l >> 31));
        key[i] = (o & ~low) | (~e & low);
      }
    }
  }
  // all bits that are set in any logit
  __device__ __forceinline__ uint32_t bits() const {
    uint32_t b = 0u;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < WORDS; ++i) b |= w[i];
    }
    return b;
  }
};
constexpr uint32_t NO_KEY = 0x00800000u;       // of ordered logits: those of -inf are below

template <int L>
__device__ __forceinline__ float sum_lanes(float v) {
#pragma unroll
  for (int o = 1; o < L; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <int L>
__device__ __forceinline__ float max_lanes(float v) {       // NaN if there is one
#pragma unroll
  for (int o = 1; o < L; o <<= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

enum Mode {
  ORDER,        // the order of the logits is all there is to it
  TOTAL,        // and the weights are softmax over all experts
  SCORED        // the choice goes by scores
};

// two best of each vector of V numbers
template <int V>
__device__ __forceinline__ float2 two_best(const float* c) {
  float best = c[0], second = -INFINITY;
#pragma unroll
  for (int i = 1; i < V; ++i) {
    second = fmaxf(second, fminf(best, c[i]));
    best = fmaxf(best, c[i]);
  }
  return make_float2(best, second);
}

// L lanes per token, EL logits per lane, lists of KP keys; V logits per load.
template <typename T, int V, int L, int EL, int KP, int MODE>
__global__ void __launch_bounds__(NT, KP == 16 ? 4 : MODE == ORDER ? (EL == 32 ? 6 : 8) : EL == 32 ? 4 : MODE == TOTAL ? 8 : 6) route_kernel(RouteArgs a) {
  extern __shared__ __align__(16) double scratch[];
  constexpr int TOKENS = 32 / L;           // of a warp at once
  constexpr int R = (KP + L - 1) / L;
  grid_launch_dependents();
  grid_dependency_wait();
  fresh(a.logits, a.bias);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, q = lane % L, mine = lane / L;
  const int E = a.E, k = a.k;
  double* const wide = scratch + (size_t)warp * (a.room / 8);
  const int index_bits = E <= 2 ? 1 : 32 - __clz(E - 1);
  const uint32_t low = (1u << index_bits) - 1u;
  const int64_t steps = ceil_div64(a.N, (int64_t)WARPS * TOKENS);
  for (int64_t step = blockIdx.x; step < steps; step += gridDim.x) {
    const int64_t t = (step * WARPS + warp) * TOKENS + mine;
    const bool in = t < a.N;
    Row<T, V, L, EL> row;
    row.load(reinterpret_cast<const T*>(a.logits) + t * E, E, q, in);
    const float m = max_lanes<L>(row.largest());
    bool bad = unusable(m);
    float denom = 1.f;
    uint32_t key[EL];
    uint32_t near = 0;                     // keys that differ by this much in their upper bits may be in any order
    uint32_t least = NO_KEY;               // keys below are none
    bool unsure = false;                   // this token's choice is made again in 64 bits
    if constexpr (MODE != SCORED) {
      row.keys(key, low, q);
      if constexpr (MODE == TOTAL) {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < EL; ++i) sum += softmax_term(row.get(i), m);
        denom = sum_lanes<L>(sum);
      }
    } else {
      float c[EL];
      if (a.softmax) {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < EL; ++i) sum += c[i] = softmax_term(row.get(i), m);
        denom = sum_lanes<L>(sum);
        const float inv = 1.f / denom;
#pragma unroll
        for (int i = 0; i < EL; ++i) c[i] *= inv;
      } else {
#pragma unroll
        for (int i = 0; i < EL; ++i)
          c[i] = reciprocal_fast(1.f + exp2_fast(fminf(row.get(i) * -LOG2E, 120.f)));
      }
      if (a.bias) {
        float worst = 0.f;
#pragma unroll
        for (int v = 0; v < EL / V; ++v) {
          const int e = (v * L + q) * V;
          if (e >= E) continue;
          float b[V];
          if (V > 1 && a.bias_vectors) {
#pragma unroll
            for (int i = 0; i < V / 4; ++i) {
              const float4 x = __ldg(reinterpret_cast<const float4*>(a.bias + e) + i);
              b[4 * i] = x.x, b[4 * i + 1] = x.y, b[4 * i + 2] = x.z, b[4 * i + 3] = x.w;
            }
          } else {
#pragma unroll
            for (int i = 0; i < V; ++i) b[i] = __ldg(a.bias + e + i);
          }
#pragma unroll
          for (int i = 0; i < V; ++i) {
            worst = max_nan(worst, b[i]);
            c[v * V + i] += b[i];
          }
        }
        bad |= unusable(max_lanes<L>(worst));
      }
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < EL; ++i) {
        if (row.get(i) == -INFINITY) c[i] = -INFINITY;
        top = fmaxf(top, c[i]);
      }
      top = max_lanes<L>(top);
      const int size = E / a.groups;
      if (a.groups > 1) {
        // The two best of each group by the token's lanes, one group each, from shared memory: out of the two best of each
        // vector where a vector lies in one group, else out of all.
        float* const rows = reinterpret_cast<float*>(wide) + mine * (2 * E + 2 * a.groups);
        float* const value = rows + 2 * E;
        const bool whole = V > 1 && size % V == 0;
        __syncwarp();
#pragma unroll
        for (int v = 0; v < EL / V; ++v) {
          const int e = (v * L + q) * V;
          if (e < E) {
            if (whole) {
              *reinterpret_cast<float2*>(rows + 2 * (e / V)) = two_best<V>(c + v * V);
            } else {
#pragma unroll
              for (int i = 0; i < V; ++i) *reinterpret_cast<float2*>(rows + 2 * (e + i)) = make_float2(c[v * V + i], -INFINITY);
            }
          }
        }
        __syncwarp();
        const int n = whole ? size / V : size;
        for (int g = q; g < a.groups; g += L) {
          float best = -INFINITY, second = -INFINITY;
          int at = lane % n;               // (another bank for each lane)
#pragma unroll 4
          for (int i = 0; i < n; ++i) {
            const float2 v = *reinterpret_cast<const float2*>(rows + 2 * (g * n + at));
            second = fmaxf(fmaxf(second, v.y), fminf(best, v.x));
            best = fmaxf(best, v.x);
            at = at + 1 == n ? 0 : at + 1;
          }
          value[g] = second > -INFINITY ? best + second : best;
          // How far that can be off: the bound of single scores, below, for both and their sum.  It goes by their size, which
          // cancels in the sum.  (No expert left: nothing to be off; a sum that is not finite is not known at all.)
          const float most = fmaxf(fabsf(best), second > -INFINITY ? fabsf(second) : 0.f);
          value[a.groups + g] = best > -INFINITY ? fmaf(most, 5e-7f, 6e-6f) : 0.f;
        }
        __syncwarp();
        uint32_t kept = 0u;
        float worst = INFINITY, other = -INFINITY;       // the least a kept group can be, the most another one
        for (int g = q; g < a.groups; g += L) {
          const float v = value[g], off = value[a.groups + g];
          int before = 0;
#pragma unroll 4
          for (int h = 0; h < a.groups; ++h) {
            const float u = value[h];
            before += u > v || (u == v && h < g);
          }
          if (before < a.top_groups) {
            kept |= 1u << g;
            worst = fminf(worst, v - off);
          } else if (off > 0.f) {
            other = fmaxf(other, fmaxf(v + off, -MAX_FINITE));
          }
        }
#pragma unroll
        for (int o = 1; o < L; o <<= 1) {
          kept |= __shfl_xor_sync(0xffffffffu, kept, o);
          worst = fminf(worst, __shfl_xor_sync(0xffffffffu, worst, o));
          other = fmaxf(other, __shfl_xor_sync(0xffffffffu, other, o));
        }
        unsure = other > -INFINITY && !(worst > other);
#pragma unroll
        for (int v = 0; v < EL / V; ++v) {
          const int e = (v * L + q) * V;
          if (whole) {
            const bool drop = (kept >> (e * a.group_magic >> 22) & 1u) == 0u;
#pragma unroll
            for (int i = 0; i < V; ++i) c[v * V + i] = drop ? -INFINITY : c[v * V + i];
          } else {
#pragma unroll
            for (int i = 0; i < V; ++i)
              if ((kept >> ((e + i) * a.group_magic >> 22) & 1u) == 0u) c[v * V + i] = -INFINITY;
          }
        }
      }
      if (a.bias) {
        // How far two c in the wrong order can be apart: the exponentials and reciprocals of each are off by 3e-7 at most, a
        // softmax's sum (37 roundings, the same for all) by 2.2e-6 of the difference of two scores, the
        // sums with the bias by half an ulp, 6e-8 (4 + |largest c|) each, the keys' own rounding by 2.4e-7 each: less than
        // 5e-6 + 1.2e-7 |largest c|.  Keys take the range of 4 below the largest c in steps of
        // 2^(2 + index bits - 32); what lies lower has the lowest key.
        const float scale = (float)(1u << (30 - index_bits)), zero = (4.f - top) * scale;
        const uint32_t most = 0xffffffffu >> index_bits;
        near = (uint32_t)fminf((6e-6f + 5e-7f * fabsf(top)) * scale, 1e9f) + 2u;
        least = 1u << index_bits;
#pragma unroll
        for (int i = 0; i < EL; ++i) {
          const uint32_t e = (uint32_t)row.expert(i, q);
          const uint32_t u = __float2uint_rz(fmaf(c[i], scale, zero));       // (below zero: 0)
          key[i] = c[i] > -INFINITY ? min(max(u, 1u), most) << index_bits | (~e & low) : 0u;
        }
      } else {
        row.keys(key, low, q);
#pragma unroll
        for (int i = 0; i < EL; ++i) key[i] = c[i] > -INFINITY ? key[i] : 0u;
      }
    }

    uint32_t list[KP];
    {
      uint32_t other[KP];
#pragma unroll
      for (int b = 0; b < EL / KP; ++b) {
#pragma unroll
        for (int i = 0; i < KP; ++i) other[i] = key[b * KP + i];
        sort_keys<KP>(other);
        if (b == 0) {
#pragma unroll
          for (int i = 0; i < KP; ++i) list[i] = other[i];
        } else {
          merge_keys<KP>(list, other);
        }
      }
#pragma unroll
      for (int o = 1; o < L; o <<= 1) {
#pragma unroll
        for (int i = 0; i < KP; ++i) other[i] = __shfl_xor_sync(0xffffffffu, list[i], o);
        merge_keys<KP>(list, other);
      }
    }
    // What the keys cannot tell apart.  (fp32 logits whose low bits are all zero have lost nothing: equal upper
    // bits are equal logits, and the index decides.)
    if (sizeof(T) == 4 || (MODE == SCORED && a.bias)) {
      bool lossy = MODE == SCORED && a.bias;
      if (!lossy) {
        uint32_t seen = row.bits() & low;
#pragma unroll
        for (int o = 1; o < L; o <<= 1) seen |= __shfl_xor_sync(0xffffffffu, seen, o);
        lossy = seen != 0u;
      }
      uint32_t last = 0;
      bool close = false;
#pragma unroll
      for (int i = 0; i < KP; ++i) {
        if (i + 1 < KP && i < k && list[i + 1] >= least)
          close |= (list[i] >> index_bits) - (list[i + 1] >> index_bits) <= near;
        if (i == k - 1) last = list[i];
      }
      if (k == KP) {                       // the best that is not in the list (whole warps: k is everyone's)
        const uint32_t bound = last >> index_bits, from = bound > near ? bound - near : 0u;
        int n = 0;
#pragma unroll
        for (int i = 0; i < EL; ++i) n += key[i] >= least && (key[i] >> index_bits) >= from;
#pragma unroll
        for (int o = 1; o < L; o <<= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
        close |= last >= least && n > k;
      }
      unsure |= lossy && close;
    }
    unsure = unsure && in && !bad;
    const bool write = in && !unsure;
    int e[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      uint32_t x = 0u;
#pragma unroll
      for (int i = 0; i < L && i + L * r < KP; ++i)
        if (q == i) x = list[i + L * r];
      e[r] = x < least || bad || !write || q + L * r >= k ? -1 : (int)(~x & low);
    }
    if (write && a.mask_bits) {
      const int nw = (E + 31) / 32;
      for (int w = q; w < nw; w += L) {
        uint32_t bits = 0u;
#pragma unroll
        for (int i = 0; i < KP; ++i) {
          const uint32_t x = ~list[i] & low;
          if (i < k && list[i] >= least && !bad && (int)(x >> 5) == w) bits |= 1u << (x & 31);
        }
        a.mask_bits[t * nw + w] = bits;
      }
    }
    put_choice<T, L, R>(a, in ? t : 0, q, e, bad, m, denom, write);
    uint32_t again = __ballot_sync(0xffffffffu, unsure && q == 0);
    while (again != 0u) {
      const int from = __ffs(again) - 1;
      again &= again - 1u;
      __syncwarp();
      route_exact<T>(a, (step * WARPS + warp) * TOKENS + from / L, wide, lane);
    }
  }
}

// -- gradient --------------------------------------------------------------------------------------------------------------
// With g_j = scale dw_j and p_j = w_j / scale, over the slots that have an expert:
//   softmax, renormalised   dl_{e_j} = p_j (g_j - sum_i p_i g_i)                 zero elsewhere
//   sigmoid, renormalised   dl_{e_j} = p_j (1 - s_{e_j}) (g_j - sum_i p_i g_i)   zero elsewhere
//   sigmoid                 dl_{e_j} = g_j s_{e_j} (1 - s_{e_j})                 zero elsewhere
//   softmax                 dl_e = s_e (sum_{j: e_j = e} g_j - sum_j s_{e_j} g_j)
// The choice itself has no gradient, nor has its bias.  L lanes have a token; the slots' shares meet in its row of
// shared memory, from which the row of dlogits is written in vectors.  The kernel's bytes are the rows', read
// (softmax over all) and written.
struct BackwardArgs {
  const void* logits;
  const int32_t* experts;
  const float *weights, *dweights;
  void* dlogits;
  int64_t N;
  int E, k;
  bool softmax, renormalise;
  float scale;
};

template <typename T, int V, int L, int EL>
__global__ void __launch_bounds__(NT, EL == 16 ? 8 : 4) route_backward_kernel(BackwardArgs a) {
  extern __shared__ __align__(16) double scratch[];
  constexpr int TOKENS = 32 / L;
  grid_launch_dependents();
  grid_dependency_wait();
  fresh(a.logits, a.experts, a.weights, a.dweights);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, q = lane % L, mine = lane / L;
  const int E = a.E, EP = (E + 3) / 4 * 4;
  float* const share = reinterpret_cast<float*>(scratch) + (size_t)(warp * TOKENS + mine) * EP;
  const float inv = 1.f / a.scale;
  const bool all = a.softmax && !a.renormalise;
  for (int i = q; i < EP; i += L) share[i] = 0.f;
  __syncwarp();
  const int64_t steps = ceil_div64(a.N, (int64_t)WARPS * TOKENS);
  for (int64_t step = blockIdx.x; step < steps; step += gridDim.x) {
    const int64_t t = (step * WARPS + warp) * TOKENS + mine;
    const bool in = t < a.N;
    const T* const l = reinterpret_cast<const T*>(a.logits) + t * E;
    T* const to = reinterpret_cast<T*>(a.dlogits) + t * E;
    Row<T, V, L, EL> row;
    if (all) row.load(l, E, q, in);
    // a lane's slots: the first stays in registers, the others (k > L) are read again
    struct Slot {
      int e;
      float g, p;
    };
    auto slot = [&](int j) {
      Slot v = {in && j < a.k ? a.experts[t * a.k + j] : -1, 0.f, 0.f};
      if ((unsigned)v.e >= (unsigned)E) {
        v.e = -1;
      } else {
        v.g = a.scale * a.dweights[t * a.k + j];
        v.p = a.weights[t * a.k + j] * inv;
      }
      return v;
    };
    const Slot mine0 = slot(q);
    float dot = 0.f;
    bool any = mine0.e >= 0;
    if (a.renormalise || a.softmax) {
      dot = mine0.p * mine0.g;
      for (int j = q + L; j < a.k; j += L) {
        const Slot v = slot(j);
        any |= v.e >= 0;
        dot = fmaf(v.p, v.g, dot);
      }
      dot = sum_lanes<L>(dot);
    }
    auto put = [&](const Slot& v) {
      if (v.e < 0) return;
      float d = a.renormalise ? v.p * (v.g - dot) : all ? v.g : v.p * v.g;
      if (!a.softmax) d *= 1.f / (1.f + expf(DT<T>::to_f(l[v.e])));          // 1 - sigmoid
      atomicAdd(&share[v.e], d);           // (an expert that is there twice has both shares)
    };
    put(mine0);
    for (int j = q + L; j < a.k; j += L) put(slot(j));
    __syncwarp();
    if (all) {
      const float m = max_lanes<L>(row.largest());
      float s[EL], sum = 0.f;
#pragma unroll
      for (int i = 0; i < EL; ++i) sum += s[i] = softmax_term(row.get(i), m);
      sum = sum_lanes<L>(sum);
      const bool chosen = sum_lanes<L>(any ? 1.f : 0.f) > 0.f;
      const float is = 1.f / sum;
#pragma unroll
      for (int v = 0; v < EL / V; ++v) {
        const int e = (v * L + q) * V;
        if (!in || e >= E) continue;
        float d[V];
        if constexpr (V == 1) {
          d[0] = share[e];
        } else {
#pragma unroll
          for (int i = 0; i < V / 4; ++i) {
            const float4 x = *(reinterpret_cast<const float4*>(share + e) + i);
            d[4 * i] = x.x, d[4 * i + 1] = x.y, d[4 * i + 2] = x.z, d[4 * i + 3] = x.w;
          }
        }
#pragma unroll
        for (int i = 0; i < V; ++i) d[i] = chosen ? s[v * V + i] * is * (d[i] - dot) : 0.f;
        if constexpr (V == 1) to[e] = DT<T>::from_f(d[0]);
        else if constexpr (V == 4) *reinterpret_cast<float4*>(to + e) = make_float4(d[0], d[1], d[2], d[3]);
        else
          *reinterpret_cast<uint4*>(to + e) = make_uint4(pack_bf16x2(d[0], d[1]), pack_bf16x2(d[2], d[3]),
                                                         pack_bf16x2(d[4], d[5]), pack_bf16x2(d[6], d[7]));
      }
    } else {
      for (int e = q * V; e < E && in; e += L * V) {
        if constexpr (V == 1) {
          to[e] = DT<T>::from_f(share[e]);
        } else {
          float4 d[V / 4];
#pragma unroll
          for (int i = 0; i < V / 4; ++i) d[i] = *(reinterpret_cast<const float4*>(share + e) + i);
          if constexpr (V == 4)
            *reinterpret_cast<float4*>(to + e) = d[0];
          else
            *reinterpret_cast<uint4*>(to + e) = make_uint4(pack_bf16x2(d[0].x, d[0].y), pack_bf16x2(d[0].z, d[0].w),
                                                           pack_bf16x2(d[1].x, d[1].y), pack_bf16x2(d[1].z, d[1].w));
        }
      }
    }
    __syncwarp();
    // back to zero, where something was
    if (mine0.e >= 0) share[mine0.e] = 0.f;
    for (int j = q + L; j < a.k; j += L) {
      const int e = slot(j).e;
      if (e >= 0) share[e] = 0.f;
    }
    __syncwarp();
  }
}

inline int route_grid(int64_t steps, int sms, int per_sm) {
  const int64_t most = (int64_t)sms * per_sm;
  return (int)(steps < most ? steps : most);
}

template <typename T, int V, int L, int EL, int KP, int MODE>
int launch_shape(RouteArgs a, int sms, cudaStream_t s) {
  constexpr int TOKENS = 32 / L;
  // one token's numbers in 64 bits, or all tokens' in 32 with their groups'
  const size_t wide = (size_t)a.E * 8, narrow = a.groups > 1 ? (size_t)TOKENS * (2 * a.E + 2 * a.groups) * 4 : 0;
  a.room = (int)(std::max(wide, narrow) + 15) / 16 * 16;
  const size_t smem = (size_t)WARPS * a.room;
  const auto k = route_kernel<T, V, L, EL, KP, MODE>;
  const int rc = device_launch_facts((const void*)k, smem, nullptr);
  if (rc != D2D_OK) return rc;
  return launch_pdl(k, dim3((unsigned)route_grid(ceil_div64(a.N, WARPS * TOKENS), sms, 16)), dim3(NT), smem, s, a);
}

// Lists of 4, 8 or 16 keys (4 of 96, 65536 tokens: lists of 8 take 23 us, lists of 4 20).  Rows that allow no vectors take the
// widest forms only.
template <typename T, int V, int L, int EL, int MODE>
int launch_list(const RouteArgs& a, int sms, cudaStream_t s) {
  if constexpr (V > 1) {
    if (a.k <= 4) return launch_shape<T, V, L, EL, 4, MODE>(a, sms, s);
    if (a.k <= 8) return launch_shape<T, V, L, EL, 8, MODE>(a, sms, s);
  }
  if constexpr (EL >= 16) return launch_shape<T, V, L, EL, 16, MODE>(a, sms, s);
  return D2D_ERR_UNSUPPORTED;
}
// Lanes per token: 32 logits a lane where their order is all (fewer merges), 16 where the scores need registers too (16384 x 256
// with groups: 32 take 28 us, 16 take 30).
template <typename T, int V, int MODE>
int launch_lanes(const RouteArgs& a, int sms, cudaStream_t s) {
  if constexpr (V > 1) {
    if (a.E <= 32 && a.k <= 8) return launch_list<T, V, 4, 8, MODE>(a, sms, s);
    if (a.E <= 64) return launch_list<T, V, 4, 16, MODE>(a, sms, s);
    if constexpr (MODE == ORDER) {
      if (a.E <= 128) return launch_list<T, V, 4, 32, MODE>(a, sms, s);
      if (a.E <= 256) return launch_list<T, V, 8, 32, MODE>(a, sms, s);
    } else {
      if (a.E <= 128) return launch_list<T, V, 8, 16, MODE>(a, sms, s);
      if (a.E <= 256) return launch_list<T, V, 8, 32, MODE>(a, sms, s);
    }
  } else {
    if (a.E <= 128) return launch_list<T, V, 8, 16, MODE>(a, sms, s);
  }
  return launch_list<T, V, 32, 32, MODE>(a, sms, s);
}
template <typename T, int V>
int launch_mode(const RouteArgs& a, int sms, cudaStream_t s) {
  if (a.bias || a.groups > 1) return launch_lanes<T, V, SCORED>(a, sms, s);
  if (a.softmax && !a.renormalise) return launch_lanes<T, V, TOTAL>(a, sms, s);
  return launch_lanes<T, V, ORDER>(a, sms, s);
}

template <typename T>
int route_t(const RouteArgs& a, int sms, cudaStream_t s) {
  if (a.k > 16) {
    const size_t smem = (size_t)WARPS * a.E * 8;
    const int rc = device_launch_facts((const void*)route_exact_kernel<T>, smem, nullptr);
    if (rc != D2D_OK) return rc;
    return launch_pdl(route_exact_kernel<T>, dim3((unsigned)route_grid(ceil_div64(a.N, WARPS), sms, 16)), dim3(NT),
                      smem, s, a);
  }
  constexpr int VW = 16 / sizeof(T);
  const bool vec = a.E % VW == 0 && (reinterpret_cast<uintptr_t>(a.logits) & 15) == 0;
  return vec ? launch_mode<T, VW>(a, sms, s) : launch_mode<T, 1>(a, sms, s);
}

template <typename T, int V, int L, int EL>
int backward_shape(const BackwardArgs& a, int sms, cudaStream_t s) {
  constexpr int TOKENS = 32 / L;
  const size_t smem = (size_t)WARPS * TOKENS * ((a.E + 3) / 4 * 4) * sizeof(float);
  const auto k = route_backward_kernel<T, V, L, EL>;
  const int rc = device_launch_facts((const void*)k, smem, nullptr);
  if (rc != D2D_OK) return rc;
  return launch_pdl(k, dim3((unsigned)route_grid(ceil_div64(a.N, WARPS * TOKENS), sms, 16)), dim3(NT), smem, s, a);
}

template <typename T>
int route_backward_t(const BackwardArgs& a, int sms, cudaStream_t s) {
  constexpr int VW = 16 / sizeof(T);
  const bool vec = a.E % VW == 0 &&
                   ((reinterpret_cast<uintptr_t>(a.logits) | reinterpret_cast<uintptr_t>(a.dlogits)) & 15) == 0;
  if (!vec) return backward_shape<T, 1, 32, 32>(a, sms, s);
  if (a.E <= 64) return backward_shape<T, VW, 4, 16>(a, sms, s);
  if (a.E <= 128) return backward_shape<T, VW, 8, 16>(a, sms, s);
  if (a.E <= 256) return backward_shape<T, VW, 16, 16>(a, sms, s);
  return backward_shape<T, VW, 32, 32>(a, sms, s);
}

}  // namespace
}  // namespace d2d
