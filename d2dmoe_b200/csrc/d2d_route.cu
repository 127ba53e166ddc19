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
// The choice is made as 64 bits make it.  What bounds a choice in 32 bits is instructions, not bytes (128 bf16
// logits are read in a fifth of the time that eight rounds of a warp-wide maximum take), so it is made on
// 32-bit keys that hold the order in their upper bits and the index in the lower ones:
//   * L lanes have a token; each sorts its keys in batches of KP with a network (Batcher's odd-even merge sort: a
//     minimum and a maximum per exchange) and merges them into a list of its KP best; log2 L butterfly merges
//     make that the token's list in every lane.
//   * The upper bits are less than the number itself.  Where two neighbours of the list, or its last one and the
//     best that is not in it, are nearer than the keys and the arithmetic before them can tell, the
//     whole warp makes that token's choice again in 64 bits.  bf16 logits without a bias fit into the
//     upper bits and never need it.
// Scores for the choice may therefore come from the fast exponential; the weights come from the accurate one.
#include <algorithm>

#include "d2d_common.cuh"

namespace d2d {
namespace {

constexpr int NT = 128;                    // threads of a block
constexpr int WARPS = NT / 32;
constexpr int MAX_E = 1024, MAX_K = 32, MAX_GROUPS = 32;
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
};

__device__ __forceinline__ bool unusable(float v) { return !(v <= MAX_FINITE); }      // NaN, +inf

// order-preserving map of a float to an unsigned integer
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t b = __float_as_uint(v);
  return b ^ (0x80000000u | (uint32_t)((int32_t)b >> 31));
}

__device__ __forceinline__ float sigmoidf(float l) { return 1.f / (1.f + expf(-l)); }

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
    // (sigmoids below e^-60 are exponentials to the last bit: their quotients do not underflow as those)
    w[r] = e[r] < 0          ? 0.f
           : !a.renormalise  ? (a.softmax ? expf(l[r] - m) / denom : sigmoidf(l[r]))
           : a.softmax || mx < -60.f ? expf(l[r] - mx)
                                     : sigmoidf(l[r]);
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
__device__ __noinline__ void route_exact(const RouteArgs& a, int64_t t, double* c, int lane) {
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
  if (scored && a.softmax && !empty) {
    total = 0.0;
    for (int e = lane; e < E; e += 32) total += exp((double)DT<T>::to_f(row[e]) - (double)m);
    total = warp_sum(total);
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
  put_choice<T, 32, 1>(a, t, lane, mine, bad, m, (float)total);
  __syncwarp();
}

template <typename T>
__global__ void __launch_bounds__(NT) route_exact_kernel(const RouteArgs a) {
  extern __shared__ __align__(16) double scratch[];
  grid_launch_dependents();
  grid_dependency_wait();
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

// V consecutive logits as floats
template <typename T, int V>
__device__ __forceinline__ void load_logits(const T* p, float* f) {
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

// L lanes per token, EL logits per lane, lists of KP keys; V logits per load.  SCORED: the choice or the weights
// need the scores of all experts.
template <typename T, int V, int L, int EL, int KP, bool SCORED>
__global__ void __launch_bounds__(NT) route_kernel(const RouteArgs a) {
  extern __shared__ __align__(16) double scratch[];
  constexpr int TOKENS = 32 / L;           // of a warp at once
  constexpr int R = (KP + L - 1) / L;
  grid_launch_dependents();
  grid_dependency_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, q = lane % L, mine = lane / L;
  const int E = a.E, k = a.k;
  // (room for the numbers of one token in 64 bits, or of all of them and their groups in 32)
  const size_t room = max((size_t)E * 8, ((size_t)TOKENS * (E + a.groups) * 4 + 7) / 8 * 8) / 8;
  double* const wide = scratch + warp * room;
  int index_bits = 1;
  while ((1 << index_bits) < E) ++index_bits;
  const uint32_t low = (1u << index_bits) - 1u;
  const int64_t steps = ceil_div64(a.N, (int64_t)WARPS * TOKENS);
  for (int64_t step = blockIdx.x; step < steps; step += gridDim.x) {
    const int64_t t = (step * WARPS + warp) * TOKENS + mine;
    const bool in = t < a.N;
    float l[EL];
    bool bad = false;
#pragma unroll
    for (int v = 0; v < EL / V; ++v) {
      const int e = (v * L + q) * V;
      if (in && e < E) {
        load_logits<T, V>(reinterpret_cast<const T*>(a.logits) + t * E + e, l + v * V);
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) l[v * V + i] = -INFINITY;
      }
    }
#pragma unroll
    for (int i = 0; i < EL; ++i) bad |= unusable(l[i]);
    uint32_t key[EL], seen = 0;
    uint32_t near = 0;                     // keys that differ by this much in their upper bits may be in any order
    bool unsure = false;                   // this token's choice is made again in 64 bits
    float m = -INFINITY, denom = 1.f;
    if constexpr (!SCORED) {
#pragma unroll
      for (int v = 0; v < EL / V; ++v)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float x = l[v * V + i];
          const uint32_t e = (uint32_t)((v * L + q) * V + i);
          if (sizeof(T) == 4 && x > -INFINITY) seen |= __float_as_uint(x);
          key[v * V + i] = x > -INFINITY ? (ordered(x) & ~low) | (low - e) : 0u;
        }
    } else {
#pragma unroll
      for (int i = 0; i < EL; ++i) m = fmaxf(m, l[i]);
#pragma unroll
      for (int o = 1; o < L; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      float c[EL];
      if (a.softmax) {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < EL; ++i) {
          c[i] = l[i] > -INFINITY ? __expf(l[i] - m) : 0.f;
          sum += c[i];
        }
#pragma unroll
        for (int o = 1; o < L; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        denom = sum;
        const float inv = 1.f / sum;
#pragma unroll
        for (int i = 0; i < EL; ++i) c[i] *= inv;
      } else if (a.bias || a.groups > 1) {
#pragma unroll
        for (int i = 0; i < EL; ++i) c[i] = __fdividef(1.f, 1.f + __expf(-fmaxf(l[i], -80.f)));
      } else {
#pragma unroll
        for (int i = 0; i < EL; ++i) c[i] = 0.f;
      }
      float top = -INFINITY;
      if (a.bias) {
#pragma unroll
        for (int v = 0; v < EL / V; ++v)
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const int e = (v * L + q) * V + i;
            const float b = e < E ? __ldg(a.bias + e) : 0.f;
            bad |= unusable(b);
            c[v * V + i] += b;
          }
      }
#pragma unroll
      for (int i = 0; i < EL; ++i) {
        if (!(l[i] > -INFINITY)) c[i] = -INFINITY;
        top = fmaxf(top, c[i]);
      }
#pragma unroll
      for (int o = 1; o < L; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      uint32_t kept = 0xffffffffu;
      const int size = E / a.groups;
      if (a.groups > 1) {
        // the two best of each group by the token's lanes, group after group, from shared memory
        float* const rows = reinterpret_cast<float*>(wide) + mine * (E + a.groups);
        __syncwarp();
#pragma unroll
        for (int v = 0; v < EL / V; ++v)
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const int e = (v * L + q) * V + i;
            if (e < E) rows[e] = c[v * V + i];
          }
        __syncwarp();
        for (int g = q; g < a.groups; g += L) {
          float best = -INFINITY, second = -INFINITY;
          int at = lane % size;            // (another bank for each lane)
          for (int i = 0; i < size; ++i) {
            const float v = rows[g * size + at];
            second = fmaxf(second, fminf(best, v));
            best = fmaxf(best, v);
            at = at + 1 == size ? 0 : at + 1;
          }
          rows[E + g] = second > -INFINITY ? best + second : best;
        }
        __syncwarp();
        kept = 0u;
        float worst = INFINITY, other = -INFINITY;       // kept, not kept
        for (int g = q; g < a.groups; g += L) {
          const float v = rows[E + g];
          int before = 0;
          for (int h = 0; h < a.groups; ++h) {
            const float u = rows[E + h];
            before += u > v || (u == v && h < g);
          }
          if (before < a.top_groups) {
            kept |= 1u << g;
            worst = fminf(worst, v);
          } else {
            other = fmaxf(other, v);
          }
        }
#pragma unroll
        for (int o = 1; o < L; o <<= 1) {
          kept |= __shfl_xor_sync(0xffffffffu, kept, o);
          worst = fminf(worst, __shfl_xor_sync(0xffffffffu, worst, o));
          other = fmaxf(other, __shfl_xor_sync(0xffffffffu, other, o));
        }
        // (two scores and their sum: twice the bound below)
        unsure = other > -INFINITY && worst - other <= 8e-6f + 1e-6f * fabsf(worst);
      }
      // Scores of the fast exponential and reciprocal are off by less than 6e-7 (softmax: 2 ulp of the exponential,
      // as much of the sum; sigmoid: less), their sums with the bias by half an ulp more: two
      // of them in the wrong order differ by less than 2e-6 + 2^-23 |c|.  Keys take the range of 4 below
      // the largest c in steps of 2^(2 + index bits - 32); what lies lower has the lowest key.
      const float scale = (float)(1u << (30 - index_bits)) * (a.bias ? 1.f : 0.f);
      near = a.bias ? (uint32_t)fminf((4e-6f + 5e-7f * fabsf(top)) * scale, 1e9f) + 2u : 0u;
#pragma unroll
      for (int v = 0; v < EL / V; ++v)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int e = (v * L + q) * V + i;
          const float x = l[v * V + i];
          const bool can = x > -INFINITY && c[v * V + i] > -INFINITY &&
                           (a.groups == 1 || (kept >> (e / size) & 1u) != 0u);
          uint32_t hi;
          if (a.bias) {
            const uint32_t u = (uint32_t)fmaxf((c[v * V + i] - top + 4.f) * scale, 1.f);
            hi = min(u, (0xffffffffu >> index_bits)) << index_bits;
          } else {
            if (sizeof(T) == 4 && can) seen |= __float_as_uint(x);
            hi = ordered(x) & ~low;
          }
          key[v * V + i] = can ? hi | (low - (uint32_t)e) : 0u;
        }
    }
#pragma unroll
    for (int o = 1; o < L; o <<= 1) bad |= (bool)__shfl_xor_sync(0xffffffffu, (int)bad, o);

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
    if (sizeof(T) == 4 || (SCORED && a.bias)) {
      bool lossy = SCORED && a.bias;
      if (!lossy) {
#pragma unroll
        for (int o = 1; o < L; o <<= 1) seen |= __shfl_xor_sync(0xffffffffu, seen, o);
        lossy = (seen & low) != 0u;
      }
      uint32_t last = 0;
      bool close = false;
#pragma unroll
      for (int i = 0; i < KP; ++i) {
        if (i + 1 < KP && i < k && list[i + 1] != 0u)
          close |= (list[i] >> index_bits) - (list[i + 1] >> index_bits) <= near;
        if (i == k - 1) last = list[i];
      }
      if (k == KP) {                       // the best that is not in the list (whole warps: k is everyone's)
        const uint32_t bound = last >> index_bits, from = bound > near ? bound - near : 1u;
        int n = 0;
#pragma unroll
        for (int i = 0; i < EL; ++i) n += key[i] != 0u && (key[i] >> index_bits) >= from;
#pragma unroll
        for (int o = 1; o < L; o <<= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
        close |= last != 0u && n > k;
      }
      unsure |= lossy && close;
    }
    unsure = unsure && in && !bad;
    int e[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      uint32_t x = 0u;
#pragma unroll
      for (int i = 0; i < L && i + L * r < KP; ++i)
        if (q == i) x = list[i + L * r];
      e[r] = x == 0u || bad || q + L * r >= k ? -1 : (int)(low - (x & low));
    }
    if (in && !unsure) {
      if (a.mask_bits) {
        const int nw = (E + 31) / 32;
        for (int w = q; w < nw; w += L) {
          uint32_t bits = 0u;
#pragma unroll
          for (int i = 0; i < KP; ++i) {
            const uint32_t x = low - (list[i] & low);
            if (i < k && list[i] != 0u && !bad && (int)(x >> 5) == w) bits |= 1u << (x & 31);
          }
          a.mask_bits[t * nw + w] = bits;
        }
      }
    }
    const bool write = in && !unsure;
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (!write) e[r] = -1;
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
// The choice itself has no gradient, nor has its bias.  A warp has a token; its row is put together in shared
// memory and written once.
template <typename T>
__global__ void __launch_bounds__(NT)
route_backward_kernel(const T* __restrict__ logits, const int32_t* __restrict__ experts,
                      const float* __restrict__ weights, const float* __restrict__ dweights,
                      T* __restrict__ dlogits, int64_t N, int E, int k, bool softmax, bool renormalise,
                      float scale) {
  extern __shared__ __align__(16) double scratch[];
  grid_launch_dependents();
  grid_dependency_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float* const row = reinterpret_cast<float*>(scratch) + (size_t)warp * E;
  const float inv = 1.f / scale;
  for (int64_t t = (int64_t)blockIdx.x * WARPS + warp; t < N; t += (int64_t)gridDim.x * WARPS) {
    const T* l = logits + t * E;
    int e = lane < k ? experts[t * k + lane] : -1;
    if ((unsigned)e >= (unsigned)E) e = -1;
    float g = 0.f, p = 0.f, le = 0.f;
    if (e >= 0) {
      g = scale * dweights[t * k + lane];
      p = weights[t * k + lane] * inv;
      le = DT<T>::to_f(l[e]);
    }
    float dot = p * g;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    const float rest = 1.f / (1.f + expf(le));           // 1 - sigmoid
    const float d = renormalise ? p * (g - dot) * (softmax ? 1.f : rest) : softmax ? g : g * p * rest;
    for (int i = lane; i < E; i += 32) row[i] = 0.f;
    __syncwarp();
    if (e >= 0) atomicAdd(&row[e], d);     // (an expert that is there twice has both shares)
    __syncwarp();
    if (softmax && !renormalise) {
      float m = -INFINITY, sum = 0.f;
      for (int i = lane; i < E; i += 32) m = fmaxf(m, DT<T>::to_f(l[i]));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      const bool any = __any_sync(0xffffffffu, e >= 0);
      for (int i = lane; i < E; i += 32) sum += expf(DT<T>::to_f(l[i]) - m);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      const float is = 1.f / sum;
      for (int i = lane; i < E; i += 32)
        dlogits[t * E + i] = DT<T>::from_f(any ? expf(DT<T>::to_f(l[i]) - m) * is * (row[i] - dot) : 0.f);
    } else {
      for (int i = lane; i < E; i += 32) dlogits[t * E + i] = DT<T>::from_f(row[i]);
    }
    __syncwarp();
  }
}

int grid_for(int64_t steps, int sms, int per_sm) {
  const int64_t most = (int64_t)sms * per_sm;
  return (int)(steps < most ? steps : most);
}

template <typename T, int V, int L, int EL, int KP>
int launch_shape(const RouteArgs& a, int sms, cudaStream_t s) {
  const bool scored = a.bias || a.groups > 1 || (a.softmax && !a.renormalise);
  const auto k = scored ? route_kernel<T, V, L, EL, KP, true> : route_kernel<T, V, L, EL, KP, false>;
  constexpr int TOKENS = 32 / L;
  const size_t room = std::max((size_t)a.E * 8, ((size_t)TOKENS * (a.E + a.groups) * 4 + 7) / 8 * 8);
  const size_t smem = WARPS * room;
  const int rc = device_launch_facts((const void*)k, smem, nullptr);
  if (rc != D2D_OK) return rc;
  return launch_pdl(k, dim3((unsigned)grid_for(ceil_div64(a.N, WARPS * TOKENS), sms, 16)), dim3(NT), smem, s, a);
}

// lists of 8 or 16; lanes per token so that each has 32 logits at most.  (Rows that allow no vectors take the widest
// forms only.)
template <typename T, int V, int L, int EL>
int launch_list(const RouteArgs& a, int sms, cudaStream_t s) {
  if constexpr (V > 1)
    if (a.k <= 8) return launch_shape<T, V, L, EL, 8>(a, sms, s);
  if constexpr (EL >= 16) return launch_shape<T, V, L, EL, 16>(a, sms, s);
  return D2D_ERR_UNSUPPORTED;
}
template <typename T, int V>
int launch_lanes(const RouteArgs& a, int sms, cudaStream_t s) {
  if constexpr (V > 1) {
    if (a.E <= 32 && a.k <= 8) return launch_list<T, V, 4, 8>(a, sms, s);
    if (a.E <= 64) return launch_list<T, V, 4, 16>(a, sms, s);
  }
  if (a.E <= 128) return launch_list<T, V, 4, 32>(a, sms, s);
  if constexpr (V > 1) {
    if (a.E <= 256) return launch_list<T, V, 8, 32>(a, sms, s);
  }
  return launch_list<T, V, 32, 32>(a, sms, s);
}

template <typename T>
int launch_t(const RouteArgs& a, int sms, cudaStream_t s) {
  if (a.k > 16) {
    const size_t smem = (size_t)WARPS * a.E * 8;
    const int rc = device_launch_facts((const void*)route_exact_kernel<T>, smem, nullptr);
    if (rc != D2D_OK) return rc;
    return launch_pdl(route_exact_kernel<T>, dim3((unsigned)grid_for(ceil_div64(a.N, WARPS), sms, 16)), dim3(NT),
                      smem, s, a);
  }
  constexpr int VW = 16 / sizeof(T);
  const bool vec = a.E % VW == 0 && (reinterpret_cast<uintptr_t>(a.logits) & 15) == 0;
  return vec ? launch_lanes<T, VW>(a, sms, s) : launch_lanes<T, 1>(a, sms, s);
}

}  // namespace

bool route_supported(int E, int k, int groups) { return E <= MAX_E && k <= MAX_K && groups <= MAX_GROUPS; }

int launch_route(const void* logits, const float* bias, int k, bool softmax, bool renormalise, float scale,
                 int groups, int top_groups, int32_t* experts, float* weights, uint32_t* mask_bits, void* dense,
                 int64_t N, int E, int dtype, cudaStream_t s) {
  int sms = 0;
  const int rc = device_launch_facts(nullptr, 0, &sms);
  if (rc != D2D_OK) return rc;
  const RouteArgs a = {logits, bias, experts, weights, mask_bits, dense, N,     E,
                       k,      groups > 1 ? groups : 1, top_groups, softmax, renormalise, scale};
  return dtype == D2D_F32 ? launch_t<float>(a, sms, s) : launch_t<bf16>(a, sms, s);
}

int launch_route_backward(const void* logits, const int32_t* experts, const float* weights,
                          const float* dweights, bool softmax, bool renormalise, float scale, void* dlogits,
                          int64_t N, int E, int k, int dtype, cudaStream_t s) {
  int sms = 0;
  int rc = device_launch_facts(nullptr, 0, &sms);
  if (rc != D2D_OK) return rc;
  const size_t smem = (size_t)WARPS * E * sizeof(float);
  const dim3 grid((unsigned)grid_for(ceil_div64(N, WARPS), sms, 16));
  if (dtype == D2D_F32)
    return launch_pdl(route_backward_kernel<float>, grid, dim3(NT), smem, s, (const float*)logits, experts, weights,
                      dweights, (float*)dlogits, N, E, k, softmax, renormalise, scale);
  return launch_pdl(route_backward_kernel<bf16>, grid, dim3(NT), smem, s, (const bf16*)logits, experts, weights,
                    dweights, (bf16*)dlogits, N, E, k, softmax, renormalise, scale);
}

}  // namespace d2d
