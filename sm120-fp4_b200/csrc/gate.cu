// Router from logits and its load-balance loss, with gradients.
//   gate     ids = the k largest logits of a token (ties: the lowest index), w_j = softmax(l)[id_j], divided by their sum if asked
//            dl = w_j (g_j - sum g w) at id_j (normalised), or p_e (g_e - sum g w) for all experts
//   balance  L = E sum_e f_e P_e, f_e = n_e / sum n, P_e = mean over live tokens of softmax(l)_e
//            dl = g E / T' p_e (f_e - sum_j p_j f_j), with f_e - 1 / E for f_e
// Measured on the GPU: gate of 16384 x 128 fp32 9.6 us (333 instructions a token, 69 % of the issue slots) and its gradient 5.7 (83, 31 %: latency), of one token 1.8; balance loss
// of 65536 x 256 bf16 14.7 us + 2, its gradient 20 (145 and 195 instructions a token, 70 and 66 % of the slots; the bytes are 5 and 10 us). Cold caches, but for the one token.
// A warp per token with its logits in registers; sums in fp32, statistics by shuffles, no atomic decides a value. A logit of -inf is an
// expert that may not be taken: a slot for which none is left gets id -1 (an empty slot of the layer) and weight 0.
#include "common.cuh"
#include "fp8_math.cuh"
#include "tcgen05.cuh"
#include <initializer_list>
#include <type_traits>

namespace b200 {

constexpr int GATE_MAXE = 512, GATE_MAXK = 16;

// Lane l holds the logits of experts l*V .. l*V + V - 1; pad for those beyond E.
template <typename T, int V, bool kVec>
__device__ __forceinline__ void load_row(const T* __restrict__ row, int E, int lane, float (&x)[V], float pad) {
  if constexpr (kVec && V * Elem<T>::kSize >= 16) {
    constexpr int P = 16 / Elem<T>::kSize;
#pragma unroll
    for (int i = 0; i < V / P; ++i) {
      const int e = lane * V + i * P;
      float v[P];
      if (e < E) unpack16<T>(__ldg(reinterpret_cast<const uint4*>(row + e)), v);      // (E is a multiple of P)
#pragma unroll
      for (int j = 0; j < P; ++j) x[i * P + j] = e < E ? v[j] : pad;
    }
  } else if constexpr (kVec && V == 4) {      // 16 bits
    const int e = lane * V;
    uint2 w = make_uint2(0u, 0u);
    if (e < E) w = __ldg(reinterpret_cast<const uint2*>(row + e));
    Elem<T>::unpack(w.x, x[0], x[1]), Elem<T>::unpack(w.y, x[2], x[3]);
    if (e >= E) x[0] = x[1] = x[2] = x[3] = pad;
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) x[j] = lane * V + j < E ? Elem<T>::load(row + lane * V + j) : pad;
  }
}
template <typename T, int V, bool kVec>
__device__ __forceinline__ void store_row(T* __restrict__ row, int E, int lane, const float (&x)[V]) {
  if constexpr (kVec && V * Elem<T>::kSize >= 16) {
    constexpr int P = 16 / Elem<T>::kSize;
#pragma unroll
    for (int i = 0; i < V / P; ++i) {
      const int e = lane * V + i * P;
      uint4 w;
      if constexpr (P == 8) w = make_uint4(Elem<T>::pack(x[8 * i], x[8 * i + 1]), Elem<T>::pack(x[8 * i + 2], x[8 * i + 3]), Elem<T>::pack(x[8 * i + 4], x[8 * i + 5]), Elem<T>::pack(x[8 * i + 6], x[8 * i + 7]));
      else w = make_uint4(__float_as_uint(x[4 * i]), __float_as_uint(x[4 * i + 1]), __float_as_uint(x[4 * i + 2]), __float_as_uint(x[4 * i + 3]));
      if (e < E) *reinterpret_cast<uint4*>(row + e) = w;
    }
  } else if constexpr (kVec && V == 4) {
    if (lane * V < E) *reinterpret_cast<uint2*>(row + lane * V) = make_uint2(Elem<T>::pack(x[0], x[1]), Elem<T>::pack(x[2], x[3]));
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (lane * V + j < E) row[lane * V + j] = Elem<T>::make(x[j]);
  }
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Softmax numerator exp(x - m) as 2^((x - m) log2(e)): the difference, the product and log2(e) are off by 2^-24, 2^-24 and 2^-26 of |x - m|, relative in the
// result, ex2 by 2^-22. (x log2(e) - m log2(e) in one fma has one rounding less, and overflows where logits are near their type's largest value.)
constexpr float kLog2e = 1.4426950408889634f;
__device__ __forceinline__ float exp_term(float x, float m) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"((x - m) * kLog2e));
  return e;
}

// Softmax numerators against the row's maximum, and the lane's share of their sum. Rows of -inf alone: zeros. An infinity or a NaN makes the row NaN.
template <int V> __device__ __forceinline__ float softmax_terms(float (&x)[V]) {
  float m = x[0];
#pragma unroll
  for (int j = 1; j < V; ++j) m = max_nan(m, x[j]);
  m = warp_max(m);
  if (m == -INFINITY) m = 0.f;
  float s = 0.f;
#pragma unroll
  for (int j = 0; j < V; ++j) x[j] = exp_term(x[j], m), s += x[j];
  return s;
}

// An unsigned number in the order of the logits: NaN above all, -0 = +0 (the addition gives the one NaN, 0x7fffffff, and no -0).
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t u = __float_as_uint(v + 0.f);
  return u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  if (k == 0xffffffffu) return NAN;
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
constexpr uint32_t kKeyMasked = 0x007fffffu;      // order_key(-inf)

// A lane's candidates in falling order. Types of 16 bits leave nine low bits of the key free: it carries the index (turned over: the lower one wins a tie), and
// one reduction over the warp gives both. In 32 bits the index is kept beside the key, and the lowest lane that holds the largest key has the lowest index.
template <int V, bool kPacked> struct Candidates {
  uint32_t key[V];
  uint32_t idx[kPacked ? 1 : V];
  __device__ __forceinline__ void order(int a, int b) {      // a's before b's
    if constexpr (kPacked) {
      const uint32_t hi = max(key[a], key[b]), lo = min(key[a], key[b]);
      key[a] = hi, key[b] = lo;
    } else {
      const bool turn = V <= 8 ? key[a] < key[b] : key[a] < key[b] || (key[a] == key[b] && idx[a] > idx[b]);
      const uint32_t k = key[a], i = idx[a];
      key[a] = turn ? key[b] : k, key[b] = turn ? k : key[b];
      idx[a] = turn ? idx[b] : i, idx[b] = turn ? i : idx[b];
    }
  }
  // Neighbours alone change places, so that equal keys stay in the order of their indexes without a look at these.
  __device__ __forceinline__ void sort_neighbours() {
#pragma unroll
    for (int n = V - 1; n > 0; --n)
#pragma unroll
      for (int i = 0; i < n; ++i) order(i, i + 1);
  }
  // Batcher's odd-even merge sort of key[kFrom .. kFrom + kCount - 1]
  template <int kFrom, int kCount, int kStep> __device__ __forceinline__ void merge() {
    if constexpr (2 * kStep < kCount) {
      merge<kFrom, kCount, 2 * kStep>();
      merge<kFrom + kStep, kCount, 2 * kStep>();
#pragma unroll
      for (int i = kFrom + kStep; i + kStep < kFrom + kCount; i += 2 * kStep) order(i, i + kStep);
    } else {
      order(kFrom, kFrom + kStep);
    }
  }
  template <int kFrom, int kCount> __device__ __forceinline__ void sort() {
    if constexpr (kCount > 1) {
      sort<kFrom, kCount / 2>();
      sort<kFrom + kCount / 2, kCount / 2>();
      merge<kFrom, kCount, 1>();
    }
  }
  __device__ __forceinline__ void pop(bool mine) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      key[i] = mine ? (i + 1 < V ? key[i + 1 < V ? i + 1 : i] : 0u) : key[i];
      if constexpr (!kPacked)
        if (i + 1 < V) idx[i] = mine ? idx[i + 1 < V ? i + 1 : i] : idx[i];
    }
  }
};

// Bound by issue (eight of 128 experts in 32 bits: 333 instructions a token; with a scan of all candidates in every round 11.2 us instead of 9.4 at 16384 tokens).
template <typename T, int V, bool kVec>
__global__ void __launch_bounds__(256) k_gate(const T* __restrict__ logits, long long stride, int tokens, int E, int k, int renorm, float* __restrict__ weights,
                                              int* __restrict__ ids) {
  constexpr bool kPacked = Elem<T>::kSize == 2;
  const int lane = threadIdx.x & 31;
  grid_dependency_wait();
  const int t = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (t >= tokens) return;
  float x[V];
  load_row<T, V, kVec>(logits + (long long)t * stride, E, lane, x, -INFINITY);
  Candidates<V, kPacked> c;
#pragma unroll
  for (int j = 0; j < V; ++j) {      // (beyond E: -inf; if such a one is taken, none but masked ones are left)
    const int e = lane * V + j;
    c.key[j] = order_key(x[j]);
    if constexpr (kPacked) c.key[j] = (c.key[j] & ~511u) | (511 - e);
    else c.idx[j] = e;
  }
  if constexpr (kPacked || V > 8) c.template sort<0, V>();
  else c.sort_neighbours();
  uint32_t mine = 0u;      // lane j: key and index of the j-th largest
  int at = -1;
#pragma unroll 2
  for (int j = 0; j < k; ++j) {
    const uint32_t top = __reduce_max_sync(0xffffffffu, c.key[0]);
    if constexpr (kPacked) {
      if (lane == j) mine = top;
      c.pop(c.key[0] == top);
    } else {
      const int src = __ffs(__ballot_sync(0xffffffffu, c.key[0] == top)) - 1;
      const int e = __shfl_sync(0xffffffffu, c.idx[0], src);
      if (lane == j) mine = top, at = e;
      c.pop(lane == src);
    }
  }
  if constexpr (kPacked) {      // the bits that carried the index were zeros in numbers from 0 on, ones below
    at = 511 - (int)(mine & 511u);
    mine = mine >= 0xfffffe00u ? 0xffffffffu : mine & 0x80000000u ? mine & ~511u : mine | 511u;
  }
  const bool live = lane < k && mine > kKeyMasked;
  const uint32_t first = __shfl_sync(0xffffffffu, mine, 0);
  const float m = first <= kKeyMasked ? 0.f : key_value(first);
  const float w = live ? exp_term(key_value(mine), m) : 0.f;
  float s = w;
  if (renorm) {
#pragma unroll
    for (int o = 8; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);      // (16 lanes have all of it)
  } else {
    s = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) s += exp_term(x[j], m);
    s = warp_sum(s);
  }
  if (lane < k) {
    weights[(long long)t * k + lane] = live ? w * __frcp_rn(s) : 0.f;
    ids[(long long)t * k + lane] = live ? at : -1;
  }
}

template <typename T, int V, bool kVec>
__global__ void __launch_bounds__(256) k_gate_backward(const float* __restrict__ grad, const float* __restrict__ weights, const int* __restrict__ ids,
                                                       const T* __restrict__ logits, long long stride, int tokens, int E, int k, int renorm, T* __restrict__ out) {
  const int lane = threadIdx.x & 31;
  grid_dependency_wait();
  const int t = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (t >= tokens) return;
  int e = -1;
  float g = 0.f, w = 0.f;
  if (lane < k) {
    e = ids[(long long)t * k + lane];
    if (e >= E) e = -1;
    if (e >= 0) g = grad[(long long)t * k + lane], w = weights[(long long)t * k + lane];
  }
  const float dot = warp_sum(g * w);
  float d[V];
  if (renorm) {
#pragma unroll
    for (int j = 0; j < V; ++j) d[j] = 0.f;
  } else {
    load_row<T, V, kVec>(logits + (long long)t * stride, E, lane, d, -INFINITY);
    const float s = warp_sum(softmax_terms<V>(d));
    const float c = s == 0.f ? 0.f : -dot / s;
#pragma unroll
    for (int j = 0; j < V; ++j) d[j] *= c;
  }
  T* row = out + (long long)t * E;
  store_row<T, V, kVec>(row, E, lane, d);
  __syncwarp();      // orders the row's stores ahead of the chosen experts'
  if (e >= 0) row[e] = Elem<T>::make(w * (g - dot));
}

// ---------------------------------------------------------------------------------------------------- balance loss
// Each block sums its tokens' probabilities per expert (fp32, a warp's tokens in order, then the warps in order) and counts its pairs; a second
// launch adds the blocks in order. part: per block E floats, E ints, live tokens.
__host__ __device__ inline int balance_words(int E) { return 2 * E + 4; }

// 64 warps an SM hide the chain load -> maximum -> sum (two tokens in hand a warp at half of that took 17.4 instead of 14.5 us at 65536 x 256).
constexpr int kBalanceRanks = 8, kBalanceBlocks = 296;
template <int V> constexpr int kBalanceWarps = V <= 8 ? 32 : 16;      // 32 KB of partial sums

template <typename T, int V, bool kVec>
__global__ void __launch_bounds__(kBalanceWarps<V> * 32, 2) k_balance_part(const T* __restrict__ logits, long long stride, int tokens, int E, const int* __restrict__ ids, int k,
                                                                           float* __restrict__ part) {
  constexpr int kWarps = kBalanceWarps<V>;
  __shared__ float sp[kWarps][32 * V];
  __shared__ int cnt[32 * V], live_n;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < 32 * V; i += kWarps * 32) cnt[i] = 0;
  if (threadIdx.x == 0) live_n = 0;
  __syncthreads();
  grid_dependency_wait();
  float acc[V];
#pragma unroll
  for (int j = 0; j < V; ++j) acc[j] = 0.f;
  int n = 0;
  for (int t = blockIdx.x * kWarps + warp; t < tokens; t += gridDim.x * kWarps) {
    const int e = lane < k ? ids[(long long)t * k + lane] : -1;
    float x[V];
    load_row<T, V, kVec>(logits + (long long)t * stride, E, lane, x, -INFINITY);
    const bool used = e >= 0 && e < E;
    if (used) atomicAdd(&cnt[e], 1);
    if (!__any_sync(0xffffffffu, used)) continue;      // an empty token
    ++n;
    const float s = warp_sum(softmax_terms<V>(x)), r = s == 0.f ? 0.f : __frcp_rn(s);
#pragma unroll
    for (int j = 0; j < V; ++j) acc[j] = fmaf(x[j], r, acc[j]);
  }
  if (lane == 0 && n) atomicAdd(&live_n, n);
#pragma unroll
  for (int j = 0; j < V; ++j) sp[warp][lane * V + j] = acc[j];
  __syncthreads();
  float* o = part + (long long)blockIdx.x * balance_words(E);
  for (int e = threadIdx.x; e < E; e += kWarps * 32) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) s += sp[i][e];
    o[e] = s;
    reinterpret_cast<int*>(o)[E + e] = cnt[e];
  }
  if (threadIdx.x == 0) reinterpret_cast<int*>(o)[2 * E] = live_n;
}

// One cluster: a block takes an eighth of the experts, a column of threads for each, every thread of which adds one of `slices` shares of the partial sums (296 at
// most: loads of a thread are in flight together); the experts' sums meet in block 0. stats: f32 [2]: 1 / pairs, E / live tokens (at least 1 of both).
__global__ void __cluster_dims__(kBalanceRanks, 1, 1) __launch_bounds__(1024)
    k_balance_sum(const float* __restrict__ part, int blocks, int E, int log_cols, float* __restrict__ loss, int* __restrict__ counts, float* __restrict__ stats) {
  __shared__ double sp[1024];
  __shared__ int sc[1024];
  __shared__ double rank_v[kBalanceRanks];      // of block 0: every block's sum of products
  __shared__ long long rank_n[kBalanceRanks];
  __shared__ int live_s;
  const int tid = threadIdx.x, cols = 1 << log_cols, col = tid & (cols - 1), slice = tid >> log_cols, slices = 1024 >> log_cols, rank = blockIdx.x;
  const int per = (E + kBalanceRanks - 1) / kBalanceRanks, e = rank * per + col, W = balance_words(E);
  cluster_arrive();      // (block 0 is there before anybody stores into it)
  grid_dependency_wait();
  double p = 0.0;
  int c = 0;
  const bool mine = col < per && e < E;
  if (mine) {
    for (int b0 = slice; b0 < blocks; b0 += slices * 10) {
      float pv[10];
      int cv[10];
#pragma unroll
      for (int i = 0; i < 10; ++i) {
        const int b = b0 + slices * i;
        pv[i] = b < blocks ? part[b * W + e] : 0.f;
        cv[i] = b < blocks ? reinterpret_cast<const int*>(part)[b * W + E + e] : 0;
      }
#pragma unroll
      for (int i = 0; i < 10; ++i) p += (double)pv[i], c += cv[i];
    }
  }
  sp[tid] = p, sc[tid] = c;
  if (rank == 0 && tid >= 992) {
    int l = 0;
    for (int b = tid - 992; b < blocks; b += 32) l += reinterpret_cast<const int*>(part)[b * W + 2 * E];
    l = __reduce_add_sync(0xffffffffu, l);
    if (tid == 992) live_s = l;
  }
  __syncthreads();
  cluster_wait();
  if (tid < 64) {      // (cols <= 64)
    double v = 0.0;
    long long n = 0;
    if (tid < cols) {
      for (int i = 1; i < slices; ++i) p += sp[i * cols + tid], c += sc[i * cols + tid];
      if (mine) counts[e] = c;
      v = p * (double)c, n = c;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o), n += __shfl_xor_sync(0xffffffffu, n, o);
    __syncwarp();
    named_bar_sync(1, 64);      // everybody has read sp and sc
    if (tid == 32) sp[0] = v, sc[0] = (int)(n & 0xffffffffll), sc[1] = (int)(n >> 32);
    named_bar_sync(1, 64);
    if (tid == 0) {
      v += sp[0], n += (long long)(((unsigned long long)(unsigned)sc[1] << 32) | (unsigned)sc[0]);
      asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(mapa_shared(smem_u32(&rank_v[rank]), 0)), "d"(v) : "memory");
      asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(mapa_shared(smem_u32(&rank_n[rank]), 0)), "l"(n) : "memory");
    }
  }
  __syncwarp();
  cluster_sync_all();
  if (rank == 0 && tid == 0) {
    double v = 0.0;
    long long n = 0;
    for (int i = 0; i < kBalanceRanks; ++i) v += rank_v[i], n += rank_n[i];
    const double live = live_s ? (double)live_s : 1.0, pairs = n ? (double)n : 1.0;
    *loss = (float)((double)E * v / (live * pairs));
    stats[0] = (float)(1.0 / pairs), stats[1] = (float)((double)E / live);
  }
}

template <typename T, int V, bool kVec>
__global__ void __launch_bounds__(256, V <= 8 ? 8 : 4) k_balance_backward(const float* __restrict__ grad, const T* __restrict__ logits, long long stride, int tokens, int E,
                                                          const int* __restrict__ ids, int k, const int* __restrict__ counts, const float* __restrict__ stats,
                                                          T* __restrict__ out) {
  const int lane = threadIdx.x & 31;
  grid_dependency_wait();
  // p_e (f_e - sum p f) is the same with f_e - 1 / E in the place of f_e, which is what is left of it where experts are used evenly, and a quotient of whole numbers:
  // (E (n_e - q) - r) / (E sum n) with sum n = q E + r. Taken from the shares themselves, the difference would drown in their roundings there.
  const float c = *grad * stats[1], inv = stats[0] / (float)E;
  int n[V], pairs = 0;
#pragma unroll
  for (int j = 0; j < V; ++j) n[j] = lane * V + j < E ? counts[lane * V + j] : 0, pairs += n[j];
  const unsigned sum = __reduce_add_sync(0xffffffffu, (unsigned)pairs), q = sum / (unsigned)E;      // (below 2^31)
  const float r = (float)(sum - q * (unsigned)E);
  float f[V];
#pragma unroll
  for (int j = 0; j < V; ++j) f[j] = lane * V + j < E ? fmaf((float)(n[j] - (int)q), (float)E, -r) * inv : 0.f;
  for (int t = blockIdx.x * 8 + (threadIdx.x >> 5); t < tokens; t += gridDim.x * 8) {
    const int e = lane < k ? ids[(long long)t * k + lane] : -1;
    float x[V];
    load_row<T, V, kVec>(logits + (long long)t * stride, E, lane, x, -INFINITY);
    if (__any_sync(0xffffffffu, e >= 0 && e < E)) {
      float s = softmax_terms<V>(x), dot = 0.f;
#pragma unroll
      for (int j = 0; j < V; ++j) dot = fmaf(x[j], f[j], dot);
#pragma unroll
      for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o), dot += __shfl_xor_sync(0xffffffffu, dot, o);
      const float r = s == 0.f ? 0.f : __frcp_rn(s), mean = dot * r, rc = r * c;
#pragma unroll
      for (int j = 0; j < V; ++j) x[j] *= rc * (f[j] - mean);
    } else {      // an empty token
#pragma unroll
      for (int j = 0; j < V; ++j) x[j] = 0.f;
    }
    store_row<T, V, kVec>(out + (long long)t * E, E, lane, x);
  }
}

// Calls `f` with the kernel's type, values per lane and whether rows are taken 8 or 16 bytes at a time.
template <typename F> static int with_type(int dtype, F&& f) {
  if (dtype == DT_BF16) return f((__nv_bfloat16*)nullptr);
  if (dtype == DT_F16) return f((__half*)nullptr);
  return f((float*)nullptr);
}
template <typename F> static int with_values(int E, F&& f) {
  if (E <= 32) return f(std::integral_constant<int, 1>());
  if (E <= 64) return f(std::integral_constant<int, 2>());
  if (E <= 128) return f(std::integral_constant<int, 4>());
  if (E <= 256) return f(std::integral_constant<int, 8>());
  return f(std::integral_constant<int, 16>());
}
static bool vec_rows(const void* p, long long stride, int E, int size) {      // every row and every lane's run on 16 bytes (8 for four 16-bit values)
  const int unit = E <= 128 && size == 2 ? 8 : 16;
  return ((uintptr_t)p % unit) == 0 && (stride * size) % unit == 0 && ((long long)E * size) % unit == 0;
}
static int balance_blocks(int tokens) {      // 16 tokens or more each
  const int want = (tokens + 15) / 16;
  return want < kBalanceBlocks ? want : kBalanceBlocks;
}

}  // namespace b200

extern "C" {

static bool words(std::initializer_list<const void*> at) {      // all on 4 bytes
  uintptr_t bits = 0;
  for (const void* p : at) bits |= (uintptr_t)p;
  return (bits & 3) == 0;
}
static int gate_args(int dtype, long long stride, int tokens, int E, int k) {
  if (dtype < 0 || dtype > 2 || tokens < 0 || E < 1 || k < 1 || k > E || (stride < E && tokens > 1)) return B200MOE_ERR_ARG;
  if (E > b200::GATE_MAXE || k > b200::GATE_MAXK || tokens > (1 << 30)) return B200MOE_ERR_LIMIT;
  return B200MOE_OK;
}

int b200moe_gate(const void* logits, int dtype, long long stride, int tokens, int E, int k, int renormalize, float* weights, int* ids, void* stream) {
  using namespace b200;
  if (int rc = gate_args(dtype, stride, tokens, E, k)) return rc;
  if (tokens == 0) return B200MOE_OK;
  if (!logits || !weights || !ids || !words({weights, ids}) || ((uintptr_t)logits & (dtype == DT_F32 ? 3 : 1))) return B200MOE_ERR_ARG;
  return with_type(dtype, [&](auto* tp) {
    using T = std::remove_pointer_t<decltype(tp)>;
    return with_values(E, [&](auto v) {
      constexpr int V = decltype(v)::value;
      const T* lp = (const T*)logits;
      void* args[] = {&lp, &stride, &tokens, &E, &k, &renormalize, &weights, &ids};
      const void* fn = vec_rows(logits, stride, E, sizeof(T)) ? (const void*)k_gate<T, V, true> : (const void*)k_gate<T, V, false>;
      return launch_kernel(fn, (tokens + 7) / 8, 256, 0, true, args, (cudaStream_t)stream);
    });
  });
}

int b200moe_gate_backward(const float* grad_weights, const float* weights, const int* ids, const void* logits, int dtype, long long stride, int tokens, int E, int k,
                          int renormalize, void* grad_logits, void* stream) {
  using namespace b200;
  if (int rc = gate_args(dtype, stride, tokens, E, k)) return rc;
  if (tokens == 0) return B200MOE_OK;
  if (!grad_weights || !weights || !ids || !grad_logits || (!renormalize && !logits) || !words({grad_weights, weights, ids}) || (((uintptr_t)logits | (uintptr_t)grad_logits) & (dtype == DT_F32 ? 3 : 1)))
    return B200MOE_ERR_ARG;
  return with_type(dtype, [&](auto* tp) {
    using T = std::remove_pointer_t<decltype(tp)>;
    return with_values(E, [&](auto v) {
      constexpr int V = decltype(v)::value;
      const T* lp = (const T*)logits;
      T* op = (T*)grad_logits;
      void* args[] = {&grad_weights, &weights, &ids, &lp, &stride, &tokens, &E, &k, &renormalize, &op};
      const bool vec = (renormalize || vec_rows(logits, stride, E, sizeof(T))) && vec_rows(grad_logits, E, E, sizeof(T));
      const void* fn = vec ? (const void*)k_gate_backward<T, V, true> : (const void*)k_gate_backward<T, V, false>;
      return launch_kernel(fn, (tokens + 7) / 8, 256, 0, true, args, (cudaStream_t)stream);
    });
  });
}

long long b200moe_balance_workspace_bytes(int tokens, int E) {
  if (tokens < 0 || E < 1) return B200MOE_ERR_ARG;
  if (E > b200::GATE_MAXE) return B200MOE_ERR_LIMIT;
  return 4ll * b200::balance_words(E) * b200::balance_blocks(tokens);
}

int b200moe_balance_loss(const void* logits, int dtype, long long stride, int tokens, int E, const int* ids, int k, float* loss, int* counts, float* stats,
                         void* workspace, long long workspace_bytes, void* stream) {
  using namespace b200;
  if (dtype < 0 || dtype > 2 || tokens < 0 || E < 1 || k < 1 || (stride < E && tokens > 1)) return B200MOE_ERR_ARG;
  if (E > GATE_MAXE || k > 32 || tokens > (1 << 30) || (long long)tokens * k > 0x7fffffff) return B200MOE_ERR_LIMIT;      // (counts of 32 bits)
  if (!loss || !counts || !stats || (tokens && (!logits || !ids || !workspace)) || ((uintptr_t)logits & (dtype == DT_F32 ? 3 : 1)) || !words({ids, loss, counts, stats, workspace}))
    return B200MOE_ERR_ARG;
  if (workspace_bytes < b200moe_balance_workspace_bytes(tokens, E)) return B200MOE_ERR_WORKSPACE;
  int blocks = balance_blocks(tokens);
  float* part = (float*)workspace;
  const int rc = tokens == 0 ? B200MOE_OK : with_type(dtype, [&](auto* tp) {
    using T = std::remove_pointer_t<decltype(tp)>;
    return with_values(E, [&](auto v) {
      constexpr int V = decltype(v)::value;
      const T* lp = (const T*)logits;
      void* args[] = {&lp, &stride, &tokens, &E, &ids, &k, &part};
      const void* fn = vec_rows(logits, stride, E, sizeof(T)) ? (const void*)k_balance_part<T, V, true> : (const void*)k_balance_part<T, V, false>;
      return launch_kernel(fn, blocks, kBalanceWarps<V> * 32, 0, true, args, (cudaStream_t)stream);
    });
  });
  if (rc) return rc;
  const float* cp = part;
  int log_cols = 5;      // columns of a block: the power of two from its eighth of the experts on, 32 at least (1024 / 32 shares are added one after the other)
  while ((1 << log_cols) < (E + kBalanceRanks - 1) / kBalanceRanks) ++log_cols;
  void* args[] = {&cp, &blocks, &E, &log_cols, &loss, &counts, &stats};
  return launch_kernel((const void*)k_balance_sum, kBalanceRanks, 1024, 0, true, args, (cudaStream_t)stream);
}

int b200moe_balance_backward(const float* grad_loss, const void* logits, int dtype, long long stride, int tokens, int E, const int* ids, int k, const int* counts,
                             const float* stats, void* grad_logits, void* stream) {
  using namespace b200;
  if (dtype < 0 || dtype > 2 || tokens < 0 || E < 1 || k < 1 || (stride < E && tokens > 1)) return B200MOE_ERR_ARG;
  if (E > GATE_MAXE || k > 32 || tokens > (1 << 30) || (long long)tokens * k > 0x7fffffff) return B200MOE_ERR_LIMIT;      // (counts of 32 bits)
  if (tokens == 0) return B200MOE_OK;
  if (!grad_loss || !logits || !ids || !counts || !stats || !grad_logits || !words({grad_loss, ids, counts, stats}) || (((uintptr_t)logits | (uintptr_t)grad_logits) & (dtype == DT_F32 ? 3 : 1))) return B200MOE_ERR_ARG;
  return with_type(dtype, [&](auto* tp) {
    using T = std::remove_pointer_t<decltype(tp)>;
    return with_values(E, [&](auto v) {
      constexpr int V = decltype(v)::value;
      const T* lp = (const T*)logits;
      T* op = (T*)grad_logits;
      void* args[] = {&grad_loss, &lp, &stride, &tokens, &E, &ids, &k, &counts, &stats, &op};
      const bool vec = vec_rows(logits, stride, E, sizeof(T)) && vec_rows(grad_logits, E, E, sizeof(T));
      const void* fn = vec ? (const void*)k_balance_backward<T, V, true> : (const void*)k_balance_backward<T, V, false>;
      const int want = (tokens + 7) / 8;
      return launch_kernel(fn, want < 1184 ? want : 1184, 256, 0, true, args, (cudaStream_t)stream);
    });
  });
}

}  // extern "C"
