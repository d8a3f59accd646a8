// FP8 quantiser: E4M3 codes with one fp32 scale per 1x128 values of a row (activations) or per 128x128 block (weights).
//   scale = fl(amax / 448), factor = fl(448 / amax), amax = max(max|x|, 1e-12); code = e4m3(fl(x * factor))
// One pass over the data: a group's values stay in registers between its maximum and its codes. HBM-bound byte movers: 3 bytes per 16-bit value (5 per 32-bit
// one) plus a scale per group. Measured: 30000 x 2048 bf16 34 us (5.5 TB/s), x 1024 fp32 23.6 us (6.6 TB/s), 128 experts' 1536 x 2048 204 us (5.9 TB/s, of 6.54 of a
// copy), 16 x 2048 1.7 us.
#include "common.cuh"
#include "fp8_math.cuh"

namespace b200 {

// A lane's 16 values, one of eight lanes that share a group of 128: their codes, and the group's scale.
template <typename T> __device__ __forceinline__ uint4 codes_of_16(const uint4 (&w)[Elem<T>::kSize], float& scale) {
  constexpr int W = Elem<T>::kSize;      // 16-byte words of 16 values
  float v[16], m = 0.f;
#pragma unroll
  for (int i = 0; i < W; ++i) unpack16<T>(w[i], v + i * (16 / W));
#pragma unroll
  for (int i = 0; i < 16; ++i) m = max_nan(m, fabsf(v[i]));
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  const Fp8Scale s = fp8_scale(m);
  scale = s.scale;
  return make_uint4(cvt_e4m3x4(v[0] * s.factor, v[1] * s.factor, v[2] * s.factor, v[3] * s.factor), cvt_e4m3x4(v[4] * s.factor, v[5] * s.factor, v[6] * s.factor, v[7] * s.factor),
                    cvt_e4m3x4(v[8] * s.factor, v[9] * s.factor, v[10] * s.factor, v[11] * s.factor),
                    cvt_e4m3x4(v[12] * s.factor, v[13] * s.factor, v[14] * s.factor, v[15] * s.factor));
}

// Rows, 16 bytes at a time: K and both row strides are multiples of 16 values, so that a lane's 16 values are whole. Eight lanes share a
// group of 128; a lane whose values lie beyond K (the last group of a row) takes part in the maximum with zeros.
template <typename T>
__global__ void __launch_bounds__(256) k_quantize_fp8_rows(const T* __restrict__ x, long long ldx, int x_rows, const int* __restrict__ src_row, int rows, int K,
                                                           uint8_t* __restrict__ codes, long long ldc, float* __restrict__ scales) {
  constexpr int W = Elem<T>::kSize;
  const int KB = (K + 127) >> 7;
  const long long units = (long long)rows * KB;
  grid_dependency_wait();
  grid_launch_dependents();
  for (long long u = (long long)blockIdx.x * 32 + (threadIdx.x >> 3); u < ((units + 3) & ~3ll); u += (long long)gridDim.x * 32) {   // (whole warps: four units each)
    const bool in = u < units;
    const int row = in ? (int)(u / KB) : 0, g = in ? (int)(u - (long long)row * KB) : 0;
    const int c = g * 128 + (threadIdx.x & 7) * 16;
    int src = row;
    if (src_row && in) src = src_row[row];
    const bool gone = src < 0 || src >= x_rows;      // an empty row: zero codes and scales
    const bool have = in && !gone && c < K;
    uint4 w[W];
#pragma unroll
    for (int i = 0; i < W; ++i) w[i] = have ? *(reinterpret_cast<const uint4*>(x + (long long)src * ldx + c) + i) : make_uint4(0u, 0u, 0u, 0u);
    float scale;
    const uint4 q = codes_of_16<T>(w, scale);
    if (!in) continue;
    if (c < K) *reinterpret_cast<uint4*>(codes + (long long)row * ldc + c) = q;
    if ((threadIdx.x & 7) == 0) scales[(long long)row * KB + g] = gone ? 0.f : scale;
  }
}

// Rows that are asked for several times (a token's copies for its experts): each source row is read and quantised once and its codes are stored to its
// destinations, which hang on a list per source row: head i32 [x_rows], next i32 [rows], made by two small kernels. The order of a list is that of the atomics,
// and does not matter: every destination gets the same bytes. Reading the source once per destination took 47 us for 4096 rows of 2816 eight times over (184 MB out
// of L2); the destinations' 92 MB are what HBM has to take.
// A list is walked by one warp for each 512 columns, 77 ns a destination. So that a row which is wanted very often is not left to them, a block of 256 destinations puts
// kFromBlock of a row on its list at most, counted by a hash of the row; the others read the row themselves, spread over the block's warps. A list then has one in
// 32 of all destinations at most (us, bounded / any length: 32768 of 2816 bf16, half of them one row, 110 / 1276; all of them, 171 / 3010; evenly spread 23.8 / 23.7).
__global__ void __launch_bounds__(256) k_no_heads(int* __restrict__ head, int x_rows) {
  grid_dependency_wait();
  grid_launch_dependents();
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i < x_rows) head[i] = -1;
}
constexpr int kLinked = 256, kFromBlock = 8, kLinkThreads = 512;      // destinations of a block
template <typename T>
__global__ void __launch_bounds__(kLinkThreads) k_link_rows(const T* __restrict__ x, long long ldx, int x_rows, const int* __restrict__ src_row, int rows, int K,
                                                            int* __restrict__ head, int* __restrict__ next, uint8_t* __restrict__ codes, long long ldc,
                                                            float* __restrict__ scales) {
  constexpr int W = Elem<T>::kSize, kAhead = 2, kHash = 1024;
  __shared__ int seen[kHash], source[kLinked], left[kLinked], left_n;
  const int tid = threadIdx.x, lane = tid & 31, r0 = blockIdx.x * kLinked, r = r0 + tid, KB = (K + 127) >> 7;
  for (int i = tid; i < kHash; i += kLinkThreads) seen[i] = 0;
  if (tid == 0) left_n = 0;
  __syncthreads();
  grid_dependency_wait();
  if (tid < kLinked && r < rows) {
    int s = src_row[r];
    if (s >= x_rows) s = -1;      // an empty row: zero codes and scales
    if (s >= 0 && atomicAdd(&seen[(uint32_t)s * 2654435769u >> 22], 1) < kFromBlock) {
      next[r] = atomicExch(head + s, r);
    } else {
      source[tid] = s;
      left[atomicAdd(&left_n, 1)] = tid;
    }
  }
  __syncthreads();
  grid_launch_dependents();      // (from the start on, the next kernel's blocks crowd onto the SMs that have none of these: 512 rows 64 times over 31 us instead of 25)
  for (int i = tid >> 5; i < left_n; i += kLinkThreads / 32) {      // a warp each
    const int at = left[i], from = source[at];
    uint8_t* to = codes + (long long)(r0 + at) * ldc;
    float* s = scales + (long long)(r0 + at) * KB;
    if (from < 0) {
      for (int j = lane; j < K / 16; j += 32) *reinterpret_cast<uint4*>(to + j * 16) = make_uint4(0u, 0u, 0u, 0u);
      for (int j = lane; j < KB; j += 32) s[j] = 0.f;
      continue;
    }
    const T* row = x + (long long)from * ldx;
    for (int c0 = 0; c0 < K; c0 += 512 * kAhead) {
      uint4 w[kAhead][W];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int c = c0 + j * 512 + lane * 16;
#pragma unroll
        for (int h = 0; h < W; ++h) w[j][h] = c < K ? *(reinterpret_cast<const uint4*>(row + c) + h) : make_uint4(0u, 0u, 0u, 0u);
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int c = c0 + j * 512 + lane * 16;
        float scale;
        const uint4 q = codes_of_16<T>(w[j], scale);
        if (c < K) *reinterpret_cast<uint4*>(to + c) = q;
        if ((lane & 7) == 0 && c < K) s[c >> 7] = scale;
      }
    }
  }
}
template <typename T>
__global__ void __launch_bounds__(256) k_quantize_fp8_copies(const T* __restrict__ x, long long ldx, int x_rows, int K, const int* __restrict__ head, const int* __restrict__ next,
                                                             uint8_t* __restrict__ codes, long long ldc, float* __restrict__ scales) {
  constexpr int W = Elem<T>::kSize;
  const int KB = (K + 127) >> 7, quads = (KB + 3) >> 2;      // a warp takes four groups of a row
  const long long u = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int row = (int)(u / quads), g = (int)(u - (long long)row * quads) * 4 + (threadIdx.x >> 3 & 3), c = g * 128 + (threadIdx.x & 7) * 16;
  grid_dependency_wait();
  grid_launch_dependents();
  if (row >= x_rows) return;      // (whole warps)
  uint4 w[W];
#pragma unroll
  for (int i = 0; i < W; ++i) w[i] = c < K ? *(reinterpret_cast<const uint4*>(x + (long long)row * ldx + c) + i) : make_uint4(0u, 0u, 0u, 0u);
  int r = head[row];
  float scale;
  const uint4 q = codes_of_16<T>(w, scale);
  while (r >= 0) {
    const int after = next[r];
    if (c < K) *reinterpret_cast<uint4*>(codes + (long long)r * ldc + c) = q;
    if ((threadIdx.x & 7) == 0 && g < KB) scales[(long long)r * KB + g] = scale;
    r = after;
  }
}

// Rows of any length, stride and alignment: a warp takes four groups of a row, four neighbouring values a lane and group, loaded kLoad at a time (what rows and strides
// allow; the loads of a warp share their sectors) and stored as one word where the rows of the codes allow it.
constexpr int kAnyGroups = 4;
template <typename T, int kLoad>
__global__ void __launch_bounds__(256) k_quantize_fp8_rows_any(const T* __restrict__ x, long long ldx, int x_rows, const int* __restrict__ src_row, int rows, int K,
                                                               uint8_t* __restrict__ codes, long long ldc, float* __restrict__ scales, int words) {
  struct alignas(sizeof(T) * kLoad) Part { T t[kLoad]; };
  const int lane = threadIdx.x & 31, KB = (K + 127) >> 7, row = blockIdx.x * 8 + (threadIdx.x >> 5);
  grid_dependency_wait();
  grid_launch_dependents();
  if (row >= rows) return;
  const int src = src_row ? src_row[row] : row;
  const bool gone = src < 0 || src >= x_rows;
  const T* from = x + (long long)(gone ? 0 : src) * ldx;
  for (int g0 = blockIdx.y * kAnyGroups; g0 < KB; g0 += gridDim.y * kAnyGroups) {
    float v[kAnyGroups][4];
#pragma unroll
    for (int j = 0; j < kAnyGroups; ++j) {      // all loads in flight
      const int c = (g0 + j) * 128 + lane * 4;
#pragma unroll
      for (int i = 0; i < 4; i += kLoad) {
        if (!gone && c + i + kLoad <= K) {
          const Part w = *reinterpret_cast<const Part*>(from + c + i);
#pragma unroll
          for (int h = 0; h < kLoad; ++h) v[j][i + h] = Elem<T>::load(&w.t[h]);
        } else {
#pragma unroll
          for (int h = 0; h < kLoad; ++h) v[j][i + h] = !gone && c + i + h < K ? Elem<T>::load(from + c + i + h) : 0.f;
        }
      }
    }
#pragma unroll
    for (int j = 0; j < kAnyGroups; ++j) {
      if (g0 + j >= KB) break;
      const int c = (g0 + j) * 128 + lane * 4;
      float m = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) m = max_nan(m, fabsf(v[j][i]));
      m = warp_max(m);
      const Fp8Scale s = fp8_scale(m);
      const uint32_t q = cvt_e4m3x4(v[j][0] * s.factor, v[j][1] * s.factor, v[j][2] * s.factor, v[j][3] * s.factor);
      uint8_t* o = codes + (long long)row * ldc + c;
      if (words && c + 4 <= K) {
        *reinterpret_cast<uint32_t*>(o) = q;
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (c + i < K) o[i] = (uint8_t)(q >> (8 * i));
      }
      if (lane == 0) scales[(long long)row * KB + g0 + j] = gone ? 0.f : s.scale;
    }
  }
}

// 128x128 blocks: one thread block each, its values in registers as they were loaded (64 a thread of 16 bits, 32 of 32). A row of the block is
// 128 consecutive values: 16 (32) lanes of 16 bytes.
template <typename T, bool kVec>
__global__ void __launch_bounds__(Elem<T>::kSize == 2 ? 256 : 512) k_quantize_fp8_blocks(const T* __restrict__ w, int N, int K, uint8_t* __restrict__ codes, long long ldc,
                                                                                         float* __restrict__ scales) {
  constexpr int kThreads = Elem<T>::kSize == 2 ? 256 : 512, kPer = 16 / Elem<T>::kSize, kLanes = 128 / kPer, kRows = kThreads / kLanes, kSteps = 128 / kRows;
  __shared__ float red[kThreads / 32];
  const int kb = blockIdx.x, nb = blockIdx.y, KB = gridDim.x, NB = gridDim.y;
  const long long e = blockIdx.z;
  const int c = kb * 128 + (threadIdx.x % kLanes) * kPer, r0 = nb * 128 + threadIdx.x / kLanes;
  const T* src = w + e * N * K + c;
  grid_dependency_wait();
  grid_launch_dependents();
  uint4 d[kSteps];
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    const int r = r0 + i * kRows;
    d[i] = make_uint4(0u, 0u, 0u, 0u);
    if constexpr (kVec) {
      if (r < N && c < K) d[i] = *reinterpret_cast<const uint4*>(src + (long long)r * K);
    } else if (r < N) {
      T t[kPer];
#pragma unroll
      for (int j = 0; j < kPer; ++j) t[j] = c + j < K ? src[(long long)r * K + j] : Elem<T>::make(0.f);
      memcpy(&d[i], t, 16);
    }
  }
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    float v[kPer];
    unpack16<T>(d[i], v);
#pragma unroll
    for (int j = 0; j < kPer; ++j) m = max_nan(m, fabsf(v[j]));
  }
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
  __syncthreads();
  m = red[0];
#pragma unroll
  for (int i = 1; i < kThreads / 32; ++i) m = max_nan(m, red[i]);
  const Fp8Scale s = fp8_scale(m);
  if (threadIdx.x == 0) scales[(e * NB + nb) * KB + kb] = s.scale;
  uint8_t* dst = codes + e * N * ldc + c;
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    const int r = r0 + i * kRows;
    if (r >= N || c >= K) continue;
    float v[kPer];
    unpack16<T>(d[i], v);
    uint32_t q[kPer / 4];
#pragma unroll
    for (int j = 0; j < kPer / 4; ++j) q[j] = cvt_e4m3x4(v[4 * j] * s.factor, v[4 * j + 1] * s.factor, v[4 * j + 2] * s.factor, v[4 * j + 3] * s.factor);
    if constexpr (kVec) {
      if constexpr (kPer == 8) *reinterpret_cast<uint2*>(dst + (long long)r * ldc) = make_uint2(q[0], q[1]);
      else *reinterpret_cast<uint32_t*>(dst + (long long)r * ldc) = q[0];
    } else {
#pragma unroll
      for (int j = 0; j < kPer; ++j)
        if (c + j < K) dst[(long long)r * ldc + j] = (uint8_t)(q[j / 4] >> (8 * (j & 3)));
    }
  }
}

// Copies by lists where rows are asked for twice or more on average and there are enough of them to pay for two more launches (us, reading the source each time / by
// lists: 8 M values 5.3 / 6.0, 10.7 M twice over 7.1 / 7.1, 16 M 9.1 / 7.3, 88 M twice over 55 / 36).
constexpr long long kListValues = 10 << 20;
static bool by_lists(int x_rows, int rows, int K) { return x_rows > 0 && rows / 2 >= x_rows && (long long)rows * K >= kListValues; }

template <typename T>
static int quantize_fp8_rows(const void* x, long long ldx, int x_rows, const int* src_row, int rows, int K, void* codes, long long ldc, float* scales, int* lists, cudaStream_t st) {
  const long long units = (long long)rows * ((K + 127) / 128);
  const bool vec = K % 16 == 0 && ldx % (16 / Elem<T>::kSize) == 0 && ldc % 16 == 0 && ((uintptr_t)x & 15) == 0 && ((uintptr_t)codes & 15) == 0;
  if (vec && lists) {
    const T* xt = (const T*)x;
    uint8_t* ct = (uint8_t*)codes;
    int *head = lists, *next = lists + x_rows;
    void* a0[] = {&head, &x_rows};
    if (int rc = launch_kernel((const void*)k_no_heads, (x_rows + 255) / 256, 256, 0, true, a0, st)) return rc;
    void* a1[] = {&xt, &ldx, &x_rows, &src_row, &rows, &K, &head, &next, &ct, &ldc, &scales};
    if (int rc = launch_kernel((const void*)k_link_rows<T>, (rows + kLinked - 1) / kLinked, kLinkThreads, 0, true, a1, st)) return rc;
    const long long warps = (long long)x_rows * ((K + 511) / 512);
    if (warps > 8ll * 0x7fffffff) return B200MOE_ERR_LIMIT;
    void* a2[] = {&xt, &ldx, &x_rows, &K, &head, &next, &ct, &ldc, &scales};
    return launch_kernel((const void*)k_quantize_fp8_copies<T>, (int)((warps + 7) / 8), 256, 0, true, a2, st);
  }
  const T* xt = (const T*)x;
  uint8_t* ct = (uint8_t*)codes;
  if (vec) {
    void* args[] = {&xt, &ldx, &x_rows, &src_row, &rows, &K, &ct, &ldc, &scales};
    const long long blocks = (units + 31) / 32;
    return launch_kernel((const void*)k_quantize_fp8_rows<T>, (int)(blocks < 1 << 30 ? blocks : 1 << 30), 256, 0, true, args, st);
  }
  int words = ldc % 4 == 0 && ((uintptr_t)codes & 3) == 0;
  void* args[] = {&xt, &ldx, &x_rows, &src_row, &rows, &K, &ct, &ldc, &scales, &words};
  const auto loads = [&](int n) { return ldx % n == 0 && (uintptr_t)x % (n * sizeof(T)) == 0; };
  const void* fn = loads(4) ? (const void*)k_quantize_fp8_rows_any<T, 4> : loads(2) ? (const void*)k_quantize_fp8_rows_any<T, 2> : (const void*)k_quantize_fp8_rows_any<T, 1>;
  const int quads = ((K + 127) / 128 + kAnyGroups - 1) / kAnyGroups;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((rows + 7) / 8, quads < 65535 ? quads : 65535), cfg.blockDim = dim3(256), cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization, attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr, cfg.numAttrs = 1;
  B200_CUDA_TRY(cudaLaunchKernelExC(&cfg, fn, args));
  return B200MOE_OK;
}

template <typename T>
static int quantize_fp8_blocks(const void* w, int E, int N, int K, void* codes, long long ldc, float* scales, cudaStream_t st) {
  const bool vec = K % 16 == 0 && ldc % 16 == 0 && ((uintptr_t)w & 15) == 0 && ((uintptr_t)codes & 15) == 0;
  const T* wt = (const T*)w;
  uint8_t* ct = (uint8_t*)codes;
  for (int e0 = 0; e0 < E; e0 += 65535) {      // (grid limit of the third dimension)
    const int n = E - e0 < 65535 ? E - e0 : 65535;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((K + 127) / 128, (N + 127) / 128, n), cfg.blockDim = dim3(Elem<T>::kSize == 2 ? 256 : 512), cfg.stream = st;
    const T* we = wt + (long long)e0 * N * K;
    uint8_t* ce = ct + (long long)e0 * N * ldc;
    float* se = scales + (long long)e0 * cfg.gridDim.x * cfg.gridDim.y;
    void* args[] = {&we, &N, &K, &ce, &ldc, &se};
    B200_CUDA_TRY(cudaLaunchKernelExC(&cfg, vec ? (const void*)k_quantize_fp8_blocks<T, true> : (const void*)k_quantize_fp8_blocks<T, false>, args));
  }
  return B200MOE_OK;
}

}  // namespace b200

extern "C" {

long long b200moe_quantize_fp8_workspace_bytes(int x_rows, int rows, int K) {
  if (x_rows < 0 || rows < 0 || K < 1) return B200MOE_ERR_ARG;
  return b200::by_lists(x_rows, rows, K) ? 4ll * ((long long)x_rows + rows) : 0;
}

int b200moe_quantize_fp8(const void* x, int dtype, long long x_stride, int x_rows, const int* src_row, int rows, int K, void* codes, long long codes_stride,
                         float* scales, void* workspace, long long workspace_bytes, void* stream) {
  using namespace b200;
  if (rows < 0 || x_rows < 0 || K < 1 || dtype < 0 || dtype > 2 || (x_stride < K && x_rows > 1) || codes_stride < K) return B200MOE_ERR_ARG;
  if (rows > (1 << 30) || x_rows > (1 << 30) || K > (1 << 30)) return B200MOE_ERR_LIMIT;
  if (rows == 0) return B200MOE_OK;      // (an empty src_row has no address)
  if (!src_row && rows != x_rows) return B200MOE_ERR_ARG;
  if ((!x && x_rows) || !codes || !scales) return B200MOE_ERR_ARG;
  const int size = dtype == DT_F32 ? 4 : 2;
  if (((uintptr_t)x & (size - 1)) || (((uintptr_t)scales | (uintptr_t)workspace | (uintptr_t)src_row) & 3)) return B200MOE_ERR_ARG;
  const long long need = src_row ? b200moe_quantize_fp8_workspace_bytes(x_rows, rows, K) : 0;
  if (need && (!workspace || workspace_bytes < need)) return B200MOE_ERR_WORKSPACE;
  cudaStream_t st = (cudaStream_t)stream;
  int* lists = need ? (int*)workspace : nullptr;
  if (dtype == DT_BF16) return quantize_fp8_rows<__nv_bfloat16>(x, x_stride, x_rows, src_row, rows, K, codes, codes_stride, scales, lists, st);
  if (dtype == DT_F16) return quantize_fp8_rows<__half>(x, x_stride, x_rows, src_row, rows, K, codes, codes_stride, scales, lists, st);
  return quantize_fp8_rows<float>(x, x_stride, x_rows, src_row, rows, K, codes, codes_stride, scales, lists, st);
}

int b200moe_quantize_fp8_blocks(const void* w, int dtype, int E, int N, int K, void* codes, long long codes_stride, float* scales, void* stream) {
  using namespace b200;
  if (E < 0 || N < 0 || K < 1 || dtype < 0 || dtype > 2 || codes_stride < K) return B200MOE_ERR_ARG;
  if (E == 0 || N == 0) return B200MOE_OK;
  if (!w || !codes || !scales) return B200MOE_ERR_ARG;
  if (N > 65535 * 128 || K > (1 << 30)) return B200MOE_ERR_LIMIT;
  const int size = dtype == DT_F32 ? 4 : 2;
  if (((uintptr_t)w & (size - 1)) || ((uintptr_t)scales & 3)) return B200MOE_ERR_ARG;
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == DT_BF16) return quantize_fp8_blocks<__nv_bfloat16>(w, E, N, K, codes, codes_stride, scales, st);
  if (dtype == DT_F16) return quantize_fp8_blocks<__half>(w, E, N, K, codes, codes_stride, scales, st);
  return quantize_fp8_blocks<float>(w, E, N, K, codes, codes_stride, scales, st);
}

}  // extern "C"
