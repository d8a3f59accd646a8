// Matrix product of E4M3 codes with fp32 scales per 1x128 values of the rows and per 128x128 block of the weights:
//   out[m, n] = sum_b sa[m, b] * sb[n / 128, b] * sum_{k in group b} a[m, k] * w[n, k]
// over one matrix, or over a matrix per expert and rows sorted by expert (the tables of the router).
//
// tcgen05 kind::f8f6f4: a group of 128 codes is four 128 x NT x 32 MMAs into a TMEM accumulator of its own, exact products and fp32 sums. The
// scales differ from group to group, so the sum over groups is taken in registers: epilogue warps read each group's accumulator and add it times
// its scale (fp32 fma), while the tensor core fills the next one. One CTA per SM; warps: epilogue | TMA producer | MMA issue | scales.
//   rows on the accumulator's lanes (kSwap false): 128 rows x NT weights, one scale a thread and group
//   weights on the lanes (kSwap true): 128 weights x NT rows; NT follows the rows there are, so that few rows cost few MMA columns, and the inner
//   size may be split over the CTAs of a cluster, which add their sums in rank order through distributed shared memory
#include "common.cuh"
#include "fp8_math.cuh"
#include "tcgen05.cuh"
#include <cudaTypedefs.h>
#include <atomic>

namespace b200 {

constexpr int MM_MAXU = 1024;                     // runs of rows (= ROUTE_MAXE, the most experts the router takes)
__device__ int g_matmul_fp8_status;               // set where a bounded wait ran out; read by b200moe_matmul_fp8_status

struct MatmulParams {
  const float *sa, *sb;
  void* out;
  const int *experts, *offsets;                   // null: one matrix, all rows
  int U, E, M, N, K, KB, NB, out_dtype, zero_rest, vec;
  long long ldo;
};

__device__ __forceinline__ void umma_f8(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate, uint32_t pred) {
  asm volatile(
      "{\n .reg .pred p, q;\n .reg .b64 a, b;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n mov.b64 a, {%1, %6};\n mov.b64 b, {%2, %6};\n"
      " @q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %3, p;\n}\n"
      ::"r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(pred), "n"(kDescHiSw128)
      : "memory");
}
// Instruction descriptor of kind::f8f6f4: fp32 accumulator (1 at bit 4), E4M3 operands (0), both K-major, N >> 3 at bit 17, M >> 4 at bit 24.
__host__ __device__ constexpr uint32_t idesc_f8(int M, int N) { return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24); }

__device__ __forceinline__ void tma_load_2d_u32(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar, uint32_t pred) {
  asm volatile(
      "{\n .reg .pred q;\n setp.ne.b32 q, %5, 0;\n"
      " @q cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n}\n"
      ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar), "r"(pred)
      : "memory");
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

template <int NT, bool kSwap> struct MmShape {
  static constexpr int kEpi = NT >= 128 ? 8 : 4;                  // epilogue warps: two per lane quadrant where a thread's columns would be more than 64 (128: kSwap false)
  static constexpr int kCols = NT / (kEpi / 4);                   // columns of a thread
  static constexpr int kThreads = (kEpi + 3) * 32;
  static constexpr int kStageBytes = 16384 + NT * 128;
  static constexpr int kRed = kSwap ? NT * 128 * 4 : 0;           // sums of a split inner size
  static constexpr int kStages = (200 * 1024 - kRed) / kStageBytes < 9 ? (200 * 1024 - kRed) / kStageBytes : 9;
  static constexpr int kBufs = 512 / NT < 8 ? 512 / NT : 8;       // accumulators in TMEM
  static constexpr int kScaleRow = kSwap ? NT : 132;              // floats of a group's scales
  static constexpr int kRows = kSwap ? NT : 128, kWeights = kSwap ? 128 : NT;      // of a tile
  static constexpr int kSmem = 1024 + kStages * kStageBytes + kRed + kBufs * kScaleRow * 4 + 2 * (MM_MAXU + 2) * 4;
  static_assert(kSmem <= 227 * 1024, "shared memory of a CTA");
};

struct MmTile { int row0, row_end, expert, n0; };

// The t-th tile: row tiles of a run and weight block side by side, so that neighbours share the weights.
template <int NT, bool kSwap>
__device__ __forceinline__ MmTile mm_tile(const MatmulParams& p, const int* first, const int* off, int t) {
  using S = MmShape<NT, kSwap>;
  int u = 0, begin = 0, end = p.M, e = 0;
  if (p.offsets) {
    int lo = 0, hi = p.U;                          // the last run whose first tile is at most t
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (first[mid] <= t) lo = mid; else hi = mid;
    }
    u = lo, t -= first[u], begin = off[u], end = off[u + 1], e = p.experts[u];
  }
  const int mt = (end - begin + S::kRows - 1) / S::kRows;
  const int n = t / mt;
  return {begin + (t - n * mt) * S::kRows, end, e, n * S::kWeights};
}

template <int DT> __device__ __forceinline__ void put(void* out, long long i, float v) {
  if constexpr (DT == DT_BF16) reinterpret_cast<__nv_bfloat16*>(out)[i] = __float2bfloat16_rn(v);
  else if constexpr (DT == DT_F16) reinterpret_cast<__half*>(out)[i] = __float2half_rn(v);
  else reinterpret_cast<float*>(out)[i] = v;
}
// n consecutive values (the whole count where vec: 16-byte stores) of a row
template <int DT, int C> __device__ __forceinline__ void put_row(void* out, long long at, const float (&v)[C], int n, bool vec) {
  if (vec && n >= C) {
    if constexpr (DT == DT_F32) {
      float4* o = reinterpret_cast<float4*>(reinterpret_cast<float*>(out) + at);
#pragma unroll
      for (int i = 0; i < C / 4; ++i) o[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    } else {
      using T = std::conditional_t<DT == DT_BF16, __nv_bfloat16, __half>;
      uint4* o = reinterpret_cast<uint4*>(reinterpret_cast<T*>(out) + at);
#pragma unroll
      for (int i = 0; i < C / 8; ++i)
        o[i] = make_uint4(Elem<T>::pack(v[8 * i], v[8 * i + 1]), Elem<T>::pack(v[8 * i + 2], v[8 * i + 3]), Elem<T>::pack(v[8 * i + 4], v[8 * i + 5]), Elem<T>::pack(v[8 * i + 6], v[8 * i + 7]));
    }
  } else {
#pragma unroll
    for (int i = 0; i < C; ++i)
      if (i < n) put<DT>(out, at + i, v[i]);
  }
}
__device__ __forceinline__ void zero_rows(const MatmulParams& p, int r0, int r1, int first, int step) {
  const int size = p.out_dtype == DT_F32 ? 4 : 2;
  for (int r = r0; r < r1; ++r) {
    uint8_t* row = reinterpret_cast<uint8_t*>(p.out) + (long long)r * p.ldo * size;
    if (p.vec) {
      for (int i = first; i < p.N * size / 16; i += step) reinterpret_cast<uint4*>(row)[i] = make_uint4(0u, 0u, 0u, 0u);
      for (int i = (p.N * size & ~15) / 2 + first; i < p.N * size / 2; i += step) reinterpret_cast<uint16_t*>(row)[i] = 0;
    } else {
      for (int i = first; i < p.N * size / 2; i += step) reinterpret_cast<uint16_t*>(row)[i] = 0;
    }
  }
}

template <int NT, bool kSwap>
__global__ void __launch_bounds__(MmShape<NT, kSwap>::kThreads, 1)
    k_matmul_fp8(const __grid_constant__ CUtensorMap map_rows, const __grid_constant__ CUtensorMap map_weights, const __grid_constant__ MatmulParams p, int split) {
  using S = MmShape<NT, kSwap>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  float* red = reinterpret_cast<float*>(smem + S::kStages * S::kStageBytes);      // [NT][128]
  float* scales = reinterpret_cast<float*>(smem + S::kStages * S::kStageBytes + S::kRed);
  int* first = reinterpret_cast<int*>(scales + S::kBufs * S::kScaleRow);
  int* off = first + MM_MAXU + 1;
  __shared__ uint64_t full[S::kStages], empty[S::kStages], acc_full[S::kBufs], acc_empty[S::kBufs], drained;
  __shared__ uint32_t tmem_base;
  __shared__ int abort_s, wsum[32];
  volatile int* abort_flag = &abort_s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  if (tid == 0) {
    for (int i = 0; i < S::kStages; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], 1);
    for (int i = 0; i < S::kBufs; ++i) mbar_init(&acc_full[i], 2), mbar_init(&acc_empty[i], S::kEpi);
    mbar_init(&drained, 1);
    abort_s = 0;
    fence_mbar_init();
    prefetch_tensormap(&map_rows), prefetch_tensormap(&map_weights);
  }
  if (warp == S::kEpi + 1) {
    tmem_alloc(&tmem_base, S::kBufs * NT);
    tmem_relinquish();
  }
  grid_dependency_wait();

  // The plan: first tile of each run. Offsets are held to 0..M and to their order, runs of an expert that is not there have no tiles.
  int tiles;
  const int ntn = (p.N + S::kWeights - 1) / S::kWeights;
  if (p.offsets) {
    for (int i = tid; i <= p.U; i += S::kThreads) off[i] = min(max(p.offsets[i], 0), p.M);
    __syncthreads();
    const int per = (p.U + S::kThreads - 1) / S::kThreads, u0 = min(tid * per, p.U), u1 = min(u0 + per, p.U);
    int n = 0;
    for (int u = u0; u < u1; ++u) {
      const int e = p.experts[u];
      first[u] = n;
      if (e >= 0 && e < p.E) n += (max(off[u + 1] - off[u], 0) + S::kRows - 1) / S::kRows * ntn;
    }
    int incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) wsum[warp] = incl;
    __syncthreads();
    int base = 0, total = 0;
    for (int w = 0; w < S::kThreads / 32; ++w) {
      if (w < warp) base += wsum[w];
      total += wsum[w];
    }
    for (int u = u0; u < u1; ++u) first[u] += base + incl - n;
    tiles = total;
  } else {
    tiles = (p.M + S::kRows - 1) / S::kRows * ntn;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tb = tmem_base;

  const int rank = split > 1 ? (int)cluster_ctarank() : 0;
  const int t0 = blockIdx.x / split, t_step = gridDim.x / split;
  const int kb0 = p.KB * rank / split, kb1 = p.KB * (rank + 1) / split;
  bool dead = false;       // a wait ran out: the rest of the tiles is walked without work, so that the barriers of a cluster still meet

  if (warp == S::kEpi) {                                             // ---- TMA producer
    const uint32_t el = elect_one();
    int st = 0, ph = 1, issued = 0;
    for (int t = t0; t < tiles; t += t_step) {
      const MmTile tl = mm_tile<NT, kSwap>(p, first, off, t);
      for (int kb = kb0; kb < kb1 && !dead; ++kb) {
        if (!mbar_wait_warp(smem_u32(&empty[st]), ph, abort_flag)) { dead = true; break; }
        const uint32_t bar = smem_u32(&full[st]), sa = smem_u32(smem + st * S::kStageBytes);
        const int wrow = tl.expert * p.N + tl.n0;
        mbar_expect_tx_u32(bar, S::kStageBytes, el);
        tma_load_2d_u32(kSwap ? sa + 16384 : sa, &map_rows, kb * 128, tl.row0, bar, el);
        tma_load_2d_u32(kSwap ? sa : sa + 16384, &map_weights, kb * 128, wrow, bar, el);
        ++issued;
        if (++st == S::kStages) st = 0, ph ^= 1;
      }
      if (split > 1) __syncwarp(), cluster_sync_all(), cluster_sync_all();
    }
    if (dead) {      // copies in flight land before the CTA may end (with a limit)
      for (int i = issued > S::kStages ? issued - S::kStages : 0; i < issued; ++i)
        for (int n = 0; n < 1 << 16 && !mbar_try_wait(&full[i % S::kStages], (i / S::kStages) & 1); ++n) {}
    }
  } else if (warp == S::kEpi + 1) {                                  // ---- MMA issue
    const uint32_t el = elect_one();
    constexpr uint32_t idesc = idesc_f8(128, NT);
    int st = 0, ph = 0, buf = 0, bph = 1;
    for (int t = t0; t < tiles; t += t_step) {
      for (int kb = kb0; kb < kb1 && !dead; ++kb) {
        if (!mbar_wait_warp(smem_u32(&acc_empty[buf]), bph, abort_flag) || !mbar_wait_warp(smem_u32(&full[st]), ph, abort_flag)) { dead = true; break; }
        tc_fence_after();
        const uint32_t a = ((smem_u32(smem + st * S::kStageBytes) >> 4) & 0x3fff) | kDescLoSw128, b = a + (16384 >> 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) umma_f8(tb + buf * NT, a + 2 * j, b + 2 * j, idesc, j != 0, el);
        umma_commit_u32(smem_u32(&empty[st]), el);
        umma_commit_u32(smem_u32(&acc_full[buf]), el);
        if (++st == S::kStages) st = 0, ph ^= 1;
        if (++buf == S::kBufs) buf = 0, bph ^= 1;
      }
      if (split > 1) __syncwarp(), cluster_sync_all(), cluster_sync_all();
    }
    if (dead) {
      umma_commit_u32(smem_u32(&drained), el);
      for (int n = 0; n < 1 << 16 && !mbar_try_wait(&drained, 0); ++n) {}
    }
  } else if (warp == S::kEpi + 2) {                                  // ---- scales: four groups ahead in registers, then a slot beside each accumulator
    constexpr int R = (S::kRows + 31) / 32;
    int buf = 0, bph = 1;
    for (int t = t0; t < tiles; t += t_step) {
      const MmTile tl = mm_tile<NT, kSwap>(p, first, off, t);
      const float* ra[R];
#pragma unroll
      for (int i = 0; i < R; ++i) ra[i] = p.sa + (long long)min(tl.row0 + lane + 32 * i, p.M - 1) * p.KB;
      const int nb = tl.n0 / 128 + (kSwap ? 0 : lane & 1);
      const float* rb = p.sb + ((long long)tl.expert * p.NB + min(nb, p.NB - 1)) * p.KB;
      float va[4][R], vb[4];
      auto fetch = [&](int kb) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int g = min(kb + j, kb1 - 1);
#pragma unroll
          for (int i = 0; i < R; ++i) va[j][i] = __ldg(ra[i] + g);
          vb[j] = __ldg(rb + g);
        }
      };
      if (!dead) fetch(kb0);
      for (int kb = kb0; kb < kb1 && !dead; kb += 4) {
        float ca[4][R], cb[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          cb[j] = vb[j];
#pragma unroll
          for (int i = 0; i < R; ++i) ca[j][i] = va[j][i];
        }
        if (kb + 4 < kb1) fetch(kb + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (kb + j >= kb1) break;
          if (!mbar_wait_warp(smem_u32(&acc_empty[buf]), bph, abort_flag)) { dead = true; break; }
          float* s = scales + buf * S::kScaleRow;
#pragma unroll
          for (int i = 0; i < R; ++i)
            if (lane + 32 * i < S::kRows) s[lane + 32 * i] = kSwap ? ca[j][i] * cb[j] : ca[j][i];
          if (!kSwap && lane < 2) s[128 + lane] = cb[j];
          __syncwarp();
          if (lane == 0) mbar_arrive(&acc_full[buf]);
          if (++buf == S::kBufs) buf = 0, bph ^= 1;
        }
      }
      if (split > 1) __syncwarp(), cluster_sync_all(), cluster_sync_all();
    }
  } else {                                                           // ---- epilogue
    const int quad = warp & 3, half = warp >> 2, col0 = half * S::kCols;
    const int l = quad * 32 + lane;                                  // accumulator lane
    int buf = 0, ph = 0;
    for (int t = t0; t < tiles; t += t_step) {
      const MmTile tl = mm_tile<NT, kSwap>(p, first, off, t);
      float acc[S::kCols];
#pragma unroll
      for (int i = 0; i < S::kCols; ++i) acc[i] = 0.f;
      for (int kb = kb0; kb < kb1 && !dead; ++kb) {
        if (!mbar_wait_warp(smem_u32(&acc_full[buf]), ph, abort_flag)) { dead = true; break; }
        tc_fence_after();
        const float* s = scales + buf * S::kScaleRow;
        const uint32_t taddr = tb + buf * NT + col0 + ((uint32_t)(quad * 32) << 16);
        const float sr = kSwap ? 0.f : s[l] * s[128 + half];
        uint32_t v[2][16];
        tmem_ld_32x32b_x16(taddr, v[0]);
#pragma unroll
        for (int c = 0; c < S::kCols / 16; ++c) {
          tmem_ld_wait();
          if (c + 1 < S::kCols / 16) tmem_ld_32x32b_x16(taddr + 16 * (c + 1), v[(c + 1) & 1]);
#pragma unroll
          for (int i = 0; i < 16; i += 4) {
            if constexpr (kSwap) {
              const float4 sc = *reinterpret_cast<const float4*>(s + col0 + c * 16 + i);
              acc[c * 16 + i] = fmaf(__uint_as_float(v[c & 1][i]), sc.x, acc[c * 16 + i]);
              acc[c * 16 + i + 1] = fmaf(__uint_as_float(v[c & 1][i + 1]), sc.y, acc[c * 16 + i + 1]);
              acc[c * 16 + i + 2] = fmaf(__uint_as_float(v[c & 1][i + 2]), sc.z, acc[c * 16 + i + 2]);
              acc[c * 16 + i + 3] = fmaf(__uint_as_float(v[c & 1][i + 3]), sc.w, acc[c * 16 + i + 3]);
            } else {
#pragma unroll
              for (int j = 0; j < 4; ++j) acc[c * 16 + i + j] = fmaf(__uint_as_float(v[c & 1][i + j]), sr, acc[c * 16 + i + j]);
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&acc_empty[buf]);
        if (++buf == S::kBufs) buf = 0, ph ^= 1;
      }
      if constexpr (!kSwap) {
        const int row = tl.row0 + l, n = tl.n0 + col0;
        if (!dead && row < tl.row_end && n < p.N) {
          const long long at = (long long)row * p.ldo + n;
          if (p.out_dtype == DT_BF16) put_row<DT_BF16>(p.out, at, acc, p.N - n, p.vec);
          else if (p.out_dtype == DT_F16) put_row<DT_F16>(p.out, at, acc, p.N - n, p.vec);
          else put_row<DT_F32>(p.out, at, acc, p.N - n, p.vec);
        }
      } else {
        if (split == 1) {
          const int n = tl.n0 + l;
          if (!dead && n < p.N) {
#pragma unroll
            for (int i = 0; i < S::kCols; ++i) {
              const int row = tl.row0 + col0 + i;
              if (row < tl.row_end) {
                const long long at = (long long)row * p.ldo + n;
                if (p.out_dtype == DT_BF16) put<DT_BF16>(p.out, at, acc[i]);
                else if (p.out_dtype == DT_F16) put<DT_F16>(p.out, at, acc[i]);
                else put<DT_F32>(p.out, at, acc[i]);
              }
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < S::kCols; ++i) red[(col0 + i) * 128 + l] = acc[i];
          __syncwarp();
          cluster_sync_all();
          if (!dead) {
            for (int i = tid + rank * S::kEpi * 32; i < NT * 128; i += split * S::kEpi * 32) {
              const int row = tl.row0 + i / 128, n = tl.n0 + (i & 127);
              if (row >= tl.row_end || n >= p.N) continue;
              float v = 0.f;
              const uint32_t mine = smem_u32(red + i);
              for (int r = 0; r < split; ++r) v += ld_cluster_f32(mapa_shared(mine, r));
              const long long at = (long long)row * p.ldo + n;
              if (p.out_dtype == DT_BF16) put<DT_BF16>(p.out, at, v);
              else if (p.out_dtype == DT_F16) put<DT_F16>(p.out, at, v);
              else put<DT_F32>(p.out, at, v);
            }
          }
          __syncwarp();
          cluster_sync_all();      // the peers' sums stay until everybody has read them
        }
      }
    }
    if (p.offsets && p.zero_rest) {      // rows outside every run, and of experts that are not there
      const int step = gridDim.x * S::kEpi * 32, me = blockIdx.x * S::kEpi * 32 + tid;
      for (int u = 0; u < p.U; ++u) {
        const int e = p.experts[u];
        if (e < 0 || e >= p.E) zero_rows(p, off[u], off[u + 1], me, step);
      }
      if (off[0] > 0) zero_rows(p, 0, off[0], me, step);
      zero_rows(p, off[p.U], p.M, me, step);
    }
  }
  if (dead) atomicExch(&g_matmul_fp8_status, 1);
  tc_fence_before();
  __syncthreads();
  if (warp == S::kEpi + 1) tmem_dealloc(tb, S::kBufs * NT);
}

static PFN_cuTensorMapEncodeTiled_v12000 map_encoder() {
  static std::atomic<void*> fn{nullptr};
  void* p = fn.load(std::memory_order_acquire);
  if (!p) {
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) return nullptr;
    fn.store(p, std::memory_order_release);
  }
  return (PFN_cuTensorMapEncodeTiled_v12000)p;
}
// E4M3 matrix of `rows` rows of K codes, `stride` bytes apart: boxes of 128 codes x box_rows, 128-byte swizzle, zeros beyond the matrix
static int codes_map(CUtensorMap* map, const void* base, long long rows, int K, long long stride, int box_rows) {
  auto enc = map_encoder();
  if (!enc) return B200MOE_ERR_DEVICE;
  cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)stride};
  cuuint32_t box[2] = {128u, (cuuint32_t)box_rows}, estr[2] = {1u, 1u};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? B200MOE_OK : B200MOE_ERR_ARG;
}

static int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  return n;
}

template <int NT, bool kSwap>
static int launch_matmul(const MatmulParams& p, const void* a, long long lda, const void* w, long long ldw, long long tiles, int split, int sms, cudaStream_t st) {
  using S = MmShape<NT, kSwap>;
  CUtensorMap rows, weights;
  if (int rc = codes_map(&rows, a, p.M, p.K, lda, S::kRows)) return rc;
  if (int rc = codes_map(&weights, w, (long long)p.E * p.N, p.K, ldw, S::kWeights)) return rc;
  const void* fn = (const void*)k_matmul_fp8<NT, kSwap>;
  B200_CUDA_TRY(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem));
  const long long most = sms / split;
  const int clusters = (int)(tiles < most ? (tiles > 0 ? tiles : 1) : most);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(clusters * split), cfg.blockDim = dim3(S::kThreads), cfg.dynamicSmemBytes = S::kSmem, cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization, attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = split, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr, cfg.numAttrs = split > 1 ? 2 : 1;
  MatmulParams q = p;
  void* args[] = {&rows, &weights, &q, &split};
  B200_CUDA_TRY(cudaLaunchKernelExC(&cfg, fn, args));
  return B200MOE_OK;
}

// Which form: rows on the lanes (128 x 256 tiles) where a run of rows fills them and the tiles fill the SMs, otherwise weights on the lanes with
// the rows' tile that a run needs; there the inner size is split while SMs are idle and a CTA keeps two groups.
static int matmul(const MatmulParams& p, const void* a, long long lda, const void* w, long long ldw, cudaStream_t st) {
  const int sms = sm_count();
  if (sms <= 0) return B200MOE_ERR_DEVICE;
  const long long runs = p.offsets ? (p.U < p.M ? p.U : p.M) : 1, mean = p.M / runs;
  const auto tiles = [&](int r, int c) { return (p.M / r + (p.offsets ? runs : (p.M % r != 0))) * ((p.N + c - 1) / c); };      // (at most)
  if (mean >= 96 && tiles(128, 256) >= sms / 2) return launch_matmul<256, false>(p, a, lda, w, ldw, tiles(128, 256), 1, sms, st);
  const int nt = mean <= 16 ? 16 : mean <= 32 ? 32 : mean <= 64 ? 64 : 128;
  const long long n = tiles(nt, 128);
  int split = 1;
  while (split < 8 && n * split * 2 <= sms && p.KB >= split * 4) split *= 2;
  switch (nt) {
    case 16: return launch_matmul<16, true>(p, a, lda, w, ldw, n, split, sms, st);
    case 32: return launch_matmul<32, true>(p, a, lda, w, ldw, n, split, sms, st);
    case 64: return launch_matmul<64, true>(p, a, lda, w, ldw, n, split, sms, st);
    default: return launch_matmul<128, true>(p, a, lda, w, ldw, n, split, sms, st);
  }
}

static int matmul_args(const void* a, long long lda, const float* sa, const void* w, long long ldw, const float* sw, int M, int N, int K, void* out, int out_dtype,
                       long long ldo) {
  if (M < 0 || N < 0 || K < 1 || out_dtype < 0 || out_dtype > 2 || lda < K || ldw < K || ldo < N) return B200MOE_ERR_ARG;
  if (M == 0 || N == 0) return B200MOE_OK;
  if (!a || !sa || !w || !sw || !out) return B200MOE_ERR_ARG;
  if ((((uintptr_t)a | (uintptr_t)w | lda | ldw) & 15) || (((uintptr_t)sa | (uintptr_t)sw) & 3) || ((uintptr_t)out & (out_dtype == DT_F32 ? 3 : 1))) return B200MOE_ERR_ARG;
  if (M > (1 << 30) || N > (1 << 30) || K > (1 << 30)) return B200MOE_ERR_LIMIT;
  return B200MOE_OK;
}
static int stores_16(const void* out, int out_dtype, long long ldo) { return ((uintptr_t)out & 15) == 0 && (ldo * (out_dtype == DT_F32 ? 4 : 2)) % 16 == 0; }

}  // namespace b200

extern "C" {

int b200moe_matmul_fp8(const void* a, long long a_stride, const float* a_scales, const void* w, long long w_stride, const float* w_scales, int M, int N, int K,
                       void* out, int out_dtype, long long out_stride, void* stream) {
  using namespace b200;
  if (int rc = matmul_args(a, a_stride, a_scales, w, w_stride, w_scales, M, N, K, out, out_dtype, out_stride)) return rc;
  if (M == 0 || N == 0) return B200MOE_OK;
  const MatmulParams p = {a_scales, w_scales, out, nullptr, nullptr, 0, 1, M, N, K, (K + 127) / 128, (N + 127) / 128, out_dtype, 0, stores_16(out, out_dtype, out_stride), out_stride};
  return matmul(p, a, a_stride, w, w_stride, (cudaStream_t)stream);
}

int b200moe_matmul_fp8_experts(const void* a, long long a_stride, const float* a_scales, int rows, const void* w, long long w_stride, const float* w_scales, int E,
                               const int* experts, const int* offsets, int runs, int N, int K, void* out, int out_dtype, long long out_stride, int zero_rest, void* stream) {
  using namespace b200;
  if (E < 1 || runs < 0) return B200MOE_ERR_ARG;
  if (int rc = matmul_args(a, a_stride, a_scales, w, w_stride, w_scales, rows, N, K, out, out_dtype, out_stride)) return rc;
  if (runs > MM_MAXU || (long long)E * N > (1ll << 31) - 512) return B200MOE_ERR_LIMIT;
  if (rows == 0 || N == 0) return B200MOE_OK;
  if (runs == 0) {
    const size_t size = out_dtype == DT_F32 ? 4 : 2;
    if (zero_rest) B200_CUDA_TRY(cudaMemset2DAsync(out, out_stride * size, 0, N * size, rows, (cudaStream_t)stream));
    return B200MOE_OK;
  }
  if (!experts || !offsets) return B200MOE_ERR_ARG;
  const MatmulParams p = {a_scales, w_scales, out, experts, offsets, runs, E, rows, N, K, (K + 127) / 128, (N + 127) / 128, out_dtype, zero_rest,
                          stores_16(out, out_dtype, out_stride), out_stride};
  return matmul(p, a, a_stride, w, w_stride, (cudaStream_t)stream);
}

int b200moe_matmul_fp8_status(void* stream) {
  int v = 0;
  B200_CUDA_TRY(cudaMemcpyFromSymbolAsync(&v, b200::g_matmul_fp8_status, sizeof v, 0, cudaMemcpyDeviceToHost, (cudaStream_t)stream));
  B200_CUDA_TRY(cudaStreamSynchronize((cudaStream_t)stream));
  if (!v) return B200MOE_OK;
  v = 0;
  B200_CUDA_TRY(cudaMemcpyToSymbolAsync(b200::g_matmul_fp8_status, &v, sizeof v, 0, cudaMemcpyHostToDevice, (cudaStream_t)stream));
  B200_CUDA_TRY(cudaStreamSynchronize((cudaStream_t)stream));
  return B200MOE_ERR_TIMEOUT;
}

}  // extern "C"
