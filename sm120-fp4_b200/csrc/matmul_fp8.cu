// Matrix product of E4M3 codes with fp32 scales per 1x128 values of the rows and per 128x128 block of the weights:
//   out[m, n] = sum_b sa[m, b] * sb[n / 128, b] * sum_{k in group b} a[m, k] * w[n, k]
// over one matrix, or over a matrix per expert and rows sorted by expert (the tables of the router).
//
// tcgen05 kind::f8f6f4: a group of 128 codes is four 128 x NT x 32 MMAs into a TMEM accumulator of its own, exact products and fp32 sums. The
// scales differ from group to group, so the sum over groups is taken in registers: epilogue warps read each group's accumulator and add it times
// its scale (fp32 fma), while the tensor core fills the next one. One CTA per SM; warps: epilogue | TMA producer | MMA issue | scales.
//   rows on the accumulator's lanes (kSwap false): 128 rows x 256 weights a CTA, one scale a thread and group; kPair: 256 x 256 of a CTA pair, each of which
//   brings half of both operands, so that shared memory takes 128 bytes a cycle at the tensor core's full rate instead of 192
//   weights on the lanes (kSwap true): 128 weights x NT rows; NT follows the rows there are, so that few rows cost few MMA columns, and the inner
//   size may be split over the CTAs of a cluster, which add their sums in rank order through distributed shared memory
// What bounds it, measured: 8192 x 4096 x 4096 in pairs takes 127 us (2150 TFLOP/s) from a cold chip and 145 us at the power limit (990 W, 1500 MHz). A step of 128 codes
// takes a pair about 780 cycles: the MMAs 512, and between them the accumulator's round trip (commit 140, reading 390 with the tensor core at
// work, arrivals and the look at the barrier 250) over two accumulators, all that TMEM holds of 256 columns. Single CTAs read 9.9 TB/s out of L2 for 128 experts of
// 1408 x 2816 and 2050 tokens (126 us). Few rows are bound by the weights' stream: 16 tokens on 128 experts of 1536 x 2048, 260 MB in 46.5 us; a step takes
// an SM 630 cycles, of which HBM's share is all.
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
  int give_up;                                    // 0; of the probe: whose waits run out at their first look
};
// Looks at a barrier until a role gives its wait up.
enum { kRoleProducer = 1, kRoleMma = 2, kRoleScales = 4, kRoleEpilogue = 8, kRoleFirstOfPair = 16 };
template <int kRole> __device__ __forceinline__ uint32_t looks_of(const MatmulParams& p, int rank) {
  return p.give_up && (p.give_up & kRole) && !(p.give_up & kRoleFirstOfPair && rank) ? 0u : 1u << 20;
}

__device__ __forceinline__ void umma_f8(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate, uint32_t pred) {
  asm volatile(
      "{\n .reg .pred p, q;\n .reg .b64 a, b;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n mov.b64 a, {%1, %6};\n mov.b64 b, {%2, %6};\n"
      " @q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %3, p;\n}\n"
      ::"r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(pred), "n"(kDescHiSw128)
      : "memory");
}
__device__ __forceinline__ void umma2_f8(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate, uint32_t pred) {
  asm volatile(
      "{\n .reg .pred p, q;\n .reg .b64 a, b;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n mov.b64 a, {%1, %6};\n mov.b64 b, {%2, %6};\n"
      " @q tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], a, b, %3, p;\n}\n"
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
// The same for a CTA pair: the copy lands in this CTA's shared memory and its bytes count at a barrier of either CTA (a cluster address).
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar, uint32_t pred) {
  asm volatile(
      "{\n .reg .pred q;\n setp.ne.b32 q, %5, 0;\n"
      " @q cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n}\n"
      ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar), "r"(pred)
      : "memory");
}
// Arrivals of one lane (pred) without a branch. The one at a barrier of any CTA of the cluster orders no memory: what it hands over is TMEM, ordered by the tcgen05
// fences, and with cluster-wide release it held the epilogue up for 900 cycles.
__device__ __forceinline__ void mbar_arrive_cluster_p(uint32_t bar, uint32_t pred) {
  asm volatile("{\n .reg .pred q;\n setp.ne.b32 q, %1, 0;\n @q mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];\n}\n" ::"r"(bar), "r"(pred) : "memory");
}
__device__ __forceinline__ void mbar_arrive_p(uint32_t bar, uint32_t pred) {
  asm volatile("{\n .reg .pred q;\n setp.ne.b32 q, %1, 0;\n @q mbarrier.arrive.shared::cta.b64 _, [%0];\n}\n" ::"r"(bar), "r"(pred) : "memory");
}
__device__ __forceinline__ bool mbar_ready(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return __all_sync(0xffffffffu, ok != 0);
}
// How many of the next `steps` steps (kPer barriers each, one a lane in order, 32 / kPer steps at most) are ready, one at least; 0 where the wait ran out. A look at a
// barrier takes 120 cycles; a look at all of them by different lanes takes no longer.
template <int kPer> __device__ __forceinline__ int mbar_wait_steps(uint32_t bar, uint32_t parity, int steps, int lane, volatile int* abort_flag, uint32_t limit = (1u << 20)) {
  uint32_t ok = 1;
  if (lane < steps * kPer)
    asm volatile("{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  const uint32_t open = ~__ballot_sync(0xffffffffu, ok != 0);
  const int ready = open ? (__ffs(open) - 1) / kPer : steps;
  __syncwarp();      // (what a lane has seen holds for all)
  if (ready) return ready < steps ? ready : steps;
  for (uint32_t it = 0; it < limit; ++it) {      // the first step: parked in the barrier
    ok = 1;
    if (lane < kPer)
      asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    if (__all_sync(0xffffffffu, ok != 0)) {
      __syncwarp();
      return 1;
    }
    if ((it & 63u) == 63u && __any_sync(0xffffffffu, *abort_flag != 0)) return 0;
  }
  *abort_flag = 1;
  return 0;
}
// mbar_wait_warp with a barrier of its own for each lane that is not done
__device__ __forceinline__ bool mbar_wait_lanes(uint32_t bar, uint32_t parity, bool done, volatile int* abort_flag, uint32_t limit = (1u << 20)) {
  for (uint32_t it = 0; it < limit; ++it) {
    uint32_t ok = 1;
    if (!done)
      asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    if (__all_sync(0xffffffffu, ok != 0)) return true;
    if ((it & 63u) == 63u && __any_sync(0xffffffffu, *abort_flag != 0)) return false;
  }
  *abort_flag = 1;
  return false;
}
__device__ __forceinline__ void st_cluster_u32(uint32_t addr, uint32_t v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }
__device__ __forceinline__ void st_cluster_f32(uint32_t addr, float v) { asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory"); }
__device__ __forceinline__ void tmem_ld_32x32b_x32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]),
        "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
template <int C> __device__ __forceinline__ void tmem_ld_cols(uint32_t taddr, uint32_t (&r)[C]) {
  if constexpr (C == 32) tmem_ld_32x32b_x32(taddr, r);
  else tmem_ld_32x32b_x16(taddr, r);
}
// a pair of fp32 fma in one instruction, each rounded as fmaf
__device__ __forceinline__ void fma2(float& a0, float& a1, uint32_t x0, uint32_t x1, float s0, float s1) {
  asm("{\n .reg .b64 a, x, s;\n mov.b64 a, {%0, %1};\n mov.b64 x, {%2, %3};\n mov.b64 s, {%4, %5};\n fma.rn.f32x2 a, x, s, a;\n mov.b64 {%0, %1}, a;\n}\n"
      : "+f"(a0), "+f"(a1) : "r"(x0), "r"(x1), "f"(s0), "f"(s1));
}
template <int R> __device__ __forceinline__ void regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R)); }
template <int R> __device__ __forceinline__ void regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R)); }

template <int NT, bool kSwap, bool kPair> struct MmShape {
  static constexpr int kEpi = NT >= 128 ? 8 : 4;                  // epilogue warps: two per lane quadrant where a thread's columns would be more than 64 (128: kSwap false)
  static constexpr int kCols = NT / (kEpi / 4);                   // columns of a thread
  static constexpr int kChunk = kCols < 32 ? kCols : 32;          // columns of a TMEM load
  // 128 sums and 64 values in flight a thread: registers go from the other warps (a warpgroup of four, one idle) to the epilogue's eight. A launch of 12 warps has
  // 168 a thread: 8 * kEpiRegs + 4 * (504 - 2 * kEpiRegs) = 12 * 168. Both shares are those with which ptxas spills nothing (192 / 120 spilled and took 148
  // instead of 126 us at 8192 x 4096 x 4096).
  static constexpr int kEpiRegs = kPair ? 184 : 176;
  static constexpr bool kSplitRegs = kCols == 128;
  static constexpr int kThreads = kSplitRegs ? 384 : (kEpi + 3) * 32;
  static constexpr int kBRows = kPair ? NT / 2 : NT;              // rows of the B operand in this CTA's shared memory
  static constexpr int kStageBytes = 16384 + kBRows * 128;
  static constexpr int kRed = kSwap ? NT * 128 * 4 : 0;           // sums of a split inner size
  static constexpr int kOutWarp = kSwap ? 0 : 8192;               // a warp's sums on their way out: two boxes of 32 rows x 128 bytes
  static constexpr int kOut = kEpi * kOutWarp;
  static constexpr int kRing = 218 * 1024 - kRed - kOut;
  static constexpr int kStages = kRing / kStageBytes < 9 ? kRing / kStageBytes : 9;
  static constexpr int kBufs = 512 / NT < 8 ? 512 / NT : 8;       // accumulators in TMEM
  static constexpr int kScaleRow = kSwap ? NT : 132;              // floats of a group's scales
  static constexpr int kAhead = kBufs < 4 ? kBufs : 4;            // steps looked at together
  static constexpr int kRows = kSwap ? NT : kPair ? 256 : 128, kWeights = kSwap ? 128 : NT;      // of a tile
  static constexpr int kSmem = 1024 + kStages * kStageBytes + kRed + kOut + kBufs * kScaleRow * 4 + 2 * (MM_MAXU + 2) * 4;
  static_assert(kSmem <= 226 * 1024, "shared memory of a CTA");
};

// First accumulator column of a warp's c-th chunk: its own half of the tile, or (kSwap, where rows may be few) chunks in turn.
template <int NT, bool kSwap, bool kPair> __device__ __forceinline__ int mm_column(int half, int c) {
  using S = MmShape<NT, kSwap, kPair>;
  return kSwap ? (c * (S::kEpi / 4) + half) * S::kChunk : half * S::kCols + c * S::kChunk;
}

struct MmTile { int row0, row_end, expert, n0; };

// Rounds of a worker (a CTA, or a pair): a tile each. kParts: the tiles that are left for the last round are cut along the inner size into as many parts as leave no
// worker without one, up to the cluster (parts of a tile are neighbours in a cluster), with two groups at least in a part; every worker has that round.
template <bool kParts> struct MmRounds {
  int tiles, worker, workers, KB, full = 0, rest = 0, log_parts = 0;
  __device__ __forceinline__ MmRounds(int tiles, int worker, int workers, int KB, int cluster) : tiles(tiles), worker(worker), workers(workers), KB(KB) {
    if constexpr (kParts) {
      full = tiles / workers, rest = tiles - full * workers, log_parts = 31 - __clz(cluster);
      while (log_parts > 0 && ((rest << log_parts) > workers || KB < (2 << log_parts))) --log_parts;
    }
  }
  __device__ __forceinline__ bool has(int i) const {
    if constexpr (kParts) return i < full + (rest > 0);
    else return i * workers + worker < tiles;
  }
  __device__ __forceinline__ bool shared(int i) const { return kParts && i == full && log_parts > 0; }
  // tile of round i (-1: none) and its groups
  __device__ __forceinline__ int tile(int i, int& kb0, int& kb1) const {
    kb0 = 0, kb1 = KB;
    if constexpr (kParts) {
      if (i == full) {
        const int j = worker >> log_parts, r = worker & ((1 << log_parts) - 1);
        kb0 = (KB * r) >> log_parts, kb1 = (KB * (r + 1)) >> log_parts;      // (KB < 2^24, at most 8 parts)
        if (j >= rest) {
          kb1 = kb0;
          return -1;
        }
        return full * workers + j;
      }
    }
    return i * workers + worker;
  }
};

// The t-th tile: row tiles of a run and weight block side by side, so that neighbours share the weights.
template <int NT, bool kSwap, bool kPair>
__device__ __forceinline__ MmTile mm_tile(const MatmulParams& p, const int* first, const int* off, int t) {
  using S = MmShape<NT, kSwap, kPair>;
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
// n values of a row, one at a time
template <int DT, int C> __device__ __forceinline__ void put_some(void* out, long long at, const float (&v)[C], int n) {
#pragma unroll
  for (int i = 0; i < C; ++i)
    if (i < n) put<DT>(out, at + i, v[i]);
}
// A warp's 32 rows x 128 columns (a row a thread) to the output, by way of boxes of 32 rows x 128 bytes in shared memory, chunks of 16 bytes turned by the row as the
// copy engine's 128-byte swizzle has them. A box goes out in one copy, which the next tile's math does not wait for: all SMs end their tiles at about the same
// time, and 5900 cycles passed until the threads' own stores (16 bytes of 32 rows an instruction) had left; a copy for each row took the engine 256 of them a
// tile. Rows beyond the run's end, and rows that do not start (or end) on 16 bytes, are stored by the warp, row by row.
template <int DT> __device__ __forceinline__ void put_rows(const MatmulParams& p, const CUtensorMap* map_out, uint8_t* buf, const float (&acc)[128], int row0, int row_end, int n,
                                                           int lane) {
  constexpr int kSize = DT == DT_F32 ? 4 : 2, kCols = 128 / kSize;      // columns of a box
  // The copy stores nothing beyond the matrix: no rows, but along a row whole 16 bytes only.
  const bool rows_whole = p.vec && (row0 + 32 <= row_end || row_end == p.M), ends_on_16 = (long long)p.N * kSize % 16 == 0;
#pragma unroll
  for (int c0 = 0; c0 < 128; c0 += kCols) {
    if (n + c0 >= p.N) break;
    uint8_t* box = buf + (c0 / kCols & 1) * 4096;
    if (lane == 0) {      // the last copy from this box has left: the tile before's, or of this tile the one before the last
      if (c0 == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
      else if (c0 >= 2 * kCols) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
    }
    __syncwarp();
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      uint4 w;
      const float* v = acc + c0 + q * 16 / kSize;
      if constexpr (DT == DT_F32) {
        w = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
      } else {
        using T = std::conditional_t<DT == DT_BF16, __nv_bfloat16, __half>;
        w = make_uint4(Elem<T>::pack(v[0], v[1]), Elem<T>::pack(v[2], v[3]), Elem<T>::pack(v[4], v[5]), Elem<T>::pack(v[6], v[7]));
      }
      *reinterpret_cast<uint4*>(box + lane * 128 + ((q ^ (lane & 7)) << 4)) = w;
    }
    if (rows_whole && (ends_on_16 || n + c0 + kCols <= p.N)) {
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0)
        asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];\n cp.async.bulk.commit_group;" ::"l"(map_out), "r"((n + c0) * kSize), "r"(row0),
                     "r"(smem_u32(box)) : "memory");
    } else {
      __syncwarp();
      const int rows = min(32, row_end - row0);
      uint8_t* o = reinterpret_cast<uint8_t*>(p.out) + ((long long)row0 * p.ldo + n + c0) * kSize;
      if (p.vec) {      // four rows an instruction
        const int left = (p.N - n - c0) * kSize - (lane & 7) * 16;      // bytes of a row from this lane's chunk on
        for (int r = lane >> 3; r < rows; r += 4) {
          const uint8_t* from = box + r * 128 + (((lane & 7) ^ (r & 7)) << 4);
          uint8_t* to = o + r * p.ldo * kSize + (lane & 7) * 16;
          if (left >= 16) *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(from);
          else
            for (int i = 0; i < left; i += kSize) {
              if constexpr (kSize == 4) *reinterpret_cast<uint32_t*>(to + i) = *reinterpret_cast<const uint32_t*>(from + i);
              else *reinterpret_cast<uint16_t*>(to + i) = *reinterpret_cast<const uint16_t*>(from + i);
            }
        }
      } else {
        const int cols = min(kCols, p.N - n - c0);
        for (int r = 0; r < rows; ++r)
#pragma unroll
          for (int i = 0; i < kCols / 32; ++i) {
            const int c = i * 32 + lane, at = c * kSize;
            const uint8_t* from = box + r * 128 + (((at >> 4) ^ (r & 7)) << 4) + (at & 15);
            uint8_t* to = o + (r * p.ldo + c) * kSize;
            if (c < cols) {
              if constexpr (kSize == 4) *reinterpret_cast<uint32_t*>(to) = *reinterpret_cast<const uint32_t*>(from);
              else *reinterpret_cast<uint16_t*>(to) = *reinterpret_cast<const uint16_t*>(from);
            }
          }
      }
    }
  }
}
// four weights' sums of a row
__device__ __forceinline__ void put_four(const MatmulParams& p, int row, int n, const float (&o)[4]) {
  const long long at = (long long)row * p.ldo + n;
  if (p.out_dtype == DT_F32) {
    if (p.vec && n + 4 <= p.N) *reinterpret_cast<float4*>(reinterpret_cast<float*>(p.out) + at) = make_float4(o[0], o[1], o[2], o[3]);
    else put_some<DT_F32>(p.out, at, o, p.N - n);
  } else if (p.out_dtype == DT_BF16) {
    if (p.vec && n + 4 <= p.N) *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(p.out) + at) = make_uint2(Elem<__nv_bfloat16>::pack(o[0], o[1]), Elem<__nv_bfloat16>::pack(o[2], o[3]));
    else put_some<DT_BF16>(p.out, at, o, p.N - n);
  } else {
    if (p.vec && n + 4 <= p.N) *reinterpret_cast<uint2*>(reinterpret_cast<__half*>(p.out) + at) = make_uint2(Elem<__half>::pack(o[0], o[1]), Elem<__half>::pack(o[2], o[3]));
    else put_some<DT_F16>(p.out, at, o, p.N - n);
  }
}
// A tile whose inner size is split over kRanks CTAs: rank r sums the columns (rows of the output) r * NT / kRanks .., to which every CTA has stored its part: red is
// [rank it came from][column][128 weights] there. Sums in rank order; a thread takes four weights of a row at a time.
template <int NT, int kRanks>
__device__ __forceinline__ void mm_add_ranks(const MatmulParams& p, const MmTile& tl, const float* red, int cluster_rank, int tid) {
  using S = MmShape<NT, true, false>;
  constexpr int kThreads = S::kEpi * 32, kItems = NT * 32 / kRanks;
  const int rank = cluster_rank & (kRanks - 1);
  for (int i = tid; i < kItems; i += kThreads) {
    const int row = tl.row0 + rank * (NT / kRanks) + i / 32, n = tl.n0 + (i & 31) * 4;
    if (row >= tl.row_end || n >= p.N) continue;
    float4 v[kRanks];
#pragma unroll
    for (int r = 0; r < kRanks; ++r) v[r] = *reinterpret_cast<const float4*>(red + (r * kItems + i) * 4);
    float o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int r = 0; r < kRanks; ++r) o[0] += v[r].x, o[1] += v[r].y, o[2] += v[r].z, o[3] += v[r].w;
    put_four(p, row, n, o);
  }
}
// Rows r0 .. r1 - 1 to zeros, by all warps of the grid that come here: a piece of 2048 bytes of a row each in turn, so that neither few long rows nor many short ones
// are left to a few SMs (32768 rows of 1536 bf16, half of them padding: 109 us, as without the zeros; with the grid's
// threads along one row, of which the first 192 have something to store, 1650). 262144 rows of 2816, half: 295 us, 193 without (737 MB at 7.2 TB/s).
__device__ __forceinline__ void zero_rows(const MatmulParams& p, int r0, int r1, int warp, int warps, int lane) {
  const int size = p.out_dtype == DT_F32 ? 4 : 2;
  const long long row_bytes = (long long)p.N * size;
  const int pieces = (int)((row_bytes + 2047) >> 11);      // (of a row: N is at most 2^30)
  const long long first = (long long)r0 * pieces, end = (long long)r1 * pieces;      // pieces are numbered from row 0 on: several short runs have different warps
  for (long long u = first + (warp + warps - (int)(first % warps)) % warps; u < end; u += warps) {
    const long long r = u / pieces, from = (u - r * pieces) << 11;
    uint8_t* at = reinterpret_cast<uint8_t*>(p.out) + r * p.ldo * size + from;
    const int n = (int)min(row_bytes - from, 2048ll), whole = p.vec ? n & ~15 : 0;
    for (int i = lane * 16; i < whole; i += 512) *reinterpret_cast<uint4*>(at + i) = make_uint4(0u, 0u, 0u, 0u);
    for (int i = whole + lane * 2; i < n; i += 64) *reinterpret_cast<uint16_t*>(at + i) = 0;
  }
}

template <int NT, bool kSwap, bool kPair>
__global__ void __launch_bounds__(MmShape<NT, kSwap, kPair>::kThreads, 1)
    k_matmul_fp8(const __grid_constant__ CUtensorMap map_rows, const __grid_constant__ CUtensorMap map_weights, const __grid_constant__ CUtensorMap map_out,
                 const __grid_constant__ MatmulParams p, int cluster) {
  using S = MmShape<NT, kSwap, kPair>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  float* red = reinterpret_cast<float*>(smem + S::kStages * S::kStageBytes);      // [NT][128]
  uint8_t* outs = smem + S::kStages * S::kStageBytes + S::kRed;      // on 1024 bytes
  float* scales = reinterpret_cast<float*>(outs + S::kOut);
  int* first = reinterpret_cast<int*>(scales + S::kBufs * S::kScaleRow);
  int* off = first + MM_MAXU + 1;
  __shared__ uint64_t full[S::kStages], empty[S::kStages], acc_full[S::kBufs], acc_empty[S::kBufs], scale_empty[S::kBufs], drained;
  __shared__ uint32_t tmem_base;
  __shared__ int abort_s, unknown_s, wsum[32];
  volatile int* abort_flag = &abort_s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  if (tid == 0) {
    for (int i = 0; i < S::kStages; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], 1);
    for (int i = 0; i < S::kBufs; ++i) mbar_init(&acc_full[i], 2), mbar_init(&acc_empty[i], kPair ? 2 * S::kEpi : S::kEpi), mbar_init(&scale_empty[i], S::kEpi);
    mbar_init(&drained, 1);
    abort_s = 0, unknown_s = 0;
    fence_mbar_init();
    prefetch_tensormap(&map_rows), prefetch_tensormap(&map_weights);
  }
  if (warp == S::kEpi + 1) {
    if constexpr (kPair) tmem_alloc2(&tmem_base, S::kBufs * NT), tmem_relinquish2();
    else tmem_alloc(&tmem_base, S::kBufs * NT), tmem_relinquish();
  }
  grid_dependency_wait();
  grid_launch_dependents();      // (the next kernel's CTAs set themselves up as this one's leave, and wait for all of it)

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
      const int rows = max(off[u + 1] - off[u], 0);
      if (e >= 0 && e < p.E) n += (rows + S::kRows - 1) / S::kRows * ntn;
      else if (rows) unknown_s = 1;
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
  if constexpr (kPair) cluster_sync_all();      // the peer's barriers and accumulators are there
  tc_fence_after();
  const uint32_t tb = tmem_base;

  const int rank = kPair || cluster > 1 ? (int)cluster_ctarank() : 0;
  const int worker = kPair ? blockIdx.x / 2 : blockIdx.x, workers = kPair ? gridDim.x / 2 : gridDim.x;
  const MmRounds<kSwap> rounds(tiles, worker, workers, p.KB, cluster);
  const int crow = kPair ? rank * 128 : 0;      // this CTA's rows of a pair's tile
  bool dead = false;       // a wait ran out: the rest of the tiles is walked without work, so that the barriers of a cluster still meet

  if (warp >= S::kEpi) {
  if constexpr (S::kSplitRegs) regs_dec<504 - 2 * S::kEpiRegs>();
  if (warp == S::kEpi) {                                             // ---- TMA producer
    const uint32_t el = elect_one();
    int st = 0, ph = 1, issued = 0;
    for (int i = 0; rounds.has(i); ++i) {
      int kb0, kb1;
      const int t = rounds.tile(i, kb0, kb1);
      const MmTile tl = mm_tile<NT, kSwap, kPair>(p, first, off, kSwap && t < 0 ? 0 : t);
      if (rounds.shared(i)) cluster_arrive();
      for (int kb = kb0; kb < kb1 && !dead; ++kb) {
        if (!mbar_wait_warp(smem_u32(&empty[st]), ph, abort_flag, looks_of<kRoleProducer>(p, rank))) { dead = true; break; }
        const uint32_t bar = smem_u32(&full[st]), sa = smem_u32(smem + st * S::kStageBytes);
        const int wrow = tl.expert * p.N + tl.n0;
        if constexpr (kPair) {      // each CTA brings its half of both operands; the bytes of both count at the leader's barrier
          const uint32_t lead = mapa_shared(bar, 0);
          mbar_expect_tx_u32(bar, 2 * S::kStageBytes, el & (rank == 0));
          tma_load_2d_pair(sa, &map_rows, kb * 128, tl.row0 + crow, lead, el);
          tma_load_2d_pair(sa + 16384, &map_weights, kb * 128, wrow + rank * S::kBRows, lead, el);
        } else {
          mbar_expect_tx_u32(bar, S::kStageBytes, el);
          tma_load_2d_u32(kSwap ? sa + 16384 : sa, &map_rows, kb * 128, tl.row0, bar, el);
          tma_load_2d_u32(kSwap ? sa : sa + 16384, &map_weights, kb * 128, wrow, bar, el);
        }
        ++issued;
        if (++st == S::kStages) st = 0, ph ^= 1;
      }
      if (rounds.shared(i)) __syncwarp(), cluster_wait(), cluster_sync_all();
    }
    // The tensor core's word that it has read a slot goes to this CTA's barriers (from the leader, in a pair): all of it arrives before the CTA may end, or it
    // would reach the barriers of the CTA that comes after it.
    if (!dead && !mbar_wait_lanes(smem_u32(&empty[lane < S::kStages ? lane : 0]), lane < st ? ph ^ 1 : ph, lane >= S::kStages, abort_flag)) dead = true;
    if (dead) {      // copies in flight land before the CTA may end (with a limit)
      if constexpr (kPair) {      // (their barriers are the first CTA's, which count both CTAs' bytes, and the other may have stopped elsewhere: 200 us)
        for (int n = 0; n < 200; ++n) __nanosleep(1000);
      } else {
        for (int i = issued > S::kStages ? issued - S::kStages : 0; i < issued; ++i)
          for (int n = 0; n < 1 << 16 && !mbar_ready(smem_u32(&full[i % S::kStages]), (i / S::kStages) & 1); ++n) {}
      }
    }
  } else if (warp == S::kEpi + 1) {                                  // ---- MMA issue
    const uint32_t el = elect_one();
    uint32_t idesc = idesc_f8(kPair ? 256 : 128, NT);
    int st = 0, ph = 0, buf = 0, bph = 1;
    for (int i = 0; rounds.has(i); ++i) {
      int kb0, kb1;
      const int t = rounds.tile(i, kb0, kb1);
      if (rounds.shared(i)) cluster_arrive();
      if constexpr (kSwap && NT > 16) {      // columns for the rows that the tile has
        const MmTile tl = mm_tile<NT, kSwap, kPair>(p, first, off, t < 0 ? 0 : t);
        idesc = idesc_f8(128, min(NT, (tl.row_end - tl.row0 + 15) & ~15));
      }
      for (int kb = kb0, ready = 0; kb < kb1 && !dead && (!kPair || rank == 0); ++kb, --ready) {
        if constexpr (S::kAhead < 4) {      // the operands first: they are there long before the accumulator is free
          if (!mbar_wait_warp(smem_u32(&full[st]), ph, abort_flag, looks_of<kRoleMma>(p, rank)) || !mbar_wait_warp(smem_u32(&acc_empty[buf]), bph, abort_flag, looks_of<kRoleMma>(p, rank))) {
            dead = true;
            break;
          }
        } else if (!ready) {      // lane 2j: the operands of the step after the next j, lane 2j + 1: its accumulator
          const int j = lane >> 1 < S::kAhead ? lane >> 1 : 0;
          int q = (lane & 1 ? buf : st) + j;
          const int wrap = lane & 1 ? S::kBufs : S::kStages;
          uint32_t par = lane & 1 ? bph : ph;
          if (q >= wrap) q -= wrap, par ^= 1;
          ready = mbar_wait_steps<2>(smem_u32(lane & 1 ? &acc_empty[q] : &full[q]), par, min(S::kAhead, kb1 - kb), lane, abort_flag, looks_of<kRoleMma>(p, rank));
          if (!ready) { dead = true; break; }
        }
        tc_fence_after();
        const uint32_t a = ((smem_u32(smem + st * S::kStageBytes) >> 4) & 0x3fff) | kDescLoSw128, b = a + (16384 >> 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (kPair) umma2_f8(tb + buf * NT, a + 2 * j, b + 2 * j, idesc, j != 0, el);
          else umma_f8(tb + buf * NT, a + 2 * j, b + 2 * j, idesc, j != 0, el);
        }
        if constexpr (kPair) {
          umma2_commit_p(&empty[st], 3, el);
          umma2_commit_p(&acc_full[buf], 3, el);
        } else {
          umma_commit_u32(smem_u32(&empty[st]), el);
          umma_commit_u32(smem_u32(&acc_full[buf]), el);
        }
        if (++st == S::kStages) st = 0, ph ^= 1;
        if (++buf == S::kBufs) buf = 0, bph ^= 1;
      }
      if (rounds.shared(i)) __syncwarp(), cluster_wait(), cluster_sync_all();
    }
    // Everything issued is done before the CTA may end, whoever else has given up (with a limit).
    if constexpr (kPair) umma2_commit_p(&drained, 1, el & (rank == 0));
    else umma_commit_u32(smem_u32(&drained), el);
    for (int n = 0; n < 1 << 16 && (!kPair || rank == 0) && !mbar_ready(smem_u32(&drained), 0); ++n) {}
  } else if (warp == S::kEpi + 2) {                                  // ---- scales: four groups ahead in registers, then a slot beside each accumulator
    constexpr int kHere = kSwap ? NT : 128, R = (kHere + 31) / 32;
    int buf = 0, bph = 1;
    for (int i = 0; rounds.has(i); ++i) {
      int kb0, kb1;
      const int t = rounds.tile(i, kb0, kb1);
      const MmTile tl = mm_tile<NT, kSwap, kPair>(p, first, off, kSwap && t < 0 ? 0 : t);
      const float* ra[R];
#pragma unroll
      for (int i = 0; i < R; ++i) ra[i] = p.sa + (long long)min(tl.row0 + crow + lane + 32 * i, p.M - 1) * p.KB;
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
      if (rounds.shared(i)) cluster_arrive();
      if (!dead && kb0 < kb1) fetch(kb0);
      for (int kb = kb0; kb < kb1 && !dead; kb += 4) {
        float ca[4][R], cb[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          cb[j] = vb[j];
#pragma unroll
          for (int i = 0; i < R; ++i) ca[j][i] = va[j][i];
        }
        if (kb + 4 < kb1) fetch(kb + 4);
        int ready = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (kb + j >= kb1) break;
          if (!ready) {
            int q = buf + (lane < S::kAhead ? lane : 0);
            uint32_t par = bph;
            if (q >= S::kBufs) q -= S::kBufs, par ^= 1;
            ready = mbar_wait_steps<1>(smem_u32(&scale_empty[q]), par, min(min(S::kAhead, 4 - j), kb1 - kb - j), lane, abort_flag, looks_of<kRoleScales>(p, rank));
            if (!ready) { dead = true; break; }
          }
          --ready;
          float* s = scales + buf * S::kScaleRow;
#pragma unroll
          for (int i = 0; i < R; ++i)
            if (lane + 32 * i < kHere) s[lane + 32 * i] = kSwap ? ca[j][i] * cb[j] : ca[j][i];
          if (!kSwap && lane < 2) s[128 + lane] = cb[j];
          __syncwarp();
          if (lane == 0) mbar_arrive(&acc_full[buf]);
          if (++buf == S::kBufs) buf = 0, bph ^= 1;
        }
      }
      if (rounds.shared(i)) __syncwarp(), cluster_wait(), cluster_sync_all();
    }
  }
  } else {                                                           // ---- epilogue
    if constexpr (S::kSplitRegs) regs_inc<S::kEpiRegs>();
    const int quad = warp & 3, half = warp >> 2, col0 = half * S::kCols;
    const int l = quad * 32 + lane;                                  // accumulator lane
    constexpr int kLogNT = NT == 16 ? 4 : NT == 32 ? 5 : NT == 64 ? 6 : NT == 128 ? 7 : 8;
    bool red_in_use = false;
    const uint32_t lead_empty = mapa_shared(smem_u32(&acc_empty[0]), 0);
    int buf = 0, ph = 0;
    for (int i = 0; rounds.has(i); ++i) {
      int kb0, kb1;
      const int t = rounds.tile(i, kb0, kb1);
      const MmTile tl = mm_tile<NT, kSwap, kPair>(p, first, off, kSwap && t < 0 ? 0 : t);
      if (rounds.shared(i)) __syncwarp(), cluster_arrive();      // this CTA is there, and its last tile's sums are read
      float acc[S::kCols];
#pragma unroll
      for (int j = 0; j < S::kCols; ++j) acc[j] = 0.f;
      const int rows = kSwap ? min(NT, tl.row_end - tl.row0) : NT;      // columns in use
      for (int kb = kb0, ready = 0; kb < kb1 && !dead; ++kb, --ready) {
        if constexpr (S::kAhead < 4) {
          if (!mbar_ready(smem_u32(&acc_full[buf]), ph) && !mbar_wait_warp(smem_u32(&acc_full[buf]), ph, abort_flag, looks_of<kRoleEpilogue>(p, rank))) { dead = true; break; }
        } else if (!ready) {
          int q = buf + (lane < S::kAhead ? lane : 0);
          uint32_t par = ph;
          if (q >= S::kBufs) q -= S::kBufs, par ^= 1;
          ready = mbar_wait_steps<1>(smem_u32(&acc_full[q]), par, min(S::kAhead, kb1 - kb), lane, abort_flag, looks_of<kRoleEpilogue>(p, rank));
          if (!ready) { dead = true; break; }
        }
        tc_fence_after();
        const float* s = scales + buf * S::kScaleRow;
        const uint32_t taddr = tb + buf * NT + ((uint32_t)(quad * 32) << 16);
        uint32_t v[2][S::kChunk];
        tmem_ld_cols<S::kChunk>(taddr + mm_column<NT, kSwap, kPair>(half, 0), v[0]);
        const float sr = kSwap ? 0.f : s[l] * s[128 + half];
#pragma unroll
        for (int c = 0; c < S::kCols / S::kChunk; ++c) {
          const int col = mm_column<NT, kSwap, kPair>(half, c);
          tmem_ld_wait();
          if (c + 1 < S::kCols / S::kChunk) {
            if (!kSwap || mm_column<NT, kSwap, kPair>(half, c + 1) < rows) tmem_ld_cols<S::kChunk>(taddr + mm_column<NT, kSwap, kPair>(half, c + 1), v[(c + 1) & 1]);
          } else {      // all of it is in registers: the tensor core may have the accumulator back
            tc_fence_before();
            __syncwarp();
            if constexpr (kPair) mbar_arrive_cluster_p(lead_empty + buf * 8, lane == 0);
            else mbar_arrive_p(smem_u32(&acc_empty[buf]), lane == 0);
            if (!kSwap) mbar_arrive_p(smem_u32(&scale_empty[buf]), lane == 0);
          }
          if (kSwap && col >= rows) continue;
#pragma unroll
          for (int i = 0; i < S::kChunk; i += 4) {
            float* o = acc + c * S::kChunk + i;
            const uint32_t* x = v[c & 1] + i;
            float4 sc = make_float4(sr, sr, sr, sr);
            if constexpr (kSwap) sc = *reinterpret_cast<const float4*>(s + col + i);
            fma2(o[0], o[1], x[0], x[1], sc.x, sc.y);
            fma2(o[2], o[3], x[2], x[3], sc.z, sc.w);
          }
        }
        if constexpr (kSwap) {      // (the slot's scales are read up to here)
          __syncwarp();
          mbar_arrive_p(smem_u32(&scale_empty[buf]), lane == 0);
        }
        if (++buf == S::kBufs) buf = 0, ph ^= 1;
      }
      if constexpr (!kSwap) {
        if (!dead) {
          const int row0 = tl.row0 + crow + quad * 32, n = tl.n0 + col0;
          uint8_t* buf = outs + warp * S::kOutWarp;
          if (row0 < tl.row_end) {
            if (p.out_dtype == DT_BF16) put_rows<DT_BF16>(p, &map_out, buf, acc, row0, tl.row_end, n, lane);
            else if (p.out_dtype == DT_F16) put_rows<DT_F16>(p, &map_out, buf, acc, row0, tl.row_end, n, lane);
            else put_rows<DT_F32>(p, &map_out, buf, acc, row0, tl.row_end, n, lane);
          }
        }
      } else {
        if (!rounds.shared(i)) {
          // to shared memory [row][128 weights] and out of it again row by row (as they stand, a store instruction writes 64 bytes of one row: 8000 cycles a tile of 64)
          if (red_in_use) named_bar_sync(1, S::kEpi * 32);      // the last tile's sums are read
#pragma unroll
          for (int c = 0; c < S::kCols / S::kChunk; ++c) {
            const int col = mm_column<NT, kSwap, kPair>(half, c);
            if (col >= rows) continue;
#pragma unroll
            for (int j = 0; j < S::kChunk; ++j) red[(col + j) * 128 + l] = acc[c * S::kChunk + j];
          }
          named_bar_sync(1, S::kEpi * 32);
          red_in_use = true;
          if (!dead && t >= 0)
            for (int j = tid; j < rows * 32; j += S::kEpi * 32) {
              const int n = tl.n0 + (j & 31) * 4;
              const float4 v = *reinterpret_cast<const float4*>(red + j * 4);
              if (n < p.N) put_four(p, tl.row0 + (j >> 5), n, {v.x, v.y, v.z, v.w});
            }
        } else {
          // each column's sums to the CTA that adds them: stores one way instead of loads there and back, and one barrier that is waited for
          __syncwarp();
          cluster_wait();
          if (t >= 0) {
            const int log_parts = rounds.log_parts, log_own = kLogNT - log_parts, here = rank & ((1 << log_parts) - 1), base = rank - here;
            const uint32_t mine = smem_u32(red) + (here << log_own) * 512 + l * 4;
            constexpr int kOwn = NT / 8;      // columns in a row that always have one owner
#pragma unroll
            for (int c = 0; c < S::kCols / S::kChunk; ++c) {
              const int col = mm_column<NT, kSwap, kPair>(half, c);
              if (col >= rows) continue;
#pragma unroll
              for (int g = 0; g < S::kChunk; g += kOwn) {
                const uint32_t to = mapa_shared(mine + ((col + g) & ((1 << log_own) - 1)) * 512, base + ((col + g) >> log_own));
#pragma unroll
                for (int j = 0; j < kOwn; ++j) st_cluster_f32(to + j * 512, acc[c * S::kChunk + g + j]);
              }
            }
          }
          __syncwarp();
          cluster_sync_all();
          if (!dead && t >= 0) {
            if (rounds.log_parts == 1) mm_add_ranks<NT, 2>(p, tl, red, rank, tid);
            else if (rounds.log_parts == 2) mm_add_ranks<NT, 4>(p, tl, red, rank, tid);
            else mm_add_ranks<NT, 8>(p, tl, red, rank, tid);
          }
        }
      }
    }
    if constexpr (!kSwap) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");      // shared memory stays until the copies have read it
    if (p.offsets && p.zero_rest) {      // rows outside every run, and of experts that are not there
      const int warps = gridDim.x * S::kEpi, me = blockIdx.x * S::kEpi + warp;
      if (unknown_s)
        for (int u = 0; u < p.U; ++u) {
          const int e = p.experts[u];
          if (e < 0 || e >= p.E) zero_rows(p, off[u], off[u + 1], me, warps, lane);
        }
      if (off[0] > 0) zero_rows(p, 0, off[0], me, warps, lane);
      zero_rows(p, off[p.U], p.M, me, warps, lane);
    }
  }
  if (dead) {
    atomicExch(&g_matmul_fp8_status, 1);
    if constexpr (kPair) st_cluster_u32(mapa_shared(smem_u32(&abort_s), rank ^ 1), 1u);      // the other CTA, which waits for this one, stops as well
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (kPair) {
    cluster_sync_all();      // nobody frees or leaves while the pair's work may still reach it
    if (warp == S::kEpi + 1) tmem_dealloc2(tb, S::kBufs * NT);
  } else {
    if (warp == S::kEpi + 1) tmem_dealloc(tb, S::kBufs * NT);
  }
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
// Matrix of `rows` rows of K bytes, `stride` bytes apart: boxes of 128 bytes x box_rows, 128-byte swizzle, zeros (or nothing stored) beyond the matrix
static int bytes_map(CUtensorMap* map, const void* base, long long rows, long long K, long long stride, int box_rows) {
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

template <int NT, bool kSwap, bool kPair>
static int launch_matmul(const MatmulParams& p, const void* a, long long lda, const void* w, long long ldw, long long tiles, int cluster, int sms, cudaStream_t st) {
  using S = MmShape<NT, kSwap, kPair>;
  CUtensorMap rows, weights, out = {};
  if (int rc = bytes_map(&rows, a, p.M, p.K, lda, kSwap ? NT : 128)) return rc;
  if (int rc = bytes_map(&weights, w, (long long)p.E * p.N, p.K, ldw, kSwap ? 128 : S::kBRows)) return rc;
  const int size = p.out_dtype == DT_F32 ? 4 : 2;
  if (!kSwap && p.vec)
    if (int rc = bytes_map(&out, p.out, p.M, (long long)p.N * size, p.ldo * size, 32)) return rc;
  const void* fn = (const void*)k_matmul_fp8<NT, kSwap, kPair>;
  static std::atomic<unsigned long long> opted_in{0};      // devices on which this form may have its shared memory
  int dev = 0;
  B200_CUDA_TRY(cudaGetDevice(&dev));
  if (dev > 63 || !(opted_in.load(std::memory_order_relaxed) >> dev & 1)) {
    B200_CUDA_TRY(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem));
    if (dev <= 63) opted_in.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  const int ranks = kPair ? 2 : cluster;
  const long long most = sms / ranks;
  const int clusters = (int)(tiles < most ? (tiles > 0 ? tiles : 1) : most);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(clusters * ranks), cfg.blockDim = dim3(S::kThreads), cfg.dynamicSmemBytes = S::kSmem, cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization, attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ranks, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr, cfg.numAttrs = ranks > 1 ? 2 : 1;
  MatmulParams q = p;
  void* args[] = {&rows, &weights, &out, &q, &cluster};
  B200_CUDA_TRY(cudaLaunchKernelExC(&cfg, fn, args));
  return B200MOE_OK;
}

// The forms with weights on the lanes: rows of a tile, and microseconds of a call and of a group, as fitted to measured calls (20 sizes from 1 x 2048 x 2048 to
// 4096 x 2816 x 704 in every form and cluster, weights in L2).
struct MmForm { int rows; float call, group; };
constexpr MmForm kMmForms[] = {{16, 4.9f, 0.17f}, {32, 5.4f, 0.22f}, {64, 6.4f, 0.30f}, {128, 10.0f, 0.35f}};
constexpr float kMmPairCall = 5.6f, kMmPairGroup = 0.48f, kMmPairRound = 0.7f;

// The largest cluster that gives its CTAs a part each: of eight CTAs only as many clusters as three quarters of the SMs hold (16 of them took two rounds: 8.2 us instead
// of 5.1 at 1 x 2048 x 2048), two where tiles are more than the SMs, for those of the last round.
static int matmul_cluster(long long tiles, int KB, int sms) {
  int cluster = 2;
  while (cluster < 8 && tiles * cluster * 2 <= (cluster == 4 ? sms * 3 / 4 : sms) && KB >= cluster * 4) cluster *= 2;
  return cluster;
}

// One matrix: the form of the least time by that model; many rows take CTA pairs (512 x 4096 x 4096: pairs 19.7 us, single CTAs of 128 x 256 21.1, weights on the
// lanes 23.0; 200 rows: 18.8, 20.0, 14.6).
// A matrix per expert: by the mean rows of a run, whose lengths the host does not know. A few rows take tiles of 16; from 8 on (3 where the inner size has four
// groups or less, and a tile's ends count for more) 128 x 256, which lose some to them while runs are alike and gain more where a few are long (us, tiles of 16 / 128 x 256, 8 rows:
// 1536 x 2048 alike 72.8 / 81.1, skewed 44.8 / 43.7; 2816 x 704 52.3 / 55.5, 41.7 / 32.9; 1536 x 512 48.0 / 45.3, 36.7 / 25.4; 3 rows of it 45.3 / 40.8, 24.0 / 22.1);
// pairs where the rows that tiles of 256 leave empty no longer matter (375 rows: pairs 229 us, single CTAs 217; 1000: 121, 125).
static int matmul(const MatmulParams& p, const void* a, long long lda, const void* w, long long ldw, cudaStream_t st) {
  const int sms = sm_count();
  if (sms <= 0) return B200MOE_ERR_DEVICE;
  int rows, cluster;
  long long n;
  if (p.offsets) {
    const long long runs = p.U < p.M ? p.U : p.M, mean = p.M / runs;
    const auto tiles = [&](int r, int c) { return (p.M / r + runs) * ((p.N + c - 1) / c); };      // (at most)
    if (mean > 512) return launch_matmul<256, false, true>(p, a, lda, w, ldw, tiles(256, 256), 1, sms, st);
    if (mean > (p.KB <= 4 ? 2 : 7)) return launch_matmul<256, false, false>(p, a, lda, w, ldw, tiles(128, 256), 1, sms, st);
    rows = 16, n = tiles(rows, 128), cluster = matmul_cluster(n, p.KB, sms);
  } else {
    const auto tiles = [&](int r, int c) { return (long long)((p.M + r - 1) / r) * ((p.N + c - 1) / c); };
    const long long pairs = tiles(256, 256), rounds = (pairs + sms / 2 - 1) / (sms / 2);
    float best = kMmPairCall + (float)rounds * (float)p.KB * kMmPairGroup + (float)(rounds - 1) * kMmPairRound;
    rows = 0;
    for (const MmForm& f : kMmForms) {
      const long long t = tiles(f.rows, 128);
      const int c = matmul_cluster(t, p.KB, sms), workers = sms / c * c;
      const long long full = t / workers, rest = t - full * workers;
      int parts = c;
      while (parts > 1 && (rest * parts > workers || p.KB < 2 * parts)) parts /= 2;
      const float time = f.call + ((float)full * (float)p.KB + (float)(rest ? (p.KB + parts - 1) / parts : 0)) * f.group + (float)(full + (rest > 0) - 1) * (f.call - 4.5f);
      if (time < best) best = time, rows = f.rows, n = t, cluster = c;
    }
    if (!rows) return launch_matmul<256, false, true>(p, a, lda, w, ldw, pairs, 1, sms, st);
  }
  switch (rows) {
    case 16: return launch_matmul<16, true, false>(p, a, lda, w, ldw, n, cluster, sms, st);
    case 32: return launch_matmul<32, true, false>(p, a, lda, w, ldw, n, cluster, sms, st);
    case 64: return launch_matmul<64, true, false>(p, a, lda, w, ldw, n, cluster, sms, st);
    default: return launch_matmul<128, true, false>(p, a, lda, w, ldw, n, cluster, sms, st);
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
static int stores_16(const void* out, int out_dtype, int N, long long ldo) {
  const int size = out_dtype == DT_F32 ? 4 : 2;
  return ((uintptr_t)out & 15) == 0 && (ldo * size) % 16 == 0 && ((long long)N + 256) * size < (1ll << 31);
}

}  // namespace b200

extern "C" {

int b200moe_matmul_fp8(const void* a, long long a_stride, const float* a_scales, const void* w, long long w_stride, const float* w_scales, int M, int N, int K,
                       void* out, int out_dtype, long long out_stride, void* stream) {
  using namespace b200;
  if (int rc = matmul_args(a, a_stride, a_scales, w, w_stride, w_scales, M, N, K, out, out_dtype, out_stride)) return rc;
  if (M == 0 || N == 0) return B200MOE_OK;
  const MatmulParams p = {a_scales, w_scales, out, nullptr, nullptr, 0, 1, M, N, K, (K + 127) / 128, (N + 127) / 128, out_dtype, 0, stores_16(out, out_dtype, N, out_stride), out_stride, 0};
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
  if (!experts || !offsets || (((uintptr_t)experts | (uintptr_t)offsets) & 3)) return B200MOE_ERR_ARG;
  const MatmulParams p = {a_scales, w_scales, out, experts, offsets, runs, E, rows, N, K, (K + 127) / 128, (N + 127) / 128, out_dtype, zero_rest,
                          stores_16(out, out_dtype, N, out_stride), out_stride, 0};
  return matmul(p, a, a_stride, w, w_stride, (cudaStream_t)stream);
}

int b200moe_matmul_fp8_probe(const void* a, long long a_stride, const float* a_scales, int rows, const void* w, long long w_stride, const float* w_scales, int E,
                             const int* experts, const int* offsets, int runs, int N, int K, void* out, int out_dtype, long long out_stride, int give_up, void* stream) {
  using namespace b200;
  if (E < 1 || runs < 0 || give_up < 0 || give_up > 31 || !experts != !offsets || (!experts && E != 1) || (((uintptr_t)experts | (uintptr_t)offsets) & 3)) return B200MOE_ERR_ARG;
  if (int rc = matmul_args(a, a_stride, a_scales, w, w_stride, w_scales, rows, N, K, out, out_dtype, out_stride)) return rc;
  if (runs > MM_MAXU || (long long)E * N > (1ll << 31) - 512) return B200MOE_ERR_LIMIT;
  if (rows == 0 || N == 0 || (experts && runs == 0)) return B200MOE_OK;
  const MatmulParams p = {a_scales, w_scales, out, experts, offsets, runs, E, rows, N, K, (K + 127) / 128, (N + 127) / 128, out_dtype, 0, stores_16(out, out_dtype, N, out_stride),
                          out_stride, give_up};
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
