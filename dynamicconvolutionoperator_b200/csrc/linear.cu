// Matrix product with bias, activation and residual in its epilogue, forward
// and backward, over row-major x [m][k] and weight [n][k] (an nn.Linear weight
// or a 1x1 convolution's).
//
//   z = x weight^T + bias,  out = act(z) + residual
// backward, with dz = dy * act'(z):
//   dx = dz weight,  dweight = dz^T x,  dbias = sum_rows dz,  dresidual = dy
//
// All three products run on one persistent tensor-core kernel,
//   D[M][N] = sum_k A(m, k) B(n, k),
// whose operands are K-major (rows of k: the forward) or MN-major (columns of
// k: weight in dx, both operands in dweight); the layout is a matter of TMA
// boxes and descriptors, so nothing is transposed in memory.
//
//   tile      128 rows x BN (64, 128 or 256) columns, K in steps of 64 (FP32:
//             32); where there is work for all, a pair of blocks shares 256 rows
//   operands  TMA, 128-byte swizzle, a ring of stages; out-of-range rows,
//             columns and k are zero filled, which covers every ragged size
//   issue     tcgen05.mma of 128 x BN x 16 by one thread; two TMEM
//             accumulators, so the epilogue of a tile overlaps the next one
//   epilogue  one or two groups of 8 warps (lane = row, two column halves; two
//             groups take the tiles in turn): TMEM -> registers,
//             bias, activation, residual -> 128-byte x 32-row boxes in shared
//             memory -> TMA store. The residual (or dy) comes through the same
//             boxes by TMA, several boxes ahead.
//
// The backward keeps x and weight only: z is computed again by the same
// product (kDz), whose epilogue turns it into dz at once. Saving z instead
// would cost m * n values of traffic twice and, rounded to 16 bits, a second
// rounding in dz. dz is rounded to the data's type, as an operand of the
// tensor cores has to be; the bias gradient sums it before that rounding.
//
// FP32 data: the tensor cores multiply bf16, so every value is split into three
// bf16 parts that hold its 24 bits, x = x0 + x1 + x2, and a K step issues the six
// products whose size is above 2^-24 of x0 y0 (exponents stay in range: bf16 has
// FP32's). Eight more warps split the operands on their way: FP32 tiles come by
// TMA, their parts go to a second ring as core matrices (16 bytes = 8 values
// along the contiguous axis). A split in a pass of its own moved 2.5 times the
// bytes (65536 x 256 -> 64, training: 199 us). Each K block has an accumulator
// of its own, and the epilogue's registers add the blocks: a chain of 384
// tensor-core additions (k = 1024) left a 2-norm error of 4.9e-6.
//
// dweight sums over all rows: its K axis is split over the SMs left without a
// tile, FP32 partials are added in a fixed order.
//
// 16-bit data, long sums: an addition in the tensor cores cuts off what lies below
// the sum's last bit, so that a chain of them is biased towards zero by up to 2^-23
// of the sum an addition (16 values of k). Same-sign fp16 data measured -3.9e-4 of
// the sum at 65536 values and -6.2e-3 at 2^20, more than half a step of bf16. An
// accumulator takes kChain values of k at most (-1.0e-4); longer sums are split, and
// their FP32 partials added (and the epilogue applied) by a kernel of its own
// (dweight of 65536 rows, 4096 x 1024 bf16: 387 -> 437 us; of 262144: 1611, 1605).
//
// Measured (bf16): 16384 x 1024 -> 4096 107 us (1280 TFLOP/s, 0.76 of the
// measured peak; without its copies 98 us), with gelu 118 us; 8192^3 760 us (1450
// TFLOP/s); 65536 x 64 -> 1728 72 us (3.3 TB/s, bound by the epilogue's chain: its
// warps' TMEM loads, stores to the boxes, fences). FP32: 8192 x 2048 -> 2048 540 us
// (127 TFLOP/s of FP32 products; bound by shared memory, through which a K block
// moves 208 KB, and by the splitting), 65536 x 256 -> 64 41 us.
//
// Up to eight rows, forward: a dot-product kernel reads the weight once at the
// memory's rate; a tensor-core tile would be 15/16 empty and its K loop serial (1024 -> 4096
// bf16: 3.2 us, 2.6 TB/s). Both at 4, 6 and 8 rows: 1024 -> 4096 bf16 6.0, 8.4, 9.8 and
// (tile) 10.3 us, 4096 -> 4096 18, 26, 32 and 25; FP32 14, 23, 26 and 126.
#include <atomic>
#include <type_traits>

#include "act.cuh"
#include "common.cuh"
#include "tc.cuh"
#include "tmap.cuh"

namespace ddpm {

namespace gencat {
int status_ptr(int** out);
int num_sms();
int max_smem_optin();
}  // namespace gencat

namespace {

constexpr int kBM = 128;
__host__ __device__ constexpr int block_k(int parts) { return parts == 3 ? 32 : 64; }
constexpr int kFirstEpi = 4;  // warps 0-3: TMA, MMA, TMEM allocation, none
constexpr int kSplitWarps = 8;  // FP32 data: warps that split operands, behind the epilogue's
__host__ __device__ constexpr int gemm_threads(int parts, int ew) {
  return 32 * (kFirstEpi + ew + (parts == 3 ? kSplitWarps : 0));
}
constexpr int kMaxStages = 8, kMaxBufs = 8;
constexpr uint64_t kWaitNs = 2000000000ull;
constexpr int kGemvRows = 8;
constexpr int kShortK = 4;  // K blocks
constexpr int kChain = 16384;  // values of k an accumulator sums (16-bit data)

enum Epi { kOut, kDz, kPartial };

struct GemmParams {
  CUtensorMap a, b, out, in;
  const void* bias;    // nullable
  const void* in_ptr;  // residual (kOut, nullable) or dy (kDz)
  void* out_ptr;
  float* colsum;       // kDz: [ceil(M / 32)][N] column sums of dz; nullable
  long long ld_in, ld_out;
  int M, N;
  int tiles_m, tiles_n, splits, num_tiles, kblocks;
  int a_mn, b_mn, tma_io, act, stages, nbuf, last_ksteps;
  uint32_t idesc;
  int* status;
};

// A box of the epilogue: 32 rows x 128 bytes (64 where half a tile is no wider).
__host__ __device__ constexpr int box_row(int bn, int es) { return bn / 2 * es < 128 ? 64 : 128; }

struct SmemLayout {
  uint32_t stage, planes, boxes, bias, total;
};
__host__ __device__ inline SmemLayout smem_layout(int cg, int parts, int bn, int ew, int row,
                                                  int stages, int nbuf) {
  SmemLayout L;
  // a stage: 64 k of 16-bit values or 32 of FP32; FP32: two sets of parts
  L.stage = (uint32_t)(kBM + bn / cg) * 128;
  L.planes = L.stage * stages;
  L.boxes = L.planes + (parts == 3 ? 2 * 3 * (kBM + bn) * 64 : 0);
  L.bias = L.boxes + ew * nbuf * 32 * row;
  L.total = L.bias + (parts == 3 ? 0 : ew * (bn / 2) * 4) + 1024;  // + alignment
  return L;
}

__device__ __forceinline__ void give_up(volatile int* abort_flag, int* status, int code) {
  *abort_flag = 1;
  atomicCAS(status, 0, code);
}

// Warp-uniform bounded wait. The copying and the issuing warp run their loops
// with all lanes and elect one only for the instruction itself: a loop that one
// lane runs keeps its descriptors in vector registers, and a product then costs
// its thread 250 clocks to issue (1.05 against 1.34 PFLOP/s at 8192^3).
template <bool kCluster = false>
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  auto try_wait = [&]() {
    if constexpr (!kCluster) {
      return tc::mbar_try_wait(bar, parity);
    } else {  // arrivals of both blocks of a pair
      uint32_t ok;
      asm volatile(
          "{\n\t.reg .pred p;\n\t"
          "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
          "selp.u32 %0, 1, 0, p;\n\t}"
          : "=r"(ok)
          : "r"(tc::smem_u32(bar)), "r"(parity)
          : "memory");
      return ok != 0;
    }
  };
  // the clock is read only once a wait has become a long one
  bool ok = false;
  for (int i = 0; i < 64 && !ok; ++i) ok = try_wait();
  if (!ok) {
    const uint64_t began = tc::globaltimer_ns();
    while (!(ok = try_wait())) {
      if ((abort_flag != nullptr && *abort_flag) || tc::globaltimer_ns() - began > kWaitNs) break;
    }
  }
  return __all_sync(0xffffffffu, ok);
}

// ------------------------------------------------------- pairs of blocks ----
// CG = 2: two blocks of a cluster work on one tile of 256 rows. Each holds its
// 128 rows of A and half the columns of B; the even block's thread issues the
// products for both (cta_group::2), which halves what a block moves through
// shared memory for the same work.
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" :::
               "memory");
}
// The even block's copy of one of this block's shared addresses.
__device__ __forceinline__ uint32_t leader_addr(const void* p) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(tc::smem_u32(p)));
  return a;
}
template <int CG>
__device__ __forceinline__ void load_box(void* dst, const void* map, int c0, int c1, uint64_t* bar,
                                         uint32_t leader_bar) {
  if constexpr (CG == 1) {
    tc::tma_load_3d(dst, map, c0, c1, 0, bar);
  } else {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile"
        ".mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(tc::smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(0), "r"(leader_bar)
        : "memory");
  }
}
template <int CG>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                    uint32_t more) {
  if constexpr (CG == 1) {
    tc::mma_f16(d, a, b, idesc, more);
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(more)
        : "memory");
  }
}
// Arrive, once the products issued so far are complete, on `bar` (of both blocks).
template <int CG> __device__ __forceinline__ void commit(uint64_t* bar) {
  if constexpr (CG == 1) {
    tc::mma_commit(bar);
  } else {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
        " [%0], %1;" ::"r"(tc::smem_u32(bar)),
        "h"((uint16_t)3)
        : "memory");
  }
}
template <int CG> __device__ __forceinline__ void arrive_leader(uint64_t* bar) {
  if constexpr (CG == 1) {
    tc::mbar_arrive(bar);
  } else {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(
                     leader_addr(bar))
                 : "memory");
  }
}
template <int CG> __device__ __forceinline__ void tmem_alloc(uint32_t* dst, uint32_t cols) {
  if constexpr (CG == 1) {
    tc::tmem_alloc(dst, cols);
    tc::tmem_relinquish();
  } else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     tc::smem_u32(dst)),
                 "r"(cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
}
template <int CG> __device__ __forceinline__ void tmem_dealloc(uint32_t at, uint32_t cols) {
  if constexpr (CG == 1)
    tc::tmem_dealloc(at, cols);
  else
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(cols)
                 : "memory");
}

// Sums over the warp's rows of 32 columns: lane l returns the sum of v[l] over
// the 32 lanes. Halves the columns a lane holds at each exchange.
__device__ __forceinline__ float column_sums(float (&v)[32], int lane) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
#pragma unroll
    for (int i = 0; i < off; ++i) {
      const bool up = lane & off;
      const float send = up ? v[i] : v[i + off];
      const float keep = up ? v[i + off] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, send, off);
    }
  }
  return v[0];
}

// Tile -> (row tile, column tile, split): column tiles of eight row tiles in
// turn, so that blocks running together share operands in L2.
__device__ __forceinline__ void tile_at(const GemmParams& p, int t, int& tm, int& tn, int& sp) {
  const int per = p.tiles_m * p.tiles_n;
  sp = t / per;
  t -= sp * per;
  const int g = t / (8 * p.tiles_n);
  const int rows = min(8, p.tiles_m - 8 * g);
  t -= g * 8 * p.tiles_n;
  tn = t / rows;
  tm = 8 * g + t - tn * rows;
}

// T: the type of out, in and bias (kPartial: out is FP32). PARTS: 1, or 3 for
// FP32 data, split into bf16 parts. CG: blocks that share a tile.
template <typename T, int BN, int PARTS, Epi kEpi, int CG, int EW>
__global__ void __launch_bounds__(gemm_threads(PARTS, EW), 1)
linear_gemm_kernel(const __grid_constant__ GemmParams p) {
  using To = typename std::conditional<kEpi == kPartial, float, T>::type;
  constexpr bool kFast = sizeof(T) == 2;
  constexpr int kGroups = EW / 8;                  // groups of 8 warps take the tiles in turn
  constexpr int kCols = BN / 2;                    // columns of a warp's part of a tile
  constexpr int kRow = box_row(BN, sizeof(To));    // bytes of a box row
  constexpr int kFirstSplit = kFirstEpi + EW;
  constexpr int kBox = 32 * kRow;
  constexpr int kCB = kRow / (int)sizeof(To);      // columns of a box
  constexpr int kBoxes = kCols / kCB;
  constexpr int kSub = kCB / 32;                   // steps of 32 columns
  constexpr int kBK = block_k(PARTS);
  constexpr int kRows64 = PARTS == 3 ? 32 : 64;    // MN-major: contiguous values of a box
  constexpr int kBNb = BN / CG;                    // columns of B this block holds
  constexpr int kPer = 16 / (int)sizeof(To);       // values of a 16-byte chunk
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full[kMaxStages], empty[kMaxStages], acc_full[2], acc_empty[2];
  __shared__ uint64_t parts_full[2], parts_empty[2];
  __shared__ uint64_t in_full[EW][kMaxBufs], drained;
  __shared__ uint32_t tmem_base_s;
  __shared__ int abort_s;
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const SmemLayout L = smem_layout(CG, PARTS, BN, EW, kRow, p.stages, p.nbuf);
  // a shuffle, so that the compiler knows the warp's number to be uniform
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? cluster_rank() : 0;
  const int first_tile = blockIdx.x / CG, tile_step = gridDim.x / CG;
  volatile int* abort_flag = &abort_s;

  if (threadIdx.x == 0) {
    for (int i = 0; i < p.stages; ++i) {
      tc::mbar_init(&full[i], 1);
      tc::mbar_init(&empty[i], PARTS == 3 ? 4 : 1);
    }
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&acc_full[i], 1);
      tc::mbar_init(&acc_empty[i], CG * 8);
      tc::mbar_init(&parts_full[i], 4);
      tc::mbar_init(&parts_empty[i], 1);
    }
    for (int w = 0; w < EW; ++w)
      for (int i = 0; i < p.nbuf; ++i) tc::mbar_init(&in_full[w][i], 1);
    tc::mbar_init(&drained, 1);
    abort_s = 0;
    tc::fence_mbar_init();
  }
  if (warp == 2) tmem_alloc<CG>(&tmem_base_s, 2 * BN);
  tc::tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();
  tc::tc_fence_after();
  const uint32_t tmem = tmem_base_s;

  auto total_blocks = [&]() {  // K blocks of all of this block's tiles
    uint32_t n = 0;
    for (int t = first_tile; t < p.num_tiles; t += tile_step) {
      const int sp = t / (p.tiles_m * p.tiles_n);
      n += (uint32_t)((long long)p.kblocks * (sp + 1) / p.splits) -
           (uint32_t)((long long)p.kblocks * sp / p.splits);
    }
    return n;
  };
  // bytes of A in a stage; of one part of A and of B
  constexpr uint32_t kStageA = kBM * 128, kPartA = kBM * kBK * 2, kPartB = kBNb * kBK * 2;
  if (warp == 0) {
    {  // ---- operand copies ----
      const bool lead = tc::elect_one();
      uint32_t it = 0;
      bool ok = true;
      for (int t = first_tile; t < p.num_tiles && ok; t += tile_step) {
        int tm, tn, sp;
        tile_at(p, t, tm, tn, sp);
        const int ra = (tm * CG + rank) * kBM, rb = tn * BN + rank * kBNb;
        const int kb0 = (int)((long long)p.kblocks * sp / p.splits);
        const int kb1 = (int)((long long)p.kblocks * (sp + 1) / p.splits);
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          const int s = it % p.stages;
          if (!warp_wait(&empty[s], ((it / p.stages) & 1) ^ 1, abort_flag)) {
            if (lead) give_up(abort_flag, p.status, 91);
            ok = false;
            break;
          }
          uint8_t* a = smem + s * L.stage;
          uint8_t* b = a + kStageA;
          uint32_t bar = 0;
          if constexpr (CG == 2) bar = leader_addr(&full[s]);
          if (lead) {
            // the even block's barrier counts both blocks' bytes
            if (rank == 0) tc::mbar_arrive_expect_tx(&full[s], CG * L.stage);
            // K-major: one box of [rows][128 bytes of k]; MN-major: a box of
            // [k][128 bytes of rows] for every 64 (FP32: 32) rows
            if (!p.a_mn) {
              load_box<CG>(a, &p.a, kb * kBK, ra, &full[s], bar);
            } else {
#pragma unroll
              for (int j = 0; j < kBM / kRows64; ++j)
                load_box<CG>(a + j * kBK * 128, &p.a, ra + j * kRows64, kb * kBK, &full[s], bar);
            }
            if (!p.b_mn) {
              load_box<CG>(b, &p.b, kb * kBK, rb, &full[s], bar);
            } else {
#pragma unroll
              for (int j = 0; j < kBNb / kRows64; ++j)
                load_box<CG>(b + j * kBK * 128, &p.b, rb + j * kRows64, kb * kBK, &full[s], bar);
            }
          }
          __syncwarp();
        }
      }
      // Copies still in flight have to land before the shared memory goes.
      if ((!ok || *abort_flag) && rank == 0 && lead) {
        const uint32_t n = it < (uint32_t)p.stages ? it : (uint32_t)p.stages;
        for (uint32_t j = it - n; j < it; ++j)
          tc::mbar_wait(&full[j % p.stages], (j / p.stages) & 1, nullptr, kWaitNs);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (rank == 0) {  // ---- products ----
      const bool lead = tc::elect_one();
      uint32_t it = 0, ti = 0;  // K blocks, accumulators
      bool ok = true;
      for (int t = first_tile; t < p.num_tiles && ok; t += tile_step) {
        int tm, tn, sp;
        tile_at(p, t, tm, tn, sp);
        const int kb0 = (int)((long long)p.kblocks * sp / p.splits);
        const int kb1 = (int)((long long)p.kblocks * (sp + 1) / p.splits);
        // An accumulator holds a tile, or (FP32 data) one K block of it: the
        // tensor cores cut off what they add to FP32 sums, and only a short
        // chain of such sums keeps FP32's digits. The epilogue adds the blocks.
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          const bool first = kb == kb0;
          if (first || PARTS == 3) {
            if (!warp_wait<CG == 2>(&acc_empty[ti & 1], ((ti >> 1) & 1) ^ 1, abort_flag)) {
              if (lead) give_up(abort_flag, p.status, 92);
              ok = false;
              break;
            }
            tc::tc_fence_after();
          }
          const uint32_t d = tmem + (ti & 1) * BN;
          // the operands' slot: the stage itself, or (FP32 data) its parts
          const int s = PARTS == 3 ? it & 1 : it % p.stages;
          const uint32_t phase = PARTS == 3 ? (it >> 1) & 1 : (it / p.stages) & 1;
          if (!warp_wait(PARTS == 3 ? &parts_full[s] : &full[s], phase, abort_flag)) {
            if (lead) give_up(abort_flag, p.status, 93);
            ok = false;
            break;
          }
          uint64_t ad, bd;
          uint32_t ak, bk;  // a K step of 16, in descriptor units of 16 bytes
          if constexpr (PARTS == 1) {
            const uint32_t sa = tc::smem_u32(smem + s * L.stage);
            const uint32_t sb = sa + kStageA;
            ad = p.a_mn ? tc::smem_desc_sw128_mn(sa, 8192) : tc::smem_desc_sw128(sa);
            bd = p.b_mn ? tc::smem_desc_sw128_mn(sb, 8192) : tc::smem_desc_sw128(sb);
            ak = (p.a_mn ? 2048 : 32) >> 4;
            bk = (p.b_mn ? 2048 : 32) >> 4;
          } else {  // core matrices, [8 values][outer index]
            const uint32_t sa = tc::smem_u32(smem + L.planes + s * 3 * (kPartA + kPartB));
            const uint32_t sb = sa + 3 * kPartA;
            ad = p.a_mn ? tc::smem_desc(sa, 128, kBK * 16) : tc::smem_desc(sa, kBM * 16, 128);
            bd = p.b_mn ? tc::smem_desc(sb, 128, kBK * 16) : tc::smem_desc(sb, BN * 16, 128);
            ak = (p.a_mn ? 256 : 2 * kBM * 16) >> 4;
            bk = (p.b_mn ? 256 : 2 * BN * 16) >> 4;
          }
          const int ksteps = kb == p.kblocks - 1 ? p.last_ksteps : kBK / 16;
          auto products = [&](auto steps) {
            if constexpr (PARTS == 1) {
#pragma unroll
              for (int ks = 0; ks < steps; ++ks)
                mma<CG>(d, ad + ks * ak, bd + ks * bk, p.idesc, (!first || ks > 0) ? 1u : 0u);
            } else {
              constexpr uint32_t ap = kPartA >> 4, bp = kPartB >> 4;
              // the small products first, while the sum is small
#pragma unroll
              for (int ks = 0; ks < steps; ++ks) {
                const uint64_t a0 = ad + ks * ak, b0 = bd + ks * bk;
                mma<CG>(d, a0 + 2 * ap, b0, p.idesc, ks > 0 ? 1u : 0u);
                mma<CG>(d, a0, b0 + 2 * bp, p.idesc, 1u);
                mma<CG>(d, a0 + ap, b0 + bp, p.idesc, 1u);
                mma<CG>(d, a0 + ap, b0, p.idesc, 1u);
                mma<CG>(d, a0, b0 + bp, p.idesc, 1u);
              }
#pragma unroll
              for (int ks = 0; ks < steps; ++ks)
                mma<CG>(d, ad + ks * ak, bd + ks * bk, p.idesc, 1u);
            }
          };
          if (lead) {
            if (ksteps == kBK / 16) products(std::integral_constant<int, kBK / 16>());
            else products(ksteps);
            commit<CG>(PARTS == 3 ? &parts_empty[s] : &empty[s]);
            if constexpr (PARTS == 3) commit<CG>(&acc_full[ti & 1]);
          }
          __syncwarp();
          if (PARTS == 3) ++ti;
        }
        if (PARTS == 1 && ok) {
          if (lead) commit<CG>(&acc_full[ti & 1]);
          __syncwarp();
          ++ti;
        }
      }
      if (lead) commit<CG>(&drained);
      __syncwarp();
    }
    // Every product has completed before the tensor memory is freed, and every
    // arrival that a commit promised to this block's barriers, those that nobody
    // else waits for among them, has come before its shared memory goes. (The
    // last phases are awaited behind `drained`: by then no barrier is more than
    // one phase behind them, so their parity tells.)
    warp_wait(&drained, 0, rank == 0 ? nullptr : abort_flag);
    const uint32_t n = total_blocks();
    const uint32_t ring = PARTS == 3 ? 2 : p.stages;
    for (uint32_t j = n > ring ? n - ring : 0; j < n; ++j)
      if (!warp_wait(PARTS == 3 ? &parts_empty[j % ring] : &empty[j % ring], (j / ring) & 1,
                     abort_flag))
        break;
    __syncwarp();
  } else if (PARTS == 3 && warp >= kFirstSplit) {  // ---- parts of FP32 operands ----
    // Two groups of four warps take the K blocks in turn, each into its own set
    // of parts. A 16-byte row of a part holds 8 values along the contiguous axis;
    // rows lie along the other one.
    const int team = (warp - kFirstSplit) >> 2;
    const int me = ((warp - kFirstSplit) & 3) * 32 + lane;
    const bool lead = tc::elect_one();
    const uint32_t blocks = total_blocks();
    auto split_operand = [&](const uint8_t* raw, uint8_t* dst, bool mn, auto width) {
      constexpr int kW = decltype(width)::value;  // rows (columns) of the operand
      constexpr uint32_t kPart = kW * kBK * 2;
#pragma unroll 4
      for (int item = me; item < kW * kBK / 8; item += 128) {
        // K-major: [k / 8][row]; MN-major: [row / 8][k]
        const int o = mn ? item % kBK : item % kW, g = mn ? item / kBK : item / kW;
        const uint8_t* line = raw + (mn ? (g / 4) * kBK * 128 + o * 128 : o * 128);
        const int c = mn ? (g % 4) * 2 : g * 2;
        const float4 lo = *reinterpret_cast<const float4*>(line + ((c ^ (o & 7)) * 16));
        const float4 hi = *reinterpret_cast<const float4*>(line + (((c + 1) ^ (o & 7)) * 16));
        const float v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
        uint32_t part[3][4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          // the first part is cut off, not rounded: it cannot overflow
          const uint32_t a = __float_as_uint(v[2 * e]), b = __float_as_uint(v[2 * e + 1]);
          part[0][e] = __byte_perm(a, b, 0x7632);
          const float ra = v[2 * e] - __uint_as_float(a & 0xffff0000u);
          const float rb = v[2 * e + 1] - __uint_as_float(b & 0xffff0000u);
          part[1][e] = pack2<__nv_bfloat16>(ra, rb);
          const float2 h = unpack2<__nv_bfloat16>(part[1][e]);
          part[2][e] = pack2<__nv_bfloat16>(ra - h.x, rb - h.y);
        }
#pragma unroll
        for (int q = 0; q < 3; ++q)
          *reinterpret_cast<uint4*>(dst + q * kPart + item * 16) =
              make_uint4(part[q][0], part[q][1], part[q][2], part[q][3]);
      }
    };
    uint8_t* dst = smem + L.planes + team * 3 * (kPartA + kPartB);
    for (uint32_t i = team; i < blocks; i += 2) {
      const uint32_t s = i % p.stages;
      if (!warp_wait(&full[s], (i / p.stages) & 1, abort_flag) ||
          !warp_wait(&parts_empty[team], ((i >> 1) & 1) ^ 1, abort_flag)) {
        if (lead) give_up(abort_flag, p.status, 96);
        break;
      }
      const uint8_t* raw = smem + s * L.stage;
      split_operand(raw, dst, p.a_mn, std::integral_constant<int, kBM>());
      split_operand(raw + kStageA, dst + 3 * kPartA, p.b_mn, std::integral_constant<int, kBNb>());
      tc::fence_proxy_async_smem();
      __syncwarp();
      if (lead) {
        tc::mbar_arrive(&empty[s]);
        tc::mbar_arrive(&parts_full[team]);
      }
    }
  } else if (warp >= kFirstEpi) {  // ---- epilogue ----
    const int ew = warp - kFirstEpi;
    const bool lead = tc::elect_one();  // copies, stores and arrivals of the warp
    const int group = ew >> 3, quad = warp & 3, part = (ew >> 2) & 1;
    uint8_t* boxes = smem + L.boxes + ew * p.nbuf * kBox;
    float* bias_s = reinterpret_cast<float*>(smem + L.bias) + ew * kCols;
    const To* in = static_cast<const To*>(p.in_ptr);
    const T* bias = static_cast<const T*>(p.bias);
    To* out = static_cast<To*>(p.out_ptr);
    const bool has_in = kEpi != kPartial && p.in_ptr != nullptr;
    const int ahead = has_in ? p.nbuf / 2 : 0;  // boxes loaded ahead
    // 16-byte chunk c of the box's row r lies at chunk c ^ swizzle(r), as TMA's
    // 64- and 128-byte swizzles have it
    auto chunk_at = [](int r, int c) {
      return kRow == 128 ? r * 128 + ((c ^ (r & 7)) * 16) : r * 64 + ((c ^ ((r >> 1) & 3)) * 16);
    };
    auto value_at = [&](int r, int c) {
      return chunk_at(r, c / kPer) + (c % kPer) * (int)sizeof(To);
    };
    uint32_t ti = group, q = 0;
    // the load cursor: box `lj` of tile `lt`
    int lt = first_tile + group * tile_step, lj = 0;
    uint32_t lq = 0;
    auto load_next = [&]() {  // the elected lane
      if (lt >= p.num_tiles) return;
      int tm, tn, sp;
      tile_at(p, lt, tm, tn, sp);
      const int c = tn * BN + part * kCols + lj * kCB, r = (tm * CG + rank) * kBM + quad * 32;
      const int b = lq % p.nbuf;
      if (c < p.N && r < p.M) {
        tc::mbar_arrive_expect_tx(&in_full[ew][b], kBox);
        tc::tma_load_3d(boxes + b * kBox, &p.in, c, r, 0, &in_full[ew][b]);
      } else {
        tc::mbar_arrive(&in_full[ew][b]);
      }
      ++lq;
      if (++lj == kBoxes) {
        lj = 0;
        lt += kGroups * tile_step;
      }
    };
    if (p.tma_io && has_in && lead)
      for (int i = 0; i < ahead; ++i) load_next();
    bool ok = true;
    for (int t = first_tile + group * tile_step; t < p.num_tiles && ok;
         t += kGroups * tile_step) {
      int tm, tn, sp;
      tile_at(p, t, tm, tn, sp);
      const int row0 = (tm * CG + rank) * kBM + quad * 32;
      const int row = row0 + lane;
      const int col0 = tn * BN + part * kCols;
      const uint32_t tcol = tmem + ((uint32_t)(quad * 32) << 16) + part * kCols;
      if constexpr (kEpi != kPartial && PARTS == 1) {
        if (bias != nullptr) {
#pragma unroll
          for (int i = lane; i < kCols; i += 32)
            bias_s[i] = col0 + i < p.N ? ldg_f32<T>(bias + col0 + i) : 0.f;
          __syncwarp();
        }
      }
      float sum[PARTS == 3 ? kCols : 1];  // FP32 data: the K blocks added up
      if constexpr (PARTS == 3) {
        const int kb0 = (int)((long long)p.kblocks * sp / p.splits);
        const int kb1 = (int)((long long)p.kblocks * (sp + 1) / p.splits);
#pragma unroll
        for (int i = 0; i < kCols; ++i) sum[i] = 0.f;
        for (int kb = kb0; kb < kb1; ++kb, ++ti) {
          ok = warp_wait(&acc_full[ti & 1], (ti >> 1) & 1, abort_flag);
          if (!ok) break;
          tc::tc_fence_after();
#pragma unroll
          for (int i = 0; i < kCols; i += 32) {
            float v[32];
            tc::tmem_ld16(tcol + (ti & 1) * BN + i, *reinterpret_cast<float(*)[16]>(v));
            tc::tmem_ld16(tcol + (ti & 1) * BN + i + 16, *reinterpret_cast<float(*)[16]>(v + 16));
            tc::tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e) sum[i + e] += v[e];
          }
          tc::tc_fence_before();
          __syncwarp();
          if (lead) arrive_leader<CG>(&acc_empty[ti & 1]);
        }
      } else {
        ok = warp_wait(&acc_full[ti & 1], (ti >> 1) & 1, abort_flag);
        tc::tc_fence_after();
      }
      if (!ok) {
        if (lead) give_up(abort_flag, p.status, 94);
        break;
      }
      // Steps of 32 columns: while one is worked on, the next one's tensor-memory
      // load is in flight (a step is a chain of latencies, and only two warps
      // share a scheduler).
      const uint32_t taddr = tcol + (ti & 1) * BN;
      float v[2][32];
      auto fetch = [&](int step, float (&d)[32]) {
        if constexpr (PARTS == 1) {
          tc::tmem_ld16(taddr + step * 32, *reinterpret_cast<float(*)[16]>(d));
          tc::tmem_ld16(taddr + step * 32 + 16, *reinterpret_cast<float(*)[16]>(d + 16));
        }
      };
      fetch(0, v[0]);
#pragma unroll (PARTS == 3 ? kBoxes : 1)
      for (int j = 0; j < kBoxes; ++j, ++q) {
        const int c0 = col0 + j * kCB;
        const int b = q % p.nbuf;
        uint8_t* box = boxes + b * kBox;
        const bool live = c0 < p.N && row0 < p.M;  // the box holds anything
        // make room, and fetch a later box of the residual
        if (p.tma_io) {
          if (lead) {
            const int pending = has_in ? p.nbuf - ahead - 1 : p.nbuf - 1;
            if (pending >= 7) tc::bulk_wait_read<7>();
            else if (pending >= 3) tc::bulk_wait_read<3>();
            else if (pending >= 1) tc::bulk_wait_read<1>();
            else tc::bulk_wait_read<0>();
            if (has_in) load_next();
          }
          __syncwarp();
        }
        if (has_in) {
          if (p.tma_io) {
            ok = warp_wait(&in_full[ew][b], (q / p.nbuf) & 1, abort_flag);
            if (!ok) {
              if (lead) give_up(abort_flag, p.status, 95);
              break;
            }
          } else if (live) {
            // rows one after the other, a lane per column
#pragma unroll
            for (int cc = 0; cc < kCB; cc += 32) {
              const int c = cc + lane;
              if (c0 + c < p.N) {
#pragma unroll 16
                for (int r = 0; r < 32; ++r)
                  if (row0 + r < p.M)
                    *reinterpret_cast<To*>(box + value_at(r, c)) =
                        in[(long long)(row0 + r) * p.ld_in + c0 + c];
              }
            }
            __syncwarp();
          }
        }
#pragma unroll
        for (int sub = 0; sub < kSub; ++sub) {
          float (&w)[32] = v[kSub == 2 ? sub : 0];
          if constexpr (PARTS == 3) {
#pragma unroll
            for (int i = 0; i < 32; ++i) w[i] = sum[j * kCB + sub * 32 + i];
          } else {
            tc::tmem_ld_wait();
            if constexpr (kSub == 2) {
              if (sub == 0) fetch(j * 2 + 1, v[1]);
              else if (j + 1 < kBoxes) fetch(j * 2 + 2, v[0]);
            }
            if (sub == kSub - 1 && j == kBoxes - 1) {  // the accumulator is free
              tc::tc_fence_before();
              __syncwarp();
              if (lead) arrive_leader<CG>(&acc_empty[ti & 1]);
            }
          }
          if (live) {
            if constexpr (kEpi != kPartial) {
              if (bias != nullptr) {
                if constexpr (PARTS == 1) {
                  const float4* bs = reinterpret_cast<const float4*>(bias_s + j * kCB + sub * 32);
#pragma unroll
                  for (int i = 0; i < 8; ++i) {
                    const float4 u = bs[i];
                    w[4 * i] += u.x;
                    w[4 * i + 1] += u.y;
                    w[4 * i + 2] += u.z;
                    w[4 * i + 3] += u.w;
                  }
                } else {  // no room for it beside the parts
#pragma unroll
                  for (int i = 0; i < 32; ++i) {
                    const int c = c0 + sub * 32 + i;
                    w[i] += ldg_f32<T>(bias + (c < p.N ? c : p.N - 1));
                  }
                }
              }
              if constexpr (kEpi == kOut) act_values<kFast, 32>(p.act, w);
              else act_slopes<kFast, 32>(p.act, w);
            }
#pragma unroll
            for (int k = 0; k < 32 / kPer; ++k) {
              uint4* at = reinterpret_cast<uint4*>(box + chunk_at(lane, sub * (32 / kPer) + k));
              if (has_in) {
                float f[kPer];
                unpack16<To>(*at, f);
#pragma unroll
                for (int i = 0; i < kPer; ++i) {
                  if constexpr (kEpi == kDz) w[k * kPer + i] *= f[i];
                  else w[k * kPer + i] += f[i];
                }
              }
              *at = pack16<To>(w + k * kPer);
            }
            if constexpr (kEpi == kDz) {
              if (p.colsum != nullptr) {
                if (row >= p.M) {
#pragma unroll
                  for (int i = 0; i < 32; ++i) w[i] = 0.f;
                }
                const float total = column_sums(w, lane);
                if (c0 + sub * 32 + lane < p.N)
                  p.colsum[(long long)(row0 / 32) * p.N + c0 + sub * 32 + lane] = total;
              }
            }
          }
          if constexpr (PARTS == 1 && kSub == 1) {
            if (j + 1 < kBoxes) fetch(j + 1, v[0]);
          }
        }
        if (live) {
          if (p.tma_io) {
            tc::fence_proxy_async_smem();
            __syncwarp();
            if (lead) tc::tma_store_3d(&p.out, box, c0, row0, sp);
          } else {
            __syncwarp();
#pragma unroll
            for (int cc = 0; cc < kCB; cc += 32) {
              const int c = cc + lane;
              if (c0 + c < p.N) {
#pragma unroll 8
                for (int r = 0; r < 32; ++r)
                  if (row0 + r < p.M)
                    out[(long long)(row0 + r) * p.ld_out + c0 + c] =
                        *reinterpret_cast<const To*>(box + value_at(r, c));
              }
            }
            __syncwarp();
          }
        }
        // a group for every box, written or not, so that counting groups
        // counts boxes
        if (p.tma_io && lead) tc::bulk_commit();
      }
      if (!ok) break;
      if constexpr (PARTS == 1) ti += kGroups;
    }
    if (p.tma_io && lead) {
      if (!ok || *abort_flag) {  // loads ahead of the failure land first
        for (uint32_t i = q; i < lq; ++i)
          tc::mbar_wait(&in_full[ew][i % p.nbuf], (i / p.nbuf) & 1, nullptr, kWaitNs);
      }
      tc::bulk_wait_all();
    }
    __syncwarp();
  }
  tc::tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();  // the pair's products and arrivals are over
  if (warp == 2) {
    tc::tc_fence_after();
    tmem_dealloc<CG>(tmem, 2 * BN);
  }
}

// --------------------------------------------------------- small kernels ----
// Rows of `src` copied to a pitch (a multiple of 8 values) that TMA can address.
template <typename T>
__global__ void __launch_bounds__(256) linear_stage_kernel(const T* __restrict__ src, long long ld,
                                                           long long rows, int cols, int pitch,
                                                           uint4* __restrict__ dst) {
  constexpr int kPer = 16 / (int)sizeof(T);
  const int per = pitch / kPer;
  const long long total = rows * per;
  const bool vec = ld * sizeof(T) % 16 == 0 && (uintptr_t)src % 16 == 0;
  for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < total;
       i += (long long)gridDim.x * blockDim.x) {
    const long long r = i / per;
    const int c = (int)(i - r * per) * kPer;
    union { uint4 u; T e[kPer]; } v;
    const T* s = src + r * ld + c;
    if (vec && c + kPer <= cols) {
      v.u = __ldg(reinterpret_cast<const uint4*>(s));
    } else {
#pragma unroll
      for (int k = 0; k < kPer; ++k) v.e[k] = c + k < cols ? s[k] : from_f32<T>(0.f);
    }
    dst[i] = v.u;
  }
}

// Column sums of `src` rows, a chunk of rows per blockIdx.y, into FP32
// partials [chunk][cols].
template <typename T>
__global__ void __launch_bounds__(256) linear_colsum_kernel(const T* __restrict__ src,
                                                            long long rows, int cols,
                                                            long long chunk,
                                                            float* __restrict__ part) {
  __shared__ float sh[8][32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  const long long r0 = blockIdx.y * chunk, r1 = min(rows, r0 + chunk);
  float a = 0.f;
  if (c < cols)
#pragma unroll 8
    for (long long r = r0 + w; r < r1; r += 8) a += to_f32<T>(src[r * cols + c]);
  sh[w][lane] = a;
  __syncthreads();
  if (w == 0 && c < cols) {
    for (int i = 1; i < 8; ++i) a += sh[i][lane];
    part[(long long)blockIdx.y * cols + c] = a;
  }
}

// out[r][c] = sum over `count` partials [count][rows][pitch].
struct Fold {
  const float* part;
  long long rows, pitch;
  int count, cols, blocks;
  void* out;
};

// A thread per value, the partials in order: few of them, many values.
template <typename T>
__global__ void __launch_bounds__(256) linear_fold_kernel(const Fold f) {
  const long long total = f.rows * f.cols;
  for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < total;
       i += (long long)gridDim.x * blockDim.x) {
    const long long r = i / f.cols;
    const float* s = f.part + r * f.pitch + (i - r * f.cols);
    float a = 0.f;
#pragma unroll 8
    for (int k = 0; k < f.count; ++k) a += s[(long long)k * f.rows * f.pitch];
    static_cast<T*>(f.out)[i] = from_f32<T>(a);
  }
}

// 32 values a block, whose 32 warps share the partials: many of them. Two sums
// in one launch (the bias's and the weight's gradient).
template <typename T>
__global__ void __launch_bounds__(1024) linear_fold_long_kernel(const Fold f0, const Fold f1) {
  __shared__ float sh[32][33];
  const bool second = (int)blockIdx.x >= f0.blocks;
  const Fold& f = second ? f1 : f0;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const long long i = (blockIdx.x - (second ? f0.blocks : 0)) * 32LL + lane;
  const long long total = f.rows * f.cols, step = f.rows * f.pitch;
  float a = 0.f;
  if (i < total) {
    const long long r = i / f.cols;
    const float* s = f.part + r * f.pitch + (i - r * f.cols);
#pragma unroll 8
    for (int k = w; k < f.count; k += 32) a += s[(long long)k * step];
  }
  sh[w][lane] = a;
  __syncthreads();
  if (w == 0 && i < total) {
    for (int k = 1; k < 32; ++k) a += sh[k][lane];
    static_cast<T*>(f.out)[i] = from_f32<T>(a);
  }
}

// The epilogue of a product whose K axis was split: the partials [splits][M][pitch]
// in order, then what the product's own epilogue does. 32 rows of 256 columns a
// block, a column a thread (kDz: its sum over the 32 rows is one of `colsum`).
struct Finish {
  const float* part;
  long long M, pitch;
  int splits, N, tiles_n, act;
  const void* bias;  // nullable
  const void* in;    // residual (kOut, nullable) or dy (kDz), [M][N]
  void* out;
  long long ld_out;
  float* colsum;     // nullable
};
template <typename T, Epi kEpi>
__global__ void __launch_bounds__(256) linear_finish_kernel(const Finish f) {
  const int tm = (int)(blockIdx.x / (unsigned)f.tiles_n);
  const int c = (int)(blockIdx.x - (unsigned)tm * f.tiles_n) * 256 + (int)threadIdx.x;
  if (c >= f.N) return;
  const long long row0 = tm * 32LL;
  const int rows = (int)min(32LL, f.M - row0);
  const float bias = f.bias ? to_f32<T>(static_cast<const T*>(f.bias)[c]) : 0.f;
  const T* in = static_cast<const T*>(f.in);
  T* out = static_cast<T*>(f.out);
  float total = 0.f;
  for (int r = 0; r < rows; r += 2) {
    float v[2] = {0.f, 0.f};
    for (int k = 0; k < f.splits; ++k)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (r + e < rows) v[e] += f.part[(k * f.M + row0 + r + e) * f.pitch + c];
    v[0] += bias;
    v[1] += bias;
    if constexpr (kEpi == kOut) act_values<sizeof(T) == 2, 2>(f.act, v);
    else act_slopes<sizeof(T) == 2, 2>(f.act, v);
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (r + e < rows) {
        const long long row = row0 + r + e;
        if (in != nullptr) {
          const float u = to_f32<T>(in[row * f.N + c]);
          v[e] = kEpi == kOut ? v[e] + u : v[e] * u;
        }
        out[row * f.ld_out + c] = from_f32<T>(v[e]);
        total += v[e];
      }
  }
  if (kEpi == kDz && f.colsum != nullptr) f.colsum[(long long)tm * f.N + c] = total;
}

// Forward of up to kGemvRows rows: a warp per output column, V values of the
// weight a lane and load, FP32 products.
template <typename T, int V, int MR>
__global__ void __launch_bounds__(256) linear_rows_kernel(const T* __restrict__ x, long long ldx,
                                                          const T* __restrict__ w,
                                                          const T* __restrict__ bias,
                                                          const T* __restrict__ res, T* out, int m,
                                                          int n, int k, int act) {
  struct alignas(sizeof(T) * V) Vt { T e[V]; };
  const int lane = threadIdx.x & 31;
  const int col = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (col >= n) return;
  const T* wr = w + (long long)col * k;
  float acc[MR];
#pragma unroll
  for (int r = 0; r < MR; ++r) acc[r] = 0.f;
#pragma unroll 4
  for (int i = lane * V; i < k; i += 32 * V) {
    const Vt wv = *reinterpret_cast<const Vt*>(wr + i);
#pragma unroll
    for (int r = 0; r < MR; ++r) {
      if (r < m) {
        const Vt xv = *reinterpret_cast<const Vt*>(x + r * ldx + i);
#pragma unroll
        for (int e = 0; e < V; ++e) acc[r] = fmaf(to_f32<T>(wv.e[e]), to_f32<T>(xv.e[e]), acc[r]);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < MR; ++r)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) acc[r] += __shfl_xor_sync(0xffffffffu, acc[r], o);
  float z[2] = {0.f, 0.f};
#pragma unroll
  for (int r = 0; r < MR; ++r)
    if (lane == r) z[0] = acc[r];
  if (lane < m) {
    if (bias != nullptr) z[0] += to_f32<T>(bias[col]);
    act_values<sizeof(T) == 2, 2>(act, z);
    const long long at = (long long)lane * n + col;
    if (res != nullptr) z[0] += to_f32<T>(res[at]);
    out[at] = from_f32<T>(z[0]);
  }
}

// ------------------------------------------------------------ host: plan ----
size_t up256(size_t v) { return (v + 255) / 256 * 256; }
int round8(int v) { return (v + 7) / 8 * 8; }

// An operand in memory: rows x cols values, `pitch` values from row to row.
struct Operand {
  const void* ptr;
  long long rows;
  int cols;
  long long pitch;
};

template <typename T> struct OpOf { using type = T; };
template <> struct OpOf<float> { using type = __nv_bfloat16; };

int small_grid(long long items) {
  const long long want = (items + 255) / 256, most = gencat::num_sms() * 8;
  return (int)(want < 1 ? 1 : want < most ? want : most);
}

size_t staged_bytes(long long rows, int cols, int es) {
  return up256((size_t)rows * round8(cols) * es);
}

template <typename T>
int stage(const void* src, long long ld, long long rows, int cols, void* dst, cudaStream_t st) {
  const int pitch = round8(cols);
  linear_stage_kernel<T><<<small_grid(rows * (pitch * (int)sizeof(T) / 16)), 256, 0, st>>>(
      static_cast<const T*>(src), ld, rows, cols, pitch, static_cast<uint4*>(dst));
  DDPM_CHECK_LAUNCH("linear_stage_kernel");
  return DDPM_OK;
}

// Tile of a product: columns, blocks that share it, epilogue warps.
struct Tile {
  int bn, cg, ew;
};

// The tile with the least estimated time: rounds of tiles over the SMs, each
// the clocks of its K blocks (the larger of what the tensor cores and the
// shared memory need: a block's operands are written once and read once per
// product) plus a constant for filling and draining.
Tile pick_tile(long long m, int n, long long k, int parts, int splits) {
  const int sms = gencat::num_sms(), bk = block_k(parts);
  const long long kb = ((k + bk - 1) / bk + splits - 1) / splits;
  Tile best{64, 1, 8};
  double least = 0;
  for (int cg = 1; cg <= (parts == 3 ? 1 : 2); ++cg)
    for (int bn = parts == 3 ? 128 : 256; bn >= (cg == 2 ? 256 : 64); bn /= 2) {
      const long long tiles =
          ((m + kBM * cg - 1) / (kBM * cg)) * ((n + bn - 1) / bn) * splits;
      const long long units = sms / cg;
      const long long rounds = (tiles + units - 1) / units;
      // FP32: splitting the operands is the longest part of a block
      const double mma = 2.0 * bn, move = 2.0 * (kBM + bn / cg);
      const double block = parts == 3 ? 150.0 + 3.2 * (kBM + bn) : mma > move ? mma : move;
      const double t = rounds * (kb * block + 1000.0 + 4.0 * bn);
      if (least == 0 || t < least) {
        least = t;
        // a short K loop leaves the epilogue as the longest part of a tile: twice
        // the warps there (65536 x k -> 1728, k = 64: 94 -> 72 us, 128: 95 -> 75, 256:
        // 97 both), which a longer one pays for with stages (384: 110 -> 121 us, 512:
        // 122 -> 155). A block on its own has no room for them
        // beside two stages, and with one a copy waits for the product before it
        // (64 x 512 -> 25600: 14.2 us, with 8 warps 9.5 us).
        best = Tile{bn, cg, cg == 2 && kb <= kShortK ? 16 : 8};
      }
    }
  return best;
}

int smem_limit() { return gencat::max_smem_optin() - 2048; }  // less the static shared memory

// Stages and boxes of a block, and their bytes. `es`: bytes of a value of out.
// As many stages as the K loop can use, at least two; what is left goes to the
// epilogue's boxes, eight a warp at most, two at least.
struct Rings {
  int stages, nbuf, smem;
};
Rings pick_rings(Tile t, int parts, int es, long long kblocks, int splits) {
  const int limit = smem_limit(), row = box_row(t.bn, es);
  auto total = [&](int s, int b) {
    return (int)smem_layout(t.cg, parts, t.bn, t.ew, row, s, b).total;
  };
  // a persistent block streams several tiles through the ring: twice a tile's
  // steps is as far ahead as it needs to look
  const long long tiles_k = (kblocks + splits - 1) / splits;
  Rings r{tiles_k * 2 < kMaxStages ? (int)tiles_k * 2 : kMaxStages, 2, 0};
  while (r.stages > 2 && total(r.stages, r.nbuf) > limit) --r.stages;
  while (r.nbuf < kMaxBufs && total(r.stages, r.nbuf + 1) <= limit) ++r.nbuf;
  r.smem = total(r.stages, r.nbuf);
  return r;
}

template <typename T, int BN, int PARTS, Epi kEpi, int CG, int EW>
int launch_gemm_as(GemmParams& p, cudaStream_t st) {
  auto fn = linear_gemm_kernel<T, BN, PARTS, kEpi, CG, EW>;
  const int limit = smem_limit();
  const Rings r = pick_rings(Tile{BN, CG, EW}, PARTS, kEpi == kPartial ? 4 : (int)sizeof(T),
                             p.kblocks, p.splits);
  if (r.smem > limit)
    return set_error(DDPM_ERR_UNSUPPORTED, "linear: %d bytes of shared memory, %d needed", limit,
                     r.smem);
  p.stages = r.stages;
  p.nbuf = r.nbuf;
  const int smem = r.smem;
  static std::atomic<unsigned long long> ready{0};  // devices whose limit is raised
  int dev = 0;
  DDPM_CUDA_TRY(cudaGetDevice(&dev));
  if (dev >= 64 || !(ready.load(std::memory_order_relaxed) >> dev & 1)) {
    DDPM_CUDA_TRY(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, limit));
    if (dev < 64) ready.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  const int units = gencat::num_sms() / CG;
  const int grid = (p.num_tiles < units ? p.num_tiles : units) * CG;
  if constexpr (CG == 1) {
    fn<<<grid, gemm_threads(PARTS, EW), smem, st>>>(p);
  } else {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(gemm_threads(PARTS, EW));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = CG;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    DDPM_CUDA_TRY(cudaLaunchKernelEx(&cfg, fn, p));
  }
  DDPM_CHECK_LAUNCH("linear_gemm_kernel");
  return DDPM_OK;
}

template <typename T, Epi kEpi>
int launch_gemm(GemmParams& p, Tile t, cudaStream_t st) {
  if constexpr (sizeof(T) == 4) {
    return t.bn == 128 ? launch_gemm_as<T, 128, 3, kEpi, 1, 8>(p, st)
                       : launch_gemm_as<T, 64, 3, kEpi, 1, 8>(p, st);
  } else {
    return t.ew == 16    ? launch_gemm_as<T, 256, 1, kEpi, 2, 16>(p, st)
           : t.cg == 2   ? launch_gemm_as<T, 256, 1, kEpi, 2, 8>(p, st)
           : t.bn == 256 ? launch_gemm_as<T, 256, 1, kEpi, 1, 8>(p, st)
           : t.bn == 128 ? launch_gemm_as<T, 128, 1, kEpi, 1, 8>(p, st)
                         : launch_gemm_as<T, 64, 1, kEpi, 1, 8>(p, st);
  }
}

int operand_map(CUtensorMap* map, const Operand& o, bool mn_major, int tile_rows, int es, bool bf16) {
  // 128 bytes along the contiguous axis; K-major: x the tile's rows, MN-major
  // (the operand's rows are the contraction's k): x a block of k
  const uint64_t dims[3] = {(uint64_t)o.cols, (uint64_t)o.rows, 1};
  const uint64_t strides[2] = {(uint64_t)o.pitch * es, (uint64_t)o.rows * o.pitch * es};
  const uint32_t box[3] = {(uint32_t)(128 / es), (uint32_t)(mn_major ? 128 / es : tile_rows), 1};
  return encode_tmap(map,
                     es == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                     : bf16  ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                             : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                     3, o.ptr, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

int io_map(CUtensorMap* map, const void* ptr, int es, bool bf16, long long rows, int cols,
           long long ld, int splits, int row_bytes) {
  const uint64_t dims[3] = {(uint64_t)cols, (uint64_t)rows, (uint64_t)splits};
  const uint64_t strides[2] = {(uint64_t)ld * es, (uint64_t)rows * ld * es};
  const uint32_t box[3] = {(uint32_t)(row_bytes / es), 32, 1};
  return encode_tmap(map,
                     es == 4  ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                     : bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                            : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                     3, ptr, dims, strides, box,
                     row_bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
}

// D[M][N] = sum over K of A and B as described above. `k` counts A's columns
// (K-major) or rows (MN-major).
struct Gemm {
  Operand a, b;
  bool a_mn, b_mn;
  long long M;
  int N;
  long long K;
  const void* bias;
  const void* in;
  long long ld_in;
  void* out;
  long long ld_out;
  int act;
  float* colsum;
  int splits;
  Tile tile;
};

bool tma_ready(const void* ptr, long long ld, int es) {
  return (uintptr_t)ptr % 16 == 0 && ld * es % 16 == 0;
}

template <typename T, Epi kEpi>
int run_gemm(const Gemm& g, cudaStream_t st) {
  using Op = typename OpOf<T>::type;
  constexpr bool kBf16 = std::is_same<Op, __nv_bfloat16>::value;
  const int es = kEpi == kPartial ? 4 : (int)sizeof(T);
  GemmParams p{};
  const int tile_m = kBM * g.tile.cg, bn = g.tile.bn;
  p.tiles_m = (int)((g.M + tile_m - 1) / tile_m);
  p.tiles_n = (g.N + bn - 1) / bn;
  p.splits = g.splits;
  p.num_tiles = p.tiles_m * p.tiles_n * g.splits;
  constexpr int kBK = block_k(sizeof(T) == 4 ? 3 : 1);
  p.kblocks = (int)((g.K + kBK - 1) / kBK);
  p.last_ksteps = (int)((g.K - (long long)(p.kblocks - 1) * kBK + 15) / 16);
  p.M = (int)g.M;
  p.N = g.N;
  p.a_mn = g.a_mn;
  p.b_mn = g.b_mn;
  p.act = g.act;
  p.bias = g.bias;
  p.in_ptr = g.in;
  p.out_ptr = g.out;
  p.ld_in = g.ld_in;
  p.ld_out = g.ld_out;
  p.colsum = g.colsum;
  p.idesc = tc::idesc_f16(tile_m, bn, kBf16, g.a_mn, g.b_mn);
  p.tma_io = tma_ready(g.out, g.ld_out, es) && (g.in == nullptr || tma_ready(g.in, g.ld_in, es));
  int rc = gencat::status_ptr(&p.status);
  if (rc) return rc;
  rc = operand_map(&p.a, g.a, g.a_mn, kBM, (int)sizeof(T), kBf16);
  if (rc) return rc;
  rc = operand_map(&p.b, g.b, g.b_mn, bn / g.tile.cg, (int)sizeof(T), kBf16);
  if (rc) return rc;
  const int row = box_row(bn, es);
  if (p.tma_io) {
    rc = io_map(&p.out, g.out, es, kBf16, g.M, g.N, g.ld_out, g.splits, row);
    if (rc) return rc;
    if (g.in != nullptr) {
      rc = io_map(&p.in, g.in, es, kBf16, g.M, g.N, g.ld_in, 1, row);
      if (rc) return rc;
    }
  }
  return launch_gemm<T, kEpi>(p, g.tile, st);
}

long long pitch4(int n) { return (n + 3) / 4 * 4; }

// Rows of a split product that are done at a time, so that its partials take no
// more than kPartBytes (or 256 rows' worth).
constexpr size_t kPartBytes = 1ull << 30;
long long part_rows(int splits, long long rows, int cols) {
  const long long fit = (long long)(kPartBytes / ((size_t)splits * pitch4(cols) * 4)) / 256 * 256;
  return rows <= fit ? rows : fit < 256 ? 256 : fit;
}
size_t part_bytes(int splits, long long rows, int cols) {
  if (splits == 1) return 0;
  const long long at_once = part_rows(splits, rows, cols);
  return (size_t)splits * (at_once < rows ? at_once : rows) * pitch4(cols) * 4;
}

// Rows m0 .. m0 + rows of a split product, into `part`.
template <typename T>
int run_partials(const Gemm& g, long long m0, long long rows, float* part, cudaStream_t st) {
  Gemm sub = g;
  const uint8_t* a = static_cast<const uint8_t*>(g.a.ptr);
  if (g.a_mn) {
    sub.a.ptr = a + m0 * sizeof(T);
    sub.a.cols = (int)rows;
  } else {
    sub.a.ptr = a + m0 * g.a.pitch * sizeof(T);
    sub.a.rows = rows;
  }
  sub.M = rows;
  sub.out = part;
  sub.ld_out = pitch4(g.N);
  sub.bias = sub.in = nullptr;
  sub.colsum = nullptr;
  return run_gemm<T, kPartial>(sub, st);
}

// A product with an epilogue, over `part` (FP32 partials) where it is split.
template <typename T, Epi kEpi>
int run_product(const Gemm& g, float* part, cudaStream_t st) {
  if constexpr (sizeof(T) == 2) {  // FP32 data needs no splits here
    if (g.splits > 1) {
      const long long step = part_rows(g.splits, g.M, g.N);
      for (long long m0 = 0; m0 < g.M; m0 += step) {
        Finish f{};
        f.part = part;
        f.M = g.M - m0 < step ? g.M - m0 : step;
        f.pitch = pitch4(g.N);
        f.splits = g.splits;
        f.N = g.N;
        f.tiles_n = (g.N + 255) / 256;
        f.act = g.act;
        f.bias = g.bias;
        f.in = g.in ? static_cast<const T*>(g.in) + m0 * g.N : nullptr;
        f.out = static_cast<T*>(g.out) + m0 * g.ld_out;
        f.ld_out = g.ld_out;
        f.colsum = g.colsum ? g.colsum + m0 / 32 * g.N : nullptr;  // m0: a multiple of 256
        const int rc = run_partials<T>(g, m0, f.M, part, st);
        if (rc) return rc;
        const long long blocks = (f.M + 31) / 32 * f.tiles_n;
        linear_finish_kernel<T, kEpi><<<(unsigned)blocks, 256, 0, st>>>(f);
        DDPM_CHECK_LAUNCH("linear_finish_kernel");
      }
      return DDPM_OK;
    }
  }
  return run_gemm<T, kEpi>(g, st);
}

// What a call has to lay out in its workspace.
struct LinearPlan {
  bool rows_path;            // the dot-product kernel
  bool stage_x, stage_w, stage_dz;
  int parts, splits_z, splits_x, splits_w;
  Tile tile_z, tile_x, tile_w;
  long long colsum_rows, colsum_chunk;
  size_t x_off, w_off, dz_off, dzp_off, colsum_off, part_off, total;
};

struct LinearShape {
  long long m;
  int n, k;
  long long ldx;
  int act, dt;
  bool aligned;  // every pointer on a 16-byte boundary
};

LinearPlan plan_linear(const LinearShape& s, bool bwd) {
  LinearPlan q{};
  const int es = dtype_size(s.dt);
  const bool f32 = s.dt == DDPM_F32;
  q.parts = f32 ? 3 : 1;
  q.rows_path = !bwd && s.m <= kGemvRows;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t o = at;
    at += up256(bytes);
    return o;
  };
  if (!q.rows_path) {
    const int whole = 16 / es;  // values of a 16-byte word
    q.stage_x = !s.aligned || s.ldx % whole;
    q.stage_w = !s.aligned || s.k % whole;
    q.x_off = q.stage_x ? take(staged_bytes(s.m, s.k, es)) : 0;
    q.w_off = q.stage_w ? take(staged_bytes(s.n, s.k, es)) : 0;
  }
  // splits that a sum over k values needs
  auto chains = [&](long long k) { return f32 ? 1 : (int)((k + kChain - 1) / kChain); };
  q.splits_z = chains(s.k);
  q.tile_z = pick_tile(s.m, s.n, s.k, q.parts, q.splits_z);
  size_t part = 0;  // the products use the partials' memory one after the other
  auto partials = [&](int splits, long long rows, int cols) {
    const size_t bytes = part_bytes(splits, rows, cols);
    if (bytes > part) part = bytes;
  };
  if (!q.rows_path && (!bwd || s.act != DDPM_ACT_NONE)) partials(q.splits_z, s.m, s.n);
  if (bwd) {
    const bool recompute = s.act != DDPM_ACT_NONE;
    // dz: recomputed, or dy, copied where TMA cannot address it
    if (recompute) q.dz_off = take((size_t)s.m * round8(s.n) * es);
    q.stage_dz = !recompute && (!s.aligned || s.n % (16 / es));
    q.dzp_off = q.stage_dz ? take(staged_bytes(s.m, s.n, es)) : 0;
    q.splits_x = chains(s.n);
    q.tile_x = pick_tile(s.m, s.k, s.n, q.parts, q.splits_x);
    partials(q.splits_x, s.m, s.k);
    if (recompute) {
      q.colsum_rows = (s.m + 31) / 32;  // a row of sums for every 32 rows
    } else {
      // rows of a chunk: enough chunks to fill the SMs, at least 64 rows each
      const long long cols = (s.n + 31) / 32;
      long long want = (long long)gencat::num_sms() * 8 / cols;
      want = want < 1 ? 1 : want;
      q.colsum_chunk = (s.m + want - 1) / want;
      if (q.colsum_chunk < 64) q.colsum_chunk = 64;
      q.colsum_rows = (s.m + q.colsum_chunk - 1) / q.colsum_chunk;
    }
    q.colsum_off = take((size_t)q.colsum_rows * s.n * 4);
    // dweight: the rows are split over the SMs that have no tile, at least four
    // K blocks a split (with two, four and eight of them: 4096 rows 256 x 256 bf16
    // 12.1, 11.3 and 12.1 us, 1024 rows 64 x 64 6.8, 7.7 and 9.6, 4096 rows
    // 256 x 256 FP32 16.9, 15.6 and 18.3)
    const int bk = block_k(q.parts);
    const long long kb = (s.m + bk - 1) / bk;
    q.tile_w = pick_tile(s.n, s.k, s.m, q.parts, 1);
    q.splits_w = 1;
    {
      const int bn = f32 || s.k <= 128 ? (s.k > 64 ? 128 : 64) : 256;
      const long long tiles = (long long)((s.n + kBM - 1) / kBM) * ((s.k + bn - 1) / bn);
      long long splits = gencat::num_sms() / tiles;
      if (splits > kb / 4) splits = kb / 4;
      const int need = chains(s.m);
      if (splits > 1) {
        // whole rounds of the SMs where the sum needs more splits
        q.splits_w = (int)((need + splits - 1) / splits * splits);
        q.tile_w = Tile{bn, 1, 8};
      } else if (need > 1) {
        q.splits_w = need;
        q.tile_w = pick_tile(s.n, s.k, s.m, q.parts, need);
      }
    }
    partials(q.splits_w, s.n, s.k);
  }
  if (part > 0) q.part_off = take(part);
  q.total = at;
  return q;
}

template <typename T>
int rows_forward(const void* x, long long ldx, const void* w, const void* bias, const void* res,
                 void* out, int m, int n, int k, int act, bool aligned, cudaStream_t st) {
  constexpr int kVec = 16 / (int)sizeof(T);
  const int grid = (n + 7) / 8;
  const bool vec = aligned && k % kVec == 0 && (m == 1 || ldx % kVec == 0);
  auto go = [&](auto fn) {
    fn<<<grid, 256, 0, st>>>(static_cast<const T*>(x), ldx, static_cast<const T*>(w),
                             static_cast<const T*>(bias), static_cast<const T*>(res),
                             static_cast<T*>(out), m, n, k, act);
  };
  if (vec) {
    if (m == 1) go(linear_rows_kernel<T, kVec, 1>);
    else if (m <= 4) go(linear_rows_kernel<T, kVec, 4>);
    else go(linear_rows_kernel<T, kVec, kGemvRows>);
  } else {
    if (m == 1) go(linear_rows_kernel<T, 1, 1>);
    else go(linear_rows_kernel<T, 1, kGemvRows>);
  }
  DDPM_CHECK_LAUNCH("linear_rows_kernel");
  return DDPM_OK;
}

int check_linear(long long m, int n, int k, long long ldx, int act, int dt) {
  DDPM_CHECK_ARG(m >= 0 && n >= 1 && k >= 1, "rows must not be negative, widths positive");
  DDPM_CHECK_ARG(ldx >= k, "row stride %lld of x is below its %d columns", ldx, k);
  DDPM_CHECK_ARG(act_known(act), "unknown activation code %d", act);
  DDPM_CHECK_ARG(dtype_size(dt) > 0, "unknown dtype code %d", dt);
  // row and column indices of tiles, and the tiles of a split, are 32-bit
  const double tiles = ((double)m / kBM + 1) * ((double)(n > k ? n : k) / 64 + 1);
  if (m >= (1LL << 31) - 256 || n >= (1 << 30) || k >= (1 << 30) || tiles >= 2e9 ||
      (double)ldx * 4 >= 1e12)
    return set_error(DDPM_ERR_UNSUPPORTED, "linear: sizes out of range");
  return DDPM_OK;
}

template <typename T>
int forward(const LinearShape& s, const LinearPlan& q, const void* x, const void* w,
            const void* bias, const void* res, void* out, uint8_t* ws, cudaStream_t st) {
  if (q.rows_path)
    return rows_forward<T>(x, s.ldx, w, bias, res, out, (int)s.m, s.n, s.k, s.act, s.aligned, st);
  int rc;
  if (q.stage_x && (rc = stage<T>(x, s.ldx, s.m, s.k, ws + q.x_off, st))) return rc;
  if (q.stage_w && (rc = stage<T>(w, s.k, s.n, s.k, ws + q.w_off, st))) return rc;
  Gemm g{};
  g.a = q.stage_x ? Operand{ws + q.x_off, s.m, s.k, round8(s.k)}
                  : Operand{x, s.m, s.k, s.ldx};
  g.b = q.stage_w ? Operand{ws + q.w_off, s.n, s.k, round8(s.k)}
                  : Operand{w, s.n, s.k, s.k};
  g.M = s.m;
  g.N = s.n;
  g.K = s.k;
  g.bias = bias;
  g.in = res;
  g.ld_in = s.n;
  g.out = out;
  g.ld_out = s.n;
  g.act = s.act;
  g.splits = q.splits_z;
  g.tile = q.tile_z;
  return run_product<T, kOut>(g, reinterpret_cast<float*>(ws + q.part_off), st);
}

template <typename T>
int backward(const LinearShape& s, const LinearPlan& q, const void* x, const void* w,
             const void* bias, const void* dy, void* gx, void* gw, void* gb, uint8_t* ws,
             cudaStream_t st) {
  int rc;
  const bool recompute = s.act != DDPM_ACT_NONE;
  if (q.stage_x && (recompute || gw) && (rc = stage<T>(x, s.ldx, s.m, s.k, ws + q.x_off, st)))
    return rc;
  if (q.stage_w && (recompute || gx) && (rc = stage<T>(w, s.k, s.n, s.k, ws + q.w_off, st)))
    return rc;
  const Operand xo = q.stage_x ? Operand{ws + q.x_off, s.m, s.k, round8(s.k)}
                               : Operand{x, s.m, s.k, s.ldx};
  const Operand wo = q.stage_w ? Operand{ws + q.w_off, s.n, s.k, round8(s.k)}
                               : Operand{w, s.n, s.k, s.k};
  float* colsum = reinterpret_cast<float*>(ws + q.colsum_off);
  float* part = reinterpret_cast<float*>(ws + q.part_off);
  const void* dz = dy;
  long long ld_dz = s.n;
  if (recompute) {
    Gemm g{};
    g.a = xo;
    g.b = wo;
    g.M = s.m;
    g.N = s.n;
    g.K = s.k;
    g.bias = bias;
    g.in = dy;
    g.ld_in = s.n;
    g.out = ws + q.dz_off;
    g.ld_out = round8(s.n);
    g.act = s.act;
    g.colsum = gb ? colsum : nullptr;
    g.splits = q.splits_z;
    g.tile = q.tile_z;
    if ((rc = run_product<T, kDz>(g, part, st))) return rc;
    dz = g.out;
    ld_dz = g.ld_out;
  } else if (gb) {
    const dim3 grid((unsigned)((s.n + 31) / 32), (unsigned)q.colsum_rows);
    linear_colsum_kernel<T><<<grid, 256, 0, st>>>(static_cast<const T*>(dy), s.m, s.n,
                                                  q.colsum_chunk, colsum);
    DDPM_CHECK_LAUNCH("linear_colsum_kernel");
  }
  Operand zo = Operand{dz, s.m, s.n, ld_dz};
  if (q.stage_dz && (gx || gw)) {
    if ((rc = stage<T>(dz, ld_dz, s.m, s.n, ws + q.dzp_off, st))) return rc;
    zo = Operand{ws + q.dzp_off, s.m, s.n, round8(s.n)};
  }
  if (gx) {
    Gemm g{};
    g.a = zo;
    g.b = wo;
    g.b_mn = true;
    g.M = s.m;
    g.N = s.k;
    g.K = s.n;
    g.out = gx;
    g.ld_out = s.k;
    g.splits = q.splits_x;
    g.tile = q.tile_x;
    if ((rc = run_product<T, kOut>(g, part, st))) return rc;
  }
  bool fold_w = gw && q.splits_w > 1;
  if (gw) {
    Gemm g{};
    g.a = zo;
    g.b = xo;
    g.a_mn = g.b_mn = true;
    g.M = s.n;
    g.N = s.k;
    g.K = s.m;
    g.splits = q.splits_w;
    g.tile = q.tile_w;
    const long long step = part_rows(q.splits_w, s.n, s.k);
    if (q.splits_w > 1 && step < s.n) {  // partials in several parts, each added up at once
      for (long long m0 = 0; m0 < s.n; m0 += step) {
        const long long rows = s.n - m0 < step ? s.n - m0 : step;
        if ((rc = run_partials<T>(g, m0, rows, part, st))) return rc;
        const Fold f{part, rows, pitch4(s.k), q.splits_w, s.k, 0,
                     static_cast<T*>(gw) + m0 * s.k};
        linear_fold_kernel<T><<<small_grid(f.rows * f.cols), 256, 0, st>>>(f);
        DDPM_CHECK_LAUNCH("linear_fold_kernel");
      }
      fold_w = false;
    } else if (q.splits_w > 1) {
      if ((rc = run_partials<T>(g, 0, s.n, part, st))) return rc;
    } else {
      g.out = gw;
      g.ld_out = s.k;
      if ((rc = run_gemm<T, kOut>(g, st))) return rc;
    }
  }
  // the sums over partials: of the bias, and of the weight where it was split
  auto blocks = [](const Fold& f) { return (int)((f.rows * f.cols + 31) / 32); };
  Fold fb{}, fw{};
  if (gb) {
    fb = Fold{colsum, 1, s.n, (int)q.colsum_rows, s.n, 0, gb};
    fb.blocks = blocks(fb);
  }
  if (fold_w) {
    fw = Fold{part, s.n, pitch4(s.k), q.splits_w, s.k, 0, gw};
    // 4096 values: 64 partials 8.5 us by warps that share them, 12.7 a thread a value;
    // 16384: 12.4 and 14.2; 65536: 22.2 and 15.8 (the whole gradient). Equal at about
    // 600 values a partial (32 partials of 16384: 11.7 both).
    if (fw.rows * fw.cols > 512LL * q.splits_w) {
      linear_fold_kernel<T><<<small_grid(fw.rows * fw.cols), 256, 0, st>>>(fw);
      DDPM_CHECK_LAUNCH("linear_fold_kernel");
    } else {
      fw.blocks = blocks(fw);
    }
  }
  if (fb.blocks + fw.blocks > 0) {
    linear_fold_long_kernel<T><<<fb.blocks + fw.blocks, 1024, 0, st>>>(fb, fw);
    DDPM_CHECK_LAUNCH("linear_fold_kernel");
  }
  return DDPM_OK;
}

int check_ws(const LinearPlan& q, const void* ws, size_t ws_bytes) {
  DDPM_CHECK_ARG((uintptr_t)ws % 256 == 0, "misaligned workspace");
  if (ws_bytes < q.total || (q.total > 0 && ws == nullptr))
    return set_error(DDPM_ERR_WORKSPACE, "linear workspace: %zu bytes needed, %zu given", q.total,
                     ws_bytes);
  return DDPM_OK;
}

}  // namespace

size_t linear_workspace_bytes(long long m, int n, int k, long long ldx, int act, int dt, int bwd,
                              int aligned) {
  const int rc = check_linear(m, n, k, ldx, act, dt);
  if (rc || m == 0) return 0;
  return plan_linear(LinearShape{m, n, k, ldx, act, dt, aligned != 0}, bwd != 0).total;
}

// For the tests: how a product runs (0 forward or dz, 1 dx, 2 dweight).
int linear_choice(long long m, int n, int k, int act, int dt, int product, int* out) {
  const int rc = check_linear(m, n, k, k, act, dt);
  if (rc) return rc;
  DDPM_CHECK_ARG(m >= 1 && product >= 0 && product <= 2 && out, "unknown product");
  const LinearPlan q = plan_linear(LinearShape{m, n, k, k, act, dt, true}, true);
  const Tile t = product == 0 ? q.tile_z : product == 1 ? q.tile_x : q.tile_w;
  const int splits = product == 0 ? q.splits_z : product == 1 ? q.splits_x : q.splits_w;
  const long long terms = product == 0 ? k : product == 1 ? n : m;
  const int bk = block_k(q.parts);
  const Rings r = pick_rings(t, q.parts, splits > 1 ? 4 : dtype_size(dt), (terms + bk - 1) / bk,
                             splits);
  const int got[6] = {t.bn, t.cg, t.ew, splits, r.stages, r.smem <= smem_limit()};
  for (int i = 0; i < 6; ++i) out[i] = got[i];
  return DDPM_OK;
}

int linear_fwd(const void* x, long long ldx, const void* w, const void* bias, const void* res,
               void* out, void* ws, size_t ws_bytes, long long m, int n, int k, int act, int dt,
               cudaStream_t st) {
  int rc = check_linear(m, n, k, ldx, act, dt);
  if (rc) return rc;
  if (m == 0) return DDPM_OK;
  DDPM_CHECK_ARG(x && w && out, "null pointer");
  const uintptr_t at = (uintptr_t)x | (uintptr_t)w | (uintptr_t)bias | (uintptr_t)res |
                       (uintptr_t)out;
  DDPM_CHECK_ARG(at % dtype_size(dt) == 0, "misaligned pointer");
  const LinearShape s{m, n, k, ldx, act, dt, at % 16 == 0};
  const LinearPlan q = plan_linear(s, false);
  rc = check_ws(q, ws, ws_bytes);
  if (rc) return rc;
  uint8_t* base = static_cast<uint8_t*>(ws);
  switch (dt) {
    case DDPM_F32: return forward<float>(s, q, x, w, bias, res, out, base, st);
    case DDPM_BF16: return forward<__nv_bfloat16>(s, q, x, w, bias, res, out, base, st);
    default: return forward<__half>(s, q, x, w, bias, res, out, base, st);
  }
}

int linear_bwd(const void* x, long long ldx, const void* w, const void* bias, const void* dy,
               void* gx, void* gw, void* gb, void* ws, size_t ws_bytes, long long m, int n, int k,
               int act, int dt, cudaStream_t st) {
  int rc = check_linear(m, n, k, ldx, act, dt);
  if (rc) return rc;
  if (m == 0) return DDPM_OK;
  DDPM_CHECK_ARG(x && w && dy, "null pointer");
  const uintptr_t at = (uintptr_t)x | (uintptr_t)w | (uintptr_t)bias | (uintptr_t)dy |
                       (uintptr_t)gx | (uintptr_t)gw | (uintptr_t)gb;
  DDPM_CHECK_ARG(at % dtype_size(dt) == 0, "misaligned pointer");
  const LinearShape s{m, n, k, ldx, act, dt, at % 16 == 0};
  const LinearPlan q = plan_linear(s, true);
  rc = check_ws(q, ws, ws_bytes);
  if (rc) return rc;
  uint8_t* base = static_cast<uint8_t*>(ws);
  switch (dt) {
    case DDPM_F32: return backward<float>(s, q, x, w, bias, dy, gx, gw, gb, base, st);
    case DDPM_BF16: return backward<__nv_bfloat16>(s, q, x, w, bias, dy, gx, gw, gb, base, st);
    default: return backward<__half>(s, q, x, w, bias, dy, gx, gw, gb, base, st);
  }
}

}  // namespace ddpm
