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
//   tile      128 rows x BN (64, 128 or 256) columns, K in steps of 64
//   operands  TMA, 128-byte swizzle, a ring of stages; out-of-range rows,
//             columns and k are zero filled, which covers every ragged size
//   issue     tcgen05.mma of 128 x BN x 16 by one thread; two TMEM
//             accumulators, so the epilogue of a tile overlaps the next one
//   epilogue  eight warps (lane = row, two column halves): TMEM -> registers,
//             bias, activation, residual -> 64-byte x 32-row boxes in shared
//             memory -> TMA store. The residual (or dy) comes through the same
//             boxes by TMA, several boxes ahead.
//
// The backward keeps x and weight only: z is computed again by the same
// product (kDz), whose epilogue turns it into dz at once. Saving z instead
// would cost m * n values of traffic twice and, rounded to 16 bits, a second
// rounding in dz. dz is rounded to the data's type, as an operand of the
// tensor cores has to be; the bias gradient sums it before that rounding.
//
// FP32 data: every operand is split once into three bf16 parts that hold its
// 24 bits, x = x0 + x1 + x2, and a K step issues the six products whose size is
// above 2^-24 of x0 y0. Exponents stay in range (bf16 has FP32's). Each K block
// has an accumulator of its own, and the epilogue's registers add the blocks: a
// chain of 384 tensor-core additions (k = 1024) left a 2-norm error of 4.9e-6.
//
// dweight sums over all rows: its K axis is split over the SMs left without a
// tile, FP32 partials are added in a fixed order.
//
// Up to eight rows, forward: a dot-product kernel reads the weight once at the
// memory's rate; a tensor-core tile would be 15/16 empty and its K loop serial.
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

constexpr int kBM = 128, kBK = 64;
constexpr int kEpiWarps = 8;
constexpr int kFirstEpi = 4;  // warps 0-3: TMA, MMA, TMEM allocation, none
constexpr int kThreads = 32 * (kFirstEpi + kEpiWarps);
constexpr int kBoxBytes = 2048;  // 32 rows x 64 bytes
constexpr int kMaxStages = 8, kMaxBufs = 8;
constexpr uint64_t kWaitNs = 2000000000ull;
constexpr int kGemvRows = 8;

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

struct SmemLayout {
  uint32_t stage, ring, boxes, total;
};
__host__ __device__ inline SmemLayout smem_layout(int parts, int bn, int stages, int nbuf) {
  SmemLayout L;
  L.stage = (uint32_t)parts * (kBM + bn) * kBK * 2;
  L.ring = 0;
  L.boxes = L.stage * stages;
  L.total = L.boxes + kEpiWarps * nbuf * kBoxBytes + 1024;  // + alignment of the base
  return L;
}

__device__ __forceinline__ void give_up(volatile int* abort_flag, int* status, int code) {
  *abort_flag = 1;
  atomicCAS(status, 0, code);
}

// Sums over the warp's rows: lane l (mod C) returns the sum of v[l] over the
// 32 lanes. Halves the columns a lane holds at each exchange.
template <int C> __device__ __forceinline__ float column_sums(float (&v)[C], int lane) {
  if constexpr (C == 16) {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], 16);
  }
#pragma unroll
  for (int off = C / 2; off > 0; off >>= 1) {
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
// FP32 data split into bf16 parts.
template <typename T, int BN, int PARTS, Epi kEpi>
__global__ void __launch_bounds__(kThreads, 1)
linear_gemm_kernel(const __grid_constant__ GemmParams p) {
  using To = typename std::conditional<kEpi == kPartial, float, T>::type;
  constexpr bool kFast = sizeof(T) == 2;
  constexpr int kCB = 64 / (int)sizeof(To);  // columns of a box
  constexpr int kHalf = BN / 2;
  constexpr int kBoxes = kHalf / kCB;        // boxes of a warp's part of a tile
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full[kMaxStages], empty[kMaxStages], acc_full[2], acc_empty[2];
  __shared__ uint64_t in_full[kEpiWarps][kMaxBufs], drained;
  __shared__ uint32_t tmem_base_s;
  __shared__ int abort_s;
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const SmemLayout L = smem_layout(PARTS, BN, p.stages, p.nbuf);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort_flag = &abort_s;

  if (threadIdx.x == 0) {
    for (int i = 0; i < p.stages; ++i) {
      tc::mbar_init(&full[i], 1);
      tc::mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&acc_full[i], 1);
      tc::mbar_init(&acc_empty[i], kEpiWarps);
    }
    for (int w = 0; w < kEpiWarps; ++w)
      for (int i = 0; i < p.nbuf; ++i) tc::mbar_init(&in_full[w][i], 1);
    tc::mbar_init(&drained, 1);
    abort_s = 0;
    tc::fence_mbar_init();
  }
  if (warp == 2) {
    tc::tmem_alloc(&tmem_base_s, 2 * BN);
    tc::tmem_relinquish();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = tmem_base_s;

  constexpr uint32_t kPartA = kBM * kBK * 2, kPartB = BN * kBK * 2;  // bytes of one part
  if (warp == 0) {
    if (lane == 0) {  // ---- operand copies ----
      uint32_t it = 0;
      bool ok = true;
      for (int t = blockIdx.x; t < p.num_tiles && ok; t += gridDim.x) {
        int tm, tn, sp;
        tile_at(p, t, tm, tn, sp);
        const int kb0 = (int)((long long)p.kblocks * sp / p.splits);
        const int kb1 = (int)((long long)p.kblocks * (sp + 1) / p.splits);
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          const int s = it % p.stages;
          if (!tc::mbar_wait(&empty[s], ((it / p.stages) & 1) ^ 1, abort_flag, kWaitNs)) {
            give_up(abort_flag, p.status, 91);
            ok = false;
            break;
          }
          uint8_t* a = smem + s * L.stage;
          uint8_t* b = a + PARTS * kPartA;
          tc::mbar_arrive_expect_tx(&full[s], L.stage);
          // K-major: one box of [parts][rows][64 k]; MN-major: a box of
          // [parts][64 k][64 rows] for every 64 rows
          if (!p.a_mn) {
            tc::tma_load_3d(a, &p.a, kb * kBK, tm * kBM, 0, &full[s]);
          } else {
#pragma unroll
            for (int j = 0; j < kBM / 64; ++j)
              tc::tma_load_3d(a + j * PARTS * 8192, &p.a, tm * kBM + j * 64, kb * kBK, 0, &full[s]);
          }
          if (!p.b_mn) {
            tc::tma_load_3d(b, &p.b, kb * kBK, tn * BN, 0, &full[s]);
          } else {
#pragma unroll
            for (int j = 0; j < BN / 64; ++j)
              tc::tma_load_3d(b + j * PARTS * 8192, &p.b, tn * BN + j * 64, kb * kBK, 0, &full[s]);
          }
        }
      }
      // Copies still in flight have to land before the block's shared memory goes.
      if (!ok || *abort_flag) {
        const uint32_t n = it < (uint32_t)p.stages ? it : (uint32_t)p.stages;
        for (uint32_t j = it - n; j < it; ++j)
          tc::mbar_wait(&full[j % p.stages], (j / p.stages) & 1, nullptr, kWaitNs);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {  // ---- products ----
      uint32_t it = 0, ti = 0;  // K blocks, accumulators
      bool ok = true;
      for (int t = blockIdx.x; t < p.num_tiles && ok; t += gridDim.x) {
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
            if (!tc::mbar_wait(&acc_empty[ti & 1], ((ti >> 1) & 1) ^ 1, abort_flag, kWaitNs)) {
              give_up(abort_flag, p.status, 92);
              ok = false;
              break;
            }
            tc::tc_fence_after();
          }
          const uint32_t d = tmem + (ti & 1) * BN;
          const int s = it % p.stages;
          if (!tc::mbar_wait(&full[s], (it / p.stages) & 1, abort_flag, kWaitNs)) {
            give_up(abort_flag, p.status, 93);
            ok = false;
            break;
          }
          tc::tc_fence_after();
          const uint32_t sa = tc::smem_u32(smem + s * L.stage);
          const uint32_t sb = sa + PARTS * kPartA;
          const uint64_t ad = p.a_mn ? tc::smem_desc_sw128_mn(sa, PARTS * 8192)
                                     : tc::smem_desc_sw128(sa);
          const uint64_t bd = p.b_mn ? tc::smem_desc_sw128_mn(sb, PARTS * 8192)
                                     : tc::smem_desc_sw128(sb);
          // descriptor units are 16 bytes
          const uint32_t ak = (p.a_mn ? 2048 : 32) >> 4, bk = (p.b_mn ? 2048 : 32) >> 4;
          const int ksteps = kb == p.kblocks - 1 ? p.last_ksteps : kBK / 16;
          if constexpr (PARTS == 1) {
            for (int ks = 0; ks < ksteps; ++ks)
              tc::mma_f16(d, ad + ks * ak, bd + ks * bk, p.idesc, (!first || ks > 0) ? 1u : 0u);
            tc::mma_commit(&empty[s]);
          } else {
            const uint32_t ap = (p.a_mn ? 8192u : kPartA) >> 4, bp = (p.b_mn ? 8192u : kPartB) >> 4;
            // the small products first, while the sum is small
            for (int ks = 0; ks < ksteps; ++ks) {
              const uint64_t a0 = ad + ks * ak, b0 = bd + ks * bk;
              tc::mma_f16(d, a0 + 2 * ap, b0, p.idesc, ks > 0 ? 1u : 0u);
              tc::mma_f16(d, a0, b0 + 2 * bp, p.idesc, 1u);
              tc::mma_f16(d, a0 + ap, b0 + bp, p.idesc, 1u);
              tc::mma_f16(d, a0 + ap, b0, p.idesc, 1u);
              tc::mma_f16(d, a0, b0 + bp, p.idesc, 1u);
            }
            for (int ks = 0; ks < ksteps; ++ks)
              tc::mma_f16(d, ad + ks * ak, bd + ks * bk, p.idesc, 1u);
            tc::mma_commit(&empty[s]);
            tc::mma_commit(&acc_full[ti & 1]);
            ++ti;
          }
        }
        if (PARTS == 1 && ok) {
          tc::mma_commit(&acc_full[ti & 1]);
          ++ti;
        }
      }
      // every product issued has completed before the tensor memory is freed
      tc::mma_commit(&drained);
      tc::mbar_wait(&drained, 0, nullptr, kWaitNs);
    }
    __syncwarp();
  } else if (warp >= kFirstEpi) {  // ---- epilogue ----
    const int ew = warp - kFirstEpi;
    const int quad = warp & 3, half = ew >> 2;
    uint8_t* boxes = smem + L.boxes + ew * p.nbuf * kBoxBytes;
    const To* in = static_cast<const To*>(p.in_ptr);
    const T* bias = static_cast<const T*>(p.bias);
    To* out = static_cast<To*>(p.out_ptr);
    const bool has_in = kEpi != kPartial && p.in_ptr != nullptr;
    const int ahead = has_in ? p.nbuf / 2 : 0;  // boxes loaded ahead
    // the block's own chunk c (16 bytes) of row r: chunk c ^ (r / 2) % 4
    const uint32_t sw = (lane >> 1) & 3;
    uint32_t ti = 0, q = 0;
    // the load cursor: box `lj` of tile `lt`
    int lt = blockIdx.x, lj = 0;
    uint32_t lq = 0;
    auto load_next = [&]() {  // lane 0
      if (lt >= p.num_tiles) return;
      int tm, tn, sp;
      tile_at(p, lt, tm, tn, sp);
      const int c = tn * BN + half * kHalf + lj * kCB, r = tm * kBM + quad * 32;
      const int b = lq % p.nbuf;
      if (c < p.N && r < p.M) {
        tc::mbar_arrive_expect_tx(&in_full[ew][b], kBoxBytes);
        tc::tma_load_3d(boxes + b * kBoxBytes, &p.in, c, r, 0, &in_full[ew][b]);
      } else {
        tc::mbar_arrive(&in_full[ew][b]);
      }
      ++lq;
      if (++lj == kBoxes) {
        lj = 0;
        lt += gridDim.x;
      }
    };
    if (p.tma_io && has_in && lane == 0)
      for (int i = 0; i < ahead; ++i) load_next();
    bool ok = true;
    for (int t = blockIdx.x; t < p.num_tiles && ok; t += gridDim.x) {
      int tm, tn, sp;
      tile_at(p, t, tm, tn, sp);
      const int row0 = tm * kBM + quad * 32;
      const int row = row0 + lane;
      const uint32_t tcol = tmem + ((uint32_t)(quad * 32) << 16) + half * kHalf;
      float sum[PARTS == 3 ? kHalf : 1];  // FP32 data: the K blocks added up
      if constexpr (PARTS == 3) {
        const int kb0 = (int)((long long)p.kblocks * sp / p.splits);
        const int kb1 = (int)((long long)p.kblocks * (sp + 1) / p.splits);
#pragma unroll
        for (int i = 0; i < kHalf; ++i) sum[i] = 0.f;
        for (int kb = kb0; kb < kb1; ++kb, ++ti) {
          ok = __all_sync(0xffffffffu, tc::mbar_wait(&acc_full[ti & 1], (ti >> 1) & 1, abort_flag,
                                                     kWaitNs));
          if (!ok) break;
          tc::tc_fence_after();
#pragma unroll
          for (int i = 0; i < kHalf; i += 32) {
            float v[32];
            tc::tmem_ld16(tcol + (ti & 1) * BN + i, *reinterpret_cast<float(*)[16]>(v));
            tc::tmem_ld16(tcol + (ti & 1) * BN + i + 16, *reinterpret_cast<float(*)[16]>(v + 16));
            tc::tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e) sum[i + e] += v[e];
          }
          tc::tc_fence_before();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(&acc_empty[ti & 1]);
        }
      } else {
        ok = __all_sync(0xffffffffu, tc::mbar_wait(&acc_full[ti & 1], (ti >> 1) & 1, abort_flag,
                                                   kWaitNs));
        tc::tc_fence_after();
      }
      if (!ok) {
        if (lane == 0) give_up(abort_flag, p.status, 94);
        break;
      }
      const uint32_t taddr = tcol + (ti & 1) * BN;
#pragma unroll (PARTS == 3 ? kBoxes : 1)
      for (int j = 0; j < kBoxes; ++j, ++q) {
        const int c0 = tn * BN + half * kHalf + j * kCB;
        const int b = q % p.nbuf;
        uint8_t* box = boxes + b * kBoxBytes;
        float v[kCB];
        if constexpr (PARTS == 3) {
#pragma unroll
          for (int i = 0; i < kCB; ++i) v[i] = sum[j * kCB + i];
        } else {
#pragma unroll
          for (int i = 0; i < kCB; i += 16)
            tc::tmem_ld16(taddr + j * kCB + i, *reinterpret_cast<float(*)[16]>(v + i));
        }
        // make room, and fetch a later box of the residual
        if (p.tma_io) {
          if (lane == 0) {
            const int pending = has_in ? p.nbuf - ahead - 1 : p.nbuf - 1;
            if (pending >= 7) tc::bulk_wait_read<7>();
            else if (pending >= 3) tc::bulk_wait_read<3>();
            else if (pending >= 1) tc::bulk_wait_read<1>();
            else tc::bulk_wait_read<0>();
            if (has_in) load_next();
          }
          __syncwarp();
        }
        if constexpr (PARTS == 1) tc::tmem_ld_wait();
        const bool live = c0 < p.N && row0 < p.M;  // the box holds anything
        if constexpr (kEpi != kPartial) {
          if (bias != nullptr && live) {
#pragma unroll
            for (int i = 0; i < kCB; ++i) {
              const int c = c0 + i < p.N ? c0 + i : p.N - 1;
              v[i] += ldg_f32<T>(bias + c);
            }
          }
          if constexpr (kEpi == kOut) act_values<kFast, kCB>(p.act, v);
          else act_slopes<kFast, kCB>(p.act, v);
        }
        if (has_in) {
          if (p.tma_io) {
            ok = __all_sync(0xffffffffu, tc::mbar_wait(&in_full[ew][b], (q / p.nbuf) & 1,
                                                       abort_flag, kWaitNs));
            if (!ok) {
              if (lane == 0) give_up(abort_flag, p.status, 95);
              break;
            }
          } else if (live) {
            // rows one after the other, a lane per column
            if (lane < kCB && c0 + lane < p.N) {
#pragma unroll 8
              for (int r = 0; r < 32; ++r) {
                if (row0 + r < p.M) {
                  const uint32_t at = r * 64 + (((lane * sizeof(To) / 16) ^ ((r >> 1) & 3)) * 16) +
                                      lane * sizeof(To) % 16;
                  *reinterpret_cast<To*>(box + at) = in[(long long)(row0 + r) * p.ld_in + c0 + lane];
                }
              }
            }
            __syncwarp();
          }
        }
        if (live) {
          union Chunk { uint4 u; To e[16 / sizeof(To)]; };
          constexpr int kPer = 16 / (int)sizeof(To);
          if constexpr (kEpi == kDz) {
            float s[kCB];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              Chunk ch;
              ch.u = *reinterpret_cast<const uint4*>(box + lane * 64 + ((k ^ sw) * 16));
#pragma unroll
              for (int i = 0; i < kPer; ++i) {
                const float dz = to_f32<To>(ch.e[i]) * v[k * kPer + i];
                ch.e[i] = from_f32<To>(dz);
                s[k * kPer + i] = row < p.M ? dz : 0.f;
              }
              *reinterpret_cast<uint4*>(box + lane * 64 + ((k ^ sw) * 16)) = ch.u;
            }
            if (p.colsum != nullptr) {
              const float total = column_sums<kCB>(s, lane);
              if (lane < kCB && c0 + lane < p.N)
                p.colsum[(long long)(tm * 4 + quad) * p.N + c0 + lane] = total;
            }
          } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              Chunk ch;
              uint4* at = reinterpret_cast<uint4*>(box + lane * 64 + ((k ^ sw) * 16));
              if (has_in) ch.u = *at;
#pragma unroll
              for (int i = 0; i < kPer; ++i) {
                float y = v[k * kPer + i];
                if (has_in) y += to_f32<To>(ch.e[i]);
                ch.e[i] = from_f32<To>(y);
              }
              *at = ch.u;
            }
          }
          if (p.tma_io) {
            tc::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              tc::tma_store_3d(&p.out, box, c0, row0, sp);
            }
          } else {
            __syncwarp();
            if (lane < kCB && c0 + lane < p.N) {
#pragma unroll 8
              for (int r = 0; r < 32; ++r) {
                if (row0 + r < p.M) {
                  const uint32_t at = r * 64 + (((lane * sizeof(To) / 16) ^ ((r >> 1) & 3)) * 16) +
                                      lane * sizeof(To) % 16;
                  out[(long long)(row0 + r) * p.ld_out + c0 + lane] =
                      *reinterpret_cast<const To*>(box + at);
                }
              }
            }
            __syncwarp();
          }
        }
        // a group for every box, written or not, so that counting groups
        // counts boxes
        if (p.tma_io && lane == 0) tc::bulk_commit();
      }
      if (!ok) break;
      if constexpr (PARTS == 1) {
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&acc_empty[ti & 1]);
        ++ti;
      }
    }
    if (p.tma_io && lane == 0) {
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
  if (warp == 2) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, 2 * BN);
  }
}

// --------------------------------------------------------- small kernels ----
// Rows of `src` as operand planes [parts][rows][pitch] (pitch a multiple of 8,
// zero padded): FP32 as three bf16 parts, 16-bit data as it is. The first part
// is cut off, not rounded, so that it never overflows; an infinity or NaN keeps
// its place in the first part.
template <typename T>
__global__ void __launch_bounds__(256) linear_stage_kernel(const T* __restrict__ src, long long ld,
                                                           long long rows, int cols, int pitch,
                                                           uint4* __restrict__ dst) {
  const int per = pitch / 8;
  const long long total = rows * per;
  const bool vec = ld * sizeof(T) % 16 == 0 && (uintptr_t)src % 16 == 0;
  for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < total;
       i += (long long)gridDim.x * blockDim.x) {
    const long long r = i / per;
    const int c = (int)(i - r * per) * 8;
    union { uint4 u[sizeof(T) / 2]; T e[8]; } v;
    const T* s = src + r * ld + c;
    if (vec && c + 8 <= cols) {
#pragma unroll
      for (int k = 0; k < (int)sizeof(T) / 2; ++k) v.u[k] = __ldg(reinterpret_cast<const uint4*>(s) + k);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) v.e[k] = c + k < cols ? s[k] : from_f32<T>(0.f);
    }
    if constexpr (sizeof(T) == 2) {
      dst[i] = v.u[0];
    } else {
      union { uint4 u; __nv_bfloat16 e[8]; } o[3];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float f = v.e[k];
        const __nv_bfloat16 h0 = __float2bfloat16_rz(f);
        const float r1 = f - __bfloat162float(h0);
        const bool fin = isfinite(f);
        const __nv_bfloat16 h1 = __float2bfloat16_rn(fin ? r1 : 0.f);
        const float r2 = fin ? r1 - __bfloat162float(h1) : 0.f;
        o[0].e[k] = h0;
        o[1].e[k] = h1;
        o[2].e[k] = __float2bfloat16_rn(r2);
      }
#pragma unroll
      for (int k = 0; k < 3; ++k) dst[k * total + i] = o[k].u;
    }
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

// out[i] = sum over `count` partials [count][size], in order.
template <typename T>
__global__ void __launch_bounds__(256) linear_fold_kernel(const float* __restrict__ part, int count,
                                                          long long rows, int cols, int pitch,
                                                          T* __restrict__ out) {
  const long long total = rows * cols;
  for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < total;
       i += (long long)gridDim.x * blockDim.x) {
    const long long r = i / cols;
    const float* s = part + r * pitch + (i - r * cols);
    float a = 0.f;
#pragma unroll 8
    for (int k = 0; k < count; ++k) a += s[(long long)k * rows * pitch];
    out[i] = from_f32<T>(a);
  }
}

// Column totals of [rows][cols] FP32 partials: 32 columns a block.
template <typename T>
__global__ void __launch_bounds__(1024) linear_fold_rows_kernel(const float* __restrict__ part,
                                                                long long rows, int cols,
                                                                T* __restrict__ out) {
  __shared__ float sh[32][33];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float a = 0.f;
  if (c < cols)
#pragma unroll 4
    for (long long r = w; r < rows; r += 32) a += part[r * cols + c];
  sh[w][lane] = a;
  __syncthreads();
  if (w == 0 && c < cols) {
    for (int i = 1; i < 32; ++i) a += sh[i][lane];
    out[c] = from_f32<T>(a);
  }
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
  float z[1] = {0.f};
#pragma unroll
  for (int r = 0; r < MR; ++r)
    if (lane == r) z[0] = acc[r];
  if (lane < m) {
    if (bias != nullptr) z[0] += to_f32<T>(bias[col]);
    act_values<sizeof(T) == 2, 1>(act, z);
    const long long at = (long long)lane * n + col;
    if (res != nullptr) z[0] += to_f32<T>(res[at]);
    out[at] = from_f32<T>(z[0]);
  }
}

// ------------------------------------------------------------ host: plan ----
size_t up256(size_t v) { return (v + 255) / 256 * 256; }
int round8(int v) { return (v + 7) / 8 * 8; }

// A tensor-core operand in memory: rows x cols of 16-bit values, `parts`
// planes of rows * pitch.
struct Operand {
  const void* ptr;
  long long rows;
  int cols;
  long long pitch;
  int parts;
};

template <typename T> struct OpOf { using type = T; };
template <> struct OpOf<float> { using type = __nv_bfloat16; };

int small_grid(long long items) {
  const long long want = (items + 255) / 256, most = 148 * 8;
  return (int)(want < 1 ? 1 : want < most ? want : most);
}

size_t plane_bytes(long long rows, int cols, int parts) {
  return up256((size_t)parts * rows * round8(cols) * 2);
}

template <typename T>
int stage(const void* src, long long ld, long long rows, int cols, void* dst, cudaStream_t st) {
  const int pitch = round8(cols);
  linear_stage_kernel<T><<<small_grid(rows * (pitch / 8)), 256, 0, st>>>(
      static_cast<const T*>(src), ld, rows, cols, pitch, static_cast<uint4*>(dst));
  DDPM_CHECK_LAUNCH("linear_stage_kernel");
  return DDPM_OK;
}

// Column tile: the widest of 256, 128, 64 that wastes less than a quarter of
// its columns more than the next narrower one and leaves a tile for every SM.
int pick_bn(long long m, int n, int most) {
  const long long tm = (m + kBM - 1) / kBM;
  for (int bn = most; bn > 64; bn /= 2) {
    const long long tn = (n + bn - 1) / bn;
    const long long narrow = (n + bn / 2 - 1) / (bn / 2);
    if (tm * tn >= gencat::num_sms() && 2 * tn - narrow <= narrow / 4) return bn;
  }
  return 64;
}

template <typename T, int BN, int PARTS, Epi kEpi>
int launch_gemm_as(GemmParams& p, cudaStream_t st) {
  auto fn = linear_gemm_kernel<T, BN, PARTS, kEpi>;
  const int tiles_k = (p.kblocks + p.splits - 1) / p.splits;
  const int limit = gencat::max_smem_optin() - 2048;  // static shared memory
  // As many stages as the K loop can use, at least two; what is left goes to
  // the epilogue's boxes, eight a warp at most, two at least.
  p.nbuf = 2;
  int stages = kMaxStages;
  auto total = [&](int s, int b) { return (int)smem_layout(PARTS, BN, s, b).total; };
  // a persistent block streams several tiles through the ring: twice a tile's
  // steps is as far ahead as it needs to look
  const int useful = tiles_k * 2 < 2 ? 2 : tiles_k * 2;
  if (stages > useful) stages = useful;
  while (stages > 1 && total(stages, p.nbuf) > limit) --stages;
  while (p.nbuf < kMaxBufs && total(stages, p.nbuf * 2) <= limit) p.nbuf *= 2;
  p.stages = stages;
  const int smem = total(stages, p.nbuf);
  DDPM_CUDA_TRY(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  const int sms = gencat::num_sms();
  const int grid = p.num_tiles < sms ? p.num_tiles : sms;
  fn<<<grid, kThreads, smem, st>>>(p);
  DDPM_CHECK_LAUNCH("linear_gemm_kernel");
  return DDPM_OK;
}

template <typename T, Epi kEpi>
int launch_gemm(GemmParams& p, int bn, cudaStream_t st) {
  if constexpr (sizeof(T) == 4) {
    return bn == 128 ? launch_gemm_as<T, 128, 3, kEpi>(p, st)
                     : launch_gemm_as<T, 64, 3, kEpi>(p, st);
  } else {
    return bn == 256   ? launch_gemm_as<T, 256, 1, kEpi>(p, st)
           : bn == 128 ? launch_gemm_as<T, 128, 1, kEpi>(p, st)
                       : launch_gemm_as<T, 64, 1, kEpi>(p, st);
  }
}

int operand_map(CUtensorMap* map, const Operand& o, bool mn_major, int tile_rows, bool bf16) {
  // K-major: [parts][rows][k], box 64 k x tile rows; MN-major: the operand's
  // rows are the contraction's k, box 64 columns x 64 k
  const uint64_t dims[3] = {(uint64_t)o.cols, (uint64_t)o.rows, (uint64_t)o.parts};
  const uint64_t strides[2] = {(uint64_t)o.pitch * 2, (uint64_t)o.rows * o.pitch * 2};
  const uint32_t box[3] = {64, (uint32_t)(mn_major ? kBK : tile_rows), (uint32_t)o.parts};
  return encode_tmap(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                     3, o.ptr, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

int io_map(CUtensorMap* map, const void* ptr, int es, bool bf16, long long rows, int cols,
           long long ld, int splits) {
  const uint64_t dims[3] = {(uint64_t)cols, (uint64_t)rows, (uint64_t)splits};
  const uint64_t strides[2] = {(uint64_t)ld * es, (uint64_t)rows * ld * es};
  const uint32_t box[3] = {(uint32_t)(64 / es), 32, 1};
  return encode_tmap(map,
                     es == 4  ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                     : bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                            : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                     3, ptr, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_64B);
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
  int splits, bn;
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
  p.tiles_m = (int)((g.M + kBM - 1) / kBM);
  p.tiles_n = (g.N + g.bn - 1) / g.bn;
  p.splits = g.splits;
  p.num_tiles = p.tiles_m * p.tiles_n * g.splits;
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
  p.idesc = tc::idesc_f16(kBM, g.bn, kBf16, g.a_mn, g.b_mn);
  p.tma_io = tma_ready(g.out, g.ld_out, es) && (g.in == nullptr || tma_ready(g.in, g.ld_in, es));
  int rc = gencat::status_ptr(&p.status);
  if (rc) return rc;
  rc = operand_map(&p.a, g.a, g.a_mn, kBM, kBf16);
  if (rc) return rc;
  rc = operand_map(&p.b, g.b, g.b_mn, g.bn, kBf16);
  if (rc) return rc;
  if (p.tma_io) {
    rc = io_map(&p.out, g.out, es, kBf16, g.M, g.N, g.ld_out, g.splits);
    if (rc) return rc;
    if (g.in != nullptr) {
      rc = io_map(&p.in, g.in, es, kBf16, g.M, g.N, g.ld_in, 1);
      if (rc) return rc;
    }
  }
  return launch_gemm<T, kEpi>(p, g.bn, st);
}

// What a call has to lay out in its workspace.
struct LinearPlan {
  bool rows_path;            // the dot-product kernel
  bool stage_x, stage_w, stage_dz;
  int parts, bn_z, bn_x, bn_w, splits_w;
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
  const int widest = f32 ? 128 : 256;
  q.parts = f32 ? 3 : 1;
  q.rows_path = !bwd && s.m <= kGemvRows;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t o = at;
    at += up256(bytes);
    return o;
  };
  if (!q.rows_path) {
    q.stage_x = f32 || !s.aligned || s.ldx % 8;
    q.stage_w = f32 || !s.aligned || s.k % 8;
    q.x_off = q.stage_x ? take(plane_bytes(s.m, s.k, q.parts)) : 0;
    q.w_off = q.stage_w ? take(plane_bytes(s.n, s.k, q.parts)) : 0;
  }
  q.bn_z = pick_bn(s.m, s.n, widest);
  if (bwd) {
    const bool recompute = s.act != DDPM_ACT_NONE;
    // dz as the data's type (recomputed), then as operand planes where that is
    // not one already
    if (recompute) q.dz_off = take((size_t)s.m * round8(s.n) * es);
    q.stage_dz = f32 || (!recompute && (!s.aligned || s.n % 8));
    q.dzp_off = q.stage_dz ? take(plane_bytes(s.m, s.n, q.parts)) : 0;
    q.bn_x = pick_bn(s.m, s.k, widest);
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
    // dweight: split the rows over the SMs, at least four K blocks a split
    const long long kb = (s.m + kBK - 1) / kBK;
    q.bn_w = s.k > 128 && widest == 256 ? 256 : s.k > 64 ? 128 : 64;
    const long long tiles = (long long)((s.n + kBM - 1) / kBM) * ((s.k + q.bn_w - 1) / q.bn_w);
    long long splits = gencat::num_sms() / tiles;
    if (splits > kb / 4) splits = kb / 4;
    q.splits_w = (int)(splits < 1 ? 1 : splits);
    if (q.splits_w > 1) q.part_off = take((size_t)q.splits_w * s.n * ((s.k + 3) / 4 * 4) * 4);
  }
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

Operand make_operand(const void* ptr, long long rows, int cols, long long pitch, int parts) {
  return Operand{ptr, rows, cols, pitch, parts};
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
  g.a = q.stage_x ? make_operand(ws + q.x_off, s.m, s.k, round8(s.k), q.parts)
                  : make_operand(x, s.m, s.k, s.ldx, 1);
  g.b = q.stage_w ? make_operand(ws + q.w_off, s.n, s.k, round8(s.k), q.parts)
                  : make_operand(w, s.n, s.k, s.k, 1);
  g.M = s.m;
  g.N = s.n;
  g.K = s.k;
  g.bias = bias;
  g.in = res;
  g.ld_in = s.n;
  g.out = out;
  g.ld_out = s.n;
  g.act = s.act;
  g.splits = 1;
  g.bn = q.bn_z;
  return run_gemm<T, kOut>(g, st);
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
  const Operand xo = q.stage_x ? make_operand(ws + q.x_off, s.m, s.k, round8(s.k), q.parts)
                               : make_operand(x, s.m, s.k, s.ldx, 1);
  const Operand wo = q.stage_w ? make_operand(ws + q.w_off, s.n, s.k, round8(s.k), q.parts)
                               : make_operand(w, s.n, s.k, s.k, 1);
  float* colsum = reinterpret_cast<float*>(ws + q.colsum_off);
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
    g.splits = 1;
    g.bn = q.bn_z;
    if ((rc = run_gemm<T, kDz>(g, st))) return rc;
    dz = g.out;
    ld_dz = g.ld_out;
  } else if (gb) {
    const dim3 grid((unsigned)((s.n + 31) / 32), (unsigned)q.colsum_rows);
    linear_colsum_kernel<T><<<grid, 256, 0, st>>>(static_cast<const T*>(dy), s.m, s.n,
                                                  q.colsum_chunk, colsum);
    DDPM_CHECK_LAUNCH("linear_colsum_kernel");
  }
  if (gb) {
    linear_fold_rows_kernel<T><<<(s.n + 31) / 32, 1024, 0, st>>>(colsum, q.colsum_rows, s.n,
                                                                 static_cast<T*>(gb));
    DDPM_CHECK_LAUNCH("linear_fold_rows_kernel");
  }
  if (!gx && !gw) return DDPM_OK;
  Operand zo = make_operand(dz, s.m, s.n, ld_dz, 1);
  if (q.stage_dz) {
    if ((rc = stage<T>(dz, ld_dz, s.m, s.n, ws + q.dzp_off, st))) return rc;
    zo = make_operand(ws + q.dzp_off, s.m, s.n, round8(s.n), q.parts);
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
    g.splits = 1;
    g.bn = q.bn_x;
    if ((rc = run_gemm<T, kOut>(g, st))) return rc;
  }
  if (gw) {
    Gemm g{};
    g.a = zo;
    g.b = xo;
    g.a_mn = g.b_mn = true;
    g.M = s.n;
    g.N = s.k;
    g.K = s.m;
    g.splits = q.splits_w;
    g.bn = q.bn_w;
    if (q.splits_w > 1) {
      const int pitch = (s.k + 3) / 4 * 4;
      g.out = ws + q.part_off;
      g.ld_out = pitch;
      if ((rc = run_gemm<T, kPartial>(g, st))) return rc;
      linear_fold_kernel<T><<<small_grid((long long)s.n * s.k), 256, 0, st>>>(
          reinterpret_cast<const float*>(ws + q.part_off), q.splits_w, s.n, s.k, pitch,
          static_cast<T*>(gw));
      DDPM_CHECK_LAUNCH("linear_fold_kernel");
    } else {
      g.out = gw;
      g.ld_out = s.k;
      if ((rc = run_gemm<T, kOut>(g, st))) return rc;
    }
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
