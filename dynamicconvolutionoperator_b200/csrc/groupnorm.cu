// Group norm with an activation over channel-last data, forward and backward.
//
//   x [N][P][C] (P pixels, channels innermost), G groups of cg = C / G channels
//   mean, rstd   per (n, g) over cnt = P * cg values, biased variance
//   z    = (x - mean) * rstd * weight[c] + bias[c],   out = act(z)
// backward, with dz = dy * act'(z) and xhat = (x - mean) * rstd:
//   dbias = sum dz, dweight = sum dz * xhat          (over n, pixels)
//   A = sum_group weight * dz / cnt, B = sum_group weight * dz * xhat / cnt
//   dx = rstd * (weight * dz - A - xhat * B)
//
// Bound: HBM. Both directions need their group's sums before the first value
// can be written, so the data is needed twice; the point of the design is that
// the second time comes from L2. One persistent launch walks chunks (R pixels
// of one sample) in order: a block sums chunk t (phase 1), and L steps later,
// when every block has passed the end of that chunk's sample, writes it
// (phase 2). L = ceil((chunks of a sample - 1) / grid), where a step of all blocks is
// up to 21 MB of x (backward: 7): 1 for a sample of 16 MB, 3 in the backward. The
// ring kernel adds two steps. So what lies between the phases is a few tens of MB.
//
// The blocks of a sample meet through a counter: the last one to add its
// partial sums folds the sample's partials in their fixed order (no floating
// point atomics: results do not depend on the order of arrival) and raises the
// sample's flag; phase 2 waits for the flag. No block waits for a phase 1
// that lies behind a wait of the same step, and the cooperative launch keeps
// all blocks resident, so the waits end; they are bounded all the same.
//
// Variance: every thread sums x - s and (x - s)^2 for its own channel about
// its first value s, then (count, mean, squared deviations) triples are merged
// exactly, so a mean far from zero costs no precision.
#include <atomic>
#include <type_traits>

#include "act.cuh"
#include "common.cuh"
#include "tc.cuh"

namespace ddpm {

namespace gencat {
int status_ptr(int** out);
int num_sms();
}  // namespace gencat

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxChannels = 65536;  // at one channel a thread: 256 tiles, fewer than the blocks
constexpr uint64_t kWaitLimitNs = 2000000000ull;

struct NormParams {
  const void* x;
  const void* dy;      // backward only
  const void* weight;  // nullable (ones)
  const void* bias;    // nullable (zeros)
  void* out;           // out, or dx (nullable in the backward)
  float2* stats;       // [N][G] mean, rstd (written by the forward)
  float2* part;        // [N * S][U] partial sums of a chunk
  float2* grp;         // backward: [N][G] A, B
  float2* wsum;        // backward: [grid / CT][C] sums of dz, dz * xhat; nullable
  unsigned* count;     // [N] arrivals, then [N] flags; zeroed before the launch
  int* status;
  long long P;
  int N, C, G, cg;
  int R, S, CT, TX, TY, U, uw;  // uw: channels of a unit (partials are kept per unit)
  long long chunks;
  int lag, act, param_f32;
  float eps;
};

template <typename T, int V> struct alignas(sizeof(T) * V) Vec { T e[V]; };

template <typename T> __device__ __forceinline__ float load_param(const void* p, int c, int f32) {
  return f32 ? __ldg(static_cast<const float*>(p) + c) : ldg_f32<T>(static_cast<const T*>(p) + c);
}

// Sum over the warp, the same in every lane.
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// What a block's threads keep for the whole launch.
template <int V> struct Column {
  int c0;        // first channel
  bool live;
  float w[V], b[V];
};

// Chunk t -> sample, first pixel, pixels.
struct Chunk {
  int n, rows;
  long long at;  // index of the first pixel over all samples
};
__device__ __forceinline__ Chunk chunk_of(const NormParams& p, long long t) {
  const long long ns = t / p.CT;
  Chunk k;
  k.n = (int)(ns / p.S);
  const int s = (int)(ns - (long long)k.n * p.S);
  const long long first = (long long)s * p.R;
  k.at = (long long)k.n * p.P + first;
  k.rows = (int)(p.P - first < p.R ? p.P - first : p.R);
  return k;
}

// The chunks of a block in order, t = block + i * grid, without a division a
// step (one tile of columns).
struct Walk {
  int n, s, dn, ds;
  __device__ __forceinline__ Walk(const NormParams& p)
      : n((int)(blockIdx.x / (unsigned)p.S)), s((int)(blockIdx.x % (unsigned)p.S)),
        dn((int)(gridDim.x / (unsigned)p.S)), ds((int)(gridDim.x % (unsigned)p.S)) {}
  __device__ __forceinline__ Chunk next(const NormParams& p) {
    Chunk k;
    k.n = n;
    const long long first = (long long)s * p.R;
    k.at = (long long)n * p.P + first;
    k.rows = (int)(p.P - first < p.R ? p.P - first : p.R);
    n += dn;
    s += ds;
    if (s >= p.S) {
      s -= p.S;
      ++n;
    }
    return k;
  }
};

__device__ __forceinline__ unsigned add_acq_rel(unsigned* p) {
  unsigned old;
  asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(old) : "l"(p) : "memory");
  return old;
}
__device__ __forceinline__ unsigned load_acquire(const unsigned* p) {
  unsigned v;
  asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ void store_release(unsigned* p, unsigned v) {
  asm volatile("st.release.gpu.global.u32 [%0], %1;" ::"l"(p), "r"(v) : "memory");
}

// (mean, squared deviations) of unit u of the tile from the per-thread pairs
// in shared memory; every lane of the warp gets the result.
__device__ __forceinline__ float2 merge_unit(const NormParams& p, const float2* sh, int u,
                                             int width, int rows, int lane) {
  const int items = p.TY * p.uw;
  const int full = rows / p.TY, rest = rows - full * p.TY;
  const float m0 = sh[u * p.uw].x;  // sums about the first mean: no digits lost to a large one
  float s = 0.f;
  for (int i = lane; i < items; i += 32) {
    const int ty = i / p.uw;
    const float k = (float)(full + (ty < rest));
    if (k > 0.f) s += k * (sh[ty * width + u * p.uw + (i - ty * p.uw)].x - m0);
  }
  const float cnt = (float)rows * (float)p.uw;
  const float mean = m0 + warp_sum(s) / cnt;
  float m2 = 0.f;
  for (int i = lane; i < items; i += 32) {
    const int ty = i / p.uw;
    const float k = (float)(full + (ty < rest));
    const float2 v = sh[ty * width + u * p.uw + (i - ty * p.uw)];
    const float d = v.x - mean;
    if (k > 0.f) m2 += v.y + k * d * d;
  }
  return make_float2(mean, warp_sum(m2));
}

__device__ __forceinline__ void count_release(unsigned* p) {
  asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(p) : "memory");
}

// Partials of a group as a warp folds them: kKept values a lane stay in
// registers for the second pass, longer lists are read twice. The loads of a
// pass are in flight together: the sample's whole grid waits for this fold.
constexpr int kKept = 12;

// Mean and rstd of group g of sample n from its chunks' partials (one warp).
__device__ __forceinline__ float2 fold_stats(const NormParams& p, int n, int g, int lane) {
  const int upg = p.U / p.G;
  const int items = p.S * upg;
  const float total = (float)((double)p.P * p.cg);
  const float* base =
      reinterpret_cast<const float*>(p.part + (long long)n * p.S * p.U + (long long)g * upg);
  const float per = (float)p.R * (float)p.uw;  // values behind a partial, and behind the last chunk's
  const float last = (float)(p.P - (long long)(p.S - 1) * p.R) * (float)p.uw;
  auto load = [&](int i) {
    const int k = upg == 1 ? i : i / upg;
    return __ldcg(reinterpret_cast<const float2*>(base) + (long long)k * p.U + (i - k * upg));
  };
  auto count = [&](int i) { return i >= items - upg ? last : per; };
  float2 v[kKept];
#pragma unroll
  for (int j = 0; j < kKept; ++j)
    if (lane + 32 * j < items) v[j] = load(lane + 32 * j);
  const float m0 = __ldcg(base);  // sums about the first mean
  float s = 0.f, m2 = 0.f;
#pragma unroll
  for (int j = 0; j < kKept; ++j)
    if (lane + 32 * j < items) s += count(lane + 32 * j) * (v[j].x - m0);
#pragma unroll 4
  for (int i = lane + 32 * kKept; i < items; i += 32) s += count(i) * (load(i).x - m0);
  const float mean = m0 + warp_sum(s) / total;
#pragma unroll
  for (int j = 0; j < kKept; ++j)
    if (lane + 32 * j < items) {
      const float d = v[j].x - mean;
      m2 += v[j].y + count(lane + 32 * j) * d * d;
    }
#pragma unroll 4
  for (int i = lane + 32 * kKept; i < items; i += 32) {
    const float2 u = load(i);
    const float d = u.x - mean;
    m2 += u.y + count(i) * d * d;
  }
  m2 = warp_sum(m2);
  return make_float2(mean, 1.f / sqrtf(m2 / total + p.eps));
}

// A and B of group g of sample n (one warp).
__device__ __forceinline__ float2 fold_sums(const NormParams& p, int n, int g, int lane) {
  const int upg = p.U / p.G;
  const int items = p.S * upg;
  const float total = (float)((double)p.P * p.cg);
  const float2* base = p.part + (long long)n * p.S * p.U + (long long)g * upg;
  float a = 0.f, b = 0.f;
#pragma unroll 8
  for (int i = lane; i < items; i += 32) {
    const int k = upg == 1 ? i : i / upg;
    const float2 v = __ldcg(&base[(long long)k * p.U + (i - k * upg)]);
    a += v.x;
    b += v.y;
  }
  a = warp_sum(a);
  b = warp_sum(b);
  return make_float2(a / total, b / total);
}

__device__ __forceinline__ float2 load_peer(const float2* p, int rank) {
  uint32_t at;
  float2 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(tc::smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory");
  return v;
}

// kCluster: the S blocks of a sample are a cluster with one chunk each, whose
// partials meet in shared memory (small samples: no counters, no waits but the
// cluster's barrier).
template <typename T, int V, bool kBwd, bool kCluster>
__global__ void __launch_bounds__(kThreads, kBwd ? 2 : 3) norm_kernel(const NormParams p) {
  constexpr bool kFast = sizeof(T) == 2;
  constexpr int kUnroll = 4;
  using Vt = Vec<T, V>;
  __shared__ float2 sh[kThreads * V];
  __shared__ float2 run[kBwd ? kThreads * V : 1];  // the block's own sums of dz, dz * xhat
  __shared__ float2 peer[kCluster ? kThreads * V : 1];    // this block's partials
  __shared__ float2 folded[kCluster ? kThreads * V : 1];  // the sample's: (mean, rstd), (A, B)
  __shared__ int sh_last, sh_abort;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int ct = (int)(blockIdx.x % p.CT);
  const int tx = tid % p.TX, ty = tid / p.TX;
  const int width = p.TX * V;  // channels of the tile (the last tile may hold fewer)
  const int tile_c = (p.C - ct * width) < width ? p.C - ct * width : width;
  Column<V> col;
  col.c0 = ct * width + tx * V;
  col.live = ty < p.TY && col.c0 < p.C;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    col.w[e] = col.live && p.weight ? load_param<T>(p.weight, col.c0 + e, p.param_f32) : 1.f;
    col.b[e] = col.live && p.bias ? load_param<T>(p.bias, col.c0 + e, p.param_f32) : 0.f;
  }
  if (tid == 0) sh_abort = 0;
  if constexpr (kBwd) {
#pragma unroll
    for (int e = 0; e < V; ++e) run[tid * V + e] = make_float2(0.f, 0.f);
  }
  const T* x = static_cast<const T*>(p.x);
  const T* dy = static_cast<const T*>(p.dy);
  T* out = static_cast<T*>(p.out);
  unsigned* flags = p.count + p.N;
  __syncthreads();

  const long long steps = (p.chunks + gridDim.x - 1) / gridDim.x;
  for (long long i = 0; i < steps + p.lag; ++i) {
    // ---- phase 1: partial sums of chunk t1 ----
    const long long t1 = i * gridDim.x + blockIdx.x;
    if (i < steps && t1 < p.chunks) {
      const Chunk k = chunk_of(p, t1);
      if (col.live) {
        const long long base = (k.at + ty) * p.C + col.c0;
        const long long pitch = (long long)p.TY * p.C;
        const int mine = (k.rows - ty + p.TY - 1) / p.TY;  // <= 0: none
        if constexpr (!kBwd) {
          float s0[V], a1[V], a2[V];
#pragma unroll
          for (int e = 0; e < V; ++e) s0[e] = a1[e] = a2[e] = 0.f;
          if (mine > 0) {
            const Vt v = *reinterpret_cast<const Vt*>(x + base);
#pragma unroll
            for (int e = 0; e < V; ++e) s0[e] = to_f32<T>(v.e[e]);
          }
          for (int r = 0; r < mine; r += kUnroll) {
            Vt v[kUnroll];
#pragma unroll
            for (int j = 0; j < kUnroll; ++j)
              if (r + j < mine) v[j] = *reinterpret_cast<const Vt*>(x + base + (r + j) * pitch);
#pragma unroll
            for (int j = 0; j < kUnroll; ++j)
              if (r + j < mine) {
#pragma unroll
                for (int e = 0; e < V; ++e) {
                  const float d = to_f32<T>(v[j].e[e]) - s0[e];
                  a1[e] += d;
                  a2[e] += d * d;
                }
              }
          }
          const float cnt = (float)(mine > 0 ? mine : 1);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float m = a1[e] / cnt;
            sh[ty * width + tx * V + e] = make_float2(s0[e] + m, fmaxf(a2[e] - a1[e] * m, 0.f));
          }
        } else {
          float mean[V], rstd[V], s1[V], s2[V];
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float2 st = __ldg(&p.stats[(long long)k.n * p.G + (col.c0 + e) / p.cg]);
            mean[e] = st.x;
            rstd[e] = st.y;
            s1[e] = s2[e] = 0.f;
          }
          for (int r = 0; r < mine; r += kUnroll) {
            Vt v[kUnroll], g[kUnroll];
#pragma unroll
            for (int j = 0; j < kUnroll; ++j)
              if (r + j < mine) {
                v[j] = *reinterpret_cast<const Vt*>(x + base + (r + j) * pitch);
                g[j] = *reinterpret_cast<const Vt*>(dy + base + (r + j) * pitch);
              }
#pragma unroll
            for (int j = 0; j < kUnroll; ++j)
              if (r + j < mine) {
                float xh[V], sl[V + V % 2];
                if constexpr (V == 1) sl[1] = 0.f;
#pragma unroll
                for (int e = 0; e < V; ++e) {
                  xh[e] = (to_f32<T>(v[j].e[e]) - mean[e]) * rstd[e];
                  sl[e] = xh[e] * col.w[e] + col.b[e];
                }
                act_slopes<kFast, V + V % 2>(p.act, sl);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                  const float dz = to_f32<T>(g[j].e[e]) * sl[e];
                  s1[e] += dz;
                  s2[e] += dz * xh[e];
                }
              }
          }
#pragma unroll
          for (int e = 0; e < V; ++e) {
            sh[ty * width + tx * V + e] = make_float2(s1[e] * col.w[e], s2[e] * col.w[e]);
            float2& q = run[tid * V + e];
            q.x += s1[e];
            q.y += s2[e];
          }
        }
      }
      __syncthreads();
      // units of this tile: groups, or single channels when the channels do
      // not fit one tile
      const int units = tile_c / p.uw;
      const int u0 = ct * width / p.uw;
      for (int u = warp; u < units; u += kWarps) {
        float2 r;
        if constexpr (!kBwd) {
          r = merge_unit(p, sh, u, width, k.rows, lane);
        } else {
          float a = 0.f, b = 0.f;
          for (int j = lane; j < p.TY * p.uw; j += 32) {
            const int yy = j / p.uw;
            const float2 v = sh[yy * width + u * p.uw + (j - yy * p.uw)];
            a += v.x;
            b += v.y;
          }
          r = make_float2(warp_sum(a), warp_sum(b));
        }
        if (lane == 0) {
          if constexpr (kCluster) peer[u] = r;
          else p.part[(t1 / p.CT) * p.U + u0 + u] = r;
        }
      }
      if constexpr (kCluster) {
        // one cluster, one sample (S > 1); a block alone may have several
        if (p.S > 1)
          asm volatile("barrier.cluster.arrive.release.aligned;\n\t"
                       "barrier.cluster.wait.acquire.aligned;" ::: "memory");
        else
          __syncthreads();
        const float total = (float)p.P * (float)p.cg;
        for (int g = warp; g < p.G; g += kWarps) {
          const bool in = lane < p.S;
          const float2 v = in ? load_peer(&peer[g], lane) : make_float2(0.f, 0.f);
          float2 r;
          if constexpr (!kBwd) {
            const float cnt = in ? (float)(min((long long)p.R, p.P - (long long)lane * p.R)) * (float)p.cg : 0.f;
            const float m0 = __shfl_sync(0xffffffffu, v.x, 0);
            const float mean = m0 + warp_sum(in ? cnt * (v.x - m0) : 0.f) / total;
            const float d = v.x - mean;
            const float m2 = warp_sum(in ? v.y + cnt * d * d : 0.f);
            r = make_float2(mean, 1.f / sqrtf(m2 / total + p.eps));
            if (lane == 0 && k.at == (long long)k.n * p.P) p.stats[(long long)k.n * p.G + g] = r;
          } else {
            r = make_float2(warp_sum(v.x) / total, warp_sum(v.y) / total);
          }
          if (lane == 0) folded[g] = r;
        }
        __syncthreads();
        // the peers' reads of this block's partials are over before it ends
        if (p.S > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
      } else {
        __syncthreads();
        if (tid == 0) {
          __threadfence();
          sh_last = add_acq_rel(&p.count[k.n]) == (unsigned)(p.S * p.CT - 1);
        }
        __syncthreads();
        if (sh_last) {  // the sample's last chunk: fold its partials
          for (int g = warp; g < p.G; g += kWarps) {
            const float2 r = kBwd ? fold_sums(p, k.n, g, lane) : fold_stats(p, k.n, g, lane);
            if (lane == 0) (kBwd ? p.grp : p.stats)[(long long)k.n * p.G + g] = r;
          }
          __threadfence();
          __syncthreads();
          if (tid == 0) store_release(&flags[k.n], 1u);
        }
      }
    }
    // ---- phase 2: write chunk t2 ----
    const long long t2 = (i - p.lag) * gridDim.x + blockIdx.x;
    if (i >= p.lag && t2 < p.chunks && (!kBwd || p.out != nullptr)) {
      const Chunk k = chunk_of(p, t2);
      if (!kCluster && tid == 0 && load_acquire(&flags[k.n]) == 0u) {
        const uint64_t began = tc::globaltimer_ns();
        while (load_acquire(&flags[k.n]) == 0u) {
          __nanosleep(32);
          if (tc::globaltimer_ns() - began > kWaitLimitNs) {
            sh_abort = 1;
            atomicCAS(p.status, 0, 90);
            break;
          }
        }
      }
      if constexpr (!kCluster) {
        __syncthreads();
        if (sh_abort) return;
      }
      if (col.live) {
        const long long base = (k.at + ty) * p.C + col.c0;
        const long long pitch = (long long)p.TY * p.C;
        const int mine = (k.rows - ty + p.TY - 1) / p.TY;
        float mean[V], rstd[V], ga[V], gb[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const int gl = (col.c0 + e) / p.cg;
          const long long g = (long long)k.n * p.G + gl;
          const float2 st = kCluster && !kBwd ? folded[gl] : __ldcg(&p.stats[g]);
          mean[e] = st.x;
          rstd[e] = st.y;
          if constexpr (kBwd) {
            const float2 ab = kCluster ? folded[gl] : __ldcg(&p.grp[g]);
            ga[e] = ab.x;
            gb[e] = ab.y;
          }
        }
        for (int r = 0; r < mine; r += kUnroll) {
          Vt v[kUnroll], d[kUnroll];
#pragma unroll
          for (int j = 0; j < kUnroll; ++j)
            if (r + j < mine) {
              v[j] = *reinterpret_cast<const Vt*>(x + base + (r + j) * pitch);
              if constexpr (kBwd) d[j] = *reinterpret_cast<const Vt*>(dy + base + (r + j) * pitch);
            }
#pragma unroll
          for (int j = 0; j < kUnroll; ++j)
            if (r + j < mine) {
              float xh[V], z[V + V % 2];
              if constexpr (V == 1) z[1] = 0.f;
#pragma unroll
              for (int e = 0; e < V; ++e) {
                xh[e] = (to_f32<T>(v[j].e[e]) - mean[e]) * rstd[e];
                z[e] = xh[e] * col.w[e] + col.b[e];
              }
              Vt o;
              if constexpr (!kBwd) {
                act_values<kFast, V + V % 2>(p.act, z);
#pragma unroll
                for (int e = 0; e < V; ++e) o.e[e] = from_f32<T>(z[e]);
              } else {
                act_slopes<kFast, V + V % 2>(p.act, z);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                  const float dz = to_f32<T>(d[j].e[e]) * z[e];
                  o.e[e] = from_f32<T>(rstd[e] * (col.w[e] * dz - ga[e] - xh[e] * gb[e]));
                }
              }
              *reinterpret_cast<Vt*>(out + base + (r + j) * pitch) = o;
            }
        }
      }
    }
  }
  if constexpr (kCluster) {
    if (p.S > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  if constexpr (kBwd) {
    if (p.wsum != nullptr) {
      __syncthreads();
      // rows of the block folded in order; one channel a thread at a time
      for (int c = tid; c < tile_c; c += kThreads) {
        float2 a = make_float2(0.f, 0.f);
        for (int yy = 0; yy < p.TY; ++yy) {
          const float2 v = run[yy * width + c];
          a.x += v.x;
          a.y += v.y;
        }
        p.wsum[(long long)(blockIdx.x / p.CT) * p.C + ct * width + c] = a;
      }
    }
  }
}

// dbias and dweight from the blocks' sums: 32 channels a block, its 8 warps
// share the rows, folded in a fixed order.
template <typename PT>
__global__ void __launch_bounds__(256) norm_param_kernel(const float2* __restrict__ sums, int rows,
                                                         int C, PT* gw, PT* gb) {
  __shared__ float2 sh[8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float2 a = make_float2(0.f, 0.f);
  if (c < C)
    for (int r = warp; r < rows; r += 8) {
      const float2 v = sums[(long long)r * C + c];
      a.x += v.x;
      a.y += v.y;
    }
  sh[warp][lane] = a;
  __syncthreads();
  if (warp == 0 && c < C) {
    for (int w = 1; w < 8; ++w) {
      a.x += sh[w][lane].x;
      a.y += sh[w][lane].y;
    }
    if (gb) gb[c] = from_f32<PT>(a.x);
    if (gw) gw[c] = from_f32<PT>(a.y);
  }
}

// ---------------------------------------------------------- ring kernel ----
// The same two phases for large, regular data (channels of a group in fours,
// 16-byte rows): one block an SM, whose warps have roles.
//   copy warp      bulk copies of chunks into a ring of shared-memory slots
//   20 work warps  phase 1 from a slot: sums of 4 channels a thread; phase 2
//                  from the same slot (or from a second copy where a sample
//                  needs more steps than the ring has slots): the result
//   4 merge warps  merge a chunk's sums, write them and count the chunk
//   4 fold warps   wait until a sample's chunks are all counted, fold its
//                  partials for phase 2
// so the copies, the sums' way through global memory and the work overlap, and
// no role waits for another's round trip: the counting is a reduction without
// an answer, and every block folds the samples that it writes, all in the same
// order. A slot holds a chunk of x (backward: of x and dy).
//
// Measured, 64 x 256 x 256 x 64 bf16 with silu: forward 271 us (4.0 TB/s of the
// 1.07 GB it has to move), backward 517 us (3.1 TB/s); the other kernel took 908
// and 2306. Neither a unit nor HBM is the limit but the steps' chains (copy, sums,
// merge, count, fold, write): larger slots (three of 64 KB instead of four of 48:
// 335 -> 290 us) help, fewer work warps (12 instead of 20) cost nothing, and a
// lag of two steps beyond what the sums need hides the folds (none: 435 us). The
// copies' L2 policies keep a chunk until its second reading (backward of a fourth
// of that size: 399 -> 271 MB read from HBM, of 268).
constexpr int kWorkWarps = 20, kMergeWarps = 4, kFoldWarps = 4;
constexpr int kWork = 32 * kWorkWarps;
constexpr int kRingThreads = kWork + 32 * (kMergeWarps + kFoldWarps + 1);
constexpr int kMaxSlots = 8, kRingGroups = 64;
constexpr int kRingSmem = 196608;     // bytes of the ring
constexpr int kSlack = 2;             // steps
// Least size of x, and the largest sample that goes to a cluster first. Measured,
// bf16 with silu, forward / backward, ring and other kernel: one sample of 1 MB (FP32)
// 13.6 / 14.4 and 16.4 / 14.3 us, of 2 MB 14.4 / 14.5 and 19.0 / 16.2; 32 samples of
// 128 KB 18.4 / 16.4 and (clusters) 10.3 / 10.7, 65 of 256 KB 23.5 / 26.7 and
// 20.3 / 24.6, 50 of 512 KB 26.7 / 34.9 and 38.4 / 48.5; 16357 of 8 KB 845 / 582 and
// 282 / 366: a step of the ring is a microsecond however little it holds.
constexpr double kRingBytes = 1e6, kClusterFirst = 262144.0;

struct RingParams {
  NormParams n;
  int slots, slot_bytes, resident;
};

struct RingShared {
  uint64_t full[kMaxSlots], empty[kMaxSlots], part[2], part_free[2], ready[2], ready_free[2];
  float2 sums[2][kWork];
  float2 stat1[kMaxSlots][kRingGroups];  // backward, phase 1: mean, rstd
  float4 stat2[2][kRingGroups];          // phase 2: mean, rstd, A, B
  int abort;
};

// The row loop of a phase, specialised for the activation.
template <typename F> __device__ __forceinline__ void with_act(int act, F&& f) {
  switch (act) {
    case DDPM_ACT_RELU: f(std::integral_constant<int, DDPM_ACT_RELU>()); break;
    case DDPM_ACT_SILU: f(std::integral_constant<int, DDPM_ACT_SILU>()); break;
    case DDPM_ACT_GELU: f(std::integral_constant<int, DDPM_ACT_GELU>()); break;
    case DDPM_ACT_GELU_TANH: f(std::integral_constant<int, DDPM_ACT_GELU_TANH>()); break;
    default: f(std::integral_constant<int, DDPM_ACT_NONE>());
  }
}

// A quad of channels as two pairs.
template <typename T> __device__ __forceinline__ void load4(const uint8_t* p, F2 (&v)[2]) {
  if constexpr (sizeof(T) == 4) {
    const float4 u = *reinterpret_cast<const float4*>(p);
    v[0] = f2(u.x, u.y);
    v[1] = f2(u.z, u.w);
  } else {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    const float2 a = unpack2<T>(u.x), b = unpack2<T>(u.y);
    v[0] = f2(a.x, a.y);
    v[1] = f2(b.x, b.y);
  }
}
template <typename T> __device__ __forceinline__ void store4(T* p, const F2 (&v)[2]) {
  const float2 a = split(v[0]), b = split(v[1]);
  if constexpr (sizeof(T) == 4)
    __stcs(reinterpret_cast<float4*>(p), make_float4(a.x, a.y, b.x, b.y));
  else
    __stcs(reinterpret_cast<uint2*>(p), make_uint2(pack2<T>(a.x, a.y), pack2<T>(b.x, b.y)));
}

// Bulk copy with an L2 policy: a chunk that is read again a few steps later is
// to stay, the second reading lets it go.
__device__ __forceinline__ void bulk_g2s_hint(void* dst, const void* src, uint32_t bytes,
                                              uint64_t* bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1], %2, [%3], %4;" ::"r"(tc::smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(tc::smem_u32(bar)), "l"(policy)
      : "memory");
}

// Warp-uniform bounded wait (the clock is read only in a long one).
__device__ __forceinline__ bool ring_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  bool ok = false;
  for (int i = 0; i < 64 && !ok; ++i) ok = tc::mbar_try_wait(bar, parity);
  if (!ok) {
    const uint64_t began = tc::globaltimer_ns();
    while (!(ok = tc::mbar_try_wait(bar, parity)))
      if (*abort_flag || tc::globaltimer_ns() - began > kWaitLimitNs) break;
  }
  return __all_sync(0xffffffffu, ok);
}

// Barrier of kCount threads that tells all of them whether any passed `bad`.
template <int kId, int kCount> __device__ __forceinline__ bool any_of(bool bad) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 q, %1, 0;\n\t"
      "bar.red.or.pred p, %2, %3, q;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)bad), "n"(kId), "n"(kCount)
      : "memory");
  return r != 0;
}

template <typename T, bool kBwd>
__global__ void __launch_bounds__(kRingThreads, 1) norm_ring_kernel(const RingParams rp) {
  constexpr bool kFast = sizeof(T) == 2;
  constexpr int kQuad = 4 * (int)sizeof(T);  // bytes of a thread's four channels
  const NormParams& p = rp.n;
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ RingShared sh;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  volatile int* abort_flag = &sh.abort;
  if (threadIdx.x == 0) {
    for (int i = 0; i < rp.slots; ++i) {
      tc::mbar_init(&sh.full[i], 1);
      tc::mbar_init(&sh.empty[i], kWorkWarps);
    }
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&sh.part[i], kWorkWarps);
      tc::mbar_init(&sh.part_free[i], kMergeWarps);
      tc::mbar_init(&sh.ready[i], kFoldWarps);
      tc::mbar_init(&sh.ready_free[i], kWorkWarps);
    }
    sh.abort = 0;
    tc::fence_mbar_init();
  }
  __syncthreads();

  const bool write = p.out != nullptr;  // the backward may want the sums only
  // steps this block has work in: its chunks are t = i * grid + block
  const int mine = ((int)p.chunks - 1 - (int)blockIdx.x) / (int)gridDim.x + 1;  // grid <= chunks
  const int steps = mine + (write ? p.lag : 0);
  auto fail = [&](int code) {
    if (lane == 0) {
      sh.abort = 1;
      atomicCAS(p.status, 0, code);
    }
  };

  if (warp == kWorkWarps + kMergeWarps + kFoldWarps) {  // ---- copies ----
    const bool lead = tc::elect_one();
    uint32_t q = 0;
    bool ok = true;
    int s = 0;             // the next slot, and the parity of its next copy
    uint32_t turn = 0;
    Walk first(p), second(p);
    uint64_t keep, drop;
    asm("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(keep));
    asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(drop));
    if (rp.resident || !write) keep = drop;  // read once
    auto fetch = [&](Walk& walk, uint64_t policy) {
      if (!ring_wait(&sh.empty[s], turn ^ 1, abort_flag)) {
        fail(102);
        ok = false;
        return;
      }
      const Chunk k = walk.next(p);
      const uint32_t bytes = (uint32_t)k.rows * p.C * sizeof(T);
      if (lead) {
        uint8_t* slot = ring + (size_t)s * rp.slot_bytes;
        const long long at = k.at * p.C * (long long)sizeof(T);
        tc::mbar_expect_tx(&sh.full[s], kBwd ? 2 * bytes : bytes);
        bulk_g2s_hint(slot, static_cast<const uint8_t*>(p.x) + at, bytes, &sh.full[s], policy);
        if constexpr (kBwd)
          bulk_g2s_hint(slot + rp.slot_bytes / 2, static_cast<const uint8_t*>(p.dy) + at, bytes,
                        &sh.full[s], policy);
      }
      if constexpr (kBwd) {
        for (int g = lane; g < p.G; g += 32) sh.stat1[s][g] = __ldg(&p.stats[(long long)k.n * p.G + g]);
      }
      __syncwarp();
      if (lead) tc::mbar_arrive(&sh.full[s]);
      ++q;
      if (++s == rp.slots) {
        s = 0;
        turn ^= 1;
      }
    };
    for (int i = 0; i < steps && ok; ++i) {
      if (i < mine) fetch(first, keep);
      if (ok && !rp.resident && write && i >= p.lag) fetch(second, drop);
    }
    if (!ok || *abort_flag) {  // what is in flight lands first
      const uint32_t n = q < (uint32_t)rp.slots ? q : (uint32_t)rp.slots;
      int never = 0;
      for (uint32_t j = q - n; j < q; ++j) ring_wait(&sh.full[j % rp.slots], (j / rp.slots) & 1, &never);
    }
  } else if (warp >= kWorkWarps + kMergeWarps) {  // ---- samples ----
    const int fw = warp - kWorkWarps - kMergeWarps;
    const unsigned all = (unsigned)p.S * kMergeWarps;
    Walk walk(p);
    int known = -1;  // the sample whose values are in the other buffer already
    for (int i = 0; write && i < mine; ++i) {
      const int b = i & 1;
      if (!ring_wait(&sh.ready_free[b], ((i >> 1) & 1) ^ 1, abort_flag)) {
        fail(97);
        break;
      }
      const bool mine_first = walk.s == 0;  // this block writes the sample's statistics
      const Chunk k = walk.next(p);
      if (k.n != known) {
        bool ok = true;
        if (load_acquire(&p.count[k.n]) != all) {
          const uint64_t began = tc::globaltimer_ns();
          while (load_acquire(&p.count[k.n]) != all) {
            __nanosleep(64);
            if (*abort_flag || tc::globaltimer_ns() - began > kWaitLimitNs) {
              ok = false;
              break;
            }
          }
        }
        if (!__all_sync(0xffffffffu, ok)) {
          fail(98);
          break;
        }
      }
      for (int g = fw; g < p.G; g += kFoldWarps) {
        float4 v;
        if (k.n == known) {
          v = sh.stat2[b ^ 1][g];
        } else if constexpr (kBwd) {
          const float2 st = __ldg(&p.stats[(long long)k.n * p.G + g]);
          const float2 ab = fold_sums(p, k.n, g, lane);
          v = make_float4(st.x, st.y, ab.x, ab.y);
        } else {
          const float2 st = fold_stats(p, k.n, g, lane);
          v = make_float4(st.x, st.y, 0.f, 0.f);
        }
        if (lane == 0) {
          sh.stat2[b][g] = v;
          if (!kBwd && mine_first) p.stats[(long long)k.n * p.G + g] = make_float2(v.x, v.y);
        }
      }
      known = k.n;
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&sh.ready[b]);
    }
  } else if (warp >= kWorkWarps) {  // ---- chunks ----
    const int fw = warp - kWorkWarps;
    const int per = p.cg / 4;  // columns of a group
    Walk walk(p);
    const bool pow2 = (per & (per - 1)) == 0;
    const int shift = __popc(per - 1);
    auto split = [&](int j, int& y, int& x) {  // entry of a group -> row, column
      y = pow2 ? j >> shift : j / per;
      x = j - y * per;
    };
    for (int i = 0; i < mine; ++i) {
      const int b = i & 1;
      if (!ring_wait(&sh.part[b], (i >> 1) & 1, abort_flag)) {
        fail(99);
        break;
      }
      const Chunk k = walk.next(p);
      const int full = (unsigned)k.rows / (unsigned)p.TY, rest = k.rows - full * p.TY;
      for (int g = fw; g < p.G; g += kMergeWarps) {
        const float2* base = sh.sums[b] + g * per;
        const int items = p.TY * per;
        float2 r;
        if constexpr (!kBwd) {
          const float m0 = base[0].x;  // sums about the first mean
          float s = 0.f, m2 = 0.f;
          for (int j = lane; j < items; j += 32) {
            int ty, cx;
            split(j, ty, cx);
            const float cnt = 4.f * (float)(full + (ty < rest));
            const float2 v = base[ty * p.TX + cx];
            if (cnt > 0.f) s += cnt * (v.x - m0);
          }
          const float mean = m0 + warp_sum(s) / ((float)k.rows * (float)p.cg);
          for (int j = lane; j < items; j += 32) {
            int ty, cx;
            split(j, ty, cx);
            const float cnt = 4.f * (float)(full + (ty < rest));
            const float2 v = base[ty * p.TX + cx];
            const float d = v.x - mean;
            if (cnt > 0.f) m2 += v.y + cnt * d * d;
          }
          r = make_float2(mean, warp_sum(m2));
        } else {
          float a = 0.f, c = 0.f;
          for (int j = lane; j < items; j += 32) {
            int ty, cx;
            split(j, ty, cx);
            const float2 v = base[ty * p.TX + cx];
            a += v.x;
            c += v.y;
          }
          r = make_float2(warp_sum(a), warp_sum(c));
        }
        if (lane == 0) p.part[((long long)i * gridDim.x + blockIdx.x) * p.G + g] = r;
      }
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&sh.part_free[b]);
      if (lane == 0) count_release(&p.count[k.n]);  // behind this lane's own partials
    }
  } else {  // ---- work ----
    const int tid = threadIdx.x;
    const int tx = tid % p.TX, ty = tid / p.TX;
    const bool live = ty < p.TY;
    const int c0 = tx * 4, g = live ? c0 / p.cg : 0;
    const int stride = p.TX * p.TY;  // quads between a thread's rows
    F2 w[2], bb[2], r1[2], r2[2];  // r1, r2: this block's sums of dz, dz * xhat
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      auto param = [&](const void* q, int c, float none) {
        return live && q ? load_param<T>(q, c, p.param_f32) : none;
      };
      w[e] = f2(param(p.weight, c0 + 2 * e, 1.f), param(p.weight, c0 + 2 * e + 1, 1.f));
      bb[e] = f2(param(p.bias, c0 + 2 * e, 0.f), param(p.bias, c0 + 2 * e + 1, 0.f));
      r1[e] = r2[e] = f2(0.f);
    }
    // the next slot to take (phase 1, and phase 2 where it has copies of its
    // own) and the slot of phase 2 where it is phase 1's
    int s1 = 0, s2 = 0;
    uint32_t turn = 0;
    Walk first(p), second(p);
    auto take = [&]() {
      if (++s1 == rp.slots) {
        s1 = 0;
        turn ^= 1;
      }
    };
    bool ok = true;
    for (int i = 0; i < steps && ok; ++i) {
      if (i < mine) {  // phase 1
        const int s = s1, b = i & 1;
        ok = ring_wait(&sh.full[s], turn, abort_flag) &&
             ring_wait(&sh.part_free[b], ((i >> 1) & 1) ^ 1, abort_flag);
        if (!ok) {
          fail(100);
          break;
        }
        const Chunk k = first.next(p);
        const uint8_t* slot = ring + (size_t)s * rp.slot_bytes;
        const int quads = k.rows * p.TX;
        if (live) {
          if constexpr (!kBwd) {
            float s0 = 0.f;
            if (tid < quads) {
              F2 v[2];
              load4<T>(slot + (size_t)tid * kQuad, v);
              s0 = split(v[0]).x;
            }
            const F2 less = f2(-s0);
            F2 a1[2] = {f2(0.f), f2(0.f)}, a2[2] = {f2(0.f), f2(0.f)};
            int count = 0;
#pragma unroll 4
            for (int j = tid; j < quads; j += stride) {
              F2 v[2];
              load4<T>(slot + (size_t)j * kQuad, v);
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const F2 d = v[e] + less;
                a1[e] = a1[e] + d;
                a2[e] = fma2(d, d, a2[e]);
              }
              count += 4;
            }
            const float2 t1 = split(a1[0] + a1[1]), t2 = split(a2[0] + a2[1]);
            const float sum = t1.x + t1.y;
            const float m = sum / (float)(count ? count : 1);
            sh.sums[b][tid] = make_float2(s0 + m, fmaxf(t2.x + t2.y - sum * m, 0.f));
          } else {
            const float2 st = sh.stat1[s][g];
            const F2 less = f2(-st.x), rstd = f2(st.y);
            F2 c1[2] = {f2(0.f), f2(0.f)}, c2[2] = {f2(0.f), f2(0.f)};
            with_act(p.act, [&](auto A) {
#pragma unroll 2
              for (int j = tid; j < quads; j += stride) {
                F2 x[2], d[2];
                load4<T>(slot + (size_t)j * kQuad, x);
                load4<T>(slot + rp.slot_bytes / 2 + (size_t)j * kQuad, d);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const F2 xh = (x[e] + less) * rstd;
                  const F2 dz = d[e] * act_slope<kFast, A.value>(fma2(xh, w[e], bb[e]));
                  c1[e] = c1[e] + dz;
                  c2[e] = fma2(dz, xh, c2[e]);
                }
              }
            });
            const float2 ta = split(fma2(w[0], c1[0], w[1] * c1[1]));
            const float2 tb = split(fma2(w[0], c2[0], w[1] * c2[1]));
            sh.sums[b][tid] = make_float2(ta.x + ta.y, tb.x + tb.y);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              r1[e] = r1[e] + c1[e];
              r2[e] = r2[e] + c2[e];
            }
          }
        }
        __syncwarp();
        if (lane == 0) {
          tc::mbar_arrive(&sh.part[b]);
          if (!rp.resident || !write) tc::mbar_arrive(&sh.empty[s]);
        }
        take();
      }
      if (write && i >= p.lag) {  // phase 2
        const int i2 = i - p.lag;
        const int b = i2 & 1;
        int s;
        if (rp.resident) {
          s = s2;
          if (++s2 == rp.slots) s2 = 0;
        } else {
          s = s1;
          ok = ring_wait(&sh.full[s], turn, abort_flag);
          take();
        }
        ok = ok && ring_wait(&sh.ready[b], (i2 >> 1) & 1, abort_flag);
        if (!ok) {
          fail(101);
          break;
        }
        const Chunk k = second.next(p);
        const uint8_t* slot = ring + (size_t)s * rp.slot_bytes;
        const int quads = k.rows * p.TX;
        if (live) {
          const float4 st = sh.stat2[b][g];
          T* out = static_cast<T*>(p.out) + k.at * p.C;
          const F2 less = f2(-st.x), rstd = f2(st.y);
          const F2 wr[2] = {w[0] * rstd, w[1] * rstd};
          if constexpr (!kBwd) {
            with_act(p.act, [&](auto A) {
#pragma unroll 2
              for (int j = tid; j < quads; j += stride) {
                F2 v[2];
                load4<T>(slot + (size_t)j * kQuad, v);
#pragma unroll
                for (int e = 0; e < 2; ++e)
                  v[e] = act_value<kFast, A.value>(fma2(v[e] + less, wr[e], bb[e]));
                store4<T>(out + (size_t)j * 4, v);
              }
            });
          } else {
            const F2 na = f2(-st.y * st.z), nb = f2(-st.y * st.w);
            with_act(p.act, [&](auto A) {
#pragma unroll 2
              for (int j = tid; j < quads; j += stride) {
                F2 x[2], d[2];
                load4<T>(slot + (size_t)j * kQuad, x);
                load4<T>(slot + rp.slot_bytes / 2 + (size_t)j * kQuad, d);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const F2 xh = (x[e] + less) * rstd;
                  const F2 dz = d[e] * act_slope<kFast, A.value>(fma2(xh, w[e], bb[e]));
                  x[e] = fma2(dz, wr[e], fma2(xh, nb, na));
                }
                store4<T>(out + (size_t)j * 4, x);
              }
            });
          }
        }
        __syncwarp();
        if (lane == 0) {
          tc::mbar_arrive(&sh.ready_free[b]);
          tc::mbar_arrive(&sh.empty[s]);
        }
      }
    }
    if constexpr (kBwd) {
      // the block's sums of a channel, its rows folded in order (the ring is
      // free: every copy has been waited for)
      if (p.wsum != nullptr && !any_of<2, kWork>(!ok)) {
        float2* run = reinterpret_cast<float2*>(ring);
        if (live) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float2 u = split(r1[e]), v = split(r2[e]);
            run[ty * p.C + c0 + 2 * e] = make_float2(u.x, v.x);
            run[ty * p.C + c0 + 2 * e + 1] = make_float2(u.y, v.y);
          }
        }
        asm volatile("bar.sync 2, %0;" ::"n"(kWork) : "memory");
        for (int c = tid; c < p.C; c += kWork) {
          float2 a = make_float2(0.f, 0.f);
          for (int y = 0; y < p.TY; ++y) {
            const float2 v = run[y * p.C + c];
            a.x += v.x;
            a.y += v.y;
          }
          p.wsum[(long long)blockIdx.x * p.C + c] = a;
        }
      }
    }
  }
}

// ------------------------------------------------------------------ plan ----
struct Plan {
  bool ring, cluster;
  int slots, slot_bytes, resident;
  int V, CT, TX, TY, U, uw, R, S, grid, lag;
  long long chunks;
  size_t part_off, grp_off, wsum_off, count_off, total;
};

int gcd_pow2(long long v, int most) {  // largest power of two <= most that divides v
  int r = most;
  while (v % r) r >>= 1;
  return r;
}

// Workspace layout of a plan.
void place(Plan* q, long long n, int G, int C, bool bwd) {
  auto up = [](size_t v) { return (v + 255) / 256 * 256; };
  q->count_off = q->part_off = q->grp_off = q->wsum_off = 0;
  if (!q->cluster) {
    q->part_off = up((size_t)n * 8);
    q->grp_off = q->part_off + up((size_t)n * q->S * q->U * 8);
    q->wsum_off = q->grp_off + (bwd ? up((size_t)n * G * 8) : 0);
  }
  q->total = q->wsum_off + (bwd ? up((size_t)(q->grid / q->CT) * C * 8) : 0);
}

// The ring kernel's plan, where it applies: rows of whole 16-byte words, groups
// of whole quads, and enough data to fill its pipeline.
bool plan_ring(Plan* q, long long n, long long P, int C, int G, int es, bool bwd, int align) {
  if (align * es < 16 || C * es % 16 || C / G % 4 || C / 4 > kWork || G > kRingGroups) return false;
  const int grid = gencat::num_sms();
  const double bytes = (double)n * P * C * es;
  if (bytes < kRingBytes) return false;
  const long long row = (long long)C * es;
  // A chunk is a slot's worth of pixels, fewer where that evens out the blocks.
  const int slots = 3;
  const int slot = kRingSmem / slots / 256 * 256;
  long long r = slot / (bwd ? 2 : 1) / row;
  if (r < 1) return false;
  const long long even = (n * P + grid - 1) / grid;
  const long long steps = (even + r - 1) / r;
  r = (even + steps - 1) / steps;
  if (r > P) r = P;
  const long long s = (P + r - 1) / r;
  if (n * s >= (1LL << 28)) return false;
  q->ring = true;
  q->slots = slots;
  q->slot_bytes = slot;
  q->V = 4;
  q->CT = 1;
  q->TX = C / 4;
  q->TY = kWork / q->TX;
  q->U = G;
  q->uw = C / G;
  q->R = (int)r;
  q->S = (int)s;
  q->chunks = n * s;
  q->grid = (int)(q->chunks < grid ? q->chunks : grid);
  q->lag = (int)((s - 1 + q->grid - 1) / q->grid);
  // more steps than the sums need: the folds' latency is then nobody's wait
  if (s > 1) q->lag += kSlack;
  q->resident = q->lag <= slots - 2;
  return true;
}

// Columns of a block of the other kernels.
void plan_tile(Plan* q, int C, int G, int align) {
  // four channels a thread: eight spill (80 registers, three blocks an SM)
  q->V = gcd_pow2(C, align < 4 ? align : 4);
  const int cols = C / q->V;
  q->CT = (cols + kThreads - 1) / kThreads;
  q->TX = (cols + q->CT - 1) / q->CT;
  q->CT = (cols + q->TX - 1) / q->TX;
  q->TY = kThreads / q->TX;
  q->U = q->CT == 1 ? G : C;
  q->uw = q->CT == 1 ? C / G : 1;
}

// Small samples: a cluster each (a single block that takes several in turn where
// there are many), at least a row of pixels for every thread row and at most 64 KB
// of x a block: 16 x 16 x 64 FP32 forward 9.0 -> 7.5 us, and two calls fewer on the
// host. (One sample of 512 KB, so at that limit: 17.2 us forward, 19.4 backward, the
// blocks that wait for one another 14.4 and 12.4; eight of them 17.4 and 19.5, and
// 19.0 and 16.5; fifty 38 and 48, and 50 and 56.)
bool plan_cluster(Plan* q, long long n, long long P, int C, int es) {
  if (q->CT != 1) return false;
  const int blocks = 3 * gencat::num_sms();
  for (int cl = 8; cl >= 1; cl /= 2) {
    const long long r = (P + cl - 1) / cl;
    if (cl > 1 && ((cl - 1) * r >= P || n * cl > blocks || r < q->TY)) continue;
    if ((double)r * C * es > 65536.0) break;
    q->cluster = true;
    q->R = (int)r;
    q->S = cl;
    q->chunks = n * cl;
    q->grid = (int)(q->chunks < blocks ? q->chunks : blocks);
    q->lag = 0;
    return true;
  }
  return false;
}

// `align`: the largest power of two (in elements, at most 16 bytes' worth)
// that divides every tensor's address.
int make_plan(Plan* q, long long n, long long P, int C, int G, int dt, bool bwd, int align) {
  const int es = dtype_size(dt);
  Plan tile{}, ring{};
  plan_tile(&tile, C, G, align);
  const bool cluster = plan_cluster(&tile, n, P, C, es);
  const bool first = cluster && (double)P * C * es <= kClusterFirst;
  *q = !first && plan_ring(&ring, n, P, C, G, es, bwd, align) ? ring : tile;
  if (q->ring || cluster) {
    place(q, n, G, C, bwd);
    return DDPM_OK;
  }
  // Two (backward) or three (forward) blocks an SM are resident by the launch
  // bounds; the launch checks it.
  const int most = gencat::num_sms() * (bwd ? 2 : 3) / q->CT * q->CT;
  // Pixels of a chunk: about 48 KB of x (24 KB in the backward, which moves
  // twice as much), fewer when that leaves blocks without work, at least two
  // a thread.
  const long long row_bytes = (long long)q->TX * q->V * es;
  const long long big = (bwd ? 24576 : 49152) / row_bytes;
  long long even = (n * P * q->CT + most - 1) / most;
  long long r = even < big ? even : big;
  if (r < 2 * q->TY) r = 2 * q->TY;
  r = (r + q->TY - 1) / q->TY * q->TY;
  if (r > P) r = P;
  q->R = (int)r;
  const long long s = (P + r - 1) / r;
  q->chunks = n * s * q->CT;
  if (q->chunks >= (1LL << 31) || s * q->CT >= (1LL << 31))
    return set_error(DDPM_ERR_UNSUPPORTED, "group norm: too many chunks");
  q->S = (int)s;
  q->grid = (int)(q->chunks < most ? q->chunks : most);
  q->lag = (int)((s * q->CT - 1 + q->grid - 1) / q->grid);
  place(q, n, G, C, bwd);
  return DDPM_OK;
}

int check_norm(long long n, long long P, int C, int G, int dt, int pdt, int act) {
  DDPM_CHECK_ARG(n >= 0 && P >= 0 && C >= 1, "sizes must not be negative, channels positive");
  DDPM_CHECK_ARG(G >= 1 && C % G == 0, "num_groups %d does not divide %d channels", G, C);
  DDPM_CHECK_ARG(dtype_size(dt) > 0, "unknown dtype code %d", dt);
  DDPM_CHECK_ARG(pdt == dt || pdt == DDPM_F32, "weight and bias must have x's dtype or be fp32");
  DDPM_CHECK_ARG(act_known(act), "unknown activation code %d", act);
  DDPM_CHECK_ARG(n < (1LL << 31) && P < (1LL << 31) && (double)n * P * C < 4e18,
                 "too many samples or pixels");
  if (C > kMaxChannels)
    return set_error(DDPM_ERR_UNSUPPORTED, "group norm supports C <= %d (got %d)", kMaxChannels, C);
  return DDPM_OK;
}

template <typename T, int V, bool kBwd>
int launch_norm(const NormParams& p, const Plan& q, cudaStream_t st) {
  if (q.cluster) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(q.grid);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = st;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = q.S;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    DDPM_CUDA_TRY(cudaLaunchKernelEx(&cfg, norm_kernel<T, V, kBwd, true>, p));
    DDPM_CHECK_LAUNCH(kBwd ? "group_norm_bwd_kernel" : "group_norm_fwd_kernel");
    return DDPM_OK;
  }
  auto fn = norm_kernel<T, V, kBwd, false>;
  if (q.S * q.CT > 1 && q.grid > 1) {
    // blocks wait for one another: all of them have to be resident
    NormParams arg = p;
    void* args[] = {&arg};
    DDPM_CUDA_TRY(cudaLaunchCooperativeKernel(reinterpret_cast<const void*>(fn), dim3(q.grid),
                                              dim3(kThreads), args, 0, st));
  } else {
    fn<<<q.grid, kThreads, 0, st>>>(p);
  }
  DDPM_CHECK_LAUNCH(kBwd ? "group_norm_bwd_kernel" : "group_norm_fwd_kernel");
  return DDPM_OK;
}

template <typename T, bool kBwd>
int launch_ring(const NormParams& p, const Plan& q, cudaStream_t st) {
  auto fn = norm_ring_kernel<T, kBwd>;
  static std::atomic<unsigned long long> ready{0};  // devices whose limit is raised
  int dev = 0;
  DDPM_CUDA_TRY(cudaGetDevice(&dev));
  if (dev >= 64 || !(ready.load(std::memory_order_relaxed) >> dev & 1)) {
    DDPM_CUDA_TRY(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingSmem));
    if (dev < 64) ready.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  RingParams arg{p, q.slots, q.slot_bytes, q.resident};
  void* args[] = {&arg};
  if (q.S > 1) {
    DDPM_CUDA_TRY(cudaLaunchCooperativeKernel(reinterpret_cast<const void*>(fn), dim3(q.grid),
                                              dim3(kRingThreads), args, (size_t)kRingSmem, st));
  } else {
    fn<<<q.grid, kRingThreads, kRingSmem, st>>>(arg);
  }
  DDPM_CHECK_LAUNCH(kBwd ? "group_norm_bwd_kernel" : "group_norm_fwd_kernel");
  return DDPM_OK;
}

template <typename T, bool kBwd>
int dispatch_norm(const NormParams& p, const Plan& q, cudaStream_t st) {
  if (q.ring) return launch_ring<T, kBwd>(p, q, st);
  switch (q.V) {
    case 4: return launch_norm<T, 4, kBwd>(p, q, st);
    case 2: return launch_norm<T, 2, kBwd>(p, q, st);
    default: return launch_norm<T, 1, kBwd>(p, q, st);
  }
}

int alignment(uintptr_t at, int es) {
  int v = 16 / es;
  while (at % ((uintptr_t)v * es)) v >>= 1;
  return v;
}

int run_norm(bool bwd, const void* x, const void* dy, const void* w, const void* b, void* out,
             void* stats, void* gw, void* gb, void* ws, size_t ws_bytes, long long n, long long P,
             int C, int G, float eps, int act, int dt, int pdt, cudaStream_t st) {
  int rc = check_norm(n, P, C, G, dt, pdt, act);
  if (rc) return rc;
  if (n == 0 || P == 0) return DDPM_OK;
  DDPM_CHECK_ARG(x && stats && (bwd ? dy != nullptr : out != nullptr), "null pointer");
  const int es = dtype_size(dt);
  const uintptr_t at = (uintptr_t)x | (uintptr_t)dy | (uintptr_t)out;
  DDPM_CHECK_ARG(at % es == 0 && (uintptr_t)stats % 8 == 0 && (uintptr_t)ws % 256 == 0,
                 "misaligned pointer");
  Plan q;
  rc = make_plan(&q, n, P, C, G, dt, bwd, alignment(at, es));
  if (rc) return rc;
  if (ws_bytes < q.total || (q.total > 0 && ws == nullptr))
    return set_error(DDPM_ERR_WORKSPACE, "group norm workspace: %zu bytes needed, %zu given",
                     q.total, ws_bytes);
  uint8_t* base = static_cast<uint8_t*>(ws);
  NormParams p{};
  p.x = x;
  p.dy = dy;
  p.weight = w;
  p.bias = b;
  p.out = out;
  p.stats = static_cast<float2*>(stats);
  p.part = reinterpret_cast<float2*>(base + q.part_off);
  p.grp = reinterpret_cast<float2*>(base + q.grp_off);
  p.wsum = bwd && (gw || gb) ? reinterpret_cast<float2*>(base + q.wsum_off) : nullptr;
  p.count = reinterpret_cast<unsigned*>(base + q.count_off);
  rc = gencat::status_ptr(&p.status);
  if (rc) return rc;
  p.P = P;
  p.N = (int)n;
  p.C = C;
  p.G = G;
  p.cg = C / G;
  p.R = q.R;
  p.S = q.S;
  p.CT = q.CT;
  p.TX = q.TX;
  p.TY = q.TY;
  p.U = q.U;
  p.uw = q.uw;
  p.chunks = q.chunks;
  p.lag = q.lag;
  p.act = act;
  p.param_f32 = pdt == DDPM_F32;
  p.eps = eps;
  if (!q.cluster) DDPM_CUDA_TRY(cudaMemsetAsync(p.count, 0, (size_t)n * 8, st));
  switch (dt) {
    case DDPM_F32:
      rc = bwd ? dispatch_norm<float, true>(p, q, st) : dispatch_norm<float, false>(p, q, st);
      break;
    case DDPM_BF16:
      rc = bwd ? dispatch_norm<__nv_bfloat16, true>(p, q, st)
               : dispatch_norm<__nv_bfloat16, false>(p, q, st);
      break;
    default:
      rc = bwd ? dispatch_norm<__half, true>(p, q, st) : dispatch_norm<__half, false>(p, q, st);
  }
  if (rc || !p.wsum) return rc;
  const int blocks = (C + 31) / 32, rows = q.grid / q.CT;
  switch (pdt) {
    case DDPM_F32:
      norm_param_kernel<<<blocks, 256, 0, st>>>(p.wsum, rows, C, (float*)gw, (float*)gb);
      break;
    case DDPM_BF16:
      norm_param_kernel<<<blocks, 256, 0, st>>>(p.wsum, rows, C, (__nv_bfloat16*)gw,
                                                (__nv_bfloat16*)gb);
      break;
    default:
      norm_param_kernel<<<blocks, 256, 0, st>>>(p.wsum, rows, C, (__half*)gw, (__half*)gb);
  }
  DDPM_CHECK_LAUNCH("group_norm_param_kernel");
  return DDPM_OK;
}

}  // namespace

// With `aligned` 0: the largest workspace any alignment of the tensors asks for.
size_t group_norm_workspace_bytes(long long n, long long P, int C, int G, int dt, int bwd,
                                  int aligned) {
  if (n <= 0 || P <= 0 || C < 1 || G < 1 || C % G || C > kMaxChannels ||
      dtype_size(dt) == 0 || n >= (1LL << 31) || P >= (1LL << 31))
    return 0;
  size_t most = 0;
  const int widest = 16 / dtype_size(dt);
  for (int align = widest; align >= (aligned ? widest : 1); align >>= 1) {
    Plan q;
    if (make_plan(&q, n, P, C, G, dt, bwd != 0, align) == DDPM_OK && q.total > most)
      most = q.total;
  }
  return most;
}

int group_norm_fwd(const void* x, const void* w, const void* b, void* out, void* stats, void* ws,
                   size_t ws_bytes, long long n, long long P, int C, int G, float eps, int act,
                   int dt, int pdt, cudaStream_t st) {
  return run_norm(false, x, nullptr, w, b, out, stats, nullptr, nullptr, ws, ws_bytes, n, P, C, G,
                  eps, act, dt, pdt, st);
}

int group_norm_bwd(const void* x, const void* dy, const void* w, const void* b, const void* stats,
                   void* gx, void* gw, void* gb, void* ws, size_t ws_bytes, long long n,
                   long long P, int C, int G, int act, int dt, int pdt, cudaStream_t st) {
  return run_norm(true, x, dy, w, b, gx, const_cast<void*>(stats), gw, gb, ws, ws_bytes, n, P, C,
                  G, 0.f, act, dt, pdt, st);
}

}  // namespace ddpm
