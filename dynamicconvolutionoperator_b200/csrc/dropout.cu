// Dropout from a counter-based generator; the mask is never stored.
//
//   out[i] = keep(offset + i) ? x[i] * (1 / (1 - p)) (+ residual[i]) : (residual[i] or 0)
//   keep(q) = philox4x32_10(counter = (q / 4, 0), key = seed)[q % 4] >= round(p * 2^32)
//
// The generator is Philox-4x32 with ten rounds (Salmon, Moraes, Dror and Shaw,
// "Parallel random numbers: as easy as 1, 2, 3", 2011): a pure function of the
// position and the seed, so the backward pass calls the same kernel on the
// gradient, and a tensor cut in pieces draws the same mask as the whole.
//
// A dropped value is selected away, not multiplied by zero: an infinity or NaN
// in a dropped place does not reach the output. The product and the residual's
// sum are formed in FP32 and rounded once.
//
// Bound: HBM (2 or 3 values moved for each one made), with the generator's
// integer multiplies close behind for 16-bit data: 20 32x32->64-bit products
// per four values. Hence one Philox block serves four neighbouring values and
// a thread handles 16 bytes (one or two blocks) per step.
//
// Measured, 268M values: bf16 264 us (4.1 TB/s; the pipe of the wide multiplies is
// 80 % busy, and neither more resident warps nor a longer grid changes it), with a
// residual 284 us (5.7 TB/s), FP32 402 us (5.3 TB/s; a copy: 329 us). An offset
// that is no multiple of four: 405 us.
#include "act.cuh"
#include "common.cuh"

namespace ddpm {

namespace gencat {
int num_sms();
}  // namespace gencat

namespace {

struct DropParams {
  const void* x;
  const void* res;       // nullable
  void* out;
  long long n;
  unsigned long long seed;
  const unsigned long long* seed_ptr;  // nullable: read on the device instead of `seed`
  unsigned long long offset;
  uint32_t threshold;    // keep iff word >= threshold
  float scale;
};

__device__ __forceinline__ void philox(uint64_t block, uint32_t k0, uint32_t k1,
                                       uint32_t (&w)[4]) {
  uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = 0, c3 = 0;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = (uint64_t)0xD2511F53u * c0;
    const uint64_t p1 = (uint64_t)0xCD9E8D57u * c2;
    c0 = (uint32_t)(p1 >> 32) ^ c1 ^ (k0 + (uint32_t)r * 0x9E3779B9u);
    c1 = (uint32_t)p1;
    c2 = (uint32_t)(p0 >> 32) ^ c3 ^ (k1 + (uint32_t)r * 0xBB67AE85u);
    c3 = (uint32_t)p0;
  }
  w[0] = c0; w[1] = c1; w[2] = c2; w[3] = c3;
}

template <bool kAll>
__device__ __forceinline__ float drop_one(const DropParams& p, uint32_t word, float x) {
  return !kAll && word >= p.threshold ? x * p.scale : 0.f;
}

// Aligned form: offset % 4 == 0 and every pointer on a 16-byte boundary. A
// thread handles kVec = 16 / sizeof(T) values (one or two generator blocks).
// kAll: p is 1.
template <typename T, bool kRes, bool kAll>
__global__ void __launch_bounds__(256) dropout_vec_kernel(const DropParams p) {
  constexpr int kVec = 16 / (int)sizeof(T);
  const uint64_t seed = p.seed_ptr ? *p.seed_ptr : p.seed;
  const uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
  const uint4* x = static_cast<const uint4*>(p.x);
  const uint4* res = static_cast<const uint4*>(p.res);
  uint4* out = static_cast<uint4*>(p.out);
  const long long nvec = p.n / kVec;
  const long long step = (long long)gridDim.x * blockDim.x;
  const uint64_t b0 = p.offset >> 2;
  const F2 scale = f2(p.scale);
  for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < nvec; i += step) {
    float v[kVec], r[kVec];
    unpack16<T>(__ldcs(x + i), v);
    if constexpr (kRes) unpack16<T>(__ldcs(res + i), r);
    uint32_t w[kVec / 4][4];
    if constexpr (!kAll) {
#pragma unroll
      for (int q = 0; q < kVec / 4; ++q) philox(b0 + (uint64_t)i * (kVec / 4) + q, k0, k1, w[q]);
    }
#pragma unroll
    for (int e = 0; e < kVec; e += 2) {
      const float2 y = split(f2(v[e], v[e + 1]) * scale);
      v[e] = !kAll && w[e / 4][e % 4] >= p.threshold ? y.x : 0.f;
      v[e + 1] = !kAll && w[e / 4][e % 4 + 1] >= p.threshold ? y.y : 0.f;
      if constexpr (kRes) {
        const float2 z = split(f2(v[e], v[e + 1]) + f2(r[e], r[e + 1]));
        v[e] = z.x;
        v[e + 1] = z.y;
      }
    }
    __stcs(out + i, pack16<T>(v));
  }
  // the last n % kVec values: the first threads of block 0 take one each
  const long long i = nvec * kVec + threadIdx.x;
  if (blockIdx.x == 0 && i < p.n) {
    uint32_t w[4];
    philox(b0 + (uint64_t)(i >> 2), k0, k1, w);
    float y = drop_one<kAll>(p, w[i & 3], to_f32<T>(static_cast<const T*>(p.x)[i]));
    if constexpr (kRes) y += to_f32<T>(static_cast<const T*>(p.res)[i]);
    static_cast<T*>(p.out)[i] = from_f32<T>(y);
  }
}

// Any offset and alignment: a thread handles the (at most four) values of one
// generator block.
template <typename T, bool kRes, bool kAll>
__global__ void __launch_bounds__(256) dropout_any_kernel(const DropParams p) {
  const uint64_t seed = p.seed_ptr ? *p.seed_ptr : p.seed;
  const uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
  const T* x = static_cast<const T*>(p.x);
  const T* res = static_cast<const T*>(p.res);
  T* out = static_cast<T*>(p.out);
  const int lead = (int)(p.offset & 3);  // lanes of the first block before position `offset`
  const long long nblk = (p.n + lead + 3) / 4;
  const long long step = (long long)gridDim.x * blockDim.x;
  for (long long b = blockIdx.x * (long long)blockDim.x + threadIdx.x; b < nblk; b += step) {
    const long long i0 = b * 4 - lead;
    float v[4], r[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool in = i0 + e >= 0 && i0 + e < p.n;
      v[e] = in ? to_f32<T>(x[i0 + e]) : 0.f;
      if constexpr (kRes) r[e] = in ? to_f32<T>(res[i0 + e]) : 0.f;
    }
    uint32_t w[4];
    philox((p.offset >> 2) + (uint64_t)b, k0, k1, w);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float y = drop_one<kAll>(p, w[e], v[e]);
      if constexpr (kRes) y += r[e];
      if (i0 + e >= 0 && i0 + e < p.n) out[i0 + e] = from_f32<T>(y);
    }
  }
}

template <typename T, bool kRes, bool kAll>
int launch_dropout_as(const DropParams& p, bool vec, cudaStream_t st) {
  const long long items = vec ? (p.n + 16 / sizeof(T) - 1) / (16 / sizeof(T)) : (p.n + 6) / 4;
  const long long most = gencat::num_sms() * 32LL;  // four rounds of eight blocks an SM
  const long long want = (items + 255) / 256;
  const int grid = (int)(want < most ? want : most);
  if (vec) dropout_vec_kernel<T, kRes, kAll><<<grid, 256, 0, st>>>(p);
  else dropout_any_kernel<T, kRes, kAll><<<grid, 256, 0, st>>>(p);
  DDPM_CHECK_LAUNCH("dropout_kernel");
  return DDPM_OK;
}

template <typename T> int launch_dropout(const DropParams& p, bool all, bool vec, cudaStream_t st) {
  if (all)
    return p.res ? launch_dropout_as<T, true, true>(p, vec, st)
                 : launch_dropout_as<T, false, true>(p, vec, st);
  return p.res ? launch_dropout_as<T, true, false>(p, vec, st)
               : launch_dropout_as<T, false, false>(p, vec, st);
}

}  // namespace

int dropout(const void* x, const void* residual, void* out, long long n, double p,
            unsigned long long seed, const void* seed_ptr, unsigned long long offset, int dt,
            cudaStream_t st) {
  DDPM_CHECK_ARG(n >= 0, "size must not be negative");
  DDPM_CHECK_ARG(p >= 0.0 && p <= 1.0, "p must be between 0 and 1, got %g", p);
  DDPM_CHECK_ARG(dtype_size(dt) > 0, "unknown dtype code %d", dt);
  if (n == 0) return DDPM_OK;
  DDPM_CHECK_ARG(offset <= UINT64_MAX - (unsigned long long)(n - 1),
                 "the positions must fit 64 bits, got offset %llu", offset);
  DDPM_CHECK_ARG(x && out, "null pointer");
  const uintptr_t es = (uintptr_t)dtype_size(dt);
  const uintptr_t at = (uintptr_t)x | (uintptr_t)residual | (uintptr_t)out;
  DDPM_CHECK_ARG(at % es == 0 && (uintptr_t)seed_ptr % 8 == 0, "misaligned pointer");
  DropParams q{};
  q.x = x;
  q.res = residual;
  q.out = out;
  q.n = n;
  q.seed = seed;
  q.seed_ptr = static_cast<const unsigned long long*>(seed_ptr);
  q.offset = offset;
  const double t = p * 4294967296.0 + 0.5;  // floor(t) = round(p * 2^32)
  const bool all = t >= 4294967296.0;
  q.threshold = all ? 0xFFFFFFFFu : (uint32_t)t;
  q.scale = p < 1.0 ? (float)(1.0 / (1.0 - p)) : 0.f;
  const bool vec = at % 16 == 0 && offset % 4 == 0;
  switch (dt) {
    case DDPM_F32: return launch_dropout<float>(q, all, vec, st);
    case DDPM_BF16: return launch_dropout<__nv_bfloat16>(q, all, vec, st);
    default: return launch_dropout<__half>(q, all, vec, st);
  }
}

}  // namespace ddpm
