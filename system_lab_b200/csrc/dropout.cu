// Dropout whose mask is a function of (seed, offset, element) and is never stored, with an optional residual:
//
//   y_e = keep_e x_e / (1 - p') + r_e,   keep_e = bits_e >= t,   t = round(65536 p),   p' = t / 65536
//
// bits_e: 16 of the 128 bits that Philox-4x32 with ten rounds (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as
// easy as 1, 2, 3", 2011) makes of key `seed` and counter (e / 8, offset): element e takes half e % 2 of word (e % 8) / 2.
// Sixteen bits keep an element's share of the ten rounds small (one block of the generator for eight elements) and set p to
// within 2^-17; the kept elements are scaled by the probability as it is then, so the mean is exact.  The gradient is the
// same kernel on dy without the residual.  x, r and y move once; bf16 is bound by its instructions (155 for eight elements, the
// rounds' 20 wide products among them) nearly as much as by memory: 8192 x 8192 in 46.3 us, 5.8 TB/s, with a residual 4096 x
// 8192 in 33.1, 6.1 TB/s.
#include "common.cuh"

namespace slab {

__device__ __forceinline__ uint4 philox(uint4 c, uint2 k) {
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t a = (uint64_t)0xD2511F53u * c.x, b = (uint64_t)0xCD9E8D57u * c.z;
    c = make_uint4((uint32_t)(b >> 32) ^ c.y ^ k.x, (uint32_t)b, (uint32_t)(a >> 32) ^ c.w ^ k.y, (uint32_t)a);
    k.x += 0x9E3779B9u;
    k.y += 0xBB67AE85u;
  }
  return c;
}

// Eight elements as they are in memory: loaded first, made numbers only behind the generator's rounds (converted where they were
// loaded, beside the branch for the tensor's end, every warp waited for memory before its rounds: 8192 x 8192 bf16, 55.8 us)
template <typename T>
struct DrRaw;
template <>
struct DrRaw<__nv_bfloat16> {
  uint4 v;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { v = __ldg(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ void load(const __nv_bfloat16* p, long left) {
    const unsigned short* b = reinterpret_cast<const unsigned short*>(p);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = (2 * i < left ? (uint32_t)b[2 * i] : 0u) | (2 * i + 1 < left ? (uint32_t)b[2 * i + 1] << 16 : 0u);
    v = make_uint4(w[0], w[1], w[2], w[3]);
  }
  __device__ __forceinline__ void get(float (&f)[8]) const { unpack8(*reinterpret_cast<const bf16x8*>(&v), f); }
};
template <>
struct DrRaw<float> {
  float v[8];
  __device__ __forceinline__ void load(const float* p) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
  __device__ __forceinline__ void load(const float* p, long left) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < left ? p[i] : 0.f;
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = v[i];
  }
};
__device__ __forceinline__ void dr_store(__nv_bfloat16* p, const float (&f)[8]) { *reinterpret_cast<bf16x8*>(p) = pack8(f); }
__device__ __forceinline__ void dr_store(float* p, const float (&f)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
}
__device__ __forceinline__ void dr_put(__nv_bfloat16* p, float v) { *p = __float2bfloat16(v); }
__device__ __forceinline__ void dr_put(float* p, float v) { *p = v; }

constexpr int DR_THREADS = 256;
constexpr long DR_MANY = 4l << 20;           // from so many bf16 elements on a thread takes DR_BLOCKS blocks of eight, whose loads and rounds
constexpr int DR_BLOCKS = 4;                 // overlap: 8192 x 8192 46.3 us, one each 59 (four million the same, 77 x 2880 3.0, one each 2.3).
                                             // fp32, which moves twice the bytes per round, takes one: 4099 x 5762 30.5, four each 32.5

// t: threshold << 16; NB: blocks of eight elements per thread
template <typename T, bool RES, int NB>
__global__ void __launch_bounds__(DR_THREADS)
dropout_kernel(const T* __restrict__ x, const T* __restrict__ res, T* __restrict__ y, long n, uint32_t t, float scale, uint64_t seed,
               const long long* __restrict__ seed_dev, uint64_t offset) {
  const long g0 = (long)blockIdx.x * (DR_THREADS * NB) + threadIdx.x;
  DrRaw<T> xs[NB], rs[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const long e = (g0 + b * DR_THREADS) * 8;
    if (e + 8 <= n) {
      xs[b].load(x + e);
      if (RES) rs[b].load(res + e);
    } else {
      xs[b].load(x + e, n - e);
      if (RES) rs[b].load(res + e, n - e);
    }
  }
  const uint64_t key = seed_dev ? (uint64_t)*seed_dev : seed;
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const long g = g0 + b * DR_THREADS, e = g * 8;
    const uint4 w = philox(make_uint4((uint32_t)g, (uint32_t)((uint64_t)g >> 32), (uint32_t)offset, (uint32_t)(offset >> 32)),
                           make_uint2((uint32_t)key, (uint32_t)(key >> 32)));
    const uint32_t words[4] = {w.x, w.y, w.z, w.w};
    float f[8], r[8];
    xs[b].get(f);
    if (RES) rs[b].get(r);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      // the upper half against t << 16 as it stands, the lower one moved up.  (A dropped element is zero whatever it was.)
      const bool keep = ((i & 1) ? words[i >> 1] : words[i >> 1] << 16) >= t;
      f[i] = keep ? (RES ? fmaf(f[i], scale, r[i]) : f[i] * scale) : (RES ? r[i] : 0.f);
    }
    if (e + 8 <= n) {
      dr_store(y + e, f);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (e + i < n) dr_put(y + e + i, f[i]);
    }
  }
}

template <typename T, int NB>
static int dropout_launch(const void* x, const void* res, void* y, long n, uint32_t t, float scale, uint64_t seed, const void* seed_dev,
                          uint64_t offset, cudaStream_t st) {
  const long per = 8l * DR_THREADS * NB, blocks = (n + per - 1) / per;
  if (blocks > 0x7fffffffl) return -12;
  if (res)
    dropout_kernel<T, true, NB><<<(unsigned)blocks, DR_THREADS, 0, st>>>((const T*)x, (const T*)res, (T*)y, n, t, scale, seed,
                                                                          (const long long*)seed_dev, offset);
  else
    dropout_kernel<T, false, NB><<<(unsigned)blocks, DR_THREADS, 0, st>>>((const T*)x, nullptr, (T*)y, n, t, scale, seed,
                                                                           (const long long*)seed_dev, offset);
  return (int)cudaGetLastError();
}

}  // namespace slab

// x, res (or null) and y [n], all bf16 or all fp32, on 16 bytes; t: elements whose 16 bits are below it are dropped (< 65536);
// seed_dev: one int64 on the device that takes the place of `seed`, or null
extern "C" int slab_dropout(const void* x, const void* res, void* y, int bf16, long n, int t, long seed, const void* seed_dev,
                            long offset, void* stream) {
  using namespace slab;
  if (n <= 0 || t < 0 || t > 65535) return -10;
  if (((size_t)x | (size_t)res | (size_t)y) & 15) return -11;
  const float scale = (float)(65536.0 / (65536 - t));
  auto* launch = !bf16 ? dropout_launch<float, 1> : n < DR_MANY ? dropout_launch<__nv_bfloat16, 1> : dropout_launch<__nv_bfloat16, DR_BLOCKS>;
  return launch(x, res, y, n, (uint32_t)t << 16, scale, (uint64_t)seed, seed_dev, (uint64_t)offset, (cudaStream_t)stream);
}
