// Embedding lookup with scaling, and its gradient.
//
//   out[t] = scale * W[token t]           dW[v] (+)= scale * sum of dout[t] over the tokens t that are v, in the order of t
//
// Both are bound by memory.  The gradient is made from sorted tokens: no atomics on values, every row of dW is written
// once, and the order of the sum is that of the positions whatever the launch.
//   sort   one block per slice of the vocabulary.  It reads all tokens (they are few and lie in L2), counts those below its
//          slice - which is where its part of the sorted list begins - and sorts its own by counting: 16 warps own
//          consecutive parts of the positions and a histogram each, so the order of equal tokens is kept.  Rows of the
//          slice that no token names are set to zero here, unless the gradient is added to an old one.
//   sum    the sorted list is cut into chunks; a group of threads, one vector of the row each, adds up a chunk's rows and
//          writes every run of equal tokens that lies in it; a run that reaches over a border leaves its pieces' sums, fp32
//   join   such runs: their pieces in order
// Sums are fp32 (the result is rounded once).  Token ids outside the table look up zeros, get no gradient, and are reported.
#include <type_traits>

#include "common.cuh"

namespace slab {

constexpr int EM_WARPS = 16;                 // of a sorting block
constexpr int EM_MAX_SLICE = 768;            // vocabulary rows per sorting block: 16 histograms of 3 KB

template <typename T, int VEC>
struct EmVec;
template <>
struct EmVec<__nv_bfloat16, 8> {
  static __device__ __forceinline__ void load(const __nv_bfloat16* p, float (&f)[8]) { unpack8(*reinterpret_cast<const bf16x8*>(p), f); }
  static __device__ __forceinline__ void store(__nv_bfloat16* p, const float (&f)[8]) { *reinterpret_cast<bf16x8*>(p) = pack8(f); }
};
template <>
struct EmVec<float, 8> {
  static __device__ __forceinline__ void load(const float* p, float (&f)[8]) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  }
  static __device__ __forceinline__ void store(float* p, const float (&f)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
  }
};
template <>
struct EmVec<__nv_bfloat16, 1> {
  static __device__ __forceinline__ void load(const __nv_bfloat16* p, float (&f)[1]) { f[0] = __bfloat162float(*p); }
  static __device__ __forceinline__ void store(__nv_bfloat16* p, const float (&f)[1]) { *p = __float2bfloat16(f[0]); }
};
template <>
struct EmVec<float, 1> {
  static __device__ __forceinline__ void load(const float* p, float (&f)[1]) { f[0] = *p; }
  static __device__ __forceinline__ void store(float* p, const float (&f)[1]) { *p = f[0]; }
};

// ---------------------------------------------------------------- lookup
template <typename TW, typename TO, int VEC>
__global__ void __launch_bounds__(256)
embedding_fwd_kernel(const long long* __restrict__ tokens, const TW* __restrict__ w, TO* __restrict__ out, long n, int vecs, int h,
                     int vocab, float scale, int* status) {
  // `vecs` vectors a row, neighbouring threads on neighbouring ones
  const long stride = (long)gridDim.x * blockDim.x;
  for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += stride) {
    const long row = i / vecs;
    const int c = (int)(i - row * vecs) * VEC;
    const long long id = tokens[row];
    float f[VEC];
    if (id >= 0 && id < vocab) {
      EmVec<TW, VEC>::load(w + (size_t)id * h + c, f);
#pragma unroll
      for (int k = 0; k < VEC; ++k) f[k] *= scale;
    } else {
#pragma unroll
      for (int k = 0; k < VEC; ++k) f[k] = 0.f;
      if (c == 0) atomicCAS(status, 0, ST_BAD_INDEX);
    }
    EmVec<TO, VEC>::store(out + (size_t)row * h + c, f);
  }
}

// ---------------------------------------------------------------- sort
// order[0 .. valid): positions of the tokens in the table, by token and then by position; *valid their number
template <typename TW>
__global__ void __launch_bounds__(EM_WARPS * 32)
embedding_sort_kernel(const long long* __restrict__ tokens, int n, int vocab, int slice, int* __restrict__ order, int* valid,
                      TW* __restrict__ dw, int h, int fill) {
  extern __shared__ int hist[];              // [warps][slice], then [slice] totals
  __shared__ int below_s, warp_sums[EM_WARPS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int v0 = blockIdx.x * slice, width = min(slice, vocab - v0);
  int* total = hist + EM_WARPS * slice;
  for (int i = threadIdx.x; i < EM_WARPS * slice; i += blockDim.x) hist[i] = 0;
  if (threadIdx.x == 0) below_s = 0;
  __syncthreads();
  // positions of a warp: whole groups of 32
  const int per = ((n + 32 * EM_WARPS - 1) / (32 * EM_WARPS)) * 32;
  const int from = min(n, warp * per), to = min(n, from + per);
  int below = 0;
  int* mine = hist + warp * slice;
#pragma unroll 4
  for (int i = from + lane; i < to; i += 32) {
    const long long id = tokens[i];
    below += id >= 0 && id < v0;
    if (id >= v0 && id < v0 + width) atomicAdd(&mine[(int)id - v0], 1);
  }
  below = __reduce_add_sync(0xffffffffu, below);
  if (lane == 0) atomicAdd(&below_s, below);
  __syncthreads();
  // a bin's histograms become the numbers of equal tokens before each warp's
  for (int b = threadIdx.x; b < slice; b += blockDim.x) {
    int sum = 0;
    if (b < width) {
#pragma unroll
      for (int w = 0; w < EM_WARPS; ++w) {
        const int c = hist[w * slice + b];
        hist[w * slice + b] = sum;
        sum += c;
      }
    }
    total[b] = sum;
  }
  __syncthreads();
  // first place of every bin: a thread has neighbouring bins
  const int each = (slice + blockDim.x - 1) / blockDim.x, b0 = threadIdx.x * each;
  int sum = 0;
  for (int b = b0; b < min(b0 + each, slice); ++b) sum += total[b];
  int scan = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, scan, o);
    if (lane >= o) scan += v;
  }
  if (lane == 31) warp_sums[warp] = scan;
  __syncthreads();
  int at = below_s + scan - sum, all = 0;
  for (int w = 0; w < EM_WARPS; ++w) {
    if (w < warp) at += warp_sums[w];
    all += warp_sums[w];
  }
  if (threadIdx.x == 0 && blockIdx.x == gridDim.x - 1) *valid = below_s + all;
  for (int b = b0; b < min(b0 + each, slice); ++b) {
    const int c = total[b];
    for (int w = 0; w < EM_WARPS && c > 0; ++w) hist[w * slice + b] += at;
    at += c;
  }
  __syncthreads();
  if (all > 0) {
    for (int i0 = from; i0 < to; i0 += 32) {
      const int i = i0 + lane;
      const long long id = i < to ? tokens[i] : -1;
      const bool in = id >= v0 && id < v0 + width;
      const int b = in ? (int)id - v0 : -1;
      if (!__any_sync(0xffffffffu, in)) continue;
      const unsigned peers = __match_any_sync(0xffffffffu, b);
      if (in) order[mine[b] + __popc(peers & ((1u << lane) - 1u))] = i;
      __syncwarp();
      if (in && (peers >> lane) == 1u) mine[b] += __popc(peers);       // the last of the equal ones
      __syncwarp();
    }
  }
  if (!fill) return;
  // rows without tokens, a warp each (their bytes are a multiple of 16 where the table's rows are)
  const long bytes = (long)h * sizeof(TW);
  for (int b = warp; b < width; b += EM_WARPS) {
    if (total[b]) continue;
    char* row = reinterpret_cast<char*>(dw) + (size_t)(v0 + b) * bytes;
    if (((reinterpret_cast<size_t>(dw) | bytes) & 15) == 0) {
      for (long i = lane * 16; i < bytes; i += 512) __stcs(reinterpret_cast<uint4*>(row + i), make_uint4(0u, 0u, 0u, 0u));
    } else {
      for (int i = lane; i < h; i += 32) reinterpret_cast<TW*>(row)[i] = TW(0.f);
    }
  }
}

// ---------------------------------------------------------------- sum
struct EmSum {
  const long long* tokens;
  const int* order;
  const int* valid;
  float* pieces;             // [chunks][2][h]: the piece of a run that comes from the chunk before, and of one that goes on
  int h, chunk;              // columns, positions per chunk
  int accumulate;
  float scale;
};
template <typename TW, int VEC>
__device__ __forceinline__ void em_write(const EmSum& p, TW* dw, long long id, int c, const float (&sum)[VEC]) {
  TW* to = dw + (size_t)id * p.h + c;
  float f[VEC], old[VEC];
  if (p.accumulate) EmVec<TW, VEC>::load(to, old);
#pragma unroll
  for (int k = 0; k < VEC; ++k) f[k] = p.accumulate ? fmaf(sum[k], p.scale, old[k]) : sum[k] * p.scale;
  EmVec<TW, VEC>::store(to, f);
}

constexpr int EM_AHEAD = 8;                  // rows in flight per thread

// block (columns / VEC threads, chunks): a row of threads sums one chunk
template <typename TW, typename TO, int VEC>
__global__ void __launch_bounds__(256)
embedding_sum_kernel(const EmSum p, const TO* __restrict__ dout, TW* __restrict__ dw) {
  const int chunk = blockIdx.x * blockDim.y + threadIdx.y;
  const int c = (blockIdx.y * blockDim.x + threadIdx.x) * VEC;
  const int valid = *p.valid, from = chunk * p.chunk;
  if (c >= p.h || from >= valid) return;
  const int to = min(valid, from + p.chunk);
  float sum[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) sum[k] = 0.f;
  long long run = p.tokens[p.order[from]];
  bool head = from > 0 && p.tokens[p.order[from - 1]] == run;          // this run began in a chunk before
  for (int i = from; i < to; i += EM_AHEAD) {
    int pos[EM_AHEAD];
    long long id[EM_AHEAD];
    float x[EM_AHEAD][VEC];
#pragma unroll
    for (int a = 0; a < EM_AHEAD; ++a) pos[a] = i + a < to ? p.order[i + a] : 0;
#pragma unroll
    for (int a = 0; a < EM_AHEAD; ++a) {
      if (i + a < to) {
        id[a] = p.tokens[pos[a]];
        EmVec<TO, VEC>::load(dout + (size_t)pos[a] * p.h + c, x[a]);
      }
    }
#pragma unroll
    for (int a = 0; a < EM_AHEAD; ++a) {
      if (i + a < to) {
        if (id[a] != run) {
          if (head) EmVec<float, VEC>::store(p.pieces + (size_t)(2 * chunk) * p.h + c, sum);
          else em_write<TW, VEC>(p, dw, run, c, sum);
          head = false;
          run = id[a];
#pragma unroll
          for (int k = 0; k < VEC; ++k) sum[k] = 0.f;
        }
#pragma unroll
        for (int k = 0; k < VEC; ++k) sum[k] += x[a][k];
      }
    }
  }
  const bool on = to < valid && p.tokens[p.order[to]] == run;          // the last run goes on in the next chunk
  if (head) EmVec<float, VEC>::store(p.pieces + (size_t)(2 * chunk) * p.h + c, sum);
  else if (on) EmVec<float, VEC>::store(p.pieces + (size_t)(2 * chunk + 1) * p.h + c, sum);
  else em_write<TW, VEC>(p, dw, run, c, sum);
}

template <typename TW, int VEC>
__global__ void __launch_bounds__(256)
embedding_join_kernel(const EmSum p, TW* __restrict__ dw) {
  const int chunk = blockIdx.x * blockDim.y + threadIdx.y;
  const int c = (blockIdx.y * blockDim.x + threadIdx.x) * VEC;
  const int valid = *p.valid, from = chunk * p.chunk, next = from + p.chunk;
  if (c >= p.h || next >= valid) return;
  // runs that begin in this chunk and go on in the next
  const long long run = p.tokens[p.order[next - 1]];
  if (p.tokens[p.order[next]] != run || (from > 0 && p.tokens[p.order[from - 1]] == run)) return;
  float sum[VEC];
  EmVec<float, VEC>::load(p.pieces + (size_t)(2 * chunk + 1) * p.h + c, sum);
  int end = chunk + 1;                       // chunks chunk + 1 .. end - 1 have a piece: the run's last position, by bisection
  {
    int lo = next, hi = valid;               // order[lo] is of the run, order[hi] is not (or behind the list)
    while (hi - lo > 1) {
      const int mid = lo + (hi - lo) / 2;
      if (p.tokens[p.order[mid]] == run) lo = mid; else hi = mid;
    }
    end = lo / p.chunk + 1;
  }
  for (int k0 = chunk + 1; k0 < end; k0 += EM_AHEAD) {
    float x[EM_AHEAD][VEC];
#pragma unroll
    for (int a = 0; a < EM_AHEAD; ++a)
      if (k0 + a < end) EmVec<float, VEC>::load(p.pieces + (size_t)(2 * (k0 + a)) * p.h + c, x[a]);
#pragma unroll
    for (int a = 0; a < EM_AHEAD; ++a) {
      if (k0 + a < end) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) sum[k] += x[a][k];
      }
    }
  }
  em_write<TW, VEC>(p, dw, run, c, sum);
}

// ---------------------------------------------------------------- launches
static int em_sms() {
  int dev = 0, n = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return n > 0 ? n : 1;
}
template <typename TW, typename TO, int VEC>
static int em_fwd(const void* tokens, const void* w, void* out, long rows, int vocab, int h, float scale, void* status, cudaStream_t st) {
  const int vecs = h / VEC;
  const long n = rows * vecs;
  const long blocks = (n + 255) / 256;
  embedding_fwd_kernel<TW, TO, VEC><<<(unsigned)(blocks < (1l << 30) ? blocks : (1l << 30)), 256, 0, st>>>(
      (const long long*)tokens, (const TW*)w, (TO*)out, n, vecs, h, vocab, scale, (int*)status);
  return (int)cudaGetLastError();
}

template <typename TW, typename TO, int VEC>
static int em_bwd(const void* tokens, const void* dout, void* dw, int* order, float* pieces, int rows, int chunk, int vocab, int h, float scale,
                  int accumulate, cudaStream_t st) {
  const int sms = em_sms();
  int* valid = order + rows;
  int slice = (vocab + 2 * sms - 1) / (2 * sms);
  slice = slice < 1 ? 1 : slice > EM_MAX_SLICE ? EM_MAX_SLICE : slice;
  const int smem = (EM_WARPS + 1) * slice * 4;
  SLAB_CUDA_CHECK(cudaFuncSetAttribute(embedding_sort_kernel<TW>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       (EM_WARPS + 1) * EM_MAX_SLICE * 4));
  embedding_sort_kernel<TW><<<(vocab + slice - 1) / slice, EM_WARPS * 32, smem, st>>>(
      (const long long*)tokens, rows, vocab, slice, order, valid, (TW*)dw, h, accumulate ? 0 : 1);
  EmSum p;
  p.tokens = (const long long*)tokens;
  p.order = order;
  p.valid = valid;
  p.pieces = pieces;
  p.h = h;
  p.chunk = chunk;
  p.accumulate = accumulate;
  p.scale = scale;
  const int vecs = h / VEC;
  int tx = 8;
  while (tx < 256 && tx < vecs) tx *= 2;
  const dim3 block(tx, 256 / tx);
  const int chunks = (rows + p.chunk - 1) / p.chunk;
  const dim3 grid((chunks + block.y - 1) / block.y, (vecs + tx - 1) / tx);
  embedding_sum_kernel<TW, TO, VEC><<<grid, block, 0, st>>>(p, (const TO*)dout, (TW*)dw);
  if (chunks > 1) embedding_join_kernel<TW, VEC><<<grid, block, 0, st>>>(p, (TW*)dw);
  return (int)cudaGetLastError();
}

template <typename F>
static int em_types(int w_bf16, int o_bf16, bool vec, F f) {
  using B = __nv_bfloat16;
  if (vec)
    return w_bf16 ? (o_bf16 ? f(B(), B(), std::integral_constant<int, 8>()) : f(B(), 0.f, std::integral_constant<int, 8>()))
                  : (o_bf16 ? f(0.f, B(), std::integral_constant<int, 8>()) : f(0.f, 0.f, std::integral_constant<int, 8>()));
  return w_bf16 ? (o_bf16 ? f(B(), B(), std::integral_constant<int, 1>()) : f(B(), 0.f, std::integral_constant<int, 1>()))
                : (o_bf16 ? f(0.f, B(), std::integral_constant<int, 1>()) : f(0.f, 0.f, std::integral_constant<int, 1>()));
}

}  // namespace slab

// tokens [rows] int64, w [vocab, h], out [rows, h]; each fp32 or bf16
extern "C" int slab_embedding_fwd(const void* tokens, const void* w, int w_bf16, void* out, int out_bf16, long rows, int vocab, int h,
                                  float scale, void* status, void* stream) {
  using namespace slab;
  if (rows <= 0 || h <= 0 || vocab < 0) return -10;
  const bool vec = h % 8 == 0 && (((size_t)w | (size_t)out) & 15) == 0;
  return em_types(w_bf16, out_bf16, vec, [&](auto a, auto b, auto v) {
    return em_fwd<decltype(a), decltype(b), decltype(v)::value>(tokens, w, out, rows, vocab, h, scale, status, (cudaStream_t)stream);
  });
}

// dw [vocab, h] (all of it written, or added to), dout [rows, h]; order: scratch of rows + 1 int32, pieces: scratch of
// ceil(rows / chunk) * 2 * h floats, chunk: positions of the sorted list that a group of threads adds up
extern "C" int slab_embedding_bwd(const void* tokens, const void* dout, int out_bf16, void* dw, int w_bf16, void* order, void* pieces,
                                  int rows, int chunk, int vocab, int h, float scale, int accumulate, void* stream) {
  using namespace slab;
  if (rows <= 0 || h <= 0 || vocab <= 0 || chunk <= 0) return -10;
  const bool vec = h % 8 == 0 && (((size_t)dw | (size_t)dout | (size_t)pieces) & 15) == 0;
  return em_types(w_bf16, out_bf16, vec, [&](auto a, auto b, auto v) {
    return em_bwd<decltype(a), decltype(b), decltype(v)::value>(tokens, dout, dw, (int*)order, (float*)pieces, rows, chunk, vocab, h, scale,
                                                                accumulate, (cudaStream_t)stream);
  });
}
