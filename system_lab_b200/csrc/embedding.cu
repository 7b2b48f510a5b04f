// Embedding lookup with scaling, and its gradient.
//
//   out[t] = scale * W[token t]           dW[v] (+)= scale * sum of dout[t] over the tokens t that are v, in the order of t
//
// Both are bound by memory.  The gradient is made from sorted tokens: no atomics on values, every row of dW is written
// once, and the order of the sum is that of the positions whatever the launch.
//   sort   one block per slice of the vocabulary.  It reads all tokens (they are few and lie in L2), counts those below its
//          slice - which is where its part of the sorted list begins - and sorts its own by counting: 32 warps own
//          consecutive parts of the positions and a histogram each, so the order of equal tokens is kept.
//   sum    the sorted list is cut into chunks; a group of threads, one vector of the row each, adds up a chunk's rows and
//          writes every run of equal tokens that lies in it; a run that reaches over a border leaves its pieces' sums, fp32
//   join   such runs: their pieces in order
// Sums are fp32 (the result is rounded once).  Token ids outside the table look up zeros, get no gradient, and are reported.
#include <type_traits>

#include "common.cuh"

namespace slab {

constexpr int EM_WARPS = 32;                 // of a sorting block
constexpr int EM_BATCH = 8;                  // tokens per lane read together
constexpr int EM_MAX_SLICE = 1536;           // vocabulary rows per sorting block: 32 histograms of 6 KB
constexpr int EM_SORT_SMEM = 220 * 1024;     // histograms, and the tokens where they fit beside them
constexpr int EM_MAX_ROWS = 1 << 30;         // of tokens, and of the table: both are counted in 32 bits, in whole groups and slices

// Vectors of a row as they are in memory (Raw: a quarter of the registers that 32-bit numbers take) and as numbers
template <typename T, int VEC>
struct EmVec;
template <>
struct EmVec<__nv_bfloat16, 8> {
  typedef uint4 Raw;
  static __device__ __forceinline__ Raw raw(const __nv_bfloat16* p) { return *reinterpret_cast<const uint4*>(p); }
  static __device__ __forceinline__ void get(const Raw& r, float (&f)[8]) { unpack8(*reinterpret_cast<const bf16x8*>(&r), f); }
  static __device__ __forceinline__ void store(__nv_bfloat16* p, const float (&f)[8]) { *reinterpret_cast<bf16x8*>(p) = pack8(f); }
};
template <>
struct EmVec<float, 8> {
  struct Raw { float4 a, b; };
  static __device__ __forceinline__ Raw raw(const float* p) { return {reinterpret_cast<const float4*>(p)[0], reinterpret_cast<const float4*>(p)[1]}; }
  static __device__ __forceinline__ void get(const Raw& r, float (&f)[8]) {
    f[0] = r.a.x; f[1] = r.a.y; f[2] = r.a.z; f[3] = r.a.w; f[4] = r.b.x; f[5] = r.b.y; f[6] = r.b.z; f[7] = r.b.w;
  }
  static __device__ __forceinline__ void store(float* p, const float (&f)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
  }
};
template <>
struct EmVec<__nv_bfloat16, 1> {
  typedef __nv_bfloat16 Raw;
  static __device__ __forceinline__ Raw raw(const __nv_bfloat16* p) { return *p; }
  static __device__ __forceinline__ void get(const Raw& r, float (&f)[1]) { f[0] = __bfloat162float(r); }
  static __device__ __forceinline__ void store(__nv_bfloat16* p, const float (&f)[1]) { *p = __float2bfloat16(f[0]); }
};
template <>
struct EmVec<float, 1> {
  typedef float Raw;
  static __device__ __forceinline__ Raw raw(const float* p) { return *p; }
  static __device__ __forceinline__ void get(const Raw& r, float (&f)[1]) { f[0] = r; }
  static __device__ __forceinline__ void store(float* p, const float (&f)[1]) { *p = f[0]; }
};
template <typename T, int VEC>
__device__ __forceinline__ void em_load(const T* p, float (&f)[VEC]) { EmVec<T, VEC>::get(EmVec<T, VEC>::raw(p), f); }

// ---------------------------------------------------------------- lookup
constexpr int EM_ROWS = 4;                   // rows of a thread, whose loads are in flight together
// block (vectors, row groups): neighbouring threads on neighbouring vectors of a row
template <typename TW, typename TO, int VEC>
__global__ void __launch_bounds__(256)
embedding_fwd_kernel(const long long* __restrict__ tokens, const TW* __restrict__ w, TO* __restrict__ out, long rows, int h, int vocab,
                     float scale, int* status) {
  const int c = (blockIdx.y * blockDim.x + threadIdx.x) * VEC;
  const long row0 = ((long)blockIdx.x * blockDim.y + threadIdx.y) * EM_ROWS;
  if (c >= h || row0 >= rows) return;
  long long id[EM_ROWS];
  float f[EM_ROWS][VEC];
#pragma unroll
  for (int i = 0; i < EM_ROWS; ++i) id[i] = row0 + i < rows ? tokens[row0 + i] : -1;
#pragma unroll
  for (int i = 0; i < EM_ROWS; ++i) {
    const bool in = id[i] >= 0 && id[i] < vocab;
#pragma unroll
    for (int k = 0; k < VEC; ++k) f[i][k] = 0.f;
    if (in) em_load<TW, VEC>(w + (size_t)id[i] * h + c, f[i]);
    else if (c == 0 && row0 + i < rows) atomicCAS(status, 0, ST_BAD_INDEX);
  }
#pragma unroll
  for (int i = 0; i < EM_ROWS; ++i) {
    if (row0 + i >= rows) break;
#pragma unroll
    for (int k = 0; k < VEC; ++k) f[i][k] *= scale;
    EmVec<TO, VEC>::store(out + (size_t)(row0 + i) * h + c, f[i]);
  }
}

// ---------------------------------------------------------------- sort
// place of a token id in the slice from v0 on: negative below it (and for negative ids), at least the slice's width above
__device__ __forceinline__ int em_bin(long long id, int v0) {
  return id < 0 ? -1 : id >= 0x7fffffffll ? 0x7fffffff : (int)id - v0;
}
// order[0 .. valid): positions of the tokens in the table, by token and then by position; *valid their number; bit v of named: some
// token is v (slices are multiples of 32 rows)
__global__ void __launch_bounds__(EM_WARPS * 32)
embedding_sort_kernel(const long long* __restrict__ tokens, int n, int vocab, int slice, int* __restrict__ order, int* valid,
                      uint32_t* __restrict__ named, int keep) {
  next_may_begin();
  extern __shared__ int hist[];              // [warps][slice], [slice] totals, and with `keep` the tokens for the second pass
  __shared__ int below_s, warp_sums[EM_WARPS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int v0 = blockIdx.x * slice, width = min(slice, vocab - v0);
  int* total = hist + EM_WARPS * slice;
  int* kept = total + slice;
  for (int i = threadIdx.x; i < EM_WARPS * slice; i += blockDim.x) hist[i] = 0;
  if (threadIdx.x == 0) below_s = 0;
  __syncthreads();
  // positions of a warp: whole groups of 32
  const int per = ((n + 32 * EM_WARPS - 1) / (32 * EM_WARPS)) * 32;
  const int from = min(n, warp * per), to = min(n, from + per);
  int below = 0;
  int* mine = hist + warp * slice;
  for (int i0 = from; i0 < to; i0 += 32 * EM_BATCH) {
    long long id[EM_BATCH];
#pragma unroll
    for (int a = 0; a < EM_BATCH; ++a) id[a] = i0 + 32 * a + lane < to ? tokens[i0 + 32 * a + lane] : -1;
#pragma unroll
    for (int a = 0; a < EM_BATCH; ++a) {
      const int b = em_bin(id[a], v0);
      below += b < 0 && id[a] >= 0;
      if (keep && i0 + 32 * a + lane < to) kept[i0 + 32 * a + lane] = b;
      if ((unsigned)b < (unsigned)width) atomicAdd(&mine[b], 1);
    }
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
    const uint32_t bits = __ballot_sync(__activemask(), sum > 0);      // (whole warps: slice is a multiple of 32)
    if ((b & 31) == 0 && b < width) named[(v0 + b) >> 5] = bits;
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
    for (int i0 = from; i0 < to; i0 += 32 * EM_BATCH) {
      int bin[EM_BATCH];
#pragma unroll
      for (int a = 0; a < EM_BATCH; ++a) {
        const int i = i0 + 32 * a + lane;
        bin[a] = i >= to ? -1 : keep ? kept[i] : em_bin(tokens[i], v0);
      }
#pragma unroll
      for (int a = 0; a < EM_BATCH; ++a) {
        const bool in = (unsigned)bin[a] < (unsigned)width;
        if (!__any_sync(0xffffffffu, in)) continue;
        const int b = in ? bin[a] : -1;
        const unsigned peers = __match_any_sync(0xffffffffu, b);
        if (in) order[mine[b] + __popc(peers & ((1u << lane) - 1u))] = i0 + 32 * a + lane;
        __syncwarp();
        if (in && (peers >> lane) == 1u) mine[b] += __popc(peers);     // the last of the equal ones
        __syncwarp();
      }
    }
  }
}

// ---------------------------------------------------------------- sum
struct EmSum {
  const long long* tokens;
  const int* order;
  const int* valid;
  float* pieces;             // [chunks][2][h]: the piece of a run that comes from the chunk before, and of one that goes on
  int2* ends;                // [chunks]: {EM_WHOLE, EM_BEGINS, token of the chunk's last run}
  int h, chunk;              // columns, positions per chunk
  int accumulate;
  float scale;
  const uint32_t* named;     // rows that some token names
  int vocab, sum_blocks;
};
template <typename TW, int VEC>
__device__ __forceinline__ void em_write(const EmSum& p, TW* dw, long long id, int c, const float (&sum)[VEC]) {
  TW* to = dw + (size_t)id * p.h + c;
  float f[VEC], old[VEC];
  if (p.accumulate) em_load<TW, VEC>(to, old);
#pragma unroll
  for (int k = 0; k < VEC; ++k) f[k] = p.accumulate ? fmaf(sum[k], p.scale, old[k]) : sum[k] * p.scale;
  EmVec<TW, VEC>::store(to, f);
}

enum { EM_WHOLE = 1, EM_BEGINS = 2 };        // a chunk lies inside one run that goes on; a run begins in it that goes on
constexpr int EM_AHEAD = 8;                  // rows in flight per thread

// block (columns / VEC threads, chunks): a row of threads sums one chunk
// Blocks from sum_blocks on set the rows that no token names to zero, a warp each: writing them is most of the time where the
// table has many more rows than the batch has tokens, and the sums, which wait for scattered rows, run beside it (8192 tokens,
// 151936 x 2048: 132 us one after the other).
template <typename TW>
__device__ __forceinline__ void em_fill(const uint32_t* named, TW* dw, int vocab, int h, int block, int blocks) {
  const int threads = blockDim.x * blockDim.y, t = threadIdx.y * blockDim.x + threadIdx.x, lane = t & 31;
  const long bytes = (long)h * sizeof(TW);
  const bool vec = ((reinterpret_cast<size_t>(dw) | bytes) & 15) == 0;
  for (long v = (long)block * (threads >> 5) + (t >> 5); v < vocab; v += (long)blocks * (threads >> 5)) {
    if (named[v >> 5] >> (v & 31) & 1u) continue;
    char* row = reinterpret_cast<char*>(dw) + (size_t)v * bytes;
    if (vec) {
      for (long i = lane * 16; i < bytes; i += 512) __stcs(reinterpret_cast<uint4*>(row + i), make_uint4(0u, 0u, 0u, 0u));
    } else {
      for (int i = lane; i < h; i += 32) reinterpret_cast<TW*>(row)[i] = TW(0.f);
    }
  }
}
template <typename TW, typename TO, int VEC>
__global__ void __launch_bounds__(256)
embedding_sum_kernel(const EmSum p, const TO* __restrict__ dout, TW* __restrict__ dw) {
  next_may_begin();
  wait_before();                             // the sorted positions
  if ((int)blockIdx.x >= p.sum_blocks) {
    if (blockIdx.y == 0) em_fill(p.named, dw, p.vocab, p.h, blockIdx.x - p.sum_blocks, gridDim.x - p.sum_blocks);
    return;
  }
  // the chunk's part of the list, from the position before it to the one behind it: {position, token}, token -1 beyond the list
  extern __shared__ int2 list_s[];
  const int chunk = blockIdx.x * blockDim.y + threadIdx.y;
  const int c = (blockIdx.y * blockDim.x + threadIdx.x) * VEC;
  const int valid = *p.valid, from = chunk * p.chunk;
  int2* list = list_s + threadIdx.y * (p.chunk + 2);
  for (int i = threadIdx.x; i < p.chunk + 2; i += blockDim.x) {
    const int at = from - 1 + i;
    int2 e = make_int2(0, -1);
    if (at >= 0 && at < valid) {
      e.x = p.order[at];
      e.y = (int)p.tokens[e.x];
    }
    list[i] = e;
  }
  __syncthreads();
  if (c >= p.h || from >= valid) return;
  const int n = min(valid - from, p.chunk);
  float sum[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) sum[k] = 0.f;
  int run = list[1].y;
  bool head = from > 0 && list[0].y == run;                            // this run began in a chunk before
  bool one = true;
  for (int i = 0; i < n; i += EM_AHEAD) {
    typename EmVec<TO, VEC>::Raw raw[EM_AHEAD];
#pragma unroll
    for (int a = 0; a < EM_AHEAD; ++a)
      if (i + a < n) raw[a] = EmVec<TO, VEC>::raw(dout + (size_t)list[1 + i + a].x * p.h + c);
#pragma unroll
    for (int a = 0; a < EM_AHEAD; ++a) {
      if (i + a < n) {
        const int id = list[1 + i + a].y;
        if (id != run) {
          if (head) EmVec<float, VEC>::store(p.pieces + (size_t)(2 * chunk) * p.h + c, sum);
          else em_write<TW, VEC>(p, dw, run, c, sum);
          head = one = false;
          run = id;
#pragma unroll
          for (int k = 0; k < VEC; ++k) sum[k] = 0.f;
        }
        float x[VEC];
        EmVec<TO, VEC>::get(raw[a], x);
#pragma unroll
        for (int k = 0; k < VEC; ++k) sum[k] += x[k];
      }
    }
  }
  const bool on = from + n < valid && list[1 + n].y == run;            // the last run goes on in the next chunk
  if (head) EmVec<float, VEC>::store(p.pieces + (size_t)(2 * chunk) * p.h + c, sum);
  else if (on) EmVec<float, VEC>::store(p.pieces + (size_t)(2 * chunk + 1) * p.h + c, sum);
  else em_write<TW, VEC>(p, dw, run, c, sum);
  if (c == 0) p.ends[chunk] = make_int2(!on ? 0 : head && one ? EM_WHOLE : EM_BEGINS, run);
}

template <typename TW, int VEC>
__global__ void __launch_bounds__(256)
embedding_join_kernel(const EmSum p, TW* __restrict__ dw) {
  wait_before();                             // the pieces
  const int chunk = blockIdx.x * blockDim.y + threadIdx.y;
  const int c = (blockIdx.y * blockDim.x + threadIdx.x) * VEC;
  const int valid = *p.valid, chunks = (valid + p.chunk - 1) / p.chunk;
  if (c >= p.h || chunk >= chunks) return;
  const int2 e = p.ends[chunk];
  if (!(e.x & EM_BEGINS)) return;
  const long long run = e.y;
  float sum[VEC];
  em_load<float, VEC>(p.pieces + (size_t)(2 * chunk + 1) * p.h + c, sum);
  int end = chunk + 1;                       // chunks chunk + 1 .. end have a piece: up to the first the run ends in
  for (bool found = false; !found;) {
    int w[EM_AHEAD];
#pragma unroll
    for (int a = 0; a < EM_AHEAD; ++a) w[a] = end + a < chunks ? p.ends[end + a].x & EM_WHOLE : 0;
#pragma unroll
    for (int a = 0; a < EM_AHEAD; ++a) {
      if (!found) ++end;
      found = found || !w[a];
    }
  }
  for (int k0 = chunk + 1; k0 < end; k0 += EM_AHEAD) {
    float x[EM_AHEAD][VEC];
#pragma unroll
    for (int a = 0; a < EM_AHEAD; ++a)
      if (k0 + a < end) em_load<float, VEC>(p.pieces + (size_t)(2 * (k0 + a)) * p.h + c, x[a]);
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
// Threads for rows of `vecs` vectors: up to 256 side by side, in slabs of about one length that end on whole warps (2880 columns
// are two slabs of 192 threads, not one of 256 and one of 104), the rest of the block for other rows.
static dim3 em_block(int vecs) {
  const int slabs = (vecs + 255) / 256, each = (vecs + slabs - 1) / slabs;
  int tx = 8;
  if (each > 16) tx = (each + 31) / 32 * 32;
  else while (tx < each) tx *= 2;
  return dim3(tx, 256 / tx > 0 ? 256 / tx : 1);
}
template <typename TW, typename TO, int VEC>
static int em_fwd(const void* tokens, const void* w, void* out, long rows, int vocab, int h, float scale, void* status, cudaStream_t st) {
  const dim3 block = em_block(h / VEC);
  const long groups = (rows + EM_ROWS - 1) / EM_ROWS;
  const dim3 grid((unsigned)((groups + block.y - 1) / block.y), (h / VEC + block.x - 1) / block.x);
  embedding_fwd_kernel<TW, TO, VEC><<<grid, block, 0, st>>>((const long long*)tokens, (const TW*)w, (TO*)out, rows, h, vocab, scale,
                                                            (int*)status);
  return (int)cudaGetLastError();
}

template <typename TW, typename TO, int VEC>
static int em_bwd(const void* tokens, const void* dout, void* dw, int* order, float* pieces, int rows, int chunk, int vocab, int h, float scale,
                  int accumulate, cudaStream_t st) {
  const int sms = em_sms();
  int* valid = order + rows;
  uint32_t* named = reinterpret_cast<uint32_t*>(valid + 1);
  // a block per SM: every block reads all tokens, which from L2 is what bounds it (32749 tokens, 32000 rows, two blocks per SM and
  // both passes from L2: 24 us)
  int slice = (vocab + sms - 1) / sms;
  slice = slice > EM_MAX_SLICE ? EM_MAX_SLICE : (slice + 31) / 32 * 32;
  const int bins = (EM_WARPS + 1) * slice * 4;
  const bool keep = rows <= (EM_SORT_SMEM - bins) / 4;
  const int smem = bins + (keep ? rows * 4 : 0);
  // (the most it ever takes, not this call's: another thread may come between the setting and the launch)
  if (smem > 48 * 1024)
    SLAB_CUDA_CHECK(cudaFuncSetAttribute(embedding_sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, EM_SORT_SMEM));
  embedding_sort_kernel<<<(vocab + slice - 1) / slice, EM_WARPS * 32, smem, st>>>((const long long*)tokens, rows, vocab, slice, order,
                                                                                  valid, named, keep ? 1 : 0);
  // (the sums take positions from what it has written: without it they must not run)
  SLAB_CUDA_CHECK(cudaGetLastError());
  EmSum p;
  p.tokens = (const long long*)tokens;
  p.order = order;
  p.valid = valid;
  p.pieces = pieces;
  p.h = h;
  p.chunk = chunk;
  p.accumulate = accumulate;
  p.scale = scale;
  const dim3 block = em_block(h / VEC);
  const int chunks = (rows + p.chunk - 1) / p.chunk;
  const dim3 grid((chunks + block.y - 1) / block.y, (h / VEC + block.x - 1) / block.x);
  p.named = named;
  p.vocab = vocab;
  p.sum_blocks = (int)grid.x;
  const int fill_blocks = accumulate ? 0 : (vocab + 7) / 8 < 8 * sms ? (vocab + 7) / 8 : 8 * sms;
  p.ends = reinterpret_cast<int2*>(pieces + (size_t)chunks * 2 * h);
  SLAB_CUDA_CHECK(launch_early(embedding_sum_kernel<TW, TO, VEC>, dim3(grid.x + fill_blocks, grid.y), block,
                               block.y * (p.chunk + 2) * sizeof(int2), st, p, (const TO*)dout, (TW*)dw));
  if (chunks > 1) SLAB_CUDA_CHECK(launch_early(embedding_join_kernel<TW, VEC>, grid, block, 0, st, p, (TW*)dw));
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

// dw [vocab, h] (all of it written, or added to), dout [rows, h]; order: scratch of rows + 1 + ceil(vocab / 32) int32, pieces: scratch of
// ceil(rows / chunk) * (2 * h + 2) floats, chunk: positions of the sorted list that a group of threads adds up; at most 2^30 tokens and
// rows of the table
extern "C" int slab_embedding_bwd(const void* tokens, const void* dout, int out_bf16, void* dw, int w_bf16, void* order, void* pieces,
                                  int rows, int chunk, int vocab, int h, float scale, int accumulate, void* stream) {
  using namespace slab;
  if (rows <= 0 || rows > EM_MAX_ROWS || h <= 0 || vocab <= 0 || vocab > EM_MAX_ROWS || chunk <= 0) return -10;
  const bool vec = h % 8 == 0 && (((size_t)dw | (size_t)dout | (size_t)pieces) & 15) == 0;
  return em_types(w_bf16, out_bf16, vec, [&](auto a, auto b, auto v) {
    return em_bwd<decltype(a), decltype(b), decltype(v)::value>(tokens, dout, dw, (int*)order, (float*)pieces, rows, chunk, vocab, h, scale,
                                                                accumulate, (cudaStream_t)stream);
  });
}
