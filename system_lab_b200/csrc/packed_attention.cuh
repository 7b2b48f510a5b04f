// What the packed-document attention kernels share: tensor memory operands, the documents' plan, item order.
#pragma once
#include "common.cuh"
#include "tma_host.cuh"

namespace slab {

constexpr int PA_TILE = 128;                 // rows of a tile, on the query and on the key side
constexpr int PA_NONE = 0x7fffffff;          // tile_lo of a tile without rows of a document

enum : int {
  ST_PATTN_Q = 40,         // waited for a query tile
  ST_PATTN_KV_FULL = 41,   // waited for a key or value tile
  ST_PATTN_EMPTY = 42,     // producer waited for a free buffer
  ST_PATTN_S = 43,         // softmax waited for scores
  ST_PATTN_P = 44,         // MMA issuer waited for probabilities (or their gradient)
  ST_PATTN_OUT = 45,       // softmax waited for the finished accumulators
  ST_PATTN_ITEM = 46,      // waited for the next item, or for room to put it
};

// The plan of a packed buffer (packed_bounds_kernel), int32:
//   doc_lo[rows], doc_hi[rows]   first row of the row's document, one past its last; a row of no document: row + 1, row
//   tile_lo[tiles], tile_hi[tiles]   least doc_lo and greatest doc_hi of the tile's rows
//   q_order, k_order [tiles], pair_order[pairs]   query tiles, key tiles, pairs of query tiles by falling work
struct PackedPlan {
  const int* doc_lo;
  const int* doc_hi;
  const int* tile_lo;
  const int* tile_hi;
  const int* q_order;
  const int* k_order;
  const int* pair_order;
  const int* end;                            // one past the plan
};
inline __host__ __device__ PackedPlan packed_plan(const int* base, int rows) {
  const int tiles = (rows + PA_TILE - 1) / PA_TILE;
  PackedPlan p;
  p.doc_lo = base;
  p.doc_hi = p.doc_lo + rows;
  p.tile_lo = p.doc_hi + rows;
  p.tile_hi = p.tile_lo + tiles;
  p.q_order = p.tile_hi + tiles;
  p.k_order = p.q_order + tiles;
  p.pair_order = p.k_order + tiles;
  p.end = p.pair_order + (tiles + 1) / 2;
  return p;
}

// ---------------------------------------------------------------- work queue
// Items are listed by falling work.  A block takes the one of its index first and then, one by one, the first that no block has
// taken: documents differ, and dealt out beforehand the last block ended a third after the mean (dk and dv, 8192 rows in
// documents of 700: 458 thousand cycles, mean 341).  A warp of its own takes and decodes them, so that no other role waits for
// the plan's dependent loads (2 to 3 thousand cycles an item), when the softmax warps are PA_EARLY steps from their item's end:
// taken as early as there is room, the first three rounds would be dealt out at once (one document of 8192 rows: dk and dv 2101
// us, 1755 so).  Issuers and copies may be an item ahead of the softmax warps; nobody waits for an item that is given out only
// once he has done something for the one before.  So issuers (and the forward pass's copies) stop at the first item without steps (all behind it, by falling
// work, have none either), finish what they have, and only then read the rest (PaReader::drain): output warps that still wait
// for the issuer's last product have not read that item, and the second one behind it needs its slot.
constexpr int PA_SLOTS = 2, PA_EARLY = 3;
struct PaQueue {
  uint64_t* full;                            // [PA_SLOTS]
  uint64_t* empty;                           // [PA_SLOTS], one arrival per reading warp
  uint64_t* want;                            // the softmax warps are near their item's end
  int4* slot;                                // [PA_SLOTS][2]
};
struct PaItem {
  int v[8];                                  // the last: steps, -1 behind the last item
};
// A reader's next item, to all lanes of its warp; false if a wait ran out
struct PaReader {
  int s = 0;
  uint32_t ph = 0;
  __device__ __forceinline__ bool next(const PaQueue& q, PaItem& it, volatile int* abort_flag, int* status);
  // reads items up to the end, for a role that has nothing to do for them
  __device__ __forceinline__ void drain(const PaQueue& q, volatile int* abort_flag, int* status);
};

// ---------------------------------------------------------------- tensor memory
// D[tmem] (+)= A[tmem] * B[smem desc]: A as 16-bit pairs, row = lane, 8 columns per 16 of the reduction.
__device__ __forceinline__ void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_st_32x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::
          "r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_32x32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void pa_tmem_ld_16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void reg_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void reg_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// A bounded wait of a whole warp (mbar_wait_warp) that is patient while rows are made again: a tile of them can take longer
// than the limit (a key tile of 64 heads x 6000 rows: some 3 s), and so can a single row (alone, some 1.1 us a pair: 64 heads x 30
// thousand rows).  Behind the abort flag stands the time at which such a row was last known to get on (pa_redone: behind every
// PA_STAMP pairs, a few milliseconds, and behind the row); the limit counts from there.
__device__ __forceinline__ bool pa_wait_slow(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* status, int code) {
#pragma unroll 1
  for (int i = 0; i < 32; ++i)
    if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = globaltimer_ns();
  uint32_t spins = 0;
  while (true) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((++spins & 255u) == 0) {
      if (*abort_flag) return false;
      if (globaltimer_ns() - t0 > SLAB_WAIT_NS) {
        const uint64_t row = *reinterpret_cast<volatile uint64_t*>(abort_flag + 1);
        if (globaltimer_ns() - row > SLAB_WAIT_NS) {
          *abort_flag = 1;
          atomicCAS(status, 0, code);
          return false;
        }
      }
    }
  }
}
__device__ __forceinline__ bool pa_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* status, int code) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  return __all_sync(0xffffffffu, pa_wait_slow(bar, parity, abort_flag, status, code));
}
__device__ __forceinline__ void pa_redone(volatile int* abort_flag) {
  if ((threadIdx.x & 31) == 0) *reinterpret_cast<volatile uint64_t*>(abort_flag + 1) = globaltimer_ns();
}
constexpr int PA_STAMP = 4096;
__device__ __forceinline__ void pa_redoing(int pair, volatile int* abort_flag) {
  if ((pair & (PA_STAMP - 1)) == PA_STAMP - 1) pa_redone(abort_flag);
}
__device__ __forceinline__ void pa_init_abort(volatile int* abort_flag) {
  abort_flag[0] = abort_flag[1] = abort_flag[2] = 0;
}

__device__ __forceinline__ bool PaReader::next(const PaQueue& q, PaItem& it, volatile int* abort_flag, int* status) {
  if (!pa_wait(&q.full[s], ph, abort_flag, status, ST_PATTN_ITEM)) return false;
  const int4 a = q.slot[2 * s], b = q.slot[2 * s + 1];
  it = {{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(&q.empty[s]);
  if (++s == PA_SLOTS) { s = 0; ph ^= 1; }
  return true;
}
__device__ __forceinline__ void PaReader::drain(const PaQueue& q, volatile int* abort_flag, int* status) {
  PaItem it;
  while (next(q, it, abort_flag, status) && it.v[7] >= 0) {}
}
// The taking warp: decode(index) makes an item of the list's index.
template <typename Decode>
__device__ __forceinline__ void pa_schedule(const PaQueue& q, int items, int* counter, Decode decode, volatile int* abort_flag,
                                            int* status) {
  int s = 0, idx = blockIdx.x;
  uint32_t ph = 1, want = 0;
  while (true) {
    if (!pa_wait(&q.empty[s], ph, abort_flag, status, ST_PATTN_ITEM)) return;
    PaItem it;
    it.v[7] = -1;
    if (idx < items) it = decode(idx);
    if ((threadIdx.x & 31) == 0) {
      q.slot[2 * s] = make_int4(it.v[0], it.v[1], it.v[2], it.v[3]);
      q.slot[2 * s + 1] = make_int4(it.v[4], it.v[5], it.v[6], it.v[7]);
      mbar_arrive(&q.full[s]);
    }
    if (idx >= items) return;
    if (++s == PA_SLOTS) { s = 0; ph ^= 1; }
    if (!pa_wait(q.want, want, abort_flag, status, ST_PATTN_ITEM)) return;
    want ^= 1;
    if (items > (int)gridDim.x) {
      if ((threadIdx.x & 31) == 0) idx = (int)gridDim.x + atomicAdd(counter, 1);
      idx = warp_uniform(idx);
    } else {
      idx = items;                           // a block for every item: nothing is counted
    }
  }
}

// Bits of the columns from .. to (any values; none where from > to) among c0 .. c0 + 31
__device__ __forceinline__ uint32_t pa_bits(int from, int to, int c0) {
  from = max(from - c0, 0);
  to = min(to - c0, 31);
  return from > to ? 0u : (0xffffffffu << from) & (0xffffffffu >> (31 - to));
}
__device__ __forceinline__ uint32_t pa_pack(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// The output's lower half.  Backward needs delta = do . o, whose error does not shrink where dp - delta does: with o as bf16 it is
// a third to a half of the error of dq and dk in short documents (0.0029 of their root mean square, 0.0023 without).  With
// gradients to come the forward pass therefore rounds half away from zero, so that fp32 bits = bf16 bits << 16 plus the lower 16
// bits as a signed number, and keeps the upper byte of those: o to 2^-16 for one byte more an element.
__device__ __forceinline__ uint32_t pa_pack_half(float lo, float hi) {
  return __byte_perm(__float_as_uint(lo) + 0x8000u, __float_as_uint(hi) + 0x8000u, 0x7632);
}
__device__ __forceinline__ uint32_t pa_rest(float a, float b, float c, float d) {
  return __byte_perm(__byte_perm(__float_as_uint(a), __float_as_uint(b), 0x0051), __byte_perm(__float_as_uint(c), __float_as_uint(d), 0x0051),
                     0x5410);
}
__device__ __forceinline__ float pa_unrest(uint32_t bf16_bits, int rest) { return __uint_as_float((bf16_bits << 16) + ((uint32_t)rest << 8)); }

// 16 neighbouring bf16 of a row, from fp32: one 32-byte store (a whole sector) where the row allows it, else up to two of 16
template <int N>
__device__ __forceinline__ void pa_put16(__nv_bfloat16* to, const uint32_t (&o)[N], int k, float f, bool wide, int left,
                                         int8_t* rest = nullptr) {
  uint32_t v[8];
  if (rest) {
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = __uint_as_float(o[k + 4 * i + e]) * f;
      v[2 * i] = pa_pack_half(x[0], x[1]);
      v[2 * i + 1] = pa_pack_half(x[2], x[3]);
      r[i] = pa_rest(x[0], x[1], x[2], x[3]);
    }
    if (wide) {
      *reinterpret_cast<uint4*>(rest) = make_uint4(r[0], r[1], r[2], r[3]);
    } else {
      if (left > 0) *reinterpret_cast<uint2*>(rest) = make_uint2(r[0], r[1]);
      if (left > 8) *reinterpret_cast<uint2*>(rest + 8) = make_uint2(r[2], r[3]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = pa_pack(__uint_as_float(o[k + 2 * i]) * f, __uint_as_float(o[k + 2 * i + 1]) * f);
  }
  if (wide) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
                 "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
  } else {
    if (left > 0) *reinterpret_cast<uint4*>(to) = make_uint4(v[0], v[1], v[2], v[3]);
    if (left > 8) *reinterpret_cast<uint4*>(to + 8) = make_uint4(v[4], v[5], v[6], v[7]);
  }
}
// two fp32 lanes in one instruction
__device__ __forceinline__ float2 pa_fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)), "l"(reinterpret_cast<uint64_t&>(c)));
  return d;
}
__device__ __forceinline__ float2 pa_add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return d;
}
__device__ __forceinline__ float2 pa_mul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return d;
}
__device__ __forceinline__ float pa_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ---------------------------------------------------------------- rows made again
// A product with tiles also multiplies what a row must not see, by zero: where that is no number, so is the result.  Rows
// whose result is not finite are therefore made again by their warp over the visible keys (queries) alone, and then hold
// what the formula gives.  A lane has four neighbouring columns.
struct PackedRows {
  const __nv_bfloat16* p;
  long ts, hs;             // token and head stride, elements
};
__device__ __forceinline__ float4 pa_row4(const PackedRows& t, int row, int head, int d) {
  const int c = (threadIdx.x & 31) * 4;
  if (c >= d) return make_float4(0.f, 0.f, 0.f, 0.f);
  const uint2 v = *reinterpret_cast<const uint2*>(t.p + (size_t)row * t.ts + (size_t)head * t.hs + c);
  const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v.x));
  const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v.y));
  return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ float pa_dot4(const float4& a, const float4& b) {
  return warp_sum(fmaf(a.x, b.x, fmaf(a.y, b.y, fmaf(a.z, b.z, a.w * b.w))));
}
__device__ __forceinline__ void pa_add4(float4& a, float f, const float4& b) {
  a.x = fmaf(f, b.x, a.x);
  a.y = fmaf(f, b.y, a.y);
  a.z = fmaf(f, b.z, a.z);
  a.w = fmaf(f, b.w, a.w);
}
__device__ __forceinline__ void pa_put4(__nv_bfloat16* to, int d, const float4& v, float f) {
  const int c = (threadIdx.x & 31) * 4;
  if (c < d) *reinterpret_cast<uint2*>(to + c) = make_uint2(pa_pack(v.x * f, v.y * f), pa_pack(v.z * f, v.w * f));
}
__device__ __forceinline__ bool pa_finite(float v) { return (__float_as_uint(v) & 0x7f800000u) != 0x7f800000u; }
__device__ __forceinline__ bool pa_nan(float v) { return (__float_as_uint(v) & 0x7fffffffu) > 0x7f800000u; }

// Largest of three in one instruction
__device__ __forceinline__ float pa_max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// The larger of two; NaN if either is
__device__ __forceinline__ float pa_max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
// 2^x for two numbers on the multiply-add units: x = n + f with n whole (adding 1.5 * 2^23 rounds it into the mantissa's low
// bits) and |f| <= 1/2; a cubic in f, fitted to 2^f for the least largest relative error (7.5e-5; probabilities are then
// rounded to bf16, 3.9e-3); n goes into the exponent.  x below -126 (-inf among it) is taken as -126, and would then weigh 2^-126,
// which is not nothing where a value is large; NaN (an infinity less itself among it) would leave the exponent's sum as a finite
// number.  Both are put right by adding x k at the end: k = 66567 * 2^-149 is 2^-126 (as the cubic has it, 8387401 * 2^-149) / 126
// rounded up, so what was cut off ends at -41 * 2^-149, which bf16 rounds to zero and no sum sees, other results change by less
// than 2^-126, and NaN stays NaN.
__device__ __forceinline__ float2 pa_exp2_fma(float2 x) {
  const float2 magic = make_float2(12582912.f, 12582912.f), k = make_float2(__uint_as_float(66567u), __uint_as_float(66567u));
  x.x = pa_max_nan(x.x, -126.f);
  x.y = pa_max_nan(x.y, -126.f);
  const float2 t = pa_add2(x, magic);
  const float2 n = pa_add2(t, make_float2(-12582912.f, -12582912.f));
  const float2 f = pa_fma2(n, make_float2(-1.f, -1.f), x);
  float2 p = pa_fma2(f, make_float2(0.05517167f, 0.05517167f), make_float2(0.24261113f, 0.24261113f));
  p = pa_fma2(p, f, make_float2(0.69326097f, 0.69326097f));
  p = pa_fma2(p, f, make_float2(0.99992806f, 0.99992806f));
  p = make_float2(__uint_as_float(__float_as_uint(p.x) + (__float_as_uint(t.x) << 23)),
                  __uint_as_float(__float_as_uint(p.y) + (__float_as_uint(t.y) << 23)));
  return pa_fma2(x, k, p);
}

// Tile of 128 rows x DP columns of one head, as boxes of 64 columns ([128 rows][128 bytes], 128-byte swizzle).  Columns at
// or beyond the head's width and rows at or beyond the buffer's end read as zero.
template <int DP>
__device__ __forceinline__ void pa_load_tile(uint8_t* dst, const CUtensorMap* map, uint64_t* bar, int head, int row) {
#pragma unroll
  for (int jb = 0; jb < DP / 64; ++jb) tma_load_3d(dst + jb * 16384, map, bar, jb * 64, head, row);
}
// S[tmem] = A B^T over the head's columns, both K-major in shared memory (descriptors of the tiles' first bytes)
template <int DP>
__device__ __forceinline__ void pa_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc) {
#pragma unroll
  for (int kk = 0; kk < DP / 16; ++kk) {
    const uint32_t off = ((kk >> 2) * 16384 + (kk & 3) * 32) >> 4;
    umma_f16(d, a + off, b + off, idesc, kk != 0 ? 1u : 0u);
  }
}

// ---------------------------------------------------------------- host
// [rows, heads, dim] with any token and head strides, read in boxes of 64 columns x 1 head x 128 rows.
inline int pa_make_map(CUtensorMap* m, const void* base, int rows, int heads, int dim, long token_stride, long head_stride) {
  TmaEncodeTiledFn enc = tma_encode_fn();
  if (!enc) return -1;
  cuuint64_t dims[3] = {(cuuint64_t)dim, (cuuint64_t)heads, (cuuint64_t)rows};
  cuuint64_t strides[2] = {(cuuint64_t)head_stride * 2, (cuuint64_t)token_stride * 2};
  cuuint32_t box[3] = {64, 1, PA_TILE};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, estr,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : -2 - (int)r;
}

}  // namespace slab
