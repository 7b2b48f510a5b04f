// Gradients of causal attention over packed documents (packed_attention.cu) for sm_100a.
//
//   p_ij = exp2(scale_log2 q_i.k_j - lse_i)     delta_i = do_i.o_i      ds_ij = p_ij (do_i.v_j - delta_i)
//   dv_j = sum_i p_ij do_i      dk_j = scale sum_i ds_ij q_i      dq_i = scale sum_j ds_ij k_j
//
// delta is made from the output with its lower half (packed_attention.cuh).  Two kernels behind the one for delta: one per query
// tile for dq, one per key tile for dk and dv.  Each makes the scores and their gradient again (7 products of 128 x 128 x D a
// tile pair where one kernel could do with 5), but no sum leaves the tensor cores before it is whole: no atomics, no fp32
// copy of dq, and the same bits every time.
//
// Roles as in the forward pass (512 threads): warps 0-3 and 4-7 take the left and the right 64 columns of every 128 x 128
// tile, a row per thread; warp 8 issues the MMAs, warp 9 the copies, warp 11 takes items; warps 12-15 store what is finished.  p
// and ds go back over the scores and products they came from, as bf16, and are the A operand of the next product from tensor
// memory.  Statistics, p - delta and all sums are fp32; p and ds are rounded to bf16 once, as operands.
//
// Bound by the chain of one tile pair: scores, p, dP, ds, product, with two hand-overs of 250 to 350 cycles beside what the
// tensor cores (half busy) and the exponentials take.  One document of 8192 rows, 64/8 heads of 128: dk and dv 1.69 ms, dq 1.30
// (1.3 PFLOP/s of the seven products, 0.79 of cuBLAS in a burst); 8192 rows in documents around 700, 32/4 heads: 382 us in all.
#include "packed_attention.cuh"

namespace slab {

constexpr int PB_THREADS = 512;
constexpr long PB_LONGEST = 1l << 18;        // steps of an item, whose end others wait for: half a second of the two that a wait may last
constexpr int PB_EVERY = 8;                  // of that many pairs of exponentials, one is made on the multiply-add units

struct PackedBwdParams {
  __nv_bfloat16 *dq, *dk, *dv;   // [rows, heads, D] contiguous
  float* partial;                // [splits][2][rows, Hkv, D]: dk and dv of a part of every group's heads, or null (splits 1)
  const float *lse, *delta;      // [Hq, tiles * 128]
  const int* plan;
  PackedRows q, k, v, dout;
  int rows, Hq, Hkv, D;
  int window;
  int splits;                    // most parts that partial has room for
  float scale, scale_log2;
  int* counter;                  // [2] items taken behind the first of every block (dk and dv, dq); [1] parts (packed_delta_kernel)
  int* status;
};

// bytes (a multiple of 16) from global to shared memory, counted on a barrier; both addresses on 16 bytes
__device__ __forceinline__ void pb_bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// The three kernels follow one another closely (launch_early).  dk and dv wait behind their set-up.  dq needs delta only, which is whole once dk and dv
// have begun, so its blocks take over SMs as those of dk and dv end; they wait for the last of them before they end
// themselves, so that what comes behind dq finds dk and dv whole.

// Query tiles that see key tile t
__device__ __forceinline__ int pb_query_tiles(const PackedPlan& plan, int t, int window) {
  int hi = plan.tile_hi[t];
  if (window > 0) hi = min(hi, t * PA_TILE + PA_TILE - 1 + window);
  return hi <= 0 ? 0 : (hi - 1) / PA_TILE - t + 1;
}
// Into how many parts a group's heads are cut for dk and dv (a whole block): a key tile's steps are a serial chain, and the longest
// should be no more than 3/2 of what an SM does in all (dq fills what is then left).  The documents decide, so it is found on the
// device; the host gives the most that there is room for.  8192 rows, 32/4 heads of 128, backward in 1 and 2 parts: documents
// around 300 rows (the longest chain is 1.4 shares) 262 and 288 us, around 2000 (1.2) 503 and 531, around 700 (1.8) 474 and 384;
// 4096 rows of one document (2.2) 738 and 456, in 4 parts the same.
__device__ __forceinline__ void pb_choose_parts(const int* base, int rows, int hq, int hkv, int window, int most, int sms, int* parts) {
  __shared__ int longest;
  __shared__ unsigned long long total;
  if (threadIdx.x == 0) { longest = 0; total = 0; }
  __syncthreads();
  const PackedPlan plan = packed_plan(base, rows);
  int l = 0;
  unsigned long long sum = 0;
  for (int t = threadIdx.x; t < (rows + PA_TILE - 1) / PA_TILE; t += blockDim.x) {
    const int n = pb_query_tiles(plan, t, window);
    l = max(l, n);
    sum += n;
  }
  atomicMax(&longest, l);
  atomicAdd(&total, sum);
  __syncthreads();
  if (threadIdx.x == 0) {
    const int group = hq / hkv;
    int s = 1;
    while (s < most && (group % s || 2l * longest * sms > 3l * (long)total * hkv * s || (long)longest * group > PB_LONGEST * s)) ++s;
    *parts = s;
  }
}

// ================================================================ delta
// DP / 8 lanes per head, eight neighbouring rows each, all of whose loads are in flight together; heads fastest, so that a block
// reads whole lines.  Rows behind the buffer's end, up to whole tiles, get zero.
template <int DP>
__global__ void __launch_bounds__(256)
packed_delta_kernel(const __nv_bfloat16* out, const int8_t* rest, const __nv_bfloat16* dout, float* delta, int rows, int padded, int hq,
                    int d, long do_ts, long do_hs, int* counter, const int* plan, int hkv, int window, int splits, int sms) {
  next_may_begin();
  if (blockIdx.x == 0) {                       // for the kernels behind this one
    if (threadIdx.x < 2) counter[threadIdx.x] = 0;
    pb_choose_parts(plan, rows, hq, hkv, window, splits, sms, counter + 2);
  }
  constexpr int LANES = DP / 8, ROWS = 8;
  const long unit = (long)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  const int c = (threadIdx.x % LANES) * 8;
  const int head = (int)(unit % hq), row0 = (int)(unit / hq) * ROWS;
  if (row0 >= padded) return;                  // (units of a warp end together: 32 / LANES divides ROWS of padded's 128)
  uint4 o[ROWS], g[ROWS];
  uint2 r[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    o[i] = g[i] = make_uint4(0u, 0u, 0u, 0u);
    r[i] = make_uint2(0u, 0u);
    if (row0 + i < rows && c < d) {
      const size_t at = ((size_t)(row0 + i) * hq + head) * d + c;
      o[i] = __ldg(reinterpret_cast<const uint4*>(out + at));
      r[i] = __ldg(reinterpret_cast<const uint2*>(rest + at));
      g[i] = __ldg(reinterpret_cast<const uint4*>(dout + (size_t)(row0 + i) * do_ts + (size_t)head * do_hs + c));
    }
  }
  float sum[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const uint32_t ow[4] = {o[i].x, o[i].y, o[i].z, o[i].w}, rw[2] = {r[i].x, r[i].y};
    float y[8];
    unpack8(*reinterpret_cast<const bf16x8*>(&g[i]), y);
    sum[i] = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t bits = (e & 1) ? ow[e >> 1] >> 16 : ow[e >> 1] & 0xffffu;
      sum[i] = fmaf(pa_unrest(bits, (int)(int8_t)(rw[e >> 2] >> (8 * (e & 3)))), y[e], sum[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
#pragma unroll
    for (int k = LANES / 2; k > 0; k >>= 1) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], k);
  }
  if (threadIdx.x % LANES == 0) {
    float4* to = reinterpret_cast<float4*>(delta + (size_t)head * padded + row0);
    to[0] = make_float4(sum[0], sum[1], sum[2], sum[3]);
    to[1] = make_float4(sum[4], sum[5], sum[6], sum[7]);
  }
}

// ================================================================ common to both
// What a row's scores are reduced by (base-2 log-sum-exp; delta), per column: one value where rows are queries, one each where
// columns are.
struct PbRow {
  float v;
  __device__ __forceinline__ float4 at(int) const { return make_float4(v, v, v, v); }
};
struct PbCols {
  const float4* p;
  __device__ __forceinline__ float4 at(int c) const { return p[c >> 2]; }
};
__device__ __forceinline__ void pb_load(uint32_t taddr, float* s) {
  tmem_ld_32x32(taddr, *reinterpret_cast<uint32_t(*)[32]>(s));
}
// 32 values to bf16, over the first 16 columns of where `to` points
__device__ __forceinline__ void pb_store(uint32_t to, const float* s) {
  uint32_t v[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) v[k] = pa_pack(s[2 * k], s[2 * k + 1]);
  tmem_st_32x16(to, v);
}
// 32 scores to probabilities; one pair in PB_EVERY is made on the multiply-add units where nothing is masked
template <bool PART, typename Stat>
__device__ __forceinline__ void pb_probs(float* s, int c0, const Stat& lse, float2 c2, uint32_t seen) {
#pragma unroll
  for (int c = 0; c < 32; c += 4) {
    const float4 b = lse.at(c0 + c);
#pragma unroll
    for (int e = 0; e < 4; e += 2) {
      float2 x = pa_fma2(make_float2(s[c + e], s[c + e + 1]), c2, e ? make_float2(-b.z, -b.w) : make_float2(-b.x, -b.y));
      if (!PART && ((c + e) / 2) % PB_EVERY == PB_EVERY - 1) {
        x = pa_exp2_fma(x);
      } else {
        x.x = pa_exp2(x.x);
        x.y = pa_exp2(x.y);
      }
      s[c + e] = !PART || (seen >> (c + e) & 1u) ? x.x : 0.f;
      s[c + e + 1] = !PART || (seen >> (c + e + 1) & 1u) ? x.y : 0.f;
    }
  }
}
// 32 probabilities times (dP - delta).  (Zero times what a hidden row holds may be no number: masked again.)
template <bool PART, typename Stat>
__device__ __forceinline__ void pb_dscores(float* s, const float* t, int c0, const Stat& delta, uint32_t seen) {
#pragma unroll
  for (int c = 0; c < 32; c += 4) {
    const float4 b = delta.at(c0 + c);
#pragma unroll
    for (int e = 0; e < 4; e += 2) {
      const float2 x = pa_mul2(make_float2(s[c + e], s[c + e + 1]),
                               pa_add2(make_float2(t[c + e], t[c + e + 1]), e ? make_float2(-b.z, -b.w) : make_float2(-b.x, -b.y)));
      s[c + e] = !PART || (seen >> (c + e) & 1u) ? x.x : 0.f;
      s[c + e + 1] = !PART || (seen >> (c + e + 1) & 1u) ? x.y : 0.f;
    }
  }
}
// What of a thread's 64 columns its row and its warp see.  The warp sees all (whole), or 32-column chunks in vis.
struct PbView {
  uint32_t seen[2], vis;                                     // what the row sees of the chunks; seen only where not whole
  bool whole;
  __device__ __forceinline__ PbView(int from, int to) {      // columns from .. to of 0 .. 63
    from = max(from, 0);
    to = min(to, 63);
    const bool none = from > to;
    seen[0] = seen[1] = 0u;
    whole = !__any_sync(0xffffffffu, from > 0 || to < 63);
    vis = 3u;
    if (!whole) {
      const int lo = __reduce_min_sync(0xffffffffu, none ? 64 : from), hi = __reduce_max_sync(0xffffffffu, none ? -1 : to);
      vis = (lo < 32 && hi >= 0 ? 1u : 0u) | (hi >= 32 ? 2u : 0u);
      seen[0] = pa_bits(from, to, 0);
      seen[1] = pa_bits(from, to, 32);
    }
  }
};
// Scores at `from` to probabilities s.  STORE: as bf16 over the scores too.
template <bool STORE, typename Stat>
__device__ __forceinline__ void pb_step_p(uint32_t from, float (&s)[64], const PbView& v, const Stat& lse, float2 c2) {
  if (v.whole) {
    pb_load(from, &s[0]);
    pb_load(from + 32, &s[32]);
    tmem_ld_wait();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      pb_probs<false>(&s[32 * h], 32 * h, lse, c2, 0u);
      if (STORE) pb_store(from + 16 * h, &s[32 * h]);
    }
    return;
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (v.vis >> h & 1u) {
      pb_load(from + 32 * h, &s[32 * h]);
      tmem_ld_wait();
      pb_probs<true>(&s[32 * h], 32 * h, lse, c2, v.seen[h]);
    } else {
#pragma unroll
      for (int c = 0; c < 32; ++c) s[32 * h + c] = 0.f;
    }
    if (STORE) pb_store(from + 16 * h, &s[32 * h]);
  }
}
// dP at `from` and probabilities s to the scores' gradient, as bf16 at `to`
template <typename Stat>
__device__ __forceinline__ void pb_step_ds(uint32_t from, uint32_t to, float (&s)[64], const PbView& v, const Stat& delta) {
  float t[64];
  if (v.whole) {
    pb_load(from, &t[0]);
    pb_load(from + 32, &t[32]);
    tmem_ld_wait();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      pb_dscores<false>(&s[32 * h], &t[32 * h], 32 * h, delta, 0u);
      pb_store(to + 16 * h, &s[32 * h]);
    }
    return;
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (v.vis >> h & 1u) {
      pb_load(from + 32 * h, &t[32 * h]);
      tmem_ld_wait();
      pb_dscores<true>(&s[32 * h], &t[32 * h], 32 * h, delta, v.seen[h]);
    }
    pb_store(to + 16 * h, &s[32 * h]);
  }
}
__device__ __forceinline__ void pb_arrive(uint64_t* bar) {
  tmem_st_wait();
  tc_fence_before();
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}
// A from tensor memory: 128 rows x 128 of the reduction, the left 64 at a, the right ones 64 columns on
template <int DP>
__device__ __forceinline__ void pb_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
#pragma unroll
  for (int kk = 0; kk < 8; ++kk)
    umma_f16_ts(d, a + (kk >> 2) * 64 + (kk & 3) * 8, b + kk * (2048 >> 4), idesc, (accumulate || kk != 0) ? 1u : 0u);
}

// ================================================================ dq
template <int DP>
struct PackedDqSmem {
  static constexpr int TILE = PA_TILE * DP * 2;
  static constexpr int KST = DP == 128 ? 3 : 5, VST = DP == 128 ? 2 : 4;
  static constexpr int Q_OFF = 1024, DO_OFF = Q_OFF + TILE, K_OFF = DO_OFF + TILE, V_OFF = K_OFF + KST * TILE,
                       TOTAL = V_OFF + VST * TILE;
  static_assert(TOTAL <= 232448, "shared memory budget");
};

struct PackedDqItem {
  int row, head, hk, j0, n;
  __device__ __forceinline__ explicit PackedDqItem(const PaItem& i) : row(i.v[0]), head(i.v[1]), hk(i.v[2]), j0(i.v[3]), n(i.v[7]) {}
};
// (sorted: the plan's order; not where every item has a block of its own)
__device__ __forceinline__ PaItem pb_dq_item(const PackedBwdParams& p, const PackedPlan& plan, int idx, bool sorted) {
  const int o = idx / p.Hq, t = sorted ? plan.q_order[o] : o, lo = plan.tile_lo[t];
  const int head = idx - o * p.Hq, row = t * PA_TILE;
  const int first = p.window > 0 ? max(lo, row - p.window + 1) : lo;
  const int j0 = lo == PA_NONE ? 0 : first / PA_TILE;
  return {{row, head, head / (p.Hq / p.Hkv), j0, 0, 0, 0, lo == PA_NONE ? 0 : t - j0 + 1}};
}

// An issuer's place in the steps of item after item
struct PbWalk {
  int n = 0, i = 0, items = 0;                 // length of the current item, steps of it done, items begun
  __device__ __forceinline__ bool due() const { return i == n; }
  __device__ __forceinline__ void begin(int len) { n = len; i = 0; ++items; }
  __device__ __forceinline__ bool first() const { return i == 0; }
  __device__ __forceinline__ bool last() const { return i == n - 1; }
  __device__ __forceinline__ uint32_t parity() const { return (items - 1) & 1; }
};

// p and ds of one pair of rows (a whole warp)
__device__ __forceinline__ float2 pb_pair(const PackedBwdParams& p, int head, int row, const float4& q, const float4& k,
                                          const float4& v, const float4& dout) {
  const size_t at = (size_t)head * ((p.rows + PA_TILE - 1) / PA_TILE * PA_TILE) + row;
  const float prob = pa_exp2(fmaf(pa_dot4(q, k), p.scale_log2, -p.lse[at]));
  return make_float2(prob, prob * (pa_dot4(dout, v) - p.delta[at]));
}
// dq of one row over its visible keys lo .. row alone (a whole warp)
__device__ __noinline__ void pb_redo_dq(const PackedBwdParams& p, int row, int head, int lo, volatile int* abort_flag) {
  const int hk = head / (p.Hq / p.Hkv);
  const float4 q = pa_row4(p.q, row, head, p.D), dout = pa_row4(p.dout, row, head, p.D);
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int j = lo; j <= row; ++j) {
    pa_redoing(j - lo, abort_flag);
    const float4 k = pa_row4(p.k, j, hk, p.D);
    const float ds = pb_pair(p, head, row, q, k, pa_row4(p.v, j, hk, p.D), dout).y;
    pa_add4(sum, ds, k);
    if (pa_nan(ds)) { sum = make_float4(ds, ds, ds, ds); break; }
  }
  pa_put4(p.dq + ((size_t)row * p.Hq + head) * p.D, p.D, sum, p.scale);
}
// dk or dv of one key row for heads h0 .. h0 + heads - 1 over the queries row .. hi - 1 alone (a whole warp)
__device__ __noinline__ void pb_redo_dkv(const PackedBwdParams& p, bool dv, int row, int hk, int h0, int heads, int part, int parts, int hi,
                                         volatile int* abort_flag) {
  const float4 k = pa_row4(p.k, row, hk, p.D), v = pa_row4(p.v, row, hk, p.D);
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  bool bad = false;
  for (int h = h0; h < h0 + heads && !bad; ++h) {
    pa_redone(abort_flag);
    for (int i = row; i < hi && !bad; ++i) {
      pa_redoing(i - row, abort_flag);
      const float4 q = pa_row4(p.q, i, h, p.D), dout = pa_row4(p.dout, i, h, p.D);
      const float2 w = pb_pair(p, h, i, q, k, v, dout);
      pa_add4(sum, dv ? w.x : w.y, dv ? dout : q);
      bad = pa_nan(dv ? w.x : w.y);
    }
  }
  if (bad) sum.x = sum.y = sum.z = sum.w = __int_as_float(0x7fffffff);
  const size_t at = ((size_t)row * p.Hkv + hk) * p.D;
  const float f = dv ? 1.f : p.scale;
  if (parts > 1) {
    const int c = (threadIdx.x & 31) * 4;
    if (c < p.D)
      *reinterpret_cast<float4*>(p.partial + (size_t)(2 * part + (dv ? 1 : 0)) * p.rows * p.Hkv * p.D + at + c) =
          make_float4(sum.x * f, sum.y * f, sum.z * f, sum.w * f);
  } else {
    pa_put4((dv ? p.dv : p.dk) + at, p.D, sum, f);
  }
}

template <int DP>
__global__ void __launch_bounds__(PB_THREADS, 1)
packed_dq_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                 const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_do,
                 const PackedBwdParams p, const int items) {
  using L = PackedDqSmem<DP>;
  constexpr int KST = L::KST, VST = L::VST;
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023u) {
    if (threadIdx.x == 0) atomicCAS(p.status, 0, ST_BAD_INDEX);
    return;
  }
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem);
  uint64_t* q_empty = q_full + 1;
  uint64_t* do_full = q_empty + 1;
  uint64_t* do_empty = do_full + 1;
  uint64_t* s_full = do_empty + 1;             // [2]
  uint64_t* dp_full = s_full + 2;
  uint64_t* ds_full = dp_full + 1;
  uint64_t* dq_full = ds_full + 1;
  uint64_t* k_full = dq_full + 1;
  uint64_t* k_empty = k_full + KST;
  uint64_t* v_full = k_empty + KST;
  uint64_t* v_empty = v_full + VST;
  PaQueue queue;
  uint64_t* dq_empty = v_empty + VST;
  queue.full = dq_empty + 1;
  queue.empty = queue.full + PA_SLOTS;
  queue.want = queue.empty + PA_SLOTS;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(queue.want + 1);
  queue.slot = reinterpret_cast<int4*>(smem + 512);
  int* lens = reinterpret_cast<int*>(smem + 768);              // [4] the issuer's items in flight
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);         // [3], see pa_wait
  uint8_t *q_s = smem + L::Q_OFF, *do_s = smem + L::DO_OFF, *k_s = smem + L::K_OFF, *v_s = smem + L::V_OFF;
  const int warp = warp_uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const PackedPlan plan = packed_plan(p.plan, p.rows);

  if (threadIdx.x == 0) {
    for (uint64_t* b = q_full; b < queue.empty; ++b) mbar_init(b, b == ds_full ? 8 : b == dq_empty ? 4 : 1);
    for (int q = 0; q < PA_SLOTS; ++q) mbar_init(&queue.empty[q], 14);           // softmax warps, output warps, issuer, copies
    mbar_init(queue.want, 1);
    pa_init_abort(abort_flag);
    fence_mbar_init();
    prefetch_tmap(&map_q);
    prefetch_tmap(&map_k);
    prefetch_tmap(&map_v);
    prefetch_tmap(&map_do);
  }
  if (warp == 8) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;            // S at 0 and 128 in turn, dP at 256, dQ at 384

  if (warp >= 8 && warp < 12) {
    reg_dec<80>();
    if (warp == 9) {
      int pos = 0, done = 0;
      bool ok = true;
      auto load = [&](uint8_t* dst, const CUtensorMap* map, uint64_t* full, uint64_t* empty, uint32_t parity, int head, int row) {
        ok = ok && pa_wait(empty, parity, abort_flag, p.status, ST_PATTN_EMPTY);
        if (ok && elect_one()) {
          mbar_arrive_expect_tx(full, L::TILE);
          pa_load_tile<DP>(dst, map, full, head, row);
        }
      };
      PaReader reader;
      PaItem next;
      while (ok && reader.next(queue, next, abort_flag, p.status)) {
        const PackedDqItem it(next);
        if (it.n < 0) break;
        if (it.n == 0) continue;
        load(q_s, &map_q, q_full, q_empty, (done & 1) ^ 1, it.head, it.row);
        for (int i = 0; ok && i < it.n; ++i, ++pos) {
          const int ks = pos % KST, vs = pos % VST, row = (it.j0 + i) * PA_TILE;
          load(k_s + ks * L::TILE, &map_k, &k_full[ks], &k_empty[ks], ((pos / KST) & 1) ^ 1, it.hk, row);
          if (i == 0) load(do_s, &map_do, do_full, do_empty, (done & 1) ^ 1, it.head, it.row);
          load(v_s + vs * L::TILE, &map_v, &v_full[vs], &v_empty[vs], ((pos / VST) & 1) ^ 1, it.hk, row);
        }
        ++done;
      }
    } else if (warp == 11) {
      pa_schedule(queue, items, p.counter + 1, [&](int idx) { return pb_dq_item(p, plan, idx, items > (int)gridDim.x); }, abort_flag, p.status);
    } else if (warp == 8) {
      constexpr uint32_t idesc_s = make_idesc(1, 1, 0, 0, PA_TILE, PA_TILE);
      constexpr uint32_t idesc_d = make_idesc(1, 1, 0, 1, PA_TILE, DP);
      constexpr uint32_t STEP = L::TILE >> 4;
      const uint64_t qd = make_smem_desc(smem_u32(q_s), 16, 1024, 2), dod = make_smem_desc(smem_u32(do_s), 16, 1024, 2);
      const uint64_t kd = make_smem_desc(smem_u32(k_s), 16, 1024, 2), vd = make_smem_desc(smem_u32(v_s), 16, 1024, 2);
      const uint64_t kt = make_smem_desc(smem_u32(k_s), 16384, 1024, 2);      // K with its rows as the reduction
      bool ok = true, more = true, empty = false;   // more: no item without steps, and not the end, has come; empty: the former has
      PaReader reader;
      // Scores run two steps ahead, dP one; each walk counts its item's steps, stages and parities (counted, not computed: see
      // elect_one).  What a product needs beside ds is waited for while others run.
      PbWalk ws, wp, wq;
      int sk = 0, sq = 0, sv = 0;              // stages of K for the scores, of K for dq, of V
      uint32_t kph = 0, vph = 0, buf = 0, qbuf = 0, dsph = 0;
      auto scores = [&]() {
        while (ok && more && ws.due()) {
          PaItem next;
          ok = reader.next(queue, next, abort_flag, p.status);
          const int n = warp_uniform(next.v[7]);
          more = ok && n > 0;
          empty = ok && n == 0;
          if (more) {
            if (lane == 0) lens[ws.items & 3] = n;
            __syncwarp();
            ws.begin(n);
          }
        }
        if (!ok || !more) return;
        ok = pa_wait(&k_full[sk], kph, abort_flag, p.status, ST_PATTN_KV_FULL);
        if (ws.first()) ok = ok && pa_wait(q_full, ws.parity(), abort_flag, p.status, ST_PATTN_Q);
        if (!ok) return;
        tc_fence_after();
        const uint64_t k0 = kd + (uint32_t)(sk * STEP);
        const uint32_t to = tmem + buf * 128;
        if (elect_one()) {
          pa_mma_ss<DP>(to, qd, k0, idesc_s);
          umma_commit(&s_full[buf]);
          if (ws.last()) umma_commit(q_empty);
        }
        ++ws.i;
        buf ^= 1;
        if (++sk == KST) { sk = 0; kph ^= 1; }
      };
      // the other walks follow the scores' items; false where there is none
      auto follow = [&](PbWalk& w) {
        if (w.due() && w.items < ws.items) w.begin(warp_uniform(lens[w.items & 3]));
        return !w.due();
      };
      bool have_p = false;                     // V of the next dP (and its item's dO) is here
      auto need_v = [&]() {
        have_p = ok && follow(wp);
        if (!have_p) return;
        ok = pa_wait(&v_full[sv], vph, abort_flag, p.status, ST_PATTN_KV_FULL);
        if (wp.first()) ok = ok && pa_wait(do_full, wp.parity(), abort_flag, p.status, ST_PATTN_Q);
      };
      auto dprob = [&]() {
        if (!ok || !have_p) return;
        const uint64_t v0 = vd + (uint32_t)(sv * STEP);
        if (elect_one()) {
          pa_mma_ss<DP>(tmem + 256, dod, v0, idesc_s);
          umma_commit(dp_full);
          umma_commit(&v_empty[sv]);
          if (wp.last()) umma_commit(do_empty);
        }
        ++wp.i;
        if (++sv == VST) { sv = 0; vph ^= 1; }
      };
      scores();
      need_v();
      tc_fence_after();
      dprob();
      scores();
      need_v();
      while (ok && follow(wq)) {
        if (wq.first()) ok = pa_wait(dq_empty, wq.parity() ^ 1, abort_flag, p.status, ST_PATTN_OUT);
        ok = ok && pa_wait(ds_full, dsph, abort_flag, p.status, ST_PATTN_P);
        if (!ok) break;
        tc_fence_after();
        const uint64_t k0 = kt + (uint32_t)(sq * STEP);
        const uint32_t from = tmem + qbuf * 128;
        const bool add = !wq.first(), last = wq.last();
        // the softmax has read dP and wants the next one soonest, unless it waits for the item's dq
        if (!last) dprob();
        if (elect_one()) {
          pb_mma_ts<DP>(tmem + 384, from, k0, idesc_d, add);
          umma_commit(&k_empty[sq]);
          if (last) umma_commit(dq_full);
        }
        if (last) dprob();
        scores();
        need_v();
        ++wq.i;
        dsph ^= 1;
        qbuf ^= 1;
        if (++sq == KST) sq = 0;
      }
      if (ok && empty) reader.drain(queue, abort_flag, p.status);
    }
  } else if (warp < 8) {
    reg_inc<176>();
    const int g = warp >> 2, lg = warp & 3;
    const uint32_t base = tmem + (uint32_t(lg * 32) << 16);
    const int padded = (p.rows + PA_TILE - 1) / PA_TILE * PA_TILE;
    int step = 0;
    bool ok = true;
    PaReader reader;
    PaItem next;
    while (reader.next(queue, next, abort_flag, p.status)) {
      const PackedDqItem it(next);
      if (it.n < 0) break;
      const int row = it.row + lg * 32 + lane;
      int lo = PA_NONE;
      if (row < p.rows) {
        lo = plan.doc_lo[row];
        if (p.window > 0) lo = max(lo, row - p.window + 1);
      }
      const bool sees = lo <= row;
      const PbRow lse = {p.lse[(size_t)it.head * padded + row]}, delta = {p.delta[(size_t)it.head * padded + row]};
      const float2 c2 = make_float2(p.scale_log2, p.scale_log2);
      const int tell = max(it.n - PA_EARLY, 0);
      if (it.n == 0 && threadIdx.x == 0) mbar_arrive(queue.want);
      for (int i = 0; i < it.n; ++i, ++step) {
        const int c0 = (it.j0 + i) * PA_TILE + g * 64;         // first key of this thread's columns
        if (i == tell && threadIdx.x == 0) mbar_arrive(queue.want);
        ok = pa_wait(&s_full[step & 1], (step >> 1) & 1, abort_flag, p.status, ST_PATTN_S);
        if (!ok) break;
        tc_fence_after();
        const PbView view(lo - c0, sees ? row - c0 : -1);
        const uint32_t s_addr = base + (step & 1) * 128 + g * 64;
        float s[64];
        pb_step_p<false>(s_addr, s, view, lse, c2);
        ok = pa_wait(dp_full, step & 1, abort_flag, p.status, ST_PATTN_S);
        if (!ok) break;
        tc_fence_after();
        pb_step_ds(base + 256 + g * 64, s_addr, s, view, delta);
        pb_arrive(ds_full);
      }
      if (!ok) break;
    }
  } else {
    reg_dec<80>();
    // output warps, a row per thread: dq of an item while the softmax warps are at the next one
    const int lg = warp & 3;
    const uint32_t base = tmem + 384 + (uint32_t(lg * 32) << 16);
    const bool wide = p.D % 16 == 0 && (reinterpret_cast<size_t>(p.dq) & 31) == 0;
    int done = 0;
    PaReader reader;
    PaItem next;
    while (reader.next(queue, next, abort_flag, p.status)) {
      const PackedDqItem it(next);
      if (it.n < 0) break;
      const int row = it.row + lg * 32 + lane;
      int lo = PA_NONE;
      if (row < p.rows) {
        lo = plan.doc_lo[row];
        if (p.window > 0) lo = max(lo, row - p.window + 1);
      }
      const bool sees = lo <= row;
      if (it.n > 0) {
        if (!pa_wait(dq_full, done & 1, abort_flag, p.status, ST_PATTN_OUT)) break;
        tc_fence_after();
        ++done;
      }
      __nv_bfloat16* dq_row = p.dq + ((size_t)row * p.Hq + it.head) * p.D;
      float sum = 0.f;
#pragma unroll 1
      for (int c = 0; c < DP; c += 16) {
        uint32_t o[16];
        if (it.n > 0) {
          pa_tmem_ld_16(base + c, o);
          tmem_ld_wait();
          if (c + 16 == DP) {                  // all read: the next item's products may come
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(dq_empty);
          }
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          if (!sees) o[e] = 0u;
          sum += fabsf(__uint_as_float(o[e]));
        }
        if (row < p.rows && c < p.D) pa_put16(dq_row + c, o, 0, p.scale, wide, p.D - c);
      }
      for (uint32_t m = __ballot_sync(0xffffffffu, sees && !pa_finite(sum)); m; m &= m - 1) {
        const int who = __ffs(m) - 1;
        __syncwarp();
        pb_redo_dq(p, it.row + lg * 32 + who, it.head, __shfl_sync(0xffffffffu, lo, who), abort_flag);
        pa_redone(abort_flag);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 100000) __nanosleep(1000);   // let copies in flight land
    __syncthreads();
  }
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (threadIdx.x == 0) wait_before();      // dk and dv
}

// ================================================================ dk, dv
template <int DP>
struct PackedDkvSmem {
  static constexpr int TILE = PA_TILE * DP * 2;
  static constexpr int ST = DP == 128 ? 2 : 3;
  static constexpr int STAT_OFF = 1024, K_OFF = STAT_OFF + 4096, V_OFF = K_OFF + TILE, Q_OFF = V_OFF + TILE,
                       DO_OFF = Q_OFF + ST * TILE, TOTAL = DO_OFF + ST * TILE;     // STAT: lse[ST][128], delta[ST][128]
  static_assert(ST * 1024 <= 4096 && K_OFF % 1024 == 0 && TOTAL <= 232448, "shared memory budget");
};

struct PackedDkvItem {
  int tile, row, hk, part;
  int h0, heads;           // query heads of this part of the group
  int tiles, n;            // query tiles of each, steps over all
  __device__ __forceinline__ explicit PackedDkvItem(const PaItem& i)
      : tile(i.v[0]), row(i.v[0] * PA_TILE), hk(i.v[1]), part(i.v[2]), h0(i.v[3]), heads(i.v[4]), tiles(i.v[5]), n(i.v[7]) {}
};
__device__ __forceinline__ PaItem pb_dkv_item(const PackedBwdParams& p, const PackedPlan& plan, int parts, int idx, bool sorted) {
  const int per = p.Hkv * parts, o = idx / per, rest = idx - o * per, G = p.Hq / p.Hkv;
  const int tile = sorted ? plan.k_order[o] : o, hk = rest / parts, part = rest - hk * parts;
  const int a = part * G / parts, b = (part + 1) * G / parts;
  const int tiles = pb_query_tiles(plan, tile, p.window);
  return {{tile, hk, part, hk * G + a, b - a, tiles, 0, tiles * (b - a)}};
}

template <int DP>
__global__ void __launch_bounds__(PB_THREADS, 1)
packed_dkv_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                  const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_do,
                  const PackedBwdParams p) {
  using L = PackedDkvSmem<DP>;
  constexpr int ST = L::ST;
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023u) {
    if (threadIdx.x == 0) atomicCAS(p.status, 0, ST_BAD_INDEX);
    return;
  }
  uint64_t* k_full = reinterpret_cast<uint64_t*>(smem);
  uint64_t* k_empty = k_full + 1;
  uint64_t* v_full = k_empty + 1;
  uint64_t* v_empty = v_full + 1;
  uint64_t* s_full = v_empty + 1;
  uint64_t* p_full = s_full + 1;
  uint64_t* dp_full = p_full + 1;
  uint64_t* ds_full = dp_full + 1;
  uint64_t* out_full = ds_full + 1;
  uint64_t* q_full = out_full + 1;
  uint64_t* q_empty = q_full + ST;
  uint64_t* do_full = q_empty + ST;
  uint64_t* do_empty = do_full + ST;
  PaQueue queue;
  uint64_t* out_empty = do_empty + ST;
  queue.full = out_empty + 1;
  queue.empty = queue.full + PA_SLOTS;
  queue.want = queue.empty + PA_SLOTS;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(queue.want + 1);
  queue.slot = reinterpret_cast<int4*>(smem + 512);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);         // [3], see pa_wait
  float* lse_s = reinterpret_cast<float*>(smem + L::STAT_OFF);
  float* delta_s = lse_s + ST * PA_TILE;
  uint8_t *k_s = smem + L::K_OFF, *v_s = smem + L::V_OFF, *q_s = smem + L::Q_OFF, *do_s = smem + L::DO_OFF;
  const int warp = warp_uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const PackedPlan plan = packed_plan(p.plan, p.rows);
  const int padded = (p.rows + PA_TILE - 1) / PA_TILE * PA_TILE;

  if (threadIdx.x == 0) {
    for (uint64_t* b = k_full; b < queue.empty; ++b) mbar_init(b, b == p_full || b == ds_full ? 8 : b == out_empty ? 4 : 1);
    for (int q = 0; q < PA_SLOTS; ++q) mbar_init(&queue.empty[q], 14);           // softmax warps, output warps, issuer, copies
    mbar_init(queue.want, 1);
    pa_init_abort(abort_flag);
    fence_mbar_init();
    prefetch_tmap(&map_q);
    prefetch_tmap(&map_k);
    prefetch_tmap(&map_v);
    prefetch_tmap(&map_do);
  }
  if (warp == 8) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  wait_before();                            // delta, and the counters
  next_may_begin();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;            // S^T at 0, dP^T at 128, dV at 256, dK at 384

  if (warp >= 8 && warp < 12) {
    reg_dec<80>();
    if (warp == 9) {
      int pos = 0, done = 0;
      bool ok = true;
      auto load = [&](uint8_t* dst, const CUtensorMap* map, uint64_t* full, uint64_t* empty, uint32_t parity, int head, int row,
                      float* stat_dst, const float* stat) {
        ok = ok && pa_wait(empty, parity, abort_flag, p.status, ST_PATTN_EMPTY);
        if (ok && elect_one()) {
          mbar_arrive_expect_tx(full, L::TILE + (stat ? PA_TILE * 4 : 0));
          pa_load_tile<DP>(dst, map, full, head, row);
          if (stat) pb_bulk_load(stat_dst, stat + (size_t)head * padded + row, PA_TILE * 4, full);
        }
      };
      PaReader reader;
      PaItem next;
      while (ok && reader.next(queue, next, abort_flag, p.status)) {
        const PackedDkvItem it(next);
        if (it.n < 0) break;
        if (it.n == 0) continue;
        load(k_s, &map_k, k_full, k_empty, (done & 1) ^ 1, it.hk, it.row, nullptr, nullptr);
        int head = it.h0, t = 0;
        for (int i = 0; ok && i < it.n; ++i, ++pos) {
          const int s = pos % ST, row = (it.tile + t) * PA_TILE;
          const uint32_t parity = ((pos / ST) & 1) ^ 1;
          load(q_s + s * L::TILE, &map_q, &q_full[s], &q_empty[s], parity, head, row, lse_s + s * PA_TILE, p.lse);
          if (i == 0) load(v_s, &map_v, v_full, v_empty, (done & 1) ^ 1, it.hk, it.row, nullptr, nullptr);
          load(do_s + s * L::TILE, &map_do, &do_full[s], &do_empty[s], parity, head, row, delta_s + s * PA_TILE, p.delta);
          if (++t == it.tiles) { t = 0; ++head; }
        }
        ++done;
      }
    } else if (warp == 11) {
      const int parts = p.counter[2], items = (p.rows + PA_TILE - 1) / PA_TILE * p.Hkv * parts;
      pa_schedule(queue, items, p.counter, [&](int idx) { return pb_dkv_item(p, plan, parts, idx, items > (int)gridDim.x); }, abort_flag,
                  p.status);
    } else if (warp == 8) {
      constexpr uint32_t idesc_s = make_idesc(1, 1, 0, 0, PA_TILE, PA_TILE);
      constexpr uint32_t idesc_d = make_idesc(1, 1, 0, 1, PA_TILE, DP);
      constexpr uint32_t STEP = L::TILE >> 4;
      const uint64_t kd = make_smem_desc(smem_u32(k_s), 16, 1024, 2), vd = make_smem_desc(smem_u32(v_s), 16, 1024, 2);
      const uint64_t qd = make_smem_desc(smem_u32(q_s), 16, 1024, 2), dod = make_smem_desc(smem_u32(do_s), 16, 1024, 2);
      const uint64_t qt = make_smem_desc(smem_u32(q_s), 16384, 1024, 2), dot = make_smem_desc(smem_u32(do_s), 16384, 1024, 2);
      bool ok = true, more = true, empty = false;   // more: no item without steps, and not the end, has come; empty: the former has
      PaReader reader;
      // (stages and parities are counted, not computed: see elect_one)
      PbWalk w;                                // the step whose scores and dP come next
      auto fetch = [&]() {
        while (ok && more && w.due()) {
          PaItem next;
          ok = reader.next(queue, next, abort_flag, p.status);
          const int n = warp_uniform(next.v[7]);
          more = ok && n > 0;
          empty = ok && n == 0;
          if (more) w.begin(n);
        }
      };
      bool done = false;                       // behind the last step
      int sa = 0, sb = 0;                      // stage of that step, of the one before
      uint32_t ph = 0, par = 0;
      auto scores = [&]() {
        if (!ok || !more) return;
        ok = pa_wait(&q_full[sa], ph, abort_flag, p.status, ST_PATTN_Q);
        if (w.first()) ok = ok && pa_wait(k_full, w.parity(), abort_flag, p.status, ST_PATTN_KV_FULL);
        if (!ok) return;
        tc_fence_after();
        const uint64_t q0 = qd + (uint32_t)(sa * STEP);
        if (elect_one()) {
          pa_mma_ss<DP>(tmem, kd, q0, idesc_s);
          umma_commit(s_full);
          if (w.last()) umma_commit(k_empty);
        }
      };
      auto dprob = [&]() {
        if (!ok || !more) return;
        ok = pa_wait(&do_full[sa], ph, abort_flag, p.status, ST_PATTN_Q);
        if (w.first()) ok = ok && pa_wait(v_full, w.parity(), abort_flag, p.status, ST_PATTN_KV_FULL);
        if (!ok) return;
        tc_fence_after();
        const uint64_t d0 = dod + (uint32_t)(sa * STEP);
        if (elect_one()) {
          pa_mma_ss<DP>(tmem + 128, vd, d0, idesc_s);
          umma_commit(dp_full);
          if (w.last()) umma_commit(v_empty);
        }
      };
      fetch();
      scores();
      dprob();
      while (ok && w.items > 0 && !done) {
        const bool add = !w.first(), last = w.last();
        if (!add) ok = pa_wait(out_empty, w.parity() ^ 1, abort_flag, p.status, ST_PATTN_OUT);
        ++w.i;                                 // now at the step behind this one
        fetch();
        done = !more;
        sb = sa;
        if (++sa == ST) { sa = 0; ph ^= 1; }
        const uint64_t d0 = dot + (uint32_t)(sb * STEP), q0 = qt + (uint32_t)(sb * STEP);
        ok = ok && pa_wait(p_full, par, abort_flag, p.status, ST_PATTN_P);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          pb_mma_ts<DP>(tmem + 256, tmem, d0, idesc_d, add);
          umma_commit(&do_empty[sb]);
        }
        scores();
        ok = ok && pa_wait(ds_full, par, abort_flag, p.status, ST_PATTN_P);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          pb_mma_ts<DP>(tmem + 384, tmem + 128, q0, idesc_d, add);
          umma_commit(&q_empty[sb]);
          if (last) umma_commit(out_full);
        }
        dprob();
        par ^= 1;
      }
      if (ok && empty) reader.drain(queue, abort_flag, p.status);
    }
  } else if (warp < 8) {
    reg_inc<176>();
    const int g = warp >> 2, lg = warp & 3;
    const uint32_t base = tmem + (uint32_t(lg * 32) << 16);
    int step = 0, slot = 0;
    uint32_t slot_parity = 0;
    bool ok = true;
    const float2 c2 = make_float2(p.scale_log2, p.scale_log2);
    PaReader reader;
    PaItem next;
    while (reader.next(queue, next, abort_flag, p.status)) {
      const PackedDkvItem it(next);
      if (it.n < 0) break;
      const int row = it.row + lg * 32 + lane;                 // key row of this thread
      int hi = 0;                                              // one past the last query row that sees it
      if (row < p.rows) {
        hi = plan.doc_hi[row];
        if (p.window > 0) hi = min(hi, row + p.window);
      }
      int t = 0;
      const int tell = max(it.n - PA_EARLY, 0);
      if (it.n == 0 && threadIdx.x == 0) mbar_arrive(queue.want);
      for (int i = 0; i < it.n; ++i, ++step) {
        const int c0 = (it.tile + t) * PA_TILE + g * 64;       // first query row of this thread's columns
        if (++t == it.tiles) t = 0;
        const PbView view(row - c0, hi - 1 - c0);
        if (i == tell && threadIdx.x == 0) mbar_arrive(queue.want);
        ok = pa_wait(s_full, step & 1, abort_flag, p.status, ST_PATTN_S) &&
             pa_wait(&q_full[slot], slot_parity, abort_flag, p.status, ST_PATTN_Q);
        if (!ok) break;
        tc_fence_after();
        float s[64];
        pb_step_p<true>(base + g * 64, s, view, PbCols{reinterpret_cast<const float4*>(lse_s + slot * PA_TILE + g * 64)}, c2);
        pb_arrive(p_full);
        ok = pa_wait(dp_full, step & 1, abort_flag, p.status, ST_PATTN_S) &&
             pa_wait(&do_full[slot], slot_parity, abort_flag, p.status, ST_PATTN_Q);
        if (!ok) break;
        tc_fence_after();
        pb_step_ds(base + 128 + g * 64, base + 128 + g * 64, s, view,
                   PbCols{reinterpret_cast<const float4*>(delta_s + slot * PA_TILE + g * 64)});
        pb_arrive(ds_full);
        if (++slot == ST) { slot = 0; slot_parity ^= 1; }
      }
      if (!ok) break;
    }
  } else {
    reg_dec<80>();
    // output warps, a row per thread: dV, then dK of an item while the softmax warps are at the next one
    const int lg = warp & 3;
    const uint32_t base = tmem + 256 + (uint32_t(lg * 32) << 16);
    const bool wide = p.D % 16 == 0 && ((reinterpret_cast<size_t>(p.dk) | reinterpret_cast<size_t>(p.dv)) & 31) == 0;
    const int parts = p.counter[2];
    int done = 0;
    PaReader reader;
    PaItem next;
    while (reader.next(queue, next, abort_flag, p.status)) {
      const PackedDkvItem it(next);
      if (it.n < 0) break;
      const int row = it.row + lg * 32 + lane;                 // key row of this thread
      int hi = 0;                                              // one past the last query row that sees it
      if (row < p.rows) {
        hi = plan.doc_hi[row];
        if (p.window > 0) hi = min(hi, row + p.window);
      }
      const bool any = hi > row;
      if (it.n > 0) {
        if (!pa_wait(out_full, done & 1, abort_flag, p.status, ST_PATTN_OUT)) break;
        tc_fence_after();
        ++done;
      }
      const size_t at = ((size_t)row * p.Hkv + it.hk) * p.D;
      float bad[2] = {0.f, 0.f};
#pragma unroll
      for (int which = 0; which < 2; ++which) {                // dV, dK
        const float f = which == 0 ? 1.f : p.scale;
        __nv_bfloat16* to = (which == 0 ? p.dv : p.dk) + at;
        float* part = p.partial + (size_t)(2 * it.part + (which == 0)) * p.rows * p.Hkv * p.D + at;
#pragma unroll 1
        for (int c = 0; c < DP; c += 16) {
          uint32_t o[16];
          if (it.n > 0) {
            pa_tmem_ld_16(base + which * 128 + c, o);
            tmem_ld_wait();
            if (which == 1 && c + 16 == DP) {                  // all read: the next item's products may come
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(out_empty);
            }
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            if (!any) o[e] = 0u;
            bad[which] += fabsf(__uint_as_float(o[e]));
          }
          if (row < p.rows) {
            if (parts > 1) {
#pragma unroll
              for (int e = 0; e < 16; e += 4)
                if (c + e < p.D)
                  *reinterpret_cast<float4*>(part + c + e) = make_float4(__uint_as_float(o[e]) * f, __uint_as_float(o[e + 1]) * f,
                                                                         __uint_as_float(o[e + 2]) * f, __uint_as_float(o[e + 3]) * f);
            } else if (c < p.D) {
              pa_put16(to + c, o, 0, f, wide, p.D - c);
            }
          }
        }
      }
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        for (uint32_t m = __ballot_sync(0xffffffffu, any && !pa_finite(bad[which])); m; m &= m - 1) {
          const int who = __ffs(m) - 1;
          __syncwarp();
          pb_redo_dkv(p, which == 0, it.row + lg * 32 + who, it.hk, it.h0, it.heads, it.part, parts, __shfl_sync(0xffffffffu, hi, who),
                      abort_flag);
          pa_redone(abort_flag);
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 100000) __nanosleep(1000);   // let copies in flight land
    __syncthreads();
  }
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// dk, dv = the parts' sums, in the parts' order
__global__ void __launch_bounds__(256)
packed_join_kernel(const float* partial, __nv_bfloat16* dk, __nv_bfloat16* dv, long n, const int* parts) {
  const int splits = *parts;
  if (splits == 1) return;                     // written by dk and dv themselves
  const long v = ((long)blockIdx.x * 256 + threadIdx.x) * 8;
  if (v >= 2 * n) return;
  float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < splits; ++s) {
    const float4* src = reinterpret_cast<const float4*>(partial + 2 * n * s + v);
    const float4 a = __ldcs(src), b = __ldcs(src + 1);
    sum[0] += a.x; sum[1] += a.y; sum[2] += a.z; sum[3] += a.w;
    sum[4] += b.x; sum[5] += b.y; sum[6] += b.z; sum[7] += b.w;
  }
  __nv_bfloat16* to = v < n ? dk + v : dv + (v - n);
  *reinterpret_cast<bf16x8*>(to) = pack8(sum);
}

template <int DP>
static int packed_bwd_launch(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const CUtensorMap& mdo,
                             const PackedBwdParams& p, cudaStream_t stream) {
  const long tiles = (p.rows + PA_TILE - 1) / PA_TILE;
  const long dq_items = tiles * p.Hq, dkv_items = tiles * p.Hkv * p.splits;
  SLAB_CUDA_CHECK(cudaFuncSetAttribute(packed_dq_kernel<DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, PackedDqSmem<DP>::TOTAL));
  SLAB_CUDA_CHECK(cudaFuncSetAttribute(packed_dkv_kernel<DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, PackedDkvSmem<DP>::TOTAL));
  const int sms = sm_count();
  SLAB_CUDA_CHECK(launch_early(packed_dkv_kernel<DP>, dim3((unsigned)(dkv_items < sms ? dkv_items : sms)), dim3(PB_THREADS),
                               PackedDkvSmem<DP>::TOTAL, stream, mq, mk, mv, mdo, p));
  SLAB_CUDA_CHECK(launch_early(packed_dq_kernel<DP>, dim3((unsigned)(dq_items < sms ? dq_items : sms)), dim3(PB_THREADS),
                               PackedDqSmem<DP>::TOTAL, stream, mq, mk, mv, mdo, p, (int)dq_items));
  if (p.splits > 1) {
    const long n = (long)p.rows * p.Hkv * p.D;
    packed_join_kernel<<<(unsigned)((2 * n / 8 + 255) / 256), 256, 0, stream>>>(p.partial, p.dk, p.dv, n, p.counter + 2);
  }
  return (int)cudaGetLastError();
}

}  // namespace slab

// Most parts that a group's heads are cut into for dk and dv (pb_choose_parts): room for so many sums.  Twice what one document
// needs, as the longest of several has less beside it.
extern "C" int slab_packed_attn_splits(int rows, int hq, int hkv, int window) {
  if (rows <= 0 || hkv <= 0 || hq % hkv || window < 0) return -10;
  const long tiles = ((long)rows + slab::PA_TILE - 1) / slab::PA_TILE;
  const long seen = window > 0 && (window + slab::PA_TILE - 2) / slab::PA_TILE + 1 < tiles ? (window + slab::PA_TILE - 2) / slab::PA_TILE + 1 : tiles;
  const int group = hq / hkv;
  // longest chain: seen * group steps; all of them: seen (tiles - (seen - 1) / 2) * hq
  const long all = (2 * tiles - seen + 1) * hkv, bound = (seen * group + slab::PB_LONGEST - 1) / slab::PB_LONGEST;
  long want = (8l * slab::sm_count() + 3 * all - 1) / (3 * all);
  want = want > bound ? want : bound;
  int s = want < group ? (int)want : group;
  while (group % s) ++s;
  return s;
}

// q, k, v, dout with token and head strides as in slab_packed_attn_fwd; out, rest, dq, dk, dv contiguous; rest and lse from the forward pass,
// delta [Hq, tiles * 128] and counter [3] int32 scratch; partial: scratch of splits * 2 * rows * Hkv * D floats where splits > 1.
extern "C" int slab_packed_attn_bwd(const void* q, const void* k, const void* v, const void* out, const void* rest,
                                    const void* dout, const void* lse,
                                    const void* plan, void* dq, void* dk, void* dv, void* delta, void* counter, void* partial, int splits,
                                    int rows, int hq, int hkv, int d, long q_ts, long q_hs, long k_ts, long k_hs, long v_ts,
                                    long v_hs, long do_ts, long do_hs, int window, float scale, void* status, void* stream) {
  using namespace slab;
  if (rows <= 0 || hq <= 0 || hkv <= 0 || hq % hkv || d <= 0 || d > 128 || d % 8 || window < 0 || !(scale > 0.f)) return -10;
  if ((q_ts | q_hs | k_ts | k_hs | v_ts | v_hs | do_ts | do_hs) & 7) return -11;
  if (splits < 1 || splits > hq / hkv || (splits > 1 && !partial)) return -13;
  tma_need_context();
  CUtensorMap mq, mk, mv, mdo;
  int rc;
  if ((rc = pa_make_map(&mq, q, rows, hq, d, q_ts, q_hs)) != 0) return rc;
  if ((rc = pa_make_map(&mk, k, rows, hkv, d, k_ts, k_hs)) != 0) return rc;
  if ((rc = pa_make_map(&mv, v, rows, hkv, d, v_ts, v_hs)) != 0) return rc;
  if ((rc = pa_make_map(&mdo, dout, rows, hq, d, do_ts, do_hs)) != 0) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  const int padded = (rows + PA_TILE - 1) / PA_TILE * PA_TILE;
  const long tiles = padded / PA_TILE;
  if (tiles * hq > 0x3fffffff || tiles * hkv * splits > 0x3fffffff) return -12;
  const long units = (long)padded / 8 * hq, per = d <= 64 ? 32 : 16;
  if (d <= 64)
    packed_delta_kernel<64><<<(unsigned)((units + per - 1) / per), 256, 0, st>>>((const __nv_bfloat16*)out, (const int8_t*)rest,
        (const __nv_bfloat16*)dout, (float*)delta, rows, padded, hq, d, do_ts, do_hs, (int*)counter,
        (const int*)plan, hkv, window, splits, sm_count());
  else
    packed_delta_kernel<128><<<(unsigned)((units + per - 1) / per), 256, 0, st>>>((const __nv_bfloat16*)out, (const int8_t*)rest,
        (const __nv_bfloat16*)dout, (float*)delta, rows, padded, hq, d, do_ts, do_hs, (int*)counter,
        (const int*)plan, hkv, window, splits, sm_count());
  // (the kernels behind it take counts from what it has written: without it they must not run)
  SLAB_CUDA_CHECK(cudaGetLastError());
  PackedBwdParams p;
  p.dq = (__nv_bfloat16*)dq;
  p.dk = (__nv_bfloat16*)dk;
  p.dv = (__nv_bfloat16*)dv;
  p.partial = (float*)partial;
  p.lse = (const float*)lse;
  p.delta = (const float*)delta;
  p.plan = (const int*)plan;
  p.q = {(const __nv_bfloat16*)q, q_ts, q_hs};
  p.k = {(const __nv_bfloat16*)k, k_ts, k_hs};
  p.v = {(const __nv_bfloat16*)v, v_ts, v_hs};
  p.dout = {(const __nv_bfloat16*)dout, do_ts, do_hs};
  p.rows = rows; p.Hq = hq; p.Hkv = hkv; p.D = d;
  p.window = window;
  p.splits = splits;
  p.counter = (int*)counter;
  p.scale = scale;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.status = (int*)status;
  return d <= 64 ? packed_bwd_launch<64>(mq, mk, mv, mdo, p, st) : packed_bwd_launch<128>(mq, mk, mv, mdo, p, st);
}
