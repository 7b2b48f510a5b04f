// Causal attention over packed documents for sm_100a: the plan of a packed buffer, and the forward pass.
//
//   o_i = sum_j p_ij v_j,  p_ij = exp(scale q_i.k_j) / sum,  over lo_i <= j <= i
//
// Documents lie one behind the other in a buffer of rows; lo_i is the first row of row i's document, or i - window + 1
// where that is later.  Tiles are cut from the buffer, not from the documents: lo grows with i, so the keys that a query
// tile sees are the tiles from its least lo to its own, whatever documents lie in it, and many short documents share one
// tile.  Rows of no document get zeros.
//
// Roles (512 threads, one persistent block per SM): warps 0-3 and 4-7 softmax, one query tile of 128 rows each, a row per
// thread; warp 8 issues the MMAs, warp 9 the copies, warp 11 takes items; warps 12-15 store finished rows.  The two query tiles
// share the key and value tiles: two heads of one group on the same rows where the group is even (nothing is masked for one
// tile only), else the next 128 rows.
// S and O live in tensor memory (2 x 128 + 2 x DP columns).  The probabilities go back over the scores they came from, as
// bf16, and are the A operand of P V from there.  While one tile's softmax runs, the tensor cores do P V of the other
// and its next scores.  O is brought to a new maximum only when a row's maximum has grown by 2^8: until then its
// probabilities are at most 2^8 too large, and so is their sum.  Statistics and sums are fp32; probabilities are rounded
// to bf16 once, as the operand of P V.
//
// Long documents are bound by the tensor cores and the exponentials side by side (8192 rows of one document, 64/8 heads of 128: 848
// us, 1.30 PFLOP/s, 0.79 of cuBLAS in a burst), short ones by their masked tiles and an item's start and end, some 5 thousand
// cycles (8192 rows in documents around 700, 32/4 heads: 115 us; 16384 rows, window 128, 64/8 heads of 64: 162 us).
#include "packed_attention.cuh"

namespace slab {

// ================================================================ plan
__global__ void packed_bounds_kernel(const int* cu, int docs, int rows, int* base, int* status) {
  const PackedPlan p = packed_plan(base, rows);
  const int row = blockIdx.x * PA_TILE + threadIdx.x;
  if (blockIdx.x == 0) {                         // offsets that fall, or pass the buffer's end, are reported
    bool bad = threadIdx.x == 0 && (cu[0] != 0 || cu[docs] > rows);
    for (int s = threadIdx.x; s < docs; s += PA_TILE) bad |= cu[s + 1] < cu[s];
    if (bad) atomicCAS(status, 0, ST_BAD_INDEX);
  }
  int lo = row + 1, hi = row;
  if (row < rows) {
    int a = 0, b = docs;                         // documents that end at or before this row
    while (a < b) {
      const int mid = (a + b) >> 1;
      if (cu[mid + 1] <= row) a = mid + 1; else b = mid;
    }
    if (a < docs && cu[a] <= row) {
      lo = max(cu[a], 0);
      hi = min(cu[a + 1], rows);
    }
    const_cast<int*>(p.doc_lo)[row] = lo;
    const_cast<int*>(p.doc_hi)[row] = hi;
  }
  int least = lo <= row ? lo : PA_NONE, most = lo <= row ? hi : 0;
  least = __reduce_min_sync(0xffffffffu, least);
  most = __reduce_max_sync(0xffffffffu, most);
  __shared__ int l[4], m[4];
  if ((threadIdx.x & 31) == 0) { l[threadIdx.x >> 5] = least; m[threadIdx.x >> 5] = most; }
  __syncthreads();
  if (threadIdx.x == 0) {
    const_cast<int*>(p.tile_lo)[blockIdx.x] = min(min(l[0], l[1]), min(l[2], l[3]));
    const_cast<int*>(p.tile_hi)[blockIdx.x] = max(max(m[0], m[1]), max(m[2], m[3]));
  }
}

// Documents of token rows [batch][seq]: one starts with every row of the batch and behind every end-of-document token.
// starts[2 t], starts[2 t + 1]: last and first start among the tile's positions (-1, PA_NONE: none).
__device__ __forceinline__ bool pa_starts(const long long* tokens, int i, int seq, long long end) {
  return i % seq == 0 || tokens[i - 1] == end;
}
__global__ void packed_starts_kernel(const long long* tokens, int rows, int seq, long long end, int* starts) {
  const int row = blockIdx.x * PA_TILE + threadIdx.x;
  const bool s = row < rows && pa_starts(tokens, row, seq, end);
  const int last = __reduce_max_sync(0xffffffffu, s ? row : -1), first = __reduce_min_sync(0xffffffffu, s ? row : PA_NONE);
  __shared__ int l[4], m[4];
  if ((threadIdx.x & 31) == 0) { l[threadIdx.x >> 5] = last; m[threadIdx.x >> 5] = first; }
  __syncthreads();
  if (threadIdx.x == 0) {
    starts[2 * blockIdx.x] = max(max(l[0], l[1]), max(l[2], l[3]));
    starts[2 * blockIdx.x + 1] = min(min(m[0], m[1]), min(m[2], m[3]));
  }
}
__global__ void packed_token_bounds_kernel(const long long* tokens, int rows, int seq, long long end, const int* starts, int* base) {
  const PackedPlan p = packed_plan(base, rows);
  const int row = blockIdx.x * PA_TILE + threadIdx.x;
  __shared__ int before, behind;
  __shared__ uint32_t mask[4];
  if (threadIdx.x == 0) { before = 0; behind = rows; }
  __syncthreads();
  int lo = 0, hi = rows;
  for (int u = threadIdx.x; u < (int)gridDim.x; u += PA_TILE) {
    if (u < (int)blockIdx.x) lo = max(lo, starts[2 * u]);
    if (u > (int)blockIdx.x) hi = min(hi, starts[2 * u + 1]);
  }
  atomicMax(&before, lo);
  atomicMin(&behind, hi);
  const uint32_t bits = __ballot_sync(0xffffffffu, row < rows && pa_starts(tokens, row, seq, end));
  if ((threadIdx.x & 31) == 0) mask[threadIdx.x >> 5] = bits;
  __syncthreads();
  // last start at or before this row, first one behind it
  lo = before;
  hi = behind;
  const int w = threadIdx.x >> 5, at = threadIdx.x & 31;
  for (int k = 0; k < 4; ++k) {
    const uint32_t le = k < w ? mask[k] : k == w ? mask[k] & (0xffffffffu >> (31 - at)) : 0u;
    if (le) lo = blockIdx.x * PA_TILE + k * 32 + 31 - __clz(le);
  }
  for (int k = 3; k >= 0; --k) {
    const uint32_t gt = k > w ? mask[k] : k == w && at < 31 ? mask[k] & (0xffffffffu << (at + 1)) : 0u;
    if (gt) hi = blockIdx.x * PA_TILE + k * 32 + __ffs(gt) - 1;
  }
  if (row < rows) {
    const_cast<int*>(p.doc_lo)[row] = lo;
    const_cast<int*>(p.doc_hi)[row] = hi;
  }
  if (threadIdx.x == 0) const_cast<int*>(p.tile_lo)[blockIdx.x] = lo;       // row 0 of the tile has its least lo
  if (row == min(rows, ((int)blockIdx.x + 1) * PA_TILE) - 1) const_cast<int*>(p.tile_hi)[blockIdx.x] = hi;
}

__device__ __forceinline__ int pa_key_tiles(const PackedPlan& p, int t) {
  const int lo = p.tile_lo[t];
  return lo == PA_NONE ? 0 : t - lo / PA_TILE + 1;
}
__device__ __forceinline__ int pa_query_tiles(const PackedPlan& p, int t) {
  const int hi = p.tile_hi[t];
  return hi == 0 ? 0 : (hi - 1) / PA_TILE - t + 1;
}
// A tile's place is the number of tiles with more work, or as much and a lower index.
__global__ void packed_order_kernel(int rows, int* base) {
  const PackedPlan p = packed_plan(base, rows);
  const int tiles = gridDim.x, pairs = (tiles + 1) / 2, t = blockIdx.x;
  auto pair_tiles = [&](int i) {
    const int n1 = 2 * i + 1 < tiles ? pa_key_tiles(p, 2 * i + 1) : 0;
    return max(n1, pa_key_tiles(p, 2 * i) + (n1 > 0));
  };
  const int nq = pa_key_tiles(p, t), nk = pa_query_tiles(p, t), np = t < pairs ? pair_tiles(t) : 0;
  int bq = 0, bk = 0, bp = 0;
  for (int u = threadIdx.x; u < tiles; u += blockDim.x) {
    const int q = pa_key_tiles(p, u), k = pa_query_tiles(p, u);
    bq += q > nq || (q == nq && u < t);
    bk += k > nk || (k == nk && u < t);
    if (u < pairs && t < pairs) {
      const int x = pair_tiles(u);
      bp += x > np || (x == np && u < t);
    }
  }
  __shared__ int sum[3];
  if (threadIdx.x < 3) sum[threadIdx.x] = 0;
  __syncthreads();
  atomicAdd(&sum[0], bq);
  atomicAdd(&sum[1], bk);
  atomicAdd(&sum[2], bp);
  __syncthreads();
  if (threadIdx.x == 0) {
    const_cast<int*>(p.q_order)[sum[0]] = t;
    const_cast<int*>(p.k_order)[sum[1]] = t;
    if (t < pairs) const_cast<int*>(p.pair_order)[sum[2]] = t;
  }
}

// ================================================================ forward
constexpr int PF_THREADS = 512;
constexpr int PF_EVERY = 8;                   // of that many pairs of exponentials, one is made on the multiply-add units
constexpr float PF_SLACK = 8.f;              // a row's maximum may be this far (log2) below the true one

struct PackedFwdParams {
  __nv_bfloat16* out;      // [rows, Hq, D]
  int8_t* rest;            // [rows, Hq, D] the output's lower half, or null
  float* lse;              // [Hq, tiles * 128], base-2 log-sum-exp of the scaled scores; +inf where a row sees nothing
  const int* plan;
  PackedRows q, k, v;
  int rows, Hq, Hkv, D;
  int window;              // 0: whole document
  int head_pairs;          // two heads of a group share a block, else two tiles of rows
  float scale_log2;        // softmax scale * log2(e)
  int* counter;            // items taken behind the first of every block, zero at launch
  int* status;
};

// A stage holds the V tile of a step and the K tile of the next one (of the next item, where the step is an item's last): they are
// used in one go and freed together.
template <int DP>
struct PackedFwdSmem {
  static constexpr int TILE = PA_TILE * DP * 2;
  static constexpr int STAGES = DP == 128 ? 2 : 4;
  static constexpr int STAT_OFF = 1024, Q_OFF = STAT_OFF + 4096, KV_OFF = Q_OFF + 2 * TILE, TOTAL = KV_OFF + STAGES * 2 * TILE;
  static_assert(TOTAL <= 232448, "shared memory budget");
};

struct PackedFwdItem {
  int row[2], head[2], hk;
  int j0, n;               // first key tile, key tiles
  __device__ __forceinline__ explicit PackedFwdItem(const PaItem& i)
      : row{i.v[0], i.v[1]}, head{i.v[2], i.v[3]}, hk(i.v[4]), j0(i.v[5]), n(i.v[7]) {}
};
// (sorted: the plan's order; not where every item has a block of its own, which spares it a dependent load)
__device__ __forceinline__ PaItem pf_item(const PackedFwdParams& p, const PackedPlan& plan, int idx, bool sorted) {
  const int tiles = (p.rows + PA_TILE - 1) / PA_TILE;
  int lo, last, row0, row1, head0, head1;
  if (p.head_pairs) {
    const int hp = p.Hq >> 1, o = idx / hp, t = sorted ? plan.q_order[o] : o;
    head0 = 2 * (idx - o * hp);
    head1 = head0 + 1;
    row0 = row1 = t * PA_TILE;
    lo = plan.tile_lo[t];
    last = t;
  } else {
    const int o = idx / p.Hq, t = 2 * (sorted ? plan.pair_order[o] : o);
    head0 = head1 = idx - o * p.Hq;
    row0 = t * PA_TILE;
    row1 = row0 + PA_TILE;
    lo = plan.tile_lo[t];
    last = t;
    if (t + 1 < tiles && plan.tile_lo[t + 1] != PA_NONE) {
      lo = min(lo, plan.tile_lo[t + 1]);
      last = t + 1;
    }
  }
  const int first = p.window > 0 ? max(lo, row0 - p.window + 1) : lo;
  const int j0 = lo == PA_NONE ? 0 : first / PA_TILE;
  return {{row0, row1, head0, head1, head0 / (p.Hq / p.Hkv), j0, 0, lo == PA_NONE ? 0 : last - j0 + 1}};
}

// One row over its visible keys lo .. row alone (a whole warp).  The values' mean is carried, not their sum, which can pass fp32
// where the mean does not (two values near the type's largest).
__device__ __noinline__ void pf_redo(const PackedFwdParams& p, int row, int head, int lo, volatile int* abort_flag) {
  const int hk = head / (p.Hq / p.Hkv), padded = (p.rows + PA_TILE - 1) / PA_TILE * PA_TILE;
  const float4 q = pa_row4(p.q, row, head, p.D);
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  float m = -INFINITY, l = 0.f;
  for (int j = lo; j <= row; ++j) {
    pa_redoing(j - lo, abort_flag);
    const float s = pa_dot4(q, pa_row4(p.k, j, hk, p.D)) * p.scale_log2;
    if (pa_nan(s)) { l = s; break; }                                   // and so is the whole row
    // (a score of -inf weighs zero; what is no number beside it makes the mean none either)
    const float top = fmaxf(m, s), old = m == -INFINITY ? 0.f : l * pa_exp2(m - top), e = s == -INFINITY ? 0.f : pa_exp2(s - top);
    l = old + e;
    const float keep = l == 0.f ? 1.f : old / l;
    o = make_float4(o.x * keep, o.y * keep, o.z * keep, o.w * keep);
    pa_add4(o, l == 0.f ? 0.f : e / l, pa_row4(p.v, j, hk, p.D));
    m = top;
    if (pa_nan(l)) break;
  }
  const float bad = __int_as_float(0x7fffffff);
  const bool none = pa_nan(l) || l == 0.f;
  if (none) o = make_float4(bad, bad, bad, bad);
  const size_t at = ((size_t)row * p.Hq + head) * p.D;
  const int c = (threadIdx.x & 31) * 4;
  if (p.rest && c < p.D) {
    const bool fin = pa_finite(o.x) && pa_finite(o.y) && pa_finite(o.z) && pa_finite(o.w);
    *reinterpret_cast<uint32_t*>(p.rest + at + c) = fin ? pa_rest(o.x, o.y, o.z, o.w) : 0u;
    if (fin) *reinterpret_cast<uint2*>(p.out + at + c) = make_uint2(pa_pack_half(o.x, o.y), pa_pack_half(o.z, o.w));
    else pa_put4(p.out + at, p.D, o, 1.f);
  } else {
    pa_put4(p.out + at, p.D, o, 1.f);
  }
  if ((threadIdx.x & 31) == 0) p.lse[(size_t)head * padded + row] = none ? bad : m + log2f(l);
}

// A row's running sums come to a maximum that has grown by more than the slack.  All rows of a warp together.
template <int DP>
__device__ __forceinline__ void pf_raise(uint32_t o_addr, float top, float& m, float2& la, float2& lb) {
  if (m == -INFINITY) m = top;                 // nothing has been added yet
  const bool grow = top > m + PF_SLACK;
  if (!__any_sync(0xffffffffu, grow)) return;
  float alpha = 1.f;
  if (grow) {
    alpha = pa_exp2(m - top);
    m = top;
  }
  la = pa_mul2(la, make_float2(alpha, alpha));
  lb = pa_mul2(lb, make_float2(alpha, alpha));
#pragma unroll 1
  for (int c = 0; c < DP; c += 16) {
    uint32_t o[16];
    pa_tmem_ld_16(o_addr + c, o);
    tmem_ld_wait();
#pragma unroll
    for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
    tmem_st_32x16(o_addr + c, o);
  }
}
__device__ __forceinline__ void pf_arrive(uint64_t* bar) {
  tmem_st_wait();
  tc_fence_before();
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

// One step of a row: scores to probabilities, which go back over them as bf16; p_full is told.  m:
// maximum (log2 units) that the sums la + lb and the output are relative to.  This form: all rows of the warp see all keys.
template <int DP>
__device__ __forceinline__ void pf_whole(uint32_t s_addr, uint32_t o_addr, float scale_log2, float& m, float2& la, float2& lb,
                                         uint64_t* p_full) {
  float s[128];
#pragma unroll
  for (int c = 0; c < 128; c += 32) tmem_ld_32x32(s_addr + c, *reinterpret_cast<uint32_t(*)[32]>(&s[c]));
  tmem_ld_wait();
  float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
  for (int k = 4; k < 124; k += 8) {
#pragma unroll
    for (int e = 0; e < 4; ++e) mx[e] = pa_max3(mx[e], s[k + 2 * e], s[k + 2 * e + 1]);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) mx[e] = fmaxf(mx[e], s[124 + e]);
  pf_raise<DP>(o_addr, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale_log2, m, la, lb);
  const float base = m == -INFINITY ? 0.f : -m;
  const float2 c2 = make_float2(scale_log2, scale_log2), b2 = make_float2(base, base);
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    uint32_t packed[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      float2 x = pa_fma2(make_float2(s[32 * c + 2 * k], s[32 * c + 2 * k + 1]), c2, b2);
      if (k % PF_EVERY == PF_EVERY - 1) {
        x = pa_exp2_fma(x);
        lb = pa_add2(lb, x);
      } else {
        x.x = pa_exp2(x.x);
        x.y = pa_exp2(x.y);
        la = pa_add2(la, x);
      }
      packed[k] = pa_pack(x.x, x.y);
    }
    tmem_st_32x16(s_addr + c * 16, packed);
  }
  pf_arrive(p_full);
}

// The other form: a row sees keys first .. lastk (none where first > lastk); chunks of 32 that no row of the warp sees (not in
// vis) are left out.  Two passes over the scores, a chunk at a time: few registers, short code.
template <int DP>
__device__ __forceinline__ void pf_part(uint32_t s_addr, uint32_t o_addr, float scale_log2, uint32_t vis, int first, int lastk,
                                        float& m, float2& la, float2& lb, uint64_t* p_full) {
  float top = -INFINITY;
#pragma unroll 1
  for (int c = 0; c < 4; ++c) {
    if (!(vis >> c & 1u)) continue;
    float s[32];
    tmem_ld_32x32(s_addr + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(&s[0]));
    tmem_ld_wait();
    const uint32_t seen = pa_bits(first, lastk, 32 * c);
    float mx[2] = {top, -INFINITY};
#pragma unroll
    for (int k = 0; k < 32; k += 2)
      mx[(k >> 1) & 1] = pa_max3(mx[(k >> 1) & 1], seen >> k & 1u ? s[k] : -INFINITY, seen >> (k + 1) & 1u ? s[k + 1] : -INFINITY);
    top = fmaxf(mx[0], mx[1]);
  }
  pf_raise<DP>(o_addr, top * scale_log2, m, la, lb);
  const float base = m == -INFINITY ? 0.f : -m;
  const float2 c2 = make_float2(scale_log2, scale_log2), b2 = make_float2(base, base);
#pragma unroll 1
  for (int c = 0; c < 4; ++c) {
    uint32_t packed[16];
    if (vis >> c & 1u) {
      float s[32];
      tmem_ld_32x32(s_addr + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(&s[0]));
      tmem_ld_wait();
      const uint32_t seen = pa_bits(first, lastk, 32 * c);
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        float2 x = pa_fma2(make_float2(s[2 * k], s[2 * k + 1]), c2, b2);
        x.x = seen >> (2 * k) & 1u ? pa_exp2(x.x) : 0.f;
        x.y = seen >> (2 * k + 1) & 1u ? pa_exp2(x.y) : 0.f;
        la = pa_add2(la, x);
        packed[k] = pa_pack(x.x, x.y);
      }
    } else {
#pragma unroll
      for (int k = 0; k < 16; ++k) packed[k] = 0u;
    }
    tmem_st_32x16(s_addr + c * 16, packed);    // (over scores that have been read)
  }
  pf_arrive(p_full);
}

template <int DP>
__global__ void __launch_bounds__(PF_THREADS, 1)
packed_fwd_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                  const __grid_constant__ CUtensorMap map_v, const PackedFwdParams p, const int items) {
  using L = PackedFwdSmem<DP>;
  constexpr int NST = L::STAGES;
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023u) {
    if (threadIdx.x == 0) atomicCAS(p.status, 0, ST_BAD_INDEX);
    return;
  }
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem);
  uint64_t* q_empty = q_full + 2;
  uint64_t* kv_full = q_empty + 2;
  uint64_t* kv_empty = kv_full + NST;
  uint64_t* s_full = kv_empty + NST;
  uint64_t* p_full = s_full + 2;
  uint64_t* o_full = p_full + 2;
  PaQueue queue;
  uint64_t* o_empty = o_full + 2;
  uint64_t* l_full = o_empty + 2;
  queue.full = l_full + 4;
  queue.empty = queue.full + PA_SLOTS;
  queue.want = queue.empty + PA_SLOTS;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(queue.want + 1);
  queue.slot = reinterpret_cast<int4*>(smem + 512);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);         // [3], see pa_wait
  float2* stat_s = reinterpret_cast<float2*>(smem + L::STAT_OFF);       // [2 items][2 tiles][128] sum and maximum of a row
  uint8_t* q_s = smem + L::Q_OFF;
  uint8_t* kv_s = smem + L::KV_OFF;
  const int warp = warp_uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const PackedPlan plan = packed_plan(p.plan, p.rows);

  if (threadIdx.x == 0) {
    for (int g = 0; g < 2; ++g) {
      mbar_init(&q_full[g], 1);
      mbar_init(&q_empty[g], 1);
      mbar_init(&s_full[g], 1);
      mbar_init(&p_full[g], 4);
      mbar_init(&o_full[g], 1);
      mbar_init(&o_empty[g], 4);
      mbar_init(&l_full[g], 4);
      mbar_init(&l_full[2 + g], 4);
    }
    for (int s = 0; s < NST; ++s) {
      mbar_init(&kv_full[s], 1);
      mbar_init(&kv_empty[s], 1);
    }
    for (int q = 0; q < PA_SLOTS; ++q) {
      mbar_init(&queue.full[q], 1);
      mbar_init(&queue.empty[q], 14);          // softmax warps, output warps, issuer, copies
    }
    mbar_init(queue.want, 1);
    pa_init_abort(abort_flag);
    fence_mbar_init();
    prefetch_tmap(&map_q);
    prefetch_tmap(&map_k);
    prefetch_tmap(&map_v);
  }
  if (warp == 8) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;            // S of tile g at 128 g, O at 256 + 128 g

  if (warp >= 8 && warp < 12) {
    reg_dec<48>();
    if (warp == 9) {
      // ------------------------------------------------------------ copies
      int st = 0, done = 0;                    // stage, items before this one
      uint32_t ph = 1;
      bool ok = true;
      int v_row = -1, v_head = 0;              // V tile of the step before, the stage's other half
      bool empty = false;                      // an item without key tiles came: so are all behind it, and the last V tile is due
      auto load_stage = [&](int k_row, int k_head) {             // (no K behind the last item's last step)
        ok = ok && pa_wait(&kv_empty[st], ph, abort_flag, p.status, ST_PATTN_EMPTY);
        if (ok && elect_one()) {
          uint8_t* to = kv_s + st * 2 * L::TILE;
          mbar_arrive_expect_tx(&kv_full[st], (v_row >= 0 ? L::TILE : 0) + (k_row >= 0 ? L::TILE : 0));
          if (v_row >= 0) pa_load_tile<DP>(to, &map_v, &kv_full[st], v_head, v_row);
          if (k_row >= 0) pa_load_tile<DP>(to + L::TILE, &map_k, &kv_full[st], k_head, k_row);
        }
        if (++st == NST) { st = 0; ph ^= 1; }
      };
      PaReader reader;
      PaItem next;
      while (ok && reader.next(queue, next, abort_flag, p.status)) {
        const PackedFwdItem it(next);
        empty = it.n == 0;
        if (it.n <= 0) break;
        load_stage(it.j0 * PA_TILE, it.hk);
        for (int g = 0; g < 2; ++g) {
          ok = ok && pa_wait(&q_empty[g], (done & 1) ^ 1, abort_flag, p.status, ST_PATTN_EMPTY);
          if (ok && elect_one()) {
            mbar_arrive_expect_tx(&q_full[g], L::TILE);
            pa_load_tile<DP>(q_s + g * L::TILE, &map_q, &q_full[g], it.head[g], it.row[g]);
          }
        }
        v_head = it.hk;
        for (int i = 0; ok && i < it.n; ++i) {
          v_row = (it.j0 + i) * PA_TILE;
          if (i + 1 < it.n) load_stage(v_row + PA_TILE, it.hk);
        }
        ++done;
      }
      if (ok && v_row >= 0) load_stage(-1, 0);
      if (ok && empty) reader.drain(queue, abort_flag, p.status);
    } else if (warp == 11) {
      pa_schedule(queue, items, p.counter, [&](int idx) { return pf_item(p, plan, idx, items > (int)gridDim.x); }, abort_flag, p.status);
    } else if (warp == 8) {
      // ------------------------------------------------------------ MMAs
      constexpr uint32_t idesc_qk = make_idesc(1, 1, 0, 0, PA_TILE, PA_TILE);
      constexpr uint32_t idesc_pv = make_idesc(1, 1, 0, 1, PA_TILE, DP);
      constexpr uint32_t STEP = L::TILE >> 4;
      const uint64_t qd = make_smem_desc(smem_u32(q_s), 16, 1024, 2);
      const uint64_t vd = make_smem_desc(smem_u32(kv_s), 16384, 1024, 2);               // key rows as the reduction
      const uint64_t kd = make_smem_desc(smem_u32(kv_s + L::TILE), 16, 1024, 2);
      PaReader reader;
      bool ok = true;
      bool empty = false;                      // an item without key tiles came: so are all behind it
      auto next_len = [&]() {                  // key tiles of the next item, 0 behind the last that has any
        PaItem next;
        ok = ok && reader.next(queue, next, abort_flag, p.status);
        const int n = ok ? warp_uniform(next.v[7]) : 0;
        empty = ok && n == 0;
        return n > 0 ? n : 0;
      };
      // This warp's own instructions bound a step once its waits (some 250 cycles each beside the softmax warps) follow one
      // another: what the next step needs is waited for and counted up before the second tile's probabilities are.  (Stages
      // and parities are counted, not computed: what the issued instructions take has to be plainly the same in all lanes,
      // see elect_one.)
      int st = 0;
      uint32_t ph = 0, pph = 0, qph = 0, oph = 1;
      int n = next_len(), i = 0;               // the step whose P V comes next: i of n
      bool last = n == 1;
      if (n > 0) {                             // scores of the first step
        ok = ok && pa_wait(&kv_full[0], 0, abort_flag, p.status, ST_PATTN_KV_FULL);
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          ok = ok && pa_wait(&q_full[g], 0, abort_flag, p.status, ST_PATTN_Q);
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
            pa_mma_ss<DP>(tmem + g * 128, qd + g * STEP, kd, idesc_qk);
            umma_commit(&s_full[g]);
            if (g == 1) umma_commit(&kv_empty[0]);
            if (last) umma_commit(&q_empty[g]);
          }
        }
        qph = 1;
        st = 1 % NST;
        if (st == 0) ph ^= 1;
        ok = ok && pa_wait(&kv_full[st], ph, abort_flag, p.status, ST_PATTN_KV_FULL);
      }
      while (ok && n > 0) {
        const bool was = last;
        const uint64_t v0 = vd + (uint32_t)(st * 2 * STEP), k0 = kd + (uint32_t)(st * 2 * STEP);
        const uint32_t fresh = i != 0 ? 1u : 0u;
        const int s0 = st;
        if (i == 0) ok = pa_wait(&o_empty[0], oph, abort_flag, p.status, ST_PATTN_OUT);
        ok = ok && pa_wait(&p_full[0], pph, abort_flag, p.status, ST_PATTN_P);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int k4 = 0; k4 < 8; ++k4)
            umma_f16_ts(tmem + 256, tmem + k4 * 8, v0 + k4 * (2048 >> 4), idesc_pv, k4 != 0 ? 1u : fresh);
          if (was) umma_commit(&o_full[0]);
        }
        const int after = was ? next_len() : n;                  // length of the item that the next step belongs to
        const bool more = after > 0;
        const bool ends = was ? after == 1 : i + 2 == n;         // whether that step is its item's last
        if (more && was) ok = ok && pa_wait(&q_full[0], qph, abort_flag, p.status, ST_PATTN_Q);
        if (!ok) break;
        if (more && elect_one()) {
          pa_mma_ss<DP>(tmem, qd, k0, idesc_qk);
          umma_commit(&s_full[0]);
          if (ends) umma_commit(&q_empty[0]);
        }
        if (more && last) ok = ok && pa_wait(&q_full[1], qph, abort_flag, p.status, ST_PATTN_Q);
        if (i == 0) {
          ok = ok && pa_wait(&o_empty[1], oph, abort_flag, p.status, ST_PATTN_OUT);
          oph ^= 1;
        }
        if (last) qph ^= 1;
        i = last ? 0 : i + 1;
        n = after;
        last = i == n - 1;
        if (++st == NST) { st = 0; ph ^= 1; }
        if (n > 0) ok = ok && pa_wait(&kv_full[st], ph, abort_flag, p.status, ST_PATTN_KV_FULL);
        ok = ok && pa_wait(&p_full[1], pph, abort_flag, p.status, ST_PATTN_P);
        pph ^= 1;
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int k4 = 0; k4 < 8; ++k4)
            umma_f16_ts(tmem + 384, tmem + 128 + k4 * 8, v0 + k4 * (2048 >> 4), idesc_pv, k4 != 0 ? 1u : fresh);
          if (was) umma_commit(&o_full[1]);
          if (more) {
            pa_mma_ss<DP>(tmem + 128, qd + STEP, k0, idesc_qk);
            umma_commit(&s_full[1]);
            if (ends) umma_commit(&q_empty[1]);
          }
          umma_commit(&kv_empty[s0]);
        }
      }
      if (ok && empty) reader.drain(queue, abort_flag, p.status);
    }
  } else if (warp < 8) {
    reg_inc<192>();
    // ------------------------------------------------------------ softmax: a query row per thread
    const int g = warp >> 2, lg = warp & 3;
    const int r128 = lg * 32 + lane;
    const uint32_t s_addr = tmem + g * 128 + (uint32_t(lg * 32) << 16);
    const uint32_t o_addr = tmem + 256 + g * 128 + (uint32_t(lg * 32) << 16);
    int step = 0, buf = 0;
    bool ok = true;
    PaReader reader;
    PaItem next;
    while (reader.next(queue, next, abort_flag, p.status)) {
      const PackedFwdItem it(next);
      if (it.n < 0) break;
      const int row = it.row[g] + r128;
      int lo = PA_NONE;                        // first key of this row
      if (row < p.rows) {
        lo = plan.doc_lo[row];
        if (p.window > 0) lo = max(lo, row - p.window + 1);
      }
      const bool sees = lo <= row;
      const int tell = max(it.n - PA_EARLY, 0);
      if (it.n == 0 && threadIdx.x == 0) mbar_arrive(queue.want);
      float m = -INFINITY;                     // maximum (log2 units) that the sums are relative to
      float2 la = make_float2(0.f, 0.f), lb = la;
      for (int i = 0; i < it.n; ++i, ++step) {
        const int kv0 = (it.j0 + i) * PA_TILE;
        if (i == tell && threadIdx.x == 0) mbar_arrive(queue.want);
        ok = pa_wait(&s_full[g], step & 1, abort_flag, p.status, ST_PATTN_S);
        if (!ok) break;
        tc_fence_after();
        // keys first .. lastk of this tile are visible to this row
        const int first = max(lo - kv0, 0), lastk = sees ? min(row - kv0, 127) : -1;
        uint32_t vis = 0u;                     // 32-key chunks of the tile that some row of the warp sees
        const bool part = __any_sync(0xffffffffu, first > 0 || lastk < 127);
        if (part) {
          const bool none = first > lastk;
          const int from = __reduce_min_sync(0xffffffffu, none ? 128 : first), to = __reduce_max_sync(0xffffffffu, none ? -1 : lastk);
#pragma unroll
          for (int c = 0; c < 4; ++c) vis |= from <= 32 * c + 31 && to >= 32 * c ? 1u << c : 0u;
        }
        if (!part)
          pf_whole<DP>(s_addr, o_addr, p.scale_log2, m, la, lb, &p_full[g]);
        else
          pf_part<DP>(s_addr, o_addr, p.scale_log2, vis, first, lastk, m, la, lb, &p_full[g]);
      }
      if (!ok) break;
      // (The output warps are done with what the item before the last one left there.  They may not have looked at the last
      // one's yet, a tile with a short item behind it: so each buffer has its barrier.)
      if (it.n > 0) {
        stat_s[(buf * 2 + g) * 128 + r128] = make_float2((la.x + la.y) + (lb.x + lb.y), m);
        __syncwarp();
        if (lane == 0) mbar_arrive(&l_full[2 * buf + g]);
        buf ^= 1;
      }
    }
  } else {
    reg_dec<80>();
    // ------------------------------------------------------------ output: both tiles of an item, while the softmax warps are at
    // the next one (the time between an item's last probabilities and its stored rows is some 5 thousand cycles)
    const int lg = warp & 3, r128 = lg * 32 + lane;
    const int tiles = (p.rows + PA_TILE - 1) / PA_TILE;
    const bool wide = p.D % 16 == 0 && ((reinterpret_cast<size_t>(p.out) | 2 * reinterpret_cast<size_t>(p.rest)) & 31) == 0;
    int done = 0;
    bool ok = true;
    PaReader reader;
    PaItem next;
    while (ok && reader.next(queue, next, abort_flag, p.status)) {
      const PackedFwdItem it(next);
      if (it.n < 0) break;
#pragma unroll 1
      for (int g = 0; g < 2 && ok; ++g) {
        const int row = (g ? it.row[1] : it.row[0]) + r128, head = g ? it.head[1] : it.head[0];
        int lo = PA_NONE;                      // first key of this row
        if (row < p.rows) {
          lo = plan.doc_lo[row];
          if (p.window > 0) lo = max(lo, row - p.window + 1);
        }
        const bool sees = lo <= row;           // (a row that sees nothing gets zeros)
        float l = 0.f, m = 0.f;
        if (it.n > 0) {
          ok = pa_wait(&l_full[2 * (done & 1) + g], (done >> 1) & 1, abort_flag, p.status, ST_PATTN_OUT) &&
               pa_wait(&o_full[g], done & 1, abort_flag, p.status, ST_PATTN_OUT);
          if (!ok) break;
          tc_fence_after();
          const float2 st = stat_s[((done & 1) * 2 + g) * 128 + r128];
          l = st.x;
          m = st.y;
        }
        const uint32_t o_addr = tmem + 256 + g * 128 + (uint32_t(lg * 32) << 16);
        __nv_bfloat16* o_row = p.out + ((size_t)row * p.Hq + head) * p.D;
        int8_t* rest = p.rest ? p.rest + ((size_t)row * p.Hq + head) * p.D : nullptr;
        const float f = sees ? 1.f / l : 0.f;
        float sum = l;                         // finite if all of the row is (or as good as: else it is made again for nothing)
#pragma unroll 1
        for (int c = 0; c < DP; c += 16) {
          uint32_t o[16];
          if (it.n > 0) {
            pa_tmem_ld_16(o_addr + c, o);
            tmem_ld_wait();
            if (c + 16 == DP) {                // all read: the next item's products may come
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&o_empty[g]);
            }
          }
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            if (!sees) o[k] = 0u;
            sum += fabsf(__uint_as_float(o[k]));
          }
          if (row < p.rows && c < p.D) pa_put16(o_row + c, o, 0, f, wide, p.D - c, rest ? rest + c : nullptr);
        }
        if (row < tiles * PA_TILE) p.lse[(size_t)head * tiles * PA_TILE + row] = sees ? m + log2f(l) : INFINITY;
        for (uint32_t again = __ballot_sync(0xffffffffu, sees && !(pa_finite(sum) && l > 0.f)); again; again &= again - 1) {
          const int who = __ffs(again) - 1;
          __syncwarp();
          pf_redo(p, row - lane + who, head, __shfl_sync(0xffffffffu, lo, who), abort_flag);
          pa_redone(abort_flag);
        }
      }
      if (it.n > 0) ++done;
    }
  }

  // ---------------------------------------------------------------- teardown
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

template <int DP>
static int packed_fwd_launch(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const PackedFwdParams& p,
                             cudaStream_t stream) {
  const int tiles = (p.rows + PA_TILE - 1) / PA_TILE;
  const long items = p.head_pairs ? (long)tiles * (p.Hq / 2) : (long)((tiles + 1) / 2) * p.Hq;
  if (items > 0x3fffffff) return -12;
  SLAB_CUDA_CHECK(cudaFuncSetAttribute(packed_fwd_kernel<DP>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       PackedFwdSmem<DP>::TOTAL));
  const int grid = items < sm_count() ? (int)items : sm_count();
  if (items > grid) SLAB_CUDA_CHECK(cudaMemsetAsync(p.counter, 0, sizeof(int), stream));
  packed_fwd_kernel<DP><<<grid, PF_THREADS, PackedFwdSmem<DP>::TOTAL, stream>>>(mq, mk, mv, p, (int)items);
  return (int)cudaGetLastError();
}

}  // namespace slab

// int32 words of a plan for `rows` rows, 2^25 at most
extern "C" int slab_packed_plan_words(int rows) {
  if (rows <= 0 || rows > 1 << 25) return -10;
  const int* base = reinterpret_cast<const int*>(16);
  return (int)(slab::packed_plan(base, rows).end - base);
}

// cu [docs + 1] int32: rows of document s are cu[s] .. cu[s + 1] - 1
extern "C" int slab_packed_plan(const void* cu, int docs, int rows, void* plan, void* status, void* stream) {
  using namespace slab;
  if (rows <= 0 || docs < 0) return -10;
  const int tiles = (rows + PA_TILE - 1) / PA_TILE;
  cudaStream_t st = (cudaStream_t)stream;
  packed_bounds_kernel<<<tiles, PA_TILE, 0, st>>>((const int*)cu, docs, rows, (int*)plan, (int*)status);
  packed_order_kernel<<<tiles, 128, 0, st>>>(rows, (int*)plan);
  return (int)cudaGetLastError();
}

// The same from token ids [batch * seq] (int64): a document ends behind every `end` token and with every row of the batch.
// starts: scratch, 2 int32 per tile.
extern "C" int slab_packed_plan_tokens(const void* tokens, int rows, int seq, long end, void* starts, void* plan, void* stream) {
  using namespace slab;
  if (rows <= 0 || seq <= 0) return -10;
  const int tiles = (rows + PA_TILE - 1) / PA_TILE;
  cudaStream_t st = (cudaStream_t)stream;
  packed_starts_kernel<<<tiles, PA_TILE, 0, st>>>((const long long*)tokens, rows, seq, end, (int*)starts);
  packed_token_bounds_kernel<<<tiles, PA_TILE, 0, st>>>((const long long*)tokens, rows, seq, end, (const int*)starts, (int*)plan);
  packed_order_kernel<<<tiles, 128, 0, st>>>(rows, (int*)plan);
  return (int)cudaGetLastError();
}

// q [rows, Hq, D], k and v [rows, Hkv, D] bf16 with the given token and head strides (elements, multiples of 8; bases on 16
// bytes), out [rows, Hq, D] contiguous, rest the same in int8 or null (lower half of the output, on 8 bytes), lse [Hq, tiles * 128] fp32, counter: scratch, one int32.  D a multiple of 8 up to 128.
extern "C" int slab_packed_attn_fwd(const void* q, const void* k, const void* v, void* out, void* rest, void* lse,
                                    const void* plan,
                                    int rows, int hq, int hkv, int d, long q_ts, long q_hs, long k_ts, long k_hs, long v_ts,
                                    long v_hs, int window, float scale, void* counter, void* status, void* stream) {
  using namespace slab;
  if (rows <= 0 || hq <= 0 || hkv <= 0 || hq % hkv || d <= 0 || d > 128 || d % 8 || window < 0 || !(scale > 0.f)) return -10;
  if ((q_ts | q_hs | k_ts | k_hs | v_ts | v_hs) & 7) return -11;
  tma_need_context();
  CUtensorMap mq, mk, mv;
  int rc;
  if ((rc = pa_make_map(&mq, q, rows, hq, d, q_ts, q_hs)) != 0) return rc;
  if ((rc = pa_make_map(&mk, k, rows, hkv, d, k_ts, k_hs)) != 0) return rc;
  if ((rc = pa_make_map(&mv, v, rows, hkv, d, v_ts, v_hs)) != 0) return rc;
  PackedFwdParams p;
  p.out = (__nv_bfloat16*)out;
  p.rest = (int8_t*)rest;
  p.lse = (float*)lse;
  p.plan = (const int*)plan;
  p.q = {(const __nv_bfloat16*)q, q_ts, q_hs};
  p.k = {(const __nv_bfloat16*)k, k_ts, k_hs};
  p.v = {(const __nv_bfloat16*)v, v_ts, v_hs};
  p.rows = rows; p.Hq = hq; p.Hkv = hkv; p.D = d;
  p.window = window;
  p.head_pairs = (hq / hkv) % 2 == 0;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.counter = (int*)counter;
  p.status = (int*)status;
  return d <= 64 ? packed_fwd_launch<64>(mq, mk, mv, p, (cudaStream_t)stream)
                 : packed_fwd_launch<128>(mq, mk, mv, p, (cudaStream_t)stream);
}
