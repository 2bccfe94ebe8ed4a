// Entry points of the paged attention: argument checks, the choice of the kernel, and the kernel that joins items which were
// cut between CTAs.
#include <cmath>

#include "attention.cuh"

namespace zt {

namespace {

constexpr int kMaxBatch = 16384;   // the division of a batch keeps one int per sequence in shared memory
constexpr int kCombineWarps = 4;   // rows per block
constexpr int kMaxStreamRows = 32; // rows per kv head up to which a pass of the streaming kernel holds all of them

// Joins the pieces of the item that is cut at the end of CTA blockIdx.x's range: one warp per row, each lane DP / 32 columns.
// Bound by memory; the pieces are mostly still in L2.
template <typename T, int DP>
__global__ void __launch_bounds__(kCombineWarps * 32) attention_combine_kernel(const __grid_constant__ AttnParams p, int R) {
  grid_launch_dependents();
  grid_dependency_wait();
  const int4 item = p.meta[blockIdx.x].cut;
  if (item.x < 0) return;
  const int row = blockIdx.y * kCombineWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (row >= item.z % 512) return;
  const int first = blockIdx.x, count = item.w - first + 1;
  constexpr int V = DP / 32, BATCH = 8;
  using Vec = std::conditional_t<V == 4, float4, float2>;
  float acc[V] = {}, sum = 0.f, top = -INFINITY;
  for (int i = 0; i < count; i += BATCH) {
    float2 ml[BATCH];
    Vec x[BATCH];
    float to = top;
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      ml[u] = make_float2(-INFINITY, 0.f), x[u] = Vec{};
      if (i + u < count) {
        const int64_t at = (int64_t)(2 * (first + i + u) + (i + u == 0 ? 1 : 0)) * R + row;
        ml[u] = p.part_ml[at];
        x[u] = *reinterpret_cast<const Vec *>(p.part_o + at * DP + lane * V);
      }
    }
#pragma unroll
    for (int u = 0; u < BATCH; ++u) to = fmaxf(to, ml[u].x);
    const float f_old = top == -INFINITY ? 0.f : exp2_fast(top - to);
    sum *= f_old;
#pragma unroll
    for (int v = 0; v < V; ++v) acc[v] *= f_old;
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      const float f = ml[u].x == -INFINITY ? 0.f : exp2_fast(ml[u].x - to);
      sum += ml[u].y * f;
#pragma unroll
      for (int v = 0; v < V; ++v) acc[v] = fmaf(f, reinterpret_cast<const float *>(&x[u])[v], acc[v]);
    }
    top = to;
  }
  if (lane * V >= p.d) return;
  const float f = top == -INFINITY ? 0.f : 1.f / sum;
  const int r = item.y + row, tok = r / p.group, qh = item.z / 512 * p.group + r % p.group;
  char *dst = reinterpret_cast<char *>(p.out) + ((item.x + tok) * p.o_st + qh * p.o_sh + lane * V) * 2;
  if constexpr (V == 4)
    *reinterpret_cast<uint2 *>(dst) = make_uint2(pack2(acc[0] * f, acc[1] * f, T(0.f)), pack2(acc[2] * f, acc[3] * f, T(0.f)));
  else
    *reinterpret_cast<uint32_t *>(dst) = pack2(acc[0] * f, acc[1] * f, T(0.f));
}

// One element of a cache.
template <typename T, bool E4M3>
__device__ __forceinline__ float cache_value(const void *base, int64_t at) {
  if constexpr (E4M3) {
    const uint2 h = e4m3x4_to_f16x4(reinterpret_cast<const uint8_t *>(base)[at]);
    return unpack2(h.x, __half(0.f)).x;
  } else {
    return (float)reinterpret_cast<const T *>(base)[at];
  }
}

// Goes through a row of the output again, by one warp, where it is not finite: unless its query or a key that it sees holds a NaN, or
// the values that it sees account for every such column, the row is computed from those keys alone.  A NaN is accounted for by
// a NaN or by infinities of both signs, an infinity by one of its sign: 0 times the value of a key that the row does not see makes a NaN
// of an infinity that it does see.
template <typename T, bool E4M3>
__device__ __noinline__ void redo_row(const AttnParams &p, int b, const SeqInfo &seq, int head, int r) {
  constexpr int V = 4;                                   // columns of a lane
  const int lane = threadIdx.x & 31, tok = r / p.group, qh = head * p.group + r % p.group;
  const int lo = key_lo(p, seq, tok), hi = key_hi(p, seq, tok);
  T *out = reinterpret_cast<T *>(p.out) + (seq.q0 + tok) * p.o_st + qh * p.o_sh;
  const T *q = reinterpret_cast<const T *>(p.q) + (seq.q0 + tok) * p.q_st + qh * p.q_sh;
  auto row_of = [&](int key, int64_t sp, int64_t ss, int64_t sh) -> int64_t {      // -1: no such page
    const int id = p.table[b * p.table_stride + page_of(p, key)];
    return id >= 0 && id < p.num_pages ? id * sp + (key - page_of(p, key) * p.page) * ss + head * sh : -1;
  };
  uint32_t nans = 0, infs[2] = {0, 0};                   // this lane's columns that are NaN, infinite (positive, negative)
  uint32_t seen_nan = 0, seen_inf[2] = {0, 0};           // columns with such a value among the keys that the row sees
  auto note = [](float x, int e, uint32_t &is_nan, uint32_t (&is_inf)[2]) {
    if (isnan(x)) is_nan |= 1u << e;
    else if (isinf(x)) is_inf[x < 0.f] |= 1u << e;
  };
  auto open = [&]() {                                    // columns that want an explanation
    return (nans & ~(seen_nan | (seen_inf[0] & seen_inf[1]))) | (infs[0] & ~seen_inf[0]) | (infs[1] & ~seen_inf[1]);
  };
#pragma unroll
  for (int e = 0; e < V; ++e)
    if (lane * V + e < p.d) note((float)out[lane * V + e], e, nans, infs);
  if (!__any_sync(0xffffffffu, open() != 0)) return;
  bool nan = false;
#pragma unroll
  for (int e = 0; e < V; ++e)
    if (lane * V + e < p.d) nan |= isnan((float)q[lane * V + e]);
  if (hi > lo && __any_sync(0xffffffffu, nan)) return;
  for (int key = hi - 1; key >= lo && __any_sync(0xffffffffu, open() != 0); --key) {
    const int64_t at = row_of(key, p.v_sp, p.v_ss, p.v_sh), k_at = row_of(key, p.k_sp, p.k_ss, p.k_sh);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      if (at < 0 || lane * V + e >= p.d) continue;
      note(cache_value<T, E4M3>(p.v, at + lane * V + e), e, seen_nan, seen_inf);
      nan |= isnan(cache_value<T, E4M3>(p.k, k_at + lane * V + e));
    }
    if (__any_sync(0xffffffffu, nan)) return;
  }
  if (!__any_sync(0xffffffffu, open() != 0)) return;
  const float mul = p.scale_log2 * (E4M3 ? p.k_scale[head] : 1.f);
  float acc[V] = {}, special[V] = {}, top = -INFINITY, sum = 0.f;      // special: values that are not finite, which no factor may touch
  for (int first = lo; first < hi; first += 32) {        // a key per lane, then its value by all lanes
    const int key = first + lane;
    float s = -INFINITY;
    if (key < hi) {
      const int64_t at = row_of(key, p.k_sp, p.k_ss, p.k_sh);
      s = 0.f;
      if (at >= 0)
        for (int e = 0; e < p.d; ++e) s = fmaf((float)q[e], cache_value<T, E4M3>(p.k, at + e), s);
      s *= mul;
    }
    float to = s;
#pragma unroll
    for (int o = 16; o; o >>= 1) to = fmaxf(to, __shfl_xor_sync(0xffffffffu, to, o));
    to = fmaxf(to, top);
    const float f = top == -INFINITY ? 0.f : exp2_fast(top - to), x = key < hi ? exp2_fast(s - (to == -INFINITY ? 0.f : to)) : 0.f;
    top = to;
    sum = sum * f + x;
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] *= f;
    for (int i = 0; i < min(32, hi - first); ++i) {
      const float xi = __shfl_sync(0xffffffffu, x, i);
      const int64_t at = row_of(first + i, p.v_sp, p.v_ss, p.v_sh);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        if (at < 0 || lane * V + e >= p.d) continue;
        const float v = cache_value<T, E4M3>(p.v, at + lane * V + e);
        if (isfinite(v)) acc[e] = fmaf(xi, v, acc[e]);
        else special[e] += v;
      }
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const float f = sum == 0.f ? 0.f : (E4M3 ? p.v_scale[head] : 1.f) / sum;
#pragma unroll
  for (int e = 0; e < V; ++e)
    if (lane * V + e < p.d) out[lane * V + e] = (T)(acc[e] * f + special[e]);
}

// The same for the pieces of the tcgen05 kernel, whose rows are neighbours in the workspace: a lane per row, a warp per 16 columns.
// A block whose CTA found outputs that are not finite goes through the rows of its items again.
template <typename T, bool E4M3, int DP>
__global__ void __launch_bounds__(DP * 2) attention_combine_rows_kernel(const __grid_constant__ AttnParams p, int R) {
  grid_launch_dependents();
  grid_dependency_wait();
  const AttnMeta &meta = p.meta[blockIdx.x];
  const int4 item = meta.cut;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row = blockIdx.y * 32 + lane, c0 = warp * 16;
  bool redo = meta.not_finite;
  if (item.x >= 0) {
    const int first = blockIdx.x, count = item.w - first + 1, n_rows = item.z % 512;
    if (row < n_rows && c0 < p.d) {
      auto slot = [&](int i) { return (int64_t)(2 * (first + i) + (i == 0 ? 1 : 0)); };
      float acc[16] = {}, sum = 0.f, top = -INFINITY;
      for (int i = 0; i < count; ++i) {
        const float2 ml = p.part_ml[slot(i) * R + row];
        const float4 *src = reinterpret_cast<const float4 *>(p.part_o) + (slot(i) * (DP / 4) + c0 / 4) * R + row;
        float4 x[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) x[q] = src[(int64_t)q * R];
        const float to = fmaxf(top, ml.x);
        const float f_old = top == -INFINITY ? 0.f : exp2_fast(top - to), f = ml.x == -INFINITY ? 0.f : exp2_fast(ml.x - to);
        top = to;
        sum = sum * f_old + ml.y * f;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          acc[4 * q] = acc[4 * q] * f_old + x[q].x * f, acc[4 * q + 1] = acc[4 * q + 1] * f_old + x[q].y * f;
          acc[4 * q + 2] = acc[4 * q + 2] * f_old + x[q].z * f, acc[4 * q + 3] = acc[4 * q + 3] * f_old + x[q].w * f;
        }
      }
      const float f = top == -INFINITY ? 0.f : 1.f / sum;
      const int r = item.y + row, tok = r / p.group, qh = item.z / 512 * p.group + r % p.group;
      uint4 *dst = reinterpret_cast<uint4 *>(reinterpret_cast<char *>(p.out) + ((item.x + tok) * p.o_st + qh * p.o_sh + c0) * 2);
#pragma unroll
      for (int q = 0; q < 2; ++q)
        if (c0 + 8 * q < p.d)
          dst[q] = make_uint4(pack2(acc[8 * q] * f, acc[8 * q + 1] * f, T(0.f)), pack2(acc[8 * q + 2] * f, acc[8 * q + 3] * f, T(0.f)),
                              pack2(acc[8 * q + 4] * f, acc[8 * q + 5] * f, T(0.f)), pack2(acc[8 * q + 6] * f, acc[8 * q + 7] * f, T(0.f)));
    }
    int others = 0;       // any CTA that worked on the cut item
    for (int i = 1 + lane; i < count; i += 32) others |= p.meta[first + i].not_finite;
    redo |= __any_sync(0xffffffffu, others) != 0;
  }
  if (!redo) return;
  __syncthreads();        // this block's part of the cut item is written
  if (item.x >= 0) {
    const SeqInfo seq = load_seq(p, meta.cut_b);
    for (int i = warp; i < 32; i += DP * 2 / 32)
      if (blockIdx.y * 32 + i < item.z % 512) redo_row<T, E4M3>(p, meta.cut_b, seq, item.z / 512, item.y + blockIdx.y * 32 + i);
  }
  if (!meta.not_finite) return;
  AttnWalk<kTcgen05Rows, kTcgen05Unit, kTcgen05Extra> it(meta.range);
  while (it.next(p)) {
    if (!it.whole) continue;      // (the block of the item's first CTA has it)
    for (int i = warp; i < 32; i += DP * 2 / 32)
      if (blockIdx.y * 32 + i < it.n_rows) redo_row<T, E4M3>(p, it.b, it.seq, it.head, it.r0 + blockIdx.y * 32 + i);
  }
}

template <typename T, bool E4M3>
cudaError_t launch_combine(const AttnParams &p, const AttnPlan &plan, cudaStream_t st) {
  if (plan.tcgen05) {
    const dim3 grid((unsigned)plan.grid, (unsigned)(plan.rows / 32)), block((unsigned)plan.dp * 2);
    return plan.dp == 64 ? launch_overlapped(attention_combine_rows_kernel<T, E4M3, 64>, grid, block, (size_t)0, st, p, plan.rows)
                         : launch_overlapped(attention_combine_rows_kernel<T, E4M3, 128>, grid, block, (size_t)0, st, p, plan.rows);
  }
  const dim3 grid((unsigned)plan.grid, (unsigned)ceil_div(plan.rows, kCombineWarps)), block(kCombineWarps * 32);
  return plan.dp == 64 ? launch_overlapped(attention_combine_kernel<T, 64>, grid, block, (size_t)0, st, p, plan.rows)
                       : launch_overlapped(attention_combine_kernel<T, 128>, grid, block, (size_t)0, st, p, plan.rows);
}

size_t align256(size_t v) { return (v + 255) / 256 * 256; }

// CTAs per sequence and kv head where block_table has room for `keys` keys each, 0: the units are dealt out.  A CTA takes 1 us for
// 64 keys, dealing and joining about 4 us, and clusters of 512 and more CTAs take longer to place than they save.  Many items even
// themselves out as they come, but one long sequence among short ones is left to its CTA: hence the bound there too.  Direct against
// dealt, ragged lengths of keys / 10 to keys (bf16, groups of 4), in us: 8 items of 4096 keys 6.6 / 10.1 (8 CTAs each), 32 of 4096
// 9.9 / 12.6 (8), 128 of 1024 11.9 / 13.0 (2) and of 2048 17.6 / 15.3, 512 of 320 12.2 / 16.5 (1), of 768 25.2 / 28.0 and of 2048
// 57.4 / 57.5, 2048 of 768 72 / 77 and of 2048 171 / 179 (e4m3: 100 / 120).
int direct_slices(int64_t keys, int64_t items, int ctas) {
  int s = 8;
  while (s > 1 && (items * s > 256 || keys <= 64 * s)) s /= 2;
  return keys <= (items >= 2 * ctas ? 2048 : 768 * s) ? s : 0;
}

AttnPlan make_plan(const zt_paged_attention_args_t &a) {
  AttnPlan plan{};
  const int group = a.kv_heads > 0 ? a.q_heads / a.kv_heads : 1;
  // rows that the longest piece of new tokens gives a kv head
  const int64_t bound = a.tokens - a.batch + 1 > 1 ? a.tokens - a.batch + 1 : 1;
  const int64_t longest = a.max_query_len > 0 && a.max_query_len < bound ? a.max_query_len : bound;
  const int64_t rows = longest * group;
  const int algo = a.algo & 0xff, hint = (a.algo >> 8) & 0xffff;
  plan.tcgen05 = algo == ZT_ALGO_TCGEN05 || (algo == ZT_ALGO_AUTO && rows > kMaxStreamRows);
  plan.dp = a.head_dim <= 64 ? 64 : 128;
  plan.rows = plan.tcgen05 ? kTcgen05Rows : rows <= 8 ? 8 : rows <= 16 ? 16 : 32;
  plan.grid = plan.tcgen05 ? sm_count() : attention_stream_grid(plan.rows);
  plan.few = rows <= 4 * plan.rows;
  const int64_t keys = (int64_t)a.page_size * a.max_blocks, items = (int64_t)a.batch * a.kv_heads;
  if (!plan.tcgen05 && items > 0) plan.slices = hint ? (hint == 1 ? 0 : hint - 1) : direct_slices(keys, items, plan.grid);
  if (plan.slices > 0) {
    plan.grid = 0;      // nothing is kept between CTAs
    return plan;
  }
  // units of the whole call at most (an item has up to three beside those of its keys)
  const int64_t unit = plan.tcgen05 ? 128 : 64, tiles = a.tokens * group / plan.rows + a.batch;
  plan.most_units = (double)tiles * a.kv_heads * (double)((int64_t)a.page_size * a.max_blocks / unit + 4);
  plan.meta_bytes = align256((size_t)plan.grid * sizeof(AttnMeta));
  plan.ml_bytes = align256((size_t)2 * plan.grid * plan.rows * sizeof(float2));
  plan.o_bytes = align256((size_t)2 * plan.grid * plan.rows * plan.dp * sizeof(float));
  return plan;
}

bool aligned(const void *ptr, const int64_t *strides, int n, int elem_bytes) {
  int64_t s = (int64_t)(reinterpret_cast<uintptr_t>(ptr) % 16);
  for (int i = 0; i < n; ++i) s |= strides[i] * elem_bytes;
  return s % 16 == 0;
}

}  // namespace
}  // namespace zt

using namespace zt;

extern "C" size_t zt_paged_attention_workspace_bytes(const zt_paged_attention_args_t *a) {
  if (!a || a->tokens <= 0 || a->q_heads <= 0 || a->kv_heads <= 0) return 256;
  return make_plan(*a).total();
}

extern "C" int zt_paged_attention(const zt_paged_attention_args_t *a, void *stream) {
  ZT_REQUIRE(a != nullptr, ZT_INVALID_ARGUMENT, "zt_paged_attention: null argument block");
  ZT_REQUIRE(a->tokens >= 0 && a->batch >= 0 && a->max_blocks >= 0 && a->num_pages >= 0 && a->max_query_len >= 0, ZT_INVALID_ARGUMENT,
             "zt_paged_attention: negative size");
  ZT_REQUIRE(a->tokens <= (1 << 30) && a->num_pages <= (1 << 30), ZT_UNSUPPORTED, "zt_paged_attention: more than 2^30 tokens or pages");
  ZT_REQUIRE(a->q_heads <= 0 || a->tokens * a->q_heads < (1 << 30), ZT_UNSUPPORTED, "zt_paged_attention: 2^30 or more query rows");
  ZT_REQUIRE(a->batch <= kMaxBatch, ZT_UNSUPPORTED, "zt_paged_attention: %d sequences, at most %d", a->batch, kMaxBatch);
  ZT_REQUIRE(a->q_heads >= 1 && a->kv_heads >= 1 && a->q_heads % a->kv_heads == 0 && a->q_heads <= 4096, ZT_INVALID_ARGUMENT,
             "zt_paged_attention: the query heads (%d) must be a multiple of the key/value heads (%d)", a->q_heads, a->kv_heads);
  ZT_REQUIRE(a->dtype == ZT_BF16 || a->dtype == ZT_F16, ZT_INVALID_ARGUMENT, "zt_paged_attention: query must be bfloat16 or float16");
  ZT_REQUIRE(a->cache_dtype == a->dtype || a->cache_dtype == ZT_E4M3, ZT_INVALID_ARGUMENT,
             "zt_paged_attention: the cache must have the type of the query or be float8_e4m3");
  const bool e4m3 = a->cache_dtype == ZT_E4M3;
  ZT_REQUIRE(a->head_dim >= 8 && a->head_dim <= 128 && a->head_dim % (e4m3 ? 16 : 8) == 0, ZT_UNSUPPORTED,
             "zt_paged_attention: head_dim must be a multiple of %d up to 128, got %d", e4m3 ? 16 : 8, a->head_dim);
  ZT_REQUIRE(a->page_size >= 1, ZT_INVALID_ARGUMENT, "zt_paged_attention: the page size must be positive");
  ZT_REQUIRE((int64_t)a->page_size * a->max_blocks <= (1 << 30), ZT_UNSUPPORTED,
             "zt_paged_attention: block_table holds more than 2^30 keys per sequence");
  ZT_REQUIRE(a->window >= 0, ZT_INVALID_ARGUMENT, "zt_paged_attention: the window must not be negative");
  ZT_REQUIRE(std::isfinite(a->scale) && a->scale > 0.f, ZT_INVALID_ARGUMENT, "zt_paged_attention: the scale must be positive and finite");
  ZT_REQUIRE(!e4m3 || (a->k_scale && a->v_scale), ZT_INVALID_ARGUMENT,
             "zt_paged_attention: a float8_e4m3 cache needs k_scale and v_scale");
  const int algo = a->algo & 0xff, hint = (a->algo >> 8) & 0xffff;
  ZT_REQUIRE((algo == ZT_ALGO_AUTO || algo == ZT_ALGO_SKINNY || algo == ZT_ALGO_TCGEN05) && a->algo >> 24 == 0 && hint <= 9, ZT_INVALID_ARGUMENT,
             "zt_paged_attention: unknown algo %d", a->algo);
  if (a->tokens == 0) return ZT_SUCCESS;
  ZT_REQUIRE(a->q && a->out && a->cu_seqlens_q, ZT_INVALID_ARGUMENT, "zt_paged_attention: null tensor pointer");
  ZT_REQUIRE(a->batch == 0 || (a->seq_lens && (a->max_blocks == 0 || a->block_table)), ZT_INVALID_ARGUMENT,
             "zt_paged_attention: null tensor pointer");
  ZT_REQUIRE(a->num_pages == 0 || (a->k_cache && a->v_cache), ZT_INVALID_ARGUMENT, "zt_paged_attention: null cache pointer");
  const int es = e4m3 ? 1 : 2;
  ZT_REQUIRE(aligned(a->q, a->q_stride, 2, 2) && aligned(a->out, a->out_stride, 2, 2), ZT_INVALID_ARGUMENT,
             "zt_paged_attention: rows of query and output must be 16-byte aligned");
  ZT_REQUIRE(a->num_pages == 0 || (aligned(a->k_cache, a->k_cache_stride, 3, es) && aligned(a->v_cache, a->v_cache_stride, 3, es)),
             ZT_INVALID_ARGUMENT, "zt_paged_attention: rows of the caches must be 16-byte aligned");
  const AttnPlan plan = make_plan(*a);
  ZT_REQUIRE(plan.most_units < 2147483648.0, ZT_UNSUPPORTED, "zt_paged_attention: more work than one call can number");
  ZT_REQUIRE(plan.total() == 0 || (a->workspace && a->workspace_bytes >= plan.total()), ZT_WORKSPACE_TOO_SMALL,
             "zt_paged_attention: workspace of %zu bytes is smaller than the %zu required", a->workspace_bytes, plan.total());
  ZT_REQUIRE((reinterpret_cast<uintptr_t>(a->workspace) & 255) == 0, ZT_INVALID_ARGUMENT,
             "zt_paged_attention: workspace must be 256-byte aligned");
  int *status = device_status_ptr();
  ZT_REQUIRE(status != nullptr, ZT_CUDA_ERROR, "zt_paged_attention: no device status word");

  AttnParams p{};
  p.q = a->q, p.out = a->out, p.k = a->k_cache, p.v = a->v_cache;
  p.q_st = a->q_stride[0], p.q_sh = a->q_stride[1], p.o_st = a->out_stride[0], p.o_sh = a->out_stride[1];
  p.k_sp = a->k_cache_stride[0], p.k_ss = a->k_cache_stride[1], p.k_sh = a->k_cache_stride[2];
  p.v_sp = a->v_cache_stride[0], p.v_ss = a->v_cache_stride[1], p.v_sh = a->v_cache_stride[2];
  p.cu = a->cu_seqlens_q, p.lens = a->seq_lens, p.table = a->block_table, p.table_stride = a->block_table_stride;
  p.k_scale = e4m3 ? a->k_scale : nullptr, p.v_scale = e4m3 ? a->v_scale : nullptr;
  p.batch = a->batch, p.tokens = (int)a->tokens, p.hq = a->q_heads, p.hkv = a->kv_heads, p.group = a->q_heads / a->kv_heads;
  p.d = a->head_dim, p.page = a->page_size, p.max_blocks = a->max_blocks, p.num_pages = (int)a->num_pages;
  p.page_shift = -1;
  for (int s = 0; s < 31; ++s)
    if (a->page_size == 1 << s) p.page_shift = s;
  p.causal = a->causal != 0, p.window = a->window < 1 << 30 ? a->window : 1 << 30 /* no context is longer */, p.scale_log2 = a->scale * 1.4426950408889634f, p.zero_tail = a->zero_tail != 0, p.few = plan.few, p.slices = plan.slices;
  char *ws = reinterpret_cast<char *>(a->workspace);
  p.meta = reinterpret_cast<AttnMeta *>(ws);
  p.part_ml = reinterpret_cast<float2 *>(ws + plan.meta_bytes);
  p.part_o = reinterpret_cast<float *>(ws + plan.meta_bytes + plan.ml_bytes);
  p.status = status;

  cudaStream_t st = (cudaStream_t)stream;
  const int rc = plan.tcgen05 ? attention_tcgen05_launch(p, plan, a->dtype, a->cache_dtype, st)
                              : attention_stream_launch(p, plan, a->dtype, a->cache_dtype, st);
  if (rc != ZT_SUCCESS || plan.slices > 0) return rc;
  ZT_CUDA_OK(a->dtype == ZT_BF16 ? (e4m3 ? launch_combine<__nv_bfloat16, true>(p, plan, st) : launch_combine<__nv_bfloat16, false>(p, plan, st))
                                 : (e4m3 ? launch_combine<__half, true>(p, plan, st) : launch_combine<__half, false>(p, plan, st)));
  return launch_status("attention_combine_kernel");
}
