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

// Four neighbouring elements of a cache.
template <typename T, bool E4M3>
__device__ __forceinline__ float4 cache_values(const void *base, int64_t at) {
  float2 lo, hi;
  if constexpr (E4M3) {
    const uint2 h = e4m3x4_to_f16x4(*reinterpret_cast<const uint32_t *>(reinterpret_cast<const uint8_t *>(base) + at));
    lo = unpack2(h.x, __half(0.f)), hi = unpack2(h.y, __half(0.f));
  } else {
    const uint2 w = *reinterpret_cast<const uint2 *>(reinterpret_cast<const T *>(base) + at);
    lo = unpack2(w.x, T(0.f)), hi = unpack2(w.y, T(0.f));
  }
  return make_float4(lo.x, lo.y, hi.x, hi.y);
}
template <typename T, bool E4M3>
__device__ __forceinline__ uint32_t not_finite_bits(uint32_t w) {
  if constexpr (E4M3) return not_finite_mask_e4m3(w);
  else return not_finite_mask(w, T(0.f));
}

constexpr int kRedoWords = 16;     // flags of a block that goes through rows again

// Which of some columns hold NaN or an infinity (positive, negative), a bit per column.
struct Special {
  uint32_t nan, inf[2];
  __device__ __forceinline__ void note(float x, int e) {
    if (isnan(x)) nan |= 1u << e;
    else if (isinf(x)) inf[x < 0.f] |= 1u << e;
  }
  __device__ __forceinline__ void note(float4 x) { note(x.x, 0), note(x.y, 1), note(x.z, 2), note(x.w, 3); }
  // Columns of an output that the values `seen` do not account for: a NaN comes of a NaN or of infinities of both signs, an infinity of
  // one of its sign.
  __device__ __forceinline__ uint32_t open(const Special &seen) const {
    return (nan & ~(seen.nan | (seen.inf[0] & seen.inf[1]))) | (inf[0] & ~seen.inf[0]) | (inf[1] & ~seen.inf[1]);
  }
};

// Goes through up to 32 neighbouring rows of an item again, by the whole block: of those whose output is not finite, unless the
// query or a key that the row sees holds a NaN, or the values that it sees account for every such column, a row is computed from
// the keys that it sees alone.  (0 times the value of a key that a row does not see is NaN where that is not finite, and makes a
// NaN of an infinity that the row does see.)
//
// The keys that all of the rows see are gone through once, by all threads; those at either end, which differ by as many tokens as there
// are rows, by a warp per row; sums are taken again four rows at a time.  With NaN among the values that most rows see, a prompt of 2048
// tokens (32 heads over 8 of 128) takes 0.5 ms instead of 0.06.  Rows that are computed again are at most a tile of rows per kv head and
// value: with NaN in the last value of 8000, which 252 rows of a chunk's last tile do not see, 8 ms instead of 0.08.  (One key after
// another in every row: 38 and 114 ms.)
template <typename T, bool E4M3, int DP>
__device__ __noinline__ void redo_rows(const AttnParams &p, int b, const SeqInfo &seq, int head, int r0, int n) {
  constexpr int NT = DP * 2, WARPS = NT / 32, PER = E4M3 ? 16 : 8, CH = DP / PER, STEP = NT / CH, AHEAD = 4;
  // flags of this block: a word per 32 columns for NaN and infinities of either sign, and whether a key holds a NaN
  // (behind the pieces in the workspace)
  uint32_t *flags = reinterpret_cast<uint32_t *>(p.part_o + (int64_t)2 * gridDim.x * kTcgen05Rows * DP) + (blockIdx.x * gridDim.y + blockIdx.y) * kRedoWords;
  uint32_t *key_nan = flags + kRedoWords - 1;
  auto seen_by_all = [&](int kind, int col) { return __ldcg(flags + 4 * kind + col / 32) >> col % 32; };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c4 = lane * 4;      // (of a row, a lane has four columns)
  auto slot_of = [&](int key, int64_t &k_at, int64_t &v_at) -> bool {             // false: no such page (zeros)
    const int page = page_of(p, key), id = p.table[b * p.table_stride + page], slot = key - page * p.page;
    k_at = id * p.k_sp + slot * p.k_ss + head * p.k_sh, v_at = id * p.v_sp + slot * p.v_ss + head * p.v_sh;
    return id >= 0 && id < p.num_pages;
  };
  auto out_row = [&](int r) { return reinterpret_cast<T *>(p.out) + (seq.q0 + r / p.group) * p.o_st + (head * p.group + r % p.group) * p.o_sh; };
  auto query_row = [&](int r) { return reinterpret_cast<const T *>(p.q) + (seq.q0 + r / p.group) * p.q_st + (head * p.group + r % p.group) * p.q_sh; };
  auto has_nan = [](float4 x) { return isnan(x.x) || isnan(x.y) || isnan(x.z) || isnan(x.w); };
  auto special_outputs = [&](int r) {
    Special x{0, {0, 0}};
    if (c4 < p.d) x.note(cache_values<T, false>(out_row(r), c4));
    return x;
  };

  __syncthreads();            // the flags of an earlier call have been read
  if (threadIdx.x < kRedoWords) flags[threadIdx.x] = 0;
  bool any = false;
  for (int i = warp; i < n; i += WARPS) any |= special_outputs(r0 + i).open({0, {0, 0}}) != 0;
  if (!__syncthreads_or(any)) return;

  // ---- the keys that all rows see ----
  int all_lo = key_lo(p, seq, (r0 + n - 1) / p.group), all_hi = key_hi(p, seq, r0 / p.group);
  {
    const int c = threadIdx.x % CH * PER, sub = threadIdx.x / CH;
    for (int first = all_lo, round = 1; first < all_hi; first += AHEAD * STEP, ++round) {
      uint4 k[AHEAD], v[AHEAD];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int key = first + u * STEP + sub;
        int64_t k_at, v_at;
        k[u] = v[u] = make_uint4(0, 0, 0, 0);
        if (key < all_hi && c < p.d && slot_of(key, k_at, v_at)) {
          constexpr int ES = E4M3 ? 1 : 2;
          k[u] = *reinterpret_cast<const uint4 *>(reinterpret_cast<const char *>(p.k) + (k_at + c) * ES);
          v[u] = *reinterpret_cast<const uint4 *>(reinterpret_cast<const char *>(p.v) + (v_at + c) * ES);
        }
      }
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const uint32_t kw[4] = {k[u].x, k[u].y, k[u].z, k[u].w}, vw[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (not_finite_bits<T, E4M3>(kw[e])) {
            bool nan = true;
            if constexpr (!E4M3) {
              const float2 x = unpack2(kw[e], T(0.f));
              nan = isnan(x.x) || isnan(x.y);
            }
            if (nan) *key_nan = 1;
          }
          if (const uint32_t bad = not_finite_bits<T, E4M3>(vw[e])) {
            Special x{0, {0, 0}};
            int at = c + e * (PER / 4);
            if constexpr (E4M3) {
              x.nan = (bad & 1) | (bad >> 7 & 2) | (bad >> 14 & 4) | (bad >> 21 & 8);
            } else {
              const float2 f = unpack2(vw[e], T(0.f));
              x.note(f.x, 0), x.note(f.y, 1);
            }
            const uint32_t bits[3] = {x.nan, x.inf[0], x.inf[1]};
#pragma unroll
            for (int kind = 0; kind < 3; ++kind)
              if (bits[kind]) atomicOr(flags + 4 * kind + at / 32, bits[kind] << at % 32);
          }
        }
      }
      if (round % 16 == 0) {      // a key of NaN, or values of NaN in all columns: nothing else matters
        bool done = false;
        if (threadIdx.x == 0) {
          done = true;
          for (int col = 0; col < p.d; col += 8) done &= (seen_by_all(0, col) & 0xffu) == 0xffu;
          done |= __ldcg(key_nan) != 0;
        }
        if (__syncthreads_or(done)) return;
      }
    }
  }
  __syncthreads();
  if (__ldcg(key_nan)) return;

  // ---- the keys that not all of them see, a row per warp: which rows need their sums again ----
  constexpr int ROWS = 32 / WARPS, G = 4;                // a warp's rows, neighbours; of those, at once
  uint32_t todo = 0, mine[ROWS];                         // mine: NaN, infinities among the values that a row sees, in this lane's columns
#pragma unroll 1
  for (int i = 0; i < ROWS; ++i) {
    mine[i] = 0;
    if (warp * ROWS + i >= n) continue;
    const int r = r0 + warp * ROWS + i, tok = r / p.group, lo = key_lo(p, seq, tok), hi = key_hi(p, seq, tok);
    const Special out = special_outputs(r);
    Special seen{0, {0, 0}};
    if (c4 < p.d) seen = {seen_by_all(0, c4) & 15, {seen_by_all(1, c4) & 15, seen_by_all(2, c4) & 15}};
    if (!__any_sync(0xffffffffu, out.open(seen) != 0)) continue;
    bool nan = false;
    if (c4 < p.d && hi > lo) nan = has_nan(cache_values<T, false>(query_row(r), c4));
    const bool some = all_hi > all_lo;
    const int before = max((some ? all_lo : hi) - lo, 0), after = some ? max(hi - all_hi, 0) : 0;
    for (int j0 = 0; j0 < before + after; j0 += 32) {
      const int j = j0 + lane;
      int64_t k_at = 0, v_at = 0;
      const bool live = j < before + after && slot_of(j < before ? lo + j : all_hi + (j - before), k_at, v_at);
      const uint32_t lives = __ballot_sync(0xffffffffu, live);
#pragma unroll 4
      for (int u = 0; u < 32; ++u) {
        const int64_t ka = __shfl_sync(0xffffffffu, k_at, u), va = __shfl_sync(0xffffffffu, v_at, u);
        if (!(lives >> u & 1) || c4 >= p.d) continue;
        seen.note(cache_values<T, E4M3>(p.v, va + c4));
        nan |= has_nan(cache_values<T, E4M3>(p.k, ka + c4));
      }
    }
    mine[i] = seen.nan | seen.inf[0] << 4 | seen.inf[1] << 8;
    if (!__any_sync(0xffffffffu, nan) && __any_sync(0xffffffffu, out.open(seen) != 0)) todo |= 1u << i;
  }

  // ---- their sums, four rows at a time over the finite values ----
  const float mul = p.scale_log2 * (E4M3 ? p.k_scale[head] : 1.f), v_scale = E4M3 ? p.v_scale[head] : 1.f;
  const int c = lane % CH * PER, sub = lane / CH;        // of a key's row: this lane's elements; key of a load
#pragma unroll 1
  for (int g = 0; g < ROWS; g += G) {
    if (!(todo >> g & 15)) continue;
    uint4 q[G][PER / 8];
    int lo[G], hi[G], first = 1 << 30, last = 0;
    float acc[G][4] = {}, top[G], sum[G];
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const bool does = todo >> (g + i) & 1;
      const int r = r0 + warp * ROWS + g + (does ? i : __ffs(todo >> g & 15) - 1), tok = r / p.group;
      lo[i] = does ? key_lo(p, seq, tok) : 0, hi[i] = does ? key_hi(p, seq, tok) : 0;
      if (hi[i] > lo[i]) first = min(first, lo[i]), last = max(last, hi[i]);
      top[i] = -INFINITY, sum[i] = 0.f;
#pragma unroll
      for (int h = 0; h < PER / 8; ++h)
        q[i][h] = c + 8 * h < p.d ? *reinterpret_cast<const uint4 *>(query_row(r) + c + 8 * h) : make_uint4(0, 0, 0, 0);
    }
    for (; first < last; first += 32) {                  // a key per lane, then its value by all lanes
      int64_t k_at = 0, v_at = 0;
      const bool live = first + lane < last && slot_of(first + lane, k_at, v_at);
      const uint32_t lives = __ballot_sync(0xffffffffu, live);
      float x[G] = {};
#pragma unroll 4
      for (int u = 0; u < CH; ++u) {                     // 32 / CH keys at once
        const int from = u * (32 / CH) + sub;
        const int64_t at = __shfl_sync(0xffffffffu, k_at, from);
        uint4 k = make_uint4(0, 0, 0, 0);
        if ((lives >> from & 1) && c < p.d) k = *reinterpret_cast<const uint4 *>(reinterpret_cast<const char *>(p.k) + (at + c) * (E4M3 ? 1 : 2));
        const uint32_t kw[4] = {k.x, k.y, k.z, k.w};
        float2 kf[PER / 2];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (E4M3) {
            const uint2 h = e4m3x4_to_f16x4(kw[e]);
            kf[2 * e] = unpack2(h.x, __half(0.f)), kf[2 * e + 1] = unpack2(h.y, __half(0.f));
          } else {
            kf[e] = unpack2(kw[e], T(0.f));
          }
        }
#pragma unroll
        for (int i = 0; i < G; ++i) {
          float2 part = make_float2(0.f, 0.f);
#pragma unroll
          for (int e = 0; e < PER / 2; ++e) {
            const uint4 &w = q[i][e / 4];
            const float2 f = unpack2(e % 4 == 0 ? w.x : e % 4 == 1 ? w.y : e % 4 == 2 ? w.z : w.w, T(0.f));
            part.x = fmaf(f.x, kf[e].x, part.x), part.y = fmaf(f.y, kf[e].y, part.y);
          }
          float s = part.x + part.y;
#pragma unroll
          for (int m = 1; m < CH; m *= 2) s += __shfl_xor_sync(0xffffffffu, s, m);
          s = __shfl_sync(0xffffffffu, s, lane % (32 / CH) * CH);
          if (lane / (32 / CH) == u) x[i] = s;
        }
      }
#pragma unroll
      for (int i = 0; i < G; ++i) {
        const bool sees = first + lane >= lo[i] && first + lane < hi[i];
        const float s = sees ? x[i] * mul : -INFINITY;
        float to = s;
#pragma unroll
        for (int o = 16; o; o >>= 1) to = fmaxf(to, __shfl_xor_sync(0xffffffffu, to, o));
        to = fmaxf(to, top[i]);
        const float f = top[i] == -INFINITY ? 0.f : exp2_fast(top[i] - to);
        x[i] = sees ? exp2_fast(s - (to == -INFINITY ? 0.f : to)) : 0.f;
        top[i] = to, sum[i] = sum[i] * f + x[i];
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][e] *= f;
      }
#pragma unroll 8
      for (int u = 0; u < 32; ++u) {
        const int64_t va = __shfl_sync(0xffffffffu, v_at, u);
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if ((lives >> u & 1) && c4 < p.d) v = cache_values<T, E4M3>(p.v, va + c4);
        v.x = isfinite(v.x) ? v.x : 0.f, v.y = isfinite(v.y) ? v.y : 0.f, v.z = isfinite(v.z) ? v.z : 0.f, v.w = isfinite(v.w) ? v.w : 0.f;
#pragma unroll
        for (int i = 0; i < G; ++i) {
          const float xi = __shfl_sync(0xffffffffu, x[i], u);
          acc[i][0] = fmaf(xi, v.x, acc[i][0]), acc[i][1] = fmaf(xi, v.y, acc[i][1]);
          acc[i][2] = fmaf(xi, v.z, acc[i][2]), acc[i][3] = fmaf(xi, v.w, acc[i][3]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < G; ++i) {
#pragma unroll
      for (int o = 16; o; o >>= 1) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], o);
      if (!(todo >> (g + i) & 1) || c4 >= p.d) continue;
      const float f = sum[i] == 0.f ? 0.f : v_scale / sum[i];
      float y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        y[e] = acc[i][e] * f;
        if (mine[g + i] >> (4 + e) & 1) y[e] += INFINITY;
        if (mine[g + i] >> (8 + e) & 1) y[e] -= INFINITY;
        if (mine[g + i] >> e & 1) y[e] = NAN;
      }
      *reinterpret_cast<uint2 *>(out_row(r0 + warp * ROWS + g + i) + c4) = make_uint2(pack2(y[0], y[1], T(0.f)), pack2(y[2], y[3], T(0.f)));
    }
  }
}

// The rows of block (x, y) of the joining kernel: the y-th 32 of the item that is cut at the end of CTA x's range and, where that CTA
// found outputs that are not finite, of its whole items.  (A function of its own, held to 64 registers:
// that it is there costs two prompts of 250 tokens 0.6 - 0.9 of 18 - 21 us; in 80 or more registers 1.3 - 4, as a third kernel 1.5 - 4.)
template <typename T, bool E4M3, int DP>
__device__ __noinline__ void redo_items(const AttnParams &p) {
  const AttnMeta &meta = p.meta[blockIdx.x];
  const int4 item = meta.cut;
  const int r32 = blockIdx.y * 32;
  if (item.x >= 0 && item.z % 512 > r32)
    redo_rows<T, E4M3, DP>(p, meta.cut_b, load_seq(p, meta.cut_b), item.z / 512, item.y + r32, min(item.z % 512 - r32, 32));
  if (!meta.not_finite) return;
  AttnWalk<kTcgen05Rows, kTcgen05Unit, kTcgen05Extra> it(meta.range);
  while (it.next(p))              // (the block of the first CTA of an item that was cut has it)
    if (it.whole && it.n_rows > r32) redo_rows<T, E4M3, DP>(p, it.b, it.seq, it.head, it.r0 + r32, min(it.n_rows - r32, 32));
}

// The same for the pieces of the tcgen05 kernel, whose rows are neighbours in the workspace: a lane per row, a warp per 16 columns.
// A block whose CTA found outputs that are not finite goes through the rows of its items again.
template <typename T, bool E4M3, int DP>
__global__ void __launch_bounds__(DP * 2, 512 / DP) attention_combine_rows_kernel(const __grid_constant__ AttnParams p, int R) {
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
  redo_items<T, E4M3, DP>(p);
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
  if (plan.tcgen05) plan.flag_bytes = align256((size_t)plan.grid * (plan.rows / 32) * kRedoWords * sizeof(uint32_t));
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
  ZT_REQUIRE(std::isfinite(a->scale * 1.4426950408889634f) && a->scale > 0.f, ZT_INVALID_ARGUMENT, "zt_paged_attention: the scale must be positive and finite");
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
  p.causal = a->causal != 0, p.zero_tail = a->zero_tail != 0;
  p.window = a->window < 1 << 30 ? a->window : 1 << 30;      // (no context is longer)
  p.scale_log2 = a->scale * 1.4426950408889634f;
  p.few = plan.few, p.slices = plan.slices;
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
