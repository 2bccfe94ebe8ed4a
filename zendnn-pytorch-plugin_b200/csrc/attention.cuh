// What the kernels of the paged attention share: parameters, the rows and keys of a tile of work, and the division of a batch
// of ragged sequences among the CTAs of a persistent grid.
//
// Rows.  The q heads of a group share a kv head, so the rows of the products are (token, head of the group) pairs of one
// sequence and kv head, token-major: row r is head r % G of new token r / G.  An item is (sequence, tile of R consecutive rows,
// kv head); its keys are those that some row of it sees, cut into units of a fixed number of keys.
//
// Work.  The units of all items, in the order (sequence, tile, kv head, unit), are dealt to the CTAs in equal contiguous ranges,
// found by every CTA for itself from the lengths in device memory: nothing about the lengths is known on the host, and a
// captured launch follows them.  An item counts for a few units more than it has, for its query rows, first and last loads and
// output (`EXTRA`, per kernel; they come before its first unit).  An item that lies in one range is written directly; one that is cut leaves unnormalised sums
// with their maxima in the workspace, at most one at either end of a CTA's range, and attention_combine_kernel joins them in CTA
// order.
#pragma once

#include <cuda_fp16.h>

#include <type_traits>

#include "tc05.cuh"

namespace zt {

struct AttnParams {
  const void *q;
  void *out;
  const void *k, *v;
  int64_t q_st, q_sh, o_st, o_sh;               // strides in elements: token, head
  int64_t k_sp, k_ss, k_sh, v_sp, v_ss, v_sh;   // page, slot, head
  const int32_t *cu, *lens, *table;
  int64_t table_stride;
  const float *k_scale, *v_scale;               // per kv head, or null
  int batch, tokens, hq, hkv, group, d;
  int page, page_shift, max_blocks, num_pages;  // page_shift: log2 of the page size, or -1
  int causal, window;                           // window 0: none
  float scale_log2;                             // softmax scale times log2(e)
  int zero_tail;                                // rows behind the last sequence are zeroed
  float *part_o;                                // [2 * grid][R][DP]
  float2 *part_ml;                              // [2 * grid][R]: maximum (log2 units), sum
  int4 *meta;                                   // [grid]: the item cut at the end of a CTA's range (b, tile, head) and the last CTA of it, or -1
  int *status;
};

struct AttnPlan {         // of one call, on the host
  bool tcgen05;
  int rows, dp, grid;     // rows per item, padded head, CTAs
  size_t meta_bytes, ml_bytes, o_bytes;
  size_t total() const { return meta_bytes + ml_bytes + o_bytes; }
};

int attention_stream_launch(const AttnParams &p, const AttnPlan &plan, int dtype, int cache_dtype, cudaStream_t st);
int attention_tcgen05_launch(const AttnParams &p, const AttnPlan &plan, int dtype, int cache_dtype, cudaStream_t st);
int attention_stream_grid();

#ifdef __CUDACC__
constexpr float kLazyRescale = 8.f;   // log2 units that a running maximum may lag behind before sums are rescaled

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// One sequence.  Lengths that do not fit are cut to what the tensors hold and reported by whoever reads the table.
struct SeqInfo {
  int q0, n, len;   // first row of the new tokens, new tokens, keys
};
__device__ __forceinline__ SeqInfo load_seq(const AttnParams &p, int b) {
  int q0 = p.cu[b], q1 = p.cu[b + 1], len = p.lens[b];
  q0 = min(max(q0, 0), p.tokens), q1 = min(max(q1, q0), p.tokens);
  const int64_t room = (int64_t)p.max_blocks * p.page;
  if (len > room) len = (int)room;
  return {q0, q1 - q0, max(len, 0)};
}
__device__ __forceinline__ bool lengths_fit(const AttnParams &p, int b) {
  const int q0 = p.cu[b], q1 = p.cu[b + 1], len = p.lens[b];
  return q0 >= 0 && q1 >= q0 && q1 <= p.tokens && len >= 0 && len <= (int64_t)p.max_blocks * p.page;
}

// Keys [lo, hi) that new token `i` of a sequence sees.
__device__ __forceinline__ int key_hi(const AttnParams &p, const SeqInfo &s, int i) {
  return p.causal ? max(min(s.len, s.len - s.n + i + 1), 0) : s.len;
}
__device__ __forceinline__ int key_lo(const AttnParams &p, const SeqInfo &s, int i) {
  return p.window > 0 ? max(s.len - s.n + i - p.window + 1, 0) : 0;
}

template <int R>
__device__ __forceinline__ int row_tiles(const AttnParams &p, const SeqInfo &s) {
  return (int)(((unsigned)s.n * (unsigned)p.group + R - 1) / R);       // (tokens * q_heads stays below 2^30)
}

// Units of UK keys of a tile: [first, first + count).  A tile that sees nothing still has one, in which its zeros are written.
struct TileUnits {
  int first, count;
};
template <int R, int UK>
__device__ __forceinline__ TileUnits tile_units(const AttnParams &p, const SeqInfo &s, int tile) {
  const int rows = s.n * p.group, r0 = tile * R, r1 = min(r0 + R, rows) - 1;
  const int lo = key_lo(p, s, r0 / p.group), hi = key_hi(p, s, r1 / p.group);
  if (hi <= lo) return {0, 1};
  return {lo / UK, (hi + UK - 1) / UK - lo / UK};
}

// Sum over the block, and the sum over the threads before this one.  `scratch`: 33 long longs of shared memory, free on entry.
template <int NT>
__device__ __forceinline__ long long block_scan(long long v, long long *scratch, long long &total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) scratch[warp] = x;
  __syncthreads();
  if (warp == 0) {
    long long w = lane < NT / 32 ? scratch[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += y;
    }
    scratch[lane] = w;
  }
  __syncthreads();
  total = scratch[NT / 32 - 1];
  const long long before = warp ? scratch[warp - 1] : 0;
  __syncthreads();
  return before + x - v;
}

// Where a CTA's range begins: units [w0, w1) of all, the first of them `offset` units into sequence b, tile `tile` (over its kv
// heads).  `per` units per CTA.
struct AttnRange {
  long long w0, w1, per, item0;   // item0: number of the first unit of (b, tile)
  int b, tile;
};

// Whole-block call.  `prefix`: batch + 1 ints of shared memory; `scratch`: 40 long longs.
template <int R, int UK, int EXTRA, int NT>
__device__ AttnRange attention_range(const AttnParams &p, int min_units, int *prefix, long long *scratch) {
  // tiles of the sequences before each sequence
  const int chunk = (p.batch + NT - 1) / NT;
  const int b0 = min((int)threadIdx.x * chunk, p.batch), b1 = min(b0 + chunk, p.batch);
  long long mine = 0;
  for (int b = b0; b < b1; ++b) {
    if (blockIdx.x == 0 && !lengths_fit(p, b)) tc::report_timeout(p.status, kStatusBadIndex);
    mine += row_tiles<R>(p, load_seq(p, b));
  }
  long long tiles;
  long long at = block_scan<NT>(mine, scratch, tiles);
  for (int b = b0; b < b1; ++b) {
    prefix[b] = (int)at;
    at += row_tiles<R>(p, load_seq(p, b));
  }
  if (threadIdx.x == 0) prefix[p.batch] = (int)tiles;
  __syncthreads();
  // units of the tiles before each thread's tiles
  const int tchunk = (int)((tiles + NT - 1) / NT);
  const int t0 = min((long long)threadIdx.x * tchunk, tiles), t1 = min((long long)t0 + tchunk, tiles);
  int b = 0;
  mine = 0;
  if (t0 < t1) {
    int lo = 0, hi = p.batch;           // the sequence of tile t0: the last with prefix <= t0
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (prefix[mid] <= t0) lo = mid;
      else hi = mid;
    }
    b = lo;
    int bb = b;
    SeqInfo s = load_seq(p, bb);
    for (int t = t0; t < t1; ++t) {
      while (t >= prefix[bb + 1]) s = load_seq(p, ++bb);
      mine += (long long)(tile_units<R, UK>(p, s, t - prefix[bb]).count + EXTRA) * p.hkv;
    }
  }
  long long total;
  at = block_scan<NT>(mine, scratch, total);
  AttnRange r;
  r.per = (total + gridDim.x - 1) / gridDim.x;
  if (r.per < min_units) r.per = min_units;
  r.w0 = min(r.per * blockIdx.x, total), r.w1 = min(r.w0 + r.per, total);
  r.b = 0, r.tile = 0, r.item0 = 0;
  if (r.w0 < r.w1) {
    if (r.w0 >= at && r.w0 < at + mine) {      // exactly one thread
      SeqInfo s = load_seq(p, b);
      for (int t = t0; t < t1; ++t) {
        while (t >= prefix[b + 1]) s = load_seq(p, ++b);
        const long long u = (long long)(tile_units<R, UK>(p, s, t - prefix[b]).count + EXTRA) * p.hkv;
        if (r.w0 < at + u) {
          scratch[36] = at, scratch[37] = b, scratch[38] = t - prefix[b];
          break;
        }
        at += u;
      }
    }
    __syncthreads();
    r.item0 = scratch[36], r.b = (int)scratch[37], r.tile = (int)scratch[38];
  }
  __syncthreads();
  return r;
}

// The pieces of items in a CTA's range, in order.
template <int R, int UK, int EXTRA>
struct AttnWalk {
  SeqInfo seq;
  int b, tile, head;
  int unit0, n_units;          // the piece's units of the item's keys
  int n_rows, r0;              // rows of the item, first of them
  bool first_piece, whole;     // the item's first unit is in this piece; all of them are

  __device__ explicit AttnWalk(const AttnRange &r)
      : seq{0, 0, 0}, b(r.b), tile(r.tile), head(-1), unit0(0), n_units(0), n_rows(0), r0(0), first_piece(false), whole(false),
        w_end_(r.w0), w1_(r.w1), per_(r.per), item0_(r.item0), h1_(-1), started_(false) {}
  __device__ bool next(const AttnParams &p) {
    for (;;) {
      const long long w = w_end_;
      if (w >= w1_) return false;
      if (!started_) seq = load_seq(p, b);
      else if (w == h1_ && head == p.hkv - 1) ++tile, item0_ = h1_;
      started_ = true;
      while (tile >= row_tiles<R>(p, seq)) seq = load_seq(p, ++b), tile = 0;   // (sequences without new tokens have no tiles)
      const TileUnits u = tile_units<R, UK>(p, seq, tile);
      const int cost = u.count + EXTRA;
      head = (int)(w - item0_) / cost;                   // units of a tile over its kv heads fit 32 bits
      const long long h0 = item0_ + (long long)head * cost;
      h1_ = h0 + cost;
      w_end_ = h1_ < w1_ ? h1_ : w1_;
      const int from = max((int)(w - h0) - EXTRA, 0), to = (int)(w_end_ - h0) - EXTRA;
      if (to <= from) continue;                          // the range ends before the item's first unit
      n_units = to - from, unit0 = u.first + from;
      r0 = tile * R, n_rows = min(seq.n * p.group - r0, R);
      first_piece = from == 0, whole = first_piece && w_end_ == h1_;
      return true;
    }
  }
  __device__ int last_cta() const { return (int)((h1_ - 1) / per_); }   // where the item ends
  __device__ int token(const AttnParams &p, int row) const { return (r0 + row) / p.group; }
  __device__ int q_head(const AttnParams &p, int row) const { return head * p.group + (r0 + row) % p.group; }

 private:
  long long w_end_, w1_, per_, item0_, h1_;
  bool started_;
};

// Row of the cache that holds a key: page id, slot in it.  An id outside the cache reads as no row and is reported.
__device__ __forceinline__ int page_of(const AttnParams &p, int key) { return p.page_shift >= 0 ? key >> p.page_shift : key / p.page; }

// Rows of `out` behind the last sequence, by all threads of the grid.
template <typename T>
__device__ __forceinline__ void zero_tail_rows(const AttnParams &p, int threads) {
  if (!p.zero_tail) return;
  const int end = min(max(p.cu[p.batch], 0), p.tokens);
  const int64_t per = (int64_t)p.hq * p.d, n = (p.tokens - end) * per;
  for (int64_t i = (int64_t)blockIdx.x * threads + threadIdx.x; i < n; i += (int64_t)gridDim.x * threads) {
    const int64_t t = end + i / per, c = i % per;
    reinterpret_cast<T *>(p.out)[t * p.o_st + (c / p.d) * p.o_sh + c % p.d] = T(0.f);
  }
}

__device__ __forceinline__ uint32_t pack2(float x, float y, __nv_bfloat16) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
  return *reinterpret_cast<const uint32_t *>(&v);
}
__device__ __forceinline__ uint32_t pack2(float x, float y, __half) {
  const __half2 v = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t *>(&v);
}
__device__ __forceinline__ float2 unpack2(uint32_t w, __nv_bfloat16) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ float2 unpack2(uint32_t w, __half) { return __half22float2(*reinterpret_cast<const __half2 *>(&w)); }
// Power of two that brings a row whose largest element is `top` to a maximum in [1, 2); none for rows of zeros or not finite.
__device__ __forceinline__ int row_exponent(float top) {
  return top > 0.f && top < __int_as_float(0x7f800000) ? min(max(ilogbf(top), -126), 126) : 0;
}
// Two e4m3 values (the low 16 bits) as halves; exact.
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t two) {
  uint32_t r;
  asm("{.reg .b16 h; cvt.u16.u32 h, %1; cvt.rn.f16x2.e4m3x2 %0, h;}" : "=r"(r) : "r"(two));
  return r;
}
#endif

}  // namespace zt
