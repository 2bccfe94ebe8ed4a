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
  int slices;                                   // streaming kernel: CTAs per sequence and kv head (0: all units are dealt out)
  int few;                                      // no sequence can have more than a few tiles of rows
  int zero_tail;                                // rows before the first sequence and behind the last are zeroed
  float *part_o;                                // [2 * grid][R][DP]
  float2 *part_ml;                              // [2 * grid][R]: maximum (log2 units), sum
  struct AttnMeta *meta;                        // [grid]
  int *status;
};

// Where a CTA's range begins: units [w0, w1) of all, w0 within the tile whose first unit (over its kv heads) is number `item0`.
// `per` units per CTA.  The host has checked that all units fit an int.
struct AttnRange {
  int w0, w1, per, item0;
  int b, tile;
};
// What a CTA leaves for the kernel that joins the cut items.
struct AttnMeta {
  int4 cut;           // the item cut at the end of its range: first new token of its sequence or -1, first row, head * 512 + rows, last CTA
  int cut_b;          // that item's sequence (tcgen05 kernel, as the rest)
  AttnRange range;
  int not_finite;     // some output of an item whose rows see different keys is not finite
};

struct AttnPlan {         // of one call, on the host
  bool tcgen05, few;
  int rows, dp, grid;     // rows per item, padded head, CTAs
  int slices;             // see AttnParams
  double most_units;
  size_t meta_bytes, ml_bytes, o_bytes, flag_bytes;
  size_t total() const { return meta_bytes + ml_bytes + o_bytes + flag_bytes; }
};

int attention_stream_launch(const AttnParams &p, const AttnPlan &plan, int dtype, int cache_dtype, cudaStream_t st);
int attention_tcgen05_launch(const AttnParams &p, const AttnPlan &plan, int dtype, int cache_dtype, cudaStream_t st);
int attention_stream_grid(int rows);

#ifdef __CUDACC__
constexpr int kTcgen05Rows = 256, kTcgen05Unit = 128, kTcgen05Extra = 3;   // rows of an item, keys of a unit, units that an item costs beside its own

constexpr float kLazyRescale = 8.f;   // log2 units that a running maximum may lag behind before sums are rescaled

// The reference of a row's exponents, to which all its probabilities and sums are relative (it cancels in the division).  In
// bf16 products it follows the maximum.  fp16 numbers end at 2^16 and, with 11 bits, at 2^-14, so there the reference lies 7
// below the maximum: the largest probability is 2^15 (with the lag), and one of 2^-21 of the largest still has its 11 bits.  Below,
// a probability is off by up to 2^-25 (half the spacing of subnormals), 2^-32 of a row's sum.  Without this, thousands of keys
// behind one that outweighs each by 2^25 were lost to the output, while the sum counts them.
template <typename M>
constexpr float kHeadroom = std::is_same_v<M, __half> ? 7.f : 0.f;
// (Rounded up, and the limit down, so that no probability passes 2^15 where scores are so large that fp32 has them 16 apart.)
template <typename M>
__device__ __forceinline__ float scaled_maximum(float best, float mul) {
  return std::is_same_v<M, __half> ? __fmul_ru(best, mul) : best * mul;
}
template <typename M>
__device__ __forceinline__ bool far_ahead(float top, float ref) {
  return top > (std::is_same_v<M, __half> ? __fadd_rd(ref, kLazyRescale + kHeadroom<M>) : ref + kLazyRescale);
}

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

// The sequence of tile t, from the tiles before each sequence: the last with prefix <= t.
__device__ __forceinline__ int first_tile_owner(const AttnParams &p, const int *prefix, int t) {
  int lo = 0, hi = p.batch;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (prefix[mid] <= t) lo = mid;
    else hi = mid;
  }
  return lo;
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

// Sum over the block, and the sum over the threads before this one.  `scratch`: 32 ints of shared memory, free on entry.
template <int NT>
__device__ __forceinline__ int block_scan(int v, int *scratch, int &total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) scratch[warp] = x;
  __syncthreads();
  int w = lane < NT / 32 ? scratch[lane] : 0, before = 0;      // every warp adds the warps' sums for itself
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += y;
  }
  total = __shfl_sync(0xffffffffu, w, NT / 32 - 1);
  before = __shfl_sync(0xffffffffu, w, warp > 0 ? warp - 1 : 0);
  return (warp ? before : 0) + x - v;
}

struct AttnScratch {
  int scan[2][32], found[3];
};

// Whole-block call.  `prefix`: batch + 1 ints of shared memory.  `few`: no sequence has more than a handful of tiles, and a thread
// goes through those of its sequences; else the tiles of all sequences are shared out evenly first.
template <int R, int UK, int EXTRA, int NT>
__device__ AttnRange attention_range(const AttnParams &p, int *prefix, AttnScratch &scratch) {
  const int chunk = (p.batch + NT - 1) / NT;
  const int b0 = min((int)threadIdx.x * chunk, p.batch), b1 = min(b0 + chunk, p.batch);
  int mine = 0, total, t0 = 0, t1 = 0, at;
  if (p.few) {
    for (int b = b0; b < b1; ++b) {
      if (blockIdx.x == 0 && !lengths_fit(p, b)) tc::report_timeout(p.status, kStatusBadIndex);
      const SeqInfo s = load_seq(p, b);
      const int n = row_tiles<R>(p, s);
      for (int t = 0; t < n; ++t) mine += (tile_units<R, UK>(p, s, t).count + EXTRA) * p.hkv;
    }
  } else {
    // tiles of the sequences before each sequence
    for (int b = b0; b < b1; ++b) {
      if (blockIdx.x == 0 && !lengths_fit(p, b)) tc::report_timeout(p.status, kStatusBadIndex);
      mine += row_tiles<R>(p, load_seq(p, b));
    }
    int tiles;
    at = block_scan<NT>(mine, scratch.scan[0], tiles);
    for (int b = b0; b < b1; ++b) {
      prefix[b] = at;
      at += row_tiles<R>(p, load_seq(p, b));
    }
    if (threadIdx.x == 0) prefix[p.batch] = tiles;
    __syncthreads();
    // units of each thread's tiles
    const int tchunk = (tiles + NT - 1) / NT;
    t0 = min((int)threadIdx.x * tchunk, tiles), t1 = min(t0 + tchunk, tiles);
    mine = 0;
    if (t0 < t1) {
      int b = first_tile_owner(p, prefix, t0);
      SeqInfo s = load_seq(p, b);
      for (int t = t0; t < t1; ++t) {
        while (t >= prefix[b + 1]) s = load_seq(p, ++b);
        mine += (tile_units<R, UK>(p, s, t - prefix[b]).count + EXTRA) * p.hkv;
      }
    }
  }
  at = block_scan<NT>(mine, scratch.scan[1], total);
  AttnRange r;
  r.per = max((total + (int)gridDim.x - 1) / (int)gridDim.x, 1);
  r.w0 = (int)min((long long)r.per * blockIdx.x, (long long)total), r.w1 = min(r.w0 + r.per, total);
  r.b = 0, r.tile = 0, r.item0 = 0;
  if (threadIdx.x == 0) scratch.found[0] = scratch.found[1] = scratch.found[2] = 0;
  __syncthreads();
  if (r.w0 < r.w1) {
    // (lengths that contradict one another can add up to more than an int, and then no thread may find w0: the walk checks what it
    // goes by, and `cut` where it ends)
    if (r.w0 >= at && r.w0 < at + mine) {      // one thread
      int b = p.few ? b0 : first_tile_owner(p, prefix, t0);
      SeqInfo s = load_seq(p, b);
      for (int t = p.few ? 0 : t0 - prefix[b];; ++t) {
        while (t >= row_tiles<R>(p, s) && b + 1 < p.batch) s = load_seq(p, ++b), t = 0;
        const int u = (tile_units<R, UK>(p, s, t).count + EXTRA) * p.hkv;
        if (r.w0 < at + u || t >= row_tiles<R>(p, s)) {
          scratch.found[0] = at, scratch.found[1] = b, scratch.found[2] = t;
          break;
        }
        at += u;
      }
    }
    __syncthreads();
    r.item0 = scratch.found[0], r.b = scratch.found[1], r.tile = scratch.found[2];
  }
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
      const int w = w_end_;
      if (w >= w1_) return false;
      if (!started_) seq = load_seq(p, b);
      else if (w == h1_ && head == p.hkv - 1) ++tile, item0_ = h1_;
      started_ = true;
      while (tile >= row_tiles<R>(p, seq)) {             // (sequences without new tokens have no tiles)
        if (++b >= p.batch) return false;
        seq = load_seq(p, b), tile = 0;
      }
      const TileUnits u = tile_units<R, UK>(p, seq, tile);
      const int cost = u.count + EXTRA;
      head = (w - item0_) / cost;
      if ((unsigned)head >= (unsigned)p.hkv) return false;
      const int h0 = item0_ + head * cost;
      h1_ = h0 + cost;
      w_end_ = min(h1_, w1_);
      const int from = max(w - h0 - EXTRA, 0), to = w_end_ - h0 - EXTRA;
      if (to <= from) continue;                          // the range ends before the item's first unit
      n_units = to - from, unit0 = u.first + from;
      r0 = tile * R, n_rows = min(seq.n * p.group - r0, R);
      first_piece = from == 0, whole = first_piece && w_end_ == h1_;
      return true;
    }
  }
  // For the kernel that joins the pieces of this item.
  __device__ int4 cut() const { return make_int4(seq.q0, r0, head * 512 + n_rows, min((h1_ - 1) / per_, (int)gridDim.x - 1)); }
  __device__ int token(const AttnParams &p, int row) const { return (r0 + row) / p.group; }
  __device__ int q_head(const AttnParams &p, int row) const { return head * p.group + (r0 + row) % p.group; }

 private:
  int w_end_, w1_, per_, item0_, h1_;
  bool started_;
};

// Entry of a sequence's row of block_table that holds the page of a key.
__device__ __forceinline__ int page_of(const AttnParams &p, int key) { return p.page_shift >= 0 ? key >> p.page_shift : key / p.page; }

// Rows of `out` before the first sequence and behind the last one, by all threads of the grid.
template <typename T>
__device__ __forceinline__ void zero_tail_rows(const AttnParams &p, int threads) {
  if (!p.zero_tail) return;
  const int end = min(max(p.cu[p.batch], 0), p.tokens), begin = min(max(p.cu[0], 0), end);
  const int vecs = p.d / 8, per = p.hq * vecs;      // (rows are whole 16-byte vectors)
  const int64_t n = (int64_t)(begin + p.tokens - end) * per;
  for (int64_t i = (int64_t)blockIdx.x * threads + threadIdx.x; i < n; i += (int64_t)gridDim.x * threads) {
    const int64_t row = i / per, t = row < begin ? row : row - begin + end;
    const int c = (int)(i % per);
    *reinterpret_cast<uint4 *>(reinterpret_cast<T *>(p.out) + t * p.o_st + (c / vecs) * p.o_sh + c % vecs * 8) = make_uint4(0, 0, 0, 0);
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
// What scores are multiplied by: a cache scale of zero becomes the smallest number there is, so that masked scores stay minus
// infinity (others come to 2^-21 at most); NaN stays NaN.
__device__ __forceinline__ float score_factor(float mul) { return mul == 0.f ? __int_as_float(1) : mul; }
// Power of two that brings a row whose largest element is `top` to a maximum in [1, 2); none for rows of zeros or not finite.
__device__ __forceinline__ int row_exponent(float top) {
  return top > 0.f && top < __int_as_float(0x7f800000) ? min(max(ilogbf(top), -126), 126) : 0;
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, int bytes) {   // the rest of the 16 is zero
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void st_shared16(uint32_t dst, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(dst), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ uint4 ld_shared16(uint32_t src) {
  uint4 x;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(src) : "memory");
  return x;
}

// Values that are not finite.  A probability of zero times such a value would reach rows that do not see its key, so where the rows
// of a tile see different keys those values are taken out of the product and added to the rows that do see them.
// Mask over the bits of the elements of `w` that are not finite: two of M, or four e4m3.
__device__ __forceinline__ uint32_t not_finite_mask(uint32_t w, __nv_bfloat16) {
  return (((w & 0x7f807f80u) + 0x00800080u) >> 15 & 0x00010001u) * 0xffffu;
}
__device__ __forceinline__ uint32_t not_finite_mask(uint32_t w, __half) {
  return (((w & 0x7c007c00u) + 0x04000400u) >> 15 & 0x00010001u) * 0xffffu;
}
__device__ __forceinline__ uint32_t not_finite_mask_e4m3(uint32_t w) {
  return (((w & 0x7f7f7f7fu) + 0x01010101u) >> 7 & 0x01010101u) * 0xffu;
}

// Four e4m3 values as halves, in order; exact.
__device__ __forceinline__ uint2 e4m3x4_to_f16x4(uint32_t four) {
  uint2 r;
  asm("{.reg .b16 l, h; mov.b32 {l, h}, %2; cvt.rn.f16x2.e4m3x2 %0, l; cvt.rn.f16x2.e4m3x2 %1, h;}" : "=r"(r.x), "=r"(r.y) : "r"(four));
  return r;
}
#endif

}  // namespace zt
