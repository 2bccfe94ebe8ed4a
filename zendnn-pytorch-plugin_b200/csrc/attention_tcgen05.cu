// Paged attention on the tensor cores of sm_100a, for chunks and prompts.
//
// An item is 256 (token, head of the group) rows of one kv head, as two tiles of 128 that share every K and V tile of 128 keys.
// Scores S = Q K^T of a tile go to tensor memory (128 columns), one thread per row turns them into probabilities, 16-bit pairs in
// 64 of the same columns, and O += P V accumulates in tensor memory with P as the tensor-memory operand.  Of the two tiles
// one is in its exponentials while the tensor core works for the other.
//
//   warps 0-3, 4-7   a row of tile 0 / 1 each thread: query rows to shared memory, running maximum and sum, probabilities, output
//   warps 8-11       K and V tiles into a ring, 32 keys each: by TMA, in boxes of 8, 16 or 32 slots of a page, where a page is whole
//                    boxes and all 32 keys are visible; else row by row, 16 bytes per asynchronous copy (any
//                    page size).  Slots past the visible keys become zeros that way, so stale contents of a page never meet the
//                    arithmetic.  e4m3 tiles come row by row into a ring of their own and from there as halves (exact)
//   warp 12          issues the MMAs
//   warp 13          walks the CTA's range and hands its pieces to the others
//
// Where the rows of an item see different keys, a probability of zero meets the values of the others, and one that is not finite
// spoils rows that do not see it.  The rows look at their output, which costs next to nothing, and note a CTA that found some not
// finite; the kernel after this one, which joins the cut items, goes through those rows again (taking such values out of the
// products here cost 10 - 40 %, by the size of the code alone).
//
// The reference of the exponents follows the row maximum only when that has run 8 (log2) ahead of it, so the rows of O are
// rescaled a few times at the start and hardly ever after; the thread that finds it does it itself.  Probabilities are rounded
// to the products' type (2^-32 of the row's sum is lost of those that are subnormals of fp16); their sum is of the unrounded fp32
// values.  e4m3: fp16 products, query rows brought below 2 by a power of
// two as in the streaming kernel.
#include <algorithm>

#include "attention.cuh"

namespace zt {

namespace {

constexpr int kTile = kTcgen05Unit;         // rows of a tile, keys of a unit
constexpr int kRows = kTcgen05Rows;
constexpr int kThreads = 512;              // four warpgroups: tile 0, tile 1, copies, MMA and walk (and two idle warps)
constexpr int kExtra = kTcgen05Extra;
constexpr int kHalf = kTile * 128;         // bytes of 64 columns of a tile: 128 rows of 128 bytes, swizzled
constexpr int kBoxSlots = 32;              // slots of a page per TMA box, at most

template <int DP, bool E4M3>
struct Smem {
  static constexpr int kTileBytes = kTile * DP * 2;
  static constexpr int kStages = E4M3 ? (DP == 128 ? 3 : 6) : DP == 128 ? 5 : 8;
  static constexpr int kLag = E4M3 ? 3 : 2;                     // stages whose row copies are in flight behind the newest
  static constexpr int kRing = 2 * kTileBytes;                  // after the two query tiles
  static constexpr int kRaw = kRing + kStages * kTileBytes;     // e4m3: tiles as they come, kLag + 1 of them
  static constexpr int kRawBytes = kTile * DP;
  static constexpr int kBytes = kRaw + (E4M3 ? (kLag + 1) * kRawBytes : 0);
};

// Registers per thread after the split; the sum over the four warpgroups is that of the launch, 4 * 128.
constexpr int kRegsRows = 152, kRegsCopy = 104, kRegsMma = 104;
static_assert(2 * kRegsRows + kRegsCopy + kRegsMma <= 4 * 128, "register split above the launch's registers");

__device__ __forceinline__ void fence_async_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Byte offset of 16-byte chunk `c` of row `row` in a tile.
__device__ __forceinline__ uint32_t tile_at(int row, int c) { return (c >> 3) * kHalf + row * 128 + (((c & 7) ^ (row & 7)) << 4); }

__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(*reinterpret_cast<unsigned long long *>(&d))
      : "l"(*reinterpret_cast<const unsigned long long *>(&a)), "l"(*reinterpret_cast<const unsigned long long *>(&b)),
        "l"(*reinterpret_cast<const unsigned long long *>(&c)));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(*reinterpret_cast<unsigned long long *>(&d))
      : "l"(*reinterpret_cast<const unsigned long long *>(&a)), "l"(*reinterpret_cast<const unsigned long long *>(&b)));
  return d;
}

// One box of a page: columns c0.., slots, head, page.
__device__ __forceinline__ void tma_load_4d_if(bool lane_does, uint32_t dst, const CUtensorMap *m, uint32_t bar, int c0, int slot, int head,
                                               int page) {
  asm volatile(
      "{.reg .pred p; setp.ne.b32 p, %0, 0;\n\t"
      "@p cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%1], [%2, {%4, %5, %6, %7}], [%3];}" ::"r"(
          (uint32_t)lane_does),
      "r"(dst), "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(c0), "r"(slot), "r"(head), "r"(page)
      : "memory");
}

__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

struct Barriers {
  uint64_t kv_full[8], kv_free[8];
  uint64_t q_full[2], s_full[2], p_half[2], p_full[2], o_full[2];
  uint64_t piece_full[4], piece_free[4];
  uint64_t drain;                // after a wait that gave up: the products that were issued
  uint32_t not_finite;           // some output that may be another row's doing
  uint32_t tmem;
};

// A piece of an item, as the walk hands it out; b < 0: there are no more.
struct Piece {
  SeqInfo seq;
  int4 cut;          // what the joining kernel is told of the item
  int b, head, unit0, n_units, r0, n_rows, first_piece, whole;
  int count[2];      // units that each tile works on, from the piece's first

  __device__ int token(const AttnParams &p, int row) const { return (r0 + row) / p.group; }
  __device__ int q_head(const AttnParams &p, int row) const { return head * p.group + (r0 + row) % p.group; }
};
constexpr int kPieces = 4;             // handed out ahead
constexpr int kPieceReaders = 13;      // warps

using Walk = AttnWalk<kRows, kTile, kExtra>;

__device__ __forceinline__ int tile_count(const AttnParams &p, const Walk &it, int i) {
  const int rows = it.n_rows - i * kTile;
  if (rows <= 0) return 0;
  const int hi = key_hi(p, it.seq, it.token(p, i * kTile + min(rows, kTile) - 1));
  return min(max((hi + kTile - 1) / kTile - it.unit0, 0), it.n_units);
}

template <typename T, bool E4M3, int DP>
__global__ void __launch_bounds__(kThreads, 1) attention_tcgen05_kernel(const __grid_constant__ AttnParams p, const __grid_constant__ CUtensorMap k_map,
                                                                        const __grid_constant__ CUtensorMap v_map, int box) {
  using M = std::conditional_t<E4M3, __half, T>;
  using L = Smem<DP, E4M3>;
  constexpr int S = L::kStages, CHUNKS = DP / 8;
  extern __shared__ unsigned char smem_raw[];
  __shared__ Barriers bars;
  __shared__ Piece pieces[kPieces];
  __shared__ AttnScratch s_scan;
  unsigned char *smem = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const uint32_t base = smem_u32(smem);
  const int warp = tc::uniform_warp(), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) tc::mbar_init(&bars.kv_full[i], 4), tc::mbar_init(&bars.kv_free[i], 1);
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&bars.q_full[i], 4), tc::mbar_init(&bars.p_half[i], 4), tc::mbar_init(&bars.p_full[i], 4);
      tc::mbar_init(&bars.s_full[i], 1), tc::mbar_init(&bars.o_full[i], 1);
    }
    for (int i = 0; i < kPieces; ++i) tc::mbar_init(&bars.piece_full[i], 1), tc::mbar_init(&bars.piece_free[i], kPieceReaders);
    tc::mbar_init(&bars.drain, 1);
    bars.not_finite = 0;
    tc::mbar_fence_init();
  }
  if (warp == 12) tc::tmem_alloc(&bars.tmem, 512);
  grid_launch_dependents();
  grid_dependency_wait();
  const AttnRange range = attention_range<kRows, kTile, kExtra, kThreads>(p, reinterpret_cast<int *>(smem), s_scan);
  zero_tail_rows<T>(p, kThreads);
  if (threadIdx.x == 0) p.meta[blockIdx.x].cut.x = -1, p.meta[blockIdx.x].range = range;
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = bars.tmem;
  bool ok = true;
  uint32_t n_piece = 0;        // pieces taken
  auto take = [&]() -> const Piece * {     // the next piece, or null (at the end, and with ok unset after a wait that gave up)
    const uint32_t i = n_piece % kPieces;
    if (!(ok = tc::warp_wait(smem_u32(&bars.piece_full[i]), (n_piece / kPieces) & 1))) return nullptr;
    ++n_piece;
    return pieces[i].b >= 0 ? &pieces[i] : nullptr;
  };
  auto give_back = [&]() {                 // of the last piece taken
    __syncwarp();
    tc::arrive_if(lane == 0, smem_u32(&bars.piece_free[(n_piece - 1) % kPieces]));
  };

  if (warp < 8) {
    // ---- a tile's rows -----------------------------------------------------------------------------------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsRows));
    const int i = warp >> 2, row = threadIdx.x & (kTile - 1);     // tile, row of it (= lane of tensor memory)
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_tmem = tmem + i * kTile + lanes, p_tmem = s_tmem + kTile / 2, o_tmem = tmem + 2 * kTile + i * kTile + lanes;
    const uint32_t s_full = smem_u32(&bars.s_full[i]), o_full = smem_u32(&bars.o_full[i]);
    const uint32_t q_full = smem_u32(&bars.q_full[i]), p_full = smem_u32(&bars.p_full[i]),
                   p_half = smem_u32(&bars.p_half[i]);
    uint32_t n_s = 0, n_o = 0;     // phases of s_full and o_full so far

    // Rows of queries come in 16 lanes (8 for heads of up to 64) to a row, so that a warp's access covers whole lines.
    constexpr int RP = 32 / CHUNKS, PASSES = 32 / RP;    // rows per pass of the warp
    const int c = lane % CHUNKS, sub = lane / CHUNKS;
    const uint32_t tile = base + i * L::kTileBytes;
    const int row0 = (warp & 3) * 32;                             // first row of the warp
    auto row_of = [&](int64_t mine, int pass) -> int64_t {        // lane's value of the row that this lane works on
      return __shfl_sync(0xffffffffu, mine, pass * RP + sub);
    };

    auto load_query = [&](const Piece &it) -> float {   // the piece's rows to shared memory; returns the factor of this row's scores
      const int r = i * kTile + row;
      const int64_t at = r < it.n_rows ? (it.seq.q0 + it.token(p, r)) * p.q_st + it.q_head(p, r) * p.q_sh : -1;
      const char *src = reinterpret_cast<const char *>(p.q);
      float mul = p.scale_log2;
      if constexpr (!E4M3) {
#pragma unroll
        for (int q = 0; q < PASSES; ++q) {
          const int64_t o = row_of(at, q);
          const bool in = o >= 0 && c * 8 < p.d;
          cp_async16(tile + tile_at(row0 + q * RP + sub, c), in ? src + (o + c * 8) * 2 : src, in ? 16 : 0);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
      } else {
        const float k_scale = p.k_scale[it.head];
        uint4 x[PASSES];
        int my_ex = 0;
#pragma unroll
        for (int q = 0; q < PASSES; ++q) {
          const int64_t o = row_of(at, q);
          x[q] = o >= 0 && c * 8 < p.d ? *reinterpret_cast<const uint4 *>(src + (o + c * 8) * 2) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int q = 0; q < PASSES; ++q) {
          const uint32_t w[4] = {x[q].x, x[q].y, x[q].z, x[q].w};
          float top = 0.f;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 f = unpack2(w[e], T(0.f));
            top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
          }
#pragma unroll
          for (int m = 1; m < CHUNKS; m *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, m));
          const int ex = row_exponent(top);
          const float down = copysignf(ldexpf(1.f, -ex), k_scale);
          uint32_t h[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 f = unpack2(w[e], T(0.f));
            h[e] = pack2(f.x * down, f.y * down, M(0.f));
          }
          st_shared16(tile + tile_at(row0 + q * RP + sub, c), h[0], h[1], h[2], h[3]);
          const int mine = __shfl_sync(0xffffffffu, ex, lane % RP * CHUNKS);
          if (lane / RP == q) my_ex = mine;
        }
        mul *= fabsf(k_scale) * ldexpf(1.f, my_ex);
      }
      return score_factor(mul);
    };
    auto query_ready = [&]() {
      if constexpr (!E4M3) asm volatile("cp.async.wait_group 0;" ::: "memory");
      fence_async_proxy();
      __syncwarp();
      tc::arrive_if(lane == 0, q_full);
    };

    const Piece *it = take();
    float mul = 0.f;
    if (it && it->count[i] > 0) {
      mul = load_query(*it);
      query_ready();
    }
    while (it) {
      const int rows = min(max(it->n_rows - i * kTile, 0), kTile), count = it->count[i], unit0 = it->unit0;
      const bool live = row < rows;
      int lo = 0, hi = 0, all_lo = 0, all_hi = 0;      // keys that this row sees; that every row of the tile sees
      if (rows > 0) {
        const int tok = it->token(p, i * kTile + (live ? row : 0));
        lo = key_lo(p, it->seq, tok), hi = live ? key_hi(p, it->seq, tok) : 0;
        if (E4M3 && hi <= lo) mul = 1.f;               // (minus infinity times a scale of NaN, in a row that sees no key)
        all_lo = key_lo(p, it->seq, it->token(p, i * kTile + rows - 1)), all_hi = key_hi(p, it->seq, it->token(p, i * kTile));
      }
      float ref = -INFINITY, sum = 0.f;
      for (int j = 0; j < count; ++j) {
        const int key0 = (unit0 + j) * kTile;
        if (!(ok = tc::warp_wait(s_full, n_s & 1))) break;
        ++n_s;
        tc::fence_after_sync();
        // Two passes over the row in pieces of 32 scores: its maximum, then the exponentials.  The last 64 scores stay in registers
        // in between and go first; their columns take the probabilities of all, so the others can be read again.
        const bool masked = key0 < all_lo || key0 + kTile > all_hi;
        auto mask = [&](uint32_t (&x)[32], int c) {
          const int f = lo - key0 - 32 * c, t = hi - key0 - 32 * c;
          const uint32_t seen = (t <= 0 ? 0u : t >= 32 ? ~0u : (1u << t) - 1) & (f <= 0 ? ~0u : f >= 32 ? 0u : ~0u << f);
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (!(seen >> e & 1)) x[e] = 0xff800000u;
        };
        float best[2] = {-INFINITY, -INFINITY};
        auto maximum = [&](const uint32_t (&x)[32]) {
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            best[0] = fmaxf(fmaxf(best[0], __uint_as_float(x[e])), __uint_as_float(x[e + 1]));
            best[1] = fmaxf(fmaxf(best[1], __uint_as_float(x[e + 2])), __uint_as_float(x[e + 3]));
          }
        };
        uint32_t x[2][32];
        tc::tmem_ld_32x32b_x32(s_tmem, x[0]);
        tc::tmem_ld_32x32b_x32(s_tmem + 32, x[1]);
        tc::tmem_ld_wait();
        if (masked) mask(x[0], 0), mask(x[1], 1);
        maximum(x[0]);
        maximum(x[1]);
        tc::tmem_ld_32x32b_x32(s_tmem + 64, x[0]);
        tc::tmem_ld_32x32b_x32(s_tmem + 96, x[1]);
        tc::tmem_ld_wait();
        if (masked) mask(x[0], 2), mask(x[1], 3);
        maximum(x[0]);
        maximum(x[1]);
        const float top = scaled_maximum<M>(fmaxf(best[0], best[1]), mul);
        if (j == 0) {
          ref = top - kHeadroom<M>;
        } else if (__any_sync(0xffffffffu, far_ahead<M>(top, ref))) {
          const float to = fmaxf(ref, top - kHeadroom<M>), f = ref == -INFINITY ? 0.f : exp2_fast(ref - to);
          if (!(ok = tc::warp_wait(o_full, (n_o - 1) & 1))) break;      // the products so far are in O
          tc::fence_after_sync();
#pragma unroll 1
          for (int c = 0; c < DP; c += 16) {
            uint32_t o[16];
            tc::tmem_ld_32x32b_x16(o_tmem + c, o);
            tc::tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            tc::tmem_st_32x32b_x16(o_tmem + c, o);
          }
          sum *= f;
          ref = to;
        }
        const float2 mul_2 = both(mul), neg_2 = both(ref == -INFINITY ? 0.f : -ref);
        float2 part[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        auto probabilities = [&](const uint32_t (&s)[32], int c) {
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            float2 y = fma2(make_float2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), mul_2, neg_2);
            y.x = exp2_fast(y.x), y.y = exp2_fast(y.y);
            part[(e >> 1) & 1] = add2(part[(e >> 1) & 1], y);
            pk[e / 2] = pack2(y.x, y.y, M(0.f));
          }
          tc::tmem_st_32x32b_x16(p_tmem + 16 * c, pk);
        };
        auto ready = [&](uint32_t bar) {      // the product of 64 keys begins while the others are in their exponentials
          tc::tmem_st_wait();
          tc::fence_before_sync();
          __syncwarp();
          tc::arrive_if(lane == 0, bar);
        };
        probabilities(x[0], 2);
        tc::tmem_ld_32x32b_x32(s_tmem, x[0]);
        probabilities(x[1], 3);
        tc::tmem_ld_32x32b_x32(s_tmem + 32, x[1]);
        ready(p_half);
        tc::tmem_ld_wait();
        if (masked) mask(x[0], 0), mask(x[1], 1);
        probabilities(x[0], 0);
        probabilities(x[1], 1);
        ready(p_full);
        part[0] = add2(part[0], part[1]);
        sum += part[0].x + part[0].y;
        ++n_o;
      }
      if (!ok) break;
      const bool whole = it->whole, watch = all_lo > unit0 * kTile || all_hi < (unit0 + count) * kTile;
      const float v_scale = E4M3 ? p.v_scale[it->head] : 1.f;
      const int slot = 2 * blockIdx.x + (it->first_piece ? 1 : 0);
      int64_t out_at = -1;
      if (live) {
        const int r = i * kTile + row;
        out_at = (it->seq.q0 + it->token(p, r)) * p.o_st + it->q_head(p, r) * p.o_sh;
      }
      if (threadIdx.x == 0 && !whole && it->first_piece) p.meta[blockIdx.x].cut = it->cut, p.meta[blockIdx.x].cut_b = it->b;
      give_back();
      // the next queries are on their way during the wait for the last product, and the tensor core has them before this output
      it = take();
      if (!ok) break;
      const bool query = it && it->count[i] > 0;
      if (query) mul = load_query(*it);
      if (count > 0) {
        if (!(ok = tc::warp_wait(o_full, (n_o - 1) & 1))) break;
        tc::fence_after_sync();
      }
      if (query) query_ready();
      if (rows > 0) {
        const float f = !whole ? v_scale : sum == 0.f ? 0.f : v_scale / sum;
        float2 zeros = both(0.f);        // not, where an output is not finite
        int64_t quad[4];       // this lane's four rows after the exchange below
#pragma unroll
        for (int r = 0; r < 4; ++r) quad[r] = __shfl_sync(0xffffffffu, out_at, (lane & ~3) + r);
#pragma unroll 1
        for (int col = 0; col < p.d; col += 32) {
          uint32_t o[32];
          if (count > 0) {
            tc::tmem_ld_32x32b_x32(o_tmem + col, o);
            tc::tmem_ld_wait();
            if (watch) {
#pragma unroll
              for (int e = 0; e < 32; e += 2)
                if (col + e < p.d) zeros = fma2(make_float2(__uint_as_float(o[e]), __uint_as_float(o[e + 1])), both(0.f), zeros);
            }
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = 0;
          }
          if (whole) {
            // 16 bytes of a row per lane would touch 32 lines at once: four lanes exchange so that each row's 64 bytes lie in a quad
            uint32_t h[4][4];
#pragma unroll
            for (int e = 0; e < 16; ++e)
              h[e / 4][e % 4] = pack2(__uint_as_float(o[2 * e]) * f, __uint_as_float(o[2 * e + 1]) * f, T(0.f));
#pragma unroll
            for (int m = 1; m <= 2; m *= 2) {
              const bool upper = lane & m;
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                if (k & m) continue;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const uint32_t got = __shfl_xor_sync(0xffffffffu, upper ? h[k][e] : h[k + m][e], m);
                  if (upper) h[k][e] = got;
                  else h[k + m][e] = got;
                }
              }
            }
            const int at = col + (lane & 3) * 8;
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (quad[r] >= 0 && at < p.d)
                *reinterpret_cast<uint4 *>(reinterpret_cast<char *>(p.out) + (quad[r] + at) * 2) = make_uint4(h[r][0], h[r][1], h[r][2], h[r][3]);
          } else if (live) {     // [slot][column / 4][row] in units of four columns: a warp's rows are neighbours
            float4 *dst = reinterpret_cast<float4 *>(p.part_o) + ((int64_t)slot * (DP / 4) + col / 4) * kRows + i * kTile + row;
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              if (col + e < DP)
                dst[(e / 4) * kRows] = make_float4(__uint_as_float(o[e]) * f, __uint_as_float(o[e + 1]) * f,
                                                   __uint_as_float(o[e + 2]) * f, __uint_as_float(o[e + 3]) * f);
          }
        }
        // (a row whose sum is not finite has it from its own scores)
        if (live && isfinite(sum) && !(zeros.x + zeros.y == 0.f)) *(volatile uint32_t *)&bars.not_finite = 1;
        if (live && !whole)    // (a NaN outweighs the other pieces' rows)
          p.part_ml[(int64_t)slot * kRows + i * kTile + row] = make_float2(sum != sum ? INFINITY : sum == 0.f ? -INFINITY : ref, sum);
      }
      tc::fence_before_sync();   // O is read before the next piece's first product, which waits for this warp's probabilities
    }
    if (!ok && lane == 0) tc::report_timeout(p.status, kStatusEpilogueTimeout);
  } else if (warp < 12) {
    // ---- K and V tiles --------------------------------------------------------------------------------------------
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsCopy));
    const int w4 = warp - 8;
    constexpr int ES = E4M3 ? 1 : 2;
    constexpr int CH = DP * ES / 16;          // 16-byte chunks of a key's row in the cache
    constexpr int RP = 32 / CH;               // rows per pass of a warp
    constexpr int PASSES = 32 / RP;
    const int c = lane % CH, sub = lane / CH;
    const int bytes = min(max(p.d * ES - c * 16, 0), 16);
    uint32_t n = 0, pending = 0;              // stages begun; which of the last have row copies that were not handed on yet
    const uint32_t raw = base + L::kRaw + w4 * (L::kRawBytes / 4) + lane * 16;      // e4m3: this lane's part of a raw tile
    // Hands stage k on; its row copies are the oldest of at most kLag + 1 groups in flight.
    auto finish = [&](uint32_t k) {
      asm volatile("cp.async.wait_group %0;" ::"n"(L::kLag) : "memory");
      if constexpr (E4M3) {
        const uint32_t st = k % S, dst = base + L::kRing + st * L::kTileBytes;
        if (k >= S && !(ok = tc::warp_wait(smem_u32(&bars.kv_free[st]), (k / S - 1) & 1))) return;
#pragma unroll
        for (int q = 0; q < PASSES; ++q) {
          const int r = w4 * 32 + q * RP + sub;
          const uint4 x = ld_shared16(raw + k % (L::kLag + 1) * L::kRawBytes + q * 512);
          const uint2 h0 = e4m3x4_to_f16x4(x.x), h1 = e4m3x4_to_f16x4(x.y), h2 = e4m3x4_to_f16x4(x.z), h3 = e4m3x4_to_f16x4(x.w);
          st_shared16(dst + tile_at(r, 2 * c), h0.x, h0.y, h1.x, h1.y);
          st_shared16(dst + tile_at(r, 2 * c + 1), h2.x, h2.y, h3.x, h3.y);
        }
      }
      fence_async_proxy();
      __syncwarp();
      tc::arrive_if(lane == 0, smem_u32(&bars.kv_full[k % S]));
      pending &= ~(1u << (k & 31));
    };
    auto finish_all = [&]() {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      for (uint32_t k = n > L::kLag ? n - L::kLag : 0; ok && k < n; ++k)
        if (pending >> (k & 31) & 1) finish(k);
    };
    // Stages lag behind only while there are others to begin: the piece after this one may be waiting for its products.
    auto take_or_finish = [&]() -> const Piece * {
      if (!__all_sync(0xffffffffu, tc::mbar_test_addr(smem_u32(&bars.piece_full[n_piece % kPieces]), (n_piece / kPieces) & 1))) finish_all();
      return ok ? take() : nullptr;
    };
    while (const Piece *piece = take_or_finish()) {
      const Piece &it = *piece;
      const int units = max(it.count[0], it.count[1]), head = it.head;
      const int k_begin = max(key_lo(p, it.seq, it.token(p, 0)), it.unit0 * kTile);
      const int k_end = min((long long)key_hi(p, it.seq, it.token(p, it.n_rows - 1)), ((long long)it.unit0 + it.n_units) * kTile);
      const char *kb = reinterpret_cast<const char *>(p.k) + head * p.k_sh * ES;
      const char *vb = reinterpret_cast<const char *>(p.v) + head * p.v_sh * ES;
      const int32_t *pages = p.table + it.b * p.table_stride;
      const int first = it.unit0 * kTile + w4 * 32 + lane;            // this lane's key of the piece's first unit
      give_back();
      auto page_id = [&](int j) -> int {
        const int key = first + j * kTile;
        if (j >= units || key < k_begin || key >= k_end) return -1;
        const int id = pages[page_of(p, key)];
        if (id >= 0 && id < p.num_pages) return id;
        tc::report_timeout(p.status, kStatusBadIndex);
        return -1;
      };
      auto slot_of = [&](int key) { return key - page_of(p, key) * p.page; };
      int ahead = page_id(0);
      for (int j = 0; j < units && ok; ++j) {
        const int id = ahead, key = first + j * kTile, slot = slot_of(key);
        ahead = page_id(j + 1);
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          const int st = n % S;
          const char *src = kv ? vb : kb;
          const int64_t sp = kv ? p.v_sp : p.k_sp, ss = kv ? p.v_ss : p.k_ss;
          bool rows = true;
          if constexpr (!E4M3) {
            if (n >= S && !(ok = tc::warp_wait(smem_u32(&bars.kv_free[st]), (n / S - 1) & 1))) break;
            if (box > 0 && __all_sync(0xffffffffu, id >= 0)) {
              // lane l of the first (boxes x halves): box l / halves of this warp's 32 keys, 64 columns of it
              constexpr int HALVES = DP / 64;
              const int b_i = lane / HALVES, half = lane % HALVES;
              const int bid = __shfl_sync(0xffffffffu, id, b_i * box & 31), bslot = __shfl_sync(0xffffffffu, slot, b_i * box & 31);
              const uint32_t full = smem_u32(&bars.kv_full[st]), dst = base + L::kRing + st * L::kTileBytes;
              tc::expect_tx_if(lane == 0, full, 32 * DP * 2);
              __syncwarp();
              tma_load_4d_if(b_i * box < 32, dst + half * kHalf + (w4 * 32 + b_i * box) * 128, kv ? &v_map : &k_map, full, half * 64, bslot,
                             head, bid);
              rows = false;
            }
          }
          if (rows) {
#pragma unroll(E4M3 ? PASSES : 2)
            for (int q = 0; q < PASSES; ++q) {
              const int r = q * RP + sub;
              const int rid = __shfl_sync(0xffffffffu, id, r), rslot = __shfl_sync(0xffffffffu, slot, r);
              const bool live = rid >= 0 && bytes > 0;
              const uint32_t dst = E4M3 ? raw + n % (L::kLag + 1) * L::kRawBytes + q * 512
                                        : base + L::kRing + st * L::kTileBytes + tile_at(w4 * 32 + r, c);
              cp_async16(dst, live ? src + (rid * sp + rslot * ss) * ES + c * 16 : src, live ? bytes : 0);
            }
            pending |= 1u << (n & 31);
          }
          asm volatile("cp.async.commit_group;" ::: "memory");
          if (n >= L::kLag && (pending >> ((n - L::kLag) & 31) & 1)) finish(n - L::kLag);
          if (!ok) break;
          ++n;
        }
      }
      if (!ok) break;
    }
    if (ok) finish_all();
    asm volatile("cp.async.wait_group 0;" ::: "memory");      // (none is left in flight by a wait that gave up)
    if (!ok)                // nor a box: each has a microsecond or so to arrive, a stage that others left incomplete its polls
      for (uint32_t k = n + 1 > S ? n + 1 - S : 0; k <= n; ++k) tc::mbar_wait(&bars.kv_full[k % S], (k / S) & 1, 1u << 10);
    if (!ok && lane == 0) tc::report_timeout(p.status, kStatusProducerTimeout);
  } else {
    // ---- MMAs -----------------------------------------------------------------------------------------------------
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsMma));
    if (warp == 12) {
      const bool leader = tc::elect_one();
      constexpr uint32_t fmt = __is_same(M, __half) ? 0u : 1u;
      const int n_cols = (p.d + 15) / 16 * 16, k_steps = n_cols / 16;
      const uint32_t i_qk = tc::instr_desc(1, fmt, fmt, kTile, kTile);
      const uint32_t i_pv = tc::instr_desc(1, fmt, fmt, kTile, n_cols) | tc::kInstrBMnMajor;
      uint32_t n = 0, n_q[2] = {0, 0}, n_p[2] = {0, 0};
      auto stage = [&](uint32_t k) { return base + L::kRing + (k % S) * L::kTileBytes; };
      auto full = [&](uint32_t k) { return tc::warp_wait(smem_u32(&bars.kv_full[k % S]), (k / S) & 1); };
      auto scores = [&](int i, uint32_t k) {      // S_i = Q_i K^T
        const uint32_t a = ((base + i * L::kTileBytes) >> 4) | (1u << 16), b = (stage(k) >> 4) | (1u << 16);   // (leading offset: unused)
        if (leader) {
          for (int s = 0; s < k_steps; ++s) {
            const uint32_t off = (s >> 2) * (kHalf >> 4) + (s & 3) * 2;
            tc::mma_f16_ss(tmem + i * kTile, tc::smem_desc_from_words(a + off, tc::kDescHiSw128),
                           tc::smem_desc_from_words(b + off, tc::kDescHiSw128), i_qk, s > 0);
          }
          tc::mma_commit(&bars.s_full[i]);
        }
        __syncwarp();
      };
      auto outputs = [&](int i, uint32_t k, int half, bool more, bool last) {    // O_i (+)= P_i V, 64 of the keys
        const uint32_t b = tc::desc_lo_mn_sw128(stage(k), kHalf) + half * (64 * 128 >> 4);
        if (leader) {
#pragma unroll
          for (int s = 0; s < 4; ++s)
            tc::mma_f16_ts(tmem + (2 + i) * kTile, tmem + i * kTile + kTile / 2 + half * 32 + s * 8,
                           tc::smem_desc_from_words(b + s * (16 * 128 >> 4), tc::kDescHiSw128), i_pv, more || s > 0);
          if (last) tc::mma_commit(&bars.o_full[i]);
        }
        __syncwarp();
      };
      auto release = [&](uint32_t k) {
        if (leader) tc::mma_commit(&bars.kv_free[k % S]);
        __syncwarp();
      };
      while (const Piece *piece = take()) {
        const int count[2] = {piece->count[0], piece->count[1]}, units = max(count[0], count[1]);
        give_back();
        for (int i = 0; i < 2 && ok; ++i)
          if (count[i] > 0) ok = tc::warp_wait(smem_u32(&bars.q_full[i]), n_q[i]++ & 1);
        if (!ok) break;
        if (units == 0) continue;
        if (!(ok = full(n))) break;
        tc::fence_after_sync();
        for (int i = 0; i < 2; ++i)
          if (count[i] > 0) scores(i, n);
        release(n);
        // stages: n is K of unit 0, then V and K alternate
        for (int j = 0; j < units && ok; ++j) {
          const uint32_t v = n + 2 * j + 1, k = v + 1;
          if (!(ok = full(v))) break;
          const bool more = j + 1 < units;
          bool have_k = false;
          for (int i = 0; i < 2; ++i) {
            if (j < count[i]) {
              if (!(ok = tc::warp_wait(smem_u32(&bars.p_half[i]), n_p[i] & 1))) break;
              tc::fence_after_sync();
              outputs(i, v, 1, j > 0, false);
              if (!(ok = tc::warp_wait(smem_u32(&bars.p_full[i]), n_p[i]++ & 1))) break;
              tc::fence_after_sync();
              outputs(i, v, 0, true, true);
            }
            if (j + 1 < count[i]) {
              if (!have_k && !(ok = full(k))) break;
              have_k = true;
              tc::fence_after_sync();
              scores(i, k);
            }
          }
          if (!ok) break;
          release(v);
          if (more) release(k);
        }
        if (!ok) break;
        n += 2 * units;
      }
      // the last arrival that the tensor core owes this CTA
      if (ok && n > 0) ok = tc::warp_wait(smem_u32(&bars.kv_free[(n - 1) % S]), ((n - 1) / S) & 1);
      if (!ok) {              // tensor memory goes back when the products that were issued are done
        if (leader) tc::mma_commit(&bars.drain);
        __syncwarp();
        tc::warp_wait(smem_u32(&bars.drain), 0);
        if (lane == 0) tc::report_timeout(p.status, kStatusMmaTimeout);
      }
    } else if (warp == 13) {
      // ---- the walk -----------------------------------------------------------------------------------------------
      Walk it(range);
      for (bool more = true; more && ok;) {
        more = it.next(p);
        const uint32_t i = n_piece % kPieces;
        if (n_piece >= kPieces && !(ok = tc::warp_wait(smem_u32(&bars.piece_free[i]), (n_piece / kPieces - 1) & 1))) break;
        if (lane == 0) {
          Piece &q = pieces[i];
          q.seq = it.seq, q.b = more ? it.b : -1, q.head = it.head, q.unit0 = it.unit0, q.n_units = it.n_units;
          q.r0 = it.r0, q.n_rows = it.n_rows, q.first_piece = it.first_piece, q.whole = it.whole;
          if (more) q.cut = it.cut(), q.count[0] = tile_count(p, it, 0), q.count[1] = tile_count(p, it, 1);
        }
        __syncwarp();
        tc::arrive_if(lane == 0, smem_u32(&bars.piece_full[i]));
        ++n_piece;
      }
      if (!ok && lane == 0) tc::report_timeout(p.status, kStatusProducerTimeout);
    }
  }
  // every product has been waited for by the rows that read it; tensor memory goes back
  tc::fence_before_sync();
  __syncthreads();
  if (threadIdx.x == 0) p.meta[blockIdx.x].not_finite = (int)*(volatile uint32_t *)&bars.not_finite;
  if (warp == 12) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, 512);
  }
}

// The cache as a tensor (column, slot, head, page) with a box of 64 columns of `box` slots.  Strides that a tensor map cannot
// hold (none, or of 2^40 bytes) leave the row copies.
template <typename T>
bool page_map(CUtensorMap *map, const AttnParams &p, const void *base, const int64_t (&strides)[3], int box) {
  const uint64_t dims[4] = {(uint64_t)p.d, (uint64_t)p.page, (uint64_t)p.hkv, (uint64_t)p.num_pages};
  uint64_t bytes[3];
  for (int i = 0; i < 3; ++i) {
    if (dims[i + 1] > 1 && (strides[i] <= 0 || strides[i] >= (int64_t)1 << 38)) return false;
    bytes[i] = dims[i + 1] > 1 ? (uint64_t)strides[i] * 2 : (uint64_t)p.d * 2;    // (of one: never used)
  }
  const uint32_t shape[4] = {64, (uint32_t)box, 1, 1};
  return make_tensor_map(map, base, __is_same(T, __half) ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, dims,
                         bytes, shape, true) == ZT_SUCCESS;
}

template <typename T, bool E4M3, int DP>
int launch(const AttnParams &p, const AttnPlan &plan, cudaStream_t st) {
  constexpr int smem = Smem<DP, E4M3>::kBytes + 1024;
  static PerDeviceOnce once;
  auto kern = attention_tcgen05_kernel<T, E4M3, DP>;
  const int rc = allow_dynamic_smem(once, kern, smem);
  if (rc != ZT_SUCCESS) return rc;
  CUtensorMap k_map{}, v_map{};
  int box = 0;
  if (!E4M3 && p.page % 8 == 0 && p.num_pages > 0) {
    box = std::min(p.page & -p.page, kBoxSlots);      // divides the page, so that no box of aligned keys spans two
    const int64_t ks[3] = {p.k_ss, p.k_sh, p.k_sp}, vs[3] = {p.v_ss, p.v_sh, p.v_sp};
    if (!page_map<T>(&k_map, p, p.k, ks, box) || !page_map<T>(&v_map, p, p.v, vs, box)) box = 0;
  }
  ZT_CUDA_OK(launch_overlapped(kern, dim3(plan.grid), dim3(kThreads), (size_t)smem, st, p, k_map, v_map, box));
  return launch_status("attention_tcgen05_kernel");
}

}  // namespace

int attention_tcgen05_launch(const AttnParams &p, const AttnPlan &plan, int dtype, int cache_dtype, cudaStream_t st) {
  const bool e4m3 = cache_dtype == ZT_E4M3, narrow = plan.dp == 64;
  if (dtype == ZT_BF16) {
    if (e4m3) return narrow ? launch<__nv_bfloat16, true, 64>(p, plan, st) : launch<__nv_bfloat16, true, 128>(p, plan, st);
    return narrow ? launch<__nv_bfloat16, false, 64>(p, plan, st) : launch<__nv_bfloat16, false, 128>(p, plan, st);
  }
  if (e4m3) return narrow ? launch<__half, true, 64>(p, plan, st) : launch<__half, true, 128>(p, plan, st);
  return narrow ? launch<__half, false, 64>(p, plan, st) : launch<__half, false, 128>(p, plan, st);
}

}  // namespace zt
