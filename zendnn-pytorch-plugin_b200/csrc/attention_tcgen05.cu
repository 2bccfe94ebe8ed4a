// Paged attention on the tensor cores of sm_100a, for chunks and prompts.
//
// An item is 256 (token, head of the group) rows of one kv head, as two tiles of 128 that share every K and V tile of 128 keys.
// Scores S = Q K^T of a tile go to tensor memory (128 columns), one thread per row turns them into probabilities that replace
// them there as 16-bit pairs, and O += P V accumulates in tensor memory with P as the tensor-memory operand.  Of the two tiles
// one is in its exponentials while the tensor core works for the other.
//
//   warps 0-3, 4-7   a row of tile 0 / 1 each thread: query rows to shared memory, running maximum and sum, probabilities, output
//   warps 8-11       K and V tiles into a ring, row by row from the pages (any page size), 16 bytes per asynchronous copy; slots past
//                    the visible keys become zeros, so stale contents of a page never meet the arithmetic.  e4m3 caches come
//                    through registers and are stored as halves (exact)
//   warp 12          issues the MMAs
//
// The reference of the exponents follows the row maximum only when that has run 8 (log2) ahead of it, so the rows of O are
// rescaled a few times at the start and hardly ever after; the thread that finds it does it itself.  Probabilities are rounded
// to the products' type; their sum is of the unrounded fp32 values.  e4m3: fp16 products, query rows brought below 2 by a power of
// two as in the streaming kernel.
#include "attention.cuh"

namespace zt {

namespace {

constexpr int kTile = 128;                 // rows of a tile, keys of a unit
constexpr int kRows = 2 * kTile;
constexpr int kThreads = 512;              // four warpgroups: tile 0, tile 1, copies, MMA (and three idle warps)
constexpr int kHalf = kTile * 128;         // bytes of 64 columns of a tile: 128 rows of 128 bytes, swizzled
constexpr int kLag = 2;                    // stages whose copies are in flight behind the newest

template <int DP>
struct Smem {
  static constexpr int kTileBytes = kTile * DP * 2;
  static constexpr int kStages = DP == 128 ? 5 : 8;
  static constexpr int kRing = 2 * kTileBytes;                  // after the two query tiles
  static constexpr int kBytes = kRing + kStages * kTileBytes;
};

// Registers per thread after the split; the sum over the four warpgroups is that of the launch, 4 * 128.
constexpr int kRegsSoftmax = 184, kRegsCopy = 88, kRegsMma = 56;
static_assert(2 * kRegsSoftmax + kRegsCopy + kRegsMma <= 4 * 128, "register split above the launch's registers");

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, int bytes) {   // the rest of the 16 is zero
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void st_shared16(uint32_t dst, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(dst), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
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

struct Barriers {
  uint64_t kv_full[8], kv_free[8];
  uint64_t q_full[2], s_full[2], p_full[2], o_full[2];
  uint32_t tmem;
};

// Units that a tile of a piece works on, from the piece's first.
template <int UK>
__device__ __forceinline__ int tile_count(const AttnParams &p, const AttnWalk<kRows, UK> &it, int i) {
  const int rows = it.n_rows - i * kTile;
  if (rows <= 0) return 0;
  const int last = i * kTile + min(rows, kTile) - 1;
  const int hi = key_hi(p, it.seq, it.token(p, last));
  return min(max((hi + UK - 1) / UK - it.unit0, 0), it.n_units);
}

template <typename T, bool E4M3, int DP>
__global__ void __launch_bounds__(kThreads, 1) attention_tcgen05_kernel(const __grid_constant__ AttnParams p) {
  using M = std::conditional_t<E4M3, __half, T>;
  using L = Smem<DP>;
  constexpr int S = L::kStages, CHUNKS = DP / 8;
  extern __shared__ unsigned char smem_raw[];
  __shared__ Barriers bars;
  __shared__ long long s_scan[40];
  unsigned char *smem = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const uint32_t base = smem_u32(smem);
  const int warp = tc::uniform_warp(), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) tc::mbar_init(&bars.kv_full[i], 4), tc::mbar_init(&bars.kv_free[i], 1);
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&bars.q_full[i], 4), tc::mbar_init(&bars.p_full[i], 4);
      tc::mbar_init(&bars.s_full[i], 1), tc::mbar_init(&bars.o_full[i], 1);
    }
    tc::mbar_fence_init();
  }
  if (warp == 12) tc::tmem_alloc(&bars.tmem, 512);
  grid_launch_dependents();
  grid_dependency_wait();
  const AttnRange range = attention_range<kRows, kTile, kThreads>(p, 1, reinterpret_cast<int *>(smem), s_scan);
  zero_tail_rows<T>(p, kThreads);
  if (threadIdx.x == 0) p.meta[blockIdx.x] = make_int4(-1, 0, 0, 0);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = bars.tmem;
  AttnWalk<kRows, kTile> it(range);
  bool ok = true;

  if (warp < 8) {
    // ---- a tile's rows -----------------------------------------------------------------------------------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    const int i = warp >> 2, row = threadIdx.x & (kTile - 1);     // tile, row of it (= lane of tensor memory)
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_tmem = tmem + i * kTile + lanes, o_tmem = tmem + 2 * kTile + i * kTile + lanes;
    const uint32_t s_full = smem_u32(&bars.s_full[i]), o_full = smem_u32(&bars.o_full[i]);
    const uint32_t q_full = smem_u32(&bars.q_full[i]), p_full = smem_u32(&bars.p_full[i]);
    uint32_t n_s = 0, n_o = 0;     // phases of s_full and o_full so far

    auto load_query = [&]() -> float {   // this thread's row of the piece to shared memory; returns the factor of its scores
      const bool live = i * kTile + row < it.n_rows;
      const int r = live ? i * kTile + row : 0;
      const char *src = reinterpret_cast<const char *>(p.q) + ((it.seq.q0 + it.token(p, r)) * p.q_st + it.q_head(p, r) * p.q_sh) * 2;
      const uint32_t dst = base + i * L::kTileBytes;
      float mul = p.scale_log2;
      if constexpr (!E4M3) {
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
          const uint4 x = live && c * 8 < p.d ? *reinterpret_cast<const uint4 *>(src + c * 16) : make_uint4(0, 0, 0, 0);
          st_shared16(dst + tile_at(row, c), x.x, x.y, x.z, x.w);
        }
      } else {
        float top = 0.f;
        uint4 x[CHUNKS];
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
          x[c] = live && c * 8 < p.d ? *reinterpret_cast<const uint4 *>(src + c * 16) : make_uint4(0, 0, 0, 0);
          const uint32_t w[4] = {x[c].x, x[c].y, x[c].z, x[c].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 f = unpack2(w[e], T(0.f));
            top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
          }
        }
        const float k_scale = p.k_scale[it.head];
        const int ex = row_exponent(top);
        const float down = copysignf(ldexpf(1.f, -ex), k_scale);
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
          const uint32_t w[4] = {x[c].x, x[c].y, x[c].z, x[c].w};
          uint32_t h[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 f = unpack2(w[e], T(0.f));
            h[e] = pack2(f.x * down, f.y * down, M(0.f));
          }
          st_shared16(dst + tile_at(row, c), h[0], h[1], h[2], h[3]);
        }
        mul *= fabsf(k_scale) * ldexpf(1.f, ex);
      }
      fence_async_proxy();
      __syncwarp();
      tc::arrive_if(lane == 0, q_full);
      return fmaxf(mul, 1e-30f);    // a scale of zero: masked scores stay minus infinity
    };

    bool has = it.next(p);
    int count = has ? tile_count(p, it, i) : 0;
    float mul = 0.f;
    if (count > 0) mul = load_query();
    while (has && ok) {
      const int rows = min(max(it.n_rows - i * kTile, 0), kTile);
      const bool live = row < rows;
      int lo = 0, hi = 0, all_lo = 0, all_hi = 0;      // keys that this row sees; that every row of the tile sees
      if (rows > 0) {
        const int tok = it.token(p, i * kTile + (live ? row : 0));
        lo = key_lo(p, it.seq, tok), hi = live ? key_hi(p, it.seq, tok) : 0;
        all_lo = key_lo(p, it.seq, it.token(p, i * kTile + rows - 1)), all_hi = key_hi(p, it.seq, it.token(p, i * kTile));
      }
      float ref = -INFINITY, sum = 0.f;
      for (int j = 0; j < count; ++j) {
        const int key0 = (it.unit0 + j) * kTile;
        if (!(ok = tc::warp_wait(s_full, n_s & 1))) break;
        ++n_s;
        tc::fence_after_sync();
        uint32_t s[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tc::tmem_ld_32x32b_x32(s_tmem + 32 * c, s[c]);
        tc::tmem_ld_wait();
        if (key0 < all_lo || key0 + kTile > all_hi) {
          const int from = lo - key0, to = hi - key0;
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (32 * c + e < from || 32 * c + e >= to) s[c][e] = 0xff800000u;
        }
        float mx[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          mx[c] = fmaxf(__uint_as_float(s[c][0]), __uint_as_float(s[c][1]));
#pragma unroll
          for (int e = 2; e < 32; e += 2) mx[c] = fmaxf(fmaxf(mx[c], __uint_as_float(s[c][e])), __uint_as_float(s[c][e + 1]));
        }
        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * mul;
        if (j == 0) {
          ref = top;
        } else if (__any_sync(0xffffffffu, top > ref + kLazyRescale)) {
          const float to = fmaxf(ref, top), f = ref == -INFINITY ? 0.f : exp2_fast(ref - to);
          if (!(ok = tc::warp_wait(o_full, (n_o - 1) & 1))) break;      // the products so far are in O
          tc::fence_after_sync();
#pragma unroll
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
        const float neg = ref == -INFINITY ? 0.f : -ref;
        const float2 mul2 = make_float2(mul, mul), neg2 = make_float2(neg, neg);
        float2 part[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            float2 x = fma2(make_float2(__uint_as_float(s[c][e]), __uint_as_float(s[c][e + 1])), mul2, neg2);
            x.x = exp2_fast(x.x), x.y = exp2_fast(x.y);
            part[(e >> 1) & 1] = add2(part[(e >> 1) & 1], x);
            pk[e / 2] = pack2(x.x, x.y, M(0.f));
          }
          tc::tmem_st_32x32b_x16(s_tmem + 16 * c, pk);
        }
        const float2 both = add2(part[0], part[1]);
        sum += both.x + both.y;
        tc::tmem_st_wait();
        tc::fence_before_sync();
        __syncwarp();
        tc::arrive_if(lane == 0, p_full);
        ++n_o;
      }
      if (!ok) break;
      // what the output needs, before the walk moves on; the next query rows go ahead of the wait for the last product
      const bool whole = it.whole;
      const int head = it.head, done = count;
      const int64_t slot_row = (int64_t)(2 * blockIdx.x + (it.first_piece ? 1 : 0)) * kRows + i * kTile + row;
      char *out = nullptr;
      if (live) {
        const int r = i * kTile + row;
        out = reinterpret_cast<char *>(p.out) + ((it.seq.q0 + it.token(p, r)) * p.o_st + it.q_head(p, r) * p.o_sh) * 2;
      }
      if (threadIdx.x == 0 && !whole && it.first_piece) p.meta[blockIdx.x] = make_int4(it.b, it.tile, head, it.last_cta);
      has = it.next(p);
      count = has ? tile_count(p, it, i) : 0;
      if (count > 0) mul = load_query();
      if (done > 0) {
        if (!(ok = tc::warp_wait(o_full, (n_o - 1) & 1))) break;
        tc::fence_after_sync();
      }
      const float v_scale = E4M3 ? p.v_scale[head] : 1.f;
      const float f = !whole ? v_scale : sum == 0.f ? 0.f : v_scale / sum;
#pragma unroll 1
      for (int c = 0; c < p.d; c += 32) {
        uint32_t o[32];
        if (done > 0) {
          tc::tmem_ld_32x32b_x32(o_tmem + c, o);
          tc::tmem_ld_wait();
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0;
        }
        if (!live) continue;
#pragma unroll
        for (int e = 0; e < 32; e += 8) {
          if (c + e >= p.d) break;
          float x[8];
#pragma unroll
          for (int q = 0; q < 8; ++q) x[q] = __uint_as_float(o[e + q]) * f;
          if (whole) {
            *reinterpret_cast<uint4 *>(out + (c + e) * 2) =
                make_uint4(pack2(x[0], x[1], T(0.f)), pack2(x[2], x[3], T(0.f)), pack2(x[4], x[5], T(0.f)), pack2(x[6], x[7], T(0.f)));
          } else {
            float4 *dst = reinterpret_cast<float4 *>(p.part_o + slot_row * DP + c + e);
            dst[0] = make_float4(x[0], x[1], x[2], x[3]), dst[1] = make_float4(x[4], x[5], x[6], x[7]);
          }
        }
      }
      // (a NaN outweighs the other pieces' rows)
      if (live && !whole) p.part_ml[slot_row] = make_float2(sum != sum ? INFINITY : sum == 0.f ? -INFINITY : ref, sum);
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
    uint32_t n = 0;                           // stages begun
    while (ok && it.next(p)) {
      const int units = max(tile_count(p, it, 0), tile_count(p, it, 1));
      const int k_begin = max(key_lo(p, it.seq, it.token(p, 0)), it.unit0 * kTile);
      const int k_end = min((long long)key_hi(p, it.seq, it.token(p, it.n_rows - 1)), ((long long)it.unit0 + it.n_units) * kTile);
      const char *kb = reinterpret_cast<const char *>(p.k) + it.head * p.k_sh * ES;
      const char *vb = reinterpret_cast<const char *>(p.v) + it.head * p.v_sh * ES;
      const int32_t *pages = p.table + it.b * p.table_stride;
      const int first = it.unit0 * kTile + w4 * 32 + lane;            // this lane's key of the piece's first unit
      auto page_id = [&](int j) -> int {
        const int key = first + j * kTile;
        if (j >= units || key < k_begin || key >= k_end) return -1;
        const int id = pages[page_of(p, key)];
        if (id >= 0 && id < p.num_pages) return id;
        tc::report_timeout(p.status, kStatusBadIndex);
        return -1;
      };
      int ahead = page_id(0);
      for (int j = 0; j < units && ok; ++j) {
        const int id = ahead, key = first + j * kTile, slot = key - page_of(p, key) * p.page;
        ahead = page_id(j + 1);
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          const int st = n % S;
          const uint32_t dst = base + L::kRing + st * L::kTileBytes;
          const char *src = kv ? vb : kb;
          const int64_t sp = kv ? p.v_sp : p.k_sp, ss = kv ? p.v_ss : p.k_ss;
          if constexpr (!E4M3) {
            if (n >= S && !(ok = tc::warp_wait_idle(smem_u32(&bars.kv_free[st]), (n / S - 1) & 1))) break;
#pragma unroll
            for (int q = 0; q < PASSES; ++q) {
              const int r = q * RP + sub;
              const int rid = __shfl_sync(0xffffffffu, id, r), rslot = __shfl_sync(0xffffffffu, slot, r);
              const bool live = rid >= 0 && bytes > 0;
              cp_async16(dst + tile_at(w4 * 32 + r, c), live ? src + (rid * sp + rslot * ss) * ES + c * 16 : src, live ? bytes : 0);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            if (n >= kLag) {     // the stage kLag behind this one has arrived
              asm volatile("cp.async.wait_group %0;" ::"n"(kLag) : "memory");
              fence_async_proxy();
              __syncwarp();
              tc::arrive_if(lane == 0, smem_u32(&bars.kv_full[(n - kLag) % S]));
            }
          } else {
            uint4 x[PASSES];     // 16 bytes of PASSES rows, in flight while the ring's slot drains
#pragma unroll
            for (int q = 0; q < PASSES; ++q) {
              const int r = q * RP + sub;
              const int rid = __shfl_sync(0xffffffffu, id, r), rslot = __shfl_sync(0xffffffffu, slot, r);
              x[q] = rid >= 0 && bytes > 0 ? *reinterpret_cast<const uint4 *>(src + rid * sp + rslot * ss + c * 16) : make_uint4(0, 0, 0, 0);
            }
            if (n >= S && !(ok = tc::warp_wait_idle(smem_u32(&bars.kv_free[st]), (n / S - 1) & 1))) break;
#pragma unroll
            for (int q = 0; q < PASSES; ++q) {
              const int r = w4 * 32 + q * RP + sub;
              st_shared16(dst + tile_at(r, 2 * c), e4m3x2_to_f16x2(x[q].x), e4m3x2_to_f16x2(x[q].x >> 16), e4m3x2_to_f16x2(x[q].y),
                          e4m3x2_to_f16x2(x[q].y >> 16));
              st_shared16(dst + tile_at(r, 2 * c + 1), e4m3x2_to_f16x2(x[q].z), e4m3x2_to_f16x2(x[q].z >> 16), e4m3x2_to_f16x2(x[q].w),
                          e4m3x2_to_f16x2(x[q].w >> 16));
            }
            fence_async_proxy();
            __syncwarp();
            tc::arrive_if(lane == 0, smem_u32(&bars.kv_full[st]));
          }
          ++n;
        }
      }
    }
    if constexpr (!E4M3) {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      fence_async_proxy();
      __syncwarp();
      if (ok)
        for (uint32_t s = n > kLag ? n - kLag : 0; s < n; ++s) tc::arrive_if(lane == 0, smem_u32(&bars.kv_full[s % S]));
    }
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
      auto outputs = [&](int i, uint32_t k, bool more) {    // O_i (+)= P_i V
        const uint32_t b = tc::desc_lo_mn_sw128(stage(k), kHalf);
        if (leader) {
#pragma unroll
          for (int s = 0; s < kTile / 16; ++s)
            tc::mma_f16_ts(tmem + (2 + i) * kTile, tmem + i * kTile + s * 8,
                           tc::smem_desc_from_words(b + s * (16 * 128 >> 4), tc::kDescHiSw128), i_pv, more || s > 0);
          tc::mma_commit(&bars.o_full[i]);
        }
        __syncwarp();
      };
      auto release = [&](uint32_t k) {
        if (leader) tc::mma_commit(&bars.kv_free[k % S]);
        __syncwarp();
      };
      while (ok && it.next(p)) {
        const int count[2] = {tile_count(p, it, 0), tile_count(p, it, 1)};
        const int units = max(count[0], count[1]);
        for (int i = 0; i < 2 && ok; ++i)
          if (count[i] > 0) ok = tc::warp_wait(smem_u32(&bars.q_full[i]), n_q[i]++ & 1);
        if (!ok || units == 0) continue;
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
              if (!(ok = tc::warp_wait(smem_u32(&bars.p_full[i]), n_p[i]++ & 1))) break;
              tc::fence_after_sync();
              outputs(i, v, j > 0);
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
        n += 2 * units;
      }
      // the last arrival that the tensor core owes this CTA
      if (ok && n > 0) ok = tc::warp_wait(smem_u32(&bars.kv_free[(n - 1) % S]), ((n - 1) / S) & 1);
      if (!ok && lane == 0) tc::report_timeout(p.status, kStatusMmaTimeout);
    }
  }
  // every product has been waited for by the rows that read it; tensor memory goes back
  tc::fence_before_sync();
  __syncthreads();
  if (warp == 12) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, 512);
  }
}

template <typename T, bool E4M3, int DP>
int launch(const AttnParams &p, const AttnPlan &plan, cudaStream_t st) {
  constexpr int smem = Smem<DP>::kBytes + 1024;
  static PerDeviceOnce once, checked;
  auto kern = attention_tcgen05_kernel<T, E4M3, DP>;
  int rc = allow_dynamic_smem(once, kern, smem);
  if (rc != ZT_SUCCESS) return rc;
  int dev = 0;
  ZT_CUDA_OK(cudaGetDevice(&dev));
  if (!checked.done[dev]) {     // the register split counts on the launch holding 128 per thread
    cudaFuncAttributes attr;
    ZT_CUDA_OK(cudaFuncGetAttributes(&attr, kern));
    ZT_REQUIRE(attr.numRegs >= 128, ZT_UNSUPPORTED, "attention_tcgen05_kernel: built with %d registers, 128 expected", attr.numRegs);
    checked.done[dev] = true;
  }
  ZT_CUDA_OK(launch_overlapped(kern, dim3(plan.grid), dim3(kThreads), (size_t)smem, st, p));
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
