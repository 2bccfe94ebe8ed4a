// Paged attention for few rows per kv head (decode, short chunks) and for every shape that has no other kernel: K and V stream
// from HBM once, with a running maximum and sum.
//
// A CTA of four warps takes units of 64 keys of an item; each warp streams its own 16 keys of every unit through a private ring
// in shared memory (16-byte asynchronous copies, whose zero fill also blanks slots past the visible keys, so stale contents of a
// page never meet the arithmetic) and keeps its own maxima, sums and output rows in registers: no barrier between warps until
// the item ends, where the four are added through shared memory.  Two or three CTAs share an SM, so that others stream while one
// is in such an end.
//
// For 16 and 32 rows those are the 16-row operand of mma.sync.m16n8k16, keys its columns; the accumulator layout of the scores is the
// operand layout of the probabilities.  For up to 8 rows (decode with groups of up to 8) they are the 8 columns instead, and keys, then
// columns of the values, the 16 rows: half as many accumulators, exponentials and products, for two transpositions of the
// probabilities per 16 keys.  One token over 700 keys 7.6 us with 16 rows, 6.8 with 8; 256 sequences of 100 - 600 keys 67.6 and 64.3;
// 17 of 9000 - 14500, heads of 64, 16.0 and 14.7; where HBM is the bound there is no difference.
//
// Bound by HBM for 16-bit caches: 64 sequences of 500 - 8000 keys (32 heads over 8, 128 wide) take 182 us, 6.3 TB/s of the 6.55 that a
// copy reaches.  An e4m3 cache takes 115 us, 5.0 TB/s: its rows are 128 bytes, 1 KB apart (16-bit heads of 64 elements, the same rows,
// reach 5.8; 6.1 with one kv head, where they are contiguous), and as many instructions go to each key for half the bytes.
//
// e4m3 keys and values become halves in registers, which is exact; the
// products then run in fp16 with query rows brought to a maximum below 2 by a power of two (what that takes from an element is
// below 2^-25 of its row's largest).  Probabilities are rounded to the type of the product (half a step of 2^-8 or 2^-11 of
// each, in fp16 2^-32 of the row's sum for those that are its subnormals; added by the tensor cores in fp32); the sum that
// divides them is of the unrounded fp32 values.
#include "attention.cuh"

namespace zt {

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kKeys = 16;                  // of a warp per unit
constexpr int kUnit = kWarps * kKeys;
constexpr int kExtra = 2;                  // units that an item costs beside its own

// Three CTAs share an SM where their rows leave the registers (up to 16 rows; 64 kept keys ahead per CTA), else two.  Decode of 64
// sequences of 500 - 8000 keys: 191 us with two, 182 with three; an e4m3 cache of 4 x 110000 keys (16 rows): 220 and 202.
template <int R>
__host__ __device__ constexpr int ctas_per_sm() { return R <= 16 ? 3 : 2; }
template <int DP, bool E4M3>
__host__ __device__ constexpr int stage_bytes() { return 2 * kKeys * DP * (E4M3 ? 1 : 2); }
template <bool E4M3, int R>
__host__ __device__ constexpr int stages() { return (E4M3 ? 2 : 1) * (R <= 16 ? 2 : 3); }
template <int DP, bool E4M3, int R>
__host__ __device__ constexpr int ring_bytes() { return kWarps * stages<E4M3, R>() * stage_bytes<DP, E4M3>(); }
template <int R, int DP>
__host__ __device__ constexpr int merge_bytes() { return kWarps * R * (DP + 8) * 4 + kWarps * R * 8 + R * 8 + R * DP * 4; }

__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ uint32_t ld_shared4(uint32_t src) {
  uint32_t x;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(x) : "r"(src) : "memory");
  return x;
}
__device__ __forceinline__ uint32_t ld_shared2(uint32_t src) {
  uint16_t x;
  asm volatile("ld.shared.b16 %0, [%1];" : "=h"(x) : "r"(src) : "memory");
  return x;
}
// Of an 8x8 matrix of 16-bit elements, two neighbours of a row in each lane.
__device__ __forceinline__ uint32_t transposed8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float4 ld_cluster16(uint32_t addr) {
  float4 x;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "r"(addr) : "memory");
  return x;
}

// An item, or a slice of its keys, of a CTA that belongs to one sequence and kv head.
struct DirectPiece {
  SeqInfo seq;
  int b, head, unit0, n_units, n_rows, r0;
  __device__ int token(const AttnParams &p, int row) const { return (r0 + row) / p.group; }
  __device__ int q_head(const AttnParams &p, int row) const { return head * p.group + (r0 + row) % p.group; }
};

// DIRECT: for short contexts, where dividing the batch and joining the pieces (two dependent steps of about 2 us and a launch) cost
// more than they even out: a cluster of p.slices CTAs per sequence and kv head, which add their rows through shared memory.  (64
// keys take a CTA 1 us, by the length of its chain of instructions: a ring of five stages instead of two changed nothing.)
template <typename T, bool E4M3, int DP, int R, bool DIRECT>
__global__ void __launch_bounds__(kThreads, ctas_per_sm<R>()) attention_stream_kernel(const __grid_constant__ AttnParams p) {
  using M = std::conditional_t<E4M3, __half, T>;
  constexpr bool NARROW = R == 8;          // the transposed form
  constexpr int MT = NARROW ? 1 : R / 16, S = stages<E4M3, R>(), SB = stage_bytes<DP, E4M3>();
  constexpr int ES = E4M3 ? 1 : 2;
  constexpr int CH = DP * ES / 16;            // 16-byte chunks of a key's row
  constexpr int KS = DP / 16;                 // 16-element steps of the score product
  constexpr int NT = DP / 8;                  // 8-column tiles of the output
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ AttnScratch s_scan;
  if constexpr (DIRECT) grid_launch_dependents();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = tc::uniform_warp();
  const int g = lane >> 2, t4 = lane & 3;
  zero_tail_rows<T>(p, kThreads);
  unsigned char *ring = smem + warp * S * SB;
  const uint32_t ring_addr = smem_u32(ring);
  float *merge_o = reinterpret_cast<float *>(smem);                                   // [warp][R][DP + 8]
  float2 *merge_ml = reinterpret_cast<float2 *>(smem + kWarps * R * (DP + 8) * 4);    // [warp][R]
  float2 *slice_ml = merge_ml + kWarps * R;                                           // DIRECT: [R], and the rows of this slice [R][DP]
  float *slice_o = reinterpret_cast<float *>(slice_ml + R);
  auto work = [&](const auto &it) {
    const SeqInfo seq = it.seq;
    const int b = it.b, head = it.head, n_units = it.n_units, unit0 = it.unit0, n_rows = it.n_rows;
    const int tok0 = it.token(p, 0), tok1 = it.token(p, n_rows - 1);
    // keys that some row sees, within this piece
    const int k_begin = max(key_lo(p, seq, tok0), unit0 * kUnit);
    const int k_end = min((long long)key_hi(p, seq, tok1), ((long long)unit0 + n_units) * kUnit);

    // ---- query rows as operand fragments (their loads go out before those of the keys wait for the page table) ----
    constexpr int HALVES = NARROW ? 1 : 2;          // of 8 rows in a fragment
    uint32_t qf[MT][KS][2 * HALVES];
    int lo[MT][2], hi[MT][2];                       // keys that the two rows of this lane's scores see
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int row = NARROW ? 2 * t4 + half : m * 16 + half * 8 + g;
        const bool live = row < n_rows;
        const int tok = it.token(p, live ? row : 0);
        lo[m][half] = live ? key_lo(p, seq, tok) : 0;
        hi[m][half] = live ? key_hi(p, seq, tok) : 0;
      }
#pragma unroll
      for (int half = 0; half < HALVES; ++half) {
        const int row = m * 16 + half * 8 + g;
        const bool live = row < n_rows;
        const int tok = it.token(p, live ? row : 0), qh = it.q_head(p, live ? row : 0);
        const char *src = reinterpret_cast<const char *>(p.q) + ((seq.q0 + tok) * p.q_st + qh * p.q_sh) * 2;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
#pragma unroll
          for (int part = 0; part < 2; ++part) {
            // e4m3: a lane's four bytes of a key are elements 4t..4t+3 of a step, whichever column of the product they are
            const int e = 16 * s + (E4M3 ? 4 * t4 + 2 * part : 8 * part + 2 * t4);
            qf[m][s][HALVES * part + half] = live && e < p.d ? *reinterpret_cast<const uint32_t *>(src + e * 2) : 0u;
          }
        }
      }
    }
    // keys that every live row sees: pieces of them need no masks
    const int all_lo = key_lo(p, seq, tok1), all_hi = key_hi(p, seq, tok0);

    // ---- the ring -------------------------------------------------------------------------------------------
    const char *kb = reinterpret_cast<const char *>(p.k) + head * p.k_sh * ES;
    const char *vb = reinterpret_cast<const char *>(p.v) + head * p.v_sh * ES;
    const int32_t *pages = p.table + b * p.table_stride;
    const int key0 = unit0 * kUnit + warp * kKeys;
    // Pages of a power of two of at least 16 slots hold a warp's 16 keys in one: a lookup is of 32 units, one per lane, and made up to
    // 64 units ahead.  Else lane 0-15 have the page and slot of a key each, two units ahead of the copies.
    const bool one_page = p.page_shift >= 4;
    auto page_id = [&](int i) -> int {
      const int first = key0 + i * kUnit, key = first + (one_page ? 0 : lane & 15);
      if (i >= n_units || (one_page ? first + kKeys : key + 1) <= k_begin || key >= k_end) return -1;
      const int id = pages[page_of(p, key)];
      if (id >= 0 && id < p.num_pages) return id;
      tc::report_timeout(p.status, kStatusBadIndex);
      return -1;
    };
    auto swizzled = [](int row, int c) { return CH == 4 ? (c ^ ((row >> 1) & 3)) : (c ^ (row & 7)); };
    int ids = page_id(one_page ? lane : 0), next_ids = page_id(one_page ? 32 + lane : 1);
    auto issue = [&](int i) {
      int id = ids;
      if (one_page) {
        id = __shfl_sync(0xffffffffu, ids, i & 31);
        if ((i & 31) == 31) ids = next_ids, next_ids = page_id(i + 33 + lane);
      } else {
        ids = next_ids, next_ids = page_id(i + 2);
      }
      if (i < n_units) {
        const int first = key0 + i * kUnit;
        constexpr int RP = 32 / CH;            // rows per pass of the warp
        const int c = lane % CH, sub = lane / CH;
        const int bytes = min(max(p.d * ES - c * 16, 0), 16);
        const uint32_t dst = ring_addr + (i % S) * SB;
        auto copy = [&](int row, bool live, const char *k, const char *v) {
          const uint32_t at = dst + row * (CH * 16) + swizzled(row, c) * 16;
          cp_async16(at, live ? k : kb, live ? bytes : 0);
          cp_async16(at + SB / 2, live ? v : vb, live ? bytes : 0);
        };
        if (one_page) {
          const int slot = (first & (p.page - 1)) + sub;
          const char *k = kb + ((int64_t)id * p.k_sp + slot * p.k_ss) * ES + c * 16, *v = vb + ((int64_t)id * p.v_sp + slot * p.v_ss) * ES + c * 16;
          const int64_t k_step = p.k_ss * (RP * ES), v_step = p.v_ss * (RP * ES);
          if (id >= 0 && first >= k_begin && first + kKeys <= k_end && p.d == DP) {      // (all of the warp)
#pragma unroll
            for (int j = 0; j < kKeys / RP; ++j) {
              const int row = j * RP + sub;
              const uint32_t at = dst + row * (CH * 16) + swizzled(row, c) * 16;
              cp_async16(at, k), cp_async16(at + SB / 2, v);
              k += k_step, v += v_step;
            }
          } else {
            const bool any = id >= 0 && bytes > 0;
#pragma unroll
            for (int j = 0; j < kKeys / RP; ++j) {
              const int row = j * RP + sub;
              copy(row, any && first + row >= k_begin && first + row < k_end, k, v);
              k += k_step, v += v_step;
            }
          }
        } else {
          const int key = first + (lane & 15), slot = key - page_of(p, key) * p.page;
#pragma unroll
          for (int j = 0; j < kKeys / RP; ++j) {
            const int row = j * RP + sub;
            const int rid = __shfl_sync(0xffffffffu, id, row), rslot = __shfl_sync(0xffffffffu, slot, row);
            copy(row, rid >= 0 && bytes > 0, kb + (rid * p.k_sp + rslot * p.k_ss) * ES + c * 16, vb + (rid * p.v_sp + rslot * p.v_ss) * ES + c * 16);
          }
        }
      }
      cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < S - 1; ++i) issue(i);

    float mul[MT][2];
    const float head_scale = p.scale_log2 * (E4M3 ? fabsf(p.k_scale[head]) : 1.f);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
      for (int half = 0; half < HALVES; ++half) {
        mul[m][half] = head_scale;
        if constexpr (E4M3) {
          float top = 0.f;
#pragma unroll
          for (int s = 0; s < KS; ++s) {
#pragma unroll
            for (int part = 0; part < 2; ++part) {
              const float2 f = unpack2(qf[m][s][HALVES * part + half], T(0.f));
              top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
            }
          }
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          const int ex = row_exponent(top);
          const float down = copysignf(ldexpf(1.f, -ex), p.k_scale[head]);
          mul[m][half] = score_factor(head_scale * ldexpf(1.f, ex));
#pragma unroll
          for (int s = 0; s < KS; ++s) {
#pragma unroll
            for (int part = 0; part < 2; ++part) {
              const float2 f = unpack2(qf[m][s][HALVES * part + half], T(0.f));
              qf[m][s][HALVES * part + half] = pack2(f.x * down, f.y * down, M(0.f));
            }
          }
        }
      }
    }

    if constexpr (NARROW) {      // from the row of this lane's query fragment to the rows of its scores
      const float mine = mul[0][0];
#pragma unroll
      for (int half = 0; half < 2; ++half) mul[0][half] = __shfl_sync(0xffffffffu, mine, (2 * t4 + half) * 4);
    }
    if constexpr (E4M3) {        // (minus infinity times a scale of NaN, in a row that sees no key)
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int half = 0; half < 2; ++half)
          if (hi[m][half] <= lo[m][half]) mul[m][half] = 1.f;
    }

    // ---- one pass over the keys -------------------------------------------------------------------------------
    // What lane (g, t) holds of the sums: rows g and g + 8 of the item, columns 8n + 2t, + 1 (o[n][2 * half + e]).  NARROW: rows
    // 2t and 2t + 1, columns 16n + g and + 8 (o[n][2 * which + half]).  (e4m3: see column() below.)
    constexpr int OT = NARROW ? NT / 2 : NT;
    float o[MT][OT][4], top[MT][2], sum[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
      for (int n = 0; n < OT; ++n) o[m][n][0] = o[m][n][1] = o[m][n][2] = o[m][n][3] = 0.f;
      top[m][0] = top[m][1] = -INFINITY;
      sum[m][0] = sum[m][1] = 0.f;
    }
    for (int i = 0; i < n_units; ++i) {
      issue(i + S - 1);
      cp_async_wait<S - 1>();
      __syncwarp();
      const uint32_t ks = ring_addr + (i % S) * SB, vs = ks + SB / 2;
      // scores
      float sc[MT][2][4];
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < 2; ++n) sc[m][n][0] = sc[m][n][1] = sc[m][n][2] = sc[m][n][3] = 0.f;
      auto frag_addr = [&](uint32_t base, int row, int c) {
        return base + row * (CH * 16) + swizzled(row, c) * 16;
      };
      if constexpr (NARROW) {      // keys are the rows of the product; even and odd steps are added apart
        if constexpr (!E4M3) {
#pragma unroll
          for (int s = 0; s < KS; ++s) {
            uint32_t kf[4];   // the step's first half: keys 0-7, keys 8-15; its second
            ldmatrix4(kf, frag_addr(ks, lane & 15, 2 * s + (lane >> 4)));
            mma16816(sc[0][s & 1], kf, qf[0][s][0], qf[0][s][1], M(0.f));
          }
        } else {
#pragma unroll
          for (int s = 0; s < KS; s += 2) {
            uint32_t kf[4];   // step s: keys 0-7, keys 8-15; step s + 1: the same
            ldmatrix4(kf, frag_addr(ks, lane & 15, s + (lane >> 4)));
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint2 x = e4m3x4_to_f16x4(kf[2 * h]), y = e4m3x4_to_f16x4(kf[2 * h + 1]);
              const uint32_t a[4] = {x.x, y.x, x.y, y.y};
              mma16816(sc[0][h], a, qf[0][s + h][0], qf[0][s + h][1], M(0.f));
            }
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[0][0][e] += sc[0][1][e];
      } else if constexpr (!E4M3) {
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          uint32_t kf[4];   // keys 0-7: both halves of the step, keys 8-15: both halves
          ldmatrix4(kf, frag_addr(ks, (lane & 7) + ((lane >> 4) << 3), 2 * s + ((lane >> 3) & 1)));
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            mma16816(sc[m][0], qf[m][s], kf[0], kf[1], M(0.f));
            mma16816(sc[m][1], qf[m][s], kf[2], kf[3], M(0.f));
          }
        }
      } else {
#pragma unroll
        for (int s = 0; s < KS; s += 2) {
          uint32_t kf[4];   // step s: keys 0-7, keys 8-15; step s + 1: the same
          ldmatrix4(kf, frag_addr(ks, (lane & 7) + (((lane >> 3) & 1) << 3), s + (lane >> 4)));
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint2 x = e4m3x4_to_f16x4(kf[2 * h]), y = e4m3x4_to_f16x4(kf[2 * h + 1]);
#pragma unroll
            for (int m = 0; m < MT; ++m) {
              mma16816(sc[m][0], qf[m][s + h], x.x, x.y, M(0.f));
              mma16816(sc[m][1], qf[m][s + h], y.x, y.y, M(0.f));
            }
          }
        }
      }
      // masks, running maximum, probabilities
      const int kbase = key0 + i * kUnit;
      const bool inside = kbase >= all_lo && kbase + kKeys <= all_hi && kbase >= k_begin && kbase + kKeys <= k_end;
      uint32_t pf[MT][4];
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        // scores of this lane's row `half`: columns 2t, 2t + 1 of both tiles of keys; NARROW: keys g and g + 8
        constexpr int PER = NARROW ? 2 : 4;
        auto score = [&](int half, int e) -> float & { return NARROW ? sc[m][0][2 * e + half] : sc[m][e >> 1][2 * half + (e & 1)]; };
        float mx[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          if (!inside) {
#pragma unroll
            for (int e = 0; e < PER; ++e) {
              const int key = kbase + (NARROW ? 8 * e + g : (e >> 1) * 8 + 2 * t4 + (e & 1));
              if (key < max(lo[m][half], k_begin) || key >= min(hi[m][half], k_end)) score(half, e) = -INFINITY;
            }
          }
          mx[half] = fmaxf(score(half, 0), score(half, 1));
          if constexpr (!NARROW) mx[half] = fmaxf(mx[half], fmaxf(score(half, 2), score(half, 3)));
          mx[half] = scaled_maximum<M>(mx[half], mul[m][half]);
        }
        // the reference of the exponents follows the maximum only when it has fallen far behind
        if (__any_sync(0xffffffffu, far_ahead<M>(mx[0], top[m][0]) || far_ahead<M>(mx[1], top[m][1]))) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            for (int v = NARROW ? 4 : 1; v < (NARROW ? 32 : 4); v *= 2) mx[half] = fmaxf(mx[half], __shfl_xor_sync(0xffffffffu, mx[half], v));
            const float to = fmaxf(top[m][half], mx[half] - kHeadroom<M>);
            const float f = top[m][half] == -INFINITY ? 0.f : exp2_fast(top[m][half] - to);
            sum[m][half] *= f;
#pragma unroll
            for (int n = 0; n < OT; ++n)
#pragma unroll
              for (int e = 0; e < 2; ++e) o[m][n][NARROW ? 2 * e + half : 2 * half + e] *= f;
            top[m][half] = to;
          }
        }
        float x[2][4];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const float neg = top[m][half] == -INFINITY ? 0.f : -top[m][half];
#pragma unroll
          for (int e = 0; e < PER; ++e) {
            x[half][e] = exp2_fast(fmaf(score(half, e), mul[m][half], neg));
            sum[m][half] += x[half][e];
          }
        }
        if constexpr (NARROW) {    // [key][row] to [row][key]
          pf[m][0] = transposed8x8(pack2(x[0][0], x[1][0], M(0.f)));
          pf[m][1] = transposed8x8(pack2(x[0][1], x[1][1], M(0.f)));
        } else {
#pragma unroll
          for (int half = 0; half < 2; ++half)
            pf[m][half] = pack2(x[half][0], x[half][1], M(0.f)), pf[m][2 + half] = pack2(x[half][2], x[half][3], M(0.f));
        }
      }
      if (!inside && tok0 != tok1) {     // rows that see different keys: values that are not finite apart
        auto bad = [&](uint32_t w) { return E4M3 ? not_finite_mask_e4m3(w) : not_finite_mask(w, M(0.f)); };
        constexpr int PER_LANE = kKeys * CH / 32;
        uint32_t any = 0;
#pragma unroll
        for (int q = 0; q < PER_LANE; ++q) {
          const uint4 x = ld_shared16(vs + (q * 32 + lane) * 16);
          any |= bad(x.x) | bad(x.y) | bad(x.z) | bad(x.w);
        }
        if (__any_sync(0xffffffffu, any != 0)) {
#pragma unroll 1
          for (int r = 0; r < kKeys; ++r) {
            const int key = kbase + r;
#pragma unroll
            for (int n = 0; n < OT; ++n) {       // this lane's two columns of tile n
              float2 f;
              if constexpr (NARROW) {
                const uint32_t w = E4M3 ? ld_shared2(frag_addr(vs, r, n) + g * 2)
                                        : ld_shared2(frag_addr(vs, r, 2 * n) + g * 2) | ld_shared2(frag_addr(vs, r, 2 * n + 1) + g * 2) << 16;
                const uint32_t x = w & bad(w);
                if constexpr (E4M3) f = unpack2(e4m3x4_to_f16x4(x).x, M(0.f));
                else f = unpack2(x, M(0.f));
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                  if (key < max(lo[0][half], k_begin) || key >= min(hi[0][half], k_end)) continue;
                  o[0][n][half] += f.x, o[0][n][2 + half] += f.y;
                }
                continue;
              }
              const uint32_t w = ld_shared4(frag_addr(vs, r, E4M3 ? n / 2 : n) + t4 * 4), x = w & bad(w);
              if constexpr (E4M3) {
                const uint2 h = e4m3x4_to_f16x4(__byte_perm(x, 0, 0x3120));
                f = unpack2(n & 1 ? h.y : h.x, M(0.f));
              } else {
                f = unpack2(x, M(0.f));
              }
#pragma unroll
              for (int m = 0; m < MT; ++m) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                  if (key < max(lo[m][half], k_begin) || key >= min(hi[m][half], k_end)) continue;
                  o[m][n][2 * half] += f.x, o[m][n][2 * half + 1] += f.y;
                }
              }
            }
          }
          __syncwarp();
#pragma unroll
          for (int q = 0; q < PER_LANE; ++q) {
            const uint32_t at = vs + (q * 32 + lane) * 16;
            const uint4 x = ld_shared16(at);
            st_shared16(at, x.x & ~bad(x.x), x.y & ~bad(x.y), x.z & ~bad(x.z), x.w & ~bad(x.w));
          }
          __syncwarp();
        }
      }
      // output rows
      if constexpr (NARROW) {      // columns are the rows of the product
        if constexpr (!E4M3) {
#pragma unroll
          for (int n = 0; n < OT; ++n) {
            uint32_t vf[4];   // keys 0-7: columns 16n.., the next eight; keys 8-15
            ldmatrix4_trans(vf, frag_addr(vs, (lane & 7) + ((lane >> 4) << 3), 2 * n + ((lane >> 3) & 1)));
            mma16816(o[0][n], vf, pf[0][0], pf[0][1], M(0.f));
          }
        } else {
#pragma unroll
          for (int n = 0; n < OT; n += 2) {
            uint32_t vf[4];   // chunk n: keys 0-7, 8-15; the next chunk.  A transposed unit is two neighbours of one key.
            ldmatrix4_trans(vf, frag_addr(vs, lane & 15, n + (lane >> 4)));
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint2 x = e4m3x4_to_f16x4(__byte_perm(vf[2 * h], 0, 0x3120)), y = e4m3x4_to_f16x4(__byte_perm(vf[2 * h + 1], 0, 0x3120));
              const uint32_t a[4] = {x.x, x.y, y.x, y.y};      // the even columns of the chunk, the odd ones
              mma16816(o[0][n + h], a, pf[0][0], pf[0][1], M(0.f));
            }
          }
        }
      } else if constexpr (!E4M3) {
#pragma unroll
        for (int n = 0; n < NT; n += 2) {
          uint32_t vf[4];   // columns 8n..: keys 0-7, 8-15; the next eight columns: the same
          ldmatrix4_trans(vf, frag_addr(vs, (lane & 7) + (((lane >> 3) & 1) << 3), n + (lane >> 4)));
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            mma16816(o[m][n], pf[m], vf[0], vf[1], M(0.f));
            mma16816(o[m][n + 1], pf[m], vf[2], vf[3], M(0.f));
          }
        }
      } else {
#pragma unroll
        for (int n = 0; n < NT; n += 4) {
          uint32_t vf[4];   // chunk n/2: keys 0-7, 8-15; the next chunk.  A transposed unit is two neighbours of one key.
          ldmatrix4_trans(vf, frag_addr(vs, (lane & 7) + (((lane >> 3) & 1) << 3), n / 2 + (lane >> 4)));
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            // the even and the odd columns of the chunk
            const uint2 x = e4m3x4_to_f16x4(__byte_perm(vf[2 * h], 0, 0x3120)), y = e4m3x4_to_f16x4(__byte_perm(vf[2 * h + 1], 0, 0x3120));
#pragma unroll
            for (int m = 0; m < MT; ++m) {
              mma16816(o[m][n + 2 * h], pf[m], x.x, y.x, M(0.f));
              mma16816(o[m][n + 2 * h + 1], pf[m], x.y, y.y, M(0.f));
            }
          }
        }
      }
      __syncwarp();   // the stage is read before the next copies overwrite it
    }
    cp_async_wait<0>();
    __syncthreads();   // the merge overlays the rings

    // ---- the four warps' rows added ----------------------------------------------------------------------------
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int v = NARROW ? 4 : 1; v < (NARROW ? 32 : 4); v *= 2) sum[m][half] += __shfl_xor_sync(0xffffffffu, sum[m][half], v);
        if (sum[m][half] != sum[m][half]) top[m][half] = INFINITY;   // a NaN outweighs the other warps' rows
        if (NARROW ? g == 0 : t4 == 0) merge_ml[warp * R + (NARROW ? 2 * t4 + half : m * 16 + half * 8 + g)] = make_float2(top[m][half], sum[m][half]);
      }
    }
    __syncthreads();
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int row = NARROW ? 2 * t4 + half : m * 16 + half * 8 + g;
        float best = -INFINITY;
#pragma unroll
        for (int v = 0; v < kWarps; ++v) best = fmaxf(best, merge_ml[v * R + row].x);
        const float f = top[m][half] == -INFINITY ? 0.f : exp2_fast(top[m][half] - best);
        float *dst = merge_o + (warp * R + row) * (DP + 8);
        if constexpr (NARROW) {
#pragma unroll
          for (int n = 0; n < OT; ++n) {
            if constexpr (E4M3) *reinterpret_cast<float2 *>(dst + 16 * n + 2 * g) = make_float2(o[m][n][half] * f, o[m][n][2 + half] * f);
            else dst[16 * n + g] = o[m][n][half] * f, dst[16 * n + 8 + g] = o[m][n][2 + half] * f;
          }
        } else if constexpr (!E4M3) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
            *reinterpret_cast<float2 *>(dst + 8 * n + 2 * t4) = make_float2(o[m][n][2 * half] * f, o[m][n][2 * half + 1] * f);
        } else {
#pragma unroll
          for (int n = 0; n < NT; n += 2)
            *reinterpret_cast<float4 *>(dst + 8 * n + 4 * t4) =
                make_float4(o[m][n][2 * half] * f, o[m][n + 1][2 * half] * f, o[m][n][2 * half + 1] * f, o[m][n + 1][2 * half + 1] * f);
        }
      }
    }
    __syncthreads();
    const float v_scale = E4M3 ? p.v_scale[head] : 1.f;
    auto write_row = [&](int row, int c, float4 acc, float f) {
      const int tok = it.token(p, row), qh = it.q_head(p, row);
      char *dst = reinterpret_cast<char *>(p.out) + ((seq.q0 + tok) * p.o_st + qh * p.o_sh + c) * 2;
      *reinterpret_cast<uint2 *>(dst) = make_uint2(pack2(acc.x * f, acc.y * f, T(0.f)), pack2(acc.z * f, acc.w * f, T(0.f)));
    };
    for (int idx = threadIdx.x; idx < n_rows * (DP / 4); idx += kThreads) {
      const int row = idx / (DP / 4), c = (idx % (DP / 4)) * 4;
      float best = -INFINITY, l = 0.f;
#pragma unroll
      for (int v = 0; v < kWarps; ++v) best = fmaxf(best, merge_ml[v * R + row].x);
#pragma unroll
      for (int v = 0; v < kWarps; ++v) {
        const float2 ml = merge_ml[v * R + row];
        l += ml.x == -INFINITY ? 0.f : ml.y * exp2_fast(ml.x - best);
      }
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int v = 0; v < kWarps; ++v) {
        const float4 x = *reinterpret_cast<const float4 *>(merge_o + (v * R + row) * (DP + 8) + c);
        acc.x += x.x, acc.y += x.y, acc.z += x.z, acc.w += x.w;
      }
      bool whole;
      if constexpr (DIRECT) whole = p.slices == 1;
      else whole = it.whole;
      if (whole) {
        if (c < p.d) write_row(row, c, acc, best == -INFINITY ? 0.f : v_scale / l);
      } else if constexpr (DIRECT) {
        *reinterpret_cast<float4 *>(slice_o + row * DP + c) = acc;
        if (c == 0) slice_ml[row] = make_float2(best, l);
      } else {
        const int slot = 2 * blockIdx.x + (it.first_piece ? 1 : 0);
        *reinterpret_cast<float4 *>(p.part_o + ((int64_t)slot * R + row) * DP + c) =
            make_float4(acc.x * v_scale, acc.y * v_scale, acc.z * v_scale, acc.w * v_scale);
        if (c == 0) p.part_ml[(int64_t)slot * R + row] = make_float2(best, l);
      }
    }
    if constexpr (DIRECT) {
      if (p.slices > 1) {          // each CTA of the cluster finishes a share of the rows
        tc::cluster_sync();
        const uint32_t o_at = smem_u32(slice_o), ml_at = smem_u32(slice_ml);
        for (int idx = (blockIdx.x % p.slices) * kThreads + threadIdx.x; idx < n_rows * (DP / 4); idx += p.slices * kThreads) {
          const int row = idx / (DP / 4), c = (idx % (DP / 4)) * 4;
          float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
          float best = -INFINITY, l = 0.f;
          for (int r = 0; r < p.slices; ++r) {
            const float top = tc::load_cluster_f32(tc::map_to_rank(ml_at + row * 8, r)), part = tc::load_cluster_f32(tc::map_to_rank(ml_at + row * 8 + 4, r));
            const float4 x = ld_cluster16(tc::map_to_rank(o_at + (row * DP + c) * 4, r));
            const float to = fmaxf(best, top), f_old = best == -INFINITY ? 0.f : exp2_fast(best - to), f = top == -INFINITY ? 0.f : exp2_fast(top - to);
            best = to, l = l * f_old + part * f;
            acc.x = acc.x * f_old + x.x * f, acc.y = acc.y * f_old + x.y * f, acc.z = acc.z * f_old + x.z * f, acc.w = acc.w * f_old + x.w * f;
          }
          if (c < p.d) write_row(row, c, acc, best == -INFINITY ? 0.f : v_scale / l);
        }
        tc::cluster_sync();        // the other CTAs have read this one's rows
      }
    } else if (threadIdx.x == 0 && !it.whole && it.first_piece) {
      p.meta[blockIdx.x].cut = it.cut();
    }
    __syncthreads();   // the merge area is read before the next rings fill it
  };

  if constexpr (DIRECT) {
    DirectPiece it;
    const int item = blockIdx.x / p.slices, slice = blockIdx.x % p.slices;
    it.b = item / p.hkv, it.head = item % p.hkv;
    if (it.head == 0 && slice == 0 && threadIdx.x == 0 && !lengths_fit(p, it.b)) tc::report_timeout(p.status, kStatusBadIndex);
    it.seq = load_seq(p, it.b);
    const int tiles = row_tiles<R>(p, it.seq);
    for (int tile = 0; tile < tiles; ++tile) {
      const TileUnits u = tile_units<R, kUnit>(p, it.seq, tile);
      const int from = u.count * slice / p.slices, to = u.count * (slice + 1) / p.slices;
      it.unit0 = u.first + from, it.n_units = to - from;
      it.r0 = tile * R, it.n_rows = min(it.seq.n * p.group - it.r0, R);
      work(it);
    }
  } else {
    const AttnRange range = attention_range<R, kUnit, kExtra, kThreads>(p, reinterpret_cast<int *>(smem), s_scan);
    if (threadIdx.x == 0) p.meta[blockIdx.x].cut.x = -1;
    AttnWalk<R, kUnit, kExtra> it(range);
    while (it.next(p)) work(it);
    // Not before the end: blocks of the joining kernel that wait beside these CTAs, and of the next call behind them, cost 64 sequences of
    // 500 - 8000 keys (e4m3) 143 us instead of 114.
    grid_launch_dependents();
  }
}

template <typename T, bool E4M3, int DP, int R, bool DIRECT>
int launch_mode(const AttnParams &p, dim3 grid, size_t prefix, cudaStream_t st) {
  constexpr int ring = ring_bytes<DP, E4M3, R>(), merge = merge_bytes<R, DP>();
  constexpr int fixed = ring > merge ? ring : merge;
  const size_t smem = prefix > fixed ? prefix : fixed;
  static PerDeviceOnce once;
  auto kern = attention_stream_kernel<T, E4M3, DP, R, DIRECT>;
  const int rc = allow_dynamic_smem(once, kern, 110 * 1024);
  if (rc != ZT_SUCCESS) return rc;
  if (!DIRECT || p.slices == 1) ZT_CUDA_OK(launch_overlapped(kern, grid, dim3(kThreads), smem, st, p));
  else ZT_CUDA_OK(launch_overlapped_cluster(kern, grid, dim3(kThreads), smem, st, dim3((unsigned)p.slices), p));
  return launch_status("attention_stream_kernel");
}
template <typename T, bool E4M3, int DP, int R>
int launch(const AttnParams &p, const AttnPlan &plan, cudaStream_t st) {
  // (the division of the batch comes before the first copy and has the shared memory to itself)
  if (plan.slices == 0) return launch_mode<T, E4M3, DP, R, false>(p, dim3(plan.grid), (size_t)(p.batch + 1) * 4, st);
  return launch_mode<T, E4M3, DP, R, true>(p, dim3((unsigned)(p.batch * p.hkv * plan.slices)), 0, st);
}
template <typename T, bool E4M3>
int launch_sized(const AttnParams &p, const AttnPlan &plan, cudaStream_t st) {
  const bool narrow = plan.dp == 64;
  if (plan.rows == 8) return narrow ? launch<T, E4M3, 64, 8>(p, plan, st) : launch<T, E4M3, 128, 8>(p, plan, st);
  if (plan.rows == 16) return narrow ? launch<T, E4M3, 64, 16>(p, plan, st) : launch<T, E4M3, 128, 16>(p, plan, st);
  return narrow ? launch<T, E4M3, 64, 32>(p, plan, st) : launch<T, E4M3, 128, 32>(p, plan, st);
}

}  // namespace

int attention_stream_grid(int rows) { return (rows <= 16 ? ctas_per_sm<16>() : ctas_per_sm<32>()) * sm_count(); }

int attention_stream_launch(const AttnParams &p, const AttnPlan &plan, int dtype, int cache_dtype, cudaStream_t st) {
  const bool e4m3 = cache_dtype == ZT_E4M3;
  if (dtype == ZT_BF16)
    return e4m3 ? launch_sized<__nv_bfloat16, true>(p, plan, st) : launch_sized<__nv_bfloat16, false>(p, plan, st);
  return e4m3 ? launch_sized<__half, true>(p, plan, st) : launch_sized<__half, false>(p, plan, st);
}

}  // namespace zt
