// Rotary positions of queries and keys, and the same with the rotated keys and the values stored in a paged cache.
//
// The first rot_dim elements of a head are pairs (a, b) -- (x[i], x[i + rot_dim/2]) or, interleaved, (x[2i], x[2i+1]) -- and pair
// i of a token at position p becomes (a cos - b sin, b cos + a sin) * factor with the angle p * inv_freq[i].  The rest of a head
// passes through.  inv_freq is fp32, positions are integers: the angle in turns is formed in fp64 (53 bits hold position times
// frequency exactly enough for positions up to 2^31), reduced to half a turn there, and only the remainder goes to fp32: a table
// in fp32 would be 0.06 radians off at position 10^6.  The angles of a token are computed once and shared by its heads.
//
// Bound by memory: every element is read once and written once.  A block takes up to eight tokens, as many as its 256 threads have
// angles to compute at once, and the first 16-byte loads are in flight meanwhile: with one token per block three quarters of the
// threads waited for the others' angles, and 8192 tokens of 64 heads took 69 us instead of 48 (5.5 TB/s).
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>

#include "tc05.cuh"

namespace zt {

namespace {

struct RopeParams {
  const char *q, *k, *v;
  char *q_out, *k_out, *k_cache, *v_cache;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh, qo_st, qo_sh, ko_st, ko_sh;   // strides in elements: token, head
  int64_t kc_sp, kc_ss, kc_sh, vc_sp, vc_ss, vc_sh;                         // cache strides: page, slot, head
  const void *positions, *slots;
  const float *inv_freq, *k_scale, *v_scale;
  int64_t capacity;   // slots of the cache
  int tokens, hq, hkv, d, rot, page, pos64, slot64, interleaved;
  int one_cache;      // keys and values have the same rows: only values are stored
  uint32_t magic_token, magic_rot, magic_rest, magic_whole;   // divisions by the items of a token, the vectors of a head's parts
  int block_tokens;
  float factor;
  int *status;
};

template <typename T>
__device__ __forceinline__ float to_f32(T v) {
  if constexpr (sizeof(T) == 4) return v;
  else if constexpr (__is_same(T, __half)) return __half2float(v);
  else return __bfloat162float(v);
}
template <typename T>
__device__ __forceinline__ T from_f32(float v) {
  if constexpr (sizeof(T) == 4) return v;
  else if constexpr (__is_same(T, __half)) return __float2half_rn(v);
  else return __float2bfloat16_rn(v);
}

__device__ __forceinline__ int64_t load_index(const void *p, int64_t i, int is64) {
  return is64 ? reinterpret_cast<const int64_t *>(p)[i] : (int64_t)reinterpret_cast<const int32_t *>(p)[i];
}

template <typename T, int VEC>
struct Pack {   // VEC elements; 16 bytes in the vector form
  T e[VEC];
};
template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> load_pack(const char *base, int64_t elem) {
  Pack<T, VEC> r;
  if constexpr (sizeof(r) == 16)
    *reinterpret_cast<uint4 *>(&r) = *reinterpret_cast<const uint4 *>(base + elem * (int64_t)sizeof(T));
  else
    r.e[0] = reinterpret_cast<const T *>(base)[elem];
  return r;
}
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3) |
         (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3) << 16;
}
// VEC values to `base`, as T or, divided by `scale` and saturated, as e4m3 (round to nearest even in both; a product with the rounded
// reciprocal would move ties, and there is none for scales below 2^-128).
template <typename T, int VEC, bool E4M3>
__device__ __forceinline__ void store_pack(char *base, int64_t elem, const float (&v)[VEC], float scale) {
  if constexpr (E4M3 && VEC == 1) {
    base[elem] = (char)__nv_cvt_float_to_fp8(__fdiv_rn(v[0], scale), __NV_SATFINITE, __NV_E4M3);
  } else if constexpr (E4M3) {
    uint32_t w[VEC / 4];
#pragma unroll
    for (int i = 0; i < VEC; i += 4)
      w[i / 4] = e4m3x4(__fdiv_rn(v[i], scale), __fdiv_rn(v[i + 1], scale), __fdiv_rn(v[i + 2], scale), __fdiv_rn(v[i + 3], scale));
    if constexpr (VEC == 8) *reinterpret_cast<uint2 *>(base + elem) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t *>(base + elem) = w[0];
  } else {
    Pack<T, VEC> r;
#pragma unroll
    for (int i = 0; i < VEC; ++i) r.e[i] = from_f32<T>(v[i]);
    if constexpr (sizeof(r) == 16)
      *reinterpret_cast<uint4 *>(base + elem * (int64_t)sizeof(T)) = *reinterpret_cast<const uint4 *>(&r);
    else
      reinterpret_cast<T *>(base)[elem] = r.e[0];
  }
}

constexpr int kRopeThreads = 256;
constexpr int kMaxHalf = 128;       // rotated pairs per head
constexpr int kMaxTokens = 8;       // of a block

// n / d for n d < 2^32, by a multiplication with `magic` = ceil(2^32 / d) (0 for d = 1).
__device__ __forceinline__ int quotient(int n, uint32_t magic) { return magic ? (int)__umulhi((uint32_t)n, magic) : n; }
uint32_t magic_of(int d) { return d > 1 ? (uint32_t)(((1ull << 32) + d - 1) / d) : 0u; }

// An item is two vectors: the two sides of the pairs of a rotated head, or two of the part of a head that passes through or of a
// value (of an odd number of vectors the last item has one).  Heads are counted through: queries, keys, values; items through the block's tokens.
// Five blocks share an SM, four with the divisions of an e4m3 cache: 8192 tokens of 64 + 8 heads take 67 us so and 79 with
// five, whose 48 registers spill (66 with products instead).
template <typename T, int VEC, bool CACHE, bool E4M3>
__global__ void __launch_bounds__(kRopeThreads, E4M3 ? 4 : 5) rope_kernel(const __grid_constant__ RopeParams p) {
  __shared__ float2 s_turn[kMaxTokens * kMaxHalf];      // [token][element of a vector][vector]: neighbouring lanes, neighbouring words
  __shared__ int64_t s_row[kMaxTokens][2];              // a token's row in the caches
  grid_launch_dependents();
  grid_dependency_wait();
  const int token0 = blockIdx.x * p.block_tokens, tokens = min(p.block_tokens, p.tokens - token0), half = p.rot / 2;
  const int per_head = half / VEC, rest = (p.d - p.rot) / VEC, whole = p.d / VEC;     // vectors
  const int rest_items = (rest + 1) / 2, whole_items = (whole + 1) / 2;
  const int heads = p.hq + p.hkv;
  const int n_rot = heads * per_head, n_rest = n_rot + heads * rest_items, n_token = n_rest + (CACHE ? p.hkv * whole_items : 0);
  const int n = tokens * n_token;

  struct Item {
    Pack<T, VEC> x0, x1;
    int token, head;
    int vec0, vec1;       // the vectors of the head, vec1 < 0: there is none
    int turn;             // rotated: number of the pair's vector, else -1
  };
  Item item{};
  auto load = [&](int it, Item &i) {
    if (it >= n) return;
    i.token = quotient(it, p.magic_token);
    it -= i.token * n_token;
    i.turn = -1;
    if (it < n_rot) {
      i.head = quotient(it, p.magic_rot);
      i.turn = it - i.head * per_head;
      i.vec0 = p.interleaved ? 2 * i.turn : i.turn;
      i.vec1 = p.interleaved ? i.vec0 + 1 : i.vec0 + per_head;
    } else if (!CACHE || it < n_rest) {
      i.head = quotient(it - n_rot, p.magic_rest);
      i.vec0 = it - n_rot - i.head * rest_items;
      i.vec1 = i.vec0 + rest_items < rest ? i.vec0 + rest_items + 2 * per_head : -1;
      i.vec0 += 2 * per_head;
    } else {
      i.head = quotient(it - n_rest, p.magic_whole);
      i.vec0 = it - n_rest - i.head * whole_items;
      i.vec1 = i.vec0 + whole_items < whole ? i.vec0 + whole_items : -1;
      i.head += heads;
    }
    const int64_t token = token0 + i.token;
    const char *in;
    int64_t at;
    if (i.head < p.hq) in = p.q, at = token * p.q_st + i.head * p.q_sh;
    else if (!CACHE || i.head < heads) in = p.k, at = token * p.k_st + (i.head - p.hq) * p.k_sh;
    else in = p.v, at = token * p.v_st + (i.head - heads) * p.v_sh;
    i.x0 = load_pack<T, VEC>(in, at + i.vec0 * VEC);
    if (i.vec1 >= 0) i.x1 = load_pack<T, VEC>(in, at + i.vec1 * VEC);
  };

  load(threadIdx.x, item);      // in flight during the angles
  if (CACHE && threadIdx.x < tokens) {
    const int64_t slot = load_index(p.slots, token0 + threadIdx.x, p.slot64);
    int64_t kc = -1, vc = 0;
    if (slot >= 0 && slot < p.capacity) {
      const int64_t page = slot / p.page, row = slot - page * p.page;
      kc = page * p.kc_sp + row * p.kc_ss;
      vc = page * p.vc_sp + row * p.vc_ss;
    } else if (slot >= p.capacity) {
      tc::report_timeout(p.status, kStatusBadIndex);
    }
    s_row[threadIdx.x][0] = kc, s_row[threadIdx.x][1] = vc;
  }
  for (int i = threadIdx.x; i < tokens * half; i += kRopeThreads) {
    const int t = i / half, pair = i - t * half;
    const double pos = (double)load_index(p.positions, token0 + t, p.pos64);
    const double turns = pos * ((double)p.inv_freq[pair] * 0.15915494309189535);   // 1 / (2 pi)
    float s, c;
    sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
    s_turn[t * half + pair % VEC * per_head + pair / VEC] = make_float2(c * p.factor, s * p.factor);
  }
  __syncthreads();

  auto process = [&](const Item &i) {
    float a[VEC], b[VEC];
    if (i.turn >= 0) {
      float u[2 * VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) u[e] = to_f32<T>(i.x0.e[e]), u[VEC + e] = to_f32<T>(i.x1.e[e]);
      const float2 *turn = s_turn + i.token * half + i.turn;
      if (p.interleaved) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float2 t = turn[e * per_head];
          const float first = u[2 * e], second = u[2 * e + 1];
          u[2 * e] = first * t.x - second * t.y, u[2 * e + 1] = second * t.x + first * t.y;
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) a[e] = u[e], b[e] = u[VEC + e];
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float2 t = turn[e * per_head];
          a[e] = u[e] * t.x - u[VEC + e] * t.y, b[e] = u[VEC + e] * t.x + u[e] * t.y;
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) a[e] = to_f32<T>(i.x0.e[e]), b[e] = to_f32<T>(i.x1.e[e]);
    }
    const int e0 = i.vec0 * VEC, e1 = i.vec1 * VEC;
    const int64_t token = token0 + i.token;
    if (i.head < p.hq) {
      const int64_t o = token * p.qo_st + i.head * p.qo_sh;
      store_pack<T, VEC, false>(p.q_out, o + e0, a, 1.f);
      if (e1 >= 0) store_pack<T, VEC, false>(p.q_out, o + e1, b, 1.f);
    } else if constexpr (CACHE) {
      const bool value = i.head >= heads;
      const int64_t row = s_row[i.token][value];
      if (s_row[i.token][0] >= 0 && (value || !p.one_cache)) {
        const int h = i.head - (value ? heads : p.hq);
        const int64_t o = row + h * (value ? p.vc_sh : p.kc_sh);
        const float scale = E4M3 ? (value ? p.v_scale[h] : p.k_scale[h]) : 1.f;
        char *base = value ? p.v_cache : p.k_cache;
        store_pack<T, VEC, E4M3>(base, o + e0, a, scale);
        if (e1 >= 0) store_pack<T, VEC, E4M3>(base, o + e1, b, scale);
      }
    } else {
      const int64_t o = token * p.ko_st + (i.head - p.hq) * p.ko_sh;
      store_pack<T, VEC, false>(p.k_out, o + e0, a, 1.f);
      if (e1 >= 0) store_pack<T, VEC, false>(p.k_out, o + e1, b, 1.f);
    }
  };
  for (int it = threadIdx.x; it < n; it += kRopeThreads) {
    process(item);
    load(it + kRopeThreads, item);
  }
}

template <typename T, int VEC>
cudaError_t launch_rope(RopeParams p, int cache, cudaStream_t st) {   // cache: 0 none, 1 of the inputs' type, 2 e4m3
  const int rot = p.rot / 2 / VEC, rest = ((p.d - p.rot) / VEC + 1) / 2, whole = (p.d / VEC + 1) / 2;      // items of a head
  p.magic_rot = magic_of(rot), p.magic_rest = magic_of(rest), p.magic_whole = magic_of(whole);
  const int items = (p.hq + p.hkv) * (rot + rest) + (cache ? p.hkv * whole : 0);
  p.magic_token = magic_of(items);
  // As many tokens as give every thread an angle, or (tokens of few items) an item; fewer where that leaves SMs with few blocks, which
  // end unevenly: 8192 tokens of 64 heads, half rotated, 55.7 us in 1024 blocks of 8 tokens, 48.4 in 2048.  (Threads without an item
  // cost more: 8192 tokens of 3 heads of 64 take 5.8 us in blocks of 8 tokens, 7.8 in blocks of 4.)
  int by_angles = p.rot > 0 ? kRopeThreads / (p.rot / 2) : kMaxTokens, by_items = ceil_div(kRopeThreads, items);
  by_angles = std::min(by_angles, ceil_div(p.tokens, 16 * sm_count()));
  by_items = std::min(by_items, ceil_div(p.tokens, 2 * sm_count()));
  int t = std::max(by_angles, by_items);
  t = t < 1 ? 1 : t > kMaxTokens ? kMaxTokens : t;
  while (t > 1 && (int64_t)items * items * t >= (int64_t)1 << 32) --t;      // quotient() is exact up to there
  p.block_tokens = t;
  const dim3 grid((unsigned)ceil_div(p.tokens, p.block_tokens)), block(kRopeThreads);
  if (cache == 0) return launch_overlapped(rope_kernel<T, VEC, false, false>, grid, block, (size_t)0, st, p);
  if (cache == 1) return launch_overlapped(rope_kernel<T, VEC, true, false>, grid, block, (size_t)0, st, p);
  return launch_overlapped(rope_kernel<T, VEC, true, true>, grid, block, (size_t)0, st, p);
}

}  // namespace
}  // namespace zt

using namespace zt;

extern "C" int zt_rope(const zt_rope_args_t *a, void *stream) {
  ZT_REQUIRE(a != nullptr, ZT_INVALID_ARGUMENT, "zt_rope: null argument block");
  ZT_REQUIRE(a->tokens >= 0 && a->tokens <= (1 << 30), ZT_INVALID_ARGUMENT, "zt_rope: token count %lld out of range",
             (long long)a->tokens);
  ZT_REQUIRE(a->q_heads >= 0 && a->kv_heads >= 0 && a->q_heads <= 4096 && a->kv_heads <= 4096 && a->head_dim >= 1 &&
                 a->head_dim <= 2 * kMaxHalf,
             ZT_INVALID_ARGUMENT, "zt_rope: need up to 4096 heads of 1 to %d elements", 2 * kMaxHalf);
  ZT_REQUIRE(a->rot_dim >= 0 && a->rot_dim % 2 == 0 && a->rot_dim <= a->head_dim, ZT_INVALID_ARGUMENT,
             "zt_rope: the rotated part of a head (%d) must be even and at most the head (%d)", a->rot_dim, a->head_dim);
  ZT_REQUIRE(a->dtype == ZT_BF16 || a->dtype == ZT_F16 || a->dtype == ZT_F32, ZT_INVALID_ARGUMENT,
             "zt_rope: query and key must be bfloat16, float16 or float32");
  const bool cache = a->k_cache != nullptr || a->v_cache != nullptr;
  ZT_REQUIRE(!cache || a->cache_dtype == a->dtype || a->cache_dtype == ZT_E4M3, ZT_INVALID_ARGUMENT,
             "zt_rope: the cache must have the type of the key or be float8_e4m3");
  ZT_REQUIRE(!cache || a->page_size >= 1, ZT_INVALID_ARGUMENT, "zt_rope: the page size must be positive");
  ZT_REQUIRE(!cache || a->num_pages >= 0, ZT_INVALID_ARGUMENT, "zt_rope: negative page count");
  if (a->tokens == 0 || a->q_heads + a->kv_heads == 0) return ZT_SUCCESS;
  ZT_REQUIRE((a->q_heads == 0 || (a->q && a->q_out)) && (a->kv_heads == 0 || a->k) && a->positions &&
                 (a->rot_dim == 0 || a->inv_freq),
             ZT_INVALID_ARGUMENT, "zt_rope: null tensor pointer");
  ZT_REQUIRE(cache ? (a->k_cache && a->v_cache && a->v && a->slots) : (a->kv_heads == 0 || a->k_out != nullptr), ZT_INVALID_ARGUMENT,
             "zt_rope: null pointer among value, slots, caches or key output");
  const bool e4m3 = cache && a->cache_dtype == ZT_E4M3;
  ZT_REQUIRE(!e4m3 || (a->k_scale && a->v_scale), ZT_INVALID_ARGUMENT, "zt_rope: a float8_e4m3 cache needs k_scale and v_scale");
  int *status = device_status_ptr();
  ZT_REQUIRE(status != nullptr, ZT_CUDA_ERROR, "zt_rope: no device status word");

  RopeParams p{};
  p.q = (const char *)a->q, p.k = (const char *)a->k, p.v = (const char *)a->v;
  p.q_out = (char *)a->q_out, p.k_out = (char *)a->k_out, p.k_cache = (char *)a->k_cache, p.v_cache = (char *)a->v_cache;
  p.q_st = a->q_stride[0], p.q_sh = a->q_stride[1], p.k_st = a->k_stride[0], p.k_sh = a->k_stride[1];
  p.v_st = a->v_stride[0], p.v_sh = a->v_stride[1];
  p.qo_st = a->q_out_stride[0], p.qo_sh = a->q_out_stride[1], p.ko_st = a->k_out_stride[0], p.ko_sh = a->k_out_stride[1];
  p.kc_sp = a->k_cache_stride[0], p.kc_ss = a->k_cache_stride[1], p.kc_sh = a->k_cache_stride[2];
  p.vc_sp = a->v_cache_stride[0], p.vc_ss = a->v_cache_stride[1], p.vc_sh = a->v_cache_stride[2];
  p.positions = a->positions, p.slots = a->slots, p.inv_freq = a->inv_freq, p.k_scale = a->k_scale, p.v_scale = a->v_scale;
  p.capacity = cache ? a->num_pages * (int64_t)a->page_size : 0;
  p.tokens = (int)a->tokens, p.hq = a->q_heads, p.hkv = a->kv_heads, p.d = a->head_dim, p.rot = a->rot_dim;
  p.page = cache ? a->page_size : 1, p.pos64 = a->positions_64, p.slot64 = a->slots_64, p.interleaved = a->interleaved != 0;
  p.factor = a->attention_factor, p.status = status;
  p.one_cache = cache && a->k_cache == a->v_cache && std::equal(a->k_cache_stride, a->k_cache_stride + 3, a->v_cache_stride);

  // 16-byte vectors where every row and both parts of a head start on one; else element by element
  const int es = a->dtype == ZT_F32 ? 4 : 2, vec = 16 / es;
  uintptr_t bits = 0;
  int64_t strides = 0;
  auto row = [&](const void *ptr, const int64_t *s) { bits |= (uintptr_t)ptr, strides |= s[0] | s[1]; };
  if (a->q_heads) row(a->q, a->q_stride), row(a->q_out, a->q_out_stride);
  if (a->kv_heads) row(a->k, a->k_stride);
  if (a->kv_heads && !cache) row(a->k_out, a->k_out_stride);
  if (cache) {
    row(a->v, a->v_stride), row(a->k_cache, a->k_cache_stride), row(a->v_cache, a->v_cache_stride);
    strides |= a->k_cache_stride[2] | a->v_cache_stride[2];
  }
  // a rotated half and the rest of a head are whole vectors; strides are counted in vectors of the inputs' type, which is at
  // least as wide as the cache's (an e4m3 vector of the same elements has 8 or 4 bytes)
  const bool wide = (a->rot_dim / 2) % vec == 0 && a->head_dim % vec == 0 && strides % vec == 0 && bits % 16 == 0;
  const int form = !cache ? 0 : e4m3 ? 2 : 1;
  const int per = wide ? vec : 1, head_items = (a->rot_dim / 2 / per) + ((a->head_dim - a->rot_dim) / per + 1) / 2;
  ZT_REQUIRE((int64_t)(a->q_heads + a->kv_heads) * head_items + (cache ? (int64_t)a->kv_heads * ((a->head_dim / per + 1) / 2) : 0) < 65536,
             ZT_UNSUPPORTED, "zt_rope: %d heads of %d elements per token are too many", a->q_heads + a->kv_heads, a->head_dim);
  cudaStream_t st = (cudaStream_t)stream;
  cudaError_t e;
  if (a->dtype == ZT_BF16)
    e = wide ? launch_rope<__nv_bfloat16, 8>(p, form, st) : launch_rope<__nv_bfloat16, 1>(p, form, st);
  else if (a->dtype == ZT_F16)
    e = wide ? launch_rope<__half, 8>(p, form, st) : launch_rope<__half, 1>(p, form, st);
  else
    e = wide ? launch_rope<float, 4>(p, form, st) : launch_rope<float, 1>(p, form, st);
  ZT_CUDA_OK(e);
  return launch_status("rope_kernel");
}
