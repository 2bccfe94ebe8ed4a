// Rotary positions of queries and keys, and the same with the rotated keys and the values stored in a paged cache.
//
// The first rot_dim elements of a head are pairs (a, b) -- (x[i], x[i + rot_dim/2]) or, interleaved, (x[2i], x[2i+1]) -- and pair
// i of a token at position p becomes (a cos - b sin, b cos + a sin) * factor with the angle p * inv_freq[i].  The rest of a head
// passes through.  inv_freq is fp32, positions are integers: the angle in turns is formed in fp64 (53 bits hold position times
// frequency exactly enough for positions up to 2^31), reduced to half a turn there, and only the remainder goes to fp32: a table
// in fp32 would be 0.06 radians off at position 10^6.  The angles of a token are computed once and shared by its heads.
//
// Bound by memory: every element is read once and written once.  A block takes one token (several where a token has few
// vectors); its threads have their 16-byte loads in flight while the angles are computed.
#include <cuda_fp16.h>
#include <cuda_fp8.h>

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
// VEC values to `base`, as T or, divided by `scale` and saturated, as e4m3 (round to nearest even in both).
template <typename T, int VEC, bool E4M3>
__device__ __forceinline__ void store_pack(char *base, int64_t elem, const float (&v)[VEC], float scale) {
  if constexpr (E4M3) {
    uint8_t b[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) b[i] = __nv_cvt_float_to_fp8(__fdiv_rn(v[i], scale), __NV_SATFINITE, __NV_E4M3);
    if constexpr (VEC == 8) *reinterpret_cast<uint2 *>(base + elem) = *reinterpret_cast<const uint2 *>(b);
    else if constexpr (VEC == 4) *reinterpret_cast<uint32_t *>(base + elem) = *reinterpret_cast<const uint32_t *>(b);
    else base[elem] = (char)b[0];
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
constexpr int kMaxTokensPerBlock = 8;

// blockDim = (threads of a token, tokens of a block).  A work item is one pair of vectors of a rotated head, one vector of the
// part of a head that passes through, or one vector of a value.
template <typename T, int VEC, bool CACHE, bool E4M3>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const RopeParams p) {
  __shared__ float2 s_turn[kMaxTokensPerBlock][kMaxHalf];
  grid_launch_dependents();
  grid_dependency_wait();
  const int token = blockIdx.x * blockDim.y + threadIdx.y, half = p.rot / 2;
  const bool live = token < p.tokens;
  const int per_head = half / VEC, rest = (p.d - p.rot) / VEC, whole = p.d / VEC;
  const int heads = p.hq + p.hkv;
  const int n_rot = heads * per_head, n_rest = heads * rest, n = live ? n_rot + n_rest + (CACHE ? p.hkv * whole : 0) : 0;

  // where the vectors of item `it` are: input, their distance, and (head, first element)
  auto locate = [&](int it, const char *&in, int64_t &at, int &gap, int &head, int &elem) {
    if (it < n_rot) {
      head = it / per_head;
      const int j = it - head * per_head;
      elem = p.interleaved ? 2 * j * VEC : j * VEC;
      gap = p.interleaved ? VEC : half;
    } else if (it < n_rot + n_rest) {
      head = (it - n_rot) / rest;
      elem = p.rot + (it - n_rot - head * rest) * VEC;
      gap = 0;
    } else {
      const int r = it - n_rot - n_rest;
      head = r / whole;
      elem = (r - head * whole) * VEC;
      gap = 0;
      in = p.v;
      at = token * p.v_st + head * p.v_sh + elem;
      head += heads;                        // heads of the values come behind those of the keys
      return;
    }
    if (head < p.hq) in = p.q, at = token * p.q_st + head * p.q_sh + elem;
    else in = p.k, at = token * p.k_st + (head - p.hq) * p.k_sh + elem;
  };

  // first item's loads before the angles, so that they are in flight meanwhile
  const char *in = nullptr;
  int64_t at = 0;
  int gap = 0, head = 0, elem = 0;
  Pack<T, VEC> x0{}, x1{};
  int it = threadIdx.x;
  if (it < n) {
    locate(it, in, at, gap, head, elem);
    x0 = load_pack<T, VEC>(in, at);
    if (gap) x1 = load_pack<T, VEC>(in, at + gap);
  }
  int64_t kc = -1, vc = 0;
  if (live) {
    const int64_t pos = load_index(p.positions, token, p.pos64);
    if constexpr (CACHE) {
      const int64_t slot = load_index(p.slots, token, p.slot64);
      if (slot >= 0 && slot < p.capacity) {
        const int64_t page = slot / p.page, row = slot - page * p.page;
        kc = page * p.kc_sp + row * p.kc_ss;
        vc = page * p.vc_sp + row * p.vc_ss;
      } else if (slot >= p.capacity && threadIdx.x == 0) {
        tc::report_timeout(p.status, kStatusBadIndex);
      }
    }
    for (int i = threadIdx.x; i < half; i += blockDim.x) {
      const double turns = (double)pos * ((double)p.inv_freq[i] * 0.15915494309189535);   // 1 / (2 pi)
      float s, c;
      sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
      s_turn[threadIdx.y][i] = make_float2(c * p.factor, s * p.factor);
    }
  }
  __syncthreads();
  while (it < n) {
    const int next = it + blockDim.x;
    float a[VEC], b[VEC];
    const bool rotated = gap != 0;
    if (rotated) {
      float u[2 * VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) u[i] = to_f32<T>(x0.e[i]), u[VEC + i] = to_f32<T>(x1.e[i]);
      const int pair = p.interleaved ? elem / 2 : elem;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float2 t = s_turn[threadIdx.y][pair + i];
        const float first = p.interleaved ? u[2 * i] : u[i], second = p.interleaved ? u[2 * i + 1] : u[VEC + i];
        a[i] = first * t.x - second * t.y;
        b[i] = second * t.x + first * t.y;
      }
      if (p.interleaved) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) u[2 * i] = a[i], u[2 * i + 1] = b[i];
#pragma unroll
        for (int i = 0; i < VEC; ++i) a[i] = u[i], b[i] = u[VEC + i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) a[i] = to_f32<T>(x0.e[i]);
    }
    const int this_head = head, this_elem = elem, this_gap = gap;
    if (next < n) {
      locate(next, in, at, gap, head, elem);
      x0 = load_pack<T, VEC>(in, at);
      if (gap) x1 = load_pack<T, VEC>(in, at + gap);
    }
    if (this_head < p.hq) {
      const int64_t o = token * p.qo_st + this_head * p.qo_sh + this_elem;
      store_pack<T, VEC, false>(p.q_out, o, a, 1.f);
      if (rotated) store_pack<T, VEC, false>(p.q_out, o + this_gap, b, 1.f);
    } else if constexpr (CACHE) {
      if (kc >= 0) {
        const int h = this_head < heads ? this_head - p.hq : this_head - heads;
        const bool value = this_head >= heads;
        const int64_t o = (value ? vc + h * p.vc_sh : kc + h * p.kc_sh) + this_elem;
        const float scale = E4M3 ? (value ? p.v_scale[h] : p.k_scale[h]) : 1.f;
        char *base = value ? p.v_cache : p.k_cache;
        store_pack<T, VEC, E4M3>(base, o, a, scale);
        if (rotated) store_pack<T, VEC, E4M3>(base, o + this_gap, b, scale);
      }
    } else {
      const int64_t o = token * p.ko_st + (this_head - p.hq) * p.ko_sh + this_elem;
      store_pack<T, VEC, false>(p.k_out, o, a, 1.f);
      if (rotated) store_pack<T, VEC, false>(p.k_out, o + this_gap, b, 1.f);
    }
    it = next;
  }
}

template <typename T, int VEC>
cudaError_t launch_rope(const RopeParams &p, int cache, cudaStream_t st) {   // cache: 0 none, 1 of the inputs' type, 2 e4m3
  const int items = (p.hq + p.hkv) * (p.rot / 2 / VEC + (p.d - p.rot) / VEC) + (cache ? p.hkv * (p.d / VEC) : 0);
  int tx = 32;
  while (tx < kRopeThreads && tx < items) tx *= 2;
  const int ty = kRopeThreads / tx;
  const dim3 grid((unsigned)ceil_div(p.tokens, ty)), block(tx, ty);
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
