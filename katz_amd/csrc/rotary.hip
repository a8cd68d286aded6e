// K14: rotary positions with several axes, on rows of q and k, or with the turned keys and the values written into the pages of a cache:
//   angle(r, j) = position[r][axis of j] * frequency[j],   (a, b) -> (a cos - b sin, b cos + a sin)   for every pair j of every head
//
// The angle is a number of whole turns and a rest; a position of 10^6 in 32 bits would leave the rest 0.06 off.  So the turns are counted in 64 bits
// (position * frequency / 2 pi less the nearest integer) and only the rest goes to 32 (off by 2^-25 turns), where sine and cosine are taken of a
// multiple of pi.  The products with the rows are in 32 bits and rounded once.
//
// Bound by memory: every element is read and written once.  A workgroup takes some rows, works their angles out once for all heads (LDS), then its
// threads go over the rows in pieces of eight elements of either half (or eight in a row), 16 bytes a load.
#include "paged_cache.h"

namespace {

struct RotaryParams {
  const void *q, *k, *v;
  void *q_out, *k_out, *v_out;   // k_out, v_out: the layer's pages where a cache is given
  const void *positions, *frequencies;
  const int32_t *table, *lengths, *slots, *places;
  const float *k_scale, *v_scale;
  long rows, ldq, ldk, ldv, ldqo, ldko;
  long k_page, k_token, k_head, v_page, v_token, v_head;
  int heads, kv_heads, d, pairs, axes, end[4];
  int position_type, frequency_32, fill, per;   // per: rows of a workgroup
  int cached, n_slots, width, pages, page;
};

constexpr int NT = 256;
constexpr double ONE_TURN = 0.15915494309189533577;   // 1 / 2 pi

// Where a row of k and v goes: its page (-1: nowhere), the place in it, and the place in the sequence (-1: the row is left out).
struct Where { int page, at, place; };

__device__ __forceinline__ Where where(const RotaryParams& p, long r) {
  Where w{-1, 0, -1};
  const long s = p.slots ? p.slots[r] : r;
  if (s < 0 || s >= p.n_slots) return w;
  int n = p.lengths[s];
  n = n < p.width * p.page ? n : p.width * p.page;
  const int t = p.places ? p.places[r] : n - 1;
  if (t < 0 || t >= n) return w;
  w.place = t;
  w.at = t % p.page;
  const int e = p.table[s * p.width + t / p.page];
  w.page = e >= 0 && e < p.pages ? e : -1;
  return w;
}

template <typename T, int N>
__device__ __forceinline__ void load(const T* from, float (&f)[N]) {
  T v[N];
  if constexpr (N == 8) __builtin_memcpy(v, __builtin_assume_aligned(from, 16), sizeof(v));
  else v[0] = from[0];
#pragma unroll
  for (int e = 0; e < N; ++e) f[e] = (float)v[e];
}
template <typename T, int N>
__device__ __forceinline__ void store(T* to, const float (&f)[N]) {
  T v[N];
#pragma unroll
  for (int e = 0; e < N; ++e) v[e] = (T)f[e];
  if constexpr (N == 8) __builtin_memcpy(__builtin_assume_aligned(to, 16), v, sizeof(v));
  else to[0] = v[0];
}
// to e4m3: the nearest code to f / scale (halves to even), no further than the largest; NaN stays one
template <int N>
__device__ __forceinline__ void store_e4m3(uint8_t* to, const float (&f)[N], float scale) {
  uint32_t w[(N + 3) / 4] = {};
  float c[N + (N & 1)];
  c[N + (N & 1) - 1] = 0.f;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const float x = f[e] / scale;
    c[e] = x > 448.f ? 448.f : x < -448.f ? -448.f : x;
  }
#if __HIP_DEVICE_COMPILE__
#pragma unroll
  for (int e = 0; e < N + (N & 1); e += 2)
    w[e / 4] = (e & 2) ? __builtin_amdgcn_cvt_pk_fp8_f32(c[e], c[e + 1], w[e / 4], true) : __builtin_amdgcn_cvt_pk_fp8_f32(c[e], c[e + 1], w[e / 4], false);
#endif
  if constexpr (N == 8) __builtin_memcpy(__builtin_assume_aligned(to, 8), w, 8);
  else to[0] = (uint8_t)w[0];
}

// Unit u of a head of d: pair(s) from u * N on while there are any, then elements that are copied.  TURN false: elements only.
template <typename T, bool E4M3, bool PAIRS, int N, bool TURN>
__device__ __forceinline__ void unit(const T* from, void* to, const float2* cs, int u, int pairs, float scale) {
  float a[N], b[N];
  const auto put = [&](int at, const float (&f)[N]) {
    if constexpr (E4M3) store_e4m3(reinterpret_cast<uint8_t*>(to) + at, f, scale);
    else store(reinterpret_cast<T*>(to) + at, f);
  };
  if constexpr (!TURN) {
    load(from + u * N, a);
    put(u * N, a);
  } else if constexpr (!PAIRS || N == 1) {
    const int turned = pairs / N;
    if (u < turned) {
      const int i = PAIRS ? 2 * u : u * N, j = PAIRS ? 2 * u + 1 : u * N + pairs;
      load(from + i, a);
      load(from + j, b);
      float x[N], y[N];
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float2 z = cs[u * N + e];
        x[e] = a[e] * z.x - b[e] * z.y;
        y[e] = b[e] * z.x + a[e] * z.y;
      }
      put(i, x);
      put(j, y);
    } else {
      const int i = 2 * pairs + (u - turned) * N;
      load(from + i, a);
      put(i, a);
    }
  } else {
    load(from + u * N, a);
    if (u * (N / 2) < pairs) {
#pragma unroll
      for (int e = 0; e < N; e += 2) {
        const float2 z = cs[u * (N / 2) + e / 2];
        const float x = a[e] * z.x - a[e + 1] * z.y;
        a[e + 1] = a[e + 1] * z.x + a[e] * z.y;
        a[e] = x;
      }
    }
    put(u * N, a);
  }
}

// N: elements of a piece, 8 where rows, heads and pairs allow it.
template <typename T, bool E4M3, bool PAIRS, int N>
__global__ __launch_bounds__(NT) void rotary_rows(const RotaryParams p) {
  extern __shared__ float2 angles[];                     // [per][pairs]
  __shared__ Where at[16];
  const int tid = threadIdx.x;
  const long first = (long)blockIdx.x * p.per;
  const int rows = (int)(p.rows - first < p.per ? p.rows - first : p.per);
  if (p.cached) {
    if (tid < rows) at[tid] = where(p, first + tid);
    __syncthreads();
  }
  for (int i = tid; i < rows * p.pairs; i += NT) {
    const int r = i / p.pairs, j = i - r * p.pairs;
    const int axis = (j >= p.end[0]) + (j >= p.end[1]) + (j >= p.end[2]);
    double t;
    if (!p.positions) t = at[r].place;
    else {
      const long x = (first + r) * p.axes + axis;
      t = p.position_type == 0 ? (double)reinterpret_cast<const int32_t*>(p.positions)[x]
          : p.position_type == 1 ? (double)reinterpret_cast<const int64_t*>(p.positions)[x] : (double)reinterpret_cast<const float*>(p.positions)[x];
    }
    t *= (p.frequency_32 ? (double)reinterpret_cast<const float*>(p.frequencies)[j] : reinterpret_cast<const double*>(p.frequencies)[j]) * ONE_TURN;
    float2 z;
    sincospif((float)(2.0 * (t - rint(t))), &z.y, &z.x);
    angles[i] = z;
  }
  __syncthreads();
  // q and k: units of a head, heads of a row, rows
  {
    const int units = PAIRS && N == 8 ? p.d / N : p.pairs / N + (p.d - 2 * p.pairs) / N, heads = p.heads + p.kv_heads;
    for (long i = tid; i < (long)rows * heads * units; i += NT) {
      const int u = (int)(i % units), hr = (int)(i / units), h = hr % heads, r = hr / heads;
      const float2* cs = angles + r * p.pairs;
      if (p.cached && at[r].place < 0) {
        if (p.fill && h < p.heads) {                     // (a unit's elements: those that it would have written)
          T* to = reinterpret_cast<T*>(p.q_out) + (first + r) * p.ldqo + (long)h * p.d;
          const float none[N] = {};
          if (PAIRS && N == 8) store(to + u * N, none);
          else if (u < p.pairs / N) {
            store(to + (PAIRS ? 2 * u : u * N), none);
            store(to + (PAIRS ? 2 * u + 1 : u * N + p.pairs), none);
          } else store(to + 2 * p.pairs + (u - p.pairs / N) * N, none);
        }
      } else if (h < p.heads) {
        unit<T, false, PAIRS, N, true>(reinterpret_cast<const T*>(p.q) + (first + r) * p.ldq + (long)h * p.d,
                                       reinterpret_cast<T*>(p.q_out) + (first + r) * p.ldqo + (long)h * p.d, cs, u, p.pairs, 1.f);
      } else {
        const int g = h - p.heads;
        const T* from = reinterpret_cast<const T*>(p.k) + (first + r) * p.ldk + (long)g * p.d;
        if (!p.cached) {
          unit<T, false, PAIRS, N, true>(from, reinterpret_cast<T*>(p.k_out) + (first + r) * p.ldko + (long)g * p.d, cs, u, p.pairs, 1.f);
        } else if (at[r].page >= 0) {
          const long to = at[r].page * p.k_page + at[r].at * p.k_token + g * p.k_head;
          unit<T, E4M3, PAIRS, N, true>(from, reinterpret_cast<char*>(p.k_out) + to * (E4M3 ? 1 : (long)sizeof(T)), cs, u, p.pairs,
                                        E4M3 && p.k_scale ? p.k_scale[g] : 1.f);
        }
      }
    }
  }
  if (p.cached) {
    const int units = p.d / N;
    for (long i = tid; i < (long)rows * p.kv_heads * units; i += NT) {
      const int u = (int)(i % units), hr = (int)(i / units), g = hr % p.kv_heads, r = hr / p.kv_heads;
      if (at[r].page < 0) continue;
      const long to = at[r].page * p.v_page + at[r].at * p.v_token + g * p.v_head;
      unit<T, E4M3, PAIRS, N, false>(reinterpret_cast<const T*>(p.v) + (first + r) * p.ldv + (long)g * p.d,
                                     reinterpret_cast<char*>(p.v_out) + to * (E4M3 ? 1 : (long)sizeof(T)), nullptr, u, 0,
                                     E4M3 && p.v_scale ? p.v_scale[g] : 1.f);
    }
  }
}

template <typename T, bool E4M3, bool PAIRS>
void launch(const RotaryParams& p, bool pieces, hipStream_t s) {
  const dim3 grid((unsigned)((p.rows + p.per - 1) / p.per));
  const size_t lds = (size_t)p.per * p.pairs * sizeof(float2);
  if (pieces) kh_launch(KH_TAG_ROTARY, rotary_rows<T, E4M3, PAIRS, 8>, grid, dim3(NT), lds, s, p);
  else kh_launch(KH_TAG_ROTARY, rotary_rows<T, E4M3, PAIRS, 1>, grid, dim3(NT), lds, s, p);
}
template <typename T, bool E4M3>
void launch(const RotaryParams& p, bool in_turn, bool pieces, hipStream_t s) {
  if (in_turn) launch<T, E4M3, true>(p, pieces, s);
  else launch<T, E4M3, false>(p, pieces, s);
}

}  // namespace

KH_EXPORT int kh_rotary(const void* q, const void* k, const void* v, void* q_out, void* k_out, const void* positions, int position_type,
                        const void* frequencies, const int64_t* section_end, int64_t axes, const KhPagedCache* cache, int64_t layer,
                        const int32_t* slots, const int32_t* places, int64_t rows, int64_t heads, int64_t kv_heads, int64_t d, int64_t ldq, int64_t ldk,
                        int64_t ldv, int64_t ldqo, int64_t ldko, int flags, int type, void* stream) {
  if (!q || !q_out || !k || !section_end || rows <= 0 || heads <= 0 || kv_heads <= 0 || d <= 0) return KH_ERR_INVALID_ARG;
  if (axes < 1 || axes > 4 || (flags & ~7) || type < 0 || type > 2 || position_type < 0 || position_type > 2) return KH_ERR_INVALID_ARG;
  for (int64_t a = 0; a < axes; ++a)
    if (section_end[a] < (a ? section_end[a - 1] : 0)) return KH_ERR_INVALID_ARG;
  const int64_t pairs = section_end[axes - 1];
  if (2 * pairs > d || (pairs > 0 && !frequencies)) return KH_ERR_INVALID_ARG;
  if (ldq < heads * d || ldqo < heads * d || ldk < kv_heads * d) return KH_ERR_INVALID_ARG;
  if (cache) {
    const int rc = kh_cache_check(cache);
    if (rc != KH_OK) return rc;
    if (!v || ldv < kv_heads * d || layer < 0 || layer >= cache->layers || cache->d != d || cache->kv_heads != kv_heads) return KH_ERR_INVALID_ARG;
    if (!slots && rows > cache->slots) return KH_ERR_INVALID_ARG;
    if (type == 2 || (cache->type != KH_E4M3 && cache->type != type)) return KH_ERR_UNSUPPORTED;
  } else if (!k_out || ldko < kv_heads * d || slots || places || (pairs > 0 && !positions)) {
    return KH_ERR_INVALID_ARG;
  }
  const uintptr_t element = type == 2 ? 4 : 2;
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)(cache ? v : k) | (uintptr_t)q_out | (uintptr_t)(cache ? q : k_out)) & (element - 1)) return KH_ERR_ALIGNMENT;
  if ((positions && ((uintptr_t)positions & (position_type == 1 ? 7 : 3))) || ((uintptr_t)frequencies & (flags & 4 ? 3 : 7))) return KH_ERR_ALIGNMENT;
  if (((uintptr_t)slots | (uintptr_t)places) & 3) return KH_ERR_ALIGNMENT;
  if (d > 1024) return KH_ERR_UNSUPPORTED;
  if (rows > (1L << 30) || heads > (1L << 20) || kv_heads > (1L << 20)) return KH_ERR_TOO_LARGE;
  RotaryParams p{};
  p.q = q, p.k = k, p.v = v, p.q_out = q_out, p.k_out = k_out, p.positions = positions, p.frequencies = frequencies, p.slots = slots, p.places = places;
  p.rows = rows, p.ldq = ldq, p.ldk = ldk, p.ldv = ldv, p.ldqo = ldqo, p.ldko = ldko;
  p.heads = (int)heads, p.kv_heads = (int)kv_heads, p.d = (int)d, p.pairs = (int)pairs, p.axes = (int)axes;
  for (int a = 0; a < 4; ++a) p.end[a] = (int)(a < axes ? section_end[a] : pairs);
  for (int a = (int)axes - 1; a < 4; ++a) p.end[a] = 1 << 30;            // (the last axis has the rest)
  p.position_type = position_type, p.frequency_32 = (flags & 4) != 0, p.fill = (flags & 2) != 0;
  if (cache) {
    const KhPagedCache& c = *cache;
    const long e = kh_cache_element(c);
    p.cached = 1, p.n_slots = (int)c.slots, p.width = (int)c.width, p.pages = (int)c.pages, p.page = (int)c.page;
    p.table = c.table, p.lengths = c.lengths;
    p.k_out = (char*)c.k + layer * c.k_layer * e, p.v_out = (char*)c.v + layer * c.v_layer * e;
    p.k_scale = c.k_scale ? c.k_scale + layer * kv_heads : nullptr, p.v_scale = c.v_scale ? c.v_scale + layer * kv_heads : nullptr;
    p.k_page = c.k_page, p.k_token = c.k_token, p.k_head = c.k_head, p.v_page = c.v_page, p.v_token = c.v_token, p.v_head = c.v_head;
  }
  const bool in_turn = flags & 1;
  // pieces of eight: whole ones in a head, its halves and its rows, at addresses of 16 bytes (the cache's are: kh_cache_check)
  const bool pieces = d % 8 == 0 && pairs % (in_turn ? 4 : 8) == 0 && (ldq | ldk | ldqo | (cache ? ldv : ldko)) % 8 == 0 && kh_aligned16(q) && kh_aligned16(k) &&
                      kh_aligned16(q_out) && kh_aligned16(cache ? v : k_out);
  // a workgroup has a row, or as many as make one angle a thread, where 2048 workgroups are left
  long per = rows / 2048;
  const long most = pairs > 0 ? (NT + pairs - 1) / pairs : 16;
  per = per < 1 ? 1 : per > most ? most : per;
  p.per = (int)(per < 16 ? per : 16);
  hipStream_t s = (hipStream_t)stream;
  const bool codes = cache && cache->type == KH_E4M3;
  if (type == 2) launch<float, false>(p, in_turn, pieces, s);
  else if (type == 0) codes ? launch<bf16_t, true>(p, in_turn, pieces, s) : launch<bf16_t, false>(p, in_turn, pieces, s);
  else codes ? launch<_Float16, true>(p, in_turn, pieces, s) : launch<_Float16, false>(p, in_turn, pieces, s);
  KH_RETURN_LAST_ERROR();
}
