// K14: rotary positions with several axes, on rows of q and k, or with the turned keys and the values written into the pages of a cache:
//   angle(r, j) = position[r][axis of j] * frequency[j],   (a, b) -> (a cos - b sin, b cos + a sin)   for every pair j of every head
//
// The angle is a number of whole turns and a rest; a position of 10^6 in 32 bits would leave the rest 0.06 off.  So the turns are counted in 64 bits
// (position * frequency / 2 pi less the nearest integer) and only the rest goes to 32 (off by 2^-26 turns), where sine and cosine are taken of a
// multiple of pi; for rows of 32 bits what it is off by turns them once more.  The products with the rows are in 32 bits and rounded once.  Codes of 8 bits have steps so wide that a key a little off in its last bits now and
// then goes to the wrong side of a border, a sixteenth away: keys that turn on the way to a code are turned and scaled in 64 bits.  A code is that of the quotient in 32
// bits, as (x.float() / scale).to(float8) has it, for values, dimensions beyond the pairs and turned keys alike: a quotient that 32 bits round to a border between two codes
// goes to the even one (one in four million; of numbers over a scale of the kind "largest / 448", many of whose quotients lie on borders, one in a thousand).
//
// Bound by memory: every element is read and written once.  A workgroup takes some rows, works their angles out once for all heads (LDS), then its
// threads go over the rows in pieces of eight elements of either half (or eight in a row), 16 bytes a load, two pieces on their way at a time
// (7904 rows of 40 heads of 64: one 19.0 us, two 15.8, three 19.8).
//
// us, the middle of 12 launches: 7904 rows of 20 + 20 heads of 64, bf16, 15.6 (5.2 TB/s in and out), 16384 of 16 + 8 of 128, fp32, 74 (5.4; four rows to a workgroup and read past the
// caches 72, but 81 behind one another), 8184 of 16 + 8 of 80 into pages 20.6 (4.1), 2 rows into pages 3.2.  Of 24: 8184 rows of 16 + 8 of 128 into bf16 pages 30 (4.5), into e4m3, every
// key turned and scaled in 64 bits, 31 (3.8), with pairs in turn 35; heads of 80 with 20 pairs, no whole eights and so an element at a time, 66 for the 14 of their bytes.
#include "paged_cache.h"
#include <type_traits>

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
  int units;                   // of a head
  KhDivide by_pairs, by_units, by_heads;
};

constexpr int NT = 256, MOST_ROWS = 16;   // threads, rows of a workgroup at most
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
// to e4m3: the nearest code to f / scale in 32 bits (halves to even), no further than the largest; NaN stays one
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

// A piece of work: unit u of a head.  Its elements are N from `first` and N from `second` on, the a and b of N pairs; with pairs in turn (and N > 1), or behind the
// pairs, only the N from `first` on.
template <typename T, bool E4M3, bool PAIRS, int N>
struct Unit {
  using Turn = typename std::conditional<E4M3, double2, float2>::type;   // cosine and sine
  const T* from;
  void* to;
  int first, second;           // second < 0: none
  const Turn* cs;              // of the first pair; nullptr: copied
  float scale;                 // of an e4m3 code
  int what;                    // 0 nothing, 1 to T, 2 to codes, 3 zeros
  float a[N], b[N];

  __device__ __forceinline__ void at(int u, int pairs, const Turn* angles) {
    second = -1;
    cs = nullptr;
    if (PAIRS && N > 1) {
      first = u * N;
      if (u * (N / 2) < pairs) cs = angles + u * (N / 2);
    } else if (u * N < pairs) {
      first = PAIRS ? 2 * u : u * N;
      second = PAIRS ? 2 * u + 1 : u * N + pairs;
      cs = angles + u * N;
    } else {
      first = u * N + pairs;                              // (2 pairs + (u - pairs / N) * N)
    }
  }
  __device__ __forceinline__ void fetch() {
    if (what == 0 || what == 3) return;
    load(from + first, a);
    if (second >= 0) load(from + second, b);
  }
  // The pair (a, b) turned by z, in the type of z and times `by`.
  template <typename X>
  static __device__ __forceinline__ void turn(float& a, float& b, const Turn& z, X by) {
    const X c = (X)z.x, s = (X)z.y, x = (X)a * c - (X)b * s, y = (X)b * c + (X)a * s;
    a = (float)(x * by);
    b = (float)(y * by);
  }
  template <typename X>
  __device__ __forceinline__ void turn_all(X by) {
    if constexpr (PAIRS && N > 1) {
#pragma unroll
      for (int e = 0; e < N; e += 2) turn<X>(a[e], a[e + 1], cs[e / 2], by);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) turn<X>(a[e], b[e], cs[e], by);
    }
  }
  __device__ __forceinline__ void finish() {
    if (what == 0) return;
    if (what == 3) {
#pragma unroll
      for (int e = 0; e < N; ++e) a[e] = b[e] = 0.f;
    }
    if (E4M3 && what == 2) {
      if (cs) {
        turn_all<double>(1.0 / (double)scale);
        scale = 1.f;
      }
      store_e4m3(reinterpret_cast<uint8_t*>(to) + first, a, scale);
      if (second >= 0) store_e4m3(reinterpret_cast<uint8_t*>(to) + second, b, scale);
    } else {
      if (cs && what == 1) turn_all<float>(1.f);
      store(reinterpret_cast<T*>(to) + first, a);
      if (second >= 0) store(reinterpret_cast<T*>(to) + second, b);
    }
  }
};

// N: elements of a piece, 8 where rows, heads and pairs allow it.
template <typename T, bool E4M3, bool PAIRS, int N>
__global__ __launch_bounds__(NT) void rotary_rows(const RotaryParams p) {
  using Piece = Unit<T, E4M3, PAIRS, N>;
  using Turn = typename Piece::Turn;
  extern __shared__ double2 lds[];                       // [per][pairs] cosines and sines
  Turn* const angles = reinterpret_cast<Turn*>(lds);
  __shared__ Where at[MOST_ROWS];
  const int tid = threadIdx.x;
  const long first = (long)blockIdx.x * p.per;
  const int rows = (int)(p.rows - first < p.per ? p.rows - first : p.per);
  // (the last wave looks the pages up while the others begin with the angles)
  if (p.cached && tid >= NT - 64 && tid - (NT - 64) < rows) at[tid - (NT - 64)] = where(p, first + tid - (NT - 64));
  if (!p.positions) __syncthreads();
  for (int i = tid; i < rows * p.pairs; i += NT) {
    const int r = (int)p.by_pairs((uint32_t)i), j = i - r * p.pairs;
    const int axis = (j >= p.end[0]) + (j >= p.end[1]) + (j >= p.end[2]);
    double t;
    if (!p.positions) t = at[r].place;
    else {
      const long x = (first + r) * p.axes + axis;
      t = p.position_type == 0 ? (double)reinterpret_cast<const int32_t*>(p.positions)[x]
          : p.position_type == 1 ? (double)reinterpret_cast<const int64_t*>(p.positions)[x] : (double)reinterpret_cast<const float*>(p.positions)[x];
    }
    t *= (p.frequency_32 ? (double)reinterpret_cast<const float*>(p.frequencies)[j] : reinterpret_cast<const double*>(p.frequencies)[j]) * ONE_TURN;
    Turn z;
    if constexpr (E4M3) sincospi(2.0 * (t - rint(t)), &z.y, &z.x);
    else {
      const double half = 2.0 * (t - rint(t));
      const float near = (float)half;
      sincospif(near, &z.y, &z.x);
      if constexpr (sizeof(T) == 4) {                     // (rows of 16 bits do not show it)
        const float rest = (float)(half - (double)near) * 3.14159265f, x = z.x;
        z.x -= z.y * rest;
        z.y += x * rest;
      }
    }
    angles[i] = z;
  }
  __syncthreads();
  // units of a head, heads of a row (of q, of k, with a cache of v), rows
  const int units = p.units, heads = p.heads + p.kv_heads, all = p.cached ? heads + p.kv_heads : heads, count = rows * all * units;
  auto piece = [&](int i, Piece& x) {
    x.what = 0;
    if (i >= count) return;
    const int hr = (int)p.by_units((uint32_t)i), u = i - hr * units, r = (int)p.by_heads((uint32_t)hr), h = hr - r * all;
    x.at(u, p.pairs, angles + r * p.pairs);
    const long row = first + r;
    if (h < p.heads) {
      x.from = reinterpret_cast<const T*>(p.q) + row * p.ldq + (long)h * p.d;
      x.to = reinterpret_cast<T*>(p.q_out) + row * p.ldqo + (long)h * p.d;
      x.what = !p.cached || at[r].place >= 0 ? 1 : p.fill ? 3 : 0;
    } else {
      const bool values = h >= heads;
      const int g = h - (values ? heads : p.heads);
      x.from = reinterpret_cast<const T*>(values ? p.v : p.k) + row * (values ? p.ldv : p.ldk) + (long)g * p.d;
      if (values) x.cs = nullptr;
      if (!p.cached) {
        x.to = reinterpret_cast<T*>(p.k_out) + row * p.ldko + (long)g * p.d;
        x.what = 1;
      } else if (at[r].page >= 0) {
        const long to = at[r].page * (values ? p.v_page : p.k_page) + at[r].at * (values ? p.v_token : p.k_token) + g * (values ? p.v_head : p.k_head);
        x.to = reinterpret_cast<char*>(values ? p.v_out : p.k_out) + to * (E4M3 ? 1 : (long)sizeof(T));
        x.what = E4M3 ? 2 : 1;
        const float* scales = values ? p.v_scale : p.k_scale;
        x.scale = E4M3 && scales ? scales[g] : 1.f;
      }
    }
  };
  for (int i = tid; i < count; i += 2 * NT) {            // two on their way at a time
    Piece x, y;
    piece(i, x);
    piece(i + NT, y);
    x.fetch();
    y.fetch();
    x.finish();
    y.finish();
  }
}

template <typename T, bool E4M3, bool PAIRS>
void launch(const RotaryParams& p, bool pieces, hipStream_t s) {
  const dim3 grid((unsigned)((p.rows + p.per - 1) / p.per));
  const size_t lds = (size_t)p.per * p.pairs * (E4M3 ? sizeof(double2) : sizeof(float2));
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
  if (rows > (1L << 30) || heads * d > (1L << 24) || kv_heads * d > (1L << 24)) return KH_ERR_TOO_LARGE;   // (a workgroup counts its pieces in 31 bits)
  RotaryParams p{.by_pairs = KhDivide(pairs > 0 ? (uint32_t)pairs : 1u), .by_units = KhDivide(1), .by_heads = KhDivide((uint32_t)(heads + kv_heads * (cache ? 2 : 1)))};
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
  p.units = pieces ? (int)(in_turn ? d / 8 : pairs / 8 + (d - 2 * pairs) / 8) : (int)(d - pairs);
  p.by_units = KhDivide((uint32_t)p.units);
  // A workgroup has a row, or as many as make 12 KB, if 2048 workgroups are left and no thread has two angles (16384 rows of 12 KB, calls behind one another: one to a workgroup
  // 74.3 us, two 77.5, four 80.7; 7904 rows of 5 KB by themselves: three 15.2, seven 16.6, one 18.3), up to twice that where its pieces then fill the threads better
  // (8184 rows of 32 heads of 80 into pages: three rows 20.9 us, four 19.2; behind one another four 18.5, six 20.0).
  const long each = (heads + kv_heads * (cache ? 2 : 1)) * p.units, bytes = (heads + kv_heads) * d * (long)element;
  long whole = pairs > 0 ? (NT + pairs - 1) / pairs : MOST_ROWS, least = rows / 2048;
  whole = whole < MOST_ROWS ? whole : MOST_ROWS;
  least = least < 12288 / bytes ? least : 12288 / bytes;
  least = least < 1 ? 1 : least < whole ? least : whole;
  double best = 0.;
  for (long n = least; n <= (least > 1 ? (2 * least < whole ? 2 * least : whole) : 1); ++n) {
    const long rounds = (n * each + 2 * NT - 1) / (2 * NT);
    const double full = (double)(n * each) / (double)(rounds * 2 * NT);
    if (full > best) best = full, p.per = (int)n;
  }
  if ((rows + p.per - 1) / p.per > (1L << 24) - 1) return KH_ERR_TOO_LARGE;     // (2^32 threads)
  hipStream_t s = (hipStream_t)stream;
  const bool codes = cache && cache->type == KH_E4M3;
  if (type == 2) launch<float, false>(p, in_turn, pieces, s);
  else if (type == 0) codes ? launch<bf16_t, true>(p, in_turn, pieces, s) : launch<bf16_t, false>(p, in_turn, pieces, s);
  else codes ? launch<_Float16, true>(p, in_turn, pieces, s) : launch<_Float16, false>(p, in_turn, pieces, s);
  KH_RETURN_LAST_ERROR();
}
