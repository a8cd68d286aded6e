// K15: attention of one token a row over a paged cache:
//   x_t = scale * q . k_t,   m = max x_t,   o = sum_t exp(x_t - m) v_t / sum_t exp(x_t - m)
//
// Bound by the bytes of the keys and values, which are read once for all query heads that share them.  The work is cut over the cache's length: the
// tiles of 128 tokens of all rows and key heads stand in one line, and every workgroup takes an equal part of it, wherever sequences end (the lengths lie on
// the device; a plan on the host would have to go by the longest).  A row and key head that one workgroup has whole is written by it; of others the
// parts are left in 32 bits (maximum, sum, unscaled output) and a second launch joins them in order.
//
// A tile is four waves of 32 tokens, each on its own until the workgroup's part ends:
//   S^T = K . Q^T     A = the keys as they lie in memory (lane l: token l % 16, 8 dimensions from 8 * (l / 16) on), B = up to 16 query heads in registers
//   O^T += V^T . P^T  A = values of 8 tokens for a dimension, put together from the loads of 8 whole rows by byte permutes in the lane, B = P
// The tokens of the keys' rows are chosen so that the scores a lane gets (query l % 16, eight tokens) are the P operand it needs: nothing crosses lanes but the
// maximum.  Neither operand goes through LDS.  P is multiplied in all 24 bits, in three pieces of 16: the matrix unit waits for memory anyway.
//
// us a launch, the middle of 12 (TB/s of keys and values): one token of 64 requests of 0 .. 8192 tokens, 32 heads of 128 on 8, bf16, 120 (5.5) and 4.9 for the join; one of 131071 tokens,
// 16 heads on 2, fp16, 27.0 (5.0) and 5.7; 2 x 77 tokens 5.7, a chain of lengths, page numbers and rows.  32 of 4096 tokens with 4 KB a token, heads of 64, 128, 256: 93, 91, 85 (5.8, 5.9, 6.3)
// on one card and 116, 113, 102 on another, with 2 KB in e4m3 87, 53, 63 and 98, 63, 66.  A copy of 1 GiB runs at 5.1 TB/s.  With each step's loads waited for where they are used: 207 and 55.  Values are read past
// the caches (126 us where that is 119), keys are not (123, and the two halves of a line that a wave asks for one after the other are both there: e4m3 78 -> 59).
#include "paged_cache.h"
#include <type_traits>

namespace {

constexpr int NW = 4, STEP = 32, TILE = NW * STEP;       // waves, tokens of a wave's step, of a tile
constexpr int QB = 16;                                  // query heads of a unit
constexpr int JT = 512, MOST = 1024;                    // threads that join, workgroups at most that share the line
constexpr int WHOLE = 4;                                // tiles that a table (or window) holds at most where units are not cut
constexpr float RESCALE_LOG2 = 8.0f;                    // the running maximum moves only for jumps above 2^8

struct PagedParams {
  const void *q, *k, *v;
  void* o;
  const int32_t *table, *row_lengths, *lengths, *slots;
  const float *k_scale, *v_scale;
  float* part;                // [2 workgroups][group][d] outputs, then [2 workgroups][group][2] maxima and sums
  int4* border;               // [workgroups]: row, unit, workgroups of the unit that a workgroup begins inside
  long ldq, ldo;
  uint32_t k_page, k_token, v_page, v_token;            // bytes
  long k_head, v_head;
  int rows, kv_heads, group, blocks, d;                 // blocks: units of a key head
  int n_slots, width, pages, page, window;
  float scale_log2;
  int fill, q_aligned;
  int whole;                  // every workgroup has a unit, and no unit parts
  int shared_lines;           // neighbouring key heads share lines of 128 bytes: neighbouring parts of the line of tiles on one XCD, whose L2 then has them
  KhDivide by_page;
};

typedef uint32_t u32x1 __attribute__((ext_vector_type(1)));
typedef _Float16 f16_t;
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

template <typename T> struct Eight;
template <> struct Eight<bf16_t> { using type = bf16x8; };
template <> struct Eight<f16_t> { using type = f16x8; };

__device__ __forceinline__ f32x4 mfma(const bf16x8& a, const bf16x8& b, const f32x4& c) {
#if __HIP_DEVICE_COMPILE__
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
#else
  return c;
#endif
}
__device__ __forceinline__ f32x4 mfma(const f16x8& a, const f16x8& b, const f32x4& c) {
#if __HIP_DEVICE_COMPILE__
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
#else
  return c;
#endif
}

__device__ __forceinline__ float swapped_max(float v) {  // over the four lanes of a query
#if __HIP_DEVICE_COMPILE__
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
#else
  return v;
#endif
}

// The codes of a word's lower or upper two bytes as two numbers of T (exact).
template <typename T, bool UP>
__device__ __forceinline__ uint32_t two_of_e4m3(uint32_t w) {
#if __HIP_DEVICE_COMPILE__
  if constexpr (sizeof(T) == 2 && __is_same(T, bf16_t)) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, UP));
  else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, UP));
#else
  return w;
#endif
}

// P in three pieces.  Of bf16 they are the upper bits of what is left each time, and P is their sum: bf16 reaches as far down as 32 bits do.  fp16 does not: P is held
// 2^7 times as large (it stays under 2^15, the running maximum may be 2^8 behind), and what a piece leaves goes to the next one 2^11 times as large, with a product of its
// own.  That is all of P down to 2^-30 of the largest, 17 bits down to 2^-36 and 11 down to 2^-42; what is lost of n weights is under n 2^-54 (of two pieces of P as it is
// n 2^-25, a hundredth of what tokens 16 below one whose value is zero give).  us: one sequence of 131071 tokens 25.1 with two pieces, 26.0 so, 28.4 with products in 32 bits.
template <typename W> struct Pieces;
template <> struct Pieces<bf16_t> {
  static constexpr float UP_LOG2 = 0.f;
  static constexpr bool APART = false;                  // whether a piece has a product of its own
  static __device__ __forceinline__ void of(const float (&p)[8], bf16x8 (&out)[3]) {
    uint32_t w[3][4];
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      float a = p[i], b = p[i + 1];
#pragma unroll
      for (int n = 0; n < 3; ++n) {
        w[n][i / 2] = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302);
        a -= __uint_as_float(__float_as_uint(a) & 0xffff0000u);
        b -= __uint_as_float(__float_as_uint(b) & 0xffff0000u);
      }
    }
#pragma unroll
    for (int n = 0; n < 3; ++n) out[n] = __builtin_bit_cast(bf16x8, u32x4{w[n][0], w[n][1], w[n][2], w[n][3]});
  }
};
template <> struct Pieces<f16_t> {
  static constexpr float UP_LOG2 = 7.f, REST = 0x1p11f;
  static constexpr bool APART = true;
  static __device__ __forceinline__ void of(const float (&p)[8], f16x8 (&out)[3]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      out[0][i] = (f16_t)p[i];
      const float rest = (p[i] - (float)out[0][i]) * REST;
      out[1][i] = (f16_t)rest;
      out[2][i] = (f16_t)((rest - (float)out[1][i]) * REST);
    }
  }
};

// a value that all lanes have, in scalar registers
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// the thread's number as something the compiler does not know: what is worked out from it stays where it is used, instead of in registers across the loop of the
// steps (heads of 128: 232 of them and 219 so, in e4m3 spills and none: 32 sequences of 4096 tokens 59 -> 53 us)
__device__ __forceinline__ int thread_here() {
  int t = threadIdx.x;
#if __HIP_DEVICE_COMPILE__
  asm volatile("" : "+v"(t));
#endif
  return t;
}

// A row's sequence: its slot (-1: none), the tokens low .. n - 1 to attend to; `tiles` tiles of 128 from `tile` on.
struct Row { int slot, n, low, tile, tiles; };

__device__ __forceinline__ Row row_of(const PagedParams& p, int slot, int n) {
  const int low = p.window > 0 && n > p.window ? n - p.window : 0, tile = low / TILE;
  return Row{slot, n, low, tile, (n + TILE - 1) / TILE - tile};
}
__device__ __forceinline__ Row row_of(const PagedParams& p, int r) {
  const int s = p.slots ? p.slots[r] : r;
  if (s < 0 || s >= p.n_slots) return row_of(p, -1, 0);
  const int n = p.row_lengths ? p.row_lengths[r] : p.lengths[s], most = p.width * p.page;
  return row_of(p, s, n < 0 ? 0 : n < most ? n : most);
}

// What a workgroup does of a unit (a row, a key head and up to 16 of its query heads): the unit in the line of tiles and the part at .. stop - 1 of it.
struct Piece {
  Row row;
  int r, unit, head, q0, queries;
  int row_at, a, b, at, stop;
};

// Shapes.  D: dimensions there is room for (d of them used: TAIL where fewer); CODES: the cache holds e4m3; EIGHT: pages of a multiple of eight tokens, so that
// the eight tokens of a lane lie on one page.
template <int D, typename T, bool CODES, bool EIGHT, bool TAIL>
struct Shape {
  using X = typename Eight<T>::type;
  using Raw = typename std::conditional<CODES, u32x2, u32x4>::type;      // eight elements of a row
  static constexpr int KK = D / 32;                     // k-steps of the scores
  static constexpr int NC = D >= 128 ? D / 128 : 1;     // pieces of a row of values in a lane
  static constexpr int VE = D >= 128 ? 8 : 4;           // elements of one
  static constexpr int ELT = CODES ? 1 : 2;
  static constexpr int VW = VE * ELT / 4;               // words of one
  using Piece = typename std::conditional<VW == 4, u32x4, typename std::conditional<VW == 2, u32x2, u32x1>::type>::type;
};

// A wave's part of a unit.  Keys and values of a step are requested as soon as the registers of the step before are free (keys behind its scores, values behind
// its products), the numbers of the pages a step earlier still, so that loads are on their way all the time.
template <int D, typename T, bool CODES, bool EIGHT, bool TAIL>
struct Wave {
  using S = Shape<D, T, CODES, EIGHT, TAIL>;
  using X = typename S::X;
  using W = typename std::conditional<CODES, bf16_t, T>::type;           // the type that values and weights are multiplied in: codes are numbers of bf16, whatever the queries are
  using X8 = typename Eight<W>::type;
  struct Pages { int k[EIGHT ? 1 : 2], v[EIGHT ? 1 : 8]; };

  X q[S::KK];
  f32x4 o[S::NC * S::VE];                               // tile c * VE + j: dimensions c * 128 + VE * (4 * (l / 16) + r) + j of query l % 16
  float m, l;
  Pages now, next;
  int t0, steps;
  typename S::Raw kr[2][S::KK];
  typename S::Piece vr[8][S::NC];

  // Tokens of lane l: of the keys 8 * (l % 16 / 4) + 4 s + l % 4, of the values (and of the scores it gets) 8 * (l / 16) + i.  One behind the end is
  // looked for at the last one.
  static __device__ __forceinline__ int key(int t0, int s) { return t0 + 8 * ((threadIdx.x & 15) >> 2) + 4 * s + (threadIdx.x & 3); }
  static __device__ __forceinline__ int value(int t0, int i) { return t0 + 8 * ((threadIdx.x & 63) >> 4) + i; }
  static __device__ __forceinline__ int kept(int t, int last) { return t < last ? t : last; }

  __device__ __forceinline__ Pages pages_of(const PagedParams& p, const Row& row, int t0) const {
    Pages e;
    const int last = EIGHT ? (row.n - 1) & ~7 : row.n - 1;
    const int32_t* pages = p.table + (long)row.slot * p.width;
#pragma unroll
    for (int s = 0; s < (EIGHT ? 1 : 2); ++s) e.k[s] = pages[p.by_page((uint32_t)kept(EIGHT ? key(t0, 0) & ~7 : key(t0, s), last))];
#pragma unroll
    for (int i = 0; i < (EIGHT ? 1 : 8); ++i) e.v[i] = pages[p.by_page((uint32_t)kept(value(t0, i), last))];
    return e;
  }
  // where a token's row lies; without a page: the first of all
  static __device__ __forceinline__ const char* place(const PagedParams& p, const char* base, int e, int t, uint32_t page, uint32_t token) {
    const bool there = (uint32_t)e < (uint32_t)p.pages;
    const uint32_t at = (uint32_t)t - p.by_page((uint32_t)t) * (uint32_t)p.page;
    return base + (uint64_t)(there ? (uint32_t)e : 0u) * page + (uint64_t)(there ? at : 0u) * token;
  }
  __device__ __forceinline__ void load_keys(const PagedParams& p, const Row& row, const char* kb, const Pages& e, int t0) {
    const int g4 = (threadIdx.x & 63) >> 4, last = EIGHT ? (row.n - 1) | 7 : row.n - 1;     // (a page of whole eights has the tokens up to there)
    const char* at[2];
    at[0] = place(p, kb, e.k[0], kept(key(t0, 0), last), p.k_page, p.k_token);
    if (EIGHT) at[1] = place(p, kb, e.k[0], kept(key(t0, 1), last), p.k_page, p.k_token);
    else at[1] = place(p, kb, e.k[EIGHT ? 0 : 1], kept(key(t0, 1), last), p.k_page, p.k_token);
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int kk = 0; kk < S::KK; ++kk) {
        const int dim = kk * 32 + g4 * 8;
        if (TAIL && kk * 32 >= p.d) kr[s][kk] = typename S::Raw{};
        else kr[s][kk] = *reinterpret_cast<const typename S::Raw*>(at[s] + (!TAIL || dim < p.d ? dim : 0) * S::ELT);
      }
  }
  __device__ __forceinline__ void load_values(const PagedParams& p, const Row& row, const char* vb, const Pages& e, int t0) {
    const int c16 = threadIdx.x & 15, last = EIGHT ? (row.n - 1) & ~7 : row.n - 1;
    const char* first = place(p, vb, e.v[0], kept(value(t0, 0), last), p.v_page, p.v_token);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const char* at = EIGHT ? first + (uint64_t)p.v_token * i : i == 0 ? first : place(p, vb, e.v[EIGHT ? 0 : i], kept(value(t0, i), last), p.v_page, p.v_token);
#pragma unroll
      for (int c = 0; c < S::NC; ++c) {
        const int dim = c * 128 + c16 * S::VE;
        vr[i][c] = __builtin_nontemporal_load(reinterpret_cast<const typename S::Piece*>(at + (!TAIL || dim < p.d ? dim : 0) * S::ELT));
      }
    }
  }

  // Requests the first step of a piece (and its queries): the tokens t0, t0 + TILE, .. of its row, `steps` times 32, of which low .. n - 1 count.
  __device__ __forceinline__ void begin(const PagedParams& p, const Piece& u, int wave) {
    const int c16 = thread_here() & 15, g4 = thread_here() >> 4 & 3;
    t0 = (u.row.tile + u.at - u.a) * TILE + wave * STEP;
    steps = u.stop - u.at;
    if (t0 + (steps - 1) * TILE >= u.row.n) --steps;     // (only the last tile may begin behind the end for some waves,
    if (t0 + STEP <= u.row.low) t0 += TILE, --steps;     //  only the first end before the window)
    if (steps > 0) {
      now = pages_of(p, u.row, t0);
      next = pages_of(p, u.row, t0 + (steps > 1 ? TILE : 0));
    }
    const T* qp = reinterpret_cast<const T*>(p.q) + (long)u.r * p.ldq + ((long)u.head * p.group + u.q0 + (c16 < u.queries ? c16 : 0)) * p.d;
#pragma unroll
    for (int kk = 0; kk < S::KK; ++kk) {
      const int dim = kk * 32 + g4 * 8;
      T e[8] = {};
      if (c16 < u.queries && (!TAIL || dim < p.d)) {
        if (p.q_aligned) __builtin_memcpy(e, __builtin_assume_aligned(qp + dim, 16), 16);
        else
#pragma unroll
          for (int i = 0; i < 8; ++i) e[i] = qp[dim + i];
      }
      __builtin_memcpy(&q[kk], e, 16);
    }
    if (steps > 0) {
      load_keys(p, u.row, reinterpret_cast<const char*>(p.k) + u.head * p.k_head, now, t0);
      load_values(p, u.row, reinterpret_cast<const char*>(p.v) + u.head * p.v_head, now, t0);
    }
  }
  __device__ __forceinline__ void run(const PagedParams& p, const Piece& u) {
#pragma unroll
    for (int i = 0; i < S::NC * S::VE; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    m = -INFINITY;
    l = 0.f;
    if (steps <= 0) return;
    const Row& row = u.row;
    const char* kb = reinterpret_cast<const char*>(p.k) + u.head * p.k_head;
    const char* vb = reinterpret_cast<const char*>(p.v) + u.head * p.v_head;
    const float factor = p.scale_log2 * (CODES && p.k_scale ? p.k_scale[u.head] : 1.f);
    for (int n = 1; n < steps; ++n) step<true>(p, row, kb, vb, factor, n + 1 < steps);
    step<false>(p, row, kb, vb, factor, false);
  }
  // MORE: another step follows, on the pages `next`; `after`: and one behind that.
  template <bool MORE>
  __device__ __forceinline__ void step(const PagedParams& p, const Row& row, const char* kb, const char* vb, float factor, bool after) {
    // scores: x[4 s + r] is token 8 * (l / 16) + 4 s + r of query l % 16
    float x[8];
    const int g4 = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      f32x4 acc{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < S::KK; ++kk) {
        typename S::Raw w = kr[s][kk];
        if (TAIL && kk * 32 + g4 * 8 >= p.d) w = typename S::Raw{};
        X a;
        if constexpr (CODES) a = __builtin_bit_cast(X, u32x4{two_of_e4m3<T, false>(w[0]), two_of_e4m3<T, true>(w[0]), two_of_e4m3<T, false>(w[1]), two_of_e4m3<T, true>(w[1])});
        else a = __builtin_bit_cast(X, w);
        acc = mfma(a, q[kk], acc);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) x[4 * s + r] = acc[r] * factor;
    }
    if constexpr (MORE) load_keys(p, row, kb, next, t0 + TILE);
    // what does not count may be anything: scores and values of tokens outside, or without a page
    const int first = value(t0, 0);
    bool good[8], whole = true;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      good[i] = (uint32_t)now.v[EIGHT ? 0 : i] < (uint32_t)p.pages && first + i >= row.low && first + i < row.n;
      whole = whole && good[i];
    }
    if (__any(!whole)) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = good[i] ? x[i] : -INFINITY;
#pragma unroll
        for (int c = 0; c < S::NC; ++c)
#pragma unroll
          for (int w = 0; w < S::VW; ++w) vr[i][c][w] = good[i] ? vr[i][c][w] : 0;
      }
    }
    float top = x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) top = fmaxf(top, x[i]);
    top = swapped_max(top);
    if (__any(top - m > RESCALE_LOG2)) {                    // (a difference of large numbers is exact, their sum with 2^3 is not)
      const float to = fmaxf(m, top), by = to == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - to);
      m = to;
      l *= by;
#pragma unroll
      for (int i = 0; i < S::NC * S::VE; ++i) o[i] *= by;
    }
    const float from = m == -INFINITY ? 0.f : m;
    float pr[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float at = x[i] - from;
      if constexpr (Pieces<W>::UP_LOG2 > 0.f) at += Pieces<W>::UP_LOG2;
      pr[i] = __builtin_amdgcn_exp2f(at);
      l += pr[i];
    }
    X8 pieces[3];
    Pieces<W>::of(pr, pieces);
#pragma unroll
    for (int c = 0; c < S::NC; ++c)
#pragma unroll
      for (int j = 0; j < S::VE; ++j) {
        u32x4 a;
#pragma unroll
        for (int h = 0; h < 4; ++h) {                 // tokens 2 h, 2 h + 1
          if constexpr (CODES) {
            const uint32_t both = __builtin_amdgcn_perm(vr[2 * h + 1][c][j / 4], vr[2 * h][c][j / 4], 0x0400u + (j % 4) * 0x0101u);
            a[h] = two_of_e4m3<W, false>(both);
          } else {
            a[h] = __builtin_amdgcn_perm(vr[2 * h + 1][c][j / 2], vr[2 * h][c][j / 2], j & 1 ? 0x07060302 : 0x05040100);
          }
        }
        const X8 value8 = __builtin_bit_cast(X8, a);
        f32x4& to = o[c * S::VE + j];
        to = mfma(value8, pieces[0], to);
        if constexpr (Pieces<W>::APART) {
          f32x4 rest = mfma(value8, pieces[2], f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
          for (int r = 0; r < 4; ++r) rest[r] *= 1.f / Pieces<W>::REST;
          rest = mfma(value8, pieces[1], rest);
#pragma unroll
          for (int r = 0; r < 4; ++r) to[r] += rest[r] * (1.f / Pieces<W>::REST);
        } else {
          to = mfma(value8, pieces[2], mfma(value8, pieces[1], to));
        }
      }
    if constexpr (MORE) {
      t0 += TILE;
      now = next;
      next = pages_of(p, row, t0 + (after ? TILE : 0));         // (before the values: its use does not wait for those)
      load_values(p, row, vb, now, t0);
    }
  }
};

template <typename T, int N>
__device__ __forceinline__ void store_row(const PagedParams& p, int row, int query, int dim, const float (&f)[N], float sum, float scale) {
  T v[N];
#pragma unroll
  for (int e = 0; e < N; ++e) v[e] = (T)(sum == 0.f ? 0.f : f[e] / sum * scale);
  __builtin_memcpy(reinterpret_cast<T*>(p.o) + (long)row * p.ldo + (long)query * p.d + dim, v, sizeof(v));
}

template <typename T>
__device__ __forceinline__ void zero_row(const PagedParams& p, int r) {
  T* to = reinterpret_cast<T*>(p.o) + (long)r * p.ldo;
  for (int i = threadIdx.x; i < p.kv_heads * p.group * p.d; i += NW * 64) to[i] = (T)0.f;
}

// Workgroups a CU, by what registers allow without spilling in the loop.  us of 32 sequences of 4096 tokens, 4096 bytes of keys and values a token in 16 bits: heads of
// 128 91 with two (three spill: 64 requests took 179 with three and 123 with two), of 64 93 with three (116 with four), of 256 85 with one; in e4m3, whose steps have
// half the bytes, of 128 84 with two and 68 with three (53 since), of 64 85 with three and 104 with four, of 256 72 with one and 63 with two.
constexpr int wgs_a_cu(int D, bool codes) { return D > 128 ? (codes ? 2 : 1) : D > 64 && !codes ? 2 : 3; }

template <int D, typename T, bool CODES, bool EIGHT, bool TAIL>
__global__ __launch_bounds__(NW * 64, wgs_a_cu(D, CODES)) void attend(const PagedParams p) {
  using S = Shape<D, T, CODES, EIGHT, TAIL>;
  constexpr int OW = D + 4;                             // floats of a query's row in LDS
  extern __shared__ float lds[];                        // [NW][QB][OW] outputs, [2][NW][QB] maxima and sums
  float* const ms = lds + NW * QB * OW;
  __shared__ int starts[NW];
  __shared__ int where[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int units = p.kv_heads * p.blocks, G = gridDim.x, w = p.shared_lines ? (int)xcd_remap(blockIdx.x, gridDim.x) : (int)blockIdx.x;

  int total = 0, W = G, begin, end;
  Piece u;
  bool active;
  if (p.whole) {                                        // a unit each
    u.r = w / units;
    const Row x = row_of(p, u.r);
    u.row = row_of(p, uniform(x.slot), uniform(x.n));
    u.row_at = 0;
    begin = (w - u.r * units) * u.row.tiles;
    end = begin + u.row.tiles;
    active = u.row.tiles > 0;
  } else {
    // the line of tiles: all of them, and the row in which this workgroup's part begins
    const int each = (p.rows + NW * 64 - 1) / (NW * 64), r0 = tid * each, r1 = r0 + each < p.rows ? r0 + each : p.rows;
    Row one{};
    int mine = 0;
    for (int r = r0; r < r1; ++r) mine += (one = row_of(p, r)).tiles;
    int before = mine;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
      const int y = __shfl_up(before, s, 64);
      if (lane >= s) before += y;
    }
    if (lane == 63) starts[wave] = before;
    if (tid < 4) where[tid] = tid == 2 ? -1 : 0;
    __syncthreads();
    before -= mine;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      if (i < wave) before += starts[i];
      total += starts[i];
    }
    total = uniform(total) * units;
    W = total < G ? total : G;                          // workgroups that have a tile
    if (tid == 0) p.border[w] = int4{-1, 0, 0, 0};
    active = w < W;
    begin = active ? (int)((long)total * w / W) : 0;
    end = active ? (int)((long)total * (w + 1) / W) : 0;
    if (active) {
      int at_row = before * units;                      // where row r begins
      for (int r = r0; r < r1; ++r) {
        if (each > 1) one = row_of(p, r);
        const int next = at_row + one.tiles * units;
        if (begin >= at_row && begin < next) {
          where[0] = r;
          where[1] = at_row;
          where[2] = one.slot;
          where[3] = one.n;
        }
        at_row = next;
      }
      __syncthreads();
      u.r = uniform(where[0]);
      u.row_at = uniform(where[1]);
      u.row = row_of(p, uniform(where[2]), uniform(where[3]));
    }
  }
  if (active) {
    // the piece from `at` on in the line; false: none (nor behind the last row, should somebody write to the lengths meanwhile)
    auto advance = [&](Piece& u, int at) {
      if (at >= end) return false;
      while (at >= u.row_at + u.row.tiles * units) {
        if (++u.r >= p.rows) return false;
        u.row_at += u.row.tiles * units;
        const Row x = row_of(p, u.r);
        u.row = row_of(p, uniform(x.slot), uniform(x.n));
      }
      u.unit = (at - u.row_at) / u.row.tiles;
      u.head = u.unit / p.blocks;
      u.q0 = (u.unit - u.head * p.blocks) * QB;
      u.queries = p.group - u.q0 < QB ? p.group - u.q0 : QB;
      u.a = u.row_at + u.unit * u.row.tiles;
      u.b = u.a + u.row.tiles;
      u.at = at;
      u.stop = u.b < end ? u.b : end;
      return true;
    };
    Wave<D, T, CODES, EIGHT, TAIL> wv;
    Piece done;
    int at = begin;
    for (bool some = false;; some = true) {
      const bool more = advance(u, at);
      if (more) wv.begin(p, u, wave);                   // (on its way while the waves' parts of the piece before it are put together)
      if (some) {
        // the waves' parts together
        const int tid = thread_here(), c16 = tid & 15, g4 = tid >> 4 & 3;
        float sum = wv.l;
        sum += __shfl_xor(sum, 16, 64);
        sum += __shfl_xor(sum, 32, 64);
        if (g4 == 0) {
          ms[wave * QB + c16] = wv.m;
          ms[(NW + wave) * QB + c16] = sum;
        }
        __syncthreads();
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < NW; ++i) top = fmaxf(top, ms[i * QB + c16]);
        const float by = wv.m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(wv.m - top);
#pragma unroll
        for (int c = 0; c < S::NC; ++c)
#pragma unroll
          for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int j = 0; j < S::VE; j += 4) {
              f32x4 f;
#pragma unroll
              for (int i = 0; i < 4; ++i) f[i] = wv.o[c * S::VE + j + i][n] * by;
              *reinterpret_cast<f32x4*>(lds + (wave * QB + c16) * OW + c * 128 + S::VE * (4 * g4 + n) + j) = f;
            }
        __syncthreads();
        const bool complete = done.a >= begin && done.b <= end;
        const long slot = 2 * (long)w + (done.a >= begin ? 1 : 0);
        const int q_max = p.group < QB ? p.group : QB;
        for (int i = tid; i < done.queries * (D / 4); i += NW * 64) {
          const int qi = i / (D / 4), dim = (i - qi * (D / 4)) * 4;
          if (TAIL && dim >= p.d) continue;
          f32x4 f{0.f, 0.f, 0.f, 0.f};
          float top_q = -INFINITY, sum_q = 0.f;
#pragma unroll
          for (int x = 0; x < NW; ++x) {
            f += *reinterpret_cast<const f32x4*>(lds + (x * QB + qi) * OW + dim);
            top_q = fmaxf(top_q, ms[x * QB + qi]);
          }
#pragma unroll
          for (int x = 0; x < NW; ++x) {
            const float mx = ms[x * QB + qi];
            sum_q += ms[(NW + x) * QB + qi] * (mx == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mx - top_q));
          }
          if (complete) {
            const float scale = CODES && p.v_scale ? p.v_scale[done.head] : 1.f;
            const float out[4] = {f[0], f[1], f[2], f[3]};
            store_row<T>(p, done.r, done.head * p.group + done.q0 + qi, dim, out, sum_q, scale);
          } else {
            *reinterpret_cast<f32x4*>(p.part + (slot * q_max + qi) * p.d + dim) = f;
            if (dim == 0) {
              float* stats = p.part + 2 * (long)G * q_max * p.d + (slot * q_max + qi) * 2;
              stats[0] = top_q;
              stats[1] = sum_q;
            }
          }
        }
        // where this workgroup begins in a unit that the one before it began: the unit's row, number and workgroups
        if (tid == 0 && done.a < begin && (long)total * (w - 1) / W <= done.a)
          p.border[w] = int4{done.r, done.unit, w - 1, (int)(((long)done.b * W - 1) / total)};
        __syncthreads();                                  // (LDS is read)
      }
      if (!more) break;
      wv.run(p, u);
      done = u;
      at = u.stop;
    }
  }
  // rows that have nothing to attend to, or no slot
  if (p.whole) {
    if (!active && w == u.r * units && (u.row.slot >= 0 || p.fill)) zero_row<T>(p, u.r);
  } else {
    for (int r = w; r < p.rows; r += G) {
      const Row row = row_of(p, r);
      if (row.tiles <= 0 && (row.slot >= 0 || p.fill)) zero_row<T>(p, r);
    }
  }
}

// The parts of a unit that several workgroups have, in their order.  Where a unit has few, a wave joins those of a query head; where it has many, a workgroup those
// of 32 of its dimensions.
struct Parts {
  int row, head, q0, first, count;
  const float *stats;
  const PagedParams& p;
  int q_max;
  // u: row, unit, first and last workgroup
  __device__ __forceinline__ Parts(const PagedParams& pp, const int4 u, int G) : p(pp) {
    row = u.x;
    head = u.y / p.blocks;
    q0 = (u.y - head * p.blocks) * QB;
    first = u.z;
    count = u.w - u.z + 1;
    q_max = p.group < QB ? p.group : QB;
    stats = p.part + 2 * (long)G * q_max * p.d;
  }
  __device__ __forceinline__ long slot(int i, int qi) const { return (2 * (long)(first + i) + (i == 0 ? 1 : 0)) * q_max + qi; }
  __device__ __forceinline__ float2 stat(int i, int qi) const { return *reinterpret_cast<const float2*>(stats + slot(i, qi) * 2); }
  __device__ __forceinline__ const float* outputs(int i, int qi) const { return p.part + slot(i, qi) * p.d; }
};

template <int D, typename T, bool CODES>
__global__ __launch_bounds__(NW * 64) void join_few(const PagedParams p, const int G) {
  constexpr int N = D / 64;
  const Parts u(p, p.border[blockIdx.x + 1], G);
  const int lane = threadIdx.x & 63, qi = blockIdx.y * NW + (threadIdx.x >> 6);
  if (u.row < 0 || qi >= u.q_max || qi >= p.group - u.q0) return;
  const int dim = lane * N, at = dim < p.d ? dim : 0;
  float f[N] = {}, top = -INFINITY, sum = 0.f;
  for (int base = 0; base < u.count; base += 64) {      // (a lane a part; the maximum only moves between rounds of 64)
    const float2 s = base + lane < u.count ? u.stat(base + lane, qi) : float2{-INFINITY, 0.f};
    float now = s.x;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) now = fmaxf(now, __shfl_xor(now, o, 64));
    now = fmaxf(now, top);
    const float old = top == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(top - now), by = s.x == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(s.x - now);
    top = now;
    float more = s.y * by;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) more += __shfl_xor(more, o, 64);
    sum = sum * old + more;
#pragma unroll
    for (int e = 0; e < N; ++e) f[e] *= old;
    const int n = u.count - base < 64 ? u.count - base : 64;
    for (int i = 0; i < n; i += 4) {                    // four on their way at a time
      float x[4][N];
#pragma unroll
      for (int k = 0; k < 4; ++k) __builtin_memcpy(x[k], u.outputs(base + (i + k < n ? i + k : i), qi) + at, sizeof(x[k]));
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float w = __shfl(by, i + k < n ? i + k : i, 64);
        if (i + k < n)
#pragma unroll
          for (int e = 0; e < N; ++e) f[e] += x[k][e] * w;
      }
    }
  }
  if (dim < p.d) store_row<T>(p, u.row, u.head * p.group + u.q0 + qi, dim, f, sum, CODES && p.v_scale ? p.v_scale[u.head] : 1.f);
}

template <typename T, bool CODES>
__global__ __launch_bounds__(JT) void join_many(const PagedParams p, const int G) {
  constexpr int DL = 8, GR = JT / DL;                   // lanes of 32 dimensions, groups that take parts in turn
  // there are few rows (fewer units than a sixteenth of the workgroups): a lane has one's tiles, and with them where this workgroup's unit lies in the line
  static_assert(MOST / 16 <= 64);
  const int units = p.kv_heads * p.blocks, r = blockIdx.x / units, unit = blockIdx.x - r * units, at_lane = threadIdx.x & 63;
  const int tiles = at_lane < p.rows ? row_of(p, at_lane).tiles : 0;
  int before = tiles;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(before, o, 64);
    if (at_lane >= o) before += y;
  }
  const int total = __shfl(before, 63, 64) * units, here = __shfl(tiles, r, 64), a = (__shfl(before, r, 64) - here) * units + unit * here, W = total < G ? total : G;
  if (here == 0) return;
  const Parts u(p, int4{r, unit, (int)(((long)(a + 1) * W - 1) / total), (int)(((long)(a + here) * W - 1) / total)}, G);
  const int qi = blockIdx.y;
  if (u.count < 2 || qi >= p.group - u.q0) return;
  __shared__ float weight[MOST], red[JT / 64], sums[JT / 64];
  __shared__ f32x4 outs[GR][DL];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, parts = u.count;
  const int g = tid / DL, dim = blockIdx.z * 32 + (tid - g * DL) * 4, at = dim < p.d ? dim : 0;
  // (the outputs of the first parts do not wait for the weights)
  f32x4 x[4];
  auto request = [&](int i) {
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = *reinterpret_cast<const f32x4*>(u.outputs(i + k * GR < parts ? i + k * GR : 0, qi) + at);
  };
  request(g);
  // what every part's outputs and sum are multiplied with
  float top = -INFINITY, sum = 0.f;
  for (int i = tid; i < parts; i += JT) top = fmaxf(top, weight[i] = u.stat(i, qi).x);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
  if (lane == 0) red[wave] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < JT / 64; ++i) top = fmaxf(top, red[i]);
  for (int i = tid; i < parts; i += JT) {
    const float mx = weight[i], by = mx == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mx - top);    // (its own: nobody else reads it before the barrier)
    weight[i] = by;
    sum += u.stat(i, qi).y * by;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
  if (lane == 0) sums[wave] = sum;
  __syncthreads();
  f32x4 f{0.f, 0.f, 0.f, 0.f};
  for (int i = g; i < parts;) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (i + k * GR < parts) f += x[k] * weight[i + k * GR];
    i += 4 * GR;
    if (i < parts) request(i);
  }
  outs[g][tid - g * DL] = f;
  __syncthreads();
#pragma unroll
  for (int s = GR / 2; s > 0; s >>= 1) {
    if (g < s) outs[g][tid - g * DL] += outs[g + s][tid - g * DL];
    __syncthreads();
  }
  if (g > 0 || dim >= p.d) return;
  sum = 0.f;
#pragma unroll
  for (int i = 0; i < JT / 64; ++i) sum += sums[i];
  const float out[4] = {outs[0][tid][0], outs[0][tid][1], outs[0][tid][2], outs[0][tid][3]};
  store_row<T>(p, u.row, u.head * p.group + u.q0 + qi, dim, out, sum, CODES && p.v_scale ? p.v_scale[u.head] : 1.f);
}

// Workgroups: as many as run at once (D 256: one a CU), but no more than there can be tiles.
// Where the table or the window has room for at most WHOLE tiles (how long the sequences are the host does not know), a workgroup has a unit, and there is no second launch: 4 sequences of 300 tokens on 8 key heads 8.9 us where line and join take 7.4 + 4.0, of 470 10.5 and 7.5 + 4.0, 256 of 300
// 61.5 and 57.8 + 3.9 (and 3 of the host's for the second launch).
// `many`: a unit has more than 16 parts or so, the workgroups by the units.  us of the join, by a wave a query head and by 32 dimensions a workgroup: 512 workgroups, heads of 128,
// 4 units 23.1 and 4.3, 16 7.5 and 4.3, 24 6.2 and 4.9, 32 5.1 and 5.1, 64 4.1 and 6.7; 768, heads of 64, 32 units 5.0 and 4.3, 48 4.4 and 4.9.
struct Plan { long workgroups; bool parts, many; };

Plan plan_of(int64_t rows, int64_t kv_heads, int64_t group, int64_t d, int64_t span, int64_t window, bool codes) {
  if (window > 0 && window + TILE - 1 < span) span = window + TILE - 1;          // (wherever it begins in a tile)
  const long tiles = (span + TILE - 1) / TILE, units = rows * kv_heads * ((group + QB - 1) / QB);
  const long at_once = 256 * wgs_a_cu((int)d, codes), n = units * tiles < at_once ? units * tiles : at_once;
  if (tiles <= WHOLE && units <= 1 << 20) return Plan{units, false, false};
  return Plan{n, true, units * 16 < n};
}

// whether all tiles can be counted in 31 bits
bool line_fits(int64_t rows, int64_t kv_heads, int64_t group, int64_t span) {
  return rows * kv_heads * ((group + QB - 1) / QB) <= (1L << 30) / ((span + TILE - 1) / TILE);
}

int64_t bytes_of(const Plan& plan, int64_t group, int64_t d) {
  if (!plan.parts) return 0;
  const int64_t q = group < QB ? group : QB;
  return plan.workgroups * 16 + 2 * plan.workgroups * q * (d + 2) * 4;
}

template <int D, typename T, bool CODES, bool EIGHT, bool TAIL>
int run(const PagedParams& p, const Plan& plan, hipStream_t s) {
  constexpr int lds = (NW * QB * (D + 4) + 2 * NW * QB) * 4;
  if (lds > 65536) {
    const hipError_t e = kh_allow_lds<attend<D, T, CODES, EIGHT, TAIL>>(lds);
    if (e != hipSuccess) return (int)e;
  }
  kh_launch(KH_TAG_PAGED_ATTENTION, attend<D, T, CODES, EIGHT, TAIL>, dim3((unsigned)plan.workgroups), dim3(NW * 64), lds, s, p);
  if (plan.parts) {
    const hipError_t e = hipGetLastError();             // (the launch behind it reads what it writes)
    if (e != hipSuccess) return (int)e;
    const unsigned borders = (unsigned)plan.workgroups - 1, queries = p.group < QB ? p.group : QB;
    if (plan.many) kh_launch(KH_TAG_PAGED_JOIN, join_many<T, CODES>, dim3((unsigned)(p.rows * p.kv_heads * p.blocks), queries, (unsigned)(p.d + 31) / 32), dim3(JT), 0, s, p, (int)plan.workgroups);
    else kh_launch(KH_TAG_PAGED_JOIN, join_few<D, T, CODES>, dim3(borders, (queries + NW - 1) / NW), dim3(NW * 64), 0, s, p, (int)plan.workgroups);
  }
  KH_RETURN_LAST_ERROR();
}
template <int D, typename T, bool CODES>
int run(const PagedParams& p, const Plan& plan, hipStream_t s) {
  if (p.page % 8 == 0) return p.d == D ? run<D, T, CODES, true, false>(p, plan, s) : run<D, T, CODES, true, true>(p, plan, s);
  return p.d == D ? run<D, T, CODES, false, false>(p, plan, s) : run<D, T, CODES, false, true>(p, plan, s);
}
template <typename T, bool CODES>
int run(const PagedParams& p, const Plan& plan, hipStream_t s) {
  return p.d <= 64 ? run<64, T, CODES>(p, plan, s) : p.d <= 128 ? run<128, T, CODES>(p, plan, s) : run<256, T, CODES>(p, plan, s);
}

}  // namespace

KH_EXPORT int64_t kh_paged_attention_workspace_bytes(int64_t rows, int64_t heads, int64_t kv_heads, int64_t d, int64_t span) {
  if (rows <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || d <= 0 || span <= 0) return KH_ERR_INVALID_ARG;
  if (d % 8 != 0 || d > 256) return KH_ERR_UNSUPPORTED;
  if (rows > (1L << 24) || heads > (1L << 16) || span > (1L << 30)) return KH_ERR_TOO_LARGE;
  if (!line_fits(rows, kv_heads, heads / kv_heads, span)) return KH_ERR_TOO_LARGE;
  return bytes_of(plan_of(rows, kv_heads, heads / kv_heads, d, span, 0, true), heads / kv_heads, d);   // (nothing has more workgroups than e4m3 without a window)
}

KH_EXPORT int kh_paged_attention(const void* q, void* o, const KhPagedCache* cache, int64_t layer, const int32_t* slots, const int32_t* lengths,
                                 void* workspace, int64_t rows, int64_t heads, int64_t ldq, int64_t ldo, int64_t window, float scale, int flags, int type,
                                 void* stream) {
  const int rc = kh_cache_check(cache);
  if (rc != KH_OK) return rc;
  const KhPagedCache& c = *cache;
  if (!q || !o || rows <= 0 || heads <= 0 || heads % c.kv_heads != 0 || window < 0 || (flags & ~1) || type < 0 || type > 1) return KH_ERR_INVALID_ARG;
  if (layer < 0 || layer >= c.layers || ldq < heads * c.d || ldo < heads * c.d || (!slots && rows > c.slots)) return KH_ERR_INVALID_ARG;
  if (c.type != KH_E4M3 && c.type != type) return KH_ERR_UNSUPPORTED;
  if ((((uintptr_t)q | (uintptr_t)o) & 1) || (((uintptr_t)slots | (uintptr_t)lengths) & 3) || !kh_aligned16(workspace)) return KH_ERR_ALIGNMENT;
  if (rows > (1L << 24) || heads > (1L << 16)) return KH_ERR_TOO_LARGE;
  const long group = heads / c.kv_heads, e = kh_cache_element(c);
  if (!line_fits(rows, c.kv_heads, group, c.width * c.page)) return KH_ERR_TOO_LARGE;
  if (window > 1L << 30) window = 0;                    // (longer than any sequence)
  const Plan plan = plan_of(rows, c.kv_heads, group, c.d, c.width * c.page, window, c.type == KH_E4M3);
  if (plan.parts && !workspace) return KH_ERR_INVALID_ARG;
  PagedParams p{q, (const char*)c.k + layer * c.k_layer * e, (const char*)c.v + layer * c.v_layer * e, o, c.table, lengths, c.lengths, slots,
                c.k_scale ? c.k_scale + layer * c.kv_heads : nullptr, c.v_scale ? c.v_scale + layer * c.kv_heads : nullptr,
                plan.parts ? (float*)((char*)workspace + plan.workgroups * 16) : nullptr, plan.parts ? (int4*)workspace : nullptr, ldq, ldo, (uint32_t)(c.k_page * e), (uint32_t)(c.k_token * e), (uint32_t)(c.v_page * e),
                (uint32_t)(c.v_token * e), c.k_head * e, c.v_head * e,
                (int)rows, (int)c.kv_heads, (int)group, (int)((group + QB - 1) / QB), (int)c.d, (int)c.slots, (int)c.width, (int)c.pages, (int)c.page,
                (int)window, scale * 1.4426950408889634f, flags & 1, 0, !plan.parts, 0, KhDivide((uint32_t)c.page)};
  // (32 sequences of 4096 tokens, 8 heads of 80 and 96 in bf16: 82 -> 77 us and 84 -> 76; heads of whole lines 91 -> 94)
  p.shared_lines = c.kv_heads > 1 && c.k_head * e % 128 != 0;
  p.q_aligned = kh_aligned16(q) && ldq % 8 == 0;
  hipStream_t s = (hipStream_t)stream;
  const bool codes = c.type == KH_E4M3;
  if (type == 0) return codes ? run<bf16_t, true>(p, plan, s) : run<bf16_t, false>(p, plan, s);
  return codes ? run<f16_t, true>(p, plan, s) : run<f16_t, false>(p, plan, s);
}
