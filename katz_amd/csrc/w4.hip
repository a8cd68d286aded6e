// K12: weights in 4 bits with a scale (and a zero point) for each group of 32, 64 or 128 along a row:
//   w[n][k] = s[n][k / G] * (q[n][k] - z[n][k / G]),   z = 8 where no zero points are given
// Quantisation, the values that codes stand for, and the linear of few and of many rows with the adapters of K1 beside it:
//   y = x w^T + b + ((x A_cat^T) * col_scale) B_cat^T (+ residual)
//
// A row of codes is its weights in order, two to a byte (the even one in the low half), filled up to 32 of them; a row of scales or
// zero points is filled up to 4.  Scales are bf16 whatever the activations' type: they have the weights' range, and the codes are
// chosen against the rounded scale.
#include "kh_common.h"
#include <type_traits>

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// Eight elements at an address that is aligned to one of them; those at and behind `left` are zero and not read.
template <typename T>
__device__ __forceinline__ void load8(const T* at, long left, T (&v)[8]) {
  if (left >= 8) {
    __builtin_memcpy(v, at, sizeof(v));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < left ? at[e] : (T)0.f;
  }
}

// Sixteen bytes that pass by: weights that are quantised, the values of codes.  Kept out of the caches they leave room for what is read again, and lines that are
// written whole need not be fetched: values of 16384 x 8192 110 -> 48 us, their codes 91 -> 76.  Of rows that are not aligned (16384 x 8191) by pieces of eight
// rather than by elements 201 -> 69.
template <typename T>
__device__ __forceinline__ void load8_once(const T* at, long left, T (&v)[8]) {
  if (left >= 8 && ((uintptr_t)at & 15) == 0) {
    u32x4 t[sizeof(v) / 16];
#pragma unroll
    for (unsigned i = 0; i < sizeof(v) / 16; ++i) t[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(at) + i);
    __builtin_memcpy(v, t, sizeof(v));
  } else {
    load8<T>(at, left, v);
  }
}
template <typename T>
__device__ __forceinline__ void store8_once(T* at, int left, const T (&v)[8]) {
  if (left >= 8 && ((uintptr_t)at & 15) == 0) {
    u32x4 t[sizeof(v) / 16];
    __builtin_memcpy(t, v, sizeof(v));
#pragma unroll
    for (unsigned i = 0; i < sizeof(v) / 16; ++i) __builtin_nontemporal_store(t[i], reinterpret_cast<u32x4*>(at) + i);
  } else if (left >= 8) {
    __builtin_memcpy(at, v, sizeof(v));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < left) at[e] = v[e];
  }
}

// ---------------------------------------------------------------- quantisation
// Rows are cut into pieces of eight, filled up to whole groups (or to a row of codes), and the pieces of all rows numbered through: a wave takes PT * 64 in a
// row, a thread one of every 64, all of whose loads are on their way before the first is used.  A group's G / 8 pieces lie in one wave, aligned.
constexpr int PT = 4;

struct Pieces {                      // of one row, and what divides a small number by that
  uint32_t per_row, magic;
  explicit Pieces(long n) : per_row((uint32_t)n), magic(n < 4 * PT * 64 ? (uint32_t)((1ull << 32) / (uint64_t)n + 1) : 0) {}
};
// Row and piece of the i-th of a thread's.  (A workgroup's first row comes from one long division; from there on numbers are below per_row + 1024.)
__device__ __forceinline__ void piece_of(const Pieces& d, int i, long& row, int& u) {
  const long first = (long)blockIdx.x * (4 * PT * 64);
  const long r0 = first / d.per_row;
  const uint32_t local = (uint32_t)(first - r0 * d.per_row) + (threadIdx.x >> 6) * (PT * 64) + i * 64 + (threadIdx.x & 63);
  const uint32_t r = d.per_row >= 4 * PT * 64 ? (local >= d.per_row ? 1u : 0u) : __umulhi(local, d.magic);   // (exact: local * per_row < 2^32)
  row = r0 + r;
  u = (int)(local - r * d.per_row);
}

struct QuantParams {
  const void* w;
  uint8_t* q;
  bf16_t* scale;
  uint8_t* zero;
  long N;
  int K, groups, gstride, words;   // words: of eight codes in a row
  Pieces pieces;
};

// The largest of a group of 4, 8 or 16 lanes, in all of them (bits of numbers that are not negative, which order like integers; a NaN is the largest).
template <int GT>
__device__ __forceinline__ int group_max(int v) {
#if __HIP_DEVICE_COMPILE__
  auto with = [](int x, auto ctrl) {
    const int y = __builtin_amdgcn_update_dpp(0, x, decltype(ctrl)::value, 0xf, 0xf, false);
    return x > y ? x : y;
  };
  v = with(v, std::integral_constant<int, 0xb1>{});    // quad_perm 1,0,3,2
  v = with(v, std::integral_constant<int, 0x4e>{});    // quad_perm 2,3,0,1
  if (GT >= 8) v = with(v, std::integral_constant<int, 0x141>{});    // row_half_mirror
  if (GT >= 16) v = with(v, std::integral_constant<int, 0x140>{});   // row_mirror
#endif
  return v;
}

template <typename T, int G, bool ZERO>
__global__ __launch_bounds__(256) void quantize_kernel(const QuantParams p) {
  constexpr int GT = G / 8;
  long row[PT];
  int u[PT];
  T v[PT][8];
#pragma unroll
  for (int i = 0; i < PT; ++i) {
    piece_of(p.pieces, i, row[i], u[i]);
    const long r = row[i] < p.N ? row[i] : p.N - 1;
    load8_once<T>((const T*)p.w + r * p.K + (long)u[i] * 8, p.K - u[i] * 8, v[i]);
  }
#pragma unroll
  for (int i = 0; i < PT; ++i) {
    if (row[i] >= p.N) break;        // (whole groups)
    float f[8];
    int hi = 0, lo = 0;              // bits of the largest value and of the largest negated one, or of the largest magnitude
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      f[e] = (float)v[i][e];
      const int bits = __float_as_int(f[e]);
      hi = max(hi, ZERO ? bits : bits & 0x7fffffff);
      if (ZERO) lo = max(lo, bits ^ (int)0x80000000);
    }
    hi = group_max<GT>(hi);
    if (ZERO) lo = group_max<GT>(lo);
    const float below = ZERO ? __int_as_float(lo) : 0.f;
    const float wide = ZERO ? (__int_as_float(hi) + below) / 15.f : __int_as_float(hi) / 7.f;
    const bf16_t sb = (bf16_t)wide;
    const float s = (float)sb;
    float z = 8.f;
    uint32_t word = 0;
    auto code = [](float r, float z) { return (uint32_t)(int)fminf(fmaxf(r + z, 0.f), 15.f); };
    if (s > 1e-30f && s < 1e30f) {
      // The quotient as a division gives it (halves have to stay halves): the reciprocal is rounded correctly, so one step from its product is the rounded
      // quotient (Markstein).
      const float inv = 1.f / s;
      auto level = [&](float a) {
        const float q = a * inv;
        return rintf(fmaf(fmaf(-q, s, a), inv, q));
      };
      if (ZERO) z = fminf(fmaxf(level(below), 0.f), 15.f);
#pragma unroll
      for (int e = 0; e < 8; ++e) word |= code(level(f[e]), z) << (4 * e);
    } else {                         // nothing but zeros, very small or very large numbers, or none: rint(a / s), 0 where that is no number
      auto level = [&](float a) {
        const float r = s > 0.f ? rintf(a / s) : 0.f;
        return r == r ? r : 0.f;
      };
      if (ZERO) z = fminf(fmaxf(level(below), 0.f), 15.f);
#pragma unroll 1
      for (int e = 0; e < 8; ++e) word |= code(level(e < 4 ? (e < 2 ? (e == 0 ? f[0] : f[1]) : (e == 2 ? f[2] : f[3])) : (e < 6 ? (e == 4 ? f[4] : f[5]) : (e == 6 ? f[6] : f[7]))), z) << (4 * e);
    }
    const int left = p.K - u[i] * 8;
    if (u[i] < p.words) {            // (behind the last weight: filling)
      if (left < 8) word = left <= 0 ? 0u : word & ((1u << (4 * left)) - 1u);
      __builtin_nontemporal_store(word, reinterpret_cast<uint32_t*>(p.q) + row[i] * p.words + u[i]);
    }
    if (u[i] % GT == 0) {
      const int g = u[i] / GT;
      p.scale[row[i] * p.gstride + g] = sb;
      if (ZERO) p.zero[row[i] * p.gstride + g] = (uint8_t)(int)z;
      if (g == p.groups - 1)
        for (int k = p.groups; k < p.gstride; ++k) {
          p.scale[row[i] * p.gstride + k] = (bf16_t)0.f;
          if (ZERO) p.zero[row[i] * p.gstride + k] = 0;
        }
    }
  }
}

// ---------------------------------------------------------------- the values that codes stand for
struct ValueParams {
  const uint32_t* q;
  const bf16_t* scale;
  const uint8_t* zero;
  void* out;
  long N;
  int K, gshift, gstride;            // gshift: log2 of a group's words of eight codes
  Pieces pieces;                     // words
};

template <typename T>
__global__ __launch_bounds__(256) void values_kernel(const ValueParams p) {
  long row[PT];
  int u[PT], z[PT];
  uint32_t word[PT];
  bf16_t s[PT];
#pragma unroll
  for (int i = 0; i < PT; ++i) {
    piece_of(p.pieces, i, row[i], u[i]);
    const long r = row[i] < p.N ? row[i] : p.N - 1;
    const int last = (p.K - 1) >> (3 + p.gshift), g = u[i] >> p.gshift;      // (words behind the last weight may lie behind the last group)
    word[i] = p.q[r * p.pieces.per_row + u[i]];
    s[i] = p.scale[r * p.gstride + (g < last ? g : last)];
    z[i] = p.zero ? p.zero[r * p.gstride + (g < last ? g : last)] : 8;
  }
#pragma unroll
  for (int i = 0; i < PT; ++i) {
    if (row[i] >= p.N) break;
    const int left = p.K - u[i] * 8;
#if __HIP_DEVICE_COMPILE__
    asm volatile("" : "+v"(z[i]));   // (masked here: at its load the compiler would wait for it, and 16384 x 8191 take 78 us instead of 71)
#endif
    const int zero = z[i] & 15;      // (as the linear takes it)
    T v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (T)((float)s[i] * (float)((int)((word[i] >> (4 * e)) & 15u) - zero));
    store8_once<T>((T*)p.out + row[i] * p.K + u[i] * 8, left, v);
  }
}

// ---------------------------------------------------------------- the linear
// Codes become operands of the matrix unit without a conversion: below the bits of a power of two P = 16, in the four upper bits of its mantissa, a code makes the
// 16 bits the number P + q, so two shifted and masked nibbles are two operands.  A second product of x with the constant -(P + z) takes P and z away again,
// exactly, in the same accumulator; scales are applied to a group's sum in 32 bits.  P is the smallest power with the codes in one binade: what the sum carries of it
// costs 32-bit sums the upper bits.  (Codes in the lower bits, under 128 in bf16 and 1024 in fp16, are one shift of eight instructions less, and left an fp16 row of x with
// a mean of 3 twice the error of its rounding.)
// The nibbles of a word come out as pairs (0,4) (1,5) (2,6) (3,7); x is put into the same order.
template <typename T> struct Num;
template <> struct Num<bf16_t> {
  static constexpr uint32_t P16 = 0x41804180u, P32 = 0x42004200u, NEG = 0x80008000u;
  static constexpr int UNIT = 3;     // where the bit of 1 is in 16 .. 32 (one further down in 32 .. 64)
  typedef bf16x8 V8;
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
#if __HIP_DEVICE_COMPILE__
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
#else
    return c;
#endif
  }
};
template <> struct Num<_Float16> {
  static constexpr uint32_t P16 = 0x4c004c00u, P32 = 0x50005000u, NEG = 0x80008000u;
  static constexpr int UNIT = 6;
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
#if __HIP_DEVICE_COMPILE__
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
#else
    return c;
#endif
  }
};

// elements 0..7 in the order 0,4,1,5,2,6,3,7
__device__ __forceinline__ u32x4 interleaved(const u32x4 v) {
#if __HIP_DEVICE_COMPILE__
  return u32x4{__builtin_amdgcn_perm(v[2], v[0], 0x05040100u), __builtin_amdgcn_perm(v[2], v[0], 0x07060302u),
               __builtin_amdgcn_perm(v[3], v[1], 0x05040100u), __builtin_amdgcn_perm(v[3], v[1], 0x07060302u)};
#else
  return v;
#endif
}

// The mask and the power of two in registers: one instruction then takes both (and-or), where two constants in the code would take two.
template <typename T>
struct Unpack {
  static constexpr int U = Num<T>::UNIT;
  uint32_t mask = 0x000f000fu << U, power = Num<T>::P16;
  __device__ __forceinline__ Unpack() {
#if __HIP_DEVICE_COMPILE__
    asm("" : "+s"(mask));
    asm("" : "+v"(power));
#endif
  }
  __device__ __forceinline__ u32x4 operator()(uint32_t word) const {
    const uint32_t second = U > 4 ? word << (U - 4) & mask : word >> (4 - U) & mask;
    return u32x4{((word << U) & mask) | power, second | power, ((word >> (8 - U)) & mask) | power, ((word >> (12 - U)) & mask) | power};
  }
};

// Lane group g (of 16 lanes) holds words 4g .. 4g+3 of a block of 128 codes of its row; afterwards words g, g+4, g+8, g+12: the k-step
// j of 32 codes takes register j of all four groups.
__device__ __forceinline__ u32x4 across_groups(u32x4 v) {
#if __HIP_DEVICE_COMPILE__
  auto a = __builtin_amdgcn_permlane32_swap(v[0], v[2], false, false);
  auto b = __builtin_amdgcn_permlane32_swap(v[1], v[3], false, false);
  auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
  auto d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
  return u32x4{c[0], c[1], d[0], d[1]};
#else
  return v;
#endif
}

struct LinParams {
  const void* x;
  const uint8_t* q;
  const bf16_t* scale;
  const uint8_t* zero;
  const void *bias, *b_cat, *residual;
  const float* t;          // [t_splits][M][R]
  void* y;
  long M, N;
  int K, R, t_splits, row_bytes, gstride;
  int dma;                 // rows of x (and of A) are aligned to four bytes
  const void* a_cat;       // few rows and a small A: every workgroup computes t by itself and keeps it in LDS from `t_at` on; else NULL
  const float* col_scale;
  int t_at;
  int b_dma;               // B_cat is aligned to four bytes
  int once;                // y of 8 MB and more is stored past the caches (616 x 10240 with rank 96 and a residual: 40.6 -> 37.4 us)
};

// The rank-R product of a 16 x 16 tile in 32 bits, a step of 16 ranks: t from LDS, or [M][R] in `splits` parts, B_cat rows of T.
template <typename T>
__device__ __forceinline__ f32x4 rank_step(const LinParams& p, const float* own, long m, long n, int r, f32x4 acc) {
  f32x4 t = f32x4{0.f, 0.f, 0.f, 0.f};
  if (own) {
    t = *reinterpret_cast<const f32x4*>(own);
  } else {
    const float* tr = p.t + m * p.R + r;
    const long part = p.M * p.R;
    for (int sp = 0; sp < p.t_splits; sp += 4) {      // four on their way at a time, added in order
      f32x4 v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = sp + i < p.t_splits ? *reinterpret_cast<const f32x4*>(tr + (sp + i) * part) : f32x4{0.f, 0.f, 0.f, 0.f};
      t = (((t + v[0]) + v[1]) + v[2]) + v[3];
    }
  }
  T b[4];
  __builtin_memcpy(b, (const T*)p.b_cat + n * p.R + r, sizeof(b));
#if __HIP_DEVICE_COMPILE__
#pragma unroll
  for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(t[e], (float)b[e], acc, 0, 0, 0);
#endif
  return acc;
}

template <int BYTES> struct Word;
template <> struct Word<1> { typedef uint8_t type; };
template <> struct Word<2> { typedef uint16_t type; };
template <> struct Word<4> { typedef uint32_t type; };
template <> struct Word<8> { typedef uint64_t type; };

typedef __attribute__((address_space(3))) void* lptr_t;

template <int VM>
__device__ __forceinline__ void wait_vm() {  // vmcnt = VM, the other counters unconstrained (gfx9 encoding)
  __builtin_amdgcn_s_waitcnt((VM & 15) | (7 << 4) | (15 << 8) | ((VM >> 4) << 14));
  asm volatile("" ::: "memory");
}

// What a wave keeps of a block of 128 codes in LDS: codes of NB x 16 rows, x in the order of its operands, scales, zero points.  P loads.
template <int G, bool ZERO, int MB, int NB, bool FOUR>
struct Stage {
  static constexpr int X = FOUR ? 1 : 4 * MB;                // loads of 1 KB
  static constexpr int S = G == 32 ? 2 : 1, Z = ZERO ? 1 : 0;  // loads of 256 bytes: four bytes of a row, the lane groups take a tile of 16 rows each
  static constexpr int P = NB + X + S + Z;
  static constexpr int WAT = 0, XAT = NB * 1024, SAT = XAT + X * 1024, ZAT = SAT + S * 256, BYTES = ZAT + Z * 256;
};

// t = (x A^T) * col_scale of up to 16 rows and RT tiles of 16 ranks into `tl`: a wave takes every LW-th step of 32 k, OWN_DEEP - 1 on their way ahead of the one that
// is multiplied (as below, in a part of LDS of its own), and the waves are summed in order.
constexpr int OWN_DEEP = 3, OWN_PITCH = 64 + 4;                 // of tl
constexpr int own_wave(int rt) { return OWN_DEEP * (1 + rt) * 1024; }
template <typename T, int LW, int RT>
__device__ __forceinline__ void own_ranks(const LinParams& p, const T* x0, int rows, char* smem, float* tl) {
#if __HIP_DEVICE_COMPILE__
  constexpr int UNIT = (1 + RT) * 1024, R = RT * 16;            // a tile of x and those of A, 1 KB each
  static_assert(16 * (R + 1) * 4 <= OWN_DEEP * UNIT && R <= OWN_PITCH - 4, "a wave's sums");
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l = lane & 15, g = lane >> 4, dr = lane >> 2, dp = lane & 3, from = (l * 4 + g) * 16;
  const T* a0 = (const T*)p.a_cat;
  const __amdgpu_buffer_rsrc_t rx = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(x0), 0, (int)(rows * p.K * 2), 0x00020000);
  const __amdgpu_buffer_rsrc_t ra = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(a0), 0, (int)(R * p.K * 2), 0x00020000);
  const int xo = ((dr < rows ? dr : rows - 1) * p.K + dp * 8) * 2, ao = (dr * p.K + dp * 8) * 2;
  const int steps = (p.K + 31) / 32, full = p.dma ? p.K / 32 : 0, mine = wave < full ? (full - 1 - wave) / LW + 1 : 0;
  char* const here = smem + wave * own_wave(RT);
  f32x4 acc[RT];
#pragma unroll
  for (int j = 0; j < RT; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto fetch = [&](int i, int st) {
    const int kb = (wave + i * LW) * 64;
    char* to = here + st * UNIT;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rx, (lptr_t)to, 16, xo, kb, 0, 0);
#pragma unroll
    for (int j = 0; j < RT; ++j) __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (lptr_t)(to + 1024 + j * 1024), 16, ao, j * 32 * p.K + kb, 0, 0);
  };
  auto use = [&](int st) {
    const char* at = here + st * UNIT + from;
    const u32x4 x = *reinterpret_cast<const u32x4*>(at);
#pragma unroll
    for (int j = 0; j < RT; ++j) acc[j] = Num<T>::mfma(x, *reinterpret_cast<const u32x4*>(at + 1024 + j * 1024), acc[j]);
  };
  if (mine > 0) fetch(0, 0);
  if (mine > 1) fetch(1, 1);
  int st = 0, i = 0;
  auto next = [&]() { st = st == 2 ? 0 : st + 1; };
  for (; i + 2 < mine; ++i) {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");          // the step before has been read; its place is the next one's
    fetch(i + 2, st == 0 ? 2 : st - 1);
    wait_vm<2 * (1 + RT)>();
    use(st);
    next();
  }
  if (i + 1 < mine) { wait_vm<1 + RT>(); use(st); next(); ++i; }
  if (i < mine) { wait_vm<0>(); use(st); }
  for (int ks = full + (wave - full % LW + LW) % LW; ks < steps; ks += LW) {     // the end of the rows, or rows that are not aligned to four bytes
    const int k = ks * 32 + g * 8;
    T v[8];
    load8<T>(x0 + (long)(l < rows ? l : rows - 1) * p.K + k, (long)p.K - k, v);
    const u32x4 x = __builtin_bit_cast(u32x4, v);
#pragma unroll
    for (int j = 0; j < RT; ++j) {
      load8<T>(a0 + (long)(j * 16 + l) * p.K + k, (long)p.K - k, v);
      acc[j] = Num<T>::mfma(x, __builtin_bit_cast(u32x4, v), acc[j]);
    }
  }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  float* part = reinterpret_cast<float*>(here);
#pragma unroll
  for (int j = 0; j < RT; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) part[(g * 4 + e) * (R + 1) + j * 16 + l] = acc[j][e];
  __syncthreads();
  for (int id = threadIdx.x; id < rows * R; id += LW * 64) {
    const int r = id / R, c = id % R;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < LW; ++w) v += reinterpret_cast<const float*>(smem + w * own_wave(RT))[r * (R + 1) + c];
    tl[r * OWN_PITCH + c] = v * p.col_scale[c];
  }
  __syncthreads();
#endif
}

// A few rows: NB * 16 columns of y (rows of codes) and MB * 16 rows of x to a workgroup.  Its LW waves take every LW-th block of 128 codes and are
// summed in order at the end.  A wave's blocks go straight to a ring of ST of its own in LDS, ST - 1 ahead of the one that is multiplied: nobody else
// reads them, so there is no barrier, and the loads in flight cost no registers.
// FOUR: at most four rows (MB 1), which lie at every fourth row of the product: then they are in the first register of every lane, and the other three
// need no scale.
template <typename T, int G, bool ZERO, int MB, int NB, int LW, int ST, bool FOUR>
__global__ __launch_bounds__(LW * 64) void w4_few_rows(const LinParams p) {
#if __HIP_DEVICE_COMPILE__
  extern __shared__ __attribute__((aligned(16))) char smem[];
  typedef Stage<G, ZERO, MB, NB, FOUR> Sg;
  constexpr int GB = 128 / G;        // groups in a block
  constexpr int SG = 4 / GB;         // k-steps in a group
  constexpr int E = FOUR ? 1 : 4;
  typedef typename Word<GB * 2>::type SW_t;
  typedef typename Word<GB>::type ZW_t;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l = lane & 15, g = lane >> 4;
  const long m0 = (long)blockIdx.y * (MB * 16), n0 = (long)blockIdx.x * (NB * 16);
  const int rows = (int)(p.M - m0 < MB * 16 ? p.M - m0 : MB * 16);
  // the workgroup's first rows, and what a lane is from there (below 2^31: K <= 2^24)
  const uint8_t* q0 = p.q + n0 * p.row_bytes;
  const bf16_t* s0 = p.scale + n0 * p.gstride;
  const uint8_t* z0 = ZERO ? p.zero + n0 * p.gstride : nullptr;
  const T* x0 = (const T*)p.x + m0 * p.K;
  const uint32_t last = (uint32_t)(p.N - 1 - n0 < NB * 16 - 1 ? p.N - 1 - n0 : NB * 16 - 1);
  // Loads to LDS: four lanes in a row take the 64 bytes of a row (a lane to every row instead costs three and a half times as much: 54 and 15 bytes a clock and CU
  // out of the L2); the reads put them in order.
  const int dr = lane >> 2, dp = lane & 3, from = (l * 4 + g) * 16;
  uint32_t qo[NB];
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const uint32_t r = j * 16 + dr;
    qo[j] = (r < last ? r : last) * (uint32_t)p.row_bytes + dp * 16;
  }
  const uint32_t mr = (g < NB ? g : NB - 1) * 16 + l, so = (mr < last ? mr : last) * (uint32_t)p.gstride;    // row whose scales the lane fetches
  int xm[MB];
  uint32_t xo[MB];
#pragma unroll
  for (int b = 0; b < MB; ++b) {
    const int r = FOUR ? l >> 2 : b * 16 + l, rd = b * 16 + dr;
    xm[b] = r < rows ? r : rows - 1;
    xo[b] = ((uint32_t)(rd < rows ? rd : rows - 1) * (uint32_t)p.K + dp * 8) * 2;
  }
  const uint32_t x4 = ((uint32_t)(g < rows ? g : rows - 1) * (uint32_t)p.K + l * 8) * 2;   // FOUR: row g, piece l
  const Unpack<T> unpack;
  const f32x4 none = f32x4{0.f, 0.f, 0.f, 0.f};
  f32x4 out[MB][NB];
#pragma unroll
  for (int b = 0; b < MB; ++b)
#pragma unroll
    for (int j = 0; j < NB; ++j) out[b][j] = none;

  auto multiply = [&](const u32x4 (&w0)[NB], const u32x4 (&x)[MB][4], const SW_t (&sw)[NB], const ZW_t (&zw)[NB], int groups) {
    u32x4 xv[MB][4];                          // groups: of this block; what rows of scales are filled up with is not used
#pragma unroll
    for (int b = 0; b < MB; ++b)
#pragma unroll
      for (int j = 0; j < 4; ++j) xv[b][j] = interleaved(x[b][j]);
    f32x4 base[MB][GB];                       // without zero points the constant is the same for all columns
    if (!ZERO) {
      constexpr uint32_t c = Num<T>::P16 | Num<T>::NEG | 0x00080008u << Num<T>::UNIT;
#pragma unroll
      for (int b = 0; b < MB; ++b)
#pragma unroll
        for (int i = 0; i < GB; ++i)
#pragma unroll
          for (int k = 0; k < SG; ++k) base[b][i] = Num<T>::mfma(xv[b][i * SG + k], u32x4{c, c, c, c}, k == 0 ? none : base[b][i]);
    }
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const u32x4 w = across_groups(w0[j]);
#pragma unroll
      for (int i = 0; i < GB; ++i) {
        const float s = i < groups ? bf16_bits_to_f32((uint32_t)(sw[j] >> (16 * i)) & 0xffffu) : 0.f;
        uint32_t c = 0;
        if (ZERO) c = (Num<T>::P16 | Num<T>::NEG) | ((uint32_t)(zw[j] >> (8 * i)) & 15u) * (0x10001u << Num<T>::UNIT);
        f32x4 acc[MB];
#pragma unroll
        for (int b = 0; b < MB; ++b) acc[b] = ZERO ? none : base[b][i];
#pragma unroll
        for (int k = 0; k < SG; ++k) {
          const u32x4 wv = unpack(w[i * SG + k]);
#pragma unroll
          for (int b = 0; b < MB; ++b) {
            acc[b] = Num<T>::mfma(xv[b][i * SG + k], wv, acc[b]);
            if (ZERO) acc[b] = Num<T>::mfma(xv[b][i * SG + k], u32x4{c, c, c, c}, acc[b]);
          }
        }
#pragma unroll
        for (int b = 0; b < MB; ++b)
#pragma unroll
          for (int e = 0; e < E; ++e) out[b][j][e] = fmaf(s, acc[b][e], out[b][j][e]);
      }
    }
  };

  const int full = p.dma ? p.K / 128 : 0, blocks = (p.row_bytes + 63) / 64;
  const int mine = wave < full ? (full - 1 - wave) / LW + 1 : 0;   // whole blocks of this wave
  char* ring = smem + wave * (ST * Sg::BYTES);
  float* const tl = reinterpret_cast<float*>(smem + p.t_at);
  if constexpr (MB == 1)
    if (p.a_cat) {
      if (p.R == 32) own_ranks<T, LW, 2>(p, x0, rows, smem, tl);
      else own_ranks<T, LW, 4>(p, x0, rows, smem, tl);
    }
  auto bytes = [](long n) { return (int)(uint32_t)(n < 0xffffffffL ? n : 0xffffffffL); };
  const __amdgpu_buffer_rsrc_t rq = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(q0), 0, bytes((p.N - n0) * p.row_bytes), 0x00020000);
  const __amdgpu_buffer_rsrc_t rx = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(x0), 0, bytes((p.M - m0) * p.K * 2), 0x00020000);
  const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<bf16_t*>(s0), 0, bytes((p.N - n0) * p.gstride * 2), 0x00020000);
  const __amdgpu_buffer_rsrc_t rz = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(ZERO ? z0 : q0), 0, bytes((p.N - n0) * p.gstride), 0x00020000);
  // the four bytes that hold a block's scales (128: half of them) or zero points
  auto s_word = [&](int kb) { return kb * GB * 2 & ~3; };
  auto z_word = [&](int kb) { return kb * GB & ~3; };
  auto fetch = [&](int i, int st) {           // the wave's i-th block into a stage
    const int kb = wave + i * LW;
    char* to = ring + st * Sg::BYTES;
#pragma unroll
    for (int j = 0; j < NB; ++j) __builtin_amdgcn_raw_ptr_buffer_load_lds(rq, (lptr_t)(to + Sg::WAT + j * 1024), 16, qo[j], kb * 64, 0, 0);
    if constexpr (FOUR) {
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rx, (lptr_t)(to + Sg::XAT), 16, x4, kb * 256, 0, 0);
    } else {
#pragma unroll
      for (int b = 0; b < MB; ++b)
#pragma unroll
        for (int j = 0; j < 4; ++j) __builtin_amdgcn_raw_ptr_buffer_load_lds(rx, (lptr_t)(to + Sg::XAT + (b * 4 + j) * 1024), 16, xo[b], kb * 256 + j * 64, 0, 0);
    }
#pragma unroll
    for (int j = 0; j < Sg::S; ++j) __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lptr_t)(to + Sg::SAT + j * 256), 4, so * 2, s_word(kb) + j * 4, 0, 0);
    if constexpr (ZERO) __builtin_amdgcn_raw_ptr_buffer_load_lds(rz, (lptr_t)(to + Sg::ZAT), 4, so, z_word(kb), 0, 0);
  };
  auto use = [&](int i, int st) {
    const int kb = wave + i * LW;
    const char* at = ring + st * Sg::BYTES;
    u32x4 w[NB], x[MB][4];
    SW_t sw[NB];
    ZW_t zw[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      w[j] = *reinterpret_cast<const u32x4*>(at + Sg::WAT + j * 1024 + from);
      const char* sa = at + Sg::SAT + (j * 16 + l) * 4;
      if constexpr (G == 32) sw[j] = (SW_t)*reinterpret_cast<const uint32_t*>(sa) | (SW_t)((uint64_t)*reinterpret_cast<const uint32_t*>(sa + 256) << 32);
      else sw[j] = (SW_t)(*reinterpret_cast<const uint32_t*>(sa) >> (kb * GB * 16 & 31));
      if constexpr (ZERO) zw[j] = (ZW_t)(*reinterpret_cast<const uint32_t*>(at + Sg::ZAT + (j * 16 + l) * 4) >> (kb * GB * 8 & 31));
    }
#pragma unroll
    for (int b = 0; b < MB; ++b)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        x[b][j] = *reinterpret_cast<const u32x4*>(at + Sg::XAT + (FOUR ? (l >> 2) * 256 + (j * 4 + g) * 16 : (b * 4 + j) * 1024 + from));
    multiply(w, x, sw, zw, GB);
  };
  {
    int st = 0;                               // stage of block i
    auto ahead = [&](int n) { return st + n < ST ? st + n : st + n - ST; };
#pragma unroll
    for (int i = 0; i < ST - 1; ++i)
      if (i < mine) fetch(i, i);
    // the adapters while the first blocks are on their way
    for (int r = wave * 16; r < p.R; r += LW * 16)
#pragma unroll
      for (int b = 0; b < MB; ++b)
#pragma unroll
        for (int j = 0; j < NB; ++j) {
          const long n = n0 + j * 16 + l;
          out[b][j] = rank_step<T>(p, MB == 1 && p.a_cat ? tl + xm[b] * OWN_PITCH + r + 4 * g : nullptr, m0 + xm[b], n < p.N ? n : p.N - 1, r + 4 * g, out[b][j]);
        }
    int i = 0;
    for (; i + ST - 1 < mine; ++i) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the block before has been read; its stage is the next one's
      fetch(i + ST - 1, ahead(ST - 1));
      wait_vm<(ST - 1) * Sg::P>();
      use(i, st);
      st = ahead(1);
    }
    if constexpr (ST > 3)
      if (i + 2 < mine) { wait_vm<2 * Sg::P>(); use(i++, st); st = ahead(1); }
    if constexpr (ST > 2)
      if (i + 1 < mine) { wait_vm<Sg::P>(); use(i++, st); st = ahead(1); }
    if (i < mine) { wait_vm<0>(); use(i, st); }
  }
  // what there is of the last block (of rows of x that are not aligned to four bytes: every block)
  for (int kb = full + (wave - full % LW + LW) % LW; kb < blocks; kb += LW) {
    u32x4 w[NB], x[MB][4];
    SW_t sw[NB];
    ZW_t zw[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const uint32_t r = j * 16 + l < (int)last ? j * 16 + l : last, rc = r * (uint32_t)p.gstride;
      w[j] = u32x4{0, 0, 0, 0};
      if (kb * 64 + g * 16 < p.row_bytes) w[j] = *reinterpret_cast<const u32x4*>(q0 + (long)kb * 64 + r * (uint32_t)p.row_bytes + g * 16);
      sw[j] = *reinterpret_cast<const SW_t*>(s0 + kb * GB + rc);           // (rows of scales and zero points are filled up to whole blocks)
      if (ZERO) zw[j] = *reinterpret_cast<const ZW_t*>(z0 + kb * GB + rc);
    }
#pragma unroll
    for (int b = 0; b < MB; ++b)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        T v[8];
        load8<T>(x0 + (long)xm[b] * p.K + (kb * 128 + j * 32 + g * 8), (long)p.K - (kb * 128 + j * 32 + g * 8), v);
        x[b][j] = __builtin_bit_cast(u32x4, v);
      }
    const int left = (p.K - kb * 128 + G - 1) / G;
    multiply(w, x, sw, zw, left < GB ? left : GB);
  }
  __syncthreads();                            // the rings are dead
  float* part = reinterpret_cast<float*>(smem);      // [LW][rows][NB * 16 + 1]
#pragma unroll
  for (int b = 0; b < MB; ++b)
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int r = FOUR ? g : b * 16 + g * 4 + e;
      if (r < rows)
#pragma unroll
        for (int j = 0; j < NB; ++j) part[(wave * rows + r) * (NB * 16 + 1) + j * 16 + l] = out[b][j][e];
    }
  __syncthreads();
  for (int i = threadIdx.x; i < rows * (NB * 16); i += LW * 64) {
    const int r = i / (NB * 16), col = i % (NB * 16);
    const long m = m0 + r, n = n0 + col;
    if (n >= p.N) continue;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < LW; ++w) v += part[(w * rows + r) * (NB * 16 + 1) + col];
    if (p.bias) v += (float)((const T*)p.bias)[n];
    if (p.residual) v += (float)((const T*)p.residual)[m * p.N + n];
    ((T*)p.y)[m * p.N + n] = (T)v;
  }
#endif
}

// Many rows: 80 rows of x (a prompt of 77 tokens) and 384 columns of y to a workgroup of eight waves, 48 columns each.  Blocks of 128 codes with their x come
// by DMA into three stages in LDS, x in the order of its operands, codes and scales to the wave that uses them.
// The numbers multiplied are 16 + q without zero points and 32 + 16 + q - z with them (z taken off in the integers, four codes at a time); what they are too
// large by is one constant then, and its product with a group's x the same for all columns: a wave computes it for 16 rows of the next block and leaves it in
// LDS, where every wave's accumulators start from it.
// A block is 1920 clocks of the matrix unit (two waves of 60 products of 16 x 16 x 32 on a SIMD), about 2100 of the vector unit (codes to operands, the scaled sum of
// every group) and 1650 of LDS: sums of a group and of the row in 32 bits each are 120 registers of the 256 that two waves leave each other.
// 616 rows, 10240 x 1280 with rank 96, by the clock of a workgroup: 2.3 us to the first block, 4.2 for the ranks, 23.6 for ten blocks (of which those instructions, one after the other, are
// 17), 2.9 for the outputs; with a residual 7 .. 8 for those, whose 25 MB all CUs move at once.
constexpr int MR_M = 5, MR_N = 3, MR_W = 8, MR_ST = 3;     // tiles of 16 rows; of 16 columns of a wave; waves; stages

template <int G, bool ZERO>
struct ManyStage {
  static constexpr int S = G == 32 ? 2 : 1, Z = ZERO ? 1 : 0, GB = 128 / G;
  static constexpr int XAT = 0, WAT = MR_M * 4096, SAT = WAT + MR_W * MR_N * 1024, ZAT = SAT + MR_W * S * 256, BYTES = ZAT + MR_W * Z * 256;
  static constexpr int SUMS = MR_ST * BYTES, RING = SUMS + 2 * GB * MR_M * 16 * 4;
  static constexpr int PITCH = MR_N * 16 + 4, OUT = MR_W * MR_M * 16 * PITCH * 4;   // the outputs in 32 bits, on their way to whole rows
  static constexpr int LDS = RING > OUT ? RING : OUT;
};

template <typename T, int G, bool ZERO>
__global__ __launch_bounds__(MR_W * 64) __attribute__((amdgpu_waves_per_eu(2, 2))) void w4_many_rows(const LinParams p) {
#if __HIP_DEVICE_COMPILE__
  extern __shared__ __attribute__((aligned(16))) char smem[];
  typedef ManyStage<G, ZERO> Sg;
  constexpr int GB = 128 / G, SG = 4 / GB;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l = lane & 15, g = lane >> 4;
  const uint32_t mt = (uint32_t)((p.M + MR_M * 16 - 1) / (MR_M * 16));
  const uint32_t unit = xcd_remap(blockIdx.x, gridDim.x);                      // an XCD has neighbouring columns, with all rows
  const long m0 = (long)(unit % mt) * (MR_M * 16), n0 = (long)(unit / mt) * (MR_W * MR_N * 16) + wave * (MR_N * 16);
  const int rows = (int)(p.M - m0 < MR_M * 16 ? p.M - m0 : MR_M * 16);
  const bool some = n0 < p.N;                                                  // (a wave past the last column repeats it)
  const long nb = some ? n0 : p.N - 1;
  const uint8_t* q0 = p.q + nb * p.row_bytes;
  const bf16_t* s0 = p.scale + nb * p.gstride;
  const uint8_t* z0 = ZERO ? p.zero + nb * p.gstride : nullptr;
  const T* x0 = (const T*)p.x + m0 * p.K;
  const uint32_t last = (uint32_t)(p.N - 1 - nb < MR_N * 16 - 1 ? p.N - 1 - nb : MR_N * 16 - 1);
  constexpr int XL = (MR_M * 4 + MR_W - 1) / MR_W;                             // loads of x of a wave, at most
  const int dr = lane >> 2, dp = lane & 3, from = (l * 4 + g) * 16;            // (as for few rows)
  uint32_t qo[MR_N], xo[XL];
#pragma unroll
  for (int j = 0; j < MR_N; ++j) {
    const uint32_t r = j * 16 + dr;
    qo[j] = (r < last ? r : last) * (uint32_t)p.row_bytes + dp * 16;
  }
#pragma unroll
  for (int i = 0; i < XL; ++i) {              // load wave + 8 i: step j of the operands of a tile of 16 rows
    const int id = wave + i * MR_W, r = (id >> 2) * 16 + dr;
    xo[i] = (uint32_t)(r < rows ? r : rows - 1) * (uint32_t)p.K + (id & 3) * 32 + dp * 8;
  }
  const uint32_t so = ((uint32_t)lane < last ? (uint32_t)lane : last) * (uint32_t)p.gstride;
  auto bytes = [](long n) { return (int)(uint32_t)(n < 0xffffffffL ? n : 0xffffffffL); };
  const __amdgpu_buffer_rsrc_t rq = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(q0), 0, bytes((p.N - nb) * p.row_bytes), 0x00020000);
  const __amdgpu_buffer_rsrc_t rx = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(x0), 0, bytes((p.M - m0) * p.K * 2), 0x00020000);
  const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<bf16_t*>(s0), 0, bytes((p.N - nb) * p.gstride * 2), 0x00020000);
  const __amdgpu_buffer_rsrc_t rz = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(ZERO ? z0 : q0), 0, bytes((p.N - nb) * p.gstride), 0x00020000);

  const int blocks = (p.row_bytes + 63) / 64, whole = p.dma ? p.K / 128 : 0, groups = (p.K + G - 1) / G;
  auto fetch = [&](int kb, int st) {
    char* to = smem + st * Sg::BYTES;
    if (kb < whole) {
#pragma unroll
      for (int i = 0; i < XL; ++i)
        if (wave + i * MR_W < MR_M * 4) __builtin_amdgcn_raw_ptr_buffer_load_lds(rx, (lptr_t)(to + Sg::XAT + (wave + i * MR_W) * 1024), 16, xo[i] * 2, kb * 256, 0, 0);
    } else {                                  // the end of the rows, or rows that are not aligned to four bytes
#pragma unroll 1
      for (int id = wave; id < MR_M * 4; id += MR_W) {
        const int r = (id >> 2) * 16 + l, k = kb * 128 + (id & 3) * 32 + g * 8;
        T v[8];
        load8<T>(x0 + (long)(r < rows ? r : rows - 1) * p.K + k, (long)p.K - k, v);
        *reinterpret_cast<u32x4*>(to + Sg::XAT + id * 1024 + from) = __builtin_bit_cast(u32x4, v);
      }
    }
#pragma unroll
    for (int j = 0; j < MR_N; ++j) __builtin_amdgcn_raw_ptr_buffer_load_lds(rq, (lptr_t)(to + Sg::WAT + (wave * MR_N + j) * 1024), 16, qo[j], kb * 64, 0, 0);
#pragma unroll
    for (int j = 0; j < Sg::S; ++j)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lptr_t)(to + Sg::SAT + (wave * Sg::S + j) * 256), 4, so * 2, (kb * GB * 2 & ~3) + j * 4, 0, 0);
    if constexpr (ZERO) __builtin_amdgcn_raw_ptr_buffer_load_lds(rz, (lptr_t)(to + Sg::ZAT + wave * 256), 4, so, kb * GB & ~3, 0, 0);
  };
  const f32x4 none = f32x4{0.f, 0.f, 0.f, 0.f};
  constexpr int U = ZERO ? Num<T>::UNIT - 1 : Num<T>::UNIT;
  constexpr uint32_t P = ZERO ? Num<T>::P32 : Num<T>::P16, over = (P | Num<T>::NEG) | (ZERO ? 0x00100010u : 0x00080008u) << U;    // -(32 + 16), -(16 + 8)
  auto x_at = [&](int st, int b, int j) { return *reinterpret_cast<const u32x4*>(smem + st * Sg::BYTES + Sg::XAT + (b * 4 + j) * 1024 + from); };
  auto sums = [&](int st, int odd) {          // a constant's products with the groups of 16 rows
    if (wave >= MR_M) return;
#pragma unroll
    for (int i = 0; i < GB; ++i) {
      f32x4 a = none;
#pragma unroll
      for (int k = 0; k < SG; ++k) a = Num<T>::mfma(x_at(st, wave, i * SG + k), u32x4{over, over, over, over}, a);
      if (l == 0) *reinterpret_cast<f32x4*>(smem + Sg::SUMS + ((odd * GB + i) * MR_M * 16 + wave * 16 + g * 4) * 4) = a;
    }
  };
  f32x4 out[MR_M][MR_N];
#pragma unroll
  for (int b = 0; b < MR_M; ++b)
#pragma unroll
    for (int j = 0; j < MR_N; ++j) out[b][j] = none;
  uint32_t low = 0x0f0f0f0fu, sixteen = 0x10101010u, power = P;
  asm("" : "+s"(low));
  asm("" : "+v"(sixteen));
  asm("" : "+s"(power));
  auto multiply = [&](int kb, int st, int odd) {
    const char* at = smem + st * Sg::BYTES;
    u32x4 w[MR_N];
    uint64_t sw[MR_N];
    uint32_t zw[MR_N];
#pragma unroll
    for (int j = 0; j < MR_N; ++j) {
      w[j] = across_groups(*reinterpret_cast<const u32x4*>(at + Sg::WAT + (wave * MR_N + j) * 1024 + from));
      const char* sa = at + Sg::SAT + wave * Sg::S * 256 + (j * 16 + l) * 4;
      sw[j] = *reinterpret_cast<const uint32_t*>(sa);
      if constexpr (G == 32) sw[j] |= (uint64_t)*reinterpret_cast<const uint32_t*>(sa + 256) << 32;
      else sw[j] >>= (kb * GB * 16 & 31);
      if constexpr (ZERO) zw[j] = *reinterpret_cast<const uint32_t*>(at + Sg::ZAT + wave * 256 + (j * 16 + l) * 4) >> (kb * GB * 8 & 31);
    }
    // Operands of the next k-step (and, where a group ends, what its sums start from) are on their way from LDS while one is multiplied: all eight waves read at
    // once after the barrier, and the matrix unit would wait for every step's reads otherwise.
    u32x4 xv[2][MR_M];
    f32x4 base[2][MR_M];
    auto step_in = [&](int t) {
#pragma unroll
      for (int b = 0; b < MR_M; ++b) {
        xv[t & 1][b] = x_at(st, b, t);
        if (t % SG == 0) base[t / SG & 1][b] = *reinterpret_cast<const f32x4*>(smem + Sg::SUMS + ((odd * GB + t / SG) * MR_M * 16 + b * 16 + g * 4) * 4);
      }
    };
    auto hold = [&](int t) {                  // (the compiler otherwise moves the reads down to their uses)
      asm volatile("" ::: "memory");
#pragma unroll
      for (int b = 0; b < MR_M; ++b) asm volatile("" : "+v"(xv[t & 1][b]));
    };
    step_in(0);
    f32x4 acc[MR_M][MR_N];
    float s[MR_N];
    uint32_t z[MR_N];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int i = t / SG;
      if (t < 3) step_in(t + 1);
      hold(t);
      if (t % SG == 0) {
#pragma unroll
        for (int j = 0; j < MR_N; ++j) {
          s[j] = kb * GB + i < groups ? bf16_bits_to_f32((uint32_t)(sw[j] >> (16 * i)) & 0xffffu) : 0.f;    // what rows of scales are filled up with is not used
          if constexpr (ZERO) z[j] = ((zw[j] >> (8 * i)) & 15u) * 0x01010101u;
        }
      }
#pragma unroll
      for (int j = 0; j < MR_N; ++j) {        // bytes of even and of odd codes, put beside one another: the order of x
        const uint32_t word = w[j][t];
        const uint32_t even = ZERO ? ((word & low) | sixteen) - z[j] : word & low;
        const uint32_t uneven = ZERO ? (((word >> 4) & low) | sixteen) - z[j] : (word >> 4) & low;
        const u32x4 wv = u32x4{__builtin_amdgcn_perm(uneven, even, 0x0c040c00u) << U | power, __builtin_amdgcn_perm(uneven, even, 0x0c050c01u) << U | power,
                               __builtin_amdgcn_perm(uneven, even, 0x0c060c02u) << U | power, __builtin_amdgcn_perm(uneven, even, 0x0c070c03u) << U | power};
#pragma unroll
        for (int b = 0; b < MR_M; ++b) acc[b][j] = Num<T>::mfma(xv[t & 1][b], wv, t % SG == 0 ? base[i & 1][b] : acc[b][j]);
      }
      if (t % SG == SG - 1)
#pragma unroll
        for (int j = 0; j < MR_N; ++j)
#pragma unroll
          for (int b = 0; b < MR_M; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e) out[b][j][e] = fmaf(s[j], acc[b][j][e], out[b][j][e]);
    }
  };
  auto barrier = []() {                       // what this wave has written to LDS is there, and everybody has arrived
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  // Workgroups of other columns begin with other blocks: rows of x are often a multiple of the memory channels' period apart, and all of them at the same
  // place of the rows would ask few channels (616 x 10240 x 1280 38.0 -> 35.0 us).
  const int rot = (int)((unit / mt) * 5 % (uint32_t)blocks);
  auto turned = [&](int i) { return i + rot < blocks ? i + rot : i + rot - blocks; };
  // The adapters' product, 32 ranks at a time, comes first through the same stages: t in three pieces of bf16 (24 bits) in the place of x, B_cat in the place of the codes.
  const bf16_t* th = (const bf16_t*)p.t;
  const int steps = p.R / 32, all = steps + blocks;
  const __amdgpu_buffer_rsrc_t rt = __builtin_amdgcn_make_buffer_rsrc(const_cast<bf16_t*>(th + m0 * p.R), 0, bytes((3 * p.M - m0) * p.R * 2), 0x00020000);
  const __amdgpu_buffer_rsrc_t rb = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>((const T*)p.b_cat + nb * p.R), 0, bytes((p.N - nb) * p.R * 2), 0x00020000);
  auto fetch_ranks = [&](int step, int st) {
    char* to = smem + st * Sg::BYTES;
#pragma unroll
    for (int i = 0; i < (3 * MR_M + MR_W - 1) / MR_W; ++i) {
      const int id = wave + i * MR_W, r = id / 3 * 16 + dr;
      if (id < 3 * MR_M)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rt, (lptr_t)(to + Sg::XAT + id * 1024), 16, (int)(((uint32_t)(r < rows ? r : rows - 1) * (uint32_t)p.R + dp * 8) * 2),
                                                 (int)((uint32_t)(id % 3 * p.M * p.R + step * 32) * 2), 0, 0);   // (below 2^32: see `many` at the entry)
    }
#pragma unroll
    for (int j = 0; j < MR_N; ++j) {
      char* at = to + Sg::WAT + (wave * MR_N + j) * 1024;
      if (p.b_dma) {
        const uint32_t r = j * 16 + dr;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, (lptr_t)at, 16, (int)(((r < last ? r : last) * (uint32_t)p.R + dp * 8) * 2), step * 64, 0, 0);
      } else {
        const uint32_t r = j * 16 + l;
        u32x4 v;
        __builtin_memcpy(&v, (const T*)p.b_cat + (nb + (r < last ? r : last)) * p.R + step * 32 + g * 8, 16);
        *reinterpret_cast<u32x4*>(at + from) = v;
      }
    }
  };
  auto multiply_ranks = [&](int st) {
    const char* at = smem + st * Sg::BYTES;
    u32x4 t[MR_M][3];
#pragma unroll
    for (int b = 0; b < MR_M; ++b)
#pragma unroll
      for (int k = 0; k < 3; ++k) t[b][k] = *reinterpret_cast<const u32x4*>(at + Sg::XAT + (3 * b + k) * 1024 + from);
    auto add = [&](int j, int k, bf16x8 v) {
#pragma unroll
      for (int b = 0; b < MR_M; ++b) out[b][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, t[b][k]), v, out[b][j], 0, 0, 0);
    };
#pragma unroll
    for (int j = 0; j < MR_N; ++j) {
      const u32x4 raw = *reinterpret_cast<const u32x4*>(at + Sg::WAT + (wave * MR_N + j) * 1024 + from);
      bf16x8 bh = __builtin_bit_cast(bf16x8, raw), bl;
      if constexpr (!__is_same(T, bf16_t)) {       // (fp16: 11 bits in two pieces)
        T v[8];
        __builtin_memcpy(v, &raw, 16);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          bh[e] = (bf16_t)(float)v[e];
          bl[e] = (bf16_t)((float)v[e] - (float)bh[e]);
        }
      }
#pragma unroll
      for (int k = 0; k < 3; ++k) add(j, k, bh);
      if constexpr (!__is_same(T, bf16_t)) {       // (the third piece's product with what is left of B is 2^-24 of the first's)
        add(j, 0, bl);
        add(j, 1, bl);
      }
    }
  };
  auto fetch_any = [&](int i, int st) {
    if (i < steps) fetch_ranks(i, st);
    else fetch(turned(i - steps), st);
  };
  fetch_any(0, 0);
  if (all > 1) fetch_any(1, 1);
  wait_vm<0>();
  barrier();
  if (steps == 0) sums(0, 0);
  int st = 0;
  auto after = [](int st) { return st == MR_ST - 1 ? 0 : st + 1; };
  for (int i = 0; i < steps; ++i) {
    wait_vm<0>();                             // this wave's share of the next block, requested a block ago
    barrier();                                // everybody's; and nobody reads the block before any more
    if (i + 2 < all) fetch_any(i + 2, after(after(st)));
    if (i + 1 == steps) sums(after(st), 0);
    multiply_ranks(st);
    st = after(st);
  }
  for (int kb = 0; kb < blocks; ++kb) {
    const int s1 = after(st);
    wait_vm<0>();
    barrier();                                // (and this block's sums)
    if (kb + 2 < blocks) fetch(turned(kb + 2), after(s1));
    if (kb + 1 < blocks) sums(s1, (kb + 1) & 1);
    multiply(turned(kb), st, kb & 1);
    st = s1;
  }
  // Outputs by way of LDS to whole rows of 768 bytes: 48 lanes of eight columns, a wave has every eighth row.  What is added to them is asked for all at once, before.
  constexpr int ROWS = MR_M * 16 / MR_W, LANES = MR_W * MR_N * 2;
  static_assert(ROWS * MR_W == MR_M * 16 && LANES <= 64, "a row to a wave");
  const long n = n0 - wave * (MR_N * 16) + lane * 8;
  const bool mine = lane < LANES && n < p.N, vec = n + 8 <= p.N;
  float bias[8];
  T res[ROWS][8];
#pragma unroll
  for (int e = 0; e < 8; ++e) bias[e] = mine && p.bias && n + e < p.N ? (float)((const T*)p.bias)[n + e] : 0.f;
  if (mine && p.residual)
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
      if (wave + i * MR_W < rows) load8<T>((const T*)p.residual + (m0 + wave + i * MR_W) * p.N + n, p.N - n, res[i]);
  barrier();                                  // the stages are dead
  float* part = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int b = 0; b < MR_M; ++b)
#pragma unroll
    for (int j = 0; j < MR_N; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) part[(wave * (MR_M * 16) + b * 16 + g * 4 + e) * Sg::PITCH + j * 16 + l] = out[b][j][e];
  barrier();
  if (!mine) return;
  const float* from_lane = part + lane / (MR_N * 2) * (MR_M * 16 * Sg::PITCH) + lane % (MR_N * 2) * 8;
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int r = wave + i * MR_W;
    if (r >= rows) break;
    T o[8];
#pragma unroll
    for (int e = 0; e < 8; e += 4) {
      const f32x4 t = *reinterpret_cast<const f32x4*>(from_lane + r * Sg::PITCH + e);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float v = t[k] + bias[e + k];
        o[e + k] = (T)(p.residual ? v + (float)res[i][e + k] : v);
      }
    }
    T* to = (T*)p.y + (m0 + r) * p.N + n;
    if (vec && p.once && ((uintptr_t)to & 15) == 0) {
      u32x4 t;
      __builtin_memcpy(&t, o, sizeof(t));
      __builtin_nontemporal_store(t, reinterpret_cast<u32x4*>(to));
    } else if (vec) {
      __builtin_memcpy(to, o, sizeof(o));
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (n + e < p.N) to[e] = o[e];
    }
  }
#endif
}

// t[split][m][r] = col_scale[r] * sum over the split's k of x[m][k] A[r][k], in 32 bits: grid (R / 16, M / 16, splits)
struct ShrinkParams {
  const void *x, *a;
  const float* col_scale;
  float* t;
  long M;
  int K, R, per;           // per: k of a split, a multiple of 32
  int pieces;              // one split, and t in three pieces of bf16 [3][M][R] instead
};
constexpr int SW = 8;      // waves of a workgroup
template <typename T>
__global__ __launch_bounds__(SW * 64) void w4_shrink(const ShrinkParams p) {
  __shared__ float part[SW][16][17];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int l = lane & 15, g = lane >> 4;
  const int r0 = blockIdx.x * 16;
  const long m0 = (long)blockIdx.y * 16;
  const T* ar = (const T*)p.a + (long)(r0 + l) * p.K;       // R % 16 == 0
  const T* xr = (const T*)p.x + (m0 + l < p.M ? m0 + l : p.M - 1) * p.K;
  const int k0 = blockIdx.z * p.per, k1 = k0 + p.per < p.K ? k0 + p.per : p.K;
  f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
  int k = k0 + wave * 32;
  for (; k + 3 * SW * 32 + 32 <= k1; k += 4 * SW * 32) {      // four steps' loads on their way at once
    u32x4 a[4], x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      __builtin_memcpy(&a[i], ar + k + i * (SW * 32) + g * 8, 16);
      __builtin_memcpy(&x[i], xr + k + i * (SW * 32) + g * 8, 16);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) acc = Num<T>::mfma(x[i], a[i], acc);
  }
  for (; k < k1; k += SW * 32) {
    T a[8], x[8];
    load8<T>(ar + k + g * 8, (long)k1 - k - g * 8, a);
    load8<T>(xr + k + g * 8, (long)k1 - k - g * 8, x);
    acc = Num<T>::mfma(__builtin_bit_cast(u32x4, x), __builtin_bit_cast(u32x4, a), acc);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) part[wave][g * 4 + e][l] = acc[e];
  __syncthreads();
  if (threadIdx.x < 256) {
    const int r = threadIdx.x >> 4, col = threadIdx.x & 15;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < SW; ++w) v += part[w][r][col];
    if (m0 + r >= p.M) return;
    v *= p.col_scale[r0 + col];
    if (p.pieces) {
      bf16_t* t = (bf16_t*)p.t + (m0 + r) * p.R + r0 + col;
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        const bf16_t hi = (bf16_t)v;
        t[k * p.M * p.R] = hi;
        v -= (float)hi;
      }
    } else {
      p.t[((long)blockIdx.z * p.M + m0 + r) * p.R + r0 + col] = v;
    }
  }
}

// Few rows with a small A: t is computed by every workgroup for itself, which reads all of A from its L2, and a launch (another 4 us of the host's) and its workspace
// are gone.  On the GPU, us in one launch | in two: one row 1280 x 640 with rank 64 5.0 | 5.6, 1280 x 1280 with 32 5.3 | 6.3 and with 64 6.5 | 6.7, 1280 x 2560 with 32
// 7.0 | 7.8, 10240 x 640 with 64 7.0 | 8.8, 65536 x 1280 with 32 31.6 | 31.9; 16 rows 1280 x 1280 with 64 7.4 | 7.7; beyond: one row 1280 x 4096 with 32 9 | 8.2,
// 1280 x 1280 with 96 8.5 | 6.9.
bool own_t(long M, long K, long R) { return (R == 32 || R == 64) && M <= 16 && R * K <= 80 << 10; }

int shrink_splits(long M, long K, long R) {
  // enough workgroups that the rows of A are read by many CUs at once, at least 512 of k each (two steps of a wave)
  const long tiles = R / 16 * ((M + 15) / 16);
  long s = tiles >= 128 ? 1 : 128 / tiles;
  const long most = (K + 511) / 512;
  if (s > most) s = most;
  if (s > 16) s = 16;
  return (int)(s < 1 ? 1 : s);
}

template <typename T, int G, bool ZERO, int MB, int NB, int LW, int ST, bool FOUR>
int launch_few_as(LinParams p, hipStream_t s) {
  const long mt = (p.M + MB * 16 - 1) / (MB * 16), rows = p.M < MB * 16 ? p.M : MB * 16;
  const int ring = LW * ST * Stage<G, ZERO, MB, NB, FOUR>::BYTES, part = (LW * (int)rows * (NB * 16 + 1) * 4 + 15) / 16 * 16;
  const int own = p.a_cat ? LW * own_wave(p.R / 16) : 0, most = ring > part ? ring : part;
  p.t_at = own > most ? own : most;
  const int lds = p.t_at + (p.a_cat ? 16 * OWN_PITCH * 4 : 0);
  if (lds > 65536) {
    const hipError_t e = kh_allow_lds<w4_few_rows<T, G, ZERO, MB, NB, LW, ST, FOUR>>(160 * 1024);      // (asked for once: the largest of all calls)
    if (e != hipSuccess) return (int)e;
  }
  kh_launch(KH_TAG_W4_LINEAR, w4_few_rows<T, G, ZERO, MB, NB, LW, ST, FOUR>, dim3((unsigned)((p.N + NB * 16 - 1) / (NB * 16)), (unsigned)mt), dim3(LW * 64), lds, s, p);
  return KH_OK;
}
// Tiles of 16 columns to a workgroup: as few as leave every CU at most one workgroup, up to four (a tile's columns share the loads of x).  Waves and stages
// as measured over N 320 .. 16384, K 640 .. 8192 (us, cold codes, groups of 64, tiles 1 | 2 | 4): one row 8192 x 8192 10.3 | 9.6 | 12.6, 16384 x 8192 18.3 | 17.5 | 18.2,
// 1280 x 5120 4.5 | 5.4 | 7.7; 16 rows 5120 x 1280 5.1 | 4.1 | 4.7, 10240 x 1280 7.6 | 5.6 | 5.1, 16384 x 8192 34.8 | 24.4 | 21.3; 32 rows 16384 x 8192 44 | 32 | 26.3.
// Four, eight or sixteen waves and two, three or four stages are within 0.5 us of one another where LDS lets two workgroups on a CU or there is only one.
template <typename T, int G, bool ZERO>
int launch_few(const LinParams& p, hipStream_t s) {
  const long nb = (p.N + 15) / 16;
  if (p.M <= 4) {
    if (nb <= 256) return launch_few_as<T, G, ZERO, 1, 1, 8, 3, true>(p, s);
    if (nb <= 512) return launch_few_as<T, G, ZERO, 1, 2, 8, 3, true>(p, s);
    return launch_few_as<T, G, ZERO, 1, 4, 8, 2, true>(p, s);
  }
  if (p.M <= 16) {
    if (nb <= 256) return launch_few_as<T, G, ZERO, 1, 1, 8, 2, false>(p, s);
    if (nb <= 512) return launch_few_as<T, G, ZERO, 1, 2, 4, 3, false>(p, s);
    return launch_few_as<T, G, ZERO, 1, 4, 8, 2, false>(p, s);
  }
  if (nb <= 256) return launch_few_as<T, G, ZERO, 2, 1, 4, 2, false>(p, s);
  if (nb <= 512) return launch_few_as<T, G, ZERO, 2, 2, 4, 2, false>(p, s);
  return launch_few_as<T, G, ZERO, 2, 4, 4, 2, false>(p, s);
}
template <typename T, int G, bool ZERO>
int launch_many(const LinParams& p, hipStream_t s) {
  const hipError_t e = kh_allow_lds<w4_many_rows<T, G, ZERO>>(ManyStage<G, ZERO>::LDS);
  if (e != hipSuccess) return (int)e;
  const long units = (p.M + MR_M * 16 - 1) / (MR_M * 16) * ((p.N + MR_W * MR_N * 16 - 1) / (MR_W * MR_N * 16));
  kh_launch(KH_TAG_W4_LINEAR, w4_many_rows<T, G, ZERO>, dim3((unsigned)units), dim3(MR_W * 64), ManyStage<G, ZERO>::LDS, s, p);
  return KH_OK;
}
// Which of the two kernels has the smaller time by what was measured over N 320 .. 16384, K 1280 .. 8192, 33 .. 2464 rows (us; a block is 128 codes): the one for many
// rows 2.25 a block and round of its workgroups on 256 CUs, whatever the rows, the one for few 0.29 ns a block of 32 x 16 and 3.4 ns beside.  few | many:
// 1280 x 1280 by 154 rows 5.7 | 28, by 616 14.1 | 28, by 2464 45 | 31; 10240 x 1280 by 154 24.4 | 28.5, by 308 41 | 29.7, by 616 74 | 32.7; 16384 x 8192 by 154
// 109 | 158, by 400 267 | 166.
bool many_rows(long M, long N, long K) {
  if (M <= 32) return false;
  const long units = (M + MR_M * 16 - 1) / (MR_M * 16) * ((N + MR_W * MR_N * 16 - 1) / (MR_W * MR_N * 16)), blocks = (K + 127) / 128;
  const double many = 6. + (double)((units + 255) / 256) * blocks * 2.25;
  const double few = 4. + (double)((M + 31) / 32) * ((N + 15) / 16) * (blocks * 0.29 + 3.4) * 1e-3;
  return many < few;
}

template <typename T>
int launch_linear(const LinParams& p, int G, bool many, hipStream_t s) {
  if (many) {
    if (p.zero) return G == 32 ? launch_many<T, 32, true>(p, s) : G == 64 ? launch_many<T, 64, true>(p, s) : launch_many<T, 128, true>(p, s);
    return G == 32 ? launch_many<T, 32, false>(p, s) : G == 64 ? launch_many<T, 64, false>(p, s) : launch_many<T, 128, false>(p, s);
  }
  if (p.zero) return G == 32 ? launch_few<T, 32, true>(p, s) : G == 64 ? launch_few<T, 64, true>(p, s) : launch_few<T, 128, true>(p, s);
  return G == 32 ? launch_few<T, 32, false>(p, s) : G == 64 ? launch_few<T, 64, false>(p, s) : launch_few<T, 128, false>(p, s);
}

bool group_ok(int64_t g) { return g == 32 || g == 64 || g == 128; }

}  // namespace

KH_EXPORT int kh_quantize_w4(const void* w, void* q, void* scale, void* zero, int64_t N, int64_t K, int64_t group, int type, void* stream) {
  if (!w || !q || !scale || N <= 0 || K <= 0 || type < 0 || type > 2) return KH_ERR_INVALID_ARG;
  if (!group_ok(group)) return KH_ERR_UNSUPPORTED;
  if (!kh_aligned16(q) || ((uintptr_t)scale & 7) || ((uintptr_t)zero & 3)) return KH_ERR_ALIGNMENT;   // (any whole rows of larger ones)
  if (K > (1L << 24) || N > (1L << 24)) return KH_ERR_TOO_LARGE;
  const long groups = (K + group - 1) / group, pieces = groups * (group / 8);
  const long wg = (N * pieces + 4 * PT * 64 - 1) / (4 * PT * 64);
  if (wg > 0x7fffffffL) return KH_ERR_TOO_LARGE;
  const dim3 grid((unsigned)wg);
  QuantParams p{w, (uint8_t*)q, (bf16_t*)scale, (uint8_t*)zero, (long)N, (int)K, (int)groups, (int)((groups + 3) / 4 * 4), (int)((K + 31) / 32 * 4), Pieces(pieces)};
  hipStream_t s = (hipStream_t)stream;
  auto go = [&](auto kernel) { kh_launch(KH_TAG_W4_QUANTIZE, kernel, grid, dim3(256), 0, s, p); };
#define KH_BY_GROUP(T)                                                                            \
  if (group == 32) zero ? go(quantize_kernel<T, 32, true>) : go(quantize_kernel<T, 32, false>);     \
  else if (group == 64) zero ? go(quantize_kernel<T, 64, true>) : go(quantize_kernel<T, 64, false>); \
  else zero ? go(quantize_kernel<T, 128, true>) : go(quantize_kernel<T, 128, false>)
  if (type == 0) { KH_BY_GROUP(bf16_t); }
  else if (type == 1) { KH_BY_GROUP(_Float16); }
  else { KH_BY_GROUP(float); }
#undef KH_BY_GROUP
  KH_RETURN_LAST_ERROR();
}

KH_EXPORT int kh_dequantize_w4(const void* q, const void* scale, const void* zero, void* out, int64_t N, int64_t K, int64_t group, int type,
                               void* stream) {
  if (!q || !scale || !out || N <= 0 || K <= 0 || type < 0 || type > 2) return KH_ERR_INVALID_ARG;
  if (!group_ok(group)) return KH_ERR_UNSUPPORTED;
  if (!kh_aligned16(q) || ((uintptr_t)scale & 7) || ((uintptr_t)zero & 3)) return KH_ERR_ALIGNMENT;   // (any whole rows of larger ones)
  if (K > (1L << 24) || N > (1L << 24)) return KH_ERR_TOO_LARGE;
  const long groups = (K + group - 1) / group, words = (K + 31) / 32 * 4;
  const long wg = (N * words + 4 * PT * 64 - 1) / (4 * PT * 64);
  if (wg > 0x7fffffffL) return KH_ERR_TOO_LARGE;
  const dim3 grid((unsigned)wg);
  ValueParams p{(const uint32_t*)q, (const bf16_t*)scale, (const uint8_t*)zero, out, (long)N, (int)K, group == 32 ? 2 : group == 64 ? 3 : 4, (int)((groups + 3) / 4 * 4), Pieces(words)};
  hipStream_t s = (hipStream_t)stream;
  auto go = [&](auto kernel) { kh_launch(KH_TAG_W4_VALUES, kernel, grid, dim3(256), 0, s, p); };
  type == 0 ? go(values_kernel<bf16_t>) : type == 1 ? go(values_kernel<_Float16>) : go(values_kernel<float>);
  KH_RETURN_LAST_ERROR();
}

namespace {

int64_t linear_workspace(int64_t M, int64_t K, int64_t R, int64_t most) {
  if (M <= 0 || K <= 0 || R < 0 || R % 32 != 0 || R > most) return KH_ERR_INVALID_ARG;
  if (R == 0 || own_t(M, K, R)) return 0;
  const int64_t parts = (int64_t)shrink_splits(M, K, R) * 4;
  return (M > 32 && parts < 6 ? 6 : parts) * M * R;         // (t in 32 bits for each split, or, for many rows, in three pieces of 16)
}

int linear(const void* x, const void* q, const void* scale, const void* zero, const void* bias, const void* a_cat, const void* b_cat,
           const float* col_scale, const void* residual, void* y, void* workspace, int64_t M, int64_t N,
           int64_t K, int64_t R, int64_t most, int64_t group, int type, void* stream) {
  if (!x || !q || !scale || !y || M <= 0 || N <= 0 || K <= 0 || R < 0 || type < 0 || type > 1) return KH_ERR_INVALID_ARG;
  const bool own = own_t(M, K, R);
  if (R > 0 && (!a_cat || !b_cat || !col_scale || (!workspace && !own))) return KH_ERR_INVALID_ARG;
  if (!group_ok(group) || R % 32 != 0) return KH_ERR_UNSUPPORTED;
  if (R > most || K > (1L << 24) || N > (1L << 24) || (M + 15) / 16 > 65535) return KH_ERR_TOO_LARGE;
  if (!kh_aligned16(q) || ((uintptr_t)scale & 7) || ((uintptr_t)zero & 3)) return KH_ERR_ALIGNMENT;   // (any whole rows of larger ones)
  if (R > 0 && ((!own && !kh_aligned16(workspace)) || ((uintptr_t)col_scale & 3))) return KH_ERR_ALIGNMENT;
  hipStream_t s = (hipStream_t)stream;
  const bool many = many_rows(M, N, K) && 3 * M * R <= 0x7fffffffL;      // (the ranks' pieces lie within 4 GB)
  const int splits = R == 0 ? 0 : many ? 1 : shrink_splits(M, K, R);
  if (R > 0 && !own) {
    const int per = (int)(((K + splits - 1) / splits + 31) / 32 * 32);
    ShrinkParams sp{x, a_cat, col_scale, (float*)workspace, (long)M, (int)K, (int)R, per, many};
    const dim3 grid((unsigned)(R / 16), (unsigned)((M + 15) / 16), (unsigned)splits);
    if (type == 0) kh_launch(KH_TAG_W4_SHRINK, w4_shrink<bf16_t>, grid, dim3(SW * 64), 0, s, sp);
    else kh_launch(KH_TAG_W4_SHRINK, w4_shrink<_Float16>, grid, dim3(SW * 64), 0, s, sp);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
  }
  LinParams p{x, (const uint8_t*)q, (const bf16_t*)scale, (const uint8_t*)zero, bias, b_cat, residual, (const float*)workspace, y, (long)M,
              (long)N, (int)K, (int)R, splits, (int)((K + 31) / 32 * 16), (int)(((K + group - 1) / group + 3) / 4 * 4),
              ((uintptr_t)x & 3) == 0 && K % 2 == 0 && (!own || ((uintptr_t)a_cat & 3) == 0), own ? a_cat : nullptr, col_scale, 0, ((uintptr_t)b_cat & 3) == 0, M * N >= 4 << 20};
  const int rc = type == 0 ? launch_linear<bf16_t>(p, (int)group, many, s) : launch_linear<_Float16>(p, (int)group, many, s);
  if (rc != KH_OK) return rc;
  KH_RETURN_LAST_ERROR();
}

}  // namespace

// Rank columns: as many as K1's entry points take, or (wide) what many adapters add up to.
constexpr int64_t RANKS = 128, RANKS_WIDE = 1 << 16;

KH_EXPORT int64_t kh_w4_linear_workspace_bytes(int64_t M, int64_t K, int64_t R) { return linear_workspace(M, K, R, RANKS); }
KH_EXPORT int64_t kh_w4_linear_wide_workspace_bytes(int64_t M, int64_t K, int64_t R) { return linear_workspace(M, K, R, RANKS_WIDE); }

KH_EXPORT int kh_w4_linear(const void* x, const void* q, const void* scale, const void* zero, const void* bias, const void* a_cat,
                           const void* b_cat, const float* col_scale, const void* residual, void* y, void* workspace, int64_t M, int64_t N,
                           int64_t K, int64_t R, int64_t group, int type, void* stream) {
  return linear(x, q, scale, zero, bias, a_cat, b_cat, col_scale, residual, y, workspace, M, N, K, R, RANKS, group, type, stream);
}
KH_EXPORT int kh_w4_linear_wide(const void* x, const void* q, const void* scale, const void* zero, const void* bias, const void* a_cat,
                                const void* b_cat, const float* col_scale, const void* residual, void* y, void* workspace, int64_t M, int64_t N,
                                int64_t K, int64_t R, int64_t group, int type, void* stream) {
  return linear(x, q, scale, zero, bias, a_cat, b_cat, col_scale, residual, y, workspace, M, N, K, R, RANKS_WIDE, group, type, stream);
}
