// K12: weights in 4 bits with a scale (and a zero point) for each group of 32, 64 or 128 along a row:
//   w[n][k] = s[n][k / G] * (q[n][k] - z[n][k / G]),   z = 8 where no zero points are given
// Quantisation, the values that codes stand for, and the linear of few and of many rows with the adapters of K1 beside it:
//   y = x w^T + b + ((x A_cat^T) * col_scale) B_cat^T (+ residual)
//
// A row of codes is its weights in order, two to a byte (the even one in the low half), filled up to 32 of them; a row of scales or
// zero points is filled up to 4.  Scales are bf16 whatever the activations' type: they have the weights' range, and the codes are
// chosen against the rounded scale.
#include "kh_common.h"

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

// ---------------------------------------------------------------- quantisation
// A thread takes eight weights of a row, G / 8 threads in a row a group.  Every row starts with a new group, so a group's threads lie
// in one wave, aligned.
struct QuantParams {
  const void* w;
  uint8_t* q;
  bf16_t* scale;
  uint8_t* zero;
  long N;
  int K, groups, gstride, words;   // words: of eight codes in a row
};

template <typename T, int G, bool ZERO>
__global__ __launch_bounds__(256) void quantize_kernel(const QuantParams p) {
  constexpr int GT = G / 8;
  const int per_row = p.groups * GT;
  const long id = (long)blockIdx.x * 256 + threadIdx.x;
  const long row = id / per_row;
  const int u = (int)(id - row * per_row);
  if (row >= p.N) return;            // (whole groups: per_row is a multiple of GT)
  T v[8];
  load8<T>((const T*)p.w + row * p.K + (long)u * 8, (long)p.K - (long)u * 8, v);
  float f[8], lo = 0.f, hi = 0.f;
  bool nan = false;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    f[e] = (float)v[e];
    nan |= f[e] != f[e];
    lo = fminf(lo, f[e]);
    hi = fmaxf(hi, f[e]);
  }
  int bad = nan;
#pragma unroll
  for (int o = GT / 2; o > 0; o >>= 1) {
    lo = fminf(lo, __shfl_xor(lo, o, 64));
    hi = fmaxf(hi, __shfl_xor(hi, o, 64));
    bad |= __shfl_xor(bad, o, 64);
  }
  float s = ZERO ? (hi - lo) / 15.f : fmaxf(hi, -lo) / 7.f;
  if (bad) s = __builtin_nanf("");
  const bf16_t sb = (bf16_t)s;
  s = (float)sb;
  const bool some = s > 0.f;
  auto level = [&](float a) {        // rint(a / s), 0 where that is no number
    const float r = some ? rintf(a / s) : 0.f;
    return r == r ? r : 0.f;
  };
  const float z = ZERO ? fminf(fmaxf(level(-lo), 0.f), 15.f) : 8.f;
  uint32_t word = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) word |= (uint32_t)(int)fminf(fmaxf(level(f[e]) + z, 0.f), 15.f) << (4 * e);
  if (u < p.words) {
    if (u * 8 >= p.K) word = 0;      // filling
    else if (p.K - u * 8 < 8) word &= (1u << (4 * (p.K - u * 8))) - 1u;
    reinterpret_cast<uint32_t*>(p.q)[row * p.words + u] = word;
  }
  const int g = u / GT;
  if (u % GT == 0) {
    p.scale[row * p.gstride + g] = sb;
    if (ZERO) p.zero[row * p.gstride + g] = (uint8_t)(int)z;
    if (g == p.groups - 1)
      for (int i = p.groups; i < p.gstride; ++i) {
        p.scale[row * p.gstride + i] = (bf16_t)0.f;
        if (ZERO) p.zero[row * p.gstride + i] = 0;
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
  int K, G, gstride, words;
};

template <typename T>
__global__ __launch_bounds__(256) void values_kernel(const ValueParams p) {
  const long id = (long)blockIdx.x * 256 + threadIdx.x;
  const long row = id / p.words;
  const int u = (int)(id - row * p.words);
  if (row >= p.N || u * 8 >= p.K) return;
  const uint32_t word = p.q[row * p.words + u];
  const long at = row * p.gstride + u * 8 / p.G;
  const float s = (float)p.scale[at];
  const int z = p.zero ? p.zero[at] : 8;
  T v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = (T)(s * (float)((int)((word >> (4 * e)) & 15u) - z));
  T* o = (T*)p.out + row * p.K + u * 8;
  if (p.K - u * 8 >= 8) {
    __builtin_memcpy(o, v, sizeof(v));
  } else {
    for (int e = 0; e < p.K - u * 8; ++e) o[e] = v[e];
  }
}

// ---------------------------------------------------------------- the linear
// Codes become operands of the matrix unit without a conversion: with the bits of a power of two P above a code (128 in bf16, 1024
// in fp16, whose unit in the last place is 1) the 16 bits are the number P + q, so two shifted and masked nibbles are two operands.
// A second product of x with the constant -(P + z) takes P and z away again, exactly, in the same accumulator; scales are applied to
// a group's sum in 32 bits.  The nibbles of a word come out as pairs (0,4) (1,5) (2,6) (3,7); x is put into the same order.
template <typename T> struct Num;
template <> struct Num<bf16_t> {
  static constexpr uint32_t P = 0x43004300u, NEG = 0x80008000u;
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
  static constexpr uint32_t P = 0x64006400u, NEG = 0x80008000u;
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

template <typename T>
__device__ __forceinline__ u32x4 operands(uint32_t word) {
  return u32x4{(word & 0x000f000fu) | Num<T>::P, ((word >> 4) & 0x000f000fu) | Num<T>::P, ((word >> 8) & 0x000f000fu) | Num<T>::P,
               ((word >> 12) & 0x000f000fu) | Num<T>::P};
}

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
};

constexpr int LW = 8;      // waves of a workgroup, which share the blocks of 128 codes

// 16 columns of y (rows of codes) and MB * 16 rows of x to a workgroup; its waves take every LW-th block of 128 codes and are summed
// in order at the end.
template <typename T, int G, bool ZERO, int MB>
__global__ __launch_bounds__(LW * 64) void w4_few_rows(const LinParams p) {
  extern __shared__ float part[];    // [LW][MB * 16][17]
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int l = lane & 15, g = lane >> 4;
  const long n = (long)blockIdx.x * 16 + l, nc = n < p.N ? n : p.N - 1;
  const long m0 = (long)blockIdx.y * (MB * 16);
  const int blocks = (p.row_bytes + 63) / 64;
  const uint8_t* qr = p.q + nc * p.row_bytes + g * 16;
  const bf16_t* sr = p.scale + nc * p.gstride;
  const uint8_t* zr = ZERO ? p.zero + nc * p.gstride : nullptr;
  const int groups = (p.K + G - 1) / G;
  constexpr int GB = 128 / G;        // groups in a block
  constexpr int SG = 4 / GB;         // k-steps in a group
  f32x4 out[MB];
#pragma unroll
  for (int b = 0; b < MB; ++b) out[b] = f32x4{0.f, 0.f, 0.f, 0.f};
  const T* xr[MB];
#pragma unroll
  for (int b = 0; b < MB; ++b) {
    const long m = m0 + b * 16 + l;
    xr[b] = (const T*)p.x + (m < p.M ? m : p.M - 1) * p.K;
  }
  for (int kb = wave; kb < blocks; kb += LW) {
    u32x4 w = u32x4{0, 0, 0, 0};
    if (kb * 64 + g * 16 < p.row_bytes) w = *reinterpret_cast<const u32x4*>(qr + (long)kb * 64);
    float s[GB];
    uint32_t c[GB];
#pragma unroll
    for (int i = 0; i < GB; ++i) {
      const int gi = kb * GB + i;
      s[i] = gi < groups ? (float)sr[gi] : 0.f;
      c[i] = (Num<T>::P | Num<T>::NEG) | (ZERO ? (gi < groups ? zr[gi] : 0u) * 0x10001u : 0x00080008u);
    }
    w = across_groups(w);
    u32x4 wv[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) wv[j] = operands<T>(w[j]);
#pragma unroll
    for (int b = 0; b < MB; ++b) {
      u32x4 xv[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int k = kb * 128 + j * 32 + g * 8;
        T v[8];
        load8<T>(xr[b] + k, (long)p.K - k, v);
        xv[j] = interleaved(__builtin_bit_cast(u32x4, v));
      }
#pragma unroll
      for (int i = 0; i < GB; ++i) {
        f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
        const u32x4 cv = u32x4{c[i], c[i], c[i], c[i]};
#pragma unroll
        for (int j = 0; j < SG; ++j) {
          acc = Num<T>::mfma(xv[i * SG + j], wv[i * SG + j], acc);
          acc = Num<T>::mfma(xv[i * SG + j], cv, acc);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) out[b][e] = fmaf(s[i], acc[e], out[b][e]);
      }
    }
  }
#pragma unroll
  for (int b = 0; b < MB; ++b)
#pragma unroll
    for (int e = 0; e < 4; ++e) part[(wave * (MB * 16) + b * 16 + g * 4 + e) * 17 + l] = out[b][e];
  __syncthreads();
  for (int i = threadIdx.x; i < MB * 256; i += LW * 64) {
    const int r = i >> 4, col = i & 15;
    const long m = m0 + r, nn = (long)blockIdx.x * 16 + col;
    if (m >= p.M || nn >= p.N) continue;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < LW; ++w) v += part[(w * (MB * 16) + r) * 17 + col];
    if (p.R > 0) {
      const T* bc = (const T*)p.b_cat + nn * p.R;
      const float* t = p.t + m * p.R;
      for (int k = 0; k < p.R; k += 8) {
        T bv[8];
        __builtin_memcpy(bv, bc + k, sizeof(bv));
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float tv = 0.f;
          for (int sp = 0; sp < p.t_splits; ++sp) tv += t[(long)sp * p.M * p.R + k + e];
          v = fmaf(tv, (float)bv[e], v);
        }
      }
    }
    if (p.bias) v += (float)((const T*)p.bias)[nn];
    if (p.residual) v += (float)((const T*)p.residual)[m * p.N + nn];
    ((T*)p.y)[m * p.N + nn] = (T)v;
  }
}

// t[split][m][r] = col_scale[r] * sum over the split's k of x[m][k] A[r][k], in 32 bits: grid (R / 16, M / 16, splits)
struct ShrinkParams {
  const void *x, *a;
  const float* col_scale;
  float* t;
  long M;
  int K, R, per;           // per: k of a split, a multiple of 32
};
template <typename T>
__global__ __launch_bounds__(LW * 64) void w4_shrink(const ShrinkParams p) {
  __shared__ float part[LW][16][17];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int l = lane & 15, g = lane >> 4;
  const int r0 = blockIdx.x * 16;
  const long m0 = (long)blockIdx.y * 16;
  const T* ar = (const T*)p.a + (long)(r0 + l) * p.K;       // R % 16 == 0
  const T* xr = (const T*)p.x + (m0 + l < p.M ? m0 + l : p.M - 1) * p.K;
  const int k0 = blockIdx.z * p.per, k1 = k0 + p.per < p.K ? k0 + p.per : p.K;
  f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int k = k0 + wave * 32; k < k1; k += LW * 32) {
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
    for (int w = 0; w < LW; ++w) v += part[w][r][col];
    if (m0 + r < p.M) p.t[((long)blockIdx.z * p.M + m0 + r) * p.R + r0 + col] = v * p.col_scale[r0 + col];
  }
}

int shrink_splits(long M, long K, long R) {
  // enough workgroups that the rows of A are read by many CUs at once, at least 1024 of k each
  const long tiles = R / 16 * ((M + 15) / 16);
  long s = tiles >= 64 ? 1 : 64 / tiles;
  const long most = (K + 1023) / 1024;
  if (s > most) s = most;
  if (s > 8) s = 8;
  return (int)(s < 1 ? 1 : s);
}

template <typename T, int G, bool ZERO>
void launch_few(const LinParams& p, hipStream_t s) {
  const unsigned nb = (unsigned)((p.N + 15) / 16);
  const long mt = (p.M + 15) / 16;
  auto go = [&](auto kernel, int mb) {
    kh_launch(KH_TAG_W4_LINEAR, kernel, dim3(nb, (unsigned)((mt + mb - 1) / mb)), dim3(LW * 64), (size_t)LW * mb * 16 * 17 * 4, s, p);
  };
  if (mt == 1) go(w4_few_rows<T, G, ZERO, 1>, 1);
  else if (mt == 2) go(w4_few_rows<T, G, ZERO, 2>, 2);
  else go(w4_few_rows<T, G, ZERO, 4>, 4);
}
template <typename T>
void launch_linear(const LinParams& p, int G, hipStream_t s) {
  if (p.zero) {
    if (G == 32) launch_few<T, 32, true>(p, s);
    else if (G == 64) launch_few<T, 64, true>(p, s);
    else launch_few<T, 128, true>(p, s);
  } else {
    if (G == 32) launch_few<T, 32, false>(p, s);
    else if (G == 64) launch_few<T, 64, false>(p, s);
    else launch_few<T, 128, false>(p, s);
  }
}

bool group_ok(int64_t g) { return g == 32 || g == 64 || g == 128; }

}  // namespace

KH_EXPORT int kh_quantize_w4(const void* w, void* q, void* scale, void* zero, int64_t N, int64_t K, int64_t group, int type, void* stream) {
  if (!w || !q || !scale || N <= 0 || K <= 0 || type < 0 || type > 2) return KH_ERR_INVALID_ARG;
  if (!group_ok(group)) return KH_ERR_UNSUPPORTED;
  if (!kh_aligned16(q) || !kh_aligned16(scale)) return KH_ERR_ALIGNMENT;
  const long groups = (K + group - 1) / group, total = N * groups * (group / 8), wg = (total + 255) / 256;
  if (K > (1L << 24) || N > (1L << 24) || wg > 0x7fffffffL) return KH_ERR_TOO_LARGE;
  QuantParams p{w, (uint8_t*)q, (bf16_t*)scale, (uint8_t*)zero, (long)N, (int)K, (int)groups, (int)((groups + 3) / 4 * 4), (int)((K + 31) / 32 * 4)};
  hipStream_t s = (hipStream_t)stream;
  auto go = [&](auto kernel) { kh_launch(KH_TAG_W4_QUANTIZE, kernel, dim3((unsigned)wg), dim3(256), 0, s, p); };
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
  if (!kh_aligned16(q) || !kh_aligned16(scale)) return KH_ERR_ALIGNMENT;
  const long groups = (K + group - 1) / group, words = (K + 31) / 32 * 4, wg = (N * words + 255) / 256;
  if (K > (1L << 24) || N > (1L << 24) || wg > 0x7fffffffL) return KH_ERR_TOO_LARGE;
  ValueParams p{(const uint32_t*)q, (const bf16_t*)scale, (const uint8_t*)zero, out, (long)N, (int)K, (int)group, (int)((groups + 3) / 4 * 4), (int)words};
  hipStream_t s = (hipStream_t)stream;
  auto go = [&](auto kernel) { kh_launch(KH_TAG_W4_VALUES, kernel, dim3((unsigned)wg), dim3(256), 0, s, p); };
  type == 0 ? go(values_kernel<bf16_t>) : type == 1 ? go(values_kernel<_Float16>) : go(values_kernel<float>);
  KH_RETURN_LAST_ERROR();
}

KH_EXPORT int64_t kh_w4_linear_workspace_bytes(int64_t M, int64_t K, int64_t R) {
  if (M <= 0 || K <= 0 || R < 0 || R % 32 != 0 || R > 128) return KH_ERR_INVALID_ARG;
  return R == 0 ? 0 : (int64_t)shrink_splits(M, K, R) * M * R * 4;
}

KH_EXPORT int kh_w4_linear(const void* x, const void* q, const void* scale, const void* zero, const void* bias, const void* a_cat,
                           const void* b_cat, const float* col_scale, const void* residual, void* y, void* workspace, int64_t M, int64_t N,
                           int64_t K, int64_t R, int64_t group, int type, void* stream) {
  if (!x || !q || !scale || !y || M <= 0 || N <= 0 || K <= 0 || R < 0 || type < 0 || type > 1) return KH_ERR_INVALID_ARG;
  if (R > 0 && (!a_cat || !b_cat || !col_scale || !workspace)) return KH_ERR_INVALID_ARG;
  if (!group_ok(group) || R % 32 != 0) return KH_ERR_UNSUPPORTED;
  if (R > 128 || K > (1L << 24) || N > (1L << 24) || (M + 15) / 16 > 65535) return KH_ERR_TOO_LARGE;
  if (!kh_aligned16(q) || !kh_aligned16(scale)) return KH_ERR_ALIGNMENT;
  hipStream_t s = (hipStream_t)stream;
  const int splits = R > 0 ? shrink_splits(M, K, R) : 0;
  if (R > 0) {
    const int per = (int)(((K + splits - 1) / splits + 31) / 32 * 32);
    ShrinkParams sp{x, a_cat, col_scale, (float*)workspace, (long)M, (int)K, (int)R, per};
    const dim3 grid((unsigned)(R / 16), (unsigned)((M + 15) / 16), (unsigned)splits);
    if (type == 0) kh_launch(KH_TAG_W4_SHRINK, w4_shrink<bf16_t>, grid, dim3(LW * 64), 0, s, sp);
    else kh_launch(KH_TAG_W4_SHRINK, w4_shrink<_Float16>, grid, dim3(LW * 64), 0, s, sp);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
  }
  LinParams p{x, (const uint8_t*)q, (const bf16_t*)scale, (const uint8_t*)zero, bias, b_cat, residual, (const float*)workspace, y, (long)M,
              (long)N, (int)K, (int)R, splits, (int)((K + 31) / 32 * 16), (int)(((K + group - 1) / group + 3) / 4 * 4)};
  if (type == 0) launch_linear<bf16_t>(p, (int)group, s);
  else launch_linear<_Float16>(p, (int)group, s);
  KH_RETURN_LAST_ERROR();
}
