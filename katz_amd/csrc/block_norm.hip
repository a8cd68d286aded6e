// K11: the norms before and after a block with the gate and the residual between them, one row in registers:
//   h' = rho * h + g * N_post(y),   u = N_pre(h')
// N is a root-mean-square or a layer norm with the affine terms that are given (or absent), g a row of gates for every row, for
// every sequence or for all.  Beside kh_layer_norm_bf16, which is one such norm of a row by itself.
//
// Statistics, sums and the row itself are held in 32 bits: u is the norm of the sum before it is rounded to the stream's type.
#include "kh_common.h"

namespace {

struct NormParams {
  const void *y, *h, *gate, *post_w, *post_b, *pre_w, *pre_b;
  void *h_out, *u;
  long M, gate_rows;   // gate_rows: rows that share a row of gates
  int D;
  float rho, eps;
  int layer, post;     // kind of the norms; whether y is normed
  int once;            // outputs larger than the caches: stored past them
};

template <typename T> __device__ __forceinline__ float to_f(T v) { return (float)v; }

// Eight elements of a row at a time: aligned to 16 bytes where rows are, else at any address, the last ones one by one
// (against single elements throughout, us: 7904 rows of 1283, stream in 32 bits, 65 -> 39, 2000 of 5001 64 -> 31, 17464 of 435 37 -> 27, 60000 of 65 45 -> 51).
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* row, int at, int D, float (&f)[8]) {
  if constexpr (VEC) {
    if (at * 8 < D) {
      T v[8];
      __builtin_memcpy(v, __builtin_assume_aligned(row + at * 8, 16), sizeof(v));
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = (float)v[e];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = 0.f;
    }
  } else if (at * 8 + 8 <= D) {
    T v[8];
    __builtin_memcpy(v, row + at * 8, sizeof(v));
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = (float)v[e];
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = at * 8 + e < D ? (float)row[at * 8 + e] : 0.f;
  }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* row, int at, int D, const float (&f)[8], int once) {
  if constexpr (VEC) {
    if (at * 8 < D) {
      T v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = (T)f[e];
      u32x4 t[sizeof(v) / 16];
      __builtin_memcpy(t, v, sizeof(v));
      u32x4* to = reinterpret_cast<u32x4*>(row + at * 8);
#pragma unroll
      for (unsigned i = 0; i < sizeof(v) / 16; ++i) {
        if (once) __builtin_nontemporal_store(t[i], to + i);
        else to[i] = t[i];
      }
    }
  } else if (at * 8 + 8 <= D) {
    T v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (T)f[e];
    __builtin_memcpy(row + at * 8, v, sizeof(v));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (at * 8 + e < D) row[at * 8 + e] = (T)f[e];
  }
}
template <bool VEC>
__device__ __forceinline__ bool inside(int at, int D, int e) {
  return VEC ? at * 8 < D : at * 8 + e < D;
}

// Sum over the NW waves of a row, in every thread; `red` is a set of NW floats that no other sum of the row uses.
template <int NW>
__device__ __forceinline__ float row_sum(float v, float* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  if constexpr (NW > 1) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) v += red[w];
  }
  return v;
}

// NW waves a row, CH pieces of eight elements a thread.
template <typename T, typename H, int NW, int CH, bool VEC>
__global__ __launch_bounds__(NW == 1 ? 256 : NW * 64) void block_norm_kernel(const NormParams p) {
  constexpr int NT = NW * 64;
  __shared__ float red[4][NW];
  const int t = NW == 1 ? threadIdx.x & 63 : threadIdx.x;
  const long row = NW == 1 ? (long)blockIdx.x * 4 + (threadIdx.x >> 6) : (long)blockIdx.x;
  if (row >= p.M) return;
  const int D = p.D;
  const float n = 1.f / (float)D;

  auto normed = [&](float (&v)[CH][8], const T* w, const T* b, float* red0, float* red1) {
    float mean = 0.f;
    if (p.layer) {
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < CH; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) s += v[k][e];   // (zeros past the row's end)
      mean = row_sum<NW>(s, red0) * n;
    }
    float q = 0.f;
#pragma unroll
    for (int k = 0; k < CH; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[k][e] = inside<VEC>(t + NT * k, D, e) ? v[k][e] - mean : 0.f;
        q = fmaf(v[k][e], v[k][e], q);
      }
    const float r = 1.f / sqrtf(row_sum<NW>(q, red1) * n + p.eps);
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      float f[8];
      if (w) load8<T, VEC>(w, t + NT * k, D, f);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[k][e] *= w ? r * f[e] : r;
      if (b) {
        load8<T, VEC>(b, t + NT * k, D, f);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[k][e] += f[e];
      }
    }
  };

  float v[CH][8];
  const H* hr = (const H*)p.h + row * D;
  if (p.y) {
    const T* yr = (const T*)p.y + row * D;
#pragma unroll
    for (int k = 0; k < CH; ++k) load8<T, VEC>(yr, t + NT * k, D, v[k]);
    if (p.post) normed(v, (const T*)p.post_w, (const T*)p.post_b, red[0], red[1]);
    const T* gr = p.gate ? (const T*)p.gate + (row / p.gate_rows) * D : nullptr;
    H* ho = (H*)p.h_out + row * D;
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      float f[8];
      if (gr) {
        load8<T, VEC>(gr, t + NT * k, D, f);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[k][e] *= f[e];
      }
      load8<H, VEC>(hr, t + NT * k, D, f);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[k][e] = fmaf(p.rho, f[e], v[k][e]);
      store8<H, VEC>(ho, t + NT * k, D, v[k], p.once);
    }
  } else {
#pragma unroll
    for (int k = 0; k < CH; ++k) load8<H, VEC>(hr, t + NT * k, D, v[k]);
  }
  if (!p.u) return;
  normed(v, (const T*)p.pre_w, (const T*)p.pre_b, red[2], red[3]);
  T* ur = (T*)p.u + row * D;
#pragma unroll
  for (int k = 0; k < CH; ++k) store8<T, VEC>(ur, t + NT * k, D, v[k], p.once);
}

template <typename T, typename H, int NW, int CH>
void launch(const NormParams& p, bool vec, hipStream_t s) {
  const dim3 grid((unsigned)(NW == 1 ? (p.M + 3) / 4 : p.M)), block(NW == 1 ? 256 : NW * 64);
  if (vec) kh_launch(KH_TAG_BLOCK_NORM, block_norm_kernel<T, H, NW, CH, true>, grid, block, 0, s, p);
  else kh_launch(KH_TAG_BLOCK_NORM, block_norm_kernel<T, H, NW, CH, false>, grid, block, 0, s, p);
}

// One wave a row where it holds the row in 32 numbers a lane and there are rows enough for all CUs, four or sixteen otherwise: 7904 rows of 1280, stream in
// 16 bits, 22.7 us with four waves and 17.0 with one (floor 15.7 at the rate of a copy), 2048 of 2048 8.3 and 10.3, one of 1280 4.0 and 5.8.  Stored past the
// caches from 8 MB on: 7904 of 1280, stream in 32 bits, 31.0 -> 23.4 us (floor 23.6), 2048 of 8192 31.0 -> 22.3.
template <typename T, typename H>
int dispatch(const NormParams& p, bool vec, hipStream_t s) {
  if (p.D <= 512) launch<T, H, 1, 1>(p, vec, s);
  else if (p.D <= 1024) launch<T, H, 1, 2>(p, vec, s);
  else if (p.D <= 1536 && p.M >= 4096) launch<T, H, 1, 3>(p, vec, s);
  else if (p.D <= 2048 && p.M >= 4096) launch<T, H, 1, 4>(p, vec, s);
  else if (p.D <= 2048) launch<T, H, 4, 1>(p, vec, s);
  else if (p.D <= 4096) launch<T, H, 4, 2>(p, vec, s);
  else if (p.D <= 8192) launch<T, H, 4, 4>(p, vec, s);
  else launch<T, H, 16, 4>(p, vec, s);
  KH_RETURN_LAST_ERROR();
}

}  // namespace

KH_EXPORT int kh_block_norm(const void* y, const void* h, const void* gate, int64_t gate_rows, const void* post_w, const void* post_b,
                            const void* pre_w, const void* pre_b, void* h_out, void* u, int64_t M, int64_t D, float residual_scale,
                            float eps, int flags, int type, int stream_type, void* stream) {
  if (!h || M <= 0 || D <= 0 || (flags & ~3) || type < 0 || type > 2 || stream_type < 0 || stream_type > 2) return KH_ERR_INVALID_ARG;
  const int post = (flags >> 1) & 1;
  if (y ? !h_out : (h_out || gate || post)) return KH_ERR_INVALID_ARG;
  if (!y && !u) return KH_ERR_INVALID_ARG;
  if ((!post && (post_w || post_b)) || (!u && (pre_w || pre_b))) return KH_ERR_INVALID_ARG;
  if (gate && (gate_rows <= 0 || gate_rows > M || M % gate_rows != 0)) return KH_ERR_INVALID_ARG;
  if (stream_type != type && stream_type != 2) return KH_ERR_UNSUPPORTED;
  if (D > 32768) return KH_ERR_TOO_LARGE;
  if (M > 0x7fffffffL || M * (D <= 1024 || (D <= 2048 && M >= 4096) ? 64 : D <= 8192 ? 256 : 1024) > 0xffff0000L) return KH_ERR_TOO_LARGE;   // (threads of a launch)
  NormParams p{y, h, gate, post_w, post_b, pre_w, pre_b, h_out, u, (long)M, (long)(gate ? gate_rows : 1), (int)D, residual_scale, eps, flags & 1, post, 0};
  auto size = [](int t) { return t == 2 ? 4 : 2; };
  p.once = M * D * ((h_out ? size(stream_type) : 0) + (u ? size(type) : 0)) >= 8 << 20;
  bool vec = D % 8 == 0;
  for (const void* a : {y, h, gate, post_w, post_b, pre_w, pre_b, (const void*)h_out, (const void*)u}) vec = vec && kh_aligned16(a);
  hipStream_t s = (hipStream_t)stream;
  if (type == 0) return stream_type == 0 ? dispatch<bf16_t, bf16_t>(p, vec, s) : dispatch<bf16_t, float>(p, vec, s);
  if (type == 1) return stream_type == 1 ? dispatch<_Float16, _Float16>(p, vec, s) : dispatch<_Float16, float>(p, vec, s);
  return dispatch<float, float>(p, vec, s);
}
