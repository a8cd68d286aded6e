// K13: linear attention with a decay for each head, beside K3: a state of dk x dv numbers a head instead of a cache of keys and values.
//   S_t = lambda_h S_{t-1} + k_t v_t^T,   o_t = scale * q_t S_t        (lambda_h = exp(log_decay[h]), S in 32 bits)
// Tokens as in K3: [B, tokens, heads * d] through strides, or packed rows with the first row of every sequence in a table (K2's).
// Query heads share the keys and values of kv_heads; every query head has its own decay and state.
//
// Prompts.  In blocks of 64 tokens the recurrence is four products for the matrix unit: with positions i, j of a block
//   o_i = scale * (sum_{j <= i} lambda^(i-j) (q_i k_j) v_j  +  lambda^(i+1) q_i S),   S' = lambda^n S + sum_j lambda^(n-1-j) k_j v_j^T
// A sequence is cut into segments of whole blocks where there are few heads: each leaves what it adds to the state (la_gain), the sums over the
// segments before each follow (la_scan), and then every segment runs on its own (la_out).
// bf16 operands carry 8 bits, so what is no input is fed to the matrix unit in pieces: scores and states as two (16 bits: their results are
// rounded to bf16), the decayed values that make the state as three (24 bits: the state stays in 32).
#include "kh_common.h"

namespace {

constexpr int C = 64;          // tokens of a block, columns of v of a workgroup

struct LaParams {
  const bf16_t *q, *k, *v;
  bf16_t* o;
  const float* log_decay;
  const float* s_in;
  float* s_out;
  const int32_t* seg_start;    // NULL: [B][T] rows through batch strides
  const int32_t* slots;
  float* ws;                   // [unit][segment][dk * 64]: a segment's gain, then the state before it
  long ldq, ldk, ldv, ldo, bsq, bsk, bsv, bso;
  long rows;                   // of packed tensors
  int B, H, share;             // share: query heads of a key head
  int T, dv, n_slots, nseg, seg;   // seg: tokens of a segment, a multiple of C
  float scale;
};

struct Unit {                  // one (sequence, head, 64 columns of v)
  int b, h, tile, len, slot;
  long q0, k0, v0, o0;         // first elements
  float g;
};

__device__ __forceinline__ bool unit_of(const LaParams& p, long u, int DK, Unit& r) {
  const int tiles = p.dv / C;
  r.tile = (int)(u % tiles);
  r.h = (int)(u / tiles % p.H);
  r.b = (int)(u / tiles / p.H);
  r.slot = p.slots ? p.slots[r.b] : r.b;
  if (r.slot < 0 || r.slot >= p.n_slots) return false;
  long row = 0;
  r.len = p.T;
  r.q0 = (long)r.b * p.bsq; r.k0 = (long)r.b * p.bsk; r.v0 = (long)r.b * p.bsv; r.o0 = (long)r.b * p.bso;
  if (p.seg_start) {           // whatever the table holds, rows stay inside the tensors
    long a = p.seg_start[r.b], e = p.seg_start[r.b + 1];
    a = a < 0 ? 0 : a > p.rows ? p.rows : a;
    e = e < a ? a : e > p.rows ? p.rows : e;
    row = a;
    r.len = (int)(e - a < p.T ? e - a : p.T);
    r.q0 = r.k0 = r.v0 = r.o0 = 0;
  }
  const int hk = r.h / p.share;
  r.q0 += row * p.ldq + (long)r.h * DK;
  r.k0 += row * p.ldk + (long)hk * DK;
  r.v0 += row * p.ldv + (long)hk * p.dv + r.tile * C;
  r.o0 += row * p.ldo + (long)r.h * p.dv + r.tile * C;
  const float g = p.log_decay[r.h];
  r.g = g < -1.0e4f ? -1.0e4f : g;     // (-inf, no memory at all, times a distance of 0 would be no number)
  return true;
}

__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) {
#if __HIP_DEVICE_COMPILE__
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
#else
  return c;
#endif
}

typedef __attribute__((address_space(3))) bf16x4* ltr_t;

// Element i of rows r .. r+3 and r+4 .. r+7 (i = lane % 16) of a bf16 tile in LDS: at = address of row (lane%16)/4 of the first four,
// column 4 (lane % 4) of the sixteen.
__device__ __forceinline__ bf16x8 transposed(const char* at, int row_bytes) {
  bf16x8 v;
#if __HIP_DEVICE_COMPILE__
  const bf16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((ltr_t)(at));
  const bf16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((ltr_t)(at + 4 * row_bytes));
#pragma unroll
  for (int e = 0; e < 4; ++e) { v[e] = a[e]; v[4 + e] = b[e]; }
#endif
  return v;
}

// The 64 x W tile of rows t0 .. t0+63 of a sequence into LDS (row pitch PITCH bytes); rows at and behind len are zero.
template <int W, int PITCH>
__device__ __forceinline__ void tile_in(const bf16_t* src, long ld, int t0, int len, char* dst) {
#pragma unroll
  for (int i = 0; i < C * W / 8 / 256; ++i) {
    const int id = i * 256 + threadIdx.x, row = id / (W / 8), piece = id % (W / 8);
    u32x4 v = u32x4{0, 0, 0, 0};
    if (t0 + row < len) v = *reinterpret_cast<const u32x4*>(src + (long)(t0 + row) * ld + piece * 8);
    *reinterpret_cast<u32x4*>(dst + row * PITCH + piece * 16) = v;
  }
}

// A state (or a segment's gain) in registers: wave w has the columns 16 w .. 16 w + 15 of the 64, lane l of a group g rows 16 t + 4 g + r of column l.
template <int DK>
struct State {
  f32x4 s[DK / 16];
};

template <int DK>
struct Shape {
  static constexpr int KP = DK * 2 + 16, VP = C * 2 + 16, PP = C * 2 + 16;   // pitches in bytes: 16-byte pieces of neighbouring rows on other banks
};

// S = lambda^n S + sum_j lambda^(n-1-j) k_j v_j^T over the n tokens of a block whose K and V lie in LDS.
template <int DK>
__device__ __forceinline__ void add_block(State<DK>& st, const char* kt, const char* vt, int n, float g) {
  typedef Shape<DK> Sh;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane & 15, grp = lane >> 4;
  bf16x8 v[2][3];
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const bf16x8 raw = transposed(vt + (32 * s + 8 * grp + (l >> 2)) * Sh::VP + wave * 32 + (l & 3) * 8, Sh::VP);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int left = n - 1 - (32 * s + 8 * grp + e);
      float w = (float)raw[e] * expf(g * (float)(left < 0 ? 0 : left));
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        v[s][i][e] = (bf16_t)w;
        w -= (float)v[s][i][e];
      }
    }
  }
  const float decay = expf(g * (float)n);
#pragma unroll
  for (int t = 0; t < DK / 16; ++t) {
#pragma unroll
    for (int e = 0; e < 4; ++e) st.s[t][e] *= decay;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const bf16x8 k = transposed(kt + (32 * s + 8 * grp + (l >> 2)) * Sh::KP + t * 32 + (l & 3) * 8, Sh::KP);
#pragma unroll
      for (int i = 0; i < 3; ++i) st.s[t] = mfma(k, v[s][i], st.s[t]);
    }
  }
}

// The state of a slot, dk x dv in rows, to and from the registers' order.
template <int DK>
__device__ __forceinline__ long state_at(const LaParams& p, const Unit& u, int t) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  return (((long)u.slot * p.H + u.h) * DK + 16 * t + 4 * (lane >> 4)) * p.dv + u.tile * C + wave * 16 + (lane & 15);
}

template <int DK>
__global__ __launch_bounds__(256) void la_gain(const LaParams p) {
  typedef Shape<DK> Sh;
  __shared__ __attribute__((aligned(16))) char kt[C * Sh::KP], vt[C * Sh::VP];
  Unit u;
  const long unit = blockIdx.x / p.nseg;
  const int sg = (int)(blockIdx.x % p.nseg);
  if (!unit_of(p, unit, DK, u)) return;
  const int t0 = sg * p.seg, t1 = u.len < t0 + p.seg ? u.len : t0 + p.seg;
  if (t0 >= t1) return;
  State<DK> st;
#pragma unroll
  for (int t = 0; t < DK / 16; ++t) st.s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int c = t0; c < t1; c += C) {
    tile_in<DK, Sh::KP>(p.k + u.k0, p.ldk, c, t1, kt);
    tile_in<C, Sh::VP>(p.v + u.v0, p.ldv, c, t1, vt);
    __syncthreads();
    add_block<DK>(st, kt, vt, t1 - c < C ? t1 - c : C, u.g);
    __syncthreads();
  }
  float* w = p.ws + (unit * p.nseg + sg) * (DK * C);
#pragma unroll
  for (int t = 0; t < DK / 16; ++t) *reinterpret_cast<f32x4*>(w + (((threadIdx.x >> 6) * (DK / 16) + t) * 64 + (threadIdx.x & 63)) * 4) = st.s[t];
}

// Gains to the states before each segment, in place; the state behind the last one to its slot.  A thread has the four rows of la_gain's lane: grid
// (DK / 16, units).
template <int DK>
__global__ __launch_bounds__(256) void la_scan(const LaParams p) {
  Unit u;
  if (!unit_of(p, blockIdx.y, DK, u)) return;
  const int t = blockIdx.x;
  const long at = state_at<DK>(p, u, t);
  f32x4 s = f32x4{0.f, 0.f, 0.f, 0.f};
  if (p.s_in)
#pragma unroll
    for (int r = 0; r < 4; ++r) s[r] = p.s_in[at + (long)r * p.dv];
  float* w = p.ws + (long)blockIdx.y * p.nseg * (DK * C) + (((threadIdx.x >> 6) * (DK / 16) + t) * 64 + (threadIdx.x & 63)) * 4;
  for (int sg = 0; sg * p.seg < u.len; ++sg, w += DK * C) {
    const f32x4 gain = *reinterpret_cast<const f32x4*>(w);
    *reinterpret_cast<f32x4*>(w) = s;
    const int n = u.len - sg * p.seg < p.seg ? u.len - sg * p.seg : p.seg;
    const float d = expf(u.g * (float)n);
#pragma unroll
    for (int r = 0; r < 4; ++r) s[r] = fmaf(d, s[r], gain[r]);
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) p.s_out[at + (long)r * p.dv] = s[r];
}

// A segment's outputs from the state before it.  nseg == 1: the whole sequence from the slot's state, whose successor it leaves.
template <int DK>
__global__ __launch_bounds__(256) void la_out(const LaParams p) {
  typedef Shape<DK> Sh;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  char* kt = smem;                         // [64][KP]
  char* qt = kt + C * Sh::KP;
  char* vt = qt + C * Sh::KP;              // [64][VP]
  char* ph = vt + C * Sh::VP;              // [64][PP]: decayed scores, upper and lower pieces
  char* pl = ph + C * Sh::PP;
  Unit u;
  const long unit = blockIdx.x / p.nseg;
  const int sg = (int)(blockIdx.x % p.nseg);
  if (!unit_of(p, unit, DK, u)) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane & 15, grp = lane >> 4;
  const int t0 = sg * p.seg, t1 = u.len < t0 + p.seg ? u.len : t0 + p.seg;
  State<DK> st;
  if (p.nseg > 1) {
    if (t0 >= t1) return;
    const float* w = p.ws + (unit * p.nseg + sg) * (DK * C);
#pragma unroll
    for (int t = 0; t < DK / 16; ++t) st.s[t] = *reinterpret_cast<const f32x4*>(w + ((wave * (DK / 16) + t) * 64 + lane) * 4);
  } else {
#pragma unroll
    for (int t = 0; t < DK / 16; ++t) {
      const long at = state_at<DK>(p, u, t);
#pragma unroll
      for (int r = 0; r < 4; ++r) st.s[t][r] = p.s_in ? p.s_in[at + (long)r * p.dv] : 0.f;
    }
  }
  // lambda^(i - j) of a tile of scores on the diagonal (rows j = 4 grp + r, column i = l) and, times lambda^(16 m), of the tiles m + 1 beside it
  float diag[4], off[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int d = l - 4 * grp - r;
    diag[r] = d < 0 ? 0.f : p.scale * expf(u.g * (float)d);
    off[r] = p.scale * expf(u.g * (float)(16 + d));
  }
  for (int c = t0; c < t1; c += C) {
    tile_in<DK, Sh::KP>(p.k + u.k0, p.ldk, c, t1, kt);
    tile_in<DK, Sh::KP>(p.q + u.q0, p.ldq, c, t1, qt);
    tile_in<C, Sh::VP>(p.v + u.v0, p.ldv, c, t1, vt);
    __syncthreads();
    // scores of the 16 tokens of this wave against those before them: column i = 16 wave + l, rows j = 16 jt + 4 grp + r
    {
      bf16x8 qf[DK / 32];
#pragma unroll
      for (int s = 0; s < DK / 32; ++s) qf[s] = *reinterpret_cast<const bf16x8*>(qt + (16 * wave + l) * Sh::KP + s * 64 + grp * 16);
      for (int jt = 0; jt <= (wave | 1); ++jt) {
        f32x4 a = f32x4{0.f, 0.f, 0.f, 0.f};
        if (jt <= wave) {
#pragma unroll
          for (int s = 0; s < DK / 32; ++s) a = mfma(*reinterpret_cast<const bf16x8*>(kt + (16 * jt + l) * Sh::KP + s * 64 + grp * 16), qf[s], a);
          const float far = jt == wave ? 1.f : expf(u.g * (float)(16 * (wave - jt - 1)));
#pragma unroll
          for (int r = 0; r < 4; ++r) a[r] *= jt == wave ? diag[r] : off[r] * far;
        }
        bf16x4 hi, lo;
#pragma unroll
        for (int r = 0; r < 4; ++r) { hi[r] = (bf16_t)a[r]; lo[r] = (bf16_t)(a[r] - (float)hi[r]); }
        const int at = (16 * wave + l) * Sh::PP + (16 * jt + 4 * grp) * 2;
        *reinterpret_cast<bf16x4*>(ph + at) = hi;
        *reinterpret_cast<bf16x4*>(pl + at) = lo;
      }
    }
    __syncthreads();
    // outputs of the 16 columns of this wave: rows of the product 4 grp + r of them, column i = 16 it + l
    bf16x8 vf[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) vf[s] = transposed(vt + (32 * s + 8 * grp + (l >> 2)) * Sh::VP + wave * 32 + (l & 3) * 8, Sh::VP);
    bf16x8 sh[DK / 32], sl[DK / 32];       // the state: k-slots e < 4 are rows 32 s + 4 grp + e, the others 16 rows further
#pragma unroll
    for (int s = 0; s < DK / 32; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = st.s[2 * s + e / 4][e % 4];
        sh[s][e] = (bf16_t)x;
        sl[s][e] = (bf16_t)(x - (float)sh[s][e]);
      }
#pragma unroll
    for (int it = 0; it < 4; ++it) {
      f32x4 a = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < DK / 32; ++s) {
        const char* at = qt + (16 * it + l) * Sh::KP + s * 64 + grp * 8;
        const bf16x4 q0 = *reinterpret_cast<const bf16x4*>(at), q1 = *reinterpret_cast<const bf16x4*>(at + 32);
        bf16x8 qf;
#pragma unroll
        for (int e = 0; e < 4; ++e) { qf[e] = q0[e]; qf[4 + e] = q1[e]; }
        a = mfma(sh[s], qf, a);
        a = mfma(sl[s], qf, a);
      }
      const float d = p.scale * expf(u.g * (float)(16 * it + l + 1));
#pragma unroll
      for (int r = 0; r < 4; ++r) a[r] *= d;
#pragma unroll
      for (int s = 0; s <= it / 2; ++s) {
        const int at = (16 * it + l) * Sh::PP + s * 64 + grp * 16;
        a = mfma(vf[s], *reinterpret_cast<const bf16x8*>(ph + at), a);
        a = mfma(vf[s], *reinterpret_cast<const bf16x8*>(pl + at), a);
      }
      const int i = c + 16 * it + l;
      if (i < t1) {
        const u32x2 v = u32x2{pack_bf16x2(a[0], a[1]), pack_bf16x2(a[2], a[3])};
        *reinterpret_cast<u32x2*>(p.o + u.o0 + (long)i * p.ldo + wave * 16 + grp * 4) = v;
      }
    }
    if (p.nseg == 1 || c + C < t1) add_block<DK>(st, kt, vt, t1 - c < C ? t1 - c : C, u.g);
    __syncthreads();
  }
  if (p.nseg == 1)
#pragma unroll
    for (int t = 0; t < DK / 16; ++t) {
      const long at = state_at<DK>(p, u, t);
#pragma unroll
      for (int r = 0; r < 4; ++r) p.s_out[at + (long)r * p.dv] = st.s[t][r];
    }
}

// One token: the state is read and written once, which bounds it.  A workgroup has 64 columns of one head: 16 threads of four columns, 16 rows at a time.
template <int DK>
__global__ __launch_bounds__(256) void la_step(const LaParams p) {
  __shared__ float red[4][C];
  Unit u;
  if (!unit_of(p, blockIdx.x, DK, u)) return;
  const int c4 = (threadIdx.x & 15) * 4, r0 = threadIdx.x >> 4;
  const float d = expf(u.g);
  const bf16x4 vb = *reinterpret_cast<const bf16x4*>(p.v + u.v0 + c4);
  const long base = (((long)u.slot * p.H + u.h) * DK) * p.dv + u.tile * C + c4;
  f32x4 s[DK / 16], o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < DK / 16; ++i) s[i] = *reinterpret_cast<const f32x4*>(p.s_in + base + (long)(r0 + 16 * i) * p.dv);
#pragma unroll
  for (int i = 0; i < DK / 16; ++i) {
    const float k = (float)p.k[u.k0 + r0 + 16 * i], q = (float)p.q[u.q0 + r0 + 16 * i];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      s[i][e] = fmaf(d, s[i][e], k * (float)vb[e]);
      o[e] = fmaf(q, s[i][e], o[e]);
    }
    *reinterpret_cast<f32x4*>(p.s_out + base + (long)(r0 + 16 * i) * p.dv) = s[i];
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    o[e] += __shfl_xor(o[e], 16, 64);
    o[e] += __shfl_xor(o[e], 32, 64);
  }
  if ((threadIdx.x & 63) < 16) *reinterpret_cast<f32x4*>(&red[threadIdx.x >> 6][c4]) = o;
  __syncthreads();
  if (threadIdx.x < C) {
    const int c = threadIdx.x;
    p.o[u.o0 + c] = (bf16_t)(p.scale * ((red[0][c] + red[1][c]) + (red[2][c] + red[3][c])));
  }
}

struct Plan { long units; int nseg, seg; };

// Segments where heads, columns and sequences alone give the CUs too little: about four workgroups a CU, two blocks of 64 tokens each at least.
Plan plan_of(long B, long H, long dv, long T) {
  Plan r;
  r.units = B * H * (dv / C);
  const long blocks = (T + C - 1) / C;
  long n = (1024 + r.units - 1) / r.units;
  if (n > (blocks + 1) / 2) n = (blocks + 1) / 2;
  if (n < 1) n = 1;
  const long per = (blocks + n - 1) / n;
  r.seg = (int)(per * C);
  r.nseg = (int)((blocks + per - 1) / per);
  return r;
}

int check(const LaParams& p, int64_t B, int64_t H, int64_t Hk, int64_t dk, int64_t dv, bool need_state) {
  if (!p.q || !p.k || !p.v || !p.o || !p.log_decay || !p.s_out || (need_state && !p.s_in)) return KH_ERR_INVALID_ARG;
  if (B <= 0 || H <= 0 || Hk <= 0 || dv <= 0 || H % Hk != 0) return KH_ERR_INVALID_ARG;
  if (p.n_slots <= 0 || (!p.slots && p.n_slots < B)) return KH_ERR_INVALID_ARG;
  if ((dk != 64 && dk != 128) || dv % C != 0 || dv > 1024) return KH_ERR_UNSUPPORTED;
  if ((p.ldq | p.ldk | p.ldv | p.ldo | p.bsq | p.bsk | p.bsv | p.bso) % 8 != 0) return KH_ERR_ALIGNMENT;
  if (!kh_aligned16(p.q) || !kh_aligned16(p.k) || !kh_aligned16(p.v) || !kh_aligned16(p.o) || !kh_aligned16(p.s_out) ||
      (p.s_in && !kh_aligned16(p.s_in)))
    return KH_ERR_ALIGNMENT;
  if (B > (1 << 20) || H > (1 << 16) || B * H * (dv / C) > (1L << 30)) return KH_ERR_TOO_LARGE;
  return KH_OK;
}

template <int DK>
int prompt(const LaParams& p, long units, hipStream_t s) {
  typedef Shape<DK> Sh;
  constexpr int lds = C * (2 * Sh::KP + Sh::VP + 2 * Sh::PP);
  if (p.nseg > 1) {
    kh_launch(KH_TAG_LINEAR_ATTENTION, la_gain<DK>, dim3((unsigned)(units * p.nseg)), dim3(256), 0, s, p);
    kh_launch(KH_TAG_LINEAR_ATTENTION, la_scan<DK>, dim3(DK / 16, (unsigned)units), dim3(256), 0, s, p);
  }
  if (lds > 65536) {
    const hipError_t e = kh_allow_lds<la_out<DK>>(lds);
    if (e != hipSuccess) return (int)e;
  }
  kh_launch(KH_TAG_LINEAR_ATTENTION, la_out<DK>, dim3((unsigned)(units * p.nseg)), dim3(256), lds, s, p);
  KH_RETURN_LAST_ERROR();
}

}  // namespace

KH_EXPORT int64_t kh_linear_attention_workspace_bytes(int64_t B, int64_t H, int64_t T, int64_t dk, int64_t dv) {
  if (B <= 0 || H <= 0 || T <= 0 || dv <= 0) return KH_ERR_INVALID_ARG;
  if ((dk != 64 && dk != 128) || dv % C != 0 || dv > 1024) return KH_ERR_UNSUPPORTED;
  if (B > (1 << 20) || H > (1 << 16) || B * H * (dv / C) > (1L << 30) || T > (1L << 30)) return KH_ERR_TOO_LARGE;
  const Plan r = plan_of(B, H, dv, T);
  return r.nseg > 1 ? (int64_t)r.units * r.nseg * dk * C * 4 : 0;
}

KH_EXPORT int kh_linear_attention_bf16(const void* q, const void* k, const void* v, void* o, const float* log_decay, const float* state_in,
                                       float* state_out, const int32_t* slots, int64_t n_slots, const int32_t* seg_start, int64_t rows,
                                       void* workspace, int64_t B, int64_t H, int64_t kv_heads, int64_t T, int64_t dk, int64_t dv, int64_t ldq,
                                       int64_t ldk, int64_t ldv, int64_t ldo, int64_t bsq, int64_t bsk, int64_t bsv, int64_t bso, float scale,
                                       void* stream) {
  if (n_slots > (1L << 30) || rows > (1L << 31)) return KH_ERR_TOO_LARGE;
  LaParams p{(const bf16_t*)q, (const bf16_t*)k, (const bf16_t*)v, (bf16_t*)o, log_decay, state_in, state_out, seg_start, slots, (float*)workspace,
             ldq, ldk, ldv, ldo, bsq, bsk, bsv, bso, (long)rows, (int)B, (int)H, kv_heads > 0 ? (int)(H / kv_heads) : 1, (int)T, (int)dv, (int)n_slots,
             1, 0, scale};
  const int rc = check(p, B, H, kv_heads, dk, dv, false);
  if (rc != KH_OK) return rc;
  if (T <= 0 || (seg_start && rows < 0)) return KH_ERR_INVALID_ARG;
  if (ldq < H * dk || ldk < kv_heads * dk || ldv < kv_heads * dv || ldo < H * dv) return KH_ERR_INVALID_ARG;
  if (T > (1L << 30)) return KH_ERR_TOO_LARGE;
  const Plan r = plan_of(B, H, dv, T);
  p.nseg = r.nseg;
  p.seg = r.seg;
  if (p.nseg > 1 && !workspace) return KH_ERR_INVALID_ARG;
  if (!kh_aligned16(workspace)) return KH_ERR_ALIGNMENT;
  if (r.units * r.nseg > 0x7fffffffL) return KH_ERR_TOO_LARGE;   // (more than 65535 units are never cut: la_scan's grid)
  return dk == 64 ? prompt<64>(p, r.units, (hipStream_t)stream) : prompt<128>(p, r.units, (hipStream_t)stream);
}

KH_EXPORT int kh_linear_attention_step_bf16(const void* q, const void* k, const void* v, void* o, const float* log_decay, const float* state_in,
                                            float* state_out, const int32_t* slots, int64_t n_slots, int64_t B, int64_t H, int64_t kv_heads,
                                            int64_t dk, int64_t dv, int64_t ldq, int64_t ldk, int64_t ldv, int64_t ldo, float scale, void* stream) {
  if (n_slots > (1L << 30)) return KH_ERR_TOO_LARGE;
  LaParams p{(const bf16_t*)q, (const bf16_t*)k, (const bf16_t*)v, (bf16_t*)o, log_decay, state_in, state_out, nullptr, slots, nullptr,
             0, 0, 0, 0, ldq, ldk, ldv, ldo, 0, (int)B, (int)H, kv_heads > 0 ? (int)(H / kv_heads) : 1, 1, (int)dv, (int)n_slots, 1, C, scale};
  const int rc = check(p, B, H, kv_heads, dk, dv, true);
  if (rc != KH_OK) return rc;
  if (ldq < H * dk || ldk < kv_heads * dk || ldv < kv_heads * dv || ldo < H * dv) return KH_ERR_INVALID_ARG;
  const long units = B * H * (dv / C);
  if (dk == 64) kh_launch(KH_TAG_LINEAR_ATTENTION, la_step<64>, dim3((unsigned)units), dim3(256), 0, (hipStream_t)stream, p);
  else kh_launch(KH_TAG_LINEAR_ATTENTION, la_step<128>, dim3((unsigned)units), dim3(256), 0, (hipStream_t)stream, p);
  KH_RETURN_LAST_ERROR();
}
