// K13: linear attention with a decay for each head, beside K3: a state of dk x dv numbers a head instead of a cache of keys and values.
//   S_t = lambda_h S_{t-1} + k_t v_t^T,   o_t = scale * q_t S_t        (lambda_h = exp(log_decay[h]), S in 32 bits)
// Tokens as in K3: [B, tokens, heads * d] through strides, or packed rows with the first row of every sequence in a table (K2's).
// Query heads share the keys and values of kv_heads; every query head has its own decay and state.
//
// Prompts.  In blocks of 64 tokens the recurrence is four products for the matrix unit: with positions i, j of a block
//   o_i = scale * (sum_{j <= i} lambda^(i-j) (q_i k_j) v_j  +  lambda^(i+1) q_i S),   S' = lambda^n S + sum_j lambda^(n-1-j) k_j v_j^T
// Where there are few heads, the blocks of all sequences of a head, one after the other, are cut into equal chunks, wherever a sequence ends: a chunk whose last
// sequence goes on in the next leaves what it adds to that state (la_gain), the sums over the chunks before each follow (la_scan), and then every chunk runs on
// its own (la_out).
// bf16 operands carry 8 bits, so what is no input (scores, states, the decayed values that make the state) is fed to the matrix unit as three pieces of 8: 24 bits,
// those of the 32-bit numbers that they are held in.  Two pieces of scores, states and of the values in chunks where no sequence ends left 2^-18 of a term and cost less (us, two | three:
// 16384 packed tokens of 16 heads of 128 on 8 122 | 135, 2 x 4096 of 20 heads of 64 46.6 | 50.1, 16 x 1024 of 16 heads of 128 83.5 | 89.4, 2 x 77 of 20 heads of 64 the same): terms that cancel
// one another lost what was left of them.
// What bounds it: of 16384 packed tokens of 16 heads of 128 on 8 the workgroups take 31 us in la_gain, 7 in la_scan and 84 .. 97 in la_out, 3 .. 4 lie between launches (the bytes of q, k, v
// and o take 42): 17 blocks a workgroup one after the other at 1.8 and 5.1 us.  Of those 5.1 products are 1.7 (126 of 16 clocks a wave, two waves on a SIMD).  The next block's loads
// are covered by the scores alone: the compiler waits for everything that is on its way in front of the state's first use in the loop, since a state comes from loads before it.
// A workgroup takes 123 KB of LDS, so there is one to a CU.
#include "kh_common.h"
#include <type_traits>

namespace {

constexpr int C = 64;          // tokens of a block; columns of v of four waves

struct LaParams {
  const bf16_t *q, *k, *v;
  bf16_t* o;
  const float* log_decay;
  const float* s_in;
  float* s_out;
  const int32_t* seg_start;    // NULL: [B][T] rows through batch strides
  const int32_t* slots;
  // [unit][chunk][dk * TV] twice: what a chunk adds to the state of its last sequence, then that state; what that sequence began with in the chunk (its slot may
  // be written by the chunk in which it ends).  Then the chunks.
  float* ws;
  long ldq, ldk, ldv, ldo, bsq, bsk, bsv, bso;
  long rows;                   // of packed tensors
  int B, H, share;             // share: query heads of a key head
  int T, dv, n_slots, chunks;  // chunks: 0 where a workgroup has a whole sequence
  float scale;
  int fill;                    // la_step: rows that are left out are zero
};

struct Unit {                  // one (sequence, head, range of columns of v)
  int b, h, tile, len, slot;
  long q0, k0, v0, o0;         // first elements
  float g;                     // log2 of the decay
};

__device__ __forceinline__ int length_of(const LaParams& p, int b, long* first = nullptr) {
  if (!p.seg_start) return p.T;
  long a = p.seg_start[b], e = p.seg_start[b + 1];      // whatever the table holds, rows stay inside the tensors
  a = a < 0 ? 0 : a > p.rows ? p.rows : a;
  e = e < a ? a : e > p.rows ? p.rows : e;
  if (first) *first = a;
  return (int)(e - a < p.T ? e - a : p.T);
}

__device__ __forceinline__ int uniform(int v) {
#if __HIP_DEVICE_COMPILE__
  return __builtin_amdgcn_readfirstlane(v);
#else
  return v;
#endif
}

__device__ __forceinline__ float decay_of(const LaParams& p, int h) {
  const float g = p.log_decay[h];
  return (g < -1.0e4f ? -1.0e4f : g) * 1.4426950408889634f;     // (-inf, no memory at all, times a distance of 0 would be no number)
}

// TV: columns of v of a unit
__device__ __forceinline__ bool unit_of(const LaParams& p, int b, int ht, int DK, int TV, Unit& r) {
  const int tiles = p.dv / TV;
  r.tile = ht % tiles;
  r.h = ht / tiles;
  r.b = b;
  r.slot = p.slots ? uniform(p.slots[r.b]) : r.b;
  if (r.slot < 0 || r.slot >= p.n_slots) return false;
  long row = 0;
  r.len = uniform(length_of(p, r.b, &row));
  row = uniform((int)row);
  r.q0 = (long)r.b * p.bsq; r.k0 = (long)r.b * p.bsk; r.v0 = (long)r.b * p.bsv; r.o0 = (long)r.b * p.bso;
  if (p.seg_start) r.q0 = r.k0 = r.v0 = r.o0 = 0;
  const int hk = r.h / p.share;
  r.q0 += row * p.ldq + (long)r.h * DK;
  r.k0 += row * p.ldk + (long)hk * DK;
  r.v0 += row * p.ldv + (long)hk * p.dv + r.tile * TV;
  r.o0 += row * p.ldo + (long)r.h * p.dv + r.tile * TV;
  r.g = decay_of(p, r.h);
  return true;
}

// lambda^n (the product's rounding is 2^-24 of the exponent, which is small wherever the power is not)
__device__ __forceinline__ float power(float g, int n) {
#if __HIP_DEVICE_COMPILE__
  return __builtin_amdgcn_exp2f(g * (float)n);
#else
  return g;
#endif
}

__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) {
#if __HIP_DEVICE_COMPILE__
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
#else
  return c;
#endif
}

typedef __attribute__((address_space(3))) void* lptr_t;
typedef __amdgpu_buffer_rsrc_t rsrc_t;

// All loads and stores but the last VM are done (they end in the order of their issue).
template <int VM = 0>
__device__ __forceinline__ void wait_vm() {
  static_assert(VM < 16, "the counter's lower four bits; the upper ones, 14 and 15, stay 0");
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(VM | (7 << 4) | (15 << 8));   // the other counters unconstrained (gfx9 encoding)
  asm volatile("" ::: "memory");
}
__device__ __forceinline__ void barrier() {                // what this wave has written to LDS is there, and everybody has arrived
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// A block's 64 x W tile in LDS, rows unpadded (they come by DMA), their 16-byte pieces swizzled so that the 16 rows of an operand lie on
// different banks.
template <int W>
struct Tile {
  static constexpr int PIECES = W / 8, ROW = W * 2, BYTES = C * ROW;
  // Sixteen rows at one piece lie on all banks, and so do the four pieces of four rows in a row that a transposing read takes.
  static __device__ __forceinline__ int swz(int row) { return (PIECES < 16 ? (row >> 1 & 1) << 2 : (row & 3) << 2) | (row >> 2 & 3); }
  // Loads of a wave of NW, and what a lane's are from the first row (below 2^31: rows of 2^24 elements and more are refused).
  template <int NW>
  struct Lanes {
    static constexpr int N = BYTES / 1024 / NW;
    uint32_t off[N];
    __device__ __forceinline__ explicit Lanes(long ld) {
      const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int id = (wave * N + i) * 64 + lane, row = id / PIECES, piece = (id % PIECES) ^ swz(row);
        off[i] = (uint32_t)row * (uint32_t)ld * 2u + (uint32_t)piece * 16u;
      }
    }
    // rows 0 .. left-1 from src; those behind them lie behind the buffer's end (ld >= W): zeros
    __device__ __forceinline__ void fetch(const bf16_t* src, long ld, int left, char* dst) const {
#if __HIP_DEVICE_COMPILE__
      const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
      const rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<bf16_t*>(src), 0, (int)(((uint32_t)((left < C ? left : C) - 1) * (uint32_t)ld + W) * 2), 0x00020000);
#pragma unroll
      for (int i = 0; i < N; ++i) __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lptr_t)(dst + (wave * N + i) * 1024), 16, off[i], 0, 0, 0);
#endif
    }
  };
  // where a lane (l = lane % 16, g = lane / 16) of an operand finds eight elements of row l from column 32 s + 8 g; rows 16 further lie 16 * ROW further
  static __device__ __forceinline__ int at8(int l, int g, int s) { return l * ROW + ((4 * s + g) ^ swz(l)) * 16; }
  // LDS addresses, for columns(), of row 8 (lane / 16) + (lane % 16) / 4 and of the row four further: a transposing read gives lane i of 16 the i-th element
  // of four rows, of which lanes 4 r .. 4 r + 3 address the r-th, four elements each.  PAIRS: the four are eight columns apart, and two tiles of 16 columns
  // make 32: lane i of tile h has column 8 (i / 4) + 4 h + i % 4.  A product whose rows are such columns leaves them in the order in which the next one takes
  // them as its operand, eight in a row to a lane.
  template <bool PAIRS>
  static __device__ __forceinline__ void column_rows(const char* t, uint32_t (&at)[2]) {
#if __HIP_DEVICE_COMPILE__
    const int lane = threadIdx.x & 63, l = lane & 15;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = 8 * (lane >> 4) + (l >> 2) + 4 * h;
      at[h] = (uint32_t)(uintptr_t)(lptr_t)(const_cast<char*>(t)) + row * ROW + ((PAIRS ? l & 3 : (l & 3) >> 1) ^ swz(row)) * 16 + (PAIRS ? 0 : (l & 1) * 8);
    }
#endif
  }
  // N operands whose lanes have the columns of tile t0 + n (N 4: t0 is a multiple of four, columns in PAIRS) of rows 32 s + 8 (lane / 16) .. + 7, s = 0, 1.  The reads are written out, with
  // their wait: in front of one of its own the compiler waits for every load that is on its way to LDS, the next block's among them.
  template <int N>
  static __device__ __forceinline__ void columns(const uint32_t (&at)[2], int t0, bf16x8 (&v)[N][2]) {
#if __HIP_DEVICE_COMPILE__
    static_assert(N == 1 || N == 4, "one or four tiles of columns");
    u32x2 r[N][4];
    const uint32_t a0 = at[0] ^ (uint32_t)(t0 << 5), b0 = at[1] ^ (uint32_t)(t0 << 5);
    if constexpr (N == 1) {
      asm volatile("ds_read_b64_tr_b16 %0, %4 offset:%7\n\tds_read_b64_tr_b16 %1, %5 offset:%7\n\tds_read_b64_tr_b16 %2, %4 offset:%6\n\tds_read_b64_tr_b16 %3, %5 offset:%6\n\t"
                   "s_waitcnt lgkmcnt(0)"
                   : "=&v"(r[0][0]), "=&v"(r[0][1]), "=&v"(r[0][2]), "=&v"(r[0][3]) : "v"(a0), "v"(b0), "i"(32 * ROW), "i"(0) : "memory");
    } else {
      const uint32_t a1 = a0 ^ 64u, b1 = b0 ^ 64u;
      asm volatile("ds_read_b64_tr_b16 %0, %16 offset:%21\n\tds_read_b64_tr_b16 %1, %17 offset:%21\n\tds_read_b64_tr_b16 %2, %16 offset:%20\n\tds_read_b64_tr_b16 %3, %17 offset:%20\n\t"
                   "ds_read_b64_tr_b16 %4, %16 offset:%23\n\tds_read_b64_tr_b16 %5, %17 offset:%23\n\tds_read_b64_tr_b16 %6, %16 offset:%22\n\tds_read_b64_tr_b16 %7, %17 offset:%22\n\t"
                   "ds_read_b64_tr_b16 %8, %18 offset:%21\n\tds_read_b64_tr_b16 %9, %19 offset:%21\n\tds_read_b64_tr_b16 %10, %18 offset:%20\n\tds_read_b64_tr_b16 %11, %19 offset:%20\n\t"
                   "ds_read_b64_tr_b16 %12, %18 offset:%23\n\tds_read_b64_tr_b16 %13, %19 offset:%23\n\tds_read_b64_tr_b16 %14, %18 offset:%22\n\tds_read_b64_tr_b16 %15, %19 offset:%22\n\t"
                   "s_waitcnt lgkmcnt(0)"
                   : "=&v"(r[0][0]), "=&v"(r[0][1]), "=&v"(r[0][2]), "=&v"(r[0][3]), "=&v"(r[1][0]), "=&v"(r[1][1]), "=&v"(r[1][2]), "=&v"(r[1][3]), "=&v"(r[2][0]), "=&v"(r[2][1]), "=&v"(r[2][2]), "=&v"(r[2][3]), "=&v"(r[3][0]), "=&v"(r[3][1]), "=&v"(r[3][2]), "=&v"(r[3][3])
                   : "v"(a0), "v"(b0), "v"(a1), "v"(b1), "i"(32 * ROW), "i"(0), "i"(8 + 32 * ROW), "i"(8) : "memory");
    }
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int s = 0; s < 2; ++s) v[n][s] = __builtin_bit_cast(bf16x8, u32x4{r[n][2 * s][0], r[n][2 * s][1], r[n][2 * s + 1][0], r[n][2 * s + 1][1]});
#endif
  }
};

// A state (or a segment's gain) in registers: wave w has the columns 16 w .. 16 w + 15, lane l of a group g the rows 16 (t & ~1) + 8 g + 4 (t & 1) + r of column l:
// a pair of tiles is eight rows in a row, an operand's order.
template <int DK>
struct State {
  f32x4 s[DK / 16];
};

__device__ __forceinline__ bool not_finite(const bf16x8 (&v)[2]) {
  uint32_t any = 0;                        // an exponent of ones carries into the sign's place
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int i = 0; i < 4; ++i) any |= (__builtin_bit_cast(u32x4, v[s])[i] & 0x7fff7fffu) + 0x00800080u;
  return (any & 0x80008000u) != 0;
}

// lambda^(n-1-j) of the tokens j = 32 s + 8 g + e of a block of n
__device__ __forceinline__ void powers(float g, int n, float (&w)[2][8]) {
  const int grp = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int left = n - 1 - (32 * s + 8 * grp + e);
      w[s][e] = power(g, left < 0 ? 0 : left);
    }
}

// Two numbers' upper pieces of bf16, which are taken off them.
__device__ __forceinline__ uint32_t take_pieces(float& x0, float& x1) {
  const uint32_t h = pack_bf16x2(x0, x1);
  x0 -= __uint_as_float(h << 16);
  x1 -= __uint_as_float(h & 0xffff0000u);
  return h;
}

// S = decay S + sum_j w_j k_j v_j^T over a block: V as the wave's columns, K in LDS; decayed values in three pieces of bf16.
template <int DK>
__device__ __forceinline__ void add_block(State<DK>& st, const bf16x8 (&raw)[2], const uint32_t (&kcol)[2], float decay, const float (&w)[2][8]) {
  u32x4 v[3][2];
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t two = __builtin_bit_cast(u32x4, raw[s])[e];
      float x0 = __uint_as_float(two << 16) * w[s][2 * e], x1 = __uint_as_float(two & 0xffff0000u) * w[s][2 * e + 1];
      v[0][s][e] = take_pieces(x0, x1);
      v[1][s][e] = take_pieces(x0, x1);
      v[2][s][e] = pack_bf16x2(x0, x1);
    }
#pragma unroll
  for (int t = 0; t < DK / 16; t += 4) {
    bf16x8 k[4][2];
    Tile<DK>::template columns<4>(kcol, t, k);
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) st.s[t + n][e] *= decay;
    auto piece = [&](int i) {
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int n = 0; n < 4; ++n) st.s[t + n] = mfma(k[n][s], __builtin_bit_cast(bf16x8, v[i][s]), st.s[t + n]);   // (four sums in turn: a product waits for the one before it in its own)
    };
    piece(0);
    piece(1);
    piece(2);
  }
}

// First row of a lane's four of tile t in a slot's state, dk x dv in rows.
template <int DK, int TV>
__device__ __forceinline__ long state_at(const LaParams& p, const Unit& u, int wave, int t) {
  const int lane = threadIdx.x & 63;
  return (((long)u.slot * p.H + u.h) * DK + 16 * (t & ~1) + 8 * (lane >> 4) + 4 * (t & 1)) * p.dv + u.tile * TV + wave * 16 + (lane & 15);
}
template <int DK>
__device__ __forceinline__ int ws_at(int wave, int t) { return ((wave * (DK / 16) + t) * 64 + (threadIdx.x & 63)) * 4; }

// The workgroup's head and columns, and its chunk or sequence.  Units that share keys and values are neighbours on one XCD; such clusters go round the eight.
template <int TV>
__device__ __forceinline__ bool work_of(const LaParams& p, int& ht, int& which) {
  const uint32_t tiles = (uint32_t)(p.dv / TV), size = tiles * (uint32_t)p.share, kv = (uint32_t)p.H / (uint32_t)p.share;
  const uint32_t local = blockIdx.x / 8, cluster = local / size * 8 + blockIdx.x % 8;
  which = (int)(cluster / kv);
  ht = (int)((cluster % kv) * size + local % size);
  return which < (p.chunks ? p.chunks : p.B);
}

// Blocks of a sequence: none where it is left out.
__device__ __forceinline__ int blocks_of(const LaParams& p, int b) {
  if (p.slots) {
    const int slot = p.slots[b];
    if (slot < 0 || slot >= p.n_slots) return 0;
  }
  return (length_of(p, b) + C - 1) / C;
}

struct Chunk {
  int b, block, count;         // its first sequence and block in it, blocks
  int tail;                    // blocks of its last sequence where that goes on in the next chunk: from the sequence's start, or, negative, from the chunk's
};
// The chunk's place among the blocks of all sequences, and the sequence that goes on (all NT threads; LDS: 8 NT / 64 + 16 bytes, dead afterwards).
template <int NT>
__device__ __forceinline__ Chunk chunk_of(const LaParams& p, int chunk, int& goes_on, char* lds) {
  constexpr int NW = NT / 64;
  long* sums = reinterpret_cast<long*>(lds);
  int* at = reinterpret_cast<int*>(lds + NW * 8);
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, per = (p.B + NT - 1) / NT;
  const int b0 = t * per < p.B ? t * per : p.B, b1 = b0 + per < p.B ? b0 + per : p.B;
  long mine = 0;
  for (int b = b0; b < b1; ++b) mine += blocks_of(p, b);
  long upto = mine;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const long v = __shfl_up(upto, o, 64);
    if (lane >= o) upto += v;
  }
  if (lane == 63) sums[wave] = upto;
  __syncthreads();
  long before = upto - mine, total = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    if (w < wave) before += sums[w];
    total += sums[w];
  }
  const uint32_t all = (uint32_t)(total < (1L << 30) ? total : 1L << 30);      // (more than that only where a table names the same rows again and again)
  const uint32_t size = (all + (uint32_t)p.chunks - 1) / (uint32_t)p.chunks;
  const long first = (long)size * chunk, next = first + size;
  auto find = [&](long target, int to) {
    if (target < before || target >= before + mine) return;
    long r = target - before;
    int b = b0;
    for (int n; b < b1 - 1 && r >= (n = blocks_of(p, b)); ++b) r -= n;
    at[to] = b;
    at[to + 1] = (int)r;
  };
  find(first, 0);
  find(next, 2);
  __syncthreads();
  Chunk c{0, 0, 0, 0};
  if (first < all) {
    c.b = __builtin_amdgcn_readfirstlane(at[0]);
    c.block = __builtin_amdgcn_readfirstlane(at[1]);
    c.count = (int)(next < all ? size : all - first);
    if (next < all) {
      goes_on = __builtin_amdgcn_readfirstlane(at[2]);
      const int done = __builtin_amdgcn_readfirstlane(at[3]);
      c.tail = done <= c.count ? done : -c.count;
    }
  }
  __syncthreads();
  return c;
}
__device__ __forceinline__ Chunk* chunks_at(const LaParams& p, int DK, int TV) {
  return reinterpret_cast<Chunk*>(p.ws + 2 * (long)p.H * (p.dv / TV) * p.chunks * (DK * TV));
}

template <int DK, int TV>
__global__ __launch_bounds__(TV * 4) void la_gain(const LaParams p) {
  constexpr int NW = TV / 16, STAGE = Tile<DK>::BYTES + Tile<TV>::BYTES;
  extern __shared__ __attribute__((aligned(16))) char smem[];   // two stages of K, V
  int ht, chunk, b = 0;
  if (!work_of<TV>(p, ht, chunk)) return;
  const Chunk ch = chunk_of<TV * 4>(p, chunk, b, smem);
  if (ht == 0 && threadIdx.x == 0) chunks_at(p, DK, TV)[chunk] = ch;
  if (ch.tail == 0) return;
  Unit u;
  if (!unit_of(p, b, ht, DK, TV, u)) return;
  const int t0 = ch.tail > 0 ? 0 : ch.block * C, t1 = t0 + (ch.tail > 0 ? ch.tail : -ch.tail) * C;     // (whole blocks: the sequence goes on)
  const typename Tile<DK>::template Lanes<NW> kl(p.ldk);
  const typename Tile<TV>::template Lanes<NW> vl(p.ldv);
  auto fetch = [&](int c, int to) {
    kl.fetch(p.k + u.k0 + (long)c * p.ldk, p.ldk, C, smem + to);
    vl.fetch(p.v + u.v0 + (long)c * p.ldv, p.ldv, C, smem + to + Tile<DK>::BYTES);
  };
  fetch(t0, 0);
  State<DK> st;
#pragma unroll
  for (int t = 0; t < DK / 16; ++t) st.s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  float w[2][8];
  powers(u.g, C, w);
  const float decay = power(u.g, C);
  uint32_t kcol[2], vcol[2];
  Tile<DK>::template column_rows<true>(smem, kcol);
  Tile<TV>::template column_rows<false>(smem + Tile<DK>::BYTES, vcol);
#pragma unroll
  for (int h = 0; h < 2; ++h) vcol[h] ^= (uint32_t)(threadIdx.x >> 6) << 5;
  for (int c = t0, st_at = 0; c < t1; c += C) {
    wait_vm();
    barrier();                             // everybody's share of this block; and nobody reads the block before any more
    const int other = STAGE - st_at;
    if (c + C < t1) fetch(c + C, other);
    bf16x8 vf[1][2];
    Tile<TV>::template columns<1>(vcol, 0, vf);
    add_block<DK>(st, vf[0], kcol, decay, w);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      vcol[h] += other - st_at;
      kcol[h] += other - st_at;
    }
    st_at = other;
  }
  float* ws = p.ws + ((long)ht * p.chunks + chunk) * (DK * TV);
#pragma unroll
  for (int t = 0; t < DK / 16; ++t) *reinterpret_cast<f32x4*>(ws + ws_at<DK>(threadIdx.x >> 6, t)) = st.s[t];
}

// Gains to the states that the next chunks begin with, in place, and the states of sequences without tokens to their slots.  A thread has the four rows of
// la_gain's lane: grid (DK / 16, units).
template <int DK, int TV>
__global__ __launch_bounds__(TV * 4) void la_scan(const LaParams p) {
  constexpr int NT = TV * 4, AHEAD = 8;
  __shared__ int empty[NT], n_empty;
  const int ht = blockIdx.y, t = blockIdx.x, wave = threadIdx.x >> 6;
  const Chunk* ch = chunks_at(p, DK, TV);
  float* w = p.ws + (long)ht * p.chunks * (DK * TV) + ws_at<DK>(wave, t);
  const long starts = (long)gridDim.y * p.chunks * (DK * TV);
  const float g = decay_of(p, ht / (p.dv / TV));
  auto start_of = [&](int b) {             // the state that a sequence begins with
    f32x4 s = f32x4{0.f, 0.f, 0.f, 0.f};
    Unit u;
    if (p.s_in && unit_of(p, b, ht, DK, TV, u)) {
      const long at = state_at<DK, TV>(p, u, wave, t);
#pragma unroll
      for (int r = 0; r < 4; ++r) s[r] = p.s_in[at + (long)r * p.dv];
    }
    return s;
  };
  f32x4 s = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int c0 = 0; c0 < p.chunks - 1; c0 += AHEAD) {     // so many on their way at a time
    f32x4 gain[AHEAD], start[AHEAD];
    int tail[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) tail[i] = c0 + i < p.chunks - 1 ? __builtin_amdgcn_readfirstlane(ch[c0 + i].tail) : 0;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      if (tail[i] != 0) gain[i] = *reinterpret_cast<const f32x4*>(w + (long)(c0 + i) * (DK * TV));
      if (tail[i] > 0) start[i] = start_of(__builtin_amdgcn_readfirstlane(ch[c0 + i + 1].b));
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      if (tail[i] == 0) continue;
      if (tail[i] > 0) {
        s = start[i];
        if (p.s_in) *reinterpret_cast<f32x4*>(w + starts + (long)(c0 + i) * (DK * TV)) = s;
      }
      const float d = power(g, C * (tail[i] > 0 ? tail[i] : -tail[i]));
#pragma unroll
      for (int r = 0; r < 4; ++r) s[r] = fmaf(d, s[r], gain[i][r]);
      *reinterpret_cast<f32x4*>(w + (long)(c0 + i) * (DK * TV)) = s;
    }
  }
  if (p.s_in == p.s_out) return;
  for (int b0 = 0; b0 < p.B; b0 += NT) {
    if (threadIdx.x == 0) n_empty = 0;
    __syncthreads();
    const int b = b0 + threadIdx.x;
    if (b < p.B && length_of(p, b) == 0) empty[atomicAdd(&n_empty, 1)] = b;       // (in any order: their slots are distinct)
    __syncthreads();
    for (int i = 0; i < n_empty; ++i) {
      Unit u;
      const int e = empty[i];
      if (!unit_of(p, e, ht, DK, TV, u)) continue;
      const f32x4 s0 = start_of(e);
      const long at = state_at<DK, TV>(p, u, wave, t);
#pragma unroll
      for (int r = 0; r < 4; ++r) p.s_out[at + (long)r * p.dv] = s0[r];
    }
    __syncthreads();
  }
}

// The outputs of a chunk, sequence by sequence from the state before it, and the states behind those that end in it.  ONE: one whole sequence.
template <int DK, int TV>
struct OutShape {
  static constexpr int PP = C * 2 + 16;    // pitch of the scores in bytes: 16-byte pieces of neighbouring rows on other banks
  static constexpr int STAGE = 2 * Tile<DK>::BYTES + Tile<TV>::BYTES, LDS = 2 * STAGE + 3 * C * PP;
};
template <int DK, int TV, bool ONE>
__global__ __launch_bounds__(TV * 4) __attribute__((amdgpu_waves_per_eu(2, 2))) void la_out(const LaParams p) {
  typedef OutShape<DK, TV> Sh;
  constexpr int NW = TV / 16;
  extern __shared__ __attribute__((aligned(16))) char smem[];   // two stages of K, Q, V; decayed scores in three pieces
  char* const ph = smem + 2 * Sh::STAGE;
  Unit u;
  int ht, which, left = 0, t0 = 0, t1;     // left: blocks of the chunk; t0, t1: tokens of the sequence
  if (!work_of<TV>(p, ht, which)) return;
  if constexpr (ONE) {
    if (!unit_of(p, which, ht, DK, TV, u)) return;
    t1 = u.len;
  } else {
    const Chunk ch = chunks_at(p, DK, TV)[which];
    left = __builtin_amdgcn_readfirstlane(ch.count);
    if (left == 0 || !unit_of(p, __builtin_amdgcn_readfirstlane(ch.b), ht, DK, TV, u)) return;
    t0 = __builtin_amdgcn_readfirstlane(ch.block) * C;
    t1 = u.len - t0 <= left * (long)C ? u.len : t0 + left * C;
  }
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane & 15, grp = lane >> 4;
  const typename Tile<DK>::template Lanes<NW> kl(p.ldk), ql(p.ldq);
  const typename Tile<TV>::template Lanes<NW> vl(p.ldv);
  auto fetch = [&](int c, int stage) {
    char* to = smem + stage;
    kl.fetch(p.k + u.k0 + (long)c * p.ldk, p.ldk, t1 - c, to);
    ql.fetch(p.q + u.q0 + (long)c * p.ldq, p.ldq, t1 - c, to + Tile<DK>::BYTES);
    vl.fetch(p.v + u.v0 + (long)c * p.ldv, p.ldv, t1 - c, to + 2 * Tile<DK>::BYTES);
  };
  if (t0 < t1) fetch(t0, 0);
  State<DK> st;
  const long slot = ((long)ht * p.chunks + which) * (DK * TV), starts = (long)p.H * (p.dv / TV) * p.chunks * (DK * TV);
  auto state_in = [&]() {                  // before token t0
    if (ONE || (t0 == 0 && (t1 == u.len || !p.s_in))) {
#pragma unroll
      for (int t = 0; t < DK / 16; ++t) {
        const long at = state_at<DK, TV>(p, u, wave, t);
#pragma unroll
        for (int r = 0; r < 4; ++r) st.s[t][r] = p.s_in ? p.s_in[at + (long)r * p.dv] : 0.f;
      }
    } else {
      const float* from = p.ws + (t0 == 0 ? starts + slot : slot - DK * TV);
#pragma unroll
      for (int t = 0; t < DK / 16; ++t) st.s[t] = *reinterpret_cast<const f32x4*>(from + ws_at<DK>(wave, t));
    }
  };
  state_in();
  // scale * lambda^(i - j) of a tile of scores on the diagonal (rows j = 4 grp + r, column i = l) and, but for lambda^(16 m), of the tiles m + 1 beside it
  float diag[4], off[4], far[3], rise[4], w[2][8];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int d = l - 4 * grp - r;
    diag[r] = d < 0 ? 0.f : p.scale * power(u.g, d);
    off[r] = p.scale * power(u.g, 16 + d);
    rise[r] = p.scale * power(u.g, 16 * r + l + 1);   // of the state, for the tokens 16 r + l
  }
#pragma unroll
  for (int m = 0; m < 3; ++m) far[m] = power(u.g, 16 * m);
  powers(u.g, C, w);
  float decay = power(u.g, C);
  // the 16 tokens whose scores a wave computes, and (of eight waves) every other tile of the tokens before them
  const int it0 = wave & 3, j0 = NW == 8 ? wave >> 2 : 0;
  constexpr int JS = NW == 8 ? 2 : 1;
  int a8[DK / 32];
#pragma unroll
  for (int s = 0; s < DK / 32; ++s) a8[s] = Tile<DK>::at8(l, grp, s);
  uint32_t kcol[2], vcol[2];
  Tile<DK>::template column_rows<true>(smem, kcol);
  Tile<TV>::template column_rows<false>(smem + 2 * Tile<DK>::BYTES, vcol);
#pragma unroll
  for (int h = 0; h < 2; ++h) vcol[h] ^= (uint32_t)wave << 5;
  const int p_to = (16 * it0 + l) * Sh::PP + (16 * j0 + 4 * grp) * 2, p_from = l * Sh::PP + grp * 16;
  // (a lane stores eight columns of one of two rows that are 16 apart)
  const int orow_at = l + 16 * (grp & 1);
  const uint32_t ocol = (wave * 16 + (grp >> 1) * 8) * 2;
  bool ends = ONE || t1 == u.len;          // the sequence, in this chunk

  int stage = 0;                           // the block's; a8, kcol and vcol lie in it
  auto block = [&](int c) {
    constexpr int KT = 0, QT = Tile<DK>::BYTES;
    const int other = Sh::STAGE - stage;
    if (c != t0) wait_vm<2>();             // (the outputs of the block before may still be on their way)
    else wait_vm();                        // (a sequence's first block: the state behind the one before is waited for with it)
    barrier();                             // everybody's share of this block; and nobody reads the block before any more
    if (c + C < t1) fetch(c + C, other);
    {
      bf16x8 qf[DK / 32];
#pragma unroll
      for (int s = 0; s < DK / 32; ++s) qf[s] = *reinterpret_cast<const bf16x8*>(smem + a8[s] + it0 * (16 * Tile<DK>::ROW) + QT);
#pragma unroll
      for (int i = 0; i < 4 / JS; ++i) {
        const int jt = j0 + JS * i;        // (the tile behind an even one on the diagonal is read with it: zeros)
        if (jt > (it0 | 1)) continue;
        f32x4 a = f32x4{0.f, 0.f, 0.f, 0.f};
        if (jt <= it0) {
#pragma unroll
          for (int s = 0; s < DK / 32; ++s) a = mfma(*reinterpret_cast<const bf16x8*>(smem + a8[s] + j0 * (16 * Tile<DK>::ROW) + JS * i * (16 * Tile<DK>::ROW) + KT), qf[s], a);
          const int m = it0 - jt;
          if (m == 0) {
#pragma unroll
            for (int r = 0; r < 4; ++r) a[r] = 4 * grp + r > l ? 0.f : a[r] * diag[r];   // (a later key may be no number)
          } else {
            const float f = m == 1 ? far[0] : m == 2 ? far[1] : far[2];
#pragma unroll
            for (int r = 0; r < 4; ++r) a[r] *= off[r] * f;
          }
        }
        float x0 = a[0], x1 = a[1], x2 = a[2], x3 = a[3];
        *reinterpret_cast<u32x2*>(ph + p_to + JS * i * 32) = u32x2{take_pieces(x0, x1), take_pieces(x2, x3)};
        *reinterpret_cast<u32x2*>(ph + C * Sh::PP + p_to + JS * i * 32) = u32x2{take_pieces(x0, x1), take_pieces(x2, x3)};
        *reinterpret_cast<u32x2*>(ph + 2 * C * Sh::PP + p_to + JS * i * 32) = u32x2{pack_bf16x2(x0, x1), pack_bf16x2(x2, x3)};
      }
    }
    // the state's share of the outputs of this wave's 16 columns: rows of the product 4 grp + r of them, columns i = 16 it + l
    f32x4 a[4];
    {
      u32x4 piece[3][DK / 32];
#pragma unroll
      for (int s = 0; s < DK / 32; ++s)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float x0 = st.s[2 * s + e / 2][2 * (e % 2)], x1 = st.s[2 * s + e / 2][2 * (e % 2) + 1];
          piece[0][s][e] = take_pieces(x0, x1);
          piece[1][s][e] = take_pieces(x0, x1);
          piece[2][s][e] = pack_bf16x2(x0, x1);
        }
#pragma unroll
      for (int it = 0; it < 4; ++it) a[it] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < DK / 32; ++s) {
        bf16x8 qf[4];
#pragma unroll
        for (int it = 0; it < 4; ++it) qf[it] = *reinterpret_cast<const bf16x8*>(smem + a8[s] + it * (16 * Tile<DK>::ROW) + QT);
#pragma unroll
        for (int i = 0; i < 3; ++i)
#pragma unroll
          for (int it = 0; it < 4; ++it) a[it] = mfma(__builtin_bit_cast(bf16x8, piece[i][s]), qf[it], a[it]);
      }
#pragma unroll
      for (int it = 0; it < 4; ++it)
#pragma unroll
        for (int r = 0; r < 4; ++r) a[it][r] *= rise[it];
    }
    bf16x8 vf[1][2];
    Tile<TV>::template columns<1>(vcol, 0, vf);
    if (__ballot(not_finite(vf[0])) != 0) {  // their products with the zeros of earlier tokens would be no numbers: taken out, and their columns marked from there on
      int first = C;
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = (float)vf[0][s][e];
          if (!(fabsf(x) <= 3.4e38f)) {
            const int j = 32 * s + 8 * grp + e;
            first = first < j ? first : j;
            vf[0][s][e] = (bf16_t)0.f;
          }
        }
      first = min(first, __shfl_xor(first, 16, 64));
      first = min(first, __shfl_xor(first, 32, 64));
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int from = __shfl(first, 4 * grp + r, 64);
#pragma unroll
        for (int it = 0; it < 4; ++it)
          if (16 * it + l >= from) a[it][r] = __builtin_nanf("");
      }
      if (first < C)
#pragma unroll
        for (int t = 0; t < DK / 16; ++t) st.s[t] = f32x4{__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
    }
    barrier();                             // the scores
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int i = 0; i < 3; ++i)
#pragma unroll
        for (int it = 2 * s; it < 4; ++it) a[it] = mfma(vf[0][s], *reinterpret_cast<const bf16x8*>(ph + i * C * Sh::PP + p_from + it * (16 * Sh::PP) + s * 64), a[it]);
    }
#if __HIP_DEVICE_COMPILE__
    const rsrc_t ro = __builtin_amdgcn_make_buffer_rsrc(p.o + u.o0 + (long)c * p.ldo, 0, (int)(uint32_t)((((t1 - c < C ? t1 - c : C) - 1) * p.ldo + TV) * 2), 0x00020000);
#endif
#pragma unroll
    for (int it = 0; it < 4; it += 2) {
      // a lane has four columns of row l of either tile; those of one tile and of the other trade places between the lanes of a pair of groups
#if __HIP_DEVICE_COMPILE__
      const auto s0 = __builtin_amdgcn_permlane16_swap(pack_bf16x2(a[it][0], a[it][1]), pack_bf16x2(a[it + 1][0], a[it + 1][1]), false, false);
      const auto s1 = __builtin_amdgcn_permlane16_swap(pack_bf16x2(a[it][2], a[it][3]), pack_bf16x2(a[it + 1][2], a[it + 1][3]), false, false);
      const int row = 16 * it + orow_at;     // (always a store: how many there are is what the next block's wait goes by)
      __builtin_amdgcn_raw_buffer_store_b128(u32x4{s0[0], s1[0], s0[1], s1[1]}, ro, c + row < t1 ? (int)((uint32_t)row * (uint32_t)p.ldo * 2u + ocol) : (int)0xfffffff0u, 0, 0);
#endif
    }
    if (ends || c + C < t1) {
      if (t1 - c < C) {
        powers(u.g, t1 - c, w);
        decay = power(u.g, t1 - c);
      }
      add_block<DK>(st, vf[0], kcol, decay, w);
    }
#pragma unroll
    for (int s = 0; s < DK / 32; ++s) a8[s] += other - stage;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      kcol[h] += other - stage;
      vcol[h] += other - stage;
    }
    stage = other;
  };
  for (;;) {
    for (int c = t0; c < t1; c += C) block(c);
    const Unit was = u;
    bool more = false;
    if constexpr (!ONE) {                  // the next sequence with tokens
      left -= (t1 - t0 + C - 1) / C;
      if (left > 0)
        for (int b = was.b + 1; b < p.B && !more; ++b) more = unit_of(p, b, ht, DK, TV, u) && u.len > 0;
      if (more) {
        t0 = 0;
        t1 = u.len <= left * (long)C ? u.len : left * C;
        barrier();                         // the stages are dead
        fetch(0, stage);
      }
    }
    if (ends)
#pragma unroll
      for (int t = 0; t < DK / 16; ++t) {
        const long at = state_at<DK, TV>(p, was, wave, t);
#pragma unroll
        for (int r = 0; r < 4; ++r) p.s_out[at + (long)r * p.dv] = st.s[t][r];
      }
    if (!more) break;
    state_in();
    ends = t1 == u.len;
    powers(u.g, C, w);
    decay = power(u.g, C);
  }
}

// One token: the state is read and written once, which bounds it (64 sequences of 32 heads of 128 x 128: 55 us, 52 at the rate of a copy).  A workgroup has 64 columns of one head: 16 threads of four columns, 16 rows at a time.
template <int DK>
__global__ __launch_bounds__(256) void la_step(const LaParams p) {
  __shared__ float red[4][C];
  Unit u;
  const int tiles = p.H * (p.dv / C);
  if (!unit_of(p, blockIdx.x / tiles, blockIdx.x % tiles, DK, C, u)) {
    if (p.fill && threadIdx.x < C) p.o[(long)u.b * p.bso + (long)u.h * p.dv + u.tile * C + threadIdx.x] = (bf16_t)0.f;
    return;
  }
  const int c4 = (threadIdx.x & 15) * 4, r0 = threadIdx.x >> 4;
  const float d = power(u.g, 1);
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

struct Plan { long heads; int tv, chunks; };      // heads: units of a sequence

// 128 columns of v to a workgroup (which computes the scores once for them) where dv has them.
// Chunks: a workgroup goes through its blocks one after the other (t_block us each, whatever else runs), so few heads are cut; but a
// chunk's state is written, read, written and read again, and the rounds that the workgroups make on 256 CUs, as many to one as its LDS holds, are whole ones.
// Measured, us for whole sequences | 8 | 12 | 16 | 25 | 32 chunks, dk x dv: 8 packed sequences of 0 .. 8192 tokens, 16384 in all, 16 heads of 128 x 128
// 530 | 220 | 157 | 134 | 170 | 157, 64 x 128 386 | 173 | 124 | 105 | 129 | 115, 128 x 64 412 | 182 | 130 | 110 | 129 | 115, 64 x 64 300 | 138 | 100 | 85 | 80 | 74;
// 16 of 1024 128 x 128 87 | 171 | 153 | 99 | 166 | 142; 2 x 4096 of 20 heads 64 x 128 193 | 90 | 70 | 92 | 79 | 91, 64 x 64 152 | 72 | 57 | 58 | 50 | 57;
// one of 1024 of 16 heads 64 x 64 39 | 21.5 | 22.5 | 22.5.  Over 36 such cases what is chosen here takes 0.3 % more than the best of 21 counts, 5 % at most.
Plan plan_of(long B, long H, long dk, long dv, long T, long rows) {
  Plan r;
  r.tv = dv % 128 == 0 ? 128 : 64;
  r.heads = H * (dv / r.tv);
  r.chunks = 0;
  const long blocks = (T + C - 1) / C, dense = B * blocks, packed = rows / C + B, all = dense < packed ? dense : packed;
  const bool wide = r.tv == 128;
  const double t_block = dk == 128 ? (wide ? 4.15 : 3.2) : wide ? 3.0 : 2.33;
  const int lds = dk == 128 ? (wide ? OutShape<128, 128>::LDS : OutShape<128, 64>::LDS) : wide ? OutShape<64, 128>::LDS : OutShape<64, 64>::LDS;
  const long slots = 256 * (160 * 1024 / lds);        // workgroups of la_out that run at once
  auto rounds = [](long wgs, long n) { return (double)((wgs + n - 1) / n); };
  double best = rounds(B * r.heads, slots) * blocks * t_block * 1.03;    // whole sequences
  if (r.heads > 65535) return r;                      // (la_scan's grid)
  static const int counts[] = {2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 13, 14, 15, 16, 18, 20, 22, 25, 28, 32, 36, 42, 51, 64, 85, 102, 128, 170, 256};
  for (const long n : counts) {
    const long size = (all + n - 1) / n;
    if (n > all || n * r.heads * dk * r.tv * 8 > 4L << 30) break;
    const double t = 14. + size * t_block * (rounds(n * r.heads, slots) + 0.5 * rounds(n * r.heads, 512)) + 0.3 * n + n * r.heads * (double)(dk * r.tv * 16) / 4e6;
    if (t < best) { best = t; r.chunks = (int)n; }
  }
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

template <int DK, int TV>
int prompt(const LaParams& p, long heads, hipStream_t s) {
  constexpr int lds = OutShape<DK, TV>::LDS, gain_lds = 2 * (Tile<DK>::BYTES + Tile<TV>::BYTES);
  const long size = p.share * (p.dv / TV), clusters = heads / size * (p.chunks ? p.chunks : p.B);
  const dim3 grid((unsigned)((clusters + 7) / 8 * 8 * size)), block(TV * 4);
  if (p.chunks == 0) {
    if (lds > 65536) {
      const hipError_t e = kh_allow_lds<la_out<DK, TV, true>>(lds);
      if (e != hipSuccess) return (int)e;
    }
    kh_launch(KH_TAG_LINEAR_ATTENTION, la_out<DK, TV, true>, grid, block, lds, s, p);
  } else {
    if (lds > 65536) {
      const hipError_t e = kh_allow_lds<la_out<DK, TV, false>>(lds);
      if (e != hipSuccess) return (int)e;
    }
    kh_launch(KH_TAG_LINEAR_ATTENTION, la_gain<DK, TV>, grid, block, gain_lds, s, p);
    hipError_t e = hipGetLastError();                 // (the launch behind it reads what it writes)
    if (e != hipSuccess) return (int)e;
    kh_launch(KH_TAG_LINEAR_ATTENTION, la_scan<DK, TV>, dim3(DK / 16, (unsigned)heads), block, 0, s, p);
    e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
    kh_launch(KH_TAG_LINEAR_ATTENTION, la_out<DK, TV, false>, grid, block, lds, s, p);
  }
  KH_RETURN_LAST_ERROR();
}

}  // namespace

KH_EXPORT int64_t kh_linear_attention_workspace_bytes(int64_t B, int64_t H, int64_t T, int64_t rows, int64_t dk, int64_t dv) {
  if (B <= 0 || H <= 0 || T <= 0 || rows <= 0 || dv <= 0) return KH_ERR_INVALID_ARG;
  if ((dk != 64 && dk != 128) || dv % C != 0 || dv > 1024) return KH_ERR_UNSUPPORTED;
  if (B > (1 << 20) || H > (1 << 16) || B * H * (dv / C) > (1L << 30) || T > (1L << 30)) return KH_ERR_TOO_LARGE;
  const Plan r = plan_of(B, H, dk, dv, T, rows);
  return r.chunks ? (int64_t)r.heads * r.chunks * dk * r.tv * 8 + r.chunks * (int64_t)sizeof(Chunk) : 0;
}

KH_EXPORT int kh_linear_attention_bf16(const void* q, const void* k, const void* v, void* o, const float* log_decay, const float* state_in,
                                       float* state_out, const int32_t* slots, int64_t n_slots, const int32_t* seg_start, int64_t rows,
                                       void* workspace, int64_t B, int64_t H, int64_t kv_heads, int64_t T, int64_t dk, int64_t dv, int64_t ldq,
                                       int64_t ldk, int64_t ldv, int64_t ldo, int64_t bsq, int64_t bsk, int64_t bsv, int64_t bso, float scale,
                                       void* stream) {
  if (n_slots > (1L << 30) || rows > (1L << 31)) return KH_ERR_TOO_LARGE;
  LaParams p{(const bf16_t*)q, (const bf16_t*)k, (const bf16_t*)v, (bf16_t*)o, log_decay, state_in, state_out, seg_start, slots, (float*)workspace,
             ldq, ldk, ldv, ldo, bsq, bsk, bsv, bso, (long)rows, (int)B, (int)H, kv_heads > 0 ? (int)(H / kv_heads) : 1, (int)T, (int)dv, (int)n_slots,
             0, scale, 0};
  const int rc = check(p, B, H, kv_heads, dk, dv, false);
  if (rc != KH_OK) return rc;
  if (T <= 0 || (seg_start && rows < 0)) return KH_ERR_INVALID_ARG;
  if (ldq < H * dk || ldk < kv_heads * dk || ldv < kv_heads * dv || ldo < H * dv) return KH_ERR_INVALID_ARG;
  if (T > (1L << 30)) return KH_ERR_TOO_LARGE;
  if ((ldq | ldk | ldv | ldo) >= (1L << 24)) return KH_ERR_TOO_LARGE;
  const Plan r = plan_of(B, H, dk, dv, T, seg_start ? (rows > 0 ? rows : 1) : B * T);
  p.chunks = r.chunks;
  if (p.chunks && !workspace) return KH_ERR_INVALID_ARG;
  if (!kh_aligned16(workspace)) return KH_ERR_ALIGNMENT;
  if (r.heads * (r.chunks ? r.chunks : B) > 0x3fffffffL) return KH_ERR_TOO_LARGE;
  hipStream_t s = (hipStream_t)stream;
  if (r.tv == 64) return dk == 64 ? prompt<64, 64>(p, r.heads, s) : prompt<128, 64>(p, r.heads, s);
  return dk == 64 ? prompt<64, 128>(p, r.heads, s) : prompt<128, 128>(p, r.heads, s);
}

KH_EXPORT int kh_linear_attention_step_bf16(const void* q, const void* k, const void* v, void* o, const float* log_decay, const float* state_in,
                                            float* state_out, const int32_t* slots, int64_t n_slots, int64_t B, int64_t H, int64_t kv_heads,
                                            int64_t dk, int64_t dv, int64_t ldq, int64_t ldk, int64_t ldv, int64_t ldo, float scale, int flags, void* stream) {
  if (flags & ~1) return KH_ERR_INVALID_ARG;
  if (n_slots > (1L << 30)) return KH_ERR_TOO_LARGE;
  LaParams p{(const bf16_t*)q, (const bf16_t*)k, (const bf16_t*)v, (bf16_t*)o, log_decay, state_in, state_out, nullptr, slots, nullptr,
             0, 0, 0, 0, ldq, ldk, ldv, ldo, 0, (int)B, (int)H, kv_heads > 0 ? (int)(H / kv_heads) : 1, 1, (int)dv, (int)n_slots, 0, scale, flags};
  const int rc = check(p, B, H, kv_heads, dk, dv, true);
  if (rc != KH_OK) return rc;
  if (ldq < H * dk || ldk < kv_heads * dk || ldv < kv_heads * dv || ldo < H * dv) return KH_ERR_INVALID_ARG;
  const long units = B * H * (dv / C);
  if (dk == 64) kh_launch(KH_TAG_LINEAR_ATTENTION, la_step<64>, dim3((unsigned)units), dim3(256), 0, (hipStream_t)stream, p);
  else kh_launch(KH_TAG_LINEAR_ATTENTION, la_step<128>, dim3((unsigned)units), dim3(256), 0, (hipStream_t)stream, p);
  KH_RETURN_LAST_ERROR();
}
