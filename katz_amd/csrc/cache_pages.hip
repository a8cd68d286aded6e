// K16: the pages of a cache: more tokens for its sequences, sequences taken over or given up, the pages in use moved together.
//
// A page is free where nobody holds it (refs 0), and whoever wants one gets the lowest: what a call does depends on the tables alone, and a pool
// fills from below.  References are counted with integer atomics (their order does not matter); pages are dealt out by one workgroup that goes over
// refs once, in order, as far as it has to.  Only the copies need the whole chip: they take their list from memory, since how many there are is not
// known to the host.
//
// Bound by the launches and the memory's latency for a few sequences, by the copies' bytes for many layers.  us, the middle of 12: three beams forked from 77 tokens, 2 layers, 6.8 + 3.4, then
// their next tokens 2.8; 48 of 8 sequences, 24 layers, 5.1 + 4.7 + 21.3 (171 MB in and out), 5.1; 490 of 2048 pages moved in 4 layers 6.4 + 102 (515 MB, 5.1 TB/s).
#include "paged_cache.h"
#include <climits>

namespace {

constexpr int NT = 1024;       // the workgroup that deals pages out
constexpr int NC = 256;        // one that copies

struct Copy { int src, dst, tokens; };

// What a call keeps in its workspace.
struct Work {
  int32_t *row;                // [slots, width] of the sequences taken over
  int32_t *length, *state;     // [slots]: new length; 0 stays, 1 takes over, 2 emptied
  int32_t *start;              // [slots]: pages wanted before
  Copy *want;                  // [slots]: the page that a slot needs a copy of (src -1: none)
  int32_t *free, *moving, *to; // [pages]
  Copy *copies;                // [max(slots, pages)]
  int32_t *count;              // of copies
};

__host__ __device__ inline long up(long n) { return (n + 3) / 4 * 4; }

inline long work_ints(long slots, long width, long pages) {
  const long most = slots > pages ? slots : pages;
  return up(slots * width) + 3 * up(slots) + up(3 * slots) + 3 * up(pages) + up(3 * most) + 4;
}
inline Work work_of(void* at, long slots, long width, long pages) {
  Work w;
  int32_t* p = (int32_t*)at;
  auto take = [&](long n) { int32_t* r = p; p += up(n); return r; };
  w.row = take(slots * width);
  w.length = take(slots);
  w.state = take(slots);
  w.start = take(slots);
  w.want = (Copy*)take(3 * slots);
  w.free = take(pages);
  w.moving = take(pages);
  w.to = take(pages);
  w.copies = (Copy*)take(3 * (slots > pages ? slots : pages));
  w.count = take(1);
  return w;
}

struct PagesParams {
  int32_t *table, *lengths, *refs;
  const int32_t* asked;        // counts or parents
  int32_t* told;               // missing or in use
  Work w;
  int slots, width, pages, page;
};

// Exclusive prefix of v over the workgroup's threads, and the sum of all.
__device__ __forceinline__ int prefix(int v, int* total, int* red) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  __syncthreads();                                      // (red may still be read from the last time)
  if (lane == 63) red[wave] = x;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) {
    if (i < wave) before += red[i];
    all += red[i];
  }
  *total = all;
  return before + x - v;
}

constexpr int EACH = 16;                                // pages a thread looks at in one go

// The counts of EACH pages from `at` on (1 behind the last).
__device__ __forceinline__ void counts_of(const int32_t* refs, int pages, int at, int (&n)[EACH]) {
  if (at + EACH <= pages && ((uintptr_t)refs & 15) == 0) {
    int4 v[EACH / 4];
#pragma unroll
    for (int i = 0; i < EACH / 4; ++i) v[i] = reinterpret_cast<const int4*>(refs + at)[i];
    __builtin_memcpy(n, v, sizeof(n));
  } else {
#pragma unroll
    for (int i = 0; i < EACH; ++i) n[i] = at + i < pages ? refs[at + i] : 1;
  }
}

// Calls take(rank, page) for the lowest `wanted` pages without references, in order, and returns how many there were.
template <typename F>
__device__ int deal(const int32_t* refs, int pages, int wanted, int* red, F take) {
  int got = 0;
  for (int base = 0; base < pages && got < wanted; base += NT * EACH) {
    const int at = base + (int)threadIdx.x * EACH;
    int n[EACH];
    counts_of(refs, pages, at, n);
    uint32_t free = 0;
#pragma unroll
    for (int i = 0; i < EACH; ++i)
      if (n[i] == 0) free |= 1u << i;
    int total;
    int rank = got + prefix(__popc(free), &total, red);
    while (free && rank < wanted) {
      take(rank++, at + __ffs(free) - 1);
      free &= free - 1;
    }
    got += total;
  }
  return got < wanted ? got : wanted;
}

__device__ __forceinline__ int clamped(int n, const PagesParams& p) {
  const int most = p.width * p.page;
  return n < 0 ? 0 : n < most ? n : most;
}

// Sequence s grows by counts[s]: the pages behind its last one, dealt out by slot and then by place.
__global__ __launch_bounds__(NT) void extend(const PagesParams p) {
  __shared__ int red[NT / 64];
  __shared__ unsigned long long all_over;               // pages that no row has room for: slots can want 2^31 each
  if (threadIdx.x == 0) all_over = 0;
  const int most = p.width * p.page;
  // a slot's tokens, its first new page and how many
  auto look = [&](int s, int* longer, int* first, int* need, int* too_long) {
    const int n = clamped(p.lengths[s], p), more = p.asked[s] > 0 ? p.asked[s] : 0, fits = more < most - n ? more : most - n;
    const long whole = ((long)n + more + p.page - 1) / p.page;
    *longer = more > 0 ? n + fits : -1;
    *first = (n + p.page - 1) / p.page;
    *need = (n + fits + p.page - 1) / p.page - *first;
    *too_long = whole > p.width ? (int)(whole - p.width) : 0;
  };
  int wanted = 0, longer = -1, first = 0, need = 0, start = 0;
  unsigned long long over = 0;
  for (int base = 0; base < p.slots; base += NT) {
    const int s = base + (int)threadIdx.x;
    int total, too_long = 0;
    longer = -1, need = 0;
    if (s < p.slots) look(s, &longer, &first, &need, &too_long);
    over += (unsigned)too_long;
    start = wanted + prefix(need, &total, red);
    if (s < p.slots && p.slots > NT) p.w.start[s] = start;
    wanted += total;
  }
  const int got = deal(p.refs, p.pages, wanted, red, [&](int rank, int page) {
    p.w.free[rank] = page;
    p.refs[page] = 1;
  });
  if (over) atomicAdd(&all_over, over);
  __syncthreads();                                      // (and what was dealt out is there for all threads)
  if (threadIdx.x == 0) {
    const unsigned long long missing = (unsigned)(wanted - got) + all_over;
    *p.told = missing < INT_MAX ? (int)missing : INT_MAX;
  }
  // a thread enters the pages of a slot, a wave those of one that gets many
  constexpr int FEW = 4;
  for (int base = 0; base < p.slots; base += NT) {
    const int s = base + (int)threadIdx.x, lane = threadIdx.x & 63;
    if (p.slots > NT) {                                 // (else it is at hand)
      int too_long;
      longer = -1, need = 0;
      if (s < p.slots) {
        look(s, &longer, &first, &need, &too_long);
        start = p.w.start[s];
      }
    }
    if (longer >= 0) {
      p.lengths[s] = longer;
      if (need <= FEW)
        for (int i = 0; i < need; ++i) p.table[(long)s * p.width + first + i] = start + i < got ? p.w.free[start + i] : -1;
    }
    for (uint64_t many = __ballot(need > FEW); many; many &= many - 1) {
      const int who = __ffsll((unsigned long long)many) - 1, f = __shfl(first, who, 64), k = __shfl(need, who, 64), from = __shfl(start, who, 64);
      int32_t* row = p.table + (long)(base + (threadIdx.x & ~63) + who) * p.width + f;
      for (int i = lane; i < k; i += 64) row[i] = from + i < got ? p.w.free[from + i] : -1;
    }
  }
}

// What slot s gives up and takes over, counted by N threads (a wave or a workgroup); its new row of pages set aside, since others still read the old one.
template <int N>
__device__ __forceinline__ void count(const PagesParams& p, int s) {
  const int lane = threadIdx.x & (N - 1), parent = p.asked[s];
  const bool takes = parent >= 0 && parent < p.slots;
  if (parent == s) {
    if (lane == 0) p.w.state[s] = 0, p.w.want[s] = Copy{-1, -1, 0};
    return;
  }
  const int32_t* mine = p.table + (long)s * p.width;
  const int used = (clamped(p.lengths[s], p) + p.page - 1) / p.page;
  for (int i = lane; i < used; i += N) {
    const int e = mine[i];
    if (e >= 0 && e < p.pages) atomicSub(p.refs + e, 1);
  }
  int32_t* row = p.w.row + (long)s * p.width;
  const int n = takes ? clamped(p.lengths[parent], p) : 0, full = n / p.page, part = n % p.page;
  // the lowest taker of a sequence whose own slot gives it up has the page not yet full as it is
  int other = 0;
  if (part) {
    other = p.asked[parent] == parent;
    for (int i = lane; i < s; i += N) other |= i != parent && p.asked[i] == parent;
  }
  const bool heir = !(N == 64 ? __any(other) : __syncthreads_or(other));
  const int32_t* theirs = p.table + (long)(takes ? parent : 0) * p.width;
  for (int i = lane; i < p.width; i += N) {
    int e = -1;
    if (i < full || (i == full && part && heir)) {
      e = theirs[i];
      if (e >= 0 && e < p.pages) atomicAdd(p.refs + e, 1);
    }
    row[i] = e;
  }
  if (lane == 0) {
    p.w.state[s] = takes ? 1 : 2;
    p.w.length[s] = n;
    const int e = part && !heir ? theirs[full] : -1;
    p.w.want[s] = e >= 0 && e < p.pages ? Copy{e, full, part} : Copy{-1, -1, 0};
  }
}
__global__ __launch_bounds__(NC) void reorder_count(const PagesParams p) {
  count<NC>(p, blockIdx.x);
}

// Pages for the copies, by slot: none of them is one that is copied, since somebody holds those.  ALL: counts first (few slots: a launch less).
template <bool ALL>
__global__ __launch_bounds__(NT) void reorder_deal(const PagesParams p) {
  __shared__ int red[NT / 64];
  if constexpr (ALL) {
    for (int s = threadIdx.x >> 6; s < p.slots; s += NT / 64) count<64>(p, s);
    __syncthreads();
  }
  int wanted = 0;
  for (int base = 0; base < p.slots; base += NT) {
    const int s = base + (int)threadIdx.x;
    const int need = s < p.slots && p.w.want[s].src >= 0;
    int total;
    const int before = prefix(need, &total, red);
    if (s < p.slots) p.w.start[s] = wanted + before;
    wanted += total;
  }
  const int got = deal(p.refs, p.pages, wanted, red, [&](int rank, int page) {
    p.w.free[rank] = page;
    p.refs[page] = 1;
  });
  if (threadIdx.x == 0) *p.told = wanted - got, *p.w.count = got;
  __syncthreads();
  for (int s = threadIdx.x; s < p.slots; s += NT) {
    const Copy c = p.w.want[s];
    const int rank = p.w.start[s];
    if (c.src < 0 || rank >= got) continue;
    const int page = p.w.free[rank];
    p.w.row[(long)s * p.width + c.dst] = page;          // (dst: the place in the row)
    p.w.copies[rank] = Copy{c.src, page, c.tokens};
  }
}

// The pages in use, their number n, and for those from n on the free ones below, both in order.
__global__ __launch_bounds__(NT) void compact_plan(const PagesParams p) {
  __shared__ int red[NT / 64];
  int used = 0, live, count[EACH];
  for (int base = 0; base < p.pages; base += NT * EACH) {
    const int at = base + (int)threadIdx.x * EACH;
    counts_of(p.refs, p.pages, at, count);
#pragma unroll
    for (int i = 0; i < EACH; ++i) used += at + i < p.pages && count[i] > 0;
  }
  prefix(used, &live, red);
  int moves = 0, holes = 0;
  for (int base = 0; base < p.pages; base += NT * EACH) {
    const int at = base + (int)threadIdx.x * EACH;
    uint32_t hole = 0, moving = 0;
    if (p.pages > NT * EACH) counts_of(p.refs, p.pages, at, count);     // (else they are at hand)
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int e = at + i;
      const bool there = e < p.pages, used = there && count[i] > 0;
      if (e < live && !used) hole |= 1u << i;
      if (there && e >= live) {
        if (used) moving |= 1u << i;
        else p.w.to[e] = e;
      }
    }
    int total;
    int rank = holes + prefix(__popc(hole), &total, red);
    holes += total;
    for (; hole; hole &= hole - 1) p.w.free[rank++] = at + __ffs(hole) - 1;
    rank = moves + prefix(__popc(moving), &total, red);
    moves += total;
    for (; moving; moving &= moving - 1) p.w.moving[rank++] = at + __ffs(moving) - 1;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < moves; i += NT) {
    const int src = p.w.moving[i], dst = p.w.free[i];
    p.w.to[src] = dst;
    p.w.copies[i] = Copy{src, dst, p.page};
    p.refs[dst] = p.refs[src];
    p.refs[src] = 0;
  }
  if (threadIdx.x == 0) *p.told = live, *p.w.count = moves;
}

struct CopyParams {
  char *k, *v;
  long k_layer, k_page, k_token, k_head, v_layer, v_page, v_token, v_head;   // in bytes
  int layers, heads, row;      // row: bytes of a token of a head
  int cut;                     // tokens of a piece of work
  int pieces;                  // of a page
  int packed;                  // the heads of a token and the tokens of a page lie behind one another
};

// Past the caches go what is written and, where pages move, what is read, which nobody reads again (us of 515 MB in and out: 104 with neither, 103 with the
// stores, 96 with both and 8192 workgroups; of 171 MB copied from 8 pages a layer to 48: 24.7, 20.5, 35).
// The rows of the list's pages, piece by piece in units of T, and beside them (the first workgroups) what the tables become.
template <typename T, bool COMPACT>
__global__ __launch_bounds__(NC) void carry_out(const PagesParams p, const CopyParams c, const int tables) {
  if ((int)blockIdx.x < tables) {
    if constexpr (COMPACT) {
      const long all = (long)p.slots * p.width;
      const int live = *p.told;
      for (long i = (long)blockIdx.x * NC + threadIdx.x; i < all; i += (long)tables * NC) {
        const int e = p.table[i];
        if (e >= live && e < p.pages) p.table[i] = p.w.to[e];
      }
    } else {
      for (int s = blockIdx.x; s < p.slots; s += tables) {
        if (p.w.state[s] == 0) continue;
        for (int i = threadIdx.x; i < p.width; i += NC) p.table[(long)s * p.width + i] = p.w.row[(long)s * p.width + i];
        if (threadIdx.x == 0) p.lengths[s] = p.w.length[s];
      }
    }
    return;
  }
  const long each = (long)c.layers * 2 * c.pieces, all = *p.w.count * each;
  for (long i = blockIdx.x - tables; i < all; i += gridDim.x - tables) {
    const Copy what = p.w.copies[i / each];
    const int j = (int)(i % each), piece = j % c.pieces, layer = j / c.pieces >> 1;
    const int first = piece * c.cut, last = first + c.cut < what.tokens ? first + c.cut : what.tokens;
    if (first >= last) continue;
    const bool values = j / c.pieces & 1;
    const long token = values ? c.v_token : c.k_token, head = values ? c.v_head : c.k_head, page = values ? c.v_page : c.k_page;
    char* base = (values ? c.v : c.k) + layer * (values ? c.v_layer : c.k_layer) + first * token;
    const char* from = base + what.src * page;
    char* to = base + what.dst * page;
    const int per = c.row / (int)sizeof(T), units = (last - first) * c.heads * per;
    for (int u0 = threadIdx.x; u0 < units; u0 += 4 * NC) {              // four on their way at a time
      T x[4];
      long off[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int u = u0 + k * NC < units ? u0 + k * NC : u0;
        off[k] = (long)u * sizeof(T);
        if (!c.packed) {
          const int row = u / per;
          off[k] = row / c.heads * token + row % c.heads * head + (u - row * per) * (long)sizeof(T);
        }
        if constexpr (COMPACT) x[k] = __builtin_nontemporal_load(reinterpret_cast<const T*>(from + off[k]));
        else x[k] = *reinterpret_cast<const T*>(from + off[k]);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (u0 + k * NC < units) __builtin_nontemporal_store(x[k], reinterpret_cast<T*>(to + off[k]));
    }
  }
}

int check(const KhPagedCache* c, const void* asked, const void* told, const void* workspace) {
  const int rc = kh_cache_check(c);
  if (rc != KH_OK) return rc;
  if (!c->refs || !asked || !told || !workspace) return KH_ERR_INVALID_ARG;
  if (((uintptr_t)asked | (uintptr_t)told) & 3) return KH_ERR_ALIGNMENT;
  if (!kh_aligned16(workspace)) return KH_ERR_ALIGNMENT;
  return KH_OK;
}

PagesParams params(const KhPagedCache& c, const void* asked, void* told, void* workspace) {
  return PagesParams{c.table, c.lengths, c.refs, (const int32_t*)asked, (int32_t*)told, work_of(workspace, c.slots, c.width, c.pages),
                     (int)c.slots, (int)c.width, (int)c.pages, (int)c.page};
}

template <bool COMPACT>
void copy(const KhPagedCache& c, const PagesParams& p, hipStream_t s) {
  const long e = kh_cache_element(c);
  CopyParams o{(char*)c.k, (char*)c.v, c.k_layer * e, c.k_page * e, c.k_token * e, c.k_head * e, c.v_layer * e, c.v_page * e, c.v_token * e, c.v_head * e,
               (int)c.layers, (int)c.kv_heads, (int)(c.d * e), 0, 0, 0};
  o.packed = c.k_head == c.d && c.v_head == c.d && c.k_token == c.d * c.kv_heads && c.v_token == c.d * c.kv_heads;
  // a piece of work: about 16 KB of a page
  const long bytes = o.row * c.kv_heads;
  o.cut = (int)(16384 / bytes < 1 ? 1 : 16384 / bytes < c.page ? 16384 / bytes : c.page);
  o.pieces = (int)((c.page + o.cut - 1) / o.cut);
  const bool wide = o.row % 16 == 0 && ((o.k_layer | o.k_page | o.k_token | o.k_head | o.v_layer | o.v_page | o.v_token | o.v_head) % 16) == 0 && kh_aligned16(c.k) &&
                    kh_aligned16(c.v);
  const long most = COMPACT ? c.pages / 2 : c.slots, works = most * c.layers * 2 * o.pieces;
  const int tables = COMPACT ? (int)(c.slots * c.width / 4096 < 1 ? 1 : c.slots * c.width / 4096 < 64 ? c.slots * c.width / 4096 : 64) : (int)(c.slots < 256 ? c.slots : 256);
  const dim3 grid((unsigned)(tables + (works < 8192 ? works : 8192)));   // (2048 workgroups move 515 MB in 100 us, 4096 in 98, 8192 in 96)
  if (wide) kh_launch(KH_TAG_CACHE_PAGES, carry_out<u32x4, COMPACT>, grid, dim3(NC), 0, s, p, o, tables);
  else kh_launch(KH_TAG_CACHE_PAGES, carry_out<u32x2, COMPACT>, grid, dim3(NC), 0, s, p, o, tables);
}

}  // namespace

KH_EXPORT int64_t kh_cache_workspace_bytes(int64_t slots, int64_t width, int64_t pages) {
  if (slots <= 0 || width <= 0 || pages <= 0) return KH_ERR_INVALID_ARG;
  if (slots > (1L << 20) || pages > (1L << 30) || width > (1L << 30) || slots * width > (1L << 30)) return KH_ERR_TOO_LARGE;
  return 4 * work_ints(slots, width, pages);
}

KH_EXPORT int kh_cache_extend(const KhPagedCache* cache, const int32_t* counts, int32_t* missing, void* workspace, void* stream) {
  const int rc = check(cache, counts, missing, workspace);
  if (rc != KH_OK) return rc;
  kh_launch(KH_TAG_CACHE_PAGES, extend, dim3(1), dim3(NT), 0, (hipStream_t)stream, params(*cache, counts, missing, workspace));
  KH_RETURN_LAST_ERROR();
}

KH_EXPORT int kh_cache_reorder(const KhPagedCache* cache, const int32_t* parents, int32_t* missing, void* workspace, void* stream) {
  const int rc = check(cache, parents, missing, workspace);
  if (rc != KH_OK) return rc;
  if (cache->slots > (1L << 16)) return KH_ERR_TOO_LARGE;           // (every slot looks through those before it)
  const PagesParams p = params(*cache, parents, missing, workspace);
  hipStream_t s = (hipStream_t)stream;
  hipError_t e;
  // one workgroup counts for few slots with short rows, a wave a slot.  us with one launch and with two, the copies' 4 among them: 4 slots with rows of 8 pages 9.9 and 12.3, of
  // 128 10.9 and 13.2, of 1024 21.5 and 14.8; 8 of 32 10.5 and 14.1, of 512 16.3 and 13.7; 16 of 8 11.3 and 14.0, of 256 14.6 and 14.1; 32 of 8 14.0 and 14.4, of 128 17.0 and 14.1.
  if (cache->slots <= 16 && cache->width <= 128) {
    kh_launch(KH_TAG_CACHE_PAGES, reorder_deal<true>, dim3(1), dim3(NT), 0, s, p);
  } else {
    kh_launch(KH_TAG_CACHE_PAGES, reorder_count, dim3((unsigned)p.slots), dim3(NC), 0, s, p);
    e = hipGetLastError();                              // (the launches behind it go by what it writes)
    if (e != hipSuccess) return (int)e;
    kh_launch(KH_TAG_CACHE_PAGES, reorder_deal<false>, dim3(1), dim3(NT), 0, s, p);
  }
  e = hipGetLastError();
  if (e != hipSuccess) return (int)e;
  copy<false>(*cache, p, s);
  KH_RETURN_LAST_ERROR();
}

KH_EXPORT int kh_cache_compact(const KhPagedCache* cache, int32_t* in_use, void* workspace, void* stream) {
  const int rc = check(cache, in_use, in_use, workspace);
  if (rc != KH_OK) return rc;
  const PagesParams p = params(*cache, in_use, in_use, workspace);
  hipStream_t s = (hipStream_t)stream;
  kh_launch(KH_TAG_CACHE_PAGES, compact_plan, dim3(1), dim3(NT), 0, s, p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return (int)e;
  copy<true>(*cache, p, s);
  KH_RETURN_LAST_ERROR();
}
