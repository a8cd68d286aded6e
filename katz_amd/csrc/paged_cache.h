// What the operators on a paged cache share: the checks of its description, and a division by the size of a page.
#pragma once
#include "kh_common.h"
#include "../../include/katz_hip.h"

constexpr int KH_E4M3 = 3;

static inline int kh_cache_element(const KhPagedCache& c) { return c.type == KH_E4M3 ? 1 : 2; }

static inline int kh_cache_check(const KhPagedCache* c) {
  if (!c || !c->k || !c->v || !c->table || !c->lengths) return KH_ERR_INVALID_ARG;
  if (c->layers <= 0 || c->pages <= 0 || c->page <= 0 || c->kv_heads <= 0 || c->d <= 0 || c->slots <= 0 || c->width <= 0) return KH_ERR_INVALID_ARG;
  if (c->type != 0 && c->type != 1 && c->type != KH_E4M3) return KH_ERR_INVALID_ARG;
  if (c->type != KH_E4M3 && (c->k_scale || c->v_scale)) return KH_ERR_INVALID_ARG;
  if (c->d % 8 != 0 || c->d > 256) return KH_ERR_UNSUPPORTED;
  const int64_t strides = c->k_layer | c->k_page | c->k_token | c->k_head | c->v_layer | c->v_page | c->v_token | c->v_head;
  if (strides < 0) return KH_ERR_INVALID_ARG;           // (one below zero: the kernels count bytes from the first element on)
  if (strides % 8 != 0) return KH_ERR_ALIGNMENT;
  const uintptr_t mask = c->type == KH_E4M3 ? 7 : 15;
  if (((uintptr_t)c->k | (uintptr_t)c->v) & mask) return KH_ERR_ALIGNMENT;
  if (((uintptr_t)c->table | (uintptr_t)c->lengths | (uintptr_t)c->refs | (uintptr_t)c->k_scale | (uintptr_t)c->v_scale) & 3) return KH_ERR_ALIGNMENT;
  if (c->pages > (1L << 30) || c->slots > (1L << 20) || c->layers > (1L << 16) || c->kv_heads > (1L << 16) || c->page > (1L << 20) ||
      c->width > (1L << 30) / c->page || c->slots * c->width > (1L << 30) || c->k_page >= (1L << 31) || c->k_token >= (1L << 31) || c->v_page >= (1L << 31) || c->v_token >= (1L << 31))
    return KH_ERR_TOO_LARGE;
  return KH_OK;
}

// t / n for 0 <= t < 2^31 by a multiplication (n is the size of a page: any number), the method of Granlund and Montgomery, "Division by Invariant Integers using
// Multiplication" (1994)
struct KhDivide {
  uint32_t n, mul, s1, s2;
  __host__ explicit KhDivide(uint32_t by) : n(by) {
    int l = 0;
    while ((1ull << l) < by) ++l;
    mul = (uint32_t)(((1ull << 32) * ((1ull << l) - by)) / by + 1);
    s1 = l > 0 ? 1 : 0;
    s2 = l > 0 ? l - 1 : 0;
  }
  __device__ __forceinline__ uint32_t operator()(uint32_t t) const {
    const uint32_t a = __umulhi(mul, t);
    return (a + ((t - a) >> s1)) >> s2;
  }
};
