// What the kernels on a cache in pages share: where an entry lies, and which tiles of its entries a token sees.
#pragma once
#include <type_traits>

#include "fhog_common.h"

namespace fhog {
namespace paged {

// j / page for 0 <= j < 2^31 without a division: with s = ceil(log2 page) and M = floor(2^(31 + s) / page) + 1 the error M page - 2^(31 + s) is at most page <= 2^s, and
// j times it below 2^(31 + s)
struct Divisor {
  uint32_t by = 1, mul = 0, shift = 0;
  Divisor() = default;
  explicit Divisor(uint32_t page) : by(page) {
    while (((uint64_t)1 << shift) < page) shift++;
    mul = (uint32_t)(((uint64_t)1 << (31 + shift)) / page + 1);
  }
  __host__ __device__ __forceinline__ uint32_t operator()(uint32_t j) const { return (uint32_t)(((uint64_t)(2 * j) * mul) >> 32) >> shift; }
};

struct Cache {
  char* keys;
  char* values;
  const int32_t* table;
  const int32_t* lengths;
  int64_t stride_p, stride_h, stride_n;   // in bytes
  int64_t stride_tb;
  Divisor page;
  int32_t pages, capacity, heads_k, batch;
  // entries of sequence b
  __device__ __forceinline__ int length(int b) const { return max(0, min(lengths[b], capacity)); }
};

inline Cache cache_of(const fhog_paged_cache& c) {
  const int es = c.dtype == FHOG_DTYPE_FP32 ? 4 : 2;
  Cache r;
  r.keys = (char*)c.keys, r.values = (char*)c.values, r.table = c.table, r.lengths = c.lengths;
  r.stride_p = c.stride_p * es, r.stride_h = c.stride_h * es, r.stride_n = c.stride_n * es, r.stride_tb = c.stride_tb;
  r.page = Divisor((uint32_t)c.page);
  r.pages = (int32_t)c.pages, r.capacity = (int32_t)(c.table_width * c.page), r.heads_k = (int32_t)c.heads_k, r.batch = (int32_t)c.batch;
  return r;
}

// Sum over the lanes up to this one, in registers
__device__ __forceinline__ int scan(int x) {
  const auto add = [&](auto control, auto mask) { x += __builtin_amdgcn_update_dpp(0, x, control.value, mask.value, 0xf, false); };
  const auto all = std::integral_constant<int, 0xf>{};
  add(std::integral_constant<int, 0x111>{}, all), add(std::integral_constant<int, 0x112>{}, all);   // the lanes 1, 2, 4 and 8 before it in its row of 16
  add(std::integral_constant<int, 0x114>{}, all), add(std::integral_constant<int, 0x118>{}, all);
  add(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{});                   // the last of the row before, into rows 1 and 3
  add(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{});                   // lane 31, into rows 2 and 3
  return x;
}

// The tiles of T entries of which a token sees some, in a row: those of the sinks that lie before its window, then the window's
template <int T>
struct Seen {
  int n, lo, sinks;     // entry j is seen iff j < n and (j >= lo or j < sinks)
  int first, skip, tiles;
  __device__ __forceinline__ Seen(int n_, int window, int sinks_) : n(n_) {
    lo = window > 0 ? max(0, n - window) : 0;
    sinks = min(sinks_, lo);
    const int all = (n + T - 1) / T;
    first = (sinks + T - 1) / T;
    skip = max(first, lo / T) - first;      // tiles between the two
    tiles = all - skip;
  }
  __device__ __forceinline__ int at(int i) const { return (i < first ? i : i + skip) * T; }
  // Where an entry that is seen comes among those of these tiles
  __device__ __forceinline__ int place(int j) const { return j < first * T ? j : j - skip * T; }
  // Tiles at most, whatever the length: the window's begin and end inside a tile
  __host__ __device__ static int64_t most(int64_t capacity, int64_t window, int64_t sinks) {
    const int64_t all = (capacity + T - 1) / T;
    if (window <= 0 || window >= capacity) return all;
    const int64_t sunk = sinks < capacity ? sinks : capacity, some = (sunk + T - 1) / T + (window + T - 2) / T + 1;
    return some < all ? some : all;
  }
  __device__ __forceinline__ bool sees(int j) const { return j < n && (j >= lo || j < sinks); }
  __device__ __forceinline__ bool whole(int j0) const { return j0 + T <= n && (j0 >= lo || j0 + T <= sinks); }
};

}  // namespace paged
}  // namespace fhog
