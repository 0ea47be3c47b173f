// New entries into a cache in pages, and the eviction of the entries of the least weight (include/fhog_hip.h).
//
// Both move rows: nothing is computed on them, and what bounds them is memory, every row in and out once, 16 bytes to a lane.
#include <algorithm>

#include "fhog_paged.h"

namespace fhog {
namespace {

using namespace paged;
constexpr int kThreads = 256;
// Rows go past the caches where they are written (a pool is larger than they are), and where they are read from it. us: 8 prompts of 4096 tokens, 8 heads, bf16, d = 128
// (158 MB) 33.0 -> 28.6, with the new rows read past them too 30.4; 32 x 8 x 4096 rows moved (1.07 GB) 219 -> 203, with two rows to a thread on the way, four 212.
__device__ __forceinline__ u32x4_t fetch_once(const char* p) { return __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(p)); }
__device__ __forceinline__ void put(char* p, u32x4_t x) { __builtin_nontemporal_store(x, reinterpret_cast<u32x4_t*>(p)); }

struct Append {
  Cache c;
  const char* k;
  const char* v;
  const int32_t* counts;
  int64_t kb, kh, kn, vb, vh, vn;   // strides in bytes
  Divisor chunks, tokens, heads;    // of a row; n; heads of keys
  uint32_t total;
};

// A thread has one chunk of a key and of its value: (sequence, head, token, chunk), the last one fastest
__global__ void __launch_bounds__(kThreads) append_entries(Append a) {
  const uint32_t id = blockIdx.x * kThreads + threadIdx.x;
  if (id >= a.total) return;
  uint32_t rest = a.chunks(id);
  const uint32_t chunk = id - rest * a.chunks.by;
  uint32_t row = a.tokens(rest);
  const int t = (int)(rest - row * a.tokens.by);
  const uint32_t b = a.heads(row), h = row - b * a.heads.by;
  const int n = max(0, a.c.lengths[b]), count = min(a.counts ? max(0, a.counts[b]) : (int)a.tokens.by, min((int)a.tokens.by, n));
  if (t >= count) return;
  const uint32_t j = n - count + t;
  if (j >= (uint32_t)a.c.capacity) return;   // a length beyond the table: what has no place is dropped, and the entries that the table has room for stay
  const u32x4_t k = *reinterpret_cast<const u32x4_t*>(a.k + b * a.kb + h * a.kh + t * a.kn + chunk * 16);
  const u32x4_t v = *reinterpret_cast<const u32x4_t*>(a.v + b * a.vb + h * a.vh + t * a.vn + chunk * 16);
  const uint32_t at = a.c.page(j);
  const int32_t page = a.c.table[b * a.c.stride_tb + at];
  if ((uint32_t)page >= (uint32_t)a.c.pages) return;
  const int64_t to = page * a.c.stride_p + h * a.c.stride_h + (j - at * a.c.page.by) * a.c.stride_n + chunk * 16;
  put(a.c.keys + to, k);
  put(a.c.values + to, v);
}

// ---- eviction ---------------------------------------------------------------------------------------------------------
struct Evict {
  Cache c;
  const float* weights;
  const int32_t* into;
  int32_t* lengths_out;
  int32_t* kept;
  float* weights_out;
  int64_t wb, wh, ib;
  int64_t budget;
  int32_t rows;             // rows that may stay: min(budget, capacity)
  int32_t sinks, recent;
  Divisor chunks;           // of a row
};

constexpr int kSelect = 1024, kWaves = kSelect / 64, kHeld = 12288;   // kHeld: entries whose ranks are held in LDS
constexpr int kCopies = 8, kDigits = 264;   // of the histogram; copies lie eight banks apart
constexpr int kRowsEach = 2;   // chunks of keys and values that a thread moves

// A number for each entry that grows with the order in which entries stay: what is protected first, then by weight, NaN last; 0 is for those that are not there
__device__ __forceinline__ uint32_t rank_of(float w, int j, int n, const Evict& e) {
  if (j < e.sinks || j >= n - e.recent) return 0xffffffffu;
  if (w != w) return 1;
  const uint32_t u = __builtin_bit_cast(uint32_t, w + 0.f);   // -0 becomes 0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Whether a number in a table names a page
__device__ __forceinline__ bool names(int32_t page, const Cache& c) { return (uint32_t)page < (uint32_t)c.pages; }
__device__ __forceinline__ int pages_of(int n, const Cache& c) { return n > 0 ? (int)c.page(n - 1) + 1 : 0; }

// Rows that stay, to their new places: the chunks of 16 bytes `id` and, kRowsEach - 1 times more, `step` further on, of the keys and values of m rows
__device__ __forceinline__ void move_chunks(const Evict& e, int b, int h, const int32_t* kept, int m, uint32_t id, uint32_t step) {
  u32x4_t k[kRowsEach], v[kRowsEach];
  int64_t dst[kRowsEach];
#pragma unroll
  for (int u = 0; u < kRowsEach; u++, id += step) {
    dst[u] = -1;
    const uint32_t i = e.chunks(id), chunk = id - i * e.chunks.by;
    if (i >= (uint32_t)m) continue;
    const uint32_t j = kept[i];
    if (j >= (uint32_t)e.c.capacity) continue;   // -1, or lengths that someone has changed meanwhile
    const uint32_t at = e.c.page(j), to = e.c.page(i);
    const int32_t from_page = e.c.table[b * e.c.stride_tb + at], to_page = e.into[b * e.ib + to];
    if (!names(from_page, e.c) || !names(to_page, e.c)) continue;
    const int64_t inside = h * e.c.stride_h + chunk * 16;
    const int64_t src = from_page * e.c.stride_p + (j - at * e.c.page.by) * e.c.stride_n + inside;
    dst[u] = to_page * e.c.stride_p + (i - to * e.c.page.by) * e.c.stride_n + inside;
    k[u] = fetch_once(e.c.keys + src), v[u] = fetch_once(e.c.values + src);
  }
#pragma unroll
  for (int u = 0; u < kRowsEach; u++)
    if (dst[u] >= 0) put(e.c.keys + dst[u], k[u]), put(e.c.values + dst[u], v[u]);
}

// Which entries of one sequence and head of keys stay. Each wave has a stretch of the entries. The rank of the last one that stays is found digit by digit, eight bits at a
// time from the top: a histogram of the digit over the entries whose higher digits are those found so far, and the digit at which the sum from above reaches
// what is still to be found. Then the entries that stay are counted, wave by wave, and written to the places that the counts give.
// What bounds it: the waits between its passes. us, 32 x 8 slices of 8192 | 4 x 4 of 1000: weights read anew in every pass 26.6 | 7.4, ranks formed once and kept in registers
// 20.2 | 10.8, in LDS 22.7 | 7.6, and there with a histogram of eight copies 19.8 | 7.7. The wave that sums a histogram clears it for the next pass, and digits that stay all together end the
// search: the whole call 230.6 -> 228.8 | 11.4 -> 10.0.
// Entries whose page is none are not there: they do not stay. Places whose page in `into` is none are passed over: there `kept` names entries that are not there, as far as there are any, so that
// an entry of nothing never comes to lie in a page that is read. The tables are looked at page by page beside the first pass, and entry by entry only where a page is missing: 0.3 us
// of 10 (4 x 4 of 1000), none of 228.
// MOVE: and are moved by the same workgroup.
template <bool MOVE>
__global__ void __launch_bounds__(kSelect) select_entries(Evict e) {
  extern __shared__ uint32_t held[];
  __shared__ __attribute__((aligned(16))) uint32_t histogram[kCopies][kDigits];   // a lane counts in copy lane % kCopies: the same digit of many lanes is not one address
  __shared__ uint32_t found[3];               // digits so far; how many of the entries of these digits stay, and whether all do
  __shared__ int counts[3][kWaves];           // entries of a wave's stretch above the rank, of the rank itself, and those that are not there
  const int b = blockIdx.x / e.c.heads_k, h = blockIdx.x - b * e.c.heads_k, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  __shared__ int with[3 * kWaves];            // by wave: whether pages lack; entries that are there, and places
  // The first wave says how many entries there are, behind the barrier that there is in any case: lengths that someone changes meanwhile make wrong results, but no waves that disagree at a barrier
  __shared__ int entries;
  const float* const w = e.weights + b * e.wb + h * e.wh;
  const int32_t* const table = e.c.table + b * e.c.stride_tb;
  const int32_t* const into = e.into + b * e.ib;
  int32_t* const kept = e.kept + (int64_t)blockIdx.x * e.budget;
  float* const out = e.weights_out + (int64_t)blockIdx.x * e.c.capacity;
  const int32_t first_into = tid < pages_of(e.rows, e.c) ? into[tid] : 0;   // pages of the tables are asked for ahead of the weights, and looked at behind them
  {
    const int n = e.c.length(b);
    if (tid == 0) entries = n;
    const int32_t first = tid < pages_of(n, e.c) ? table[tid] : 0;
    for (int j = tid; j < min(n, kHeld); j += kSelect) held[j] = rank_of(w[j], j, n, e);
    const auto lacks = [&](const int32_t* pages, int32_t first, int n) {   // a page of n entries, in this wave's share
      bool none = !names(first, e.c);
      for (int i = tid + kSelect; i < pages_of(n, e.c); i += kSelect) none = none || !names(pages[i], e.c);
      return __builtin_amdgcn_ballot_w64(none) != 0;
    };
    const int lack = (lacks(table, first, n) ? 1 : 0) | (lacks(into, first_into, e.rows) ? 2 : 0);
    if (lane == 0) with[wave] = lack;
  }
  for (int i = tid; i < kCopies * kDigits; i += kSelect) (&histogram[0][0])[i] = 0;
  __syncthreads();
  const int n = __builtin_amdgcn_readfirstlane(entries), lack = with[lane % kWaves];
  const bool gaps = __builtin_amdgcn_ballot_w64(lack & 1) != 0, closed = __builtin_amdgcn_ballot_w64(lack & 2) != 0;
  int here = n, open = e.rows;   // entries that are there, and places
  if (gaps || closed) {
    const auto share = [&](const int32_t* pages, int n) {
      int sum = 0;
      for (int i = tid; i < pages_of(n, e.c); i += kSelect)
        if (names(pages[i], e.c)) sum += min((int)e.c.page.by, n - i * (int)e.c.page.by);
      return scan(sum);
    };
    const int some_here = share(table, n), some_open = share(into, e.rows);
    if (lane == 63) with[kWaves + wave] = some_here, with[2 * kWaves + wave] = some_open;
    if (gaps)
      for (int j = tid; j < min(n, kHeld); j += kSelect)
        if (!names(table[e.c.page(j)], e.c)) held[j] = 0;
    __syncthreads();
    const int upto = scan(lane < 2 * kWaves ? with[kWaves + lane] : 0);
    here = __builtin_amdgcn_readlane(upto, kWaves - 1), open = __builtin_amdgcn_readlane(upto, 2 * kWaves - 1) - here;
  }
  const int m = min(here, open);
  const int stretch = ((n + kWaves - 1) / kWaves + 63) & ~63, begin = min(n, wave * stretch), end = min(n, begin + stretch);
  // f(j, rank) for the wave's entries in order, 64 at a time; all lanes take part
  const auto each = [&](auto f) {
    int j = begin + lane;
    for (; j - lane < min(end, kHeld); j += 64) f(j, j < end ? held[j] : 0);
    for (; j - lane < end; j += 64) f(j, j >= end || (gaps && !names(table[e.c.page(j)], e.c)) ? 0 : rank_of(w[j], j, n, e));
  };
  if (!closed) {
    if (h == 0 && tid == 0) e.lengths_out[b] = m;
    for (int64_t i = m + tid; i < e.budget; i += kSelect) kept[i] = -1;
    for (int i = m + tid; i < e.c.capacity; i += kSelect) out[i] = 0.f;
  }
  uint32_t rank = 0;
  int ties = 0;
  if (0 < m && m < here) {
    ties = n;
    uint32_t above = 0;
    int need = m;
    for (int shift = 24;; shift -= 8) {
      each([&](int j, uint32_t r) {
        const uint32_t digit = r >> shift & 255;
        const bool in = r != 0 && (shift == 24 || r >> (shift + 8) == above);
        if (in) atomicAdd(&histogram[lane % kCopies][digit], 1u);
      });
      __syncthreads();
      if (wave == 0) {
        // lane l has the digits 4 l .. 4 l + 3; sum of the digits from there up
        u32x4_t c = {0, 0, 0, 0};
#pragma unroll
        for (int x = 0; x < kCopies; x++) {
          u32x4_t& counted = *reinterpret_cast<u32x4_t*>(&histogram[x][4 * lane]);
          c += counted, counted = u32x4_t{0, 0, 0, 0};   // for the next pass
        }
        const uint32_t sum = c[0] + c[1] + c[2] + c[3], upto = scan((int)sum);
        uint32_t over = __builtin_amdgcn_readlane(upto, 63) - upto;   // entries of higher digits than this lane's
        const uint32_t up = over + sum;
        if (over < (uint32_t)need && up >= (uint32_t)need) {   // one lane alone
          int i = 3;
          while (over + c[i] < (uint32_t)need) over += c[i], i--;
          found[0] = above << 8 | (4 * lane + i), found[1] = need - over, found[2] = c[i] == need - over;
        }
      }
      __syncthreads();
      above = found[0], need = (int)found[1];
      if (found[2]) {   // all of these digits, and of higher ones
        rank = above << shift;
        break;
      }
      if (shift == 0) {
        rank = above, ties = need;
        break;
      }
    }
  }
  int over = 0, same = 0, gone = 0;
  each([&](int j, uint32_t r) {
    over += __builtin_popcountll(__builtin_amdgcn_ballot_w64(j < end && r > rank));
    same += __builtin_popcountll(__builtin_amdgcn_ballot_w64(j < end && r == rank));
    if (closed) gone += __builtin_popcountll(__builtin_amdgcn_ballot_w64(j < end && r == 0));
  });
  if (lane == 0) counts[0][wave] = over, counts[1][wave] = same, counts[2][wave] = gone;
  __syncthreads();
  over = same = gone = 0;
  for (int i = 0; i < wave; i++) over += counts[0][i], same += counts[1][i], gone += counts[2][i];
  const uint64_t below = ((uint64_t)1 << lane) - 1;
  const auto list = [&](int i, int j) { out[i] = __builtin_bit_cast(float, j); };   // closed: what stays in order, and behind it what is not there, until places are dealt out
  const auto listed = [&](int i) { return __builtin_bit_cast(int, out[i]); };
  each([&](int j, uint32_t r) {
    const uint64_t o = __builtin_amdgcn_ballot_w64(j < end && r > rank), s = __builtin_amdgcn_ballot_w64(j < end && r == rank);
    const int same_before = same + __builtin_popcountll(s & below), at = over + __builtin_popcountll(o & below) + min(same_before, ties);
    if (j < end && at < m && (r > rank || (r == rank && same_before < ties))) {   // at >= m: of lengths that someone has changed meanwhile
      if (closed) list(at, j);
      else kept[at] = j, out[at] = w[j];
    }
    over += __builtin_popcountll(o), same += __builtin_popcountll(s);
    if (closed) {
      const uint64_t g = __builtin_amdgcn_ballot_w64(j < end && r == 0);
      const int to = here + gone + __builtin_popcountll(g & below);
      if (j < end && r == 0 && to < n) list(to, j);
      gone += __builtin_popcountll(g);
    }
  });
  int length = m;
  if (closed) {
    const int part = ((e.rows + kWaves - 1) / kWaves + 63) & ~63, first = min(e.rows, wave * part), last = min(e.rows, first + part);
    const auto open_at = [&](int i) { return i < last && names(into[e.c.page(i)], e.c); };
    int before = 0;   // open places
    for (int i = first + lane; i - lane < last; i += 64) before += __builtin_popcountll(__builtin_amdgcn_ballot_w64(open_at(i)));
    __syncthreads();   // the list is there, and the counts have been read
    if (lane == 0) counts[0][wave] = before;
    if (tid == 0) entries = 0;
    __syncthreads();
    before = 0;
    for (int i = 0; i < wave; i++) before += counts[0][i];
    for (int i = first + lane; i - lane < last; i += 64) {
      const bool is = open_at(i);
      const uint64_t o = __builtin_amdgcn_ballot_w64(is);
      const int k = before + __builtin_popcountll(o & below);   // open places in front of it; i - k closed ones
      if (i < last) kept[i] = k >= m ? -1 : is ? listed(k) : i - k < n - here ? listed(here + i - k) : -1;
      if (is && k == m - 1) entries = i + 1;
      before += __builtin_popcountll(o);
    }
    for (int64_t i = e.rows + tid; i < e.budget; i += kSelect) kept[i] = -1;
    __syncthreads();   // the list has been read
    length = entries;
    if (h == 0 && tid == 0) e.lengths_out[b] = length;
    for (int i = tid; i < e.c.capacity; i += kSelect) {
      const int j = i < length && names(into[e.c.page(i)], e.c) ? kept[i] : -1;
      out[i] = (uint32_t)j < (uint32_t)n ? w[j] : 0.f;
    }
  }
  if constexpr (MOVE) {
    __syncthreads();   // all of `kept` is there
    for (uint32_t id = tid; id < (uint32_t)length * e.chunks.by; id += kRowsEach * kSelect) move_chunks(e, b, h, kept, length, id, kSelect);
  }
}

__global__ void __launch_bounds__(kThreads) move_entries(Evict e) {
  const int b = blockIdx.y / e.c.heads_k, h = blockIdx.y - b * e.c.heads_k;
  move_chunks(e, b, h, e.kept + (int64_t)blockIdx.y * e.budget, e.rows, blockIdx.x * kRowsEach * kThreads + threadIdx.x, kThreads);
}

uint32_t row_chunks(const fhog_paged_cache& c) { return (uint32_t)(c.d * (c.dtype == FHOG_DTYPE_FP32 ? 4 : 2) / 16); }

}  // namespace

hipError_t launch_paged_append(const fhog_paged_append_args* a, hipStream_t s) {
  Append p;
  const int es = a->cache.dtype == FHOG_DTYPE_FP32 ? 4 : 2;
  p.c = cache_of(a->cache), p.k = (const char*)a->k, p.v = (const char*)a->v, p.counts = a->counts;
  p.kb = a->stride_kb * es, p.kh = a->stride_kh * es, p.kn = a->stride_kn * es, p.vb = a->stride_vb * es, p.vh = a->stride_vh * es, p.vn = a->stride_vn * es;
  p.chunks = Divisor(row_chunks(a->cache)), p.tokens = Divisor((uint32_t)a->n), p.heads = Divisor((uint32_t)a->cache.heads_k);
  p.total = (uint32_t)(a->cache.batch * a->cache.heads_k * a->n * p.chunks.by);
  hipLaunchKernelGGL(append_entries, dim3((p.total + kThreads - 1) / kThreads), dim3(kThreads), 0, s, p);
  return hipGetLastError();
}

hipError_t launch_paged_evict(const fhog_paged_evict_args* a, hipStream_t s) {
  Evict e;
  e.c = cache_of(a->cache), e.weights = a->weights, e.into = a->into, e.lengths_out = a->lengths_out, e.kept = a->kept, e.weights_out = a->weights_out;
  e.wb = a->stride_wb, e.wh = a->stride_wh, e.ib = a->stride_ib, e.budget = a->budget;
  e.rows = (int32_t)(a->budget < e.c.capacity ? a->budget : e.c.capacity);
  // beyond the capacity all entries are protected either way
  e.sinks = (int32_t)(a->sinks < e.c.capacity ? a->sinks : e.c.capacity), e.recent = (int32_t)(a->recent < e.c.capacity ? a->recent : e.c.capacity);
  e.chunks = Divisor(row_chunks(a->cache));
  const unsigned slices = (unsigned)(a->cache.batch * a->cache.heads_k);
  const size_t lds = std::min(e.c.capacity, kHeld) * sizeof(uint32_t);
  // In one launch up to 96 KiB of rows to a slice, where that is nowhere slower. us, one launch | two, d = 64, slices of 64 | 98 | 128 | 179 KB: 16 slices 10.0 | 12.9, 11.0 | 12.9, 12.2 | 13.0, 15.0 | 13.0;
  // 64 10.2 | 12.8, 12.8 | 12.8, 15.4 | 13.5, 19.4 | 15.0; 128 11.4 | 13.2, 14.3 | 14.4, 17.7 | 16.1, 22.0 | 19.4; 256 13.2 | 15.8, 17.1 | 19.2, 21.4 | 23.0, 27.0 | 28.7
  if ((int64_t)e.rows * e.chunks.by * 32 <= 96 << 10) {
    hipLaunchKernelGGL(select_entries<true>, dim3(slices), dim3(kSelect), lds, s, e);
    return hipGetLastError();
  }
  hipLaunchKernelGGL(select_entries<false>, dim3(slices), dim3(kSelect), lds, s, e);
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess) return err;
  hipLaunchKernelGGL(move_entries, dim3((unsigned)(((int64_t)e.rows * e.chunks.by + kThreads * kRowsEach - 1) / (kThreads * kRowsEach)), slices), dim3(kThreads), 0, s, e);
  return hipGetLastError();
}

}  // namespace fhog
