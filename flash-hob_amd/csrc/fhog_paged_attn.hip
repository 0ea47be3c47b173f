// Attention of one new token of each sequence over a cache in pages.
//
//   s_hj = scale q_h . k_gj, L_h = ln sum_j exp s_hj, O_h = sum_j exp(s_hj - L_h) v_gj;   W'_gj = W_gj + sum_(h of g) exp(s_hj - L_h)
//
// over the entries j that the token sees; g: the head of keys that head h of queries belongs to.
//
// What bounds it: memory, every key and value once (4 flop to a byte with one head of queries to one of keys, 64 with 16). So no key and no value goes through LDS: a wave takes
// tiles of its own, straight into the registers that the matrix instructions read. The waves meet twice: behind the first one's finding out what there is to do (the lengths of all sequences, where
// tiles are dealt out: 12.1 -> 13.0 us for one sequence of 4096), and at the end.
//
// A tile is 32 entries (16 of fp32). The heads of queries of a head of keys are the columns, up to 16 of them; more take workgroups of their own. S^T = K Q^T
// with 16x16 products: lane l has row l % 16 of K, 16 bytes at a time, and gets column l % 16 of S^T, entries 4 (l / 16) + 0..3 of each 16. These are, with
// the entries counted in that order, the B operand of O^T = V^T P^T as they lie. Its A operand wants a channel to a lane and entries along it. A lane
// therefore loads the entries of its own group (l / 16), channels c (l % 16) .. + c - 1 with c = d / 16, which fills a row of a page with 16 lanes, and turns the
// 8 x c block that it has in its own registers: product i of c takes channel c m + i as its row m, so the results of a lane are c consecutive channels.
#include <algorithm>
#include <type_traits>

#include "fhog_paged.h"

namespace fhog {
namespace {

using namespace paged;
constexpr int kThreads = 256, kWaves = 4, kColumns = 16;
constexpr float kLn2 = 0.6931471805599453f;

struct Token {
  Cache c;
  const char* q;
  char* o;
  float* lse;
  const float* weights_in;
  float* weights_out;
  int64_t qb, qh, ob, oh;          // in bytes
  int64_t wib, wih, wob, woh;
  int32_t heads_q, group, columns; // group: heads of queries of a head of keys; columns: workgroups that they take
  int32_t window, sinks;
  int32_t units, slots;            // workgroups to a head of keys and 16 of its heads of queries: about, and at most
  int32_t dealt;                   // the tiles of all sequences are dealt out over them (Deal); else a workgroup has a sequence
  float scale_log2;
  float* part;                     // [slot][16][d]
  f32x2_t* stats;                  // [slot][16]: maximum in log2 units, sum
  f32x2_t* whole;                  // [batch * heads_q]: the same of rows that one workgroup had for itself
  float* scores;                   // [batch * heads_q][row]: scores in log2 units, of the tiles of which some entry is seen, in their order
  int64_t row;
};

template <int DT>
struct Type;   // by FHOG_DTYPE_*
template <>
struct Type<FHOG_DTYPE_BF16> {
  typedef __bf16 T;
};
template <>
struct Type<FHOG_DTYPE_FP16> {
  typedef _Float16 T;
};
template <>
struct Type<FHOG_DTYPE_FP32> {
  typedef float T;
};

template <int BYTES>
struct Words {
  typedef uint32_t type __attribute__((ext_vector_type(BYTES / 4)));
};
template <>
struct Words<4> {
  typedef uint32_t type;
};
template <int W>
__device__ __forceinline__ uint32_t word(const typename Words<4 * W>::type& v, int i) {
  if constexpr (W == 1) return v;
  else return v[i];
}

// ONCE: past the caches. TB/s of a loop of 16-byte loads over 2 GiB 6.2 -> 7.1; us, d = 128, bf16, 8 heads of keys 32 x 16384 326 -> 302, 64 x 2048 93 -> 84. For rows of 256 bytes
// and more (rows of 128 are read half a line at a time: d = 64, 24 x 700 15 -> 17) that one workgroup alone reads (64 heads of queries to 2 of keys, 32 x 16384: 113, else 150).
template <bool ONCE, typename V>
__device__ __forceinline__ V fetch(const char* p) {
  if constexpr (ONCE) return __builtin_nontemporal_load(reinterpret_cast<const V*>(p));
  else return *reinterpret_cast<const V*>(p);
}

typedef __attribute__((__vector_size__(8 * sizeof(_Float16)))) _Float16 f16x8_t;
template <int DT>
__device__ __forceinline__ f32x4_t mfma16(u32x4_t a, u32x4_t b, f32x4_t c) {
  if constexpr (DT == FHOG_DTYPE_FP16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
// The bits of a vector's element as a number; handed over by value: of an element itself __builtin_bit_cast takes the vector's first
__device__ __forceinline__ float number(uint32_t bits) { return __builtin_bit_cast(float, bits); }
template <int DT>
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
  typedef typename Type<DT>::T T;
  typedef T pair __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, pair{(T)lo, (T)hi});
}
// Two weights, not negative, cut to the type, and what that leaves of them. The rest of a weight that is not 0 is not 0 either, or infinite values would turn into NaN
template <int DT>
__device__ __forceinline__ u32x2_t cut(float lo, float hi) {
  if constexpr (DT == FHOG_DTYPE_FP16) {
    const auto first = __builtin_amdgcn_cvt_pkrtz(lo, hi);
    const auto rest = __builtin_amdgcn_cvt_pkrtz(__builtin_fmaf((float)first[0], -1.f, lo), __builtin_fmaf((float)first[1], -1.f, hi));
    const uint32_t bits = __builtin_bit_cast(uint32_t, first), not0 = (bits + 0x7fff7fffu) >> 15 & 0x00010001u;
    return u32x2_t{bits, __builtin_bit_cast(uint32_t, rest) | not0};
  } else {
    const uint32_t a = __builtin_bit_cast(uint32_t, lo), b = __builtin_bit_cast(uint32_t, hi);
    const auto left = [](float x, uint32_t bits) { return __builtin_fmaf(x, 1.f + 0x1p-22f, -number(bits & 0xffff0000u)); };
    return u32x2_t{__builtin_amdgcn_perm(b, a, 0x07060302), pack<DT>(left(lo, a), left(hi, b))};
  }
}

// What weights of fp16 are multiplied by on their way into the product: with references within 2^4 of the maximum they reach 2^15 there, and the steps of 2^-24 that fp16 has at its lower end
// are 2^-35 of the largest weight, not 2^-24. Without it many weak entries vanished beside a strong one: of 8192 that each weigh e^-17.4 of it a fourth of their sum.
template <int DT>
constexpr float kLift = DT == FHOG_DTYPE_FP16 ? 2048.f : 1.f;

// Entries of a tile
template <int DT>
constexpr int kTile = DT == FHOG_DTYPE_FP32 ? 16 : 32;
int tile_of(int dtype) { return dtype == FHOG_DTYPE_FP32 ? kTile<FHOG_DTYPE_FP32> : kTile<FHOG_DTYPE_BF16>; }

// How the tiles of all sequences are dealt out over about t.units workgroups (dealt): a sequence goes to as many as its share of all tiles comes to, rounded, and one at least. So a long
// sequence among short ones has many, whatever the table has room for. By a wave, lane b of each 64 sequences. Else every sequence has one workgroup.
template <int TILE>
struct Deal {
  const Token& t;
  int lane, share = 1;   // tiles of a workgroup, about
  int n0;                // tiles of this lane's sequence of the first 64
  __device__ __forceinline__ int tiles(int b) const { return b < t.c.batch ? Seen<TILE>(t.c.length(b), t.window, t.sinks).tiles : 0; }
  __device__ __forceinline__ int mine(int b) const { return b == 0 ? n0 : tiles(b + lane); }
  __device__ __forceinline__ int parts(int n) const { return n == 0 ? 0 : max(1, (n + share / 2) / share); }
  __device__ __forceinline__ static int last(int x) { return __builtin_amdgcn_readlane(x, 63); }
  __device__ __forceinline__ Deal(const Token& t_, int lane_) : t(t_), lane(lane_) {
    n0 = tiles(lane);
    int total = last(scan(n0));
    for (int b = 64; b < t.c.batch; b += 64) total += last(scan(tiles(b + lane)));
    share = max(kWaves, (total + t.units - 1) / t.units);
  }
  // The sequence that workgroup `unit` has a part of, -1 if none; the part, and how many there are
  __device__ __forceinline__ int find(int unit, int& part, int& count) const {
    for (int b = 0, before = 0; b < t.c.batch; b += 64) {
      const int n = parts(mine(b)), upto = scan(n);
      const uint64_t hit = __builtin_amdgcn_ballot_w64(before + upto > unit);
      if (hit != 0) {
        const int l = __builtin_ctzll(hit);
        count = __builtin_amdgcn_readlane(n, l);
        part = unit - (before + __builtin_amdgcn_readlane(upto, l) - count);
        return b + l;
      }
      before += last(upto);
    }
    return -1;
  }
  // The first workgroup of sequence b, and how many it has
  __device__ __forceinline__ int first(int b, int& count) const {
    int before = 0;
    for (int i = 0; i + 64 <= b; i += 64) before += last(scan(parts(mine(i))));
    const int n = parts(mine(b & ~63)), upto = scan(n);
    count = __builtin_amdgcn_readlane(n, b & 63);
    return before + __builtin_amdgcn_readlane(upto, b & 63) - count;
  }
};

// Where the parts of a sequence lie: in the slots of its workgroups
template <int TILE>
struct Shares {
  int first = 0, parts = 1;
  __device__ __forceinline__ Shares(const Token& t, int b, int lane) {
    if (t.dealt) first = Deal<TILE>(t, lane).first(__builtin_amdgcn_readfirstlane(b), parts);
  }
  __device__ __forceinline__ int64_t slot(const Token& t, int column, int part) const { return (int64_t)column * t.slots + min(first + part, t.slots - 1); }
};

// PAGES16: pages of a multiple of 16 entries, so that 16 in a row share one. WEIGHTS: scores are kept. ONCE: as in fetch.
template <int DT, int D, bool PAGES16, bool WEIGHTS, bool ONCE>
__global__ void __launch_bounds__(kThreads, 2) attend(Token t) {
  constexpr bool WIDE = DT == FHOG_DTYPE_FP32;
  typedef typename Type<DT>::T T;
  constexpr int TILE = kTile<DT>, SUB = TILE / 16;     // entries of a tile; 16 at a time
  constexpr float JUMP = DT == FHOG_DTYPE_FP16 ? 4.f : 8.f;
  constexpr int STEPS = D * (int)sizeof(T) / 64;          // 16-byte pieces of a row that a lane has (four lanes to a row)
  constexpr int C = D / 16;                               // channels of a lane in V and O
  constexpr int VB = C * sizeof(T), VW = VB >= 16 ? 4 : VB / 4, VN = VB >= 16 ? VB / 16 : 1;   // bytes of them, words of a load, loads
  typedef typename Words<4 * VW>::type VWord;
  __shared__ float tops[kWaves][kColumns], sums[kWaves][kColumns];
  __shared__ float rows[kWaves][kColumns][D + 4];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m = lane & 15, quarter = lane >> 4;
  // Workgroups of the same entries, for other heads of queries, come eight ids apart: on the same XCD, where the second one finds what the first one read
  const uint32_t turn = blockIdx.x / (8 * t.columns), inside = blockIdx.x - turn * (8 * t.columns), unit = 8 * turn + (inside & 7);
  const int own = unit / t.c.heads_k, g = unit - own * t.c.heads_k;   // those that there is nothing for come last
  if (own >= t.slots) return;
  const int column = g * t.columns + (inside >> 3), first_head = (inside >> 3) * kColumns;
  const int heads = min(kColumns, t.group - first_head);
  const char* const keys = t.c.keys + (int64_t)g * t.c.stride_h;
  const char* const values = t.c.values + (int64_t)g * t.c.stride_h;
  // a lane's bytes from the first of 16 entries that lie in a row
  const uint32_t stride = (uint32_t)t.c.stride_n, key_off = m * stride + quarter * 16;
  uint32_t value_off[4];
#pragma unroll
  for (int x = 0; x < 4; x++) value_off[x] = (4 * quarter + x) * stride + m * VB;

  // The first wave finds out what there is to do and says so: lengths that someone changes meanwhile make wrong results, but no waves that disagree on them at a barrier
  __shared__ int task[4];   // sequence, its entries, the tiles of this workgroup: the first one, and the one behind the last
  __shared__ bool task_shared;
  if (wave == 0) {
    int b = own, part = 0, parts = 1;
    if (t.dealt) b = Deal<TILE>(t, lane).find(own, part, parts);
    if (lane == 0) {
      const int n = b < 0 ? 0 : t.c.length(b);
      const int64_t tiles = Seen<TILE>(n, t.window, t.sinks).tiles;
      task[0] = b, task[1] = n, task[2] = (int)(tiles * part / parts), task[3] = (int)(tiles * (part + 1) / parts), task_shared = parts > 1;
    }
  }
  __syncthreads();
  const auto told = [&](int i) { return __builtin_amdgcn_readfirstlane(task[i]); };
  const int b = told(0), begin = told(2), end = told(3);
  if (b < 0) return;
  const bool shared = task_shared;
  const int64_t slot = (int64_t)column * t.slots + own;
  const int64_t row0 = (int64_t)b * t.heads_q + g * t.group + first_head;   // of (batch * heads_q)
  const Seen<TILE> seen(told(1), t.window, t.sinks);
  u32x4_t q[STEPS];
#pragma unroll
  for (int s = 0; s < STEPS; s++) {
    q[s] = u32x4_t{0, 0, 0, 0};
    if (m < heads) q[s] = *reinterpret_cast<const u32x4_t*>(t.q + b * t.qb + (int64_t)(g * t.group + first_head + m) * t.qh + s * 64 + quarter * 16);
  }
  float top = -INFINITY, sum = 0.f;   // of column m; the sum is this lane's share
  f32x4_t acc[C];
#pragma unroll
  for (int i = 0; i < C; i++) acc[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  const int32_t* const table = t.c.table + b * t.c.stride_tb;
  // Where the entries of a tile lie. `hidden`: some of them are not there or not seen, the same for the wave
  struct Place {
    int j0;
    bool hidden;
    int64_t at[SUB];   // in bytes from the pool's head g, -1: nowhere; of 16 entries in a row (PAGES16), else of entry m of 16, and of those that are seen alone
  };
  const auto locate = [&](int i) {
    Place p;
    p.j0 = seen.at(i), p.hidden = !seen.whole(p.j0);
#pragma unroll
    for (int u = 0; u < SUB; u++) {
      const int j = p.j0 + 16 * u + (PAGES16 ? 0 : m);
      uint32_t index = t.c.page(j);
      int32_t page = -1;
      if constexpr (PAGES16) {
        index = __builtin_amdgcn_readfirstlane(index);
        if (j < seen.n) page = table[index];
        page = __builtin_amdgcn_readfirstlane(page);
      } else {
        if (seen.sees(j)) page = table[index];
      }
      const bool found = (uint32_t)page < (uint32_t)t.c.pages;
      p.at[u] = found ? page * t.c.stride_p + (j - (int)(index * t.c.page.by)) * t.c.stride_n : -1;
      p.hidden = p.hidden || (PAGES16 ? !found : __builtin_amdgcn_ballot_w64(!found) != 0);
    }
    return p;
  };
  // Whether entry `from` of 16 is there, and where; from: this lane's or another's
  const auto entry = [&](const Place& p, int u, int from, int64_t& at) {
    if constexpr (PAGES16) {
      at = p.at[u];
      return at >= 0 && seen.sees(p.j0 + 16 * u + from);
    } else {
      at = (int64_t)((uint64_t)(uint32_t)__shfl((int)(p.at[u] >> 32), from) << 32 | (uint32_t)__shfl((int)p.at[u], from));
      return at >= 0;
    }
  };
  u32x4_t k[SUB][STEPS];
  VWord v[SUB][4][VN];
  uint32_t there = 0;   // bit 4 u + x: value x of the lane's four of 16 entries is there; looked at where some are not
  const auto load_keys = [&](const Place& p) {
    const auto all = [&](auto guard) {
#pragma unroll
      for (int u = 0; u < SUB; u++) {
        const char* const from = keys + p.at[u] + (PAGES16 ? key_off : quarter * 16);
        const bool ok = !guard.value || (p.at[u] >= 0 && (!PAGES16 || seen.sees(p.j0 + 16 * u + m)));
#pragma unroll
        for (int s = 0; s < STEPS; s++) k[u][s] = ok ? fetch<ONCE, u32x4_t>(from + s * 64) : u32x4_t{0, 0, 0, 0};
      }
    };
    if (p.hidden) all(std::true_type{});
    else all(std::false_type{});
  };
  const auto load_values = [&](const Place& p) {
    const auto all = [&](auto guard) {
#pragma unroll
      for (int u = 0; u < SUB; u++)
#pragma unroll
        for (int x = 0; x < 4; x++) {
          int64_t at;
          const bool seen_here = entry(p, u, 4 * quarter + x, at), ok = !guard.value || seen_here;
          if (guard.value) there = ok ? there | 1u << (4 * u + x) : there & ~(1u << (4 * u + x));
          const char* const from = values + at + (PAGES16 ? value_off[x] : m * VB);
#pragma unroll
          for (int y = 0; y < VN; y++) v[u][x][y] = ok ? fetch<ONCE, VWord>(from + y * 16) : VWord(0u);
        }
    };
    if (p.hidden) all(std::true_type{});
    else all(std::false_type{});
  };
  // A tile's keys are asked for once those of the tile before have been multiplied, its values once those have: into the same registers, with the other half of
  // a tile's work to hide behind. us, 64 x 2048, 8 heads of keys, bf16, d = 128 86.5 -> 84.5, 16 x 4096 with weights 55.8 -> 53.4
  Place p;
  if (begin + wave < end) p = locate(begin + wave), load_keys(p), load_values(p);
  for (int i = begin + wave; i < end; i += kWaves) {
    const bool hidden = p.hidden, more = i + kWaves < end;
    if (more) p = locate(i + kWaves);
    // S^T of the tile, in log2 units
    f32x4_t x[SUB];
#pragma unroll
    for (int u = 0; u < SUB; u++) {
      f32x4_t s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < STEPS; c++) {
        if constexpr (WIDE) {
#pragma unroll
          for (int e = 0; e < 4; e++) s = __builtin_amdgcn_mfma_f32_16x16x4f32(number(k[u][c][e]), number(q[c][e]), s, 0, 0, 0);
        } else {
          s = mfma16<DT>(k[u][c], q[c], s);
        }
      }
      x[u] = s * t.scale_log2;
      if (hidden) {
#pragma unroll
        for (int e = 0; e < 4; e++) x[u][e] = there >> (4 * u + e) & 1 ? x[u][e] : -INFINITY;   // the entries of this lane's values are those of its scores
      }
      if (WEIGHTS && m < heads) *reinterpret_cast<f32x4_t*>(t.scores + (row0 + m) * t.row + i * TILE + 16 * u + 4 * quarter) = x[u];
    }
    if (more) load_keys(p);
    float high = x[0][0];
#pragma unroll
    for (int u = 0; u < SUB; u++) high = fmaxf(fmaxf(high, fmaxf(x[u][0], x[u][1])), fmaxf(x[u][2], x[u][3]));
    high = fmaxf(high, __shfl_xor(high, 16));
    high = fmaxf(high, __shfl_xor(high, 32));
    // The reference of the exponentials follows the maximum only in jumps of more than 8 (in log2 units; fp16: kLift): weights may then reach 2^8, which costs no precision,
    // and the sums are scaled again only now and then
    const float next = high > top + JUMP ? high : top;
    const float ref = next == -INFINITY ? 0.f : next;   // a column that has seen nothing yet
    if (__builtin_amdgcn_ballot_w64(next > top) != 0) {
      const float by = __builtin_amdgcn_exp2f(top - ref);
      sum *= by;
#pragma unroll
      for (int c = 0; c < C; c++) acc[c] *= by;
    }
    top = next;
#pragma unroll
    for (int u = 0; u < SUB; u++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        x[u][e] = __builtin_amdgcn_exp2f(x[u][e] - ref);
        sum += x[u][e];
      }
    // O^T += V^T P^T
    if constexpr (WIDE) {
#pragma unroll
      for (int u = 0; u < SUB; u++)
#pragma unroll
        for (int e = 0; e < 4; e++)
#pragma unroll
          for (int c = 0; c < C; c++) acc[c] = __builtin_amdgcn_mfma_f32_16x16x4f32(number(word<VW>(v[u][e][c / VW], c % VW)), x[u][e], acc[c], 0, 0, 0);
    } else {
#pragma unroll
      for (int u = 0; u < SUB; u += 2) {
        // The products' other factor, the values, has 16 bits, so a weight enters in two terms of its type, what it is cut to and what that leaves: off by 2^-15 of a weight in
        // bf16 and 2^-19 in fp16 (and 2^-35 of the largest), where one term is by 2^-8 and 2^-11. The matrix pipe has little else to do: us, one
        // term | two: bf16, d = 128 32 x 16384 291 | 291, 64 x 2048 84.5 | 84.4, d = 32 32 x 8192 56.2 | 56.3; fp16, d = 64, window 700 of 24 x 3001, where its latency shows, 13.9 | 14.5
        u32x4_t weights, rest;
#pragma unroll
        for (int y = 0; y < 4; y++) {
          const u32x2_t both = cut<DT>(x[u + y / 2][2 * (y % 2)] * kLift<DT>, x[u + y / 2][2 * (y % 2) + 1] * kLift<DT>);
          weights[y] = both[0], rest[y] = both[1];
        }
#pragma unroll
        for (int c = 0; c < C; c += 2) {
          const int w = c / 2;   // the word of channels c, c + 1
          u32x4_t even, odd;
#pragma unroll
          for (int y = 0; y < 4; y++) {
            const uint32_t lo = word<VW>(v[u + y / 2][2 * (y % 2)][0], w), hi = word<VW>(v[u + y / 2][2 * (y % 2) + 1][0], w);
            even[y] = __builtin_amdgcn_perm(hi, lo, 0x05040100), odd[y] = __builtin_amdgcn_perm(hi, lo, 0x07060302);
          }
          acc[c] = mfma16<DT>(even, rest, mfma16<DT>(even, weights, acc[c]));
          acc[c + 1] = mfma16<DT>(odd, rest, mfma16<DT>(odd, weights, acc[c + 1]));
        }
      }
    }
    if (more) load_values(p);
  }

  // The waves' results on one maximum, joined in their order
  sum += __shfl_xor(sum, 16);
  sum += __shfl_xor(sum, 32);
  if (quarter == 0) tops[wave][m] = top;
  __syncthreads();
  float all = tops[0][m];
#pragma unroll
  for (int w = 1; w < kWaves; w++) all = fmaxf(all, tops[w][m]);
  const float by = __builtin_amdgcn_exp2f(top - (all == -INFINITY ? 0.f : all));
  if (quarter == 0) sums[wave][m] = sum * by;
#pragma unroll
  for (int c = 0; c < C; c++)
#pragma unroll
    for (int r = 0; r < 4; r++) rows[wave][m][C * (4 * quarter + r) + c] = acc[c][r] * (by / kLift<DT>);
  __syncthreads();
  for (int at = tid * 4; at < kColumns * D; at += kThreads * 4) {
    const int h = at / D, c = at % D;
    if (h >= heads) break;
    f32x4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kWaves; w++) o += *reinterpret_cast<const f32x4_t*>(&rows[w][h][c]);
    if (shared) {
      *reinterpret_cast<f32x4_t*>(t.part + (slot * kColumns + h) * D + c) = o;
    } else {
      float total = sums[0][h];
#pragma unroll
      for (int w = 1; w < kWaves; w++) total += sums[w][h];
      o *= total > 0.f ? 1.f / total : total == 0.f ? 0.f : total;   // nothing seen: 0
      char* const to = t.o + b * t.ob + (int64_t)(g * t.group + first_head + h) * t.oh + c * sizeof(T);
      if constexpr (WIDE) *reinterpret_cast<f32x4_t*>(to) = o;
      else *reinterpret_cast<u32x2_t*>(to) = u32x2_t{pack<DT>(o[0], o[1]), pack<DT>(o[2], o[3])};
    }
  }
  if (tid < heads) {
    float total = sums[0][tid], high = tops[0][tid];
#pragma unroll
    for (int w = 1; w < kWaves; w++) total += sums[w][tid], high = fmaxf(high, tops[w][tid]);
    if (shared) {
      t.stats[slot * kColumns + tid] = f32x2_t{high, total};
    } else {
      if (WEIGHTS) t.whole[row0 + tid] = f32x2_t{high, total};
      t.lse[row0 + tid] = total == 0.f ? -INFINITY : (high + __builtin_amdgcn_logf(total)) * kLn2;
    }
  }
}

// Maximum, in log2 units, and sum over the parts of head `head` of a column, by the lanes of a wave
template <int TILE>
__device__ __forceinline__ f32x2_t joined(const Token& t, const Shares<TILE>& of, int column, int head, int lane) {
  float high = -INFINITY, total = 0.f;
  for (int i = lane; i < of.parts; i += 64) high = fmaxf(high, t.stats[of.slot(t, column, i) * kColumns + head][0]);
#pragma unroll
  for (int d = 1; d < 64; d *= 2) high = fmaxf(high, __shfl_xor(high, d));
  const float ref = high == -INFINITY ? 0.f : high;
  for (int i = lane; i < of.parts; i += 64) {
    const f32x2_t s = t.stats[of.slot(t, column, i) * kColumns + head];
    total += s[1] * __builtin_amdgcn_exp2f(s[0] - ref);
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) total += __shfl_xor(total, d);
  return f32x2_t{high, total};
}

// O and L of a row that several workgroups have shared: a lane has four channels, groups of D / 4 lanes take the parts in turn. (With one group and part after part 32 parts of 16
// rows took 21 us, each load waiting for the one before; so 4.) Rows of sequences without entries, which no workgroup had.
template <int DT, int D>
__device__ __forceinline__ void join_row(const Token& t, int64_t row, int tid) {
  constexpr bool WIDE = DT == FHOG_DTYPE_FP32;
  constexpr int LANES = D / 4, GROUPS = kThreads / LANES;
  __shared__ f32x4_t sums[GROUPS][LANES];
  const int group = tid / LANES, c = tid % LANES * 4, b = (int)(row / t.heads_q), h = (int)(row - (int64_t)b * t.heads_q);
  __shared__ int parts;   // as the first wave has them: all waves are to agree on whether there is something to do
  const Shares<kTile<DT>> of(t, b, tid & 63);
  if (tid == 0) parts = of.parts;
  __syncthreads();
  if (parts == 1) return;
  const int g = h / t.group, inside = h - g * t.group, column = g * t.columns + inside / kColumns, head = inside % kColumns;
  const f32x2_t all = joined(t, of, column, head, tid & 63);   // every wave for itself
  const float ref = all[0] == -INFINITY ? 0.f : all[0];
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int i = group; i < of.parts; i += GROUPS) {
    const int64_t at = of.slot(t, column, i) * kColumns + head;
    o += *reinterpret_cast<const f32x4_t*>(t.part + at * D + c) * __builtin_amdgcn_exp2f(t.stats[at][0] - ref);
  }
  sums[group][tid % LANES] = o;
  __syncthreads();
  if (group != 0) return;
  for (int i = 1; i < GROUPS; i++) o += sums[i][tid];
  o *= all[1] > 0.f ? 1.f / all[1] : all[1] == 0.f ? 0.f : all[1];
  char* const to = t.o + b * t.ob + h * t.oh + c * sizeof(typename Type<DT>::T);
  if constexpr (WIDE) *reinterpret_cast<f32x4_t*>(to) = o;
  else *reinterpret_cast<u32x2_t*>(to) = u32x2_t{pack<DT>(o[0], o[1]), pack<DT>(o[2], o[3])};
  if (c == 0) t.lse[row] = all[1] == 0.f ? -INFINITY : (all[0] + __builtin_amdgcn_logf(all[1])) * kLn2;
}

constexpr int kEntries = 4 * kThreads;   // of the weights that a workgroup adds to

// The weights of kEntries entries of a head of keys: what was kept of their scores, on the joined statistics
template <int DT>
__device__ __forceinline__ void add_weights(const Token& t, int64_t id, int tid) {
  constexpr int kHeads = 64, kGroup = 4;   // heads of queries at a time
  __shared__ float lse[kHeads];
  const int blocks = (t.c.capacity + kEntries - 1) / kEntries;
  const int64_t slice = id / blocks;
  const int b = (int)(slice / t.c.heads_k), g = (int)(slice - (int64_t)b * t.c.heads_k), j0 = (int)(id - slice * blocks) * kEntries + tid;
  const Seen<kTile<DT>> seen(t.c.length(b), t.window, t.sinks);
  const int64_t row0 = (int64_t)b * t.heads_q + g * t.group;
  const float* const in = t.weights_in + b * t.wib + g * t.wih;
  float* const out = t.weights_out + b * t.wob + g * t.woh;
  float w[4];
#pragma unroll
  for (int i = 0; i < 4; i++) w[i] = j0 + i * kThreads < t.c.capacity ? in[j0 + i * kThreads] : 0.f;
  const float* const scores = t.scores + row0 * t.row;
  int place[4];
#pragma unroll
  for (int i = 0; i < 4; i++) place[i] = seen.sees(j0 + i * kThreads) ? seen.place(j0 + i * kThreads) : -1;
  float s[kGroup][4];
  const auto load = [&](int h0) {   // of kGroup heads
#pragma unroll
    for (int h = 0; h < kGroup; h++)
#pragma unroll
      for (int i = 0; i < 4; i++) s[h][i] = h0 + h < t.group && place[i] >= 0 ? scores[(h0 + h) * t.row + place[i]] : -INFINITY;
  };
  load(0);   // before the statistics, for which it does not have to wait
  const Shares<kTile<DT>> of(t, b, tid & 63);
  for (int h0 = 0; h0 < t.group; h0 += kHeads) {
    const int heads = min(kHeads, t.group - h0);
    __syncthreads();
    for (int h = tid >> 6; h < heads; h += kWaves) {
      const f32x2_t all = of.parts > 1 ? joined(t, of, g * t.columns + (h0 + h) / kColumns, (h0 + h) % kColumns, tid & 63) : seen.tiles ? t.whole[row0 + h0 + h] : f32x2_t{0.f, 0.f};
      if ((tid & 63) == 0) lse[h] = all[1] == 0.f ? INFINITY : all[0] + __builtin_amdgcn_logf(all[1]);
    }
    __syncthreads();
    for (int h1 = 0; h1 < heads; h1 += kGroup) {
#pragma unroll
      for (int h = 0; h < kGroup; h++)
        if (h1 + h < heads)
#pragma unroll
          for (int i = 0; i < 4; i++) w[i] = s[h][i] == -INFINITY ? w[i] : w[i] + __builtin_amdgcn_exp2f(s[h][i] - lse[h1 + h]);   // else as it was, also -0
      load(h0 + h1 + kGroup);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; i++)
    if (j0 + i * kThreads < t.c.capacity) out[j0 + i * kThreads] = w[i];
}

// What is left after the parts, in one launch: workgroups that join rows, and those that add weights behind them
template <int DT, int D>
__global__ void __launch_bounds__(kThreads) join_parts(Token t, int rows) {
  if ((int)blockIdx.x < rows) join_row<DT, D>(t, blockIdx.x, threadIdx.x);
  else add_weights<DT>(t, (int64_t)blockIdx.x - rows, threadIdx.x);
}

// How the tiles of a call are dealt out, and what that leaves in the workspace
struct Plan {
  int units, slots;
  bool dealt;
  int64_t row;   // scores of a row
  size_t part_bytes, stats_bytes, whole_bytes, score_bytes;
  size_t bytes() const { return part_bytes + stats_bytes + whole_bytes + score_bytes; }
};

size_t up16(size_t n) { return (n + 15) & ~(size_t)15; }

Plan plan_of(const fhog_paged_attn_args* a) {
  Plan p;
  const fhog_paged_cache& c = a->cache;
  const int64_t tile = tile_of(c.dtype), capacity = c.table_width * c.page;
  int64_t most = capacity;   // entries that a token may see
  if (a->window > 0 && a->window < capacity) most = std::min(capacity, a->window + std::min(a->sinks, capacity) + 2 * tile);
  const int64_t tiles = (most + tile - 1) / tile, group = a->heads_q / c.heads_k, columns = c.heads_k * ((group + kColumns - 1) / kColumns), slices = c.batch * columns;
  // Two workgroups to a CU, as few as keep memory busy: what is split has to be joined. us at 512 | 768 | 1024 workgroups, bf16, d = 128, 8 heads of keys, when each sequence had
  // as many parts as the longest would need: 1 x 32768 28.5 | 31.0 | 30.5, 8 x 4096 28.2 | 29.4 | 29.0, 64 x 2048 84.5 | 90.5 | 90.6. Dealt out by their lengths: 16384 beside 31 of 500
  // 138 -> 30, beside 63 of 100 240 -> 30, 8192 and 300 in turn 136 -> 99; 8 x 4096 28.5 -> 29.2, 1 x 4096 12.1 -> 13.0, which is what finding out costs. So not where one workgroup
  // reads up to 256 KiB, 512 where every CU has one (dealt out | not, 8 sequences of 600 d = 128 14.6 | 16.4, d = 64 11.9 | 9.7, 1 x 300 11.6 | 9.4; 32 of 1000 d = 128 29.9 | 25.8,
  // d = 64 19.1 | 13.8), or where there are two to a CU, of sequences too short to leave much of the GPU idle at the end.
  const int64_t bytes = most * 2 * c.d * (c.dtype == FHOG_DTYPE_FP32 ? 4 : 2);
  p.dealt = bytes > (slices < 256 ? 256 << 10 : 512 << 10) && c.batch <= 512 && (slices < 512 || bytes >= 2 << 20) && tiles * c.batch < ((int64_t)1 << 30);
  // Beyond 1 MiB to a workgroup more of them, which start as others end: ragged lengths even out better. us, 32 sequences of 12000 to 16384 304 -> 291, 64 of 500 to 8192 238 -> 190, 16 of
  // 2000 to 16384 113 -> 110; with 512 KiB to each 302, 197, 111
  const int64_t many = std::min<int64_t>(2048, std::max<int64_t>(512, bytes * c.batch * c.heads_k >> 20));
  p.units = (int)(p.dealt ? std::max<int64_t>(1, std::min(many / columns, (tiles * c.batch + kWaves - 1) / kWaves)) : c.batch);
  p.slots = (int)(p.dealt ? p.units + c.batch : c.batch);   // a part is rounded up by less than one for each sequence
  // A window sees as many entries of a wide table as of one cut to it: with 64 sequences of 64 heads, 131072 entries and window 700 the scores take 12.6 MB, not 2.1 GB
  p.row = tile * (c.dtype == FHOG_DTYPE_FP32 ? Seen<kTile<FHOG_DTYPE_FP32>>::most(capacity, a->window, a->sinks) : Seen<kTile<FHOG_DTYPE_BF16>>::most(capacity, a->window, a->sinks));
  const int64_t slots = p.slots * columns, rows = c.batch * a->heads_q;
  p.part_bytes = p.dealt ? sizeof(float) * slots * kColumns * c.d : 0;
  p.stats_bytes = p.dealt ? sizeof(f32x2_t) * slots * kColumns : 0;
  p.whole_bytes = a->weights_out ? up16(sizeof(f32x2_t) * rows) : 0;
  p.score_bytes = a->weights_out ? sizeof(float) * rows * p.row : 0;
  return p;
}

template <int DT, int D>
hipError_t launch_d(const Token& t, hipStream_t s) {
  const int64_t units = (int64_t)t.slots * t.c.heads_k;
  const dim3 grid((unsigned)((units + 7) / 8 * 8 * t.columns));
  const bool pages16 = t.c.page.by % 16 == 0;
  const auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, s, t); };
  const auto pick = [&](auto once) {
    constexpr bool ONCE = decltype(once)::value;
    if (t.weights_out) pages16 ? go(attend<DT, D, true, true, ONCE>) : go(attend<DT, D, false, true, ONCE>);
    else pages16 ? go(attend<DT, D, true, false, ONCE>) : go(attend<DT, D, false, false, ONCE>);
  };
  constexpr bool WHOLE_LINES = D * sizeof(typename Type<DT>::T) >= 256;
  if (WHOLE_LINES && t.columns == 1) pick(std::bool_constant<WHOLE_LINES>{});
  else pick(std::false_type{});
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || (!t.dealt && !t.weights_out)) return e;
  const int64_t rows = t.dealt ? (int64_t)t.c.batch * t.heads_q : 0;
  const int64_t weights = t.weights_out ? (int64_t)t.c.batch * t.c.heads_k * ((t.c.capacity + kEntries - 1) / kEntries) : 0;
  hipLaunchKernelGGL((join_parts<DT, D>), dim3((unsigned)(rows + weights)), dim3(kThreads), 0, s, t, (int)rows);
  return hipGetLastError();
}
template <int DT>
hipError_t launch_t(const Token& t, int64_t d, hipStream_t s) {
  switch (d) {
    case 32: return launch_d<DT, 32>(t, s);
    case 64: return launch_d<DT, 64>(t, s);
    default: return launch_d<DT, 128>(t, s);
  }
}

}  // namespace

size_t paged_attn_bytes(const fhog_paged_attn_args* a) { return plan_of(a).bytes(); }

hipError_t launch_paged_attn(const fhog_paged_attn_args* a, hipStream_t s) {
  const Plan p = plan_of(a);
  const int es = a->cache.dtype == FHOG_DTYPE_FP32 ? 4 : 2;
  Token t;
  t.c = cache_of(a->cache);
  t.q = (const char*)a->q, t.o = (char*)a->o, t.lse = a->lse, t.weights_in = a->weights_in, t.weights_out = a->weights_out;
  t.qb = a->stride_qb * es, t.qh = a->stride_qh * es, t.ob = a->stride_ob * es, t.oh = a->stride_oh * es;
  t.wib = a->stride_wib, t.wih = a->stride_wih, t.wob = a->stride_wob, t.woh = a->stride_woh;
  t.heads_q = (int32_t)a->heads_q, t.group = (int32_t)(a->heads_q / a->cache.heads_k), t.columns = (t.group + kColumns - 1) / kColumns;
  t.window = (int32_t)std::min<int64_t>(a->window, INT32_MAX), t.sinks = (int32_t)std::min<int64_t>(a->sinks, t.c.capacity);
  t.units = p.units, t.slots = p.slots, t.dealt = p.dealt, t.scale_log2 = a->scale * kLog2e, t.row = p.row;
  char* const ws = (char*)a->ws;
  t.part = (float*)ws, t.stats = (f32x2_t*)(ws + p.part_bytes);
  t.whole = (f32x2_t*)(ws + p.part_bytes + p.stats_bytes), t.scores = (float*)(ws + p.part_bytes + p.stats_bytes + p.whole_bytes);
  switch (a->cache.dtype) {
    case FHOG_DTYPE_FP32: return launch_t<FHOG_DTYPE_FP32>(t, a->cache.d, s);
    case FHOG_DTYPE_FP16: return launch_t<FHOG_DTYPE_FP16>(t, a->cache.d, s);
    default: return launch_t<FHOG_DTYPE_BF16>(t, a->cache.d, s);
  }
}

}  // namespace fhog
