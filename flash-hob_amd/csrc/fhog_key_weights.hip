// The weight that each key got from the queries of a prompt:
//
//   out_j = sum_h sum_i exp(scale q_hi . k_j - L_hi)
//
// over the heads h of queries of the key's head and the queries i that see key j: the column sums of attention's weights, recomputed from Q, K and L. Nothing of shape
// (N_Q, N_K) is stored.
//
// A workgroup owns 128 NK keys, 32 NK to a wave, in registers, and streams the queries of all heads of its group through LDS, 64 at a time. S = Q K^T with 32x32
// products puts a key into a lane and 16 queries into its registers, so the sum over the queries is a lane's own until the end. The tiles of queries that a
// workgroup would go through are cut into pieces of equal length, one to a workgroup, where there are several they leave partial sums, which a second kernel
// adds in their order: a causal mask leaves the first keys many times the work of the last, and a sink all of it.
//
// What bounds it: the instructions of a SIMD. A block of 32 x 32 pairs takes d / 16 matrix instructions of 32 cycles and 48 vector instructions, 16 of them exponentials at half
// rate: 256 cycles each at d = 128. The matrix instructions of one wave run beside the exponentials of another: three workgroups to a CU, four below d = 128. bf16, 16 heads x 16384
// causal, four to one of keys, d = 128: 540 us (557 on another card), 1020 TFLOP/s, 86 % of what a large library product of bf16 matrices reaches here, which takes no exponentials.
#include <algorithm>

#include "fhog_small.h"

namespace fhog {
using namespace bf16k;
namespace {

constexpr int kThreads = 256;
// Queries of a stage. Rows of 512 bytes in stages of 64 leave room in LDS for one workgroup, of 32 for three: fp32, d = 128, us 16 x 8192 1642 -> 1120 (122 TFLOP/s of the 154 that a
// large library product reaches), 8 x 2048 74 -> 59, 16 x 4096, window 512 130 -> 103
constexpr int rows_of(int bytes) { return bytes > 256 ? 32 : 64; }
// Stages in LDS: the one that is read, the one after it, which has landed so that its statistics can be made ready, and one that is on its way
constexpr int kRing = 3;

struct Weigh {
  const char* q;
  const char* k;
  const float* lse;
  const int32_t* lengths;
  float* out;
  float* part;                                // [piece][batch * heads_k][n_k]
  int64_t qb, qh, qn, kb, kh, kn, ob, oh;     // of q and k in bytes
  int32_t batch, heads_q, heads_k, group, n_q, n_k;
  int32_t causal, off, window, sinks;         // key j is seen by query i iff j <= i + off and (i + off - j < window or j < sinks)
  int32_t tiles, pieces, chunk;               // of keys; pieces of a tile of keys at most; stages of a piece
  float scale_log2;
};

// Pieces into which the stages of a tile of keys go: as few as hold `chunk` each at most, the same number in every kernel
__device__ __forceinline__ int pieces_of(int steps, const Weigh& w) { return steps == 0 ? 0 : (steps - 1) / w.chunk + 1; }

// Which queries see a key
struct Queries {
  int n_q, n_k, off, window, sinks, causal;
  // length: of the sequence, where there are lengths; padding is as if it were not there
  __device__ __forceinline__ Queries(const Weigh& w, int length) : n_q(w.n_q), n_k(w.n_k), off(w.off), window(w.window), sinks(w.sinks), causal(w.causal) {
    if (w.lengths) {
      n_k = max(0, min(length, n_k));
      n_q = max(0, min(n_k - off, n_q));
    }
  }
  __device__ __forceinline__ int first(int j) const { return causal ? max(0, j - off) : 0; }
  __device__ __forceinline__ int last(int j) const { return causal && j >= sinks && j - off < n_q - window ? j - off + window - 1 : n_q - 1; }
  // stages of ROWS queries of which some see some of the keys [j, j + n)
  template <int ROWS>
  __device__ __forceinline__ void stages(int j, int n, int& begin, int& end) const {
    begin = end = 0;
    if (j >= n_k || n_q == 0) return;
    const int to = j < sinks ? n_q - 1 : last(min(j + n, n_k) - 1);
    begin = first(j) / ROWS, end = max(begin, to / ROWS + 1);
    if (first(j) >= n_q) end = begin;
  }
};

template <int DT>
struct Type;
template <>
struct Type<FHOG_DTYPE_BF16> {
  typedef uint16_t T;
};
template <>
struct Type<FHOG_DTYPE_FP16> {
  typedef uint16_t T;
};
template <>
struct Type<FHOG_DTYPE_FP32> {
  typedef float T;
};

// The bits of a vector's element as a number; handed over by value: of an element itself __builtin_bit_cast takes the vector's first
__device__ __forceinline__ float number(uint32_t bits) { return __builtin_bit_cast(float, bits); }

// rows of BYTES bytes in LDS: chunk ch of row r lies at ch ^ swizzle(r), so that the 16-byte reads of a column of rows meet no bank twice
template <int BYTES>
__device__ __forceinline__ int swizzle(int r) {
  return swz<(BYTES > 256 ? 128 : BYTES / 2)>(r);
}

// Workgroups of a CU that the registers are to leave room for; the stages in LDS do. us, 16 x 16384 causal, 64 keys to a wave: d = 128 with two
// workgroups 605, with three 538, with two that take the exponentials of one tile of queries behind the matrix products of the next 619; d = 64 with three 368, with four 355
template <int DT, int D>
constexpr int kWorkgroups = D == 128 || DT == FHOG_DTYPE_FP32 ? 3 : 4;

template <int DT, int D, int NK>
__global__ void __launch_bounds__(kThreads, (kWorkgroups<DT, D>)) weigh(Weigh w) {
  constexpr bool WIDE = DT == FHOG_DTYPE_FP32, F16 = DT == FHOG_DTYPE_FP16;
  constexpr int BYTES = D * (int)sizeof(typename Type<DT>::T), CHUNKS = BYTES / 16, PER_LOAD = 64 / CHUNKS, ROWS = rows_of(BYTES), LOADS = ROWS / PER_LOAD / 4;
  constexpr int TILE = ROWS * BYTES, STAGE = TILE + 256, KEYS = 128 * NK, STEPS = CHUNKS / 2;
  extern __shared__ __attribute__((aligned(16))) char smem[];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 31, h = lane >> 5;
  // Workgroup ids go round the eight XCDs: one piece of every tile after the other, so that those that have no such piece are spread over them, each piece beginning a
  // tile further on, so that those of a tile are too. (Tile after tile, 64 tiles of 16 pieces left half of the XCDs idle: us, 16 x 16384 causal, d = 128 1082, so 650.)
  const int piece = blockIdx.x / w.tiles, g = blockIdx.y, b = blockIdx.z;
  int tile = blockIdx.x - piece * w.tiles + piece % w.tiles;
  if (tile >= w.tiles) tile -= w.tiles;
  int length = 0;
  if (w.lengths) {   // one thread reads it: lengths that someone changes meanwhile make wrong results, but no waves that disagree at a barrier
    __shared__ int read;
    if (tid == 0) read = w.lengths[b];
    __syncthreads();
    length = __builtin_amdgcn_readfirstlane(read);
  }
  const Queries geo(w, length);
  const int k0 = tile * KEYS, kw = k0 + 32 * NK * wave;
  int begin, end;
  geo.template stages<ROWS>(k0, KEYS, begin, end);
  const int each = end - begin, steps = w.group * each, pieces = pieces_of(steps, w);
  if (piece >= max(pieces, w.pieces == 1 ? 1 : 0)) return;
  const int from = piece * w.chunk, to = from + min(steps - from, w.chunk);

  u32x4_t key[NK][STEPS];
  int lo[NK], hi[NK];                              // queries that see this lane's keys
  int any_lo = INT32_MAX, any_hi = -1, whole_lo = 0, whole_hi = INT32_MAX;   // ... some of the wave's, and all of them
#pragma unroll
  for (int x = 0; x < NK; x++) {
    const int j0 = kw + 32 * x, j = j0 + n, last = min(j0 + 31, geo.n_k - 1);
    const char* const row = w.k + b * w.kb + g * w.kh + (int64_t)max(0, min(j, geo.n_k - 1)) * w.kn + 16 * h;
#pragma unroll
    for (int s = 0; s < STEPS; s++) key[x][s] = geo.n_k > 0 ? *reinterpret_cast<const u32x4_t*>(row + 32 * s) : u32x4_t{0, 0, 0, 0};
    lo[x] = geo.first(j), hi[x] = j < geo.n_k ? geo.last(j) : -1;
    any_lo = min(any_lo, geo.first(j0)), any_hi = max(any_hi, j0 >= geo.n_k ? -1 : j0 < geo.sinks ? geo.n_q - 1 : geo.last(last));
    whole_lo = max(whole_lo, geo.first(j0 + 31)), whole_hi = min(whole_hi, j0 + 31 >= geo.n_k ? -1 : geo.last(max(j0, min(geo.sinks, j0 + 31))));
  }
  float sum[NK] = {};
  // staging: straight into LDS, 1 KiB to an instruction; rows past the end are copies of the last
  uint32_t off[LOADS];
  const auto offset = [&](int u, int valid) {
    const int r = (wave + 4 * u) * PER_LOAD + lane / CHUNKS, pc = lane % CHUNKS;
    return (uint32_t)(min(r, valid - 1) * (uint32_t)w.qn) + (uint32_t)((pc ^ swizzle<BYTES>(r)) << 4);
  };
#pragma unroll
  for (int u = 0; u < LOADS; u++) off[u] = offset(u, ROWS);
  const uint32_t ring = lds_addr(smem);
  int t = begin;            // of the stage that is issued next; its queries, its statistics, and where it goes
  const int64_t row0 = (int64_t)b * w.heads_q + g * w.group, stage_bytes = ROWS * w.qn;
  const char* src = w.q + b * w.qb + (int64_t)g * w.group * w.qh + begin * stage_bytes;
  const float* lse = w.lse + row0 * w.n_q + begin * ROWS;
  uint32_t into = ring;
  if (each > 0) {
    const int head = from / each;
    t = begin + from - head * each, src += head * w.qh + (t - begin) * stage_bytes, lse += (int64_t)head * w.n_q + (t - begin) * ROWS;
  }
  const int64_t back = w.qh - (each - 1) * stage_bytes, lse_back = w.n_q - (int64_t)(each - 1) * ROWS;   // to the first stage of the next head
  const auto issue = [&] {
    const int valid = geo.n_q - t * ROWS;
    if (valid >= ROWS) {
      if (wave == 3) smallk::stage_words(into + TILE, lse + lane % ROWS);
#pragma unroll
      for (int u = 0; u < LOADS; u++) Dma<64>::issue_one(into + (wave + 4 * u) * 1024, off[u], (const __bf16*)src);
    } else {
      keep_branch();
      if (wave == 3) smallk::stage_words(into + TILE, lse + min(lane % ROWS, valid - 1));
#pragma unroll
      for (int u = 0; u < LOADS; u++) Dma<64>::issue_one(into + (wave + 4 * u) * 1024, offset(u, valid), (const __bf16*)src);
    }
    into = into == ring + (kRing - 1) * STAGE ? ring : into + STAGE;
    if (++t == end) t = begin, src += back, lse += lse_back;
    else src += stage_bytes, lse += ROWS;
  };
  // L in log2 units: it and the score are rounded there apart, 1.5e-7 of the weights (5e-8 if their difference were, which takes an instruction more to a score). A query that saw nothing has no weights to give, whatever it holds: it becomes 0, exp(0 - infinity)
  const auto make_ready = [&](char* stage) {
    float* const at = reinterpret_cast<float*>(stage + TILE) + lane;
    const float l = *at;
    *at = l == -INFINITY ? INFINITY : l * kLog2e;
    for (uint64_t empty = __builtin_amdgcn_ballot_w64(lane < ROWS && l == -INFINITY); empty != 0; empty &= empty - 1)
      for (int c = lane; c < BYTES / 4; c += 64) reinterpret_cast<uint32_t*>(stage + __builtin_ctzll(empty) * BYTES)[c] = 0;
  };
  for (int i = 0; i < kRing - 1 && from + i < to; i++) issue();
  wait_vm0();   // the keys and the first stages; with the builtin, or the compiler waits for the keys, and for the stages under way, in every tile
  __syncthreads();
  if (from < to && wave == 0) make_ready(smem);
  char* stage = smem;
  __syncthreads();
  int now = each > 0 ? begin + from % each : 0;
  for (int step = from; step < to; step++) {
    const bool more = step + kRing - 1 < to;
    if (more) issue();
    char* const after = stage == smem + (kRing - 1) * STAGE ? smem : stage + STAGE;
    if (step + 1 < to && wave == (step & 3)) make_ready(after);
#pragma unroll
    for (int u = 0; u < ROWS / 32; u++) {
      const int i0 = now * ROWS + 32 * u;
      if (i0 > any_hi || i0 + 31 < any_lo) continue;   // no query of the tile sees a key of this wave
      constexpr int AHEAD = STEPS < 3 ? STEPS : 3;
      const char* const row = stage + (32 * u + n) * BYTES;
      u32x4_t a[AHEAD];
      const auto read = [&](int c) { a[c % AHEAD] = *reinterpret_cast<const u32x4_t*>(row + (((2 * c + h) ^ swizzle<BYTES>(n)) << 4)); };
#pragma unroll
      for (int c = 0; c < AHEAD - 1; c++) read(c);
      f32x16_t scores[NK];
#pragma unroll
      for (int c = 0; c < STEPS; c++) {
        if (c + AHEAD - 1 < STEPS) read(c + AHEAD - 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int x = 0; x < NK; x++) {
          if (c == 0) scores[x] = f32x16_t{0};
          if constexpr (WIDE) {
#pragma unroll
            for (int e = 0; e < 4; e++) scores[x] = __builtin_amdgcn_mfma_f32_32x32x2f32(number(a[c % AHEAD][e]), number(key[x][c][e]), scores[x], 0, 0, 0);
          } else {
            scores[x] = mfma<F16>(__builtin_bit_cast(bf16x8_t, a[c % AHEAD]), __builtin_bit_cast(bf16x8_t, key[x][c]), scores[x]);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      f32x4_t stats[4];   // L of the lane's 16 queries: 8 g + 4 h + e
#pragma unroll
      for (int e = 0; e < 4; e++) stats[e] = *reinterpret_cast<const f32x4_t*>(stage + TILE + (32 * u + 8 * e + 4 * h) * 4);
      const auto weight = [&](int x, int r) { return __builtin_amdgcn_exp2f(__builtin_fmaf(scores[x][r], w.scale_log2, -stats[r / 4][r % 4])); };
      // sums of tiles, then of their sums: a sum over many queries is rounded once for each tile, not for each query
      if (i0 >= whole_lo && i0 + 31 <= whole_hi) {
#pragma unroll
        for (int x = 0; x < NK; x++) {
          float part[2] = {weight(x, 0), weight(x, 1)};
#pragma unroll
          for (int r = 2; r < 16; r++) part[r % 2] += weight(x, r);
          sum[x] += part[0] + part[1];
        }
      } else {   // some queries do not see some keys
        keep_branch();
#pragma unroll
        for (int x = 0; x < NK; x++) {
          float all = 0.f;
#pragma unroll
          for (int r = 0; r < 16; r++) {
            const int i = i0 + 8 * (r / 4) + 4 * h + r % 4;
            const float p = weight(x, r);
            all += i >= lo[x] && i <= hi[x] ? p : 0.f;
          }
          sum[x] += all;
        }
      }
    }
    if (++now == end) now = begin;
    stage = after;
    dma_wait();   // the stage after the next one has landed
    __syncthreads();
  }
  // A query that saw nothing is 0 in LDS, which makes NaN of keys that are infinite or NaN. So where a sum is NaN the wave forms it once more, straight from memory and from the queries that
  // saw something alone; it stays NaN if one of these sees such a key. (Looked at in the loop, in place of this, L cost all calls 1 to 6 %.)
  bool nan = false;
#pragma unroll
  for (int x = 0; x < NK; x++) nan = nan || sum[x] != sum[x];
  if (__builtin_amdgcn_ballot_w64(nan) != 0) {
    float anew[NK] = {};
    int at = lane;
    asm volatile("" : "+v"(at));   // what follows is formed here, and not held in registers through the loop above
    const int n = at & 31, h = at >> 5;
    int head = from / each;
    now = begin + from - head * each;
#pragma unroll 1
    for (int step = from; step < to; step++) {
      const char* const rows = w.q + b * w.qb + (int64_t)(g * w.group + head) * w.qh + 16 * h;
      const float* const L = w.lse + (row0 + head) * w.n_q;
#pragma unroll 1
      for (int i0 = now * ROWS; i0 < (now + 1) * ROWS; i0 += 32) {
        if (i0 > any_hi || i0 + 31 < any_lo) continue;
        const char* const row = rows + min(i0 + n, geo.n_q - 1) * w.qn;
#pragma unroll
        for (int x = 0; x < NK; x++) {
          const char* const keys = w.k + b * w.kb + g * w.kh + (int64_t)min(kw + 32 * x + n, geo.n_k - 1) * w.kn + 16 * h;
          f32x16_t scores = {0};
#pragma unroll
          for (int c = 0; c < STEPS; c++) {
            __builtin_amdgcn_sched_barrier(0);   // one load after the other: registers are the loop's above
            const u32x4_t a = *reinterpret_cast<const u32x4_t*>(row + 32 * c), of = *reinterpret_cast<const u32x4_t*>(keys + 32 * c);
            if constexpr (WIDE) {
#pragma unroll
              for (int e = 0; e < 4; e++) scores = __builtin_amdgcn_mfma_f32_32x32x2f32(number(a[e]), number(of[e]), scores, 0, 0, 0);
            } else {
              scores = mfma<F16>(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, of), scores);
            }
          }
#pragma unroll
          for (int r = 0; r < 16; r++) {
            __builtin_amdgcn_sched_barrier(0);
            const int i = i0 + 8 * (r / 4) + 4 * h + r % 4;
            const float l = L[min(i, geo.n_q - 1)], p = __builtin_amdgcn_exp2f(__builtin_fmaf(scores[r], w.scale_log2, -(l * kLog2e)));
            anew[x] += i >= lo[x] && i <= hi[x] && l != -INFINITY ? p : 0.f;
          }
        }
      }
      if (++now == end) now = begin, head++;
    }
#pragma unroll
    for (int x = 0; x < NK; x++) sum[x] = sum[x] != sum[x] ? anew[x] : sum[x];
  }
#pragma unroll
  for (int x = 0; x < NK; x++) {
    const float total = sum[x] + __shfl_xor(sum[x], 32);
    const int j = kw + 32 * x + n;
    if (h != 0 || j >= w.n_k) continue;
    if (w.pieces > 1) w.part[(((int64_t)piece * w.batch + b) * w.heads_k + g) * w.n_k + j] = total;
    else w.out[b * w.ob + g * w.oh + j] = total;
  }
}

template <int KEYS, int ROWS>
__global__ void __launch_bounds__(kThreads) add_pieces(Weigh w) {
  const int j = blockIdx.x * kThreads + threadIdx.x, g = blockIdx.y, b = blockIdx.z;
  if (j >= w.n_k) return;
  const Queries geo(w, w.lengths ? w.lengths[b] : 0);
  int begin, end;
  geo.template stages<ROWS>(j / KEYS * KEYS, KEYS, begin, end);
  const int pieces = pieces_of(w.group * (end - begin), w);
  const int64_t slice = (int64_t)w.heads_k * w.batch * w.n_k;
  const float* const part = w.part + ((int64_t)b * w.heads_k + g) * w.n_k + j;
  float sum = 0.f;
  for (int i = 0; i < pieces; i += 8) {   // eight on their way at a time, added in their order
    float of[8];
#pragma unroll
    for (int e = 0; e < 8; e++) of[e] = i + e < pieces ? part[(i + e) * slice] : 0.f;
#pragma unroll
    for (int e = 0; e < 8; e++) sum += of[e];
  }
  w.out[b * w.ob + g * w.oh + j] = sum;
}

// Pieces at most: a workspace of that many rows like the result's, whatever the length (131072 tokens, 4 heads of keys: 134 MB), and a grid of 2^23 workgroups
constexpr int64_t kPieces = 64;

// Keys of a workgroup and how the queries of one are cut
struct Plan {
  int nk, pieces, chunk;
  int64_t tiles;
  size_t bytes;
};

Plan plan_of(const fhog_key_weights_args* a) {
  Plan p;
  const int64_t slices = a->batch * a->heads_k, group = a->heads_q / a->heads_k, rows = rows_of((int)a->d * (a->dtype == FHOG_DTYPE_FP32 ? 4 : 2)), all = (a->n_q + rows - 1) / rows;
  const bool banded = a->causal != FHOG_MASK_NONE && a->window > 0 && a->window < a->n_q;
  // stages of a tile of keys in one head of queries: those of the tile with the most, and about those of all of them together
  const auto stages = [&](int64_t keys, int64_t& most, int64_t& total) {
    p.tiles = (a->n_k + keys - 1) / keys;
    const int64_t band = banded ? std::min(all, (a->window + keys) / rows + 2) : all;
    most = a->sinks > 0 ? all : band;
    const int64_t seen = a->causal == FHOG_MASK_NONE ? a->n_k : a->n_k - a->n_q / 2;   // keys of a query, about, without a window
    total = std::max(p.tiles, banded ? std::min(p.tiles, (a->n_q + a->window + keys - 1) / keys) * band : all * ((seen + keys - 1) / keys));
  };
  // 64 keys to a wave where there is work for it: half the reads of LDS, but fewer workgroups and coarser masks. us, 32 | 64 keys, bf16, heads x length: d = 128 causal 16 x 16384
  // 631 | 534, 16 x 8192 179 | 153, 32 x 4096 99 | 86, 64 x 2048 56.7 | 59.7, 16 x 3000 36.8 | 39.2, 8 x 512 10.8 | 18.1, window 2048 of 16 x 16384 175 | 159, window 1024 134 | 140;
  // d = 64 16 x 16384 386 | 354, 32 x 4096 67 | 62, 32 x 2048 25.5 | 33.4, window 2048 112 | 110; d = 32 16 x 16384 295 | 290, 16 x 8192 98 | 91
  int64_t most, total;
  p.nk = 2, stages(256, most, total);
  if (a->dtype == FHOG_DTYPE_FP32 || (banded && a->window < 2048) || total * group * slices < 12288) p.nk = 1, stages(128, most, total);
  // Eight pieces to a CU, as long as that leaves pieces worth their beginning, and short enough to even out the end of the launch. us, at most 16 | 24 | 32 | 48 | 64 stages, 32 keys to
  // a wave, 16 x 16384: d = 128 651 | 642 | 628 | 650 | 660, d = 64 399 | 394 | 391 | 410 | 418; four | eight pieces to a CU, 64 keys to a wave: 16 x 8192 172 | 154; at least 6 | 8 stages:
  // 16 x 3000 39.1 | 36.9, 8 x 512 12.0 | 10.8 (which then needs no second kernel); of a band, whose tiles have few, 3 | 5 | 8: fp16 48 x 1537, window 400, d = 64 23.0 | 22.3 | 26.1, bf16 64 x 1000,
  // window 128 17.9 | 17.5 | 21.0, 32 x 2048, window 512 24.0 | 23.0 | 23.6, d = 128 8 x 3000, window 1000 19.1 | 18.3 | 20.1, 16 x 4096, window 256 30.1 | 28.5 | 26.8; of fp32, whose stages take
  // eight times as long, 3 | 5 | 8: d = 64 16 x 2048 56.5 | 65.7 | 60.6, 8 x 4096 106 | 116 | 130, 8 x 512 14.5 | 19.7 | 24.2, 64 x 300 19.5 | 17.5 | 17.5, d = 128 32 x 1024 59 | 67 | 67, d = 32 4 x 3000 26 | 32 | 36
  const int64_t least = a->dtype == FHOG_DTYPE_FP32 ? 3 : p.nk == 1 && banded ? 5 : 8;
  int64_t chunk = std::min<int64_t>(32, std::max(least, (total * group * slices + 2047) / 2048));
  if (banded) {   // most tiles have as many stages: cut them evenly, not into full pieces and a short one
    const int64_t mine = group * std::min(all, (a->window + 128 * p.nk) / rows + 2), n = std::max<int64_t>(1, (mine + chunk / 2) / chunk);
    chunk = (mine + n - 1) / n;
  }
  chunk = std::max(chunk, (most * group + kPieces - 1) / kPieces);
  p.pieces = (int)std::max<int64_t>(1, (most * group + chunk - 1) / chunk);
  p.chunk = (int)std::max(chunk, p.pieces == 1 ? most * group : 0);
  p.bytes = p.pieces > 1 ? sizeof(float) * p.pieces * slices * a->n_k : 0;
  return p;
}

template <int DT, int D, int NK>
hipError_t launch_d(const Weigh& w, hipStream_t s) {
  constexpr int BYTES = D * (int)sizeof(typename Type<DT>::T), ROWS = rows_of(BYTES), STAGE = ROWS * BYTES + 256, LDS = kRing * STAGE;
  static_assert(LDS <= 64 << 10, "what a launch may ask for without further ado");
  hipLaunchKernelGGL((weigh<DT, D, NK>), dim3((unsigned)(w.tiles * w.pieces), (unsigned)w.heads_k, (unsigned)w.batch), dim3(kThreads), LDS, s, w);
  if (w.pieces > 1) hipLaunchKernelGGL((add_pieces<128 * NK, ROWS>), dim3((unsigned)((w.n_k + kThreads - 1) / kThreads), (unsigned)w.heads_k, (unsigned)w.batch), dim3(kThreads), 0, s, w);
  return hipGetLastError();
}
template <int DT, int NK>
hipError_t launch_t(const Weigh& w, int64_t d, hipStream_t s) {
  return d == 32 ? launch_d<DT, 32, NK>(w, s) : d == 64 ? launch_d<DT, 64, NK>(w, s) : launch_d<DT, 128, NK>(w, s);
}

}  // namespace

size_t key_weights_bytes(const fhog_key_weights_args* a) { return plan_of(a).bytes; }

hipError_t launch_key_weights(const fhog_key_weights_args* a, hipStream_t s) {
  const Plan p = plan_of(a);
  const int es = a->dtype == FHOG_DTYPE_FP32 ? 4 : 2;
  Weigh w;
  w.q = (const char*)a->q, w.k = (const char*)a->k, w.lse = a->lse, w.lengths = a->lengths, w.out = a->out, w.part = (float*)a->ws;
  w.qb = a->stride_qb * es, w.qh = a->stride_qh * es, w.qn = a->stride_qn * es, w.kb = a->stride_kb * es, w.kh = a->stride_kh * es, w.kn = a->stride_kn * es;
  w.ob = a->stride_ob, w.oh = a->stride_oh;
  w.batch = (int32_t)a->batch, w.heads_q = (int32_t)a->heads_q, w.heads_k = (int32_t)a->heads_k, w.group = w.heads_q / w.heads_k;
  w.n_q = (int32_t)a->n_q, w.n_k = (int32_t)a->n_k;
  w.causal = a->causal != FHOG_MASK_NONE, w.off = a->causal == FHOG_MASK_BOTTOM_RIGHT ? w.n_k - w.n_q : 0;
  w.window = a->window > 0 && a->window < w.n_q + (int64_t)w.n_k ? (int32_t)a->window : w.n_q + w.n_k;
  w.sinks = (int32_t)std::min<int64_t>(a->sinks, a->n_k);
  w.tiles = (int32_t)p.tiles, w.pieces = p.pieces, w.chunk = p.chunk, w.scale_log2 = a->scale * kLog2e;
  if (a->dtype == FHOG_DTYPE_FP32) return launch_t<FHOG_DTYPE_FP32, 1>(w, a->d, s);
  if (a->dtype == FHOG_DTYPE_FP16) return p.nk == 1 ? launch_t<FHOG_DTYPE_FP16, 1>(w, a->d, s) : launch_t<FHOG_DTYPE_FP16, 2>(w, a->d, s);
  return p.nk == 1 ? launch_t<FHOG_DTYPE_BF16, 1>(w, a->d, s) : launch_t<FHOG_DTYPE_BF16, 2>(w, a->d, s);
}

}  // namespace fhog
