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
// What bounds it: vector instructions, three of them and an exponential to 2 d flop of a pair.
#include <algorithm>

#include "fhog_bf16_util.h"

namespace fhog {
using namespace bf16k;
namespace {

constexpr int kThreads = 256, kRows = 64;   // queries of a stage

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

// Which queries see a key
struct Queries {
  int n_q, n_k, off, window, sinks, causal;
  __device__ __forceinline__ Queries(const Weigh& w, int b) : n_q(w.n_q), n_k(w.n_k), off(w.off), window(w.window), sinks(w.sinks), causal(w.causal) {
    if (w.lengths) {   // padding is as if it were not there
      n_k = max(0, min(w.lengths[b], n_k));
      n_q = max(0, min(n_k - off, n_q));
    }
  }
  __device__ __forceinline__ int first(int j) const { return causal ? max(0, j - off) : 0; }
  __device__ __forceinline__ int last(int j) const { return causal && j >= sinks && j - off < n_q - window ? j - off + window - 1 : n_q - 1; }
  // stages of 64 queries of which some see some of the keys [j, j + n)
  __device__ __forceinline__ void stages(int j, int n, int& begin, int& end) const {
    begin = end = 0;
    if (j >= n_k || n_q == 0) return;
    const int to = j < sinks ? n_q - 1 : last(min(j + n, n_k) - 1);
    begin = first(j) / kRows, end = max(begin, to / kRows + 1);
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

template <int DT, int D, int NK>
__global__ void __launch_bounds__(kThreads, 2) weigh(Weigh w) {
  constexpr bool WIDE = DT == FHOG_DTYPE_FP32, F16 = DT == FHOG_DTYPE_FP16;
  constexpr int BYTES = D * (int)sizeof(typename Type<DT>::T), CHUNKS = BYTES / 16, PER_LOAD = 64 / CHUNKS, LOADS = kRows / PER_LOAD / 4;
  constexpr int TILE = kRows * BYTES, STAGE = TILE + kRows * 4, KEYS = 128 * NK, STEPS = CHUNKS / 2;
  extern __shared__ __attribute__((aligned(16))) char smem[];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 31, h = lane >> 5;
  const int tile = blockIdx.x / w.pieces, piece = blockIdx.x - tile * w.pieces, g = blockIdx.y, b = blockIdx.z;
  const Queries geo(w, b);
  const int k0 = tile * KEYS, kw = k0 + 32 * NK * wave;
  int begin, end;
  geo.stages(k0, KEYS, begin, end);
  const int each = end - begin, steps = w.group * each, from = piece * w.chunk, to = min(steps, from + w.chunk);
  if (w.pieces > 1 && from >= steps) return;

  u32x4_t key[NK][STEPS];
  int lo[NK], hi[NK];                              // queries that see this lane's keys
  int whole_lo[NK], whole_hi[NK], any_lo[NK], any_hi[NK];   // ... all of the wave's 32, and some of them
#pragma unroll
  for (int x = 0; x < NK; x++) {
    const int j0 = kw + 32 * x, j = j0 + n, last = min(j0 + 31, geo.n_k - 1);
    const char* const row = w.k + b * w.kb + g * w.kh + (int64_t)max(0, min(j, geo.n_k - 1)) * w.kn + 16 * h;
#pragma unroll
    for (int s = 0; s < STEPS; s++) key[x][s] = geo.n_k > 0 ? *reinterpret_cast<const u32x4_t*>(row + 32 * s) : u32x4_t{0, 0, 0, 0};
    lo[x] = geo.first(j), hi[x] = j < geo.n_k ? geo.last(j) : -1;
    any_lo[x] = geo.first(j0), any_hi[x] = j0 >= geo.n_k ? -1 : j0 < geo.sinks ? geo.n_q - 1 : geo.last(last);
    whole_lo[x] = geo.first(j0 + 31), whole_hi[x] = j0 + 31 >= geo.n_k ? -1 : geo.last(max(j0, min(geo.sinks, j0 + 31)));
  }
  float sum[NK] = {};

  // staging: straight into LDS, 1 KiB to an instruction; rows past the end are copies of the last
  uint32_t off[LOADS];
  const auto offset = [&](int u, int valid) {
    const int r = (wave + 4 * u) * PER_LOAD + lane / CHUNKS, pc = lane % CHUNKS;
    return (uint32_t)(min(r, valid - 1) * (uint32_t)w.qn) + (uint32_t)((pc ^ swizzle<BYTES>(r)) << 4);
  };
#pragma unroll
  for (int u = 0; u < LOADS; u++) off[u] = offset(u, kRows);
  const uint32_t ring = lds_addr(smem);
  float stat = 0.f;
  int head = 0, t = begin;   // of the stage that is issued next
  if (each > 0) head = from / each, t = begin + from - head * each;
  const auto issue = [&](int slot) {
    const int64_t row = ((int64_t)b * w.heads_q + g * w.group + head);
    const char* const src = w.q + b * w.qb + (int64_t)(g * w.group + head) * w.qh + (int64_t)t * kRows * w.qn;
    const int valid = geo.n_q - t * kRows;
    if (tid < kRows) stat = *(global_f32_ptr)(w.lse + row * w.n_q + min(t * kRows + tid, geo.n_q - 1));
#pragma unroll
    for (int u = 0; u < LOADS; u++)
      Dma<64>::issue_one(ring + slot * STAGE + (wave + 4 * u) * 1024, valid >= kRows ? off[u] : offset(u, valid), (const __bf16*)src);
    if (++t == end) t = begin, head++;
  };
  // A query that saw nothing has no weights to give: exp(s - infinity)
  const auto publish = [&](int slot) {
    if (tid < kRows) reinterpret_cast<float*>(smem + slot * STAGE + TILE)[tid] = stat == -INFINITY ? INFINITY : stat * kLog2e;
  };
  if (from < to) {
    issue(0);
    wait_vm0();
    publish(0);
  }
  dma_wait();
  __syncthreads();
  int now = each > 0 ? begin + from % each : 0;
  for (int step = from; step < to; step++) {
    const int slot = (step - from) & 1;
    if (step + 1 < to) issue(slot ^ 1);
    const char* const stage = smem + slot * STAGE;
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const int i0 = now * kRows + 32 * u;
      bool dead = true;
#pragma unroll
      for (int x = 0; x < NK; x++) dead = dead && (i0 > any_hi[x] || i0 + 31 < any_lo[x]);
      if (dead) continue;   // no query of the tile sees a key of this wave
      f32x16_t s[NK];
#pragma unroll
      for (int x = 0; x < NK; x++) s[x] = f32x16_t{0};
#pragma unroll
      for (int c = 0; c < STEPS; c++) {
        const u32x4_t a = *reinterpret_cast<const u32x4_t*>(stage + (32 * u + n) * BYTES + (((2 * c + h) ^ swizzle<BYTES>(32 * u + n)) << 4));
#pragma unroll
        for (int x = 0; x < NK; x++) {
          if constexpr (WIDE) {
#pragma unroll
            for (int e = 0; e < 4; e++) s[x] = __builtin_amdgcn_mfma_f32_32x32x2f32(number(a[e]), number(key[x][c][e]), s[x], 0, 0, 0);
          } else {
            s[x] = mfma<F16>(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, key[x][c]), s[x]);
          }
        }
      }
      f32x4_t l[4];   // of the lane's 16 queries: 8 g + 4 h + e
#pragma unroll
      for (int e = 0; e < 4; e++) l[e] = *reinterpret_cast<const f32x4_t*>(stage + TILE + (32 * u + 8 * e + 4 * h) * 4);
#pragma unroll
      for (int x = 0; x < NK; x++) {
#pragma unroll
        for (int r = 0; r < 16; r++) s[x][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x][r], w.scale_log2, -l[r / 4][r % 4]));
        if (i0 < whole_lo[x] || i0 + 31 > whole_hi[x]) {   // the same for the wave
          keep_branch();
#pragma unroll
          for (int r = 0; r < 16; r++) {
            const int i = i0 + 8 * (r / 4) + 4 * h + r % 4;
            s[x][r] = i >= lo[x] && i <= hi[x] ? s[x][r] : 0.f;
          }
        }
        // in pairs: a sum over many tiles loses a rounding for each tile, not for each query
#pragma unroll
        for (int d = 8; d; d /= 2)
#pragma unroll
          for (int r = 0; r < d; r++) s[x][r] += s[x][r + d];
        sum[x] += s[x][0];
      }
    }
    if (++now == end) now = begin;
    if (step + 1 < to) {
      wait_vm0();
      publish(slot ^ 1);
    }
    dma_wait();
    __syncthreads();
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

template <int KEYS>
__global__ void __launch_bounds__(kThreads) add_pieces(Weigh w) {
  const int j = blockIdx.x * kThreads + threadIdx.x, g = blockIdx.y, b = blockIdx.z;
  if (j >= w.n_k) return;
  const Queries geo(w, b);
  int begin, end;
  geo.stages(j / KEYS * KEYS, KEYS, begin, end);
  const int pieces = (w.group * (end - begin) + w.chunk - 1) / w.chunk;
  const int64_t slice = (int64_t)w.heads_k * w.batch * w.n_k;
  const float* const part = w.part + ((int64_t)b * w.heads_k + g) * w.n_k + j;
  float sum = 0.f;
  for (int i = 0; i < pieces; i++) sum += part[i * slice];
  w.out[b * w.ob + g * w.oh + j] = sum;
}

// Keys of a workgroup and how the queries of one are cut
struct Plan {
  int nk, pieces, chunk;
  int64_t tiles;
  size_t bytes;
};

Plan plan_of(const fhog_key_weights_args* a) {
  Plan p;
  const int64_t slices = a->batch * a->heads_k, group = a->heads_q / a->heads_k;
  const int64_t window = a->causal != FHOG_MASK_NONE && a->window > 0 ? std::min(a->window, a->n_k) : a->n_k;
  p.nk = a->dtype == FHOG_DTYPE_FP32 ? 1 : 2;
  const int64_t keys = 128 * p.nk;
  p.tiles = (a->n_k + keys - 1) / keys;
  // stages of the tile of keys with the most, and about how many there are in all
  const int64_t all = (a->n_q + kRows - 1) / kRows, most = a->sinks > 0 || window >= a->n_k ? all : std::min(all, (window + keys) / kRows + 2);
  const int64_t mean = a->causal == FHOG_MASK_NONE ? all : std::min(most, (a->n_q < a->n_k ? all : all / 2 + 1));
  const int64_t total = mean * group * p.tiles * slices;
  const int64_t chunk = std::max<int64_t>(8, (total + 1535) / 1536);
  p.pieces = (int)std::max<int64_t>(1, (most * group + chunk - 1) / chunk);
  p.chunk = p.pieces == 1 ? (int)(most * group) : (int)chunk;
  p.bytes = p.pieces > 1 ? sizeof(float) * p.pieces * slices * a->n_k : 0;
  return p;
}

template <int DT, int D, int NK>
hipError_t launch_d(const Weigh& w, hipStream_t s) {
  constexpr int STAGE = kRows * D * (int)sizeof(typename Type<DT>::T) + kRows * 4;
  const hipError_t e = allow_dynamic_lds<weigh<DT, D, NK>>(2 * STAGE);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((weigh<DT, D, NK>), dim3((unsigned)(w.tiles * w.pieces), (unsigned)w.heads_k, (unsigned)w.batch), dim3(kThreads), 2 * STAGE, s, w);
  if (w.pieces > 1) hipLaunchKernelGGL((add_pieces<128 * NK>), dim3((unsigned)((w.n_k + kThreads - 1) / kThreads), (unsigned)w.heads_k, (unsigned)w.batch), dim3(kThreads), 0, s, w);
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
  switch (a->dtype) {
    case FHOG_DTYPE_FP32: return launch_t<FHOG_DTYPE_FP32, 1>(w, a->d, s);
    case FHOG_DTYPE_FP16: return launch_t<FHOG_DTYPE_FP16, 2>(w, a->d, s);
    default: return launch_t<FHOG_DTYPE_BF16, 2>(w, a->d, s);
  }
}

}  // namespace fhog
