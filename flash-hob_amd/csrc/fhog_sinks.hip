// What masks with sinks need beside the sweeps: the rows of dK, dV (dK2, dV2) of the sinks, and the join of forwards whose keys went to several workgroups.
//
// A key j < sinks is seen by every query from the diagonal on, n_q - j + ... of them, the other keys by a window's length: as rows of an ordinary
// workgroup of the key-tiled sweep the sinks would keep it busy n_q / window times as long as the others. The sweep therefore treats them as keys of the band, and
// a launch behind it computes their rows over ALL their queries and puts them in place: workgroups of 32 sinks with four waves on the same rows (of split
// products also 64 with two and 128 with one, as their terms fit the LDS), the queries dealt out over `parts` workgroups (rules::sink_parts), whose fp32 sums are added here in a fixed order and rounded once. Where they can, those workgroups
// come last in the launch of the key-tiled sweep itself (rules::sinks_ride).
#include "fhog_rules.h"
#include "fhog_split_util.h"

namespace fhog {
using namespace splitk;
namespace {

constexpr int kLanes = 8;   // lanes that share the parts of four columns

// Sums of four columns over the parts: lane i of LANES adds parts i, i + LANES, .., four loads at a time, and the lanes' sums are added pairwise, which gives all of
// them the same bits. With eight lanes up to 32 parts are one round trip to memory (one thread to all the parts of four columns took 5.0 us for 16
// parts, four lanes 4.2, eight 2.5); up to four parts are that for one lane, and eight lanes take 7.8 us for two parts of 4800 rows of 64.
template <int LANES>
__device__ __forceinline__ f32x4_t sum_parts(const float* from, int parts, int64_t stride, int lane) {
  f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
  for (int i = lane; i < parts; i += 4 * LANES) {
    f32x4_t x[4];
#pragma unroll
    for (int u = 0; u < 4; u++) {
      x[u] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      if (i + u * LANES < parts) x[u] = *reinterpret_cast<const f32x4_t*>(from + (i + u * LANES) * stride);
    }
    sum += (x[0] + x[1]) + (x[2] + x[3]);
  }
#pragma unroll
  for (int m = 1; m < LANES; m *= 2)
#pragma unroll
    for (int e = 0; e < 4; e++) sum[e] += __shfl_xor(sum[e], m);
  return sum;
}

template <typename T>
__device__ __forceinline__ void store4(T* to, f32x4_t x) {
  if constexpr (sizeof(T) == 4) *reinterpret_cast<f32x4_t*>(to) = x;
  else *reinterpret_cast<u32x2_t*>(to) = pack4<Terms<T>::F16>(x[0], x[1], x[2], x[3]);
}

// Rows [part][first | second][batch * sinks][d] -> the first `sinks` rows of two tensors; LANES threads to four columns of a row of one
struct SinkRows {
  const float* part;
  void *first, *second;
  int64_t stride_b, stride_n;
  int32_t parts, batch, sinks, d;
  float scale;   // of the first tensor
};
template <typename T, int LANES>
__global__ void __launch_bounds__(256) add_sink_parts(SinkRows a) {
  const int64_t idx = ((int64_t)blockIdx.x * 256 + threadIdx.x) / LANES, rows = (int64_t)a.batch * a.sinks;
  const int per_row = a.d / 4, lane = threadIdx.x % LANES;
  if (idx >= 2 * rows * per_row) return;   // LANES at a time
  const bool second = idx >= rows * per_row;
  const int64_t row = idx / per_row - (second ? rows : 0);
  const int col = (int)(idx % per_row) * 4;
  const f32x4_t sum = sum_parts<LANES>(a.part + ((second ? rows : 0) + row) * a.d + col, a.parts, 2 * rows * a.d, lane);
  if (lane == 0) store4((T*)(second ? a.second : a.first) + row / a.sinks * a.stride_b + row % a.sinks * a.stride_n + col, sum * (second ? 1.f : a.scale));
}

template <typename T>
hipError_t launch_add_t(const SinkRows& a, hipStream_t s) {
  const int64_t columns = (int64_t)a.batch * a.sinks * (a.d / 4) * 2;   // fours of them
  if (a.parts <= 4) hipLaunchKernelGGL((add_sink_parts<T, 1>), dim3((unsigned)((columns + 255) / 256)), dim3(256), 0, s, a);
  else hipLaunchKernelGGL((add_sink_parts<T, kLanes>), dim3((unsigned)((columns * kLanes + 255) / 256)), dim3(256), 0, s, a);
  return hipGetLastError();
}

hipError_t launch_add(const SinkRows& a, int dtype, hipStream_t s) {
  return dtype == FHOG_DTYPE_FP32 ? launch_add_t<float>(a, s) : dtype == FHOG_DTYPE_FP16 ? launch_add_t<_Float16>(a, s) : launch_add_t<__bf16>(a, s);
}

// O_i = sum_p 2^(m_p - M) acc_p / l, l = sum_p 2^(m_p - M) l_p, L_i = ln 2 (M + log2 l). A part that saw no key of the row has m = -inf, l = 0 and a row of
// zeros. kLanes threads to four columns of a row: lane i takes parts i, i + 8, .. and up to two of them, 16 parts in all, wait for no more than one round trip.
template <typename T>
__global__ void __launch_bounds__(256) join_forward(AttnParams p) {
  const PartialRows part(p);
  const int64_t idx = ((int64_t)blockIdx.x * 256 + threadIdx.x) / kLanes;
  const int per_row = p.d / 4, lane = threadIdx.x % kLanes;
  const int64_t row = idx / per_row;
  const int col = (int)(idx % per_row) * 4;
  if (row >= part.rows) return;   // kLanes at a time
  float top = -INFINITY, l = 0.f;
  f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
  for (int i = lane; i < p.n_split; i += 2 * kLanes) {   // on the maximum so far
    f32x2_t ml[2];
    f32x4_t x[2];
#pragma unroll
    for (int u = 0; u < 2; u++) {
      ml[u] = f32x2_t{-INFINITY, 0.f}, x[u] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      if (i + u * kLanes < p.n_split) ml[u] = part.stats(i + u * kLanes)[row], x[u] = *reinterpret_cast<const f32x4_t*>(part.row(i + u * kLanes, row) + col);
    }
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const float more = fmaxf(top, ml[u][0]), ref = more == -INFINITY ? 0.f : more;
      const float old = __builtin_amdgcn_exp2f(top - ref), w = __builtin_amdgcn_exp2f(ml[u][0] - ref);
      l = __builtin_fmaf(l, old, ml[u][1] * w);
      sum = sum * old + x[u] * w;
      top = more;
    }
  }
  float all = top;
#pragma unroll
  for (int m = 1; m < kLanes; m *= 2) all = fmaxf(all, __shfl_xor(all, m));
  const float mine = __builtin_amdgcn_exp2f(top - (all == -INFINITY ? 0.f : all));
  l *= mine, sum *= mine;
#pragma unroll
  for (int m = 1; m < kLanes; m *= 2) {
    l += __shfl_xor(l, m);
#pragma unroll
    for (int e = 0; e < 4; e++) sum[e] += __shfl_xor(sum[e], m);
  }
  if (lane != 0) return;
  const int64_t to = row / p.n_q * p.stride_qb + row % p.n_q * p.stride_qn + col;
  store4((T*)p.o + to, sum * (1.f / l));
  if (col == 0) p.lse[row] = (all + __builtin_amdgcn_logf(l)) * 0.6931471805599453f;   // v_log_f32 is log2
}

}  // namespace

hipError_t launch_join_forward(const AttnParams& p, int dtype, hipStream_t s) {
  const dim3 grid((unsigned)(((int64_t)p.batch * p.n_q * (p.d / 4) * kLanes + 255) / 256));
  switch (dtype) {
    case FHOG_DTYPE_FP32: hipLaunchKernelGGL(join_forward<float>, grid, dim3(256), 0, s, p); break;
    case FHOG_DTYPE_FP16: hipLaunchKernelGGL(join_forward<_Float16>, grid, dim3(256), 0, s, p); break;
    default: hipLaunchKernelGGL(join_forward<__bf16>, grid, dim3(256), 0, s, p);
  }
  return hipGetLastError();
}

hipError_t launch_sink_keys(const AttnParams& p, int dtype, bool swept, hipStream_t s) {
  AttnParams a = p;
  sinks_alone(a);
  const bool bit16 = dtype != FHOG_DTYPE_FP32 && p.d != 32;
  const hipError_t e = swept ? hipSuccess : bit16 ? launch_small_sink_bwd(a, s) : launch_attn_split_parts(a, dtype, true, s);
  if (e != hipSuccess || !a.part) return e;
  return launch_add({a.part, a.dk, a.dv, a.stride_kb, a.stride_kn, a.n_split, a.batch, a.n_k, a.d, a.scale}, dtype, s);
}

hipError_t launch_sink_keys(const Params& p, int dtype, bool split_products, bool swept, hipStream_t s) {
  Params a = p;
  sinks_alone(a);
  const hipError_t e = swept ? hipSuccess : split_products ? launch_split_sink_grads(a, dtype, s) : launch_small_sink_grads(a, s);
  if (e != hipSuccess || !a.part) return e;
  return launch_add({a.part, a.dk2, a.dv2, a.stride_kb, a.stride_kn, a.n_split, a.batch, a.n_k, a.d, a.scale}, dtype, s);
}

}  // namespace fhog
