// 16-bit kernels for launches too small to fill the GPU (d = 64 and 128): the default schedule of the double-backward in two
// launches (row statistics; dQ2, ddO beside dK2, dV2) and the first-order passes in two (forward; dQ beside dK, dV).
//
// A workgroup is 4 wave64, W = 4 or 2 of them on the SAME 32 stationary rows: each takes every W-th streamed tile, staged by itself
// in LDS of its own, so the sweep has no barrier, and the partial results of the W waves are added through LDS in their order.
// Against four waves on 128 rows that is W times the workgroups with a W-th of the tiles each; every tile is read from L2 once per 32
// rows instead of once per 128. The two tilings of a backward pass do not depend on each other and share a launch: dK and dV need
// d = rowsum(O dO) of the queries that they stream and take it from the staged rows themselves.
//
// What bounds them: latency. One round trip for the resident rows and the first tiles, the blocks of a wave one after the other (0.9 to
// 1.8 us each at d = 128, 0.5 to 1.1 at d = 64), an exchange through LDS and the stores. us, 128-row kernels -> here, bf16 causal:
//   2 x 256   d = 128: forward 11.3 -> 7.2, first backward 25.5 -> 11.6, double-backward 52.0 -> 22.7; d = 64: 8.7 -> 5.4, 20.2 -> 7.2, 39.3 -> 14.9
//   1 x 4096  d = 128: forward 93 -> 33, first backward 187 -> 76; d = 64: 74 -> 23, 160 -> 38
// One wave of such a workgroup keeps a SIMD to itself: at d = 128 the sweeps for dQ2, ddO and dK2, dV2 take 510 registers, which their
// two output accumulators and the resident rows do not leave room to halve.
#include "fhog_small.h"

namespace fhog {
using namespace bf16k;
using namespace smallk;
namespace {

// ---- double-backward: d, dd, b ------------------------------------------------------------------------------------------
template <int D>
constexpr int stats_lds = WAVES * n_buffers<D, 4> * 4 * TS * 2 * D;

template <bool F16, int D, int MASK, int W>
__global__ void __launch_bounds__(256, 2) small_stats(Params p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr int KK = D / 16, NC = D / 32, ROWS = TS * WAVES / W, NT = 4, TILE = TS * 2 * D, STAGE = NT * TILE, NBUF = n_buffers<D, NT>;
  int bh, tile;
  if (!decode_block<MASK>((p.n_q + ROWS - 1) / ROWS, p.batch, MASK != MASK_NONE, p.tile_major, bh, tile)) return;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int group = wave / W, ws = wave % W;   // row group of the wave, and which of its streamed tiles it takes
  const int n = lane & 31, h = lane >> 5;
  const int q0 = tile * ROWS + TS * group, qi = q0 + n, qr = min(qi, p.n_q - 1);   // queries past the end compute on a copy of the last row
  const int64_t qoff = (int64_t)bh * p.stride_qb, koff = (int64_t)bh * p.stride_kb, row = (int64_t)bh * p.n_q + qr;
  const __bf16* const src[NT] = {(const __bf16*)p.k + koff, (const __bf16*)p.ddk + koff, (const __bf16*)p.v + koff, (const __bf16*)p.ddv + koff};

  StreamKeys<MASK> geo(p.mask_off, p.window, p.n_k, p.sinks);
  int j_begin, j_end;
  geo.tile_range(q0, TS, j_begin, j_end);
  Dma<D, 1> dma;
  dma.init(p.stride_kn, 0, lane);
  const auto issue = [&](int j, uint32_t lds) { dma.template issue_all<NT>(lds, TILE, src, geo.offset(j, p.stride_kn), 0, geo.end(j) - geo.at(j)); };
  char* const ring = smem + wave * NBUF * STAGE;
  first_tiles<W, NBUF, STAGE>(j_begin + ws, j_end, ring, issue);

  bf16x8_t Qb[KK], ddQb[KK], dOb[KK], Ob[KK];
  load_resident<D>(Qb, (const __bf16*)p.q + qoff, p.stride_qn, qr, h);
  load_resident<D>(ddQb, (const __bf16*)p.ddq + qoff, p.stride_qn, qr, h);
  load_resident<D>(dOb, (const __bf16*)p.dO + qoff, p.stride_qn, qr, h);
  load_resident<D>(Ob, (const __bf16*)p.o + qoff, p.stride_qn, qr, h);
  const float l_log2 = p.lse[row] * kLog2e, c_scale_log2 = p.scale * kLog2e;
  float dsum = half_row_dot<F16, D>(Ob, dOb);   // d_i = sum_c O_ic dO_ic (fhog/triton_bwdbwd.py:580)
  dsum += __shfl_xor(dsum, 32);
  wait_vm0();

  int aoff[KK], troff[NC][2];
  lane_offsets<D>(lane, aoff, troff);
  float red[5] = {};   // sum P E, and over keys of P ddS, v ddS, v and P with v = P u
  f32x16_t none[NC];
  own_tiles<W, NBUF, STAGE, NT * Dma<D, 1>::IPT>(j_begin + ws, j_end, ring, issue, [&](const char* stage, int j) {
    const int k0 = geo.at(j);
    const bool masked = geo.partial(k0, q0, geo.sink(j));
    int lo = 0, hi = 0;
    if (masked) keep_branch(), geo.limits(k0, qi, h, lo, hi, geo.sink(j));
    q_block<F16, D, 5>(stage, aoff, troff, Qb, ddQb, dOb, masked, lo, hi, c_scale_log2, l_log2, p.scale, dsum, 0.f, 0.f, red[0], red[1],
                       red[2], red[3], red[4], none, none);
  });
  __syncthreads();   // the stages are no longer read
  float* const x = reinterpret_cast<float*>(smem) + lane;
#pragma unroll
  for (int i = 0; i < 5; i++) x[(wave * 5 + i) * 64] = red[i];
  __syncthreads();
  if (ws != 0) return;
#pragma unroll
  for (int i = 0; i < 5; i++) {
#pragma unroll
    for (int w = 1; w < W; w++) red[i] += x[((wave + w) * 5 + i) * 64];
    red[i] += __shfl_xor(red[i], 32);
  }
  if (h != 0 || qi >= p.n_q) return;
  const float dd = red[1] * p.scale;
  p.ws_d[row] = dsum;
  p.ws_dd[row] = dd;
  p.ws_b[row] = __builtin_fmaf(-dd, __builtin_fmaf(dsum, red[4], red[3]), __builtin_fmaf(p.scale, red[2], red[0]));
}

// ---- double-backward: dQ2, ddO (workgroups [0, q_blocks)) and dK2, dV2 (the others) -----------------------------------------
template <bool F16, int D, int MASK, int W>
__device__ __forceinline__ void grads_q(const Params& p, char* smem) {
  constexpr int KK = D / 16, NC = D / 32, ROWS = TS * WAVES / W, NT = 4, TILE = TS * 2 * D, STAGE = NT * TILE, NBUF = n_buffers<D, NT>;
  int bh, tile;
  if (!decode_block<MASK>((p.n_q + ROWS - 1) / ROWS, p.batch, MASK != MASK_NONE, p.tile_major, bh, tile)) return;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int group = wave / W, ws = wave % W;   // row group of the wave, and which of its streamed tiles it takes
  const int n = lane & 31, h = lane >> 5;
  const int q0 = tile * ROWS + TS * group, qi = q0 + n, qr = min(qi, p.n_q - 1);
  const int64_t qoff = (int64_t)bh * p.stride_qb, koff = (int64_t)bh * p.stride_kb, row = (int64_t)bh * p.n_q + qr;
  const __bf16* const src[NT] = {(const __bf16*)p.k + koff, (const __bf16*)p.ddk + koff, (const __bf16*)p.v + koff, (const __bf16*)p.ddv + koff};

  StreamKeys<MASK> geo(p.mask_off, p.window, p.n_k, p.sinks);
  int j_begin, j_end;
  geo.tile_range(q0, TS, j_begin, j_end);
  Dma<D, 1> dma;
  dma.init(p.stride_kn, 0, lane);
  const auto issue = [&](int j, uint32_t lds) { dma.template issue_all<NT>(lds, TILE, src, geo.offset(j, p.stride_kn), 0, geo.end(j) - geo.at(j)); };
  char* const ring = smem + wave * NBUF * STAGE;
  first_tiles<W, NBUF, STAGE>(j_begin + ws, j_end, ring, issue);

  bf16x8_t Qb[KK], ddQb[KK], dOb[KK];
  load_resident<D>(Qb, (const __bf16*)p.q + qoff, p.stride_qn, qr, h);
  load_resident<D>(ddQb, (const __bf16*)p.ddq + qoff, p.stride_qn, qr, h);
  load_resident<D>(dOb, (const __bf16*)p.dO + qoff, p.stride_qn, qr, h);
  const float l_log2 = p.lse[row] * kLog2e, c_scale_log2 = p.scale * kLog2e;
  const float dsum = p.ws_d[row], dd = p.ws_dd[row], kc = __builtin_fmaf(dd, dsum, p.ws_b[row]);
  wait_vm0();

  int aoff[KK], troff[NC][2];
  lane_offsets<D>(lane, aoff, troff);
  f32x16_t acc_dq[NC], acc_ddo[NC];
#pragma unroll
  for (int cb = 0; cb < NC; cb++) acc_dq[cb] = f32x16_t{0}, acc_ddo[cb] = f32x16_t{0};
  float none[5] = {};
  own_tiles<W, NBUF, STAGE, NT * Dma<D, 1>::IPT>(j_begin + ws, j_end, ring, issue, [&](const char* stage, int j) {
    const int k0 = geo.at(j);
    const bool masked = geo.partial(k0, q0, geo.sink(j));
    int lo = 0, hi = 0;
    if (masked) keep_branch(), geo.limits(k0, qi, h, lo, hi, geo.sink(j));
    q_block<F16, D, 3>(stage, aoff, troff, Qb, ddQb, dOb, masked, lo, hi, c_scale_log2, l_log2, p.scale, dsum, dd, kc, none[0], none[1],
                       none[2], none[3], none[4], acc_dq, acc_ddo);
  });
  __syncthreads();   // the stages are no longer read
  f32x16_t acc[2 * NC];
#pragma unroll
  for (int cb = 0; cb < NC; cb++) acc[cb] = acc_dq[cb], acc[NC + cb] = acc_ddo[cb];
  f32x4_t out[2 * NC][4 / W];
  add_waves<W>(acc, smem, group, ws, lane, out);
  if (qi >= p.n_q) return;
  store_part<F16, NC, 4 / W>((uint16_t*)p.dq2 + qoff + (int64_t)qi * p.stride_qn, out, p.scale, ws, h);
  store_part<F16, NC, 4 / W>((uint16_t*)p.ddo + qoff + (int64_t)qi * p.stride_qn, out + NC, 1.f, ws, h);
}

template <int D>
constexpr int grads_lds = max_of(WAVES * n_buffers<D, 4> * max_of(4 * TS * 2 * D, grads_k_stage<D>), add_waves_bytes(2 * D / 32));

// MASK_SINK, small_bwd too: behind both come the workgroups that sum up the rows of the sinks (fhog_sinks.hip)
template <bool F16, int D, int MASK, int W>
__global__ void __launch_bounds__(256, D == 64 ? 2 : 1) small_grads(Params p, int q_blocks) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  if constexpr (MASK == MASK_SINK) {
    const int id = sink_workgroup(p.part_s ? p.sinks : 0, p.batch * p.n_split_s);
    if (id >= 0) {
      sinks_alone(p);
      return grads_k<F16, D, MASK_BAND, WAVES, true>(p, smem, id);
    }
  }
  if ((int)blockIdx.x < q_blocks) grads_q<F16, D, MASK, W>(p, smem);
  else grads_k<F16, D, MASK, W>(p, smem, (int)blockIdx.x - q_blocks);
}

// ---- first order: forward ---------------------------------------------------------------------------------------------------
template <int D>
constexpr int fwd_lds = max_of(WAVES * n_buffers<D, 2> * 2 * TS * 2 * D, add_waves_bytes(D / 32) + WAVES * 2 * 64 * 4);

// PARTS: the streamed keys are dealt out over n_split workgroups, which leave fp32 rows and their maximum and sum in p.part (PartialRows) where there are several
template <bool F16, int D, int MASK, int W, bool PARTS = false>
__global__ void __launch_bounds__(256, 2) small_fwd(AttnParams p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr int KK = D / 16, NC = D / 32, ROWS = TS * WAVES / W, NT = 2, TILE = TS * 2 * D, STAGE = NT * TILE, NBUF = n_buffers<D, NT>;
  int bh, tile;
  if (!decode_block<MASK>((p.n_q + ROWS - 1) / ROWS, p.batch * (PARTS ? p.n_split : 1), MASK != MASK_NONE, MASK != MASK_NONE, bh, tile)) return;
  const int part = PARTS ? bh % p.n_split : 0;
  if (PARTS) bh /= p.n_split;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int group = wave / W, ws = wave % W;   // row group of the wave, and which of its streamed tiles it takes
  const int n = lane & 31, h = lane >> 5;
  const int q0 = tile * ROWS + TS * group, qi = q0 + n, qr = min(qi, p.n_q - 1);
  const int64_t qoff = (int64_t)bh * p.stride_qb, koff = (int64_t)bh * p.stride_kb;
  const __bf16* const src[NT] = {(const __bf16*)p.k + koff, (const __bf16*)p.v + koff};
  StreamKeys<MASK> geo(p.mask_off, p.window, p.n_k, p.sinks);
  int j_begin, j_end;
  geo.tile_range(q0, TS, j_begin, j_end);
  if (PARTS) split_range(part, p.n_split, j_begin, j_end);
  Dma<D, 1> dma;
  dma.init(p.stride_kn, 0, lane);
  const auto issue = [&](int j, uint32_t lds) { dma.template issue_all<NT>(lds, TILE, src, geo.offset(j, p.stride_kn), 0, geo.end(j) - geo.at(j)); };
  char* const ring = smem + wave * NBUF * STAGE;
  first_tiles<W, NBUF, STAGE>(j_begin + ws, j_end, ring, issue);
  bf16x8_t Qb[KK];
  load_resident<D>(Qb, (const __bf16*)p.q + qoff, p.stride_qn, qr, h);
  wait_vm0();
  const float c_scale_log2 = p.scale * kLog2e;
  int aoff[KK], troff[NC][2];
  lane_offsets<D>(lane, aoff, troff);
  float m = -INFINITY, l = 0.f;
  f32x16_t acc[1][NC];
#pragma unroll
  for (int cb = 0; cb < NC; cb++) acc[0][cb] = f32x16_t{0};
  own_tiles<W, NBUF, STAGE, NT * Dma<D, 1>::IPT>(j_begin + ws, j_end, ring, issue, [&](const char* stage, int j) {
    const int k0 = geo.at(j);
    const bool masked = geo.partial(k0, q0, geo.sink(j));
    int lo = 0, hi = 0;
    if (masked) keep_branch(), geo.limits(k0, qi, h, lo, hi, geo.sink(j));
    fwd_block<F16, D>(stage, aoff, troff, Qb, masked, lo, hi, c_scale_log2, m, l, acc);
  });
  __syncthreads();
  // the waves' rows on one maximum; a wave that has seen no key of a row has l = 0 and m = -inf there
  float* const ml = reinterpret_cast<float*>(smem + add_waves_bytes(NC)) + lane;
  ml[wave * 2 * 64] = m, ml[(wave * 2 + 1) * 64] = l;
  __syncthreads();
  float m_all = -INFINITY, l_all = 0.f;
#pragma unroll
  for (int w = group * W; w < group * W + W; w++) m_all = fmaxf(m_all, ml[w * 2 * 64]);
  const float m_ref = m_all == -INFINITY ? 0.f : m_all;
#pragma unroll
  for (int w = group * W; w < group * W + W; w++) l_all = __builtin_fmaf(ml[(w * 2 + 1) * 64], __builtin_amdgcn_exp2f(ml[w * 2 * 64] - m_ref), l_all);
  const float mine = __builtin_amdgcn_exp2f(m - m_ref);
#pragma unroll
  for (int cb = 0; cb < NC; cb++)
#pragma unroll
    for (int r = 0; r < 16; r++) acc[0][cb][r] *= mine;
  f32x4_t out[NC][4 / W];
  add_waves<W>(acc[0], smem, group, ws, lane, out);
  l_all += __shfl_xor(l_all, 32);
  if (qi >= p.n_q) return;
  if (PARTS && p.n_split > 1) {
    const PartialRows rows(p);
    store_partial<NC, 4 / W>(rows.row(part, (int64_t)bh * p.n_q + qi), out, ws, h);
    if (ws == 0 && h == 0) rows.stats(part)[(int64_t)bh * p.n_q + qi] = f32x2_t{m_all, l_all};
    return;
  }
  store_part<F16, NC, 4 / W>((uint16_t*)p.o + qoff + (int64_t)qi * p.stride_qn, out, 1.f / l_all, ws, h);
  if (ws == 0 && h == 0) p.lse[(int64_t)bh * p.n_q + qi] = (m_all + __builtin_amdgcn_logf(l_all)) * 0.6931471805599453f;   // v_log_f32 is log2
}

// ---- first order: dQ (workgroups [0, q_blocks)) and dK, dV (the others) ---------------------------------------------------------
template <bool F16, int D, int MASK, int W>
__device__ __forceinline__ void bwd_q(const AttnParams& p, char* smem) {
  constexpr int KK = D / 16, NC = D / 32, ROWS = TS * WAVES / W, NT = 2, TILE = TS * 2 * D, STAGE = NT * TILE, NBUF = n_buffers<D, NT>;
  int bh, tile;
  if (!decode_block<MASK>((p.n_q + ROWS - 1) / ROWS, p.batch, MASK != MASK_NONE, p.tile_major_q != 0, bh, tile)) return;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int group = wave / W, ws = wave % W;   // row group of the wave, and which of its streamed tiles it takes
  const int n = lane & 31, h = lane >> 5;
  const int q0 = tile * ROWS + TS * group, qi = q0 + n, qr = min(qi, p.n_q - 1);
  const int64_t qoff = (int64_t)bh * p.stride_qb, koff = (int64_t)bh * p.stride_kb, row = (int64_t)bh * p.n_q + qr;
  const __bf16* const src[NT] = {(const __bf16*)p.k + koff, (const __bf16*)p.v + koff};
  StreamKeys<MASK> geo(p.mask_off, p.window, p.n_k, p.sinks);
  int j_begin, j_end;
  geo.tile_range(q0, TS, j_begin, j_end);
  Dma<D, 1> dma;
  dma.init(p.stride_kn, 0, lane);
  const auto issue = [&](int j, uint32_t lds) { dma.template issue_all<NT>(lds, TILE, src, geo.offset(j, p.stride_kn), 0, geo.end(j) - geo.at(j)); };
  char* const ring = smem + wave * NBUF * STAGE;
  first_tiles<W, NBUF, STAGE>(j_begin + ws, j_end, ring, issue);
  bf16x8_t Qb[KK], dOb[KK], Ob[KK];
  load_resident<D>(Qb, (const __bf16*)p.q + qoff, p.stride_qn, qr, h);
  load_resident<D>(dOb, (const __bf16*)p.dO + qoff, p.stride_qn, qr, h);
  load_resident<D>(Ob, (const __bf16*)p.o + qoff, p.stride_qn, qr, h);
  const float l_log2 = p.lse[row] * kLog2e, c_scale_log2 = p.scale * kLog2e;
  float dsum = half_row_dot<F16, D>(Ob, dOb);
  dsum += __shfl_xor(dsum, 32);
  wait_vm0();
  int aoff[KK], troff[NC][2];
  lane_offsets<D>(lane, aoff, troff);
  f32x16_t acc[1][NC];
#pragma unroll
  for (int cb = 0; cb < NC; cb++) acc[0][cb] = f32x16_t{0};
  own_tiles<W, NBUF, STAGE, NT * Dma<D, 1>::IPT>(j_begin + ws, j_end, ring, issue, [&](const char* stage, int j) {
    const int k0 = geo.at(j);
    const bool masked = geo.partial(k0, q0, geo.sink(j));
    int lo = 0, hi = 0;
    if (masked) keep_branch(), geo.limits(k0, qi, h, lo, hi, geo.sink(j));
    bwd_q_block<F16, D>(stage, aoff, troff, Qb, dOb, masked, lo, hi, c_scale_log2, l_log2, dsum, acc);
  });
  __syncthreads();
  f32x4_t out[NC][4 / W];
  add_waves<W>(acc[0], smem, group, ws, lane, out);
  if (qi >= p.n_q) return;
  store_part<F16, NC, 4 / W>((uint16_t*)p.dq + qoff + (int64_t)qi * p.stride_qn, out, p.scale, ws, h);
  if (ws == 0 && h == 0) p.ws_d[row] = dsum;
}

template <int D>
constexpr int bwd_lds = max_of(max_of(WAVES * n_buffers<D, 2> * 2 * TS * 2 * D, WAVES * bwd_k_buffers<D, true> * bwd_k_stage<D, true>), add_waves_bytes(2 * D / 32));

template <bool F16, int D, int MASK, int W>
__global__ void __launch_bounds__(256, D == 64 ? 2 : 1) small_bwd(AttnParams p, int q_blocks) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  if constexpr (MASK == MASK_SINK) {
    const int id = sink_workgroup(p.part ? p.sinks : 0, p.batch * p.n_split);
    if (id >= 0) {
      sinks_alone(p);
      return bwd_k<F16, D, MASK_BAND, WAVES, true>(p, smem, id);
    }
  }
  if ((int)blockIdx.x < q_blocks) bwd_q<F16, D, MASK, W>(p, smem);
  else bwd_k<F16, D, MASK, W>(p, smem, (int)blockIdx.x - q_blocks);
}

// The rows of dK, dV (dK2, dV2) of the sinks, over all queries that see them: p.n_k is the number of sinks there, and there is no window
template <bool F16, int D>
__global__ void __launch_bounds__(256, D == 64 ? 2 : 1) sink_bwd(AttnParams p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  bwd_k<F16, D, MASK_BAND, WAVES, true, false>(p, smem, blockIdx.x);
}
template <bool F16, int D>
__global__ void __launch_bounds__(256, D == 64 ? 2 : 1) sink_grads(Params p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  grads_k<F16, D, MASK_BAND, WAVES, true>(p, smem, blockIdx.x);
}

template <auto Kernel, typename... Args>
hipError_t launch(unsigned grid, int lds, hipStream_t s, Args... args) {
  const hipError_t e = allow_dynamic_lds<Kernel>(lds);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(Kernel, dim3(grid), dim3(64 * WAVES), lds, s, args...);
  return hipGetLastError();
}

template <int W>
unsigned blocks(int rows, int batch) { return grid_blocks((rows + TS * WAVES / W - 1) / (TS * WAVES / W), batch); }

template <bool F16, int D, int MASK, int W>
hipError_t bwdbwd_d(const Params& p, hipStream_t s) {
  static_assert(stats_lds<D> <= 160 * 1024 && grads_lds<D> <= 160 * 1024, "the stages of four waves have to fit the LDS");
  const unsigned gq = blocks<W>(p.n_q, p.batch), gk = blocks<W>(p.n_k, p.batch), gs = MASK == MASK_SINK && p.part_s ? blocks<WAVES>(p.sinks, p.batch * p.n_split_s) : 0;
  const hipError_t e = launch<small_stats<F16, D, MASK, W>>(gq, stats_lds<D>, s, p);
  return e != hipSuccess ? e : launch<small_grads<F16, D, MASK, W>>(gq + gk + gs, grads_lds<D>, s, p, (int)gq);
}

template <bool F16, int D, int MASK, int W>
hipError_t attn_d(const AttnParams& p, bool backward, hipStream_t s) {
  static_assert(fwd_lds<D> <= 160 * 1024 && bwd_lds<D> <= 160 * 1024, "the stages of four waves have to fit the LDS");
  const unsigned gq = blocks<W>(p.n_q, p.batch), gk = blocks<W>(p.n_k, p.batch), gs = MASK == MASK_SINK && p.part ? blocks<WAVES>(p.sinks, p.batch * p.n_split) : 0;
  if (!backward) return launch<small_fwd<F16, D, MASK, W>>(gq, fwd_lds<D>, s, p);
  return launch<small_bwd<F16, D, MASK, W>>(gq + gk + gs, bwd_lds<D>, s, p, (int)gq);
}

template <bool F16, int D>
hipError_t fwd_parts_d(const AttnParams& p, hipStream_t s) { return launch<small_fwd<F16, D, MASK_SINK, WAVES, true>>(blocks<WAVES>(p.n_q, p.batch * p.n_split), fwd_lds<D>, s, p); }
template <bool F16, int D>
hipError_t sink_bwd_d(const AttnParams& p, hipStream_t s) { return launch<sink_bwd<F16, D>>(blocks<WAVES>(p.n_k, p.batch * p.n_split), sink_bwd_lds<D>, s, p); }
template <bool F16, int D>
hipError_t sink_grads_d(const Params& p, hipStream_t s) { return launch<sink_grads<F16, D>>(blocks<WAVES>(p.n_k, p.batch * p.n_split), grads_lds<D>, s, p); }

}  // namespace

#define FHOG_SMALL_W(FN, F, DD, M, ...) (waves == 4 ? FN<F, DD, M, 4>(__VA_ARGS__) : FN<F, DD, M, 2>(__VA_ARGS__))
#define FHOG_SMALL(FN, F, DD, ...)                                          \
  (mask == MASK_NONE ? FHOG_SMALL_W(FN, F, DD, MASK_NONE, __VA_ARGS__)      \
                     : mask == MASK_CAUSAL ? FHOG_SMALL_W(FN, F, DD, MASK_CAUSAL, __VA_ARGS__) \
                     : mask == MASK_SINK ? FHOG_SMALL_W(FN, F, DD, MASK_SINK, __VA_ARGS__) : FHOG_SMALL_W(FN, F, DD, MASK_BAND, __VA_ARGS__))

hipError_t launch_small_bwdbwd(const Params& p, int waves, hipStream_t s) {
  const int mask = mask_mode(p);
  if (p.f16) return p.d == 128 ? FHOG_SMALL(bwdbwd_d, true, 128, p, s) : FHOG_SMALL(bwdbwd_d, true, 64, p, s);
  return p.d == 128 ? FHOG_SMALL(bwdbwd_d, false, 128, p, s) : FHOG_SMALL(bwdbwd_d, false, 64, p, s);
}

hipError_t launch_small_attn(const AttnParams& p, bool backward, int waves, hipStream_t s) {
  const int mask = mask_mode(p);
  if (p.f16) return p.d == 128 ? FHOG_SMALL(attn_d, true, 128, p, backward, s) : FHOG_SMALL(attn_d, true, 64, p, backward, s);
  return p.d == 128 ? FHOG_SMALL(attn_d, false, 128, p, backward, s) : FHOG_SMALL(attn_d, false, 64, p, backward, s);
}
#undef FHOG_SMALL
#undef FHOG_SMALL_W

hipError_t launch_small_fwd_parts(const AttnParams& p, hipStream_t s) {
  if (p.f16) return p.d == 128 ? fwd_parts_d<true, 128>(p, s) : fwd_parts_d<true, 64>(p, s);
  return p.d == 128 ? fwd_parts_d<false, 128>(p, s) : fwd_parts_d<false, 64>(p, s);
}

hipError_t launch_small_sink_bwd(const AttnParams& p, hipStream_t s) {
  if (p.f16) return p.d == 128 ? sink_bwd_d<true, 128>(p, s) : sink_bwd_d<true, 64>(p, s);
  return p.d == 128 ? sink_bwd_d<false, 128>(p, s) : sink_bwd_d<false, 64>(p, s);
}

hipError_t launch_small_sink_grads(const Params& p, hipStream_t s) {
  if (p.f16) return p.d == 128 ? sink_grads_d<true, 128>(p, s) : sink_grads_d<true, 64>(p, s);
  return p.d == 128 ? sink_grads_d<false, 128>(p, s) : sink_grads_d<false, 64>(p, s);
}

}  // namespace fhog
