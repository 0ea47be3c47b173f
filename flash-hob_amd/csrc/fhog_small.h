// Four wave64 on the same 32 stationary rows (gfx950): staging, exchange and the key-tiled sweeps of the 16-bit kernels for small launches (fhog_small.hip), which the rows
// of the sinks (fhog_attn.hip, fhog_bf16.hip) run on as well.
#pragma once
#include "fhog_bf16_blocks.h"

namespace fhog {
namespace smallk {
using namespace bf16k;

constexpr int WAVES = 4;

__device__ __forceinline__ void lds_reads_done() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// 64 lanes x 4 bytes from the lanes' addresses to 256 contiguous bytes of LDS; counted like the loads of Dma
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void stage_words(uint32_t lds, const float* src) {
  const uint32_t m0 = __builtin_amdgcn_readfirstlane(lds);
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dword %1, off\n\t" ::"s"(m0), "v"(src) : "memory", "m0");
}
#pragma clang diagnostic pop

// The streamed tiles of one wave: every W-th one of [begin, end), in a ring of NBUF stages of its own.
// issue(t, lds): requests tile t into the stage at LDS address lds, COUNT loads.
template <int W, int NBUF, int STAGE, int COUNT, typename Issue, typename Block>
__device__ __forceinline__ void own_tiles(int begin, int end, char* ring, const Issue& issue, const Block& block) {
  const uint32_t lds = lds_addr(ring);
  int t = begin;
  bool landed = true;   // first_tiles' requests: every caller has waited for them
  for (int slot = 0; t < end; t += W) {
    if (!landed) {
      // what may still travel is the tile behind this one
      if (NBUF == 2 && t + W < end) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(COUNT) : "memory");
      else dma_wait();
    }
    block(ring + slot * STAGE, t);
    lds_reads_done();   // the stage is overwritten next
    if (t + NBUF * W < end) issue(t + NBUF * W, lds + slot * STAGE);
    landed = landed && NBUF == 2 && t == begin;   // the second tile was requested beside the first
    if (NBUF == 2) slot ^= 1;
  }
}
template <int W, int NBUF, int STAGE, typename Issue>
__device__ __forceinline__ void first_tiles(int begin, int end, char* ring, const Issue& issue) {
  if (begin < end) issue(begin, lds_addr(ring));
  if (NBUF == 2 && begin + W < end) issue(begin + W, lds_addr(ring) + STAGE);
}

// Adds the accumulators of the W waves of a row group: its wave ws returns registers 16/W ws .. of every one, four at a time, summed in
// the order of the waves.
template <int W, int NV>
__device__ __forceinline__ void add_waves(const f32x16_t (&acc)[NV], char* smem, int group, int ws, int lane, f32x4_t (&out)[NV][4 / W]) {
  constexpr int G = 4 / W;   // groups of four registers that a wave returns
  f32x4_t* const x = reinterpret_cast<f32x4_t*>(smem) + group * (W * W * NV * G * 64) + lane;
#pragma unroll
  for (int v = 0; v < NV; v++)
#pragma unroll
    for (int g = 0; g < 4; g++)
      x[(((g / G * W + ws) * NV + v) * G + g % G) * 64] = f32x4_t{acc[v][4 * g], acc[v][4 * g + 1], acc[v][4 * g + 2], acc[v][4 * g + 3]};
  __syncthreads();
#pragma unroll
  for (int v = 0; v < NV; v++)
#pragma unroll
    for (int g = 0; g < G; g++) {
      out[v][g] = x[((ws * W * NV + v) * G + g) * 64];
#pragma unroll
      for (int w = 1; w < W; w++) out[v][g] += x[(((ws * W + w) * NV + v) * G + g) * 64];
    }
}
constexpr int add_waves_bytes(int nv) { return 16 * nv * 64 * 16; }

// The columns of a row whose registers add_waves returned: 32 cb + 8 (G ws + g) + 4 h .. + 3, from out[cb][g]
template <bool F16, int NC, int G>
__device__ __forceinline__ void store_part(uint16_t* row, const f32x4_t (*out)[G], float scale, int ws, int h) {
#pragma unroll
  for (int cb = 0; cb < NC; cb++)
#pragma unroll
    for (int g = 0; g < G; g++)
      *reinterpret_cast<u32x2_t*>(row + 32 * cb + 8 * (G * ws + g) + 4 * h) =
          pack4<F16>(out[cb][g][0] * scale, out[cb][g][1] * scale, out[cb][g][2] * scale, out[cb][g][3] * scale);
}

// ... as fp32 numbers
template <int NC, int G>
__device__ __forceinline__ void store_partial(float* row, const f32x4_t (*out)[G], int ws, int h) {
#pragma unroll
  for (int cb = 0; cb < NC; cb++)
#pragma unroll
    for (int g = 0; g < G; g++) *reinterpret_cast<f32x4_t*>(row + 32 * cb + 8 * (G * ws + g) + 4 * h) = out[cb][g];
}

template <int D>
__device__ __forceinline__ void lane_offsets(int lane, int (&aoff)[D / 16], int (&troff)[D / 32][2]) {
#pragma unroll
  for (int kk = 0; kk < D / 16; kk++) aoff[kk] = tile_off<D>(lane & 31, 2 * kk + (lane >> 5));
#pragma unroll
  for (int cb = 0; cb < D / 32; cb++) troff[cb][0] = tr_lane_off_acc<D>(cb, 0, lane), troff[cb][1] = tr_lane_off_acc<D>(cb, 1, lane);
}

template <bool F16, int D>
__device__ __forceinline__ float half_row_dot(const bf16x8_t (&a)[D / 16], const bf16x8_t (&b)[D / 16]) {
  float sum = 0.f;
#pragma unroll
  for (int kk = 0; kk < D / 16; kk++)
#pragma unroll
    for (int e = 0; e < 8; e++) sum = __builtin_fmaf(to_f32<F16>(a[kk][e]), to_f32<F16>(b[kk][e]), sum);
  return sum;
}

// Stages of a wave's ring: as many as let four waves stay within the 160 KiB of a CU
template <int D, int NT>
constexpr int n_buffers = 2 * WAVES * NT * TS * 2 * D <= 128 * 1024 ? 2 : 1;

constexpr int max_of(int a, int b) { return a > b ? a : b; }
// ---- double-backward: dK2, dV2 --------------------------------------------------------------------------------------------
template <int D>
constexpr int grads_k_stage = 3 * TS * 2 * D + 4 * TS * 4;   // Q, ddQ, dO tiles and the statistics of their rows

// PARTS: the streamed queries are dealt out over n_split workgroups, whose partial results are fp32 rows [part][dK2 | dV2][batch * n_k][D] in p.part
template <bool F16, int D, int MASK, int W, bool PARTS = false, int NBUF = n_buffers<D, 4>>
__device__ __forceinline__ void grads_k(const Params& p, char* smem, int id) {
  constexpr int KK = D / 16, NC = D / 32, ROWS = TS * WAVES / W, NT = 3, TILE = TS * 2 * D, STAGE = grads_k_stage<D>;
  int bh, tile;
  if (!decode_block<MASK>((p.n_k + ROWS - 1) / ROWS, p.batch * (PARTS ? p.n_split : 1), false, p.tile_major, bh, tile, false, id)) return;
  const int part = PARTS ? bh % p.n_split : 0;
  if (PARTS) bh /= p.n_split;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int group = wave / W, ws = wave % W;
  const int n = lane & 31, h = lane >> 5;
  const int k0 = tile * ROWS + TS * group, kj = k0 + n, kr = min(kj, p.n_k - 1);   // keys past the end compute on a copy of the last row
  const int64_t qoff = (int64_t)bh * p.stride_qb, koff = (int64_t)bh * p.stride_kb, srow = (int64_t)bh * p.n_q;
  const __bf16* const src[NT] = {(const __bf16*)p.q + qoff, (const __bf16*)p.ddq + qoff, (const __bf16*)p.dO + qoff};

  const StreamQueries<MASK> geo(p.mask_off, p.window, p.n_q);
  int t_begin, t_end;
  geo.tile_range(k0, TS, t_begin, t_end);
  if (PARTS) split_range(part, p.n_split, t_begin, t_end);
  Dma<D, 1> dma;
  dma.init(p.stride_qn, 0, lane);
  const auto issue = [&](int t, uint32_t lds) {
    const int64_t q = srow + min(t * TS + n, p.n_q - 1);
    dma.template issue_all<NT>(lds, TILE, src, (int64_t)t * TS * p.stride_qn, 0, p.n_q - t * TS);
    stage_words(lds + NT * TILE, (h ? p.ws_d : p.lse) + q);
    stage_words(lds + NT * TILE + 2 * TS * 4, (h ? p.ws_b : p.ws_dd) + q);
  };
  char* const ring = smem + wave * NBUF * STAGE;
  first_tiles<W, NBUF, STAGE>(t_begin + ws, t_end, ring, issue);

  bf16x8_t Kb[KK], ddKb[KK], Vb[KK], ddVb[KK];
  load_resident<D>(Kb, (const __bf16*)p.k + koff, p.stride_kn, kr, h);
  load_resident<D>(ddKb, (const __bf16*)p.ddk + koff, p.stride_kn, kr, h);
  load_resident<D>(Vb, (const __bf16*)p.v + koff, p.stride_kn, kr, h);
  load_resident<D>(ddVb, (const __bf16*)p.ddv + koff, p.stride_kn, kr, h);
  wait_vm0();
  const float c_scale_log2 = p.scale * kLog2e;
  int aoff[KK], troff[NC][2];
  lane_offsets<D>(lane, aoff, troff);
  f32x16_t acc_dk[NC], acc_dv[NC];
#pragma unroll
  for (int cb = 0; cb < NC; cb++) acc_dk[cb] = f32x16_t{0}, acc_dv[cb] = f32x16_t{0};
  own_tiles<W, NBUF, STAGE, NT * Dma<D, 1>::IPT + 2>(t_begin + ws, t_end, ring, issue, [&](char* stage, int t) {
    // L, d, dd, b as they lie in memory -> L log2(e), -d, dd, -(dd d + b)
    float* const stat = reinterpret_cast<float*>(stage + NT * TILE);
    const float l = stat[n], d = stat[TS + n], dd = stat[2 * TS + n], b = stat[3 * TS + n];
    stat[h * TS + n] = h ? -d : l * kLog2e;
    if (h) stat[3 * TS + n] = -__builtin_fmaf(dd, d, b);
    k_block<F16, D>(geo, stage, aoff, troff, Kb, ddKb, Vb, ddVb, t * TS, k0, kj, h, c_scale_log2, p.scale, acc_dk, acc_dv);
  });
  __syncthreads();
  f32x16_t acc[2 * NC];
#pragma unroll
  for (int cb = 0; cb < NC; cb++) acc[cb] = acc_dk[cb], acc[NC + cb] = acc_dv[cb];
  f32x4_t out[2 * NC][4 / W];
  add_waves<W>(acc, smem, group, ws, lane, out);
  if (kj >= p.n_k) return;
  if (PARTS && p.part) {
    float* const to = p.part + ((int64_t)part * 2 * p.batch * p.n_k + (int64_t)bh * p.n_k + kj) * D;
    store_partial<NC, 4 / W>(to, out, ws, h);
    store_partial<NC, 4 / W>(to + (int64_t)p.batch * p.n_k * D, out + NC, ws, h);
    return;
  }
  store_part<F16, NC, 4 / W>((uint16_t*)p.dk2 + koff + (int64_t)kj * p.stride_kn, out, p.scale, ws, h);
  store_part<F16, NC, 4 / W>((uint16_t*)p.dv2 + koff + (int64_t)kj * p.stride_kn, out + NC, 1.f, ws, h);
}

// ---- first order: dK, dV --------------------------------------------------------------------------------------------------
// Q, dO and, without a sweep for dQ before it (OWN_D), O tiles; L log2(e) and d of their rows
template <int D, bool OWN_D>
constexpr int bwd_k_stage = (OWN_D ? 3 : 2) * TS * 2 * D + 2 * TS * 4;
template <int D, bool OWN_D>
constexpr int bwd_k_buffers = 2 * WAVES * bwd_k_stage<D, OWN_D> <= (OWN_D ? 128 : 160) * 1024 ? 2 : 1;

template <bool F16, int D, int MASK, int W, bool PARTS = false, bool OWN_D = true>   // PARTS: as in grads_k; without OWN_D behind a sweep for dQ
__device__ __forceinline__ void bwd_k(const AttnParams& p, char* smem, int id) {
  constexpr int KK = D / 16, NC = D / 32, ROWS = TS * WAVES / W, TILE = TS * 2 * D;
  constexpr int NT = OWN_D ? 3 : 2, STAGE = bwd_k_stage<D, OWN_D>, NBUF = bwd_k_buffers<D, OWN_D>;
  int bh, tile;
  if (!decode_block<MASK>((p.n_k + ROWS - 1) / ROWS, p.batch * (PARTS ? p.n_split : 1), false, p.tile_major_k != 0, bh, tile, false, id)) return;
  const int part = PARTS ? bh % p.n_split : 0;
  if (PARTS) bh /= p.n_split;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int group = wave / W, ws = wave % W;
  const int n = lane & 31, h = lane >> 5;
  const int k0 = tile * ROWS + TS * group, kj = k0 + n, kr = min(kj, p.n_k - 1);
  const int64_t qoff = (int64_t)bh * p.stride_qb, koff = (int64_t)bh * p.stride_kb, srow = (int64_t)bh * p.n_q;
  // bwd_k_block reads Q, dO and, behind them, the statistics; O lies at the end of a stage
  const __bf16* const src[2] = {(const __bf16*)p.q + qoff, (const __bf16*)p.dO + qoff};
  const __bf16* const src_o[1] = {(const __bf16*)p.o + qoff};
  constexpr int STAT = 2 * TILE, O = 2 * TILE + 2 * TS * 4;
  const StreamQueries<MASK> geo(p.mask_off, p.window, p.n_q);
  int t_begin, t_end;
  geo.tile_range(k0, TS, t_begin, t_end);
  if (PARTS) split_range(part, p.n_split, t_begin, t_end);
  Dma<D, 1> dma;
  dma.init(p.stride_qn, 0, lane);
  const auto issue = [&](int t, uint32_t lds) {
    const int64_t adv = (int64_t)t * TS * p.stride_qn;
    dma.template issue_all<2>(lds, TILE, src, adv, 0, p.n_q - t * TS);
    if (OWN_D) dma.template issue_all<1>(lds + O, TILE, src_o, adv, 0, p.n_q - t * TS);
    stage_words(lds + STAT, (OWN_D || !h ? p.lse : p.ws_d) + srow + min(t * TS + n, p.n_q - 1));
  };
  char* const ring = smem + wave * NBUF * STAGE;
  first_tiles<W, NBUF, STAGE>(t_begin + ws, t_end, ring, issue);
  bf16x8_t Kb[KK], Vb[KK];
  load_resident<D>(Kb, (const __bf16*)p.k + koff, p.stride_kn, kr, h);
  load_resident<D>(Vb, (const __bf16*)p.v + koff, p.stride_kn, kr, h);
  wait_vm0();
  const float c_scale_log2 = p.scale * kLog2e;
  int aoff[KK], troff[NC][2];
  lane_offsets<D>(lane, aoff, troff);
  f32x16_t acc[2][NC];
#pragma unroll
  for (int cb = 0; cb < NC; cb++) acc[0][cb] = f32x16_t{0}, acc[1][cb] = f32x16_t{0};
  own_tiles<W, NBUF, STAGE, NT * Dma<D, 1>::IPT + 1>(t_begin + ws, t_end, ring, issue, [&](char* stage, int t) {
    float* const stat = reinterpret_cast<float*>(stage + STAT);
    if constexpr (OWN_D) {
      bf16x8_t Ob[KK], dOb[KK];
#pragma unroll
      for (int kk = 0; kk < KK; kk++) Ob[kk] = lds_read128(stage + O, aoff[kk]), dOb[kk] = lds_read128(stage + TILE, aoff[kk]);
      float d = half_row_dot<F16, D>(Ob, dOb);
      d += __shfl_xor(d, 32);
      const float l = stat[n];
      stat[h * TS + n] = h ? d : l * kLog2e;
    } else if (!h) {
      stat[n] *= kLog2e;
    }
    bwd_k_block<F16, D>(geo, stage, aoff, troff, Kb, Vb, t * TS, k0, kj, h, c_scale_log2, acc);
  });
  __syncthreads();
  f32x16_t all[2 * NC];
#pragma unroll
  for (int cb = 0; cb < NC; cb++) all[cb] = acc[0][cb], all[NC + cb] = acc[1][cb];
  f32x4_t out[2 * NC][4 / W];
  add_waves<W>(all, smem, group, ws, lane, out);
  if (kj >= p.n_k) return;
  if (PARTS && p.part) {
    float* const to = p.part + ((int64_t)part * 2 * p.batch * p.n_k + (int64_t)bh * p.n_k + kj) * D;
    store_partial<NC, 4 / W>(to, out, ws, h);
    store_partial<NC, 4 / W>(to + (int64_t)p.batch * p.n_k * D, out + NC, ws, h);
    return;
  }
  store_part<F16, NC, 4 / W>((uint16_t*)p.dk + koff + (int64_t)kj * p.stride_kn, out, p.scale, ws, h);
  store_part<F16, NC, 4 / W>((uint16_t*)p.dv + koff + (int64_t)kj * p.stride_kn, out + NC, 1.f, ws, h);
}

template <int D>
constexpr int sink_bwd_lds = max_of(WAVES * bwd_k_buffers<D, false> * bwd_k_stage<D, false>, add_waves_bytes(2 * D / 32));

// Of the workgroups that sum up the rows of the sinks, the last ones of a launch (none without sinks): this one's number among them, negative for the others
__device__ __forceinline__ int sink_workgroup(int sinks, int slices) { return (int)blockIdx.x - (int)gridDim.x + (int)grid_blocks((sinks + TS - 1) / TS, slices); }

}  // namespace smallk
}  // namespace fhog
