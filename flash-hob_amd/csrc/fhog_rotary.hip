// Rotary positions: the pairs of channels of a query or key, turned by angles that grow with the token's position on one to four axes.
//
//   angle = p[axis(f)] theta^(-2 f / rotary_dim), f = 0 .. rotary_dim / 2 - 1;  (u, w) -> (u cos - w sin, w cos + u sin)
//
// on the pair (f, f + rotary_dim / 2), or (2 f, 2 f + 1) interleaved; the channels from rotary_dim on pass. The rotation is linear and orthogonal: its adjoint, and with
// it every derivative, is the rotation by the negative angle (inverse).
//
// A far position turns the first frequencies millions of times, so the number of turns is formed in 64 bits: p (theta^(-2f/rd) / 2 pi) is right to
// (6 + |ln theta|) 2^-53 of itself (the position, 1 / 2 pi, two products and the power, a step of 2^-52, are rounded, and so is its exponent, which ln theta multiplies),
// with theta >= 1 an angle to 2^-50 p at most. The nearest quarter is taken off exactly, and what is left, an eighth of a turn at most either way, goes through the sine's and cosine's own power series in single precision
// (terms up to x^9 and x^8: the first ones left out are 2e-9 and 3e-8 at pi / 4; with the roundings 6e-8 and 9.3e-8 off at most, over four million angles).
//
// What bounds it: memory, every channel in and out once. A thread owns V pairs of one token (two loads and two stores of 16 bytes) and keeps their sines and cosines in
// registers while it goes through the heads, of queries and keys alike; nothing is shared, so there is neither LDS nor a barrier.
#include <math.h>

#include "fhog_common.h"

namespace fhog {
namespace {

constexpr int kThreads = 256;

struct Heads {
  const void* in;
  void* out;
  int64_t in_b, in_h, in_n, out_b, out_h, out_n;   // strides in elements
};
struct Rotary {
  Heads q, k;
  const void* positions;
  int64_t pos_a, pos_b, pos_n;
  int64_t tokens;              // batch * n
  int32_t n, heads_q, heads;   // heads: of q and k together
  int32_t d, half, group;      // half: pairs of a row; group: heads that a workgroup goes through
  int32_t axes, first[3];      // first frequency of the second, third and fourth axis
  int32_t inverse;
  double turns[FHOG_ROTARY_MAX_D / 2];   // of one step of position, by frequency
};

template <typename P>
__device__ __forceinline__ double position(const Rotary& r, int a, int64_t b, int64_t t) {
  return (double)static_cast<const P*>(r.positions)[a * r.pos_a + b * r.pos_b + t * r.pos_n];
}

// sine and cosine of `turns` turns
__device__ __forceinline__ void sin_cos(double turns, float& s, float& c) {
  const double quarters = __builtin_rint(4 * turns);
  const float x = (float)(__builtin_fma(quarters, -0.25, turns) * 6.283185307179586);   // the difference is exact
  const float x2 = x * x;
  const auto next = [x2](float sum, float term) { return __builtin_fmaf(sum, x2, term); };
  const float sine = __builtin_fmaf(x * x2, next(next(next(1.f / 362880, -1.f / 5040), 1.f / 120), -1.f / 6), x);
  const float cosine = next(next(next(next(1.f / 40320, -1.f / 720), 1.f / 24), -0.5f), 1.f);
  const int quadrant = (int)(quarters - 4 * __builtin_floor(0.25 * quarters));   // quarters may lie beyond an int's range
  const bool odd = quadrant & 1;
  s = odd ? cosine : sine, c = odd ? sine : cosine;
  if (quadrant & 2) s = -s;
  if ((quadrant + 1) & 2) c = -c;
}

template <typename T, int V>
struct Vec {
  T v[V];
};

// V: pairs of a thread. LAYOUT 0: (f, f + half), 1: interleaved. P: type of the positions
template <typename T, int V, int LAYOUT, typename P>
__global__ void __launch_bounds__(kThreads) rotary(Rotary r) {
  typedef Vec<T, V> __attribute__((aligned(V * sizeof(T)))) Chunk;
  const int items = r.d / (2 * V);   // of a row: V pairs each, or 2 V channels that pass
  const int64_t id = (int64_t)blockIdx.x * kThreads + threadIdx.x, token = id / items;
  if (token >= r.tokens) return;
  const int item = (int)(id - token * items), f0 = item * V;
  const int64_t b = token / r.n, t = token - b * r.n;
  const bool turned = f0 < r.half;
  // the thread's two chunks: of the pairs, or consecutive ones
  const int c0 = LAYOUT == 0 && turned ? f0 : 2 * f0, c1 = LAYOUT == 0 && turned ? f0 + r.half : 2 * f0 + V;
  float s[V], c[V];
#pragma unroll
  for (int i = 0; i < V; i++) s[i] = 0.f, c[i] = 1.f;
  if (turned) {
    double p[4];
#pragma unroll
    for (int a = 0; a < 4; a++) p[a] = a < r.axes ? position<P>(r, a, b, t) : 0;
#pragma unroll
    for (int i = 0; i < V; i++) {
      const int f = f0 + i;
      double at = p[0];
#pragma unroll
      for (int a = 1; a < 4; a++) at = a < r.axes && f >= r.first[a - 1] ? p[a] : at;
      sin_cos(at * r.turns[f], s[i], c[i]);
      if (r.inverse) s[i] = -s[i];
    }
  }
  const int h0 = blockIdx.y * r.group, h1 = min(h0 + r.group, r.heads);
  const auto one = [&](int h, Chunk (&x)[2]) {
    const Heads& g = h < r.heads_q ? r.q : r.k;
    const T* const from = static_cast<const T*>(g.in) + b * g.in_b + (h < r.heads_q ? h : h - r.heads_q) * g.in_h + t * g.in_n;
    x[0] = *reinterpret_cast<const Chunk*>(from + c0), x[1] = *reinterpret_cast<const Chunk*>(from + c1);
  };
  const auto put = [&](int h, const Chunk (&x)[2]) {
    Chunk y[2];
    if (turned) {
#pragma unroll
      for (int i = 0; i < V; i++) {
        const int e0 = LAYOUT == 0 ? i : 2 * i, e1 = LAYOUT == 0 ? V + i : 2 * i + 1;
        const float u = (float)x[e0 / V].v[e0 % V], w = (float)x[e1 / V].v[e1 % V];
        y[e0 / V].v[e0 % V] = (T)__builtin_fmaf(u, c[i], -(w * s[i]));   // written out: the same bits from chunks and pair by pair
        y[e1 / V].v[e1 % V] = (T)__builtin_fmaf(w, c[i], u * s[i]);
      }
    } else {
      y[0] = x[0], y[1] = x[1];
    }
    const Heads& g = h < r.heads_q ? r.q : r.k;
    T* const to = static_cast<T*>(g.out) + b * g.out_b + (h < r.heads_q ? h : h - r.heads_q) * g.out_h + t * g.out_n;
    *reinterpret_cast<Chunk*>(to + c0) = y[0], *reinterpret_cast<Chunk*>(to + c1) = y[1];
  };
  for (int h = h0; h < h1; h++) {
    Chunk x[2];
    one(h, x);
    put(h, x);
  }
}

template <typename T, int V, int LAYOUT>
hipError_t launch_p(const Rotary& r, int positions, dim3 grid, hipStream_t s) {
  switch (positions) {
    case FHOG_POSITIONS_INT32: hipLaunchKernelGGL((rotary<T, V, LAYOUT, int32_t>), grid, dim3(kThreads), 0, s, r); break;
    case FHOG_POSITIONS_INT64: hipLaunchKernelGGL((rotary<T, V, LAYOUT, int64_t>), grid, dim3(kThreads), 0, s, r); break;
    default: hipLaunchKernelGGL((rotary<T, V, LAYOUT, float>), grid, dim3(kThreads), 0, s, r);
  }
  return hipGetLastError();
}

template <typename T, int V>
hipError_t launch_v(Rotary r, const fhog_rotary_args* a, hipStream_t s) {
  const int64_t blocks = (r.tokens * (r.d / (2 * V)) + kThreads - 1) / kThreads;
  // Heads to a workgroup: as few as give 2048 workgroups, eight for every CU, and all of them where the tokens alone do
  int64_t groups = (2048 + blocks - 1) / blocks;
  if (groups > r.heads) groups = r.heads;
  r.group = (int32_t)((r.heads + groups - 1) / groups);
  const dim3 grid((unsigned)blocks, (unsigned)((r.heads + r.group - 1) / r.group));
  return a->interleaved ? launch_p<T, V, 1>(r, a->position_type, grid, s) : launch_p<T, V, 0>(r, a->position_type, grid, s);
}

// Chunks of 16 bytes where every row lies on a multiple of them and the pairs come in whole chunks, else pair by pair
template <typename T>
hipError_t launch_t(const Rotary& r, const fhog_rotary_args* a, hipStream_t s) {
  constexpr int V = 16 / sizeof(T);
  bool wide = a->d % (2 * V) == 0 && a->rotary_dim % (2 * V) == 0;
  const auto fits = [&](const Heads& h) {
    wide = wide && (reinterpret_cast<uintptr_t>(h.in) | reinterpret_cast<uintptr_t>(h.out)) % 16 == 0 &&
           (h.in_b | h.in_h | h.in_n | h.out_b | h.out_h | h.out_n) % V == 0;
  };
  fits(r.q);
  if (a->heads_k > 0) fits(r.k);
  return wide ? launch_v<T, V>(r, a, s) : launch_v<T, 1>(r, a, s);
}

// Turns of one step of position. 64 powers take the host 2 us, so a thread keeps the last table: it depends on theta and the number of pairs alone.
void turns_of(double theta, int half, double* turns) {
  thread_local double kept[FHOG_ROTARY_MAX_D / 2];
  thread_local double kept_theta = 0;
  thread_local int kept_half = 0;
  if (theta != kept_theta || half != kept_half) {
    for (int f = 0; f < half; f++) kept[f] = pow(theta, -(double)f / half) * 0.15915494309189533577;   // 1 / 2 pi
    kept_theta = theta, kept_half = half;
  }
  for (int f = 0; f < half; f++) turns[f] = kept[f];
}

}  // namespace

hipError_t launch_rotary(const fhog_rotary_args* a, hipStream_t s) {
  Rotary r = {};
  r.q = {a->q, a->q_out, a->stride_qb, a->stride_qh, a->stride_qn, a->stride_qob, a->stride_qoh, a->stride_qon};
  r.k = {a->k, a->k_out, a->stride_kb, a->stride_kh, a->stride_kn, a->stride_kob, a->stride_koh, a->stride_kon};
  r.positions = a->positions, r.pos_a = a->stride_pa, r.pos_b = a->stride_pb, r.pos_n = a->stride_pn;
  r.tokens = a->batch * a->n, r.n = (int32_t)a->n;
  r.heads_q = (int32_t)a->heads_q, r.heads = (int32_t)(a->heads_q + a->heads_k);
  r.d = (int32_t)a->d, r.half = (int32_t)(a->rotary_dim / 2);
  r.axes = a->axes;
  for (int i = 0, at = 0; i < 3; i++) r.first[i] = i + 1 < a->axes ? (at += a->sections[i]) : 0;
  r.inverse = a->inverse;
  turns_of(a->theta, r.half, r.turns);
  switch (a->dtype) {
    case FHOG_DTYPE_FP32: return launch_t<float>(r, a, s);
    case FHOG_DTYPE_FP16: return launch_t<_Float16>(r, a, s);
    default: return launch_t<__bf16>(r, a, s);
  }
}

}  // namespace fhog
