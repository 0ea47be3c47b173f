// C ABI of libfhog_hip.so: argument validation, kernel-family selection, pass sequencing.
// Replaces the host side of flash_bwdbwd (fhog/triton_bwdbwd.py:557-648).
#include <math.h>
#include <stdarg.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include <algorithm>
#include <atomic>
#include <utility>

#include "fhog_common.h"
#include "fhog_rules.h"

// Workspace of fhog_bwdbwd_static_ws: device memory that belongs to the loaded library, so that the entry point never
// allocates. Every GPU the library runs on holds its own copy at its own address until the process ends; the name below
// is only a host-side handle, the address on the current device comes from hipGetSymbolAddress (scratch_on_device).
static __device__ __align__(256) unsigned char scratch[FHOG_STATIC_WS_BYTES];

namespace {

using namespace fhog::rules;

thread_local char g_err[512] = "";

int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

// the staging loads address a 32-row tile with 32-bit byte offsets per lane: 32 rows * stride * 2 bytes must fit
constexpr int64_t kMaxRowStride = (int64_t)1 << 24;

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// FHOG_OK or the error for a mask that does not apply to the shape
int check_mask(int32_t causal, int64_t window, int64_t n_q, int64_t n_k) {
  if (causal < FHOG_MASK_NONE || causal > FHOG_MASK_BOTTOM_RIGHT) return fail(FHOG_E_CAUSAL, "causal must be 0, 1 or 2");
  if (causal == FHOG_MASK_TOP_LEFT && n_q != n_k)
    return fail(FHOG_E_CAUSAL, "causal (top-left) needs n_q == n_k (got %lld, %lld)", (long long)n_q, (long long)n_k);
  if (causal == FHOG_MASK_BOTTOM_RIGHT && n_k < n_q)
    return fail(FHOG_E_CAUSAL, "causal (bottom-right) needs n_k >= n_q (got %lld, %lld)", (long long)n_k, (long long)n_q);
  if (window < 0) return fail(FHOG_E_CAUSAL, "window must be >= 0");
  if (window > 0 && causal == FHOG_MASK_NONE) return fail(FHOG_E_CAUSAL, "a window needs a causal mask");
  return FHOG_OK;
}
int validate(const fhog_bwdbwd_args* a) {
  if (!a) return fail(FHOG_E_NULL, "args is NULL");
  const void* ptrs[] = {a->q, a->k, a->v, a->o, a->dO, a->ddq, a->ddk, a->ddv, a->lse, a->dq2, a->dk2, a->dv2, a->ddo, a->ws};
  const char* names[] = {"q", "k", "v", "o", "dO", "ddq", "ddk", "ddv", "lse", "dq2", "dk2", "dv2", "ddo", "ws"};
  for (int i = 0; i < 14; i++)
    if (!ptrs[i]) return fail(FHOG_E_NULL, "pointer '%s' is NULL", names[i]);
  if (a->dtype != FHOG_DTYPE_BF16 && a->dtype != FHOG_DTYPE_FP32 && a->dtype != FHOG_DTYPE_FP16)
    return fail(FHOG_E_DTYPE, "unknown dtype %d", a->dtype);
  if (a->impl != FHOG_IMPL_AUTO && a->impl != FHOG_IMPL_FP32 && a->impl != FHOG_IMPL_BF16)
    return fail(FHOG_E_IMPL, "unknown impl %d", a->impl);
  if (a->schedule < FHOG_SCHEDULE_FOUR_PASS || a->schedule > FHOG_SCHEDULE_THREE_SWEEP)
    return fail(FHOG_E_SCHEDULE, "unknown schedule %d", a->schedule);
  if (a->batch < 1 || a->n_q < 1 || a->n_k < 1)
    return fail(FHOG_E_SHAPE, "batch, n_q, n_k must be >= 1 (got %lld, %lld, %lld)", (long long)a->batch, (long long)a->n_q,
                (long long)a->n_k);
  if (a->batch > 65535) return fail(FHOG_E_SHAPE, "batch %lld above 65535 (batch * head slices) is not supported", (long long)a->batch);
  if (a->n_q > (1 << 24) || a->n_k > (1 << 24)) return fail(FHOG_E_SHAPE, "n_q/n_k above 2^24 not supported");
  if (a->batch * a->n_q >= (int64_t)1 << 31) return fail(FHOG_E_SHAPE, "batch*n_q must be below 2^31");
  if (a->d != 32 && a->d != 64 && a->d != 128) return fail(FHOG_E_SHAPE, "head dim %lld not in {32, 64, 128}", (long long)a->d);
  if (const int rc = check_mask(a->causal, a->window, a->n_q, a->n_k)) return rc;
  if (!isfinite(a->scale)) return fail(FHOG_E_SCALE, "scale is not finite");
  if (a->ws_bytes != 0 && a->ws_bytes < (int64_t)(3 * a->batch * a->n_q * sizeof(float)))
    return fail(FHOG_E_SHAPE, "ws_bytes %lld is below the minimum of 3 * batch * n_q floats", (long long)a->ws_bytes);
  const int vec = a->dtype == FHOG_DTYPE_FP32 ? 4 : 8;  // elements per 16 bytes
  if (a->stride_qn < a->d || a->stride_kn < a->d) return fail(FHOG_E_STRIDE, "row stride smaller than d");
  if (a->stride_qn > kMaxRowStride || a->stride_kn > kMaxRowStride) return fail(FHOG_E_STRIDE, "row stride above 2^24 elements");
  if (a->stride_qn % vec || a->stride_kn % vec || a->stride_qb % vec || a->stride_kb % vec)
    return fail(FHOG_E_STRIDE, "strides must be multiples of %d elements (16 bytes)", vec);
  if (a->batch > 1 && (a->stride_qb < a->n_q * a->stride_qn || a->stride_kb < a->n_k * a->stride_kn))
    return fail(FHOG_E_STRIDE, "batch stride smaller than one (n, d) slice");
  for (int i = 0; i < 14; i++)
    if (!aligned16(ptrs[i])) return fail(FHOG_E_ALIGN, "pointer '%s' is not 16-byte aligned", names[i]);
  if (a->impl == FHOG_IMPL_BF16) {
    if (a->dtype == FHOG_DTYPE_FP32) return fail(FHOG_E_DTYPE, "impl=bf16 needs bf16 or fp16 tensors");
    if (!fhog::bf16_shape_supported(a->n_q, a->n_k, a->d, a->causal))
      return fail(FHOG_E_SHAPE, "impl=bf16 needs d in {64,128}");
  }
  return FHOG_OK;
}

int select_impl(const fhog_bwdbwd_args* a) {
  if (a->impl == FHOG_IMPL_FP32) return FHOG_IMPL_FP32;
  if (a->impl == FHOG_IMPL_BF16) return FHOG_IMPL_BF16;
  if (a->dtype != FHOG_DTYPE_FP32 && fhog::bf16_shape_supported(a->n_q, a->n_k, a->d, a->causal)) return FHOG_IMPL_BF16;
  return FHOG_IMPL_FP32;
}

fhog::Params to_params(const fhog_bwdbwd_args* a) {
  fhog::Params p;
  p.q = a->q;
  p.k = a->k;
  p.v = a->v;
  p.o = a->o;
  p.dO = a->dO;
  p.ddq = a->ddq;
  p.ddk = a->ddk;
  p.ddv = a->ddv;
  p.lse = a->lse;
  p.dq2 = a->dq2;
  p.dk2 = a->dk2;
  p.dv2 = a->dv2;
  p.ddo = a->ddo;
  const int64_t rows = a->batch * a->n_q;
  p.ws_d = a->ws;
  p.ws_dd = a->ws + rows;
  p.ws_b = a->ws + 2 * rows;
  p.stride_qb = a->stride_qb;
  p.stride_qn = a->stride_qn;
  p.stride_kb = a->stride_kb;
  p.stride_kn = a->stride_kn;
  p.batch = (int32_t)a->batch;
  p.n_q = (int32_t)a->n_q;
  p.n_k = (int32_t)a->n_k;
  p.d = (int32_t)a->d;
  p.scale = a->scale;
  p.causal = a->causal != FHOG_MASK_NONE;
  p.f16 = a->dtype == FHOG_DTYPE_FP16;
  mask_params(a->causal, a->window, a->n_q, a->n_k, &p.mask_off, &p.window);
  p.sinks = 0, p.n_split_s = 1, p.part_s = nullptr;
  p.n_split = 1;
  p.part = nullptr;
  const int order = fhog::tuning().order;
  p.tile_major = order < 0 ? p.causal : order;
  p.n_split_k = 1, p.tile_major_k = p.tile_major, p.part_k = nullptr;
  return p;
}

// Pass 3 or 7 (q_pass, 0: none) and pass 4 (k_side) of the 16-bit kernels, in one launch
int run_grads(const fhog_bwdbwd_args* a, const fhog::Params& base, int q_pass, bool k_side, hipStream_t s) {
  fhog::Params p = base;
  if (q_pass && k_side) {
    joint_splits(a, p, q_pass, &p.n_split, &p.n_split_k);
  } else {
    p.n_split = q_pass ? launch_split_of(a, p, FHOG_IMPL_BF16, q_pass) : 1;
    p.n_split_k = k_side ? launch_split_of(a, p, FHOG_IMPL_BF16, FHOG_PASS_DK_DV) : 1;
  }
  grads_order(a, q_pass != 0, k_side, p);
  p.part = reinterpret_cast<float*>(reinterpret_cast<char*>(a->ws) + stats_bytes(a));
  p.part_k = p.part + (p.n_split > 1 ? p.n_split * (split_bytes(a, FHOG_PASS_DQ_DDO) / sizeof(float)) : 0);
  const hipError_t e = fhog::launch_bf16_grads(p, q_pass, k_side, s);
  if (e != hipSuccess) return fail(FHOG_E_LAUNCH, "passes %d and %d: HIP error %d (%s)", q_pass, k_side ? FHOG_PASS_DK_DV : 0, (int)e, hipGetErrorString(e));
  return FHOG_OK;
}

int run_pass(const fhog_bwdbwd_args* a, const fhog::Params& base, int impl, int pass, hipStream_t s) {
  if (pass > FHOG_PASS_DD_B && impl != FHOG_IMPL_BF16)
    return fail(FHOG_E_PASS, "pass %d exists in the 16-bit MFMA family only (bf16 / fp16 tensors, d in {64, 128})", pass);
  if (pass == FHOG_PASS_STAGE1 && a->d != 64)
    return fail(FHOG_E_PASS, "pass %d (three sweeps in one launch) exists for d = 64 only", pass);
  if (impl == FHOG_IMPL_BF16 && (pass == FHOG_PASS_DQ_DDO || pass == FHOG_PASS_DQ)) return run_grads(a, base, pass, false, s);
  if (impl == FHOG_IMPL_BF16 && pass == FHOG_PASS_DK_DV) return run_grads(a, base, 0, true, s);
  fhog::Params p = base;
  p.n_split = launch_split_of(a, p, impl, pass);
  pass_order(a, pass, p);
  p.part = reinterpret_cast<float*>(reinterpret_cast<char*>(a->ws) + stats_bytes(a));
  hipError_t e;
  if (pass == FHOG_PASS_D)
    e = fhog::launch_rowdot(p, a->dtype, s);
  else if (impl == FHOG_IMPL_BF16)
    e = fhog::launch_bf16_pass(p, pass, s);
  else
    e = fhog::launch_split_pass(p, a->dtype, pass, s);
  if (e != hipSuccess) return fail(FHOG_E_LAUNCH, "pass %d: HIP error %d (%s)", pass == fhog::kPassGrads ? FHOG_PASS_DQ_DDO : pass, (int)e, hipGetErrorString(e));
  return FHOG_OK;
}

// bf16 / fp16 tensors with d in {64, 128} run on the 16-bit MFMA kernels, everything else (fp32 tensors, d = 32) on the
// split-product ones
bool attn_on_16bit_kernels(const fhog_attn_args* a) { return a->dtype != FHOG_DTYPE_FP32 && (a->d == 64 || a->d == 128); }

int validate_attn(const fhog_attn_args* a, int backward) {
  if (!a) return fail(FHOG_E_NULL, "args is NULL");
  const void* ptrs[] = {a->q, a->k, a->v, a->o, a->lse, a->dO, a->dq, a->dk, a->dv, a->ws};
  const char* names[] = {"q", "k", "v", "o", "lse", "dO", "dq", "dk", "dv", "ws"};
  const int n_ptr = backward ? 10 : 5;
  for (int i = 0; i < n_ptr; i++) {
    if (!ptrs[i]) return fail(FHOG_E_NULL, "pointer '%s' is NULL", names[i]);
    if (!aligned16(ptrs[i])) return fail(FHOG_E_ALIGN, "pointer '%s' is not 16-byte aligned", names[i]);
  }
  if (a->dtype != FHOG_DTYPE_BF16 && a->dtype != FHOG_DTYPE_FP16 && a->dtype != FHOG_DTYPE_FP32)
    return fail(FHOG_E_DTYPE, "unknown dtype %d", a->dtype);
  if (a->batch < 1 || a->batch > 65535) return fail(FHOG_E_SHAPE, "batch %lld outside 1..65535", (long long)a->batch);
  if (a->n_q < 1 || a->n_k < 1 || a->n_q > (1 << 24) || a->n_k > (1 << 24) || a->batch * a->n_q >= (int64_t)1 << 31)
    return fail(FHOG_E_SHAPE, "n_q/n_k out of range");
  if (const int rc = check_mask(a->causal, a->window, a->n_q, a->n_k)) return rc;
  if (a->d != 32 && a->d != 64 && a->d != 128) return fail(FHOG_E_SHAPE, "head dim %lld not in {32, 64, 128}", (long long)a->d);
  if (!isfinite(a->scale)) return fail(FHOG_E_SCALE, "scale is not finite");
  // the 16-bit forward takes the running maximum of the raw scores and scales it afterwards, which needs scale > 0
  if (attn_on_16bit_kernels(a) && a->scale <= 0.f)
    return fail(FHOG_E_SCALE, "the 16-bit kernels need a positive scale (got %g)", (double)a->scale);
  const int vec = a->dtype == FHOG_DTYPE_FP32 ? 4 : 8;  // elements per 16 bytes
  if (a->stride_qn < a->d || a->stride_kn < a->d) return fail(FHOG_E_STRIDE, "row stride smaller than d");
  if (a->stride_qn > kMaxRowStride || a->stride_kn > kMaxRowStride) return fail(FHOG_E_STRIDE, "row stride above 2^24 elements");
  if (a->stride_qn % vec || a->stride_kn % vec || a->stride_qb % vec || a->stride_kb % vec)
    return fail(FHOG_E_STRIDE, "strides must be multiples of %d elements (16 bytes)", vec);
  if (a->batch > 1 && (a->stride_qb < a->n_q * a->stride_qn || a->stride_kb < a->n_k * a->stride_kn))
    return fail(FHOG_E_STRIDE, "batch stride smaller than one (n, d) slice");
  return FHOG_OK;
}

fhog::AttnParams to_attn_params(const fhog_attn_args* a) {
  fhog::AttnParams p;
  p.q = a->q;
  p.k = a->k;
  p.v = a->v;
  p.o = a->o;
  p.lse = a->lse;
  p.dO = a->dO;
  p.dq = a->dq;
  p.dk = a->dk;
  p.dv = a->dv;
  p.ws_d = a->ws;
  p.stride_qb = a->stride_qb;
  p.stride_qn = a->stride_qn;
  p.stride_kb = a->stride_kb;
  p.stride_kn = a->stride_kn;
  p.batch = (int32_t)a->batch;
  p.n_q = (int32_t)a->n_q;
  p.n_k = (int32_t)a->n_k;
  p.d = (int32_t)a->d;
  p.scale = a->scale;
  p.causal = a->causal != FHOG_MASK_NONE;
  p.f16 = a->dtype == FHOG_DTYPE_FP16;
  mask_params(a->causal, a->window, a->n_q, a->n_k, &p.mask_off, &p.window);
  p.sinks = 0, p.n_split = 1, p.part = nullptr;
  // as in run_pass: tile-major with a mask, until a slice alone has tiles enough to balance the end of a launch
  const int order = fhog::tuning().order;
  p.tile_major_q = order < 0 ? (p.causal && a->n_q < 16384) : order;
  p.tile_major_k = order < 0 ? (p.causal && a->n_k < 16384) : order;
  return p;
}

int dtype_bytes(int dtype) { return dtype == FHOG_DTYPE_FP32 ? 4 : 2; }
// Sinks of a mask, or the error for a number that is none
int check_sinks(int64_t sinks) { return sinks < 0 ? fail(FHOG_E_CAUSAL, "sinks must be >= 0 (got %lld)", (long long)sinks) : FHOG_OK; }
int32_t sinks_of(const fhog_attn_args* a, int64_t sinks) { return fhog::rules::sinks_of(sinks, a->window, a->n_k); }
int32_t sinks_of(const fhog_bwdbwd_args* a, int64_t sinks) { return fhog::rules::sinks_of(sinks, a->window, a->n_k); }

int forward_parts(const fhog_attn_args* a, int32_t sinks) {
  return fhog::rules::forward_parts(a->batch, a->n_q, a->n_k, a->d, a->window, sinks, dtype_bytes(a->dtype));
}

// Row sums d of a first backward, rounded up so that what follows stays 16-byte aligned
size_t row_bytes(const fhog_attn_args* a) { return ((size_t)a->batch * a->n_q * sizeof(float) + 15) & ~(size_t)15; }

size_t attn_sinks_bytes(const fhog_attn_args* a, int64_t sinks, int backward) {
  const int32_t n = sinks_of(a, sinks);
  if (backward) return n ? row_bytes(a) + sink_bytes(a->batch, n, a->n_q, a->d, dtype_bytes(a->dtype), false) : (size_t)a->batch * a->n_q * sizeof(float);
  return n ? forward_part_bytes(a->batch, a->n_q, a->d, forward_parts(a, n)) : 0;
}

// A workspace of the entry points with sinks: there, aligned and as large as the call needs
int check_ws(const void* ws, int64_t have, size_t need) {
  if (need == 0) return FHOG_OK;
  if (!ws) return fail(FHOG_E_NULL, "pointer 'ws' is NULL");
  if (!aligned16(ws)) return fail(FHOG_E_ALIGN, "pointer 'ws' is not 16-byte aligned");
  if (have < 0 || (size_t)have < need) return fail(FHOG_E_SHAPE, "ws_bytes %lld is below the %zu bytes that this call needs", (long long)have, need);
  return FHOG_OK;
}

// Whether the rows of a (batch, heads, n, d) output lie apart: from the shortest stride up, each has to pass what lies below it
bool rows_apart(int64_t batch, int64_t heads, int64_t n, int64_t d, int64_t stride_b, int64_t stride_h, int64_t stride_n) {
  struct Dim {
    int64_t size;
    __int128 stride;
  } dims[] = {{batch, stride_b}, {heads, stride_h}, {n, stride_n}};
  for (Dim& x : dims) x.stride = x.size == 1 ? 0 : x.stride < 0 ? -x.stride : x.stride;   // a dimension of one is never stepped along
  std::sort(dims, dims + 3, [](const Dim& x, const Dim& y) { return x.stride < y.stride; });
  __int128 extent = d;
  for (const Dim& x : dims) {
    if (x.size == 1) continue;
    if (x.stride < extent) return false;
    extent += (x.size - 1) * x.stride;
  }
  return true;
}

int validate_rotary(const fhog_rotary_args* a) {
  if (!a) return fail(FHOG_E_NULL, "args is NULL");
  if (a->dtype != FHOG_DTYPE_BF16 && a->dtype != FHOG_DTYPE_FP16 && a->dtype != FHOG_DTYPE_FP32) return fail(FHOG_E_DTYPE, "unknown dtype %d", a->dtype);
  if (a->batch < 0 || a->n < 0 || a->heads_q < 1 || a->heads_k < 0)
    return fail(FHOG_E_SHAPE, "batch, n and heads_k must be >= 0, heads_q >= 1 (got %lld, %lld, %lld, %lld)", (long long)a->batch, (long long)a->n,
                (long long)a->heads_k, (long long)a->heads_q);
  if (a->n > INT32_MAX || a->batch > INT32_MAX || a->heads_q > 65535 || a->heads_k > 65535 || a->heads_q + a->heads_k > 65535)
    return fail(FHOG_E_SHAPE, "more than 2^31 - 1 rows or slices, or 65535 heads of queries and keys, are not supported");
  if (a->d < 2 || a->d > FHOG_ROTARY_MAX_D || a->d % 2) return fail(FHOG_E_SHAPE, "head dim %lld is not an even number in 2..%d", (long long)a->d, FHOG_ROTARY_MAX_D);
  if (a->rotary_dim < 2 || a->rotary_dim > a->d || a->rotary_dim % 2)
    return fail(FHOG_E_SHAPE, "rotary_dim %lld is not an even number in 2..%lld", (long long)a->rotary_dim, (long long)a->d);
  // a thread for each, in whole workgroups: a launch has fewer than 2^32
  if (a->n > 0 && a->batch > ((int64_t)UINT32_MAX - 255) / (a->d / 2) / a->n) return fail(FHOG_E_SHAPE, "batch * n * d / 2 above 2^32 - 256 is not supported");
  if (a->axes < 1 || a->axes > FHOG_ROTARY_MAX_AXES) return fail(FHOG_E_ROTARY, "axes must be 1..%d (got %d)", FHOG_ROTARY_MAX_AXES, a->axes);
  int64_t sum = 0;
  for (int i = 0; i < a->axes; i++) {
    if (a->sections[i] < 0) return fail(FHOG_E_ROTARY, "section %d is negative", i);
    sum += a->sections[i];
  }
  if (sum != a->rotary_dim / 2) return fail(FHOG_E_ROTARY, "the sections hold %lld frequencies, rotary_dim %lld has %lld", (long long)sum, (long long)a->rotary_dim, (long long)(a->rotary_dim / 2));
  if (!(a->theta > 0) || !isfinite(a->theta)) return fail(FHOG_E_ROTARY, "theta must be a positive number (got %g)", a->theta);
  if (a->position_type < FHOG_POSITIONS_INT32 || a->position_type > FHOG_POSITIONS_FP32) return fail(FHOG_E_ROTARY, "unknown type of positions %d", a->position_type);
  if (a->batch == 0 || a->n == 0) return FHOG_OK;   // nothing is read or written
  const void* ptrs[] = {a->q, a->q_out, a->positions, a->k, a->k_out};
  const char* names[] = {"q", "q_out", "positions", "k", "k_out"};
  const int align = a->dtype == FHOG_DTYPE_FP32 ? 4 : 2;
  for (int i = 0; i < (a->heads_k > 0 ? 5 : 3); i++) {
    if (!ptrs[i]) return fail(FHOG_E_NULL, "pointer '%s' is NULL", names[i]);
    if (reinterpret_cast<uintptr_t>(ptrs[i]) % (i == 2 ? (a->position_type == FHOG_POSITIONS_INT64 ? 8 : 4) : align))
      return fail(FHOG_E_ALIGN, "pointer '%s' is not aligned to its type", names[i]);
  }
  // rows that share an address would be written by several threads
  if (!rows_apart(a->batch, a->heads_q, a->n, a->d, a->stride_qob, a->stride_qoh, a->stride_qon) ||
      (a->heads_k > 0 && (a->q_out == a->k_out || !rows_apart(a->batch, a->heads_k, a->n, a->d, a->stride_kob, a->stride_koh, a->stride_kon))))
    return fail(FHOG_E_STRIDE, "rows of an output overlap");
  return FHOG_OK;
}

bool dtype_known(int dtype) { return dtype == FHOG_DTYPE_BF16 || dtype == FHOG_DTYPE_FP32 || dtype == FHOG_DTYPE_FP16; }
bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }
constexpr int64_t kMaxEntries = (int64_t)1 << 30;   // of a sequence
constexpr int64_t kMaxIndex = (int64_t)INT32_MAX - 255;

// Strides of rows that are read 16 bytes at a time; dimensions of one are never stepped along
int check_strides(const char* name, int dtype, const int64_t (&size)[3], const int64_t (&stride)[3]) {
  const int64_t vec = 16 / dtype_bytes(dtype);
  for (int i = 0; i < 3; i++)
    if (size[i] > 1 && stride[i] % vec) return fail(FHOG_E_STRIDE, "strides of '%s' must be multiples of %lld elements (16 bytes)", name, (long long)vec);
  return FHOG_OK;
}
int check_pointer(const char* name, const void* p, bool wide) {
  if (!p) return fail(FHOG_E_NULL, "pointer '%s' is NULL", name);
  if (wide ? !aligned16(p) : !aligned4(p)) return fail(FHOG_E_ALIGN, "pointer '%s' is not %s-byte aligned", name, wide ? "16" : "4");
  return FHOG_OK;
}

int validate_cache(const fhog_paged_cache& c, bool written) {
  if (!dtype_known(c.dtype)) return fail(FHOG_E_DTYPE, "unknown dtype %d", c.dtype);
  if (c.d != 32 && c.d != 64 && c.d != 128) return fail(FHOG_E_SHAPE, "head dim %lld not in {32, 64, 128}", (long long)c.d);
  if (c.batch < 0 || c.heads_k < 1 || c.batch > 65535 || c.heads_k > 65535 || c.batch * c.heads_k > 65535)
    return fail(FHOG_E_SHAPE, "%lld sequences of %lld heads of keys: expected 1 head or more, and 65535 or fewer of all sequences together", (long long)c.batch, (long long)c.heads_k);
  if (c.pages < 1 || c.pages > INT32_MAX) return fail(FHOG_E_PAGED, "%lld pages: expected 1 to 2^31 - 1", (long long)c.pages);
  if (c.page < 1 || c.table_width < 1 || c.page > kMaxEntries || c.table_width > kMaxEntries / c.page)
    return fail(FHOG_E_PAGED, "pages of %lld entries, %lld to a sequence: expected 1 or more of each, and 2^30 entries or fewer of a sequence", (long long)c.page, (long long)c.table_width);
  if (const int rc = check_strides("keys", c.dtype, {c.pages, c.heads_k, c.page}, {c.stride_p, c.stride_h, c.stride_n})) return rc;
  if (c.page > 1 && (c.stride_n < c.d || c.stride_n > kMaxRowStride)) return fail(FHOG_E_STRIDE, "entries of a page have to lie d to 2^24 elements apart (got %lld)", (long long)c.stride_n);
  if ((c.pages > 1 && c.stride_p < 0) || (c.heads_k > 1 && c.stride_h < 0)) return fail(FHOG_E_STRIDE, "strides of pages and heads of keys must not be negative");
  if (!rows_apart(c.pages, c.heads_k, c.page, c.d, c.stride_p, c.stride_h, c.stride_n)) return fail(FHOG_E_STRIDE, "entries of the pages overlap");
  if (c.batch == 0) return FHOG_OK;
  for (const auto& x : {std::make_pair("keys", c.keys), std::make_pair("values", c.values)})
    if (const int rc = check_pointer(x.first, x.second, true)) return rc;
  if (const int rc = check_pointer("table", c.table, false)) return rc;
  if (const int rc = check_pointer("lengths", c.lengths, false)) return rc;
  if (written && c.keys == c.values) return fail(FHOG_E_PAGED, "keys and values lie in the same place");
  return FHOG_OK;
}

int validate_append(const fhog_paged_append_args* a) {
  if (!a) return fail(FHOG_E_NULL, "args is NULL");
  const fhog_paged_cache& c = a->cache;
  if (const int rc = validate_cache(c, true)) return rc;
  if (a->n < 0 || a->n > kMaxEntries) return fail(FHOG_E_SHAPE, "n must be 0 to 2^30 (got %lld)", (long long)a->n);
  if (c.batch == 0 || a->n == 0) return FHOG_OK;
  if (a->n > kMaxIndex / (c.d * dtype_bytes(c.dtype) / 16) / (c.batch * c.heads_k)) return fail(FHOG_E_SHAPE, "more than 2^31 - 256 pieces of 16 bytes are not supported");
  if (const int rc = check_strides("k", c.dtype, {c.batch, c.heads_k, a->n}, {a->stride_kb, a->stride_kh, a->stride_kn})) return rc;
  if (const int rc = check_strides("v", c.dtype, {c.batch, c.heads_k, a->n}, {a->stride_vb, a->stride_vh, a->stride_vn})) return rc;
  if (const int rc = check_pointer("k", a->k, true)) return rc;
  if (const int rc = check_pointer("v", a->v, true)) return rc;
  return a->counts ? check_pointer("counts", a->counts, false) : FHOG_OK;
}

int validate_paged_attn(const fhog_paged_attn_args* a) {
  if (!a) return fail(FHOG_E_NULL, "args is NULL");
  const fhog_paged_cache& c = a->cache;
  if (const int rc = validate_cache(c, false)) return rc;
  if (a->heads_q < 1 || a->heads_q > 65535 || a->heads_q % c.heads_k || c.batch * a->heads_q > INT32_MAX / 128)
    return fail(FHOG_E_SHAPE, "%lld heads of queries and %lld of keys: expected a multiple, 65535 or fewer, and 2^24 - 1 or fewer of all sequences together", (long long)a->heads_q,
                (long long)c.heads_k);
  if (!isfinite(a->scale)) return fail(FHOG_E_SCALE, "scale is not finite");
  if (a->window < 0) return fail(FHOG_E_CAUSAL, "window must be >= 0");
  if (const int rc = check_sinks(a->sinks)) return rc;
  const int64_t capacity = c.page * c.table_width;
  if (c.batch * c.heads_k * ((capacity + 1023) / 1024) > kMaxIndex / 2) return fail(FHOG_E_SHAPE, "more than 2^40 entries of all sequences together are not supported");
  if (c.batch == 0) return FHOG_OK;
  if (const int rc = check_strides("q", c.dtype, {c.batch, a->heads_q, 1}, {a->stride_qb, a->stride_qh, 0})) return rc;
  if (const int rc = check_strides("o", c.dtype, {c.batch, a->heads_q, 1}, {a->stride_ob, a->stride_oh, 0})) return rc;
  if (!rows_apart(c.batch, a->heads_q, 1, c.d, a->stride_ob, a->stride_oh, 0)) return fail(FHOG_E_STRIDE, "rows of an output overlap");
  if (const int rc = check_pointer("q", a->q, true)) return rc;
  if (const int rc = check_pointer("o", a->o, true)) return rc;
  if (const int rc = check_pointer("lse", a->lse, false)) return rc;
  if (!a->weights_in != !a->weights_out) return fail(FHOG_E_NULL, "one of weights_in and weights_out is NULL");
  if (!a->weights_out) return FHOG_OK;
  if (c.batch * a->heads_q + c.batch * c.heads_k * ((capacity + 1023) / 1024) >= 1 << 24)   // workgroups of the launch that adds them
    return fail(FHOG_E_SHAPE, "weights of more than about 2^34 entries, of all sequences and heads of keys together, are not supported");
  if (const int rc = check_pointer("weights_in", a->weights_in, false)) return rc;
  if (const int rc = check_pointer("weights_out", a->weights_out, false)) return rc;
  if (!rows_apart(c.batch, c.heads_k, 1, capacity, a->stride_wob, a->stride_woh, 0)) return fail(FHOG_E_STRIDE, "rows of an output overlap");
  return FHOG_OK;
}

int validate_key_weights(const fhog_key_weights_args* a) {
  if (!a) return fail(FHOG_E_NULL, "args is NULL");
  if (!dtype_known(a->dtype)) return fail(FHOG_E_DTYPE, "unknown dtype %d", a->dtype);
  if (a->d != 32 && a->d != 64 && a->d != 128) return fail(FHOG_E_SHAPE, "head dim %lld not in {32, 64, 128}", (long long)a->d);
  if (a->batch < 0 || a->batch > 65535 || a->heads_k < 1 || a->heads_k > 65535 || a->heads_q < 1 || a->heads_q > 65535 || a->heads_q % a->heads_k)
    return fail(FHOG_E_SHAPE, "%lld sequences, %lld heads of queries and %lld of keys: expected 65535 or fewer, the heads a multiple", (long long)a->batch, (long long)a->heads_q,
                (long long)a->heads_k);
  if (a->n_q < 1 || a->n_k < 1 || a->n_q > (1 << 24) || a->n_k > (1 << 24)) return fail(FHOG_E_SHAPE, "n_q/n_k out of range");
  if ((a->n_q + 63) / 64 * (a->heads_q / a->heads_k) > kMaxIndex / 2) return fail(FHOG_E_SHAPE, "more than 2^36 queries to a head of keys are not supported");
  if (const int rc = check_mask(a->causal, a->window, a->n_q, a->n_k)) return rc;
  if (const int rc = check_sinks(a->sinks)) return rc;
  if (!isfinite(a->scale)) return fail(FHOG_E_SCALE, "scale is not finite");
  if (a->lengths && a->causal == FHOG_MASK_NONE) return fail(FHOG_E_CAUSAL, "lengths need a causal mask, under which padding comes last");
  if (a->batch == 0) return FHOG_OK;
  if (const int rc = check_strides("q", a->dtype, {a->batch, a->heads_q, a->n_q}, {a->stride_qb, a->stride_qh, a->stride_qn})) return rc;
  if (const int rc = check_strides("k", a->dtype, {a->batch, a->heads_k, a->n_k}, {a->stride_kb, a->stride_kh, a->stride_kn})) return rc;
  if ((a->n_q > 1 && (a->stride_qn < 0 || a->stride_qn > kMaxRowStride)) || (a->n_k > 1 && (a->stride_kn < 0 || a->stride_kn > kMaxRowStride)))
    return fail(FHOG_E_STRIDE, "row stride outside 0..2^24 elements");
  if (const int rc = check_pointer("q", a->q, true)) return rc;
  if (const int rc = check_pointer("k", a->k, true)) return rc;
  if (const int rc = check_pointer("lse", a->lse, false)) return rc;
  if (const int rc = check_pointer("out", a->out, false)) return rc;
  if (a->lengths)
    if (const int rc = check_pointer("lengths", a->lengths, false)) return rc;
  if (!rows_apart(a->batch, a->heads_k, 1, a->n_k, a->stride_ob, a->stride_oh, 0)) return fail(FHOG_E_STRIDE, "rows of an output overlap");
  return FHOG_OK;
}

int validate_evict(const fhog_paged_evict_args* a) {
  if (!a) return fail(FHOG_E_NULL, "args is NULL");
  const fhog_paged_cache& c = a->cache;
  if (const int rc = validate_cache(c, true)) return rc;
  if (a->budget < 1 || a->budget > kMaxEntries) return fail(FHOG_E_PAGED, "budget must be 1 to 2^30 (got %lld)", (long long)a->budget);
  if (a->sinks < 0 || a->recent < 0 || a->sinks > a->budget || a->recent > a->budget - a->sinks)
    return fail(FHOG_E_PAGED, "sinks (%lld) and recent (%lld) must be >= 0 and within the budget (%lld) together", (long long)a->sinks, (long long)a->recent, (long long)a->budget);
  const int64_t capacity = c.page * c.table_width, rows = std::min(a->budget, capacity);
  if (a->into_width < 1 || a->into_width > kMaxEntries / c.page || a->into_width * c.page < rows)
    return fail(FHOG_E_PAGED, "'into' has %lld pages of %lld entries: expected room for %lld", (long long)a->into_width, (long long)c.page, (long long)rows);
  if (rows * (c.d * dtype_bytes(c.dtype) / 16) > kMaxIndex) return fail(FHOG_E_SHAPE, "more than 2^31 - 256 pieces of 16 bytes to a head are not supported");
  if (c.batch == 0) return FHOG_OK;
  const void* ptrs[] = {a->weights, a->into, a->lengths_out, a->kept, a->weights_out};
  const char* names[] = {"weights", "into", "lengths_out", "kept", "weights_out"};
  for (int i = 0; i < 5; i++)
    if (const int rc = check_pointer(names[i], ptrs[i], false)) return rc;
  if (a->weights == a->weights_out) return fail(FHOG_E_PAGED, "weights_out is the array 'weights'");
  if (a->into == c.table) return fail(FHOG_E_PAGED, "'into' is the table of the cache: entries would be written over others that are still to be read");
  if (a->lengths_out == c.lengths) return fail(FHOG_E_PAGED, "lengths_out are the lengths of the cache, which are still being read");
  return FHOG_OK;
}

// Address of `scratch` on the current device, looked up once per device (the first call there) and kept.
constexpr int kMaxDevices = 64;
std::atomic<void*> g_scratch_ptr[kMaxDevices];

int scratch_on_device(void** out) {
  int dev = -1;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return fail(FHOG_E_LAUNCH, "hipGetDevice: HIP error %d (%s)", (int)e, hipGetErrorString(e));
  if (dev < 0 || dev >= kMaxDevices) return fail(FHOG_E_LAUNCH, "device ordinal %d outside 0..%d", dev, kMaxDevices - 1);
  void* ptr = g_scratch_ptr[dev].load(std::memory_order_acquire);
  if (!ptr) {
    e = hipGetSymbolAddress(&ptr, HIP_SYMBOL(scratch));
    if (e != hipSuccess || !ptr)
      return fail(FHOG_E_LAUNCH, "hipGetSymbolAddress(scratch) on device %d: HIP error %d (%s)", dev, (int)e, hipGetErrorString(e));
    g_scratch_ptr[dev].store(ptr, std::memory_order_release);   // concurrent first calls store the same address
  }
  *out = ptr;
  return FHOG_OK;
}

}  // namespace

namespace fhog {
const Tuning& tuning() {
  static const Tuning t = [] {
    Tuning r;
    const char* env = getenv("FHOG_TUNE");
    if (!env) return r;
    char buf[256];
    if (strlen(env) >= sizeof(buf)) fprintf(stderr, "libfhog_hip: FHOG_TUNE is longer than %zu characters; the rest is ignored\n", sizeof(buf) - 1);
    strncpy(buf, env, sizeof(buf) - 1);
    buf[sizeof(buf) - 1] = 0;
    // 0 / 1 switches; anything else is reported and ignored
    const auto flag = [](const char* key, const char* val, int* out) {
      if (!strcmp(val, "0") || !strcmp(val, "1")) *out = val[0] - '0';
      else fprintf(stderr, "libfhog_hip: FHOG_TUNE: value '%s' of '%s' is not 0 or 1; ignored\n", val, key);
    };
    char* save = nullptr;
    for (char* tok = strtok_r(buf, ",", &save); tok; tok = strtok_r(nullptr, ",", &save)) {
      char* eq = strchr(tok, '=');
      if (!eq) {
        fprintf(stderr, "libfhog_hip: FHOG_TUNE: '%s' is not key=value; ignored\n", tok);
        continue;
      }
      *eq = 0;
      const char* val = eq + 1;
      if (!strcmp(tok, "b8")) flag(tok, val, &r.b8);
      else if (!strcmp(tok, "split")) flag(tok, val, &r.split);
      else if (!strcmp(tok, "dd64")) flag(tok, val, &r.dd64);
      else if (!strcmp(tok, "stage64")) flag(tok, val, &r.stage64);
      else if (!strcmp(tok, "stage1")) flag(tok, val, &r.stage1);
      else if (!strcmp(tok, "few")) flag(tok, val, &r.few);
      else if (!strcmp(tok, "small")) {
        if (!strcmp(val, "0") || !strcmp(val, "2") || !strcmp(val, "4")) r.small = val[0] - '0';
        else fprintf(stderr, "libfhog_hip: FHOG_TUNE: small is '0', '2' or '4', not '%s'; ignored\n", val);
      }
      else if (!strcmp(tok, "order")) {
        if (!strcmp(val, "tile")) r.order = 1;
        else if (!strcmp(val, "slice")) r.order = 0;
        else fprintf(stderr, "libfhog_hip: FHOG_TUNE: order is 'slice' or 'tile', not '%s'; ignored\n", val);
      } else {
        fprintf(stderr, "libfhog_hip: FHOG_TUNE: unknown key '%s'; ignored\n", tok);
      }
    }
    return r;
  }();
  return t;
}
}  // namespace fhog

extern "C" {

size_t fhog_attn_args_size(void) { return sizeof(fhog_attn_args); }

int fhog_attn_validate(const fhog_attn_args* args, int backward) { return validate_attn(args, backward); }

int fhog_attn_fwd(const fhog_attn_args* args, void* hip_stream) {
  const int rc = validate_attn(args, 0);
  if (rc != FHOG_OK) return rc;
  const int small = attn_on_16bit_kernels(args) ? small_waves(Small::forward, args) : 0;
  const hipError_t e = small ? fhog::launch_small_attn(to_attn_params(args), false, small, (hipStream_t)hip_stream)
                       : attn_on_16bit_kernels(args) ? fhog::launch_attn_bf16(to_attn_params(args), 0, (hipStream_t)hip_stream)
                                                   : fhog::launch_attn_split(to_attn_params(args), args->dtype, false, (hipStream_t)hip_stream);
  if (e != hipSuccess) return fail(FHOG_E_LAUNCH, "attention forward: HIP error %d (%s)", (int)e, hipGetErrorString(e));
  return FHOG_OK;
}

int fhog_attn_bwd(const fhog_attn_args* args, void* hip_stream) {
  const int rc = validate_attn(args, 1);
  if (rc != FHOG_OK) return rc;
  const fhog::AttnParams p = to_attn_params(args);
  hipError_t e;
  if (!attn_on_16bit_kernels(args)) {
    e = fhog::launch_attn_split(p, args->dtype, true, (hipStream_t)hip_stream);
  } else if (const int small = small_waves(Small::backward, args)) {
    e = fhog::launch_small_attn(p, true, small, (hipStream_t)hip_stream);
  } else {
    e = fhog::launch_attn_bf16(p, 1, (hipStream_t)hip_stream);   // dQ, and the row sums d that the kernel for dK and dV reads
    if (e == hipSuccess) e = fhog::launch_attn_bf16(p, 2, (hipStream_t)hip_stream);
  }
  if (e != hipSuccess) return fail(FHOG_E_LAUNCH, "attention backward: HIP error %d (%s)", (int)e, hipGetErrorString(e));
  return FHOG_OK;
}

size_t fhog_attn_sinks_workspace_bytes(const fhog_attn_args* args, int64_t sinks, int backward) {
  fhog_attn_args a;
  if (!args) return 0;
  a = *args;
  if (backward && !a.ws) a.ws = (float*)a.q;   // not there yet: its size is the question
  if (validate_attn(&a, backward) != FHOG_OK || check_sinks(sinks) != FHOG_OK) return 0;
  return attn_sinks_bytes(&a, sinks, backward);
}

int fhog_attn_fwd_sinks(const fhog_attn_args* args, int64_t sinks, void* ws, int64_t ws_bytes, void* hip_stream) {
  if (const int rc = validate_attn(args, 0)) return rc;
  if (const int rc = check_sinks(sinks)) return rc;
  if (const int rc = check_ws(ws, ws_bytes, attn_sinks_bytes(args, sinks, 0))) return rc;
  const int32_t n = sinks_of(args, sinks);
  if (n == 0) return fhog_attn_fwd(args, hip_stream);
  const hipStream_t s = (hipStream_t)hip_stream;
  fhog::AttnParams p = to_attn_params(args);
  p.sinks = n;
  const int parts = forward_parts(args, n);
  const bool bit16 = attn_on_16bit_kernels(args);
  hipError_t e;
  if (parts > 0) {
    p.n_split = parts, p.part = (float*)ws;
    e = bit16 ? fhog::launch_small_fwd_parts(p, s) : fhog::launch_attn_split_parts(p, args->dtype, false, s);
    if (e == hipSuccess && parts > 1) e = fhog::launch_join_forward(p, args->dtype, s);
  } else if (const int small = bit16 ? sink_small_waves(Small::forward, args) : 0) {
    e = fhog::launch_small_attn(p, false, small, s);
  } else {
    e = bit16 ? fhog::launch_attn_bf16(p, 0, s) : fhog::launch_attn_split(p, args->dtype, false, s);
  }
  if (e != hipSuccess) return fail(FHOG_E_LAUNCH, "attention forward: HIP error %d (%s)", (int)e, hipGetErrorString(e));
  return FHOG_OK;
}

int fhog_attn_bwd_sinks(const fhog_attn_args* args, int64_t sinks, int64_t ws_bytes, void* hip_stream) {
  if (const int rc = validate_attn(args, 1)) return rc;
  if (const int rc = check_sinks(sinks)) return rc;
  if (const int rc = check_ws(args->ws, ws_bytes, attn_sinks_bytes(args, sinks, 1))) return rc;
  const int32_t n = sinks_of(args, sinks);
  if (n == 0) return fhog_attn_bwd(args, hip_stream);
  const hipStream_t s = (hipStream_t)hip_stream;
  fhog::AttnParams p = to_attn_params(args);
  p.sinks = n;
  const int parts = sink_parts(args->batch, n, args->n_q, args->d, dtype_bytes(args->dtype), false);
  float* const part = reinterpret_cast<float*>(reinterpret_cast<char*>(args->ws) + row_bytes(args));
  const bool bit16 = attn_on_16bit_kernels(args);
  const int small = bit16 ? sink_small_waves(Small::backward, args) : 0;
  const bool swept = fhog::rules::sinks_ride(p, dtype_bytes(args->dtype), bit16, small);
  hipError_t e = hipSuccess;
  if (bit16 && !small) e = fhog::launch_attn_bf16(p, 1, s);
  if (swept) p.n_split = parts, p.part = part;
  if (e == hipSuccess)
    e = !bit16 ? fhog::launch_attn_split(p, args->dtype, true, s) : small ? fhog::launch_small_attn(p, true, small, s) : fhog::launch_attn_bf16(p, 2, s);
  if (e == hipSuccess) {
    p.n_split = parts, p.part = swept || parts > 1 ? part : nullptr;
    e = fhog::launch_sink_keys(p, args->dtype, swept, s);
  }
  if (e != hipSuccess) return fail(FHOG_E_LAUNCH, "attention backward: HIP error %d (%s)", (int)e, hipGetErrorString(e));
  return FHOG_OK;
}

size_t fhog_bwdbwd_sinks_workspace_bytes(const fhog_bwdbwd_args* args, int64_t sinks) {
  if (validate(args) != FHOG_OK || check_sinks(sinks) != FHOG_OK) return 0;
  const size_t hint = workspace_hint(args, to_params(args), select_impl(args));
  const int32_t n = sinks_of(args, sinks);
  return n ? ((hint + 15) & ~(size_t)15) + sink_bytes(args->batch, n, args->n_q, args->d, dtype_bytes(args->dtype), true) : hint;
}

int fhog_bwdbwd_sinks(const fhog_bwdbwd_args* args, int64_t sinks, void* hip_stream) {
  if (const int rc = validate(args)) return rc;
  if (const int rc = check_sinks(sinks)) return rc;
  const int32_t n = sinks_of(args, sinks);
  if (n == 0) return fhog_bwdbwd(args, hip_stream);
  if (args->schedule != FHOG_SCHEDULE_FUSED_STATS) return fail(FHOG_E_SCHEDULE, "sinks run under schedule %d alone (got %d)", FHOG_SCHEDULE_FUSED_STATS, args->schedule);
  const size_t of_sinks = sink_bytes(args->batch, n, args->n_q, args->d, dtype_bytes(args->dtype), true);
  if (const int rc = check_ws(args->ws, args->ws_bytes, stats_bytes(args) + of_sinks)) return rc;
  const hipStream_t s = (hipStream_t)hip_stream;
  const int impl = select_impl(args);
  fhog_bwdbwd_args a = *args;   // the sweeps have what lies before the partial results of the sinks, which are a multiple of 16 bytes
  a.ws_bytes = (args->ws_bytes & ~(int64_t)15) - (int64_t)of_sinks;
  fhog::Params p = to_params(&a);
  p.sinks = n, p.n_split_s = sink_parts(a.batch, n, a.n_q, a.d, dtype_bytes(a.dtype), true);
  float* const part = reinterpret_cast<float*>(reinterpret_cast<char*>(a.ws) + a.ws_bytes);
  const int small = impl == FHOG_IMPL_BF16 ? sink_small_waves(Small::double_backward, args) : 0;
  const bool swept = fhog::rules::sinks_ride(p, dtype_bytes(a.dtype), impl == FHOG_IMPL_BF16, small);
  if (swept) p.part_s = part;
  hipError_t e = hipSuccess;
  if (small) {
    e = fhog::launch_small_bwdbwd(p, small, s);
  } else {
    if (const int rc = run_pass(&a, p, impl, FHOG_PASS_DD_B, s)) return rc;
    if (const int rc = impl == FHOG_IMPL_BF16 ? run_grads(&a, p, FHOG_PASS_DQ_DDO, true, s) : run_pass(&a, p, impl, fhog::kPassGrads, s)) return rc;
  }
  p.part_s = swept || p.n_split_s > 1 ? part : nullptr;
  if (e == hipSuccess) e = fhog::launch_sink_keys(p, args->dtype, impl != FHOG_IMPL_BF16, swept, s);
  if (e != hipSuccess) return fail(FHOG_E_LAUNCH, "HIP error %d (%s)", (int)e, hipGetErrorString(e));
  return FHOG_OK;
}

size_t fhog_rotary_args_size(void) { return sizeof(fhog_rotary_args); }

int fhog_rotary_validate(const fhog_rotary_args* args) { return validate_rotary(args); }

int fhog_rotary(const fhog_rotary_args* args, void* hip_stream) {
  if (const int rc = validate_rotary(args)) return rc;
  if (args->batch == 0 || args->n == 0) return FHOG_OK;
  const hipError_t e = fhog::launch_rotary(args, (hipStream_t)hip_stream);
  if (e != hipSuccess) return fail(FHOG_E_LAUNCH, "rotary positions: HIP error %d (%s)", (int)e, hipGetErrorString(e));
  return FHOG_OK;
}

size_t fhog_paged_append_args_size(void) { return sizeof(fhog_paged_append_args); }

int fhog_paged_append_validate(const fhog_paged_append_args* args) { return validate_append(args); }

int fhog_paged_append(const fhog_paged_append_args* args, void* hip_stream) {
  if (const int rc = validate_append(args)) return rc;
  if (args->cache.batch == 0 || args->n == 0) return FHOG_OK;
  const hipError_t e = fhog::launch_paged_append(args, (hipStream_t)hip_stream);
  if (e != hipSuccess) return fail(FHOG_E_LAUNCH, "paged append: HIP error %d (%s)", (int)e, hipGetErrorString(e));
  return FHOG_OK;
}

size_t fhog_paged_attn_args_size(void) { return sizeof(fhog_paged_attn_args); }

int fhog_paged_attn_validate(const fhog_paged_attn_args* args) { return validate_paged_attn(args); }

size_t fhog_paged_attn_workspace_bytes(const fhog_paged_attn_args* args) { return validate_paged_attn(args) == FHOG_OK && args->cache.batch ? fhog::paged_attn_bytes(args) : 0; }

int fhog_paged_attn(const fhog_paged_attn_args* args, void* hip_stream) {
  if (const int rc = validate_paged_attn(args)) return rc;
  if (args->cache.batch == 0) return FHOG_OK;
  if (const int rc = check_ws(args->ws, args->ws_bytes, fhog::paged_attn_bytes(args))) return rc;
  const hipError_t e = fhog::launch_paged_attn(args, (hipStream_t)hip_stream);
  if (e != hipSuccess) return fail(FHOG_E_LAUNCH, "paged attention: HIP error %d (%s)", (int)e, hipGetErrorString(e));
  return FHOG_OK;
}

size_t fhog_key_weights_args_size(void) { return sizeof(fhog_key_weights_args); }

int fhog_key_weights_validate(const fhog_key_weights_args* args) { return validate_key_weights(args); }

size_t fhog_key_weights_workspace_bytes(const fhog_key_weights_args* args) { return validate_key_weights(args) == FHOG_OK && args->batch ? fhog::key_weights_bytes(args) : 0; }

int fhog_key_weights(const fhog_key_weights_args* args, void* hip_stream) {
  if (const int rc = validate_key_weights(args)) return rc;
  if (args->batch == 0) return FHOG_OK;
  if (const int rc = check_ws(args->ws, args->ws_bytes, fhog::key_weights_bytes(args))) return rc;
  const hipError_t e = fhog::launch_key_weights(args, (hipStream_t)hip_stream);
  if (e != hipSuccess) return fail(FHOG_E_LAUNCH, "weights of keys: HIP error %d (%s)", (int)e, hipGetErrorString(e));
  return FHOG_OK;
}

size_t fhog_paged_evict_args_size(void) { return sizeof(fhog_paged_evict_args); }

int fhog_paged_evict_validate(const fhog_paged_evict_args* args) { return validate_evict(args); }

int fhog_paged_evict(const fhog_paged_evict_args* args, void* hip_stream) {
  if (const int rc = validate_evict(args)) return rc;
  if (args->cache.batch == 0) return FHOG_OK;
  const hipError_t e = fhog::launch_paged_evict(args, (hipStream_t)hip_stream);
  if (e != hipSuccess) return fail(FHOG_E_LAUNCH, "paged eviction: HIP error %d (%s)", (int)e, hipGetErrorString(e));
  return FHOG_OK;
}

int fhog_abi_version(void) { return FHOG_ABI_VERSION; }

size_t fhog_bwdbwd_args_size(void) { return sizeof(fhog_bwdbwd_args); }

size_t fhog_bwdbwd_workspace_bytes(int64_t batch, int64_t n_q) {
  if (batch < 0 || n_q < 0) return 0;
  return (size_t)3 * (size_t)batch * (size_t)n_q * sizeof(float);
}

size_t fhog_bwdbwd_workspace_hint(const fhog_bwdbwd_args* args) {
  if (validate(args) != FHOG_OK) return 0;
  return workspace_hint(args, to_params(args), select_impl(args));
}

int fhog_validate(const fhog_bwdbwd_args* args) { return validate(args); }

int fhog_select_impl(const fhog_bwdbwd_args* args) {
  const int rc = validate(args);
  if (rc != FHOG_OK) return rc;
  return select_impl(args);
}

int fhog_bwdbwd_pass(const fhog_bwdbwd_args* args, int pass, void* hip_stream) {
  const int rc = validate(args);
  if (rc != FHOG_OK) return rc;
  if (pass < FHOG_PASS_D || pass > FHOG_PASS_STAGE1) return fail(FHOG_E_PASS, "unknown pass %d", pass);
  const fhog::Params p = to_params(args);
  return run_pass(args, p, select_impl(args), pass, (hipStream_t)hip_stream);
}

int fhog_bwdbwd(const fhog_bwdbwd_args* args, void* hip_stream) {
  const int rc = validate(args);
  if (rc != FHOG_OK) return rc;
  const fhog::Params p = to_params(args);
  const int impl = select_impl(args);
  // Small launches: the default schedule in two launches. The schedules that take ddO out of the third sweep do the same as long as
  // that is one round of the CUs (us, 2 x 86, d = 64: 41 -> 13), their own sweeps beyond.
  int small = 0;
  if (impl == FHOG_IMPL_BF16 && (args->schedule == FHOG_SCHEDULE_FUSED_STATS ||
                                 (args->schedule != FHOG_SCHEDULE_FOUR_PASS && ((args->n_q + 127) / 128 + (args->n_k + 127) / 128) * args->batch <= 128)))
    small = small_waves(Small::double_backward, args->batch, args->n_q, args->n_k, args->d, args->causal, args->window);
  if (small) {
    const hipError_t e = fhog::launch_small_bwdbwd(p, small, (hipStream_t)hip_stream);
    if (e != hipSuccess) return fail(FHOG_E_LAUNCH, "HIP error %d (%s)", (int)e, hipGetErrorString(e));
    return FHOG_OK;
  }
  // Pass sequences. The first statistics sweep writes d_i itself: no separate launch for it.
  // The schedules that take ddO out of the third sweep exist in the 16-bit family; the split-product family runs the
  // fused one for them.
  // The last sweep of a sequence shares its launch with pass 4, stage 1 apart, which pass 4 follows in one of its own.
  static const int four[] = {FHOG_PASS_DD, FHOG_PASS_B, FHOG_PASS_DQ_DDO, 0};
  static const int stage1[] = {FHOG_PASS_STAGE1, FHOG_PASS_DK_DV, 0};
  static const int fused[] = {FHOG_PASS_DD_B, FHOG_PASS_DQ_DDO, 0};
  static const int ddo_early[] = {FHOG_PASS_DD, FHOG_PASS_B_DDO, FHOG_PASS_DQ, 0};
  static const int three[] = {FHOG_PASS_DD_B_DDO, FHOG_PASS_DQ, 0};
  const int* order = four;
  const bool split_products = impl != FHOG_IMPL_BF16;
  // d = 64, launch large enough to fill the GPU: the reference's own arrangement of its four passes, sweeps 1-3 in one launch
  if (args->schedule == FHOG_SCHEDULE_FOUR_PASS && impl == FHOG_IMPL_BF16 && args->d == 64 && fhog::tuning().stage1 != 0 &&
      granted_split(args, impl, FHOG_PASS_DQ_DDO) == 1 && granted_split(args, impl, FHOG_PASS_DD) == 1)
    order = stage1;
  if (args->schedule == FHOG_SCHEDULE_FUSED_STATS || (split_products && args->schedule != FHOG_SCHEDULE_FOUR_PASS)) order = fused;
  const bool splits = splits_instead(args, p, impl);
  if (args->schedule == FHOG_SCHEDULE_THREE_SWEEP && splits) order = fused;
  if (args->schedule == FHOG_SCHEDULE_DDO_EARLY && impl == FHOG_IMPL_BF16 && !splits) order = ddo_early;
  if (args->schedule == FHOG_SCHEDULE_THREE_SWEEP && impl == FHOG_IMPL_BF16 && !splits) order = three;
  for (; *order; order++) {
    const bool last_two = *order == FHOG_PASS_DQ_DDO || *order == FHOG_PASS_DQ;
    const int r = !last_two ? run_pass(args, p, impl, *order, (hipStream_t)hip_stream)
                  : split_products ? run_pass(args, p, impl, fhog::kPassGrads, (hipStream_t)hip_stream)
                                   : run_grads(args, p, *order, true, (hipStream_t)hip_stream);
    if (r != FHOG_OK) return r;
  }
  return FHOG_OK;
}

int fhog_bwdbwd_static_ws(const fhog_bwdbwd_args* args, void* hip_stream) {
  if (!args) return fail(FHOG_E_NULL, "args is NULL");
  void* ws = nullptr;
  if (const int rc = scratch_on_device(&ws)) return rc;
  fhog_bwdbwd_args a = *args;   // the caller's ws / ws_bytes are not read
  a.ws = static_cast<float*>(ws);
  a.ws_bytes = 0;
  if (const int rc = validate(&a)) return rc;
  const size_t need = fhog_bwdbwd_workspace_bytes(a.batch, a.n_q);
  if (need > (size_t)FHOG_STATIC_WS_BYTES)
    return fail(FHOG_E_SHAPE,
                "fhog_bwdbwd_static_ws: batch*n_q = %lld rows need %zu bytes of row statistics, the static workspace holds %zu "
                "(at most %zu rows); use fhog_bwdbwd with a caller-owned workspace",
                (long long)(a.batch * a.n_q), need, (size_t)FHOG_STATIC_WS_BYTES, (size_t)FHOG_STATIC_WS_BYTES / 12);
  a.ws_bytes = FHOG_STATIC_WS_BYTES;   // small launches split their streamed side as far as the rest of the array allows
  return fhog_bwdbwd(&a, hip_stream);
}

size_t fhog_static_ws_bytes(void) { return (size_t)FHOG_STATIC_WS_BYTES; }

int fhog_probe_mfma_rate(float* out, int blocks, int trips, int data_mode, double* flops, void* hip_stream) {
  if (!out || !flops) return fail(FHOG_E_NULL, "out or flops is NULL");
  const int mix = data_mode & 7, waves = (data_mode & 8) ? 4 : 8;
  if (blocks < 1 || blocks > 65535 || trips < 1 || data_mode < 0 || data_mode > 13 || mix > 5)
    return fail(FHOG_E_SHAPE, "blocks in 1..65535, trips >= 1, data_mode 0..5 or 8..13");
  const hipError_t e = fhog::launch_mfma_rate(out, blocks, trips, mix, waves, (hipStream_t)hip_stream);
  if (e != hipSuccess) return fail(FHOG_E_LAUNCH, "MFMA rate probe: HIP error %d (%s)", (int)e, hipGetErrorString(e));
  *flops = (double)blocks * waves * trips * 32.0 * 32768.0;
  return FHOG_OK;
}

const char* fhog_last_error(void) { return g_err; }

}  // extern "C"
