// Shared pieces of the shared-prefix attention kernels (prefix_decode.cu,
// prefix_prefill.cu): the call's parameters, their host checks and the online
// softmax's small functions.
#pragma once

#include <atomic>

#include "common.cuh"

namespace kani {
namespace prefix {

// Grants a kernel its most dynamic shared memory on the current device, once per
// device (the call costs about a microsecond); 0 or a cudaError_t.
template <typename Kernel>
int grant_smem(Kernel kern, size_t bytes, std::atomic<uint64_t>& granted) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0) dev = 63;
  const uint64_t bit = 1ull << (dev & 63);
  if (dev < 63 && (granted.load(std::memory_order_relaxed) & bit)) return 0;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e != cudaSuccess) return (int)e;
  granted.fetch_or(bit, std::memory_order_relaxed);
  return 0;
}

struct Params {
  const void* q;
  int64_t qb, qt, qh;  // strides of q [B, T, Hq, D] (T = 1 in the decode form)
  const void* k;
  const void* v;
  int64_t cb, ch, cs;  // strides of the caches [B, Hk, S, D]
  int64_t cache_len;
  const int64_t* kv_len;
  const int64_t* q_len;  // prefill: valid queries per stream (NULL: all of them)
  const void* pk;
  const void* pv;
  int64_t ph, ps;  // strides of the prefix [Hk, P, D]
  int64_t prefix_rows;
  const int64_t* prefix_len;  // NULL: prefix_rows
  float qscale;               // scale * log2(e)
  float* scores;
  int64_t sb, sh;  // strides of scores [B, Hk, S]
  void* out;
  int64_t ob, ot, oh;  // strides of out [B, T, Hq, D]
  int32_t* err;
  int batch, tokens, hq, hk, group;
};

// What both entry points refuse, and the strides of dimensions of one element,
// which are never followed, set to 0.
inline int check_params(Params& p, int32_t dtype, int64_t batch, int64_t tokens, int32_t hq, int32_t hk, int32_t d,
                        float scale) {
  if (hk == 0 || hq % hk != 0 || !p.q || !p.kv_len || !p.out || (p.cache_len > 0 && (!p.k || !p.v)) ||
      (p.prefix_rows > 0 && (!p.pk || !p.pv)) || !(scale >= 0.f) || scale > 3.0e38f)
    return KANI_ERR_INVALID_ARG;
  if (dtype != KANI_DTYPE_BF16 && dtype != KANI_DTYPE_F16)
    return dtype == KANI_DTYPE_F32 ? KANI_ERR_UNSUPPORTED : KANI_ERR_DTYPE;
  if ((d != 64 && d != 128) || hq / hk > 8 || batch > 65535 || hk > 65535 || tokens > (1 << 24) ||
      p.cache_len > (1 << 30) || p.prefix_rows > (1 << 30))
    return KANI_ERR_UNSUPPORTED;
  if (batch == 1) p.qb = p.cb = p.sb = p.ob = 0;
  if (tokens == 1) p.qt = p.ot = 0;
  if (hq == 1) p.qh = p.oh = 0;
  if (hk == 1) p.ch = p.ph = p.sh = 0;
  if (p.cache_len <= 1) p.cs = 0;
  if (p.prefix_rows <= 1) p.ps = 0;
  // rows, heads and queries that are one and the same memory make no tensor map
  if ((p.cs == 0 && p.cache_len > 1) || (p.ps == 0 && p.prefix_rows > 1) || (p.qh == 0 && hq > 1) ||
      (p.qt == 0 && tokens > 1))
    return KANI_ERR_UNSUPPORTED;
  for (int64_t x : {p.qb, p.qt, p.qh, p.cb, p.ch, p.cs, p.ph, p.ps, p.ob, p.ot, p.oh})
    if (x % 8 != 0) return KANI_ERR_UNSUPPORTED;
  for (const void* x : {p.q, p.k, p.v, p.pk, p.pv, (const void*)p.out})
    if (!aligned16(x)) return KANI_ERR_UNSUPPORTED;
  p.batch = (int)batch;
  p.tokens = (int)tokens;
  p.hq = hq;
  p.hk = hk;
  p.group = hq / hk;
  // 0 times an infinite (masked) logit has to stay infinite
  p.qscale = scale > 1e-30f ? scale * 1.4426950408889634f : 1e-30f;
  return KANI_OK;
}

// a length read on the device, held to [0, most] and flagged where it was outside
__device__ __forceinline__ int checked_len(int64_t n, int64_t most, int32_t* err, bool tell) {
  if ((n > most || n < 0) && tell && err != nullptr) atomicOr(err, KANI_FLAG_SLOT_OOB);
  return (int)(n < 0 ? 0 : (n > most ? most : n));
}

// 2^x with the hardware approximation (ex2.approx: relative error ~2^-22)
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// factor that brings sums relative to the maximum m to the maximum mnew; the empty
// sum's m is -inf
__device__ __forceinline__ float merge_weight(float m, float mnew) {
  return m == -INFINITY ? 0.f : ex2(m - mnew);
}

}  // namespace prefix
}  // namespace kani
