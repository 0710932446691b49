// GQA attention of a batch of streams that share a long prefix (sm_100a).
//
// Every stream b has its own static cache (rows [0, kv_len[b])) and all of them
// read the same prefix rows [0, prefix_len) first.  With query head hq and KV
// head h = hq / G,
//     out = softmax_j(scale * q . k_j) v_j   over the prefix rows, then the own rows;
// a query that sees no row gets zeros.  Two forms:
//   * decode: one query per stream, which sees all of its own valid rows, and
//     optionally scores[b, h, j] += sum over the group of its weight on row j;
//   * prefill: query i < q_len[b] is the stream's own row kv_len[b] - q_len[b] + i
//     and sees its own rows up to that one; queries past q_len[b] get zeros.
//
// One block per (query, KV head, stream), one warp per query head: every lane
// holds D / 32 dims of the query and of the running weighted sum (fp32), and a
// warp walks the rows with an online softmax (running maximum and sum).
#include <algorithm>

#include "common.cuh"

namespace kani {
namespace {

struct PrefixAttnParams {
  const void* q;
  int64_t qb, qt, qh;  // strides of q [B, T, Hq, D]
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
  int64_t ob, ot, oh;
  int32_t* err;
  int group, tokens;
};

// a length read on the device, held to [0, most] and flagged where it was outside
__device__ __forceinline__ int64_t checked_len(int64_t n, int64_t most, int32_t* err, bool tell) {
  if ((n > most || n < 0) && tell && err != nullptr) atomicOr(err, KANI_FLAG_SLOT_OOB);
  return n < 0 ? 0 : (n > most ? most : n);
}

template <typename T, int D>
__global__ void prefix_attn_kernel(PrefixAttnParams p) {
  constexpr int E = D / 32;
  const int t = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __shared__ float s_m[8], s_l[8];
  const bool tell = threadIdx.x == 0 && t == 0 && h == 0;
  const int64_t plen = p.prefix_len ? checked_len(*p.prefix_len, p.prefix_rows, p.err, tell && b == 0) : p.prefix_rows;
  int64_t own = checked_len(p.kv_len[b], p.cache_len, p.err, tell);
  const int64_t ql = p.q_len ? checked_len(p.q_len[b], p.tokens, p.err, tell) : p.tokens;
  T* o = static_cast<T*>(p.out) + b * p.ob + (int64_t)t * p.ot + (int64_t)(h * p.group + warp) * p.oh + lane * E;
  if (t >= ql) {
    for (int e = 0; e < E; ++e) o[e] = Elem<T>::from_f(0.f);
    return;
  }
  if (p.tokens > 1 || p.q_len) {
    if (own < ql && tell && p.err) atomicOr(p.err, KANI_FLAG_SLOT_OOB);
    own = min(own, max(own - ql, (int64_t)0) + t + 1);
  }
  const T* q = static_cast<const T*>(p.q) + b * p.qb + (int64_t)t * p.qt + (int64_t)(h * p.group + warp) * p.qh + lane * E;
  const T* pk = static_cast<const T*>(p.pk) + h * p.ph + lane * E;
  const T* pv = static_cast<const T*>(p.pv) + h * p.ph + lane * E;
  const T* k = static_cast<const T*>(p.k) + b * p.cb + h * p.ch + lane * E;
  const T* v = static_cast<const T*>(p.v) + b * p.cb + h * p.ch + lane * E;
  float qf[E], acc[E];
  for (int e = 0; e < E; ++e) {
    qf[e] = Elem<T>::to_f(q[e]) * p.qscale;
    acc[e] = 0.f;
  }
  auto dot = [&](const T* row) {
    float s = 0.f;
    for (int e = 0; e < E; ++e) s = fmaf(qf[e], Elem<T>::to_f(row[e]), s);
    for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    return s;
  };
  float m = -INFINITY, l = 0.f;
  for (int64_t j = 0; j < plen + own; ++j) {
    const float s = dot(j < plen ? pk + j * p.ps : k + (j - plen) * p.cs);
    const T* vr = j < plen ? pv + j * p.ps : v + (j - plen) * p.cs;
    const float mn = fmaxf(m, s), corr = m == -INFINITY ? 0.f : exp2f(m - mn), w = exp2f(s - mn);
    l = fmaf(l, corr, w);
    for (int e = 0; e < E; ++e) acc[e] = fmaf(acc[e], corr, w * Elem<T>::to_f(vr[e]));
    m = mn;
  }
  for (int e = 0; e < E; ++e) o[e] = Elem<T>::from_f(l == 0.f ? 0.f : acc[e] / l);
  if (p.scores == nullptr) return;
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
  __syncthreads();
  float* sc = p.scores + b * p.sb + h * p.sh;
  for (int64_t j = warp; j < own; j += p.group) {
    float add = 0.f;
    for (int g = 0; g < p.group; ++g) {
      const T* qg = static_cast<const T*>(p.q) + b * p.qb + (int64_t)(h * p.group + g) * p.qh + lane * E;
      for (int e = 0; e < E; ++e) qf[e] = Elem<T>::to_f(qg[e]) * p.qscale;
      add += exp2f(dot(k + j * p.cs) - s_m[g]) / s_l[g];
    }
    if (lane == 0) sc[j] += add;
  }
}

int prefix_attention(int32_t dtype, int64_t batch, int64_t tokens, int32_t num_q_heads, int32_t num_kv_heads,
                     int32_t head_dim, PrefixAttnParams p, float scale, void* workspace, int64_t workspace_bytes,
                     void* stream) {
  if (batch < 0 || tokens < 0 || num_q_heads < 0 || num_kv_heads < 0 || head_dim < 0 || p.cache_len < 0 ||
      p.prefix_rows < 0 || workspace_bytes < 0)
    return KANI_ERR_INVALID_ARG;
  if (batch == 0 || tokens == 0 || num_q_heads == 0) return KANI_OK;
  if (num_kv_heads == 0 || num_q_heads % num_kv_heads != 0 || !p.q || !p.kv_len || !p.out ||
      (p.cache_len > 0 && (!p.k || !p.v)) || (p.prefix_rows > 0 && (!p.pk || !p.pv)) || !(scale >= 0.f) ||
      scale > 3.0e38f)
    return KANI_ERR_INVALID_ARG;
  if (dtype != KANI_DTYPE_BF16 && dtype != KANI_DTYPE_F16)
    return dtype == KANI_DTYPE_F32 ? KANI_ERR_UNSUPPORTED : KANI_ERR_DTYPE;
  p.group = num_q_heads / num_kv_heads;
  p.tokens = (int)tokens;
  if ((head_dim != 64 && head_dim != 128) || p.group > 8 || batch > 65535 || num_kv_heads > 65535 ||
      tokens > (1 << 24) || p.cache_len > (1 << 30) || p.prefix_rows > (1 << 30))
    return KANI_ERR_UNSUPPORTED;
  const int64_t st[] = {p.qb, p.qt, p.qh, p.cb, p.ch, p.cs, p.ph, p.ps, p.ob, p.ot, p.oh};
  for (int64_t x : st)
    if (x % 8 != 0) return KANI_ERR_UNSUPPORTED;
  for (const void* x : {p.q, p.k, p.v, p.pk, p.pv, (const void*)p.out})
    if (!aligned16(x)) return KANI_ERR_UNSUPPORTED;
  p.qscale = scale * 1.4426950408889634f;
  const dim3 grid((unsigned)tokens, (unsigned)num_kv_heads, (unsigned)batch);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto go = [&]<typename T>() {
    if (head_dim == 64) prefix_attn_kernel<T, 64><<<grid, 32 * p.group, 0, s>>>(p);
    else prefix_attn_kernel<T, 128><<<grid, 32 * p.group, 0, s>>>(p);
    return launch_status();
  };
  return dtype == KANI_DTYPE_BF16 ? go.template operator()<__nv_bfloat16>() : go.template operator()<__half>();
}

}  // namespace
}  // namespace kani

extern "C" int64_t kani_prefix_decode_workspace(int64_t batch, int32_t num_q_heads, int32_t num_kv_heads,
                                                int32_t head_dim, int64_t cache_len, int64_t prefix_rows,
                                                int32_t with_scores) {
  return 0;
}

extern "C" int64_t kani_prefix_prefill_workspace(int64_t batch, int64_t tokens, int32_t num_q_heads,
                                                 int32_t num_kv_heads, int32_t head_dim, int64_t cache_len,
                                                 int64_t prefix_rows) {
  return 0;
}

extern "C" int kani_prefix_decode_attention(
    int32_t dtype, int64_t batch, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, const void* q,
    int64_t q_batch_stride, int64_t q_head_stride, const void* k_cache, const void* v_cache,
    int64_t cache_batch_stride, int64_t cache_head_stride, int64_t cache_slot_stride, int64_t cache_len,
    const int64_t* kv_len, const void* prefix_k, const void* prefix_v, int64_t prefix_head_stride,
    int64_t prefix_row_stride, int64_t prefix_rows, const int64_t* prefix_len, float scale, float* scores,
    int64_t scores_batch_stride, int64_t scores_head_stride, void* out, int64_t out_batch_stride,
    int64_t out_head_stride, void* workspace, int64_t workspace_bytes, int32_t* err_flag, void* stream) {
  kani::PrefixAttnParams p = {};
  p.q = q;
  p.qb = q_batch_stride;
  p.qh = q_head_stride;
  p.k = k_cache;
  p.v = v_cache;
  p.cb = cache_batch_stride;
  p.ch = cache_head_stride;
  p.cs = cache_slot_stride;
  p.cache_len = cache_len;
  p.kv_len = kv_len;
  p.pk = prefix_k;
  p.pv = prefix_v;
  p.ph = prefix_head_stride;
  p.ps = prefix_row_stride;
  p.prefix_rows = prefix_rows;
  p.prefix_len = prefix_len;
  p.scores = scores;
  p.sb = scores_batch_stride;
  p.sh = scores_head_stride;
  p.out = out;
  p.ob = out_batch_stride;
  p.oh = out_head_stride;
  p.err = err_flag;
  return kani::prefix_attention(dtype, batch, 1, num_q_heads, num_kv_heads, head_dim, p, scale, workspace,
                                workspace_bytes, stream);
}

extern "C" int kani_prefix_prefill_attention(
    int32_t dtype, int64_t batch, int64_t tokens, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
    const void* q, int64_t q_batch_stride, int64_t q_token_stride, int64_t q_head_stride, const void* k_cache,
    const void* v_cache, int64_t cache_batch_stride, int64_t cache_head_stride, int64_t cache_slot_stride,
    int64_t cache_len, const int64_t* kv_len, const int64_t* q_len, const void* prefix_k, const void* prefix_v,
    int64_t prefix_head_stride, int64_t prefix_row_stride, int64_t prefix_rows, const int64_t* prefix_len,
    float scale, void* out, int64_t out_batch_stride, int64_t out_token_stride, int64_t out_head_stride,
    void* workspace, int64_t workspace_bytes, int32_t* err_flag, void* stream) {
  kani::PrefixAttnParams p = {};
  p.q = q;
  p.qb = q_batch_stride;
  p.qt = q_token_stride;
  p.qh = q_head_stride;
  p.k = k_cache;
  p.v = v_cache;
  p.cb = cache_batch_stride;
  p.ch = cache_head_stride;
  p.cs = cache_slot_stride;
  p.cache_len = cache_len;
  p.kv_len = kv_len;
  p.q_len = q_len;
  p.pk = prefix_k;
  p.pv = prefix_v;
  p.ph = prefix_head_stride;
  p.ps = prefix_row_stride;
  p.prefix_rows = prefix_rows;
  p.prefix_len = prefix_len;
  p.out = out;
  p.ob = out_batch_stride;
  p.ot = out_token_stride;
  p.oh = out_head_stride;
  p.err = err_flag;
  return kani::prefix_attention(dtype, batch, tokens, num_q_heads, num_kv_heads, head_dim, p, scale, workspace,
                                workspace_bytes, stream);
}
