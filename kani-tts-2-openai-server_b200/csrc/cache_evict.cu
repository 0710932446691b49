// Eviction from the static KV caches by accumulated attention weight (sm_100a).
//
// For every stream b and KV head h with n = kv_len[b] > budget rows, keep
//   * the first `protect` rows and the last `recent` rows,
//   * of the rows between, the budget - protect - recent with the highest
//     scores[b, h, j] (ties: the lowest slot; NaN counts as the lowest score),
// and move them, in slot order, to rows [0, budget) of the destination caches (the
// caches themselves, or others).  Scores move along; those past the new length
// become zero.  K / V rows past the new length stay as they were.  Streams of at
// most `budget` rows keep all of them.
//
// One block per (b, h).  The lowest kept score is found by a binary search over
// its bits; a scan over the slots then gives every kept row its destination.  In
// place, row i comes from a slot >= i, so each step of 256 rows is read before
// any of it is written, and no later step reads what it wrote.
#include "common.cuh"

namespace kani {
namespace {

constexpr int kEvictThreads = 256;

struct EvictParams {
  const void* k;
  const void* v;
  int64_t cb, ch, cs;  // byte strides of the caches [B, Hk, S, D]
  int64_t cache_len;
  const float* scores;
  int64_t sb, sh;
  const int64_t* kv_len;
  int64_t budget, recent, protect;
  void* k_out;
  void* v_out;
  int64_t cbo, cho, cso;
  float* scores_out;
  int64_t sbo, sho;
  int64_t out_len;
  int64_t* len_out;
  int32_t* kept;  // [B, Hk, budget] or NULL
  int row_vecs;   // 16-byte vectors per row
  int32_t* err;
};

// a score's bits in an order where unsigned comparison is the score's; NaN lowest
__device__ __forceinline__ uint32_t score_key(float f) {
  if (isnan(f)) return 0u;
  const uint32_t u = __float_as_uint(f + 0.f);  // -0 -> +0
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

__device__ int block_sum(int x, int* red) {
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = x;
  __syncthreads();
  int s = 0;
  for (int w = 0; w < kEvictThreads / 32; ++w) s += red[w];
  __syncthreads();
  return s;
}

// exclusive prefix sum of a flag over the block, and the block's total
__device__ int block_rank(bool f, int* red, int& total) {
  const unsigned m = __ballot_sync(0xffffffffu, f);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (lane == 0) red[warp] = __popc(m);
  __syncthreads();
  int before = 0;
  total = 0;
  for (int w = 0; w < kEvictThreads / 32; ++w) {
    if (w < warp) before += red[w];
    total += red[w];
  }
  __syncthreads();
  return before + __popc(m & ((1u << lane) - 1u));
}

__global__ void __launch_bounds__(kEvictThreads) cache_evict_kernel(EvictParams p) {
  __shared__ int red[kEvictThreads / 32];
  __shared__ int s_src[kEvictThreads];
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  int64_t n = p.kv_len[b];
  if ((n < 0 || n > p.cache_len) && h == 0 && tid == 0 && p.err) atomicOr(p.err, KANI_FLAG_SLOT_OOB);
  n = n < 0 ? 0 : (n > p.cache_len ? p.cache_len : n);
  const float* sc = p.scores + b * p.sb + h * p.sh;
  const int64_t keep = n < p.budget ? n : p.budget;
  const int64_t lo = n > p.budget ? p.protect : n, hi = n > p.budget ? n - p.recent : n;
  const int64_t most = n > p.budget ? p.budget - p.protect - p.recent : 0;
  // the largest threshold that at least `most` of the rows between reach
  uint32_t thr = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t t = thr | (1u << bit);
    int c = 0;
    for (int64_t j = lo + tid; j < hi; j += kEvictThreads) c += score_key(sc[j]) >= t;
    if (block_sum(c, red) >= most) thr = t;
  }
  int above = 0;
  for (int64_t j = lo + tid; j < hi; j += kEvictThreads) above += score_key(sc[j]) > thr;
  const int64_t ties = most - block_sum(above, red);  // rows at the threshold that stay
  int64_t dst0 = 0, tie0 = 0;
  for (int64_t j0 = 0; j0 < n; j0 += kEvictThreads) {
    const int64_t j = j0 + tid;
    const bool in = j < n, mid = in && j >= lo && j < hi;
    const uint32_t key = mid ? score_key(sc[j]) : 0u;
    int total;
    const bool tie = mid && key == thr;
    const int tr = block_rank(tie, red, total);
    const bool stay = in && (!mid || key > thr || (tie && tie0 + tr < ties));
    tie0 += total;
    const int rank = block_rank(stay, red, total);
    if (stay) s_src[rank] = (int)j;
    __syncthreads();
    const bool row = tid < total;
    const int64_t src = row ? s_src[tid] : 0, dst = dst0 + tid;
    for (int c = 0; c < 2 * p.row_vecs; ++c) {
      const int vec = c >> 1;
      const char* in_ = static_cast<const char*>(c & 1 ? p.v : p.k) + b * p.cb + h * p.ch + src * p.cs + vec * 16;
      char* out_ = static_cast<char*>(c & 1 ? p.v_out : p.k_out) + b * p.cbo + h * p.cho + dst * p.cso + vec * 16;
      uint4 x;
      if (row) x = ld16(in_);
      __syncthreads();
      if (row) st16(out_, x);
    }
    const float f = row ? sc[src] : 0.f;
    __syncthreads();
    if (row) {
      p.scores_out[b * p.sbo + h * p.sho + dst] = f;
      if (p.kept) p.kept[((int64_t)b * gridDim.x + h) * p.budget + dst] = (int32_t)src;
    }
    dst0 += total;
    __syncthreads();
  }
  for (int64_t j = keep + tid; j < p.out_len; j += kEvictThreads) p.scores_out[b * p.sbo + h * p.sho + j] = 0.f;
  if (p.kept)
    for (int64_t j = keep + tid; j < p.budget; j += kEvictThreads)
      p.kept[((int64_t)b * gridDim.x + h) * p.budget + j] = -1;
  if (h == 0 && tid == 0) p.len_out[b] = keep;
}

}  // namespace
}  // namespace kani

extern "C" int kani_cache_evict(int32_t dtype, int64_t batch, int32_t num_kv_heads, int32_t head_dim,
                                const void* k_cache, const void* v_cache, int64_t cache_batch_stride,
                                int64_t cache_head_stride, int64_t cache_slot_stride, int64_t cache_len,
                                const float* scores, int64_t scores_batch_stride, int64_t scores_head_stride,
                                const int64_t* kv_len, int64_t budget, int64_t recent, int64_t protect, void* k_out,
                                void* v_out, int64_t out_batch_stride, int64_t out_head_stride,
                                int64_t out_slot_stride, int64_t out_len, float* scores_out,
                                int64_t scores_out_batch_stride, int64_t scores_out_head_stride, int64_t* len_out,
                                int32_t* kept_out, int32_t* err_flag, void* stream) {
  using namespace kani;
  if (batch < 0 || num_kv_heads < 0 || head_dim < 0 || cache_len < 0 || out_len < 0 || budget < 0 || recent < 0 ||
      protect < 0 || recent > budget || protect > budget - recent || budget > out_len)
    return KANI_ERR_INVALID_ARG;
  if (dtype != KANI_DTYPE_F32 && dtype != KANI_DTYPE_BF16 && dtype != KANI_DTYPE_F16) return KANI_ERR_DTYPE;
  if (batch == 0 || num_kv_heads == 0) return KANI_OK;
  const int es = dtype == KANI_DTYPE_F32 ? 4 : 2;
  const bool rows = cache_len > 0 && out_len > 0 && head_dim > 0;
  if (!kv_len || !len_out || kv_len == len_out ||
      (rows && (!k_cache || !v_cache || !k_out || !v_out || !scores || !scores_out || k_cache == v_cache || k_out == v_out)))
    return KANI_ERR_INVALID_ARG;
  // in place is all of k, v and scores in place
  const bool in_place = rows && k_out == k_cache;
  if (rows && ((v_out == v_cache) != in_place || (scores_out == scores) != in_place)) return KANI_ERR_INVALID_ARG;
  if (in_place && (out_batch_stride != cache_batch_stride || out_head_stride != cache_head_stride ||
                   out_slot_stride != cache_slot_stride || out_len != cache_len ||
                   scores_out_batch_stride != scores_batch_stride || scores_out_head_stride != scores_head_stride))
    return KANI_ERR_INVALID_ARG;
  const int64_t st[] = {cache_batch_stride, cache_head_stride, cache_slot_stride,
                        out_batch_stride,   out_head_stride,   out_slot_stride};
  for (int64_t x : st)
    if (x * es % 16 != 0) return KANI_ERR_UNSUPPORTED;
  if ((int64_t)head_dim * es % 16 != 0 || head_dim > 256 || batch > 65535 || num_kv_heads > 65535 ||
      cache_len > (1 << 30) || out_len > (1 << 30) || !aligned16(k_cache) || !aligned16(v_cache) ||
      !aligned16(k_out) || !aligned16(v_out))
    return KANI_ERR_UNSUPPORTED;
  EvictParams p = {};
  p.k = k_cache;
  p.v = v_cache;
  p.cb = cache_batch_stride * es;
  p.ch = cache_head_stride * es;
  p.cs = cache_slot_stride * es;
  p.cache_len = cache_len;
  p.scores = scores;
  p.sb = scores_batch_stride;
  p.sh = scores_head_stride;
  p.kv_len = kv_len;
  p.budget = budget;
  p.recent = recent;
  p.protect = protect;
  p.k_out = k_out;
  p.v_out = v_out;
  p.cbo = out_batch_stride * es;
  p.cho = out_head_stride * es;
  p.cso = out_slot_stride * es;
  p.scores_out = scores_out;
  p.sbo = scores_out_batch_stride;
  p.sho = scores_out_head_stride;
  p.out_len = out_len;
  p.len_out = len_out;
  p.kept = kept_out;
  p.row_vecs = head_dim * es / 16;
  p.err = err_flag;
  cache_evict_kernel<<<dim3((unsigned)num_kv_heads, (unsigned)batch), kEvictThreads, 0,
                       static_cast<cudaStream_t>(stream)>>>(p);
  return launch_status();
}
