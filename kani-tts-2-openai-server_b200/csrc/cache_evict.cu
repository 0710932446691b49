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
// Moving the kept rows bounds it.  A cluster of 1, 2, 4 or 8 CTAs works on one
// (b, h): every CTA finds the kept rows for itself and moves its share of the columns
// of the rows [K | V], so in-place moves of different CTAs never meet.
// (Out of place, further clusters may share the rows of long caches.)
//   * Selection: the scores' bits in an order where unsigned comparison is theirs; the
//     most-th largest by radix selection over digits of 11, 11 and 10 bits, with a
//     histogram in shared memory; ties beyond it go by slot.  Counts are integers, so
//     the order of the atomics does not matter.
//   * Compaction: kept slots of a chunk by ballots and a scan over the warps, as a
//     list in shared memory; then 16-byte pieces of the listed rows, four in flight
//     per thread.  In place, kept row i comes from a slot >= i: each step's pieces are
//     all read before any is written, and no later step reads a row that was written.
//   * Scores stay in registers between the passes where the cache is one chunk; CTA 0
//     writes the moved ones once every CTA of the cluster has read the chunk.
#include <cooperative_groups.h>

#include "common.cuh"

namespace cg = cooperative_groups;

namespace kani {
namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kBins = 2048, kDigits = kBins / kThreads;
constexpr int kInFlight = 4;  // 16-byte pieces per thread and step

struct EvictParams {
  const char* k;
  const char* v;
  int64_t cb, ch, cs;  // byte strides of the caches [B, Hk, S, D]
  int64_t cache_len;
  const float* scores;
  int64_t sb, sh;
  const int64_t* kv_len;
  int64_t budget, recent, protect;
  char* k_out;
  char* v_out;
  int64_t cbo, cho, cso;
  float* scores_out;
  int64_t sbo, sho;
  int64_t out_len;
  int64_t* len_out;
  int32_t* kept;  // [B, Hk, budget] or NULL
  int row_vecs;   // 16-byte pieces per row of K or V
  int in_place;
  int32_t* err;
};

// a score's bits in an order where unsigned comparison is the score's; NaN lowest
__device__ __forceinline__ uint32_t score_key(uint32_t u) {
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0u;
  if (u == 0x80000000u) u = 0u;  // -0 is 0
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// exclusive sum over the block's warps of one number per warp (given in all its
// lanes), and the total; `red` holds kWarps ints
__device__ __forceinline__ int warps_before(int x, int* red, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  __syncthreads();  // the last use of red is over
  if (lane == 0) red[warp] = x;
  __syncthreads();
  int v = lane < kWarps ? red[lane] : 0, sum = v;
#pragma unroll
  for (int o = 1; o < kWarps; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += y;
  }
  total = __shfl_sync(0xffffffffu, sum, kWarps - 1);
  return __shfl_sync(0xffffffffu, sum - v, warp);
}

template <int ITEMS>
__global__ void __launch_bounds__(kThreads, 2) cache_evict_kernel(const EvictParams p) {
  constexpr int CHUNK = kThreads * ITEMS;  // slots per chunk; warp w has ITEMS * 32 of them in a row
  extern __shared__ int s_list[];               // kept slots of the chunk
  __shared__ int hist[kBins];
  __shared__ int red[kWarps];
  __shared__ int s_digit, s_need;
  cg::cluster_group cluster = cg::this_cluster();
  const int ncl = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  // out of place, several clusters may share the kept rows of one (b, h); the first does the rest
  const int parts = (int)gridDim.x / ncl, part = (int)blockIdx.x / ncl;
  const bool lead = rank == 0 && part == 0;
  const int h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int64_t len = p.kv_len[b];
  if ((len < 0 || len > p.cache_len) && lead && h == 0 && tid == 0 && p.err) atomicOr(p.err, KANI_FLAG_SLOT_OOB);
  const int n = (int)(len < 0 ? 0 : (len > p.cache_len ? p.cache_len : len));
  const bool cut = n > p.budget;
  const int keep = cut ? (int)p.budget : n;
  // rows [lo, hi) compete for `most` places; the others stay
  const int lo = cut ? (int)p.protect : n, hi = cut ? n - (int)p.recent : n;
  const int most = cut ? (int)(p.budget - p.protect - p.recent) : 0;
  const float* sc = p.scores + b * p.sb + h * p.sh;
  const int chunks = (n + CHUNK - 1) / CHUNK;

  uint32_t raw[ITEMS];
  auto slot = [&](int c, int i) { return c * CHUNK + warp * (ITEMS * 32) + i * 32 + lane; };
  auto load = [&](int c) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) raw[i] = slot(c, i) < n ? __float_as_uint(sc[slot(c, i)]) : 0u;
  };
  if (chunks > 0) load(0);

  // ---- the lowest kept score of the competing rows, and how many rows tie for it
  uint32_t thr = 0xffffffffu;
  int ties = 0;
  if (most > 0) {
    int need = most;
    uint32_t prefix = 0;
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
      for (int i = tid; i < kBins; i += kThreads) hist[i] = 0;
      __syncthreads();
#pragma unroll 1
      for (int c = 0; c < chunks; ++c) {
        if (chunks > 1) load(c);
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
          const int j = slot(c, i);
          const uint32_t key = score_key(raw[i]);
          const bool in = j >= lo && j < hi && (pass == 0 || (key >> (shift + bits)) == prefix);
          if (in) atomicAdd(&hist[(key >> shift) & ((1u << bits) - 1u)], 1);
        }
      }
      __syncthreads();
      // digits from the highest down: thread t has kDigits of them
      const int top = kBins - 1 - kDigits * tid;
      int mine[kDigits], sum = 0;
#pragma unroll
      for (int i = 0; i < kDigits; ++i) sum += mine[i] = hist[top - i];
      int before = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += y;
      }
      int total;
      const int wsum = __shfl_sync(0xffffffffu, before, 31);
      before += warps_before(wsum, red, total) - sum;
      if (before < need && need <= before + sum) {
#pragma unroll
        for (int i = 0; i < kDigits; ++i) {
          if (need > before && need <= before + mine[i]) {
            s_digit = top - i;
            s_need = need - before;
          }
          before += mine[i];
        }
      }
      __syncthreads();
      prefix = (prefix << bits) | (uint32_t)s_digit;
      need = s_need;
    }
    thr = prefix;
    ties = need;
  }

  // ---- the kept slots in order, chunk by chunk, and their rows
  const int w0 = rank * 2 * p.row_vecs / ncl, wn = (rank + 1) * 2 * p.row_vecs / ncl - w0;  // pieces of [K | V]
  const int shift = (wn & (wn - 1)) == 0 ? __ffs(wn) - 1 : -1;
  const char* kin = p.k + b * p.cb + h * p.ch;
  const char* vin = p.v + b * p.cb + h * p.ch;
  char* kout = p.k_out + b * p.cbo + h * p.cho;
  char* vout = p.v_out + b * p.cbo + h * p.cho;
  float* so = p.scores_out + b * p.sbo + h * p.sho;
  int32_t* kept = p.kept ? p.kept + ((int64_t)b * gridDim.y + h) * p.budget : nullptr;
  int dst0 = 0, tie0 = 0;
#pragma unroll 1
  for (int c = 0; c < chunks; ++c) {
    if (chunks > 1) load(c);
    if (p.in_place && ncl > 1) cluster.sync();  // the chunk's scores are in every CTA's registers
    int sure = 0, tied = 0;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int j = slot(c, i);
      const uint32_t key = score_key(raw[i]);
      const bool mid = j >= lo && j < hi;
      sure += __popc(__ballot_sync(0xffffffffu, j < n && (!mid || key > thr)));
      tied += __popc(__ballot_sync(0xffffffffu, mid && key == thr));
    }
    int all_tied, total;
    int tie = tie0 + warps_before(tied, red, all_tied);  // tied rows before this warp's
    const int stay = sure + min(max(ties - tie, 0), tied);
    int at = warps_before(stay, red, total);  // kept rows of the chunk before this warp's
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int j = slot(c, i);
      const uint32_t key = score_key(raw[i]);
      const bool mid = j >= lo && j < hi, tied_row = mid && key == thr;
      const unsigned below = (1u << lane) - 1u, tm = __ballot_sync(0xffffffffu, tied_row);
      const bool stays = j < n && (!mid || key > thr || (tied_row && tie + __popc(tm & below) < ties));
      const unsigned sm = __ballot_sync(0xffffffffu, stays);
      if (stays) {
        const int r = at + __popc(sm & below);
        s_list[r] = j;
        if (lead) {
          so[dst0 + r] = __uint_as_float(raw[i]);
          if (kept) kept[dst0 + r] = j;
        }
      }
      tie += __popc(tm);
      at += __popc(sm);
    }
    __syncthreads();  // the list is complete

    // pieces: index = row * wn + piece
    const int64_t first = (int64_t)total * part / parts * wn, pieces = (int64_t)total * (part + 1) / parts * wn;
    auto where = [&](int64_t i, int& r, int& w) {
      if (shift >= 0) {
        r = (int)(i >> shift);
        w = w0 + (int)(i & (wn - 1));
      } else {
        r = (int)(i / wn);
        w = w0 + (int)(i % wn);
      }
    };
    for (int64_t i0 = first; i0 < pieces; i0 += kThreads * kInFlight) {
      uint4 x[kInFlight];
      char* to[kInFlight];
#pragma unroll
      for (int u = 0; u < kInFlight; ++u) {
        const int64_t i = i0 + u * kThreads + tid;
        to[u] = nullptr;
        if (i < pieces) {
          int r, w;
          where(i, r, w);
          const int src = s_list[r], dst = dst0 + r;
          if (!p.in_place || src != dst) {
            const bool val = w >= p.row_vecs;
            const int64_t off = (int64_t)(val ? w - p.row_vecs : w) * 16;
            x[u] = ld16_stream((val ? vin : kin) + src * p.cs + off);
            to[u] = (val ? vout : kout) + dst * p.cso + off;
          }
        }
      }
      if (p.in_place) __syncthreads();  // every piece of this step is in registers
#pragma unroll
      for (int u = 0; u < kInFlight; ++u)
        if (to[u] != nullptr) st16(to[u], x[u]);
    }
    dst0 += total;
    tie0 += all_tied;
    if (c + 1 < chunks) __syncthreads();  // the list may be overwritten
  }
  if (p.in_place && ncl > 1 && chunks == 0) cluster.sync();
  if (lead) {
    for (int64_t j = keep + tid; j < p.out_len; j += kThreads) so[j] = 0.f;
    if (kept)
      for (int64_t j = keep + tid; j < p.budget; j += kThreads) kept[j] = -1;
    if (h == 0 && tid == 0) p.len_out[b] = keep;
  }
}

template <int ITEMS>
int launch_evict(const EvictParams& p, int ncl, int parts, int hk, int batch, cudaStream_t s) {
  auto kern = cache_evict_kernel<ITEMS>;
  const size_t smem = (size_t)kThreads * ITEMS * sizeof(int);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(ncl * parts), (unsigned)hk, (unsigned)batch);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ncl;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
  note_launch();
  return e == cudaSuccess ? KANI_OK : (int)e;
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
  if (head_dim == 0 || !kv_len || !len_out || kv_len == len_out ||
      (cache_len > 0 && (!k_cache || !v_cache || !scores || k_cache == v_cache)) ||
      (out_len > 0 && (!k_out || !v_out || !scores_out || k_out == v_out)))
    return KANI_ERR_INVALID_ARG;
  // in place is all of k, v and scores in place
  const bool in_place = cache_len > 0 && k_out == k_cache;
  if (cache_len > 0 && ((v_out == v_cache) != in_place || (scores_out == scores) != in_place))
    return KANI_ERR_INVALID_ARG;
  if (in_place && (out_batch_stride != cache_batch_stride || out_head_stride != cache_head_stride ||
                   out_slot_stride != cache_slot_stride || out_len != cache_len ||
                   scores_out_batch_stride != scores_batch_stride || scores_out_head_stride != scores_head_stride))
    return KANI_ERR_INVALID_ARG;
  // the strides of dimensions of one element are never followed
  if (batch == 1) cache_batch_stride = out_batch_stride = 0;
  if (num_kv_heads == 1) cache_head_stride = out_head_stride = 0;
  if (cache_len <= 1) cache_slot_stride = 0;
  if (out_len <= 1) out_slot_stride = 0;
  for (int64_t x : {cache_batch_stride, cache_head_stride, cache_slot_stride, out_batch_stride, out_head_stride,
                    out_slot_stride})
    if (x * es % 16 != 0) return KANI_ERR_UNSUPPORTED;
  if ((int64_t)head_dim * es % 16 != 0 || head_dim > 256 || batch > 65535 || num_kv_heads > 65535 ||
      cache_len > (1 << 30) || out_len > (1 << 30) || !aligned16(k_cache) || !aligned16(v_cache) ||
      !aligned16(k_out) || !aligned16(v_out))
    return KANI_ERR_UNSUPPORTED;
  EvictParams p = {};
  p.k = static_cast<const char*>(k_cache);
  p.v = static_cast<const char*>(v_cache);
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
  p.k_out = static_cast<char*>(k_out);
  p.v_out = static_cast<char*>(v_out);
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
  p.in_place = in_place;
  // enough CTAs for two per SM, each with 32 bytes or more of a row
  int ncl = 1;
  while (ncl < 8 && batch * num_kv_heads * ncl * 2 <= 2 * sm_count() && ncl * 2 <= p.row_vecs) ncl *= 2;
  // in place a cluster's columns are all the split there is; elsewhere more clusters may
  // share the rows, each after a selection of its own, while 128 KB are left to each CTA
  // (8 x 2 caches, 4 MB kept of each: 72.2 us alone, 62.4 with two; one stream's 8 x 128 KB:
  // 7.2 us alone, 9.8 with four)
  int parts = 1;
  if (!in_place && ncl == 8)
    while (parts < 4 && batch * num_kv_heads * ncl * parts * 2 <= 2 * sm_count() &&
           budget * p.row_vecs * 32 / (ncl * parts * 2) >= 128 << 10)
      parts *= 2;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // Few slots per thread where the cache is short; chunks of 8192 where it is long.  (Blocks
  // of 1024 threads, one chunk for 16384 slots, leave room for 15 clusters of 8 on the GPU:
  // 8 x 2 caches of up to 16384 rows 75.2 us, with 512 threads 72.3; 64 x 8 caches of up to
  // 2048 rows 59.7 us with 512 threads, 60.8 with 256, 69.0 with 1024.)
  if (cache_len <= 2048) return launch_evict<4>(p, ncl, parts, num_kv_heads, (int)batch, s);
  return launch_evict<16>(p, ncl, parts, num_kv_heads, (int)batch, s);
}
