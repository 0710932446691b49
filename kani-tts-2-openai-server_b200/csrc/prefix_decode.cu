// GQA decode attention of a batch of streams that share a long prefix (sm_100a).
//
// Every stream b has its own static cache (rows [0, kv_len[b])) and all of them
// read the same prefix rows [0, prefix_len) first.  With query head hq and KV
// head h = hq / G,
//     out[b, hq] = sum_j w_j v_j,  w_j = e^(scale q . k_j) / sum_i e^(scale q . k_i),
// j over the prefix rows, then the own rows; zeros where there is no row.  Optionally
// scores[b, h, j] += sum over the group of w_j, for the own rows.
//
// Memory bounds it: each own row is read once, for the G query heads together.
// One cluster of 1, 2, 4 or 8 CTAs per (b, h), the rows split evenly over its
// CTAs and their 4 warps.  A warp keeps its own ring of STAGES x KEYS rows,
// filled by 16-byte asynchronous copies (any row stride; rows past the end are
// filled with zeros, so what lies there is never read) and meets no block barrier
// until its rows are done.  Both products run on mma.m16n8k16 with fp32 sums, the
// query heads as its 16 rows: S = Q K^T has the G <= 8 heads in rows 0..7; for
// O = P V the weights are split in two, hi = round(p) in rows 0..7 and
// lo = round(p - hi) in rows 8..15 of the same instruction, so weights keep 16
// (bf16) or more bits at no cost.  K and V rows lie in shared memory with their
// 16-byte pieces XOR-ed by the row, which serves ldmatrix without bank conflicts.
// The running maximum moves only when some logit passes it by 2^8 (the weights
// stay below 2^8, far from overflow), so rescaling is rare.
//
// Partials (maximum, sum, weighted V) are merged over the CTA's warps in shared
// memory and over the cluster in rank 0's, in a fixed order.  For the scores each
// CTA keeps its rows' logits (shared memory, or the workspace for long caches) and
// adds e^(s - m) / l once rank 0 has handed out the cluster's m and l.
#include <cooperative_groups.h>

#include <algorithm>

#include "prefix_attn.cuh"

namespace cg = cooperative_groups;

namespace kani {
namespace {

using prefix::ex2;
using prefix::merge_weight;
using prefix::Params;

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr float kMaxSlack = 8.f;             // the running maximum may lag by this many powers of 2
constexpr int64_t kLogitSmem = 32 * 1024;    // logits kept in shared memory up to this many bytes

struct DecodeParams : Params {
  float* logits;      // workspace [B, Hq, cache_len] when they do not fit in shared memory
  int logit_rows;     // else rows per CTA
};

__device__ __forceinline__ uint32_t smem32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}

template <bool TRANS>
__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  if constexpr (TRANS)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

template <typename T>
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  if constexpr (std::is_same_v<T, __nv_bfloat16>)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, "
        "%2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, "
        "%2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// (a, b) rounded to T as one register, and what the rounding left of them
template <typename T>
__device__ __forceinline__ void split_pair(float a, float b, uint32_t& hi, uint32_t& lo) {
  const T ha = Elem<T>::from_f(a), hb = Elem<T>::from_f(b);
  const T la = Elem<T>::from_f(a - Elem<T>::to_f(ha)), lb = Elem<T>::from_f(b - Elem<T>::to_f(hb));
  uint16_t u[4];
  memcpy(&u[0], &ha, 2);
  memcpy(&u[1], &hb, 2);
  memcpy(&u[2], &la, 2);
  memcpy(&u[3], &lb, 2);
  hi = u[0] | ((uint32_t)u[1] << 16);
  lo = u[2] | ((uint32_t)u[3] << 16);
}

template <int D, int KEYS, int STAGES>
constexpr size_t kRingBytes = (size_t)kWarps * STAGES * 2 * KEYS * D * 2;

template <typename T, int D, int KEYS, int STAGES>
__global__ void __launch_bounds__(kThreads) prefix_decode_kernel(const __grid_constant__ DecodeParams p) {
  constexpr int ROW = D * 2;             // bytes
  constexpr int CH = ROW / 16;           // 16-byte pieces per row
  constexpr int TILE = KEYS * ROW;       // one stage's K (or V) rows
  constexpr int PART = D + 2;            // floats of a head's partial: m, l, weighted V
  extern __shared__ __align__(128) unsigned char smem[];
  cg::cluster_group cluster = cg::this_cluster();
  const int ncl = (int)gridDim.x, rank = (int)blockIdx.x;
  const int h = blockIdx.y, b = blockIdx.z, G = p.group;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t4 = lane & 3;  // this lane's head (row) and pair of columns in a product
  float* gathered = reinterpret_cast<float*>(smem + kRingBytes<D, KEYS, STAGES>);  // [ncl][G][PART], rank 0's is used
  float* stat = gathered + ncl * G * PART;                                           // [G][2]: m, 1 / l
  float* s_logits = stat + 2 * G;                                                    // [G][logit_rows]

  const bool tell = rank == 0 && h == 0 && tid == 0;
  const int plen = p.prefix_len ? prefix::checked_len(*p.prefix_len, p.prefix_rows, p.err, tell && b == 0)
                                : (int)p.prefix_rows;
  const int own = prefix::checked_len(p.kv_len[b], p.cache_len, p.err, tell);
  // this CTA's rows: [p0, p0 + np) of the prefix, then [o0, o0 + no) of the stream
  const int pc = (plen + ncl - 1) / ncl, oc = (own + ncl - 1) / ncl;
  const int p0 = min(rank * pc, plen), np = min(pc, plen - p0);
  const int o0 = min(rank * oc, own), no = min(oc, own - o0);
  const int n = np + no;
  // this warp's: [w0, w0 + wn) of those, a multiple of 16 for all but the last
  const int wc = ((n + kWarps - 1) / kWarps + 15) & ~15;
  const int w0 = min(warp * wc, n), wn = min(wc, n - w0);

  const char* kp = reinterpret_cast<const char*>(static_cast<const T*>(p.pk) + h * p.ph + (int64_t)p0 * p.ps);
  const char* vp = reinterpret_cast<const char*>(static_cast<const T*>(p.pv) + h * p.ph + (int64_t)p0 * p.ps);
  const char* ko = reinterpret_cast<const char*>(static_cast<const T*>(p.k) + b * p.cb + h * p.ch + (int64_t)o0 * p.cs);
  const char* vo = reinterpret_cast<const char*>(static_cast<const T*>(p.v) + b * p.cb + h * p.ch + (int64_t)o0 * p.cs);
  const int64_t pstep = p.ps * 2, ostep = p.cs * 2;

  const uint32_t ring = smem32(smem) + (uint32_t)warp * STAGES * 2 * TILE;
  const int rl = lane / CH, cl = lane % CH;
  auto issue = [&](int it) {
    const uint32_t kt = ring + (uint32_t)(it % STAGES) * 2 * TILE;
#pragma unroll
    for (int i = 0; i < KEYS * CH / 32; ++i) {
      const int r = i * (32 / CH) + rl;
      const int j = w0 + it * KEYS + r;  // row of the CTA
      const bool valid = it * KEYS + r < wn;
      const uint32_t dst = kt + (uint32_t)(r * ROW + ((cl ^ (r & 7)) << 4));
      const int64_t off = (j < np ? j * pstep : (int64_t)(j - np) * ostep) + cl * 16;
      const char* ks = j < np ? kp : ko;
      const char* vs = j < np ? vp : vo;
      copy16(dst, valid ? ks + off : static_cast<const char*>(p.q), valid);
      copy16(dst + TILE, valid ? vs + off : static_cast<const char*>(p.q), valid);
    }
  };
  const int nit = (wn + KEYS - 1) / KEYS;
#pragma unroll
  for (int it = 0; it < STAGES - 1; ++it) {
    if (it < nit) issue(it);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }

  // Q as the A operand: head g's dims 2 t4.. of each 16-wide step (rows 8..15 are zero)
  uint32_t qa[D / 16][2];
  {
    const T* q = static_cast<const T*>(p.q) + b * p.qb + (int64_t)(h * G + g) * p.qh + 2 * t4;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
      qa[s][0] = g < G ? __ldcg(reinterpret_cast<const unsigned int*>(q + s * 16)) : 0u;
      qa[s][1] = g < G ? __ldcg(reinterpret_cast<const unsigned int*>(q + s * 16 + 8)) : 0u;
    }
  }
  float acc[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
  float m = -INFINITY, l = 0.f;

  for (int it = 0; it < nit; ++it) {
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
    __syncwarp();
    if (it + STAGES - 1 < nit) issue(it + STAGES - 1);  // the stage of the step before, which every lane has left
    asm volatile("cp.async.commit_group;" ::: "memory");
    const uint32_t kt = ring + (uint32_t)(it % STAGES) * 2 * TILE, vt = kt + TILE;
#pragma unroll
    for (int kb = 0; kb < KEYS; kb += 16) {
      const int left = wn - it * KEYS - kb;  // valid rows of these 16
      if (left <= 0) break;
      float c[2][4] = {};
      {
        const int r = kb + ((lane >> 4) << 3) + (lane & 7);
#pragma unroll
        for (int s = 0; s < D / 16; ++s) {
          uint32_t f[4];
          ldmatrix4<false>(kt + (uint32_t)(r * ROW + (((2 * s + ((lane >> 3) & 1)) ^ (r & 7)) << 4)), f);
          mma<T>(c[0], qa[s][0], 0u, qa[s][1], 0u, f[0], f[1]);
          mma<T>(c[1], qa[s][0], 0u, qa[s][1], 0u, f[2], f[3]);
        }
      }
      float s[4];
      float mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[i] = (i >> 1) * 8 + 2 * t4 + (i & 1) < left ? c[i >> 1][i & 1] * p.qscale : -INFINITY;
        mx = fmaxf(mx, s[i]);
      }
      if (p.scores != nullptr && g < G) {
        const int j = w0 + it * KEYS + kb + 2 * t4 - np;  // own row of the CTA
        float* lg = p.logits ? p.logits + ((int64_t)b * p.hq + h * G + g) * p.cache_len + o0 : s_logits + g * p.logit_rows;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int jj = j + (i >> 1) * 8 + (i & 1);
          if (jj >= 0 && jj < no) lg[jj] = s[i];
        }
      }
      if (__any_sync(0xffffffffu, mx > m + kMaxSlack)) {
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float mn = fmaxf(m, mx), w = merge_weight(m, mn);
        l *= w;
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][e] *= w;
        m = mn;
      }
      const float ms = m == -INFINITY ? 0.f : m;
      float w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = ex2(s[i] - ms);
      l += (w[0] + w[1]) + (w[2] + w[3]);
      uint32_t a[4];
      split_pair<T>(w[0], w[1], a[0], a[1]);
      split_pair<T>(w[2], w[3], a[2], a[3]);
      const int r = kb + (lane & 15);
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        uint32_t f[4];
        ldmatrix4<true>(vt + (uint32_t)(r * ROW + (((2 * i + (lane >> 4)) ^ (r & 7)) << 4)), f);
        mma<T>(acc[2 * i], a[0], a[1], a[2], a[3], f[0], f[1]);
        mma<T>(acc[2 * i + 1], a[0], a[1], a[2], a[3], f[2], f[3]);
      }
    }
  }
  l += __shfl_xor_sync(0xffffffffu, l, 1);
  l += __shfl_xor_sync(0xffffffffu, l, 2);

  // this warp's partial, into its own (now idle) ring
  __syncwarp();
  float* mine = reinterpret_cast<float*>(smem + (size_t)warp * STAGES * 2 * TILE);
  if (g < G) {
    float* w = mine + g * PART;
    if (t4 == 0) {
      w[0] = m;
      w[1] = l;
    }
#pragma unroll
    for (int i = 0; i < D / 8; ++i) {
      w[2 + i * 8 + 2 * t4] = acc[i][0] + acc[i][2];
      w[3 + i * 8 + 2 * t4] = acc[i][1] + acc[i][3];
    }
  }
  __syncthreads();
  if (ncl > 1) cluster.sync();  // every CTA of the cluster runs: rank 0's memory may be written
  float* dst = ncl > 1 ? cluster.map_shared_rank(gathered, 0) : gathered;
  for (int t = tid; t < G * D; t += kThreads) {
    const int hd = t / D, d = t % D;
    const float* w = reinterpret_cast<const float*>(smem) + hd * PART;
    constexpr int WS = STAGES * 2 * TILE / 4;
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) mx = fmaxf(mx, w[i * WS]);
    float ls = 0.f, as = 0.f;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      const float f = merge_weight(w[i * WS], mx);
      ls += w[i * WS + 1] * f;
      as += w[i * WS + 2 + d] * f;
    }
    float* o = dst + (rank * G + hd) * PART;
    o[2 + d] = as;
    if (d == 0) {
      o[0] = mx;
      o[1] = ls;
    }
  }
  if (ncl > 1) cluster.sync(); else __syncthreads();
  if (rank == 0) {
    for (int t = tid; t < G * D; t += kThreads) {
      const int hd = t / D, d = t % D;
      float mx = -INFINITY;
      for (int r = 0; r < ncl; ++r) mx = fmaxf(mx, gathered[(r * G + hd) * PART]);
      float ls = 0.f, as = 0.f;
      for (int r = 0; r < ncl; ++r) {
        const float* o = gathered + (r * G + hd) * PART;
        const float f = merge_weight(o[0], mx);
        ls += o[1] * f;
        as += o[2 + d] * f;
      }
      static_cast<T*>(p.out)[b * p.ob + (int64_t)(h * G + hd) * p.oh + d] = Elem<T>::from_f(ls == 0.f ? 0.f : as / ls);
      if (d == 0 && p.scores != nullptr)
        for (int r = 0; r < ncl; ++r) {
          float* st = ncl > 1 ? cluster.map_shared_rank(stat, r) : stat;
          st[2 * hd] = mx == -INFINITY ? 0.f : mx;
          st[2 * hd + 1] = ls == 0.f ? 0.f : 1.f / ls;
        }
    }
  }
  if (p.scores == nullptr) return;
  if (ncl > 1) cluster.sync(); else __syncthreads();
  float* sc = p.scores + b * p.sb + h * p.sh + o0;
  for (int j = tid; j < no; j += kThreads) {
    float add = 0.f;
    for (int hd = 0; hd < G; ++hd) {
      const float s = p.logits ? p.logits[((int64_t)b * p.hq + h * G + hd) * p.cache_len + o0 + j]
                               : s_logits[hd * p.logit_rows + j];
      add += ex2(s - stat[2 * hd]) * stat[2 * hd + 1];
    }
    sc[j] += add;
  }
}

template <typename T, int D, int KEYS, int STAGES>
int launch_decode(DecodeParams& p, int ncl, cudaStream_t s) {
  auto kern = prefix_decode_kernel<T, D, KEYS, STAGES>;
  const size_t smem = kRingBytes<D, KEYS, STAGES> +
                      4 * ((size_t)ncl * p.group * (D + 2) + 2 * p.group + (size_t)p.group * p.logit_rows);
  const cudaError_t a = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (a != cudaSuccess) return (int)a;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ncl, (unsigned)p.hk, (unsigned)p.batch);
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

// CTAs per (stream, KV head): as many as still fit the GPU at two per SM
int cluster_size(int64_t batch, int32_t hk) {
  int ncl = 8;
  while (ncl > 1 && batch * hk * ncl > 2 * sm_count()) ncl >>= 1;
  return ncl;
}

// rows of logits that a CTA keeps in shared memory; 0: they go to the workspace
int logit_rows(int group, int64_t cache_len, int ncl) {
  const int64_t rows = (cache_len + ncl - 1) / ncl;
  return rows * group * 4 <= kLogitSmem ? (int)rows : 0;
}

}  // namespace
}  // namespace kani

extern "C" int64_t kani_prefix_decode_workspace(int64_t batch, int32_t num_q_heads, int32_t num_kv_heads,
                                                int32_t head_dim, int64_t cache_len, int64_t prefix_rows,
                                                int32_t with_scores) {
  using namespace kani;
  if (batch <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || cache_len <= 0 || !with_scores) return 0;
  if (logit_rows(num_q_heads / num_kv_heads, cache_len, cluster_size(batch, num_kv_heads)) > 0) return 0;
  return batch * num_q_heads * cache_len * 4;
}

extern "C" int kani_prefix_decode_attention(
    int32_t dtype, int64_t batch, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, const void* q,
    int64_t q_batch_stride, int64_t q_head_stride, const void* k_cache, const void* v_cache,
    int64_t cache_batch_stride, int64_t cache_head_stride, int64_t cache_slot_stride, int64_t cache_len,
    const int64_t* kv_len, const void* prefix_k, const void* prefix_v, int64_t prefix_head_stride,
    int64_t prefix_row_stride, int64_t prefix_rows, const int64_t* prefix_len, float scale, float* scores,
    int64_t scores_batch_stride, int64_t scores_head_stride, void* out, int64_t out_batch_stride,
    int64_t out_head_stride, void* workspace, int64_t workspace_bytes, int32_t* err_flag, void* stream) {
  using namespace kani;
  if (batch < 0 || num_q_heads < 0 || num_kv_heads < 0 || head_dim < 0 || cache_len < 0 || prefix_rows < 0 ||
      workspace_bytes < 0)
    return KANI_ERR_INVALID_ARG;
  if (batch == 0 || num_q_heads == 0) return KANI_OK;
  DecodeParams p = {};
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
  p.scores = cache_len > 0 ? scores : nullptr;
  p.sb = scores_batch_stride;
  p.sh = scores_head_stride;
  p.out = out;
  p.ob = out_batch_stride;
  p.oh = out_head_stride;
  p.err = err_flag;
  if (const int bad = prefix::check_params(p, dtype, batch, 1, num_q_heads, num_kv_heads, head_dim, scale)) return bad;
  const int64_t need = kani_prefix_decode_workspace(batch, num_q_heads, num_kv_heads, head_dim, cache_len, prefix_rows,
                                                    p.scores != nullptr);
  if (workspace_bytes < need || (need > 0 && (!workspace || !aligned16(workspace)))) return KANI_ERR_INVALID_ARG;
  const int ncl = cluster_size(batch, num_kv_heads);
  p.logit_rows = p.scores ? logit_rows(p.group, cache_len, ncl) : 0;
  p.logits = p.scores && !p.logit_rows ? static_cast<float*>(workspace) : nullptr;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto go = [&]<typename T>() {
    return head_dim == 64 ? launch_decode<T, 64, 32, 3>(p, ncl, s) : launch_decode<T, 128, 16, 3>(p, ncl, s);
  };
  return dtype == KANI_DTYPE_BF16 ? go.template operator()<__nv_bfloat16>() : go.template operator()<__half>();
}
