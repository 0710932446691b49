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
#include "prefix_flash.cuh"

namespace cg = cooperative_groups;

namespace kani {
namespace {

using prefix::ex2;
using prefix::merge_weight;
using prefix::Params;

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr float kMaxSlack = 8.f;             // the running maximum may lag by this many powers of 2
constexpr int64_t kSharedBytes = 128 << 20;  // prefix bytes (K and V), times the streams, from which it is read once
constexpr int64_t kLogitSmem = 32 * 1024;    // logits kept in shared memory up to this many bytes

struct DecodeParams : Params {
  float* logits;     // workspace [B, Hq, cache_len] when they do not fit in shared memory
  int logit_rows;    // else rows per CTA
  int by_length;     // blocks take the streams in the order of their lengths
  int step;          // launched as a programmatic dependent of the launch that writes q and the newest rows
  int parts;         // the prefix's partials (0: this kernel reads the prefix rows itself)
  const float* acc;  // [parts][B, Hq][D]
  const float* ml;   // [parts][B, Hq][2]
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

// After the last row the rings are idle: each warp's holds its own partial first, and
// in rank 0's the partials of the cluster's CTAs r = warp and r = warp + 4 behind it.
template <int D>
constexpr int kPartBytes = (8 * (D + 2) * 4 + 127) / 128 * 128;
constexpr int kMaxParts = 16;  // of the prefix; 8 heads' factors of all partials fit the first slot
template <int D>
constexpr int kFirstSlot = kPartBytes<D> > 8 * (kMaxParts + 8) * 4 ? kPartBytes<D> : 8 * (kMaxParts + 8) * 4;

template <typename T, int D, int KEYS, int STAGES>
__global__ void __launch_bounds__(kThreads) prefix_decode_kernel(const __grid_constant__ DecodeParams p) {
  constexpr int ROW = D * 2;             // bytes
  constexpr int CH = ROW / 16;           // 16-byte pieces per row
  constexpr int TILE = KEYS * ROW;       // one stage's K (or V) rows
  constexpr int PART = D + 2;            // floats of a head's partial: m, l, weighted V
  extern __shared__ __align__(128) unsigned char smem[];
  cg::cluster_group cluster = cg::this_cluster();
  const int ncl = (int)gridDim.x, rank = (int)blockIdx.x;
  const int h = blockIdx.y, G = p.group;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int b = blockIdx.z;
  if (p.by_length) {
    // blocks start in the order of z: the longest stream first, so that the last ones
    // to start are short (64 streams of 120..1500 rows: 24.9 us against 30.8)
    int* len = reinterpret_cast<int*>(smem);
    __shared__ int s_b;
    const int n = p.batch <= tid ? -1 : (int)min(max(p.kv_len[tid], (int64_t)0), p.cache_len);
    len[tid] = n;
    __syncthreads();
    int before = 0;
#pragma unroll 4
    for (int j = 0; j < p.batch; j += 4) {
      const int4 o = *reinterpret_cast<const int4*>(len + j);
      before += (o.x > n || (o.x == n && j < tid)) + (o.y > n || (o.y == n && j + 1 < tid)) +
                (o.z > n || (o.z == n && j + 2 < tid)) + (o.w > n || (o.w == n && j + 3 < tid));
    }
    if (n >= 0 && before == b) s_b = tid;
    __syncthreads();
    b = s_b;
  }
  const int g = lane >> 2, t4 = lane & 3;  // this lane's head (row) and pair of columns in a product
  constexpr int WRING = STAGES * 2 * TILE;  // bytes of a warp's ring
  static_assert(kFirstSlot<D> + 2 * kPartBytes<D> <= WRING, "the partials fit the rings");
  auto gathered = [&](int r, int hd) {  // CTA r's partial of a head (rank 0's memory)
    return reinterpret_cast<float*>(smem + (r & 3) * WRING + kFirstSlot<D> + (r >> 2) * kPartBytes<D>) + hd * PART;
  };
  float* stat = reinterpret_cast<float*>(smem + kRingBytes<D, KEYS, STAGES>);  // [G][2]: m, 1 / l
  float* s_logits = stat + 2 * G;                                              // [G][logit_rows]

  const bool tell = rank == 0 && h == 0 && tid == 0;
  const int plen = p.parts        ? 0
                   : p.prefix_len ? prefix::checked_len(*p.prefix_len, p.prefix_rows, p.err, tell && b == 0)
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

  const uint32_t ring = smem32(smem) + (uint32_t)warp * WRING;
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
  auto first_steps = [&] {
#pragma unroll
    for (int it = 0; it < STAGES - 1; ++it) {
      if (it < nit) issue(it);
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
  };
  // As a step's dependent launch (p.step), the first rows stream in while the launch
  // before still runs, but in the warp where they hold the stream's newest row, the one
  // which that launch may be writing.
  const bool newest = no > 0 && o0 + no == own && w0 + wn == n;
  const bool early = p.step && !(newest && nit < STAGES);
  if (early) first_steps();
  if (p.step) griddep_wait();  // q and the newest row
  if (!early) first_steps();

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
  float* mine = reinterpret_cast<float*>(smem + (size_t)warp * WRING);
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
  for (int t = tid; t < G * D; t += kThreads) {
    const int hd = t / D, d = t % D;
    const float* w = reinterpret_cast<const float*>(smem) + hd * PART;
    constexpr int WS = WRING / 4;
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
    float* o = gathered(rank, hd);
    if (ncl > 1) o = cluster.map_shared_rank(o, 0);
    o[2 + d] = as;
    if (d == 0) {
      o[0] = mx;
      o[1] = ls;
    }
  }
  if (ncl > 1) cluster.sync(); else __syncthreads();
  // The rows above streamed in while the prefix launch ran; its partials (and the
  // memory written below) only now.  Every block waits, so this launch ends after it.
  griddep_wait();
  if (rank == 0) {
    // factor of every partial (the prefix's, then the cluster's), and 1 / sum
    const int64_t row = (int64_t)b * p.hq + h * G, nrows = (int64_t)p.batch * p.hq;
    const int np_ = p.parts, all = np_ + ncl;
    float* fac = reinterpret_cast<float*>(smem);  // [G][all], in the first slot
    for (int hd = warp; hd < G; hd += kWarps) {
      float mx = -INFINITY, ls = 0.f;
      auto ml = [&](int i) {
        return i < np_ ? *reinterpret_cast<const float2*>(p.ml + (i * nrows + row + hd) * 2)
                       : *reinterpret_cast<const float2*>(gathered(i - np_, hd));
      };
      for (int i = lane; i < all; i += 32) mx = fmaxf(mx, ml(i).x);
      for (int x = 16; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
      for (int i = lane; i < all; i += 32) {
        const float2 v = ml(i);
        const float f = merge_weight(v.x, mx);
        fac[hd * all + i] = f;
        ls += v.y * f;
      }
      for (int x = 16; x > 0; x >>= 1) ls += __shfl_xor_sync(0xffffffffu, ls, x);
      const float inv = ls == 0.f ? 0.f : 1.f / ls;
      __syncwarp();
      for (int i = lane; i < all; i += 32) fac[hd * all + i] *= inv;
      if (p.scores != nullptr && lane < ncl) {
        float* st = ncl > 1 ? cluster.map_shared_rank(stat, lane) : stat;
        st[2 * hd] = mx == -INFINITY ? 0.f : mx;
        st[2 * hd + 1] = inv;
      }
    }
    __syncthreads();
    for (int t = tid; t < G * D; t += kThreads) {
      const int hd = t / D, d = t % D;
      float as = 0.f;
      const float* pa = p.acc + (row + hd) * D + d;
#pragma unroll 8
      for (int i = 0; i < np_; ++i) as = fmaf(pa[i * nrows * D], fac[hd * all + i], as);
#pragma unroll
      for (int r = 0; r < 8; ++r)
        if (r < ncl) as = fmaf(gathered(r, hd)[2 + d], fac[hd * all + np_ + r], as);
      static_cast<T*>(p.out)[b * p.ob + (int64_t)(h * G + hd) * p.oh + d] = Elem<T>::from_f(as);
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
                      4 * (2 * p.group + (size_t)p.group * p.logit_rows);
  static std::atomic<uint64_t> granted{0};
  if (const int e = prefix::grant_smem(kern, kRingBytes<D, KEYS, STAGES> + 4 * 2 * 8 + kLogitSmem, granted)) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ncl, (unsigned)p.hk, (unsigned)p.batch);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ncl;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.parts || p.step ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
  note_launch();
  return e == cudaSuccess ? KANI_OK : (int)e;
}

struct DecodePlan {
  int ncl;         // CTAs per (stream, KV head)
  int logit_rows;  // rows of logits that a CTA keeps in shared memory; 0: in the workspace
  int parts;       // partial results of the prefix per query; 0: no launch for it
  prefix::FlashSplit split;
  int64_t logits, acc, ml;  // bytes of the workspace's sections
};

DecodePlan plan_decode(int64_t batch, int hq, int hk, int d, int64_t cache_len, int64_t prefix_rows, bool scores) {
  DecodePlan p = {};
  // as many CTAs as still fit the GPU at two per SM
  p.ncl = 8;
  while (p.ncl > 1 && batch * hk * p.ncl > 2 * sm_count()) p.ncl >>= 1;
  const int64_t rows = (cache_len + p.ncl - 1) / p.ncl;
  if (scores && rows * (hq / hk) * 4 <= kLogitSmem) p.logit_rows = (int)rows;
  if (scores && !p.logit_rows) p.logits = batch * hq * cache_len * 4;
  // The prefix in a launch of its own, for all streams, costs 3-6 us; read by every
  // stream's blocks it costs L2 bandwidth in the streams' number.  Measured (8 KV heads
  // of 64, up to 500 own rows; own launch / read by each, us):
  //    32 MiB in all: 16 streams x 1024 rows 11.7 / 10.4, 64 x 256 18.0 / 15.2
  //    64 MiB: 16 x 2048 12.5 / 14.6, 32 x 1024 12.3 / 16.2, 64 x 512 18.5 / 19.7
  //    96 MiB: 32 x 1536 12.9 / 20.6, 64 x 768 19.2 / 24.2, 128 x 384 27.7 / 29.9
  //   128 MiB: 16 x 4096 16.2 / 23.4, 64 x 1024 19.4 / 28.9, 128 x 512 28.9 / 33.4
  // The own launch rounds the prefix's weights to the storage type, these blocks keep
  // them in two halves (result off by 2.1e-3 of its norm against 1.7e-3 in bf16): up to
  // 128 MiB the closer result is kept, at 1.1 to 1.6 times the time from 64 MiB on.
  if (prefix_rows > 0 && batch * prefix_rows * hk * d * 4 >= kSharedBytes) {
    p.split = prefix::flash_split(1, batch, hq, hk, prefix_rows, kMaxParts);
    p.parts = p.split.parts;
    p.acc = (int64_t)p.parts * batch * hq * d * 4;
    p.ml = (int64_t)p.parts * batch * hq * 2 * 4;
  }
  return p;
}

}  // namespace
}  // namespace kani

extern "C" int64_t kani_prefix_decode_workspace(int64_t batch, int32_t num_q_heads, int32_t num_kv_heads,
                                                int32_t head_dim, int64_t cache_len, int64_t prefix_rows,
                                                int32_t with_scores) {
  if (batch <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 || cache_len < 0 || prefix_rows < 0 ||
      num_q_heads % num_kv_heads != 0 || num_q_heads / num_kv_heads > 8)
    return 0;
  const kani::DecodePlan p =
      kani::plan_decode(batch, num_q_heads, num_kv_heads, head_dim, cache_len, prefix_rows, with_scores && cache_len > 0);
  return p.logits + p.acc + p.ml;
}

namespace {
int prefix_decode_impl(
    int32_t dtype, int64_t batch, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, const void* q,
    int64_t q_batch_stride, int64_t q_head_stride, const void* k_cache, const void* v_cache,
    int64_t cache_batch_stride, int64_t cache_head_stride, int64_t cache_slot_stride, int64_t cache_len,
    const int64_t* kv_len, const void* prefix_k, const void* prefix_v, int64_t prefix_head_stride,
    int64_t prefix_row_stride, int64_t prefix_rows, const int64_t* prefix_len, float scale, float* scores,
    int64_t scores_batch_stride, int64_t scores_head_stride, void* out, int64_t out_batch_stride,
    int64_t out_head_stride, void* workspace, int64_t workspace_bytes, int32_t* err_flag, void* stream,
    bool step) {
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
  const DecodePlan plan =
      plan_decode(batch, num_q_heads, num_kv_heads, head_dim, cache_len, prefix_rows, p.scores != nullptr);
  const int64_t need = plan.logits + plan.acc + plan.ml;
  if (workspace_bytes < need || (need > 0 && (!workspace || !aligned16(workspace)))) return KANI_ERR_INVALID_ARG;
  char* ws = static_cast<char*>(workspace);
  float* acc = reinterpret_cast<float*>(ws);
  float* ml = reinterpret_cast<float*>(ws + plan.acc);
  p.acc = acc;
  p.ml = ml;
  p.parts = plan.parts;
  // behind the prefix launch, which itself waits for the launch before, nothing is pending
  p.step = step && !plan.parts;
  // Finding a block's place costs it up to 0.4 us: worth it while the blocks make few
  // waves (64 streams x 8 heads), not for more (128 x 8, 20 rows each: 24.1 us without
  // it, 26.8 with).
  p.by_length = batch > 1 && batch <= kThreads && batch * num_kv_heads * plan.ncl <= 4 * sm_count();
  p.logit_rows = plan.logit_rows;
  p.logits = plan.logits ? reinterpret_cast<float*>(ws + plan.acc + plan.ml) : nullptr;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (plan.parts) {  // the prefix for all streams at once: the streams are the tokens of one sequence
    prefix::Params f = p;
    f.qt = p.qb;
    f.qb = 0;
    const int rc = prefix::launch_flash(f, dtype, head_dim, 1, (int)batch, false, plan.split, ml, acc, step, s);
    if (rc != KANI_OK) return rc;
  }
  auto go = [&]<typename T>() {
    // Rings of 64 KB, three blocks per SM; of 48 KB where those make two waves of the blocks
    // and four per SM make one (64 streams of 880 rows: 30.3 us with 64 KB, 23.8 with 48;
    // behind a prefix launch, which takes the shared memory of one, 25.7 and 28.6).
    const int64_t blocks = batch * num_kv_heads * plan.ncl;
    const bool small = !plan.parts && blocks > 3 * sm_count() && blocks <= 4 * sm_count();
    if (head_dim == 64)
      return small ? launch_decode<T, 64, 16, 3>(p, plan.ncl, s) : launch_decode<T, 64, 32, 2>(p, plan.ncl, s);
    return launch_decode<T, 128, 16, 2>(p, plan.ncl, s);
  };
  return dtype == KANI_DTYPE_BF16 ? go.template operator()<__nv_bfloat16>() : go.template operator()<__half>();
}
}  // namespace

extern "C" int kani_prefix_decode_attention(
    int32_t dtype, int64_t batch, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, const void* q,
    int64_t q_batch_stride, int64_t q_head_stride, const void* k_cache, const void* v_cache,
    int64_t cache_batch_stride, int64_t cache_head_stride, int64_t cache_slot_stride, int64_t cache_len,
    const int64_t* kv_len, const void* prefix_k, const void* prefix_v, int64_t prefix_head_stride,
    int64_t prefix_row_stride, int64_t prefix_rows, const int64_t* prefix_len, float scale, float* scores,
    int64_t scores_batch_stride, int64_t scores_head_stride, void* out, int64_t out_batch_stride,
    int64_t out_head_stride, void* workspace, int64_t workspace_bytes, int32_t* err_flag, void* stream) {
  return prefix_decode_impl(dtype, batch, num_q_heads, num_kv_heads, head_dim, q, q_batch_stride, q_head_stride, k_cache, v_cache,
                            cache_batch_stride, cache_head_stride, cache_slot_stride, cache_len, kv_len, prefix_k,
                            prefix_v, prefix_head_stride, prefix_row_stride, prefix_rows, prefix_len, scale, scores,
                            scores_batch_stride, scores_head_stride, out, out_batch_stride, out_head_stride, workspace,
                            workspace_bytes, err_flag, stream, false);
}

extern "C" int kani_prefix_decode_attention_step(
    int32_t dtype, int64_t batch, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, const void* q,
    int64_t q_batch_stride, int64_t q_head_stride, const void* k_cache, const void* v_cache,
    int64_t cache_batch_stride, int64_t cache_head_stride, int64_t cache_slot_stride, int64_t cache_len,
    const int64_t* kv_len, const void* prefix_k, const void* prefix_v, int64_t prefix_head_stride,
    int64_t prefix_row_stride, int64_t prefix_rows, const int64_t* prefix_len, float scale, float* scores,
    int64_t scores_batch_stride, int64_t scores_head_stride, void* out, int64_t out_batch_stride,
    int64_t out_head_stride, void* workspace, int64_t workspace_bytes, int32_t* err_flag, void* stream) {
  return prefix_decode_impl(dtype, batch, num_q_heads, num_kv_heads, head_dim, q, q_batch_stride, q_head_stride, k_cache, v_cache,
                            cache_batch_stride, cache_head_stride, cache_slot_stride, cache_len, kv_len, prefix_k,
                            prefix_v, prefix_head_stride, prefix_row_stride, prefix_rows, prefix_len, scale, scores,
                            scores_batch_stride, scores_head_stride, out, out_batch_stride, out_head_stride, workspace,
                            workspace_bytes, err_flag, stream, true);
}
