// GQA attention of many queries over a prefix shared by the batch and, causally,
// over each stream's own rows, on the tensor cores (tcgen05, sm_100a).
//
// Query i < q_len[b] of stream b is the stream's own cache row kv_len[b] - q_len[b] + i;
// it sees the prefix rows [0, prefix_len) and the own rows up to its own:
//     out[b, i, hq] = softmax_j(scale * q . k_j) v_j;   queries from q_len[b] on get zeros.
// The decode form runs the same kernel over the prefix alone, with the streams in
// the place of the tokens, so the prefix is read once for the whole batch.
//
// One CTA per 128 query rows of a KV head (row = token * G + head of the group: the
// G heads share each K and V tile), over tiles of 64 rows, two CTAs per SM:
//   * warp 4 brings Q once and K / V tiles through a ring of stages by TMA
//     (128-byte swizzle);
//   * warp 5 issues the MMAs: S = Q K^T (both operands in shared memory, S in two
//     tensor-memory buffers, so the next S is computed while this one is worked on)
//     and O += P V with P taken from tensor memory and V as it lies (rows = keys: an
//     MN-major operand);
//   * warps 0..3 hold one query row per thread: p = 2^(s c - m) and their sum in
//     fp32; P is rounded to the storage type (bf16 / fp16: half a step of it relative
//     to each weight, as the result's own rounding) and replaces S in tensor memory.
// The running maximum moves only when a tile's weights sum to more than 2^10, so most
// tiles need no search for it, and O is rescaled (read from and written back to tensor
// memory) a few times per row at most; p stays below 2^10, which both types hold.
//
// Rows that a tile holds beyond what its queries may see are masked in S, and their
// V is replaced by zeros in shared memory where nobody may see it or where it is not
// finite (0 * inf would reach every row); values that are not finite and that later
// queries of the tile do see are added to those at the end.
//
// A grid of few CTAs splits the rows over a cluster of 2, 4 or 8: every CTA leaves its
// O in its own (by then idle) operand memory, and CTA r joins rows [128 r / n, ..) of
// all of them through distributed shared memory, in the order of the splits.
#include <cooperative_groups.h>

#include <algorithm>

#include "prefix_attn.cuh"
#include "prefix_flash.cuh"
#include "tc_common.cuh"

namespace cg = cooperative_groups;

namespace kani {
namespace prefix {
namespace {

constexpr int kRows = 128;   // query rows per CTA: the MMA's M
constexpr int kKeys = 64;    // K / V rows per tile
constexpr int kSoftmaxThreads = 128;
constexpr int kFlashThreads = kSoftmaxThreads + 64;
constexpr uint32_t kTmemCols = 256;  // S: 2 x 64, O: D
constexpr uint32_t kTmemO = 128;
constexpr float kMaxSum = 1024.f;
constexpr int kMaxStages = 4;

template <int D> struct FlashShape {
  static constexpr int kStages = D == 64 ? 4 : 2;
  // One pair of weights in so many by polynomial instead of the special-function unit,
  // which takes 8 cycles for a warp's 32: with D = 64 that unit is the busiest (4 x 4096
  // tokens behind 4096 rows: none 589 us, one in 4 568, one in 6 562, one in 8 563), with
  // D = 128 the products weigh twice as much (3 x 777 tokens: none 53.8-55.8 us, one in 4
  // 54.3-54.4, between runs on one GPU and on several: no gain).
  static constexpr int kFmaOneIn = D == 64 ? 6 : 0;
  static constexpr uint32_t kQBytes = kRows * D * 2;
  static constexpr uint32_t kTileBytes = kKeys * D * 2;
  // 2 CTAs per SM by shared memory, so two blocks' 256 columns fill tensor memory
  static_assert((size_t)kRows * (D + 4) * 4 <= kQBytes + (size_t)kStages * 2 * kTileBytes, "O fits the operands' memory");
  static constexpr size_t kSmem = 1024 + kQBytes + (size_t)kStages * 2 * kTileBytes;
};

struct FlashParams {
  CUtensorMap q, pk, pv, k, v;
  const int64_t* kv_len;
  const int64_t* q_len;
  const int64_t* prefix_len;
  const void* v_raw;
  int64_t vb, vh, vs;  // strides of the own V rows (elements)
  void* out;
  int64_t ob, ot, oh;
  float* ml;   // partials [splits / cluster][rows][2]; NULL: write out
  float* acc;  // [splits / cluster][rows][D]
  int64_t rows;  // batch * tokens * hq
  int32_t* err;
  float qscale;
  int tokens, group, hq, tpt, splits, cluster, m_tiles;
  int prefix_rows, cache_len;  // cache_len 0: prefix only
  int b_step, h_step;          // 0 where the own caches' batch / head dimension is expanded
  int ph_step, qb_step;
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3,
                                            uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
      : "memory");
}

// D[tmem] (+)= A[tmem] * B[smem]
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1u : 0u)
      : "memory");
}

// MN-major 128-byte-swizzle operand: 64 elements of a key's row are contiguous,
// 8 keys make an atom of 1024 bytes (stride offset), 64-wide column blocks lie
// kKeys rows apart (leading offset)
__device__ __forceinline__ uint64_t desc_v(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3fffu) | ((uint64_t)((kKeys * 128) >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}

#define KANI_R4(v, i) "=r"(v[i]), "=r"(v[i + 1]), "=r"(v[i + 2]), "=r"(v[i + 3])
#define KANI_W4(v, i) "r"(v[i]), "r"(v[i + 1]), "r"(v[i + 2]), "r"(v[i + 3])

// 32 consecutive 32-bit columns of this warp's lanes (not waited on)
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : KANI_R4(v, 0), KANI_R4(v, 4), KANI_R4(v, 8), KANI_R4(v, 12), KANI_R4(v, 16), KANI_R4(v, 20), KANI_R4(v, 24),
        KANI_R4(v, 28)
      : "r"(addr)
      : "memory");
}

__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
      KANI_W4(v, 0), KANI_W4(v, 4), KANI_W4(v, 8), KANI_W4(v, 12), KANI_W4(v, 16), KANI_W4(v, 20), KANI_W4(v, 24),
      KANI_W4(v, 28)
      : "memory");
}
#undef KANI_R4
#undef KANI_W4

__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void mbar_init_n(uint32_t bar, uint32_t n) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(n) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  uint32_t u;
  if constexpr (std::is_same_v<T, __nv_bfloat16>) {
    const __nv_bfloat162 x = __floats2bfloat162_rn(a, b);
    memcpy(&u, &x, 4);
  } else {
    const __half2 x = __floats2half2_rn(a, b);
    memcpy(&u, &x, 4);
  }
  return u;
}

// whether a 16-bit value is infinite or NaN
template <typename T>
__device__ __forceinline__ bool not_finite16(uint32_t bits) {
  constexpr uint32_t e = std::is_same_v<T, __nv_bfloat16> ? 0x7f80u : 0x7c00u;
  return (bits & e) == e;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// 2^x on the FMA pipes: x = n + f with n the nearest integer (read off the low bits of
// x + 1.5 * 2^23), 2^f by a polynomial of degree 4 fitted to the least relative error on
// [-1/2, 1/2] (2.7e-6, under a hundredth of half a step of fp16), n added to the
// exponent.  x is held to [-126, 127]: what lies below counts as 2^-126, what lies above
// is far past kMaxSum and is done again.  A NaN stays one up to the last step, where its
// bits (0x7fffffff, as the arithmetic makes them) give the largest finite number: past
// kMaxSum too.
__device__ __forceinline__ float clamp_exponent(float x) {
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(x) : "f"(-126.f));
  asm("min.NaN.f32 %0, %0, %1;" : "+f"(x) : "f"(127.f));
  return x;
}
__device__ __forceinline__ float2 exp2_fma(float2 x) {
  x.x = clamp_exponent(x.x);
  x.y = clamp_exponent(x.y);
  const float2 magic = make_float2(12582912.f, 12582912.f);
  const float2 t = __fadd2_rn(x, magic);
  const float2 n = __fadd2_rn(t, make_float2(-12582912.f, -12582912.f));
  const float2 f = __fadd2_rn(x, make_float2(-n.x, -n.y));
  auto k = [](float v) { return make_float2(v, v); };
  float2 p = __ffma2_rn(k(0.009570102207362652f), f, k(0.05591785907745361f));
  p = __ffma2_rn(p, f, k(0.240247443318367f));
  p = __ffma2_rn(p, f, k(0.6931217908859253f));
  p = __ffma2_rn(p, f, k(0.9999992847442627f));
  return make_float2(__int_as_float(__float_as_int(p.x) + (__float_as_int(t.x) << 23)),
                     __int_as_float(__float_as_int(p.y) + (__float_as_int(t.y) << 23)));
}

// one lane of a converged warp (which the compiler knows to be one)
__device__ __forceinline__ bool elect_one() {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok));
  return ok != 0;
}

struct FlashBars {
  uint64_t q, pv;
  uint64_t kv_full[kMaxStages], kv_empty[kMaxStages];
  uint64_t s_full[2], p_full[2];
};

template <typename T, int D>
__global__ void __launch_bounds__(kFlashThreads, 2) prefix_flash_kernel(const __grid_constant__ FlashParams p) {
  using Shape = FlashShape<D>;
  constexpr int ST = Shape::kStages;
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(8) FlashBars bars;
  __shared__ uint32_t s_tmem;
  __shared__ int s_failed, s_poison;
  __shared__ float2 s_ml[kRows];  // with a cluster: this CTA's maximum and sum of each row
  constexpr int RED = D + 4;      // floats per row of O left in shared memory (16-byte steps between rows)

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int split = (int)blockIdx.x % p.splits;
  const int m_tile = p.m_tiles - 1 - (int)blockIdx.x / p.splits;  // the longest rows first
  const int h = blockIdx.y, b = blockIdx.z, G = p.group;
  const int t0 = m_tile * p.tpt;  // first token of the tile
  const uint32_t base = (tc::smem_addr(smem_raw) + 1023u) & ~1023u;
  const uint32_t q_smem = base, ring = base + Shape::kQBytes;

  if (warp == 5) tc::tmem_alloc(&s_tmem, kTmemCols);
  if (warp == 4 && lane < 5) tc::prefetch_map(lane == 0 ? &p.q : lane == 1 ? &p.pk : lane == 2 ? &p.pv : lane == 3 ? &p.k : &p.v);
  if (tid == 0) {
    s_failed = 0;
    s_poison = 0;
    tc::mbar_init(tc::smem_addr(&bars.q));
    tc::mbar_init(tc::smem_addr(&bars.pv));
    for (int i = 0; i < ST; ++i) {
      tc::mbar_init(tc::smem_addr(&bars.kv_full[i]));
      tc::mbar_init(tc::smem_addr(&bars.kv_empty[i]));
    }
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(tc::smem_addr(&bars.s_full[i]));
      mbar_init_n(tc::smem_addr(&bars.p_full[i]), 4);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  griddep_wait();

  const bool tell = tid == 0 && blockIdx.x == 0 && h == 0;
  const int plen = p.prefix_len ? checked_len(*p.prefix_len, p.prefix_rows, p.err, tell && b == 0) : p.prefix_rows;
  int own = 0, ql = p.tokens, start = 0;
  if (p.kv_len) {
    own = checked_len(p.kv_len[b], p.cache_len, p.err, tell);
    if (p.q_len) ql = checked_len(p.q_len[b], p.tokens, p.err, tell);
    if (own < ql && tell && p.err) atomicOr(p.err, KANI_FLAG_SLOT_OOB);
    start = max(own - ql, 0);
  }
  // own rows that the tile's last real token sees
  const int t_end = min(t0 + p.tpt, ql);
  const int vis = t_end > t0 ? min(own, start + t_end) : 0;
  const int np = t_end > t0 ? (plen + kKeys - 1) / kKeys : 0;
  const int tiles = np + (vis + kKeys - 1) / kKeys;
  const int first = (int)((int64_t)tiles * split / p.splits);
  const int nt = (int)((int64_t)tiles * (split + 1) / p.splits) - first;

  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = s_tmem;
  // only now: a dependent of this launch may rely on the launches before it, and one that
  // needs tensor memory must not come between this block and its own
  griddep_launch_dependents();

  // n finished (or, for partials, unnormalised) columns from c on of the tile's row r
  auto store = [&](int r, int c, float2 ml, const float* f, int n) {
    const int tok = t0 + r / G, hq = h * G + r % G;
    if (p.ml) {
      const int64_t at = (int64_t)(split / p.cluster) * p.rows + ((int64_t)b * p.tokens + tok) * p.hq + hq;
      if (c == 0) *reinterpret_cast<float2*>(p.ml + at * 2) = ml;
      for (int i = 0; i < n; i += 4)
        *reinterpret_cast<float4*>(p.acc + at * D + c + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
    } else {
      T* o = static_cast<T*>(p.out) + b * p.ob + (int64_t)tok * p.ot + (int64_t)hq * p.oh + c;
      for (int i = 0; i < n; i += 8) st16(o + i, pack16<T>(f + i));
    }
  };
  auto stage_k = [&](int j) { return ring + (uint32_t)(j % ST) * 2u * Shape::kTileBytes; };
  auto bar = [&](const uint64_t& x) { return tc::smem_addr(&x); };

  if (warp == 4) {
    if (nt > 0 && elect_one()) {
      tc::expect_tx(bar(bars.q), (uint32_t)(G * p.tpt) * D * 2);
#pragma unroll
      for (int c = 0; c < D / 64; ++c)
        tma_load_4d(q_smem + c * kRows * 128, &p.q, c * 64, h * G, t0, b * p.qb_step, bar(bars.q));
      int issued = 0;
      for (int j = 0; j < nt; ++j) {
        if (j >= ST && !tc::wait(bar(bars.kv_empty[j % ST]), (uint32_t)((j / ST - 1) & 1))) break;
        const uint32_t full = bar(bars.kv_full[j % ST]);
        tc::expect_tx(full, 2 * Shape::kTileBytes);
        const int jt = first + j;
        const bool pre = jt < np;
        const int row = (pre ? jt : jt - np) * kKeys;
        const int ch = pre ? h * p.ph_step : h * p.h_step, cb = pre ? 0 : b * p.b_step;
        const CUtensorMap* mk = pre ? &p.pk : &p.k;
        const CUtensorMap* mv = pre ? &p.pv : &p.v;
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
          tma_load_4d(stage_k(j) + c * kKeys * 128, mk, c * 64, row, ch, cb, full);
          tma_load_4d(stage_k(j) + Shape::kTileBytes + c * kKeys * 128, mv, c * 64, row, ch, cb, full);
        }
        issued = j + 1;
      }
      // every copy has landed before the block may end
      bool ok = tc::wait(bar(bars.q), 0u) && issued == nt;
      for (int j = max(0, issued - ST); j < issued; ++j)
        ok &= tc::wait(bar(bars.kv_full[j % ST]), (uint32_t)((j / ST) & 1));
      if (!ok) atomicOr(&s_failed, 1);
    }
  } else if (warp == 5) {
    if (nt > 0 && elect_one()) {
      const uint32_t id_s = tc::idesc_f16<T>(kRows, kKeys);
      const uint32_t id_o = tc::idesc_f16<T>(kRows, D) | (1u << 16);  // B is MN-major
      auto qk = [&](int j) {
        if (!tc::wait(bar(bars.kv_full[j % ST]), (uint32_t)((j / ST) & 1))) return false;
        tc::fence_after_sync();
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
          tc::mma_f16(tmem + (uint32_t)(j & 1) * 64u,
                      tc::desc_sw128(q_smem + (uint32_t)(i >> 2) * (kRows * 128) + (uint32_t)(i & 3) * 32u),
                      tc::desc_sw128(stage_k(j) + (uint32_t)(i >> 2) * (kKeys * 128) + (uint32_t)(i & 3) * 32u), id_s,
                      i > 0);
        tc::commit(bar(bars.s_full[j & 1]));
        return true;
      };
      bool ok = tc::wait(bar(bars.q), 0u) && qk(0);
      for (int j = 0; ok && j < nt; ++j) {
        if (j + 1 < nt && !(ok = qk(j + 1))) break;
        if (!(ok = tc::wait(bar(bars.p_full[j & 1]), (uint32_t)((j >> 1) & 1)))) break;
        tc::fence_after_sync();
#pragma unroll
        for (int i = 0; i < kKeys / 16; ++i)
          mma_f16_ts(tmem + kTmemO, tmem + (uint32_t)(j & 1) * 64u + (uint32_t)i * 8u,
                     desc_v(stage_k(j) + Shape::kTileBytes + (uint32_t)i * 2048u), id_o, j > 0 || i > 0);
        tc::commit(bar(bars.kv_empty[j % ST]));
        tc::commit(bar(bars.pv));
      }
      // the last product is done before tensor memory is freed, its arrivals before the block ends
      if (ok) ok = tc::wait(bar(bars.pv), (uint32_t)((nt - 1) & 1)) &&
                   tc::wait(bar(bars.kv_empty[(nt - 1) % ST]), (uint32_t)(((nt - 1) / ST) & 1));
      if (!ok) atomicOr(&s_failed, 1);
    }
  } else {
    // ---- one query row per thread
    const int tok = t0 + tid / G;
    const bool row_ok = tid < G * p.tpt && tok < p.tokens;
    const bool real = row_ok && tok < ql;
    const int lim = real ? min(own, start + tok + 1) : 0;  // own rows that this row sees
    const int all = min(own, start + t0 + 1);              // own rows that every real row sees
    const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
    float m = -INFINITY, l = 0.f;
    bool ok = true, live = real;  // live: the row's maximum may still move
    auto wait_all = [&](const uint64_t& x, uint32_t parity) {  // the same answer in all lanes
      return ok = __all_sync(0xffffffffu, tc::wait(bar(x), parity));
    };
    for (int j = 0; j < nt; ++j) {
      if (!wait_all(bars.s_full[j & 1], (uint32_t)((j >> 1) & 1))) break;
      tc::fence_after_sync();
      const uint32_t sp = lanes + (uint32_t)(j & 1) * 64u;
      const int jt = first + j;
      const bool pre = jt < np;
      const int row0 = (pre ? jt : jt - np) * kKeys;
      const bool ragged = row0 + kKeys > (pre ? plen : all);  // some row may not see all of the tile
      const int n = ragged ? (pre ? (real ? plen : 0) : lim) - row0 : kKeys;  // of them this row sees the first n
      auto load_s = [&](uint32_t (&s)[64]) {
        tmem_ld32(sp, s);
        tmem_ld32(sp + 32u, s + 32);
        tmem_wait_ld();
        if (ragged) {
#pragma unroll
          for (int i = 0; i < 64; ++i)
            if (i >= n) s[i] = 0xff800000u;  // -inf
        }
      };
      // The weights relative to the maximum so far, without looking for a new one: a
      // sum that passes 2^10 (or a row that has no maximum yet) shows that it is needed.
      // Only such rows move, so a row's result does not depend on the others of its warp.
      uint32_t pk[32];
      float tile_sum = 0.f;
      auto weights = [&](auto mixed, auto always, bool want) {
        const float ms = m == -INFINITY ? 0.f : m;
        const float2 c2 = make_float2(p.qscale, p.qscale), m2 = make_float2(-ms, -ms);
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        uint32_t s[64];
        load_s(s);
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const float2 x = __ffma2_rn(make_float2(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), c2, m2);
          float2 w;
          if constexpr (decltype(mixed)::value && Shape::kFmaOneIn > 0)
            w = i % Shape::kFmaOneIn == 0 ? exp2_fma(x) : make_float2(ex2(x.x), ex2(x.y));
          else
            w = make_float2(ex2(x.x), ex2(x.y));
          sum[i & 1] = __fadd2_rn(sum[i & 1], w);
          const uint32_t both = pack2<T>(w.x, w.y);
          pk[i] = decltype(always)::value || want ? both : pk[i];
        }
        if (decltype(always)::value || want) tile_sum = (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
      };
      // A row whose logits have all been -inf asks again in every tile, one that has met a
      // NaN does not.  The rows beside it are served as ever: the pass is left out only
      // where no row has a maximum to go by, as in the first tile.
      bool move = live && m == -INFINITY && n > 0;
      bool pass = !__any_sync(0xffffffffu, move);
      if (!pass) pass = __any_sync(0xffffffffu, m != -INFINITY);
      if (pass) {
        if (ragged) weights(std::false_type{}, std::true_type{}, true);
        else weights(std::true_type{}, std::true_type{}, true);
        move = move || (live && tile_sum > kMaxSum);
      }
      if (__any_sync(0xffffffffu, move)) {
        float mx = -INFINITY;
        {
          uint32_t s[64];
          load_s(s);
#pragma unroll
          for (int i = 0; i < 64; i += 2) mx = max3(mx, __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
        }
        const float mn = move ? fmaxf(m, mx * p.qscale) : m, w = move ? merge_weight(m, mn) : 1.f;
        if (j > 0) {
          if (!wait_all(bars.pv, (uint32_t)((j - 1) & 1))) break;
          tc::fence_after_sync();
          l *= w;
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            uint32_t o[32];
            tmem_ld32(lanes + kTmemO + (uint32_t)c, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * w);
            tmem_st32(lanes + kTmemO + (uint32_t)c, o);
          }
        }
        m = mn;
        weights(std::false_type{}, std::false_type{}, !pass || move);
        live = live && tile_sum == tile_sum;
      }
      l += tile_sum;
      tmem_st32(sp, pk);  // over S, which has been read
      if (ragged) {
        // V rows that no query of the tile may see become zero; so do values that are
        // not finite in rows that only some of them see (added again at the end)
        if (!wait_all(bars.kv_full[j % ST], (uint32_t)((j / ST) & 1))) break;
        const int end = (pre ? plen : vis) - row0, some = (pre ? plen : all) - row0;
        for (int i = tid; i < kKeys * D / 8; i += kSoftmaxThreads) {
          const int c = i / (kKeys * 8), r = i / 8 % kKeys;
          if (r < some) continue;
          const uint32_t at = stage_k(j) + Shape::kTileBytes + (uint32_t)(c * kKeys * 128 + r * 128 + (((i & 7) ^ (r & 7)) << 4));
          uint4 x = make_uint4(0u, 0u, 0u, 0u);
          if (r < end) {
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w)
                         : "r"(at));
            uint32_t w[4] = {x.x, x.y, x.z, x.w};
            bool bad = false;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if (not_finite16<T>(w[e])) w[e] &= 0xffff0000u, bad = true;
              if (not_finite16<T>(w[e] >> 16)) w[e] &= 0xffffu, bad = true;
            }
            if (!bad) continue;
            s_poison = 1;
            x = make_uint4(w[0], w[1], w[2], w[3]);
          }
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(x.x), "r"(x.y), "r"(x.z), "r"(x.w)
                       : "memory");
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      }
      tmem_wait_st();
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(bars.p_full[j & 1]));
    }
    if (ok && nt > 0) wait_all(bars.pv, (uint32_t)((nt - 1) & 1));
    if (!ok) atomicOr(&s_failed, 1);
    tc::fence_after_sync();
    asm volatile("bar.sync 1, 128;" ::: "memory");  // every warp's s_poison
    const int poisoned = *(volatile int*)&s_poison;
    const bool seen = ok && nt > 0 && real && l != 0.f;
    const float inv = p.ml || p.cluster > 1 ? 1.f : (seen ? 1.f / l : 0.f);
    float* red = reinterpret_cast<float*>(smem_raw + (base - tc::smem_addr(smem_raw))) + tid * RED;
    if (p.cluster > 1) s_ml[tid] = make_float2(m, seen ? l : 0.f);
#pragma unroll 1
    for (int c = 0; c < D; c += 32) {
      float f[32];
      if (nt > 0 && ok) {
        uint32_t raw[32];
        tmem_ld32(lanes + kTmemO + (uint32_t)c, raw);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; ++i) f[i] = seen ? __uint_as_float(raw[i]) * inv : 0.f;
        if (poisoned) {
          // own rows of this CTA's partly visible tiles that this row does see
          const int lo = max(all / kKeys * kKeys, (max(first, np) - np) * kKeys), hi = min(lim, (first + nt - np) * kKeys);
          for (int r = lo; r < hi; ++r) {
            const uint16_t* vr = static_cast<const uint16_t*>(p.v_raw) + b * p.vb + h * p.vh + (int64_t)r * p.vs + c;
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (r >= all && not_finite16<T>(vr[i])) f[i] += tc::from_bits16<T>(vr[i]);
          }
        }
        if (p.cluster > 1) {  // (every operand has been read: the last product is done)
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            *reinterpret_cast<float4*>(red + c + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) f[i] = 0.f;
      }
      if (p.cluster == 1 && row_ok) store(tid, c, make_float2(m, seen ? l : 0.f), f, 32);
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  if (warp == 5) tc::tmem_free(tmem, kTmemCols);
  if (tid == 0 && s_failed && p.err) atomicOr(p.err, KANI_FLAG_TIMEOUT);
  if (p.cluster == 1) return;
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();  // every CTA's O lies in its shared memory
  const int rank = (int)cluster.block_rank(), share = kRows / p.cluster;
  const float* red0 = reinterpret_cast<const float*>(smem_raw + (base - tc::smem_addr(smem_raw)));
  for (int i = tid; i < share * (D / 8); i += kFlashThreads) {
    const int r = rank * share + i / (D / 8), c = i % (D / 8) * 8;
    if (r >= G * p.tpt || t0 + r / G >= p.tokens) continue;
    float2 st[8];
    float mx = -INFINITY;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      st[k] = k < p.cluster ? *cluster.map_shared_rank(&s_ml[r], k) : make_float2(-INFINITY, 0.f);
      mx = fmaxf(mx, st[k].x);
    }
    float4 a[8], e[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      a[k] = e[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (st[k].y != 0.f) {  // else that CTA's tiles hold nothing for this row (or there is none)
        const float* o = cluster.map_shared_rank(red0 + r * RED + c, k);
        a[k] = *reinterpret_cast<const float4*>(o);
        e[k] = *reinterpret_cast<const float4*>(o + 4);
      }
    }
    float ls = 0.f, f[8] = {};
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float w = merge_weight(st[k].x, mx);
      ls += st[k].y * w;
      f[0] += a[k].x * w, f[1] += a[k].y * w, f[2] += a[k].z * w, f[3] += a[k].w * w;
      f[4] += e[k].x * w, f[5] += e[k].y * w, f[6] += e[k].z * w, f[7] += e[k].w * w;
    }
    if (!p.ml) {
      const float inv = ls == 0.f ? 0.f : 1.f / ls;
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = ls == 0.f ? 0.f : f[k] * inv;
    }
    store(r, c, make_float2(mx, ls), f, 8);
  }
  cluster.sync();  // the other CTAs have read this one's memory
}

// {64 elements, n1, n2, n3} map of 16-bit rows, in boxes of 64 x b1 x b2; strides in elements
bool encode_4d(CUtensorMap* map, bool bf16, const void* base, int d, int64_t n1, int64_t s1, int64_t n2, int64_t s2,
               int64_t n3, int64_t s3, int b1, int b2) {
  // the stride of a dimension of one element is never followed, but has to be valid
  auto st = [&](int64_t n, int64_t s) { return (cuuint64_t)(n > 1 ? s : d) * 2u; };
  const cuuint64_t dims[4] = {(cuuint64_t)d, (cuuint64_t)n1, (cuuint64_t)n2, (cuuint64_t)n3};
  const cuuint64_t strides[3] = {st(n1, s1), st(n2, s2), st(n3, s3)};
  const cuuint32_t box[4] = {64u, (cuuint32_t)b1, (cuuint32_t)b2, 1u};
  return tc::encode_map(map, bf16, base, 4, dims, strides, box);
}

int64_t m_tiles_of(int64_t tokens, int group) {
  const int tpt = kRows / group;
  return (tokens + tpt - 1) / tpt;
}

}  // namespace

FlashSplit flash_split(int64_t batch, int64_t tokens, int hq, int hk, int64_t rows, int most_parts) {
  const int64_t ctas = batch * hk * m_tiles_of(tokens, hq / hk);
  const int64_t tiles = std::max<int64_t>(1, (rows + kKeys - 1) / kKeys);
  FlashSplit s = {1, 1};
  while (s.cluster < 8 && ctas * s.cluster * 2 <= 2 * sm_count() && s.cluster * 2 <= tiles) s.cluster *= 2;
  if (s.cluster == 8)
    s.parts = (int)std::max<int64_t>(1, std::min<int64_t>({sm_count() / (ctas * 8), tiles / 32, most_parts}));
  return s;
}

template <typename T, int D>
static int launch_flash_t(const FlashParams& f, int hk, int batch, bool dependent, cudaStream_t s) {
  auto kern = prefix_flash_kernel<T, D>;
  static std::atomic<uint64_t> granted{0};
  if (const int e = grant_smem(kern, FlashShape<D>::kSmem, granted)) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(f.m_tiles * f.splits), (unsigned)hk, (unsigned)batch);
  cfg.blockDim = dim3(kFlashThreads);
  cfg.dynamicSmemBytes = FlashShape<D>::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)f.cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = dependent ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, f);
  note_launch();
  return e == cudaSuccess ? KANI_OK : (int)e;
}

int launch_flash(const Params& p, int32_t dtype, int d, int batch, int tokens, bool own_rows, FlashSplit split,
                 float* ml, float* acc, bool dependent, cudaStream_t s) {
  const bool bf16 = dtype == KANI_DTYPE_BF16;
  FlashParams f;
  memset(&f, 0, sizeof(f));
  f.tpt = kRows / p.group;
  // the expanded dimensions (stride 0) of Q and the caches are one element to the copies
  const bool qb = batch > 1 && p.qb != 0;
  f.qb_step = qb;
  f.b_step = p.cb != 0;
  f.h_step = p.ch != 0;
  f.ph_step = p.ph != 0;
  bool enc = encode_4d(&f.q, bf16, p.q, d, p.hq, p.qh, tokens, p.qt, qb ? batch : 1, p.qb, p.group, f.tpt);
  f.pk = f.pv = f.k = f.v = f.q;
  if (p.prefix_rows > 0)
    for (int i = 0; i < 2; ++i)
      enc = enc && encode_4d(i ? &f.pv : &f.pk, bf16, i ? p.pv : p.pk, d, p.prefix_rows, p.ps, f.ph_step ? p.hk : 1, p.ph,
                             1, 0, kKeys, 1);
  if (own_rows && p.cache_len > 0)
    for (int i = 0; i < 2; ++i)
      enc = enc && encode_4d(i ? &f.v : &f.k, bf16, i ? p.v : p.k, d, p.cache_len, p.cs, f.h_step ? p.hk : 1, p.ch,
                             f.b_step ? batch : 1, p.cb, kKeys, 1);
  if (!enc) return KANI_ERR_UNSUPPORTED;
  f.kv_len = own_rows ? p.kv_len : nullptr;
  f.q_len = p.q_len;
  f.prefix_len = p.prefix_len;
  f.v_raw = p.v;
  f.vb = p.cb;
  f.vh = p.ch;
  f.vs = p.cs;
  f.out = p.out;
  f.ob = p.ob;
  f.ot = p.ot;
  f.oh = p.oh;
  f.ml = ml;
  f.acc = acc;
  f.rows = (int64_t)batch * tokens * p.hq;
  f.err = p.err;
  f.qscale = p.qscale;
  f.tokens = tokens;
  f.group = p.group;
  f.hq = p.hq;
  f.cluster = split.cluster;
  f.splits = split.cluster * split.parts;
  f.m_tiles = (int)m_tiles_of(tokens, p.group);
  f.prefix_rows = (int)p.prefix_rows;
  f.cache_len = own_rows ? (int)p.cache_len : 0;
  if (bf16)
    return d == 64 ? launch_flash_t<__nv_bfloat16, 64>(f, p.hk, batch, dependent, s)
                   : launch_flash_t<__nv_bfloat16, 128>(f, p.hk, batch, dependent, s);
  return d == 64 ? launch_flash_t<__half, 64>(f, p.hk, batch, dependent, s)
                 : launch_flash_t<__half, 128>(f, p.hk, batch, dependent, s);
}

}  // namespace prefix
}  // namespace kani

extern "C" int kani_prefix_prefill_attention(
    int32_t dtype, int64_t batch, int64_t tokens, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
    const void* q, int64_t q_batch_stride, int64_t q_token_stride, int64_t q_head_stride, const void* k_cache,
    const void* v_cache, int64_t cache_batch_stride, int64_t cache_head_stride, int64_t cache_slot_stride,
    int64_t cache_len, const int64_t* kv_len, const int64_t* q_len, const void* prefix_k, const void* prefix_v,
    int64_t prefix_head_stride, int64_t prefix_row_stride, int64_t prefix_rows, const int64_t* prefix_len,
    float scale, void* out, int64_t out_batch_stride, int64_t out_token_stride, int64_t out_head_stride,
    int32_t* err_flag, void* stream) {
  using namespace kani;
  if (batch < 0 || tokens < 0 || num_q_heads < 0 || num_kv_heads < 0 || head_dim < 0 || cache_len < 0 ||
      prefix_rows < 0)
    return KANI_ERR_INVALID_ARG;
  if (batch == 0 || tokens == 0 || num_q_heads == 0) return KANI_OK;
  prefix::Params p = {};
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
  if (const int bad = prefix::check_params(p, dtype, batch, tokens, num_q_heads, num_kv_heads, head_dim, scale))
    return bad;
  return prefix::launch_flash(p, dtype, head_dim, (int)batch, (int)tokens, true,
                              prefix::flash_split(batch, tokens, num_q_heads, num_kv_heads, prefix_rows + cache_len, 1),
                              nullptr, nullptr, false, static_cast<cudaStream_t>(stream));
}
