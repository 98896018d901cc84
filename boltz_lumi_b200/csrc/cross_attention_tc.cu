// Cross attention forward on tcgen05 tensor cores (bf16; see cross_attention.cuh).
//
// One CTA = kTiles tiles of 128 query rows of one (sample, head) over key tiles
// of 64.  Warp 0 feeds the tiles by TMA, warp 1 issues the MMAs, and four softmax
// warps per query tile own one row per thread (TMEM lane = row):
//   * S = Q K^T into one of two TMEM buffers per query tile (128 x 64, fp32), so the
//     next tile's S is computed while this tile's softmax runs;
//   * the thread reads its 64 scores (tcgen05.ld), adds the bias row from shared
//     memory (128-byte swizzle: conflict-free 16-byte reads), takes p = exp2 and
//     writes P as bf16 over the S columns it came from;
//   * O += P V with P from TMEM and V in its natural [key][d] order (MN-major);
//     O is rescaled only when a row's maximum grew by more than 2^8.
// What bounds it: one exponential per score (16 per clock and SM) and, with a bias,
// the bias bytes through L2; the products are a third of that.  Two query tiles per
// CTA halve the K / V bytes that each score costs; with few tiles one per CTA
// spreads them over more SMs.
#include "cross_attention.cuh"
#include "tc.cuh"

namespace bl {
namespace xa {
namespace {

constexpr int kBQ = 128, kBK = 64;
constexpr float kRescale = 8.f;  // log2 of the growth of a maximum that rescales O

template <int kTiles, int kBlocks, bool kBias> struct Shape {  // kBlocks: 64-column blocks of d
  static constexpr int kSoftWarps = 4 * kTiles, kThreads = (2 + kSoftWarps) * 32;
  static constexpr int kKvStages = kBias ? (kBlocks == 2 && kTiles == 2 ? 2 : 3) : (kBlocks == 2 ? 3 : 4);
  static constexpr int kBiasStages = kBlocks == 2 ? 2 : (kTiles == 2 ? 3 : 2);
  static constexpr int kQ = kBQ * 128 * kBlocks;         // bytes of one query tile
  static constexpr int kK = kBK * 128 * kBlocks;         // bytes of a K or V tile
  static constexpr int kB = kBias ? kBQ * kBK * 2 : 0;   // bytes of a bias tile
  static constexpr int kKvOff = kTiles * kQ;
  static constexpr int kBiasOff = kKvOff + kKvStages * 2 * kK;
  static constexpr int kMaskOff = kBiasOff + kTiles * kBiasStages * kB;  // [softmax warp][64] fp32
  static constexpr int kBarOff = kMaskOff + kSoftWarps * kBK * 4;
  static constexpr int kBytes = kBarOff + 384 + 1024;
  static constexpr uint32_t kTmem = kTiles == 2 ? 512 : 256;
  static constexpr uint32_t kOCol = kTiles * 2 * kBK;    // O of tile t at kOCol + t * 128
};

struct TcArgs {
  Args a;
  int q_tiles;  // CTAs per (sample, head)
  unsigned int *status;
};

__device__ __forceinline__ void tma_load_4d(void *dst, const CUtensorMap *map, uint64_t *bar, int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(smem_addr(dst)), "l"(map), "r"(smem_addr(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}
// 128-byte swizzle, K-major (LBO unused), 8-row groups 1024 bytes apart.
__device__ __forceinline__ uint64_t desc_k(uint32_t saddr) {
  return uint64_t((saddr & 0x3FFFFu) >> 4) | (uint64_t(1) << 16) | (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) |
         (uint64_t(2) << 61);
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint64_t pack2(uint32_t lo, uint32_t hi) { return (uint64_t(hi) << 32) | lo; }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity, unsigned int *status, unsigned code) {
  return __all_sync(0xffffffffu, tc::mbar_wait(bar, parity, status, code));
}

template <int kTiles, int kBlocks, bool kBias>
__global__ void __launch_bounds__(Shape<kTiles, kBlocks, kBias>::kThreads, kTiles == 1 ? 2 : 1)
    flash_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                    const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_bias,
                    const TcArgs x) {
  using S = Shape<kTiles, kBlocks, kBias>;
  constexpr int KV = S::kKvStages, BS = S::kBiasStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + S::kBarOff);
  uint64_t *q_full = bars;
  uint64_t *kv_full = q_full + 1;              // [KV] K and V of a key tile landed
  uint64_t *kv_empty = kv_full + KV;           // [KV] its P.V products are done
  uint64_t *b_full = kv_empty + KV;            // [tile][BS] bias block landed
  uint64_t *b_empty = b_full + kTiles * BS;    // [tile][BS] the softmax warps have read it
  uint64_t *s_full = b_empty + kTiles * BS;    // [tile][2] S in TMEM
  uint64_t *p_full = s_full + kTiles * 2;      // [tile][2] P in TMEM (and O rescaled if needed)
  uint64_t *pv_done = p_full + kTiles * 2;     // [tile][2] P.V of that buffer is done
  uint64_t *o_full = pv_done + kTiles * 2;     // [tile] every P.V is done
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(o_full + kTiles);
  int *last_key = reinterpret_cast<int *>(tmem_slot + 1);

  const Args &a = x.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int tile, h, b;
  decode_cta(a, blockIdx.x, x.q_tiles, a.heads, tile, h, b);
  const int q0 = tile * kTiles * kBQ, hk = h / a.group, bb = b / a.share;
  const int live = a.nq - q0 > kBQ ? kTiles : 1;  // query tiles with rows

  if (tid == 0) {
    tc::mbar_init(q_full, 1);
    for (int i = 0; i < KV; ++i) tc::mbar_init(kv_full + i, 1), tc::mbar_init(kv_empty + i, 1);
    for (int i = 0; i < kTiles * BS; ++i) tc::mbar_init(b_full + i, 1), tc::mbar_init(b_empty + i, 4);
    for (int i = 0; i < kTiles * 2; ++i)
      tc::mbar_init(s_full + i, 1), tc::mbar_init(p_full + i, 4), tc::mbar_init(pv_done + i, 1);
    for (int i = 0; i < kTiles; ++i) tc::mbar_init(o_full + i, 1);
    tc::fence_mbar_init();
    *last_key = -1;
  }
  if (warp == 1) {
    tc::tmem_alloc(tmem_slot, S::kTmem);
    tc::tmem_relinquish();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // Key tiles past the last kept key (a padded batch) are not visited.
  int keys = a.nk;
  if (a.mask_kind == kMaskKeep) {
    const uint8_t *mask = static_cast<const uint8_t *>(a.mask) + b * a.mask_sb;
    for (int end = a.nk; end > 0; end -= 8 * S::kThreads) {
      int best = -1;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int j = end - 1 - e * S::kThreads - tid;
        if (j >= 0 && mask[j] && best < j) best = j;
      }
      if (best >= 0) atomicMax(last_key, best);
      if (__syncthreads_or(best >= 0)) break;
    }
    keys = *last_key + 1;
  }
  const int n_tiles = (keys + kBK - 1) / kBK;

  if (warp == 0) {
    // ---------------- TMA producer ----------------
    if (lane == 0 && n_tiles > 0) {
      tc::prefetch_tmap(&map_q);
      tc::prefetch_tmap(&map_k);
      tc::prefetch_tmap(&map_v);
      tc::mbar_arrive_expect_tx(q_full, live * S::kQ);
      for (int t = 0; t < live; ++t)
        for (int c = 0; c < kBlocks; ++c)
          tma_load_4d(smem + t * S::kQ + c * kBQ * 128, &map_q, q_full, 64 * c, q0 + t * kBQ, h, b);
      bool ok = true;
      for (int j = 0; j < n_tiles && ok; ++j) {
        const int s = j % KV;
        if (j >= KV && !(ok = tc::mbar_wait(kv_empty + s, ((j / KV) & 1) ^ 1u, x.status, 0x301))) break;
        uint8_t *st = smem + S::kKvOff + s * 2 * S::kK;
        tc::mbar_arrive_expect_tx(kv_full + s, 2 * S::kK);
        for (int c = 0; c < kBlocks; ++c) tma_load_4d(st + c * kBK * 128, &map_k, kv_full + s, 64 * c, j * kBK, hk, b);
        for (int c = 0; c < kBlocks; ++c)
          tma_load_4d(st + S::kK + c * kBK * 128, &map_v, kv_full + s, 64 * c, j * kBK, hk, b);
        if constexpr (kBias) {
          const int bs = j % BS;
          for (int t = 0; t < live; ++t) {
            uint64_t *full = b_full + t * BS + bs;
            if (j >= BS && !(ok = tc::mbar_wait(b_empty + t * BS + bs, ((j / BS) & 1) ^ 1u, x.status, 0x302))) break;
            tc::mbar_arrive_expect_tx(full, S::kB);
            tma_load_4d(smem + S::kBiasOff + (t * BS + bs) * S::kB, &map_bias, full, j * kBK, q0 + t * kBQ, h, bb);
          }
        }
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    if (lane == 0 && n_tiles > 0 && tc::mbar_wait(q_full, 0, x.status, 0x303)) {
      constexpr uint32_t idesc_s = tc::idesc_bf16(kBQ, kBK, false, false);
      const int steps = (a.d + 15) / 16;  // columns past d are zero
      const uint32_t idesc_pv = tc::idesc_bf16(kBQ, 16 * steps, false, true);
      const uint32_t base = smem_addr(smem);
      auto issue_s = [&](int t, int j) {
        const int s = j % KV, buf = j & 1;
        if (!tc::mbar_wait(kv_full + s, (j / KV) & 1, x.status, 0x304)) return false;
        // The buffer held P of tile j - 2: its P.V must have read it.
        if (j >= 2 && !tc::mbar_wait(pv_done + t * 2 + buf, ((j - 2) >> 1) & 1, x.status, 0x305)) return false;
        tc::tc_fence_after();
        const uint32_t q = base + t * S::kQ, k = base + S::kKvOff + s * 2 * S::kK;
        for (int e = 0; e < steps; ++e)
          tc::umma_f16_ss(tmem + (t * 2 + buf) * kBK, desc_k(q + (e >> 2) * kBQ * 128 + (e & 3) * 32),
                          desc_k(k + (e >> 2) * kBK * 128 + (e & 3) * 32), idesc_s, e != 0);
        tc::umma_commit(s_full + t * 2 + buf);
        return true;
      };
      bool ok = true;
      for (int t = 0; t < live && ok; ++t) ok = issue_s(t, 0);
      for (int j = 0; j < n_tiles && ok; ++j) {
        const int s = j % KV, buf = j & 1;
        for (int t = 0; t < live && ok; ++t) {
          if (j + 1 < n_tiles && !(ok = issue_s(t, j + 1))) break;
          if (!(ok = tc::mbar_wait(p_full + t * 2 + buf, (j >> 1) & 1, x.status, 0x306))) break;
          tc::tc_fence_after();
          const uint32_t v = base + S::kKvOff + s * 2 * S::kK + S::kK;
#pragma unroll
          for (int e = 0; e < kBK / 16; ++e)
            tc::umma_f16_ts(tmem + S::kOCol + t * 128, tmem + (t * 2 + buf) * kBK + e * 8,
                            tc::desc_sw128(v + e * 2048, kBK * 128), idesc_pv, (j | e) != 0);
          tc::umma_commit(pv_done + t * 2 + buf);
          if (t + 1 == live) tc::umma_commit(kv_empty + s);
          if (j + 1 == n_tiles) tc::umma_commit(o_full + t);
        }
      }
    }
  } else {
    // ---------------- softmax and epilogue: one query row per thread ----------------
    const int t = (warp - 2) >> 2, quarter = warp & 3;
    const int row = quarter * 32 + lane, i = q0 + t * kBQ + row;
    const uint32_t lanes = tmem + (uint32_t(quarter * 32) << 16);
    const uint32_t o_col = lanes + S::kOCol + t * 128;
    float *mk = reinterpret_cast<float *>(smem + S::kMaskOff) + (warp - 2) * kBK;  // this warp's copy
    const int d16 = (a.d + 15) / 16;
    float m = -INFINITY;           // reference of the exponentials
    uint64_t sum2 = 0;             // two partial row sums
    bool ok = t < live;
    float mv[2] = {0.f, 0.f};
    if (ok && n_tiles > 0)
#pragma unroll
      for (int e = 0; e < 2; ++e) mv[e] = mask_value(a, b, lane + 32 * e);
    for (int j = 0; j < n_tiles && ok; ++j) {
      const int buf = j & 1;
      // Mask of this tile (and the keys past nk), from the values read one tile ago.
      const bool masked = __any_sync(0xffffffffu, mv[0] != 0.f || mv[1] != 0.f);
      const uint32_t cut0 = __ballot_sync(0xffffffffu, mv[0] == -INFINITY), cut1 = __ballot_sync(0xffffffffu, mv[1] == -INFINITY);
      if (masked) {
        __syncwarp();
        mk[lane] = mv[0], mk[lane + 32] = mv[1];
        __syncwarp();
      }
      if (j + 1 < n_tiles)
#pragma unroll
        for (int e = 0; e < 2; ++e) mv[e] = mask_value(a, b, (j + 1) * kBK + lane + 32 * e);
      if (!(ok = warp_wait(s_full + t * 2 + buf, (j >> 1) & 1, x.status, 0x307))) break;
      tc::tc_fence_after();
      uint32_t sv[2][32];
      tc::tmem_ld_32x32b_x32(lanes + (t * 2 + buf) * kBK, sv[0]);
      tc::tmem_ld_32x32b_x32(lanes + (t * 2 + buf) * kBK + 32, sv[1]);
      const int bs = j % BS;
      if constexpr (kBias) {
        if (!(ok = warp_wait(b_full + t * BS + bs, (j / BS) & 1, x.status, 0x308))) {
          tc::tmem_ld_wait();
          break;
        }
      }
      tc::tmem_ld_wait_regs(sv[0], sv[1]);
      uint64_t y[32];  // the scores, in pairs
      const uint64_t scale2 = dup2(a.scale);
      if constexpr (kBias) {
        const uint32_t brow = smem_addr(smem + S::kBiasOff + (t * BS + bs) * S::kB) + row * 128;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const uint4 v = lds128(brow + ((c ^ (row & 7)) << 4));
          const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int p = 4 * c + e;
            y[p] = fma2(pack2(sv[p >> 4][(2 * p) & 31], sv[p >> 4][(2 * p + 1) & 31]), scale2,
                        pack2(w[e] << 16, w[e] & 0xffff0000u));
          }
        }
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(b_empty + t * BS + bs);
      } else {
#pragma unroll
        for (int p = 0; p < 32; ++p)
          y[p] = mul2(pack2(sv[p >> 4][(2 * p) & 31], sv[p >> 4][(2 * p + 1) & 31]), scale2);
      }
      if (masked) {
#pragma unroll
        for (int p = 0; p < 32; ++p) {
          const float2 mp = *reinterpret_cast<const float2 *>(mk + 2 * p);
          const float lo = mp.x == -INFINITY ? mp.x : lo_f(y[p]) + mp.x, hi = mp.y == -INFINITY ? mp.y : hi_f(y[p]) + mp.y;
          y[p] = pack2(__float_as_uint(lo), __float_as_uint(hi));
        }
        if (cut0 | cut1) {
          // V rows of left-out keys must be zero: a zero weight times what they hold may not be.
          if (a.mask_kind == kMaskKeep) {
            const int s = j % KV, key = row >> 1;
            if (((key < 32 ? cut0 >> key : cut1 >> (key - 32)) & 1) != 0) {
              tc::mbar_wait(kv_full + s, (j / KV) & 1, x.status, 0x30B);  // complete: S came from this stage
              uint8_t *v = smem + S::kKvOff + s * 2 * S::kK + S::kK + key * 128 + (row & 1) * 64;
#pragma unroll
              for (int c = 0; c < kBlocks; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  *reinterpret_cast<uint4 *>(v + c * kBK * 128 + e * 16) = make_uint4(0u, 0u, 0u, 0u);
            }
            tc::fence_proxy_async_smem();
          }
        }
      }
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int p = 0; p < 32; ++p) mx[p & 3] = fmaxf(mx[p & 3], fmaxf(lo_f(y[p]), hi_f(y[p])));
      const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
      const bool grow = j > 0 && (top - m) * kLog2e > kRescale;  // NaN (both -inf): no
      if (__any_sync(0xffffffffu, grow)) {
        if (!(ok = warp_wait(pv_done + t * 2 + ((j - 1) & 1), ((j - 1) >> 1) & 1, x.status, 0x309))) break;
        tc::tc_fence_after();
        const float alpha = grow ? fast_exp2((m - top) * kLog2e) : 1.f;
        for (int c = 0; c < d16; ++c) {
          uint32_t o[16];
          tc::tmem_ld_32x32b_x16(o_col + 16 * c, o);
          tc::tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
          tc::tmem_st_32x32b_x16(o_col + 16 * c, o);
        }
        sum2 = mul2(sum2, dup2(alpha));
      }
      if (j == 0 || grow) m = top;
      uint32_t p16[2][16];
      if (__any_sync(0xffffffffu, m < -1e37f && m != -INFINITY)) {
        // A row of the type's lowest values: subtract before the change of base, which would overflow.
        const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int p = 0; p < 32; ++p) {
          const float e0 = fast_exp2((lo_f(y[p]) - base) * kLog2e), e1 = fast_exp2((hi_f(y[p]) - base) * kLog2e);
          sum2 = add2(sum2, pack2(__float_as_uint(e0), __float_as_uint(e1)));
          p16[p >> 4][p & 15] = pack_bf16x2(e0, e1);
        }
      } else {
        const uint64_t log2e2 = dup2(kLog2e), base2 = dup2(m == -INFINITY ? 0.f : -m * kLog2e);
#pragma unroll
        for (int p = 0; p < 32; ++p) {
          const uint64_t z = fma2(y[p], log2e2, base2);
          const float e0 = fast_exp2(lo_f(z)), e1 = fast_exp2(hi_f(z));
          sum2 = add2(sum2, pack2(__float_as_uint(e0), __float_as_uint(e1)));
          p16[p >> 4][p & 15] = pack_bf16x2(e0, e1);
        }
      }
      tc::tmem_st_32x32b_x16(lanes + (t * 2 + buf) * kBK, p16[0]);
      tc::tmem_st_32x32b_x16(lanes + (t * 2 + buf) * kBK + 16, p16[1]);
      tc::tmem_st_wait();
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(p_full + t * 2 + buf);
    }
    // Epilogue: o / l, the gate, one rounding.
    if (t < live && ok) {
      if (n_tiles > 0) ok = warp_wait(o_full + t, 0, x.status, 0x30A);
      tc::tc_fence_after();
      const float l = lo_f(sum2) + hi_f(sum2), inv = l == 0.f ? 0.f : 1.f / l;
      using T = __nv_bfloat16;
      const int64_t at = ((int64_t(b) * a.nq + i) * a.heads + h) * a.d;
      const T *gate = a.gate.p ? static_cast<const T *>(a.gate.p) + b * a.gate.sb + int64_t(i) * a.gate.si + h * a.gate.sh
                               : nullptr;
      T *out = static_cast<T *>(a.out) + at, *low = a.low ? static_cast<T *>(a.low) + at : nullptr;
      if (ok) {
        for (int c = 0; c < d16; ++c) {
          uint32_t o[16];
          if (n_tiles > 0) {
            tc::tmem_ld_32x32b_x16(o_col + 16 * c, o);
            tc::tmem_ld_wait();
          }
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int c0 = 16 * c + 8 * half;
            if (i >= a.nq || c0 >= a.d) continue;  // d is a multiple of 8
            uint4 gv = make_uint4(0u, 0u, 0u, 0u);
            if (gate) gv = *reinterpret_cast<const uint4 *>(gate + c0);
            const uint32_t gw[4] = {gv.x, gv.y, gv.z, gv.w};
            uint32_t ov[4], lv[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float u = n_tiles > 0 ? __uint_as_float(o[8 * half + 2 * e]) * inv : 0.f;
              float w = n_tiles > 0 ? __uint_as_float(o[8 * half + 2 * e + 1]) * inv : 0.f;
              if (gate) {
                u *= 1.f / (1.f + expf(-bf16_lo(gw[e])));
                w *= 1.f / (1.f + expf(-bf16_hi(gw[e])));
              }
              ov[e] = pack_bf16x2(u, w);
              lv[e] = pack_bf16x2(u - bf16_lo(ov[e]), w - bf16_hi(ov[e]));
            }
            *reinterpret_cast<uint4 *>(out + c0) = make_uint4(ov[0], ov[1], ov[2], ov[3]);
            if (low) *reinterpret_cast<uint4 *>(low + c0) = make_uint4(lv[0], lv[1], lv[2], lv[3]);
          }
        }
        if (a.lse && i < a.nq) {
          float *st = a.lse + (int64_t(b) * a.heads + h) * a.nq + i;
          st[0] = l == 0.f ? -INFINITY : m;
          st[a.lse_plane()] = l == 0.f ? 0.f : logf(l);
        }
      }
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, S::kTmem);
  }
}

// Map of a [batch][rows][heads][d] view: box of 64 columns x box_rows rows; false where TMA cannot describe it.
bool rows_map(CUtensorMap *map, const Rows &r, int d, int rows, int heads, int batch, int box_rows) {
  const int64_t strides[3] = {r.si, r.sh, r.sb};
  const int sizes[3] = {rows, heads, batch};
  uint64_t dims[4] = {uint64_t(d), uint64_t(rows), uint64_t(heads), uint64_t(batch)}, bytes[3];
  for (int e = 0; e < 3; ++e) {
    if (sizes[e] > 1 && strides[e] <= 0) return false;
    bytes[e] = sizes[e] > 1 ? uint64_t(strides[e]) * 2 : 16;
    if (bytes[e] >= (uint64_t(1) << 40)) return false;
  }
  const uint32_t box[4] = {64, uint32_t(box_rows), 1, 1};
  return encode_tmap(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, r.p, dims, bytes, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int kTiles, int kBlocks, bool kBias>
int launch_tc(const Args &a, const CUtensorMap (&maps)[4], cudaStream_t stream) {
  using S = Shape<kTiles, kBlocks, kBias>;
  static_assert(S::kBytes <= 232448, "shared memory");
  TcArgs x;
  x.a = a;
  x.q_tiles = (a.nq + kTiles * kBQ - 1) / (kTiles * kBQ);
  x.status = device_status_ptr();
  BL_REQUIRE(x.status, "bl_cross_attention: device status word unavailable");
  const int64_t ctas = int64_t(x.q_tiles) * a.heads * a.batch;
  BL_REQUIRE(ctas < (int64_t(1) << 31), "bl_cross_attention: too many query tiles");
  auto kernel = flash_tc_kernel<kTiles, kBlocks, kBias>;
  BL_CUDA(ensure_smem_limit(reinterpret_cast<const void *>(kernel), S::kBytes));
  kernel<<<unsigned(ctas), S::kThreads, S::kBytes, stream>>>(maps[0], maps[1], maps[2], maps[3], x);
  BL_LAUNCH_CHECK();
  return BL_OK;
}

}  // namespace

// Runs the tensor-core kernel and sets *taken where it covers the call.
int forward_tc(const Args &a, cudaStream_t stream, bool *taken) {
  *taken = false;
  if (a.nq < 65 || a.nk < 64 || !(a.scale > 0.f) || (a.bias && !a.bias_vec)) return BL_OK;
  CUtensorMap maps[4];
  const int kv_heads = a.heads / a.group;
  if (!rows_map(&maps[0], a.q, a.d, a.nq, a.heads, a.batch, kBQ) ||
      !rows_map(&maps[1], a.k, a.d, a.nk, kv_heads, a.batch, kBK) ||
      !rows_map(&maps[2], a.v, a.d, a.nk, kv_heads, a.batch, kBK))
    return BL_OK;
  maps[3] = maps[0];
  if (a.bias) {
    const Rows r{a.bias, a.bias_sb, a.bias_si, a.bias_sh};
    if (!rows_map(&maps[3], r, a.nk, a.nq, a.heads, a.batch / a.share, kBQ)) return BL_OK;
  }
  *taken = true;
  const bool wide = a.d > 64;
  // Two query tiles per CTA once they still give every SM a CTA.
  const bool two = int64_t((a.nq + 2 * kBQ - 1) / (2 * kBQ)) * a.heads * a.batch >= num_sms();
  if (a.bias) {
    if (two) return wide ? launch_tc<2, 2, true>(a, maps, stream) : launch_tc<2, 1, true>(a, maps, stream);
    return wide ? launch_tc<1, 2, true>(a, maps, stream) : launch_tc<1, 1, true>(a, maps, stream);
  }
  if (two) return wide ? launch_tc<2, 2, false>(a, maps, stream) : launch_tc<2, 1, false>(a, maps, stream);
  return wide ? launch_tc<1, 2, false>(a, maps, stream) : launch_tc<1, 1, false>(a, maps, stream);
}

}  // namespace xa
}  // namespace bl
