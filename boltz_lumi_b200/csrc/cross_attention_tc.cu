// Cross attention forward on tcgen05 tensor cores (bf16; see cross_attention.cuh).
//
// One CTA = kTiles tiles of 128 query rows of one (sample, head) over key tiles
// of 64.  Warp 0 feeds the tiles by TMA, warps 1 and 2 issue the MMAs of one query tile
// each (a single issuer would wait for one tile's P before the other's next S), and
// four softmax warps per query tile own one row per thread (TMEM lane = row):
//   * S = Q K^T into TMEM (128 x 64, fp32); the thread reads its 64 scores into
//     registers, which frees S at once: the next tile's product runs under this
//     tile's softmax (with P written over S it had to wait for P.V);
//   * the thread adds the bias row from shared memory (128-byte swizzle: conflict-free
//     16-byte reads), takes p = exp2 and writes P as bf16 to one of two TMEM buffers;
//   * O += P V with P from TMEM and V in its natural [key][d] order (MN-major);
//     O is rescaled only when a row's maximum grew by more than 2^8 (a published refinement of the
//     online softmax: any reference near the maximum serves, as P and the row sum share it).
// P is rounded to bf16 for its product; the row sum adds the fp32 values.
// 2 x 16 x 2048 x 8190 x 48 with one bias: 385 us (floor 92 us: 606 MB, nearly all the bias); 4 x 16(4) x
// 777 x 2048 x 128 without: 112 us, 465 TFLOP/s.  What bounds it: the softmax warps' chain per tile, two
// warps per scheduler deep (1430 cycles per 128 x 64 scores, of which the exponentials, 16 per clock and
// SM, are 512 and issue some 500), and whole waves (256 CTAs over 148 SMs: two).  Two query tiles per
// CTA halve the K / V bytes that each score costs; with few tiles one per CTA
// spreads them over more SMs, and a cluster of CTAs divides the keys of one tile
// and joins its parts through distributed shared memory (one launch, fixed order).
#include <array>

#include "cross_attention_tc.cuh"

namespace bl {
namespace xa {
namespace {

constexpr int kBQ = 128, kBK = 64;
constexpr float kRescale = 8.f;  // log2 of the growth of a maximum that rescales O

template <int kTiles, int kBlocks, bool kBias> struct Shape {  // kBlocks: 64-column blocks of d
  static constexpr int kSoftWarps = 4 * kTiles, kThreads = (4 + kSoftWarps) * 32;
  // Registers per thread after the split: launched with 168 (384 threads) or 128 (256 threads,
  // two CTAs per SM), the first four warps give up what the softmax warps take.
  static constexpr int kFew = 40, kMany = kTiles == 2 ? 232 : 216;
  static_assert(128 * kFew + 128 * kTiles * kMany <= (kTiles == 2 ? 384 * 168 : 256 * 128), "register split");
  static constexpr int kKvStages = kBias ? (kBlocks == 2 && kTiles == 2 ? 2 : 3) : (kBlocks == 2 ? 3 : 4);
  static constexpr int kBiasStages = kBlocks == 2 ? 2 : (kTiles == 2 ? 3 : 2);
  static constexpr int kQ = kBQ * 128 * kBlocks;         // bytes of one query tile
  static constexpr int kK = kBK * 128 * kBlocks;         // bytes of a K or V tile
  static constexpr int kB = kBias ? kBQ * kBK * 2 : 0;   // bytes of a bias tile
  static constexpr int kKvOff = kTiles * kQ;
  static constexpr int kBiasOff = kKvOff + kKvStages * 2 * kK;
  static constexpr int kMaskOff = kBiasOff + kTiles * kBiasStages * kB;  // [softmax warp][64] fp32
  static constexpr int kBitsOff = kMaskOff + kSoftWarps * kBK * 4;  // [kMaskWords] bits of keys to look at
  static constexpr int kBarOff = kBitsOff + kMaskWords * 4;
  static constexpr int kBytes = kBarOff + 384 + 1024;
  static constexpr uint32_t kTmem = kTiles == 2 ? 512 : 256;
  // TMEM columns of tile t, from 256 t on: S (64), P of even and odd key tiles (32 each), O (128).
  static constexpr uint32_t kPCol = 64, kOCol = 128;
};

struct TcArgs {
  Args a;
  int q_tiles;  // CTAs (clusters) per (sample, head)
  int split;    // CTAs of a cluster that divide the keys
  unsigned int *status;
};

// Joins the parts of a cluster's CTAs (in the order of their keys): a thread has one row and every
// split-th group of four columns.
__device__ __forceinline__ void merge_rows(const Args &a, const void *part, const void *stat, int split, int rank, int row,
                                           int q0, int h, int b) {
  const int i = q0 + row;
  if (i >= a.nq) return;
  const float *st = static_cast<const float *>(stat);
  float weight[8], top = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    weight[e] = e < split ? peer(st + row, uint32_t(e)) : -INFINITY;
    top = fmaxf(top, weight[e]);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    weight[e] = weight[e] == -INFINITY ? 0.f : fast_exp2((weight[e] - top) * kLog2e);
    if (e < split) l = fmaf(weight[e], peer(st + kBQ + row, uint32_t(e)), l);
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  using T = __nv_bfloat16;
  const int64_t at = ((int64_t(b) * a.nq + i) * a.heads + h) * a.d;
  const T *gate = a.gate.p ? static_cast<const T *>(a.gate.p) + b * a.gate.sb + int64_t(i) * a.gate.si + h * a.gate.sh : nullptr;
  for (int c = rank; 4 * c < a.d; c += split) {
    float o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < split) {
        const float4 v = peer4(static_cast<const float4 *>(part) + c * kBQ + row, uint32_t(e));
        o[0] = fmaf(weight[e], v.x, o[0]), o[1] = fmaf(weight[e], v.y, o[1]);
        o[2] = fmaf(weight[e], v.z, o[2]), o[3] = fmaf(weight[e], v.w, o[3]);
      }
    uint2 g = make_uint2(0u, 0u);
    if (gate) g = *reinterpret_cast<const uint2 *>(gate + 4 * c);
    const float gv[4] = {bf16_lo(g.x), bf16_hi(g.x), bf16_lo(g.y), bf16_hi(g.y)};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      o[e] *= inv;
      if (gate) o[e] *= 1.f / (1.f + expf(-gv[e]));
    }
    const uint2 hi = make_uint2(pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]));
    *reinterpret_cast<uint2 *>(static_cast<T *>(a.out) + at + 4 * c) = hi;
    if (a.low)
      *reinterpret_cast<uint2 *>(static_cast<T *>(a.low) + at + 4 * c) =
          make_uint2(pack_bf16x2(o[0] - bf16_lo(hi.x), o[1] - bf16_hi(hi.x)), pack_bf16x2(o[2] - bf16_lo(hi.y), o[3] - bf16_hi(hi.y)));
  }
  if (a.lse && rank == 0) {
    float *to = a.lse + (int64_t(b) * a.heads + h) * a.nq + i;
    to[0] = l == 0.f ? -INFINITY : top;
    to[a.lse_plane()] = l == 0.f ? 0.f : logf(l);
  }
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
  uint64_t *s_full = b_empty + kTiles * BS;    // [tile] S in TMEM
  uint64_t *s_free = s_full + kTiles;          // [tile] S is in the softmax warps' registers
  uint64_t *p_full = s_free + kTiles;          // [tile][2] P in TMEM (and O rescaled if needed)
  uint64_t *pv_done = p_full + kTiles * 2;     // [tile][2] P.V of that buffer is done
  uint64_t *o_full = pv_done + kTiles * 2;     // [tile] every P.V is done
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(o_full + kTiles);
  int *last_key = reinterpret_cast<int *>(tmem_slot + 1);

  const Args &a = x.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int tile, h, b;
  const int split = kTiles == 1 ? x.split : 1, rank = split > 1 ? int(blockIdx.x) % split : 0;
  decode_cta(a, blockIdx.x / split, x.q_tiles, a.heads, tile, h, b);
  const int q0 = tile * kTiles * kBQ, hk = h / a.group, bb = b / a.share;
  const int live = a.nq - q0 > kBQ ? kTiles : 1;  // query tiles with rows

  if (tid == 0) {
    tc::mbar_init(q_full, 1);
    for (int i = 0; i < KV; ++i) tc::mbar_init(kv_full + i, 1), tc::mbar_init(kv_empty + i, live);
    for (int i = 0; i < kTiles * BS; ++i) tc::mbar_init(b_full + i, 1), tc::mbar_init(b_empty + i, 4);
    for (int i = 0; i < kTiles * 2; ++i) tc::mbar_init(p_full + i, 4), tc::mbar_init(pv_done + i, 1);
    for (int i = 0; i < kTiles; ++i)
      tc::mbar_init(s_full + i, 1), tc::mbar_init(s_free + i, 4), tc::mbar_init(o_full + i, 1);
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
  // One bit per key: left out (or, with an additive mask, changed by it).  Reading the mask
  // tile by tile cost 400 of 2500 cycles per tile.  Key tiles past the last kept key (a
  // padded batch) are not visited.
  uint32_t *bits = reinterpret_cast<uint32_t *>(smem + S::kBitsOff);
  const bool use_bits = a.nk <= 32 * kMaskWords;
  int keys = a.nk;
  if (a.mask_kind != kMaskNone && use_bits) {
    int best = -1;
    for (int w = tid; w < (n_words(a.nk) + 1) / 2 * 2; w += S::kThreads) {
      const uint32_t word = mask_word(a, b, w);
      bits[w] = word;
      if (word != 0xffffffffu) best = 32 * w + 31 - __clz(~word);
    }
    if (a.mask_kind == kMaskKeep) {
      if (best >= 0) atomicMax(last_key, best);
      __syncthreads();
      keys = *last_key + 1;
    } else {
      __syncthreads();
    }
  }
  // Key tiles [lo, lo + n_tiles).
  const int all_tiles = (keys + kBK - 1) / kBK, lo = int(int64_t(rank) * all_tiles / split);
  const int n_tiles = int(int64_t(rank + 1) * all_tiles / split) - lo;

  if (warp < 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::kFew));
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
        if (j >= KV && !(ok = wait_phase(kv_empty + s, ((j / KV) & 1) ^ 1u, x.status, 0x301))) break;
        uint8_t *st = smem + S::kKvOff + s * 2 * S::kK;
        tc::mbar_arrive_expect_tx(kv_full + s, 2 * S::kK);
        for (int c = 0; c < kBlocks; ++c) tma_load_4d(st + c * kBK * 128, &map_k, kv_full + s, 64 * c, (lo + j) * kBK, hk, b);
        for (int c = 0; c < kBlocks; ++c)
          tma_load_4d(st + S::kK + c * kBK * 128, &map_v, kv_full + s, 64 * c, (lo + j) * kBK, hk, b);
        if constexpr (kBias) {
          const int bs = j % BS;
          for (int t = 0; t < live; ++t) {
            uint64_t *full = b_full + t * BS + bs;
            if (j >= BS && !(ok = wait_phase(b_empty + t * BS + bs, ((j / BS) & 1) ^ 1u, x.status, 0x302))) break;
            tc::mbar_arrive_expect_tx(full, S::kB);
            tma_load_4d(smem + S::kBiasOff + (t * BS + bs) * S::kB, &map_bias, full, (lo + j) * kBK, q0 + t * kBQ, h, bb);
          }
        }
      }
    }
  } else if (warp < 1 + kTiles) {
    // ---------------- MMA issuer of one query tile ----------------
    const int t = warp - 1;
    if (lane == 0 && t < live && n_tiles > 0 && wait_phase(q_full, 0, x.status, 0x303)) {
      constexpr uint32_t idesc_s = tc::idesc_bf16(kBQ, kBK, false, false);
      const int steps = (a.d + 15) / 16;  // columns past d are zero
      const uint32_t idesc_pv = tc::idesc_bf16(kBQ, 16 * steps, false, true);
      const uint32_t rows = low_k(smem_addr(smem)), cols = low_mn(smem_addr(smem), kBK * 128), q = rows + (t * S::kQ >> 4);
      auto issue_s = [&](int j) {
        const int s = j % KV;
        if (!wait_phase(kv_full + s, (j / KV) & 1, x.status, 0x304)) return false;
        if (j > 0 && !wait_phase(s_free + t, (j - 1) & 1, x.status, 0x305)) return false;
        tc::tc_fence_after();
        mma_rows_ss<kBlocks>(tmem + t * 256, q, kBQ * 128, rows + ((S::kKvOff + s * 2 * S::kK) >> 4), kBK * 128, idesc_s, false);
        tc::umma_commit(s_full + t);
        return true;
      };
      bool ok = issue_s(0);
      for (int j = 0; j < n_tiles && ok; ++j) {
        const int s = j % KV, buf = j & 1;
        if (j + 1 < n_tiles && !(ok = issue_s(j + 1))) break;
        if (!(ok = wait_phase(p_full + t * 2 + buf, (j >> 1) & 1, x.status, 0x306))) break;
        tc::tc_fence_after();
        mma_cols_ts<kBK / 16>(tmem + t * 256 + S::kOCol, tmem + t * 256 + S::kPCol + buf * 32,
                              cols + ((S::kKvOff + s * 2 * S::kK + S::kK) >> 4), idesc_pv, j != 0);
        tc::umma_commit(pv_done + t * 2 + buf);
        tc::umma_commit(kv_empty + s);
        if (j + 1 == n_tiles) tc::umma_commit(o_full + t);
      }
    }
  } else if (warp >= 4) {
    // ---------------- softmax and epilogue: one query row per thread ----------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(S::kMany));
    const int t = (warp - 4) >> 2, quarter = warp & 3;
    const int row = quarter * 32 + lane, i = q0 + t * kBQ + row;
    const uint32_t lanes = tmem + (uint32_t(quarter * 32) << 16) + t * 256;
    const uint32_t o_col = lanes + S::kOCol;
    float *mk = reinterpret_cast<float *>(smem + S::kMaskOff) + (warp - 4) * kBK;  // this warp's additive mask values
    const int d16 = (a.d + 15) / 16;
    float m = -INFINITY;  // reference of the exponentials
    uint64_t sum2 = 0;    // two partial row sums
    bool ok = t < live;
    // The scores of a tile are fetched from TMEM while the tile before it is being
    // exponentiated: the load's latency would otherwise be paid per tile.
    uint32_t sv[2][32];
    auto fetch = [&](int j) {
      if (!(ok = warp_wait(s_full + t, j & 1, x.status, 0x307))) return;
      tc::tc_fence_after();
      tc::tmem_ld_32x32b_x32(lanes, sv[0]);
      tc::tmem_ld_32x32b_x32(lanes + 32, sv[1]);
    };
    if (ok && n_tiles > 0) fetch(0);
    for (int j = 0; j < n_tiles && ok; ++j) {
      const int buf = j & 1, bs = j % BS, k0 = (lo + j) * kBK;
      // Keys of this tile that the mask touches, and keys past nk.
      uint32_t cut[2] = {0u, 0u};
      if (a.mask_kind == kMaskNone) {
        const int left = a.nk - k0;
        if (left < kBK) cut[0] = left < 32 ? ~0u << left : 0u, cut[1] = left <= 32 ? ~0u : ~0u << (left - 32);
      } else if (use_bits) {
        const uint2 w = *reinterpret_cast<const uint2 *>(bits + 2 * (lo + j));
        cut[0] = w.x, cut[1] = w.y;
      } else {
#pragma unroll
        for (int e = 0; e < 2; ++e)
          cut[e] = __ballot_sync(0xffffffffu, mask_value(a, b, k0 + 32 * e + lane) != 0.f);
      }
      const bool masked = (cut[0] | cut[1]) != 0;
      if (masked && a.mask_kind == kMaskAdd) {
        __syncwarp();
#pragma unroll
        for (int e = 0; e < 2; ++e) mk[lane + 32 * e] = mask_value(a, b, k0 + 32 * e + lane);
        __syncwarp();
      }
      if constexpr (kBias) {
        if (!(ok = warp_wait(b_full + t * BS + bs, (j / BS) & 1, x.status, 0x308))) break;
      }
      tc::tmem_ld_wait_regs(sv[0], sv[1]);
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(s_free + t);
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
      } else {
#pragma unroll
        for (int p = 0; p < 32; ++p)
          y[p] = mul2(pack2(sv[p >> 4][(2 * p) & 31], sv[p >> 4][(2 * p + 1) & 31]), scale2);
      }
      if (masked) {
        if (a.mask_kind == kMaskAdd) {
#pragma unroll
          for (int p = 0; p < 32; ++p) {
            const float2 mp = *reinterpret_cast<const float2 *>(mk + 2 * p);
            const float lo = mp.x == -INFINITY ? mp.x : lo_f(y[p]) + mp.x, hi = mp.y == -INFINITY ? mp.y : hi_f(y[p]) + mp.y;
            y[p] = pack2(__float_as_uint(lo), __float_as_uint(hi));
          }
        } else {
#pragma unroll
          for (int p = 0; p < 32; ++p) {
            const uint32_t c = cut[p >> 4] >> (2 * p & 31);
            y[p] = pack2(c & 1 ? 0xff800000u : uint32_t(y[p]), c & 2 ? 0xff800000u : uint32_t(y[p] >> 32));
          }
        }
        // V rows of left-out keys must be zero: a zero weight times what they hold may not be.
        if (a.mask_kind == kMaskKeep) {
          const int s = j % KV, key = row >> 1;
          if ((key < 32 ? cut[0] >> key : cut[1] >> (key - 32)) & 1) {
            wait_phase(kv_full + s, (j / KV) & 1, x.status, 0x30B);  // complete: S came from this stage
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
      float mx[8];
#pragma unroll
      for (int p = 0; p < 8; ++p) mx[p] = fmaxf(lo_f(y[p]), hi_f(y[p]));
#pragma unroll
      for (int p = 8; p < 32; ++p) mx[p & 7] = fmaxf(mx[p & 7], fmaxf(lo_f(y[p]), hi_f(y[p])));
      const float top = fmaxf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), fmaxf(fmaxf(mx[4], mx[5]), fmaxf(mx[6], mx[7])));
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
      // P of tile j - 2 was in this buffer.  Its P.V has read it: it was issued before S of
      // this tile, whose commit (s_full) covers every earlier product of that thread.
      const uint32_t p_col = lanes + S::kPCol + buf * 32;
      const bool far = __any_sync(0xffffffffu, far_row(m));  // every score has been looked at: the bias is in registers
      if constexpr (kBias) {
        tc::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(b_empty + t * BS + bs);
      }
      if (far) {
        const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t p16[16];
#pragma unroll
          for (int p = 0; p < 16; ++p) {
            const uint64_t z = y[16 * half + p];
            const float e0 = fast_exp2((lo_f(z) - base) * kLog2e), e1 = fast_exp2((hi_f(z) - base) * kLog2e);
            sum2 = add2(sum2, pack2(__float_as_uint(e0), __float_as_uint(e1)));
            p16[p] = pack_bf16x2(e0, e1);
          }
          tc::tmem_st_32x32b_x16(p_col + 16 * half, p16);
        }
        if (j + 1 < n_tiles) fetch(j + 1);
      } else {
        const uint64_t log2e2 = dup2(kLog2e), base2 = dup2(m == -INFINITY ? 0.f : -m * kLog2e);
        uint64_t other = 0;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t p16[16];
#pragma unroll
          for (int p = 0; p < 16; ++p) {
            const uint64_t z = fma2(y[16 * half + p], log2e2, base2);
            const float e0 = fast_exp2(lo_f(z)), e1 = fast_exp2(hi_f(z));
            uint64_t &to = p & 1 ? other : sum2;
            to = add2(to, pack2(__float_as_uint(e0), __float_as_uint(e1)));
            p16[p] = pack_bf16x2(e0, e1);
          }
          tc::tmem_st_32x32b_x16(p_col + 16 * half, p16);
          if (half == 0 && j + 1 < n_tiles) fetch(j + 1);
        }
        sum2 = add2(sum2, other);
      }
      tc::tmem_st_wait();
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(p_full + t * 2 + buf);
    }
    // Epilogue: o / l, the gate, one rounding.
    if (t < live) {
      tc::tmem_ld_wait();
      if (ok && n_tiles > 0) ok = warp_wait(o_full + t, 0, x.status, 0x30A);
      tc::tc_fence_after();
      const float l = lo_f(sum2) + hi_f(sum2), inv = l == 0.f ? 0.f : 1.f / l;
      using T = __nv_bfloat16;
      const int64_t at = ((int64_t(b) * a.nq + i) * a.heads + h) * a.d;
      const T *gate = a.gate.p ? static_cast<const T *>(a.gate.p) + b * a.gate.sb + int64_t(i) * a.gate.si + h * a.gate.sh
                               : nullptr;
      T *out = static_cast<T *>(a.out) + at, *low = a.low ? static_cast<T *>(a.low) + at : nullptr;
      if (ok && kTiles == 1 && split > 1) {
        // This CTA's part of the row, for the cluster: O where K and V were, [4 columns][row].
        float4 *part = reinterpret_cast<float4 *>(smem + S::kKvOff);
        float *stat = reinterpret_cast<float *>(smem + S::kMaskOff);
        for (int c = 0; c < d16; ++c) {
          uint32_t o[16];
          if (n_tiles > 0) {
            tc::tmem_ld_32x32b_x16(o_col + 16 * c, o);
            tc::tmem_ld_wait();
          }
#pragma unroll
          for (int e = 0; e < 4; ++e)
            part[(4 * c + e) * kBQ + row] =
                n_tiles > 0 ? make_float4(__uint_as_float(o[4 * e]), __uint_as_float(o[4 * e + 1]),
                                          __uint_as_float(o[4 * e + 2]), __uint_as_float(o[4 * e + 3]))
                            : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        stat[row] = l == 0.f ? -INFINITY : m, stat[kBQ + row] = l;
      } else if (ok) {
        for (int c = 0; c < d16; ++c) {
          uint32_t o[16];
          if (n_tiles > 0) {
            tc::tmem_ld_32x32b_x16(o_col + 16 * c, o);
            tc::tmem_ld_wait();
          }
#pragma unroll
          for (int e8 = 0; e8 < 2; ++e8) {
            const int c0 = 16 * c + 8 * e8;
            if (i >= a.nq || c0 >= a.d) continue;  // d is a multiple of 8
            uint4 gv = make_uint4(0u, 0u, 0u, 0u);
            if (gate) gv = *reinterpret_cast<const uint4 *>(gate + c0);
            const uint32_t gw[4] = {gv.x, gv.y, gv.z, gv.w};
            uint32_t ov[4], lv[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float u = n_tiles > 0 ? __uint_as_float(o[8 * e8 + 2 * e]) * inv : 0.f;
              float w = n_tiles > 0 ? __uint_as_float(o[8 * e8 + 2 * e + 1]) * inv : 0.f;
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
        if (a.lse && i < a.nq) {  // (a cluster's rows: merge_rows)
          float *st = a.lse + (int64_t(b) * a.heads + h) * a.nq + i;
          st[0] = l == 0.f ? -INFINITY : m;
          st[a.lse_plane()] = l == 0.f ? 0.f : logf(l);
        }
      }
    }
  }
  if (kTiles == 1 && split > 1) {
    __syncwarp();
    cluster_barrier();
    if (warp >= 4) merge_rows(a, smem + S::kKvOff, smem + S::kMaskOff, split, rank, tid - 128, q0, h, b);
    __syncwarp();
    cluster_barrier();  // until every part has been read
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, S::kTmem);
  }
}

// Clusters of s CTAs that the device holds at once (asked of the first device in use: only the choice of a split hangs on it).
template <int kTiles, int kBlocks, bool kBias> int active_clusters(int s) {
  using S = Shape<kTiles, kBlocks, kBias>;
  static const std::array<int, 9> table = [] {
    std::array<int, 9> t{};
    for (int e = 1; e <= 8; ++e) {
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = unsigned(e), attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
      cudaLaunchConfig_t config = {};
      config.gridDim = dim3(unsigned(e)), config.blockDim = dim3(S::kThreads), config.dynamicSmemBytes = S::kBytes;
      config.attrs = attr, config.numAttrs = 1;
      int n = 0;
      if (cudaOccupancyMaxActiveClusters(&n, flash_tc_kernel<kTiles, kBlocks, kBias>, &config) != cudaSuccess || n < 1) {
        cudaGetLastError();
        n = num_sms() / e;
      }
      t[e] = n < 1 ? 1 : n;
    }
    return t;
  }();
  return table[s];
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
  x.split = 1;
  if (kTiles == 1) {
    // Few CTAs: a cluster divides the keys, by the waves that it takes (128 queries, 8 heads: 33 -> 12 us at
    // 1024 keys, 164 -> 29 us at 8192; 2 x 16 x 384 x 1734 without a mask: 46 -> 39 us).
    const int64_t work = (a.nk + kBK - 1) / kBK;
    double best = 0.;
    for (int e = 1; e <= 8 && (e == 1 || e <= work); ++e) {
      const int64_t held = active_clusters<kTiles, kBlocks, kBias>(e), waves = (ctas + held - 1) / held;
      const double cost = double(waves) / e + 0.02 * (e > 1);
      if (e == 1 || cost < best) best = cost, x.split = e;
    }
  }
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(unsigned(ctas * x.split)), config.blockDim = dim3(S::kThreads);
  config.dynamicSmemBytes = S::kBytes, config.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(x.split), attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
  config.attrs = attr, config.numAttrs = x.split > 1 ? 1 : 0;
  BL_CUDA(cudaLaunchKernelEx(&config, kernel, maps[0], maps[1], maps[2], maps[3], x));
  BL_LAUNCH_CHECK();
  return BL_OK;
}

}  // namespace

// Runs the tensor-core kernel and sets *taken where it covers the call.
int forward_tc(const Args &a, cudaStream_t stream, bool *taken) {
  *taken = false;
  if (a.nk < 64 || !(a.scale > 0.f) || (a.bias && !a.bias_vec)) return BL_OK;
  if (!worth_tiles(a)) return BL_OK;
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
  // Two query tiles per CTA once they still give every SM a CTA.  (Up to 128 queries the second tile has no rows: one tile
  // per CTA and two CTAs per SM would take 66 against 95 us at 1024 heads x 128 x 512 x 32, 140 against 122 us at d = 128.)
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
