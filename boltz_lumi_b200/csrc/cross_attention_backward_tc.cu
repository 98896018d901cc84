// Cross attention gradients on tcgen05 tensor cores (bf16; see cross_attention_backward.cu
// for the formulas).
//
//   queries_tc_kernel  one CTA = 128 query rows of one (sample, head) over key tiles of 64:
//                      S = Q K^T and dP = dO V^T in TMEM, dS = p (dP - delta) as bf16 in TMEM,
//                      dQ += dS K; dS itself is the bias gradient where no sample shares the bias.
//   keys_tc_kernel     one CTA = 128 keys of one (sample, key/value head) over query tiles of 64 of
//                      every head that reads them: S^T = K Q^T and dP^T = V dO^T, P^T and dS^T as
//                      bf16 in TMEM, dV += P^T dO, dK += dS^T Q (a gated dO in two bf16 terms).
//
//   bias_tc_kernel     the gradient of a bias that several samples share (see there).
//
// Both: warp 0 feeds the tiles by TMA; warps 1 to 3 issue the MMAs of the scores, of dP and of the
// gradients (an MMA of 64 columns costs its issuer 50 to 90 cycles, so one issuer was the limit: 179
// against 133 us for dQ at 4 x 16 x 777 x 2048 x 128); warps 4..7 and 8..11 take turns over the
// tiles, a thread per resident row (TMEM lane), in two halves of 32 scores.  S and dP have two
// buffers, so one set's products run under the other's arithmetic.  There is no row maximum to
// agree on: the forward's statistics give p directly.  A gated do enters dP and dV as two bf16 terms.
// P^T and dS^T (dS in the query kernel) are rounded to bf16 once, as the operands of their products; an unshared
// bias' gradient is that dS.  A shared one adds dS in fp32 and rounds the sum.
//
// Against the same loops on warp products: 4 x 16(4) x 777 x 2048 x 128 without bias, dk/dv 446 ->
// 138 us, dq 435 -> 133 us (five products, 620 TFLOP/s); 2 x 16 x 384 x 1734 x 48 with a shared bias and a
// gate, dk/dv 72 -> 48 us, dq 97 -> 35 us, dbias 87 -> 36 us.  What bounds them: at d = 128 the MMAs' operands (an
// SS product of 64 columns reads 6 KB of shared memory in 48 cycles) beside 2 x 900 cycles of
// exponentials and conversions per tile and set; at d = 48 that arithmetic and a CTA's start and end,
// some 8000 of 59000 cycles; CTAs come in whole waves (448 over 148 SMs: four).
#include "cross_attention_backward.cuh"
#include "cross_attention_tc.cuh"

namespace bl {
namespace xa {
namespace {

constexpr int kRowsTc = 128, kTileTc = 64, kThreadsTc = 12 * 32;
using Bf = __nv_bfloat16;

struct BackTc {
  BackArgs x;
  int tiles;  // resident row tiles per (sample, head)
  unsigned int *status;
};

template <int kBlocks, bool kBias, bool kLow> struct QShape {
  static constexpr int kRes = kRowsTc * 128 * kBlocks;  // bytes of a resident 128-row tile
  static constexpr int kStr = kTileTc * 128 * kBlocks;  // bytes of a streamed 64-row tile
  static constexpr int kB = kBias ? kRowsTc * kTileTc * 2 : 0;
  // A tile's load takes about as long as two tiles' arithmetic: K, which dQ still reads, needs the
  // longest ring, V is free after dP.
  static constexpr int kKStages = kBlocks == 1 ? 6 : kLow && kBias ? 3 : kLow || kBias ? 4 : 5;
  static constexpr int kVStages = kKStages - 1, kBiasStages = kBlocks == 1 ? 4 : 2;
  static constexpr int kResident = kLow ? 3 : 2;  // Q, dO, do - bf16(do)
  static constexpr int kKOff = kResident * kRes, kVOff = kKOff + kKStages * kStr;
  static constexpr int kBiasOff = kVOff + kVStages * kStr;
  static constexpr int kMaskOff = kBiasOff + (kBias ? kBiasStages * kB : 0);  // [warp][32] additive mask values
  static constexpr int kBitsOff = kMaskOff + 8 * 32 * 4;
  static constexpr int kBarOff = kBitsOff + kMaskWords * 4;
  static constexpr int kBytes = kBarOff + 512 + 1024;
};
// TMEM columns: two buffers of S and dP (64 each), two of dS (32 each), dQ.
constexpr uint32_t kSCol = 0, kDpCol = 64, kPair = 128, kDsCol = 256, kDqCol = 320;

template <int kBlocks, bool kBias, bool kLow>
__global__ void __launch_bounds__(kThreadsTc, 1)
    queries_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_do,
                      const __grid_constant__ CUtensorMap map_low, const __grid_constant__ CUtensorMap map_k,
                      const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_bias,
                      const BackTc p) {
  using S = QShape<kBlocks, kBias, kLow>;
  constexpr int KS = S::kKStages, VS = S::kVStages, BS = S::kBiasStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + S::kBarOff);
  uint64_t *res_full = bars;             // resident tiles landed
  uint64_t *k_full = res_full + 1;       // [KS] K of a key tile landed
  uint64_t *k_empty = k_full + KS;       // [KS] dQ has read it
  uint64_t *v_full = k_empty + KS;       // [VS] V landed
  uint64_t *v_empty = v_full + VS;       // [VS] dP has read it
  uint64_t *b_full = v_empty + VS;       // [BS] bias block landed
  uint64_t *b_empty = b_full + BS;       // [BS] it has been read
  uint64_t *s_full = b_empty + BS;       // [2] S and dP in TMEM
  uint64_t *ds_full = s_full + 2;        // [2] they have been read, dS is in TMEM
  uint64_t *dq_full = ds_full + 2;       // every product is done
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(dq_full + 1);
  int *last_key = reinterpret_cast<int *>(tmem_slot + 1);
  const Args &a = p.x.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int tile, h, b;
  decode_cta(a, blockIdx.x, p.tiles, a.heads, tile, h, b);
  const int q0 = tile * kRowsTc, hk = h / a.group, bb = b / a.share;
  if (tid == 0) {
    tc::mbar_init(res_full, 1);
    for (int i = 0; i < KS; ++i) tc::mbar_init(k_full + i, 1), tc::mbar_init(k_empty + i, 1);
    for (int i = 0; i < VS; ++i) tc::mbar_init(v_full + i, 1), tc::mbar_init(v_empty + i, 1);
    for (int i = 0; i < BS; ++i) tc::mbar_init(b_full + i, 1), tc::mbar_init(b_empty + i, 4);
    for (int i = 0; i < 2; ++i) tc::mbar_init(s_full + i, 2), tc::mbar_init(ds_full + i, 4);
    tc::mbar_init(dq_full, 1);
    tc::fence_mbar_init();
    *last_key = -1;
  }
  if (warp == 1) {
    tc::tmem_alloc(tmem_slot, 512);
    tc::tmem_relinquish();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  uint32_t *bits = reinterpret_cast<uint32_t *>(smem + S::kBitsOff);
  const bool use_bits = a.nk <= 32 * kMaskWords;
  int keys = a.nk;
  if (a.mask_kind != kMaskNone && use_bits) {
    int best = -1;
    for (int w = tid; w < (n_words(a.nk) + 1) / 2 * 2; w += kThreadsTc) {
      const uint32_t word = mask_word(a, b, w);
      bits[w] = word;
      if (word != 0xffffffffu) best = 32 * w + 31 - __clz(~word);
    }
    if (a.mask_kind == kMaskKeep && best >= 0) atomicMax(last_key, best);
    __syncthreads();
    // Key tiles past the last kept key add nothing to dq; where dbias is written here they are
    // visited all the same, to write their zeros.
    if (a.mask_kind == kMaskKeep && !(kBias && p.x.dbias && a.share == 1)) keys = *last_key + 1;
  }
  const int n = (keys + kTileTc - 1) / kTileTc;

  if (warp == 0) {
    if (lane == 0 && n > 0) {
      tc::mbar_arrive_expect_tx(res_full, S::kResident * S::kRes);
      for (int c = 0; c < kBlocks; ++c) {
        tma_load_4d(smem + c * kRowsTc * 128, &map_q, res_full, 64 * c, q0, h, b);
        tma_load_4d(smem + S::kRes + c * kRowsTc * 128, &map_do, res_full, 64 * c, q0, h, b);
        if (kLow) tma_load_4d(smem + 2 * S::kRes + c * kRowsTc * 128, &map_low, res_full, 64 * c, q0, h, b);
      }
      for (int j = 0; j < n; ++j) {
        const int ks = j % KS, vs = j % VS;
        if (j >= KS && !wait_phase(k_empty + ks, ((j / KS) & 1) ^ 1u, p.status, 0x401)) break;
        tc::mbar_arrive_expect_tx(k_full + ks, S::kStr);
        for (int c = 0; c < kBlocks; ++c)
          tma_load_4d(smem + S::kKOff + ks * S::kStr + c * kTileTc * 128, &map_k, k_full + ks, 64 * c, j * kTileTc, hk, b);
        if (j >= VS && !wait_phase(v_empty + vs, ((j / VS) & 1) ^ 1u, p.status, 0x40B)) break;
        tc::mbar_arrive_expect_tx(v_full + vs, S::kStr);
        for (int c = 0; c < kBlocks; ++c)
          tma_load_4d(smem + S::kVOff + vs * S::kStr + c * kTileTc * 128, &map_v, v_full + vs, 64 * c, j * kTileTc, hk, b);
        if constexpr (kBias) {
          const int bs = j % BS;
          if (j >= BS && !wait_phase(b_empty + bs, ((j / BS) & 1) ^ 1u, p.status, 0x402)) break;
          tc::mbar_arrive_expect_tx(b_full + bs, S::kB);
          tma_load_4d(smem + S::kBiasOff + bs * S::kB, &map_bias, b_full + bs, j * kTileTc, q0, h, bb);
        }
      }
    }
  } else if (warp < 3) {
    // ---------------- S (warp 1) and dP (warp 2), two tiles ahead of dQ ----------------
    if (lane == 0 && n > 0 && wait_phase(res_full, 0, p.status, 0x403)) {
      constexpr uint32_t idesc_s = tc::idesc_bf16(kRowsTc, kTileTc, false, false);
      const uint32_t base = low_k(smem_addr(smem));
      for (int j = 0; j < n; ++j) {
        const int set = j & 1, st = warp == 1 ? j % KS : j % VS;
        // This buffer's scores are in registers.
        if (j >= 2 && !wait_phase(ds_full + set, ((j - 2) >> 1) & 1, p.status, 0x404)) break;
        if (warp == 1) {
          if (!wait_phase(k_full + st, (j / KS) & 1, p.status, 0x405)) break;
          tc::tc_fence_after();
          mma_rows_ss<kBlocks>(tmem + set * kPair + kSCol, base, kRowsTc * 128, base + ((S::kKOff + st * S::kStr) >> 4),
                               kTileTc * 128, idesc_s, false);
          tc::umma_commit(s_full + set);
        } else {
          if (!wait_phase(v_full + st, (j / VS) & 1, p.status, 0x406)) break;
          tc::tc_fence_after();
          const uint32_t v = base + ((S::kVOff + st * S::kStr) >> 4);
          mma_rows_ss<kBlocks>(tmem + set * kPair + kDpCol, base + (S::kRes >> 4), kRowsTc * 128, v, kTileTc * 128, idesc_s, false);
          if (kLow)
            mma_rows_ss<kBlocks>(tmem + set * kPair + kDpCol, base + (2 * S::kRes >> 4), kRowsTc * 128, v, kTileTc * 128, idesc_s,
                                 true);
          tc::umma_commit(s_full + set);
          tc::umma_commit(v_empty + st);
        }
      }
    }
  } else if (warp == 3) {
    if (lane == 0) {
      const uint32_t idesc_dq = tc::idesc_bf16(kRowsTc, (a.d + 15) / 16 * 16, false, true);
      const uint32_t base = low_mn(smem_addr(smem), kTileTc * 128);
      for (int j = 0; j < n; ++j) {
        const int ks = j % KS;
        if (!wait_phase(ds_full + (j & 1), (j >> 1) & 1, p.status, 0x40C) || !wait_phase(k_full + ks, (j / KS) & 1, p.status, 0x40D))
          break;
        tc::tc_fence_after();
        mma_cols_ts<kTileTc / 16>(tmem + kDqCol, tmem + kDsCol + (j & 1) * 32, base + ((S::kKOff + ks * S::kStr) >> 4), idesc_dq,
                                  j != 0);
        tc::umma_commit(k_empty + ks);
        if (j + 1 == n) tc::umma_commit(dq_full);
      }
    }
  } else if (warp >= 4) {
    const int set = (warp - 4) >> 2, quarter = warp & 3, row = quarter * 32 + lane, i = q0 + row;
    const uint32_t lanes = tmem + (uint32_t(quarter * 32) << 16);
    float *mk = reinterpret_cast<float *>(smem + S::kMaskOff) + (warp - 4) * 32;
    float m = INFINITY, nl = 0.f, delta = 0.f;
    if (i < a.nq) {
      const int64_t at = (int64_t(b) * a.heads + h) * a.nq + i;
      m = row_max(a.lse[at]), nl = -kLog2e * a.lse[a.lse_plane() + at], delta = p.x.delta[at];
    }
    const bool far = __any_sync(0xffffffffu, far_row(m));
    const uint64_t c2 = dup2(m == INFINITY ? -INFINITY : fmaf(-m, kLog2e, nl)), delta2 = dup2(-delta), scale2 = dup2(a.scale);
    const uint64_t log2e2 = dup2(kLog2e);
    Bf *dbias = kBias && p.x.dbias && a.share == 1 && i < a.nq
                    ? static_cast<Bf *>(p.x.dbias) + ((int64_t(b) * a.heads + h) * a.nq + i) * p.x.dbias_ld
                    : nullptr;
    bool ok = true;
    for (int j = set; j < n && ok; j += 2) {
      const int bs = j % BS;
#pragma unroll 1
      for (int half = 0; half < 2 && ok; ++half) {
        const int k0 = j * kTileTc + 32 * half;
        uint32_t cut = 0;
        if (a.mask_kind == kMaskNone) {
          const int left = a.nk - k0;
          if (left < 32) cut = left <= 0 ? ~0u : ~0u << left;
        } else if (use_bits) {
          cut = bits[2 * j + half];
        } else {
          cut = __ballot_sync(0xffffffffu, mask_value(a, b, k0 + lane) != 0.f);
        }
        const bool adds = cut && a.mask_kind == kMaskAdd;
        if (adds) {
          const float v = mask_value(a, b, k0 + lane);
          __syncwarp();
          mk[lane] = v == -INFINITY ? 0.f : v;
          cut = __ballot_sync(0xffffffffu, v == -INFINITY);  // from here on: keys that count nothing
          __syncwarp();
        }
        if (half == 0) {
          if (!(ok = warp_wait(s_full + set, (j >> 1) & 1, p.status, 0x407))) break;
          tc::tc_fence_after();
          if constexpr (kBias) ok = warp_wait(b_full + bs, (j / BS) & 1, p.status, 0x408);
          if (!ok) break;
        }
        uint32_t sv[32], dv[32];
        tc::tmem_ld_32x32b_x32(lanes + set * kPair + kSCol + 32 * half, sv);
        tc::tmem_ld_32x32b_x32(lanes + set * kPair + kDpCol + 32 * half, dv);
        tc::tmem_ld_wait_regs(sv, dv);
        uint64_t y[16];
        if constexpr (kBias) {
          const uint32_t brow = smem_addr(smem + S::kBiasOff + bs * S::kB) + row * 128;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const uint4 v = lds128(brow + (((4 * half + c) ^ (row & 7)) << 4));
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
              y[4 * c + e] = fma2(pack2(sv[8 * c + 2 * e], sv[8 * c + 2 * e + 1]), scale2, pack2(w[e] << 16, w[e] & 0xffff0000u));
          }
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) y[e] = mul2(pack2(sv[2 * e], sv[2 * e + 1]), scale2);
        }
        if (adds)
#pragma unroll
          for (int e = 0; e < 16; ++e) y[e] = add2(y[e], *reinterpret_cast<const uint64_t *>(mk + 2 * e));
        uint32_t ds[16];
        if (far)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            y[e] = pack2(__float_as_uint(fmaf(lo_f(y[e]) - m, kLog2e, nl)), __float_as_uint(fmaf(hi_f(y[e]) - m, kLog2e, nl)));
        else
#pragma unroll
          for (int e = 0; e < 16; ++e) y[e] = fma2(y[e], log2e2, c2);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const uint64_t prob = pack2(__float_as_uint(fast_exp2(lo_f(y[e]))), __float_as_uint(fast_exp2(hi_f(y[e]))));
          const uint64_t g = mul2(prob, add2(pack2(dv[2 * e], dv[2 * e + 1]), delta2));
          ds[e] = pack_bf16x2(lo_f(g), hi_f(g));
        }
        if (cut) {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const uint32_t c = cut >> (2 * e);
            ds[e] &= (c & 1 ? 0u : 0xffffu) | (c & 2 ? 0u : 0xffff0000u);
          }
          // K rows of left-out keys must be zero before dS meets them in dQ.
          if (a.mask_kind == kMaskKeep) {
            const int ks = j % KS, key = 8 * quarter + (lane >> 2);
            if (cut >> key & 1) {
              wait_phase(k_full + ks, (j / KS) & 1, p.status, 0x409);  // complete: S came from this stage
              uint8_t *k = smem + S::kKOff + ks * S::kStr + (32 * half + key) * 128 + (lane & 3) * 32;
#pragma unroll
              for (int c = 0; c < kBlocks; ++c)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                  *reinterpret_cast<uint4 *>(k + c * kTileTc * 128 + e * 16) = make_uint4(0u, 0u, 0u, 0u);
            }
            tc::fence_proxy_async_smem();
          }
        }
        // dQ has read the dS of tile j - 2 in this buffer.
        if (half == 0 && j >= 2 && !(ok = warp_wait(k_empty + (j - 2) % KS, ((j - 2) / KS) & 1, p.status, 0x40E))) break;
        tc::tmem_st_32x32b_x16(lanes + kDsCol + set * 32 + 16 * half, ds);
        // The bias block is free once its values have gone into dS.  Released right after its loads, the next block
        // overtook them where the stores of dbias held them up.
        if (kBias && half == 1) {
          tc::fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(b_empty + bs);
        }
        if (kBias && dbias) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int k = k0 + 8 * c;
            if (k + 8 <= a.nk)
              *reinterpret_cast<uint4 *>(dbias + k) = make_uint4(ds[4 * c], ds[4 * c + 1], ds[4 * c + 2], ds[4 * c + 3]);
            else
#pragma unroll
              for (int e = 0; e < 8; ++e)
                if (k + e < a.nk) reinterpret_cast<uint16_t *>(dbias)[k + e] = uint16_t(ds[4 * c + (e >> 1)] >> (16 * (e & 1)));
          }
        }
      }
      if (!ok) break;
      tc::tmem_st_wait();
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(ds_full + set);
    }
    if (ok && n > 0) ok = warp_wait(dq_full, 0, p.status, 0x40A);
    tc::tc_fence_after();
    if (ok) {
      Bf *dq = static_cast<Bf *>(p.x.dq) + ((int64_t(b) * a.nq + i) * a.heads + h) * a.d;
      for (int c = set; c < (a.d + 15) / 16; c += 2) {
        uint32_t o[16];
        if (n > 0) {
          tc::tmem_ld_32x32b_x16(lanes + kDqCol + 16 * c, o);
          tc::tmem_ld_wait();
        }
#pragma unroll
        for (int e8 = 0; e8 < 2; ++e8) {
          const int c0 = 16 * c + 8 * e8;
          if (i >= a.nq || c0 >= a.d) continue;
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            w[e] = n > 0 ? pack_bf16x2(__uint_as_float(o[8 * e8 + 2 * e]) * a.scale, __uint_as_float(o[8 * e8 + 2 * e + 1]) * a.scale)
                         : 0u;
          *reinterpret_cast<uint4 *>(dq + c0) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, 512);
  }
}

template <int kBlocks, bool kBias, bool kLow> struct KShape {
  static constexpr int kRes = kRowsTc * 128 * kBlocks, kStr = kTileTc * 128 * kBlocks;
  static constexpr int kPer = kLow ? 3 : 2;  // streamed tiles: Q, dO, do - bf16(do)
  static constexpr int kB = kBias ? kTileTc * kRowsTc * 2 : 0;
  static constexpr int kStages = kBlocks == 1 ? (kBias ? 4 : 5) : kLow && kBias ? 2 : kLow || kBias ? 3 : 4;
  static constexpr int kStrOff = 2 * kRes;  // K, V
  static constexpr int kBiasOff = kStrOff + kStages * kPer * kStr;
  static constexpr int kStatOff = kBiasOff + kStages * kB;  // [stage]{reference, -log2 sum, base-2 offset, -delta}[64]
  static constexpr int kBarOff = kStatOff + kStages * 4 * kTileTc * 4 + kStages * 16;
  static constexpr int kBytes = kBarOff + 256 + 1024;
};
// TMEM columns: two buffers of S^T and dP^T (64 each), of P^T and dS^T (32 each), dV, dK.  With wide
// rows P^T and dS^T take the first columns of S^T and dP^T instead.
template <int kBlocks> struct KCols {
  static constexpr uint32_t pt = kBlocks == 1 ? 256 : kSCol, pt_step = kBlocks == 1 ? 32 : kPair;
  static constexpr uint32_t ds = kBlocks == 1 ? 320 : kDpCol, dv = kBlocks == 1 ? 384 : 256, dk = dv + 64 * kBlocks;
};

template <int kBlocks, bool kBias, bool kLow>
__global__ void __launch_bounds__(kThreadsTc, 1)
    keys_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_do,
                   const __grid_constant__ CUtensorMap map_low, const __grid_constant__ CUtensorMap map_k,
                   const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_bias, const BackTc p) {
  using S = KShape<kBlocks, kBias, kLow>;
  using C = KCols<kBlocks>;
  constexpr int ST = S::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + S::kBarOff);
  uint64_t *res_full = bars;             // K and V landed
  uint64_t *st_full = res_full + 1;      // [ST] Q, dO and the bias block of a query tile landed
  uint64_t *st_empty = st_full + ST;     // [ST] dV and dK have read them
  uint64_t *stat_full = st_empty + ST;   // [ST] the rows' statistics are in shared memory
  uint64_t *stat_empty = stat_full + ST; // [ST] they (and the bias block) have been read
  uint64_t *s_full = stat_empty + ST;    // [2] S^T and dP^T in TMEM
  uint64_t *ps_full = s_full + 2;        // [2] P^T and dS^T in TMEM
  uint64_t *pv_done = ps_full + 2;       // [2] dV has read P^T
  uint64_t *d_full = pv_done + 2;        // every product is done
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(d_full + 1);
  float *stats = reinterpret_cast<float *>(smem + S::kStatOff);
  int *far_flag = reinterpret_cast<int *>(stats + ST * 4 * kTileTc);  // [ST], 16 bytes apart
  const Args &a = p.x.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, kv_heads = a.heads / a.group;
  int tile, hk, b;
  decode_cta(a, blockIdx.x, p.tiles, kv_heads, tile, hk, b);
  const int j0 = tile * kRowsTc, bb = b / a.share;
  if (tid == 0) {
    tc::mbar_init(res_full, 1);
    for (int i = 0; i < ST; ++i) {
      tc::mbar_init(st_full + i, 1), tc::mbar_init(st_empty + i, 1);
      tc::mbar_init(stat_full + i, 1), tc::mbar_init(stat_empty + i, 4);
    }
    for (int i = 0; i < 2; ++i) tc::mbar_init(s_full + i, 2), tc::mbar_init(ps_full + i, 4), tc::mbar_init(pv_done + i, 1);
    tc::mbar_init(d_full, 1);
    tc::fence_mbar_init();
  }
  if (warp == 1) {
    tc::tmem_alloc(tmem_slot, 512);
    tc::tmem_relinquish();
  }
  const bool keeps = tid < kRowsTc && mask_value(a, b, j0 + tid) != -INFINITY;
  tc::tc_fence_before();
  const bool any = __syncthreads_or(keeps);
  tc::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int q_tiles = (a.nq + kTileTc - 1) / kTileTc, n = any ? q_tiles * a.group : 0;

  if (warp == 0) {
    if (lane == 0 && n > 0) {
      tc::mbar_arrive_expect_tx(res_full, 2 * S::kRes);
      for (int c = 0; c < kBlocks; ++c) {
        tma_load_4d(smem + c * kRowsTc * 128, &map_k, res_full, 64 * c, j0, hk, b);
        tma_load_4d(smem + S::kRes + c * kRowsTc * 128, &map_v, res_full, 64 * c, j0, hk, b);
      }
      for (int u = 0; u < n; ++u) {
        const int s = u % ST, h = hk * a.group + u / q_tiles, i0 = u % q_tiles * kTileTc;
        if (u >= ST && !wait_phase(st_empty + s, ((u / ST) & 1) ^ 1u, p.status, 0x411)) break;
        if (kBias && u >= ST && !wait_phase(stat_empty + s, ((u / ST) & 1) ^ 1u, p.status, 0x412)) break;
        uint8_t *st = smem + S::kStrOff + s * S::kPer * S::kStr;
        tc::mbar_arrive_expect_tx(st_full + s, S::kPer * S::kStr + S::kB);
        for (int c = 0; c < kBlocks; ++c) {
          tma_load_4d(st + c * kTileTc * 128, &map_q, st_full + s, 64 * c, i0, h, b);
          tma_load_4d(st + S::kStr + c * kTileTc * 128, &map_do, st_full + s, 64 * c, i0, h, b);
          if (kLow) tma_load_4d(st + 2 * S::kStr + c * kTileTc * 128, &map_low, st_full + s, 64 * c, i0, h, b);
        }
        if constexpr (kBias)  // two blocks of 64 keys
          for (int c = 0; c < 2; ++c)
            tma_load_4d(smem + S::kBiasOff + s * S::kB + c * kTileTc * 128, &map_bias, st_full + s, j0 + 64 * c, i0, h, bb);
      }
    }
  } else if (warp == 1) {
    // ---------------- S^T ----------------
    if (lane == 0 && n > 0 && wait_phase(res_full, 0, p.status, 0x413)) {
      constexpr uint32_t idesc_s = tc::idesc_bf16(kRowsTc, kTileTc, false, false);
      const uint32_t base = low_k(smem_addr(smem));
      for (int u = 0; u < n; ++u) {
        const int s = u % ST, set = u & 1;
        // The scores of this buffer are in registers (and what overwrote them has been read).
        if (u >= 2 && !wait_phase((kBlocks == 1 ? ps_full : pv_done) + set, ((u - 2) >> 1) & 1, p.status, 0x415)) break;
        if (!wait_phase(st_full + s, (u / ST) & 1, p.status, 0x414)) break;
        tc::tc_fence_after();
        mma_rows_ss<kBlocks>(tmem + set * kPair + kSCol, base, kRowsTc * 128, base + ((S::kStrOff + s * S::kPer * S::kStr) >> 4),
                             kTileTc * 128, idesc_s, false);
        tc::umma_commit(s_full + set);
      }
    }
  } else if (warp == 2) {
    // ---------------- statistics of the query rows, a tile at a time, and dP^T ----------------
    float m[2], nl[2], dl[2];
    auto fetch = [&](int u) {
      const int h = hk * a.group + u / q_tiles, i0 = u % q_tiles * kTileTc;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int i = i0 + lane + 32 * e;
        const int64_t at = (int64_t(b) * a.heads + h) * a.nq + i;
        m[e] = i < a.nq ? a.lse[at] : -INFINITY;
        nl[e] = i < a.nq ? a.lse[a.lse_plane() + at] : 0.f;
        dl[e] = i < a.nq ? p.x.delta[at] : 0.f;
      }
    };
    constexpr uint32_t idesc_s = tc::idesc_bf16(kRowsTc, kTileTc, false, false);
    const uint32_t base = low_k(smem_addr(smem));
    bool ok = n > 0 && warp_wait(res_full, 0, p.status, 0x41C);
    if (ok) fetch(0);
    for (int u = 0; u < n && ok; ++u) {
      const int s = u % ST, set = u & 1;
      if (u >= ST && !(ok = warp_wait(stat_empty + s, ((u / ST) & 1) ^ 1u, p.status, 0x417))) break;
      float *st = stats + s * 4 * kTileTc;
      bool any_far = false;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = lane + 32 * e;
        const float top = row_max(m[e]), off = -kLog2e * nl[e];
        st[r] = top, st[kTileTc + r] = off, st[3 * kTileTc + r] = -dl[e];
        st[2 * kTileTc + r] = top == INFINITY ? -INFINITY : fmaf(-top, kLog2e, off);
        any_far |= far_row(top);
      }
      any_far = __any_sync(0xffffffffu, any_far);
      if (lane == 0) far_flag[4 * s] = any_far;
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(stat_full + s);
      if (u + 1 < n) fetch(u + 1);
      if (lane == 0) {
        ok = u < 2 || (kBlocks == 1 ? wait_phase(ps_full + set, ((u - 2) >> 1) & 1, p.status, 0x41D)
                                    : wait_phase(st_empty + (u - 2) % ST, ((u - 2) / ST) & 1, p.status, 0x41D));
        ok = ok && wait_phase(st_full + s, (u / ST) & 1, p.status, 0x41E);
        if (ok) {
          tc::tc_fence_after();
          const uint32_t d = base + ((S::kStrOff + s * S::kPer * S::kStr + S::kStr) >> 4);
          mma_rows_ss<kBlocks>(tmem + set * kPair + kDpCol, base + (S::kRes >> 4), kRowsTc * 128, d, kTileTc * 128, idesc_s, false);
          if (kLow)
            mma_rows_ss<kBlocks>(tmem + set * kPair + kDpCol, base + (S::kRes >> 4), kRowsTc * 128, d + (S::kStr >> 4),
                                 kTileTc * 128, idesc_s, true);
          tc::umma_commit(s_full + set);
        }
      }
      ok = __all_sync(0xffffffffu, ok);
    }
  } else if (warp == 3) {
    // ---------------- dV and dK ----------------
    if (lane == 0) {
      const uint32_t idesc_d = tc::idesc_bf16(kRowsTc, (a.d + 15) / 16 * 16, false, true);
      const uint32_t base = low_mn(smem_addr(smem), kTileTc * 128);
      for (int u = 0; u < n; ++u) {
        const int s = u % ST, set = u & 1;
        if (!wait_phase(ps_full + set, (u >> 1) & 1, p.status, 0x416) || !wait_phase(st_full + s, (u / ST) & 1, p.status, 0x41F))
          break;
        tc::tc_fence_after();
        const uint32_t q = base + ((S::kStrOff + s * S::kPer * S::kStr) >> 4), d = q + (S::kStr >> 4);
        const uint32_t pt = tmem + C::pt + set * C::pt_step, ds = tmem + C::ds + set * C::pt_step;
        mma_cols_ts<kTileTc / 16>(tmem + C::dv, pt, d, idesc_d, u != 0);
        if (kLow) mma_cols_ts<kTileTc / 16>(tmem + C::dv, pt, d + (S::kStr >> 4), idesc_d, true);
        tc::umma_commit(pv_done + set);
        mma_cols_ts<kTileTc / 16>(tmem + C::dk, ds, q, idesc_d, u != 0);
        tc::umma_commit(st_empty + s);
        if (u + 1 == n) tc::umma_commit(d_full);
      }
    }
  } else if (warp >= 4) {
    const int set = (warp - 4) >> 2, quarter = warp & 3, row = quarter * 32 + lane, j = j0 + row;
    const uint32_t lanes = tmem + (uint32_t(quarter * 32) << 16);
    const float mkv = mask_value(a, b, j);
    const bool out = mkv == -INFINITY;
    const uint64_t scale2 = dup2(a.scale), log2e2 = dup2(kLog2e), mk2 = dup2(out ? 0.f : mkv);
    bool ok = true;
    const uint32_t pair = lanes + set * kPair;
    for (int u = set; u < n && ok; u += 2) {
      const int s = u % ST;
      if (!(ok = warp_wait(stat_full + s, (u / ST) & 1, p.status, 0x419) &&
                 (!kBias || warp_wait(st_full + s, (u / ST) & 1, p.status, 0x41A)) &&
                 warp_wait(s_full + set, (u >> 1) & 1, p.status, 0x418)))
        break;
      tc::tc_fence_after();
#pragma unroll 1
      for (int half = 0; half < 2; ++half) {
        uint32_t sv[32], dv[32];
        tc::tmem_ld_32x32b_x32(pair + kSCol + 32 * half, sv);
        tc::tmem_ld_32x32b_x32(pair + kDpCol + 32 * half, dv);
        tc::tmem_ld_wait_regs(sv, dv);
        const float *st = stats + s * 4 * kTileTc + 32 * half;
        const bool far = far_flag[4 * s] != 0;
        // bias(q, key): 64-key block row / 64, row q of 128 bytes, 16-byte chunk (key / 8) ^ (q & 7).
        const uint8_t *bias = smem + S::kBiasOff + s * S::kB + (row >> 6) * kTileTc * 128 + 32 * half * 128 + (row & 7) * 2;
        const int chunk = (row & 63) >> 3;
        uint32_t pt[16], ds[16];
        uint64_t z[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          if constexpr (kBias) {
            const uint32_t b0 = *reinterpret_cast<const uint16_t *>(bias + (2 * e) * 128 + ((chunk ^ ((2 * e) & 7)) << 4));
            const uint32_t b1 = *reinterpret_cast<const uint16_t *>(bias + (2 * e + 1) * 128 + ((chunk ^ ((2 * e + 1) & 7)) << 4));
            z[e] = add2(fma2(pack2(sv[2 * e], sv[2 * e + 1]), scale2, pack2(b0 << 16, b1 << 16)), mk2);
          } else {
            z[e] = fma2(pack2(sv[2 * e], sv[2 * e + 1]), scale2, mk2);
          }
        }
        if (far)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            z[e] = pack2(__float_as_uint(fmaf(lo_f(z[e]) - st[2 * e], kLog2e, st[kTileTc + 2 * e])),
                         __float_as_uint(fmaf(hi_f(z[e]) - st[2 * e + 1], kLog2e, st[kTileTc + 2 * e + 1])));
        else
#pragma unroll
          for (int e = 0; e < 16; ++e) z[e] = fma2(z[e], log2e2, *reinterpret_cast<const uint64_t *>(st + 2 * kTileTc + 2 * e));
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float p0 = fast_exp2(lo_f(z[e])), p1 = fast_exp2(hi_f(z[e]));
          const uint64_t prob = pack2(__float_as_uint(p0), __float_as_uint(p1));
          const uint64_t g = mul2(prob, add2(pack2(dv[2 * e], dv[2 * e + 1]), *reinterpret_cast<const uint64_t *>(st + 3 * kTileTc + 2 * e)));
          pt[e] = out ? 0u : pack_bf16x2(p0, p1);
          ds[e] = out ? 0u : pack_bf16x2(lo_f(g), hi_f(g));
        }
        // Wide rows: over columns that this half or the first one has read.  Else dV and dK have
        // read what tile u - 2 left here.
        if (kBlocks == 1 && half == 0 && u >= 2 && !(ok = warp_wait(st_empty + (u - 2) % ST, ((u - 2) / ST) & 1, p.status, 0x420)))
          break;
        tc::tmem_st_32x32b_x16(lanes + C::pt + set * C::pt_step + 16 * half, pt);
        tc::tmem_st_32x32b_x16(lanes + C::ds + set * C::pt_step + 16 * half, ds);
      }
      if (!ok) break;
      tc::tmem_st_wait();
      tc::tc_fence_before();
      if (kBias) tc::fence_proxy_async_smem();  // the bias block has been read
      __syncwarp();
      if (lane == 0) {
        tc::mbar_arrive(stat_empty + s);
        tc::mbar_arrive(ps_full + set);
      }
    }
    if (ok && n > 0) ok = warp_wait(d_full, 0, p.status, 0x41B);
    tc::tc_fence_after();
    if (ok) {
      const int64_t at = ((int64_t(b) * a.nk + j) * kv_heads + hk) * a.d;
      for (int c = set; c < (a.d + 15) / 16; c += 2) {
        uint32_t gv[16], gk[16];
        if (n > 0) {
          tc::tmem_ld_32x32b_x16(lanes + C::dv + 16 * c, gv);
          tc::tmem_ld_32x32b_x16(lanes + C::dk + 16 * c, gk);
          tc::tmem_ld_wait();
        }
#pragma unroll
        for (int e8 = 0; e8 < 2; ++e8) {
          const int c0 = 16 * c + 8 * e8;
          if (j >= a.nk || c0 >= a.d) continue;
          uint32_t wv[4], wk[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int o = 8 * e8 + 2 * e;
            wv[e] = n > 0 ? pack_bf16x2(__uint_as_float(gv[o]), __uint_as_float(gv[o + 1])) : 0u;
            wk[e] = n > 0 ? pack_bf16x2(__uint_as_float(gk[o]) * a.scale, __uint_as_float(gk[o + 1]) * a.scale) : 0u;
          }
          *reinterpret_cast<uint4 *>(static_cast<Bf *>(p.x.dv) + at + c0) = make_uint4(wv[0], wv[1], wv[2], wv[3]);
          *reinterpret_cast<uint4 *>(static_cast<Bf *>(p.x.dk) + at + c0) = make_uint4(wk[0], wk[1], wk[2], wk[3]);
        }
      }
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, 512);
  }
}

// Gradient of a bias that several samples share: one CTA = 128 query rows of one (bias, head) over a
// range of key tiles; for each tile the samples' Q, dO, K and V stream through a three-stage ring and the
// threads add up dS in registers.  Bound by those reads from L2 (64 KB per 128 x 64 scores, some 5 TB/s).  d <= 64 (two 64-column blocks would leave one stage).
template <bool kLow> struct BShape {
  static constexpr int kRes = kRowsTc * 128, kStr = kTileTc * 128, kPer = kLow ? 3 : 2;
  static constexpr int kStage = kPer * kRes + 2 * kStr;  // Q, dO, do - bf16(do), K, V
  static constexpr int kB = kRowsTc * kTileTc * 2;
  static constexpr int kStages = 3, kBiasOff = kStages * kStage, kMaskOff = kBiasOff + 2 * kB, kBarOff = kMaskOff + 8 * 32 * 4;
  static constexpr int kBytes = kBarOff + 256 + 1024;
};

template <bool kLow>
__global__ void __launch_bounds__(kThreadsTc, 1)
    bias_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_do,
                   const __grid_constant__ CUtensorMap map_low, const __grid_constant__ CUtensorMap map_k,
                   const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_bias, const BackTc p,
                   int ranges) {
  using S = BShape<kLow>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + S::kBarOff);
  constexpr int ST = S::kStages;
  uint64_t *st_full = bars, *st_empty = bars + ST;    // [ST] a sample's tiles landed; its products are done
  uint64_t *b_full = st_empty + ST, *b_empty = b_full + 2;  // [2] bias block landed; it has been read
  uint64_t *s_full = b_empty + 2, *s_free = s_full + 2;     // [2] S and dP in TMEM; in registers
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(s_free + 2);
  const Args &a = p.x.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int64_t at = blockIdx.x;
  const int range = int(at % ranges);
  at /= ranges;
  const int q0 = int(at % p.tiles) * kRowsTc;
  at /= p.tiles;
  const int h = int(at % a.heads), bb = int(at / a.heads), hk = h / a.group;
  const int key_tiles = (a.nk + kTileTc - 1) / kTileTc;
  const int t0 = int(int64_t(range) * key_tiles / ranges), t1 = int(int64_t(range + 1) * key_tiles / ranges);
  const int n = (t1 - t0) * a.share;  // (key tile, sample) steps
  if (tid == 0) {
    for (int i = 0; i < ST; ++i) tc::mbar_init(st_full + i, 1), tc::mbar_init(st_empty + i, 2);
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(b_full + i, 1), tc::mbar_init(b_empty + i, 8);
      tc::mbar_init(s_full + i, 2), tc::mbar_init(s_free + i, 8);
    }
    tc::fence_mbar_init();
  }
  if (warp == 1) {
    tc::tmem_alloc(tmem_slot, 256);
    tc::tmem_relinquish();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  if (warp == 0) {
    if (lane == 0)
      for (int u = 0; u < n; ++u) {
        const int s = u % ST, jt = u / a.share, b = bb * a.share + u % a.share, j0 = (t0 + jt) * kTileTc;
        if (u >= ST && !wait_phase(st_empty + s, ((u / ST) & 1) ^ 1u, p.status, 0x421)) break;
        uint8_t *st = smem + s * S::kStage;
        tc::mbar_arrive_expect_tx(st_full + s, S::kStage);
        tma_load_4d(st, &map_q, st_full + s, 0, q0, h, b);
        tma_load_4d(st + S::kRes, &map_do, st_full + s, 0, q0, h, b);
        if (kLow) tma_load_4d(st + 2 * S::kRes, &map_low, st_full + s, 0, q0, h, b);
        tma_load_4d(st + S::kPer * S::kRes, &map_k, st_full + s, 0, j0, hk, b);
        tma_load_4d(st + S::kPer * S::kRes + S::kStr, &map_v, st_full + s, 0, j0, hk, b);
        if (u % a.share == 0) {
          const int bs = jt & 1;
          if (jt >= 2 && !wait_phase(b_empty + bs, ((jt >> 1) & 1) ^ 1u, p.status, 0x422)) break;
          tc::mbar_arrive_expect_tx(b_full + bs, S::kB);
          tma_load_4d(smem + S::kBiasOff + bs * S::kB, &map_bias, b_full + bs, j0, q0, h, bb);
        }
      }
  } else if (warp < 3) {
    // ---------------- S (warp 1) and dP (warp 2) ----------------
    if (lane == 0) {
      constexpr uint32_t idesc = tc::idesc_bf16(kRowsTc, kTileTc, false, false);
      const uint32_t base = low_k(smem_addr(smem));
      for (int u = 0; u < n; ++u) {
        const int s = u % ST, buf = u & 1;
        if (!wait_phase(st_full + s, (u / ST) & 1, p.status, 0x423)) break;
        if (u >= 2 && !wait_phase(s_free + buf, ((u - 2) >> 1) & 1, p.status, 0x424)) break;
        tc::tc_fence_after();
        const uint32_t q = base + (s * S::kStage >> 4), k = q + (S::kPer * S::kRes >> 4);
        if (warp == 1) {
          mma_rows_ss<1>(tmem + buf * kPair + kSCol, q, 0, k, 0, idesc, false);
        } else {
#pragma unroll
          for (int t = 1; t < S::kPer; ++t)
            mma_rows_ss<1>(tmem + buf * kPair + kDpCol, q + (t * S::kRes >> 4), 0, k + (S::kStr >> 4), 0, idesc, t > 1);
        }
        tc::umma_commit(s_full + buf);
        tc::umma_commit(st_empty + s);
      }
    }
  } else if (warp >= 4) {
    const int half = (warp - 4) >> 2, quarter = warp & 3, row = quarter * 32 + lane, i = q0 + row;
    const uint32_t lanes = tmem + (uint32_t(quarter * 32) << 16);
    float *mk = reinterpret_cast<float *>(smem + S::kMaskOff) + (warp - 4) * 32;
    const uint64_t scale2 = dup2(a.scale), log2e2 = dup2(kLog2e);
    uint64_t acc[16];
    // A step's statistics and mask values are fetched a step ahead.
    float m, nl, delta, mv;
    auto fetch = [&](int u) {
      const int b = bb * a.share + u % a.share;
      m = -INFINITY, nl = delta = 0.f;
      if (i < a.nq) {
        const int64_t r = (int64_t(b) * a.heads + h) * a.nq + i;
        m = a.lse[r], nl = a.lse[a.lse_plane() + r], delta = p.x.delta[r];
      }
      mv = mask_value(a, b, (t0 + u / a.share) * kTileTc + 32 * half + lane);
    };
    if (n > 0) fetch(0);
    for (int u = 0; u < n; ++u) {
      const int jt = u / a.share, first = u % a.share == 0, buf = u & 1;
      const int k0 = (t0 + jt) * kTileTc + 32 * half;
      m = row_max(m), nl *= -kLog2e;
      const bool adds = __any_sync(0xffffffffu, mv != 0.f && mv != -INFINITY);
      const uint32_t cut = __ballot_sync(0xffffffffu, mv == -INFINITY);
      if (adds) {
        __syncwarp();
        mk[lane] = mv == -INFINITY ? 0.f : mv;
        __syncwarp();
      }
      const bool far = __any_sync(0xffffffffu, far_row(m));
      const uint64_t c2 = dup2(m == INFINITY ? -INFINITY : fmaf(-m, kLog2e, nl)), delta2 = dup2(-delta);
      const float m_now = m, nl_now = nl;
      if (u + 1 < n) fetch(u + 1);
      if (!warp_wait(s_full + buf, (u >> 1) & 1, p.status, 0x425)) break;
      tc::tc_fence_after();
      uint32_t sv[32], dv[32];
      tc::tmem_ld_32x32b_x32(lanes + buf * kPair + kSCol + 32 * half, sv);
      tc::tmem_ld_32x32b_x32(lanes + buf * kPair + kDpCol + 32 * half, dv);
      const bool ok = !first || warp_wait(b_full + (jt & 1), (jt >> 1) & 1, p.status, 0x426);
      tc::tmem_ld_wait_regs(sv, dv);
      if (!ok) break;
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(s_free + buf);
      const uint32_t brow = smem_addr(smem + S::kBiasOff + (jt & 1) * S::kB) + row * 128;
      uint64_t z[16];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const uint4 v = lds128(brow + (((4 * half + c) ^ (row & 7)) << 4));
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          z[4 * c + e] = fma2(pack2(sv[8 * c + 2 * e], sv[8 * c + 2 * e + 1]), scale2, pack2(w[e] << 16, w[e] & 0xffff0000u));
      }
      if (adds)
#pragma unroll
        for (int e = 0; e < 16; ++e) z[e] = add2(z[e], *reinterpret_cast<const uint64_t *>(mk + 2 * e));
      if (far)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          z[e] = pack2(__float_as_uint(fmaf(lo_f(z[e]) - m_now, kLog2e, nl_now)), __float_as_uint(fmaf(hi_f(z[e]) - m_now, kLog2e, nl_now)));
      else
#pragma unroll
        for (int e = 0; e < 16; ++e) z[e] = fma2(z[e], log2e2, c2);
#pragma unroll
      for (int e = 0; e < 16; ++e)
        z[e] = mul2(pack2(__float_as_uint(fast_exp2(lo_f(z[e]))), __float_as_uint(fast_exp2(hi_f(z[e])))),
                    add2(pack2(dv[2 * e], dv[2 * e + 1]), delta2));
      if (cut)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const uint32_t out = cut >> (2 * e);
          z[e] = pack2(out & 1 ? 0u : uint32_t(z[e]), out & 2 ? 0u : uint32_t(z[e] >> 32));
        }
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[e] = first ? z[e] : add2(acc[e], z[e]);
      if ((u + 1) % a.share == 0) {
        if (i < a.nq) {
          Bf *dst = static_cast<Bf *>(p.x.dbias) + ((int64_t(bb) * a.heads + h) * a.nq + i) * p.x.dbias_ld;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = pack_bf16x2(lo_f(acc[4 * c + e]), hi_f(acc[4 * c + e]));
            const int k = k0 + 8 * c;
            if (k + 8 <= a.nk)
              *reinterpret_cast<uint4 *>(dst + k) = make_uint4(w[0], w[1], w[2], w[3]);
            else
#pragma unroll
              for (int e = 0; e < 8; ++e)
                if (k + e < a.nk) reinterpret_cast<uint16_t *>(dst)[k + e] = uint16_t(w[e >> 1] >> (16 * (e & 1)));
          }
        }
        tc::fence_proxy_async_smem();  // the bias block has been read
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(b_empty + (jt & 1));
      }
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, 256);
  }
}

// The six maps of a kernel whose resident tiles are 128 rows; false where TMA cannot describe one.
bool back_maps(CUtensorMap (&m)[6], const BackArgs &x, bool queries_resident) {
  const Args &a = x.a;
  const int kv_heads = a.heads / a.group, qr = queries_resident ? kRowsTc : kTileTc, kr = queries_resident ? kTileTc : kRowsTc;
  const Rows dout{x.dout, int64_t(a.nq) * a.heads * a.d, int64_t(a.heads) * a.d, a.d};
  Rows low = dout;
  if (x.dlow) low.p = x.dlow;
  if (!rows_map(&m[0], a.q, a.d, a.nq, a.heads, a.batch, qr) || !rows_map(&m[1], dout, a.d, a.nq, a.heads, a.batch, qr) ||
      !rows_map(&m[2], low, a.d, a.nq, a.heads, a.batch, qr) || !rows_map(&m[3], a.k, a.d, a.nk, kv_heads, a.batch, kr) ||
      !rows_map(&m[4], a.v, a.d, a.nk, kv_heads, a.batch, kr))
    return false;
  m[5] = m[0];
  const Rows bias{a.bias, a.bias_sb, a.bias_si, a.bias_sh};
  return !a.bias || rows_map(&m[5], bias, a.nk, a.nq, a.heads, a.batch / a.share, qr);
}

bool back_covered(const Args &a) {
  return a.nk >= 64 && worth_tiles(a) && !(a.bias && !a.bias_vec) && a.batch > 0;
}

template <typename K> int back_launch(K kernel, int bytes, const BackTc &p, int64_t ctas, const CUtensorMap (&m)[6], cudaStream_t stream) {
  BL_REQUIRE(p.status, "bl_cross_attention_backward: device status word unavailable");
  BL_REQUIRE(ctas < (int64_t(1) << 31), "bl_cross_attention_backward: too many tiles");
  BL_CUDA(ensure_smem_limit(reinterpret_cast<const void *>(kernel), bytes));
  kernel<<<unsigned(ctas), kThreadsTc, bytes, stream>>>(m[0], m[1], m[2], m[3], m[4], m[5], p);
  BL_LAUNCH_CHECK();
  return BL_OK;
}

}  // namespace

#define BL_PICK(KERNEL, SHAPE, W, B, L)                                                                       \
  do {                                                                                                        \
    static_assert(SHAPE<W, B, L>::kBytes <= 232448, "shared memory");                                         \
    return back_launch(KERNEL<W, B, L>, SHAPE<W, B, L>::kBytes, p, ctas, maps, stream);                       \
  } while (0)
#define BL_DISPATCH(KERNEL, SHAPE)                                                                            \
  do {                                                                                                        \
    if (a.d > 64) {                                                                                           \
      if (a.bias) { if (x.dlow) BL_PICK(KERNEL, SHAPE, 2, true, true); BL_PICK(KERNEL, SHAPE, 2, true, false); } \
      if (x.dlow) BL_PICK(KERNEL, SHAPE, 2, false, true);                                                     \
      BL_PICK(KERNEL, SHAPE, 2, false, false);                                                                \
    }                                                                                                         \
    if (a.bias) { if (x.dlow) BL_PICK(KERNEL, SHAPE, 1, true, true); BL_PICK(KERNEL, SHAPE, 1, true, false); } \
    if (x.dlow) BL_PICK(KERNEL, SHAPE, 1, false, true);                                                       \
    BL_PICK(KERNEL, SHAPE, 1, false, false);                                                                  \
  } while (0)

int queries_tc(const BackArgs &x, cudaStream_t stream, bool *taken) {
  const Args &a = x.a;
  CUtensorMap maps[6];
  *taken = back_covered(a) && back_maps(maps, x, true);
  if (!*taken) return BL_OK;
  BackTc p{x, (a.nq + kRowsTc - 1) / kRowsTc, device_status_ptr()};
  const int64_t ctas = int64_t(p.tiles) * a.heads * a.batch;
  BL_DISPATCH(queries_tc_kernel, QShape);
}

int keys_tc(const BackArgs &x, cudaStream_t stream, bool *taken) {
  const Args &a = x.a;
  CUtensorMap maps[6];
  *taken = back_covered(a) && back_maps(maps, x, false);
  if (!*taken) return BL_OK;
  BackTc p{x, (a.nk + kRowsTc - 1) / kRowsTc, device_status_ptr()};
  const int64_t ctas = int64_t(p.tiles) * (a.heads / a.group) * a.batch;
  BL_DISPATCH(keys_tc_kernel, KShape);
}

int bias_tc(const BackArgs &x, cudaStream_t stream, bool *taken) {
  const Args &a = x.a;
  CUtensorMap maps[6];
  *taken = a.d <= 64 && back_covered(a) && back_maps(maps, x, true);
  if (!*taken) return BL_OK;
  BackTc p{x, (a.nq + kRowsTc - 1) / kRowsTc, device_status_ptr()};
  BL_REQUIRE(p.status, "bl_cross_attention_backward: device status word unavailable");
  // Few row tiles: the keys are divided so that one wave of CTAs (one per SM) covers them.
  const int64_t base = int64_t(p.tiles) * a.heads * (a.batch / a.share), key_tiles = (a.nk + kTileTc - 1) / kTileTc;
  int64_t ranges = num_sms() / base;
  ranges = ranges < 1 ? 1 : ranges > key_tiles ? key_tiles : ranges;
  BL_REQUIRE(base * ranges < (int64_t(1) << 31), "bl_cross_attention_backward: too many bias blocks");
  auto kernel = x.dlow ? bias_tc_kernel<true> : bias_tc_kernel<false>;
  const int bytes = x.dlow ? BShape<true>::kBytes : BShape<false>::kBytes;
  static_assert(BShape<true>::kBytes <= 232448, "shared memory");
  BL_CUDA(ensure_smem_limit(reinterpret_cast<const void *>(kernel), bytes));
  kernel<<<unsigned(base * ranges), kThreadsTc, bytes, stream>>>(maps[0], maps[1], maps[2], maps[3], maps[4], maps[5], p,
                                                                 int(ranges));
  BL_LAUNCH_CHECK();
  return BL_OK;
}

}  // namespace xa
}  // namespace bl
