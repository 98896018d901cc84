// Parts shared by the tcgen05 cross-attention kernels.
#pragma once

#include "cross_attention.cuh"
#include "tc.cuh"

namespace bl {
namespace xa {
namespace {

constexpr int kMaskWords = 2048;  // keys whose mask is kept as bits in shared memory, / 32

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
// Bounded wait that polls: tc::mbar_wait's timer read and timed suspension lengthen the
// chain of waits per tile (5 % of the kernel); the timer is read once in 4096 polls.
__device__ __forceinline__ bool wait_phase(uint64_t *bar, uint32_t parity, unsigned int *status, unsigned code) {
  uint64_t start = 0;
  for (uint32_t spin = 1;; ++spin) {
    if (tc::mbar_try_wait(bar, parity)) return true;
    if ((spin & 4095u) == 0) {
      if (*reinterpret_cast<volatile unsigned int *>(status) != 0u) return false;
      const uint64_t now = tc::global_timer_ns();
      if (start == 0) start = now;
      if (now - start > tc::kWaitLimitNs) {
        atomicCAS(status, 0u, code);
        return false;
      }
    }
  }
}
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity, unsigned int *status, unsigned code) {
  return __all_sync(0xffffffffu, wait_phase(bar, parity, status, code));
}

// The MMA issuers compute only the low words of descriptors (address, offset between blocks) and
// unroll over the K steps: building 64-bit descriptors in a loop took 92 cycles per MMA of 64
// columns, this 53, of which 48 are the operands' shared-memory reads.
__device__ __forceinline__ uint32_t low_k(uint32_t saddr) { return uint32_t(desc_k(saddr)); }
__device__ __forceinline__ uint32_t low_mn(uint32_t saddr, uint32_t block_bytes) {
  return uint32_t(tc::desc_sw128(saddr, block_bytes));
}
__device__ __forceinline__ uint64_t with_low(uint32_t low) {
  return uint64_t(low) | uint64_t(1024 >> 4) << 32 | uint64_t(1) << 46 | uint64_t(2) << 61;
}
// D (+)= A B^T over kBlocks * 64 columns: A and B rows of 128-byte swizzled 64-column blocks that are
// a_block and b_block bytes apart, their descriptors' low words.  Columns past d are zero and
// multiplied all the same: a test per step costs more than the steps.
template <int kBlocks>
__device__ __forceinline__ void mma_rows_ss(uint32_t d_tmem, uint32_t a, int a_block, uint32_t b, int b_block,
                                            uint32_t idesc, bool add) {
#pragma unroll
  for (int e = 0; e < 4 * kBlocks; ++e)
    tc::umma_f16_ss(d_tmem, with_low(a + (e >> 2) * (a_block >> 4) + (e & 3) * 2),
                    with_low(b + (e >> 2) * (b_block >> 4) + (e & 3) * 2), idesc, add || e != 0);
}
// D (+)= A B over 16 kSteps rows of B: A 16-bit pairs in TMEM, B rows of 128 bytes, low_mn's word.
template <int kSteps>
__device__ __forceinline__ void mma_cols_ts(uint32_t d_tmem, uint32_t a_tmem, uint32_t b, uint32_t idesc, bool add) {
#pragma unroll
  for (int e = 0; e < kSteps; ++e) tc::umma_f16_ts(d_tmem, a_tmem + e * 8, with_low(b + e * 128), idesc, add || e != 0);
}

// A row whose reference m is far from zero: m is subtracted from its scores before the change of base.  Else -m log2(e) is
// rounded once into an offset of the exponents (and once more with the log of the sum in the gradients), which costs
// at most |m| 2^-23 of a probability: 2^-13 here, a 32nd of what rounding it to bf16 does.  Without the limit a sample whose
// keys are all masked by -1e6 came out 2.3 times further off than its bounds, by -1e9 with gradients of 1e7, by -1e10 as NaN.
constexpr float kFar = 1024.f;
__device__ __forceinline__ bool far_row(float m) { return fabsf(m) > kFar && fabsf(m) != INFINITY; }

__device__ __forceinline__ int n_words(int nk) { return (nk + 31) / 32; }
// At most 64 queries leave half or more of a tile's rows idle: taken over many keys while the heads do not fill the
// GPU.  Forward and gradients of 32 queries in us (d = 64, no bias, no mask), against the kernels on warp products, which
// divide the keys among clusters too: 8 heads, 256 keys 13 / 24 against 16 / 26, 4096 keys 22 / 79 against 25 / 46; 64 heads,
// 256 keys 17 / 26 against 16 / 28, 4096 keys 49 / 169 against 41 / 124; 148 heads, 1024 keys 28 / 87 against 29 / 79; past
// the limit, 192 heads, 256 keys 28 / 48 against 17 / 40, 512 heads, 1024 keys 83 / 286 against 49 / 200.  At 128 keys
// (every head count) the warp products are as fast or faster.  The rule follows the forward of few heads; gradients over
// 1024 keys or more and the forward of 64 heads are slower by it.
inline bool worth_tiles(const Args &a) {
  return a.nq > 64 || (a.nk >= 256 && int64_t(a.heads) * a.batch <= num_sms());
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

}  // namespace
}  // namespace xa
}  // namespace bl
