// Shared parts of the cross-attention kernels: arguments, tile loads and warp products.
//
//   x[b, h, i, j] = (q[b, i, h] . k[b, j, h']) scale + bias[b / share, h, i, j] + mk[b, j],  h' = h / (heads / kv_heads)
//   p = softmax_j(x)  (a row whose keys are all left out: p = 0)
//   o = sum_j p v[b, j, h'],  out = sigmoid(gate) o
// mk is 0, -inf for a left-out key, or inf (mask - 1) with an additive mask.
//
// The warp products take 16 x K times K x 8 steps of mma.sync: bf16 operands
// directly; fp32 operands as tf32 pairs x = hi + lo (11 significant bits each,
// hi rounded, lo truncated), with lo hi + hi lo + hi hi accumulated in fp32: the
// dropped terms are below 3 2^-21 of a product.
#pragma once

#include "common.cuh"

namespace bl {
namespace xa {

enum MaskKind { kMaskNone = 0, kMaskKeep = 1, kMaskAdd = 2 };

struct Rows {  // a [batch][rows][heads][d] view with contiguous d
  const void *p;
  int64_t sb, si, sh;
};

struct Args {
  Rows q, k, v, gate;  // gate.p may be null
  const void *bias;    // null: none; element (b', h, i, j) at b'*bias_sb + h*bias_sh + i*bias_si + j
  int64_t bias_sb, bias_sh, bias_si;
  int bias_vec;        // bias rows start on 16-byte boundaries
  int share;           // samples per bias (1 without bias)
  const void *mask;    // kMaskKeep: uint8, kMaskAdd: fp32; [batch][nk] with row stride mask_sb
  int64_t mask_sb;
  int mask_kind;
  float inf, scale;
  int batch, heads, group, nq, nk, d;  // group: query heads per key/value head
  void *out;    // [batch][nq][heads][d]
  void *low;    // like out, or null: what rounding to bf16 took from out, itself rounded to bf16
  float *lse;   // [2][batch][heads][nq] or null: a reference of the row's scores, log of the sum relative to it
  __host__ __device__ int64_t lse_plane() const { return int64_t(batch) * heads * nq; }
};

template <typename T> struct Type;
template <> struct Type<__nv_bfloat16> {
  static constexpr int kVec = 8, kPad = 8;  // elements per 16 bytes; row padding: 16-byte matrix rows hit distinct banks
};
template <> struct Type<float> {
  static constexpr int kVec = 4, kPad = 4;  // rows = 4 mod 32 banks: both fragment patterns are conflict-free
};
template <typename T, int DP> constexpr int kLd = DP + Type<T>::kPad;

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ uint32_t smem_addr(const void *p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void cp16(void *dst, const void *src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(dst)), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void cp_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Shared memory of the cluster's other CTAs.
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float peer(const float *local, uint32_t rank) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_addr(local)), "r"(rank));
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote) : "memory");
  return v;
}

__device__ __forceinline__ float4 peer4(const float4 *local, uint32_t rank) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_addr(local)), "r"(rank));
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(remote)
               : "memory");
  return v;
}

// Rows [row0, row0 + kRows) of a view's (b, h) slab into shared [kRows][kLd];
// rows past n and columns past d are zero.  `tid` of `threads` threads.
template <typename T, int DP, int kRows>
__device__ __forceinline__ void load_rows(T *dst, const T *src, int64_t stride, int row0, int n, int d, int tid,
                                          int threads) {
  constexpr int kVec = Type<T>::kVec, kChunks = DP / kVec;
#pragma unroll 4
  for (int u = tid; u < kRows * kChunks; u += threads) {
    const int r = u / kChunks, c = u % kChunks * kVec;
    const bool ok = row0 + r < n && c < d;
    cp16(dst + r * kLd<T, DP> + c, ok ? src + (row0 + r) * stride + c : src, ok ? 16 : 0);
  }
}

// The bias block of query rows [i0, i0 + rows) and keys [j0, j0 + kCols) into
// shared [rows][kCols + 8] (elements past the ends: any finite or zero value;
// the callers leave their scores out).
template <typename T, int kCols>
__device__ __forceinline__ void load_bias(T *dst, const T *bias, const Args &a, int i0, int rows, int j0, int tid,
                                          int threads) {
  constexpr int kVec = Type<T>::kVec, kChunks = kCols / kVec;
  if (a.bias_vec) {
#pragma unroll 4
    for (int u = tid; u < rows * kChunks; u += threads) {
      const int r = u / kChunks, c = u % kChunks * kVec;
      const int left = a.nk - j0 - c;
      const int bytes = i0 + r < a.nq && left > 0 ? (left < kVec ? left * int(sizeof(T)) : 16) : 0;
      cp16(dst + r * (kCols + 8) + c, bytes ? bias + int64_t(i0 + r) * a.bias_si + j0 + c : bias, bytes);
    }
  } else {
    for (int u = tid; u < rows * kCols; u += threads) {
      const int r = u / kCols, c = u % kCols;
      T x = T(0.f);
      if (i0 + r < a.nq && j0 + c < a.nk) x = bias[int64_t(i0 + r) * a.bias_si + j0 + c];
      dst[r * (kCols + 8) + c] = x;
    }
  }
}

// Two neighbouring elements of an fp32 bias row from an even column, `left` of the row at hand (the others 0).
__device__ __forceinline__ float2 bias_pair(const Args &a, const float *p, int left) {
  if (a.bias_vec && left > 1) return *reinterpret_cast<const float2 *>(p);
  return make_float2(left > 0 ? p[0] : 0.f, left > 1 ? p[1] : 0.f);
}

// mk of key j (see above); keys past nk are left out.
__device__ __forceinline__ float mask_value(const Args &a, int b, int j) {
  if (j >= a.nk) return -INFINITY;
  if (a.mask_kind == kMaskNone) return 0.f;
  if (a.mask_kind == kMaskKeep)
    return static_cast<const uint8_t *>(a.mask)[b * a.mask_sb + j] ? 0.f : -INFINITY;
  return a.inf * (static_cast<const float *>(a.mask)[b * a.mask_sb + j] - 1.f);
}

// Bits of keys [32 w, 32 w + 32): left out by a keep mask, changed by an additive one, or past nk.
__device__ __forceinline__ uint32_t mask_word(const Args &a, int b, int w) {
  uint32_t word = 0;
  const int j0 = 32 * w;
  if (a.mask_kind == kMaskKeep) {
    const uint8_t *m = static_cast<const uint8_t *>(a.mask) + b * a.mask_sb + j0;
    if (j0 + 32 <= a.nk && (reinterpret_cast<uintptr_t>(m) & 15) == 0) {
      const uint4 v[2] = {reinterpret_cast<const uint4 *>(m)[0], reinterpret_cast<const uint4 *>(m)[1]};
      const uint32_t u[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w};
#pragma unroll
      for (int e = 0; e < 8; ++e)  // 0xff where a byte is zero; its low bits gathered to four
        word |= ((__vcmpeq4(u[e], 0u) & 0x01010101u) * 0x10204080u >> 28) << (4 * e);
    } else {
#pragma unroll
      for (int e = 0; e < 32; ++e) word |= uint32_t(j0 + e >= a.nk || m[e] == 0) << e;
    }
  } else {
#pragma unroll 8
    for (int e = 0; e < 32; ++e) word |= uint32_t(mask_value(a, b, j0 + e) != 0.f) << e;
  }
  return word;
}

// Two neighbouring elements of a shared row.
__device__ __forceinline__ float2 load2(const float *p) { return *reinterpret_cast<const float2 *>(p); }
__device__ __forceinline__ float2 load2(const __nv_bfloat16 *p) {
  const uint32_t v = *reinterpret_cast<const uint32_t *>(p);
  return make_float2(bf16_lo(v), bf16_hi(v));
}
__device__ __forceinline__ void store2(float *p, float x, float y) { *reinterpret_cast<float2 *>(p) = make_float2(x, y); }
__device__ __forceinline__ void store2(__nv_bfloat16 *p, float x, float y) {
  *reinterpret_cast<uint32_t *>(p) = pack_bf16x2(x, y);
}

// ---------------------------------------------------------------------------
// Warp products (fragment layouts of mma.sync m16n8: row g = lane / 4 and g + 8,
// columns 2 (lane % 4) and + 1 of each 8-column tile)
// ---------------------------------------------------------------------------
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], const void *p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(smem_addr(p)));
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], const void *p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(smem_addr(p)));
}
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
               "{%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma8(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
               "{%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
__device__ __forceinline__ void split_tf32(float x, uint32_t &hi, uint32_t &lo) {
  hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;  // half a step away from zero, then cut: nearest
  lo = __float_as_uint(x - __uint_as_float(hi)) & 0xffffe000u;
}

// acc[NT][4] += A B^T over DP: A = 16 shared rows, B = 8 NT shared rows (both [row][kLd]).
template <int NT, int DP>
__device__ __forceinline__ void mma_rows(float (&acc)[NT][4], const __nv_bfloat16 *a, const __nv_bfloat16 *b, int lane) {
  constexpr int ld = kLd<__nv_bfloat16, DP>;
  const __nv_bfloat16 *ap = a + (lane & 15) * ld + (lane >> 4) * 8;
  const __nv_bfloat16 *bp = b + ((lane & 7) + ((lane >> 4) << 3)) * ld + ((lane >> 3) & 1) * 8;
#pragma unroll
  for (int kk = 0; kk < DP / 16; ++kk) {
    uint32_t ar[4];
    ldsm4(ar, ap + kk * 16);
#pragma unroll
    for (int n = 0; n < NT; n += 2) {
      uint32_t br[4];
      ldsm4(br, bp + n * 8 * ld + kk * 16);
      mma16(acc[n], ar, br[0], br[1]);
      mma16(acc[n + 1], ar, br[2], br[3]);
    }
  }
}
// fp32: the two small products have accumulators of their own (the tensor core cuts every
// running sum towards zero, so a sum of 3 n terms would drift three times as far).
template <int NT, int DP>
__device__ __forceinline__ void mma_rows(float (&acc)[NT][4], const float *a, const float *b, int lane) {
  constexpr int ld = kLd<float, DP>, kN = NT < 4 ? NT : 4;
  const int g = lane >> 2, t = lane & 3;
  const float *ap = a + g * ld + t, *bp = b + g * ld + t;
#pragma unroll
  for (int n0 = 0; n0 < NT; n0 += kN) {
    float small[kN][4];
#pragma unroll
    for (int n = 0; n < kN; ++n) small[n][0] = small[n][1] = small[n][2] = small[n][3] = 0.f;
#pragma unroll 4
    for (int kk = 0; kk < DP / 8; ++kk) {
      uint32_t ah[4], al[4], bh[kN][2], bl[kN][2];
      split_tf32(ap[kk * 8], ah[0], al[0]);
      split_tf32(ap[kk * 8 + 8 * ld], ah[1], al[1]);
      split_tf32(ap[kk * 8 + 4], ah[2], al[2]);
      split_tf32(ap[kk * 8 + 8 * ld + 4], ah[3], al[3]);
#pragma unroll
      for (int n = 0; n < kN; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) split_tf32(bp[(n0 + n) * 8 * ld + kk * 8 + 4 * e], bh[n][e], bl[n][e]);
#pragma unroll
      for (int n = 0; n < kN; ++n) mma8(small[n], al, bh[n]);
#pragma unroll
      for (int n = 0; n < kN; ++n) mma8(acc[n0 + n], ah, bh[n]);
#pragma unroll
      for (int n = 0; n < kN; ++n) mma8(small[n], ah, bl[n]);
    }
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[n0 + n][e] += small[n][e];
  }
}

// acc[DP / 8][4] += P V: P = a 16 x 8 KT fragment in registers (accumulator
// layout), V = 8 KT shared rows [row][kLd].  fp32: the tf32 A layout wants
// columns t and t + 4 where the accumulator holds 2 t and 2 t + 1; the sum
// over rows of V does not care, so V's rows are read in the matching order.
// A tile's sum starts at zero and is added to acc in fp32: run through the tensor
// core over all tiles, a sum over 2860 keys came out 1.1e-6 low, added 4e-7.
template <int KT, int DP>
__device__ __forceinline__ void mma_acc(float (&acc)[DP / 8][4], const float (&p)[KT][4], const __nv_bfloat16 *v,
                                        int lane) {
  constexpr int ld = kLd<__nv_bfloat16, DP>;
  const __nv_bfloat16 *vp = v + (lane & 15) * ld + (lane >> 4) * 8;
#pragma unroll
  for (int kk = 0; kk < KT / 2; ++kk) {
    const uint32_t ar[4] = {pack_bf16x2(p[2 * kk][0], p[2 * kk][1]), pack_bf16x2(p[2 * kk][2], p[2 * kk][3]),
                            pack_bf16x2(p[2 * kk + 1][0], p[2 * kk + 1][1]),
                            pack_bf16x2(p[2 * kk + 1][2], p[2 * kk + 1][3])};
#pragma unroll
    for (int n = 0; n < DP / 8; n += 2) {
      uint32_t br[4];
      ldsm4_t(br, vp + kk * 16 * ld + n * 8);
      mma16(acc[n], ar, br[0], br[1]);
      mma16(acc[n + 1], ar, br[2], br[3]);
    }
  }
}
template <int KT, int DP>
__device__ __forceinline__ void mma_acc(float (&acc)[DP / 8][4], const float (&p)[KT][4], const float *v, int lane) {
  constexpr int ld = kLd<float, DP>;
  const int g = lane >> 2, t = lane & 3;
  const float *vp = v + 2 * t * ld + g;
#pragma unroll
  for (int n0 = 0; n0 < DP / 8; n0 += 4) {
    float main[4][4], small[4][4];
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) main[n][e] = small[n][e] = 0.f;
#pragma unroll
    for (int kk = 0; kk < KT; ++kk) {
      uint32_t ah[4], al[4], bh[4][2], bl[4][2];
      split_tf32(p[kk][0], ah[0], al[0]);
      split_tf32(p[kk][2], ah[1], al[1]);
      split_tf32(p[kk][1], ah[2], al[2]);
      split_tf32(p[kk][3], ah[3], al[3]);
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) split_tf32(vp[(kk * 8 + e) * ld + (n0 + n) * 8], bh[n][e], bl[n][e]);
#pragma unroll
      for (int n = 0; n < 4; ++n) mma8(small[n], al, bh[n]);
#pragma unroll
      for (int n = 0; n < 4; ++n) mma8(main[n], ah, bh[n]);
#pragma unroll
      for (int n = 0; n < 4; ++n) mma8(small[n], ah, bl[n]);
    }
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[n0 + n][e] += main[n][e] + small[n][e];
  }
}

// CTA index -> (tile, head, sample): samples that share a bias are neighbours
// (their bias block is read from HBM once), then the tiles of one head.
__device__ __forceinline__ void decode_cta(const Args &a, int64_t x, int tiles, int heads, int &tile, int &h, int &b) {
  const int s = int(x % a.share);
  x /= a.share;
  tile = int(x % tiles);
  x /= tiles;
  h = int(x % heads);
  b = int(x / heads) * a.share + s;
}

// Zero the shared rows of left-out keys: whatever the caller keeps there
// (infinities and NaN included) must not meet a zero weight in a product.
template <typename T, int DP, int kRows>
__device__ __forceinline__ void clear_left_out(T *rows, const float *mk, int tid, int threads) {
  constexpr int kChunks = DP / Type<T>::kVec;
  for (int u = tid; u < kRows * kChunks; u += threads)
    if (mk[u / kChunks] == -INFINITY)
      *reinterpret_cast<uint4 *>(rows + (u / kChunks) * kLd<T, DP> + u % kChunks * Type<T>::kVec) =
          make_uint4(0u, 0u, 0u, 0u);
}

// CTAs of a cluster that divide `tiles` key tiles, two or more each, where `ctas` clusters leave SMs without
// two CTAs (128 threads or fewer each).
inline int key_split(int64_t ctas, int64_t tiles) {
  const int64_t room = ctas > 0 ? 2 * int64_t(num_sms()) / ctas : 1, most = room < tiles / 2 ? room : tiles / 2;
  return most < 1 ? 1 : most > 8 ? 8 : int(most);
}
template <typename K, typename... A>
cudaError_t launch_clusters(K kernel, int64_t ctas, int split, int threads, size_t smem, cudaStream_t stream, A... args) {
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(unsigned(ctas * split)), config.blockDim = dim3(unsigned(threads));
  config.dynamicSmemBytes = smem, config.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(split), attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
  config.attrs = attr, config.numAttrs = split > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&config, kernel, args...);
}
// Four fp32 values to a row of the type.
__device__ __forceinline__ void store4(float *p, const float (&v)[4]) { *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]); }
__device__ __forceinline__ void store4(__nv_bfloat16 *p, const float (&v)[4]) {
  *reinterpret_cast<uint2 *>(p) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
}

// cross_attention.cu
Args make_args(const bl_cross_attention_args *x);
int check(const char *name, const Args &a, int64_t kv_heads, int dtype);
// cross_attention_tc.cu
int forward_tc(const Args &a, cudaStream_t stream, bool *taken);

}  // namespace xa
}  // namespace bl
