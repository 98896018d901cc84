// Cross attention to states of another length, forward (see cross_attention.cuh).
//
// flash_kernel: one CTA = up to 64 query rows of one (sample, head), 16 per
// warp; key tiles of kBN stream through a two-stage cp.async ring (K, V, the
// bias block in bf16) while the previous tile is computed; running maximum and sum in
// fp32 registers; the [Nq, Nk] scores never exist in memory.  Few CTAs become clusters
// that divide the keys.  640 fp32 windows of 32 x 128, 4 heads of 32: 59 us (floor 19 us: 124 MB);
// bound by the issue of the split products and their latency at 18 warps per SM.
#include <array>

#include "cross_attention.cuh"

namespace bl {
namespace xa {
namespace {

template <typename T, int DP> constexpr int kBN = sizeof(T) == 4 ? 32 : 64;

template <typename T, int DP> struct FlashSmem {
  static constexpr int bn = kBN<T, DP>, ld = kLd<T, DP>;
  static size_t bytes(int rows, bool bias) {
    return size_t(rows) * ld * sizeof(T) + 2 * (2 * bn * ld * sizeof(T) + bn * 4) +
           (bias && sizeof(T) == 2 ? 2 * size_t(rows) * (bn + 8) * sizeof(T) : 0);
  }
};

template <int DP> constexpr int kPartLd = DP + 4;

// Joins the parts of a cluster's CTAs in the order of their keys: a thread takes four columns of a row at a time.
template <typename T, int DP>
__device__ __forceinline__ void join_parts(const Args &a, const float *part, const float *stat, int rows, int split, int rank,
                                           int i0, int h, int b) {
  for (int u = rank * blockDim.x + threadIdx.x; u < rows * (DP / 4); u += split * blockDim.x) {
    const int row = u / (DP / 4), c = u % (DP / 4) * 4, i = i0 + row;
    if (i >= a.nq || c >= a.d) continue;
    float top = -INFINITY, l = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
    for (int e = 0; e < split; ++e) top = fmaxf(top, peer(stat + row, uint32_t(e)));
    for (int e = 0; e < split; ++e) {
      const float m = peer(stat + row, uint32_t(e));
      if (m == -INFINITY) continue;
      const float weight = fast_exp2((m - top) * kLog2e);
      l = fmaf(weight, peer(stat + rows + row, uint32_t(e)), l);
      const float4 v = peer4(reinterpret_cast<const float4 *>(part + row * kPartLd<DP> + c), uint32_t(e));
      x[0] = fmaf(weight, v.x, x[0]), x[1] = fmaf(weight, v.y, x[1]);
      x[2] = fmaf(weight, v.z, x[2]), x[3] = fmaf(weight, v.w, x[3]);
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int64_t at = ((int64_t(b) * a.nq + i) * a.heads + h) * a.d + c;
    const T *gr = a.gate.p ? static_cast<const T *>(a.gate.p) + b * a.gate.sb + i * a.gate.si + h * a.gate.sh + c : nullptr;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[e] *= inv;
      if (gr) x[e] *= 1.f / (1.f + expf(-load_as_float(gr + e)));
    }
    store4(static_cast<T *>(a.out) + at, x);
    if constexpr (sizeof(T) == 2)
      if (a.low) {
        const float y[4] = {x[0] - bf16r(x[0]), x[1] - bf16r(x[1]), x[2] - bf16r(x[2]), x[3] - bf16r(x[3])};
        store4(static_cast<T *>(a.low) + at, y);
      }
    if (a.lse && c == 0) {
      float *st = a.lse + (int64_t(b) * a.heads + h) * a.nq + i;
      st[0] = l == 0.f ? -INFINITY : top;
      st[a.lse_plane()] = l == 0.f ? 0.f : logf(l);
    }
  }
}

// kSplit: as a cluster of `split` CTAs.  (A variant of its own: its registers cost the other 5 to 10 %.)
template <typename T, int DP, bool kSplit> __global__ void __launch_bounds__(128) flash_kernel(const Args a, int tiles, int clusters) {
  constexpr int BN = kBN<T, DP>, NT = BN / 8, ld = kLd<T, DP>, ND = DP / 8;
  extern __shared__ float4 smem4[];
  const int threads = blockDim.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rows = threads / 2;  // 16 per warp
  T *qs = reinterpret_cast<T *>(smem4);
  T *ks = qs + rows * ld, *vs = ks + 2 * BN * ld;
  float *mks = reinterpret_cast<float *>(vs + 2 * BN * ld);
  T *bs = reinterpret_cast<T *>(mks + 2 * BN);
  int tile, h, b;
  const int split = kSplit ? clusters : 1, rank = kSplit ? int(blockIdx.x) % split : 0;
  decode_cta(a, blockIdx.x / split, tiles, a.heads, tile, h, b);
  const int i0 = tile * rows, hk = h / a.group;
  const T *q = static_cast<const T *>(a.q.p) + b * a.q.sb + h * a.q.sh;
  const T *k = static_cast<const T *>(a.k.p) + b * a.k.sb + hk * a.k.sh;
  const T *v = static_cast<const T *>(a.v.p) + b * a.v.sb + hk * a.v.sh;
  const T *bias = a.bias ? static_cast<const T *>(a.bias) + (b / a.share) * a.bias_sb + h * a.bias_sh : nullptr;

  auto load = [&](int j, int buf) {
    load_rows<T, DP, BN>(ks + buf * BN * ld, k, a.k.si, j * BN, a.nk, a.d, tid, threads);
    load_rows<T, DP, BN>(vs + buf * BN * ld, v, a.v.si, j * BN, a.nk, a.d, tid, threads);
    if (sizeof(T) == 2 && bias) load_bias<T, BN>(bs + buf * rows * (BN + 8), bias, a, i0, rows, j * BN, tid, threads);
    cp_commit();
  };
  for (int u = tid; u < rows * (DP / Type<T>::kVec); u += threads) {
    const int r = u / (DP / Type<T>::kVec), c = u % (DP / Type<T>::kVec) * Type<T>::kVec;
    const bool ok = i0 + r < a.nq && c < a.d;
    cp16(qs + r * ld + c, ok ? q + int64_t(i0 + r) * a.q.si + c : q, ok ? 16 : 0);
  }
  // Key tiles [first, n_tiles).
  const int all_tiles = (a.nk + BN - 1) / BN, first = int(int64_t(rank) * all_tiles / split);
  const int n_tiles = int(int64_t(rank + 1) * all_tiles / split);
  if (n_tiles > first) load(first, 0);
  // mk of a tile: read into registers a tile ahead, put into shared memory after that tile's products.
  float mv[2];
  bool odd = false;
  auto get_mask = [&](int j) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int u = tid + e * threads;
      mv[e] = u < BN ? mask_value(a, b, j * BN + u) : 0.f;
    }
  };
  auto put_mask = [&](int buf) {
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (tid + e * threads < BN) mks[buf * BN + tid + e * threads] = mv[e];
    odd = mv[0] != 0.f || mv[1] != 0.f;
  };
  get_mask(first);
  put_mask(0);

  const int g = lane >> 2, t = lane & 3;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  float o[ND][4];
#pragma unroll
  for (int n = 0; n < ND; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;

  // fp32 bias: straight into registers (the staged blocks left room for 6 CTAs of 64 threads per SM, not 9).
  float2 bv[sizeof(T) == 4 ? NT : 1][2];
  for (int j = first; j < n_tiles; ++j) {
    const int buf = (j - first) & 1;
    if constexpr (sizeof(T) == 4)
      if (bias) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int i = i0 + warp * 16 + g + 8 * r;
          const float *br = bias + int64_t(i) * a.bias_si + j * BN + 2 * t;
#pragma unroll
          for (int n = 0; n < NT; ++n) bv[n][r] = bias_pair(a, br + n * 8, i < a.nq ? a.nk - j * BN - n * 8 - 2 * t : 0);
        }
      }
    if (j + 1 < n_tiles) {
      load(j + 1, buf ^ 1);
      cp_wait<1>();
    } else {
      cp_wait<0>();
    }
    const bool masked = __syncthreads_or(odd);
    if (j + 1 < n_tiles) get_mask(j + 1);
    const float *mk = mks + buf * BN;
    T *vt = vs + buf * BN * ld;
    if (masked && a.mask_kind == kMaskKeep) {
      if (__syncthreads_and((tid >= BN || mk[tid] == -INFINITY) && (tid + threads >= BN || mk[tid + threads] == -INFINITY))) {
        if (j + 1 < n_tiles) put_mask(buf ^ 1);
        continue;  // every key of the tile is left out
      }
      clear_left_out<T, DP, BN>(vt, mk, tid, threads);
      __syncthreads();
    }
    if (i0 + warp * 16 < a.nq) {
      float s[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
      mma_rows<NT, DP>(s, qs + warp * 16 * ld, ks + buf * BN * ld, lane);
      const T *br = bs + buf * rows * (BN + 8) + (warp * 16 + g) * (BN + 8) + 2 * t;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float2 b0 = make_float2(0.f, 0.f), b1 = b0;
        if constexpr (sizeof(T) == 4) {
          if (bias) b0 = bv[n][0], b1 = bv[n][1];
        } else {
          if (bias) b0 = load2(br + n * 8), b1 = load2(br + 8 * (BN + 8) + n * 8);
        }
        s[n][0] = fmaf(s[n][0], a.scale, b0.x), s[n][1] = fmaf(s[n][1], a.scale, b0.y);
        s[n][2] = fmaf(s[n][2], a.scale, b1.x), s[n][3] = fmaf(s[n][3], a.scale, b1.y);
        if (masked) {
          const float2 mv = load2(mk + n * 8 + 2 * t);
          s[n][0] = mv.x == -INFINITY ? mv.x : s[n][0] + mv.x, s[n][1] = mv.y == -INFINITY ? mv.y : s[n][1] + mv.y;
          s[n][2] = mv.x == -INFINITY ? mv.x : s[n][2] + mv.x, s[n][3] = mv.y == -INFINITY ? mv.y : s[n][3] + mv.y;
        }
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float mx = m[r];
#pragma unroll
        for (int n = 0; n < NT; ++n) mx = fmaxf(mx, fmaxf(s[n][2 * r], s[n][2 * r + 1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        // Subtract first, then change base: a mask of the type's lowest value stays finite.
        const float base = mx == -INFINITY ? 0.f : mx;
        const float alpha = fast_exp2((m[r] - base) * kLog2e);
        m[r] = mx;
        float sum = 0.f;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float p = fast_exp2((s[n][2 * r + e] - base) * kLog2e);
            s[n][2 * r + e] = p;
            sum += p;
          }
        l[r] = fmaf(l[r], alpha, sum);
#pragma unroll
        for (int n = 0; n < ND; ++n) o[n][2 * r] *= alpha, o[n][2 * r + 1] *= alpha;
      }
      mma_acc<NT, DP>(o, s, vt, lane);
    }
    if (j + 1 < n_tiles) put_mask(buf ^ 1);
    __syncthreads();
  }

  cp_wait_all();
  T *out = static_cast<T *>(a.out);
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
  }
  if constexpr (kSplit) {  // the cluster's parts, through shared memory
    float *part = reinterpret_cast<float *>(smem4), *stat = part + rows * kPartLd<DP>;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = warp * 16 + g + 8 * r;
#pragma unroll
      for (int n = 0; n < ND; ++n) store2(part + row * kPartLd<DP> + n * 8 + 2 * t, o[n][2 * r], o[n][2 * r + 1]);
      if (t == 0) stat[row] = l[r] == 0.f ? -INFINITY : m[r], stat[rows + row] = l[r];
    }
    cluster_barrier();
    join_parts<T, DP>(a, part, stat, rows, split, rank, i0, h, b);
    cluster_barrier();  // until every part has been read
    return;
  }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int i = i0 + warp * 16 + g + 8 * r;
    if (i >= a.nq) continue;
    const float inv = l[r] == 0.f ? 0.f : 1.f / l[r];
    const int64_t at = ((int64_t(b) * a.nq + i) * a.heads + h) * a.d;
    const T *gr = a.gate.p ? static_cast<const T *>(a.gate.p) + b * a.gate.sb + i * a.gate.si + h * a.gate.sh : nullptr;
#pragma unroll
    for (int n = 0; n < ND; ++n) {
      const int c = n * 8 + 2 * t;
      if (c >= a.d) continue;
      float x = o[n][2 * r] * inv, y = o[n][2 * r + 1] * inv;
      if (gr) {
        const float2 gv = load2(gr + c);
        x *= 1.f / (1.f + expf(-gv.x)), y *= 1.f / (1.f + expf(-gv.y));
      }
      store2(out + at + c, x, y);
      if constexpr (sizeof(T) == 2)
        if (a.low) store2(static_cast<T *>(a.low) + at + c, x - bf16r(x), y - bf16r(y));
    }
    if (a.lse && t == 0) {
      float *st = a.lse + (int64_t(b) * a.heads + h) * a.nq + i;
      st[0] = l[r] == 0.f ? -INFINITY : m[r];
      st[a.lse_plane()] = l[r] == 0.f ? 0.f : logf(l[r]);
    }
  }
}

template <typename T, int DP> int launch_flash(const Args &a, cudaStream_t stream) {
  const int warps = a.nq >= 64 ? 4 : (a.nq + 15) / 16, rows = 16 * warps;
  const int64_t tiles = (a.nq + rows - 1) / rows, ctas = tiles * a.heads * a.batch;
  BL_REQUIRE(ctas < (int64_t(1) << 31), "bl_cross_attention: too many query tiles");
  const size_t smem = FlashSmem<T, DP>::bytes(rows, a.bias != nullptr);
  // Few CTAs: a cluster divides the keys.
  const int split = key_split(ctas, (a.nk + kBN<T, DP> - 1) / kBN<T, DP>);
  auto kernel = split > 1 ? flash_kernel<T, DP, true> : flash_kernel<T, DP, false>;
  BL_CUDA(ensure_smem_limit(reinterpret_cast<const void *>(kernel), 232448));
  BL_CUDA(launch_clusters(kernel, ctas, split, 32 * warps, smem, stream, a, int(tiles), split));
  BL_LAUNCH_CHECK();
  return BL_OK;
}

// ---------------------------------------------------------------------------
// Few query rows (the serving step): one CTA, or a cluster of `split` CTAs, per
// (sample, key/value head).  The nq * group rows that read the same keys form
// one 16-row tile; each warp takes every fourth chunk of kKC keys through a
// ring of its own (no CTA barrier in the loop) and keeps its own maximum, sum
// and output.  The warps' parts are merged in shared memory, the CTAs' parts
// through distributed shared memory: one launch, no workspace, fixed order.
// Bound by reading K and V once: 84 MB (5 samples, 16 heads on 4, 16384 keys of 64) in 25 us,
// 3.3 TB/s; clusters of 6 cover 120 of the 148 SMs, and a call of a few us ends before HBM is at its rate.
// ---------------------------------------------------------------------------
constexpr int kStepRows = 16;

template <typename T, int DP> struct Step {
  // Eight warps (two per scheduler: a chunk is a chain of some 600 instructions) with two
  // chunks each in flight; wide rows leave room for four warps with three.
  static constexpr int warps = DP == 128 ? 4 : 8, stages = DP == 128 ? 3 : 2;
  static constexpr int kc = (sizeof(T) == 4 && DP >= 64) ? 16 : 32, ld = kLd<T, DP>;
  static constexpr int kv = kc * ld;              // elements of a K or V chunk
  static constexpr int bias = kStepRows * (kc + 8);
  static constexpr int stage_bytes = (2 * kv + bias) * int(sizeof(T)) + kc * 4;
  static constexpr int q_bytes = kStepRows * ld * int(sizeof(T));
  static constexpr int ring_bytes = warps * stages * stage_bytes;
  static constexpr int part_bytes = (warps * kStepRows * (DP + 2) + 2 * kStepRows) * 4;
  static constexpr int bits_off = q_bytes + (ring_bytes > part_bytes ? ring_bytes : part_bytes);
  // Keep mask of the CTA's keys as bits, where it fits.
  static constexpr int mask_words = (232448 - bits_off) / 4 < 2048 ? (232448 - bits_off) / 4 : 2048;
  static constexpr int bytes = bits_off + mask_words * 4;
};

template <typename T, int DP>
__global__ void __launch_bounds__(32 * Step<T, DP>::warps) step_kernel(const Args a, int split) {
  using S = Step<T, DP>;
  constexpr int kStepWarps = S::warps, kStepStages = S::stages;
  constexpr int KC = S::kc, NT = KC / 8, ld = S::ld, ND = DP / 8, kVec = Type<T>::kVec, kChunks = DP / kVec;
  extern __shared__ float4 smem4[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  T *qs = reinterpret_cast<T *>(smem4);
  char *ring = reinterpret_cast<char *>(smem4) + S::q_bytes;
  char *mine = ring + warp * kStepStages * S::stage_bytes;
  const int kv_heads = a.heads / a.group, rank = int(blockIdx.x) % split, bh = int(blockIdx.x) / split;
  const int b = bh / kv_heads, hk = bh % kv_heads, rows = a.nq * a.group;
  const T *q = static_cast<const T *>(a.q.p) + b * a.q.sb + hk * a.group * a.q.sh;
  const T *k = static_cast<const T *>(a.k.p) + b * a.k.sb + hk * a.k.sh;
  const T *v = static_cast<const T *>(a.v.p) + b * a.v.sb + hk * a.v.sh;
  const T *bias = a.bias ? static_cast<const T *>(a.bias) + (b / a.share) * a.bias_sb + hk * a.group * a.bias_sh : nullptr;
  for (int u = tid; u < kStepRows * kChunks; u += 32 * kStepWarps) {
    const int r = u / kChunks, c = u % kChunks * kVec;
    const bool ok = r < rows && c < a.d;
    cp16(qs + r * ld + c, ok ? q + r / a.group * a.q.si + r % a.group * a.q.sh + c : q, ok ? 16 : 0);
  }
  cp_commit();
  const int64_t chunks = (a.nk + KC - 1) / KC;
  const int c_begin = int(rank * chunks / split), c_end = int((rank + 1) * chunks / split);
  // The mask decides which rows are loaded, so it has to be there ahead of them: read chunk by chunk it cost
  // 6 of 29 us at 5 samples of 16384 keys.
  uint32_t *bits = reinterpret_cast<uint32_t *>(reinterpret_cast<char *>(smem4) + S::bits_off);
  const int w0 = int(int64_t(c_begin) * KC / 32), words = int((int64_t(c_end) * KC + 31) / 32) - w0;
  const bool use_bits = a.mask_kind == kMaskKeep && words <= S::mask_words;
  int next = c_begin + warp;  // chunk to issue
  float mk_next = lane < KC && next < c_end ? mask_value(a, b, next * KC + lane) : -INFINITY;
  int put = 0;
  // Keys that are left out are not loaded: their rows are zero whatever they hold.
  auto issue = [&](bool first) {
    if (next < c_end) {
      char *st = mine + put * S::stage_bytes;
      T *kt = reinterpret_cast<T *>(st), *vt = kt + S::kv, *bt = vt + S::kv;
      float *mk = reinterpret_cast<float *>(bt + S::bias);
      const int j0 = next * KC;
      if (use_bits && !first) {
        const int j = next * KC;
        mk_next = bits[(j >> 5) - w0] >> ((j & 31) + (lane & (KC - 1))) & 1 ? -INFINITY : 0.f;
      }
      if (lane < KC) mk[lane] = mk_next;
      // Lane: chunk c of rows r0, r0 + kStep, ...
      constexpr int kStep = 32 / kChunks > 0 ? 32 / kChunks : 1;
      const int r0 = lane / kChunks, c = lane % kChunks * kVec;
      const uint32_t gone = __ballot_sync(0xffffffffu, mk_next == -INFINITY);
      const T *kp = k + int64_t(j0 + r0) * a.k.si + c, *vp = v + int64_t(j0 + r0) * a.v.si + c;
      const int64_t k_step = kStep * a.k.si, v_step = kStep * a.v.si;
#pragma unroll 4
      for (int r = r0; r < KC; r += kStep, kp += k_step, vp += v_step) {
        const bool ok = (gone >> r & 1) == 0 && c < a.d;
        cp16(kt + r * ld + c, ok ? kp : k, ok ? 16 : 0);
        cp16(vt + r * ld + c, ok ? vp : v, ok ? 16 : 0);
      }
      if (bias) {
        for (int u = lane; u < rows * (KC / kVec); u += 32) {
          const int r = u / (KC / kVec), c = u % (KC / kVec) * kVec, left = a.nk - j0 - c;
          const T *src = bias + int64_t(r / a.group) * a.bias_si + r % a.group * a.bias_sh + j0 + c;
          T *dst = bt + r * (KC + 8) + c;
          if (a.bias_vec) {
            const int bytes = left > 0 ? (left < kVec ? left * int(sizeof(T)) : 16) : 0;
            cp16(dst, bytes ? src : bias, bytes);
          } else {
#pragma unroll
            for (int e = 0; e < kVec; ++e) dst[e] = e < left ? src[e] : T(0.f);
          }
        }
      }
      next += kStepWarps;
      if (!use_bits || first) mk_next = lane < KC && next < c_end ? mask_value(a, b, next * KC + lane) : -INFINITY;
    }
    cp_commit();
    put = put + 1 == kStepStages ? 0 : put + 1;
  };
#pragma unroll
  for (int e = 0; e < kStepStages - 1; ++e) issue(true);
  if (use_bits)
    for (int w = tid; w < words; w += 32 * kStepWarps) bits[w] = mask_word(a, b, w0 + w);
  cp_wait<kStepStages - 1>();
  __syncthreads();  // Q and the mask

  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[ND][4];
#pragma unroll
  for (int n = 0; n < ND; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
  int take = 0;
  for (int c = c_begin + warp; c < c_end; c += kStepWarps) {
    issue(false);
    cp_wait<kStepStages - 1>();
    __syncwarp();
    const char *st = mine + take * S::stage_bytes;
    const T *kt = reinterpret_cast<const T *>(st), *vt = kt + S::kv, *bt = vt + S::kv;
    const float *mk = reinterpret_cast<const float *>(bt + S::bias);
    take = take + 1 == kStepStages ? 0 : take + 1;
    if (__any_sync(0xffffffffu, lane < KC && mk[lane & (KC - 1)] != -INFINITY)) {
      float s[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
      mma_rows<NT, DP>(s, qs, kt, lane);
      const T *br = bt + g * (KC + 8) + 2 * t;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float2 b0 = make_float2(0.f, 0.f), b1 = b0;
        if (bias) {
          if (g < rows) b0 = load2(br + n * 8);
          if (g + 8 < rows) b1 = load2(br + 8 * (KC + 8) + n * 8);
        }
        const float2 mv = load2(mk + n * 8 + 2 * t);
        s[n][0] = mv.x == -INFINITY ? mv.x : fmaf(s[n][0], a.scale, b0.x) + mv.x;
        s[n][1] = mv.y == -INFINITY ? mv.y : fmaf(s[n][1], a.scale, b0.y) + mv.y;
        s[n][2] = mv.x == -INFINITY ? mv.x : fmaf(s[n][2], a.scale, b1.x) + mv.x;
        s[n][3] = mv.y == -INFINITY ? mv.y : fmaf(s[n][3], a.scale, b1.y) + mv.y;
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float mx = m[r];
#pragma unroll
        for (int n = 0; n < NT; ++n) mx = fmaxf(mx, fmaxf(s[n][2 * r], s[n][2 * r + 1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float base = mx == -INFINITY ? 0.f : mx;
        const float alpha = fast_exp2((m[r] - base) * kLog2e);
        m[r] = mx;
        float sum = 0.f;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            s[n][2 * r + e] = fast_exp2((s[n][2 * r + e] - base) * kLog2e);
            sum += s[n][2 * r + e];
          }
        l[r] = fmaf(l[r], alpha, sum);
        if (__any_sync(0xffffffffu, alpha != 1.f))
#pragma unroll
          for (int n = 0; n < ND; ++n) o[n][2 * r] *= alpha, o[n][2 * r + 1] *= alpha;
      }
      mma_acc<NT, DP>(o, s, vt, lane);
    }
    __syncwarp();
  }
  cp_wait_all();
  __syncthreads();  // the ring is free: the warps' parts go there
  float *po = reinterpret_cast<float *>(ring);              // [warp][row][DP]
  float *pm = po + kStepWarps * kStepRows * DP;             // [warp][row]
  float *pl = pm + kStepWarps * kStepRows;                  // [warp][row]
  float *cm = pl + kStepWarps * kStepRows, *cl = cm + kStepRows;  // the CTA's
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    const int at = warp * kStepRows + g + 8 * r;
    if (t == 0) pm[at] = m[r], pl[at] = l[r];
#pragma unroll
    for (int n = 0; n < ND; ++n) store2(po + at * DP + n * 8 + 2 * t, o[n][2 * r], o[n][2 * r + 1]);
  }
  __syncthreads();
  for (int u = tid; u < rows * DP; u += 32 * kStepWarps) {
    const int r = u / DP;
    float mx = pm[r];
#pragma unroll
    for (int w = 1; w < kStepWarps; ++w) mx = fmaxf(mx, pm[w * kStepRows + r]);
    const float base = mx == -INFINITY ? 0.f : mx;
    float sum = 0.f, x = 0.f;
#pragma unroll
    for (int w = 0; w < kStepWarps; ++w) {
      const float f = fast_exp2((pm[w * kStepRows + r] - base) * kLog2e);
      sum = fmaf(pl[w * kStepRows + r], f, sum);
      x = fmaf(po[w * kStepRows * DP + u], f, x);
    }
    po[u] = x;  // this element of the other warps' parts is read by this thread alone
    if (u % DP == 0) cm[r] = mx, cl[r] = sum;
  }
  if (split > 1) cluster_barrier(); else __syncthreads();
  T *out = static_cast<T *>(a.out);
  const int pairs = rows * (a.d / 2);
  const int u_end = (rank + 1) * pairs / split;
  for (int u = rank * pairs / split + tid; u < u_end; u += 32 * kStepWarps) {
    const int r = u / (a.d / 2), c = 2 * (u % (a.d / 2));
    float mx = -INFINITY, sum = 0.f, x = 0.f, y = 0.f;
    if (split > 1) {
      for (int p = 0; p < split; ++p) mx = fmaxf(mx, peer(cm + r, p));
      const float base = mx == -INFINITY ? 0.f : mx;
#pragma unroll 4
      for (int p = 0; p < split; ++p) {
        const float f = fast_exp2((peer(cm + r, p) - base) * kLog2e);
        sum = fmaf(peer(cl + r, p), f, sum);
        x = fmaf(peer(po + r * DP + c, p), f, x);
        y = fmaf(peer(po + r * DP + c + 1, p), f, y);
      }
    } else {
      mx = cm[r], sum = cl[r], x = po[r * DP + c], y = po[r * DP + c + 1];
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    x *= inv, y *= inv;
    const int i = r / a.group, h = hk * a.group + r % a.group;
    if (a.gate.p) {
      const float2 gv = load2(static_cast<const T *>(a.gate.p) + b * a.gate.sb + i * a.gate.si + h * a.gate.sh + c);
      x *= 1.f / (1.f + expf(-gv.x)), y *= 1.f / (1.f + expf(-gv.y));
    }
    const int64_t at = ((int64_t(b) * a.nq + i) * a.heads + h) * a.d + c;
    store2(out + at, x, y);
    if constexpr (sizeof(T) == 2)
      if (a.low) store2(static_cast<T *>(a.low) + at, x - bf16r(x), y - bf16r(y));
    if (a.lse && c == 0) {
      float *st = a.lse + (int64_t(b) * a.heads + h) * a.nq + i;
      st[0] = sum == 0.f ? -INFINITY : mx;
      st[a.lse_plane()] = sum == 0.f ? 0.f : logf(sum);
    }
  }
  if (split > 1) cluster_barrier();  // peers may still be reading this CTA's parts
}

// Clusters of s CTAs that the device holds at once (1 / s of its SMs where the query fails; asked of the first device in
// use: only the choice of a split hangs on it).
template <typename T, int DP> int active_clusters(int s) {
  using S = Step<T, DP>;
  static const std::array<int, 9> table = [] {
    std::array<int, 9> t{};
    for (int e = 1; e <= 8; ++e) {
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = unsigned(e), attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
      cudaLaunchConfig_t config = {};
      config.gridDim = dim3(unsigned(e)), config.blockDim = dim3(32 * S::warps), config.dynamicSmemBytes = S::bytes;
      config.attrs = attr, config.numAttrs = 1;
      int n = 0;
      if (cudaOccupancyMaxActiveClusters(&n, step_kernel<T, DP>, &config) != cudaSuccess || n < 1) {
        cudaGetLastError();
        n = num_sms() / e;
      }
      t[e] = n < 1 ? 1 : n;
    }
    return t;
  }();
  return table[s];
}

template <typename T, int DP> int launch_step(const Args &a, cudaStream_t stream) {
  using S = Step<T, DP>;
  static_assert(S::bytes <= 232448, "shared memory");
  const int64_t slabs = int64_t(a.batch) * (a.heads / a.group);
  BL_CUDA(ensure_smem_limit(reinterpret_cast<const void *>(step_kernel<T, DP>), S::bytes));
  // The split with the fewest waves per CTA's share of the keys, at least one chunk per warp.  (At 20 slabs a fixed split
  // of eight takes two waves: it took 62 us where six took 31, which later steps brought to 25.)
  int split = 1;
  double best = 0.;
  for (int e = 1; e <= 8 && (e == 1 || a.nk >= int64_t(e) * S::warps * S::kc); ++e) {
    const int64_t waves = (slabs + active_clusters<T, DP>(e) - 1) / active_clusters<T, DP>(e);
    const double cost = double(waves) / e + 0.02 * (e > 1);  // a cluster's merge costs a little
    if (e == 1 || cost < best) best = cost, split = e;
  }
  BL_REQUIRE(slabs * split < (int64_t(1) << 31), "bl_cross_attention: too many samples");
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(unsigned(slabs * split));
  config.blockDim = dim3(32 * S::warps);
  config.dynamicSmemBytes = S::bytes;
  config.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(split);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  config.attrs = attr;
  config.numAttrs = split > 1 ? 1 : 0;
  BL_CUDA(cudaLaunchKernelEx(&config, step_kernel<T, DP>, a, split));
  BL_LAUNCH_CHECK();
  return BL_OK;
}

template <typename T> int forward(const Args &a, cudaStream_t stream) {
  if (int64_t(a.nq) * a.group <= kStepRows) {
    if (a.d <= 32) return launch_step<T, 32>(a, stream);
    if (a.d <= 64) return launch_step<T, 64>(a, stream);
    return launch_step<T, 128>(a, stream);
  }
  if (sizeof(T) == 2) {
    bool taken = false;
    if (int rc = forward_tc(a, stream, &taken)) return rc;
    if (taken) return BL_OK;
  }
  if (a.d <= 32) return launch_flash<T, 32>(a, stream);
  if (a.d <= 64) return launch_flash<T, 64>(a, stream);
  return launch_flash<T, 128>(a, stream);
}

bool rows_ok(const Rows &r, int vec) {
  return aligned_to(r.p, 16) && r.sb % vec == 0 && r.si % vec == 0 && r.sh % vec == 0;
}

}  // namespace

int check(const char *name, const Args &a, int64_t kv_heads, int dtype) {
  BL_REQUIRE(dtype == BL_F32 || dtype == BL_BF16, "%s: dtype must be fp32 or bf16", name);
  BL_REQUIRE(a.batch >= 0 && a.nq >= 0 && a.nk >= 0 && a.heads >= 1 && kv_heads >= 1, "%s: bad shape", name);
  BL_REQUIRE(a.heads % kv_heads == 0, "%s: key/value heads must divide the query heads", name);
  BL_REQUIRE(a.d >= 8 && a.d <= 128 && a.d % 8 == 0, "%s: head_dim must be a multiple of 8, at most 128", name);
  BL_REQUIRE(a.share >= 1 && a.batch % a.share == 0, "%s: the samples per bias must divide the batch", name);
  BL_REQUIRE(a.mask_kind >= kMaskNone && a.mask_kind <= kMaskAdd, "%s: unknown mask kind", name);
  const int vec = dtype == BL_F32 ? 4 : 8;
  if (a.batch == 0 || a.nq == 0) return BL_OK;
  BL_REQUIRE(a.q.p && a.out && (a.nk == 0 || (a.k.p && a.v.p)), "%s: null pointer", name);
  BL_REQUIRE(a.mask_kind == kMaskNone || a.mask || a.nk == 0, "%s: the mask is missing", name);
  BL_REQUIRE(rows_ok(a.q, vec) && rows_ok(a.k, vec) && rows_ok(a.v, vec) && rows_ok(a.gate, vec) && aligned_to(a.out, 16) &&
                 aligned_to(a.low, 16),
             "%s: q, k, v, gate and out rows must start on 16-byte boundaries", name);
  return BL_OK;
}

Args make_args(const bl_cross_attention_args *x) {
  Args a{};
  const int vec = x->dtype == BL_F32 ? 4 : 8;
  a.q = {x->q, x->q_stride[0], x->q_stride[1], x->q_stride[2]};
  a.k = {x->k, x->k_stride[0], x->k_stride[1], x->k_stride[2]};
  a.v = {x->v, x->v_stride[0], x->v_stride[1], x->v_stride[2]};
  a.gate = {x->gate, x->gate_stride[0], x->gate_stride[1], x->gate_stride[2]};
  a.bias = x->bias;
  a.bias_sb = x->bias_stride[0], a.bias_sh = x->bias_stride[1], a.bias_si = x->bias_stride[2];
  a.bias_vec = aligned_to(x->bias, 16) && a.bias_sb % vec == 0 && a.bias_sh % vec == 0 && a.bias_si % vec == 0;
  a.share = x->bias ? int(x->bias_share) : 1;
  a.mask = x->mask, a.mask_sb = x->mask_stride, a.mask_kind = x->mask_kind;
  a.inf = x->inf, a.scale = x->scale;
  a.batch = int(x->batch), a.heads = int(x->heads), a.nq = int(x->nq), a.nk = int(x->nk), a.d = int(x->head_dim);
  a.group = x->kv_heads > 0 ? int(x->heads / x->kv_heads) : 1;
  a.out = x->out, a.low = x->dtype == BL_BF16 ? x->low : nullptr, a.lse = x->lse;
  return a;
}

}  // namespace xa
}  // namespace bl

using namespace bl;

extern "C" int bl_cross_attention(const bl_cross_attention_args *x, void *stream) {
  BL_REQUIRE(x, "bl_cross_attention: null arguments");
  BL_REQUIRE(x->batch < (1 << 30) && x->heads < (1 << 16) && x->kv_heads < (1 << 16) && x->nq < (1 << 30) &&
                 x->nk < (1 << 30) && x->head_dim < (1 << 16) && x->bias_share < (1 << 30),
             "bl_cross_attention: shape too large");
  const xa::Args a = xa::make_args(x);
  if (int rc = xa::check("bl_cross_attention", a, x->kv_heads, x->dtype)) return rc;
  if (a.batch == 0 || a.nq == 0) return BL_OK;
  return x->dtype == BL_F32 ? xa::forward<float>(a, as_stream(stream)) : xa::forward<__nv_bfloat16>(a, as_stream(stream));
}
