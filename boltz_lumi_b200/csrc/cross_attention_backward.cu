// Cross attention to states of another length, gradients (see cross_attention.cuh).
//
//   do = dy sigmoid(gate),  delta = sum_e do o,  dgate = dy o sigmoid(gate) (1 - sigmoid(gate))
//   p = softmax(x),  ds = p (do . v - delta)
//   dv = sum_i p do,  dk = scale sum_i ds q,  dq = scale sum_j ds k,  dbias = sum over the sharing samples of ds
//
// The scores are recomputed tile by tile and never stored.  Every output has
// one owner, so there are no atomics and the same inputs give the same bits:
//   rows_kernel    one pass over dy and out: delta, do, dgate.  Where one key dominates a
//                  row, do . v and delta cancel, so in bf16 both need more than 8 bits: delta
//                  takes out with the part that its rounding took (`low`), and a gated do
//                  goes into do . v (and dv, whose p is rounded already) as two bf16 terms;
//   keys_kernel    one CTA = 64 keys of one (sample, key/value head): dk and dv,
//                  summed over the query tiles of every head that shares them;
//   queries_kernel one CTA = up to 64 query rows of one (sample, head): dq, and
//                  dbias where no other sample shares the bias;
//   bias_kernel    one CTA = one block of a shared bias: dbias summed over its samples;
//   window_kernel  all four gradients of small fp32 windows at once.
// bf16 goes to cross_attention_backward_tc.cu (measured there) where back_covered says so: 64 keys or more,
// more than 64 queries (or what worth_tiles allows), operands that tensor maps describe, bias rows
// on 16-byte boundaries; a shared bias' gradient also wants d <= 64 (bias_tc).  The rest stays here.  What
// bounds these kernels is the issue of the warp products: in fp32 each is three (tf32 pairs), and a CTA's
// 16-row products read and split every operand tile again (10 x 8 x 96 x 6619 x 48, fp32, one bias
// per five samples: 2.1 ms, 11 TFLOP/s of the formula's products, where the plain form's library products take
// 1.85 ms; 22 x 16 x 33 x 752 x 128: 3 % slower than they).  A shared bias' gradient at d = 128, bf16, 2 x 16 x 384 x
// 1734: 148 us here beside 128 us for the other gradients on tiles (at d = 64 37 beside 108).  Half the tile (16 rows) at d = 128, for two CTAs per SM, was
// faster with few queries (961 -> 783 us) and slower else (1715 -> 1960 us).
#include "cross_attention_backward.cuh"

namespace bl {
namespace xa {
namespace {

// Query rows per tile of keys_kernel and key columns per tile of the others.
template <typename T, int DP> constexpr int kTile = (sizeof(T) == 4 || DP == 128) ? 32 : 64;

// p and ds of one score, given the row's maximum m, -log2 of its sum and delta.  m is
// subtracted before the change of base: in a row of the type's lowest values the sum
// would vanish in m + log(sum).  Left-out keys contribute nothing whatever their operands hold.
__device__ __forceinline__ void grad_score(float &s, float &dp, float scale, float bias, float mk, float m, float nl,
                                           float delta) {
  const bool out = mk == -INFINITY;
  const float x = fmaf(s, scale, bias) + mk;
  const float p = out ? 0.f : fast_exp2(fmaf(x - m, kLog2e, nl));
  s = p;
  dp = out ? 0.f : p * (dp - delta);
}

// Eight lanes per row of d elements.
template <typename T> __global__ void __launch_bounds__(256) rows_kernel(const BackArgs x, int64_t rows) {
  constexpr int kVec = Type<T>::kVec;
  const Args &a = x.a;
  const int64_t r = (int64_t(blockIdx.x) * blockDim.x + threadIdx.x) >> 3;
  const int part = threadIdx.x & 7;
  float sum = 0.f;
  if (r < rows) {
    const int h = int(r % a.heads);
    const int64_t bi = r / a.heads, i = bi % a.nq, b = bi / a.nq;
    const T *dy = static_cast<const T *>(x.dy) + r * a.d, *y = static_cast<const T *>(a.out) + r * a.d;
    const T *low = a.low ? static_cast<const T *>(a.low) + r * a.d : nullptr;
    const T *g = a.gate.p ? static_cast<const T *>(a.gate.p) + b * a.gate.sb + i * a.gate.si + h * a.gate.sh : nullptr;
    T *dout = g ? static_cast<T *>(const_cast<void *>(x.dout)) + r * a.d : nullptr;
    T *dl = x.dlow ? static_cast<T *>(const_cast<void *>(x.dlow)) + r * a.d : nullptr;
    T *dg = g ? static_cast<T *>(x.dgate) + r * a.d : nullptr;
    for (int c = part * kVec; c < a.d; c += 8 * kVec) {
#pragma unroll
      for (int e = 0; e < kVec; e += 2) {
        const float2 u = load2(dy + c + e);
        float2 w = load2(y + c + e);
        if (low) {
          const float2 z = load2(low + c + e);
          w.x += z.x, w.y += z.y;
        }
        if (g) {
          const float2 z = load2(g + c + e);
          const float s0 = 1.f / (1.f + expf(-z.x)), s1 = 1.f / (1.f + expf(-z.y));
          const float d0 = u.x * s0, d1 = u.y * s1;
          store2(dout + c + e, d0, d1);
          if constexpr (sizeof(T) == 2) store2(dl + c + e, d0 - bf16r(d0), d1 - bf16r(d1));
          // do o = dy out; 1 - sigmoid(z) = sigmoid(-z)
          store2(dg + c + e, u.x * w.x * (1.f / (1.f + expf(z.x))), u.y * w.y * (1.f / (1.f + expf(z.y))));
        }
        sum = fmaf(u.x, w.x, fmaf(u.y, w.y, sum));
      }
    }
  }
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (r < rows && part == 0) {
    const int h = int(r % a.heads);
    const int64_t bi = r / a.heads;
    x.delta[((bi / a.nq) * a.heads + h) * a.nq + bi % a.nq] = sum;
  }
}

__device__ __forceinline__ void cp4(float *dst, const float *src, bool ok) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_addr(dst)), "l"(src), "r"(ok ? 4 : 0) : "memory");
}

constexpr int kKeys = 64;

template <typename T, int DP> size_t keys_smem(bool bias, bool low) {
  constexpr int ld = kLd<T, DP>, BQ = kTile<T, DP>;
  return (2 * kKeys * ld + (low ? 6 : 4) * BQ * ld) * sizeof(T) + 6 * BQ * 4 + (bias && sizeof(T) == 2 ? 2 * BQ * (kKeys + 8) * sizeof(T) : 0);
}

template <typename T, int DP> __global__ void __launch_bounds__(128) keys_kernel(const BackArgs x, int tiles) {
  constexpr int BQ = kTile<T, DP>, NT = BQ / 8, ld = kLd<T, DP>, ND = DP / 8, kThreads = 128;
  const Args &a = x.a;
  extern __shared__ float4 smem4[];
  T *ks = reinterpret_cast<T *>(smem4), *vs = ks + kKeys * ld;
  T *qs = vs + kKeys * ld, *ds = qs + 2 * BQ * ld, *dls = ds + 2 * BQ * ld;
  float *ls = reinterpret_cast<float *>(dls + (x.dlow ? 2 * BQ * ld : 0)), *lg = ls + 2 * BQ, *del = lg + 2 * BQ;
  T *bs = reinterpret_cast<T *>(del + 2 * BQ);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int kv_heads = a.heads / a.group;
  int tile, hk, b;
  decode_cta(a, blockIdx.x, tiles, kv_heads, tile, hk, b);
  const int j0 = tile * kKeys;
  const T *k = static_cast<const T *>(a.k.p) + b * a.k.sb + hk * a.k.sh;
  const T *v = static_cast<const T *>(a.v.p) + b * a.v.sb + hk * a.v.sh;
  load_rows<T, DP, kKeys>(ks, k, a.k.si, j0, a.nk, a.d, tid, kThreads);
  load_rows<T, DP, kKeys>(vs, v, a.v.si, j0, a.nk, a.d, tid, kThreads);
  float mk[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) mk[r] = mask_value(a, b, j0 + warp * 16 + g + 8 * r);
  const bool any = __syncthreads_or(mk[0] != -INFINITY || mk[1] != -INFINITY);

  const int q_tiles = (a.nq + BQ - 1) / BQ, steps = any ? q_tiles * a.group : 0;
  auto load = [&](int u, int buf) {
    const int h = hk * a.group + u / q_tiles, i0 = u % q_tiles * BQ;
    const T *q = static_cast<const T *>(a.q.p) + b * a.q.sb + h * a.q.sh;
    const T *d = static_cast<const T *>(x.dout) + (int64_t(b) * a.nq * a.heads + h) * a.d;
    load_rows<T, DP, BQ>(qs + buf * BQ * ld, q, a.q.si, i0, a.nq, a.d, tid, kThreads);
    load_rows<T, DP, BQ>(ds + buf * BQ * ld, d, int64_t(a.heads) * a.d, i0, a.nq, a.d, tid, kThreads);
    if (x.dlow)
      load_rows<T, DP, BQ>(dls + buf * BQ * ld, static_cast<const T *>(x.dlow) + (int64_t(b) * a.nq * a.heads + h) * a.d,
                           int64_t(a.heads) * a.d, i0, a.nq, a.d, tid, kThreads);
    if (tid < BQ) {
      const int64_t at = (int64_t(b) * a.heads + h) * a.nq;
      const bool ok = i0 + tid < a.nq;
      if (ok)
        cp4(ls + buf * BQ + tid, a.lse + at + i0 + tid, true);
      else  // a row past the last: p = 0 whatever the mask adds (0 for its reference made exp(mask term) of it)
        ls[buf * BQ + tid] = -INFINITY;
      cp4(lg + buf * BQ + tid, a.lse + a.lse_plane() + at + (ok ? i0 + tid : 0), ok);
      cp4(del + buf * BQ + tid, x.delta + at + (ok ? i0 + tid : 0), ok);
    }
    if (sizeof(T) == 2 && a.bias) {
      const T *bias = static_cast<const T *>(a.bias) + (b / a.share) * a.bias_sb + h * a.bias_sh;
      load_bias<T, kKeys>(bs + buf * BQ * (kKeys + 8), bias, a, i0, BQ, j0, tid, kThreads);
    }
    cp_commit();
  };
  if (steps > 0) load(0, 0);
  float dk[ND][4], dv[ND][4];
#pragma unroll
  for (int n = 0; n < ND; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) dk[n][e] = dv[n][e] = 0.f;

  // fp32 bias: straight into registers (see flash_kernel).
  float bv[sizeof(T) == 4 ? NT : 1][4];
  for (int u = 0; u < steps; ++u) {
    const int buf = u & 1;
    if constexpr (sizeof(T) == 4)
      if (a.bias) {
        const int h = hk * a.group + u / q_tiles, i0 = u % q_tiles * BQ + 2 * t, j = j0 + warp * 16 + g;
        const T *br = static_cast<const T *>(a.bias) + (b / a.share) * a.bias_sb + h * a.bias_sh + i0 * a.bias_si + j;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            bv[n][e] = i0 + n * 8 + (e & 1) < a.nq && j + (e >> 1) * 8 < a.nk ? br[(n * 8 + (e & 1)) * a.bias_si + (e >> 1) * 8] : 0.f;
      }
    if (u + 1 < steps) {
      load(u + 1, buf ^ 1);
      cp_wait<1>();
    } else {
      cp_wait<0>();
    }
    __syncthreads();
    if (j0 + warp * 16 < a.nk) {
      const T *qt = qs + buf * BQ * ld, *dt = ds + buf * BQ * ld;
      float s[NT][4], dp[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = dp[n][e] = 0.f;
      mma_rows<NT, DP>(s, ks + warp * 16 * ld, qt, lane);
      if (x.dlow) mma_rows<NT, DP>(dp, vs + warp * 16 * ld, dls + buf * BQ * ld, lane);
      mma_rows<NT, DP>(dp, vs + warp * 16 * ld, dt, lane);
      const T *bp = bs + buf * BQ * (kKeys + 8) + 2 * t * (kKeys + 8) + warp * 16 + g;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float2 lv = load2(ls + buf * BQ + n * 8 + 2 * t), dl = load2(del + buf * BQ + n * 8 + 2 * t);
        const float2 ll = load2(lg + buf * BQ + n * 8 + 2 * t);
        const float m0 = row_max(lv.x), m1 = row_max(lv.y), n0 = -kLog2e * ll.x, n1 = -kLog2e * ll.y;
        float bq[4] = {0.f, 0.f, 0.f, 0.f};
        if (a.bias) {
          if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int e = 0; e < 4; ++e) bq[e] = bv[n][e];
          } else {
            const T *p = bp + n * 8 * (kKeys + 8);
            bq[0] = load_as_float(p), bq[1] = load_as_float(p + kKeys + 8);
            bq[2] = load_as_float(p + 8), bq[3] = load_as_float(p + kKeys + 16);
          }
        }
        grad_score(s[n][0], dp[n][0], a.scale, bq[0], mk[0], m0, n0, dl.x);
        grad_score(s[n][1], dp[n][1], a.scale, bq[1], mk[0], m1, n1, dl.y);
        grad_score(s[n][2], dp[n][2], a.scale, bq[2], mk[1], m0, n0, dl.x);
        grad_score(s[n][3], dp[n][3], a.scale, bq[3], mk[1], m1, n1, dl.y);
      }
      if (x.dlow) mma_acc<NT, DP>(dv, s, dls + buf * BQ * ld, lane);
      mma_acc<NT, DP>(dv, s, dt, lane);
      mma_acc<NT, DP>(dk, dp, qt, lane);
    }
    __syncthreads();
  }
  cp_wait_all();
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int j = j0 + warp * 16 + g + 8 * r;
    if (j >= a.nk) continue;
    const int64_t at = ((int64_t(b) * a.nk + j) * kv_heads + hk) * a.d;
#pragma unroll
    for (int n = 0; n < ND; ++n) {
      const int c = n * 8 + 2 * t;
      if (c >= a.d) continue;
      store2(static_cast<T *>(x.dk) + at + c, dk[n][2 * r] * a.scale, dk[n][2 * r + 1] * a.scale);
      store2(static_cast<T *>(x.dv) + at + c, dv[n][2 * r], dv[n][2 * r + 1]);
    }
  }
}

template <typename T, int DP> size_t queries_smem(int rows, bool bias, bool low) {
  constexpr int ld = kLd<T, DP>, BN = kTile<T, DP>;
  return ((low ? 3 : 2) * size_t(rows) * ld + 4 * BN * ld) * sizeof(T) + 2 * BN * 4 + (bias && sizeof(T) == 2 ? 2 * size_t(rows) * (BN + 8) * sizeof(T) : 0);
}

// ds of two neighbouring keys of one row into the bias gradient's row.
template <typename T> __device__ __forceinline__ void store_bias(T *row, int j, int nk, float x, float y) {
  if (j + 1 < nk)
    store2(row + j, x, y);
  else if (j < nk)
    store_from_float(row + j, x);
}

// kSplit: see flash_kernel.
template <typename T, int DP, bool kSplit> __global__ void __launch_bounds__(128) queries_kernel(const BackArgs x, int tiles, int clusters) {
  constexpr int BN = kTile<T, DP>, NT = BN / 8, ld = kLd<T, DP>, ND = DP / 8;
  const Args &a = x.a;
  extern __shared__ float4 smem4[];
  const int threads = blockDim.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rows = threads / 2;
  const int g = lane >> 2, t = lane & 3;
  T *qs = reinterpret_cast<T *>(smem4), *ds = qs + rows * ld, *dls = ds + rows * ld;
  T *ks = dls + (x.dlow ? rows * ld : 0), *vs = ks + 2 * BN * ld;
  float *mks = reinterpret_cast<float *>(vs + 2 * BN * ld);
  T *bs = reinterpret_cast<T *>(mks + 2 * BN);
  int tile, h, b;
  const int split = kSplit ? clusters : 1, rank = kSplit ? int(blockIdx.x) % split : 0;
  decode_cta(a, blockIdx.x / split, tiles, a.heads, tile, h, b);
  const int i0 = tile * rows, hk = h / a.group;
  const T *q = static_cast<const T *>(a.q.p) + b * a.q.sb + h * a.q.sh;
  const T *k = static_cast<const T *>(a.k.p) + b * a.k.sb + hk * a.k.sh;
  const T *v = static_cast<const T *>(a.v.p) + b * a.v.sb + hk * a.v.sh;
  const T *dout = static_cast<const T *>(x.dout) + (int64_t(b) * a.nq * a.heads + h) * a.d;
  const T *bias = a.bias ? static_cast<const T *>(a.bias) + (b / a.share) * a.bias_sb + h * a.bias_sh : nullptr;
  T *dbias = x.dbias && a.share == 1 ? static_cast<T *>(x.dbias) + (int64_t(b) * a.heads + h) * a.nq * x.dbias_ld : nullptr;
  auto load = [&](int j, int buf) {
    load_rows<T, DP, BN>(ks + buf * BN * ld, k, a.k.si, j * BN, a.nk, a.d, tid, threads);
    load_rows<T, DP, BN>(vs + buf * BN * ld, v, a.v.si, j * BN, a.nk, a.d, tid, threads);
    if (sizeof(T) == 2 && bias) load_bias<T, BN>(bs + buf * rows * (BN + 8), bias, a, i0, rows, j * BN, tid, threads);
    cp_commit();
  };
  constexpr int kChunks = DP / Type<T>::kVec;
  for (int u = tid; u < rows * kChunks; u += threads) {
    const int r = u / kChunks, c = u % kChunks * Type<T>::kVec;
    const bool ok = i0 + r < a.nq && c < a.d;
    cp16(qs + r * ld + c, ok ? q + int64_t(i0 + r) * a.q.si + c : q, ok ? 16 : 0);
    cp16(ds + r * ld + c, ok ? dout + int64_t(i0 + r) * a.heads * a.d + c : dout, ok ? 16 : 0);
    if (x.dlow) {
      const T *low = static_cast<const T *>(x.dlow) + (int64_t(b) * a.nq * a.heads + h) * a.d;
      cp16(dls + r * ld + c, ok ? low + int64_t(i0 + r) * a.heads * a.d + c : low, ok ? 16 : 0);
    }
  }
  // Key tiles [first, n_tiles).
  const int all_tiles = (a.nk + BN - 1) / BN, first = int(int64_t(rank) * all_tiles / split);
  const int n_tiles = int(int64_t(rank + 1) * all_tiles / split);
  if (n_tiles > first) load(first, 0);
  float m[2], nl[2], delta[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int i = i0 + warp * 16 + g + 8 * r;
    const int64_t at = (int64_t(b) * a.heads + h) * a.nq + i;
    m[r] = i < a.nq ? row_max(a.lse[at]) : INFINITY;
    nl[r] = i < a.nq ? -kLog2e * a.lse[a.lse_plane() + at] : 0.f;
    delta[r] = i < a.nq ? x.delta[at] : 0.f;
  }
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
  float dq[ND][4];
#pragma unroll
  for (int n = 0; n < ND; ++n) dq[n][0] = dq[n][1] = dq[n][2] = dq[n][3] = 0.f;

  float2 bv[sizeof(T) == 4 ? NT : 1][2];  // fp32 bias (see flash_kernel)
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
    T *kt = ks + buf * BN * ld, *vt = vs + buf * BN * ld;
    if (masked && a.mask_kind == kMaskKeep) {
      clear_left_out<T, DP, BN>(kt, mk, tid, threads);
      clear_left_out<T, DP, BN>(vt, mk, tid, threads);
      __syncthreads();
    }
    if (i0 + warp * 16 < a.nq) {
      float s[NT][4], dp[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = dp[n][e] = 0.f;
      mma_rows<NT, DP>(s, qs + warp * 16 * ld, kt, lane);
      if (x.dlow) mma_rows<NT, DP>(dp, dls + warp * 16 * ld, vt, lane);
      mma_rows<NT, DP>(dp, ds + warp * 16 * ld, vt, lane);
      const T *br = bs + buf * rows * (BN + 8) + (warp * 16 + g) * (BN + 8) + 2 * t;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float2 b0 = make_float2(0.f, 0.f), b1 = b0, m2 = b0;
        if constexpr (sizeof(T) == 4) {
          if (bias) b0 = bv[n][0], b1 = bv[n][1];
        } else {
          if (bias) b0 = load2(br + n * 8), b1 = load2(br + 8 * (BN + 8) + n * 8);
        }
        if (masked) m2 = load2(mk + n * 8 + 2 * t);
        grad_score(s[n][0], dp[n][0], a.scale, b0.x, m2.x, m[0], nl[0], delta[0]);
        grad_score(s[n][1], dp[n][1], a.scale, b0.y, m2.y, m[0], nl[0], delta[0]);
        grad_score(s[n][2], dp[n][2], a.scale, b1.x, m2.x, m[1], nl[1], delta[1]);
        grad_score(s[n][3], dp[n][3], a.scale, b1.y, m2.y, m[1], nl[1], delta[1]);
      }
      if (dbias) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int i = i0 + warp * 16 + g + 8 * r;
          if (i < a.nq) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
              store_bias(dbias + i * x.dbias_ld, j * BN + n * 8 + 2 * t, a.nk, dp[n][2 * r], dp[n][2 * r + 1]);
          }
        }
      }
      mma_acc<NT, DP>(dq, dp, kt, lane);
    }
    if (j + 1 < n_tiles) put_mask(buf ^ 1);
    __syncthreads();
  }
  cp_wait_all();
  if constexpr (kSplit) {  // the cluster's parts are added through shared memory, in the order of their keys
    float *part = reinterpret_cast<float *>(smem4);
    constexpr int pl = DP + 4;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int n = 0; n < ND; ++n)
        store2(part + (warp * 16 + g + 8 * r) * pl + n * 8 + 2 * t, dq[n][2 * r], dq[n][2 * r + 1]);
    cluster_barrier();
    for (int u = rank * threads + tid; u < rows * (DP / 4); u += split * threads) {
      const int row = u / (DP / 4), c = u % (DP / 4) * 4, i = i0 + row;
      if (i >= a.nq || c >= a.d) continue;
      float y[4] = {0.f, 0.f, 0.f, 0.f};
      for (int e = 0; e < split; ++e) {
        const float4 w = peer4(reinterpret_cast<const float4 *>(part + row * pl + c), uint32_t(e));
        y[0] += w.x, y[1] += w.y, y[2] += w.z, y[3] += w.w;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] *= a.scale;
      store4(static_cast<T *>(x.dq) + ((int64_t(b) * a.nq + i) * a.heads + h) * a.d + c, y);
    }
    cluster_barrier();  // until every part has been read
    return;
  }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int i = i0 + warp * 16 + g + 8 * r;
    if (i >= a.nq) continue;
    T *dst = static_cast<T *>(x.dq) + ((int64_t(b) * a.nq + i) * a.heads + h) * a.d;
#pragma unroll
    for (int n = 0; n < ND; ++n) {
      const int c = n * 8 + 2 * t;
      if (c < a.d) store2(dst + c, dq[n][2 * r] * a.scale, dq[n][2 * r + 1] * a.scale);
    }
  }
}

template <typename T, int DP> size_t bias_smem(int rows, bool low) {
  constexpr int ld = kLd<T, DP>, BN = kTile<T, DP>;
  return ((low ? 6 : 4) * size_t(rows) * ld + 4 * BN * ld + size_t(rows) * (BN + 8)) * sizeof(T) + 2 * BN * 4;
}

// dbias block [rows x BN] of one shared bias: the samples stream through a two-stage ring.
template <typename T, int DP> __global__ void __launch_bounds__(128) bias_kernel(const BackArgs x, int tiles, int cols) {
  constexpr int BN = kTile<T, DP>, NT = BN / 8, ld = kLd<T, DP>;
  const Args &a = x.a;
  extern __shared__ float4 smem4[];
  const int threads = blockDim.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rows = threads / 2;
  const int g = lane >> 2, t = lane & 3;
  T *qs = reinterpret_cast<T *>(smem4), *ds = qs + 2 * rows * ld, *dls = ds + 2 * rows * ld;
  T *ks = dls + (x.dlow ? 2 * rows * ld : 0), *vs = ks + 2 * BN * ld;
  T *bs = vs + 2 * BN * ld;
  float *mks = reinterpret_cast<float *>(bs + rows * (BN + 8));
  int64_t at = blockIdx.x;
  const int j0 = int(at % cols) * BN;
  at /= cols;
  const int i0 = int(at % tiles) * rows;
  at /= tiles;
  const int h = int(at % a.heads), bb = int(at / a.heads), hk = h / a.group;
  auto load = [&](int s, int buf) {
    const int b = bb * a.share + s;
    const T *q = static_cast<const T *>(a.q.p) + b * a.q.sb + h * a.q.sh;
    const T *dout = static_cast<const T *>(x.dout) + (int64_t(b) * a.nq * a.heads + h) * a.d;
    constexpr int kChunks = DP / Type<T>::kVec;
    for (int u = tid; u < rows * kChunks; u += threads) {
      const int r = u / kChunks, c = u % kChunks * Type<T>::kVec;
      const bool ok = i0 + r < a.nq && c < a.d;
      cp16(qs + (buf * rows + r) * ld + c, ok ? q + int64_t(i0 + r) * a.q.si + c : q, ok ? 16 : 0);
      cp16(ds + (buf * rows + r) * ld + c, ok ? dout + int64_t(i0 + r) * a.heads * a.d + c : dout, ok ? 16 : 0);
      if (x.dlow) {
        const T *low = static_cast<const T *>(x.dlow) + (int64_t(b) * a.nq * a.heads + h) * a.d;
        cp16(dls + (buf * rows + r) * ld + c, ok ? low + int64_t(i0 + r) * a.heads * a.d + c : low, ok ? 16 : 0);
      }
    }
    load_rows<T, DP, BN>(ks + buf * BN * ld, static_cast<const T *>(a.k.p) + b * a.k.sb + hk * a.k.sh, a.k.si, j0, a.nk,
                         a.d, tid, threads);
    load_rows<T, DP, BN>(vs + buf * BN * ld, static_cast<const T *>(a.v.p) + b * a.v.sb + hk * a.v.sh, a.v.si, j0, a.nk,
                         a.d, tid, threads);
    cp_commit();
    for (int u = tid; u < BN; u += threads) mks[buf * BN + u] = mask_value(a, b, j0 + u);
  };
  load_bias<T, BN>(bs, static_cast<const T *>(a.bias) + bb * a.bias_sb + h * a.bias_sh, a, i0, rows, j0, tid, threads);
  load(0, 0);
  float acc[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
  const int i_lo = i0 + warp * 16 + g;
  for (int s0 = 0; s0 < a.share; ++s0) {
    const int buf = s0 & 1;
    if (s0 + 1 < a.share) {
      load(s0 + 1, buf ^ 1);
      cp_wait<1>();
    } else {
      cp_wait<0>();
    }
    const int64_t row = (int64_t(bb * a.share + s0) * a.heads + h) * a.nq + i_lo;
    const float *lg = a.lse + a.lse_plane() + row;
    const float m0 = i_lo < a.nq ? row_max(a.lse[row]) : INFINITY, m1 = i_lo + 8 < a.nq ? row_max(a.lse[row + 8]) : INFINITY;
    const float n0 = i_lo < a.nq ? -kLog2e * lg[0] : 0.f, n1 = i_lo + 8 < a.nq ? -kLog2e * lg[8] : 0.f;
    const float d0 = i_lo < a.nq ? x.delta[row] : 0.f, d1 = i_lo + 8 < a.nq ? x.delta[row + 8] : 0.f;
    __syncthreads();
    if (i0 + warp * 16 < a.nq) {
      float s[NT][4], dp[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = dp[n][e] = 0.f;
      mma_rows<NT, DP>(s, qs + (buf * rows + warp * 16) * ld, ks + buf * BN * ld, lane);
      if (x.dlow) mma_rows<NT, DP>(dp, dls + (buf * rows + warp * 16) * ld, vs + buf * BN * ld, lane);
      mma_rows<NT, DP>(dp, ds + (buf * rows + warp * 16) * ld, vs + buf * BN * ld, lane);
      const T *br = bs + (warp * 16 + g) * (BN + 8) + 2 * t;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float2 b0 = load2(br + n * 8), b1 = load2(br + 8 * (BN + 8) + n * 8);
        const float2 m2 = load2(mks + buf * BN + n * 8 + 2 * t);
        grad_score(s[n][0], dp[n][0], a.scale, b0.x, m2.x, m0, n0, d0);
        grad_score(s[n][1], dp[n][1], a.scale, b0.y, m2.y, m0, n0, d0);
        grad_score(s[n][2], dp[n][2], a.scale, b1.x, m2.x, m1, n1, d1);
        grad_score(s[n][3], dp[n][3], a.scale, b1.y, m2.y, m1, n1, d1);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[n][e] += dp[n][e];
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int i = i_lo + 8 * r;
    if (i >= a.nq) continue;
    T *dst = static_cast<T *>(x.dbias) + ((int64_t(bb) * a.heads + h) * a.nq + i) * x.dbias_ld;
#pragma unroll
    for (int n = 0; n < NT; ++n) store_bias(dst, j0 + n * 8 + 2 * t, a.nk, acc[n][2 * r], acc[n][2 * r + 1]);
  }
}

// fp32 windows (17 to 32 queries, at most 128 keys, heads of their own): everything a (sample,
// head) needs fits in shared memory, so one CTA makes all four gradients from one set of scores,
// five products instead of the nine of the kernels above, and reads each tensor once.  Warp w
// has query rows 16 (w & 1) and keys 32 (w / 2); P and dS go through shared memory to the keys'
// products (16 keys per warp), dq is summed over the four key blocks.  The CTA walks the samples
// that share a bias, dbias stays in its registers.  96 biases x 4 samples of 32 x 128, 4 heads of 32:
// 67 us (150 with the kernels above; 76 with the bias read after the score products); bound by the split products' issue and latency, not by bytes
// (floor 17 us).
constexpr int kWinThreads = 256, kWinRows = 32, kWinKeys = 128, kWinLd = kWinKeys + 4;

template <int DP> constexpr size_t window_smem() {
  return (2 * kWinRows * kLd<float, DP> + 2 * kWinKeys * kLd<float, DP> + kWinRows * kWinLd + kWinKeys + 3 * kWinRows) * 4;
}
static_assert(kWinKeys * kLd<float, 32> >= kWinRows * kWinLd, "P takes V's place");

// acc[DP / 8][4] += A^T B over the kWinRows rows of A ([row][kWinLd], 16 columns from `a`) and B ([row][kLd]).
// A step's rows are taken in the order 0, 2, 4, 6, 1, 3, 5, 7: without bank conflicts.
template <int DP> __device__ __forceinline__ void mma_cols(float (&acc)[DP / 8][4], const float *a, const float *b, int lane) {
  constexpr int ld = kLd<float, DP>;
  const int g = lane >> 2, t = lane & 3;
  const float *ap = a + 2 * t * kWinLd + g, *bp = b + 2 * t * ld + g;
#pragma unroll
  for (int n0 = 0; n0 < DP / 8; n0 += 4) {
    float small[4][4];
#pragma unroll
    for (int n = 0; n < 4; ++n) small[n][0] = small[n][1] = small[n][2] = small[n][3] = 0.f;
#pragma unroll
    for (int kk = 0; kk < kWinRows / 8; ++kk) {
      uint32_t ah[4], al[4], bh[4][2], bl[4][2];
#pragma unroll
      for (int e = 0; e < 4; ++e) split_tf32(ap[(kk * 8 + (e >> 1)) * kWinLd + (e & 1) * 8], ah[e], al[e]);
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) split_tf32(bp[(kk * 8 + e) * ld + (n0 + n) * 8], bh[n][e], bl[n][e]);
#pragma unroll
      for (int n = 0; n < 4; ++n) mma8(small[n], al, bh[n]);
#pragma unroll
      for (int n = 0; n < 4; ++n) mma8(acc[n0 + n], ah, bh[n]);
#pragma unroll
      for (int n = 0; n < 4; ++n) mma8(small[n], ah, bl[n]);
    }
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[n0 + n][e] += small[n][e];
  }
}

template <int DP> __global__ void __launch_bounds__(kWinThreads, 2) window_kernel(const BackArgs x, int samples) {
  constexpr int ld = kLd<float, DP>, ND = DP / 8, NT = 4;
  const Args &a = x.a;
  extern __shared__ float4 smem4[];
  float *qs = reinterpret_cast<float *>(smem4), *dos = qs + kWinRows * ld, *ks = dos + kWinRows * ld, *vs = ks + kWinKeys * ld;
  float *dss = vs + kWinKeys * ld, *mks = dss + kWinRows * kWinLd, *st = mks + kWinKeys;
  float *ps = vs, *red = ks;  // once V, then K have been read
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int r0 = 16 * (warp & 1), c0 = 32 * (warp >> 1), key0 = 16 * warp;
  const int h = int(blockIdx.x % a.heads), b0 = int(blockIdx.x / a.heads) * samples;
  float *dbias = x.dbias ? static_cast<float *>(x.dbias) + (int64_t(b0 / a.share) * a.heads + h) * a.nq * x.dbias_ld : nullptr;
  const float *bias = a.bias ? static_cast<const float *>(a.bias) + (b0 / a.share) * a.bias_sb + h * a.bias_sh : nullptr;
  float sum[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n) sum[n][0] = sum[n][1] = sum[n][2] = sum[n][3] = 0.f;
  for (int b = b0; b < b0 + samples; ++b) {
    const float *q = static_cast<const float *>(a.q.p) + b * a.q.sb + h * a.q.sh;
    const float *k = static_cast<const float *>(a.k.p) + b * a.k.sb + h * a.k.sh;
    const float *v = static_cast<const float *>(a.v.p) + b * a.v.sb + h * a.v.sh;
    const float *dout = static_cast<const float *>(x.dout) + (int64_t(b) * a.nq * a.heads + h) * a.d;
    load_rows<float, DP, kWinRows>(qs, q, a.q.si, 0, a.nq, a.d, tid, kWinThreads);
    load_rows<float, DP, kWinRows>(dos, dout, int64_t(a.heads) * a.d, 0, a.nq, a.d, tid, kWinThreads);
    load_rows<float, DP, kWinKeys>(ks, k, a.k.si, 0, a.nk, a.d, tid, kWinThreads);
    load_rows<float, DP, kWinKeys>(vs, v, a.v.si, 0, a.nk, a.d, tid, kWinThreads);
    cp_commit();
    float2 bv[NT][2];  // the bias, in flight under the tiles' copies
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int i = r0 + g + 8 * r;
      const float *br = bias + int64_t(i) * a.bias_si + c0 + 2 * t;
#pragma unroll
      for (int n = 0; n < NT; ++n)
        bv[n][r] = bias ? bias_pair(a, br + n * 8, i < a.nq ? a.nk - c0 - n * 8 - 2 * t : 0) : make_float2(0.f, 0.f);
    }
    bool gone = false;
    if (tid < kWinKeys) {
      const float mk = mask_value(a, b, tid);
      mks[tid] = mk;
      gone = mk == -INFINITY;
    } else if (tid < kWinKeys + kWinRows) {
      const int i = tid - kWinKeys;
      const int64_t at = (int64_t(b) * a.heads + h) * a.nq + i;
      st[i] = i < a.nq ? row_max(a.lse[at]) : INFINITY;
      st[kWinRows + i] = i < a.nq ? -kLog2e * a.lse[a.lse_plane() + at] : 0.f;
      st[2 * kWinRows + i] = i < a.nq ? x.delta[at] : 0.f;
    }
    cp_wait_all();
    if (__syncthreads_or(gone)) {
      clear_left_out<float, DP, kWinKeys>(ks, mks, tid, kWinThreads);
      clear_left_out<float, DP, kWinKeys>(vs, mks, tid, kWinThreads);
      __syncthreads();
    }
    float s[NT][4], dp[NT][4], dq[ND][4];
#pragma unroll
    for (int n = 0; n < ND; ++n) dq[n][0] = dq[n][1] = dq[n][2] = dq[n][3] = 0.f;
    if (c0 < a.nk) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = dp[n][e] = 0.f;
      mma_rows<NT, DP>(s, qs + r0 * ld, ks + c0 * ld, lane);
      mma_rows<NT, DP>(dp, dos + r0 * ld, vs + c0 * ld, lane);
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int i = r0 + g + 8 * r;
        const float m = st[i], nl = st[kWinRows + i], delta = st[2 * kWinRows + i];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const int j = c0 + n * 8 + 2 * t;
          const float2 mk = load2(mks + j);
          grad_score(s[n][2 * r], dp[n][2 * r], a.scale, bv[n][r].x, mk.x, m, nl, delta);
          grad_score(s[n][2 * r + 1], dp[n][2 * r + 1], a.scale, bv[n][r].y, mk.y, m, nl, delta);
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[n][e] += dp[n][e];
      mma_acc<NT, DP>(dq, dp, ks + c0 * ld, lane);
    }
    __syncthreads();
    if (c0 < a.nk)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int at = (r0 + g + 8 * r) * kWinLd + c0 + n * 8 + 2 * t;
          store2(ps + at, s[n][2 * r], s[n][2 * r + 1]);
          store2(dss + at, dp[n][2 * r], dp[n][2 * r + 1]);
        }
    // dq of this key block, where K was.
#pragma unroll
    for (int n = 0; n < ND; ++n)
#pragma unroll
      for (int r = 0; r < 2; ++r)
        store2(red + ((warp >> 1) * kWinRows + r0 + g + 8 * r) * ld + n * 8 + 2 * t, dq[n][2 * r], dq[n][2 * r + 1]);
    __syncthreads();
    if (key0 < a.nk) {
      const int64_t at = ((int64_t(b) * a.nk + key0 + g) * a.heads + h) * a.d;
      auto product = [&](const float *left, const float *right, void *to, float scale) {
        float acc[ND][4];
#pragma unroll
        for (int n = 0; n < ND; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
        mma_cols<DP>(acc, left + key0, right, lane);
#pragma unroll
        for (int r = 0; r < 2; ++r)
          if (key0 + g + 8 * r < a.nk)
#pragma unroll
            for (int n = 0; n < ND; ++n)
              if (n * 8 + 2 * t < a.d)
                store2(static_cast<float *>(to) + at + int64_t(8 * r) * a.heads * a.d + n * 8 + 2 * t, scale * acc[n][2 * r],
                       scale * acc[n][2 * r + 1]);
      };
      product(ps, dos, x.dv, 1.f);
      product(dss, qs, x.dk, a.scale);
    }
    for (int u = tid; u < kWinRows * (DP / 4); u += kWinThreads) {
      const int i = u / (DP / 4), c = u % (DP / 4) * 4;
      if (i >= a.nq || c >= a.d) continue;
      float4 w = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float4 y = *reinterpret_cast<const float4 *>(red + (e * kWinRows + i) * ld + c);
        w.x += y.x, w.y += y.y, w.z += y.z, w.w += y.w;
      }
      *reinterpret_cast<float4 *>(static_cast<float *>(x.dq) + ((int64_t(b) * a.nq + i) * a.heads + h) * a.d + c) =
          make_float4(w.x * a.scale, w.y * a.scale, w.z * a.scale, w.w * a.scale);
    }
    __syncthreads();
  }
  if (dbias && c0 < a.nk)
#pragma unroll
    for (int r = 0; r < 2; ++r)
      if (r0 + g + 8 * r < a.nq)
#pragma unroll
        for (int n = 0; n < NT; ++n)
          store_bias(dbias + (r0 + g + 8 * r) * x.dbias_ld, c0 + n * 8 + 2 * t, a.nk, sum[n][2 * r], sum[n][2 * r + 1]);
}

// *taken where the windows' kernel has run.  At 32 x 128 x 4 heads it takes 12 us against 23 of the kernels above for
// 4 biases of one sample, 30 against 41 for 16 biases of 4, but a CTA that walks many samples alone is slower (107
// against 60 us for 1 bias of 16).  Below 17 queries or 33 keys half of its warps idle (43 against 39 us at 16 x 33).
template <int DP> int launch_window(const BackArgs &x, cudaStream_t stream, bool *taken) {
  const Args &a = x.a;
  const int samples = x.dbias ? a.share : 1;
  const int64_t ctas = int64_t(a.batch / samples) * a.heads;
  *taken = a.group == 1 && a.nq > 16 && a.nq <= kWinRows && a.nk > 32 && a.nk <= kWinKeys &&
           (samples <= 4 || ctas >= 2 * num_sms());
  if (!*taken) return BL_OK;
  BL_REQUIRE(ctas < (int64_t(1) << 31), "bl_cross_attention_backward: too many windows");
  BL_CUDA(ensure_smem_limit(reinterpret_cast<const void *>(window_kernel<DP>), 232448));
  window_kernel<DP><<<unsigned(ctas), kWinThreads, window_smem<DP>(), stream>>>(x, samples);
  BL_LAUNCH_CHECK();
  return BL_OK;
}

template <typename T, int DP> int launch(const BackArgs &x, cudaStream_t stream) {
  const Args &a = x.a;
  const bool biased = a.bias != nullptr;
  const int64_t rows_total = int64_t(a.batch) * a.nq * a.heads;
  BL_REQUIRE(rows_total < (int64_t(1) << 35), "bl_cross_attention_backward: too many query rows");
  rows_kernel<T><<<unsigned((rows_total + 31) / 32), 256, 0, stream>>>(x, rows_total);
  BL_LAUNCH_CHECK();
  bool taken = false;
  if constexpr (sizeof(T) == 4 && DP <= 64) {
    if (int rc = launch_window<DP>(x, stream, &taken)) return rc;
    if (taken) return BL_OK;
  }
  if (sizeof(T) == 2)
    if (int rc = keys_tc(x, stream, &taken)) return rc;
  if (a.nk > 0 && !taken) {
    const int64_t tiles = (a.nk + kKeys - 1) / kKeys, ctas = tiles * (a.heads / a.group) * a.batch;
    BL_REQUIRE(ctas < (int64_t(1) << 31), "bl_cross_attention_backward: too many key tiles");
    BL_CUDA(ensure_smem_limit(reinterpret_cast<const void *>(keys_kernel<T, DP>), 232448));
    keys_kernel<T, DP><<<unsigned(ctas), 128, keys_smem<T, DP>(biased, x.dlow != nullptr), stream>>>(x, int(tiles));
    BL_LAUNCH_CHECK();
  }
  const int warps = a.nq >= 64 ? 4 : (a.nq + 15) / 16, rows = 16 * warps;
  const int64_t tiles = (a.nq + rows - 1) / rows, ctas = tiles * a.heads * a.batch;
  BL_REQUIRE(ctas < (int64_t(1) << 31), "bl_cross_attention_backward: too many query tiles");
  taken = false;
  if (sizeof(T) == 2)
    if (int rc = queries_tc(x, stream, &taken)) return rc;
  if (!taken) {
    const int split = key_split(ctas, (a.nk + kTile<T, DP> - 1) / kTile<T, DP>);
    auto kernel = split > 1 ? queries_kernel<T, DP, true> : queries_kernel<T, DP, false>;
    BL_CUDA(ensure_smem_limit(reinterpret_cast<const void *>(kernel), 232448));
    BL_CUDA(launch_clusters(kernel, ctas, split, 32 * warps, queries_smem<T, DP>(rows, biased, x.dlow != nullptr), stream, x,
                            int(tiles), split));
    BL_LAUNCH_CHECK();
  }
  taken = false;
  if (sizeof(T) == 2 && x.dbias && a.share > 1)
    if (int rc = bias_tc(x, stream, &taken)) return rc;
  if (x.dbias && a.share > 1 && a.nk > 0 && !taken) {
    const int cols = (a.nk + kTile<T, DP> - 1) / kTile<T, DP>;
    const int64_t blocks = tiles * cols * a.heads * (a.batch / a.share);
    BL_REQUIRE(blocks < (int64_t(1) << 31), "bl_cross_attention_backward: too many bias blocks");
    BL_CUDA(ensure_smem_limit(reinterpret_cast<const void *>(bias_kernel<T, DP>), 232448));
    bias_kernel<T, DP><<<unsigned(blocks), 32 * warps, bias_smem<T, DP>(rows, x.dlow != nullptr), stream>>>(x, int(tiles), cols);
    BL_LAUNCH_CHECK();
  }
  return BL_OK;
}

template <typename T> int backward(const BackArgs &x, cudaStream_t stream) {
  if (x.a.d <= 32) return launch<T, 32>(x, stream);
  if (x.a.d <= 64) return launch<T, 64>(x, stream);
  return launch<T, 128>(x, stream);
}

int64_t delta_bytes(int64_t batch, int64_t heads, int64_t nq) { return (batch * heads * nq * 4 + 15) / 16 * 16; }

}  // namespace
}  // namespace xa
}  // namespace bl

using namespace bl;

extern "C" int64_t bl_cross_attention_workspace(const bl_cross_attention_args *x) {
  if (!x || x->batch <= 0 || x->heads <= 0 || x->nq <= 0 || x->head_dim <= 0) return 0;
  const int64_t rows = x->batch * x->nq * x->heads;
  // delta; with a gate do, as fp32 or as two bf16 planes
  return xa::delta_bytes(x->batch, x->heads, x->nq) + (x->gate ? rows * x->head_dim * 4 : 0);
}

extern "C" int bl_cross_attention_backward(const bl_cross_attention_args *x, const void *dy, void *dq, void *dk, void *dv,
                                           void *dbias, int64_t dbias_ld, void *dgate, void *workspace,
                                           int64_t workspace_bytes, void *stream) {
  BL_REQUIRE(x, "bl_cross_attention_backward: null arguments");
  BL_REQUIRE(x->batch < (1 << 30) && x->heads < (1 << 16) && x->kv_heads < (1 << 16) && x->nq < (1 << 30) &&
                 x->nk < (1 << 30) && x->head_dim < (1 << 16) && x->bias_share < (1 << 30),
             "bl_cross_attention_backward: shape too large");
  xa::BackArgs y{};
  y.a = xa::make_args(x);
  const xa::Args &a = y.a;
  if (int rc = xa::check("bl_cross_attention_backward", a, x->kv_heads, x->dtype)) return rc;
  cudaStream_t st = as_stream(stream);
  const size_t size = x->dtype == BL_F32 ? 4 : 2;
  if (a.batch == 0) return BL_OK;
  if (a.nq == 0) {
    if (a.nk == 0) return BL_OK;
    BL_REQUIRE(dk && dv, "bl_cross_attention_backward: null pointer");
    const size_t bytes = size_t(a.batch) * a.nk * size_t(x->kv_heads) * a.d * size;
    BL_CUDA(cudaMemsetAsync(dk, 0, bytes, st));
    BL_CUDA(cudaMemsetAsync(dv, 0, bytes, st));
    return BL_OK;
  }
  const int64_t need = bl_cross_attention_workspace(x);
  BL_REQUIRE(workspace && workspace_bytes >= need && aligned_to(workspace, 16),
             "bl_cross_attention_backward: needs a 16-byte aligned workspace of %lld bytes", (long long)need);
  BL_REQUIRE(dy && a.lse && dq && (a.nk == 0 || (dk && dv)) && (!dbias || a.bias) && (!a.gate.p || dgate),
             "bl_cross_attention_backward: null pointer");
  BL_REQUIRE(aligned_to(dy, 16) && aligned_to(dq, 16) && aligned_to(dk, 16) && aligned_to(dv, 16) && aligned_to(dgate, 16) &&
                 aligned_to(dbias, 16) && dbias_ld % 8 == 0 && (!dbias || dbias_ld >= a.nk),
             "bl_cross_attention_backward: gradients must be 16-byte aligned, the bias gradient's rows of a multiple of 8 "
             "elements");
  y.dy = dy;
  y.delta = static_cast<float *>(workspace);
  y.dout = a.gate.p ? static_cast<char *>(workspace) + xa::delta_bytes(a.batch, a.heads, a.nq) : dy;
  if (a.gate.p && x->dtype == BL_BF16)
    y.dlow = static_cast<const __nv_bfloat16 *>(y.dout) + int64_t(a.batch) * a.nq * a.heads * a.d;
  y.dq = dq, y.dk = dk, y.dv = dv, y.dgate = dgate, y.dbias = dbias, y.dbias_ld = dbias_ld;
  return x->dtype == BL_F32 ? xa::backward<float>(y, st) : xa::backward<__nv_bfloat16>(y, st);
}
