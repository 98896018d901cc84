// Learned relative positions by buckets, and the gradients of their tables.
//
// 1. Encoding of a pair tensor (AF3 supplementary Algorithm 3, upstream
//    RelativePositionEncoder):
//      out[b, i, j] = W[:, p] + W[:, R + t] + [entity_i = entity_j] W[:, 2 R] + W[:, 2 R + 1 + c],  R = 2 r + 2
//      p = clip(residue_i - residue_j + r, 0, 2 r)  same chain (asym), else 2 r + 1
//      t = clip(token_i - token_j + r, 0, 2 r)      same chain and residue, else 2 r + 1
//      c = 2 s + 1  same chain (fix_sym: entities differ), else clip(sym_i - sym_j + s, 0, 2 s)
//    The one-hot features and their product with W never exist: a pair's row is
//    the sum of at most four rows of W^T, which sits in shared memory.
// 2. Bias of attention heads, queries and keys of any two lengths:
//      out[b, h, i, j] = table[u][h],  u = lut[clip(q_pos_i - k_pos_j, -D, D) + D], other group: the last bucket
//
// Both forwards are bound by their HBM writes and both gradients by reading
// the upstream gradient once.  The gradients are deterministic: every partial
// sum belongs to one thread, and partials are added in a fixed order.
#include <type_traits>

#include "common.cuh"

namespace bl {
namespace {

constexpr int kMaxSmem = 232448;  // 227 KB: the limit of one CTA

// ---------------------------------------------------------------------------
// Encoding
// ---------------------------------------------------------------------------
struct EncArgs {
  const int64_t *residue, *asym, *entity, *token, *sym;  // [batch][n]
  int n, channels, rows;                                 // rows: columns of W
  int r, s, fix_sym;
  int64_t batch;
};

// The picks of pair (i, j), packed: residue row (bits 0..9), token row
// (10..19), chain-copy row (20..29), entities agree (30).
__device__ __forceinline__ uint32_t clip_offset(int64_t a, int64_t b, int m) {
  const int64_t d = a - b;
  return uint32_t(d < -m ? 0 : d > m ? 2 * m : int(d) + m);
}
__device__ __forceinline__ uint32_t pick(const EncArgs &a, int64_t i, int64_t j) {
  const int64_t ri = a.residue[i], rj = a.residue[j];
  const bool chain = a.asym[i] == a.asym[j], agree = a.entity[i] == a.entity[j];
  const uint32_t apart = 2 * a.r + 1;
  const uint32_t p = chain ? clip_offset(ri, rj, a.r) : apart;
  const uint32_t t = apart + 1 + (chain && ri == rj ? clip_offset(a.token[i], a.token[j], a.r) : apart);
  const bool other = a.fix_sym ? !agree : chain;
  const uint32_t c = 2 * (apart + 1) + 1 + (other ? 2 * a.s + 1 : clip_offset(a.sym[i], a.sym[j], a.s));
  return p | (t << 10) | (c << 20) | (uint32_t(agree) << 30);
}

// W[c0 .. c0 + kC)[rows] -> shared [rows][kC + 4], by 4-byte asynchronous copies: all of a
// thread's are in flight at once (a load-store loop took 40 of 63 us at 512 tokens).  Eight
// lanes read eight consecutive columns of one W row (a full 32-byte sector), four rows
// per warp step; the padded row keeps the 32 transposed writes in distinct banks.
template <int kC> __device__ __forceinline__ void load_rows(float *dst, const float *w, const EncArgs &a, int c0) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int c = lane >> 3;
  for (int r0 = 0; r0 < a.rows; r0 += 8) {
    const int row = r0 + (lane & 7);
    for (int q = warp; q < kC / 4; q += warps) {
      const bool ok = row < a.rows && c0 + 4 * q + c < a.channels;
      if (row < a.rows) {
        const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(dst + row * (kC + 4) + 4 * q + c));
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to),
                     "l"(w + (ok ? int64_t(c0 + 4 * q + c) * a.rows + row : 0)), "r"(ok ? 4 : 0)
                     : "memory");
      }
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

__device__ __forceinline__ float4 add4(float4 a, float4 b) {
  return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w);
}

// kLanes lanes (4 channels each) per pair; a warp step writes 32 / kLanes
// pairs.  A warp takes 32 consecutive pairs of one row i: lane l computes the
// picks of pair j0 + l, the others receive them by shuffle.  The sum of the
// token, entity and chain rows repeats along most of a row, so it stays in
// registers until its picks change: one shared load per pair and lane.
template <typename Out, int kLanes, bool kAdd>
__global__ void __launch_bounds__(256) encoding_kernel(const float *w, const EncArgs a, Out *out) {
  constexpr int kC = 4 * kLanes, kLd = kC + 4, kPairs = 32 / kLanes;
  extern __shared__ float4 smem4[];
  float *rows = reinterpret_cast<float *>(smem4);
  const int c0 = blockIdx.y * kC;
  load_rows<kC>(rows, w, a, c0);
  __syncthreads();
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int sub = lane / kLanes, c = 4 * (lane % kLanes);
  const int n = a.n, segments = (n + 31) / 32;
  const bool live = c0 + c < a.channels;
  const uint32_t units = uint32_t(a.batch * n * segments);  // below 2^31: checked by the host
  const float *col = rows + c;
  uint32_t held = 0xffffffffu;
  float4 base = make_float4(0.f, 0.f, 0.f, 0.f);
  for (uint32_t u = blockIdx.x * warps + (threadIdx.x >> 5); u < units; u += gridDim.x * warps) {
    const uint32_t row = u / uint32_t(segments);  // b * n + i
    const int j0 = int(u - row * segments) * 32;
    const int64_t i = row, b0 = row / uint32_t(n) * n;
    const uint32_t mine = j0 + lane < n ? pick(a, i, b0 + j0 + lane) : 0u;
    const int count = n - j0 < 32 ? n - j0 : 32;
    Out *dst = out + (i * n + j0) * a.channels + c0 + c;
#pragma unroll 4
    for (int t = 0; t < count; t += kPairs) {
      const int jj = t + sub;
      const uint32_t v = __shfl_sync(0xffffffffu, mine, jj & 31);
      if (jj < count && live) {
        if ((v >> 10) != held) {
          held = v >> 10;
          base = add4(*reinterpret_cast<const float4 *>(col + ((v >> 10) & 1023u) * kLd),
                      *reinterpret_cast<const float4 *>(col + ((v >> 20) & 1023u) * kLd));
          if (v >> 30) base = add4(base, *reinterpret_cast<const float4 *>(col + (4 * a.r + 4) * kLd));
        }
        float4 y = add4(*reinterpret_cast<const float4 *>(col + (v & 1023u) * kLd), base);
        Out *p = dst + int64_t(jj) * a.channels;
        if constexpr (sizeof(Out) == 4) {
          if (kAdd) y = add4(y, *reinterpret_cast<const float4 *>(p));
          *reinterpret_cast<float4 *>(p) = y;
        } else {
          *reinterpret_cast<uint2 *>(p) = make_uint2(pack_bf16x2(y.x, y.y), pack_bf16x2(y.z, y.w));
        }
      }
    }
  }
}

// Gradient of W.  A group of two warps covers 128 channels (two per lane) and owns
// a private [rows][128] table in shared memory, each element of which one lane
// alone updates.  A group walks diagonals: from pair (i0, j) it visits
// (i0 + s, (j + s) mod n) for up to kSteps rows, every load a coalesced half of a
// pair row, all of a walk's loads in flight at once.  Along a diagonal of one chain
// the offsets, so the picks, do not change: the sum of the pairs stays in registers
// and goes to the table rows of its picks when one of them changes.
constexpr int kGroups = 3;  // private tables per CTA (71 KB each at r = 32, s = 2)
template <typename In> constexpr int kSteps = sizeof(In) == 4 ? 32 : 64;

template <typename In>
__global__ void __launch_bounds__(kGroups * 64) encoding_grad_kernel(const In *grad, const EncArgs a, float *partial) {
  constexpr int kS = kSteps<In>;
  extern __shared__ float4 smem4[];
  float *tables = reinterpret_cast<float *>(smem4);
  const int groups = blockDim.x / 64, size = a.rows * 128;
  for (int i = threadIdx.x; i < groups * size / 4; i += blockDim.x) smem4[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  __syncthreads();
  const int lane = threadIdx.x & 31, group = threadIdx.x / 64;
  const int ch = threadIdx.x % 64 * 2, c0 = blockIdx.y * 128;
  const bool live = c0 + ch < a.channels;  // channels is even
  float2 *mine = reinterpret_cast<float2 *>(tables + group * size + ch);
  const int n = a.n, blocks = (n + kS - 1) / kS;
  const uint32_t units = uint32_t(a.batch * blocks * n);
  const int64_t step = (int64_t(n) + 1) * a.channels, wrap = int64_t(n) * a.channels;
  float2 run = make_float2(0.f, 0.f);
  uint32_t held = 0xffffffffu;
  auto put = [&](uint32_t row) {
    float2 v = mine[row * 64];
    v.x += run.x, v.y += run.y;
    mine[row * 64] = v;
  };
  auto flush = [&]() {
    put(held & 1023u), put((held >> 10) & 1023u), put((held >> 20) & 1023u);
    if (held >> 30) put(4 * a.r + 4);
    run = make_float2(0.f, 0.f);
  };
  for (uint32_t u = blockIdx.x * groups + group; u < units; u += gridDim.x * groups) {
    const uint32_t ib = u / uint32_t(n), b = ib / uint32_t(blocks);
    const int j = int(u - ib * n), i0 = int(ib - b * blocks) * kS;
    const int64_t b0 = int64_t(b) * n;
    const int count = n - i0 < kS ? n - i0 : kS;
    const In *p = grad + ((b0 + i0) * n + j) * a.channels + c0 + ch;
    typename std::conditional<sizeof(In) == 4, float2, uint32_t>::type x[kS];
    int col = j;
#pragma unroll
    for (int s = 0; s < kS; ++s) {
      if (s < count && live) {
        if constexpr (sizeof(In) == 4)
          x[s] = __ldcs(reinterpret_cast<const float2 *>(p));
        else
          x[s] = __ldcs(reinterpret_cast<const unsigned int *>(p));
      } else {
        x[s] = {};
      }
      p += step;
      if (++col == n) col = 0, p -= wrap;
    }
    uint32_t packed[kS / 32];
#pragma unroll
    for (int e = 0; e < kS / 32; ++e) {
      const int s = 32 * e + lane;
      packed[e] = s < count ? pick(a, b0 + i0 + s, b0 + (j + s) % n) : 0u;
    }
#pragma unroll
    for (int s = 0; s < kS; ++s) {
      if (s >= count) break;
      const uint32_t v = __shfl_sync(0xffffffffu, packed[s / 32], s % 32);
      if (v != held) {
        if (held != 0xffffffffu) flush();
        held = v;
      }
      if constexpr (sizeof(In) == 4)
        run.x += x[s].x, run.y += x[s].y;
      else
        run.x += bf16_lo(x[s]), run.y += bf16_hi(x[s]);
    }
  }
  if (held != 0xffffffffu) flush();
  __syncthreads();
  // partial[cta][channel chunk][row][128]
  float4 *dst = reinterpret_cast<float4 *>(partial + (int64_t(blockIdx.x) * gridDim.y + blockIdx.y) * size);
  for (int i = threadIdx.x; i < size / 4; i += blockDim.x) {
    float4 v = smem4[i];
    for (int g = 1; g < groups; ++g) v = add4(v, smem4[g * (size / 4) + i]);
    dst[i] = v;
  }
}

// dw[c][row] = sum over CTAs of partial[cta][c / 128][row][c % 128]; 8 threads per output, joined in a fixed order.
__global__ void __launch_bounds__(256) encoding_grad_sum_kernel(const float *partial, int ctas, int chunks, int rows,
                                                                int channels, float *dw) {
  __shared__ float part[8][33];
  const int lane = threadIdx.x & 31, way = threadIdx.x >> 5;
  const int64_t size = int64_t(chunks) * rows * 128;
  const int64_t at = int64_t(blockIdx.x) * 32 + lane;
  float v = 0.f;
  if (at < size)
    for (int k = way; k < ctas; k += 8) v += partial[k * size + at];
  part[way][lane] = v;
  __syncthreads();
  if (way == 0 && at < size) {
    for (int k = 1; k < 8; ++k) v += part[k][lane];
    const int c = int(at / (int64_t(rows) * 128)) * 128 + int(at % 128), row = int(at / 128 % rows);
    if (c < channels) dw[int64_t(c) * rows + row] = v;
  }
}

int encoding_check(const char *name, const EncArgs &a, int64_t n, int64_t channels, int64_t r, int64_t s) {
  BL_REQUIRE(a.batch >= 0 && n >= 0 && n <= (1 << 15) && a.batch <= (1 << 20), "%s: bad shape", name);
  BL_REQUIRE(a.batch * n * ((n + 31) / 32) < (int64_t(1) << 31), "%s: too many token pairs", name);
  BL_REQUIRE(channels >= 4 && channels <= 4096 && channels % 4 == 0, "%s: channels must be a multiple of 4, at most 4096",
             name);
  BL_REQUIRE(r >= 0 && s >= 0 && r <= 96 && s <= 16, "%s: r_max must lie in [0, 96], s_max in [0, 16]", name);
  BL_REQUIRE(a.batch == 0 || n == 0 || (a.residue && a.asym && a.entity && a.token && a.sym), "%s: null pointer", name);
  return BL_OK;
}

int encoding_grad_groups(int rows) {  // private tables that fit in 227 KB
  const int fit = kMaxSmem / (rows * 128 * 4);
  return fit < kGroups ? fit : kGroups;
}
int64_t encoding_grad_ctas(int64_t batch, int64_t n, int rows, int chunks) {
  const int64_t units = batch * ((n + 31) / 32) * n, groups = encoding_grad_groups(rows);
  const int64_t want = (units + groups - 1) / groups, cap = (num_sms() + chunks - 1) / chunks;
  return want < 1 ? 1 : want < cap ? want : cap;
}

// ---------------------------------------------------------------------------
// Bias of attention heads
// ---------------------------------------------------------------------------
struct BiasArgs {
  const int64_t *q_pos, *k_pos, *q_group, *k_group;  // [batch][nq], [batch][nk]; groups may be null
  const int *lut;                                    // [2 * distance + 1]
  int distance, buckets, heads, nq, nk;
  int64_t batch;
  int64_t sb, sh, sq;  // element strides of the planes
};

// lut as 16-bit entries in shared memory; entries outside [0, buckets) become the last bucket.
__device__ __forceinline__ void load_lut(uint16_t *dst, const BiasArgs &a) {
  for (int i = threadIdx.x; i < 2 * a.distance + 1; i += blockDim.x) {
    const uint32_t u = uint32_t(a.lut[i]), last = uint32_t(a.buckets - 1);
    dst[i] = uint16_t(u < last ? u : last);
  }
}
__device__ __forceinline__ int bucket_of(const uint16_t *lut, const BiasArgs &a, int64_t q, int64_t k, bool same) {
  const int64_t d = q - k;
  const int at = d < -a.distance ? 0 : d > a.distance ? 2 * a.distance : int(d) + a.distance;
  return same ? lut[at] : a.buckets - 1;
}

// A thread keeps four key columns and their positions, computes their buckets
// once per query row and writes them for every head (16 or 8 bytes per store).
constexpr int kBiasThreads = 128, kBiasCols = 4 * kBiasThreads;

template <typename Out>
__global__ void __launch_bounds__(kBiasThreads) bias_kernel(const float *table, const BiasArgs a, Out *out, int q_rows,
                                                            int vector) {
  extern __shared__ float4 smem4[];
  float *tab = reinterpret_cast<float *>(smem4);                      // [heads][buckets]
  uint16_t *lut = reinterpret_cast<uint16_t *>(tab + a.heads * a.buckets);
  for (int i = threadIdx.x; i < a.heads * a.buckets; i += kBiasThreads)
    tab[i % a.heads * a.buckets + i / a.heads] = table[i];
  load_lut(lut, a);
  __syncthreads();
  const int64_t b = blockIdx.z;
  const int j = blockIdx.x * kBiasCols + 4 * threadIdx.x;
  if (j >= a.nk) return;
  const int count = a.nk - j < 4 ? a.nk - j : 4;
  int64_t kp[4], kg[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int64_t at = b * a.nk + j + (e < count ? e : 0);
    kp[e] = a.k_pos[at];
    kg[e] = a.k_group ? a.k_group[at] : 0;
  }
  const int i0 = blockIdx.y * q_rows, i1 = i0 + q_rows < a.nq ? i0 + q_rows : a.nq;
  for (int i = i0; i < i1; ++i) {
    const int64_t qp = a.q_pos[b * a.nq + i], qg = a.q_group ? a.q_group[b * a.nq + i] : 0;
    int u[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) u[e] = bucket_of(lut, a, qp, kp[e], qg == kg[e]);
    Out *p = out + b * a.sb + int64_t(i) * a.sq + j;
    const float *row = tab;
#pragma unroll 4
    for (int h = 0; h < a.heads; ++h, row += a.buckets, p += a.sh) {
      const float y[4] = {row[u[0]], row[u[1]], row[u[2]], row[u[3]]};
      if (vector && count == 4) {
        if constexpr (sizeof(Out) == 4)
          __stcs(reinterpret_cast<float4 *>(p), make_float4(y[0], y[1], y[2], y[3]));
        else
          __stcs(reinterpret_cast<uint2 *>(p), make_uint2(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])));
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (e < count) store_from_float(p + e, y[e]);
      }
    }
  }
}

// Four neighbouring elements of a row as loaded.
template <typename T> struct Quad;
template <> struct Quad<float> {
  using type = float4;
  static __device__ __forceinline__ float4 load(const float *p, int count, bool vector) {
    if (vector) return __ldcs(reinterpret_cast<const float4 *>(p));
    return make_float4(p[0], count > 1 ? p[1] : 0.f, count > 2 ? p[2] : 0.f, count > 3 ? p[3] : 0.f);
  }
  static __device__ __forceinline__ float get(const float4 &v, int e) {
    return e == 0 ? v.x : e == 1 ? v.y : e == 2 ? v.z : v.w;
  }
};
template <> struct Quad<__nv_bfloat16> {
  using type = uint2;
  static __device__ __forceinline__ uint2 load(const __nv_bfloat16 *p, int count, bool vector) {
    if (vector) return __ldcs(reinterpret_cast<const uint2 *>(p));
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = e < count ? __bfloat162float(p[e]) : 0.f;
    return make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));  // exact
  }
  static __device__ __forceinline__ float get(const uint2 &v, int e) {
    return e == 0 ? bf16_lo(v.x) : e == 1 ? bf16_hi(v.x) : e == 2 ? bf16_lo(v.y) : bf16_hi(v.y);
  }
};

// Gradient of the table.  A thread owns four key columns of kHeads heads and
// walks down the query rows with one running sum per column and head; when a
// column's bucket changes, its sums go to the thread's own column of the
// shared histogram [bucket][head][thread] (bank = thread: no conflicts, no
// atomics).  The bucket of a (row, column) is computed once for kHeads heads.
template <typename In, int kHeads>
__global__ void __launch_bounds__(kBiasThreads) bias_grad_kernel(const In *grad, const BiasArgs a, int q_rows,
                                                                 int vector, float *partial) {
  extern __shared__ float4 smem4[];
  float *hist = reinterpret_cast<float *>(smem4);
  uint16_t *lut = reinterpret_cast<uint16_t *>(hist + a.buckets * kHeads * kBiasThreads);
  for (int i = threadIdx.x; i < a.buckets * kHeads * kBiasThreads; i += kBiasThreads) hist[i] = 0.f;
  load_lut(lut, a);
  __syncthreads();
  float *mine = hist + threadIdx.x;
  const int h0 = blockIdx.y * kHeads, heads = a.heads - h0 < kHeads ? a.heads - h0 : kHeads;
  // Four columns per thread, consecutive over all samples: no thread idles at a row's end.
  const int quads = (a.nk + 3) / 4, row_blocks = (a.nq + q_rows - 1) / q_rows;
  const uint32_t all_quads = uint32_t(a.batch * quads), col_blocks = (all_quads + kBiasThreads - 1) / kBiasThreads;
  const uint32_t units = col_blocks * row_blocks;
  for (uint32_t u = blockIdx.x; u < units; u += gridDim.x) {
    const uint32_t rb = u / col_blocks, quad = (u - rb * col_blocks) * kBiasThreads + threadIdx.x;
    if (quad >= all_quads) continue;
    const int64_t b = quad / uint32_t(quads);
    const int j = 4 * int(quad - uint32_t(b) * quads);
    const int i0 = int(rb) * q_rows, i1 = i0 + q_rows < a.nq ? i0 + q_rows : a.nq;
    const int count = a.nk - j < 4 ? a.nk - j : 4;
    int64_t kp[4], kg[4];
    int held[4];
    float run[4][kHeads];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int64_t at = b * a.nk + j + (e < count ? e : 0);
      kp[e] = a.k_pos[at];
      kg[e] = a.k_group ? a.k_group[at] : 0;
      held[e] = -1;
#pragma unroll
      for (int h = 0; h < kHeads; ++h) run[e][h] = 0.f;
    }
    const In *base = grad + b * a.sb + h0 * a.sh + j;
    auto load = [&](int i, typename Quad<In>::type (&x)[kHeads]) {
#pragma unroll
      for (int h = 0; h < kHeads; ++h) {
        x[h] = {};
        if (h < heads) x[h] = Quad<In>::load(base + h * a.sh + int64_t(i) * a.sq, count, vector && count == 4);
      }
    };
    auto take = [&](int i, const typename Quad<In>::type (&x)[kHeads]) {
      const int64_t qp = a.q_pos[b * a.nq + i], qg = a.q_group ? a.q_group[b * a.nq + i] : 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int v = bucket_of(lut, a, qp, kp[e], qg == kg[e]);
        if (v != held[e]) {
          if (held[e] >= 0) {
#pragma unroll
            for (int h = 0; h < kHeads; ++h) {
              mine[(held[e] * kHeads + h) * kBiasThreads] += run[e][h];
              run[e][h] = 0.f;
            }
          }
          held[e] = v;
        }
#pragma unroll
        for (int h = 0; h < kHeads; ++h) run[e][h] += Quad<In>::get(x[h], e);
      }
    };
    constexpr int kAhead = 4;  // rows in flight
    int i = i0;
    for (; i + kAhead <= i1; i += kAhead) {
      typename Quad<In>::type x[kAhead][kHeads];
#pragma unroll
      for (int r = 0; r < kAhead; ++r) load(i + r, x[r]);
#pragma unroll
      for (int r = 0; r < kAhead; ++r) take(i + r, x[r]);
    }
    for (; i < i1; ++i) {
      typename Quad<In>::type x[kHeads];
      load(i, x);
      take(i, x);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (held[e] >= 0) {
#pragma unroll
        for (int h = 0; h < kHeads; ++h) mine[(held[e] * kHeads + h) * kBiasThreads] += run[e][h];
      }
  }
  __syncthreads();
  // partial[head group][cta][bucket][kHeads]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float *dst = partial + (int64_t(blockIdx.y) * gridDim.x + blockIdx.x) * a.buckets * kHeads;
  for (int k = warp; k < a.buckets * kHeads; k += kBiasThreads / 32) {
    const float *row = hist + k * kBiasThreads + lane;
    const float v = warp_sum((row[0] + row[32]) + (row[64] + row[96]));
    if (lane == 0) dst[k] = v;
  }
}

// dtable[bucket][head] = sum over CTAs; one warp per output.
__global__ void __launch_bounds__(256) bias_grad_sum_kernel(const float *partial, int ctas, int buckets, int heads,
                                                            int per_group, float *dtable) {
  const int at = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (at >= buckets * heads) return;
  const int u = at / heads, h = at % heads;
  const float *src = partial + int64_t(h / per_group) * ctas * buckets * per_group + u * per_group + h % per_group;
  float v = 0.f;
  for (int k = lane; k < ctas; k += 32) v += src[int64_t(k) * buckets * per_group];
  v = warp_sum(v);
  if (lane == 0) dtable[at] = v;
}

int bias_check(const char *name, const BiasArgs &a) {
  BL_REQUIRE(a.batch >= 0 && a.nq >= 0 && a.nk >= 0 && a.batch < 65536, "%s: bad shape", name);
  BL_REQUIRE(a.heads >= 1 && a.heads <= 1024 && a.buckets >= 1 && a.buckets <= 256 && a.distance >= 0 && a.distance <= 8192,
             "%s: heads must lie in [1, 1024], buckets in [1, 256] and the clipping distance in [0, 8192]", name);
  BL_REQUIRE(int64_t(a.heads) * a.buckets <= 40960, "%s: heads * buckets must be at most 40960", name);
  BL_REQUIRE(a.lut, "%s: lut is required", name);
  BL_REQUIRE(a.batch == 0 || a.nq == 0 || a.nk == 0 || (a.q_pos && a.k_pos), "%s: positions are required", name);
  BL_REQUIRE(a.batch * ((a.nk + 3) / 4) * int64_t(a.nq) < (int64_t(1) << 38) && a.batch * a.nk < (int64_t(1) << 31),
             "%s: shape too large", name);
  BL_REQUIRE(!a.q_group == !a.k_group, "%s: give both groups or neither", name);
  return BL_OK;
}

int bias_lut_bytes(int distance) { return (2 * distance + 1) * 2; }
int bias_grad_heads(int buckets) { return buckets <= 48 ? 4 : 1; }  // 2 KB (4 heads) or 0.5 KB (1) per bucket
// Launch shape of the table gradient: three CTAs per SM (67 KB of histogram at 33 buckets x 4 heads), and rows per
// unit such that a CTA has about eight units to even out, in whole groups of four rows.
struct BiasGrad {
  int per, groups, rows;
  int64_t ctas;
};
BiasGrad bias_grad_shape(int64_t batch, int64_t heads, int64_t nq, int64_t nk, int buckets) {
  BiasGrad g;
  g.per = bias_grad_heads(buckets);
  g.groups = int((heads + g.per - 1) / g.per);
  const int64_t cols = (batch * ((nk + 3) / 4) + kBiasThreads - 1) / kBiasThreads;
  const int64_t cap = (3 * num_sms() + g.groups - 1) / g.groups;
  int64_t rows = nq * cols / (8 * cap) / 4 * 4;
  g.rows = int(rows < 4 ? 4 : rows > 64 ? 64 : rows);
  const int64_t units = cols * ((nq + g.rows - 1) / g.rows);
  g.ctas = units < 1 ? 1 : units < cap ? units : cap;
  return g;
}

bool vector_planes(const void *p, const BiasArgs &a, int dtype) {
  return aligned_to(p, dtype == BL_F32 ? 16 : 8) && a.sb % 4 == 0 && a.sh % 4 == 0 && a.sq % 4 == 0;
}

}  // namespace
}  // namespace bl

using namespace bl;

extern "C" int bl_relative_position_encoding(const float *weight, const int64_t *residue, const int64_t *asym,
                                             const int64_t *entity, const int64_t *token, const int64_t *sym,
                                             int64_t batch, int64_t n, int64_t channels, int64_t r_max, int64_t s_max,
                                             int fix_sym, void *out, int out_dtype, int add, void *stream) {
  EncArgs a{residue, asym, entity, token, sym, int(n), int(channels), int(4 * r_max + 2 * s_max + 7), int(r_max),
            int(s_max), fix_sym, batch};
  if (int rc = encoding_check("bl_relative_position_encoding", a, n, channels, r_max, s_max)) return rc;
  BL_REQUIRE(out_dtype == BL_F32 || out_dtype == BL_BF16, "bl_relative_position_encoding: dtype must be fp32 or bf16");
  BL_REQUIRE(!add || out_dtype == BL_F32, "bl_relative_position_encoding: adding needs an fp32 output");
  if (batch == 0 || n == 0) return BL_OK;
  BL_REQUIRE(weight && out && aligned_to(out, 16), "bl_relative_position_encoding: null or unaligned pointer");
  // 128 channels per CTA once every SM has several warps of pairs to write;
  // 32 for fewer pairs (or channels): a quarter of the table to load per CTA
  // and four times the CTAs.
  const int64_t units = batch * n * ((n + 31) / 32);
  const bool wide = channels % 128 == 0 && units >= 16 * int64_t(num_sms());
  const int kc = wide ? 128 : 32;
  const int smem = a.rows * (kc + 4) * 4, chunks = int((channels + kc - 1) / kc);
  auto kernel = out_dtype == BL_F32
                    ? (add ? (wide ? encoding_kernel<float, 32, true> : encoding_kernel<float, 8, true>)
                           : (wide ? encoding_kernel<float, 32, false> : encoding_kernel<float, 8, false>))
                    : nullptr;
  auto kernel16 = wide ? encoding_kernel<__nv_bfloat16, 32, false> : encoding_kernel<__nv_bfloat16, 8, false>;
  const void *fn = kernel ? reinterpret_cast<const void *>(kernel) : reinterpret_cast<const void *>(kernel16);
  BL_CUDA(ensure_smem_limit(fn, kMaxSmem));
  const int64_t fit = kMaxSmem / (smem + 1024), per_sm = fit < 1 ? 1 : fit < 8 ? fit : 8;
  const int64_t want = (units + 7) / 8, cap = (per_sm * num_sms() + chunks - 1) / chunks;
  dim3 grid(unsigned(want < cap ? want : cap), unsigned(chunks));
  if (kernel)
    kernel<<<grid, 256, smem, as_stream(stream)>>>(weight, a, static_cast<float *>(out));
  else
    kernel16<<<grid, 256, smem, as_stream(stream)>>>(weight, a, static_cast<__nv_bfloat16 *>(out));
  BL_LAUNCH_CHECK();
  return BL_OK;
}

extern "C" int64_t bl_relative_position_encoding_workspace(int64_t batch, int64_t n, int64_t channels, int64_t r_max,
                                                           int64_t s_max) {
  if (batch <= 0 || n <= 0 || channels <= 0 || r_max < 0 || s_max < 0 || r_max > 96 || s_max > 16) return 0;
  const int rows = int(4 * r_max + 2 * s_max + 7), chunks = int((channels + 127) / 128);
  return encoding_grad_ctas(batch, n, rows, chunks) * chunks * rows * 128 * 4;
}

extern "C" int bl_relative_position_encoding_backward(const void *grad, int dtype, const int64_t *residue,
                                                      const int64_t *asym, const int64_t *entity, const int64_t *token,
                                                      const int64_t *sym, int64_t batch, int64_t n, int64_t channels,
                                                      int64_t r_max, int64_t s_max, int fix_sym, float *dweight,
                                                      void *workspace, int64_t workspace_bytes, void *stream) {
  EncArgs a{residue, asym, entity, token, sym, int(n), int(channels), int(4 * r_max + 2 * s_max + 7), int(r_max),
            int(s_max), fix_sym, batch};
  if (int rc = encoding_check("bl_relative_position_encoding_backward", a, n, channels, r_max, s_max)) return rc;
  BL_REQUIRE(dtype == BL_F32 || dtype == BL_BF16, "bl_relative_position_encoding_backward: dtype must be fp32 or bf16");
  BL_REQUIRE(dweight, "bl_relative_position_encoding_backward: null pointer");
  cudaStream_t st = as_stream(stream);
  if (batch == 0 || n == 0) {
    BL_CUDA(cudaMemsetAsync(dweight, 0, size_t(channels) * a.rows * 4, st));
    return BL_OK;
  }
  BL_REQUIRE(grad && aligned_to(grad, dtype == BL_F32 ? 8 : 4),
             "bl_relative_position_encoding_backward: null or unaligned pointer");
  const int64_t need = bl_relative_position_encoding_workspace(batch, n, channels, r_max, s_max);
  BL_REQUIRE(workspace && workspace_bytes >= need && aligned_to(workspace, 16),
             "bl_relative_position_encoding_backward: needs a workspace of %lld bytes", (long long)need);
  const int chunks = int((channels + 127) / 128), groups = encoding_grad_groups(a.rows);
  const int64_t ctas = encoding_grad_ctas(batch, n, a.rows, chunks);
  const int smem = groups * a.rows * 128 * 4;
  float *part = static_cast<float *>(workspace);
  dim3 grid{unsigned(ctas), unsigned(chunks)};
  if (dtype == BL_F32) {
    BL_CUDA(ensure_smem_limit(reinterpret_cast<const void *>(encoding_grad_kernel<float>), kMaxSmem));
    encoding_grad_kernel<float><<<grid, groups * 64, smem, st>>>(static_cast<const float *>(grad), a, part);
  } else {
    BL_CUDA(ensure_smem_limit(reinterpret_cast<const void *>(encoding_grad_kernel<__nv_bfloat16>), kMaxSmem));
    encoding_grad_kernel<__nv_bfloat16>
        <<<grid, groups * 64, smem, st>>>(static_cast<const __nv_bfloat16 *>(grad), a, part);
  }
  BL_LAUNCH_CHECK();
  const int64_t size = int64_t(chunks) * a.rows * 128;
  encoding_grad_sum_kernel<<<unsigned((size + 31) / 32), 256, 0, st>>>(part, int(ctas), chunks, a.rows, a.channels,
                                                                       dweight);
  BL_LAUNCH_CHECK();
  return BL_OK;
}

extern "C" int bl_relative_position_bias(const float *table, const int64_t *q_pos, const int64_t *k_pos, const int *lut,
                                         int64_t distance, const int64_t *q_group, const int64_t *k_group,
                                         int64_t batch, int64_t heads, int64_t nq, int64_t nk, int64_t buckets,
                                         void *out, int out_dtype, int64_t sb, int64_t sh, int64_t sq, void *stream) {
  BL_REQUIRE(nq < (1 << 30) && nk < (1 << 30) && heads < (1 << 20) && buckets < (1 << 20) && distance < (1 << 20),
             "bl_relative_position_bias: shape too large");
  BiasArgs a{q_pos, k_pos, q_group, k_group, lut, int(distance), int(buckets), int(heads), int(nq), int(nk), batch,
             sb, sh, sq};
  if (int rc = bias_check("bl_relative_position_bias", a)) return rc;
  BL_REQUIRE(out_dtype == BL_F32 || out_dtype == BL_BF16, "bl_relative_position_bias: dtype must be fp32 or bf16");
  if (batch == 0 || nq == 0 || nk == 0) return BL_OK;
  BL_REQUIRE(table && out, "bl_relative_position_bias: null pointer");
  const int smem = a.heads * a.buckets * 4 + bias_lut_bytes(a.distance);
  const int64_t col_blocks = (nk + kBiasCols - 1) / kBiasCols;
  // Query rows per CTA: about eight CTAs per SM in all, at most 32 rows each.
  const int64_t want = 8 * int64_t(num_sms());
  int64_t rows = (nq * col_blocks * batch + want - 1) / want;
  rows = rows < 1 ? 1 : rows > 32 ? 32 : rows;
  while ((nq + rows - 1) / rows > 65535) rows *= 2;
  dim3 grid{unsigned(col_blocks), unsigned((nq + rows - 1) / rows), unsigned(batch)};
  const int vec = vector_planes(out, a, out_dtype);
  if (out_dtype == BL_F32) {
    BL_CUDA(ensure_smem_limit(reinterpret_cast<const void *>(bias_kernel<float>), kMaxSmem));
    bias_kernel<float><<<grid, kBiasThreads, smem, as_stream(stream)>>>(table, a, static_cast<float *>(out), int(rows), vec);
  } else {
    BL_CUDA(ensure_smem_limit(reinterpret_cast<const void *>(bias_kernel<__nv_bfloat16>), kMaxSmem));
    bias_kernel<__nv_bfloat16>
        <<<grid, kBiasThreads, smem, as_stream(stream)>>>(table, a, static_cast<__nv_bfloat16 *>(out), int(rows), vec);
  }
  BL_LAUNCH_CHECK();
  return BL_OK;
}

extern "C" int64_t bl_relative_position_bias_workspace(int64_t batch, int64_t heads, int64_t nq, int64_t nk,
                                                       int64_t buckets) {
  if (batch <= 0 || heads <= 0 || heads > 1024 || nq <= 0 || nk <= 0 || buckets <= 0 || buckets > 256) return 0;
  const BiasGrad g = bias_grad_shape(batch, heads, nq, nk, int(buckets));
  return g.ctas * g.groups * buckets * g.per * 4;
}

extern "C" int bl_relative_position_bias_backward(const void *grad, int dtype, int64_t sb, int64_t sh, int64_t sq,
                                                  const int64_t *q_pos, const int64_t *k_pos, const int *lut,
                                                  int64_t distance, const int64_t *q_group, const int64_t *k_group,
                                                  int64_t batch, int64_t heads, int64_t nq, int64_t nk, int64_t buckets,
                                                  float *dtable, void *workspace, int64_t workspace_bytes,
                                                  void *stream) {
  BL_REQUIRE(nq < (1 << 30) && nk < (1 << 30) && heads < (1 << 20) && buckets < (1 << 20) && distance < (1 << 20),
             "bl_relative_position_bias_backward: shape too large");
  BiasArgs a{q_pos, k_pos, q_group, k_group, lut, int(distance), int(buckets), int(heads), int(nq), int(nk), batch,
             sb, sh, sq};
  if (int rc = bias_check("bl_relative_position_bias_backward", a)) return rc;
  BL_REQUIRE(dtype == BL_F32 || dtype == BL_BF16, "bl_relative_position_bias_backward: dtype must be fp32 or bf16");
  BL_REQUIRE(dtable, "bl_relative_position_bias_backward: null pointer");
  cudaStream_t st = as_stream(stream);
  if (batch == 0 || nq == 0 || nk == 0) {
    BL_CUDA(cudaMemsetAsync(dtable, 0, size_t(heads) * buckets * 4, st));
    return BL_OK;
  }
  const int64_t need = bl_relative_position_bias_workspace(batch, heads, nq, nk, buckets);
  BL_REQUIRE(grad && workspace && workspace_bytes >= need && aligned_to(workspace, 4),
             "bl_relative_position_bias_backward: needs grad and a workspace of %lld bytes", (long long)need);
  const BiasGrad shape = bias_grad_shape(batch, heads, nq, nk, a.buckets);
  const int per = shape.per, groups = shape.groups, rows = shape.rows;
  const int64_t ctas = shape.ctas;
  const int smem = a.buckets * per * kBiasThreads * 4 + bias_lut_bytes(a.distance);
  float *part = static_cast<float *>(workspace);
  const int vec = vector_planes(grad, a, dtype);
  dim3 grid{unsigned(ctas), unsigned(groups)};
#define BL_BIAS_GRAD(T, K)                                                                                        \
  do {                                                                                                            \
    BL_CUDA(ensure_smem_limit(reinterpret_cast<const void *>(bias_grad_kernel<T, K>), kMaxSmem));                     \
    bias_grad_kernel<T, K><<<grid, kBiasThreads, smem, st>>>(static_cast<const T *>(grad), a, rows, vec, part);   \
  } while (0)
  if (dtype == BL_F32) {
    if (per == 4) BL_BIAS_GRAD(float, 4); else BL_BIAS_GRAD(float, 1);
  } else {
    if (per == 4) BL_BIAS_GRAD(__nv_bfloat16, 4); else BL_BIAS_GRAD(__nv_bfloat16, 1);
  }
#undef BL_BIAS_GRAD
  BL_LAUNCH_CHECK();
  bias_grad_sum_kernel<<<unsigned((a.buckets * a.heads + 7) / 8), 256, 0, st>>>(part, int(ctas), a.buckets, a.heads, per,
                                                                              dtable);
  BL_LAUNCH_CHECK();
  return BL_OK;
}
