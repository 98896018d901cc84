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
// the upstream gradient once.  Encoding of 512 tokens, 128 fp32 channels: 31 us for 134 MB (4.3 TB/s; a plain
// fill of the same tensor 21 us; the table's load and the launch are the rest).  Its gradient at 424 tokens: 40 us
// for 92 MB, of which the partial sums' kernel is 4 us; six private tables of 36 KB leave six warps per SM, 1.5 per
// scheduler, whose latency is the limit: they issue in 25 % of the cycles, and of 6.0 cycles per issue 1.7 wait for an
// instruction's own latency, 1.5 for loads and 0.6 for shared memory (DRAM at 30 %).  Bias planes of 16 x 2048 x 8190 in bf16: 97 us for 537 MB (5.5 TB/s; a plain fill 74 to 90 us).
// Table gradient of 2 x 16 x 768 x 1134 fp32: 47 us for 112 MB, 12 us of it clearing and adding up the histograms.  The gradients are deterministic: every partial
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
// The features of a pair as loaded: looked at only later, so that the loads stay in flight.
struct PairFeatures {
  int64_t ri, rj, ai, aj, ei, ej, ti, tj, si, sj;
};
__device__ __forceinline__ PairFeatures pair_features(const EncArgs &a, int64_t i, int64_t j) {
  return {a.residue[i], a.residue[j], a.asym[i],  a.asym[j], a.entity[i],
          a.entity[j],  a.token[i],   a.token[j], a.sym[i],  a.sym[j]};
}
__device__ __forceinline__ uint32_t pick(const EncArgs &a, const PairFeatures &f) {
  const bool chain = f.ai == f.aj, agree = f.ei == f.ej;
  const uint32_t apart = 2 * a.r + 1;
  const uint32_t p = chain ? clip_offset(f.ri, f.rj, a.r) : apart;
  const uint32_t t = apart + 1 + (chain && f.ri == f.rj ? clip_offset(f.ti, f.tj, a.r) : apart);
  const bool other = a.fix_sym ? !agree : chain;
  const uint32_t c = 2 * (apart + 1) + 1 + (other ? 2 * a.s + 1 : clip_offset(f.si, f.sj, a.s));
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

__device__ __forceinline__ void put4(float *p, float4 y) { *reinterpret_cast<float4 *>(p) = y; }
__device__ __forceinline__ void put4(__nv_bfloat16 *p, float4 y) {
  *reinterpret_cast<uint2 *>(p) = make_uint2(pack_bf16x2(y.x, y.y), pack_bf16x2(y.z, y.w));
}

// kLanes lanes (4 channels each) per pair; a warp step writes 32 / kLanes
// pairs.  A warp takes 32 consecutive pairs of one row i: lane l computes the
// picks of pair j0 + l, the others receive them by shuffle.  The sum of the
// token, entity and chain rows repeats along most of a row, so it stays in
// registers: one shared load per pair and lane.
template <typename Out, int kLanes, bool kAdd>
__global__ void __launch_bounds__(1024) encoding_kernel(const float *w, const EncArgs a, Out *out) {
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
  auto hold = [&](uint32_t key) {
    held = key;
    base = add4(*reinterpret_cast<const float4 *>(col + (key & 1023u) * kLd),
                *reinterpret_cast<const float4 *>(col + ((key >> 10) & 1023u) * kLd));
    if (key >> 20) base = add4(base, *reinterpret_cast<const float4 *>(col + (4 * a.r + 4) * kLd));
  };
  auto write = [&](Out *p, uint32_t row) {
    float4 y = add4(*reinterpret_cast<const float4 *>(col + row * kLd), base);
    if constexpr (kAdd) y = add4(y, *reinterpret_cast<const float4 *>(p));
    put4(p, y);
  };
  for (uint32_t u = blockIdx.x * warps + (threadIdx.x >> 5); u < units; u += gridDim.x * warps) {
    const uint32_t row = u / uint32_t(segments);  // b * n + i
    const int j0 = int(u - row * segments) * 32;
    const int64_t i = row, b0 = row / uint32_t(n) * n;
    const int count = n - j0 < 32 ? n - j0 : 32;
    uint32_t mine = 0;
    if (lane < count) mine = pick(a, pair_features(a, i, b0 + j0 + lane));
    const uint32_t key = __shfl_sync(0xffffffffu, mine, 0) >> 10;
    Out *p = out + (i * n + j0 + sub) * a.channels + c0 + c;
    const int64_t step = int64_t(kPairs) * a.channels;
    if (count == 32 && __all_sync(0xffffffffu, (mine >> 10) == key)) {
      // One base for the whole segment.
      if (key != held) hold(key);
#pragma unroll 8
      for (int t = 0; t < 32; t += kPairs, p += step) {
        const uint32_t v = __shfl_sync(0xffffffffu, mine, t + sub) & 1023u;
        if (kLanes == 32 || live) write(p, v);
      }
    } else {
      for (int t = 0; t < count; t += kPairs, p += step) {
        const uint32_t v = __shfl_sync(0xffffffffu, mine, (t + sub) & 31);
        if (t + sub < count && live) {
          if ((v >> 10) != held) hold(v >> 10);
          write(p, v & 1023u);
        }
      }
    }
  }
}

// Gradient of W.  A warp covers 64 channels (two per lane) and owns a private
// [rows][64] table in shared memory, each element of which one lane alone
// updates.  It walks diagonals: from pair (i0, j) it visits (i0 + s, (j + s) mod n)
// for up to kSteps rows, every load a whole pair row, two walks' loads in flight at
// once.  Along a diagonal of one chain the offsets, so the picks, do not change: the
// sum of the pairs stays in registers and goes to the table rows of its picks when one
// of them changes.
// (128 channels per warp leave three warps per SM: 53 us at 424 tokens in fp32, 57 in bf16, against 40 and 39.)
constexpr int kGradCh = 64, kGroups = 6;  // private tables per CTA (36 KB each at r = 32, s = 2)
constexpr int kSteps = 16;

__device__ __forceinline__ float2 as_float2(float2 v) { return v; }
__device__ __forceinline__ float2 as_float2(uint32_t v) { return make_float2(bf16_lo(v), bf16_hi(v)); }
__device__ __forceinline__ float2 sum2(float2 a, float2 b) { return make_float2(a.x + b.x, a.y + b.y); }

template <typename In>
__global__ void __launch_bounds__(kGroups * 32) encoding_grad_kernel(const In *grad, const EncArgs a, float *partial) {
  constexpr int kS = kSteps;
  using Raw = typename std::conditional<sizeof(In) == 4, float2, uint32_t>::type;
  extern __shared__ float4 smem4[];
  float *tables = reinterpret_cast<float *>(smem4);
  const int groups = blockDim.x / 32, size = a.rows * kGradCh;
  for (int i = threadIdx.x; i < groups * size / 4; i += blockDim.x) smem4[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  __syncthreads();
  const int lane = threadIdx.x & 31, group = threadIdx.x / 32, ch = 2 * lane, c0 = blockIdx.y * kGradCh;
  const bool live = c0 + ch < a.channels;  // channels is a multiple of 4
  float2 *mine = reinterpret_cast<float2 *>(tables + group * size + ch);
  const int n = a.n, blocks = (n + kS - 1) / kS;
  const uint32_t units = uint32_t(a.batch * blocks * n);
  const int64_t step = (int64_t(n) + 1) * a.channels, wrap = int64_t(n) * a.channels;
  float2 run = make_float2(0.f, 0.f);
  uint32_t held = 0xffffffffu;
  auto put = [&](uint32_t row) { mine[row * 32] = sum2(mine[row * 32], run); };
  auto flush = [&]() {
    put(held & 1023u), put((held >> 10) & 1023u), put((held >> 20) & 1023u);
    if (held >> 30) put(4 * a.r + 4);
    run = make_float2(0.f, 0.f);
  };
  struct Walk {
    Raw x[kS];
    PairFeatures f;  // of step `lane`
    int count;
  };
  auto load = [&](uint32_t u, Walk &w) {
    const uint32_t ib = u / uint32_t(n), b = ib / uint32_t(blocks);
    const int j = int(u - ib * n), i0 = int(ib - b * blocks) * kS;
    const int64_t b0 = int64_t(b) * n;
    w.count = u >= units ? 0 : n - i0 < kS ? n - i0 : kS;
    const In *p = grad + ((b0 + i0) * n + j) * a.channels + c0 + ch;
    const int turn = n - j;  // first step past the row's end (s < count <= n: at most one turn)
    const int last = live ? w.count : 0;
    if (last == kS && turn >= kS) {
#pragma unroll
      for (int s = 0; s < kS; ++s, p += step) w.x[s] = __ldcs(reinterpret_cast<const Raw *>(p));
    } else {
#pragma unroll
      for (int s = 0; s < kS; ++s) {
        if (s == turn) p -= wrap;
        w.x[s] = {};
        if (s < last) w.x[s] = __ldcs(reinterpret_cast<const Raw *>(p));
        p += step;
      }
    }
    const int col = j + lane >= n ? j + lane - n : j + lane;
    if (lane < w.count) w.f = pair_features(a, b0 + i0 + lane, b0 + col);
  };
  auto sum = [&](const Walk &w) {
    if (w.count == 0) return;
    const uint32_t packed = lane < w.count ? pick(a, w.f) : 0u;
    const uint32_t first = __shfl_sync(0xffffffffu, packed, 0);
    if (__all_sync(0xffffffffu, lane >= w.count || packed == first)) {  // one pick for the walk (rows past it are zero)
      if (first != held) {
        if (held != 0xffffffffu) flush();
        held = first;
      }
      float2 part = make_float2(0.f, 0.f);
#pragma unroll
      for (int s = 0; s < kS; ++s) part = sum2(part, as_float2(w.x[s]));
      run = sum2(run, part);
    } else {
#pragma unroll
      for (int s = 0; s < kS; ++s) {
        if (s < w.count) {
          const uint32_t v = __shfl_sync(0xffffffffu, packed, s);
          if (v != held) {
            if (held != 0xffffffffu) flush();
            held = v;
          }
          run = sum2(run, as_float2(w.x[s]));
        }
      }
    }
  };
  const uint32_t hop = gridDim.x * groups;
  Walk one, two;
  uint32_t u = blockIdx.x * groups + group;
  load(u, one);
  for (; u < units; u += 2 * hop) {
    load(u + hop, two);
    sum(one);
    load(u + 2 * hop, one);
    sum(two);
  }
  if (held != 0xffffffffu) flush();
  __syncthreads();
  // partial[cta][channel chunk][row][kGradCh]
  float4 *dst = reinterpret_cast<float4 *>(partial + (int64_t(blockIdx.x) * gridDim.y + blockIdx.y) * size);
  for (int i = threadIdx.x; i < size / 4; i += blockDim.x) {
    float4 v = smem4[i];
    for (int g = 1; g < groups; ++g) v = add4(v, smem4[g * (size / 4) + i]);
    dst[i] = v;
  }
}

// dw[c][row] = sum over CTAs of partial[cta][c / kGradCh][row][c % kGradCh]; 8 threads per output, joined in a fixed order.
__global__ void __launch_bounds__(256) encoding_grad_sum_kernel(const float *partial, int ctas, int chunks, int rows,
                                                                int channels, float *dw) {
  __shared__ float part[8][33];
  const int lane = threadIdx.x & 31, way = threadIdx.x >> 5;
  const int64_t size = int64_t(chunks) * rows * kGradCh;
  const int64_t at = int64_t(blockIdx.x) * 32 + lane;
  float v = 0.f;
  if (at < size)
    for (int k = way; k < ctas; k += 8) v += partial[k * size + at];
  part[way][lane] = v;
  __syncthreads();
  if (way == 0 && at < size) {
    for (int k = 1; k < 8; ++k) v += part[k][lane];
    const int c = int(at / (int64_t(rows) * kGradCh)) * kGradCh + int(at % kGradCh), row = int(at / kGradCh % rows);
    if (c < channels) dw[int64_t(c) * rows + row] = v;
  }
}

int encoding_check(const char *name, const EncArgs &a, int64_t n, int64_t channels, int64_t r, int64_t s) {
  BL_REQUIRE(a.batch >= 0 && n >= 0 && n <= (1 << 15) && a.batch <= (1 << 20), "%s: bad shape", name);
  BL_REQUIRE(a.batch * n * ((n + 15) / 16) < (int64_t(1) << 30), "%s: too many token pairs", name);
  BL_REQUIRE(channels >= 4 && channels <= 4096 && channels % 4 == 0, "%s: channels must be a multiple of 4, at most 4096",
             name);
  BL_REQUIRE(r >= 0 && s >= 0 && r <= 96 && s <= 16, "%s: r_max must lie in [0, 96], s_max in [0, 16]", name);
  BL_REQUIRE(a.batch == 0 || n == 0 || (a.residue && a.asym && a.entity && a.token && a.sym), "%s: null pointer", name);
  return BL_OK;
}

int encoding_grad_groups(int rows) {  // private tables that fit in 227 KB
  const int fit = kMaxSmem / (rows * kGradCh * 4);
  return fit < kGroups ? fit : kGroups;
}
int64_t encoding_grad_ctas(int64_t batch, int64_t n, int rows, int chunks) {
  const int64_t units = batch * ((n + kSteps - 1) / kSteps) * n, groups = encoding_grad_groups(rows);
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
// Four key columns of one sample.  Positions relative to the sample's first key and groups as 32
// bits where they fit (`wide`: they do not, and are read again as 64 bits).
constexpr int kFits = 1 << 29;
struct Columns {
  int k[4], g[4];
  int64_t at;  // index of the first column
  int count;   // columns that exist
  bool wide;
};
__device__ __forceinline__ Columns load_columns(const BiasArgs &a, int64_t b, int j) {
  Columns c;
  c.at = b * a.nk + j;
  c.count = a.nk - j < 4 ? a.nk - j : 4;
  c.wide = false;
  const int64_t base = a.k_pos[b * a.nk];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int64_t at = c.at + (e < c.count ? e : 0), k = a.k_pos[at] - base, g = a.k_group ? a.k_group[at] : 0;
    c.k[e] = int(k), c.g[e] = int(g);
    c.wide |= k < -kFits || k > kFits || g != int64_t(int(g));
  }
  return c;
}
// Query rows [i0, i0 + rows) of sample b into shared memory: position relative to the sample's first
// key as 32 bits (saturated: at least kFits from any key that fits), group, whether the group fits.
__device__ __forceinline__ void load_rows_info(int4 *dst, const BiasArgs &a, int64_t b, int i0, int step, int rows) {
  const int64_t base = a.k_pos[b * a.nk];
  for (int r = threadIdx.x; r < rows; r += blockDim.x) {
    const int64_t at = b * a.nq + i0 + int64_t(r) * step, d = a.q_pos[at] - base, g = a.q_group ? a.q_group[at] : 0;
    const int q = d < -2 * int64_t(kFits) ? -2 * kFits : d > 2 * int64_t(kFits) - 1 ? 2 * kFits - 1 : int(d);
    dst[r] = make_int4(q, int(g), g == int64_t(int(g)), i0 + r * step);
  }
}
// Buckets of one query row.
__device__ __forceinline__ void buckets_of(int (&u)[4], const uint16_t *lut, const BiasArgs &a, const Columns &c, int64_t b,
                                           const int4 &r) {
  if (!c.wide) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int at = min(max(r.x - c.k[e], -a.distance), a.distance);
      u[e] = lut[a.distance + at];
      if (r.y != c.g[e] || !r.z) u[e] = a.buckets - 1;
    }
  } else {
    const int64_t q = a.q_pos[b * a.nq + r.w], g = a.q_group ? a.q_group[b * a.nq + r.w] : 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int64_t at = c.at + (e < c.count ? e : 0), d = q - a.k_pos[at];
      const int x = d < -a.distance ? 0 : d > a.distance ? 2 * a.distance : int(d) + a.distance;
      u[e] = !a.k_group || g == a.k_group[at] ? int(lut[x]) : a.buckets - 1;
    }
  }
}

// A thread keeps four key columns and their positions, computes their buckets
// once per query row and writes them for every head (16 or 8 bytes per store).
// The table sits in shared memory as [bucket][heads + 4]: one 16-byte load gives a
// column's value for four heads, and rows of different buckets start in different
// banks (heads a multiple of 8, padded: 4 (heads / 4 + 1) words apart, odd multiples
// of 4).  With [head][bucket] and a load per value the kernel took 28 instructions
// per store and 115 us for 537 MB.
constexpr int kBiasThreads = 128, kBiasCols = 4 * kBiasThreads;
constexpr int kRowsPerCta = 4;
constexpr int kBiasRows = 512;  // query rows whose positions sit in shared memory at a time

__host__ __device__ inline int table_ld(int heads) { return (heads + 7) / 8 * 8 + 4; }

template <typename Out>
__global__ void __launch_bounds__(kBiasThreads) bias_kernel(const float *table, const BiasArgs a, Out *out, int vector) {
  extern __shared__ float4 smem4[];
  const int ld = table_ld(a.heads);
  int4 *info = reinterpret_cast<int4 *>(smem4);
  float *tab = reinterpret_cast<float *>(info + kBiasRows);  // [buckets][ld]
  uint16_t *lut = reinterpret_cast<uint16_t *>(tab + a.buckets * ld);
  for (int i = threadIdx.x; i < a.heads * a.buckets; i += kBiasThreads) tab[i / a.heads * ld + i % a.heads] = table[i];
  load_lut(lut, a);
  // blockIdx.x keeps its column block and walks the rows r, r + runs, ...: the rows that all CTAs
  // write at a time are neighbours.
  const int64_t b = blockIdx.z;
  const int j = blockIdx.x * kBiasCols + 4 * threadIdx.x;
  const bool active = j < a.nk;
  Columns c{};
  if (active) c = load_columns(a, b, j);
  const bool whole = vector && c.count == 4;
  const int rows = (a.nq - int(blockIdx.y) + int(gridDim.y) - 1) / int(gridDim.y), full = a.heads & ~3;
  for (int r0 = 0; r0 < rows; r0 += kBiasRows) {
    const int now = rows - r0 < kBiasRows ? rows - r0 : kBiasRows;
    __syncthreads();
    load_rows_info(info, a, b, blockIdx.y + r0 * gridDim.y, gridDim.y, now);
    __syncthreads();
    if (!active) continue;
    for (int t = 0; t < now; ++t) {
      const int4 r = info[t];
      int u[4];
      buckets_of(u, lut, a, c, b, r);
      const float *row[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) row[e] = tab + u[e] * ld;
      Out *p = out + b * a.sb + int64_t(r.w) * a.sq + j;
      auto four = [&](int h, float (&v)[4][4]) {  // [head][column]
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float4 f = *reinterpret_cast<const float4 *>(row[e] + h);
          v[0][e] = f.x, v[1][e] = f.y, v[2][e] = f.z, v[3][e] = f.w;
        }
      };
      if (whole) {
#pragma unroll 4
        for (int h = 0; h < full; h += 4) {
          float v[4][4];
          four(h, v);
#pragma unroll
          for (int g = 0; g < 4; ++g, p += a.sh) put4(p, make_float4(v[g][0], v[g][1], v[g][2], v[g][3]));
        }
        if (full < a.heads) {
          float v[4][4];
          four(full, v);
#pragma unroll
          for (int g = 0; g < 3; ++g, p += a.sh)
            if (full + g < a.heads) put4(p, make_float4(v[g][0], v[g][1], v[g][2], v[g][3]));
        }
      } else {
        for (int h = 0; h < a.heads; ++h, p += a.sh)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (e < c.count) store_from_float(p + e, row[e][h]);
      }
    }
  }
}

// Four neighbouring elements of a row as loaded.
template <typename T> struct Quad;
template <> struct Quad<float> {
  using type = float4;
  static __device__ __forceinline__ float4 load(const float *p) { return __ldcs(reinterpret_cast<const float4 *>(p)); }
  static __device__ __forceinline__ float4 load_part(const float *p, int count) {
    return make_float4(p[0], count > 1 ? p[1] : 0.f, count > 2 ? p[2] : 0.f, count > 3 ? p[3] : 0.f);
  }
  static __device__ __forceinline__ float get(const float4 &v, int e) {
    return e == 0 ? v.x : e == 1 ? v.y : e == 2 ? v.z : v.w;
  }
};
template <> struct Quad<__nv_bfloat16> {
  using type = uint2;
  static __device__ __forceinline__ uint2 load(const __nv_bfloat16 *p) {
    return __ldcs(reinterpret_cast<const uint2 *>(p));
  }
  static __device__ __forceinline__ uint2 load_part(const __nv_bfloat16 *p, int count) {
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
// kVector: the four columns in one load (rows on 16-byte boundaries; 8 in bf16); else one by one.
// One row at a time with enough warps per SM: two rows ahead in registers took 36 against 32 us at
// 2 x 16 x 768 x 1024, and 67 against 45 us with unaligned rows (1134 keys).
template <typename In, int kHeads, bool kVector>
__global__ void __launch_bounds__(kBiasThreads) bias_grad_kernel(const In *grad, const BiasArgs a, int q_rows,
                                                                 float *partial) {
  using Four = typename Quad<In>::type;
  extern __shared__ float4 smem4[];
  int4 *info = reinterpret_cast<int4 *>(smem4);
  float *hist = reinterpret_cast<float *>(info + kBiasRows);
  uint16_t *lut = reinterpret_cast<uint16_t *>(hist + a.buckets * kHeads * kBiasThreads);
  for (int i = threadIdx.x; i < a.buckets * kHeads * kBiasThreads / 4; i += kBiasThreads)
    reinterpret_cast<float4 *>(hist)[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  load_lut(lut, a);
  float *mine = hist + threadIdx.x;
  const int h0 = blockIdx.y * kHeads, heads = a.heads - h0 < kHeads ? a.heads - h0 : kHeads;
  // A sample's columns in equal blocks of at most 128 x 4.
  const int quads = (a.nk + 3) / 4, col_blocks = (quads + kBiasThreads - 1) / kBiasThreads;
  const int width = (quads + col_blocks - 1) / col_blocks, row_blocks = (a.nq + q_rows - 1) / q_rows;
  const int64_t units = a.batch * col_blocks * row_blocks;
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int rb = int(u % row_blocks), cb = int(u / row_blocks % col_blocks);
    const int64_t b = u / row_blocks / col_blocks;
    const int i0 = rb * q_rows, rows = a.nq - i0 < q_rows ? a.nq - i0 : q_rows;
    const int j = 4 * (cb * width + int(threadIdx.x));
    const bool active = int(threadIdx.x) < width && j < a.nk;
    __syncthreads();
    load_rows_info(info, a, b, i0, 1, rows);
    __syncthreads();
    if (!active) continue;
    const Columns c = load_columns(a, b, j);
    int held[4];
    float run[4][kHeads];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      held[e] = -1;
#pragma unroll
      for (int h = 0; h < kHeads; ++h) run[e][h] = 0.f;
    }
    auto take = [&](int r, const Four (&x)[kHeads]) {
      int v[4];
      buckets_of(v, lut, a, c, b, info[r]);
      if (((v[0] ^ held[0]) | (v[1] ^ held[1]) | (v[2] ^ held[2]) | (v[3] ^ held[3])) != 0) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (v[e] != held[e]) {
            if (held[e] >= 0) {
              float *to = mine + held[e] * kHeads * kBiasThreads;
#pragma unroll
              for (int h = 0; h < kHeads; ++h) {
                to[h * kBiasThreads] += run[e][h];
                run[e][h] = 0.f;
              }
            }
            held[e] = v[e];
          }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int h = 0; h < kHeads; ++h) run[e][h] += Quad<In>::get(x[h], e);
    };
    const In *p = grad + b * a.sb + h0 * a.sh + int64_t(i0) * a.sq + j;
    for (int t = 0; t < rows; ++t, p += a.sq) {
      Four x[kHeads];
#pragma unroll
      for (int h = 0; h < kHeads; ++h) {
        x[h] = {};
        if (h < heads)
          x[h] = kVector && c.count == 4 ? Quad<In>::load(p + h * a.sh) : Quad<In>::load_part(p + h * a.sh, c.count);
      }
      take(t, x);
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
  // A thread sums a row of 128 in 16-byte steps, starting at a place of its own: no two lanes of a
  // phase meet in a bank.
  float *dst = partial + (int64_t(blockIdx.y) * gridDim.x + blockIdx.x) * a.buckets * kHeads;
  for (int k = threadIdx.x; k < a.buckets * kHeads; k += kBiasThreads) {
    const float4 *row = reinterpret_cast<const float4 *>(hist + k * kBiasThreads);
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int e = 0; e < kBiasThreads / 4; ++e) v = add4(v, row[(e + k) % (kBiasThreads / 4)]);
    dst[k] = (v.x + v.y) + (v.z + v.w);
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
// 2 KB (4 heads) or 0.5 KB (1) of histogram per bucket.  Four heads share the index work of a row while two CTAs fit an SM:
// 2 x 16 x 768 x 1134 fp32, cold, 33 buckets 58 us with four heads and 120 with one, 48 buckets 93 and 120, 65 to 92 buckets (one
// CTA per SM) 128 and 120.
int bias_grad_heads(int buckets) { return buckets <= 48 ? 4 : 1; }
// Launch shape of the table gradient: up to three CTAs per SM (67 KB of histogram at 33 buckets x 4 heads), each with
// one column block and one run of rows, in whole groups of four rows.
struct BiasGrad {
  int per, groups, rows;
  int64_t ctas;
};
BiasGrad bias_grad_shape(int64_t batch, int64_t heads, int64_t nq, int64_t nk, int buckets) {
  BiasGrad g;
  g.per = bias_grad_heads(buckets);
  g.groups = int((heads + g.per - 1) / g.per);
  const int64_t cols = batch * (((nk + 3) / 4 + kBiasThreads - 1) / kBiasThreads);
  const int64_t cap = (3 * num_sms() + g.groups - 1) / g.groups;
  int64_t runs = cap / cols;
  runs = runs < 1 ? 1 : runs > (nq + 7) / 8 ? (nq + 7) / 8 : runs;
  const int64_t rows = ((nq + runs - 1) / runs + 3) / 4 * 4;
  g.rows = int(rows > kBiasRows ? kBiasRows : rows);
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
  // One CTA per SM when wide: every CTA loads the table (71 KB), and three per SM spent 10 us at 512 tokens on it.
  const int threads = wide ? 1024 : 256, warps = threads / 32;
  const int64_t fit = kMaxSmem / (smem + 1024), per_sm = wide || fit < 1 ? 1 : fit < 8 ? fit : 8;
  const int64_t want = (units + warps - 1) / warps, cap = (per_sm * num_sms() + chunks - 1) / chunks;
  dim3 grid(unsigned(want < cap ? want : cap), unsigned(chunks));
  if (kernel)
    kernel<<<grid, threads, smem, as_stream(stream)>>>(weight, a, static_cast<float *>(out));
  else
    kernel16<<<grid, threads, smem, as_stream(stream)>>>(weight, a, static_cast<__nv_bfloat16 *>(out));
  BL_LAUNCH_CHECK();
  return BL_OK;
}

extern "C" int64_t bl_relative_position_encoding_workspace(int64_t batch, int64_t n, int64_t channels, int64_t r_max,
                                                           int64_t s_max) {
  if (batch <= 0 || n <= 0 || channels <= 0 || r_max < 0 || s_max < 0 || r_max > 96 || s_max > 16) return 0;
  const int rows = int(4 * r_max + 2 * s_max + 7), chunks = int((channels + kGradCh - 1) / kGradCh);
  return encoding_grad_ctas(batch, n, rows, chunks) * chunks * rows * kGradCh * 4;
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
  BL_REQUIRE(grad && aligned_to(grad, dtype == BL_F32 ? 16 : 8),
             "bl_relative_position_encoding_backward: null or unaligned pointer");
  const int64_t need = bl_relative_position_encoding_workspace(batch, n, channels, r_max, s_max);
  BL_REQUIRE(workspace && workspace_bytes >= need && aligned_to(workspace, 16),
             "bl_relative_position_encoding_backward: needs a workspace of %lld bytes", (long long)need);
  const int chunks = int((channels + kGradCh - 1) / kGradCh), groups = encoding_grad_groups(a.rows);
  const int64_t ctas = encoding_grad_ctas(batch, n, a.rows, chunks);
  const int smem = groups * a.rows * kGradCh * 4;
  float *part = static_cast<float *>(workspace);
  dim3 grid{unsigned(ctas), unsigned(chunks)};
  if (dtype == BL_F32) {
    BL_CUDA(ensure_smem_limit(reinterpret_cast<const void *>(encoding_grad_kernel<float>), kMaxSmem));
    encoding_grad_kernel<float><<<grid, groups * 32, smem, st>>>(static_cast<const float *>(grad), a, part);
  } else {
    BL_CUDA(ensure_smem_limit(reinterpret_cast<const void *>(encoding_grad_kernel<__nv_bfloat16>), kMaxSmem));
    encoding_grad_kernel<__nv_bfloat16>
        <<<grid, groups * 32, smem, st>>>(static_cast<const __nv_bfloat16 *>(grad), a, part);
  }
  BL_LAUNCH_CHECK();
  const int64_t size = int64_t(chunks) * a.rows * kGradCh;
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
  const int smem = kBiasRows * 16 + table_ld(a.heads) * a.buckets * 4 + bias_lut_bytes(a.distance);
  const int64_t col_blocks = (nk + kBiasCols - 1) / kBiasCols;
  // Four rows per CTA, fewer while that leaves SMs without eight CTAs.  (Long runs of rows write in
  // many places at once: filling the planes alone takes 90 us in runs of 28 rows, 77 us row by row.)
  const int64_t least = 8 * int64_t(num_sms()) / (col_blocks * batch);
  int64_t runs = (nq + kRowsPerCta - 1) / kRowsPerCta;
  runs = runs < least ? (least < nq ? least : nq) : runs;
  runs = runs > 65535 ? 65535 : runs;
  dim3 grid{unsigned(col_blocks), unsigned(runs), unsigned(batch)};
  const int vec = vector_planes(out, a, out_dtype);
  if (out_dtype == BL_F32) {
    BL_CUDA(ensure_smem_limit(reinterpret_cast<const void *>(bias_kernel<float>), kMaxSmem));
    bias_kernel<float><<<grid, kBiasThreads, smem, as_stream(stream)>>>(table, a, static_cast<float *>(out), vec);
  } else {
    BL_CUDA(ensure_smem_limit(reinterpret_cast<const void *>(bias_kernel<__nv_bfloat16>), kMaxSmem));
    bias_kernel<__nv_bfloat16>
        <<<grid, kBiasThreads, smem, as_stream(stream)>>>(table, a, static_cast<__nv_bfloat16 *>(out), vec);
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
  const int smem = kBiasRows * 16 + a.buckets * per * kBiasThreads * 4 + bias_lut_bytes(a.distance);
  float *part = static_cast<float *>(workspace);
  const int vec = vector_planes(grad, a, dtype);
  dim3 grid{unsigned(ctas), unsigned(groups)};
#define BL_BIAS_GRAD(T, K, V)                                                                                   \
  do {                                                                                                          \
    BL_CUDA(ensure_smem_limit(reinterpret_cast<const void *>(bias_grad_kernel<T, K, V>), kMaxSmem));            \
    bias_grad_kernel<T, K, V><<<grid, kBiasThreads, smem, st>>>(static_cast<const T *>(grad), a, rows, part);   \
  } while (0)
#define BL_BIAS_GRAD_BY(T)                                                                                      \
  do {                                                                                                          \
    if (per == 4) { if (vec) BL_BIAS_GRAD(T, 4, true); else BL_BIAS_GRAD(T, 4, false); }                        \
    else { if (vec) BL_BIAS_GRAD(T, 1, true); else BL_BIAS_GRAD(T, 1, false); }                                 \
  } while (0)
  if (dtype == BL_F32) BL_BIAS_GRAD_BY(float); else BL_BIAS_GRAD_BY(__nv_bfloat16);
#undef BL_BIAS_GRAD_BY
#undef BL_BIAS_GRAD
  BL_LAUNCH_CHECK();
  bias_grad_sum_kernel<<<unsigned((a.buckets * a.heads + 7) / 8), 256, 0, st>>>(part, int(ctas), a.buckets, a.heads, per,
                                                                              dtable);
  BL_LAUNCH_CHECK();
  return BL_OK;
}
