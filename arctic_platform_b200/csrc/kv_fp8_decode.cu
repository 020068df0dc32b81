// Decode attention (one query token per sequence, or few of them: apb_kv8_few) over the 8-bit cache (layout: kv_fp8.cuh).
//
// Bound by the stream of codes: a page of 16 tokens and one key head is 32 D + 32 bytes that up to 16 query heads share.  A warp walks
// pages by itself, two at a time: a TMA copy brings a page's keys and values into its ring of shared memory (swizzled, so that the
// 16-byte reads below meet no bank twice) while the two before are worked on, the 32 exponents go to registers, a word per lane.
//
// Both products run on m16n8k16 MMAs in fp16, transposed: S^T = K Q^T and O^T += V^T W^T.  The 16 rows of a tile are tokens or
// dimensions, its 8 columns the heads of a group.  Codes become fp16 numbers exactly, by one instruction per pair; which dimension is
// which k index of the first product and which row of the second is free, so lanes take 16 neighbouring codes each and nothing is
// transposed in memory.  (The tcgen05 tile has 128 rows where a key head has 4 to 8 query heads.)
//
// fp16 holds codes, but not their scales: those stay outside the products.  Queries are scaled by a power of two per head so that the
// largest is about 2^14 (what fp16 drops is below 2^-38 of it); a score is (product) * 2^(key exponent) * constant.  A value's
// exponent belongs to its weight: with y = score + value exponent, weights are 2^(y - M + 14) against the running maximum M of y, not
// of the scores, so that the largest weight is always 2^14 and what falls out of fp16's range is below 2^-38 of the largest term.  They
// are rounded to 11 bits.  The sum of the softmax runs beside it in fp32 against the maximum of the scores, by lane: only M has to be
// common to the lanes of a head while the walk lasts.
//
// Measured: 128 sequences of 1365 to 4096 tokens, 32 / 8 heads of 128, 127 us (5.6 TB/s, 0.85 of a copy; the copies alone take 113); 2 of
// 36864, 32 / 4 heads, 23.2; 41 of 500 to 1500, 16 / 8 heads, 22.7; one of 384, 6.3.
#include <cuda_fp16.h>

#include "host_utils.cuh"
#include "kv_fp8.cuh"
#include "paged_mma.cuh"

namespace apb {

struct Kv8Decode {
  const __nv_bfloat16* q;    // [B, Hq, D], rows ldq elements apart
  long long ldq;
  const uint8_t* data;       // [pages, Hkv, block]
  const int* table;          // [B, max_pages], rows ld_table apart
  long long ld_table;
  int max_pages, pages;
  const int* lengths;        // [B]
  __nv_bfloat16* out;
  long long ldo;
  int B, Hq, Hkv;
  int groups;                // of 8 H query heads (ROWS: heads of some tokens) per key head
  int splits;                // parts of a sequence: CTAs of a cluster
  float scale_log2;
  int* status;
  const int* starts;         // ROWS [B + 1]: where the query tokens of a sequence begin in q and out
  const int* active;         // null, or [B]: sequences that are taken as empty where it is not above 0
  __device__ __forceinline__ int length(int b) const { return active && active[b] <= 0 ? 0 : lengths[b]; }
};

constexpr float kKv8Top = 14.f;          // log2 of the largest weight and (about) of the largest query element
constexpr int kKv8Stages = 2;            // of a warp's ring, two pages each
constexpr float kKv8None = -1.7e38f;     // a maximum of nothing: finite, so that differences of such are numbers

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <int D, int H, int WARPS>
struct Kv8DecodeCfg {
  static constexpr int kStage = 64 * D;                              // codes of two pages
  static constexpr int kRing = kKv8Stages * kStage;
  static constexpr int kHeads = 8 * H;
  static constexpr int kJoin = (WARPS + 1) * kHeads * (D + 4) * 4;   // the warps' results and the CTA's, in place of the rings
  static constexpr int kMain = WARPS * kRing > kJoin ? WARPS * kRing : kJoin;
  static constexpr int kSmem = kMain + WARPS * kKv8Stages * 8 + 1024;
};

// What a warp has of its heads: a lane has heads 2 (lane % 4) and the next of every group of 8, of them the dimensions
// D/8 (lane / 4) + [0, D/8) and the softmax sums of tokens lane / 4 and lane / 4 + 8 of its pages.
// ROWS: heads of several tokens, which differ in how many of the sequence's last tokens they do not see.
template <int D, int H, bool ROWS = false>
struct Kv8Heads {
  static constexpr int KS = D / 16;       // k steps of the first product, tiles of 16 dimensions of the second
  uint32_t qb[H][KS][2];
  float c[H][2];                          // score per unit of the product, in log2
  float o[H][KS][4];
  float top[H][2];                        // M
  float m[H][2], l[H][2];
  int unseen[ROWS ? H : 1][2];

  // q_of(head): where its query is
  template <typename Q>
  __device__ __forceinline__ void start(Q q_of, int heads, float scale_log2, int lane) {
    const int g = lane >> 2, c4 = lane & 3;
#pragma unroll
    for (int h = 0; h < H; ++h) {
      const int head = 8 * h + g;
      float x[KS * 4], most = 0.f;
#pragma unroll
      for (int i = 0; i < KS / 2; ++i) {
        uint4 r = make_uint4(0, 0, 0, 0);
        if (head < heads) r = *reinterpret_cast<const uint4*>(q_of(head) + c4 * (D / 4) + i * 8);
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          x[i * 8 + 2 * k] = __uint_as_float(w[k] << 16);
          x[i * 8 + 2 * k + 1] = __uint_as_float(w[k] & 0xFFFF0000u);
        }
      }
#pragma unroll
      for (int i = 0; i < KS * 4; ++i) most = fmaxf(most, fabsf(x[i]));
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
      const int e = max(static_cast<int>(__float_as_uint(most) >> 23) - 127, -100) - static_cast<int>(kKv8Top);
      const float f = exp2_int(-e);
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        qb[h][k][0] = pack_f16x2(x[4 * k] * f, x[4 * k + 1] * f);
        qb[h][k][1] = pack_f16x2(x[4 * k + 2] * f, x[4 * k + 3] * f);
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int e2 = __shfl_sync(0xffffffffu, e, 4 * (2 * c4 + k));
        c[h][k] = scale_log2 * exp2_int(e2);
        top[h][k] = m[h][k] = kKv8None;
        l[h][k] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < KS; ++i) o[h][i][0] = o[h][i][1] = o[h][i][2] = o[h][i][3] = 0.f;
    }
  }

  // The codes of two pages at `stage`, their exponents of tokens g and g + 8 in `ex` (255: no such page); `left` of their tokens
  // count.  Two at a time: the chains of one hide those of the other, and what is done once per maximum is done half as often.
  __device__ __forceinline__ void pages(uint32_t stage, const uint32_t (&ex)[2], int left, int lane) {
    const int g = lane >> 2, c4 = lane & 3;
    float s[2][H][4];
#pragma unroll
    for (int pg = 0; pg < 2; ++pg)
#pragma unroll
      for (int h = 0; h < H; ++h) s[pg][h][0] = s[pg][h][1] = s[pg][h][2] = s[pg][h][3] = 0.f;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      const int chunk = D == 128 ? (2 * c4 + i) ^ g : c4 ^ (g >> 1);
      uint4 lo[2], hi[2];
#pragma unroll
      for (int pg = 0; pg < 2; ++pg) {
        lo[pg] = lds128(stage + pg * 32 * D + g * D + chunk * 16);
        hi[pg] = lds128(stage + pg * 32 * D + (g + 8) * D + chunk * 16);
      }
#pragma unroll
      for (int w = 0; w < 4; ++w)
#pragma unroll
        for (int pg = 0; pg < 2; ++pg) {
          const uint32_t wl = w == 0 ? lo[pg].x : w == 1 ? lo[pg].y : w == 2 ? lo[pg].z : lo[pg].w;
          const uint32_t wh = w == 0 ? hi[pg].x : w == 1 ? hi[pg].y : w == 2 ? hi[pg].z : hi[pg].w;
          uint32_t a0, a1, a2, a3;
          e4m3x4_to_f16(wl, a0, a2);
          e4m3x4_to_f16(wh, a1, a3);
#pragma unroll
          for (int h = 0; h < H; ++h) mma_f16(s[pg][h], a0, a1, a2, a3, qb[h][4 * i + w][0], qb[h][4 * i + w][1]);
        }
    }
    // tokens g, g + 8 of the first page and of the second
    float f[4], y[4];
    bool in[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const uint32_t k = (ex[t >> 1] >> (8 * (t & 1))) & 255, v = (ex[t >> 1] >> (16 + 8 * (t & 1))) & 255;
      in[t] = g + 8 * t < left && k != 255;
      f[t] = __uint_as_float(k << 23);
      y[t] = static_cast<float>(static_cast<int>(v) - 127);
    }
    uint32_t pb[2][H][2];
#pragma unroll
    for (int h = 0; h < H; ++h) {
      float w[2][4], grown[2];
      bool grew = false;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float x[4], sum = 0.f;
#pragma unroll
        for (int t = 0; t < 4; ++t)
          x[t] = in[t] && (!ROWS || g + 8 * t < left - unseen[h][e]) ? s[t >> 1][h][2 * (t & 1) + e] * (f[t] * c[h][e]) : -INFINITY;
        const float m_new = fmaxf(fmaxf(m[h][e], fmaxf(x[0], x[1])), fmaxf(x[2], x[3]));
#pragma unroll
        for (int t = 0; t < 4; ++t) sum += ex2(x[t] - m_new);
        l[h][e] = l[h][e] * ex2(m[h][e] - m_new) + sum;
        m[h][e] = m_new;
#pragma unroll
        for (int t = 0; t < 4; ++t) x[t] += y[t];
        float mx = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
#pragma unroll
        for (int k = 4; k < 32; k <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, k));
        grown[e] = fmaxf(top[h][e], mx);
        grew |= grown[e] > top[h][e];
#pragma unroll
        for (int t = 0; t < 4; ++t) w[e][t] = ex2(x[t] - (grown[e] - kKv8Top));
      }
      if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float alpha = ex2(top[h][e] - grown[e]);
          top[h][e] = grown[e];
#pragma unroll
          for (int i = 0; i < KS; ++i) {
            o[h][i][e] *= alpha;
            o[h][i][2 + e] *= alpha;
          }
        }
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) pb[t >> 1][h][t & 1] = transpose_8x8(pack_f16x2(w[0][t], w[1][t]));
    }
#pragma unroll
    for (int pg = 0; pg < 2; ++pg) {
      // values of tokens 2 c4, 2 c4 + 1 and the same + 8
      constexpr int W = D / 32;             // words of a lane's dimensions
      uint32_t x[4][W];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int t = 2 * c4 + (k & 1) + 8 * (k >> 1);
        const uint32_t row = stage + pg * 32 * D + (16 + t) * D;
        if constexpr (D == 128) {
          const uint4 r = lds128(row + ((g ^ (t & 7)) << 4));
          x[k][0] = r.x, x[k][1] = r.y, x[k][2] = r.z, x[k][3] = r.w;
        } else {
          const uint2 r = lds64(row + (((g >> 1) ^ ((t >> 1) & 3)) << 4) + (g & 1) * 8);
          x[k][0] = r.x, x[k][1] = r.y;
        }
      }
      if (left < 32) {                // what lies behind the last token may be anything, and 0 times no number is none
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (16 * pg + 2 * c4 + (k & 1) + 8 * (k >> 1) >= left)
#pragma unroll
            for (int w = 0; w < W; ++w) x[k][w] = 0u;
      }
#pragma unroll
      for (int w = 0; w < W; ++w)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          uint32_t a0, a1, a2, a3;
          e4m3x4_to_f16(__byte_perm(x[0][w], x[1][w], u ? 0x7362 : 0x5140), a0, a1);
          e4m3x4_to_f16(__byte_perm(x[2][w], x[3][w], u ? 0x7362 : 0x5140), a2, a3);
#pragma unroll
          for (int h = 0; h < H; ++h) mma_f16(o[h][2 * w + u], a0, a1, a2, a3, pb[pg][h][0], pb[pg][h][1]);
        }
    }
  }

  // sums of a head over its lanes; m and l are then the same in all of them
  __device__ __forceinline__ void finish() {
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float mx = m[h][e];
#pragma unroll
        for (int k = 4; k < 32; k <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, k));
        float sum = l[h][e] * ex2(m[h][e] - mx);
#pragma unroll
        for (int k = 4; k < 32; k <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
        m[h][e] = mx;
        l[h][e] = sum;
      }
  }
};

// From numerators in units of 2^(M - 14) and a sum in units of 2^m to results.
struct Kv8Final {
  float f, inv;
  __device__ __forceinline__ Kv8Final(float top, float m, float l) {
    const bool some = l != 0.f;
    inv = some ? 1.f / l : 0.f;
    f = some ? exp2f((top - m - kKv8Top) * 0.5f) : 0.f;       // half of it: values may be far from 1
  }
  __device__ __forceinline__ float operator()(float o) const { return inv == 0.f ? 0.f : o * inv * f * f; }
};

// A warp's ring: copies of two pages each under way while the two before are worked on.
template <int D>
struct Kv8Copies {
  const CUtensorMap* map;
  const Kv8Decode& p;
  uint8_t* ring;
  uint64_t* full;
  int lane;
  __device__ __forceinline__ int checked(int id) const {
    if (static_cast<unsigned>(id) < static_cast<unsigned>(p.pages)) return id;
    if (p.status) atomicCAS(p.status, 0, kBadTable);
    return -1;
  }
  // copy number j, of pages id0 and (two) id1; `ex`: this lane's exponents, 255s where there is no page
  __device__ __forceinline__ void ask(int j, int id0, int id1, bool two, int kvh, uint32_t (&ex)[2]) const {
    const int block0 = id0 * p.Hkv + kvh, block1 = id1 * p.Hkv + kvh, behind = p.pages * p.Hkv;       // behind the cache are zeros
    if (lane == 0) {
      uint64_t* bar = &full[j % kKv8Stages];
      mbar_expect_tx(bar, (two ? 2 : 1) * 32 * D);
      tma_load_3d(ring + j % kKv8Stages * 64 * D, map, bar, 0, 0, id0 < 0 ? behind : block0);
      if (two) tma_load_3d(ring + j % kKv8Stages * 64 * D + 32 * D, map, bar, 0, 0, id1 < 0 ? behind : block1);
    }
    const uint8_t* at = p.data + 2 * Kv8<D>::kHalf + (lane & 28);
    ex[0] = id0 < 0 ? ~0u : __ldcg(reinterpret_cast<const uint32_t*>(at + static_cast<long long>(block0) * Kv8<D>::kBlock));
    ex[1] = !two || id1 < 0 ? ~0u : __ldcg(reinterpret_cast<const uint32_t*>(at + static_cast<long long>(block1) * Kv8<D>::kBlock));
  }
  __device__ __forceinline__ bool wait(int j) const {
    return __all_sync(0xffffffffu, mbar_wait(&full[j % kKv8Stages], (j / kKv8Stages) & 1, p.status, kTimeoutFull));
  }
  __device__ __forceinline__ uint32_t stage(int j) const { return smem_u32(ring) + j % kKv8Stages * 64 * D; }
  __device__ __forceinline__ void give_up() const {       // copies that are late may still write to the ring
    const uint64_t t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 100000ull) {
    }
  }
};

template <int D, int H, int WARPS, bool ROWS>
__global__ void __launch_bounds__(32 * WARPS)
kv8_decode_kernel(const __grid_constant__ CUtensorMap map, const Kv8Decode p) {
  using Cfg = Kv8DecodeCfg<D, H, WARPS>;
  extern __shared__ uint8_t kv8_smem[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(kv8_smem) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::kMain);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = blockIdx.x % p.splits, unit = blockIdx.x / p.splits;
  const int group = unit % p.groups, kvh = unit / p.groups % p.Hkv, b = unit / p.groups / p.Hkv;
  const int R = p.Hq / p.Hkv;
  uint64_t* full = bars + warp * kKv8Stages;
  if (lane == 0) {
    for (int s = 0; s < kKv8Stages; ++s) mbar_init(&full[s], 1);
    mbar_fence_init();
    tma_prefetch_desc(&map);
  }
  __syncwarp();
  pdl_entry();

  const int token0 = ROWS ? p.starts[b] : b, tokens = ROWS ? p.starts[b + 1] - token0 : 1;
  const int heads = min(Cfg::kHeads, tokens * R - group * Cfg::kHeads);
  if (heads <= 0) return;
  // of a head of the group: its token of the sequence's, its place among the key head's
  auto token_of = [&](int head) { return ROWS ? (group * Cfg::kHeads + head) / R : 0; };
  auto row_of = [&](int head, long long ld) {
    const int t = token_of(head);
    return (token0 + t) * ld + (kvh * R + group * Cfg::kHeads + head - t * R) * D;
  };
  int len = p.length(b);
  if (len > p.max_pages * kKv8Page) {
    if (threadIdx.x == 0 && p.status) atomicCAS(p.status, 0, kBadTable);
    len = p.max_pages * kKv8Page;
  }
  const int n_pages = (max(len, 0) + kKv8Page - 1) / kKv8Page, pairs = (n_pages + 1) / 2;
  const int per = (pairs + p.splits - 1) / p.splits, p0 = split * per, p1 = min(pairs, p0 + per);
  const int first = p0 + warp, n = (p1 - first + WARPS - 1) / WARPS;      // pairs of pages first, first + WARPS, ... (n <= 0: none)
  const int* table = p.table + b * p.ld_table;
  Kv8Copies<D> copies{&map, p, smem + warp * Cfg::kRing, full, lane};
  int ids = 0;                              // of pairs [j & ~15, + 16) of the walk, two lanes each
  uint32_t next[2] = {~0u, ~0u};
  auto issue = [&](int j) {
    if ((j & 15) == 0) {
      const int at = 2 * (first + (j + (lane >> 1)) * WARPS) + (lane & 1);
      ids = copies.checked(j + (lane >> 1) < n && at < n_pages ? table[at] : 0);
    }
    const int id0 = __shfl_sync(0xffffffffu, ids, 2 * (j & 15)), id1 = __shfl_sync(0xffffffffu, ids, 2 * (j & 15) + 1);
    if (j < n) copies.ask(j, id0, id1, 2 * (first + j * WARPS) + 1 < n_pages, kvh, next);
  };
  Kv8Heads<D, H, ROWS> acc;
  issue(0);
  acc.start([&](int head) { return p.q + row_of(head, p.ldq); }, heads, p.scale_log2, lane);
  if constexpr (ROWS) {
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
      for (int e = 0; e < 2; ++e) acc.unseen[h][e] = tokens - 1 - token_of(min(8 * h + 2 * (lane & 3) + e, heads - 1));
  }
  bool ok = true;
#pragma unroll 1
  for (int j = 0; j < n; ++j) {
    const uint32_t ex[2] = {next[0], next[1]};
    issue(j + 1);
    ok = copies.wait(j);
    if (!ok) break;
    acc.pages(copies.stage(j), ex, len - 2 * (first + j * WARPS) * kKv8Page, lane);
    __syncwarp();
  }
  if (!ok) copies.give_up();
  acc.finish();

  // the warps of the CTA, then the CTAs of the cluster
  __syncthreads();
  constexpr int kHeads = Cfg::kHeads;
  float* wo = reinterpret_cast<float*>(smem);                // [WARPS][kHeads][D]
  float* ws = wo + WARPS * kHeads * D;                       // [WARPS][kHeads][4]: M, m, l
  float* co = ws + WARPS * kHeads * 4;                       // [kHeads][D]
  float* cs = co + kHeads * D;                               // [kHeads][4]
#pragma unroll
  for (int h = 0; h < H; ++h)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int head = 8 * h + 2 * (lane & 3) + e, at = warp * kHeads + head;
      constexpr int N = D / 8;
      float* dst = wo + at * D + (lane >> 2) * N;
#pragma unroll
      for (int i = 0; i < N / 2; ++i) *reinterpret_cast<float2*>(dst + 2 * i) = make_float2(acc.o[h][i][e], acc.o[h][i][2 + e]);
      if (lane < 4) {
        ws[at * 4] = acc.top[h][e];
        ws[at * 4 + 1] = acc.m[h][e];
        ws[at * 4 + 2] = acc.l[h][e];
      }
    }
  __syncthreads();
  // joins `parts` results of one head and dimension, in the order of their places
  auto join = [&](int parts, auto top_of, auto m_of, auto l_of, auto o_of, float& top, float& m, float& l, float& o) {
    top = m = kKv8None;
    for (int k = 0; k < parts; ++k) top = fmaxf(top, top_of(k)), m = fmaxf(m, m_of(k));
    l = o = 0.f;
    for (int k = 0; k < parts; ++k) {
      const float lk = l_of(k);
      if (lk == 0.f) continue;                               // nothing seen
      const float mk = m_of(k), tk = top_of(k);
      l += lk * ex2(mk - m);
      o += o_of(k) * ex2(tk - top);
    }
  };
  auto finished = [&](int head, int d, float top, float m, float l, float o) {
    p.out[row_of(head, p.ldo) + d] = __float2bfloat16(Kv8Final(top, m, l)(o));
  };
  for (int i = threadIdx.x; i < heads * D; i += 32 * WARPS) {
    const int head = i / D, d = i % D;
    auto at = [&](int k) { return k * kHeads + head; };
    float top, m, l, o;
    join(WARPS, [&](int k) { return ws[at(k) * 4]; }, [&](int k) { return ws[at(k) * 4 + 1]; }, [&](int k) { return ws[at(k) * 4 + 2]; },
         [&](int k) { return wo[at(k) * D + d]; }, top, m, l, o);
    if (p.splits == 1) {
      finished(head, d, top, m, l, o);
    } else {
      co[i] = o;
      if (d == 0) cs[head * 4] = top, cs[head * 4 + 1] = m, cs[head * 4 + 2] = l;
    }
  }
  if (p.splits > 1) {
    cluster_sync_all();
    for (int i = threadIdx.x + split * 32 * WARPS; i < heads * D; i += p.splits * 32 * WARPS) {
      const int head = i / D, d = i % D;
      const uint32_t s_at = smem_u32(cs + head * 4), o_at = smem_u32(co + i);
      float top, m, l, o;
      join(p.splits, [&](int k) { return ld_cluster_f32(map_to_cta(s_at, k)); }, [&](int k) { return ld_cluster_f32(map_to_cta(s_at, k) + 4); },
           [&](int k) { return ld_cluster_f32(map_to_cta(s_at, k) + 8); }, [&](int k) { return ld_cluster_f32(map_to_cta(o_at, k)); }, top, m, l, o);
      finished(head, d, top, m, l, o);
    }
    cluster_sync_all();
  }
}

// All pages of all sequences in one row, cut into equal shares: a CTA walks its share through whichever units (sequence, key head, group
// of query heads) it meets, its warps take the pairs of pages of a unit in turn, and the copies of the next unit's pages are on
// their way while this one's results are joined.  A unit that lies in one share is finished there; of one that crosses borders every share
// leaves its part, and kv8_join_kernel joins them.
struct Kv8Parts {
  float *o, *s;               // [CTAs][2] rows: of the unit that began in front of the share, of one that goes on behind it; a row is
                              // [8 H][D] numerators, [8 H][4]: M, m, l
  int4* crossing;             // the unit that begins in a CTA and goes on behind it: sequence, unit of it, CTAs (0: none), the first of
                              // them; by CTA, or by unit where there are fewer of those
  bool by_unit;
  int least;                  // pages of a share at least
};
constexpr int kKv8Warps = 4;

template <int D, int H>
struct Kv8StreamCfg {
  static constexpr int kRing = kKv8Stages * 64 * D;
  static constexpr int kJoin = kKv8Warps * 4 * (D + 4) * 4;          // four heads of every warp
  static constexpr int kSmem = kKv8Warps * kRing + kJoin + kKv8Warps * kKv8Stages * 8 + 64 + 1024;
};

// Parts of a head added up, V dimensions a lane.
template <int V>
struct Kv8Joined {
  float top = kKv8None, m = kKv8None, l = 0.f, o[V] = {};
  __device__ __forceinline__ void add(const float4& s, const float (&v)[V]) {
    const float t1 = fmaxf(top, s.x), m1 = fmaxf(m, s.y), fo = ex2(top - t1), gn = ex2(s.x - t1);
    l = l * ex2(m - m1) + s.z * ex2(s.y - m1);
#pragma unroll
    for (int x = 0; x < V; ++x) o[x] = o[x] * fo + v[x] * gn;
    top = t1, m = m1;
  }
  __device__ __forceinline__ void store(__nv_bfloat16* out) const {
    const Kv8Final fin(top, m, l);
#pragma unroll
    for (int x = 0; x < V; x += 2) *reinterpret_cast<uint32_t*>(out + x) = pack_bf16x2(fin(o[x]), fin(o[x + 1]));
  }
};
template <int V>
__device__ __forceinline__ void kv8_load_part(const float* o, const float* sums, bool there, float4& s, float (&v)[V]) {
  s = make_float4(kKv8None, kKv8None, 0.f, 0.f);
#pragma unroll
  for (int x = 0; x < V; ++x) v[x] = 0.f;
  if (!there) return;
  s = __ldcg(reinterpret_cast<const float4*>(sums));
#pragma unroll
  for (int x = 0; x < V; x += 2) {
    const float2 y = __ldcg(reinterpret_cast<const float2*>(o + x));
    v[x] = y.x, v[x + 1] = y.y;
  }
}

template <int D, int H>
__global__ void __launch_bounds__(32 * kKv8Warps, H == 1 ? 3 : 2)
kv8_decode_stream_kernel(const __grid_constant__ CUtensorMap map, const Kv8Decode p, const Kv8Parts parts) {
  using Cfg = Kv8StreamCfg<D, H>;
  constexpr int kHeads = 8 * H, kThreads = 32 * kKv8Warps;
  extern __shared__ uint8_t kv8_smem[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(kv8_smem) + 1023) & ~uintptr_t(1023));
  float* jo = reinterpret_cast<float*>(smem + kKv8Warps * Cfg::kRing);          // [warps][4][D]
  float* js = jo + kKv8Warps * 4 * D;                                           // [warps][4][4]: M, m, l
  uint64_t* bars = reinterpret_cast<uint64_t*>(js + kKv8Warps * 4 * 4);
  // sequence that the share begins in, pages in front of it; sums of the warps
  int* found = reinterpret_cast<int*>(bars + kKv8Warps * kKv8Stages);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int R = p.Hq / p.Hkv, U = p.Hkv * p.groups;
  uint64_t* full = bars + warp * kKv8Stages;
  if (lane == 0) {
    for (int s = 0; s < kKv8Stages; ++s) mbar_init(&full[s], 1);
    mbar_fence_init();
    tma_prefetch_desc(&map);
  }
  pdl_entry();

  auto tokens_of = [&](int b) { return min(max(p.length(b), 0), p.max_pages * kKv8Page); };
  auto pages_of = [&](int b) { return (tokens_of(b) + kKv8Page - 1) / kKv8Page; };
  int from, to, share;        // this share; pages of all but the last ones
  {
    const int per = (p.B + kThreads - 1) / kThreads, b0 = min(p.B, static_cast<int>(threadIdx.x) * per), b1 = min(p.B, b0 + per);
    int mine = 0;
    for (int b = b0; b < b1; ++b) {
      mine += pages_of(b);
      if (p.length(b) > p.max_pages * kKv8Page && p.status) atomicCAS(p.status, 0, kBadTable);
    }
    int end = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, end, o);
      if (lane >= o) end += t;
    }
    if (lane == 31) found[2 + warp] = end;
    __syncthreads();
    int at = end - mine, total = 0;
#pragma unroll
    for (int k = 0; k < kKv8Warps; ++k) {
      if (k < warp) at += found[2 + k];
      total += found[2 + k];
    }
    total *= U;
    constexpr int kRound = 2 * kKv8Warps;            // pages that the warps take at a time
    const int even = (total + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x);
    share = (max(parts.least, even) + kRound - 1) / kRound * kRound;
    from = min(total, static_cast<int>(blockIdx.x) * share);
    to = min(total, from + share);
    if (from < to && at * U <= from && from < (at + mine) * U) {
      int b = b0;
      for (;; ++b) {
        const int np = pages_of(b);
        if (from < (at + np) * U) break;
        at += np;
      }
      found[0] = b;
      found[1] = at;
    }
    if (threadIdx.x == 0 && !parts.by_unit) parts.crossing[blockIdx.x] = make_int4(0, 0, 0, 0);
    for (int b = blockIdx.x; b < p.B; b += gridDim.x)       // sequences without tokens
      if (pages_of(b) == 0) {
        for (int i = threadIdx.x; i < p.Hq * D; i += kThreads) p.out[b * p.ldo + i] = __float2bfloat16(0.f);
        if (parts.by_unit)
          for (int i = threadIdx.x; i < U; i += kThreads) parts.crossing[b * U + i] = make_int4(0, 0, 0, 0);
      }
    __syncthreads();
    if (from == to) return;
  }
  // where a walk through the share is: pages [j, end) of unit u of sequence b, which has np pages; `left` pages of the share from j on
  struct Cursor {
    int b, u, j, np, left;
    __device__ __forceinline__ int pages() const { return min(np - j, left); }
  };
  Cursor c;
  c.b = found[0];
  c.np = pages_of(c.b);
  {
    const int in = from - found[1] * U;
    c.u = in / c.np;
    c.j = in - c.u * c.np;
    c.left = to - from;
  }
  auto next_unit = [&](Cursor& x) {           // there is one: pages of the share are left
    x.left -= x.pages();
    x.j = 0;
    if (x.left > 0 && ++x.u == U) {
      x.u = 0;
      do ++x.b;
      while ((x.np = pages_of(x.b)) == 0);
    }
  };
  Kv8Copies<D> copies{&map, p, smem + warp * Cfg::kRing, full, lane};
  Cursor f = c;               // of the copies
  int pair = warp, ids_at = -64, ids = 0, asked = 0;      // pair of f's pages; ids: of pairs [ids_at, + 64) by fours, two lanes each
  uint32_t next[2] = {~0u, ~0u};
  auto issue = [&]() {
    while (f.left > 0 && 2 * pair >= f.pages()) {
      next_unit(f);
      pair = warp;
      ids_at = -64;
    }
    if (f.left <= 0) return;
    const int n = f.pages();
    if (pair >= ids_at + 64) {
      ids_at = pair;
      const int at = 2 * (pair + (lane >> 1) * kKv8Warps) + (lane & 1);
      ids = copies.checked(at < n ? p.table[f.b * p.ld_table + f.j + at] : 0);
    }
    const int i = (pair - ids_at) / kKv8Warps * 2, id0 = __shfl_sync(0xffffffffu, ids, i), id1 = __shfl_sync(0xffffffffu, ids, i + 1);
    copies.ask(asked++, id0, id1, 2 * pair + 1 < n, f.u / p.groups, next);
    pair += kKv8Warps;
  };
  issue();
  Kv8Heads<D, H> acc;
  bool ok = true;
  int copy = 0, at = from;
  while (c.left > 0) {
    const int n = c.pages(), pairs = (n + 1) / 2, len = tokens_of(c.b);
    const int group = c.u % p.groups, head0 = c.u / p.groups * R + group * kHeads, heads = min(kHeads, R - group * kHeads);
    acc.start([&](int head) { return p.q + c.b * p.ldq + (head0 + head) * D; }, heads, p.scale_log2, lane);
#pragma unroll 1
    for (int k = warp; k < pairs && ok; k += kKv8Warps, ++copy) {
      const uint32_t ex[2] = {next[0], next[1]};
      issue();
      ok = copies.wait(copy);
      if (!ok) break;
      acc.pages(copies.stage(copy), ex, min(len - (c.j + 2 * k) * kKv8Page, (n - 2 * k) * kKv8Page), lane);
      __syncwarp();
    }
    acc.finish();
    const bool whole = n == c.np;
    const long long row0 = (static_cast<long long>(blockIdx.x) * 2 + (at - c.j < from ? 0 : 1)) * kHeads;
    // the warps' results, four heads at a time
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll 1
    for (int h4 = 8 * h; h4 < min(heads, 8 * h + 8); h4 += 4) {
      constexpr int N = D / 8;
      if ((lane & 3) / 2 == h4 / 4 % 2) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int row = warp * 4 + 2 * (lane & 1) + e;
          float* dst = jo + row * D + (lane >> 2) * N;
#pragma unroll
          for (int i = 0; i < N / 2; ++i) *reinterpret_cast<float2*>(dst + 2 * i) = make_float2(acc.o[h][i][e], acc.o[h][i][2 + e]);
          if (lane < 4) *reinterpret_cast<float4*>(js + row * 4) = make_float4(acc.top[h][e], acc.m[h][e], acc.l[h][e], 0.f);
        }
      }
      __syncthreads();
#pragma unroll
      for (int i = threadIdx.x; i < 4 * D; i += kThreads) {
        const int head = h4 + i / D, d = i % D;
        if (head >= heads) break;
        Kv8Joined<1> sum;
#pragma unroll
        for (int k = 0; k < kKv8Warps; ++k) {
          const float v[1] = {jo[k * 4 * D + i]};
          sum.add(*reinterpret_cast<const float4*>(js + (k * 4 + i / D) * 4), v);
        }
        if (whole) {
          p.out[c.b * p.ldo + (head0 + head) * D + d] = __float2bfloat16(Kv8Final(sum.top, sum.m, sum.l)(sum.o[0]));
        } else {
          parts.o[(row0 + head) * D + d] = sum.o[0];
          if (d == 0) *reinterpret_cast<float4*>(parts.s + (row0 + head) * 4) = make_float4(sum.top, sum.m, sum.l, 0.f);
        }
      }
      __syncthreads();
    }
    if (threadIdx.x == 0 && c.j == 0) {
      const int ctas = (at + c.np - 1) / share - static_cast<int>(blockIdx.x) + 1;
      if (parts.by_unit || ctas > 1)
        parts.crossing[parts.by_unit ? c.b * U + c.u : blockIdx.x] = make_int4(c.b, c.u, ctas > 1 ? ctas : 0, blockIdx.x);
    }
    at += n;
    next_unit(c);
  }
  if (!ok) copies.give_up();
}

// Joins the parts of the units that cross borders between CTAs; KB parts are loaded at a time.  WARPS > 1: a CTA per unit and head, its
// warps take the parts in turn and one joins theirs; else a warp per head.
template <int D, int H, int WARPS, int KB>
__global__ void __launch_bounds__(32 * (WARPS > 1 ? WARPS : 16)) kv8_join_kernel(const Kv8Decode p, const Kv8Parts parts) {
  pdl_wait();
  constexpr int kHeads = 8 * H, V = D / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int4 unit = __ldcg(parts.crossing + blockIdx.x);
  const int n = unit.z, R = p.Hq / p.Hkv, group = unit.y % p.groups, heads = min(kHeads, R - group * kHeads);
  const int head = WARPS > 1 ? blockIdx.y : warp, first = WARPS > 1 ? warp : 0;
  if (n == 0 || head >= heads) return;
  Kv8Joined<V> sum;
  for (int k0 = first; k0 < n; k0 += WARPS * KB) {
    float4 s[KB];
    float v[KB][V];
#pragma unroll
    for (int i = 0; i < KB; ++i) {
      const int k = k0 + WARPS * i;
      const long long row = ((static_cast<long long>(unit.w) + k) * 2 + (k == 0)) * kHeads + head;
      kv8_load_part<V>(parts.o + row * D + lane * V, parts.s + row * 4, k < n, s[i], v[i]);
    }
#pragma unroll
    for (int i = 0; i < KB; ++i) sum.add(s[i], v[i]);
  }
  if constexpr (WARPS > 1) {
    __shared__ float so[WARPS][D];
    __shared__ float4 ss[WARPS];
#pragma unroll
    for (int x = 0; x < V; ++x) so[warp][lane * V + x] = sum.o[x];
    if (lane == 0) ss[warp] = make_float4(sum.top, sum.m, sum.l, 0.f);
    __syncthreads();
    if (warp) return;
    for (int k = 1; k < WARPS; ++k) {
      float v[V];
#pragma unroll
      for (int x = 0; x < V; ++x) v[x] = so[k][lane * V + x];
      sum.add(ss[k], v);
    }
  }
  sum.store(p.out + unit.x * p.ldo + (unit.y / p.groups * R + group * kHeads + head) * D + lane * V);
}

// [blocks][32 rows of D codes]: what lies behind a block's codes is passed over
static int kv8_map(CUtensorMap* map, const void* data, int D, long long blocks) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) return -1;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(D), 32, static_cast<cuuint64_t>(blocks)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(32 * D + 32)};
  const cuuint32_t box[3] = {static_cast<cuuint32_t>(D), 32, 1}, one[3] = {1, 1, 1};
  return static_cast<int>(fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(data), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                             D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE));
}

template <int D, int H, int WARPS, bool ROWS = false>
static int launch_kv8_decode(const CUtensorMap& map, const Kv8Decode& p, cudaStream_t s) {
  constexpr int smem = Kv8DecodeCfg<D, H, WARPS>::kSmem;
  static bool configured[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!configured[dev & 63]) {
    cudaError_t e = cudaFuncSetAttribute(kv8_decode_kernel<D, H, WARPS, ROWS>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return static_cast<int>(e);
    configured[dev & 63] = true;
  }
  return static_cast<int>(launch_kernel_clusters(kv8_decode_kernel<D, H, WARPS, ROWS>, dim3(p.B * p.Hkv * p.groups * p.splits), dim3(32 * WARPS), smem,
                                                 p.splits, s, map, p));
}

// Places of a table that count: as many as a sequence of up to 2^31 tokens has, so that their tokens fit 32 bits.
static int table_width(int max_pages) { return max_pages < (1 << 27) ? max_pages : (1 << 27) - 1; }

// CTAs that a unit is cut into, of more than 4 pages, as long as all have a place.  An SM holds 3 (registers), 2 of heads of 128 with rows of
// several tokens in two groups.  Those in a second wave cost most of a walk: 10 x 4 tokens behind 1500, 32 / 8 heads of 128, 40 us as 320 CTAs
// and 32 as 160; 20 x 4 56 and 36.
static int kv8_splits(long long units, int longest, int places = 3) {
  int splits = 1;
  while (splits < 8 && units * splits * 2 <= places * sm_count() && splits * 8 < longest) splits *= 2;
  return splits;
}
static int kv8_stream_ctas(int H) { return sm_count() * (H == 1 ? 3 : 2); }

template <int D, int H>
static int launch_kv8_stream(const CUtensorMap& map, const Kv8Decode& p, const Kv8Parts& parts, cudaStream_t s) {
  constexpr int smem = Kv8StreamCfg<D, H>::kSmem;
  static bool configured[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!configured[dev & 63]) {
    cudaError_t e = cudaFuncSetAttribute(kv8_decode_stream_kernel<D, H>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return static_cast<int>(e);
    configured[dev & 63] = true;
  }
  const int ctas = kv8_stream_ctas(H);
  const int rc = static_cast<int>(launch_kernel(kv8_decode_stream_kernel<D, H>, dim3(ctas), dim3(32 * kKv8Warps), smem, s, map, p, parts));
  if (rc) return rc;
  const int heads = p.Hq / p.Hkv < 8 * H ? p.Hq / p.Hkv : 8 * H, units = p.B * p.Hkv * p.groups;
  if (parts.by_unit)          // parts of a unit: more than one on the mean
    return static_cast<int>(launch_kernel_after(kv8_join_kernel<D, H, 8, 8>, dim3(units, heads), dim3(256), 0, s, p, parts));
  return static_cast<int>(launch_kernel_after(kv8_join_kernel<D, H, 1, 2>, dim3(ctas), dim3(32 * heads), 0, s, p, parts));
}

}  // namespace apb

extern "C" {
using namespace apb;

// Bytes of scratch that apb_kv8_decode should get for sequences of up to `longest` pages; 0: none, a cluster per unit is sooner done.
//
// Times are counted in rounds, in which the four warps of a CTA take two pages each: a CTA of a unit walks its part of the longest sequence
// while others idle or wait for a place (a quarter of a walk where CTAs go in more than one wave and lengths differ); even shares
// cost all pages over all places and about 6 rounds for finding them, for the parts and for the join.  Measured, unit / shares, 32 / 8
// heads: 41 x 500..1500 tokens 22 / 28 us, 128 x 333..1000 41 / 49, 1 x 6000 11.6 / 13.0, 4 x 4000..12000 21.6 / 23.8; 1 x 36864 40.5 /
// 21.5, 16 x 4000..12000 57 / 54, 64 x 1667..5000 93 / 83; 32 / 4 heads, 2 x 36864 42 / 23.
long long apb_kv8_decode_scratch(int B, int longest, int Hq, int Hkv, int D) {
  const int R = Hq / Hkv, H = R > 8 ? 2 : 1, places = kv8_stream_ctas(H);
  const double units = static_cast<double>(B) * Hkv * ((R + 8 * H - 1) / (8 * H));
  const int splits = kv8_splits(static_cast<long long>(units), longest);
  const double walk = longest / (8.0 * splits), waves = units * splits / places;
  const double unit = walk * (waves > 1 ? waves + 0.25 : 1.0), shares = units * longest / (8.0 * places) + 6.0;
  return unit <= shares ? 0 : static_cast<long long>(places) * (2 * 8 * H * (D + 4) * 4 + 16);
}

// scratch: null, or what apb_kv8_decode_scratch says; active: null, or [B], sequences without are taken as empty
int apb_kv8_decode(const void* q, long long ldq, const void* data, const int* table, long long ld_table, int max_pages, int pages,
                   const int* lengths, const int* active, void* out, long long ldo, int B, int longest, int Hq, int Hkv, int D, float scale,
                   void* scratch, cudaStream_t s) {
  if (B <= 0) return 0;
  if ((D != 64 && D != 128) || Hkv < 1 || Hq % Hkv || pages < 1 || max_pages < 0 || static_cast<long long>(pages) * Hkv >= (1ll << 31) - 1 ||
      ldq % 8 || ldo % 2 || reinterpret_cast<uintptr_t>(q) % 16 || reinterpret_cast<uintptr_t>(out) % 4 || reinterpret_cast<uintptr_t>(data) % 16 ||
      reinterpret_cast<uintptr_t>(scratch) % 16)
    return kBadArgument;
  max_pages = table_width(max_pages);
  const int R = Hq / Hkv, H = R > 8 ? 2 : 1, groups = (R + 8 * H - 1) / (8 * H);
  const long long units = static_cast<long long>(B) * Hkv * groups;
  CUtensorMap map;
  const int rc = kv8_map(&map, data, D, static_cast<long long>(pages) * Hkv);
  if (rc) return 1000 + rc;
  Kv8Decode p = {static_cast<const __nv_bfloat16*>(q), ldq, static_cast<const uint8_t*>(data), table, ld_table, max_pages, pages, lengths,
                 static_cast<__nv_bfloat16*>(out), ldo, B, Hq, Hkv, groups, 1, scale * 1.4426950408889634f, status_device_ptr(), nullptr,
                 active};
  if (scratch && units * max_pages < (1ll << 30)) {          // shares count pages in 32 bits, of as many as a table could name
    const long long rows = static_cast<long long>(kv8_stream_ctas(H)) * 2 * 8 * H;
    Kv8Parts parts;
    parts.o = static_cast<float*>(scratch);
    parts.s = parts.o + rows * D;
    parts.crossing = reinterpret_cast<int4*>(parts.s + rows * 4);
    parts.by_unit = units * 4 <= kv8_stream_ctas(H);
    parts.least = 2 * kKv8Warps;
    if (D == 128) return H == 1 ? launch_kv8_stream<128, 1>(map, p, parts, s) : launch_kv8_stream<128, 2>(map, p, parts, s);
    return H == 1 ? launch_kv8_stream<64, 1>(map, p, parts, s) : launch_kv8_stream<64, 2>(map, p, parts, s);
  }
  p.splits = kv8_splits(units, longest);
  if (units * p.splits >= (1ll << 31)) return kBadArgument;
  if (D == 128) return H == 1 ? launch_kv8_decode<128, 1, 4>(map, p, s) : launch_kv8_decode<128, 2, 4>(map, p, s);
  return H == 1 ? launch_kv8_decode<64, 1, 4>(map, p, s) : launch_kv8_decode<64, 2, 4>(map, p, s);
}

// Attention of few query tokens of each sequence, causal, 16 of them times the query heads of a key head at most: sequence b has those from
// starts[b] to starts[b + 1], at the end of its lengths[b] tokens, `most` at most; q, out [rows, Hq, D].  A unit's rows are then heads of
// several tokens.  (A third group of 8 rows was slower than 128-row tiles: 20 rows, 16 x 1500 tokens 33 us against 27.)
int apb_kv8_few(const void* q, long long ldq, const void* data, const int* table, long long ld_table, int max_pages, int pages, const int* lengths,
                const int* starts, void* out, long long ldo, int B, int most, int longest, int Hq, int Hkv, int D, float scale, cudaStream_t s) {
  if (B <= 0 || most <= 0) return 0;
  if ((D != 64 && D != 128) || Hkv < 1 || Hq % Hkv || pages < 1 || max_pages < 0 || static_cast<long long>(pages) * Hkv >= (1ll << 31) - 1 ||
      ldq % 8 || reinterpret_cast<uintptr_t>(q) % 16 || reinterpret_cast<uintptr_t>(data) % 16)
    return kBadArgument;
  const long long rows = static_cast<long long>(most) * (Hq / Hkv), units = static_cast<long long>(B) * Hkv;
  if (rows > 16) return kBadArgument;
  max_pages = table_width(max_pages);
  CUtensorMap map;
  const int rc = kv8_map(&map, data, D, static_cast<long long>(pages) * Hkv);
  if (rc) return 1000 + rc;
  Kv8Decode p = {static_cast<const __nv_bfloat16*>(q), ldq, static_cast<const uint8_t*>(data), table, ld_table, max_pages, pages, lengths,
                 static_cast<__nv_bfloat16*>(out), ldo, B, Hq, Hkv, 1, kv8_splits(units, longest, rows > 8 && D == 128 ? 2 : 3),
                 scale * 1.4426950408889634f, status_device_ptr(), starts, nullptr};
  if (units * p.splits >= (1ll << 31)) return kBadArgument;
  if (D == 128) return rows <= 8 ? launch_kv8_decode<128, 1, 4, true>(map, p, s) : launch_kv8_decode<128, 2, 4, true>(map, p, s);
  return rows <= 8 ? launch_kv8_decode<64, 1, 4, true>(map, p, s) : launch_kv8_decode<64, 2, 4, true>(map, p, s);
}
}
