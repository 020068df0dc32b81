// Decode attention (one query token per sequence) over the 8-bit cache (layout: kv_fp8.cuh).
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
// of the scores, so that the largest weight is always 2^14 and what falls out of fp16's range is below 2^-38 of the largest term.  They are rounded to
// 11 bits.  The sum of the softmax runs beside it in fp32 against the maximum of the scores, by lane: only M has to be common to
// the lanes of a head while the walk lasts.
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
  int groups;                // of 8 H query heads per key head
  int splits;                // parts of a sequence: CTAs of a cluster
  float scale_log2;
  int* status;
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
template <int D, int H>
struct Kv8Heads {
  static constexpr int KS = D / 16;       // k steps of the first product, tiles of 16 dimensions of the second
  uint32_t qb[H][KS][2];
  float c[H][2];                          // score per unit of the product, in log2
  float o[H][KS][4];
  float top[H][2];                        // M
  float m[H][2], l[H][2];

  __device__ __forceinline__ void start(const __nv_bfloat16* q, int heads, float scale_log2, int lane) {
    const int g = lane >> 2, c4 = lane & 3;
#pragma unroll
    for (int h = 0; h < H; ++h) {
      const int head = 8 * h + g;
      float x[KS * 4], most = 0.f;
#pragma unroll
      for (int i = 0; i < KS / 2; ++i) {
        uint4 r = make_uint4(0, 0, 0, 0);
        if (head < heads) r = *reinterpret_cast<const uint4*>(q + head * D + c4 * (D / 4) + i * 8);
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
        for (int t = 0; t < 4; ++t) x[t] = in[t] ? s[t >> 1][h][2 * (t & 1) + e] * (f[t] * c[h][e]) : -INFINITY;
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

template <int D, int H, int WARPS>
__global__ void __launch_bounds__(32 * WARPS)
kv8_decode_kernel(const __grid_constant__ CUtensorMap map, const Kv8Decode p) {
  using Cfg = Kv8DecodeCfg<D, H, WARPS>;
  extern __shared__ uint8_t kv8_smem[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(kv8_smem) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::kMain);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = blockIdx.x % p.splits, unit = blockIdx.x / p.splits;
  const int group = unit % p.groups, kvh = unit / p.groups % p.Hkv, b = unit / p.groups / p.Hkv;
  const int R = p.Hq / p.Hkv, head0 = kvh * R + group * Cfg::kHeads, heads = min(Cfg::kHeads, R - group * Cfg::kHeads);
  uint64_t* full = bars + warp * kKv8Stages;
  if (lane == 0) {
    for (int s = 0; s < kKv8Stages; ++s) mbar_init(&full[s], 1);
    mbar_fence_init();
    tma_prefetch_desc(&map);
  }
  __syncwarp();
  pdl_entry();

  int len = p.lengths[b];
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
  Kv8Heads<D, H> acc;
  issue(0);
  acc.start(p.q + b * p.ldq + head0 * D, heads, p.scale_log2, lane);
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
    p.out[b * p.ldo + (head0 + head) * D + d] = __float2bfloat16(Kv8Final(top, m, l)(o));
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

template <int D, int H, int WARPS>
static int launch_kv8_decode(const CUtensorMap& map, const Kv8Decode& p, cudaStream_t s) {
  constexpr int smem = Kv8DecodeCfg<D, H, WARPS>::kSmem;
  static bool configured[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!configured[dev & 63]) {
    cudaError_t e = cudaFuncSetAttribute(kv8_decode_kernel<D, H, WARPS>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return static_cast<int>(e);
    configured[dev & 63] = true;
  }
  return static_cast<int>(launch_kernel_clusters(kv8_decode_kernel<D, H, WARPS>, dim3(p.B * p.Hkv * p.groups * p.splits), dim3(32 * WARPS), smem,
                                                 p.splits, s, map, p));
}

}  // namespace apb

extern "C" {
using namespace apb;

int apb_kv8_decode(const void* q, long long ldq, const void* data, const int* table, long long ld_table, int max_pages, int pages,
                   const int* lengths, void* out, long long ldo, int B, int Hq, int Hkv, int D, float scale, cudaStream_t s) {
  if (B <= 0) return 0;
  if ((D != 64 && D != 128) || Hkv < 1 || Hq % Hkv || pages < 1 || max_pages < 0 || static_cast<long long>(pages) * Hkv >= (1ll << 31) - 1 ||
      ldq % 8 || reinterpret_cast<uintptr_t>(q) % 16 || reinterpret_cast<uintptr_t>(data) % 16)
    return kBadArgument;
  const int R = Hq / Hkv, H = R > 8 ? 2 : 1, groups = (R + 8 * H - 1) / (8 * H);
  const long long units = static_cast<long long>(B) * Hkv * groups;
  int splits = 1;
  while (splits < 8 && units * splits * 2 <= 3 * sm_count() && splits * 8 < max_pages) splits *= 2;
  if (units * splits >= (1ll << 31)) return kBadArgument;
  CUtensorMap map;
  const int rc = kv8_map(&map, data, D, static_cast<long long>(pages) * Hkv);
  if (rc) return 1000 + rc;
  const Kv8Decode p = {static_cast<const __nv_bfloat16*>(q), ldq, static_cast<const uint8_t*>(data), table, ld_table, max_pages, pages, lengths,
                       static_cast<__nv_bfloat16*>(out), ldo, B, Hq, Hkv, groups, splits, scale * 1.4426950408889634f, status_device_ptr()};
  if (D == 128) return H == 1 ? launch_kv8_decode<128, 1, 4>(map, p, s) : launch_kv8_decode<128, 2, 4>(map, p, s);
  return H == 1 ? launch_kv8_decode<64, 1, 4>(map, p, s) : launch_kv8_decode<64, 2, 4>(map, p, s);
}
}
