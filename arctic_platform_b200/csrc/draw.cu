// Tokens drawn from rows of logits with given random numbers: temperature, top-k, min-p, top-p, then the first token, in the order of the
// vocabulary, at which the running mass of what stays passes u of the whole.
//
// Mathematics.  Every restriction keeps the logits from a threshold on, so a row comes down to one threshold: the top_k-th largest logit; the
// least logit with exp((l - max) / T) >= min_p; the least logit of which the strictly larger ones hold less than top_p of what stayed so far.
// Masses and their sums are 64-bit numbers: an fp32 running sum is off by 2^-24 of itself at best, a hundredth of one token's mass in a flat row
// of 151936, which would put one draw of a hundred on the neighbour's side of a border.  Nothing is added by floating atomics, so that the same
// numbers give the same token every time.
//
// Layout.  One CTA of 32 warps a row, or a cluster of 2, 4 or 8 where the rows leave SMs idle.  One walk reads a part from global memory, finds the
// largest logit and adds up the masses (of exp(l / T) itself: 64-bit numbers have the range, so nothing waits for the largest); a warp has a
// contiguous range, so that a draw from the whole distribution is then a search in 32 sums, in the 32 of that range and in some
// hundred elements.  A part that fits shared memory is kept there for further walks, a longer one is read again from L2.  A threshold is found
// by histograms that the CTAs of a cluster read from one another; where one CTA has a long row, only of what lies near it, as a sample tells.
//
// Measured: 128 rows of 151936 in fp32 from the whole distribution 31 us (2.5 TB/s; the first walk, where 64-bit arithmetic and loads meet, three
// quarters of it), with a nucleus of 0.95 104 us (chains of short steps of one CTA behind two walks), one row of 151936 in a cluster of 8
// 19 us (latency).
#include "common.cuh"
#include "draw_noise.cuh"
#include "host_utils.cuh"

namespace apb {

constexpr int kDrawThreads = 1024;
constexpr int kDrawWarps = kDrawThreads / 32;
constexpr int kDrawClasses = 2048;
constexpr int kDrawPer = kDrawClasses / kDrawThreads;      // classes of a thread
constexpr int kDrawLanes = kDrawThreads / 256;             // threads that compare one element with its class
constexpr int kDrawRanges = kDrawWarps / 4;                // ranges of a lane, of those of 8 parts
constexpr int kDrawBatch = 8;              // elements of a lane in flight in the first walk
constexpr int kDrawGroup = 4;             // elements of a lane side by side in later ones: longer code does not fit the instruction cache
constexpr int kDrawFew = 256;             // elements of a class that are compared with one another
constexpr int kDrawKept = 24 * 1024;      // elements of a part that is kept in shared memory
constexpr int kDrawBytes = 176 * 1024;    // shared memory for the part and for the lists of elements that a nucleus can reach
constexpr int kDrawMost = 3 << 17;        // elements of a row: units of 2^-45 of their masses add up in 64 bits, limbs of 12 bits in 32

struct DrawArgs {
  const void* logits;
  long long ld;
  const float* temperature;   // [B] each, or null: the same number for all rows
  const int* top_k;
  const float* top_p;
  const float* min_p;
  float temperature_all, top_p_all, min_p_all;
  int top_k_all;
  const void* u;              // [B] fp32 or fp64; null: noise of every token by a hash of (seed, step, row, token)
  const int* step;            // on the device, with `seed_dev` too: a captured launch sees new values
  const int* seed_dev;        // or null: `seed`
  uint32_t seed;
  int u64;
  int V, parts, per, room;    // per: elements of a part; room: of a lane's list
  int* tokens;
  float* logprobs;
};

__device__ __forceinline__ uint32_t draw_key(float z) {      // larger logit, larger key
  const uint32_t u = __float_as_uint(z);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float draw_unkey(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }
__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ unsigned long long ld_cluster_u64(uint32_t a) {
  unsigned long long v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ unsigned long long warp_scan_u64(unsigned long long v, int lane) {     // sum up to and with this lane
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long t = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += t;
  }
  return v;
}

// One value of every warp of the row: lane w of v[p] has that of warp w of part p (`none` behind the last part).
__device__ __forceinline__ void row_f32(const float (&own)[kDrawWarps], int parts, int lane, float none, float (&v)[8]) {
#pragma unroll
  for (int p = 0; p < 8; ++p) v[p] = p < parts && lane < kDrawWarps ? ld_cluster_f32(map_to_cta(smem_u32(&own[lane]), p)) : none;
}
__device__ __forceinline__ float row_max(const float (&own)[kDrawWarps], int parts, int lane) {
  float v[8];
  row_f32(own, parts, lane, -INFINITY, v);
  return warp_max(fmaxf(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), fmaxf(fmaxf(v[4], v[5]), fmaxf(v[6], v[7]))));
}
__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ double warp_scan_f64(double v, int lane) {      // sum up to and with this lane
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double t = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += t;
  }
  return v;
}
__device__ __forceinline__ double row_sum(const double (&own)[kDrawWarps], int parts, int lane) {
  double v[8], s = 0;
#pragma unroll
  for (int p = 0; p < 8; ++p)
    v[p] = p < parts && lane < kDrawWarps ? __longlong_as_double(ld_cluster_u64(map_to_cta(smem_u32(&own[lane]), p))) : 0.0;
#pragma unroll
  for (int p = 0; p < 8; ++p) s += v[p];
  return warp_sum_f64(s);
}
__device__ __forceinline__ int row_min(const int (&own)[kDrawWarps], int parts, int lane) {
  int s = 0x7fffffff;
#pragma unroll
  for (int p = 0; p < 8; ++p)
    if (p < parts && lane < kDrawWarps) s = min(s, static_cast<int>(ld_cluster_u32(map_to_cta(smem_u32(&own[lane]), p))));
  return __reduce_min_sync(0xffffffffu, s);
}
__device__ __forceinline__ void row_sync(int parts) {       // the CTAs of a row; what they wrote to their shared memory is there
  if (parts > 1) cluster_sync_all();
  else __syncthreads();
}

// exp2(x / 64) of a 64-bit number, x from -2^16 to 2^16: x split into a whole number, whose power is a table's and an exponent, and a rest of at
// most 1/2, whose power is its series to the third term (the fourth is below 4e-11 of the result).  The high word of a table's entry is less by
// its index at the place from which the shifted whole number carries into the exponent, so that one addition sets both.  7 operations in 64
// bits with the addition of the result to a sum.  The table has a copy for every two lanes: a load takes 2 passes through shared
// memory, where one table of 1024 entries and a series shorter by a term takes 6 and no less time in all.
struct DrawPower {
  double y, power;                        // the result is their product
};
__device__ __forceinline__ DrawPower draw_power(double l, double scale, const double* table) {      // x = l scale; table: this lane's
  constexpr double kShift = 6755399441055744.0;                    // 1.5 2^52: adding it leaves the nearest whole number in the low bits
  constexpr double kA = 0.69314718055994530942 / 64;
  const double t = fma(l, scale, kShift);
  const int k = __double2loint(t);
  const double r = fma(l, scale, kShift - t);
  const double e = table[(k & 63) << 4];
  return {fma(r, fma(r, fma(r, kA * kA * kA / 6, kA * kA / 2), kA), 1.0),
          __hiloint2double(__double2hiint(e) + (k << 14), __double2loint(e))};
}

template <typename T>
__device__ __forceinline__ float draw_logit(T x) {
  const float z = static_cast<float>(x);
  return z == z ? z : -INFINITY;          // what is not a number is never drawn
}

struct DrawShared {
  double table[64][16];                     // 2^(j / 64), the high word less by j << 14; a copy for every two lanes: their own banks
  uint32_t hist[4][kDrawClasses];           // of the classes: limbs of the masses, or elements
  float list[2][kDrawFew];                  // this CTA's elements of the class that holds a threshold (by rank, by mass)
  float all[kDrawFew];                      // the row's
  unsigned long long weight[kDrawFew];
  double warp_mass[2][kDrawWarps], sub[kDrawWarps], before;
  unsigned long long scan[kDrawWarps], above;
  float warp_f[2][kDrawWarps], warp_key[kDrawWarps];
  int warp_i[kDrawWarps];
  int list_n[2], limb[2], warp_n[kDrawWarps], chosen, owner;
};

constexpr int kDrawShared = (sizeof(DrawShared) + 15) / 16 * 16;
static_assert(kDrawShared + kDrawBytes <= 227 * 1024, "shared memory of one CTA");

// This CTA's part of a row: `n` elements from `src` on, KEPT: in shared memory, element i at z[i].  16-byte words of the row: the first
// one begins at element `head`.
template <typename T, bool KEPT>
struct DrawRow {
  static constexpr int kVec = 16 / sizeof(T);
  const T* src;
  float* z;
  int n, parts, head, words;
  float m, cut;        // cut: below it a mass is nothing
  double scale;        // 64 log2(e) / T
  const double* table;
  bool flat;           // the largest logit is infinite: equal ones stand for 0, all others for -inf

  __device__ __forceinline__ float seen(float l) const { return flat ? (l == INFINITY ? 0.f : -INFINITY) : l; }
  __device__ __forceinline__ float at(int i) const { return seen(KEPT ? z[i] : draw_logit(src[i])); }
  __device__ __forceinline__ void word(int w, float (&l)[kVec]) const {
    if constexpr (KEPT) {
      const float4* f = reinterpret_cast<const float4*>(z + head + w * kVec);
#pragma unroll
      for (int j = 0; j < kVec; j += 4) {
        const float4 v = f[j / 4];
        l[j] = v.x;
        l[j + 1] = v.y;
        l[j + 2] = v.z;
        l[j + 3] = v.w;
      }
    } else {
      const uint4 raw = reinterpret_cast<const uint4*>(src + head)[w];
      const T* x = reinterpret_cast<const T*>(&raw);
#pragma unroll
      for (int j = 0; j < kVec; ++j) l[j] = draw_logit(x[j]);
    }
  }
  // Elements of a warp: whole words, the first warp's range begins with the elements in front of them, the last one's ends with those behind.
  __device__ __forceinline__ int per_warp() const { return (words + kDrawWarps - 1) / kDrawWarps; }
  __device__ __forceinline__ int from(int warp) const { return warp == 0 ? 0 : head + min(warp * per_warp(), words) * kVec; }
  __device__ __forceinline__ int to(int warp) const { return warp == kDrawWarps - 1 ? n : head + min((warp + 1) * per_warp(), words) * kVec; }
  // f(logits) over the elements of this warp, kDrawGroup of a lane at a time, two words on their way meanwhile; places behind the last hold
  // `none`
  template <typename F>
  __device__ __forceinline__ void walk(int warp, int lane, float none, F f) const {
    const int w1 = min((warp + 1) * per_warp(), words);
    int w = min(warp * per_warp(), words) + lane;
    float next[2][kVec];
    if (w < w1) word(w, next[0]);
    if (w + 32 < w1) word(w + 32, next[1]);
#pragma unroll 1
    for (; w < w1; w += 32) {
      float x[kVec];
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        x[j] = next[0][j];
        next[0][j] = next[1][j];
      }
      if (w + 64 < w1) word(w + 64, next[1]);
#pragma unroll
      for (int g = 0; g < kVec; g += kDrawGroup) {
        float l[kDrawGroup];
#pragma unroll
        for (int j = 0; j < kDrawGroup; ++j) l[j] = seen(x[g + j]);
        f(l);
      }
    }
    const int tail = head + words * kVec;
    const int edge = warp == 0 && lane < head ? lane : warp == kDrawWarps - 1 && tail + lane < n ? tail + lane : -1;
    if (edge >= 0) {
      float l[kDrawGroup];
      l[0] = at(edge);
#pragma unroll
      for (int j = 1; j < kDrawGroup; ++j) l[j] = none;
      f(l);
    }
  }

  // exp((l - m) / T)
  __device__ __forceinline__ double mass(float l) const {
    const DrawPower q = draw_power(static_cast<double>(fmaxf(l, cut)) - static_cast<double>(m), scale, table);
    return l >= cut ? q.y * q.power : 0.0;
  }
  // of those >= bound, together
  __device__ __forceinline__ double masses(const float (&l)[kDrawGroup], float bound) const {
    double s[2] = {0.0, 0.0};
    bool any = false;
#pragma unroll
    for (int j = 0; j < kDrawGroup; ++j) any |= l[j] >= bound;
    if (!any) return 0.0;
#pragma unroll
    for (int j = 0; j < kDrawGroup; ++j) s[j & 1] += l[j] >= bound ? mass(l[j]) : 0.0;
    return s[0] + s[1];
  }
  // the same in whole units of 2^-45
  __device__ __forceinline__ unsigned long long units_of(double mass) const {
    return static_cast<unsigned long long>(__double_as_longlong(fma(mass, 0x1p45, 4503599627370496.0))) - 0x4330000000000000ull;
  }
  __device__ __forceinline__ unsigned long long units(float l) const { return units_of(mass(l)); }
};

// The threshold of a restriction on the elements that each(f) gives f, a warp's share to each warp (all that can matter of them): the least logit of
// which the strictly larger ones count (MASS: weigh) less than `target`, `above` of which lies in elements that are not given; none that is
// given lies above `top`.  NaN if there is none.  The same in every CTA of the row.
template <bool MASS, typename Row, typename Each>
__device__ float draw_threshold(const Row& r, DrawShared& sh, Each each, int elements, float per_class, unsigned long long target,
                                float top, unsigned long long above) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // Sums of limbs over `elements` elements of this CTA have to fit 32 bits: additions of 32 bits are carried out by shared memory, those of 64
  // are a loop of comparisons.
  const int limb = elements <= 65536 ? 16 : 13;
  if (tid == 0) sh.limb[MASS] = limb;
  // Classes of a level: 2048 equal steps down from the largest logit (the last takes what is left), 2048 steps of that class, then the bytes
  // of the logits' order, the highest first.
  uint32_t prefix = 0;
  int first = 0, second = 0;
  for (int level = 0; level < 6; ++level) {
    const int shift = 40 - 8 * level;       // level 2: the highest byte
    // whether an element belongs to the classes chosen so far; its class of this level
    auto in_chosen = [&](float l, int& c) {
      const float x = l == top ? 0.f : (top - l) * per_class;
      c = static_cast<int>(fminf(x, kDrawClasses - 1.f));
      if (level == 0) return true;
      if (c != first) return false;
      c = static_cast<int>(fminf((x - static_cast<float>(first)) * kDrawClasses, kDrawClasses - 1.f));
      if (level == 1) return true;
      if (c != second) return false;
      const uint32_t key = draw_key(l);
      c = 255 - static_cast<int>((key >> shift) & 255u);
      return level == 2 || (key >> (shift + 8)) == prefix;
    };
    uint32_t(*h)[kDrawClasses] = sh.hist;   // the others have read it when they come to the row's wait behind
#pragma unroll
    for (int q = 0; q < (MASS ? 4 : 1); ++q)
#pragma unroll
      for (int i = 0; i < kDrawPer; ++i) h[q][tid + i * kDrawThreads] = 0;
    if (tid == 0) sh.chosen = -1;
    __syncthreads();
    each([&](const float (&l)[kDrawGroup]) {
      int c[kDrawGroup];
      bool in[kDrawGroup];
#pragma unroll
      for (int j = 0; j < kDrawGroup; ++j) in[j] = in_chosen(l[j], c[j]) && l[j] == l[j];
      if constexpr (!MASS) {
#pragma unroll
        for (int j = 0; j < kDrawGroup; ++j)
          if (in[j]) atomicAdd(&h[0][c[j]], 1u);
      } else {
        unsigned long long w[kDrawGroup];
#pragma unroll
        for (int j = 0; j < kDrawGroup; ++j) w[j] = r.units(l[j]);       // at most 2^45: 3 limbs of 16 bits, 4 of 13
#pragma unroll
        for (int j = 0; j < kDrawGroup; ++j) {
          if (!in[j]) continue;
          const uint32_t mask = (1u << limb) - 1u;
          atomicAdd(&h[0][c[j]], static_cast<uint32_t>(w[j]) & mask);
          atomicAdd(&h[1][c[j]], static_cast<uint32_t>(w[j] >> limb) & mask);
          const uint32_t rest = static_cast<uint32_t>(w[j] >> (2 * limb));         // most have no more
          if (rest) {
            atomicAdd(&h[2][c[j]], rest & mask);
            if (rest >> limb) atomicAdd(&h[3][c[j]], rest >> limb);
          }
        }
      }
    });
    row_sync(r.parts);
    {
      // neighbouring classes to a thread; then a scan from the highest on
      int limbs[8];
#pragma unroll
      for (int p = 0; p < 8; ++p) limbs[p] = MASS && p < r.parts ? static_cast<int>(ld_cluster_u32(map_to_cta(smem_u32(&sh.limb[MASS]), p))) : 0;
      unsigned long long v[kDrawPer] = {}, own = 0;
#pragma unroll
      for (int q = 0; q < (MASS ? 4 : 1); ++q)
#pragma unroll
        for (int p = 0; p < 8; ++p)
          if (p < r.parts) {
            const uint32_t from = map_to_cta(smem_u32(&h[q][kDrawPer * tid]), p);
#pragma unroll
            for (int i = 0; i < kDrawPer; i += 2) {
              const unsigned long long x = ld_cluster_u64(from + 4 * i);
              v[i] += (x & 0xffffffffull) << (q * limbs[p]);
              v[i + 1] += (x >> 32) << (q * limbs[p]);
            }
          }
#pragma unroll
      for (int i = 0; i < kDrawPer; ++i) own += v[i];
      const unsigned long long upto = warp_scan_u64(own, lane);
      if (lane == 31) sh.scan[warp] = upto;
      if (tid == 0) sh.list_n[MASS] = 0;
      __syncthreads();
      unsigned long long before = above + upto - own;
      for (int w = 0; w < warp; ++w) before += sh.scan[w];
#pragma unroll
      for (int i = 0; i < kDrawPer; ++i) {
        if (before < target && before + v[i] >= target) {
          sh.chosen = kDrawPer * tid + i;
          sh.above = before;
        }
        before += v[i];
      }
    }
    __syncthreads();
    const int chosen = sh.chosen;
    if (chosen < 0) {
      row_sync(r.parts);
      return NAN;
    }
    above = sh.above;
    if (level == 5) {                         // all bytes: one value
      row_sync(r.parts);
      return draw_unkey(prefix << 8 | (255u - chosen));
    }
    each([&](const float (&l)[kDrawGroup]) {
#pragma unroll
      for (int j = 0; j < kDrawGroup; ++j) {
        int c;
        if (l[j] == l[j] && in_chosen(l[j], c) && c == chosen) {
          const int to = atomicAdd(&sh.list_n[MASS], 1);
          if (to < kDrawFew) sh.list[MASS][to] = l[j];
        }
      }
    });
    row_sync(r.parts);
    const int ns = lane < r.parts ? static_cast<int>(ld_cluster_u32(map_to_cta(smem_u32(&sh.list_n[MASS]), lane))) : 0;
    const int few = __reduce_add_sync(0xffffffffu, ns);
    if (few <= kDrawFew) {
      // the parts' lists one behind another: a warp per part
      if (warp < r.parts) {
        const int to = __reduce_add_sync(0xffffffffu, lane < warp ? ns : 0), have = __shfl_sync(0xffffffffu, ns, warp);
        for (int i = lane; i < have; i += 32) {
          const float l = ld_cluster_f32(map_to_cta(smem_u32(&sh.list[MASS][i]), warp));
          sh.all[to + i] = l;
          if (MASS) sh.weight[to + i] = r.units(l);
        }
      }
      __syncthreads();
      // some lanes an element: what is strictly larger, each lane in its share of the list
      float least = INFINITY;
      const int e = tid / kDrawLanes;
      unsigned long long larger = 0;
      const float l = e < few ? sh.all[e] : INFINITY;
      for (int j = tid % kDrawLanes; j < few; j += kDrawLanes)
        if (sh.all[j] > l) larger += MASS ? sh.weight[j] : 1ull;
#pragma unroll
      for (int o = 1; o < kDrawLanes; o <<= 1) larger += __shfl_xor_sync(0xffffffffu, larger, o);
      if (e < few && above + larger < target) least = l;
      least = -warp_max(-least);
      if (lane == 0) sh.warp_f[1][warp] = least;
      __syncthreads();
      least = -warp_max(-sh.warp_f[1][lane % kDrawWarps]);
      return least;
    }
    if (level == 0)
      first = chosen;
    else if (level == 1)
      second = chosen;
    else
      prefix = level == 2 ? 255u - chosen : prefix << 8 | (255u - chosen);
    row_sync(r.parts);                        // what was read here is written again
  }
  return -INFINITY;
}

// A sample of a row, 32 words of every 256: where what it weighs from below comes to 0.8 and to 1.25 of `left`, the mass that a nucleus leaves
// out (but 16 of the sample above the first).  The nucleus' border lies between, but for bad luck, which draw_threshold sees.  Classes are
// those of draw_threshold from `m` down to `widest`.  One CTA a row.
template <typename Row>
__device__ void draw_bracket(const Row& r, DrawShared& sh, double left, float inv_t, float threshold, float per_class, float widest, float& lower,
                             float& upper) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
#pragma unroll
  for (int i = 0; i < kDrawPer; ++i) sh.hist[0][tid + i * kDrawThreads] = sh.hist[1][tid + i * kDrawThreads] = 0;
  if (tid == 0) sh.chosen = kDrawClasses - 1;
  __syncthreads();
  // 2^20 stand for `left`; no more than 2^16 for one, so that an eighth of the largest row adds up in 32 bits
  static_assert((kDrawMost / 8 + 8192) * 65537ll < 1ll << 32, "weights of a sample");
  const float lift = static_cast<float>(log(8 * 0x1p20 / left));
  uint32_t last = 0, lasts = 0;               // of the last class, which has most
  for (int w = warp * 256 + lane; w < r.words; w += kDrawWarps * 256) {
    float x[Row::kVec];
    r.word(w, x);
#pragma unroll
    for (int j = 0; j < Row::kVec; ++j) {
      const float l = x[j];
      const int c = static_cast<int>(fminf((r.m - l) * per_class, kDrawClasses - 1.f));
      const uint32_t weight = l >= threshold ? static_cast<uint32_t>(fminf(__expf((l - r.m) * inv_t + lift), 65536.f) + 0.5f) : 0u;
      if (c < kDrawClasses - 1) {
        if (l >= threshold) {
          atomicAdd(&sh.hist[0][c], weight);
          atomicAdd(&sh.hist[1][c], 1u);
        }
      } else {
        last += weight;
        lasts += l >= threshold;
      }
    }
  }
  last = __reduce_add_sync(0xffffffffu, last);
  lasts = __reduce_add_sync(0xffffffffu, lasts);
  if (lane == 0) {
    atomicAdd(&sh.hist[0][kDrawClasses - 1], last);
    atomicAdd(&sh.hist[1][kDrawClasses - 1], lasts);
  }
  __syncthreads();
  constexpr unsigned long long kWeight = (1ull << 40) - 1;      // the weight; above it the number
  unsigned long long v[kDrawPer], own = 0;
#pragma unroll
  for (int i = 0; i < kDrawPer; ++i) {
    v[i] = sh.hist[0][kDrawPer * tid + i] | static_cast<unsigned long long>(sh.hist[1][kDrawPer * tid + i]) << 40;
    own += v[i];
  }
  const unsigned long long upto = warp_scan_u64(own, lane);
  if (lane == 31) sh.scan[warp] = upto;
  __syncthreads();
  unsigned long long before = upto - own, all = 0;
  for (int w = 0; w < kDrawWarps; ++w) {
    if (w < warp) before += sh.scan[w];
    all += sh.scan[w];
  }
  auto below = [&](unsigned long long x) { return static_cast<uint32_t>((all & kWeight) - (x & kWeight)); };
  auto low = [&](unsigned long long x) { return below(x) <= 838861u && (x >> 40) >= 16; };
  auto high = [&](unsigned long long x) { return below(x) >= 1310720u; };
#pragma unroll
  for (int i = 0; i < kDrawPer; ++i) {
    const unsigned long long x = before + v[i];
    const bool first = kDrawPer * tid + i == 0;
    if (low(x) && (first || !low(before))) sh.chosen = kDrawPer * tid + i;
    if (!high(x) && (first || high(before))) sh.owner = kDrawPer * tid + i;       // one there always is: nothing lies below the last
    before = x;
  }
  __syncthreads();
  lower = sh.chosen == kDrawClasses - 1 ? widest : fmaxf(widest, r.m - (sh.chosen + 1) / per_class);
  upper = sh.owner == 0 ? INFINITY : fmaxf(lower, r.m - sh.owner / per_class);
}

// GIVEN: by a given number, else by noise
template <typename T, bool KEPT, bool GIVEN>
__global__ void __launch_bounds__(kDrawThreads, 1) draw_kernel(const DrawArgs a) {
  pdl_entry();
  extern __shared__ __align__(16) unsigned char draw_smem[];
  DrawShared& sh = *reinterpret_cast<DrawShared*>(draw_smem);
  float* const draw_buffer = reinterpret_cast<float*>(draw_smem + kDrawShared);
  using Row = DrawRow<T, KEPT>;
  const int b = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int begin = min(part * a.per, a.V), n = min(a.V - begin, a.per);
  Row r;
  r.src = static_cast<const T*>(a.logits) + b * a.ld + begin;
  r.n = n;
  r.parts = a.parts;
  r.head = min(static_cast<int>((-(reinterpret_cast<uintptr_t>(r.src)) & 15) / sizeof(T)), n);
  r.words = (n - r.head) / Row::kVec;
  r.table = &sh.table[0][lane & 15];
  r.flat = false;
  r.z = draw_buffer + (4 - r.head % 4) % 4;           // words of the row on words of the buffer
  float* const heavy = draw_buffer + (KEPT ? a.per + 4 : 0) + warp * 32 * a.room;
  const float p = a.top_p ? a.top_p[b] : a.top_p_all;
  const bool by_mass = p < 1.f;

  for (int i = tid; i < 1024; i += kDrawThreads) {
    const double e = exp2((i >> 4) / 64.0);
    sh.table[i >> 4][i & 15] = __hiloint2double(__double2hiint(e) - ((i >> 4) << 14), __double2loint(e));
  }
  const float temperature = a.temperature ? a.temperature[b] : a.temperature_all;
  const bool greedy = !(temperature > 0.f);
  const float t = greedy ? 1.f : fminf(temperature, 1e30f);
  r.scale = 64 * 1.4426950408889634 / static_cast<double>(t);
  __syncthreads();

  // the first walk: the largest logit, masses exp(l / T) of this warp's range; KEPT: the part into shared memory
  // 2^-1000: what lies below is taken as that, as what is no number is; what lies too far above 0 is seen by the largest, and its sums are not used
  const float reach_of = 693.f * t;
  float m = -INFINITY;
  double mine = 0.0;
  {
    // the stages of all elements of a batch side by side: an operation in 64 bits has its result some ten times later than one in 32
    auto take = [&](const float (&l)[kDrawBatch]) {
      double sum[2] = {0.0, 0.0};
#pragma unroll
      for (int j = 0; j < kDrawBatch; ++j) {
        m = fmaxf(m, l[j]);
        const DrawPower q = draw_power(static_cast<double>(fmaxf(l[j], -reach_of)), r.scale, r.table);
        sum[j & 1] = fma(q.y, q.power, sum[j & 1]);
      }
      mine += sum[0] + sum[1];
    };
    const int tail = r.head + r.words * Row::kVec;
    const int edge = warp == 0 && lane < r.head ? lane : warp == kDrawWarps - 1 && tail + lane < n ? tail + lane : -1;
    if (edge >= 0) {
      const float l = draw_logit(r.src[edge]);
      if (KEPT) r.z[edge] = l;
      m = fmaxf(m, l);
      const DrawPower q = draw_power(static_cast<double>(fmaxf(l, -reach_of)), r.scale, r.table);
      mine += q.y * q.power;
    }
    const uint4* s4 = reinterpret_cast<const uint4*>(r.src + r.head);
    const int w1 = min((warp + 1) * r.per_warp(), r.words);
    constexpr int kWords = kDrawBatch / Row::kVec;
    uint4 next[kWords];                       // of the batch after this one
    int w = min(warp * r.per_warp(), r.words) + lane;
    auto fetch = [&](int at) {
#pragma unroll
      for (int q = 0; q < kWords; ++q)
        if (at + 32 * q < w1) next[q] = s4[at + 32 * q];
    };
    fetch(w);
    for (; w < w1; w += 32 * kWords) {
      float l[kDrawBatch];
#pragma unroll
      for (int q = 0; q < kWords; ++q) {
        const bool on = w + 32 * q < w1;
        const T* x = reinterpret_cast<const T*>(&next[q]);
#pragma unroll
        for (int j = 0; j < Row::kVec; j += 4) {
          float4 f = make_float4(static_cast<float>(x[j]), static_cast<float>(x[j + 1]), static_cast<float>(x[j + 2]), static_cast<float>(x[j + 3]));
          if (KEPT && on)
            reinterpret_cast<float4*>(r.z + r.head + (w + 32 * q) * Row::kVec)[j / 4] =
                make_float4(draw_logit(f.x), draw_logit(f.y), draw_logit(f.z), draw_logit(f.w));
          if (!on) f = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
          l[q * Row::kVec + j] = f.x;
          l[q * Row::kVec + j + 1] = f.y;
          l[q * Row::kVec + j + 2] = f.z;
          l[q * Row::kVec + j + 3] = f.w;
        }
      }
      fetch(w + 32 * kWords);
      take(l);
    }
  }
  m = warp_max(m);
  mine = warp_sum_f64(mine);
  if (lane == 0) {
    sh.warp_f[0][warp] = m;
    sh.warp_mass[0][warp] = mine;
  }
  row_sync(a.parts);
  m = row_max(sh.warp_f[0], a.parts, lane);
  if (m == -INFINITY) {                      // nothing to draw from
    if (part == 0 && tid == 0) {
      a.tokens[b] = 0;
      a.logprobs[b] = -INFINITY;
    }
    row_sync(a.parts);
    return;
  }
  r.flat = m == INFINITY;
  // the first walk's sums say nothing where the largest logit lies near or beyond what they tell apart
  const bool redo = !(fabsf(m) <= 600.f * t);
  if (r.flat) m = 0.f;
  const float inv_t = 1.f / t;
  r.m = m;
  r.cut = m - 693.f * t;                      // 2^-1000 of the largest's mass, as far as a table and 64 bits reach
  const int k = a.top_k ? a.top_k[b] : a.top_k_all;
  const float least_share = a.min_p ? a.min_p[b] : a.min_p_all, mp = fminf(least_share, 1.f);
  const bool by_rank = k > 0 && k < a.V, by_share = least_share > 0.f;
  // exp((l - m) / T) of this warp's elements >= bound
  auto weigh = [&](float bound, int slot) {
    double s0 = 0.0;
    r.walk(warp, lane, NAN, [&](const float (&l)[kDrawGroup]) { s0 += r.masses(l, bound); });
    s0 = warp_sum_f64(s0);
    if (lane == 0) sh.warp_mass[slot][warp] = s0;
  };
  int slot = 0;                               // of warp_mass: the other one may still be read
  double factor = 1.0;                        // from the sums' unit to the largest's mass
  if (redo) {
    weigh(-INFINITY, slot = 1);
    row_sync(a.parts);
  } else {
    const DrawPower q = draw_power(-static_cast<double>(m), r.scale, r.table);
    factor = q.y * q.power;
  }
  const double all_mass = row_sum(sh.warp_mass[slot], a.parts, lane) * factor;        // of the unrestricted row
  if (greedy) {
    int first = 0x7fffffff;
    const int hi = r.to(warp);
    for (int i = r.from(warp) + lane; i < hi; i += 32)
      if (r.at(i) == m) first = min(first, begin + i);
    first = __reduce_min_sync(0xffffffffu, first);
    if (lane == 0) sh.warp_i[warp] = first;
    row_sync(a.parts);
    if (part == 0 && warp == 0) {
      first = row_min(sh.warp_i, a.parts, lane);
      if (lane == 0) {
        a.tokens[b] = first;
        a.logprobs[b] = static_cast<float>(-log(all_mass));
      }
    }
    row_sync(a.parts);
    return;
  }

  // what stays: logits >= threshold
  float threshold = -INFINITY;
  if (by_rank)
    threshold = draw_threshold<false>(r, sh, [&](auto f) { r.walk(warp, lane, NAN, f); }, n, 64.f * inv_t, static_cast<unsigned long long>(k), m, 0ull);
  if (by_share) {
    // the least fp32 number l with (l - m) / T >= log(min_p), in 64 bits; from a rounded guess it is a step or two
    const double need = log(static_cast<double>(mp)) * static_cast<double>(t);
    auto stays = [&](float l) { return static_cast<double>(l) - static_cast<double>(m) >= need; };
    float l = static_cast<float>(static_cast<double>(m) + need);
    for (int i = 0; i < 4 && !stays(l); ++i) l = draw_unkey(draw_key(l) + 1u);
    for (int i = 0; i < 4 && l > -INFINITY && stays(draw_unkey(draw_key(l) - 1u)); ++i) l = draw_unkey(draw_key(l) - 1u);
    threshold = fmaxf(threshold, fminf(l, m));
  }
  if (by_mass) {
    double total = all_mass;
    if (by_rank || by_share) {
      weigh(threshold, slot ^= 1);
      row_sync(a.parts);
      total = row_sum(sh.warp_mass[slot], a.parts, lane);
    }
    // larger < p total; in units, whose sums over the elements are off by less than the least step of p
    const double share = p > 0.f ? static_cast<double>(p) * total : 0.0;
    const unsigned long long target = max(1ull, static_cast<unsigned long long>(ceil(share * 0x1p45)));
    // Elements below the V-th part of what the nucleus leaves out weigh less than that together: they are outside of it.  What is above goes
    // into a list (of 151936 logits some hundreds to some ten thousands), and only its elements are sorted into classes.
    const double least = (total - share) / static_cast<double>(a.V) * 0x1p45 - 1.0;
    float reach = threshold;
    if (least > 0.0) {
      // lower by more than the roundings of masses, of l and of its fp32 number
      const double under = log(least * 0x1p-45) - 1e-5;
      reach = fmaxf(reach, static_cast<float>(static_cast<double>(m) + static_cast<double>(t) * under) - 1e-6f * fabsf(m));
    }
    const bool ranged = reach > -INFINITY && reach < m;
    const float widest = reach, per_class = ranged ? fminf((kDrawClasses - 0.1f) / (m - reach), 1e30f) : 64.f * inv_t;
    // Of a long row a sample says roughly where the border is: only what lies near it is then sorted, what lies above is added up, and nothing else
    // is listed.  (128 rows of 151936, top_p = 0.95: 103 us, 182 with everything above `widest` sorted.)  Should the border lie elsewhere, it
    // is sought once more without, as it is where the lists do not hold what lies above: 44032 of 151936 logits, which the nuclei of flat rows
    // exceed (T = 1, top_p 0.95: 242 us; T = 1.3: 316; in 16 bits 507 and 323).
    float upper = INFINITY;
    bool narrow = !KEPT && a.parts == 1 && !redo && ranged && least > 0.0;
    if (narrow) draw_bracket(r, sh, total - share, inv_t, threshold, per_class, widest, reach, upper);
    double s0 = 0.0;
    float border;
#pragma unroll 1
    for (;;) {
      // each lane's, in a column of its own of the warp's list: from the front those up to `upper`, from the back those above
      const int nowhere = (a.room - 1) * 32 + lane;      // the column's last place takes what is not listed: a store less to decide about
      int front = lane, back = nowhere - 32;             // upper >= reach: what is above `upper` is in
      r.walk(warp, lane, NAN, [&](const float (&l)[kDrawGroup]) {
#pragma unroll
        for (int j = 0; j < kDrawGroup; ++j) {       // no branches (170 us with them): nearly every warp has some of both kinds
          const int in = l[j] >= reach, is_high = l[j] >= upper;
          heavy[front > back || !in ? nowhere : is_high ? back : front] = l[j];
          back -= is_high * 32;
          front += (in - is_high) * 32;
        }
      });
      const int have = front / 32, high = (nowhere - 32 - back) / 32;
      const int most = __reduce_max_sync(0xffffffffu, have), together = __reduce_add_sync(0xffffffffu, have);
      const bool listed = __reduce_max_sync(0xffffffffu, have + high) < a.room;       // else the warp's range takes the list's place
      if (lane == 0) sh.warp_n[warp] = together;
      const bool full = __syncthreads_or(!listed);
      const int elements = __reduce_add_sync(0xffffffffu, lane < kDrawWarps ? sh.warp_n[lane] : 0);
      auto each = [&](auto f) {
        if (!listed) {
          r.walk(warp, lane, NAN, [&](float (&l)[kDrawGroup]) {
#pragma unroll
            for (int j = 0; j < kDrawGroup; ++j) l[j] = l[j] >= reach ? l[j] : NAN;
            f(l);
          });
          return;
        }
#pragma unroll 1
        for (int i = 0; i < most; i += kDrawGroup) {
          float l[kDrawGroup];
#pragma unroll
          for (int j = 0; j < kDrawGroup; ++j) l[j] = i + j < have ? heavy[(i + j) * 32 + lane] : NAN;
          f(l);
        }
      };
      s0 = 0.0;
      unsigned long long above = 0;
      if (narrow && !full) {
#pragma unroll 1
        for (int i = 0; i < high; i += kDrawGroup) {
          double s[2] = {0.0, 0.0};
#pragma unroll
          for (int j = 0; j < kDrawGroup; ++j) {
            const double q = r.mass(i + j < high ? heavy[nowhere - 32 * (1 + i + j)] : NAN);
            s[j & 1] += q;
            above += r.units_of(q);
          }
          s0 += s[0] + s[1];
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) above += __shfl_xor_sync(0xffffffffu, above, o);
        if (lane == 0) sh.scan[warp] = above;
        __syncthreads();
        above = 0;
        for (int w = 0; w < kDrawWarps; ++w) above += sh.scan[w];
      }
      border = narrow && full ? NAN : draw_threshold<true>(r, sh, each, elements, per_class, target, upper < m ? upper : m, above);
      if (!narrow && !(border == border)) border = reach;
      if (border == border) {
        each([&](const float (&l)[kDrawGroup]) { s0 += r.masses(l, border); });
        break;
      }
      narrow = false;
      reach = widest;
      upper = INFINITY;
    }
    threshold = fmaxf(threshold, border);
    s0 = warp_sum_f64(s0);
    slot ^= 1;
    if (lane == 0) sh.warp_mass[slot][warp] = s0;
  }

  if constexpr (!GIVEN) {
    // The largest of l / T and a noise of each token's own, numbers and rounding as in decode.cu's draws: a restriction changes what is drawn only
    // where it leaves that token out, and logits that differ in their last bits seldom change it.
    const uint32_t step = a.step ? static_cast<uint32_t>(*a.step) : 0u, seed = a.seed_dev ? static_cast<uint32_t>(*a.seed_dev) : a.seed;
    const uint32_t base = noise_base(seed, step, b);
    float best = -INFINITY;
    int best_i = 0x7fffffff;
    const int hi = r.to(warp);
#pragma unroll 4
    for (int i = r.from(warp) + lane; i < hi; i += 32) {
      const float l = r.at(i);
      if (!(l >= threshold)) continue;
      const float key = l * inv_t + draw_noise(base, begin + i);
      if (key > best) {
        best = key;
        best_i = begin + i;
      }
    }
    auto join = [&]() {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const float key = __shfl_xor_sync(0xffffffffu, best, o);
        const int i = __shfl_xor_sync(0xffffffffu, best_i, o);
        if (key > best || (key == best && i < best_i)) {
          best = key;
          best_i = i;
        }
      }
    };
    join();
    if (lane == 0) {
      sh.warp_key[warp] = best;
      sh.warp_i[warp] = best_i;
    }
    row_sync(a.parts);
    if (part == 0 && warp == 0) {
      best = -INFINITY;
      best_i = 0x7fffffff;
      for (int p = 0; p < a.parts; ++p) {
        if (lane >= kDrawWarps) break;
        const float key = ld_cluster_f32(map_to_cta(smem_u32(&sh.warp_key[lane]), p));
        const int i = static_cast<int>(ld_cluster_u32(map_to_cta(smem_u32(&sh.warp_i[lane]), p)));
        if (key > best || (key == best && i < best_i)) {
          best = key;
          best_i = i;
        }
      }
      __syncwarp();
      join();
      if (lane == 0) {
        // the largest always stays, so there is one; its key can be -inf only where T is so small that l / T is
        const int i = best_i < a.V ? best_i : 0;
        const float l = r.seen(draw_logit(static_cast<const T*>(a.logits)[b * a.ld + i]));
        a.tokens[b] = i;
        a.logprobs[b] = static_cast<float>((static_cast<double>(l) - static_cast<double>(m)) / static_cast<double>(t) - log(all_mass));
      }
    }
    row_sync(a.parts);
  } else {
    double u = a.u64 ? static_cast<const double*>(a.u)[b] : static_cast<double>(static_cast<const float*>(a.u)[b]);
    // 1 and above, and what is not a number, stand for the largest number below 1
    u = u < 1.0 ? fmax(u, 0.0) : 1.0 - 0x1p-52;
    // Masses of what stays.  The first walk's sums hold 2^-1000 for every element below that, which is next to nothing beside any u but those next
    // to 0 (torch.rand gives 0 once in 2^24): these want to know which ranges have any mass.
    const bool restricted = by_rank || by_share || by_mass, weighed = restricted || redo || u < 0x1p-60;
    if (restricted || (weighed && !redo)) {
      if (!by_mass) weigh(threshold, slot ^= 1);
      factor = 1.0;
      row_sync(a.parts);
    }
    if (warp == 0) {
      // the ranges of up to 8 parts, some a lane; a target that roundings put behind the last of their sums lies in the last that has mass
      double v[kDrawRanges], total = 0.0;
      const int q = lane / 4;
#pragma unroll
      for (int j = 0; j < kDrawRanges; ++j)        // relative to the largest's
        v[j] = q < a.parts ? __longlong_as_double(ld_cluster_u64(map_to_cta(smem_u32(&sh.warp_mass[slot][lane % 4 * kDrawRanges + j]), q))) * factor : 0.0;
#pragma unroll
      for (int j = 0; j < kDrawRanges; ++j) total += v[j];
      const double upto = warp_scan_f64(total, lane);
      const double target = u * __shfl_sync(0xffffffffu, upto, 31);
      // a range of the first walk's with less than 2^-80 may have none: its sum is what its elements' places are worth
      const double none = weighed ? 0.0 : 0x1p-80;
      const unsigned behind = __ballot_sync(0xffffffffu, total > none && target < upto), some = __ballot_sync(0xffffffffu, total > none);
      const int owner = behind ? __ffs(behind) - 1 : 31 - __clz(some);
      double before = __shfl_up_sync(0xffffffffu, upto, 1);
      if (lane == 0) before = 0.0;
      if (lane == owner) {
        int range = 0;
        double begins = before;
        bool found = false;
#pragma unroll
        for (int j = 0; j < kDrawRanges; ++j) {
          if (!found && v[j] > none) {
            range = j;
            begins = before;
          }
          before += v[j];
          found = found || (v[j] > none && target < before);
        }
        sh.owner = lane * kDrawRanges + range;
        sh.before = target - begins;            // within the range
      }
    }
    __syncthreads();
    if (sh.owner / kDrawWarps == part) {
      // the range again, a run to each warp; then the run element by element
      const double target = sh.before;
      const int lo = r.from(sh.owner % kDrawWarps), hi = r.to(sh.owner % kDrawWarps), run = (hi - lo + kDrawWarps - 1) / kDrawWarps;
      const int r0 = min(lo + warp * run, hi), r1 = min(r0 + run, hi);
      // of a run up to 256 elements stay in registers: their loads go out together, and the search takes them from there
      constexpr int kHeld = 8;
      float l[kHeld];
      double w[kHeld], s = 0.0;
#pragma unroll
      for (int j = 0; j < kHeld; ++j) l[j] = r0 + 32 * j + lane < r1 ? r.at(r0 + 32 * j + lane) : -INFINITY;
#pragma unroll
      for (int j = 0; j < kHeld; ++j) {
        w[j] = r0 + 32 * j < r1 && l[j] >= threshold ? r.mass(l[j]) : 0.0;
        s += w[j];
      }
      for (int i = r0 + 32 * kHeld + lane; i < r1; i += 32) {
        const float x = r.at(i);
        if (x >= threshold) s += r.mass(x);
      }
      s = warp_sum_f64(s);
      if (lane == 0) sh.sub[warp] = s;
      __syncthreads();
      const double mass = lane < kDrawWarps ? sh.sub[lane] : 0.0, upto = warp_scan_f64(mass, lane);
      const unsigned some = __ballot_sync(0xffffffffu, mass > 0.0), behind = __ballot_sync(0xffffffffu, mass > 0.0 && target < upto);
      const int at = behind ? __ffs(behind) - 1 : 31 - __clz(some);
      double before = __shfl_sync(0xffffffffu, upto - mass, at);
      if (warp == at) {
        int drawn = -1;                         // the first behind which the target does not lie, or the last with any mass
        auto search = [&](int i0, double x) {
          const double upto_x = before + warp_scan_f64(x, lane);
          const unsigned held = __ballot_sync(0xffffffffu, x > 0.0), hit = __ballot_sync(0xffffffffu, x > 0.0 && target < upto_x);
          if (hit) {
            drawn = i0 + __ffs(hit) - 1;
            return true;
          }
          if (held) drawn = i0 + 31 - __clz(held);
          before = __shfl_sync(0xffffffffu, upto_x, 31);
          return false;
        };
        bool found = false;
#pragma unroll
        for (int j = 0; j < kHeld; ++j)
          if (!found && r0 + 32 * j < r1) found = search(r0 + 32 * j, w[j]);
        for (int i0 = r0 + 32 * kHeld; i0 < r1 && !found; i0 += 32) {
          const float x = i0 + lane < r1 ? r.at(i0 + lane) : -INFINITY;
          found = search(i0, i0 + lane < r1 && x >= threshold ? r.mass(x) : 0.0);
        }
        if (lane == 0) {
          const float x = r.at(drawn);
          a.tokens[b] = begin + drawn;
          a.logprobs[b] = static_cast<float>((static_cast<double>(x) - static_cast<double>(m)) / static_cast<double>(t) - log(all_mass));
        }
      }
    }
    row_sync(a.parts);                          // nobody leaves while its shared memory may be read
  }
}

template <typename T, bool KEPT, bool GIVEN>
static int launch_draw_as(const DrawArgs& a, int B, cudaStream_t s) {
  static int allowed[64] = {0};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!allowed[dev & 63]) {
    const cudaError_t e = cudaFuncSetAttribute(draw_kernel<T, KEPT, GIVEN>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               kDrawShared + kDrawBytes);
    if (e != cudaSuccess) return static_cast<int>(e);
    allowed[dev & 63] = 1;
  }
  return static_cast<int>(launch_kernel_clusters(draw_kernel<T, KEPT, GIVEN>, dim3(static_cast<unsigned>(B) * a.parts), dim3(kDrawThreads),
                                                 kDrawShared + kDrawBytes, a.parts, s, a));
}

template <typename T>
static int launch_draw(DrawArgs a, int B, cudaStream_t s) {
  // as many parts as leave every CTA an SM of its own, of no fewer than 4096 elements
  int parts = 1;
  while (parts < 8 && static_cast<long long>(B) * parts * 2 <= sm_count() && a.V / parts > 8192) parts *= 2;
  a.parts = parts;
  a.per = ((a.V + parts - 1) / parts + 7) / 8 * 8;
  const bool kept = a.per <= kDrawKept;
  a.room = (kDrawBytes / 4 - (kept ? a.per + 4 : 0)) / kDrawThreads;
  if (!a.u) return kept ? launch_draw_as<T, true, false>(a, B, s) : launch_draw_as<T, false, false>(a, B, s);
  return kept ? launch_draw_as<T, true, true>(a, B, s) : launch_draw_as<T, false, true>(a, B, s);
}

}  // namespace apb

extern "C" {

// logits [B, V], row stride ld: type 0 fp32, 1 bf16, 2 fp16.  Of each setting a tensor [B] (fp32, top_k int32) or null and one number
// for all rows: temperature (<= 0: the first of the largest logits), top_k (<= 0: off), top_p (>= 1: off), min_p (<= 0: off).  u [B] in
// [0, 1): fp32, or fp64 with u64; null: the largest of logit / T and noise of each token's own, a hash of *seed_dev (null: seed), *step (null:
// 0), the row and the token.  tokens [B] int32, logprobs [B] fp32.  V up to 393216.
int apb_draw(const void* logits, int type, long long ld, const float* temperature, float temperature_all, const int* top_k, int top_k_all,
             const float* top_p, float top_p_all, const float* min_p, float min_p_all, const void* u, int u64, unsigned seed,
             const int* seed_dev, const int* step, int B, int V, int* tokens, float* logprobs, cudaStream_t s) {
  using namespace apb;
  if (B <= 0) return 0;
  if (!logits || !tokens || !logprobs || V < 1 || V > kDrawMost || type < 0 || type > 2) return kBadArgument;
  DrawArgs a{logits, ld, temperature, top_k, top_p, min_p, temperature_all, top_p_all, min_p_all, top_k_all,
             u, step, seed_dev, static_cast<uint32_t>(seed), u64, V, 1, 0, 0, tokens, logprobs};
  if (type == 0) return launch_draw<float>(a, B, s);
  if (type == 1) return launch_draw<__nv_bfloat16>(a, B, s);
  return launch_draw<__half>(a, B, s);
}
}
