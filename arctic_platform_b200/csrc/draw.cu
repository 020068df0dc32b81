// Tokens drawn from rows of logits with given random numbers: temperature, top-k, min-p, top-p, then the first token, in the order of the
// vocabulary, at which the running mass of what stays passes u of the whole.
//
// Mathematics.  Every restriction keeps the logits from a threshold on, so a row comes down to one threshold: the top_k-th largest
// logit; the least logit with exp((l - max) / T) >= min_p; the least logit of which the strictly larger ones hold less than top_p of what
// stayed so far.  Masses are exp((l - max) / T) in 64 bits, rounded to whole multiples of 2^-45: sums of whole numbers do not depend on
// their order, and a draw next to a border comes out as it does in 64-bit arithmetic (fp32 masses put one draw of some hundred, from
// flat rows of 151936, on the neighbour's side).
//
// Layout.  A cluster of CTAs per row, each with a part of it in shared memory, so that the row is read from global memory once and walked
// several times.  A threshold is found by histograms of 256 classes (an eighth of a nat each, then the bytes of the logit's order) that all CTAs of the
// cluster read from one another, until few elements are left in the class that holds it.
#include "common.cuh"
#include "host_utils.cuh"

namespace apb {

constexpr int kDrawThreads = 512;
constexpr int kDrawWarps = kDrawThreads / 32;
constexpr int kDrawClasses = 256;
constexpr int kDrawFew = 256;             // elements of a class that are compared with one another
constexpr int kDrawMaxPart = 48 * 1024;   // elements of a row in one CTA's shared memory

struct DrawArgs {
  const void* logits;
  long long ld;
  const float* temperature;   // [B] each, or null: the same number for all rows
  const int* top_k;
  const float* top_p;
  const float* min_p;
  float temperature_all, top_p_all, min_p_all;
  int top_k_all;
  const void* u;              // [B] fp32 or fp64; null: a hash of (seed, step, row)
  const int* step;
  uint32_t seed;
  int u64;
  int V, parts, per;
  int* tokens;
  float* logprobs;
};

__device__ __forceinline__ uint32_t draw_key(float z) {      // larger logit, larger key
  const uint32_t u = __float_as_uint(z);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float draw_unkey(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }
__device__ __forceinline__ uint32_t draw_hash(uint32_t x) {
  x ^= x >> 16;
  x *= 0x7feb352dU;
  x ^= x >> 15;
  x *= 0x846ca68bU;
  x ^= x >> 16;
  return x;
}
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
__device__ __forceinline__ unsigned long long warp_sum_u64(unsigned long long v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
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

template <typename T>
__device__ __forceinline__ float draw_logit(T x) {
  const float z = static_cast<float>(x);
  return z == z ? z : -INFINITY;          // what is not a number is never drawn
}

// z[shift + i] = element begin + i of the row, i < n; returns this thread's largest.  The shift puts 16-byte words of the row on 16-byte
// words of the buffer.
template <typename T>
__device__ __forceinline__ float draw_load(const T* __restrict__ src, int n, float* buffer, int& shift) {
  constexpr int kVec = 16 / sizeof(T);
  const int ahead = static_cast<int>((-(reinterpret_cast<uintptr_t>(src)) & 15) / sizeof(T));
  const int head = min(ahead, n), words = (n - head) / kVec, tail = head + words * kVec;
  shift = (4 - head % 4) % 4;
  float* z = buffer + shift;
  float m = -INFINITY;
  if (static_cast<int>(threadIdx.x) < head) {
    z[threadIdx.x] = draw_logit(src[threadIdx.x]);
    m = z[threadIdx.x];
  }
  const uint4* s4 = reinterpret_cast<const uint4*>(src + head);
#pragma unroll 4
  for (int w = threadIdx.x; w < words; w += kDrawThreads) {
    const uint4 raw = s4[w];
    const T* x = reinterpret_cast<const T*>(&raw);
    float4* to = reinterpret_cast<float4*>(z + head + w * kVec);
#pragma unroll
    for (int j = 0; j < kVec; j += 4) {
      const float4 f = make_float4(draw_logit(x[j]), draw_logit(x[j + 1]), draw_logit(x[j + 2]), draw_logit(x[j + 3]));
      to[j / 4] = f;
      m = fmaxf(fmaxf(m, fmaxf(f.x, f.y)), fmaxf(f.z, f.w));
    }
  }
  for (int i = tail + threadIdx.x; i < n; i += kDrawThreads) {
    z[i] = draw_logit(src[i]);
    m = fmaxf(m, z[i]);
  }
  return m;
}

struct DrawShared {
  uint32_t hist[2][4][kDrawClasses];        // three 16-bit limbs of the masses, counts (two copies: one is read while the next is filled)
  float list[kDrawFew];                     // this CTA's elements of the class
  float all[kDrawFew];                      // the cluster's
  unsigned long long weight[kDrawFew];
  unsigned long long warp_mass[kDrawWarps];
  unsigned long long above, total;
  float warp_f[kDrawWarps];
  int warp_i[kDrawWarps];
  float part_max, part_sum, threshold;
  int part_first, list_n, chosen, in_class, owner;
  unsigned long long before;
};

struct DrawRow {
  const float* z;      // this CTA's part
  int n, parts, part;
  float m, inv_t;
  double scale;        // log2(e) / T

  // mass in units of 2^-45; rounded to nearest: rounding down would take 2^-46 from every token of the tail, to one side
  __device__ __forceinline__ unsigned long long mass(float l) const {
    if (l == m) return 1ull << 45;
    const double x = (static_cast<double>(l) - static_cast<double>(m)) * scale;
    if (!(x > -47.0)) return 0ull;
    return static_cast<unsigned long long>(__double2ll_rn(exp2(x + 45.0)));
  }
  __device__ __forceinline__ int first_class(float l) const {
    if (l == m) return 0;
    return static_cast<int>(fminf((m - l) * inv_t * 8.f, static_cast<float>(kDrawClasses - 1)));
  }
};

// The threshold of a restriction on the elements >= floor: the least logit of which the strictly larger ones count less than `target`
// (MASS: weigh less than `share` / 2^64 of all).  The same in every CTA of the cluster.
template <bool MASS>
__device__ float draw_threshold(const DrawRow& r, DrawShared& sh, float floor, unsigned long long target, unsigned long long share, int& round) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  unsigned long long above = 0;             // of the elements in higher classes
  uint32_t prefix = 0;
  int first = 0;
  for (int level = 0; level < 5; ++level, ++round) {
    const int shift = 32 - 8 * level;       // level 1: the highest byte
    uint32_t(*h)[kDrawClasses] = sh.hist[round & 1];
    for (int i = tid; i < 4 * kDrawClasses; i += kDrawThreads) (&h[0][0])[i] = 0;
    __syncthreads();
    for (int i = tid; i < r.n; i += kDrawThreads) {
      const float l = r.z[i];
      if (!(l >= floor)) continue;
      int c = r.first_class(l);
      if (level > 0) {
        if (c != first) continue;
        const uint32_t key = draw_key(l);
        if (level > 1 && (key >> (shift + 8)) != prefix) continue;
        c = 255 - static_cast<int>((key >> shift) & 255u);
      }
      atomicAdd(&h[3][c], 1u);
      if (MASS) {
        const unsigned long long w = r.mass(l);          // at most 2^45; a class has at most 2^16 elements of this CTA
        if (w & 0xffffu) atomicAdd(&h[0][c], static_cast<uint32_t>(w & 0xffffu));
        if ((w >> 16) & 0xffffu) atomicAdd(&h[1][c], static_cast<uint32_t>((w >> 16) & 0xffffu));
        if (w >> 32) atomicAdd(&h[2][c], static_cast<uint32_t>(w >> 32));
      }
    }
    cluster_sync_all();
    if (warp < 8) {
      // one class a thread; then a scan from the highest on
      unsigned long long v = 0;
      uint32_t count = 0;
      for (int p = 0; p < r.parts; ++p) {
        const uint32_t at = map_to_cta(smem_u32(&h[0][tid]), p);
        count += ld_cluster_u32(at + 3 * kDrawClasses * 4);
        if (MASS)
          v += ld_cluster_u32(at) + (static_cast<unsigned long long>(ld_cluster_u32(at + kDrawClasses * 4)) << 16) +
               (static_cast<unsigned long long>(ld_cluster_u32(at + 2 * kDrawClasses * 4)) << 32);
      }
      if (!MASS) v = count;
      const unsigned long long upto = warp_scan_u64(v, lane);
      if (lane == 31) sh.warp_mass[warp] = upto;
      asm volatile("bar.sync 1, 256;" ::: "memory");
      unsigned long long lower = above;
      for (int w = 0; w < warp; ++w) lower += sh.warp_mass[w];
      if (MASS && level == 0) {
        unsigned long long total = 0;
        for (int w = 0; w < 8; ++w) total += sh.warp_mass[w];
        // larger < p total, in whole numbers: larger < ceil(p total); the largest always stay
        target = max(1ull, __umul64hi(share, total) + (share * total != 0ull ? 1ull : 0ull));
        if (tid == 0) sh.total = target;
      }
      const unsigned long long before = lower + upto - v;
      if (before < target && before + v >= target) {
        sh.chosen = tid;
        sh.in_class = static_cast<int>(count);
        sh.above = before;
      }
    }
    __syncthreads();
    if (MASS && level == 0) target = sh.total;
    above = sh.above;
    const int chosen = sh.chosen, few = sh.in_class;
    if (level == 0)
      first = chosen;
    else
      prefix = level == 1 ? 255u - chosen : prefix << 8 | (255u - chosen);
    __syncthreads();                          // what was read here is written again
    if (level == 4) {                         // all bytes: one value
      ++round;
      return draw_unkey(prefix);
    }
    if (few <= kDrawFew) {
      if (tid == 0) sh.list_n = 0;
      __syncthreads();
      for (int i = tid; i < r.n; i += kDrawThreads) {
        const float l = r.z[i];
        if (!(l >= floor) || r.first_class(l) != first) continue;
        if (level > 0 && (draw_key(l) >> shift) != prefix) continue;
        sh.list[atomicAdd(&sh.list_n, 1)] = l;
      }
      cluster_sync_all();
      // the parts' lists one behind another: a warp per part
      if (warp < r.parts) {
        int at = 0;
        for (int p = 0; p < warp; ++p) at += static_cast<int>(ld_cluster_u32(map_to_cta(smem_u32(&sh.list_n), p)));
        const int n = static_cast<int>(ld_cluster_u32(map_to_cta(smem_u32(&sh.list_n), warp)));
        for (int i = lane; i < n; i += 32) {
          const float l = ld_cluster_f32(map_to_cta(smem_u32(&sh.list[i]), warp));
          sh.all[at + i] = l;
          if (MASS) sh.weight[at + i] = r.mass(l);
        }
      }
      __syncthreads();
      float least = INFINITY;
      if (tid < few) {
        const float l = sh.all[tid];
        unsigned long long larger = above;
        for (int j = 0; j < few; ++j)
          if (sh.all[j] > l) larger += MASS ? sh.weight[j] : 1ull;
        if (larger < target) least = l;
      }
      least = -warp_max(-least);
      if (lane == 0) sh.warp_f[warp] = least;
      __syncthreads();
      for (int w = 0; w < kDrawWarps; ++w) least = fminf(least, sh.warp_f[w]);
      __syncthreads();
      cluster_sync_all();                     // the lists may be written again
      ++round;
      return least;
    }
  }
  return floor;
}

template <typename T>
__global__ void __launch_bounds__(kDrawThreads) draw_kernel(const DrawArgs a) {
  pdl_entry();
  extern __shared__ __align__(16) float draw_buffer[];
  __shared__ DrawShared sh;
  const int b = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int begin = min(part * a.per, a.V), n = min(a.V - begin, a.per);
  const T* src = static_cast<const T*>(a.logits) + b * a.ld + begin;
  int shift;
  float m = draw_load(src, n, draw_buffer, shift);
  const float* z = draw_buffer + shift;
  m = warp_max(m);
  if (lane == 0) sh.warp_f[warp] = m;
  __syncthreads();
  for (int w = 0; w < kDrawWarps; ++w) m = fmaxf(m, sh.warp_f[w]);
  if (tid == 0) sh.part_max = m;
  cluster_sync_all();
  for (int p = 0; p < a.parts; ++p) m = fmaxf(m, ld_cluster_f32(map_to_cta(smem_u32(&sh.part_max), p)));

  const float temperature = a.temperature ? a.temperature[b] : a.temperature_all;
  const bool greedy = !(temperature > 0.f);
  const float t = greedy ? 1.f : temperature;
  DrawRow r{z, n, a.parts, part, m, 1.f / t, 1.4426950408889634 / static_cast<double>(t)};
  if (m == -INFINITY) {                      // nothing to draw from
    if (part == 0 && tid == 0) {
      a.tokens[b] = 0;
      a.logprobs[b] = -INFINITY;
    }
    cluster_sync_all();
    return;
  }
  // denominator of the unrestricted row
  float sum = 0.f;
  int first = 0x7fffffff;
  for (int i = tid; i < n; i += kDrawThreads) {
    const float l = z[i];
    sum += l == m ? 1.f : __expf((l - m) * r.inv_t);
    if (l == m) first = min(first, begin + i);
  }
  sum = warp_sum(sum);
  first = __reduce_min_sync(0xffffffffu, first);
  __syncthreads();
  if (lane == 0) {
    sh.warp_f[warp] = sum;
    sh.warp_i[warp] = first;
  }
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kDrawWarps; ++w) {
      sum += sh.warp_f[w];
      first = min(first, sh.warp_i[w]);
    }
    sh.part_sum = sum;
    sh.part_first = first;
  }
  __syncthreads();
  auto whole_sum = [&]() {
    float s = 0.f;
    for (int p = 0; p < a.parts; ++p) s += ld_cluster_f32(map_to_cta(smem_u32(&sh.part_sum), p));
    return s;
  };
  if (greedy) {
    cluster_sync_all();
    if (part == 0 && tid == 0) {
      for (int p = 0; p < a.parts; ++p) first = min(first, static_cast<int>(ld_cluster_u32(map_to_cta(smem_u32(&sh.part_first), p))));
      a.tokens[b] = first;
      a.logprobs[b] = -logf(whole_sum());
    }
    cluster_sync_all();
    return;
  }

  // what stays: logits >= threshold
  float threshold = -INFINITY;
  int round = 0;
  const int k = a.top_k ? a.top_k[b] : a.top_k_all;
  if (k > 0 && k < a.V) threshold = draw_threshold<false>(r, sh, -INFINITY, static_cast<unsigned long long>(k), 0ull, round);
  const float mp = fminf(a.min_p ? a.min_p[b] : a.min_p_all, 1.f);
  if (mp > 0.f && m < INFINITY) {
    // the least fp32 number l with (l - m) / T >= log(min_p), in 64 bits; from a rounded guess it is a step or two
    const double need = log(static_cast<double>(mp)) * static_cast<double>(t);
    auto stays = [&](float l) { return static_cast<double>(l) - static_cast<double>(m) >= need; };
    float l = static_cast<float>(static_cast<double>(m) + need);
    for (int i = 0; i < 4 && !stays(l); ++i) l = draw_unkey(draw_key(l) + 1u);
    for (int i = 0; i < 4 && l > -INFINITY && stays(draw_unkey(draw_key(l) - 1u)); ++i) l = draw_unkey(draw_key(l) - 1u);
    threshold = fmaxf(threshold, fminf(l, m));
  }
  const float p = a.top_p ? a.top_p[b] : a.top_p_all;
  if (p < 1.f) {
    const unsigned long long share = p > 0.f ? static_cast<unsigned long long>(static_cast<double>(p) * 18446744073709551616.0) : 0ull;
    threshold = fmaxf(threshold, draw_threshold<true>(r, sh, threshold, 0ull, share, round));
  }

  // masses of what stays, in whole ranges of a warp
  const int range = (n + kDrawWarps * 32 - 1) / (kDrawWarps * 32) * 32;
  const int lo = min(warp * range, n), hi = min(lo + range, n);
  unsigned long long mine = 0;
  for (int i = lo + lane; i < hi; i += 32)
    if (z[i] >= threshold) mine += r.mass(z[i]);
  mine = warp_sum_u64(mine);
  if (lane == 0) sh.warp_mass[warp] = mine;
  cluster_sync_all();
  if (warp == 0) {
    // 16 ranges of up to 8 parts, four a lane
    unsigned long long v[4], total = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int q = lane * 4 + j;
      v[j] = q / kDrawWarps < a.parts ? ld_cluster_u64(map_to_cta(smem_u32(&sh.warp_mass[q % kDrawWarps]), q / kDrawWarps)) : 0ull;
      total += v[j];
    }
    const unsigned long long upto = warp_scan_u64(total, lane);
    const unsigned long long all = __shfl_sync(0xffffffffu, upto, 31);
    unsigned long long u;
    if (a.u == nullptr) {
      const uint32_t step = a.step ? static_cast<uint32_t>(*a.step) : 0u;
      const uint32_t base = draw_hash(a.seed ^ (step * 0x9E3779B9u)) ^ draw_hash(static_cast<uint32_t>(b) * 0x85ebca6bU + 1u);
      u = static_cast<unsigned long long>(draw_hash(base + 0x9E3779B9u)) << 32 | draw_hash(base ^ 0x85ebca6bU);
    } else {
      const double x = a.u64 ? static_cast<const double*>(a.u)[b] : static_cast<double>(static_cast<const float*>(a.u)[b]);
      // 1 and above, and what is not a number, stand for the last number below 1
      u = x < 1.0 ? (x > 0.0 ? static_cast<unsigned long long>(x * 18446744073709551616.0) : 0ull) : ~0ull;
    }
    const unsigned long long target = __umul64hi(u, all);       // floor(u all) < all
    unsigned long long before = upto - total;
    if (before <= target && target < upto) {
      int j = 0;
#pragma unroll
      for (int i = 0; i < 3; ++i)
        if (j == i && target >= before + v[i]) {
          before += v[i];
          j = i + 1;
        }
      sh.owner = lane * 4 + j;
      sh.before = target - before;            // within the range
    }
  }
  __syncthreads();
  if (sh.owner / kDrawWarps == part && sh.owner % kDrawWarps == warp) {
    const unsigned long long target = sh.before;
    // runs of the range, one a lane; then the run element by element
    const int run = (hi - lo + 31) / 32, r0 = min(lo + lane * run, hi), r1 = min(r0 + run, hi);
    unsigned long long s = 0;
    for (int i = r0; i < r1; ++i)
      if (z[i] >= threshold) s += r.mass(z[i]);
    const unsigned long long upto = warp_scan_u64(s, lane);
    const int at = __ffs(__ballot_sync(0xffffffffu, target < upto)) - 1;
    unsigned long long before = __shfl_sync(0xffffffffu, upto - s, at);
    const int e0 = __shfl_sync(0xffffffffu, r0, at), e1 = __shfl_sync(0xffffffffu, r1, at);
    for (int i0 = e0; i0 < e1; i0 += 32) {
      const int i = i0 + lane;
      const unsigned long long w = i < e1 && z[i] >= threshold ? r.mass(z[i]) : 0ull;
      const unsigned long long sum_w = before + warp_scan_u64(w, lane);
      const unsigned hit = __ballot_sync(0xffffffffu, target < sum_w);
      if (hit) {
        if (lane == __ffs(hit) - 1) {
          a.tokens[b] = begin + i;
          const double x = z[i] == m ? 0.0 : (static_cast<double>(z[i]) - static_cast<double>(m)) / static_cast<double>(t);
          a.logprobs[b] = static_cast<float>(x - static_cast<double>(logf(whole_sum())));
        }
        break;
      }
      before = __shfl_sync(0xffffffffu, sum_w, 31);
    }
  }
  cluster_sync_all();                         // nobody leaves while its shared memory may be read
}

template <typename T>
static int launch_draw(DrawArgs a, int B, cudaStream_t s) {
  // parts of about 19000 elements, two CTAs of which an SM holds; more parts where rows are too few for the GPU
  int parts = 1;
  while (parts < 8 && ((a.V + parts - 1) / parts > 20480 || (static_cast<long long>(B) * parts * 2 <= 2 * sm_count() && a.V / parts > 4096))) parts *= 2;
  a.parts = parts;
  a.per = ((a.V + parts - 1) / parts + 7) / 8 * 8;
  if (a.per > kDrawMaxPart) return kBadArgument;
  const size_t smem = (static_cast<size_t>(a.per) + 4) * sizeof(float);
  static int allowed[64] = {0};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!allowed[dev & 63]) {
    const cudaError_t e = cudaFuncSetAttribute(draw_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (kDrawMaxPart + 4) * 4);
    if (e != cudaSuccess) return static_cast<int>(e);
    allowed[dev & 63] = 1;
  }
  return static_cast<int>(launch_kernel_clusters(draw_kernel<T>, dim3(static_cast<unsigned>(B) * parts), dim3(kDrawThreads), smem, parts, s, a));
}

}  // namespace apb

extern "C" {

// logits [B, V], row stride ld: type 0 fp32, 1 bf16, 2 fp16.  Of each setting a tensor [B] (fp32, top_k int32) or null and one number
// for all rows: temperature (<= 0: the first of the largest logits), top_k (<= 0: off), top_p (>= 1: off), min_p (<= 0: off).  u [B] in
// [0, 1): fp32, or fp64 with u64; null: a hash of seed, *step (null: 0) and the row.  tokens [B] int32, logprobs [B] fp32.  V up to 8 * 49152.
int apb_draw(const void* logits, int type, long long ld, const float* temperature, float temperature_all, const int* top_k, int top_k_all,
             const float* top_p, float top_p_all, const float* min_p, float min_p_all, const void* u, int u64, unsigned seed, const int* step,
             int B, int V, int* tokens, float* logprobs, cudaStream_t s) {
  using namespace apb;
  if (B <= 0) return 0;
  if (!logits || !tokens || !logprobs || V < 1 || V > 8 * kDrawMaxPart || type < 0 || type > 2) return kBadArgument;
  DrawArgs a{logits, ld, temperature, top_k, top_p, min_p, temperature_all, top_p_all, min_p_all, top_k_all,
             u, step, static_cast<uint32_t>(seed), u64, V, 1, 0, tokens, logprobs};
  if (type == 0) return launch_draw<float>(a, B, s);
  if (type == 1) return launch_draw<__nv_bfloat16>(a, B, s);
  return launch_draw<__half>(a, B, s);
}
}
