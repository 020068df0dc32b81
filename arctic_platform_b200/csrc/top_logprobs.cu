// The k most likely tokens of rows of logits, largest first, the lowest index first where logits are equal; their log-probabilities and the log of
// the mass of all other tokens.
//
// Mathematics.  One pass.  A candidate is a logit's order and its index in one 64-bit number, larger for larger logits and, of equal ones, for
// the lower index, so that the k largest numbers are the answer.  A buffer takes what reaches a bound that k candidates are known to reach: at
// first k of the threads' largest ones, later k of the buffer, whenever it has grown; what falls out of the buffer, or never reached the
// bound, can no longer be among the k and adds exp(l) to the sum of the others.  That sum is therefore formed from them alone: one minus
// the named tokens' share would keep nothing of it where they hold all but a little.  A bound is found bit by bit, by counting what
// reaches it, and only until few more than k do (2000 cycles; sorting the buffer of 1024 instead took 17000, and 0.69 ms the pass over 2048
// rows of 151936 where HBM wants 0.19).
//
// Layout.  One CTA walks a row, or each CTA of a cluster a part of it where rows are few, and the first one sorts what all have kept.
//
// Measured: 2048 rows of 151936 in fp32, k = 64, 344 us (3.6 TB/s, issue slots 66 % busy: instructions bound it); 256 rows of 248320 in bf16, k = 128,
// 100 us; 333 rows of 32000, k = 20, 29 us.
#include "common.cuh"
#include "host_utils.cuh"

namespace apb {

constexpr int kTopMost = 1024;            // k
constexpr float kTopLog2e = 1.44269504088896340736f;

struct TopArgs {
  const void* logits;
  long long ld;
  const float* row_scale;                 // [N] or null
  float scale;
  int V, k, parts, per;
  float* logprobs;                        // [N, k]
  int* ids;                               // [N, k]
  float* rest;                            // [N]
};

__device__ __forceinline__ uint32_t top_key(float z) {
  const uint32_t u = __float_as_uint(z);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float top_unkey(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }
__device__ __forceinline__ float top_value(unsigned long long c) { return top_unkey(static_cast<uint32_t>(c >> 32)); }
__device__ __forceinline__ unsigned long long top_candidate(float z, int i) {
  return static_cast<unsigned long long>(top_key(z)) << 32 | (0xffffffffu - static_cast<uint32_t>(i));
}

// 2^((z - ref) scale2), z <= ref: the difference first, as a product of a large logit would lose the digits that tell it from its neighbours.
__device__ __forceinline__ float top_power(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float top_mass(float z, float ref, float scale2) { return z == ref ? 1.f : top_power((z - ref) * scale2); }

// 64 entries of a warp, a: those of lane, b: those 32 behind; steps of a bitonic network over runs of `run` that begin `stride` apart, for entries
// whose place is base + lane and base + 32 + lane.
__device__ __forceinline__ void top_steps(unsigned long long& a, unsigned long long& b, int base, int run, int stride) {
  const int lane = threadIdx.x & 31;
  if (stride == 32) {
    if ((a < b) == (((base + lane) & run) == 0)) {
      const unsigned long long t = a;
      a = b;
      b = t;
    }
    stride = 16;
  }
  for (; stride > 0; stride >>= 1) {
    const unsigned long long c = __shfl_xor_sync(0xffffffffu, a, stride), d = __shfl_xor_sync(0xffffffffu, b, stride);
    const bool first = (lane & stride) == 0;
    const bool larger_a = first == (((base + lane) & run) == 0), larger_b = first == (((base + 32 + lane) & run) == 0);
    a = (a < c) == larger_a ? c : a;
    b = (b < d) == larger_b ? d : b;
  }
}
__device__ __forceinline__ void top_sort_64(unsigned long long& a, unsigned long long& b, int base) {
  for (int run = 2; run <= 64; run <<= 1) top_steps(a, b, base, run, run >> 1);
}

// The first `size` (a power of 2 from 64 on) entries of the buffer in falling order (all threads).  Entries at most 32 apart meet in a warp's
// registers, those further apart in shared memory.
template <int THREADS>
__device__ void top_sort(unsigned long long* buf, int size) {
  const int lane = threadIdx.x & 31;
  __syncthreads();
  for (int base = (threadIdx.x >> 5) * 64; base < size; base += 2 * THREADS) {
    unsigned long long a = buf[base + lane], b = buf[base + 32 + lane];
    top_sort_64(a, b, base);
    buf[base + lane] = a;
    buf[base + 32 + lane] = b;
  }
  __syncthreads();
  for (int run = 128; run <= size; run <<= 1) {
    for (int stride = run >> 1; stride >= 64; stride >>= 1) {
      for (int t = threadIdx.x; t < size / 2; t += THREADS) {
        const int i = 2 * t - (t & (stride - 1)), j = i + stride;
        const unsigned long long a = buf[i], b = buf[j];
        if ((a < b) == ((i & run) == 0)) {
          buf[i] = b;
          buf[j] = a;
        }
      }
      __syncthreads();
    }
    for (int base = (threadIdx.x >> 5) * 64; base < size; base += 2 * THREADS) {
      unsigned long long a = buf[base + lane], b = buf[base + 32 + lane];
      top_steps(a, b, base, run, 32);
      buf[base + lane] = a;
      buf[base + 32 + lane] = b;
    }
    __syncthreads();
  }
}

// A number that at least `want` candidates reach, of each thread one or two (TWO) by their orders' keys (0: none): each warp's share-th largest, the
// least of these.  0 where a warp has too few.  About twice `want` reach it if they lie in any order.
template <int THREADS, bool TWO>
__device__ unsigned long long top_rough_bound(uint32_t a, uint32_t b, int want, unsigned long long* ends) {
  constexpr int kWarps = THREADS / 32;
  const int lane = threadIdx.x & 31, share = (want + kWarps - 1) / kWarps - 1;         // index of it
  if (share >= (TWO ? 64 : 32)) return 0;
#pragma unroll
  for (int run = 2; run <= (TWO ? 64 : 32); run <<= 1) {
    if (TWO && run == 64) {
      const uint32_t t = max(a, b);
      b = min(a, b);
      a = t;
    }
#pragma unroll
    for (int stride = run == 64 ? 16 : run >> 1; stride > 0; stride >>= 1) {
      const uint32_t c = __shfl_xor_sync(0xffffffffu, a, stride);
      const bool first = (lane & stride) == 0;
      const bool falls = run == 32 || run == 64 || (lane & run) == 0;         // of 64 the first 32 fall, the others rise until they meet
      a = first == falls ? max(a, c) : min(a, c);
      if (TWO) {
        const uint32_t d = __shfl_xor_sync(0xffffffffu, b, stride);
        const bool falls_b = run == 64 || (run == 32 ? false : (lane & run) == 0);
        b = first == falls_b ? max(b, d) : min(b, d);
      }
    }
  }
  const uint32_t low = __shfl_sync(0xffffffffu, share < 32 ? a : b, share & 31);
  if (lane == 0) ends[threadIdx.x >> 5] = static_cast<unsigned long long>(low) << 32;
  __syncthreads();
  unsigned long long x = ends[0];
  for (int w = 1; w < kWarps; ++w) x = ends[w] < x ? ends[w] : x;
  return x;
}

// A number that at least `want` of the CTA's candidates reach (E of a thread, 0: none), the largest one with so many unless no more than
// `enough` reach a smaller one already.
template <int THREADS, int E>
__device__ unsigned long long top_bound(const unsigned long long (&c)[E], int want, int enough, unsigned long long (&ends)[2][THREADS / 32]) {
  // the bits that all have in common need no counting
  unsigned long long lo = ~0ull, hi = 0;
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (c[e] != 0) {
      lo = c[e] < lo ? c[e] : lo;
      hi = c[e] > hi ? c[e] : hi;
    }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long a = __shfl_xor_sync(0xffffffffu, lo, o), b = __shfl_xor_sync(0xffffffffu, hi, o);
    lo = a < lo ? a : lo;
    hi = b > hi ? b : hi;
  }
  if ((threadIdx.x & 31) == 0) {
    ends[0][threadIdx.x >> 5] = lo;
    ends[1][threadIdx.x >> 5] = hi;
  }
  __syncthreads();
  for (int w = 0; w < THREADS / 32; ++w) {
    lo = ends[0][w] < lo ? ends[0][w] : lo;
    hi = ends[1][w] > hi ? ends[1][w] : hi;
  }
  const int from = 63 - __clzll(static_cast<long long>(lo ^ hi));           // the highest bit in which they differ, -1: none
  unsigned long long x = from < 0 ? lo : from == 63 ? 0ull : hi >> (from + 1) << (from + 1);
#pragma unroll 1
  for (int bit = from; bit >= 0; --bit) {
    const unsigned long long t = x | 1ull << bit;
    int reach = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) reach += __syncthreads_count(c[e] >= t);
    if (reach >= want) {
      x = t;
      if (reach <= enough) break;
    }
  }
  return x;
}

template <typename T, int ROOM, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) top_kernel(const TopArgs a) {
  pdl_entry();
  __shared__ unsigned long long buf[ROOM];
  __shared__ float warp_s[THREADS / 32], part_ref, part_s, shared_log;
  __shared__ int held, part_held;
  __shared__ unsigned long long ends[2][THREADS / 32];
  constexpr int kVec = 16 / sizeof(T);
  constexpr int kAtOnce = 16;             // elements of a thread between two looks at the buffer
  constexpr int kWords = kAtOnce / kVec;
  constexpr int kWarps = THREADS / 32;
  const int row = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int begin = min(part * a.per, a.V), n = min(a.V - begin, a.per), k = a.k;
  const T* src = static_cast<const T*>(a.logits) + row * a.ld + begin;
  const float scale2 = a.scale * (a.row_scale ? a.row_scale[row] : 1.f) * kTopLog2e;
  constexpr int kOwn = ROOM / THREADS;              // candidates of the buffer that a thread looks at
  float sum = 0.f, ref = -INFINITY;                     // of the others' masses against `ref`, which none of them is above
  float bound_z = -INFINITY;                            // candidates reach the bound with more than this, or with as much and no higher index
  int bound_i = 0x7fffffff;
  unsigned long long bound = 0;
  const int crowd = max(ROOM / 2, k + ROOM / 4);        // held entries from which on a new bound pays
  const int loose = k + k / 4 + 8;                      // candidates that a bound may leave before the last
  if (tid == 0) held = 0;
  __syncthreads();

  auto set_bound = [&](unsigned long long x) {
    const uint32_t key = static_cast<uint32_t>(x >> 32), low = static_cast<uint32_t>(x);
    if (x <= bound || key < 0x007fffffu) return;        // below -inf: all reach it
    bound = x;
    bound_z = key == 0x7fffffffu ? 0.f : top_unkey(key);            // the place of -0, which no candidate has
    bound_i = key == 0x7fffffffu || low < 0x80000000u ? 0x7fffffff : static_cast<int>(0xffffffffu - low);
    sum = sum == 0.f ? 0.f : sum * top_mass(ref, bound_z, scale2);
    ref = bound_z;
  };
  auto reaches = [&](float z, int at) { return z > bound_z || (z == bound_z && at <= bound_i); };
  // a new bound, which at least k of the `have` entries of the buffer reach, as `enough` says; what does not goes into the sum
  auto squeeze = [&](int have, int enough, bool last) {
    unsigned long long c[kOwn];
#pragma unroll
    for (int e = 0; e < kOwn; ++e) c[e] = tid + e * THREADS < have ? buf[tid + e * THREADS] : 0;
    if (have > k) {
      // roughly first, if that leaves few enough
      unsigned long long x = 0;
      if (kOwn == 2 && !last) {
        x = top_rough_bound<THREADS, true>(static_cast<uint32_t>(c[0] >> 32), static_cast<uint32_t>(c[1] >> 32), k, ends[0]);
        int reach = 0;
#pragma unroll
        for (int e = 0; e < kOwn; ++e) reach += __syncthreads_count(c[e] != 0 && c[e] >= x);
        if (reach > crowd - ROOM / 8) x = 0;
      }
      if (x == 0) x = top_bound<THREADS>(c, k, enough, ends);
      if (tid == 0) held = 0;
      __syncthreads();
      set_bound(x);
#pragma unroll
      for (int e = 0; e < kOwn; ++e) {
        if (c[e] >= x && c[e] != 0) buf[atomicAdd(&held, 1)] = c[e];
        else if (c[e] != 0 && top_value(c[e]) > -INFINITY) sum += top_mass(top_value(c[e]), ref, scale2);
      }
    } else if (tid == 0) {
      held = have;
    }
    __syncthreads();
  };
  auto clean = [](float f) { return f == f ? f + 0.f : -INFINITY; };     // no number: the least likely; -0 is as large as 0
  // the elements of one step, as they are: what does not reach the bound into the sum, the others into the buffer
  auto take = [&](float (&z)[kAtOnce], int at0, uint32_t there) {
    auto at = [&](int j) { return at0 + (j / kVec) * THREADS * kVec + j % kVec; };
    float most = z[0];
#pragma unroll
    for (int j = 1; j < kAtOnce; ++j) most = fmaxf(most, z[j]);
    // what is below the bound goes into the sum; no number is below it, places without an element hold -inf
    float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      const float y = top_power((z[j] - ref) * scale2);
      s[j & 3] += z[j] < bound_z ? y : 0.f;
    }
    sum += (s[0] + s[1]) + (s[2] + s[3]);
    uint32_t waiting = 0;
    if (most >= bound_z || bound_z == -INFINITY) {
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j)
        if (!(z[j] < bound_z)) waiting |= 1u << j;
      waiting &= there;
    }
    for (;;) {
      uint32_t left = 0;
      bool full = false;
      while (waiting) {
        const int j = __ffs(waiting) - 1;
        waiting &= waiting - 1;
        float zj = z[0];
#pragma unroll
        for (int i = 1; i < kAtOnce; ++i)
          if (i == j) zj = z[i];
        zj = clean(zj);
        if (!reaches(zj, at(j))) {
          if (zj > -INFINITY) sum += top_mass(zj, ref, scale2);
          continue;
        }
        const int slot = atomicAdd(&held, 1);
        if (slot < ROOM) buf[slot] = top_candidate(zj, at(j));
        else left |= 1u << j;
        full |= slot >= crowd;
      }
      if (!__syncthreads_or(left != 0 || full)) break;
      const int have = min(held, ROOM);
      __syncthreads();
      squeeze(have, loose, false);
      if (!__syncthreads_or(left != 0)) break;
      waiting = left;
    }
  };
  auto number = [&](T x) { return clean(static_cast<float>(x)); };

  const int ahead = static_cast<int>((-(reinterpret_cast<uintptr_t>(src)) & 15) / sizeof(T));
  const int head = min(ahead, n), words = (n - head) / kVec, tail = head + words * kVec;
  const uint4* s4 = reinterpret_cast<const uint4*>(src + head);
  auto fetch = [&](uint4 (&raw)[kWords], int w0) {
#pragma unroll
    for (int q = 0; q < kWords; ++q) {
      const int w = w0 + q * THREADS + tid;
      raw[q] = w < words ? __ldcs(s4 + w) : make_uint4(0, 0, 0, 0);
    }
  };
  uint4 next[kWords];
  fetch(next, 0);
  for (int w0 = 0; w0 < words; w0 += kWords * THREADS) {
    float z[kAtOnce];
    uint32_t there = 0;
#pragma unroll
    for (int q = 0; q < kWords; ++q) {
      const T* x = reinterpret_cast<const T*>(&next[q]);
#pragma unroll
      for (int j = 0; j < kVec; ++j) z[q * kVec + j] = static_cast<float>(x[j]);
      if (w0 + q * THREADS + tid < words) {
        there |= ((1u << kVec) - 1u) << (q * kVec);
      } else {
#pragma unroll
        for (int j = 0; j < kVec; ++j) z[q * kVec + j] = -INFINITY;
      }
    }
    fetch(next, w0 + kWords * THREADS);
    const int at0 = begin + head + (w0 + tid) * kVec;
    if (w0 == 0 && k <= THREADS && words > THREADS) {
      // of the threads' largest elements k reach the bound.  Every thread has at least its first word.
      uint32_t best = 0;
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j)
        if ((there >> j) & 1u) best = max(best, top_key(clean(z[j])));
      set_bound(top_rough_bound<THREADS, false>(best, 0, k, ends[0]));
    }
    take(z, at0, there);
  }
  {
    // in front of the first and behind the last whole word: at most 14 elements
    float z[kAtOnce];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) z[j] = -INFINITY;
    const int i = tid < head ? tid : tail + tid - head;
    if (i < n) z[0] = static_cast<float>(src[i]);
    take(z, begin + i, i < n ? 1u : 0u);
  }
  const int sorted = max(64, 1 << (32 - __clz(k - 1 | 1)));         // entries that are sorted in the end: a power of 2, at least k
  {
    const int have = min(held, ROOM);
    __syncthreads();
    squeeze(have, a.parts > 1 ? ROOM / a.parts : sorted, true);
  }

  // a sum over the CTA
  auto join = [&](float s) {
    s = warp_sum(s);
    if (lane == 0) warp_s[warp] = s;
    __syncthreads();
    s = 0.f;
    for (int w = 0; w < kWarps; ++w) s += warp_s[w];
    __syncthreads();
    return s;
  };
  // in order; what is behind the k goes to the others, against the k-th, which no reference is above
  auto finish = [&](int have) {
    for (int i = have + tid; i < sorted; i += THREADS) buf[i] = 0;
    top_sort<THREADS>(buf, sorted);
    const float last = top_value(buf[k - 1]);
    sum = sum == 0.f ? 0.f : sum * top_mass(ref, last, scale2);
    ref = last;
    for (int i = k + tid; i < sorted; i += THREADS)
      if (buf[i] != 0 && top_value(buf[i]) > -INFINITY) sum += top_mass(top_value(buf[i]), ref, scale2);
  };
  int have = held;
  if (a.parts > 1) {
    const float s = join(sum);
    if (tid == 0) {
      part_ref = ref;
      part_s = s;
      part_held = have;
    }
    cluster_sync_all();
    if (part == 0) {
      for (int p = 1; p < a.parts; ++p) {
        int other;
        asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(other) : "r"(map_to_cta(smem_u32(&part_held), p)) : "memory");
        for (int i = tid; i < other; i += THREADS) {
          unsigned long long c;
          asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(c) : "r"(map_to_cta(smem_u32(&buf[i]), p)) : "memory");
          buf[have + i] = c;
        }
        have += other;                    // each has at most ROOM / parts
      }
      sum = 0.f;
      __syncthreads();
      squeeze(have, sorted, true);
      finish(held);
      if (tid == 0)
        for (int p = 0; p < a.parts; ++p) {
          const float r = ld_cluster_f32(map_to_cta(smem_u32(&part_ref), p)), t = ld_cluster_f32(map_to_cta(smem_u32(&part_s), p));
          if (!(t <= 0.f)) sum += t * top_mass(r, ref, scale2);
        }
    }
    cluster_sync_all();                   // nobody leaves while its buffer may be read
    if (part != 0) return;
  } else {
    finish(have);
  }
  float others = join(sum);

  // denominator: the others and the k
  const float top = top_value(buf[0]);
  const float scale = a.scale * (a.row_scale ? a.row_scale[row] : 1.f);
  float log_others = -INFINITY;           // against `top`
  if (others > 1e-25f) {
    log_others = (ref == top ? 0.f : (ref - top) * scale) + logf(others);
  } else if (k < a.V && top_value(buf[k - 1]) > -INFINITY) {
    // all of them so far below the k-th (57 nats) that their masses against it are lost, or among them what is no number: the row again, against
    // their largest
    const T* all = static_cast<const T*>(a.logits) + row * a.ld;
    const unsigned long long last = buf[k - 1];
    float most = -INFINITY;
    for (int i = tid; i < a.V; i += THREADS) {
      const float z = number(all[i]);
      if (top_candidate(z, i) < last) most = fmaxf(most, z);
    }
    most = warp_max(most);
    if (lane == 0) warp_s[warp] = most;
    __syncthreads();
    for (int w = 0; w < kWarps; ++w) most = fmaxf(most, warp_s[w]);
    __syncthreads();
    sum = 0.f;
    for (int i = tid; i < a.V; i += THREADS) {
      const float z = number(all[i]);
      if (z > -INFINITY && top_candidate(z, i) < last) sum += top_mass(z, most, scale2);
    }
    others = join(sum);
    if (others > 0.f) log_others = (most - top) * scale + logf(others);
  }
  float named = 0.f;
  for (int i = tid; i < k; i += THREADS) named += top_mass(top_value(buf[i]), top, scale2);
  named = join(named);
  if (tid == 0) {
    others = expf(log_others);
    const float log_all = logf(named + others);
    shared_log = log_all;
    // near 1 the logarithm of the others' share is that of one minus the named tokens'
    a.rest[row] = top == -INFINITY ? -INFINITY : named < others ? log1pf(-named / (named + others)) : log_others - log_all;
  }
  __syncthreads();
  for (int i = tid; i < k; i += THREADS) {
    const float z = top_value(buf[i]);
    a.ids[static_cast<long long>(row) * k + i] = static_cast<int>(0xffffffffu - static_cast<uint32_t>(buf[i]));
    a.logprobs[static_cast<long long>(row) * k + i] = top == -INFINITY ? -INFINITY : (z == top ? 0.f : (z - top) * scale) - shared_log;
  }
}

template <typename T, int ROOM, int THREADS>
static int launch_top_as(TopArgs a, int N, cudaStream_t s) {
  // parts of a row where the GPU has room for more CTAs than rows, as long as their candidates fit the first one's buffer
  int parts = 1;
  while (parts < 8 && static_cast<long long>(N) * parts * 2 <= 1024 / THREADS * sm_count() && a.V / parts > 16 * THREADS && 2 * parts * a.k <= ROOM)
    parts *= 2;
  a.parts = parts;
  a.per = ((a.V + parts - 1) / parts + 7) / 8 * 8;
  return static_cast<int>(launch_kernel_clusters(top_kernel<T, ROOM, THREADS>, dim3(static_cast<unsigned>(N) * parts), dim3(THREADS), 0, parts, s, a));
}

template <typename T>
static int launch_top(const TopArgs& a, int N, cudaStream_t s) {
  // 256 threads, four CTAs an SM, wait for one another less, but their buffer is filled more often.  Where both break even goes with the rows: near
  // k = 220 for 2048 rows of 151936 (k = 64 / 96 / 128 / 192: 344 / 364 / 390 / 469 us, 412 / 422 / 446 / 475 with 512), 160 for 333 and 200 for
  // 1024 of 32000, but below 48 for 256 long rows in 16 bits (248320, k = 64 / 96 / 128 / 192: 97 / 99 / 113 / 131 us, 93 / 90 / 101 / 101)
  if (a.k <= 96) return launch_top_as<T, 512, 256>(a, N, s);
  return a.k <= 256 ? launch_top_as<T, 1024, 512>(a, N, s) : launch_top_as<T, 2048, 512>(a, N, s);
}

}  // namespace apb

extern "C" {

// logits [N, V], row stride ld: type 0 fp32, 1 bf16, 2 fp16; 1 <= k <= min(V, 1024); log-probabilities are those of logits * scale (times
// row_scale [N] where it is given), both positive.  logprobs [N, k] fp32, ids [N, k] int32, rest [N] fp32 (-inf for k = V).
int apb_top_logprobs(const void* logits, int type, long long ld, const float* row_scale, float scale, int N, int V, int k, float* logprobs,
                     int* ids, float* rest, cudaStream_t s) {
  using namespace apb;
  if (N <= 0) return 0;
  if (!logits || !logprobs || !ids || !rest || V < 1 || k < 1 || k > V || k > kTopMost || type < 0 || type > 2) return kBadArgument;
  TopArgs a{logits, ld, row_scale, scale, V, k, 1, 0, logprobs, ids, rest};
  if (type == 0) return launch_top<float>(a, N, s);
  if (type == 1) return launch_top<__nv_bfloat16>(a, N, s);
  return launch_top<__half>(a, N, s);
}
}
