// The k most likely tokens of rows of logits, largest first, the lowest index first where logits are equal; their log-probabilities and the log of
// the mass of all other tokens.
//
// Mathematics.  One pass.  A candidate is a logit's order and its index in one 64-bit number, larger for larger logits and, of equal ones, for
// the lower index, so that the k largest numbers are the answer.  A buffer takes what is above the k-th largest number seen when it was
// last sorted; what falls out of it, or never was above that, can no longer be among the k and adds exp(l) to the sum of the others.  That sum
// is therefore formed from them alone: one minus the named tokens' share would keep nothing of it where they hold all but a little.
//
// Layout.  One CTA walks a row, or each CTA of a cluster a part of it where rows are few, and the first one sorts what the others kept.
#include "common.cuh"
#include "host_utils.cuh"

namespace apb {

constexpr int kTopThreads = 1024;
constexpr int kTopRoom = 2048;            // candidates that the buffer holds
constexpr int kTopMost = 1024;            // k

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
__device__ __forceinline__ float top_value(unsigned long long c) {
  const uint32_t k = static_cast<uint32_t>(c >> 32);
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
__device__ __forceinline__ unsigned long long top_candidate(float z, int i) {
  return static_cast<unsigned long long>(top_key(z)) << 32 | (0xffffffffu - static_cast<uint32_t>(i));
}

// Sum of exp((l - m) scale) against a running maximum.
struct TopSum {
  float m = -INFINITY, s = 0.f;
  __device__ __forceinline__ void add(float z) {
    if (z > m) {
      s = (m == -INFINITY ? 0.f : s * __expf(m - z)) + 1.f;
      m = z;
    } else if (z > -INFINITY) {
      s += z == m ? 1.f : __expf(z - m);
    }
  }
  __device__ __forceinline__ void join(float m2, float s2) {
    const float mn = fmaxf(m, m2);
    if (mn == -INFINITY) return;
    s = (m == mn ? s : s * __expf(m - mn)) + (m2 == mn ? s2 : s2 * __expf(m2 - mn));
    m = mn;
  }
};

// The buffer in falling order (all threads).
__device__ void top_sort(unsigned long long* buf) {
  for (int size = 2; size <= kTopRoom; size <<= 1)
    for (int stride = size >> 1; stride > 0; stride >>= 1) {
      __syncthreads();
      const int i = 2 * threadIdx.x - (threadIdx.x & (stride - 1)), j = i + stride;
      const unsigned long long a = buf[i], b = buf[j];
      if ((a < b) == ((i & size) == 0)) {
        buf[i] = b;
        buf[j] = a;
      }
    }
  __syncthreads();
}

template <typename T>
__global__ void __launch_bounds__(kTopThreads) top_kernel(const TopArgs a) {
  pdl_entry();
  __shared__ unsigned long long buf[kTopRoom];
  __shared__ float warp_m[32], warp_s[32], part_m, part_s;
  __shared__ int held, part_held;
  constexpr int kVec = 16 / sizeof(T);
  constexpr int kAtOnce = 8;              // elements of a thread between two looks at the buffer
  const int row = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int begin = min(part * a.per, a.V), n = min(a.V - begin, a.per), k = a.k;
  const T* src = static_cast<const T*>(a.logits) + row * a.ld + begin;
  const float scale = a.scale * (a.row_scale ? a.row_scale[row] : 1.f);
  TopSum sum;
  unsigned long long least = 0;           // the k-th largest when the buffer was last sorted; everything is above 0
  if (tid == 0) held = 0;
  __syncthreads();

  // sorts, keeps the k largest and counts the others into the sum
  auto squeeze = [&](int have) {
    for (int i = have + tid; i < kTopRoom; i += kTopThreads) buf[i] = 0;
    top_sort(buf);
    for (int i = k + tid; i < have; i += kTopThreads) sum.add(top_value(buf[i]) * scale);
    __syncthreads();
    if (tid == 0) held = min(have, k);
    least = have >= k ? buf[k - 1] : 0;
    __syncthreads();
  };
  // the elements of one step: what is not above `least` into the sum, the others into the buffer
  auto take = [&](const float (&z)[kAtOnce], const int (&at)[kAtOnce], uint32_t there) {
    uint32_t waiting = 0;
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j)
      if ((there >> j) & 1u) {
        if (top_candidate(z[j], at[j]) > least) waiting |= 1u << j;
        else sum.add(z[j] * scale);
      }
    for (;;) {
      uint32_t left = 0;
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j)
        if ((waiting >> j) & 1u) {
          const int slot = atomicAdd(&held, 1);
          if (slot < kTopRoom) buf[slot] = top_candidate(z[j], at[j]);
          else left |= 1u << j;
        }
      if (!__syncthreads_or(left != 0)) break;
      squeeze(kTopRoom);
      waiting = 0;
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j)
        if ((left >> j) & 1u) {
          if (top_candidate(z[j], at[j]) > least) waiting |= 1u << j;
          else sum.add(z[j] * scale);
        }
    }
  };
  auto number = [](T x) {
    const float f = static_cast<float>(x);
    return f == f ? f + 0.f : -INFINITY;  // what is not a number is the least likely; -0 is as large as 0
  };

  const int ahead = static_cast<int>((-(reinterpret_cast<uintptr_t>(src)) & 15) / sizeof(T));
  const int head = min(ahead, n), words = (n - head) / kVec, tail = head + words * kVec;
  const uint4* s4 = reinterpret_cast<const uint4*>(src + head);
  constexpr int kWords = kAtOnce / kVec;
  for (int w0 = 0; w0 < words; w0 += kWords * kTopThreads) {
    float z[kAtOnce];
    int at[kAtOnce];
    uint32_t there = 0;
    uint4 raw[kWords];
#pragma unroll
    for (int q = 0; q < kWords; ++q) {
      const int w = w0 + q * kTopThreads + tid;
      raw[q] = w < words ? s4[w] : make_uint4(0, 0, 0, 0);
      if (w < words) there |= ((1u << kVec) - 1u) << (q * kVec);
    }
#pragma unroll
    for (int q = 0; q < kWords; ++q) {
      const T* x = reinterpret_cast<const T*>(&raw[q]);
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        z[q * kVec + j] = number(x[j]);
        at[q * kVec + j] = begin + head + (w0 + q * kTopThreads + tid) * kVec + j;
      }
    }
    take(z, at, there);
  }
  {
    // in front of the first and behind the last whole word: at most 14 elements
    float z[kAtOnce];
    int at[kAtOnce];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      z[j] = 0.f;
      at[j] = 0;
    }
    const int i = tid < head ? tid : tail + tid - head;
    const bool one = i < n;
    if (one) {
      z[0] = number(src[i]);
      at[0] = begin + i;
    }
    take(z, at, one ? 1u : 0u);
  }
  squeeze(min(held, kTopRoom));

  // the parts' candidates into the first one's buffer
  float m = warp_max(sum.m);
  float s = sum.m == -INFINITY ? 0.f : sum.s * __expf(sum.m - m);
  s = warp_sum(s);
  if (lane == 0) {
    warp_m[warp] = m;
    warp_s[warp] = s;
  }
  __syncthreads();
  if (a.parts > 1) {
    if (warp == 0) {
      const float wm = warp_m[lane], mm = warp_max(wm);
      const float ss = warp_sum(wm == -INFINITY ? 0.f : warp_s[lane] * __expf(wm - mm));
      if (lane == 0) {
        part_m = mm;
        part_s = ss;
        part_held = held;
      }
    }
    cluster_sync_all();
    if (part == 0) {
      int have = held;
      sum.m = -INFINITY;
      sum.s = 0.f;
      for (int p = 0; p < a.parts; ++p) {
        if (tid == 0)
          sum.join(ld_cluster_f32(map_to_cta(smem_u32(&part_m), p)), ld_cluster_f32(map_to_cta(smem_u32(&part_s), p)));
        if (p == 0) continue;
        int other;
        asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(other) : "r"(map_to_cta(smem_u32(&part_held), p)) : "memory");
        for (int i = tid; i < other; i += kTopThreads) {
          unsigned long long c;
          asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(c) : "r"(map_to_cta(smem_u32(&buf[i]), p)) : "memory");
          buf[have + i] = c;
        }
        have += other;                    // parts * k <= kTopRoom
      }
      __syncthreads();
      squeeze(have);
      m = warp_max(sum.m);
      s = warp_sum(sum.m == -INFINITY ? 0.f : sum.s * __expf(sum.m - m));
      if (lane == 0) {
        warp_m[warp] = m;
        warp_s[warp] = s;
      }
      __syncthreads();
    }
    cluster_sync_all();                   // nobody leaves while its buffer may be read
    if (part != 0) return;
  }

  // denominator: the others and the k
  const float top = top_value(buf[0]) * scale;
  __shared__ float named_sum;
  __syncthreads();
  float others_m = -INFINITY, others = 0.f;
  if (warp == 0) {
    const float wm = warp_m[lane];
    others_m = warp_max(wm);
    others = warp_sum(wm == -INFINITY ? 0.f : warp_s[lane] * __expf(wm - others_m));
  }
  float named = 0.f;
  for (int i = tid; i < k; i += kTopThreads) {
    const float z = top_value(buf[i]) * scale;
    named += z == top ? 1.f : expf(z - top);
  }
  named = warp_sum(named);
  __syncthreads();
  if (lane == 0) warp_s[warp] = named;
  __syncthreads();
  if (warp == 0) {
    named = warp_sum(warp_s[lane]);
    const float log_others = others_m == -INFINITY ? -INFINITY : others_m - top + logf(others);     // also where the share itself is 0
    others = expf(log_others);
    if (lane == 0) {
      const float log_all = logf(named + others);
      named_sum = log_all;
      // near 1 the logarithm of the others' share is that of one minus the named tokens'
      a.rest[row] = top == -INFINITY ? -INFINITY : named < others ? log1pf(-named / (named + others)) : log_others - log_all;
    }
  }
  __syncthreads();
  for (int i = tid; i < k; i += kTopThreads) {
    const float z = top_value(buf[i]) * scale;
    a.ids[static_cast<long long>(row) * k + i] = static_cast<int>(0xffffffffu - static_cast<uint32_t>(buf[i]));
    a.logprobs[static_cast<long long>(row) * k + i] = top == -INFINITY ? -INFINITY : (z == top ? 0.f : z - top) - named_sum;
  }
}

template <typename T>
static int launch_top(TopArgs a, int N, cudaStream_t s) {
  // parts of a row where the GPU has room for more CTAs than rows (two a SM), as long as their candidates fit the first one's buffer
  int parts = 1;
  while (parts < 8 && static_cast<long long>(N) * parts * 2 <= 2 * sm_count() && a.V / parts > 8192 && 2 * parts * a.k <= kTopRoom) parts *= 2;
  a.parts = parts;
  a.per = ((a.V + parts - 1) / parts + 7) / 8 * 8;
  return static_cast<int>(launch_kernel_clusters(top_kernel<T>, dim3(static_cast<unsigned>(N) * parts), dim3(kTopThreads), 0, parts, s, a));
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
