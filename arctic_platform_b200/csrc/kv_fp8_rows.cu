// Rows of keys and values into the 8-bit cache and back (layout: kv_fp8.cuh).
//
// Both are bound by memory: a row of D values moves 2 D (4 D from fp32) + D + 1 bytes on its way in, D + 1 + 2 D on its way out.
// D / 8 lanes share a row, eight neighbouring values each, so that 16-byte accesses to the values and 8-byte ones to the codes cover
// whole sectors; the largest magnitude of a row is found by shuffles among them, and nothing is read twice.  (Lanes that walked over
// rows one at a time kept too little on its way, and a 64-bit division per row: 2.9 TB/s in, 4.1 out.)  Measured, 8 heads of 128, bf16:
// 16384 tokens 36 us in and out (4.7 TB/s); 36864 tokens of 4 heads 20.2 us out (5.6 TB/s, 0.86 of a copy; issue slots are 76 % busy).
#include <cuda_fp16.h>

#include "host_utils.cuh"
#include "kv_fp8.cuh"

namespace apb {

struct Kv8Rows {
  const void *k, *v;       // [T, H, D] with the given strides in elements
  long long ldk, lhk, ldv, lhv;
  const int* slots;        // page * 16 + token in the page; below 0: none
  uint8_t* data;           // [pages, H, block]
  int T, H;
  int slots_end;           // pages * 16
  int* status;
};

// Eight neighbouring values as they lie in memory.
template <typename T>
struct Eight {
  uint4 r[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) r[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    if constexpr (sizeof(T) == 2) {
      const uint32_t w[4] = {r[0].x, r[0].y, r[0].z, r[0].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        v[4 * i] = __uint_as_float(r[i].x), v[4 * i + 1] = __uint_as_float(r[i].y);
        v[4 * i + 2] = __uint_as_float(r[i].z), v[4 * i + 3] = __uint_as_float(r[i].w);
      }
    }
  }
};
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]);
template <>
__device__ __forceinline__ void store8<__nv_bfloat16>(__nv_bfloat16* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) =
      make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}
template <>
__device__ __forceinline__ void store8<float>(float* p, const float (&v)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}

// A warp takes the same 32 / kLanes rows of AT tokens behind one another, all of their loads on the way before the first is used: tokens
// that lie in one page share its exponents' sector.  AT = 4 moves the most; where there are fewer runs than fill the GPU, AT = 1 is
// sooner done (a step of 128 tokens: 2.0 us instead of 2.8).
template <int D, int AT>
struct RowsWalk {
  static constexpr int kLanes = D / 8, kRows = 32 / kLanes;
  int t, row, part;         // first token, this lane's row of the 2 H, eight values of it
  bool there;
  __device__ __forceinline__ RowsWalk(const Kv8Rows& p, int per_token) {
    const int w = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    t = w / per_token;
    row = (w - t * per_token) * kRows + lane / kLanes;
    there = row < 2 * p.H;
    t *= AT;
    part = lane % kLanes;
  }
};

template <typename T, int D, int AT>
__global__ void __launch_bounds__(256) kv8_write_kernel(const Kv8Rows p, int per_token) {
  pdl_entry();
  const RowsWalk<D, AT> at(p, per_token);
  if (at.t >= p.T) return;
  const int row = min(at.row, 2 * p.H - 1), which = row >= p.H, h = row - which * p.H;      // all lanes stay for the shuffles
  const T* from = static_cast<const T*>(which ? p.v : p.k) + h * (which ? p.lhv : p.lhk) + at.part * 8;
  const long long ld = which ? p.ldv : p.ldk;
  int slot[AT];
  Eight<T> x[AT];
#pragma unroll
  for (int i = 0; i < AT; ++i) {
    const int t = min(at.t + i, p.T - 1);
    slot[i] = at.t + i < p.T ? p.slots[t] : -1;
    x[i].load(from + t * ld);
  }
  uint8_t* const to = p.data + static_cast<long long>(h) * Kv8<D>::kBlock;
#pragma unroll
  for (int i = 0; i < AT; ++i) {
    float v[8], most = 0.f;
    x[i].get(v);
#pragma unroll
    for (int k = 0; k < 8; ++k) most = fmaxf(most, fabsf(v[k]));
#pragma unroll
    for (int o = 1; o < RowsWalk<D, AT>::kLanes; o <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    if (!at.there || slot[i] < 0) continue;
    if (slot[i] >= p.slots_end) {
      if (p.status) atomicCAS(p.status, 0, kBadTable);
      continue;
    }
    const int e = kv8_exponent(most), token = slot[i] % kKv8Page;
    const float f = exp2_int(-e);
    uint16_t c[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) c[k] = e4m3_pair(v[2 * k] * f, v[2 * k + 1] * f);
    uint8_t* block = to + static_cast<long long>(slot[i] / kKv8Page) * p.H * Kv8<D>::kBlock;
    *reinterpret_cast<uint2*>(block + which * Kv8<D>::kHalf + token * D + at.part * 8) =
        make_uint2(c[0] | static_cast<uint32_t>(c[1]) << 16, c[2] | static_cast<uint32_t>(c[3]) << 16);
    if (at.part == 0) block[2 * Kv8<D>::kHalf + kv8_exponent_at(token, which)] = static_cast<uint8_t>(e + 127);
  }
}

template <typename T, int D, int AT>
__global__ void __launch_bounds__(256) kv8_read_kernel(const Kv8Rows p, int per_token, T* out_k, T* out_v) {
  pdl_entry();
  const RowsWalk<D, AT> at(p, per_token);
  if (at.t >= p.T || !at.there) return;
  const int which = at.row >= p.H, h = at.row - which * p.H;
  const uint8_t* const from = p.data + static_cast<long long>(h) * Kv8<D>::kBlock;
  int slot[AT], e[AT];
  uint2 c[AT];
#pragma unroll
  for (int i = 0; i < AT; ++i) slot[i] = at.t + i < p.T ? p.slots[at.t + i] : -1;
#pragma unroll
  for (int i = 0; i < AT; ++i) {
    c[i] = make_uint2(0, 0);
    e[i] = 0;
    if (slot[i] >= p.slots_end) {
      if (p.status) atomicCAS(p.status, 0, kBadTable);
    } else if (slot[i] >= 0) {
      const int token = slot[i] % kKv8Page;
      const uint8_t* block = from + static_cast<long long>(slot[i] / kKv8Page) * p.H * Kv8<D>::kBlock;
      c[i] = *reinterpret_cast<const uint2*>(block + which * Kv8<D>::kHalf + token * D + at.part * 8);
      e[i] = block[2 * Kv8<D>::kHalf + kv8_exponent_at(token, which)];
    }
  }
#pragma unroll
  for (int i = 0; i < AT; ++i) {
    if (at.t + i >= p.T) break;
    const float f = exp2f(static_cast<float>(e[i]) - 127.f);
    const uint16_t pair[4] = {static_cast<uint16_t>(c[i].x), static_cast<uint16_t>(c[i].x >> 16), static_cast<uint16_t>(c[i].y),
                              static_cast<uint16_t>(c[i].y >> 16)};
    float v[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t y = e4m3_to_f16x2(pair[k]);
      const float2 z = __half22float2(*reinterpret_cast<const __half2*>(&y));
      v[2 * k] = z.x * f;
      v[2 * k + 1] = z.y * f;
    }
    store8((which ? out_v : out_k) + (static_cast<long long>(at.t + i) * p.H + h) * D + at.part * 8, v);
  }
}

// Behind the split-K qkv projection of a decode step: sums [B, (Hq + 2 H) D] in fp32 (cleared as they are read), RMSNorm and rotate-half
// RoPE of q and k per head, q to bf16, k and v rounded to bf16 and into their slots, as decode_qkv_post_kernel and kv8_write_kernel
// would leave them.  One warp per token and head; bound by launch and latency.
struct Kv8QkvPost {
  float* acc;
  long long ld_acc;
  const __nv_bfloat16 *wq, *wk;      // null: no norm
  const float *cos_t, *sin_t;        // [positions, D / 2]
  const int *pos, *slots;
  __nv_bfloat16* q_out;              // [B, Hq, D]
  uint8_t* data;
  int B, Hq, H, slots_end, positions;      // positions: rows of cos and sin
  float eps;
  int* status;
};
template <int D>
__global__ void __launch_bounds__(256) kv8_qkv_post_kernel(const Kv8QkvPost p) {
  pdl_entry();
  constexpr int E = D / 64;
  const int lane = threadIdx.x & 31, heads = p.Hq + 2 * p.H, w = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (w >= p.B * heads) return;
  const int t = w / heads, h = w - t * heads;
  float* src = p.acc + t * p.ld_acc + static_cast<long long>(h) * D;
  float a[E], b[E];
#pragma unroll
  for (int j = 0; j < E; ++j) {
    a[j] = src[lane * E + j];
    b[j] = src[D / 2 + lane * E + j];
    src[lane * E + j] = 0.f;
    src[D / 2 + lane * E + j] = 0.f;
  }
  const bool is_q = h < p.Hq, is_v = h >= p.Hq + p.H;
  const int pos = p.pos[t];
  const bool lost = static_cast<unsigned>(pos) >= static_cast<unsigned>(p.positions);      // the tables have no such row
  const int to = p.slots[t], slot = lost ? -1 : to;
  if (lost) {
    if (to >= 0 && p.status) atomicCAS(p.status, 0, kBadTable);          // of an idle row any position will do
#pragma unroll
    for (int j = 0; j < E; ++j) a[j] = b[j] = 0.f;
  } else if (!is_v) {
    const __nv_bfloat16* weight = is_q ? p.wq : p.wk;
    if (weight) {
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < E; ++j) ss += a[j] * a[j] + b[j] * b[j];
      const float rstd = rsqrtf(warp_sum(ss) / D + p.eps);
#pragma unroll
      for (int j = 0; j < E; ++j) {
        a[j] *= rstd * __bfloat162float(weight[lane * E + j]);
        b[j] *= rstd * __bfloat162float(weight[D / 2 + lane * E + j]);
      }
    }
    const long long at = static_cast<long long>(pos) * (D / 2) + lane * E;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const float c = p.cos_t[at + j], s = p.sin_t[at + j], x = a[j] * c - b[j] * s;
      b[j] = b[j] * c + a[j] * s;
      a[j] = x;
    }
  }
  if (is_q) {
    __nv_bfloat16* dst = p.q_out + (static_cast<long long>(t) * p.Hq + h) * D;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      dst[lane * E + j] = __float2bfloat16(a[j]);
      dst[D / 2 + lane * E + j] = __float2bfloat16(b[j]);
    }
    return;
  }
  float most = 0.f;
#pragma unroll
  for (int j = 0; j < E; ++j) {
    a[j] = __bfloat162float(__float2bfloat16(a[j]));
    b[j] = __bfloat162float(__float2bfloat16(b[j]));
    most = fmaxf(most, fmaxf(fabsf(a[j]), fabsf(b[j])));
  }
  most = warp_max(most);
  if (slot < 0) return;
  if (slot >= p.slots_end) {
    if (p.status) atomicCAS(p.status, 0, kBadTable);
    return;
  }
  const int e = kv8_exponent(most), token = slot % kKv8Page;
  const float f = exp2_int(-e);
  uint8_t* block = p.data + (static_cast<long long>(slot / kKv8Page) * p.H + (h - p.Hq - (is_v ? p.H : 0))) * Kv8<D>::kBlock;
  uint8_t* row = block + is_v * Kv8<D>::kHalf + token * D;
  if constexpr (E == 2) {
    *reinterpret_cast<uint16_t*>(row + lane * 2) = e4m3_pair(a[0] * f, a[1] * f);
    *reinterpret_cast<uint16_t*>(row + D / 2 + lane * 2) = e4m3_pair(b[0] * f, b[1] * f);
  } else {
    const uint16_t c = e4m3_pair(a[0] * f, b[0] * f);
    row[lane] = static_cast<uint8_t>(c);
    row[D / 2 + lane] = static_cast<uint8_t>(c >> 8);
  }
  if (lane == 0) block[2 * Kv8<D>::kHalf + kv8_exponent_at(token, is_v)] = static_cast<uint8_t>(e + 127);
}

// kernel<AT> for the AT that fits
template <int D, typename K4, typename K1, typename... Args>
static int launch_rows(K4 four, K1 one, const Kv8Rows& p, cudaStream_t s, Args... args) {
  const int per_token = (2 * p.H + RowsWalk<D, 1>::kRows - 1) / RowsWalk<D, 1>::kRows;
  const bool few = static_cast<long long>(p.T) * per_token <= sm_count() * 32ll;
  const long long warps = (static_cast<long long>(p.T) + 3) / (few ? 1 : 4) * per_token;
  if (warps >= 1ll << 31) return kBadArgument;
  const dim3 grid(static_cast<unsigned>((warps + 7) / 8));
  return static_cast<int>(few ? launch_kernel(one, grid, dim3(256), 0, s, p, per_token, args...)
                              : launch_kernel(four, grid, dim3(256), 0, s, p, per_token, args...));
}

}  // namespace apb

extern "C" {
using namespace apb;

// k, v: [T, H, D] of bf16 (dtype 0) or fp32 (1), strides of tokens and heads in elements, rows on 16-byte boundaries; slots [T];
// data [pages, H, 32 D + 32].
int apb_kv8_write(const void* k, long long ldk, long long lhk, const void* v, long long ldv, long long lhv, const int* slots, void* data,
                  int T, int H, int D, int pages, int dtype, cudaStream_t s) {
  if (T <= 0) return 0;
  const int unit = dtype == 0 ? 8 : 4;
  if ((D != 64 && D != 128) || H < 1 || pages < 0 || pages > (1 << 27) || (dtype != 0 && dtype != 1) || ldk % unit || lhk % unit ||
      ldv % unit || lhv % unit || reinterpret_cast<uintptr_t>(k) % 16 || reinterpret_cast<uintptr_t>(v) % 16 ||
      reinterpret_cast<uintptr_t>(data) % 16)
    return kBadArgument;
  Kv8Rows p = {k, v, ldk, lhk, ldv, lhv, slots, static_cast<uint8_t*>(data), T, H, pages * kKv8Page, status_device_ptr()};
  using bf16 = __nv_bfloat16;
  if (dtype == 0)
    return D == 128 ? launch_rows<128>(kv8_write_kernel<bf16, 128, 4>, kv8_write_kernel<bf16, 128, 1>, p, s)
                    : launch_rows<64>(kv8_write_kernel<bf16, 64, 4>, kv8_write_kernel<bf16, 64, 1>, p, s);
  return D == 128 ? launch_rows<128>(kv8_write_kernel<float, 128, 4>, kv8_write_kernel<float, 128, 1>, p, s)
                  : launch_rows<64>(kv8_write_kernel<float, 64, 4>, kv8_write_kernel<float, 64, 1>, p, s);
}

// out_k, out_v: [T, H, D] of bf16 (dtype 0) or fp32 (1); zeros where slots[t] is below 0.
int apb_kv8_read(const void* data, const int* slots, void* out_k, void* out_v, int T, int H, int D, int pages, int dtype, cudaStream_t s) {
  if (T <= 0) return 0;
  if ((D != 64 && D != 128) || H < 1 || pages < 0 || pages > (1 << 27) || (dtype != 0 && dtype != 1) ||
      reinterpret_cast<uintptr_t>(data) % 16 || reinterpret_cast<uintptr_t>(out_k) % 16 || reinterpret_cast<uintptr_t>(out_v) % 16)
    return kBadArgument;
  Kv8Rows p = {};
  p.slots = slots;
  p.data = static_cast<uint8_t*>(const_cast<void*>(data));
  p.T = T;
  p.H = H;
  p.slots_end = pages * kKv8Page;
  p.status = status_device_ptr();
  if (dtype == 0) {
    using bf16 = __nv_bfloat16;
    auto *ok = static_cast<bf16*>(out_k), *ov = static_cast<bf16*>(out_v);
    return D == 128 ? launch_rows<128>(kv8_read_kernel<bf16, 128, 4>, kv8_read_kernel<bf16, 128, 1>, p, s, ok, ov)
                    : launch_rows<64>(kv8_read_kernel<bf16, 64, 4>, kv8_read_kernel<bf16, 64, 1>, p, s, ok, ov);
  }
  auto *ok = static_cast<float*>(out_k), *ov = static_cast<float*>(out_v);
  return D == 128 ? launch_rows<128>(kv8_read_kernel<float, 128, 4>, kv8_read_kernel<float, 128, 1>, p, s, ok, ov)
                  : launch_rows<64>(kv8_read_kernel<float, 64, 4>, kv8_read_kernel<float, 64, 1>, p, s, ok, ov);
}

// acc [B, (Hq + 2 H) D] fp32, left as zeros; wq, wk [D] bf16 or null; cos, sin [positions, D / 2]; q_out [B, Hq, D] bf16.
int apb_kv8_qkv_post(float* acc, long long ld_acc, const void* wq, const void* wk, const float* cos_t, const float* sin_t, const int* pos,
                     const int* slots, void* q_out, void* data, int B, int Hq, int H, int D, int pages, int positions, float eps,
                     cudaStream_t s) {
  if (B <= 0) return 0;
  if ((D != 64 && D != 128) || H < 1 || Hq < 1 || positions < 0 || pages < 0 || pages > (1 << 27) || reinterpret_cast<uintptr_t>(data) % 16)
    return kBadArgument;
  const Kv8QkvPost p = {acc, ld_acc, static_cast<const __nv_bfloat16*>(wq), static_cast<const __nv_bfloat16*>(wk), cos_t, sin_t, pos, slots,
                        static_cast<__nv_bfloat16*>(q_out), static_cast<uint8_t*>(data), B, Hq, H, pages * kKv8Page, positions, eps,
                        status_device_ptr()};
  const dim3 grid(static_cast<unsigned>((static_cast<long long>(B) * (Hq + 2 * H) + 7) / 8));
  return static_cast<int>(D == 128 ? launch_kernel(kv8_qkv_post_kernel<128>, grid, dim3(256), 0, s, p)
                                   : launch_kernel(kv8_qkv_post_kernel<64>, grid, dim3(256), 0, s, p));
}
}
