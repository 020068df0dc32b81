// Rows of keys and values into the 8-bit cache and back (layout: kv_fp8.cuh).
//
// Both are bound by memory: a row of D values moves 2 D (4 D from fp32) + D + 1 bytes on its way in, D + 1 + 2 D on its way out.
// D / 8 lanes share a row, eight neighbouring values each, so that 16-byte accesses to the values and 8-byte ones to the codes cover
// whole sectors; the largest magnitude of a row is found by shuffles among them, and nothing is read twice.  (Lanes that walked over
// rows one at a time kept too little on its way, and a 64-bit division per row: 2.9 TB/s in, 4.1 out.)
#include <cuda_fp16.h>

#include "host_utils.cuh"
#include "kv_fp8.cuh"

namespace apb {

struct Kv8Rows {
  const void* x[2];        // keys and values: [T, H, D] with the given strides in elements
  long long ld[2], lh[2];
  const int* slots;        // page * 16 + token in the page; below 0: none
  uint8_t* data;           // [pages, H, block]
  int T, H;
  int slots_end;           // pages * 16
  int* status;
};

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]);
template <>
__device__ __forceinline__ void load8<__nv_bfloat16>(const __nv_bfloat16* p, float (&v)[8]) {
  const uint4 r = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
template <>
__device__ __forceinline__ void load8<float>(const float* p, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float4 r = reinterpret_cast<const float4*>(p)[i];
    v[4 * i] = r.x, v[4 * i + 1] = r.y, v[4 * i + 2] = r.z, v[4 * i + 3] = r.w;
  }
}
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

// A warp has kAtOnce runs of rows of one token, 32 / kLanes rows each: all of their loads are on their way before the first is used.
constexpr int kAtOnce = 4;
template <int D>
struct RowsWalk {
  static constexpr int kLanes = D / 8, kRows = 32 / kLanes, kPerWarp = kRows * kAtOnce;
  int t, row0, part;        // token, first row of this lane's of its 2 H, eight values of it
  __device__ __forceinline__ bool start(const Kv8Rows& p, int warps_per_token) {
    const int w = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    t = w / warps_per_token;
    row0 = (w - t * warps_per_token) * kPerWarp + lane / kLanes;
    part = lane % kLanes;
    return t < p.T;
  }
};

template <typename T, int D>
__global__ void __launch_bounds__(256) kv8_write_kernel(const Kv8Rows p, int warps_per_token) {
  pdl_entry();
  using Walk = RowsWalk<D>;
  Walk at;
  if (!at.start(p, warps_per_token)) return;
  const int slot = p.slots[at.t];
  float v[kAtOnce][8];
#pragma unroll
  for (int i = 0; i < kAtOnce; ++i) {
    const int row = min(at.row0 + i * Walk::kRows, 2 * p.H - 1), which = row >= p.H, h = row - which * p.H;      // all lanes stay for the shuffles
    load8(static_cast<const T*>(p.x[which]) + at.t * p.ld[which] + h * p.lh[which] + at.part * 8, v[i]);
  }
  if (slot < 0) return;
  if (slot >= p.slots_end) {
    if (p.status) atomicCAS(p.status, 0, kBadTable);
    return;
  }
  const int token = slot % kKv8Page;
  uint8_t* page = p.data + static_cast<long long>(slot / kKv8Page) * p.H * Kv8<D>::kBlock;
#pragma unroll
  for (int i = 0; i < kAtOnce; ++i) {
    const int row = at.row0 + i * Walk::kRows, which = row >= p.H, h = row - which * p.H;
    float most = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) most = fmaxf(most, fabsf(v[i][k]));
#pragma unroll
    for (int o = 1; o < Walk::kLanes; o <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    if (row >= 2 * p.H) continue;
    const int e = kv8_exponent(most);
    const float f = exp2_int(-e);
    uint16_t c[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) c[k] = e4m3_pair(v[i][2 * k] * f, v[i][2 * k + 1] * f);
    uint8_t* block = page + h * Kv8<D>::kBlock;
    *reinterpret_cast<uint2*>(block + which * Kv8<D>::kHalf + token * D + at.part * 8) =
        make_uint2(c[0] | static_cast<uint32_t>(c[1]) << 16, c[2] | static_cast<uint32_t>(c[3]) << 16);
    if (at.part == 0) block[2 * Kv8<D>::kHalf + kv8_exponent_at(token, which)] = static_cast<uint8_t>(e + 127);
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(256) kv8_read_kernel(const Kv8Rows p, int warps_per_token, T* out_k, T* out_v) {
  pdl_entry();
  using Walk = RowsWalk<D>;
  Walk at;
  if (!at.start(p, warps_per_token)) return;
  int slot = p.slots[at.t];
  if (slot >= p.slots_end) {
    if (p.status) atomicCAS(p.status, 0, kBadTable);
    slot = -1;
  }
  const int token = slot % kKv8Page;
  const uint8_t* page = p.data + static_cast<long long>(slot / kKv8Page) * p.H * Kv8<D>::kBlock;
  uint2 c[kAtOnce];
  int e[kAtOnce];
#pragma unroll
  for (int i = 0; i < kAtOnce; ++i) {
    const int row = at.row0 + i * Walk::kRows, which = row >= p.H, h = row - which * p.H;
    const uint8_t* block = page + h * Kv8<D>::kBlock;
    c[i] = make_uint2(0, 0);
    e[i] = 0;
    if (row < 2 * p.H && slot >= 0) {
      c[i] = *reinterpret_cast<const uint2*>(block + which * Kv8<D>::kHalf + token * D + at.part * 8);
      e[i] = block[2 * Kv8<D>::kHalf + kv8_exponent_at(token, which)];
    }
  }
#pragma unroll
  for (int i = 0; i < kAtOnce; ++i) {
    const int row = at.row0 + i * Walk::kRows, which = row >= p.H, h = row - which * p.H;
    if (row >= 2 * p.H) break;
    const float f = exp2f(static_cast<float>(e[i]) - 127.f);
    const uint16_t pair[4] = {static_cast<uint16_t>(c[i].x), static_cast<uint16_t>(c[i].x >> 16), static_cast<uint16_t>(c[i].y),
                              static_cast<uint16_t>(c[i].y >> 16)};
    float v[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t x = e4m3_to_f16x2(pair[k]);
      const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&x));
      v[2 * k] = y.x * f;
      v[2 * k + 1] = y.y * f;
    }
    store8((which ? out_v : out_k) + (static_cast<long long>(at.t) * p.H + h) * D + at.part * 8, v);
  }
}

template <int D, typename K, typename... Args>
static int launch_rows(K kernel, const Kv8Rows& p, cudaStream_t s, Args... args) {
  const int per_token = (2 * p.H + RowsWalk<D>::kPerWarp - 1) / RowsWalk<D>::kPerWarp;
  const long long blocks = (static_cast<long long>(p.T) * per_token + 7) / 8;
  if (blocks * 8 >= 1ll << 31) return kBadArgument;
  return static_cast<int>(launch_kernel(kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, s, p, per_token, args...));
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
  Kv8Rows p = {{k, v}, {ldk, ldv}, {lhk, lhv}, slots, static_cast<uint8_t*>(data), T, H, pages * kKv8Page, status_device_ptr()};
  if (dtype == 0) return D == 128 ? launch_rows<128>(kv8_write_kernel<__nv_bfloat16, 128>, p, s) : launch_rows<64>(kv8_write_kernel<__nv_bfloat16, 64>, p, s);
  return D == 128 ? launch_rows<128>(kv8_write_kernel<float, 128>, p, s) : launch_rows<64>(kv8_write_kernel<float, 64>, p, s);
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
    auto *ok = static_cast<__nv_bfloat16*>(out_k), *ov = static_cast<__nv_bfloat16*>(out_v);
    return D == 128 ? launch_rows<128>(kv8_read_kernel<__nv_bfloat16, 128>, p, s, ok, ov) : launch_rows<64>(kv8_read_kernel<__nv_bfloat16, 64>, p, s, ok, ov);
  }
  auto *ok = static_cast<float*>(out_k), *ov = static_cast<float*>(out_v);
  return D == 128 ? launch_rows<128>(kv8_read_kernel<float, 128>, p, s, ok, ov) : launch_rows<64>(kv8_read_kernel<float, 64>, p, s, ok, ov);
}
}
