// Attention over the 8-bit cache (layout: kv_fp8.cuh): one warp walk per query row and head.
#include <cuda_fp16.h>

#include "host_utils.cuh"
#include "kv_fp8.cuh"

namespace apb {

struct Kv8Attn {
  const __nv_bfloat16* q;    // [rows, Hq, D], rows ldq elements apart
  long long ldq;
  const uint8_t* data;       // [pages, Hkv, block]
  const int* table;          // [entries, ...], rows ld_table apart
  long long ld_table;
  int max_pages, pages;
  const int* lengths;        // [entries] tokens of the cache
  const int* row_entry;      // [rows] or null: row i belongs to entry i and sees all of its tokens
  const int* row_last;       // [rows] last position that a row sees
  __nv_bfloat16* out;
  long long ldo;
  int rows, Hq, Hkv;
  float scale_log2;
  int* status;
};

// A CTA has one query row and head, each of its 4 warps every fourth token; a lane has D / 32 neighbouring dimensions.
template <int D>
__global__ void __launch_bounds__(128) kv8_rows_attention_kernel(const Kv8Attn p) {
  pdl_entry();
  constexpr int N = D / 32;
  const int row = blockIdx.x / p.Hq, head = blockIdx.x % p.Hq, kvh = head / (p.Hq / p.Hkv);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int entry = p.row_entry ? p.row_entry[row] : row;
  int len = p.lengths[entry];
  if (p.row_last) len = min(len, p.row_last[row] + 1);
  if (len > p.max_pages * kKv8Page) {
    if (p.status) atomicCAS(p.status, 0, kBadTable);
    len = p.max_pages * kKv8Page;
  }
  float q[N], o[N] = {}, m = -INFINITY, l = 0.f;
  for (int i = 0; i < N; ++i) q[i] = __bfloat162float(p.q[row * p.ldq + head * D + lane * N + i]) * p.scale_log2;
  auto get = [&](const uint8_t* codes, float f, float (&x)[N]) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const uint32_t y = e4m3_to_f16x2(*reinterpret_cast<const uint16_t*>(codes + lane * N + i));
      const float2 z = __half22float2(*reinterpret_cast<const __half2*>(&y));
      x[i] = z.x * f;
      x[i + 1] = z.y * f;
    }
  };
  for (int t = warp; t < len; t += 4) {
    const int page = p.table[entry * p.ld_table + t / kKv8Page], token = t % kKv8Page;
    if (static_cast<unsigned>(page) >= static_cast<unsigned>(p.pages)) {
      if (p.status) atomicCAS(p.status, 0, kBadTable);
      continue;
    }
    const uint8_t* block = p.data + (static_cast<long long>(page) * p.Hkv + kvh) * Kv8<D>::kBlock;
    float x[N], s = 0.f;
    get(block + token * D, exp2f(block[2 * Kv8<D>::kHalf + kv8_exponent_at(token, 0)] - 127.f), x);
#pragma unroll
    for (int i = 0; i < N; ++i) s += q[i] * x[i];
    s = warp_sum(s);
    const float m_new = fmaxf(m, s), use = m_new == -INFINITY ? 0.f : m_new, alpha = exp2f(m - use), w = exp2f(s - use);
    get(block + Kv8<D>::kHalf + token * D, exp2f(block[2 * Kv8<D>::kHalf + kv8_exponent_at(token, 1)] - 127.f), x);
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = o[i] * alpha + w * x[i];
    l = l * alpha + w;
    m = m_new;
  }
  __shared__ float sm[4], sl[4], so[4][D];
  if (lane == 0) sm[warp] = m, sl[warp] = l;
  for (int i = 0; i < N; ++i) so[warp][lane * N + i] = o[i];
  __syncthreads();
  const float most = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  float total = 0.f, f[4];
  for (int w = 0; w < 4; ++w) {
    f[w] = sm[w] == -INFINITY ? 0.f : exp2f(sm[w] - most);
    total += sl[w] * f[w];
  }
  for (int d = threadIdx.x; d < D; d += 128) {
    float v = 0.f;
    for (int w = 0; w < 4; ++w) v += f[w] == 0.f ? 0.f : so[w][d] * f[w];
    p.out[row * p.ldo + head * D + d] = __float2bfloat16(total != 0.f ? v / total : 0.f);
  }
}

}  // namespace apb

extern "C" {
using namespace apb;

int apb_kv8_rows_attention(const void* q, long long ldq, const void* data, const int* table, long long ld_table, int max_pages, int pages,
                           const int* lengths, const int* row_entry, const int* row_last, void* out, long long ldo, int rows, int Hq,
                           int Hkv, int D, float scale, cudaStream_t s) {
  if (rows <= 0) return 0;
  if ((D != 64 && D != 128) || Hkv < 1 || Hq % Hkv || pages < 0) return kBadArgument;
  const Kv8Attn p = {static_cast<const __nv_bfloat16*>(q), ldq, static_cast<const uint8_t*>(data), table, ld_table, max_pages, pages,
                     lengths, row_entry, row_last, static_cast<__nv_bfloat16*>(out), ldo, rows, Hq, Hkv, scale * 1.4426950408889634f,
                     status_device_ptr()};
  const dim3 grid(static_cast<unsigned>(rows) * Hq);
  return static_cast<int>(D == 128 ? launch_kernel(kv8_rows_attention_kernel<128>, grid, dim3(128), 0, s, p)
                                   : launch_kernel(kv8_rows_attention_kernel<64>, grid, dim3(128), 0, s, p));
}
}
