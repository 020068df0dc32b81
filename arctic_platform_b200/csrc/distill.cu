// Distillation from a teacher's most likely tokens through the lm head, around the two vocabulary products of the log-prob head.
//
// A row names K tokens with the teacher's log-probabilities lq, and may give the log of the mass of all other tokens, lqr.  With the
// student's p = softmax(z), z = hidden @ weight^T * scale, and its mass pr of the tokens not named, over the K (+ 1) classes
//   F = sum q (lq - lp) (+ qr (lqr - lpr)),   R = sum p (lp - lq) (+ pr (lpr - lqr)),   value = (1 - mix) F + mix R.
// With Q = sum q (+ qr) and E = sum p (lp - lq + 1) (+ pr (lpr - lqr + 1)):
//   d value / d z_v = (1 - mix) (p_v Q - q_v) + mix p_v (lp_v - lq_v + 1 - E)     for a named token,
//                   = p_v c,  c = (1 - mix) (Q - qr / pr) + mix (lpr - lqr + 1 - E)  for any other (without the class of the others
//                                                                                  qr / pr = 0 and lpr - lqr + 1 = 0).
// So the rows' gradient is dense only as a multiple of p, which is what the log-prob head's backward epilogue writes; the K named places
// (and the label's) are put over it afterwards.  Where pr is so small that p_v leaves fp32's range it is a multiple of p_v / pr instead, a softmax
// of the others alone.
//
//   named    one CTA per row: the row's names in rising order for the product's epilogue; logits of the named tokens and the label as
//            dot products.  An entry below 0 or beyond the vocabulary names nothing, a token named again counts once, by
//            its first entry.
//   product  CTA pairs (gemm_tcgen05_2cta.cu), records of every 128 columns without the named ones and, where there is room, their exponentials
//   combine  one warp per row: statistics, value, log-prob and entropy of the label's distribution, c and the named places' gradients, in 64 bits
//   rows     the coefficient of p in the backward pass; spread  the kept exponentials times it (or the product again); places  the named places
//            and the label's over that
//
// Why the named logits are dot products of their own instead of columns taken out of the product's tiles: the named tokens carry nearly all of
// the mass and of the gradient, and a tensor core's running sum of all H terms is less exact than 64-bit sums of eight products each.
// It costs a read of K rows of the weight for every row (4096 rows with 64 names, H = 2560: 0.23 ms of 8.3).
//
// d(logits) is rounded to bf16, the type in which the tensor cores take it with a bf16 weight: an entry is off by 2^-8 of itself at most, and a
// gradient in norm by 2.3 to 2.5e-3 where its own rounding to bf16 makes 1.7e-3.  That is one more rounding of the named entries, which hold
// nearly all of it; that of the kept exponentials does not show in three digits.  A second product for what the rounding leaves would take another
// 4.4 of 8.3 ms.
//
// Time of a whole pass and its gradients at 4096 x 151936 x 2560: 8.3 ms, of which the product 2.17 (with the exponentials kept), spread 0.42,
// d_hidden 2.12 and d_weight 2.25 (cuBLAS's sustained rate gives 2.25 for each); 10.0 with the logits formed again.  At H = 1024, 549 rows
// 0.79 ms (0.93).
#include "common.cuh"
#include "gemm_common.cuh"
#include "host_utils.cuh"

namespace apb {

constexpr int kMostNamed = 256;
constexpr int kNoName = 0x7fffffff;

__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float dot8(const uint4& a, const uint4& b, float s) {
  const uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&x[i]));
    const float2 g = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&y[i]));
    s = fmaf(f.x, g.x, s);
    s = fmaf(f.y, g.y, s);
  }
  return s;
}

// names [N, K] as given; sorted [N, K] and where every 128 columns of the vocabulary have theirs in it (the product's named_at); logit [N, K + 1]:
// of every entry (-inf where it names nothing), then of the label.
__global__ void __launch_bounds__(256)
distill_named_kernel(const __nv_bfloat16* __restrict__ hidden, long long ldh, const __nv_bfloat16* __restrict__ weight, long long ldw,
                     const int* __restrict__ names, const int* __restrict__ labels, const float* __restrict__ row_scale, float scale, int K,
                     int V, int H, int* __restrict__ sorted, uint16_t* __restrict__ named_at, double* __restrict__ logit) {
  __shared__ int name[kMostNamed];
  __shared__ int kept[kMostNamed];
  const long long row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid < K) {
    const int id = names[row * K + tid];
    name[tid] = id >= 0 && id < V ? id : kNoName;
  }
  __syncthreads();
  if (tid < K) {
    int id = name[tid];
    for (int j = 0; j < tid; ++j)
      if (name[j] == id) id = kNoName;
    kept[tid] = id;
  }
  __syncthreads();
  if (tid < K) {
    const int id = kept[tid];
    int rank = 0;
    for (int j = 0; j < K; ++j) rank += kept[j] < id || (kept[j] == id && j < tid);
    sorted[row * K + rank] = id;
    name[rank] = id;
  }
  __syncthreads();
  const int tiles = K > 0 ? (V + 127) / 128 : 0;
  for (int t = tid; t < tiles; t += 256) {
    int lo = 0, hi = K;                  // first entry of this tile or behind it
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (name[mid] < t * 128) lo = mid + 1;
      else hi = mid;
    }
    while (hi < K && name[hi] < V && name[hi] >> 7 == t) ++hi;
    named_at[row * tiles + t] = static_cast<uint16_t>(hi > lo ? lo | (hi - lo) << 8 : 0);     // K <= 256, at most 128 in a tile
  }
  const float rs = scale * (row_scale ? row_scale[row] : 1.f);
  const uint4* h = reinterpret_cast<const uint4*>(hidden + row * ldh);
  const int chunks = H / 8;
  for (int k = warp; k <= K; k += 8) {
    const int id = k < K ? kept[k] : labels[row];
    double s = 0.0;                        // products of two bf16 numbers are exact in fp32, eight of them add up there
    const bool there = id >= 0 && id < V;
    if (there) {
      const uint4* w = reinterpret_cast<const uint4*>(weight + static_cast<long long>(id) * ldw);
      for (int c = lane; c < chunks; c += 32) s += static_cast<double>(dot8(h[c], w[c], 0.f));
      s = warp_sum_f64(s);
    }
    if (lane == 0) logit[row * (K + 1) + k] = there ? s * static_cast<double>(rs) : -INFINITY;
  }
}

struct DistillRows {
  const float4* partial;     // [N][tiles] records of the columns not named
  const double* logit;       // [N, K + 1]
  const float* teacher;      // [N, K] log-probabilities
  const float* rest;         // [N] log of the others' mass, or null
  float* value;              // [N]
  float* lp;
  float* ent;
  double* lse;
  float* ref;                // d value / d z_v of a token not named is others exp(z_v - ref); lse in fp32, or that of the others alone
  float* others;
  float* named_grad;         // [N, K] d value / d z of the named ones
  int tiles, K, N;
  float mix;
};

// Logits of the named tokens, the log-sum-exp and the terms of the value and of its gradient are 64-bit numbers here.  A divergence is a small
// difference of log-probabilities, themselves differences of numbers around 16, and in fp32 was off by up to 1e-5 of itself where rows are
// few.  The terms of a gradient cancel where a student is sure or near its teacher: in fp32 they left 1e-7 times the upstream gradient.
// x * y, 0 where x is: a class without mass adds nothing, whatever its logarithm is
__device__ __forceinline__ float mass_times(float x, float y) { return x > 0.f ? x * y : 0.f; }
__device__ __forceinline__ double mass_times(double x, double y) { return x > 0.0 ? x * y : 0.0; }

// Where the log of the others' mass is below this their probabilities come near the end of fp32's range (2^-126, 87 below the largest), but not the
// gradient that the teacher's mass of them asks for: it is formed from their shares of their own sum.
constexpr double kLeastRest = -69.0;

constexpr int kRecords = 8;      // of a lane in flight (549 rows of 1187 records: 8 us, 27 with one)

__global__ void __launch_bounds__(256) distill_combine_kernel(const DistillRows a) {
  const int row = (blockIdx.x * blockDim.x + threadIdx.x) >> 5, lane = threadIdx.x & 31;
  if (row >= a.N) return;
  const float4* pr = a.partial + static_cast<long long>(row) * a.tiles;
  const double* zk = a.logit + static_cast<long long>(row) * (a.K + 1);
  const float* lq = a.teacher + static_cast<long long>(row) * a.K;
  float m = -INFINITY, s = 0.f, e = 0.f;                // of the tokens not named
  for (int t0 = lane; t0 < a.tiles; t0 += 32 * kRecords) {
    float4 v[kRecords];
    float mn = m;
#pragma unroll
    for (int i = 0; i < kRecords; ++i) {
      v[i] = t0 + 32 * i < a.tiles ? pr[t0 + 32 * i] : make_float4(-INFINITY, 0.f, 0.f, 0.f);
      mn = fmaxf(mn, v[i].x);
    }
    const float c0 = m == -INFINITY ? 0.f : __expf(m - mn);
    s *= c0;
    e *= c0;
#pragma unroll
    for (int i = 0; i < kRecords; ++i) {
      const float c = v[i].x == -INFINITY ? 0.f : __expf(v[i].x - mn);
      s = fmaf(v[i].y, c, s);
      e = fmaf(v[i].z, c, e);
    }
    m = mn;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o), e2 = __shfl_xor_sync(0xffffffffu, e, o);
    const float mn = fmaxf(m, m2);
    const float c0 = m == -INFINITY ? 0.f : __expf(m - mn), c1 = m2 == -INFINITY ? 0.f : __expf(m2 - mn);
    s = s * c0 + s2 * c1;
    e = e * c0 + e2 * c1;
    m = mn;
  }
  float top = m;
  for (int k = lane; k < a.K; k += 32) top = fmaxf(top, static_cast<float>(zk[k]));
  top = warp_max(top);
  double st = 0.0, et = 0.0;
  for (int k = lane; k < a.K; k += 32) {
    const double z = zk[k];
    if (z == -INFINITY) continue;
    const double x = exp(z - top);
    st += x;
    et += x * z;
  }
  st = warp_sum_f64(st);
  et = warp_sum_f64(et);
  const double shift = m == -INFINITY ? 0.0 : exp(static_cast<double>(m) - top);
  const double sum = st + s * shift;
  const double lse = top + log(sum);
  const float ent = static_cast<float>(lse - (et + e * shift) / sum);
  // classes
  const bool bucket = a.rest != nullptr;
  const double mix = a.mix, one_way = 1.0 - mix;
  const double rest_lp = s > 0.f ? m + log(static_cast<double>(s)) - lse : -INFINITY, rest_p = exp(rest_lp);
  const double lqr = bucket ? a.rest[row] : -INFINITY, qr = exp(lqr);
  double F = 0.0, R = 0.0, Q = 0.0, E = 0.0;
  for (int k = lane; k < a.K; k += 32) {
    const double z = zk[k];
    if (z == -INFINITY) continue;
    const double lp = z - lse, l = lq[k], q = exp(l);
    F += mass_times(q, l - lp);
    Q += q;
    if (a.mix != 0.f) {
      const double p = exp(lp);
      R += mass_times(p, lp - l);
      E += mass_times(p, lp - l + 1.0);
    }
  }
  F = warp_sum_f64(F);
  Q = warp_sum_f64(Q);
  R = warp_sum_f64(R);
  E = warp_sum_f64(E);
  const bool far = bucket && s > 0.f && rest_lp < kLeastRest;
  double c = 0.0;
  if (bucket) {
    F += mass_times(qr, lqr - rest_lp);
    Q += qr;
    if (!far && s > 0.f) c = -one_way * (qr / rest_p);
    if (a.mix != 0.f) {
      R += mass_times(rest_p, rest_lp - lqr);
      E += mass_times(rest_p, rest_lp - lqr + 1.0);
      if (rest_p > 0.0) c += mix * (rest_lp - lqr + 1.0);
    }
  }
  c += one_way * Q;
  if (a.mix != 0.f) c -= mix * E;
  if (far) c = mass_times(rest_p, c) - one_way * qr;           // c pr, without the quotient
  for (int k = lane; k < a.K; k += 32) {
    const double z = zk[k];
    double g = 0.0;
    if (z != -INFINITY) {
      const double lp = z - lse, p = exp(lp), l = lq[k];
      g = one_way * (p * Q - exp(l));
      if (a.mix != 0.f) g += mix * mass_times(p, lp - l + 1.0 - E);
    }
    a.named_grad[static_cast<long long>(row) * a.K + k] = static_cast<float>(g);
  }
  if (lane == 0) {
    a.value[row] = static_cast<float>(a.mix == 0.f ? F : one_way * F + mix * R);
    a.lp[row] = static_cast<float>(zk[a.K] - lse);
    a.ent[row] = ent;
    a.lse[row] = lse;
    a.ref[row] = static_cast<float>(far ? lse + rest_lp : lse);
    a.others[row] = static_cast<float>(c);
  }
}

// The upstream gradient of a log-prob that would give every token not named what it gets: minus the coefficient of exp(z - ref).  Where ref is not
// the log-sum-exp, the others' probabilities add up to less than e^-69, and the entropy's gradient of them, below 100 times that, is left out.
__global__ void __launch_bounds__(256)
distill_rows_kernel(const float* __restrict__ g_value, const float* __restrict__ g_lp, const float* __restrict__ g_ent,
                    const float* __restrict__ others, const double* __restrict__ lse, const float* __restrict__ ref, int N,
                    float* __restrict__ out, int* __restrict__ no_label, float* __restrict__ out_ent) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= N) return;
  const float g = g_value ? g_value[i] : 0.f, gl = g_lp ? g_lp[i] : 0.f, l = static_cast<float>(lse[i]), r = ref[i];
  out[i] = (r == l ? gl : gl * expf(r - l)) - (g == 0.f ? 0.f : g * others[i]);
  no_label[i] = -1;
  if (g_ent) out_ent[i] = r == l ? g_ent[i] : 0.f;
}

// d(logits) of the tokens not named from what the forward product kept of them, exp(z - m) of every 128 columns' largest m in bf16: times
// exp(m - ref) and the row's coefficient.  One CTA per row, 16 bytes a thread; bound by memory (4096 x 151936: 2.5 GB, 0.4 ms, where forming the
// logits again takes 2.1).  The named places hold zeros.  A value is rounded twice, by 2^-8 at most each time; the named tokens, which
// carry nearly all of a row's gradient, and the label are written from fp32 behind this.
__global__ void __launch_bounds__(256)
distill_spread_kernel(const uint4* __restrict__ kept, const float4* __restrict__ partial, const float* __restrict__ glp,
                      const float* __restrict__ ref, const float* __restrict__ row_scale, float scale, int V, uint4* __restrict__ d) {
  const long long row = blockIdx.x;
  const int units = V / 8, tiles = (V + 127) / 128;
  const float c = -glp[row] * scale * (row_scale ? row_scale[row] : 1.f), l = ref[row];
#pragma unroll 4
  for (int u = threadIdx.x; u < units; u += 256) {
    const uint4 x = __ldcs(kept + row * units + u);
    const float m = partial[row * tiles + u / 16].x, f = m == -INFINITY ? 0.f : c * __expf(m - l);
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]));
      o[i] = pack_bf16x2(v.x * f, v.y * f);
    }
    d[row * units + u] = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

__global__ void __launch_bounds__(256) distill_round_kernel(const float4* __restrict__ x, uint2* __restrict__ y, long long n) {
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
    const float4 v = x[i];
    y[i] = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
  }
}

// One warp per row: the places of the named tokens, and the label's, in d(logits) [N, V] bf16.  Log-probabilities come from the 64-bit
// log-sum-exp, and the label's 1 - p from its own: where a student is sure of a token, 1 - p of an fp32 log-sum-exp around 50 is off by 2e-6.
__global__ void __launch_bounds__(256)
distill_places_kernel(const int* __restrict__ names, const int* __restrict__ labels, const double* __restrict__ logit,
                      const float* __restrict__ named_grad, const float* __restrict__ others, const double* __restrict__ lse,
                      const float* __restrict__ ref, const float* __restrict__ ent, const float* __restrict__ g_value, const float* __restrict__ g_lp,
                      const float* __restrict__ g_ent, const float* __restrict__ row_scale, float scale, int K, int V, int N,
                      __nv_bfloat16* __restrict__ d, long long ldd) {
  const int row = (blockIdx.x * blockDim.x + threadIdx.x) >> 5, lane = threadIdx.x & 31;
  if (row >= N) return;
  const double* zk = logit + static_cast<long long>(row) * (K + 1);
  const int label = labels[row];
  const float rs = scale * (row_scale ? row_scale[row] : 1.f);
  const float gv = g_value ? g_value[row] : 0.f, gl = g_lp ? g_lp[row] : 0.f, ge = g_ent ? g_ent[row] : 0.f, en = ent[row];
  const double l = lse[row];
  __nv_bfloat16* to = d + row * ldd;
  bool label_named = false;
  for (int k = lane; k < K; k += 32) {
    if (zk[k] == -INFINITY) continue;
    const int id = names[static_cast<long long>(row) * K + k];
    const float lp = static_cast<float>(zk[k] - l), p = expf(lp);
    const float g = (gv == 0.f ? 0.f : gv * named_grad[static_cast<long long>(row) * K + k]) - ge * mass_times(p, lp + en);
    if (id == label) label_named = true;
    to[id] = __float2bfloat16_rn((g - gl * (id == label ? expm1f(lp) : p)) * rs);
  }
  label_named = __any_sync(0xffffffffu, label_named);
  if (lane == 0 && !label_named && label >= 0 && label < V) {
    const float lp = static_cast<float>(zk[K] - l), p = expf(lp);
    const float share = expf(static_cast<float>(zk[K] - ref[row]));
    to[label] = __float2bfloat16_rn(((gv == 0.f ? 0.f : gv * others[row] * share) - gl * expm1f(lp) - ge * mass_times(p, lp + en)) * rs);
  }
}

int launch_gemm_pair(const CUtensorMap& ta, const CUtensorMap& tb, const GemmParams& p, cudaStream_t stream);

}  // namespace apb

extern "C" {

int apb_lmhead_dlogits(const void* hidden, const void* weight, const int* labels, const float* row_scale, const float* lse, const float* ent,
                       const float* g_lp, const float* g_ent, void* dlogits, int M, int V, int H, long long ldh, long long ldw, long long ldd,
                       float scale, cudaStream_t stream);
int apb_gemm_bf16(const void* A, const void* B, void* C, int M, int N, int K, long long lda, long long ldb, long long ldc, int a_mn, int b_mn,
                  int epi, int splits, float alpha, const void* bias, void* C2, long long ldc2, const void* tile_map, int num_map_tiles,
                  long long b_rows, int bn, int max_ctas, cudaStream_t stream);

// hidden [N, H] and weight [V, H] bf16 (H, V and the strides multiples of 8, 16-byte aligned), labels [N], names [N, K] int32 (K <= 256),
// teacher [N, K] fp32, rest [N] fp32 or null, row_scale [N] or null (then `scale` alone).  Scratch: sorted [N, K] int32 and
// behind it [N][ceil(V / 128)] uint16, partial [N][ceil(V / 128)][4] fp32.  Kept for the backward pass: logit [N, K + 1] and
// lse [N] fp64, named_grad [N, K], others, ref, ent [N] and, if not null, kept [N, V] bf16 (then partial too).
int apb_lmhead_distill_fwd(const void* hidden, const void* weight, const int* labels, const int* names, const float* teacher,
                           const float* rest, const float* row_scale, float* partial, int* sorted, double* logit, float* value, float* lp,
                           float* ent, double* lse, float* ref, float* others, float* named_grad, void* kept, int N, int V, int H, int K, long long ldh,
                           long long ldw, float scale, float mix, cudaStream_t stream) {
  using namespace apb;
  if (N <= 0) return 0;
  if (!hidden || !weight || !labels || !partial || !value || !lp || !ent || !lse || !ref || !others || !logit || K < 0 || K > kMostNamed ||
      (K > 0 && (!names || !teacher || !sorted || !named_grad)) || V <= 0 || H <= 0 || (H % 8) || (V % 8) || (ldh % 8) || (ldw % 8) ||
      ((reinterpret_cast<uintptr_t>(hidden) | reinterpret_cast<uintptr_t>(weight)) & 15))
    return kBadArgument;
  distill_named_kernel<<<N, 256, 0, stream>>>(static_cast<const __nv_bfloat16*>(hidden), ldh, static_cast<const __nv_bfloat16*>(weight),
                                              ldw, names, labels, row_scale, scale, K, V, H, sorted,
                                              reinterpret_cast<uint16_t*>(sorted + static_cast<long long>(N) * K), logit);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return static_cast<int>(e);
  CUtensorMap ta, tb;
  int rc = make_tmap_2d(&ta, hidden, 2, N, H, ldh, 64, 128);
  if (rc) return 1000 + rc;
  rc = make_tmap_2d(&tb, weight, 2, V, H, ldw, 64, 128);
  if (rc) return 2000 + rc;
  GemmParams p{};
  p.M = N;
  p.N = V;
  p.K = H;
  p.epi = kEpiRestPartial;
  p.C = kept;
  p.ldc = V;
  p.splits = 1;
  p.alpha = scale;
  p.row_scale = row_scale;
  p.partial = partial;
  p.named = sorted;
  p.named_at = reinterpret_cast<const uint16_t*>(sorted + static_cast<long long>(N) * K);
  p.n_named = K;
  p.status = status_device_ptr();
  rc = launch_gemm_pair(ta, tb, p, stream);
  if (rc) return rc;
  DistillRows a{reinterpret_cast<const float4*>(partial), logit, teacher, rest, value, lp, ent, lse, ref, others, named_grad, (V + 127) / 128, K, N,
                mix};
  distill_combine_kernel<<<(N + 7) / 8, 256, 0, stream>>>(a);
  return static_cast<int>(cudaGetLastError());
}

// The backward pass of N rows of a forward pass: d(logits) [N, V] bf16, of it d_hidden [N, H] bf16 and d_weight [V, H] (bf16, or fp32 that is
// added to), either may be null.  d(logits): the coefficients of the probabilities; probability times coefficient, from what the forward
// pass kept or, without it or with g_ent, by the product again; the named tokens' places and the label's.  g_value, g_lp, g_ent [N] fp32:
// upstream gradients (null: none); the others as kept by the forward pass.  Scratch: scratch [3 N] words of 32 bits; total [N, H] fp32 or null:
// then d_hidden's product is cut along the vocabulary.
int apb_lmhead_distill_bwd(const void* hidden, const void* weight, const int* names, const int* labels, const float* row_scale,
                           const double* logit, const float* named_grad, const float* others, const double* lse, const float* ref, const float* ent,
                           const float* g_value, const float* g_lp, const float* g_ent, const void* kept, const float* partial, float* scratch,
                           void* dlogits, void* d_hidden, float* total, void* d_weight, int weight_f32, int N, int V, int H, int K,
                           long long ldh, long long ldw, float scale, cudaStream_t stream) {
  using namespace apb;
  if (N <= 0) return 0;
  if (!hidden || !weight || !labels || !logit || !others || !lse || !ref || !ent || !scratch || !dlogits || K < 0 || K > kMostNamed ||
      (K > 0 && (!names || !named_grad)) || V <= 0 || H <= 0 || (V % 8) || (H % 8) || (kept && !partial))
    return kBadArgument;
  int* no_label = reinterpret_cast<int*>(scratch + N);
  float* ent_rows = scratch + 2ll * N;
  distill_rows_kernel<<<(N + 255) / 256, 256, 0, stream>>>(g_value, g_lp, g_ent, others, lse, ref, N, scratch, no_label, ent_rows);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return static_cast<int>(e);
  int rc = 0;
  if (kept && !g_ent) {
    distill_spread_kernel<<<N, 256, 0, stream>>>(static_cast<const uint4*>(kept), reinterpret_cast<const float4*>(partial), scratch, ref, row_scale,
                                                 scale, V, static_cast<uint4*>(dlogits));
    rc = static_cast<int>(cudaGetLastError());
  } else {
    rc = apb_lmhead_dlogits(hidden, weight, no_label, row_scale, ref, ent, scratch, g_ent ? ent_rows : nullptr, dlogits, N, V, H, ldh, ldw, V, scale, stream);
  }
  if (rc) return rc;
  distill_places_kernel<<<(N + 7) / 8, 256, 0, stream>>>(names, labels, logit, named_grad, others, lse, ref, ent, g_value, g_lp, g_ent, row_scale,
                                                         scale, K, V, N, static_cast<__nv_bfloat16*>(dlogits), V);
  e = cudaGetLastError();
  if (e != cudaSuccess) return static_cast<int>(e);
  if (d_hidden && total) {
    e = cudaMemsetAsync(total, 0, sizeof(float) * N * H, stream);
    if (e != cudaSuccess) return static_cast<int>(e);
    rc = apb_gemm_bf16(dlogits, weight, total, N, H, V, V, ldw, H, 0, 1, kEpiF32Accum, 1, 1.f, nullptr, nullptr, 0, nullptr, 0, 0, 0, 0, stream);
    if (rc) return rc;
    const long long n = static_cast<long long>(N) * H / 4, grid = (n + 255) / 256, cap = 8ll * sm_count();
    distill_round_kernel<<<static_cast<int>(grid < cap ? grid : cap), 256, 0, stream>>>(reinterpret_cast<const float4*>(total),
                                                                                       static_cast<uint2*>(d_hidden), n);
    rc = static_cast<int>(cudaGetLastError());
  } else if (d_hidden) {
    rc = apb_gemm_bf16(dlogits, weight, d_hidden, N, H, V, V, ldw, H, 0, 1, kEpiBf16, 1, 1.f, nullptr, nullptr, 0, nullptr, 0, 0, 0, 0, stream);
  }
  if (rc || !d_weight) return rc;
  return apb_gemm_bf16(dlogits, hidden, d_weight, V, H, N, V, ldh, H, 1, 1, weight_f32 ? kEpiF32Accum : kEpiBf16, 1, 1.f, nullptr, nullptr, 0,
                       nullptr, 0, 0, 0, 0, stream);
}
}
