// Attention of chunks of query tokens over the 8-bit cache (layout: kv_fp8.cuh) on tcgen05 tensor cores.
//
// A tile holds 128 rows: the query heads of one key head for 128 / heads neighbouring tokens, so that short chunks fill it too.  A CTA
// (or a pair of them) walks work items of one or two such tiles over a range of 128-token blocks: S = Q K^T and O += P V by MMAs of 128 x
// 128 per CTA, S and O in tensor memory, P over S, one softmax warpgroup per tile, one thread per row.
//
// Keys and values are bf16 operands here: kind::f16 wants both sides in 16 bits, and queries and weights do not fit 8.  Pages come by
// bulk copies into a staging ring as they lie in the cache; one or two warpgroups turn them into swizzled bf16 tiles.  A code becomes
// a bf16 number by moving its bits (exponents off by 120), two at a time, and one multiplication by a power of two, which also brings
// in its token's exponent relative to a reference: for keys the block's largest exponent (and 16), which the softmax multiplies by, for values
// one that moves only when a block's is larger by 2^8 or more, and O with it.  Nothing is rounded: 2^-120 of the reference is far below
// what counts (tokens more than 2^100 smaller than the largest of their sequence lose bits).
//
// What bounds it.  A block of two tiles is 2050 clocks of MMAs and 2050 of exponentials, of which a warp by itself gets half the rate,
// beside turning codes into tiles (3000 by one warpgroup), and the three wait for one another.  Hence the pair: its MMAs of 256 rows take
// half of the keys and half of the values' columns from either CTA, so that each turns half of the codes.  And weights are taken
// relative to a reference that stays while they fit (the softmax below), in one pass over the scores.  Both together took 512 new tokens
// of a 16896-token conversation (32/8 heads of 128) from 181 to 164 us, 851 TFLOP/s (one CTA per item with this softmax: 179); four prompts
// of up to 4096 tokens from 397 to 357.  (156 and 347 before the pair's tiles were released at the cluster's scope, see the warp that
// does it.)  The chain of a tile is what is left: 2300 clocks of softmax, 260 until the issuing warp knows, 1470 until the next scores.  S in
// halves of 64 columns with buffers of their own was slower (an MMA of 64 columns takes 0.7 of one of 128), and so were two threads per
// row (they have to agree on the reference: 171 us where this form took 148).  Looking for codes that are no numbers costs 10 us.
// Short chunks (5 draft tokens: 28 us where the bytes take 4.8) have one tile of 20 rows, for which all codes are turned into tiles: two
// warpgroups do that there (one: 31), 2000 clocks a block.  Of up to 16 rows most go the way of decode attention instead (apb_kv8_few).
//
// Items over long contexts are cut along the keys where there are too few to fill the GPU (csrc/runtime_kv8.cpp); their parts are
// joined by kv8_chunk_join_kernel.
#include <type_traits>

#include "attention_common.cuh"
#include "host_utils.cuh"
#include "kv_fp8.cuh"

namespace apb {

struct Kv8Item {
  int row0, tokens;        // first query token, tokens of both tiles
  int seq, kvh, head0, heads;
  int pos0, len;           // position of the first token (may be below 0), tokens of the sequence
  int block0, blocks;      // of 128 tokens
  int part;                // where its results go: tile of the scratch, -1: the output
  int pad;
};
struct Kv8Chunk {
  const Kv8Item* items;    // of CTA c: [first[c], first[c + 1])
  const int* first;
  const uint8_t* data;
  const int* table;        // [sequences, ...]
  long long ld_table;
  __nv_bfloat16* out;
  long long ldo;
  float* part_o;           // [tiles][128][D], normalised
  float* part_s;           // [tiles][128][2]: maximum in log2, sum
  int Hkv, hp, tp;         // heads and tokens of a tile
  float scale_log2;        // above 0
  uint32_t key_sign;       // sign bits of a pair of bf16 where the scale is below 0
  int* status;
};

constexpr float kKcRoom = 1.1e12f;          // 2^40: what a row's weights of a block may sum up to
constexpr int kKcBlock = 128;
constexpr int kKcStages = 2, kKcMeta = 4;

// kTwo: a CTA per item of one or two tiles.
// kDual: items of one tile each; the two softmax groups take every second block of it and join what they have at the item's end.
// kPair: two CTAs per item, whose tiles have 256 rows, 128 for each; a CTA makes the half of the keys and the half of the values'
// columns that its partner's tensor core then reads as well.
enum Kv8ChunkForm : int { kTwo, kDual, kPair };

template <int D, int FORM>
struct Kv8ChunkCfg {
  static constexpr int kTile = 128 * D * 2, kKv = FORM == kPair ? kTile / 2 : kTile;            // bytes of a tile of queries, of the ring
  static constexpr int kQ = FORM == kDual ? 1 : 2, kRing = FORM == kTwo ? 3 : FORM == kDual ? 4 : 6;      // tiles
  // Warpgroups: issue, one or two that turn codes into tiles, one of softmax per tile.  Registers move between them; their sum is what
  // the block was launched with.
  static constexpr int kConvert = FORM != kTwo ? 8 : 4, kThreads = 128 + 32 * kConvert + 256;         // warps that turn codes into tiles
  static constexpr int kRegsIssue = FORM != kTwo ? 56 : 80, kRegsConvert = FORM != kTwo ? 72 : 96, kRegsSoftmax = FORM != kTwo ? 136 : 168;
  static_assert(kRegsIssue * 128 + kRegsConvert * 32 * kConvert + kRegsSoftmax * 256 <= (FORM != kTwo ? 96 : 128) * kThreads, "registers");
  static constexpr int kStage = 8 * Kv8<D>::kBlock;
  static constexpr int kSmem = kQ * kTile + kRing * kKv + kKcStages * kStage + 2048 + 384;
  static_assert(kSmem <= 227 * 1024, "shared memory of one CTA");
};

__device__ __forceinline__ void bulk_load(void* smem_dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(smem_dst)), "l"(src),
               "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
// A load whose bytes are counted on a barrier that may live in the partner CTA.
__device__ __forceinline__ void tma_load_3d_pair(void* smem_dst, const CUtensorMap* map, uint32_t bar_cluster_addr, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
          smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar_cluster_addr), "r"(x), "r"(y), "r"(z)
      : "memory");
}
// An arrival at a barrier of either CTA that orders no accesses to shared memory: for what lies in tensor memory, which tcgen05's fences
// order with it.
__device__ __forceinline__ void mbar_arrive_relaxed(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ void umma_bf16_ts_pair(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n\t"
      "}\n" ::"r"(tmem_d),
      "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Arrive on the barrier at this place in both CTAs once every MMA issued so far is done.
__device__ __forceinline__ void tc_commit_both(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
               "h"(static_cast<uint16_t>(3))
               : "memory");
}
// Four codes times 2^-120 as bf16 pairs, times their factor: a byte with its sign eight times in front of it, moved by four bits, has sign,
// exponent and mantissa in their places.
__device__ __forceinline__ void e4m3x4_to_bf16(uint32_t w, uint32_t factor, uint32_t& lo, uint32_t& hi) {
  uint32_t x, y;
  asm("prmt.b32 %0, %1, 0, 0x9180;" : "=r"(x) : "r"(w));
  asm("prmt.b32 %0, %1, 0, 0xB3A2;" : "=r"(y) : "r"(w));
  x = (x * 16u) & 0x87F087F0u;
  y = (y * 16u) & 0x87F087F0u;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(lo) : "r"(x), "r"(factor));
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(hi) : "r"(y), "r"(factor));
}
// Puts no numbers where codes are none.
__device__ __forceinline__ void e4m3x4_nan(uint32_t w, uint32_t& lo, uint32_t& hi) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if ((w >> (8 * i) & 0x7F) == 0x7F) (i < 2 ? lo : hi) |= i & 1 ? 0x7FC00000u : 0x7FC0u;
}

template <int D, int FORM>
__global__ void __launch_bounds__(Kv8ChunkCfg<D, FORM>::kThreads, 1)
    kv8_chunk_kernel(const __grid_constant__ CUtensorMap tma_q, const Kv8Chunk p) {
  using Cfg = Kv8ChunkCfg<D, FORM>;
  constexpr bool DUAL = FORM == kDual, PAIR = FORM == kPair;
  constexpr int kConvert = Cfg::kConvert;
  constexpr int kCtas = PAIR ? 2 : 1;
  // Parts of a block's columns that softmax threads hand over one by one, so that the values' product of one runs beside the softmax of
  // the next.  One for kPair, whose CTAs would have to meet twice as often: 169 us for 146 without the look for numbers.
  constexpr int kHalves = PAIR ? 1 : 2, kCols = kKcBlock / kHalves;
  constexpr int kRing = Cfg::kRing, kChunks = D / 64;
  extern __shared__ __align__(1024) uint8_t kc_smem[];
  uint8_t* smem = kc_smem;
  pdl_entry();
  if (smem_u32(smem) & 1023) {             // the tiles' swizzle goes by the address
    if (threadIdx.x == 0 && p.status) atomicCAS(p.status, 0, kBadArgument);
    return;
  }
  uint8_t* smem_q = smem;
  uint8_t* smem_kv = smem + Cfg::kQ * Cfg::kTile;
  uint8_t* smem_st = smem_kv + kRing * Cfg::kKv;
  uint8_t* smem_x = smem_st + kKcStages * Cfg::kStage;        // [2] 1 KB through which the softmax threads of a group pass numbers of rows
  uint64_t* st_full = reinterpret_cast<uint64_t*>(smem_x + 2048);
  uint64_t* st_empty = st_full + kKcStages;
  uint64_t* kv_full = st_empty + kKcStages;
  uint64_t* kv_empty = kv_full + kRing;
  uint64_t* q_full = kv_empty + kRing;
  uint64_t* q_empty = q_full + 1;
  uint64_t* s_full = q_empty + 1;      // [2]
  uint64_t* p_full = s_full + 2;       // [2][2] of the halves
  uint64_t* o_full = p_full + 4;       // [2][2] after a half's product, but for the last one's only at the end of an item
  uint64_t* meet = o_full + 4;         // [4] kDual: the two warps of 32 rows
  int2* meta = reinterpret_cast<int2*>(meet + 4);             // [kKcMeta] reference exponents of a block's keys and values
  int* other_ev = reinterpret_cast<int*>(meta + kKcMeta);     // [2][4] kDual: what a group's O is in units of, for 32 rows each
  uint64_t* kv_made = reinterpret_cast<uint64_t*>(other_ev + 8);      // kPair: [kRing] this CTA's part of a tile
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(kv_made + (PAIR ? kRing : 0));
  static_assert((2 * kKcStages + (PAIR ? 3 : 2) * kRing + 2 + 10 + 4) * 8 + kKcMeta * 8 + 36 <= 384, "barriers");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t cta = PAIR ? cluster_cta_rank() : 0;          // 0 issues the products of both
  if (threadIdx.x == 0) {
    for (int s = 0; s < kKcStages; ++s) {
      mbar_init(&st_full[s], 1);
      mbar_init(&st_empty[s], kConvert);
    }
    for (int s = 0; s < kRing; ++s) {
      mbar_init(&kv_full[s], PAIR ? kCtas : kConvert);
      mbar_init(&kv_empty[s], 1);
      if constexpr (PAIR) mbar_init(&kv_made[s], kConvert);
    }
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int g = 0; g < 2; ++g) {
      mbar_init(&s_full[g], 1);
      mbar_init(&p_full[g * 2], kCtas * 4);
      mbar_init(&p_full[g * 2 + 1], kCtas * 4);
      mbar_init(&o_full[g * 2], 1);
      mbar_init(&o_full[g * 2 + 1], 1);
    }
    for (int i = 0; i < 4; ++i) mbar_init(&meet[i], 2);
    mbar_fence_init();
    tma_prefetch_desc(&tma_q);
  }
  if (warp == 1) {
    if constexpr (PAIR) {
      tmem_alloc_pair(tmem_holder, 512);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(tmem_holder, 512);
      tmem_relinquish();
    }
  }
  // rows that no query fills stay zeros
  for (int i = threadIdx.x; i < Cfg::kQ * Cfg::kTile / 16; i += Cfg::kThreads) reinterpret_cast<uint4*>(smem_q)[i] = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync_all();                // both CTAs' barriers are there before anybody signals the partner
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;

  const int item0 = p.first[blockIdx.x / kCtas], item1 = p.first[blockIdx.x / kCtas + 1];
  // To the warp that issues: weights are in tensor memory, scores may be written over.
  auto arrive_issuer = [&](uint64_t* bar) {
    if constexpr (PAIR)
      mbar_arrive_relaxed(map_to_cta(smem_u32(bar), 0));
    else
      mbar_arrive(bar);
  };
  auto commit = [&](uint64_t* bar) {
    if constexpr (PAIR)
      tc_commit_both(bar);
    else
      tc_commit(bar);
  };
  auto wait = [&](uint64_t* bar, uint32_t parity, int code) {      // of a whole warp
    const bool r = __all_sync(0xffffffffu, mbar_wait<PAIR>(bar, parity, p.status, code));
    tc_fence_after();
    return r;
  };
  auto next = [](int& slot, uint32_t& phase, int n) {
    if (++slot == n) {
      slot = 0;
      phase ^= 1;
    }
  };

  // Commits arrive by themselves, in pairs from the partner's tensor core too: the block does not leave before the last ones have, those of
  // every tile that is still in the ring (a slot that was never taken counts as given back).
  auto ring_given_back = [&](int slot, uint32_t phase) {
    for (int i = 0; i < kRing && wait(&kv_empty[slot], phase ^ 1, kTimeoutEmpty); ++i) next(slot, phase, kRing);
  };

  auto convert = [&]() {
    // ---------------------------------------------------------------- codes to tiles
    const int part = warp - 4;
    // Keys' exponents are taken relative to 16 above their largest: they are at most 2^-7 then, and 128 products with queries of any size
    // fit fp32.  Less where the reference times the scale would come near the end of fp32: queries for which the rest matters have scores
    // behind that end.
    const int most_ref = min(111, 110 + 127 - static_cast<int>(__float_as_uint(p.scale_log2) >> 23));
    bool ok = true;
    int st = 0, slot = 0;
    uint32_t st_phase = 0, phase = 0, n_blocks = 0;
    for (int at = item0; at < item1 && ok; ++at) {
      const int blocks = p.items[at].blocks, left0 = p.items[at].len - p.items[at].block0 * kKcBlock;
      int vref = 0;
      for (int j = 0; j < blocks && ok; ++j) {
        ok = wait(&st_full[st], st_phase, kTimeoutFull);
        if (!ok) break;
        const int valid = min(kKcBlock, left0 - j * kKcBlock);
        const uint8_t* stage = smem_st + st * Cfg::kStage;
        int kmax = 0, vmax = 0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int word = lane + 32 * i, t = (word >> 3) * kKv8Page + (word & 7);
          const uint32_t e = *reinterpret_cast<const uint32_t*>(stage + (word >> 3) * Kv8<D>::kBlock + 2 * Kv8<D>::kHalf + (word & 7) * 4);
          if (t < valid) kmax = max(kmax, static_cast<int>(e & 255)), vmax = max(vmax, static_cast<int>(e >> 16 & 255));
          if (t + 8 < valid) kmax = max(kmax, static_cast<int>(e >> 8 & 255)), vmax = max(vmax, static_cast<int>(e >> 24));
        }
        kmax = __reduce_max_sync(0xffffffffu, kmax);
        vmax = __reduce_max_sync(0xffffffffu, vmax);
        if (j == 0 || vmax > vref + 7) vref = vmax;       // factors up to 2^127 do without a new one
        const int kref = kmax + min(max(most_ref + 127 - kmax, 0), 16);
        if (part == 0 && lane == 0) meta[n_blocks % kKcMeta] = make_int2(kref - 127, vref - 127);
        ++n_blocks;
        const bool ragged = valid < kKcBlock;
        auto tile = [&](auto value) {
          constexpr int kValue = decltype(value)::value;
          ok = wait(&kv_empty[slot], phase ^ 1, kTimeoutEmpty);
          if (!ok) return;
          // A lane has the same 16 columns of some tokens.  Eight neighbouring lanes read eight places of 16 bytes that lie in different
          // banks, and so do the two they write to: one token's whole row, half of them with their two units the other way around, or
          // (PAIR's values, half a row) those of a token and of another two pages on.
          constexpr bool kHalfRow = PAIR && kValue;
          constexpr int kUnits = (kHalfRow ? D / 2 : D) / 16, kRows = PAIR && !kValue ? 64 : 128;           // units of a row; tokens
          constexpr int kAt = kRows * kUnits / (32 * kConvert);
          const int c = kHalfRow ? lane & 3 : lane % kUnits;
          const int t0 = kHalfRow ? (lane >> 2 & 1) * 32 + part * 4 + (lane >> 3) : (part * 32 + lane) / kUnits;
          const bool swap = kHalfRow ? lane >> 2 & 1 : c >> 2;
          const int u0 = kHalfRow ? 2 * c + swap : 2 * (c & 3) + swap;
          // tokens from a lane's first to its k-th
          auto after = [](int k) { return kHalfRow ? (k * 4 * kConvert & 31) + 64 * (k * 4 * kConvert >> 5) : k * (32 * kConvert / kUnits); };
          static_assert(kHalfRow || 32 * kConvert / kUnits % 16 == 0, "a lane's tokens have the same place in their pages");
          const int t_half = PAIR && !kValue ? static_cast<int>(cta) * 64 : 0;       // the first token of the tile
          const uint32_t page0 = smem_u32(stage) + ((t0 + t_half) >> 4) * Kv8<D>::kBlock;
          const uint32_t codes = page0 + kValue * Kv8<D>::kHalf + (t0 & 15) * D + c * 16 + (kHalfRow ? cta * (D / 2) : 0);
          const uint32_t exps = page0 + 2 * Kv8<D>::kHalf + kv8_exponent_at(t0 & 15, kValue);
          const uint32_t to = smem_u32(smem_kv) + slot * Cfg::kKv + (c >> 2) * kRows * 128 + t0 * 128, u = (u0 ^ (t0 & 7)) << 4;
          const uint32_t sign = kValue ? 0u : p.key_sign;
          const int up = 127 + 120 - (kValue ? vref : kref);
          uint4 w[kAt];
          int e[kAt];
#pragma unroll
          for (int k = 0; k < kAt; ++k) {
            w[k] = lds128(codes + after(k) / 16 * Kv8<D>::kBlock);
            e[k] = lds8(exps + after(k) / 16 * Kv8<D>::kBlock);
          }
          uint32_t none_of = 0;          // the top bit of a byte: some code there was no number
          auto turn = [&](uint4 r, int exponent, int later, bool none) {
            uint32_t f = static_cast<uint32_t>(max(exponent + up, 0)) * 0x00800080u + sign;      // two exponents
            if (ragged && t_half + t0 + later >= valid) r = make_uint4(0, 0, 0, 0), f = 0;
            none_of |= ((r.x & 0x7F7F7F7Fu) + 0x01010101u) | ((r.y & 0x7F7F7F7Fu) + 0x01010101u);
            none_of |= ((r.z & 0x7F7F7F7Fu) + 0x01010101u) | ((r.w & 0x7F7F7F7Fu) + 0x01010101u);
            if (swap) r = make_uint4(r.z, r.w, r.x, r.y);
            uint4 a, b;
            e4m3x4_to_bf16(r.x, f, a.x, a.y);
            e4m3x4_to_bf16(r.y, f, a.z, a.w);
            e4m3x4_to_bf16(r.z, f, b.x, b.y);
            e4m3x4_to_bf16(r.w, f, b.z, b.w);
            if (none) {
              e4m3x4_nan(r.x, a.x, a.y);
              e4m3x4_nan(r.y, a.z, a.w);
              e4m3x4_nan(r.z, b.x, b.y);
              e4m3x4_nan(r.w, b.z, b.w);
            }
            sts128(to + later * 128 + u, a);
            sts128(to + later * 128 + (u ^ 16), b);
          };
#pragma unroll
          for (int k = 0; k < kAt; ++k) turn(w[k], e[k], after(k), false);
          if (none_of & 0x80808080u) {          // hardly ever: once more
#pragma unroll 1
            for (int k = 0; k < kAt; ++k)
              turn(lds128(codes + after(k) / 16 * Kv8<D>::kBlock), lds8(exps + after(k) / 16 * Kv8<D>::kBlock), after(k), true);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(PAIR ? &kv_made[slot] : &kv_full[slot]);
          next(slot, phase, kRing);
        };
        tile(std::integral_constant<int, 0>());
        if (ok) tile(std::integral_constant<int, 1>());
        if (!ok) break;
        if (lane == 0) mbar_arrive(&st_empty[st]);
        next(st, st_phase, kKcStages);
      }
    }
    if (!PAIR && ok) ring_given_back(slot, phase);
  };

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Cfg::kRegsIssue));
    if (warp == 0) {
      // ---------------------------------------------------------------- copies
      bool ok = true;
      int slot = 0;
      uint32_t phase = 0, n_q = 0;
      for (int at = item0; at < item1 && ok; ++at) {
        const Kv8Item w = p.items[at];
        if (w.blocks == 0) continue;
        const int tiles = !DUAL && w.tokens > kCtas * p.tp ? 2 : 1, pages = (w.len + kKv8Page - 1) / kKv8Page;
        const int* table = p.table + w.seq * p.ld_table;
        auto page_of = [&](int j) {        // of block j, a lane each
          const int i = (w.block0 + j) * 8 + lane;
          return j < w.blocks && lane < 8 && i < pages ? table[i] : -1;
        };
        int id = page_of(0);
        ok = wait(q_empty, (n_q & 1) ^ 1, kTimeoutEmpty);
        if (!ok) break;
        ++n_q;
        if (lane == 0) {
          if (cta == 0) mbar_expect_tx(q_full, kCtas * tiles * kChunks * 128 * p.hp * p.tp);
          const uint32_t bar = PAIR ? map_to_cta(smem_u32(q_full), 0) : 0;
          for (int g = 0; g < tiles; ++g)
            for (int c = 0; c < kChunks; ++c) {
              uint8_t* to = smem_q + g * Cfg::kTile + c * 16384;
              const int row = w.row0 + (g * kCtas + static_cast<int>(cta)) * p.tp;
              if constexpr (PAIR)
                tma_load_3d_pair(to, &tma_q, bar, c * 64, w.head0, row);
              else
                tma_load_3d(to, &tma_q, q_full, c * 64, w.head0, row);
            }
        }
        for (int j = 0; j < w.blocks; ++j) {
          const int id_next = page_of(j + 1);
          ok = wait(&st_empty[slot], phase ^ 1, kTimeoutEmpty);
          if (!ok) break;
          const int n = __popc(__ballot_sync(0xffffffffu, id >= 0));
          if (lane == 0) mbar_expect_tx(&st_full[slot], n * Kv8<D>::kBlock);
          __syncwarp();
          if (id >= 0)
            bulk_load(smem_st + slot * Cfg::kStage + lane * Kv8<D>::kBlock,
                      p.data + (static_cast<long long>(id) * p.Hkv + w.kvh) * Kv8<D>::kBlock, Kv8<D>::kBlock, &st_full[slot]);
          __syncwarp();
          id = id_next;
          next(slot, phase, kKcStages);
        }
      }
      if (ok) ok = wait(q_empty, (n_q & 1) ^ 1, kTimeoutEmpty);          // the last commit, as with the ring's
      if (!ok) {
        const uint64_t t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 100000ull) {
        }
      }
    } else if (warp == 1 && cta == 0) {
      // ---------------------------------------------------------------- products (one elected lane issues)
      const uint32_t idesc_s = umma_idesc_bf16(kCtas * 128, kKcBlock, 0, 0), idesc_o = umma_idesc_bf16(kCtas * 128, D, 0, 1);
      const uint64_t desc_q = umma_smem_desc(smem_u32(smem_q), 0, 1024), desc_k = umma_smem_desc(smem_u32(smem_kv), 0, 1024);
      const uint64_t desc_v = umma_smem_desc(smem_u32(smem_kv), 16384, 1024);
      constexpr uint32_t kT = Cfg::kTile >> 4, kKvT = Cfg::kKv >> 4;
      auto issue_s = [&](uint32_t g, uint32_t slot, uint32_t q) {
        const uint32_t d = tmem_base + g * 128;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint64_t a = desc_q + q * kT + (k / 4) * 1024 + (k % 4) * 2;
          const uint64_t b = desc_k + slot * kKvT + (k / 4) * (1024 / kCtas) + (k % 4) * 2;
          if constexpr (PAIR)
            umma_bf16_ss_pair(d, a, b, idesc_s, k > 0 ? 1u : 0u);
          else
            umma_bf16_ss(d, a, b, idesc_s, k > 0 ? 1u : 0u);
        }
        commit(&s_full[g]);
      };
      // the h-th part of the block's columns
      auto issue_o = [&](uint32_t g, uint32_t h, uint32_t slot, bool first) {
#pragma unroll
        for (int k = 0; k < kCols / 16; ++k) {
          const uint32_t d = tmem_base + 256 + g * 128, a = tmem_base + g * 128 + h * 32 + k * 8;
          const uint64_t b = desc_v + slot * kKvT + (h * 4 + k) * 128;
          if constexpr (PAIR)
            umma_bf16_ts_pair(d, a, b, idesc_o, (!first || k > 0) ? 1u : 0u);
          else
            umma_bf16_ts(d, a, b, idesc_o, (!first || k > 0) ? 1u : 0u);
        }
      };
      int slot = 0;
      uint32_t phase = 0, n_q = 0, done[2] = {0, 0};
      auto wait_slot = [&]() {
        const bool r = wait(&kv_full[slot], phase, kTimeoutFull);
        next(slot, phase, kRing);
        return r;
      };
      bool ok = true;
      uint32_t tile = 0;               // kDual: number of the item's first tile
      for (int at = item0; at < item1 && ok; ++at) {
        const int blocks = p.items[at].blocks, tiles = !DUAL && p.items[at].tokens > kCtas * p.tp ? 2 : 1;
        if (blocks == 0) continue;
        if constexpr (DUAL) {
          auto wait_tile = [&](uint32_t t) { return wait(&kv_full[t % kRing], (t / kRing) & 1, kTimeoutFull); };
          auto scores = [&](int j) {   // of block j, when its keys are there
            const uint32_t t = tile + 2 * j;
            if (!wait_tile(t)) return false;
            if (elect_one()) {
              issue_s(j & 1, t % kRing, 0);
              commit(&kv_empty[t % kRing]);
              if (j + 1 == blocks) commit(q_empty);
            }
            __syncwarp();
            return true;
          };
          ok = wait(q_full, n_q & 1, kTimeoutFull) && scores(0) && (blocks == 1 || scores(1));
          ++n_q;
          for (int j = 0; j < blocks && ok; ++j) {
            const uint32_t g = j & 1, t = tile + 2 * j + 1;
            ok = wait_tile(t);
            for (int h = 0; h < 2 && ok; ++h) {
              ok = wait(&p_full[g * 2 + h], done[g] >> 1 & 1, kTimeoutTmemEmpty);
              if (!ok) break;
              ++done[g];
              if (elect_one()) {
                issue_o(g, h, t % kRing, j < 2 && h == 0);
                commit(&o_full[g * 2 + h]);
                if (h == 1) commit(&kv_empty[t % kRing]);
              }
              __syncwarp();
            }
            if (!ok) break;
            if (j + 2 < blocks) ok = scores(j + 2);
          }
          tile += 2 * blocks;
          continue;
        }
        int sk = slot;
        ok = wait(q_full, n_q & 1, kTimeoutFull) && wait_slot();
        if (!ok) break;
        ++n_q;
        if (elect_one()) {
          for (int g = 0; g < tiles; ++g) issue_s(g, sk, g);
          commit(&kv_empty[sk]);
          if (blocks == 1) commit(q_empty);
        }
        __syncwarp();
        for (int j = 0; j < blocks && ok; ++j) {
          const bool more = j + 1 < blocks;
          const int sv = slot;
          ok = wait_slot();
          sk = slot;
          if constexpr (kHalves == 1) {
            if (ok && more) ok = wait_slot();          // ahead of the weights, not between them and their product
            if (!ok) break;
            for (int g = 0; g < tiles && ok; ++g) {
              ok = wait(&p_full[g * 2], done[g] & 1, kTimeoutTmemEmpty);
              if (!ok) break;
              ++done[g];
              if (elect_one()) {
                issue_o(g, 0, sv, j == 0);
                if (more)
                  issue_s(g, sk, g);      // over P, which the product above reads first: the tensor core keeps the order of issue
                else
                  commit(&o_full[g * 2]);
                if (g == tiles - 1) {
                  commit(&kv_empty[sv]);
                  if (more) commit(&kv_empty[sk]);
                  if (j + 2 == blocks) commit(q_empty);
                }
              }
              __syncwarp();
            }
          } else {
            for (int g = 0; g < tiles && ok; ++g) {
              for (int h = 0; h < 2 && ok; ++h) {
                ok = wait(&p_full[g * 2 + h], done[g] >> 1 & 1, kTimeoutTmemEmpty);
                if (!ok) break;
                ++done[g];
                if (elect_one()) {
                  issue_o(g, h, sv, j == 0 && h == 0);
                  commit(&o_full[g * 2 + h]);
                  if (h == 1 && g == tiles - 1) commit(&kv_empty[sv]);
                }
                __syncwarp();
                if (!more || h == 0) continue;
                if (g == 0 && !(ok = wait_slot())) break;
                if (elect_one()) {
                  issue_s(g, sk, g);
                  if (g == tiles - 1) {
                    commit(&kv_empty[sk]);
                    if (j + 2 == blocks) commit(q_empty);
                  }
                }
                __syncwarp();
              }
            }
          }
        }
      }
    } else if (PAIR && warp == 2) {
      // ---------------------------------------------------------------- tiles made, to the CTA that issues
      // Tiles are stores to shared memory that the products of another CTA's thread read: they have to be released at the cluster's scope.
      // By the warps that make them that takes 1000 clocks a tile, for their own stores to settle (512 tokens behind 16384: 202 us where no
      // release took 148); a warp that has none passes on what it has acquired (164 where none took 156).
      int tiles = 0;
      for (int at = item0; at < item1; ++at) tiles += 2 * p.items[at].blocks;
      int slot = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int i = 0; i < tiles && ok; ++i) {
        ok = wait(&kv_made[slot], phase, kTimeoutFull);
        if (!ok) break;
        if (lane == 0) mbar_arrive_cluster(map_to_cta(smem_u32(&kv_full[slot]), 0));
        next(slot, phase, kRing);
      }
      if (ok) ring_given_back(slot, phase);
    }
  } else if (warp < 4 + kConvert) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Cfg::kRegsConvert));
    convert();
  } else {
    // ------------------------------------------------------------------ softmax groups
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Cfg::kRegsSoftmax));
    const int g = (warp - 4 - kConvert) >> 2, quarter = warp & 3, row = quarter * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t t_s0 = tmem_base + lane_off + g * 128;        // scores; weights go over the first half of them
    const uint32_t t_o = tmem_base + lane_off + 256 + g * 128;
    const int row_token = (DUAL ? 0 : (g * kCtas + static_cast<int>(cta)) * p.tp) + row / p.hp, row_head = row % p.hp;
    uint32_t parts_seen = 0, blocks_all = 0, items = 0, met = 0;
    bool ok = true;
    auto meet_other = [&]() {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&meet[quarter]);
      return wait(&meet[quarter], met++ & 1, kTimeoutTmemFull);
    };
    for (int at = item0; at < item1 && ok; ++at) {
      const Kv8Item w = p.items[at];
      if (!DUAL && g > 0 && w.tokens <= kCtas * p.tp) {
        blocks_all += w.blocks;
        continue;
      }
      const int seen = min(w.len, w.pos0 + row_token + 1) - w.block0 * kKcBlock;      // tokens of the range that the row sees (or more)
      auto asked_for = [&]() { return row < p.hp * p.tp && row_token < w.tokens && row_head < w.heads; };
      // rows that nobody asked for: whatever their weights are, nothing is stored (of two tiles few are such, and the test costs them 2%)
      const bool idle = DUAL && !__any_sync(0xffffffffu, asked_for());
      float m_ref = -INFINITY;             // what weights are relative to: a score of the row not far below its largest
      uint64_t l2 = 0;
      int ev = 0;
      const int mine_n = kHalves * (DUAL ? (w.blocks + 1 - g) / 2 : w.blocks);          // this group's parts of blocks
      for (int k = 0; k < mine_n; ++k) {
        const int j = DUAL ? k / kHalves * 2 + g : k / kHalves, h = k % kHalves;
        const uint32_t t_s = t_s0 + h * 64;
        if (h == 0) ok = wait(&s_full[g], parts_seen / kHalves & 1, kTimeoutTmemFull);
        if (!ok) break;
        ++parts_seen;
        if (idle) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive_issuer(&p_full[g * 2 + h]);
          continue;
        }
        const int2 ref = meta[(blocks_all + j) % kKcMeta];
        const float c1 = fmaxf(p.scale_log2 * exp2_int(ref.x), 1.2e-38f);
        const uint64_t c2 = xtc_pair(c1, c1);
        const int limit = seen - j * kKcBlock - h * 64;
        const bool masked = __any_sync(0xffffffffu, limit < kCols);
        if (k == 0) ev = ref.y;
        float alpha = 1.f;
        auto mask = [&](int c, uint32_t (&x)[16]) {
          if (masked) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (c * 16 + i >= limit) x[i] = 0xff800000u;
          }
        };
        // Once through the scores, 16 columns at a time and the next ones on their way.  The reference stays while weights fit in: any will
        // do as long as nothing overflows, and bf16 has the range.  Where a block's sum passes 2^40 its weights are taken again, with
        // the row's maximum as the reference (scores that spread by 130 nats, so that most blocks of some row do: 4.0 us a block for 2.4).
        // Weights are rounded to bf16, the type of the values' tiles, by half a step of 2^-8 each.  Behind a reference that is not the row's
        // maximum the largest weight is rounded as well: errors of rows with few large weights are 2.2e-3 of their norm instead of 1.8e-3
        // (of which 1.7e-3 are the output's own rounding), of others 2.4e-3 instead of 2.3e-3.  Sums of the rounded weights would mend
        // most of it and take 10% longer.
        constexpr int kRuns = kCols / 16;
        uint32_t pk[kCols / 2];
        uint64_t sum = 0;
        bool anew = __any_sync(0xffffffffu, m_ref == -INFINITY && limit > 0);
#pragma unroll 1
        for (int turn = 0; turn < 2; ++turn) {
          uint32_t v[2][16];
          tmem_ld_32x16(t_s, v[0]);
          tmem_ld_wait(v[0]);
          if (anew) {
            float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int c = 0; c < kRuns; ++c) {
              tmem_ld_32x16(t_s + (c + 1) % kRuns * 16, v[(c + 1) & 1]);
              mask(c, v[c & 1]);
#pragma unroll
              for (int i = 0; i < 16; i += 2)
                mx[(i >> 1) & 1] = fmaxf(fmaxf(mx[(i >> 1) & 1], __uint_as_float(v[c & 1][i])), __uint_as_float(v[c & 1][i + 1]));
              tmem_ld_wait(v[(c + 1) & 1]);
            }
            const float m_new = fmaxf(m_ref, fmaxf(mx[0], mx[1]) * c1);
            alpha = m_ref == -INFINITY ? 0.f : xtc_ex2(m_ref - m_new);
            m_ref = m_new;
          }
          const float m_use = m_ref == -INFINITY ? 0.f : m_ref;
          const uint64_t nm2 = xtc_pair(-m_use, -m_use);
          uint64_t part[2] = {0, 0};
#pragma unroll
          for (int c = 0; c < kRuns; ++c) {
            if (c + 1 < kRuns) tmem_ld_32x16(t_s + (c + 1) * 16, v[(c + 1) & 1]);
            mask(c, v[c & 1]);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              float2 f = xtc_unpair(xtc_fma2(xtc_pair(__uint_as_float(v[c & 1][2 * i]), __uint_as_float(v[c & 1][2 * i + 1])), c2, nm2));
              f.x = xtc_ex2(f.x);
              f.y = xtc_ex2(f.y);
              part[i & 1] = xtc_add2(part[i & 1], xtc_pair(f.x, f.y));
              pk[c * 8 + i] = pack_bf16x2(f.x, f.y);
            }
            if (c + 1 < kRuns) tmem_ld_wait(v[(c + 1) & 1]);
          }
          sum = xtc_add2(part[0], part[1]);
          const float2 f = xtc_unpair(sum);
          if (anew || !__any_sync(0xffffffffu, !(f.x + f.y <= kKcRoom))) break;
          anew = true;
        }
        if (k > 0 && (anew || ev != ref.y)) {
          // O with what came before: issued ahead of this S, but for the product of the block's first half
          if (h == 1 && !(ok = wait(&o_full[g * 2], (parts_seen - 1) / kHalves & 1, kTimeoutTmemFull))) break;
          l2 = xtc_mul2(l2, xtc_pair(alpha, alpha));
          const float ao = alpha * exp2_int(max(ev - ref.y, -126));
          const uint64_t a2 = xtc_pair(ao, ao);
          uint32_t r[16];
#pragma unroll
          for (int c = 0; c < D / 16; ++c) {
            tmem_ld_32x16(t_o + c * 16, r);
            tmem_ld_wait(r);
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
              const float2 f = xtc_unpair(xtc_mul2(xtc_pair(__uint_as_float(r[i]), __uint_as_float(r[i + 1])), a2));
              r[i] = __float_as_uint(f.x);
              r[i + 1] = __float_as_uint(f.y);
            }
            tmem_st_32x16(t_o + c * 16, r);
          }
        }
        ev = ref.y;
#pragma unroll
        for (int c = 0; c < kCols / 64; ++c) tmem_st_32x32(t_s0 + h * 32 + c * 32, *reinterpret_cast<const uint32_t(*)[32]>(pk + c * 32));
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_issuer(&p_full[g * 2 + h]);
        l2 = xtc_add2(l2, sum);
      }
      blocks_all += w.blocks;
      if (!ok) break;
      if (mine_n > 0) {
        ok = wait(&o_full[g * 2 + kHalves - 1], (kHalves == 1 ? items : (parts_seen - 1) >> 1) & 1, kTimeoutTmemFull);
        if (!ok) break;
        ++items;
      }
      // output = own O * f0 * 2^ev + the other group's O * f1 * 2^ev1; kDual: half of the columns per group
      const float2 lp = xtc_unpair(l2);
      float l = lp.x + lp.y;
      float f0 = l == 0.f ? 0.f : 1.f / l, f1 = 0.f;
      const float e0 = exp2_int(ev);
      float e1 = 0.f;
      constexpr int kOut = DUAL ? D / 2 : D;
      const int col0 = DUAL ? g * kOut : 0;
      if constexpr (DUAL) {
        float* y = reinterpret_cast<float*>(smem_x) + row;            // [2] groups of [128] references and [128] sums
        y[g * 256] = m_ref;
        y[g * 256 + 128] = l;
        if (lane == 0) other_ev[g * 4 + quarter] = ev;
        ok = meet_other();
        if (!ok) break;
        const float m1 = y[(1 - g) * 256], l1 = y[(1 - g) * 256 + 128];
        const float m = fmaxf(m_ref, m1), a0 = l == 0.f ? 0.f : xtc_ex2(m_ref - m), a1 = l1 == 0.f ? 0.f : xtc_ex2(m1 - m);
        l = g == 0 ? l * a0 + l1 * a1 : l1 * a1 + l * a0;
        m_ref = m;
        f0 = a0 == 0.f ? 0.f : a0 / l;
        f1 = a1 == 0.f ? 0.f : a1 / l;
        e1 = exp2_int(other_ev[(1 - g) * 4 + quarter]);
      }
      const bool mine = asked_for();
      __nv_bfloat16* dst = p.out + (static_cast<long long>(w.row0) + row_token) * p.ldo + (w.head0 + row_head) * D;
      const long long part = (static_cast<long long>(w.part) + (DUAL ? 0 : g * kCtas + static_cast<int>(cta))) * 128 + row;
#pragma unroll 1
      for (int c = col0; c < (idle ? col0 : col0 + kOut); c += 16) {
        uint32_t r[16];
        float f[16];
        if (mine_n > 0) {
          tmem_ld_32x16(t_o + c, r);
          tmem_ld_wait(r);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) f[i] = f0 == 0.f ? 0.f : __uint_as_float(r[i]) * f0 * e0;
        if (DUAL && (g == 0 ? w.blocks > 1 : w.blocks > 0)) {          // the other group has some
          tmem_ld_32x16(t_o + (g == 0 ? 128 : -128) + c, r);
          tmem_ld_wait(r);
#pragma unroll
          for (int i = 0; i < 16; ++i) f[i] += f1 == 0.f ? 0.f : __uint_as_float(r[i]) * f1 * e1;
        }
        if (mine) {
          if (w.part < 0) {
#pragma unroll
            for (int q = 0; q < 2; ++q)
              *reinterpret_cast<uint4*>(dst + c + q * 8) =
                  make_uint4(pack_bf16x2(f[q * 8], f[q * 8 + 1]), pack_bf16x2(f[q * 8 + 2], f[q * 8 + 3]), pack_bf16x2(f[q * 8 + 4], f[q * 8 + 5]),
                             pack_bf16x2(f[q * 8 + 6], f[q * 8 + 7]));
          } else {
#pragma unroll
            for (int q = 0; q < 4; ++q)
              *reinterpret_cast<float4*>(p.part_o + part * D + c + q * 4) = make_float4(f[q * 4], f[q * 4 + 1], f[q * 4 + 2], f[q * 4 + 3]);
          }
        }
      }
      if (w.part >= 0 && mine && (!DUAL || g == 0)) *reinterpret_cast<float2*>(p.part_s + part * 2) = make_float2(m_ref, l);
      tc_fence_before();
      if (DUAL && !(ok = meet_other())) break;          // the next item's products write over both groups' O
    }
    // the last commit that no reference asked for
    if (kHalves == 2 && ok && parts_seen > 0) wait(&o_full[g * 2], (parts_seen / 2 - 1) & 1, kTimeoutTmemFull);
  }

  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync_all();                // nobody's memory is still a target of the partner
  if (warp == 1) {
    tc_fence_after();
    if constexpr (PAIR)
      tmem_dealloc_pair(tmem_base, 512);
    else
      tmem_dealloc(tmem_base, 512);
  }
}

// Joins the parts of tiles that were cut along the keys; a warp per row.
struct Kv8ChunkJoin {
  int row0, tokens, head0, heads, part, parts, step, pad;       // the tile's rows; its parts: scratch tiles part, part + step, ...
};
template <int D>
__global__ void __launch_bounds__(128) kv8_chunk_join_kernel(const Kv8Chunk p, const Kv8ChunkJoin* __restrict__ joins) {
  constexpr int V = D / 32, KB = 4;
  const Kv8ChunkJoin w = joins[blockIdx.x];
  const int row = blockIdx.y * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31, token = row / p.hp, head = row % p.hp;
  if (token >= min(w.tokens, p.tp) || head >= w.heads) return;
  float m = -INFINITY, l = 0.f, o[V] = {};
  for (int k0 = 0; k0 < w.parts; k0 += KB) {
    float2 s[KB];
    float v[KB][V];
#pragma unroll
    for (int k = 0; k < KB; ++k) {
      const long long at = (static_cast<long long>(w.part) + (k0 + k) * w.step) * 128 + row;
      const bool there = k0 + k < w.parts;
      s[k] = there ? *reinterpret_cast<const float2*>(p.part_s + at * 2) : make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int i = 0; i < V; ++i) v[k][i] = there ? p.part_o[at * D + lane * V + i] : 0.f;
    }
#pragma unroll
    for (int k = 0; k < KB; ++k) {
      if (s[k].y == 0.f) continue;
      const float m1 = fmaxf(m, s[k].x), a = m == -INFINITY ? 0.f : xtc_ex2(m - m1), b = s[k].y * (s[k].x == -INFINITY ? 1.f : xtc_ex2(s[k].x - m1));
      l = l * a + b;
#pragma unroll
      for (int i = 0; i < V; ++i) o[i] = o[i] * a + v[k][i] * b;
      m = m1;
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  __nv_bfloat16* dst = p.out + (static_cast<long long>(w.row0) + token) * p.ldo + (w.head0 + head) * D + lane * V;
#pragma unroll
  for (int i = 0; i < V; i += 2) *reinterpret_cast<uint32_t*>(dst + i) = pack_bf16x2(o[i] * inv, o[i + 1] * inv);
}

template <int D, int FORM>
static int launch_kv8_chunk(const CUtensorMap& tq, const Kv8Chunk& p, int workers, const Kv8ChunkJoin* joins, int n_joins, cudaStream_t s) {
  static bool configured[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!configured[dev & 63]) {
    cudaError_t e = cudaFuncSetAttribute(kv8_chunk_kernel<D, FORM>, cudaFuncAttributeMaxDynamicSharedMemorySize, Kv8ChunkCfg<D, FORM>::kSmem);
    if (e != cudaSuccess) return static_cast<int>(e);
    configured[dev & 63] = true;
  }
  constexpr int kCtas = FORM == kPair ? 2 : 1;
  using Cfg = Kv8ChunkCfg<D, FORM>;
  cudaError_t e = launch_kernel_clusters(kv8_chunk_kernel<D, FORM>, dim3(workers * kCtas), dim3(Cfg::kThreads), Cfg::kSmem, kCtas, s, tq, p);
  if (e != cudaSuccess || n_joins == 0) return static_cast<int>(e);
  kv8_chunk_join_kernel<D><<<dim3(n_joins, (p.hp * p.tp + 3) / 4), 128, 0, s>>>(p, joins);
  return static_cast<int>(cudaGetLastError());
}

}  // namespace apb

extern "C" {
using namespace apb;

// q [T, Hq, D], out [T, Hq, D] (rows on 16-byte boundaries); items [..][12], first [workers + 1], joins [n_joins][8] and the form of the
// workers (CTAs or pairs) as apb_rt_kv8_plan makes them; scratch: part_tiles * 128 * (D + 2) floats.
int apb_kv8_chunk(const void* q, long long ldq, const void* data, const int* table, long long ld_table, const int* items, const int* first,
                  int workers, const int* joins, int n_joins, int part_tiles, int form, void* scratch, void* out, long long ldo, int T,
                  int Hq, int Hkv, int D, float scale, cudaStream_t s) {
  if (workers <= 0) return 0;
  if (form < kTwo || form > kPair || (form == kPair && D != 128)) return kBadArgument;
  if ((D != 64 && D != 128) || Hkv < 1 || Hq % Hkv || ldq % 8 || ldo % 8 || reinterpret_cast<uintptr_t>(q) % 16 ||
      reinterpret_cast<uintptr_t>(out) % 16 || reinterpret_cast<uintptr_t>(data) % 16 || reinterpret_cast<uintptr_t>(items) % 16)
    return kBadArgument;
  const int R = Hq / Hkv, hp = R < 128 ? R : 128, tp = 128 / hp;
  CUtensorMap tq;
  const uint64_t dims[3] = {static_cast<uint64_t>(D), static_cast<uint64_t>(Hq), static_cast<uint64_t>(T)};
  const uint64_t strides[2] = {static_cast<uint64_t>(D) * 2, static_cast<uint64_t>(ldq) * 2};
  const uint32_t box[3] = {64, static_cast<uint32_t>(hp), static_cast<uint32_t>(tp)};
  const int rc = make_tmap_nd(&tq, q, 2, 3, dims, strides, box);
  if (rc) return 1000 + rc;
  float* part_o = static_cast<float*>(scratch);
  Kv8Chunk p = {reinterpret_cast<const Kv8Item*>(items), first, static_cast<const uint8_t*>(data), table, ld_table,
                static_cast<__nv_bfloat16*>(out), ldo, part_o, part_o + static_cast<long long>(part_tiles) * 128 * D, Hkv, hp, tp,
                fabsf(scale) * 1.4426950408889634f, scale < 0.f ? 0x80008000u : 0u, status_device_ptr()};
  const Kv8ChunkJoin* j = reinterpret_cast<const Kv8ChunkJoin*>(joins);
  if (D == 64 && form == kDual) return launch_kv8_chunk<64, kDual>(tq, p, workers, j, n_joins, s);
  if (D == 64) return launch_kv8_chunk<64, kTwo>(tq, p, workers, j, n_joins, s);
  if (form == kPair) return launch_kv8_chunk<128, kPair>(tq, p, workers, j, n_joins, s);
  if (form == kDual) return launch_kv8_chunk<128, kDual>(tq, p, workers, j, n_joins, s);
  return launch_kv8_chunk<128, kTwo>(tq, p, workers, j, n_joins, s);
}
}
