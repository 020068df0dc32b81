// Attention of chunks of query tokens over the 8-bit cache (layout: kv_fp8.cuh) on tcgen05 tensor cores.
//
// A tile holds 128 rows: the query heads of one key head for 128 / heads neighbouring tokens, so that short chunks fill it too.  A CTA
// walks work items of one or two such tiles over a range of 128-token blocks: S = Q K^T and O += P V by 128 x 128 MMAs, S and O in
// tensor memory, P over S, one softmax warpgroup per tile, as in attention_fwd.cu.
//
// Keys and values are bf16 operands here: kind::f16 wants both sides in 16 bits, and queries and weights do not fit 8.  Pages come by
// bulk copies into a staging ring as they lie in the cache; two warps turn them into swizzled bf16 tiles, which serves both query
// tiles.  A code becomes a bf16 number by moving its bits (exponents off by 120), two at a time, and one multiplication by a power of
// two, which also brings in its token's exponent relative to a reference: for keys the block's largest exponent, which the softmax
// multiplies by, for values one that moves only when a block's is larger by 2^8 or more, and O with it.  Nothing is rounded: 2^-120
// of the reference is far below what counts (tokens more than 2^100 smaller than the largest of their sequence lose bits).
//
// Items over long contexts are cut along the keys where there are too few to fill the GPU (csrc/runtime_kv8.cpp); their parts are
// joined by kv8_chunk_join_kernel.
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

// Four warpgroups: issue, codes to tiles, two of softmax.  Registers move between them: 80 + 96 + 2 * 168 = 4 * 128, what the block was
// launched with.
constexpr int kKcThreads = 512;
constexpr int kKcConvert = 4;               // warps that turn codes into tiles
constexpr int kKcRegsIssue = 80, kKcRegsConvert = 96, kKcRegsSoftmax = 168;
constexpr int kKcBlock = 128;
constexpr int kKcStages = 2, kKcMeta = 4;

template <int D, bool DUAL>
struct Kv8ChunkCfg {
  static constexpr int kTile = 128 * D * 2;
  static constexpr int kQ = DUAL ? 1 : 2, kRing = DUAL ? 4 : 3;      // tiles
  static constexpr int kStage = 8 * Kv8<D>::kBlock;
  static constexpr int kSmem = (kQ + kRing) * kTile + kKcStages * kStage + 256 + (DUAL ? 1024 : 0) + 1024;
  static_assert(kSmem <= 227 * 1024, "shared memory of one CTA");
};

__device__ __forceinline__ void bulk_load(void* smem_dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(smem_dst)), "l"(src),
               "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
// Four codes times 2^-120 as bf16 pairs, each times its factor
__device__ __forceinline__ void e4m3x4_to_bf16(uint32_t w, uint32_t factor, uint32_t& lo, uint32_t& hi) {
  const uint32_t a = __byte_perm(w, 0, 0x1404), b = __byte_perm(w, 0, 0x3424);
  const uint32_t x = (a & 0x80008000u) | ((a >> 4) & 0x07F007F0u), y = (b & 0x80008000u) | ((b >> 4) & 0x07F007F0u);
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(lo) : "r"(x), "r"(factor));
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(hi) : "r"(y), "r"(factor));
}

// DUAL: items of one tile each; the two softmax groups take every second block of it and join what they have at the item's end.
template <int D, bool DUAL>
__global__ void __launch_bounds__(kKcThreads, 1) kv8_chunk_kernel(const __grid_constant__ CUtensorMap tma_q, const Kv8Chunk p) {
  using Cfg = Kv8ChunkCfg<D, DUAL>;
  constexpr int kRing = Cfg::kRing, kChunks = D / 64;
  extern __shared__ uint8_t kc_smem[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(kc_smem) + 1023) & ~uintptr_t(1023));
  uint8_t* smem_q = smem;
  uint8_t* smem_kv = smem + Cfg::kQ * Cfg::kTile;
  uint8_t* smem_st = smem_kv + kRing * Cfg::kTile;
  uint64_t* st_full = reinterpret_cast<uint64_t*>(smem_st + kKcStages * Cfg::kStage);
  uint64_t* st_empty = st_full + kKcStages;
  uint64_t* kv_full = st_empty + kKcStages;
  uint64_t* kv_empty = kv_full + kRing;
  uint64_t* q_full = kv_empty + kRing;
  uint64_t* q_empty = q_full + 1;
  uint64_t* s_full = q_empty + 1;      // [2]
  uint64_t* p_full = s_full + 2;       // [2]
  uint64_t* o_full = p_full + 2;       // [2] once per item
  uint64_t* pair = o_full + 2;         // DUAL: both softmax groups
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(pair + 1);
  int2* meta = reinterpret_cast<int2*>(tmem_holder + 2);      // [kKcMeta] reference exponents of a block's keys and values
  float* other = reinterpret_cast<float*>(st_full) + 64;      // [2][128] DUAL: a number per row and group
  int* other_ev = reinterpret_cast<int*>(meta + kKcMeta);     // [2]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kKcStages; ++s) {
      mbar_init(&st_full[s], 1);
      mbar_init(&st_empty[s], kKcConvert);
    }
    for (int s = 0; s < kRing; ++s) {
      mbar_init(&kv_full[s], kKcConvert);
      mbar_init(&kv_empty[s], 1);
    }
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int g = 0; g < 2; ++g) {
      mbar_init(&s_full[g], 1);
      mbar_init(&p_full[g], 128);
      mbar_init(&o_full[g], 1);
    }
    mbar_init(pair, 256);
    mbar_fence_init();
    tma_prefetch_desc(&tma_q);
  }
  if (warp == 1) {
    tmem_alloc(tmem_holder, 512);
    tmem_relinquish();
  }
  // rows that no query fills stay zeros
  for (int i = threadIdx.x; i < Cfg::kQ * Cfg::kTile / 16; i += kKcThreads) reinterpret_cast<uint4*>(smem_q)[i] = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;

  const int item0 = p.first[blockIdx.x], item1 = p.first[blockIdx.x + 1];
  auto wait = [&](uint64_t* bar, uint32_t parity, int code) {      // of a whole warp
    const bool r = __all_sync(0xffffffffu, mbar_wait(bar, parity, p.status, code));
    tc_fence_after();
    return r;
  };
  auto next = [](int& slot, uint32_t& phase, int n) {
    if (++slot == n) {
      slot = 0;
      phase ^= 1;
    }
  };

  auto convert = [&]() {
    // ---------------------------------------------------------------- codes to tiles
    const int part = warp - 4;
    constexpr int kUnits = D / 16;         // of 16 codes in a row
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
        if (part == 0 && lane == 0) meta[n_blocks % kKcMeta] = make_int2(kmax - 127, vref - 127);
        ++n_blocks;
#pragma unroll 1
        for (int which = 0; which < 2 && ok; ++which) {
          const int ref = which ? vref : kmax;
          const uint32_t sign = which ? 0u : p.key_sign;
          ok = wait(&kv_empty[slot], phase ^ 1, kTimeoutEmpty);
          if (!ok) break;
          // A lane has the same 16 columns of every kStep-th token; the upper half of a row takes its two units the other
          // way around, so that no bank is met twice.
          const int c = lane % kUnits, u0 = 2 * (c & 3) + (c >> 2), t0 = (part * 32 + lane) / kUnits;
          constexpr int kStep = 32 * kKcConvert / kUnits, kAt = 4;           // tokens between a lane's, of them at a time
          const bool swap = c >> 2, ragged = valid < kKcBlock;
          const uint32_t tile = smem_u32(smem_kv) + slot * Cfg::kTile + (c >> 2) * 16384;
          const uint32_t codes = smem_u32(stage) + which * Kv8<D>::kHalf + c * 16, exps = smem_u32(stage) + 2 * Kv8<D>::kHalf;
#pragma unroll 1
          for (int i = t0; i < 128; i += kStep * kAt) {
            uint4 w[kAt];
            int e[kAt];
#pragma unroll
            for (int k = 0; k < kAt; ++k) {
              const int t = i + k * kStep;
              w[k] = lds128(codes + (t >> 4) * Kv8<D>::kBlock + (t & 15) * D);
              e[k] = lds8(exps + (t >> 4) * Kv8<D>::kBlock + kv8_exponent_at(t & 15, which));
            }
#pragma unroll
            for (int k = 0; k < kAt; ++k) {
              const int t = i + k * kStep;
              uint32_t f = static_cast<uint32_t>(max(127 + 120 + e[k] - ref, 0)) << 7;
              f = f << 16 | f | sign;
              if (ragged && t >= valid) w[k] = make_uint4(0, 0, 0, 0), f = 0;
              uint4 a, b;
              e4m3x4_to_bf16(swap ? w[k].z : w[k].x, f, a.x, a.y);
              e4m3x4_to_bf16(swap ? w[k].w : w[k].y, f, a.z, a.w);
              e4m3x4_to_bf16(swap ? w[k].x : w[k].z, f, b.x, b.y);
              e4m3x4_to_bf16(swap ? w[k].y : w[k].w, f, b.z, b.w);
              const uint32_t row = tile + t * 128, u = (u0 ^ (t & 7)) << 4;
              sts128(row + u, a);
              sts128(row + (u ^ 16), b);
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&kv_full[slot]);
          next(slot, phase, kRing);
        }
        if (!ok) break;
        if (lane == 0) mbar_arrive(&st_empty[st]);
        next(st, st_phase, kKcStages);
      }
    }
  };

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kKcRegsIssue));
    if (warp == 0) {
      // ---------------------------------------------------------------- copies
      bool ok = true;
      int slot = 0;
      uint32_t phase = 0, n_q = 0;
      for (int at = item0; at < item1 && ok; ++at) {
        const Kv8Item w = p.items[at];
        if (w.blocks == 0) continue;
        const int tiles = !DUAL && w.tokens > p.tp ? 2 : 1, pages = (w.len + kKv8Page - 1) / kKv8Page;
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
          mbar_expect_tx(q_full, tiles * kChunks * 128 * p.hp * p.tp);
          for (int g = 0; g < tiles; ++g)
            for (int c = 0; c < kChunks; ++c)
              tma_load_3d(smem_q + g * Cfg::kTile + c * 16384, &tma_q, q_full, c * 64, w.head0, w.row0 + g * p.tp);
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
      if (!ok) {
        const uint64_t t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 100000ull) {
        }
      }
    } else if (warp == 1) {
      // ---------------------------------------------------------------- products (one elected lane issues)
      const uint32_t idesc_s = umma_idesc_bf16(128, kKcBlock, 0, 0), idesc_o = umma_idesc_bf16(128, D, 0, 1);
      const uint64_t desc_q = umma_smem_desc(smem_u32(smem_q), 0, 1024), desc_k = umma_smem_desc(smem_u32(smem_kv), 0, 1024);
      const uint64_t desc_v = umma_smem_desc(smem_u32(smem_kv), 16384, 1024);
      constexpr uint32_t kT = Cfg::kTile >> 4;
      auto issue_s = [&](uint32_t g, uint32_t slot, uint32_t q) {
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          umma_bf16_ss(tmem_base + g * 128, desc_q + q * kT + (k / 4) * 1024 + (k % 4) * 2, desc_k + slot * kT + (k / 4) * 1024 + (k % 4) * 2,
                       idesc_s, k > 0 ? 1u : 0u);
        tc_commit(&s_full[g]);
      };
      auto issue_o = [&](uint32_t g, uint32_t slot, bool first) {
#pragma unroll
        for (int k = 0; k < kKcBlock / 16; ++k)
          umma_bf16_ts(tmem_base + 256 + g * 128, tmem_base + g * 128 + k * 8, desc_v + slot * kT + k * 128, idesc_o, (!first || k > 0) ? 1u : 0u);
      };
      int slot = 0;
      uint32_t phase = 0, n_q = 0, done[2] = {0, 0};
      auto wait_slot = [&]() {
        const bool r = wait(&kv_full[slot], phase, kTimeoutFull);
        next(slot, phase, kRing);
        return r;
      };
      bool ok = true;
      uint32_t tile = 0;               // DUAL: number of the item's first tile
      for (int at = item0; at < item1 && ok; ++at) {
        const int blocks = p.items[at].blocks, tiles = !DUAL && p.items[at].tokens > p.tp ? 2 : 1;
        if (blocks == 0) continue;
        if constexpr (DUAL) {
          auto wait_tile = [&](uint32_t t) { return wait(&kv_full[t % kRing], (t / kRing) & 1, kTimeoutFull); };
          auto scores = [&](int j) {   // of block j, when its keys are there
            const uint32_t t = tile + 2 * j;
            if (!wait_tile(t)) return false;
            if (elect_one()) {
              issue_s(j & 1, t % kRing, 0);
              tc_commit(&kv_empty[t % kRing]);
              if (j + 1 == blocks) tc_commit(q_empty);
            }
            __syncwarp();
            return true;
          };
          ok = wait(q_full, n_q & 1, kTimeoutFull) && scores(0) && (blocks == 1 || scores(1));
          ++n_q;
          for (int j = 0; j < blocks && ok; ++j) {
            const uint32_t g = j & 1, t = tile + 2 * j + 1;
            ok = wait_tile(t) && wait(&p_full[g], done[g] & 1, kTimeoutTmemEmpty);
            if (!ok) break;
            ++done[g];
            if (elect_one()) {
              issue_o(g, t % kRing, j < 2);
              tc_commit(&kv_empty[t % kRing]);
              if (j + 2 >= blocks) tc_commit(&o_full[g]);
            }
            __syncwarp();
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
          tc_commit(&kv_empty[sk]);
          if (blocks == 1) tc_commit(q_empty);
        }
        __syncwarp();
        for (int j = 0; j < blocks && ok; ++j) {
          const bool more = j + 1 < blocks;
          const int sv = slot;
          ok = wait_slot();
          sk = slot;
          if (ok && more) ok = wait_slot();
          if (!ok) break;
          for (int g = 0; g < tiles && ok; ++g) {
            ok = wait(&p_full[g], done[g] & 1, kTimeoutTmemEmpty);
            if (!ok) break;
            ++done[g];
            if (elect_one()) {
              issue_o(g, sv, j == 0);
              if (more)
                issue_s(g, sk, g);      // over P, which the product above reads first: the tensor core keeps the order of issue
              else
                tc_commit(&o_full[g]);
              if (g == tiles - 1) {
                tc_commit(&kv_empty[sv]);
                if (more) tc_commit(&kv_empty[sk]);
                if (j + 2 == blocks) tc_commit(q_empty);
              }
            }
            __syncwarp();
          }
        }
      }
    }
  } else if (warp < 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kKcRegsConvert));
    convert();
  } else {
    // ------------------------------------------------------------------ softmax groups
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kKcRegsSoftmax));
    const int g = (warp >> 2) - 2, quarter = warp & 3, row = quarter * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t t_s = tmem_base + lane_off + g * 128, t_o = tmem_base + lane_off + 256 + g * 128;
    const int row_token = (DUAL ? 0 : g * p.tp) + row / p.hp, row_head = row % p.hp;
    uint32_t blocks_seen = 0, blocks_all = 0, items = 0, met = 0;
    bool ok = true;
    auto meet = [&]() {                // the other group
      tc_fence_before();
      mbar_arrive(pair);
      return wait(pair, met++ & 1, kTimeoutTmemFull);
    };
    for (int at = item0; at < item1 && ok; ++at) {
      const Kv8Item w = p.items[at];
      if (!DUAL && g > 0 && w.tokens <= p.tp) {
        blocks_all += w.blocks;
        continue;
      }
      const int seen = min(w.len, w.pos0 + row_token + 1) - w.block0 * kKcBlock;      // tokens of the range that the row sees (or more)
      float m_run = -INFINITY;
      uint64_t l2 = 0;
      int ev = 0;
      const int mine_n = DUAL ? (w.blocks + 1 - g) / 2 : w.blocks;          // blocks of this group
      for (int k = 0; k < mine_n; ++k) {
        const int j = DUAL ? 2 * k + g : k;
        ok = wait(&s_full[g], blocks_seen & 1, kTimeoutTmemFull);
        if (!ok) break;
        ++blocks_seen;
        const int2 ref = meta[(blocks_all + j) % kKcMeta];
        const float c1 = fmaxf(p.scale_log2 * exp2_int(ref.x), 1.2e-38f);
        const uint64_t c2 = xtc_pair(c1, c1);
        const int limit = seen - j * kKcBlock;
        const bool masked = __any_sync(0xffffffffu, limit < kKcBlock);
        // twice through the scores, 32 columns at a time and the next ones on their way: all 128 in registers spilled
        uint32_t v[2][32];
        auto mask = [&](int c, uint32_t (&x)[32]) {
          if (masked) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (c * 32 + i >= limit) x[i] = 0xff800000u;
          }
        };
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        tmem_ld_32x32(t_s, v[0]);
        tmem_ld_wait(v[0]);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          tmem_ld_32x32(t_s + ((c + 1) & 3) * 32, v[(c + 1) & 1]);
          mask(c, v[c & 1]);
#pragma unroll
          for (int i = 0; i < 32; i += 2)
            mx[(i >> 1) & 3] = fmaxf(fmaxf(mx[(i >> 1) & 3], __uint_as_float(v[c & 1][i])), __uint_as_float(v[c & 1][i + 1]));
          tmem_ld_wait(v[(c + 1) & 1]);
        }
        const float m_new = fmaxf(m_run, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * c1);
        if (k == 0) ev = ref.y;
        if (__any_sync(0xffffffffu, m_new > m_run) || ev != ref.y) {
          if (k > 0) {           // O holds the blocks before this one: their product was issued ahead of this S
            const float alpha = m_run == -INFINITY ? 0.f : xtc_ex2(m_run - m_new);
            l2 = xtc_mul2(l2, xtc_pair(alpha, alpha));
            const float ao = alpha * exp2_int(max(ev - ref.y, -126));
            const uint64_t a2 = xtc_pair(ao, ao);
            uint32_t r[2][16];
            tmem_ld_32x16(t_o, r[0]);
            tmem_ld_wait(r[0]);
#pragma unroll
            for (int c = 0; c < D / 16; ++c) {
              if (c + 1 < D / 16) tmem_ld_32x16(t_o + (c + 1) * 16, r[(c + 1) & 1]);
#pragma unroll
              for (int i = 0; i < 16; i += 2) {
                const float2 f = xtc_unpair(xtc_mul2(xtc_pair(__uint_as_float(r[c & 1][i]), __uint_as_float(r[c & 1][i + 1])), a2));
                r[c & 1][i] = __float_as_uint(f.x);
                r[c & 1][i + 1] = __float_as_uint(f.y);
              }
              tmem_st_32x16(t_o + c * 16, r[c & 1]);
              if (c + 1 < D / 16) tmem_ld_wait(r[(c + 1) & 1]);
            }
          }
          m_run = m_new;
          ev = ref.y;
        }
        const float m_use = m_run == -INFINITY ? 0.f : m_run;
        const uint64_t nm2 = xtc_pair(-m_use, -m_use);
        uint64_t sum[2] = {0, 0};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          if (c < 3) tmem_ld_32x32(t_s + (c + 1) * 32, v[(c + 1) & 1]);
          mask(c, v[c & 1]);
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float2 f = xtc_unpair(xtc_fma2(xtc_pair(__uint_as_float(v[c & 1][2 * i]), __uint_as_float(v[c & 1][2 * i + 1])), c2, nm2));
            f.x = xtc_ex2(f.x);
            f.y = xtc_ex2(f.y);
            sum[i & 1] = xtc_add2(sum[i & 1], xtc_pair(f.x, f.y));
            pk[i] = pack_bf16x2(f.x, f.y);
          }
          if (c < 3) tmem_ld_wait(v[(c + 1) & 1]);
          tmem_st_32x16(t_s + c * 16, pk);
        }
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&p_full[g]);
        l2 = xtc_add2(l2, xtc_add2(sum[0], sum[1]));
      }
      blocks_all += w.blocks;
      if (!ok) break;
      if (mine_n > 0) {
        ok = wait(&o_full[g], items & 1, kTimeoutTmemFull);
        if (!ok) break;
        ++items;
      }
      const float2 lp = xtc_unpair(l2);
      float l = lp.x + lp.y;
      // output = (own O * f0 + the other group's O * f1): DUAL, a half of the columns each
      float f0 = l == 0.f ? 0.f : exp2_int(ev) / l, f1 = 0.f;
      if constexpr (DUAL) {
        auto pass = [&](float x) {       // this row's number of the other group
          other[g * 128 + row] = x;
          ok = ok && meet();
          const float y = other[(1 - g) * 128 + row];
          ok = ok && meet();
          return y;
        };
        if (row == 0) other_ev[g] = ev;
        const float m1 = pass(m_run), l1 = pass(l);
        if (!ok) break;
        const float m = fmaxf(m_run, m1), a0 = l == 0.f ? 0.f : xtc_ex2(m_run - m), a1 = l1 == 0.f ? 0.f : xtc_ex2(m1 - m);
        const int ev1 = other_ev[1 - g];
        l = l * a0 + l1 * a1;
        m_run = m;
        f0 = a0 == 0.f ? 0.f : a0 * exp2_int(ev) / l;
        f1 = a1 == 0.f ? 0.f : a1 * exp2_int(ev1) / l;
      }
      const bool mine = row < p.hp * p.tp && row_token < w.tokens && row_head < w.heads;
      __nv_bfloat16* dst = p.out + (static_cast<long long>(w.row0) + row_token) * p.ldo + (w.head0 + row_head) * D;
      const long long part = (static_cast<long long>(w.part) + (DUAL ? 0 : g)) * 128 + row;
      constexpr int kPer = DUAL ? D / 64 : D / 32;           // runs of 32 columns per group
#pragma unroll 1
      for (int c = DUAL ? g * kPer : 0; c < (DUAL ? (g + 1) * kPer : kPer); ++c) {
        uint32_t r[32];
        float f[32];
        if (mine_n > 0) {
          tmem_ld_32x32(t_o + c * 32, r);
          tmem_ld_wait(r);
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) f[i] = f0 == 0.f ? 0.f : __uint_as_float(r[i]) * f0;
        if (DUAL && (g == 0 ? w.blocks > 1 : w.blocks > 0)) {          // the other group has some
          tmem_ld_32x32(t_o + (g == 0 ? 128 : -128) + c * 32, r);
          tmem_ld_wait(r);
#pragma unroll
          for (int i = 0; i < 32; ++i) f[i] += f1 == 0.f ? 0.f : __uint_as_float(r[i]) * f1;
        }
        if (mine) {
          if (w.part < 0) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
              *reinterpret_cast<uint4*>(dst + c * 32 + q * 8) =
                  make_uint4(pack_bf16x2(f[q * 8], f[q * 8 + 1]), pack_bf16x2(f[q * 8 + 2], f[q * 8 + 3]), pack_bf16x2(f[q * 8 + 4], f[q * 8 + 5]),
                             pack_bf16x2(f[q * 8 + 6], f[q * 8 + 7]));
          } else {
#pragma unroll
            for (int q = 0; q < 8; ++q)
              *reinterpret_cast<float4*>(p.part_o + part * D + c * 32 + q * 4) = make_float4(f[q * 4], f[q * 4 + 1], f[q * 4 + 2], f[q * 4 + 3]);
          }
        }
      }
      if (w.part >= 0 && mine && (!DUAL || g == 0)) *reinterpret_cast<float2*>(p.part_s + part * 2) = make_float2(m_run, l);
      tc_fence_before();
      if (DUAL && !(ok = meet())) break;          // the next item's products write over both groups' O
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
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

template <int D, bool DUAL>
static int launch_kv8_chunk(const CUtensorMap& tq, const Kv8Chunk& p, int grid, const Kv8ChunkJoin* joins, int n_joins, cudaStream_t s) {
  static bool configured[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!configured[dev & 63]) {
    cudaError_t e = cudaFuncSetAttribute(kv8_chunk_kernel<D, DUAL>, cudaFuncAttributeMaxDynamicSharedMemorySize, Kv8ChunkCfg<D, DUAL>::kSmem);
    if (e != cudaSuccess) return static_cast<int>(e);
    configured[dev & 63] = true;
  }
    kv8_chunk_kernel<D, DUAL><<<grid, kKcThreads, Kv8ChunkCfg<D, DUAL>::kSmem, s>>>(tq, p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || n_joins == 0) return static_cast<int>(e);
  kv8_chunk_join_kernel<D><<<dim3(n_joins, (p.hp * p.tp + 3) / 4), 128, 0, s>>>(p, joins);
  return static_cast<int>(cudaGetLastError());
}

}  // namespace apb

extern "C" {
using namespace apb;

// q [T, Hq, D], out [T, Hq, D] (rows on 16-byte boundaries); one_tile: no item has two tiles; items [..][12], first [ctas + 1], joins [n_joins][8] as apb_rt_kv8_plan makes
// them; scratch: part_tiles * 128 * (D + 2) floats.
int apb_kv8_chunk(const void* q, long long ldq, const void* data, const int* table, long long ld_table, const int* items, const int* first,
                  int ctas, const int* joins, int n_joins, int part_tiles, int one_tile, void* scratch, void* out, long long ldo, int T, int Hq, int Hkv, int D,
                  float scale, cudaStream_t s) {
  if (ctas <= 0) return 0;
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
  if (one_tile) return D == 128 ? launch_kv8_chunk<128, true>(tq, p, ctas, j, n_joins, s) : launch_kv8_chunk<64, true>(tq, p, ctas, j, n_joins, s);
  return D == 128 ? launch_kv8_chunk<128, false>(tq, p, ctas, j, n_joins, s) : launch_kv8_chunk<64, false>(tq, p, ctas, j, n_joins, s);
}
}
