// Flash-attention backward for head_dim 128 on sm_100a (MHA and GQA) with ranges of queries for every key, capped scores and a distance
// bias (attn_mods.cuh).
//
// One CTA per (128-key tile, KV head or part of its query heads, sequence); it walks over the 64-row query tiles of its query heads
// between its first key's first query and its last key's last one.  Everything is computed with the keys in the TMEM lanes.  Per step
// five tcgen05 GEMMs:
//   S^T = K Q^T         dP^T = V dO^T                  (fp32 in TMEM, one key per lane, one query per column)
//   P^T = exp(score(S^T) - lse),  dS^T = P^T * (dP^T - D) * (1 - tanh^2 with a cap)   (bf16 back into TMEM, dS^T also into shared memory)
//   dV += P^T dO        dK += dS^T Q                   (A operand from TMEM; accumulated in TMEM over the whole walk)
//   dQ^T = K^T dS^T     -> TMEM -> shared memory -> added to a global fp32 dQ accumulator by TMA reduce-add
// Roles:
//   warps 0-7, 8-15  softmax of the even / odd steps, two threads per key (32 queries each)
//   warps 16-19      dQ^T: out of TMEM, transposed through shared memory, one TMA reduce-add per warp and step
//   warp 20          TMA producer: K and V once, then Q and dO through a ring of three stages
//   warps 21, 22     MMA issuers: the gradients of a step; S^T and dP^T of the step after next, into the columns that those leave
//   warp 23          the query rows' statistics for the ring, read one step ahead; clears padded rows of tiles that have some
// TMEM (512 columns): dV, dK (128 each) and two sets (even / odd steps) of [S^T | dP^T], 64 columns each: P^T and dS^T
// (bf16, 8 + 8 columns per 16 queries) replace S^T once it has been read, dQ^T replaces dP^T.  So the softmax of one step runs under
// the MMAs of its neighbours.  Bound: about 1700 cycles of MMA per step (S^T, dP^T and dQ^T with N = 64 take 48 instead of 32 cycles per
// instruction: shared memory delivers 128 bytes a cycle), and about 2300 of the shared-memory port with what else a step moves through it, 176 KB of
// operands, 32 of loads, 16 of dS^T and 64 of dQ^T; 2750 pass.
// bf16, 32 heads, causal, 1 x 8192: 1510 us with the passes before and after (82), 910 TFLOP/s; scores capped 1700; 32 / 8 heads in packed documents
// of 5 to 8000 tokens 425.  Straight from registers (`red`) dQ took 1670 instead of 1520; with K and V loaded behind the ranges, 1520.
// With a distance bias 8 to 16 bytes a thread spill.
// D = rowsum(dO * O) comes from a small pre-pass; scale and bf16 of dQ are applied by a post-pass, of dK at the end.
#include "attn_bwd_common.cuh"
#include "attn_mods.cuh"
#include "common.cuh"
#include "yafsdp_b200.h"

YF_TU_STATUS()

namespace {

constexpr int ATOM = 16384;        // [128 rows x 64 bf16], 128-byte swizzle
constexpr int TILE = 2 * ATOM;     // K or V: [128 x 128] bf16
constexpr int QATOM = 8192;        // [64 rows x 64 bf16]
constexpr int QTILE = 2 * QATOM;   // Q or dO of a step: [64 x 128] bf16
constexpr int STAGES = 3;          // ring of Q, dO and statistics
constexpr int BWD_THREADS = 768;
constexpr int DS_BYTES = ATOM;     // dS^T of a step: [128 keys x 64 queries] bf16
constexpr int DQ_BYTES = BQ * HD * 4;
constexpr int STAT_FLOATS = 2 * BQ;  // per stage: -lse * log2(e), -D
constexpr int BWD_SMEM = 1024 + 2 * TILE + STAGES * 2 * QTILE + 2 * DS_BYTES + DQ_BYTES + STAGES * STAT_FLOATS * 4 + 256;
static_assert(BWD_SMEM <= 232448, "shared memory of one CTA");
constexpr float LOG2E = 1.4426950408889634f;

struct BwdArgs {
  const float* lse;    // [B, Hq, S]
  const float* delta;  // [B, Hq, S]
  float4* dkv_parts;   // head_parts > 1: every part's own fp32 sums (part_tile), dK without scale; else null
  int S, B, Hq, Hkv;
  int head_group;      // order of the CTAs (head_group_order)
  int head_parts;      // CTAs that share a key tile of a KV head, each with a part of its query heads
  float scale, scale_log2;
  const int2* query_spans;  // [B, S] ranges of keys by query; null: causal
  AttnMods mods;
};

template <int MODS>
__global__ void __launch_bounds__(BWD_THREADS, 1)
attn_mods_bwd_kernel(const __grid_constant__ CUtensorMap tma_q, const __grid_constant__ CUtensorMap tma_k,
                     const __grid_constant__ CUtensorMap tma_v, const __grid_constant__ CUtensorMap tma_do,
                     const __grid_constant__ CUtensorMap tma_dq, const __grid_constant__ CUtensorMap tma_dk,
                     const __grid_constant__ CUtensorMap tma_dv, BwdArgs args) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sK = smem;
  uint8_t* sV = sK + TILE;
  uint8_t* sRing = sV + TILE;                      // stage s: Q at sRing + s * 2 * QTILE, dO at + QTILE
  uint8_t* sdS = sRing + STAGES * 2 * QTILE;       // even / odd steps
  uint8_t* sdQ = sdS + 2 * DS_BYTES;               // warp w of the dQ warps: [64 queries x 32 dims] fp32 at w * 8192
  float* sStat = reinterpret_cast<float*>(sdQ + DQ_BYTES);
  uint64_t* bars = reinterpret_cast<uint64_t*>(sStat + STAGES * STAT_FLOATS);
  uint64_t* kv_land = bars;                 // bytes of K and V, and of a stage's Q and dO, before padded rows are cleared
  uint64_t* q_land = bars + 1;              // [STAGES]
  uint64_t* kv_full = q_land + STAGES;
  uint64_t* q_full = kv_full + 1;           // [STAGES] ready, with the statistics
  uint64_t* q_empty = q_full + STAGES;      // [STAGES]
  uint64_t* sdp_full = q_empty + STAGES;    // [2] even / odd steps, as all that follow
  uint64_t* pds_ready = sdp_full + 2;
  uint64_t* dq_full = pds_ready + 2;
  uint64_t* vk_done = dq_full + 2;
  uint64_t* dq_read = vk_done + 2;
  uint64_t* all_done = dq_read + 2;         // every MMA of the walk (waiting two phases ahead on vk_done would not do)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(all_done + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  int jt, bh;  // key tile (under the causal mask the first ones have the longest walks), (sequence, KV head, part)
  const int n_kt = (args.S + BKV - 1) / BKV;
  head_group_order((int)blockIdx.x, n_kt, args.B * args.Hkv * args.head_parts, args.head_group, jt, bh);
  const int part = bh % args.head_parts, hk = (bh / args.head_parts) % args.Hkv, b = bh / (args.head_parts * args.Hkv);
  const int heads = args.Hq / args.Hkv / args.head_parts;  // query heads of this CTA
  const int h0 = hk * (args.Hq / args.Hkv) + part * heads;
  const int kv0 = jt * BKV;
  const int n_qt = (args.S + BQ - 1) / BQ;
  // ranges of queries by key, padded tokens by tile
  const int2* spans = args.mods.spans == nullptr ? nullptr : args.mods.spans + (long long)b * args.S;
  const int* padding = args.mods.spans == nullptr ? nullptr : args.mods.padding + (long long)b * n_kt;
  if (threadIdx.x == 0) {
    mbar_init(kv_land, 1);
    mbar_fence_init();
    // K and V do not depend on the ranges, whose loads take as long
    mbar_expect_tx(kv_land, 2 * TILE);
    tma_load_3d(sK, &tma_k, kv_land, hk * HD, kv0, b);
    tma_load_3d(sK + ATOM, &tma_k, kv_land, hk * HD + 64, kv0, b);
    tma_load_3d(sV, &tma_v, kv_land, hk * HD, kv0, b);
    tma_load_3d(sV + ATOM, &tma_v, kv_land, hk * HD + 64, kv0, b);
    tma_prefetch_desc(&tma_q);
    tma_prefetch_desc(&tma_do);
    tma_prefetch_desc(&tma_dq);
    mbar_init(kv_full, 1);
    mbar_init(all_done, 1);
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&q_land[i], 1);
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sdp_full[i], 1);
      mbar_init(&pds_ready[i], 8);
      mbar_init(&dq_full[i], 1);
      mbar_init(&vk_done[i], 1);
      mbar_init(&dq_read[i], 4);
    }
    mbar_fence_init();
  }
  int i_start = kv0 / BQ, per_head = n_qt - i_start;  // query tiles [i_start, + per_head)
  int dead_keys = 0;                                  // padded ones of this tile
  if (spans != nullptr) {
    const int keys = min(BKV, args.S - kv0);
    const int2 a = __ldg(spans + kv0), z = __ldg(spans + kv0 + keys - 1);
    dead_keys = __ldg(padding + jt);
    i_start = max(a.x, 0) / BQ;
    per_head = (min(z.y, args.S) + BQ - 1) / BQ - i_start;
    if (dead_keys >= keys || per_head < 0) per_head = 0;  // nothing but padding
  }
  const int n_it = per_head * heads;

  if (warp == 21) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const uint32_t tdV = tmem_base + 256, tdK = tmem_base + 384;  // set p of S^T | dP^T: tmem_base + 128 p, + 64

  if (warp == 20) {
    if (n_it > 0 && elect_one()) {
      int h = h0, i = 0;
      for (int it = 0, st = 0, ph = 1; it < n_it; ++it) {
        if (!mbar_wait(&q_empty[st], ph, 500)) break;
        const int q0 = (i_start + i) * BQ;
        uint8_t* sQ = sRing + st * 2 * QTILE;
        uint8_t* sdO = sQ + QTILE;
        mbar_expect_tx(&q_land[st], 2 * QTILE);
        tma_load_3d(sQ, &tma_q, &q_land[st], h * HD, q0, b);
        tma_load_3d(sQ + QATOM, &tma_q, &q_land[st], h * HD + 64, q0, b);
        tma_load_3d(sdO, &tma_do, &q_land[st], h * HD, q0, b);
        tma_load_3d(sdO + QATOM, &tma_do, &q_land[st], h * HD + 64, q0, b);
        if (++i == per_head) { i = 0; ++h; }
        if (++st == STAGES) { st = 0; ph ^= 1; }
      }
    }
  } else if (warp == 23) {
    // statistics of a step's 64 query rows, read one step ahead; rows past the end of the sequence: a probability of zero
    int h = h0, i = 0;
    float nl[2], dl[2];
    auto fetch = [&]() {
      const int q0 = (i_start + i) * BQ;
      const long long at = ((long long)b * args.Hq + h) * args.S + q0;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = lane + 32 * e;
        const bool ok = q0 + r < args.S;
        nl[e] = ok ? args.lse[at + r] * -LOG2E : -INFINITY;
        dl[e] = ok ? args.delta[at + r] : 0.f;
      }
    };
    if (n_it > 0) fetch();
    if (__all_sync(0xffffffffu, mbar_wait(kv_land, 0, 502))) {  // (without queries too: the tiles have to land before the block ends)
      if (n_it > 0) {
        if (dead_keys > 0) {  // dQ^T = K^T dS^T would multiply what padding holds by zeros
          zero_padded_rows(sK, ATOM, BKV, kv0, args.S, spans);
          fence_proxy_async_smem();
          __syncwarp();
        }
        if (lane == 0) mbar_arrive(kv_full);
      }
    }
    for (int it = 0, st = 0, ph = 1; it < n_it; ++it) {
      if (!__all_sync(0xffffffffu, mbar_wait(&q_empty[st], ph, 501))) break;
      float* stat = sStat + st * STAT_FLOATS;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        stat[lane + 32 * e] = nl[e];
        stat[BQ + lane + 32 * e] = -dl[e];
      }
      if (!__all_sync(0xffffffffu, mbar_wait(&q_land[st], ph ^ 1, 503))) break;
      const int q0 = (i_start + i) * BQ;
      if (padding != nullptr && __ldg(padding + q0 / BKV) > 0) {  // dK and dV: as above
        uint8_t* sQ = sRing + st * 2 * QTILE;
        zero_padded_rows(sQ, QATOM, BQ, q0, args.S, spans);
        zero_padded_rows(sQ + QTILE, QATOM, BQ, q0, args.S, spans);
        fence_proxy_async_smem();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full[st]);
      if (++i == per_head) { i = 0; ++h; }
      if (it + 1 < n_it) fetch();
      if (++st == STAGES) { st = 0; ph ^= 1; }
    }
  } else if (warp == 21) {
    // the gradients of a step.  (One thread for all MMAs spent its time waiting for the products in front of the next ones: 2750 cycles a step.)
    if (n_it > 0 && elect_one()) {
      const uint32_t id_g = umma_idesc_bf16(128, HD, 0, 1);    // dV, dK: A from TMEM (K = queries), dO / Q MN-major
      const uint32_t id_q = umma_idesc_bf16(128, BQ, 1, 1);    // dQ^T: K tile MN-major (M = head dim), dS^T MN-major
      const uint64_t mK = umma_smem_desc_sw128(smem_u32(sK), ATOM, 1024);
      const uint64_t mQ = umma_smem_desc_sw128(smem_u32(sRing), QATOM, 1024);
      const uint64_t mS = umma_smem_desc_sw128(smem_u32(sdS), ATOM, 1024);
      // descriptor addresses advance in units of 16 bytes
      for (int it = 0, st = 0; it < n_it; ++it) {
        const int p = it & 1;
        if (!mbar_wait(&pds_ready[p], (it >> 1) & 1, 514)) break;
        tc_fence_after();
        const uint32_t t = tmem_base + p * 128;
        const uint64_t ds = mS + (uint32_t)(p * (DS_BYTES >> 4));
#pragma unroll
        for (int e = 0; e < BKV / 16; ++e)  // dQ^T first: the dQ warps fetch it under dV and dK
          tc_mma_bf16(t + 64, mK + e * (2048 >> 4), ds + e * (2048 >> 4), id_q, e != 0);
        tc_commit(&dq_full[p]);
        const uint64_t q = mQ + (uint32_t)(st * (2 * QTILE >> 4));
#pragma unroll
        for (int e = 0; e < BQ / 16; ++e)  // 16 queries: 8 TMEM columns of P^T, 16 rows of dO
          tc_mma_bf16_ts(tdV, t + e * 16, q + ((QTILE + e * 2048) >> 4), id_g, (it | e) != 0);
#pragma unroll
        for (int e = 0; e < BQ / 16; ++e)
          tc_mma_bf16_ts(tdK, t + e * 16 + 8, q + (e * 2048 >> 4), id_g, (it | e) != 0);
        tc_commit(&vk_done[p]);
        tc_commit(&q_empty[st]);
        if (++st == STAGES) st = 0;
        if (it + 1 == n_it) tc_commit(all_done);
      }
    }
  } else if (warp == 22) {
    // S^T and dP^T of a step into its set: S^T once dV and dK of two steps before have read P^T and dS^T there, dP^T once the dQ warps have
    // read dQ^T
    if (n_it > 0 && elect_one()) {
      const uint32_t id_s = umma_idesc_bf16(128, BQ, 0, 0);    // both operands K-major (K = head dim)
      const uint64_t kK = umma_smem_desc_sw128(smem_u32(sK), 0, 1024), kV = umma_smem_desc_sw128(smem_u32(sV), 0, 1024);
      const uint64_t kQ = umma_smem_desc_sw128(smem_u32(sRing), 0, 1024);
      bool alive = mbar_wait(kv_full, 0, 510);
      for (int it = 0, st = 0, ph = 0; it < n_it && alive; ++it) {
        const int p = it & 1, par = ((it >> 1) & 1) ^ 1;  // parity of step it - 2
        if (!mbar_wait(&q_full[st], ph, 511) || (it >= 2 && !mbar_wait(&vk_done[p], par, 512))) break;
        tc_fence_after();
        const uint64_t q = kQ + (uint32_t)(st * (2 * QTILE >> 4));
        const uint32_t t = tmem_base + p * 128;
#pragma unroll
        for (int e = 0; e < HD / 16; ++e)
          tc_mma_bf16(t, kK + (((e >> 2) * ATOM + (e & 3) * 32) >> 4), q + (((e >> 2) * QATOM + (e & 3) * 32) >> 4), id_s, e != 0);
        if (it >= 2 && !mbar_wait(&dq_read[p], par, 513)) break;
        tc_fence_after();
#pragma unroll
        for (int e = 0; e < HD / 16; ++e)
          tc_mma_bf16(t + 64, kV + (((e >> 2) * ATOM + (e & 3) * 32) >> 4), q + ((QTILE + (e >> 2) * QATOM + (e & 3) * 32) >> 4), id_s, e != 0);
        tc_commit(&sdp_full[p]);
        if (++st == STAGES) { st = 0; ph ^= 1; }
      }
    }
  } else if (warp < 16) {
    const int p = warp >> 3;                  // even or odd steps
    const int half = (warp >> 2) & 1;         // of the step's queries
    const int row = (warp & 3) * 32 + lane;   // key inside the tile == TMEM lane
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t t = tmem_base + lane_off + p * 128 + half * 32;
    const int key = kv0 + row;
    const float sl2 = args.scale_log2;
    uint8_t* ds_row = sdS + p * DS_BYTES + row * 128;
    int2 span = make_int2(key, args.S);       // queries [x, y) that see this key
    if (spans != nullptr || key >= args.S) {
      span = key < args.S ? __ldg(spans + key) : make_int2(0, 0);
      span = make_int2(max(span.x, 0), min(span.y, args.S));  // ranges put together by hand may reach beyond the row
    }
    const float cap_sq = (MODS & MOD_CAP) ? -1.f / (args.mods.cap_log2 * args.mods.cap_log2) : 0.f;
    int h = h0 + (n_it == 0 ? 0 : p / per_head);
    bool alive = true;
    int st = p, ph = 0, i = n_it == 0 ? 0 : p % per_head;  // ring stage and its parity, query tile of step p
    for (int it = p; it < n_it; it += 2) {
      const int q0 = (i_start + i) * BQ + half * 32;
      // a bounded wait that runs out ends the warp's work (the lanes decide together: TMEM accesses are warp-wide)
      if (!__all_sync(0xffffffffu, mbar_wait(&q_full[st], ph, 520) && mbar_wait(&sdp_full[p], (it >> 1) & 1, 521))) { alive = false; break; }
      tc_fence_after();
      const float4* stat = reinterpret_cast<const float4*>(sStat + st * STAT_FLOATS) + half * 8;
      // the queries of the 32 that see this key
      const bool any_hidden = __any_sync(0xffffffffu, q0 < span.x || q0 + 32 > span.y);
      uint32_t seen = bit_range(span.x - q0, span.y - q0);
      const float slope = (MODS & MOD_BIAS) ? __ldg(args.mods.slopes + h) * LOG2E : 0.f;
      // 16 queries at a time, so that everything stays in registers: a spill goes to the L2, as shared memory leaves no L1
#pragma unroll 1
      for (int c = 0; c < 2; ++c, seen >>= 16) {
        uint32_t s[16], dp[16], pk[8], dk[8];
        tmem_ld16(t + c * 16, s);
        tmem_ld16(t + 64 + c * 16, dp);
        tmem_ld_wait();
        if (MODS & MOD_CAP) cap_scores(s, args.mods);
        const uint64_t one = f32x2(1.f, 1.f), cap2 = f32x2(cap_sq, cap_sq);
        uint64_t slopes2[8];  // 1 - tanh^2
        if (MODS & MOD_CAP) {
#pragma unroll
          for (int v = 0; v < 8; ++v) {
            const uint64_t y = f32x2(__uint_as_float(s[2 * v]), __uint_as_float(s[2 * v + 1]));
            slopes2[v] = fma_f32x2(mul_f32x2(y, y), cap2, one);
          }
        }
        if (MODS & MOD_BIAS) add_bias(s, (MODS & MOD_CAP) ? 1.f : sl2, slope, (float)(q0 + c * 16 - key), span.x < key ? 0 : 1);
        const float m = (MODS & (MOD_CAP | MOD_BIAS)) ? 1.f : sl2;
        const uint64_t m2 = f32x2(m, m);
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const float4 nl = stat[c * 4 + v], nd = stat[BQ / 4 + c * 4 + v];
          float x[4], g[4];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint64_t n2 = e == 0 ? f32x2(nl.x, nl.y) : f32x2(nl.z, nl.w), d2 = e == 0 ? f32x2(nd.x, nd.y) : f32x2(nd.z, nd.w);
            const int at = 4 * v + 2 * e;
            const float2 y = f32x2_split(fma_f32x2(f32x2(__uint_as_float(s[at]), __uint_as_float(s[at + 1])), m2, n2));
            x[2 * e] = fast_exp2(y.x);
            x[2 * e + 1] = fast_exp2(y.y);
            uint64_t z = mul_f32x2(add_f32x2(f32x2(__uint_as_float(dp[at]), __uint_as_float(dp[at + 1])), d2), f32x2(x[2 * e], x[2 * e + 1]));
            if (MODS & MOD_CAP) z = mul_f32x2(z, slopes2[2 * v + e]);
            const float2 w = f32x2_split(z);
            g[2 * e] = w.x;
            g[2 * e + 1] = w.y;
          }
          if (any_hidden) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (!((seen >> (4 * v + e)) & 1u)) x[e] = g[e] = 0.f;
          }
          pk[2 * v] = pack_bf16x2(x[0], x[1]);
          pk[2 * v + 1] = pack_bf16x2(x[2], x[3]);
          dk[2 * v] = pack_bf16x2(g[0], g[1]);
          dk[2 * v + 1] = pack_bf16x2(g[2], g[3]);
        }
        // over the part of S^T that this thread has read: P^T, then dS^T
        tmem_st8(t + c * 16, pk);
        tmem_st8(t + c * 16 + 8, dk);
#pragma unroll
        for (int v = 0; v < 2; ++v)
          *reinterpret_cast<uint4*>(ds_row + (((half * 4 + c * 2 + v) ^ (row & 7)) << 4)) = make_uint4(dk[4 * v], dk[4 * v + 1], dk[4 * v + 2], dk[4 * v + 3]);
      }
      tmem_st_wait();
      fence_proxy_async_smem();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&pds_ready[p]);
      i += 2;
      while (i >= per_head) { i -= per_head; ++h; }
      st += 2;
      if (st >= STAGES) { st -= STAGES; ph ^= 1; }
    }
    // The results: the even steps' warps write dV, the odd steps' warps dK (TMEM lane == key), 64 head dims each.  They go out through the ring
    // and TMA, which leaves out the rows past the end; with parts of a key tile straight to their place.  Nothing but padding: zeros.
    alive = n_it == 0 || (alive && __all_sync(0xffffffffu, mbar_wait(all_done, 0, 522)));
    if (alive) {
      tc_fence_after();
      const uint32_t src = (p == 0 ? tdV : tdK) + lane_off + half * 64;
      const float f = p == 0 ? 1.f : args.scale;
      // a key that only one query sees, which sees nothing else
      bool alone = false;
      if (p == 1 && span.y - span.x == 1) alone = sees_one_key(args.query_spans, (long long)b * args.S + span.x, span.x, args.S);
      uint8_t* stage = sRing + p * 2 * QTILE + half * ATOM + (warp & 3) * 32 * 128;
#pragma unroll 1
      for (int c = 0; c < 2; ++c) {
        uint32_t r[32];
        if (n_it > 0) {
          tmem_ld32(src + c * 32, r);
          tmem_ld_wait();
        }
        if (n_it == 0 || alone) {
#pragma unroll
          for (int e = 0; e < 32; ++e) r[e] = 0u;
        }
        if (args.dkv_parts != nullptr) {
          if (key < args.S) {
            float4* dst = args.dkv_parts + part_tile(part, args.B, b, n_kt, jt, args.Hkv, hk, p == 0 ? 1 : 0) + row + (half * 16 + c * 8) * BKV;
#pragma unroll
            for (int v = 0; v < 8; ++v)
              dst[v * BKV] = make_float4(__uint_as_float(r[4 * v]), __uint_as_float(r[4 * v + 1]), __uint_as_float(r[4 * v + 2]), __uint_as_float(r[4 * v + 3]));
          }
        } else {
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            uint4 w;
            w.x = pack_bf16x2(__uint_as_float(r[8 * v + 0]) * f, __uint_as_float(r[8 * v + 1]) * f);
            w.y = pack_bf16x2(__uint_as_float(r[8 * v + 2]) * f, __uint_as_float(r[8 * v + 3]) * f);
            w.z = pack_bf16x2(__uint_as_float(r[8 * v + 4]) * f, __uint_as_float(r[8 * v + 5]) * f);
            w.w = pack_bf16x2(__uint_as_float(r[8 * v + 6]) * f, __uint_as_float(r[8 * v + 7]) * f);
            *reinterpret_cast<uint4*>(stage + lane * 128 + (((c * 4 + v) ^ (lane & 7)) << 4)) = w;
          }
        }
      }
      if (args.dkv_parts == nullptr) {
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          tma_store_3d(p == 0 ? &tma_dv : &tma_dk, stage, hk * HD + half * 64, kv0 + (warp & 3) * 32, b);
          tma_store_commit();
          tma_store_wait_read0();  // the rest of the way is not this block's
        }
      }
    }
    tc_fence_before();
  } else if (warp < 20) {
    const int w = warp & 3;                   // head dims [32 w, +32) == TMEM lanes
    float* stg = reinterpret_cast<float*>(sdQ) + w * (BQ * 32);
    int h = h0, i = 0;
    for (int it = 0; it < n_it; ++it) {
      const int p = it & 1;
      if (!__all_sync(0xffffffffu, mbar_wait(&dq_full[p], (it >> 1) & 1, 530))) break;
      tc_fence_after();
      const uint32_t t = tmem_base + ((uint32_t)(w * 32) << 16) + p * 128 + 64;
      if (lane == 0) tma_store_wait_read0();  // the reduce of the step before has finished reading the block
      __syncwarp();
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t r[32];
        tmem_ld32(t + c * 32, r);
        tmem_ld_wait();
        if (c == 1) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&dq_read[p]);
        }
#pragma unroll
        for (int e = 0; e < 32; ++e) stg[(c * 32 + e) * 32 + lane] = __uint_as_float(r[e]);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        // rows past the end of the sequence are clipped by the tensor map
        tma_reduce_add_3d(&tma_dq, stg, h * HD + w * 32, (i_start + i) * BQ, b);
        tma_store_commit();
      }
      if (++i == per_head) { i = 0; ++h; }
    }
    if (lane == 0) tma_store_wait_read0();
    tc_fence_before();
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 21) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

struct Maps {
  const CUtensorMap *q, *k, *v, *d_o, *dq, *dk, *dv;
};
template <int MODS>
int launch(const Maps& m, const BwdArgs& a, int grid, cudaStream_t st) {
  static bool optin[64] = {};  // the shared-memory opt-in is a per-device attribute
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -1;
  if (!optin[dev]) {
    cudaError_t e = cudaFuncSetAttribute(attn_mods_bwd_kernel<MODS>, cudaFuncAttributeMaxDynamicSharedMemorySize, BWD_SMEM);
    if (e != cudaSuccess) return -(int)e;
    optin[dev] = true;
  }
  attn_mods_bwd_kernel<MODS><<<grid, BWD_THREADS, BWD_SMEM, st>>>(*m.q, *m.k, *m.v, *m.d_o, *m.dq, *m.dk, *m.dv, a);
  return -(int)cudaGetLastError();
}

int capped_blocks(long long threads) {
  const long long blocks = (threads + 255) / 256, cap = (long long)yf_num_sms() * 8;
  return (int)(blocks < cap ? blocks : cap);
}

}  // namespace

// Backward of yf_attn_fwd_mods: spans, key_spans and padding as yf_document_mask gives them (all null: causal), out_lo as the forward pass left it,
// or null.  Scratch, results and head_parts as in yf_attn_bwd_parts.
extern "C" int yf_attn_bwd_mods(const void* q, const void* k, const void* v, const void* out, const void* out_lo, const void* dout, const float* lse,
                                float* delta, float* dq_accum, float* dkv_parts, long long dkv_floats, int head_parts, void* dq, void* dk, void* dv,
                                int B, int S, int Hq, int Hkv, long long q_stride, long long k_stride, long long v_stride, long long o_stride,
                                long long do_stride, long long dq_stride, long long dkv_stride, float scale, float softcap, const float* slopes,
                                const int* spans, const int* key_spans, const int* padding, void* stream) {
  if (B <= 0 || S <= 0 || Hq <= 0 || Hkv <= 0 || (Hq % Hkv)) return -1;
  if (!(softcap >= 0.f) || !(scale > 0.f) || (key_spans != nullptr) != (padding != nullptr) || (key_spans != nullptr) != (spans != nullptr)) return -1;
  if ((reinterpret_cast<uintptr_t>(key_spans) | reinterpret_cast<uintptr_t>(spans)) & 7) return -1;
  if (head_parts < 1 || (Hq / Hkv) % head_parts || (head_parts > 1) != (dkv_parts != nullptr)) return -1;
  const int n_kt = (S + BKV - 1) / BKV;
  if (dkv_parts != nullptr && dkv_floats < 4 * part_tile(head_parts, B, 0, n_kt, 0, Hkv, 0, 0)) return -1;
  if ((q_stride % 8) || (k_stride % 8) || (v_stride % 8) || (o_stride % 8) || (do_stride % 8) || (dq_stride % 8) || (dkv_stride % 8)) return -1;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(out) |
       reinterpret_cast<uintptr_t>(out_lo) | reinterpret_cast<uintptr_t>(dout) | reinterpret_cast<uintptr_t>(dq) | reinterpret_cast<uintptr_t>(dk) |
       reinterpret_cast<uintptr_t>(dv) | reinterpret_cast<uintptr_t>(dq_accum) | reinterpret_cast<uintptr_t>(dkv_parts)) & 15)
    return -1;
  const long long ctas = (long long)n_kt * B * Hkv * head_parts, T = (long long)B * S;
  if (ctas > 0x7fffffffll) return -1;
  const uint64_t wq = (uint64_t)Hq * HD, wk = (uint64_t)Hkv * HD;
  Maps m;
  m.q = yf_tensor_map_3d(q, wq, S, B, q_stride, (uint64_t)S * q_stride, 64, BQ, 1, 2, 1);
  m.k = yf_tensor_map_3d(k, wk, S, B, k_stride, (uint64_t)S * k_stride, 64, BKV, 1, 2, 1);
  m.v = yf_tensor_map_3d(v, wk, S, B, v_stride, (uint64_t)S * v_stride, 64, BKV, 1, 2, 1);
  m.d_o = yf_tensor_map_3d(dout, wq, S, B, do_stride, (uint64_t)S * do_stride, 64, BQ, 1, 2, 1);
  m.dq = yf_tensor_map_3d(dq_accum, wq, S, B, wq, (uint64_t)S * wq, 32, BQ, 1, 4, 0);
  m.dk = yf_tensor_map_3d(dk, wk, S, B, dkv_stride, (uint64_t)S * dkv_stride, 64, 32, 1, 2, 1);
  m.dv = yf_tensor_map_3d(dv, wk, S, B, dkv_stride, (uint64_t)S * dkv_stride, 64, 32, 1, 2, 1);
  if (!m.q || !m.k || !m.v || !m.d_o || !m.dq || !m.dk || !m.dv) return -2;
  if (int rc = yf_tu_bind_status()) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  BwdArgs a;
  a.lse = lse;
  a.delta = delta;
  a.dkv_parts = reinterpret_cast<float4*>(dkv_parts);
  a.S = S; a.B = B; a.Hq = Hq; a.Hkv = Hkv;
  a.head_parts = head_parts;
  a.head_group = head_group_size(n_kt, B * Hkv * head_parts, T * Hq * HD * 4, yf_num_sms());  // the dQ accumulator
  a.scale = scale;
  a.scale_log2 = scale * LOG2E;
  a.query_spans = reinterpret_cast<const int2*>(spans);
  a.mods = attn_mods(scale, softcap, slopes, key_spans, padding);
  // D, and the dQ accumulator cleared on the way
  const auto pre = out_lo != nullptr ? attn_delta_kernel<true> : attn_delta_kernel<false>;
  pre<<<capped_blocks(T * Hq * 16), 256, 0, st>>>(reinterpret_cast<const __nv_bfloat16*>(out), reinterpret_cast<const __nv_bfloat16*>(out_lo),
                                                  reinterpret_cast<const __nv_bfloat16*>(dout), delta, dq_accum, B, S, Hq, o_stride, do_stride);
  const auto main = softcap > 0.f ? (slopes != nullptr ? launch<MOD_CAP | MOD_BIAS> : launch<MOD_CAP>)
                                  : (slopes != nullptr ? launch<MOD_BIAS> : launch<0>);
  if (int rc = main(m, a, (int)ctas, st)) return rc;
  const long long items = T * Hq * 8 + (dkv_parts ? (long long)B * n_kt * Hkv * 2 * BKV * 8 : 0);
  attn_convert_kernel<true><<<capped_blocks(items), 256, 0, st>>>(dq_accum, a.dkv_parts, head_parts, nullptr, reinterpret_cast<__nv_bfloat16*>(dq),
                                                            reinterpret_cast<__nv_bfloat16*>(dk), reinterpret_cast<__nv_bfloat16*>(dv), B, S, Hq, Hkv,
                                                            dq_stride, dkv_stride, scale, a.query_spans);
  return -(int)cudaGetLastError();
}
