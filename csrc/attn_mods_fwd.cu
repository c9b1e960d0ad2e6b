// Flash-attention forward for head_dim 128 on sm_100a (MHA and GQA) with ranges of keys for every query, capped scores and a distance
// bias (attn_mods.cuh).
//
// A piece of work is (256 query rows, query head, sequence) as two tiles of 128 rows (one tile where every piece then still finds an SM of its own).
// A tile walks over the half blocks of 64 keys between its first row's first key and its last row's last one.  Every piece has a block in the
// grid, the long causal ones first, but a block that has issued its last loads claims the next one that has not started: over packed documents
// a piece has a few half blocks only, and a block's start and end (some 5000 cycles with no MMA) cost as much as they do.  Roles:
//   warp 0        producer: claims pieces; TMA of Q through three places, K and V in tiles of 128 keys through two stages each; clears the padded rows
//                 of V tiles that have some
//   warp 1        MMA: O += P V, half block by half block, the tiles in turn
//   warps 18, 19  MMA: S = Q K^T, one warp for each tile, half block by half block
//   warps 2-9     softmax of tile 0, warps 10-17 of tile 1: two threads per query row (TMEM lane == row), 32 keys of a half block each
// A tile's output leaves through the place of its Q, which is why there are three: the next piece's first tile has its Q, and S, while this one's goes out.
// TMEM (512 columns): S_0, S_1, O_0, O_1, 128 columns of fp32 each.  S_i is two halves of 64 columns which take turns; a thread's P (bf16, 16 columns)
// takes the place of half of the S that it has read into registers, and is the MMA's A operand from there, under the softmax of the other half.
// The exponent's reference maximum is only moved when some row of a warp has grown by more than 2^40 since it was set (then its pair of
// warps rescales its rows of O in TMEM and their sums); the final division by the row sum makes the result exact again.  A row's bits depend
// on the 32 rows that share its warps.
// Bound: per 64 keys of two tiles the products take 1280 cycles (an MMA of 16 x 128 rows 48 at N = 64 and 64 at N = 128), the exponentials 1024, on
// different pipes; about 2100 pass.  A softmax warp spends 600 to 1000 of its 2000 on exponentials and the rest on latencies (S out of TMEM 350,
// the maximum 150, the pair's barrier 240, P into TMEM and the next S 400), and the four of an SM partition tend to do either together.  What was tried:
// S for 128 keys at once, 1024 cycles of products (599 us at the sizes below, where halves took 515: its next S waits for the whole P); one thread that
// issues for both tiles (643); a warp for 64 keys, the two of a row in turn (562: S waits for a longer softmax); the tiles' exponentials in turn (540); the
// exponentials before it is known whether a row has grown (511, packed 144: they are taken twice too often).
// bf16, 32 heads, causal, 1 x 8192: 502 us, 1095 TFLOP/s; in packed documents of 5 to 8000 tokens 135 us, 155 with a block for each piece; scores
// capped 672 us.  64 heads, 2 x 4096 with prefixes and a distance bias 757 us.
#include "attn_mods.cuh"
#include "common.cuh"
#include "yafsdp_b200.h"

YF_TU_STATUS()

namespace {

constexpr int HD = 128;        // head dim
constexpr int BQ = 128;        // query rows per tile
constexpr int BKV = 128;       // keys per tile of K and V
constexpr int HKV = 64;        // keys per half block
constexpr int ATOM = 16384;    // bytes of one [128 rows x 64 bf16] swizzled block
constexpr int TILE = 2 * ATOM; // one 128x128 bf16 tile
constexpr int FWD_THREADS = 640;  // producer warp, three MMA warps, sixteen softmax warps
constexpr int QST = 3, KST = 2, VST = 2;  // tiles of Q, stages of K and V
constexpr int FWD_SMEM = (QST + KST + VST) * TILE + 2 * 2 * BQ * 4 /*between the threads of a row*/ + 384;
static_assert(FWD_SMEM <= 232448, "shared memory of one CTA");
constexpr float LOG2E = 1.4426950408889634f;

struct FwdArgs {
  __nv_bfloat16* out;
  float* lse;
  long long out_stride;  // elements between token rows of out
  int S, B, Hq, Hkv;
  float scale_log2;      // softmax scale * log2(e)
  float scale;
  int tiles;             // query tiles per piece of work: two, or one where even so every piece finds an SM of its own
  int more;              // whether there are more pieces than SMs
  AttnMods mods;
};

template <int MODS>
__global__ void __launch_bounds__(FWD_THREADS, 1)
attn_mods_fwd_kernel(const __grid_constant__ CUtensorMap tma_q, const __grid_constant__ CUtensorMap tma_k,
                     const __grid_constant__ CUtensorMap tma_v, const __grid_constant__ CUtensorMap tma_o,
                     const __grid_constant__ CUtensorMap tma_lo, FwdArgs args) {
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* sQ = smem;                   // stage s at + s * TILE, as the next two
  uint8_t* sK = sQ + QST * TILE;
  uint8_t* sV = sK + KST * TILE;
  float* sRow = reinterpret_cast<float*>(sV + VST * TILE);  // [tile][thread of the row][row]
  uint64_t* bars = reinterpret_cast<uint64_t*>(sRow + 2 * 2 * BQ);
  uint64_t* q_full = bars;              // [QST] per stage
  uint64_t* q_empty = q_full + QST;
  uint64_t* k_full = q_empty + QST;     // [KST]
  uint64_t* k_empty = k_full + KST;
  uint64_t* v_full = k_empty + KST;     // [VST]
  uint64_t* v_empty = v_full + VST;
  uint64_t* s_full = v_empty + VST;     // [2][2] per tile and half, as the next two
  uint64_t* p_ready = s_full + 4;
  uint64_t* o_done = p_ready + 4;
  uint64_t* v_land = o_done + 4;        // a V tile with padded rows has landed, to be cleared before it counts as full
  uint64_t* work_full = v_land + 1;    // [2] per slot of `work`
  uint64_t* work_empty = work_full + 2;
  uint64_t* claimed = work_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(claimed + 1);
  // [2][4] per tile and pair of warps: 1 + the half block at which one of them has given up
  volatile int* dead = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int4* claim = reinterpret_cast<int4*>((reinterpret_cast<uintptr_t>(tmem_slot + 9) + 15) & ~(uintptr_t)15);
  // [2][2] {a piece's query tile, head, sequence, q_places() or 0: no piece}, {its half blocks [x, y), [z, w) of the two tiles}
  int4* work = claim + 1;
  // nothing but this array is in shared memory, so it starts on the boundary that the swizzled tiles need
  if ((smem_u32(smem) & 1023) != 0) {
    if (threadIdx.x == 0) yf_raise(YF_ERR_BAD_ARGUMENT, 430);
    return;
  }

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int n_tiles_kv = (args.S + BKV - 1) / BKV;
  const int kv_heads_div = args.Hq / args.Hkv;
  auto load = [&](uint8_t* dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int b) {
    mbar_expect_tx(bar, TILE);
    tma_load_3d(dst, map, bar, x, y, b);
    tma_load_3d(dst + ATOM, map, bar, x + 64, y, b);
  };
  // whether the work that starts at q0 has a second tile
  auto two = [&](int q0) { return args.tiles == 2 && q0 + BQ < args.S; };
  // half blocks [x, y) and [z, w) of the piece's two tiles; 0, 0 when the sequence ends before, for nothing but padding, or without a second tile
  auto ranges = [&](int q0, int b) {
    int from[2], to[2];
    if (args.mods.spans == nullptr) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        from[i] = 0;
        to[i] = (min(q0 + (i + 1) * BQ, args.S) + HKV - 1) / HKV;
      }
    } else {
      const int2* spans = args.mods.spans + (long long)b * args.S;
      const int* padding = args.mods.padding + (long long)b * n_tiles_kv;
      int2 a[2], z[2];
      int dead_rows[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {  // all loads at once: a row past the end stands for one in front of it
        const int row0 = min(q0 + i * BQ, args.S - 1);
        a[i] = __ldg(spans + row0);
        z[i] = __ldg(spans + min(row0 + BQ - 1, args.S - 1));
        dead_rows[i] = __ldg(padding + row0 / BQ);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        from[i] = max(a[i].x, 0) / HKV;
        to[i] = dead_rows[i] >= min(BQ, args.S - q0 - i * BQ) ? 0 : (min(z[i].y, args.S) + HKV - 1) / HKV;
      }
    }
    if (!two(q0)) to[1] = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (from[i] >= to[i]) from[i] = to[i] = 0;
    return make_int4(from[0], to[0], from[1], to[1]);
  };
  // the query position is the slowest index: under the causal mask the long rows of all heads start first
  auto piece_tile = [&](int z) { return (int)gridDim.z - 1 - z; };
  // The tiles of Q that a launch's blocks load, in their order: place m is stage m % 3, for the (m / 3)-th time.  For a piece in a byte for each tile:
  // stage, parity of the time, whether it is loaded; `m` counts on (from 0 again at 6).
  auto q_places = [&](int m, bool load0, bool load1) {
    int w = 128;
    if (load0) { w |= (m % QST) | (m / QST) << 2 | 8; m = m == 2 * QST - 1 ? 0 : m + 1; }
    w |= load1 ? ((m % QST) | (m / QST) << 2 | 8) << 8 : 0;
    return w;
  };
  auto q_stage = [&](int w, int i) { return (w >> (8 * i)) & 3; };
  auto q_phase = [&](int w, int i) { return (w >> (8 * i + 2)) & 1; };
  auto q_loaded = [&](int w, int i) { return ((w >> (8 * i + 3)) & 1) != 0; };
  if (threadIdx.x == 0) {
    for (int s = 0; s < QST; ++s) mbar_init(&q_full[s], 1);
    mbar_fence_init();
    // Q does not depend on the ranges, whose loads take as long
    const int qt = piece_tile((int)blockIdx.z), q0 = qt * args.tiles * BQ, h = (int)blockIdx.x, b = (int)blockIdx.y;
    load(sQ, &tma_q, &q_full[0], h * HD, q0, b);
    if (two(q0)) load(sQ + TILE, &tma_q, &q_full[1], h * HD, q0 + BQ, b);
    tma_prefetch_desc(&tma_k);
    tma_prefetch_desc(&tma_v);
    tma_prefetch_desc(&tma_o);
    work[0] = make_int4(qt, h, b, q_places(0, true, two(q0)));
    work[1] = ranges(q0, b);
  }
  if (threadIdx.x == 64) {
    for (int s = 0; s < KST; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 2);  // one arrival for each tile
    }
    for (int s = 0; s < VST; ++s) {
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    for (int s = 0; s < QST; ++s) mbar_init(&q_empty[s], 8);  // one arrival per softmax warp of the tile, as for p_ready
    for (int s = 0; s < 4; ++s) {
      mbar_init(&s_full[s], 1);
      mbar_init(&p_ready[s], 8);
      mbar_init(&o_done[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&work_full[s], 1);
      mbar_init(&work_empty[s], 19);  // the warps but the producer's
    }
    mbar_init(v_land, 1);
    mbar_init(claimed, 1);
    for (int s = 0; s < 8; ++s) dead[s] = 0;
    mbar_fence_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  // The roles but the producer: wait until piece number n (or that there is none) stands in its slot of `work`
  auto piece_there = [&](int n) { return n == 0 || (args.more && mbar_wait(&work_full[n & 1], ((n - 1) >> 1) & 1, 404)); };
  int4 piece, range;
  auto next_piece = [&](int n) {
    if (!piece_there(n)) return false;
    piece = work[(n & 1) * 2];
    range = work[(n & 1) * 2 + 1];
    mbar_arrive(&work_empty[n & 1]);
    return piece.w != 0;
  };
  auto first_block = [&]() { return (range.x < range.y && range.z < range.w ? min(range.x, range.z) : range.x < range.y ? range.x : range.z) >> 1; };
  auto end_block = [&]() { return (max(range.y, range.w) + 1) >> 1; };
  if (warp == 0) {
    // the whole warp, since it clears the padded rows of the V tiles that have some; K of a block comes before V of the block before
    int landed = 0, ks = 0, kp = 1, vs = 0, vp = 1, m = 0;
    piece = work[0];
    range = work[1];
    bool ok = true;
    for (int n = 0; ok; ++n) {
      const int b = piece.z, h = piece.y, kv_x = h / kv_heads_div * HD, q0 = piece.x * args.tiles * BQ;
      const int2* spans = args.mods.spans == nullptr ? nullptr : args.mods.spans + (long long)b * args.S;
      const int* padding = args.mods.spans == nullptr ? nullptr : args.mods.padding + (long long)b * n_tiles_kv;
      const int j_first = first_block(), j_end = end_block();
      const bool has0 = range.x < range.y, has1 = range.z < range.w;
      const int ask = max(j_first, j_end - 2);  // before the last loads, and not earlier: a piece that is claimed waits for this CTA
      bool asked = false;
      auto claim_next = [&]() {
        if (lane == 0) {
          mbar_expect_tx(claimed, 16);
          claim_block(claim, claimed);
        }
        asked = true;
      };
      // Q of the second tile lands where the first tile of the piece before had its own, through which its output leaves
      auto load_q = [&](int i) {
        if (!q_loaded(piece.w, i)) return true;
        const int s = q_stage(piece.w, i);
        if (!mbar_wait(&q_empty[s], q_phase(piece.w, i) ^ 1, 405)) return false;
        load(sQ + s * TILE, &tma_q, &q_full[s], h * HD, q0 + i * BQ, b);
        return true;
      };
      if (args.more && j_first >= j_end) claim_next();
      int dead_rows = padding != nullptr && j_first < j_end ? __ldg(padding + j_first) : 0;
      for (int j = j_first; j <= j_end && j_first < j_end; ++j) {
        if (args.more && j == ask) claim_next();
        if (lane == 0 && j < j_end) {
          ok = ok && mbar_wait(&k_empty[ks], kp, 400);
          if (ok) load(sK + ks * TILE, &tma_k, &k_full[ks], kv_x, j * BKV, b);
          if (++ks == KST) { ks = 0; kp ^= 1; }
          if (n > 0 && j == j_first && ok) ok = load_q(0);
        }
        ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
        if (!ok) break;
        if (j == j_first) continue;
        const bool clear = dead_rows > 0;
        if (padding != nullptr && j < j_end) dead_rows = __ldg(padding + j);
        ok = __all_sync(0xffffffffu, mbar_wait(&v_empty[vs], vp, 401));
        if (!ok) break;
        if (lane == 0) load(sV + vs * TILE, &tma_v, clear ? v_land : &v_full[vs], kv_x, (j - 1) * BKV, b);
        if (clear) {
          ok = __all_sync(0xffffffffu, mbar_wait(v_land, landed & 1, 402));
          if (!ok) break;
          ++landed;
          zero_padded_rows(sV + vs * TILE, ATOM, BKV, (j - 1) * BKV, args.S, spans);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&v_full[vs]);
        }
        if (++vs == VST) { vs = 0; vp ^= 1; }
        if (n > 0 && lane == 0 && j == j_first + 1) ok = load_q(1);
      }
      ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
      // a tile without keys: its Q has to land before the place is used again or the block ends
      if (n == 0 && !has0) mbar_wait(&q_full[0], 0, 403);
      if (n == 0 && !has1 && two(q0)) mbar_wait(&q_full[1], 0, 403);
      m = (m + (q_loaded(piece.w, 0) ? 1 : 0) + (q_loaded(piece.w, 1) ? 1 : 0)) % (2 * QST);
      if (!asked) break;
      const bool answered = __all_sync(0xffffffffu, mbar_wait(claimed, n & 1, 406));
      if (!answered || !ok) break;
      uint3 at;
      const bool got = claimed_block(claim, at);
      fence_proxy_async_smem();  // the next answer is written behind these reads
      __syncwarp();
      piece = range = make_int4(0, 0, 0, 0);
      if (got) {
        piece = make_int4(piece_tile((int)at.z), (int)at.x, (int)at.y, 0);
        range = ranges(piece.x * args.tiles * BQ, piece.z);
        piece.w = q_places(m, range.x < range.y, range.z < range.w);
      }
      if (n > 0) ok = __all_sync(0xffffffffu, mbar_wait(&work_empty[(n + 1) & 1], ((n - 1) >> 1) & 1, 407));
      if (!ok) break;
      if (lane == 0) {
        work[((n + 1) & 1) * 2] = piece;
        work[((n + 1) & 1) * 2 + 1] = range;
        mbar_arrive(&work_full[(n + 1) & 1]);
      }
      if (!got) break;
    }
  } else if (warp == 1) {
    // O += P V, the tiles in turn
    if (elect_one()) {
      const uint32_t idesc_o = umma_idesc_bf16(BQ, HD, 0, 1);    // P from TMEM (K = keys), V MN-major
      const uint64_t dV = umma_smem_desc_sw128(smem_u32(sV), ATOM, 1024);
      int vs = 0, vp = 0;
      uint32_t pp = 0;  // phase of p_ready, a bit for each
      bool alive = true;
      for (int n = 0; alive && next_piece(n); ++n) {
        const int j_end = end_block();
        for (int j = first_block(); j < j_end && alive; ++j) {
          alive = mbar_wait(&v_full[vs], vp, 410);
          if (!alive) break;
#pragma unroll 1
          for (int x = 0; x < 4; ++x) {
            const int i = x & 1, u = x >> 1, t = 2 * j + u, lo = i == 0 ? range.x : range.z, hi = i == 0 ? range.y : range.w;
            if (t < lo || t >= hi) continue;
            if (!mbar_wait(&p_ready[i * 2 + u], (pp >> x) & 1, 411)) { alive = false; break; }
            pp ^= 1u << x;
            tc_fence_after();
            const uint64_t v = dV + (uint32_t)(vs * (TILE >> 4) + u * (HKV * 128 >> 4));
            const uint32_t p = tmem_base + i * 128 + u * HKV;
#pragma unroll
            for (int e = 0; e < HKV / 16; ++e)  // 16 keys: 8 TMEM columns of P, 16 rows of V; two of them a thread
              tc_mma_bf16_ts(tmem_base + 256 + i * 128, p + (e >> 1) * 32 + (e & 1) * 8, v + e * (2048 >> 4), idesc_o, t != lo || e != 0);
            tc_commit(&o_done[i * 2 + u]);
          }
          tc_commit(&v_empty[vs]);
          if (++vs == VST) { vs = 0; vp ^= 1; }
        }
      }
    }
  } else if (warp >= 18) {
    // S = Q K^T, one thread for each tile.  S of half block t goes into the columns that P of t - 2 held: P V of t - 2 is waited for, the order
    // of MMAs with different accumulators is not promised.
    const int i = warp - 18;
    if (elect_one()) {
      const uint32_t idesc_s = umma_idesc_bf16(BQ, HKV, 0, 0);   // Q, K both K-major (K = head dim)
      const uint64_t dQ = umma_smem_desc_sw128(smem_u32(sQ), 0, 1024);
      const uint64_t dK = umma_smem_desc_sw128(smem_u32(sK), 0, 1024);
      int ks = 0, kp = 0;  // stage and phase of the block whose K comes next
      uint32_t op = 3;             // phase of o_done, a bit for each half: the first time nothing is waited for
      auto next_k = [&]() {
        if (++ks == KST) { ks = 0; kp ^= 1; }
      };
      auto pass = [&](int blocks) {  // that only the other tile walks over: passed on as soon as they are there
        for (; blocks > 0; --blocks) {
          if (!mbar_wait(&k_full[ks], kp, 412 + i)) return false;
          mbar_arrive(&k_empty[ks]);
          next_k();
        }
        return true;
      };
      bool alive = true;
      for (int n = 0; alive && next_piece(n); ++n) {
        const int lo = i == 0 ? range.x : range.z, hi = i == 0 ? range.y : range.w, j_first = first_block(), j_end = end_block();
        if (lo < hi) {
          const int place = q_stage(piece.w, i);
          const uint64_t q = dQ + (uint32_t)(place * (TILE >> 4));
          alive = pass((lo >> 1) - j_first) && mbar_wait(&q_full[place], q_phase(piece.w, i), 414 + i);
          for (int t = lo; t < hi && alive; ++t) {
            const int u = t & 1;
            alive = (u != 0 && t != lo) || mbar_wait(&k_full[ks], kp, 416 + i);
            alive = alive && mbar_wait(&o_done[i * 2 + u], (op >> u) & 1, 418 + i);
            if (!alive) break;
            op ^= 1u << u;
            tc_fence_after();
            // descriptor addresses advance in units of 16 bytes; half a tile of K is 64 rows of 128 bytes further on in either column block
            const uint64_t k = dK + (uint32_t)(ks * (TILE >> 4) + u * (HKV * 128 >> 4));
#pragma unroll
            for (int e = 0; e < HD / 16; ++e) {
              const uint32_t off = ((e >> 2) * ATOM + (e & 3) * 32) >> 4;
              tc_mma_bf16(tmem_base + i * 128 + u * HKV, q + off, k + off, idesc_s, e != 0);
            }
            tc_commit(&s_full[i * 2 + u]);
            if (u == 1 || t == hi - 1) {  // the last S of its block
              tc_commit(&k_empty[ks]);
              next_k();
            }
          }
          alive = alive && pass(j_end - ((hi + 1) >> 1));
        } else {
          alive = pass(j_end - j_first);
        }
      }
    }
  } else {
    const int i = (warp - 2) >> 3;           // tile
    const int half = ((warp - 2) >> 2) & 1;  // of a half block's keys, of the columns of O
    const int q = warp & 3;                  // a warp may only touch TMEM lanes [32*(warp%4), +32)
    const int bar = 1 + i * 4 + q;           // barrier of the two warps that share 32 rows
    const uint32_t lane_off = (uint32_t)(q * 32) << 16;
    const uint32_t tS = tmem_base + lane_off + i * 128, tO = tmem_base + lane_off + 256 + i * 128 + half * 64;
    float* mine = sRow + (i * 2 + half) * BQ + q * 32 + lane;
    float* theirs = sRow + (i * 2 + (half ^ 1)) * BQ + q * 32 + lane;
    volatile int* gone = dead + i * 4 + q;
    const float sl2 = args.scale_log2;
    // The reference maximum is moved when a row's maximum exceeds it by 2^40: P, its sums and O in fp32 keep their relative accuracy at any
    // reference, and stay finite for V up to 10^22 over 10^4 keys.  (By 2^8, with the distance bias of the 64 heads 832 instead of 757 us.)
    constexpr float RESCALE_LOG2 = 40.f;
    // scores that were transformed are in units of log2 already
    const float to_log2 = (MODS & (MOD_CAP | MOD_BIAS)) ? 1.f : sl2;
    uint32_t ph = 0;                         // phase of s_full and o_done, a bit for each half
    bool alive = true;
    for (int n = 0;; ++n) {
      // both warps of a pair go on or neither does: they meet at barriers, which have no limit
      alive = __all_sync(0xffffffffu, piece_there(n));
      if (n > 0 && args.more && named_bar_or(bar, 64, !alive)) alive = false;
      const int4* now = work + (n & 1) * 2;
      if (!alive || now[0].w == 0) break;
      const int lo = i == 0 ? now[1].x : now[1].z, hi = i == 0 ? now[1].y : now[1].w;
      const int qrow = now[0].x * args.tiles * BQ + i * BQ + q * 32 + lane;
      float m_run = -INFINITY;                 // reference maximum of the exponent
      float l_run = 0.f;                       // sum over this thread's keys
      float l_off = 0.f;                       // what rounding to bf16 adds to the largest of every 32 keys
      int2 span = make_int2(0, qrow + 1);      // keys [x, y) of this row
      if (args.mods.spans != nullptr || qrow >= args.S) {
        span = qrow < args.S ? __ldg(args.mods.spans + (long long)now[0].z * args.S + qrow) : make_int2(0, 0);
        span = make_int2(max(span.x, 0), min(span.y, args.S));  // ranges put together by hand may reach beyond the row
      }
      const float slope = (MODS & MOD_BIAS) ? args.mods.slopes[now[0].y] * LOG2E : 0.f;
      float top = -INFINITY;                   // exponent of the largest P, of the half block before for a while
      auto add_off = [&]() {  // under the next half block's maximum (causal 520 us, 529 at once)
        const float p = fast_exp2(top);
        l_off += __bfloat162float(__float2bfloat16_rn(p)) - p;
      };
      const bool worked = lo < hi;
      for (int t = lo; t < hi; ++t) {
        const int u = t & 1;
        // a bounded wait that runs out ends the work of the two warps: they meet at the barrier below, so the one that gives up says so there
        // (the lanes of a warp decide together: TMEM accesses are warp-wide)
        alive = alive && __all_sync(0xffffffffu, mbar_wait(&s_full[i * 2 + u], (ph >> u) & 1, 420 + i));
        ph ^= 1u << u;
        const int kv0 = t * HKV + half * 32;
        uint32_t sc[32];
        if (!alive) *gone = t + 1;
        tc_fence_after();
        tmem_ld32(tS + u * HKV + half * 32, sc);  // (of a dead walk too: branches around it cost a move for each score)
        tmem_ld_wait();
        if (MODS & MOD_CAP) cap_scores(sc, args.mods);
        if (MODS & MOD_BIAS) add_bias(sc, (MODS & MOD_CAP) ? 1.f : sl2, slope, (float)(kv0 - qrow), span.y > qrow + 1 ? 0 : -1);
        if (kv0 < span.x || kv0 + 32 > span.y) {  // the ends of a row's range
          const uint32_t seen = bit_range(span.x - kv0, span.y - kv0);
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (!((seen >> e) & 1u)) sc[e] = 0xff800000u;  // -inf
        }
        float mx2[2] = {__uint_as_float(sc[0]), __uint_as_float(sc[1])};
#pragma unroll
        for (int e = 2; e < 30; e += 4) {
          mx2[0] = fmax3(mx2[0], __uint_as_float(sc[e]), __uint_as_float(sc[e + 1]));
          mx2[1] = fmax3(mx2[1], __uint_as_float(sc[e + 2]), __uint_as_float(sc[e + 3]));
        }
        const float mx = fmaxf(fmax3(mx2[0], __uint_as_float(sc[30]), __uint_as_float(sc[31])), mx2[1]);
        add_off();
        const bool grew = !alive || (mx != -INFINITY && (m_run == -INFINITY || (mx - m_run) * to_log2 > RESCALE_LOG2));
        if (named_bar_or(bar, 64, grew)) {
          if (*gone == t + 1) { alive = false; break; }  // not a later half block's: who gives up there waits for this warp there
          *mine = mx;
          named_bar_sync(bar, 64);
          const float m_new = fmaxf(m_run, fmaxf(mx, *theirs));
          if (__any_sync(0xffffffffu, m_run != -INFINITY)) {
            // O holds sums relative to the old maximum: wait for the last P V to land, then scale this warp's part of the rows
            alive = __all_sync(0xffffffffu, mbar_wait(&o_done[i * 2 + (u ^ 1)], ((ph >> (u ^ 1)) & 1) ^ 1, 422 + i));
            if (!alive) continue;  // to the next barrier, where the other warp learns of it
            tc_fence_after();
            const float alpha = (m_run == -INFINITY) ? 0.f : fast_exp2((m_run - m_new) * to_log2);
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
              uint32_t r[16];
              tmem_ld16(tO + c * 16, r);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 16; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) * alpha);
              tmem_st16(tO + c * 16, r);
            }
            l_run *= alpha;
            l_off *= alpha;
          }
          m_run = m_new;
        }
        const float neg_ms = (m_run == -INFINITY) ? 0.f : -m_run * to_log2;
        uint64_t sum = f32x2(0.f, 0.f);
        uint32_t packed[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          // (pairs of products in one instruction cost moves here, 520 us)
          const float2 y = make_float2(fmaf(__uint_as_float(sc[2 * e]), to_log2, neg_ms), fmaf(__uint_as_float(sc[2 * e + 1]), to_log2, neg_ms));
          const float p0 = fast_exp2(y.x), p1 = fast_exp2(y.y);
          sum = add_f32x2(sum, f32x2(p0, p1));
          packed[e] = pack_bf16x2(p0, p1);
        }
        tmem_st16(tS + u * HKV + half * 32, packed);
        top = fmaf(mx, to_log2, neg_ms);
        const float2 two = f32x2_split(sum);
        l_run += two.x + two.y;
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_ready[i * 2 + u]);
      }
      // what the piece is, once more: the loop above has no registers for it
      const int h = now[0].y, b = now[0].z, row0 = qrow - lane;
      const int places = now[0].w;
      if (!worked) {  // nothing but padding, or no tile here: zeros
        if (qrow < args.S && i < args.tiles) {
          const long long at = ((long long)b * args.S + qrow) * args.out_stride + h * HD + half * 64;
#pragma unroll
          for (int v = 0; v < 8; ++v) {
            reinterpret_cast<uint4*>(args.out + at)[v] = make_uint4(0u, 0u, 0u, 0u);
            if (args.mods.out_lo != nullptr) reinterpret_cast<uint4*>(args.mods.out_lo + at)[v] = make_uint4(0u, 0u, 0u, 0u);
          }
          if (half == 0) args.lse[((long long)b * args.Hq + h) * args.S + qrow] = -INFINITY;
        }
      } else {
        // the output of the last half block, and the sum of both threads
        const int u = (hi - 1) & 1;
        alive = alive && __all_sync(0xffffffffu, mbar_wait(&o_done[i * 2 + u], ((ph >> u) & 1) ^ 1, 424 + i));
        add_off();
        *mine = l_run;
        if (named_bar_or(bar, 64, !alive)) alive = false;
        l_run = half == 0 ? l_run + *theirs : *theirs + l_run;
        named_bar_sync(bar, 64);
        *mine = l_off;
        named_bar_sync(bar, 64);
        l_off += *theirs;
      }
      if (worked && alive) {
        tc_fence_after();
        // P V has the rounded P of the largest keys, and so has the sum that it is divided by (0.0021 instead of 0.0023 of O off over documents of
        // some 400 tokens, and one key alone gives exactly its V).  The backward pass works with unrounded P: lse takes their sum.
        const float l = l_run, inv = (l > 0.f) ? 1.f / (l + l_off) : 0.f;
        // The warp's 32 rows x 64 columns go out through the place of Q, which the tile's last product has read, and TMA (which leaves out the
        // rows past the end): a thread's own 16 bytes at a time touch 32 lines with each instruction.
        uint8_t* stage = sQ + q_stage(places, i) * TILE + half * ATOM + q * 32 * 128;
#pragma unroll 1
        for (int low = 0; low < (args.mods.out_lo != nullptr ? 2 : 1); ++low) {  // the output, then what its rounding left over
          if (low != 0) {
            if (lane == 0) tma_store_wait_read0();
            __syncwarp();
          }
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t r[32];
            tmem_ld32(tO + c * 32, r);
            tmem_ld_wait();
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              uint32_t w[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float x = __uint_as_float(r[8 * v + 2 * e]) * inv, y = __uint_as_float(r[8 * v + 2 * e + 1]) * inv;
                w[e] = pack_bf16x2(x, y);
                const float2 z = unpack_bf16x2(w[e]);
                if (low != 0) w[e] = pack_bf16x2(x - z.x, y - z.y);
              }
              *reinterpret_cast<uint4*>(stage + lane * 128 + (((4 * c + v) ^ (lane & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_3d(low != 0 ? &tma_lo : &tma_o, stage, h * HD + half * 64, row0, b);
            tma_store_commit();
          }
        }
        if (half == 0 && qrow < args.S)
          args.lse[((long long)b * args.Hq + h) * args.S + qrow] =
              (l > 0.f) ? (m_run * ((MODS & (MOD_CAP | MOD_BIAS)) ? 0.6931471805599453f : args.scale) + logf(l)) : -INFINITY;
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&work_empty[n & 1]);
        if (q_loaded(places, i)) {
          tma_store_wait_read0();  // the rest of the way is not this block's
          mbar_arrive(&q_empty[q_stage(places, i)]);
        }
      }
      if (!alive) break;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

template <int MODS>
int launch(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const CUtensorMap& mo, const CUtensorMap& ml, const FwdArgs& a,
           cudaStream_t st) {
  static bool optin[64] = {};  // the shared-memory opt-in is a per-device attribute
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -1;
  if (!optin[dev]) {
    cudaError_t e = cudaFuncSetAttribute(attn_mods_fwd_kernel<MODS>, cudaFuncAttributeMaxDynamicSharedMemorySize, FWD_SMEM);
    if (e != cudaSuccess) return -(int)e;
    optin[dev] = true;
  }
  if (int rc = yf_tu_bind_status()) return rc;
  dim3 grid(a.Hq, a.B, (a.S + a.tiles * BQ - 1) / (a.tiles * BQ));
  attn_mods_fwd_kernel<MODS><<<grid, FWD_THREADS, FWD_SMEM, st>>>(mq, mk, mv, mo, ml, a);
  return -(int)cudaGetLastError();
}

}  // namespace

// As yf_attn_fwd, with row pitches of their own for k and v, scores capped at +-softcap (0: not) and less slopes[h] * distance (null: not), keys
// by `spans` and `padding` as yf_document_mask gives them (both null: causal).  Rows without a key: zeros, lse -inf.  out_lo (may be null):
// what the rounding of `out` left over, for the backward pass.
extern "C" int yf_attn_fwd_mods(const void* q, const void* k, const void* v, void* out, void* out_lo, float* lse, int B, int S, int Hq, int Hkv,
                                long long q_stride, long long k_stride, long long v_stride, long long out_stride, float scale, float softcap,
                                const float* slopes, const int* spans, const int* padding, void* stream) {
  if (B <= 0 || B > 65535 || S <= 0 || Hq <= 0 || Hkv <= 0 || (Hq % Hkv) || (q_stride % 8) || (k_stride % 8) || (v_stride % 8) || (out_stride % 8)) return -1;
  if (!(softcap >= 0.f) || !(scale > 0.f) || (spans != nullptr) != (padding != nullptr) || (reinterpret_cast<uintptr_t>(spans) & 7)) return -1;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
       reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(out_lo)) & 15)
    return -1;
  const CUtensorMap* mq = yf_tensor_map_3d(q, (uint64_t)Hq * HD, S, B, q_stride, (uint64_t)S * q_stride, 64, BQ, 1, 2, 1);
  const CUtensorMap* mk = yf_tensor_map_3d(k, (uint64_t)Hkv * HD, S, B, k_stride, (uint64_t)S * k_stride, 64, BKV, 1, 2, 1);
  const CUtensorMap* mv = yf_tensor_map_3d(v, (uint64_t)Hkv * HD, S, B, v_stride, (uint64_t)S * v_stride, 64, BKV, 1, 2, 1);
  const CUtensorMap* mo = yf_tensor_map_3d(out, (uint64_t)Hq * HD, S, B, out_stride, (uint64_t)S * out_stride, 64, 32, 1, 2, 1);
  const CUtensorMap* ml = out_lo == nullptr ? mo : yf_tensor_map_3d(out_lo, (uint64_t)Hq * HD, S, B, out_stride, (uint64_t)S * out_stride, 64, 32, 1, 2, 1);
  if (!mq || !mk || !mv || !mo || !ml) return -2;
  FwdArgs a;
  a.out = reinterpret_cast<__nv_bfloat16*>(out);
  a.lse = lse;
  a.out_stride = out_stride;
  a.S = S; a.B = B; a.Hq = Hq; a.Hkv = Hkv;
  a.scale = scale;
  a.scale_log2 = scale * LOG2E;
  // 1 x 512 tokens, 32 heads 13.0 us with one tile a piece, 15.2 with two; 1 x 777, 16 heads 17.1 and 19.7; 1 x 333, 40 heads 11.4 and 11.1
  a.tiles = (long long)((S + BQ - 1) / BQ) * Hq * B <= yf_num_sms() ? 1 : 2;
  a.more = (long long)((S + BQ * a.tiles - 1) / (BQ * a.tiles)) * Hq * B > yf_num_sms();
  a.mods = attn_mods(scale, softcap, slopes, spans, padding);
  a.mods.out_lo = reinterpret_cast<__nv_bfloat16*>(out_lo);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (softcap > 0.f) return slopes != nullptr ? launch<MOD_CAP | MOD_BIAS>(*mq, *mk, *mv, *mo, *ml, a, st) : launch<MOD_CAP>(*mq, *mk, *mv, *mo, *ml, a, st);
  return slopes != nullptr ? launch<MOD_BIAS>(*mq, *mk, *mv, *mo, *ml, a, st) : launch<0>(*mq, *mk, *mv, *mo, *ml, a, st);
}
