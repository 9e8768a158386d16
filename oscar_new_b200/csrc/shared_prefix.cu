// Decode attention of requests that share a prefix: the INT2 history of the prefix is read,
// dequantised and multiplied once per group of requests instead of once per request.
//
// A group's rows (members x queries x query heads of a KV head) are packed into tiles of
// 128 rows, and one CTA attends a tile to a run of 64-token history tiles of one KV head:
//   packed slots   one 4-D TMA copy per tile (144 of a slot's 160 bytes, 64 tokens of one
//                  head, no multicast) into a 4-stage ring;
//   operands       four warps expand the keys and four the values into bf16 tiles
//                  (128-byte swizzle): a token has only four levels bf16(c * s + z) per
//                  vector, kept in two registers, and one PRMT whose selector nibbles come
//                  from one IMAD fetches two elements.  Bytes hold dims 4i .. 4i + 3, so a
//                  PRMT yields dims (p, 4 + p) or (8 + p, 12 + p): every 16-dim block is
//                  kept transposed (position 4p + i holds dim 4i + p), the query is stored in
//                  the same order and the output is transposed back when it is written;
//   S = Q K^T      tcgen05.mma kind::f16, M = 128 rows, N = 64 tokens, K = 256, with the
//                  queries as the tensor-memory A operand (no shared-memory traffic);
//   softmax        thread = row = TMEM lane, running max re-based lazily, P as bf16 over
//                  its own scores in tensor memory;
//   O += P V       P from tensor memory, V MN-major, M = 128, N = 256, K = 64.
// Tensor memory: O 256 columns, Q 128, S / P 2 x 64.  The range is the same for all rows
// of a group: [sink, end), end = the shortest of the members' prefix lengths and recent
// windows (oscar_prepare_shared_prefix); what lies behind it for a member stays with the
// per-request kernels.  Tokens outside the range get zero levels (their slots may hold
// anything) and -inf scores.  Split partials (normalised O, lse) join the merge of the step.
//
// Every wait is bounded; a wait that gives up sets the status word, the CTA's rows get
// lse = -inf, copies in flight land and issued MMAs complete before tensor memory is freed.
#include <climits>
#include <cstring>

#include "shared_prefix.cuh"
#include "tcgen05.cuh"

namespace oscar {
namespace {

// ----------------------------------------------------------------------------
// plan
// ----------------------------------------------------------------------------
constexpr int kPlanThreads = 1024;
constexpr int kPlanMaxReqs = 8192;
constexpr int kItemCost = 4;  // an item's fixed cost (start, merge of its partial) in tiles

struct PlanParams {
  const int32_t *qstarts, *seq_lens, *counts, *groups, *prefix_lens;
  int32_t *plan;
  int32_t max_reqs, items, splits, sms;
  oscar_geometry geo;
};

OSCAR_DEVINL int warp_sum(int v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// splits of a group of `tiles` tiles at about `span` tiles each
OSCAR_DEVINL int splits_of(int tiles, int span, int most) { return max(1, min(most, (tiles + span - 1) / span)); }

__global__ void __launch_bounds__(kPlanThreads) shared_plan_kernel(const PlanParams P) {
  extern __shared__ int32_t sm[];
  const oscar_geometry &g = P.geo;
  const int nr = min(P.counts[0], P.max_reqs), active = P.counts[1];
  int32_t *s_label = sm, *s_limit = sm + P.max_reqs;          // group label; end of the shareable history
  int32_t *s_rows = sm + 2 * P.max_reqs;                      // group start: row tiles (0: not a start)
  int32_t *s_tiles = sm + 3 * P.max_reqs;                     // group start: history tiles
  __shared__ int32_t s_cost[32], s_span[32], s_total, s_row_tiles, s_scan[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int32_t *ends = P.plan + kSharedHead, *used = ends + (P.max_reqs + 3) / 4 * 4;
  SharedItem *items = reinterpret_cast<SharedItem *>(used + (P.max_reqs + 3) / 4 * 4);
  if (tid == 0) s_total = s_row_tiles = 0;
  for (int r = tid; r < P.max_reqs; r += kPlanThreads) {
    int label = -1, limit = INT_MAX;
    if (r < nr) {
      const int q0 = min(P.qstarts[r], active), q1 = min(P.qstarts[r + 1], active), qlen = q1 - q0;
      label = P.groups[r];
      if (qlen > 0) {
        const int prefix = P.seq_lens[r] - qlen, sink = min(g.sink, prefix);
        limit = min(P.prefix_lens[r], max(sink, prefix - g.recent));
      }
    }
    s_label[r] = label, s_limit[r] = limit, s_rows[r] = 0, s_tiles[r] = 0;
    ends[r] = 0, used[r] = 0;
  }
  __syncthreads();
  // one warp per run of equal labels: its active members, the shortest limit
  for (int r = warp; r < nr; r += 32) {
    const int label = s_label[r];
    if (label < 0 || (r > 0 && s_label[r - 1] == label)) continue;
    int members = 0, leader = INT_MAX, limit = INT_MAX, stop = nr;
    for (int base = r; base < nr; base += 32) {
      const int j = base + lane;
      const bool same = j < nr && s_label[j] == label;
      const uint32_t other = __ballot_sync(0xffffffffu, !same);
      const int run = other ? __ffs(other) - 1 : 32;
      const int lim = lane < run ? s_limit[j] : INT_MAX;
      const bool is_active = lane < run && lim != INT_MAX;
      members += __popc(__ballot_sync(0xffffffffu, is_active));
      limit = min(limit, __reduce_min_sync(0xffffffffu, lim));
      leader = min(leader, __reduce_min_sync(0xffffffffu, is_active ? j : INT_MAX));
      if (run < 32) {
        stop = base + run;
        break;
      }
    }
    const int64_t reach = (int64_t)g.table_stride * kKernelBlock;
    if (limit > reach) limit = (int)reach;
    if (members < 2 || limit <= g.sink) continue;
    const int tok0 = min(P.qstarts[r], active), tok1 = min(P.qstarts[stop], active);
    const int rows = (tok1 - tok0) * g.group;
    for (int j = r + lane; j < stop; j += 32) ends[j] = limit;
    if (lane == 0) {
      s_limit[r] = stop;  // read by this warp alone: from here on the request behind the group
      s_rows[r] = (rows + kSharedRows - 1) / kSharedRows;
      s_tiles[r] = (limit + kSharedTile - 1) / kSharedTile - g.sink / kSharedTile;
      used[r] = leader;  // until the splits are known
    }
  }
  __syncthreads();
  {
    int mine = 0, mine_rows = 0;
    for (int r = tid; r < nr; r += kPlanThreads) mine += s_rows[r] * s_tiles[r], mine_rows += s_rows[r];
    mine = warp_sum(mine), mine_rows = warp_sum(mine_rows);
    if (lane == 0 && mine_rows) atomicAdd(&s_total, mine), atomicAdd(&s_row_tiles, mine_rows);
  }
  __syncthreads();
  const int64_t total = (int64_t)s_total * g.kv_heads;
  if (total == 0 || s_row_tiles > P.items) {  // nothing shared, or more row tiles than the plan holds
    for (int r = tid; r < nr; r += kPlanThreads) ends[r] = 0, used[r] = 0;
    if (tid == 0) P.plan[0] = 0;
    return;
  }
  // 32 candidate spans, one per warp: around one wave of CTAs, then 2 .. 17 waves; the
  // cheapest in (waves x (longest split + fixed cost)) wins, the first among equals
  {
    const int64_t base = max((int64_t)1, (total + P.sms - 1) / P.sms);
    const int64_t want = warp < 16 ? base + base * warp / 16 : (base + warp - 15) / (warp - 14);
    const int span = (int)min((int64_t)1 << 24, max((int64_t)1, want));
    int count = 0, longest = 0;
    for (int r = lane; r < nr; r += 32) {
      if (!s_rows[r]) continue;
      const int k = splits_of(s_tiles[r], span, P.splits);
      count += s_rows[r] * k;
      longest = max(longest, (s_tiles[r] + k - 1) / k);
    }
    count = warp_sum(count);
    longest = __reduce_max_sync(0xffffffffu, longest);
    if (lane == 0) {
      const int64_t waves = ((int64_t)count * g.kv_heads + P.sms - 1) / P.sms;
      const int64_t cost = waves * (longest + kItemCost);
      s_cost[warp] = count > P.items ? INT_MAX : (int)min((int64_t)INT_MAX - 1, cost);
      s_span[warp] = span;
    }
  }
  __syncthreads();
  int span = 1 << 24;  // no candidate fits the item list: one split per row tile
  {
    const int cost = s_cost[lane], best = __reduce_min_sync(0xffffffffu, cost);
    const uint32_t at = __ballot_sync(0xffffffffu, cost == best);
    if (best != INT_MAX) span = s_span[__ffs(at) - 1];
  }
  int done = 0;
  for (int base = 0; base < nr; base += kPlanThreads) {
    const int r = base + tid;
    const int mt = r < nr ? s_rows[r] : 0;
    const int k = mt ? splits_of(s_tiles[r], span, P.splits) : 0;
    int v = mt * k;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    if (lane == 31) s_scan[warp] = v;
    __syncthreads();
    int s = s_scan[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += u;
    }
    const int before = done + (warp ? __shfl_sync(0xffffffffu, s, (warp + 31) & 31) : 0) + v - mt * k;
    done += __shfl_sync(0xffffffffu, s, 31);
    __syncthreads();
    if (r < nr) s_label[r] = before;  // first item of the group that starts here
  }
  __syncthreads();
  for (int r = warp; r < nr; r += 32) {
    const int mt = s_rows[r];
    if (!mt) continue;
    const int tiles = s_tiles[r], k = splits_of(tiles, span, P.splits), first = s_label[r], stop = s_limit[r];
    const int leader = used[r], end = ends[r];
    const int tok0 = min(P.qstarts[r], active), rows = (min(P.qstarts[stop], active) - tok0) * g.group;
    const int tile0 = g.sink / kSharedTile;
    for (int i = lane; i < mt * k; i += 32) {
      const int m = i / k, s = i % k;
      SharedItem it;
      it.tok0 = tok0, it.row0 = m * kSharedRows, it.rows = min(kSharedRows, rows - m * kSharedRows);
      it.leader = leader, it.end = end, it.slot = s;
      it.tile0 = tile0 + (int)((int64_t)tiles * s / k);
      it.tile1 = tile0 + (int)((int64_t)tiles * (s + 1) / k);
      items[first + i] = it;
    }
    __syncwarp();
    for (int j = r + lane; j < stop; j += 32) used[j] = k;
  }
  if (tid == 0) P.plan[0] = done;
}

// ----------------------------------------------------------------------------
// attention
// ----------------------------------------------------------------------------
constexpr int kSpPacked = 144;                           // bytes of a slot that are copied
constexpr int kSpStageBytes = kSharedTile * kSpPacked;   // 9 KiB
constexpr int kSpStages = 4;
constexpr int kSpTileBytes = kSharedTile * kDim * 2;     // 32 KiB: 4 boxes of [64 tokens][64 dims]
constexpr int kSpBox = kSpTileBytes / 4;
constexpr int kSpWarps = 14;  // 0-3 softmax, 4 loader, 5 MMA issuer, 6-9 keys, 10-13 values
constexpr int kSpThreads = 32 * kSpWarps;
constexpr uint32_t kSpColO = 0, kSpColQ = 256, kSpColS = 384, kSpCols = 512;
constexpr float kSpSlack = 8.f;  // re-base a row when its max grows past 2^8
constexpr uint32_t kSpProbeNs = 4000;

// kind::f16, bf16 operands, fp32 accumulator, M = 128; S: B K-major, N = 64; P V: B
// MN-major, N = 256
constexpr uint32_t kSpIdescS = (1u << 4) | (1u << 7) | (1u << 10) | ((64u >> 3) << 17) | ((128u >> 4) << 24);
constexpr uint32_t kSpIdescPV =
    (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((256u >> 3) << 17) | ((128u >> 4) << 24);

struct SpParams {
  CUtensorMap hmap;  // history as [pages][page tokens][heads][160 bytes]
  const __nv_bfloat16 *query;
  const int32_t *table, *plan;
  const SharedItem *items;
  float *partials, *lse;
  int32_t split_slots, slot_base;
  oscar_geometry geo;
  float scale_log2;
  int32_t *status;
  int32_t item_cap;
  int32_t withhold;
  uint32_t wait_probes;
};

struct SpSmem {
  uint64_t packed_full[kSpStages], packed_empty[kSpStages];
  uint64_t k_full[2], v_full[2], s_full[2], p_full[2], pv_done[2], q_full, drained;
  uint32_t tmem;
  int32_t abort;
};
constexpr int kSpSmemBytes = 4 * kSpTileBytes + kSpStages * kSpStageBytes + (int)sizeof(SpSmem) + 1024;
static_assert(kSpSmemBytes <= 227 * 1024, "shared memory budget");

// Bounded wait (a probe may suspend the thread for a few us); gives up at the probe limit
// or as soon as another role has raised the abort flag.
OSCAR_DEVINL bool sp_wait(uint64_t *bar, uint32_t parity, SpSmem &S, const SpParams &P) {
  for (uint32_t i = 0; i < P.wait_probes; ++i) {
    if (mbar_try_wait_sleep(bar, parity, kSpProbeNs)) return true;
    if (*reinterpret_cast<volatile int32_t *>(&S.abort)) return false;
  }
  atomicExch(&S.abort, 1);
  return false;
}

// The same for a whole warp: all lanes go on, or none.
OSCAR_DEVINL bool sp_wait_warp(uint64_t *bar, uint32_t parity, SpSmem &S, const SpParams &P) {
  return __all_sync(0xffffffffu, sp_wait(bar, parity, S, P));
}

OSCAR_DEVINL void tma_load_4d(uint32_t dst, const CUtensorMap *map, int x, int y, int z, int w, uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
      : "memory");
}

// 32 codes-words of one token's half vector (two 64-dim boxes) -> bf16 rows of two boxes.
OSCAR_DEVINL void expand_half(uint8_t *tile, int token, int box0, const uint32_t (&w)[8], uint32_t sz, bool live) {
  const float s = half_bits_to_float(sz & 0xffffu), z = half_bits_to_float(sz >> 16);
  const uint32_t l01 = pack_bf162(z, __fadd_rn(s, z));
  const uint32_t l23 = pack_bf162(__fadd_rn(2.f * s, z), __fadd_rn(3.f * s, z));
  const uint32_t lo = live ? prmt(l01, l23, 0x6420u) : 0u, hi = live ? prmt(l01, l23, 0x7531u) : 0u;
  uint8_t *row = tile + box0 * kSpBox + token * 128;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    uint32_t r[8];
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const uint32_t sel = ((w[k] >> (2 * p)) & 0x03030303u) * 0x11u + 0x40404040u;
      r[2 * p] = prmt(lo, hi, sel);
      r[2 * p + 1] = prmt(lo, hi, sel >> 16);
    }
    uint8_t *dst = row + (k >> 2) * kSpBox;
    const int chunk = 2 * (k & 3);
    *reinterpret_cast<uint4 *>(dst + ((chunk ^ (token & 7)) << 4)) = make_uint4(r[0], r[1], r[2], r[3]);
    *reinterpret_cast<uint4 *>(dst + (((chunk + 1) ^ (token & 7)) << 4)) = make_uint4(r[4], r[5], r[6], r[7]);
  }
}

__global__ void __launch_bounds__(kSpThreads, 1) shared_prefix_kernel(const __grid_constant__ SpParams P) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *kt = smem, *vt = smem + 2 * kSpTileBytes, *packed = smem + 4 * kSpTileBytes;
  SpSmem &S = *reinterpret_cast<SpSmem *>(packed + kSpStages * kSpStageBytes);
  const oscar_geometry &g = P.geo;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int heads = g.kv_heads;
  const int64_t work = (int64_t)min(P.plan[0], P.item_cap) * heads;
  if (blockIdx.x >= work) return;

  if (tid == 0) {
    for (int i = 0; i < kSpStages; ++i) {
      mbar_init(&S.packed_full[i], 1);
      mbar_init(&S.packed_empty[i], 8);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&S.k_full[b], 4);
      mbar_init(&S.v_full[b], 4);
      mbar_init(&S.s_full[b], 1);
      mbar_init(&S.p_full[b], 4);
      mbar_init(&S.pv_done[b], 1);
    }
    mbar_init(&S.q_full, 4);
    mbar_init(&S.drained, 1);
    S.abort = 0;
    fence_mbarrier_init();
  }
  if (warp == 5) tmem_alloc(&S.tmem, kSpCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = S.tmem;

  // Tiles are numbered over all items of the CTA (T): buffer T & 1, phase (T >> 1) & 1.
  if (warp == 4) {
    if (lane == 0) {
      // ---- loader ----
      int T = 0;
      bool ok = true;
      for (int64_t w = blockIdx.x; w < work && ok; w += gridDim.x) {
        const SharedItem it = P.items[w / heads];
        const int head = (int)(w % heads);
        const int32_t *row = P.table + (int64_t)it.leader * g.table_stride;
        for (int t = it.tile0; t < it.tile1; ++t, ++T) {
          const int st = T % kSpStages;
          const int pos = t * kSharedTile;
          const int64_t slot = (int64_t)row[pos / kKernelBlock] * kKernelBlock + pos % kKernelBlock;
          if (T >= kSpStages && !sp_wait(&S.packed_empty[st], (T / kSpStages - 1) & 1, S, P)) {
            ok = false;
            break;
          }
          if (T == P.withhold && blockIdx.x == 0) {  // test hook: this tile never arrives
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(&S.packed_full[st], kSpStageBytes);
          tma_load_4d(smem_u32(packed + st * kSpStageBytes), &P.hmap, 0, head, (int)(slot % g.block_tokens),
                      (int)(slot / g.block_tokens), &S.packed_full[st]);
        }
      }
      // copies in flight land before the CTA exits (an aborted CTA has readers no more)
      for (int i = max(0, T - kSpStages); i < T; ++i)
        (void)mbar_wait_bounded(&S.packed_full[i % kSpStages], (i / kSpStages) & 1);
    }
  } else if (warp == 5) {
    if (lane == 0) {
      // ---- MMA issuer ----
      int T = 0, n = 0;
      bool ok = true;
      auto scores = [&](int i) {
        if (!ok || !sp_wait(&S.k_full[i & 1], (i >> 1) & 1, S, P)) {
          ok = false;
          return;
        }
        tc_fence_after();
        const uint32_t k0 = smem_u32(kt + (i & 1) * kSpTileBytes);
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            umma_f16_ts(tmem + kSpColS + 64 * (i & 1), tmem + kSpColQ + 8 * (4 * b + kk),
                        smem_desc(k0 + b * kSpBox + kk * 32, 16, 1024), kSpIdescS, (b | kk) != 0 ? 1u : 0u);
        umma_commit(&S.s_full[i & 1]);
      };
      for (int64_t w = blockIdx.x; w < work && ok; w += gridDim.x, ++n) {
        const SharedItem it = P.items[w / heads];
        const int tiles = it.tile1 - it.tile0;
        if (!sp_wait(&S.q_full, n & 1, S, P)) {
          ok = false;
          break;
        }
        tc_fence_after();
        scores(T);
        if (tiles > 1) scores(T + 1);
        for (int j = 0; j < tiles && ok; ++j) {
          const int i = T + j, b = i & 1;
          if (!sp_wait(&S.p_full[b], (i >> 1) & 1, S, P) || !sp_wait(&S.v_full[b], (i >> 1) & 1, S, P)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t v0 = smem_u32(vt + b * kSpTileBytes);
#pragma unroll
          for (int kk = 0; kk < kSharedTile / 16; ++kk)
            umma_f16_ts(tmem + kSpColO, tmem + kSpColS + 64 * b + 8 * kk, smem_desc(v0 + kk * 2048, kSpBox, 1024),
                        kSpIdescPV, (j | kk) != 0 ? 1u : 0u);
          umma_commit(&S.pv_done[b]);
          if (j + 2 < tiles) {  // its scores take the columns that P of this tile is read from
            if (!sp_wait(&S.pv_done[b], (i >> 1) & 1, S, P)) {
              ok = false;
              break;
            }
            scores(i + 2);
          }
        }
        T += tiles;
      }
      umma_commit(&S.drained);
      (void)mbar_wait_bounded(&S.drained, 0);
    }
  } else if (warp >= 6) {
    // ---- operands: thread = token x half vector ----
    const bool value = warp >= 10;
    const int w4 = (warp - 6) & 3;
    const int token = 32 * (w4 & 1) + lane, box0 = 2 * (w4 >> 1);
    uint64_t *full = value ? S.v_full : S.k_full, *freed = value ? S.pv_done : S.s_full;
    uint8_t *tiles = value ? vt : kt;
    int T = 0;
    bool ok = true;
    for (int64_t w = blockIdx.x; w < work && ok; w += gridDim.x) {
      const SharedItem it = P.items[w / heads];
      for (int t = it.tile0; t < it.tile1; ++t, ++T) {
        const int st = T % kSpStages, b = T & 1;
        if (!sp_wait_warp(&S.packed_full[st], (T / kSpStages) & 1, S, P)) {
          ok = false;
          break;
        }
        const uint4 *src = reinterpret_cast<const uint4 *>(packed + st * kSpStageBytes + token * kSpPacked);
        uint32_t words[8], sz;
        if (!value) {
          const uint4 a = src[box0], c = src[box0 + 1];
          sz = reinterpret_cast<const uint32_t *>(src)[16];
          words[0] = a.x, words[1] = a.y, words[2] = a.z, words[3] = a.w;
          words[4] = c.x, words[5] = c.y, words[6] = c.z, words[7] = c.w;
        } else {  // value codes start one word into the 16-byte vectors
          const uint4 a = src[4 + box0], c = src[5 + box0];
          words[0] = a.y, words[1] = a.z, words[2] = a.w, words[3] = c.x;
          words[4] = c.y, words[5] = c.z, words[6] = c.w;
          words[7] = reinterpret_cast<const uint32_t *>(src + 6 + box0)[0];
          sz = reinterpret_cast<const uint32_t *>(src)[33];
        }
        if (T >= 2 && !sp_wait_warp(&freed[b], ((T >> 1) - 1) & 1, S, P)) {
          ok = false;
          break;
        }
        const int pos = t * kSharedTile + token;
        expand_half(tiles + b * kSpTileBytes, token, box0, words, sz, pos >= g.sink && pos < it.end);
        fence_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&S.packed_empty[st]);
          mbar_arrive(&full[b]);
        }
      }
    }
  } else {
    // ---- softmax: thread = row = TMEM lane ----
    const int row = 32 * warp + lane;
    const uint32_t lane_base = tmem + ((uint32_t)(32 * warp) << 16);
    int T = 0;
    bool ok = true;
    for (int64_t w = blockIdx.x; w < work && ok; w += gridDim.x) {
      const SharedItem it = P.items[w / heads];
      const int head = (int)(w % heads);
      const bool live = row < it.rows;
      const int64_t qrow = (int64_t)(it.tok0 + (it.row0 + row) / g.group) * heads * g.group + head * g.group +
                           (it.row0 + row) % g.group;
      const uint4 *q = reinterpret_cast<const uint4 *>(P.query + qrow * kDim);
#pragma unroll 1
      for (int b = 0; b < 4; ++b) {
        uint32_t v[32];
#pragma unroll
        for (int u = 0; u < 4; ++u) {  // 16 dims: transposed 4 x 4
          const uint4 x = live ? q[8 * b + 2 * u] : make_uint4(0, 0, 0, 0);
          const uint4 y = live ? q[8 * b + 2 * u + 1] : make_uint4(0, 0, 0, 0);
          const uint32_t d[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
          for (int p = 0; p < 4; ++p)
#pragma unroll
            for (int a = 0; a < 2; ++a)
              v[8 * u + 2 * p + a] = prmt(d[4 * a + p / 2], d[4 * a + 2 + p / 2], p & 1 ? 0x7632u : 0x5410u);
        }
        tmem_store32(lane_base + kSpColQ + 32 * b, v);
      }
      tmem_store_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&S.q_full);

      float m = -INFINITY, l = 0.f;
      const int tiles = it.tile1 - it.tile0;
      for (int j = 0; j < tiles; ++j) {
        const int i = T + j, b = i & 1, pos = (it.tile0 + j) * kSharedTile;
        if (!sp_wait_warp(&S.s_full[b], (i >> 1) & 1, S, P)) {
          ok = false;
          break;
        }
        tc_fence_after();
        uint32_t lo[32], hi[32];
        tmem_load32x2(lane_base + kSpColS + 64 * b, lo, lane_base + kSpColS + 64 * b + 32, hi);
        float x[64];
#pragma unroll
        for (int c = 0; c < 32; ++c) x[c] = __uint_as_float(lo[c]), x[32 + c] = __uint_as_float(hi[c]);
        if (pos < g.sink || pos + kSharedTile > it.end) {
#pragma unroll
          for (int c = 0; c < 64; ++c)
            if (pos + c < g.sink || pos + c >= it.end) x[c] = -INFINITY;
        }
        float t32[32];
#pragma unroll
        for (int c = 0; c < 32; ++c) t32[c] = fmaxf(x[c], x[c + 32]);
#pragma unroll
        for (int k = 16; k >= 1; k >>= 1)
#pragma unroll
          for (int c = 0; c < k; ++c) t32[c] = fmaxf(t32[c], t32[c + k]);
        const float top = t32[0] * P.scale_log2;
        const bool rebase = m != -INFINITY && top > m + kSpSlack;
        if (m == -INFINITY) m = top;
        if (__any_sync(0xffffffffu, rebase)) {
          const float alpha = rebase ? ex2(m - top) : 1.f;
          if (rebase) {
            m = top;
            l *= alpha;
          }
          if (!sp_wait_warp(&S.pv_done[(i - 1) & 1], ((i - 1) >> 1) & 1, S, P)) {
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll 1
          for (int cb = 0; cb < 8; ++cb) {
            uint32_t o[32];
            tmem_load32(lane_base + kSpColO + 32 * cb, o);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            tmem_store32(lane_base + kSpColO + 32 * cb, o);
          }
        }
        const float base = m == -INFINITY ? 0.f : m;
        uint32_t pk[32];
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < 32; ++c) {
          const float p0 = ex2(fmaf(x[2 * c], P.scale_log2, -base)), p1 = ex2(fmaf(x[2 * c + 1], P.scale_log2, -base));
          acc[c & 3] += p0 + p1;
          pk[c] = pack_bf162(p0, p1);
        }
        l += (acc[0] + acc[1]) + (acc[2] + acc[3]);
        tmem_store32(lane_base + kSpColS + 64 * b, pk);
        tmem_store_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&S.p_full[b]);
      }
      T += tiles;
      // ---- epilogue: O / l and the lse ----
      if (ok) ok = sp_wait_warp(&S.pv_done[(T - 1) & 1], ((T - 1) >> 1) & 1, S, P);
      const int64_t out = qrow * P.split_slots + P.slot_base + it.slot;
      if (!ok) {
        if (live) P.lse[out] = -INFINITY;
        break;
      }
      tc_fence_after();
      const bool any = l > 0.f || l != l;  // a row of NaN scores stays NaN
      const float inv = any ? 1.f / l : 0.f;
      if (live) P.lse[out] = any ? m * 0.69314718055994531f + logf(l) : -INFINITY;
#pragma unroll 1
      for (int cb = 0; cb < 8; ++cb) {
        uint32_t o[32];
        tmem_load32(lane_base + kSpColO + 32 * cb, o);
        if (live && any) {
          float4 *dst = reinterpret_cast<float4 *>(P.partials + out * kDim + 32 * cb);
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              dst[4 * u + k] = make_float4(__uint_as_float(o[16 * u + k]) * inv, __uint_as_float(o[16 * u + 4 + k]) * inv,
                                           __uint_as_float(o[16 * u + 8 + k]) * inv,
                                           __uint_as_float(o[16 * u + 12 + k]) * inv);
        }
      }
      tc_fence_before();
    }
    if (!ok) {  // the CTA's remaining rows count for nothing
      if (lane == 0 && P.status) atomicExch(P.status, OSCAR_ERR_TIMEOUT);
      for (int64_t w = blockIdx.x; w < work; w += gridDim.x) {
        const SharedItem it = P.items[w / heads];
        const int head = (int)(w % heads);
        if (row < it.rows) {
          const int64_t qrow = (int64_t)(it.tok0 + (it.row0 + row) / g.group) * heads * g.group + head * g.group +
                               (it.row0 + row) % g.group;
          P.lse[qrow * P.split_slots + P.slot_base + it.slot] = -INFINITY;
        }
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(tmem, kSpCols);
  }
}

}  // namespace

int shared_prefix_launch(const SharedLaunch &L, cudaStream_t stream, int priority) {
  const oscar_geometry &g = L.geo;
  if (encode_fn() == nullptr || g.slot_bytes != 160 || (reinterpret_cast<uintptr_t>(L.history) & 15))
    return OSCAR_ERR_UNSUPPORTED;
  SpParams P;
  memset(&P, 0, sizeof(P));
  cuuint64_t dims[4] = {160, (cuuint64_t)g.kv_heads, (cuuint64_t)g.block_tokens, (cuuint64_t)L.num_pages};
  cuuint64_t strides[3] = {160, (cuuint64_t)g.kv_heads * 160, (cuuint64_t)g.page_bytes};
  cuuint32_t box[4] = {(cuuint32_t)kSpPacked, 1u, (cuuint32_t)kSharedTile, 1u};
  cuuint32_t estr[4] = {1u, 1u, 1u, 1u};
  if (encode_fn()(&P.hmap, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<uint8_t *>(L.history), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return OSCAR_ERR_INVALID;
  P.query = L.query;
  P.table = L.table, P.plan = L.plan;
  P.items = reinterpret_cast<const SharedItem *>(L.plan + kSharedHead + 2 * shared_up4(L.max_reqs));
  P.partials = L.partials, P.lse = L.lse, P.split_slots = L.split_slots, P.slot_base = L.slot_base;
  P.geo = g;
  P.scale_log2 = L.scale_log2;
  P.status = L.status;
  P.item_cap = L.items;
  P.withhold = test_hook_withhold();
  P.wait_probes = test_hook_wait_probes();
  if (!ensure_dynamic_smem<shared_prefix_kernel>(kSpSmemBytes)) return OSCAR_ERR_LAUNCH;
  cudaLaunchConfig_t cfg = {};
  const int64_t most = (int64_t)L.items * g.kv_heads;
  cfg.gridDim = dim3((unsigned)(most < sm_count() ? most : sm_count()));
  cfg.blockDim = dim3(kSpThreads);
  cfg.dynamicSmemBytes = kSpSmemBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributePriority;
  attr[0].val.priority = priority;
  cfg.attrs = attr;
  cfg.numAttrs = priority != 0 ? 1 : 0;
  if (cudaLaunchKernelEx(&cfg, shared_prefix_kernel, P) != cudaSuccess) {
    cudaGetLastError();
    return OSCAR_ERR_LAUNCH;
  }
  OSCAR_CHECK_LAUNCH();
  return OSCAR_OK;
}

}  // namespace oscar

using namespace oscar;

extern "C" int oscar_shared_prefix_layout(int32_t max_reqs, int64_t tokens, int32_t hq, int32_t kv_heads,
                                          int64_t *sizes) {
  if (!sizes || max_reqs < 1 || max_reqs > kPlanMaxReqs || tokens < 0 || tokens > INT32_MAX || hq < 1 || kv_heads < 1 ||
      hq % kv_heads || hq > (1 << 16))
    return OSCAR_ERR_INVALID;
  // row tiles of all groups (each has two members or more), and four waves of splits
  const int64_t groups = (tokens < max_reqs ? tokens : max_reqs) / 2;
  const int64_t items = tokens * (hq / kv_heads) / kSharedRows + groups + 1 + (4 * 148 + kv_heads - 1) / kv_heads;
  if (items > (1 << 26)) return OSCAR_ERR_INVALID;
  sizes[0] = items;
  sizes[1] = shared_words(max_reqs, items);
  return OSCAR_OK;
}

extern "C" int oscar_prepare_shared_prefix(const int32_t *qstarts, const int32_t *seq_lens, const int32_t *counts,
                                           const int32_t *groups, const int32_t *prefix_lens, int32_t max_reqs,
                                           int32_t items, int32_t splits, oscar_geometry geo, int32_t *plan,
                                           void *stream) {
  if (!paged_geometry_ok(geo) || max_reqs < 1 || max_reqs > kPlanMaxReqs || items < 1 || splits < 1 || splits > 63 ||
      !qstarts || !seq_lens || !counts || !groups || !prefix_lens || !plan || (reinterpret_cast<uintptr_t>(plan) & 15))
    return OSCAR_ERR_INVALID;
  PlanParams P{};
  P.qstarts = qstarts, P.seq_lens = seq_lens, P.counts = counts, P.groups = groups, P.prefix_lens = prefix_lens;
  P.plan = plan, P.max_reqs = max_reqs, P.items = items, P.splits = splits, P.sms = sm_count(), P.geo = geo;
  const size_t smem = (size_t)4 * max_reqs * sizeof(int32_t);
  if (!ensure_dynamic_smem<shared_plan_kernel>(smem)) return OSCAR_ERR_LAUNCH;
  shared_plan_kernel<<<1, kPlanThreads, smem, (cudaStream_t)stream>>>(P);
  OSCAR_CHECK_LAUNCH();
  return OSCAR_OK;
}
