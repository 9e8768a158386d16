// Decode attention of requests that share a prefix: the INT2 history of the prefix is read,
// dequantised and multiplied once per group of requests instead of once per request.
//
// A group's rows (members x queries x query heads of a KV head) are packed into tiles of
// 128 rows, and one CTA attends a tile to a run of 64-token history tiles of one KV head:
//   packed slots   one 4-D TMA copy per tile (144 of a slot's 160 bytes, 64 tokens of one
//                  head, no multicast) into a 6-stage ring;
//   operands       four warps expand the keys and four the values into bf16 tiles
//                  (128-byte swizzle): a token has only four levels bf16(c * s + z) per
//                  vector, kept in two registers, and one PRMT whose selector nibbles come
//                  from one IMAD fetches two elements.  Bytes hold dims 4i .. 4i + 3, so a
//                  PRMT yields dims (p, 4 + p) or (8 + p, 12 + p): every 16-dim block is
//                  kept transposed (position 4p + i holds dim 4i + p), the query is stored in
//                  the same order and the output is transposed back when it is written;
//   S = Q K^T      tcgen05.mma kind::f16, M = 128 rows, N = 64 tokens, K = 256, with the
//                  queries as the tensor-memory A operand (no shared-memory traffic);
//   softmax        thread = row = TMEM lane; two sets of four warps take the tiles in turn.  A
//                  row's weights are taken relative to the max of the item's first tile, with
//                  no max per tile: a tile whose weights sum to more than 2^15 (they could
//                  leave fp16) re-bases its row, rescales O and takes its weights again, and
//                  each set passes the base on to the other's next tile;
//   O += P V       fp16: P from tensor memory, V MN-major, M = 128, N = 256, K = 64.  fp16
//                  weights are off by 2^-12 where bf16 ones would be by 2^-9; the value
//                  levels go in times 2^-3, which keeps them in range (|s c + z| < 2^18) and
//                  exact down to 2^-11 (below, off by less than 2^-8 of a code's step).
// Tensor memory, all of it: O 256 columns, Q 128, S 64, P 2 x 32.  One warp issues the MMAs in
// the order S of tile t, P V of tile t - 3: while P V runs, the softmax loads the scores and
// frees their columns for the next S (two issuers would share the tensor cores between both
// and hold S back).  It issues from converged code with constant operands: an MMA whose
// operands have to be moved into uniform registers first takes 70 to 94 cycles to issue
// whatever its size, one with constant ones 32 (M 128, N 64, K 16), the tensor cores' rate.
// The range is the same for all rows of a group: [sink, end), end = the shortest of the
// members' prefix lengths and recent windows (oscar_prepare_shared_prefix); what lies behind
// it for a member stays with the per-request kernels.  Tokens outside the range get zero
// levels (their slots may hold anything) and -inf scores.  Split partials (normalised O, lse)
// join the merge of the step.
//
// 64 requests on 32K shared tokens (24 / 4 heads, 52 GFLOP): 75 us beside the step's other
// kernels, 0.7 PFLOP/s; a tile takes about 2000 cycles where the tensor cores need 1040 and
// the integer pipe 1190: the issue of four warps per scheduler bounds it.  16 operand warps
// (their registers come out of the softmax's) take 5 % longer.
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
constexpr int kPlanThreads = 256, kPlanWarps = kPlanThreads / 32;
constexpr int kPlanSpans = 32;  // candidate split lengths
constexpr int kPlanMaxReqs = 8192;
// The step's other kernels (own histories, windows) need SMs that the prefix CTAs, which fill
// theirs, leave free, or they run behind them.  Their work in 64-token tiles of one KV head
// counts 0.8 + 0.85 per row tile of theirs against a prefix tile: 64 requests on one 32K
// prompt take 104 us with 44 SMs left (the best of 0, 16, .., 56) and 124 us with none.
constexpr float kSideBase = 0.8f, kSidePerTile = 0.85f;
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
  int32_t *s_seq = sm + 4 * P.max_reqs;                       // tokens of the request
  int32_t *s_tok = sm + 5 * P.max_reqs;                       // first token in the step
  __shared__ int32_t s_cost[kPlanSpans], s_span[kPlanSpans], s_row_tiles, s_side, s_scan[kPlanWarps];
  __shared__ unsigned long long s_total;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int32_t *ends = P.plan + kSharedHead, *used = ends + (P.max_reqs + 3) / 4 * 4;
  SharedItem *items = reinterpret_cast<SharedItem *>(used + (P.max_reqs + 3) / 4 * 4);
  if (tid == 0) s_total = 0, s_row_tiles = s_side = 0;
  for (int r = tid; r < P.max_reqs; r += kPlanThreads) {
    int label = -1, limit = INT_MAX;
    if (r < nr) {
      const int seq = P.seq_lens[r], shares = P.prefix_lens[r];
      label = P.groups[r];
      const int q0 = min(P.qstarts[r], active), q1 = min(P.qstarts[r + 1], active), qlen = q1 - q0;
      if (qlen > 0) {
        const int prefix = seq - qlen, sink = min(g.sink, prefix);
        limit = min(shares, max(sink, prefix - g.recent));
      }
      s_tok[r] = q0, s_seq[r] = seq;
      if (r == nr - 1) s_tok[nr] = q1;
    }
    s_label[r] = label, s_limit[r] = limit, s_rows[r] = 0, s_tiles[r] = 0;
    ends[r] = 0, used[r] = 0;
  }
  __syncthreads();
  // one warp per run of equal labels: its active members, the shortest limit
  for (int r = warp; r < nr; r += kPlanWarps) {
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
    const int rows = (s_tok[stop] - s_tok[r]) * g.group;
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
    unsigned long long mine = 0;
    int mine_rows = 0, side = 0;
    for (int r = tid; r < nr; r += kPlanThreads) {
      mine += (unsigned long long)s_rows[r] * s_tiles[r], mine_rows += s_rows[r];
      // what the request has for itself, once per task of query_tile queries
      const int qlen = s_tok[r + 1] - s_tok[r], own = max(0, s_seq[r] - max(0, ends[r] - g.sink));
      if (qlen > 0) {
        const int rows = min(qlen, g.query_tile) * g.group, tasks = (qlen + g.query_tile - 1) / g.query_tile;
        const float cost = (kSideBase + kSidePerTile * ((rows + 7) / 8)) * tasks * own * (1.f / kSharedTile);
        side += (int)fminf(cost, 1e6f);
      }
    }
    if (mine) atomicAdd(&s_total, mine);  // few starts
    mine_rows = warp_sum(mine_rows), side = warp_sum(side);
    if (lane == 0) atomicAdd(&s_side, side), atomicAdd(&s_row_tiles, mine_rows);
  }
  __syncthreads();
  if (s_total == 0 || s_row_tiles > P.items) {  // nothing shared, or more row tiles than the plan holds
    for (int r = tid; r < nr; r += kPlanThreads) ends[r] = 0, used[r] = 0;
    if (tid == 0) P.plan[0] = 0, P.plan[1] = P.sms;
    return;
  }
  // The choice of the split length only weighs costs: 32-bit arithmetic, saturated.
  const uint32_t heads = g.kv_heads, total = (uint32_t)min(s_total * heads, 1ull << 30);
  const float side = (float)s_side * heads;
  const uint32_t sms = P.sms - (uint32_t)(min(0.5f, side / (side + total)) * P.sms);
  // candidate spans: around one wave of CTAs, then 2 .. 17 waves; the cheapest in (waves x
  // (longest split + fixed cost)) wins, the first among equals
  for (int c = warp; c < kPlanSpans; c += kPlanWarps) {
    const uint32_t base = (total + sms - 1) / sms;
    const int span = (int)(c < 16 ? base + base / 16 * c + base % 16 * c / 16 : (base + c - 15) / (c - 14));
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
      const float waves = ceilf((float)count * heads / sms);
      s_cost[c] = count > P.items ? INT_MAX : (int)fminf(waves * (longest + kItemCost), 2e9f);
      s_span[c] = span;
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
    int s = lane < kPlanWarps ? s_scan[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += u;
    }
    const int ahead = __shfl_sync(0xffffffffu, s, (warp + 31) & 31);
    const int before = done + (warp ? ahead : 0) + v - mt * k;
    done += __shfl_sync(0xffffffffu, s, 31);
    __syncthreads();
    if (r < nr) s_label[r] = before;  // first item of the group that starts here
  }
  __syncthreads();
  for (int r = warp; r < nr; r += kPlanWarps) {
    const int mt = s_rows[r];
    if (!mt) continue;
    const int tiles = s_tiles[r], k = splits_of(tiles, span, P.splits), first = s_label[r], stop = s_limit[r];
    const int leader = used[r], end = ends[r];
    const int tok0 = s_tok[r], rows = (s_tok[stop] - tok0) * g.group;
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
  if (tid == 0) P.plan[0] = done, P.plan[1] = sms;
}

// ----------------------------------------------------------------------------
// attention
// ----------------------------------------------------------------------------
constexpr int kSpPacked = 144;                           // bytes of a slot that are copied
constexpr int kSpStageBytes = kSharedTile * kSpPacked;   // 9 KiB
constexpr int kSpStages = 6;
constexpr int kSpTileBytes = kSharedTile * kDim * 2;     // 32 KiB: 4 boxes of [64 tokens][64 dims]
constexpr int kSpBox = kSpTileBytes / 4;
// 0-3 and 4-7 softmax, 8 loader, 9 MMA issuer, 10-11 idle, 12-15 keys, 16-19
// values.  Registers: 640 threads launch with 96, the softmax warpgroups take
// 144 of what the others (64) give back: 256 * 144 + 384 * 64 = 640 * 96.
constexpr int kSpWarps = 20;
constexpr int kSpLoader = 8, kSpIssue = 9, kSpKeys = 12, kSpValues = 16;
constexpr int kSpLag = 3;  // tiles between a score tile and its P V in the order of issue
constexpr int kSpRegsMany = 144, kSpRegsFew = 64;
constexpr int kSpThreads = 32 * kSpWarps;
constexpr uint32_t kSpColO = 0, kSpColQ = 256, kSpColS = 384, kSpColP = 448, kSpCols = 512;
// Weights are 2^(score - base) with base = max - 4 when it is set: fp16 then holds weights
// down to 2^-28 of the largest, and a tile may sum to 2^15 before its row takes a new base.
constexpr float kSpMostWeight = 32768.f, kSpHeadroom = 4.f;
constexpr float kSpValueScale = 0.125f;
constexpr uint32_t kSpProbeNs = 4000;

// kind::f16, fp32 accumulator, M = 128; S: bf16, B K-major, N = 64; P V: fp16, B MN-major,
// N = 256
constexpr uint32_t kSpIdescS = (1u << 4) | (1u << 7) | (1u << 10) | ((64u >> 3) << 17) | ((128u >> 4) << 24);
constexpr uint32_t kSpIdescPV = (1u << 4) | (1u << 16) | ((256u >> 3) << 17) | ((128u >> 4) << 24);

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
  // a plan of another step must not reach outside this one's buffers
  int64_t n;
  int32_t table_rows;
  int32_t item_cap;
  int32_t withhold;
  uint32_t wait_probes;
};

struct SpSmem {
  uint64_t packed_full[kSpStages], packed_empty[kSpStages];
  // A parity wait is right only while its barrier is at most one phase ahead of what the
  // waiter has seen: by buffer (T & 1) where a role waits for every tile of the buffer, by
  // T & 3 where the softmax sets also look at each other's tiles.
  uint64_t s_ready[2];   // the keys of tile T are expanded and the scores of tile T - 1 loaded
  uint64_t pv_ready[2];  // the values of tile T are expanded and its P stored
  uint64_t s_full[2];    // S of tile T is done: scores to load, keys' buffer free
  uint64_t pv_done[4];
  uint64_t base_left[4];            // per 32 rows, phase = tile: its rows' bases are in `base`
  uint64_t q_full, sums_left[4];   // phase = item
  uint64_t drained;
  float base[128], sum[2][128];
  uint32_t tmem;
  int32_t abort;
};
constexpr int kSpStageRow = 36;  // floats of a staged row of 32: 16-byte accesses hit distinct banks
constexpr int kSpStagingBytes = 8 * 32 * kSpStageRow * 4;
constexpr int kSpSmemBytes =
    4 * kSpTileBytes + kSpStages * kSpStageBytes + kSpStagingBytes + (int)sizeof(SpSmem) + 1024;
static_assert(kSpSmemBytes <= 227 * 1024, "shared memory budget");

// Bounded wait (a probe may suspend the thread for a few us); gives up at the probe limit
// or as soon as another role has raised the abort flag.
OSCAR_DEVINL bool sp_wait(uint64_t *bar, uint32_t parity, SpSmem &S, const SpParams &P) {
  if (mbar_test(bar, parity)) return true;  // half the latency of a try_wait when there is nothing to wait for
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

// One lane of a converged warp: its MMA operands stay in uniform registers.
OSCAR_DEVINL bool elect_one() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(p));
  return p != 0;
}

// d = a * b + c on two fp32 at once
OSCAR_DEVINL uint64_t pack_f32x2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
OSCAR_DEVINL void unpack_f32x2(uint64_t v, float &lo, float &hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
OSCAR_DEVINL uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
OSCAR_DEVINL uint64_t add_f32x2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// The eight code words of two 64-dim boxes of one token -> operand rows: bf16 levels
// (keys) or fp16 levels of the bf16 ones times kSpValueScale (values).
OSCAR_DEVINL void expand_half(uint8_t *tile, int token, int box0, const uint32_t (&w)[8], uint32_t sz, bool live,
                              bool value) {
  const float s = half_bits_to_float(sz & 0xffffu), z = half_bits_to_float(sz >> 16);
  uint32_t l01 = pack_bf162(z, __fadd_rn(s, z)), l23 = pack_bf162(__fadd_rn(2.f * s, z), __fadd_rn(3.f * s, z));
  if (value) {
    l01 = pack_half2(bf16_bits_to_float(l01 & 0xffffu) * kSpValueScale, bf16_bits_to_float(l01 >> 16) * kSpValueScale);
    l23 = pack_half2(bf16_bits_to_float(l23 & 0xffffu) * kSpValueScale, bf16_bits_to_float(l23 >> 16) * kSpValueScale);
  }
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

// The MMAs of one tile in buffer B (constant operands).
template <int B>
OSCAR_DEVINL void issue_scores(uint32_t k0) {
#pragma unroll
  for (int k = 0; k < 16; ++k)
    umma_f16_ts(kSpColS, kSpColQ + 8 * k, smem_desc(k0 + B * kSpTileBytes + (k >> 2) * kSpBox + (k & 3) * 32, 16, 1024),
                kSpIdescS, k != 0 ? 1u : 0u);
}
template <int B>
OSCAR_DEVINL void issue_values(uint32_t v0, uint32_t accumulate) {
#pragma unroll
  for (int k = 0; k < kSharedTile / 16; ++k)
    umma_f16_ts(kSpColO, kSpColP + 32 * B + 8 * k, smem_desc(v0 + B * kSpTileBytes + k * 2048, kSpBox, 1024), kSpIdescPV,
                k != 0 ? 1u : accumulate);
}

__global__ void __launch_bounds__(kSpThreads, 1) shared_prefix_kernel(const __grid_constant__ SpParams P) {
  extern __shared__ uint8_t smem_raw[];
  // an offset keeps the address space (a pointer rounded as an integer makes every access generic)
  uint8_t *smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  uint8_t *kt = smem, *vt = smem + 2 * kSpTileBytes, *packed = smem + 4 * kSpTileBytes;
  float *staging = reinterpret_cast<float *>(packed + kSpStages * kSpStageBytes);
  SpSmem &S = *reinterpret_cast<SpSmem *>(packed + kSpStages * kSpStageBytes + kSpStagingBytes);
  const oscar_geometry &g = P.geo;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int heads = g.kv_heads;
  const int64_t work = (int64_t)min(P.plan[0], P.item_cap) * heads;
  const int ctas = min((int)gridDim.x, P.plan[1]);
  if (blockIdx.x >= ctas || blockIdx.x >= work) return;

  if (tid == 0) {
    for (int i = 0; i < kSpStages; ++i) {
      mbar_init(&S.packed_full[i], 1);
      mbar_init(&S.packed_empty[i], 8);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&S.s_ready[b], 8);
      mbar_init(&S.pv_ready[b], 8);
      mbar_init(&S.s_full[b], 1);
    }
    for (int i = 0; i < 4; ++i) mbar_init(&S.pv_done[i], 1);
    mbar_init(&S.q_full, 8);
    for (int i = 0; i < 4; ++i) {
      mbar_init(&S.base_left[i], 1);
      mbar_init(&S.sums_left[i], 2);
    }
    mbar_init(&S.drained, 1);
    S.abort = 0;
    fence_mbarrier_init();
  }
  if (warp == kSpIssue) tmem_alloc(&S.tmem, kSpCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // all columns are allocated, so they start at 0: constant addresses below
  if (S.tmem != 0) return;  // uniform; cannot happen

  // Tiles are numbered over all items of the CTA (T).
  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSpRegsMany));
    // ---- softmax: thread = row = TMEM lane; set `half` takes the tiles T of its parity ----
    const int half = warp >> 2, quarter = warp & 3, row = 32 * quarter + lane;
    const uint32_t lane_base = (uint32_t)(32 * quarter) << 16;
    if (half == 0 && lane == 0) mbar_arrive(&S.s_ready[0]);  // no scores before tile 0
    int T = 0, n = 0;
    bool ok = true;
    for (int64_t w = blockIdx.x; w < work && ok; w += ctas, ++n) {
      const SharedItem it = P.items[w / heads];
      const int head = (int)(w % heads);
      const bool live = row < it.rows && it.tok0 + (it.row0 + row) / g.group < P.n;
      const int64_t qrow = (int64_t)(it.tok0 + (it.row0 + row) / g.group) * heads * g.group + head * g.group +
                           (it.row0 + row) % g.group;
      const uint4 *q = reinterpret_cast<const uint4 *>(P.query + qrow * kDim) + 16 * half;
#pragma unroll
      for (int b = 0; b < 2; ++b) {
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
        tmem_store32(lane_base + kSpColQ + 64 * half + 32 * b, v);
      }
      tmem_store_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&S.q_full);

      float m = -INFINITY, l = 0.f;  // base (log2) of the weights, and this set's sum of them
      const int end_T = T + it.tile1 - it.tile0;
      const uint64_t scale2 = pack_f32x2(P.scale_log2, P.scale_log2);
      for (int i = T + ((T ^ half) & 1); i < end_T; i += 2) {
        const int b = i & 1, pos = (it.tile0 + i - T) * kSharedTile;
        if (!sp_wait_warp(&S.s_full[b], (i >> 1) & 1, S, P)) {
          ok = false;
          break;
        }
        tc_fence_after();
        uint32_t lo[32], hi[32];
        tmem_load32x2(lane_base + kSpColS, lo, lane_base + kSpColS + 32, hi);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&S.s_ready[(i + 1) & 1]);
        if (pos < g.sink || pos + kSharedTile > it.end) {
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            if (pos + c < g.sink || pos + c >= it.end) lo[c] = 0xff800000u;
            if (pos + 32 + c < g.sink || pos + 32 + c >= it.end) hi[c] = 0xff800000u;
          }
        }
        auto largest = [&]() {
          float t[8];
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            t[c] = fmaxf(__uint_as_float(lo[c]), __uint_as_float(hi[c]));
#pragma unroll
            for (int k = 1; k < 4; ++k)
              t[c] = fmaxf(t[c], fmaxf(__uint_as_float(lo[c + 8 * k]), __uint_as_float(hi[c + 8 * k])));
          }
#pragma unroll
          for (int k = 4; k >= 1; k >>= 1)
#pragma unroll
            for (int c = 0; c < k; ++c) t[c] = fmaxf(t[c], t[c + k]);
          return t[0] * P.scale_log2 - kSpHeadroom;
        };
        uint32_t pk[32];
        auto weights = [&](float base) {  // P of the tile relative to 2^base; returns their sum
          if (base == -INFINITY) base = 0.f;
          const uint64_t neg2 = pack_f32x2(-base, -base);
          uint64_t acc[2] = {0, 0};
          auto pairs = [&](const uint32_t(&v)[32], int at) {
#pragma unroll
            for (int c = 0; c < 16; ++c) {
              float p0, p1;
              unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(v[2 * c]), __uint_as_float(v[2 * c + 1])), scale2, neg2),
                           p0, p1);
              p0 = ex2(p0), p1 = ex2(p1);
              acc[c & 1] = add_f32x2(acc[c & 1], pack_f32x2(p0, p1));
              pk[at + c] = pack_half2(p0, p1);
            }
          };
          pairs(lo, 0);
          pairs(hi, 16);
          float a, b2;
          unpack_f32x2(add_f32x2(acc[0], acc[1]), a, b2);
          return a + b2;
        };
        // the base that the tile before left; the second tile's set learns it here
        bool checked = i <= T + 1, fresh = false;
        if (checked) {
          if (i > 0 && !sp_wait_warp(&S.base_left[quarter], (i - 1) & 1, S, P)) {
            ok = false;
            break;
          }
          m = i == T ? largest() : S.base[row];
        }
        float sum = 0.f;
#pragma unroll 1
        while (ok) {  // once, but for rows that re-base
          sum = weights(m);
          if (!checked) {
            checked = true;
            if (!(ok = sp_wait_warp(&S.base_left[quarter], (i - 1) & 1, S, P))) break;
            const float now = S.base[row];
            if (__any_sync(0xffffffffu, now != m && m == m)) {  // the other set re-based meanwhile
              l *= m == -INFINITY ? 0.f : ex2(m - now);
              m = now;
              continue;
            }
          }
          // weights too large for fp16 (or all of the row's scores so far -inf): a new base
          const bool high = !fresh && (!(sum <= kSpMostWeight) || (m == -INFINITY && i > T));
          if (!__any_sync(0xffffffffu, high)) break;
          fresh = true;
          const float top = fmaxf(m, largest());
          const float alpha = high && m != -INFINITY ? ex2(m - top) : 1.f;
          if (i > T) {
            if (!(ok = sp_wait_warp(&S.pv_done[(i - 1) & 3], ((i - 1) >> 2) & 1, S, P))) break;
            tc_fence_after();
#pragma unroll 1
            for (int cb = 0; cb < 16; ++cb) {
              uint32_t o[16];
              tmem_load16(kSpColO + lane_base + 16 * cb, o);
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
              tmem_store16(kSpColO + lane_base + 16 * cb, o);
            }
          }
          if (high) {
            l *= alpha;
            m = top;
          }
        }
        if (!ok) break;
        l += sum;
        S.base[row] = m;
        __syncwarp();
        if (lane == 0) mbar_arrive(&S.base_left[quarter]);
        if (i >= 2 && !sp_wait_warp(&S.pv_done[(i - 2) & 3], ((i - 2) >> 2) & 1, S, P)) {  // its P is read
          ok = false;
          break;
        }
        tc_fence_after();
        tmem_store32(lane_base + kSpColP + 32 * b, pk);
        tmem_store_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&S.pv_ready[b]);
      }
      T = end_T;
      // ---- epilogue: O / l and the lse; each set writes half of every row ----
      if (ok) ok = sp_wait_warp(&S.base_left[quarter], (T - 1) & 1, S, P);
      float last = 0.f;
      if (ok) {
        last = S.base[row];
        S.sum[half][row] = m == last ? l : (m == -INFINITY ? 0.f : l * ex2(m - last));
        __syncwarp();
        if (lane == 0) mbar_arrive(&S.sums_left[quarter]);
        ok = sp_wait_warp(&S.sums_left[quarter], n & 1, S, P);
      }
      if (ok) ok = sp_wait_warp(&S.pv_done[(T - 1) & 3], ((T - 1) >> 2) & 1, S, P);
      if (!ok) break;
      const int64_t out = qrow * P.split_slots + P.slot_base + it.slot;
      const float total = S.sum[0][row] + S.sum[1][row];
      tc_fence_after();
      const bool any = total > 0.f || total != total;  // a row of NaN scores stays NaN
      const float inv = any ? (1.f / kSpValueScale) / total : 0.f;
      if (live && half == 0) P.lse[out] = any ? last * 0.69314718055994531f + logf(total) : -INFINITY;
      // through shared memory, so that a store instruction writes 128 bytes of each of 4 rows
      // (a thread's own row alone would be 32 lines per instruction)
      float *stage = staging + warp * kSpStageRow * 32;
      float *row_out[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int r = 4 * k + (lane >> 3);
        const int64_t at = __shfl_sync(0xffffffffu, out, r);
        const bool writes = __shfl_sync(0xffffffffu, (int)(live && any), r);
        row_out[k] = writes ? P.partials + at * kDim + 128 * half + 4 * (lane & 7) : nullptr;
      }
#pragma unroll 1
      for (int cb = 0; cb < 4; ++cb) {
        uint32_t o[32];
        tmem_load32(lane_base + kSpColO + 128 * half + 32 * cb, o);
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            *reinterpret_cast<float4 *>(stage + lane * kSpStageRow + 16 * u + 4 * k) =
                make_float4(__uint_as_float(o[16 * u + k]) * inv, __uint_as_float(o[16 * u + 4 + k]) * inv,
                            __uint_as_float(o[16 * u + 8 + k]) * inv, __uint_as_float(o[16 * u + 12 + k]) * inv);
        __syncwarp();
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (row_out[k])
            *reinterpret_cast<float4 *>(row_out[k] + 32 * cb) =
                *reinterpret_cast<const float4 *>(stage + (4 * k + (lane >> 3)) * kSpStageRow + 4 * (lane & 7));
        __syncwarp();
      }
      tc_fence_before();
    }
    if (!ok) {  // the CTA's remaining rows count for nothing
      if (lane == 0 && P.status) atomicExch(P.status, OSCAR_ERR_TIMEOUT);
      for (int64_t w = blockIdx.x; w < work; w += ctas) {
        const SharedItem it = P.items[w / heads];
        const int head = (int)(w % heads);
        if (row < it.rows && it.tok0 + (it.row0 + row) / g.group < P.n) {
          const int64_t qrow = (int64_t)(it.tok0 + (it.row0 + row) / g.group) * heads * g.group + head * g.group +
                               (it.row0 + row) % g.group;
          P.lse[qrow * P.split_slots + P.slot_base + it.slot] = -INFINITY;
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kSpRegsFew));
    if (warp == kSpLoader) {
      if (lane == 0) {
        // ---- loader ----
        int T = 0;
        bool ok = true;
        for (int64_t w = blockIdx.x; w < work && ok; w += ctas) {
          const SharedItem it = P.items[w / heads];
          const int head = (int)(w % heads);
          const int32_t *row = P.table + (int64_t)min((uint32_t)it.leader, (uint32_t)P.table_rows - 1) * g.table_stride;
          for (int t = it.tile0; t < it.tile1; ++t, ++T) {
            const int st = T % kSpStages;
            const int pos = t * kSharedTile;
            const int64_t slot = (int64_t)row[min(pos / kKernelBlock, g.table_stride - 1)] * kKernelBlock + pos % kKernelBlock;
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
    } else if (warp == kSpIssue) {
      // ---- MMAs: S of tile i, then P V of tile i - 3 ----
      if (elect_one()) {
        int T = 0, n = 0;
        bool ok = true;
        for (int64_t w = blockIdx.x; w < work && ok; w += ctas, ++n) {
          const SharedItem it = P.items[w / heads];
          const int end_T = T + it.tile1 - it.tile0;
          ok = sp_wait(&S.q_full, n & 1, S, P);
          for (int i = T; i < end_T + kSpLag && ok; ++i) {
            // both waits first: S and P V then enter the tensor cores' queue without a gap,
            // and the P V at its end covers the commits and the next waits
            const int j = i - kSpLag;
            ok = (i >= end_T || sp_wait(&S.s_ready[i & 1], (i >> 1) & 1, S, P)) &&
                 (j < T || sp_wait(&S.pv_ready[j & 1], (j >> 1) & 1, S, P));
            if (!ok) break;
            tc_fence_after();
            if (i < end_T) {
              if (i & 1)
                issue_scores<1>(smem_u32(kt));
              else
                issue_scores<0>(smem_u32(kt));
              umma_commit(&S.s_full[i & 1]);
            }
            if (j >= T) {
              if (j & 1)
                issue_values<1>(smem_u32(vt), j != T ? 1u : 0u);
              else
                issue_values<0>(smem_u32(vt), j != T ? 1u : 0u);
              umma_commit(&S.pv_done[j & 3]);
            }
          }
          T = end_T;
        }
        umma_commit(&S.drained);
        (void)mbar_wait_bounded(&S.drained, 0);
      }
    } else if (warp >= kSpKeys) {
      // ---- operands: thread = token x half vector ----
      const bool value = warp >= kSpValues;
      const int w4 = (warp - kSpKeys) & 3;
      const int token = 32 * (w4 & 1) + lane, box0 = 2 * (w4 >> 1);
      uint64_t *full = value ? S.pv_ready : S.s_ready;
      uint8_t *tiles = value ? vt : kt;
      int T = 0;
      bool ok = true;
      for (int64_t w = blockIdx.x; w < work && ok; w += ctas) {
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
          // the buffer is free once the MMAs of tile T - 2 are done
          if (T >= 2 && !(value ? sp_wait_warp(&S.pv_done[(T - 2) & 3], ((T - 2) >> 2) & 1, S, P)
                                : sp_wait_warp(&S.s_full[b], ((T >> 1) - 1) & 1, S, P))) {
            ok = false;
            break;
          }
          const int pos = t * kSharedTile + token;
          expand_half(tiles + b * kSpTileBytes, token, box0, words, sz, pos >= g.sink && pos < it.end, value);
          fence_async_smem();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&S.packed_empty[st]);
            mbar_arrive(&full[b]);
          }
        }
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == kSpIssue) {
    tc_fence_after();
    tmem_dealloc(0, kSpCols);
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
  P.table = L.table, P.plan = L.plan, P.n = L.n, P.table_rows = L.table_rows;
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
  const size_t smem = ((size_t)6 * max_reqs + 1) * sizeof(int32_t);
  if (!ensure_dynamic_smem<shared_plan_kernel>(smem)) return OSCAR_ERR_LAUNCH;
  shared_plan_kernel<<<1, kPlanThreads, smem, (cudaStream_t)stream>>>(P);
  OSCAR_CHECK_LAUNCH();
  return OSCAR_OK;
}
