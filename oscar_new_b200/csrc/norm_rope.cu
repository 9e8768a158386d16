// Per-head norm of queries and keys and the position rotation, in one pass over the rows
// that then enter rotate_store and the attention (the reference leaves both to the model).
//
//   y = x * rsqrt(mean(x^2) + eps) * (w + offset);  pairs (a, b) of the first `rotary`
//   dims turn to (a cos - b sin, b cos + a sin) with the position's table row; the pairs
//   are (i, i + rotary / 2), or (2 i, 2 i + 1) when interleaved.
//
// Everything is fp32 between the bf16 input and the one rounding of the output.  A warp
// owns one token's run of query or key heads; a lane holds 8 dims of a row as four pairs
// that turn together (two 8-byte loads: dims 4l and rotary / 2 + 4l of a turning lane in the
// split form, 8l and 8l + 4 else), so the only exchange is the sum of squares.  With the
// weights inside the rotation's coefficients (cos 1, sin 0 for dims that do not turn) a pair
// is six multiplies and adds for all lanes alike:
//   y_a = r (x_a (w_a cos) - x_b (w_b sin)),  y_b = r (x_b (w_b cos) + x_a (w_a sin)).
// The first rows are asked for before the position is known.
//
// Measured on a B200: 16384 tokens, 24 + 4 heads, 64 rotary dims, bf16 (475 MB): 91 us, 5.2
// TB/s; with one 16-byte load a lane and the partner of a pair shuffled in, 122 us.
#include <algorithm>

#include "common.cuh"

namespace oscar {
namespace {

constexpr int kNrWarps = 8, kNrBlocks = 4;  // 32 warps per SM
constexpr int kNrRows = 2;                  // rows in flight per warp (1: 109 us, 4: 109 us and spills)

struct NrParams {
  const __nv_bfloat16 *q, *k;
  int64_t qs0, qs1, ks0, ks1;
  __nv_bfloat16 *qo, *ko;
  int64_t qos0, qos1, kos0, kos1;
  const void *qw, *kw, *positions, *table;
  int64_t max_positions;
  int64_t n;
  int32_t hq, hkv, rotary, weight_f32, table_f32, positions_64;
  int32_t q_runs, runs, run;  // runs of queries and in all per token, heads per run
  float eps, offset;
  const int32_t *counts;
  int32_t *status;
};

// Four consecutive fp32 or bf16 values.
OSCAR_DEVINL void load_floats(float (&v)[4], const void *base, int64_t at, bool f32) {
  if (f32) {
    const float4 x = __ldg(reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(base) + at));
    v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
  } else {
    const uint2 x = __ldg(reinterpret_cast<const uint2 *>(reinterpret_cast<const __nv_bfloat16 *>(base) + at));
    v[0] = bf16_bits_to_float(x.x & 0xffffu), v[1] = bf16_bits_to_float(x.x >> 16);
    v[2] = bf16_bits_to_float(x.y & 0xffffu), v[3] = bf16_bits_to_float(x.y >> 16);
  }
}

OSCAR_DEVINL void unpack4(const uint2 &v, float (&x)[4]) {
  x[0] = bf16_bits_to_float(v.x & 0xffffu), x[1] = __uint_as_float(v.x & 0xffff0000u);
  x[2] = bf16_bits_to_float(v.y & 0xffffu), x[3] = __uint_as_float(v.y & 0xffff0000u);
}

template <bool INTERLEAVED>
__global__ void __launch_bounds__(32 * kNrWarps, kNrBlocks) qk_norm_rope_kernel(const NrParams P) {
  const int lane = threadIdx.x & 31;
  const int64_t unit = (int64_t)blockIdx.x * kNrWarps + (threadIdx.x >> 5);
  const int64_t token = unit / P.runs;
  const int run = (int)(unit - token * P.runs);
  if (token >= P.n || (P.counts && token >= P.counts[1])) return;
  const bool isq = run < P.q_runs;
  const int h0 = (isq ? run : run - P.q_runs) * P.run, heads = min(P.run, (isq ? P.hq : P.hkv) - h0);
  const int half = P.rotary >> 1;
  const bool turns = 8 * lane < P.rotary;
  const int off0 = !INTERLEAVED && turns ? 4 * lane : 8 * lane, off1 = !INTERLEAVED && turns ? half + 4 * lane : 8 * lane + 4;
  const int64_t s1 = isq ? P.qs1 : P.ks1, o1 = isq ? P.qos1 : P.kos1;
  const __nv_bfloat16 *src = (isq ? P.q + token * P.qs0 : P.k + token * P.ks0) + h0 * s1;
  __nv_bfloat16 *dst = (isq ? P.qo + token * P.qos0 : P.ko + token * P.kos0) + h0 * o1;
  uint2 raw[kNrRows][2];
#pragma unroll
  for (int i = 0; i < kNrRows; ++i)
    if (i < heads) {
      raw[i][0] = *reinterpret_cast<const uint2 *>(src + i * s1 + off0);
      raw[i][1] = *reinterpret_cast<const uint2 *>(src + i * s1 + off1);
    }
  src += kNrRows * s1;
  const int64_t position = P.positions_64 ? __ldg(reinterpret_cast<const long long *>(P.positions) + token)
                                          : (int64_t)__ldg(reinterpret_cast<const int32_t *>(P.positions) + token);
  float w0[4], w1[4], c[4] = {1.f, 1.f, 1.f, 1.f}, s[4] = {0.f, 0.f, 0.f, 0.f};
  load_floats(w0, isq ? P.qw : P.kw, off0, P.weight_f32);
  load_floats(w1, isq ? P.qw : P.kw, off1, P.weight_f32);
  if (P.rotary > 0 && (position < 0 || position >= P.max_positions)) {  // the token's rows stay unwritten
    if (lane == 0 && P.status) atomicExch(P.status, OSCAR_ERR_INVALID);
    return;
  }
  if (turns) {
    load_floats(c, P.table, position * P.rotary + 4 * lane, P.table_f32);
    load_floats(s, P.table, position * P.rotary + half + 4 * lane, P.table_f32);
  }
  // pair e: dims (off0 + e, off1 + e), or adjacent dims when interleaved; coefficients of
  // y_a: aa x_a - ab x_b, of y_b: bb x_b + ba x_a
  float aa[4], ab[4], bb[4], ba[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float wa = P.offset + (INTERLEAVED ? (e < 2 ? w0[2 * e] : w1[2 * e - 4]) : w0[e]);
    const float wb = P.offset + (INTERLEAVED ? (e < 2 ? w0[2 * e + 1] : w1[2 * e - 3]) : w1[e]);
    aa[e] = wa * c[e], ab[e] = wb * s[e], bb[e] = wb * c[e], ba[e] = wa * s[e];
  }
  for (int h = 0; h < heads; h += kNrRows) {
#pragma unroll
    for (int i = 0; i < kNrRows; ++i) {
      if (h + i >= heads) break;
      float x0[4], x1[4];
      unpack4(raw[i][0], x0);
      unpack4(raw[i][1], x1);
      if (h + i + kNrRows < heads) {
        raw[i][0] = *reinterpret_cast<const uint2 *>(src + i * s1 + off0);
        raw[i][1] = *reinterpret_cast<const uint2 *>(src + i * s1 + off1);
      }
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) ss = fmaf(x0[e], x0[e], fmaf(x1[e], x1[e], ss));
#pragma unroll
      for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float r = rsqrtf(ss * (1.f / kDim) + P.eps);
      float y0[4], y1[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float a = INTERLEAVED ? (e < 2 ? x0[2 * e] : x1[2 * e - 4]) : x0[e];
        const float b = INTERLEAVED ? (e < 2 ? x0[2 * e + 1] : x1[2 * e - 3]) : x1[e];
        const float ya = r * (a * aa[e] - b * ab[e]), yb = r * (b * bb[e] + a * ba[e]);
        if (INTERLEAVED) {
          if (e < 2)
            y0[2 * e] = ya, y0[2 * e + 1] = yb;
          else
            y1[2 * e - 4] = ya, y1[2 * e - 3] = yb;
        } else {
          y0[e] = ya, y1[e] = yb;
        }
      }
      // Dims that do not turn met their lane partner with coefficient 0, and an infinite one
      // (r = 0 then) made NaN of them: without it, in rows that hold one (90.3 -> 91.2 us).
      if (!(ss < INFINITY) && !turns) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          y0[e] = r * (x0[e] * (INTERLEAVED ? (e & 1 ? bb[e >> 1] : aa[e >> 1]) : aa[e]));
          y1[e] = r * (x1[e] * (INTERLEAVED ? (e & 1 ? bb[2 + (e >> 1)] : aa[2 + (e >> 1)]) : bb[e]));
        }
      }
      *reinterpret_cast<uint2 *>(dst + i * o1 + off0) = make_uint2(pack_bf162(y0[0], y0[1]), pack_bf162(y0[2], y0[3]));
      *reinterpret_cast<uint2 *>(dst + i * o1 + off1) = make_uint2(pack_bf162(y1[0], y1[1]), pack_bf162(y1[2], y1[3]));
    }
    src += kNrRows * s1, dst += kNrRows * o1;
  }
}

}  // namespace
}  // namespace oscar

using namespace oscar;

extern "C" int oscar_qk_norm_rope(const void *query, int64_t qs0, int64_t qs1, const void *key, int64_t ks0,
                                  int64_t ks1, int64_t n, int32_t hq, int32_t hkv, const void *q_weight,
                                  const void *k_weight, int32_t weight_f32, float weight_offset, float eps,
                                  const void *positions, int32_t positions_64, const void *cos_sin,
                                  int32_t table_f32, int64_t max_positions, int32_t rotary, int32_t interleaved,
                                  const int32_t *counts, void *query_out, int64_t qos0, int64_t qos1, void *key_out,
                                  int64_t kos0, int64_t kos1, int32_t *status, void *stream) {
  if (n < 0 || hq < 0 || hkv < 0 || hq > (1 << 16) || hkv > (1 << 16) || rotary < 0 || rotary > kDim || rotary % 16 ||
      max_positions < 0 || !(eps >= 0.f))
    return OSCAR_ERR_INVALID;
  if (n == 0 || hq + hkv == 0) return OSCAR_OK;
  if (!positions || (rotary && !cos_sin) || (hq && (!query || !query_out)) || (hkv && (!key || !key_out)) ||
      !q_weight || !k_weight)
    return OSCAR_ERR_INVALID;
  const uintptr_t rows = reinterpret_cast<uintptr_t>(query) | reinterpret_cast<uintptr_t>(key) |
                         reinterpret_cast<uintptr_t>(query_out) | reinterpret_cast<uintptr_t>(key_out) |
                         reinterpret_cast<uintptr_t>(q_weight) | reinterpret_cast<uintptr_t>(k_weight) |
                         reinterpret_cast<uintptr_t>(cos_sin);
  if ((rows & 15) || qs0 % 8 || qs1 % 8 || ks0 % 8 || ks1 % 8 || qos0 % 8 || qos1 % 8 || kos0 % 8 || kos1 % 8)
    return OSCAR_ERR_INVALID;
  NrParams P{};
  P.q = reinterpret_cast<const __nv_bfloat16 *>(query), P.qs0 = qs0, P.qs1 = qs1;
  P.k = reinterpret_cast<const __nv_bfloat16 *>(key), P.ks0 = ks0, P.ks1 = ks1;
  P.qo = reinterpret_cast<__nv_bfloat16 *>(query_out), P.qos0 = qos0, P.qos1 = qos1;
  P.ko = reinterpret_cast<__nv_bfloat16 *>(key_out), P.kos0 = kos0, P.kos1 = kos1;
  P.qw = q_weight, P.kw = k_weight, P.weight_f32 = weight_f32, P.offset = weight_offset, P.eps = eps;
  P.positions = positions, P.positions_64 = positions_64;
  P.table = cos_sin, P.table_f32 = table_f32, P.max_positions = max_positions, P.rotary = rotary;
  P.n = n, P.hq = hq, P.hkv = hkv, P.counts = counts, P.status = status;
  // few tokens: a warp per row (latency); many: runs of heads share the token's table row
  P.run = n * (hq + hkv) <= 148 * 32 ? 1 : 8;
  P.q_runs = (hq + P.run - 1) / P.run;
  P.runs = P.q_runs + (hkv + P.run - 1) / P.run;
  const int64_t blocks = (n * P.runs + kNrWarps - 1) / kNrWarps;
  if (blocks > INT32_MAX) return OSCAR_ERR_INVALID;
  if (interleaved)
    qk_norm_rope_kernel<true><<<(unsigned)blocks, 32 * kNrWarps, 0, (cudaStream_t)stream>>>(P);
  else
    qk_norm_rope_kernel<false><<<(unsigned)blocks, 32 * kNrWarps, 0, (cudaStream_t)stream>>>(P);
  OSCAR_CHECK_LAUNCH();
  return OSCAR_OK;
}
