// Per-head norm of queries and keys and the position rotation, in one pass over the rows
// that then enter rotate_store and the attention (the reference leaves both to the model).
//
//   y = x * rsqrt(mean(x^2) + eps) * (w + offset);  pairs (a, b) of the first `rotary`
//   dims turn to (a cos - b sin, b cos + a sin) with the position's table row; the pairs
//   are (i, i + rotary / 2), or (2 i, 2 i + 1) when interleaved.
//
// Everything is fp32 between the bf16 input and the one rounding of the output.  A warp
// owns one token's run of heads: lane l holds dims 8l .. 8l + 7 of a row (one 16-byte
// load), the row's sum of squares is five shuffles, and the pair partner of the split
// form sits rotary / 16 lanes away (rotary a multiple of 16), so nothing goes through
// shared memory.  The token's cos / sin and both weights stay in registers over its heads.
#include <algorithm>

#include "common.cuh"

namespace oscar {
namespace {

constexpr int kNrWarps = 8;

struct NrParams {
  const __nv_bfloat16 *q, *k;
  int64_t qs0, qs1, ks0, ks1;
  __nv_bfloat16 *qo, *ko;
  int64_t qos0, qos1, kos0, kos1;
  const void *qw, *kw, *positions, *table;
  int64_t max_positions;
  int64_t n;
  int32_t hq, hkv, rotary, weight_f32, table_f32, positions_64;
  int32_t runs, run;  // runs per token, heads per run
  float eps, offset;
  const int32_t *counts;
  int32_t *status;
};

// COUNT consecutive fp32 or bf16 values, 8-byte aligned (COUNT 4) or 16-byte aligned (8)
template <int COUNT>
OSCAR_DEVINL void load_floats(float (&v)[8], const void *base, int64_t at, bool f32) {
  if (f32) {
    const float4 *src = reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(base) + at);
#pragma unroll
    for (int i = 0; i < COUNT / 4; ++i) {
      const float4 x = __ldg(src + i);
      v[4 * i] = x.x, v[4 * i + 1] = x.y, v[4 * i + 2] = x.z, v[4 * i + 3] = x.w;
    }
  } else {
    const uint2 *src = reinterpret_cast<const uint2 *>(reinterpret_cast<const __nv_bfloat16 *>(base) + at);
#pragma unroll
    for (int i = 0; i < COUNT / 4; ++i) {
      const uint2 x = __ldg(src + i);
      v[4 * i] = bf16_bits_to_float(x.x & 0xffffu), v[4 * i + 1] = bf16_bits_to_float(x.x >> 16);
      v[4 * i + 2] = bf16_bits_to_float(x.y & 0xffffu), v[4 * i + 3] = bf16_bits_to_float(x.y >> 16);
    }
  }
}

template <bool INTERLEAVED>
__global__ void __launch_bounds__(32 * kNrWarps) qk_norm_rope_kernel(const NrParams P) {
  const int lane = threadIdx.x & 31;
  const int64_t unit = (int64_t)blockIdx.x * kNrWarps + (threadIdx.x >> 5);
  const int64_t token = unit / P.runs;
  const int h0 = (int)(unit % P.runs) * P.run, heads = P.hq + P.hkv;
  if (token >= P.n || (P.counts && token >= P.counts[1])) return;
  const int64_t position = P.positions_64 ? __ldg(reinterpret_cast<const long long *>(P.positions) + token)
                                          : (int64_t)__ldg(reinterpret_cast<const int32_t *>(P.positions) + token);
  if (position < 0 || position >= P.max_positions) {  // the token's rows stay unwritten
    if (lane == 0 && P.status) atomicExch(P.status, OSCAR_ERR_INVALID);
    return;
  }
  const int half = P.rotary >> 1;
  const bool turns = 8 * lane < P.rotary;
  const bool first = 8 * lane < half;
  const int partner = !turns ? lane : (first ? lane + half / 8 : lane - half / 8);
  float cosv[8], sinv[8];
  if (turns) {
    const int64_t row = position * P.rotary;
    if (INTERLEAVED) {
      load_floats<4>(cosv, P.table, row + 4 * lane, P.table_f32);
      load_floats<4>(sinv, P.table, row + half + 4 * lane, P.table_f32);
    } else {
      const int at = first ? 8 * lane : 8 * lane - half;
      load_floats<8>(cosv, P.table, row + at, P.table_f32);
      load_floats<8>(sinv, P.table, row + half + at, P.table_f32);
      if (first) {
#pragma unroll
        for (int e = 0; e < 8; ++e) sinv[e] = -sinv[e];
      }
    }
  }
  float w[2][8];
  load_floats<8>(w[0], P.qw, 8 * lane, P.weight_f32);
  load_floats<8>(w[1], P.kw, 8 * lane, P.weight_f32);
#pragma unroll
  for (int e = 0; e < 8; ++e) w[0][e] += P.offset, w[1][e] += P.offset;

  constexpr int B = 4;  // rows in flight per warp
  const int h1 = min(h0 + P.run, heads);
  for (int hb = h0; hb < h1; hb += B) {
    uint4 raw[B];
#pragma unroll
    for (int i = 0; i < B; ++i) {
      const int h = hb + i;
      if (h < h1) {
        const __nv_bfloat16 *src = h < P.hq ? P.q + token * P.qs0 + h * P.qs1 : P.k + token * P.ks0 + (h - P.hq) * P.ks1;
        raw[i] = *reinterpret_cast<const uint4 *>(src + 8 * lane);
      }
    }
#pragma unroll
    for (int i = 0; i < B; ++i) {
      const int h = hb + i;
      if (h >= h1) break;
      const uint32_t word[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
      float x[8], ss = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[2 * e] = bf16_bits_to_float(word[e] & 0xffffu), x[2 * e + 1] = bf16_bits_to_float(word[e] >> 16);
        ss = fmaf(x[2 * e], x[2 * e], fmaf(x[2 * e + 1], x[2 * e + 1], ss));
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float r = rsqrtf(ss * (1.f / kDim) + P.eps);
      const bool isq = h < P.hq;
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] *= r * (isq ? w[0][e] : w[1][e]);
      if (INTERLEAVED) {
        if (turns) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float a = x[2 * e], b = x[2 * e + 1];
            x[2 * e] = a * cosv[e] - b * sinv[e];
            x[2 * e + 1] = b * cosv[e] + a * sinv[e];
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float other = __shfl_sync(0xffffffffu, x[e], partner);
          if (turns) x[e] = x[e] * cosv[e] + other * sinv[e];
        }
      }
      __nv_bfloat16 *dst =
          isq ? P.qo + token * P.qos0 + h * P.qos1 : P.ko + token * P.kos0 + (h - P.hq) * P.kos1;
      *reinterpret_cast<uint4 *>(dst + 8 * lane) =
          make_uint4(pack_bf162(x[0], x[1]), pack_bf162(x[2], x[3]), pack_bf162(x[4], x[5]), pack_bf162(x[6], x[7]));
    }
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
  const int heads = hq + hkv;
  P.run = n * heads <= 148 * 16 ? 1 : std::min(heads, 8);
  P.runs = (heads + P.run - 1) / P.run;
  const int64_t blocks = (n * P.runs + kNrWarps - 1) / kNrWarps;
  if (blocks > INT32_MAX) return OSCAR_ERR_INVALID;
  if (interleaved)
    qk_norm_rope_kernel<true><<<(unsigned)blocks, 32 * kNrWarps, 0, (cudaStream_t)stream>>>(P);
  else
    qk_norm_rope_kernel<false><<<(unsigned)blocks, 32 * kNrWarps, 0, (cudaStream_t)stream>>>(P);
  OSCAR_CHECK_LAUNCH();
  return OSCAR_OK;
}
