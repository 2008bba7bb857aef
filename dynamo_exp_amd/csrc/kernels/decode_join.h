// Flash-decoding's balanced parts and the join of them, for the decode kernels whose heads are 128 wide.
#pragma once
#include "common.h"

namespace {

constexpr int kHeadDim = 128;

// tokens per partition when a context of ctx tokens is split into n balanced
// parts, rounded up to `align` (the workgroup's 4-wave chunk stride), or to
// half or a quarter of it where a part is no longer: a CU takes 55 cycles for
// a KB of K or V however its lanes lie, so a part of 128 tokens holds its CU
// for 3500 while most of the chip has none.  Eight layers in a graph, one
// sequence of 700 tokens 71 -> 64 us; four layers, one of 150 36.4 -> 33.7,
// two of 500 44.6 -> 36.6, four of 700 45.6 -> 40.0, 32 / 8 heads.
__device__ __forceinline__ int balanced_part(int ctx, int n, int align) {
  const int per = (ctx + n - 1) / n;
  align = per <= align / 4 ? align / 4 : per <= align / 2 ? align / 2 : align;
  return (per + align - 1) / align * align;
}

// (the callers' rows have their elements' alignment, no more)
typedef float f32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef float f32x2_a4 __attribute__((ext_vector_type(2), aligned(4)));
typedef unsigned int u32x2_a2 __attribute__((ext_vector_type(2), aligned(2)));

// merge flash-decoding partitions: grid (Hq, B), block kHeadDim threads.  Latency-bound (a head's parts are a few KB): the
// context, the parts' (m, l) and the first 4 AHEAD parts' rows are all asked for at once, whether the parts exist or not, and
// four groups of 32 lanes x 4 columns sum every fourth part.  In a captured step, a layer's attention at 32 / 8 heads, us,
// part by part with one column a thread before: one sequence of 700 tokens 10.5 -> 9.3, of 4000 19.6 -> 11.1, four of
// 1500 15.7 -> 12.5.
template <int AHEAD>
__global__ void __launch_bounds__(kHeadDim) decode_reduce_kernel(bf16_t* __restrict__ out, const float* __restrict__ tmp_out,
                                                          const float* __restrict__ tmp_ml,
                                                          const int* __restrict__ ctx_lens, int n_parts, int align, int most) {
  __shared__ __attribute__((aligned(16))) f32x4 other[kHeadDim / 4];
  const int qh = blockIdx.x, b = blockIdx.y, nqh = gridDim.x;
  const int lane = threadIdx.x & 63, grp = threadIdx.x >> 5, col = 4 * (threadIdx.x & 31);
  const int64_t row0 = ((int64_t)b * nqh + qh) * n_parts;
  const f32x2_a4* ml = reinterpret_cast<const f32x2_a4*>(tmp_ml) + row0;
  const float* rows = tmp_out + row0 * kHeadDim + col;
  const f32x2_a4 first = ml[min(lane, n_parts - 1)];
  f32x4 x[AHEAD];
#pragma unroll
  for (int k = 0; k < AHEAD; ++k) x[k] = *reinterpret_cast<const f32x4_a4*>(rows + (int64_t)min(grp + 4 * k, n_parts - 1) * kHeadDim);
  const int ctx = min(ctx_lens[b], most);
  bf16_t* o = out + ((int64_t)b * nqh + qh) * kHeadDim + col;
  if (ctx <= 0) {  // a graph bucket's padding row (context 0): no partition wrote it
    if (grp == 0) *reinterpret_cast<u32x2_a2*>(o) = u32x2_a2{0u, 0u};
    return;
  }
  const int part_size = balanced_part(ctx, n_parts, align);
  const int np = min((ctx + part_size - 1) / part_size, n_parts);
  float M = lane < np ? first.x : -1e30f;
  for (int p = lane + 64; p < np; p += 64) M = fmaxf(M, ml[p].x);
  M = wave_reduce_max(M);
  const float w0 = lane < np ? exp2f(first.x - M) * first.y : 0.f;
  float den = w0;
  for (int p = lane + 64; p < np; p += 64) den += exp2f(ml[p].x - M) * ml[p].y;
  den = wave_reduce_sum(den);
  f32x4 num = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int k = 0; k < AHEAD; ++k) {
    const float w = __shfl(w0, grp + 4 * k, 64);
    if (grp + 4 * k < np) num += w * x[k];  // (a part that does not exist may hold anything)
  }
  for (int p0 = 4 * AHEAD; p0 < np; p0 += 16)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int p = p0 + grp + 4 * k, q = min(p, np - 1);
      const f32x4 y = *reinterpret_cast<const f32x4_a4*>(rows + (int64_t)q * kHeadDim);
      float w = __shfl(w0, q & 63, 64);
      if (p0 >= 64) w = exp2f(ml[q].x - M) * ml[q].y;
      if (p < np) num += w * y;
    }
#pragma unroll
  for (int i = 0; i < 4; ++i) num[i] = halves_sum(num[i]);
  if (grp == 2) other[threadIdx.x & 31] = num;
  __syncthreads();
  if (grp) return;
  num += other[threadIdx.x];
  u32x2_a2 pk = {0u, 0u};
  if (den != 0.f) pk = u32x2_a2{pack_bf16x2(num[0] / den, num[1] / den), pack_bf16x2(num[2] / den, num[3] / den)};
  *reinterpret_cast<u32x2_a2*>(o) = pk;
}

// (with few parts the rows that are not there only cost time: 44 sequences of 76 tokens in two parts, three layers 41.5 us
// asking for 16, 43.0 for 32)
// most: the length that longer contexts were cut to)
inline void join(bf16_t* out, const float* tmp_out, const float* tmp_ml, const int* ctx, int n_q_heads, int batch, int n_parts, int align,
                 hipStream_t st, int most = 0x7fffffff) {
  const dim3 grid(n_q_heads, batch);
  if (n_parts > 16) decode_reduce_kernel<8><<<grid, kHeadDim, 0, st>>>(out, tmp_out, tmp_ml, ctx, n_parts, align, most);
  else decode_reduce_kernel<4><<<grid, kHeadDim, 0, st>>>(out, tmp_out, tmp_ml, ctx, n_parts, align, most);
}

}  // namespace
