// Products of few rows with weights in 4 bits, for gfx950:  y[m, n] = sum_k x[m, k] (c[n, k] - z[n, k / g]) s[n, k / g]
// c, z in 0..15, s bf16, groups of g = 32, 64 or 128 columns; x and y bf16, sums in fp32.
//
// Bound by the weights' bytes: each is read once by one wave and goes straight into a matrix product's A operand (16 weight rows),
// the x rows are its 16 columns.  A code becomes bf16 by being put in the mantissa of 128 (0x4300 | c = 128 + c, exact), two by
// one and-or; what that adds is taken off group by group, with the sum of the group's x from a product with ones:
//   sum x (c - z) = sum x (128 + c) - (128 + z) sum x
// The two sums are exact to fp32's 2^-24 of their size, 136 / 4.6 times the wanted one's at random codes: 2^-19, against the
// 2^-8 of y's own rounding.
//
// Weights are laid out once (ops.w4_pack): [N / 16][K / 128][lane][4] words, lane = 16 (k quarter) + row, word s the lane's eight
// columns 32 s + 8 (lane / 16) .. of the 128, column 2 i in nibble i, 2 i + 1 in nibble 4 + i: one 1 KB load of a wave is 16 rows x
// 128 columns.  Scales [N / 16][K / g][16] bf16, zeros (128 + z) the same in bytes.  The K axis is split over the waves of a
// workgroup, whose sums are added in LDS in the waves' order.
#include "block8.h"

namespace {

struct W4Args {
  bf16_t* y;
  const bf16_t* x;
  const raw4* w;
  const uint16_t* s;
  const uint8_t* z;
  int64_t ldy, ldx;
  int M, N, K, chunks;  // chunks of 128 columns, the last one perhaps not whole
};

__device__ __forceinline__ bf16x8_t codes_bf16(uint32_t w) {
  raw4 o;
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = ((w >> (4 * i)) & 0x000F000Fu) | 0x43004300u;
  return __builtin_bit_cast(bf16x8_t, o);
}

// RT: 16-row tiles of weights a wave; T: 16-row tiles of x; GS: k steps of 32 in a group
template <int RT, int T, int GS, bool ZERO>
__global__ void __launch_bounds__(512) w4_kernel(const W4Args a) {
  extern __shared__ __attribute__((aligned(16))) float red[];  // [waves][RT][T][16 tokens][16 rows]
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int r = lane & 15, q = lane >> 4;
  const int tiles = (a.N + 15) >> 4, nt0 = blockIdx.x * RT, m0 = blockIdx.y * (16 * T);
  constexpr int GC = 4 / GS;  // groups in a chunk
  const int groups = (a.K + 32 * GS - 1) / (32 * GS);
  const raw4 kOnes = {0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u};

  f32x4 acc[RT][T];
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int t = 0; t < T; ++t) acc[i][t] = f32x4{0.f, 0.f, 0.f, 0.f};

  const bf16_t* xp[T];
#pragma unroll
  for (int t = 0; t < T; ++t) xp[t] = a.x + (int64_t)min(m0 + 16 * t + r, a.M - 1) * a.ldx + 8 * q;

  struct Chunk {
    raw4 w[RT], x[T][4];
    raw2 s[RT][GC];
    uint32_t z[RT][GC];
  };
  auto load = [&](int kc, Chunk& c) {
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const int nt = min(nt0 + i, tiles - 1);
      c.w[i] = __builtin_nontemporal_load(a.w + ((int64_t)nt * a.chunks + kc) * 64 + lane);
#pragma unroll
      for (int g = 0; g < GC; ++g) {
        const int64_t at = ((int64_t)nt * groups + min(kc * GC + g, groups - 1)) * 16 + 4 * q;
        c.s[i][g] = *reinterpret_cast<const raw2*>(a.s + at);
        if constexpr (ZERO) c.z[i][g] = *reinterpret_cast<const uint32_t*>(a.z + at);
      }
    }
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int k = 128 * kc + 32 * s;
      const bool in = k < a.K;  // (K is a multiple of 32)
#pragma unroll
      for (int t = 0; t < T; ++t) {
        c.x[t][s] = *reinterpret_cast<const raw4*>(xp[t] + (in ? k : 0));
        if (!in) c.x[t][s] = raw4{0u, 0u, 0u, 0u};
      }
    }
  };
  auto compute = [&](const Chunk& c) {
#pragma unroll
    for (int g = 0; g < GC; ++g) {
      f32x4 xs[T];
#pragma unroll
      for (int t = 0; t < T; ++t) {
        xs[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = g * GS; s < (g + 1) * GS; ++s)
          xs[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, kOnes), __builtin_bit_cast(bf16x8_t, c.x[t][s]), xs[t], 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        f32x4 part[T];
#pragma unroll
        for (int t = 0; t < T; ++t) part[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = g * GS; s < (g + 1) * GS; ++s) {
          const bf16x8_t w = codes_bf16(c.w[i][s]);
#pragma unroll
          for (int t = 0; t < T; ++t) part[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, __builtin_bit_cast(bf16x8_t, c.x[t][s]), part[t], 0, 0, 0);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float sc = e & 1 ? bf16hi(c.s[i][g][e >> 1]) : bf16lo(c.s[i][g][e >> 1]);
          const float zc = ZERO ? (float)((c.z[i][g] >> (8 * e)) & 0xffu) : 136.f;
#pragma unroll
          for (int t = 0; t < T; ++t) acc[i][t][e] += sc * (part[t][e] - zc * xs[t][e]);
        }
      }
    }
  };
  Chunk c0, c1;
  int kc = wid;
  if (kc < a.chunks) load(kc, c0);
  while (kc < a.chunks) {
    if (kc + waves < a.chunks) load(kc + waves, c1);
    compute(c0);
    kc += waves;
    if (kc >= a.chunks) break;
    if (kc + waves < a.chunks) load(kc + waves, c0);
    compute(c1);
    kc += waves;
  }
  // lane (q, r): rows 4 q + e of a tile, token r
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int t = 0; t < T; ++t) *reinterpret_cast<f32x4*>(red + (((wid * RT + i) * T + t) * 16 + r) * 16 + 4 * q) = acc[i][t];
  __syncthreads();
  for (int o = threadIdx.x; o < RT * T * 256; o += blockDim.x) {
    const int n = o & 15, i = (o >> 4) % RT, m = (o >> 4) / RT;  // rows of tiles next to each other, then tokens
    const int row = 16 * (nt0 + i) + n, tok = m0 + m;
    if (row >= a.N || tok >= a.M) continue;
    float sum = 0.f;
    for (int w = 0; w < waves; ++w) sum += red[(((w * RT + i) * T + (m >> 4)) * 16 + (m & 15)) * 16 + n];
    a.y[(int64_t)tok * a.ldy + row] = f32_to_bf16(sum);
  }
}

template <int RT, int T, int GS, bool ZERO> int launch(const W4Args& a, int waves, hipStream_t st) {
  const size_t lds = (size_t)waves * RT * T * 1024;
  if (lds > 64 * 1024) return -3;
  const dim3 grid(((a.N + 15) / 16 + RT - 1) / RT, (a.M + 16 * T - 1) / (16 * T));
  w4_kernel<RT, T, GS, ZERO><<<grid, 64 * waves, lds, st>>>(a);
  return (int)hipGetLastError();
}

template <int RT, int T> int launch_group(const W4Args& a, int group, int waves, hipStream_t st) {
  const bool z = a.z != nullptr;
  switch (group) {
    case 32: return z ? launch<RT, T, 1, true>(a, waves, st) : launch<RT, T, 1, false>(a, waves, st);
    case 64: return z ? launch<RT, T, 2, true>(a, waves, st) : launch<RT, T, 2, false>(a, waves, st);
    case 128: return z ? launch<RT, T, 4, true>(a, waves, st) : launch<RT, T, 4, false>(a, waves, st);
  }
  return -1;
}

}  // namespace

extern "C" int dx_w4_gemm(void* y, int64_t ldy, const void* x, int64_t ldx, const void* w, const void* s, const void* z, int M, int N, int K,
                          int group, hipStream_t stream) {
  if (M < 0 || N < 1 || K < 32 || K % group || ldx % 8) return -1;
  if (M == 0) return 0;
  W4Args a{};
  a.y = (bf16_t*)y, a.x = (const bf16_t*)x, a.w = (const raw4*)w, a.s = (const uint16_t*)s, a.z = (const uint8_t*)z;
  a.ldy = ldy, a.ldx = ldx, a.M = M, a.N = N, a.K = K, a.chunks = (K + 127) / 128;
  int waves = 8;
  while (waves > 1 && waves > a.chunks) waves >>= 1;
  if (M <= 16) return launch_group<1, 1>(a, group, waves, stream);
  if (M <= 32) return launch_group<1, 2>(a, group, waves, stream);
  return launch_group<1, 4>(a, group, waves, stream);
}
