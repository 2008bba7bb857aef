// Products of few rows with weights in 4 bits, for gfx950:  y[m, n] = sum_k x[m, k] (c[n, k] - z[n, k / g]) s[n, k / g]
// c, z in 0..15, s bf16, groups of g = 32, 64 or 128 columns; x and y bf16, sums in fp32.
//
// Bound by the weights' bytes: each is read once by one wave and goes straight into a matrix product's B operand (16 weight rows),
// the x rows are the rows of A.  A code becomes bf16 by being put in the mantissa of 128 (0x4300 | c = 128 + c, exact), two by
// one and-or; what that adds is taken off group by group, with the sum of the group's x from a product with ones:
//   sum x (c - z) = sum x (128 + c) - (128 + z) sum x
// The two sums are off by 2^-24 of their size an addition.  Beside the wanted sum that size is 136 / 4.6 where x has mean zero and codes are
// random (2^-19, against the 2^-8 of y's own rounding), and grows with the root of the group where x has a common part: 136 sqrt(128) / 4.6,
// 330 times (2^-15).  Where x is infinite, or so large that 143 x is, they leave no number, and the result is summed column by column.
//
// Weights are laid out once (ops.w4_pack): [N / 16][K / 128][lane][4] words, lane = 16 (k quarter) + row, word s the lane's eight
// columns 32 s + 8 (lane / 16) .. of the 128, column 2 i in nibble i, 2 i + 1 in nibble 4 + i: one 1 KB load of a wave is 16 rows x
// 128 columns.  Scales [N / 16][K / 128][row][group] bf16, zeros (128 + z) the same in bytes: a lane's products are all of one row.
// The K axis is split over the waves of a workgroup, whose sums are added in LDS in the waves' order, and over workgroups where rows
// are few (their sums in fp32, added by a second kernel).  x rows come from L2 once for RT tiles.
//
// One row of 4096 x 4096 4.4 us, of 28672 x 4096 (groups of 64, zeros) 13.5 (4.7 TB/s of weights), 16 rows of 4096 x 14336 (groups of 32,
// zeros) 14.3, of which the joined halves of K take 2.4: the latency of seven chunks a wave.
//
// More than 16 rows are bands of 16, workgroups of their own, while there is little work; then (w4_wide_kernel) x would come from L2 more often
// than the weights from HBM (64 rows of 28672 x 4096 50 us, now 31), so a workgroup's eight waves, four tile pairs by two halves of
// 256 columns, read it from LDS, staged a step ahead.
#include "block8.h"

#include <type_traits>

namespace {

struct W4Args {
  bf16_t* y;
  float* ws;  // [splits][M][N], where K is split over workgroups
  const bf16_t* x;
  const raw4* w;
  const uint16_t* s;
  const uint8_t* z;
  int64_t ldy, ldx;
  int M, N, K, chunks;  // chunks of 128 columns, the last one perhaps not whole
};

// (`base` is 0x43004300 in a vector register: with both constants in scalar ones the and-or would be two instructions)
__device__ __forceinline__ bf16x8_t codes_bf16(uint32_t w, uint32_t base) {
  raw4 o;
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = ((w >> (4 * i)) & 0x000F000Fu) | base;
  return __builtin_bit_cast(bf16x8_t, o);
}

__device__ __forceinline__ bool finite(float x) { return fabsf(x) < INFINITY; }

// A result by its definition, column by column, over the chunks of 128 columns that a workgroup has (`per` of them side by side): where x is
// infinite, or 143 x is, (128 + c) x and (128 + z) x leave no number between them.  Only such results come here.
template <int GS, bool ZERO> __device__ __forceinline__ float sum_by_column(const W4Args& a, int row, int tok, int per) {
  constexpr int GC = 4 / GS;
  const bf16_t* x = a.x + (int64_t)tok * a.ldx;
  float sum = 0.f;
  for (int c0 = per * blockIdx.z; c0 < a.chunks; c0 += per * gridDim.z)
    for (int c = c0; c < min(c0 + per, a.chunks); ++c) {
      const int64_t at = (int64_t)(row >> 4) * a.chunks + c;
      for (int s = 0; s < 4 && 128 * c + 32 * s < a.K; ++s) {
        const int64_t group = (at * 16 + (row & 15)) * GC + s / GS;
        const float sc = bf16lo((uint32_t)a.s[group]), zc = ZERO ? (float)a.z[group] - 128.f : 8.f;
        for (int q = 0; q < 4; ++q) {
          const uint32_t w = reinterpret_cast<const uint32_t*>(a.w + at * 64 + 16 * q + (row & 15))[s];
          for (int e = 0; e < 8; ++e) {
            const float code = (float)((w >> (4 * (e / 2 + 4 * (e & 1)))) & 15u);
            sum += bf16lo((uint32_t)*reinterpret_cast<const uint16_t*>(x + 128 * c + 32 * s + 8 * q + e)) * ((code - zc) * sc);
          }
        }
        if (sum != sum) return sum;  // (and so it stays)
      }
    }
  return sum;
}

// RT: 16-row tiles of weights a wave; T: tiles of 4 E rows of x (E of every four rows of A); GS: k steps of 32 in a group; DW: chunks on
// their way
template <int RT, int T, int E, int GS, bool ZERO, int DW>
__global__ void __launch_bounds__(512) w4_kernel(const W4Args a) {
  extern __shared__ __attribute__((aligned(16))) float red[];  // [waves][RT][T][4 E tokens][16 rows]
  static_assert(DW % 2 == 0, "x alternates between two places");
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int r = lane & 15, q = lane >> 4;
  const int tiles = (a.N + 15) >> 4, nt0 = blockIdx.x * RT, m0 = blockIdx.y * (4 * E * T);
  constexpr int GC = 4 / GS;  // groups in a chunk
  uint32_t base = 0x43004300u;
  asm("" : "+v"(base));
  const raw4 kOnes = {0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u};

  float acc[RT][T][E];
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int e = 0; e < E; ++e) acc[i][t][e] = 0.f;

  struct Chunk {
    raw4 w[RT];
    uint32_t s[RT][(GC + 1) / 2], z[RT];
  };
  struct Rows {
    raw4 x[T][4];
  };
  const bf16_t* xp[T];  // row 4 i + j of A is token E i + j % E
#pragma unroll
  for (int t = 0; t < T; ++t) xp[t] = a.x + (int64_t)min(m0 + 4 * E * t + E * (r >> 2) + (r & (E - 1)), a.M - 1) * a.ldx + 8 * q;
  int64_t tile_at[RT];  // first chunk of a tile (one behind the last is the last again, and goes nowhere)
#pragma unroll
  for (int i = 0; i < RT; ++i) tile_at[i] = (int64_t)min(nt0 + i, tiles - 1) * a.chunks;
  const int step = waves * gridDim.z, first = wid + waves * blockIdx.z;  // this wave's chunks: first, first + step, ..
  const int n = a.chunks > first ? (a.chunks - first + step - 1) / step : 0;
  auto load_w = [&](int j, Chunk& c) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const int64_t at = tile_at[i] + first + j * step;
      c.w[i] = __builtin_nontemporal_load(a.w + at * 64 + lane);
      const uint16_t* s = a.s + (at * 16 + r) * GC;
      const uint8_t* z = a.z + (at * 16 + r) * GC;
      if constexpr (GC == 1) {
        c.s[i][0] = *s;
        if constexpr (ZERO) c.z[i] = *z;
      } else if constexpr (GC == 2) {
        c.s[i][0] = *reinterpret_cast<const uint32_t*>(s);
        if constexpr (ZERO) c.z[i] = *reinterpret_cast<const uint16_t*>(z);
      } else {
        const raw2 v = *reinterpret_cast<const raw2*>(s);
        c.s[i][0] = v[0], c.s[i][1] = v[1];
        if constexpr (ZERO) c.z[i] = *reinterpret_cast<const uint32_t*>(z);
      }
    }
  };
  auto load_x = [&](int j, Rows& c) __attribute__((always_inline)) {
    const int k0 = 128 * (first + j * step);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int k = k0 + 32 * s < a.K ? k0 + 32 * s : 0;  // (behind the columns, whose scales are 0, any x of the row will do)
#pragma unroll
      for (int t = 0; t < T; ++t) c.x[t][s] = *reinterpret_cast<const raw4*>(xp[t] + k);
    }
  };
  auto compute = [&](const Chunk& c, const Rows& y) __attribute__((always_inline)) {
#pragma unroll
    for (int g = 0; g < GC; ++g) {
      f32x4 xs[T];
#pragma unroll
      for (int t = 0; t < T; ++t) {
        xs[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = g * GS; s < (g + 1) * GS; ++s)
          xs[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, y.x[t][s]), __builtin_bit_cast(bf16x8_t, kOnes), xs[t], 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        f32x4 part[T];
#pragma unroll
        for (int t = 0; t < T; ++t) part[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = g * GS; s < (g + 1) * GS; ++s) {
          const bf16x8_t w = codes_bf16(c.w[i][s], base);
#pragma unroll
          for (int t = 0; t < T; ++t) part[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, y.x[t][s]), w, part[t], 0, 0, 0);
        }
        const float sc = g & 1 ? bf16hi(c.s[i][g >> 1]) : bf16lo(c.s[i][g >> 1]);
        const float zc = ZERO ? (float)((c.z[i] >> (8 * g)) & 0xffu) : 136.f;
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
          for (int e = 0; e < E; ++e) acc[i][t][e] += sc * (part[t][e] - zc * xs[t][e]);
      }
    }
  };
  if (n > 0) {
    Chunk c[DW];
    Rows y[2];
#pragma unroll
    for (int u = 0; u < DW - 1; ++u) load_w(min(u, n - 1), c[u]);
    load_x(0, y[0]);
    int j = 0;
    for (; j + 2 * DW - 1 <= n; j += DW) {  // (no load of these lies in a branch: each is waited for by count)
#pragma unroll
      for (int u = 0; u < DW; ++u) {
        load_x(j + u + 1, y[(u + 1) & 1]);
        load_w(j + u + DW - 1, c[(u + DW - 1) % DW]);
        __builtin_amdgcn_sched_barrier(0);
        compute(c[u], y[u & 1]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    for (; j < n; j += DW)
#pragma unroll
      for (int u = 0; u < DW; ++u)
        if (j + u < n) {
          if (j + u + 1 < n) load_x(j + u + 1, y[(u + 1) & 1]);
          if (j + u + DW - 1 < n) load_w(j + u + DW - 1, c[(u + DW - 1) % DW]);
          compute(c[u], y[u & 1]);
        }
  }
  // lane (q, r): tokens E q + e of row r
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int e = 0; e < E; ++e) red[((wid * RT + i) * T + t) * (64 * E) + (E * q + e) * 16 + r] = acc[i][t][e];
  __syncthreads();
  for (int o = threadIdx.x; o < RT * T * E * 64; o += blockDim.x) {
    const int i = o / (T * E * 64), in = o % (T * E * 64);  // (in: token, then row)
    const int row = 16 * (nt0 + i) + (o & 15), tok = m0 + (in >> 4);
    if (row >= a.N || tok >= a.M) continue;
    float sum = 0.f;
    for (int w = 0; w < waves; ++w) sum += red[w * (RT * T * E * 64) + o];
    if (!finite(sum)) sum = sum_by_column<GS, ZERO>(a, row, tok, waves);
    if (gridDim.z == 1) a.y[(int64_t)tok * a.ldy + row] = f32_to_bf16(sum);
    else a.ws[((int64_t)blockIdx.z * a.M + tok) * a.N + row] = sum;
  }
}

// 16 T rows of x; waves: four pairs of 16-row weight tiles by the two chunks of a step of 256 columns
template <int T, int GS, bool ZERO>
__global__ void __launch_bounds__(512) w4_wide_kernel(const W4Args a) {
  constexpr int RT = 2, GC = 4 / GS, XN = T;  // 16-byte pieces of x a thread stages in a step
  __shared__ __attribute__((aligned(16))) raw4 img[2][16 * T * 32];  // [row][piece ^ row % 16]: a wave's reads meet all banks
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, q = lane >> 4, half = wid >> 2;
  const int tiles = (a.N + 15) >> 4, nt0 = (blockIdx.x * 4 + (wid & 3)) * RT, m0 = blockIdx.y * (16 * T);
  uint32_t base = 0x43004300u;
  asm("" : "+v"(base));
  const raw4 kOnes = {0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u};
  f32x4 acc[RT][T];
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int t = 0; t < T; ++t) acc[i][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  struct Chunk {
    raw4 w[RT];
    uint32_t s[RT][(GC + 1) / 2], z[RT];
  };
  int64_t tile_at[RT];
#pragma unroll
  for (int i = 0; i < RT; ++i) tile_at[i] = (int64_t)min(nt0 + i, tiles - 1) * a.chunks;
  const int pairs = (a.chunks + 1) >> 1, first = blockIdx.z, step = gridDim.z;
  const int n = pairs > first ? (pairs - first + step - 1) / step : 0;
  const bf16_t* xp[XN];
  int col[XN], to[XN];
#pragma unroll
  for (int i = 0; i < XN; ++i) {
    const int at = threadIdx.x + 512 * i, row = at >> 5, piece = at & 31;
    xp[i] = a.x + (int64_t)min(m0 + row, a.M - 1) * a.ldx;
    col[i] = 8 * piece;
    to[i] = row * 32 + (piece ^ (row & 15));
  }
  raw4 xr[XN];
  auto load = [&](int j, Chunk& c) __attribute__((always_inline)) {
    const int pair = first + min(j, n - 1) * step;
    const int kc = min(2 * pair + half, a.chunks - 1);
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const int64_t at = tile_at[i] + kc;
      c.w[i] = __builtin_nontemporal_load(a.w + at * 64 + lane);
      const uint16_t* s = a.s + (at * 16 + r) * GC;
      const uint8_t* z = a.z + (at * 16 + r) * GC;
      if constexpr (GC == 1) {
        c.s[i][0] = *s;
        if constexpr (ZERO) c.z[i] = *z;
      } else if constexpr (GC == 2) {
        c.s[i][0] = *reinterpret_cast<const uint32_t*>(s);
        if constexpr (ZERO) c.z[i] = *reinterpret_cast<const uint16_t*>(z);
      } else {
        const raw2 v = *reinterpret_cast<const raw2*>(s);
        c.s[i][0] = v[0], c.s[i][1] = v[1];
        if constexpr (ZERO) c.z[i] = *reinterpret_cast<const uint32_t*>(z);
      }
    }
#pragma unroll
    for (int i = 0; i < XN; ++i) {
      const int k = 256 * pair + col[i];
      xr[i] = *reinterpret_cast<const raw4*>(xp[i] + (k < a.K ? k : 0));  // (behind the columns, whose scales are 0, any x of the row will do)
    }
  };
  auto store = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < XN; ++i) img[buf][to[i]] = xr[i];
  };
  auto compute = [&](const Chunk& c, const raw4* x) __attribute__((always_inline)) {
#pragma unroll
    for (int g = 0; g < GC; ++g) {
      f32x4 xs[T], part[RT][T];
#pragma unroll
      for (int t = 0; t < T; ++t) {
        xs[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < RT; ++i) part[i][t] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
#pragma unroll
      for (int s = g * GS; s < (g + 1) * GS; ++s) {
        bf16x8_t w[RT];
#pragma unroll
        for (int i = 0; i < RT; ++i) w[i] = codes_bf16(c.w[i][s], base);
#pragma unroll
        for (int t = 0; t < T; ++t) {
          const bf16x8_t f = __builtin_bit_cast(bf16x8_t, x[(16 * t + r) * 32 + ((16 * half + 4 * s + q) ^ r)]);
          xs[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f, __builtin_bit_cast(bf16x8_t, kOnes), xs[t], 0, 0, 0);
#pragma unroll
          for (int i = 0; i < RT; ++i) part[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f, w[i], part[i][t], 0, 0, 0);
        }
      }
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        const float sc = g & 1 ? bf16hi(c.s[i][g >> 1]) : bf16lo(c.s[i][g >> 1]);
        const float zc = ZERO ? (float)((c.z[i] >> (8 * g)) & 0xffu) : 136.f;
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][t][e] += sc * (part[i][t][e] - zc * xs[t][e]);
      }
    }
  };
  if (n > 0) {
    Chunk c[2];
    load(0, c[0]);
    store(0);
    __syncthreads();
    auto turn = [&](auto now_, int j) __attribute__((always_inline)) {
      constexpr int now = decltype(now_)::value;
      load(j + 1, c[now ^ 1]);
      __builtin_amdgcn_sched_barrier(0);
      if (2 * (first + j * step) + half < a.chunks) compute(c[now], img[now]);
      __builtin_amdgcn_sched_barrier(0);
      store(now ^ 1);
      __syncthreads();
    };
    for (int j = 0; j < n; j += 2) {
      turn(std::integral_constant<int, 0>{}, j);
      if (j + 1 < n) turn(std::integral_constant<int, 1>{}, j + 1);
    }
  }
  // the second half's sums to the first; lane (q, r): tokens 4 q + e of row r
  f32x4* red = reinterpret_cast<f32x4*>(img);
  __syncthreads();
  if (half) {
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int t = 0; t < T; ++t) red[(((wid & 3) * RT + i) * T + t) * 64 + lane] = acc[i][t];
  }
  __syncthreads();
  if (half) return;
  bool odd = false;
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int t = 0; t < T; ++t) {
      acc[i][t] += red[((wid * RT + i) * T + t) * 64 + lane];
      const int row = 16 * (nt0 + i) + r;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int tok = m0 + 16 * t + 4 * q + e;
        if (row < a.N && tok < a.M) {
          if (gridDim.z == 1) a.y[(int64_t)tok * a.ldy + row] = f32_to_bf16(acc[i][t][e]);
          else a.ws[((int64_t)blockIdx.z * a.M + tok) * a.N + row] = acc[i][t][e];
          odd |= !finite(acc[i][t][e]);
        }
      }
    }
  if (!odd) return;
#pragma unroll 1
  for (int o = 0; o < RT * T * 4; ++o) {  // (a lane's results once more: the sums are in registers, which have no number at run time)
    const int row = 16 * (nt0 + o / (T * 4)) + r, tok = m0 + 16 * (o / 4 % T) + 4 * q + o % 4;
    if (row >= a.N || tok >= a.M) continue;
    bf16_t* y = a.y + (int64_t)tok * a.ldy + row;
    float* part = a.ws + ((int64_t)blockIdx.z * a.M + tok) * a.N + row;
    if (finite(gridDim.z == 1 ? bf16lo((uint32_t)*reinterpret_cast<const uint16_t*>(y)) : *part)) continue;
    const float sum = sum_by_column<GS, ZERO>(a, row, tok, 2);
    if (gridDim.z == 1) *y = f32_to_bf16(sum);
    else *part = sum;
  }
}

// y = the splits' sums, in their order
__global__ void __launch_bounds__(256) w4_sum_kernel(bf16_t* __restrict__ y, int64_t ldy, const float* __restrict__ ws, int M, int N, int splits) {
  const int n = blockIdx.x * 256 + threadIdx.x, m = blockIdx.y;
  if (n >= N) return;
  float sum = 0.f;
#pragma unroll 8
  for (int s = 0; s < splits; ++s) sum += ws[((int64_t)s * M + m) * N + n];
  y[(int64_t)m * ldy + n] = f32_to_bf16(sum);
}

template <int RT, int T, int E, int GS, bool ZERO> int launch(const W4Args& a, int waves, int splits, hipStream_t st) {
  const size_t lds = (size_t)waves * RT * T * E * 256;
  if (lds > 64 * 1024 || waves < 1 || waves > 8 || splits < 1 || (splits > 1 && a.ws == nullptr)) return -3;
  const dim3 grid(((a.N + 15) / 16 + RT - 1) / RT, (a.M + 4 * E * T - 1) / (4 * E * T), splits);
  w4_kernel<RT, T, E, GS, ZERO, 2><<<grid, 64 * waves, lds, st>>>(a);
  if (splits > 1) w4_sum_kernel<<<dim3((a.N + 255) / 256, a.M), 256, 0, st>>>(a.y, a.ldy, a.ws, a.M, a.N, splits);
  return (int)hipGetLastError();
}

template <int RT, int T, int E> int launch_group(const W4Args& a, int group, int waves, int splits, hipStream_t st) {
  const bool z = a.z != nullptr;
  switch (group) {
    case 32: return z ? launch<RT, T, E, 1, true>(a, waves, splits, st) : launch<RT, T, E, 1, false>(a, waves, splits, st);
    case 64: return z ? launch<RT, T, E, 2, true>(a, waves, splits, st) : launch<RT, T, E, 2, false>(a, waves, splits, st);
    case 128: return z ? launch<RT, T, E, 4, true>(a, waves, splits, st) : launch<RT, T, E, 4, false>(a, waves, splits, st);
  }
  return -1;
}

template <int T> int launch_wide(const W4Args& a, int group, int splits, hipStream_t st) {
  const dim3 grid(((a.N + 15) / 16 + 7) / 8, (a.M + 16 * T - 1) / (16 * T), splits);
  const bool z = a.z != nullptr;
#define DX_W4W(GS)                                                  \
  do {                                                              \
    if (z) w4_wide_kernel<T, GS, true><<<grid, 512, 0, st>>>(a);    \
    else w4_wide_kernel<T, GS, false><<<grid, 512, 0, st>>>(a);     \
  } while (0)
  switch (group) {
    case 32: DX_W4W(1); break;
    case 64: DX_W4W(2); break;
    case 128: DX_W4W(4); break;
    default: return -1;
  }
#undef DX_W4W
  if (splits > 1) w4_sum_kernel<<<dim3((a.N + 255) / 256, a.M), 256, 0, st>>>(a.y, a.ldy, a.ws, a.M, a.N, splits);
  return (int)hipGetLastError();
}

}  // namespace

extern "C" int dx_w4_gemm(void* y, int64_t ldy, const void* x, int64_t ldx, const void* w, const void* s, const void* z, float* ws, int M, int N, int K,
                          int group, int waves, int rt, int splits, hipStream_t stream) {
  if (M < 0 || N < 1 || K < 32 || K % group || ldx % 8) return -1;
  if (M == 0) return 0;
  W4Args a{};
  a.y = (bf16_t*)y, a.ws = ws, a.x = (const bf16_t*)x, a.w = (const raw4*)w, a.s = (const uint16_t*)s, a.z = (const uint8_t*)z;
  a.ldy = ldy, a.ldx = ldx, a.M = M, a.N = N, a.K = K, a.chunks = (K + 127) / 128;
#define DX_W4(T_, E_)                                                                        \
  do {                                                                                       \
    if (rt == 4) return launch_group<4, T_, E_>(a, group, waves, splits, stream);            \
    if (rt == 2) return launch_group<2, T_, E_>(a, group, waves, splits, stream);            \
    return launch_group<1, T_, E_>(a, group, waves, splits, stream);                         \
  } while (0)
  if (splits < 1 || (splits > 1 && ws == nullptr)) return -3;
  if (rt > 0) {
    if (M <= 4) DX_W4(1, 1);
    if (M <= 8) DX_W4(1, 2);
    DX_W4(1, 4);
  }
  return M <= 32 ? launch_wide<2>(a, group, splits, stream) : launch_wide<4>(a, group, splits, stream);
#undef DX_W4
}
