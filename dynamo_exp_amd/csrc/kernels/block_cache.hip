// Rotary positions and the append to the 8-bit KV cache whose scales belong to a block and head (block8.h), and the read-back
// of its blocks as bf16, for gfx950.
//
// Of a run of tokens that goes into one block (offsets o .. o + n - 1), with a = max |x| over the run's finite values of one
// head's K (rotated, in fp32) or V:
//   need = the smallest power of two with a <= M need (M = 127 or 448),  new = max(old, need)  (old: 0 where o = 0)
//   codes = round_half_even(x / new);  where new != old the o rows in front become round(code old / new)
// A power of two makes every step of this exact but the roundings themselves: e4m3 codes move without loss (but for its
// subnormals), and a move at least doubles an int8 block's step, so all of a code's roundings sum to less than one step.  The
// exponent comes from the bits of a, no division is near a border.
//
// A unit is one run's K or V of one head, in a workgroup: eight lanes a row, each with eight columns of either half, the rows
// of a block in registers between the maximum and the rounding, so each value is read once.  Runs are found where the slots
// stop rising by one: a workgroup looks a window of tokens over at once and takes the runs that begin in it, those of at most
// eight rows (decode steps') a wave each, side by side.  Windows of 32 tokens, 4 where tokens are few: a window in which no run
// begins costs its workgroup a launch and a load, 1 us of a CU's five places (6520 tokens of 8 heads in blocks of 64, windows of 8
// and no runs a wave: 25 us for K and V; now 21, and 36 with Q of 32 heads, which is a copy and takes 19 of its own: 3.3 TB/s).  64 tokens of
// 64 sequences: 4.6 us, the latency of slots, rows, positions and table in turn.
#include "block8.h"

namespace {

constexpr int D = 128, kThreads = 256;
constexpr int kRows = kThreads / 8;  // rows of a pass
constexpr int kMostBlock = 128;

// smallest 2^e with a <= most 2^e, e >= -126 (a finite, >= 0)
template <int CODE> __device__ __forceinline__ float power_scale(float a) {
  // a = m 2^k, m in [0.5, 1); 127 = 0.9921875 2^7, 448 = 0.875 2^9
  constexpr uint32_t kTop = CODE == kInt8 ? 0x7E0000u : 0x600000u;
  constexpr int kExp = CODE == kInt8 ? 7 : 9;
  const uint32_t b = __float_as_uint(a);
  const int k = (int)(b >> 23) - 126;
  const int e = k - kExp + ((b & 0x7FFFFFu) > kTop ? 1 : 0);
  return __uint_as_float((uint32_t)(max(e, -126) + 127) << 23);
}

// four values (already over the scale) as codes: half-even; int8 keeps +-127 and has no NaN (0), e4m3 keeps +-448
template <int CODE> __device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
  auto cl = [](float x) {
    constexpr float m = CODE == kInt8 ? 127.f : 448.f;
    const float y = fminf(fmaxf(x, -m), m);
    if constexpr (CODE == kInt8) return x == x ? y : 0.f;
    return x == x ? y : x;
  };
  if constexpr (CODE == kE4m3) {
    const int w = __builtin_amdgcn_cvt_pk_fp8_f32(cl(a), cl(b), 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(cl(c), cl(d), w, true);
  } else {
    auto q = [&](float x) { return (uint32_t)(int)rintf(cl(x)) & 0xffu; };
    return q(a) | q(b) << 8 | q(c) << 16 | q(d) << 24;
  }
}

struct AppendArgs {
  const bf16_t *q, *k, *v;       // rows of heads, `stride` elements apart
  bf16_t* q_out;                 // rotated Q (rows q_out_stride apart); nullptr: no Q here
  const void* positions;         // (not read without cos_sin)
  const float* cos_sin;          // [positions, 128]; nullptr: K as it comes
  const float* row_scale;        // nullptr, or a factor of every row
  const int64_t* slots;          // nullptr: nothing is appended
  uint8_t *k_codes, *v_codes;
  float *k_scales, *v_scales;
  int64_t stride, q_out_stride;
  int64_t num_slots;
  int tokens, n_q, n_kv, bs_shift, pos_i64, rotate_q, units_x, window, last_position;
};

__device__ __forceinline__ int64_t position(const AppendArgs& g, int64_t t) {
  const int64_t p = g.pos_i64 ? static_cast<const int64_t*>(g.positions)[t] : (int64_t)static_cast<const int32_t*>(g.positions)[t];
  return min(max(p, (int64_t)0), (int64_t)g.last_position);  // (a row of the table, whatever is asked for)
}

// one run: by a workgroup, or (WAVE) n rows by a wave
template <int CODE, int PASSES, bool WAVE>
__device__ __forceinline__ void append_run(const AppendArgs& g, int64_t t0, int64_t slot, int n, int head, int is_v, float* red) {
  constexpr int STEP = WAVE ? 8 : kRows;  // rows of a pass
  const int bs = 1 << g.bs_shift, lane = threadIdx.x & 63, row = (WAVE ? lane : (int)threadIdx.x) >> 3, j = threadIdx.x & 7;
  const int64_t block = slot >> g.bs_shift;
  const int off = (int)(slot & (bs - 1));
  const int64_t at = block * g.n_kv + head;
  float* scale_at = (is_v ? g.v_scales : g.k_scales) + at;
  uint8_t* codes = (is_v ? g.v_codes : g.k_codes) + (at << g.bs_shift) * D + 8 * j;
  const float held = off > 0 ? *scale_at : 0.f;
  const float old = held > 0.f && held < INFINITY ? held : 0.f;
  // the rows that may be the run's, asked for with what says how many are: 8 j .. + 7 and 64 + 8 j .. + 7 of a row a lane
  const bf16_t* src = (is_v ? g.v : g.k) + t0 * g.stride + head * D + 8 * j;
  const bool turn = !is_v && g.cos_sin != nullptr;
  const int most = min(WAVE ? n : bs - off, (int)min(g.tokens - t0, (int64_t)kMostBlock));
  raw4 lo[PASSES], hi[PASSES];
  int64_t pos[PASSES];
  float rsc[PASSES];
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int i = p * STEP + row;
    if (i < most) {
      lo[p] = *reinterpret_cast<const raw4*>(src + i * g.stride);
      hi[p] = *reinterpret_cast<const raw4*>(src + i * g.stride + 64);
      pos[p] = turn ? position(g, t0 + i) : 0;
      rsc[p] = g.row_scale != nullptr ? g.row_scale[t0 + i] : 1.f;
    }
  }
  if constexpr (!WAVE) {  // the run's length: up to where the slots stop rising by one, or the block ends
    n = 0;
#pragma unroll
    for (int h = 0; h < kMostBlock / 64; ++h) {
      const int i = 64 * h + lane;
      const bool on = i < most && g.slots[t0 + i] == slot + i;
      const uint64_t m = __builtin_amdgcn_ballot_w64(!on);
      if (n == 64 * h) n += m ? __builtin_ctzll(m) : 64;
    }
  }
  float x[PASSES][16];
  float amax = 0.f;
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int i = p * STEP + row;
    if (i < n) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        x[p][2 * k] = bf16lo(lo[p][k]) * rsc[p], x[p][2 * k + 1] = bf16hi(lo[p][k]) * rsc[p];
        x[p][8 + 2 * k] = bf16lo(hi[p][k]) * rsc[p], x[p][9 + 2 * k] = bf16hi(hi[p][k]) * rsc[p];
      }
      if (turn) {
        const float* cs = g.cos_sin + pos[p] * D + 8 * j;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const f32x4 c = *reinterpret_cast<const f32x4*>(cs + 4 * h), s = *reinterpret_cast<const f32x4*>(cs + 64 + 4 * h);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float u = x[p][4 * h + k], w = x[p][8 + 4 * h + k];
            x[p][4 * h + k] = u * c[k] - w * s[k];
            x[p][8 + 4 * h + k] = w * c[k] + u * s[k];
          }
        }
      }
#pragma unroll
      for (int c = 0; c < 16; ++c) {
        const float a = fabsf(x[p][c]);
        amax = a < INFINITY ? fmaxf(amax, a) : amax;
      }
    }
  }
  amax = wave_reduce_max(amax);
  if constexpr (!WAVE) {
    if (lane == 0) red[threadIdx.x >> 6] = amax;
    __syncthreads();  // (every wave has read the old scale by now)
    amax = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  }
  const float now = fmaxf(old, power_scale<CODE>(amax));
  const float inv = 1.f / now;
  if ((WAVE ? lane : (int)threadIdx.x) == 0) *scale_at = now;
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int i = p * STEP + row;
    if (i < n) {
      uint8_t* dst = codes + (int64_t)(off + i) * D;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        raw2 w;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float* y = &x[p][8 * h + 4 * k];
          w[k] = codes4<CODE>(y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv);
        }
        *reinterpret_cast<raw2*>(dst + 64 * h) = w;
      }
    }
  }
  if (off > 0 && now != held) {
    const float ratio = old / now;
    for (int i = row; i < off; i += STEP) {
      uint8_t* dst = codes + (int64_t)i * D;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        raw2 w = *reinterpret_cast<const raw2*>(dst + 64 * h);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float f[4];
          widen4<CODE>(w[k], f);
          w[k] = codes4<CODE>(f[0] * ratio, f[1] * ratio, f[2] * ratio, f[3] * ratio);
        }
        *reinterpret_cast<raw2*>(dst + 64 * h) = w;
      }
    }
  }
  if constexpr (!WAVE) __syncthreads();  // (the maxima's place is used again by the next run)
}

template <int CODE, int PASSES>
__global__ void __launch_bounds__(kThreads) block_append_kernel(const AppendArgs g) {
  __shared__ float red[4];
  const int lane = threadIdx.x & 63;
  if ((int)blockIdx.x < g.units_x) {  // units: windows x heads x (K, V)
    const int per = 2 * g.n_kv;
    const int64_t w0 = (int64_t)(blockIdx.x / per) * g.window;
    const int u = blockIdx.x % per, head = u >> 1, is_v = u & 1;
    // every lane looks at one token and the one in front of it, eight tokens past the window too: there its last runs may end
    int64_t slot = -1;
    bool begins = false;
    if (lane <= g.window + 8 && w0 + lane < g.tokens) {
      slot = g.slots[w0 + lane];
      const int64_t before = g.slots[max(w0 + lane - 1, (int64_t)0)];
      const bool inside = w0 + lane > 0 && (slot & ((1 << g.bs_shift) - 1)) != 0 && before == slot - 1;
      begins = slot >= 0 && slot < g.num_slots && !inside;
    }
    // a run ends at the next one, at a token that has no place, or behind the last token
    const uint64_t starts = __builtin_amdgcn_ballot_w64(begins), runs = starts & ((1ull << g.window) - 1);
    const uint64_t ends = starts | __builtin_amdgcn_ballot_w64(lane <= g.window + 8 && (slot < 0 || slot >= g.num_slots));
    auto slot_of = [&](int i) {
      const uint32_t lo = __builtin_amdgcn_readlane((int)slot, i), hi = __builtin_amdgcn_readlane((int)(slot >> 32), i);
      return (int64_t)((uint64_t)hi << 32 | lo);
    };
    auto rows_of = [&](int i) {  // (more than eight where the window does not say)
      const uint64_t next = i < 63 ? ends >> (i + 1) : 0;
      return next ? __builtin_ctzll(next) + 1 : 64;
    };
    for (uint64_t m = runs; m; m &= m - 1) {
      const int i = __builtin_ctzll(m);
      if (rows_of(i) > 8) append_run<CODE, PASSES, false>(g, w0 + i, slot_of(i), 0, head, is_v, red);
    }
    int k = 0;
    for (uint64_t m = runs; m; m &= m - 1) {
      const int i = __builtin_ctzll(m), n = rows_of(i);
      if (n <= 8 && (k++ & 3) == (int)(threadIdx.x >> 6)) append_run<CODE, 1, true>(g, w0 + i, slot_of(i), n, head, is_v, red);
    }
    return;
  }
  // Q: a token a wave, eight lanes a head; a lane's cosines and sines serve its heads, four of them on their way at once
  const int64_t t = (int64_t)(blockIdx.x - g.units_x) * 4 + (threadIdx.x >> 6);
  if (t >= g.tokens) return;
  const float rsc = g.row_scale != nullptr ? g.row_scale[t] : 1.f;
  const float* cs = g.rotate_q && g.cos_sin != nullptr ? g.cos_sin + position(g, t) * D : nullptr;
  const int j = lane & 7;
  f32x4 c[2] = {{1.f, 1.f, 1.f, 1.f}, {1.f, 1.f, 1.f, 1.f}}, s[2] = {};
  if (cs != nullptr) {
#pragma unroll
    for (int h = 0; h < 2; ++h) c[h] = *reinterpret_cast<const f32x4*>(cs + 8 * j + 4 * h), s[h] = *reinterpret_cast<const f32x4*>(cs + 64 + 8 * j + 4 * h);
  }
  const bf16_t* src = g.q + t * g.stride + 8 * j;
  bf16_t* dst = g.q_out + t * g.q_out_stride + 8 * j;
  constexpr int kHeads = 4;
  for (int h0 = lane >> 3; h0 < g.n_q; h0 += 8 * kHeads) {
    raw4 a[kHeads], b[kHeads];
#pragma unroll
    for (int k = 0; k < kHeads; ++k) {
      const int h = min(h0 + 8 * k, g.n_q - 1);
      a[k] = *reinterpret_cast<const raw4*>(src + h * D);
      b[k] = *reinterpret_cast<const raw4*>(src + h * D + 64);
    }
#pragma unroll
    for (int k = 0; k < kHeads; ++k) {
      raw4 oa, ob;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float u[2] = {bf16lo(a[k][i]) * rsc, bf16hi(a[k][i]) * rsc}, w[2] = {bf16lo(b[k][i]) * rsc, bf16hi(b[k][i]) * rsc};
        float x[2], y[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float cc = c[i >> 1][2 * (i & 1) + e], ss = s[i >> 1][2 * (i & 1) + e];
          x[e] = cs != nullptr ? u[e] * cc - w[e] * ss : u[e];
          y[e] = cs != nullptr ? w[e] * cc + u[e] * ss : w[e];
        }
        oa[i] = pack_bf16x2(x[0], x[1]), ob[i] = pack_bf16x2(y[0], y[1]);
      }
      if (h0 + 8 * k < g.n_q) {
        *reinterpret_cast<raw4*>(dst + (h0 + 8 * k) * D) = oa;
        *reinterpret_cast<raw4*>(dst + (h0 + 8 * k) * D + 64) = ob;
      }
    }
  }
}

// Blocks as bf16: grid (blocks per sequence, sequences, 2 = K / V times pieces); dst_table[i][j] takes block j of sequence i (dense: that is
// i max_blocks + j, and written here), blocks past the sequence's length are left.  Bound by HBM; a thread has its loads of a piece on their way at once (105 blocks of 64 x 8 heads,
// K and V: 11.6 us, 3.5 TB/s read and written).
constexpr int kVecs = 4, kPiece = kThreads * 16 * kVecs;

template <int CODE>
__global__ void __launch_bounds__(kThreads)
    block_dequant_kernel(const uint8_t* __restrict__ kc, const uint8_t* __restrict__ vc, const float* __restrict__ k_scales,
                         const float* __restrict__ v_scales, bf16_t* __restrict__ ks, bf16_t* __restrict__ vs,
                         const int* __restrict__ block_tables, int bt_stride, const int* __restrict__ ctx_lens,
                         int* __restrict__ dst_table, int dense, int max_blocks, int num_blocks, int dst_blocks, int n_kv, int bs_shift) {
  const int j = blockIdx.x, i = blockIdx.y, which = blockIdx.z & 1;
  const int64_t at_table = (int64_t)i * max_blocks + j;
  if (dense && blockIdx.z == 0 && threadIdx.x == 0) dst_table[at_table] = (int)at_table;
  if (((int64_t)j << bs_shift) >= ctx_lens[i]) return;
  const int src = block_tables[(int64_t)i * bt_stride + j], dst = dense ? (int)at_table : dst_table[at_table];
  if ((unsigned)src >= (unsigned)num_blocks || (unsigned)dst >= (unsigned)dst_blocks) return;
  const int elems = n_kv << bs_shift << 7;
  const uint8_t* from = (which ? vc : kc) + (int64_t)src * elems;
  bf16_t* to = (which ? vs : ks) + (int64_t)dst * elems;
  const float* scales = (which ? v_scales : k_scales) + (int64_t)src * n_kv;
  const int e0 = (blockIdx.z >> 1) * kPiece + threadIdx.x * 16;
  raw4 w[kVecs];
  float s[kVecs];
#pragma unroll
  for (int n = 0; n < kVecs; ++n) {
    const int e = e0 + n * kThreads * 16, at = e < elems ? e : 0;
    w[n] = *reinterpret_cast<const raw4*>(from + at);
    s[n] = scales[at >> (bs_shift + 7)];
  }
#pragma unroll
  for (int n = 0; n < kVecs; ++n) {
    const int e = e0 + n * kThreads * 16;
    if (e >= elems) return;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const raw2 a = widen4_bf16<CODE, true>(w[n][2 * h], s[n]), b = widen4_bf16<CODE, true>(w[n][2 * h + 1], s[n]);
      *reinterpret_cast<raw4*>(to + e + 8 * h) = raw4{a[0], a[1], b[0], b[1]};
    }
  }
}

}  // namespace

// code: 0 int8, 1 e4m3fn.  q, k, v: bf16 rows `stride` elements apart, 16-byte aligned; q_out nullptr: K and V alone;
// slots nullptr: Q alone.
extern "C" int dx_block_append(const void* q, const void* k, const void* v, int64_t stride, void* q_out, int64_t q_out_stride,
                               const void* positions, int pos_i64, const float* cos_sin, int n_positions, const float* row_scale, const int64_t* slots,
                               void* k_codes, void* v_codes, float* k_scales, float* v_scales, int tokens, int n_q, int n_kv,
                               int head_dim, int block_size, int num_blocks, int rotate_q, int code, hipStream_t stream) {
  if (head_dim != D || block_size < 16 || block_size > kMostBlock || (block_size & (block_size - 1)) || stride % 8 || q_out_stride % 8 ||
      (cos_sin != nullptr && n_positions < 1))
    return -1;
  if (tokens <= 0) return 0;
  AppendArgs g{};
  g.q = (const bf16_t*)q, g.k = (const bf16_t*)k, g.v = (const bf16_t*)v, g.q_out = (bf16_t*)q_out;
  g.positions = positions, g.cos_sin = cos_sin, g.row_scale = row_scale, g.slots = slots;
  g.k_codes = (uint8_t*)k_codes, g.v_codes = (uint8_t*)v_codes, g.k_scales = k_scales, g.v_scales = v_scales;
  g.stride = stride, g.q_out_stride = q_out_stride;
  g.tokens = tokens, g.n_q = n_q, g.n_kv = n_kv, g.bs_shift = __builtin_ctz((unsigned)block_size);
  g.num_slots = (int64_t)num_blocks << g.bs_shift;
  g.pos_i64 = pos_i64, g.rotate_q = rotate_q, g.last_position = n_positions - 1;
  g.window = tokens > 512 ? 32 : 4;
  const int64_t units = slots ? (int64_t)((tokens + g.window - 1) / g.window) * 2 * n_kv : 0;
  const int64_t grid = units + (q_out ? (tokens + 3) / 4 : 0);
  if (grid == 0) return 0;
  if (grid > 0x7fffffff) return -2;
  g.units_x = (int)units;
#define DX_APPEND(C)                                                                      \
  do {                                                                                    \
    if (block_size <= 32) block_append_kernel<C, 1><<<(unsigned)grid, kThreads, 0, stream>>>(g);           \
    else if (block_size == 64) block_append_kernel<C, 2><<<(unsigned)grid, kThreads, 0, stream>>>(g);      \
    else block_append_kernel<C, 4><<<(unsigned)grid, kThreads, 0, stream>>>(g);                            \
  } while (0)
  if (code == kE4m3) DX_APPEND(kE4m3);
  else DX_APPEND(kInt8);
#undef DX_APPEND
  return (int)hipGetLastError();
}

extern "C" int dx_block_dequant(const void* kc, const void* vc, const float* k_scales, const float* v_scales, void* ks, void* vs,
                                const int* block_tables, int bt_stride, const int* ctx_lens, int* dst_table, int dense, int n_seqs,
                                int max_blocks, int num_blocks, int dst_blocks, int n_kv, int block_size, int head_dim, int code,
                                hipStream_t stream) {
  if (head_dim != D || block_size < 16 || (block_size & (block_size - 1))) return -1;
  if (n_seqs == 0 || max_blocks == 0) return 0;
  const int64_t elems = (int64_t)n_kv * block_size * D, pieces = (elems + kPiece - 1) / kPiece;
  if (elems > 0x3fffffff || pieces > 32767 || n_seqs > 65535) return -2;
  const dim3 grid(max_blocks, n_seqs, (unsigned)(2 * pieces));
  const int shift = __builtin_ctz((unsigned)block_size);
  auto go = [&](auto kernel) {
    kernel<<<grid, kThreads, 0, stream>>>((const uint8_t*)kc, (const uint8_t*)vc, k_scales, v_scales, (bf16_t*)ks, (bf16_t*)vs,
                                          block_tables, bt_stride, ctx_lens, dst_table, dense, max_blocks, num_blocks, dst_blocks, n_kv, shift);
  };
  if (code == kE4m3) go(block_dequant_kernel<kE4m3>);
  else go(block_dequant_kernel<kInt8>);
  return (int)hipGetLastError();
}
