// Paged causal prompt attention (ragged chunks behind cached tokens, grouped heads of 128) over the 8-bit cache whose scales
// belong to a block and head (block8.h), for gfx950:
//   out[i, h] = sum_j p_j vs_j v_j,  p = softmax_j(scale ks_j (q_i . k_j)),  j <= position of i (causal) or j < ctx
// with k_j, v_j the codes of token j and ks_j, vs_j the scales of its block.
//
// Bound by the matrix products and the exponentials of long chunks and by the cache's bytes of short ones.  A workgroup takes 32 rows a
// wave of one key/value head, a row being one query head of one token (token-major: row = token G + head), so that chunks of few tokens
// fill waves at any group size, and a wave's rows span few positions.  Tiles of 64 keys: their codes are asked for a tile ahead, 16
// bytes a lane, and become bf16, which holds them exactly, in swizzled LDS images (a workgroup widens a code once for all its rows).
// S^T = K Q^T and O^T = V^T P^T on 32 x 32 x 16 products: a lane's scores are one row's, the softmax is lane-local but for one exchange
// between the halves, the weights are the second product's operand as they are, V is read transposed, and the row sum is taken of the
// bf16 weights that the second product sees (rounded to 2^-8 of themselves), two by an instruction.  The running maximum moves when a
// tile's exceeds it by 2^8.
//
// Scales stay out of the products and cost no instruction a score: ks is a factor of the scores; O is held in units of the largest vs
// that the workgroup has come upon, and what a tile's vs is of the unit is added to its exponents; the row sum's ones are its inverse
// (2^-100 at least: what lies further apart is taken for that, and weights under 2^-26 of it are lost to the row sum).
//
// 8000 tokens of 64 / 8 heads, e4m3: 925 us, 1133 TFLOP/s (matrix cores busy half of the cycles, vector issue two thirds, the clock at 1.9
// GHz); two of up to 5000, 32 / 8 heads, int8: 372 to 389; six chunks behind up to 900 tokens, e4m3: 40 to 42; 16 tokens behind 20000: 22 with the join.
// One to four tokens behind 20000 (block_rows_kernel) 15, eight 19, with the join.
//
// Few rows behind many keys are split over the keys (the plan says where), each part leaves its sums in fp32, and a second kernel
// joins them.
#include "block8.h"

#include <type_traits>

namespace {

constexpr int D = 128, BQ = 32;
constexpr float kRescale = 8.0f;
constexpr int kItem = 6;  // seq, first row, first key, end of the keys, place of its sums (or -1), rows of the sequence
constexpr int kFewRows = 32;  // rows that block_rows_kernel takes
constexpr int kJoin = 4;  // seq, first row, first place, places
typedef float f32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ int swz(int row) { return ((row & 3) << 2) | ((row >> 2) & 3); }
__device__ __forceinline__ int tile_off(int row, int ch) { return row * 256 + 16 * (ch ^ swz(row)); }

struct PrefillArgs {
  bf16_t* out;
  float *ws_o, *ws_ml;
  const bf16_t* q;
  const uint8_t *k, *v;
  const float *ks, *vs;
  const int *block_tables, *cu, *ctx_lens, *work;
  int64_t q_stride;
  int bt_stride, bt_cols, n_kv, G, bs_shift, num_blocks, causal, tile, tokens;  // tile: rows of a place of sums
  float scale_log2e;
};

// a pair of bf16 times another, added to a sum in fp32
__device__ __forceinline__ float sum2(uint32_t a, uint32_t b, float c) {
  typedef __bf16 pair __attribute__((ext_vector_type(2)));
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(pair, a), __builtin_bit_cast(pair, b), c, false);
}

// the larger of two scores, NaN where one is: an instruction for two more (fmaxf would quiet each score first)
__device__ __forceinline__ float top(float x, float y) { return __builtin_elementwise_maximum(x, y); }

// The new tokens of a sequence, wherever the step says they are: first and count, among those that there are.
struct Tokens {
  int first, n;
};
__device__ __forceinline__ Tokens tokens_of(const int* cu, int seq, int tokens) {
  const int first = min(max(__builtin_amdgcn_readfirstlane(cu[seq]), 0), tokens);
  return {first, min(max(__builtin_amdgcn_readfirstlane(cu[seq + 1]), first), tokens) - first};
}

// A sequence that has other rows than the plan's: those that no item has are NaN (the items' own are so by their row sum).
__device__ __forceinline__ void rows_without_item(const PrefillArgs& a, int kvh, const Tokens& at, int from) {
  const int n = (at.n * a.G - from) * (D / 8);
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int f = from + i / (D / 8), tok = f / a.G;
    *reinterpret_cast<raw4*>(a.out + ((int64_t)(at.first + tok) * a.n_kv * a.G + kvh * a.G + f - tok * a.G) * D + 8 * (i % (D / 8))) =
        raw4{0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u};
  }
}

template <int I> using at_t = std::integral_constant<int, I>;

// RW: row waves of 32 rows; KW: waves that share a tile's keys (1: 64 keys, or 4: 128, 32 each); ONE: a wave's keys of a tile lie in one block
template <int CODE, int RW, int KW, bool ONE>
__global__ void __launch_bounds__(64 * RW * KW, 2) block_prefill_kernel(const PrefillArgs a) {
  static_assert(KW == 1 || KW == 4, "keys of a tile");
  constexpr int BKV = KW == 1 ? 64 : 128, kTileBytes = BKV * D * 2;
  constexpr int NW = RW * KW, PIECES = BKV / 8 / NW;  // pieces of 8 rows of a tile that a wave brings
  constexpr int SUBS = KW == 1 ? 2 : 1;         // 32-key pieces of a tile that a wave multiplies
  constexpr int NG = ONE ? 1 : 2 * SUBS;        // scales of a wave's keys of a tile
  constexpr bool kPhases = RW == 8;             // two halves of the waves, in turn with products and with the softmax
  __shared__ __attribute__((aligned(16))) char smem[2 * 2 * kTileBytes];
  const int* item = a.work + (int64_t)blockIdx.y * kItem;
  const int kvh = blockIdx.x, G = a.G;
  const int seq = __builtin_amdgcn_readfirstlane(item[0]), row0 = __builtin_amdgcn_readfirstlane(item[1]);
  const int key0 = __builtin_amdgcn_readfirstlane(item[2]), key1 = __builtin_amdgcn_readfirstlane(item[3]), place = __builtin_amdgcn_readfirstlane(item[4]);
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rw = wid % RW, kw = wid / RW;
  const int r = lane & 31, h = lane >> 5;
  const int* bt = a.block_tables + (int64_t)seq * a.bt_stride;
  // the blocks of the tiles, 64 at a time, a lane each (a table's columns are all that may be read of it)
  int first = key0 >> a.bs_shift, ids = bt[min(first + lane, a.bt_cols - 1)];
  const Tokens mine = tokens_of(a.cu, seq, a.tokens);
  const int q_start = mine.first, qlen = mine.n;
  const int ctx = __builtin_amdgcn_readfirstlane((int)min((int64_t)a.ctx_lens[seq], (int64_t)a.bt_cols << a.bs_shift));
  const int last = max(ctx - 1, 0) >> a.bs_shift;
  // ... and what becomes of their scales: a score's factor (never 0: a masked score is -infinity times it), the logarithm of vs in
  // units of the largest so far, and its inverse as a pair of bf16
  float sc_l, lg_l, unit = 0x1p-126f;
  uint32_t ones_l;
  float ks, vs;
  auto ask = [&]() __attribute__((always_inline)) {
    ids = (unsigned)ids < (unsigned)a.num_blocks ? ids : 0;
    ks = a.ks[(int64_t)ids * a.n_kv + kvh], vs = a.vs[(int64_t)ids * a.n_kv + kvh];
  };
  auto scales = [&]() __attribute__((always_inline)) {
    sc_l = fmaxf(ks * a.scale_log2e, 0x1p-126f);
    const float top = wave_reduce_max(first + lane <= last ? vs : 0.f);  // (a scale behind the context may be anything)
    unit = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(fmaxf(unit, top))));
    const float part = fmaxf(vs * __builtin_amdgcn_rcpf(unit), 0x1p-100f), inv = __builtin_amdgcn_rcpf(part);  // (of powers of two: exact)
    lg_l = __builtin_amdgcn_logf(part);
    ones_l = pack_bf16x2(inv, inv);
  };
  ask();
  const int pos0 = ctx - qlen, rows = qlen * G, planned = __builtin_amdgcn_readfirstlane(item[5]);
  if (rows != planned && key0 == 0 && row0 + BQ * RW >= planned) rows_without_item(a, kvh, mine, planned);
  const int w0 = row0 + BQ * rw, f = w0 + r;
  const bool valid = f < rows;
  const int tok = f / G, hq = f - tok * G;
  const int my_pos = a.causal ? pos0 + tok : ctx - 1;
  const int wave_min = a.causal ? pos0 + w0 / G : ctx - 1;
  const int wave_max = w0 >= rows ? -1 : a.causal ? pos0 + min(w0 + BQ - 1, rows - 1) / G : ctx - 1;
  const int wg_max = a.causal ? pos0 + min(row0 + BQ * RW - 1, rows - 1) / G : ctx - 1;
  const int kv_end = min(min(key1, ctx), wg_max + 1);
  const int n_tiles = max(kv_end - key0 + BKV - 1, 0) / BKV;

  // ---- a tile's codes: piece p of this wave is rows 8 (PIECES wid + p) .. + 7, a lane 16 columns of one of them
  raw4 kr[PIECES], vr[PIECES];
  uint32_t ones_now[NG];  // of the tile whose weights are here
  auto at_block = [&](int j) __attribute__((always_inline)) { return min(j >> a.bs_shift, last) - first; };
  auto window = [&](int t0, int t1) __attribute__((always_inline)) {  // the blocks of tiles t0 to t1 are among the 64 here
    if (min((key0 + (t1 + 1) * BKV - 1) >> a.bs_shift, last) - first >= 64) {
      first = (key0 + t0 * BKV) >> a.bs_shift;
      ids = bt[min(first + lane, a.bt_cols - 1)];
      ask();
      scales();
    }
  };
  auto load = [&](const uint8_t* from, int t, raw4(&to)[PIECES]) __attribute__((always_inline)) {
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
      const int j = key0 + t * BKV + 8 * (PIECES * wid + p);
      const int64_t block = (int64_t)__builtin_amdgcn_readlane(ids, at_block(j)) * a.n_kv + kvh;
      const uint8_t* at = from + ((block << a.bs_shift) + (j & ((1 << a.bs_shift) - 1))) * D;  // (the same in all lanes)
      to[p] = *reinterpret_cast<const raw4*>(at + (uint32_t)(lane >> 3) * D + 16 * (lane & 7));
    }
  };
  // (whatever lies behind the context may be a NaN)
  auto behind = [&](int t, raw4(&x)[PIECES]) __attribute__((always_inline)) {
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
      const bool none = key0 + t * BKV + 8 * (PIECES * wid + p) + (lane >> 3) >= ctx;
#pragma unroll
      for (int i = 0; i < 4; ++i) x[p][i] = none ? 0u : x[p][i];
    }
  };
  int to_off[PIECES][2];
#pragma unroll
  for (int p = 0; p < PIECES; ++p)
#pragma unroll
    for (int i = 0; i < 2; ++i) to_off[p][i] = tile_off(8 * (PIECES * wid + p) + (lane >> 3), 2 * (lane & 7) + i);
  auto store = [&](int image, const raw4(&x)[PIECES]) __attribute__((always_inline)) {
#pragma unroll
    for (int p = 0; p < PIECES; ++p)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const raw2 lo = widen4_bf16<CODE, false>(x[p][2 * i], 1.f), hi = widen4_bf16<CODE, false>(x[p][2 * i + 1], 1.f);
        *reinterpret_cast<raw4*>(smem + image + to_off[p][i]) = raw4{lo[0], lo[1], hi[0], hi[1]};
      }
  };
  if (n_tiles > 0) {
    load(a.k, 0, kr);
    if constexpr (!kPhases) load(a.v, 0, vr);
  }
  u16x8 qf[8];
  {
    const bf16_t* qp = a.q + (int64_t)(q_start + tok) * a.q_stride + (int64_t)(kvh * G + hq) * D + 8 * h;
#pragma unroll
    for (int s = 0; s < 8; ++s) qf[s] = valid ? *reinterpret_cast<const u16x8*>(qp + 16 * s) : u16x8{{0, 0, 0, 0}};
  }
  scales();  // (behind the loads that do not need them)
  float unit_o = unit;  // what this wave's O is in
  f32x16 o_acc[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) o_acc[i] = f32x16{};
  float m_i = -1e30f, l_i = rows == planned ? 0.f : __builtin_nanf("");  // (l: of this lane's keys)
  f32x16 s0, s1;                  // a tile's scores
  u16x8 pf[2][2];                 // its weights
  auto weights = [&](int j0) __attribute__((always_inline)) {
    if (j0 + 32 * SUBS - 1 > wave_min || j0 + 32 * SUBS > ctx) {  // the diagonal, or the context's end
      const int lim = min(my_pos, ctx - 1) - j0 - 4 * h;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int off = (i & 3) + 8 * (i >> 2);
        s0[i] = off > lim ? -INFINITY : s0[i];
        if constexpr (SUBS == 2) s1[i] = off + 32 > lim ? -INFINITY : s1[i];
      }
    }
    // a score's factor, and what its exponent is short of: one of a tile, or one each 16 keys (group 2 sub + s2 of this wave's)
    float sc[2][2], lg[2][2];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const int i = at_block(j0 + 16 * g);
      const float x = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(sc_l), i));
      const float y = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(lg_l), i));
      if (NG == 1) sc[0][0] = sc[0][1] = sc[1][0] = sc[1][1] = x, lg[0][0] = lg[0][1] = lg[1][0] = lg[1][1] = y;
      else sc[g >> 1][g & 1] = x, lg[g >> 1][g & 1] = y;
      ones_now[g] = __builtin_amdgcn_readlane(ones_l, i);
    }
    float t_s;
    if constexpr (ONE) {
      float ta = s0[0], tb = s0[1];
      if constexpr (SUBS == 2) ta = top(ta, s1[0]), tb = top(tb, s1[1]);
#pragma unroll
      for (int i = 2; i < 16; i += 2) {
        ta = top(ta, s0[i]), tb = top(tb, s0[i + 1]);
        if constexpr (SUBS == 2) ta = top(ta, s1[i]), tb = top(tb, s1[i + 1]);
      }
      t_s = over_halves(top(ta, tb), top) * sc[0][0];  // (scales are positive)
    } else {
      t_s = -INFINITY;
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2) {
        float ta = s0[8 * s2], tb = SUBS == 2 ? s1[8 * s2] : -INFINITY;
#pragma unroll
        for (int i = 8 * s2 + 1; i < 8 * s2 + 8; ++i) {
          ta = top(ta, s0[i]);
          if constexpr (SUBS == 2) tb = top(tb, s1[i]);
        }
        t_s = top(t_s, ta * sc[0][s2]);
        if constexpr (SUBS == 2) t_s = top(t_s, tb * sc[1][s2]);
      }
      t_s = over_halves(t_s, top);
    }
    const float m_new = t_s > m_i + kRescale ? t_s : m_i;
    const float alpha = fast_exp2(m_i - m_new);
    m_i = m_new;
#pragma unroll
    for (int s2 = 0; s2 < 2; ++s2) {
      const float b0 = m_new - lg[0][s2], b1 = SUBS == 2 ? m_new - lg[SUBS - 1][s2] : 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int i = 8 * s2 + 2 * w;
        pf[0][s2].w[w] = pack_bf16x2(fast_exp2(s0[i] * sc[0][s2] - b0), fast_exp2(s0[i + 1] * sc[0][s2] - b0));
        if constexpr (SUBS == 2) pf[1][s2].w[w] = pack_bf16x2(fast_exp2(s1[i] * sc[1][s2] - b1), fast_exp2(s1[i + 1] * sc[1][s2] - b1));
      }
    }
    l_i *= alpha;
    if (unit_o != unit || __builtin_amdgcn_ballot_w64(alpha != 1.f)) {
      const float both = alpha * (unit_o * __builtin_amdgcn_rcpf(unit));
      unit_o = unit;
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) o_acc[dt] *= both;
    }
  };
  // pair i of a wave's 8 SUBS pairs of weights, added to the row sum
  auto add_pair = [&](int i) __attribute__((always_inline)) {
    const int sub = i >> 3, s2 = (i >> 2) & 1;
    l_i = sum2(pf[sub][s2].w[i & 3], ones_now[NG == 1 ? 0 : 2 * sub + s2], l_i);
  };
  auto mfma = [](const u16x8& x, const u16x8& y, const f32x16& c) __attribute__((always_inline)) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, x), __builtin_bit_cast(bf16x8_t, y), c, 0, 0, 0);
  };
  // ---- fragments, by one address each of K and V: what a fragment's place differs by is an exclusive or, or a constant.  (The addresses
  // are taken anew in each tile: there are not registers for a place each.)
  int kbase = tile_off(r, h), vbase = tile_off(4 * h + ((lane & 15) >> 2), 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) + 8 * (lane & 1);
  auto again = [&]() __attribute__((always_inline)) { asm volatile("" : "+v"(kbase), "+v"(vbase)); };
  auto kfrag = [&](int image, int i) __attribute__((always_inline)) {  // columns 16 (i % 8) .. + 15 of keys 32 (i / 8) .. + 31
    return __builtin_bit_cast(u16x8, *reinterpret_cast<const raw4*>(smem + (kbase ^ (32 * (i & 7))) + image + 8192 * (i >> 3)));
  };
  auto vfrag = [&](int image, int i) __attribute__((always_inline)) {  // columns 32 (i % 4) .. + 31 of keys 16 (i / 4) .. + 15
    const char* at = smem + image + 4096 * (i >> 2);
    const i16x4 lo = read_tr16((const lds_i16x4*)(at + (vbase ^ (64 * (i & 3)))));
    const i16x4 hi = read_tr16((const lds_i16x4*)(at + (vbase ^ (64 * (i & 3) + 32)) + 2048));
    return __builtin_bit_cast(u16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  };
  // Products FROM .. TO of the scores' (0 .. 15) and values' (16 .. 31), in one line with their fragments kAhead ahead; between(i) comes
  // behind product i.
  constexpr int kAhead = 4;
  auto line = [&](auto from_, auto to_, int k_image, int v_image, auto between) __attribute__((always_inline)) {
    constexpr int FROM = decltype(from_)::value, TO = decltype(to_)::value;
    u16x8 x[kAhead];
    auto read = [&](int i) __attribute__((always_inline)) { return i < 16 ? kfrag(k_image, i) : vfrag(v_image, i - 16); };
    if constexpr (FROM == 0) s0 = s1 = f32x16{};
#pragma unroll
    for (int i = 0; i < kAhead; ++i) x[i] = read(FROM + i);
    __builtin_amdgcn_sched_group_barrier(0x100, FROM < 16 ? kAhead : 2 * kAhead, 0);
#pragma unroll
    for (int i = FROM; i < TO; ++i) {
      const u16x8 now = x[(i - FROM) % kAhead];
      if (i + kAhead < TO) x[(i - FROM) % kAhead] = read(i + kAhead);
      if (i < 8) s0 = mfma(now, qf[i & 7], s0);
      else if (i < 16) s1 = mfma(now, qf[i & 7], s1);
      else o_acc[i & 3] = mfma(now, pf[(i >> 3) & 1][(i >> 2) & 1], o_acc[i & 3]);
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      if (i + kAhead < TO && i + kAhead < 16) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      else if (i + kAhead < TO) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
      between(i);
    }
  };
  auto nothing = [](int) {};

  const int jw = key0 + 32 * SUBS * kw;  // this wave's first key of a tile
  if constexpr (kPhases) {
    // The products of one half of the waves run while the other half has its softmax: left to themselves the two waves of a SIMD, held
    // together by the barriers, come to either at once, and wait.  Products of t read K of t and V of t - 1; the row sum of t - 1 and a
    // wave's part of the next K go with them, its part of the next V with the softmax, so that the two take about as long.  Half h is a
    // meeting behind half 0: it brings V a tile further.  us, 5000 + 4000 tokens of 32 / 8 heads, int8: no phases 411, with these
    // 328; without priority for the products 344, K and V brought with the products 342, with the softmax 350.
    const int late = wid / 4;  // (the waves of a SIMD are one of either half)
    auto meet = [&]() __attribute__((always_inline)) {
      __builtin_amdgcn_sched_barrier(0);
      __syncthreads();
      __builtin_amdgcn_sched_barrier(0);
    };
    auto k_at = [](int t) { return (t & 1) * kTileBytes; };
    auto v_at = [](int t) { return (2 + (t & 1)) * kTileBytes; };
    const int end = n_tiles - 1;  // (behind the last tile that one again, read by none)
    auto bring_v = [&](int t) __attribute__((always_inline)) {
      behind(min(t, end), vr);
      store(v_at(t), vr);
      load(a.v, min(t + 1, end), vr);
    };
    auto bring_k = [&](int t) __attribute__((always_inline)) {
      behind(min(t, end), kr);
      store(k_at(t), kr);
      load(a.k, min(t + 1, end), kr);
    };
    if (n_tiles > 0) {
      window(0, min(2, end));
      bring_k(0);
      load(a.v, 0, vr);
      meet();
      if (late) {
        bring_v(0);
        meet();
      }
      line(at_t<0>{}, at_t<16>{}, k_at(0), 0, nothing);
      bring_k(1);
      for (int t = 0; t < end; ++t) {
        meet();
        __builtin_amdgcn_s_setprio(0);
        window(t, min(t + 3, end));
        bring_v(t + late);
        weights(jw + t * BKV);
        again();
        meet();
        __builtin_amdgcn_s_setprio(1);
        line(at_t<0>{}, at_t<32>{}, k_at(t + 1), v_at(t), [&](int i) __attribute__((always_inline)) {
          if (i >= 14 && i < 30) add_pair(i - 14);
        });
        bring_k(t + 2);
      }
      meet();
      window(end, end);
      weights(jw + end * BKV);
      bring_v(end + late);
      again();
      meet();
      line(at_t<16>{}, at_t<32>{}, 0, v_at(end), [&](int i) __attribute__((always_inline)) { add_pair(i - 16); });
      if (!late) meet();
    }
  } else {
    auto image = [](int t) { return (t & 1) * 2 * kTileBytes; };
    if (n_tiles > 0) {
      behind(0, kr);
      store(image(0), kr);
      behind(0, vr);
      store(image(0) + kTileBytes, vr);
    }
    __syncthreads();
    for (int t = 0; t < n_tiles; ++t) {
      window(t, min(t + 1, n_tiles - 1));
      if (t + 1 < n_tiles) {
        load(a.k, t + 1, kr);
        load(a.v, t + 1, vr);
      }
      const int j0 = jw + t * BKV;
      if (j0 <= wave_max) {
        const int kb = image(t) + 8192 * SUBS * kw, vb = kb + kTileBytes;
        again();
        line(at_t<0>{}, at_t<8 * SUBS>{}, kb, 0, nothing);
        weights(j0);
        line(at_t<16>{}, at_t<16 + 8 * SUBS>{}, 0, vb, [&](int i) __attribute__((always_inline)) { add_pair(i - 16); });
      }
      if (t + 1 < n_tiles) {
        behind(t + 1, kr);
        store(image(t + 1), kr);
        behind(t + 1, vr);
        store(image(t + 1) + kTileBytes, vr);
      }
      __syncthreads();
    }
  }

  // ---- lane (r, h) holds columns 32 dt + 8 g + 4 h .. + 3 of its row
  l_i = halves_sum(l_i);
#pragma unroll
  for (int dt = 0; dt < 4; ++dt) o_acc[dt] *= unit_o;
  if constexpr (KW > 1) {  // the waves of the other keys hand their sums to those of the first
    float* so = reinterpret_cast<float*>(smem);  // [KW - 1][RW][64 lanes] x 64 values, a lane's apart by 64 so that a wave's lie together
    float* sml = so + (KW - 1) * RW * (BQ * D);
    static_assert((KW - 1) * RW * (BQ * D + 128) * 4 <= 4 * kTileBytes, "the images hold the sums");
    if (kw) {
      const int at = (kw - 1) * RW + rw;
#pragma unroll
      for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) so[at * (BQ * D) + (dt * 16 + i) * 64 + lane] = o_acc[dt][i];
      sml[at * 128 + lane] = m_i, sml[at * 128 + 64 + lane] = l_i;
    }
    __syncthreads();
    if (kw) return;
    float m[KW - 1], M = m_i;
#pragma unroll
    for (int k = 0; k < KW - 1; ++k) M = fmaxf(M, m[k] = sml[(k * RW + rw) * 128 + lane]);
    const float e0 = fast_exp2(m_i - M);
    l_i *= e0;
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) o_acc[dt] *= e0;
#pragma unroll
    for (int k = 0; k < KW - 1; ++k) {
      const float e = fast_exp2(m[k] - M);
      l_i += e * sml[(k * RW + rw) * 128 + 64 + lane];
#pragma unroll
      for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) o_acc[dt][i] += e * so[(k * RW + rw) * (BQ * D) + (dt * 16 + i) * 64 + lane];
    }
    m_i = M;
  }
  if (place >= 0) {  // the sums as they are
    const int64_t row = ((int64_t)place * a.n_kv + kvh) * a.tile + BQ * rw + r;
    if (valid) {
#pragma unroll
      for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<f32x4*>(a.ws_o + row * D + 32 * dt + 8 * g + 4 * h) =
              f32x4{o_acc[dt][4 * g], o_acc[dt][4 * g + 1], o_acc[dt][4 * g + 2], o_acc[dt][4 * g + 3]};
      if (h == 0) *reinterpret_cast<f32x2*>(a.ws_ml + row * 2) = f32x2{m_i, l_i};
    }
    return;
  }
  const float inv_l = l_i != 0.f ? 1.f / l_i : 0.f;
  bf16_t* op = a.out + ((int64_t)(q_start + tok) * a.n_kv * G + kvh * G + hq) * D;
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int g = 0; g < 4; g += 2) {
      uint2 x, y;
      x.x = pack_bf16x2(o_acc[dt][4 * g + 0] * inv_l, o_acc[dt][4 * g + 1] * inv_l);
      x.y = pack_bf16x2(o_acc[dt][4 * g + 2] * inv_l, o_acc[dt][4 * g + 3] * inv_l);
      y.x = pack_bf16x2(o_acc[dt][4 * g + 4] * inv_l, o_acc[dt][4 * g + 5] * inv_l);
      y.y = pack_bf16x2(o_acc[dt][4 * g + 6] * inv_l, o_acc[dt][4 * g + 7] * inv_l);
      const auto sx = __builtin_amdgcn_permlane32_swap(x.x, y.x, false, false);
      const auto sy = __builtin_amdgcn_permlane32_swap(x.y, y.y, false, false);
      if (valid)  // after the swaps: every lane takes part in them
        *reinterpret_cast<uint4*>(op + dt * 32 + 8 * g + 8 * h) = make_uint4(sx[0], sy[0], sx[1], sy[1]);
    }
}

// Few rows (16 CG of a key/value head at most) behind their keys: a decode step's kernel with more columns.  Bound by the cache's bytes: the
// waves of a workgroup take chunks of 32 keys in turn, each for all rows, with K and V on their way a chunk ahead and no barrier between
// them (the tiles above would leave waves without rows, and stage for 64 rows what 128 could use).  16 x 16 x 32 products: rows are the
// columns of S^T = K Q^T and O^T = V^T P^T; ks is a factor of the scores, vs of the weights (a lane's eight keys lie in one block); V
// goes through a wave's own image in LDS.
constexpr int CH = 32;
__device__ __forceinline__ int vimg_off(int row, int ch) { return row * 256 + 16 * (ch ^ (((row & 3) << 2) | ((row >> 2) & 3))); }

template <int CODE, int CG>
__global__ void __launch_bounds__(256, 2) block_rows_kernel(const PrefillArgs a) {
  __shared__ __attribute__((aligned(16))) char image[4 * CH * D * 2];
  __shared__ float st_m[4 * 16 * CG], st_l[4 * 16 * CG];
  const int* item = a.work + (int64_t)blockIdx.y * kItem;
  const int kvh = blockIdx.x, G = a.G;
  const int seq = __builtin_amdgcn_readfirstlane(item[0]), key0 = __builtin_amdgcn_readfirstlane(item[2]), key1 = __builtin_amdgcn_readfirstlane(item[3]);
  const int place = __builtin_amdgcn_readfirstlane(item[4]);
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, r = lane & 15;
  const Tokens mine = tokens_of(a.cu, seq, a.tokens);
  const int q_start = mine.first, qlen = mine.n;
  const int ctx = __builtin_amdgcn_readfirstlane((int)min((int64_t)a.ctx_lens[seq], (int64_t)a.bt_cols << a.bs_shift));
  const int rows = min(qlen * G, 16 * CG), pos0 = ctx - qlen, planned = __builtin_amdgcn_readfirstlane(item[5]);
  if (qlen * G != planned && key0 == 0) rows_without_item(a, kvh, mine, planned);
  if (rows == 0) return;
  const int p0 = key0, p1 = min(key1, ctx);
  char* vimg = image + wid * (CH * D * 2);

  raw4 qf[CG][4];
  int lim[CG];  // the last key a column sees (columns behind the rows hold the last row, and go nowhere)
#pragma unroll
  for (int c = 0; c < CG; ++c) {
    const int f = max(min(16 * c + r, rows - 1), 0), tok = f / G, hq = f - tok * G;
    lim[c] = a.causal ? pos0 + tok : ctx - 1;
#pragma unroll
    for (int s = 0; s < 4; ++s) qf[c][s] = *reinterpret_cast<const raw4*>(a.q + (int64_t)(q_start + tok) * a.q_stride + (int64_t)(kvh * G + hq) * D + 8 * (4 * g + s));
  }
  const int first_lim = a.causal ? pos0 : ctx - 1;  // keys up to here are seen by every row

  const int* bt = a.block_tables + (int64_t)seq * a.bt_stride;
  const int last = max(ctx - 1, 0) >> a.bs_shift;
  int first = p0 >> a.bs_shift, ids;
  auto fetch = [&]() {
    const int id = bt[min(first + lane, last)];
    ids = (unsigned)id < (unsigned)a.num_blocks ? id : 0;
  };
  fetch();
  auto block_at = [&](int i) {
    if (i - first >= 64) {  // (chunks only go up)
      first = i;
      fetch();
    }
    return __builtin_amdgcn_readlane(ids, max(i - first, 0));
  };

  f32x4 oacc[CG][8];
  float m_i[CG], l_i[CG];
#pragma unroll
  for (int c = 0; c < CG; ++c) {
    m_i[c] = -1e30f, l_i[c] = qlen * G == planned ? 0.f : __builtin_nanf("");
#pragma unroll
    for (int db = 0; db < 8; ++db) oacc[c][db] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const int n_chunks = max(p1 - p0 + CH - 1, 0) / CH;
  raw4 kf[2][2];
  raw2 vr[8];
  float ks_l, vs_l;
  auto load = [&](int c) {
    const int cb = p0 + c * CH;
    const int cb1 = cb + 16 < p1 ? cb + 16 : cb;
    const int64_t row0 = (int64_t)block_at(cb >> a.bs_shift) * a.n_kv + kvh, row1 = (int64_t)block_at(cb1 >> a.bs_shift) * a.n_kv + kvh;
    const int in = (1 << a.bs_shift) - 1;
    const int64_t base0 = ((row0 << a.bs_shift) + (cb & in)) * D, base1 = ((row1 << a.bs_shift) + (cb1 & in)) * D;
    const int64_t srow = g < 2 ? row0 : row1;
    ks_l = a.ks[srow];
    vs_l = a.vs[srow];
#pragma unroll
    for (int bb = 0; bb < 2; ++bb) {
      const int t = 8 * (r >> 2) + 4 * bb + (r & 3);
      const uint8_t* p = a.k + (t < 16 ? base0 : base1) + (t & 15) * D + 32 * g;
      kf[bb][0] = *reinterpret_cast<const raw4*>(p);
      kf[bb][1] = *reinterpret_cast<const raw4*>(p + 16);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) vr[k] = *reinterpret_cast<const raw2*>(a.v + (k < 4 ? base0 : base1) + (4 * (k & 3) + g) * D + 8 * r);
  };
  auto step = [&](auto more_, int c) {
    constexpr bool more = decltype(more_)::value;
    const int cb = p0 + c * CH;
    const bool ragged = cb + CH > p1, masked = ragged || cb + CH - 1 > first_lim;
    f32x4 sacc[CG][2];
#pragma unroll
    for (int bb = 0; bb < 2; ++bb) {
#pragma unroll
      for (int cg = 0; cg < CG; ++cg) sacc[cg][bb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const raw2 lo = widen4_bf16<CODE, false>(kf[bb][s >> 1][2 * (s & 1)], 1.f), hi = widen4_bf16<CODE, false>(kf[bb][s >> 1][2 * (s & 1) + 1], 1.f);
#pragma unroll
        for (int cg = 0; cg < CG; ++cg)
          sacc[cg][bb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, raw4{lo[0], lo[1], hi[0], hi[1]}),
                                                                 __builtin_bit_cast(bf16x8_t, qf[cg][s]), sacc[cg][bb], 0, 0, 0);
      }
    }
    if (ragged) {  // (weights of 0 meet zeros: whatever lies behind the context may be a NaN)
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (cb + 4 * k + g >= p1) vr[k] = raw2{0u, 0u};
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const raw2 lo = widen4_bf16<CODE, false>(vr[k][0], 1.f), hi = widen4_bf16<CODE, false>(vr[k][1], 1.f);
      *reinterpret_cast<raw4*>(vimg + vimg_off(4 * k + g, r)) = raw4{lo[0], lo[1], hi[0], hi[1]};
    }
    const float kscale = ks_l * a.scale_log2e, vscale = vs_l;
    if constexpr (more) load(c + 4);
    raw4 pf[CG];
#pragma unroll
    for (int cg = 0; cg < CG; ++cg) {
      float t[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) t[j] = sacc[cg][j >> 2][j & 3] * kscale;
      if (masked) {
        const int end = min(lim[cg], p1 - 1);
#pragma unroll
        for (int j = 0; j < 8; ++j) t[j] = cb + 8 * g + j > end ? -INFINITY : t[j];
      }
      float cmax = fmaxf(fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])), fmaxf(fmaxf(t[4], t[5]), fmaxf(t[6], t[7])));
      cmax = over_row_pairs(halves_max(cmax), [](float x, float y) { return fmaxf(x, y); });
      const float m_new = cmax > m_i[cg] + kRescale ? cmax : m_i[cg];
      const float alpha = fast_exp2(m_i[cg] - m_new);
      m_i[cg] = m_new;
      float ps = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float x = fast_exp2(t[2 * w] - m_new), y = fast_exp2(t[2 * w + 1] - m_new);
        ps += x + y;
        pf[cg][w] = pack_bf16x2(x * vscale, y * vscale);
      }
      if (ragged) {  // (a scale behind the context may be anything)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          if (cb + 8 * g + 2 * w >= p1) pf[cg][w] &= 0xffff0000u;
          if (cb + 8 * g + 2 * w + 1 >= p1) pf[cg][w] &= 0x0000ffffu;
        }
      }
      l_i[cg] = l_i[cg] * alpha + ps;
      if (__builtin_amdgcn_ballot_w64(alpha != 1.f)) {
#pragma unroll
        for (int db = 0; db < 8; ++db) oacc[cg][db] *= alpha;
      }
    }
#pragma unroll
    for (int db = 0; db < 8; ++db) {
      const int qq = r >> 2, pp = r & 3;
      const i16x4 lo = read_tr16((const lds_i16x4*)(vimg + vimg_off(8 * g + qq, 2 * db + (pp >> 1)) + 8 * (pp & 1)));
      const i16x4 hi = read_tr16((const lds_i16x4*)(vimg + vimg_off(8 * g + 4 + qq, 2 * db + (pp >> 1)) + 8 * (pp & 1)));
      const bf16x8_t v = __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
      for (int cg = 0; cg < CG; ++cg) oacc[cg][db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, __builtin_bit_cast(bf16x8_t, pf[cg]), oacc[cg][db], 0, 0, 0);
    }
  };
  int c = wid;
  if (c < n_chunks) {
    load(c);
    for (; c + 4 < n_chunks; c += 4) step(std::true_type{}, c);
    step(std::false_type{}, c);
  }

  // the waves' (O, m, l), 16 rows at a time, each in its own image; lane (g, r) holds columns 16 db + 4 g .. of a row
#pragma unroll
  for (int cg = 0; cg < CG; ++cg) {
    const float l_tot = over_row_pairs(halves_sum(l_i[cg]), [](float x, float y) { return x + y; });
    if (g == 0) st_m[(wid * CG + cg) * 16 + r] = m_i[cg], st_l[(wid * CG + cg) * 16 + r] = l_tot;
  }
#pragma unroll
  for (int cg = 0; cg < CG; ++cg) {
    if (16 * cg >= rows) break;
    if (cg) __syncthreads();
    float* so = reinterpret_cast<float*>(vimg) + r * D + 4 * g;
#pragma unroll
    for (int db = 0; db < 8; ++db) *reinterpret_cast<f32x4*>(so + 16 * db) = oacc[cg][db];
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * D / 4; i += 256) {
      const int in = i / (D / 4), d = 4 * (i % (D / 4)), f = 16 * cg + in;
      if (f >= rows) break;
      float m[4], M = -1e30f, den = 0.f;
      f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < 4; ++w) M = fmaxf(M, m[w] = st_m[(w * CG + cg) * 16 + in]);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float e = fast_exp2(m[w] - M);
        sum += e * *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(image + w * (CH * D * 2)) + in * D + d);
        den += e * st_l[(w * CG + cg) * 16 + in];
      }
      if (place >= 0) {
        const int64_t row = ((int64_t)place * a.n_kv + kvh) * kFewRows + f;
        *reinterpret_cast<f32x4*>(a.ws_o + row * D + d) = sum;
        if (d == 0) *reinterpret_cast<f32x2*>(a.ws_ml + row * 2) = f32x2{M, den};
      } else {
        const float inv = den != 0.f ? 1.f / den : 0.f;
        const int tok = f / G, hq = f - tok * G;
        *reinterpret_cast<uint2*>(a.out + ((int64_t)(q_start + tok) * a.n_kv * G + kvh * G + hq) * D + d) =
            uint2{pack_bf16x2(sum[0] * inv, sum[1] * inv), pack_bf16x2(sum[2] * inv, sum[3] * inv)};
      }
    }
  }
}

// A row's parts' sums under a common maximum, over their common sum: by 32 lanes x 4 columns where parts are few, eight rows a
// workgroup, by all eight groups of 32 lanes where they are many, each taking every eighth part, two of them on their way at once.
template <int GROUPS>
__global__ void __launch_bounds__(256) block_prefill_join_kernel(bf16_t* __restrict__ out, const float* __restrict__ ws_o, const float* __restrict__ ws_ml,
                                                                 const int* __restrict__ joins, const int* __restrict__ cu, int tokens, int n_kv, int G, int tile) {
  __shared__ __attribute__((aligned(16))) f32x4 other[8][D / 4];
  __shared__ float dens[8];
  const int grp = threadIdx.x >> 5, col = threadIdx.x & 31, in = blockIdx.x * (8 / GROUPS) + grp / GROUPS, kvh = blockIdx.y;
  const int* item = joins + (int64_t)blockIdx.z * kJoin;
  const int seq = item[0], f = item[1] + in, place = item[2], n = item[3];
  const Tokens mine = tokens_of(cu, seq, tokens);
  const int q_start = mine.first, rows = mine.n * G;
  if (in >= tile || f >= rows) return;  // (of one row: all of the workgroup)
  const int64_t step = (int64_t)n_kv * tile, row = ((int64_t)place * n_kv + kvh) * tile + in;
  float M = -1e30f;
  for (int p = col; p < n; p += 32) M = fmaxf(M, ws_ml[(row + p * step) * 2]);
#pragma unroll
  for (int d = 16; d; d >>= 1) M = fmaxf(M, __shfl_xor(M, d, 64));
  float den = 0.f;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  for (int p = grp % GROUPS; p < n; p += 2 * GROUPS) {
    const int p2 = min(p + GROUPS, n - 1);
    const f32x2 ml = *reinterpret_cast<const f32x2*>(ws_ml + (row + p * step) * 2), ml2 = *reinterpret_cast<const f32x2*>(ws_ml + (row + p2 * step) * 2);
    const f32x4 x = *reinterpret_cast<const f32x4*>(ws_o + (row + p * step) * D + 4 * col), x2 = *reinterpret_cast<const f32x4*>(ws_o + (row + p2 * step) * D + 4 * col);
    const float w = fast_exp2(ml.x - M), w2 = p + GROUPS < n ? fast_exp2(ml2.x - M) : 0.f;
    den += w * ml.y + w2 * ml2.y;
    sum += w * x + w2 * x2;
  }
  if constexpr (GROUPS > 1) {
    other[grp][col] = sum;
    if (col == 0) dens[grp] = den;
    __syncthreads();
    if (grp) return;
#pragma unroll
    for (int k = 1; k < 8; ++k) sum += other[k][col], den += dens[k];
  }
  const float inv = den != 0.f ? 1.f / den : 0.f;
  const int tok = f / G, hq = f - tok * G;
  *reinterpret_cast<uint2*>(out + ((int64_t)(q_start + tok) * n_kv * G + kvh * G + hq) * D + 4 * col) =
      uint2{pack_bf16x2(sum[0] * inv, sum[1] * inv), pack_bf16x2(sum[2] * inv, sum[3] * inv)};
}

// rows: those of the longest joined item; parts: of the most cut one
void join_parts(const PrefillArgs& a, const int* joins, int n_joins, int rows, int parts, int tile, hipStream_t stream) {
  if (!n_joins) return;
  if (parts <= 4)
    block_prefill_join_kernel<1><<<dim3((rows + 7) / 8, a.n_kv, n_joins), 256, 0, stream>>>(a.out, a.ws_o, a.ws_ml, joins, a.cu, a.tokens, a.n_kv, a.G, tile);
  else
    block_prefill_join_kernel<8><<<dim3(rows, a.n_kv, n_joins), 256, 0, stream>>>(a.out, a.ws_o, a.ws_ml, joins, a.cu, a.tokens, a.n_kv, a.G, tile);
}

}  // namespace

// q [T, Hq, 128] rows q_stride apart (16-byte aligned); out [T, Hq, 128]; tokens: T; work [n_work + n_few][6] (tiles, then sequences of few rows),
// joins [n_joins + n_few_joins][4] and the places of their sums (ws_o [places, Hkv, tile, 128], ws_ml [..., 2] fp32; few: [places, Hkv,
// 32, ...]) as the plan says; join_rows, most_parts: rows and parts that a joined item has at most; tile: rows of a work item (64, 128, 256); few_groups: 16s of rows (1, 2).  code: 0 int8, 1 e4m3fn.
extern "C" int dx_block_prefill(void* out, float* ws_o, float* ws_ml, float* few_o, float* few_ml, const void* q, int64_t q_stride, const void* k,
                                const void* v, const float* ks, const float* vs, const int* block_tables, int bt_stride, int bt_cols, const int* cu,
                                const int* ctx_lens, const int* work, int n_work, int n_few, const int* joins, int n_joins, int n_few_joins, int join_rows,
                                int few_join_rows, int most_parts, int few_most_parts, int tile, int few_groups, int n_q, int n_kv, int head_dim, int block_size, int num_blocks, int tokens, float scale, int causal, int code,
                                hipStream_t stream) {
  if (head_dim != D || block_size < 16 || (block_size & (block_size - 1)) || n_kv < 1 || n_kv > 65535 || tokens < 0 || n_q < 1 || n_q % n_kv || q_stride % 8 || bt_cols < 1 ||
      (tile != 64 && tile != 128 && tile != 256) || (few_groups != 1 && few_groups != 2) || n_work > 65535 || n_few > 65535 || n_joins > 65535 ||
      n_few_joins > 65535 || (n_joins && (join_rows < 1 || join_rows > tile)) || (n_few_joins && (few_join_rows < 1 || few_join_rows > kFewRows)))
    return -1;
  PrefillArgs a{};
  a.out = (bf16_t*)out, a.ws_o = ws_o, a.ws_ml = ws_ml, a.q = (const bf16_t*)q;
  a.k = (const uint8_t*)k, a.v = (const uint8_t*)v, a.ks = ks, a.vs = vs;
  a.block_tables = block_tables, a.cu = cu, a.ctx_lens = ctx_lens, a.work = work;
  a.q_stride = q_stride, a.bt_stride = bt_stride, a.bt_cols = bt_cols;
  a.n_kv = n_kv, a.G = n_q / n_kv, a.bs_shift = __builtin_ctz((unsigned)block_size), a.num_blocks = num_blocks, a.causal = causal, a.tokens = tokens;
  a.scale_log2e = scale * 1.4426950408889634f;
  if (n_work) {
    const dim3 grid(n_kv, n_work);
    a.tile = tile;
#define DX_BPT(C, RW, KW, ONE) block_prefill_kernel<C, RW, KW, ONE><<<grid, 64 * RW * KW, 0, stream>>>(a)
#define DX_BP(C)                                                                                      \
  do {                                                                                                \
    if (tile == 256) block_size >= 64 ? DX_BPT(C, 8, 1, true) : DX_BPT(C, 8, 1, false);               \
    else if (tile == 128) block_size >= 64 ? DX_BPT(C, 4, 1, true) : DX_BPT(C, 4, 1, false);          \
    else block_size >= 32 ? DX_BPT(C, 2, 4, true) : DX_BPT(C, 2, 4, false);                           \
  } while (0)
    if (code == kE4m3) DX_BP(kE4m3);
    else DX_BP(kInt8);
#undef DX_BP
#undef DX_BPT
    join_parts(a, joins, n_joins, join_rows, most_parts, tile, stream);
  }
  if (n_few) {
    a.work = work + kItem * n_work, a.ws_o = few_o, a.ws_ml = few_ml;
    const dim3 grid(n_kv, n_few);
#define DX_BR(C)                                                                       \
  do {                                                                                 \
    if (few_groups == 1) block_rows_kernel<C, 1><<<grid, 256, 0, stream>>>(a);         \
    else block_rows_kernel<C, 2><<<grid, 256, 0, stream>>>(a);                         \
  } while (0)
    if (code == kE4m3) DX_BR(kE4m3);
    else DX_BR(kInt8);
#undef DX_BR
    join_parts(a, joins + kJoin * n_joins, n_few_joins, few_join_rows, few_most_parts, kFewRows, stream);
  }
  return (int)hipGetLastError();
}
