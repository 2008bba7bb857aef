// Paged causal prompt attention (ragged chunks behind cached tokens, grouped heads of 128) over the 8-bit cache whose scales
// belong to a block and head (block8.h), for gfx950:
//   out[i, h] = sum_j p_j v_j,  p = softmax_j(scale q_i . k_j),  j <= position of i (causal) or j < ctx
// with k_j, v_j the cache's values, rounded to bf16 where their scales are no powers of two.
//
// Bound by the matrix products of long chunks and by the cache's bytes of short ones.  A workgroup takes 32 rows a wave of one
// key/value head, a row being one query head of one token (token-major: row = token G + head), so that chunks of few tokens fill
// waves at any group size, and a wave's rows span few positions.  Tiles of 64 keys: their codes are asked for a tile ahead, 16
// bytes a lane, and become bf16 in a swizzled double-buffered LDS image behind the tile's products (a workgroup widens a code once
// for all its rows).  S^T = K Q^T and O^T = V^T P^T on 32 x 32 x 16 products: a lane's scores are one row's, the softmax is
// lane-local but for one exchange between the halves, the weights are the second product's operand as they are, V is read
// transposed, and the row sum is a product with ones (of the bf16 weights that the second product sees).  The running maximum
// moves when a tile's exceeds it by 2^8.
//
// Few rows behind many keys are split over the keys (the plan says where), each part leaves its sums in fp32, and a second kernel
// joins them.
#include "block8.h"

#include <type_traits>

namespace {

constexpr int D = 128, BQ = 32, BKV = 64;
constexpr int kTileBytes = BKV * D * 2;
constexpr int kItem = 6;  // seq, first row, first key, end of the keys, place of its sums (or -1), 0
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
  int bt_stride, bt_cols, n_kv, G, bs_shift, num_blocks, causal;
  float scale_log2e;
};

template <int CODE, int NW>
__global__ void __launch_bounds__(64 * NW, 2) block_prefill_kernel(const PrefillArgs a) {
  constexpr float kRescale = 8.0f;
  constexpr int PIECES = 8 / NW;  // pieces of 8 rows of a tile that a wave brings
  __shared__ __attribute__((aligned(16))) char smem[2 * 2 * kTileBytes];
  const int* item = a.work + (int64_t)blockIdx.y * kItem;
  const int kvh = blockIdx.x, G = a.G;
  const int seq = __builtin_amdgcn_readfirstlane(item[0]), row0 = __builtin_amdgcn_readfirstlane(item[1]);
  const int key0 = __builtin_amdgcn_readfirstlane(item[2]), key1 = __builtin_amdgcn_readfirstlane(item[3]), place = __builtin_amdgcn_readfirstlane(item[4]);
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 31, h = lane >> 5;
  const int q_start = __builtin_amdgcn_readfirstlane(a.cu[seq]), qlen = __builtin_amdgcn_readfirstlane(a.cu[seq + 1]) - q_start;
  const int ctx = __builtin_amdgcn_readfirstlane((int)min((int64_t)a.ctx_lens[seq], (int64_t)a.bt_cols << a.bs_shift));
  const int pos0 = ctx - qlen, rows = qlen * G;
  const int w0 = row0 + BQ * wid, f = w0 + r;
  const bool valid = f < rows;
  const int tok = f / G, hq = f - tok * G;
  const int my_pos = a.causal ? pos0 + tok : ctx - 1;
  const int wave_min = a.causal ? pos0 + w0 / G : ctx - 1;
  const int wave_max = w0 >= rows ? -1 : a.causal ? pos0 + min(w0 + BQ - 1, rows - 1) / G : ctx - 1;
  const int wg_max = a.causal ? pos0 + min(row0 + BQ * NW - 1, rows - 1) / G : ctx - 1;
  const int kv_end = min(min(key1, ctx), wg_max + 1);
  const int n_tiles = max(kv_end - key0 + BKV - 1, 0) / BKV;

  u16x8 qf[8];
  {
    const bf16_t* qp = a.q + (int64_t)(q_start + tok) * a.q_stride + (int64_t)(kvh * G + hq) * D + 8 * h;
#pragma unroll
    for (int s = 0; s < 8; ++s) qf[s] = valid ? *reinterpret_cast<const u16x8*>(qp + 16 * s) : u16x8{{0, 0, 0, 0}};
  }
  int koff[8], voff[4][2];
#pragma unroll
  for (int s = 0; s < 8; ++s) koff[s] = tile_off(r, 2 * s + h);
  {
    const int g16 = (lane >> 4) & 1, qq = (lane & 15) >> 2, pp = lane & 3;
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) {
      const int ch = dt * 4 + 2 * g16 + (pp >> 1);
      voff[dt][0] = tile_off(4 * h + qq, ch) + 8 * (pp & 1);
      voff[dt][1] = tile_off(4 * h + qq + 8, ch) + 8 * (pp & 1);
    }
  }
  // ---- a tile's codes: piece p of this wave is rows 8 (PIECES wid + p) .. + 7, a lane 16 columns of one of them
  const int* bt = a.block_tables + (int64_t)seq * a.bt_stride;
  const int last = max(ctx - 1, 0) >> a.bs_shift;
  int first = -64, ids = 0;
  raw4 kr[PIECES], vr[PIECES];
  float ksc[PIECES], vsc[PIECES];
  auto load = [&](int t) __attribute__((always_inline)) {
    const int j0 = key0 + t * BKV;
    if (min((j0 + BKV - 1) >> a.bs_shift, last) - first >= 64) {  // 64 entries of the table at a time, a lane each
      first = j0 >> a.bs_shift;
      const int id = bt[min(first + lane, last)];
      ids = (unsigned)id < (unsigned)a.num_blocks ? id : 0;
    }
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
      const int at = 8 * (PIECES * wid + p), j = j0 + at;
      const int64_t block = (int64_t)__builtin_amdgcn_readlane(ids, min(j >> a.bs_shift, last) - first) * a.n_kv + kvh;
      const int64_t base = ((block << a.bs_shift) + (j & ((1 << a.bs_shift) - 1)) + (lane >> 3)) * D + 16 * (lane & 7);
      ksc[p] = a.ks[block], vsc[p] = a.vs[block];
      kr[p] = *reinterpret_cast<const raw4*>(a.k + base);
      vr[p] = *reinterpret_cast<const raw4*>(a.v + base);
      if (j + (lane >> 3) >= ctx) kr[p] = vr[p] = raw4{0u, 0u, 0u, 0u};  // (whatever lies behind the context may be a NaN)
    }
  };
  auto store = [&](char* kb) __attribute__((always_inline)) {
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
      const int row = 8 * (PIECES * wid + p) + (lane >> 3);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int to = tile_off(row, 2 * (lane & 7) + c);
        const raw2 k0 = widen4_bf16<CODE, true>(kr[p][2 * c], ksc[p]), k1 = widen4_bf16<CODE, true>(kr[p][2 * c + 1], ksc[p]);
        const raw2 v0 = widen4_bf16<CODE, true>(vr[p][2 * c], vsc[p]), v1 = widen4_bf16<CODE, true>(vr[p][2 * c + 1], vsc[p]);
        *reinterpret_cast<raw4*>(kb + to) = raw4{k0[0], k0[1], k1[0], k1[1]};
        *reinterpret_cast<raw4*>(kb + kTileBytes + to) = raw4{v0[0], v0[1], v1[0], v1[1]};
      }
    }
  };

  f32x16 o_acc[4], l_acc = f32x16{};
#pragma unroll
  for (int i = 0; i < 4; ++i) o_acc[i] = f32x16{};
  float m_i = -1e30f;
  const bf16x8_t kOnes = __builtin_bit_cast(bf16x8_t, u16x8{{0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u}});
  const f32x2 sc2 = {a.scale_log2e, a.scale_log2e};
  auto vread = [&](const char* vb, int i) __attribute__((always_inline)) {  // columns 32 (i % 4) .. + 31 of keys 16 (i / 4) .. + 15
    const i16x4 lo = read_tr16((const lds_i16x4*)(vb + i / 4 * 4096 + voff[i % 4][0]));
    const i16x4 hi = read_tr16((const lds_i16x4*)(vb + i / 4 * 4096 + voff[i % 4][1]));
    return __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  };
  auto compute = [&](const char* kb, int t) __attribute__((always_inline)) {
    const int j0 = key0 + t * BKV;
    if (j0 > wave_max) return;
    const bool live1 = j0 + 32 <= wave_max;
    f32x16 s0 = f32x16{}, s1 = f32x16{};
    auto kread = [&](int i) __attribute__((always_inline)) { return __builtin_bit_cast(bf16x8_t, *reinterpret_cast<const raw4*>(kb + 8192 * (i >> 3) + koff[i & 7])); };
#pragma unroll
    for (int s = 0; s < 8; ++s) s0 = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kread(s), __builtin_bit_cast(bf16x8_t, qf[s]), s0, 0, 0, 0);
    if (live1) {
#pragma unroll
      for (int s = 0; s < 8; ++s) s1 = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kread(8 + s), __builtin_bit_cast(bf16x8_t, qf[s]), s1, 0, 0, 0);
    }
    if (j0 + BKV - 1 > wave_min || j0 + BKV > ctx) {  // the diagonal, or the context's end
      const int lim = min(my_pos, ctx - 1) - j0 - 4 * h;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int off = (i & 3) + 8 * (i >> 2);
        s0[i] = off > lim ? -INFINITY : s0[i];
        s1[i] = off + 32 > lim ? -INFINITY : s1[i];
      }
    }
    float ta = fmaxf(s0[0], s1[0]), tb = fmaxf(s0[1], s1[1]);
#pragma unroll
    for (int i = 2; i < 16; i += 2) {
      ta = fmaxf(fmaxf(ta, s0[i]), s1[i]);
      tb = fmaxf(fmaxf(tb, s0[i + 1]), s1[i + 1]);
    }
    const float t_s = halves_max(fmaxf(ta, tb)) * a.scale_log2e;
    const float m_new = t_s > m_i + kRescale ? t_s : m_i;
    const float alpha = fast_exp2(m_i - m_new);
    m_i = m_new;
    const f32x2 nm2 = {-m_new, -m_new};
    u16x8 pf[2][2];
#pragma unroll
    for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int i = 8 * s2 + 2 * w;
        const f32x2 a0 = f32x2{s0[i], s0[i + 1]} * sc2 + nm2;
        const f32x2 a1 = f32x2{s1[i], s1[i + 1]} * sc2 + nm2;
        pf[0][s2].w[w] = pack_bf16x2(fast_exp2(a0.x), fast_exp2(a0.y));
        pf[1][s2].w[w] = pack_bf16x2(fast_exp2(a1.x), fast_exp2(a1.y));
      }
    if (__builtin_amdgcn_ballot_w64(alpha != 1.f)) {
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) o_acc[dt] *= alpha;
      l_acc *= alpha;
    }
    const char* vb = kb + kTileBytes;
#pragma unroll
    for (int sub = 0; sub < 2; ++sub)
      if (sub == 0 || live1) {
#pragma unroll
        for (int i = 8 * sub; i < 8 * sub + 8; ++i) {
          const bf16x8_t p = __builtin_bit_cast(bf16x8_t, pf[sub][(i >> 2) & 1]);
          o_acc[i & 3] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vread(vb, i), p, o_acc[i & 3], 0, 0, 0);
          if ((i & 3) == 3) l_acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kOnes, p, l_acc, 0, 0, 0);
        }
      }
  };

  if (n_tiles > 0) {
    load(0);
    store(smem);
  }
  __syncthreads();
  for (int t = 0; t < n_tiles; ++t) {
    char *now = smem + (t & 1) * 2 * kTileBytes, *next = smem + ((t + 1) & 1) * 2 * kTileBytes;
    if (t + 1 < n_tiles) load(t + 1);
    compute(now, t);
    if (t + 1 < n_tiles) store(next);
    __syncthreads();
  }

  // ---- lane (r, h) holds columns 32 dt + 8 g + 4 h .. + 3 of its row
  const float l_i = l_acc[0];
  if (place >= 0) {  // (the sums as they are; rows that are none hold zeros)
    const int64_t row = ((int64_t)place * a.n_kv + kvh) * (BQ * NW) + BQ * wid + r;
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4*>(a.ws_o + row * D + 32 * dt + 8 * g + 4 * h) =
            f32x4{o_acc[dt][4 * g], o_acc[dt][4 * g + 1], o_acc[dt][4 * g + 2], o_acc[dt][4 * g + 3]};
    if (h == 0) *reinterpret_cast<f32x2*>(a.ws_ml + row * 2) = f32x2{m_i, l_i};
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

// one row a wave: its parts' sums under a common maximum, over their common sum
__global__ void __launch_bounds__(256) block_prefill_join_kernel(bf16_t* __restrict__ out, const float* __restrict__ ws_o, const float* __restrict__ ws_ml,
                                                                 const int* __restrict__ joins, const int* __restrict__ cu, int n_kv, int G, int tile) {
  const int lane = threadIdx.x & 63, in = blockIdx.x * 4 + (threadIdx.x >> 6), kvh = blockIdx.y;
  const int* item = joins + (int64_t)blockIdx.z * kJoin;
  const int seq = item[0], f = item[1] + in, place = item[2], n = item[3];
  const int q_start = cu[seq], rows = (cu[seq + 1] - q_start) * G;
  if (f >= rows) return;
  const int64_t step = (int64_t)n_kv * tile, row = ((int64_t)place * n_kv + kvh) * tile + in;
  float M = -1e30f;
  for (int p = lane; p < n; p += 64) M = fmaxf(M, ws_ml[(row + p * step) * 2]);
  M = wave_reduce_max(M);
  float den = 0.f;
  f32x2 sum = {0.f, 0.f};
#pragma unroll 4
  for (int p = 0; p < n; ++p) {
    const f32x2 ml = *reinterpret_cast<const f32x2*>(ws_ml + (row + p * step) * 2);
    const f32x2 x = *reinterpret_cast<const f32x2*>(ws_o + (row + p * step) * D + 2 * lane);
    const float w = fast_exp2(ml.x - M);
    den += w * ml.y;
    sum += w * x;
  }
  const float inv = den != 0.f ? 1.f / den : 0.f;
  const int tok = f / G, hq = f - tok * G;
  reinterpret_cast<uint32_t*>(out + ((int64_t)(q_start + tok) * n_kv * G + kvh * G + hq) * D)[lane] = pack_bf16x2(sum.x * inv, sum.y * inv);
}

}  // namespace

// q [T, Hq, 128] rows q_stride apart (16-byte aligned); out [T, Hq, 128]; work [n_work][6], joins [n_joins][4] and the places of their
// sums (ws_o [places, Hkv, 32 waves, 128], ws_ml [..., 2] fp32) as the plan says.  code: 0 int8, 1 e4m3fn.
extern "C" int dx_block_prefill(void* out, float* ws_o, float* ws_ml, const void* q, int64_t q_stride, const void* k, const void* v, const float* ks,
                                const float* vs, const int* block_tables, int bt_stride, int bt_cols, const int* cu, const int* ctx_lens,
                                const int* work, int n_work, const int* joins, int n_joins, int waves, int n_q, int n_kv, int head_dim,
                                int block_size, int num_blocks, float scale, int causal, int code, hipStream_t stream) {
  if (head_dim != D || block_size < 16 || (block_size & (block_size - 1)) || n_kv < 1 || n_kv > 65535 || n_q % n_kv || q_stride % 8 || bt_cols < 1 ||
      (waves != 4 && waves != 8) || n_work > 65535 || n_joins > 65535)
    return -1;
  if (n_work == 0) return 0;
  PrefillArgs a{};
  a.out = (bf16_t*)out, a.ws_o = ws_o, a.ws_ml = ws_ml, a.q = (const bf16_t*)q;
  a.k = (const uint8_t*)k, a.v = (const uint8_t*)v, a.ks = ks, a.vs = vs;
  a.block_tables = block_tables, a.cu = cu, a.ctx_lens = ctx_lens, a.work = work;
  a.q_stride = q_stride, a.bt_stride = bt_stride, a.bt_cols = bt_cols;
  a.n_kv = n_kv, a.G = n_q / n_kv, a.bs_shift = __builtin_ctz((unsigned)block_size), a.num_blocks = num_blocks, a.causal = causal;
  a.scale_log2e = scale * 1.4426950408889634f;
  const dim3 grid(n_kv, n_work);
#define DX_BP(C)                                                                       \
  do {                                                                                 \
    if (waves == 8) block_prefill_kernel<C, 8><<<grid, 512, 0, stream>>>(a);           \
    else block_prefill_kernel<C, 4><<<grid, 256, 0, stream>>>(a);                      \
  } while (0)
  if (code == kE4m3) DX_BP(kE4m3);
  else DX_BP(kInt8);
#undef DX_BP
  if (n_joins)
    block_prefill_join_kernel<<<dim3(8 * waves, n_kv, n_joins), 256, 0, stream>>>((bf16_t*)out, ws_o, ws_ml, joins, cu, n_kv, n_q / n_kv, 32 * waves);
  return (int)hipGetLastError();
}
