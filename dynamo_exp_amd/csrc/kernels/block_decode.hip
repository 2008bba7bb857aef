// Paged decode attention (one query row per sequence, grouped heads of 128) over the 8-bit cache whose scales belong to a block
// and head (block8.h), for gfx950:
//   out[b, h] = sum_j p_j vs_j v_j,  p = softmax_j(scale ks_j (q . k_j)),  j < ctx[b];  0 where ctx[b] is 0
// with k_j, v_j the codes of token j and ks_j, vs_j the scales of its block.
//
// Bound by HBM: a (token, head) row of codes is read once, 2 x 128 bytes, and serves the G query heads of its group, which are
// columns of the matrix products.  Balanced parts of a context, joined by a second kernel, as in the bf16 form
// (decode_join.h); a workgroup's waves take chunks of 32 tokens in turn, their K and V on their way a chunk ahead.  Four waves, or eight
// where contexts are short and few enough to be left whole (at most 768 tokens, a workgroup a CU): the join, a launch of its own, costs
// more than two chunks more.
//
// Codes widen to bf16 exactly, so the products see them without their scales: ks is a factor of a lane's scores (a lane's eight
// tokens lie in one half of a chunk, thus in one block of 16 or more), and vs one of its weights before they are rounded to bf16
// for the second product (relative 2^-8 each, as in the bf16 form; a power of two leaves that rounding as it is).  The row sum is
// taken of the unrounded weights in fp32.
//
// 96 sequences of up to 3150 tokens, 32 / 8 heads, int8: 89 us, 5.5 TB/s; three of up to 60001, 64 / 8 heads, e4m3: 38.5 us with the join, 5.4
// TB/s; one of 700 8.7 us, 44 of up to 76 in blocks of 16 5.5, both latency.
//
// Layouts of a chunk (lane = 16 g + r): S^T row block bb, row rho -> token 8 (rho >> 2) + 4 bb + (rho & 3), so that a lane's eight
// scores of head r are tokens 8 g .. 8 g + 7 and, as bf16, the B operand of O^T = V^T P^T.  K comes straight from global memory (a
// lane's 32 bytes are columns 32 g ..), V goes through a wave's own 8 KB image in LDS and is read transposed.
#include "block8.h"
#include "decode_join.h"

#include <type_traits>

namespace {

constexpr int D = kHeadDim, CH = 32;

__device__ __forceinline__ int vimg_off(int row, int ch) {  // byte offset of 16-B chunk ch of row in a wave's image
  return row * 256 + 16 * (ch ^ (((row & 3) << 2) | ((row >> 2) & 3)));
}
template <typename F> __device__ __forceinline__ float over_groups(float x, F f) { return over_row_pairs(over_halves(x, f), f); }

struct DecodeArgs {
  bf16_t* out;
  float *tmp_out, *tmp_ml;
  const bf16_t* q;
  const uint8_t *k, *v;
  const float *ks, *vs;
  const int *block_tables, *ctx_lens;
  int64_t q_stride;
  int bt_stride, bt_cols, n_kv, G, bs_shift, num_blocks;
  float scale_log2e;
};

template <int CODE, int NW>
__global__ void __launch_bounds__(64 * NW, NW == 4 ? 3 : 2) block_decode_kernel(const DecodeArgs a) {
  constexpr int kThreads = 64 * NW;
  constexpr float kRescale = 8.0f;  // the running maximum moves when a chunk's exceeds it by 2^8
  __shared__ __attribute__((aligned(16))) char image[NW * CH * D * 2];
  __shared__ float st_m[NW * 16], st_l[NW * 16];
  const int pid = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z, n_parts = gridDim.x, G = a.G;
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, r = lane & 15;
  const int64_t qh0 = ((int64_t)b * a.n_kv + kvh) * G;
  // the part's blocks, 64 at a time, a lane each; the first 64 of the context are asked for beside its length, not behind it (a table's
  // columns are all that may be read of it)
  const int* bt = a.block_tables + (int64_t)b * a.bt_stride;
  int first = 0, ids = bt[min(lane, a.bt_cols - 1)];
  raw4 qf[4];
#pragma unroll
  for (int s = 0; s < 4; ++s)  // (columns behind the heads hold the last one's, and go nowhere)
    qf[s] = *reinterpret_cast<const raw4*>(a.q + b * a.q_stride + (int64_t)(kvh * G + min(r, G - 1)) * D + 8 * (4 * g + s));
  const int ctx = __builtin_amdgcn_readfirstlane((int)min((int64_t)a.ctx_lens[b], (int64_t)a.bt_cols << a.bs_shift));
  if (ctx <= 0) {
    if (n_parts == 1)
      for (int i = threadIdx.x; i < G * D / 2; i += kThreads) reinterpret_cast<uint32_t*>(a.out + qh0 * D)[i] = 0;
    return;  // (of several parts, the join writes the zeros)
  }
  const int part = balanced_part(ctx, n_parts, 4 * CH);
  const int p0 = pid * part;
  if (p0 >= ctx) return;
  const int p1 = min(p0 + part, ctx);
  char* vimg = image + wid * (CH * D * 2);

  const int last = (ctx - 1) >> a.bs_shift;
  auto fetch = [&]() { ids = bt[min(first + lane, last)]; };
  if ((p1 - 1) >> a.bs_shift >= 64) {
    first = p0 >> a.bs_shift;
    fetch();
  }
  auto block_at = [&](int i) {
    if (i - first >= 64) {  // (chunks only go up)
      first = i;
      fetch();
    }
    const int id = __builtin_amdgcn_readlane(ids, max(i - first, 0));
    return (unsigned)id < (unsigned)a.num_blocks ? id : 0;
  };

  f32x4 oacc[8];
#pragma unroll
  for (int db = 0; db < 8; ++db) oacc[db] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m_i = -1e30f, l_i = 0.f;

  const int n_chunks = (p1 - p0 + CH - 1) / CH;
  raw4 kf[2][2];
  raw2 vr[8];
  float ks_l, vs_l;
  auto load = [&](int c) {
    const int cb = p0 + c * CH;
    // the two halves of 16 tokens, each in one block; one that starts behind the part is the first again (its rows are masked)
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
      kf[bb][0] = __builtin_nontemporal_load(reinterpret_cast<const raw4*>(p));
      kf[bb][1] = __builtin_nontemporal_load(reinterpret_cast<const raw4*>(p + 16));
    }
#pragma unroll
    for (int k = 0; k < 8; ++k)
      vr[k] = __builtin_nontemporal_load(reinterpret_cast<const raw2*>(a.v + (k < 4 ? base0 : base1) + (4 * (k & 3) + g) * D + 8 * r));
  };
  auto step = [&](auto more_, int c) {
    constexpr bool more = decltype(more_)::value;
    const int cb = p0 + c * CH;
    const bool partial = !more && cb + CH > p1;
    f32x4 sacc[2];
#pragma unroll
    for (int bb = 0; bb < 2; ++bb) {
      sacc[bb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const raw2 lo = widen4_bf16<CODE, false>(kf[bb][s >> 1][2 * (s & 1)], 1.f), hi = widen4_bf16<CODE, false>(kf[bb][s >> 1][2 * (s & 1) + 1], 1.f);
        sacc[bb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, raw4{lo[0], lo[1], hi[0], hi[1]}),
                                                           __builtin_bit_cast(bf16x8_t, qf[s]), sacc[bb], 0, 0, 0);
      }
    }
    if (partial) {  // (weights of 0 meet zeros: whatever lies behind the context may be a NaN)
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
    if constexpr (more) load(c + NW);
    float t[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) t[j] = sacc[j >> 2][j & 3] * kscale;
    if (partial) {
#pragma unroll
      for (int j = 0; j < 8; ++j) t[j] = cb + 8 * g + j >= p1 ? -INFINITY : t[j];
    }
    float cmax = fmaxf(fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])), fmaxf(fmaxf(t[4], t[5]), fmaxf(t[6], t[7])));
    cmax = over_groups(cmax, [](float x, float y) { return fmaxf(x, y); });
    const float m_new = cmax > m_i + kRescale ? cmax : m_i;
    const float alpha = fast_exp2(m_i - m_new);
    m_i = m_new;
    raw4 pf;
    float ps = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float x = fast_exp2(t[2 * w] - m_new), y = fast_exp2(t[2 * w + 1] - m_new);
      ps += x + y;
      pf[w] = pack_bf16x2(x * vscale, y * vscale);
    }
    if (partial) {  // (a scale behind the context may be anything)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        if (cb + 8 * g + 2 * w >= p1) pf[w] &= 0xffff0000u;
        if (cb + 8 * g + 2 * w + 1 >= p1) pf[w] &= 0x0000ffffu;
      }
    }
    l_i = l_i * alpha + ps;
    if (__builtin_amdgcn_ballot_w64(alpha != 1.f)) {
#pragma unroll
      for (int db = 0; db < 8; ++db) oacc[db] *= alpha;
    }
    const bf16x8_t pfrag = __builtin_bit_cast(bf16x8_t, pf);
#pragma unroll
    for (int db = 0; db < 8; ++db) {
      const int qq = r >> 2, pp = r & 3;
      const i16x4 lo = read_tr16((const lds_i16x4*)(vimg + vimg_off(8 * g + qq, 2 * db + (pp >> 1)) + 8 * (pp & 1)));
      const i16x4 hi = read_tr16((const lds_i16x4*)(vimg + vimg_off(8 * g + 4 + qq, 2 * db + (pp >> 1)) + 8 * (pp & 1)));
      oacc[db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7)), pfrag,
                                                         oacc[db], 0, 0, 0);
    }
  };
  int c = wid;
  if (c < n_chunks) {
    load(c);
    for (; c + NW < n_chunks; c += NW) step(std::true_type{}, c);
    step(std::false_type{}, c);
  }

  // a wave's (O, m, l) into its own image: lane (g, r < G) holds columns 16 db + 4 g .. of head r
  const float l_tot = over_groups(l_i, [](float x, float y) { return x + y; });
  if (r < G) {
    float* so = reinterpret_cast<float*>(vimg) + r * D + 4 * g;
#pragma unroll
    for (int db = 0; db < 8; ++db) *reinterpret_cast<f32x4*>(so + 16 * db) = oacc[db];
    if (g == 0) st_m[wid * 16 + r] = m_i, st_l[wid * 16 + r] = l_tot;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < G * D / 4; i += kThreads) {
    const int h = i / (D / 4), d = 4 * (i % (D / 4));
    float m[NW], l[NW], M = -1e30f;
    f32x4 o[NW];
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      m[w] = st_m[w * 16 + h], l[w] = st_l[w * 16 + h];
      o[w] = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(image + w * (CH * D * 2)) + h * D + d);
      M = fmaxf(M, m[w]);
    }
    float den = 0.f;
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float f = exp2f(m[w] - M);
      sum += f * o[w];
      den += f * l[w];
    }
    f32x4 val;
#pragma unroll
    for (int j = 0; j < 4; ++j) val[j] = den != 0.f ? sum[j] / den : 0.f;
    const int64_t qh = qh0 + h;
    if (n_parts == 1) {
      *reinterpret_cast<u32x2_a2*>(a.out + qh * D + d) = u32x2_a2{pack_bf16x2(val[0], val[1]), pack_bf16x2(val[2], val[3])};
    } else {
      const int64_t row = qh * n_parts + pid;
      *reinterpret_cast<f32x4_a4*>(a.tmp_out + row * D + d) = val;
      if (d == 0) *reinterpret_cast<f32x2_a4*>(a.tmp_ml + row * 2) = f32x2_a4{M, den};
    }
  }
}

}  // namespace

// q [B, Hq, 128] rows q_stride apart (16-byte aligned); out [B, Hq, 128]; block_tables [B, bt_cols], rows bt_stride apart; tmp_out
// [B, Hq, n_parts, 128], tmp_ml [B, Hq, n_parts, 2] fp32 (n_parts > 1 alone).  code: 0 int8, 1 e4m3fn.
extern "C" int dx_block_decode(void* out, float* tmp_out, float* tmp_ml, const void* q, int64_t q_stride, const void* k, const void* v,
                               const float* ks, const float* vs, const int* block_tables, int bt_stride, int bt_cols, const int* ctx_lens,
                               int batch, int n_q, int n_kv, int head_dim, int block_size, int num_blocks, int n_parts, float scale, int code,
                               hipStream_t stream) {
  if (head_dim != D || block_size < 16 || (block_size & (block_size - 1)) || n_parts < 1 || n_kv < 1 || n_q < 1 || n_q % n_kv || n_q / n_kv > 16 ||
      q_stride % 8 || batch > 65535 || n_kv > 65535 || bt_cols < 1)
    return -1;
  if (batch == 0) return 0;
  DecodeArgs a{};
  a.out = (bf16_t*)out, a.tmp_out = tmp_out, a.tmp_ml = tmp_ml, a.q = (const bf16_t*)q;
  a.k = (const uint8_t*)k, a.v = (const uint8_t*)v, a.ks = ks, a.vs = vs;
  a.block_tables = block_tables, a.ctx_lens = ctx_lens, a.q_stride = q_stride, a.bt_stride = bt_stride, a.bt_cols = bt_cols;
  a.n_kv = n_kv, a.G = n_q / n_kv, a.bs_shift = __builtin_ctz((unsigned)block_size), a.num_blocks = num_blocks;
  a.scale_log2e = scale * 1.4426950408889634f;
  const dim3 grid(n_parts, n_kv, batch);
  const bool eight = n_parts == 1 && (int64_t)batch * n_kv <= 256;
#define DX_BD(C)                                                               \
  do {                                                                         \
    if (eight) block_decode_kernel<C, 8><<<grid, 512, 0, stream>>>(a);         \
    else block_decode_kernel<C, 4><<<grid, 256, 0, stream>>>(a);               \
  } while (0)
  if (code == kE4m3) DX_BD(kE4m3);
  else DX_BD(kInt8);
#undef DX_BD
  if (n_parts > 1) join(a.out, tmp_out, tmp_ml, ctx_lens, n_q, batch, n_parts, 4 * CH, stream,
                        (int)min((int64_t)bt_cols * block_size, (int64_t)0x7fffffff));
  return (int)hipGetLastError();
}
