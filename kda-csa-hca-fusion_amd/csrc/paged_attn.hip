// Attention of a chunk of new tokens over the paged HCA cache (gfx950).
//
// Query p = ctx + i, head h of a sequence, q^ = q / max(||q||, 1e-12) (or q):
//   keys (which are the values too)  the compressed rows b < (p + 1) / m2 and the
//   window rows of positions max(0, p - win + 1) .. p
//   s = scale q^ K^T,  out = sum_k e^(s_k) K_k / (sum_k e^(s_k) + e^sink_h)
// and 0 where no key is visible (/root/reference/ops_hca.py:132-194 over a cache,
// /root/reference/ops_decoding_cache.py:1268-1395; chunks of one token are its
// decode step). The query is rounded to bf16 and so are the weights e^(s - M) in
// the second product, whose factors the matrix instruction takes in bf16; keys
// are exact in bf16 in every storage format, scores, sums and outputs are fp32.
//
// All heads share the keys (MQA), so the query rows of a sequence are its tokens
// times its heads, nh rows a token, and a 16-row MFMA tile may hold rows of
// several tokens: each lane masks its own row. A workgroup takes RG groups of
// 16 rows and streams the union of their keys through LDS, KC rows at a time:
// page entries two tiles ahead, rows one tile ahead in registers, converted to
// bf16 once on their way into LDS for all of the workgroup's rows. Where a step
// has few rows (one token of 16 heads is one group) the workgroup's waves split
// each tile's keys instead (KG waves a group) and their sums are joined at the
// end; long contexts are cut into ranges of keys, one workgroup each, whose
// partial sums a second kernel joins, so that a few sequences fill the device.
//
// A key row that is not finite (E8M0 code 255, or a non-finite bf16 channel)
// sits in LDS as zeros beside a NaN that is added to its scores: rows that do
// not see it stay as they are (0 times NaN would reach them in the second
// product), rows that do become NaN.

#include "paged.h"

namespace kch {

namespace {

constexpr int KC = 128;  // key rows of an LDS tile

// The keys of query tokens [ta, tb] (indices into the chunk) of a sequence: the
// first nc compressed rows, then nw window rows from position wlo on.
struct KeySpan {
  uint32_t nc, wlo, nw;
};
__device__ __forceinline__ uint32_t visible_blocks(const PagedAttnParams& p, uint32_t pos) {
  return min((pos + 1) / (uint32_t)p.m2, (uint32_t)p.pool.nbp << p.pool.log2page);
}
__device__ __forceinline__ KeySpan key_span(const PagedAttnParams& p, const PagedSeq& sq, int ta, int tb) {
  KeySpan k;
  const uint32_t pa = sq.ctx + ta, pb = sq.ctx + tb;
  k.nc = visible_blocks(p, pb);
  k.wlo = pa + 1 > (uint32_t)p.win ? pa + 1 - p.win : 0;
  k.nw = p.win > 0 && p.pool.nrp > 0 ? pb - k.wlo + 1 : 0;
  return k;
}
// Keys of one range: split_keys, or more where the spans are longer than the
// launch was laid out for.
__device__ __forceinline__ uint32_t range_keys(const PagedAttnParams& p, uint32_t total) {
  const uint32_t need = (total + p.nsplit - 1) / p.nsplit;
  return max((uint32_t)p.split_keys, (need + KC - 1) / KC * KC);
}

// RG groups of 16 rows, QW of them a wave, KG waves share a group's keys.
template <int HD, int FMT, int RG, int QW, int KG, typename T>
__global__ __launch_bounds__(64 * (RG / QW) * KG) void paged_attn_kernel(PagedAttnParams p) {
  using W = MqaWave<HD>;
  constexpr int NWV = RG / QW * KG, NTH = 64 * NWV;
  constexpr int ROWS = 16 * RG;
  constexpr int EPL = FMT == PF_BF16 ? 8 : 16;  // row elements of a lane's 16 bytes
  constexpr int TPR = HD / EPL;                 // lanes per key row
  constexpr int RSTEP = NTH / TPR;              // key rows of a load instruction of the workgroup
  constexpr int NLD = KC / RSTEP;
  static_assert(NLD >= 1 && KC % RSTEP == 0 && RSTEP % 16 == 0, "tile loads");
  static_assert(KG <= KC / 32, "a wave takes whole 32-key steps");
  __shared__ __attribute__((aligned(16))) bf16_t tile[2][KC * HD];
  __shared__ __attribute__((aligned(16))) float poison[2][KC];
  __shared__ int any_bad;  // some row so far is not finite
  __shared__ float join_ml[KG > 1 ? NWV : 1][16][2];

  const int tid = threadIdx.x;
  const PagedPool& pl = p.pool;
  if (blockIdx.y == (unsigned)pl.S) {  // the rows behind the last sequence
    if (blockIdx.z) return;
    const long long n0 = (long long)max(0, min(pl.cu[pl.S], pl.N)) * p.nh * HD, n1 = (long long)pl.N * p.nh * HD;
    for (long long i = n0 + 8ll * (blockIdx.x * NTH + tid); i < n1; i += 8ll * gridDim.x * NTH)
#pragma unroll
      for (int e = 0; e < 8; e += 4) Store4<T>::run(static_cast<T*>(p.out) + i + e, f32x4{0.f, 0.f, 0.f, 0.f}, 1.f);
    return;
  }
  const PagedSeq sq = paged_seq(pl, blockIdx.y);
  const int nrow = sq.len * p.nh;  // N nh is below 2^31
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63, q4 = lane >> 4, n = lane & 15;
  const int rg = wv / KG, kg = wv % KG;
  const uint32_t ring_cap = (uint32_t)pl.nrp << pl.log2page;
  const int lmask = (1 << pl.log2page) - 1;
  const int* const btab = pl.block_table + (size_t)sq.slot * pl.nbp;
  const int* const rtab = pl.ring_table + (size_t)sq.slot * pl.nrp;
  const TileOffsets<HD> to;

  // (r0 + the grid's rows cannot pass 2^31: both are at most N nh plus a tile)
  for (int r0 = blockIdx.x * ROWS; r0 < nrow; r0 += gridDim.x * ROWS) {
    const int ta = r0 / p.nh, tb = (min(r0 + ROWS, nrow) - 1) / p.nh;
    const KeySpan sp = key_span(p, sq, ta, tb);
    const uint32_t total = sp.nc + sp.nw;
    const uint32_t per = range_keys(p, total);
    const uint32_t k0 = per * blockIdx.z;
    if (k0 >= total && blockIdx.z) continue;
    const uint32_t k1 = min(total, k0 + per);
    const bool whole = total <= per;  // no other range: the output itself

    // Tile loads: thread tid takes 16 bytes (part tid % TPR) of key rows
    // tid / TPR + RSTEP i of the tile. Rows past k1, and rows whose table entry
    // names no page of the pool, are zeros.
    const int lrow = tid / TPR, lch = tid % TPR;
    const uint32_t wr = sp.nw ? sp.wlo % ring_cap : 0;
    int pg[NLD];
    uint4 pf[NLD];
    int code[NLD];
    auto line_of = [&](uint32_t j, bool& blk) -> uint32_t {
      blk = j < sp.nc;
      if (blk) return j;
      uint32_t r = wr + (j - sp.nc);
      return r >= ring_cap ? r % ring_cap : r;
    };
    auto load_pages = [&](uint32_t t0) {
#pragma unroll
      for (int i = 0; i < NLD; ++i) {
        const uint32_t j = t0 + lrow + RSTEP * i;
        pg[i] = -1;
        if (j < k1) {
          bool blk;
          const uint32_t r = line_of(j, blk);
          pg[i] = (blk ? btab : rtab)[r >> pl.log2page];
        }
      }
    };
    auto load_rows = [&](uint32_t t0) {
#pragma unroll
      for (int i = 0; i < NLD; ++i) {
        const uint32_t j = t0 + lrow + RSTEP * i;
        bool blk;
        const uint32_t r = line_of(j, blk);
        const bool ok = (unsigned)pg[i] < (unsigned)pl.P;
        const long long pr = ok ? ((long long)pg[i] << pl.log2page) + (r & lmask) : 0;
        pf[i] = make_uint4(0, 0, 0, 0);
        code[i] = 127;
        if (ok) {
          pf[i] = *reinterpret_cast<const uint4*>(static_cast<const char*>(pl.rows) +
                                                  (pr * TPR + lch) * 16);
          if constexpr (FMT != PF_BF16) code[i] = pl.scales[pr];
        }
      }
    };
    auto store_rows_lds = [&](int buf) {
      bool bad_any = false;
#pragma unroll
      for (int i = 0; i < NLD; ++i) {
        const int row = lrow + RSTEP * i;
        bf16_t* dst = tile[buf] + row * HD;
        const int sw = tile_swz<HD>(row & 15);
        if constexpr (FMT == PF_BF16) {
          const uint32_t w[4] = {pf[i].x, pf[i].y, pf[i].z, pf[i].w};
          bool bad = false;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            bad |= (w[e] & 0x7f80u) == 0x7f80u || (w[e] & 0x7f800000u) == 0x7f800000u;
          // the whole row is bad where one of its lanes is
          const unsigned long long g = __ballot(bad) >> (lane & ~(TPR - 1)) & ((1ull << TPR) - 1);
          if (g) pf[i] = make_uint4(0, 0, 0, 0);
          *reinterpret_cast<uint4*>(dst + 8 * (lch ^ sw)) = pf[i];
          if (lch == 0) poison[buf][row] = g ? __uint_as_float(0x7fc00000u) : 0.f;
          bad_any |= g != 0;
        } else {
          const bool bad = code[i] == kScaleNan;
          const float sc = row_scale(bad ? 127 : code[i]);
          const uint32_t keep = bad ? 0u : 0xffffffffu;
          const uint2 a = dequant4_bf16<FMT>(pf[i].x & keep, sc), b = dequant4_bf16<FMT>(pf[i].y & keep, sc);
          const uint2 c = dequant4_bf16<FMT>(pf[i].z & keep, sc), d = dequant4_bf16<FMT>(pf[i].w & keep, sc);
          *reinterpret_cast<uint4*>(dst + 8 * ((2 * lch) ^ sw)) = make_uint4(a.x, a.y, b.x, b.y);
          *reinterpret_cast<uint4*>(dst + 8 * ((2 * lch + 1) ^ sw)) = make_uint4(c.x, c.y, d.x, d.y);
          if (lch == 0) poison[buf][row] = bad ? __uint_as_float(0x7fc00000u) : 0.f;
          bad_any |= bad;
        }
      }
      if (bad_any) any_bad = 1;
    };

    // the first tile's rows are in flight while the queries load
    const uint32_t nt = (k1 - min(k0, k1) + KC - 1) / KC;
    if (nt) {
      load_pages(k0);
      load_rows(k0);
      load_pages(k0 + KC);
    }

    W w[QW];
    uint32_t vis[QW], lo[QW], hi[QW];  // this lane's row: keys [0, vis) and [lo, hi)
    int head[QW];
#pragma unroll
    for (int u = 0; u < QW; ++u) {
      const int r = r0 + 16 * (QW * rg + u) + n;
      const bool live = r < nrow;
      const int rr = live ? r : nrow - 1;
      const int tok = rr / p.nh;
      head[u] = rr - tok * p.nh;
      const T* qrow = static_cast<const T*>(p.q) + ((long long)sq.row0 * p.nh + rr) * HD;
      w[u].template init_always<T>(qrow, live, p.normalize_q != 0, p.scale);
      const uint32_t pos = sq.ctx + tok;
      vis[u] = live ? visible_blocks(p, pos) : 0;
      lo[u] = hi[u] = 0;
      if (live && sp.nw) {
        const uint32_t f = pos + 1 > (uint32_t)p.win ? pos + 1 - p.win : 0;
        lo[u] = sp.nc + (f - sp.wlo);
        hi[u] = sp.nc + (pos - sp.wlo) + 1;
      }
    }

    // 32 keys (tile rows from `rows`, key index j0 of the first)
    auto keys32 = [&](const bf16_t* rows, const float* pz, bool bad, uint32_t j0) {
      f32x4 sa[QW], sb[QW];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        bf16x8 kf[W::NS];
#pragma unroll
        for (int s = 0; s < W::NS; ++s) kf[s] = *reinterpret_cast<const bf16x8*>(rows + 16 * HD * h + to.key(s));
#pragma unroll
        for (int u = 0; u < QW; ++u) {
          if (h == 0) sa[u] = w[u].scores(kf);
          else sb[u] = w[u].scores(kf);
        }
      }
      bf16x8 pb[QW];
#pragma unroll
      for (int u = 0; u < QW; ++u) {
        float sc[8] = {sa[u][0], sa[u][1], sa[u][2], sa[u][3], sb[u][0], sb[u][1], sb[u][2], sb[u][3]};
        if (bad) {
#pragma unroll
          for (int e = 0; e < 8; ++e) sc[e] += pz[4 * q4 + (e < 4 ? e : 12 + e)];
        }
        const bool full = j0 + 32 <= k1 && (j0 + 32 <= vis[u] || (j0 >= lo[u] && j0 + 32 <= hi[u]));
        if (__ballot(!full)) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const uint32_t j = j0 + 4 * q4 + (e < 4 ? e : 12 + e);
            const bool ok = j < k1 && (j < vis[u] || (j >= lo[u] && j < hi[u]));
            sc[e] = ok ? sc[e] : -INFINITY;
          }
        }
        pb[u] = w[u].softmax32(sc);
      }
#pragma unroll
      for (int t = 0; t < W::NT; ++t) {
        const bf16x8 va = W::vt_frag(rows, to, t);
#pragma unroll
        for (int u = 0; u < QW; ++u)
          w[u].o[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, pb[u], w[u].o[t], 0, 0, 0);
      }
    };

    if (tid == 0) any_bad = 0;
    __syncthreads();  // the buffers of the last row tile are free
    if (nt) store_rows_lds(0);
    __syncthreads();
    for (uint32_t t = 0; t < nt; ++t) {
      const int buf = t & 1;
      const uint32_t j0 = k0 + t * KC;
      if (t + 1 < nt) {
        load_rows(j0 + KC);
        load_pages(j0 + 2 * KC);
      }
      const bool bad = any_bad != 0;  // (set early for the next tile: this one's poison is 0)
#pragma unroll
      for (int s = 0; s < KC / 32 / KG; ++s) {
        const int at = 32 * (s * KG + kg);
        if (j0 + at < k1) keys32(tile[buf] + at * HD, poison[buf] + at, bad, j0 + at);
      }
      if (t + 1 < nt) store_rows_lds(buf ^ 1);
      __syncthreads();
    }

    // sums of the row: over its four lanes, then over the waves that shared it
    char* const stage = reinterpret_cast<char*>(&tile[0][0]) + wv * 16 * HD * 4;
    static_assert(NWV * 16 * HD * 4 <= (int)sizeof(tile), "the staged outputs fit in the tiles");
#pragma unroll
    for (int u = 0; u < QW; ++u) w[u].finalize();
    if constexpr (KG > 1) {
      static_assert(QW == 1, "waves that share keys take one group");
      float* const ob = reinterpret_cast<float*>(stage);
#pragma unroll
      for (int t = 0; t < W::NT; ++t) *reinterpret_cast<f32x4*>(ob + (t * 64 + lane) * 4) = w[0].o[t];
      if (q4 == 0) {
        join_ml[wv][n][0] = w[0].M;
        join_ml[wv][n][1] = w[0].L;
      }
      __syncthreads();
      if (kg == 0) {
        float M = w[0].M;
#pragma unroll
        for (int g = 1; g < KG; ++g) M = fmaxf(M, join_ml[wv + g][n][0]);
        const float f0 = fast_exp2(w[0].M - M);
        w[0].L *= f0;
#pragma unroll
        for (int t = 0; t < W::NT; ++t) w[0].o[t] *= f0;
#pragma unroll
        for (int g = 1; g < KG; ++g) {
          const float f = fast_exp2(join_ml[wv + g][n][0] - M);
          w[0].L += f * join_ml[wv + g][n][1];
          const float* og = reinterpret_cast<const float*>(stage + g * 16 * HD * 4);
#pragma unroll
          for (int t = 0; t < W::NT; ++t) w[0].o[t] += f * *reinterpret_cast<const f32x4*>(og + (t * 64 + lane) * 4);
        }
        w[0].M = M;
      }
      __syncthreads();  // the partial outputs are read before their place is staged over
      if (kg != 0) continue;
    }
#pragma unroll
    for (int u = 0; u < QW; ++u) {
      const int r = r0 + 16 * (QW * rg + u);
      if (u > 0) wave_lds_sync();
      if (r >= nrow) break;
      const int live = min(16, nrow - r);
      const long long g = (long long)sq.row0 * p.nh + r;
      if (whole) {
        const float f = w[u].finish(p.sink != nullptr, p.sink ? p.sink[head[u]] : 0.f);
        store_rows<HD, T>(w[u].o, f, static_cast<T*>(p.out) + g * HD, live, stage);
      } else {
        const long long gp = (long long)blockIdx.z * pl.N * p.nh + g;
        store_rows<HD, float>(w[u].o, 1.f, p.part_o + gp * HD, live, stage);
        if (q4 == 0 && n < live) {
          p.part_ml[2 * (gp + n)] = w[u].M;
          p.part_ml[2 * (gp + n) + 1] = w[u].L;
        }
      }
    }
  }
}

// Joins the ranges of rows that have more than one: HD / 8 lanes a row.
template <int HD, typename T>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedAttnParams p, int tile_rows) {
  constexpr int LPR = HD / 8;
  const PagedSeq sq = paged_seq(p.pool, blockIdx.y);
  const int nrow = sq.len * p.nh;
  const int ch = 8 * (threadIdx.x % LPR);
  for (int r = blockIdx.x * (256 / LPR) + threadIdx.x / LPR; r < nrow; r += gridDim.x * (256 / LPR)) {
    const int r0 = r / tile_rows * tile_rows;
    const KeySpan sp = key_span(p, sq, r0 / p.nh, (min(r0 + tile_rows, nrow) - 1) / p.nh);
    const uint32_t total = sp.nc + sp.nw, per = range_keys(p, total);
    if (total <= per) continue;
    const int ns = (int)((total + per - 1) / per);
    const long long g = (long long)sq.row0 * p.nh + r, stride = (long long)p.pool.N * p.nh;
    float M = kMFloor;
    for (int s = 0; s < ns; ++s) M = fmaxf(M, p.part_ml[2 * (g + s * stride)]);
    float L = 0.f, o[8] = {};
    for (int s = 0; s < ns; ++s) {
      const float* ml = p.part_ml + 2 * (g + s * stride);
      const float f = fast_exp2(ml[0] - M);
      float v[8];
      Load8<float>::run(p.part_o + (g + s * stride) * HD + ch, v);
      L = fmaf(f, ml[1], L);
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = fmaf(f, v[i], o[i]);
    }
    float den = L;
    if (p.sink) den += fast_exp2(p.sink[r % p.nh] * kLog2eF - M);
    // as MqaWave::finish, with a NaN sum kept
    const float f = L == 0.f ? 0.f : 1.f / den;
    T* dst = static_cast<T*>(p.out) + g * HD + ch;
#pragma unroll
    for (int i = 0; i < 8; i += 4) Store4<T>::run(dst + i, f32x4{o[i], o[i + 1], o[i + 2], o[i + 3]}, f);
  }
}

// Row groups of a workgroup for rows query rows a sequence: all of them up to 4
// groups (fewer groups leave waves to split the keys), else 8.
int row_groups(long long rows) { return rows <= 16 ? 1 : rows <= 32 ? 2 : rows <= 64 ? 4 : 8; }

template <int HD, int FMT, typename T>
void attn_launch(const PagedAttnParams& p, int rows, hipStream_t s) {
  const long long nrow = (long long)p.max_len * p.nh;
  const dim3 grid((unsigned)((nrow + rows - 1) / rows), (unsigned)(p.pool.S + (p.zero_tail ? 1 : 0)),
                  (unsigned)p.nsplit);
#define KCH_PA(RG, QW, KG) \
  hipLaunchKernelGGL((paged_attn_kernel<HD, FMT, RG, QW, KG, T>), grid, dim3(64 * RG / QW * KG), 0, s, p)
  if (rows == 16) KCH_PA(1, 1, 4);
  else if (rows == 32) KCH_PA(2, 1, 2);
  else if (rows == 64) KCH_PA(4, 1, 1);
  else KCH_PA(8, 1, 1);
#undef KCH_PA
  if (p.nsplit > 1) {
    constexpr int RPB = 256 / (HD / 8);
    const dim3 jg((unsigned)((nrow + RPB - 1) / RPB), (unsigned)p.pool.S);
    hipLaunchKernelGGL((paged_join_kernel<HD, T>), jg, dim3(256), 0, s, p, rows);
  }
}

template <int HD, int FMT>
void attn_launch_t(const PagedAttnParams& p, int dtype, int rows, hipStream_t s) {
  if (dtype == DT_BF16) attn_launch<HD, FMT, bf16_t>(p, rows, s);
  else if (dtype == DT_F16) attn_launch<HD, FMT, _Float16>(p, rows, s);
  else attn_launch<HD, FMT, float>(p, rows, s);
}

}  // namespace

PagedAttnPlan paged_attn_plan(int S, int N, int nh, int c, int m2, int win, int max_len, int max_ctx) {
  PagedAttnPlan pl;
  const long long nrow = (long long)max_len * nh;
  pl.rows = 16 * row_groups(nrow);
  const long long tiles = (nrow + pl.rows - 1) / pl.rows * S;
  const long long keys = ((long long)max_ctx + max_len) / m2 + win + (pl.rows + nh - 1) / nh;
  // two workgroups for each of 256 CUs; a range no shorter than four tiles
  const long long want = 512 / (tiles > 0 ? tiles : 1);
  long long per = want > 1 ? (keys + want - 1) / want : keys;
  per = ((per < 4 * KC ? 4 * KC : per) + KC - 1) / KC * KC;
  pl.nsplit = (int)((keys + per - 1) / per);
  if (pl.nsplit < 1) pl.nsplit = 1;
  pl.split_keys = (int)(per < (1ll << 30) ? per : (1ll << 30));
  pl.bytes = pl.nsplit > 1 ? (size_t)pl.nsplit * N * nh * (c + 2) * sizeof(float) : 0;
  return pl;
}

hipError_t paged_attn_dispatch(const PagedAttnParams& p, const PagedAttnPlan& plan, int format, int dtype,
                               hipStream_t s) {
  if (p.pool.c == 128) {
    if (format == PF_BF16) attn_launch_t<128, PF_BF16>(p, dtype, plan.rows, s);
    else if (format == PF_E4M3) attn_launch_t<128, PF_E4M3>(p, dtype, plan.rows, s);
    else attn_launch_t<128, PF_INT8>(p, dtype, plan.rows, s);
  } else {
    if (format == PF_BF16) attn_launch_t<64, PF_BF16>(p, dtype, plan.rows, s);
    else if (format == PF_E4M3) attn_launch_t<64, PF_E4M3>(p, dtype, plan.rows, s);
    else attn_launch_t<64, PF_INT8>(p, dtype, plan.rows, s);
  }
  return hipGetLastError();
}

}  // namespace kch
