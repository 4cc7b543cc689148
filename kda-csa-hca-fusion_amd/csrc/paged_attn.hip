// Attention of a chunk of new tokens over the paged HCA cache (gfx950).
//
// Query p = ctx + i, head h of a sequence, q^ = q / max(||q||, 1e-12) (or q):
//   keys (which are the values too)  the compressed rows b < (p + 1) / m2 and the
//   window rows of positions max(0, p - win + 1) .. p
//   s = scale q^ K^T,  out = sum_k e^(s_k) K_k / (sum_k e^(s_k) + e^sink_h)
// and 0 where no key is visible (/root/reference/ops_hca.py:132-194 over a cache,
// /root/reference/ops_decoding_cache.py:1268-1395; chunks of one token are its
// decode step). The products take 16-bit operands: bf16, which has the range of fp32 that
// unnormalised queries and rows scaled by any power of two need and holds the rows of
// every storage format exactly; fp16, finer by three bits, where the queries are fp16, for
// what such a model's rows are fits it (paged.h). Scores, sums and outputs are fp32.
// A query enters as it is, times a power of two, and what is left of 1 / ||q|| multiplies
// the scores with the scale: a 16-bit query is not rounded again (but for fp16 channels
// below 2^-14 of the row's length, to 2^-25 of it). A second rounding took a bf16 output
// from 0.0020 off to 0.0026, where its own rounding leaves 0.0017. The weights
// e^(s - M) are rounded to the products' type, as such queries' outputs are. An fp32 query
// and its weights enter as the three bf16 parts that they are the sums of, three products
// for one, and its output is off by what fp32 sums are (with one bf16 part of each by 2e-3).
// That takes 48 us a call where bf16 queries take 31 (128 tokens of a batch), 240 where they
// take 116 (prompt chunks), and no longer for short contexts.
//
// All heads share the keys (MQA), so the query rows of a sequence are its tokens
// times its heads, nh rows a token, and a 16-row MFMA tile may hold rows of
// several tokens: each lane masks its own row. A workgroup takes RG groups of
// 16 rows and streams the union of their keys through LDS, KC rows at a time:
// page entries two tiles ahead, rows one tile ahead in registers, converted to
// bf16 once on their way into LDS for all of the workgroup's rows
// (paged_attn_kernel). Where a sequence has few rows (one token of 16 heads is one
// group) the call is bound by the rows' bytes, and the waves of a workgroup split
// the keys: each takes 32-key steps of its own through its own LDS, one in flight
// beside the one in LDS, without a barrier, and the waves' sums are joined at the end
// (paged_token_kernel). Long contexts are cut into ranges of keys, one workgroup
// each, whose partial sums a second kernel joins, so that a few sequences fill the
// device.
//
// A key row that is not finite (E8M0 code 255, or a non-finite bf16 channel)
// sits in LDS as zeros beside a NaN that is added to its scores: rows that do
// not see it stay as they are (0 times NaN would reach them in the second
// product), rows that do become NaN. A NaN among the e4m3 codes of a row is looked for
// where it matters, in a step that some row masks: its scores are NaN, and then the
// values go into the second product with zeros in its place (values_or_zero).
// (It costs 3%; looked for in the codes themselves 5 to 10%, with a copy of the products for
// it, which spills, 40%.)
//
// Measured (16 heads of 128, e4m3 rows, blocks of 128 tokens, a window of 128):
//   one token for each of 128 contexts of 512K to 1M tokens  31 us a call (traced, 28.6 to
//     31.0 and 4.4 to 4.6 the join), for 99.6 MB 3.2 TB/s (a large copy 5.1): bound by the
//     rows' bytes, by ranges that end at different times and by the join's launch
//   one token behind 5003, 51 KB  9.4 us: latencies one after another (the step's
//     arrays, page entries, rows, the second of a wave's steps, the waves' join)
//   up to 2048 tokens behind 64K to 128K in each of 8 sequences  116 us a call, 609 TFLOP/s
//     (130 to 137 under the tracer): the issue of vector instructions beside the products
//     (77 a 16 products, most of them the softmax; products busy for 35% of the cycles)

#include "paged.h"

namespace kch {

namespace {

constexpr int KC = 128;       // key rows of an LDS tile
constexpr int kStepUnit = 8;  // 32-key steps of a range: two a wave

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
// The same keys as 32-key steps of paged_token_kernel: nb steps of compressed
// rows, then nw of window rows. Where pages hold whole steps (at least 32 rows) a
// step never leaves its page: window steps then start at a multiple of 32 of the
// ring, woff rows before the first one.
struct KeySteps {
  uint32_t nb, nw, woff;
};
__device__ __forceinline__ KeySteps key_steps(const PagedAttnParams& p, const KeySpan& sp) {
  KeySteps k;
  k.nb = (sp.nc + 31) / 32;
  const uint32_t cap = (uint32_t)p.pool.nrp << p.pool.log2page;
  k.woff = sp.nw && p.pool.log2page >= 5 ? (sp.wlo % cap) & 31 : 0;
  k.nw = sp.nw ? (k.woff + sp.nw + 31) / 32 : 0;
  return k;
}
// Length of a range, in units of the kernel that takes it: the plan's, or more where
// the spans are longer than the launch was laid out for.
__device__ __forceinline__ uint32_t range_len(const PagedAttnParams& p, uint32_t total, uint32_t unit) {
  const uint32_t need = (total + p.nsplit - 1) / p.nsplit;
  return max((uint32_t)p.range, (need + unit - 1) / unit * unit);
}

// Output rows n0 .. n1 - 1 as zeros, by the workgroup.
template <int HD, typename T>
__device__ __forceinline__ void zero_rows(const PagedAttnParams& p, long long n0, long long n1) {
  for (long long i = n0 * HD + 4ll * threadIdx.x; i < n1 * HD; i += 4ll * blockDim.x)
    Store4<T>::run(static_cast<T*>(p.out) + i, f32x4{0.f, 0.f, 0.f, 0.f}, 1.f);
}
// Rows [r0, r1) as zeros, a share of each workgroup of the grid row.
template <int HD, typename T>
__device__ __forceinline__ void zero_shared(const PagedAttnParams& p, long long r0, long long r1) {
  const long long per = (r1 - r0 + gridDim.x - 1) / gridDim.x, at = r0 + per * blockIdx.x;
  zero_rows<HD, T>(p, at, min(r1, at + per));
}
// The rows that no workgroup computes, as zeros: those ahead of the first and behind the last
// sequence (a grid row of their own), the whole chunk of a sequence that is passed over,
// and what a chunk has past max_len.
template <int HD, typename T>
__device__ __forceinline__ void zero_ends(const PagedAttnParams& p) {
  if (blockIdx.z) return;
  const long long nh = p.nh, N = p.pool.N;
  zero_shared<HD, T>(p, 0, nh * max(0, min(p.pool.cu[0], p.pool.N)));
  zero_shared<HD, T>(p, nh * max(0, min(p.pool.cu[p.pool.S], p.pool.N)), nh * N);
}
template <int HD, typename T>
__device__ __forceinline__ void zero_rest(const PagedAttnParams& p, const PagedSeq& sq) {
  if (!p.zero_tail || blockIdx.z) return;
  const long long nh = p.nh;
  if (sq.len == 0)
    zero_shared<HD, T>(p, nh * max(0, min(sq.row0, p.pool.N)), nh * min(sq.end, p.pool.N));
  else if (sq.len > p.max_len)
    zero_shared<HD, T>(p, nh * (sq.row0 + p.max_len), nh * (sq.row0 + sq.len));
}
__device__ __forceinline__ int computed_rows(const PagedAttnParams& p, const PagedSeq& sq) {
  return min(sq.len, p.max_len) * p.nh;  // N nh is below 2^30
}

// The type of the products for queries of type T.
template <typename T> struct Prod { typedef bf16_t type; };
template <> struct Prod<_Float16> { typedef _Float16 type; };

// MqaWave for queries of type T. A product has kParts of them: an fp32 value is the sum of
// three bf16 ones (hi + mid + lo, 24 significant bits), and the keys are one exactly.
template <int HD, typename T> struct PagedWave : MqaWave<HD, typename Prod<T>::type> {
  typedef typename Prod<T>::type E;
  typedef MqaWave<HD, E> Base;
  typedef typename Base::v8 v8;
  typedef typename Base::f32x8 f32x8;
  static constexpr int kParts = __is_same(T, float) ? 3 : 1;
  v8 qx[kParts > 1 ? kParts - 1 : 1][Base::NS];  // mid and lo (hi: qf)

  // x's bf16 parts, the largest first.
  static __device__ __forceinline__ void parts(f32x8 x, v8 (&p)[kParts]) {
#pragma unroll
    for (int i = 0; i < kParts; ++i) {
      p[i] = __builtin_convertvector(x, v8);
      if (i + 1 < kParts) x -= __builtin_convertvector(p[i], f32x8);
    }
  }
  // The query of this lane's row, at q_row (always readable; zeros where it is not `keep`).
  // Normalised, it enters times the power of two of 1 / ||q||; the rest of that, in [1, 2),
  // goes into the scores' factor. (1 / ||q|| of an infinite sum of squares is 0, and so is
  // the query, its infinities NaN.)
  __device__ __forceinline__ void query(const T* q_row, bool keep, bool normalise, float scale) {
    const int q = lane_id() >> 4;
    float f[Base::NS][8], ss = 0.f;
#pragma unroll
    for (int s = 0; s < Base::NS; ++s) {
      Load8<T>::run(q_row + 32 * s + 8 * q, f[s]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        f[s][i] = keep ? f[s][i] : 0.f;
        ss += f[s][i] * f[s][i];
      }
    }
    const uint32_t inv = __float_as_uint(normalise ? l2_inv(colq_sum(ss)) : 1.f);
    const float two = __uint_as_float(inv & 0x7f800000u), rest = __uint_as_float((inv & 0x7fffffu) | 0x3f800000u);
    Base::setup(f, false, 0.f);
    Base::qscale2 = fmaxf(fabsf(scale) * kLog2eF * rest, 1e-30f);
    Base::thr = (kMFloor + kRescaleLog2) / Base::qscale2;
#pragma unroll
    for (int s = 0; s < Base::NS; ++s) {
      f32x8 x;
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = f[s][i] * (scale < 0.f ? -two : two);
      v8 p[kParts];
      parts(x, p);
      Base::qf[s] = p[0];
#pragma unroll
      for (int i = 1; i < kParts; ++i) qx[i - 1][s] = p[i];
    }
  }
  __device__ __forceinline__ void nothing() {
    float z[Base::NS][8] = {};
    Base::setup(z, false, 1.f);
  }
  // S^T accumulator of 16 key rows, the least part first.
  __device__ __forceinline__ f32x4 scores(const v8 (&k)[Base::NS]) const {
    f32x4 st = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = kParts - 1; i >= 0; --i)
#pragma unroll
      for (int s = 0; s < Base::NS; ++s) st = Mfma16<E>::run(k[s], i ? qx[i ? i - 1 : 0][s] : Base::qf[s], st);
    return st;
  }
  __device__ __forceinline__ void softmax(const float (&sc)[8], v8 (&p)[kParts]) { parts(Base::weights32(sc), p); }
  __device__ __forceinline__ void add(int t, v8 v, const v8 (&p)[kParts]) {
#pragma unroll
    for (int i = kParts - 1; i >= 0; --i) Base::o[t] = Mfma16<E>::run(v, p[i], Base::o[t]);
  }
};

// Whether a lane of the wave holds a NaN.
__device__ __forceinline__ bool any_nan(const float (&sc)[8]) {
  bool n = false;
#pragma unroll
  for (int e = 0; e < 8; ++e) n |= sc[e] != sc[e];
  return __ballot(n) != 0ull;
}
// Eight values, 0 for NaN.
template <typename V> __device__ __forceinline__ V values_or_zero(V v) {
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = v[e] == v[e] ? v[e] : 0;
  return v;
}

// One 16-row group's output, or its partial sums for the join of its ranges.
template <int HD, int FMT, typename T, typename E>
__device__ __forceinline__ void store_group(const PagedAttnParams& p, const MqaWave<HD, E>& w, long long g, int live,
                                            bool whole, int head, void* stage) {
  constexpr float unit = 1.f / PagedKey<FMT, E>::held;
  if (whole) {
    const float f = unit * w.finish(p.sink != nullptr, p.sink ? p.sink[head] : 0.f);
    store_rows<HD, T>(w.o, f, static_cast<T*>(p.out) + g * HD, live, stage);
    return;
  }
  const int n = lane_id() & 15;
  const long long gp = (long long)blockIdx.z * p.pool.N * p.nh + g;
  store_rows<HD, float>(w.o, unit, p.part_o + gp * HD, live, stage);
  if (lane_id() < 16 && n < live) {
    p.part_ml[2 * (gp + n)] = w.M;
    p.part_ml[2 * (gp + n) + 1] = w.L;
  }
}

// Up to 16 QW rows of a sequence and a range of 32-key steps, which the four waves take
// in turn. BIG: pages of at least 32 rows (one table entry a step). No load is behind a
// branch (a wait there would drain every load in flight): past the end the last
// step is read again.
// Workgroups a CU at least (as many as leave registers for a step in flight without spilling).
constexpr int token_min_blocks(int HD, int FMT, int QW, bool f32) {
  const int n = (QW == 1 ? 3 : 2) - (HD == 128 && FMT == PF_BF16 ? 1 : 0);
  return f32 && n > 1 ? n - 1 : n;
}
template <int HD, int FMT, int QW, bool BIG, typename T>
__global__ __launch_bounds__(256, token_min_blocks(HD, FMT, QW, __is_same(T, float))) void paged_token_kernel(PagedAttnParams p) {
  typedef typename Prod<T>::type E;
  typedef PagedKey<FMT, E> Key;
  using W = PagedWave<HD, T>;
  typedef typename W::v8 v8;
  constexpr int ROWB = FMT == PF_BF16 ? 2 * HD : HD;  // bytes of a key row
  constexpr int TPR = ROWB / 16;                      // lanes per key row
  constexpr int RPI = 64 / TPR;                       // key rows of a load
  constexpr int NLI = 32 / RPI;                       // loads of a step
  constexpr int NP = BIG ? 1 : NLI;                   // table entries of a lane
  __shared__ __attribute__((aligned(16))) E stage_all[4][32 * HD];
  __shared__ float ml[4][16][2];
  __shared__ float poison[4][32];
  const PagedPool& pl = p.pool;
  if (blockIdx.y == (unsigned)pl.S) return zero_ends<HD, T>(p);
  const PagedSeq sq = paged_seq(pl, blockIdx.y);
  const int nrow = computed_rows(p, sq);
  zero_rest<HD, T>(p, sq);
  const int wv = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int lane = lane_id(), q4 = lane >> 4, n = lane & 15;
  const int lrow = lane / TPR, lch = lane % TPR;
  const uint32_t cap = (uint32_t)pl.nrp << pl.log2page;
  const uint32_t lmask = (1u << pl.log2page) - 1;
  E* const stage = stage_all[wv];
  const TileOffsets<HD> to;

  const int r0 = blockIdx.x * 16 * QW;
  if (r0 >= nrow) return;
  const KeySpan sp = key_span(p, sq, r0 / p.nh, (min(r0 + 16 * QW, nrow) - 1) / p.nh);
  const KeySteps ks = key_steps(p, sp);
  const uint32_t total = ks.nb + ks.nw, per = range_len(p, total, kStepUnit);
  const uint32_t s0 = per * blockIdx.z, s1 = min(total, s0 + per);
  if (s0 >= total && blockIdx.z) return;
  const bool whole = total <= per;  // no other range: the output itself
  const int* const btab = pl.block_table + (size_t)sq.slot * pl.nbp;
  const int* const rtab = pl.ring_table + (size_t)sq.slot * pl.nrp;
  const uint32_t wr = sp.nw ? sp.wlo % cap - ks.woff : 0;  // ring row of the first window step

  W w[QW];
  int head[QW];
  if (s0 < s1) {
    const int nb = ks.nb, last = s1 - 1;
    const uint32_t bwidth = pl.nbp, rwidth = pl.nrp;
    struct Step {
      uint4 v[NLI];
      int code[NLI];
      int ok;  // bit i: the row of load i is a row of the pool
    };
    auto step_row = [&](int i) { return (uint32_t)(RPI * i + lrow); };
    auto ring_row = [&](uint32_t r) { return r >= cap ? r - cap : r; };
    auto load_page = [&](int st, int (&pg)[NP]) {
      st = min(st, last);
      const int d = st - nb;  // (a signed compare stays on the scalar unit)
      const bool blk = d < 0;
      const int* const tab = blk ? btab : rtab;
      const uint32_t f = blk ? 32 * st : wr + 32 * d, width = blk ? bwidth : rwidth;
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        uint32_t r = BIG ? f : f + step_row(i);
        if (!blk) r = ring_row(r);
        pg[i] = tab[min(r >> pl.log2page, width - 1)];
      }
    };
    auto load_step = [&](int st, const int (&pg)[NP], Step& s) {
      st = min(st, last);
      const int d = st - nb;
      const bool blk = d < 0;
      const uint32_t f = blk ? 32 * st : wr + 32 * d;
      if constexpr (BIG) {  // one page: a scalar address, the lane's offset in it and constants
        const int page = __builtin_amdgcn_readfirstlane(pg[0]);
        const bool ok = (unsigned)page < (unsigned)pl.P;
        const long long pr = ((long long)(ok ? page : 0) << pl.log2page) + ((blk ? f : ring_row(f)) & lmask);
        const char* const base = static_cast<const char*>(pl.rows) + pr * ROWB;
        const uint8_t* const sb = pl.scales + pr;
#pragma unroll
        for (int i = 0; i < NLI; ++i) {
          s.v[i] = *reinterpret_cast<const uint4*>(base + (lrow * ROWB + 16 * lch) + i * RPI * ROWB);
          if constexpr (FMT != PF_BF16) s.code[i] = sb[lrow + i * RPI];
        }
        s.ok = ok ? 0xff : 0;
      } else {
        s.ok = 0;
#pragma unroll
        for (int i = 0; i < NLI; ++i) {
          const bool ok = (unsigned)pg[i] < (unsigned)pl.P;
          uint32_t r = f + step_row(i);
          if (!blk) r = ring_row(r);
          const long long pr = ((long long)(ok ? pg[i] : 0) << pl.log2page) + (r & lmask);
          s.v[i] = *reinterpret_cast<const uint4*>(static_cast<const char*>(pl.rows) + pr * ROWB + 16 * lch);
          if constexpr (FMT != PF_BF16) s.code[i] = pl.scales[pr];
          s.ok |= (ok ? 1 : 0) << i;
        }
      }
    };
    // a step in flight, and the table entry of the one after it. The loads keep this
    // order everywhere: a wait counts the loads issued after the one it waits for.
    int pg[NP];
    Step sa;
    int st = s0 + wv;
    auto next = [&](int at) {
      __builtin_amdgcn_sched_barrier(0);
      load_step(at, pg, sa);
      __builtin_amdgcn_sched_barrier(0);
      load_page(at + 4, pg);
      __builtin_amdgcn_sched_barrier(0);
    };
    load_page(st, pg);
    next(st);

    // the queries, while the first steps' rows are in flight; this lane's row sees
    // block rows below vis, and window rows [lo, hi) counted from the first window step's
    uint32_t vis[QW], lo[QW], hi[QW];
#pragma unroll
    for (int u = 0; u < QW; ++u) {
      const int r = r0 + 16 * u + n;
      const bool live = r < nrow;
      const int rr = live ? r : nrow - 1;
      const int tok = rr / p.nh;
      head[u] = rr - tok * p.nh;
      w[u].query(static_cast<const T*>(p.q) + ((long long)sq.row0 * p.nh + rr) * HD, live, p.normalize_q != 0,
                 p.scale / Key::held);
      const uint32_t pos = sq.ctx + tok;
      const uint32_t f = pos + 1 > (uint32_t)p.win ? pos + 1 - p.win : 0;
      // (a padding row is never stored: it masks nothing)
      vis[u] = live ? visible_blocks(p, pos) : 0xffffffffu;
      lo[u] = live ? ks.woff + (f - sp.wlo) : 0;
      hi[u] = live ? ks.woff + (pos - sp.wlo) + 1 : 0xffffffffu;
    }

    bool any_bad = false;
    // a step's rows into the wave's LDS
    auto put = [&](int st, Step& s) {
      const int d = st - nb;
      const bool blk = d < 0;
      const uint32_t j0 = 32 * (blk ? st : d);  // block row, or window row, of the step's first
      // rows that no query of the workgroup sees, or that are none of the pool: zeros
      const uint32_t ua = blk ? 0 : ks.woff, ub = blk ? sp.nc : ks.woff + sp.nw;
      if (!(BIG && s.ok && j0 >= ua && j0 + 32 <= ub)) {
#pragma unroll
        for (int i = 0; i < NLI; ++i) {
          const uint32_t j = j0 + step_row(i);
          const bool ok = (s.ok >> i & 1) && j >= ua && j < ub;
          s.v[i] = ok ? s.v[i] : make_uint4(0, 0, 0, 0);
          if constexpr (FMT != PF_BF16) s.code[i] = ok ? s.code[i] : 127;
        }
      }
      bool bad[NLI], some = false;
#pragma unroll
      for (int i = 0; i < NLI; ++i) {
        if constexpr (FMT == PF_BF16) {
          const uint32_t x[4] = {s.v[i].x, s.v[i].y, s.v[i].z, s.v[i].w};
          bad[i] = false;
#pragma unroll
          for (int e = 0; e < 4; ++e) bad[i] |= (x[e] & 0x7fffu) > Key::top || (x[e] >> 16 & 0x7fffu) > Key::top;
        } else {
          bad[i] = s.code[i] > Key::top;
        }
        some |= bad[i];
      }
      wave_lds_sync();  // the previous step's reads of the stage are done
      any_bad = __ballot(some) != 0ull;
      if (any_bad) {  // (rare) such a row as zeros, and NaN beside it
#pragma unroll
        for (int i = 0; i < NLI; ++i) {
          const unsigned long long g = __ballot(bad[i]) >> (lane & ~(TPR - 1)) & ((1ull << TPR) - 1);
          s.v[i] = g ? make_uint4(0, 0, 0, 0) : s.v[i];
          if constexpr (FMT != PF_BF16) s.code[i] = g ? 127 : s.code[i];
          if (lch == 0) poison[wv][step_row(i)] = g ? __uint_as_float(0x7fc00000u) : 0.f;
        }
      }
#pragma unroll
      for (int i = 0; i < NLI; ++i) {
        const uint32_t row = step_row(i);
        E* const dst = stage + row * HD;
        const int sw = tile_swz<HD>(row & 15);
        if constexpr (FMT == PF_BF16) {
          *reinterpret_cast<uint4*>(dst + 8 * (lch ^ sw)) = bf16_pairs<E>(s.v[i]);
        } else {
          const float sc = Key::held * __uint_as_float((uint32_t)s.code[i] << 23);
          const uint2 a = dequant4<FMT, E>(s.v[i].x, sc), c = dequant4<FMT, E>(s.v[i].y, sc);
          const uint2 d = dequant4<FMT, E>(s.v[i].z, sc), e = dequant4<FMT, E>(s.v[i].w, sc);
          *reinterpret_cast<uint4*>(dst + 8 * ((2 * lch) ^ sw)) = make_uint4(a.x, a.y, c.x, c.y);
          *reinterpret_cast<uint4*>(dst + 8 * ((2 * lch + 1) ^ sw)) = make_uint4(d.x, d.y, e.x, e.y);
        }
      }
      wave_lds_sync();  // staged rows visible to the whole wave
    };
    auto use = [&](int st) {
      const int d = st - nb;
      const bool blk = d < 0;
      const uint32_t j0 = 32 * (blk ? st : d);
      f32x4 ra[QW], rb[QW];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        v8 kf[W::NS];
#pragma unroll
        for (int e = 0; e < W::NS; ++e) kf[e] = *reinterpret_cast<const v8*>(stage + 16 * HD * h + to.key(e));
#pragma unroll
        for (int u = 0; u < QW; ++u) {
          if (h == 0) ra[u] = w[u].scores(kf);
          else rb[u] = w[u].scores(kf);
        }
      }
      v8 pb8[QW][W::kParts];
      bool holes = false;  // a NaN that some row does not see
#pragma unroll
      for (int u = 0; u < QW; ++u) {
        float sc[8] = {ra[u][0], ra[u][1], ra[u][2], ra[u][3], rb[u][0], rb[u][1], rb[u][2], rb[u][3]};
        if (any_bad) {
#pragma unroll
          for (int e = 0; e < 8; ++e) sc[e] += poison[wv][4 * q4 + (e < 4 ? e : 12 + e)];
        }
        const uint32_t la = blk ? 0 : lo[u], lb = blk ? vis[u] : hi[u];
        if (__ballot(j0 < la || j0 + 32 > lb)) {
          if constexpr (FMT == PF_E4M3) holes |= any_nan(sc);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const uint32_t j = j0 + 4 * q4 + (e < 4 ? e : 12 + e);
            sc[e] = j >= la && j < lb ? sc[e] : -INFINITY;
          }
        }
        w[u].softmax(sc, pb8[u]);
      }
#pragma unroll
      for (int t0 = 0; t0 < W::NT; t0 += 4) {
        v8 va[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) va[t] = W::vt_frag(stage, to, t0 + t);
        if (FMT == PF_E4M3 && holes) {
#pragma unroll
          for (int t = 0; t < 4; ++t) va[t] = values_or_zero(va[t]);
        }
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int u = 0; u < QW; ++u) w[u].add(t0 + t, va[t], pb8[u]);
      }
    };

    // a step's registers are free once it is in LDS: the next one's load goes out before
    // the products
    for (; st <= last; st += 4) {
      put(st, sa);
      next(st + 4);
      use(st);
    }
  } else {
#pragma unroll
    for (int u = 0; u < QW; ++u) {
      w[u].nothing();
      head[u] = 0;
    }
  }

  // the four waves' sums, a 16-row group at a time
#pragma unroll
  for (int u = 0; u < QW; ++u) {
    w[u].finalize();
    float* const ob = reinterpret_cast<float*>(stage_all) + wv * 16 * HD;
    __syncthreads();
#pragma unroll
    for (int t = 0; t < W::NT; ++t) *reinterpret_cast<f32x4*>(ob + (t * 64 + lane) * 4) = w[u].o[t];
    if (q4 == 0) {
      ml[wv][n][0] = w[u].M;
      ml[wv][n][1] = w[u].L;
    }
    __syncthreads();
    if (wv == u % 4) {
      float M = ml[0][n][0];
#pragma unroll
      for (int g = 1; g < 4; ++g) M = fmaxf(M, ml[g][n][0]);
      w[u].M = M;
      w[u].L = 0.f;
#pragma unroll
      for (int t = 0; t < W::NT; ++t) w[u].o[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const float f = fast_exp2(ml[g][n][0] - M);
        w[u].L += f * ml[g][n][1];
        const float* og = reinterpret_cast<const float*>(stage_all) + g * 16 * HD;
#pragma unroll
        for (int t = 0; t < W::NT; ++t) w[u].o[t] += f * *reinterpret_cast<const f32x4*>(og + (t * 64 + lane) * 4);
      }
    }
    __syncthreads();  // the sums are read before their place is staged over
    const int r = r0 + 16 * u;
    if (wv == u % 4 && r < nrow)
      store_group<HD, FMT, T>(p, w[u], (long long)sq.row0 * p.nh + r, min(16, nrow - r), whole, head[u], ob);
  }
}

// The keys below k1 that a token of a tile sees: [0, vis) and [lo, hi). All grow with the
// token.
struct RowKeys {
  uint32_t vis, lo, hi;
};
__device__ __forceinline__ RowKeys row_keys(const PagedAttnParams& p, const PagedSeq& sq, const KeySpan& sp,
                                            int tok, uint32_t k1) {
  const uint32_t pos = sq.ctx + tok, f = pos + 1 > (uint32_t)p.win ? pos + 1 - p.win : 0;
  RowKeys k;
  k.vis = min(visible_blocks(p, pos), k1);
  k.lo = sp.nw ? min(sp.nc + (f - sp.wlo), k1) : 0;
  k.hi = sp.nw ? min(sp.nc + (pos - sp.wlo) + 1, k1) : 0;
  return k;
}

// RG groups of 16 rows of a sequence, QW of them a wave, and a range of keys. Two
// workgroups of 8 waves a CU (128 registers): 132 us where one took 156, for 8 chunks of up
// to 2048 tokens behind 128K. Two groups a wave on half as many waves, with the next
// step's scores between this one's softmax, halve the LDS reads and nearly the vector
// instructions, but two waves a SIMD wait for LDS: 122 us there, and 76 where this
// takes 71 for 16 chunks without a context, 167 where it takes 143 on bf16 rows (125 us
// for this one then).
template <int HD, int FMT, int RG, int QW, typename T>
__global__ __launch_bounds__(64 * (RG / QW), RG == 8 && !__is_same(T, float) ? 4 : 2) void paged_attn_kernel(PagedAttnParams p) {
  typedef typename Prod<T>::type E;
  typedef PagedKey<FMT, E> Key;
  using W = PagedWave<HD, T>;
  typedef typename W::v8 v8;
  constexpr int NWV = RG / QW, NTH = 64 * NWV;
  constexpr int ROWS = 16 * RG;
  constexpr int EPL = FMT == PF_BF16 ? 8 : 16;  // row elements of a lane's 16 bytes
  constexpr int TPR = HD / EPL;                 // lanes per key row
  constexpr int RSTEP = NTH / TPR;              // key rows of a load instruction of the workgroup
  constexpr int NLD = KC / RSTEP;
  static_assert(NLD >= 1 && KC % RSTEP == 0 && RSTEP % 16 == 0, "tile loads");
  __shared__ __attribute__((aligned(16))) E tile[2][KC * HD];
  __shared__ __attribute__((aligned(16))) float poison[2][KC];
  __shared__ int any_bad;  // some row so far is not finite

  const int tid = threadIdx.x;
  const PagedPool& pl = p.pool;
  if (blockIdx.y == (unsigned)pl.S) return zero_ends<HD, T>(p);
  const PagedSeq sq = paged_seq(pl, blockIdx.y);
  const int nrow = computed_rows(p, sq);
  zero_rest<HD, T>(p, sq);
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63, q4 = lane >> 4, n = lane & 15;
  const uint32_t ring_cap = (uint32_t)pl.nrp << pl.log2page;
  const int lmask = (1 << pl.log2page) - 1;
  const int* const btab = pl.block_table + (size_t)sq.slot * pl.nbp;
  const int* const rtab = pl.ring_table + (size_t)sq.slot * pl.nrp;
  const TileOffsets<HD> to;

  const int r0 = blockIdx.x * ROWS;
  if (r0 >= nrow) return;
  const int ta = r0 / p.nh, tb = (min(r0 + ROWS, nrow) - 1) / p.nh;
  const KeySpan sp = key_span(p, sq, ta, tb);
  const uint32_t total = sp.nc + sp.nw;
  const uint32_t per = range_len(p, total, KC);
  const uint32_t k0 = per * blockIdx.z;
  if (k0 >= total && blockIdx.z) return;
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
      E* dst = tile[buf] + row * HD;
      const int sw = tile_swz<HD>(row & 15);
      if constexpr (FMT == PF_BF16) {
        const uint32_t w[4] = {pf[i].x, pf[i].y, pf[i].z, pf[i].w};
        bool bad = false;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          bad |= (w[e] & 0x7fffu) > Key::top || (w[e] >> 16 & 0x7fffu) > Key::top;
        // the whole row is bad where one of its lanes is
        const unsigned long long g = __ballot(bad) >> (lane & ~(TPR - 1)) & ((1ull << TPR) - 1);
        if (g) pf[i] = make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(dst + 8 * (lch ^ sw)) = bf16_pairs<E>(pf[i]);
        if (lch == 0) poison[buf][row] = g ? __uint_as_float(0x7fc00000u) : 0.f;
        bad_any |= g != 0;
      } else {
        const bool bad = code[i] > Key::top;
        const float sc = Key::held * row_scale(bad ? 127 : code[i]);
        const uint32_t keep = bad ? 0u : 0xffffffffu;
        const uint2 a = dequant4<FMT, E>(pf[i].x & keep, sc), b = dequant4<FMT, E>(pf[i].y & keep, sc);
        const uint2 c = dequant4<FMT, E>(pf[i].z & keep, sc), d = dequant4<FMT, E>(pf[i].w & keep, sc);
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
  RowKeys first[QW], final_[QW];
  bool seen[QW];
  int head[QW];
#pragma unroll
  for (int u = 0; u < QW; ++u) {
    const int r = r0 + 16 * (QW * wv + u) + n;
    const bool live = r < nrow;
    const int rr = live ? r : nrow - 1;
    const int tok = rr / p.nh;
    head[u] = rr - tok * p.nh;
    const T* qrow = static_cast<const T*>(p.q) + ((long long)sq.row0 * p.nh + rr) * HD;
    w[u].query(qrow, live, p.normalize_q != 0, p.scale / Key::held);
    const RowKeys k = row_keys(p, sq, sp, tok, k1);
    // (a padding row is never stored: it masks nothing)
    vis[u] = live ? k.vis : k1;
    lo[u] = k.lo;
    hi[u] = k.hi;
    // the group's first and last rows bound what its rows see
    const int g0 = r0 + 16 * (QW * wv + u), g1 = min(g0 + 15, nrow - 1);
    seen[u] = g0 < nrow;
    first[u] = row_keys(p, sq, sp, min(g0, nrow - 1) / p.nh, k1);
    final_[u] = row_keys(p, sq, sp, g1 / p.nh, k1);
  }

  // values read this many 16-column tiles ahead of their products: four, where 128 registers
  // hold them beside the e4m3 rows' look for NaN (that spills at 128 columns: 156 us for 116; bf16
  // rows 138 for 142, 64 columns 78 for 81)
  constexpr int kPv = RG == 8 && HD == 128 && FMT == PF_E4M3 ? 1 : 4;
  // 32 keys (tile rows from `rows`, key index j0 of the first)
  auto keys32 = [&](const E* rows, const float* pz, bool bad, uint32_t j0) {
    f32x4 sa[QW], sb[QW];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      v8 kf[W::NS];
#pragma unroll
      for (int s = 0; s < W::NS; ++s) kf[s] = *reinterpret_cast<const v8*>(rows + 16 * HD * h + to.key(s));
#pragma unroll
      for (int u = 0; u < QW; ++u) {
        if (h == 0) sa[u] = w[u].scores(kf);
        else sb[u] = w[u].scores(kf);
      }
    }
    v8 pb[QW][W::kParts];
    bool holes = false;  // a NaN that some row does not see
#pragma unroll
    for (int u = 0; u < QW; ++u) {
      float sc[8] = {sa[u][0], sa[u][1], sa[u][2], sa[u][3], sb[u][0], sb[u][1], sb[u][2], sb[u][3]};
      if (bad) {
#pragma unroll
        for (int e = 0; e < 8; ++e) sc[e] += pz[4 * q4 + (e < 4 ? e : 12 + e)];
      }
      if (!(j0 + 32 <= first[u].vis || (j0 >= final_[u].lo && j0 + 32 <= first[u].hi))) {
        if constexpr (FMT == PF_E4M3) holes |= any_nan(sc);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t j = j0 + 4 * q4 + (e < 4 ? e : 12 + e);
          const bool ok = (j < vis[u]) | (j - lo[u] < hi[u] - lo[u]);
          sc[e] = ok ? sc[e] : -INFINITY;
        }
      }
      w[u].softmax(sc, pb[u]);
    }
    // a wave at its products goes before those at their softmax (8 short-context chunks
    // 82.6 -> 76.8 us, long ones 126 -> 122)
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int t0 = 0; t0 < W::NT; t0 += kPv) {
      v8 va[kPv];
#pragma unroll
      for (int t = 0; t < kPv; ++t) va[t] = W::vt_frag(rows, to, t0 + t);
      if (FMT == PF_E4M3 && holes) {
#pragma unroll
        for (int t = 0; t < kPv; ++t) va[t] = values_or_zero(va[t]);
      }
#pragma unroll
      for (int t = 0; t < kPv; ++t)
#pragma unroll
        for (int u = 0; u < QW; ++u) w[u].add(t0 + t, va[t], pb[u]);
    }
    __builtin_amdgcn_s_setprio(0);
  };

  if (tid == 0) any_bad = 0;
  __syncthreads();
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
    for (int s = 0; s < KC / 32; ++s) {
      const int at = 32 * s;
      // (a step that none of the wave's rows sees is passed over)
      bool some = false;
#pragma unroll
      for (int u = 0; u < QW; ++u)
        some |= seen[u] && (j0 + at < final_[u].vis || (j0 + at < final_[u].hi && j0 + at + 32 > first[u].lo));
      if (some) keys32(tile[buf] + at * HD, poison[buf] + at, bad, j0 + at);
    }
    if (t + 1 < nt) store_rows_lds(buf ^ 1);
    __syncthreads();
  }

  char* const stage = reinterpret_cast<char*>(&tile[0][0]) + wv * 16 * HD * 4;
  static_assert(NWV * 16 * HD * 4 <= (int)sizeof(tile), "the staged outputs fit in the tiles");
#pragma unroll
  for (int u = 0; u < QW; ++u) {
    const int r = r0 + 16 * (QW * wv + u);
    if (u > 0) wave_lds_sync();
    if (r >= nrow) break;
    w[u].finalize();
    store_group<HD, FMT, T>(p, w[u], (long long)sq.row0 * p.nh + r, min(16, nrow - r), whole, head[u], stage);
  }
}

// Joins the ranges of rows that have more than one: HD / 8 lanes a row.
template <int HD, typename T>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedAttnParams p) {
  constexpr int LPR = HD / 8;
  const PagedSeq sq = paged_seq(p.pool, blockIdx.y);
  const int nrow = computed_rows(p, sq);
  const int ch = 8 * (threadIdx.x % LPR);
  for (int r = blockIdx.x * (256 / LPR) + threadIdx.x / LPR; r < nrow; r += gridDim.x * (256 / LPR)) {
    const int r0 = r / p.rows * p.rows;
    const KeySpan sp = key_span(p, sq, r0 / p.nh, (min(r0 + p.rows, nrow) - 1) / p.nh);
    const KeySteps ks = key_steps(p, sp);
    const bool steps = p.rows <= kPagedTokenRows;
    const uint32_t total = steps ? ks.nb + ks.nw : sp.nc + sp.nw, per = range_len(p, total, steps ? kStepUnit : KC);
    if (total <= per) continue;
    const int ns = (int)((total + per - 1) / per);
    const long long g = (long long)sq.row0 * p.nh + r, stride = (long long)p.pool.N * p.nh;
    // eight ranges' sums in flight together (past the last one it again, with weight 0)
    float M = kMFloor, L = 0.f, o[8] = {};
    for (int s0 = 0; s0 < ns; s0 += 8) {
      float2 ml[8];
      float v[8][8];
#pragma unroll
      for (int s = 0; s < 8; ++s) {
        const long long at = g + min(s0 + s, ns - 1) * stride;
        ml[s] = *reinterpret_cast<const float2*>(p.part_ml + 2 * at);
        Load8<float>::run(p.part_o + at * HD + ch, v[s]);
      }
      float mx = M;
#pragma unroll
      for (int s = 0; s < 8; ++s) mx = fmaxf(mx, ml[s].x);
      const float f0 = fast_exp2(M - mx);
      L *= f0;
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] *= f0;
      M = mx;
#pragma unroll
      for (int s = 0; s < 8; ++s) {
        if (s0 + s >= ns) break;
        const float f = fast_exp2(ml[s].x - M);
        L = fmaf(f, ml[s].y, L);
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = fmaf(f, v[s][i], o[i]);
      }
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

template <int HD, int FMT, typename T>
void attn_launch(const PagedAttnParams& p, hipStream_t s) {
  const long long nrow = (long long)p.max_len * p.nh;
  const dim3 grid((unsigned)((nrow + p.rows - 1) / p.rows), (unsigned)(p.pool.S + (p.zero_tail ? 1 : 0)),
                  (unsigned)p.nsplit);
  const bool big = p.pool.log2page >= 5;
#define KCH_PT(QW, BIG) hipLaunchKernelGGL((paged_token_kernel<HD, FMT, QW, BIG, T>), grid, dim3(256), 0, s, p)
#define KCH_PA(RG, QW) hipLaunchKernelGGL((paged_attn_kernel<HD, FMT, RG, QW, T>), grid, dim3(64 * RG / QW), 0, s, p)
  if (p.rows == 16 && big) KCH_PT(1, true);
  else if (p.rows == 16) KCH_PT(1, false);
  else if (p.rows == 32 && big) KCH_PT(2, true);
  else if (p.rows == 32) KCH_PT(2, false);
  else if (p.rows == 64) KCH_PA(4, 1);
  else KCH_PA(8, 1);
#undef KCH_PT
#undef KCH_PA
  if (p.nsplit > 1) {
    constexpr int RPB = 256 / (HD / 8);
    const dim3 jg((unsigned)((nrow + RPB - 1) / RPB), (unsigned)p.pool.S);
    hipLaunchKernelGGL((paged_join_kernel<HD, T>), jg, dim3(256), 0, s, p);
  }
}

template <int HD, int FMT>
void attn_launch_t(const PagedAttnParams& p, int dtype, hipStream_t s) {
  if (dtype == DT_BF16) attn_launch<HD, FMT, bf16_t>(p, s);
  else if (dtype == DT_F16) attn_launch<HD, FMT, _Float16>(p, s);
  else attn_launch<HD, FMT, float>(p, s);
}

}  // namespace

PagedAttnPlan paged_attn_plan(int S, int N, int nh, int c, int m2, int win, int max_len, int max_ctx) {
  PagedAttnPlan pl;
  const long long nrow = (long long)max_len * nh;
  pl.rows = nrow <= 16 ? 16 : nrow <= 32 ? 32 : nrow <= 64 ? 64 : 128;
  const bool steps = pl.rows <= kPagedTokenRows;
  const long long tiles = (nrow + pl.rows - 1) / pl.rows * S;
  const long long keys = ((long long)max_ctx + max_len) / m2 + win + (pl.rows + nh - 1) / nh;
  // units of a range: 32-key steps, or keys, a tile at a time
  const long long unit = steps ? kStepUnit : KC, total = steps ? keys / 32 + 3 : keys;
  // workgroups for each of 256 CUs, and no range too short to be worth its join
  const long long want = (pl.rows == 16 ? 768 : 512) / (tiles > 0 ? tiles : 1), least = steps ? 2 * kStepUnit : 4 * KC;
  long long per = want > 1 ? (total + want - 1) / want : total;
  per = ((per < least ? least : per) + unit - 1) / unit * unit;
  pl.nsplit = (int)((total + per - 1) / per);
  if (pl.nsplit < 1) pl.nsplit = 1;
  pl.range = (int)(per < (1ll << 30) ? per : (1ll << 30));
  pl.bytes = pl.nsplit > 1 ? (size_t)pl.nsplit * N * nh * (c + 2) * sizeof(float) : 0;
  return pl;
}

hipError_t paged_attn_dispatch(const PagedAttnParams& p, int format, int dtype, hipStream_t s) {
  if (p.pool.c == 128) {
    if (format == PF_BF16) attn_launch_t<128, PF_BF16>(p, dtype, s);
    else if (format == PF_E4M3) attn_launch_t<128, PF_E4M3>(p, dtype, s);
    else attn_launch_t<128, PF_INT8>(p, dtype, s);
  } else {
    if (format == PF_BF16) attn_launch_t<64, PF_BF16>(p, dtype, s);
    else if (format == PF_E4M3) attn_launch_t<64, PF_E4M3>(p, dtype, s);
    else attn_launch_t<64, PF_INT8>(p, dtype, s);
  }
  return hipGetLastError();
}

}  // namespace kch
