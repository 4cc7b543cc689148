// The paged HCA cache: a chunk's tokens quantised as they are written, and rows
// read back (gfx950).
//
// paged_append_kernel. Token p = ctx + i of a sequence, block b = p / m2, j = p %
// m2, per channel z = Z + B_pos[j]:
//   window row   C_p / max(||C_p||, 1e-12) at ring row p % (ring's rows)
//   block row    r / max(||r||, 1e-12), r = sum_j softmax_j(z) C_j, on b's end
// both quantised row by row (paged.h). The softmax runs over the block's tokens
// in one pass with a running maximum, sum and weighted sum per channel (fp32);
// what a chunk leaves of a block, these three numbers, is all that the next call
// needs: 12 c bytes a sequence, where keeping the tokens themselves takes
// 4 m2 c (64 KB at m2 = 128, c = 128) and a second pass at the block's end.
// (csa_compress_kv, /root/reference/ops_csa.py:198-234; the accumulation per token,
// /root/reference/ops_decoding_cache.py:1200-1267.)
//
// A workgroup of 8 waves takes one block (of one wave where blocks or chunks have few
// tokens): its rows 16 bytes a lane (HD / 8 lanes a row), so a row's norm and maximum
// are reductions over neighbouring lanes, C and Z are read once for both outputs,
// and a block of 128 tokens is in flight at once. The workgroup of a sequence's first
// block also takes the block that the chunk leaves open, because it alone may read
// the sequence's old sums: no other workgroup writes them. Both are parts of blocks:
// half of the waves take each at the same time (one after the other, they were
// the kernel's time: 16 chunks of up to 2048 tokens 16.4 us, now 13.2 for 12.7 MB, 1 TB/s;
// 2.5 us at the rate of a large copy). Bound by what one workgroup does in a row: the
// step's arrays, the block's rows, its sums over the waves, the quantised row.

#include <cfloat>

#include "paged.h"

namespace kch {

namespace {

// Reductions over groups of 8 or 16 neighbouring lanes on the vector unit's own lane
// moves (a shuffle through LDS takes some hundred cycles a step): pairs, quads, then the
// mirrored half rows and rows.
template <int CTRL> __device__ __forceinline__ float dpp_move(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, false));
}
template <int W, typename F> __device__ __forceinline__ float group_reduce(float v, F f) {
  static_assert(W == 8 || W == 16, "lanes of a row");
  v = f(v, dpp_move<0xb1>(v));    // quad_perm 1 0 3 2
  v = f(v, dpp_move<0x4e>(v));    // quad_perm 2 3 0 1
  v = f(v, dpp_move<0x141>(v));   // row_half_mirror
  if constexpr (W == 16) v = f(v, dpp_move<0x140>(v));  // row_mirror
  return v;
}
template <int W> __device__ __forceinline__ float group_sum(float v) {
  return group_reduce<W>(v, [](float a, float b) { return a + b; });
}
template <int W> __device__ __forceinline__ float group_amax(float v) {
  return group_reduce<W>(v, [](float a, float b) { return amax_nan(a, b); });
}

// e^(a - b) of softmax references: a = -inf (nothing summed yet) gives 0, also
// where b is -inf. (A reference of the type's lowest value is one like any other: a block
// masked with it weighs its tokens alike.)
__device__ __forceinline__ float ref_exp(float a, float b) { return exp_hw(a - fmaxf(b, -FLT_MAX)); }

// One softmax state (max, sum, weighted sum) joined into another.
struct Sums {
  float m, l, a;
  __device__ __forceinline__ void join(float m2, float l2, float a2) {
    const float mn = fmaxf(m, m2), f = ref_exp(m, mn), g = ref_exp(m2, mn);
    l = l * f + l2 * g;
    a = a * f + a2 * g;
    m = mn;
  }
};

template <int HD, int FMT, int NWV, typename T>
__global__ __launch_bounds__(64 * NWV) void paged_append_kernel(PagedAppendParams p) {
  constexpr int LPR = HD / 8;        // lanes per row
  constexpr int RPW = 64 / LPR;      // rows of a wave at a time
  constexpr int BR = NWV == 1 ? 4 : 2;  // rows of a lane whose loads are in flight together
  typedef typename PagedFmt<FMT>::elem elem;
  __shared__ float red[NWV * RPW][3][HD];
  const PagedSeq sq = paged_seq(p.pool, blockIdx.y);
  if (sq.len == 0) return;
  const int wv = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int lane = lane_id(), sub = lane / LPR, ch = 8 * (lane % LPR);
  const uint32_t m2 = p.m2, end = sq.ctx + sq.len;
  const uint32_t b0 = sq.ctx / m2, bl = (end - 1) / m2;  // blocks touched
  const bool open = end != (bl + 1) * m2;
  const uint32_t cap = (uint32_t)p.pool.nrp << p.pool.log2page;
  float* const state = p.state + (size_t)sq.slot * 3 * HD;
  elem* const rows = static_cast<elem*>(p.pool.rows);

  // block b on the waves w0 .. w0 + nw - 1 (every wave of the workgroup is in such a call)
  auto block = [&](uint32_t b, int w0, int nw) {
    const int step = nw * RPW;                        // rows of these waves at a time, and sums of a channel
    const int parts = NWV == 1 ? step : 64 * nw / HD;  // of them the last wave joins
    const uint32_t lo = max(b * m2, sq.ctx), hi = min((b + 1) * m2, end);
    const uint32_t rlo = cap > 0 ? lo % cap : 0;  // ring row of the first token
    // what the end needs of memory, asked for at the start: the sums carried in (lane's
    // channels CPL lane ..), and the block's own row
    constexpr int CPL = HD / 64;
    const bool carried = b == b0 && sq.ctx != b0 * m2, ends = (b + 1) * m2 <= end;
    Sums s[CPL];
#pragma unroll
    for (int k = 0; k < CPL; ++k) {
      const int c = CPL * lane + k;
      s[k] = carried ? Sums{state[c], state[HD + c], state[2 * HD + c]} : Sums{-INFINITY, 0.f, 0.f};
    }
    const long long pr = ends ? pool_row(p.pool, p.pool.block_table, p.pool.nbp, sq.slot, b) : -1;
    float m[8], l[8], a[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      m[i] = -INFINITY;
      l[i] = a[i] = 0.f;
    }
    for (uint32_t r0 = lo; r0 < hi; r0 += step * BR) {
      float c8[BR][8], z8[BR][8], b8[BR][8];
      long long at[BR];  // pool row of the token's window row, or -1
#pragma unroll
      for (int u = 0; u < BR; ++u) {
        const uint32_t pos = r0 + u * step + (wv - w0) * RPW + sub;
        at[u] = -1;
        if (pos < hi) {
          const long long row = sq.row0 + (int)(pos - sq.ctx);
          Load8<T>::run(static_cast<const T*>(p.C) + row * p.ldc + ch, c8[u]);
          Load8<T>::run(static_cast<const T*>(p.Z) + row * p.ldz + ch, z8[u]);
          Load8<float>::run(p.B_pos + (size_t)(pos - b * m2) * HD + ch, b8[u]);
          uint32_t r = rlo + (pos - lo);
          if (r >= cap) r = r - cap < cap || cap == 0 ? r - cap : r % cap;
          // (a later token of the chunk may take its place)
          if (cap > 0 && end - pos <= cap) at[u] = pool_row(p.pool, p.pool.ring_table, p.pool.nrp, sq.slot, r);
        }
      }
#pragma unroll
      for (int u = 0; u < BR; ++u) {
        const uint32_t pos = r0 + u * step + (wv - w0) * RPW + sub;
        const bool live = pos < hi;
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          c8[u][i] = live ? c8[u][i] : 0.f;
          z8[u][i] = live ? z8[u][i] + b8[u][i] : -INFINITY;
          ss += c8[u][i] * c8[u][i];
        }
        if (cap == 0 || r0 + u * step >= hi) continue;  // (uniform)
        const float inv = p.normalize ? l2_inv(group_sum<LPR>(ss)) : 1.f;
        float x[8], mx = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[i] = c8[u][i] * inv;
          mx = amax_nan(mx, x[i]);
        }
        if constexpr (FMT == PF_BF16) {
          if (not_finite(group_amax<LPR>(mx)))
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(0x7fc00000u);
          if (at[u] >= 0) *reinterpret_cast<bf16x8*>(rows + at[u] * HD + ch) = to_bf16x8(x);
        } else {
          const int code = row_scale_code<FMT>(group_amax<LPR>(mx));
          if (at[u] >= 0) {
            *reinterpret_cast<uint2*>(rows + at[u] * HD + ch) =
                make_uint2(quant4<FMT>(x[0], x[1], x[2], x[3], code), quant4<FMT>(x[4], x[5], x[6], x[7], code));
            if (ch == 0) p.pool.scales[at[u]] = (uint8_t)code;
          }
        }
      }
      // one reference for the batch, so that a channel rescales once for it
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float mn = m[i];
#pragma unroll
        for (int u = 0; u < BR; ++u) mn = fmaxf(mn, z8[u][i]);
        const float f = ref_exp(m[i], mn);
        l[i] *= f;
        a[i] *= f;
        m[i] = mn;
      }
#pragma unroll
      for (int u = 0; u < BR; ++u) {
        if (r0 + u * step >= hi) continue;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float e = ref_exp(z8[u][i], m[i]);
          l[i] += e;
          // a masked token's value does not enter, whatever it is
          a[i] = e != 0.f ? fmaf(e, c8[u][i], a[i]) : a[i];
        }
      }
    }
    // the sums of all row slots that had a token, `parts` at a time, then one wave
    const int slots = (int)min((uint32_t)step, hi - lo), e0 = w0 * RPW;
    const int slot = wv * RPW + sub;
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
      *reinterpret_cast<float4*>(&red[slot][0][ch + i]) = make_float4(m[i], m[i + 1], m[i + 2], m[i + 3]);
      *reinterpret_cast<float4*>(&red[slot][1][ch + i]) = make_float4(l[i], l[i + 1], l[i + 2], l[i + 3]);
      *reinterpret_cast<float4*>(&red[slot][2][ch + i]) = make_float4(a[i], a[i + 1], a[i + 2], a[i + 3]);
    }
    __syncthreads();
    if constexpr (NWV > 1) {
      const int t = threadIdx.x - 64 * w0, c = t % HD, part = t / HD;
      Sums t0{-INFINITY, 0.f, 0.f};
      for (int e = part; e < slots; e += parts) t0.join(red[e0 + e][0][c], red[e0 + e][1][c], red[e0 + e][2][c]);
      // (entry `part` is this thread's own)
      red[e0 + part][0][c] = t0.m;
      red[e0 + part][1][c] = t0.l;
      red[e0 + part][2][c] = t0.a;
      __syncthreads();
    }
    if (wv == w0) {
      float x[CPL], ss = 0.f, mx = 0.f;
      for (int e = e0; e < e0 + min(parts, slots); ++e)
#pragma unroll
        for (int k = 0; k < CPL; ++k) {
          const int c = CPL * lane + k;
          s[k].join(red[e][0][c], red[e][1][c], red[e][2][c]);
        }
      if (ends) {
#pragma unroll
        for (int k = 0; k < CPL; ++k) {
          x[k] = s[k].l == 0.f ? 0.f : s[k].a / s[k].l;  // a channel without a weight: 0
          ss += x[k] * x[k];
        }
        const float inv = p.normalize ? l2_inv(wave_sum(ss)) : 1.f;
#pragma unroll
        for (int k = 0; k < CPL; ++k) {
          x[k] *= inv;
          mx = amax_nan(mx, x[k]);
        }
#pragma unroll
        for (int k = 32; k >= 1; k >>= 1) mx = amax_nan(mx, __shfl_xor(mx, k));
        if (pr >= 0) {
          elem* dst = rows + pr * HD + CPL * lane;
          if constexpr (FMT == PF_BF16) {
#pragma unroll
            for (int k = 0; k < CPL; ++k) dst[k] = (bf16_t)(not_finite(mx) ? __uint_as_float(0x7fc00000u) : x[k]);
          } else {
            const int code = row_scale_code<FMT>(mx);
            const uint32_t w = quant4<FMT>(x[0], CPL > 1 ? x[CPL - 1] : 0.f, 0.f, 0.f, code);
            if constexpr (CPL == 2) *reinterpret_cast<uint16_t*>(dst) = (uint16_t)w;
            else *dst = (uint8_t)w;
            if (lane == 0) p.pool.scales[pr] = (uint8_t)code;
          }
        }
      } else {
#pragma unroll
        for (int k = 0; k < CPL; ++k) {
          const int c = CPL * lane + k;
          state[c] = s[k].m;
          state[HD + c] = s[k].l;
          state[2 * HD + c] = s[k].a;
        }
      }
    }
    __syncthreads();  // red is free again
  };

  // the open block is the first workgroup's, which reads the old sums
  const bool two = blockIdx.x == 0 && open && bl > b0;
  const uint32_t last = open && bl > b0 ? bl - 1 : bl;
  uint32_t b = b0 + blockIdx.x;
  if (two) {
    if constexpr (NWV > 1) {
      block(wv < NWV / 2 ? b0 : bl, wv < NWV / 2 ? 0 : NWV / 2, NWV / 2);
    } else {
      block(b0, 0, 1);
      block(bl, 0, 1);
    }
    b += gridDim.x;
  }
  for (; b <= last; b += gridDim.x) block(b, 0, NWV);
}

template <int HD, int FMT, int NWV>
void append_launch_w(const PagedAppendParams& p, int dtype, hipStream_t s) {
  const dim3 grid((unsigned)((p.max_len + p.m2 - 2) / p.m2 + 1), (unsigned)p.pool.S), block(64 * NWV);
  if (dtype == DT_BF16) hipLaunchKernelGGL((paged_append_kernel<HD, FMT, NWV, bf16_t>), grid, block, 0, s, p);
  else if (dtype == DT_F16) hipLaunchKernelGGL((paged_append_kernel<HD, FMT, NWV, _Float16>), grid, block, 0, s, p);
  else hipLaunchKernelGGL((paged_append_kernel<HD, FMT, NWV, float>), grid, block, 0, s, p);
}
template <int HD, int FMT>
void append_launch(const PagedAppendParams& p, int dtype, hipStream_t s) {
  // tokens of a block in this call; a wave takes 4 (8) of 128 (64) channels at a time.
  // Measured (us with 1 / 8 / 16 waves, 128 channels, bf16 into e4m3): few blocks, chunks of 1, 8,
  // 16, 32, 64, 96, 128 tokens of 4 sequences 3.7 / 3.9 / 4.9, 4.6 / 4.4 / 5.5, 6.0 / 4.6 / 5.7, 9.1 / 5.2 /
  // 6.1, 15.8 / 6.2 / 6.9, 22.2 / 7.6 / 8.0, 29.3 / 9.3 / 9.2; many, 64 chunks of 500 in blocks of 8, 16, 20, 32,
  // 64, 72, 128 18.1 / 62 / 84, 10.6 / 34.5 / 45, 11.5 / 31.8 / 39.5, 18.2 / 21.6 / 25.8, 29.5 / 16.1 / 17.2, 40.7 /
  // 22.7 / 22.1, 54.9 / 14.9 / 13.9. So one wave up to 16 tokens costs few blocks up to 1.4 us and saves
  // many 24 to 44; from 17 to 32 it is the other way round by 2 to 4 us and 3 to 20. Past 64, 16 waves are
  // within 11% of 8, better from 128 on; at 64 channels 8 stay the better by up to 30% below 128.
  const int n = min(p.max_len, p.m2);
  if (n <= 16) append_launch_w<HD, FMT, 1>(p, dtype, s);
  else if (n <= 64) append_launch_w<HD, FMT, 8>(p, dtype, s);
  else append_launch_w<HD, FMT, 16>(p, dtype, s);
}

// paged_read_kernel: output row j of a sequence is row (first + j) % capacity of
// its slot's table. A workgroup takes kReadRows consecutive output rows: a thread
// a row finds its sequence (counting the entries of cu up to the first row, 64 a wave
// instruction, then walking) and its pool row, into LDS; then the rows stream
// through, 16 channels a lane, all of a thread's loads before its first store. Bound by
// the bytes: 16 caches of up to 1M tokens as bf16, 49 MB, in 12 us, 4.1 TB/s (with a lane
// looking its rows up one after the other 13.3).
constexpr int kReadRows = 128;

template <typename OT> __device__ __forceinline__ void store16(OT* p, const float* f) {
  if constexpr (sizeof(OT) == 4) {
#pragma unroll
    for (int i = 0; i < 16; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
  } else {
    typedef OT v8 __attribute__((ext_vector_type(8)));
#pragma unroll
    for (int i = 0; i < 16; i += 8) {
      v8 v;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = (OT)f[i + e];
      *reinterpret_cast<v8*>(p + i) = v;
    }
  }
}

template <int HD, int FMT, typename OT>
__global__ __launch_bounds__(256) void paged_read_kernel(PagedReadParams p) {
  constexpr int LPR = HD / 16, RSTEP = 256 / LPR, NR = kReadRows / RSTEP;
  constexpr int NV = FMT == PF_BF16 ? 2 : 1;  // 16-byte loads of a lane's 16 channels
  constexpr long long kZero = -1, kSkip = -2;
  typedef typename PagedFmt<FMT>::elem elem;
  __shared__ long long src_row[kReadRows];
  const PagedPool& pl = p.pool;
  const int lane = lane_id(), base = blockIdx.x * kReadRows;
  if (threadIdx.x < kReadRows) {
    const int row = base + threadIdx.x;
    long long pr = kSkip;
    int seq = -1;  // the last sequence that starts at or before row `base`
    for (int i = 0; i <= pl.S; i += 64) {
      const bool le = i + lane <= pl.S && pl.cu[i + lane] <= base;
      const int n = __popcll(__ballot(le));
      seq += n;
      if (n < 64) break;
    }
    if (row < pl.N) {
      while (seq + 1 <= pl.S && pl.cu[seq + 1] <= row) ++seq;
      if (seq >= 0 && seq < pl.S) {
        const uint32_t cap = (uint32_t)pl.nbp << pl.log2page;
        const int slot = pl.slots[seq];
        const uint32_t first = pl.ctx ? pl.ctx[seq] : 0, at = row - pl.cu[seq];
        pr = kZero;
        if (cap > 0 && (unsigned)slot < (unsigned)pl.n_slots)
          pr = pool_row(pl, pl.block_table, pl.nbp, slot, (first + at) % cap);
      } else if (p.zero_tail) {
        pr = kZero;
      }
    }
    src_row[threadIdx.x] = pr;
  }
  __syncthreads();
  const int lr = threadIdx.x / LPR, ch = 16 * (threadIdx.x % LPR);
  uint4 v[NR][NV];
  int code[NR];
  long long pr[NR];
#pragma unroll
  for (int k = 0; k < NR; ++k) {
    pr[k] = src_row[k * RSTEP + lr];
    const long long at = pr[k] < 0 ? 0 : pr[k];  // (row 0 of the pool is there: P >= 1)
    const uint4* src = reinterpret_cast<const uint4*>(static_cast<const elem*>(pl.rows) + at * HD + ch);
#pragma unroll
    for (int e = 0; e < NV; ++e) v[k][e] = src[e];
    if constexpr (FMT != PF_BF16) code[k] = pl.scales[at];
  }
#pragma unroll
  for (int k = 0; k < NR; ++k) {
    if (pr[k] == kSkip) continue;
    float f[16];
    if constexpr (FMT == PF_BF16) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t w[4] = {v[k][e].x, v[k][e].y, v[k][e].z, v[k][e].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          f[8 * e + 2 * i] = __uint_as_float(w[i] << 16);
          f[8 * e + 2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
      }
    } else {
      const uint32_t w[4] = {v[k][0].x, v[k][0].y, v[k][0].z, v[k][0].w};
      const float sc = row_scale(code[k]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (FMT == PF_E4M3) {
          const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(w[i], false);
          const auto b = __builtin_amdgcn_cvt_pk_f32_fp8(w[i], true);
          f[4 * i] = a[0]; f[4 * i + 1] = a[1]; f[4 * i + 2] = b[0]; f[4 * i + 3] = b[1];
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) f[4 * i + e] = (float)(int8_t)(w[i] >> (8 * e));
        }
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) f[i] *= sc;
    }
    if (pr[k] == kZero)
#pragma unroll
      for (int i = 0; i < 16; ++i) f[i] = 0.f;
    store16<OT>(static_cast<OT*>(p.out) + (size_t)(base + k * RSTEP + lr) * HD + ch, f);
  }
}

template <int HD, int FMT>
void read_launch(const PagedReadParams& p, int odtype, hipStream_t s) {
  const dim3 grid((unsigned)((p.pool.N + kReadRows - 1) / kReadRows)), block(256);
  if (odtype == DT_BF16) hipLaunchKernelGGL((paged_read_kernel<HD, FMT, bf16_t>), grid, block, 0, s, p);
  else if (odtype == DT_F16) hipLaunchKernelGGL((paged_read_kernel<HD, FMT, _Float16>), grid, block, 0, s, p);
  else hipLaunchKernelGGL((paged_read_kernel<HD, FMT, float>), grid, block, 0, s, p);
}

}  // namespace

#define KCH_PAGED_FMT(FN, P, ...)                                       \
  do {                                                                  \
    if ((P).pool.c == 128) {                                            \
      if (format == PF_BF16) FN<128, PF_BF16>(P, __VA_ARGS__);          \
      else if (format == PF_E4M3) FN<128, PF_E4M3>(P, __VA_ARGS__);     \
      else FN<128, PF_INT8>(P, __VA_ARGS__);                            \
    } else {                                                            \
      if (format == PF_BF16) FN<64, PF_BF16>(P, __VA_ARGS__);           \
      else if (format == PF_E4M3) FN<64, PF_E4M3>(P, __VA_ARGS__);      \
      else FN<64, PF_INT8>(P, __VA_ARGS__);                             \
    }                                                                   \
  } while (0)

hipError_t paged_append_dispatch(const PagedAppendParams& p, int format, int dtype, hipStream_t s) {
  KCH_PAGED_FMT(append_launch, p, dtype, s);
  return hipGetLastError();
}

hipError_t paged_read_dispatch(const PagedReadParams& p, int format, int odtype, hipStream_t s) {
  KCH_PAGED_FMT(read_launch, p, odtype, s);
  return hipGetLastError();
}

}  // namespace kch
