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
// A workgroup takes one block: its rows 16 bytes a lane (HD / 8 lanes a row), so
// a row's norm and maximum are reductions over neighbouring lanes, and C and Z
// are read once for both outputs. The workgroup of a sequence's first block also
// takes the block that the chunk leaves open, because it alone may read the
// sequence's old sums: no other workgroup writes them.

#include "paged.h"

namespace kch {

namespace {

// Reductions over groups of W neighbouring lanes.
template <int W> __device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int m = W / 2; m >= 1; m >>= 1) v += __shfl_xor(v, m);
  return v;
}
template <int W> __device__ __forceinline__ float group_amax(float v) {
#pragma unroll
  for (int m = W / 2; m >= 1; m >>= 1) v = amax_nan(v, __shfl_xor(v, m));
  return v;
}

// e^(a - b) of softmax references: a = -inf (nothing summed yet) gives 0, also
// where b is -inf.
__device__ __forceinline__ float ref_exp(float a, float b) { return exp_hw(a - fmaxf(b, -3e38f)); }

constexpr int kBatchRows = 4;  // rows of a lane whose loads are in flight together

template <int HD, int FMT, typename T>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedAppendParams p) {
  constexpr int LPR = HD / 8;        // lanes per row
  constexpr int RPW = 64 / LPR;      // rows of a wave at a time
  constexpr int STEP = 4 * RPW;      // rows of the workgroup at a time
  typedef typename PagedFmt<FMT>::elem elem;
  __shared__ float red[4][3][HD];
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

  auto block = [&](uint32_t b) {
    const uint32_t lo = max(b * m2, sq.ctx), hi = min((b + 1) * m2, end);
    float m[8], l[8], a[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      m[i] = -INFINITY;
      l[i] = a[i] = 0.f;
    }
    for (uint32_t r0 = lo; r0 < hi; r0 += STEP * kBatchRows) {
      float c8[kBatchRows][8], z8[kBatchRows][8];
#pragma unroll
      for (int u = 0; u < kBatchRows; ++u) {
        const uint32_t pos = r0 + u * STEP + wv * RPW + sub;
        if (pos < hi) {
          const long long row = sq.row0 + (int)(pos - sq.ctx);
          Load8<T>::run(static_cast<const T*>(p.C) + row * p.ldc + ch, c8[u]);
          Load8<T>::run(static_cast<const T*>(p.Z) + row * p.ldz + ch, z8[u]);
        }
      }
#pragma unroll
      for (int u = 0; u < kBatchRows; ++u) {
        const uint32_t pos = r0 + u * STEP + wv * RPW + sub;
        const bool live = pos < hi;
        float b8[8];
        if (live) Load8<float>::run(p.B_pos + (size_t)(pos - b * m2) * HD + ch, b8);
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          c8[u][i] = live ? c8[u][i] : 0.f;
          z8[u][i] = live ? z8[u][i] + b8[i] : -INFINITY;
          ss += c8[u][i] * c8[u][i];
        }
        // the window row, unless a later token of this chunk takes its place
        if (cap > 0) {
          const float inv = p.normalize ? l2_inv(group_sum<LPR>(ss)) : 1.f;
          float x[8], mx = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            x[i] = c8[u][i] * inv;
            mx = amax_nan(mx, x[i]);
          }
          if constexpr (FMT != PF_BF16) mx = group_amax<LPR>(mx);
          const long long pr = live && end - pos <= cap
                                   ? pool_row(p.pool, p.pool.ring_table, p.pool.nrp, sq.slot, pos % cap)
                                   : -1;
          if (pr >= 0) {
            if constexpr (FMT == PF_BF16) {
              *reinterpret_cast<bf16x8*>(rows + pr * HD + ch) = to_bf16x8(x);
            } else {
              const int code = row_scale_code<FMT>(mx);
              *reinterpret_cast<uint2*>(rows + pr * HD + ch) =
                  make_uint2(quant4<FMT>(x[0], x[1], x[2], x[3], code), quant4<FMT>(x[4], x[5], x[6], x[7], code));
              if (ch == 0) p.pool.scales[pr] = (uint8_t)code;
            }
          }
        }
      }
      // one reference for the batch, so that a channel rescales once for it
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float mn = m[i];
#pragma unroll
        for (int u = 0; u < kBatchRows; ++u) mn = fmaxf(mn, z8[u][i]);
        const float f = ref_exp(m[i], mn);
        l[i] *= f;
        a[i] *= f;
        m[i] = mn;
#pragma unroll
        for (int u = 0; u < kBatchRows; ++u) {
          const float e = ref_exp(z8[u][i], mn);
          l[i] += e;
          // a masked token's value does not enter, whatever it is
          a[i] = e != 0.f ? fmaf(e, c8[u][i], a[i]) : a[i];
        }
      }
    }
    // the rows of the wave, then the four waves
#pragma unroll
    for (int i = 0; i < 8; ++i) {
#pragma unroll
      for (int s = LPR; s < 64; s <<= 1) {
        const float mo = __shfl_xor(m[i], s), lo_ = __shfl_xor(l[i], s), ao = __shfl_xor(a[i], s);
        const float mn = fmaxf(m[i], mo), f = ref_exp(m[i], mn), g = ref_exp(mo, mn);
        l[i] = l[i] * f + lo_ * g;
        a[i] = a[i] * f + ao * g;
        m[i] = mn;
      }
      if (sub == 0) {
        red[wv][0][ch + i] = m[i];
        red[wv][1][ch + i] = l[i];
        red[wv][2][ch + i] = a[i];
      }
    }
    __syncthreads();
    if (wv == 0) {
      constexpr int CPL = HD / 64;  // channels per lane
      const bool carried = b == b0 && sq.ctx != b0 * m2;
      const bool ends = (b + 1) * m2 <= end;
      float x[CPL], mm[CPL], ll[CPL], aa[CPL], ss = 0.f, mx = 0.f;
#pragma unroll
      for (int k = 0; k < CPL; ++k) {
        const int c = CPL * lane + k;
        float mn = carried ? state[c] : -INFINITY, ls = carried ? state[HD + c] : 0.f,
              as = carried ? state[2 * HD + c] : 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float mo = red[w][0][c], mt = fmaxf(mn, mo), f = ref_exp(mn, mt), g = ref_exp(mo, mt);
          ls = ls * f + red[w][1][c] * g;
          as = as * f + red[w][2][c] * g;
          mn = mt;
        }
        mm[k] = mn;
        ll[k] = ls;
        aa[k] = as;
        x[k] = ls == 0.f ? 0.f : as / ls;  // a channel without a weight: 0
        ss += x[k] * x[k];
      }
      if (ends) {
        const float inv = p.normalize ? l2_inv(wave_sum(ss)) : 1.f;
#pragma unroll
        for (int k = 0; k < CPL; ++k) {
          x[k] *= inv;
          mx = amax_nan(mx, x[k]);
        }
        const long long pr = pool_row(p.pool, p.pool.block_table, p.pool.nbp, sq.slot, b);
        if constexpr (FMT != PF_BF16) mx = group_amax<64>(mx);
        if (pr >= 0) {
          elem* dst = rows + pr * HD + CPL * lane;
          if constexpr (FMT == PF_BF16) {
#pragma unroll
            for (int k = 0; k < CPL; ++k) dst[k] = (bf16_t)x[k];
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
          state[c] = mm[k];
          state[HD + c] = ll[k];
          state[2 * HD + c] = aa[k];
        }
      }
    }
    __syncthreads();  // red is free again
  };

  // the open block is the first workgroup's, after the sums it read
  const uint32_t last = open && bl > b0 ? bl - 1 : bl;
  for (uint32_t b = b0 + blockIdx.x; b <= last; b += gridDim.x) block(b);
  if (blockIdx.x == 0 && last < bl) block(bl);
}

template <int HD, int FMT>
void append_launch(const PagedAppendParams& p, int dtype, hipStream_t s) {
  const dim3 grid((unsigned)((p.max_len + p.m2 - 2) / p.m2 + 1), (unsigned)p.pool.S), block(256);
  if (dtype == DT_BF16) hipLaunchKernelGGL((paged_append_kernel<HD, FMT, bf16_t>), grid, block, 0, s, p);
  else if (dtype == DT_F16) hipLaunchKernelGGL((paged_append_kernel<HD, FMT, _Float16>), grid, block, 0, s, p);
  else hipLaunchKernelGGL((paged_append_kernel<HD, FMT, float>), grid, block, 0, s, p);
}

// paged_read_kernel: output row j of a sequence is row (first + j) % capacity of
// its slot's table. 16 channels a lane; a workgroup takes kReadRows consecutive
// output rows, whose sequences it finds by counting the entries of cu up to them
// (64 a wave instruction) and then walks.
constexpr int kReadRows = 128;

template <int HD, int FMT, typename OT>
__global__ __launch_bounds__(256) void paged_read_kernel(PagedReadParams p) {
  constexpr int LPR = HD / 16, RSTEP = 256 / LPR;
  typedef typename PagedFmt<FMT>::elem elem;
  const PagedPool& pl = p.pool;
  const int lane = lane_id(), ch = 16 * (threadIdx.x % LPR);
  const int base = blockIdx.x * kReadRows;
  int seq = -1;  // the last sequence that starts at or before row `base`
  for (int i = 0; i <= pl.S; i += 64) {
    const bool le = i + lane <= pl.S && pl.cu[i + lane] <= base;
    const int n = __popcll(__ballot(le));
    seq += n;
    if (n < 64) break;
  }
  const uint32_t cap = (uint32_t)pl.nbp << pl.log2page;
  OT* out = static_cast<OT*>(p.out);
#pragma unroll 4
  for (int k = 0; k < kReadRows / RSTEP; ++k) {
    const int row = base + k * RSTEP + (int)threadIdx.x / LPR;
    if (row >= pl.N) break;
    while (seq + 1 <= pl.S && pl.cu[seq + 1] <= row) ++seq;
    long long pr = -1;
    if (seq >= 0 && seq < pl.S) {
      const int slot = pl.slots[seq];
      const uint32_t first = pl.ctx ? pl.ctx[seq] : 0, at = row - pl.cu[seq];
      if (cap > 0 && (unsigned)slot < (unsigned)pl.n_slots)
        pr = pool_row(pl, pl.block_table, pl.nbp, slot, (first + at) % cap);
    } else if (!p.zero_tail) {
      continue;
    }
    float f[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) f[i] = 0.f;
    if (pr >= 0) {
      const elem* src = static_cast<const elem*>(pl.rows) + pr * HD + ch;
      if constexpr (FMT == PF_BF16) {
        Load8<bf16_t>::run(src, f);
        Load8<bf16_t>::run(src + 8, f + 8);
      } else {
        const uint4 w = *reinterpret_cast<const uint4*>(src);
        const float sc = row_scale(pl.scales[pr]);
        const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (FMT == PF_E4M3) {
            const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(ww[i], false);
            const auto b = __builtin_amdgcn_cvt_pk_f32_fp8(ww[i], true);
            f[4 * i] = a[0]; f[4 * i + 1] = a[1]; f[4 * i + 2] = b[0]; f[4 * i + 3] = b[1];
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) f[4 * i + e] = (float)(int8_t)(ww[i] >> (8 * e));
          }
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) f[i] *= sc;
      }
    }
    OT* dst = out + (size_t)row * HD + ch;
#pragma unroll
    for (int i = 0; i < 16; i += 4) Store4<OT>::run(dst + i, f32x4{f[i], f[i + 1], f[i + 2], f[i + 3]}, 1.f);
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
