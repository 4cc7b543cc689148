// Few rows times a matrix of 4-bit weights with group scales (gfx950):
//   y[m, n] = sum_k x[m, k] s[k / G, n] (q[n, k] - z[k / G, n])  (+ res[m, n])
// q the 4-bit codes, two a byte (low nibble: even k), rows of K / 2 bytes; s in
// x's type; z uint8, or 8 everywhere. x and y bf16 or fp16, sums fp32, rounded once.
//
// It serves the layer projections of a decode step, as kch_linear_rows does, with a
// quarter of the bytes; what bounds it is the stream of the codes.
//
// y^T = W x^T on v_mfma_f32_16x16x32: A is a 16-row tile of W, B x^T (zero past
// M). A code becomes a 16-bit float without arithmetic: the nibble in the low
// mantissa bits of 128 (bf16) or 1024 (fp16) is 128 + q (1024 + q) exactly, one
// and-or for two codes. The offset and the zero point leave with the sum of x
// over the group: sum x (q - z) = sum x (128 + q) - (128 + z) sum x, both in
// fp32, the second sum by the same instruction with a tile of ones, which puts it
// where the first one is. Each group is then scaled in fp32 (so no weight is
// rounded to 16 bits).
//
// A lane loads 16 bytes, 32 codes of its row (4 lanes cover 128 consecutive k), and
// the four words change places among the four lanes of a row (a 4 x 4 transpose
// with the row swaps) so that an MFMA step holds 32 consecutive k and a group
// is whole steps.

#include "attn_common.h"
#include "kch_kernels.h"

namespace kch {

namespace {

template <typename T> struct W4Type;
template <> struct W4Type<bf16_t> {
  typedef bf16x8 v8;
  static constexpr uint32_t magic = 0x43004300u;  // 128
  static constexpr float offset = 128.f;
  static constexpr uint32_t one2 = 0x3f803f80u;
  static __device__ __forceinline__ f32x4 mfma(v8 a, v8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <> struct W4Type<_Float16> {
  typedef f16x8 v8;
  static constexpr uint32_t magic = 0x64006400u;  // 1024
  static constexpr float offset = 1024.f;
  static constexpr uint32_t one2 = 0x3c003c00u;
  static __device__ __forceinline__ f32x4 mfma(v8 a, v8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};

// Words of the four lanes {r, r + 16, r + 32, r + 48}: lane group q's register j
// becomes lane group j's register q.
__device__ __forceinline__ void transpose4(uint32_t (&w)[4]) {
  auto a = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
  auto b = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
  auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
  auto d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
  w[0] = c[0]; w[1] = c[1]; w[2] = d[0]; w[3] = d[1];
}

// KW waves share a 16-row tile of W and its K range, 128 k at a time in turn.
template <typename T, int KW, int G, bool ZP>
__global__ __launch_bounds__(64 * KW) void linear_w4_kernel(LinearW4Params p) {
  using W = W4Type<T>;
  typedef typename W::v8 v8;
  constexpr int U = 2;      // 128-k pieces of a wave whose loads are in flight together
  constexpr int SPG = G / 32;  // MFMA steps of a group
  __shared__ float part[KW][16][17];
  const int wv = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int lane = lane_id(), r = lane & 15, q = lane >> 4;
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16;
  const int K = p.K, N = p.N;
  // rows past N read row N - 1 again (never stored)
  const uint4* wrow = reinterpret_cast<const uint4*>(p.w + (size_t)min(n0 + r, N - 1) * (K / 2)) + q;
  const bool mok = m0 + r < p.M;
  const T* xrow = static_cast<const T*>(p.x) + (size_t)(mok ? m0 + r : 0) * p.ldx + 8 * q;
  const T* const sc = static_cast<const T*>(p.scales);
  const int np = (K + 127) / 128;
  const int ns = n0 + 4 * q;  // the lane's four rows of y^T
  uint4 ones_w = make_uint4(W::one2, W::one2, W::one2, W::one2);
  const v8 ones = __builtin_bit_cast(v8, ones_w);
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  const uint4 z4 = make_uint4(0, 0, 0, 0);
  for (int p0 = wv; p0 < np; p0 += KW * U) {
    uint4 wq[U], xq[U][4];
    float s[U][4 / SPG][4], z[U][4 / SPG][4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int pc = p0 + u * KW, k0 = 128 * pc;
      wq[u] = pc < np && k0 + 32 * q < K ? wrow[4 * pc] : z4;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        xq[u][j] = mok && pc < np && k0 + 32 * j < K ? *reinterpret_cast<const uint4*>(xrow + k0 + 32 * j) : z4;
#pragma unroll
      for (int g = 0; g < 4 / SPG; ++g) {
        const int k = k0 + G * g;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool ok = pc < np && k < K;
          const size_t at = (size_t)(ok ? k / G : 0) * N + min(ns + e, N - 1);
          s[u][g][e] = ok ? to_f32(sc[at]) : 0.f;
          z[u][g][e] = W::offset + (ZP ? (float)p.zeros[at] : 8.f);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      uint32_t w4[4] = {wq[u].x, wq[u].y, wq[u].z, wq[u].w};
      transpose4(w4);
      f32x4 raw = {0.f, 0.f, 0.f, 0.f}, sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        // codes (e, e + 4) of the word in the halves of register e, and x alike
        uint4 a;
        a.x = (w4[j] & 0x000f000fu) | W::magic;
        a.y = ((w4[j] >> 4) & 0x000f000fu) | W::magic;
        a.z = ((w4[j] >> 8) & 0x000f000fu) | W::magic;
        a.w = ((w4[j] >> 12) & 0x000f000fu) | W::magic;
        const uint4 x = xq[u][j];
        uint4 b;
        b.x = __builtin_amdgcn_perm(x.z, x.x, 0x05040100u);
        b.y = __builtin_amdgcn_perm(x.z, x.x, 0x07060302u);
        b.z = __builtin_amdgcn_perm(x.w, x.y, 0x05040100u);
        b.w = __builtin_amdgcn_perm(x.w, x.y, 0x07060302u);
        const v8 bv = __builtin_bit_cast(v8, b);
        raw = W::mfma(__builtin_bit_cast(v8, a), bv, raw);
        sum = W::mfma(ones, bv, sum);
        if (j % SPG == SPG - 1) {
          const int g = j / SPG;
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[e] = fmaf(s[u][g][e], fmaf(-z[u][g][e], sum[e], raw[e]), acc[e]);
          raw = sum = f32x4{0.f, 0.f, 0.f, 0.f};
        }
      }
    }
  }
  // acc[e]: y^T[n0 + 4 q + e][m0 + r]
#pragma unroll
  for (int e = 0; e < 4; ++e) part[wv][r][4 * q + e] = acc[e];
  __syncthreads();
  for (int t = threadIdx.x; t < 256; t += 64 * KW) {
    const int m = t >> 4, n = t & 15;
    if (m0 + m >= p.M || n0 + n >= N) continue;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < KW; ++w) v += part[w][m][n];
    if (p.res) v += to_f32(static_cast<const T*>(p.res)[(size_t)(m0 + m) * p.ldr + n0 + n]);
    static_cast<T*>(p.y)[(size_t)(m0 + m) * p.ldy + n0 + n] = from_f32<T>(v);
  }
}

template <typename T, int G>
void w4_launch(const LinearW4Params& p, hipStream_t s) {
  const dim3 grid((unsigned)((p.N + 15) / 16), (unsigned)((p.M + 15) / 16));
  if (p.zeros) hipLaunchKernelGGL((linear_w4_kernel<T, 4, G, true>), grid, dim3(256), 0, s, p);
  else hipLaunchKernelGGL((linear_w4_kernel<T, 4, G, false>), grid, dim3(256), 0, s, p);
}

template <typename T>
void w4_launch_g(const LinearW4Params& p, hipStream_t s) {
  if (p.group == 32) w4_launch<T, 32>(p, s);
  else if (p.group == 64) w4_launch<T, 64>(p, s);
  else w4_launch<T, 128>(p, s);
}

}  // namespace

hipError_t linear_w4_dispatch(const LinearW4Params& p, int dtype, hipStream_t s) {
  if (dtype == DT_BF16) w4_launch_g<bf16_t>(p, s);
  else w4_launch_g<_Float16>(p, s);
  return hipGetLastError();
}

}  // namespace kch
