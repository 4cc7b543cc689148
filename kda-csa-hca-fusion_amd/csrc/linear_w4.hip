// Few rows times a matrix of 4-bit weights with group scales (gfx950):
//   y[m, n] = sum_k x[m, k] s[k / G, n] (q[n, k] - z[k / G, n])  (+ res[m, n])
// q the 4-bit codes, two a byte (low nibble: even k), rows of K / 2 bytes; s in
// x's type; z uint8, or 8 everywhere. x and y bf16 or fp16, sums fp32, rounded once.
//
// It serves the layer projections of a decode step, as kch_linear_rows does, with a
// quarter of the bytes; what bounds it is the stream of the codes. Every 16 rows read and unpack
// them again: 64 rows of N 16384, K 8192 take 65 us where the bf16 product takes 47, 512 475
// and 116 (N = K = 2048: 8.5 and 19, 25 and 20).
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

// y[m, n] term by term, in fp64: for sums that came out infinite or NaN. An infinite x, or sums
// of 128 x past fp32's range, meet their own negative in the offset's sum, where the
// definition's product is an infinity or finite.
template <typename T>
__device__ __forceinline__ float w4_terms(const LinearW4Params& p, int m, int n) {
  const T* const x = static_cast<const T*>(p.x) + (size_t)m * p.ldx;
  const uint32_t* const w = reinterpret_cast<const uint32_t*>(p.w + (size_t)n * (p.K / 2));
  double sum = 0.0;
#pragma unroll 1
  for (int k = 0; k < p.K; k += 8) {
    const size_t g = (size_t)(k / p.group) * p.N + n;
    const float s = to_f32(static_cast<const T*>(p.scales)[g]);
    const int z = p.zeros ? p.zeros[g] : 8;
    const uint32_t c = w[k / 8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      sum += (double)to_f32(x[k + i]) * ((double)s * ((int)(c >> (4 * i) & 15u) - z));
  }
  return (float)sum;
}

// What a wave holds of 128 consecutive k: its tiles' codes, x, and per group the scales
// (4 of 16 bits) and zero points (4 bytes) of the lane's rows of y^T.
template <int NT, int G> struct W4Piece {
  uint4 w[NT], x[4];
  uint2 s[128 / G][NT];
  uint32_t z[128 / G][NT];
};

// A workgroup takes NT 16-row tiles of W, its KW waves the K range 128 k at a time in
// turn. The tiles of a wave share x (at M = 16 its rows are four times a tile's codes) and
// the tile of ones. x is read by whole 128-byte lines and changes places through the wave's
// LDS: in the order of its MFMA operand, 64 bytes of each of 16 rows an instruction, it
// bound the kernel (16 rows, N 4096, K 8192: 13.7 against 10.1 us). VEC: N is a multiple of 4,
// four scales are one load. The loop has no load behind a branch: a wait there would drain
// every load in flight (the same kernel with such loads took 145 us where it took 43).
// At 16 rows, N 16384, K 8192 17.3 us a call (traced 19.1 to 19.4), 4.1 TB/s; 13.9 us is what its 71 MB take at the rate of a
// large copy. Past the stream it is the 56 vector instructions a tile and 128 k, mostly the
// codes' unpacking.
template <typename T, int NT, int KW, int G, bool ZP, bool VEC, bool KT>
__global__ __launch_bounds__(64 * KW) void linear_w4_kernel(LinearW4Params p) {
  using W = W4Type<T>;
  typedef typename W::v8 v8;
  typedef W4Piece<NT, G> Piece;
  constexpr int NG = 128 / G;
  constexpr int XB = 4096, PB = 16 * (16 * NT + 1) * 4;  // bytes of a wave's x and of its partial tiles
  __shared__ __attribute__((aligned(16))) char lds[KW * (XB > PB ? XB : PB)];
  float (*const part)[16][16 * NT + 1] = reinterpret_cast<float (*)[16][16 * NT + 1]>(lds);
  const int wv = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int lane = lane_id(), r = lane & 15, q = lane >> 4;
  const int n0 = blockIdx.x * 16 * NT, m0 = blockIdx.y * 16;
  const int K = p.K, N = p.N;
  // rows past M and N read the last one again: their results are never stored
  const T* const xa = static_cast<const T*>(p.x) + (size_t)min(m0 + lane / 8, p.M - 1) * p.ldx + 8 * (lane & 7);
  const T* const xb = static_cast<const T*>(p.x) + (size_t)min(m0 + 8 + lane / 8, p.M - 1) * p.ldx + 8 * (lane & 7);
  uint4* const xl = reinterpret_cast<uint4*>(lds) + 256 * wv;
  const uint4* wrow[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t)
    wrow[t] = reinterpret_cast<const uint4*>(p.w + (size_t)min(n0 + 16 * t + r, N - 1) * (K / 2)) + q;
  const uint16_t* const sc = static_cast<const uint16_t*>(p.scales);

  // TAIL: the last piece where K is no multiple of 128; what lies past K is read from
  // inside the row and meets zeros of x
  auto load = [&](Piece& c, int pc, auto tail) {
    constexpr bool TAIL = decltype(tail)::value;
    const int k0 = 128 * pc;
#pragma unroll
    for (int t = 0; t < NT; ++t) c.w[t] = wrow[t][TAIL && k0 + 32 * q >= K ? -q : 4 * pc];
    const int kl = 8 * (lane & 7), ka = k0 + kl, kb = ka + 64;  // this lane's k of its two lines
    const bool pa = TAIL && ka >= K, pb = TAIL && kb >= K;         // (past the row: its start instead)
    c.x[0] = *reinterpret_cast<const uint4*>(xa + (pa ? -kl : k0));
    c.x[1] = *reinterpret_cast<const uint4*>(xa + (pb ? -kl : k0 + 64));
    c.x[2] = *reinterpret_cast<const uint4*>(xb + (pa ? -kl : k0));
    c.x[3] = *reinterpret_cast<const uint4*>(xb + (pb ? -kl : k0 + 64));
    if (pa) c.x[0] = c.x[2] = make_uint4(0, 0, 0, 0);
    if (pb) c.x[1] = c.x[3] = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const size_t row = (size_t)(TAIL ? min(k0 / G + g, K / G - 1) : k0 / G + g) * N;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int n = n0 + 16 * t + 4 * q;
        if constexpr (VEC) {
          const size_t at = row + min(n, N - 4);
          c.s[g][t] = *reinterpret_cast<const uint2*>(sc + at);
          if constexpr (ZP) c.z[g][t] = *reinterpret_cast<const uint32_t*>(p.zeros + at);
        } else {
          uint32_t v[4], z = 0;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const size_t at = row + min(n + e, N - 1);
            v[e] = sc[at];
            if constexpr (ZP) z |= (uint32_t)p.zeros[at] << (8 * e);
          }
          c.s[g][t] = make_uint2(v[0] | v[1] << 16, v[2] | v[3] << 16);
          if constexpr (ZP) c.z[g][t] = z;
        }
      }
    }
  };

  const v8 ones = __builtin_bit_cast(v8, make_uint4(W::one2, W::one2, W::one2, W::one2));
  f32x4 acc[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};

  auto use = [&](Piece& c) {
    uint32_t w4[NT][4];
    v8 bx[4];
    wave_lds_sync();
    const int ra = lane / 8, ch = lane & 7;
    xl[16 * ra + (ch ^ ra)] = c.x[0];
    xl[16 * ra + ((8 + ch) ^ ra)] = c.x[1];
    xl[16 * (8 + ra) + (ch ^ (8 + ra))] = c.x[2];
    xl[16 * (8 + ra) + ((8 + ch) ^ (8 + ra))] = c.x[3];
    wave_lds_sync();
#pragma unroll
    for (int j = 0; j < 4; ++j) c.x[j] = xl[16 * r + ((4 * j + q) ^ r)];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      w4[t][0] = c.w[t].x; w4[t][1] = c.w[t].y; w4[t][2] = c.w[t].z; w4[t][3] = c.w[t].w;
      transpose4(w4[t]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      // codes (e, e + 4) of a word come out in the halves of register e: x alike
      const uint4 x = c.x[j];
      uint4 b;
      b.x = __builtin_amdgcn_perm(x.z, x.x, 0x05040100u);
      b.y = __builtin_amdgcn_perm(x.z, x.x, 0x07060302u);
      b.z = __builtin_amdgcn_perm(x.w, x.y, 0x05040100u);
      b.w = __builtin_amdgcn_perm(x.w, x.y, 0x07060302u);
      bx[j] = __builtin_bit_cast(v8, b);
    }
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      // sum x, and what the offset (and a zero point of 8) adds to every code: the
      // products start from its negative
      f32x4 sum = {0.f, 0.f, 0.f, 0.f}, base;
#pragma unroll
      for (int j = g * G / 32; j < (g + 1) * G / 32; ++j) sum = W::mfma(ones, bx[j], sum);
#pragma unroll
      for (int e = 0; e < 4; ++e) base[e] = -(W::offset + (ZP ? 0.f : 8.f)) * sum[e];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        f32x4 raw = base;
#pragma unroll
        for (int j = g * G / 32; j < (g + 1) * G / 32; ++j) {
          const uint32_t w = w4[t][j];
          uint4 a;
          a.x = (w & 0x000f000fu) | W::magic;
          a.y = ((w >> 4) & 0x000f000fu) | W::magic;
          a.z = ((w >> 8) & 0x000f000fu) | W::magic;
          a.w = ((w >> 12) & 0x000f000fu) | W::magic;
          raw = W::mfma(__builtin_bit_cast(v8, a), bx[j], raw);
        }
        const uint32_t sw[2] = {c.s[g][t].x, c.s[g][t].y};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float s = to_f32(__builtin_bit_cast(T, (uint16_t)(sw[e >> 1] >> (16 * (e & 1)))));
          const float d = ZP ? fmaf(-(float)((c.z[g][t] >> (8 * e)) & 255u), sum[e], raw[e]) : raw[e];
          acc[t][e] = fmaf(s, d, acc[t][e]);
        }
      }
    }
  };

  // two pieces in turn: the next one's loads are in flight while one is used (past the
  // end the last one again, from the cache); KT: K has a tail past its last 128, which
  // comes first, beside the first piece (its code alone, unused, cost the large case 8%)
  const std::integral_constant<bool, false> whole{};
  const int nf = K / 128;
  Piece c0, c1;
  if (wv < nf) load(c0, wv, whole);
  if (KT && wv == nf % KW) {
    load(c1, nf, std::integral_constant<bool, true>{});
    use(c1);
  }
  if (wv < nf) {
    for (int pc = wv; pc < nf; pc += 2 * KW) {
      load(c1, min(pc + KW, nf - 1), whole);
      use(c0);
      load(c0, min(pc + 2 * KW, nf - 1), whole);
      if (pc + KW < nf) use(c1);
    }
  }
  __syncthreads();  // the partial tiles go where x was
  // acc[t][e]: y^T[n0 + 16 t + 4 q + e][m0 + r]
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) part[wv][r][16 * t + 4 * q + e] = acc[t][e];
  __syncthreads();
  for (int i = threadIdx.x; i < 256 * NT; i += 64 * KW) {
    const int m = i / (16 * NT), n = i % (16 * NT);
    if (m0 + m >= p.M || n0 + n >= N) continue;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < KW; ++w) v += part[w][m][n];
    if (!(fabsf(v) < INFINITY)) v = w4_terms<T>(p, m0 + m, n0 + n);
    if (p.res) v += to_f32(static_cast<const T*>(p.res)[(size_t)(m0 + m) * p.ldr + n0 + n]);
    static_cast<T*>(p.y)[(size_t)(m0 + m) * p.ldy + n0 + n] = from_f32<T>(v);
  }
}

template <typename T, int NT, int G, bool VEC>
void w4_launch(const LinearW4Params& p, hipStream_t s) {
  const dim3 grid((unsigned)((p.N + 16 * NT - 1) / (16 * NT)), (unsigned)((p.M + 15) / 16)), block(512);
#define KCH_W4(ZP, KT) hipLaunchKernelGGL((linear_w4_kernel<T, NT, 8, G, ZP, VEC, KT>), grid, block, 0, s, p)
  if constexpr (G < 128) {
    if (p.K % 128) {
      if (p.zeros) KCH_W4(true, true);
      else KCH_W4(false, true);
      return;
    }
  }
  if (p.zeros) KCH_W4(true, false);
  else KCH_W4(false, false);
#undef KCH_W4
}

template <typename T, int NT, bool VEC>
void w4_launch_g(const LinearW4Params& p, hipStream_t s) {
  if (p.group == 32) w4_launch<T, NT, 32, VEC>(p, s);
  else if (p.group == 64) w4_launch<T, NT, 64, VEC>(p, s);
  else w4_launch<T, NT, 128, VEC>(p, s);
}

// Tiles of a workgroup of 8 waves (one a CU): as many as leave a workgroup for each of 256
// CUs. Measured (us, bf16, groups of 128, weights from HBM) with 1 / 2 / 4 tiles: one row, N 2048,
// K 2048 4.1 / 4.8 / 6.6; 16 rows, N 4096, K 8192 10.1 / 12.0 / 18.2, N 8192, K 2048 7.4 /
// 6.2 / 8.9, N 16384, K 8192 29.1 / 22.1 / 20.3.
template <typename T>
void w4_launch_n(const LinearW4Params& p, hipStream_t s) {
  const long long tiles = (long long)((p.N + 15) / 16) * ((p.M + 15) / 16);
  if (p.N % 4 || ((uintptr_t)p.scales & 7) || ((uintptr_t)p.zeros & 3)) w4_launch_g<T, 1, false>(p, s);
  else if (tiles >= 1024) w4_launch_g<T, 4, true>(p, s);
  else if (tiles >= 512) w4_launch_g<T, 2, true>(p, s);
  else w4_launch_g<T, 1, true>(p, s);
}

}  // namespace

hipError_t linear_w4_dispatch(const LinearW4Params& p, int dtype, hipStream_t s) {
  if (dtype == DT_BF16) w4_launch_n<bf16_t>(p, s);
  else w4_launch_n<_Float16>(p, s);
  return hipGetLastError();
}

}  // namespace kch
