// Linears in 8-bit integers: rows quantised with one scale each, and their product with a weight held in
// 8 bits with one scale per output channel.
//
//   a_r = max_k |x_rk|,  s_r = a_r / 127,  q_rk = rne(127 x_rk / a_r)
//   y_mn = act( sx_m sw_n sum_k qx_mk qw_nk + b_n + r_mn )
//
// The sum is an integer (|sum| <= 127^2 K < 2^31 for every K the host accepts), so it is exact in any
// order: tiles, k-splits and batch sizes never change a bit of the result.
#include "common.h"

enum { ACT_NONE = 0, ACT_GELU = 1, ACT_QUICK_GELU = 2, ACT_GEGLU = 3 };

// 16-bit element <-> float; EL 0: bf16, 1: fp16
template <int EL>
__device__ __forceinline__ float dec16(uint32_t v) {
  if constexpr (EL == 0) return __uint_as_float(v << 16);
  else return (float)__builtin_bit_cast(_Float16, (uint16_t)v);
}
template <int EL>
__device__ __forceinline__ uint32_t enc16(float f) {
  if constexpr (EL == 0) return f2bf(f);
  else return __builtin_bit_cast(uint16_t, (_Float16)f);
}

__device__ __forceinline__ float act_f(float y, int act) {
  if (act == ACT_GELU) return gelu_f(y);
  if (act == ACT_QUICK_GELU) return y * __builtin_amdgcn_rcpf(1.f + fast_exp(-1.702f * y));
  return y;
}

// ---------------------------------------------------------------------------------------------
// Row quantisation.  A half step k + 1/2 of r = 127 x / a is an exact ratio of the row's numbers: 254 x and
// (2k + 1) a are multiples of x's last bit, so an r that is not on a half step is at least (k + 1/2) 2^-19
// away from it (11-bit fp16 significands; bf16: 2^-16).  x * (127 / a) in fp32 is off by less than 2^-23 of
// itself, so rounding it to 21 significant bits puts every exact half step back on its place and moves
// nothing across one: q is the correctly rounded (half to even) quotient, bit for bit that of a 64-bit
// division, for four VALU operations instead of a division.
__device__ __forceinline__ uint32_t quant_one(float x, float inv) {
  const float r = __uint_as_float((__float_as_uint(x * inv) + 4u) & ~7u);
  return __float_as_uint(r + 12582912.f);       // 1.5 2^23: r's integer in the low bits (the low byte is q)
}
// 127 / a with x pre-scaled by `up` where 127 / a would leave the fp32 range (a below 2^-100: bf16 only)
__device__ __forceinline__ void quant_scale(float a, float& s, float& inv, float& up) {
  up = a < 7.888609e-31f ? 1.2676506e30f : 1.f;      // 2^-100, 2^100
  const bool fine = a <= 3.4028235e38f;               // false for inf and NaN
  s = fine ? a / 127.f : __builtin_nanf("");
  inv = fine && a > 0.f ? 127.f / (a * up) : 0.f;
}

// 8 values as 8 bytes: the low bytes of the four + four integers
__device__ __forceinline__ uint2 quant8(const float (&f)[8], float inv, float up) {
  uint32_t w[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const uint32_t a = quant_one(f[4 * e] * up, inv), b = quant_one(f[4 * e + 1] * up, inv);
    const uint32_t c = quant_one(f[4 * e + 2] * up, inv), d = quant_one(f[4 * e + 3] * up, inv);
    w[e] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0c0c0400u), __builtin_amdgcn_perm(b, a, 0x0c0c0400u),
                                 0x05040100u);
  }
  return make_uint2(w[0], w[1]);
}
template <int EL>
__device__ __forceinline__ void dec8(uint4 v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = dec16<EL>(w[i] & 0xffffu);
    f[2 * i + 1] = dec16<EL>(w[i] >> 16);
  }
}
// sum / maximum over the T threads (64: a wave, 256: the block) that share a row; fixed order
template <int T, bool MAX>
__device__ __forceinline__ float row_reduce(float v, float* red) {
  v = MAX ? wave_max(v) : wave_sum(v);
  if constexpr (T == 256) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = MAX ? fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])) : (red[0] + red[1]) + (red[2] + red[3]);
  }
  return v;
}

// One row per T threads (T = 64: four rows per workgroup), held in registers: V vectors of 8 elements per thread,
// K <= 8 T V, K % 8 == 0, 16-byte aligned rows.  LN: LayerNorm in fp32 first (two exact passes over the
// registers), the normalised row not rounded before it is quantised.  Bound by memory: 2 bytes read and 1
// written per element in one pass.
template <int EL, bool LN, int T, int V>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const uint16_t* __restrict__ x, long ldx,
                                                            const uint16_t* __restrict__ gamma,
                                                            const uint16_t* __restrict__ beta, float eps,
                                                            int8_t* __restrict__ q, int ldq,
                                                            float* __restrict__ scale, long rows, int K) {
  __shared__ float red[4];
  const int t = threadIdx.x % T;
  const long row = blockIdx.x * (256L / T) + threadIdx.x / T;
  if (T == 64 && row >= rows) return;
  const uint16_t* xr = x + row * ldx;
  const int NV = K >> 3;
  float f[V][8];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int v = t + T * i;
    dec8<EL>(v < NV ? ld16(xr + 8 * v) : make_uint4(0, 0, 0, 0), f[i]);
  }
  if constexpr (LN) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) s += f[i][e];
    const float mean = row_reduce<T, false>(s, red) / (float)K;
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (t + T * i < NV) {
#pragma unroll
        for (int e = 0; e < 8; ++e) ss += (f[i][e] - mean) * (f[i][e] - mean);
      }
    const float rstd = rsqrtf(row_reduce<T, false>(ss, red) / (float)K + eps);
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (t + T * i < NV) {
        float g[8], b[8];
        dec8<EL>(ld16(gamma + 8 * (t + T * i)), g);
        dec8<EL>(ld16(beta + 8 * (t + T * i)), b);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[i][e] = (f[i][e] - mean) * rstd * g[e] + b[e];
      }
  }
  float a = 0.f;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      bad |= f[i][e] != f[i][e];
      a = fmaxf(a, fabsf(f[i][e]));
    }
  a = row_reduce<T, true>(bad ? INFINITY : a, red);
  float s, inv, up;
  quant_scale(a, s, inv, up);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int v = t + T * i;
    if (8 * v < ldq)
      *reinterpret_cast<uint2*>(q + row * ldq + 8 * v) =
          v < NV && inv != 0.f ? quant8(f[i], inv, up) : make_uint2(0u, 0u);
  }
  if (t == 0) scale[row] = s;
}

// Any K, alignment and length: one row per workgroup, read again for every pass (from the caches).
template <int EL, bool LN>
__global__ void __launch_bounds__(256) quantize_rows_any_kernel(const uint16_t* __restrict__ x, long ldx,
                                                                const uint16_t* __restrict__ gamma,
                                                                const uint16_t* __restrict__ beta, float eps,
                                                                int8_t* __restrict__ q, int ldq,
                                                                float* __restrict__ scale, int K) {
  __shared__ float red[4];
  const long row = blockIdx.x;
  const uint16_t* xr = x + row * ldx;
  float mean = 0.f, rstd = 1.f;
  if constexpr (LN) {
    float sum = 0.f, ss = 0.f;
    for (int k = threadIdx.x; k < K; k += 256) sum += dec16<EL>(xr[k]);
    mean = row_reduce<256, false>(sum, red) / (float)K;
    for (int k = threadIdx.x; k < K; k += 256) {
      const float d = dec16<EL>(xr[k]) - mean;
      ss += d * d;
    }
    rstd = rsqrtf(row_reduce<256, false>(ss, red) / (float)K + eps);
  }
  auto y = [&](int k) {
    const float v = dec16<EL>(xr[k]);
    return LN ? (v - mean) * rstd * dec16<EL>(gamma[k]) + dec16<EL>(beta[k]) : v;
  };
  float a = 0.f;
  bool bad = false;
  for (int k = threadIdx.x; k < K; k += 256) {
    const float f = y(k);
    bad |= f != f;
    a = fmaxf(a, fabsf(f));
  }
  a = row_reduce<256, true>(bad ? INFINITY : a, red);
  float s, inv, up;
  quant_scale(a, s, inv, up);
  for (int k = threadIdx.x; k < ldq; k += 256)
    q[row * ldq + k] = k < K && inv != 0.f ? (int8_t)quant_one(y(k) * up, inv) : 0;
  if (threadIdx.x == 0) scale[row] = s;
}

// ---------------------------------------------------------------------------------------------
struct LinArgs {
  const int8_t* x;       // [M, ldx] rows, zero from K to the next multiple of 16
  const int8_t* w;       // [N, ldw]
  const float* sx;
  const float* sw;
  const uint16_t* b;     // [N] or null
  const uint16_t* res;   // [M, N] or null
  uint16_t* y;           // [M, N] (N / 2 for geglu)
  long ldx, ldw;
  int M, N, K, act;
};

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

// 32x32x32 step of int8 products.  Lane l holds row / column l & 31 of A / B at k = 16 (l >> 5) .. + 15, and of the
// result column l & 31 at rows 8 (i >> 2) + 4 (l >> 5) + (i & 3), i = 0 .. 15.
__device__ __forceinline__ i32x16 mma_i8(uint4 a, uint4 b, i32x16 c) {
  return __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
}
// 16 bytes per lane straight into LDS (lane-linear from the wave-uniform lds) through a buffer resource over
// [base, base + nbytes): a lane whose offset lies past it writes zeros.
__device__ __forceinline__ void dma_i8(const int8_t* base, int nbytes, void* lds, unsigned off) {
  __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(base), 0, nbytes, 0x00020000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)lds, 16, off, 0, 0, 0);
}
template <int N>
__device__ __forceinline__ void wait_dma() {                      // at most N of this wave's loads still in flight
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | 0x70 | 0xF00);
}
template <int V>
struct Stage {
  static constexpr int value = V;
};

// Epilogue of one 32 (tokens) x 32 W (channels) strip of a wave: the fp32 results cross a wave-private LDS patch
// (a lane holds 4 channels of one token; the stores want runs of channels), then residual, activation
// and one rounding to the output type; 16 bytes per lane where N allows it.
template <int EL, int W>
__device__ __forceinline__ void store_strip(const LinArgs& p, const float* patch, int m0, int n0, int NO, int act) {
  constexpr int LD = 32 * W + 4;
  const int lane = threadIdx.x & 63;
  auto finish = [&](float y, long at) {
    if (p.res) y += dec16<EL>(p.res[at]);
    return act_f(y, act);
  };
  if (NO % 8 == 0) {
    constexpr int LPR = 4 * W;                                    // lanes per row, 8 channels each
#pragma unroll
    for (int it = 0; it < 32 * LPR / 64; ++it) {
      const int r = (it * 64 + lane) / LPR, c = (it * 64 + lane) % LPR * 8;
      if (m0 + r >= p.M || n0 + c >= NO) continue;
      const long at = (long)(m0 + r) * NO + n0 + c;
      float f[8];
      *reinterpret_cast<float4*>(f) = *reinterpret_cast<const float4*>(patch + r * LD + c);
      *reinterpret_cast<float4*>(f + 4) = *reinterpret_cast<const float4*>(patch + r * LD + c + 4);
      if (p.res) {
        float g[8];
        dec8<EL>(ld16(p.res + at), g);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] += g[e];
      }
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        w[e] = enc16<EL>(act_f(f[2 * e], act)) | (enc16<EL>(act_f(f[2 * e + 1], act)) << 16);
      st16(p.y + at, make_uint4(w[0], w[1], w[2], w[3]));
    }
  } else {
    for (int e = lane; e < 32 * 32 * W; e += 64) {
      const int r = e / (32 * W), c = e % (32 * W);
      if (m0 + r >= p.M || n0 + c >= NO) continue;
      const long at = (long)(m0 + r) * NO + n0 + c;
      p.y[at] = (uint16_t)enc16<EL>(finish(patch[r * LD + c], at));
    }
  }
}

// BM tokens x BN weight rows per workgroup, WM x WN waves, K in tiles of 128 bytes: both operands go straight to
// LDS (ring of NS stages, NS - 1 tiles in flight, counted waits, one barrier per tile), chunks XOR-swizzled
// by the row on the source address so that fragment reads touch every bank once.  W is the A operand: a
// lane's accumulators are 4 consecutive channels of one token.
// GLU: 32-row groups of the W tile alternate value rows and gate rows of the same channels, so both
// halves of an output meet in one lane.
template <int EL, bool GLU, int BM, int BN, int WM, int WN, int NS>
__global__ void __launch_bounds__(64 * WM * WN, 1) linear_int8_kernel(LinArgs p) {
  constexpr int NW = WM * WN, TM = BM / WM / 32, TN = BN / WN / 32;
  constexpr int XCH = BM / 8 / NW, WCH = BN / 8 / NW;             // DMA instructions per wave and tile (8 rows each)
  constexpr int LPT = XCH + WCH, STAGE = (BM + BN) * 128;
  constexpr int PW = GLU ? TN / 2 : TN;                           // 32-channel groups a wave puts out
  static_assert(XCH * 8 * NW == BM && WCH * 8 * NW == BN && (!GLU || TN % 2 == 0), "tile shape");
  static_assert(32 * (32 * PW + 4) * 4 * NW <= NS * STAGE, "patches fit the ring");
  __shared__ __attribute__((aligned(16))) int8_t ring[NS][STAGE];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN, col = lane & 31, half = lane >> 5;
  const int NO = GLU ? p.N / 2 : p.N;                             // output channels
  constexpr int BO = GLU ? BN / 2 : BN;                           // ... per workgroup
  // tile order: XCD-contiguous, in groups of 8 token tiles x all channel tiles (token tile fastest), so the
  // tiles in flight on an XCD share rows of both operands in its L2
  const int mt = (p.M + BM - 1) / BM, nt = (NO + BO - 1) / BO;
  const int lin = xcd_remap(blockIdx.x, mt * nt);
  const int grp = lin / (8 * nt), in = lin - grp * 8 * nt, gm = min(8, mt - 8 * grp);
  const int m0 = (8 * grp + in % gm) * BM, n0 = in / gm * BO;

  const int kp = (p.K + 15) & ~15;                                // bytes of a row that are loaded
  const int nk = (kp + 127) / 128;
  const int8_t* xb = p.x + (long)m0 * p.ldx;
  const int8_t* wb = GLU ? p.w : p.w + (long)n0 * p.ldw;
  const int xbytes = (int)min((long)min(BM, p.M - m0) * p.ldx, 0x7fffffffL);
  constexpr unsigned OOB = 0x80000000u;
  unsigned xo[XCH];
  int kc[XCH > WCH ? XCH : WCH];                                  // byte of the row a DMA lane starts at
#pragma unroll
  for (int i = 0; i < XCH; ++i) {
    const int r = 8 * (wave + NW * i) + (lane >> 3), c = (lane & 7) ^ ((r >> 1) & 7);
    xo[i] = m0 + r < p.M ? (unsigned)(r * (int)p.ldx + 16 * c) : OOB;
  }
  // W rows: 64-bit row starts for GLU (two far row groups), offsets in the tile otherwise
  unsigned wo[WCH];
  const int8_t* wrow[GLU ? WCH : 1];
#pragma unroll
  for (int i = 0; i < WCH; ++i) {
    const int r = 8 * (wave + NW * i) + (lane >> 3), c = (lane & 7) ^ ((r >> 1) & 7);
    if constexpr (GLU) {
      const int n = n0 + (r >> 6) * 32 + (r & 31);
      wo[i] = n < NO ? 16 * c : OOB;
      wrow[i] = nullptr;
    } else {
      wo[i] = n0 + r < NO ? (unsigned)(r * (int)p.ldw + 16 * c) : OOB;
    }
  }
#pragma unroll
  for (int i = 0; i < (XCH > WCH ? XCH : WCH); ++i) {
    const int r = 8 * (wave + NW * i) + (lane >> 3);
    kc[i] = 16 * ((lane & 7) ^ ((r >> 1) & 7));
  }
  (void)wrow;
  auto issue = [&](auto stage, int kt) __attribute__((always_inline)) {
    int8_t* dst = ring[decltype(stage)::value];
    const int k0 = 128 * kt;
    const bool tail = k0 + 128 > kp;
#pragma unroll
    for (int i = 0; i < XCH; ++i) {
      unsigned off = xo[i];
      if (tail && k0 + kc[i] >= kp) off = OOB;
      dma_i8(xb + k0, xbytes - k0, dst + 1024 * (wave + NW * i), off);
    }
#pragma unroll
    for (int i = 0; i < WCH; ++i) {
      unsigned off = wo[i];
      if (tail && k0 + kc[i] >= kp) off = OOB;
      if constexpr (GLU) {
        // the 8 rows of one DMA instruction lie in one group: a uniform base, rows ldw apart
        const int r = 8 * (wave + NW * i), n = n0 + (r >> 6) * 32 + (r & 31);
        const int8_t* base = p.w + (long)((r >> 5) & 1 ? NO + n : n) * p.ldw + k0;
        const int left = min(8, NO - n);
        if (off != OOB) off += (unsigned)((lane >> 3) * (int)p.ldw);
        dma_i8(base, left > 0 ? left * (int)p.ldw - k0 : 0, dst + BM * 128 + 1024 * (wave + NW * i), off);
      } else {
        dma_i8(wb + k0, (int)min((long)min(BN, NO - n0) * p.ldw, 0x7fffffffL) - k0,
               dst + BM * 128 + 1024 * (wave + NW * i), off);
      }
    }
  };

  i32x16 acc[TN][TM];
#pragma unroll
  for (int a = 0; a < TN; ++a)
#pragma unroll
    for (int b = 0; b < TM; ++b) acc[a][b] = (i32x16){};

  auto step = [&](auto stage, int kt) __attribute__((always_inline)) {
    constexpr int S = decltype(stage)::value;
    if (kt + NS - 2 < nk) wait_dma<(NS - 2) * LPT>();
    else wait_dma<0>();
    __builtin_amdgcn_s_barrier();                                 // tile kt is in LDS for every wave
    if (kt + NS - 1 < nk) issue(Stage<(S + NS - 1) % NS>(), kt + NS - 1);   // that stage was read at kt - 1
    const int8_t* sx = ring[S] + wm * (BM / WM) * 128;
    const int8_t* sw = ring[S] + (BM + wn * (BN / WN)) * 128;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      const int at = 128 * col + 16 * ((2 * ks + half) ^ ((col >> 1) & 7));
      uint4 af[TN], bf[TM];
#pragma unroll
      for (int a = 0; a < TN; ++a) af[a] = ld16(sw + 4096 * a + at);
#pragma unroll
      for (int b = 0; b < TM; ++b) bf[b] = ld16(sx + 4096 * b + at);
#pragma unroll
      for (int a = 0; a < TN; ++a)
#pragma unroll
        for (int b = 0; b < TM; ++b) acc[a][b] = mma_i8(af[a], bf[b], acc[a][b]);
    }
  };
  issue(Stage<0>(), 0);
  if (NS > 2 && 1 < nk) issue(Stage<1>(), 1);
  if (NS > 3 && 2 < nk) issue(Stage<2 % NS>(), 2);
  for (int kt = 0; kt < nk; kt += NS) {
    step(Stage<0>(), kt);
    if (kt + 1 < nk) step(Stage<1>(), kt + 1);
    if constexpr (NS > 2) {
      if (kt + 2 < nk) step(Stage<2 % NS>(), kt + 2);
    }
    if constexpr (NS > 3) {
      if (kt + 3 < nk) step(Stage<3 % NS>(), kt + 3);
    }
  }
  __syncthreads();                                                // the ring becomes the waves' patches

  float* patch = reinterpret_cast<float*>(&ring[0][0]) + wave * 32 * (32 * PW + 4);
  const int nw = n0 + wn * 32 * PW;                               // this wave's first output channel
#pragma unroll
  for (int b = 0; b < TM; ++b) {
    const int m = m0 + wm * (BM / WM) + 32 * b;
    const float sx = m + col < p.M ? p.sx[m + col] : 0.f;
#pragma unroll
    for (int g = 0; g < PW; ++g)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const int c = 32 * g + 2 * i + 4 * half;
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int n = min(nw + c + e, NO - 1);                  // channels past the last one are not stored
          y[e] = (float)acc[GLU ? 2 * g : g][b][i + e] * sx * p.sw[n];
          if (p.b) y[e] += dec16<EL>(p.b[n]);
          if constexpr (GLU) {
            float gate = (float)acc[2 * g + 1][b][i + e] * sx * p.sw[NO + n];
            if (p.b) gate += dec16<EL>(p.b[NO + n]);
            y[e] *= gelu_f(gate);
          }
        }
        *reinterpret_cast<float4*>(patch + col * (32 * PW + 4) + c) = make_float4(y[0], y[1], y[2], y[3]);
      }
    store_strip<EL, PW>(p, patch, m, nw, NO, GLU ? ACT_NONE : p.act);
  }
}

template <int EL, bool LN>
static void launch_quantize(const uint16_t* x, long ldx, const uint16_t* g, const uint16_t* b, float eps, int8_t* q,
                            int ldq, float* scale, long rows, int K, hipStream_t stream) {
  const bool vec = K % 8 == 0 && ldx % 8 == 0 && (size_t)x % 16 == 0 && (size_t)g % 16 == 0 && (size_t)b % 16 == 0;
  const int nv = (ldq + 7) / 8;                                   // vectors a row's threads write
#define QROWS(T, V)                                                                                            \
  quantize_rows_kernel<EL, LN, T, V><<<dim3((unsigned)((rows + 256 / T - 1) / (256 / T))), 256, 0, stream>>>(   \
      x, ldx, g, b, eps, q, ldq, scale, rows, K)
  if (!vec || nv > 2048)
    quantize_rows_any_kernel<EL, LN><<<dim3((unsigned)rows), 256, 0, stream>>>(x, ldx, g, b, eps, q, ldq, scale, K);
  else if (nv <= 64) QROWS(64, 1);
  else if (nv <= 128) QROWS(64, 2);
  else if (nv <= 256) QROWS(256, 1);
  else if (nv <= 512) QROWS(256, 2);
  else if (nv <= 1024) QROWS(256, 4);
  else QROWS(256, 8);
#undef QROWS
}

// x [rows, K] 16-bit (row stride ldx elements) -> q [rows, ldq] int8, scale [rows]; gamma / beta: LayerNorm first
ARB_API int arb_quantize_rows(const void* x, long ldx, const void* gamma, const void* beta, float eps, void* q, int ldq,
                              void* scale, long rows, int K, int el, hipStream_t stream) {
  if (rows <= 0 || rows > 0x7fffffffL || K <= 0 || ldq < K || ldq % 16 || ldq - K >= 16 ||
      (gamma == nullptr) != (beta == nullptr))
    return -1;
  const uint16_t *xp = (const uint16_t*)x, *g = (const uint16_t*)gamma, *b = (const uint16_t*)beta;
#define QUANT(EL, LN) \
  launch_quantize<EL, LN>(xp, ldx, g, b, eps, (int8_t*)q, ldq, (float*)scale, rows, K, stream)
  if (gamma) {
    if (el) QUANT(1, true); else QUANT(0, true);
  } else {
    if (el) QUANT(1, false); else QUANT(0, false);
  }
#undef QUANT
  return (int)hipGetLastError();
}

template <int EL, bool GLU, int BM, int BN, int WM, int WN, int NS>
static void launch_tiles(const LinArgs& p, hipStream_t s) {
  const int NO = GLU ? p.N / 2 : p.N, BO = GLU ? BN / 2 : BN;
  const long tiles = (long)((p.M + BM - 1) / BM) * ((NO + BO - 1) / BO);
  linear_int8_kernel<EL, GLU, BM, BN, WM, WN, NS><<<dim3((unsigned)tiles), 64 * WM * WN, 0, s>>>(p);
}

template <int EL, bool GLU>
static void launch_linear(const LinArgs& p, hipStream_t s) {
  auto tiles = [&](long bm, long bn) { return ((p.M + bm - 1) / bm) * ((p.N + bn - 1) / bn); };
  if (tiles(256, 256) >= 256) launch_tiles<EL, GLU, 256, 256, 2, 4, 2>(p, s);
  else if (tiles(128, 128) >= 256) launch_tiles<EL, GLU, 128, 128, 2, 2, 3>(p, s);
  else launch_tiles<EL, GLU, 64, 128, 2, 2, 4>(p, s);
}

ARB_API int arb_linear_int8(const void* x, long ldx, const void* sx, const void* w, long ldw, const void* sw,
                            const void* b, const void* res, void* y, int M, int N, int K, int act, int el,
                            hipStream_t stream) {
  const int kp = (K + 15) / 16 * 16;
  if (M <= 0 || N <= 0 || K <= 0 || K > 133000 || ldx < kp || ldw < kp || ldx % 16 || ldw % 16 || act < 0 || act > 3 ||
      (act == ACT_GEGLU && (N % 2 || res)))
    return -1;
  if (ldx >= (1L << 22) || ldw >= (1L << 22)) return -1;          // 31-bit byte offsets inside a tile
  LinArgs p{(const int8_t*)x, (const int8_t*)w, (const float*)sx, (const float*)sw, (const uint16_t*)b,
            (const uint16_t*)res, (uint16_t*)y, ldx, ldw, M, N, K, act};
  if (act == ACT_GEGLU) {
    if (el) launch_linear<1, true>(p, stream);
    else launch_linear<0, true>(p, stream);
  } else {
    if (el) launch_linear<1, false>(p, stream);
    else launch_linear<0, false>(p, stream);
  }
  return (int)hipGetLastError();
}
