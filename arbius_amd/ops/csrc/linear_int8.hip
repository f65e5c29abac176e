// Linears in 8-bit integers: rows quantised with one scale each, and their product with a weight held in
// 8 bits with one scale per output channel.
//
//   a_r = max_k |x_rk|,  s_r = a_r / 127,  q_rk = rne(127 x_rk / a_r)
//   y_mn = act( sx_m sw_n sum_k qx_mk qw_nk + b_n + r_mn )
//
// The sum is an integer (|sum| <= 128^2 K < 2^31 for every K the host accepts), so it is exact in any
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

// the activation of 8 values (uniform branch outside the loop)
__device__ __forceinline__ void act8(float (&y)[8], int act) {
  if (act == ACT_GELU) {
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = gelu_f(y[e]);
  } else if (act == ACT_QUICK_GELU) {
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] *= __builtin_amdgcn_rcpf(1.f + fast_exp(-1.702f * y[e]));
  }
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
// 8 elements from p (EW: at any element, else 16-byte aligned)
template <bool EW>
__device__ __forceinline__ uint4 ld8(const uint16_t* p) {
  if constexpr (!EW) return ld16(p);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = p[2 * i] | (uint32_t)p[2 * i + 1] << 16;
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// sum / maximum over the T threads that share a row (8 .. 64 lanes of a wave, or the block of 256); fixed order
template <int T, bool MAX>
__device__ __forceinline__ float row_reduce(float v, float* red) {
#pragma unroll
  for (int o = T < 64 ? T / 2 : 32; o > 0; o >>= 1) {
    const float u = __shfl_xor(v, o, 64);
    v = MAX ? fmaxf(v, u) : v + u;
  }
  if constexpr (T == 256) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = MAX ? fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])) : (red[0] + red[1]) + (red[2] + red[3]);
  }
  return v;
}

// A row on T threads, V vectors of 8 elements each (thread t: vectors t, t + T, ..; zeros behind the row): its values
// (LN: of LayerNorm in fp32, two exact passes over the registers, the normalised row not rounded before it is
// quantised), scale and reciprocal.
template <int EL, bool LN, int T, int V, bool EW = false>
__device__ __forceinline__ void row_values(const uint4 (&raw)[V], int t, int K, const uint16_t* __restrict__ gamma,
                                           const uint16_t* __restrict__ beta, float eps, float* red,
                                           float (&f)[V][8], float& s, float& inv, float& up) {
  const int NV = K >> 3;
#pragma unroll
  for (int i = 0; i < V; ++i) dec8<EL>(raw[i], f[i]);
  if constexpr (LN) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += f[i][e];
    const float mean = row_reduce<T, false>(sum, red) / (float)K;
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (t + T * i < NV) {
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(f[i][e] - mean, f[i][e] - mean, ss);
      }
    const float rstd = rsqrtf(row_reduce<T, false>(ss, red) / (float)K + eps);
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (t + T * i < NV) {
        float g[8], b[8];
        dec8<EL>(ld8<EW>(gamma + 8 * (t + T * i)), g);
        dec8<EL>(ld8<EW>(beta + 8 * (t + T * i)), b);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[i][e] = fmaf((f[i][e] - mean) * rstd, g[e], b[e]);
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
  quant_scale(row_reduce<T, true>(bad ? INFINITY : a, red), s, inv, up);
}

// One row per T threads: K <= 8 T V, K % 8 == 0, 16-byte aligned rows, gamma and beta (EW: at any element, read by
// elements - the order of LayerNorm's sums is K's, not the address's).  Bound by memory: 2 bytes read and 1 written
// per element in one pass (16384 x 8192 in 84 us, 4.8 TB/s; LayerNorm 65536 x 320 in 17 us, 3.7 TB/s; 1232 x 4096 in
// 4.6 us, where the launch counts).
template <int EL, bool LN, int T, int V, bool EW>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const uint16_t* __restrict__ x, long ldx,
                                                            const uint16_t* __restrict__ gamma,
                                                            const uint16_t* __restrict__ beta, float eps,
                                                            int8_t* __restrict__ q, int ldq,
                                                            float* __restrict__ scale, long rows, int K) {
  __shared__ float red[4];
  const int t = threadIdx.x % T;
  const long row = blockIdx.x * (256L / T) + threadIdx.x / T;
  if (T < 256 && row >= rows) return;
  const uint16_t* xr = x + row * ldx;
  const int NV = K >> 3;
  uint4 raw[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int v = t + T * i;
    raw[i] = v < NV ? ld8<EW>(xr + 8 * v) : make_uint4(0, 0, 0, 0);
  }
  float f[V][8], s, inv, up;
  row_values<EL, LN, T, V, EW>(raw, t, K, gamma, beta, eps, red, f, s, inv, up);
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
  bool vec;              // 16-byte accesses to y and res: N (N / 2) % 8 == 0, res aligned
};

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

// 32x32x32 step of int8 products.  Lane l holds row / column l & 31 of A / B at k = 16 (l >> 5) .. + 15, and of the
// result column l & 31 at rows 8 (i >> 2) + 4 (l >> 5) + (i & 3), i = 0 .. 15.
__device__ __forceinline__ i32x16 mma_i8(uint4 a, uint4 b, i32x16 c) {
  return __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
}
// 16 bytes per lane from base + off + k0 straight into LDS (lane-linear from the wave-uniform lds); a lane with
// off = kZeros writes zeros.  base and k0 are uniform: a load costs its own instruction and the LDS address.
constexpr unsigned kZeros = 0x80000000u;
__device__ __forceinline__ void dma_i8(const int8_t* base, void* lds, unsigned off, int k0) {
  __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(base), 0, 0x7fffffff, 0x00020000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)lds, 16, off, k0, 0, 0);
}
template <int N>
__device__ __forceinline__ void wait_dma() {                      // at most N of this wave's loads still in flight
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | 0x70 | 0xF00);
}
// Every LDS read of this wave has its data, then the workgroup meets: whoever refills a stage behind this barrier finds
// no read of it under way (a read's own wait may stand behind the barrier, in front of the product that uses it).
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_s_waitcnt(0xC07F);                             // lgkmcnt 0; DMA counted elsewhere
  __builtin_amdgcn_s_barrier();
}
template <int V>
struct Stage {
  static constexpr int value = V;
};
template <int S>
__device__ __forceinline__ int8_t* ring_of(int8_t* r0, int8_t* r1, int8_t* r2, int8_t* r3) {
  if constexpr (S == 0) return r0;
  else if constexpr (S == 1) return r1;
  else if constexpr (S == 2) return r2;
  else return r3;
}

// Scales and biases of a workgroup's tile.  They are read before the K loop (one row and one channel per thread, in
// registers meanwhile) and reach LDS after it: the epilogue waits for no memory.
template <int BM, int BN>
struct TileScales {
  float sx[BM], sw[BN], bias[BN];
};
template <int EL, int BM, int BN, int NT>
struct ScaleRegs {
  static constexpr int NX = (BM + NT - 1) / NT, NWR = (BN + NT - 1) / NT;
  float sx[NX], sw[NWR];
  uint16_t bias[NWR];
  // row(r): the weight row of row r of the W tile, -1 past the last one
  template <typename F>
  __device__ __forceinline__ void load(const LinArgs& p, int m0, F row) {
#pragma unroll
    for (int i = 0; i < NX; ++i) {
      const int m = m0 + (int)threadIdx.x + NT * i;
      sx[i] = p.sx ? p.sx[min(m, p.M - 1)] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < NWR; ++i) {
      const int n = max(0, row(min((int)threadIdx.x + NT * i, BN - 1)));
      sw[i] = p.sw[n];
      bias[i] = p.b ? p.b[n] : 0;
    }
  }
  __device__ __forceinline__ void store(TileScales<BM, BN>& t, bool tokens = true) const {
#pragma unroll
    for (int i = 0; i < NX; ++i)
      if (tokens && (int)threadIdx.x + NT * i < BM) t.sx[threadIdx.x + NT * i] = sx[i];
#pragma unroll
    for (int i = 0; i < NWR; ++i)
      if ((int)threadIdx.x + NT * i < BN) {
        t.sw[threadIdx.x + NT * i] = sw[i];
        t.bias[threadIdx.x + NT * i] = dec16<EL>(bias[i]);
      }
  }
};

// Two floats as two 16-bit values, rounded to nearest even (one instruction each pair)
template <int EL>
__device__ __forceinline__ uint32_t enc16x2(float a, float b) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  if constexpr (EL == 0) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, bf16x2));
  } else {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, f16x2));
  }
}

// A lane's 8 channels (GLU: and their gates), the same for every token it finishes.
template <bool GLU>
struct Lane8 {
  float sw[8], bias[8], gsw[GLU ? 8 : 1], gbias[GLU ? 8 : 1];
  template <int GATE>
  __device__ __forceinline__ void read(const float* s, const float* b) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      sw[e] = s[e];
      bias[e] = b[e];
      if constexpr (GLU) {
        gsw[e] = s[GATE + e];
        gbias[e] = b[GATE + e];
      }
    }
  }
};

// Channels n .. + 7 of token m: the KW partial sums of the patches, scales, bias, residual, activation, one
// rounding.  off: the values' place in a patch, their gates (GLU) GATE further on.
template <int EL, bool GLU, int KW, int GATE, bool VEC>
__device__ __forceinline__ void finish8(const LinArgs& p, const int* const (&patch)[KW], int off, float sx,
                                        const Lane8<GLU>& ch, int m, int n, int NO) {
  const uint16_t* __restrict__ res = p.res;
  uint16_t* __restrict__ y = p.y;
  auto sums = [&](int at, float (&f)[8]) {
    int t[8];
#pragma unroll
    for (int w = 0; w < KW; ++w) {
      const int4 u = *reinterpret_cast<const int4*>(patch[w] + off + at);
      const int4 v = *reinterpret_cast<const int4*>(patch[w] + off + at + 4);
      const int uv[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) t[e] = w ? t[e] + uv[e] : uv[e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = (float)t[e] * sx;
  };
  float f[8];
  sums(0, f);
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = fmaf(f[e], ch.sw[e], ch.bias[e]);
  if constexpr (GLU) {
    float g[8];
    sums(GATE, g);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] *= gelu_f(fmaf(g[e], ch.gsw[e], ch.gbias[e]));
  }
  if (m >= p.M) return;
  const long at = (long)m * NO + n;
  if constexpr (VEC) {
    if (n >= NO) return;
    if (res) {
      float g[8];
      dec8<EL>(ld16(res + at), g);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] += g[e];
    }
    if constexpr (!GLU) act8(f, p.act);
    st16(y + at, make_uint4(enc16x2<EL>(f[0], f[1]), enc16x2<EL>(f[2], f[3]), enc16x2<EL>(f[4], f[5]),
                            enc16x2<EL>(f[6], f[7])));
  } else {
    if (res) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (n + e < NO) f[e] += dec16<EL>(res[at + e]);
    }
    if constexpr (!GLU) act8(f, p.act);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (n + e < NO) y[at + e] = (uint16_t)enc16<EL>(f[e]);
  }
}

// Tile of workgroup `lin`: XCD-contiguous, in groups of 8 token tiles x all channel tiles (token tile fastest), so
// the tiles in flight on an XCD share rows of both operands in its L2.
__device__ __forceinline__ void tile_of(int mt, int nt, int& m, int& n) {
  const int lin = xcd_remap(blockIdx.x, mt * nt);
  const int grp = lin / (8 * nt), in = lin - grp * 8 * nt, gm = min(8, mt - 8 * grp);
  m = 8 * grp + in % gm;
  n = in / gm;
}

// A strip of 32 tokens x 32 TN weight rows as integers into a patch [32][32 TN + 4].
template <int TM, int TN>
__device__ __forceinline__ void put_strip(const i32x16 (&acc)[TN][TM], int b, int* patch) {
  const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
#pragma unroll
  for (int a = 0; a < TN; ++a)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const i32x16& x = acc[a][b];
      *reinterpret_cast<int4*>(patch + col * (32 * TN + 4) + 32 * a + 2 * i + 4 * half) =
          make_int4(x[i], x[i + 1], x[i + 2], x[i + 3]);
    }
}

// BM tokens x BN weight rows per workgroup, WM x WN waves, K in tiles of 128 bytes: both operands go straight to
// LDS (ring of NS stages, NS - 1 tiles in flight, counted waits, one barrier per tile), chunks XOR-swizzled
// by the row on the source address so that fragment reads touch every bank once.  W is the A operand: a
// lane's accumulators are 4 consecutive channels of one token; the epilogue takes them through an LDS
// patch, so that a lane stores (and loads residuals) 8 channels wide with their scales in registers.
// GLU: 32-row groups of the W tile alternate value rows and gate rows of the same channels, so both
// halves of an output meet in one lane.
// Bound by the matrix cores from 256 x 256 tiles on (16384 x 8192 x 8192: 928 - 955 us, 2300 - 2370 Top/s; a library
// product of that kind 2138), by LDS reads and the latency of a K step where a CU has one 64 x 128 tile
// (1232 x 4096 -> 1024: 14.1 - 15 us, 690 - 730 Top/s).
template <int EL, bool GLU, int BM, int BN, int WM, int WN, int NS>
__global__ void __launch_bounds__(64 * WM * WN, 1) linear_int8_kernel(LinArgs p) {
  constexpr int NW = WM * WN, TM = BM / WM / 32, TN = BN / WN / 32;
  constexpr int PRE = TM + TN <= 3 ? 4 : TM + TN <= 4 ? 2 : 1;    // K steps whose fragments are read together
  constexpr int XCH = BM / 8 / NW, WCH = BN / 8 / NW;             // DMA instructions per wave and tile (8 rows each)
  constexpr int LPT = XCH + WCH, STAGE = (BM + BN) * 128;
  static_assert(XCH * 8 * NW == BM && WCH * 8 * NW == BN && (!GLU || TN % 2 == 0), "tile shape");
  constexpr int LD = 32 * TN + 4, PATCH = 32 * LD;                // a wave's epilogue patch (ints)
  static_assert(PATCH * 4 * (NW / 2) <= STAGE, "half of the patches fit a ring stage");
  __shared__ TileScales<BM, BN> scales;
  // one __shared__ object per stage, each reached through compile-time stage numbers only: hipcc then knows that
  // reads of one stage do not depend on the loads into the others, and leaves those in flight
  __shared__ __attribute__((aligned(16))) int8_t ring0[STAGE];
  __shared__ __attribute__((aligned(16))) int8_t ring1[STAGE];
  __shared__ __attribute__((aligned(16))) int8_t ring2[NS > 2 ? STAGE : 16];
  __shared__ __attribute__((aligned(16))) int8_t ring3[NS > 3 ? STAGE : 16];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN, col = lane & 31, half = lane >> 5;
  const int NO = GLU ? p.N / 2 : p.N;                             // output channels
  constexpr int BO = GLU ? BN / 2 : BN;                           // ... per workgroup
  int m0, n0;
  tile_of((p.M + BM - 1) / BM, (NO + BO - 1) / BO, m0, n0);
  m0 *= BM;
  n0 *= BO;
  ScaleRegs<EL, BM, BN, 64 * NW> sr;
  sr.load(p, m0, [&](int r) {
    const int n = GLU ? n0 + (r >> 6) * 32 + (r & 31) : n0 + r;
    return n >= NO ? -1 : GLU && ((r >> 5) & 1) ? NO + n : n;
  });

  const int kp = (p.K + 15) & ~15;                                // bytes of a row that are loaded
  const int nk = (kp + 127) / 128;
  const int8_t* xb = p.x + (long)m0 * p.ldx;
  unsigned xo[XCH], wo[WCH];
  const int8_t* wb[WCH];                                          // uniform: an instruction's 8 rows are of one kind
  int kc[XCH > WCH ? XCH : WCH];                                  // byte of the K tile a lane starts at
#pragma unroll
  for (int i = 0; i < (XCH > WCH ? XCH : WCH); ++i) {
    const int r = 8 * (wave + NW * i) + (lane >> 3);
    kc[i] = 16 * ((lane & 7) ^ ((r >> 1) & 7));
  }
#pragma unroll
  for (int i = 0; i < XCH; ++i) {
    const int r = 8 * (wave + NW * i) + (lane >> 3);
    xo[i] = m0 + r < p.M ? (unsigned)(r * (int)p.ldx + kc[i]) : kZeros;
  }
#pragma unroll
  for (int i = 0; i < WCH; ++i) {
    const int r0 = 8 * (wave + NW * i), r = r0 + (lane >> 3);
    const int row = GLU ? (r >> 6) * 32 + (r & 31) : r;           // of the tile's value rows / gate rows
    wb[i] = p.w + ((GLU && ((r0 >> 5) & 1) ? NO : 0) + (long)n0) * p.ldw;
    wo[i] = n0 + row < NO ? (unsigned)(row * (int)p.ldw + kc[i]) : kZeros;
  }
  auto issue = [&](auto stage, int kt) __attribute__((always_inline)) {
    int8_t* dst = ring_of<decltype(stage)::value>(ring0, ring1, ring2, ring3);
    const int k0 = 128 * kt;
    if (k0 + 128 <= kp) {
#pragma unroll
      for (int i = 0; i < XCH; ++i) dma_i8(xb, dst + 1024 * (wave + NW * i), xo[i], k0);
#pragma unroll
      for (int i = 0; i < WCH; ++i) dma_i8(wb[i], dst + BM * 128 + 1024 * (wave + NW * i), wo[i], k0);
    } else {                                                      // the row ends inside the tile
#pragma unroll
      for (int i = 0; i < XCH; ++i)
        dma_i8(xb, dst + 1024 * (wave + NW * i), k0 + kc[i] < kp ? xo[i] : kZeros, k0);
#pragma unroll
      for (int i = 0; i < WCH; ++i)
        dma_i8(wb[i], dst + BM * 128 + 1024 * (wave + NW * i), k0 + kc[i] < kp ? wo[i] : kZeros, k0);
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
    const int8_t* st = ring_of<S>(ring0, ring1, ring2, ring3);
    const int8_t* sx = st + wm * (BM / WM) * 128;
    const int8_t* sw = st + (BM + wn * (BN / WN)) * 128;
    // Fragments are read PRE steps of 32 at a time, all before the products that use them (left to itself hipcc
    // puts every read right in front of its product and waits out the LDS latency four times a tile).
    uint4 af[2][PRE][TN], bf[2][PRE][TM];
    auto read = [&](int k) __attribute__((always_inline)) {
      const int at = 128 * col + 16 * ((2 * k + half) ^ ((col >> 1) & 7));
#pragma unroll
      for (int a = 0; a < TN; ++a) af[k / PRE & 1][k % PRE][a] = ld16(sw + 4096 * a + at);
#pragma unroll
      for (int b = 0; b < TM; ++b) bf[k / PRE & 1][k % PRE][b] = ld16(sx + 4096 * b + at);
    };
#pragma unroll
    for (int k = 0; k < PRE; ++k) read(k);
#pragma unroll
    for (int g = 0; g < 4 / PRE; ++g) {
      if (g + 1 < 4 / PRE) {
#pragma unroll
        for (int k = 0; k < PRE; ++k) read((g + 1) * PRE + k);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int k = 0; k < PRE; ++k)
#pragma unroll
        for (int a = 0; a < TN; ++a)
#pragma unroll
          for (int b = 0; b < TM; ++b) acc[a][b] = mma_i8(af[g & 1][k][a], bf[g & 1][k][b], acc[a][b]);
      __builtin_amdgcn_sched_barrier(0);
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
  sr.store(scales);
  __syncthreads();                                                // the ring becomes the waves' patches

  int* patch = reinterpret_cast<int*>(wave < NW / 2 ? ring0 : ring1) + wave % (NW / 2) * PATCH;
  const int* const patches[1] = {patch};
  constexpr int OW = GLU ? 16 * TN : 32 * TN, LPR = OW / 8, RPI = 64 / LPR;   // channels of a strip, lanes, rows
  const int c = lane % LPR * 8, pc = GLU ? c / 32 * 64 + c % 32 : c, n = n0 + wn * OW + c;
  Lane8<GLU> ch;
  ch.template read<32>(scales.sw + wn * 32 * TN + pc, scales.bias + wn * 32 * TN + pc);
  auto strips = [&](auto vec) __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < TM; ++b) {
      put_strip<TM, TN>(acc, b, patch);
#pragma unroll
      for (int it = 0; it < 32 / RPI; ++it) {
        const int r = it * RPI + lane / LPR, mr = wm * (BM / WM) + 32 * b + r;
        finish8<EL, GLU, 1, 32, decltype(vec)::value != 0>(p, patches, r * LD + pc, scales.sx[mr], ch, m0 + mr, n, NO);
      }
    }
  };
  if (p.vec) strips(Stage<1>());
  else strips(Stage<0>());
}

__device__ __forceinline__ uint4 load_i8(const int8_t* base, unsigned off, int k0) {
  __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(base), 0, 0x7fffffff, 0x00020000);
  return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(r, off, k0, 0));
}

// Few tokens (at most 16): 16 TN weight rows per workgroup, and its KW waves split K.  No LDS-DMA and no barrier in the
// loop: each wave keeps two K tiles of 128 bytes in flight in its own registers, a lane's 16 bytes being its
// 16x16x64 MFMA fragment as it lies in memory.  The integer partial sums of the waves meet in LDS.
// MR > 0 (at most MR tokens, K <= 8192): x comes in 16 bits and every workgroup quantises it for itself, into LDS,
// while its weights are on their way - a few KB from the L2 instead of a launch.  The quantisation is exact, so
// this gives the bits of quantize_rows.
// Bound by the read of the weight and the latency of one pass over it: 1 x 2048 -> 8192 in 7.1 us with the weight in
// memory, 2.4 TB/s, in 5.2 with it in the caches (quantisation launched apart: 8.8 and 6.5).  4 tokens: 8.9 (9.0), and
// one launch less for the host; more are quantised apart.
template <int EL, bool GLU, int TN, int KW, int MR>
__global__ void __launch_bounds__(64 * KW, 2) linear_int8_direct_kernel(LinArgs p, const uint16_t* __restrict__ x16,
                                                                        long ldx16) {
  constexpr int BM = 16, BN = 16 * TN, BO = GLU ? BN / 2 : BN, LD = BN + 4, NT = 64 * KW;
  constexpr int KMAX = 8192, QLD = KMAX + 16;                     // (16 bytes apart: rows start on other banks)
  static_assert(!GLU || TN % 2 == 0, "value and gate groups");
  static_assert(MR == 0 || KMAX / 8 <= 2 * NT, "two vectors a thread");
  __shared__ __attribute__((aligned(16))) int patch[KW][BM * LD];
  __shared__ __attribute__((aligned(16))) int8_t sq[MR ? MR * QLD : 16];
  __shared__ float sred[MR ? MR : 1][KW];
  __shared__ TileScales<BM, BN> scales;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r16 = lane & 15, g = lane >> 4;
  const int NO = GLU ? p.N / 2 : p.N;
  const int n0 = xcd_remap(blockIdx.x, (NO + BO - 1) / BO) * BO;
  const int kp = (p.K + 15) & ~15, nk = (kp + 127) / 128;

  uint4 xv[MR ? MR : 1][2];
  if constexpr (MR > 0) {                                         // before the weights: loads return in order
#pragma unroll
    for (int r = 0; r < MR; ++r)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int v = tid + NT * j;
        xv[r][j] = 8 * v < p.K ? ld16(x16 + min(r, p.M - 1) * ldx16 + 8 * v) : make_uint4(0, 0, 0, 0);
      }
  }
  // rows past the last one repeat it: their results are not stored.  GLU: 16-row groups alternate values and gates
  const unsigned xo = MR ? 0u : (unsigned)(min(r16, p.M - 1) * (int)p.ldx + 16 * g);
  unsigned wo[TN];
#pragma unroll
  for (int a = 0; a < TN; ++a) {
    const int r = GLU ? 16 * (a >> 1) + r16 : 16 * a + r16;
    wo[a] = (unsigned)(min(r, NO - 1 - n0) * (int)p.ldw + 16 * g);
  }
  const int8_t* wb = p.w + (long)n0 * p.ldw;
  const int8_t* gb = GLU ? wb + (long)NO * p.ldw : wb;

  uint4 xf[2][2], wf[2][2][TN];
  auto load = [&](auto buf, int kt) __attribute__((always_inline)) {
    constexpr int B = decltype(buf)::value;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int k0 = 128 * kt + 64 * s;
      const unsigned past = k0 + 16 * g < kp ? 0u : kZeros;       // chunks behind the row
#pragma unroll
      for (int a = 0; a < TN; ++a) wf[B][s][a] = load_i8(GLU && (a & 1) ? gb : wb, wo[a] | past, k0);
      if constexpr (MR == 0) xf[B][s] = load_i8(p.x, xo | past, k0);
    }
  };
  if (wave < nk) load(Stage<0>(), wave);
  if (wave + KW < nk) load(Stage<1>(), wave + KW);
  ScaleRegs<EL, BM, BN, NT> sr;
  sr.load(p, 0, [&](int r) {
    const int n = GLU ? n0 + (r >> 5) * 16 + (r & 15) : n0 + r;
    return n >= NO ? -1 : GLU && ((r >> 4) & 1) ? NO + n : n;
  });
  if constexpr (MR > 0) {
#pragma unroll
    for (int r = 0; r < MR; ++r) {
      float a = 0.f;
      bool bad = false;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float f[8];
        dec8<EL>(xv[r][j], f);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          bad |= f[e] != f[e];
          a = fmaxf(a, fabsf(f[e]));
        }
      }
      a = wave_max(bad ? INFINITY : a);
      if (lane == 0) sred[r][wave] = a;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < MR; ++r) {
      float a = sred[r][0];
#pragma unroll
      for (int w = 1; w < KW; ++w) a = fmaxf(a, sred[r][w]);
      float s, inv, up;
      quant_scale(a, s, inv, up);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int v = tid + NT * j;
        if (8 * v < 128 * nk) {                                   // zeros to the end of the last K tile
          float f[8];
          dec8<EL>(xv[r][j], f);
          *reinterpret_cast<uint2*>(sq + r * QLD + 8 * v) = inv != 0.f ? quant8(f, inv, up) : make_uint2(0u, 0u);
        }
      }
      if (tid == 0) scales.sx[r] = s;
    }
    __syncthreads();
  }
  i32x4 acc[TN];
#pragma unroll
  for (int a = 0; a < TN; ++a) acc[a] = (i32x4){};
  auto mma = [&](auto buf, int kt) __attribute__((always_inline)) {
    constexpr int B = decltype(buf)::value;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      if constexpr (MR > 0) xf[B][s] = ld16(sq + min(r16, MR - 1) * QLD + 128 * kt + 64 * s + 16 * g);
#pragma unroll
      for (int a = 0; a < TN; ++a)
        acc[a] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, wf[B][s][a]),
                                                       __builtin_bit_cast(i32x4, xf[B][s]), acc[a], 0, 0, 0);
    }
  };
  for (int kt = wave; kt < nk; kt += 2 * KW) {
    mma(Stage<0>(), kt);
    if (kt + 2 * KW < nk) load(Stage<0>(), kt + 2 * KW);
    if (kt + KW < nk) {
      mma(Stage<1>(), kt + KW);
      if (kt + 3 * KW < nk) load(Stage<1>(), kt + 3 * KW);
    }
  }
  // result column lane & 15 (token), rows 4 (lane >> 4) .. + 3 (channels)
#pragma unroll
  for (int a = 0; a < TN; ++a) *reinterpret_cast<i32x4*>(&patch[wave][r16 * LD + 16 * a + 4 * g]) = acc[a];
  sr.store(scales, MR == 0);
  __syncthreads();
  const int* patches[KW];
#pragma unroll
  for (int w = 0; w < KW; ++w) patches[w] = patch[w];
  constexpr int LPR = BO / 8;
  for (int e = tid; e < BM * LPR; e += NT) {
    const int r = e / LPR, c = e % LPR * 8, pc = GLU ? c / 16 * 32 + c % 16 : c;
    if (r >= p.M) break;
    Lane8<GLU> ch;
    ch.template read<16>(scales.sw + pc, scales.bias + pc);
    if (p.vec) finish8<EL, GLU, KW, 16, true>(p, patches, r * LD + pc, scales.sx[r], ch, r, n0 + c, NO);
    else finish8<EL, GLU, KW, 16, false>(p, patches, r * LD + pc, scales.sx[r], ch, r, n0 + c, NO);
  }
}

// Short rows (K <= 32 KS), many of them: LayerNorm, quantisation and product in one kernel, x read once and never
// written in 8 bits.  A wave owns 32 tokens: it quantises them as quantize_rows_kernel does (the same lanes per row,
// the same bits), 64 / T rows at a time, through LDS into the B operand's layout, and their fragments stay in
// registers while the workgroup walks its weight rows, 64 at a time (GLU: 32 values and their 32 gates), through two
// LDS stages.  A token's scale is a register of its lanes, so the epilogue runs in the accumulators' layout and only
// the finished 16-bit channels cross lanes (LDS patch) for 16-byte stores.
// Bound by the VALU (quantisation, scales, GELU) next to the write of y: LayerNorm 65536 x 320 -> 960 in 48 - 49
// us with x and y's memory in the 256 MB cache (3.5 TB/s of them; quantised apart 69), 57 with x from memory, 61 - 68
// with new memory for y too; 16384 x 640 -> 5120 geglu in 84 - 86 us launch behind launch, 91 - 94 alone (apart 106).
template <int EL, bool GLU, bool LN, int KS, int NW>
__global__ void __launch_bounds__(64 * NW, 2) linear_int8_rows_kernel(LinArgs p, const uint16_t* __restrict__ x16,
                                                                      long ldx16, const uint16_t* __restrict__ gamma,
                                                                      const uint16_t* __restrict__ beta, float eps,
                                                                      int splits) {
  constexpr int BM = 32 * NW, OW = GLU ? 32 : 64, STAGE = KS * 32 * 64, NDMA = 2 * KS / NW, PR = OW + 8;
  constexpr int LPR = OW / 8, RPI = 64 / LPR, NST = 32 / RPI;     // stores: lanes per row, rows each, per chunk
  static_assert(NW % 4 == 0 && 2 * KS % NW == 0, "one row group per wave");
  __shared__ __attribute__((aligned(16))) int8_t st0[STAGE];
  __shared__ __attribute__((aligned(16))) int8_t st1[STAGE];
  __shared__ __attribute__((aligned(16))) uint16_t patch[NW][32 * PR];
  __shared__ __attribute__((aligned(16))) float schan[NW][2][64];
  __shared__ float stok[NW][32];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int NO = GLU ? p.N / 2 : p.N, chunks = (NO + OW - 1) / OW;
  const int lin = xcd_remap(blockIdx.x, (p.M + BM - 1) / BM * splits), rt = lin / splits, sp = lin - rt * splits;
  const int per = (chunks + splits - 1) / splits, c0 = min(chunks, sp * per), c1 = min(chunks, c0 + per);
  const int m0 = rt * BM + 32 * wave, m = m0 + col;
  const int kp = (p.K + 15) & ~15;

  // weight stage: 64-byte K tiles of 64 rows, 16-byte chunks XOR-swizzled by the row; instruction q = wave + NW i
  // fills rows 16 (q & 3) .. + 15 of K tile q >> 2
  const int wrow = 16 * (wave & 3) + (lane >> 2), kc = 16 * ((lane & 3) ^ ((wrow >> 2) & 3));
  const bool gate = GLU && (wave & 2);
  const int orow = gate ? wrow - 32 : wrow;                       // of the chunk's value / gate rows
  auto issue = [&](int c, int8_t* dst) __attribute__((always_inline)) {
    const int8_t* base = p.w + ((gate ? NO : 0) + (long)c * OW) * p.ldw;
    const unsigned off = c * OW + orow < NO ? (unsigned)(orow * (int)p.ldw + kc) : kZeros;
#pragma unroll
    for (int i = 0; i < NDMA; ++i) {
      const int k0 = 64 * ((wave >> 2) + NW / 4 * i);
      dma_i8(base, dst + 1024 * (wave + NW * i), k0 + kc < kp ? off : kZeros, k0);
    }
  };
  // channel `lane` of a chunk (GLU: values, then gates): read a chunk ahead
  float csw = 0.f;
  uint32_t cb = 0;
  auto channels = [&](int c) __attribute__((always_inline)) {
    const int n = min(c * OW + (GLU ? col : lane), NO - 1), row = GLU && half ? NO + n : n;
    csw = p.sw[row];
    cb = p.b ? p.b[row] : 0;
  };

  if (c0 >= c1) return;
  // ---- the wave's tokens, RP rows at a time through its part of the weight stages
  constexpr int T = KS == 10 ? 8 : 16, V = 5, RI = 64 / T, RP = 2 * STAGE / NW / (32 * KS), SWZ = KS == 10 ? 3 : 7;
  static_assert(8 * T * V == 32 * KS && RP * NW * 32 * KS == 2 * STAGE && 32 % RP == 0 && RP % RI == 0, "passes");
  int8_t* const mine = (wave < NW / 2 ? st0 : st1) + wave % (NW / 2) * (RP * 32 * KS);
  const int t = lane % T, NV = p.K >> 3;
  auto fetch = [&](int r, uint4 (&raw)[V]) __attribute__((always_inline)) {   // row r of the wave's 32
    const uint16_t* xr = x16 + (long)min(m0 + r, p.M - 1) * ldx16;
#pragma unroll
    for (int i = 0; i < V; ++i) raw[i] = t + T * i < NV ? ld16(xr + 8 * (t + T * i)) : make_uint4(0, 0, 0, 0);
  };
  auto swz = [](int r) { return SWZ == 3 ? (r >> 2) & 3 : (r >> 1) & 7; };   // 16-byte units of a staged row, by bank
  uint4 xq[KS], raw[V];
  fetch(lane / T, raw);
#pragma unroll
  for (int pass = 0; pass < 32 / RP; ++pass) {
#pragma unroll 1
    for (int it = 0; it < RP / RI; ++it) {
      const int r = it * RI + lane / T, next = pass * RP + r + RI;
      uint4 now[V];
#pragma unroll
      for (int i = 0; i < V; ++i) now[i] = raw[i];
      if (next < 32) fetch(next, raw);
      float f[V][8], s, inv, up;
      row_values<EL, LN, T, V>(now, t, p.K, gamma, beta, eps, nullptr, f, s, inv, up);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int v = t + T * i;
        *reinterpret_cast<uint2*>(mine + r * (32 * KS) + 16 * ((v >> 1) ^ swz(r)) + 8 * (v & 1)) =
            v < NV && inv != 0.f ? quant8(f[i], inv, up) : make_uint2(0u, 0u);
      }
      if (t == 0) stok[wave][pass * RP + r] = s;
    }
    if (RP == 32 || col / RP == pass) {
      const int r = col % RP;
#pragma unroll
      for (int s = 0; s < KS; ++s) xq[s] = ld16(mine + r * (32 * KS) + 16 * ((2 * s + half) ^ swz(r)));
    }
  }
  const float sx = stok[wave][col];
  __syncthreads();                                                // the stages are the weight's from here on

  // ---- the workgroup's weight rows
  const int sw0 = col * 64 + 16 * (half ^ ((col >> 2) & 3)), sw1 = col * 64 + 16 * ((2 + half) ^ ((col >> 2) & 3));
  uint16_t* const pt = patch[wave];
  float* const sc = schan[wave][0];
  auto put_channels = [&]() __attribute__((always_inline)) {      // (a wave's own LDS: in order, no barrier)
    sc[lane] = csw;
    sc[64 + lane] = dec16<EL>(cb);
  };
  auto product = [&](const int8_t* st, i32x16 (&acc)[2]) __attribute__((always_inline)) {
    acc[0] = acc[1] = (i32x16){};
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int t = 0; t < 2; ++t)
        acc[t] = mma_i8(ld16(st + 4096 * (s >> 1) + 2048 * t + (s & 1 ? sw1 : sw0)), xq[s], acc[t]);
  };
  auto finish = [&](int c, const i32x16 (&acc)[2], auto plain) __attribute__((always_inline)) {
    const int n0 = c * OW;
#pragma unroll
    for (int t = 0; t < (GLU ? 1 : 2); ++t)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const int ch = 32 * t + 2 * i + 4 * half;                 // channels ch .. + 3 of the chunk
        const f32x4 w = *reinterpret_cast<const f32x4*>(sc + ch), b = *reinterpret_cast<const f32x4*>(sc + 64 + ch);
        float f[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = fmaf((float)acc[t][i + e] * sx, w[e], b[e]);
        if constexpr (GLU) {
          const f32x4 gw = *reinterpret_cast<const f32x4*>(sc + 32 + ch);
          const f32x4 gb = *reinterpret_cast<const f32x4*>(sc + 96 + ch);
#pragma unroll
          for (int e = 0; e < 4; ++e) f[e] *= gelu_f(fmaf((float)acc[1][i + e] * sx, gw[e], gb[e]));
        } else if constexpr (decltype(plain)::value == 0) {
          if (p.res && m < p.M && n0 + ch < NO) {
            const uint2 r = *reinterpret_cast<const uint2*>(p.res + (long)m * NO + n0 + ch);
            f[0] += dec16<EL>(r.x & 0xffffu);
            f[1] += dec16<EL>(r.x >> 16);
            f[2] += dec16<EL>(r.y & 0xffffu);
            f[3] += dec16<EL>(r.y >> 16);
          }
          if (p.act == ACT_GELU) {
#pragma unroll
            for (int e = 0; e < 4; ++e) f[e] = gelu_f(f[e]);
          } else if (p.act == ACT_QUICK_GELU) {
#pragma unroll
            for (int e = 0; e < 4; ++e) f[e] *= __builtin_amdgcn_rcpf(1.f + fast_exp(-1.702f * f[e]));
          }
        }
        *reinterpret_cast<uint2*>(pt + col * PR + ch) = make_uint2(enc16x2<EL>(f[0], f[1]), enc16x2<EL>(f[2], f[3]));
      }
    if constexpr (decltype(plain)::value == 1) {                  // fragments four ahead, a product, some epilogue
      __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
      for (int i = 0; i < 2 * KS; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, GLU ? 320 / (2 * KS) : 120 / (2 * KS), 0);
      }
    }
    put_channels();                                               // the next chunk's: does not wait for the stores
    const int r = lane / LPR, cc = lane % LPR * 8;
    uint16_t* y = p.y + (long)(m0 + r) * NO + n0 + cc;
    if (m0 + 32 <= p.M && n0 + OW <= NO) {                        // uniform
      uint4 v[NST];
#pragma unroll
      for (int i = 0; i < NST; ++i) v[i] = ld16(pt + (r + RPI * i) * PR + cc);
#pragma unroll
      for (int i = 0; i < NST; ++i) st16(y + (long)RPI * i * NO, v[i]);
      asm volatile("" ::: "memory");
      wait_dma<NST>();                                            // all but these stores: the other stage has arrived
    } else {
#pragma unroll
      for (int i = 0; i < NST; ++i)
        if (m0 + r + RPI * i < p.M && n0 + cc < NO) st16(y + (long)RPI * i * NO, ld16(pt + (r + RPI * i) * PR + cc));
      asm volatile("" ::: "memory");
      wait_dma<0>();
    }
  };
  issue(c0, st0);
  channels(c0);
  put_channels();
  wait_dma<0>();
  lds_barrier();
  if constexpr (KS == 10) {
    // Chunk c's product next to chunk c - 1's epilogue, so that matrix cores and VALU work side by side (65536 x 320
    // -> 960 behind a LayerNorm 54.8 -> 49.9 us; at KS 20, with twice the fragments to hold, it is a tenth slower)
    auto step = [&](int c, const int8_t* st, int8_t* other, i32x16 (&acc)[2], const i32x16 (&last)[2])
                    __attribute__((always_inline)) {
      if (c + 1 < c1) issue(c + 1, other);
      channels(c);
      product(st, acc);
      if (GLU || (!p.res && p.act == ACT_NONE)) finish(c - 1, last, Stage<1>());
      else finish(c - 1, last, Stage<0>());
      lds_barrier();
    };
    i32x16 acc0[2], acc1[2];
    if (c0 + 1 < c1) issue(c0 + 1, st1);
    product(st0, acc0);
    wait_dma<0>();
    lds_barrier();
    for (int c = c0 + 1; c < c1; c += 2) {
      step(c, st1, st0, acc1, acc0);
      if (c + 1 >= c1) {
        acc0[0] = acc1[0];
        acc0[1] = acc1[1];
        break;
      }
      step(c + 1, st0, st1, acc0, acc1);
    }
    finish(c1 - 1, acc0, Stage<0>());
  } else {
    i32x16 acc[2];
    for (int c = c0; c < c1; c += 2) {
      if (c + 1 < c1) {
        issue(c + 1, st1);
        channels(c + 1);
      }
      product(st0, acc);
      finish(c, acc, Stage<0>());
      lds_barrier();
      if (c + 1 >= c1) break;
      if (c + 2 < c1) {
        issue(c + 2, st0);
        channels(c + 2);
      }
      product(st1, acc);
      finish(c + 1, acc, Stage<0>());
      lds_barrier();
    }
  }
}

template <int EL, bool LN>
static int launch_quantize(const uint16_t* x, long ldx, const uint16_t* g, const uint16_t* b, float eps, int8_t* q,
                            int ldq, float* scale, long rows, int K, hipStream_t stream) {
  const bool vec = K % 8 == 0 && ldx % 8 == 0 && (size_t)x % 16 == 0 && (size_t)g % 16 == 0 && (size_t)b % 16 == 0;
  const int nv = (ldq + 7) / 8;                                   // vectors a row's threads write
#define QROWS(T, V)                                                                                              \
  do {                                                                                                           \
    const dim3 grid((unsigned)((rows + 256 / T - 1) / (256 / T)));                                               \
    if (vec) quantize_rows_kernel<EL, LN, T, V, false><<<grid, 256, 0, stream>>>(x, ldx, g, b, eps, q, ldq, scale, \
                                                                                 rows, K);                       \
    else quantize_rows_kernel<EL, LN, T, V, LN><<<grid, 256, 0, stream>>>(x, ldx, g, b, eps, q, ldq, scale, rows, \
                                                                          K);                                    \
  } while (0)
  // Lanes per row.  LN: by K alone (its sums' order must not depend on the rows of the batch, nor on where they lie),
  // about 5 vectors a lane.  Without LN every choice gives the same bits: few rows are spread over whole workgroups.
  const bool few = !LN && rows < 4096, any = !(vec || (LN && K % 8 == 0)) || nv > 2048;
  // a launch has fewer than 2^32 threads
  if (rows * (any || nv > 320 ? 256 : nv > 160 ? 64 : nv > 80 ? 32 : nv > 40 ? 16 : 8) >= (1L << 32) - 256) return -1;
  if (any) {
    quantize_rows_any_kernel<EL, LN><<<dim3((unsigned)rows), 256, 0, stream>>>(x, ldx, g, b, eps, q, ldq, scale, K);
  } else if (few && nv <= 256) {
    if constexpr (!LN) {
      if (nv <= 64) QROWS(64, 1);
      else QROWS(256, 1);
    }
  } else if (nv <= 40) {
    QROWS(8, 5);
  } else if (nv <= 80) {
    QROWS(16, 5);
  } else if (nv <= 160) {
    QROWS(32, 5);
  } else if (nv <= 320 && !few) {
    QROWS(64, 5);
  } else if (nv <= 512) {
    QROWS(256, 2);
  } else if (nv <= 1024) {
    QROWS(256, 4);
  } else {
    QROWS(256, 8);
  }
#undef QROWS
  return (int)hipGetLastError();
}

// x [rows, K] 16-bit (row stride ldx elements) -> q [rows, ldq] int8, scale [rows]; gamma / beta: LayerNorm first
ARB_API int arb_quantize_rows(const void* x, long ldx, const void* gamma, const void* beta, float eps, void* q, int ldq,
                              void* scale, long rows, int K, int el, hipStream_t stream) {
  if (rows <= 0 || rows > 0x7fffffffL || K <= 0 || ldq < K || ldq % 16 || ldq - K >= 16 ||
      (gamma == nullptr) != (beta == nullptr))
    return -1;
  const uint16_t *xp = (const uint16_t*)x, *g = (const uint16_t*)gamma, *b = (const uint16_t*)beta;
#define QUANT(EL, LN) \
  return launch_quantize<EL, LN>(xp, ldx, g, b, eps, (int8_t*)q, ldq, (float*)scale, rows, K, stream)
  if (gamma) {
    if (el) QUANT(1, true); else QUANT(0, true);
  } else {
    if (el) QUANT(1, false); else QUANT(0, false);
  }
#undef QUANT
}

template <int EL, bool GLU, int MR>
static int launch_direct(const LinArgs& p, hipStream_t s, const uint16_t* x16 = nullptr, long ldx16 = 0) {
  const int NO = GLU ? p.N / 2 : p.N, BO = GLU ? 16 : 32;
  if (NO >= 1 << 26) return -1;                                   // a launch has fewer than 2^32 threads
  linear_int8_direct_kernel<EL, GLU, 2, 8, MR><<<dim3((unsigned)((NO + BO - 1) / BO)), 512, 0, s>>>(p, x16, ldx16);
  return (int)hipGetLastError();
}

template <int EL, bool GLU, int BM, int BN, int WM, int WN, int NS>
static int launch_tiles(const LinArgs& p, hipStream_t s) {
  const int NO = GLU ? p.N / 2 : p.N, BO = GLU ? BN / 2 : BN;
  const long tiles = ((p.M + BM - 1L) / BM) * ((NO + BO - 1L) / BO);
  if (tiles * 64 * WM * WN >= (1L << 32)) return -1;              // a launch has fewer threads
  linear_int8_kernel<EL, GLU, BM, BN, WM, WN, NS><<<dim3((unsigned)tiles), 64 * WM * WN, 0, s>>>(p);
  return (int)hipGetLastError();
}

// Kernel by size (the sums are exact: every choice gives the same bits).  Measured, us, the product alone:
//                              256x256  64x128 ring 2  64x128 ring 4  direct 16x32
//   16384 x 8192 x 8192            918           1337           1544         10676
//   65536 x 320 -> 960            49.9           57.5           97.7           287
//   4096 x 1280 -> 1280           21.5           14.7           18.2          74.1
//   1232 x 4096 -> 1024           47.1           20.2           14.0          55.3
//   162 x 2048 -> 6144            26.7           11.9            8.5          27.8
//   1 x 2048 -> 8192              24.9           11.8            8.6           6.2
// 256 x 256 from one tile per CU on; below, 64 x 128 with two stages while two and more workgroups share a CU
// and hide each other's latency, with four where a CU has one; up to 16 tokens the weight alone counts.
template <int EL, bool GLU>
static int launch_linear(const LinArgs& p, hipStream_t s) {
  auto tiles = [&](long bm, long bn) { return ((p.M + bm - 1) / bm) * ((p.N + bn - 1) / bn); };
  constexpr int WN = GLU ? 2 : 4;                                 // value and gate groups share a wave
  if (p.M <= 16) return launch_direct<EL, GLU, 0>(p, s);
  if (tiles(256, 256) >= 256) return launch_tiles<EL, GLU, 256, 256, 2, 4, 2>(p, s);
  if (tiles(64, 128) >= 512) return launch_tiles<EL, GLU, 64, 128, 2, WN, 2>(p, s);
  return launch_tiles<EL, GLU, 64, 128, 2, WN, 4>(p, s);
}

template <int EL, bool GLU, bool LN>
static int launch_rows(const LinArgs& p, const uint16_t* x, long ldx, const uint16_t* g, const uint16_t* b, float eps,
                       hipStream_t s) {
  const bool wide = p.K > 320;
  const int chunks = GLU ? (p.N / 2 + 31) / 32 : (p.N + 63) / 64, bm = wide ? 256 : 128;
  const long tiles = (p.M + bm - 1L) / bm;
  const int splits = (int)max(1L, min((wide ? 256 : 512) / tiles, (long)chunks));
  if (tiles * splits * 2 * bm >= (1L << 32)) return -1;           // a launch has fewer threads
  const dim3 grid((unsigned)(tiles * splits));
  if (wide) linear_int8_rows_kernel<EL, GLU, LN, 20, 8><<<grid, 512, 0, s>>>(p, x, ldx, g, b, eps, splits);
  else linear_int8_rows_kernel<EL, GLU, LN, 10, 4><<<grid, 256, 0, s>>>(p, x, ldx, g, b, eps, splits);
  return (int)hipGetLastError();
}

// Whether a product of 16-bit rows without LayerNorm quantises them itself: up to 4 tokens.  (Behind a LayerNorm the
// sums would run in another order than for longer batches.)
ARB_API int arb_linear_int8_few(const void* x, long ldx, int M, int K) {
  return M <= 4 && K <= 8192 && K % 8 == 0 && ldx % 8 == 0 && (size_t)x % 16 == 0;
}

// sx != null: x int8 rows (stride ldx bytes) with scales sx.  sx null: x 16-bit rows (stride ldx elements), which are
// quantised (gamma / beta: LayerNorm first) into ws - M rows of K rounded up to 16 bytes, then M scales (unused, may be
// null, where arb_linear_int8_few says 1).
ARB_API int arb_linear_int8(const void* x, long ldx, const void* sx, const void* gamma, const void* beta, float eps,
                            void* ws, const void* w, long ldw, const void* sw, const void* b, const void* res,
                            void* y, int M, int N, int K, int act, int el, hipStream_t stream) {
  const int kp = (K + 15) / 16 * 16;
  if (M <= 0 || N <= 0 || K <= 0 || K > 131071 || ldw < kp || ldw % 16 || act < 0 || act > 3 ||
      (act == ACT_GEGLU && (N % 2 || res)))
    return -1;
  LinArgs p{(const int8_t*)x, (const int8_t*)w, (const float*)sx, (const float*)sw, (const uint16_t*)b,
            (const uint16_t*)res, (uint16_t*)y, ldx, ldw, M, N, K, act,
            (act == ACT_GEGLU ? N / 2 : N) % 8 == 0 && (size_t)res % 16 == 0 && (size_t)y % 16 == 0};
  if (ldw >= (1L << 22)) return -1;                               // 31-bit offsets in a tile
  if (sx == nullptr && !gamma && arb_linear_int8_few(x, ldx, M, K)) {
    const uint16_t* x16 = (const uint16_t*)x;
#define FEW(EL, GLU) \
  return M == 1 ? launch_direct<EL, GLU, 1>(p, stream, x16, ldx) : launch_direct<EL, GLU, 4>(p, stream, x16, ldx)
    if (act == ACT_GEGLU) {
      if (el) FEW(1, true); else FEW(0, true);
    } else {
      if (el) FEW(1, false); else FEW(0, false);
    }
#undef FEW
  }
  // Many short rows: one kernel.  Measured against the quantisation and the product apart, us:
  //                       8192 rows   16384   32768   65536
  //   320 -> 2560 geglu   28.6/36.4 43.3/54.6 71.8/92.1 124/173      640 -> 5120 geglu  52.6/64.0 87.7/106 156/200
  //   320 -> 1280 gelu          -   36.9/49.8 58.8/76.5 100/128      512 -> 2048 gelu          -  56.4/57.4 95.2/105
  //   320 -> 960 (LN)           -   25.9/23.9 33.1/39.7 49.9/69.1    640 -> 1920               -  44.3/43.1 67.1/77.5
  // (4096 rows: 22.4/19.3 and 36.7/40.9 with geglu; the quantising prologue has too few rows to hide behind)
  const int many = act == ACT_GEGLU ? 8192 : act == ACT_NONE ? 32768 : 16384;
  if (sx == nullptr && p.vec && K <= 640 && M >= many && K % 8 == 0 && ldx % 8 == 0 &&
      ((size_t)x | (size_t)gamma | (size_t)beta) % 16 == 0) {
    const uint16_t *xp = (const uint16_t*)x, *g = (const uint16_t*)gamma, *be = (const uint16_t*)beta;
#define ROWS(EL, GLU)                                                            \
  return g ? launch_rows<EL, GLU, true>(p, xp, ldx, g, be, eps, stream)          \
           : launch_rows<EL, GLU, false>(p, xp, ldx, g, be, eps, stream)
    if (act == ACT_GEGLU) {
      if (el) ROWS(1, true); else ROWS(0, true);
    } else {
      if (el) ROWS(1, false); else ROWS(0, false);
    }
#undef ROWS
  }
  if (sx == nullptr) {
    if (ws == nullptr) return -1;
    float* scale = (float*)((int8_t*)ws + (size_t)M * kp);
    const int rc = arb_quantize_rows(x, ldx, gamma, beta, eps, ws, kp, scale, M, K, el, stream);
    if (rc != 0) return rc;
    p.x = (const int8_t*)ws;
    p.ldx = kp;
    p.sx = scale;
  }
  if (p.ldx < kp || p.ldx % 16 || p.ldx >= (1L << 22)) return -1;
  if (act == ACT_GEGLU) return el ? launch_linear<1, true>(p, stream) : launch_linear<0, true>(p, stream);
  return el ? launch_linear<1, false>(p, stream) : launch_linear<0, false>(p, stream);
}
