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
__device__ __forceinline__ int quant_one(float x, float inv) {
  const float r = __uint_as_float((__float_as_uint(x * inv) + 4u) & ~7u);
  return (int)__float_as_uint(r + 12582912.f);       // 1.5 2^23: r's integer in the low bits (the low byte is q)
}
// 127 / a with x pre-scaled by `up` where 127 / a would leave the fp32 range (a below 2^-100: bf16 only)
__device__ __forceinline__ void quant_scale(float a, float& s, float& inv, float& up) {
  up = a < 7.888609e-31f ? 1.2676506e30f : 1.f;      // 2^-100, 2^100
  const bool fine = a <= 3.4028235e38f;               // false for inf and NaN
  s = fine ? a / 127.f : __builtin_nanf("");
  inv = fine && a > 0.f ? 127.f / (a * up) : 0.f;
}

template <int EL>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const uint16_t* __restrict__ x, long ldx,
                                                            int8_t* __restrict__ q, int ldq,
                                                            float* __restrict__ scale, int K) {
  const long row = blockIdx.x;
  const uint16_t* xr = x + row * ldx;
  __shared__ float red[4];
  float a = 0.f;
  bool bad = false;
  for (int k = threadIdx.x; k < K; k += 256) {
    const float f = fabsf(dec16<EL>(xr[k]));
    bad |= !(f <= 3.4028235e38f);
    a = fmaxf(a, f);
  }
  if (bad) a = INFINITY;
  a = wave_max(a);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = a;
  __syncthreads();
  a = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  float s, inv, up;
  quant_scale(a, s, inv, up);
  for (int k = threadIdx.x; k < ldq; k += 256)
    q[row * ldq + k] = k < K && inv != 0.f ? (int8_t)quant_one(dec16<EL>(xr[k]) * up, inv) : 0;
  if (threadIdx.x == 0) scale[row] = s;
}

// LayerNorm in fp32, then the quantisation of the normalised row (not rounded in between).
template <int EL>
__global__ void __launch_bounds__(256) ln_quantize_rows_kernel(const uint16_t* __restrict__ x, long ldx,
                                                               const uint16_t* __restrict__ gamma,
                                                               const uint16_t* __restrict__ beta, float eps,
                                                               int8_t* __restrict__ q, int ldq,
                                                               float* __restrict__ scale, int K) {
  const long row = blockIdx.x;
  const uint16_t* xr = x + row * ldx;
  __shared__ float red[4];
  auto block_sum = [&](float v) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
  };
  float sum = 0.f;
  for (int k = threadIdx.x; k < K; k += 256) sum += dec16<EL>(xr[k]);
  const float mean = block_sum(sum) / (float)K;
  float ss = 0.f;
  for (int k = threadIdx.x; k < K; k += 256) {
    const float d = dec16<EL>(xr[k]) - mean;
    ss += d * d;
  }
  const float rstd = rsqrtf(block_sum(ss) / (float)K + eps);
  auto y = [&](int k) { return (dec16<EL>(xr[k]) - mean) * rstd * dec16<EL>(gamma[k]) + dec16<EL>(beta[k]); };
  float a = 0.f;
  bool bad = false;
  for (int k = threadIdx.x; k < K; k += 256) {
    const float f = fabsf(y(k));
    bad |= !(f <= 3.4028235e38f);
    a = fmaxf(a, f);
  }
  if (bad) a = INFINITY;
  a = wave_max(a);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = a;
  __syncthreads();
  a = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
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
  int M, N, K;
};

template <int EL, int ACT>
__global__ void __launch_bounds__(256) linear_int8_kernel(LinArgs p) {
  const int NO = ACT == ACT_GEGLU ? p.N / 2 : p.N;
  const int n = blockIdx.y * 256 + threadIdx.x, m = blockIdx.x;
  if (n >= NO) return;
  auto dot = [&](int row) {
    int acc = 0;
    const int* a = (const int*)(p.x + m * p.ldx);
    const int* b = (const int*)(p.w + row * p.ldw);
    for (int k = 0; k < (p.K + 3) / 4; ++k) acc = __builtin_amdgcn_sdot4(a[k], b[k], acc, false);
    float y = (float)acc * p.sx[m] * p.sw[row];
    if (p.b) y += dec16<EL>(p.b[row]);
    return y;
  };
  float y = dot(n);
  if (p.res) y += dec16<EL>(p.res[(long)m * p.N + n]);
  if (ACT == ACT_GEGLU) y *= gelu_f(dot(NO + n));
  else y = act_f(y, ACT);
  p.y[(long)m * NO + n] = (uint16_t)enc16<EL>(y);
}

// x [rows, K] 16-bit (row stride ldx elements) -> q [rows, ldq] int8, scale [rows]; gamma / beta: LayerNorm first
ARB_API int arb_quantize_rows(const void* x, long ldx, const void* gamma, const void* beta, float eps, void* q, int ldq,
                              void* scale, long rows, int K, int el, hipStream_t stream) {
  if (rows <= 0 || rows > 0x7fffffffL || K <= 0 || ldq < K || ldq % 16 || ldq - K >= 16 ||
      (gamma == nullptr) != (beta == nullptr))
    return -1;
  const dim3 grid((unsigned)rows);
  const uint16_t *xp = (const uint16_t*)x, *g = (const uint16_t*)gamma, *b = (const uint16_t*)beta;
  if (gamma) {
    if (el) ln_quantize_rows_kernel<1><<<grid, 256, 0, stream>>>(xp, ldx, g, b, eps, (int8_t*)q, ldq, (float*)scale, K);
    else ln_quantize_rows_kernel<0><<<grid, 256, 0, stream>>>(xp, ldx, g, b, eps, (int8_t*)q, ldq, (float*)scale, K);
  } else {
    if (el) quantize_rows_kernel<1><<<grid, 256, 0, stream>>>(xp, ldx, (int8_t*)q, ldq, (float*)scale, K);
    else quantize_rows_kernel<0><<<grid, 256, 0, stream>>>(xp, ldx, (int8_t*)q, ldq, (float*)scale, K);
  }
  return (int)hipGetLastError();
}

template <int EL>
static void launch_linear(const LinArgs& p, int act, hipStream_t s) {
  const int NO = act == ACT_GEGLU ? p.N / 2 : p.N;
  const dim3 grid(p.M, (NO + 255) / 256);
  switch (act) {
    case ACT_GELU: linear_int8_kernel<EL, ACT_GELU><<<grid, 256, 0, s>>>(p); break;
    case ACT_QUICK_GELU: linear_int8_kernel<EL, ACT_QUICK_GELU><<<grid, 256, 0, s>>>(p); break;
    case ACT_GEGLU: linear_int8_kernel<EL, ACT_GEGLU><<<grid, 256, 0, s>>>(p); break;
    default: linear_int8_kernel<EL, ACT_NONE><<<grid, 256, 0, s>>>(p); break;
  }
}

ARB_API int arb_linear_int8(const void* x, long ldx, const void* sx, const void* w, long ldw, const void* sw,
                            const void* b, const void* res, void* y, int M, int N, int K, int act, int el,
                            hipStream_t stream) {
  const int kp = (K + 15) / 16 * 16;
  if (M <= 0 || N <= 0 || K <= 0 || K > 133000 || ldx < kp || ldw < kp || ldx % 16 || ldw % 16 || act < 0 || act > 3 ||
      (act == ACT_GEGLU && (N % 2 || res)))
    return -1;
  LinArgs p{(const int8_t*)x, (const int8_t*)w, (const float*)sx, (const float*)sw, (const uint16_t*)b,
            (const uint16_t*)res, (uint16_t*)y, ldx, ldw, M, N, K};
  if (el) launch_linear<1>(p, act, stream);
  else launch_linear<0>(p, act, stream);
  return (int)hipGetLastError();
}
