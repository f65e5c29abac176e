// Attention with masks and score transforms (forward, bf16 / fp16, fp32 softmax and accumulation).
//
//   s_ij = cap tanh(scale q_i.k_j / cap) - slope_h |p_i - j|          (cap, slope optional)
//   o_i  = sum_j softmax_j(s_ij) v_j  over the keys the masks leave, 0 where they leave none
//
// with p_i = start_b + i the position of query i.  Every mask (lengths, documents, causal, prefix) leaves a
// query ONE run of keys [lo, hi), so a row carries two integers instead of a mask:
//   documents: [off_t, off_t+1) of the document t that holds p_i (none: empty)
//   causal:    hi <= max(p_i + 1, first key of the document + prefix)
//   lengths:   hi <= length_b
// Keys outside the run never reach the result, whatever their bits are (NaN and infinities included).
#include "common.h"

struct MaskedArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* o;
  long q_sb, q_sn, q_sh, k_sb, k_sn, k_sh, v_sb, v_sn, v_sh, o_sb, o_sn, o_sh;
  int B, H, Hkv, Nq, Nk, D;
  int causal, q_start;
  const int* q_starts;   // [B] or null: q_start
  const int* lengths;    // [B] or null
  const int* docs;       // [B or 1, n_docs + 1] or null
  long docs_sb;
  int n_docs;
  const int* prefix;     // [B] (no documents) or one per document
  long prefix_sb;
  const float* slopes;   // [H] or null
  float scale, softcap;  // softcap 0: none
};

template <int EL>
__device__ __forceinline__ float ma_dec(uint16_t v) {
  if constexpr (EL == 0) return bf2f(v);
  else return (float)__builtin_bit_cast(_Float16, v);
}
template <int EL>
__device__ __forceinline__ uint16_t ma_enc(float f) {
  if constexpr (EL == 0) return f2bf(f);
  else return __builtin_bit_cast(uint16_t, (_Float16)f);
}

__device__ __forceinline__ long query_position(const MaskedArgs& a, int b, int i) {
  return (long)(a.q_starts ? a.q_starts[b] : a.q_start) + i;
}

// The run [lo, hi) of keys of query i.  Device data (lengths, offsets, prefixes, starts) is clamped, so no
// value of it can lead outside [0, Nk).
__device__ __forceinline__ void key_run(const MaskedArgs& a, int b, int i, int& lo, int& hi) {
  const long p = query_position(a, b, i);
  long l = 0, r = a.Nk;
  int t = 0;
  if (a.docs) {
    const int* off = a.docs + b * a.docs_sb;
    int x = 0, y = a.n_docs + 1;               // first index with off > p, in [0, n_docs + 1]
    while (x < y) {
      const int mid = (x + y) >> 1;
      if (off[mid] <= p) x = mid + 1;
      else y = mid;
    }
    t = x - 1;
    if (t < 0 || t >= a.n_docs) {
      lo = hi = 0;
      return;
    }
    l = max(l, (long)off[t]);
    r = min(r, (long)off[t + 1]);
  }
  if (a.causal) {
    long seen = p + 1;
    if (a.prefix) seen = max(seen, l + a.prefix[b * a.prefix_sb + t]);
    r = min(r, seen);
  }
  if (a.lengths) r = min(r, (long)a.lengths[b]);
  r = max(r, 0L);
  lo = (int)min(l, (long)a.Nk);
  hi = (int)r;
  if (lo >= hi) lo = hi = 0;
}

// One wave per (batch, head, query): lanes over the head dimension.
template <int EL>
__global__ void __launch_bounds__(64) masked_attention_row_kernel(MaskedArgs a) {
  const int i = blockIdx.x % a.Nq, h = (blockIdx.x / a.Nq) % a.H, b = blockIdx.x / a.Nq / a.H, lane = threadIdx.x;
  const int hk = h / (a.H / a.Hkv);
  const uint16_t* q = a.q + b * a.q_sb + i * a.q_sn + h * a.q_sh;
  float qv[4], acc[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) qv[e] = lane + 64 * e < a.D ? ma_dec<EL>(q[lane + 64 * e]) * a.scale : 0.f;
  int lo, hi;
  key_run(a, b, i, lo, hi);
  const long p = query_position(a, b, i);
  for (int j = lo; j < hi; ++j) {
    const uint16_t* k = a.k + b * a.k_sb + (long)j * a.k_sn + hk * a.k_sh;
    const uint16_t* v = a.v + b * a.v_sb + (long)j * a.v_sn + hk * a.v_sh;
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (lane + 64 * e < a.D) s += qv[e] * ma_dec<EL>(k[lane + 64 * e]);
    s = wave_sum(s);
    if (a.softcap > 0.f) s = a.softcap * tanhf(s / a.softcap);
    if (a.slopes) s -= a.slopes[h] * fabsf((float)(p - j));
    const float mn = fmaxf(m, s), w = mn == -INFINITY && s == s ? 0.f : __expf(s - mn);
    const float c = m == -INFINITY ? 0.f : __expf(m - mn);
    m = mn;
    l = l * c + w;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (lane + 64 * e < a.D) acc[e] = acc[e] * c + w * ma_dec<EL>(v[lane + 64 * e]);
  }
  uint16_t* o = a.o + b * a.o_sb + i * a.o_sn + h * a.o_sh;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (lane + 64 * e < a.D) o[lane + 64 * e] = ma_enc<EL>(l == 0.f ? 0.f : acc[e] / l);
}

// strides: {q, k, v, o} x {batch, token, head} elements; ints: {B, H, Hkv, Nq, Nk, D, causal, q_start, n_docs,
// docs_sb, prefix_sb}
ARB_API int arb_masked_attention(const void* q, const void* k, const void* v, void* o, const long* strides,
                                 const long* ints, const void* q_starts, const void* lengths, const void* docs,
                                 const void* prefix, const void* slopes, float scale, float softcap, int el,
                                 hipStream_t stream) {
  MaskedArgs a;
  a.q = (const uint16_t*)q; a.k = (const uint16_t*)k; a.v = (const uint16_t*)v; a.o = (uint16_t*)o;
  a.q_sb = strides[0]; a.q_sn = strides[1]; a.q_sh = strides[2];
  a.k_sb = strides[3]; a.k_sn = strides[4]; a.k_sh = strides[5];
  a.v_sb = strides[6]; a.v_sn = strides[7]; a.v_sh = strides[8];
  a.o_sb = strides[9]; a.o_sn = strides[10]; a.o_sh = strides[11];
  a.B = (int)ints[0]; a.H = (int)ints[1]; a.Hkv = (int)ints[2]; a.Nq = (int)ints[3]; a.Nk = (int)ints[4];
  a.D = (int)ints[5]; a.causal = (int)ints[6]; a.q_start = (int)ints[7]; a.n_docs = (int)ints[8];
  a.docs_sb = ints[9]; a.prefix_sb = ints[10];
  a.q_starts = (const int*)q_starts; a.lengths = (const int*)lengths; a.docs = (const int*)docs;
  a.prefix = (const int*)prefix; a.slopes = (const float*)slopes;
  a.scale = scale;
  a.softcap = softcap;
  if (a.B <= 0 || a.Nq <= 0 || a.Nk <= 0 || a.H <= 0 || a.Hkv <= 0 || a.H % a.Hkv || a.D <= 0 || a.D % 8 || a.D > 256)
    return -1;
  if ((long)a.Nq * a.H * a.B > 0x7fffffffL) return -1;
  const dim3 grid((unsigned)(a.Nq * a.H * a.B));
  if (el) masked_attention_row_kernel<1><<<grid, 64, 0, stream>>>(a);
  else masked_attention_row_kernel<0><<<grid, 64, 0, stream>>>(a);
  return (int)hipGetLastError();
}
