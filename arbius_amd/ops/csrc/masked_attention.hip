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
  int splits;            // key ranges per row tile; 1: o is written, else po / pml
  float* po;             // [splits, B, Hkv, G Nq, D] fp32 partial sums
  float2* pml;           // [splits, B, Hkv, G Nq] (running maximum, sum)
};

template <int EL>
__device__ __forceinline__ float ma_dec(uint16_t v) {
  if constexpr (EL == 0) return bf2f(v);
  else return (float)__builtin_bit_cast(_Float16, v);
}
template <int EL>
__device__ __forceinline__ bool not_finite(uint32_t v) {
  constexpr uint32_t EXP = EL == 0 ? 0x7f80u : 0x7c00u;
  return (v & EXP) == EXP;
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

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// 32x32x16 matrix product step.  Lane l holds row / column l & 31 of A / B at k = 8 (l >> 5) .. + 7, and of the
// result column l & 31 at rows 8 (i >> 2) + 4 (l >> 5) + (i & 3), i = 0 .. 15.
template <int EL>
__device__ __forceinline__ f32x16 mma32(uint4 a, uint4 b, f32x16 c) {
  if constexpr (EL == 0)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                  0);
}

template <int EL>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  return (uint32_t)ma_enc<EL>(lo) | ((uint32_t)ma_enc<EL>(hi) << 16);
}

// 16 bytes per lane straight into LDS (lane-linear from the wave-uniform lds) through a buffer resource over
// [base, base + nbytes): a lane whose offset lies past it writes zeros.
__device__ __forceinline__ void dma_lds16(const void* base, int nbytes, void* lds, unsigned off) {
  __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, nbytes, 0x00020000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)lds, 16, off, 0, 0, 0);
}

__device__ __forceinline__ int wave_imin(int v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = min(v, __shfl_xor(v, o, 64));
  return v;
}
__device__ __forceinline__ int wave_imax(int v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = max(v, __shfl_xor(v, o, 64));
  return v;
}

enum { MA_PLAIN = 0, MA_CAP = 1, MA_BIAS = 2 };   // score transforms (bits)

// One workgroup (4 waves): 128 QT rows of one (batch, key / value head), against one range of keys.  A row is a
// (query, head of the group) pair, query major, so the G heads that share keys and values share their tiles.
//
// * S^T = K Q^T on 32x32x16 MFMA: a lane owns ONE row (column l & 31) and 16 of every 32 keys, so the row
//   maximum is a max3 tree plus one lane swap, and the sum needs none until the end.
// * P^T leaves the S^T accumulators as the B operand of O^T = V^T P^T, in the key order the accumulators have;
//   V^T comes from the row-major tile through the transposing LDS read in that same order.
// * K / V tiles of 64 keys go straight to LDS (double buffer, one barrier per tile).  Rows past the last key
//   any row of the workgroup sees arrive as zeros (buffer range check), so memory behind a sequence is
//   never multiplied.  16-byte chunks (K) and 32-byte pairs (V) are XOR-swizzled by the row on the source
//   address: fragment reads touch every bank once.
// * Tiles inside every row's run of keys skip the mask; the running maximum is kept until it grows by more than
//   8 (log2 units), so the accumulators are rescaled only on the few tiles that need it.
// * A masked key has P = 0 exactly, but 0 * V is NaN for a NaN or infinite V.  The result shows that (every
//   poisoned sum is NaN or infinite), and only then the workgroup runs a second pass: V's NaNs and infinities
//   are zeroed in LDS and added, one key at a time, to the rows that do see the key.  All other rows repeat
//   the first pass's arithmetic: their bits do not depend on what masked places hold.
template <int EL, int DC, int QT, int TR>
__global__ void __launch_bounds__(256, (DC <= 128 && QT * DC <= 128) ? 2 : 1) masked_attention_kernel(MaskedArgs a) {
  constexpr int KS = DC / 16, DT = DC / 32;
  constexpr int RB = DC <= 64 ? 64 : DC <= 128 ? 128 : 256;       // LDS row (elements)
  constexpr int RCH = RB / 8;                                     // 16-byte chunks per LDS row
  constexpr int STAGE = 64 * RB * 2;
  constexpr int NDMA = 64 * RCH / 256;                            // DMA instructions per wave, K and V each
  __shared__ __attribute__((aligned(16))) uint16_t s0[STAGE];
  __shared__ __attribute__((aligned(16))) uint16_t s1[STAGE];
  __shared__ int sred[8];
  __shared__ int sflag[64];

  const int G = a.H / a.Hkv, R = G * a.Nq;
  const int nrt = (R + 128 * QT - 1) / (128 * QT);
  const int total = nrt * a.splits * a.Hkv * a.B;
  int lin = xcd_remap(blockIdx.x, total);
  const int split = lin % a.splits;
  lin /= a.splits;
  const int rt = nrt - 1 - lin % nrt;                             // causal: the longest tiles start first
  lin /= nrt;
  const int hk = lin % a.Hkv, b = lin / a.Hkv;

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int D = a.D;

  // ---- rows: key runs, positions, Q fragments
  int row[QT], lo[QT], hi[QT];
  long pos[QT];
  float slope[QT];
  uint4 qf[QT][KS];
  int wlo = 0x7fffffff, whi = 0, wmaxlo = 0, wminhi = 0x7fffffff;
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    row[qt] = rt * 128 * QT + (wave * QT + qt) * 32 + col;
    const bool ok = row[qt] < R;
    const int i = (ok ? row[qt] : 0) / G, g = (ok ? row[qt] : 0) - i * G, h = hk * G + g;
    key_run(a, b, i, lo[qt], hi[qt]);
    pos[qt] = query_position(a, b, i);
    slope[qt] = 0.f;
    if constexpr ((TR & MA_BIAS) != 0)
      if (a.slopes) slope[qt] = a.slopes[h] * -1.4426950408889634f;
    if (!ok) lo[qt] = hi[qt] = 0;
    if (ok) {
      if (lo[qt] < hi[qt]) {
        wlo = min(wlo, lo[qt]);
        whi = max(whi, hi[qt]);
      }
      wmaxlo = max(wmaxlo, lo[qt]);
      wminhi = min(wminhi, hi[qt]);
    }
    const uint16_t* q = a.q + b * a.q_sb + i * a.q_sn + h * a.q_sh;
    const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;       // the scale's sign goes to Q, exactly
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int d = 16 * s + 8 * half;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (ok && d < D) {
        v = ld16(q + d);
        v.x ^= flip; v.y ^= flip; v.z ^= flip; v.w ^= flip;
      }
      qf[qt][s] = v;
    }
  }
  wlo = wave_imin(wlo);
  whi = wave_imax(whi);
  wmaxlo = wave_imax(wmaxlo);
  wminhi = wave_imin(wminhi);
  if (lane == 0) {
    sred[wave] = wlo;
    sred[4 + wave] = whi;
  }
  __syncthreads();
  const int glo = min(min(sred[0], sred[1]), min(sred[2], sred[3]));
  const int ghi = max(max(sred[4], sred[5]), max(sred[6], sred[7]));
  // this split's tiles: [k0, k1)
  const int tiles = ghi > glo ? (ghi - glo + 63) / 64 : 0;
  const int per = (tiles + a.splits - 1) / a.splits;
  const int k0 = __builtin_amdgcn_readfirstlane(glo + 64 * min(tiles, split * per));
  const int k1 = __builtin_amdgcn_readfirstlane(min(ghi, glo + 64 * min(tiles, (split + 1) * per)));
  wlo = __builtin_amdgcn_readfirstlane(wlo);
  whi = __builtin_amdgcn_readfirstlane(whi);
  wmaxlo = __builtin_amdgcn_readfirstlane(wmaxlo);
  wminhi = __builtin_amdgcn_readfirstlane(wminhi);

  // ---- DMA geometry: instruction n of wave w fills chunks [64 (w + 4 n), + 64) of the tile image
  const char* kbase = (const char*)(a.k + b * a.k_sb + hk * a.k_sh);
  const char* vbase = (const char*)(a.v + b * a.v_sb + hk * a.v_sh);
  const int ksn = (int)a.k_sn * 2, vsn = (int)a.v_sn * 2;         // bytes (64 rows stay below 2^31: checked)
  unsigned ko[NDMA], vo[NDMA];
#pragma unroll
  for (int n = 0; n < NDMA; ++n) {
    const int c = 64 * (wave + 4 * n) + lane, r = c / RCH, at = c % RCH;
    const int kc = RB == 64 ? at ^ ((r >> 1) & 7) : at ^ (r & 15);
    const int vc = RB == 64 ? at ^ (((r >> 1) & 3) << 1) : at ^ ((r & 7) << 1);
    ko[n] = kc * 8 < D ? (unsigned)(r * ksn + kc * 16) : 0x80000000u;
    vo[n] = vc * 8 < D ? (unsigned)(r * vsn + vc * 16) : 0x80000000u;
  }
  auto issue = [&](int kv, uint16_t* dst) __attribute__((always_inline)) {
    const int rows = min(64, k1 - kv);
    const char* kb = kbase + (long)kv * ksn;
    const char* vb = vbase + (long)kv * vsn;
#pragma unroll
    for (int n = 0; n < NDMA; ++n) dma_lds16(kb, rows * ksn, dst + 512 * (wave + 4 * n), ko[n]);
#pragma unroll
    for (int n = 0; n < NDMA; ++n) dma_lds16(vb, rows * vsn, dst + 64 * RB + 512 * (wave + 4 * n), vo[n]);
  };

  f32x16 o[QT][DT];
  float m[QT], l[QT];
  const float c1 = fabsf(a.scale) * 1.4426950408889634f;
  // cap tanh(t) log2(e) = C - 2 C / (1 + exp2(2 log2(e) t)), t = scale s / cap
  const float capc = a.softcap * 1.4426950408889634f;
  const float capk = a.softcap > 0.f ? 2.f * c1 / a.softcap : 0.f;

  auto tile = [&](int kv, const uint16_t* sk, bool careful) __attribute__((always_inline)) {
    if (kv + 64 <= wlo || kv >= whi) return;                      // no row of this wave sees the tile
    const uint16_t* sv = sk + 64 * RB;
    f32x16 st[QT][2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) st[qt][t] = (f32x16){};
      const int r = 32 * t + col;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int c = 2 * s + half;
        const uint4 kf = ld16(sk + r * RB + 8 * (RB == 64 ? c ^ ((r >> 1) & 7) : c ^ (r & 15)));
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) st[qt][t] = mma32<EL>(kf, qf[qt][s], st[qt][t]);
      }
    }
    const bool full = kv >= wmaxlo && kv + 64 <= wminhi;          // wave-uniform
    uint4 pf[QT][4];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      // scores in log2 units (plain: still raw, the scale rides on the exp2 argument's fma)
      if constexpr (TR != MA_PLAIN) {
        const float d0 = (float)(pos[qt] - (kv + 4 * half));
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float x;
            if constexpr ((TR & MA_CAP) != 0) {
              const float e = __builtin_amdgcn_exp2f(st[qt][t][i] * capk);
              x = fmaf(-2.f * capc, __builtin_amdgcn_rcpf(1.f + e), capc);
            } else {
              x = st[qt][t][i] * c1;
            }
            if constexpr ((TR & MA_BIAS) != 0)
              x = fmaf(slope[qt], fabsf(d0 - (float)(32 * t + 8 * (i >> 2) + (i & 3))), x);
            st[qt][t][i] = x;
          }
      }
      if (!full) {
        const int first = lo[qt] - kv - 4 * half, count = hi[qt] - lo[qt];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int key = 32 * t + 8 * (i >> 2) + (i & 3);
            st[qt][t][i] = (unsigned)(key - first) < (unsigned)count ? st[qt][t][i] : -INFINITY;
          }
      }
      float mx = vmax3(st[qt][0][0], st[qt][0][1], st[qt][0][2]);
#pragma unroll
      for (int i = 3; i < 31; i += 2) mx = vmax3(mx, st[qt][i >> 4][i & 15], st[qt][(i + 1) >> 4][(i + 1) & 15]);
      mx = max_xor32(vmax2(mx, st[qt][1][15]));
      if constexpr (TR == MA_PLAIN) mx *= c1;
      const bool grow = mx > m[qt] + 8.f;
      if (__any(grow)) {
        const float to = grow ? mx : m[qt];
        const float alpha = m[qt] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[qt] - to);
        if (grow) {
          m[qt] = to;
          l[qt] *= alpha;
        }
        const float by = grow ? alpha : 1.f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[qt][dt] *= by;
      }
      const float mu = m[qt] == -INFINITY ? 0.f : m[qt];
      float sum = 0.f;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float x = TR == MA_PLAIN ? fmaf(st[qt][t][i], c1, -mu) : st[qt][t][i] - mu;
          st[qt][t][i] = __builtin_amdgcn_exp2f(x);
          sum += st[qt][t][i];
        }
      l[qt] += sum;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const f32x16& x = st[qt][u >> 1];
        const int e = 8 * (u & 1);
        pf[qt][u] = make_uint4(pack2<EL>(x[e], x[e + 1]), pack2<EL>(x[e + 2], x[e + 3]),
                               pack2<EL>(x[e + 4], x[e + 5]), pack2<EL>(x[e + 6], x[e + 7]));
      }
    }
    // ---- O^T += V^T P^T
    const int vr = 4 * half + ((lane & 15) >> 2), vp = (lane >> 4) & 1, vw = 4 * (lane & 3);
    auto vfrag = [&](int dt, int u) __attribute__((always_inline)) {
      const int r = 16 * u + vr, p = 2 * dt + vp;
      const uint16_t* v0 = sv + r * RB + 16 * (RB == 64 ? p ^ ((r >> 1) & 3) : p ^ (r & 7)) + vw;
      const int r1 = r + 8;
      const uint16_t* v1 = sv + r1 * RB + 16 * (RB == 64 ? p ^ ((r1 >> 1) & 3) : p ^ (r1 & 7)) + vw;
      const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(LDS_PTR(s16x4, v0));
      const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16(LDS_PTR(s16x4, v1));
      const uint2 xx = __builtin_bit_cast(uint2, x), yy = __builtin_bit_cast(uint2, y);
      return make_uint4(xx.x, xx.y, yy.x, yy.y);
    };
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint4 v = vfrag(dt, u);
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) o[qt][dt] = mma32<EL>(v, pf[qt][u], o[qt][dt]);
      }
    if (careful) {                                                // uniform
      for (int j = 0; j < 64; ++j) {
        if (!sflag[j]) continue;
        const uint16_t* v = (const uint16_t*)(vbase + (long)(kv + j) * vsn);
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) {
          const bool sees = kv + j >= lo[qt] && kv + j < hi[qt];
#pragma unroll
          for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int d = 32 * dt + 8 * (i >> 2) + 4 * half + (i & 3);
              const uint16_t x = sees && d < D ? v[d] : 0;
              if (not_finite<EL>(x)) o[qt][dt][i] += ma_dec<EL>(x);
            }
        }
      }
    }
  };
  // pass 1: the NaNs and infinities of the V tile become zeros, their keys are flagged
  auto clean = [&](int kv, uint16_t* sk) __attribute__((always_inline)) {
    if (tid < 64) sflag[tid] = 0;
    __syncthreads();
    for (int c = tid; c < 64 * RCH; c += 256) {
      uint4 v = ld16(sk + 64 * RB + 8 * c);
      uint32_t w[4] = {v.x, v.y, v.z, v.w};
      bool any = false;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (not_finite<EL>(w[e] & 0xffffu)) any = true, w[e] &= 0xffff0000u;
        if (not_finite<EL>(w[e] >> 16)) any = true, w[e] &= 0xffffu;
      }
      if (any) {
        st16(sk + 64 * RB + 8 * c, make_uint4(w[0], w[1], w[2], w[3]));
        sflag[c / RCH] = 1;
      }
    }
    __syncthreads();
  };

  for (int pass = 0; pass < 2; ++pass) {
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      m[qt] = -INFINITY;
      l[qt] = 0.f;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[qt][dt] = (f32x16){};
    }
    // stage roles are static (loop unrolled by 2): DMA into one stage while the other is read; a stage is
    // refilled only after the barrier that retired its last reads
    if (k0 < k1) issue(k0, s0);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    for (int kv = k0; kv < k1; kv += 128) {
      if (kv + 64 < k1) issue(kv + 64, s1);
      if (pass) clean(kv, s0);
      tile(kv, s0, pass);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      if (kv + 64 >= k1) break;
      if (kv + 128 < k1) issue(kv + 128, s0);
      if (pass) clean(kv + 64, s1);
      tile(kv + 64, s1, pass);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
    }
    bool bad = false;
#pragma unroll
    for (int qt = 0; qt < QT; ++qt)
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) bad |= !(fabsf(o[qt][dt][i]) <= 3.4028235e38f);
    if (pass || !__syncthreads_or(bad)) break;
  }

  // ---- one sum over the two lanes of a row, then the row (or its part of it)
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const float sum = sum_xor32(l[qt]);
    if (row[qt] >= R) continue;
    if (a.splits > 1) {
      const long at = (((long)split * a.B + b) * a.Hkv + hk) * R + row[qt];
      if (half == 0) a.pml[at] = make_float2(m[qt], sum);
      float* po = a.po + at * D;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          const int d = 32 * dt + 2 * i + 4 * half;
          if (d < D)
            *reinterpret_cast<f32x4*>(po + d) =
                (f32x4){o[qt][dt][i], o[qt][dt][i + 1], o[qt][dt][i + 2], o[qt][dt][i + 3]};
        }
      continue;
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const int i0 = row[qt] / G, h = hk * G + row[qt] - i0 * G;
    uint16_t* out = a.o + b * a.o_sb + i0 * a.o_sn + h * a.o_sh;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const int d = 32 * dt + 2 * i + 4 * half;
        if (d < D) {
          const f32x16& x = o[qt][dt];
          *reinterpret_cast<uint2*>(out + d) = make_uint2(pack2<EL>(x[i] * inv, x[i + 1] * inv),
                                                          pack2<EL>(x[i + 2] * inv, x[i + 3] * inv));
        }
      }
  }
}

// Joins the splits of a row: o = sum_s 2^(m_s - m) po_s / sum_s 2^(m_s - m) l_s, in split order.  One wave per row.
template <int EL>
__global__ void __launch_bounds__(256) masked_attention_join_kernel(MaskedArgs a) {
  const int G = a.H / a.Hkv, R = G * a.Nq, lane = threadIdx.x & 63;
  const long rows = (long)a.B * a.Hkv * R, at = blockIdx.x * 4L + (threadIdx.x >> 6);
  if (at >= rows) return;
  float m = -INFINITY;
  for (int s = 0; s < a.splits; ++s) m = fmaxf(m, a.pml[s * rows + at].x);
  if (m == -INFINITY) m = 0.f;
  float sum = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
  const int d = 4 * lane;
  for (int s = 0; s < a.splits; ++s) {
    const float2 ml = a.pml[s * rows + at];
    if (ml.x == -INFINITY && ml.y == 0.f) continue;               // nothing seen
    const float w = __builtin_amdgcn_exp2f(ml.x - m);
    sum += w * ml.y;
    if (d < a.D) {
      const float4 p = *reinterpret_cast<const float4*>(a.po + (s * rows + at) * a.D + d);
      acc[0] += w * p.x; acc[1] += w * p.y; acc[2] += w * p.z; acc[3] += w * p.w;
    }
  }
  if (d >= a.D) return;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int r = (int)(at % R), hk = (int)(at / R % a.Hkv), b = (int)(at / R / a.Hkv), i = r / G;
  uint16_t* o = a.o + b * a.o_sb + i * a.o_sn + (hk * G + r - i * G) * a.o_sh + d;
  *reinterpret_cast<uint2*>(o) =
      make_uint2(pack2<EL>(acc[0] * inv, acc[1] * inv), pack2<EL>(acc[2] * inv, acc[3] * inv));
}

template <int EL, int DC, int QT>
static void launch_masked(const MaskedArgs& a, hipStream_t s) {
  const long nrt = ((long)(a.H / a.Hkv) * a.Nq + 128 * QT - 1) / (128 * QT);
  const dim3 grid((unsigned)(nrt * a.splits * a.Hkv * a.B));
  const bool bias = a.slopes != nullptr || a.scale == 0.f;        // scale 0: masked scores must not be scaled
  if (a.softcap > 0.f) {
    if (bias) masked_attention_kernel<EL, DC, QT, MA_CAP | MA_BIAS><<<grid, 256, 0, s>>>(a);
    else masked_attention_kernel<EL, DC, QT, MA_CAP><<<grid, 256, 0, s>>>(a);
  } else {
    if (bias) masked_attention_kernel<EL, DC, QT, MA_BIAS><<<grid, 256, 0, s>>>(a);
    else masked_attention_kernel<EL, DC, QT, MA_PLAIN><<<grid, 256, 0, s>>>(a);
  }
  if (a.splits > 1) {
    const long rows = (long)a.B * a.H * a.Nq;
    masked_attention_join_kernel<EL><<<dim3((unsigned)((rows + 3) / 4)), 256, 0, s>>>(a);
  }
}

template <int EL>
static int dispatch_masked(const MaskedArgs& a, hipStream_t s) {
  if (a.D <= 32) launch_masked<EL, 32, 1>(a, s);
  else if (a.D <= 64) launch_masked<EL, 64, 1>(a, s);
  else if (a.D <= 96) launch_masked<EL, 96, 1>(a, s);
  else if (a.D <= 128) launch_masked<EL, 128, 1>(a, s);
  else if (a.D <= 160) launch_masked<EL, 160, 1>(a, s);
  else launch_masked<EL, 256, 1>(a, s);
  return (int)hipGetLastError();
}

// Key ranges per row tile: split while the launch has fewer than 512 workgroups (two per CU) and every range
// keeps 4 tiles.  `batch`: the canonical batch under batch-invariant planning, so a sequence's ranges do not
// depend on what shares its launch.
static int masked_splits(long batch, int H, int Hkv, int Nq, int Nk) {
  const long nrt = ((long)(H / Hkv) * Nq + 127) / 128, wgs = nrt * Hkv * batch;
  const long most = (Nk + 255) / 256;
  long s = (512 + wgs - 1) / wgs;
  s = s < most ? s : most;
  return (int)(s < 1 ? 1 : s > 128 ? 128 : s);
}

// bytes of workspace (0: none); also the split count is fixed by these arguments alone
ARB_API size_t arb_masked_attention_workspace(int B, long batch, int H, int Hkv, int Nq, int Nk, int D) {
  const int s = masked_splits(batch, H, Hkv, Nq, Nk);
  return s > 1 ? (size_t)s * B * H * Nq * (D + 2) * sizeof(float) : 0;
}

// dims: {q, k, v, o} x {batch, token, head} strides in elements, then {B, H, Hkv, Nq, Nk, D, causal, q_start,
// n_docs, docs_sb, prefix_sb, canonical batch}
ARB_API int arb_masked_attention(const void* q, const void* k, const void* v, void* o, const void* dims,
                                 const void* q_starts, const void* lengths, const void* docs, const void* prefix,
                                 const void* slopes, void* ws, float scale, float softcap, int el,
                                 hipStream_t stream) {
  long strides[12], ints[12];
  __builtin_memcpy(strides, dims, sizeof(strides));
  __builtin_memcpy(ints, (const char*)dims + sizeof(strides), sizeof(ints));
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
  if (a.B <= 0 || a.Nq <= 0 || a.Nk <= 0 || a.H <= 0 || a.Hkv <= 0 || a.H % a.Hkv || a.D <= 0 || a.D % 8 ||
      a.D > 256 || ints[11] <= 0)
    return -1;
  // a tile's 64 rows are addressed by 31-bit byte offsets; its row range check needs rows apart
  if (a.k_sn < a.D || a.v_sn < a.D || a.k_sn >= (1L << 23) || a.v_sn >= (1L << 23)) return -1;
  const long rows = (long)a.B * a.H * a.Nq;
  a.splits = masked_splits(ints[11], a.H, a.Hkv, a.Nq, a.Nk);
  if ((long)(a.H / a.Hkv) * a.Nq > 0x7fffffffL - 256 || (rows + 127) * a.splits > 0x7fffffffL) return -1;
  if (a.splits > 1 && ws == nullptr) return -1;
  a.po = (float*)ws;
  a.pml = a.splits > 1 ? (float2*)((float*)ws + (size_t)a.splits * rows * a.D) : nullptr;
  return el ? dispatch_masked<1>(a, stream) : dispatch_masked<0>(a, stream);
}
