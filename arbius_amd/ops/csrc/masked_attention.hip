// Entry points of the masked attention (masked_attention.inc) and its bf16 kernels; the fp16 ones are a source of
// their own (masked_attention_f16.hip), the two compile side by side.
#include "masked_attention.inc"

int dispatch_masked_f16(const MaskedArgs& a, hipStream_t s);

// How a call's keys are divided.  `batch`: the canonical batch under batch-invariant planning, so that a sequence's
// parts do not depend on what shares its launch.
struct KeyPlan {
  int splits, wk;
};
static KeyPlan key_plan(long batch, int H, int Hkv, int Nq, int Nk, int D) {
  const long rows = (long)(H / Hkv) * Nq, wgs = (rows + 127) / 128 * Hkv * batch;
  // Key ranges (a second kernel joins them): up to two workgroups per CU, 128 keys each at least, and not where
  // the partial sums written and read (8 D bytes a row and range) pass the keys and values read (4 D a key).  Measured,
  // us, 32 heads on 8: one token x 4, 65536 keys, 16 ranges 193, 8 ranges 229; one token x 16, 4096 keys, 4 ranges 60,
  // 8 ranges 61, 2 ranges 70; 16 heads on 4: 16 tokens, 8192 keys, 64 ranges 24, 8 ranges 29.
  long s = (512 + wgs - 1) / wgs;
  s = min(min(s, (Nk + 127L) / 128), min(256L, Nk / (2 * rows)));
  s = max(s, 1L);
  // 8 waves where a CU gets one workgroup and the keys are many (causal, us, against 4: 4096 tokens x 8 heads x 128
  // 69 / 87, 2 x 2047 x 8 x 80 36 / 41, 8192 x 4 x 64 82 / 105); with more workgroups a second one is the second wave
  // (8 x 2048 x 16 x 64 144 / 114)
  const int wk = wgs * s <= 256 && Nk >= 512 && rows > 32 && D <= 128 ? 2 : 1;
  return {(int)s, wk};
}

// bytes of workspace (0: none)
ARB_API size_t arb_masked_attention_workspace(int B, long batch, int H, int Hkv, int Nq, int Nk, int D) {
  const KeyPlan kp = key_plan(batch, H, Hkv, Nq, Nk, D);
  return kp.splits > 1 ? (size_t)kp.splits * B * H * Nq * (D + 2) * sizeof(float) : 0;
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
  for (int i = 0; i < 9; ++i)                                     // int counts, a tile past the last key too
    if (ints[i] > 0x7fffffffL - (i == 7 ? 0 : 1024)) return -1;
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
  // a tile's keys (at most 128) are addressed by 31-bit byte offsets; its row range check needs rows apart
  if (a.k_sn < a.D || a.v_sn < a.D || a.k_sn >= (1L << 22) || a.v_sn >= (1L << 22)) return -1;
  const long rows = (long)a.B * a.H * a.Nq;
  const KeyPlan kp = key_plan(ints[11], a.H, a.Hkv, a.Nq, a.Nk, a.D);
  a.splits = kp.splits;
  a.wk = kp.wk;
  const long group = (long)(a.H / a.Hkv) * a.Nq, wgs = (group + 127) / 128 * a.Hkv * a.B;
  // a launch has fewer than 2^32 threads
  if (group > 0x7fffffffL - 256 || wgs * a.splits >= (1L << 23) || (a.splits > 1 && rows >= (1L << 24))) return -1;
  if (a.splits > 1 && ws == nullptr) return -1;
  a.po = (float*)ws;
  a.pml = a.splits > 1 ? (float2*)((float*)ws + (size_t)a.splits * rows * a.D) : nullptr;
  return el ? dispatch_masked_f16(a, stream) : dispatch_masked<0>(a, stream);
}
