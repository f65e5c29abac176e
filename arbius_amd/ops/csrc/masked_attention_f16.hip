// fp16 kernels of the masked attention (masked_attention.inc).
#include "masked_attention.inc"

int dispatch_masked_f16(const MaskedArgs& a, hipStream_t s) { return dispatch_masked<1>(a, s); }
