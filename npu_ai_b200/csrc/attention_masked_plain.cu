// attention_masked_plain.cu - the masked attention kernels with no change to the scores (causal, prefix, document and length masks).
#include "attention_masked.cuh"

namespace npub200 {

template int launch_masked_for<0>(int64_t, int, const CUtensorMap&, const CUtensorMap&, const CUtensorMap&,
                                  const MaskedArgs&, dim3, cudaStream_t, int);

}  // namespace npub200
