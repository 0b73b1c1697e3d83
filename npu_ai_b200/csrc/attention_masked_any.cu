// attention_masked_any.cu - the masked attention kernels with any combination.
#include "attention_masked.cuh"

namespace npub200 {

template int launch_masked_for<kFeatAny>(int64_t, int, const CUtensorMap&, const CUtensorMap&, const CUtensorMap&,
                                  const MaskedArgs&, dim3, cudaStream_t, int);

}  // namespace npub200
