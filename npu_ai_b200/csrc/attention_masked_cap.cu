// attention_masked_cap.cu - the masked attention kernels with capped scores.
#include "attention_masked.cuh"

namespace npub200 {

template int launch_masked_for<kFeatCap>(int64_t, int, const CUtensorMap&, const CUtensorMap&, const CUtensorMap&,
                                  const MaskedArgs&, dim3, cudaStream_t, int);

}  // namespace npub200
