// attention_masked_tensor.cu - the masked attention kernels with a mask tensor that has a row for each query.
#include "attention_masked.cuh"

namespace npub200 {

template int launch_masked_for<kFeatMask>(int64_t, int, const CUtensorMap&, const CUtensorMap&, const CUtensorMap&,
                                  const MaskedArgs&, dim3, cudaStream_t, int);

}  // namespace npub200
