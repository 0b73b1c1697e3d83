// attention_masked_distance.cu - the masked attention kernels with a bias by distance.
#include "attention_masked.cuh"

namespace npub200 {

template int launch_masked_for<kFeatDistance>(int64_t, int, const CUtensorMap&, const CUtensorMap&, const CUtensorMap&,
                                  const MaskedArgs&, dim3, cudaStream_t, int);

}  // namespace npub200
