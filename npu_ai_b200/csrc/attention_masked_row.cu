// attention_masked_row.cu - the masked attention kernels with a mask tensor whose rows the queries share.
#include "attention_masked.cuh"

namespace npub200 {

template int launch_masked_for<kFeatMaskRow>(int64_t, int, const CUtensorMap&, const CUtensorMap&, const CUtensorMap&,
                                     const MaskedArgs&, dim3, cudaStream_t, int);

}  // namespace npub200
