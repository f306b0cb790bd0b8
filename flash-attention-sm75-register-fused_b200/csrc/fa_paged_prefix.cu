// Paged attention in two passes over different keys (shared prefixes): the decode and chunk
// kernels again, with fp32 results of the first pass and the join in the second
// (kPartRows), beside the plain ones of fa_fwd_sm100.cu, whose code this leaves as it was (as a
// run-time choice it cost them 2 to 8 %).  And the summed weights of chunks.
#define FA_PART_ROWS 1
#include "fa_device.cuh"
#include "fa_paged_chunk.cuh"
#include "fa_paged_decode.cuh"
#include "fa_paged_weights_chunk.cuh"

namespace fa {

cudaError_t read_status_prefix(unsigned long long* out, bool reset) { return read_status_word(out, reset); }

}  // namespace fa
