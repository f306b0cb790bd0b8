// Paged attention in two passes over different keys (shared prefixes): the decode and chunk
// kernels again, with fp32 results of the first pass and the join in the second
// (kPartRows), beside the plain ones of fa_fwd_sm100.cu, whose code this leaves as it was (as a
// run-time choice it cost them 2 to 8 %).  And the summed weights of chunks.
//
// A prefix is computed once for all rows behind it: the first pass sees its tokens as one
// sequence, of many rows, over the prefix's keys (few rows: the decode kernel, else the
// tensor cores), the second every sequence over its own keys.  Measured, 8 KV heads, d = 128, GQA
// 4, and in brackets the same batch as sequences that each have the prefix in their table:
// 64 single tokens behind 8192 bf16 keys, up to 1024 of their own, 63 us (143); 48 behind
// 16384 e4m3 keys 81 (186); 8 behind 1024 21 (16: two passes and a join have their fixed
// costs); 8 x 512 tokens behind 8192 540 (498: chunks fill the tensor cores' tiles by
// themselves, and the first pass's 67 MB of fp32 rows are written and read).
#define FA_PART_ROWS 1
#include "fa_device.cuh"
#include "fa_paged_chunk.cuh"
#include "fa_paged_decode.cuh"
#include "fa_paged_weights_chunk.cuh"

namespace fa {

cudaError_t read_status_prefix(unsigned long long* out, bool reset) { return read_status_word(out, reset); }

}  // namespace fa
