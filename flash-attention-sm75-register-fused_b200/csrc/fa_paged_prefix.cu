// Paged attention in two passes over different keys (shared prefixes): the decode and chunk
// kernels again, with fp32 results of the first pass and the join in the second
// (kPartRows), beside the plain ones of fa_fwd_sm100.cu, whose code this leaves as it was (as a
// run-time choice it cost them 2 to 8 %).  And the summed weights of chunks.
//
// A prefix is computed once for all rows behind it: the first pass sees its tokens as one
// sequence, of many rows, over the prefix's keys (few rows: the decode kernel, else the
// tensor cores), the second every sequence over its own keys.  Measured, calls among others, 8 KV
// heads, d = 128, GQA 4, and in brackets the same batch as sequences that each have the prefix
// in their table: 64 single tokens behind 8192 bf16 keys, up to 1024 of their own, 61 us (135);
// 48 behind 16384 e4m3 keys 79 (181); 512 tokens and 31 single ones behind 8192 130 (192); 8
// behind 1024 19 (15: two passes and a join have their fixed costs); 32 x 4 drafts of d = 64
// behind three prefixes 41 (31: the first pass reads every unit in four warps); 8 x 512 tokens
// behind 8192 522 to 593 from run to run (498 to 551: chunks fill the tensor cores' tiles by
// themselves, and the first pass's 67 MB of fp32 rows are written and read).
#define FA_PART_ROWS 1
#include "fa_device.cuh"
#include "fa_paged_chunk.cuh"
#include "fa_paged_decode.cuh"
#include "fa_paged_weights_chunk.cuh"

namespace fa {

cudaError_t read_status_prefix(unsigned long long* out, bool reset) { return read_status_word(out, reset); }

}  // namespace fa
