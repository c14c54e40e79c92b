// Host side of the ragged step's calls: the checks their arguments share.
#pragma once

namespace rlse {

// RLSE_OK, or a failure recorded for the call `what`.
int validate_chunk_shape(const char* what, int num_seqs, int total_tokens, int max_tokens, int Hq,
                         int Hkv, int mbps, int window, int sinks);

}  // namespace rlse
