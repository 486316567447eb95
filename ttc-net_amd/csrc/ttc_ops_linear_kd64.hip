// ttc_ops_linear_kd64.hip -- the chunked sweep's kernels for keys of up to 64 elements.
#include "ttc_ops_linear_chunk.hpp"

TTC_CHUNK_UNIT(__bf16, 64)
TTC_CHUNK_UNIT(float, 64)
