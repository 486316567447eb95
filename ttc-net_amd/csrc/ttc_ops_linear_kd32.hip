// ttc_ops_linear_kd32.hip -- the chunked sweep's kernels for keys of up to 32 elements.
#include "ttc_ops_linear_chunk.hpp"

TTC_CHUNK_UNIT(__bf16, 32)
TTC_CHUNK_UNIT(float, 32)
