// ttc_ops_linear_kd128.hip -- the chunked sweep's kernels for keys of up to 128 elements.
#include "ttc_ops_linear_chunk.hpp"

TTC_CHUNK_UNIT(__bf16, 128)
TTC_CHUNK_UNIT(float, 128)
