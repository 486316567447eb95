// ttc_ops_delta_kd32.hip -- the gated delta rule's chunk kernels for keys of up to 32.
#include "ttc_ops_delta_chunk.hpp"

TTC_DELTA_UNIT(__bf16, 32)
TTC_DELTA_UNIT(float, 32)
