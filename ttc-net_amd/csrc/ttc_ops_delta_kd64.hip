// ttc_ops_delta_kd64.hip -- the gated delta rule's chunk kernels for keys of up to 64.
#include "ttc_ops_delta_chunk.hpp"

TTC_DELTA_UNIT(__bf16, 64)
TTC_DELTA_UNIT(float, 64)
