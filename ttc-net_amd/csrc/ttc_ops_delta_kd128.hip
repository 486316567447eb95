// ttc_ops_delta_kd128.hip -- the gated delta rule's chunk kernels for keys of up to 128.
#include "ttc_ops_delta_chunk.hpp"

TTC_DELTA_UNIT(__bf16, 128)
TTC_DELTA_UNIT(float, 128)
