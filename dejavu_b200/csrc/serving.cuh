// What the kernels of the serving library share.
#pragma once
#include "../../include/dejavu_b200_serving.h"
#include "dtype.cuh"
#include "serving_plan.cuh"

namespace djv {

// table entries and positions that each kernel refused (djv_paged_faults)
unsigned append_faults(), decode_faults();
// waits that ran out (djv_serving_timeouts)
unsigned decode_timeouts(), packed_timeouts();

struct Pool {  // strides in elements
  long long ld_page, ld_head, ld_slot;
};

inline bool is_dtype(int dtype) { return dtype == DJV_DTYPE_F16 || dtype == DJV_DTYPE_BF16 || dtype == DJV_DTYPE_F32; }

}  // namespace djv
