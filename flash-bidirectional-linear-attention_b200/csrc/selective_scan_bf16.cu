// The selective scan's kernels for __nv_bfloat16 inputs.
#include "selective_scan_kernels.cuh"

template struct fbla::scan::Launcher<__nv_bfloat16>;
