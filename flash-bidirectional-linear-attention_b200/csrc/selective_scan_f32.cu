// The selective scan's kernels for float inputs.
#include "selective_scan_kernels.cuh"

template struct fbla::scan::Launcher<float>;
