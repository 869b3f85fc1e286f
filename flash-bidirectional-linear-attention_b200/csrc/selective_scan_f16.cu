// The selective scan's kernels for __half inputs.
#include "selective_scan_kernels.cuh"

template struct fbla::scan::Launcher<__half>;
