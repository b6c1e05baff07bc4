#include "mx_inst.cuh"
gz::MxEntry gz::mx_kernels_nvfp4(int config, bool gated) { return gz::inst::mx_entry_for<true>(config, gated); }
