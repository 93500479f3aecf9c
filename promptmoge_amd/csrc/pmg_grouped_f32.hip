#include "pmg_grouped_kernels.h"

template int pmg::launch_experts<float>(pmg::GroupArgs&, bool, hipStream_t);
template int pmg::launch_lora<float>(pmg::GroupArgs&, bool, bool, hipStream_t);
