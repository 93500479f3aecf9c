#include "pmg_grouped_kernels.h"

template int pmg::launch_experts<_Float16>(pmg::GroupArgs&, bool, hipStream_t);
template int pmg::launch_lora<_Float16>(pmg::GroupArgs&, bool, bool, hipStream_t);
