#include "pmg_grouped_kernels.h"

template int pmg::launch_experts<__bf16>(pmg::GroupArgs&, bool, hipStream_t);
template int pmg::launch_lora<__bf16>(pmg::GroupArgs&, bool, bool, hipStream_t);
