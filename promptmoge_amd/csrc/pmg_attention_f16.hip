#include "pmg_attention.h"

namespace pmg {
int launch_attention_f16(AttnArgs& a, hipStream_t s) { return launch_attention_t<_Float16>(a, s); }
}  // namespace pmg
