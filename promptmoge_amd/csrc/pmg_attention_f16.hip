#include "pmg_attention.h"

namespace pmg {
int launch_attention_f16(AttnArgs& a, int waves, hipStream_t s) { return launch_attention_t<_Float16>(a, waves, s); }
}  // namespace pmg
