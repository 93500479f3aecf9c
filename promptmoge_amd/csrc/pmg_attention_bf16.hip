#include "pmg_attention.h"

namespace pmg {
int launch_attention_bf16(AttnArgs& a, hipStream_t s) { return launch_attention_t<__bf16>(a, s); }
}  // namespace pmg
