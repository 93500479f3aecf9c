#include "pmg_attention.h"

namespace pmg {
int launch_attention_f32(AttnArgs& a, hipStream_t s) { return launch_attention_t<float>(a, s); }
}  // namespace pmg
