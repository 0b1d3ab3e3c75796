// The bf16 instances of csrc/linattn_mix.h.
#include "linattn_mix.h"

namespace xrl {

int launch_mix_bf16(const mix_t& m, int da, int dc, hipStream_t s) { return launch_mix<bf16_t>(m, da, dc, s); }
int init_mix_bf16() { return init_mix<bf16_t>(); }

}  // namespace xrl
