// The f32 instances of csrc/linattn_mix.h.
#include "linattn_mix.h"

namespace xrl {

int launch_mix_f32(const mix_t& m, int da, int dc, hipStream_t s) { return launch_mix<float>(m, da, dc, s); }
int init_mix_f32() { return init_mix<float>(); }

}  // namespace xrl
