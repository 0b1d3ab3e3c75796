// The bf16 instances of csrc/linattn_mix.h.
#include "linattn_mix.h"

namespace xrl {

// da, dc: the largest of the jobs'
int launch_mix_bf16(const mix_t& m, int da, int dc, hipStream_t s) {
    if (da <= 32) return dc <= 16 ? launch_mix_size<bf16_t, 16, 32, 1>(m, dc, s) : dc <= 32 ? launch_mix_size<bf16_t, 16, 32, 2>(m, dc, s) : launch_mix_size<bf16_t, 16, 32, 4>(m, dc, s);
    if (da <= 64) return dc <= 32 ? launch_mix_size<bf16_t, 16, 64, 2>(m, dc, s) : launch_mix_size<bf16_t, 16, 64, 4>(m, dc, s);
    return dc <= 64 ? launch_mix_size<bf16_t, 32, 128, 2>(m, dc, s) : launch_mix_size<bf16_t, 32, 128, 4>(m, dc, s);
}

// the instances that take close to 64 KB of LDS
int init_mix_bf16() {
    if (int rc = init_mix_as<bf16_t, 32, 128, 2>()) return rc;
    return init_mix_as<bf16_t, 32, 128, 4>();
}

}  // namespace xrl
