// The f32 instances of csrc/linattn_mix.h.
#include "linattn_mix.h"

namespace xrl {

// da, dc: the largest of the jobs'
int launch_mix_f32(const mix_t& m, int da, int dc, hipStream_t s) {
    if (da <= 16) return dc <= 16 ? launch_mix_size<float, 16, 16, 1>(m, dc, s) : dc <= 32 ? launch_mix_size<float, 16, 16, 2>(m, dc, s) : launch_mix_size<float, 16, 16, 4>(m, dc, s);
    if (da <= 32) return dc <= 16 ? launch_mix_size<float, 16, 32, 1>(m, dc, s) : dc <= 32 ? launch_mix_size<float, 16, 32, 2>(m, dc, s) : launch_mix_size<float, 16, 32, 4>(m, dc, s);
    if (da <= 64) return dc <= 32 ? launch_mix_size<float, 16, 64, 2>(m, dc, s) : launch_mix_size<float, 16, 64, 4>(m, dc, s);
    return dc <= 64 ? launch_mix_size<float, 16, 128, 4>(m, dc, s) : launch_mix_size<float, 16, 128, 8>(m, dc, s);
}

// the instances that take more than 64 KB of LDS
int init_mix_f32() {
    if (int rc = init_mix_as<float, 16, 64, 4>()) return rc;
    if (int rc = init_mix_as<float, 16, 128, 4>()) return rc;
    return init_mix_as<float, 16, 128, 8>();
}

}  // namespace xrl
