// The f32 instances of csrc/linattn_mix.h.  da, dc: the largest of the jobs'.
#include "linattn_mix.h"

#define MIX_F32(F, ...)                                                                                                                        \
    if (da <= 16) { if (dc <= 16) return F<float, 16, 16, 1>(__VA_ARGS__); if (dc <= 32) return F<float, 16, 16, 2>(__VA_ARGS__); return F<float, 16, 16, 4>(__VA_ARGS__); } \
    if (da <= 32) { if (dc <= 16) return F<float, 16, 32, 1>(__VA_ARGS__); if (dc <= 32) return F<float, 16, 32, 2>(__VA_ARGS__); return F<float, 16, 32, 4>(__VA_ARGS__); } \
    if (da <= 64) { if (dc <= 32) return F<float, 16, 64, 2>(__VA_ARGS__); return F<float, 16, 64, 4>(__VA_ARGS__); }                                \
    if (dc <= 64) return F<float, 16, 128, 4>(__VA_ARGS__);                                                                                          \
    return F<float, 16, 128, 8>(__VA_ARGS__);

namespace xrl {

int launch_mix_f32(const mix_t& m, int da, int dc, hipStream_t s) { MIX_F32(launch_mix_size, m, dc, s) }
int mix_resident_f32(int da, int dc) { MIX_F32(mix_resident, ) }

// the instances that take more than 64 KB of LDS
int init_mix_f32() {
    if (int rc = init_mix_as<float, 16, 64, 4>()) return rc;
    if (int rc = init_mix_as<float, 16, 128, 4>()) return rc;
    return init_mix_as<float, 16, 128, 8>();
}

}  // namespace xrl
