// The bf16 instances of csrc/linattn_mix.h.  da, dc: the largest of the jobs'.
#include "linattn_mix.h"

#define MIX_BF16(F, ...)                                                                                                                         \
    if (da <= 32) { if (dc <= 16) return F<bf16_t, 16, 32, 1>(__VA_ARGS__); if (dc <= 32) return F<bf16_t, 16, 32, 2>(__VA_ARGS__); return F<bf16_t, 16, 32, 4>(__VA_ARGS__); } \
    if (da <= 64) { if (dc <= 32) return F<bf16_t, 16, 64, 2>(__VA_ARGS__); return F<bf16_t, 16, 64, 4>(__VA_ARGS__); }                                \
    if (dc <= 64) return F<bf16_t, 32, 128, 2>(__VA_ARGS__);                                                                                           \
    return F<bf16_t, 32, 128, 4>(__VA_ARGS__);

namespace xrl {

int launch_mix_bf16(const mix_t& m, int da, int dc, hipStream_t s) { MIX_BF16(launch_mix_size, m, dc, s) }
int mix_resident_bf16(int da, int dc) { MIX_BF16(mix_resident, ) }

// the instances that take close to 64 KB of LDS, or more
int init_mix_bf16() {
    if (int rc = init_mix_as<bf16_t, 32, 128, 2>()) return rc;
    return init_mix_as<bf16_t, 32, 128, 4>();
}

}  // namespace xrl
