// Distillation of a categorical policy from a teacher's top logits (include/xrl_hip.h: xrl_distill_loss): the loss of every row and its
// gradient in one launch.  With m the row's maximum and Z = sum_a exp((s_a - m) / tau),
//     log p_a = (s_a - m) / tau - log Z,   loss = w tau^2 sum_k q_k (log q_k - log p_{i_k}),   d s_a = g w tau (p_a - q_a).
// Bound by memory: the logits are read, their gradient is written.
#include "io16.h"

namespace xrl {

constexpr int DISTILL_MAX_K = 256;

template <typename E>
__global__ void __launch_bounds__(256) distill_kernel(xrl_distill_t p) {
    __shared__ float scratch[16];
    __shared__ int ti[DISTILL_MAX_K];
    __shared__ float tq[DISTILL_MAX_K];
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x, A = p.A, K = p.K;
    const E* s = (const E*)p.logits + row * p.ld;
    E* d = p.d_logits ? (E*)p.d_logits + row * p.ld_d : nullptr;
    const float* av = p.avail ? p.avail + row * A : nullptr;
    const float w = p.weight ? p.weight[row] : 1.f, inv_tau = 1.f / p.temperature;
    float m = -INFINITY, tl = -INFINITY, z_at = 0.f;
    int idx = -1;
    if (w != 0.f) {
        if (tid < K) {
            idx = p.teacher_idx[row * K + tid];
            if (idx < 0 || idx >= A || (av && av[idx] == 0.f)) idx = -1;
            else {
                tl = io_load((const E*)p.teacher_logits + row * K + tid);
                z_at = io_load(s + idx);
                if (tl == -INFINITY) idx = -1;
            }
        }
        for (int a = tid; a < A; a += 256)
            if (!av || av[a] != 0.f) m = fmaxf(m, io_load(s + a));
    }
    auto block_max = [&](float v) {
        for (int off = 32; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor(v, off, 64));
        __syncthreads();
        if ((tid & 63) == 0) scratch[tid >> 6] = v;
        __syncthreads();
        return fmaxf(fmaxf(scratch[0], scratch[1]), fmaxf(scratch[2], scratch[3]));
    };
    m = block_max(m);
    const float tm = block_max(tl);
    const int valid = __syncthreads_count(idx >= 0);
    if (valid == 0 || m == -INFINITY) {
        if (d) for (int a = tid; a < A; a += 256) io_store(d + a, 0.f);
        if (tid == 0) p.loss[row] = 0.f;
        return;
    }
    float z = 0.f;
    for (int a = tid; a < A; a += 256)
        if (!av || av[a] != 0.f) z += expf((io_load(s + a) - m) * inv_tau);
    z = block_sum(z, scratch);
    const float te = idx >= 0 ? expf((tl - tm) * inv_tau) : 0.f;
    const float tsum = block_sum(te, scratch);
    const float q = te / tsum, lz = logf(z);
    float term = 0.f;
    if (q != 0.f) term = q * (((tl - tm) * inv_tau - logf(tsum)) - ((z_at - m) * inv_tau - lz));
    term = block_sum(term, scratch);
    if (tid == 0) p.loss[row] = w * p.temperature * p.temperature * term;
    if (!d) return;
    const float c = p.grad_scale * w * p.temperature, inv_z = 1.f / z;
    ti[tid] = idx; tq[tid] = q;
    for (int a = tid; a < A; a += 256) {
        const bool open = !av || av[a] != 0.f;
        io_store(d + a, open ? c * (expf((io_load(s + a) - m) * inv_tau) * inv_z) : 0.f);
    }
    __syncthreads();
    if (idx >= 0) {                       // the first of the entries that name an action writes for all of them
        float qs = 0.f;
        bool first = true;
        for (int j = 0; j < K; ++j)
            if (ti[j] == idx) { qs += tq[j]; first = first && j >= tid; }
        if (first) io_store(d + idx, c * (expf((z_at - m) * inv_tau) * inv_z - qs));
    }
}

}  // namespace xrl

using namespace xrl;

extern "C" int xrl_distill_loss(const xrl_distill_t* pp, xrl_stream_t stream) {
    XRL_CHECK_ARG(pp != nullptr);
    const xrl_distill_t& p = *pp;
    XRL_CHECK_ARG(p.N >= 0 && p.N <= 0x7fffffff && p.A >= 1 && p.K >= 1 && p.K <= DISTILL_MAX_K);
    XRL_CHECK_ARG((p.dtype == XRL_F32 || p.dtype == XRL_BF16) && p.temperature > 0.f);
    if (p.N == 0) return XRL_OK;
    XRL_CHECK_ARG(p.logits && p.teacher_idx && p.teacher_logits && p.loss);
    if (p.dtype == XRL_F32) hipLaunchKernelGGL(distill_kernel<float>, dim3((unsigned)p.N), dim3(256), 0, as_stream(stream), p);
    else hipLaunchKernelGGL(distill_kernel<bf16_t>, dim3((unsigned)p.N), dim3(256), 0, as_stream(stream), p);
    XRL_CHECK_LAUNCH();
    return XRL_OK;
}
