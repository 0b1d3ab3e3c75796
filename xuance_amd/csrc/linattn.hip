// Linear attention with one decay per head (include/xrl_hip.h: xrl_linattn_*): whole sequences, their gradients, one acting step.
//
// One operator carries all of it.  With a_i, b_j of width da and c_j of width dc,
//     mix_i = sum_{j <= i, same segment} lam^(i-j) (a_i . b_j) c_j + lam^(i+off) a_i S_in,     S: [da][dc]
// is the forward pass for (a, b, c) = (q, k, v) and the gradients for
//     d_q: (d_out, v, k), S_in = state^T;     d_k: (v, d_out, q) and d_v: (k, q, d_out) in reversed time, S_in = d_state_out(^T), off = 0,
// because S_t meets d S_t exactly where o_t meets q_t.  A launch runs one job (forward) or three (backward) of it.
#include "io16.h"

namespace xrl {

struct mix_job_t {
    const void* a; const void* b; const void* c; void* out;
    int64_t sa[3], sb[3], sc[3], so[3];
    int da, dc;
    const float* s_in; float* s_out;      // [B][H][dk][dv], element (d, e) at d * sd + e * se
    int sd, se;
    int reverse, off;
    float scale_p, scale_s, scale_b;      // of the products a.b, of a S, of b (x) c in the state
};
struct mix_t {
    mix_job_t job[3];
    const float* log_decay; const int32_t* lengths; const float* reset;
    int T, B, H, kv;
};

// The recurrence, one token after another: a workgroup holds the state columns [64 z, 64 z + 64) of one row, head and job.
template <typename E>
__global__ void __launch_bounds__(256) linattn_mix_kernel(mix_t p) {
    const mix_job_t& J = p.job[blockIdx.y];
    const int bh = blockIdx.x, b = bh / p.H, h = bh % p.H;
    const int col = threadIdx.x & 63, grp = threadIdx.x >> 6, e = blockIdx.z * 64 + col;
    if ((int)blockIdx.z * 64 >= J.dc) return;
    __shared__ float la[128], lb[128], part[4][64];
    const int n = p.lengths ? min(max(p.lengths[b], 0), p.T) : p.T;
    const float lam = expf(fminf(p.log_decay[h], 0.f));
    const bool own = e < J.dc;
    float s[32];
#pragma unroll
    for (int m = 0; m < 32; ++m) {
        const int d = grp + 4 * m;
        s[m] = (J.s_in && own && d < J.da) ? J.s_in[(size_t)bh * p.kv + (size_t)d * J.sd + (size_t)e * J.se] : 0.f;
    }
    const E* pa = (const E*)J.a + b * J.sa[1] + h * J.sa[2];
    const E* pb = (const E*)J.b + b * J.sb[1] + h * J.sb[2];
    const E* pc = (const E*)J.c + b * J.sc[1] + h * J.sc[2];
    E* po = (E*)J.out + b * J.so[1] + h * J.so[2];
    // off = 1: S decays before every token; off = 0 (reversed time): S_in meets the first token as it is, and S leaves decayed
    for (int i = 0; i < n; ++i) {
        const int64_t t = J.reverse ? n - 1 - i : i;
        __syncthreads();
        if (threadIdx.x < 128) la[threadIdx.x] = threadIdx.x < J.da ? io_load(pa + t * J.sa[0] + threadIdx.x) : 0.f;
        else lb[threadIdx.x - 128] = threadIdx.x - 128 < J.da ? io_load(pb + t * J.sb[0] + threadIdx.x - 128) : 0.f;
        const float c = own ? io_load(pc + t * J.sc[0] + e) : 0.f;
        // a reset before step t cuts t off from what came before; in reversed time from what came after: the reset of step t + 1
        const int64_t rt = J.reverse ? t + 1 : t;
        const bool cut = p.reset && rt < n && p.reset[rt * p.B + b] != 0.f;
        const float keep = cut ? 0.f : (J.off == 1 || i > 0) ? lam : 1.f;
        __syncthreads();
        float acc_p = 0.f, acc_s = 0.f;
#pragma unroll
        for (int m = 0; m < 32; ++m) {
            const int d = grp + 4 * m;
            const float prev = cut ? 0.f : keep * s[m], now = lb[d] * c;
            acc_s += la[d] * prev;
            acc_p += la[d] * now;
            s[m] = prev + J.scale_b * now;
        }
        part[grp][col] = J.scale_s * acc_s + J.scale_p * acc_p;
        __syncthreads();
        if (grp == 0 && own) io_store(po + t * J.so[0] + e, (part[0][col] + part[1][col]) + (part[2][col] + part[3][col]));
    }
    for (int64_t t = n; t < p.T; ++t)
        if (grp == 0 && own) io_store(po + t * J.so[0] + e, 0.f);
    if (J.s_out && own) {
        const float last = (J.off == 0 && n > 0) ? ((p.reset && p.reset[b] != 0.f) ? 0.f : lam) : 1.f;
#pragma unroll
        for (int m = 0; m < 32; ++m) {
            const int d = grp + 4 * m;
            if (d < J.da) J.s_out[(size_t)bh * p.kv + (size_t)d * J.sd + (size_t)e * J.se] = last == 0.f ? 0.f : last * s[m];
        }
    }
}

// One token: read S, decay, add k (x) v, read out with q, write S.  A workgroup takes one row and head; thread = 4 columns of S.
template <typename E, bool VEC>
__global__ void __launch_bounds__(256) linattn_step_kernel(xrl_linattn_t p) {
    __shared__ f32x4_t part[256];
    const int bh = blockIdx.x, b = bh / p.H, h = bh % p.H;
    const int nc = (p.dv + 3) >> 2, groups = blockDim.x / nc;
    const int c4 = threadIdx.x % nc, g = threadIdx.x / nc;
    const float lam = expf(fminf(p.log_decay[h], 0.f));
    const bool cut = p.reset && p.reset[b] != 0.f;
    const E* q = (const E*)p.q + b * p.stride_q[1] + h * p.stride_q[2];
    const E* k = (const E*)p.k + b * p.stride_k[1] + h * p.stride_k[2];
    const E* v = (const E*)p.v + b * p.stride_v[1] + h * p.stride_v[2];
    f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
    if (g < groups) {
        f32x4_t vv;
#pragma unroll
        for (int m = 0; m < 4; ++m) vv[m] = 4 * c4 + m < p.dv ? io_load(v + 4 * c4 + m) : 0.f;
        for (int d = g; d < p.dk; d += groups) {
            const int64_t at = ((int64_t)bh * p.dk + d) * p.dv + 4 * c4;
            f32x4_t s = {0.f, 0.f, 0.f, 0.f};
            if (!cut) {
                if (VEC) s = *reinterpret_cast<const f32x4_t*>(p.state + at);
                else
#pragma unroll
                    for (int m = 0; m < 4; ++m) s[m] = 4 * c4 + m < p.dv ? p.state[at + m] : 0.f;
            }
            const float kd = io_load(k + d), qd = io_load(q + d);
#pragma unroll
            for (int m = 0; m < 4; ++m) { s[m] = lam * s[m] + kd * vv[m]; acc[m] += qd * s[m]; }
            if (VEC) *reinterpret_cast<f32x4_t*>(p.state_out + at) = s;
            else
#pragma unroll
                for (int m = 0; m < 4; ++m)
                    if (4 * c4 + m < p.dv) p.state_out[at + m] = s[m];
        }
    }
    part[threadIdx.x] = acc;
    __syncthreads();
    if ((int)threadIdx.x < p.dv) {
        float o = 0.f;
        for (int r = 0; r < groups; ++r) o += part[r * nc + (threadIdx.x >> 2)][threadIdx.x & 3];
        io_store((E*)p.out + b * p.stride_out[1] + h * p.stride_out[2] + threadIdx.x, p.scale * o);
    }
}

static int check_sizes(const xrl_linattn_t& p) {
    XRL_CHECK_ARG(p.T >= 0 && p.B >= 0 && p.H >= 1 && p.dk >= 1 && p.dk <= 128 && p.dv >= 1 && p.dv <= 128);
    XRL_CHECK_ARG((int64_t)p.B * p.H <= 0x7fffffff);
    XRL_CHECK_ARG(p.dtype == XRL_F32 || p.dtype == XRL_BF16);
    return XRL_OK;
}

static void set_strides(int64_t* d, const int64_t* s) { d[0] = s[0]; d[1] = s[1]; d[2] = s[2]; }

static mix_job_t forward_job(const xrl_linattn_t& p) {
    mix_job_t j{};
    j.a = p.q; j.b = p.k; j.c = p.v; j.out = p.out;
    set_strides(j.sa, p.stride_q); set_strides(j.sb, p.stride_k); set_strides(j.sc, p.stride_v); set_strides(j.so, p.stride_out);
    j.da = p.dk; j.dc = p.dv; j.s_in = p.state; j.s_out = p.state_out; j.sd = p.dv; j.se = 1;
    j.off = 1; j.scale_p = j.scale_s = p.scale; j.scale_b = 1.f;
    return j;
}

static void backward_jobs(const xrl_linattn_t& p, mix_job_t* j) {
    mix_job_t& q = j[0];
    q.a = p.d_out; q.b = p.v; q.c = p.k; q.out = p.d_q;
    set_strides(q.sa, p.stride_d_out); set_strides(q.sb, p.stride_v); set_strides(q.sc, p.stride_k); set_strides(q.so, p.stride_d_q);
    q.da = p.dv; q.dc = p.dk; q.s_in = p.state; q.sd = 1; q.se = p.dv;
    q.off = 1; q.scale_p = q.scale_s = p.scale; q.scale_b = 1.f;
    mix_job_t& k = j[1];
    k.a = p.v; k.b = p.d_out; k.c = p.q; k.out = p.d_k;
    set_strides(k.sa, p.stride_v); set_strides(k.sb, p.stride_d_out); set_strides(k.sc, p.stride_q); set_strides(k.so, p.stride_d_k);
    k.da = p.dv; k.dc = p.dk; k.s_in = p.d_state_out; k.sd = 1; k.se = p.dv;
    k.reverse = 1; k.off = 0; k.scale_p = k.scale_b = p.scale; k.scale_s = 1.f;
    mix_job_t& v = j[2];
    v.a = p.k; v.b = p.q; v.c = p.d_out; v.out = p.d_v;
    set_strides(v.sa, p.stride_k); set_strides(v.sb, p.stride_q); set_strides(v.sc, p.stride_d_out); set_strides(v.so, p.stride_d_v);
    v.da = p.dk; v.dc = p.dv; v.s_in = p.d_state_out; v.s_out = p.d_state; v.sd = p.dv; v.se = 1;
    v.reverse = 1; v.off = 0; v.scale_p = v.scale_b = p.scale; v.scale_s = 1.f;
}

static int run_jobs(const xrl_linattn_t& p, mix_t& m, int n_jobs, xrl_stream_t stream) {
    m.log_decay = p.log_decay; m.lengths = p.lengths; m.reset = p.reset;
    m.T = p.T; m.B = p.B; m.H = p.H; m.kv = p.dk * p.dv;
    const dim3 grid(p.B * p.H, n_jobs, 2);
    if (p.dtype == XRL_F32) hipLaunchKernelGGL(linattn_mix_kernel<float>, grid, dim3(256), 0, as_stream(stream), m);
    else hipLaunchKernelGGL(linattn_mix_kernel<bf16_t>, grid, dim3(256), 0, as_stream(stream), m);
    XRL_CHECK_LAUNCH();
    return XRL_OK;
}

}  // namespace xrl

using namespace xrl;

extern "C" int64_t xrl_linattn_workspace_floats(const xrl_linattn_t* p, int backward) {
    (void)backward;
    if (!p || check_sizes(*p)) return XRL_EINVAL;
    return 0;
}

extern "C" int xrl_linattn_forward(const xrl_linattn_t* pp, xrl_stream_t stream) {
    XRL_CHECK_ARG(pp != nullptr);
    const xrl_linattn_t& p = *pp;
    if (int rc = check_sizes(p)) return rc;
    XRL_CHECK_ARG(p.log_decay && (p.T == 0 || p.B == 0 || (p.q && p.k && p.v && p.out)));
    if (p.B == 0) return XRL_OK;
    mix_t m{};
    m.job[0] = forward_job(p);
    return run_jobs(p, m, 1, stream);
}

extern "C" int xrl_linattn_backward(const xrl_linattn_t* pp, xrl_stream_t stream) {
    XRL_CHECK_ARG(pp != nullptr);
    const xrl_linattn_t& p = *pp;
    if (int rc = check_sizes(p)) return rc;
    XRL_CHECK_ARG(p.log_decay && (p.T == 0 || p.B == 0 || (p.q && p.k && p.v && p.d_out && p.d_q && p.d_k && p.d_v)));
    XRL_CHECK_ARG(!p.d_state || p.d_state != p.d_state_out);         // d_k's job reads d_state_out while d_v's writes d_state
    if (p.B == 0) return XRL_OK;
    mix_t m{};
    backward_jobs(p, m.job);
    return run_jobs(p, m, 3, stream);
}

extern "C" int xrl_linattn_step(const xrl_linattn_t* pp, xrl_stream_t stream) {
    XRL_CHECK_ARG(pp != nullptr);
    const xrl_linattn_t& p = *pp;
    if (int rc = check_sizes(p)) return rc;
    XRL_CHECK_ARG(p.T == 1);
    if (p.B == 0) return XRL_OK;
    XRL_CHECK_ARG(p.q && p.k && p.v && p.out && p.log_decay && p.state && p.state_out);
    const bool vec = p.dv % 4 == 0 && ((reinterpret_cast<uintptr_t>(p.state) | reinterpret_cast<uintptr_t>(p.state_out)) & 15) == 0;
    const int threads = 256;
    const dim3 grid(p.B * p.H);
    if (p.dtype == XRL_F32) {
        if (vec) hipLaunchKernelGGL((linattn_step_kernel<float, true>), grid, dim3(threads), 0, as_stream(stream), p);
        else hipLaunchKernelGGL((linattn_step_kernel<float, false>), grid, dim3(threads), 0, as_stream(stream), p);
    } else {
        if (vec) hipLaunchKernelGGL((linattn_step_kernel<bf16_t, true>), grid, dim3(threads), 0, as_stream(stream), p);
        else hipLaunchKernelGGL((linattn_step_kernel<bf16_t, false>), grid, dim3(threads), 0, as_stream(stream), p);
    }
    XRL_CHECK_LAUNCH();
    return XRL_OK;
}
