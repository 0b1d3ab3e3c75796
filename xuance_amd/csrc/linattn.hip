// Linear attention with one decay per head (include/xrl_hip.h: xrl_linattn_*): whole sequences, their gradients, one acting step.
//
// One operator carries all of it.  With a_i, b_j of width da and c_j of width dc,
//     mix_i = sum_{j <= i, same segment} lam^(i-j) (a_i . b_j) c_j + lam^(i+off) a_i S_in,     S: [da][dc]
// is the forward pass for (a, b, c) = (q, k, v) and the gradients for
//     d_q: (d_out, v, k), S_in = state^T;     d_k: (v, d_out, q) and d_v: (k, q, d_out) in reversed time, S_in = d_state_out(^T), off = 0,
// because S_t meets d S_t exactly where o_t meets q_t.  A launch runs one job (forward) or three (backward) of it.
#include "args.h"
#include "linattn_mix.h"

namespace xrl {

// The segments of a split time axis joined: every segment's own state becomes the state before it, S_in carried on past the last one is s_out.
struct scan_job_t {
    float* states; const float* carry;            // [row and head][segment][kv], [row and head][segment][2]
    const float* s_in; float* s_out;              // NULL or [B][H][.][.]
    int dc, sd, se;
    int stop_at_first;                            // s_out is 0 where the first step has a reset (reversed time)
};
struct scan_t {
    scan_job_t job[2];
    const float* reset; const int32_t* lengths;
    int T, H, kv, n_seg;
};

// Bound by memory, a read and a write of every state: 8 x 64 states of 128 x 128, 67 MB, 20 us (all requested at once: the same).
__global__ void __launch_bounds__(256) linattn_scan_kernel(scan_t p) {
    const scan_job_t& J = p.job[blockIdx.z];
    const int bh = blockIdx.y, x = blockIdx.x * 256 + threadIdx.x;
    if (x >= p.kv) return;
    const int64_t at = (int64_t)bh * p.kv + (int64_t)(x / J.dc) * J.sd + (int64_t)(x % J.dc) * J.se;
    float* s = J.states + (int64_t)bh * p.n_seg * p.kv + x;
    const float* c = J.carry + (int64_t)bh * p.n_seg * 2;
    float cur = J.s_in ? J.s_in[at] : 0.f;
    for (int i = 0; i < p.n_seg; i += 8) {
        float own[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) own[q] = i + q < p.n_seg ? s[(int64_t)(i + q) * p.kv] : 0.f;
#pragma unroll
        for (int q = 0; q < 8; ++q)
            if (i + q < p.n_seg) {
                s[(int64_t)(i + q) * p.kv] = cur;
                const float keep = c[2 * (i + q)];
                cur = keep < 0.f ? own[q] : __builtin_fmaf(cur, keep, cur * c[2 * (i + q) + 1]) + own[q];
            }
    }
    if (J.s_out) {
        const int b = bh / p.H;
        const bool none = J.stop_at_first && p.reset && p.reset[b] != 0.f && p.T > 0 && (!p.lengths || p.lengths[b] > 0);
        J.s_out[at] = none ? 0.f : cur;
    }
}

// One token: read S, decay, add k (x) v, read out with q, write S.  A workgroup takes one row and head; thread = 4 columns of S.
// Bound by memory, the state in and out: 4096 rows, 4 heads of 64 x 64, 537 MB in 98 us, 5.5 TB/s.
template <typename E, bool VEC>
__global__ void __launch_bounds__(256) linattn_step_kernel(xrl_linattn_t p) {
    __shared__ f32x4_t part[256];
    const int bh = blockIdx.x, b = bh / p.H, h = bh % p.H;
    const int nc = (p.dv + 3) >> 2, groups = blockDim.x / nc;
    const int c4 = threadIdx.x % nc, g = threadIdx.x / nc;
    // the decay as two floats, as in the sequence form: of a long memory one alone is off by a fair part of what it forgets (-1e-6: 1.3 %)
    const float gl = p.log_decay[h];
    const double decay = exp((double)(gl > 0.f ? 0.f : gl < -1e30f ? -1e30f : gl));
    const float lam = (float)decay, lam_low = (float)(decay - (double)lam);
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
            for (int m = 0; m < 4; ++m) {
                s[m] = __builtin_fmaf(s[m], lam, __builtin_fmaf(s[m], lam_low, kd * vv[m]));
                acc[m] += qd * s[m];
            }
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
    XRL_CHECK_ARG((int64_t)p.B * p.H <= 1 << 24);
    XRL_CHECK_ARG(p.dtype == XRL_F32 || p.dtype == XRL_BF16);
    return XRL_OK;
}

static void set_strides(int64_t* d, const int64_t* s) { d[0] = s[0]; d[1] = s[1]; d[2] = s[2]; }

static arg_t rows_arg(const char* name, const xrl_linattn_t& p, const void* ptr, const int64_t* s, int d, bool out) {
    return arg_t{name, ptr, p.dtype == XRL_F32 ? 4 : 2, 4, {p.T, p.B, p.H, d}, {s[0], s[1], s[2], 1}, out};
}
static arg_t dense_arg(const char* name, const void* ptr, int64_t n, bool out) { return arg_t{name, ptr, 4, 1, {n}, {1}, out}; }

static int check_tensors(const xrl_linattn_t& p, bool backward) {
    const int64_t states = (int64_t)p.B * p.H * p.dk * p.dv;
    const arg_t q = rows_arg("q", p, p.q, p.stride_q, p.dk, false), k = rows_arg("k", p, p.k, p.stride_k, p.dk, false),
                v = rows_arg("v", p, p.v, p.stride_v, p.dv, false), state = dense_arg("state", p.state, states, false),
                decay = dense_arg("log_decay", p.log_decay, p.H, false), reset = dense_arg("reset", p.reset, (int64_t)p.T * p.B, false),
                lengths = dense_arg("lengths", p.lengths, p.B, false);
    const int64_t ws = p.workspace ? p.workspace_floats : 0;
    if (!backward) {
        const arg_t a[] = {rows_arg("out", p, p.out, p.stride_out, p.dv, true), dense_arg("state_out", p.state_out, states, true),
                           dense_arg("workspace", p.workspace, ws, true), q, k, v, state, decay, reset, lengths};
        const int pairs[][2] = {{1, 6}};
        return check_args(a, 10, pairs, 1);
    }
    const arg_t a[] = {rows_arg("d_q", p, p.d_q, p.stride_d_q, p.dk, true), rows_arg("d_k", p, p.d_k, p.stride_d_k, p.dk, true),
                       rows_arg("d_v", p, p.d_v, p.stride_d_v, p.dv, true), dense_arg("d_state", p.d_state, states, true),
                       dense_arg("workspace", p.workspace, ws, true), q, k, v, rows_arg("d_out", p, p.d_out, p.stride_d_out, p.dv, false),
                       state, dense_arg("d_state_out", p.d_state_out, states, false), decay, reset, lengths};
    return check_args(a, 14, nullptr, 0);
}

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

// Segments that the time axis of every row is cut into, so that few rows fill the chip.  In units of one chunk's time, n segments cost
//     ceil(rows heads jobs n / slots) (chunks / n + 2)       the launch itself: its workgroups by turns, each its chunks and its start,
//   + ceil(... states n / slots) (chunks / n + 2) / 2 + 3    for n > 1 the pass over the segments' own states, their joining and two launches,
//   + rows heads states n dk dv / 2^21                       and the states' way through memory;
// the cheapest n up to 64 is taken.  Measured, forward / backward in us, * where the rule goes:
//   8 rows, 8 heads, 4096 steps, 128 wide, bf16:    n = 1 367 / 379,  4 162 / 359,  8 153* / 371*,  16 176 / 404
//   1 row, 8 heads, 32768 steps, 128 wide, bf16:    16 281 / 389,  32 171 / 363 (21: 353*),  64 155* / 376,  128 182 / 426
//   2 rows, 4 heads, 8192 steps, 64 wide, f32:      1 719 / 724,  8 141 / 147,  16 80 / 112,  32 54* / 93*
//   16 rows, 8 heads, 1024 steps, 128 wide, bf16:   1 98 / 145*,  2 100 / 198,  4 92* / 212
// Backward the rule is up to 3 % from the best of these: a compute unit's second workgroup gains less than the rule's slots say.
static int segments(const xrl_linattn_t& p, int n_jobs) {
    const int64_t units = (int64_t)p.B * p.H, wide = p.dk > p.dv ? p.dk : p.dv, da = n_jobs > 1 ? wide : p.dk, dc = n_jobs > 1 ? wide : p.dv;
    const int chunks = (p.T + CH - 1) / CH, states = n_jobs > 1 ? 2 : 1;
    if (units == 0 || chunks < 8 || units * n_jobs >= 4096) return 1;
    const int64_t slots = 256 * (int64_t)(p.dtype == XRL_F32 ? mix_resident_f32((int)da, (int)dc) : mix_resident_bf16((int)da, (int)dc));
    int best = 1;
    double least = 0;
    for (int n = 1; n <= 64 && n <= chunks / 4; ++n) {
        const double each = (double)chunks / n + 2, turns = (double)((units * n_jobs * n + slots - 1) / slots), turns_s = (double)((units * states * n + slots - 1) / slots);
        const double cost = turns * each + (n > 1 ? turns_s * each / 2 + 3 + (double)(units * states * n * p.dk * p.dv) / (1 << 21) : 0);
        if (n == 1 || cost < least) { best = n; least = cost; }
    }
    return best;
}

static int64_t split_floats(const xrl_linattn_t& p, int n_seg, int n_states) {
    return n_seg > 1 ? (int64_t)n_states * p.B * p.H * n_seg * (p.dk * p.dv + 2) : 0;
}

static int launch(const xrl_linattn_t& p, const mix_t& m, hipStream_t s) {
    int da = 0, dc = 0;
    for (int i = 0; i < m.n_jobs; ++i) { da = da > m.job[i].da ? da : m.job[i].da; dc = dc > m.job[i].dc ? dc : m.job[i].dc; }
    return p.dtype == XRL_F32 ? launch_mix_f32(m, da, dc, s) : launch_mix_bf16(m, da, dc, s);
}

// jobs: the outputs to make; holder[i]: the job whose split states job i starts from, itself or one of the same state transposed
static int run_jobs(const xrl_linattn_t& p, mix_t& m, int n_jobs, const int* holder, hipStream_t s) {
    m.log_decay = p.log_decay; m.lengths = p.lengths; m.reset = p.reset;
    m.T = p.T; m.B = p.B; m.H = p.H; m.kv = p.dk * p.dv; m.n_jobs = n_jobs;
    m.n_seg = segments(p, n_jobs);
    for (int i = 0; i < n_jobs; ++i) m.job[i].s_row = m.kv;
    if (m.n_seg == 1) return launch(p, m, s);
    mix_t st = m;
    scan_t sc{};
    sc.reset = p.reset; sc.lengths = p.lengths; sc.T = p.T; sc.H = p.H; sc.kv = m.kv; sc.n_seg = m.n_seg;
    const int64_t bhs = (int64_t)p.B * p.H * m.n_seg;
    int n = 0, slot[3] = {0, 0, 0};
    for (int i = 0; i < n_jobs; ++i)
        if (holder[i] == i) slot[i] = n++;
    float* carries = p.workspace + n * bhs * m.kv;
    for (int i = 0; i < n_jobs; ++i) {
        if (holder[i] != i) continue;
        const mix_job_t& j = m.job[i];
        mix_job_t& t = st.job[slot[i]];
        t = j;
        t.s_in = nullptr;
        t.s_out = p.workspace + slot[i] * bhs * m.kv;
        t.carry = carries + slot[i] * bhs * 2;
        scan_job_t& q = sc.job[slot[i]];
        q.states = t.s_out; q.carry = t.carry; q.s_in = j.s_in; q.s_out = j.s_out; q.dc = j.dc; q.sd = j.sd; q.se = j.se; q.stop_at_first = j.off == 0;
    }
    st.n_jobs = n; st.states_only = 1;
    if (int rc = launch(p, st, s)) return rc;
    hipLaunchKernelGGL(linattn_scan_kernel, dim3((m.kv + 255) / 256, p.B * p.H, n), dim3(256), 0, s, sc);
    XRL_CHECK_LAUNCH();
    for (int i = 0; i < n_jobs; ++i) {
        mix_job_t& j = m.job[i];
        j.s_in = p.workspace + slot[holder[i]] * bhs * m.kv;
        if (holder[i] == i) { j.sd = j.dc; j.se = 1; }
        else { j.sd = 1; j.se = m.job[holder[i]].dc; }
    }
    return launch(p, m, s);
}

int init_linattn() {
    if (int rc = init_mix_f32()) return rc;
    return init_mix_bf16();
}

}  // namespace xrl

using namespace xrl;

extern "C" int64_t xrl_linattn_workspace_floats(const xrl_linattn_t* p, int backward) {
    if (!p || check_sizes(*p)) return XRL_EINVAL;
    return split_floats(*p, segments(*p, backward ? 3 : 1), backward ? 2 : 1);
}

extern "C" int xrl_linattn_forward(const xrl_linattn_t* pp, xrl_stream_t stream) {
    XRL_CHECK_ARG(pp != nullptr);
    const xrl_linattn_t& p = *pp;
    if (int rc = check_sizes(p)) return rc;
    XRL_CHECK_ARG(p.log_decay && (p.T == 0 || p.B == 0 || (p.q && p.k && p.v && p.out)));
    if (p.B == 0) return XRL_OK;
    if (int rc = check_tensors(p, false)) return rc;
    const int64_t need = xrl_linattn_workspace_floats(pp, 0);
    XRL_CHECK_ARG(need == 0 || (p.workspace && p.workspace_floats >= need));
    mix_t m{};
    m.job[0] = forward_job(p);
    const int holder[1] = {0};
    return run_jobs(p, m, 1, holder, as_stream(stream));
}

extern "C" int xrl_linattn_backward(const xrl_linattn_t* pp, xrl_stream_t stream) {
    XRL_CHECK_ARG(pp != nullptr);
    const xrl_linattn_t& p = *pp;
    if (int rc = check_sizes(p)) return rc;
    XRL_CHECK_ARG(p.log_decay && (p.T == 0 || p.B == 0 || (p.q && p.k && p.v && p.d_out && p.d_q && p.d_k && p.d_v)));
    if (p.B == 0) return XRL_OK;
    if (int rc = check_tensors(p, true)) return rc;                  // d_state is not d_state_out: d_k's job reads it while d_v's writes
    const int64_t need = xrl_linattn_workspace_floats(pp, 1);
    XRL_CHECK_ARG(need == 0 || (p.workspace && p.workspace_floats >= need));
    mix_t m{};
    backward_jobs(p, m.job);
    const int holder[3] = {0, 2, 2};                                 // d_k starts from the same states as d_v, transposed
    return run_jobs(p, m, 3, holder, as_stream(stream));
}

extern "C" int xrl_linattn_step(const xrl_linattn_t* pp, xrl_stream_t stream) {
    XRL_CHECK_ARG(pp != nullptr);
    const xrl_linattn_t& p = *pp;
    if (int rc = check_sizes(p)) return rc;
    XRL_CHECK_ARG(p.T == 1);
    if (p.B == 0) return XRL_OK;
    XRL_CHECK_ARG(p.q && p.k && p.v && p.out && p.log_decay && p.state && p.state_out);
    if (int rc = check_tensors(p, false)) return rc;
    const bool vec = p.dv % 4 == 0 && ((reinterpret_cast<uintptr_t>(p.state) | reinterpret_cast<uintptr_t>(p.state_out)) & 15) == 0;
    const int threads = 256;
    const int64_t most = p.H < 1 << 23 ? (1 << 23) / p.H : 1, e = p.dtype == XRL_F32 ? 4 : 2;       // rows of a launch, which takes under 2^32 threads
    XRL_CHECK_ARG(p.H < 1 << 24);
    for (int64_t first = 0; first < p.B; first += most) {
        xrl_linattn_t r = p;
        r.B = (int)(p.B - first < most ? p.B - first : most);
        r.q = (const char*)p.q + first * p.stride_q[1] * e;
        r.k = (const char*)p.k + first * p.stride_k[1] * e;
        r.v = (const char*)p.v + first * p.stride_v[1] * e;
        r.out = (char*)p.out + first * p.stride_out[1] * e;
        r.state = p.state + first * p.H * p.dk * p.dv;
        r.state_out = p.state_out + first * p.H * p.dk * p.dv;
        if (p.reset) r.reset = p.reset + first;
        const dim3 grid(r.B * r.H);
        if (p.dtype == XRL_F32) {
            if (vec) hipLaunchKernelGGL((linattn_step_kernel<float, true>), grid, dim3(threads), 0, as_stream(stream), r);
            else hipLaunchKernelGGL((linattn_step_kernel<float, false>), grid, dim3(threads), 0, as_stream(stream), r);
        } else {
            if (vec) hipLaunchKernelGGL((linattn_step_kernel<bf16_t, true>), grid, dim3(threads), 0, as_stream(stream), r);
            else hipLaunchKernelGGL((linattn_step_kernel<bf16_t, false>), grid, dim3(threads), 0, as_stream(stream), r);
        }
        XRL_CHECK_LAUNCH();
    }
    return XRL_OK;
}
