// The norms before and after a residual block, fused with the block's gate and residual scale (include/xrl_hip.h: xrl_block_norm_*).
//
//     p = norm(u) w_post + b_post,   y = x + scale act(gate) p,   n = norm(y) w_pre + b_pre
//
// Bound by memory: forward 3 reads + 2 writes, backward 5 reads + 3 writes of N x D values and nothing saved in between -- the backward
// pass recomputes p, y and both statistics from the x, u and gate it needs anyway.  A row lives in the registers of L lanes, 8 values
// each, from its one load to its one store; the parameters and the gradient sums over the rows stay in registers over all rows of a
// workgroup.  Those sums leave as one line of partials per workgroup and a second launch adds the lines in a fixed order (no atomics).
#include "args.h"
#include "io16.h"

namespace xrl {

constexpr int NV = 8;                  // values of a row per lane

// The build keeps products and sums apart (-ffp-contract=off); here they are fused by hand, a third of the vector instructions, which come close to
// the memory's time for 16-bit rows.
__device__ __forceinline__ float fma_f(float a, float b, float c) { return __builtin_fmaf(a, b, c); }

// act_apply_c with the sigmoid from v_exp_f32 and v_rcp_f32 (a unit in the last place each) instead of expf and a division
template <int ACT>
__device__ __forceinline__ float gate_act_c(float z) {
    if (ACT == XRL_ACT_SIGMOID) return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * z));
    return act_apply_c<ACT>(z);
}
constexpr int NORM_SUMS = 5;           // d_scale, d_w_post, d_b_post, d_w_pre, d_b_pre

template <int L>
struct norm_geom {
    static constexpr int THREADS = L < 256 ? (L > 64 ? L : 256) : L;
    static constexpr int ROWS = L > 64 ? 1 : THREADS / L;        // rows of a workgroup at a time
    static constexpr int WAVES = THREADS / 64;
};

// eight neighbouring values of a row as they are stored; absent ones 0
template <typename E>
struct row8 {
    static constexpr int PER = row16<E>::PER, N = NV / PER;
    u32x4_t v[N];
    __device__ __forceinline__ void load(const E* row, int at, int D) {
        typedef row16<E> R;
#pragma unroll
        for (int q = 0; q < N; ++q) { const u32x4_t zero = {0, 0, 0, 0}; v[q] = zero; }
        if (at + NV <= D) {
#pragma unroll
            for (int q = 0; q < N; ++q) v[q] = R::load(row + at + PER * q);
        } else if (at < D) {
#pragma unroll
            for (int m = 0; m < NV; ++m)
                if (at + m < D) R::put(v[m / PER], m % PER, R::bits(row + at + m));
        }
    }
    __device__ __forceinline__ void get(float (&f)[NV]) const {
#pragma unroll
        for (int m = 0; m < NV; ++m) f[m] = row16<E>::get(v[m / PER], m % PER);
    }
    static __device__ __forceinline__ void store(E* row, int at, int D, const float (&f)[NV]) {
        typedef row16<E> R;
        if (at + NV <= D) {
#pragma unroll
            for (int q = 0; q < N; ++q) R::store(row + at + PER * q, R::pack(f + PER * q));
        } else if (at < D) {
#pragma unroll
            for (int m = 0; m < NV; ++m)
                if (at + m < D) io_store(row + at + m, f[m]);
        }
    }
};

__device__ __forceinline__ void norm_param(const float* p, int at, int D, float missing, float (&v)[NV]) {
#pragma unroll
    for (int m = 0; m < NV; ++m) v[m] = at + m < D ? (p ? p[at + m] : missing) : 0.f;
}

// Sums over the L lanes of a row.  Across waves through LDS with one barrier: consecutive sums use other slots of `scratch`, and a slot
// comes round again only two barriers later.
template <int L>
struct row_sum_t {
    float2 (*scratch)[16];
    int slot;
    __device__ __forceinline__ float2 operator()(float a, float b) {
#pragma unroll
        for (int off = (L < 64 ? L : 64) / 2; off > 0; off >>= 1) { a += __shfl_xor(a, off, 64); b += __shfl_xor(b, off, 64); }
        if (L > 64) {
            const int w = threadIdx.x >> 6;
            slot = slot == 2 ? 0 : slot + 1;
            if ((threadIdx.x & 63) == 0) scratch[slot][w] = make_float2(a, b);
            __syncthreads();
            a = b = 0.f;
#pragma unroll
            for (int i = 0; i < L / 64; ++i) { a += scratch[slot][i].x; b += scratch[slot][i].y; }
        }
        return make_float2(a, b);
    }
    __device__ __forceinline__ float operator()(float a) {
#pragma unroll
        for (int off = (L < 64 ? L : 64) / 2; off > 0; off >>= 1) a += __shfl_xor(a, off, 64);
        if (L > 64) {
            const int w = threadIdx.x >> 6;
            slot = slot == 2 ? 0 : slot + 1;
            if ((threadIdx.x & 63) == 0) scratch[slot][w].x = a;
            __syncthreads();
            a = 0.f;
#pragma unroll
            for (int i = 0; i < L / 64; ++i) a += scratch[slot][i].x;
        }
        return a;
    }
};

// v := (v - mean) r (layer) or v r; returns r.  The variance is taken of the centred values (no difference of large sums).
template <int L, bool LN>
__device__ __forceinline__ float normalize(float (&v)[NV], int at, int D, float inv_d, float eps, row_sum_t<L>& sum) {
    if (LN) {
        float s = 0.f;
#pragma unroll
        for (int m = 0; m < NV; ++m) s += v[m];
        const float mean = sum(s) * inv_d;
#pragma unroll
        for (int m = 0; m < NV; ++m) v[m] = at + m < D ? v[m] - mean : 0.f;
    }
    float q = 0.f;
#pragma unroll
    for (int m = 0; m < NV; ++m) q = fma_f(v[m], v[m], q);
    const float r = 1.f / sqrtf(fma_f(sum(q), inv_d, eps));
#pragma unroll
    for (int m = 0; m < NV; ++m) v[m] *= r;
    return r;
}

template <typename E, int L, bool LN>
__global__ void __launch_bounds__(norm_geom<L>::THREADS) block_norm_fwd_kernel(xrl_block_norm_t p) {
    using G = norm_geom<L>;
    __shared__ float2 scratch[3][16];
    row_sum_t<L> sum{scratch, 0};
    const int lane = threadIdx.x % L, at = lane * NV, D = p.D;
    const float inv_d = 1.f / (float)D;
    float sc[NV], w0[NV], b0[NV], w1[NV], b1[NV];
    norm_param(p.scale, at, D, 1.f, sc);
    norm_param(p.w_post, at, D, 1.f, w0);
    norm_param(p.b_post, at, D, 0.f, b0);
    norm_param(p.w_pre, at, D, 1.f, w1);
    norm_param(p.b_pre, at, D, 0.f, b1);
    row8<E> rx, ru, rg;
    auto request = [&](int64_t row) {
        const int width = row < p.N ? D : 0;
        ru.load((const E*)p.u + row * p.ld_u, at, width);
        rx.load((const E*)p.x + row * p.ld_x, at, width);
        if (p.gate) rg.load((const E*)p.gate + row * p.ld_gate, at, width);
    };
    constexpr bool AHEAD = L < 1024;                                 // 1024 threads leave no registers for it
    if (AHEAD) request((int64_t)blockIdx.x * G::ROWS + threadIdx.x / L);
    const int64_t step = (int64_t)gridDim.x * G::ROWS;
    for (int64_t base = (int64_t)blockIdx.x * G::ROWS; base < p.N; base += step) {       // whole workgroups go round: barriers inside
        const int64_t row = base + threadIdx.x / L;
        const bool live = row < p.N;
        float x[NV], u[NV], g[NV] = {};
        if (!AHEAD) request(row);
        ru.get(u); rx.get(x);
        if (p.gate) rg.get(g);
        if (AHEAD && base + step < p.N) request(row + step);         // the next row is on its way while this one is worked on
        normalize<L, LN>(u, at, D, inv_d, p.eps, sum);
        if (p.gate) {
            XRL_ACT_DISPATCH(p.gate_act, _Pragma("unroll") for (int m = 0; m < NV; ++m) g[m] = gate_act_c<ACT>(g[m]);)
        }
#pragma unroll
        for (int m = 0; m < NV; ++m) {
            const float b = fma_f(u[m], w0[m], b0[m]);
            x[m] = fma_f(p.gate ? g[m] * sc[m] : sc[m], b, x[m]);
        }
        if (live) row8<E>::store((E*)p.y + row * p.ld_y, at, D, x);
        if (p.n) {
            normalize<L, LN>(x, at, D, inv_d, p.eps, sum);
#pragma unroll
            for (int m = 0; m < NV; ++m) x[m] = fma_f(x[m], w1[m], b1[m]);
            if (live) row8<E>::store((E*)p.n + row * p.ld_n, at, D, x);
        }
    }
}

// d := r (d - xhat mean(d xhat) [- mean(d)]): gradient through the normalisation
template <int L, bool LN>
__device__ __forceinline__ void normalize_back(float (&d)[NV], const float (&xhat)[NV], float r, int at, int D, float inv_d,
                                               row_sum_t<L>& sum) {
    float a = 0.f, b = 0.f;
#pragma unroll
    for (int m = 0; m < NV; ++m) { a = fma_f(d[m], xhat[m], a); if (LN) b += d[m]; }
    if (LN) { const float2 t = sum(a, b); a = t.x * inv_d; b = t.y * inv_d; }
    else a = sum(a) * inv_d;
#pragma unroll
    for (int m = 0; m < NV; ++m) d[m] = at + m < D ? r * fma_f(-xhat[m], a, LN ? d[m] - b : d[m]) : 0.f;
}

template <typename E, int L, bool LN>
__global__ void __launch_bounds__(norm_geom<L>::THREADS) block_norm_bwd_kernel(xrl_block_norm_t p) {
    using G = norm_geom<L>;
    __shared__ float2 scratch[3][16];
    row_sum_t<L> sum{scratch, 0};
    const int lane = threadIdx.x % L, at = lane * NV, D = p.D;
    const float inv_d = 1.f / (float)D;
    float sc[NV], w0[NV], b0[NV], w1[NV];
    norm_param(p.scale, at, D, 1.f, sc);
    norm_param(p.w_post, at, D, 1.f, w0);
    norm_param(p.b_post, at, D, 0.f, b0);
    norm_param(p.w_pre, at, D, 1.f, w1);
    float acc[NORM_SUMS][NV] = {};
    // the next row is on its way while this one is worked on; 1024 threads leave no registers for that
    constexpr bool AHEAD = L < 1024;
    row8<E> rx, ru_, rg, ry_, rn;
    auto request = [&](int64_t row) {
        const int width = row < p.N ? D : 0;
        ru_.load((const E*)p.u + row * p.ld_u, at, width);
        rx.load((const E*)p.x + row * p.ld_x, at, width);
        if (p.gate) rg.load((const E*)p.gate + row * p.ld_gate, at, width);
        if (p.d_y) ry_.load((const E*)p.d_y + row * p.ld_d_y, at, width);
        if (p.d_n) rn.load((const E*)p.d_n + row * p.ld_d_n, at, width);
    };
    if (AHEAD) request((int64_t)blockIdx.x * G::ROWS + threadIdx.x / L);
    const int64_t step = (int64_t)gridDim.x * G::ROWS;
    for (int64_t base = (int64_t)blockIdx.x * G::ROWS; base < p.N; base += step) {
        const int64_t row = base + threadIdx.x / L;
        const bool live = row < p.N;
        float x[NV], u[NV], g[NV] = {}, dy[NV] = {}, dn[NV] = {}, t[NV];
        if (!AHEAD) request(row);
        ru_.get(u); rx.get(x);
        if (p.gate) rg.get(g);
        if (p.d_y) ry_.get(dy);
        if (p.d_n) rn.get(dn);
        if (AHEAD && base + step < p.N) request(row + step);
        const float ru = normalize<L, LN>(u, at, D, inv_d, p.eps, sum);
        if (p.gate) {
            XRL_ACT_DISPATCH(p.gate_act, _Pragma("unroll") for (int m = 0; m < NV; ++m) g[m] = gate_act_c<ACT>(g[m]);)
        }
        float pm[NV];                                                // the normed block before gate and scale
#pragma unroll
        for (int m = 0; m < NV; ++m) pm[m] = fma_f(u[m], w0[m], b0[m]);
        if (p.d_n) {
#pragma unroll
            for (int m = 0; m < NV; ++m) x[m] = fma_f(p.gate ? g[m] * sc[m] : sc[m], pm[m], x[m]);
            const float ry = normalize<L, LN>(x, at, D, inv_d, p.eps, sum);
#pragma unroll
            for (int m = 0; m < NV; ++m) { acc[3][m] = fma_f(dn[m], x[m], acc[3][m]); acc[4][m] += dn[m]; t[m] = dn[m] * w1[m]; }
            normalize_back<L, LN>(t, x, ry, at, D, inv_d, sum);
#pragma unroll
            for (int m = 0; m < NV; ++m) dy[m] += t[m];
        }
        if (live) row8<E>::store((E*)p.d_x + row * p.ld_d_x, at, D, dy);
        // y = x + scale a p: with a the activated gate
#pragma unroll
        for (int m = 0; m < NV; ++m) {
            const float da = p.gate ? dy[m] * g[m] : dy[m], dp = da * sc[m];
            acc[0][m] = fma_f(da, pm[m], acc[0][m]);
            acc[1][m] = fma_f(dp, u[m], acc[1][m]);
            acc[2][m] += dp;
            t[m] = dp * w0[m];
            dy[m] *= sc[m] * pm[m];                                  // gradient of the activated gate
        }
        if (p.d_gate) {
            XRL_ACT_DISPATCH(p.gate_act, _Pragma("unroll") for (int m = 0; m < NV; ++m) g[m] = dy[m] * act_grad_c<ACT>(g[m]);)
            if (live) row8<E>::store((E*)p.d_gate + row * p.ld_d_gate, at, D, g);
        }
        normalize_back<L, LN>(t, u, ru, at, D, inv_d, sum);
        if (live) row8<E>::store((E*)p.d_u + row * p.ld_d_u, at, D, t);
    }
    // partial sums: over the rows of a wave, then over the waves (in wave order), one line per workgroup
    float* line = p.workspace + (size_t)blockIdx.x * NORM_SUMS * D;
    __shared__ float part[L > 64 ? 1 : G::WAVES][L > 64 ? 1 : L * NV];
#pragma unroll
    for (int s = 0; s < NORM_SUMS; ++s) {
        if (L < 64) {
#pragma unroll
            for (int off = L; off < 64; off <<= 1)
#pragma unroll
                for (int m = 0; m < NV; ++m) acc[s][m] += __shfl_xor(acc[s][m], off, 64);
        }
        if (L > 64) {
#pragma unroll
            for (int m = 0; m < NV; ++m) {
                if (at + m < D) line[s * D + at + m] = acc[s][m];
            }
        } else {
            __syncthreads();
            if ((int)(threadIdx.x & 63) < L) {
#pragma unroll
                for (int m = 0; m < NV; ++m) part[threadIdx.x >> 6][at + m] = acc[s][m];
            }
            __syncthreads();
            for (int e = threadIdx.x; e < D; e += G::THREADS) {
                float t = 0.f;
#pragma unroll
                for (int w = 0; w < G::WAVES; ++w) t += part[w][e];
                line[s * D + e] = t;
            }
        }
    }
}

// out[s][e] = sum of the workgroups' lines, 64 groups of lines a column, met in a fixed order
__global__ void __launch_bounds__(1024) block_norm_sums_kernel(xrl_block_norm_t p, int lines) {
    __shared__ float part[64][17];
    const int c = threadIdx.x & 15, r = threadIdx.x >> 4, width = NORM_SUMS * p.D;
    const int col = blockIdx.x * 16 + c;
    float t = 0.f;
    if (col < width)
        for (int i = r; i < lines; i += 64) t += p.workspace[(size_t)i * width + col];
    part[r][c] = t;
    __syncthreads();
    if (threadIdx.x < 16 && col < width) {
        float a = 0.f;
        for (int i = 0; i < 64; ++i) a += part[i][c];
        float* outs[NORM_SUMS] = {p.d_scale, p.d_w_post, p.d_b_post, p.d_w_pre, p.d_b_pre};
#pragma unroll
        for (int s = 0; s < NORM_SUMS; ++s)
            if (outs[s] && col / p.D == s) outs[s][col % p.D] = a;
    }
}

static int norm_lanes(int D) {
    int L = 8;
    while (L * NV < D) L *= 2;
    return L;
}

// workgroups of the backward pass: enough to fill the chip twice over, each with rows to keep its parameters and sums for
static int norm_lines(const xrl_block_norm_t& p) {
    const int L = norm_lanes(p.D), threads = L < 256 ? (L > 64 ? L : 256) : L, rows = L > 64 ? 1 : threads / L;
    const int64_t most = 512 * 256 / threads, need = (p.N + rows - 1) / rows;
    return (int)(need < most ? need : most);
}

static int check_norm(const xrl_block_norm_t& p) {
    XRL_CHECK_ARG(p.N >= 0 && p.D >= 1 && p.D <= 8192);
    XRL_CHECK_ARG((p.dtype == XRL_F32 || p.dtype == XRL_BF16) && (p.kind == XRL_NORM_RMS || p.kind == XRL_NORM_LAYER));
    XRL_CHECK_ARG(p.gate_act >= XRL_ACT_NONE && p.gate_act <= XRL_ACT_SIGMOID && p.eps > 0.f);
    return XRL_OK;
}

static int check_norm_tensors(const xrl_block_norm_t& p, bool backward) {
    const int e = p.dtype == XRL_F32 ? 4 : 2;
    auto rows = [&](const char* name, const void* ptr, int64_t ld, bool out) { return arg_t{name, ptr, e, 2, {p.N, p.D}, {ld, 1}, out}; };
    auto vec = [&](const char* name, const void* ptr, bool out) { return arg_t{name, ptr, 4, 1, {p.D}, {1}, out}; };
    const arg_t x = rows("x", p.x, p.ld_x, false), u = rows("u", p.u, p.ld_u, false), g = rows("gate", p.gate, p.ld_gate, false),
                sc = vec("scale", p.scale, false), w0 = vec("w_post", p.w_post, false), b0 = vec("b_post", p.b_post, false),
                w1 = vec("w_pre", p.w_pre, false), b1 = vec("b_pre", p.b_pre, false);
    if (!backward) {
        const arg_t a[] = {rows("y", p.y, p.ld_y, true), rows("n", p.n, p.ld_n, true), x, u, g, sc, w0, b0, w1, b1};
        const int pairs[][2] = {{0, 2}};
        return check_args(a, 10, pairs, 1);
    }
    const arg_t a[] = {rows("d_x", p.d_x, p.ld_d_x, true), rows("d_u", p.d_u, p.ld_d_u, true), rows("d_gate", p.d_gate, p.ld_d_gate, true),
                       vec("d_scale", p.d_scale, true), vec("d_w_post", p.d_w_post, true), vec("d_b_post", p.d_b_post, true),
                       vec("d_w_pre", p.d_w_pre, true), vec("d_b_pre", p.d_b_pre, true),
                       arg_t{"workspace", p.workspace, 4, 1, {p.workspace ? p.workspace_floats : 0}, {1}, true},
                       rows("d_y", p.d_y, p.ld_d_y, false), rows("d_n", p.d_n, p.ld_d_n, false), x, u, g, sc, w0, b0, w1, b1};
    const int pairs[][2] = {{0, 9}};
    return check_args(a, 19, pairs, 1);
}

template <typename E, bool LN>
static void launch_norm(const xrl_block_norm_t& p, bool backward, hipStream_t s) {
    const int L = norm_lanes(p.D);
#define NORM_CASE(LL)                                                                                                            \
    case LL: {                                                                                                                   \
        using G = norm_geom<LL>;                                                                                                 \
        if (backward) hipLaunchKernelGGL((block_norm_bwd_kernel<E, LL, LN>), dim3(norm_lines(p)), dim3(G::THREADS), 0, s, p); \
        else {                                                                                                                   \
            const int64_t need = (p.N + G::ROWS - 1) / G::ROWS, most = 1024 * 256 / G::THREADS;                                  \
            hipLaunchKernelGGL((block_norm_fwd_kernel<E, LL, LN>), dim3((int)(need < most ? need : most)), dim3(G::THREADS), 0, s, p); \
        }                                                                                                                        \
    } break;
    switch (L) { NORM_CASE(8) NORM_CASE(16) NORM_CASE(32) NORM_CASE(64) NORM_CASE(128) NORM_CASE(256) NORM_CASE(512) NORM_CASE(1024) }
#undef NORM_CASE
}

static int run_norm(const xrl_block_norm_t& p, bool backward, hipStream_t s) {
    const bool ln = p.kind == XRL_NORM_LAYER;
    if (p.dtype == XRL_F32) { if (ln) launch_norm<float, true>(p, backward, s); else launch_norm<float, false>(p, backward, s); }
    else { if (ln) launch_norm<bf16_t, true>(p, backward, s); else launch_norm<bf16_t, false>(p, backward, s); }
    XRL_CHECK_LAUNCH();
    return XRL_OK;
}

}  // namespace xrl

using namespace xrl;

extern "C" int64_t xrl_block_norm_workspace_floats(const xrl_block_norm_t* p) {
    if (!p || check_norm(*p)) return XRL_EINVAL;
    return (int64_t)norm_lines(*p) * NORM_SUMS * p->D;
}

extern "C" int xrl_block_norm_forward(const xrl_block_norm_t* pp, xrl_stream_t stream) {
    XRL_CHECK_ARG(pp != nullptr);
    const xrl_block_norm_t& p = *pp;
    if (int rc = check_norm(p)) return rc;
    if (p.N == 0) return XRL_OK;
    XRL_CHECK_ARG(p.x && p.u && p.y);
    if (int rc = check_norm_tensors(p, false)) return rc;
    return run_norm(p, false, as_stream(stream));
}

extern "C" int xrl_block_norm_backward(const xrl_block_norm_t* pp, xrl_stream_t stream) {
    XRL_CHECK_ARG(pp != nullptr);
    const xrl_block_norm_t& p = *pp;
    if (int rc = check_norm(p)) return rc;
    XRL_CHECK_ARG(!p.d_gate || p.gate);
    XRL_CHECK_ARG(p.N == 0 || (p.x && p.u && p.d_x && p.d_u && (p.d_y || p.d_n) && p.workspace));
    XRL_CHECK_ARG(p.workspace_floats >= (int64_t)norm_lines(p) * NORM_SUMS * p.D);
    if (int rc = check_norm_tensors(p, true)) return rc;
    if (p.N > 0)
        if (int rc = run_norm(p, true, as_stream(stream))) return rc;
    if (p.d_scale || p.d_w_post || p.d_b_post || p.d_w_pre || p.d_b_pre) {
        hipLaunchKernelGGL(block_norm_sums_kernel, dim3((NORM_SUMS * p.D + 15) / 16), dim3(1024), 0, as_stream(stream), p, norm_lines(p));
        XRL_CHECK_LAUNCH();
    }
    return XRL_OK;
}
