// The norms before and after a residual block, fused with the block's gate and residual scale (include/xrl_hip.h: xrl_block_norm_*).
//
//     p = norm(u) w_post + b_post,   y = x + scale act(gate) p,   n = norm(y) w_pre + b_pre
//
// Bound by memory: forward 3 reads + 2 writes, backward 5 reads + 3 writes of N x D values and nothing saved in between -- the backward
// pass recomputes p, y and both statistics from the x, u and gate it needs anyway.  A row lives in the registers of L lanes, 8 values
// each, from its one load to its one store; the gradient sums over the rows stay in registers over all rows of a workgroup, the parameters in LDS.
// Those sums leave as one line of partials per workgroup and a second launch adds the lines in a fixed order (no atomics).
// Measured, forward and backward with its sums: 65536 x 256 f32 with a gate, rms 64 us (5.2 TB/s) and 110 us (4.9), as a copy; 30011 x 2048 bf16, layer,
// 131 us (4.7) and 216 us (4.6): a row of 2048 is four waves that meet six times, and the vector instructions of two or three rows a CU do not hide that.
#include "args.h"
#include "io16.h"
#include "lanes.h"

namespace xrl {

constexpr int NV = 8;                  // values of a row per lane

// The build keeps products and sums apart (-ffp-contract=off); here they are fused by hand, a third of the vector instructions, which come close to
// the memory's time for 16-bit rows.
__device__ __forceinline__ float fma_f(float a, float b, float c) { return __builtin_fmaf(a, b, c); }

// act_apply_c with the sigmoid a from v_exp_f32 and v_rcp_f32 (a unit in the last place each) instead of expf and a division.  The exponential's argument
// is rounded too, so a is off by up to ((1 - a) (1.5 |z| + 2) + 3) 2^-24 of itself: far out, where a is small, by |z| of its last places.
template <int ACT>
__device__ __forceinline__ float gate_act_c(float z) {
    if (ACT == XRL_ACT_SIGMOID) return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * z));
    return act_apply_c<ACT>(z);
}
// Sums over the rows, with a the activated gate, uhat and yhat the normalised u and y:  S0 = sum a d_y,  S1 = sum a d_y uhat,  S2 = sum d_n yhat,
// S3 = sum d_n.  They give d_scale = w_post S1 + b_post S0, d_w_post = scale S1, d_b_post = scale S0, d_w_pre = S2, d_b_pre = S3.  (Where w_post uhat
// and b_post cancel in p over all rows, d_scale is off by the roundings of uhat, which p has too, and by those of the two sums.)
constexpr int NORM_SUMS = 4;

// FULL below: rows of exactly 8 L values, without the checks of a row's end (30011 x 2048 bf16: with the sums by lanes.h 431 -> 386 us)
template <int L>
struct norm_geom {
    static constexpr int THREADS = L < 256 ? (L > 64 ? L : 256) : L;
    static constexpr int ROWS = L > 64 ? 1 : THREADS / L;        // rows of a workgroup at a time
    static constexpr int WAVES = THREADS / 64;
};

// eight neighbouring values of a row as they are stored; absent ones 0
template <typename E, bool FULL>
struct row8 {
    static constexpr int PER = row16<E>::PER, N = NV / PER;
    u32x4_t v[N];
    __device__ __forceinline__ void load(const E* row, int at, int D) {
        typedef row16<E> R;
#pragma unroll
        for (int q = 0; q < N; ++q) { const u32x4_t zero = {0, 0, 0, 0}; v[q] = zero; }
        if (FULL ? D > 0 : at + NV <= D) {
#pragma unroll
            for (int q = 0; q < N; ++q) v[q] = R::load(row + at + PER * q);
        } else if (!FULL && at < D) {
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
        if (FULL || at + NV <= D) {
#pragma unroll
            for (int q = 0; q < N; ++q) R::store(row + at + PER * q, R::pack(f + PER * q));
        } else if (at < D) {
#pragma unroll
            for (int m = 0; m < NV; ++m)
                if (at + m < D) io_store(row + at + m, f[m]);
        }
    }
};

// A row's parameters in LDS, 16 bytes a lane and read: kept in registers they would cost 8 each and with them every third or second wave.
template <int L>
struct norm_params {
    f32x4_t (*lds)[2][L];                                            // [parameter][half][lane]
    __device__ __forceinline__ void fill(int which, const float* p, float missing, int D) {
        for (int c = threadIdx.x; c < 2 * L; c += norm_geom<L>::THREADS) {
            const int half = c / L, l = c % L;
            f32x4_t v;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int e = l * NV + 4 * half + i;
                v[i] = e < D ? (p ? p[e] : missing) : 0.f;
            }
            lds[which][half][l] = v;
        }
    }
    __device__ __forceinline__ void get(int which, int lane, float (&v)[NV]) const {
        asm volatile("" : "+v"(lane));                               // read again for every use
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const f32x4_t q = lds[which][half][lane];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[4 * half + i] = q[i];
        }
    }
};

// Sums over the L lanes of a row.  Across waves through LDS with one barrier: consecutive sums use other slots of `scratch`, and a slot
// comes round again only two barriers later.
template <int L>
struct row_sum_t {
    float2 (*scratch)[16];
    int slot;
    __device__ __forceinline__ float2 operator()(float a, float b) {
        a = lane_sum<L < 64 ? L : 64>(a);
        b = lane_sum<L < 64 ? L : 64>(b);
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
        a = lane_sum<L < 64 ? L : 64>(a);
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
template <int L, bool LN, bool FULL>
__device__ __forceinline__ float normalize(float (&v)[NV], int at, int D, float inv_d, float eps, row_sum_t<L>& sum) {
    if (LN) {
        float s = 0.f;
#pragma unroll
        for (int m = 0; m < NV; ++m) s += v[m];
        const float mean = sum(s) * inv_d;
#pragma unroll
        for (int m = 0; m < NV; ++m) v[m] = FULL || at + m < D ? v[m] - mean : 0.f;
    }
    float q = 0.f;
#pragma unroll
    for (int m = 0; m < NV; ++m) q = fma_f(v[m], v[m], q);
    const float r = 1.f / sqrtf(fma_f(sum(q), inv_d, eps));
#pragma unroll
    for (int m = 0; m < NV; ++m) v[m] *= r;
    return r;
}

template <typename E, int L, bool LN, bool FULL>
__global__ void __launch_bounds__(norm_geom<L>::THREADS) block_norm_fwd_kernel(xrl_block_norm_t p) {
    using G = norm_geom<L>;
    __shared__ float2 scratch[3][16];
    row_sum_t<L> sum{scratch, 0};
    const int lane = threadIdx.x % L, at = lane * NV, D = p.D;
    const float inv_d = 1.f / (float)D;
    __shared__ f32x4_t pars[3][2][L];                                // the shifts in registers: five here, 40 KB for 2048 values, leave room for three waves
    norm_params<L> par{pars};
    par.fill(0, p.scale, 1.f, D); par.fill(1, p.w_post, 1.f, D); par.fill(2, p.w_pre, 1.f, D);
    float b0[NV], b1[NV];
#pragma unroll
    for (int m = 0; m < NV; ++m) {
        b0[m] = p.b_post && at + m < D ? p.b_post[at + m] : 0.f;
        b1[m] = p.b_pre && at + m < D ? p.b_pre[at + m] : 0.f;
    }
    __syncthreads();
    row8<E, FULL> rx, ru, rg;
    auto request = [&](int64_t row) {
        const int width = row < p.N ? D : 0;
        ru.load((const E*)p.u + row * p.ld_u, at, width);
        rx.load((const E*)p.x + row * p.ld_x, at, width);
        if (p.gate) rg.load((const E*)p.gate + row * p.ld_gate, at, width);
    };
    constexpr bool AHEAD = L < 1024;                                 // 1024 threads leave no registers for it; both passes of 2048 bf16: 471 -> 431 us
    if (AHEAD) request((int64_t)blockIdx.x * G::ROWS + threadIdx.x / L);
    const int64_t step = (int64_t)gridDim.x * G::ROWS;
    for (int64_t base = (int64_t)blockIdx.x * G::ROWS; base < p.N; base += step) {       // whole workgroups go round: barriers inside
        const int64_t row = base + threadIdx.x / L;
        const bool live = row < p.N;
        float x[NV], u[NV], g[NV];
        if (!AHEAD) request(row);
        ru.get(u); rx.get(x);
        if (p.gate) rg.get(g);
        if (AHEAD && base + step < p.N) request(row + step);         // the next row is on its way while this one is worked on
        normalize<L, LN, FULL>(u, at, D, inv_d, p.eps, sum);
        if (p.gate) {
            XRL_ACT_DISPATCH(p.gate_act, _Pragma("unroll") for (int m = 0; m < NV; ++m) g[m] = gate_act_c<ACT>(g[m]);)
        } else {
#pragma unroll
            for (int m = 0; m < NV; ++m) g[m] = 1.f;
        }
        float w[NV];
        par.get(1, lane, w);
#pragma unroll
        for (int m = 0; m < NV; ++m) u[m] = fma_f(u[m], w[m], b0[m]);
        par.get(0, lane, w);
#pragma unroll
        for (int m = 0; m < NV; ++m) x[m] = fma_f(g[m] * w[m], u[m], x[m]);
        if (live) row8<E, FULL>::store((E*)p.y + row * p.ld_y, at, D, x);
        if (p.n) {
            normalize<L, LN, FULL>(x, at, D, inv_d, p.eps, sum);
            par.get(2, lane, w);
#pragma unroll
            for (int m = 0; m < NV; ++m) x[m] = fma_f(x[m], w[m], b1[m]);
            if (live) row8<E, FULL>::store((E*)p.n + row * p.ld_n, at, D, x);
        }
    }
}

// d := r (d - xhat mean(d xhat) [- mean(d)]): gradient through the normalisation
template <int L, bool LN, bool FULL>
__device__ __forceinline__ void normalize_back(float (&d)[NV], const float (&xhat)[NV], float r, int at, int D, float inv_d,
                                               row_sum_t<L>& sum) {
    float a = 0.f, b = 0.f;
#pragma unroll
    for (int m = 0; m < NV; ++m) { a = fma_f(d[m], xhat[m], a); if (LN) b += d[m]; }
    if (LN) { const float2 t = sum(a, b); a = t.x * inv_d; b = t.y * inv_d; }
    else a = sum(a) * inv_d;
#pragma unroll
    for (int m = 0; m < NV; ++m) d[m] = FULL || at + m < D ? r * fma_f(-xhat[m], a, LN ? d[m] - b : d[m]) : 0.f;
}

template <typename E, int L, bool LN, bool FULL>
__global__ void __launch_bounds__(norm_geom<L>::THREADS) block_norm_bwd_kernel(xrl_block_norm_t p) {
    using G = norm_geom<L>;
    __shared__ float2 scratch[3][16];
    row_sum_t<L> sum{scratch, 0};
    const int lane = threadIdx.x % L, at = lane * NV, D = p.D;
    const float inv_d = 1.f / (float)D;
    __shared__ f32x4_t pars[4][2][L];
    norm_params<L> par{pars};
    par.fill(0, p.scale, 1.f, D); par.fill(1, p.w_post, 1.f, D); par.fill(2, p.b_post, 0.f, D); par.fill(3, p.w_pre, 1.f, D);
    __syncthreads();
    float acc[NORM_SUMS][NV] = {};
    // the next row is on its way while this one is worked on; 1024 threads leave no registers for that
    constexpr bool AHEAD = L < 1024;
    row8<E, FULL> rx, ru_, rg, ry_, rn;
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
        float x[NV], u[NV], g[NV], dy[NV] = {}, dn[NV] = {}, t[NV];
        if (!AHEAD) request(row);
        ru_.get(u); rx.get(x);
        if (p.gate) rg.get(g);
        if (p.d_y) ry_.get(dy);
        if (p.d_n) rn.get(dn);
        if (AHEAD && base + step < p.N) request(row + step);
        const float ru = normalize<L, LN, FULL>(u, at, D, inv_d, p.eps, sum);
        if (p.gate) {
            XRL_ACT_DISPATCH(p.gate_act, _Pragma("unroll") for (int m = 0; m < NV; ++m) g[m] = gate_act_c<ACT>(g[m]);)
        } else {
#pragma unroll
            for (int m = 0; m < NV; ++m) g[m] = 1.f;
        }
        float w[NV], sc[NV], pm[NV];                                 // pm: the block's part before gate and scale
        par.get(1, lane, w); par.get(2, lane, pm);
#pragma unroll
        for (int m = 0; m < NV; ++m) pm[m] = fma_f(u[m], w[m], pm[m]);
        if (p.d_n) {
            par.get(0, lane, sc);
#pragma unroll
            for (int m = 0; m < NV; ++m) x[m] = fma_f(g[m] * sc[m], pm[m], x[m]);
            const float ry = normalize<L, LN, FULL>(x, at, D, inv_d, p.eps, sum);
            par.get(3, lane, w);
#pragma unroll
            for (int m = 0; m < NV; ++m) { acc[2][m] = fma_f(dn[m], x[m], acc[2][m]); acc[3][m] += dn[m]; t[m] = dn[m] * w[m]; }
            normalize_back<L, LN, FULL>(t, x, ry, at, D, inv_d, sum);
#pragma unroll
            for (int m = 0; m < NV; ++m) dy[m] += t[m];
        }
        if (live) row8<E, FULL>::store((E*)p.d_x + row * p.ld_d_x, at, D, dy);
        // y = x + scale a p: with a the activated gate
        par.get(0, lane, sc); par.get(1, lane, w);
#pragma unroll
        for (int m = 0; m < NV; ++m) {
            const float da = dy[m] * g[m];
            acc[0][m] += da;
            acc[1][m] = fma_f(da, u[m], acc[1][m]);
            t[m] = da * sc[m] * w[m];
            dy[m] *= sc[m] * pm[m];                                  // gradient of the activated gate
        }
        if (p.d_gate) {
            XRL_ACT_DISPATCH(p.gate_act, _Pragma("unroll") for (int m = 0; m < NV; ++m) g[m] = dy[m] * act_grad_c<ACT>(g[m]);)
            if (live) row8<E, FULL>::store((E*)p.d_gate + row * p.ld_d_gate, at, D, g);
        }
        normalize_back<L, LN, FULL>(t, u, ru, at, D, inv_d, sum);
        if (live) row8<E, FULL>::store((E*)p.d_u + row * p.ld_d_u, at, D, t);
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

// The sums of the workgroups' lines, 64 groups of lines a column, met in a fixed order, and what they give.  A workgroup has 16 columns of S0 and S1
// or of S2 and S3.
__global__ void __launch_bounds__(1024) block_norm_sums_kernel(xrl_block_norm_t p, int lines) {
    __shared__ float part[2][64][17];
    const int c = threadIdx.x & 15, r = threadIdx.x >> 4, width = NORM_SUMS * p.D, e = blockIdx.x * 16 + c;
    const float* first = p.workspace + (size_t)blockIdx.y * 2 * p.D + e;
    float s = 0.f, t = 0.f;
    if (e < p.D)
        for (int i = r; i < lines; i += 64) {
            s += first[(size_t)i * width];
            t += first[(size_t)i * width + p.D];
        }
    part[0][r][c] = s;
    part[1][r][c] = t;
    __syncthreads();
    if (threadIdx.x < 16 && e < p.D) {
        s = t = 0.f;
        for (int i = 0; i < 64; ++i) { s += part[0][i][c]; t += part[1][i][c]; }
        if (blockIdx.y == 0) {
            const float sc = p.scale ? p.scale[e] : 1.f;
            if (p.d_scale) p.d_scale[e] = fma_f(p.w_post ? p.w_post[e] : 1.f, t, p.b_post ? p.b_post[e] * s : 0.f);
            if (p.d_w_post) p.d_w_post[e] = sc * t;
            if (p.d_b_post) p.d_b_post[e] = sc * s;
        } else {
            if (p.d_w_pre) p.d_w_pre[e] = s;
            if (p.d_b_pre) p.d_b_pre[e] = t;
        }
    }
}

static int norm_lanes(int D) {
    int L = 8;
    while (L * NV < D) L *= 2;
    return L;
}

// workgroups of the backward pass: as many as the registers let the chip hold (of 256 threads two a CU in f32, three in bf16), each with its rows
static int norm_lines(const xrl_block_norm_t& p) {
    const int L = norm_lanes(p.D), threads = L < 256 ? (L > 64 ? L : 256) : L, rows = L > 64 ? 1 : threads / L;
    const int64_t most = threads > 256 ? 256 : (p.dtype == XRL_F32 ? 512 : 768) * 256 / threads, need = (p.N + rows - 1) / rows;
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

template <typename E, bool LN, bool FULL>
static void launch_norm(const xrl_block_norm_t& p, bool backward, hipStream_t s) {
    const int L = norm_lanes(p.D);
#define NORM_CASE(LL)                                                                                                            \
    case LL: {                                                                                                                   \
        using G = norm_geom<LL>;                                                                                                 \
        if (backward) hipLaunchKernelGGL((block_norm_bwd_kernel<E, LL, LN, FULL>), dim3(norm_lines(p)), dim3(G::THREADS), 0, s, p); \
        else {                                                                                                                   \
            const int64_t need = (p.N + G::ROWS - 1) / G::ROWS, most = 1024 * 256 / G::THREADS;                                  \
            hipLaunchKernelGGL((block_norm_fwd_kernel<E, LL, LN, FULL>), dim3((int)(need < most ? need : most)), dim3(G::THREADS), 0, s, p); \
        }                                                                                                                        \
    } break;
    switch (L) { NORM_CASE(8) NORM_CASE(16) NORM_CASE(32) NORM_CASE(64) NORM_CASE(128) NORM_CASE(256) NORM_CASE(512) NORM_CASE(1024) }
#undef NORM_CASE
}

static int run_norm(const xrl_block_norm_t& p, bool backward, hipStream_t s) {
    const bool ln = p.kind == XRL_NORM_LAYER;
    const bool full = p.D == norm_lanes(p.D) * NV;
#define NORM_RUN(E, LN) do { if (full) launch_norm<E, LN, true>(p, backward, s); else launch_norm<E, LN, false>(p, backward, s); } while (0)
    if (p.dtype == XRL_F32) { if (ln) NORM_RUN(float, true); else NORM_RUN(float, false); }
    else { if (ln) NORM_RUN(bf16_t, true); else NORM_RUN(bf16_t, false); }
#undef NORM_RUN
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
        hipLaunchKernelGGL(block_norm_sums_kernel, dim3((p.D + 15) / 16, 2), dim3(1024), 0, as_stream(stream), p, norm_lines(p));
        XRL_CHECK_LAUNCH();
    }
    return XRL_OK;
}
