// Distillation of a categorical policy from a teacher's top logits (include/xrl_hip.h: xrl_distill_loss): the loss of every row and its
// gradient in one launch.  With m the row's maximum and Z = sum_a exp((s_a - m) / tau),
//     log p_a = (s_a - m) / tau - log Z,   loss = w tau^2 sum_k q_k (log q_k - log p_{i_k}),   d s_a = g w tau (p_a - q_a).
//
// Bound by memory: the logits are read once, their gradient is written once.  A row is held in registers from the one to the other, by 8 to 64
// lanes of a wave (up to 512 actions) or by a workgroup (up to 256 KB a row, 128 KB in 16 bits); only longer rows are read twice.  Rows of any width keep 16-byte
// accesses: the hardware takes them at any address, and a last part of a row that is shorter goes element by element.  An unavailable or
// absent action counts as -inf, which needs no case of its own afterwards.  q_k meets p at the lane that holds action i_k, so no element is
// stored twice; entries that name the same action are added up by the first of them, in their order (no float atomics).
#include "args.h"
#include "io16.h"

namespace xrl {

constexpr int DISTILL_MAX_K = 256;
constexpr float LOG2E = 1.4426950408889634f;

// elements [at, at + PER) of a row of A; absent and unavailable ones -inf
template <typename E>
__device__ __forceinline__ u32x4_t distill_load(const E* s, const float* av, int at, int A) {
    typedef row16<E> R;
    u32x4_t v = {R::LOW, R::LOW, R::LOW, R::LOW};
    if (at + R::PER <= A) {
        v = R::load(s + at);
        if (av) {
#pragma unroll
            for (int q = 0; q < R::PER / 4; ++q) {
                const f32x4_t a = *reinterpret_cast<const f32x4_any_t*>(av + at + 4 * q);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (a[j] == 0.f) R::put(v, 4 * q + j, R::LOW & (sizeof(E) == 4 ? 0xffffffffu : 0xffffu));
            }
        }
    } else if (at < A) {
#pragma unroll
        for (int j = 0; j < R::PER; ++j)
            if (at + j < A && (!av || av[at + j] != 0.f)) R::put(v, j, R::bits(s + at + j));
    }
    return v;
}

template <typename E>
__device__ __forceinline__ void distill_store(E* d, int at, int A, const float* f) {
    typedef row16<E> R;
    if (at + R::PER <= A) R::store(d + at, R::pack(f));
    else {
#pragma unroll
        for (int j = 0; j < R::PER; ++j)
            if (at + j < A) io_store(d + at + j, f[j]);
    }
}

// a teacher entry of action i and logit t: the action again or -1 (no entry: t is -inf too), and the policy's logit of the action
template <typename E>
__device__ __forceinline__ int distill_entry(int i, float& t, const E* s, const float* av, int A, float& z) {
    if (i < 0 || i >= A || t == -INFINITY) i = -1;
    else {
        z = io_load(s + i);
        if (av && av[i] == 0.f) i = -1;
    }
    if (i < 0) t = -INFINITY;
    return i;
}
// for a maximum: fmaxf passes over a NaN, which has to reach the result
__device__ __forceinline__ float nan_as_inf(float t) { return t != t ? INFINITY : t; }

__device__ __forceinline__ void wave_lds_fence() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); __builtin_amdgcn_wave_barrier(); }

// Rows of up to 8 L actions: L lanes a row, 8 neighbouring actions a lane, no barrier.  LDS of a row: its entries (action, weight, policy's logit) and
// one word per action, first the smallest entry that names it, then that action's teacher weight.
template <typename E, int L>
__global__ void __launch_bounds__(256) distill_lanes_kernel(xrl_distill_t p) {
    typedef row16<E> R;
    constexpr int ROWS = 256 / L, PER = R::PER, NV = 8 / PER;
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    const int slot = threadIdx.x / L, lane = threadIdx.x % L, A = p.A, K = p.K;
    int* at_action = reinterpret_cast<int*>(lds) + slot * 8 * L;
    int* ti = reinterpret_cast<int*>(lds) + ROWS * 8 * L + slot * K;
    float* tq = reinterpret_cast<float*>(lds) + ROWS * 8 * L + ROWS * K + slot * K;
    float* tz = tq + ROWS * K;
    const int64_t row = (int64_t)blockIdx.x * ROWS + slot;
    if (row >= p.N) return;
    auto sum = [&](float v) {
#pragma unroll
        for (int off = L / 2; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
        return v;
    };
    auto top = [&](float v) {
#pragma unroll
        for (int off = L / 2; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor(v, off, 64));
        return v;
    };
    const float w = p.weight ? p.weight[row] : 1.f, kt = LOG2E / p.temperature, inv_tau = 1.f / p.temperature;
    const E* s = (const E*)p.logits + row * p.ld;
    const float* av = p.avail ? p.avail + row * A : nullptr;
    u32x4_t v[NV];
#pragma unroll
    for (int q = 0; q < NV; ++q) v[q] = distill_load<E>(s, av, w != 0.f ? 8 * lane + PER * q : A, A);
    float tm = -INFINITY, m = -INFINITY;
    for (int k = lane; k < K; k += L) {
        float t = -INFINITY, z = 0.f;
        int i = -1;
        if (w != 0.f) {
            t = io_load((const E*)p.teacher_logits + row * K + k);
            i = distill_entry<E>(p.teacher_idx[row * K + k], t, s, av, A, z);
        }
        ti[k] = i; tq[k] = t; tz[k] = z;
        tm = fmaxf(tm, nan_as_inf(t));
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) { m = fmaxf(m, R::get(v[j / PER], j % PER)); at_action[8 * lane + j] = 0x7fffffff; }
    tm = top(tm); m = top(m);
    float any = 0.f, ts = 0.f, z = 0.f;
    wave_lds_fence();
    for (int k = lane; k < K; k += L)
        if (ti[k] >= 0) {
            any = 1.f;
            const float e = __builtin_amdgcn_exp2f((tq[k] - tm) * kt);
            tq[k] = e;
            ts += e;
            atomicMin(&at_action[ti[k]], k);
        }
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) { f[j] = __builtin_amdgcn_exp2f((R::get(v[j / PER], j % PER) - m) * kt); z += f[j]; }
    any = top(any); ts = sum(ts); z = sum(z);
    const bool live = any != 0.f && m != -INFINITY && w != 0.f;
    const float lz = logf(z), lt = logf(ts), inv_t = 1.f / ts;
    float term = 0.f;
    bool twice = false;
    wave_lds_fence();
    for (int k = lane; k < K; k += L)
        if (ti[k] >= 0) {
            const float q = tq[k] * inv_t;
            // tq is exp of the teacher's (t - max) / tau: its logarithm again costs less than keeping both
            if (q != 0.f) term += q * ((logf(tq[k]) - lt) - ((tz[k] - m) * inv_tau - lz));
            tq[k] = q;
            twice = twice || at_action[ti[k]] != k;
        }
    term = sum(term);
    if (lane == 0) p.loss[row] = live ? w * p.temperature * p.temperature * term : 0.f;
    if (!p.d_logits) return;
    wave_lds_fence();
    const bool repeats = __any(twice);
    for (int k = lane; k < K; k += L) {
        const int i = ti[k];
        if (i >= 0 && at_action[i] == k) {
            float q = tq[k];
            if (repeats)
                for (int j = k + 1; j < K; ++j)
                    if (ti[j] == i) q += tq[j];
            tz[k] = q;
        } else tz[k] = -1.f;
    }
    wave_lds_fence();
    for (int k = lane; k < K; k += L)
        if (ti[k] >= 0 && !(tz[k] < 0.f)) at_action[ti[k]] = __float_as_int(tz[k]);
    wave_lds_fence();
    const float c = live ? p.grad_scale * w * p.temperature : 0.f, inv_z = 1.f / z;
    E* d = (E*)p.d_logits + row * p.ld_d;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int q = at_action[8 * lane + j];
        const float pr = f[j] * inv_z;
        f[j] = live ? c * (q == 0x7fffffff ? pr : pr - __int_as_float(q)) : 0.f;
    }
#pragma unroll
    for (int q = 0; q < NV; ++q) distill_store<E>(d, 8 * lane + PER * q, A, f + PER * q);
}

// sums or maxima of two values over a workgroup of T threads; every call uses another part of `scratch`
template <int T, bool MAX>
__device__ __forceinline__ float2 block_pair(float a, float b, float2* scratch) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const float x = __shfl_xor(a, off, 64), y = __shfl_xor(b, off, 64);
        a = MAX ? fmaxf(a, x) : a + x;
        b = MAX ? fmaxf(b, y) : b + y;
    }
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = make_float2(a, b);
    lds_barrier();
    float2 r = scratch[0];
#pragma unroll
    for (int i = 1; i < T / 64; ++i) {
        const float2 o = scratch[i];
        r.x = MAX ? fmaxf(r.x, o.x) : r.x + o.x;
        r.y = MAX ? fmaxf(r.y, o.y) : r.y + o.y;
    }
    return r;
}

// Rows of up to T NV 16 bytes: a workgroup a row, NV pieces of 16 bytes a thread; entry k belongs to thread k.
template <typename E, int T, int NV>
__global__ void __launch_bounds__(T) distill_row_kernel(xrl_distill_t p) {
    typedef row16<E> R;
    constexpr int PER = R::PER;
    __shared__ float2 scratch[3][T / 64];
    __shared__ int ti[DISTILL_MAX_K], next[DISTILL_MAX_K], head[T];
    __shared__ float tq[DISTILL_MAX_K];
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x, A = p.A, K = p.K;
    const E* s = (const E*)p.logits + row * p.ld;
    E* d = p.d_logits ? (E*)p.d_logits + row * p.ld_d : nullptr;
    const float* av = p.avail ? p.avail + row * A : nullptr;
    const float w = p.weight ? p.weight[row] : 1.f, kt = LOG2E / p.temperature, inv_tau = 1.f / p.temperature;
    u32x4_t v[NV];
    float m = -INFINITY, tl = -INFINITY, z_at = 0.f;
    int idx = -1;
    if (w != 0.f) {
        if (tid < K) { idx = p.teacher_idx[row * K + tid]; tl = io_load((const E*)p.teacher_logits + row * K + tid); }
#pragma unroll
        for (int q = 0; q < NV; ++q) v[q] = distill_load<E>(s, av, (tid + q * T) * PER, A);
        idx = distill_entry<E>(idx, tl, s, av, A, z_at);
#pragma unroll
        for (int q = 0; q < NV; ++q)
#pragma unroll
            for (int j = 0; j < PER; ++j) m = fmaxf(m, R::get(v[q], j));
    }
    if (tid < K) ti[tid] = idx;
    head[tid] = -1;
    const float2 tops = block_pair<T, true>(m, nan_as_inf(tl), scratch[0]);
    const float tm = tops.y;
    m = tops.x;
    if (tm == -INFINITY || m == -INFINITY) {                     // weight 0, no entry, no available logit
        const float zero[PER] = {};
        if (d)
#pragma unroll
            for (int q = 0; q < NV; ++q)
                if ((tid + q * T) * PER < A) distill_store<E>(d, (tid + q * T) * PER, A, zero);
        if (tid == 0) p.loss[row] = 0.f;
        return;
    }
    float z = 0.f;
#pragma unroll
    for (int q = 0; q < NV; ++q)
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const float e = __builtin_amdgcn_exp2f((R::get(v[q], j) - m) * kt);
            z += e;
            if (sizeof(E) == 4) R::put(v[q], j, __float_as_uint(e));           // 16-bit rows keep their logits and take the exponential again
        }
    const float te = idx >= 0 ? __builtin_amdgcn_exp2f((tl - tm) * kt) : 0.f;
    const float2 sums = block_pair<T, false>(z, te, scratch[1]);
    const float inv_z = 1.f / sums.x, qk = te / sums.y;
    if (tid < K) tq[tid] = qk;
    float term = 0.f;
    if (qk != 0.f) term = qk * (((tl - tm) * inv_tau - logf(sums.y)) - ((z_at - m) * inv_tau - logf(sums.x)));
    const float2 loss = block_pair<T, false>(term, 0.f, scratch[2]);
    if (tid == 0) p.loss[row] = w * p.temperature * p.temperature * loss.x;
    if (!d) return;
    if (idx >= 0) {                                              // the first entry that names its action carries the weight of all of them
        float q = 0.f;
        bool first = true;
        for (int k = 0; k < K; ++k)
            if (ti[k] == idx) { first = first && k >= tid; if (k >= tid) q += tq[k]; }
        if (first) {
            tl = q;
            next[tid] = atomicExch(&head[(idx / PER) % T], tid);  // a list for the thread that holds the action
        } else idx = -1;
    }
    lds_barrier();                                               // everyone has summed: tq may now hold the sums
    if (idx >= 0) tq[tid] = tl;
    lds_barrier();
    const float c = p.grad_scale * w * p.temperature;
    const int mine = head[tid];
#pragma unroll
    for (int q = 0; q < NV; ++q) {
        const int at = (tid + q * T) * PER;
        if (at >= A) continue;
        float f[PER];
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const float e = sizeof(E) == 4 ? R::get(v[q], j) : __builtin_amdgcn_exp2f((R::get(v[q], j) - m) * kt);
            f[j] = e * inv_z;
        }
        for (int k = mine; k >= 0; k = next[k]) {
            const int j = ti[k] - at;
#pragma unroll
            for (int i = 0; i < PER; ++i) f[i] = i == j ? f[i] - tq[k] : f[i];
        }
#pragma unroll
        for (int j = 0; j < PER; ++j) f[j] *= c;
        distill_store<E>(d, at, A, f);
    }
}

// Longer rows: one pass for the maximum and the sum together, a second one for the gradient.
template <typename E>
__global__ void __launch_bounds__(1024) distill_long_kernel(xrl_distill_t p) {
    typedef row16<E> R;
    constexpr int PER = R::PER, T = 1024;
    __shared__ float2 scratch[4][T / 64];
    __shared__ int ti[DISTILL_MAX_K];
    __shared__ float tq[DISTILL_MAX_K];
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x, A = p.A, K = p.K;
    const E* s = (const E*)p.logits + row * p.ld;
    E* d = p.d_logits ? (E*)p.d_logits + row * p.ld_d : nullptr;
    const float* av = p.avail ? p.avail + row * A : nullptr;
    const float w = p.weight ? p.weight[row] : 1.f, kt = LOG2E / p.temperature, inv_tau = 1.f / p.temperature;
    float m = -INFINITY, z = 0.f, tl = -INFINITY, z_at = 0.f;
    int idx = -1;
    if (w != 0.f) {
        if (tid < K) { idx = p.teacher_idx[row * K + tid]; tl = io_load((const E*)p.teacher_logits + row * K + tid); }
        idx = distill_entry<E>(idx, tl, s, av, A, z_at);
        for (int64_t at = (int64_t)tid * PER; at < A; at += T * PER) {
            const u32x4_t v = distill_load<E>(s, av, (int)at, A);
            float top = m;
#pragma unroll
            for (int j = 0; j < PER; ++j) top = fmaxf(top, R::get(v, j));
            if (top > -INFINITY) {
                z *= __builtin_amdgcn_exp2f((m - top) * kt);
#pragma unroll
                for (int j = 0; j < PER; ++j) z += __builtin_amdgcn_exp2f((R::get(v, j) - top) * kt);
                m = top;
            }
        }
    }
    if (tid < K) ti[tid] = idx;
    const float2 tops = block_pair<T, true>(m, nan_as_inf(tl), scratch[0]);
    const float mine = m, tm = tops.y;
    m = tops.x;
    if (tm == -INFINITY || m == -INFINITY) {
        const float zero[PER] = {};
        if (d) for (int64_t at = (int64_t)tid * PER; at < A; at += T * PER) distill_store<E>(d, (int)at, A, zero);
        if (tid == 0) p.loss[row] = 0.f;
        return;
    }
    z = mine > -INFINITY ? z * __builtin_amdgcn_exp2f((mine - m) * kt) : 0.f;
    const float te = idx >= 0 ? __builtin_amdgcn_exp2f((tl - tm) * kt) : 0.f;
    const float2 sums = block_pair<T, false>(z, te, scratch[1]);
    const float inv_z = 1.f / sums.x, qk = te / sums.y;
    if (tid < K) tq[tid] = qk;
    float term = 0.f;
    if (qk != 0.f) term = qk * (((tl - tm) * inv_tau - logf(sums.y)) - ((z_at - m) * inv_tau - logf(sums.x)));
    const float2 loss = block_pair<T, false>(term, 0.f, scratch[2]);
    if (tid == 0) p.loss[row] = w * p.temperature * p.temperature * loss.x;
    if (!d) return;
    const float c = p.grad_scale * w * p.temperature;
    for (int64_t at = (int64_t)tid * PER; at < A; at += T * PER) {
        const u32x4_t v = distill_load<E>(s, av, (int)at, A);
        float f[PER];
#pragma unroll
        for (int j = 0; j < PER; ++j) f[j] = c * (__builtin_amdgcn_exp2f((R::get(v, j) - m) * kt) * inv_z);
        distill_store<E>(d, (int)at, A, f);
    }
    __syncthreads();                                             // the entries' elements are written over, by the first entry of each action
    if (idx >= 0) {
        float q = 0.f;
        bool first = true;
        for (int k = 0; k < K; ++k)
            if (ti[k] == idx) { first = first && k >= tid; q += tq[k]; }
        if (first) io_store(d + idx, c * (__builtin_amdgcn_exp2f((z_at - m) * kt) * inv_z - q));
    }
}

template <typename E>
static void launch_distill(const xrl_distill_t& p, hipStream_t st) {
    const int A = p.A;
    const int64_t bytes = (int64_t)A * (int)sizeof(E);
    const unsigned n = (unsigned)p.N;
#define DISTILL_LANES(L)                                                                                                             \
    hipLaunchKernelGGL((distill_lanes_kernel<E, L>), dim3((n + 256 / L - 1) / (256 / L)), dim3(256), 4 * (256 / L) * (8 * L + 3 * p.K), st, p)
#define DISTILL_ROW(T, NV) hipLaunchKernelGGL((distill_row_kernel<E, T, NV>), dim3(n), dim3(T), 0, st, p)
    if (A <= 64 && p.K <= 64) DISTILL_LANES(8);                  // more entries a row leave no LDS for 32 rows
    else if (A <= 128 && p.K <= 128) DISTILL_LANES(16);
    else if (A <= 256) DISTILL_LANES(32);
    else if (A <= 512) DISTILL_LANES(64);
    else if (bytes <= 256 * 16) DISTILL_ROW(256, 1);
    else if (bytes <= 256 * 32) DISTILL_ROW(256, 2);
    else if (bytes <= 256 * 64) DISTILL_ROW(256, 4);
    else if (bytes <= 512 * 64) DISTILL_ROW(512, 4);
    else if (bytes <= 512 * 128) DISTILL_ROW(512, 8);
    else if (bytes <= 1024 * 128) DISTILL_ROW(1024, 8);
    else if (sizeof(E) == 4 && bytes <= 1024 * 256) DISTILL_ROW(1024, (sizeof(E) == 4 ? 16 : 8));      // 8 x 16 bf16 a thread do not fit the registers
    else hipLaunchKernelGGL(distill_long_kernel<E>, dim3(n), dim3(1024), 0, st, p);
#undef DISTILL_ROW
#undef DISTILL_LANES
}

}  // namespace xrl

using namespace xrl;

extern "C" int xrl_distill_loss(const xrl_distill_t* pp, xrl_stream_t stream) {
    XRL_CHECK_ARG(pp != nullptr);
    const xrl_distill_t& p = *pp;
    XRL_CHECK_ARG(p.N >= 0 && p.N <= 0x7fffffff && p.A >= 1 && p.A <= 1 << 30 && p.K >= 1 && p.K <= DISTILL_MAX_K);
    XRL_CHECK_ARG((p.dtype == XRL_F32 || p.dtype == XRL_BF16) && p.temperature > 0.f);
    if (p.N == 0) return XRL_OK;
    XRL_CHECK_ARG(p.logits && p.teacher_idx && p.teacher_logits && p.loss);
    const int e = p.dtype == XRL_F32 ? 4 : 2;
    const arg_t a[] = {{"d_logits", p.d_logits, e, 2, {p.N, p.A}, {p.ld_d, 1}, true}, {"loss", p.loss, 4, 1, {p.N}, {1}, true},
                       {"logits", p.logits, e, 2, {p.N, p.A}, {p.ld, 1}, false}, {"teacher_idx", p.teacher_idx, 4, 2, {p.N, p.K}, {p.K, 1}, false},
                       {"teacher_logits", p.teacher_logits, e, 2, {p.N, p.K}, {p.K, 1}, false}, {"avail", p.avail, 4, 2, {p.N, p.A}, {p.A, 1}, false},
                       {"weight", p.weight, 4, 1, {p.N}, {1}, false}};
    const int pairs[][2] = {{0, 2}};
    if (int rc = check_args(a, 7, pairs, 1)) return rc;
    if (p.dtype == XRL_F32) launch_distill<float>(p, as_stream(stream));
    else launch_distill<bf16_t>(p, as_stream(stream));
    XRL_CHECK_LAUNCH();
    return XRL_OK;
}
