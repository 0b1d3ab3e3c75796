// Distillation of a categorical policy from a teacher's top logits (include/xrl_hip.h: xrl_distill_loss): the loss of every row and its
// gradient in one launch.  With m the row's maximum and Z = sum_a exp((s_a - m) / tau),
//     log p_a = (s_a - m) / tau - log Z,   loss = w tau^2 sum_k q_k (log q_k - log p_{i_k}),   d s_a = g w tau (p_a - q_a).
//
// Bound by memory: the logits are read once, their gradient is written once.  A row is held in registers from the one to the other, by 8 to 64
// lanes of a wave (up to 512 actions), by a wave (up to 16 KB a row, 24 KB in 16 bits) or by a workgroup (up to 256 KB, 128 KB in 16 bits); only
// longer rows are read twice.  Rows of any width keep 16-byte accesses: the hardware takes them at any address, and a last part of a row that is
// shorter goes element by element.  An unavailable or absent action counts as -inf, which needs no case of its own afterwards.  Entries that name
// the same action are added up by the first of them, in their order (no float atomics).
// Measured, logits and gradient counted: 8192 x 4099 bf16 32 us (4.2 TB/s), 8388 x 4000 f32 49 us (5.5), 4096 x 50257 f32 366 us (4.5; a copy of
// this size reaches 5.4), 33554 x 1000 bf16 42 us (3.2: the work on the entries shows), 256 x 18 9.7 us (the call and its launch).
#include "args.h"
#include "io16.h"
#include "lanes.h"

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
__device__ __forceinline__ void wave_lds_fence() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); __builtin_amdgcn_wave_barrier(); }

// Rows of up to 8 L actions: L lanes a row, 8 neighbouring actions a lane, no barrier.  LDS of a row: its entries (action, weight, policy's logit) and
// one word per action, first the smallest entry that names it, then that action's teacher weight.  65536 x 512 f32: 70 us, 3.9 TB/s.
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
        tm = nan_max(tm, t);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) { m = nan_max(m, R::get(v[j / PER], j % PER)); at_action[8 * lane + j] = 0x7fffffff; }
    tm = lane_max<L>(tm); m = lane_max<L>(m);
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
    any = lane_max<L>(any); ts = lane_sum<L>(ts); z = lane_sum<L>(z);
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
    term = lane_sum<L>(term);
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

// sums or maxima of two values over a workgroup of T threads; every call uses another part of `scratch`.  For T = 64 they are
// over the wave, and no `scratch` is used.
template <int T, bool MAX>
__device__ __forceinline__ float2 block_pair(float a, float b, float2* scratch) {
    a = MAX ? lane_max<64>(a) : lane_sum<64>(a);
    b = MAX ? lane_max<64>(b) : lane_sum<64>(b);
    if (T == 64) return make_float2(a, b);
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = make_float2(a, b);
    lds_barrier();
    float2 r = scratch[0];
#pragma unroll
    for (int i = 1; i < T / 64; ++i) {
        const float2 o = scratch[i];
        r.x = MAX ? nan_max(r.x, o.x) : r.x + o.x;
        r.y = MAX ? nan_max(r.y, o.y) : r.y + o.y;
    }
    return r;
}

// Rows of up to NV KB: a wave a row, KV entries a lane (entry k in lane k % 64), no barrier and no LDS.  Many waves hide each other's latencies, so
// the entries' actions are simply stored a second time, behind the row's own stores.
template <typename E, int NV, int KV>
__global__ void __launch_bounds__(256) distill_wave_kernel(xrl_distill_t p) {
    typedef row16<E> R;
    constexpr int PER = R::PER;
    const int lane = threadIdx.x & 63, A = p.A, K = p.K, t0 = lane * PER;
    const int64_t row = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (row >= p.N) return;
    const float kt = LOG2E / p.temperature, inv_tau = 1.f / p.temperature;
    typedef const __attribute__((address_space(4))) float* scalar_t;
    const float w = p.weight ? ((scalar_t)(uintptr_t)p.weight)[row] : 1.f;
    const E* s = (const E*)p.logits + row * p.ld;
    E* d = p.d_logits ? (E*)p.d_logits + row * p.ld_d : nullptr;
    const float* av = p.avail ? p.avail + row * A : nullptr;
    u32x4_t v[NV];
    float m = -INFINITY, tm = -INFINITY, tl[KV], z_at[KV];
    int idx[KV];
#pragma unroll
    for (int e = 0; e < KV; ++e) { idx[e] = -1; tl[e] = -INFINITY; z_at[e] = 0.f; }
    if (w != 0.f) {
#pragma unroll
        for (int e = 0; e < KV; ++e)
            if (lane + 64 * e < K) {
                idx[e] = p.teacher_idx[row * K + lane + 64 * e];
                tl[e] = io_load((const E*)p.teacher_logits + row * K + lane + 64 * e);
            }
#pragma unroll
        for (int q = 0; q < NV; ++q) v[q] = distill_load<E>(s + q * 64 * PER, av ? av + q * 64 * PER : nullptr, t0, A - q * 64 * PER);
#pragma unroll
        for (int e = 0; e < KV; ++e) {
            idx[e] = distill_entry<E>(idx[e], tl[e], s, av, A, z_at[e]);
            tm = nan_max(tm, tl[e]);
        }
#pragma unroll
        for (int q = 0; q < NV; ++q)
#pragma unroll
            for (int j = 0; j < PER; ++j) m = nan_max(m, R::get(v[q], j));
    }
    const float2 tops = block_pair<64, true>(m, tm, nullptr);
    tm = tops.y;
    m = tops.x;
    if (tm == -INFINITY || m == -INFINITY) {                     // weight 0, no entry, no available logit
        const float zero[PER] = {};
        if (d)
#pragma unroll
            for (int q = 0; q < NV; ++q)
                if (t0 < A - q * 64 * PER) distill_store<E>(d + q * 64 * PER, t0, A - q * 64 * PER, zero);
        if (lane == 0) p.loss[row] = 0.f;
        return;
    }
    float z = 0.f, te[KV], ts = 0.f, term = 0.f;
#pragma unroll
    for (int q = 0; q < NV; ++q) {
        if (sizeof(E) == 2) asm volatile("" : "+v"(v[q]));       // unpacked anew for each use: kept, it would take twice the registers
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const float e = __builtin_amdgcn_exp2f((R::get(v[q], j) - m) * kt);
            z += e;
            if (sizeof(E) == 4) R::put(v[q], j, __float_as_uint(e));                // 16-bit rows keep their logits and take the exponential again
        }
    }
#pragma unroll
    for (int e = 0; e < KV; ++e) {
        te[e] = idx[e] >= 0 ? __builtin_amdgcn_exp2f((tl[e] - tm) * kt) : 0.f;
        ts += te[e];
    }
    const float2 sums = block_pair<64, false>(z, ts, nullptr);
    const float c = p.grad_scale * w * p.temperature, ci = c / sums.x, lz = logf(sums.x), lt = logf(sums.y);
#pragma unroll
    for (int e = 0; e < KV; ++e) {
        te[e] /= sums.y;
        if (te[e] != 0.f) term += te[e] * (((tl[e] - tm) * inv_tau - lt) - ((z_at[e] - m) * inv_tau - lz));
    }
    term = lane_sum<64>(term);
    if (lane == 0) p.loss[row] = w * p.temperature * p.temperature * term;
    if (!d) return;
    // entries that name one action: found by every entry's action in turn, which no entry without one can meet
    uint64_t repeats = 0;
    int name[KV];
#pragma unroll
    for (int e = 0; e < KV; ++e) name[e] = idx[e] >= 0 ? idx[e] : -1 - (lane + 64 * e);
#pragma unroll
    for (int e = 0; e < KV; ++e)
        for (int k = 0; k < (K - 64 * e < 64 ? K - 64 * e : 64); ++k) {
            const int i = __builtin_amdgcn_readlane(name[e], k);
            uint64_t others = 0;
#pragma unroll
            for (int o = 0; o < KV; ++o) {
                uint64_t same = __ballot(name[o] == i);
                if (o == e) same &= same - 1;                    // the lowest lane of this word is at most k: a second one shows the repeat
                others |= o < e ? 0 : same;
            }
            repeats |= others;
        }
    if (repeats) {                                               // by the first of them, all in their order
        float all[KV];
#pragma unroll
        for (int o = 0; o < KV; ++o) all[o] = 0.f;
#pragma unroll
        for (int e = 0; e < KV; ++e)
            for (int k = 0; k < (K - 64 * e < 64 ? K - 64 * e : 64); ++k) {
                const int i = __builtin_amdgcn_readlane(name[e], k);
                const float q = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(te[e]), k));
#pragma unroll
                for (int o = 0; o < KV; ++o)
                    if (i == name[o]) {
                        all[o] += q;
                        if (64 * e + k < 64 * o + lane) idx[o] = -1;
                    }
            }
#pragma unroll
        for (int o = 0; o < KV; ++o) te[o] = all[o];
    }
#pragma unroll
    for (int q = 0; q < NV; ++q) {
        if (t0 >= A - q * 64 * PER) continue;
        if (sizeof(E) == 2) asm volatile("" : "+v"(v[q]));
        float f[PER];
#pragma unroll
        for (int j = 0; j < PER; ++j)
            f[j] = ci * (sizeof(E) == 4 ? R::get(v[q], j) : __builtin_amdgcn_exp2f((R::get(v[q], j) - m) * kt));
        distill_store<E>(d + q * 64 * PER, t0, A - q * 64 * PER, f);
    }
    __threadfence_block();                                       // the row's stores come first
#pragma unroll
    for (int e = 0; e < KV; ++e)
        if (idx[e] >= 0) io_store(d + idx[e], ci * __builtin_amdgcn_exp2f((z_at[e] - m) * kt) - c * te[e]);
}

// Rows of up to T NV 16 bytes: a workgroup a row at a time, NV pieces of 16 bytes a thread; entry k belongs to thread k.  An entry meets its
// action in the thread that holds it, by a list in LDS whose first two actions the thread keeps.  The next row is requested piece by piece
// as this one's gradient is stored.
template <typename E, int T, int NV>
__global__ void __launch_bounds__(T) distill_row_kernel(xrl_distill_t p) {
    typedef row16<E> R;
    constexpr int PER = R::PER;
    __shared__ float2 scratch[3][T / 64];
    __shared__ int ti[DISTILL_MAX_K], next[DISTILL_MAX_K], head[T];
    __shared__ float tq[DISTILL_MAX_K];
    const int tid = threadIdx.x, A = p.A, K = p.K;
    const float kt = LOG2E / p.temperature, inv_tau = 1.f / p.temperature;
    typedef const __attribute__((address_space(4))) float* scalar_t;
    auto weight = [&](int64_t row) { return p.weight ? ((scalar_t)(uintptr_t)p.weight)[row] : 1.f; };
    u32x4_t v[NV];
    int idx = -1;
    float tl = -INFINITY, w = weight(blockIdx.x);
    auto entries = [&](int64_t row) {
        idx = -1; tl = -INFINITY;
        if (tid < K) { idx = p.teacher_idx[row * K + tid]; tl = io_load((const E*)p.teacher_logits + row * K + tid); }
    };
    const int t0 = tid * PER;                                         // this thread's actions are q T PER + t0 + 0..PER-1
    auto anew = [&]() {                                               // 16-bit rows are unpacked for each use: kept unpacked they would take twice the registers
        if (sizeof(E) == 2)
#pragma unroll
            for (int q = 0; q < NV; ++q) asm volatile("" : "+v"(v[q]));
    };
    auto piece = [&](int64_t row, int q) {
        const int64_t at = (int64_t)row * p.ld + q * T * PER;
        v[q] = distill_load<E>((const E*)p.logits + at, p.avail ? p.avail + row * A + q * T * PER : nullptr, t0, A - q * T * PER);
    };
    if (w != 0.f) {
        entries(blockIdx.x);
#pragma unroll
        for (int q = 0; q < NV; ++q) piece(blockIdx.x, q);
    }
    for (int64_t row = blockIdx.x; row < p.N; row += gridDim.x) {
        const int64_t ahead = row + gridDim.x;
        const float w_ahead = ahead < p.N ? weight(ahead) : 0.f;
        E* d = p.d_logits ? (E*)p.d_logits + row * p.ld_d : nullptr;
        head[tid] = -1;
        lds_barrier();
        float m = -INFINITY;
        float z_at = 0.f;
        if (w != 0.f) {
            idx = distill_entry<E>(idx, tl, (const E*)p.logits + row * p.ld, p.avail ? p.avail + row * A : nullptr, A, z_at);
            if (tid < K) {
                ti[tid] = idx;
                if (idx >= 0) next[tid] = atomicExch(&head[(idx / PER) % T], tid);
            }
#pragma unroll
            for (int q = 0; q < NV; ++q)
#pragma unroll
                for (int j = 0; j < PER; ++j) m = nan_max(m, R::get(v[q], j));
        }
        const float2 tops = block_pair<T, true>(m, w != 0.f ? tl : -INFINITY, scratch[0]);
        const float tm = tops.y;
        m = tops.x;
        const bool live = tm != -INFINITY && m != -INFINITY;           // weight 0, no entry, no available logit: 0
        float c = 0.f, ci = 0.f;
        const int mine = live ? head[tid] : -1;
        if (live) {
            anew();
            float z = 0.f;
#pragma unroll
            for (int q = 0; q < NV; ++q)
#pragma unroll
                for (int j = 0; j < PER; ++j) {
                    const float e = __builtin_amdgcn_exp2f((R::get(v[q], j) - m) * kt);
                    z += e;
                    if (sizeof(E) == 4) R::put(v[q], j, __float_as_uint(e));       // 16-bit rows keep their logits and take the exponential again
                }
            const float te = idx >= 0 ? __builtin_amdgcn_exp2f((tl - tm) * kt) : 0.f;
            const float2 sums = block_pair<T, false>(z, te, scratch[1]);
            const float qk = te / sums.y;
            if (tid < K) tq[tid] = qk;
            float term = 0.f;
            if (qk != 0.f) term = qk * (((tl - tm) * inv_tau - logf(sums.y)) - ((z_at - m) * inv_tau - logf(sums.x)));
            const float2 loss = block_pair<T, false>(term, 0.f, scratch[2]);
            if (tid == 0) p.loss[row] = w * p.temperature * p.temperature * loss.x;
            c = p.grad_scale * w * p.temperature;
            ci = c / sums.x;
        } else if (tid == 0) p.loss[row] = 0.f;
        if (w_ahead != 0.f) entries(ahead);
        anew();
        // the list's actions in their order, each with the weights of all entries that name it, by the first of them: two in registers
        int at1 = -1, at2 = -1, last = -1;
        float q1 = 0.f, q2 = 0.f;
        auto next_action = [&](int& at, float& q) {
            int k = DISTILL_MAX_K;                                   // the smallest entry behind `last` whose action no earlier one names
            for (int o = mine; o >= 0; o = next[o]) {
                if (o <= last || o >= k) continue;
                bool first = true;
                for (int e = mine; e >= 0 && first; e = next[e]) first = e >= o || ti[e] != ti[o];
                if (first) k = o;
            }
            if (k == DISTILL_MAX_K) return false;
            at = ti[k]; q = tq[k];
            for (int low = k;;) {
                int least = DISTILL_MAX_K;
                for (int o = mine; o >= 0; o = next[o])
                    if (ti[o] == at && o > low && o < least) least = o;
                if (least == DISTILL_MAX_K) break;
                q += tq[least];
                low = least;
            }
            last = k;
            return true;
        };
        bool more = false;
        if (mine >= 0 && next_action(at1, q1) && next_action(at2, q2)) more = true;
#pragma unroll
        for (int q = 0; q < NV; ++q) {
            const int left = A - q * T * PER;
            if (d && t0 < left) {
                float f[PER];
                if (!live) {
#pragma unroll
                    for (int j = 0; j < PER; ++j) f[j] = 0.f;
                } else {
#pragma unroll
                    for (int j = 0; j < PER; ++j)
                        f[j] = ci * (sizeof(E) == 4 ? R::get(v[q], j) : __builtin_amdgcn_exp2f((R::get(v[q], j) - m) * kt));
                    const int i1 = at1 - q * T * PER - t0, i2 = at2 - q * T * PER - t0;
                    if ((unsigned)i1 < (unsigned)PER || (unsigned)i2 < (unsigned)PER) {
#pragma unroll
                        for (int j = 0; j < PER; ++j) {
                            f[j] = j == i1 ? f[j] - c * q1 : f[j];
                            f[j] = j == i2 ? f[j] - c * q2 : f[j];
                        }
                    }
                    if (more) {
                        const int kept = last;
                        int at = -1;
                        float w_at = 0.f;
                        while (next_action(at, w_at)) {
                            const int i = at - q * T * PER - t0;
#pragma unroll
                            for (int j = 0; j < PER; ++j) f[j] = j == i ? f[j] - c * w_at : f[j];
                        }
                        last = kept;
                    }
                }
                distill_store<E>(d + q * T * PER, t0, left, f);
            }
            if (w_ahead != 0.f) piece(ahead, q);
        }
        w = w_ahead;
        lds_barrier();                                               // the lists are read to the end before the next row's are begun
    }
}

// Longer rows: one pass for the maximum and the sum together, a second one for the gradient.  1000 x 100000 f32: 227 us, 5.3 TB/s of the three passes
// through memory.
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
            for (int j = 0; j < PER; ++j) top = nan_max(top, R::get(v, j));
            if (top != -INFINITY) {
                z *= __builtin_amdgcn_exp2f((m - top) * kt);
#pragma unroll
                for (int j = 0; j < PER; ++j) z += __builtin_amdgcn_exp2f((R::get(v, j) - top) * kt);
                m = top;
            }
        }
    }
    if (tid < K) ti[tid] = idx;
    const float2 tops = block_pair<T, true>(m, tl, scratch[0]);
    const float mine = m, tm = tops.y;
    m = tops.x;
    if (tm == -INFINITY || m == -INFINITY) {
        const float zero[PER] = {};
        if (d) for (int64_t at = (int64_t)tid * PER; at < A; at += T * PER) distill_store<E>(d, (int)at, A, zero);
        if (tid == 0) p.loss[row] = 0.f;
        return;
    }
    z = mine != -INFINITY ? z * __builtin_amdgcn_exp2f((mine - m) * kt) : 0.f;
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

// as many workgroups as the chip holds at a time, each with its rows
template <typename E, int T, int NV>
static void launch_distill_row(const xrl_distill_t& p, hipStream_t st) {
    static const int held = [] {
        int n = 0;
        if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&n, distill_row_kernel<E, T, NV>, T, 0) != hipSuccess || n < 1) n = 1;
        return 256 * n;
    }();
    hipLaunchKernelGGL((distill_row_kernel<E, T, NV>), dim3((unsigned)(p.N < held ? p.N : held)), dim3(T), 0, st, p);
}

template <typename E>
static void launch_distill(const xrl_distill_t& p, hipStream_t st) {
    const int A = p.A;
    const int64_t bytes = (int64_t)A * (int)sizeof(E);
    const unsigned n = (unsigned)p.N;
#define DISTILL_LANES(L)                                                                                                             \
    hipLaunchKernelGGL((distill_lanes_kernel<E, L>), dim3((n + 256 / L - 1) / (256 / L)), dim3(256), 4 * (256 / L) * (8 * L + 3 * p.K), st, p)
#define DISTILL_ROW(T, NV) launch_distill_row<E, T, NV>(p, st)
#define DISTILL_WAVE(NV)                                                                                                             \
    if (p.K <= 64) hipLaunchKernelGGL((distill_wave_kernel<E, NV, 1>), dim3((n + 3) / 4), dim3(256), 0, st, p);                      \
    else hipLaunchKernelGGL((distill_wave_kernel<E, NV, 4>), dim3((n + 3) / 4), dim3(256), 0, st, p)
    // A wave a row against a workgroup of 256 a row, both in registers: 8186 x 4099 bf16 33 us against 71, 33554 x 1000 47 against 295, 4194 x 8000
    // f32 53 against 66: no barriers, and as many rows in flight as waves.  Pieces in steps, since each piece that a row does not have still costs
    // its exponentials (16-bit rows of 20 and 24 KB: 31 us for 64 MB in a wave, 38 in a workgroup of 512).  Above them 512 threads up to 32 KB and 1024
    // behind: 134 MB in rows of 64000 bytes took 90 us in 512 threads, 67 MB in rows of 60000 bytes 38 us in 1024.  One list for all K: a lane has room for 4 entries where K is over 64.
    if (A <= 64 && p.K <= 64) DISTILL_LANES(8);                  // more entries a row leave no LDS for 32 rows
    else if (A <= 128 && p.K <= 128) DISTILL_LANES(16);
    else if (A <= 256) DISTILL_LANES(32);
    else if (A <= 512) DISTILL_LANES(64);
    else if (bytes <= (sizeof(E) == 4 ? 16 : 24) * 1024) {
        if (bytes <= 2 * 1024) { DISTILL_WAVE(2); }
        else if (bytes <= 4 * 1024) { DISTILL_WAVE(4); }
        else if (bytes <= 6 * 1024) { DISTILL_WAVE(6); }
        else if (bytes <= 8 * 1024) { DISTILL_WAVE(8); }
        else if (bytes <= 10 * 1024) { DISTILL_WAVE(10); }
        else if (bytes <= 12 * 1024) { DISTILL_WAVE(12); }
        else if (bytes <= 16 * 1024) { DISTILL_WAVE(16); }
        else if (bytes <= 20 * 1024) { DISTILL_WAVE((sizeof(E) == 4 ? 16 : 20)); }
        else { DISTILL_WAVE((sizeof(E) == 4 ? 16 : 24)); }
    }
    else if (bytes <= 512 * 48) DISTILL_ROW(512, 3);
    else if (bytes <= 512 * 64) DISTILL_ROW(512, 4);
    else if (bytes <= 1024 * 48) DISTILL_ROW(1024, 3);
    else if (bytes <= 1024 * 64) DISTILL_ROW(1024, 4);
    else if (bytes <= 1024 * 96) DISTILL_ROW(1024, 6);
    else if (bytes <= 1024 * 128) DISTILL_ROW(1024, 8);
    else if (sizeof(E) == 4 && bytes <= 1024 * 160) DISTILL_ROW(1024, (sizeof(E) == 4 ? 10 : 8));       // 8 x 16 bf16 a thread do not fit the registers
    else if (sizeof(E) == 4 && bytes <= 1024 * 208) DISTILL_ROW(1024, (sizeof(E) == 4 ? 13 : 8));
    else if (sizeof(E) == 4 && bytes <= 1024 * 256) DISTILL_ROW(1024, (sizeof(E) == 4 ? 16 : 8));
    else hipLaunchKernelGGL(distill_long_kernel<E>, dim3(n), dim3(1024), 0, st, p);
#undef DISTILL_WAVE
#undef DISTILL_ROW
#undef DISTILL_LANES
}

}  // namespace xrl

using namespace xrl;

extern "C" int xrl_distill_loss(const xrl_distill_t* pp, xrl_stream_t stream) {
    XRL_CHECK_ARG(pp != nullptr);
    const xrl_distill_t& p = *pp;
    XRL_CHECK_ARG(p.N >= 0 && p.N <= 0x7fffffff && p.A >= 1 && p.A <= 1 << 30 && p.K >= 1 && p.K <= DISTILL_MAX_K);
    XRL_CHECK_ARG((p.dtype == XRL_F32 || p.dtype == XRL_BF16) && p.temperature >= 1e-18f && p.temperature <= 1e18f);
    if (p.N == 0) return XRL_OK;
    XRL_CHECK_ARG(p.logits && p.teacher_idx && p.teacher_logits && p.loss);
    const int e = p.dtype == XRL_F32 ? 4 : 2;
    const arg_t a[] = {{"d_logits", p.d_logits, e, 2, {p.N, p.A}, {p.ld_d, 1}, true}, {"loss", p.loss, 4, 1, {p.N}, {1}, true},
                       {"logits", p.logits, e, 2, {p.N, p.A}, {p.ld, 1}, false}, {"teacher_idx", p.teacher_idx, 4, 2, {p.N, p.K}, {p.K, 1}, false},
                       {"teacher_logits", p.teacher_logits, e, 2, {p.N, p.K}, {p.K, 1}, false}, {"avail", p.avail, 4, 2, {p.N, p.A}, {p.A, 1}, false},
                       {"weight", p.weight, 4, 1, {p.N}, {1}, false}};
    const int pairs[][2] = {{0, 2}};
    if (int rc = check_args(a, 7, pairs, 1)) return rc;
    // a launch takes under 2^32 threads, and a row 1024 of them at most
    for (int64_t first = 0; first < p.N; first += 1 << 21) {
        xrl_distill_t r = p;
        r.N = p.N - first < 1 << 21 ? p.N - first : 1 << 21;
        r.logits = (const char*)p.logits + first * p.ld * e;
        r.teacher_idx = p.teacher_idx + first * p.K;
        r.teacher_logits = (const char*)p.teacher_logits + first * p.K * e;
        if (p.avail) r.avail = p.avail + first * p.A;
        if (p.weight) r.weight = p.weight + first;
        r.loss = p.loss + first;
        if (p.d_logits) r.d_logits = (char*)p.d_logits + first * p.ld_d * e;
        if (p.dtype == XRL_F32) launch_distill<float>(r, as_stream(stream));
        else launch_distill<bf16_t>(r, as_stream(stream));
        XRL_CHECK_LAUNCH();
    }
    return XRL_OK;
}
