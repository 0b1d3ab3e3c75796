// The chunked form of the operator of csrc/linattn.hip (see there), one workgroup per row, head, job and segment of the time axis:
//     mix_i = sum_{j <= i} lam^(i-j) (a_i . b_j) c_j + lam^(i+off) a_i S_in .
// With i, j counted inside a chunk of 64 steps and S the state before it,
//     O^T = S^T A^T diag(lam^(i+off)) + C^T P^T,   P_ij = lam^(i-j) (a_i . b_j) for j <= i,   S := lam^64 S + B^T diag(lam^(64-j-off)) C,
// four matrix products of a 64-step chunk instead of 64 dependent steps.
//
// Layout.  Wave w owns columns [16 w, 16 w + 16) of c, O and S; S stays in its accumulator registers for the whole segment.  The 16 x 16
// matrix instructions return D[m][n] with lane = n + 16 g holding m = 4 g + r and take an operand's k values as m or n = lane % 16, k by g.  Since
// the order of k inside a product is free as long as both operands agree, S [d][e] as returned (e = lane % 16, d = 4 g + r) IS the operand
// S^T of the first product, and P^T as returned leaves for LDS with four neighbouring j per lane.  So only the chunk's a, b, c and P pass through
// LDS.  The next chunk's rows are requested into registers before the current one is multiplied.
//
// Precision.  f32: f32 matrix instructions throughout.  bf16: products of stored bf16 values are exact and accumulate in f32; P and S enter their
// products as two bf16 parts (off by 2^-17 at most, the stored result by 2^-9), the weighted c enters the state as three (exact), so a state is as
// good as f32 sums make it.  Powers of lam are made in f64; lam^64, applied to the state at every chunk, keeps its rounding error as a second float.
#pragma once
#include "io16.h"

namespace xrl {

struct mix_job_t {
    const void* a; const void* b; const void* c; void* out;
    int64_t sa[3], sb[3], sc[3], so[3];
    int da, dc;
    const float* s_in; float* s_out;      // [B][H][.][.], element (d, e) of a row and head at d * sd + e * se
    int sd, se;
    int64_t s_row;                        // s_in: from row and head (and segment) to the next
    int reverse, off;
    int vec;                              // bit 0 a, 1 b, 2 c, 3 out: rows allow 16-byte (out: 4-element) accesses
    float scale_p, scale_s, scale_b;      // of the products a.b, of a S, of b (x) c in the state
    float* carry;                         // pass over the states of segments: what a segment multiplies the state by
};
struct mix_t {
    mix_job_t job[3];
    const float* log_decay; const int32_t* lengths; const float* reset;
    int T, B, H, kv;
    int n_jobs, n_seg, seg_chunks;
    int states_only;                      // write every segment's own state to s_out [row and head][segment] and its carry
};

constexpr int CH = 64;                    // steps of a chunk

template <typename E> struct mix_ops;

template <> struct mix_ops<float> {
    static constexpr int KB = 16, PAD = 4, PLANES = 1;          // k of one operand fragment, row padding in LDS, planes of P
    typedef f32x4_t frag;
    // four values of a row of LDS, k = 16 p + 4 g + r
    static __device__ __forceinline__ frag row(const float* r, int p, int g) { return *reinterpret_cast<const f32x4_t*>(r + 16 * p + 4 * g); }
    static __device__ __forceinline__ frag row_natural(const float* r, int p, int g) { return row(r, p, g); }
    // a column: rows 16 p + 4 g + r
    static __device__ __forceinline__ frag column(const float* base, int stride, int p, int g, int col) {
        const float* at = base + (16 * p + 4 * g) * stride + col;
        const f32x4_t v = {at[0], at[stride], at[2 * stride], at[3 * stride]};
        return v;
    }
    static __device__ __forceinline__ f32x4_t mfma(frag a, frag b, f32x4_t c) {
#pragma unroll
        for (int r = 0; r < 4; ++r) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[r], b[r], c, 0, 0, 0);
        return c;
    }
    // (state tiles as returned) x row fragment
    static __device__ __forceinline__ f32x4_t mfma_state(const f32x4_t* s, int p, frag b, f32x4_t c) { return mfma(s[p], b, c); }
    // column fragment x weights, as the second operand of the state's product
    struct weighted { frag v; };
    static __device__ __forceinline__ weighted weigh(frag v, const float* w) {
        weighted t;
#pragma unroll
        for (int r = 0; r < 4; ++r) t.v[r] = v[r] * w[r];
        return t;
    }
    static __device__ __forceinline__ f32x4_t mfma_weighted(frag a, const weighted& w, f32x4_t c) { return mfma(a, w.v, c); }
    static __device__ __forceinline__ void store_p(float* p, int plane, f32x4_t v) { (void)plane; *reinterpret_cast<f32x4_t*>(p) = v; }
    static __device__ __forceinline__ f32x4_t mfma_p(frag c, const float* p, int plane, int q, int g, f32x4_t o) { (void)plane; return mfma(c, row(p, q, g), o); }
    static __device__ __forceinline__ void store_out(float* o, f32x4_t v, bool vec, int left) {
        if (vec) { if (left > 0) *reinterpret_cast<f32x4_t*>(o) = v; }
        else
#pragma unroll
            for (int r = 0; r < 4; ++r) if (r < left) o[r] = v[r];
    }
};

template <> struct mix_ops<bf16_t> {
    static constexpr int KB = 32, PAD = 8, PLANES = 2;
    typedef u32x4_t frag;                                        // eight bf16
    typedef unsigned short u16;
    static __device__ __forceinline__ u32x2_t two(const bf16_t* p) { return *reinterpret_cast<const u32x2_t*>(p); }
    // k = 32 p + 4 g + r and 32 p + 16 + 4 g + r: the order in which two state tiles hold their rows
    static __device__ __forceinline__ frag row(const bf16_t* r, int p, int g) {
        const u32x2_t x = two(r + 32 * p + 4 * g), y = two(r + 32 * p + 16 + 4 * g);
        const frag v = {x.x, x.y, y.x, y.y};
        return v;
    }
    static __device__ __forceinline__ frag row_natural(const bf16_t* r, int p, int g) { return *reinterpret_cast<const u32x4_t*>(r + 32 * p + 8 * g); }
    // a column, rows 32 p + 8 g + 0..7, by the transposing LDS read (lane q of 16 names row q / 4, columns 4 (q % 4) and receives column q of
    // four rows).  col: the first of the 16 columns.
    static __device__ __forceinline__ frag column(const bf16_t* base, int stride, int p, int g, int col) {
        const int q = threadIdx.x & 15;
        typedef short s16x4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) s16x4* lptr;
        const bf16_t* at = base + (32 * p + 8 * g + (q >> 2)) * stride + (col - q) + 4 * (q & 3);
        const u32x2_t x = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lptr)at));
        const u32x2_t y = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lptr)(at + 4 * stride)));
        const frag v = {x.x, x.y, y.x, y.y};
        return v;
    }
    static __device__ __forceinline__ f32x4_t mfma(frag a, frag b, f32x4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ void split2(float x0, float x1, unsigned& h, unsigned& l) {
        h = cvt_pk_bf16(x0, x1);
        l = cvt_pk_bf16(x0 - __uint_as_float(h << 16), x1 - __uint_as_float(h & 0xffff0000u));
    }
    static __device__ __forceinline__ f32x4_t mfma_state(const f32x4_t* s, int p, frag b, f32x4_t c) {
        frag h, l;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const f32x4_t t = s[2 * p + (q >> 1)];
            unsigned x, y;
            split2(t[2 * (q & 1)], t[2 * (q & 1) + 1], x, y);
            h[q] = x; l[q] = y;
        }
        return mfma(h, b, mfma(l, b, c));
    }
    struct weighted { frag h, m, l; };
    static __device__ __forceinline__ weighted weigh(frag v, const float* w) {
        weighted t;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            unsigned x, y, z;
            split3_pair(__uint_as_float(v[q] << 16) * w[2 * q], __uint_as_float(v[q] & 0xffff0000u) * w[2 * q + 1], x, y, z);
            t.h[q] = x; t.m[q] = y; t.l[q] = z;
        }
        return t;
    }
    static __device__ __forceinline__ f32x4_t mfma_weighted(frag a, const weighted& w, f32x4_t c) { return mfma(a, w.h, mfma(a, w.m, mfma(a, w.l, c))); }
    static __device__ __forceinline__ void store_p(bf16_t* p, int plane, f32x4_t v) {
        unsigned h0, l0, h1, l1;
        split2(v[0], v[1], h0, l0);
        split2(v[2], v[3], h1, l1);
        const u32x2_t h = {h0, h1}, l = {l0, l1};
        *reinterpret_cast<u32x2_t*>(p) = h;
        *reinterpret_cast<u32x2_t*>(p + plane) = l;
    }
    static __device__ __forceinline__ f32x4_t mfma_p(frag c, const bf16_t* p, int plane, int q, int g, f32x4_t o) {
        return mfma(c, row_natural(p, q, g), mfma(c, row_natural(p + plane, q, g), o));
    }
    static __device__ __forceinline__ void store_out(bf16_t* o, f32x4_t v, bool vec, int left) {
        if (vec) {
            const u32x2_t t = {cvt_pk_bf16(v[0], v[1]), cvt_pk_bf16(v[2], v[3])};
            if (left > 0) *reinterpret_cast<u32x2_t*>(o) = t;
        } else
#pragma unroll
            for (int r = 0; r < 4; ++r) if (r < left) io_store(o + r, v[r]);
    }
};

// 64 rows of a tensor on their way from memory to LDS: N 16-byte pieces per thread, pieces of a row by neighbouring threads
template <typename E, int D, int NT>
struct mix_stage_t {
    static constexpr int PER = 16 / sizeof(E), ROW = D / PER, N = (CH * ROW + NT - 1) / NT, STRIDE = D + mix_ops<E>::PAD;
    u32x4_t v[N];
    // rows first .. first + 63 of n (in reversed time the rows counted from the end); absent rows and columns read as 0
    __device__ __forceinline__ void load(const E* base, int64_t stride, int first, int n, int reverse, int d, bool vec, int tid) {
#pragma unroll
        for (int q = 0; q < N; ++q) {
            const int at = tid + q * NT, r = at / ROW, c = (at % ROW) * PER, i = first + r;
            u32x4_t x = {0, 0, 0, 0};
            if ((N * NT == CH * ROW || r < CH) && i < n && c < d) {
                const E* row = base + (int64_t)(reverse ? n - 1 - i : i) * stride + c;
                if (vec) x = *reinterpret_cast<const u32x4_t*>(row);
                else {
                    if (sizeof(E) == 4) {
#pragma unroll
                        for (int m = 0; m < 4; ++m) x[m] = c + m < d ? reinterpret_cast<const unsigned*>(row)[m] : 0u;
                    } else {
#pragma unroll
                        for (int m = 0; m < 8; ++m) {
                            const unsigned e = c + m < d ? reinterpret_cast<const unsigned short*>(row)[m] : 0u;
                            x[m >> 1] |= e << (16 * (m & 1));
                        }
                    }
                }
            }
            v[q] = x;
        }
    }
    __device__ __forceinline__ void store(E* lds, int tid) const {
#pragma unroll
        for (int q = 0; q < N; ++q) {
            const int at = tid + q * NT, r = at / ROW, c = (at % ROW) * PER;
            if (N * NT == CH * ROW || r < CH) *reinterpret_cast<u32x4_t*>(lds + r * STRIDE + c) = v[q];
        }
    }
};

template <typename E, int DA, int NW>
struct mix_geom {
    static constexpr int DC = 16 * NW, NT = 64 * NW, SA = DA + mix_ops<E>::PAD, SC = DC + mix_ops<E>::PAD, SP = CH + mix_ops<E>::PAD;
    static constexpr int A = 0, B = A + CH * SA, C = B + CH * SA, P = C + CH * SC, END = P + mix_ops<E>::PLANES * CH * SP;
    static constexpr int BYTES = END * (int)sizeof(E);
};

template <typename E, int DA, int NW>
__global__ void __launch_bounds__(64 * NW) linattn_mix_kernel(mix_t p) {
    typedef mix_ops<E> M;
    typedef mix_geom<E, DA, NW> G;
    constexpr int NT = G::NT, NPA = DA / M::KB, NPC = CH / M::KB, TPP = M::KB / 16;      // fragments over DA, over a chunk; tiles per fragment
    extern __shared__ __attribute__((aligned(16))) unsigned char lds_raw[];
    E* la = reinterpret_cast<E*>(lds_raw) + G::A;
    E* lb = reinterpret_cast<E*>(lds_raw) + G::B;
    E* lc = reinterpret_cast<E*>(lds_raw) + G::C;
    E* lp = reinterpret_cast<E*>(lds_raw) + G::P;
    __shared__ float pw[CH + 1], wq[CH], wb[CH];
    __shared__ int seg_of[CH];
    // workgroups of one row and head follow each other on one XCD (ids go round the 8 of them): its jobs share their reads in that L2
    const int lin = blockIdx.x, turn = lin >> 3;
    const int job_i = turn % p.n_jobs, unit = (turn / p.n_jobs) * 8 + (lin & 7);
    if (unit >= p.B * p.H * p.n_seg) return;
    const mix_job_t& J = p.job[job_i];
    const int bh = unit / p.n_seg, seg = unit % p.n_seg, b = bh / p.H, h = bh % p.H;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), ln = lane & 15, g = lane >> 4;
    const int n = p.lengths ? min(max(p.lengths[b], 0), p.T) : p.T;
    const int c_first = seg * p.seg_chunks, c_end = min(c_first + p.seg_chunks, (n + CH - 1) / CH);
    const int da = J.da, dc = J.dc;
    const E* pa = (const E*)J.a + b * J.sa[1] + h * J.sa[2];
    const E* pb = (const E*)J.b + b * J.sb[1] + h * J.sb[2];
    const E* pc = (const E*)J.c + b * J.sc[1] + h * J.sc[2];
    E* po = (E*)J.out + b * J.so[1] + h * J.so[2];
    float gl = p.log_decay[h];
    gl = gl > 0.f ? 0.f : gl < -1e30f ? -1e30f : gl;
    if (tid <= CH) pw[tid] = (float)exp((double)gl * tid);
    if (NT == 64 && tid == 0) pw[CH] = (float)exp((double)gl * CH);
    const int n_last = n - (n - 1) / CH * CH;                       // steps of the row's last chunk (n > 0)
    const double full = exp((double)gl * CH), part = exp((double)gl * n_last);
    const float full_h = (float)full, full_l = (float)(full - (double)full_h), part_h = (float)part, part_l = (float)(part - (double)part_h);

    f32x4_t S[DA / 16];
    {
        const float* s = J.s_in ? J.s_in + ((int64_t)bh * p.n_seg + seg) * J.s_row : nullptr;
        const int e = 16 * w + ln;
#pragma unroll
        for (int t = 0; t < DA / 16; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int d = 16 * t + 4 * g + r;
                S[t][r] = (s && d < da && e < dc) ? s[d * J.sd + e * J.se] : 0.f;
            }
    }
    if (!p.states_only) {
        // P's tiles above the diagonal that share a fragment with one on it are read and stay 0
        if (TPP == 2)
            for (int at = tid; at < 2 * 32 * M::PLANES; at += NT) {
                const int plane = at / 64, r = at % 64, i = (r >> 4) * 32 + (r & 15);      // rows 0..15 and 32..47
                if (r < 32) {
                    u32x4_t* z = reinterpret_cast<u32x4_t*>(lp + plane * CH * G::SP + i * G::SP + (i & 32) + 16);
                    const u32x4_t zero = {0, 0, 0, 0};
                    z[0] = zero; z[1] = zero;
                }
            }
        // rows behind the sequence: 0
        const int lo = max(n, c_first * CH), hi = min(p.T, (c_first + p.seg_chunks) * CH);
        for (int64_t at = (int64_t)lo * dc + tid; at < (int64_t)hi * dc; at += NT) io_store(po + (at / dc) * J.so[0] + at % dc, 0.f);
    }

    // weights of the scores: lam^(16 dist + ln - (4 g + r)), masked above the diagonal, for the four distances of two tiles
    lds_barrier();
    float wd[4][4];
#pragma unroll
    for (int dist = 0; dist < 4; ++dist)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int k = 16 * dist + ln - 4 * g - r;
            wd[dist][r] = k >= 0 ? J.scale_p * pw[k] : 0.f;
        }

    mix_stage_t<E, DA, NT> ra, rb;
    mix_stage_t<E, G::DC, NT> rc;
    float rflag = 0.f;
    auto request = [&](int c) {
        const int first = c * CH;
        if (!p.states_only) ra.load(pa, J.sa[0], first, n, J.reverse, da, J.vec & 1, tid);
        rb.load(pb, J.sb[0], first, n, J.reverse, da, J.vec & 2, tid);
        rc.load(pc, J.sc[0], first, n, J.reverse, dc, J.vec & 4, tid);
        if (p.reset) {
            // what came before step i is cut off: by the reset of step i; in reversed time by that of the step behind it
            const int i = first + lane, t = J.reverse ? n - i : i;
            rflag = (i < n && t < n) ? p.reset[(int64_t)t * p.B + b] : 0.f;
        }
    };
    bool cut_any = false;
    if (c_first < c_end) request(c_first);
    for (int c = c_first; c < c_end; ++c) {
        const int nv = min(CH, n - c * CH);
        unsigned long long cuts = 0;
        if (p.reset) cuts = __ballot(rflag != 0.f);
        cut_any = cut_any || cuts != 0;
        if (!p.states_only) ra.store(la, tid);
        rb.store(lb, tid);
        rc.store(lc, tid);
        const int n_cuts = __popcll(cuts);
        if (tid < CH) {
            const int k = __popcll(cuts & (~0ull >> (63 - tid)));      // cuts up to and including this step
            seg_of[tid] = k;
            wq[tid] = k == 0 ? J.scale_s * pw[tid + J.off] : 0.f;
            wb[tid] = (tid < nv && k == n_cuts) ? J.scale_b * pw[nv - tid - J.off] : 0.f;
        }
        lds_barrier();
        if (c + 1 < c_end) request(c + 1);
        f32x4_t O[4];
        if (!p.states_only) {
            // P^T tiles on and below the diagonal, dealt out to the waves
            for (int t = w; t < 10; t += NW) {
                const int it = t < 1 ? 0 : t < 3 ? 1 : t < 6 ? 2 : 3, jt = t - it * (it + 1) / 2;
                f32x4_t s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int q = 0; q < NPA; ++q) s = M::mfma(M::row(lb + (16 * jt + ln) * G::SA, q, g), M::row(la + (16 * it + ln) * G::SA, q, g), s);
                const int dist = it - jt;
#pragma unroll
                for (int r = 0; r < 4; ++r) s[r] *= dist == 0 ? wd[0][r] : dist == 1 ? wd[1][r] : dist == 2 ? wd[2][r] : wd[3][r];
                if (cuts) {
                    const int k = seg_of[16 * it + ln];
#pragma unroll
                    for (int r = 0; r < 4; ++r) s[r] = seg_of[16 * jt + 4 * g + r] == k ? s[r] : 0.f;
                }
                M::store_p(lp + (16 * it + ln) * G::SP + 16 * jt + 4 * g, CH * G::SP, s);
            }
#pragma unroll
            for (int it = 0; it < 4; ++it) {
                f32x4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int q = 0; q < NPA; ++q) o = M::mfma_state(S, q, M::row(la + (16 * it + ln) * G::SA, q, g), o);
                const float f = wq[16 * it + ln];
#pragma unroll
                for (int r = 0; r < 4; ++r) o[r] *= f;
                O[it] = o;
            }
            lds_barrier();
        }
        {
            const bool last = nv < CH || (c + 1) * CH == n;
            float ch = full_h, cl = full_l;
            if (last) { ch = part_h; cl = part_l; }
            if (cuts) ch = cl = 0.f;
#pragma unroll
            for (int t = 0; t < DA / 16; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) S[t][r] = __builtin_fmaf(S[t][r], ch, S[t][r] * cl);
        }
#pragma unroll
        for (int q = 0; q < NPC; ++q) {
            const typename M::frag cf = M::column(lc, G::SC, q, g, 16 * w + ln);
            if (!p.states_only) {
#pragma unroll
                for (int it = 0; it < 4; ++it)
                    if (q * TPP <= it) O[it] = M::mfma_p(cf, lp + (16 * it + ln) * G::SP, CH * G::SP, q, g, O[it]);
            }
            float wv[M::KB / 4];
#pragma unroll
            for (int r = 0; r < M::KB / 4; ++r) wv[r] = wb[M::KB * q + (M::KB / 4) * g + r];
            const typename M::weighted cw = M::weigh(cf, wv);
#pragma unroll
            for (int t = 0; t < DA / 16; ++t) S[t] = M::mfma_weighted(M::column(lb, G::SA, q, g, 16 * t + ln), cw, S[t]);
        }
        if (!p.states_only) {
            const int e = 16 * w + 4 * g;
#pragma unroll
            for (int it = 0; it < 4; ++it) {
                const int i = c * CH + 16 * it + ln;
                if (i < n) M::store_out(po + (int64_t)(J.reverse ? n - 1 - i : i) * J.so[0] + e, O[it], J.vec & 8, dc - e);
            }
        }
        lds_barrier();
    }
    const int e = 16 * w + ln;
    if (p.states_only) {
        const int64_t at = ((int64_t)bh * p.n_seg + seg);
        float* s = J.s_out + at * J.da * J.dc;
#pragma unroll
        for (int t = 0; t < DA / 16; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int d = 16 * t + 4 * g + r;
                if (d < da && e < dc) s[d * dc + e] = S[t][r];
            }
        if (tid == 0) {
            const int steps = max(0, min(n, (c_first + p.seg_chunks) * CH) - c_first * CH);
            const double f = exp((double)gl * steps);
            J.carry[2 * at] = cut_any ? 0.f : (float)f;
            J.carry[2 * at + 1] = cut_any ? 0.f : (float)(f - (double)(float)f);
        }
    } else if (J.s_out && p.n_seg == 1) {
        const bool none = J.off == 0 && n > 0 && p.reset && p.reset[b] != 0.f;      // the gradient stops at a reset before the first step
#pragma unroll
        for (int t = 0; t < DA / 16; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int d = 16 * t + 4 * g + r;
                if (d < da && e < dc) J.s_out[(int64_t)bh * p.kv + (int64_t)d * J.sd + (int64_t)e * J.se] = none ? 0.f : S[t][r];
            }
    }
}

template <typename E, int DA, int NW>
static int launch_mix_as(const mix_t& m, hipStream_t s) {
    typedef mix_geom<E, DA, NW> G;
    static_assert(G::BYTES + 1200 <= 160 * 1024, "LDS");
    const int64_t units = ((int64_t)m.B * m.H * m.n_seg + 7) / 8 * 8;
    hipLaunchKernelGGL((linattn_mix_kernel<E, DA, NW>), dim3((unsigned)(units * m.n_jobs)), dim3(64 * NW), G::BYTES, s, m);
    XRL_CHECK_LAUNCH();
    return XRL_OK;
}

template <typename E, int DA, int NW>
static int init_mix_as() {
    XRL_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(linattn_mix_kernel<E, DA, NW>), hipFuncAttributeMaxDynamicSharedMemorySize,
                                      mix_geom<E, DA, NW>::BYTES));
    return XRL_OK;
}

// the instances that take more than 64 KB of LDS
template <typename E>
static int init_mix() {
    if (int rc = init_mix_as<E, 64, 4>()) return rc;
    if (int rc = init_mix_as<E, 64, 8>()) return rc;
    if (int rc = init_mix_as<E, 128, 4>()) return rc;
    return init_mix_as<E, 128, 8>();
}

// da, dc: the largest of the jobs'
template <typename E>
static int launch_mix(const mix_t& m, int da, int dc, hipStream_t s) {
    const int nw = dc <= 16 ? 1 : dc <= 32 ? 2 : dc <= 64 ? 4 : 8;
    if (sizeof(E) == 4 && da <= 16) {
        if (nw == 1) return launch_mix_as<E, sizeof(E) == 4 ? 16 : 32, 1>(m, s);
        if (nw == 2) return launch_mix_as<E, sizeof(E) == 4 ? 16 : 32, 2>(m, s);
        if (nw == 4) return launch_mix_as<E, sizeof(E) == 4 ? 16 : 32, 4>(m, s);
        return launch_mix_as<E, sizeof(E) == 4 ? 16 : 32, 8>(m, s);
    }
    if (da <= 32) {
        if (nw == 1) return launch_mix_as<E, 32, 1>(m, s);
        if (nw == 2) return launch_mix_as<E, 32, 2>(m, s);
        if (nw == 4) return launch_mix_as<E, 32, 4>(m, s);
        return launch_mix_as<E, 32, 8>(m, s);
    }
    if (da <= 64) {
        if (nw <= 2) return launch_mix_as<E, 64, 2>(m, s);
        if (nw == 4) return launch_mix_as<E, 64, 4>(m, s);
        return launch_mix_as<E, 64, 8>(m, s);
    }
    if (nw <= 4) return launch_mix_as<E, 128, 4>(m, s);
    return launch_mix_as<E, 128, 8>(m, s);
}

int launch_mix_f32(const mix_t& m, int da, int dc, hipStream_t s);
int launch_mix_bf16(const mix_t& m, int da, int dc, hipStream_t s);
int init_mix_f32();
int init_mix_bf16();

}  // namespace xrl
