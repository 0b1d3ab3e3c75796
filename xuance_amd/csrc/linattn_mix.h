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
// Precision.  f32: f32 matrix instructions throughout.  bf16: products of stored bf16 values are exact and accumulate in f32; the f32 operands that
// are made here (P, S, the weighted c) enter their products as three bf16 parts, which together are the f32 value (csrc/split3.h).  So either type
// computes what f32 sums make of its inputs, and a bf16 result is rounded once, where it is stored.  Powers of lam are made in f64; lam^64, applied
// to the state at every chunk, keeps its rounding error as a second float.
//
// Bound.  f32: the matrix instructions (half of a large product's rate): 256 rows x 256 steps, 4 heads of 64: 91 us forward, 229 us the three gradients,
// in a run of hundreds of passes (the first 20 after a pause take a fifth more).
// bf16, heads of 128: a chunk takes a compute unit 10.9 k cycles, 35% of them matrix instructions, 46% vector instructions (three-part operands, decays),
// 35% LDS, mostly one after another in the two workgroups that registers and LDS allow; 8 ragged rows x 4096 steps, 8 heads: 77 us forward and 35 + 16 us for
// the states of its segments and their joining, 220 us and 66 + 29 us the gradients.  (With two-part operands, 17 bits of them, 9.7 k cycles a chunk; in turn on one
// card: this case 373 us with two, 429 with three.)
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
    float scale_p, scale_s, scale_b;      // of the products a.b, of a S, of b (x) c in the state
    float* carry;                         // pass over the states of segments: what a segment multiplies the state by; below 0 where a reset ends it
};
struct mix_t {
    mix_job_t job[3];
    const float* log_decay; const int32_t* lengths; const float* reset;
    int T, B, H, kv;
    int n_jobs, n_seg, n_slices;          // every row is cut into n_seg segments of equally many chunks, by its own length
    int states_only;                      // write every segment's own state to s_out [row and head][segment] and its carry
};

constexpr int CH = 64;                    // steps of a chunk

template <typename E, int TS> struct mix_ops;

// Operands by fragments: KB values of k of 16 rows or columns.  A product of fragments takes STEPS matrix instructions; an f32 operand that is made
// here (P, the state, the weighted c) takes P_PARTS, S_PARTS, W_PARTS fragments.
template <> struct mix_ops<float, 16> {
    static constexpr int KB = 16, PAD_A = 4, PAD_B = 4, PAD_C = 4, PAD_P = 4, SLOTS = 4, STEPS = 4, P_PARTS = 1, S_PARTS = 1, W_PARTS = 1;
    typedef f32x4_t frag;
    typedef f32x4_t acc;
    // four values of a row of LDS, k = 16 p + 4 g + r
    static __device__ __forceinline__ frag row(const float* r, int p, int g) { return *reinterpret_cast<const f32x4_t*>(r + 16 * p + 4 * g); }
    static __device__ __forceinline__ frag row_natural(const float* r, int p, int g) { return row(r, p, g); }
    // a column: rows 16 p + 4 g + r
    static __device__ __forceinline__ frag column(const float* base, int stride, int p, int g, int col) {
        const float* at = base + (16 * p + 4 * g) * stride + col;
        const f32x4_t v = {at[0], at[stride], at[2 * stride], at[3 * stride]};
        return v;
    }
    static __device__ __forceinline__ acc mfma(frag a, frag b, acc c, int step) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a[step], b[step], c, 0, 0, 0); }
    static __device__ __forceinline__ void of_state(const acc* s, int p, frag (&f)[1]) { f[0] = s[p]; }
    static __device__ __forceinline__ void weigh(frag v, const float* w, frag (&f)[1]) {
#pragma unroll
        for (int r = 0; r < 4; ++r) f[0][r] = v[r] * w[r];
    }
    static __device__ __forceinline__ void store_p(float* p, int plane, f32x4_t v) { (void)plane; *reinterpret_cast<f32x4_t*>(p) = v; }
    static __device__ __forceinline__ void store_out(float* o, f32x4_t v) { *reinterpret_cast<f32x4_any_t*>(o) = v; }
};

// what both tile sizes of bf16 share
struct mix_bf16 {
    // LDS rows: read 8 bytes of each of 16 rows at a time (a), by transposing reads of 32 bytes of 4 rows (c), both (b) or 16 bytes of 8 rows (P); each wants
    // its rows to fall behind each other in the 32 banks.  With 8 for all, half of the cycles that LDS was busy were conflicts.
    static constexpr int PAD_A = 4, PAD_B = 8, PAD_C = 16, PAD_P = 8, SLOTS = 8, STEPS = 1, P_PARTS = 3, S_PARTS = 3, W_PARTS = 3;
    typedef u32x4_t frag;                                        // eight bf16
    static __device__ __forceinline__ u32x2_t two(const bf16_t* p) { return *reinterpret_cast<const u32x2_t*>(p); }
    static __device__ __forceinline__ frag join(u32x2_t x, u32x2_t y) { return frag{x.x, x.y, y.x, y.y}; }
    // eight rows of a column by two transposing LDS reads: lane q of 16 names row q / 4, columns 4 (q % 4) and receives column q of four rows
    static __device__ __forceinline__ frag column16(const bf16_t* first, int stride) {
        const int q = threadIdx.x & 15;
        typedef short s16x4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) s16x4* lptr;
        const bf16_t* at = first + (q >> 2) * stride + 4 * (q & 3);
        return join(__builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lptr)at)),
                    __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lptr)(at + 4 * stride))));
    }
    static __device__ __forceinline__ void weigh(frag v, const float* w, frag (&f)[3]) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            unsigned h, m, l;
            split3_pair(__uint_as_float(v[q] << 16) * w[2 * q], __uint_as_float(v[q] & 0xffff0000u) * w[2 * q + 1], h, m, l);
            f[0][q] = h; f[1][q] = m; f[2][q] = l;
        }
    }
    static __device__ __forceinline__ void store_p(bf16_t* p, int plane, f32x4_t v) {
        unsigned h0, m0, l0, h1, m1, l1;
        split3_pair(v[0], v[1], h0, m0, l0);
        split3_pair(v[2], v[3], h1, m1, l1);
        const u32x2_t h = {h0, h1}, m = {m0, m1}, l = {l0, l1};
        *reinterpret_cast<u32x2_t*>(p) = h;
        *reinterpret_cast<u32x2_t*>(p + plane) = m;
        *reinterpret_cast<u32x2_t*>(p + 2 * plane) = l;
    }
    static __device__ __forceinline__ void store_out(bf16_t* o, f32x4_t v) {
        typedef u32x2_t any_t __attribute__((aligned(2)));
        *reinterpret_cast<any_t*>(o) = u32x2_t{cvt_pk_bf16(v[0], v[1]), cvt_pk_bf16(v[2], v[3])};
    }
};

template <> struct mix_ops<bf16_t, 16> : mix_bf16 {
    static constexpr int KB = 32;
    typedef f32x4_t acc;
    // k = 32 p + 4 g + r and 32 p + 16 + 4 g + r: the order in which two state tiles hold their rows
    static __device__ __forceinline__ frag row(const bf16_t* r, int p, int g) { return join(two(r + 32 * p + 4 * g), two(r + 32 * p + 16 + 4 * g)); }
    static __device__ __forceinline__ frag row_natural(const bf16_t* r, int p, int g) { return *reinterpret_cast<const u32x4_t*>(r + 32 * p + 8 * g); }
    static __device__ __forceinline__ frag column(const bf16_t* base, int stride, int p, int g, int col) {
        return column16(base + (32 * p + 8 * g) * stride + (col & ~15), stride);
    }
    static __device__ __forceinline__ acc mfma(frag a, frag b, acc c, int) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ void of_state(const acc* s, int p, frag (&f)[3]) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const acc t = s[2 * p + (q >> 1)];
            unsigned h, m, l;
            split3_pair(t[2 * (q & 1)], t[2 * (q & 1) + 1], h, m, l);
            f[0][q] = h; f[1][q] = m; f[2][q] = l;
        }
    }
};

// tiles of 32: half the LDS reads for the same products, twice the accumulators
template <> struct mix_ops<bf16_t, 32> : mix_bf16 {
    static constexpr int KB = 16;
    typedef f32x16_t acc;
    // k = 16 p + 4 g + r and 16 p + 8 + 4 g + r: the order in which half a state tile holds its rows
    static __device__ __forceinline__ frag row(const bf16_t* r, int p, int g) { return join(two(r + 16 * p + 4 * g), two(r + 16 * p + 8 + 4 * g)); }
    static __device__ __forceinline__ frag row_natural(const bf16_t* r, int p, int g) { return *reinterpret_cast<const u32x4_t*>(r + 16 * p + 8 * g); }
    static __device__ __forceinline__ frag column(const bf16_t* base, int stride, int p, int g, int col) {
        return column16(base + (16 * p + 8 * g) * stride + (col & ~15), stride);
    }
    static __device__ __forceinline__ acc mfma(frag a, frag b, acc c, int) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ void of_state(const acc* s, int p, frag (&f)[3]) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            unsigned h, m, l;
            split3_pair(s[p >> 1][8 * (p & 1) + 2 * q], s[p >> 1][8 * (p & 1) + 2 * q + 1], h, m, l);
            f[0][q] = h; f[1][q] = m; f[2][q] = l;
        }
    }
};

// s elements off the low end of 16 bytes, 0 in at the high end
template <typename E>
__device__ __forceinline__ u32x4_t drop_low(u32x4_t v, int s) {
    const int bits = s * 8 * (int)sizeof(E), words = bits >> 5, rest = bits & 31;
    u32x4_t a;
#pragma unroll
    for (int m = 0; m < 4; ++m) {
        unsigned x = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (m + k < 4) x = words == k ? v[m + k] : x;
        a[m] = x;
    }
    if (sizeof(E) == 2 && rest) {
#pragma unroll
        for (int m = 0; m < 4; ++m) a[m] = (a[m] >> 16) | (m < 3 ? a[m + 1] << 16 : 0u);
    }
    return a;
}

// 64 rows of a tensor on their way from memory to LDS: N 16-byte pieces per thread, pieces of a row by neighbouring threads.  Rows come in
// the order of memory and are turned round in LDS for reversed time.  Requests are never conditional -- a load under a branch makes the
// compiler wait for all loads wherever one is used -- but stay inside the tensor: rows behind the sequence are requested as its last one,
// pieces behind the row's end from its last 16 bytes; store() puts that right.
// FULL: d is D, and 64 rows span less than 2 GB: an address is a scalar base and a 32-bit offset that the thread keeps.
template <typename E, int D, int NT, bool FULL, int PAD>
struct mix_stage_t {
    static constexpr int PER = 16 / sizeof(E), ROW = D / PER, N = (CH * ROW + NT - 1) / NT, STRIDE = D + PAD, STEP = NT / ROW;
    static constexpr bool ALL = N * NT == CH * ROW;             // else the threads left over request what is there already, and store nothing
    u32x4_t v[N];
    const E* base;
    int64_t stride;
    int d, n, reverse;
    __device__ __forceinline__ void begin(const E* base_, int64_t stride_, int d_, int n_, int reverse_) {
        base = base_; stride = stride_; d = d_; n = n_; reverse = reverse_;
    }
    // this thread's first row and its element of a row
    static __device__ __forceinline__ int first_row(int tid) { return ALL ? tid / ROW : min(tid / ROW, CH - 1); }
    static __device__ __forceinline__ int first_at(int tid) { return (tid % ROW) * PER; }
    // steps first .. first + 63 of n > first
    __device__ __forceinline__ void load(int first, int tid) {
        const int row0 = first_row(tid), at0 = first_at(tid);
        const int left = n - first, low = reverse ? left - CH : first;          // memory row of the chunk's first row (can be below 0)
        const int row_min = reverse ? max(CH - left, 0) : 0, row_max = reverse ? CH - 1 : min(left, CH) - 1;
        const char* at = reinterpret_cast<const char*>(base + (int64_t)low * stride);
        if (FULL && left >= CH) {
            const unsigned off0 = (unsigned)row0 * (unsigned)((int)stride * (int)sizeof(E)) + (unsigned)at0 * (unsigned)sizeof(E);
#pragma unroll
            for (int q = 0; q < N; ++q) v[q] = row16<E>::load(reinterpret_cast<const E*>(at + (int64_t)(q * STEP) * stride * (int)sizeof(E) + off0));
        } else {
#pragma unroll
            for (int q = 0; q < N; ++q) {
                const E* row = reinterpret_cast<const E*>(at) + (int64_t)min(max(row0 + q * STEP, row_min), row_max) * stride;
                if (FULL || d >= PER) v[q] = row16<E>::load(row + (FULL ? at0 : min(at0, d - PER)));
                else {
#pragma unroll
                    for (int m = 0; m < PER; ++m) row16<E>::put(v[q], m, row16<E>::bits(row + min(at0 + m, d - 1)));
                }
            }
        }
    }
    __device__ __forceinline__ void store(E* lds, int left, int tid) {
        const int row0 = first_row(tid), at0 = first_at(tid);
        if (!FULL || left < CH) {
#pragma unroll
            for (int q = 0; q < N; ++q) {
                const int row = row0 + q * STEP;
                const u32x4_t zero = {0, 0, 0, 0};
                if (!FULL) {
                    if (d < PER) {
#pragma unroll
                        for (int m = 0; m < PER; ++m)
                            if (at0 + m >= d) row16<E>::put(v[q], m, 0u);
                    } else if (at0 + PER > d) v[q] = at0 < d ? drop_low<E>(v[q], at0 + PER - d) : zero;
                }
                if ((reverse ? CH - 1 - row : row) >= left) v[q] = zero;
            }
        }
        if (ALL || tid < CH * ROW) {
            E* to = lds + (reverse ? CH - 1 - row0 : row0) * STRIDE + at0;
            const int step = reverse ? -STEP * STRIDE : STEP * STRIDE;
#pragma unroll
            for (int q = 0; q < N; ++q) {
                if (STRIDE * sizeof(E) % 16 == 0) *reinterpret_cast<u32x4_t*>(to + q * step) = v[q];
                else {
                    *reinterpret_cast<u32x2_t*>(to + q * step) = u32x2_t{v[q].x, v[q].y};
                    *reinterpret_cast<u32x2_t*>(to + q * step + PER / 2) = u32x2_t{v[q].z, v[q].w};
                }
            }
        }
    }
};

constexpr int up(int bytes) { return (bytes + 1279) / 1280 * 1280; }                   // LDS is given out in pieces of this size

template <typename E, int TS, int DA, int NW>
struct mix_geom {
    typedef mix_ops<E, TS> M;
    static constexpr int DC = TS * NW, NT = 64 * NW, SA = DA + M::PAD_A, SB = DA + M::PAD_B, SC = DC + M::PAD_C, SP = CH + M::PAD_P;
    static constexpr int P_SIZE = M::P_PARTS * CH * SP, P_TILES = (CH / TS) * (CH / TS + 1) / 2, MINE = (P_TILES + NW - 1) / NW;
    // P in the place of A, which costs a barrier, where a wave's tiles of P fit its registers and a third workgroup fits the compute unit for it:
    // 256 rows of 256 steps, 4 heads of 64, f32, forward and backward 349 us with two workgroups, 319 with three
    static constexpr int OTHER = 1280, OVER_SIZE = P_SIZE > CH * SA ? P_SIZE : CH * SA;
    static constexpr bool OVER = M::KB == TS && MINE <= 3 && 160 * 1024 / up((CH * (SA + SB + SC) + P_SIZE) * (int)sizeof(E) + OTHER) == 2 &&
                                 160 * 1024 / up((OVER_SIZE + CH * (SB + SC)) * (int)sizeof(E) + OTHER) == 3;
    static constexpr int A = 0, B = A + (OVER ? OVER_SIZE : CH * SA), C = B + CH * SB, P = OVER ? A : C + CH * SC, END = OVER ? C + CH * SC : P + P_SIZE;
    static constexpr int BYTES = END * (int)sizeof(E), HELD = 160 * 1024 / up(BYTES + OTHER);          // workgroups that LDS has room for
    static constexpr int MIN_WAVES = OVER ? 3 : NW * HELD >= 8 ? 2 : 1;
};

// between scheduling fences: V vector instructions behind each of N matrix instructions, which run meanwhile
template <int N, int V>
__device__ __forceinline__ void mix_interleave(bool both) {
    if (both) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, V, 0);
        }
    }
    __builtin_amdgcn_sched_barrier(0);
}

template <typename E, int TS, int DA, int NW, bool FULL>
__global__ void __launch_bounds__(64 * NW, (mix_geom<E, TS, DA, NW>::MIN_WAVES)) linattn_mix_kernel(mix_t p) {
    typedef mix_ops<E, TS> M;
    typedef mix_geom<E, TS, DA, NW> G;
    typedef typename M::frag frag;
    typedef typename M::acc acc;
    constexpr int NT = G::NT, TILES = DA / TS, IT = CH / TS, NPA = DA / M::KB, NPC = CH / M::KB;       // tiles of S and of O; fragments over DA, over a chunk
    constexpr int AR = TS * TS / 64, QUADS = AR / 4;               // a lane's values of a tile, in runs of four neighbouring rows: 8 quad + 4 g (32) or 4 g
    constexpr int PLANE = CH * G::SP;
    extern __shared__ __attribute__((aligned(16))) unsigned char lds_raw[];
    E* la = reinterpret_cast<E*>(lds_raw) + G::A;
    E* lb = reinterpret_cast<E*>(lds_raw) + G::B;
    E* lc = reinterpret_cast<E*>(lds_raw) + G::C;
    E* lp = reinterpret_cast<E*>(lds_raw) + G::P;
    // powers of lam: 0..64 and that of the last chunk's steps (of the last two also the rounding error); those of the scores by i - j + 32, 0 for i < j; weights of c by step, of
    // whole chunks without a cut [0] and of the chunk at hand otherwise [1]
    __shared__ float pw[CH + 2], pw_low[2], score_w[CH + 32], wb[2][CH];
    __shared__ unsigned char seg_of[CH];
    static_assert(sizeof(pw) + sizeof(pw_low) + sizeof(score_w) + sizeof(wb) + sizeof(seg_of) <= G::OTHER, "LDS");
    // workgroups of one row and head follow each other on one XCD (ids go round the 8 of them): its jobs share their reads in that L2
    const int lin = blockIdx.x, turn = lin >> 3, both = turn % (p.n_jobs * p.n_slices);
    const int job_i = both / p.n_slices, unit = turn / (p.n_jobs * p.n_slices) * 8 + (lin & 7);
    if (unit >= p.B * p.H * p.n_seg) return;
    const mix_job_t& J = p.job[job_i];
    const int seg = unit % p.n_seg, h = unit / p.n_seg % p.H, nth = unit / p.n_seg / p.H;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), ln0 = lane % TS, g0 = lane / TS;
    typedef const __attribute__((address_space(4))) int* scalar_int_t;
    int b = nth;
    if (p.lengths && p.B <= 64) {
        // few rows: the longest first, so that the last workgroups to end are short ones (8 ragged rows of 4096 steps, forward and backward, 433 -> 411 us;
        // more rows even out by themselves)
        const int mine = lane < p.B ? min(max(p.lengths[lane], 0), p.T) : -1;
        int longer = 0;
        for (int k = 0; k < p.B; ++k) {
            const int other = __builtin_amdgcn_readlane(mine, k);
            longer += other > mine || (other == mine && k < lane) ? 1 : 0;
        }
        b = __builtin_ctzll(__ballot(lane < p.B && longer == nth));
    }
    const int bh = b * p.H + h;
    const int n = p.lengths ? min(max(((scalar_int_t)(uintptr_t)p.lengths)[b], 0), p.T) : p.T;
    const int seg_chunks = ((n + CH - 1) / CH + p.n_seg - 1) / p.n_seg, c_first = seg * seg_chunks, c_end = min(c_first + seg_chunks, (n + CH - 1) / CH);
    const int c0 = (both % p.n_slices) * G::DC;                     // the slice of c's columns
    const int da = FULL ? DA : J.da, dc = FULL ? G::DC : min(J.dc - c0, G::DC), reverse = J.reverse, off = J.off;
    if (!FULL && dc <= 0) return;                                   // a job of fewer columns than the widest
    const bool states_only = p.states_only;
    const float scale_p = J.scale_p, scale_s = J.scale_s, scale_b = J.scale_b;
    const float* reset = p.reset;
    E* po = (E*)J.out + b * J.so[1] + h * J.so[2] + c0;
    const int64_t so = J.so[0];

    mix_stage_t<E, DA, NT, FULL, M::PAD_A> ra;
    mix_stage_t<E, DA, NT, FULL, M::PAD_B> rb;
    mix_stage_t<E, G::DC, NT, FULL, M::PAD_C> rc;
    ra.begin((const E*)J.a + b * J.sa[1] + h * J.sa[2], J.sa[0], da, n, reverse);
    rb.begin((const E*)J.b + b * J.sb[1] + h * J.sb[2], J.sb[0], da, n, reverse);
    rc.begin((const E*)J.c + b * J.sc[1] + h * J.sc[2] + c0, J.sc[0], dc, n, reverse);
    float rflag = 0.f;
    auto request = [&](int c, int tid) {
        const int first = c * CH;
        if (!states_only) ra.load(first, tid);
        rb.load(first, tid);
        rc.load(first, tid);
        if (reset) {
            // what came before step i is cut off: by the reset of step i; in reversed time by that of the step behind it
            const int i = first + lane, t = reverse ? n - i : i;
            rflag = reset[(int64_t)min(max(t, 0), n - 1) * p.B + b];           // of another step where there is none: see below
        }
    };
    typedef const __attribute__((address_space(4))) float* scalar_t;
    float gl = ((scalar_t)(uintptr_t)p.log_decay)[h];               // before the rows are requested: vector loads come back in order
    if (c_first < c_end) request(c_first, tid);
    gl = gl > 0.f ? 0.f : gl < -1e30f ? -1e30f : gl;
    const int n_last = n - (n - 1) / CH * CH;                       // steps of the row's last chunk (n > 0)
    for (int k = tid; k < CH + 2; k += NT) {
        const double f = exp((double)gl * (k <= CH ? k : n_last));
        pw[k] = (float)f;
        if (k >= CH) pw_low[k - CH] = (float)(f - (double)(float)f);
    }
    acc S[TILES];
    {
        const float* s = J.s_in;
        const int e = TS * w + ln0;
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int r = 0; r < AR; ++r) S[t][r] = 0.f;
        if (s) {
            s += ((int64_t)bh * p.n_seg + seg) * J.s_row + (c0 + e) * J.se;
            const int sd = J.sd;
#pragma unroll
            for (int t = 0; t < TILES; ++t)
#pragma unroll
                for (int r = 0; r < AR; ++r) {
                    const int d = TS * t + 8 * (r >> 2) + 4 * g0 + (r & 3);
                    if (FULL || (d < da && e < dc)) S[t][r] = s[d * sd];
                }
        }
    }
    if (!states_only) {
        // P's tiles above the diagonal that share a fragment with one on it are read and stay 0
        if (M::KB > TS)
            for (int at = tid; at < 32 * M::P_PARTS; at += NT) {
                const int i = ((at >> 4) & 1) * 32 + (at & 15);                           // rows 0..15 and 32..47
                u32x4_t* z = reinterpret_cast<u32x4_t*>(lp + (at >> 5) * PLANE + i * G::SP + (i & 32) + 16);
                const u32x4_t zero = {0, 0, 0, 0};
                z[0] = zero; z[1] = zero;
            }
        // rows behind the sequence: 0
        constexpr int PIECES = G::DC / 4;
        for (int r = n + seg * (NT / PIECES) + tid / PIECES; r < p.T; r += p.n_seg * (NT / PIECES)) {
            const int e = tid % PIECES * 4;
            E* o = po + (int64_t)r * so + e;
            if (e + 4 <= dc) M::store_out(o, f32x4_t{0.f, 0.f, 0.f, 0.f});
            else
                for (int m = 0; e + m < dc; ++m) io_store(o + m, 0.f);
        }
    }
    lds_barrier();
    for (int k = tid; k < CH + 32; k += NT) score_w[k] = k < 32 ? 0.f : scale_p * pw[k - 32];
    if (tid < CH) {
        wb[0][tid] = scale_b * pw[CH - tid - off];
    }

    bool cut_any = false;
    for (int c = c_first; c < c_end; ++c) {
        const int left = n - c * CH;
        int ln = ln0, g = g0, tx = tid;
        asm volatile("" : "+v"(ln), "+v"(g), "+v"(tx));             // addresses are made anew: kept over the loop they would not fit the registers
        unsigned long long cuts = 0;
        if (reset) {
            const int i = c * CH + lane;
            cuts = __ballot(rflag != 0.f && i < n && (!reverse || i > 0));
        }
        cut_any = cut_any || cuts != 0;
        if (!states_only) ra.store(la, left, tx);
        rb.store(lb, left, tx);
        rc.store(lc, left, tx);
        const int own_w = cuts != 0 || left < CH ? 1 : 0;
        if (own_w && tid < CH) {
            const int nv = min(left, CH), k = __popcll(cuts & (~0ull >> (63 - tid)));      // cuts up to and including this step
            const float x = pw[max(nv - tid - off, 0)];
            seg_of[tid] = (unsigned char)k;
            wb[1][tid] = tid < nv && k == __popcll(cuts) ? scale_b * x : 0.f;
        }
        lds_barrier();
        if (c + 1 < c_end) request(c + 1, tx);
        acc O[IT];
        if (!states_only) {
            // P^T tiles on and below the diagonal, dealt out to the waves, up to three at a time
            constexpr int ALL_P = G::P_TILES, MINE = G::MINE, AT_ONCE = MINE < 3 ? MINE : 3;
            acc s[AT_ONCE];
            int it[AT_ONCE], jt[AT_ONCE];
            auto store_scores = [&](int t0) {
#pragma unroll
                for (int k = 0; k < AT_ONCE; ++k)
#pragma unroll
                    for (int x = 0; x < QUADS; ++x)
                        if (t0 + k < MINE)
                            M::store_p(lp + (TS * it[k] + ln) * G::SP + TS * jt[k] + 8 * x + 4 * g, PLANE,
                                       f32x4_t{s[k][4 * x], s[k][4 * x + 1], s[k][4 * x + 2], s[k][4 * x + 3]});
            };
#pragma unroll
            for (int t0 = 0; t0 < MINE; t0 += AT_ONCE) {
                const E *ax[AT_ONCE], *bx[AT_ONCE];
                float sw[AT_ONCE][AR];
#pragma unroll
                for (int k = 0; k < AT_ONCE; ++k) {
                    const int t = min(w + (t0 + k) * NW, ALL_P - 1);                  // a wave without one repeats the last: the same values again
                    it[k] = t < 1 ? 0 : t < 3 ? 1 : t < 6 ? 2 : 3;
                    jt[k] = t - it[k] * (it[k] + 1) / 2;
#pragma unroll
                    for (int r = 0; r < AR; ++r) s[k][r] = 0.f;
                    ax[k] = la + (TS * it[k] + ln) * G::SA;
                    bx[k] = lb + (TS * jt[k] + ln) * G::SB;
                }
                frag fa[2][AT_ONCE], fb[2][AT_ONCE];
#pragma unroll
                for (int q = 0; q <= NPA; ++q) {                                      // one fragment ahead of the matrix instructions
                    if (q < NPA) {
#pragma unroll
                        for (int k = 0; k < AT_ONCE; ++k) { fb[q & 1][k] = M::row(bx[k], q, g); fa[q & 1][k] = M::row(ax[k], q, g); }
                    } else {
#pragma unroll
                        for (int k = 0; k < AT_ONCE; ++k)
#pragma unroll
                            for (int r = 0; r < AR; ++r) sw[k][r] = (score_w + (5 + ln - 4 * g + TS * (it[k] - jt[k])))[27 - 8 * (r >> 2) - (r & 3)];
                    }
                    if (q > 0) {
#pragma unroll
                        for (int x = 0; x < M::STEPS; ++x)
#pragma unroll
                            for (int k = 0; k < AT_ONCE; ++k)
                                if (t0 + k < MINE) s[k] = M::mfma(fb[(q - 1) & 1][k], fa[(q - 1) & 1][k], s[k], x);
                    }
                    if (TS == 32) __builtin_amdgcn_sched_barrier(0);    // fragments of two steps at a time: more do not fit the registers
                }
#pragma unroll
                for (int k = 0; k < AT_ONCE; ++k)
#pragma unroll
                    for (int r = 0; r < AR; ++r) s[k][r] *= sw[k][r];
                if (cuts) {
#pragma unroll
                    for (int k = 0; k < AT_ONCE; ++k) {
                        const int m = seg_of[TS * it[k] + ln];
#pragma unroll
                        for (int r = 0; r < AR; ++r) s[k][r] = seg_of[TS * jt[k] + 8 * (r >> 2) + 4 * g + (r & 3)] == m ? s[k][r] : 0.f;
                    }
                }
                if (!G::OVER) store_scores(t0);
            }
#pragma unroll
            for (int it = 0; it < IT; ++it)
#pragma unroll
                for (int r = 0; r < AR; ++r) O[it][r] = 0.f;
            frag fa[2][IT], fs[2][M::S_PARTS];
            float fq[IT];
#pragma unroll
            for (int q = -1; q < NPA; ++q) {                                          // the next fragments are made while these are multiplied
#pragma unroll
                for (int it = 0; it < IT; ++it) {
                    if (q + 1 < NPA) fa[(q + 1) & 1][it] = M::row(la + (TS * it + ln) * G::SA, q + 1, g);
                    else fq[it] = scale_s * pw[TS * it + ln + off];
                }
                if (q >= 0) {
#pragma unroll
                    for (int part = M::S_PARTS - 1; part >= 0; --part)
#pragma unroll
                        for (int x = 0; x < M::STEPS; ++x)
#pragma unroll
                            for (int it = 0; it < IT; ++it) O[it] = M::mfma(fs[q & 1][part], fa[q & 1][it], O[it], x);
                }
                if (q + 1 < NPA) M::of_state(S, q + 1, fs[(q + 1) & 1]);
                if (TS == 32) mix_interleave<IT * M::S_PARTS, 8>(q >= 0 && q + 1 < NPA);
            }
#pragma unroll
            for (int it = 0; it < IT; ++it)
#pragma unroll
                for (int r = 0; r < AR; ++r) O[it][r] *= fq[it];
            if (cuts)                                                // a choice, no factor of 0: the state that a reset ends may be anything
#pragma unroll
                for (int it = 0; it < IT; ++it) {
                    const bool after = seg_of[TS * it + ln] != 0;
#pragma unroll
                    for (int r = 0; r < AR; ++r) O[it][r] = after ? 0.f : O[it][r];
                }
            if (G::OVER) {
                lds_barrier();                                       // A has been read by all
                store_scores(0);
            }
            lds_barrier();
        }
        const bool last = left <= CH;
        const float ch = pw[last ? CH + 1 : CH], cl = pw_low[last ? 1 : 0];
        // where half of the state or more is gone a chunk later, the rounding of lam^64 does not add up over the chunks
        const bool two = __builtin_amdgcn_readfirstlane(ch > 0.5f);
        frag cf[NPC];
#pragma unroll
        for (int q = 0; q < NPC; ++q) cf[q] = M::column(lc, G::SC, q, g, TS * w + ln);
#pragma unroll
        for (int q = 0; q < (NPC > TILES ? NPC : TILES); ++q) {
            if (q < NPC && !states_only) {
                frag fp[M::P_PARTS][IT];
#pragma unroll
                for (int part = 0; part < M::P_PARTS; ++part)
#pragma unroll
                    for (int it = 0; it < IT; ++it)
                        if (q * M::KB < TS * (it + 1)) fp[part][it] = M::row_natural(lp + part * PLANE + (TS * it + ln) * G::SP, q, g);
#pragma unroll
                for (int part = M::P_PARTS - 1; part >= 0; --part)
#pragma unroll
                    for (int x = 0; x < M::STEPS; ++x)
#pragma unroll
                        for (int it = 0; it < IT; ++it)
                            if (q * M::KB < TS * (it + 1)) O[it] = M::mfma(cf[q], fp[part][it], O[it], x);
            }
            if (q < TILES) {
                if (cuts) {
#pragma unroll
                    for (int r = 0; r < AR; ++r) S[q][r] = 0.f;
                } else if (two) {
#pragma unroll
                    for (int r = 0; r < AR; ++r) S[q][r] = __builtin_fmaf(S[q][r], ch, S[q][r] * cl);
                } else {
#pragma unroll
                    for (int r = 0; r < AR; ++r) S[q][r] *= ch;
                }
            }
        }
        frag cw[2][M::W_PARTS];
#pragma unroll
        for (int q = -1; q < NPC; ++q) {
            frag fb[TILES];
            if (q >= 0)
#pragma unroll
                for (int t = 0; t < TILES; ++t) fb[t] = M::column(lb, G::SB, q, g, TS * t + ln);
            float wv[M::SLOTS];
            if (q + 1 < NPC) {
#pragma unroll
                for (int r = 0; r < M::SLOTS; ++r) wv[r] = wb[own_w][M::KB * (q + 1) + M::SLOTS * g + r];
            }
            if (q >= 0) {
#pragma unroll
                for (int part = M::W_PARTS - 1; part >= 0; --part) {
#pragma unroll
                    for (int x = 0; x < M::STEPS; ++x)
#pragma unroll
                        for (int t = 0; t < TILES; ++t) S[t] = M::mfma(fb[t], cw[q & 1][part], S[t], x);
                }
            }
            if (q + 1 < NPC) M::weigh(cf[q + 1], wv, cw[(q + 1) & 1]);
            if (TS == 32) mix_interleave<TILES * M::W_PARTS, 5>(q >= 0 && q + 1 < NPC);
        }
        if (!states_only) {
            // rows of O in the order of memory, as the stage's
            const int low = reverse ? left - CH : c * CH, e = TS * w + 4 * g;
            E* at = po + (int64_t)low * so + (int64_t)(reverse ? TS - 1 - ln : ln) * so + e;
#pragma unroll
            for (int it = 0; it < IT; ++it) {
                E* o = at + (int64_t)(TS * (reverse ? IT - 1 - it : it)) * so;
                if (TS * it + ln < left) {
#pragma unroll
                    for (int x = 0; x < QUADS; ++x) {
                        if (FULL || e + 8 * x + 4 <= dc) M::store_out(o + 8 * x, f32x4_t{O[it][4 * x], O[it][4 * x + 1], O[it][4 * x + 2], O[it][4 * x + 3]});
                        else
#pragma unroll
                            for (int r = 0; r < 4; ++r) if (e + 8 * x + r < dc) io_store(o + 8 * x + r, O[it][4 * x + r]);
                    }
                }
            }
        }
        lds_barrier();
    }
    const int e = TS * w + ln0;
    if (states_only) {
        const int64_t at = ((int64_t)bh * p.n_seg + seg);
        float* s = J.s_out + at * p.kv + c0;
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int r = 0; r < AR; ++r) {
                const int d = TS * t + 8 * (r >> 2) + 4 * g0 + (r & 3);
                if (d < da && e < dc) s[d * J.dc + e] = S[t][r];
            }
        if (tid == 0 && c0 == 0) {
            const int steps = max(0, min(n, (c_first + seg_chunks) * CH) - c_first * CH);
            const double f = exp((double)gl * steps);
            J.carry[2 * at] = cut_any ? -1.f : (float)f;
            J.carry[2 * at + 1] = cut_any ? 0.f : (float)(f - (double)(float)f);
        }
    } else if (J.s_out && p.n_seg == 1) {
        const bool none = J.off == 0 && n > 0 && p.reset && p.reset[b] != 0.f;      // the gradient stops at a reset before the first step
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int r = 0; r < AR; ++r) {
                const int d = TS * t + 8 * (r >> 2) + 4 * g0 + (r & 3);
                if (d < da && e < dc) J.s_out[(int64_t)bh * p.kv + d * J.sd + (c0 + e) * J.se] = none ? 0.f : S[t][r];
            }
    }
}

template <typename E, int TS, int DA, int NW, bool FULL>
static int launch_mix_as(mix_t m, int dc, hipStream_t s) {
    typedef mix_geom<E, TS, DA, NW> G;
    static_assert(G::BYTES + 1500 <= 160 * 1024, "LDS");
    m.n_slices = (dc + G::DC - 1) / G::DC;
    const int64_t units = ((int64_t)m.B * m.H * m.n_seg + 7) / 8 * 8, grid = units * m.n_jobs * m.n_slices;
    XRL_CHECK_ARG(grid * G::NT < 1ll << 32);                         // threads of a launch
    hipLaunchKernelGGL((linattn_mix_kernel<E, TS, DA, NW, FULL>), dim3((unsigned)grid), dim3(64 * NW), G::BYTES, s, m);
    XRL_CHECK_LAUNCH();
    return XRL_OK;
}

template <typename E, int TS, int DA, int NW>
static int launch_mix_size(const mix_t& m, int dc, hipStream_t s) {
    bool full = true;
    for (int i = 0; i < m.n_jobs; ++i) {
        const mix_job_t& j = m.job[i];
        full = full && j.da == DA && j.dc == dc && dc % (TS * NW) == 0;
        const int64_t most = (1ll << 31) / (CH * (int)sizeof(E));
        full = full && j.sa[0] < most && j.sb[0] < most && j.sc[0] < most;
    }
    return full ? launch_mix_as<E, TS, DA, NW, true>(m, dc, s) : launch_mix_as<E, TS, DA, NW, false>(m, dc, s);
}

// what a compute unit holds of an instance's workgroups
template <typename E, int TS, int DA, int NW>
static int mix_resident() {
    typedef mix_geom<E, TS, DA, NW> G;
    const int by_lds = G::HELD, by_registers = (G::OVER ? 12 : 8) / NW > 0 ? (G::OVER ? 12 : 8) / NW : 1;
    return by_lds < by_registers ? by_lds : by_registers;
}

template <typename E, int TS, int DA, int NW>
static int init_mix_as() {
    const int bytes = mix_geom<E, TS, DA, NW>::BYTES;
    XRL_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(linattn_mix_kernel<E, TS, DA, NW, true>), hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
    XRL_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(linattn_mix_kernel<E, TS, DA, NW, false>), hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
    return XRL_OK;
}

int launch_mix_f32(const mix_t& m, int da, int dc, hipStream_t s);
int launch_mix_bf16(const mix_t& m, int da, int dc, hipStream_t s);
int init_mix_f32();
int init_mix_bf16();
int mix_resident_f32(int da, int dc);
int mix_resident_bf16(int da, int dc);

}  // namespace xrl
