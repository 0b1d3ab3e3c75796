// Fused rollout step: ONE launch per vector step of the on-policy agent loop (ppo_agent.py:113-177) for a
// device-resident CartPole.  See include/xrl_hip.h (xrl_rollout_step_t) for the dataflow contract.
//
// Why: at the reference's sizes (256..1024 envs, 34k-parameter net) a vector step is ~17 MFLOP and ~20 KB of
// traffic -- far below one launch's worth of roofline work -- so the step is bound by *dependent latencies*: kernel
// boundaries (1.6 us each) and global-memory round trips (~1 us each right after a boundary; measured with the
// shader-clock stamps behind p.dbg).  The design therefore minimises round trips, not bytes or flops:
//   * one launch; a workgroup keeps a 32-row tile of every activation level in LDS for the whole MLP;
//   * every global load the kernel will ever need is ISSUED in the first few hundred cycles: biases and the small
//     layers' weights are copied into an LDS parameter cache, the first big layer's B-fragments go straight into
//     registers (16 x 16 B per lane), raw observations / flags for the statistics are loaded at the same time, so all of
//     them share one round trip that ends at the first barrier;
//   * statistics that couple all envs are recomputed per workgroup from the (tiny) previous-step arrays instead of
//     being synchronised across workgroups.
//
// MFMA mapping (64-wide wavefronts): v_mfma_f32_32x32x2_f32, the tile's 32 rows are M, each of the 8 waves owns 32-column
// output tiles.  A-fragments are ds_read_b128 from the LDS activations (row stride roundup8(width)+4 floats:
// conflict-free), B-fragments are 4 consecutive k of one weight row per lane (ds_read_b128 from the parameter cache or a
// 16-byte global load); as in gemm.hip lane-half h consumes k = 8q+4h+s so both operands share one k permutation.
// Layers with fewer than 8 column tiles split K over waves and reduce the partial tiles through LDS in wave order.
#include "common.h"
#include "rng.h"
#include "cartpole.h"
#include "mlp_tile.h"

namespace xrl {

// Layer roles (host order = execution order): layers[0] is the first layer (K = D = 4, evaluated on the VALU while the
// observation is normalised -- bitwise the same k-ordered fma chain the MFMA would produce), the last n_head layers all
// write the head level and are merged into ONE block-structured layer in the LDS cache, everything between runs on MFMA.
__global__ void __launch_bounds__(FUSED_THREADS) rollout_step_cartpole_kernel(xrl_rollout_step_t p) {
#pragma clang fp contract(off)
    extern __shared__ __attribute__((aligned(16))) float lds[];
    __shared__ double part[2 * NW * 4];
    __shared__ float s_mean[4], s_std[4];
    __shared__ float s_ret[2];

    constexpr int D = 4;
    const int tid = threadIdx.x, n = p.n, A = p.A;
    long long* dbg = p.dbg;
    int dbi = 0;
    const bool dbg_me = dbg && tid == 0 && (int)blockIdx.x == (int)dbg[63];   // dbg[63] selects the stamped workgroup
#define STAMP() do { if (dbg_me) dbg[dbi++] = clock64(); } while (0)
    STAMP();
    // workgroup role: with role_split the actor and critic branches of an act tile run in different workgroups
    //   role 0: act tile, actor branch (+ sampling, physics, bookkeeping)      role 1: act tile, critic branch -> val_slot
    //   role 2: bootstrap tile (critic branch only when role_split) -> bootv[t-1]
    const int n_act_tiles = (n + FT - 1) / FT;
    const int group = blockIdx.x / n_act_tiles, tile = blockIdx.x - group * n_act_tiles;
    const int role = p.boot_only ? 2 : (p.role_split ? group : (group == 0 ? 0 : 2));
    const bool boot = role == 2;
    const bool do_actor = !p.role_split ? !boot : role == 0;          // computes the actor columns / logits
    const bool do_critic = !p.role_split || role != 0;                // computes the critic columns / value
    const int e0 = tile * FT;
    const int lane = tid & 63, wave = tid >> 6, li_ = lane & 31, lh_ = lane >> 5;
    const int nL = p.n_layers, nH = p.n_head_layers, nLv = p.n_levels;
    const int first_mid = 1, end_mid = nL - nH;                      // MFMA layers [first_mid, end_mid)

    // ---- LDS carve (uniform arithmetic): activation levels 1.., split-K scratch, parameter cache
    int lvl_off[XRL_FUSED_MAX_LEVELS], lvl_ld[XRL_FUSED_MAX_LEVELS];  // small, fully unrolled uses only
    int off = 0;
#pragma unroll
    for (int l = 0; l < XRL_FUSED_MAX_LEVELS; ++l) {
        lvl_ld[l] = l < nLv ? level_ld(p.level_width[l]) : 0;
        lvl_off[l] = off;
        if (l >= 1 && l < nLv) off += FT * lvl_ld[l];
    }
    const int acts_end = off;
    float* red = lds + off;             off += NW * 32 * 33;
    const xrl_fused_layer_t& L0 = p.layers[0];
    off = (off + 3) / 4 * 4;
    const int c_w0 = off;               off += L0.N * 4;              // first layer weights [N0][4]
    const int c_b0 = off;               off += (L0.N + 3) / 4 * 4;
    int c_bm[XRL_FUSED_MAX_LAYERS], c_wm[XRL_FUSED_MAX_LAYERS];
#pragma unroll
    for (int l = 0; l < XRL_FUSED_MAX_LAYERS; ++l) {
        c_bm[l] = off; c_wm[l] = -1;
        if (l >= first_mid && l < end_mid) {
            off += (p.layers[l].N + 3) / 4 * 4;
            if (layer_small(p.layers[l].N, p.layers[l].K)) { c_wm[l] = off; off += p.layers[l].N * level_ld(p.layers[l].K); }
        }
    }
    const int KH = p.level_width[nLv - 2], NH = p.level_width[nLv - 1], ldH = level_ld(KH);
    const int c_wh = off;               off += NH * ldH;              // merged head weights [NH][ldH]
    const int c_bh = off;               off += (NH + 3) / 4 * 4;

    // ---- issue EVERY global load now.  (1) B-fragments of the first big MFMA layer straight into registers
    float4 pf[PD];
    int pf_layer = -1;
#pragma unroll
    for (int l = 1; l < XRL_FUSED_MAX_LAYERS; ++l) {
        if (pf_layer < 0 && l >= first_mid && l < end_mid && c_wm[l] < 0) {
            const xrl_fused_layer_t& L = p.layers[l];
            const float* Wg = p.params + L.w_off;
            if ((L.N + 31) / 32 >= NW && (L.K & 7) == 0 && ((reinterpret_cast<uintptr_t>(Wg) & 15) == 0)) {
                pf_layer = l;
                const int kq = L.K / 8;
                if (p.frag_image) {
                    // fragment-ordered copy (xrl_pack_rollout_cache): tile, chunk q, lane l -> one contiguous 1 KB per load
                    const int my_tile = (p.role_split && !do_actor ? p.split_col / 32 : 0) + wave;
                    const float4* fr = reinterpret_cast<const float4*>(p.frag_image) +
                                       (size_t)min(my_tile, (L.N + 31) / 32 - 1) * kq * 64 + lane;
#pragma unroll
                    for (int q = 0; q < PD; ++q) pf[q] = q < kq ? fr[q * 64] : make_float4(0.f, 0.f, 0.f, 0.f);
                } else {
                    const int my_tile = (p.role_split && !do_actor ? p.split_col / 32 : 0) + wave;
                    const float* wrow = Wg + (size_t)min(my_tile * 32 + li_, L.N - 1) * L.K + 4 * lh_;
#pragma unroll
                    for (int q = 0; q < PD; ++q) pf[q] = q < kq ? *reinterpret_cast<const float4*>(wrow + q * 8) : make_float4(0.f, 0.f, 0.f, 0.f);
                }
            }
        }
    }
    // (2) this thread's row of the tile (16 threads share a row) and, for act tiles, its share of ALL raw observations
    const int r = tid >> 4, sub = tid & 15, e_row = e0 + r;
    float4 xrow = make_float4(0.f, 0.f, 0.f, 0.f);
    if (e_row < n) xrow = *reinterpret_cast<const float4*>((boot ? p.xnext_in : p.obs_raw_in) + (size_t)e_row * D);
    // (2b) the tail (sampling + physics) runs on lanes 0..31: fetch their env state now instead of after the MLP
    double cps[4] = {0.0, 0.0, 0.0, 0.0};
    int cp_steps0 = 0, cp_ep0 = 0;
    float cp_score0 = 0.f, rtrack0 = 0.f;
    if (!boot && tid < FT && e0 + tid < n) {
        const int et = e0 + tid;
        cps[0] = p.cp_state[(size_t)et * 4 + 0]; cps[1] = p.cp_state[(size_t)et * 4 + 1];
        cps[2] = p.cp_state[(size_t)et * 4 + 2]; cps[3] = p.cp_state[(size_t)et * 4 + 3];
        cp_steps0 = p.cp_steps[et]; cp_ep0 = p.cp_episodes[et]; cp_score0 = p.cp_score[et]; rtrack0 = p.ret_track[et];
    }
    double s1 = 0.0, s2 = 0.0;                                      // sums for dimension d = tid & 3
    unsigned long long ended_mask[16];
    float rfin[16];
    float ret_m0 = 0.f, ret_v0 = 1.f, st_mean = 0.f, st_var = 1.f;
    double ret_c0 = 0.0, st_cnt = 0.0;
    if (!boot) {
        if (p.use_obsnorm) {
            float sv[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) { const int i = tid + j * FUSED_THREADS; sv[j] = i < n * D ? p.obs_raw_in[i] : 0.f; }
#pragma unroll
            for (int j = 0; j < 8; ++j) { const double v = (double)sv[j]; s1 += v; s2 += v * v; }
        }
        if (wave == 0) {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const int e = j * 64 + lane;
                const bool in = e < n;
                rfin[j] = in ? p.ret_final_in[e] : 0.f;               // loaded up front: no memory access inside the merge loop
                ended_mask[j] = __ballot(in && p.ended_in[e] != 0);
            }
            ret_m0 = p.ret_stats_in[0]; ret_v0 = p.ret_stats_in[1]; ret_c0 = *p.ret_count_in;
        }
        if (tid < D && p.use_obsnorm) { st_mean = p.obs_stats_in[tid]; st_var = p.obs_stats_in[D + tid]; st_cnt = *p.obs_count_in; }
    }
    // (3) the LDS parameter cache is a flat copy of the image xrl_pack_rollout_cache built once per rollout (same layout:
    //     first-layer W | b | middle biases (+ small middle weights, zero padded) | merged head W | head b): every
    //     thread issues its <= 4 independent 16-byte loads back to back, so the whole cache costs ONE round trip.
    const int pc_base = c_w0, pc_floats = off - c_w0;
    float4 img[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int i4 = (tid + j * FUSED_THREADS) * 4;
        img[j] = i4 < pc_floats ? *reinterpret_cast<const float4*>(p.cache_image + i4) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    for (int i4 = (tid + 4 * FUSED_THREADS) * 4; i4 < pc_floats; i4 += FUSED_THREADS * 4)      // larger nets: plain tail
        *reinterpret_cast<float4*>(&lds[pc_base + i4]) = *reinterpret_cast<const float4*>(p.cache_image + i4);
    // (4) zero the activation tiles (padding columns must read as zero) while the loads are in flight
    for (int i = tid; i < acts_end; i += FUSED_THREADS) lds[i] = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int i4 = (tid + j * FUSED_THREADS) * 4;
        if (i4 < pc_floats) *reinterpret_cast<float4*>(&lds[pc_base + i4]) = img[j];
    }

    if (!boot) {
        // ---- deferred ret_rms.update() of the episodes that ended at the previous step, in env order (ppo_agent.py:146-149)
        if (wave == 0) {
            float mean = ret_m0, var = ret_v0;
            double count = ret_c0;
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                unsigned long long mm = ended_mask[j];
                while (mm) {                                            // wave-uniform loop over finished envs
                    const int bpos = __ffsll((long long)mm) - 1; mm &= mm - 1;
                    const float bm = __shfl(rfin[j], bpos, 64);
                    const double tot = count + 1.0; const float delta = bm - mean;
                    const float new_mean = mean + delta * 1.0f / (float)tot;
                    const float M2 = var * (float)count + 0.f + (delta * delta) * (float)count * 1.0f / (float)tot;
                    mean = new_mean; var = M2 / (float)tot; count = tot;
                }
            }
            if (lane == 0) {
                s_ret[0] = mean; s_ret[1] = var;
                if (blockIdx.x == 0) { p.ret_stats_out[0] = mean; p.ret_stats_out[1] = var; *p.ret_count_out = count; }
            }
        }
        // ---- obs_rms.update(obs) over ALL envs, recomputed per workgroup: one pass, sum / sum of squares in float64
        if (p.use_obsnorm) {
            for (int o = 32; o >= D; o >>= 1) { s1 += __shfl_xor(s1, o, 64); s2 += __shfl_xor(s2, o, 64); }
            if (lane < D) { part[wave * 4 + lane] = s1; part[NW * 4 + wave * 4 + lane] = s2; }
        }
    }
    STAMP();
    __syncthreads();
    STAMP();
    if (!boot) {
        if (tid < D) {
            if (p.use_obsnorm) {
                double a = 0.0, b = 0.0;
                for (int w = 0; w < NW; ++w) { a += part[w * 4 + tid]; b += part[NW * 4 + w * 4 + tid]; }
                const double m = a / n;
                const float bm = (float)m;                              // np.mean -> float32
                const float bstd = (float)sqrt(fmax(b / n - m * m, 0.0));          // np.std -> float32
                const float bv = bstd * bstd;                           // batch_var = np.square(batch_std)
                const double cnt = st_cnt, tot = cnt + (double)n;
                const float mean = st_mean, var = st_var;
                const float delta = bm - mean;                          // update_from_moments (statistic_tools.py:173-185)
                const float new_mean = mean + delta * (float)n / (float)tot;
                const float m_a = var * (float)cnt, m_b = bv * (float)n;
                const float M2 = m_a + m_b + (delta * delta) * (float)cnt * (float)n / (float)tot;
                const float new_var = M2 / (float)tot;
                s_mean[tid] = new_mean; s_std[tid] = sqrtf(new_var);
                if (blockIdx.x == 0) {
                    p.obs_stats_out[tid] = new_mean; p.obs_stats_out[D + tid] = new_var;
                    if (tid == 0) *p.obs_count_out = tot;
                }
            } else { s_mean[tid] = 0.f; s_std[tid] = 1.f; }
        }
        __syncthreads();
        if (p.use_obsnorm) {
            xrow.x = fminf(fmaxf((xrow.x - s_mean[0]) / (s_std[0] + 1e-8f), -p.obs_range), p.obs_range);
            xrow.y = fminf(fmaxf((xrow.y - s_mean[1]) / (s_std[1] + 1e-8f), -p.obs_range), p.obs_range);
            xrow.z = fminf(fmaxf((xrow.z - s_mean[2]) / (s_std[2] + 1e-8f), -p.obs_range), p.obs_range);
            xrow.w = fminf(fmaxf((xrow.w - s_mean[3]) / (s_std[3] + 1e-8f), -p.obs_range), p.obs_range);
        }
        if (sub == 0 && e_row < n && role == 0) *reinterpret_cast<float4*>(p.obs_slot + (size_t)e_row * D) = xrow;   // memory.observations[t]
    }
    STAMP();
    // ---- first layer on the VALU: out = act(fma(x3,w3, fma(x2,w2, fma(x1,w1, x0*w0))) + b), 16 threads per row
    {
        float* o1 = lds + lvl_off[L0.out_level] + L0.out_off + r * lvl_ld[L0.out_level];
        XRL_ACT_DISPATCH(L0.act,
            for (int c = sub; c < L0.N; c += 16) {
                const float4 w = *reinterpret_cast<const float4*>(&lds[c_w0 + c * 4]);
                float acc = __fmaf_rn(xrow.x, w.x, 0.f);
                acc = __fmaf_rn(xrow.y, w.y, acc);
                acc = __fmaf_rn(xrow.z, w.z, acc);
                acc = __fmaf_rn(xrow.w, w.w, acc);
                o1[c] = act_apply_c<ACT>(acc + lds[c_b0 + c]);
            })
    }
    __syncthreads();
    STAMP();
    // ---- middle layers on the matrix cores
#ifdef XRL_TILE_PROBE
    if (dbg_me) { g_probe = dbg + 16; g_probe_i = 0; }
#endif
#pragma unroll
    for (int l = 1; l < XRL_FUSED_MAX_LAYERS; ++l) {
        if (l >= first_mid && l < end_mid) {
            const xrl_fused_layer_t& L = p.layers[l];
            const int tb = p.role_split ? (do_actor ? 0 : p.split_col / 32) : 0;
            const int te = p.role_split ? (do_actor ? p.split_col / 32 : (L.N + 31) / 32) : -1;
            fused_layer(p.params + L.w_off, c_wm[l] >= 0 ? lds + c_wm[l] : nullptr, level_ld(L.K), lds + c_bm[l], L.K, L.N, L.act,
                        lds + lvl_off[L.in_level] + L.in_off, lvl_ld[L.in_level],
                        lds + lvl_off[L.out_level] + L.out_off, lvl_ld[L.out_level], red, pf, l == pf_layer, nullptr, 0, tb, te);
            STAMP();
        }
    }
    // ---- all heads as one block-structured layer from the LDS cache (per-head activation is the identity for the
    //      categorical actor and the critic)
    if (NH <= 8)
        narrow_layer_valu(lds + c_wh, ldH, lds + c_bh, KH, NH, XRL_ACT_NONE, lds + lvl_off[nLv - 2], lvl_ld[nLv - 2],
                          lds + lvl_off[nLv - 1], lvl_ld[nLv - 1]);
    else
        fused_layer(nullptr, lds + c_wh, ldH, lds + c_bh, KH, NH, XRL_ACT_NONE, lds + lvl_off[nLv - 2], lvl_ld[nLv - 2],
                    lds + lvl_off[nLv - 1], lvl_ld[nLv - 1], red, pf, false);
    STAMP();
    const float* heads = lds + lvl_off[nLv - 1];
    const int ldh = lvl_ld[nLv - 1];

    if (tid >= FT) return;
    const int e = e0 + tid;
    if (e >= n) return;
    const float* h = heads + tid * ldh;
    if (boot) {                                                         // V(next_obs_{t-1}) -> bootv[t-1]
        if (p.bootv_prev) p.bootv_prev[e] = h[A];
        if (dbg_me) { dbg[dbi++] = clock64(); dbg[15] = dbi; }
        return;
    }
    if (role == 1) { p.val_slot[e] = h[A]; return; }                   // critic workgroup of an act tile
    // ---- get_actions (core/on_policy.py:128-169): sample, log-prob, value; store (ppo_agent.py:128)
    const uint32_t step = p.step + (p.step_dev ? *p.step_dev : 0u);
    int a = 0;
    float logp;
    {
        uint32_t rr[4];
        philox4x32(p.seed, (uint32_t)e, step, STREAM_ACTION, rr);
        const float u = u01(rr[0]);
        float mx = h[0];
        for (int j = 1; j < A; ++j) mx = fmaxf(mx, h[j]);
        float se = 0.f;
        for (int j = 0; j < A; ++j) se += expf(h[j] - mx);
        const float lse = mx + logf(se);
        a = A - 1;
        float c = 0.f;
        for (int j = 0; j < A; ++j) { c += expf(h[j] - lse); if (c > u) { a = j; break; } }
        logp = h[a] - lse;
    }
    STAMP();
    p.act_slot[e] = (float)a;
    if (!p.role_split) p.val_slot[e] = h[A];
    p.logp_slot[e] = logp;
    // ---- envs.step(acts): physics + DummyVecEnv auto-reset
    double* s = p.cp_state + (size_t)e * 4;
    double x, xd, th, thd;
    bool term;
    cartpole_advance(cps, a, x, xd, th, thd, term);
    const int steps = cp_steps0 + 1;
    const bool trunc = steps >= p.max_steps;
    const float nobs[4] = {(float)x, (float)xd, (float)th, (float)thd};
    const float score = cp_score0 + 1.0f;
    float robs[4] = {nobs[0], nobs[1], nobs[2], nobs[3]};
    if (term || trunc) {
        const int ep = cp_ep0 + 1;
        p.cp_episodes[e] = ep;
        cartpole_reset(s, p.env_seed, e, (uint32_t)ep);
        p.cp_steps[e] = 0; p.cp_score[e] = 0.f;
        robs[0] = (float)s[0]; robs[1] = (float)s[1]; robs[2] = (float)s[2]; robs[3] = (float)s[3];
        atomicAdd(&p.cp_stats[0], 1.0); atomicAdd(&p.cp_stats[1], (double)score); atomicAdd(&p.cp_stats[2], (double)steps);
    } else {
        s[0] = x; s[1] = xd; s[2] = th; s[3] = thd;
        p.cp_steps[e] = steps; p.cp_score[e] = score;
    }
    STAMP();
    // ---- bookkeeping (ppo_agent.py:128,144-157)
    const float reward = 1.0f;
    float rstd = sqrtf(s_ret[1]);
    rstd = fminf(fmaxf(rstd, 0.1f), 100.f);
    float rn = reward;
    if (p.use_rewnorm) rn = fminf(fmaxf(reward / rstd, -p.rew_range), p.rew_range);
    p.rew_slot[e] = rn;
    p.term_slot[e] = term ? 1.f : 0.f;
    p.seg_slot[e] = (term || trunc || p.last_step) ? (uint8_t)(1 | (term ? 6 : 0)) : (uint8_t)0;
    const float tr = p.gamma * rtrack0 + reward;
    if (term || trunc) { p.ret_final_out[e] = tr; p.ended_out[e] = 1; p.ret_track[e] = 0.f; }
    else { p.ended_out[e] = 0; p.ret_track[e] = tr; }
    float4 ro = make_float4(robs[0], robs[1], robs[2], robs[3]), xn;
    *reinterpret_cast<float4*>(p.obs_raw_out + (size_t)e * 4) = ro;    // buf_obs for the next step (reset_obs on episode end)
    float nv[4];
#pragma unroll
    for (int d = 0; d < 4; ++d) {
        float v = nobs[d];
        if (p.use_obsnorm) { v = (v - s_mean[d]) / (s_std[d] + 1e-8f); v = fminf(fmaxf(v, -p.obs_range), p.obs_range); }
        nv[d] = v;
    }
    xn = make_float4(nv[0], nv[1], nv[2], nv[3]);
    *reinterpret_cast<float4*>(p.xnext_out + (size_t)e * 4) = xn;      // get_terminated_values input (on_policy.py:109)
    if (dbg_me) { dbg[dbi++] = clock64(); dbg[15] = dbi; }
}

// Builds the parameter-cache image (same carve as the kernel above, offsets relative to the image start).
__global__ void __launch_bounds__(256) pack_rollout_cache_kernel(xrl_rollout_step_t p, float* __restrict__ image,
                                                                 float* __restrict__ frag) {
    const int nL = p.n_layers, nH = p.n_head_layers, nLv = p.n_levels, end_mid = nL - nH;
    const int tid = blockIdx.x * blockDim.x + threadIdx.x, nt = gridDim.x * blockDim.x;
    if (frag) {
        // first middle layer that qualifies for register prefetch (same test as the step kernel)
        for (int l = 1; l < end_mid; ++l) {
            const xrl_fused_layer_t& L = p.layers[l];
            if (!layer_small(L.N, L.K) && (L.N + 31) / 32 >= NW && (L.K & 7) == 0) {
                const int kq = L.K / 8, total = ((L.N + 31) / 32) * kq * 64 * 4;
                for (int i = tid; i < total; i += nt) {
                    const int sidx = i & 3, ln = (i >> 2) & 63, q = (i >> 8) % kq, t = (i >> 8) / kq;
                    const int row = min(t * 32 + (ln & 31), L.N - 1), k = q * 8 + 4 * (ln >> 5) + sidx;
                    frag[i] = p.params[L.w_off + (size_t)row * L.K + k];
                }
                break;
            }
        }
    }
    const xrl_fused_layer_t& L0 = p.layers[0];
    int off = 0;
    const int c_w0 = off; off += L0.N * 4;
    const int c_b0 = off; off += (L0.N + 3) / 4 * 4;
    for (int i = tid; i < L0.N * 4; i += nt) image[c_w0 + i] = p.params[L0.w_off + i];
    for (int i = tid; i < (L0.N + 3) / 4 * 4; i += nt) image[c_b0 + i] = i < L0.N ? p.params[L0.b_off + i] : 0.f;
    for (int l = 1; l < end_mid; ++l) {
        const xrl_fused_layer_t& L = p.layers[l];
        const int nb = (L.N + 3) / 4 * 4;
        for (int i = tid; i < nb; i += nt) image[off + i] = i < L.N ? p.params[L.b_off + i] : 0.f;
        off += nb;
        if (layer_small(L.N, L.K)) {
            const int ldw = level_ld(L.K);
            for (int i = tid; i < L.N * ldw; i += nt) { const int r = i / ldw, k = i - r * ldw; image[off + i] = k < L.K ? p.params[L.w_off + (size_t)r * L.K + k] : 0.f; }
            off += L.N * ldw;
        }
    }
    const int KH = p.level_width[nLv - 2], NH = p.level_width[nLv - 1], ldH = level_ld(KH);
    const int c_wh = off; off += NH * ldH;
    const int c_bh = off;
    for (int i = tid; i < NH * ldH; i += nt) {                          // merged heads: W_h[out_off+j][in_off+k] = W_l[j][k]
        const int row = i / ldH, k = i - row * ldH;
        float v = 0.f;
        for (int l = end_mid; l < nL; ++l) {
            const xrl_fused_layer_t& L = p.layers[l];
            if (row >= L.out_off && row < L.out_off + L.N && k >= L.in_off && k < L.in_off + L.K)
                v = p.params[L.w_off + (size_t)(row - L.out_off) * L.K + (k - L.in_off)];
        }
        image[c_wh + i] = v;
    }
    for (int i = tid; i < (NH + 3) / 4 * 4; i += nt) {
        float v = 0.f;
        for (int l = end_mid; l < nL; ++l) {
            const xrl_fused_layer_t& L = p.layers[l];
            if (i >= L.out_off && i < L.out_off + L.N) v = p.params[L.b_off + i - L.out_off];
        }
        image[c_bh + i] = v;
    }
}

static size_t fused_cache_floats(const xrl_rollout_step_t& p) {
    size_t floats = (size_t)p.layers[0].N * 4 + (p.layers[0].N + 3) / 4 * 4;
    for (int l = 1; l < p.n_layers - p.n_head_layers; ++l) {
        floats += (p.layers[l].N + 3) / 4 * 4;
        if (layer_small(p.layers[l].N, p.layers[l].K)) floats += (size_t)p.layers[l].N * level_ld(p.layers[l].K);
    }
    const int NH = p.level_width[p.n_levels - 1], KH = p.level_width[p.n_levels - 2];
    floats += (size_t)NH * level_ld(KH) + (NH + 3) / 4 * 4;
    return floats;
}

static size_t fused_lds_bytes(const xrl_rollout_step_t& p) {
    size_t floats = 0;
    for (int l = 1; l < p.n_levels; ++l) floats += (size_t)FT * level_ld(p.level_width[l]);
    floats += NW * 32 * 33;                                           // split-K reduction scratch
    floats += (size_t)p.layers[0].N * 4 + (p.layers[0].N + 3) / 4 * 4;
    for (int l = 1; l < p.n_layers - p.n_head_layers; ++l) {
        floats += (p.layers[l].N + 3) / 4 * 4;
        if (layer_small(p.layers[l].N, p.layers[l].K)) floats += (size_t)p.layers[l].N * level_ld(p.layers[l].K);
    }
    const int NH = p.level_width[p.n_levels - 1], KH = p.level_width[p.n_levels - 2];
    floats += (size_t)NH * level_ld(KH) + (NH + 3) / 4 * 4;
    return floats * sizeof(float);
}

}  // namespace xrl

using namespace xrl;

namespace xrl { int init_ppo_fused(); int init_linattn(); }      // (csrc/ppo_fused.hip, csrc/linattn.hip; internal: not part of the C ABI)
extern "C" int xrl_pack_rollout_cache2(const xrl_rollout_step_t* pp, float* image, int64_t image_floats, float* frag,
                                       xrl_stream_t stream);

extern "C" int xrl_init(void) {
    if (int rc = init_ppo_fused()) return rc;
    if (int rc = init_linattn()) return rc;
    // kernels that carve more than 64 KB of dynamic LDS need the attribute; set it outside any graph capture
    XRL_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(rollout_step_cartpole_kernel),
                                      hipFuncAttributeMaxDynamicSharedMemorySize, 144 * 1024));
    return XRL_OK;
}

extern "C" int xrl_rollout_step_cartpole(const xrl_rollout_step_t* pp, xrl_stream_t stream) {
    XRL_CHECK_ARG(pp != nullptr);
    const xrl_rollout_step_t& p = *pp;
    XRL_CHECK_ARG(p.params && p.n > 0 && p.D == 4 && p.A >= 2 && !p.gaussian);
    XRL_CHECK_ARG(p.n_layers >= 1 && p.n_layers <= XRL_FUSED_MAX_LAYERS && p.n_levels >= 2 && p.n_levels <= XRL_FUSED_MAX_LEVELS);
    XRL_CHECK_ARG(p.level_width[0] == p.D && p.level_width[p.n_levels - 1] >= p.A + 1);
    XRL_CHECK_ARG(p.n_head_layers >= 1 && p.n_head_layers < p.n_layers && p.layers[0].K == 4 && p.layers[0].in_level == 0);
    XRL_CHECK_ARG(p.n <= 1024);
    XRL_CHECK_ARG(p.xnext_in != nullptr && p.cache_image != nullptr && (reinterpret_cast<uintptr_t>(p.cache_image) & 15) == 0);
    if (!p.boot_only) {
        XRL_CHECK_ARG(p.obs_raw_in && p.obs_raw_out && p.xnext_out && p.obs_stats_in && p.obs_stats_out && p.obs_count_in &&
                      p.obs_count_out && p.ret_stats_in && p.ret_stats_out && p.ret_count_in && p.ret_count_out &&
                      p.ended_in && p.ended_out && p.ret_final_in && p.ret_final_out && p.ret_track);
        XRL_CHECK_ARG(p.obs_slot && p.act_slot && p.val_slot && p.logp_slot && p.rew_slot && p.term_slot && p.seg_slot);
        XRL_CHECK_ARG(p.cp_state && p.cp_steps && p.cp_episodes && p.cp_score && p.cp_stats);
    } else {
        XRL_CHECK_ARG(p.bootv_prev != nullptr);
    }
    const size_t lds_bytes = fused_lds_bytes(p);
    XRL_CHECK_ARG(lds_bytes <= 144 * 1024);
    const int n_tiles = (p.n + FT - 1) / FT;
    if (p.role_split) XRL_CHECK_ARG(p.split_col > 0 && p.split_col % 32 == 0 && p.n_layers - p.n_head_layers == 2);
    const int act_groups = p.role_split ? 2 : 1;
    const int grid = p.boot_only ? n_tiles : (p.bootv_prev ? (act_groups + 1) * n_tiles : act_groups * n_tiles);
    hipLaunchKernelGGL(rollout_step_cartpole_kernel, dim3(grid), dim3(FUSED_THREADS), lds_bytes, as_stream(stream), p);
    XRL_CHECK_LAUNCH();
    return XRL_OK;
}

extern "C" int xrl_pack_rollout_cache(const xrl_rollout_step_t* pp, float* image, int64_t image_floats, xrl_stream_t stream) {
    return xrl_pack_rollout_cache2(pp, image, image_floats, nullptr, stream);
}

extern "C" int xrl_pack_rollout_cache2(const xrl_rollout_step_t* pp, float* image, int64_t image_floats, float* frag,
                                       xrl_stream_t stream) {
    XRL_CHECK_ARG(pp && image && pp->params);
    const xrl_rollout_step_t& p = *pp;
    XRL_CHECK_ARG(p.n_layers >= 2 && p.n_layers <= XRL_FUSED_MAX_LAYERS && p.n_head_layers >= 1 && p.n_head_layers < p.n_layers);
    XRL_CHECK_ARG((int64_t)fused_cache_floats(p) <= image_floats);
    hipLaunchKernelGGL(pack_rollout_cache_kernel, dim3(32), dim3(256), 0, as_stream(stream), p, image, frag);
    XRL_CHECK_LAUNCH();
    return XRL_OK;
}

extern "C" int64_t xrl_rollout_cache_floats(const xrl_rollout_step_t* pp) {
    return pp ? (int64_t)fused_cache_floats(*pp) : -1;
}
