// The selective state space scan, forward (state_space.cuh has the formulas and how lanes and waves share the work), and its single-token step.
//
// What bounds the scan: the vector ALU, busy 88 to 90 % of the time (8192 x 4096 x 16 191 us, 4 x 2048 x 2048 x 16 72, with the states for a backward pass some 90).  A state and token cost 11.3 issue slots in all: a
// multiplication and an exponential (two slots) for the decay, two for the walk from zero and two for the other; the rest are step sizes, gates, sums over lanes and what
// brings operands into place.  Against that stand 8 bytes of x, dt, z and y a channel and token of bf16.
#include "hdla_launch.h"
#include "state_space.cuh"
#include "state_space_ends.h"

namespace hdla {

template <typename T, int LPC, int TOK, int W, bool VEC>
__global__ __launch_bounds__(64 * W) void scan_tokens_kernel(ScanArgs p) {
    using Lane = ScanLane<LPC, TOK>;
    constexpr int CHN = Lane::CHN, V = Lane::V, TILE = W * TOK, PITCH = ss_pitch(TOK);
    static_assert(W >= 4, "a thread a state of the 64 lanes");
    // a wave's own: its arrays lie at fixed distances, so that a lane holds one address for all of them
    struct Mine { f32x4 B[TOK * LPC], C[TOK * LPC]; float d[CHN * PITCH], x[CHN * PITCH]; };
    struct Meet { f32x4 P[W][64], E[W][64]; };
    __shared__ __attribute__((aligned(16))) Mine mine[W];
    __shared__ Meet meet;
    __shared__ float bias[CHN], skip[CHN];                // (in registers they are what does not fit)

    int unit, block;
    if (!scan_work(blockIdx.x, p.blocks, unit, block)) return;
    const Unit U(p, unit);
    if (!U.ok) return;
    const int n = U.n;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane_id(), tid = threadIdx.x;
    const Lane L(p, block);
    Mine& my = mine[w];
    const int64_t bos = U.bos;
    const int len = U.to;
    const long long batch = p.cu ? 0 : n, row0 = p.cu ? bos : (long long)n * p.T;
    f32x4 A2 = zero4();
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (j < L.left) A2[j] = ld_decay(p.A, p.A_f32, (long long)L.d * p.S + 4 * L.q + j);
    if (tid < CHN) {
        const bool in = (block % p.per_group) * CHN + tid < p.DD / p.G;
        bias[tid] = p.bias && in ? ld_param(p.bias, p.bias_f32, L.d0 + tid) : 0.f;
        skip[tid] = p.D && in ? ld_param(p.D, p.D_f32, L.d0 + tid) : 0.f;
    }
    __syncthreads();
    // The state that enters the tile, one of the 256 states of the block a thread of the first four waves: number tid of meet.E's rows
    const int ec = (tid >> 2) / LPC, es = 4 * ((tid >> 2) % LPC) + (tid & 3);
    const bool chains = tid < 256, there = chains && (block % p.per_group) * CHN + ec < p.DD / p.G && es < p.S;
    const long long state = ((long long)n * p.DD + L.d0 + ec) * p.S + es;
    float enters = there && p.h0 ? p.h0[state] : 0.f;
    if (chains)
        for (int i = 0; i < U.index; ++i) {
            const float* const left = ends_of(p, unit - U.index + i, block) + tid;
            enters = __builtin_fmaf(left[256], enters, left[0]);
        }

    float* const ckpt = p.ckpt ? ckpt_of(p, n, bos, block) : nullptr;
    Raw<T, V, VEC> rx, rdt, rz;
    StatesOf<T, LPC, TOK, VEC> rB, rC;
    const long long first = bos + U.from + w * TOK;
    Cursor<T> cx(row_of<T>(p.x, batch, first) + L.d0, p.x.row * TILE), cdt(row_of<T>(p.dt, batch, first) + L.d0, p.dt.row * TILE),
        cz(row_of<T>(p.z, batch, first) + L.d0, p.z.row * TILE), cB(row_of<T>(p.B, batch, first) + L.group * p.B_group, p.B.row * TILE),
        cC(row_of<T>(p.C, batch, first) + L.group * p.C_group, p.C.row * TILE),
        cy(static_cast<const T*>(p.y) + (row0 + U.from + w * TOK) * p.DD + L.d0, (long long)p.DD * TILE);
    const uint32_t ox = L.offset(p.x.row, sizeof(T)), odt = L.offset(p.dt.row, sizeof(T)), oz = L.offset(p.z.row, sizeof(T)), oy = L.offset(p.DD, sizeof(T));
    auto request = [&](int t0) __attribute__((always_inline)) {
        const int tokens = min(max(len - t0, 0), TOK);
        const bool live = L.tok < tokens && L.carried > 0;
        rx.load(cx.rows(), live ? ox : NOWHERE, L.carried);
        rdt.load(cdt.rows(), live ? odt : NOWHERE, L.carried);
        if (p.z.p) rz.load(cz.rows(), live ? oz : NOWHERE, L.carried);
        else rz.clear();
        rB.load(cB, (uint32_t)p.B.row, tokens, p.S);
        rC.load(cC, (uint32_t)p.C.row, tokens, p.S);
        cx.next(); cdt.next(); cz.next(); cB.next(); cC.next();
    };
    request(U.from + w * TOK);
    for (int tile = U.from; tile < len; tile += TILE) {
        const int t0 = tile + w * TOK, tokens = min(max(len - t0, 0), TOK);
        float x[V], z[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            x[i] = rx[i];
            z[i] = rz[i];
            float e;
            const float v = rdt[i] + bias[L.ch + i], delta = L.tok < tokens ? (p.softplus ? softplus<T>(v, e) : v) : 0.f;
            if (L.tok < TOK) {
                my.d[(L.ch + i) * PITCH + L.tok] = delta;
                my.x[(L.ch + i) * PITCH + L.tok] = delta * x[i];
            }
        }
        rB.put(my.B);
        rC.put(my.C);
        request(t0 + TILE);
        wave_lds_fence();
        // from zero: the decays stay in registers
        f32x4 a[TOK], b[TOK], E = zero4();                // decays, and what each token adds
        float sum = 0.f;
        const float *const mine_d = &my.d[L.c * PITCH], *const mine_x = &my.x[L.c * PITCH];
        float dl = mine_d[0], dx = mine_x[0];
        b[0] = my.B[L.q];
#pragma unroll
        for (int k = 0; k < TOK; ++k) {
            // (the next token's operands are on their way while this one's are worked on)
            float dl1 = 0.f, dx1 = 0.f;
            if (k + 1 < TOK) { dl1 = mine_d[k + 1]; dx1 = mine_x[k + 1]; b[k + 1] = my.B[(k + 1) * LPC + L.q]; }
            sum += dl;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                a[k][j] = __builtin_amdgcn_exp2f(dl * A2[j]);
                b[k][j] *= dx;
                E[j] = __builtin_fmaf(a[k][j], E[j], b[k][j]);
            }
            dl = dl1;
            dx = dx1;
            apart();
        }
        f32x4 P;
#pragma unroll
        for (int j = 0; j < 4; ++j) P[j] = __builtin_amdgcn_exp2f(sum * A2[j]);
        meet.P[w][l] = P;
        meet.E[w][l] = E;
        __syncthreads();
        if (chains) {
            float* const e = reinterpret_cast<float*>(meet.E) + tid;
            const float* const f = reinterpret_cast<const float*>(meet.P) + tid;
#pragma unroll
            for (int k = 0; k < W; k += 4) {
                float ends[4], decays[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) { ends[i] = e[(k + i) * 256]; decays[i] = f[(k + i) * 256]; }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    e[(k + i) * 256] = enters;
                    enters = __builtin_fmaf(decays[i], enters, ends[i]);
                }
            }
        }
        __syncthreads();
        f32x4 h = meet.E[w][l];
        if (ckpt && (t0 & ((1 << p.every_log2) - 1)) == 0 && tokens > 0)
            *reinterpret_cast<f32x4*>(ckpt + (long long)(t0 >> p.every_log2) * p.blocks * 256 + l * 4) = h;
        float y[TOK];
        f32x4 cc = my.C[L.q];
#pragma unroll
        for (int k = 0; k < TOK; ++k) {
            const f32x4 c1 = k + 1 < TOK ? my.C[(k + 1) * LPC + L.q] : zero4();
            float s = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                h[j] = __builtin_fmaf(a[k][j], h[j], b[k][j]);
                s = __builtin_fmaf(h[j], cc[j], s);
            }
            y[k] = s;
            cc = c1;
            apart();
        }
        sum_channel<LPC>(y);
        if (L.q == 0) {
#pragma unroll
            for (int k = 0; k < TOK; k += 4) *reinterpret_cast<f32x4*>(&my.d[L.c * PITCH + k]) = f32x4{y[k], y[k + 1], y[k + 2], y[k + 3]};
        }
        wave_lds_fence();
        float o[V], g[V];
        if (p.z.p) sigmoid_each<T, V>(z, g);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            o[i] = __builtin_fmaf(skip[L.ch + i], x[i], my.d[(L.ch + i) * PITCH + min(L.tok, TOK - 1)]);
            if (p.z.p) o[i] *= z[i] * g[i];
        }
        if (L.tok < tokens && L.carried > 0)
            st_values<T, V, VEC>(at(const_cast<T*>(cy.p), oy), o, L.carried);
        cy.next();
        wave_lds_fence();                                 // the next tile's operands go where y is
    }
    if (there && p.ht && U.to == U.len) p.ht[state] = enters;
}

// One token of each sequence: lpc lanes a channel, four states each; a thread takes NB sequences one behind the other, whose states are on their way together and whose
// decays, skip and bias are the same.  Bound by HBM: 8 bytes a state.  us, one sequence a thread with loads of single elements -> this: 256 x 4096 x 16 42.2 -> 25.7
// (5.6 TB/s).
template <typename T, int NB, bool VEC>
__global__ __launch_bounds__(256) void scan_step_kernel(ScanArgs p, int lpc_log2) {
    const int lpc = 1 << lpc_log2;
    const long long at = (long long)blockIdx.x * 256 + threadIdx.x, channel = at >> lpc_log2;
    const int q = (int)(at & (lpc - 1));
    const bool in = channel < p.DD;                       // (lanes of a channel are neighbours: they are out together)
    const int d = in ? (int)channel : 0, g = d / (p.DD / p.G), left = in ? min(max(p.S - 4 * q, 0), 4) : 0, n0 = blockIdx.y * NB, many = min(NB, p.N - n0);
    f32x4 h[NB], A = zero4();
    Raw<T, 4, VEC> B[NB], C[NB];
    Raw<T, 1, true> x[NB], dt[NB], z[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        const int n = n0 + min(i, many - 1);
        h[i] = left ? ld_states(p.h0 + ((long long)n * p.DD + d) * p.S + 4 * q, left, VEC) : zero4();
        B[i].clear();
        C[i].clear();
        if (left) {
            B[i].load(static_cast<const T*>(p.B.p) + n * p.B.batch + g * p.B_group + 4 * q, left);
            C[i].load(static_cast<const T*>(p.C.p) + n * p.C.batch + g * p.C_group + 4 * q, left);
        }
        x[i].load(static_cast<const T*>(p.x.p) + n * p.x.batch + d, 1);
        dt[i].load(static_cast<const T*>(p.dt.p) + n * p.dt.batch + d, 1);
        if (p.z.p) z[i].load(static_cast<const T*>(p.z.p) + n * p.z.batch + d, 1);
        else z[i].clear();
    }
    const long long a0 = (long long)d * p.S + 4 * q;
    if (VEC && p.A_f32 && left) A = *reinterpret_cast<const f32x4*>(static_cast<const float*>(p.A) + a0);
    else
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < left) A[j] = ld_param(p.A, p.A_f32, a0 + j);
#pragma unroll
    for (int j = 0; j < 4; ++j) A[j] = decay_exponent(A[j]);
    const float bias = p.bias ? ld_param(p.bias, p.bias_f32, d) : 0.f, D = p.D ? ld_param(p.D, p.D_f32, d) : 0.f;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        float e;
        const float v = dt[i][0] + bias, delta = p.softplus ? softplus<T>(v, e) : v, add = delta * x[i][0];
        float y = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            h[i][j] = __builtin_fmaf(__builtin_amdgcn_exp2f(delta * A[j]), h[i][j], add * B[i][j]);
            y = __builtin_fmaf(h[i][j], C[i][j], y);
        }
        y = sum_lanes(y, lpc);
        if (i >= many) continue;
        const long long ch = (long long)(n0 + i) * p.DD + d;
        if (left) st_states(p.ht + ch * p.S + 4 * q, h[i], left, VEC);
        if (in && q == 0) {
            y = __builtin_fmaf(D, x[i][0], y);
            if (p.z.p) {
                float zz[1] = {z[i][0]}, s[1];
                sigmoid_each<T, 1>(zz, s);
                y *= zz[0] * s[0];
            }
            st_elem(static_cast<T*>(p.y) + ch, y);
        }
    }
}

template <typename T, int LPC, int W, bool VEC> static void launch_tokens(const ScanArgs& a, hipStream_t s) {
    hipLaunchKernelGGL((scan_tokens_kernel<T, LPC, SS_TOK, W, VEC>), dim3((unsigned)scan_workgroups(a.blocks, a.units)), dim3(64 * W), 0, s, a);
}
// Waves of a workgroup.  Where the registers of four waves a SIMD suffice: eight, two workgroups a compute unit, if there are as many; else sixteen.  Where they don't: twelve.
// Short sequences: four.  us, eight / twelve / sixteen (and 16 tokens a wave, eight waves): 8192 x 4096 channels, 256 workgroups, 245 / 214 / 195 (215); 4 x 2048 x 2048, 512 of them,
// 72 / 84 / 77 (94).  Four / eight: 8 x 64 x 2048 11 / 14, 256 x 32 x 2048 156 / 303, 64 x 128 x 2048 100 / 122, but 4 x 128 x 1024, 256 workgroups, 10.2 / 8.5.
template <typename T, int LPC, bool VEC> static void launch_lpc(const ScanArgs& a, hipStream_t s) {
    constexpr bool lean = LPC == 8 || (VEC && sizeof(T) == 2 && LPC >= 4);
    const int average = a.T / (a.cu ? a.N : 1);
    const bool many = scan_workgroups(a.blocks, a.units) >= 512;
    if (average <= 64 || (average <= 128 && many)) launch_tokens<T, LPC, 4, VEC>(a, s);
    else if constexpr (!lean) launch_tokens<T, LPC, 12, VEC>(a, s);
    else if (many) launch_tokens<T, LPC, 8, VEC>(a, s);
    else launch_tokens<T, LPC, 16, VEC>(a, s);
}
template <typename T> static hipError_t launch_scan(const ScanArgs& a, const ScanPlan& s, hipStream_t st) {
    if (s.seg) {
        const hipError_t e = launch_scan_ends<T>(a, s, false, st);
        if (e != hipSuccess) return e;
    }
    switch (s.lpc) {
#define HDLA_SCAN_CASE(LPCV)                                  \
    case LPCV:                                                \
        if (s.vec) launch_lpc<T, LPCV, true>(a, st);          \
        else launch_lpc<T, LPCV, false>(a, st);               \
        break;
        HDLA_SCAN_CASE(2)
        HDLA_SCAN_CASE(4)
        HDLA_SCAN_CASE(8)
        HDLA_SCAN_CASE(16)
#undef HDLA_SCAN_CASE
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace hdla

using namespace hdla;

extern "C" int hdla_state_space_version(void) { return HDLA_STATE_SPACE_VERSION; }
extern "C" size_t hdla_scan_fwd_workspace_bytes(const hdla_scan_dims* dims) {
    ScanPlan s;
    if (scan_plan(dims, s)) return 0;
    scan_segments(dims, s, SEGMENT_COST_FORWARD, s.blocks);
    return ends_bytes(s);
}
extern "C" int hdla_scan_fwd(const hdla_scan_dims* dims, const void* x, const void* dt, const void* A, const void* B, const void* C, const void* D, const void* z,
                             const void* dt_bias, const float* h0, void* y, float* ht, void* states, size_t states_bytes, void* workspace, size_t workspace_bytes, void* stream) {
    ScanPlan s;
    const int rc = scan_plan(dims, s);
    if (rc) return rc;
    if (!A || (s.rows > 0 && (!x || !dt || !B || !C || !y))) return HDLA_ERR_NULL;
    if (!fits(y, 16) || !fits(h0, 16) || !fits(ht, 16)) return HDLA_ERR_ALIGN;
    if (states && (!fits(states, 16) || states_bytes < (size_t)s.ckpt * s.blocks * 1024)) return HDLA_ERR_WORKSPACE;
    if (!s.units) return HDLA_OK;
    scan_segments(dims, s, SEGMENT_COST_FORWARD, s.blocks);
    if (s.seg && (!workspace || !fits(workspace, 16) || workspace_bytes < ends_bytes(s))) return HDLA_ERR_WORKSPACE;
    ScanArgs a = scan_args(dims, s, x, dt, A, B, C, D, z, dt_bias);
    a.h0 = h0; a.ht = ht; a.y = y; a.ckpt = static_cast<float*>(states); a.ends = static_cast<float*>(workspace);
    s.vec = scan_vec(dims, s, a);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (a.cu) {
        PackedOut out{};
        out.add(y, (long long)dims->D * (dims->dtype == HDLA_BF16 ? 2 : 4));
        const hipError_t e = launch_clear_uncovered(a.cu, a.N, a.T, out, st);
        if (e != hipSuccess) return (int)e;
    }
    const hipError_t e = dims->dtype == HDLA_BF16 ? launch_scan<bf16>(a, s, st) : launch_scan<float>(a, s, st);
    return e == hipSuccess ? HDLA_OK : (int)e;
}
extern "C" size_t hdla_scan_states_bytes(const hdla_scan_dims* dims) {
    ScanPlan s;
    return scan_plan(dims, s) ? 0 : (size_t)s.ckpt * s.blocks * 1024;
}
extern "C" int hdla_scan_step(const hdla_scan_dims* dims, const void* x, const void* dt, const void* A, const void* B, const void* C, const void* D, const void* z,
                              const void* dt_bias, const float* state, void* y, float* new_state, void* stream) {
    ScanPlan s;
    const int rc = scan_plan(dims, s);
    if (rc) return rc;
    if (dims->T != 1 || dims->cu_seqlens) return HDLA_ERR_SHAPE;
    if (!dims->N) return HDLA_OK;
    if (!x || !dt || !A || !B || !C || !y || !state || !new_state) return HDLA_ERR_NULL;
    if (!fits(y, 16) || !fits(state, 16) || !fits(new_state, 16)) return HDLA_ERR_ALIGN;
    ScanArgs a = scan_args(dims, s, x, dt, A, B, C, D, z, dt_bias);
    a.h0 = state; a.ht = new_state; a.y = y;
    int log2 = 0;
    while ((4 << log2) < dims->S) ++log2;
    // four sequences a thread where that leaves every compute unit sixteen waves.  us, one / four, of 4096 channels with 16 states: 4 sequences 3.4 / 4.9, 32 of them (the half of
    // that) 6.0 / 6.5, 64 9.1 / 9.1, 256 27.5 / 24.6
    const long long blocks = (((long long)a.DD << log2) + 255) / 256;
    const int nb = blocks * ((a.N + 3) / 4) >= 1024 ? 4 : 1;
    const long long rows = (a.N + nb - 1) / nb;
    if (blocks > 0x7fffffffLL || rows > 65535) return HDLA_ERR_SHAPE;
    const int es = dims->dtype == HDLA_BF16 ? 2 : 4;
    bool vec = dims->S % 4 == 0 && fits(a.A, 16) && a.B_group % 4 == 0 && a.C_group % 4 == 0;
    for (const Operand* o : {&a.B, &a.C}) vec = vec && fits(o->p, 4 * es) && o->batch % 4 == 0;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const dim3 grid((unsigned)blocks, (unsigned)rows), block(256);
#define HDLA_STEP(T, NB)                                                                                          \
    if (vec) hipLaunchKernelGGL((scan_step_kernel<T, NB, true>), grid, block, 0, st, a, log2);                     \
    else hipLaunchKernelGGL((scan_step_kernel<T, NB, false>), grid, block, 0, st, a, log2)
    if (dims->dtype == HDLA_BF16) {
        if (nb == 4) { HDLA_STEP(bf16, 4); } else { HDLA_STEP(bf16, 1); }
    } else {
        if (nb == 4) { HDLA_STEP(float, 4); } else { HDLA_STEP(float, 1); }
    }
#undef HDLA_STEP
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? HDLA_OK : (int)e;
}
