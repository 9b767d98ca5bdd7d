// Segments of the selective scan: what each leaves if nothing enters it, and its decays.  From the front the state behind its last token, from the back the gradient of
// the state before its first one: G_t = exp(delta_t A) (G_{t+1} + C_t e_t), e_t = dy_t silu(z_t).
//
// A workgroup has a segment of a block of channels; each of its eight waves walks an eighth of the tokens by itself, and they meet once, at the end.  Bound by the vector ALU:
// half of the issue slots a state and token that the scan takes, from the back a sixth.
#include "state_space_ends.h"

namespace hdla {

template <typename T, int LPC, bool VEC, bool BACK>
__global__ __launch_bounds__(512) void scan_ends_kernel(ScanArgs p) {
    constexpr int TOK = SS_TOK, W = 8, PITCH = ss_pitch(TOK);
    using Lane = ScanLane<LPC, TOK>;
    constexpr int CHN = Lane::CHN, V = Lane::V;
    struct Mine { f32x4 B[TOK * LPC]; float d[CHN * PITCH], x[CHN * PITCH]; };
    struct Meet { f32x4 P[W][64], E[W][64]; };
    __shared__ __attribute__((aligned(16))) Mine mine[W];
    __shared__ Meet meet;
    int unit, block;
    if (!scan_work(blockIdx.x, p.blocks, unit, block)) return;
    const Unit U(p, unit);
    if (!U.ok || (BACK ? U.index == 0 : U.to == U.len)) return;           // (nothing comes behind it)
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane_id(), tid = threadIdx.x;
    const Lane L(p, block);
    Mine& my = mine[w];
    const long long batch = p.cu ? 0 : U.n, row0 = p.cu ? U.bos : (long long)U.n * p.T;
    f32x4 A2 = zero4(), E = zero4();
    float bias[V], sum = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (j < L.left) A2[j] = ld_decay(p.A, p.A_f32, (long long)L.d * p.S + 4 * L.q + j);
#pragma unroll
    for (int i = 0; i < V; ++i) bias[i] = p.bias && i < L.carried ? ld_param(p.bias, p.bias_f32, L.dv + i) : 0.f;
    const int pieces = (U.to - U.from + W * TOK - 1) / (W * TOK), start = U.from + w * pieces * TOK, begin = BACK ? start + (pieces - 1) * TOK : start;
    const long long first = U.bos + begin, way = BACK ? -TOK : TOK;
    const Operand& in = BACK ? p.C : p.B;
    Cursor<T> cdt(row_of<T>(p.dt, batch, first) + L.d0, p.dt.row * way), cB(row_of<T>(in, batch, first) + L.group * (BACK ? p.C_group : p.B_group), in.row * way),
        cx(BACK ? static_cast<const T*>(p.dy) + (row0 + begin) * p.DD + L.d0 : row_of<T>(p.x, batch, first) + L.d0, (BACK ? (long long)p.DD : p.x.row) * way),
        cz(row_of<T>(p.z, batch, first) + L.d0, p.z.row * way);
    const uint32_t odt = L.offset(p.dt.row, sizeof(T)), ox = L.offset(BACK ? (long long)p.DD : p.x.row, sizeof(T)), oz = L.offset(p.z.row, sizeof(T));
    Raw<T, V, VEC> rx, rdt, rz;
    StatesOf<T, LPC, TOK, VEC> rB;
    auto request = [&](int t0) __attribute__((always_inline)) {
        const int tokens = min(max(U.to - t0, 0), TOK);
        const bool live = L.tok < tokens && L.carried > 0;
        rx.load(cx.rows(), live ? ox : NOWHERE, L.carried);
        rdt.load(cdt.rows(), live ? odt : NOWHERE, L.carried);
        if (BACK && p.z.p) rz.load(cz.rows(), live ? oz : NOWHERE, L.carried);
        else rz.clear();
        rB.load(cB, (uint32_t)in.row, tokens, p.S);
        cx.next(); cdt.next(); cz.next(); cB.next();
    };
    request(begin);
    for (int piece = 0, t0 = begin; piece < pieces; ++piece, t0 += (int)way) {
        const int tokens = min(max(U.to - t0, 0), TOK);
        float z[V], g[V];
#pragma unroll
        for (int i = 0; i < V; ++i) z[i] = rz[i];
        if (BACK && p.z.p) sigmoid_each<T, V>(z, g);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float e;
            const float v = rdt[i] + bias[i], delta = L.tok < tokens ? (p.softplus ? softplus<T>(v, e) : v) : 0.f;
            if (L.tok < TOK) {
                my.d[(L.ch + i) * PITCH + L.tok] = delta;
                my.x[(L.ch + i) * PITCH + L.tok] = BACK ? (p.z.p ? rx[i] * (z[i] * g[i]) : rx[i]) : delta * rx[i];
            }
        }
        rB.put(my.B);
        if (piece + 1 < pieces) request(t0 + (int)way);
        wave_lds_fence();
        const float *const mine_d = &my.d[L.c * PITCH], *const mine_x = &my.x[L.c * PITCH];
#pragma unroll
        for (int i = 0; i < TOK; ++i) {
            const int k = BACK ? TOK - 1 - i : i;
            const f32x4 b = my.B[k * LPC + L.q];
            const float dl = mine_d[k], u = mine_x[k];
            sum += dl;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float a = __builtin_amdgcn_exp2f(dl * A2[j]);
                E[j] = BACK ? a * __builtin_fmaf(u, b[j], E[j]) : __builtin_fmaf(a, E[j], u * b[j]);
            }
        }
        wave_lds_fence();
    }
    f32x4 P;
#pragma unroll
    for (int j = 0; j < 4; ++j) P[j] = __builtin_amdgcn_exp2f(sum * A2[j]);
    meet.P[w][l] = P;
    meet.E[w][l] = E;
    __syncthreads();
    if (tid >= 256) return;
    float end = 0.f, decay = 1.f;
#pragma unroll
    for (int i = 0; i < W; ++i) {
        const int k = (BACK ? W - 1 - i : i) * 256 + tid;
        const float f = reinterpret_cast<const float*>(meet.P)[k];
        end = __builtin_fmaf(f, end, reinterpret_cast<const float*>(meet.E)[k]);
        decay *= f;
    }
    float* const to = ends_of(p, unit, block) + tid;
    to[0] = end;
    to[256] = decay;
}

template <typename T, int LPC> static void launch_ends(const ScanArgs& a, bool vec, bool back, hipStream_t s) {
    const dim3 grid((unsigned)scan_workgroups(a.blocks, a.units)), block(512);
    if (back) {
        if (vec) hipLaunchKernelGGL((scan_ends_kernel<T, LPC, true, true>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((scan_ends_kernel<T, LPC, false, true>), grid, block, 0, s, a);
    } else {
        if (vec) hipLaunchKernelGGL((scan_ends_kernel<T, LPC, true, false>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((scan_ends_kernel<T, LPC, false, false>), grid, block, 0, s, a);
    }
}
template <typename T> hipError_t launch_scan_ends(const ScanArgs& a, const ScanPlan& s, bool back, hipStream_t stream) {
    switch (s.lpc) {
        case 2: launch_ends<T, 2>(a, s.vec, back, stream); break;
        case 4: launch_ends<T, 4>(a, s.vec, back, stream); break;
        case 8: launch_ends<T, 8>(a, s.vec, back, stream); break;
        case 16: launch_ends<T, 16>(a, s.vec, back, stream); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}
template hipError_t launch_scan_ends<bf16>(const ScanArgs&, const ScanPlan&, bool, hipStream_t);
template hipError_t launch_scan_ends<float>(const ScanArgs&, const ScanPlan&, bool, hipStream_t);

}  // namespace hdla
