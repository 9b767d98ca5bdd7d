// The selective state space scan's backward pass.  With e_t = dy_t silu(z_t) and G_t the gradient of h_t,
//     G_t = C_t e_t + exp(delta_{t+1} A) G_{t+1};   u_t = exp(delta_t A) h_{t-1};
//     dC_t = sum_d e h;  dB_t = sum_d G delta x;  dx = delta sum_s G B + D e;  d delta = sum_s G (A u + x B);  dA = sum_t G delta u;
//     dD = sum_t e x;  dz = dy (C . h + D x) silu'(z);  dh_0 = exp(delta_1 A) G_1.
// Tiles of 64 or 32 tokens, the last first, each from the state that the forward pass left at its first token.  A wave scans its eight tokens forwards and backwards
// from zero; both chains over the waves' pieces run at once, four waves each (of four waves: one behind the other); then it walks them again with what enters, states and decays in registers.
//
// What bounds it: the vector ALU, busy 76 % of the time (4 x 2048 x 2048 x 16 some 285 us, and 22 for the sums of dB and dC): 30 issue slots a state and token in all (27 instructions; an
// exponential and a lane swap are two slots), of which two are the exponential, fifteen the other arithmetic of the four walks, six the sums over channels for dB and dC, two the sums over
// a channel's lanes and five what there is once for a token and channel: step sizes, gates, results, addresses.
#include "column_sums.cuh"
#include "hdla_launch.h"
#include "state_space.cuh"
#include "state_space_ends.h"

namespace hdla {

// x and y of all lanes: their sums over pairs of lanes that are 32 (16) apart, x's in the lower half (the even rows of 16), y's in the upper (odd ones)
__device__ __forceinline__ float fold32(float x, float y) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_int(x), __float_as_int(y), false, false);
    return __int_as_float(r[0]) + __int_as_float(r[1]);
}
__device__ __forceinline__ float fold16(float x, float y) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_int(x), __float_as_int(y), false, false);
    return __int_as_float(r[0]) + __int_as_float(r[1]);
}

template <typename T, int LPC, int TOK, int W, bool VEC>
__global__ __launch_bounds__(64 * W) void scan_grad_kernel(ScanArgs p) {
    using Lane = ScanLane<LPC, TOK>;
    constexpr int CHN = Lane::CHN, V = Lane::V, TILE = W * TOK, PITCH = ss_pitch(TOK);
    static_assert(W == 4 || W == 8, "a thread a state for either chain, or for both");
    // a wave's own: its arrays lie at fixed distances, so that a lane holds one address for all of them
    struct Mine { f32x4 B[TOK * LPC], C[TOK * LPC]; float d[CHN * PITCH], x[CHN * PITCH], e[CHN * PITCH], y[CHN * PITCH]; };
    struct Meet { f32x4 P[W][64], E[W][64], G[W][64]; };
    __shared__ __attribute__((aligned(16))) Mine mine[W];
    __shared__ Meet meet;

    int slot, block;
    if (!scan_work(blockIdx.x, p.take * p.G, slot, block)) return;
    if (p.take < p.per_group) block = block / p.take * p.per_group + p.first + block % p.take;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane_id(), tid = threadIdx.x;
    const Lane L(p, block);
    Mine& my = mine[w];
    f32x4 A2 = zero4(), dA = zero4();
    float bias[V], D[V], dD[V], dbias[V];
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (j < L.left) A2[j] = ld_decay(p.A, p.A_f32, (long long)L.d * p.S + 4 * L.q + j);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        bias[i] = p.bias && i < L.carried ? ld_param(p.bias, p.bias_f32, L.dv + i) : 0.f;
        D[i] = p.D && i < L.carried ? ld_param(p.D, p.D_f32, L.dv + i) : 0.f;
        dD[i] = dbias[i] = 0.f;
    }
    // a thread a state: the first four waves chain the states, the other four (if there are) their gradients
    const int e = tid & 255, ec = (e >> 2) / LPC, es = 4 * ((e >> 2) % LPC) + (e & 3);
    const bool forwards = tid < 256, backwards = W < 8 || tid >= 256, there = (block % p.per_group) * CHN + ec < p.DD / p.G && es < p.S;

    for (int unit = slot; unit < p.units; unit += p.slots) {
        const Unit U(p, unit);
        if (!U.ok) continue;                              // (the same on all threads)
        const int n = U.n, len = U.to;
        const int64_t bos = U.bos;
        const long long batch = p.cu ? 0 : n, row0 = p.cu ? bos : (long long)n * p.T;
        const long long state = ((long long)n * p.DD + L.d0 + ec) * p.S + es;
        float enters = backwards && there && p.dht ? p.dht[state] : 0.f;
        if (backwards)
            for (int i = U.segments(p) - 1; i > U.index; --i) {
                const float* const left = ends_of(p, unit - U.index + i, block) + e;
                enters = __builtin_fmaf(left[256], enters, left[0]);
            }

        const int tiles = (len + TILE - 1) / TILE, until = U.from / TILE;
        const long long first = bos + (long long)(tiles - 1) * TILE + w * TOK, frow = row0 + (long long)(tiles - 1) * TILE + w * TOK;
        Cursor<T> cx(row_of<T>(p.x, batch, first) + L.d0, -p.x.row * TILE), cdt(row_of<T>(p.dt, batch, first) + L.d0, -p.dt.row * TILE),
            cz(row_of<T>(p.z, batch, first) + L.d0, -p.z.row * TILE), cB(row_of<T>(p.B, batch, first) + L.group * p.B_group, -p.B.row * TILE),
            cC(row_of<T>(p.C, batch, first) + L.group * p.C_group, -p.C.row * TILE),
            cdy(static_cast<const T*>(p.dy) + frow * p.DD + L.d0, -(long long)p.DD * TILE);
        long long at_row = frow * p.DD + L.d0;            // dy and the gradients lie alike
        const uint32_t ox = L.offset(p.x.row, sizeof(T)), odt = L.offset(p.dt.row, sizeof(T)), oz = L.offset(p.z.row, sizeof(T)), oy = L.offset(p.DD, sizeof(T));
        Raw<T, V, VEC> rx, rdt, rz, rdy;
        StatesOf<T, LPC, TOK, VEC> rB, rC;
        auto request = [&](int t0) __attribute__((always_inline)) {
            const int tokens = t0 < U.from ? 0 : min(max(len - t0, 0), TOK);
            const bool live = L.tok < tokens && L.carried > 0;
            rx.load(cx.rows(), live ? ox : NOWHERE, L.carried);
            rdt.load(cdt.rows(), live ? odt : NOWHERE, L.carried);
            if (p.z.p) rz.load(cz.rows(), live ? oz : NOWHERE, L.carried);
            else rz.clear();
            rdy.load(cdy.rows(), live ? oy : NOWHERE, L.carried);
            rB.load(cB, (uint32_t)p.B.row, tokens, p.S);
            rC.load(cC, (uint32_t)p.C.row, tokens, p.S);
            cx.next(); cdt.next(); cz.next(); cdy.next(); cB.next(); cC.next();
        };
        const float* const entered = ckpt_of(p, n, bos, block);
        // this block's part of dB and dC: [block of the group in this pass][B, C][row][group][S]
        const long long inner = (long long)p.G * p.S, half = p.rows * inner;
        float* const part0 = p.part_bc + 2 * half * (block % p.per_group - p.first) + (long long)L.group * p.S;
        request((tiles - 1) * TILE + w * TOK);
        for (int tile = tiles - 1; tile >= until; --tile) {
            const int t0 = tile * TILE + w * TOK, tokens = min(max(len - t0, 0), TOK);
            const float left = forwards ? entered[tile * (p.blocks * 256LL) + e] : 0.f;
            float x[V], z[V], dy[V], v[V], ev[V], gz[V], delta[V], ee[V];
#pragma unroll
            for (int i = 0; i < V; ++i) { x[i] = rx[i]; z[i] = rz[i]; dy[i] = rdy[i]; v[i] = rdt[i] + bias[i]; }
            if (p.z.p) sigmoid_each<T, V>(z, gz);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                delta[i] = L.tok < tokens ? (p.softplus ? softplus<T>(v[i], ev[i]) : v[i]) : 0.f;
                ee[i] = p.z.p ? dy[i] * (z[i] * gz[i]) : dy[i];
                const int place = (L.ch + i) * PITCH + L.tok;
                if (L.tok < TOK) {
                    my.d[place] = delta[i];
                    my.x[place] = delta[i] * x[i];
                    my.e[place] = ee[i];
                }
            }
            rB.put(my.B);
            rC.put(my.C);
            request(t0 - TILE);
            wave_lds_fence();
            f32x4 a[TOK], add[TOK], E = zero4(), G = zero4();         // decays; what each token adds
            const float *const mine_d = &my.d[L.c * PITCH], *const mine_x = &my.x[L.c * PITCH], *const mine_e = &my.e[L.c * PITCH];
            float sum = 0.f;
            // (in all the walks: the next token's operands are on their way while this one's are worked on)
            {
                f32x4 b = my.B[L.q];
                float dl = mine_d[0], u = mine_x[0];
#pragma unroll
                for (int k = 0; k < TOK; ++k) {
                    f32x4 b1;
                    float dl1, u1;
                    if (k + 1 < TOK) { b1 = my.B[(k + 1) * LPC + L.q]; dl1 = mine_d[k + 1]; u1 = mine_x[k + 1]; }
                    sum += dl;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        a[k][j] = __builtin_amdgcn_exp2f(dl * A2[j]);
                        add[k][j] = u * b[j];
                        E[j] = __builtin_fmaf(a[k][j], E[j], add[k][j]);
                    }
                    apart();
                    if (k + 1 < TOK) { b = b1; dl = dl1; u = u1; }
                }
            }
            {
                f32x4 cc = my.C[(TOK - 1) * LPC + L.q];
                float et = mine_e[TOK - 1];
#pragma unroll
                for (int k = TOK - 1; k >= 0; --k) {
                    f32x4 c1;
                    float e1;
                    if (k) { c1 = my.C[(k - 1) * LPC + L.q]; e1 = mine_e[k - 1]; }
#pragma unroll
                    for (int j = 0; j < 4; ++j) G[j] = a[k][j] * __builtin_fmaf(cc[j], et, G[j]);
                    apart();
                    if (k) { cc = c1; et = e1; }
                }
            }
            f32x4 P;
#pragma unroll
            for (int j = 0; j < 4; ++j) P[j] = __builtin_amdgcn_exp2f(sum * A2[j]);
            meet.P[w][l] = P;
            meet.E[w][l] = E;
            meet.G[w][l] = G;
            __syncthreads();
            {
                const float* const f = reinterpret_cast<const float*>(meet.P) + e;
                float decays[W], ends[W];
#pragma unroll
                for (int i = 0; i < W; ++i) decays[i] = f[i * 256];
                if (forwards) {
                    float* const at = reinterpret_cast<float*>(meet.E) + e;
                    float h = left;
#pragma unroll
                    for (int i = 0; i < W; ++i) ends[i] = at[i * 256];
#pragma unroll
                    for (int i = 0; i < W; ++i) {
                        at[i * 256] = h;
                        h = __builtin_fmaf(decays[i], h, ends[i]);
                    }
                }
                if (backwards) {
                    float* const at = reinterpret_cast<float*>(meet.G) + e;
#pragma unroll
                    for (int i = 0; i < W; ++i) ends[i] = at[i * 256];
#pragma unroll
                    for (int i = W - 1; i >= 0; --i) {
                        at[i * 256] = enters;
                        enters = __builtin_fmaf(decays[i], enters, ends[i]);
                    }
                }
            }
            __syncthreads();
            const f32x4 first = meet.E[w][l];
            G = meet.G[w][l];
            f32x4 h[TOK];
            {
                f32x4 cc = my.C[L.q];
#pragma unroll
                for (int k = 0; k < TOK; ++k) {
                    f32x4 c1;
                    if (k + 1 < TOK) c1 = my.C[(k + 1) * LPC + L.q];
                    float y[1] = {0.f};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        h[k][j] = __builtin_fmaf(a[k][j], k ? h[k - 1][j] : first[j], add[k][j]);
                        y[0] = __builtin_fmaf(h[k][j], cc[j], y[0]);
                    }
                    sum_channel<LPC>(y);
                    my.y[L.c * PITCH + k] = y[0];        // (the same from all lanes of the channel)
                    apart();
                    if (k + 1 < TOK) cc = c1;
                }
            }
            wave_lds_fence();                             // B and C are read again, not kept
            f32x4 b = my.B[(TOK - 1) * LPC + L.q], cc = my.C[(TOK - 1) * LPC + L.q];
            float dl = mine_d[TOK - 1], u = mine_x[TOK - 1], et = mine_e[TOK - 1];
#pragma unroll
            for (int k = TOK - 1; k >= 0; --k) {
                f32x4 b1, c1;
                float dl1, u1, e1;
                if (k) { b1 = my.B[(k - 1) * LPC + L.q]; c1 = my.C[(k - 1) * LPC + L.q]; dl1 = mine_d[k - 1]; u1 = mine_x[k - 1]; e1 = mine_e[k - 1]; }
                float s[2] = {0.f, 0.f}, db[4], dc[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float g = __builtin_fmaf(cc[j], et, G[j]);
                    dc[j] = et * h[k][j];
                    db[j] = g * u;
                    s[0] = __builtin_fmaf(g, b[j], s[0]);
                    G[j] = a[k][j] * g;
                    const float through = G[j] * (k ? h[k - 1][j] : first[j]);
                    s[1] = __builtin_fmaf(through, A2[j], s[1]);
                    dA[j] = __builtin_fmaf(through, dl, dA[j]);
                }
                // over the wave's channels: lanes with the same states
                float f0 = fold16(fold32(db[0], dc[0]), fold32(db[1], dc[1])), f1 = fold16(fold32(db[2], dc[2]), fold32(db[3], dc[3]));
                if constexpr (LPC < 16) { f0 += dpp0<0x128>(f0); f1 += dpp0<0x128>(f1); }      // row_ror:8
                if constexpr (LPC < 8) { f0 += dpp0<0x124>(f0); f1 += dpp0<0x124>(f1); }
                if constexpr (LPC < 4) { f0 += dpp0<0x122>(f0); f1 += dpp0<0x122>(f1); }
                sum_channel<LPC>(s);
                // (what this token had there has been read: B, C, delta, delta x)
                my.d[L.c * PITCH + k] = s[0];
                my.x[L.c * PITCH + k] = s[1];
                if ((l & 15) < LPC) {
                    float* const to = reinterpret_cast<float*>(&(l < 32 ? my.B : my.C)[k * LPC + (l & 15)]) + ((l >> 4) & 1);
                    to[0] = f0;
                    to[2] = f1;
                }
                apart();
                if (k) { b = b1; cc = c1; dl = dl1; u = u1; et = e1; }
            }
            wave_lds_fence();
            float gx[V], gdt[V], gzz[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int place = (L.ch + i) * PITCH + min(L.tok, TOK - 1);
                const float gb = my.d[place], ga = my.x[place] * LN2, inner = __builtin_fmaf(D[i], x[i], my.y[place]);
                gx[i] = __builtin_fmaf(D[i], ee[i], gb * delta[i]);
                gdt[i] = __builtin_fmaf(gb, x[i], ga);
                if (p.softplus) gdt[i] *= softplus_slope(v[i], ev[i]);
                if (p.z.p) gzz[i] = dy[i] * inner * (gz[i] * __builtin_fmaf(z[i], 1.f - gz[i], 1.f));
                if (L.tok < tokens) {
                    dD[i] = __builtin_fmaf(ee[i], x[i], dD[i]);
                    dbias[i] += gdt[i];
                }
            }
            if (L.tok < tokens && L.carried > 0) {
                st_values<T, V, VEC>(at(static_cast<T*>(p.dx) + at_row, oy), gx, L.carried);
                st_values<T, V, VEC>(at(static_cast<T*>(p.ddt) + at_row, oy), gdt, L.carried);
                if (p.z.p) st_values<T, V, VEC>(at(static_cast<T*>(p.dz) + at_row, oy), gzz, L.carried);
            }
            at_row -= (long long)TILE * p.DD;
            asm("" : "+s"(at_row));
            {
                float* const to = part0 + (row0 + t0) * inner;
                constexpr int PIECES = TOK * LPC < 64 ? 1 : TOK * LPC / 64;
#pragma unroll
                for (int i = 0; i < PIECES; ++i) {
                    const int piece = i * 64 + l, t = piece / LPC, s = piece % LPC * 4;
                    if (t < tokens && s < p.S) {
                        st_states(to + t * inner + s, my.B[piece], p.S - s, VEC);
                        st_states(to + half + t * inner + s, my.C[piece], p.S - s, VEC);
                    }
                }
            }
            wave_lds_fence();
        }
        if (backwards && there && p.dh0 && U.index == 0) p.dh0[state] = enters;
    }
    // what the waves have of dA, dD and d bias
    __syncthreads();
    meet.E[w][l] = dA;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        // over the tokens
#pragma unroll
        for (int m = CHN / V; m < 64; m *= 2) { dD[i] += __shfl_xor(dD[i], m); dbias[i] += __shfl_xor(dbias[i], m); }
        if (l < CHN / V) { my.d[L.ch + i] = dD[i]; my.x[L.ch + i] = dbias[i]; }
    }
    __syncthreads();
    if (forwards) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < W; ++i) s += reinterpret_cast<const float*>(meet.E)[i * 256 + e];
        if (there) p.part_own[(long long)slot * p.DD * (p.S + 2) + (long long)(L.d0 + ec) * p.S + es] = s;
    }
    if (backwards && e < CHN && (block % p.per_group) * CHN + e < p.DD / p.G) {
        float s = 0.f, b = 0.f;
#pragma unroll
        for (int i = 0; i < W; ++i) { s += mine[i].d[e]; b += mine[i].x[e]; }
        float* const to = p.part_own + (long long)slot * p.DD * (p.S + 2) + (long long)p.DD * p.S + L.d0 + e;
        to[0] = s;
        to[p.DD] = b;
    }
}

// Partial sums of dB and dC are a fp32 copy of both for every block of 64 / lanes channels: with more channels and states they outgrow everything else (8192 channels with 64 states: 64
// times x in bf16).  So a pass takes as many blocks of a group as fit into PARTS_MOST, and the next one goes on with their sums, which lie in front of its own parts: the same additions in the
// same order as in one pass.  ms a training step and GB of parts, in one pass / so, with 4096 channels and 64 states in bf16: 4 x 2048 tokens 3.91 and 4.3 / 3.95 and 2.2, 1 x 32768 (whose
// passes are cut into segments) 16.1 and 17.2 / 17.7 and 2.2.
constexpr size_t PARTS_MOST = (size_t)2 << 30;
static size_t part_floats(const hdla_scan_dims* d, const ScanPlan& s) { return 2 * (size_t)s.rows * d->G * d->S; }
static void grad_plan(const hdla_scan_dims* d, ScanPlan& s) {
    const size_t one = part_floats(d, s) * 4;
    s.take = s.per_group;
    s.passes = 1;
    if (s.per_group * one > PARTS_MOST) {
        // (as many as are whole rounds of two workgroups a compute unit, where a round fits)
        const long long most = std::max<size_t>(PARTS_MOST / one, 1), full = std::max(1LL, 512 / ((long long)d->G * d->N)), round = most < full ? 1 : full;
        const long long rounds = (s.per_group + round - 1) / round, passes = (rounds + most / round - 1) / (most / round);
        s.take = (int)((rounds + passes - 1) / passes * round);
        s.passes = (s.per_group + s.take - 1) / s.take;
    }
    scan_segments(d, s, SEGMENT_COST_BACKWARD, s.take * d->G);
    // Workgroups walk sequences, or segments, in turns so that their partial sums of dA, dD and d bias stay few: as many as fill the device a few times
    s.slots = (int)std::min<long long>(s.units, std::max(1LL, 2048LL / (s.take * d->G)));
}
// partial sums of dB and dC, [sum of earlier passes, where there are several; blocks of a group in a pass][2][rows][G][S], and behind them those of dA, dD and d bias, [slots][D S + 2 D],
// and segments' ends
static size_t bc_bytes(const hdla_scan_dims* d, const ScanPlan& s) { return ((s.take + (s.passes > 1)) * part_floats(d, s) * 4 + 15) / 16 * 16; }
static size_t own_bytes(const hdla_scan_dims* d, const ScanPlan& s) { return ((size_t)s.slots * d->D * (d->S + 2) * 4 + 15) / 16 * 16; }
static size_t grad_bytes(const hdla_scan_dims* d, const ScanPlan& s) { return std::max<size_t>(bc_bytes(d, s) + own_bytes(d, s) + ends_bytes(s), 16); }
template <typename T, int LPC, int W> static void launch_grad_waves(const ScanArgs& a, bool vec, hipStream_t s) {
    constexpr int TOK = SS_TOK;
    const dim3 grid((unsigned)scan_workgroups(a.take * a.G, a.slots)), block(64 * W);
    if (vec) hipLaunchKernelGGL((scan_grad_kernel<T, LPC, TOK, W, true>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((scan_grad_kernel<T, LPC, TOK, W, false>), grid, block, 0, s, a);
}
template <typename T, int LPC> static void launch_grad(const ScanArgs& a, bool vec, hipStream_t s) {
    static_assert(SS_TILE_MANY == 4 * SS_TOK && SS_TILE_FEW == 8 * SS_TOK && SS_TILE_MANY == 1 << 5 && SS_TILE_FEW == 1 << 6, "a tile begins where a state is left");
    if (a.every_log2 == 5) launch_grad_waves<T, LPC, 4>(a, vec, s);
    else launch_grad_waves<T, LPC, 8>(a, vec, s);
}
template <typename T> static hipError_t launch_scan_grad(const ScanArgs& a, const ScanPlan& s, hipStream_t st) {
    switch (s.lpc) {
        case 2: launch_grad<T, 2>(a, s.vec, st); break;
        case 4: launch_grad<T, 4>(a, s.vec, st); break;
        case 8: launch_grad<T, 8>(a, s.vec, st); break;
        case 16: launch_grad<T, 16>(a, s.vec, st); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace hdla

using namespace hdla;

extern "C" size_t hdla_scan_workspace_bytes(const hdla_scan_dims* dims) {
    ScanPlan s;
    if (scan_plan(dims, s)) return 0;
    grad_plan(dims, s);
    return grad_bytes(dims, s);
}
extern "C" int hdla_scan_bwd(const hdla_scan_dims* dims, const void* x, const void* dt, const void* A, const void* B, const void* C, const void* D, const void* z,
                             const void* dt_bias, const void* dy, const float* dht, const void* states, size_t states_bytes, void* dx, void* ddt, void* dA, void* dB,
                             void* dC, void* dD, void* dz, void* ddt_bias, float* dh0, void* workspace, size_t workspace_bytes, void* stream) {
    ScanPlan s;
    const int rc = scan_plan(dims, s);
    if (rc) return rc;
    if (!A || !dA || (D && !dD) || (dt_bias && !ddt_bias)) return HDLA_ERR_NULL;
    if (s.rows > 0 && (!x || !dt || !B || !C || !dy || !dx || !ddt || !dB || !dC || !states || (z && !dz))) return HDLA_ERR_NULL;
    for (const void* q : {dy, (const void*)dht, states, (const void*)dx, (const void*)ddt, (const void*)dB, (const void*)dC, (const void*)dz, (const void*)dh0})
        if (!fits(q, 16)) return HDLA_ERR_ALIGN;
    grad_plan(dims, s);
    if (!workspace || !fits(workspace, 16) || workspace_bytes < grad_bytes(dims, s)) return HDLA_ERR_WORKSPACE;
    if (s.rows > 0 && states_bytes < (size_t)s.ckpt * s.blocks * 1024) return HDLA_ERR_WORKSPACE;
    ScanArgs a = scan_args(dims, s, x, dt, A, B, C, D, z, dt_bias);
    a.dy = dy; a.dht = dht; a.ckpt = static_cast<float*>(const_cast<void*>(states));
    a.dx = dx; a.ddt = ddt; a.dz = dz; a.dh0 = dh0;
    char* const base = static_cast<char*>(workspace);
    float* const sums = reinterpret_cast<float*>(base);   // of earlier passes, where there are several
    a.part_bc = sums + (s.passes > 1 ? part_floats(dims, s) : 0);
    a.part_own = reinterpret_cast<float*>(base + bc_bytes(dims, s));
    a.ends = reinterpret_cast<float*>(base + bc_bytes(dims, s) + own_bytes(dims, s));
    s.vec = scan_vec(dims, s, a);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const int es = dims->dtype == HDLA_BF16 ? 2 : 4;
    if (a.cu) {
        PackedOut out{};
        for (void* o : {dx, ddt, dz}) out.add(o, (long long)dims->D * es);
        const hipError_t e = launch_clear_uncovered(a.cu, a.N, a.T, out, st);
        if (e != hipSuccess) return (int)e;
    }
    if (s.seg) {
        const hipError_t e = dims->dtype == HDLA_BF16 ? launch_scan_ends<bf16>(a, s, true, st) : launch_scan_ends<float>(a, s, true, st);
        if (e != hipSuccess) return (int)e;
    }
    ColumnSums k{};
    k.part = a.part_own; k.rows = s.slots;
    k.add(dA, a.A_f32, (long long)dims->D * dims->S);
    k.add(D ? dD : nullptr, a.D_f32, dims->D);
    k.add(dt_bias ? ddt_bias : nullptr, a.bias_f32, dims->D);
    const long long inner = (long long)dims->G * dims->S;
    for (int pass = 0; pass < s.passes; ++pass) {
        a.first = pass * s.take;
        a.take = std::min(s.take, s.per_group - a.first);
        hipError_t e = !s.units ? hipSuccess : dims->dtype == HDLA_BF16 ? launch_scan_grad<bf16>(a, s, st) : launch_scan_grad<float>(a, s, st);
        if (e != hipSuccess) return (int)e;
        const bool last = pass + 1 == s.passes;
        ColumnSums c{};
        c.part = pass ? sums : a.part_bc; c.rows = a.take + (pass > 0);
        c.cu = a.cu; c.N = a.N; c.T = a.T; c.per_token = inner; c.tokens_end = 2 * s.rows * inner;
        if (last) {
            c.add(dB, es == 4, s.rows * inner);
            c.add(dC, es == 4, s.rows * inner);
        } else {
            c.add(sums, true, 2 * s.rows * inner);        // (a thread writes where it has read)
        }
        e = launch_column_sums(c, st, last ? k : ColumnSums{});
        if (e != hipSuccess) return (int)e;
    }
    return HDLA_OK;
}
