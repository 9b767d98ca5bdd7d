// The norms around a block, with its gate and the residual stream: what the block gave, normalised (or not), gated and scaled, is added to the stream, and the sum is
// normalised for the next block.  Per row of E channels:
//     p = x / rms(x) post_weight  (or x);   u = p act(gate)  (or p);   r = residual + scale u;   y = r / rms(r) weight;   rms(v) = sqrt(mean v^2 + eps)
// Backward, from dy and dr (rhat = r / rms(r), xhat = x / rms(x)), with everything formed again from the inputs:
//     m = dy weight;  dr += (m - rhat mean(m rhat)) / rms(r);   dresidual = dr;   dweight = sum dy rhat;   dscale = sum dr u;   du = scale dr;
//     dgate = du p act'(gate);   dp = du act(gate);   dpost_weight = sum dp xhat;   q = dp post_weight;  dx = (q - xhat mean(q xhat)) / rms(x)
//
// Streams through HBM: forward reads x, gate, residual and writes y, r; backward reads these, dy, dr and writes dx, dgate, dresidual.  A row lies in the registers
// of one wave, or of two, four or eight waves of a workgroup where it is long, 16 bytes a lane and piece; its sums are taken across lanes without LDS (several waves' through it).
// 16384 x 4096 in bf16 with an fp32 stream: forward 177 us, 5.3 TB/s, what a large copy reaches; 8192 x 2048 in bf16 forward 28 us, backward 58, the sums of the weights' gradients 9.
// Workgroups stride over rows: weights are read once, and the gradients of weights and scale stay in registers until a workgroup leaves one row of partial sums.
#include "column_sums.cuh"
#include "hdla_common.cuh"
#include "state_space.cuh"

#include <algorithm>

namespace hdla {

struct BlockNormArgs {
    const void *x, *residual, *weight, *post, *gate, *scale, *dy, *dr;
    void *y, *r, *dx, *dresidual, *dgate;
    float* part;                   // [workgroups][3][E]: dweight, dpost, dscale
    long long rows;
    int E, pieces, w_f32, p_f32, s_f32, act, post_norm;
    float factor, inv_e, eps;      // the scale where it is a number
};
enum { ACT_NONE, ACT_SIGMOID, ACT_SILU };

// Which channel is element j of a lane's piece i: N neighbours a lane where rows start on 16 bytes (VEC), else neighbours on neighbouring lanes, so that loads of single
// elements still come as whole lines (10833 rows of 3791 channels, fp32 stream, forward: 357 us with eight neighbours a lane, so 180).
template <int N, int LANES, bool VEC> __device__ __forceinline__ int channel(int i, int j, int lane) { return VEC ? (i * LANES + lane) * N + j : (i * N + j) * LANES + lane; }

// a lane's piece i of a vector; beyond its end, or without one, `none`
template <int N, int LANES, bool VEC> __device__ __forceinline__ void ld_vector(const void* v, int f32, int E, int i, int lane, float none, float (&f)[N]) {
#pragma unroll
    for (int j = 0; j < N; ++j) f[j] = none;
    if (!v) return;
    if constexpr (VEC) {
        const int e = channel<N, LANES, VEC>(i, 0, lane);
        if (e >= E) return;
#pragma unroll
        for (int k = 0; k < N; k += 4) {
            const f32x4 r = f32 ? *reinterpret_cast<const f32x4*>(static_cast<const float*>(v) + e + k) : to_f32(ld_frag(static_cast<const bf16*>(v) + e + k));
#pragma unroll
            for (int j = 0; j < 4; ++j) f[k + j] = r[j];
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int e = channel<N, LANES, VEC>(i, j, lane);
            if (e < E) f[j] = ld_param(v, f32, e);
        }
    }
}
// A lane's pieces of one row as they come from memory: 16 bytes of x's type each.  Lanes behind the row's end, and rows behind the last, ask for nothing and get zeros.
template <typename X, int N, int NV, int LANES, bool VEC> struct RowOf {
    Raw<X, N, VEC> p[NV];
    __device__ __forceinline__ void load(const void* base, long long row, bool live, int E, int lane) {
        const auto rows = __builtin_amdgcn_make_buffer_rsrc(const_cast<X*>(static_cast<const X*>(base) + row * E), 0, NOWHERE_FROM, 0x00027000);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if constexpr (VEC) {
                const int e = channel<N, LANES, VEC>(i, 0, lane);
                p[i].load(rows, live && e < E ? e * (uint32_t)sizeof(X) : NOWHERE, N);
            } else {
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const int e = channel<N, LANES, VEC>(i, j, lane);
                    const uint32_t off = live && e < E ? e * (uint32_t)sizeof(X) : NOWHERE;
                    if constexpr (sizeof(X) == 2) p[i].w[j] = __builtin_amdgcn_raw_buffer_load_b16(rows, off, 0, 0);
                    else p[i].w[j] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rows, off, 0, 0));
                }
            }
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < NV; ++i) p[i].clear();
    }
};
template <typename T, int N, int LANES, bool VEC> __device__ __forceinline__ void st_row(void* base, long long row, int E, int i, int lane, const float (&f)[N]) {
    T* const to = static_cast<T*>(base) + row * E;
    if constexpr (VEC) {
        const int e = channel<N, LANES, VEC>(i, 0, lane);
        if (e < E) st_values<T, N, VEC>(to + e, f, N);
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int e = channel<N, LANES, VEC>(i, j, lane);
            if (e < E) st_elem(to + e, f[j]);
        }
    }
}
// act(g) and its derivative.  The sigmoid's is s (1 - s), and 1 - s = s exp(-g): formed so because of an open gate the difference of one and nearly one is its roundings (a gate
// of 12: 1 % off; above 17: zero).  An exponential that is infinite meets s = 0: bounded, their product is zero.
template <typename T, int N> __device__ __forceinline__ void activate(int act, const float (&g)[N], float (&a)[N], float (&da)[N]) {
    if (act == ACT_NONE) {
#pragma unroll
        for (int i = 0; i < N; ++i) { a[i] = g[i]; da[i] = 1.f; }
        return;
    }
    float s[N];
    sigmoid_each<T, N>(g, s);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        a[i] = act == ACT_SILU ? g[i] * s[i] : s[i];
        da[i] = act == ACT_SILU ? s[i] * __builtin_fmaf(g[i], 1.f - s[i], 1.f) : s[i] * (s[i] * __builtin_amdgcn_fmed3f(exp_t<T>(-g[i]), 0.f, 3.402823466e38f));
    }
}

// Sums over a row: the lanes of a wave, or of several in a workgroup, whose threads all make the same calls; alternating halves of LDS, so one barrier a call
template <int WAVES, int N> struct RowSum {
    float* lds;
    int half = 0;
    __device__ __forceinline__ void operator()(float (&x)[N]) {
        sum_lanes<N>(x, 64);
        if constexpr (WAVES > 1) {
            float* const s = lds + half * WAVES * N;
            if ((threadIdx.x & 63) == 0)
#pragma unroll
                for (int i = 0; i < N; ++i) s[(threadIdx.x >> 6) % WAVES * N + i] = x[i];
            __syncthreads();
#pragma unroll
            for (int i = 0; i < N; ++i) {
                x[i] = s[i];
#pragma unroll
                for (int k = 1; k < WAVES; ++k) x[i] += s[k * N + i];
            }
            half ^= 1;
        }
    }
};

// x and gate of T, residual, r of S.  NV pieces of N channels a lane; WAVES waves a row, a workgroup of four waves (eight of a row of eight).  A row's pieces are on
// their way while the row before it is worked on.
template <int WAVES> struct RowShare {
    static constexpr int THREADS = WAVES == 8 ? 512 : 256, LANES = 64 * WAVES, ROWS = THREADS / LANES;
    long long row, step;
    int lane;
    __device__ __forceinline__ RowShare() {
        const int mine = __builtin_amdgcn_readfirstlane(threadIdx.x / LANES);
        row = (long long)blockIdx.x * ROWS + mine;
        step = (long long)gridDim.x * ROWS;
        lane = threadIdx.x - mine * LANES;
    }
    // (every wave of a workgroup makes as many turns)
    __device__ __forceinline__ int turns(long long rows) const { return (int)((rows - (long long)blockIdx.x * ROWS + step - 1) / step); }
};
template <typename T, typename S, int NV, int WAVES, bool VEC>
__global__ __launch_bounds__(RowShare<WAVES>::THREADS) void block_norm_kernel(BlockNormArgs p) {
    using Share = RowShare<WAVES>;
    constexpr int N = 16 / sizeof(T), LANES = Share::LANES;
    __shared__ float lds[Share::ROWS][2 * WAVES];
    Share at;
    RowSum<WAVES, 1> sum{lds[threadIdx.x / LANES]};
    RowOf<T, N, NV, LANES, VEC> rx, rg;
    RowOf<S, N, NV, LANES, VEC> rr;
    auto request = [&](long long row) __attribute__((always_inline)) {
        const bool live = row < p.rows;
        rx.load(p.x, row, live, p.E, at.lane);
        if (p.gate) rg.load(p.gate, row, live, p.E, at.lane);
        else rg.clear();
        if (p.residual) rr.load(p.residual, row, live, p.E, at.lane);
        else rr.clear();
    };
    request(at.row);
    float w[NV][N], pw[NV][N], sc[NV][N];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        ld_vector<N, LANES, VEC>(p.weight, p.w_f32, p.E, i, at.lane, 1.f, w[i]);
        ld_vector<N, LANES, VEC>(p.post, p.p_f32, p.E, i, at.lane, 1.f, pw[i]);
        ld_vector<N, LANES, VEC>(p.scale, p.s_f32, p.E, i, at.lane, p.factor, sc[i]);
    }
    for (int turn = at.turns(p.rows); turn > 0; --turn, at.row += at.step) {
        const int E = at.row < p.rows ? p.E : 0;
        float x[NV][N], r[NV][N], g[NV][N];
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < N; ++j) { x[i][j] = rx.p[i][j]; r[i][j] = rr.p[i][j]; g[i][j] = rg.p[i][j]; }
        if (turn > 1) request(at.row + at.step);
        float inv = 1.f;
        if (p.post_norm) {
            float s[1] = {0.f};
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < N; ++j) s[0] = __builtin_fmaf(x[i][j], x[i][j], s[0]);
            sum(s);
            inv = 1.f / sqrtf(__builtin_fmaf(s[0], p.inv_e, p.eps));
        }
        float s[1] = {0.f};
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float a[N], da[N];
            if (p.gate) activate<T, N>(p.act, g[i], a, da);
#pragma unroll
            for (int j = 0; j < N; ++j) {
                float u = x[i][j] * inv * pw[i][j];
                if (p.gate) u *= a[j];
                r[i][j] = __builtin_fmaf(u, sc[i][j], r[i][j]);
                s[0] = __builtin_fmaf(r[i][j], r[i][j], s[0]);
            }
        }
        sum(s);
        const float ir = 1.f / sqrtf(__builtin_fmaf(s[0], p.inv_e, p.eps));
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float y[N];
#pragma unroll
            for (int j = 0; j < N; ++j) y[j] = r[i][j] * ir * w[i][j];
            st_row<T, N, LANES, VEC>(p.y, at.row, E, i, at.lane, y);
            st_row<S, N, LANES, VEC>(p.r, at.row, E, i, at.lane, r[i]);
        }
    }
}

template <typename T, typename S, int NV, int WAVES, bool VEC>
__global__ __launch_bounds__(RowShare<WAVES>::THREADS) void block_norm_grad_kernel(BlockNormArgs p) {
    using Share = RowShare<WAVES>;
    constexpr int N = 16 / sizeof(T), LANES = Share::LANES, ROWS = Share::ROWS;
    __shared__ float lds[ROWS][2 * WAVES * 2], lds1[ROWS][2 * WAVES];
    __shared__ float meet[ROWS > 1 ? (ROWS - 1) * NV * N * LANES : 1];
    Share at;
    RowSum<WAVES, 1> sum1{lds1[threadIdx.x / LANES]};
    RowSum<WAVES, 2> sum2{lds[threadIdx.x / LANES]};
    RowOf<T, N, NV, LANES, VEC> rx, rg, rdy;
    RowOf<S, N, NV, LANES, VEC> rr, rdr;
    auto request = [&](long long row) __attribute__((always_inline)) {
        const bool live = row < p.rows;
        rx.load(p.x, row, live, p.E, at.lane);
        if (p.gate) rg.load(p.gate, row, live, p.E, at.lane);
        else rg.clear();
        if (p.residual) rr.load(p.residual, row, live, p.E, at.lane);
        else rr.clear();
        if (p.dy) rdy.load(p.dy, row, live, p.E, at.lane);
        else rdy.clear();
        if (p.dr) rdr.load(p.dr, row, live, p.E, at.lane);
        else rdr.clear();
    };
    const int turns = at.turns(p.rows);
    if (turns > 0) request(at.row);
    float w[NV][N], pw[NV][N], sc[NV][N], acc[3][NV][N];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        ld_vector<N, LANES, VEC>(p.weight, p.w_f32, p.E, i, at.lane, 1.f, w[i]);
        ld_vector<N, LANES, VEC>(p.post, p.p_f32, p.E, i, at.lane, 1.f, pw[i]);
        ld_vector<N, LANES, VEC>(p.scale, p.s_f32, p.E, i, at.lane, p.factor, sc[i]);
#pragma unroll
        for (int k = 0; k < 3; ++k)
#pragma unroll
            for (int j = 0; j < N; ++j) acc[k][i][j] = 0.f;
    }
    for (int turn = turns; turn > 0; --turn, at.row += at.step) {
        const int E = at.row < p.rows ? p.E : 0;          // (places behind the last row: zeros, and no roots of eps, which may be zero, so that they add nothing to the sums)
        // xhat; r; dy, then the gradient of xhat; the gradient of r; act(gate) and its derivative
        float x[NV][N], r[NV][N], m[NV][N], t[NV][N], a[NV][N], da[NV][N];
        float inv = 1.f, s1[1] = {0.f};
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float g[N];
#pragma unroll
            for (int j = 0; j < N; ++j) {
                x[i][j] = rx.p[i][j];
                r[i][j] = rr.p[i][j];
                m[i][j] = rdy.p[i][j];
                t[i][j] = rdr.p[i][j];
                g[j] = rg.p[i][j];
                a[i][j] = 1.f;
                da[i][j] = 0.f;
                s1[0] = __builtin_fmaf(x[i][j], x[i][j], s1[0]);
            }
            if (p.gate) activate<T, N>(p.act, g, a[i], da[i]);
        }
        if (turn > 1) request(at.row + at.step);
        if (p.post_norm) {
            sum1(s1);
            inv = E ? 1.f / sqrtf(__builtin_fmaf(s1[0], p.inv_e, p.eps)) : 0.f;
        }
        float s2[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < N; ++j) {
                x[i][j] *= inv;
                r[i][j] = __builtin_fmaf(sc[i][j], x[i][j] * pw[i][j] * a[i][j], r[i][j]);
                s2[0] = __builtin_fmaf(r[i][j], r[i][j], s2[0]);
                s2[1] = __builtin_fmaf(m[i][j] * w[i][j], r[i][j], s2[1]);
            }
        sum2(s2);
        const float ir = E ? 1.f / sqrtf(__builtin_fmaf(s2[0], p.inv_e, p.eps)) : 0.f, along = s2[1] * ir * p.inv_e;
        s1[0] = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float dg[N];
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const float rh = r[i][j] * ir, pv = x[i][j] * pw[i][j];
                t[i][j] = __builtin_fmaf(ir, m[i][j] * w[i][j] - rh * along, t[i][j]);
                acc[0][i][j] = __builtin_fmaf(m[i][j], rh, acc[0][i][j]);
                acc[2][i][j] = __builtin_fmaf(t[i][j], pv * a[i][j], acc[2][i][j]);
                const float du = t[i][j] * sc[i][j], dp = du * a[i][j];
                dg[j] = du * pv * da[i][j];
                acc[1][i][j] = __builtin_fmaf(dp, x[i][j], acc[1][i][j]);
                m[i][j] = dp * pw[i][j];
                s1[0] = __builtin_fmaf(m[i][j], x[i][j], s1[0]);
            }
            if (p.gate) st_row<T, N, LANES, VEC>(p.dgate, at.row, E, i, at.lane, dg);
            if (p.dresidual) st_row<S, N, LANES, VEC>(p.dresidual, at.row, E, i, at.lane, t[i]);
        }
        float back = 0.f;
        if (p.post_norm) { sum1(s1); back = s1[0] * p.inv_e; }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float d[N];
#pragma unroll
            for (int j = 0; j < N; ++j) d[j] = p.post_norm ? inv * (m[i][j] - x[i][j] * back) : m[i][j];
            st_row<T, N, LANES, VEC>(p.dx, at.row, E, i, at.lane, d);
        }
    }
    // rows that a workgroup has side by side: their sums meet in LDS
    float* const to = p.part + (long long)blockIdx.x * 3 * p.E;
    const int mine = threadIdx.x / LANES;
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        if constexpr (ROWS > 1) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < N; ++j)
                    if (mine) meet[((mine - 1) * NV * N + i * N + j) * LANES + at.lane] = acc[k][i][j];
            __syncthreads();
            if (mine) continue;
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < N; ++j)
#pragma unroll
                    for (int o = 0; o < ROWS - 1; ++o) acc[k][i][j] += meet[(o * NV * N + i * N + j) * LANES + at.lane];
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const int e = channel<N, LANES, VEC>(i, j, at.lane);
                if (e < p.E) to[k * p.E + e] = acc[k][i][j];
            }
        }
    }
}

constexpr int BLOCK_NORM_MOST = 4096;     // a row lies in the registers of eight waves at the most
struct BlockNormCfg { int nv, waves; bool vec; long long wgs; };
constexpr long long BLOCK_NORM_WGS = 2048, BLOCK_NORM_GRAD_WGS = 768;
static int block_norm_config(const hdla_block_norm_dims* d, bool bwd, BlockNormCfg& c, const void* weight = nullptr, const void* post = nullptr, const void* scale = nullptr) {
    if (!d) return HDLA_ERR_NULL;
    for (int t : {d->dtype, d->residual_dtype, d->weight_dtype, d->post_dtype, d->scale_dtype})
        if (t != HDLA_BF16 && t != HDLA_FP32) return HDLA_ERR_DTYPE;
    if (d->dtype == HDLA_FP32 && d->residual_dtype != HDLA_FP32) return HDLA_ERR_DTYPE;
    if (d->rows < 0 || d->rows > (1LL << 40) || d->E < 1 || !(d->eps >= 0.f) || d->act < ACT_NONE || d->act > ACT_SILU) return HDLA_ERR_SHAPE;
    if (d->E > BLOCK_NORM_MOST) return HDLA_ERR_SHAPE;
    const int n = d->dtype == HDLA_BF16 ? 8 : 4, pieces = (d->E + n - 1) / n;
    // one piece a lane, up to 512 lanes; two pieces of half as many lanes are alike (8192 x 4096 in bf16, forward and backward 205 us; so 201)
    c.waves = pieces <= 64 ? 1 : pieces <= 128 ? 2 : pieces <= 256 || (pieces <= 512 && n == 4) ? 4 : 8;
    c.nv = pieces > 64 * c.waves ? 2 : 1;
    const long long per = c.waves >= 4 ? 1 : 4 / c.waves, need = (d->rows + per - 1) / per, most = bwd ? BLOCK_NORM_GRAD_WGS : BLOCK_NORM_WGS;
    // as many as are resident, with as many rows each as the others.  us, forward and backward, of 512 / 768 / 1024 workgroups backward (forward 1024, 2048 and 4096 are alike):
    // 8192 x 2048 in bf16 107 / 96 / 106, 16384 x 1024 103 / 87 / 92, 16384 x 4096 491 / 490 / 487
    const long long turns = (need + most - 1) / most;
    c.wgs = std::max(1LL, turns ? (need + turns - 1) / turns : 1);
    c.vec = d->E % n == 0;
    for (const void* q : {weight, post, scale}) c.vec = c.vec && fits(q, 16);
    return HDLA_OK;
}
static BlockNormArgs block_norm_args(const hdla_block_norm_dims* d) {
    BlockNormArgs a{};
    a.rows = d->rows; a.E = d->E; a.act = d->act; a.post_norm = d->post_norm != 0;
    a.w_f32 = d->weight_dtype == HDLA_FP32; a.p_f32 = d->post_dtype == HDLA_FP32; a.s_f32 = d->scale_dtype == HDLA_FP32;
    a.factor = d->factor; a.inv_e = 1.f / (float)d->E; a.eps = d->eps;
    return a;
}
template <typename T, typename S, int NV, int WAVES> static void launch_norm_of(const BlockNormArgs& a, const BlockNormCfg& c, bool bwd, hipStream_t s) {
    const dim3 grid((unsigned)c.wgs), block(RowShare<WAVES>::THREADS);
    if (bwd) {
        if (c.vec) hipLaunchKernelGGL((block_norm_grad_kernel<T, S, NV, WAVES, true>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((block_norm_grad_kernel<T, S, NV, WAVES, false>), grid, block, 0, s, a);
    } else {
        if (c.vec) hipLaunchKernelGGL((block_norm_kernel<T, S, NV, WAVES, true>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((block_norm_kernel<T, S, NV, WAVES, false>), grid, block, 0, s, a);
    }
}
template <typename T, typename S> static hipError_t launch_block_norm(const BlockNormArgs& a, const BlockNormCfg& c, bool bwd, hipStream_t s) {
    constexpr int WIDE = sizeof(T) == 4 ? 2 : 1;          // pieces of the widest rows
    if (c.waves == 1) launch_norm_of<T, S, 1, 1>(a, c, bwd, s);
    else if (c.waves == 2) launch_norm_of<T, S, 1, 2>(a, c, bwd, s);
    else if (c.waves == 4 && c.nv == 1) launch_norm_of<T, S, 1, 4>(a, c, bwd, s);
    else if (c.waves == 4) launch_norm_of<T, S, WIDE, 4>(a, c, bwd, s);
    else launch_norm_of<T, S, WIDE, 8>(a, c, bwd, s);
    return hipGetLastError();
}
static hipError_t launch_any(const hdla_block_norm_dims* d, const BlockNormArgs& a, const BlockNormCfg& c, bool bwd, hipStream_t s) {
    if (d->dtype == HDLA_FP32) return launch_block_norm<float, float>(a, c, bwd, s);
    return d->residual_dtype == HDLA_FP32 ? launch_block_norm<bf16, float>(a, c, bwd, s) : launch_block_norm<bf16, bf16>(a, c, bwd, s);
}

}  // namespace hdla

using namespace hdla;

extern "C" int hdla_block_norm_fwd(const hdla_block_norm_dims* dims, const void* x, const void* residual, const void* weight, const void* post_weight, const void* gate,
                                   const void* scale, void* y, void* r, void* stream) {
    BlockNormCfg c;
    const int rc = block_norm_config(dims, false, c, weight, post_weight, scale);
    if (rc) return rc;
    if (dims->rows == 0) return HDLA_OK;
    if (!x || !y || !r) return HDLA_ERR_NULL;
    for (const void* q : {x, residual, gate, (const void*)y, (const void*)r})
        if (!fits(q, 16)) return HDLA_ERR_ALIGN;
    BlockNormArgs a = block_norm_args(dims);
    a.x = x; a.residual = residual; a.weight = weight; a.post = post_weight; a.gate = gate; a.scale = scale; a.y = y; a.r = r;
    const hipError_t e = launch_any(dims, a, c, false, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? HDLA_OK : (int)e;
}
extern "C" size_t hdla_block_norm_workspace_bytes(const hdla_block_norm_dims* dims) {
    BlockNormCfg c;
    return block_norm_config(dims, true, c) ? 0 : (size_t)c.wgs * 3 * dims->E * 4;
}
extern "C" int hdla_block_norm_bwd(const hdla_block_norm_dims* dims, const void* x, const void* residual, const void* weight, const void* post_weight, const void* gate,
                                   const void* scale, const void* dy, const void* dr, void* dx, void* dresidual, void* dweight, void* dpost_weight, void* dgate,
                                   void* dscale, void* workspace, size_t workspace_bytes, void* stream) {
    BlockNormCfg c;
    const int rc = block_norm_config(dims, true, c, weight, post_weight, scale);
    if (rc) return rc;
    if ((weight && !dweight) || (post_weight && !dpost_weight) || (scale && !dscale)) return HDLA_ERR_NULL;
    if (dims->rows > 0 && (!x || !dx || (gate && !dgate))) return HDLA_ERR_NULL;
    for (const void* q : {x, residual, gate, dy, dr, (const void*)dx, (const void*)dresidual, (const void*)dgate})
        if (!fits(q, 16)) return HDLA_ERR_ALIGN;
    if (!workspace || !fits(workspace, 16) || workspace_bytes < hdla_block_norm_workspace_bytes(dims)) return HDLA_ERR_WORKSPACE;
    BlockNormArgs a = block_norm_args(dims);
    a.x = x; a.residual = residual; a.weight = weight; a.post = post_weight; a.gate = gate; a.scale = scale; a.dy = dy; a.dr = dr;
    a.dx = dx; a.dresidual = dresidual; a.dgate = dgate;
    a.part = static_cast<float*>(workspace);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    hipError_t e = launch_any(dims, a, c, true, s);       // (no rows: one workgroup leaves zeros)
    if (e != hipSuccess) return (int)e;
    if (!weight && !post_weight && !scale) return HDLA_OK;
    ColumnSums k{};
    k.part = a.part; k.rows = c.wgs;
    k.add(weight ? dweight : nullptr, a.w_f32, dims->E);
    k.add(post_weight ? dpost_weight : nullptr, a.p_f32, dims->E);
    k.add(scale ? dscale : nullptr, a.s_f32, dims->E);
    e = launch_column_sums(k, s);
    return e == hipSuccess ? HDLA_OK : (int)e;
}
