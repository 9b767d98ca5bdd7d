// The norms around a block, with its gate and the residual stream: what the block gave, normalised (or not), gated and scaled, is added to the stream, and the sum is
// normalised for the next block.  Per row of E channels:
//     p = x / rms(x) post_weight  (or x);   u = p act(gate)  (or p);   r = residual + scale u;   y = r / rms(r) weight;   rms(v) = sqrt(mean v^2 + eps)
// Backward, from dy and dr (rhat = r / rms(r), xhat = x / rms(x)), with everything formed again from the inputs:
//     m = dy weight;  dr += (m - rhat mean(m rhat)) / rms(r);   dresidual = dr;   dweight = sum dy rhat;   dscale = sum dr u;   du = scale dr;
//     dgate = du p act'(gate);   dp = du act(gate);   dpost_weight = sum dp xhat;   q = dp post_weight;  dx = (q - xhat mean(q xhat)) / rms(x)
//
// Streams through HBM: forward reads x, gate, residual and writes y, r; backward reads these, dy, dr and writes dx, dgate, dresidual.  A row lies in the registers
// of one wave, or of the four waves of a workgroup where it is long, 16 bytes a lane and piece; its sums are taken across lanes without LDS (a workgroup's four through it).
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

// N channels from e on; beyond the row's end (it need not be a multiple of N where VEC is false) zeros
template <typename T, int N, bool VEC> __device__ __forceinline__ void ld_row(const void* base, long long row, int E, int e, float (&f)[N]) {
    Raw<T, N, VEC> r;
    r.clear();
    if (e < E) r.load(static_cast<const T*>(base) + row * E + e, E - e);
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = r[i];
}
template <int N, bool VEC> __device__ __forceinline__ void ld_vector(const void* v, int f32, int E, int e, float none, float (&f)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = v && e + i < E ? ld_param(v, f32, e + i) : none;
}
template <typename T, int N, bool VEC> __device__ __forceinline__ void st_row(void* base, long long row, int E, int e, const float (&f)[N]) {
    if (e < E) st_values<T, N, VEC>(static_cast<T*>(base) + row * E + e, f, E - e);
}
// act(g) and its derivative
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
        da[i] = act == ACT_SILU ? s[i] * __builtin_fmaf(g[i], 1.f - s[i], 1.f) : s[i] * (1.f - s[i]);
    }
}

// Sums over a row: the lanes of a wave, or (WAVES = 4) of a workgroup, whose threads all make the same calls; alternating halves of LDS, so one barrier a call
template <int WAVES, int N> struct RowSum {
    float* lds;
    int half = 0;
    __device__ __forceinline__ void operator()(float (&x)[N]) {
        sum_lanes<N>(x, 64);
        if constexpr (WAVES > 1) {
            float* const s = lds + half * WAVES * N;
            if ((threadIdx.x & 63) == 0)
#pragma unroll
                for (int i = 0; i < N; ++i) s[(threadIdx.x >> 6) * N + i] = x[i];
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

// x and gate of T, residual, r of S.  NV pieces of N channels a lane; WAVES waves a row
template <typename T, typename S, int NV, int WAVES, bool VEC>
__global__ __launch_bounds__(WAVES == 8 ? 512 : 256) void block_norm_kernel(BlockNormArgs p) {
    constexpr int N = 16 / sizeof(T), LANES = 64 * WAVES, ROWS = WAVES == 1 ? 4 : 1;
    __shared__ float lds[2 * WAVES];
    RowSum<WAVES, 1> sum{lds};
    const int lane = threadIdx.x % LANES;
    float w[NV][N], pw[NV][N], sc[NV][N];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int e = (i * LANES + lane) * N;
        ld_vector<N, VEC>(p.weight, p.w_f32, p.E, e, 1.f, w[i]);
        ld_vector<N, VEC>(p.post, p.p_f32, p.E, e, 1.f, pw[i]);
        ld_vector<N, VEC>(p.scale, p.s_f32, p.E, e, p.factor, sc[i]);
    }
    for (long long first = (long long)blockIdx.x * ROWS; first < p.rows; first += (long long)gridDim.x * ROWS) {
        const long long row = first + threadIdx.x / LANES;
        const bool live = row < p.rows;
        const int E = live ? p.E : 0;
        float x[NV][N], r[NV][N], g[NV][N];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int e = (i * LANES + lane) * N;
            ld_row<T, N, VEC>(p.x, row, E, e, x[i]);
            if (p.residual) ld_row<S, N, VEC>(p.residual, row, E, e, r[i]);
            if (p.gate) ld_row<T, N, VEC>(p.gate, row, E, e, g[i]);
        }
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
                u *= sc[i][j];
                r[i][j] = p.residual ? r[i][j] + u : u;
                s[0] = __builtin_fmaf(r[i][j], r[i][j], s[0]);
            }
        }
        sum(s);
        const float ir = 1.f / sqrtf(__builtin_fmaf(s[0], p.inv_e, p.eps));
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int e = (i * LANES + lane) * N;
            float y[N];
#pragma unroll
            for (int j = 0; j < N; ++j) y[j] = r[i][j] * ir * w[i][j];
            st_row<T, N, VEC>(p.y, row, E, e, y);
            st_row<S, N, VEC>(p.r, row, E, e, r[i]);
        }
    }
}

// (four channels a lane and piece: their sums' registers are three times theirs. )
template <typename T, typename S, int NV, int WAVES, bool VEC>
__global__ __launch_bounds__(WAVES == 8 ? 512 : 256) void block_norm_grad_kernel(BlockNormArgs p) {
    constexpr int N = 4, LANES = 64 * WAVES, ROWS = WAVES == 1 ? 4 : 1;
    __shared__ float lds[2 * WAVES * 2], lds1[2 * WAVES];
    __shared__ f32x4 meet[WAVES == 1 ? 3 * NV * 64 : 1];
    RowSum<WAVES, 1> sum1{lds1};
    RowSum<WAVES, 2> sum2{lds};
    const int lane = threadIdx.x % LANES;
    f32x4 acc[3][NV];
#pragma unroll
    for (int k = 0; k < 3; ++k)
#pragma unroll
        for (int i = 0; i < NV; ++i) acc[k][i] = zero4();
    for (long long first = (long long)blockIdx.x * ROWS; first < p.rows; first += (long long)gridDim.x * ROWS) {
        const long long row = first + threadIdx.x / LANES;
        const bool live = row < p.rows;
        const int E = live ? p.E : 0;
        float x[NV][N], r[NV][N], m[NV][N], t[NV][N];    // xhat; r, then rhat; dy; the gradient of r
        float inv = 1.f, s1[1] = {0.f};
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int e = (i * LANES + lane) * N;
            ld_row<T, N, VEC>(p.x, row, E, e, x[i]);
            if (p.residual) ld_row<S, N, VEC>(p.residual, row, E, e, r[i]);
            else
#pragma unroll
                for (int j = 0; j < N; ++j) r[i][j] = 0.f;
            if (p.dy) ld_row<T, N, VEC>(p.dy, row, E, e, m[i]);
            else
#pragma unroll
                for (int j = 0; j < N; ++j) m[i][j] = 0.f;
            if (p.dr) ld_row<S, N, VEC>(p.dr, row, E, e, t[i]);
            else
#pragma unroll
                for (int j = 0; j < N; ++j) t[i][j] = 0.f;
#pragma unroll
            for (int j = 0; j < N; ++j) s1[0] = __builtin_fmaf(x[i][j], x[i][j], s1[0]);
        }
        if (p.post_norm) {
            sum1(s1);
            inv = 1.f / sqrtf(__builtin_fmaf(s1[0], p.inv_e, p.eps));
        }
        float s2[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int e = (i * LANES + lane) * N;
            float w[N], pw[N], sc[N], g[N], a[N], da[N];
            ld_vector<N, VEC>(p.weight, p.w_f32, p.E, e, 1.f, w);
            ld_vector<N, VEC>(p.post, p.p_f32, p.E, e, 1.f, pw);
            ld_vector<N, VEC>(p.scale, p.s_f32, p.E, e, p.factor, sc);
            if (p.gate) { ld_row<T, N, VEC>(p.gate, row, E, e, g); activate<T, N>(p.act, g, a, da); }
#pragma unroll
            for (int j = 0; j < N; ++j) {
                x[i][j] *= inv;
                float u = x[i][j] * pw[j];
                if (p.gate) u *= a[j];
                r[i][j] = __builtin_fmaf(sc[j], u, r[i][j]);
                s2[0] = __builtin_fmaf(r[i][j], r[i][j], s2[0]);
                s2[1] = __builtin_fmaf(m[i][j] * w[j], r[i][j], s2[1]);
            }
        }
        sum2(s2);
        const float ir = 1.f / sqrtf(__builtin_fmaf(s2[0], p.inv_e, p.eps)), along = s2[1] * ir * p.inv_e;
        s1[0] = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int e = (i * LANES + lane) * N;
            float w[N], pw[N], sc[N], g[N], a[N], da[N], dg[N];
            ld_vector<N, VEC>(p.weight, p.w_f32, p.E, e, 1.f, w);
            ld_vector<N, VEC>(p.post, p.p_f32, p.E, e, 1.f, pw);
            ld_vector<N, VEC>(p.scale, p.s_f32, p.E, e, p.factor, sc);
            if (p.gate) { ld_row<T, N, VEC>(p.gate, row, E, e, g); activate<T, N>(p.act, g, a, da); }
            f32x4 dw = acc[0][i], dp = acc[1][i], ds = acc[2][i];
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const float rh = r[i][j] * ir;
                t[i][j] = __builtin_fmaf(ir, m[i][j] * w[j] - rh * along, t[i][j]);
                dw[j] = __builtin_fmaf(m[i][j], rh, dw[j]);
                const float pv = x[i][j] * pw[j];
                ds[j] = __builtin_fmaf(t[i][j], p.gate ? pv * a[j] : pv, ds[j]);
                float du = t[i][j] * sc[j];
                if (p.gate) { dg[j] = du * pv * da[j]; du *= a[j]; }
                dp[j] = __builtin_fmaf(du, x[i][j], dp[j]);
                m[i][j] = du * pw[j];
                s1[0] = __builtin_fmaf(m[i][j], x[i][j], s1[0]);
            }
            acc[0][i] = dw; acc[1][i] = dp; acc[2][i] = ds;
            if (p.gate) st_row<T, N, VEC>(p.dgate, row, E, e, dg);
            if (p.dresidual) st_row<S, N, VEC>(p.dresidual, row, E, e, t[i]);
        }
        float back = 0.f;
        if (p.post_norm) { sum1(s1); back = s1[0] * p.inv_e; }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int e = (i * LANES + lane) * N;
            float d[N];
#pragma unroll
            for (int j = 0; j < N; ++j) d[j] = p.post_norm ? inv * (m[i][j] - x[i][j] * back) : m[i][j];
            st_row<T, N, VEC>(p.dx, row, E, e, d);
        }
    }
    float* const to = p.part + (long long)blockIdx.x * 3 * p.E;
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        if constexpr (WAVES == 1) {                       // the four waves hold the same channels
            const int wave = threadIdx.x >> 6;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (wave) meet[((wave - 1) * NV + i) * 64 + lane] = acc[k][i];
            __syncthreads();
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (!wave) acc[k][i] += (meet[i * 64 + lane] + meet[(NV + i) * 64 + lane]) + meet[(2 * NV + i) * 64 + lane];
            if (wave) continue;
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int e = (i * LANES + lane) * N;
            const f32x4 v = acc[k][i];
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (e + j < p.E) to[k * p.E + e + j] = v[j];
        }
    }
}

constexpr int BLOCK_NORM_MOST = 4096;     // a row lies in the registers of eight waves at the most
struct BlockNormCfg { int nv, waves; bool vec; long long wgs; };
static int block_norm_config(const hdla_block_norm_dims* d, bool bwd, BlockNormCfg& c) {
    if (!d) return HDLA_ERR_NULL;
    for (int t : {d->dtype, d->residual_dtype, d->weight_dtype, d->post_dtype, d->scale_dtype})
        if (t != HDLA_BF16 && t != HDLA_FP32) return HDLA_ERR_DTYPE;
    if (d->dtype == HDLA_FP32 && d->residual_dtype != HDLA_FP32) return HDLA_ERR_DTYPE;
    if (d->rows < 0 || d->rows > (1LL << 40) || d->E < 1 || !(d->eps >= 0.f) || d->act < ACT_NONE || d->act > ACT_SILU) return HDLA_ERR_SHAPE;
    if (d->E > BLOCK_NORM_MOST) return HDLA_ERR_SHAPE;
    const int n = bwd || d->dtype == HDLA_FP32 ? 4 : 8, pieces = (d->E + n - 1) / n;
    c.waves = pieces <= 64 ? 1 : pieces <= 512 ? 4 : 8;
    c.nv = 1;
    while (c.nv * 64 * c.waves < pieces) c.nv *= 2;
    const long long per = c.waves == 1 ? 4 : 1, need = (d->rows + per - 1) / per;
    c.wgs = std::max(1LL, std::min(need, bwd ? 1024LL : 4096LL));
    c.vec = d->E % n == 0;
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
    const dim3 grid((unsigned)c.wgs), block(WAVES == 8 ? 512 : 256);
    if (bwd) {
        if (c.vec) hipLaunchKernelGGL((block_norm_grad_kernel<T, S, NV, WAVES, true>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((block_norm_grad_kernel<T, S, NV, WAVES, false>), grid, block, 0, s, a);
    } else {
        if (c.vec) hipLaunchKernelGGL((block_norm_kernel<T, S, NV, WAVES, true>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((block_norm_kernel<T, S, NV, WAVES, false>), grid, block, 0, s, a);
    }
}
template <typename T, typename S> static hipError_t launch_block_norm(const BlockNormArgs& a, const BlockNormCfg& c, bool bwd, hipStream_t s) {
    if (c.waves == 1) launch_norm_of<T, S, 1, 1>(a, c, bwd, s);
    else if (c.waves == 4 && c.nv == 1) launch_norm_of<T, S, 1, 4>(a, c, bwd, s);
    else if (c.waves == 4) launch_norm_of<T, S, 2, 4>(a, c, bwd, s);
    else launch_norm_of<T, S, 2, 8>(a, c, bwd, s);
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
    const int rc = block_norm_config(dims, false, c);
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
    const int rc = block_norm_config(dims, true, c);
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
    const struct { void* out; bool f32; } sums[3] = {{weight ? dweight : nullptr, a.w_f32 != 0}, {post_weight ? dpost_weight : nullptr, a.p_f32 != 0}, {scale ? dscale : nullptr, a.s_f32 != 0}};
    for (int i = 0; i < 3; ++i) {
        if (!sums[i].out) continue;
        ColumnSums k{};
        k.part = a.part + (long long)i * dims->E; k.rows = c.wgs;
        k.add(sums[i].out, sums[i].f32, dims->E);
        k.apart = 3LL * dims->E;
        e = launch_column_sums(k, s);
        if (e != hipSuccess) return (int)e;
    }
    return HDLA_OK;
}
