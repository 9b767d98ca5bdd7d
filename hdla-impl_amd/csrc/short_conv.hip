// Short causal convolution over the tokens of each channel, W taps (2, 3 or 4), optionally followed by silu:
//     p_t = bias + sum_j w_j x_{t-W+1+j};   y_t = p_t or p_t sigmoid(p_t)
// where x before a sequence's first token is its state (the W - 1 inputs before it), or zero.  Backward, with g_t = dy_t act'(p_t):
//     dx_t = sum_j w_{W-1-j} g_{t+j} (+ what reaches x_t through the final state);   dw_j = sum_t g_t x_{t-W+1+j};   dbias = sum_t g_t
//
// Streams through HBM (forward: read x, write y; backward: read x, dy, write dx).  A thread owns V neighbouring channels of a run of consecutive tokens:
// its taps come from registers, and x is read again only where runs meet.  16384 x 4096 in bf16, 4 taps with silu: forward 50 us, 5.4 TB/s, what a large
// copy reaches.  8192 x 2048: forward 20 us, backward 32 us and 4 us for the sums of dw and dbias.
#include "column_sums.cuh"
#include "hdla_common.cuh"
#include "state_space.cuh"

#include <algorithm>

namespace hdla {

struct ConvArgs {
    Operand x;
    const void *weight, *bias, *state, *dy, *dlast;      // state, dlast [N, W-1, D]
    void *y, *last, *dx, *dstate;
    float* part;                                         // [rows of partial sums][D * W + D]
    const int64_t* cu;
    int T, N, D, w_f32, b_f32, silu;
    int cols, runs;                                      // column groups of V channels; runs of tokens a sequence (packed: of all tokens)
    long long threads;                                   // of the runs; those behind them take the states
};

// V channels of W taps, [V][W] as they lie
template <int W, int V> __device__ __forceinline__ void ld_taps(const void* w, int f32, long long at, float (&t)[V][W]) {
    constexpr int N = V * W;
    if constexpr (V > 1) {
        if (f32) {
#pragma unroll
            for (int i = 0; i < N; i += 4) {
                const f32x4 r = *reinterpret_cast<const f32x4*>(static_cast<const float*>(w) + at + i);
#pragma unroll
                for (int j = 0; j < 4; ++j) t[(i + j) / W][(i + j) % W] = r[j];
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; i += 4) {
                const f32x4 r = to_f32(ld_frag(static_cast<const bf16*>(w) + at + i));
#pragma unroll
                for (int j = 0; j < 4; ++j) t[(i + j) / W][(i + j) % W] = r[j];
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) t[i / W][i % W] = ld_param(w, f32, at + i);
    }
}

// The sequence that a token of a packed batch belongs to; tokens of none have len 0
struct Where {
    int n;
    int64_t bos, eos;
    __device__ __forceinline__ void find(const ConvArgs& p, int64_t t) {
        // as many sequences as end at or before t, by halves
        int lo = 0, hi = p.N;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (p.cu[mid + 1] <= t) lo = mid + 1;
            else hi = mid;
        }
        n = lo;
        bounds(p, t);
    }
    __device__ __forceinline__ void bounds(const ConvArgs& p, int64_t t) {
        if (n < p.N) packed_bounds(p.cu, n, p.T, bos, eos);
        if (n >= p.N || t < bos || t >= eos) { bos = t + 1; eos = t + 1; }     // (of none)
    }
    __device__ __forceinline__ void next(const ConvArgs& p, int64_t t) {
        while (n < p.N && p.cu[n + 1] <= t) ++n;
        bounds(p, t);
    }
};

template <typename T, int W, int V> struct ConvRow {
    // V elements of row i (from its first token, negative: of its state) of sequence n
    static __device__ __forceinline__ Raw<T, V, (V > 1)> get(const ConvArgs& p, int n, int64_t bos, int64_t i, int col) {
        Raw<T, V, (V > 1)> r;
        r.clear();
        if (i >= 0) {
            const long long batch = p.cu ? 0 : n;
            r.load(static_cast<const T*>(p.x.p) + batch * p.x.batch + (bos + i) * p.x.row + col, V);
        } else if (p.state && i >= -(W - 1)) {
            r.load(static_cast<const T*>(p.state) + ((long long)n * (W - 1) + (W - 1 + i)) * p.D + col, V);
        }
        return r;
    }
};

// A thread behind the runs': one row of a final state
template <typename T, int W, int V> __device__ __forceinline__ void conv_last(const ConvArgs& p, long long at) {
    const int col = (int)(at % p.cols) * V;
    const long long r = at / p.cols;
    const int i = (int)(r % (W - 1));
    const long long n = r / (W - 1);
    if (n >= p.N) return;
    int64_t bos = 0, eos = p.T;
    if (p.cu) packed_bounds(p.cu, (int)n, p.T, bos, eos);
    const Raw<T, V, (V > 1)> x = ConvRow<T, W, V>::get(p, (int)n, bos, eos - bos - (W - 1) + i, col);
    float f[V];
#pragma unroll
    for (int k = 0; k < V; ++k) f[k] = x[k];
    st_values<T, V, (V > 1)>(static_cast<T*>(p.last) + (n * (W - 1) + i) * p.D + col, f, V);
}

// The taps of tokens: rows of x as they come from memory, `before` the W - 1 in front of those in `now`
template <int W, int STEP, typename R> __device__ __forceinline__ const R& tap(const R (&before)[W - 1], const R (&now)[STEP], int i) {
    return i < W - 1 ? before[i < W - 1 ? i : 0] : now[i >= W - 1 ? i - (W - 1) : 0];
}
template <typename T, int W, int V, int STEP, bool PACKED>
__global__ __launch_bounds__(256) void short_conv_kernel(ConvArgs p, int steps) {
    using R = Raw<T, V, (V > 1)>;
    const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
    if (id >= p.threads) { if (p.last) conv_last<T, W, V>(p, id - p.threads); return; }
    const int col = (int)(id % p.cols) * V;
    const long long r = id / p.cols;
    const int n = PACKED ? 0 : (int)(r / p.runs);
    int64_t t0 = (r - (long long)n * p.runs) * steps * STEP;
    // (rows behind the last, asked for with a step of others, are the last one once more)
    const T* const x0 = static_cast<const T*>(p.x.p) + n * p.x.batch + col;
    auto row = [&](int64_t t, R& to) __attribute__((always_inline)) { to.load(x0 + min(t, (int64_t)p.T - 1) * p.x.row, V); };
    R before[W - 1], now[STEP], next[STEP];
#pragma unroll
    for (int i = 0; i < STEP; ++i) row(t0 + i, now[i]);
    float w[V][W], b[V];
    ld_taps<W, V>(p.weight, p.w_f32, (long long)col * W, w);
#pragma unroll
    for (int k = 0; k < V; ++k) b[k] = p.bias ? ld_param(p.bias, p.b_f32, col + k) : 0.f;
    // (before a packed batch's first token nothing is read: these rows are of another sequence, or of none)
#pragma unroll
    for (int i = 0; i < W - 1; ++i) {
        const int64_t t = t0 - (W - 1) + i;
        before[i] = PACKED ? ConvRow<T, W, V>::get(p, 0, 0, max(t, (int64_t)0), col) : ConvRow<T, W, V>::get(p, n, 0, t, col);
    }
    Where s{n, 0, p.T};
    if (PACKED) s.find(p, t0);
    T* y = static_cast<T*>(p.y) + ((long long)n * p.T + t0) * p.D + col;
    for (int step = 0; step < steps && t0 < p.T; ++step, t0 += STEP) {
        if (step + 1 < steps) {
#pragma unroll
            for (int i = 0; i < STEP; ++i) row(t0 + STEP + i, next[i]);
        }
#pragma unroll
        for (int i = 0; i < STEP; ++i) {
            const int64_t t = t0 + i;
            if (t < p.T) {
                float f[V];
#pragma unroll
                for (int k = 0; k < V; ++k) f[k] = b[k];
                bool none = false, early = false;
                if (PACKED) {
                    if (t >= s.eos) s.next(p, t);
                    none = t < s.bos;
                    early = t - s.bos < W - 1;
                }
                if (!early) {
#pragma unroll
                    for (int j = 0; j < W; ++j)
#pragma unroll
                        for (int k = 0; k < V; ++k) f[k] = __builtin_fmaf(w[k][j], tap<W, STEP>(before, now, i + j)[k], f[k]);
                } else if (!none) {
#pragma unroll
                    for (int j = 0; j < W; ++j) {
                        const R e = ConvRow<T, W, V>::get(p, s.n, s.bos, t - s.bos - (W - 1) + j, col);
#pragma unroll
                        for (int k = 0; k < V; ++k) f[k] = __builtin_fmaf(w[k][j], e[k], f[k]);
                    }
                }
                if (p.silu) {
                    float g[V];
                    sigmoid_each<T, V>(f, g);
#pragma unroll
                    for (int k = 0; k < V; ++k) f[k] *= g[k];
                }
                if (none) {
#pragma unroll
                    for (int k = 0; k < V; ++k) f[k] = 0.f;
                }
                st_values<T, V, (V > 1)>(y, f, V);
            }
            y += p.D;
        }
#pragma unroll
        for (int i = 0; i < W - 1; ++i) before[i] = now[STEP - (W - 1) + i];
#pragma unroll
        for (int i = 0; i < STEP; ++i) now[i] = next[i];
    }
}

// g of token i of sequence n (its pre-activation once more from its taps); zero behind the sequence
template <typename T, int W, int V>
__device__ __forceinline__ void conv_g(const ConvArgs& p, const float (&w)[V][W], const float (&b)[V], const float (&x)[W][V], const Raw<T, V, (V > 1)>& dy, float (&g)[V]) {
#pragma unroll
    for (int k = 0; k < V; ++k) g[k] = dy[k];
    if (p.silu) {
        float f[V], s[V];
#pragma unroll
        for (int k = 0; k < V; ++k) {
            f[k] = b[k];
#pragma unroll
            for (int j = 0; j < W; ++j) f[k] = __builtin_fmaf(w[k][j], x[j][k], f[k]);
        }
        sigmoid_each<T, V>(f, s);
#pragma unroll
        for (int k = 0; k < V; ++k) g[k] *= s[k] * __builtin_fmaf(f[k], 1.f - s[k], 1.f);
    }
}

// A thread behind the runs': one row of an initial state's gradient, row i being W - 1 - i tokens before the sequence
template <typename T, int W, int V> __device__ __forceinline__ void conv_dstate(const ConvArgs& p, long long at) {
    const int col = (int)(at % p.cols) * V;
    const long long r = at / p.cols;
    const int i = (int)(r % (W - 1));
    const long long n = r / (W - 1);
    if (n >= p.N) return;
    int64_t bos = 0, eos = p.T;
    if (p.cu) packed_bounds(p.cu, (int)n, p.T, bos, eos);
    const int64_t len = eos - bos, row0 = p.cu ? bos : n * p.T;
    float w[V][W], b[V], d[V];
    ld_taps<W, V>(p.weight, p.w_f32, (long long)col * W, w);
#pragma unroll
    for (int k = 0; k < V; ++k) { b[k] = p.bias ? ld_param(p.bias, p.b_f32, col + k) : 0.f; d[k] = 0.f; }
    // token t's tap j meets row t + j of [state, tokens]
#pragma unroll
    for (int t = 0; t < W - 1; ++t) {
        if (t < len && t <= i) {
            float x[W][V], g[V];
#pragma unroll
            for (int j = 0; j < W; ++j) {
                const Raw<T, V, (V > 1)> e = ConvRow<T, W, V>::get(p, (int)n, bos, t - (W - 1) + j, col);
#pragma unroll
                for (int k = 0; k < V; ++k) x[j][k] = e[k];
            }
            Raw<T, V, (V > 1)> dy;
            dy.load(static_cast<const T*>(p.dy) + (row0 + t) * p.D + col, V);
            conv_g<T, W, V>(p, w, b, x, dy, g);
#pragma unroll
            for (int j = 0; j < W; ++j)
                if (j == i - t)
#pragma unroll
                    for (int k = 0; k < V; ++k) d[k] = __builtin_fmaf(w[k][j], g[k], d[k]);
        }
    }
    if (p.dlast && i >= len) {                            // a sequence of fewer tokens hands its state's later rows on
        Raw<T, V, (V > 1)> e;
        e.load(static_cast<const T*>(p.dlast) + (n * (W - 1) + (i - len)) * p.D + col, V);
#pragma unroll
        for (int k = 0; k < V; ++k) d[k] += e[k];
    }
    st_values<T, V, (V > 1)>(static_cast<T*>(p.dstate) + (n * (W - 1) + i) * p.D + col, d, V);
}

// A workgroup is 64 columns (fewer where there are fewer) x 4 runs of steps x STEP tokens: their sums of dw and dbias meet in LDS.  A run walks its tokens and the
// W - 1 behind them: g_t from its taps, then dx_{t-W+1}, which by then has all the g that it needs.
template <typename T, int W, int V, int STEP, bool PACKED>
__global__ __launch_bounds__(256) void short_conv_grad_kernel(ConvArgs p, int steps, long long col_blocks, long long row_blocks) {
    using R = Raw<T, V, (V > 1)>;
    __shared__ float red[3][V * (W + 1)][64];
    if (blockIdx.x >= col_blocks * row_blocks) {
        if (p.dstate) conv_dstate<T, W, V>(p, (blockIdx.x - col_blocks * row_blocks) * 256 + threadIdx.x);
        return;
    }
    const int c = (int)(blockIdx.x % col_blocks) * 64 + (threadIdx.x & 63), wave = threadIdx.x >> 6;
    const long long r = blockIdx.x / col_blocks * 4 + wave;
    const int col = c * V, n = PACKED ? 0 : (int)(r / p.runs);
    const int64_t first = (r - (long long)n * p.runs) * steps * STEP;
    const bool live = c < p.cols && r < (long long)(PACKED ? 1 : p.N) * p.runs && first < p.T;
    float dw[V][W], db[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
        db[k] = 0.f;
#pragma unroll
        for (int j = 0; j < W; ++j) dw[k][j] = 0.f;
    }
    if (live) {
        const int64_t end = min(first + (int64_t)steps * STEP, (int64_t)p.T);          // of this run's own tokens
        const T *const x0 = static_cast<const T*>(p.x.p) + n * p.x.batch + col, *const dy0 = static_cast<const T*>(p.dy) + (long long)n * p.T * p.D + col;
        T* const dx0 = static_cast<T*>(p.dx) + (long long)n * p.T * p.D + col;
        // (rows behind the last, asked for with a step of others, are the last one once more)
        auto rows = [&](int64_t t, R& x, R& dy) __attribute__((always_inline)) {
            const int64_t at = min(t, (int64_t)p.T - 1);
            x.load(x0 + at * p.x.row, V);
            dy.load(dy0 + at * p.D, V);
        };
        R before[W - 1], x[STEP], dy[STEP], xn[STEP], dyn[STEP];
#pragma unroll
        for (int i = 0; i < STEP; ++i) rows(first + i, x[i], dy[i]);
        float w[V][W], b[V], ring[W][V];                  // ring: g of the last W tokens
        ld_taps<W, V>(p.weight, p.w_f32, (long long)col * W, w);
#pragma unroll
        for (int k = 0; k < V; ++k) {
            b[k] = p.bias ? ld_param(p.bias, p.b_f32, col + k) : 0.f;
#pragma unroll
            for (int j = 0; j < W; ++j) ring[j][k] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < W - 1; ++i) {
            const int64_t t = first - (W - 1) + i;
            before[i] = PACKED ? ConvRow<T, W, V>::get(p, 0, 0, max(t, (int64_t)0), col) : ConvRow<T, W, V>::get(p, n, 0, t, col);
        }
        Where q{n, 0, p.T}, s{n, 0, p.T};                 // of the token whose g is formed; of the one whose dx is
        if (PACKED) { q.find(p, first); s = q; }
        for (int64_t t0 = first; t0 < end + (W - 1); t0 += STEP) {
            if (t0 + STEP < end + (W - 1)) {
#pragma unroll
                for (int i = 0; i < STEP; ++i) rows(t0 + STEP + i, xn[i], dyn[i]);
            }
#pragma unroll
            for (int i = 0; i < STEP; ++i) {
                const int64_t t = t0 + i, to = t - (W - 1);
                float g[V];
#pragma unroll
                for (int k = 0; k < V; ++k) g[k] = 0.f;
                bool none = t >= p.T || t >= end + (W - 1), early = false;
                if (PACKED && !none) {
                    if (t >= q.eos) q.next(p, t);
                    none = t < q.bos;
                    early = t - q.bos < W - 1;
                }
                if (!none) {
                    float xf[W][V];
#pragma unroll
                    for (int j = 0; j < W; ++j)
#pragma unroll
                        for (int k = 0; k < V; ++k) xf[j][k] = tap<W, STEP>(before, x, i + j)[k];
                    if (PACKED && early) {
#pragma unroll
                        for (int j = 0; j < W; ++j) {
                            const R e = ConvRow<T, W, V>::get(p, q.n, q.bos, t - q.bos - (W - 1) + j, col);
#pragma unroll
                            for (int k = 0; k < V; ++k) xf[j][k] = e[k];
                        }
                    }
                    conv_g<T, W, V>(p, w, b, xf, dy[i], g);
                    if (t < end) {
#pragma unroll
                        for (int k = 0; k < V; ++k) {
                            db[k] += g[k];
#pragma unroll
                            for (int j = 0; j < W; ++j) dw[k][j] = __builtin_fmaf(g[k], xf[j][k], dw[k][j]);
                        }
                    }
                }
#pragma unroll
                for (int j = 0; j < W - 1; ++j)
#pragma unroll
                    for (int k = 0; k < V; ++k) ring[j][k] = ring[j + 1][k];
#pragma unroll
                for (int k = 0; k < V; ++k) ring[W - 1][k] = g[k];
                if (to >= first && to < end) {
                    if (PACKED && to >= s.eos) s.next(p, to);
                    float d[V];
#pragma unroll
                    for (int k = 0; k < V; ++k) d[k] = 0.f;
#pragma unroll
                    for (int m = 0; m < W; ++m) {         // g_{to + m} through tap W - 1 - m (none behind the last token: g is zero there)
                        if (!PACKED || to + m < s.eos) {
#pragma unroll
                            for (int k = 0; k < V; ++k) d[k] = __builtin_fmaf(w[k][W - 1 - m], ring[m][k], d[k]);
                        }
                    }
                    if (PACKED && to < s.bos) {
#pragma unroll
                        for (int k = 0; k < V; ++k) d[k] = 0.f;
                    } else if (p.dlast && s.eos - to <= W - 1) {
                        R e;
                        e.load(static_cast<const T*>(p.dlast) + ((long long)s.n * (W - 1) + (W - 1 - (s.eos - to))) * p.D + col, V);
#pragma unroll
                        for (int k = 0; k < V; ++k) d[k] += e[k];
                    }
                    st_values<T, V, (V > 1)>(dx0 + to * p.D, d, V);
                }
            }
#pragma unroll
            for (int i = 0; i < W - 1; ++i) before[i] = x[STEP - (W - 1) + i];
#pragma unroll
            for (int i = 0; i < STEP; ++i) { x[i] = xn[i]; dy[i] = dyn[i]; }
        }
    }
    if (wave) {
#pragma unroll
        for (int k = 0; k < V; ++k) {
            red[wave - 1][k * (W + 1) + W][threadIdx.x & 63] = db[k];
#pragma unroll
            for (int j = 0; j < W; ++j) red[wave - 1][k * (W + 1) + j][threadIdx.x & 63] = dw[k][j];
        }
    }
    __syncthreads();
    if (wave || c >= p.cols) return;
    float* const to = p.part + blockIdx.x / col_blocks * ((long long)p.D * (W + 1));
#pragma unroll
    for (int k = 0; k < V; ++k) {
#pragma unroll
        for (int j = 0; j <= W; ++j) {
            float v = j < W ? dw[k][j < W ? j : 0] : db[k];
#pragma unroll
            for (int i = 0; i < 3; ++i) v += red[i][k * (W + 1) + j][threadIdx.x & 63];
            if (j < W) to[(long long)(col + k) * W + j] = v;
            else to[(long long)p.D * W + col + k] = v;
        }
    }
}

// One token: the state's rows and x are the taps
template <typename T, int W, int V>
__global__ __launch_bounds__(256) void short_conv_step_kernel(ConvArgs p) {
    const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
    if (id >= p.threads) return;
    const int col = (int)(id % p.cols) * V;
    const long long n = id / p.cols;
    float w[V][W], f[V], row[V];
    Raw<T, V, (V > 1)> x[W];
#pragma unroll
    for (int j = 0; j < W - 1; ++j) x[j].load(static_cast<const T*>(p.state) + (n * (W - 1) + j) * p.D + col, V);
    x[W - 1].load(static_cast<const T*>(p.x.p) + n * p.x.batch + col, V);
    ld_taps<W, V>(p.weight, p.w_f32, (long long)col * W, w);
#pragma unroll
    for (int k = 0; k < V; ++k) {
        f[k] = p.bias ? ld_param(p.bias, p.b_f32, col + k) : 0.f;
#pragma unroll
        for (int j = 0; j < W; ++j) f[k] = __builtin_fmaf(w[k][j], x[j][k], f[k]);
    }
    if (p.silu) {
        float g[V];
        sigmoid_each<T, V>(f, g);
#pragma unroll
        for (int k = 0; k < V; ++k) f[k] *= g[k];
    }
    st_values<T, V, (V > 1)>(static_cast<T*>(p.y) + n * p.D + col, f, V);
#pragma unroll
    for (int j = 1; j < W; ++j) {
#pragma unroll
        for (int k = 0; k < V; ++k) row[k] = x[j][k];
        st_values<T, V, (V > 1)>(static_cast<T*>(p.last) + (n * (W - 1) + j - 1) * p.D + col, row, V);
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------
constexpr int CONV_STEP = 8;
// Steps of a run: the more, the fewer tokens are read twice; as many runs as give every compute unit `waves` waves.  Forward, 16384 x 4096: 50 us with 16
// waves (four steps a run), 64 with 8, 54 with 32.
static int conv_steps(long long rows, long long cols, int T, int waves, int most) {
    const long long threads = waves * 64LL * 256, steps = rows * cols / (threads * CONV_STEP);
    return (int)std::max(1LL, std::min<long long>({steps, (long long)most, (T + CONV_STEP - 1) / CONV_STEP}));
}
static int conv_check(const hdla_conv_dims* d) {
    if (!d) return HDLA_ERR_NULL;
    for (int t : {d->dtype, d->weight_dtype, d->bias_dtype})
        if (t != HDLA_BF16 && t != HDLA_FP32) return HDLA_ERR_DTYPE;
    const bool none = d->B == 0 && d->N == 0;             // no sequences
    if ((!none && (d->B < 1 || d->N < 1)) || d->T < 0 || d->D < 1 || d->W < 2 || d->W > 4 || d->T > (1 << 30) || d->D > (1 << 24)) return HDLA_ERR_SHAPE;
    if (d->cu_seqlens ? d->B != 1 : d->N != d->B) return HDLA_ERR_SEQ;
    if ((long long)d->B * d->T > 0x7fffffffLL) return HDLA_ERR_SHAPE;
    return HDLA_OK;
}
// V channels a thread where everything lies on multiples of them (V elements of x, V W of the weight), else one
static bool conv_vec(const hdla_conv_dims* d, int v, const ConvArgs& a) {
    const int bytes = v * (d->dtype == HDLA_BF16 ? 2 : 4);
    if (d->D % v || d->x_row % v || d->x_batch % v || !fits(a.x.p, std::min(bytes, 16))) return false;
    return fits(a.weight, d->weight_dtype == HDLA_BF16 ? 8 : 16);
}
static ConvArgs conv_args(const hdla_conv_dims* d, const void* x, const void* weight, const void* bias, const void* state) {
    ConvArgs a{};
    a.x = {x, d->x_batch, d->x_row};
    a.weight = weight; a.bias = bias; a.state = state;
    a.cu = d->cu_seqlens; a.T = d->T; a.N = d->N; a.D = d->D;
    a.w_f32 = d->weight_dtype == HDLA_FP32; a.b_f32 = d->bias_dtype == HDLA_FP32; a.silu = d->silu != 0;
    return a;
}
#define HDLA_CONV_WIDTHS(CASE) CASE(2) CASE(3) CASE(4)

template <typename T, int V> static hipError_t launch_conv(ConvArgs a, int W, hipStream_t s) {
    a.cols = a.D / V;
    const int steps = conv_steps((long long)a.T * (a.cu ? 1 : a.N), a.cols, a.T, 16, 8);
    a.runs = (a.T + steps * CONV_STEP - 1) / (steps * CONV_STEP);
    a.threads = (long long)a.cols * a.runs * (a.cu ? 1 : a.N);
    const long long all = a.threads + (a.last ? (long long)a.cols * (W - 1) * a.N : 0), blocks = (all + 255) / 256;
    if (blocks > 0x7fffffffLL) return hipErrorInvalidValue;
    if (!blocks) return hipSuccess;
    switch (W) {
#define HDLA_CASE(WW)                                                                                                                            \
    case WW:                                                                                                                                     \
        if (a.cu) hipLaunchKernelGGL((short_conv_kernel<T, WW, V, CONV_STEP, true>), dim3((unsigned)blocks), dim3(256), 0, s, a, steps);         \
        else hipLaunchKernelGGL((short_conv_kernel<T, WW, V, CONV_STEP, false>), dim3((unsigned)blocks), dim3(256), 0, s, a, steps);             \
        break;
        HDLA_CONV_WIDTHS(HDLA_CASE)
#undef HDLA_CASE
    }
    return hipGetLastError();
}
template <typename T, int V> static hipError_t launch_conv_step(ConvArgs a, int W, hipStream_t s) {
    a.cols = a.D / V;
    a.threads = (long long)a.cols * a.N;
    const long long blocks = (a.threads + 255) / 256;
    if (blocks > 0x7fffffffLL) return hipErrorInvalidValue;
    switch (W) {
#define HDLA_CASE(WW) case WW: hipLaunchKernelGGL((short_conv_step_kernel<T, WW, V>), dim3((unsigned)blocks), dim3(256), 0, s, a); break;
        HDLA_CONV_WIDTHS(HDLA_CASE)
#undef HDLA_CASE
    }
    return hipGetLastError();
}
// Steps of a run of the backward pass, its runs, and the rows of partial sums that they leave: four runs a row
struct ConvGradPlan { int steps; long long runs, rows; };
static ConvGradPlan conv_grad_plan(const hdla_conv_dims* d) {
    ConvGradPlan g;
    g.steps = conv_steps((long long)d->T * d->B, (d->D + 3) / 4, d->T, 6, 8);
    g.runs = (d->T + g.steps * CONV_STEP - 1) / (g.steps * CONV_STEP);
    g.rows = (g.runs * (d->cu_seqlens ? 1 : d->N) + 3) / 4;
    return g;
}
template <typename T, int V> static hipError_t launch_conv_grad(ConvArgs a, int W, const ConvGradPlan& g, hipStream_t s) {
    a.cols = a.D / V;
    a.runs = (int)g.runs;
    const long long col_blocks = (a.cols + 63) / 64, states = a.dstate ? ((long long)a.cols * (W - 1) * a.N + 255) / 256 : 0, blocks = col_blocks * g.rows + states;
    if (blocks > 0x7fffffffLL) return hipErrorInvalidValue;
    if (!blocks) return hipSuccess;
    switch (W) {
#define HDLA_CASE(WW)                                                                                                                                                  \
    case WW:                                                                                                                                                           \
        if (a.cu) hipLaunchKernelGGL((short_conv_grad_kernel<T, WW, V, CONV_STEP, true>), dim3((unsigned)blocks), dim3(256), 0, s, a, g.steps, col_blocks, g.rows);    \
        else hipLaunchKernelGGL((short_conv_grad_kernel<T, WW, V, CONV_STEP, false>), dim3((unsigned)blocks), dim3(256), 0, s, a, g.steps, col_blocks, g.rows);        \
        break;
        HDLA_CONV_WIDTHS(HDLA_CASE)
#undef HDLA_CASE
    }
    return hipGetLastError();
}

}  // namespace hdla

using namespace hdla;

extern "C" int hdla_short_conv_fwd(const hdla_conv_dims* dims, const void* x, const void* weight, const void* bias, const void* state, void* y, void* last,
                                   void* stream) {
    const int rc = conv_check(dims);
    if (rc) return rc;
    if (!weight || ((long long)dims->B * dims->T > 0 && (!x || !y))) return HDLA_ERR_NULL;
    for (const void* q : {state, (const void*)y, (const void*)last})
        if (!fits(q, 16)) return HDLA_ERR_ALIGN;
    ConvArgs a = conv_args(dims, x, weight, bias, state);
    a.y = y; a.last = last;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    hipError_t e;
    if (dims->dtype == HDLA_BF16) e = conv_vec(dims, 8, a) ? launch_conv<bf16, 8>(a, dims->W, s) : launch_conv<bf16, 1>(a, dims->W, s);
    else e = conv_vec(dims, 4, a) ? launch_conv<float, 4>(a, dims->W, s) : launch_conv<float, 1>(a, dims->W, s);
    return e == hipSuccess ? HDLA_OK : (int)e;
}
extern "C" int hdla_short_conv_step(const hdla_conv_dims* dims, const void* x, const void* weight, const void* bias, const void* state, void* y, void* new_state,
                                    void* stream) {
    const int rc = conv_check(dims);
    if (rc) return rc;
    if (dims->T != 1 || dims->cu_seqlens) return HDLA_ERR_SHAPE;
    if (!dims->N) return HDLA_OK;
    if (!x || !weight || !state || !y || !new_state) return HDLA_ERR_NULL;
    for (const void* q : {state, (const void*)y, (const void*)new_state})
        if (!fits(q, 16)) return HDLA_ERR_ALIGN;
    ConvArgs a = conv_args(dims, x, weight, bias, state);
    a.y = y; a.last = new_state;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    hipError_t e;
    if (dims->dtype == HDLA_BF16) e = conv_vec(dims, 8, a) ? launch_conv_step<bf16, 8>(a, dims->W, s) : launch_conv_step<bf16, 1>(a, dims->W, s);
    else e = conv_vec(dims, 4, a) ? launch_conv_step<float, 4>(a, dims->W, s) : launch_conv_step<float, 1>(a, dims->W, s);
    return e == hipSuccess ? HDLA_OK : (int)e;
}
extern "C" size_t hdla_short_conv_workspace_bytes(const hdla_conv_dims* dims) {
    return conv_check(dims) ? 0 : std::max<size_t>((size_t)conv_grad_plan(dims).rows * dims->D * (dims->W + 1) * 4, 16);
}
extern "C" int hdla_short_conv_bwd(const hdla_conv_dims* dims, const void* x, const void* weight, const void* bias, const void* state, const void* dy, const void* dlast,
                                   void* dx, void* dweight, void* dbias, void* dstate, void* workspace, size_t workspace_bytes, void* stream) {
    const int rc = conv_check(dims);
    if (rc) return rc;
    if (!weight || !dweight || (bias && !dbias) || ((long long)dims->B * dims->T > 0 && (!x || !dy || !dx))) return HDLA_ERR_NULL;
    for (const void* q : {state, dy, dlast, (const void*)dx, (const void*)dstate})
        if (!fits(q, 16)) return HDLA_ERR_ALIGN;
    if (!workspace || !fits(workspace, 16) || workspace_bytes < hdla_short_conv_workspace_bytes(dims)) return HDLA_ERR_WORKSPACE;
    ConvArgs a = conv_args(dims, x, weight, bias, state);
    a.dy = dy; a.dlast = dlast; a.dx = dx; a.dstate = dstate;
    a.part = static_cast<float*>(workspace);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const ConvGradPlan g = conv_grad_plan(dims);
    hipError_t e;
    // four channels a thread also in bf16: eight need the registers of twice as many sums (8192 x 2048, forward and backward 69 us; so 56)
    if (dims->dtype == HDLA_BF16) e = conv_vec(dims, 4, a) ? launch_conv_grad<bf16, 4>(a, dims->W, g, s) : launch_conv_grad<bf16, 1>(a, dims->W, g, s);
    else e = conv_vec(dims, 4, a) ? launch_conv_grad<float, 4>(a, dims->W, g, s) : launch_conv_grad<float, 1>(a, dims->W, g, s);
    if (e != hipSuccess) return (int)e;
    ColumnSums c{};
    c.part = a.part; c.rows = g.rows;
    c.add(dweight, a.w_f32, (long long)dims->D * dims->W);
    c.add(bias ? dbias : nullptr, a.b_f32, dims->D);
    e = launch_column_sums(c, s);
    return e == hipSuccess ? HDLA_OK : (int)e;
}
