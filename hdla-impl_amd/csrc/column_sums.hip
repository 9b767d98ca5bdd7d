// Bound by HBM where there are many columns, by the latency of a few rounds of loads where there are few; what it measured stands at the passes that leave the partial results.
#include "column_sums.cuh"

namespace hdla {

// PH threads a column, each every PH-th row; their sums are added in order
template <int PH> __global__ __launch_bounds__(256) void column_sums_kernel(ColumnSums s) {
    constexpr int COLS = 256 / PH;
    __shared__ float red[PH > 1 ? PH : 1][COLS];
    const int c = threadIdx.x % COLS, ph = threadIdx.x / COLS;
    const long long col = (long long)blockIdx.x * COLS + c;
    int decreases = 0;
    if (s.cu) {
        for (int n = threadIdx.x; n < s.N; n += 256) decreases |= s.cu[n + 1] < s.cu[n];
        decreases = __syncthreads_or(decreases);
    }
    bool covered = true;
    if (s.cu && col < s.tokens_end) {
        const long long t = col / s.per_token % s.T;
        if (!decreases) covered = t >= s.cu[0] && t < s.cu[s.N];
        else {
            covered = false;
            for (int n = 0; n < s.N && !covered; ++n) {
                int64_t bos, eos;
                packed_bounds(s.cu, n, s.T, bos, eos);
                covered = t >= bos && t < eos;
            }
        }
    }
    float sum = 0.f;
    if (col < s.columns && covered) {
        const float* p = s.part + col;
#pragma unroll 8
        for (long long r = ph; r < s.rows; r += PH) sum += p[r * s.apart];
    }
    if constexpr (PH > 1) {
        red[ph][c] = sum;
        __syncthreads();
        if (ph) return;
#pragma unroll
        for (int i = 1; i < PH; ++i) sum += red[i][c];
    }
    if (col >= s.columns) return;
    int at = 0;
    while (at + 1 < s.results && col >= s.end[at]) ++at;
    const long long e = col - (at ? s.end[at - 1] : 0);
    if (!s.out[at]) return;
    if (s.f32[at]) static_cast<float*>(s.out[at])[e] = sum;
    else st_elem(static_cast<bf16*>(s.out[at]) + e, sum);
}

hipError_t launch_column_sums(const ColumnSums& sums, hipStream_t stream) {
    ColumnSums s = sums;
    if (!s.columns) return hipSuccess;
    if (!s.apart) s.apart = s.columns;
    // us, 1 / 16 threads a column: 745 rows of 6144 columns (a norm's weights) 36 / 9, 104 of 10240 (a convolution's) 5.2 / 4.0; 128 of 262144 (a scan's dB and dC) 22 with either
    const int ph = s.rows < 8 || s.columns >= 65536 * 4 ? 1 : 16;
    const long long blocks = (s.columns * ph + 255) / 256;
    if (blocks > 0x7fffffffLL) return hipErrorInvalidValue;
    if (ph == 1) hipLaunchKernelGGL(column_sums_kernel<1>, dim3((unsigned)blocks), dim3(256), 0, stream, s);
    else hipLaunchKernelGGL(column_sums_kernel<16>, dim3((unsigned)blocks), dim3(256), 0, stream, s);
    return hipGetLastError();
}

}  // namespace hdla
