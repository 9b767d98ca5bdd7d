// Bound by HBM where there are many columns, by the latency of a few rounds of loads where there are few; what it measured stands at the passes that leave the partial results.
#include "column_sums.cuh"

namespace hdla {

// `phases` threads a column, each every so many-th row; their sums are added in order.  Two lots of partial results in one launch: the workgroups from `first` on have the other's.
__global__ __launch_bounds__(256) void column_sums_kernel(ColumnSums one, ColumnSums other, unsigned first) {
    __shared__ float red[256];
    const ColumnSums& s = blockIdx.x < first ? one : other;
    const int cols = 256 / s.phases, c = threadIdx.x & (cols - 1), ph = threadIdx.x / cols;
    const long long col = (long long)(blockIdx.x < first ? blockIdx.x : blockIdx.x - first) * cols + c;
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
        for (long long r = ph; r < s.rows; r += s.phases) sum += p[r * s.apart];
    }
    if (s.phases > 1) {
        red[threadIdx.x] = sum;
        __syncthreads();
        if (ph) return;
        for (int i = 1; i < s.phases; ++i) sum += red[i * cols + c];
    }
    if (col >= s.columns) return;
    int at = 0;
    while (at + 1 < s.results && col >= s.end[at]) ++at;
    const long long e = col - (at ? s.end[at - 1] : 0);
    if (!s.out[at]) return;
    if (s.f32[at]) static_cast<float*>(s.out[at])[e] = sum;
    else st_elem(static_cast<bf16*>(s.out[at]) + e, sum);
}

// threads a column, and the workgroups
static long long shares(ColumnSums& s) {
    if (!s.apart) s.apart = s.columns;
    // us, 1 / 16 threads a column: 745 rows of 6144 columns (a norm's weights) 36 / 9, 104 of 10240 (a convolution's) 5.2 / 4.0; 128 of 262144 (a scan's dB and dC) 22 with either
    s.phases = s.rows < 8 || s.columns >= 65536 * 4 ? 1 : 16;
    return (s.columns * s.phases + 255) / 256;
}
hipError_t launch_column_sums(const ColumnSums& sums, hipStream_t stream, const ColumnSums& more) {
    ColumnSums one = sums, other = more;
    const long long first = shares(one), blocks = first + shares(other);
    if (blocks > 0x7fffffffLL) return hipErrorInvalidValue;
    if (!blocks) return hipSuccess;
    hipLaunchKernelGGL(column_sums_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, one, other, (unsigned)first);
    return hipGetLastError();
}

}  // namespace hdla
