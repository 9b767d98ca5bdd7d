// Sums over the rows of partial results [rows][columns] in 32 bits, in the order of the rows: what workgroups left of gradients that all of them
// add to (weights, vectors, inputs that channels share).  The columns go to up to four results one behind the other, in 32 bits or rounded once to bf16.
#pragma once
#include "hdla_common.cuh"

namespace hdla {

struct ColumnSums {
    const float* part;
    int phases;                       // (the launch's)
    long long columns, rows, apart;   // apart: elements from one row to the next (0: columns)
    int results;
    long long end[4];             // of each result's columns
    void* out[4];
    int f32[4];
    // results whose columns are tokens (packed batches: those of no sequence become zero, whatever `part` holds there)
    const int64_t* cu;
    int N, T;
    long long per_token, tokens_end;
    // the next n columns (o null: of no use)
    void add(void* o, bool is_f32, long long n) {
        if (!n) return;
        const long long at = results ? end[results - 1] : 0;
        out[results] = o;
        f32[results] = is_f32;
        end[results++] = at + n;
        columns = at + n;
    }
};
hipError_t launch_column_sums(const ColumnSums& s, hipStream_t stream, const ColumnSums& more = ColumnSums{});

}  // namespace hdla
