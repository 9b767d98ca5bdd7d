// What the kernels of the selective state space scan share: how its operands lie, how a wave takes them, and the step sizes.
//
// Per channel d with S states, decays A [D, S] (as they enter the exponent) and per-token B, C [G, S] that D / G channels share:
//     delta_t = softplus(dt_t + bias);   h_t = exp(delta_t A) h_{t-1} + delta_t x_t B_t;   y_t = (C_t . h_t + D x_t) silu(z_t)
//
// Lanes: LPC lanes of a wave hold the states of one channel, four each, and a wave has 64 / LPC channels and L tokens at a time.  The W waves
// of a workgroup take consecutive pieces of L tokens.  Every wave scans its piece from zero, the pieces' decays and ends meet in LDS, where one thread
// a state chains them, and the wave walks its piece once more from the state that enters it.  The exponentials are formed once, two
// issue slots each (8.1 cycles a wave where a multiplication takes 4.1), and stay in registers for the second walk: that one costs two slots a state.
#pragma once
#include "hdla_common.cuh"
#include "row_tile.cuh"
#include "../../include/hdla_state_space.h"

#include <algorithm>

namespace hdla {

typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// floats from one channel to the next of a piece of L tokens in LDS: 16 bytes aligned, neighbours on other banks
constexpr int ss_pitch(int L) { return L + 4; }
constexpr int SS_TOK = 8;             // tokens of a wave at a time
// Tokens between the states that a forward pass leaves for the backward pass: a tile of that pass, of four waves where there are workgroups for two on every compute unit,
// whose barriers then fall into each other's work, else of eight.  us a training step, eight / four: 4 x 2048 x 2048 (512 workgroups of four waves) 432 / 416, 2503 x 520 in fp32 (264) 152 / 181.
constexpr int SS_TILE_FEW = 64, SS_TILE_MANY = 32;      // (2^6, 2^5)

// element (b, t, .) of an operand: base + b batch + t row.  A wave's tokens are reached by 32-bit offsets from its first one's row.
struct Operand {
    const void* p;
    long long batch, row;
};
constexpr long long ROW_MOST = 1 << 24;      // elements; 16 rows of 4 bytes reach 2^30
template <typename T> __device__ __forceinline__ const T* row_of(const Operand& o, long long batch, long long t) {
    return static_cast<const T*>(o.p) + batch * o.batch + t * o.row;
}
struct ScanArgs {
    Operand x, dt, z, B, C;           // z.p may be null; B, C: + group
    long long B_group, C_group;
    const void *A, *D, *bias;         // D, bias may be null
    int A_f32, D_f32, bias_f32;
    const float* h0;                  // [N, D, S], may be null
    float* ht;                        // [N, D, S], may be null
    void* y;                          // [rows, D]
    float* ckpt;                      // [slots][blocks][64][4], may be null
    const int64_t* cu;
    int T, N, DD, S, G, softplus;
    int per_group, blocks;            // channel blocks of a group, of all of them
    int every_log2;                   // of SS_TILE_FEW or SS_TILE_MANY
    // backward
    const void* dy;                   // [rows, D]
    const float* dht;
    void *dx, *ddt, *dz;              // [rows, D]
    float *part_bc, *part_own, *dh0;
    long long rows;
    int slots;                        // units (sequences, or segments of them) at a time
    int first, take;                  // blocks of each group that a pass has, from the first on
    // segments: 0, or how many tokens one has; `units` of them, and for each [blocks][256] what it leaves if nothing enters, and [blocks][256] its decays
    int seg, units;
    float* ends;
};
constexpr int SS_SEGMENT = 128;       // segments are multiples of it

// V elements of T as they come from memory; VEC: with loads of several, else (rows at any address) one by one
template <typename T, int V, bool VEC> struct Raw;
template <int V> struct Raw<bf16, V, true> {
    static constexpr int NW = V < 2 ? 1 : V / 2;
    uint32_t w[NW];
    __device__ __forceinline__ void load(const bf16* p, int) {
        if constexpr (V == 1) w[0] = p->x;
        else if constexpr (V == 4) { const u32x2 r = *reinterpret_cast<const u32x2*>(p); w[0] = r[0]; w[1] = r[1]; }
        else { const u32x4 r = *reinterpret_cast<const u32x4*>(p); w[0] = r[0]; w[1] = r[1]; w[2] = r[2]; w[3] = r[3]; }
    }
    template <typename R> __device__ __forceinline__ void load(R rows, uint32_t off, int) {
        if constexpr (V == 1) w[0] = __builtin_amdgcn_raw_buffer_load_b16(rows, off, 0, 0);
        else if constexpr (V == 2) w[0] = __builtin_amdgcn_raw_buffer_load_b32(rows, off, 0, 0);
        else if constexpr (V == 4) { const u32x2 r = __builtin_amdgcn_raw_buffer_load_b64(rows, off, 0, 0); w[0] = r[0]; w[1] = r[1]; }
        else { const u32x4 r = __builtin_amdgcn_raw_buffer_load_b128(rows, off, 0, 0); w[0] = r[0]; w[1] = r[1]; w[2] = r[2]; w[3] = r[3]; }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < NW; ++i) w[i] = 0;
    }
    __device__ __forceinline__ float operator[](int i) const { return __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16); }
};
constexpr uint32_t NOWHERE = 0x80000000u, NOWHERE_FROM = 0x7fffffffu;    // an offset that a buffer's loads answer with zero, and where these begin
template <int V> struct Raw<bf16, V, false> {
    uint32_t w[V];
    // (the first n)
    __device__ __forceinline__ void load(const bf16* p, int n) {
#pragma unroll
        for (int i = 0; i < V; ++i) w[i] = i < n ? p[i].x : 0;
    }
    template <typename R> __device__ __forceinline__ void load(R rows, uint32_t off, int n) {
#pragma unroll
        for (int i = 0; i < V; ++i) w[i] = __builtin_amdgcn_raw_buffer_load_b16(rows, i < n ? off + 2 * i : NOWHERE, 0, 0);
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < V; ++i) w[i] = 0;
    }
    __device__ __forceinline__ float operator[](int i) const { return __uint_as_float(w[i] << 16); }
};
template <int V, bool VEC> struct Raw<float, V, VEC> {
    float w[V];
    __device__ __forceinline__ void load(const float* p, int n) {
        if constexpr (VEC && V % 4 == 0) {
#pragma unroll
            for (int i = 0; i < V; i += 4) {
                const f32x4 r = *reinterpret_cast<const f32x4*>(p + i);
#pragma unroll
                for (int j = 0; j < 4; ++j) w[i + j] = r[j];
            }
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) w[i] = i < n ? p[i] : 0.f;
        }
    }
    template <typename R> __device__ __forceinline__ void load(R rows, uint32_t off, int n) {
        if constexpr (VEC && V % 4 == 0) {
#pragma unroll
            for (int i = 0; i < V; i += 4) {
                const u32x4 r = __builtin_amdgcn_raw_buffer_load_b128(rows, off + 4 * i, 0, 0);
#pragma unroll
                for (int j = 0; j < 4; ++j) w[i + j] = __uint_as_float(r[j]);
            }
        } else if constexpr (VEC && V == 2) {
            const u32x2 r = __builtin_amdgcn_raw_buffer_load_b64(rows, off, 0, 0);
            w[0] = __uint_as_float(r[0]);
            w[1] = __uint_as_float(r[1]);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) w[i] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rows, i < n ? off + 4 * i : NOWHERE, 0, 0));
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < V; ++i) w[i] = 0.f;
    }
    __device__ __forceinline__ float operator[](int i) const { return w[i]; }
};
// the first n of V results, rounded to nearest
template <typename T, int V, bool VEC> __device__ __forceinline__ void st_values(T* p, const float (&x)[V], int n) {
    if constexpr (VEC && V == 8 && sizeof(T) == 2) {
        const s16x4 lo = to_frag<T>(f32x4{x[0], x[1], x[2], x[3]}).v, hi = to_frag<T>(f32x4{x[4], x[5], x[6], x[7]}).v;
        *reinterpret_cast<s16x8*>(p) = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    } else if constexpr (VEC && V == 2 && sizeof(T) == 2) {
        *reinterpret_cast<uint32_t*>(p) = __builtin_bit_cast(u32x2, to_frag<T>(f32x4{x[0], x[1], 0.f, 0.f}).v)[0];
    } else if constexpr (VEC && V == 2) {
        *reinterpret_cast<u32x2*>(p) = u32x2{__float_as_uint(x[0]), __float_as_uint(x[1])};
    } else if constexpr (VEC && V % 4 == 0) {
#pragma unroll
        for (int i = 0; i < V; i += 4) st_frag(p + i, to_frag<T>(f32x4{x[i], x[i + 1], x[i + 2], x[i + 3]}));
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < n) st_elem(p + i, x[i]);
    }
}

__device__ __forceinline__ float ld_param(const void* p, int f32, long long i) {
    return f32 ? static_cast<const float*>(p)[i] : ld_elem(static_cast<const bf16*>(p) + i);
}
// A decay as it stands in the exponent, in base 2.  The lowest finite number for minus infinity, whose product with a step size of zero is no number: so a place without a token,
// and a token that is passed over, leave a state as it is.
__device__ __forceinline__ float decay_exponent(float A) {
    const float a = A * LOG2E;
    return a < -3.402823466e38f ? -3.402823466e38f : a;
}
__device__ __forceinline__ float ld_decay(const void* p, int f32, long long i) { return decay_exponent(ld_param(p, f32, i)); }
// four states of a channel, the first `n` of which there are
__device__ __forceinline__ f32x4 ld_states(const float* p, int n, bool whole) {
    if (whole) return *reinterpret_cast<const f32x4*>(p);
    f32x4 r = zero4();
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (j < n) r[j] = p[j];
    return r;
}
__device__ __forceinline__ void st_states(float* p, f32x4 x, int n, bool whole) {
    if (whole) { *reinterpret_cast<f32x4*>(p) = x; return; }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (j < n) p[j] = x[j];
}

// softplus(v) = max(v, 0) + log(1 + e), e = exp(-|v|) <= 1, and log(1 + e) = 2 artanh(s), s = e / (2 + e) <= 1/3: 2 artanh(s) / s as a polynomial in s^2 (a fit of least
// largest relative error over 0 .. 1/9, off by 8e-9, an eighth of a rounding).  No logarithm, whose hardware form loses what is small beside one.
template <typename T> __device__ __forceinline__ float softplus(float v, float& e) {
    e = exp_t<T>(-fabsf(v));
    const float s = e * __builtin_amdgcn_rcpf(2.f + e), q = s * s;
    float r = 0.28178343f;
    r = __builtin_fmaf(r, q, 0.27960610f);
    r = __builtin_fmaf(r, q, 0.40024909f);
    r = __builtin_fmaf(r, q, 0.66666317f);
    r = __builtin_fmaf(r, q, 2.f);
    return __builtin_fmaf(s, r, fmaxf(v, 0.f));
}
// its derivative, from that exponential
__device__ __forceinline__ float softplus_slope(float v, float e) { return (v < 0.f ? e : 1.f) * __builtin_amdgcn_rcpf(1.f + e); }
// The hardware's reciprocal, a unit in the last place at the most; of an exponential that is infinite, zero.
template <typename T, int N> __device__ __forceinline__ void sigmoid_each(const float (&x)[N], float (&s)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = __builtin_amdgcn_rcpf(1.f + exp_t<T>(-x[i]));
}

constexpr float LN2 = 0.69314718055994530942f;

// Which unit and block of channels a workgroup has.  Workgroups go to the eight XCDs in turns, and neighbouring blocks share cache lines: each XCD has an eighth of the
// blocks, of all units, so that units of unequal lengths leave none idle.  (Units one behind the other on an XCD instead: 2000 tokens in segments of 768, one of three sequences being
// 1500 long, backward 129 us; so 68.)  Fewer than 16 blocks would leave XCDs without one: these are dealt out as they come.
constexpr int XCDS = 8;
inline __host__ __device__ int blocks_an_xcd(int blocks) { return blocks < 2 * XCDS ? 0 : (blocks + XCDS - 1) / XCDS; }
inline long long scan_workgroups(int blocks, long long units) { return blocks_an_xcd(blocks) ? (long long)XCDS * blocks_an_xcd(blocks) * units : blocks * units; }
__device__ __forceinline__ bool scan_work(int id, int blocks, int& unit, int& block) {
    const int most = blocks_an_xcd(blocks);
    if (!most) {
        unit = id / blocks;
        block = id - unit * blocks;
        return true;
    }
    const int xcd = id % XCDS, k = id / XCDS, first = xcd * blocks / XCDS;
    unit = k / most;
    block = first + k - unit * most;
    return block < (xcd + 1) * blocks / XCDS;
}

// A wave's rows of an operand, tile after tile: the address of its first token's and how far the next tile's are.  (Formed anew in every tile the products
// of strides are some 150 scalar instructions, as long as half of the vector ones.)
template <typename T> struct Cursor {
    const T* p;
    long long step;
    __device__ __forceinline__ Cursor(const T* first, long long s) : p(first), step(s) {}
    // (opaque: the compiler would otherwise go back to products of the tile's number)
    __device__ __forceinline__ void next() { p += step; asm("" : "+s"(p)); }
    // The rows from there on: loads at NOWHERE give zero, which lanes without a token or a channel ask for.  (Under a condition instead every loaded register has a zero
    // beside it that lives through the loop.)
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t rows() const { return __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(p), 0, NOWHERE_FROM, 0x00027000); }
};

// The piece of work that a workgroup has: a sequence, or (p.seg) a segment of one.  Packed sequences' counts of segments are not known to the host: sequence n has
// the units from bos / seg + n on, which never overlap; those that no segment has are idle (`ok`).
struct Unit {
    int n, index, len, from, to;      // of its sequence: number of the segment, tokens, first token, one behind the last
    int64_t bos;
    bool ok;
    __device__ __forceinline__ Unit(const ScanArgs& p, int unit) {
        n = unit;
        index = 0;
        if (p.seg && !p.cu) {
            const int per = (p.T + p.seg - 1) / p.seg;
            n = unit / per;
            index = unit - n * per;
        } else if (p.seg) {
            int lo = 0, hi = p.N - 1;                     // the last sequence that begins at or before this unit
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (first(p, mid) <= unit) lo = mid;
                else hi = mid - 1;
            }
            n = lo;
            index = unit - (int)first(p, n);
        }
        bos = 0;
        int64_t eos = p.T;
        if (p.cu) packed_bounds(p.cu, n, p.T, bos, eos);
        len = (int)(eos - bos);
        ok = index >= 0 && (index == 0 || (long long)index * p.seg < len);
        from = p.seg ? index * p.seg : 0;
        to = p.seg ? min(len, from + p.seg) : len;
    }
    static __device__ __forceinline__ int64_t first(const ScanArgs& p, int n) { return min(max(p.cu[n], (int64_t)0), (int64_t)p.T) / p.seg + n; }
    __device__ __forceinline__ int segments(const ScanArgs& p) const { return p.seg ? max(1, (len + p.seg - 1) / p.seg) : 1; }
};
__device__ __forceinline__ float* ends_of(const ScanArgs& p, long long unit, int block) { return p.ends + (unit * p.blocks + block) * 512; }

// Where a lane stands: as a scanner (channel c, states 4 q .. 4 q + 3) and as a carrier of operands and results (token tok of the piece, V channels from ch)
template <int LPC, int TOKENS> struct ScanLane {
    static constexpr int CHN = 64 / LPC, V = TOKENS > LPC ? TOKENS / LPC : 1;
    int c, q, tok, ch, d0, d, dv, left, carried, group;
    bool live;
    __device__ __forceinline__ ScanLane(const ScanArgs& p, int block) {
        const int l = lane_id(), size = p.DD / p.G;
        group = block / p.per_group;
        const int first = (block - group * p.per_group) * CHN;
        d0 = group * size + first;
        c = l / LPC;
        q = l % LPC;
        d = d0 + c;
        live = first + c < size;
        left = live ? min(max(p.S - 4 * q, 0), 4) : 0;           // states of this lane that there are
        tok = l / (CHN / V);                                      // (LPC = 16, eight tokens: beyond them on half of the lanes)
        ch = l % (CHN / V) * V;
        dv = d0 + ch;
        carried = min(max(size - first - ch, 0), V);             // channels of these V that there are
    }
    // bytes from the wave's first token's row, at channel d0, to this carrier's channels of its token
    __device__ __forceinline__ uint32_t offset(long long row, int size) const { return ((uint32_t)tok * (uint32_t)row + (uint32_t)ch) * (uint32_t)size; }
};

// B or C of a wave's piece, its tokens x 4 LPC states, as fp32 in LDS: [tok][quad]
template <typename T, int LPC, int TOKENS, bool VEC> struct StatesOf {
    static constexpr int PIECES = TOKENS * LPC < 64 ? 1 : TOKENS * LPC / 64;
    Raw<T, 4, VEC> r[PIECES];
    __device__ __forceinline__ void load(const Cursor<T>& base, uint32_t row, int tokens, int S) {
        const auto rows = base.rows();
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int e = i * 64 + lane_id(), t = e / LPC, s = e % LPC * 4;
            r[i].load(rows, t < tokens && s < S ? (t * row + s) * (uint32_t)sizeof(T) : NOWHERE, S - s);
        }
    }
    __device__ __forceinline__ void put(f32x4* lds) const {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int e = i * 64 + lane_id();
            if (PIECES * 64 <= TOKENS * LPC || e < TOKENS * LPC) lds[e] = f32x4{r[i][0], r[i][1], r[i][2], r[i][3]};
        }
    }
};

// Tokens stay in their order: left to itself the scheduler asks for the operands of all of them at once, and spills.
__device__ __forceinline__ void apart() { __builtin_amdgcn_sched_barrier(0); }

// sums over the LPC lanes of a channel
template <int LPC, int N> __device__ __forceinline__ void sum_channel(float (&x)[N]) { sum_lanes<N>(x, LPC); }

// A block's states in the first slot of a sequence, of those that a forward pass leaves: packed sequences' counts of slots are not known to the host, and these never overlap
__device__ __forceinline__ float* ckpt_of(const ScanArgs& p, int n, int64_t bos, int block) {
    const long long slot = p.cu ? (bos >> p.every_log2) + n : (long long)n * ((p.T + (1 << p.every_log2) - 1) >> p.every_log2);
    return p.ckpt + (slot * p.blocks + block) * 256;
}
inline long long ckpt_slots(bool packed, long long T, long long N, int every) {
    return packed ? T / every + N + 1 : N * ((T + every - 1) / every);
}

// ---- host side: what both passes and the workspace sizes go by ---------------------------------------------------------
inline int lanes_of(int S) { return S <= 8 ? 2 : S <= 16 ? 4 : S <= 32 ? 8 : 16; }

// What both passes and the workspace sizes go by
struct ScanPlan {
    int lpc, per_group, blocks, slots, seg, every, take, passes;
    bool vec;
    long long rows, ckpt, units;
};
// Segments fill the device where there are few (sequence, channel block) pairs, at `cost` times the work.  In tokens that a compute unit walks: whole sequences (of packed
// ones the longest is taken for twice the average) against segments of the length that is best, which have to gain an eighth.  `at_once`: channel blocks that are worked on
// together.
inline void scan_segments(const hdla_scan_dims* d, ScanPlan& s, float cost, int at_once) {
    constexpr long long CUS = 256;
    if (!d->N) return;
    const bool packed = d->cu_seqlens != nullptr;
    const long long average = d->T / (packed ? d->N : 1), longest = packed && d->N > 1 ? std::min<long long>(2 * average, d->T) : d->T;
    const long long wide = scan_workgroups(at_once, 1);
    auto rounds = [](long long wgs) { return (wgs + CUS - 1) / CUS; };
    const long long all = wide * d->N;
    float best = 0.875f * (float)std::max<long long>(longest, rounds(all) * average);
    s.seg = 0;
    s.units = d->N;
    for (long long seg = 2 * SS_SEGMENT; seg < longest; seg += seg < 8 * SS_SEGMENT ? SS_SEGMENT : seg / 4 / SS_SEGMENT * SS_SEGMENT) {
        const long long busy = packed ? d->T / seg + (d->N + 1) / 2 : d->N * ((d->T + seg - 1) / seg), units = packed ? d->T / seg + d->N : busy;
        if (units * (s.blocks + 8) > 0x7fffffffLL) continue;
        // (and what is chained in front of a segment, some two tokens each of those before it, and a launch)
        const float t = cost * (float)(rounds(busy * wide) * seg) + 2.f * (float)(longest / seg) + 128.f;
        if (t < best) { best = t; s.seg = (int)seg; s.units = units; }
    }
}
inline size_t ends_bytes(const ScanPlan& s) { return s.seg ? (size_t)s.units * s.blocks * 512 * 4 : 0; }
constexpr float SEGMENT_COST_FORWARD = 1.6f, SEGMENT_COST_BACKWARD = 1.25f;
inline bool fits(const void* p, int to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

inline int scan_plan(const hdla_scan_dims* d, ScanPlan& s) {
    if (!d) return HDLA_ERR_NULL;
    if (d->dtype != HDLA_BF16 && d->dtype != HDLA_FP32) return HDLA_ERR_DTYPE;
    for (int t : {d->A_dtype, d->D_dtype, d->bias_dtype})
        if (t != HDLA_BF16 && t != HDLA_FP32) return HDLA_ERR_DTYPE;
    const bool none = d->B == 0 && d->N == 0;             // no sequences
    if ((!none && (d->B < 1 || d->N < 1)) || d->T < 0 || d->D < 1 || d->S < 1 || d->S > 64 || d->G < 1 || d->D % d->G) return HDLA_ERR_SHAPE;
    if (d->cu_seqlens ? d->B != 1 : d->N != d->B) return HDLA_ERR_SEQ;
    if (d->T > (1 << 30) || d->D > ROW_MOST) return HDLA_ERR_SHAPE;
    for (long long r : {d->x_row, d->dt_row, d->z_row, d->B_row, d->C_row})
        if (r < 0 || r > ROW_MOST) return HDLA_ERR_SHAPE;
    s.lpc = lanes_of(d->S);
    const int channels = 64 / s.lpc, size = d->D / d->G;
    s.per_group = (size + channels - 1) / channels;
    s.blocks = d->G * s.per_group;
    s.rows = (long long)d->B * d->T;
    if ((long long)(s.blocks + 8) * d->N > 0x7fffffffLL || s.rows > 0x7fffffffLL) return HDLA_ERR_SHAPE;
    s.every = scan_workgroups(s.blocks, d->N) >= 512 ? SS_TILE_MANY : SS_TILE_FEW;
    s.ckpt = ckpt_slots(d->cu_seqlens != nullptr, d->T, d->N, s.every);
    s.slots = 1;
    s.seg = 0;
    s.units = d->N;
    return HDLA_OK;
}
// Loads of V elements (channels) and of four (states): where everything lies on multiples of them
inline bool scan_vec(const hdla_scan_dims* d, const ScanPlan& s, const ScanArgs& a) {
    const int es = d->dtype == HDLA_BF16 ? 2 : 4, v = std::max(1, SS_TOK / s.lpc), size = d->D / d->G;
    if (size % v || d->S % 4) return false;
    const int bytes = std::min(v * es, 16);
    for (const Operand* o : {&a.x, &a.dt, &a.z})
        if (o->p && (!fits(o->p, bytes) || o->batch % v || o->row % v)) return false;
    if (a.B_group % 4 || a.C_group % 4) return false;
    for (const Operand* o : {&a.B, &a.C})
        if (!fits(o->p, 4 * es) || o->batch % 4 || o->row % 4) return false;
    return true;
}

inline ScanArgs scan_args(const hdla_scan_dims* d, const ScanPlan& s, const void* x, const void* dt, const void* A, const void* B, const void* C, const void* D,
                          const void* z, const void* bias) {
    ScanArgs a{};
    a.x = {x, d->x_batch, d->x_row}; a.dt = {dt, d->dt_batch, d->dt_row}; a.z = {z, d->z_batch, d->z_row};
    a.B = {B, d->B_batch, d->B_row}; a.C = {C, d->C_batch, d->C_row};
    a.A = A; a.D = D; a.bias = bias;
    a.B_group = d->B_group; a.C_group = d->C_group;
    a.A_f32 = d->A_dtype == HDLA_FP32; a.D_f32 = d->D_dtype == HDLA_FP32; a.bias_f32 = d->bias_dtype == HDLA_FP32;
    a.cu = d->cu_seqlens; a.T = d->T; a.N = d->N; a.DD = d->D; a.S = d->S; a.G = d->G; a.softplus = d->softplus != 0;
    a.per_group = s.per_group; a.blocks = s.blocks; a.every_log2 = s.every == SS_TILE_MANY ? 5 : 6; a.rows = s.rows; a.slots = s.slots;
    a.seg = s.seg; a.units = (int)s.units;
    return a;
}

}  // namespace hdla
