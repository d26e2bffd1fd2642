// A linear attention with one decay for each head: what its kernels share (head_decay.cu, head_decay_tc.cu).
//
//   S_t = e^{g_t} S_{t-1} + k_t v_t^T;    o_t = scale S_t^T q_t          S [dim, vdim] per (sequence, head), float
//
// A sequence's tokens are cut into segments.  With c_i = g_1 + .. + g_i counted from a segment's start and the state S_0 there:
//
//   o_i = scale (e^{c_i} S_0^T q_i + sum_{j <= i} e^{c_i - c_j} (q_i . k_j) v_j)
//   S_L = e^{c_L} S_0 + U,    U = sum_j e^{c_L - c_j} k_j v_j^T
//
// Only S_0 -> S_L has to follow one another.  So: every segment's U side by side, a pass over the segments of a (sequence, head)
// that leaves S_0 where each U was, and every segment's outputs side by side.
#pragma once
#include "common.cuh"

#define HD_MAX_DIM 256

struct HeadDecayArgs {
    const void *q, *k, *v, *gate;   // rows of [H dim], [G dim], [G vdim], [H vdim]; gate and norm may be null (together)
    const float* g;                 // [nt or 1, H] logarithms of the decays
    const float* norm;              // [H vdim]
    const float* state;             // [n_slots] rows of [H, dim, vdim]
    float* new_state;               // may be `state`
    void* out;                      // rows of [H vdim]
    const int *seq_start, *slots;
    float* work;                    // [heads of a portion][max_segs][dim][vdim]: U, then S_0
    float* seg_g;                   // [heads of a portion][max_segs]: c_L
    long long ldq, ldk, ldv, ldgate, ldo, pitch, new_pitch;
    long long g_stride;             // 0: one row of decays for all tokens
    int nt, B, H, G, dim, vdim, n_slots, max_segs, seg;
    int h0, heads;                  // the portion's first head and its heads
    float scale, eps;
};

// The logarithm of a decay as the kernels take it: above 0 counts as 0; at -104 e^g is below every float, so nothing is lost
// by that floor, and infinities stay out of the sums.  NaN stays NaN.
__device__ __forceinline__ float hd_log_decay(float g) { return g < -104.f ? -104.f : g > 0.f ? 0.f : g; }

struct HdSegment {
    int b, t0, n, first;            // sequence (-1: none), first token in the step, tokens, and the number of its sequence's first segment
};

// The numbers of a sequence's segments start at seq_start[b] / seg + b: these are far enough apart (its ceil(n / seg) segments end
// before (seq_start[b] + n) / seg + b + 1), below nt / seg + B, and ascend with b, so a warp finds the sequence of a segment
// 32 guesses at a time.  All lanes of a warp call; sequences whose bounds or slot are not what they may be are left out.
__device__ __forceinline__ bool hd_sequence(const HeadDecayArgs& p, int b, int& t0, int& n, int& slot) {
    t0 = p.seq_start[b];
    n = p.seq_start[b + 1] - t0;
    slot = p.slots[b];
    return t0 >= 0 && n >= 0 && n <= p.nt - t0 && slot >= 0 && slot < p.n_slots;
}
__device__ __forceinline__ HdSegment hd_find(const HeadDecayArgs& p, int x) {
    const int lane = threadIdx.x & 31;
    int lo = 0, size = p.B;
    while (size > 1) {
        const int step = (size + 31) / 32, b = lo + lane * step;
        const bool before = lane * step < size && p.seq_start[b] / p.seg + b <= x;
        const int n = max(1, __popc(__ballot_sync(0xffffffffu, before)));
        lo += (n - 1) * step;
        size = min(step, p.B - lo);
    }
    HdSegment s{-1, 0, 0, 0};
    int t0, n, slot;
    if (!hd_sequence(p, lo, t0, n, slot)) return s;
    const int i = x - (t0 / p.seg + lo);
    if (i < 0 || (long long)i * p.seg >= n) return s;
    s.b = lo;
    s.t0 = t0 + i * p.seg;
    s.n = min(p.seg, n - i * p.seg);
    s.first = t0 / p.seg + lo;
    return s;
}

// A sum held as a float and what its rounding left: differences of far sums of strong decays keep their last bits.
struct HdSum {
    float hi, lo;
};
__device__ __forceinline__ float hd_minus(HdSum a, HdSum b) { return (a.hi - b.hi) + (a.lo - b.lo); }

// c_i for the n <= 64 tokens from t0 on, by the first warp; the others wait at the caller's barrier.  In 64 bits.
__device__ __forceinline__ void hd_sums(const HeadDecayArgs& p, int h, int t0, int n, HdSum* c) {
    if (threadIdx.x >= 32) return;
    const int lane = threadIdx.x;
    float g[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) g[u] = p.g[(size_t)(p.g_stride ? t0 + min(lane + 32 * u, n - 1) : 0) * p.g_stride + h];
    double x[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) x[u] = lane + 32 * u < n ? (double)hd_log_decay(g[u]) : 0.0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const double v = __shfl_up_sync(0xffffffffu, x[u], o);
            if (lane >= o) x[u] += v;
        }
    x[1] += __shfl_sync(0xffffffffu, x[0], 31);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const float hi = (float)x[u];
        if (lane + 32 * u < n) c[lane + 32 * u] = HdSum{hi, (float)(x[u] - (double)hi)};
    }
}

// Segments of B sequences of nt tokens in all, at most.
static inline long long hd_segments(int nt, int B, int seg) { return (long long)nt / seg + B; }

// What every launcher asks of its sizes.
static inline int hd_check(const HeadDecayArgs& p) {
    if (p.nt < 0 || p.B < 0 || p.H <= 0 || p.G <= 0 || p.H % p.G || p.dim <= 0 || p.vdim <= 0 || p.n_slots < 0 ||
        p.ldq < (long long)p.H * p.dim || p.ldk < (long long)p.G * p.dim || p.ldv < (long long)p.G * p.vdim ||
        p.ldo < (long long)p.H * p.vdim || (p.gate && p.ldgate < (long long)p.H * p.vdim) || !p.gate != !p.norm ||
        p.pitch < (long long)p.H * p.dim * p.vdim || p.new_pitch < (long long)p.H * p.dim * p.vdim ||
        (p.g_stride != 0 && p.g_stride < p.H))
        return TB_ERR_ARG;
    if (p.dim > HD_MAX_DIM || p.vdim > HD_MAX_DIM || p.H > 65535) return TB_ERR_UNSUPPORTED;
    return 0;
}
