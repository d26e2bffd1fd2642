// Linear attention with one decay for each head (mathematics: head_decay.cuh), any head sizes up to 256, float or bfloat16.
//
//   hd_update_kernel   a block = a segment x a head x 64 x 64 entries of U
//   hd_pass_kernel     a thread = four (or one) entries of the state of a (sequence, head): walks the segments, leaves S_0 where U was
//   hd_rows_kernel     a block = a segment x a head: scores, outputs, and with a gate the heads' norm
//   hd_rates_kernel    the decays of a mixer whose input makes them
//   hd_short_kernel    the three in one, a block = a sequence x a head, for steps of up to 64 tokens with heads of up to 64
//   hd_step_kernel     one token per sequence: a block = a sequence x a head, the state once through the registers
//
// Segments of 64 tokens: the scores of a segment are one tile in shared memory.  Float throughout.  Bound by latency with few segments (a block of
// 256 threads an SM) and by multiply-adds with many: 2 sequences of 200 to 700 tokens, 8 heads of 96 x 80 in float, update 17, pass 6, rows
// with gate 31 us (59 the call; with plain multiply-adds instead of two an instruction 3 more).
#include "head_decay.cuh"
#include "memory_common.cuh"

#define HD_SEG 64
#define HD_STEP_NT 256
#define HD_STEP_U 16
#define HD_PAD 68               // pitch of a tile of 64 columns

// ROWS x 64 entries of a block of 256 threads, all asked for together; they are stored later, so that a tile is on its way while the one
// before it is multiplied.
template <int ROWS, typename Load>
__device__ __forceinline__ void hd_ask(float (&x)[ROWS / 4], Load load) {
#pragma unroll
    for (int u = 0; u < ROWS / 4; ++u) x[u] = load((int)(threadIdx.x >> 6) + 4 * u, (int)(threadIdx.x & 63));
}
template <int ROWS, typename Store>
__device__ __forceinline__ void hd_put(const float (&x)[ROWS / 4], Store store) {
#pragma unroll
    for (int u = 0; u < ROWS / 4; ++u) store((int)(threadIdx.x >> 6) + 4 * u, (int)(threadIdx.x & 63), x[u]);
}
// r += four entries of a row times four of another, 4 x 4 results a thread
__device__ __forceinline__ void hd_fma16(const float* a_row, const float* b_row, F2 (&r)[4][2]) {
    const float4 a = *reinterpret_cast<const float4*>(a_row), b = *reinterpret_cast<const float4*>(b_row);
    const float av[4] = {a.x, a.y, a.z, a.w};
    F2 b0, b1;
    b0.f = make_float2(b.x, b.y);
    b1.f = make_float2(b.z, b.w);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        F2 x;
        x.f = make_float2(av[i], av[i]);
        r[i][0] = fma2(x, b0, r[i][0]);
        r[i][1] = fma2(x, b1, r[i][1]);
    }
}
__device__ __forceinline__ void hd_zero(F2 (&r)[4][2]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i][0].f = r[i][1].f = make_float2(0.f, 0.f);
}
__device__ __forceinline__ float hd_of(const F2 (&r)[4][2], int i, int l) { return l & 1 ? r[i][l >> 1].f.y : r[i][l >> 1].f.x; }

// ---- U of a segment ----------------------------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(256) hd_update_kernel(const HeadDecayArgs p) {
    pdl_sync();
    __shared__ __align__(16) float ks[32][HD_PAD], vs[32][HD_PAD];
    __shared__ HdSum c[HD_SEG];
    const int h = p.h0 + blockIdx.y;
    const HdSegment s = hd_find(p, blockIdx.x);
    if (s.b < 0) return;
    const int tiles = (p.vdim + 63) / 64, r0 = blockIdx.z / tiles * 64, c0 = blockIdx.z % tiles * 64;
    hd_sums(p, h, s.t0, s.n, c);
    __syncthreads();
    const int kv = h / (p.H / p.G);
    const T* k = static_cast<const T*>(p.k) + (size_t)s.t0 * p.ldk + (size_t)kv * p.dim;
    const T* v = static_cast<const T*>(p.v) + (size_t)s.t0 * p.ldv + (size_t)kv * p.vdim;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const HdSum last = c[s.n - 1];
    F2 acc[4][2];
    hd_zero(acc);
    float kx[8], vx[8];
    auto ask = [&](int j0) {
        hd_ask<32>(kx, [&](int j, int r) { return j0 + j < s.n && r0 + r < p.dim ? ldf(k + (size_t)(j0 + j) * p.ldk + r0 + r) : 0.f; });
        hd_ask<32>(vx, [&](int j, int r) { return j0 + j < s.n && c0 + r < p.vdim ? ldf(v + (size_t)(j0 + j) * p.ldv + c0 + r) : 0.f; });
    };
    ask(0);
    for (int j0 = 0; j0 < s.n; j0 += 32) {
        hd_put<32>(kx, [&](int j, int r, float x) { ks[j][r] = j0 + j < s.n ? x * expf(hd_minus(last, c[j0 + j])) : 0.f; });
        hd_put<32>(vx, [&](int j, int r, float x) { vs[j][r] = x; });
        __syncthreads();
        if (j0 + 32 < s.n) ask(j0 + 32);
#pragma unroll 8
        for (int j = 0; j < 32; ++j) hd_fma16(&ks[j][ty * 4], &vs[j][tx * 4], acc);
        __syncthreads();
    }
    const size_t at = (size_t)blockIdx.y * p.max_segs + blockIdx.x;
    float* u = p.work + at * p.dim * p.vdim;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int l = 0; l < 4; ++l) {
            const int r = r0 + ty * 4 + i, col = c0 + tx * 4 + l;
            if (r < p.dim && col < p.vdim) u[(size_t)r * p.vdim + col] = hd_of(acc, i, l);
        }
    if (blockIdx.z == 0 && threadIdx.x == 0) p.seg_g[at] = last.hi + last.lo;
}

// ---- from segment to segment ---------------------------------------------------------------------------------------
template <int V>
__global__ void __launch_bounds__(256) hd_pass_kernel(const HeadDecayArgs p) {
    pdl_sync();
    const int b = blockIdx.x, h = p.h0 + blockIdx.y, size = p.dim * p.vdim;
    const int e = (blockIdx.z * 256 + threadIdx.x) * V;
    int t0, n, slot;
    if (!hd_sequence(p, b, t0, n, slot) || e >= size) return;
    float S[V];
    dm_load<float, V>(p.state + (size_t)slot * p.pitch + (size_t)h * size + e, S);
    const int segs = (n + p.seg - 1) / p.seg;
    const size_t first = (size_t)blockIdx.y * p.max_segs + t0 / p.seg + b;
    float* w = p.work + first * size + e;
    constexpr int U = 4;
    for (int i0 = 0; i0 < segs; i0 += U) {
        float u[U][V], d[U];
#pragma unroll
        for (int i = 0; i < U; ++i)
            if (i0 + i < segs) {
                dm_load<float, V>(w + (size_t)(i0 + i) * size, u[i]);
                d[i] = p.seg_g[first + i0 + i];
            }
#pragma unroll
        for (int i = 0; i < U; ++i)
            if (i0 + i < segs) {
                dm_store<V>(w + (size_t)(i0 + i) * size, S);
                const float f = expf(d[i]);
#pragma unroll
                for (int l = 0; l < V; ++l) S[l] = S[l] * f + u[i][l];
            }
    }
    dm_store<V>(p.new_state + (size_t)slot * p.new_pitch + (size_t)h * size + e, S);
}

// ---- a segment's outputs --------------------------------------------------------------------------------------------
// The rows of a segment, 4 x 4 a thread and tile of 64 columns, scaled, normed and gated where that is asked for.  A row's gate is asked for
// before the row ahead of it is stored (where registers hold both): behind a store that may change it a load waits for its turn.
template <typename T, int TILES>
__device__ __forceinline__ void hd_leave(const HeadDecayArgs& p, const HdSegment& s, int h, const F2 (&o)[TILES][4][2]) {
    const int vdim = p.vdim, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    T* out = static_cast<T*>(p.out) + (size_t)s.t0 * p.ldo + (size_t)h * vdim;
    const T* gate = static_cast<const T*>(p.gate) + (p.gate ? (size_t)s.t0 * p.ldgate + (size_t)h * vdim : 0);
    constexpr bool AHEAD = TILES <= 2;
    float z[2][TILES][4], nw[TILES][4];
    auto ask = [&](int i) {
        if (!p.gate || ty * 4 + i >= s.n) return;
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int l = 0; l < 4; ++l) {
                const int col = t * 64 + tx * 4 + l;
                if (col < vdim) z[i & 1][t][l] = ldf(gate + (size_t)(ty * 4 + i) * p.ldgate + col);
            }
    };
    if (p.gate)
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int l = 0; l < 4; ++l) {
                const int col = t * 64 + tx * 4 + l;
                if (col < vdim) nw[t][l] = p.norm[(size_t)h * vdim + col];
            }
    if (AHEAD) ask(0);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int qi = ty * 4 + i;
        if (!AHEAD) ask(i);
        else if (i + 1 < 4) ask(i + 1);
        float sq = 0.f;
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int l = 0; l < 4; ++l) {
                const float y = hd_of(o[t], i, l) * p.scale;
                sq += y * y;
            }
#pragma unroll
        for (int m = 8; m > 0; m >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, m);
        if (qi >= s.n) continue;
        const float rs = 1.0f / sqrtf(sq / (float)vdim + p.eps);
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int l = 0; l < 4; ++l) {
                const int col = t * 64 + tx * 4 + l;
                if (col >= vdim) continue;
                float y = hd_of(o[t], i, l) * p.scale;
                if (p.gate) y = y * rs * nw[t][l] * (z[i & 1][t][l] / (1.0f + expf(-z[i & 1][t][l])));
                stf(out + (size_t)qi * p.ldo + col, y);
            }
    }
}

// o += P V for n keys, P by [key][query].  The keys that all four of this thread's rows see, and the last three one row after the other: a
// weight of 0 is not multiplied with a value that may be no number.
__device__ __forceinline__ void hd_weigh(const float* p_s, const float* v_s, int n, F2 (&o)[4][2]) {
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4, whole = min(n, ty * 4 + 1);
    if (ty * 4 >= n) return;
#pragma unroll 4
    for (int j = 0; j < whole; ++j) hd_fma16(p_s + j * HD_PAD + ty * 4, v_s + j * HD_PAD + tx * 4, o);
#pragma unroll
    for (int c1 = 1; c1 < 4; ++c1) {
        const int j = ty * 4 + c1;
        if (j >= n) break;
        const float4 b = *reinterpret_cast<const float4*>(v_s + j * HD_PAD + tx * 4);
        F2 b0, b1;
        b0.f = make_float2(b.x, b.y);
        b1.f = make_float2(b.z, b.w);
#pragma unroll
        for (int i = c1; i < 4; ++i) {
            F2 w;
            const float x = p_s[j * HD_PAD + ty * 4 + i];
            w.f = make_float2(x, x);
            o[i][0] = fma2(w, b0, o[i][0]);
            o[i][1] = fma2(w, b1, o[i][1]);
        }
    }
}

// 16 x 16 threads, 4 x 4 results each; columns 64 at a time.  TILES: tiles of 64 columns of vdim.
// `c`: shared memory for the segment's sums, which are made here.  S: the state that the segment starts with.
template <typename T, int TILES>
__device__ __forceinline__ void hd_rows(const HeadDecayArgs& p, const HdSegment& s, int h, const float* S, float* hd_sm, HdSum* c) {
    const int dim = p.dim, vdim = p.vdim;
    float* q_s = hd_sm;                          // [dim][HD_PAD]: q transposed, by token
    float* p_s = q_s + (size_t)dim * HD_PAD;     // [HD_SEG][HD_PAD]: weights transposed, [key][query]
    float* x_s = p_s + HD_SEG * HD_PAD;          // [64][HD_PAD]: keys transposed, states, values
    const int kv = h / (p.H / p.G);
    const T* q = static_cast<const T*>(p.q) + (size_t)s.t0 * p.ldq + (size_t)h * dim;
    const T* k = static_cast<const T*>(p.k) + (size_t)s.t0 * p.ldk + (size_t)kv * dim;
    const T* v = static_cast<const T*>(p.v) + (size_t)s.t0 * p.ldv + (size_t)kv * vdim;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    float x[HD_SEG / 4];                // the tile that comes next
    auto ask_q = [&](int d0) { hd_ask<HD_SEG>(x, [&](int i, int r) { return i < s.n && d0 + r < dim ? ldf(q + (size_t)i * p.ldq + d0 + r) : 0.f; }); };
    auto ask_k = [&](int d0) { hd_ask<HD_SEG>(x, [&](int j, int r) { return j < s.n && d0 + r < dim ? ldf(k + (size_t)j * p.ldk + d0 + r) : 0.f; }); };
    auto ask_s = [&](int c0, int d0) {
        hd_ask<HD_SEG>(x, [&](int r, int col) { return d0 + r < dim && c0 + col < vdim ? S[(size_t)(d0 + r) * vdim + c0 + col] : 0.f; });
    };
    auto ask_v = [&](int c0) { hd_ask<HD_SEG>(x, [&](int j, int col) { return j < s.n && c0 + col < vdim ? ldf(v + (size_t)j * p.ldv + c0 + col) : 0.f; }); };
    ask_q(0);
    hd_sums(p, h, s.t0, s.n, c);
    for (int d0 = 0; d0 < dim; d0 += 64) {
        hd_put<HD_SEG>(x, [&](int i, int r, float y) { if (d0 + r < dim) q_s[(d0 + r) * HD_PAD + i] = y; });
        if (d0 + 64 < dim) ask_q(d0 + 64);
    }
    // scores, rows = queries ty * 4 .., columns = keys tx * 4 ..
    F2 acc[4][2];
    hd_zero(acc);
    ask_k(0);
    for (int d0 = 0; d0 < dim; d0 += 64) {
        const int here = min(64, dim - d0);
        hd_put<HD_SEG>(x, [&](int j, int r, float y) { x_s[r * HD_PAD + j] = y; });
        __syncthreads();
        if (d0 + 64 < dim) ask_k(d0 + 64);
        else ask_s(0, 0);
#pragma unroll 4
        for (int r = 0; r < here; ++r) hd_fma16(q_s + (size_t)(d0 + r) * HD_PAD + ty * 4, x_s + r * HD_PAD + tx * 4, acc);
        __syncthreads();
    }
    // a query sees the keys up to its own; the others' weights are 0 and their values are not multiplied at all
#pragma unroll
    for (int l = 0; l < 4; ++l) {
        const int j = tx * 4 + l;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int qi = ty * 4 + i;
            p_s[j * HD_PAD + qi] = j <= qi && qi < s.n ? hd_of(acc, i, l) * expf(hd_minus(c[qi], c[j])) : 0.f;
        }
    }
    float from_start[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) from_start[i] = ty * 4 + i < s.n ? expf(c[ty * 4 + i].hi + c[ty * 4 + i].lo) : 0.f;
    F2 o[TILES][4][2];
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
        const int c0 = t * 64;
        hd_zero(o[t]);
        if (c0 >= vdim) continue;
        for (int d0 = 0; d0 < dim; d0 += 64) {
            const int here = min(64, dim - d0);
            hd_put<HD_SEG>(x, [&](int r, int col, float y) { x_s[r * HD_PAD + col] = y; });
            __syncthreads();
            if (d0 + 64 < dim) ask_s(c0, d0 + 64);
            else ask_v(c0);
#pragma unroll 4
            for (int r = 0; r < here; ++r) hd_fma16(q_s + (size_t)(d0 + r) * HD_PAD + ty * 4, x_s + r * HD_PAD + tx * 4, o[t]);
            __syncthreads();
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            F2 f;
            f.f = make_float2(from_start[i], from_start[i]);
            o[t][i][0] = mul2(o[t][i][0], f);
            o[t][i][1] = mul2(o[t][i][1], f);
        }
        hd_put<HD_SEG>(x, [&](int j, int col, float y) { x_s[j * HD_PAD + col] = y; });
        __syncthreads();
        if (t + 1 < TILES && c0 + 64 < vdim) ask_s(c0 + 64, 0);
        hd_weigh(p_s, x_s, s.n, o[t]);
        __syncthreads();
    }
    hd_leave<T, TILES>(p, s, h, o);
}

template <typename T, int TILES>
__global__ void __launch_bounds__(256, 2) hd_rows_kernel(const HeadDecayArgs p) {
    pdl_sync();
    extern __shared__ __align__(16) float hd_sm[];
    __shared__ HdSum c[HD_SEG];
    const HdSegment s = hd_find(p, blockIdx.x);
    if (s.b < 0) return;
    hd_rows<T, TILES>(p, s, p.h0 + blockIdx.y, p.work + ((size_t)blockIdx.y * p.max_segs + blockIdx.x) * p.dim * p.vdim, hd_sm, c);
}

// ---- a step of up to 64 tokens, heads of up to 64 entries: all of a (sequence, head) in one block --------------------
// Every sequence is one segment, and q, k, v and the state are a tile each: asked for together, multiplied from shared memory.
template <typename T>
__global__ void __launch_bounds__(256) hd_short_kernel(const HeadDecayArgs p) {
    pdl_sync();
    extern __shared__ __align__(16) float hd_sm[];
    __shared__ HdSum c[HD_SEG];
    __shared__ float w_s[HD_SEG];
    const int b = blockIdx.x, h = blockIdx.y, dim = p.dim, vdim = p.vdim, size = dim * vdim;
    int t0, n, slot;
    if (!hd_sequence(p, b, t0, n, slot)) return;
    const float* S = p.state + (size_t)slot * p.pitch + (size_t)h * size;
    float* N = p.new_state + (size_t)slot * p.new_pitch + (size_t)h * size;
    if (n == 0) {
        for (int e = threadIdx.x; e < size; e += 256) N[e] = S[e];
        return;
    }
    constexpr int TILE = HD_SEG * HD_PAD;
    float *q_s = hd_sm, *k_t = q_s + TILE, *k_s = k_t + TILE, *v_s = k_s + TILE, *s_s = v_s + TILE, *p_s = s_s + TILE;     // [entry][token] the first two
    const int kv = h / (p.H / p.G), tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const T* q = static_cast<const T*>(p.q) + (size_t)t0 * p.ldq + (size_t)h * dim;
    const T* k = static_cast<const T*>(p.k) + (size_t)t0 * p.ldk + (size_t)kv * dim;
    const T* v = static_cast<const T*>(p.v) + (size_t)t0 * p.ldv + (size_t)kv * vdim;
    {
        float xq[HD_SEG / 4], xk[HD_SEG / 4], xv[HD_SEG / 4], xs[HD_SEG / 4];
        hd_ask<HD_SEG>(xq, [&](int j, int r) { return j < n && r < dim ? ldf(q + (size_t)j * p.ldq + r) : 0.f; });
        hd_ask<HD_SEG>(xk, [&](int j, int r) { return j < n && r < dim ? ldf(k + (size_t)j * p.ldk + r) : 0.f; });
        hd_ask<HD_SEG>(xs, [&](int r, int col) { return r < dim && col < vdim ? S[(size_t)r * vdim + col] : 0.f; });
        hd_ask<HD_SEG>(xv, [&](int j, int col) { return j < n && col < vdim ? ldf(v + (size_t)j * p.ldv + col) : 0.f; });
        hd_sums(p, h, t0, n, c);
        hd_put<HD_SEG>(xq, [&](int j, int r, float x) { q_s[r * HD_PAD + j] = x; });
        hd_put<HD_SEG>(xk, [&](int j, int r, float x) { k_t[r * HD_PAD + j] = k_s[j * HD_PAD + r] = x; });
        hd_put<HD_SEG>(xs, [&](int r, int col, float x) { s_s[r * HD_PAD + col] = x; });
        hd_put<HD_SEG>(xv, [&](int j, int col, float x) { v_s[j * HD_PAD + col] = x; });
    }
    __syncthreads();
    const HdSum last = c[n - 1];
    if (threadIdx.x < n) w_s[threadIdx.x] = expf(hd_minus(last, c[threadIdx.x]));
    F2 acc[4][2], o[1][4][2];
    hd_zero(acc);
    hd_zero(o[0]);
    if (ty * 4 < n) {
#pragma unroll 4
        for (int r = 0; r < dim; ++r) {
            hd_fma16(q_s + r * HD_PAD + ty * 4, k_t + r * HD_PAD + tx * 4, acc);
            hd_fma16(q_s + r * HD_PAD + ty * 4, s_s + r * HD_PAD + tx * 4, o[0]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int qi = ty * 4 + i;
            const float f = qi < n ? expf(c[qi].hi + c[qi].lo) : 0.f;
            F2 f2;
            f2.f = make_float2(f, f);
            o[0][i][0] = mul2(o[0][i][0], f2);
            o[0][i][1] = mul2(o[0][i][1], f2);
#pragma unroll
            for (int l = 0; l < 4; ++l) {
                const int j = tx * 4 + l;
                p_s[j * HD_PAD + qi] = j <= qi && qi < n ? hd_of(acc, i, l) * expf(hd_minus(c[qi], c[j])) : 0.f;
            }
        }
    }
    __syncthreads();
    hd_weigh(p_s, v_s, n, o[0]);
    hd_zero(acc);
    if (ty * 4 < dim && tx * 4 < vdim) {
#pragma unroll 4
        for (int j = 0; j < n; ++j) {
            const float4 a = *reinterpret_cast<const float4*>(k_s + j * HD_PAD + ty * 4);
            const float w = w_s[j], row[4] = {a.x * w, a.y * w, a.z * w, a.w * w};
            const float4 x = *reinterpret_cast<const float4*>(v_s + j * HD_PAD + tx * 4);
            F2 b0, b1;
            b0.f = make_float2(x.x, x.y);
            b1.f = make_float2(x.z, x.w);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                F2 y;
                y.f = make_float2(row[i], row[i]);
                acc[i][0] = fma2(y, b0, acc[i][0]);
                acc[i][1] = fma2(y, b1, acc[i][1]);
            }
        }
        const float f = expf(last.hi + last.lo);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int l = 0; l < 4; ++l) {
                const int r = ty * 4 + i, col = tx * 4 + l;
                if (r < dim && col < vdim) N[(size_t)r * vdim + col] = f * s_s[r * HD_PAD + col] + hd_of(acc, i, l);
            }
    }
    hd_leave<T, 1>(p, HdSegment{b, t0, n, 0}, h, o);
}

// ---- one token per sequence ---------------------------------------------------------------------------------------
// The state goes through the registers once, S' = e^g S + k v^T and its q^T S' on the way: bound by memory.  16 rows of 256 threads in flight, read and
// written past the caches that others use: 64 sequences of 32 heads of 128 x 128 45 us, 6.0 TB/s (512 threads 63 us, 1,024 67); one
// sequence 6 us.
// V: columns a thread and access (four where rows and heads are whole 16-byte pieces); NT threads, U rows asked for together.
template <typename T, int V, int NT, int U>
__global__ void __launch_bounds__(NT) hd_step_kernel(const HeadDecayArgs p) {
    extern __shared__ __align__(16) float hd_sm[];
    __shared__ float red[33];
    const int b = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, dim = p.dim, vdim = p.vdim;
    const int nc = vdim / V, R = NT / nc;   // columns' threads, groups of rows
    const int vp = (vdim + 3) / 4 * 4;
    float* q_s = hd_sm;                     // [dim] each
    float* k_s = q_s + dim;
    float* o_s = hd_sm + (2 * dim + 3) / 4 * 4;     // [R][vp]
    pdl_sync();
    const int slot = p.slots[b];
    if (slot < 0 || slot >= p.n_slots) return;
    const int rg = tid / nc, c = (tid - rg * nc) * V;
    const float* S = p.state + (size_t)slot * p.pitch + (size_t)h * dim * vdim;
    float* N = p.new_state + (size_t)slot * p.new_pitch + (size_t)h * dim * vdim;
    float s[U][V];
    auto fetch = [&](int r0) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (r0 + u * R < dim) {
                const float* at = S + (size_t)(r0 + u * R) * vdim + c;
                if constexpr (V == 4) {
                    const float4 f = __ldcs(reinterpret_cast<const float4*>(at));       // read once
                    s[u][0] = f.x; s[u][1] = f.y; s[u][2] = f.z; s[u][3] = f.w;
                } else {
                    s[u][0] = __ldcs(at);
                }
            }
    };
    if (rg < R) fetch(rg);
    const int kv = h / (p.H / p.G);
    const T* q = static_cast<const T*>(p.q) + (size_t)b * p.ldq + (size_t)h * dim;
    const T* k = static_cast<const T*>(p.k) + (size_t)b * p.ldk + (size_t)kv * dim;
    if (tid < dim) {
        q_s[tid] = ldf(q + tid) * p.scale;
        k_s[tid] = ldf(k + tid);
    }
    const float decay = expf(hd_log_decay(p.g[(size_t)b * p.g_stride + h]));
    float v[V] = {};
    if (rg < R) {
        const T* vr = static_cast<const T*>(p.v) + (size_t)b * p.ldv + (size_t)kv * vdim + c;
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = ldf(vr + e);
    }
    float gate = 0.f, nw = 0.f;
    if (p.gate && tid < vdim) {
        gate = ldf(static_cast<const T*>(p.gate) + (size_t)b * p.ldgate + (size_t)h * vdim + tid);
        nw = p.norm[(size_t)h * vdim + tid];
    }
    __syncthreads();
    if (rg < R) {
        float acc[V] = {};
        for (int r0 = rg; r0 < dim; r0 += R * U) {
            if (r0 != rg) fetch(r0);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int r = r0 + u * R;
                if (r >= dim) break;
                const float qq = q_s[r], kk = k_s[r];
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    s[u][e] = s[u][e] * decay + kk * v[e];
                    acc[e] += s[u][e] * qq;
                }
                float* at = N + (size_t)r * vdim + c;
                if constexpr (V == 4) __stcs(reinterpret_cast<float4*>(at), make_float4(s[u][0], s[u][1], s[u][2], s[u][3]));
                else __stcs(at, s[u][0]);
            }
        }
#pragma unroll
        for (int e = 0; e < V; ++e) o_s[rg * vp + c + e] = acc[e];
    }
    __syncthreads();
    float o = 0.f;
    if (tid < vdim)
        for (int i = 0; i < R; ++i) o += o_s[i * vp + tid];
    if (p.gate) {
        const float rs = 1.0f / sqrtf(block_sum(o * o, red) / (float)vdim + p.eps);
        o *= rs * nw * (gate / (1.0f + expf(-gate)));
    }
    if (tid < vdim) stf(static_cast<T*>(p.out) + (size_t)b * p.ldo + (size_t)h * vdim + tid, o);
}

// ---- g = -exp(rate) softplus(a + bias) -----------------------------------------------------------------------------
__global__ void __launch_bounds__(256) hd_rates_kernel(const float* __restrict__ a, const float* __restrict__ rate,
                                                       const float* __restrict__ bias, float* __restrict__ g, int n, int H) {
    pdl_sync();
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const float z = a[i] + bias[i % H];
    g[i] = -expf(rate[i % H]) * (fmaxf(z, 0.f) + log1pf(expf(-fabsf(z))));
}

// ---- launchers ------------------------------------------------------------------------------------------------------
// Four entries of the states an access: rows, heads and slots are whole 16-byte pieces.
static bool hd_fours(const HeadDecayArgs& p) {
    return p.vdim % 4 == 0 && p.pitch % 4 == 0 && p.new_pitch % 4 == 0 && (((uintptr_t)p.state | (uintptr_t)p.new_state) & 15) == 0;
}

template <typename T, int TILES>
static void hd_rows_launch(const HeadDecayArgs& p, cudaStream_t s) {
    const size_t smem = ((size_t)p.dim + HD_SEG + 64) * HD_PAD * sizeof(float);
    static PerDevice allowed;
    tb_allow_smem(allowed, (const void*)hd_rows_kernel<T, TILES>, ((size_t)HD_MAX_DIM + HD_SEG + 64) * HD_PAD * sizeof(float));
    TB_LAUNCH((hd_rows_kernel<T, TILES>), dim3(p.max_segs, p.heads), 256, smem, s, p);
}
// One kernel instead of three, and no scratch.  us of a call among others / of the kernels alone in a graph, this kernel and the three, heads
// of 64 x 64: bfloat16 (the three on tcgen05), 8 heads, 8 tokens 15 / 9.7 and 24 / 13.5, 33 tokens 15 / 13.3 and 24 / 14.0, 64 tokens 17 / 16.7
// and 24 / 13.9; 32 heads, 64 tokens in 8 sequences 15 / 11.4 and 26 / 24.6, in 32 sequences 35 / 34.9 and 64 / 62.9; float, 8 heads, 33 tokens
// 15 / 11.1 and 22 / 19.5, 64 tokens 15 / 13.4 and 22 / 20.4, 32 heads in 32 sequences 33 / 33.1 and 70 / 69.1.  Where only the kernels
// count, one bfloat16 sequence of more than some 35 tokens would have up to 4.5 us less with the three; prompts are calls, which are 7 us less with one.
static bool hd_is_short(int nt, int dim, int vdim) { return nt <= HD_SEG && dim <= 64 && vdim <= 64; }

// work: floats of scratch, `heads` heads of it (max_segs (dim vdim + 1) each); that many heads are done together.
template <typename T>
static int hd_prompt_launch(HeadDecayArgs p, int heads, cudaStream_t s) {
    const int rc = hd_check(p);
    if (rc) return rc;
    if (heads <= 0 || ((uintptr_t)p.work & 15)) return TB_ERR_ARG;
    if (p.B == 0) return 0;
    p.seg = HD_SEG;
    if (hd_is_short(p.nt, p.dim, p.vdim)) {
        constexpr size_t smem = 6 * (size_t)HD_SEG * HD_PAD * sizeof(float);
        static PerDevice allowed;
        tb_allow_smem(allowed, (const void*)hd_short_kernel<T>, smem);
        TB_LAUNCH((hd_short_kernel<T>), dim3(p.B, p.H), 256, smem, s, p);
        return tb_last_error();
    }
    const long long segs = hd_segments(p.nt, p.B, p.seg);
    if (p.max_segs < segs) return TB_ERR_ARG;
    p.max_segs = (int)segs;
    const int size = p.dim * p.vdim, tiles = ((p.dim + 63) / 64) * ((p.vdim + 63) / 64);
    p.seg_g = p.work + (size_t)heads * p.max_segs * size;
    for (p.h0 = 0; p.h0 < p.H; p.h0 += heads) {
        const int here = p.H - p.h0 < heads ? p.H - p.h0 : heads;
        p.heads = here;
        if (p.nt) TB_LAUNCH((hd_update_kernel<T>), dim3(p.max_segs, here, tiles), 256, 0, s, p);
        if (hd_fours(p)) TB_LAUNCH((hd_pass_kernel<4>), dim3(p.B, here, (size / 4 + 255) / 256), 256, 0, s, p);
        else TB_LAUNCH((hd_pass_kernel<1>), dim3(p.B, here, (size + 255) / 256), 256, 0, s, p);
        if (!p.nt) continue;        // sequences without tokens: their states alone
        if (p.vdim <= 64) hd_rows_launch<T, 1>(p, s);
        else if (p.vdim <= 128) hd_rows_launch<T, 2>(p, s);
        else hd_rows_launch<T, 4>(p, s);
    }
    return tb_last_error();
}

template <typename T>
static int hd_step_launch(const HeadDecayArgs& p, cudaStream_t s) {
    const int rc = hd_check(p);
    if (rc) return rc;
    if (p.B == 0) return 0;
    const bool four = hd_fours(p);
    constexpr int NT = HD_STEP_NT;
    const int R = NT / (p.vdim / (four ? 4 : 1)), vp = (p.vdim + 3) / 4 * 4;
    const size_t smem = ((2 * (size_t)p.dim + 3) / 4 * 4 + (size_t)R * vp) * sizeof(float);
    if (four) TB_LAUNCH((hd_step_kernel<T, 4, NT, HD_STEP_U>), dim3(p.B, p.H), NT, smem, s, p);
    else TB_LAUNCH((hd_step_kernel<T, 1, NT, HD_STEP_U>), dim3(p.B, p.H), NT, smem, s, p);
    return tb_last_error();
}

extern "C" {
// 0: one kernel does all, no scratch is wanted.  -1: more segments than 32 bits count.
int tb_head_decay_segments(int nt, int B, int dim, int vdim) {
    const long long segs = hd_is_short(nt, dim, vdim) ? 0 : hd_segments(nt, B, HD_SEG);
    return segs > 0x7fffffffLL ? -1 : (int)segs;
}

int tb_head_decay_rates(const float* a, const float* rate, const float* bias, float* g, int nt, int H, cudaStream_t s) {
    if (nt < 0 || H <= 0 || (long long)nt * H > 0x7fffffffLL - 256) return TB_ERR_ARG;
    if (nt == 0) return 0;
    TB_LAUNCH((hd_rates_kernel), (nt * H + 255) / 256, 256, 0, s, a, rate, bias, g, nt * H, H);
    return tb_last_error();
}

#define TB_HEAD_DECAY(SFX, T)                                                                                              \
    int tb_head_decay_##SFX(const void* q, const void* k, const void* v, const void* gate, long long ldq, long long ldk,   \
                            long long ldv, long long ldgate, const float* g, long long g_stride, const float* norm,        \
                            const float* state, float* new_state, long long pitch, long long new_pitch, void* out,         \
                            long long ldo, const int* seq_start, const int* slots, float* work, int max_segs, int heads,   \
                            int nt, int B, int H, int G, int dim, int vdim, int n_slots, float scale, float eps,           \
                            cudaStream_t s) {                                                                              \
        return hd_prompt_launch<T>(HeadDecayArgs{q, k, v, gate, g, norm, state, new_state, out, seq_start, slots, work,    \
                                                 nullptr, ldq, ldk, ldv, ldgate, ldo, pitch, new_pitch, g_stride, nt, B,   \
                                                 H, G, dim, vdim, n_slots, max_segs, HD_SEG, 0, H, scale, eps}, heads, s); \
    }                                                                                                                      \
    int tb_head_decay_step_##SFX(const void* q, const void* k, const void* v, const void* gate, long long ldq,             \
                                 long long ldk, long long ldv, long long ldgate, const float* g, long long g_stride,       \
                                 const float* norm, const float* state, float* new_state, long long pitch,                 \
                                 long long new_pitch, void* out, long long ldo, const int* slots, int B, int H, int G,     \
                                 int dim, int vdim, int n_slots, float scale, float eps, cudaStream_t s) {                 \
        return hd_step_launch<T>(HeadDecayArgs{q, k, v, gate, g, norm, state, new_state, out, nullptr, slots, nullptr,     \
                                               nullptr, ldq, ldk, ldv, ldgate, ldo, pitch, new_pitch, g_stride, B, B, H,   \
                                               G, dim, vdim, n_slots, 0, HD_SEG, 0, H, scale, eps}, s);                    \
    }
TB_HEAD_DECAY(f32, float)
TB_HEAD_DECAY(bf16, __nv_bfloat16)
}

#include "tape.h"
TB_TAPE_REGISTER(tb_head_decay_rates)
TB_TAPE_REGISTER(tb_head_decay_f32)
TB_TAPE_REGISTER(tb_head_decay_bf16)
TB_TAPE_REGISTER(tb_head_decay_step_f32)
TB_TAPE_REGISTER(tb_head_decay_step_bf16)
