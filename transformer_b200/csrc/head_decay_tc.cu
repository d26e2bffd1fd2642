// Linear attention with one decay for each head (mathematics: head_decay.cuh): prompts in bfloat16 on the tcgen05 tensor cores, key heads of up
// to 128 entries and value heads of up to 256, in multiples of eight.
//
//   hd_update_tc_kernel   a block = a segment x a head: U = K'^T V (dim x vdim, in tensor memory), K'_j = e^{c_L - c_j} k_j
//   hd_pass_tc_kernel     a thread = four entries of the state of a (sequence, head): walks the segments, leaves S_0 in bfloat16
//   hd_rows_tc_kernel     a block = 128 tokens of a segment x a head: O = e^{c_i} (Q S_0), then += P V for each 128 keys up to its own,
//                         P = (Q K^T) e^{c_i - c_j}; with a gate the heads' norm at the end
//
// The states stay in float: K' is written as three bfloat16s, the value and what its rounding left twice (over K and beside it), and all are
// multiplied with V into the same accumulator, so U has float's error (with two of them 2^-18 of a term may be left out, which showed: the
// states were more than 1e-6 of their norm off).  P, and the copy of S_0 that outputs are made from, are rounded to bfloat16 once: the outputs,
// which are rounded to it themselves, are 2.1e-3 to 2.3e-3 of their norm off 64 bits instead of 1.7e-3.  Each in two bfloat16s they are 1.7e-3 off,
// and a call in a graph takes, with P alone, with S_0 alone and with both so: 2,048 tokens of 32 heads 50, 54 and 55 us for 48; 11,875 in 11
// sequences 253, 267 and 284 for 237; 8,192 of 16 92, 107 and 109 for 89.
// A factor e^{c_i - c_j} is one exponential for a row and 32 keys times one for a key and the end of its 32, both at most 1; inside
// the 32 x 32 on the diagonal, where the first would grow, one exponential each.  P takes its place over the scores in tensor memory (the A
// operand of the second product).  Copies by TMA (3-D maps [tokens, heads, entries]: entries behind a head's are zeros), products issued
// by one warp, eight warps for the rows, two blocks an SM.  Every wait is bounded.
//
// Bound by latency: copies, scores, weights, products and gate of a tile follow one another, some 12,000 clocks of which two blocks an SM (tensor
// memory has room for no third) cover a part.  2,048 tokens of 32 heads of 128 x 128, us: update 18, pass 10, rows with
// gate 30 (the call 50, 1.8 TB/s of what it has to read and write); 11,875 tokens in 11 sequences 79, 40, 131 (238); 8,192 tokens of 16 heads
// 33, 13, 53 (90).
#include <algorithm>

#include "head_decay.cuh"
#include "memory_common.cuh"
#include "tc_common.cuh"

#define HT_TILE 128
#define HT_HALF 64              // rows of a TMA box, and keys that the update takes together
#define HT_TILES 2              // tiles of a segment.  us in a graph with 1 and 2: 2,048 tokens of 32 heads 57 and 48, 11,875 in 11 sequences 293 and
                                // 236, 8,192 of 16 106 and 88 (twice the states' way through memory), 6 narrow sequences 40 and 38; 4 left the
                                // SMs with few long blocks
#define HT_SEG (HT_TILES * HT_TILE)
#define HT_WORKERS 256          // eight warps: two for each 32 lanes of tensor memory, half of the columns each
#define HT_THREADS (64 + HT_WORKERS)
#define HT_LOG2E 1.4426950408889634f

struct HdTcArgs {
    HeadDecayArgs p;
    __nv_bfloat16* starts;          // [heads of a portion][max_segs][dim][vdim]
    float* sums;                    // [heads of a portion][max_segs][HT_RECORD]
    int* error;
    int heads_u, heads_r;           // heads that a block goes through, one after the other
};

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}
__device__ __forceinline__ uint64_t ht_desc(uint32_t smem_addr, uint32_t lbo) {     // MN-major: column boxes lbo apart, 8 rows 1024 bytes
    uint64_t d = 0;
    d |= (uint64_t)((smem_addr & 0x3FFFFu) >> 4);
    d |= (uint64_t)((lbo >> 4) & 0x3FFF) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
__device__ __forceinline__ void ht_fetch_map(const CUtensorMap* map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}
// 16 packed pairs over 16 columns of this thread's lane (tcgen05.wait::st comes before they are handed over)
__device__ __forceinline__ void ht_store16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
        "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void ht_store32(uint32_t taddr, const float (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
        ::"r"(taddr), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]),
        "f"(v[9]), "f"(v[10]), "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15]), "f"(v[16]), "f"(v[17]),
        "f"(v[18]), "f"(v[19]), "f"(v[20]), "f"(v[21]), "f"(v[22]), "f"(v[23]), "f"(v[24]), "f"(v[25]), "f"(v[26]),
        "f"(v[27]), "f"(v[28]), "f"(v[29]), "f"(v[30]), "f"(v[31])
        : "memory");
}
__device__ __forceinline__ float ht_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 128 rows of one head from token t on, in boxes of 64 rows and 64 columns, the columns' boxes HT_TILE rows apart
template <int BOXES>
__device__ __forceinline__ void ht_load_tile(uint32_t dst, const CUtensorMap* map, uint32_t bar, int head, int t) {
#pragma unroll
    for (int b = 0; b < BOXES; ++b)
#pragma unroll
        for (int r = 0; r < HT_TILE; r += HT_HALF) tma_load_3d(dst + b * (HT_TILE * 128) + r * 128, map, bar, b * 64, head, t + r);
}

// y s(z) for two pairs, s(z) = z / (1 + e^-z).  The reciprocal on the multiply-add units, which have time where the exponential unit has
// none, by Newton and Raphson's steps r (2 - x r) from a start that is a subtraction of x's bits (the known piecewise linear approximation
// by a float's exponent and fraction taken as one number): 0x7ef311c0 less the bits of x in [1, 2^116) is 1 / x within 5.1 %, and each step
// squares that (6.7e-6 after two).  Below -80, where s lies between 0 and -1.5e-33, the reciprocal is 0 whatever the steps make of it, so that a
// gate of the type's lowest value closes its channel; times -inf that is no number, as in the other kernels.
__device__ __forceinline__ F2 ht_gated(F2 y, float z0, float z1) {
    F2 z, t, nx, r, m, c;
    z.f = make_float2(z0, z1);
    c.f = make_float2(-HT_LOG2E, -HT_LOG2E);
    t = mul2(z, c);
    t.f = make_float2(ht_ex2(t.f.x), ht_ex2(t.f.y));
    c.f = make_float2(-1.f, -1.f);
    nx = fma2(t, c, c);             // -(1 + e)
    r.f = make_float2(__uint_as_float(0xfef311c0u - __float_as_uint(nx.f.x)), __uint_as_float(0xfef311c0u - __float_as_uint(nx.f.y)));
    c.f = make_float2(2.f, 2.f);
    m = fma2(nx, r, c);
    r = mul2(r, m);
    m = fma2(nx, r, c);
    r = mul2(r, m);
    r.f = make_float2(z0 < -80.f ? 0.f : r.f.x, z1 < -80.f ? 0.f : r.f.y);
    return mul2(y, mul2(z, r));
}

// The decays of a segment's tokens in blocks of 32: e_j = the sum behind token j to its block's end, l_j = up to and with token j from its
// block's start, and the sums before each block in 64 bits, so that no sum of few tokens is a difference of long ones.  The blocks that
// make U leave them in scratch for those that make the outputs: a record of l [seg], e^{e_j} [seg], the sums before the blocks, and a
// number for each of their worker warps that is not 0 if U has an entry that is no number there (which it has in a whole column where a value
// of the segment is none: whatever it is multiplied with, the result is none).  A decay that is none is in e of the tokens before it, which
// only tokens behind it may use: within a block the outputs take l, which has it from its token on.
#define HT_BLOCKS (HT_SEG / 32)
struct alignas(16) HtSums {
    float e[HT_SEG];
    double before[HT_BLOCKS + 2];
};
#define HT_RECORD_BEFORE (2 * HT_SEG)
#define HT_RECORD_BAD (HT_RECORD_BEFORE + 2 * (HT_BLOCKS + 2))
#define HT_RECORD (HT_RECORD_BAD + HT_WORKERS / 32)
#define HT_DECAYS (HT_SEG / HT_WORKERS)         // tokens of a worker
static_assert(HT_SEG % HT_WORKERS == 0 && HT_BLOCKS < 32, "a worker's tokens, and the blocks' sums in one warp");
// This worker's tokens' decays, asked for ahead of ht_sums.
__device__ __forceinline__ void ht_decays(const HeadDecayArgs& p, int h, int t0, int n, int tid, float (&x)[HT_DECAYS]) {
#pragma unroll
    for (int u = 0; u < HT_DECAYS; ++u) x[u] = p.g[(size_t)(p.g_stride ? t0 + min(tid + HT_WORKERS * u, n - 1) : 0) * p.g_stride + h];
}
// By the workers (tid 0..255), which leave together.
__device__ __forceinline__ void ht_sums(const HeadDecayArgs& p, int n, int tid, const float (&x)[HT_DECAYS], HtSums& s, float* __restrict__ record) {
    const int lane = tid & 31;
#pragma unroll
    for (int u = 0; u < HT_DECAYS; ++u) {
        const int i = tid + HT_WORKERS * u;
        float l = i < n ? hd_log_decay(x[u]) : 0.f, e = __shfl_down_sync(0xffffffffu, l, 1);
        if (lane == 31) e = 0.f;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const float a = __shfl_up_sync(0xffffffffu, l, o), b = __shfl_down_sync(0xffffffffu, e, o);
            if (lane >= o) l += a;
            if (lane + o < 32) e += b;
        }
        s.e[i] = e;
        if (lane == 31) s.before[i >> 5] = (double)l;
        record[i] = l;
        record[HT_SEG + i] = ht_ex2(e * HT_LOG2E);
    }
    asm volatile("bar.sync 1, 256;" ::: "memory");
    if (tid < 32) {         // the blocks' sums, to those before each
        double v = lane < HT_BLOCKS ? s.before[lane] : 0.0;
#pragma unroll
        for (int o = 1; o < HT_BLOCKS; o <<= 1) {
            const double a = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += a;
        }
        const double before = __shfl_up_sync(0xffffffffu, v, 1);
        if (lane <= HT_BLOCKS) {
            s.before[lane] = lane ? before : 0.0;
            reinterpret_cast<double*>(record + HT_RECORD_BEFORE)[lane] = lane ? before : 0.0;
        }
    }
    asm volatile("bar.sync 1, 256;" ::: "memory");
}

// ---- U of a segment -----------------------------------------------------------------------------------------------------
// A block takes its segment's heads one after the other, 64 keys at a time: copies (two stages of K and V) and decays run ahead into the
// next head, and a head's U leaves while the next one's keys are multiplied (two accumulators).  What rounding left of K' has room for
// one stage, so the next keys are weighted when the product before them is done.  U has its entries in the order
// [vdim / 4][dim][4]: a warp's 32 rows of four columns are 512 bytes on end.
template <int KB, int VB>
__global__ void __launch_bounds__(HT_THREADS, VB == 4 ? 1 : 2)
hd_update_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const HdTcArgs a) {
    if (threadIdx.x == 0) {
        ht_fetch_map(&map_k);
        ht_fetch_map(&map_v);
    }
    pdl_sync();
    constexpr int DK = KB * 64, DV = VB * 64;
    constexpr uint32_t BOX = HT_HALF * 128, K_BYTES = KB * BOX, V_BYTES = VB * BOX, STAGE = K_BYTES + V_BYTES, TMEM_COLS = 2 * DV;
    extern __shared__ __align__(1024) uint8_t smem_raw[];       // two stages of K (then K') and V; what one and two roundings left of K'
    const HeadDecayArgs& p = a.p;
    const uint32_t base = smem_u32(smem_raw);
    uint8_t* rest = smem_raw + 2 * STAGE;
    uint64_t* bars = reinterpret_cast<uint64_t*>(rest + 2 * K_BYTES);
    HtSums* sums = reinterpret_cast<HtSums*>(bars + 12);        // by the head's parity
    uint32_t& tmem_slot = *reinterpret_cast<uint32_t*>(bars + 11);
    const int warp = warp_number(), lane = threadIdx.x & 31;
    const int at0 = blockIdx.y * a.heads_u;             // of the portion
    const uint32_t bar0 = smem_u32(bars);
    auto full = [&](int s) { return bar0 + 8u * s; };
    auto ready = [&](int s) { return bar0 + 16 + 8u * s; };
    auto empty = [&](int s) { return bar0 + 32 + 8u * s; };
    auto u_full = [&](int s) { return bar0 + 48 + 8u * s; };
    auto u_empty = [&](int s) { return bar0 + 64 + 8u * s; };
    if (base & 1023u) {
        if (threadIdx.x == 0) atomicCAS(a.error, 0, 49);
        return;
    }
    if (threadIdx.x == 0) {
        for (int s = 0; s < 2; ++s) {
            mbar_init(full(s), 1);
            mbar_init(ready(s), HT_WORKERS / 32);
            mbar_init(empty(s), 1);
            mbar_init(u_full(s), 1);
            mbar_init(u_empty(s), HT_WORKERS / 32);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    if (warp == 1) tmem_alloc(smem_u32(&tmem_slot), TMEM_COLS);
    const HdSegment s = hd_find(p, blockIdx.x);
    // no such segment: no heads, so that no warp waits for another
    const int tiles = (s.n + HT_HALF - 1) / HT_HALF, heads = tiles ? min(a.heads_u, p.heads - at0) : 0, steps = tiles * heads;
    auto copy = [&](int it) {
        const int i = it / tiles, t = s.t0 + (it - i * tiles) * HT_HALF, kv = (p.h0 + at0 + i) / (p.H / p.G);
        if (elect_one()) {
            const uint32_t sk = base + (it & 1) * STAGE, sv = sk + K_BYTES;
            mbar_expect_tx(full(it & 1), K_BYTES + V_BYTES);
#pragma unroll
            for (int b = 0; b < KB; ++b) tma_load_3d(sk + b * BOX, &map_k, full(it & 1), b * 64, kv, t);
#pragma unroll
            for (int b = 0; b < VB; ++b) tma_load_3d(sv + b * BOX, &map_v, full(it & 1), b * 64, kv, t);
        }
        __syncwarp();
    };
    // the first copies do not wait for the other warps: this one has made their barriers
    if (warp == 0 && steps > 0) copy(0);
    if (warp == 0 && steps > 1) copy(1);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    if (warp == 0) {
        int issued = min(steps, 2);
        for (int it = 2; it < steps; ++it) {
            if (!mbar_wait_warp(empty(it & 1), ((it >> 1) - 1) & 1, a.error, 41)) break;
            copy(it);
            issued = it + 1;
        }
        if (*(volatile int*)a.error != 0)           // no copy is left under way
            for (int it = max(0, issued - 2); it < issued; ++it) mbar_wait(full(it & 1), (it >> 1) & 1, a.error, 41);
    } else if (warp == 1) {
        // A = K'^T and B = V, both with the tokens along the rows of their tiles (MN-major)
        const uint32_t idesc = umma_idesc(DK, DV) | (1u << 15) | (1u << 16);
        bool ok = true;
        for (int i = 0, it = 0; i < heads && ok; ++i) {
            if (i >= 2) ok = mbar_wait_warp(u_empty(i & 1), ((i >> 1) - 1) & 1, a.error, 42);
            for (int j = 0; j < tiles && ok; ++j, ++it) {
                ok = mbar_wait_warp(ready(it & 1), (it >> 1) & 1, a.error, 42);
                if (!ok) break;
                tc_fence_after();
                if (elect_one()) {
                    const uint32_t sk = base + (it & 1) * STAGE, sv = sk + K_BYTES, sr = base + 2 * STAGE, to = tmem + (i & 1) * DV;
                    const int ks = (min(HT_HALF, s.n - j * HT_HALF) + 15) / 16;
                    for (int k = 0; k < ks; ++k) {
                        const uint64_t dv = ht_desc(sv + k * 2048, BOX);
                        umma_bf16(to, ht_desc(sk + k * 2048, BOX), dv, idesc, (j | k) != 0);
                        umma_bf16(to, ht_desc(sr + k * 2048, BOX), dv, idesc, 1);
                        umma_bf16(to, ht_desc(sr + K_BYTES + k * 2048, BOX), dv, idesc, 1);
                    }
                    umma_commit(empty(it & 1));
                    if (j == tiles - 1) umma_commit(u_full(i & 1));
                }
                __syncwarp();
            }
        }
    } else if (steps > 0) {
        const int tid = threadIdx.x - 64, quad = warp & 3, key = tid & 63, part = tid >> 6;
        bool ok = true;
        float x[HT_DECAYS];
        ht_decays(p, p.h0 + at0, s.t0, s.n, tid, x);
        auto leave = [&](int i) {           // U of head i
            ok = ok && mbar_wait_warp(u_full(i & 1), (i >> 1) & 1, a.error, 44);
            tc_fence_after();
            if (!ok) return;
            // accumulators of 64 rows lie in the first 16 lanes of each warp's 32
            const size_t at = (size_t)(at0 + i) * p.max_segs + blockIdx.x;
            const int r = DK == 128 ? quad * 32 + lane : quad * 16 + lane, c_lo = (tid >> 7) * (DV / 2);
            const bool mine = r < p.dim && (DK == 128 || lane < 16);
            float4* u = reinterpret_cast<float4*>(p.work + at * p.dim * p.vdim) + r;
            float bad = 0.f;            // 0 times the entries: 0, or NaN
#pragma unroll 1
            for (int c0 = c_lo; c0 < c_lo + DV / 2; c0 += 32) {
                float o[32];
                tmem_ld32(tmem + (i & 1) * DV + ((uint32_t)(quad * 32) << 16) + c0, o);
                if (mine) {
#pragma unroll
                    for (int e = 0; e < 32; ++e) bad = fmaf(o[e], 0.f, bad);
#pragma unroll
                    for (int e = 0; e < 32; e += 4)
                        if (c0 + e < p.vdim) u[(size_t)((c0 + e) >> 2) * p.dim] = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                }
            }
            const bool some = __any_sync(0xffffffffu, !(bad == 0.f));
            if (lane == 0) a.sums[at * HT_RECORD + HT_RECORD_BAD + (tid >> 5)] = some ? 1.f : 0.f;
            tc_fence_before();
            __syncwarp();
            if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(u_empty(i & 1)) : "memory");
        };
        for (int i = 0, it = 0; i < heads; ++i) {
            HtSums& sum = sums[i & 1];
            const size_t at = (size_t)(at0 + i) * p.max_segs + blockIdx.x;
            ht_sums(p, s.n, tid, x, sum, a.sums + at * HT_RECORD);
            if (i + 1 < heads) ht_decays(p, p.h0 + at0 + i + 1, s.t0, s.n, tid, x);
            const double end = sum.before[(s.n + 31) / 32];
            for (int j = 0; j < tiles; ++j, ++it) {
                ok = ok && mbar_wait_warp(full(it & 1), (it >> 1) & 1, a.error, 43);
                if (it > 0) ok = ok && mbar_wait_warp(empty(~it & 1), ((it - 1) >> 1) & 1, a.error, 43);
                if (!ok) continue;
                const int token = j * HT_HALF + key;
                const bool there = token < s.n;
                const float w = there ? expf(sum.e[token] + (float)(end - sum.before[(token >> 5) + 1])) : 0.f;
                F2 w2;
                w2.f = make_float2(w, w);
                uint8_t *row = smem_raw + (it & 1) * STAGE + key * 128, *left = rest + key * 128;
                // four threads a key, a quarter of its 16-byte pieces each
#pragma unroll
                for (int c = 0; c < 2 * KB; ++c) {
                    const int piece = part * 2 * KB + c;
                    const int offset = (piece >> 3) * BOX + (((piece & 7) ^ (key & 7)) << 4);
                    uint4* here = reinterpret_cast<uint4*>(row + offset);
                    const uint4 raw = there ? *here : make_uint4(0u, 0u, 0u, 0u);
                    const uint32_t in[4] = {raw.x, raw.y, raw.z, raw.w};
                    uint32_t part3[3][4];       // the value, and what is left of it twice
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        F2 f;
                        f.f = make_float2(__uint_as_float(in[e] << 16), __uint_as_float(in[e] & 0xffff0000u));
                        f = mul2(f, w2);
#pragma unroll
                        for (int r = 0; r < 3; ++r) {
                            const __nv_bfloat162 q = __floats2bfloat162_rn(f.f.x, f.f.y);
                            part3[r][e] = *reinterpret_cast<const uint32_t*>(&q);
                            f.f = make_float2(f.f.x - __uint_as_float(part3[r][e] << 16), f.f.y - __uint_as_float(part3[r][e] & 0xffff0000u));
                        }
                    }
                    *here = make_uint4(part3[0][0], part3[0][1], part3[0][2], part3[0][3]);
                    *reinterpret_cast<uint4*>(left + offset) = make_uint4(part3[1][0], part3[1][1], part3[1][2], part3[1][3]);
                    *reinterpret_cast<uint4*>(left + K_BYTES + offset) = make_uint4(part3[2][0], part3[2][1], part3[2][2], part3[2][3]);
                }
                if (!there) {           // another sequence's values: 0 times one that is no number would not be 0
#pragma unroll
                    for (int c = 0; c < 2 * VB; ++c) {
                        const int piece = part * 2 * VB + c;
                        *reinterpret_cast<uint4*>(row + K_BYTES + (piece >> 3) * BOX + (piece & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(ready(it & 1)) : "memory");
            }
            if (tid == 0) p.seg_g[at] = (float)end;
            if (i > 0) leave(i - 1);
        }
        leave(heads - 1);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) tmem_dealloc(tmem, TMEM_COLS);
}

// ---- from segment to segment ------------------------------------------------------------------------------------------------
// Four entries a thread, a warp 8 rows of 16 columns: whole sectors of the states' order and of U's.  U: segments asked for together.
template <int U>
__global__ void __launch_bounds__(256) hd_pass_tc_kernel(const HdTcArgs a) {
    pdl_sync();
    const HeadDecayArgs& p = a.p;
    const int b = blockIdx.x, h = p.h0 + blockIdx.y, size = p.dim * p.vdim, across = (p.vdim + 15) / 16;
    const int lane = threadIdx.x & 31, patch = blockIdx.z * 8 + (threadIdx.x >> 5), down = patch / across;
    const int r = down * 8 + (lane & 7), c = (patch - down * across) * 16 + (lane >> 3) * 4;
    int t0, n, slot;
    if (!hd_sequence(p, b, t0, n, slot) || r >= p.dim || c >= p.vdim) return;
    const int e = r * p.vdim + c;
    auto once = [](const float* at, float (&f)[4]) {         // read here for the last time
        const float4 x = __ldcs(reinterpret_cast<const float4*>(at));
        f[0] = x.x; f[1] = x.y; f[2] = x.z; f[3] = x.w;
    };
    float S[4];
    once(p.state + (size_t)slot * p.pitch + (size_t)h * size + e, S);
    const int segs = (n + HT_SEG - 1) / HT_SEG;
    const size_t first = (size_t)blockIdx.y * p.max_segs + t0 / HT_SEG + b;
    const float* __restrict__ w = p.work + first * size + ((size_t)(c >> 2) * p.dim + r) * 4;
    const float* __restrict__ gs = p.seg_g + first;
    __nv_bfloat16* __restrict__ st = a.starts + first * size + e;
    for (int i0 = 0; i0 < segs; i0 += U) {
        float u[U][4], d[U];
#pragma unroll
        for (int i = 0; i < U; ++i)
            if (i0 + i < segs) {
                once(w + (size_t)(i0 + i) * size, u[i]);
                d[i] = gs[i0 + i];
            }
#pragma unroll
        for (int i = 0; i < U; ++i)
            if (i0 + i < segs) {
                const __nv_bfloat162 lo = __floats2bfloat162_rn(S[0], S[1]), hi = __floats2bfloat162_rn(S[2], S[3]);
                *reinterpret_cast<uint2*>(st + (size_t)(i0 + i) * size) =
                    make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
                const float f = expf(d[i]);
#pragma unroll
                for (int l = 0; l < 4; ++l) S[l] = S[l] * f + u[i][l];
            }
    }
    __stcs(reinterpret_cast<float4*>(p.new_state + (size_t)slot * p.new_pitch + (size_t)h * size + e), make_float4(S[0], S[1], S[2], S[3]));
}

// ---- outputs -------------------------------------------------------------------------------------------------------------------
// A weight of 0 times a value that is no number would reach the rows before it: where the segment has one, such values of the 128 keys that
// a block's rows share are made 0 for the product, and the rows that do see them become NaN at the end.  The rows of other sequences
// behind the segment's last are made 0 always (`look`: the others are looked through).
// Two threads a key, half of each box's 64 entries.
template <int VB>
__device__ __forceinline__ void ht_clear(uint8_t* v, int key, int half, bool there, bool look, volatile uint32_t* found) {
    uint8_t* row = v + key * 128;
    if (!there) {
#pragma unroll
        for (int i = 0; i < VB * 4; ++i) *reinterpret_cast<uint4*>(row + (i >> 2) * (HT_TILE * 128) + half * 64 + (i & 3) * 16) = make_uint4(0u, 0u, 0u, 0u);
        return;
    }
    if (!look) return;
    const __nv_bfloat162 zero = __float2bfloat162_rn(0.f);
    __nv_bfloat162 sum[4] = {zero, zero, zero, zero};     // of 0 times the entries: 0, or NaN
#pragma unroll 1
    for (int b = 0; b < VB; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint4 x = *reinterpret_cast<const uint4*>(row + b * (HT_TILE * 128) + (((half * 4 + i) ^ (key & 7)) << 4));
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[e] = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&w[e]), zero, sum[e]);
        }
    sum[0] = __hadd2(__hadd2(sum[0], sum[1]), __hadd2(sum[2], sum[3]));
    if ((*reinterpret_cast<const uint32_t*>(&sum[0]) & 0x7fff7fffu) == 0) return;
    *found = 1;
    for (int i = 0; i < VB * 16; ++i) {
        uint32_t* w = reinterpret_cast<uint32_t*>(row + (i >> 4) * (HT_TILE * 128) + (((half * 4 + ((i >> 2) & 3)) ^ (key & 7)) << 4)) + (i & 3);
        *w = finite_pair(*w);
    }
}

// The row's outputs in the channels where one of the block's tokens up to its own has a value that is no number (gated: all of them, through
// the norm); `seen`: the block's values.
__device__ __noinline__ void ht_unclear(const __nv_bfloat16* seen, long long ldv, int vdim, int c_lo, int c_hi, int row, bool all, uint8_t* mine) {
    bool any = false;
    for (int pass = 0; pass < (all ? 2 : 1); ++pass)
        for (int c = 0; c < vdim; ++c) {
            bool bad = pass == 1 && any;
            for (int k = 0; k <= row && !bad; ++k) bad = !(fabsf(__bfloat162float(seen[(size_t)k * ldv + c])) < INFINITY);
            any = any || bad;
            if (bad && c >= c_lo && c < c_hi)
                *reinterpret_cast<uint16_t*>(mine + (c >> 6) * (HT_TILE * 128) + ((((c & 63) >> 3) ^ (row & 7)) << 4) + (c & 7) * 2) = 0x7fff;
        }
}

struct alignas(16) HtRowsShared {
    float record[2][HT_RECORD];          // of the head, by its parity
    float norm[2][256];
    float squares[2][HT_TILE];
};

// A block takes the heads of its 128 tokens one after the other.  Three places in shared memory: Q's (X), K's (Y), and one that holds S_0
// and then V.  When the last scores are done the gate comes to X, where the outputs are staged, and the next head's Q to Y (the two change
// roles); when the last P V is done the next S_0 comes.  The two halves of tensor memory change roles likewise: the next head's Q S_0 goes
// where P was while the outputs leave the other half.
template <int KB, int VB>
__global__ void __launch_bounds__(HT_THREADS, VB == 4 ? 1 : 2)
hd_rows_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                  const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_s,
                  const __grid_constant__ CUtensorMap map_g, const __grid_constant__ CUtensorMap map_o, const HdTcArgs a) {
    if (threadIdx.x == 0) {
        ht_fetch_map(&map_q);
        ht_fetch_map(&map_k);
        ht_fetch_map(&map_v);
        ht_fetch_map(&map_s);
        ht_fetch_map(&map_o);
        if (a.p.gate) ht_fetch_map(&map_g);
    }
    pdl_sync();
    constexpr int DK = KB * 64, DV = VB * 64, WIDE = KB > VB ? KB : VB, HALF_COLS = DV > HT_TILE ? DV : HT_TILE;
    constexpr uint32_t BOX = HT_TILE * 128, K_BYTES = KB * BOX, V_BYTES = VB * BOX, S_BOX = DK * 128, PLACE = WIDE * BOX, TMEM_COLS = 2 * HALF_COLS;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    const HeadDecayArgs& p = a.p;
    const uint32_t base = smem_u32(smem_raw), sv = base + 2 * PLACE;
    auto sx = [&](int i) { return base + (i & 1) * PLACE; };
    auto sy = [&](int i) { return base + (~i & 1) * PLACE; };
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem_raw + 3 * PLACE);
    HtRowsShared& sh = *reinterpret_cast<HtRowsShared*>(bars + 16);
    uint32_t& tmem_slot = *reinterpret_cast<uint32_t*>(bars + 14);
    volatile uint32_t* cleared = reinterpret_cast<volatile uint32_t*>(bars + 15);       // by the head's parity
    const int warp = warp_number(), lane = threadIdx.x & 31;
    const int x = blockIdx.x / HT_TILES, at0 = blockIdx.y * a.heads_r, heads = min(a.heads_r, p.heads - at0);
    const uint32_t bar0 = smem_u32(bars), q_full = bar0, k_full = bar0 + 8, k_empty = bar0 + 16, v_full = bar0 + 24, v_empty = bar0 + 32,
                   s_full = bar0 + 40, p_ready = bar0 + 48, o_start = bar0 + 56, o_done = bar0 + 64, g_full = bar0 + 72, x_free = bar0 + 80;
    auto r_full = [&](int i) { return bar0 + 88 + 8u * (i & 1); };
    if (base & 1023u) {
        if (threadIdx.x == 0) atomicCAS(a.error, 0, 49);
        return;
    }
    if (threadIdx.x == 0) {
        cleared[0] = cleared[1] = 0;
        mbar_init(q_full, 1);
        mbar_init(k_full, 1);
        mbar_init(k_empty, 1);
        mbar_init(v_full, 1);
        mbar_init(v_empty, 1);
        mbar_init(s_full, 1);
        mbar_init(p_ready, HT_WORKERS / 32);
        mbar_init(o_start, 1);
        mbar_init(o_done, 1);
        mbar_init(g_full, 1);
        mbar_init(x_free, HT_WORKERS / 32);
        mbar_init(r_full(0), 1);
        mbar_init(r_full(1), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    if (warp == 1) tmem_alloc(smem_u32(&tmem_slot), TMEM_COLS);
    const HdSegment s = hd_find(p, x);
    const int last = blockIdx.x - x * HT_TILES;              // this block's tile of its segment
    const int q0 = s.t0 + last * HT_TILE, nq = min(HT_TILE, s.n - last * HT_TILE);      // nq <= 0: no such tile
    const int n_k = last + 1, n_v = last + 2;               // phases of a head: tiles of keys; S_0 and tiles of values
    auto kv_of = [&](int i) { return (p.h0 + at0 + i) / (p.H / p.G); };
    // by one lane
    auto load_q = [&](int i) {
        mbar_expect_tx(q_full, K_BYTES);
        ht_load_tile<KB>(sx(i), &map_q, q_full, p.h0 + at0 + i, q0);
    };
    auto load_s = [&](int i) {
        mbar_expect_tx(v_full, VB * S_BOX);
#pragma unroll
        for (int b = 0; b < VB; ++b) tma_load_3d(sv + b * S_BOX, &map_s, v_full, b * 64, 0, (at0 + i) * p.max_segs + x);
    };
    auto load_k = [&](int i, int j) {
        mbar_expect_tx(k_full, K_BYTES);
        ht_load_tile<KB>(sy(i), &map_k, k_full, kv_of(i), s.t0 + j * HT_TILE);
    };
    auto load_record = [&](int i) {
        const uint32_t bytes = HT_RECORD * 4, nb = p.gate ? p.vdim * 4 : 0;
        mbar_expect_tx(r_full(i), bytes + nb);
        bulk_load(smem_u32(sh.record[i & 1]), a.sums + ((size_t)(at0 + i) * p.max_segs + x) * HT_RECORD, bytes, r_full(i));
        if (nb) bulk_load(smem_u32(sh.norm[i & 1]), p.norm + (size_t)(p.h0 + at0 + i) * p.vdim, nb, r_full(i));
    };
    // the first copies do not wait for the other warps: this one has made their barriers
    if (warp == 0 && nq > 0 && elect_one()) {
        load_record(0);
        load_q(0);
        load_s(0);
        load_k(0, 0);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    auto tmem_o = [&](int i) { return tmem + (i & 1) * HALF_COLS; };
    auto tmem_s = [&](int i) { return tmem + (~i & 1) * HALF_COLS; };
    if (nq <= 0) {
    } else if (warp == 0) {
        int qs = 1, ks = 1, vs = 1, gs = 0, rs = 1;         // copies begun so far
        bool ok = true;
        for (int i = 0; i < heads && ok; ++i) {
            if (i > 0) {
                ok = mbar_wait_warp(x_free, (i - 1) & 1, a.error, 45);
                if (!ok) break;
                if (elect_one()) load_k(i, 0);
                __syncwarp();
                ++ks;
            }
            if (i + 1 < heads) {
                if (elect_one()) load_record(i + 1);
                __syncwarp();
                ++rs;
            }
            for (int j = 0; j <= last && ok; ++j) {
                ok = mbar_wait_warp(v_empty, (i * n_v + j) & 1, a.error, 45);
                if (!ok) break;
                if (elect_one()) {
                    mbar_expect_tx(v_full, V_BYTES);
                    ht_load_tile<VB>(sv, &map_v, v_full, kv_of(i), s.t0 + j * HT_TILE);
                }
                __syncwarp();
                ++vs;
                ok = mbar_wait_warp(k_empty, (i * n_k + j) & 1, a.error, 45);
                if (!ok) break;
                if (j < last) {
                    if (elect_one()) load_k(i, j + 1);
                    __syncwarp();
                    ++ks;
                    continue;
                }
                if (p.gate) {
                    if (elect_one()) {
                        mbar_expect_tx(g_full, V_BYTES);
                        ht_load_tile<VB>(sx(i), &map_g, g_full, p.h0 + at0 + i, q0);
                    }
                    __syncwarp();
                    ++gs;
                }
                if (i + 1 < heads) {
                    if (elect_one()) load_q(i + 1);
                    __syncwarp();
                    ++qs;
                }
            }
            if (ok && i + 1 < heads) {
                ok = mbar_wait_warp(v_empty, (i * n_v + n_v - 1) & 1, a.error, 45);
                if (!ok) break;
                if (elect_one()) load_s(i + 1);
                __syncwarp();
                ++vs;
            }
        }
        if (*(volatile int*)a.error != 0) {         // no copy is left under way
            mbar_wait(q_full, (qs - 1) & 1, a.error, 45);
            mbar_wait(k_full, (ks - 1) & 1, a.error, 45);
            mbar_wait(v_full, (vs - 1) & 1, a.error, 45);
            if (gs) mbar_wait(g_full, (gs - 1) & 1, a.error, 45);
            for (int i = max(0, rs - 2); i < rs; ++i) mbar_wait(r_full(i), (i >> 1) & 1, a.error, 45);
        }
    } else if (warp == 1) {
        const uint32_t idesc_s = umma_idesc(HT_TILE, HT_TILE), idesc_o = umma_idesc(HT_TILE, DV) | (1u << 16);
        bool ok = true;
        for (int i = 0; i < heads && ok; ++i) {
            const uint32_t sq = sx(i), sk = sy(i), to = tmem_o(i), ts = tmem_s(i);
            auto scores = [&]() {
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < DK / 16; ++k)
                        umma_bf16(ts, umma_desc(sq + (k / 4) * BOX) + 2 * (k % 4), umma_desc(sk + (k / 4) * BOX) + 2 * (k % 4), idesc_s, k != 0);
                    umma_commit(s_full);
                    umma_commit(k_empty);
                }
                __syncwarp();
            };
            // S_0 came when the last P V was done, so its P may be written over
            ok = mbar_wait_warp(q_full, i & 1, a.error, 46) && mbar_wait_warp(v_full, (i * n_v) & 1, a.error, 46);
            if (!ok) break;
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < DK / 16; ++k)
                    umma_bf16(to, umma_desc(sq + (k / 4) * BOX) + 2 * (k % 4), ht_desc(sv + k * 2048, S_BOX), idesc_o, k != 0);
                umma_commit(o_start);
                umma_commit(v_empty);
            }
            __syncwarp();
            if (i > 0) ok = mbar_wait_warp(x_free, (i - 1) & 1, a.error, 46);       // the outputs have left where the scores go
            ok = ok && mbar_wait_warp(k_full, (i * n_k) & 1, a.error, 46);
            if (!ok) break;
            tc_fence_after();
            scores();
            for (int j = 0; j <= last && ok; ++j) {
                ok = mbar_wait_warp(p_ready, (i * n_k + j) & 1, a.error, 46) && mbar_wait_warp(v_full, (i * n_v + j + 1) & 1, a.error, 46);
                if (!ok) break;
                tc_fence_after();
                if (elect_one()) {
                    const int steps = j < last ? HT_TILE / 16 : (nq + 15) / 16;
                    // 16 keys are 8 columns of packed pairs; the second 64 keys' lie where their own scores began
                    for (int k = 0; k < steps; ++k)
                        umma_bf16_ts(to, ts + 8 * k + (k < 4 ? 0 : 32), ht_desc(sv + k * 2048, BOX), idesc_o, 1);
                    umma_commit(v_empty);
                    umma_commit(o_done);
                }
                __syncwarp();
                if (j < last) {         // the next scores go where P is
                    ok = mbar_wait_warp(o_done, (i * n_k + j) & 1, a.error, 46) && mbar_wait_warp(k_full, (i * n_k + j + 1) & 1, a.error, 46);
                    if (!ok) break;
                    tc_fence_after();
                    scores();
                }
            }
        }
    } else {
        const int tid = threadIdx.x - 64, quad = warp & 3, half = tid >> 7, row = quad * 32 + lane, c_lo = half * (DV / 2);
        const uint32_t lane_sel = (uint32_t)(quad * 32) << 16;
        const bool in = row < nq;
        const int mine_at = last * HT_TILE + row;
        bool ok = true;             // a warp that gave up goes on to the barriers of the others, and to nothing else
        for (int i = 0; i < heads; ++i) {
            const uint32_t to = tmem_o(i) + lane_sel, ts = tmem_s(i) + lane_sel;
            const float* record = sh.record[i & 1];
            const double* before = reinterpret_cast<const double*>(record + HT_RECORD_BEFORE);
            ok = ok && mbar_wait_warp(r_full(i), (i >> 1) & 1, a.error, 47);
            const bool look = __any_sync(0xffffffffu, lane < HT_WORKERS / 32 && record[HT_RECORD_BAD + (lane & 7)] != 0.f);
            const float l_row = record[mine_at], l_row2 = l_row * HT_LOG2E;
            const double at_block = before[last * 4 + quad];
            ok = ok && mbar_wait_warp(o_start, i & 1, a.error, 47);
            tc_fence_after();
            if (ok) {
                const float f = ht_ex2((l_row + (float)at_block) * HT_LOG2E);
#pragma unroll 1
                for (int c0 = c_lo; c0 < c_lo + DV / 2; c0 += 32) {
                    float o[32];
                    tmem_ld32(to + c0, o);
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] *= f;
                    ht_store32(to + c0, o);
                }
            }
            for (int j = 0; j <= last; ++j) {
                ok = ok && mbar_wait_warp(s_full, (i * n_k + j) & 1, a.error, 47);
                tc_fence_after();
                if (!ok) break;
#pragma unroll 1
                for (int b = 2 * half; b < 2 * half + 2; ++b) {
                    uint32_t w[16];
                    float v[32];
                    if (j < last || b <= quad) tmem_ld32(ts + 32 * b, v);
                    if (j < last || b < quad) {
                        F2 f;
                        const float r = in ? ht_ex2((l_row + (float)(at_block - before[j * 4 + b + 1])) * HT_LOG2E) : 0.f;
                        f.f = make_float2(r, r);
                        const float4* fk = reinterpret_cast<const float4*>(record + HT_SEG + j * HT_TILE + 32 * b);
#pragma unroll
                        for (int c = 0; c < 8; ++c) {
                            const float4 y = fk[c];
                            F2 s0, s1, y0, y1;
                            s0.f = make_float2(v[4 * c], v[4 * c + 1]);
                            s1.f = make_float2(v[4 * c + 2], v[4 * c + 3]);
                            y0.f = make_float2(y.x, y.y);
                            y1.f = make_float2(y.z, y.w);
                            s0 = mul2(mul2(s0, f), y0);
                            s1 = mul2(mul2(s1, f), y1);
                            const __nv_bfloat162 h0 = __floats2bfloat162_rn(s0.f.x, s0.f.y), h1 = __floats2bfloat162_rn(s1.f.x, s1.f.y);
                            w[2 * c] = *reinterpret_cast<const uint32_t*>(&h0);
                            w[2 * c + 1] = *reinterpret_cast<const uint32_t*>(&h1);
                        }
                    } else if (b == quad) {
                        const float4* lk = reinterpret_cast<const float4*>(record + j * HT_TILE + 32 * b);
#pragma unroll
                        for (int c = 0; c < 8; ++c) {
                            const float4 y = lk[c];
                            const float z[4] = {y.x, y.y, y.z, y.w};
                            float o[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[e] = 4 * c + e <= lane ? v[4 * c + e] * ht_ex2(fmaf(z[e], -HT_LOG2E, l_row2)) : 0.f;
                            const __nv_bfloat162 h0 = __floats2bfloat162_rn(o[0], o[1]), h1 = __floats2bfloat162_rn(o[2], o[3]);
                            w[2 * c] = *reinterpret_cast<const uint32_t*>(&h0);
                            w[2 * c + 1] = *reinterpret_cast<const uint32_t*>(&h1);
                        }
                    } else {
#pragma unroll
                        for (int c = 0; c < 16; ++c) w[c] = 0u;
                    }
                    ht_store16(ts + 16 * b + 32 * half, w);         // over scores that this warp has read
                }
                if (j == last && (look || nq < HT_TILE)) {
                    ok = mbar_wait_warp(v_full, (i * n_v + j + 1) & 1, a.error, 47);
                    if (!ok) break;
                    ht_clear<VB>(smem_raw + 2 * PLACE, tid & 127, half, (tid & 127) < nq, look, cleared + (i & 1));
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                }
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                tc_fence_before();
                __syncwarp();
                if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(p_ready) : "memory");
            }
            ok = ok && mbar_wait_warp(o_done, (i * n_k + last) & 1, a.error, 48);
            tc_fence_after();
            float by = p.scale;
            if (p.gate) {
                if (ok) {
                    float sq = 0.f;
#pragma unroll 1
                    for (int c0 = c_lo; c0 < c_lo + DV / 2; c0 += 32) {
                        float o[32];
                        tmem_ld32(to + c0, o);
#pragma unroll
                        for (int e = 0; e < 32; ++e) sq += o[e] * o[e];
                    }
                    sh.squares[half][row] = sq;
                }
                ok = ok && mbar_wait_warp(g_full, i & 1, a.error, 48);
            }
            asm volatile("bar.sync 1, 256;" ::: "memory");          // the halves' squares; cleared, as any of the warps left it
            // the next head's: the one before it, whose word that was, is behind all warps
            if (tid == 0) cleared[~i & 1] = 0;
            if (!ok) continue;
            if (p.gate) by *= rsqrtf((sh.squares[0][row] + sh.squares[1][row]) * (p.scale * p.scale) / (float)p.vdim + p.eps);
            // the row's outputs go where its gate is (16-byte pieces in the order of the TMA's swizzle) ...
            const int h = p.h0 + at0 + i;
            uint8_t* stage = smem_raw + (i & 1) * PLACE;
            uint8_t* mine = stage + row * 128;
            const float* norm = sh.norm[i & 1];
#pragma unroll 1
            for (int c0 = c_lo; c0 < c_lo + DV / 2; c0 += 32) {
                float o[32];
                tmem_ld32(to + c0, o);
#pragma unroll
                for (int c = 0; c < 32; c += 8) {
                    uint8_t* at = mine + (c0 >> 6) * BOX + (((((c0 & 32) + c) >> 3) ^ (row & 7)) << 4);
                    float y[8];
                    if (p.gate) {
                        float z[8];
                        Vec16<__nv_bfloat16>::unpack(*reinterpret_cast<const uint4*>(at), z);
                        const float4 w0 = *reinterpret_cast<const float4*>(norm + c0 + c), w1 = *reinterpret_cast<const float4*>(norm + c0 + c + 4);
                        const float w[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
                        F2 by2;
                        by2.f = make_float2(by, by);
#pragma unroll
                        for (int e = 0; e < 8; e += 2) {
                            F2 v, u;
                            v.f = make_float2(o[c + e], o[c + e + 1]);
                            u.f = make_float2(w[e], w[e + 1]);
                            v = ht_gated(mul2(mul2(v, by2), u), z[e], z[e + 1]);
                            y[e] = v.f.x;
                            y[e + 1] = v.f.y;
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e) y[e] = o[c + e] * by;
                    }
                    store8(reinterpret_cast<__nv_bfloat16*>(at), y);
                }
            }
            if (cleared[i & 1] && in)
                ht_unclear(static_cast<const __nv_bfloat16*>(p.v) + (size_t)q0 * p.ldv + (size_t)kv_of(i) * p.vdim, p.ldv, p.vdim, c_lo,
                           min(p.vdim, c_lo + DV / 2), row, p.gate != nullptr, mine);
            tc_fence_before();
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");        // read by a copy, or written over by the next head's K
            __syncwarp();
            // ... and leave: whole tiles of whole boxes by TMA, 32 rows a warp, others in whole lines, the warp's rows one after the other
            if (VB > 1 && nq == HT_TILE) {
                if (elect_one()) {
#pragma unroll
                    for (int c = 0; c < DV / 2; c += 64)
                        if (c_lo + c < p.vdim)
                            asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];"
                                         ::"l"(&map_o), "r"(smem_u32(stage) + ((c_lo + c) >> 6) * BOX + quad * (32 * 128)), "r"(c_lo + c), "r"(h),
                                         "r"(q0 + quad * 32) : "memory");
                    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                    asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                }
            } else {
                const int pieces = max(0, min(p.vdim, c_lo + DV / 2) - c_lo) >> 3, rows = max(0, min(32, nq - quad * 32));
                __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(p.out) + (size_t)(q0 + quad * 32) * p.ldo + (size_t)h * p.vdim + c_lo;
#pragma unroll 4
                for (int e = lane; e < rows * pieces; e += 32) {
                    const int r = e / pieces, at = e - r * pieces, c = c_lo / 8 + at, rr = quad * 32 + r;
                    const uint4 y = *reinterpret_cast<const uint4*>(stage + rr * 128 + (c >> 3) * BOX + (((c & 7) ^ (rr & 7)) << 4));
                    *reinterpret_cast<uint4*>(dst + (size_t)r * p.ldo + at * 8) = y;
                }
            }
            __syncwarp();
            if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(x_free) : "memory");
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) tmem_dealloc(tmem, TMEM_COLS);
}

// ---- launchers --------------------------------------------------------------------------------------------------------------------
template <int KB, int VB>
static void ht_launch(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const CUtensorMap& ms, const CUtensorMap& mg,
                      const CUtensorMap& mo, const HdTcArgs& a, cudaStream_t s) {
    const HeadDecayArgs& p = a.p;
    constexpr int WIDE = KB > VB ? KB : VB;
    // the update: K's and V's boxes of half the rows in two stages, and K's twice for what rounding left
    const size_t box = (size_t)HT_TILE * 128, smem_u = (2 * KB + VB) * box + 12 * 8 + 2 * sizeof(HtSums),
                 smem_r = 3 * WIDE * box + 16 * 8 + sizeof(HtRowsShared);
    static PerDevice allowed_u, allowed_r;
    tb_allow_smem(allowed_u, (const void*)hd_update_tc_kernel<KB, VB>, smem_u);
    tb_allow_smem(allowed_r, (const void*)hd_rows_tc_kernel<KB, VB>, smem_r);
    if (p.nt) TB_LAUNCH((hd_update_tc_kernel<KB, VB>), dim3(p.max_segs, (p.heads + a.heads_u - 1) / a.heads_u), HT_THREADS, smem_u, s, mk, mv, a);
    // one wave of blocks is bound by the latency of its loads, more by memory: us of the whole call in a graph with 8 and 4 at a time, 8,192 tokens
    // of 16 heads of 128 88 and 99, 2,048 of 32 47.1 and 47.5, 6 sequences of 100 to 1,500 of 16 of 64 x 128 37.1 and 36.3 (all of one
    // wave: 8), 11,875 in 11 sequences of 32 heads 250 and 235 (4.8 waves: 4)
    const dim3 grid(p.B, p.heads, (p.dim / 8 * ((p.vdim + 15) / 16) + 7) / 8);
    if ((long long)grid.x * grid.y * grid.z <= 148 * 8) TB_LAUNCH((hd_pass_tc_kernel<8>), grid, 256, 0, s, a);
    else TB_LAUNCH((hd_pass_tc_kernel<4>), grid, 256, 0, s, a);
    if (p.nt) TB_LAUNCH((hd_rows_tc_kernel<KB, VB>), dim3(p.max_segs * HT_TILES, (p.heads + a.heads_r - 1) / a.heads_r), HT_THREADS, smem_r, s, mq, mk, mv, ms, mg, mo, a);
}

extern "C" {
// Floats of scratch a head: U, S_0 (bfloat16), the tokens' decays and the segments'.  0: these kernels do not take such heads.
long long tb_head_decay_tc_work(int nt, int B, int dim, int vdim) {
    if (dim <= 0 || vdim <= 0 || dim % 8 || vdim % 8 || dim > 128 || vdim > 256) return 0;
    const long long segs = hd_segments(nt, B, HT_SEG), size = (long long)dim * vdim;
    return (segs * (size + size / 2 + HT_RECORD) + segs + 3) / 4 * 4;
}

int tb_head_decay_tc_bf16(const void* q, const void* k, const void* v, const void* gate, long long ldq, long long ldk, long long ldv,
                          long long ldgate, const float* g, long long g_stride, const float* norm, const float* state, float* new_state,
                          long long pitch, long long new_pitch, void* out, long long ldo, const int* seq_start, const int* slots,
                          float* work, int heads, int nt, int B, int H, int G, int dim, int vdim, int n_slots, float scale,
                          float eps, cudaStream_t s) {
    HdTcArgs a{HeadDecayArgs{q, k, v, gate, g, norm, state, new_state, out, seq_start, slots, work, nullptr, ldq, ldk, ldv, ldgate, ldo,
                             pitch, new_pitch, g_stride, nt, B, H, G, dim, vdim, n_slots, 0, HT_SEG, 0, H, scale, eps},
               nullptr, nullptr, nullptr, 1, 1};
    HeadDecayArgs& p = a.p;
    const int rc = hd_check(p);
    if (rc) return rc;
    if (heads <= 0 || ((uintptr_t)work & 15)) return TB_ERR_ARG;
    if (!tb_head_decay_tc_work(nt, B, dim, vdim)) return TB_ERR_UNSUPPORTED;
    if (ldq % 8 || ldk % 8 || ldv % 8 || ldo % 8 || ldgate % 8 || pitch % 4 || new_pitch % 4 ||
        (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)gate | (uintptr_t)out | (uintptr_t)state | (uintptr_t)new_state |
          (uintptr_t)norm) & 15))
        return TB_ERR_UNSUPPORTED;
    if (B == 0) return 0;
    const long long segs = hd_segments(nt, B, p.seg);
    if (segs * HT_TILES > 0x7fffffffLL) return TB_ERR_UNSUPPORTED;
    p.max_segs = (int)segs;
    if (heads > H) heads = H;
    const size_t size = (size_t)dim * vdim, all = (size_t)heads * p.max_segs;
    a.starts = reinterpret_cast<__nv_bfloat16*>(work + all * size);
    a.sums = work + all * size + all * (size / 2);
    p.seg_g = a.sums + all * HT_RECORD;
    a.error = tc_error_ptr();
    if (!a.error) return tb_last_error();
    // Heads a block: the next one's copies run ahead, but longer blocks leave the SMs less evenly.  Up to four, where three rounds of blocks
    // over their places (two an SM) remain.  us of a call in a graph, 1, 2 and 4 heads a block of the update / of the rows, the other by the
    // rule: 11,875 tokens in 11 sequences of 32 heads of 128 239, 235 and 252 / 245, 236 and 235 (6 / 12 rounds: 2 / 4); 8,192 of 16 88, 85 and
    // 91 / 88, 87 and 87 (1.8 / 3.6: 1); 2,048 of 32 47, 50 and 63 / 47, 48 and 60 (1 / 1.9: 1); 6 sequences of 100 to 1,500 of 16 heads of
    // 64 x 128 37, 42 and 49 / 37, 36 and 46 (1.3 / 2.6: 1)
    const long long places = 2 * 148;
    auto per_block = [&](long long blocks) { return (int)std::max(1LL, std::min({4LL, (long long)heads, blocks * heads / (3 * places)})); };
    a.heads_u = per_block(p.max_segs);
    a.heads_r = per_block((long long)p.max_segs * HT_TILES);
    const int kb = (dim + 63) / 64, vb = vdim <= 64 ? 1 : vdim <= 128 ? 2 : 4;
    CUtensorMap mq, mk, mv, ms, mo, mg = {};
    const int rows = nt > 0 ? nt : 1;
    if (make_map_3d(&mq, q, dim, H, rows, dim, ldq, 1, HT_HALF) || make_map_3d(&mk, k, dim, G, rows, dim, ldk, 1, HT_HALF) ||
        make_map_3d(&mv, v, vdim, G, rows, vdim, ldv, 1, HT_HALF) ||
        make_map_3d(&mo, out, vdim, H, rows, vdim, ldo, 1, 32) || make_map_3d(&ms, a.starts, vdim, dim, (long long)all, vdim, (long long)size, kb * 64, 1) ||
        (gate && make_map_3d(&mg, gate, vdim, H, rows, vdim, ldgate, 1, HT_HALF)))
        return TB_ERR_UNSUPPORTED;
    for (p.h0 = 0; p.h0 < H; p.h0 += heads) {
        p.heads = H - p.h0 < heads ? H - p.h0 : heads;
        if (kb == 1) {
            if (vb == 1) ht_launch<1, 1>(mq, mk, mv, ms, mg, mo, a, s);
            else if (vb == 2) ht_launch<1, 2>(mq, mk, mv, ms, mg, mo, a, s);
            else ht_launch<1, 4>(mq, mk, mv, ms, mg, mo, a, s);
        } else {
            if (vb == 1) ht_launch<2, 1>(mq, mk, mv, ms, mg, mo, a, s);
            else if (vb == 2) ht_launch<2, 2>(mq, mk, mv, ms, mg, mo, a, s);
            else ht_launch<2, 4>(mq, mk, mv, ms, mg, mo, a, s);
        }
    }
    return tb_last_error();
}
}

#include "tape.h"
TB_TAPE_REGISTER(tb_head_decay_tc_bf16)
