// The choice of experts within groups, from router logits x [nt, E] in float:
//
//   s = softmax(x) or sigmoid(x);   c = s + bias (the bias steers the choice alone)
//   a group's worth = the sum of its group_top (1 or 2) largest c;  the groups_use worthiest groups stay
//   the k largest c of those are chosen, in descending order;  w = s of the chosen, / their sum with `renorm`, times `scale`
//
// Equal c, or groups of equal worth, go to the lower index.  An expert with logit -inf has s = 0 (in a row of nothing else too); NaN ranks
// below -inf, and in a group's worth it counts as -inf, as inf - inf does, so the k indices of a row always differ; chosen scores that are
// all 0 stay 0 when they are renormalized.
//
// A warp per token, a lane the PER neighbouring experts from lane * PER on: the lowest lane among equals has the lowest index, so
// a choice is one redux over order-preserving keys, a ballot and a shuffle.  Without a bias c and x have the same order, and the
// logits themselves are compared.  With one, or where sums of scores decide, values closer than what float rounding can turn round
// are decided again in 64 bits (float: expf 2 ulp, two more roundings, the sum's): a row in some hundreds.
// Bound by integer and select instructions, some 1,370 a token: 8,191 tokens, the 8 of 256 experts in 4 of 8 groups, 16 us by itself and 14
// behind another (0.6 TB/s of logits), of which a few rows in 64 bits are the last 1 to 3; 2,039 tokens, 4 of 60, 4 and 3 us; 8 tokens likewise.
#include "common.cuh"

#define RG_MAX_E 1024
#define RG_MAX_K 30
#define RG_MAX_GROUPS 32
#define RG_WARPS 8

struct RouterGroupArgs {
    const float* logits;            // [nt] rows of E, ld apart
    const float* bias;              // [E] or null
    int* idx;                       // [nt, k]
    float* w;
    long long ld;
    int nt, E, k, groups, groups_use, group_top, softmax, renorm;
    float scale;
};

// larger value <=> larger key; NaN 1; 0 is left for what cannot be chosen (any more)
__device__ __forceinline__ unsigned rg_key(float c) {
    const unsigned b = __float_as_uint(c + 0.0f);
    return c != c ? 1u : b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float rg_value(unsigned key) {
    return key == 1u ? __int_as_float(0x7fc00000) : __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// Entries e0 .. e0 + PER - 1 of a row of E, `none` behind its end; four an access where they lie so.
template <int PER>
__device__ __forceinline__ void rg_load(const float* __restrict__ row, int e0, int E, float none, float (&x)[PER]) {
    if constexpr (PER >= 4) {
        if (((uintptr_t)row & 15) == 0 && e0 + PER <= E) {
#pragma unroll
            for (int i = 0; i < PER; i += 4) {
                const float4 f = *reinterpret_cast<const float4*>(row + e0 + i);
                x[i] = f.x;
                x[i + 1] = f.y;
                x[i + 2] = f.z;
                x[i + 3] = f.w;
            }
            return;
        }
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) x[i] = e0 + i < E ? row[e0 + i] : none;
}

// The choice in 64 bits: called for the few rows where float cannot tell.  Returns this lane's choice (lane < k).
template <int PER>
__device__ __noinline__ int rg_choose64(const RouterGroupArgs& p, const float* row, float mx, int lane) {
    const double lowest = -INFINITY;
    const int size = p.E / p.groups;
    double c[PER];
    unsigned open = 0u, none = 0u;  // which of the lane's may be chosen, and which are NaN
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int e = lane * PER + i;
        const float x = e < p.E ? row[e] : -INFINITY;
        c[i] = p.softmax ? exp((double)x - (double)mx) : 1.0 / (1.0 + exp(-(double)x));
        if (e < p.E) open |= 1u << i;
    }
    if (p.softmax) {
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < PER; ++i) sum += c[i];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        const double inv = sum == 0.0 ? 0.0 : 1.0 / sum;
#pragma unroll
        for (int i = 0; i < PER; ++i) c[i] *= inv;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        if (p.bias && (open >> i & 1u)) c[i] += (double)p.bias[lane * PER + i];
        if (c[i] != c[i]) {
            c[i] = lowest;
            none |= 1u << i;
        }
    }
    if (p.groups > 1) {
        double worth = lowest;      // of group `lane`
        for (int g = 0; g < p.groups; ++g) {
            const int from = g * size - lane * PER;         // the group among this lane's
            double a = lowest, b = lowest;      // its two largest
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (i >= from && i < from + size) {
                    b = fmax(b, fmin(a, c[i]));
                    a = fmax(a, c[i]);
                }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                const double oa = __shfl_xor_sync(0xffffffffu, a, o), ob = __shfl_xor_sync(0xffffffffu, b, o);
                b = fmax(fmin(a, oa), fmax(b, ob));
                a = fmax(a, oa);
            }
            if (lane == g) worth = p.group_top == 2 && size > 1 ? a + b : a;
        }
        if (worth != worth) worth = lowest;
        int place = 0;
        for (int g = 0; g < p.groups; ++g) {
            const double other = __shfl_sync(0xffffffffu, worth, g);
            place += other > worth || (other == worth && g < lane);
        }
        const unsigned kept = __ballot_sync(0xffffffffu, lane < p.groups && place < p.groups_use);
        for (int g = 0; g < p.groups; ++g) {
            const int from = g * size - lane * PER;
            if (kept >> g & 1u) continue;
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (i >= from && i < from + size) open &= ~(1u << i);
        }
    }
    // without a bias experts are compared by their logits, here as everywhere
    if (!p.bias) {
        none = 0u;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const float x = lane * PER + i < p.E ? row[lane * PER + i] : 0.f;
            c[i] = x;
            none |= x != x ? 1u << i : 0u;
        }
    }
    // larger value <=> larger key, NaN below -inf, 0 for what cannot be chosen (any more)
    unsigned long long key[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const unsigned long long b = (unsigned long long)__double_as_longlong(c[i] + 0.0);
        key[i] = !(open >> i & 1u) ? 0ull : none >> i & 1u ? 1ull : b >> 63 ? ~b : b | 1ull << 63;
    }
    int mine = 0;
    for (int j = 0; j < p.k; ++j) {
        unsigned long long best = key[0];
        int at = 0;
#pragma unroll
        for (int i = 1; i < PER; ++i) {
            at = key[i] > best ? i : at;
            best = key[i] > best ? key[i] : best;
        }
        // the largest of the warp by halves; the lowest lane among equals has the lowest index
        const unsigned hi = (unsigned)(best >> 32), lo = (unsigned)best;
        const unsigned most_hi = __reduce_max_sync(0xffffffffu, hi);
        const unsigned most_lo = __reduce_max_sync(0xffffffffu, hi == most_hi ? lo : 0u);
        const int from = __ffs(__ballot_sync(0xffffffffu, hi == most_hi && lo == most_lo)) - 1;
        const int e = __shfl_sync(0xffffffffu, lane * PER + at, from);
        if (lane == from)
#pragma unroll
            for (int i = 0; i < PER; ++i) key[i] = i == at ? 0ull : key[i];
        if (lane == j) mine = e;
    }
    return mine;
}

template <int PER>
__global__ void __launch_bounds__(RG_WARPS * 32) router_groups_kernel(const __grid_constant__ RouterGroupArgs p) {
    extern __shared__ float rg_sm[];        // [RG_WARPS][E + E / 32 + 1] where groups' worths are found
    pdl_sync();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long t = (long long)blockIdx.x * RG_WARPS + warp;
    if (t >= p.nt) return;
    const float* row = p.logits + t * p.ld;
    const int E = p.E, e0 = lane * PER;
    float x[PER];
    rg_load<PER>(row, e0, E, -INFINITY, x);
    // scores, as far as they are asked for
    const bool sums = p.groups > 1 && p.group_top == 2;     // sums of scores decide
    const bool by_logit = !p.bias;
    float mx = 0.f, inv = 1.f;
    if (p.softmax && (p.bias || sums || !p.renorm)) {
        mx = x[0];
#pragma unroll
        for (int i = 1; i < PER; ++i) mx = fmaxf(mx, x[i]);
        mx = warp_max(mx);
        if (mx == -INFINITY) mx = 0.f;      // a row of masked experts: scores of 0
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < PER; ++i) sum += expf(x[i] - mx);
        sum = warp_sum(sum);
        inv = sum == 0.f ? 0.f : 1.0f / sum;
    }
    auto score = [&](float v) { return p.softmax ? expf(v - mx) * inv : 1.0f / (1.0f + expf(-v)); };
    unsigned key[PER];
    float c[PER];
    if (by_logit && !sums) {
#pragma unroll
        for (int i = 0; i < PER; ++i) c[i] = x[i];
    } else {
        // the hardware's exponential and reciprocal (2 and 1 ulp, and the argument's rounding): off by 3e-7 of the largest score at most,
        // within what `loose` below allows for
        const float by = p.softmax ? 1.4426950408889634f : -1.4426950408889634f;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            float y;
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"((x[i] - mx) * by));
            if (p.softmax) y *= inv;
            else asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(1.0f + y));
            c[i] = y;
        }
        if (p.bias) {
            float b[PER];
            rg_load<PER>(p.bias, e0, E, 0.f, b);
#pragma unroll
            for (int i = 0; i < PER; ++i) c[i] += b[i];
        }
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) key[i] = e0 + i < E ? rg_key(by_logit ? x[i] : c[i]) : 0u;
    // what float may have turned round: scores up to `top`, each off by up to 4 (sigmoid) or 24 (softmax, its sum included)
    // half steps of it, and the roundings of the sums that were compared
    const float loose = (p.softmax ? 24.f * inv : 4.f) * 1.2e-7f;
    bool again = false;
    if (p.groups > 1) {
        // 32 / groups lanes (a power of two) find a group's worth
        float* cs = rg_sm + (size_t)warp * (E + E / 32 + 1);
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (e0 + i < E) cs[e0 + i + ((e0 + i) >> 5)] = c[i] != c[i] ? -INFINITY : c[i];
        __syncwarp();
        const int size = E / p.groups;
        const float per_size = 1.0f / (float)size;      // (e + 1/2) / size is at least 1 / 2048 from a whole number
        int L = 1;
        while (2 * L * p.groups <= 32) L *= 2;
        const int g = lane / L, part = lane - g * L;
        float a = -INFINITY, b = -INFINITY;
        if (g < p.groups)
            for (int i = part; i < size; i += L) {
                const int e = g * size + i;
                const float v = cs[e + (e >> 5)];
                b = fmaxf(b, fminf(a, v));
                a = fmaxf(a, v);
            }
        for (int o = L >> 1; o > 0; o >>= 1) {
            const float oa = __shfl_xor_sync(0xffffffffu, a, o), ob = __shfl_xor_sync(0xffffffffu, b, o);
            b = fmaxf(fminf(a, oa), fmaxf(b, ob));
            a = fmaxf(a, oa);
        }
        float worth = p.group_top == 2 && size > 1 ? a + b : a;
        if (worth != worth) worth = -INFINITY;      // a bias of inf and one of -inf
        int place = 0;
        for (int j = 0; j < p.groups; ++j) {
            const float other = __shfl_sync(0xffffffffu, worth, j * L);
            place += other > worth || (other == worth && j < g);
        }
        const bool in = g < p.groups && place < p.groups_use;
        if (!(by_logit && !sums) && p.groups_use < p.groups) {
            float least = in ? worth : INFINITY, most = g < p.groups && !in ? worth : -INFINITY;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                least = fminf(least, __shfl_xor_sync(0xffffffffu, least, o));
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
            }
            again = least - most <= 4.f * loose + 2.5e-7f * (fabsf(least) + fabsf(most));
        }
        const unsigned kept = __ballot_sync(0xffffffffu, in);
        if (size % PER == 0) {          // a lane's experts are of one group
            if (!(kept >> ((int)((e0 + 0.5f) * per_size) * L & 31) & 1u))
#pragma unroll
                for (int i = 0; i < PER; ++i) key[i] = 0u;
        } else
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (!(kept >> ((int)((e0 + i + 0.5f) * per_size) * L & 31) & 1u)) key[i] = 0u;
    }
    // the k largest, and where float may have turned values round the two that would come next
    unsigned my_key = 0u;
    int mine = 0;
    const int rounds = by_logit ? p.k : p.k + 2;
    if constexpr (PER <= 8) {
        // a lane's own in descending order first (neighbours change places only if the later is larger, so equals stay in order), their
        // places in four bits each: the lane that a round takes from moves up
        unsigned place[PER], places = 0u;
#pragma unroll
        for (int i = 0; i < PER; ++i) place[i] = i;
#pragma unroll
        for (int turn = 0; turn < PER; ++turn)
#pragma unroll
            for (int i = turn & 1; i + 1 < PER; i += 2) {
                const bool swap = key[i + 1] > key[i];
                const unsigned k0 = key[i], p0 = place[i];
                key[i] = swap ? key[i + 1] : k0;
                key[i + 1] = swap ? k0 : key[i + 1];
                place[i] = swap ? place[i + 1] : p0;
                place[i + 1] = swap ? p0 : place[i + 1];
            }
#pragma unroll
        for (int i = 0; i < PER; ++i) places |= place[i] << (4 * i);
        for (int j = 0; j < rounds; ++j) {
            const unsigned best = __reduce_max_sync(0xffffffffu, key[0]);
            const int from = __ffs(__ballot_sync(0xffffffffu, key[0] == best)) - 1;
            const int e = __shfl_sync(0xffffffffu, e0 + (int)(places & 15u), from);
            if (lane == from) {
#pragma unroll
                for (int i = 0; i + 1 < PER; ++i) key[i] = key[i + 1];
                key[PER - 1] = 0u;
                places >>= 4;
            }
            if (lane == j) {
                my_key = best;
                mine = e;
            }
        }
    } else {
        unsigned most = key[0];
#pragma unroll
        for (int i = 1; i < PER; ++i) most = max(most, key[i]);
        for (int j = 0; j < rounds; ++j) {
            const unsigned best = __reduce_max_sync(0xffffffffu, most);
            const int from = __ffs(__ballot_sync(0xffffffffu, most == best)) - 1;
            int at = PER;
#pragma unroll
            for (int i = PER - 1; i >= 0; --i) at = key[i] == best ? i : at;
            const int e = __shfl_sync(0xffffffffu, e0 + at, from);
            if (lane != from) at = PER;
            most = 0u;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                key[i] = i == at ? 0u : key[i];
                most = max(most, key[i]);
            }
            if (lane == j) {
                my_key = best;
                mine = e;
            }
        }
    }
    const bool have = lane < rounds && my_key != 0u;        // fewer than k + 2 may be left
    if (!have) mine = 0;
    float mine_x = have ? row[mine] : 0.f;
    if (!by_logit) {
        // a lane's value against its follower's
        const float v = rg_value(my_key), b = have ? p.bias[mine] : 0.f, nv = __shfl_down_sync(0xffffffffu, v, 1);
        const float nx = __shfl_down_sync(0xffffffffu, mine_x, 1), nb = __shfl_down_sync(0xffffffffu, b, 1);
        const bool followed = __shfl_down_sync(0xffffffffu, (int)have, 1) && have && lane + 1 < rounds;
        const bool near = followed && v - nv <= 2.f * loose + 1.3e-7f * (fabsf(v) + fabsf(nv));
        const unsigned nears = __ballot_sync(0xffffffffu, near);
        const unsigned closes = __ballot_sync(0xffffffffu, near && !(mine_x == nx && b == nb));
        if (!again) {
            if ((nears >> (p.k - 1) & 3u) == 3u) {
                again = true;       // one that was not looked at may belong among the chosen
            } else if ((closes & ((1u << p.k) - 1u)) && p.softmax) {
                again = true;       // a sum over all experts is wanted
            } else if (closes & ((1u << p.k) - 1u)) {
                // the candidates in 64 bits, a lane each, to their places by counting; NaN, which compares with nothing, behind all numbers
                const double d = have && lane <= p.k ? 1.0 / (1.0 + exp(-(double)mine_x)) + (double)b : 0.0;
                const bool counts = have && lane <= p.k;
                int place = 0;
                for (int j = 0; j <= p.k; ++j) {
                    const double od = __shfl_sync(0xffffffffu, d, j);
                    const int oe = __shfl_sync(0xffffffffu, mine, j);
                    const int there = __shfl_sync(0xffffffffu, (int)counts, j);
                    const bool on = od != od, dn = d != d;
                    place += there && (od > d || (dn && !on) || ((od == d || (on && dn)) && oe < mine));
                }
                const int was = mine;
                for (int j = 0; j <= p.k; ++j) {
                    const int to = __shfl_sync(0xffffffffu, counts ? place : 32, j), e = __shfl_sync(0xffffffffu, was, j);
                    if (lane == to) mine = e;
                }
                if (lane < p.k) mine_x = row[mine];
            }
        }
    }
    if (__any_sync(0xffffffffu, again)) {
        mine = rg_choose64<PER>(p, row, mx, lane);
        if (lane < p.k) mine_x = row[mine];
    }
    // weights
    float s = 0.f;
    if (p.renorm) {
        // against the largest chosen logit, so that small scores keep their ratios
        float m = lane < p.k ? mine_x : -INFINITY;
        m = warp_max(m);
        if (!p.softmax) m = fminf(m, 0.f);
        if (m == -INFINITY) m = 0.f;
        if (lane < p.k) s = p.softmax ? expf(mine_x - m) : m < 0.f ? expf(mine_x - m) / (1.0f + expf(mine_x)) : 1.0f / (1.0f + expf(-mine_x));
        const float sum = warp_sum(s);
        if (sum != 0.f) s /= sum;
    } else if (lane < p.k) {
        s = score(mine_x);
    }
    if (lane < p.k) {
        p.idx[t * p.k + lane] = mine;
        p.w[t * p.k + lane] = s * p.scale;
    }
}

template <int PER>
static void router_groups_launch(const RouterGroupArgs& p, cudaStream_t s) {
    const size_t smem = p.groups > 1 ? (size_t)RG_WARPS * (p.E + p.E / 32 + 1) * sizeof(float) : 0;
    TB_LAUNCH((router_groups_kernel<PER>), (p.nt - 1) / RG_WARPS + 1, RG_WARPS * 32, smem, s, p);
}

extern "C" int tb_router_groups(const float* logits, long long ld, const float* bias, int* idx, float* w, int nt, int E, int k,
                                int groups, int groups_use, int group_top, int softmax, int renorm, float scale, cudaStream_t s) {
    if (nt < 0 || E <= 0 || k <= 0 || groups <= 0 || E % groups || groups_use <= 0 || groups_use > groups || ld < E ||
        k > E / groups * groups_use || group_top < 1 || group_top > 2)
        return TB_ERR_ARG;
    if (E > RG_MAX_E || k > RG_MAX_K || groups > RG_MAX_GROUPS) return TB_ERR_UNSUPPORTED;
    if (nt == 0) return 0;
    const RouterGroupArgs p{logits, bias, idx, w, ld, nt, E, k, groups, groups_use, group_top, softmax, renorm, scale};
    if (E <= 32) router_groups_launch<1>(p, s);
    else if (E <= 64) router_groups_launch<2>(p, s);
    else if (E <= 128) router_groups_launch<4>(p, s);
    else if (E <= 256) router_groups_launch<8>(p, s);
    else if (E <= 512) router_groups_launch<16>(p, s);
    else router_groups_launch<32>(p, s);
    return tb_last_error();
}

#include "tape.h"
TB_TAPE_REGISTER(tb_router_groups)
