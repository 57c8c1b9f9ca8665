// trench-gguf_amd/csrc/route.cuh - a router's choice of experts and the grouping of the rows by expert.
//
// Choice: score = softmax or sigmoid of a token's logits; key = score + bias, or the logit itself where there is no
// bias and one group (both scores rise with it). With groups, a group counts by the sum of its two largest keys and the
// `keep` best groups stay. The k largest keys are taken, a tie at the lowest index; weight = scale * score, over the sum
// of the taken scores with `renorm`. A NaN logit or key counts as minus infinity, which is never taken: what is left
// over gets id -1 and weight 0.
#pragma once
#include "common.cuh"

struct RouteArgs {
    const void *logits;
    int64_t ld;                 // elements from token to token
    const float *bias;
    int32_t *ids;
    float *weights;
    int64_t ntok;
    int nexp, k, ngroup, keep;
    float scale;
    int sigmoid, renorm;
};

// the other lane of each pair at distance 1, 2, 4, 8 (within rows of 16 lanes, as a reduction needs it), 16 and 32
template <int STEP> DEV float rt_other(float v) {
    if (STEP >= 16) return __shfl_xor(v, STEP, 64);
    constexpr int CTRL = STEP == 1 ? 0xB1 : STEP == 2 ? 0x4E : STEP == 4 ? 0x141 : 0x140;   // quads, half mirror, mirror
    return ffrom((uint32_t)__builtin_amdgcn_mov_dpp((int)fbits(v), CTRL, 0xf, 0xf, true));
}
DEV float rt_max(float v) {     // over the wave, in every lane
    v = fmaxf(v, rt_other<1>(v));
    v = fmaxf(v, rt_other<2>(v));
    v = fmaxf(v, rt_other<4>(v));
    v = fmaxf(v, rt_other<8>(v));
    v = fmaxf(v, rt_other<16>(v));
    return fmaxf(v, rt_other<32>(v));
}
DEV float rt_sum(float v) {
    v += rt_other<1>(v);
    v += rt_other<2>(v);
    v += rt_other<4>(v);
    v += rt_other<8>(v);
    v += rt_other<16>(v);
    return v + rt_other<32>(v);
}
// a value that at least `count` lanes reach: the smallest of the maxima of as many groups of lanes
DEV float rt_reached(float v, int count) {
    const int g = count > 32 ? 1 : count > 16 ? 2 : count > 8 ? 4 : count > 4 ? 8 : count > 2 ? 16 : 32;   // lanes a group
    float o;
#define RT_STEP(S) o = rt_other<S>(v); v = S < g ? fmaxf(v, o) : fminf(v, o)
    RT_STEP(1);
    RT_STEP(2);
    RT_STEP(4);
    RT_STEP(8);
    RT_STEP(16);
    RT_STEP(32);
#undef RT_STEP
    return v;
}
template <int SRC> DEV float rt_load(const void *p, int64_t i) {
    if (SRC == T_F32) return ((const float *)p)[i];
    const uint32_t h = ((const uint16_t *)p)[i];
    return SRC == T_BF16 ? ffrom(h << 16) : h2f(h);
}

#define RT_NONE (-__builtin_inff())

// One wave a token; lane l holds experts l, l + 64, ... The k largest keys are found in one pass: the smallest of the
// maxima of at least k groups of lanes is reached by at least k keys, so only the keys that reach it (about three times
// k) can be among them; they are moved to one a lane in index order and each counts the ones ahead of it. Where more than
// 64 reach it, the largest is taken k times instead. A score is computed only where it is needed: logits order the
// experts by themselves unless a bias or groups come in, and the sum over all cancels with renorm. Instructions bound
// it: 16384 tokens of 384 experts take 16.5 us (taking the largest key k times over took 26.6), 0.8 TB/s.
template <int SRC, int P>
__global__ __launch_bounds__(256) void k_route(RouteArgs a) {
    __shared__ float keys[4][64 * P], gs[4][64];
    __shared__ int2 cand[4][64];                            // (key, expert)
    __shared__ int cid[4][64];
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t t = (int64_t)blockIdx.x * 4 + wave;
    const bool live = t < a.ntok;
    const int64_t row = (live ? t : a.ntok - 1) * a.ld;
    float x[P], key[P];
    float mx = RT_NONE;
#pragma unroll
    for (int j = 0; j < P; ++j) {
        const int e = j * 64 + lane;
        float v = e < a.nexp ? rt_load<SRC>(a.logits, row + e) : RT_NONE;
        v = v == v ? fminf(v, 3.402823466e38f) : RT_NONE;
        x[j] = v;
        mx = fmaxf(mx, v);
    }
    const bool by_logit = !a.bias && a.ngroup == 1;
    float z = 1.f;
    if (!a.sigmoid) {
        mx = rt_max(mx);
        if (!by_logit || !a.renorm) {
            float s = 0.f;
#pragma unroll
            for (int j = 0; j < P; ++j) s += x[j] == RT_NONE ? 0.f : expf(x[j] - mx);
            z = rt_sum(s);
            z = z > 0.f ? z : 1.f;
        }
    }
    auto score = [&](float v) { return v == RT_NONE ? 0.f : a.sigmoid ? 1.f / (1.f + expf(-v)) : expf(v - mx) / z; };
    if (by_logit) {
#pragma unroll
        for (int j = 0; j < P; ++j) key[j] = x[j];
    } else {
#pragma unroll
        for (int j = 0; j < P; ++j) {
            const int e = j * 64 + lane;
            float v = score(x[j]);
            if (a.bias && e < a.nexp) v += a.bias[e];
            key[j] = v == v && x[j] != RT_NONE ? v : RT_NONE;
        }
    }
    if (a.ngroup > 1) {         // (uniform)
#pragma unroll
        for (int j = 0; j < P; ++j) keys[wave][j * 64 + lane] = key[j];
        __builtin_amdgcn_wave_barrier();
        const int per = a.nexp / a.ngroup;
        float best = RT_NONE, next = RT_NONE;
        if (lane < a.ngroup) {
            for (int i = 0; i < per; ++i) {
                const float v = keys[wave][lane * per + i];
                next = fmaxf(next, fminf(best, v));
                best = fmaxf(best, v);
            }
        }
        const float g = next == RT_NONE ? best : best + next;
        gs[wave][lane] = g;
        __builtin_amdgcn_wave_barrier();
        int ahead = 0;          // groups that come before this one
        for (int i = 0; i < a.ngroup; ++i) ahead += gs[wave][i] > g || (gs[wave][i] == g && i < lane);
        const uint64_t kept = __ballot(lane < a.ngroup && ahead < a.keep);
#pragma unroll
        for (int j = 0; j < P; ++j) {
            const int e = j * 64 + lane;
            if (e < a.nexp && !((kept >> (e / per)) & 1)) key[j] = RT_NONE;
        }
    }
    float top = key[0];
#pragma unroll
    for (int j = 1; j < P; ++j) top = fmaxf(top, key[j]);
    const float bound = rt_reached(top, a.k);
    int n = 0;                  // the keys that reach it (none of minus infinity), in index order
#pragma unroll
    for (int j = 0; j < P; ++j) {
        const bool on = key[j] >= bound && key[j] != RT_NONE;
        const uint64_t who = __ballot(on);
        const int at = n + __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0));
        if (on && at < 64) cand[wave][at] = make_int2((int)fbits(key[j]), j * 64 + lane);
        n += __popcll(who);
    }
    __builtin_amdgcn_wave_barrier();
    int rank = 64, id = -1;     // this lane's candidate, if it is among the k
    if (n <= 64) {
        // keys as whole numbers in the same order: one from before this lane is ahead if it is not less, one from behind if
        // it is more (lanes past n hold less than all)
        const int2 c = cand[wave][lane];
        const int b = c.x == (int)0x80000000 ? 0 : c.x;     // (minus zero ties with zero)
        const int mine = lane < n ? (b < 0 ? b ^ 0x7fffffff : b) : (int)0x80000000;
        id = lane < n ? c.y : -1;
        int ahead = 0;
        for (int i0 = 0; i0 < n; i0 += 8) {
#pragma unroll
            for (int i = i0; i < i0 + 8; ++i) ahead += __builtin_amdgcn_readlane(mine, i) > (i < lane ? mine - 1 : mine);
        }
        if (lane < n && ahead < a.k) rank = ahead;
    } else {
        for (int r = 0; r < a.k; ++r) {                     // (n > 64 >= k: there is one every time)
            float v = key[0];
#pragma unroll
            for (int j = 1; j < P; ++j) v = fmaxf(v, key[j]);
            const float m = rt_max(v);
            int best = -1;
#pragma unroll
            for (int j = 0; j < P; ++j) {
                const uint64_t who = __ballot(key[j] == m);
                if (best < 0 && who) best = j * 64 + __ffsll((unsigned long long)who) - 1;
            }
#pragma unroll
            for (int j = 0; j < P; ++j)
                if (j * 64 + lane == best) key[j] = RT_NONE;
            if (lane == r) {
                rank = r;
                id = best;
            }
        }
    }
    __builtin_amdgcn_wave_barrier();
    if (lane < a.k) cid[wave][lane] = -1;
    __builtin_amdgcn_wave_barrier();
    if (rank < a.k) cid[wave][rank] = id;
    __builtin_amdgcn_wave_barrier();
    const int my_id = lane < a.k ? cid[wave][lane] : -1;
    float my = 0.f;
    if (my_id >= 0) {
        float v = rt_load<SRC>(a.logits, row + my_id);
        my = score(fminf(v, 3.402823466e38f));
    }
    float sum = 0.f;            // of the scores, best first
    for (int r = 0; r < a.k; ++r) sum += ffrom((uint32_t)__builtin_amdgcn_readlane((int)fbits(my), r));
    if (live && lane < a.k) {
        const float w = !a.renorm ? my : sum > 0.f ? my / sum : 0.f;
        a.ids[t * a.k + lane] = my_id;
        a.weights[t * a.k + lane] = w * a.scale;
    }
}

// ---- grouping: assignments (flat ids [n]) sorted by expert, in order within each. Chunks of 512 assignments a wave, a
// workgroup each (of 8 waves: every chunk reads the counts of all, so few are better, and many share the work; one of 4 where
// that holds the whole call): counts per chunk and expert, then every chunk places its own.
#define RG_SMALL 2048
#define RG_BLOCK 4096
#define RG_CHUNKS 128
#define RG_MAXE 1024

// the lanes of a wave find those with their number by its bits
DEV uint64_t rg_same(int id, bool on) {
    uint64_t same = __ballot(on);
#pragma unroll
    for (int j = 0; j < 10; ++j) {
        const uint64_t bit = __ballot((id >> j) & 1);
        same &= (id >> j) & 1 ? bit : ~bit;
    }
    return same;
}

// counts[chunk][e]
__global__ __launch_bounds__(1024) void k_group_count(const int32_t *__restrict__ ids, int64_t n, int nexp, int64_t chunk,
                                                     int32_t *__restrict__ counts) {
    __shared__ int hist[RG_MAXE];
    const int tid = threadIdx.x;
    for (int e = tid; e < nexp; e += 1024) hist[e] = 0;
    __syncthreads();
    const int64_t i0 = (int64_t)blockIdx.x * chunk, i1 = i0 + chunk < n ? i0 + chunk : n;
    for (int64_t b = i0; b < i1; b += 8192) {
        int32_t id[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) id[r] = b + r * 1024 + tid < i1 ? ids[b + r * 1024 + tid] : -1;
#pragma unroll
        for (int r = 0; r < 8; ++r)
            if ((uint32_t)id[r] < (uint32_t)nexp) atomicAdd(&hist[id[r]], 1);
    }
    __syncthreads();
    for (int e = tid; e < nexp; e += 1024) counts[(int64_t)blockIdx.x * nexp + e] = hist[e];
}

// offsets [nexp + 1], rows [n] (the token of each sorted assignment), slots [n] (its flat index); the places past
// offsets[nexp] (ids that name no expert) get -1. counts is null where there is one chunk. Each of the NW waves places its
// share of the chunk, 64 assignments at a time: the place of each is the expert's next and the number of its own before it.
// 131072 assignments of 384 experts take 3.1 us to count and 10.6 to place, most of it the counts of all chunks on their way.
template <int NW>
__global__ __launch_bounds__(NW * 64) void k_group_place(const int32_t *__restrict__ ids, int64_t n, int k, int nexp,
                                                         int64_t chunk, const int32_t *__restrict__ counts,
                                                         int32_t *__restrict__ offsets, int32_t *__restrict__ rows,
                                                         int32_t *__restrict__ slots) {
    constexpr int PER = RG_MAXE / (NW * 64);
    __shared__ int part[NW], place[NW][RG_MAXE];
    const int tid = threadIdx.x, lane = lane_id(), wave = tid >> 6, me = blockIdx.x, nchunk = gridDim.x;
    const int64_t i0 = me * chunk, i1 = i0 + chunk < n ? i0 + chunk : n, w0 = i0 + wave * (chunk / NW);
    const int64_t w1 = w0 + chunk / NW < i1 ? w0 + chunk / NW : i1;
    // this thread's experts: the whole call's totals and what earlier chunks hold
    int total[PER] = {}, before[PER] = {};
    if (nchunk > 1) {
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int e = PER * tid + j;
            if (e >= nexp) continue;
#pragma unroll 16
            for (int c = 0; c < nchunk; ++c) {
                const int v = counts[(int64_t)c * nexp + e];
                total[j] += v;
                before[j] += c < me ? v : 0;
            }
        }
    }
    for (int e = lane; e < nexp; e += 64) place[wave][e] = 0;
    int32_t id[8];                              // 512 assignments at a time, the loads together
    auto load = [&](int64_t b) {
#pragma unroll
        for (int r = 0; r < 8; ++r) id[r] = b + r * 64 + lane < w1 ? ids[b + r * 64 + lane] : -1;
    };
    for (int64_t b = w0; b < w1; b += 512) {
        load(b);
#pragma unroll
        for (int r = 0; r < 8; ++r)
            if ((uint32_t)id[r] < (uint32_t)nexp) atomicAdd(&place[wave][id[r]], 1);
    }
    __syncthreads();
    int sum = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int e = PER * tid + j;
        if (nchunk == 1 && e < nexp) {
            for (int w = 0; w < NW; ++w) total[j] += place[w][e];
        }
        sum += total[j];
    }
    int inc = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int up = __shfl_up(inc, o, 64);
        if (lane >= o) inc += up;
    }
    if (lane == 63) part[wave] = inc;
    __syncthreads();
    int base = inc - sum, all = 0;
    for (int w = 0; w < NW; ++w) {
        base += w < wave ? part[w] : 0;
        all += part[w];
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int e = PER * tid + j;
        if (e < nexp) {
            if (me == 0) offsets[e] = base;
            int p = base + before[j], c[NW];    // where each wave's first of this expert goes
#pragma unroll
            for (int w = 0; w < NW; ++w) c[w] = place[w][e];
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                place[w][e] = p;
                p += c[w];
            }
        }
        base += total[j];
    }
    if (me == 0 && tid == 0) offsets[nexp] = all;
    __syncthreads();
    for (int64_t b = w0; b < w1; b += 512) {
        if (w1 - w0 > 512) load(b);             // (otherwise they are still there)
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            const bool on = (uint32_t)id[r] < (uint32_t)nexp;
            const uint64_t same = rg_same(id[r], on);
            if (on) {
                const uint32_t i = (uint32_t)(b + r * 64 + lane);
                const int rank = __popcll(same & ((1ull << lane) - 1));
                const int p = place[wave][id[r]] + rank;
                rows[p] = (int32_t)(i / (uint32_t)k);
                slots[p] = (int32_t)i;
                if (rank == 0) place[wave][id[r]] += __popcll(same);
            }
        }
    }
    // (each chunk clears its share of what no expert took)
    for (int64_t i = i0 + tid; i < i1; i += NW * 64) {
        if (i >= all) {
            rows[i] = -1;
            slots[i] = -1;
        }
    }
}
