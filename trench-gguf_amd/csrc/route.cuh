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

DEV float rt_max(float v) {     // over the wave, in every lane
#pragma unroll
    for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}
DEV float rt_sum(float v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
template <int SRC> DEV float rt_load(const void *p, int64_t i) {
    if (SRC == T_F32) return ((const float *)p)[i];
    const uint32_t h = ((const uint16_t *)p)[i];
    return SRC == T_BF16 ? ffrom(h << 16) : h2f(h);
}

#define RT_NONE (-__builtin_inff())

// one wave a token; lane l holds experts l * P .. l * P + P - 1
template <int SRC, int P>
__global__ __launch_bounds__(256) void k_route(RouteArgs a) {
    __shared__ float keys[4][64 * P], gs[4][64];
    const int lane = lane_id(), wave = threadIdx.x >> 6;
    const int64_t t = (int64_t)blockIdx.x * 4 + wave;
    const bool live = t < a.ntok;
    const int64_t row = (live ? t : a.ntok - 1) * a.ld;
    float x[P], score[P], key[P];
    float mx = RT_NONE;
#pragma unroll
    for (int j = 0; j < P; ++j) {
        const int e = lane * P + j;
        float v = e < a.nexp ? rt_load<SRC>(a.logits, row + e) : RT_NONE;
        v = v == v ? fminf(v, 3.402823466e38f) : RT_NONE;
        x[j] = v;
        mx = fmaxf(mx, v);
    }
    float z = 1.f;
    if (a.sigmoid) {
#pragma unroll
        for (int j = 0; j < P; ++j) score[j] = 1.f / (1.f + expf(-x[j]));
    } else {
        mx = rt_max(mx);
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < P; ++j) {
            score[j] = x[j] == RT_NONE ? 0.f : expf(x[j] - mx);
            s += score[j];
        }
        z = rt_sum(s);
        z = z > 0.f ? z : 1.f;
#pragma unroll
        for (int j = 0; j < P; ++j) score[j] = score[j] / z;
    }
    const bool by_logit = !a.bias && a.ngroup == 1;
#pragma unroll
    for (int j = 0; j < P; ++j) {
        const int e = lane * P + j;
        float v = by_logit ? x[j] : score[j];
        if (a.bias && e < a.nexp) v += a.bias[e];
        key[j] = v == v && x[j] != RT_NONE ? v : RT_NONE;
    }
    if (a.ngroup > 1) {         // (uniform)
#pragma unroll
        for (int j = 0; j < P; ++j) keys[wave][lane * P + j] = key[j];
        __syncthreads();
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
        __syncthreads();
        int ahead = 0;          // groups that come before this one
        for (int i = 0; i < a.ngroup; ++i) ahead += gs[wave][i] > g || (gs[wave][i] == g && i < lane);
        const uint64_t kept = __ballot(lane < a.ngroup && ahead < a.keep);
#pragma unroll
        for (int j = 0; j < P; ++j) {
            const int e = lane * P + j;
            if (e < a.nexp && !((kept >> (e / per)) & 1)) key[j] = RT_NONE;
        }
    }
    int my_id = -1;
    float my_w = 0.f, sum = 0.f;
    for (int r = 0; r < a.k; ++r) {
        float v = key[0];
#pragma unroll
        for (int j = 1; j < P; ++j) v = fmaxf(v, key[j]);
        const float m = rt_max(v);
        if (m == RT_NONE) break;            // (uniform)
        const int owner = __ffsll((unsigned long long)__ballot(v == m)) - 1;
        int at = 0;
        float s = 0.f;
        bool found = false;
#pragma unroll
        for (int j = 0; j < P; ++j) {
            const bool hit = !found && key[j] == m;
            at = hit ? j : at;
            s = hit ? score[j] : s;
            found |= hit;
            if (hit && lane == owner) key[j] = RT_NONE;
        }
        s = __shfl(s, owner, 64);
        at = __shfl(at, owner, 64);
        sum += s;
        if (lane == r) {
            my_id = owner * P + at;
            my_w = s;
        }
    }
    if (live && lane < a.k) {
        const float w = !a.renorm ? my_w : sum > 0.f ? my_w / sum : 0.f;
        a.ids[t * a.k + lane] = my_id;
        a.weights[t * a.k + lane] = w * a.scale;
    }
}

// ---- grouping: assignments (flat ids [n]) sorted by expert, in order within each. Chunks of RG_CHUNK assignments, a
// workgroup each: counts per expert and chunk, then every chunk places its own from the counts of all.
#define RG_CHUNK 2048
#define RG_MAXE 1024

// counts[e][chunk]
__global__ __launch_bounds__(256) void k_group_count(const int32_t *__restrict__ ids, int64_t n, int nexp, int nchunk,
                                                     int32_t *__restrict__ counts) {
    __shared__ int hist[RG_MAXE];
    for (int e = threadIdx.x; e < nexp; e += 256) hist[e] = 0;
    __syncthreads();
    const int64_t i0 = (int64_t)blockIdx.x * RG_CHUNK, i1 = i0 + RG_CHUNK < n ? i0 + RG_CHUNK : n;
    for (int64_t i = i0 + threadIdx.x; i < i1; i += 256) {
        const uint32_t e = (uint32_t)ids[i];
        if (e < (uint32_t)nexp) atomicAdd(&hist[e], 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < nexp; e += 256) counts[(int64_t)e * nchunk + blockIdx.x] = hist[e];
}

// offsets [nexp + 1], rows [n] (the token of each sorted assignment), slots [n] (its flat index); the places past
// offsets[nexp] (ids that name no expert) get -1. counts is null where there is one chunk.
__global__ __launch_bounds__(256) void k_group_place(const int32_t *__restrict__ ids, int64_t n, int k, int nexp,
                                                     int nchunk, const int32_t *__restrict__ counts,
                                                     int32_t *__restrict__ offsets, int32_t *__restrict__ rows,
                                                     int32_t *__restrict__ slots) {
    __shared__ int total[RG_MAXE], before[RG_MAXE], part[4], place[4][RG_MAXE];
    const int tid = threadIdx.x, lane = lane_id(), wave = tid >> 6, chunk = blockIdx.x;
    const int64_t i0 = (int64_t)chunk * RG_CHUNK, i1 = i0 + RG_CHUNK < n ? i0 + RG_CHUNK : n;
    for (int e = tid; e < 4 * RG_MAXE; e += 256) (&place[0][0])[e] = 0;
    __syncthreads();
    // each wave counts its own quarter of the chunk
    const int64_t w0 = i0 + wave * (RG_CHUNK / 4);
    int32_t id[RG_CHUNK / 256];
#pragma unroll
    for (int r = 0; r < RG_CHUNK / 256; ++r) {
        const int64_t i = w0 + r * 64 + lane;
        id[r] = i < i1 ? ids[i] : -1;
        if ((uint32_t)id[r] < (uint32_t)nexp) atomicAdd(&place[wave][id[r]], 1);
        else id[r] = -1;
    }
    __syncthreads();
    // the whole call's totals and what earlier chunks hold
    if (nchunk == 1) {
        for (int e = tid; e < nexp; e += 256) {
            total[e] = place[0][e] + place[1][e] + place[2][e] + place[3][e];
            before[e] = 0;
        }
    } else {
        for (int e = wave; e < nexp; e += 4) {
            int s = 0, b = 0;
            for (int c = lane; c < nchunk; c += 64) {
                const int v = counts[(int64_t)e * nchunk + c];
                s += v;
                b += c < chunk ? v : 0;
            }
#pragma unroll
            for (int o = 32; o; o >>= 1) {
                s += __shfl_xor(s, o, 64);
                b += __shfl_xor(b, o, 64);
            }
            if (lane == 0) {
                total[e] = s;
                before[e] = b;
            }
        }
    }
    __syncthreads();
    // exclusive scan of the totals: 4 experts a thread
    int t[4], sum = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        t[j] = 4 * tid + j < nexp ? total[4 * tid + j] : 0;
        sum += t[j];
    }
    int inc = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int up = __shfl_up(inc, o, 64);
        if (lane >= o) inc += up;
    }
    if (lane == 63) part[wave] = inc;
    __syncthreads();
    int base = inc - sum;
    for (int w = 0; w < wave; ++w) base += part[w];
    const int all = part[0] + part[1] + part[2] + part[3];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int e = 4 * tid + j;
        if (e < nexp) {
            if (chunk == 0) offsets[e] = base;
            int p = base + before[e];           // where each wave's first of this expert goes
            for (int w = 0; w < 4; ++w) {
                const int c = place[w][e];
                place[w][e] = p;
                p += c;
            }
        }
        base += t[j];
    }
    if (chunk == 0 && tid == 0) offsets[nexp] = all;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < RG_CHUNK / 256; ++r) {
        const int64_t i = w0 + r * 64 + lane;
        const bool on = id[r] >= 0;
        uint64_t same = __ballot(on);
#pragma unroll
        for (int b = 0; b < 10; ++b) {
            const uint64_t bit = __ballot((id[r] >> b) & 1);
            same &= (id[r] >> b) & 1 ? bit : ~bit;
        }
        if (on) {
            const int rank = __popcll(same & ((1ull << lane) - 1));
            const int p = place[wave][id[r]] + rank;
            rows[p] = (int32_t)(i / k);
            slots[p] = (int32_t)i;
            if (rank == 0) place[wave][id[r]] += __popcll(same);
        }
    }
    // (each chunk clears its share of what no expert took)
    for (int64_t i = i0 + tid; i < i1; i += 256) {
        if (i >= all) {
            rows[i] = -1;
            slots[i] = -1;
        }
    }
}
