// trench-gguf_amd/csrc/mxmul.cuh - products of rows with stored MXFP4 matrices: y[r][n] = sum_k x[r][k] w[e][n][k],
// with e the matrix of r's group, and with SwiGLU of two such products, y = g / (1 + exp(-g)) * u.
//
// The weights come packed (mxfp4.cuh). BF16 rows meet them as BF16: a code times its scale is exact there, products are
// exact in f32 and the sums are held in f32. F32 and F16 rows come as sums of 3 and 2 BF16 rows (k_mx_split), summed
// piece by piece into the same f32 sums, so no bit of them is lost. Packed MXFP4 rows meet the packed weights in the
// scaled matrix instructions. A product is a matrix instruction with w's rows as its rows and x's as its columns, so a
// lane ends up with 4 consecutive outputs of one row. The order of k inside an instruction is free as long as both
// sides agree: lane group q takes k = 32 q .. 32 q + 31 of every 128, which are one 16-byte piece of codes under one
// scale, and instruction c of four takes 8 c .. 8 c + 7 of those.
#pragma once
#include "mxfp4.cuh"

typedef int mx_i8 __attribute__((ext_vector_type(8)));

struct MxMulArgs {
    const uint8_t *x;           // BF16 rows (pieces of F16 and F32 rows one after the other), or codes (rows layout)
    const uint8_t *xs;          // scales (rows layout)
    int64_t nx, xrow;           // rows of x and bytes from row to row
    int64_t kx;                 // BF16: values of a row that are there, its pieces together (the rest counts as zero)
    int pieces;
    const uint8_t *w, *ws, *u, *us;     // codes and scales (tiles layout), u and us of the second product
    int64_t nmat, ne1, strips;  // strips of 16 rows of a matrix
    int nk;                     // 128-value pieces of a row of w that hold values
    int nc;                     // 512-value pieces of a row of w (the last may be part padding)
    const int32_t *offsets, *rows;
    int64_t m;
    void *y;
    int ytype;
    int mt;                     // row tiles of the grid (an upper bound with offsets)
};

static __device__ __align__(16) uint32_t mx_zero[4];

DEV uint32_t mx_bf16(float f) {          // to nearest even; NaN stays one
    const uint32_t u = fbits(f);
    if ((u & 0x7fffffffu) > 0x7f800000u) return (u >> 16) | 0x40u;
    return (u + 0x7fffu + ((u >> 16) & 1)) >> 16;
}
DEV uint32_t mx_f16(float f) {
    union { _Float16 h; uint16_t u; } c = {(_Float16)f};
    return c.u;
}

DEV float mx_glu(float g, float u) { return g / (1.f + expf(-g)) * u; }

// y[row][n .. n + 3], the part of it that is there
DEV void mx_store4(const MxMulArgs &a, int64_t row, int64_t n, const float (&v)[4]) {
    const int64_t at = row * a.ne1 + n;
    const bool whole = n + 4 <= a.ne1 && a.ne1 % 4 == 0;
    if (a.ytype == T_F32) {
        float *y = (float *)a.y + at;
        if (whole) {
            *(float4 *)y = make_float4(v[0], v[1], v[2], v[3]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (n + i < a.ne1) y[i] = v[i];
        }
    } else {
        uint16_t *y = (uint16_t *)a.y + at;
        uint32_t h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = a.ytype == T_BF16 ? mx_bf16(v[i]) : mx_f16(v[i]);
        if (whole) {
            *(uint2 *)y = make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (n + i < a.ne1) y[i] = (uint16_t)h[i];
        }
    }
}

// group e's rows [r0, r1), kept inside [0, m) whatever the offsets say; group nmat is what no expert has
DEV void mx_group(const MxMulArgs &a, int64_t e, int64_t &r0, int64_t &r1) {
    if (!a.offsets) {
        r0 = e ? a.m : 0;
        r1 = a.m;
        return;
    }
    const int64_t o0 = a.offsets[e], o1 = e < a.nmat ? a.offsets[e + 1] : a.m;
    r0 = o0 < 0 ? 0 : o0 > a.m ? a.m : o0;
    r1 = o1 < r0 ? r0 : o1 > a.m ? a.m : o1;
}

// the row of x that output row r reads, or -1
DEV int64_t mx_row(const MxMulArgs &a, int64_t r) {
    const int64_t i = a.rows ? a.rows[r] : r;
    return i >= 0 && i < a.nx ? i : -1;
}

// 8 codes -> 8 BF16 at scale s (a power of two as f32)
DEV mx_bf8 mx_widen(uint32_t codes, float s) {
    union { mx_bf2 v[4]; mx_bf8 b; } r;
    r.v[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 0);
    r.v[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 1);
    r.v[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 2);
    r.v[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 3);
    return r.b;
}

DEV mx_i8 mx_wide(uint4 v) { return mx_i8{(int)v.x, (int)v.y, (int)v.z, (int)v.w, 0, 0, 0, 0}; }

// ---- few rows a group: a workgroup owns 16 columns of one group, its 8 waves split k by 128-value pieces and their
// sums meet in LDS in a fixed order; MF x 16 rows at a time. grid (ceil(ne1 / 16), groups + 1)
template <bool FP4, int MF, bool GLU>
__global__ __launch_bounds__(512) void k_mx_rows(MxMulArgs a) {
    constexpr int G = GLU ? 2 : 1;
    __shared__ mx_f4 red[8][MF * G][64];
    const int tid = threadIdx.x, lane = lane_id(), wave = tid >> 6, q = lane >> 4;
    const int64_t e = blockIdx.y, n0 = (int64_t)blockIdx.x * 16;
    int64_t r0, r1;
    mx_group(a, e, r0, r1);
    if (e == a.nmat) {          // rows that belong to no expert
        for (int64_t i = r0 * 4 + tid; i < r1 * 4; i += 512) {
            const float z[4] = {0.f, 0.f, 0.f, 0.f};
            if (n0 + 4 * (i & 3) < a.ne1) mx_store4(a, i >> 2, n0 + 4 * (i & 3), z);
        }
        return;
    }
    const int64_t strip = e * a.strips + blockIdx.x;
    const uint8_t *wp[2] = {a.w + strip * a.nc * 4096 + 16 * lane, GLU ? a.u + strip * a.nc * 4096 + 16 * lane : nullptr};
    const uint8_t *sp[2] = {a.ws + strip * a.nc * 256 + 4 * lane, GLU ? a.us + strip * a.nc * 256 + 4 * lane : nullptr};
    for (int64_t m0 = r0; m0 < r1; m0 += 16 * MF) {
        mx_f4 acc[MF][G];
        const uint8_t *xp[MF];
        const uint8_t *xsp[MF];
#pragma unroll
        for (int f = 0; f < MF; ++f) {
            const int64_t r = m0 + 16 * f + (lane & 15);
            const int64_t i = mx_row(a, r < r1 ? r : r1 - 1);
            xp[f] = a.x + (i < 0 ? 0 : i) * a.xrow;
            xsp[f] = FP4 ? a.xs + (i < 0 ? 0 : i) * 16 + 4 * q : nullptr;
#pragma unroll
            for (int g = 0; g < G; ++g) acc[f][g] = mx_f4{0.f, 0.f, 0.f, 0.f};
        }
        for (int p = 0; p < a.pieces; ++p) {
            for (int c = wave; c < a.nk; c += 8) {
                uint4 wq[G];
                uint32_t sc[G];
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    wq[g] = *(const uint4 *)(wp[g] + (int64_t)c * 1024);
                    sc[g] = sp[g][(c >> 2) * 256 + (c & 3)];
                }
                if (FP4) {
#pragma unroll
                    for (int f = 0; f < MF; ++f) {
                        const uint4 xq = *(const uint4 *)(xp[f] + (int64_t)c * 64 + 16 * q);
                        const uint32_t xsc = xsp[f][(c >> 2) * a.nx * 16 + (c & 3)];
#pragma unroll
                        for (int g = 0; g < G; ++g)
                            acc[f][g] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                                mx_wide(wq[g]), mx_wide(xq), acc[f][g], 4, 4, 0, (int)sc[g], 0, (int)xsc);
                    }
                } else {
                    const int s = p * a.nk + c;
                    const bool in = (int64_t)s * 128 + 32 * q < a.kx;
                    mx_bf8 xv[MF][4];
#pragma unroll
                    for (int f = 0; f < MF; ++f) {
                        const uint8_t *xc = xp[f] + (int64_t)s * 256 + 64 * q;
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            xv[f][j] = *(const mx_bf8 *)(in ? xc + 16 * j : (const uint8_t *)mx_zero);
                    }
#pragma unroll
                    for (int g = 0; g < G; ++g) {
                        const float scale = ffrom(sc[g] << 23);
                        const uint32_t cw[4] = {wq[g].x, wq[g].y, wq[g].z, wq[g].w};
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const mx_bf8 wv = mx_widen(cw[j], scale);
#pragma unroll
                            for (int f = 0; f < MF; ++f)
                                acc[f][g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wv, xv[f][j], acc[f][g], 0, 0, 0);
                        }
                    }
                }
            }
        }
#pragma unroll
        for (int f = 0; f < MF; ++f)
#pragma unroll
            for (int g = 0; g < G; ++g) red[wave][f * G + g][lane] = acc[f][g];
        __syncthreads();
        for (int f = wave; f < MF; f += 8) {
            float v[G][4];
#pragma unroll
            for (int g = 0; g < G; ++g) {
                mx_f4 s = red[0][f * G + g][lane];
#pragma unroll
                for (int w = 1; w < 8; ++w) s += red[w][f * G + g][lane];
#pragma unroll
                for (int i = 0; i < 4; ++i) v[g][i] = s[i];
            }
            const int64_t r = m0 + 16 * f + (lane & 15), n = n0 + 4 * q;
            if (r < r1 && n < a.ne1) {
                const bool on = mx_row(a, r) >= 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (GLU) v[0][i] = mx_glu(v[0][i], v[G - 1][i]);
                    if (!on) v[0][i] = 0.f;
                }
                mx_store4(a, r, n, v[0]);
            }
        }
        __syncthreads();
    }
}

// ---- many rows: tiles of TM rows by TN columns

// the row tile t of the grid: its group and rows. Groups take ceil(rows / TM) tiles each, in order, the rows of no
// expert last. False for a tile past the last.
template <int TM> DEV bool mx_tile(const MxMulArgs &a, int t, int64_t &e, int64_t &r0, int64_t &r1) {
    if (!a.offsets) {
        e = 0;
        r0 = (int64_t)t * TM;
        r1 = a.m < r0 + TM ? a.m : r0 + TM;
        return r0 < a.m;
    }
    const int lane = lane_id();
    int base = 0;
    for (int64_t g0 = 0; g0 <= a.nmat; g0 += 64) {
        int64_t s0 = 0, s1 = 0;
        if (g0 + lane <= a.nmat) mx_group(a, g0 + lane, s0, s1);
        const int cnt = (int)((s1 - s0 + TM - 1) / TM);
        int inc = cnt;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int up = __shfl_up(inc, o, 64);
            if (lane >= o) inc += up;
        }
        const uint64_t here = __ballot(base + inc > t);
        if (here) {
            const int l = __ffsll((unsigned long long)here) - 1;
            const int skip = base + __shfl(inc, l, 64) - __shfl(cnt, l, 64);
            const int s0i = __shfl((int)s0, l, 64), s1i = __shfl((int)s1, l, 64);
            e = g0 + l;
            r0 = (int64_t)s0i + (int64_t)(t - skip) * TM;
            r1 = r0 + TM < s1i ? r0 + TM : s1i;
            return true;
        }
        base += __shfl(inc, 63, 64);
    }
    return false;
}

// 16 bytes a lane from g to l + 16 * lane (l the same in the wave), without registers between. Written out because the
// compiler lets every later read of LDS wait for the builtin's loads, which are for the buffer that is not being read:
// products then wait for the loads of the next step in every step. It names no register that the load writes; mx_sync
// waits for it. (The wait states are those of reading m0 after a scalar write.)
DEV void mx_to_lds(const void *g, void *l) {
    const uint32_t at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void *)l;
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
                 :: "s"(__builtin_amdgcn_readfirstlane(at)), "v"(g) : "memory");
}
// the loads into LDS have landed, for every wave
DEV void mx_sync() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

// WM x WN waves, each FM x 16 rows by FN x 16 columns (with GLU the first half of its FN strips are w's and the second
// the same columns of u). x goes through LDS, 256 bytes of every row a step (128 BF16 values or 512 codes), in two
// buffers: piece 4c + q of a row's 16, which lane group q takes into product c, lies at (4c + q) ^ (row & 15), so that
// the reads of 16 rows spread over the banks. A wave's weights go straight to its registers, a kilobyte of a strip at a
// time and one ahead: as codes they are a quarter of what BF16 rows take, and half of them are read twice.
template <bool FP4, int WM, int WN, int FM, int FN, bool GLU>
__global__ __launch_bounds__(WM * WN * 64) void k_mx_tile(MxMulArgs a) {
    constexpr int TM = WM * FM * 16, NS = WN * FN / (GLU ? 2 : 1), NO = NS * 16, NW = WM * WN, LD = TM / 4 / NW;
    constexpr int FH = GLU ? FN / 2 : FN;                   // strips of one matrix
    __shared__ __align__(1024) uint8_t xs[2 * TM * 256];
    __shared__ __align__(16) uint8_t xsc[FP4 ? 2 * TM * 16 : 16];
    const int tid = threadIdx.x, lane = lane_id(), q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave / WN, wn = wave % WN;
    const int nt = (int)((a.strips + NS - 1) / NS), total = nt * a.mt, per = (total + 7) / 8;
    const int id = (int)(blockIdx.x % 8) * per + (int)(blockIdx.x / 8);
    if ((int)(blockIdx.x / 8) >= per || id >= total) return;
    int64_t e, r0, r1;
    if (!mx_tile<TM>(a, id / nt, e, r0, r1)) return;
    const int64_t s0 = (int64_t)(id % nt) * NS;             // the tile's first strip
    if (e == a.nmat) {
        const float z[4] = {0.f, 0.f, 0.f, 0.f};
        for (int64_t i = tid; i < (r1 - r0) * (NO / 4); i += NW * 64) {
            const int64_t n = s0 * 16 + 4 * (i % (NO / 4));
            if (n < a.ne1) mx_store4(a, r0 + i / (NO / 4), n, z);
        }
        return;
    }
    // where this lane's 16-byte pieces of x come from
    const uint8_t *xp[LD];
#pragma unroll
    for (int i = 0; i < LD; ++i) {
        const int row = (wave * LD + i) * 4 + (lane >> 4);
        const int64_t r = r0 + row < r1 ? r0 + row : r1 - 1;
        const int64_t j = mx_row(a, r);
        const int p = (lane & 15) ^ (row & 15);
        xp[i] = a.x + (j < 0 ? 0 : j) * a.xrow + 16 * (FP4 ? p : 4 * (p & 3) + (p >> 2));
    }
    const uint8_t *sp = a.xs;               // FP4: a row's scales of 512 values, a lane each of the first TM
    if (FP4) {
        const int64_t r = r0 + tid < r1 ? r0 + tid : r1 - 1;
        const int64_t j = mx_row(a, r);
        sp += (j < 0 ? 0 : j) * 16;
    }
    const uint8_t *wp[FN], *wsp[FN];        // (uniform) this wave's strips, those past the last the last
#pragma unroll
    for (int f = 0; f < FN; ++f) {
        const int64_t t = s0 + wn * FH + f % FH, strip = e * a.strips + (t < a.strips ? t : a.strips - 1);
        wp[f] = (f < FH ? a.w : a.u) + strip * a.nc * 4096;
        wsp[f] = (f < FH ? a.ws : a.us) + strip * a.nc * 256;
    }
    mx_f4 acc[FN][FM];
#pragma unroll
    for (int f = 0; f < FN; ++f)
#pragma unroll
        for (int g = 0; g < FM; ++g) acc[f][g] = mx_f4{0.f, 0.f, 0.f, 0.f};
    const int steps = FP4 ? a.nc : a.nk * a.pieces;
    // part j of 4 of step s into its buffer
    auto stage = [&](int s, int j) {
        uint8_t *buf = xs + (s & 1) * (TM * 256);
        if (!FP4 && (int64_t)s * 128 + 128 > a.kx) {        // (the last step, of rows that end inside it)
#pragma unroll
            for (int i = j * LD / 4; i < (j + 1) * LD / 4; ++i) {
                const int p = (lane & 15) ^ (((wave * LD + i) * 4 + (lane >> 4)) & 15);
                const bool in = (int64_t)s * 128 + 8 * (4 * (p & 3) + (p >> 2)) < a.kx;
                mx_to_lds(in ? xp[i] : (const uint8_t *)mx_zero, buf + (wave * LD + i) * 1024);
            }
        } else {
#pragma unroll
            for (int i = j * LD / 4; i < (j + 1) * LD / 4; ++i) {
                mx_to_lds(xp[i], buf + (wave * LD + i) * 1024);
                xp[i] += 256;
            }
        }
        if (FP4 && j == 3 && wave * 64 < TM) mx_to_lds(sp + (int64_t)s * a.nx * 16, xsc + (s & 1) * (TM * 16) + wave * 1024);
    };
    uint4 wq[FN], wn_[FN];
    uint32_t sc[FN], sn[FN];
    auto fetch = [&](int c) {               // the weights' piece c
#pragma unroll
        for (int f = 0; f < FN; ++f) wn_[f] = *(const uint4 *)(wp[f] + (int64_t)c * 1024 + 16 * lane);
    };
    auto scales = [&](int c) {              // and the scales of its 512 values
#pragma unroll
        for (int f = 0; f < FN; ++f) sn[f] = *(const uint32_t *)(wsp[f] + (int64_t)c * 256 + 4 * lane);
    };
    int c = 0;                              // BF16: the piece at hand
#pragma unroll
    for (int j = 0; j < 4; ++j) stage(0, j);
    fetch(0);
    scales(0);
    mx_sync();
#pragma unroll 1
    for (int s = 0; s < steps; ++s) {
        const uint8_t *b = xs + (s & 1) * (TM * 256) + (wm * FM * 16 + (lane & 15)) * 256;
        const bool more = s + 1 < steps;
        uint32_t xc[FP4 ? FM : 1];
        const int next = FP4 ? s + 1 : c + 1 < a.nk ? c + 1 : 0;
        if (FP4) {
#pragma unroll
            for (int g = 0; g < FM; ++g)
                xc[g] = *(const uint32_t *)(xsc + (s & 1) * (TM * 16) + ((wm * FM + g) * 16 + (lane & 15)) * 16 + 4 * q);
#pragma unroll
            for (int f = 0; f < FN; ++f) sc[f] = sn[f];
            if (more) scales(next);
        } else {
#pragma unroll
            for (int f = 0; f < FN; ++f) {
                wq[f] = wn_[f];
                sc[f] = ((sn[f] >> (8 * (c & 3))) & 255) << 23;
            }
            if (more) {
                fetch(next);
                if ((next & 3) == 0) scales(next >> 2);
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (FP4) {
                if (4 * s + j >= a.nk) continue;            // (padding)
#pragma unroll
                for (int f = 0; f < FN; ++f) wq[f] = wn_[f];
                if (j < 3 || more) fetch(4 * s + j + 1);    // (the last piece of a row is followed by its scales at least)
            }
            if (more) stage(s + 1, j);
            mx_bf8 wv[FN];
            if (!FP4) {
#pragma unroll
                for (int f = 0; f < FN; ++f)
                    wv[f] = mx_widen(j == 0 ? wq[f].x : j == 1 ? wq[f].y : j == 2 ? wq[f].z : wq[f].w, ffrom(sc[f]));
            }
#pragma unroll
            for (int g = 0; g < FM; ++g) {
                const uint4 xv = *(const uint4 *)(b + g * 4096 + (((4 * j + q) ^ (lane & 15)) * 16));
                union { uint4 u; mx_bf8 b; } xb = {xv};
#pragma unroll
                for (int f = 0; f < FN; ++f) {
                    if (FP4) {
                        const mx_i8 wi = mx_wide(wq[f]), xi = mx_wide(xv);
                        const int ws = (int)sc[f], xw = (int)xc[FP4 ? g : 0];
                        acc[f][g] = j == 0   ? __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wi, xi, acc[f][g], 4, 4, 0, ws, 0, xw)
                                    : j == 1 ? __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wi, xi, acc[f][g], 4, 4, 1, ws, 1, xw)
                                    : j == 2 ? __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wi, xi, acc[f][g], 4, 4, 2, ws, 2, xw)
                                             : __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wi, xi, acc[f][g], 4, 4, 3, ws, 3, xw);
                    } else {
                        acc[f][g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wv[f], xb.b, acc[f][g], 0, 0, 0);
                    }
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        if (!FP4) c = next;
        mx_sync();
    }
#pragma unroll
    for (int g = 0; g < FM; ++g) {
        const int64_t r = r0 + (wm * FM + g) * 16 + (lane & 15);
        if (r >= r1) continue;
        const bool on = mx_row(a, r) >= 0;
#pragma unroll
        for (int f = 0; f < FH; ++f) {
            const int64_t n = (s0 + wn * FH + f) * 16 + 4 * q;
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = acc[f][g][i];
                if (GLU) v[i] = mx_glu(v[i], acc[(f + FH) % FN][g][i]);
                if (!on) v[i] = 0.f;
            }
            if (n < a.ne1) mx_store4(a, r, n, v);
        }
    }
}
