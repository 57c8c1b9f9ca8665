// trench-gguf_amd/csrc/mxfp4.cuh - microscaled 4-bit floats: rounding to MXFP4, its packed layout, and the exact
// split of wider rows into BF16 summands.
//
// A block of 32 values shares the scale 2^(e - 127), e = floor(log2(largest magnitude)) - 2 + 127 clamped to [0, 252]
// (the largest e2m1 value is 6 = 1.5 * 2^2), and each value becomes the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 with its
// sign; a tie goes to the smaller magnitude, a magnitude past 6 to 6, and a value that rounds to zero is +0. The
// division by the scale is a multiplication by a power of two and so exact. NaN counts as zero, an infinity as the
// largest magnitude there is.
//
// Two layouts for products, of rows padded to np = n_per_row rounded up to 512, the padding zero codes at zero scales:
//   rows (what products multiply; any row can be picked): codes [nrow][np / 2] bytes, value 2i in the low nibble of byte
//     i; then scales [np / 512][nrow][16], block 4c + q of the 16 at byte 4q + c.
//   tiles (stored matrices, each padded to whole strips of 16 rows): codes [strip][np / 128][64][16], piece 16q + r the
//     codes of row r's block q of the 128; then scales [strip][np / 512][64][4], byte c of piece 16q + r row r's block
//     4c + q. A strip's 128 columns are one kilobyte in the order in which the lanes of a 16 x 16 x 128 product take
//     them, so a wave loads its operand from 8 whole lines (from rows 3584 bytes apart the same bytes came as 16 half
//     lines, and the products waited for the loads: 4096 x 2048 x 7168 took 183 us with the rows of x left out and 135
//     with these loads left out too).
#pragma once
#include "common.cuh"

typedef __bf16 mx_bf8 __attribute__((ext_vector_type(8)));
typedef __bf16 mx_bf2 __attribute__((ext_vector_type(2)));
typedef float mx_f4 __attribute__((ext_vector_type(4)));

#define MX_PAD 512
inline __host__ __device__ int64_t mx_padded(int64_t n) { return (n + MX_PAD - 1) / MX_PAD * MX_PAD; }

// n / d for n < 2^31 as a multiplication and a shift
struct MxDiv {
    uint32_t d, mul, shift;
    DEV uint32_t div(uint32_t n) const { return (uint32_t)(((uint64_t)__umulhi(n, mul) + n) >> shift); }
};
inline MxDiv mx_div(uint32_t d) {
    uint32_t s = 0;
    while ((1ull << s) < d) ++s;
    return MxDiv{d, (uint32_t)((((1ull << s) - d) << 32) / d + 1), s};
}

template <int CTRL> DEV uint32_t mx_quad(uint32_t v) {      // a fixed exchange within each 4 lanes
    return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xf, 0xf, true);
}

// four nibbles -> the low nibbles of four bytes
DEV uint32_t mx_spread(uint32_t h) {
    h = (h | (h << 8)) & 0x00ff00ffu;
    return (h | (h << 4)) & 0x0f0f0f0fu;
}
// the low nibbles of four bytes -> four nibbles
DEV uint32_t mx_gather(uint32_t b) {
    b = (b | (b >> 4)) & 0x00ff00ffu;
    return (b | (b >> 8)) & 0xffffu;
}

// 8 source values
template <int SRC> DEV void mx_load8(const void *src, int64_t i, float (&v)[8]) {
    if (SRC == T_F32) {
        const float4 a = *(const float4 *)((const float *)src + i), b = *(const float4 *)((const float *)src + i + 4);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
        const uint4 a = *(const uint4 *)((const uint16_t *)src + i);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (SRC == T_BF16) {
                v[2 * j] = ffrom(w[j] << 16);
                v[2 * j + 1] = ffrom(w[j] & 0xffff0000u);
            } else {
                union { uint32_t u; _Float16 h[2]; } c = {w[j]};
                v[2 * j] = (float)c.h[0];
                v[2 * j + 1] = (float)c.h[1];
            }
        }
    }
}

// the code of v at the scale whose reciprocal is inv
DEV uint32_t mx_code(float v, float inv) {
    const float t = fabsf(v) * inv;
    const uint32_t c = (uint32_t)(t > 0.25f) + (t > 0.75f) + (t > 1.25f) + (t > 1.75f) + (t > 2.5f) + (t > 3.5f) +
                       (t > 5.f);
    return c ? c | ((fbits(v) >> 28) & 8u) : 0u;
}

// 8 codes and their block's scale exponent -> 8 BF16 values (exact: a value is at least 2^-128)
DEV uint4 mx_values(uint32_t codes, uint32_t e) {
    const float s = ffrom(e << 23);
    union { mx_bf2 v[4]; uint4 u; } r;
    r.v[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 0);
    r.v[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 1);
    r.v[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 2);
    r.v[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 3);
    return r.u;
}

struct MxQuantArgs {
    const void *src;
    int64_t ld;                 // source elements from row to row (MXFP4: unused, rows are whole blocks)
    uint8_t *dst, *scales;      // blocks, or codes and scales
    uint16_t *values;           // BF16, or null
    int64_t ncol, nrow;         // columns, and rows of a matrix (rows: of all of them together)
    int64_t row0;               // the launch's first strip
    uint32_t nblk, nb;          // blocks of this launch (blocks), and those of a row
    MxDiv row;                  // blocks of a row (blocks), strips of a matrix
};

enum { MX_BLOCKS = 0, MX_ROWS = 1, MX_TILES = 2 };

// 8 values of a block (quarter a of it): the source's, zero where the block holds none
template <int SRC> DEV void mx_source(const MxQuantArgs &p, int64_t row, uint32_t col, bool real, int a, float (&v)[8],
                                      uint32_t (&raw)[3]) {
    if (SRC == T_MXFP4) {
        const uint8_t *blk = (const uint8_t *)p.src + (real ? row * p.nb + col : 0) * 17;
        raw[2] = blk[0];
        __builtin_memcpy(&raw[0], blk + 1 + 8 * (a & 1), 8);
        if (!real) raw[0] = raw[1] = raw[2] = 0;
    } else {
        mx_load8<SRC>(p.src, (real ? row * p.ld + (int64_t)col * 32 : 0) + 8 * a, v);
        if (!real) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = 0.f;
        }
    }
}
// their codes and the block's scale exponent (over the 4 lanes that share it)
template <int SRC> DEV uint32_t mx_encode(int a, const float (&v)[8], const uint32_t (&raw)[3], uint32_t &e) {
    uint32_t codes = 0;
    if (SRC == T_MXFP4) {
        const int sh = 4 * (a >> 1);
        codes = mx_gather((raw[0] >> sh) & 0x0f0f0f0fu) | (mx_gather((raw[1] >> sh) & 0x0f0f0f0fu) << 16);
        e = raw[2];
    } else {
        float m = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(v[j]));             // (a NaN is passed over)
        m = fmaxf(m, ffrom(mx_quad<0xB1>(fbits(m))));
        m = fmaxf(m, ffrom(mx_quad<0x4E>(fbits(m))));
        const int x = (int)(fbits(m) >> 23) - 2;
        e = (uint32_t)(x < 0 ? 0 : x > 252 ? 252 : x);
        const float inv = ffrom((254 - e) << 23);
#pragma unroll
        for (int j = 0; j < 8; ++j) codes |= mx_code(v[j], inv) << (4 * j);
    }
    return codes;
}

// blocks: four lanes a block, 8 values a lane, MX_U blocks a lane; the 17-byte blocks of a workgroup leave through LDS
#define MX_U 4
template <int SRC>
__global__ __launch_bounds__(256) void k_mx_blocks(MxQuantArgs p) {
    __shared__ __align__(16) uint8_t out[MX_U * 64 * 17];
    const int tid = threadIdx.x, a = tid & 3;
    const uint32_t b0 = blockIdx.x * (MX_U * 64) + (tid >> 2);
    float v[MX_U][8];
    uint32_t raw[3], row[MX_U], col[MX_U];
#pragma unroll
    for (int u = 0; u < MX_U; ++u) {
        const uint32_t b = b0 + 64 * u < p.nblk ? b0 + 64 * u : p.nblk - 1;
        row[u] = p.row.div(b);
        col[u] = b - row[u] * p.row.d;
        mx_source<SRC>(p, row[u], col[u], true, a, v[u], raw);
    }
#pragma unroll
    for (int u = 0; u < MX_U; ++u) {
        uint32_t e;
        const uint32_t codes = mx_encode<SRC>(a, v[u], raw, e);
        if (p.values && b0 + 64 * u < p.nblk)
            *(uint4 *)(p.values + (int64_t)row[u] * p.ncol + col[u] * 32 + 8 * a) = mx_values(codes, e);
        // ggml's block: e, then byte j = value j | value j + 16 << 4; lane a gets bytes 4a .. 4a + 3
        const uint32_t lo = mx_quad<0x50>(codes) >> (16 * (a & 1)), hi = mx_quad<0xFA>(codes) >> (16 * (a & 1));
        const uint32_t w = mx_spread(lo & 0xffffu) | (mx_spread(hi & 0xffffu) << 4);
        uint8_t *o = out + (u * 64 + (tid >> 2)) * 17;
        if (a == 0) o[0] = (uint8_t)e;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[1 + 4 * a + j] = (uint8_t)(w >> (8 * j));
    }
    __syncthreads();
    const uint32_t first = blockIdx.x * (MX_U * 64);
    const uint32_t n = (p.nblk - first < MX_U * 64 ? p.nblk - first : MX_U * 64) * 17;
    uint8_t *d = p.dst + (int64_t)first * 17;
    for (uint32_t i = tid * 16; i < n; i += 256 * 16) {
        if (i + 16 <= n) {
            *(uint4 *)(d + i) = *(const uint4 *)(out + i);
        } else {
            for (uint32_t j = i; j < n; ++j) d[j] = out[j];
        }
    }
}

// rows and tiles: a workgroup writes 512 columns of 16 rows, four pieces of 128; grid (np / 512, strips of the launch).
// (Rows made block by block, a row's scales of 512 columns apart from the next row's in time and place, took 46 us of
// 8192 x 7168 BF16 values, and MX_ROWS_US so: 16 rows' scales are two whole lines.)
template <int SRC, bool TILES>
__global__ __launch_bounds__(256) void k_mx_strips(MxQuantArgs p) {
    __shared__ uint32_t es[64];
    const int tid = threadIdx.x, a = tid & 3, q = (tid >> 2) & 3, r = tid >> 4;
    const uint32_t strip = (uint32_t)p.row0 + blockIdx.y, mat = p.row.div(strip);
    const int64_t in_mat = (int64_t)(strip - mat * p.row.d) * 16 + r, row = mat * p.nrow + in_mat;
    const bool has = in_mat < p.nrow;
    float v[4][8];
    uint32_t raw[4][3];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const uint32_t col = blockIdx.x * 16 + 4 * c + q;
        mx_source<SRC>(p, row, col, has && col < p.nb, a, v[c], raw[c]);
    }
    uint8_t *d = TILES ? p.dst + ((int64_t)strip * gridDim.x + blockIdx.x) * 4096 + (16 * q + r) * 16 + 4 * a
                       : p.dst + (row * gridDim.x + blockIdx.x) * 256 + 16 * q + 4 * a;
    uint32_t all = 0;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const uint32_t col = blockIdx.x * 16 + 4 * c + q;
        uint32_t e;
        const uint32_t codes = mx_encode<SRC>(a, v[c], raw[c], e);
        all |= e << (8 * c);
        if (TILES || has) *(uint32_t *)(d + c * (TILES ? 1024 : 64)) = codes;
        if (p.values && has && col < p.nb)
            *(uint4 *)(p.values + row * p.ncol + col * 32 + 8 * a) = mx_values(codes, e);
    }
    if (a == 0) es[TILES ? 16 * q + r : 4 * r + q] = all;
    __syncthreads();
    if (TILES) {
        if (tid < 64) *(uint32_t *)(p.scales + ((int64_t)strip * gridDim.x + blockIdx.x) * 256 + 4 * tid) = es[tid];
    } else if (tid < 64 && (int64_t)strip * 16 + (tid >> 2) < p.nrow) {       // (rows: one matrix of them all)
        *(uint32_t *)(p.scales + ((int64_t)blockIdx.x * p.nrow + (int64_t)strip * 16) * 16 + 4 * tid) = es[tid];
    }
}

// F32 / F16 rows as sums of BF16 rows: the top 16 bits, then those of the rest, which holds every bit of an F16 value
// in 2 pieces and of an F32 value in 3 (8 bits each). out [nrow][PIECES][kp], kp = ncol rounded up to 128, zero-padded;
// one lane 8 values; grid (ceil(kp / 8 / 256), rows)
template <int SRC, int PIECES>
__global__ __launch_bounds__(256) void k_mx_split(const void *__restrict__ src, int64_t ld, int64_t ncol, int64_t kp,
                                                  int64_t nrow, uint16_t *__restrict__ out) {
    const int64_t c = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
    if (c >= kp) return;
    for (int64_t r = blockIdx.y; r < nrow; r += gridDim.y) {
        float v[8];
        if (c < ncol) {
            mx_load8<SRC>(src, r * ld + c, v);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = 0.f;
        }
#pragma unroll
        for (int q = 0; q < PIECES; ++q) {
            uint32_t w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t b = fbits(v[j]);
                const bool fin = (b & 0x7f800000u) != 0x7f800000u;
                w[j] = (b >> 16) | (!fin && (b & 0x7fffffu) ? 0x40u : 0u);      // (a NaN stays one)
                v[j] = fin ? v[j] - ffrom(b & 0xffff0000u) : 0.f;
            }
            *(uint4 *)(out + (r * PIECES + q) * kp + c) =
                make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
        }
    }
}
