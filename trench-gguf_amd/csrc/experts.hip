// trench-gguf_amd/csrc/experts.hip - the expert-layer entry points of libgpuq.so: rounding to MXFP4, products with
// stored MXFP4 matrices, a router's choice of experts and the grouping of rows by expert (declared, with their
// conventions, in include/gpuq.h).
#include <hip/hip_runtime.h>

#include "mxfp4.cuh"
#include "mxmul.cuh"
#include "route.cuh"

__attribute__((visibility("hidden"))) int gq_device(void);      // the device gpuq_init chose, -1 before it

namespace {

bool float_type(int t) { return t == T_F32 || t == T_F16 || t == T_BF16; }
int64_t type_size(int t) { return t == T_F32 ? 4 : 2; }
bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }
constexpr int64_t MAX_BLOCKS = (int64_t)1 << 30;                // of a launch (32-bit block numbers)
constexpr int64_t MAX_ROWS = (int64_t)1 << 30;

int64_t packed_bytes(int64_t nrow, int64_t n) { return nrow * (mx_padded(n) / 2 + mx_padded(n) / 32); }

// a row length of whole blocks whose padded rows stay countable
bool cols_ok(int64_t n) { return n > 0 && n % 32 == 0 && n <= (int64_t)1 << 24; }

template <int SRC> void launch_quantize(bool packed, const MxQuantArgs &p, hipStream_t st) {
    const unsigned grid = (unsigned)((p.nblk + MX_U * 64 - 1) / (MX_U * 64));
    if (packed) hipLaunchKernelGGL((k_mx_quantize<SRC, true>), dim3(grid), dim3(256), 0, st, p);
    else hipLaunchKernelGGL((k_mx_quantize<SRC, false>), dim3(grid), dim3(256), 0, st, p);
}

int pieces_of(int x_type) { return x_type == T_F32 ? 3 : x_type == T_F16 ? 2 : 1; }
int64_t round128(int64_t n) { return (n + 127) / 128 * 128; }

template <int MF> void launch_rows(bool fp4, bool glu, const MxMulArgs &a, hipStream_t st) {
    const dim3 grid((unsigned)((a.ne1 + 15) / 16), (unsigned)(a.offsets ? a.nmat + 1 : 1));
#define MX_ROWS(F, G) hipLaunchKernelGGL((k_mx_rows<F, MF, G>), grid, dim3(512), 0, st, a)
    if (fp4) {
        if (glu) MX_ROWS(true, true);
        else MX_ROWS(true, false);
    } else {
        if (glu) MX_ROWS(false, true);
        else MX_ROWS(false, false);
    }
#undef MX_ROWS
}

template <int WM, int WN, int FM, int FN> bool launch_tile(bool fp4, bool glu, MxMulArgs &a, hipStream_t st) {
    constexpr int TM = WM * FM * 16, TN = WN * FN * 16;
    const int64_t no = glu ? TN / 2 : TN, nt = (a.ne1 + no - 1) / no;
    const int64_t mt = (a.m + TM - 1) / TM + (a.offsets ? a.nmat + 1 : 0);
    if (nt * mt >= ((int64_t)1 << 30)) return false;
    a.mt = (int)mt;
    const dim3 grid((unsigned)((nt * mt + 7) / 8 * 8)), block(WM * WN * 64);
    if (fp4) {
        if (glu) hipLaunchKernelGGL((k_mx_tile4<WM, WN, FM, FN, true>), grid, block, 0, st, a);
        else hipLaunchKernelGGL((k_mx_tile4<WM, WN, FM, FN, false>), grid, block, 0, st, a);
    } else {
        if (glu) hipLaunchKernelGGL((k_mx_tile<WM, WN, FM, FN, true>), grid, block, 0, st, a);
        else hipLaunchKernelGGL((k_mx_tile<WM, WN, FM, FN, false>), grid, block, 0, st, a);
    }
    return true;
}

template <int SRC> bool launch_route(const RouteArgs &a, hipStream_t st) {
    const dim3 grid((unsigned)((a.ntok + 3) / 4));
    if (a.nexp <= 64) hipLaunchKernelGGL((k_route<SRC, 1>), grid, dim3(256), 0, st, a);
    else if (a.nexp <= 128) hipLaunchKernelGGL((k_route<SRC, 2>), grid, dim3(256), 0, st, a);
    else if (a.nexp <= 256) hipLaunchKernelGGL((k_route<SRC, 4>), grid, dim3(256), 0, st, a);
    else if (a.nexp <= 384) hipLaunchKernelGGL((k_route<SRC, 6>), grid, dim3(256), 0, st, a);
    else if (a.nexp <= 512) hipLaunchKernelGGL((k_route<SRC, 8>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((k_route<SRC, 16>), grid, dim3(256), 0, st, a);
    return hipGetLastError() == hipSuccess;
}

}  // namespace

extern "C" size_t gpuq_mxfp4_packed_bytes(int64_t nrow, int64_t n_per_row) {
    if (nrow <= 0 || nrow >= ((int64_t)1 << 40) / 32 || !cols_ok(n_per_row)) return 0;
    return (size_t)packed_bytes(nrow, n_per_row);
}

extern "C" size_t gpuq_mxfp4_quantize_dev(int src_type, const void *d_src, int64_t nrow, int64_t n_per_row, int64_t ld,
                                          int packed, void *d_dst, void *d_values, void *stream) {
    if (gq_device() < 0 || !d_src || !d_dst || !gpuq_mxfp4_packed_bytes(nrow, n_per_row)) return 0;
    if (packed != 0 && packed != 1) return 0;
    if (!aligned16(d_dst) || !aligned16(d_values)) return 0;
    if (src_type == T_MXFP4) {
        if (!packed || ld != n_per_row) return 0;
    } else if (!float_type(src_type) || ld < n_per_row || ld > ((int64_t)1 << 40) || !aligned16(d_src) ||
               ld * type_size(src_type) % 16) {
        return 0;
    }
    const int64_t nb = n_per_row / 32, stored = packed ? mx_padded(n_per_row) / 32 : nb, rows_max = MAX_BLOCKS / stored;
    uint8_t *dst = (uint8_t *)d_dst, *scales = dst + nrow * stored * 16;
    for (int64_t r = 0; r < nrow; r += rows_max) {
        const int64_t n = nrow - r < rows_max ? nrow - r : rows_max;
        MxQuantArgs p;
        p.src = (const uint8_t *)d_src + (src_type == T_MXFP4 ? r * nb * 17 : r * ld * type_size(src_type));
        p.ld = ld;
        p.dst = dst + r * stored * (packed ? 16 : 17);
        p.scales = packed ? scales + r * stored : nullptr;
        p.values = d_values ? (uint16_t *)d_values + r * n_per_row : nullptr;
        p.ncol = n_per_row;
        p.nblk = (uint32_t)(n * stored);
        p.nb = (uint32_t)nb;
        p.row = mx_div((uint32_t)stored);
        switch (src_type) {
            case T_F32: launch_quantize<T_F32>(packed != 0, p, (hipStream_t)stream); break;
            case T_F16: launch_quantize<T_F16>(packed != 0, p, (hipStream_t)stream); break;
            case T_BF16: launch_quantize<T_BF16>(packed != 0, p, (hipStream_t)stream); break;
            default: hipLaunchKernelGGL((k_mx_quantize<T_MXFP4, true>), dim3((unsigned)((p.nblk + MX_U * 64 - 1) / (MX_U * 64))),
                                        dim3(256), 0, (hipStream_t)stream, p);
        }
        if (hipGetLastError() != hipSuccess) return 0;
    }
    return (size_t)(nrow * stored * 17);
}

extern "C" size_t gpuq_mxfp4_matmul_work(int x_type, int64_t nx, int64_t ne0) {
    if (pieces_of(x_type) == 1 || nx <= 0 || nx > MAX_ROWS || !cols_ok(ne0)) return 0;
    return (size_t)(nx * pieces_of(x_type) * round128(ne0) * 2);
}

extern "C" size_t gpuq_mxfp4_matmul_dev(int x_type, const void *d_x, int64_t nx, int64_t ld, const void *d_w,
                                        const void *d_up, int64_t nmat, int64_t ne1, int64_t ne0,
                                        const int32_t *d_offsets, const int32_t *d_rows, int64_t m, int y_type,
                                        void *d_y, void *d_work, void *stream) {
    const bool fp4 = x_type == T_MXFP4;
    if (gq_device() < 0 || !d_x || !d_w || !d_y || (!fp4 && !float_type(x_type)) || !float_type(y_type)) return 0;
    if (nmat <= 0 || nmat > 65534 || ne1 <= 0 || ne1 > MAX_ROWS || !cols_ok(ne0) || nx <= 0 || nx > MAX_ROWS || m <= 0 ||
        m > MAX_ROWS || (nmat > 1 && !d_offsets) || (!d_rows && m > nx))
        return 0;
    if (!aligned16(d_x) || !aligned16(d_w) || !aligned16(d_up) || !aligned16(d_y) || ((uintptr_t)d_offsets & 3) ||
        ((uintptr_t)d_rows & 3))
        return 0;
    if (fp4 ? ld != ne0 : ld < ne0 || ld > ((int64_t)1 << 40) || ld * type_size(x_type) % 16) return 0;
    const int pieces = pieces_of(x_type);
    if (pieces > 1 && (!d_work || !aligned16(d_work))) return 0;
    const hipStream_t st = (hipStream_t)stream;
    const int64_t np = mx_padded(ne0), wcodes = nmat * ne1 * (np / 2);
    MxMulArgs a = {};
    a.nx = nx;
    a.w = (const uint8_t *)d_w;
    a.ws = a.w + wcodes;
    a.u = (const uint8_t *)d_up;
    a.us = d_up ? a.u + wcodes : nullptr;
    a.nmat = nmat;
    a.ne1 = ne1;
    a.np = np;
    a.nk = (int)(round128(ne0) / 128);
    a.offsets = d_offsets;
    a.rows = d_rows;
    a.m = m;
    a.y = d_y;
    a.ytype = y_type;
    a.pieces = pieces;
    if (fp4) {
        a.x = (const uint8_t *)d_x;
        a.xs = a.x + nx * (np / 2);
        a.xrow = np / 2;
    } else if (pieces == 1) {
        a.x = (const uint8_t *)d_x;
        a.xrow = ld * 2;
        a.kx = ne0;
    } else {
        const int64_t kp = round128(ne0);
        const dim3 grid((unsigned)((kp / 8 + 255) / 256), (unsigned)(nx < 65535 ? nx : 65535));
        if (x_type == T_F32)
            hipLaunchKernelGGL((k_mx_split<T_F32, 3>), grid, dim3(256), 0, st, d_x, ld, ne0, kp, nx, (uint16_t *)d_work);
        else
            hipLaunchKernelGGL((k_mx_split<T_F16, 2>), grid, dim3(256), 0, st, d_x, ld, ne0, kp, nx, (uint16_t *)d_work);
        a.x = (const uint8_t *)d_work;
        a.xrow = kp * 2 * pieces;
        a.kx = kp * pieces;
        a.piece = kp * 2;
    }
    const bool glu = d_up != nullptr;
    const int64_t per = m / nmat;                               // rows a group, on average
    if (per <= 16) launch_rows<1>(fp4, glu, a, st);
    else if (per <= 64) launch_rows<4>(fp4, glu, a, st);
    else if (per < 256) {
        if (!launch_tile<2, 2, 4, 4>(fp4, glu, a, st)) return 0;
    } else if (!launch_tile<2, 4, 8, 4>(fp4, glu, a, st)) {
        return 0;
    }
    return hipGetLastError() == hipSuccess ? (size_t)(m * ne1 * type_size(y_type)) : 0;
}

extern "C" int gpuq_route_dev(int type, const void *d_logits, int64_t ntok, int64_t ld, int nexp, int k, int sigmoid,
                              const float *d_bias, int ngroup, int keep, int renorm, float scale, int32_t *d_ids,
                              float *d_weights, void *stream) {
    if (gq_device() < 0 || !float_type(type) || !d_logits || !d_ids || !d_weights || ntok <= 0 || ntok > MAX_ROWS ||
        nexp <= 0 || nexp > RG_MAXE || ld < nexp || k <= 0 || k > 64 || k > nexp)
        return 1;
    if (ngroup <= 0 || ngroup > 64 || nexp % ngroup || keep <= 0 || keep > ngroup) return 1;
    if (((uintptr_t)d_logits & (type_size(type) - 1)) || ((uintptr_t)d_bias & 3) || ((uintptr_t)d_ids & 3) ||
        ((uintptr_t)d_weights & 3))
        return 1;
    const RouteArgs a = {d_logits, ld, d_bias, d_ids, d_weights, ntok, nexp, k, ngroup, keep, scale, sigmoid != 0, renorm != 0};
    const hipStream_t st = (hipStream_t)stream;
    const bool ok = type == T_F32 ? launch_route<T_F32>(a, st) : type == T_F16 ? launch_route<T_F16>(a, st)
                                                                              : launch_route<T_BF16>(a, st);
    return ok ? 0 : 4;
}

extern "C" size_t gpuq_route_group_work(int64_t n, int nexp) {
    if (n <= RG_CHUNK || n > MAX_ROWS || nexp <= 0 || nexp > RG_MAXE) return 0;
    return (size_t)((n + RG_CHUNK - 1) / RG_CHUNK * nexp * 4);
}

extern "C" int gpuq_route_group_dev(const int32_t *d_ids, int64_t ntok, int k, int nexp, int32_t *d_offsets,
                                    int32_t *d_rows, int32_t *d_slots, void *d_work, void *stream) {
    if (gq_device() < 0 || !d_ids || !d_offsets || !d_rows || !d_slots || ntok <= 0 || k <= 0 || nexp <= 0 ||
        nexp > RG_MAXE || ntok > MAX_ROWS || ntok * k > MAX_ROWS)
        return 1;
    if (((uintptr_t)d_ids | (uintptr_t)d_offsets | (uintptr_t)d_rows | (uintptr_t)d_slots | (uintptr_t)d_work) & 3) return 1;
    const int64_t n = ntok * k;
    const int nchunk = (int)((n + RG_CHUNK - 1) / RG_CHUNK);
    if (nchunk > 1 && !d_work) return 1;
    const hipStream_t st = (hipStream_t)stream;
    if (nchunk > 1)
        hipLaunchKernelGGL(k_group_count, dim3(nchunk), dim3(256), 0, st, d_ids, n, nexp, nchunk, (int32_t *)d_work);
    hipLaunchKernelGGL(k_group_place, dim3(nchunk), dim3(256), 0, st, d_ids, n, k, nexp, nchunk,
                       nchunk > 1 ? (const int32_t *)d_work : nullptr, d_offsets, d_rows, d_slots);
    return hipGetLastError() == hipSuccess ? 0 : 4;
}
