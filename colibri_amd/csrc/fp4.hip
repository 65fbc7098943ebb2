// fp4.hip -- MXFP4 on the device: rows quantized to e2m1 codes with e8m0 scales
// per 32 columns and back, and products of such rows with resident MXFP4
// matrices, one matrix or one per expert over sorted rows
// (coli_hip_mxfp4_quantize_dev, coli_hip_fp4_matmul_a4_dev, coli_hip_experts_a4_dev).
//
// y[r, o] = sum_b 2^(ex[r, b] + ew[o, b] - 254) sum_{k in b} cx[r, k] cw[o, k], on
// v_mfma_scale_f32_16x16x128_f8f6f4 with both operands e2m1: the unit reads codes and
// scales as they are stored and no conversion is left. Lane (c, g) of an operand
// holds the 32 codes of row c's block g of the 128 columns, and their scale.
#include "coli_hip_host.h"
#include "coli_rows.h"

#include "coli_backend_abi.h"
#include "coli_hip_ext.h"

#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <vector>

typedef int i32x8 __attribute__((ext_vector_type(8)));

// ---------------------------------------------------------------------------
// quantization
// ---------------------------------------------------------------------------
// Eight elements of a row from column c on, zeros past its end, by loads that stay
// inside the row: moved back where they would pass the end, and shifted to their
// places again (no lane takes a branch of its own; see row4 in coli_device.h).
// FORM 0: n % 8 == 0, 1: any n >= 8, 2: n < 8.
template <typename T, int FORM> __device__ __forceinline__ void row8(const T *xr, int c, int n, float (&v)[8]) {
    if constexpr (FORM == 2) {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = (float)*GPTR(T, xr + min(c + i, n - 1));
    } else {
        const int p = min(c, n - 8);
        el_load<T, 8>(xr + p, v);
        if constexpr (FORM == 1) {
            const int d = c - p;
#pragma unroll
            for (int b = 1; b < 8; b <<= 1)
#pragma unroll
                for (int i = 0; i + b < 8; i++) v[i] = d & b ? v[i + b] : v[i];
        }
    }
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = c + i < n ? v[i] : 0.0f;
}

// The eight codes of a lane and the scale byte of its four lanes' block. a / 6 with
// a = m 2^e lies in (2^(e-3), 2^(e-2)] up to m = 1.5 and in (2^(e-2), 2^(e-1)) beyond,
// so 2^ceil(log2(a / 6)) is read off a's bits: adding just under half of the mantissa's
// range carries into the exponent beyond 1.5. The conversion divides by the scale
// exactly and rounds once, to nearest even: no choice is left to rounding.
__device__ __forceinline__ uint32_t mx_codes(const float (&v)[8], uint32_t &byte) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xF, 0xF, false));
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xF, 0xF, false));
    const uint32_t e = (m + 0x3fffffu) >> 23;
    byte = m == 0 ? 127u : m >= 0x7f800000u ? 255u : max(e, 3u) - 2u;
    const float scale = __uint_as_float(byte << 23);
    uint32_t u = 0;
    u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, v[0], v[1], scale, 0);
    u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, v[2], v[3], scale, 1);
    u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, v[4], v[5], scale, 2);
    u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, v[6], v[7], scale, 3);
    return byte == 255u ? 0u : u;
}

struct QuantArgs {
    const void *x;
    uint8_t *q4, *e8;
    int rows, cols, cp;   // columns, and as written: cp (operand form, a multiple of 256) or cols
    int lpr;              // log2 of the lanes that take a row's octets
};

// Lanes of a row take its octets in turn, four to a block of 32. Native bytes, or
// (OPERAND) rows of cp / 2 and cp / 32 bytes with zeros past the row's end.
template <typename T, int FORM, bool OPERAND> __device__ __forceinline__ void quant_rows(const QuantArgs &a, int blk) {
    const int r = (blk << (8 - a.lpr)) + (threadIdx.x >> a.lpr);
    const int o0 = threadIdx.x & ((1 << a.lpr) - 1);
    if (r >= a.rows) return;
    const T *xr = (const T *)a.x + (size_t)r * a.cols;
    const int end = OPERAND ? a.cp : (a.cols + 31) / 32 * 32;
    const size_t qs = OPERAND ? a.cp / 2 : (a.cols + 1) / 2, es = OPERAND ? a.cp / 32 : (a.cols + 31) / 32;
    for (int c = 8 * o0; c < end; c += 8 << a.lpr) {
        float v[8];
        uint32_t byte;
        row8<T, FORM>(xr, c, a.cols, v);
        const uint32_t u = mx_codes(v, byte);
        uint8_t *q = a.q4 + (size_t)r * qs + c / 2;
        if (OPERAND) {
            *(uint32_t *)q = u;
        } else if (c + 8 <= a.cols) {
            *(u32a1 *)q = u;
        } else {
            for (int i = 0; c + 2 * i < a.cols; i++) q[i] = (uint8_t)(u >> (8 * i));
        }
        if ((threadIdx.x & 3) == 0) a.e8[(size_t)r * es + c / 32] = (uint8_t)byte;
    }
}
template <typename T, int FORM> __global__ __launch_bounds__(256) void coli_mx_quant(QuantArgs a) {
    quant_rows<T, FORM, false>(a, blockIdx.x);
}

// Back: eight columns a lane.
struct DequantArgs {
    const uint8_t *q4, *e8;
    void *y;
    int rows, cols, lpr;
};
template <typename T> __global__ __launch_bounds__(256) void coli_mx_dequant(DequantArgs a) {
    typedef float float2v __attribute__((ext_vector_type(2)));
    const int r = (blockIdx.x << (8 - a.lpr)) + (threadIdx.x >> a.lpr);
    const int o0 = threadIdx.x & ((1 << a.lpr) - 1), qs = (a.cols + 1) / 2;
    if (r >= a.rows) return;
    const uint8_t *q = a.q4 + (size_t)r * qs, *e8 = a.e8 + (size_t)r * ((a.cols + 31) / 32);
    T *y = (T *)a.y + (size_t)r * a.cols;
    for (int c = 8 * o0; c < a.cols; c += 8 << a.lpr) {
        uint32_t u;
        if (qs >= 4) {
            const int p = min(c / 2, qs - 4);
            u = *GPTR(u32a1, q + p) >> (8 * (c / 2 - p));
        } else {
            u = q[0] | q[min(1, qs - 1)] << 8 | q[min(2, qs - 1)] << 16;
        }
        const float s = __uint_as_float((uint32_t)e8[c / 32] << 23);
        const float2v f[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(u, 1.0f, 0), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(u, 1.0f, 1),
                              __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(u, 1.0f, 2), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(u, 1.0f, 3)};
        float o[8];
#pragma unroll
        for (int i = 0; i < 8; i++) o[i] = f[i >> 1][i & 1] * s;
        if (c + 8 <= a.cols) {
            el_store<T, 8>(y + c, o);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (c + i < a.cols) y[c + i] = (T)o[i];
        }
    }
}

// ---------------------------------------------------------------------------
// products
// ---------------------------------------------------------------------------
struct Fp4Mat {
    const uint8_t *w0, *s0, *w1, *s1;   // matrix or gate, up
};
struct Fp4Item {
    int mat, r0, nrows, pad;            // rows [r0, r0 + nrows) of the output times matrix mat
};
struct Fp4Args {
    const Fp4Mat *mats;        // device; null: mat0, and item i is rows [i tile, ..) of S
    Fp4Mat mat0;
    const Fp4Item *items;
    const int *n_items;
    int S, tile;
    int nrt, nq, O;
    int rtb;                   // row-tile blocks of an item
    const uint8_t *xq, *xe;    // operand rows: cp / 2 codes, cp / 32 scales
    int cp;
    const int *src;            // sorted row -> K x row + k (null: the row itself)
    int K, rows;
    const uint8_t *zero;
    float *y;
    float limit;
};

// The items of sorted rows: tiles of `tile` rows of each expert. Offsets are taken
// within 0..N, and no more items are written than there is room for.
struct ItemArgs {
    const int *offsets;
    int E, N, tile, room;
    Fp4Item *items;
    int *n_items;
};
__device__ __forceinline__ void fp4_items(const ItemArgs &a) {
    __shared__ int tmp[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int base = 0;
    for (int e0 = 0; e0 < a.E; e0 += 256) {
        const int e = e0 + tid;
        int r0 = 0, n = 0;
        if (e < a.E) {
            r0 = min(max(a.offsets[e], 0), a.N);
            n = max(0, min(max(a.offsets[e + 1], 0), a.N) - r0);
        }
        const int tiles = (n + a.tile - 1) / a.tile;
        int s = tiles;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int u = __shfl_up(s, o);
            if (lane >= o) s += u;
        }
        if (lane == 63) tmp[wave] = s;
        __syncthreads();
        int at = base + s - tiles;
        for (int w = 0; w < 4; w++) {
            if (w < wave) at += tmp[w];
            base += tmp[w];
        }
        __syncthreads();
        for (int i = 0; i < tiles && at + i < a.room; i++)
            a.items[at + i] = {e, r0 + i * a.tile, min(a.tile, n - i * a.tile), 0};
    }
    if (tid == 0) *a.n_items = min(base, a.room);
}

// The rows' operands and, in the last workgroup (it.items), the items.
template <int FORM> __global__ __launch_bounds__(256) void coli_fp4_prep(QuantArgs a, ItemArgs it, int nblk) {
    if (blockIdx.x == (unsigned)nblk) fp4_items(it);
    else quant_rows<float, FORM, true>(a, blockIdx.x);
}

// 4x4 dword transpose across the four 16-lane rows: the stored tile gives lane (c,
// s) eight codes of each of the four blocks; after it lane (c, g) has block g's 32.
__device__ __forceinline__ i32x8 fp4_tile(u32x4 x) {
    const auto a = __builtin_amdgcn_permlane32_swap(x[0], x[2], false, false);
    const auto b = __builtin_amdgcn_permlane32_swap(x[1], x[3], false, false);
    const auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
    const auto d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
    return (i32x8){(int)c[0], (int)c[1], (int)d[0], (int)d[1], 0, 0, 0, 0};
}

// Rows [0, 16 NM) of an item and R weight tiles (DUAL: the gate and the up tile) a
// workgroup; its W waves take the 128-column steps in turn and add up in LDS, in the
// order of the waves.
template <int NM, int R, bool DUAL, int W> __global__ __launch_bounds__(64 * W) void coli_fp4_few(Fp4Args a) {
    constexpr int U = 2;   // steps whose loads are requested together
    __shared__ floatx4 part[W][R][NM][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, g = lane >> 4;
    const int item = blockIdx.x / a.rtb, rb = blockIdx.x - item * a.rtb;
    Fp4Item it = {0, item * a.tile, 0, 0};
    Fp4Mat mat = a.mat0;
    if (a.mats) {
        if (item >= *a.n_items) return;
        it = a.items[item];
        mat = a.mats[it.mat];
    } else {
        it.nrows = min(a.tile, a.S - it.r0);
    }
    const uint8_t *w[R], *sc[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
        const int rt = min(DUAL ? rb : rb * R + r, a.nrt - 1);
        const size_t t0 = (size_t)rt * a.nq;
        w[r] = uniform_ptr(DUAL && r ? mat.w1 : mat.w0) + t0 * COLI_TILE_BYTES;
        sc[r] = uniform_ptr(DUAL && r ? mat.s1 : mat.s0) + t0 * 64;
    }
    const uint8_t *xq[NM], *xe[NM];
#pragma unroll
    for (int m = 0; m < NM; m++) {
        int x = it.r0 + min(16 * m + c, it.nrows - 1);
        if (a.src) {
            x = a.src[x];
            x = x < 0 ? -1 : x / a.K;
        }
        const bool in = (unsigned)x < (unsigned)a.rows;
        xq[m] = (in ? a.xq + (size_t)x * (a.cp / 2) : a.zero) + 16 * g;
        xe[m] = in ? a.xe + (size_t)x * (a.cp / 32) : a.zero;
    }
    floatx4 acc[R][NM];
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
        for (int m = 0; m < NM; m++) acc[r][m] = (floatx4){0.f, 0.f, 0.f, 0.f};
    for (int q0 = wave; q0 < a.nq; q0 += W * U) {
        u32x4 wv[U][R], xv[U][NM];
        uint32_t ws[U][R], xs[U][NM];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int q = min(q0 + W * u, a.nq - 1);
#pragma unroll
            for (int r = 0; r < R; r++) {
                wv[u][r] = *GPTR(u32x4, w[r] + (size_t)q * COLI_TILE_BYTES + lane * 16);
                ws[u][r] = *GPTR(uint32_t, sc[r] + (size_t)q * 64 + c * 4);
            }
#pragma unroll
            for (int m = 0; m < NM; m++) {
                xv[u][m] = *GPTR(u32x4, xq[m] + (size_t)q * 64);
                xs[u][m] = *GPTR(uint32_t, xe[m] + (size_t)q * 4);
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (q0 + W * u >= a.nq) break;
            i32x8 wo[R];
#pragma unroll
            for (int r = 0; r < R; r++) wo[r] = fp4_tile(wv[u][r]);
#pragma unroll
            for (int m = 0; m < NM; m++) {
                const i32x8 xo = {(int)xv[u][m][0], (int)xv[u][m][1], (int)xv[u][m][2], (int)xv[u][m][3], 0, 0, 0, 0};
#pragma unroll
                for (int r = 0; r < R; r++)
                    acc[r][m] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wo[r], xo, acc[r][m], 4, 4, 0,
                                                                                (int)(ws[u][r] >> (8 * g)), 0,
                                                                                (int)(xs[u][m] >> (8 * g)));
            }
        }
    }
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
        for (int m = 0; m < NM; m++) part[wave][r][m][lane] = acc[r][m];
    __syncthreads();
    // lane (c, g): row 16 m + c, outputs 16 rt + 4 g ..
    constexpr int RT = DUAL ? 1 : R;
    for (int k = wave; k < RT * NM; k += W) {
        const int r = k / NM, m = k - r * NM;
        floatx4 v = part[0][r][m][lane], u = {};
#pragma unroll
        for (int q = 1; q < W; q++) v += part[q][r][m][lane];
        if constexpr (DUAL) {
            u = part[0][1][m][lane];
#pragma unroll
            for (int q = 1; q < W; q++) u += part[q][1][m][lane];
        }
        const int row = 16 * m + c, o = 16 * (DUAL ? rb : rb * R + r) + 4 * g;
        if (row >= it.nrows) continue;
        float *y = a.y + (size_t)(it.r0 + row) * a.O + o;
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (o + i < a.O) y[i] = DUAL ? swiglu_out(v[i], u[i], a.limit) : v[i];
    }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
static int lanes_log2(int cols) {   // lanes of a row: its octets, 4 to 256
    int l = 2;
    while (l < 8 && (8 << l) < cols) l++;
    return l;
}

static size_t mx_q4_bytes(int rows, int cols) { return (size_t)rows * ((cols + 1) / 2); }
static size_t mx_e8_bytes(int rows, int cols) { return (size_t)rows * ((cols + 31) / 32); }

template <typename T> static void quant_launch(const QuantArgs &a, hipStream_t st) {
    const dim3 g((unsigned)((a.rows + (256 >> a.lpr) - 1) / (256 >> a.lpr)));
    if (a.cols < 8) hipLaunchKernelGGL((coli_mx_quant<T, 2>), g, dim3(256), 0, st, a);
    else if (a.cols % 8) hipLaunchKernelGGL((coli_mx_quant<T, 1>), g, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((coli_mx_quant<T, 0>), g, dim3(256), 0, st, a);
}
static int quantize(DevCtx *ctx, const void *x, int dtype, int rows, int cols, uint8_t *q4, uint8_t *e8) {
    const QuantArgs a = {x, q4, e8, rows, cols, cols, lanes_log2(cols)};
    if (dtype == 0) quant_launch<float>(a, ctx->stream);
    else if (dtype == 1) quant_launch<_Float16>(a, ctx->stream);
    else quant_launch<__bf16>(a, ctx->stream);
    return hip_check(hipGetLastError(), "mxfp4 quantize");
}

#define COLI_MX_MAX 16777215   // rows and columns of a call (a grid of 256-thread workgroups by row)
static bool mx_shape_ok(int dtype, int rows, int cols) {
    return dtype >= 0 && dtype <= 2 && rows >= 0 && rows <= COLI_MX_MAX && cols >= 1 && cols <= COLI_MX_MAX;
}

extern "C" int coli_hip_mxfp4_quantize_dev(int device, const void *x, int dtype, int rows, int cols, unsigned char *q4,
                                           unsigned char *e8) {
    if (fault_injected()) return 0;
    if (!mx_shape_ok(dtype, rows, cols) || (rows && (!x || !q4 || !e8))) return 0;
    const size_t qb = mx_q4_bytes(rows, cols), eb = mx_e8_bytes(rows, cols);
    if (!outputs_apart({{q4, qb}, {e8, eb}, {x, (size_t)rows * cols * (dtype ? 2 : 4)}}, 2)) return 0;
    DevCtx *ctx = ctx_of(device);
    if (!bind_ctx(ctx)) return 0;
    if (!rows) return 1;
    forget_emitted(ctx, q4, qb);
    forget_emitted(ctx, e8, eb);
    return quantize(ctx, x, dtype, rows, cols, q4, e8);
}

extern "C" int coli_hip_mxfp4_dequantize_dev(int device, const unsigned char *q4, const unsigned char *e8, int rows,
                                             int cols, void *y, int dtype) {
    if (fault_injected()) return 0;
    if (!mx_shape_ok(dtype, rows, cols) || (rows && (!y || !q4 || !e8))) return 0;
    const size_t yb = (size_t)rows * cols * (dtype ? 2 : 4);
    if (!outputs_apart({{y, yb}, {q4, mx_q4_bytes(rows, cols)}, {e8, mx_e8_bytes(rows, cols)}}, 1)) return 0;
    DevCtx *ctx = ctx_of(device);
    if (!bind_ctx(ctx)) return 0;
    if (!rows) return 1;
    forget_emitted(ctx, y, yb);
    const DequantArgs a = {q4, e8, y, rows, cols, lanes_log2(cols)};
    const dim3 g((unsigned)((rows + (256 >> a.lpr) - 1) / (256 >> a.lpr)));
    if (dtype == 0) hipLaunchKernelGGL(coli_mx_dequant<float>, g, dim3(256), 0, ctx->stream, a);
    else if (dtype == 1) hipLaunchKernelGGL(coli_mx_dequant<_Float16>, g, dim3(256), 0, ctx->stream, a);
    else hipLaunchKernelGGL(coli_mx_dequant<__bf16>, g, dim3(256), 0, ctx->stream, a);
    return hip_check(hipGetLastError(), "mxfp4 dequantize");
}

// Native bytes on the device, then the upload from there (its scales come from the
// host, where the tensor's scale range is looked at too).
extern "C" int coli_hip_tensor_quantize_mxfp4(ColiCudaTensor **tensor, const void *weights_dev, int dtype, int I, int O,
                                              int device) {
    if (!tensor || *tensor || !weights_dev || !mx_shape_ok(dtype, O, I) || O < 1) return 0;
    DevCtx *ctx = ctx_of(device);
    if (!bind_ctx(ctx)) return 0;
    const size_t qb = (mx_q4_bytes(O, I) + 255) & ~(size_t)255, eb = mx_e8_bytes(O, I);
    if (!reserve(ctx, &ctx->stage_w, qb + eb, 0)) return 0;
    uint8_t *q4 = (uint8_t *)ctx->stage_w.p, *e8 = q4 + qb;
    std::vector<uint8_t> host(eb);
    if (!quantize(ctx, weights_dev, dtype, O, I, q4, e8) ||
        !hip_check(hipStreamSynchronize(ctx->stream), "tensor quantize") ||
        !hip_check(hipMemcpy(host.data(), e8, eb, hipMemcpyDeviceToHost), "scale download"))
        return 0;
    return upload_impl(tensor, q4, nullptr, host.data(), 7, I, O, device, 32, 1);
}

// Rows of x as operands of the products (and the items of sorted rows beside it).
#define COLI_FP4_TILE 64
static int fp4_prep(DevCtx *ctx, const float *x, int rows, int I, const ItemArgs *it, Fp4Args *a) {
    const int cp = (I + 255) / 256 * 256;
    const size_t qb = ((size_t)rows * (cp / 2) + 255) & ~(size_t)255, eb = (size_t)rows * (cp / 32);
    if (!reserve_kept(ctx, &ctx->fp4_x, qb + eb, 0)) return 0;
    uint8_t *p = (uint8_t *)ctx->fp4_x.p;
    const QuantArgs q = {x, p, p + qb, rows, I, cp, lanes_log2(cp)};
    const int nblk = (rows + (256 >> q.lpr) - 1) / (256 >> q.lpr);
    const dim3 g(nblk + (it ? 1 : 0));
    const ItemArgs none = {};
    if (I < 8) hipLaunchKernelGGL(coli_fp4_prep<2>, g, dim3(256), 0, ctx->stream, q, it ? *it : none, nblk);
    else if (I % 8) hipLaunchKernelGGL(coli_fp4_prep<1>, g, dim3(256), 0, ctx->stream, q, it ? *it : none, nblk);
    else hipLaunchKernelGGL(coli_fp4_prep<0>, g, dim3(256), 0, ctx->stream, q, it ? *it : none, nblk);
    if (!hip_check(hipGetLastError(), "fp4 operands")) return 0;
    a->xq = p;
    a->xe = p + qb;
    a->cp = cp;
    a->rows = rows;
    a->zero = (const uint8_t *)ctx->zeros.p;
    return 1;
}

// The launch over n_items items of tiles of a.tile rows.
static int fp4_run(DevCtx *ctx, Fp4Args &a, int n_items, bool dual) {
    const int W = 8;
    a.rtb = dual ? a.nrt : (a.nrt + 1) / 2;
    if ((int64_t)n_items * a.rtb * 64 * W >= ((int64_t)1 << 32)) return 0;
    const dim3 g((unsigned)n_items * a.rtb);
    if (dual) hipLaunchKernelGGL((coli_fp4_few<4, 2, true, W>), g, dim3(64 * W), 0, ctx->stream, a);
    else hipLaunchKernelGGL((coli_fp4_few<4, 2, false, W>), g, dim3(64 * W), 0, ctx->stream, a);
    return hip_check(hipGetLastError(), "fp4 product");
}

#define COLI_FP4_MAX_I (COLI_ZERO_BYTES * 2)   // an operand row is no longer than the zeros

int matmul_a4_dev(DevCtx *ctx, ColiCudaTensor *t, float *y_dev, const float *x_dev, int S) {
    Fp4Args a = {};
    if (t->I > (int)COLI_FP4_MAX_I) return 0;
    forget_emitted(ctx, y_dev, (size_t)S * t->O * 4);
    if (!fp4_prep(ctx, x_dev, S, t->I, nullptr, &a)) return 0;
    a.mat0 = {t->w, (const uint8_t *)t->sc, nullptr, nullptr};
    a.S = S;
    a.tile = COLI_FP4_TILE;
    a.nrt = t->nrt;
    a.nq = t->nq;
    a.O = t->O;
    a.K = 1;
    a.y = y_dev;
    return fp4_run(ctx, a, (S + a.tile - 1) / a.tile, false);
}

extern "C" int coli_hip_fp4_matmul_a4_dev(ColiCudaTensor *t, float *y_dev, const float *x_dev, int S) {
    if (fault_injected()) return 0;
    if (!t || t->kind != COLI_KIND_FP4 || !y_dev || !x_dev || S < 1 || S > COLI_MX_MAX ||
        ranges_overlap(y_dev, (size_t)S * t->O * 4, x_dev, (size_t)S * t->I * 4))
        return 0;
    DevCtx *ctx = ctx_of(t->device);
    if (!bind_ctx(ctx)) return 0;
    return matmul_a4_dev(ctx, t, y_dev, x_dev, S);
}

struct ColiHipExperts {
    int device, E, I, O, nrt, nq, dual;
    float limit;
    Fp4Mat *mats;   // device
};

extern "C" void coli_hip_experts_free(ColiHipExperts *x) {
    if (!x) return;
    DevCtx *ctx = ctx_of(x->device);
    if (ctx) {
        bind_ctx(ctx);
        (void)hipStreamSynchronize(ctx->stream);
    }
    if (x->mats) (void)hipFree(x->mats);
    std::free(x);
}

extern "C" int coli_hip_experts_create(ColiHipExperts **out, int device, int E, ColiCudaTensor *const *gates,
                                       ColiCudaTensor *const *ups, float swiglu_limit) {
    if (!out || E < 1 || E > 1024 || !gates) return 0;
    DevCtx *ctx = ctx_of(device);
    if (!bind_ctx(ctx)) return 0;
    std::vector<Fp4Mat> m(E);
    for (int e = 0; e < E; e++)
        for (int k = 0; k < (ups ? 2 : 1); k++) {
            const ColiCudaTensor *t = k ? ups[e] : gates[e];
            if (!t || t->kind != COLI_KIND_FP4 || t->device != device || t->I != gates[0]->I || t->O != gates[0]->O ||
                t->I > (int)COLI_FP4_MAX_I) {
                std::fprintf(stderr, "[HIP] experts: expert %d is not an MXFP4 tensor of this device and shape\n", e);
                return 0;
            }
            (k ? m[e].w1 : m[e].w0) = t->w;
            (k ? m[e].s1 : m[e].s0) = (const uint8_t *)t->sc;
        }
    ColiHipExperts *x = (ColiHipExperts *)std::calloc(1, sizeof(ColiHipExperts));
    if (!x) return 0;
    x->device = device;
    x->E = E;
    x->I = gates[0]->I;
    x->O = gates[0]->O;
    x->nrt = gates[0]->nrt;
    x->nq = gates[0]->nq;
    x->dual = ups != nullptr;
    x->limit = swiglu_limit;
    if (!hip_check(hipMalloc((void **)&x->mats, E * sizeof(Fp4Mat)), "expert set") ||
        !hip_check(hipMemcpy(x->mats, m.data(), E * sizeof(Fp4Mat), hipMemcpyHostToDevice), "expert set")) {
        coli_hip_experts_free(x);
        return 0;
    }
    *out = x;
    return 1;
}

extern "C" int coli_hip_experts_a4_dev(ColiHipExperts *x, float *y, const float *xr, int rows, const int *src, int K,
                                       const int *offsets, int N) {
    if (fault_injected()) return 0;
    if (!x || rows < 0 || rows > COLI_MX_MAX || N < 0 || N > (1 << 30) || K < 1 || (N && (!y || !offsets || !xr || !rows)))
        return 0;
    const size_t yb = (size_t)N * x->O * 4;
    if (!outputs_apart({{y, yb}, {xr, (size_t)rows * x->I * 4}, {src, (size_t)N * 4}, {offsets, (size_t)(x->E + 1) * 4}}, 1))
        return 0;
    DevCtx *ctx = ctx_of(x->device);
    if (!bind_ctx(ctx)) return 0;
    if (!N) return 1;
    forget_emitted(ctx, y, yb);
    ItemArgs it = {};
    it.offsets = offsets;
    it.E = x->E;
    it.N = N;
    it.tile = COLI_FP4_TILE;
    it.room = (int)std::min<int64_t>(N, N / it.tile + x->E);
    if (!reserve_kept(ctx, &ctx->fp4_items, 256 + (size_t)it.room * sizeof(Fp4Item), 0)) return 0;
    it.n_items = (int *)ctx->fp4_items.p;
    it.items = (Fp4Item *)((uint8_t *)ctx->fp4_items.p + 256);
    Fp4Args a = {};
    if (!fp4_prep(ctx, xr, rows, x->I, &it, &a)) return 0;
    a.mats = x->mats;
    a.items = it.items;
    a.n_items = it.n_items;
    a.tile = it.tile;
    a.nrt = x->nrt;
    a.nq = x->nq;
    a.O = x->O;
    a.src = src;
    a.K = K;
    a.y = y;
    a.limit = x->limit;
    return fp4_run(ctx, a, it.room, x->dual != 0);
}
