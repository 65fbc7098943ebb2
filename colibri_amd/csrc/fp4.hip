// fp4.hip -- MXFP4 on the device: rows quantized to e2m1 codes with e8m0 scales
// per 32 columns and back, and products of such rows with resident MXFP4
// matrices, one matrix or one per expert over sorted rows
// (coli_hip_mxfp4_quantize_dev, coli_hip_fp4_matmul_a4_dev, coli_hip_experts_a4_dev).
//
// y[r, o] = sum_b 2^(ex[r, b] + ew[o, b] - 254) sum_{k in b} cx[r, k] cw[o, k], on
// v_mfma_scale_f32_{16x16x128,32x32x64}_f8f6f4 with both operands e2m1: the unit reads codes
// and scales as they are stored and no conversion is left. A lane of an operand holds the
// 32 codes of one block of a row, and their scale. Products are exact and sums f32.
//
// Two kernels. coli_fp4_few streams the weights (a token through 4096 x 14336 7.6 us, 4.1
// TB/s, what a plain read of so small a matrix reaches; the pairs that 16 rows select of
// 256, 0.88 GB, in 130 us, 6.7 TB/s). coli_fp4_many is bound by the matrix units' power: 2048 x
// 14336 x 4096 in 66 us, 3.6 PFLOP/s, 47 us with its loads, LDS reads and turns left out
// (the card lowers its clock to 1.6 GHz under MFMAs of random codes); of the rest 13 us go
// with the loads, whatever they hit: weights five steps ahead instead of two, weights that a
// second group of waves shares, and hot lines alone change nothing.
// coli_fp4_prep quantizes the rows ahead of them, at the rate of a copy.
#include "coli_hip_host.h"
#include "coli_rows.h"

#include "coli_backend_abi.h"
#include "coli_hip_ext.h"

#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <type_traits>
#include <vector>

typedef int i32x8 __attribute__((ext_vector_type(8)));

// ---------------------------------------------------------------------------
// quantization
// ---------------------------------------------------------------------------
// V elements of a row from column c on, zeros past its end, by loads that stay inside
// the row: moved back where they would pass the end, and shifted to their places again
// (no lane takes a branch of its own; see row4 in coli_device.h).
// FORM 0: n % V == 0, 1: any n >= V, 2: n < V.
template <typename T, int FORM, int V, bool NT = false> __device__ __forceinline__ void row_vec(const T *xr, int c, int n, float (&v)[V]) {
    if constexpr (FORM == 2) {
#pragma unroll
        for (int i = 0; i < V; i++) v[i] = (float)*GPTR(T, xr + min(c + i, n - 1));
    } else {
        const int p = min(c, n - V);
        el_load<T, V, NT>(xr + p, v);
        if constexpr (FORM == 1) {
            const int d = c - p;
#pragma unroll
            for (int b = 1; b < V; b <<= 1)
#pragma unroll
                for (int i = 0; i + b < V; i++) v[i] = d & b ? v[i + b] : v[i];
        }
    }
#pragma unroll
    for (int i = 0; i < V; i++) v[i] = c + i < n ? v[i] : 0.0f;
}

// The V codes of a lane and the scale byte of its 32 / V lanes' block. a / 6 with
// a = m 2^e lies in (2^(e-3), 2^(e-2)] up to m = 1.5 and in (2^(e-2), 2^(e-1)) beyond,
// so 2^ceil(log2(a / 6)) is read off a's bits: adding just under half of the mantissa's
// range carries into the exponent beyond 1.5. The conversion divides by the scale
// exactly and rounds once, to nearest even: no choice is left to rounding.
template <int V> __device__ __forceinline__ uint32_t mx_codes(const float (&v)[V], uint32_t &byte) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < V; i++) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xF, 0xF, false));
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xF, 0xF, false));
    if constexpr (V == 4) m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x141, 0xF, 0xF, false));
    const uint32_t e = (m + 0x3fffffu) >> 23;
    byte = m == 0 ? 127u : m >= 0x7f800000u ? 255u : max(e, 3u) - 2u;
    const float scale = __uint_as_float(byte << 23);
    uint32_t u = 0;
    u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, v[0], v[1], scale, 0);
    u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, v[2], v[3], scale, 1);
    if constexpr (V == 8) {
        u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, v[4], v[5], scale, 2);
        u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, v[6], v[7], scale, 3);
    }
    return byte == 255u ? 0u : u;
}

struct QuantArgs {
    const void *x;
    uint8_t *q4, *e8;
    int rows, cols, cp;   // columns, and as written: cp (operand form, a multiple of 256) or cols
    int lpr, chunks;      // log2 of the lanes that a row has, workgroups that share a row
};

// A lane takes 16 bytes of a row at a time, so that neighbours load whole cache lines
// (8000 f32 rows of 14336 and back 227 us with 8 elements, 217 with 4).
// Native bytes, or (OPERAND) rows of cp / 2 and cp / 32 bytes with zeros past the row's
// end, and behind the last row one of zeros.
template <typename T, int FORM, bool OPERAND> __device__ __forceinline__ void quant_rows(const QuantArgs &a, int blk) {
    constexpr int V = 16 / sizeof(T);
    const int grp = blk / a.chunks, r = (grp << (8 - a.lpr)) + (threadIdx.x >> a.lpr);
    const int o0 = ((blk - grp * a.chunks) << a.lpr) + (threadIdx.x & ((1 << a.lpr) - 1));
    if (r >= a.rows + (OPERAND ? 1 : 0)) return;
    const bool zero = OPERAND && r == a.rows;
    const T *xr = (const T *)a.x + (size_t)(zero ? 0 : r) * a.cols;
    const int end = OPERAND ? a.cp : (a.cols + 31) / 32 * 32;
    const size_t qs = OPERAND ? a.cp / 2 : (a.cols + 1) / 2, es = OPERAND ? a.cp / 32 : (a.cols + 31) / 32;
    for (int c = V * o0; c < end; c += (V << a.lpr) * a.chunks) {
        float v[V];
        uint32_t byte;
        row_vec<T, FORM, V, true>(xr, c, a.cols, v);   // (read once, past the caches: 8000 f32 rows of 14336 and back 264 -> 229 us)
        if constexpr (OPERAND) {
#pragma unroll
            for (int i = 0; i < V; i++) v[i] = zero ? 0.0f : v[i];
        }
        const uint32_t u = mx_codes<V>(v, byte);
        uint8_t *q = a.q4 + (size_t)r * qs + c / 2;
        if (OPERAND || c + V <= a.cols) {
            if constexpr (V == 8) *(u32a1 *)q = u;
            else *(u16a1 *)q = (uint16_t)u;
        } else {
            for (int i = 0; c + 2 * i < a.cols; i++) q[i] = (uint8_t)(u >> (8 * i));
        }
        if ((threadIdx.x & (32 / V - 1)) == 0) a.e8[(size_t)r * es + c / 32] = (uint8_t)byte;
    }
}
template <typename T, int FORM> __global__ __launch_bounds__(256) void coli_mx_quant(QuantArgs a) {
    quant_rows<T, FORM, false>(a, blockIdx.x);
}

// Back: eight columns a lane.
struct DequantArgs {
    const uint8_t *q4, *e8;
    void *y;
    int rows, cols, lpr, chunks;
};
template <typename T, bool NT> __global__ __launch_bounds__(256) void coli_mx_dequant(DequantArgs a) {
    typedef float float2v __attribute__((ext_vector_type(2)));
    const int grp = blockIdx.x / a.chunks, r = (grp << (8 - a.lpr)) + (threadIdx.x >> a.lpr), qs = (a.cols + 1) / 2;
    const int o0 = ((blockIdx.x - grp * a.chunks) << a.lpr) + (threadIdx.x & ((1 << a.lpr) - 1));
    if (r >= a.rows) return;
    const uint8_t *q = a.q4 + (size_t)r * qs, *e8 = a.e8 + (size_t)r * ((a.cols + 31) / 32);
    T *y = (T *)a.y + (size_t)r * a.cols;
    for (int c = 8 * o0; c < a.cols; c += (8 << a.lpr) * a.chunks) {
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
            el_store<T, 8, NT>(y + c, o);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (c + i < a.cols) y[c + i] = el_of<T>(o[i]);
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
    Fp4Mat mat;
    int r0, nrows;                      // rows [r0, r0 + nrows) of the output times mat
};
struct Fp4Args {
    const Fp4Item *items;      // device; null: mat0, and item i is rows [i tile, ..) of S
    const int *n_items;
    Fp4Mat mat0;
    int S, tile;
    int nrt, nq, O;
    int rtb;                   // row-tile blocks of an item
    const uint8_t *xq, *xe;    // operand rows: cp / 2 codes, cp / 32 scales; row `rows` is zeros
    const float *x;            // or the rows themselves, of width I (the kernel quantizes them)
    int cp, I;
    int splits, sps;           // K splits (many rows of one matrix): 256-column stages of each
    float *part;               // their sums [split][S][O]
    const int *src;            // sorted row -> K x row + k (null: the row itself)
    int K, rows;
    float *y;
    int group;                 // items of a group (coli_fp4_many)
    float limit;
    int item0;                 // the launch's first item
};

// The items of sorted rows: tiles of `tile` rows of each expert. Offsets are taken
// within 0..N, and no more items are written than there is room for.
struct ItemArgs {
    const int *offsets;
    int E, N, tile, room;
    const Fp4Mat *mats;
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
            a.items[at + i] = {a.mats[e], r0 + i * a.tile, min(a.tile, n - i * a.tile)};
    }
    if (tid == 0) *a.n_items = min(base, a.room);
}

// The rows' operands and, in the first workgroup (it.items), the items: placed last it
// would end after the others.
template <int FORM> __global__ __launch_bounds__(256) void coli_fp4_prep(QuantArgs a, ItemArgs it) {
    const int first = it.items ? 1 : 0;
    if ((int)blockIdx.x < first) fp4_items(it);
    else quant_rows<float, FORM, true>(a, blockIdx.x - first);
}

// swiglu_out on the hardware's exp2 and reciprocal (a step of each, beside products whose
// sums carry more): exp(-g) = 2^h (1 + l ln 2) with h + l = -g log2(e) in two parts, right
// to 5 x 2^-24 for gates from COLI_FP4_LOW up. A third of the instructions of expf and the
// division, which a short product shows (16384 rows through 8 pairs of 2048 x 1024 68.0 -> 61.8
// us, through 64 pairs 98.0 -> 89.3).
// LOW: gates below it too, whose sigmoid is exp(g) in f32 and (from -87.34 down) below the
// normal range, where the reciprocal is 0: 2^n 2^f in two steps, the up scaled by 2^-64
// meanwhile, so that nothing is lost that the result can hold. Where 2^-64 takes a small up out of
// range the result is below it too: |g| exp(g) < 2^-119. Gates below -300 count as -300: the
// result is 0 for every finite up.
#define COLI_FP4_LOW -87.0f
template <bool LOW> __device__ __forceinline__ float fp4_swiglu(float g, float u, float limit) {
    if (limit > 0.0f) {   // (compared, not fminf: a NaN stays one)
        g = g > limit ? limit : g;
        u = u > limit ? limit : u < -limit ? -limit : u;
    }
    const float c = fminf(fmaxf(g, -128.0f), 128.0f);   // beyond, the sigmoid is 1 in f32, or 0 (LOW has it)
    const float h = c * -1.44269504f, l = fmaf(c, -1.44269504f, -h) + c * -1.92596303e-8f;
    const float e = __builtin_amdgcn_exp2f(h) * fmaf(l, 0.693147181f, 1.0f);
    const float y = g * __builtin_amdgcn_rcpf(1.0f + e) * u;
    if constexpr (!LOW) return y;
    const float d = fmaxf(g, -300.0f), n = rintf(d * 1.44269504f), f = fmaf(d, 1.44269504f, -n) + d * 1.92596303e-8f;
    const float z = __builtin_ldexpf(d * __builtin_amdgcn_exp2f(f) * (u * 0x1p-64f), (int)n + 64);
    return g < COLI_FP4_LOW && g > -INFINITY ? z : y;
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

// Few rows: [0, 16 NM) of an item times R weight tiles (DUAL: the gate and the up tile) a
// workgroup; its eight waves take the 128-column steps in turn, U of them requested
// together, and add up in LDS, in the order of the waves. The weights' stream is the
// bound.
// FORM (of row_vec; -1: operands in memory): the workgroup quantizes the rows itself, into
// LDS, behind its first weights' loads. That saves the operands' launch where the rows
// are so few that 512 threads have done them before the weights are there.
#define COLI_FP4_WAVES 8
template <int NM, int R, bool DUAL, int FORM> __global__ __launch_bounds__(64 * COLI_FP4_WAVES) void coli_fp4_few(Fp4Args a) {
    constexpr int W = COLI_FP4_WAVES, U = NM == 1 ? 4 : 2;
    constexpr bool OWN = FORM >= 0;
    __shared__ floatx4 part[W][R][NM][64];
    extern __shared__ __attribute__((aligned(16))) uint8_t xl[];   // (OWN) codes, then scales
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, g = lane >> 4;
    const int in = blockIdx.x / a.rtb, rb = blockIdx.x - in * a.rtb, item = a.item0 + in;
    Fp4Item it = {a.mat0, item * a.tile, min(a.tile, a.S - item * a.tile)};
    if (a.items) {
        if (item >= *a.n_items) return;
        it = a.items[item];
    }
    const Fp4Mat mat = it.mat;
    const uint8_t *w[R], *sc[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
        const int rt = min(DUAL ? rb : rb * R + r, a.nrt - 1);
        const size_t t0 = (size_t)rt * a.nq;
        w[r] = uniform_ptr(DUAL && r ? mat.w1 : mat.w0) + t0 * COLI_TILE_BYTES;
        sc[r] = uniform_ptr(DUAL && r ? mat.s1 : mat.s0) + t0 * 64;
    }
    const int qs = a.cp / 2, es = a.cp / 32;
    const uint8_t *xq[NM], *xe[NM];
#pragma unroll
    for (int m = 0; m < NM; m++) {
        int x = it.r0 + min(16 * m + c, it.nrows - 1);
        if (a.src) {
            x = a.src[x];
            x = x < 0 ? -1 : x / a.K;
        }
        if ((unsigned)x >= (unsigned)a.rows) x = a.rows;
        xq[m] = OWN ? xl + x * qs + 16 * g : a.xq + (size_t)x * qs + 16 * g;
        xe[m] = OWN ? xl + a.rows * qs + x * es : a.xe + (size_t)x * es;
    }
    floatx4 acc[R][NM];
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
        for (int m = 0; m < NM; m++) acc[r][m] = (floatx4){0.f, 0.f, 0.f, 0.f};
    u32x4 wv[U][R], xv[U][NM];
    uint32_t ws[U][R], xs[U][NM];
    auto load_w = [&](int q0) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int q = min(q0 + W * u, a.nq - 1);
#pragma unroll
            for (int r = 0; r < R; r++) {
                wv[u][r] = __builtin_nontemporal_load(GPTR(u32x4, w[r] + (size_t)q * COLI_TILE_BYTES + lane * 16));
                ws[u][r] = *GPTR(uint32_t, sc[r] + (size_t)q * 64 + c * 4);
            }
        }
    };
    auto compute = [&](int q0) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int q = min(q0 + W * u, a.nq - 1);
#pragma unroll
            for (int m = 0; m < NM; m++) {
                xv[u][m] = OWN ? *(const u32x4 *)(xq[m] + q * 64) : (u32x4)*GPTR(u32x4, xq[m] + (size_t)q * 64);
                xs[u][m] = OWN ? *(const uint32_t *)(xe[m] + q * 4) : *GPTR(uint32_t, xe[m] + (size_t)q * 4);
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
    };
    load_w(wave);
    if constexpr (OWN) {
        const int opr = a.cp / 8;   // octets of a row
        for (int o = threadIdx.x; o < a.rows * opr; o += 64 * W) {
            const int r = o / opr, k = 8 * (o - r * opr);
            float v[8];
            uint32_t byte;
            row_vec<float, FORM, 8>(a.x + (size_t)r * a.I, k, a.I, v);
            const uint32_t u = mx_codes<8>(v, byte);
            *(uint32_t *)(xl + r * qs + k / 2) = u;
            if ((threadIdx.x & 3) == 0) xl[a.rows * qs + r * es + k / 32] = (uint8_t)byte;
        }
        __syncthreads();
    }
    compute(wave);
    for (int q0 = wave + W * U; q0 < a.nq; q0 += W * U) {
        load_w(q0);
        compute(q0);
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
        if constexpr (DUAL) {
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = fp4_swiglu<true>(v[i], u[i], a.limit);
        }
        if (o + 4 <= a.O) {
            *(f4u *)y = v;
        } else {
#pragma unroll
            for (int i = 0; i < 3; i++)
                if (o + i < a.O) y[i] = v[i];
        }
    }
}

// Many rows: 128 rows x 16 weight tiles (DUAL: 8 gate and 8 up tiles) a workgroup of
// four waves, each all the rows and four tiles as two operands of 32 rows on
// v_mfma_scale_f32_32x32x64_f8f6f4: 16 MFMAs a wave and step of 128 columns, on 4 KiB of
// weights, which go straight to registers, and 8 KiB of rows from LDS. (One wave issues
// the 16x16x128 form every 29 cycles, four waves a SIMD every 18; the 32x32x64 form,
// twice the work, runs at its 32 from one wave: 8.9 PFLOP/s of zeros on the card, 6.8 of
// random codes, where 16x16x128 reaches 6.8 and 5.4.)
// The rows come by LDS DMA two steps at a time (128 bytes of a row: a whole cache line)
// into a ring of three stages; 16-byte pieces are stored XORed with a key of the row,
// so that the rows of an operand read hit different banks.
// Loads retire in order: a wave that has used the weights of a step has all the DMAs
// requested before them, so the ring costs one barrier a stage and no wait of its own.
// (The DMAs are buffer loads: the compiler takes global_load_lds for a flat access and
// waits for every load in flight at the next use of any.)
// Weights rotate through three sets of registers, one in use, one being turned, one
// being loaded, without a copy: six steps (three stages) are written out.
#define COLI_FP4_MANY 128
struct FmGeom {
    static constexpr int kRows = COLI_FP4_MANY * 128;   // a stage's codes: 256 columns
    static constexpr int kStage = kRows + COLI_FP4_MANY * 8;
    static constexpr int kPD = 3;
};
typedef __attribute__((address_space(3))) uint8_t lds_u8;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t fp4_rsrc(const void *p, uint32_t n) {
    return __builtin_amdgcn_make_buffer_rsrc((void *)p, 0, n, 0x00020000);
}
__device__ __forceinline__ i32x8 fp4_op(u32x4 v) { return (i32x8){(int)v[0], (int)v[1], (int)v[2], (int)v[3], 0, 0, 0, 0}; }
// The results of a wave's operands. Lane (n, g), register i: row 8 (i / 4) + 4 g + i % 4 of the
// block, output n of the operand's 32: a store fills whole cache lines of two rows.
template <int NB, bool DUAL, bool NT, bool LOW> __device__ __forceinline__ void fp4_store(
    const Fp4Args &a, const Fp4Item &it, const int (&rt)[2], int split, int n, int g, const floatx16 (&acc)[2][NB]) {
#pragma unroll
    for (int r = 0; r < (DUAL ? 1 : 2); r++) {
        const int o = 16 * rt[r] + n;
        float *y = (a.splits > 1 ? a.part + (size_t)split * a.S * a.O : a.y) + (size_t)it.r0 * a.O + o;
        if (o >= a.O) continue;
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int row = 32 * b + 8 * (i >> 2) + 4 * g + (i & 3);
                float v = acc[r][b][i];
                if constexpr (DUAL) v = fp4_swiglu<LOW>(v, acc[1][b][i], a.limit);
                if (row >= it.nrows) continue;
                if constexpr (NT) __builtin_nontemporal_store(v, y + (size_t)row * a.O);
                else y[(size_t)row * a.O] = v;
            }
    }
}
// NB: 32-row blocks
template <int NB, bool DUAL, bool NT> __device__ __forceinline__ void fp4_many(const Fp4Args &a, const Fp4Item &it, int rb,
                                                                      int split, lds_u8 *lds) {
    using G = FmGeom;
    const Fp4Mat &mat = it.mat;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 31, g = lane >> 5;
    // operand r: two row tiles from rt[r] on (DUAL: the gate's and the up's of the same)
    int rt[2];
    __amdgpu_buffer_rsrc_t wr[2], sr[2];
    uint32_t wo[2], so[2];
#pragma unroll
    for (int r = 0; r < 2; r++) {
        rt[r] = DUAL ? (rb * 4 + wave) * 2 : (rb * 4 + wave) * 4 + 2 * r;
        const int t = min(rt[r], a.nrt - 1), two = min(2, a.nrt - t);   // past the last tile it is read again
        const size_t t0 = (size_t)t * a.nq;
        wr[r] = fp4_rsrc(uniform_ptr(DUAL && r ? mat.w1 : mat.w0) + t0 * COLI_TILE_BYTES, two * a.nq * COLI_TILE_BYTES);
        sr[r] = fp4_rsrc(uniform_ptr(DUAL && r ? mat.s1 : mat.s0) + t0 * 64, two * a.nq * 64);
        const int k = min(n >> 4, two - 1) * a.nq;
        wo[r] = k * COLI_TILE_BYTES + (32 * g + (n & 15)) * 16;   // slices 2 g and (256 bytes on) 2 g + 1 of row n
        so[r] = k * 64 + (n & 15) * 4;
    }
    const int s0 = split * a.sps, ns = min(a.cp / 256, s0 + a.sps);   // this workgroup's stages
    // Loaded: lane (n, g) has slices 2 g, 2 g + 1 of row n, a dword of each block. Turned:
    // its four dwords of block 2 t + g in wv[.][r][t], those that the lane 32 away had by
    // v_permlane32_swap. Scales: shifted so that bytes 0 and 2 are blocks g, 2 + g.
    u32x4 wv[3][2][2];
    uint32_t ws[3][2];
    auto load_w = [&](int p, int r, int q) {
        q = min(q, a.nq - 1);
        wv[p][r][0] = __builtin_amdgcn_raw_buffer_load_b128(wr[r], wo[r], q * COLI_TILE_BYTES, 0);
        wv[p][r][1] = __builtin_amdgcn_raw_buffer_load_b128(wr[r], wo[r] + 256, q * COLI_TILE_BYTES, 0);
        ws[p][r] = __builtin_amdgcn_raw_buffer_load_b32(sr[r], so[r], q * 64, 0);
    };
#pragma unroll
    for (int r = 0; r < 2; r++) load_w(0, r, 2 * s0);   // (ahead of the rows, whose addresses are loads away)
#pragma unroll
    for (int r = 0; r < 2; r++) load_w(1, r, 2 * s0 + 1);
    // operand row of the item's row r (a.rows: zeros), relative to the item's first (or
    // the zeros) where there is no src: offsets of 32 bits, see coli_hip_experts_a4_dev
    const int base = a.src ? 0 : min(it.r0, a.rows);
    auto row_of = [&](int r) {
        int x = it.r0 + min(r, it.nrows - 1);
        if (a.src) {
            x = a.src[x];
            x = x < 0 ? -1 : x / a.K;
        }
        return (uint32_t)(((unsigned)x < (unsigned)a.rows ? x : a.rows) - base);
    };
    const uint32_t qs = a.cp / 2, es = a.cp / 32;
    const __amdgpu_buffer_rsrc_t xqr = fp4_rsrc(a.xq + (size_t)base * qs, 0xffffffffu);
    const __amdgpu_buffer_rsrc_t xer = fp4_rsrc(a.xe + (size_t)base * es, 0xffffffffu);
    // codes: DMA k of the wave covers rows 8 (4 k + wave) .. + 7; scales: rows 32 wave + l / 2
    uint32_t xa[NB];
#pragma unroll
    for (int k = 0; k < NB; k++) {
        const int r = 8 * (4 * k + wave) + (lane >> 3);
        xa[k] = row_of(r) * qs + 16 * ((lane & 7) ^ ((r >> 1) & 7));
    }
    const uint32_t xs = row_of(32 * wave + (lane >> 1)) * es + 4 * (lane & 1);
    auto issue = [&](int s, lds_u8 *st) {
        s = min(s, ns - 1);
#pragma unroll
        for (int k = 0; k < NB; k++)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(xqr, (lds_void *)(st + (4 * k + wave) * 1024), 16, xa[k], s * 128, 0, 0);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(xer, (lds_void *)(st + G::kRows + wave * 256), 4, xs, s * 8, 0, 0);
    };
    auto turn = [&](int p, int r) {
        const u32x4 x = wv[p][r][0], y = wv[p][r][1];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const auto u = __builtin_amdgcn_permlane32_swap(x[2 * t], x[2 * t + 1], false, false);
            const auto v = __builtin_amdgcn_permlane32_swap(y[2 * t], y[2 * t + 1], false, false);
            wv[p][r][t] = (u32x4){u[0], v[0], u[1], v[1]};
        }
        ws[p][r] >>= 8 * g;
        asm("" : "+v"(ws[p][r]));   // (left alone, the shift moves to the use behind the loop's start, and its wait with it)
    };
    floatx16 acc[2][NB];
#pragma unroll
    for (int r = 0; r < 2; r++)
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int i = 0; i < 16; i++) acc[r][b][i] = 0.0f;
    // the lane's 16 bytes of a block's row n: step h, blocks 2 t + g
    int xo[4];
#pragma unroll
    for (int k = 0; k < 4; k++) xo[k] = n * 128 + 16 * ((2 * k + g) ^ ((n >> 1) & 7));
    u32x4 xv[3][2];   // the rows of this group, the next and the one after it
    u32x2 xe[NB];     // the stage's row scales
    int ev[2];        // this group's and the next's, shifted
    auto read_x = [&](int p, int t, int h, int b, const lds_u8 *st) {
        xv[p][t] = *(const __attribute__((address_space(3))) u32x4 *)(st + b * 4096 + xo[2 * h + t]);
    };
    auto read_e = [&](int b, const lds_u8 *st) {
        xe[b] = *(const __attribute__((address_space(3))) u32x2 *)(st + G::kRows + (32 * b + n) * 8);
    };
    // Group (step h of stage s, block b of rows): four MFMAs, each with its share of the
    // other work, in the order written here (left to the compiler, loads bunch up and
    // operands are read right before their use: 2048 x 14336 x 4096 73 us, so 66).
    // Beside them: reads of the rows two groups on, loads of the weights two steps on,
    // turns of the next step's weights, and in the second step the DMAs two stages on,
    // behind the barrier: by then every wave has the next stage's rows in and is done with
    // the stage before this one.
    constexpr int NG = 2 * NB;   // groups of a stage
    auto group = [&](int s, auto kt, auto gt, lds_u8 *const *slot) {
        constexpr int k3 = decltype(kt)::value, k = decltype(gt)::value, h = k / NB, b = k % NB, kk = 2 * k3 + h;
        constexpr int cur = kk % 3, nxt = (kk + 1) % 3, ld = (kk + 2) % 3;
        constexpr int gi = k3 * NG + k, p = gi % 3, pf = (gi + 2) % 3;          // row sets: this group's, that to fill
        constexpr int fk = (k + 2) % NG, fh = fk / NB, fb = fk % NB;            // the group two on
        constexpr int nk = (k + 1) % NG, nh = nk / NB, nb = nk % NB;            // and one on
        const lds_u8 *fst = slot[k + 2 < NG ? k3 : (k3 + 1) % 3];
        constexpr int every = NB / 2, r = b / every;                            // an operand of weights every so many groups
        const int q = min(2 * s + h + 2, a.nq - 1), sd = min(s + 2, ns - 1);
        auto mfma = [&](auto rt, auto tt) {
            constexpr int rr = decltype(rt)::value, t = decltype(tt)::value;
            acc[rr][b] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fp4_op(xv[p][t]), fp4_op(wv[cur][rr][t]), acc[rr][b], 4, 4, 2 * t,
                                                                         ev[gi & 1], 2 * t, (int)ws[cur][rr]);
        };
        auto dma = [&](int d) {   // d: 0 .. NB - 1 the codes, NB the scales
            lds_u8 *st = slot[(k3 + 2) % 3];
            if (d < NB)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(xqr, (lds_void *)(st + (4 * d + wave) * 1024), 16, xa[d], sd * 128, 0, 0);
            else if (d == NB)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(xer, (lds_void *)(st + G::kRows + wave * 256), 4, xs, sd * 8, 0, 0);
        };
        using C0 = std::integral_constant<int, 0>;
        using C1 = std::integral_constant<int, 1>;
        if constexpr (h == 1 && b == 0) {
            __builtin_amdgcn_s_waitcnt(0x0f76);   // vmcnt(6): all but the first step's weights, so the next stage's DMAs
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
        }
        mfma(C0{}, C0{});
        read_x(pf, 0, fh, fb, fst);
        if constexpr (b % every == 0) wv[ld][r][0] = __builtin_amdgcn_raw_buffer_load_b128(wr[r], wo[r], q * COLI_TILE_BYTES, 0);
        __builtin_amdgcn_sched_barrier(0);
        mfma(C1{}, C0{});
        if constexpr (fh == 0) read_e(fb, fst);
        if constexpr (h == 1) dma(b * (NB == 2 ? 2 : 1));
        if constexpr (b % every == every - 1) {
            const u32x4 x = wv[nxt][r][0], y = wv[nxt][r][1];
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const auto u = __builtin_amdgcn_permlane32_swap(x[2 * t], x[2 * t + 1], false, false);
                const auto v = __builtin_amdgcn_permlane32_swap(y[2 * t], y[2 * t + 1], false, false);
                wv[nxt][r][t] = (u32x4){u[0], v[0], u[1], v[1]};
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        mfma(C0{}, C1{});
        read_x(pf, 1, fh, fb, fst);
        if constexpr (b % every == 0) wv[ld][r][1] = __builtin_amdgcn_raw_buffer_load_b128(wr[r], wo[r] + 256, q * COLI_TILE_BYTES, 0);
        __builtin_amdgcn_sched_barrier(0);
        mfma(C1{}, C1{});
        if constexpr (b % every == 0) ws[ld][r] = __builtin_amdgcn_raw_buffer_load_b32(sr[r], so[r], q * 64, 0);
        if constexpr (b % every == every - 1) {
            ws[nxt][r] >>= 8 * g;
            asm("" : "+v"(ws[nxt][r]));   // (left alone, the shift moves to its use behind the loop's start, and the wait with it)
        }
        if constexpr (h == 1 && (NB == 2 || b == NB - 1)) dma(NB == 2 ? 2 * b + 1 : NB);
        ev[(gi + 1) & 1] = (int)(xe[nb][nh] >> (8 * g));
        __builtin_amdgcn_sched_barrier(0);
    };
    lds_u8 *const slot[3] = {lds, lds + G::kStage, lds + 2 * G::kStage};
    asm volatile("" ::"v"(lds) : "memory");
    issue(s0, slot[0]);
    issue(s0 + 1, slot[1]);
#pragma unroll
    for (int r = 0; r < 2; r++) turn(0, r);
    __builtin_amdgcn_s_waitcnt(0);   // (a builtin: the compiler counts on from it)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int k = 0; k < 2; k++) {   // (two groups: k < NB)
        read_x(k, 0, 0, k, slot[0]);
        read_x(k, 1, 0, k, slot[0]);
        read_e(k, slot[0]);
    }
    ev[0] = (int)(xe[0][0] >> (8 * g));
    __builtin_amdgcn_sched_barrier(0);
    auto stage = [&](int s, auto kt) {
        group(s, kt, std::integral_constant<int, 0>{}, slot);
        group(s, kt, std::integral_constant<int, 1>{}, slot);
        group(s, kt, std::integral_constant<int, 2>{}, slot);
        group(s, kt, std::integral_constant<int, 3>{}, slot);
        if constexpr (NB == 4) {
            group(s, kt, std::integral_constant<int, 4>{}, slot);
            group(s, kt, std::integral_constant<int, 5>{}, slot);
            group(s, kt, std::integral_constant<int, 6>{}, slot);
            group(s, kt, std::integral_constant<int, 7>{}, slot);
        }
    };
    for (int s = s0;;) {
        stage(s, std::integral_constant<int, 0>{});
        if (++s >= ns) break;
        stage(s, std::integral_constant<int, 1>{});
        if (++s >= ns) break;
        stage(s, std::integral_constant<int, 2>{});
        if (++s >= ns) break;
    }
    // the last DMAs write this workgroup's LDS: none may outlive it
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if constexpr (DUAL) {   // gates below COLI_FP4_LOW are rare: looked for by their bits, once for the wave
        uint32_t m = 0;
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int i = 0; i < 16; i++) m = max(m, __float_as_uint(acc[0][b][i]));
        if (__any(m > __float_as_uint(COLI_FP4_LOW))) {
            fp4_store<NB, DUAL, NT, true>(a, it, rt, split, n, g, acc);
            return;
        }
    }
    fp4_store<NB, DUAL, NT, false>(a, it, rt, split, n, g, acc);
}
// Workgroups of one XCD (every eighth) take consecutive tiles, a group of items' tiles of
// one block of weights before the next block's, so that both stay in its L2: eight items
// of one matrix (one item at a time: 8192 x 8192 x 2048 100 -> 112 us), one where experts
// have few tiles and their weights are the stream (64 pairs of 2048 x 1024, 256 rows each
// 89 -> 85 us; 16 pairs of 7168 x 2048, 750 rows each 280 -> 287).
// NT: y past the caches (a template's: of two stores under a branch the compiler makes one
// and drops the hint).
template <bool DUAL, bool NT> __global__ __launch_bounds__(256, 2) void coli_fp4_many(Fp4Args a, int n_items) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];   // FmGeom::kPD stages
    const int n = a.items ? min(*a.n_items - a.item0, n_items) : n_items;   // (none left: 0 or less)
    const int total = n * a.rtb * a.splits, per = (total + 7) / 8, j = blockIdx.x >> 3;
    int id = (blockIdx.x & 7) * per + j;
    if (j >= per || id >= total) return;
    const int split = id / (n * a.rtb);
    id -= split * n * a.rtb;
    const int grp = id / (a.group * a.rtb), in = id - grp * a.group * a.rtb, gi = min(a.group, n - grp * a.group);
    const int item = a.item0 + grp * a.group + in % gi, rb = in / gi;
    Fp4Item it = {a.mat0, item * a.tile, min(a.tile, a.S - item * a.tile)};
    if (a.items) it = a.items[item];
    if (it.nrows <= 64) fp4_many<2, DUAL, NT>(a, it, rb, split, (lds_u8 *)lds);
    else fp4_many<4, DUAL, NT>(a, it, rb, split, (lds_u8 *)lds);
}

// The K splits' sums in their order: n outputs, four a thread.
__global__ __launch_bounds__(256) void coli_fp4_join(const float *part, int splits, size_t n, float *y) {
    const size_t i = ((size_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i + 4 <= n) {
        floatx4 v = {};
        for (int p = 0; p < splits; p++) v += *GPTR(f4u, part + p * n + i);
        *(f4u *)(y + i) = v;
    } else {
        for (size_t k = i; k < n; k++) {
            float v = 0.0f;
            for (int p = 0; p < splits; p++) v += part[p * n + k];
            y[k] = v;
        }
    }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
static int lanes_log2(int cols, int V) {   // lanes of a row, V columns each: a block's to 256
    int l = V == 4 ? 3 : 2;
    while (l < 8 && (V << l) < cols) l++;
    return l;
}

// Workgroups for rows of `cols` columns: groups of rows, and a row of more than one step
// of 256 lanes by several: where groups are few, up to 2048 in all (8192 rows of 7168 bf16:
// 55 us whole, 59 in pieces), and where f32 rows are many and more than six steps long
// (operands and their product through 1024 outputs: 2048 rows of 14336 61 -> 57 us, 3000 of
// 7168 52.5 -> 51.8; but 8000 of 4096 51 -> 52.6, 600 of 14336 30 -> 33. At the step, rows of
// 14336 and back: 1024 of them, in two pieces, 28.0, 1025 in eight 29.6, whole 30.1).
static unsigned mx_grid(int rows, int cols, int V, int lpr, int *chunks) {
    const unsigned groups = (unsigned)((rows + (256 >> lpr) - 1) / (256 >> lpr)), steps = (unsigned)((cols + (V << lpr) - 1) / (V << lpr));
    const unsigned most = V == 4 && groups > 1024 && steps > 6 ? (8192 + groups) / groups : 2048 / groups;
    *chunks = (int)std::max(1u, std::min(steps, most));
    return groups * *chunks;
}

static size_t mx_q4_bytes(int rows, int cols) { return (size_t)rows * ((cols + 1) / 2); }
static size_t mx_e8_bytes(int rows, int cols) { return (size_t)rows * ((cols + 31) / 32); }

template <typename T> static void quant_launch(QuantArgs &a, hipStream_t st) {
    constexpr int V = 16 / sizeof(T);
    a.lpr = lanes_log2(a.cols, V);
    const dim3 g(mx_grid(a.rows, a.cols, V, a.lpr, &a.chunks));
    if (a.cols < V) hipLaunchKernelGGL((coli_mx_quant<T, 2>), g, dim3(256), 0, st, a);
    else if (a.cols % V) hipLaunchKernelGGL((coli_mx_quant<T, 1>), g, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((coli_mx_quant<T, 0>), g, dim3(256), 0, st, a);
}
template <typename T> static void dequant_launch(const DequantArgs &a, dim3 g, bool nt, hipStream_t st) {
    // (f32: a lane's 32 bytes are two stores of half lines, which past the caches are
    // written twice: 8000 rows of 14336 and back 229 -> 305 us)
    if (nt && sizeof(T) == 2) hipLaunchKernelGGL((coli_mx_dequant<T, sizeof(T) == 2>), g, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((coli_mx_dequant<T, false>), g, dim3(256), 0, st, a);
}
static int quantize(DevCtx *ctx, const void *x, int dtype, int rows, int cols, uint8_t *q4, uint8_t *e8) {
    QuantArgs a = {x, q4, e8, rows, cols, cols, 0, 1};
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
    DequantArgs a = {q4, e8, y, rows, cols, lanes_log2(cols, 8), 1};
    const dim3 g(mx_grid(rows, cols, 8, a.lpr, &a.chunks));
    const bool nt = yb > ((size_t)128 << 20);   // more than the 256 MB cache keeps for whoever reads y next
    if (dtype == 0) dequant_launch<float>(a, g, nt, ctx->stream);
    else if (dtype == 1) dequant_launch<_Float16>(a, g, nt, ctx->stream);
    else dequant_launch<__bf16>(a, g, nt, ctx->stream);
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
static int fp4_prep(DevCtx *ctx, const float *x, int rows, int I, const ItemArgs *it, Fp4Args *a) {
    const int cp = (I + 255) / 256 * 256;
    const size_t n = (size_t)rows + 1, qb = (n * (cp / 2) + 255) & ~(size_t)255, eb = n * (cp / 32);
    if (!reserve_kept(ctx, &ctx->fp4_x, qb + eb, 0)) return 0;
    uint8_t *p = (uint8_t *)ctx->fp4_x.p;
    QuantArgs q = {x, p, p + qb, rows, I, cp, lanes_log2(cp, 4), 1};
    const int nblk = (int)mx_grid(rows + 1, cp, 4, q.lpr, &q.chunks);
    const dim3 g(nblk + (it ? 1 : 0));
    const ItemArgs none = {};
    if (I < 4) hipLaunchKernelGGL(coli_fp4_prep<2>, g, dim3(256), 0, ctx->stream, q, it ? *it : none);
    else if (I % 4) hipLaunchKernelGGL(coli_fp4_prep<1>, g, dim3(256), 0, ctx->stream, q, it ? *it : none);
    else hipLaunchKernelGGL(coli_fp4_prep<0>, g, dim3(256), 0, ctx->stream, q, it ? *it : none);
    if (!hip_check(hipGetLastError(), "fp4 operands")) return 0;
    a->xq = p;
    a->xe = p + qb;
    a->cp = cp;
    a->rows = rows;
    return 1;
}

// How S rows of a matrix are multiplied: rows of a tile (COLI_FP4_MANY: that kernel),
// row tiles a workgroup of the kernel of few rows, K splits of the one of many, and
// whether the former quantizes the rows itself.
struct Fp4Plan {
    int tile, R, splits;
    bool own;
};
// Row tiles a workgroup: as many as leave most CUs one, since each workgroup reads all the
// rows' operands (4096 x 14336, us with 1 / 2 / 4: 16 rows 13.9 / 11.0 / 9.7, 64 rows 37 /
// 23 / 18; 14336 x 4096, 16 rows: 15.1 / 17.7 / 21.3).
static int fp4_row_tiles(const DevCtx *ctx, int nrt, bool dual) {
    int R = 1;
    while (!dual && R < 4 && nrt / (2 * R) >= ctx->cu_count * 4 / 5) R *= 2;
    return R;
}
static const char *fp4_pin(void) { return std::getenv("COLI_HIP_FP4"); }
static Fp4Plan fp4_plan(const DevCtx *ctx, const ColiCudaTensor *t, int S) {
    const int cp = (t->I + 255) / 256 * 256, cus = ctx->cu_count;
    Fp4Plan p = {S <= 16 ? 16 : S <= 32 ? 32 : 64, fp4_row_tiles(ctx, t->nrt, false), 1, false};
    // Quantizing the rows in every workgroup against a launch of their own (3 us): up to
    // 16384 columns in all, 49152 where there is a workgroup a CU at most (14336 x 4096, 3
    // rows: 13.9 / 14.2 us, 4096 x 14336 with four tiles a workgroup, 4 rows 8.4 / 8.9, 8
    // rows 9.9 / 9.2; 7168 x 2048, 8 rows 10.6 / 10.6).
    const int64_t cols = (int64_t)S * cp;
    p.own = S <= 32 && t->I >= 8 && cols <= (t->nrt <= cus ? 49152 : 16384);
    if (p.own)   // few columns: each workgroup's share of the work is small beside its latency
        while (p.R > 1 && cols * (t->nrt / (p.R / 2)) <= (int64_t)4096 * 1024) p.R /= 2;
    // The kernel of many rows, modelled in us from measurements: 8 and a stage of 256
    // columns 0.72 (1.06 with every CU at it), each further workgroup of a CU as much
    // again, a join of K splits 2.5 and 0.3 a MB of sums. The other: 5.5, the weights at
    // 6.5 TB/s for each tile of rows, the rows' operands, once for each workgroup, at 5
    // TB/s, and the results at 2.5 TB/s.
    const int ns = cp / 256, wgs = (S + COLI_FP4_MANY - 1) / COLI_FP4_MANY * ((t->nrt + 15) / 16);
    double best = 1e30;
    for (int P = 1; P <= 32 && P <= ns; P *= 2) {
        const int sps = (ns + P - 1) / P, n = wgs * P;
        const double full = std::min(1.0, (double)n / cus);
        const double us = 8.0 + sps * (0.72 + 0.34 * full) * std::max(1.0, (double)n / cus) +
                          (P > 1 ? 2.5 + 0.3e-6 * 4.0 * P * (double)S * t->O : 0.0);
        if (us < best) {
            best = us;
            p.splits = P;
        }
    }
    const int nwg = (t->nrt + p.R - 1) / p.R, tiles = (S + p.tile - 1) / p.tile;
    const double few = 5.5 + tiles * (double)t->w_bytes / 6.5e6 +
                       0.2e-6 * nwg * (double)S * cp * 0.53 * std::max(1.0, 0.8 * cus / (nwg * tiles)) +
                       0.4e-6 * 4.0 * S * t->O;
    const char *pin = fp4_pin();
    if (pin ? std::strcmp(pin, "many") == 0 : S > 16 && best < few) {
        p.tile = COLI_FP4_MANY;
        p.own = false;
    }
    return p;
}

template <int NM, int FORM> static void few_launch(const Fp4Args &a, dim3 g, bool dual, int R, hipStream_t st) {
    const dim3 b(64 * COLI_FP4_WAVES);
    const size_t own = FORM < 0 ? 0 : (size_t)a.rows * (a.cp / 2 + a.cp / 32);
    if constexpr (FORM < 0) {   // (rows of pairs come as operands)
        if (dual) {
            hipLaunchKernelGGL((coli_fp4_few<NM, 2, true, FORM>), g, b, 0, st, a);
            return;
        }
    }
    if (R == 4) hipLaunchKernelGGL((coli_fp4_few<NM, 4, false, FORM>), g, b, own, st, a);
    else if (R == 2) hipLaunchKernelGGL((coli_fp4_few<NM, 2, false, FORM>), g, b, own, st, a);
    else hipLaunchKernelGGL((coli_fp4_few<NM, 1, false, FORM>), g, b, own, st, a);
}

// Workgroups of an item, and how many items a launch takes: 2^32 threads are its limit. 0 where
// one item has more (beyond 2^27 - 16 outputs).
static int fp4_blocks(int nrt, bool dual, const Fp4Plan &plan, int *rtb) {
    const int R = plan.tile == COLI_FP4_MANY ? (dual ? 8 : 16) : plan.R;
    *rtb = (nrt + R - 1) / R;
    return (int)(((1 << 23) - 1) / ((int64_t)*rtb * plan.splits));
}

// The launches over n_items items of tiles of a.tile rows, `rows` in all.
static int fp4_run(DevCtx *ctx, Fp4Args &a, int n_items, int rows, bool dual, const Fp4Plan &plan) {
    const int most = fp4_blocks(a.nrt, dual, plan, &a.rtb);
    if (!most) return 0;
    if (a.tile == COLI_FP4_MANY) {
        a.sps = (a.cp / 256 + plan.splits - 1) / plan.splits;
        a.splits = (a.cp / 256 + a.sps - 1) / a.sps;
        if (a.splits > 1 && !reserve_kept(ctx, &ctx->fp4_part, (size_t)a.splits * a.S * a.O * 4, 0)) return 0;
        a.part = (float *)ctx->fp4_part.p;
        // Outputs beyond half of the 256 MB cache go past it (8192 x 4096 x 14336 380 -> 290
        // us); smaller ones may be there still when they are read (2048 rows: no difference).
        const bool nt = a.splits == 1 && (size_t)rows * a.O * 4 > ((size_t)128 << 20);
        const size_t shm = FmGeom::kPD * FmGeom::kStage;
        for (a.item0 = 0; a.item0 < n_items; a.item0 += most) {
            const int n = std::min(most, n_items - a.item0);
            const dim3 g((unsigned)(n * a.rtb * a.splits + 7) / 8 * 8);
            if (dual && nt) hipLaunchKernelGGL((coli_fp4_many<true, true>), g, dim3(256), shm, ctx->stream, a, n);
            else if (dual) hipLaunchKernelGGL((coli_fp4_many<true, false>), g, dim3(256), shm, ctx->stream, a, n);
            else if (nt) hipLaunchKernelGGL((coli_fp4_many<false, true>), g, dim3(256), shm, ctx->stream, a, n);
            else hipLaunchKernelGGL((coli_fp4_many<false, false>), g, dim3(256), shm, ctx->stream, a, n);
            if (!hip_check(hipGetLastError(), "fp4 product")) return 0;
        }
        if (a.splits > 1) {
            const size_t n = (size_t)a.S * a.O;
            hipLaunchKernelGGL(coli_fp4_join, dim3((unsigned)((n + 1023) / 1024)), dim3(256), 0, ctx->stream, a.part, a.splits, n, a.y);
        }
        return hip_check(hipGetLastError(), "fp4 join");
    }
    const int R = plan.R;
    for (a.item0 = 0; a.item0 < n_items; a.item0 += most) {
        const dim3 g((unsigned)std::min(most, n_items - a.item0) * a.rtb);
        if (a.x && a.I % 8 && a.tile <= 16) few_launch<1, 1>(a, g, dual, R, ctx->stream);
        else if (a.x && a.I % 8) few_launch<2, 1>(a, g, dual, R, ctx->stream);
        else if (a.x && a.tile <= 16) few_launch<1, 0>(a, g, dual, R, ctx->stream);
        else if (a.x) few_launch<2, 0>(a, g, dual, R, ctx->stream);
        else if (a.tile <= 16) few_launch<1, -1>(a, g, dual, R, ctx->stream);
        else if (a.tile <= 32) few_launch<2, -1>(a, g, dual, R, ctx->stream);
        else few_launch<4, -1>(a, g, dual, R, ctx->stream);
        if (!hip_check(hipGetLastError(), "fp4 product")) return 0;
    }
    return 1;
}

#define COLI_FP4_MAX_I (1 << 21)       // a tile's operand rows lie within 2 GiB (128 MiB)
#define COLI_FP4_MAX_ROWS (1 << 23)

int matmul_a4_dev(DevCtx *ctx, ColiCudaTensor *t, float *y_dev, const float *x_dev, int S) {
    Fp4Args a = {};
    if (t->I > COLI_FP4_MAX_I || S > COLI_FP4_MAX_ROWS) return 0;
    const Fp4Plan plan = fp4_plan(ctx, t, S);
    if (!fp4_blocks(t->nrt, false, plan, &a.rtb)) return 0;
    forget_emitted(ctx, y_dev, (size_t)S * t->O * 4);
    a.tile = plan.tile;
    if (plan.own) {
        a.x = x_dev;
        a.I = t->I;
        a.cp = (t->I + 255) / 256 * 256;
        a.rows = S;
    } else if (!fp4_prep(ctx, x_dev, S, t->I, nullptr, &a)) {
        return 0;
    }
    a.mat0 = {t->w, (const uint8_t *)t->sc, nullptr, nullptr};
    a.S = S;
    a.group = 8;
    a.nrt = t->nrt;
    a.nq = t->nq;
    a.O = t->O;
    a.K = 1;
    a.y = y_dev;
    return fp4_run(ctx, a, (S + a.tile - 1) / a.tile, S, false, plan);
}

extern "C" int coli_hip_fp4_matmul_a4_dev(ColiCudaTensor *t, float *y_dev, const float *x_dev, int S) {
    if (fault_injected()) return 0;
    if (!t || t->kind != COLI_KIND_FP4 || !y_dev || !x_dev || S < 1 || S > COLI_FP4_MAX_ROWS ||
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
                t->I > COLI_FP4_MAX_I) {
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
    if (!x || rows < 0 || rows > COLI_FP4_MAX_ROWS || N < 0 || N > COLI_FP4_MAX_ROWS || K < 1 || (N && (!y || !offsets || !xr || !rows)))
        return 0;
    const size_t yb = (size_t)N * x->O * 4;
    if (!outputs_apart({{y, yb}, {xr, (size_t)rows * x->I * 4}, {src, (size_t)N * 4}, {offsets, (size_t)(x->E + 1) * 4}}, 1))
        return 0;
    DevCtx *ctx = ctx_of(x->device);
    if (!bind_ctx(ctx)) return 0;
    if (!N) return 1;
    ItemArgs it = {};
    it.offsets = offsets;
    it.mats = x->mats;
    it.E = x->E;
    it.N = N;
    // Tiles by the rows of an expert, were all that have some alike (us with tiles of 16 /
    // of 128 rows on that kernel: 64 pairs of 2048 x 1024, 256 rows 25.6 / 29.3, 512 28.5 /
    // 30.3, 1024 41 / 31; 32 pairs of 7168 x 2048, 256 rows 90 / 96, 512 137 / 99).
    const int mean = N / std::min(N, x->E);
    const char *pin = fp4_pin();
    Fp4Plan plan = {mean <= 8 ? 16 : COLI_FP4_MANY, fp4_row_tiles(ctx, x->nrt, x->dual != 0), 1, false};
    // (that kernel's rows lie within 2 GiB of their first, so of x where src chooses them)
    const size_t xb = ((size_t)rows + 1) * (((size_t)x->I + 255) / 256 * 128);
    if (src && xb > ((size_t)1 << 31)) plan.tile = mean <= 16 ? 16 : 64;
    else if (pin) plan.tile = std::strcmp(pin, "many") == 0 ? COLI_FP4_MANY : mean <= 16 ? 16 : mean <= 32 ? 32 : 64;
    Fp4Args a = {};
    if (!fp4_blocks(x->nrt, x->dual != 0, plan, &a.rtb)) return 0;
    forget_emitted(ctx, y, yb);
    it.tile = plan.tile;
    it.room = (int)std::min<int64_t>(N, N / it.tile + x->E);
    if (!reserve_kept(ctx, &ctx->fp4_items, 256 + (size_t)it.room * sizeof(Fp4Item), 0)) return 0;
    it.n_items = (int *)ctx->fp4_items.p;
    it.items = (Fp4Item *)((uint8_t *)ctx->fp4_items.p + 256);
    if (!fp4_prep(ctx, xr, rows, x->I, &it, &a)) return 0;
    a.items = it.items;
    a.n_items = it.n_items;
    a.tile = it.tile;
    a.group = mean < 512 ? 1 : 8;
    a.nrt = x->nrt;
    a.nq = x->nq;
    a.O = x->O;
    a.src = src;
    a.K = K;
    a.y = y;
    a.limit = x->limit;
    return fp4_run(ctx, a, it.room, N, x->dual != 0, plan);
}
