// gemm_t.hip -- the input gradient of a resident projection: dx = dy W.
//
//   dx[s, i] = sum_o dy[s, o] n[o, i] sc[o, i / 32]
//
// The sum runs over O, along which the tiles hold one row a lane and the group
// scales change, so neither the forward's operand layout nor its scaling of
// results fits. Both are turned round in registers:
//   * A wave takes half a tile quad, 64 columns: lane (o = lane % 16, c =
//     lane / 16) loads dwords 2 h, 2 h + 1 of its 16 bytes, 8 nibbles of
//     columns 64 h + 32 j + 8 c + t. An 8 x 8 nibble transpose among the eight
//     lanes o % 8 (three exchanges: nibbles, bytes, halfwords with lanes ^1,
//     ^2, ^4) makes t the lane and o % 8 the nibble; one exchange with lane ^8
//     and one v_permlane32_swap then put o / 8 into lane bit 5 and the columns'
//     j into lane bit 3. Lane l holds column 64 h + 32 (l / 8 % 2) + 16 r + 8 (l / 16 % 2)
//     + l % 8 in register r, rows 8 (l / 32) + 0..7: the B operand of
//     v_mfma_f32_32x32x16_f16. About 1.3 instructions a weight, no LDS.
//   * A weight enters as n sc 2^-Eg in fp16 hi + lo, Eg the exponent of its
//     column group's largest scale over all rows of W (it must be one: the sum
//     over the rows is taken before it is applied); dy as fp16 hi + lo under its
//     row's exponent (2^-22). hi hi + hi lo + lo hi are summed in f32. Weights of
//     MXFP4 (lo is zero and left out) and of fp16 scales are exact while their
//     scale is within 2^-35 and 2^-22 of that largest one; f32 scales enter as two
//     fp16, to 3 x 2^-22 within 2^-11 of it. Smaller scales lose places to fp16's
//     least one: a weight is off by at most 8 x 2^-32 of the largest scale (MXFP4
//     7 x 2^-37) beside that, and zero where its scale is below. The forward, which
//     applies scales to results, does not lose them. The scales are kept a second
//     time per tensor, by column group with eight rows' worth in 16 bytes
//     (coli_t_scales, made on first use).
//
// Many rows run at the rate of a large library product: 2048 x 4096 x 14336
// int4, three products, 600 us, 1.2 PFLOP/s of fp16 products (8192^3 by the
// library: 1.07), the matrix units busy for 54 % of the cycles, waves waiting for
// a third of theirs; 512 rows 187 us with the join (7 us) and the build of dy's
// operands (16 us, 59 MB at 3.8 TB/s) to come. f32 scales (a second plane of them)
// take 3 to 6 % longer: whole calls of 512 rows 183 us against 177. Few rows: see
// coli_gemm_t_few.
#include "coli_hip_host.h"
#include "coli_device.h"

#include "coli_backend_abi.h"
#include "coli_hip_ext.h"

#include <algorithm>
#include <cstdlib>
#include <cstring>

// ---------------------------------------------------------------------------
// scales by column group
// ---------------------------------------------------------------------------
// Workgroup q: the four column groups of tile quad q. sct[plane][4 q + j][octet]
// holds eight rows' scales times 2^-Eg (int4: odd rows also / 16, their nibbles
// unpack as 16 n; plane 1: the rest that fp16 leaves of an f32 scale).
template <int KIND>
__global__ __launch_bounds__(256) void coli_t_scales(const void *__restrict__ sc, int nrt, int nq, int noct,
                                                     _Float16 *__restrict__ sct, int *__restrict__ ge) {
    __shared__ float mx[256];
    __shared__ int es[4];
    const int q = blockIdx.x, tid = threadIdx.x;
    auto scale = [&](int o, int j) -> float {
        if (o >= nrt * 16) return 0.0f;
        const size_t at = ((size_t)(o >> 4) * nq + q) * 64 + (o & 15) * 4 + j;
        if constexpr (KIND == COLI_KIND_I4_H) return (float)((const _Float16 *)sc)[at];
        else if constexpr (KIND == COLI_KIND_I4_F) return ((const float *)sc)[at];
        else return __uint_as_float((uint32_t)((const uint8_t *)sc)[at] << 23);
    };
    float m = 0.0f;
    for (int e = tid; e < nrt * 64; e += 256) {
        const float s = fabsf(scale(e >> 2, e & 3));   // e & 3 == tid & 3
        if (s < INFINITY) m = fmaxf(m, s);
    }
    mx[tid] = m;
    __syncthreads();
    if (tid < 4) {
        for (int k = tid; k < 256; k += 4) m = fmaxf(m, mx[k]);
        int E = 0;
        if (m > 0.0f) {
            frexpf(m, &E);       // m in [2^(E-1), 2^E)
            // int4: |16 n| (s / 16) <= 128 * 2^8; e2m1: 6 * 2^12
            E -= KIND == COLI_KIND_FP4 ? 13 : 12;
        }
        es[tid] = E;
        ge[4 * q + tid] = E;
    }
    __syncthreads();
    const size_t plane = (size_t)nq * 4 * noct * 8;
    for (int e = tid; e < 4 * noct * 8; e += 256) {
        const int j = e / (noct * 8), k = e - j * noct * 8;
        const int o = (k & ~7) + t_order(KIND != COLI_KIND_FP4, k & 7);
        float s = ldexpf(scale(o, j), -es[j]);
        if (KIND != COLI_KIND_FP4 && (o & 1)) s *= 0.0625f;
        const _Float16 h = (_Float16)s;
        const size_t at = ((size_t)4 * q + j) * noct * 8 + k;
        sct[at] = h;
        if constexpr (KIND == COLI_KIND_I4_F) sct[plane + at] = (_Float16)(s - (float)h);
    }
}

// ---------------------------------------------------------------------------
// dy as fp16 hi + lo
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(1024) void coli_t_prep_rows(ColiTPrepArgs a) { coli_t_prep_block(a, blockIdx.x); }

// ---------------------------------------------------------------------------
// the product
// ---------------------------------------------------------------------------
struct GemmTArgs {
    const uint8_t *w;            // tiles [nrt][nq]
    const _Float16 *sct;
    const int *ge;               // [4 nq]
    const _Float16 *hi, *lo;     // [noct][Sp][8] (coli_gemm_t)
    const int *exps;             // [S]
    size_t Sp;
    const float *dy;             // [S][O] (coli_gemm_t_few)
    int O;                       // its columns, at least 4
    int nrt, nq, noct, I, S;
    int splits, per;             // K split: steps of 32 rows of W each
    float *out;                  // [splits][S][I]
};

// 8 x 8 nibble transpose among lanes l ^ 0..7 (nibble t of lane o -> nibble o of lane t).
struct NibT {
    uint32_t rot, keep, bsel, hsel;
};
__device__ __forceinline__ NibT nib_consts(int lane) {
    NibT c;
    c.rot = lane & 1 ? 4u : 28u;                      // rotate right by
    c.keep = lane & 1 ? 0xF0F0F0F0u : 0x0F0F0F0Fu;
    // perm(x, y): bytes 4-7 are x's
    c.bsel = lane & 2 ? 0x07030501u : 0x02060004u;
    c.hsel = lane & 4 ? 0x07060302u : 0x01000504u;
    return c;
}
__device__ __forceinline__ uint32_t nib_transpose(uint32_t x, const NibT &c) {
    uint32_t y = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0xB1, 0xF, 0xF, false);        // lane ^ 1
    y = __builtin_amdgcn_alignbit(y, y, c.rot);
    x = (x & c.keep) | (y & ~c.keep);
    y = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x4E, 0xF, 0xF, false);                 // lane ^ 2
    x = __builtin_amdgcn_perm(x, y, c.bsel);
    y = (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, 0x104, 0xF, 0x5, false);           // lane + 4
    y = (uint32_t)__builtin_amdgcn_update_dpp((int)y, (int)x, 0x114, 0xF, 0xA, false);           // lane - 4
    return __builtin_amdgcn_perm(x, y, c.hsel);
}

// The two dwords (columns 32 j + ...) of a lane as two B operands' nibbles.
__device__ __forceinline__ void half_quad(uint32_t d0, uint32_t d1, const NibT &c, uint32_t &b0, uint32_t &b1) {
    d0 = nib_transpose(d0, c);
    d1 = nib_transpose(d1, c);
    // lane bit 3 <-> register (lane ^ 8), then lane bit 5 <-> register
    const uint32_t e0 = (uint32_t)__builtin_amdgcn_update_dpp((int)d0, (int)d1, 0x128, 0xF, 0xC, false);
    const uint32_t e1 = (uint32_t)__builtin_amdgcn_update_dpp((int)d1, (int)d0, 0x128, 0xF, 0x3, false);
    const auto r = __builtin_amdgcn_permlane32_swap(e0, e1, false, false);
    b0 = r[0];
    b1 = r[1];
}

// hi (and lo) of eight weights from their nibbles and scales.
template <int KIND>
__device__ __forceinline__ void t_weights(uint32_t nib, half8v s, half8v s2, half8v &hi, half8v &lo) {
    const half8v n = unpack_b<KIND>(nib);
    hi = n * s;   // (pairs: v_pk_mul_f16)
    if constexpr (KIND == COLI_KIND_FP4) {
        (void)lo;
    } else {
#pragma unroll
        for (int p = 0; p < 4; p++) {
            const half2v nn = {n[2 * p], n[2 * p + 1]}, ss = {s[2 * p], s[2 * p + 1]}, hh = {hi[2 * p], hi[2 * p + 1]};
            half2v l = __builtin_elementwise_fma(nn, ss, -hh);   // exact: 15 bits less 11
            if constexpr (KIND == COLI_KIND_I4_F) {
                const half2v s2p = {s2[2 * p], s2[2 * p + 1]};
                l = __builtin_elementwise_fma(nn, s2p, l);
            }
            lo[2 * p] = l[0];
            lo[2 * p + 1] = l[1];
        }
    }
}

// One K step's products: a lane's dwords d of two row tiles' half-quad, their
// scales, and dy's octets in LDS ([part][octet][BM rows][8]).
template <int KIND, int MT>
__device__ __forceinline__ void t_products(const uint32_t (&d)[2][2], const half8v (&sc)[2], const half8v (&sc2)[2],
                                           const NibT &nc, const uint8_t *as, int lane, floatx16 (&acc)[MT][2]) {
    constexpr int BM = 32 * MT;
#pragma unroll
    for (int t = 0; t < 2; t++) {
        uint32_t b[2];
        half_quad(d[t][0], d[t][1], nc, b[0], b[1]);
        half8v bh[2], bl[2];
#pragma unroll
        for (int r = 0; r < 2; r++) t_weights<KIND>(b[r], sc[t], sc2[t], bh[r], bl[r]);
        const uint8_t *ap = as + (size_t)((2 * t + (lane >> 5)) * BM + (lane & 31)) * 16;
#pragma unroll
        for (int m = 0; m < MT; m++) {
            const half8v ah = *(const half8v *)(ap + m * 32 * 16);
            const half8v al = *(const half8v *)(ap + (4 * BM + m * 32) * 16);
#pragma unroll
            for (int r = 0; r < 2; r++) {
                acc[m][r] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, bh[r], acc[m][r], 0, 0, 0);
                acc[m][r] = __builtin_amdgcn_mfma_f32_32x32x16_f16(al, bh[r], acc[m][r], 0, 0, 0);
                if constexpr (KIND != COLI_KIND_FP4)
                    acc[m][r] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, bl[r], acc[m][r], 0, 0, 0);
            }
        }
    }
}

// Many rows: workgroup (64 WN columns, 32 MT rows, K split); WK wave groups
// share its K steps (32 rows of W: two row tiles) and are joined in LDS at the
// end. A step's dy octets are staged in LDS (two buffers), the weights and
// scales of the next step are requested before this one's products. 2048 x 4096
// x 14336 int4: 600 us; with one wave group, one wave a SIMD, 686 us.
template <int KIND, int MT, int WN, int WK>
__global__ __launch_bounds__(64 * WN * WK, 2) void coli_gemm_t(GemmTArgs a) {
    constexpr int BM = 32 * MT, NT = 64 * WN, CH = 8 * BM;   // 16-byte chunks of a step: 2 parts x 4 octets x BM rows
    constexpr int CPT = CH / NT;
    static_assert(CH % NT == 0, "whole chunks a thread");
    constexpr int STAGE = 8 * BM * 16;
    constexpr int JOIN = WK * (WK - 1) * (32 / WK) * NT * 4;
    constexpr int LDS = 2 * WK * STAGE > JOIN ? 2 * WK * STAGE : JOIN;
    __shared__ __attribute__((aligned(16))) uint8_t lds[LDS];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wn = wave % WN, wk = wave / WN;
    const int gt = tid - wk * NT;                              // thread within its K group
    const int hq = blockIdx.x * WN + wn, q = min(hq >> 1, a.nq - 1), h = hq & 1;   // half-quad
    const int row0 = blockIdx.y * BM;
    const int k0 = blockIdx.z * a.per, k1 = min((a.noct + 3) / 4, k0 + a.per);
    const int nstep = (k1 - k0 + WK - 1) / WK;
    const NibT nc = nib_consts(lane);
    // (a base of the whole wave and a 32-bit offset of the lane: no address
    // arithmetic on the VALU)
    const uint8_t *wp = a.w + (size_t)q * COLI_TILE_BYTES + 8 * h;
    const uint32_t wo = lane * 16;
    const size_t wstride = (size_t)a.nq * COLI_TILE_BYTES;
    const size_t plane = (size_t)a.nq * 4 * a.noct * 16;
    // lane bit 3: the column group, lane bit 5: the octet of a row tile
    const uint8_t *sp = (const uint8_t *)a.sct + ((size_t)4 * q + 2 * h) * a.noct * 16;
    const uint32_t so = (uint32_t)((lane >> 3 & 1) * a.noct + (lane >> 5)) * 16;
    floatx16 acc[MT][2];
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int r = 0; r < 2; r++)
#pragma unroll
            for (int i = 0; i < 16; i++) acc[m][r][i] = 0.0f;
    u32x2 wd[2];
    half8v sc[2], sc2[2];
    u32x4 ad[CPT];
    auto load_w = [&](int step) {
        step = min(step, k1 - 1);
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const uint8_t *wb = wp + min(2 * step + t, a.nrt - 1) * wstride;   // (past the last row tile: zero scales)
            const uint8_t *sb = sp + (size_t)(4 * step + 2 * t) * 16;
            wd[t] = *GPTR(u32x2, wb + wo);
            sc[t] = *GPTR(half8v, sb + so);
            if constexpr (KIND == COLI_KIND_I4_F) sc2[t] = *GPTR(half8v, sb + plane + so);
        }
    };
    auto load_a = [&](int step) {
        step = min(step, k1 - 1);
#pragma unroll
        for (int i = 0; i < CPT; i++) {
            // chunk c: part c / (4 BM) (the same for the whole workgroup), octet c / BM % 4, row c % BM
            static_assert(4 * BM % NT == 0, "a load is of one part");
            const int c = gt + i * NT;
            const uint8_t *ab = (const uint8_t *)(i * NT >= 4 * BM ? a.lo : a.hi) + ((size_t)4 * step * a.Sp + row0) * 16;
            ad[i] = *GPTR(u32x4, ab + (uint32_t)((c / BM % 4) * (uint32_t)a.Sp + c % BM) * 16);
        }
    };
    auto store_a = [&](int buf) {
#pragma unroll
        for (int i = 0; i < CPT; i++) *(u32x4 *)(lds + (size_t)(buf * WK + wk) * STAGE + (size_t)(gt + i * NT) * 16) = ad[i];
    };
    load_w(k0 + wk);
    load_a(k0 + wk);
    store_a(0);
    __syncthreads();
    for (int it = 0; it < nstep; it++) {
        const int step = k0 + it * WK + wk;
        uint32_t w0[2][2];
        half8v s0[2], s1[2];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            w0[t][0] = wd[t][0];
            w0[t][1] = wd[t][1];
            s0[t] = sc[t];
            s1[t] = sc2[t];
        }
        load_a(step + WK);
        load_w(step + WK);
        if (step < k1) t_products<KIND, MT>(w0, s0, s1, nc, lds + (size_t)((it & 1) * WK + wk) * STAGE, lane, acc);
        if (it + 1 < nstep) store_a((it + 1) & 1);
        __syncthreads();
    }
    // lane: column l % 32 of the operand; register i: row 8 (i / 4) + 4 (l / 32) + i % 4
    const int c0 = 128 * q + 64 * h + 32 * (lane >> 3 & 1) + 8 * (lane >> 4 & 1) + (lane & 7);
    const int E = a.ge[4 * q + 2 * h + (lane >> 3 & 1)];
    float *out = a.out + (size_t)blockIdx.z * a.S * a.I;
    // group g finishes registers i with i / (16 / WK) == g: the others' are
    // handed over through LDS, [g][the other][r][i][thread]
    constexpr int NI = 16 / WK;
    float *js = (float *)lds;
    auto at = [&](int g, int s, int r, int i) { return (((g * (WK - 1) + (s < g ? s : s - 1)) * 2 + r) * NI + i) * NT + gt; };
#pragma unroll
    for (int m = 0; m < MT; m++) {
        if (m) __syncthreads();
#pragma unroll
        for (int g = 0; g < WK; g++)
            if (g != wk)
#pragma unroll
                for (int r = 0; r < 2; r++)
#pragma unroll
                    for (int i = 0; i < NI; i++) js[at(g, wk, r, i)] = acc[m][r][g * NI + i];
        __syncthreads();
#pragma unroll
        for (int g = 0; g < WK; g++)
            if (g == wk)
#pragma unroll
                for (int i = 0; i < NI; i++) {
                    const int k = g * NI + i, row = row0 + 32 * m + 8 * (k >> 2) + 4 * (lane >> 5) + (k & 3);
                    const int e = E + a.exps[min(row, a.S - 1)];
#pragma unroll
                    for (int r = 0; r < 2; r++) {
                        float v = acc[m][r][k];
#pragma unroll
                        for (int s = 0; s < WK; s++)
                            if (s != g) v += js[at(g, s, r, i)];
                        if (row < a.S && hq < 2 * a.nq && c0 + 16 * r < a.I)
                            out[(size_t)row * a.I + c0 + 16 * r] = ldexpf(v, e);
                    }
                }
    }
}

// Few rows or a small W (t_plan): workgroup (tile quad, 32 rows, K split), eight
// waves that take its K steps in turn, each with all 128 columns and its own copy of the step's
// dy: read as f32 and converted on its way into the wave's LDS, under the
// exponent of the row's part in this split (the splits' sums are f32 already).
// No launch builds operands, and no barrier holds the waves together before
// their sums are joined. Transpose, unpack and conversion are about 450 VALU
// instructions a step of 4096 weights: 64 rows of 14336 x 4096 int4 (33 MB) take
// 46 us, the busy CUs' VALU issuing for 62 % of their cycles and waves waiting for
// 40 % of theirs; 16 rows of 7168 x 2048 MXFP4 (8.4 MB) 8.7 us and the join 2.8,
// latency. A 64-row form spilled its accumulators, so every 32 rows read and
// unpack the weights again.
template <int KIND, bool ODD>
__global__ __launch_bounds__(512, 2) void coli_gemm_t_few(GemmTArgs a) {
    constexpr int BM = 32, W = 8, CPT = 4 * BM / 64, STAGE = 8 * BM * 16, PD = 2;
    // the join: two accumulators of every wave at a time
    constexpr int LDS = 2 * W * 16 * 64 * 4;
    static_assert(W * STAGE <= LDS, "the waves' stages");
    __shared__ __attribute__((aligned(16))) uint8_t lds[LDS];
    __shared__ int rexp[BM];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int q = blockIdx.x, row0 = blockIdx.y * BM, live = min(BM, a.S - row0);
    const int k0 = blockIdx.z * a.per, k1 = min((a.noct + 3) / 4, k0 + a.per);
    const NibT nc = nib_consts(lane);
    // (a base of the whole wave and a 32-bit offset of the lane: no address
    // arithmetic on the VALU)
    const uint8_t *wp = a.w + (size_t)q * COLI_TILE_BYTES;
    const uint32_t wo = lane * 16;
    const size_t wstride = (size_t)a.nq * COLI_TILE_BYTES;
    const size_t plane = (size_t)a.nq * 4 * a.noct * 16;
    // lane bit 3: the column group of a half, lane bit 5: the octet of a row tile
    const uint8_t *sp = (const uint8_t *)a.sct + (size_t)4 * q * a.noct * 16;
    const uint32_t so = (uint32_t)((lane >> 3 & 1) * a.noct + (lane >> 5)) * 16;
    const float *dy = a.dy + (size_t)row0 * a.O;
    floatx16 acc[2][1][2];
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
        for (int r = 0; r < 2; r++)
#pragma unroll
            for (int i = 0; i < 16; i++) acc[h][0][r][i] = 0.0f;
    struct Step {
        u32x4 w[2];
        half8v s[2][2], s2[2][2];   // [half][row tile]
    };
    Step st[PD];
    float af[CPT][8];
    int ae[CPT];
    auto load_w = [&](int step, Step &p) {
        step = min(step, k1 - 1);
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const uint8_t *wb = wp + min(2 * step + t, a.nrt - 1) * wstride;   // (past the last row tile: zero scales)
            p.w[t] = *GPTR(u32x4, wb + wo);
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const uint8_t *sb = sp + ((size_t)2 * h * a.noct + 4 * step + 2 * t) * 16;
                p.s[h][t] = *GPTR(half8v, sb + so);
                if constexpr (KIND == COLI_KIND_I4_F) p.s2[h][t] = *GPTR(half8v, sb + plane + so);
            }
        }
    };
    // chunk c of a step: octet c % 4 of row c / 4 (a chunk of rows past S: skipped
    // where all of a load's are, else some row's, not kept)
    auto load_a = [&](int step) {
        step = min(step, k1 - 1);
#pragma unroll
        for (int i = 0; i < CPT; i++) {
            if (16 * i >= live) continue;
            const int c = lane + i * 64;
            t_load8<ODD>(dy + (uint32_t)(min(c >> 2, live - 1) * a.O), 4 * step + (c & 3), a.O, af[i]);
        }
    };
#pragma unroll
    for (int p = 0; p < PD; p++) load_w(k0 + wave + p * W, st[p]);
#pragma unroll
    for (int i = 0; i < CPT; i++)
#pragma unroll
        for (int e = 0; e < 8; e++) af[i][e] = 0.0f;
    load_a(k0 + wave);
    {
        // the rows' exponents over this split's columns
        constexpr int TPR = 64 * W / BM;   // threads a row
        const int r = tid / TPR;
        float m = 0.0f;
        const float *xr = dy + (size_t)min(r, live - 1) * a.O;
        // (requested eight at a time: the split's first products wait for this)
        for (int c = 32 * k0 + 4 * (tid % TPR); c < 32 * k1; c += 32 * TPR) {
            floatx4 v[8];
#pragma unroll
            for (int u = 0; u < 8; u++) v[u] = row4<ODD>(xr, min(c + 4 * u * TPR, 32 * k1 - 4), a.O);
#pragma unroll
            for (int u = 0; u < 8; u++)
                m = fmaxf(m, fmaxf(fmaxf(fabsf(v[u][0]), fabsf(v[u][1])), fmaxf(fabsf(v[u][2]), fabsf(v[u][3]))));
        }
#pragma unroll
        for (int o = 1; o < TPR; o <<= 1) m = fmaxf(m, __shfl_xor(m, o));
        if (tid % TPR == 0) rexp[r] = t_exponent(m);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < CPT; i++) ae[i] = rexp[(lane + i * 64) >> 2];
    }
    uint8_t *mine = lds + wave * STAGE;
    auto one = [&](int step, Step &p) {
#pragma unroll
        for (int i = 0; i < CPT; i++) {
            if (16 * i >= live) continue;   // (rows that are not kept: whatever LDS holds)
            const int c = lane + i * 64;
            half8v hv, lv;
            t_split8(af[i], KIND != COLI_KIND_FP4, ae[i], hv, lv);
            *(half8v *)(mine + ((c & 3) * BM + (c >> 2)) * 16) = hv;
            *(half8v *)(mine + ((4 + (c & 3)) * BM + (c >> 2)) * 16) = lv;
        }
        load_a(step + W);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // the wave's other lanes' chunks
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const uint32_t d[2][2] = {{p.w[0][2 * h], p.w[0][2 * h + 1]}, {p.w[1][2 * h], p.w[1][2 * h + 1]}};
            t_products<KIND, 1>(d, p.s[h], p.s2[h], nc, mine, lane, acc[h]);
        }
        load_w(step + PD * W, p);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // read before the next step's writes
    };
    for (int step = k0 + wave; step < k1; step += PD * W) {
        one(step, st[0]);
        if (step + W < k1) one(step + W, st[1]);
    }
    // wave w finishes registers 2 w, 2 w + 1 of both operands r
    float *js = (float *)lds;
    const int c0 = 128 * q + 32 * (lane >> 3 & 1) + 8 * (lane >> 4 & 1) + (lane & 7);
    float *out = a.out + ((size_t)blockIdx.z * a.S + row0) * a.I;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int E = a.ge[4 * q + 2 * h + (lane >> 3 & 1)];
        __syncthreads();
#pragma unroll
        for (int r = 0; r < 2; r++)
#pragma unroll
            for (int i = 0; i < 16; i++) js[((r * 16 + i) * W + wave) * 64 + lane] = acc[h][0][r][i];
        __syncthreads();
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int i = 2 * wave + u, row = 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3);
#pragma unroll
            for (int r = 0; r < 2; r++) {
                float v = js[(r * 16 + i) * W * 64 + lane];
#pragma unroll
                for (int s = 1; s < W; s++) v += js[((r * 16 + i) * W + s) * 64 + lane];
                const int c = c0 + 64 * h + 16 * r;
                if (row < live && c < a.I) out[(size_t)row * a.I + c] = ldexpf(v, E + rexp[row]);
            }
        }
    }
}

// dy of fewer than four columns as rows of four.
__global__ void coli_t_pad(const float *__restrict__ dy, float *__restrict__ to, int S, int O) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i < 4 * S) to[i] = (i & 3) < O ? dy[(size_t)(i >> 2) * O + (i & 3)] : 0.0f;
}

// Sum of the K splits, in order.
__global__ __launch_bounds__(256) void coli_t_join(const float *__restrict__ part, float *__restrict__ out, size_t n,
                                                   int splits) {
    const size_t i = ((size_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i + 4 <= n && n % 4 == 0) {
        floatx4 s = *GPTR(floatx4, part + i);
        for (int p = 1; p < splits; p++) s += *GPTR(floatx4, part + p * n + i);
        if (((uintptr_t)out & 15) == 0) {
            *(floatx4 *)(out + i) = s;
        } else {
            for (int k = 0; k < 4; k++) out[i + k] = s[k];
        }
    } else {
        for (size_t k = i; k < n && k < i + 4; k++) {
            float s = part[k];
            for (int p = 1; p < splits; p++) s += part[p * n + k];
            out[k] = s;
        }
    }
}

// Source-layout int4 whose groups are not multiples of 32 columns: one thread
// a column, rows of W in turn (the forward's scalar kernel, turned round).
__global__ __launch_bounds__(256) void coli_t_generic(const uint8_t *__restrict__ w, const float *__restrict__ sc, int gs,
                                                      int ng, int I, int O, const float *__restrict__ dy,
                                                      float *__restrict__ dx) {
    const int i = blockIdx.x * 256 + threadIdx.x, s = blockIdx.y;
    if (i >= I) return;
    const size_t rb = (size_t)(I + 1) / 2;
    const float *d = dy + (size_t)s * O;
    float acc = 0.0f;
    for (int o = 0; o < O; o++) {
        const int u = w[o * rb + (i >> 1)] >> (i & 1 ? 4 : 0) & 15;
        acc += d[o] * ((float)(u - 8) * sc[(size_t)o * ng + i / gs]);
    }
    dx[(size_t)s * I + i] = acc;
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
static int t_octets(const ColiCudaTensor *t) { return (t->nrt + 1) / 2 * 4; }

// The tensor's scales by column group: made on first use, rebuilt by
// fill_tensor after an update.
int build_t_scales(DevCtx *ctx, ColiCudaTensor *t, bool update_only) {
    if (t->kind == COLI_KIND_GENERIC || (update_only && !t->sct)) return 1;
    const int noct = t_octets(t), planes = t->kind == COLI_KIND_I4_F ? 2 : 1;
    const size_t sb = (size_t)planes * t->nq * 4 * noct * 16, bytes = sb + (size_t)t->nq * 4 * sizeof(int);
    const bool first = !t->sct;
    if (first) {
        // laid out by a graph they would be missing in every call before its replay
        hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
        if (!hip_check(hipStreamIsCapturing(ctx->stream, &cap), "transposed scales") || cap != hipStreamCaptureStatusNone)
            return 0;
        if (!hip_check(hipMalloc(&t->sct, bytes), "transposed scales")) return 0;
        t->sct_ge = (int *)((uint8_t *)t->sct + sb);
    }
#define COLI_TS(KD)                                                                                            \
    hipLaunchKernelGGL((coli_t_scales<KD>), dim3(t->nq), dim3(256), 0, ctx->stream, t->sc, t->nrt, t->nq, noct, \
                       (_Float16 *)t->sct, t->sct_ge)
    if (t->kind == COLI_KIND_I4_H) COLI_TS(COLI_KIND_I4_H);
    else if (t->kind == COLI_KIND_I4_F) COLI_TS(COLI_KIND_I4_F);
    else COLI_TS(COLI_KIND_FP4);
#undef COLI_TS
    const int ok = hip_check(hipGetLastError(), "transposed scales");
    if (first && ok) {
        t->sct_bytes = bytes;
        t->accounted += bytes;
        ctx->tensor_bytes += bytes;
    } else if (first) {
        (void)hipFree(t->sct);
        t->sct = nullptr;
    }
    return ok;
}

template <int KIND>
static void launch_gemm_t(const GemmTArgs &a, bool few, hipStream_t st) {
    const dim3 grid(a.nq, (a.S + 31) / 32, a.splits);
    if (few && a.O % 4 == 0)
        hipLaunchKernelGGL((coli_gemm_t_few<KIND, false>), grid, dim3(512), 0, st, a);
    else if (few)
        hipLaunchKernelGGL((coli_gemm_t_few<KIND, true>), grid, dim3(512), 0, st, a);
    else
        hipLaunchKernelGGL((coli_gemm_t<KIND, 4, 4, 2>), dim3((a.nq + 1) / 2, (a.S + 127) / 128, a.splits), dim3(512), 0, st, a);
}

// Which kernel, and its K splits, by the modelled time in us. A workgroup of
// either (eight waves of about 200 registers) has a CU to itself, so rounds of
// workgroups; a split adds its sums written and read again, and a launch to
// join them.
//   coli_gemm_t: 128 rows and two quads a workgroup, a step of 32 rows of W 1.4
//   us with three products (int4), 0.9 with two (all CUs busy: 2048 x 4096 x
//   14336 and 512 x 7168 x 2048), about eight steps before the first; the dy
//   operands' build 7 us and its bytes. Splits measured: 512 x 4096 x 14336 2 /
//   4 / 8: 285 / 196 / 213 us; 512 x 7168 x 2048 MXFP4 1 / 2 / 3: 83 / 65 / 85.
//   coli_gemm_t_few: eight steps, one a wave, 2.5 us (2.1 with two products),
//   and 8 us. Up to 32 rows it is the faster one at every size; more, while its
//   workgroups fit one round. Both measured, rows x I x O, few / many: int4 160
//   x 6400 x 2176 28 / 42 us, 192 49 / 43; 64 x 14336 x 4096 48 / 67, 66 78 /
//   62; 512 x 768 x 1920 18 / 36; MXFP4 128 x 7168 x 2048 21 / 34, 192 40 / 40;
//   192 x 2048 x 7168 38 / 43, 320 61 / 52.
struct TPlan {
    bool few;
    int splits;
};
static TPlan t_plan(const ColiCudaTensor *t, int S, int cus, int steps) {
    const bool fp4 = t->kind == COLI_KIND_FP4;
    const double mb = (double)S * t->I * 4e-6;
    auto join = [&](int s) { return s > 1 ? (s + 1) * mb / 4 + 3 : 0.0; };
    auto rounds = [&](long blocks) { return (double)((blocks + cus - 1) / cus); };
    const long fb = (long)((S + 31) / 32) * t->nq, mbk = (long)((S + 127) / 128) * ((t->nq + 1) / 2);
    // few: a workgroup a CU, a step for each of its waves at least
    TPlan best = {true, (int)std::max(1L, std::min((long)cus / fb, (long)steps / 8))};
    double least = 8 + (fp4 ? 2.1 : 2.5) * rounds(fb * best.splits) * ((steps + 8 * best.splits - 1) / (8 * best.splits)) + join(best.splits);
    const double prep = 7 + (double)S * t->O * 8e-6 / 4;
    int force = 0;   // COLI_HIP_GEMM_T=few|many pins the kernel (tuning and tests)
    if (const char *e = std::getenv("COLI_HIP_GEMM_T")) force = std::strcmp(e, "few") == 0 ? 1 : (std::strcmp(e, "many") == 0 ? -1 : 0);
    if (force > 0) return best;
    if (force < 0) least = 1e30;
    for (int s = 1; s <= 32 && s * 8 <= std::max(8, steps); s++) {
        const double us = prep + (fp4 ? 0.9 : 1.4) * rounds(mbk * s) * ((steps + s - 1) / s + 8) + join(s);
        if (us < least) {
            least = us;
            best = {false, s};
        }
    }
    return best;
}

int gemm_t_plan(DevCtx *ctx, ColiCudaTensor *t, const float *dy, int S, GemmTPlan *g) {
    *g = GemmTPlan{};
    if (t->kind == COLI_KIND_GENERIC) return 1;
    if (!t->sct && !build_t_scales(ctx, t, false)) return 0;
    const int noct = t_octets(t), steps = noct / 4;
    const TPlan pl = t_plan(t, S, ctx->cu_count ? ctx->cu_count : 256, steps);
    const bool few = pl.few;
    const size_t Sp = few ? 0 : ((size_t)S + 127) & ~(size_t)127, fb = (size_t)noct * Sp * 16;
    int splits = pl.splits;
    const int per = (steps + splits - 1) / splits;
    splits = (steps + per - 1) / per;
    const size_t eb = (Sp * sizeof(int) + 255) & ~(size_t)255;
    const size_t pb = splits > 1 ? (size_t)splits * S * t->I * sizeof(float) : 0;
    const size_t db = t->O < 4 ? (size_t)S * 16 : 0;
    if (2 * fb + eb + pb + db && !reserve_kept(ctx, &ctx->gt, 2 * fb + eb + pb + db, 0)) return 0;
    uint8_t *p = (uint8_t *)ctx->gt.p;
    g->few = few;
    g->splits = splits;
    g->per = per;
    g->part = (float *)(p + 2 * fb + eb);
    g->parts = splits > 1 ? splits : 0;
    ColiTPrepArgs &a = g->prep;
    a.dy = dy;
    if (db) {   // (the kernels load four columns at a time)
        a.dy = (float *)(p + 2 * fb + eb + pb);
        hipLaunchKernelGGL(coli_t_pad, dim3((4 * S + 255) / 256), dim3(256), 0, ctx->stream, dy, (float *)a.dy, S, t->O);
        if (!hip_check(hipGetLastError(), "gradient rows padding")) return 0;
    }
    a.hi = (_Float16 *)p;
    a.lo = (_Float16 *)(p + fb);
    a.exps = (int *)(p + 2 * fb);
    a.Sp = Sp;
    a.S = S;
    a.K = std::max(4, t->O);
    a.noct = noct;
    a.int4 = t->kind != COLI_KIND_FP4;
    a.nblocks = few ? 0 : (S + 3) / 4;
    return 1;
}

int gemm_t_run(DevCtx *ctx, ColiCudaTensor *t, float *dx, const float *dy, int S, const GemmTPlan &g, bool with_join) {
    forget_emitted(ctx, dx, (size_t)S * t->I * sizeof(float));
    hipStream_t st = ctx->stream;
    if (t->kind == COLI_KIND_GENERIC) {
        hipLaunchKernelGGL(coli_t_generic, dim3((t->I + 255) / 256, S), dim3(256), 0, st, t->w, (const float *)t->sc, t->gs,
                           t->ng_src, t->I, t->O, dy, dx);
        return hip_check(hipGetLastError(), "generic gradient");
    }
    if (g.prep.nblocks) {
        hipLaunchKernelGGL(coli_t_prep_rows, dim3(g.prep.nblocks), dim3(1024), 0, st, g.prep);
        if (!hip_check(hipGetLastError(), "gradient rows")) return 0;
    }
    GemmTArgs a = {};
    a.w = t->w;
    a.sct = (const _Float16 *)t->sct;
    a.ge = t->sct_ge;
    a.hi = g.prep.hi;
    a.lo = g.prep.lo;
    a.exps = g.prep.exps;
    a.Sp = g.prep.Sp;
    a.dy = g.prep.dy;
    a.O = g.prep.K;
    a.nrt = t->nrt;
    a.nq = t->nq;
    a.noct = g.prep.noct;
    a.I = t->I;
    a.S = S;
    a.splits = g.splits;
    a.per = g.per;
    a.out = g.parts ? g.part : dx;
    if (t->kind == COLI_KIND_I4_H) launch_gemm_t<COLI_KIND_I4_H>(a, g.few, st);
    else if (t->kind == COLI_KIND_I4_F) launch_gemm_t<COLI_KIND_I4_F>(a, g.few, st);
    else launch_gemm_t<COLI_KIND_FP4>(a, g.few, st);
    if (!hip_check(hipGetLastError(), "input gradient")) return 0;
    if (!with_join || !g.parts) return 1;
    const size_t n = (size_t)S * t->I;
    hipLaunchKernelGGL(coli_t_join, dim3((unsigned)((n + 1023) / 1024)), dim3(256), 0, st, a.out, dx, n, g.splits);
    return hip_check(hipGetLastError(), "input gradient join");
}

extern "C" int coli_hip_gemm_t_dev(ColiCudaTensor *t, float *dx_dev, const float *dy_dev, int S) {
    if (fault_injected()) return 0;
    if (!tensor_computable(t) || !dx_dev || !dy_dev || S < 1 || S > COLI_GRAD_MAX_ROWS ||
        ranges_overlap(dx_dev, (size_t)S * t->I * 4, dy_dev, (size_t)S * t->O * 4))
        return 0;
    DevCtx *ctx = ctx_of(t->device);
    if (!bind_ctx(ctx)) return 0;
    GemmTPlan g;
    return gemm_t_plan(ctx, t, dy_dev, S, &g) && gemm_t_run(ctx, t, dx_dev, dy_dev, S, g, true);
}
