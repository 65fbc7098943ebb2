// balance.hip -- per-expert counts and the load-balance loss of routed rows, by
// sequence, with the gradient of the router's logits.
//
// For sequence i (rows [offsets[i], offsets[i + 1]) that the mask keeps, n_i of
// them) with c_e live selections of expert e, C = sum c_e:
//   p_te  = exp(u(z_te)) / sum_j exp(u(z_tj)),  u(z) = z (softmax routing),
//           log sigmoid(z) (modes 1, 2), 1/2 log softplus(z) (mode 3): the
//           router's scores divided by their sum
//   loss  = sum_e f_e P_e,  f_e = E c_e / C,  P_e = (1 / n_i) sum_t p_te
//   dz_te = p_te (w_e - sum_j w_j p_tj) u'(z_te),  w_e = dloss f_e / n_i
// (the counts carry no gradient). Both passes are bound by the logits' bytes:
// T E 4 read forward, read and written backward.
//
// A row is held by 16 lanes (float4 v of lane l: columns 64 v + 4 l), so a wave
// runs four rows at once, every reduction of a row is four DPP steps, and one
// load instruction of a row group reads 256 contiguous bytes. All sums are f32,
// the counts integers; they are joined in a fixed order (no float atomics).
#include "coli_hip_host.h"
#include "coli_device.h"

#include "coli_backend_abi.h"
#include "coli_hip_ext.h"

#include <algorithm>

#define COLI_BAL_MAX_SEQS 16384
#define COLI_BAL_MAX_ROWS (1 << 24)
// Rows one workgroup finishes alone, loss included.
#define COLI_BAL_SINGLE 128

struct BalanceArgs {
    const float *z;            // [nch][T][E]: logits, or column-chunk partials added in chunk order
    size_t chstride;
    int nch;
    const int *idx, *keff;     // [T][K], [T] or null
    const uint8_t *mask;       // [T] or null
    const int *off;            // [n + 1] or null: one sequence of all rows
    int n, T, E, K, mode, R;   // R: rows per workgroup
    int vec;                   // E % 4 == 0 and every row 16-byte aligned
    float *loss;               // [n]
    int *counts, *rows;        // [n][E], [n]
    // partial sums of workgroup b's rows of sequence i, slot b + i (the pairs
    // (b, i) that share rows are ordered, and b + i grows along them)
    float *ps;                 // [slots][Ep]
    int *pc;                   // [slots][Ep]
    int *pn;                   // [slots][2]: rows, selections
    int Ep;                    // E rounded up to 64
    float *lossp;              // [n][Ep / 64]
    int *arrive;               // [n], zero between launches
    // backward
    const float *dloss;
    float *dz;
};

// Sum over each 16-lane row (DPP: neighbours, pairs, halves of 8, halves of 16).
__device__ __forceinline__ float dpp_sum16(float v) {
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xB1, 0xF, 0xF, false));
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4E, 0xF, 0xF, false));
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x141, 0xF, 0xF, false));
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x140, 0xF, 0xF, false));
}
__device__ __forceinline__ int dpp_sum16i(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x141, 0xF, 0xF, false);
    return v + __builtin_amdgcn_update_dpp(0, v, 0x140, 0xF, 0xF, false);
}

// The row's logits; columns past E read -inf, which every score maps to 0.
template <int NV>
__device__ __forceinline__ void bal_load(const BalanceArgs &a, int row, int l, float (&v)[4 * NV]) {
    const float *zr = a.z + (size_t)row * a.E;
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int e = 64 * i + 4 * l;
        if (a.vec) {
            const floatx4 t = e < a.E ? *GPTR(floatx4, zr + e) : (floatx4){-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int k = 0; k < 4; k++) v[4 * i + k] = t[k];
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++) v[4 * i + k] = e + k < a.E ? zr[e + k] : -INFINITY;
        }
    }
    for (int ch = 1; ch < a.nch; ch++) {
        const float *zc = zr + (size_t)ch * a.chstride;
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (64 * i + 4 * l + k < a.E) v[4 * i + k] += zc[64 * i + 4 * l + k];
    }
}

// v: logits in, p out; with GRAD, up: u'(z). The hardware's exp2, log2, rcp and
// sqrt (1 ulp each) are used: a p is off by a few 2^-23. Scores so small that
// their sum would lose bits (every z below about -27) go by their logarithm
// instead, where both u are linear to within f32: z, or z / 2 in mode 3. A row
// of nothing but -inf has p = 0.
template <int NV, bool GRAD>
__device__ __forceinline__ void bal_prob(int mode, float (&v)[4 * NV], float (&up)[4 * NV]) {
    float z[4 * NV], sum = 0.0f;
#pragma unroll
    for (int k = 0; k < 4 * NV; k++) z[k] = v[k];
    if (mode) {
#pragma unroll
        for (int k = 0; k < 4 * NV; k++) {
            const float t = __expf(-fabsf(z[k])), w = 1.0f + t, r = __builtin_amdgcn_rcpf(w);
            const bool pos = z[k] >= 0.0f;
            const float sg = pos ? r : t * r;
            if (mode == 3) {
                // log(1 + t) = t log(w) / (w - 1): the rounding of w cancels
                const float d = w - 1.0f, lg = d > 0.0f ? t * (__logf(w) * __builtin_amdgcn_rcpf(d)) : t;
                const float sp = (pos ? z[k] : 0.0f) + lg;
                v[k] = __builtin_amdgcn_sqrtf(sp);
                if constexpr (GRAD) up[k] = z[k] < -15.0f ? 0.5f : 0.5f * sg * __builtin_amdgcn_rcpf(sp);
            } else {
                v[k] = sg;
                if constexpr (GRAD) up[k] = pos ? t * r : r;
            }
            if (z[k] != z[k]) v[k] = z[k];
            sum += v[k];
        }
        sum = dpp_sum16(sum);
    }
    if (!mode || sum < 1e-12f) {
        float m = -INFINITY;
#pragma unroll
        for (int k = 0; k < 4 * NV; k++) m = fmaxf(m, z[k]);
        m = dpp_max16(m);
        const float c = mode == 3 ? 0.5f : 1.0f;
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < 4 * NV; k++) {
            // (m = -inf: only -inf and NaN in the row; NaN stays)
            v[k] = z[k] == -INFINITY ? 0.0f : __expf(c * (z[k] - m));
            if constexpr (GRAD)
                if (!mode) up[k] = 1.0f;
            s += v[k];
        }
        sum = dpp_sum16(s);
    }
    const float r = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int k = 0; k < 4 * NV; k++) v[k] *= r;
}

// First sequence that ends after `row`: the offsets up to it, counted by the block.
__device__ __forceinline__ int bal_first(const BalanceArgs &a, int row) {
    if (!a.off) return 0;
    int c = 0;
    for (int j0 = 0; j0 < a.n; j0 += blockDim.x) {
        const int j = j0 + threadIdx.x;
        c += __syncthreads_count(j < a.n && a.off[j + 1] <= row);
    }
    return c;
}
__device__ __forceinline__ int bal_begin(const BalanceArgs &a, int i) {
    return a.off ? min(max(a.off[i], 0), a.T) : 0;
}
__device__ __forceinline__ int bal_end(const BalanceArgs &a, int i) {
    return a.off ? min(max(a.off[i + 1], 0), a.T) : a.T;
}

// Sums of each workgroup's R rows by sequence; with SINGLE (one workgroup for
// all rows) the outputs themselves.
template <int NV, bool SINGLE>
__global__ __launch_bounds__(256) void coli_balance_rows(BalanceArgs a) {
    __shared__ float red[4][64 * NV];
    __shared__ int cnt[64 * NV];
    __shared__ int seg_n[2];
    __shared__ float wsum[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l = lane & 15, g = lane >> 4;
    const int b = blockIdx.x, r0 = b * a.R, r1 = min(a.T, r0 + a.R);
    if constexpr (SINGLE) {
        for (size_t e = tid; e < (size_t)a.n * a.E; e += 256) a.counts[e] = 0;
        for (int i = tid; i < a.n; i += 256) {
            a.loss[i] = 0.0f;
            a.rows[i] = 0;
        }
    }
    int i = bal_first(a, r0);
    int row = i < a.n ? max(r0, bal_begin(a, 0)) : r1;
    if constexpr (SINGLE) __syncthreads();
    while (row < r1 && i < a.n) {
        const int end = bal_end(a, i);
        if (end <= row) {
            i++;
            continue;
        }
        const int hi = min(end, r1);
        for (int e = tid; e < 64 * NV; e += 256) cnt[e] = 0;
        if (tid < 2) seg_n[tid] = 0;
        __syncthreads();
        // selections: (row, slot) pairs over the threads
        int nsel = 0, nrow = 0;
        const int npair = (hi - row) * a.K;
        for (int s = tid; s < npair; s += 256) {
            const int t = row + s / a.K, kk = s - s / a.K * a.K;
            if (a.mask && !a.mask[t]) continue;
            const int e = a.idx[(size_t)t * a.K + kk];
            if (kk < (a.keff ? a.keff[t] : a.K) && e >= 0 && e < a.E) {
                atomicAdd(cnt + e, 1);
                nsel++;
            }
        }
        float acc[4 * NV];
#pragma unroll
        for (int k = 0; k < 4 * NV; k++) acc[k] = 0.0f;
        for (int t0 = row + 4 * wave; t0 < hi; t0 += 16) {
            const int t = t0 + g;
            const bool live = t < hi && (!a.mask || a.mask[t]);
            float v[4 * NV], none[4 * NV];
            bal_load<NV>(a, t < hi ? t : t0, l, v);
            bal_prob<NV, false>(a.mode, v, none);
            if (live) {
                nrow += l == 0;
#pragma unroll
                for (int k = 0; k < 4 * NV; k++) acc[k] += v[k];
            }
        }
        if (nsel) atomicAdd(seg_n + 1, nsel);
        if (nrow) atomicAdd(seg_n, nrow);
#pragma unroll
        for (int k = 0; k < 4 * NV; k++) {
            acc[k] += __shfl_xor(acc[k], 16);
            acc[k] += __shfl_xor(acc[k], 32);
        }
        if (g == 0)
#pragma unroll
            for (int v = 0; v < NV; v++)
                *(floatx4 *)&red[wave][64 * v + 4 * l] =
                    (floatx4){acc[4 * v], acc[4 * v + 1], acc[4 * v + 2], acc[4 * v + 3]};
        __syncthreads();
        const int n = seg_n[0], C = seg_n[1];
        if constexpr (SINGLE) {
            float d = 0.0f;
            for (int e = tid; e < a.E; e += 256) {
                const float P = (red[0][e] + red[1][e]) + (red[2][e] + red[3][e]);
                a.counts[(size_t)i * a.E + e] = cnt[e];
                d += (float)cnt[e] * P;
            }
#pragma unroll
            for (int o = 32; o; o >>= 1) d += __shfl_xor(d, o);
            if (lane == 0) wsum[wave] = d;
            __syncthreads();
            if (tid == 0) {
                a.rows[i] = n;
                a.loss[i] = C && n ? ((wsum[0] + wsum[1]) + (wsum[2] + wsum[3])) * ((float)a.E / (float)C / (float)n) : 0.0f;
            }
        } else {
            const size_t slot = (size_t)(b + i);
            for (int e = tid; e < a.Ep; e += 256) {
                a.ps[slot * a.Ep + e] = (red[0][e] + red[1][e]) + (red[2][e] + red[3][e]);
                a.pc[slot * a.Ep + e] = cnt[e];
            }
            if (tid < 2) a.pn[2 * slot + tid] = seg_n[tid];
        }
        __syncthreads();
        row = hi;
        if (row >= end) i++;
    }
}

// Joins a sequence's partial sums, 64 columns a workgroup (16 lanes of four
// columns x blockDim / 16 groups of slots); the workgroup that arrives last
// adds the loss's pieces in column order.
template <int NT>
__global__ __launch_bounds__(NT) void coli_balance_join(BalanceArgs a) {
    constexpr int G = NT / 16;
    __shared__ floatx4 sp[G][16];
    __shared__ int sc[G][64], sn[G][2];
    const int i = blockIdx.x, eb = blockIdx.y, neb = gridDim.y, tid = threadIdx.x, l = tid & 15, g = tid >> 4;
    const int lo = bal_begin(a, i), hi = bal_end(a, i);
    const int b0 = lo / a.R, b1 = hi > lo ? (hi - 1) / a.R : b0 - 1;
    floatx4 s = (floatx4){0.f, 0.f, 0.f, 0.f};
    int c[4] = {0, 0, 0, 0}, n0 = 0, n1 = 0;
#pragma unroll 4
    for (int b = b0 + g; b <= b1; b += G) {
        const size_t slot = (size_t)(b + i);
        const floatx4 x = *GPTR(floatx4, a.ps + slot * a.Ep + 64 * eb + 4 * l);
        const u32x4 y = *GPTR(u32x4, a.pc + slot * a.Ep + 64 * eb + 4 * l);
        n0 += a.pn[2 * slot];
        n1 += a.pn[2 * slot + 1];
        s += x;
#pragma unroll
        for (int k = 0; k < 4; k++) c[k] += (int)y[k];
    }
    sp[g][l] = s;
#pragma unroll
    for (int k = 0; k < 4; k++) sc[g][4 * l + k] = c[k];
    if (l == 0) {
        sn[g][0] = n0;
        sn[g][1] = n1;
    }
    __syncthreads();
    if (tid < 64) {
        const int e = 64 * eb + tid;
        float P = 0.0f;
        int C = 0, n = 0, cn = 0;
        for (int q = 0; q < G; q++) {
            P += sp[q][tid >> 2][tid & 3];
            cn += sc[q][tid];
            n += sn[q][0];
            C += sn[q][1];
        }
        if (e < a.E) a.counts[(size_t)i * a.E + e] = cn;
        float d = (float)cn * P;
#pragma unroll
        for (int o = 32; o; o >>= 1) d += __shfl_xor(d, o);
        if (tid == 0) {
            const float f = C && n ? (float)a.E / (float)C / (float)n : 0.0f;
            // the first workgroup of the sequence writes the row count; every
            // one publishes its piece and counts itself in
            if (eb == 0) a.rows[i] = n;
            if (neb == 1) {
                a.loss[i] = f != 0.0f ? d * f : 0.0f;
            } else {
                __hip_atomic_store(a.lossp + (size_t)i * neb + eb, d, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                const int at = __hip_atomic_fetch_add(a.arrive + i, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
                if (at == neb - 1) {
                    float t = 0.0f;
                    for (int q = 0; q < neb; q++)
                        t += __hip_atomic_load(a.lossp + (size_t)i * neb + q, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                    a.loss[i] = f != 0.0f ? t * f : 0.0f;
                    __hip_atomic_store(a.arrive + i, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                }
            }
        }
    }
}

// dz of each workgroup's R rows; rows of no sequence are left as they were.
template <int NV>
__global__ __launch_bounds__(256) void coli_balance_grad(BalanceArgs a) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l = lane & 15, g = lane >> 4;
    const int r0 = blockIdx.x * a.R, r1 = min(a.T, r0 + a.R);
    int i = bal_first(a, r0);
    int row = i < a.n ? max(r0, bal_begin(a, 0)) : r1;
    while (row < r1 && i < a.n) {
        const int end = bal_end(a, i);
        if (end <= row) {
            i++;
            continue;
        }
        const int hi = min(end, r1);
        float w[4 * NV];
        int C = 0;
#pragma unroll
        for (int v = 0; v < NV; v++)
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int e = 64 * v + 4 * l + k;
                const int c = e < a.E ? a.counts[(size_t)i * a.E + e] : 0;
                w[4 * v + k] = (float)c;
                C += c;
            }
        C = dpp_sum16i(C);
        const int n = a.rows[i];
        const float f = C > 0 && n > 0 ? a.dloss[i] * ((float)a.E / (float)C / (float)n) : 0.0f;
#pragma unroll
        for (int k = 0; k < 4 * NV; k++) w[k] *= f;
        for (int t0 = row + 4 * wave; t0 < hi; t0 += 16) {
            const int t = t0 + g;
            float v[4 * NV], up[4 * NV];
            bal_load<NV>(a, t < hi ? t : t0, l, v);
            bal_prob<NV, true>(a.mode, v, up);
            float d = 0.0f;
#pragma unroll
            for (int k = 0; k < 4 * NV; k++) d += w[k] * v[k];
            d = dpp_sum16(d);
            const bool live = t < hi && f != 0.0f && (!a.mask || a.mask[t]);
            if (t >= hi) continue;
            float *dr = a.dz + (size_t)t * a.E;
#pragma unroll
            for (int q = 0; q < NV; q++) {
                const int e = 64 * q + 4 * l;
                floatx4 o;
#pragma unroll
                for (int k = 0; k < 4; k++) o[k] = live ? v[4 * q + k] * (w[4 * q + k] - d) * up[4 * q + k] : 0.0f;
                if (a.vec) {
                    if (e < a.E) *(floatx4 *)(dr + e) = o;
                } else {
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        if (e + k < a.E) dr[e + k] = o[k];
                }
            }
        }
        row = hi;
        if (row >= end) i++;
    }
}

static int nv_of(int E) { return E <= 64 ? 1 : E <= 128 ? 2 : E <= 256 ? 4 : E <= 384 ? 6 : E <= 512 ? 8 : 16; }
#define COLI_BAL_NV(E, CALL)          \
    switch (nv_of(E)) {               \
    case 1: CALL(1); break;           \
    case 2: CALL(2); break;           \
    case 4: CALL(4); break;           \
    case 6: CALL(6); break;           \
    case 8: CALL(8); break;           \
    default: CALL(16); break;         \
    }

static bool balance_shape_ok(int n, int T, int E, int mode) {
    return n >= 1 && n <= COLI_BAL_MAX_SEQS && T >= 1 && T <= COLI_BAL_MAX_ROWS && E >= 1 && E <= 1024 && mode >= 0 &&
           mode <= 3;
}

int run_balance(DevCtx *ctx, const float *z, int nch, size_t chstride, const int *idx, const int *keff,
                const uint8_t *mask, const int *off, int n, int T, int E, int K, int mode, float *loss, int *counts,
                int *rows) {
    if (!balance_shape_ok(n, T, E, mode) || K < 1 || K > 64 || K > E) return 0;
    BalanceArgs a = {};
    a.z = z;
    a.nch = nch;
    a.chstride = chstride;
    a.idx = idx;
    a.keff = keff;
    a.mask = mask;
    a.off = off;
    a.n = n;
    a.T = T;
    a.E = E;
    a.K = K;
    a.mode = mode;
    a.vec = E % 4 == 0 && ((uintptr_t)z & 15) == 0;
    a.loss = loss;
    a.counts = counts;
    a.rows = rows;
    forget_emitted(ctx, loss, (size_t)n * sizeof(float));
    forget_emitted(ctx, counts, (size_t)n * E * sizeof(int));
    forget_emitted(ctx, rows, (size_t)n * sizeof(int));
    hipStream_t st = ctx->stream;
    if (T <= COLI_BAL_SINGLE && n <= 64) {
        a.R = T;
#define COLI_BAL_ONE(NV) hipLaunchKernelGGL((coli_balance_rows<NV, true>), dim3(1), dim3(256), 0, st, a)
        COLI_BAL_NV(E, COLI_BAL_ONE)
#undef COLI_BAL_ONE
        return hip_check(hipGetLastError(), "balance");
    }
    // 16 rows a step of a workgroup; about 1024 workgroups once there are rows for them
    a.R = std::max(16, (T + 1023) / 1024 + 15 & ~15);
    const int nb = (T + a.R - 1) / a.R;
    const size_t slots = (size_t)nb + n;
    a.Ep = (E + 63) / 64 * 64;
    const int neb = a.Ep / 64;
    const size_t ps_b = slots * a.Ep * 4, pn_b = (slots * 8 + 255) & ~(size_t)255, lp_b = ((size_t)n * neb * 4 + 255) & ~(size_t)255;
    if (!reserve_kept(ctx, &ctx->bal, 2 * ps_b + pn_b + lp_b, 0) ||
        !reserve_kept(ctx, &ctx->bal_cnt, (size_t)COLI_BAL_MAX_SEQS * sizeof(int), 1))
        return 0;
    uint8_t *p = (uint8_t *)ctx->bal.p;
    a.ps = (float *)p;
    a.pc = (int *)(p + ps_b);
    a.pn = (int *)(p + 2 * ps_b);
    a.lossp = (float *)(p + 2 * ps_b + pn_b);
    a.arrive = (int *)ctx->bal_cnt.p;
#define COLI_BAL_ROWS(NV) hipLaunchKernelGGL((coli_balance_rows<NV, false>), dim3(nb), dim3(256), 0, st, a)
    COLI_BAL_NV(E, COLI_BAL_ROWS)
#undef COLI_BAL_ROWS
    if (!hip_check(hipGetLastError(), "balance rows")) return 0;
    if (nb / n > 16)
        hipLaunchKernelGGL((coli_balance_join<1024>), dim3(n, neb), dim3(1024), 0, st, a);
    else
        hipLaunchKernelGGL((coli_balance_join<256>), dim3(n, neb), dim3(256), 0, st, a);
    return hip_check(hipGetLastError(), "balance join");
}

extern "C" int coli_hip_balance_dev(int device, const float *logits, const int *idx, const int *keff,
                                    const unsigned char *mask, const int *offsets, int n, int T, int E, int K,
                                    int route_mode, float *loss, int *counts, int *rows) {
    if (fault_injected()) return 0;
    if (!logits || !idx || !loss || !counts || !rows || (!offsets && n != 1)) return 0;
    DevCtx *ctx = ctx_of(device);
    if (!bind_ctx(ctx)) return 0;
    return run_balance(ctx, logits, 1, 0, idx, keff, mask, offsets, n, T, E, K, route_mode, loss, counts, rows);
}

extern "C" int coli_hip_balance_grad_dev(int device, const float *logits, const unsigned char *mask,
                                         const int *offsets, int n, int T, int E, int route_mode, const float *dloss,
                                         const int *counts, const int *rows, float *dlogits) {
    if (fault_injected()) return 0;
    if (!logits || !dloss || !counts || !rows || !dlogits || (!offsets && n != 1) ||
        !balance_shape_ok(n, T, E, route_mode))
        return 0;
    DevCtx *ctx = ctx_of(device);
    if (!bind_ctx(ctx)) return 0;
    forget_emitted(ctx, dlogits, (size_t)T * E * sizeof(float));
    BalanceArgs a = {};
    a.z = logits;
    a.nch = 1;
    a.mask = mask;
    a.off = offsets;
    a.n = n;
    a.T = T;
    a.E = E;
    a.mode = route_mode;
    a.vec = E % 4 == 0 && (((uintptr_t)logits | (uintptr_t)dlogits) & 15) == 0;
    a.counts = (int *)counts;
    a.rows = (int *)rows;
    a.dloss = dloss;
    a.dz = dlogits;
    a.R = std::max(16, (T + 2047) / 2048 + 15 & ~15);
    const int nb = (T + a.R - 1) / a.R;
#define COLI_BAL_GRAD(NV) hipLaunchKernelGGL((coli_balance_grad<NV>), dim3(nb), dim3(256), 0, ctx->stream, a)
    COLI_BAL_NV(E, COLI_BAL_GRAD)
#undef COLI_BAL_GRAD
    return hip_check(hipGetLastError(), "balance gradient");
}
