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
// A row is held by L = 16, 32 or 64 lanes (float4 v of lane l: columns 4 L v +
// 4 l), at most sixteen columns a lane, so a wave runs four rows at once up to
// 256 experts, and the reductions of a row are lane permutes on the VALU. All sums are f32,
// the counts integers; they are joined in a fixed order (no float atomics).
//
// Measured, 65536 rows of 384 experts: softmax and sigmoid forward 26 us with the
// join's 7 (101 MB of logits, 20 us of them at 5 TB/s), backward 35 us (201 MB,
// 5.7 TB/s, the logits partly cached); sqrt-softplus, whose four hardware
// functions an element meet the bytes, 36 and 40 us. Rows a workgroup, forward
// (mode 0): 16 / 32 / 64 / 128: 36 / 29 / 26 / 26 us; backward 34 to 36 us for
// all of them. 64 rows of 64 experts: one workgroup, 6.8 us, latency; it takes
// several sequences one after the other, a step of 64 rows each.
#include "coli_hip_host.h"
#include "coli_device.h"

#include "coli_backend_abi.h"
#include "coli_hip_ext.h"

#include <algorithm>
#include <initializer_list>

#define COLI_BAL_MAX_SEQS 16384
#define COLI_BAL_MAX_ROWS (1 << 24)

struct BalanceArgs {
    const float *z;            // [nch][T][E]: logits, or column-chunk partials added in chunk order
    int nch;
    const int *state;          // null, or a MoE layer's state, which holds T and z
    const int *idx, *keff;     // [T][K], [T] or null
    const uint8_t *mask;       // [T] or null
    const int *off;            // [n + 1] or null: one sequence of all rows
    int n, T, E, K, R;         // R: rows per workgroup
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
// Sum, maximum over the L lanes of a row.
template <int L> __device__ __forceinline__ float bal_sum(float v) {
    v = dpp_sum16(v);
    if constexpr (L >= 32) {
        const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    }
    if constexpr (L >= 64) {
        const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(b[0]) + __uint_as_float(b[1]);
    }
    return v;
}
template <int L> __device__ __forceinline__ float bal_max(float v) {
    v = dpp_max16(v);
    if constexpr (L >= 32) v = fmaxf(v, __shfl_xor(v, 16));
    if constexpr (L >= 64) v = fmaxf(v, __shfl_xor(v, 32));
    return v;
}
template <int L> __device__ __forceinline__ int bal_sumi(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x141, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x140, 0xF, 0xF, false);
    if constexpr (L >= 32) v += __shfl_xor(v, 16);
    if constexpr (L >= 64) v += __shfl_xor(v, 32);
    return v;
}

// T and z of the layer's last forward (0 rows: none has run).
__device__ __forceinline__ void bal_last(BalanceArgs &a) {
    if (!a.state) return;
    a.T = a.state[4];
    a.z = *(const float *const *)(a.state + 6);
}

// Columns that every E taking this form has (nv_of): its blocks up to there are whole.
template <int L, int NV> constexpr int bal_whole() {
    return L == 16 ? (NV == 1 ? 0 : 32 * NV) : L == 32 ? (NV == 3 ? 256 : 384) : 512;
}

// The row's logits; columns past E read -inf, which every score maps to 0. No
// lane takes a branch of its own (see row4): four columns a load, moved back
// where they would pass E, and with ROW 1 (E % 4 != 0) shifted to their places
// again; ROW 2 (E < 4): one column a load.
template <int L, int NV, int ROW>
__device__ __forceinline__ void bal_load(const BalanceArgs &a, int row, int l, float (&v)[4 * NV]) {
    const float *zr = a.z + (size_t)row * a.E;
    auto block = [&](const float *p, int i) -> floatx4 {
        const int e = 4 * L * i + 4 * l;
        if constexpr (ROW == 2)
            return (floatx4){p[min(e, a.E - 1)], p[min(e + 1, a.E - 1)], p[min(e + 2, a.E - 1)], p[min(e + 3, a.E - 1)]};
        floatx4 t = *GPTR(f4u, p + min(e, a.E - 4));
        if constexpr (ROW == 1) {
            if (4 * L * (i + 1) > bal_whole<L, NV>()) {
                const int d = e - min(e, a.E - 4);
                const bool d1 = d & 1, d2 = d & 2;
                t = (floatx4){d1 ? t[1] : t[0], d1 ? t[2] : t[1], d1 ? t[3] : t[2], t[3]};
                t = (floatx4){d2 ? t[2] : t[0], d2 ? t[3] : t[1], t[2], t[3]};
            }
        }
        return t;
    };
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const floatx4 t = block(zr, i);
#pragma unroll
        for (int k = 0; k < 4; k++) v[4 * i + k] = t[k];
    }
    for (int ch = 1; ch < a.nch; ch++)
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const floatx4 t = block(zr + (size_t)ch * a.T * a.E, i);
#pragma unroll
            for (int k = 0; k < 4; k++) v[4 * i + k] += t[k];
        }
#pragma unroll
    for (int i = 0; i < NV; i++)
        if (4 * L * (i + 1) > bal_whole<L, NV>()) {
#pragma unroll
            for (int k = 0; k < 4; k++) v[4 * i + k] = 4 * L * i + 4 * l + (ROW ? k : 0) < a.E ? v[4 * i + k] : -INFINITY;
        }
}

// v: the row's logits in; out, scores whose sum over the row (`sum`) they are to
// be divided by: p = v / sum. GRAD: v u'(z) instead, and ws = sum_e w_e v_e, so
// that the row is held once. The hardware's exp2, log2, rcp and rsq (1 ulp each)
// are used, and their rounded arguments count for more the farther a logit lies:
// a p is off by up to about (|z| + 8) 2^-23 of itself (z under the row's maximum
// in mode 0; at z = -20 the library's expf is off by one 2^-23). A score below 2^-126
// is zero. So scores so small that others of the row would be lost beside them, or
// their sum lose bits, go by their logarithm instead, under the row's maximum, where
// both u are linear to within f32: z where all of them are below about -27, z / 2 in
// mode 3 below about -16 (its softplus leaves the normal range at -87, where a
// score e^(z / 2) would still be 2^-24 of the row's at -54).
// A row of nothing but -inf has p = 0.
template <int L, int NV, int MODE, int ROW, bool GRAD>
__device__ __forceinline__ void bal_scores(const BalanceArgs &a, int row, int l, const float *w, float (&v)[4 * NV],
                                           float &sum, float &ws) {
    sum = ws = 0.0f;
    auto add = [&](int k, float s, float up) {
        sum += s;
        if constexpr (GRAD) ws += w[k] * s;
        v[k] = GRAD ? s * up : s;
    };
    if constexpr (MODE == 3) {
#pragma unroll
        for (int k = 0; k < 4 * NV; k++) {
            const float z = v[k], t = __expf(-fabsf(z)), o = 1.0f + t;
            // log(1 + t) = log o + (t - (o - 1)) / o but for the square of o's
            // rounding; 1 / o <= 1 is left out of that last place
            const float sp = fmaxf(z, 0.0f) + (__logf(o) + (t - (o - 1.0f)));
            const float q = __builtin_amdgcn_rsqf(fmaxf(sp, 1e-37f));
            float up = 1.0f;
            if constexpr (GRAD) {
                const float r = __builtin_amdgcn_rcpf(o);
                up = z < -15.0f ? 0.5f : 0.5f * (z >= 0.0f ? r : t * r) * (q * q);
            }
            add(k, z == z ? sp * q : z, up);
        }
    } else if constexpr (MODE == 1) {
#pragma unroll
        for (int k = 0; k < 4 * NV; k++) {
            const float z = v[k], t = __expf(-fabsf(z)), r = __builtin_amdgcn_rcpf(1.0f + t);
            add(k, z >= 0.0f ? r : t * r, z >= 0.0f ? t * r : r);
        }
    }
    if (MODE) sum = bal_sum<L>(sum);
    if (MODE == 0 || sum < (MODE == 3 ? 3e-4f : 1e-12f)) {
        if (MODE) bal_load<L, NV, ROW>(a, row, l, v);
        float m = -INFINITY;
#pragma unroll
        for (int k = 0; k < 4 * NV; k++) m = fmaxf(m, v[k]);
        m = bal_max<L>(m);
        sum = ws = 0.0f;
#pragma unroll
        for (int k = 0; k < 4 * NV; k++) {
            // (m = -inf: only -inf and NaN in the row; NaN stays). u' where every
            // score is small: 1, or 1 / 2 in mode 3.
            const float c = MODE == 3 ? 0.5f : 1.0f;
            add(k, v[k] == -INFINITY ? 0.0f : __expf(c * (v[k] - m)), c);
        }
        sum = bal_sum<L>(sum);
    }
    if constexpr (GRAD) ws = bal_sum<L>(ws);
}

// The sequences' offsets, clamped to the rows; in LDS where they fit (each
// lookup of a row's sequence reads a few, one after the other).
#define COLI_BAL_OFF 1024
struct BalOff {
    const int *lds, *off;
    int n, T;
    __device__ int get(int i) const {
        if (!off) return i ? T : 0;
        return min(max(n < COLI_BAL_OFF ? lds[i] : off[i], 0), T);
    }
};
// First sequence that ends after `row`: the offsets up to it, counted by the block.
__device__ __forceinline__ int bal_first(const BalanceArgs &a, int row, int *s_off) {
    if (!a.off) return 0;
    int c = 0;
    if (threadIdx.x == 0) s_off[0] = a.off[0];
    for (int j0 = 0; j0 < a.n; j0 += blockDim.x) {
        const int j = j0 + threadIdx.x;
        const int o = j < a.n ? a.off[j + 1] : 0;
        if (j < a.n && a.n < COLI_BAL_OFF) s_off[j + 1] = o;
        c += __syncthreads_count(j < a.n && o <= row);
    }
    return c;
}

// Sums of each workgroup's R rows by sequence; with SINGLE (one workgroup for
// all rows, sixteen waves) the outputs themselves. A wave takes 64 / L rows of each
// step from the workgroup's first; the first step's logits are requested before
// the rows' sequences are known.
template <int L, int NV, int MODE, int ROW, bool SINGLE>
__global__ __launch_bounds__(SINGLE ? 1024 : 256, 4) void coli_balance_rows(BalanceArgs a) {
    constexpr int W = SINGLE ? 16 : 4, NT = 64 * W, RW = 64 / L, RS = RW * W, COLS = 4 * L * NV;
    __shared__ float red[W][COLS];
    __shared__ int cnt[COLS];
    __shared__ int seg_n[2], s_off[COLI_BAL_OFF];
    __shared__ float wsum[W];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l = lane % L, g = lane / L;
    bal_last(a);
    const int b = blockIdx.x, r0 = b * a.R, r1 = min(a.T, r0 + a.R);
    float v[4 * NV];
    int have = 0;   // the step whose rows v holds
    const bool none = a.state && r0 >= r1;   // fewer rows than the launch allows for
    if (!none) bal_load<L, NV, ROW>(a, min(r0 + RW * wave + g, r1 - 1), l, v);
    if constexpr (SINGLE) {
        for (int e = tid; e < a.n * a.E; e += NT) a.counts[e] = 0;
        for (int i = tid; i < a.n; i += NT) {
            a.loss[i] = 0.0f;
            a.rows[i] = 0;
        }
    }
    if (none) return;
    int i = bal_first(a, r0, s_off);
    const BalOff off = {s_off, a.off, a.n, a.T};
    if (!a.off || SINGLE) __syncthreads();
    int row = i < a.n ? max(r0, off.get(0)) : r1;
    while (row < r1 && i < a.n) {
        const int end = off.get(i + 1);
        if (end <= row) {
            i++;
            continue;
        }
        const int hi = min(end, r1);
        for (int e = tid; e < COLS; e += NT) cnt[e] = 0;
        if (tid < 2) seg_n[tid] = 0;
        __syncthreads();
        // selections: (row, slot) pairs over the threads
        int nsel = 0, nrow = 0;
        const int npair = (hi - row) * a.K;
        for (int s = tid; s < npair; s += NT) {
            const int t = row + s / a.K, kk = s - s / a.K * a.K;
            const int e = a.idx[(size_t)t * a.K + kk], ke = a.keff ? a.keff[t] : a.K;
            const bool live = !a.mask || a.mask[t];
            if (live && kk < ke && e >= 0 && e < a.E) {
                atomicAdd(cnt + e, 1);
                nsel++;
            }
        }
        float acc[4 * NV];
#pragma unroll
        for (int k = 0; k < 4 * NV; k++) acc[k] = 0.0f;
        for (int s = (row - r0) / RS; r0 + RS * s < hi; s++) {
            const int t = r0 + RS * s + RW * wave + g;
            const bool in = t >= row && t < hi, live = in && (!a.mask || a.mask[t]);
            float sum, ws;
            if (have != s) bal_load<L, NV, ROW>(a, min(t, r1 - 1), l, v);
            bal_scores<L, NV, MODE, ROW, false>(a, min(t, r1 - 1), l, nullptr, v, sum, ws);
            if (live) {
                const float r = sum == 0.0f ? 0.0f : 1.0f / sum;
                nrow += l == 0;
#pragma unroll
                for (int k = 0; k < 4 * NV; k++) acc[k] += v[k] * r;
            }
            have = s + 1;
            if (r0 + RS * have < r1) bal_load<L, NV, ROW>(a, min(t + RS, r1 - 1), l, v);
            else have = -1;
        }
        if (nsel) atomicAdd(seg_n + 1, nsel);
        if (nrow) atomicAdd(seg_n, nrow);
#pragma unroll
        for (int k = 0; k < 4 * NV; k++) {
            if (L < 32) acc[k] += __shfl_xor(acc[k], 16);
            if (L < 64) acc[k] += __shfl_xor(acc[k], 32);
        }
        if (g == 0)
#pragma unroll
            for (int v = 0; v < NV; v++)
                *(floatx4 *)&red[wave][4 * L * v + 4 * l] =
                    (floatx4){acc[4 * v], acc[4 * v + 1], acc[4 * v + 2], acc[4 * v + 3]};
        __syncthreads();
        auto total = [&](int e) {
            float v = red[0][e];
#pragma unroll
            for (int q = 1; q < W; q++) v += red[q][e];
            return v;
        };
        if constexpr (SINGLE) {
            const int n = seg_n[0], C = seg_n[1];
            float d = 0.0f;
            for (int e = tid; e < a.E; e += NT) {
                a.counts[(size_t)i * a.E + e] = cnt[e];
                d += (float)cnt[e] * total(e);
            }
#pragma unroll
            for (int o = 32; o; o >>= 1) d += __shfl_xor(d, o);
            if (lane == 0) wsum[wave] = d;
            __syncthreads();
            if (tid == 0) {
                for (int q = 1; q < W; q++) d += wsum[q];
                a.rows[i] = n;
                a.loss[i] = C && n ? d * ((float)a.E / (float)C / (float)n) : 0.0f;
            }
        } else {
            const size_t slot = (size_t)(b + i);
            for (int e = tid; e < a.Ep; e += NT) {
                a.ps[slot * a.Ep + e] = total(e);
                a.pc[slot * a.Ep + e] = cnt[e];
            }
            if (tid < 2) a.pn[2 * slot + tid] = seg_n[tid];
        }
        __syncthreads();
        row = hi;
        if (row >= end) i++;
    }
}

// Joins a sequence's partial sums. A workgroup (sequence, 64 NB columns) has
// 1024 / (16 NB) groups of slots, each of 16 NB lanes of four columns. With
// all columns in one workgroup the loss is complete; else (a long sequence) the
// one that arrives last adds the pieces in column order.
template <int NB>
__global__ __launch_bounds__(1024) void coli_balance_join(BalanceArgs a) {
    constexpr int L = 16 * NB, G = 1024 / L;
    __shared__ floatx4 sp[G][L];
    __shared__ __attribute__((aligned(16))) int sc[G][4 * L];
    __shared__ int sn[G][2];
    __shared__ float wsum[16];
    const int i = blockIdx.x, eb = blockIdx.y, neb = gridDim.y, tid = threadIdx.x, l = tid % L, g = tid / L;
    bal_last(a);
    const BalOff off = {nullptr, a.off, COLI_BAL_OFF, a.T};
    const int lo = off.get(i), hi = off.get(i + 1);
    const int b0 = lo / a.R, b1 = hi > lo ? (hi - 1) / a.R : b0 - 1;
    const int col = 4 * (L * eb + l);
    floatx4 s = (floatx4){0.f, 0.f, 0.f, 0.f};
    u32x4 c = (u32x4){0u, 0u, 0u, 0u};
    int n0 = 0, n1 = 0;
    if (g < G && col < a.Ep) {
        for (int b = b0 + g; b <= b1; b += 4 * G) {
            floatx4 x[4];
            u32x4 y[4];
            int m0[4], m1[4];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const size_t slot = (size_t)(min(b + u * G, b1) + i);
                x[u] = *GPTR(floatx4, a.ps + slot * a.Ep + col);
                y[u] = *GPTR(u32x4, a.pc + slot * a.Ep + col);
                m0[u] = a.pn[2 * slot];
                m1[u] = a.pn[2 * slot + 1];
            }
#pragma unroll
            for (int u = 0; u < 4; u++)
                if (b + u * G <= b1) {
                    s += x[u];
                    c += y[u];
                    n0 += m0[u];
                    n1 += m1[u];
                }
        }
    }
    if (g < G) {
        sp[g][l] = s;
        *(u32x4 *)&sc[g][4 * l] = c;
        if (l == 0) {
            sn[g][0] = n0;
            sn[g][1] = n1;
        }
    }
    __syncthreads();
    float d = 0.0f;
    for (int e = tid; e < 4 * L; e += 1024) {
        float P = 0.0f;
        int cn = 0;
#pragma unroll
        for (int q = 0; q < G; q++) {
            P += ((const float *)sp[q])[e];
            cn += sc[q][e];
        }
        if (4 * L * eb + e < a.E) a.counts[(size_t)i * a.E + 4 * L * eb + e] = cn;
        d += (float)cn * P;
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) d += __shfl_xor(d, o);
    if ((tid & 63) == 0) wsum[tid >> 6] = d;
    __syncthreads();
    if (tid) return;
    int n = 0, C = 0;
    for (int q = 0; q < G; q++) {
        n += sn[q][0];
        C += sn[q][1];
    }
    for (int q = 1; q < 16; q++) d += wsum[q];
    const float f = C && n ? (float)a.E / (float)C / (float)n : 0.0f;
    if (eb == 0) a.rows[i] = n;
    if (neb > 1) {
        // publish the piece where every XCD sees it, then count it in
        __hip_atomic_store(a.lossp + (size_t)i * neb + eb, d, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const int at = __hip_atomic_fetch_add(a.arrive + i, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
        if (at != neb - 1) return;
        d = 0.0f;
        for (int q = 0; q < neb; q++)
            d += __hip_atomic_load(a.lossp + (size_t)i * neb + q, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(a.arrive + i, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    a.loss[i] = f != 0.0f ? d * f : 0.0f;
}

// dz of each workgroup's R rows; rows of no sequence are left as they were.
template <int L, int NV, int MODE, int ROW>
__global__ __launch_bounds__(256, 4) void coli_balance_grad(BalanceArgs a) {
    constexpr int RW = 64 / L, RS = 4 * RW;
    __shared__ int s_off[COLI_BAL_OFF];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l = lane % L, g = lane / L;
    const int r0 = blockIdx.x * a.R, r1 = min(a.T, r0 + a.R);
    float v[4 * NV];
    int have = 0;   // the step whose rows v holds
    bal_load<L, NV, ROW>(a, min(r0 + RW * wave + g, r1 - 1), l, v);
    int i = bal_first(a, r0, s_off);
    const BalOff off = {s_off, a.off, a.n, a.T};
    int row = i < a.n ? max(r0, off.get(0)) : r1;
    while (row < r1 && i < a.n) {
        const int end = off.get(i + 1);
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
                const int e = 4 * L * v + 4 * l + k;
                const int c = e < a.E ? a.counts[(size_t)i * a.E + e] : 0;
                w[4 * v + k] = (float)c;
                C += c;
            }
        C = bal_sumi<L>(C);
        const int n = a.rows[i];
        const float f = C > 0 && n > 0 ? a.dloss[i] * ((float)a.E / (float)C / (float)n) : 0.0f;
#pragma unroll
        for (int k = 0; k < 4 * NV; k++) w[k] *= f;
        for (int s = (row - r0) / RS; r0 + RS * s < hi; s++) {
            const int t = r0 + RS * s + RW * wave + g;
            const bool in = t >= row && t < hi, live = in && f != 0.0f && (!a.mask || a.mask[t]);
            float sum, ws;
            if (have != s) bal_load<L, NV, ROW>(a, min(t, r1 - 1), l, v);
            have = -1;
            bal_scores<L, NV, MODE, ROW, true>(a, min(t, r1 - 1), l, w, v, sum, ws);
            const float r = sum == 0.0f ? 0.0f : 1.0f / sum, d = ws * r;
            if (!in) continue;
            float *dr = a.dz + (size_t)t * a.E;
#pragma unroll
            for (int q = 0; q < NV; q++) {
                const int e = 4 * L * q + 4 * l;
                floatx4 o;
#pragma unroll
                for (int k = 0; k < 4; k++) o[k] = live ? v[4 * q + k] * r * (w[4 * q + k] - d) : 0.0f;
                if (e + 4 <= a.E) {
                    *(f4u *)(dr + e) = o;
                } else {
#pragma unroll
                    for (int k = 0; k < 3; k++)
                        if (e + k < a.E) dr[e + k] = o[k];
                }
            }
        }
        row = hi;
        if (row >= end) i++;
    }
}

// (modes 1 and 2 score alike)
#define COLI_BAL_SCORE(mode, CALL, L, NV, ROW) \
    if ((mode) == 0) CALL(L, NV, 0, ROW);      \
    else if ((mode) == 3) CALL(L, NV, 3, ROW); \
    else CALL(L, NV, 1, ROW)
#define COLI_BAL_MODE(mode, CALL, L, NV)                           \
    if (a.E % 4 == 0) { COLI_BAL_SCORE(mode, CALL, L, NV, 0); }    \
    else { COLI_BAL_SCORE(mode, CALL, L, NV, 1); }
// lanes a row and float4 a lane (bal_whole knows the ranges)
#define COLI_BAL_CALL(mode, CALL)                                                    \
    if (a.E < 4) { COLI_BAL_SCORE(mode, CALL, 16, 1, 2); }                           \
    else if (a.E <= 64) { COLI_BAL_MODE(mode, CALL, 16, 1) }                         \
    else if (a.E <= 128) { COLI_BAL_MODE(mode, CALL, 16, 2) }                        \
    else if (a.E <= 256) { COLI_BAL_MODE(mode, CALL, 16, 4) }                        \
    else if (a.E <= 384) { COLI_BAL_MODE(mode, CALL, 32, 3) }                        \
    else if (a.E <= 512) { COLI_BAL_MODE(mode, CALL, 32, 4) }                        \
    else { COLI_BAL_MODE(mode, CALL, 64, 4) }

static bool balance_shape_ok(int n, int T, int E, int mode) {
    return n >= 1 && n <= COLI_BAL_MAX_SEQS && T >= 1 && T <= COLI_BAL_MAX_ROWS && E >= 1 && E <= 1024 && mode >= 0 &&
           mode <= 3;
}

int run_balance(DevCtx *ctx, const float *z, int nch, const int *idx, const int *keff, const uint8_t *mask,
                const int *off, int n, int T, int E, int K, int mode, float *loss, int *counts, int *rows,
                const BalanceLast *last) {
    const size_t rows4 = (size_t)T * 4;
    if (!balance_shape_ok(n, T, E, mode) || K < 1 || K > 64 || K > E ||
        !outputs_apart({{loss, (size_t)n * 4}, {counts, (size_t)n * E * 4}, {rows, (size_t)n * 4}, {z, rows4 * E}, {idx, rows4 * K},
                        {keff, rows4}, {mask, last ? 1 : (size_t)T}, {off, (size_t)(n + 1) * 4}}, 3))
        return 0;   // (last: the mask may be shorter than the guess)
    BalanceArgs a = {};
    a.z = z;
    a.nch = nch;
    a.state = last ? last->state : nullptr;
    a.idx = idx;
    a.keff = keff;
    a.mask = mask;
    a.off = off;
    a.n = n;
    a.T = T;
    a.E = E;
    a.K = K;
    a.loss = loss;
    a.counts = counts;
    a.rows = rows;
    forget_emitted(ctx, loss, (size_t)n * sizeof(float));
    forget_emitted(ctx, counts, (size_t)n * E * sizeof(int));
    forget_emitted(ctx, rows, (size_t)n * sizeof(int));
    hipStream_t st = ctx->stream;
    const int most = last ? last->max_rows : T;   // rows that the launches must hold for
    // up to four steps of one workgroup: one launch, loss included
    if (T <= (E <= 256 ? 256 : E <= 512 ? 128 : 64) && n <= 64) {
        a.R = most;
#define COLI_BAL_ONE(L, NV, M, ROW) hipLaunchKernelGGL((coli_balance_rows<L, NV, M, ROW, true>), dim3(1), dim3(1024), 0, st, a)
        COLI_BAL_CALL(mode, COLI_BAL_ONE)
#undef COLI_BAL_ONE
        return hip_check(hipGetLastError(), "balance");
    }
    // 16 rows a step of a workgroup; about 1024 workgroups once there are rows for them
    a.R = std::max(16, (most + 1023) / 1024 + 15 & ~15);
    const int nb = (most + a.R - 1) / a.R;
    const size_t slots = (size_t)nb + n;
    a.Ep = (E + 63) / 64 * 64;
    // slots of a sequence: few, one workgroup adds all its columns; many, one for each 64
    const bool many = nb / n > 64;
    const int neb = many ? a.Ep / 64 : 1;
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
#define COLI_BAL_ROWS(L, NV, M, ROW) hipLaunchKernelGGL((coli_balance_rows<L, NV, M, ROW, false>), dim3(nb), dim3(256), 0, st, a)
    COLI_BAL_CALL(mode, COLI_BAL_ROWS)
#undef COLI_BAL_ROWS
    if (!hip_check(hipGetLastError(), "balance rows")) return 0;
#define COLI_BAL_JOIN(NB) hipLaunchKernelGGL((coli_balance_join<NB>), dim3(n, neb), dim3(1024), 0, st, a)
    if (many || E <= 64) COLI_BAL_JOIN(1);
    else if (E <= 128) COLI_BAL_JOIN(2);
    else if (E <= 256) COLI_BAL_JOIN(4);
    else if (E <= 384) COLI_BAL_JOIN(6);
    else if (E <= 512) COLI_BAL_JOIN(8);
    else COLI_BAL_JOIN(16);
#undef COLI_BAL_JOIN
    return hip_check(hipGetLastError(), "balance join");
}

extern "C" int coli_hip_balance_dev(int device, const float *logits, const int *idx, const int *keff,
                                    const unsigned char *mask, const int *offsets, int n, int T, int E, int K,
                                    int route_mode, float *loss, int *counts, int *rows) {
    if (fault_injected()) return 0;
    if (!logits || !idx || !loss || !counts || !rows || (!offsets && n != 1)) return 0;
    DevCtx *ctx = ctx_of(device);
    if (!bind_ctx(ctx)) return 0;
    return run_balance(ctx, logits, 1, idx, keff, mask, offsets, n, T, E, K, route_mode, loss, counts, rows);
}

extern "C" int coli_hip_balance_grad_dev(int device, const float *logits, const unsigned char *mask,
                                         const int *offsets, int n, int T, int E, int route_mode, const float *dloss,
                                         const int *counts, const int *rows, float *dlogits) {
    if (fault_injected()) return 0;
    if (!logits || !dloss || !counts || !rows || !dlogits || (!offsets && n != 1) ||
        !balance_shape_ok(n, T, E, route_mode) ||
        (dlogits != logits && ranges_overlap(dlogits, (size_t)T * E * 4, logits, (size_t)T * E * 4)) ||
        !outputs_apart({{dlogits, (size_t)T * E * 4}, {mask, (size_t)T}, {offsets, (size_t)(n + 1) * 4}, {dloss, (size_t)n * 4},
                        {counts, (size_t)n * E * 4}, {rows, (size_t)n * 4}}, 1))
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
    a.counts = (int *)counts;
    a.rows = (int *)rows;
    a.dloss = dloss;
    a.dz = dlogits;
    a.R = std::max(16, (T + 2047) / 2048 + 15 & ~15);
    const int nb = (T + a.R - 1) / a.R;
#define COLI_BAL_GRAD(L, NV, M, ROW) hipLaunchKernelGGL((coli_balance_grad<L, NV, M, ROW>), dim3(nb), dim3(256), 0, ctx->stream, a)
    COLI_BAL_CALL(route_mode, COLI_BAL_GRAD)
#undef COLI_BAL_GRAD
    return hip_check(hipGetLastError(), "balance gradient");
}
